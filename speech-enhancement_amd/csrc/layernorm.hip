// Layer norm over the last axis, forward and backward, fp32 / bf16 / fp16 storage with fp32 arithmetic.
//
//   mu = sum_c x / C,  var = sum_c (x - mu)^2 / C,  s = 1 / sqrt(var + eps),  h = (x - mu) s,  y = h w + b
//   a = dy w,  dx = s (a - mean_c(a) - h mean_c(a h)),  dw_c = sum_r dy h,  db_c = sum_r dy
//
// Bound by memory: the forward reads x and writes y, the backward reads x and dy and writes dx, each once. A row
// lies in the registers of NT threads (16, 64, 256 or 1024; 16 elements a thread), so the mean, then the squared
// deviations from it (no cancelling difference of two large sums) and the output all come from one read. The
// weight's and bias's gradients are sums over rows: every thread adds its columns of the rows that its block
// takes in registers, the block's row groups are added in order through LDS, each block writes one partial row, and
// ln_finish_kernel adds those in order: no atomics, the same bits every time.
#include "common.hpp"

#include <algorithm>

namespace {

constexpr int kElems = 16;   // elements of a row that one thread holds

template <typename T, int V> struct alignas(sizeof(T) * V) Pack { T v[V]; };

struct LnArgs {
  const void* x;
  const void* dy;
  const void* w;      // may be NULL (1)
  const void* b;      // may be NULL (0)
  void* out;          // y or dx, rows of C
  float* save;        // [2][rows]: mean, 1 / sqrt(var + eps); may be NULL in the forward
  float* part;        // [grid][2][C] (backward with gradients of w / b), or NULL
  long long rows, sx, sdy;
  int C, wf32;        // wf32: w and b are fp32 beside a 16-bit x
  float eps, inv_c;
};

template <typename T, int V>
__device__ __forceinline__ void load_vec(const void* p, long long at, bool f32, float (&v)[V]) {
  if (f32) {
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = static_cast<const float*>(p)[at + j];
  } else {
    const Pack<T, V> t = *reinterpret_cast<const Pack<T, V>*>(static_cast<const T*>(p) + at);
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = (float)t.v[j];
  }
}

template <typename T, int V>
__device__ __forceinline__ void store_vec(T* p, const float (&v)[V]) {
  Pack<T, V> t;
#pragma unroll
  for (int j = 0; j < V; ++j) t.v[j] = (T)v[j];
  *reinterpret_cast<Pack<T, V>*>(p) = t;
}

// Sums of N values over the NT threads of a row, left in all of them. NT > 64: the block is one row group; `red`
// alternates between two halves from call to call, so one barrier a call is enough.
template <int NT, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float* red, int& flip) {
#pragma unroll
  for (int o = (NT < 64 ? NT : 64) / 2; o > 0; o >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor(v[i], o, 64);
  if constexpr (NT > 64) {
    constexpr int NW = NT / 64;
    float* r = red + flip * (2 * 16);
    flip ^= 1;
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int i = 0; i < N; ++i) r[i * 16 + (threadIdx.x >> 6)] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float s = 0.f;
#pragma unroll
      for (int k = 0; k < NW; ++k) s += r[i * 16 + k];
      v[i] = s;
    }
  }
}

template <typename T, int V, int NT>
__global__ void __launch_bounds__(NT > 256 ? NT : 256) ln_fwd_kernel(const LnArgs a) {
  constexpr int NB = NT > 256 ? NT : 256, RPB = NB / NT, IT = kElems / V;
  __shared__ float red[2 * 2 * 16];
  int flip = 0;
  const int t = threadIdx.x % NT, g = threadIdx.x / NT;
  T* y = static_cast<T*>(a.out);
  float w[IT][V], b[IT][V];   // the thread's columns, for all its rows
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    const int c = (i * NT + t) * V;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      w[i][j] = 1.f;
      b[i][j] = 0.f;
    }
    if (a.w && c < a.C) load_vec<T, V>(a.w, c, a.wf32, w[i]);
    if (a.b && c < a.C) load_vec<T, V>(a.b, c, a.wf32, b[i]);
  }
  for (long long r0 = (long long)blockIdx.x * RPB; r0 < a.rows; r0 += (long long)gridDim.x * RPB) {
    const long long row = r0 + g;
    const bool on = row < a.rows;
    float x[IT][V], s[1] = {0.f};
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int c = (i * NT + t) * V;
#pragma unroll
      for (int j = 0; j < V; ++j) x[i][j] = 0.f;
      if (on && c < a.C) load_vec<T, V>(a.x, row * a.sx + c, false, x[i]);
#pragma unroll
      for (int j = 0; j < V; ++j) s[0] += x[i][j];
    }
    row_sum<NT, 1>(s, red, flip);
    const float mean = s[0] * a.inv_c;
    s[0] = 0.f;
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int c = (i * NT + t) * V;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        x[i][j] = c < a.C ? x[i][j] - mean : 0.f;
        s[0] += x[i][j] * x[i][j];
      }
    }
    row_sum<NT, 1>(s, red, flip);
    const float rstd = 1.f / sqrtf(s[0] * a.inv_c + a.eps);
    if (a.save && on && t == 0) {
      a.save[row] = mean;
      a.save[a.rows + row] = rstd;
    }
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int c = (i * NT + t) * V;
      if (!on || c >= a.C) continue;
      float o[V];
#pragma unroll
      for (int j = 0; j < V; ++j) o[j] = x[i][j] * rstd * w[i][j] + b[i][j];
      store_vec<T, V>(y + row * a.C + c, o);
    }
  }
}

template <typename T, int V, int NT>
__global__ void __launch_bounds__(NT > 256 ? NT : 256) ln_bwd_kernel(const LnArgs a) {
  constexpr int NB = NT > 256 ? NT : 256, RPB = NB / NT, IT = kElems / V;
  __shared__ float red[2 * 2 * 16];
  __shared__ float sum[RPB > 1 ? 2 * NT * kElems : 1];
  int flip = 0;
  const int t = threadIdx.x % NT, g = threadIdx.x / NT;
  T* dx = static_cast<T*>(a.out);
  float w[IT][V], aw[IT][V], ab[IT][V];
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    const int c = (i * NT + t) * V;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      w[i][j] = 1.f;
      aw[i][j] = ab[i][j] = 0.f;
    }
    if (a.w && c < a.C) load_vec<T, V>(a.w, c, a.wf32, w[i]);
  }
  for (long long r0 = (long long)blockIdx.x * RPB; r0 < a.rows; r0 += (long long)gridDim.x * RPB) {
    const long long row = r0 + g;
    const bool on = row < a.rows;
    const float mean = on ? a.save[row] : 0.f, rstd = on ? a.save[a.rows + row] : 0.f;
    float h[IT][V], d[IT][V], s[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int c = (i * NT + t) * V;
#pragma unroll
      for (int j = 0; j < V; ++j) h[i][j] = d[i][j] = 0.f;
      if (on && c < a.C) {
        load_vec<T, V>(a.x, row * a.sx + c, false, h[i]);
        load_vec<T, V>(a.dy, row * a.sdy + c, false, d[i]);
#pragma unroll
        for (int j = 0; j < V; ++j) h[i][j] = (h[i][j] - mean) * rstd;
      }
#pragma unroll
      for (int j = 0; j < V; ++j) {
        aw[i][j] += d[i][j] * h[i][j];
        ab[i][j] += d[i][j];
        d[i][j] *= w[i][j];
        s[0] += d[i][j];
        s[1] += d[i][j] * h[i][j];
      }
    }
    if (a.out) {
      row_sum<NT, 2>(s, red, flip);
      const float m0 = s[0] * a.inv_c, m1 = s[1] * a.inv_c;
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        const int c = (i * NT + t) * V;
        if (!on || c >= a.C) continue;
        float o[V];
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] = rstd * (d[i][j] - m0 - h[i][j] * m1);
        store_vec<T, V>(dx + row * a.C + c, o);
      }
    }
  }
  if (!a.part) return;
  float* part = a.part + (long long)blockIdx.x * 2 * a.C;
  if constexpr (RPB > 1) {   // the row groups of the block, added in order
    for (int k = 0; k < RPB; ++k) {
      if (g == k)
#pragma unroll
        for (int i = 0; i < IT; ++i)
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const int c = (i * NT + t) * V + j;
            sum[c] = k ? sum[c] + aw[i][j] : aw[i][j];
            sum[NT * kElems + c] = k ? sum[NT * kElems + c] + ab[i][j] : ab[i][j];
          }
      __syncthreads();
    }
    for (int c = threadIdx.x; c < a.C; c += NB) {
      part[c] = sum[c];
      part[a.C + c] = sum[NT * kElems + c];
    }
  } else {
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int c = (i * NT + t) * V;
      if (c >= a.C) continue;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        part[c + j] = aw[i][j];
        part[a.C + c + j] = ab[i][j];
      }
    }
  }
}

// Rows wider than 1024 threads hold (16384): three passes over the row, which the L2 keeps, one element a load. Not
// made fast: 2048 x 20000 fp32 forward 111 us (3.0 TB/s), 2048 x 40000 bf16 270 us (1.2 TB/s).
template <typename T>
__global__ void __launch_bounds__(1024) ln_fwd_wide_kernel(const LnArgs a) {
  __shared__ float red[2 * 2 * 16];
  int flip = 0;
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + row * a.sx;
    T* y = static_cast<T*>(a.out) + row * a.C;
    float s[1] = {0.f};
    for (int c = threadIdx.x; c < a.C; c += 1024) s[0] += (float)x[c];
    row_sum<1024, 1>(s, red, flip);
    const float mean = s[0] * a.inv_c;
    s[0] = 0.f;
    for (int c = threadIdx.x; c < a.C; c += 1024) {
      const float d = (float)x[c] - mean;
      s[0] += d * d;
    }
    row_sum<1024, 1>(s, red, flip);
    const float rstd = 1.f / sqrtf(s[0] * a.inv_c + a.eps);
    if (a.save && threadIdx.x == 0) {
      a.save[row] = mean;
      a.save[a.rows + row] = rstd;
    }
    for (int c = threadIdx.x; c < a.C; c += 1024) {
      float w[1] = {1.f}, b[1] = {0.f};
      if (a.w) load_vec<T, 1>(a.w, c, a.wf32, w);
      if (a.b) load_vec<T, 1>(a.b, c, a.wf32, b);
      y[c] = (T)(((float)x[c] - mean) * rstd * w[0] + b[0]);
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(1024) ln_bwd_wide_kernel(const LnArgs a) {
  __shared__ float red[2 * 2 * 16];
  int flip = 0;
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + row * a.sx;
    const T* dy = static_cast<const T*>(a.dy) + row * a.sdy;
    T* dx = static_cast<T*>(a.out) + row * a.C;
    const float mean = a.save[row], rstd = a.save[a.rows + row];
    float s[2] = {0.f, 0.f}, w[1] = {1.f};
    for (int c = threadIdx.x; c < a.C; c += 1024) {
      if (a.w) load_vec<T, 1>(a.w, c, a.wf32, w);
      const float d = (float)dy[c] * w[0];
      s[0] += d;
      s[1] += d * (((float)x[c] - mean) * rstd);
    }
    row_sum<1024, 2>(s, red, flip);
    const float m0 = s[0] * a.inv_c, m1 = s[1] * a.inv_c;
    for (int c = threadIdx.x; c < a.C; c += 1024) {
      if (a.w) load_vec<T, 1>(a.w, c, a.wf32, w);
      dx[c] = (T)(rstd * ((float)dy[c] * w[0] - m0 - ((float)x[c] - mean) * rstd * m1));
    }
  }
}

// dw / db of wide rows: one thread a column, block y the rows y, y + gridDim.y, ...
template <typename T>
__global__ void __launch_bounds__(256) ln_cols_wide_kernel(const LnArgs a) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= a.C) return;
  float sw = 0.f, sb = 0.f;
  for (long long row = blockIdx.y; row < a.rows; row += gridDim.y) {
    const float d = (float)static_cast<const T*>(a.dy)[row * a.sdy + c];
    sb += d;
    sw += d * (((float)static_cast<const T*>(a.x)[row * a.sx + c] - a.save[row]) * a.save[a.rows + row]);
  }
  float* part = a.part + (long long)blockIdx.y * 2 * a.C;
  part[c] = sw;
  part[a.C + c] = sb;
}

// dw (blockIdx.y 0) and db (1): the partial rows, 16 slices of them a column, each slice in row order, then the
// slices in order
template <typename T>
__global__ void __launch_bounds__(1024) ln_finish_kernel(const float* __restrict__ part, int parts, int C, int wf32,
                                                         void* dw, void* db) {
  __shared__ float s[16][64];
  const int l = threadIdx.x & 63, k = threadIdx.x >> 6, c = blockIdx.x * 64 + l;
  void* out = blockIdx.y ? db : dw;
  if (!out) return;
  const int per = (parts + 15) / 16, p0 = k * per, p1 = min(parts, p0 + per);
  const float* p = part + (long long)blockIdx.y * C + c;
  float v = 0.f;
  if (c < C)
#pragma unroll 8
    for (int i = p0; i < p1; ++i) v += p[(long long)i * 2 * C];
  s[k][l] = v;
  __syncthreads();
  if (k || c >= C) return;
  for (int i = 1; i < 16; ++i) v += s[i][l];
  if (wf32) static_cast<float*>(out)[c] = v;
  else static_cast<T*>(out)[c] = (T)v;
}

// V and NT of a row: V by the alignment of every pointer and row start, NT the smallest that holds the row
struct LnPlan {
  int V, NT;   // NT 0: wider than the registers of 1024 threads
};

LnPlan plan_of(int C, int es, bool al16, bool al2) {   // al2: aligned to two elements
  LnPlan p;
  p.V = al16 ? 16 / es : al2 ? 2 : 1;
  p.NT = 0;
  for (int nt : {16, 64, 256, 1024})
    if (!p.NT && (long long)nt * kElems >= C) p.NT = nt;
  return p;
}

inline bool aligned(const void* p, long long stride_bytes, int n) {
  return ((uintptr_t)p % n) == 0 && stride_bytes % n == 0;
}

// Workgroups that stay, each with its columns' weights in registers (read for every row they made the forward at 32768 x 4096
// bf16 130 us). 1536 (six a CU) and 1024 were chosen at that size (256 threads a row); 768, 1024, 1536 and 2048 forward,
// 512, 768, 1024 and 2048 backward take, in us:
//   threads  rows x columns       forward             backward
//   16       65536 x 64 bf16      9   8   7   8       17  17  19  27
//   64       25792 x 514 fp32     19  19  20  20      42  39  37  43
//   64       65536 x 200 bf16     15  14  12  14      26  26  27  37
//   256      32768 x 4096 bf16    142 120 103 123     184 160 167 193
//   1024     4096 x 16384 bf16    54  70  57  59      105 133 127 178   (a third of them forward, half backward)
constexpr int kFwdGroups = 1536;
constexpr int kMaxParts = 1024;

// partial rows of the backward: the grid of ln_bwd_kernel
int parts_of(long long rows, int C) {
  const LnPlan p = plan_of(C, 4, true, true);
  const int rpb = p.NT && p.NT < 256 ? 256 / p.NT : 1;
  const int most = p.NT == 1024 || !p.NT ? kMaxParts / 2 : kMaxParts;
  return (int)std::max<long long>(1, std::min<long long>((rows + rpb - 1) / rpb, most));
}

template <typename T, int V>
void launch_fwd(const LnArgs& a, int NT, unsigned grid, hipStream_t st) {
  if (NT == 16) hipLaunchKernelGGL((ln_fwd_kernel<T, V, 16>), dim3(grid), dim3(256), 0, st, a);
  else if (NT == 64) hipLaunchKernelGGL((ln_fwd_kernel<T, V, 64>), dim3(grid), dim3(256), 0, st, a);
  else if (NT == 256) hipLaunchKernelGGL((ln_fwd_kernel<T, V, 256>), dim3(grid), dim3(256), 0, st, a);
  else hipLaunchKernelGGL((ln_fwd_kernel<T, V, 1024>), dim3(grid), dim3(1024), 0, st, a);
}

template <typename T, int V>
void launch_bwd(const LnArgs& a, int NT, unsigned grid, hipStream_t st) {
  if (NT == 16) hipLaunchKernelGGL((ln_bwd_kernel<T, V, 16>), dim3(grid), dim3(256), 0, st, a);
  else if (NT == 64) hipLaunchKernelGGL((ln_bwd_kernel<T, V, 64>), dim3(grid), dim3(256), 0, st, a);
  else if (NT == 256) hipLaunchKernelGGL((ln_bwd_kernel<T, V, 256>), dim3(grid), dim3(256), 0, st, a);
  else hipLaunchKernelGGL((ln_bwd_kernel<T, V, 1024>), dim3(grid), dim3(1024), 0, st, a);
}

template <typename T>
int run_fwd(const LnArgs& a, hipStream_t st) {
  constexpr int es = sizeof(T), we = 16 / es;
  const long long ce = (long long)a.C * es;
  auto all = [&](int n) {
    return aligned(a.x, a.sx * es, n) && aligned(a.out, ce, n) && ce % n == 0 &&
           (a.wf32 || (aligned(a.w, 0, n) && aligned(a.b, 0, n)));
  };
  const LnPlan p = plan_of(a.C, es, all(16), all(2 * es));
  if (!p.NT) {
    hipLaunchKernelGGL(ln_fwd_wide_kernel<T>, dim3((unsigned)std::min<long long>(a.rows, 1024)), dim3(1024), 0, st, a);
  } else {
    const int rpb = p.NT < 256 ? 256 / p.NT : 1;
    const unsigned grid = (unsigned)std::min<long long>((a.rows + rpb - 1) / rpb, p.NT == 1024 ? kFwdGroups / 3 : kFwdGroups);
    if (p.V == we) launch_fwd<T, we>(a, p.NT, grid, st);
    else if (p.V == 2) launch_fwd<T, 2>(a, p.NT, grid, st);
    else launch_fwd<T, 1>(a, p.NT, grid, st);
  }
  SE_LAUNCH_CHECK();
  return SE_OK;
}

template <typename T>
int run_bwd(const LnArgs& a, int parts, void* dw, void* db, hipStream_t st) {
  constexpr int es = sizeof(T), we = 16 / es;
  const long long ce = (long long)a.C * es;
  auto all = [&](int n) {
    return aligned(a.x, a.sx * es, n) && aligned(a.dy, a.sdy * es, n) && aligned(a.out, ce, n) && ce % n == 0 &&
           (a.wf32 || aligned(a.w, 0, n));
  };
  const LnPlan p = plan_of(a.C, es, all(16), all(2 * es));
  if (!p.NT) {
    if (a.out) {
      hipLaunchKernelGGL(ln_bwd_wide_kernel<T>, dim3((unsigned)std::min<long long>(a.rows, 1024)), dim3(1024), 0, st, a);
      SE_LAUNCH_CHECK();
    }
    if (a.part)
      hipLaunchKernelGGL(ln_cols_wide_kernel<T>, dim3(se::ceil_div(a.C, 256), parts), dim3(256), 0, st, a);
  } else {
    if (p.V == we) launch_bwd<T, we>(a, p.NT, parts, st);
    else if (p.V == 2) launch_bwd<T, 2>(a, p.NT, parts, st);
    else launch_bwd<T, 1>(a, p.NT, parts, st);
  }
  SE_LAUNCH_CHECK();
  if (a.part) {
    hipLaunchKernelGGL(ln_finish_kernel<T>, dim3(se::ceil_div(a.C, 64), 2), dim3(1024), 0, st, a.part, parts, a.C,
                       a.wf32, dw, db);
    SE_LAUNCH_CHECK();
  }
  return SE_OK;
}

int check(long long rows, int C, int dtype, int wdtype) {
  if (rows <= 0 || C <= 0) return SE_E_ARG;
  if (dtype != SE_DTYPE_F32 && dtype != SE_DTYPE_BF16 && dtype != SE_DTYPE_F16) return SE_E_ARG;
  if (wdtype != dtype && wdtype != SE_DTYPE_F32) return SE_E_ARG;
  if (C > (1 << 30)) return SE_E_UNSUPPORTED;   // column indices are 32-bit
  return SE_OK;
}

}  // namespace

extern "C" int se_layer_norm_fwd(const void* x, long long x_stride, long long rows, int C, const void* weight,
                                 const void* bias, float eps, void* y, float* save, int dtype, int wdtype,
                                 void* stream) {
  const int rc = check(rows, C, dtype, wdtype);
  if (rc != SE_OK) return rc;
  if (!x || !y || x_stride < 0 || (x_stride < C && rows > 1)) return SE_E_ARG;
  LnArgs a{};
  a.x = x; a.w = weight; a.b = bias; a.out = y; a.save = save;
  a.rows = rows; a.sx = x_stride; a.C = C; a.eps = eps; a.inv_c = 1.f / (float)C;
  a.wf32 = dtype != SE_DTYPE_F32 && wdtype == SE_DTYPE_F32;
  hipStream_t st = se::as_stream(stream);
  if (dtype == SE_DTYPE_F32) return run_fwd<float>(a, st);
  if (dtype == SE_DTYPE_BF16) return run_fwd<__bf16>(a, st);
  return run_fwd<_Float16>(a, st);
}

extern "C" size_t se_layer_norm_workspace_size(long long rows, int C) {
  if (rows <= 0 || C <= 0) return 0;
  return (size_t)parts_of(rows, C) * 2 * C * sizeof(float);
}

extern "C" int se_layer_norm_bwd(const void* dy, long long dy_stride, const void* x, long long x_stride,
                                 long long rows, int C, const void* weight, const float* save, void* dx, void* dw,
                                 void* db, int dtype, int wdtype, void* ws, size_t ws_bytes, void* stream) {
  const int rc = check(rows, C, dtype, wdtype);
  if (rc != SE_OK) return rc;
  if (!dy || !x || !save || (!dx && !dw && !db)) return SE_E_ARG;
  if (x_stride < 0 || dy_stride < 0 || (rows > 1 && (x_stride < C || dy_stride < C))) return SE_E_ARG;
  const bool need = dw || db;
  if (need && (!ws || ws_bytes < se_layer_norm_workspace_size(rows, C))) return SE_E_WORKSPACE;
  LnArgs a{};
  a.x = x; a.dy = dy; a.w = weight; a.out = dx; a.save = const_cast<float*>(save);
  a.part = need ? static_cast<float*>(ws) : nullptr;
  a.rows = rows; a.sx = x_stride; a.sdy = dy_stride; a.C = C; a.inv_c = 1.f / (float)C;
  a.wf32 = dtype != SE_DTYPE_F32 && wdtype == SE_DTYPE_F32;
  const int parts = parts_of(rows, C);
  hipStream_t st = se::as_stream(stream);
  if (dtype == SE_DTYPE_F32) return run_bwd<float>(a, parts, dw, db, st);
  if (dtype == SE_DTYPE_BF16) return run_bwd<__bf16>(a, parts, dw, db, st);
  return run_bwd<_Float16>(a, parts, dw, db, st);
}
