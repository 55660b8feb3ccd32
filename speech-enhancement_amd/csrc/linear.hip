// The product with bias, activation and residual in its epilogue, and its gradients:
//
//   z = x W^T + b,  y = act(z) + r                         x [M, K], W [N, K], r and y [M, N]
//   g = dy act'(z),  dx = g W,  dW = g^T x,  db_n = sum_m g
//
// One GEMM kernel on v_mfma_f32_32x32x16_{bf16,f16} serves all three products. Each operand has a free index (a row of
// the tile) and the reduced one; it is stored with either of them contiguous:
//   KC  element (r, k) at r ld + k: x and W in the forward, g in dx
//   RC  element (r, k) at k ld + r: W in dx, g and x in dW
// Tiles of 64 reduced indices go from memory to LDS without passing registers (buffer_load ... lds, 16 bytes a lane),
// while the tile before them is multiplied. KC tiles are read back by ds_read_b128, RC tiles by
// ds_read_b64_tr_b16, which hands every lane four consecutive k of its own row. A direct load leaves lane l's
// 16 bytes at l * 16, so the image is swizzled on the side of memory: which chunk of its row a lane fetches.
//
// fp32 storage: each operand is split beforehand into two fp16 planes x 2^(14 - e) = hi + lo (22 significant bits),
// e from the largest magnitude of its own free index (a row of x has its own scale, so a loud frame costs a quiet one
// no digits, and an infinity stays in its row), and the kernel walks k three times: hi hi, hi lo, lo hi; the
// epilogue multiplies by 2^(ea + eb - 28).
#include "common.hpp"

#include <algorithm>

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef unsigned short u16;

constexpr int kBK = 64;
constexpr int kTop = 14;

struct Epi {
  void* C;              // [M][N]
  void* z;              // pre-activation in the storage type, or NULL
  const void* bias;     // [N], or NULL
  const void* res;      // [M][N] at ldr, or NULL
  const short* ea;      // power of two of each row of A and of B (fp32), or NULL
  const short* eb;
  long long ldc, ldr;   // z has rows of N
  int act;
};

struct GemmArgs {
  const u16* A[2];      // planes (one, or hi and lo)
  const u16* B[2];
  long long lda, ldb;   // elements between the rows of the stored matrix
  long long a_bytes, b_bytes;
  float* slab;          // splits > 1: [splits][M][N]
  int M, N;             // rows of A and of B
  int K, ksteps;        // reduced length, its tiles
  int steps, per;       // terms * ksteps, and how many of them a split takes
  int splits;
  Epi e;
};

__device__ __forceinline__ float act_of(int act, float z) {
  switch (act) {
    case SE_LINACT_RELU: return z > 0.f ? z : (z == z ? 0.f : z);
    case SE_LINACT_GELU: return 0.5f * z * (1.f + erff(z * 0.70710678118654752f));
    case SE_LINACT_GELU_TANH: return 0.5f * z * (1.f + tanhf(0.79788456080286536f * (z + 0.044715f * z * z * z)));
    case SE_LINACT_SILU: return z / (1.f + expf(-z));
    default: return z;
  }
}

__device__ __forceinline__ float slope_of(int act, float z) {
  switch (act) {
    case SE_LINACT_RELU: return z > 0.f ? 1.f : 0.f;
    case SE_LINACT_GELU:
      return 0.5f * (1.f + erff(z * 0.70710678118654752f)) + z * 0.3989422804014327f * expf(-0.5f * z * z);
    case SE_LINACT_GELU_TANH: {
      const float t = tanhf(0.79788456080286536f * (z + 0.044715f * z * z * z));
      return 0.5f * (1.f + t) + 0.5f * z * (1.f - t * t) * 0.79788456080286536f * (1.f + 0.134145f * z * z);
    }
    case SE_LINACT_SILU: {
      const float p = 1.f / (1.f + expf(-z));
      return p * (1.f + z * (1.f - p));
    }
    default: return 1.f;
  }
}

// four consecutive columns n .. n + 3 of row m, out of the accumulators or the slabs
template <typename S>
__device__ __forceinline__ void epilogue4(const Epi& e, int M, int N, int m, int n, float (&v)[4], bool vec) {
  struct alignas(4 * sizeof(S)) P { S x[4]; };
  if (m >= M || n >= N) return;
  const int left = N - n;
  if (e.ea) {
    const int s = e.ea[m] - 2 * kTop;
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = __builtin_ldexpf(v[j], s + (j < left ? e.eb[n + j] : 0));
  }
  const long long o = (long long)m * e.ldc + n, oz = (long long)m * N + n, orr = (long long)m * e.ldr + n;
  if (e.bias) {
    const S* b = static_cast<const S*>(e.bias) + n;
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] += j < left ? (float)b[j] : 0.f;
  }
  if (vec && left >= 4) {
    P t;
    if (e.z) {
#pragma unroll
      for (int j = 0; j < 4; ++j) t.x[j] = (S)v[j];
      *reinterpret_cast<P*>(static_cast<S*>(e.z) + oz) = t;
    }
    if (e.act)
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = act_of(e.act, v[j]);
    if (e.res) {
      const P r = *reinterpret_cast<const P*>(static_cast<const S*>(e.res) + orr);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] += (float)r.x[j];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) t.x[j] = (S)v[j];
    *reinterpret_cast<P*>(static_cast<S*>(e.C) + o) = t;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (j >= left) continue;
      if (e.z) static_cast<S*>(e.z)[oz + j] = (S)v[j];
      float r = e.act ? act_of(e.act, v[j]) : v[j];
      if (e.res) r += (float)static_cast<const S*>(e.res)[orr + j];
      static_cast<S*>(e.C)[o + j] = (S)r;
    }
  }
}

// whether rows of C, z and the residual take four columns in one access
template <typename S>
__device__ __forceinline__ bool vec_of(const Epi& e, int N) {
  const unsigned long long al = 4 * sizeof(S) - 1;
  return ((unsigned long long)e.C & al) == 0 && e.ldc % 4 == 0 && (!e.z || (N % 4 == 0 && ((unsigned long long)e.z & al) == 0)) &&
         (!e.res || (((unsigned long long)e.res & al) == 0 && e.ldr % 4 == 0));
}

typedef __attribute__((address_space(3))) void* lds_ptr;

// One operand's tile of R rows x 64 k, stored by NW waves; see the head comment for the two forms.
template <bool KC, int R, int NW>
struct Tile {
  static constexpr int kInstr = R / 8 / NW;              // 1 KB wave loads of each wave
  static constexpr int kRowsRC = 512 / R;                // stored rows (k) of one wave load
  static constexpr int kMask = (R / 16 < 8 ? R / 16 : 8) - 1;
  static_assert(R / 8 % NW == 0, "whole wave loads");
  static_assert(KC || (NW * kRowsRC) % 8 == 0, "a lane's swizzle does not change from load to load");

  // byte offset of this lane's 16 bytes from the tile's first element, without the load's uniform part
  static __device__ __forceinline__ unsigned lane_offset(int lane, int wave, long long ld) {
    if constexpr (KC) {
      return (unsigned)((lane >> 3) * ld * 2) + (((lane & 7) ^ (lane >> 3)) * 16);
    } else {
      const int k = wave * kRowsRC + lane / (R / 8), c = lane % (R / 8);
      return (unsigned)((lane / (R / 8)) * ld * 2) + ((c ^ (2 * (k & kMask))) * 16);
    }
  }
  // k of this lane's chunk within the tile (KC)
  static __device__ __forceinline__ int lane_k(int lane) { return ((lane & 7) ^ (lane >> 3)) * 8; }

  static __device__ __forceinline__ void load(const u16* base, long long at, long long bytes, long long ld, int kleft,
                                              unsigned off, int lane, int wave, u16* lds) {
    const long long left = bytes - at * 2;
    const int rec = left <= 0 ? 0 : (int)(left < 0x7ffffff0LL ? left : 0x7ffffff0LL);
    const __amdgpu_buffer_rsrc_t r =
        __builtin_amdgcn_make_buffer_rsrc(se::uniform_ptr(base + at), (short)0, __builtin_amdgcn_readfirstlane(rec), 0x00020000);
    if constexpr (KC)
      if (kleft < kBK && lane_k(lane) >= kleft) off = 0x80000000u;   // behind the row's end: zeros
#pragma unroll
    for (int q = 0; q < kInstr; ++q) {
      const int i = q * NW + wave;
      const int so = (int)((KC ? 8 : kRowsRC) * ld * 2) * i;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_ptr)(lds + i * 512), 16, (int)off,
                                               __builtin_amdgcn_readfirstlane(so), 0, 0);
    }
  }

  // this lane's eight k (kk + 8 (lane / 32) ..) of row f0 + (lane & 31)
  static __device__ __forceinline__ s16x8 fragment(const u16* lds, int f0, int kk, int lane) {
    if constexpr (KC) {
      const int row = f0 + (lane & 31), c = (kk >> 3) + (lane >> 5);
      return *reinterpret_cast<const s16x8*>(lds + row * kBK + ((c ^ (row & 7)) * 8));
    } else {
      s16x4 h[2];
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int k = kk + 8 * (lane >> 5) + 4 * q + ((lane & 15) >> 2);
        const int col = f0 + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
        const u16* p = lds + k * R + (((col >> 3) ^ (2 * (k & kMask))) * 8) + (col & 7);
        h[q] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p);
      }
      return __builtin_shufflevector(h[0], h[1], 0, 1, 2, 3, 4, 5, 6, 7);
    }
  }
};

template <typename H>
__device__ __forceinline__ f32x16 mfma(s16x8 a, s16x8 b, f32x16 c) {
  if constexpr (__is_same(H, __bf16))
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// consecutive workgroups go to the eight XCDs in turn: give each XCD a run of neighbouring tiles, eight rows of
// tiles deep, so that its L2 serves the operands they share
__device__ __forceinline__ void tile_of(int id, int MT, int NT, int& mt, int& nt) {
  const int total = MT * NT, x = id & 7, q = total >> 3, r = total & 7;
  id = x * q + min(x, r) + (id >> 3);
  constexpr int G = 8;
  const int band = id / (G * NT), first = band * G, deep = min(G, MT - first), in = id - band * G * NT;
  mt = first + in % deep;
  nt = in / deep;
}

// H: the products' type; S: the storage type of C, z, bias and residual (H, or float)
template <typename H, typename S, bool AKC, bool BKC, int BM, int BN, int WM, int WN>
__global__ void __launch_bounds__(WM * WN * 64, 2) linear_gemm_kernel(const GemmArgs a) {
  constexpr int NW = WM * WN, TM = BM / WM, TN = BN / WN, FM = TM / 32, FN = TN / 32;
  using TA = Tile<AKC, BM, NW>;
  using TB = Tile<BKC, BN, NW>;
  __shared__ __attribute__((aligned(16))) u16 sA0[BM * kBK], sB0[BN * kBK], sA1[BM * kBK], sB1[BN * kBK];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int MT = (a.M + BM - 1) / BM, NT = (a.N + BN - 1) / BN;
  int mt, nt;
  tile_of(blockIdx.x, MT, NT, mt, nt);
  const int m0 = mt * BM, n0 = nt * BN;
  const int wm = (wave % WM) * TM, wn = (wave / WM) * TN;
  const int s0 = blockIdx.y * a.per, s1 = min(a.steps, s0 + a.per);
  const unsigned offA = TA::lane_offset(lane, wave, a.lda), offB = TB::lane_offset(lane, wave, a.ldb);

  auto load = [&](int s, u16* la, u16* lb) __attribute__((always_inline)) {
    const int term = s / a.ksteps, k0 = (s - term * a.ksteps) * kBK, kleft = a.K - k0;
    const u16* pa = a.A[term == 2];
    const u16* pb = a.B[term == 1];
    TA::load(pa, AKC ? m0 * a.lda + k0 : k0 * a.lda + m0, a.a_bytes, a.lda, kleft, offA, lane, wave, la);
    TB::load(pb, BKC ? n0 * a.ldb + k0 : k0 * a.ldb + n0, a.b_bytes, a.ldb, kleft, offB, lane, wave, lb);
    __builtin_amdgcn_sched_barrier(0);   // the scheduler would sink the loads to the barrier that waits for them
  };

  f32x16 acc[FN][FM];
#pragma unroll
  for (int i = 0; i < FN; ++i)
#pragma unroll
    for (int j = 0; j < FM; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

  auto compute = [&](const u16* la, const u16* lb) __attribute__((always_inline)) {
#pragma unroll
    for (int kk = 0; kk < kBK; kk += 16) {
      s16x8 fa[FM], fb[FN];
#pragma unroll
      for (int j = 0; j < FM; ++j) fa[j] = TA::fragment(la, wm + 32 * j, kk, lane);
#pragma unroll
      for (int i = 0; i < FN; ++i) fb[i] = TB::fragment(lb, wn + 32 * i, kk, lane);
#pragma unroll
      for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int j = 0; j < FM; ++j) acc[i][j] = mfma<H>(fb[i], fa[j], acc[i][j]);
    }
  };

  if (s0 < s1) {
    load(s0, sA0, sB0);
    __syncthreads();
    int s = s0;
    for (; s + 2 < s1; s += 2) {
      load(s + 1, sA1, sB1);
      compute(sA0, sB0);
      __syncthreads();
      load(s + 2, sA0, sB0);
      compute(sA1, sB1);
      __syncthreads();
    }
    if (s + 1 < s1) {
      load(s + 1, sA1, sB1);
      compute(sA0, sB0);
      __syncthreads();
      compute(sA1, sB1);
    } else {
      compute(sA0, sB0);
    }
  }

  // block (i, j): this lane's column of the accumulator is row m, its registers 4 q .. 4 q + 3 four consecutive n
  const bool vec = vec_of<S>(a.e, a.N);
  float* slab = a.slab ? a.slab + (long long)blockIdx.y * a.M * a.N : nullptr;
#pragma unroll
  for (int j = 0; j < FM; ++j) {
    const int m = m0 + wm + 32 * j + (lane & 31);
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int n = n0 + wn + 32 * i + 8 * q + 4 * (lane >> 5);
        float v[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = acc[i][j][4 * q + r];
        if (!slab) {
          epilogue4<S>(a.e, a.M, a.N, m, n, v, vec);
        } else if (m < a.M) {
          float* p = slab + (long long)m * a.N + n;
          if (a.N % 4 == 0 && n < a.N) *reinterpret_cast<f32x4*>(p) = (f32x4){v[0], v[1], v[2], v[3]};
          else
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (n + r < a.N) p[r] = v[r];
        }
      }
  }
}

// the slabs of a split product, added in order, and the epilogue
template <typename S>
__global__ void __launch_bounds__(256) linear_join_kernel(const GemmArgs a) {
  const int N4 = (a.N + 3) / 4;
  const long long total = (long long)a.M * N4, mn = (long long)a.M * a.N;
  const bool vec = vec_of<S>(a.e, a.N), whole = a.N % 4 == 0;
  for (long long i = blockIdx.x * 256LL + threadIdx.x; i < total; i += gridDim.x * 256LL) {
    const int m = (int)(i / N4), n = (int)(i - (long long)m * N4) * 4;
    const float* p = a.slab + (long long)m * a.N + n;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    if (whole) {
      for (int s = 0; s < a.splits; ++s) {
        const f32x4 t = *reinterpret_cast<const f32x4*>(p + s * mn);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] += t[j];
      }
    } else {
      for (int s = 0; s < a.splits; ++s)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (n + j < a.N) v[j] += p[s * mn + j];
    }
    epilogue4<S>(a.e, a.M, a.N, m, n, v, vec);
  }
}

// ------------------------------------------------------------------ operands laid out
// [R][C] at ld -> rows of Cp = C rounded up to 8, zeros behind C (a matrix whose rows do not start on 16 bytes)
__global__ void __launch_bounds__(256) linear_pack_kernel(const u16* __restrict__ x, long long ld, int R, int C, int Cp,
                                                          u16* __restrict__ out) {
  const int per = Cp / 8;
  const long long total = (long long)R * per;
  for (long long i = blockIdx.x * 256LL + threadIdx.x; i < total; i += gridDim.x * 256LL) {
    const int r = (int)(i / per), c = (int)(i - (long long)r * per) * 8;
    const u16* p = x + r * ld + c;
    s16x8 v;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = c + j < C ? (short)p[j] : (short)0;
    *reinterpret_cast<s16x8*>(out + (long long)r * Cp + c) = v;
  }
}

// e with amax < 2^e; 2^(14 - e) stays a normal number
__device__ __forceinline__ int exp_of(float amax) {
  return max((int)(__builtin_bit_cast(unsigned, amax) >> 23) - 126, -112);
}
__device__ __forceinline__ float finite_abs(float x) { return fabsf(x) < INFINITY ? fabsf(x) : 0.f; }
__device__ __forceinline__ void split(float x, int e, _Float16& hi, _Float16& lo) {
  const float s = __builtin_ldexpf(x, kTop - e);
  hi = (_Float16)s;
  lo = fabsf(x) < INFINITY ? (_Float16)(s - (float)hi) : (_Float16)0.f;
}

// fp32 [R][C] at ld -> planes of rows Cp, one power of two a row (four rows a workgroup)
__global__ void __launch_bounds__(256) linear_split_rows_kernel(const float* __restrict__ x, long long ld, int R, int C,
                                                                int Cp, _Float16* __restrict__ hi,
                                                                _Float16* __restrict__ lo, short* __restrict__ ex) {
  const int r = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (r >= R) return;
  const float* p = x + r * ld;
  float m = 0.f;
  for (int c = lane; c < C; c += 64) m = fmaxf(m, finite_abs(p[c]));
  const int e = exp_of(se::wave_max(m));
  if (lane == 0) ex[r] = (short)e;
  for (int c = lane; c < Cp; c += 64) {
    _Float16 h, l;
    split(c < C ? p[c] : 0.f, e, h, l);
    hi[(long long)r * Cp + c] = h;
    lo[(long long)r * Cp + c] = l;
  }
}

// the same with one power of two a column: the columns' largest magnitudes over chunks of rows, then the planes
__global__ void __launch_bounds__(256) linear_col_max_kernel(const float* __restrict__ x, long long ld, int R, int C,
                                                             int rows, float* __restrict__ part) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= C) return;
  const int r0 = blockIdx.y * rows, r1 = min(R, r0 + rows);
  float m = 0.f;
#pragma unroll 8
  for (int r = r0; r < r1; ++r) m = fmaxf(m, finite_abs(x[r * ld + c]));
  part[(long long)blockIdx.y * C + c] = m;
}
__global__ void __launch_bounds__(256) linear_col_exp_kernel(const float* __restrict__ part, int parts, int C,
                                                             short* __restrict__ ex) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= C) return;
  float m = 0.f;
#pragma unroll 8
  for (int i = 0; i < parts; ++i) m = fmaxf(m, part[(long long)i * C + c]);
  ex[c] = (short)exp_of(m);
}
__global__ void __launch_bounds__(256) linear_split_cols_kernel(const float* __restrict__ x, long long ld, int R, int C,
                                                                int Cp, const short* __restrict__ ex,
                                                                _Float16* __restrict__ hi, _Float16* __restrict__ lo) {
  const long long total = (long long)R * Cp;
  for (long long i = blockIdx.x * 256LL + threadIdx.x; i < total; i += gridDim.x * 256LL) {
    const int r = (int)(i / Cp), c = (int)(i - (long long)r * Cp);
    _Float16 h, l;
    split(c < C ? x[r * ld + c] : 0.f, c < C ? ex[c] : 0, h, l);
    hi[i] = h;
    lo[i] = l;
  }
}

// g = dy act'(z) in rows of Np (zeros behind N), and each chunk of rows' column sums of g. z NULL: g = dy; g NULL: the
// sums alone. A workgroup takes 64 columns and `rows` rows, four rows at a time.
template <typename S>
__global__ void __launch_bounds__(256) linear_slope_kernel(const S* __restrict__ dy, long long ld, const S* __restrict__ z,
                                                           int act, int M, int N, int Np, int rows, S* __restrict__ g,
                                                           float* __restrict__ part) {
  __shared__ float sum[4][64];
  const int l = threadIdx.x & 63, w = threadIdx.x >> 6, n = blockIdx.x * 64 + l;
  const int r0 = blockIdx.y * rows, r1 = min(M, r0 + rows);
  float s = 0.f;
  if (n < Np)
#pragma unroll 4
    for (int r = r0 + w; r < r1; r += 4) {
      float v = 0.f;
      if (n < N) {
        v = (float)dy[r * ld + n];
        if (z) v *= slope_of(act, (float)z[(long long)r * N + n]);
      }
      if (g) g[(long long)r * Np + n] = (S)v;
      s += v;
    }
  if (!part) return;
  sum[w][l] = s;
  __syncthreads();
  if (w == 0 && n < N) part[(long long)blockIdx.y * N + n] = (sum[0][l] + sum[1][l]) + (sum[2][l] + sum[3][l]);
}

template <typename S>
__global__ void __launch_bounds__(1024) linear_bias_kernel(const float* __restrict__ part, int parts, int N,
                                                           S* __restrict__ db) {
  __shared__ float s[16][64];
  const int l = threadIdx.x & 63, k = threadIdx.x >> 6, n = blockIdx.x * 64 + l;
  const int per = (parts + 15) / 16, p0 = k * per, p1 = min(parts, p0 + per);
  float v = 0.f;
  if (n < N)
#pragma unroll 8
    for (int i = p0; i < p1; ++i) v += part[(long long)i * N + n];
  s[k][l] = v;
  __syncthreads();
  if (k || n >= N) return;
  for (int i = 1; i < 16; ++i) v += s[i][l];
  db[n] = (S)v;
}

// ------------------------------------------------------------------ host
struct Carve {   // a workspace, or (base NULL) its size
  char* base;
  size_t at = 0;
  template <typename T> T* take(long long n) {
    T* p = reinterpret_cast<T*>(base + at);
    at += ((size_t)n * sizeof(T) + 255) / 256 * 256;
    return base ? p : nullptr;
  }
};

struct Mat {            // an operand as the kernel reads it
  const u16* p[2];
  const short* ex;
  long long ld, bytes;
};

inline int up8(int n) { return (n + 7) / 8 * 8; }
inline unsigned blocks_for(long long n) { return (unsigned)std::min<long long>((n + 255) / 256, 8192); }

// A pass of the product: lays its operands out, multiplies, joins. `run` false: takes the workspace, launches nothing.
struct Pass {
  Carve ws;
  bool run;
  hipStream_t st;
  int rc = SE_OK;
  void launched() {
    if (rc == SE_OK && hipGetLastError() != hipSuccess) rc = SE_E_LAUNCH;
  }

  // 16-bit [R][C] at ld, as it is or packed
  Mat half(const void* x, long long ld, int R, int C) {
    Mat m{};
    if (ld % 8 == 0 && C % 8 == 0 && ((uintptr_t)x & 15) == 0) {
      m.p[0] = static_cast<const u16*>(x);
      m.ld = ld;
      m.bytes = ((long long)(R - 1) * ld + C) * 2;
      return m;
    }
    const int Cp = up8(C);
    u16* out = ws.take<u16>((long long)R * Cp);
    if (run) {
      hipLaunchKernelGGL(linear_pack_kernel, dim3(blocks_for((long long)R * Cp / 8)), dim3(256), 0, st,
                         static_cast<const u16*>(x), ld, R, C, Cp, out);
      launched();
    }
    m.p[0] = out;
    m.ld = Cp;
    m.bytes = (long long)R * Cp * 2;
    return m;
  }
  // fp32 [R][C] at ld as two planes, powers of two by row or by column
  Mat planes(const void* xv, long long ld, int R, int C, bool by_row) {
    const float* x = static_cast<const float*>(xv);
    Mat m{};
    const int Cp = up8(C);
    _Float16* hi = ws.take<_Float16>((long long)R * Cp);
    _Float16* lo = ws.take<_Float16>((long long)R * Cp);
    short* ex = ws.take<short>(by_row ? R : C);
    const int rows = std::max(64, (R + 255) / 256), parts = (R + rows - 1) / rows;
    float* part = by_row ? nullptr : ws.take<float>((long long)parts * C);
    if (run && by_row) {
      hipLaunchKernelGGL(linear_split_rows_kernel, dim3((R + 3) / 4), dim3(256), 0, st, x, ld, R, C, Cp, hi, lo, ex);
      launched();
    } else if (run) {
      hipLaunchKernelGGL(linear_col_max_kernel, dim3((C + 255) / 256, parts), dim3(256), 0, st, x, ld, R, C, rows, part);
      hipLaunchKernelGGL(linear_col_exp_kernel, dim3((C + 255) / 256), dim3(256), 0, st, part, parts, C, ex);
      hipLaunchKernelGGL(linear_split_cols_kernel, dim3(blocks_for((long long)R * Cp)), dim3(256), 0, st, x, ld, R, C,
                         Cp, ex, hi, lo);
      launched();
    }
    m.p[0] = reinterpret_cast<const u16*>(hi);
    m.p[1] = reinterpret_cast<const u16*>(lo);
    m.ex = ex;
    m.ld = Cp;
    m.bytes = (long long)R * Cp * 2;
    return m;
  }

  template <typename H, typename S, bool AKC, bool BKC>
  void product(const Mat& A, const Mat& B, int M, int N, int K, const Epi& e) {
    constexpr int BM = 128, BN = 128;
    GemmArgs a{};
    a.M = M; a.N = N; a.K = K;
    a.lda = A.ld; a.ldb = B.ld; a.a_bytes = A.bytes; a.b_bytes = B.bytes;
    for (int i = 0; i < 2; ++i) { a.A[i] = A.p[i]; a.B[i] = B.p[i]; }
    a.e = e;
    a.e.ea = A.ex; a.e.eb = B.ex;
    a.ksteps = (K + kBK - 1) / kBK;
    const int terms = __is_same(S, float) ? 3 : 1;
    const long long tiles = (long long)((M + BM - 1) / BM) * ((N + BN - 1) / BN), steps = (long long)terms * a.ksteps;
    if (tiles > 0x7fffffffLL || steps > 0x7fffffffLL || A.ld > (1 << 21) || B.ld > (1 << 21)) { rc = SE_E_UNSUPPORTED; return; }
    a.steps = (int)steps;
    // two workgroups share a CU: split the reduction until 512 run, eight tiles of it at least to a split
    int splits = 1;
    if (tiles < 384) splits = (int)std::max<long long>(1, std::min<long long>(512 / tiles, steps / 8));
    a.per = (a.steps + splits - 1) / splits;
    a.splits = (a.steps + a.per - 1) / a.per;
    if (a.splits > 1) a.slab = ws.take<float>((long long)a.splits * M * N);
    if (!run || rc != SE_OK) return;
    hipLaunchKernelGGL((linear_gemm_kernel<H, S, AKC, BKC, BM, BN, 2, 2>), dim3((unsigned)tiles, a.splits), dim3(256), 0,
                       st, a);
    launched();
    if (a.splits > 1) {
      hipLaunchKernelGGL(linear_join_kernel<S>, dim3(blocks_for((long long)M * ((N + 3) / 4))), dim3(256), 0, st, a);
      launched();
    }
  }
};

template <typename S> struct Product { using H = S; };
template <> struct Product<float> { using H = _Float16; };

template <typename S>
int forward(const se_linear_desc* d, const void* x, const void* w, const void* bias, const void* res, void* y, void* z,
            Pass& p) {
  using H = typename Product<S>::H;
  constexpr bool f32 = __is_same(S, float);
  const Mat A = f32 ? p.planes(x, d->ldx, d->M, d->K, true) : p.half(x, d->ldx, d->M, d->K);
  const Mat B = f32 ? p.planes(w, d->ldw, d->N, d->K, true) : p.half(w, d->ldw, d->N, d->K);
  Epi e{};
  e.C = y; e.z = z; e.bias = bias; e.res = res; e.ldc = d->N; e.ldr = d->ldr; e.act = d->act;
  p.template product<H, S, true, true>(A, B, d->M, d->N, d->K, e);
  return p.rc;
}

template <typename S>
int backward(const se_linear_desc* d, const void* dy, const void* x, const void* w, const void* z, void* dx, void* dw,
             void* db, Pass& p) {
  using H = typename Product<S>::H;
  constexpr bool f32 = __is_same(S, float);
  const int M = d->M, N = d->N, K = d->K;
  const bool sloped = d->act != SE_LINACT_NONE, prod = dx || dw;
  // g: dy itself where nothing multiplies it and the product can read it as it lies
  const bool as_is = !sloped && (f32 || (d->ldr % 8 == 0 && N % 8 == 0 && ((uintptr_t)dy & 15) == 0));
  const int Np = f32 ? N : up8(N);
  S* g = prod && !as_is ? p.ws.template take<S>((long long)M * Np) : nullptr;
  const int rows = std::max(64, (int)(((long long)M + 127) / 128)), parts = (M + rows - 1) / rows;
  float* part = db ? p.ws.template take<float>((long long)parts * N) : nullptr;
  if (p.run && (part || g)) {
    hipLaunchKernelGGL(linear_slope_kernel<S>, dim3((Np + 63) / 64, parts), dim3(256), 0, p.st,
                       static_cast<const S*>(dy), d->ldr, sloped ? static_cast<const S*>(z) : nullptr, d->act, M, N, Np,
                       rows, g, part);
    p.launched();
    if (part) {
      hipLaunchKernelGGL(linear_bias_kernel<S>, dim3((N + 63) / 64), dim3(1024), 0, p.st, part, parts, N,
                         static_cast<S*>(db));
      p.launched();
    }
  }
  const void* gp = as_is ? dy : g;
  const long long ldg = as_is ? d->ldr : Np;
  if (dx) {
    const Mat A = f32 ? p.planes(gp, ldg, M, N, true) : p.half(gp, ldg, M, as_is ? N : Np);
    const Mat B = f32 ? p.planes(w, d->ldw, N, K, false) : p.half(w, d->ldw, N, K);
    Epi e{};
    e.C = dx; e.ldc = K;
    p.template product<H, S, true, false>(A, B, M, K, N, e);
  }
  if (dw) {
    const Mat A = f32 ? p.planes(gp, ldg, M, N, false) : p.half(gp, ldg, M, as_is ? N : Np);
    const Mat B = f32 ? p.planes(x, d->ldx, M, K, false) : p.half(x, d->ldx, M, K);
    Epi e{};
    e.C = dw; e.ldc = K;
    p.template product<H, S, false, false>(A, B, N, K, M, e);
  }
  return p.rc;
}

int check(const se_linear_desc* d) {
  if (!d || d->M <= 0 || d->N <= 0 || d->K <= 0) return SE_E_ARG;
  if (d->dtype != SE_DTYPE_F32 && d->dtype != SE_DTYPE_BF16 && d->dtype != SE_DTYPE_F16) return SE_E_ARG;
  if (d->act < SE_LINACT_NONE || d->act > SE_LINACT_SILU) return SE_E_ARG;
  if (d->ldw < d->K || d->ldx < 0 || (d->M > 1 && d->ldx < d->K) || d->ldr < 0 || (d->M > 1 && d->ldr && d->ldr < d->N))
    return SE_E_ARG;
  if (d->N > (1 << 21) || d->K > (1 << 21) || d->ldw > (1LL << 21) || d->ldx > (1LL << 21) || d->ldr > (1LL << 21))
    return SE_E_UNSUPPORTED;   // a tile's byte offsets are 32-bit
  return SE_OK;
}

#define SE_LIN_SWITCH(dtype, CALL)                        \
  switch (dtype) {                                        \
    case SE_DTYPE_F32: { using S = float; return CALL; }  \
    case SE_DTYPE_BF16: { using S = __bf16; return CALL; } \
    default: { using S = _Float16; return CALL; }         \
  }

int forward_any(const se_linear_desc* d, const void* x, const void* w, const void* bias, const void* res, void* y, void* z,
                Pass& p) {
  SE_LIN_SWITCH(d->dtype, (forward<S>(d, x, w, bias, res, y, z, p)))
}
int backward_any(const se_linear_desc* d, const void* dy, const void* x, const void* w, const void* z, void* dx, void* dw,
                 void* db, Pass& p) {
  SE_LIN_SWITCH(d->dtype, (backward<S>(d, dy, x, w, z, dx, dw, db, p)))
}

}  // namespace

extern "C" size_t se_linear_fwd_workspace_size(const se_linear_desc* d, const void* x, const void* w) {
  if (check(d) != SE_OK) return 0;
  Pass p{Carve{nullptr}, false, nullptr};
  forward_any(d, x, w, nullptr, nullptr, nullptr, nullptr, p);
  return p.ws.at;
}

extern "C" int se_linear_fwd(const se_linear_desc* d, const void* x, const void* w, const void* bias, const void* residual,
                             void* y, void* z, void* ws, size_t ws_bytes, void* stream) {
  const int rc = check(d);
  if (rc != SE_OK) return rc;
  if (!x || !w || !y) return SE_E_ARG;
  const size_t need = se_linear_fwd_workspace_size(d, x, w);
  if (need && (!ws || ws_bytes < need)) return SE_E_WORKSPACE;
  Pass p{Carve{static_cast<char*>(ws)}, true, se::as_stream(stream)};
  return forward_any(d, x, w, bias, residual, y, z, p);
}

extern "C" size_t se_linear_bwd_workspace_size(const se_linear_desc* d, const void* dy, const void* x, const void* w,
                                               int want_dx, int want_dw, int want_db) {
  if (check(d) != SE_OK) return 0;
  Pass p{Carve{nullptr}, false, nullptr};
  char some;   // only asked whether it is there
  backward_any(d, dy, x, w, nullptr, want_dx ? &some : nullptr, want_dw ? &some : nullptr, want_db ? &some : nullptr, p);
  return p.ws.at;
}

extern "C" int se_linear_bwd(const se_linear_desc* d, const void* dy, const void* x, const void* w, const void* z, void* dx,
                             void* dw, void* db, void* ws, size_t ws_bytes, void* stream) {
  const int rc = check(d);
  if (rc != SE_OK) return rc;
  if (!dy || (dx && !w) || (dw && !x) || (!dx && !dw && !db) || (d->act != SE_LINACT_NONE && !z)) return SE_E_ARG;
  if (d->M > 1 && d->ldr < d->N) return SE_E_ARG;
  const size_t need = se_linear_bwd_workspace_size(d, dy, x, w, dx != nullptr, dw != nullptr, db != nullptr);
  if (need && (!ws || ws_bytes < need)) return SE_E_WORKSPACE;
  Pass p{Carve{static_cast<char*>(ws)}, true, se::as_stream(stream)};
  return backward_any(d, dy, x, w, z, dx, dw, db, p);
}
