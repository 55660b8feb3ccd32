// AdamW over many tensors in one launch, its states held in 8 bits or in 32 beside fp32, bf16 or fp16 parameters.
//
//   m' = m + (1 - b1)(g - m),  v' = b2 v + (1 - b2) g^2
//   p' = p (1 - lr wd) - lr / (1 - b1^t) m' / (sqrt(v') / sqrt(1 - b2^t) + eps)
//
// 32: m and v in fp32. 8: m and q = sqrt(v) as e4m3 values times one power of two for each 128 consecutive
// elements of a tensor (codes [numel], exponents k + 127 [ceil(numel / 128)]). q rather than v: half the binades, so
// e4m3's 18 below the block's largest cover gradients down to 2^-18 of it. k is the smallest with amax <= 448 2^k.
// m', v' ((1 - b2) g before times g) and q are fp32 values, each operation rounded once in the order it is written in, the same at 8
// and at 32 bits, and a code is the exact rounding of the fp32 value: a program that takes the step in elementary fp32
// operations holds the same codes, however often it is taken (a code that differs moves the next step's parameter by up
// to a tenth of lr). Rounding is stochastic: the magnitude in grid steps plus u = (h + 1/2) / 65536, rounded down, h the
// low (m) or high (q) half of a hash of (seed, step, tensor, element). To the nearest, a state would stand still: a step
// moves v by 1 - b2 = 0.001 of it, half a grid step is 2^-4. The hash is a counter's, so the replicas of a data-parallel
// run, which share seed and gradients, keep the same states. A positive q is stored as at least the smallest value: as 0
// it would leave m' / eps. The parameter moves by m' and v' before they are rounded to codes.
//
// Bound by memory: at 8 bits an element of an fp32 parameter reads and writes 16.06 bytes. The table of tensors goes in
// the kernel's arguments (no copy, no device table to keep alive, 48 tensors a launch); a workgroup takes one
// chunk of 2048 consecutive elements of one tensor, eight a thread, so 16 lanes share a block's exponent. 336 M fp32
// parameters with 8-bit states: 1.01 ms, 5.3 TB/s (a large copy: 5.0); 67 M bf16 ones with 32-bit states: 297 us, 5.0.
#include "common.hpp"

#include <cmath>

namespace {

constexpr int kThr = 256, kPer = 8, kChunk = kThr * kPer, kBlock = SE_ADAMW_BLOCK, kMost = 48;
constexpr long long kMostChunks = 0xffffff;   // a launch has less than 2^32 threads
static_assert(kBlock == 16 * kPer, "sixteen lanes share an exponent");

struct Tensor {
  void* p;
  const void* g;
  void* m;
  void* v;          // v (32) or q (8)
  unsigned char* mk;
  unsigned char* vk;
  long long n;
  unsigned key;
  unsigned vec;     // every pointer aligned for eight elements
};
struct Table {
  Tensor t[kMost];
  unsigned first[kMost + 1];   // chunks before tensor i
  int n;
};
struct Hyper {
  float decay, w1, b2, omb2, inv_bc2_sqrt, eps, neg_step;
};
static_assert(sizeof(Table) + sizeof(Hyper) <= 4096, "kernel arguments");

__device__ __host__ __forceinline__ unsigned mix(unsigned x) {
  x = (x ^ (x >> 15)) * 0x6A09E667u;   // the fractional bits of sqrt 2, of sqrt 3, of the golden ratio and of pi
  x = (x ^ (x >> 13)) * 0xBB67AE85u;
  return x ^ (x >> 16);
}

template <typename T>
__device__ __forceinline__ void load8(const T* p, bool vec, int left, float (&v)[8]) {
  struct alignas(16) P { T x[16 / sizeof(T)]; };
  if (vec && left >= 8) {
#pragma unroll
    for (int q = 0; q < (int)(8 * sizeof(T) / 16); ++q) {
      const P t = reinterpret_cast<const P*>(p)[q];
#pragma unroll
      for (int j = 0; j < (int)(16 / sizeof(T)); ++j) v[q * (16 / sizeof(T)) + j] = (float)t.x[j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < left ? (float)p[j] : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, bool vec, int left, const float (&v)[8]) {
  struct alignas(16) P { T x[16 / sizeof(T)]; };
  if (vec && left >= 8) {
#pragma unroll
    for (int q = 0; q < (int)(8 * sizeof(T) / 16); ++q) {
      P t;
#pragma unroll
      for (int j = 0; j < (int)(16 / sizeof(T)); ++j) t.x[j] = (T)v[q * (16 / sizeof(T)) + j];
      reinterpret_cast<P*>(p)[q] = t;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < left) p[j] = (T)v[j];
  }
}

typedef float f32x2 __attribute__((ext_vector_type(2)));

// eight e4m3 codes times 2^k
__device__ __forceinline__ void load_codes(const unsigned char* p, bool vec, int left, unsigned kcode, float (&v)[8]) {
  unsigned w[2] = {0u, 0u};
  if (vec && left >= 8) {
    const uint2 t = *reinterpret_cast<const uint2*>(p);
    w[0] = t.x; w[1] = t.y;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < left) w[j >> 2] |= (unsigned)p[j] << (8 * (j & 3));
  }
  const float s = __builtin_bit_cast(float, kcode << 23);   // kcode >= 1
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[q], false);
    const f32x2 b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[q], true);
    v[4 * q] = a.x * s; v[4 * q + 1] = a.y * s; v[4 * q + 2] = b.x * s; v[4 * q + 3] = b.y * s;
  }
}

// m' and v' from m and v, no two operations joined into one rounding
__device__ __forceinline__ void moments(const Hyper& h, float g, float& m, float& v) {
#pragma clang fp contract(off)
  m = m + h.w1 * (g - m);
  v = h.b2 * v + h.omb2 * g * g;
}

// k + 127 of the block that this thread's sixteen lanes hold: amax over their finite values
__device__ __forceinline__ unsigned block_exp(const float (&v)[8]) {
  float m = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float a = fabsf(v[j]);
    m = fmaxf(m, a < INFINITY ? a : 0.f);
  }
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
  const unsigned b = __builtin_bit_cast(unsigned, m);
  const int k = (int)(b >> 23) - 8 + ((b & 0x7fffffu) > 0x600000u);   // 448 = 1.75 2^8
  return (unsigned)max(k, 1);
}

// e4m3 code of x 2^-k, rounded stochastically by the 16 bits h; NaN for what is not finite. z, its fraction and 1 - u are
// fp32 numbers without an error, so that the comparison is the exact one (z + u would be rounded, at times up to the border).
__device__ __forceinline__ unsigned code_of(float x, float inv, unsigned h, bool floor1) {
#pragma clang fp contract(off)
  const float a = fabsf(x);
  const float y = a * inv;
  const int e = max((int)(__builtin_bit_cast(unsigned, y) >> 23) - 127, -6);
  const float z = __builtin_ldexpf(y, 3 - e);   // 8 .. 16, or less below 2^-6
  const float f = floorf(z);
  const bool up = z - f >= ((float)(0xffffu - h) + 0.5f) * 0x1p-16f;
  unsigned c = (unsigned)(((e + 7) << 3) + (int)f - 8 + up);
  if (floor1 && a > 0.f) c = max(c, 1u);
  if (!(a < INFINITY)) c = 0x7fu;
  return c | ((__builtin_bit_cast(unsigned, x) >> 24) & 0x80u);
}

// eight codes in two words
__device__ __forceinline__ void store_codes(unsigned char* p, bool vec, int left, unsigned w0, unsigned w1) {
  if (vec && left >= 8) {
    *reinterpret_cast<uint2*>(p) = uint2{w0, w1};
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < left) p[j] = (unsigned char)((j < 4 ? w0 : w1) >> (8 * (j & 3)));
  }
}

template <typename T, bool Q8>
__global__ void __launch_bounds__(kThr) adamw_multi_kernel(const Table tab, const Hyper h) {
  int lo = 0, hi = tab.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (tab.first[mid] <= blockIdx.x) lo = mid; else hi = mid - 1;
  }
  const Tensor& t = tab.t[lo];
  const long long i = (long long)(blockIdx.x - tab.first[lo]) * kChunk + threadIdx.x * kPer;
  // every lane stays for the block's shuffles; lanes behind the end hold zeros and write nothing
  const int left = (int)max(0LL, min(t.n - i, (long long)kPer));
  const bool vec = t.vec;
  T* P = static_cast<T*>(t.p) + i;
  float p[8], g[8], m[8], v[8];
  load8(P, vec, left, p);
  load8(static_cast<const T*>(t.g) + i, vec, left, g);
  unsigned mk = 1u, vk = 1u;
  if constexpr (Q8) {
    if (left > 0) {
      mk = max((unsigned)t.mk[i / kBlock], 1u);
      vk = max((unsigned)t.vk[i / kBlock], 1u);
    }
    load_codes(static_cast<unsigned char*>(t.m) + i, vec, left, mk, m);
    load_codes(static_cast<unsigned char*>(t.v) + i, vec, left, vk, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= v[j];
  } else {
    load8(static_cast<float*>(t.m) + i, vec, left, m);
    load8(static_cast<float*>(t.v) + i, vec, left, v);
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    moments(h, g[j], m[j], v[j]);
    const float q = sqrtf(v[j]);
    p[j] = p[j] * h.decay + h.neg_step * m[j] / (q * h.inv_bc2_sqrt + h.eps);
    if constexpr (Q8) v[j] = q;
  }
  store8(P, vec, left, p);
  if constexpr (Q8) {
    const unsigned base = (unsigned)i * 0x9E3779B1u + (unsigned)(i >> 32) * 0x243F6A89u + t.key;
    const unsigned nmk = block_exp(m), nvk = block_exp(v);
    const float mi = __builtin_bit_cast(float, (254u - nmk) << 23), vi = __builtin_bit_cast(float, (254u - nvk) << 23);
    unsigned char* cm = static_cast<unsigned char*>(t.m) + i;
    unsigned char* cv = static_cast<unsigned char*>(t.v) + i;
    unsigned wm[2] = {0u, 0u}, wv[2] = {0u, 0u};
#pragma unroll
    for (int j = 0; j < 8; ++j) {   // i is a multiple of 8: the upper half is the same for all eight
      const unsigned r = mix(base + j * 0x9E3779B1u);
      wm[j >> 2] |= code_of(m[j], mi, r & 0xffffu, false) << (8 * (j & 3));
      wv[j >> 2] |= code_of(v[j], vi, r >> 16, true) << (8 * (j & 3));
    }
    store_codes(cm, vec, left, wm[0], wm[1]);
    store_codes(cv, vec, left, wv[0], wv[1]);
    if (left > 0 && (threadIdx.x & 15) == 0) {
      t.mk[i / kBlock] = (unsigned char)nmk;
      t.vk[i / kBlock] = (unsigned char)nvk;
    }
  } else {
    store8(static_cast<float*>(t.m) + i, vec, left, m);
    store8(static_cast<float*>(t.v) + i, vec, left, v);
  }
}

template <typename T>
void launch(const Table& tab, const Hyper& h, int bits, unsigned grid, hipStream_t st) {
  if (bits == 8) hipLaunchKernelGGL((adamw_multi_kernel<T, true>), dim3(grid), dim3(kThr), 0, st, tab, h);
  else hipLaunchKernelGGL((adamw_multi_kernel<T, false>), dim3(grid), dim3(kThr), 0, st, tab, h);
}

}  // namespace

extern "C" int se_adamw_multi(const se_adamw_tensor* tensors, int n, int dtype, int bits, double lr, double beta1,
                              double beta2, double eps, double weight_decay, long long step,
                              unsigned long long seed, void* stream) {
  if (n < 0 || (n && !tensors) || step < 1) return SE_E_ARG;
  if (dtype != SE_DTYPE_F32 && dtype != SE_DTYPE_BF16 && dtype != SE_DTYPE_F16) return SE_E_ARG;
  if (bits != 8 && bits != 32) return SE_E_ARG;
  if (!(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0)) return SE_E_ARG;
  for (int i = 0; i < n; ++i) {
    const se_adamw_tensor& s = tensors[i];
    if (s.numel < 0) return SE_E_ARG;
    if (s.numel == 0) continue;
    if (!s.param || !s.grad || !s.exp_avg || !s.exp_avg_sq) return SE_E_ARG;
    if (bits == 8 && (!s.exp_avg_scale || !s.exp_avg_sq_scale)) return SE_E_ARG;
    if (s.numel > (long long)kChunk * kMostChunks) return SE_E_UNSUPPORTED;
  }
  Hyper h;
  h.decay = (float)(1.0 - lr * weight_decay);
  h.w1 = (float)(1.0 - beta1);
  h.b2 = (float)beta2;
  h.omb2 = (float)(1.0 - beta2);
  h.inv_bc2_sqrt = (float)(1.0 / std::sqrt(1.0 - std::pow(beta2, (double)step)));
  h.eps = (float)eps;
  h.neg_step = (float)(-(lr / (1.0 - std::pow(beta1, (double)step))));
  const unsigned k0 = mix(mix((unsigned)seed + mix((unsigned)(seed >> 32))) + (unsigned)step);   // mix(0) is 0
  hipStream_t st = se::as_stream(stream);
  Table tab;
  tab.n = 0;
  unsigned long long chunks = 0;
  for (int i = 0; i <= n; ++i) {
    const bool end = i == n;
    const long long c = end ? 0 : (tensors[i].numel + kChunk - 1) / kChunk;
    if (tab.n && (end || tab.n == kMost || chunks + c > (unsigned long long)kMostChunks)) {
      tab.first[tab.n] = (unsigned)chunks;
      if (dtype == SE_DTYPE_F32) launch<float>(tab, h, bits, (unsigned)chunks, st);
      else if (dtype == SE_DTYPE_BF16) launch<__bf16>(tab, h, bits, (unsigned)chunks, st);
      else launch<_Float16>(tab, h, bits, (unsigned)chunks, st);
      SE_LAUNCH_CHECK();
      tab.n = 0;
      chunks = 0;
    }
    if (end || c == 0) continue;
    const se_adamw_tensor& s = tensors[i];
    Tensor& t = tab.t[tab.n];
    t.p = s.param; t.g = s.grad; t.m = s.exp_avg; t.v = s.exp_avg_sq;
    t.mk = static_cast<unsigned char*>(s.exp_avg_scale);
    t.vk = static_cast<unsigned char*>(s.exp_avg_sq_scale);
    t.n = s.numel;
    t.key = mix(k0 + (unsigned)i);
    const int sa = bits == 8 ? 8 : 16;
    t.vec = ((uintptr_t)s.param | (uintptr_t)s.grad) % 16 == 0 && ((uintptr_t)s.exp_avg | (uintptr_t)s.exp_avg_sq) % sa == 0;
    tab.first[tab.n++] = (unsigned)chunks;
    chunks += c;
  }
  return SE_OK;
}
