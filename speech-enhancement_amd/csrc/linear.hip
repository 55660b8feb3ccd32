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
// fp32 storage, but for small products (linear_plain_kernel): each operand is split beforehand into fp16 x 2^(14 - e) = hi + lo (22 significant bits), e from the
// largest magnitude of its own free index (a row of x has its own scale, so a loud frame costs a quiet one no digits, and
// an infinity stays in its row). 32 k of hi and the same 32 of lo lie side by side, 64 k of a tile, whose products are hi hi,
// hi lo and lo hi; the epilogue multiplies by 2^(ea + eb - 28).
//
// Rounded on the way in 16 bits, beside the result: z, which the backward reads (in fp32 it would add half to what the
// forward writes), and g, which the products take as 16-bit operands. The slope is that of the rounded z. Against products
// of an unrounded g the gradients' error grows from 0.0017 to 0.0024 (bf16, root of the mean square, relative) where there is an
// activation; without one nothing but the result is rounded.
//
// What bounds it: at 128 x 128 the LDS (a wave's 64 x 64 asks for a fragment a product, 192 KB of reads and writes to
// 256 cycles of products); at 256 x 256 in four waves of 128 x 128 (half as many) the matrix unit is busy 76 % of a CU's
// cycles in dW, 70 % in dx and 61 % in the forward, whose rounds' epilogues nothing covers, and the clock falls to
// 1.65 GHz. 8192^3 bf16: 828 us, 1.33 PFLOP/s (in 128 x 128: 1023; eight waves of 128 x 64 took 901 where the same step
// in four took 853). 16384 x 4096 x 8192 bf16 inside a training pass, hot: forward 1.10 ms, dx 0.97, dW 0.88;
// 25792 x 512 x 2048: 75, 58 and 84 us; 9002 x 514 x 1030 fp32: 63, 48 and 58 us. Tried and slower: stores straight
// from the accumulators (32 bytes of a row at a time; 16384 x 8192 outputs over 128: 185 us against 141), workgroups
// that stay and load their next tile under the epilogue (1 to 9 %); the order of k rotated between workgroups changed
// less than 2 %.
#include "common.hpp"

#include <algorithm>
#include <cmath>
#include <type_traits>

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
constexpr int kMostLd = 1 << 21;   // elements between rows that the tiled product reads: its byte offsets in a tile are 32-bit

struct Epi {
  void* C;              // [M][N]
  void* z;              // pre-activation in the storage type, or NULL
  const void* bias;     // [N], or NULL
  const void* res;      // [M][N] at ldr, or NULL
  const short* ea;      // power of two of each row of A and of B (fp32), or NULL
  const short* eb;
  long long ldc, ldr, ldz;
  int act;
};

struct GemmArgs {
  const u16* A;
  const u16* B;
  long long lda, ldb;   // elements between the rows of the stored matrix
  long long a_bytes, b_bytes;
  float* slab;          // splits > 1: [splits][M][N]
  int M, N;             // rows of A and of B
  int K;                // reduced length as it is stored (fp32: hi and lo)
  int steps, per;       // its tiles, and how many of them a split takes
  int splits;
  Epi e;
};

// The activations by the hardware's exponential and reciprocal (1 ulp each): sigma(t) = 1 / (1 + 2^(-t log2 e)).
__device__ __forceinline__ float sigmoid_fast(float t) {
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.4426950408889634f * t));
}
// Phi(z), and phi(z): for fp32 storage by erf; for 16 bits Phi(-|z|) = phi(z) Q(t) t sqrt(pi / 2), t = 1 / (1 + 0.44 |z| / sqrt 2), Q
// of degree 5 fitted to exp(x^2) erfc(x) / t (least largest relative error over x up to 9.6, by reweighted least squares):
// Phi is 5.5e-6 of itself off in either tail, a hundredth of an fp16 half step, besides what the rounding of z^2 / 2 does
// to the exponential (z^2 2^-24 of it).
template <bool FAST>
__device__ __forceinline__ float normal_cdf(float z, float& phi) {
  const float e = __builtin_amdgcn_exp2f(-0.72134752044448170f * z * z);   // exp(-z^2 / 2)
  phi = 0.3989422804014327f * e;
  if constexpr (FAST) {
    const float t = __builtin_amdgcn_rcpf(1.f + 0.44f * 0.70710678118654752f * fabsf(z));
    const float q = 0.5f * e * t * (0.24856107f + t * (0.24256903f + t * (0.26358819f + t * (0.040727897f + t * (0.35065521f + t * -0.14610657f)))));
    return z < 0.f ? q : 1.f - q;
  } else {
    return z < 0.f ? 0.5f * erfcf(-0.70710678118654752f * z) : 0.5f + 0.5f * erff(0.70710678118654752f * z);
  }
}
// the argument of the tanh form: z (1 + tanh c(z + a z^3)) / 2 = z sigma(2 c (z + a z^3))
__device__ __forceinline__ float tanh_arg(float z) { return 1.5957691216057308f * (z + 0.044715f * z * z * z); }

template <bool FAST, int V>
__device__ __forceinline__ void act_of(int act, float (&v)[V]) {
  switch (act) {   // one branch for the V values
    case SE_LINACT_RELU:
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = v[j] < 0.f ? 0.f : v[j];   // a NaN stays
      break;
    case SE_LINACT_GELU:
#pragma unroll
      for (int j = 0; j < V; ++j) {
        float phi;
        v[j] *= normal_cdf<FAST>(v[j], phi);
      }
      break;
    case SE_LINACT_GELU_TANH:
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] *= sigmoid_fast(tanh_arg(v[j]));
      break;
    case SE_LINACT_SILU:
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] *= sigmoid_fast(v[j]);
      break;
    default: break;
  }
}

// v *= act'(z)
template <bool FAST, int V>
__device__ __forceinline__ void slope_of(int act, const float (&z)[V], float (&v)[V]) {
  switch (act) {
    case SE_LINACT_RELU:
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = z[j] <= 0.f ? 0.f : v[j];
      break;
    case SE_LINACT_GELU:
#pragma unroll
      for (int j = 0; j < V; ++j) {
        float phi;
        const float c = normal_cdf<FAST>(z[j], phi);
        v[j] *= c + z[j] * phi;
      }
      break;
    case SE_LINACT_GELU_TANH:
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float p = sigmoid_fast(tanh_arg(z[j]));
        v[j] *= p + z[j] * p * (1.f - p) * (1.5957691216057308f * (1.f + 0.134145f * fminf(z[j] * z[j], 1e30f)));
      }
      break;
    case SE_LINACT_SILU:
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float p = sigmoid_fast(z[j]);
        v[j] *= p * (1.f + z[j] * (1.f - p));
      }
      break;
    default: break;
  }
}

template <typename S, int V> struct alignas(sizeof(S) * V > 16 ? 16 : sizeof(S) * V) Pack { S x[V]; };
template <typename S, int V>
__device__ __forceinline__ void load_pack(const S* p, float (&v)[V]) {
  const Pack<S, V> t = *reinterpret_cast<const Pack<S, V>*>(p);
#pragma unroll
  for (int j = 0; j < V; ++j) v[j] = (float)t.x[j];
}
template <typename S, int V>
__device__ __forceinline__ void store_pack(S* p, const float (&v)[V]) {
  Pack<S, V> t;
#pragma unroll
  for (int j = 0; j < V; ++j) t.x[j] = (S)v[j];
  *reinterpret_cast<Pack<S, V>*>(p) = t;
}

// what V consecutive columns n .. (all inside) have for every row
template <typename S, int V>
struct Cols {
  float bias[V];
  int eb[V];
  __device__ __forceinline__ void load(const Epi& e, int n) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      bias[j] = 0.f;
      eb[j] = 0;
    }
    if (e.bias) load_pack<S, V>(static_cast<const S*>(e.bias) + n, bias);
    if (e.ea)
#pragma unroll
      for (int j = 0; j < V; ++j) eb[j] = e.eb[n + j] - 2 * kTop;
  }
};

// those columns of row m, out of the sums; res: the residual's values, or zeros. Every row is aligned for V.
template <typename S, int V>
__device__ __forceinline__ void epilogue(const Epi& e, const Cols<S, V>& cols, long long m, int n, float (&v)[V],
                                         const float (&res)[V], int ea) {
  if constexpr (sizeof(S) == 4)   // fp32: the planes' powers of two (0 where there are none)
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = __builtin_ldexpf(v[j], ea + cols.eb[j]);
#pragma unroll
  for (int j = 0; j < V; ++j) v[j] += cols.bias[j];
  if (e.z) store_pack<S, V>(static_cast<S*>(e.z) + m * e.ldz + n, v);
  act_of<sizeof(S) == 2, V>(e.act, v);
#pragma unroll
  for (int j = 0; j < V; ++j) v[j] += res[j];
  store_pack<S, V>(static_cast<S*>(e.C) + m * e.ldc + n, v);
}

// whether the rows of C, z, the residual and the bias take V columns in one access (z's rows are laid out for it)
template <typename S, int V>
__device__ __forceinline__ bool vec_of(const Epi& e, int N) {
  constexpr unsigned long long al = (sizeof(S) * V > 16 ? 16 : sizeof(S) * V) - 1;
  return N % V == 0 && (((unsigned long long)e.C | (unsigned long long)e.bias | (unsigned long long)e.res) & al) == 0 &&
         e.ldc % V == 0 && (!e.res || e.ldr % V == 0);
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

  // the matrix from element `at` on, `bytes` in all: reads behind its end give zeros
  static __device__ __forceinline__ __amdgpu_buffer_rsrc_t source(const u16* base, long long at, long long bytes) {
    const long long left = bytes - at * 2;
    const int rec = left <= 0 ? 0 : (int)(left < 0x7ffffff0LL ? left : 0x7ffffff0LL);
    return __builtin_amdgcn_make_buffer_rsrc(se::uniform_ptr(base + at), (short)0, __builtin_amdgcn_readfirstlane(rec), 0x00020000);
  }
  // wave load q of kInstr: 1 KB of the tile
  static __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t r, unsigned off, int ld, int wave, int q, u16* lds) {
    const int i = q * NW + wave;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_ptr)(lds + i * 512), 16, (int)off,
                                             __builtin_amdgcn_readfirstlane((KC ? 8 : kRowsRC) * 2 * i * ld), 0, 0);
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

// 32 rows of TN sums from `turn` through the epilogue (or into the slab), V columns a lane. Stores and loads complete in the
// order they were asked for, so the loop waits for no load behind a store but the residuals', eight turns' together.
template <typename S, int V, bool RES, int TN, int PITCH>
__device__ __forceinline__ void drain(const GemmArgs& a, float* slab, const float* turn, int lane, int mb, int nb,
                                      const float* bias, const int* eb, const int* ea) {
  constexpr int kWide = TN < 64 * V ? TN : 64 * V, kLanes = kWide / V, kRows = 64 / kLanes;
  constexpr int kU = 32 / kRows < 8 ? 32 / kRows : 8;
#pragma unroll 1
  for (int c0 = 0; c0 < TN; c0 += kWide) {
    const int c = c0 + (lane % kLanes) * V, n = nb + c;
    const bool on = n < a.N;   // V divides N
    float cb[V];
    int ce[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      cb[j] = bias[c + j];
      ce[j] = sizeof(S) == 4 ? eb[c + j] : 0;
    }
#pragma unroll 1
    for (int r0 = 0; r0 < 32; r0 += kU * kRows) {
      float v[kU * V], res[RES ? kU * V : 1];
      const int first = r0 + lane / kLanes;
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        const int r = first + u * kRows;
        float t[V];
        load_pack<float, V>(turn + r * PITCH + c, t);
#pragma unroll
        for (int j = 0; j < V; ++j) v[u * V + j] = t[j];
        if constexpr (RES) {
          const bool in = on && mb + r < a.M;
          load_pack<S, V>(static_cast<const S*>(a.e.res) + (in ? (mb + r) * a.e.ldr + n : 0), t);
#pragma unroll
          for (int j = 0; j < V; ++j) res[u * V + j] = t[j];
        }
      }
      auto put = [&](auto* to, long long ld) __attribute__((always_inline)) {
        using O = std::remove_pointer_t<decltype(to)>;
#pragma unroll
        for (int u = 0; u < kU; ++u) {
          const int m = mb + first + u * kRows;
          float t[V];
#pragma unroll
          for (int j = 0; j < V; ++j) t[j] = v[u * V + j];
          if (on && m < a.M) store_pack<O, V>(to + m * ld + n, t);
        }
      };
      if (slab) {
        put(slab, a.N);
        continue;
      }
#pragma unroll
      for (int u = 0; u < kU; ++u)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          if constexpr (sizeof(S) == 4) v[u * V + j] = __builtin_ldexpf(v[u * V + j], ea[first + u * kRows] + ce[j]);
          v[u * V + j] += cb[j];
        }
      if (a.e.z) put(static_cast<S*>(a.e.z), a.e.ldz);
      act_of<sizeof(S) == 2, kU * V>(a.e.act, v);
      if constexpr (RES)
#pragma unroll
        for (int j = 0; j < kU * V; ++j) v[j] += res[j];
      put(static_cast<S*>(a.e.C), a.e.ldc);
    }
  }
}

// H: the products' type; S: the storage type of C, z, bias and residual (H, or float); RES: there is a residual
template <typename H, typename S, bool AKC, bool BKC, bool RES, int BM, int BN, int WM, int WN>
__global__ void __launch_bounds__(WM * WN * 64, BM == 256 && WM * WN == 4 ? 1 : 2) linear_gemm_kernel(const GemmArgs a) {
  constexpr int NW = WM * WN, TM = BM / WM, TN = BN / WN, FM = TM / 32, FN = TN / 32;
  using TA = Tile<AKC, BM, NW>;
  using TB = Tile<BKC, BN, NW>;
  __shared__ __attribute__((aligned(16))) u16 sA0[BM * kBK], sB0[BN * kBK], sA1[BM * kBK], sB1[BN * kBK];
  // what the epilogue needs of its columns and rows: nothing may be waited for from memory behind the first store
  constexpr bool f32 = sizeof(S) == 4;
  __shared__ __attribute__((aligned(16))) float sBias[BN];
  __shared__ __attribute__((aligned(16))) int sEb[f32 ? BN : 4], sEa[f32 ? BM : 4];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int MT = (a.M + BM - 1) / BM, NT = (a.N + BN - 1) / BN;
  int mt, nt;
  tile_of(blockIdx.x, MT, NT, mt, nt);
  const int m0 = mt * BM, n0 = nt * BN;
  const int wm = (wave % WM) * TM, wn = (wave / WM) * TN;
  const int s0 = blockIdx.y * a.per, s1 = min(a.steps, s0 + a.per);
  if (!a.slab) {
    for (int i = threadIdx.x; i < BN; i += NW * 64) {
      const bool in = n0 + i < a.N;
      sBias[i] = in && a.e.bias ? (float)static_cast<const S*>(a.e.bias)[n0 + i] : 0.f;
      if constexpr (f32) sEb[i] = in && a.e.eb ? a.e.eb[n0 + i] - 2 * kTop : 0;
    }
    if constexpr (f32)
      for (int i = threadIdx.x; i < BM; i += NW * 64) sEa[i] = m0 + i < a.M && a.e.ea ? a.e.ea[m0 + i] : 0;
  }
  const unsigned offA = TA::lane_offset(lane, wave, a.lda), offB = TB::lane_offset(lane, wave, a.ldb);

  // where the tile after the one that is being loaded lies: its sources, and the lanes' offsets into them
  struct Next {
    __amdgpu_buffer_rsrc_t a, b;
    unsigned oa, ob;
  } next;
  auto aim = [&](int s) __attribute__((always_inline)) {
    const int k0 = s * kBK, kleft = a.K - k0;
    const bool on = s < s1;   // behind the last one: nothing is read
    next.a = TA::source(a.A, AKC ? m0 * a.lda + k0 : k0 * a.lda + m0, on ? a.a_bytes : 0);
    next.b = TB::source(a.B, BKC ? n0 * a.ldb + k0 : k0 * a.ldb + n0, on ? a.b_bytes : 0);
    // KC, behind the row's end: zeros
    next.oa = AKC && kleft < kBK && TA::lane_k(lane) >= kleft ? 0x80000000u : offA;
    next.ob = BKC && kleft < kBK && TB::lane_k(lane) >= kleft ? 0x80000000u : offB;
  };
  constexpr int kLoads = TA::kInstr + TB::kInstr;
  auto load = [&](int from, int to, u16* la, u16* lb) __attribute__((always_inline)) {
#pragma unroll
    for (int q = 0; q < kLoads; ++q) {
      if (q < from || q >= to) continue;
      if (q < TA::kInstr) TA::load(next.a, next.oa, (int)a.lda, wave, q, la);
      else TB::load(next.b, next.ob, (int)a.ldb, wave, q - TA::kInstr, lb);
    }
  };

  f32x16 acc[FN][FM];
#pragma unroll
  for (int i = 0; i < FN; ++i)
#pragma unroll
    for (int j = 0; j < FM; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

  // The fragments of the next sixteen k are read while the matrix unit works on these; the last sixteen of a tile come
  // after the barrier that opens the next tile, so that its first fragments, and the loads into the tile just left,
  // are under way meanwhile.
  s16x8 fa[2][FM], fb[2][FN], fl[f32 ? FN : 1];
  auto readA = [&](s16x8 (&f)[FM], const u16* la, int kk) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < FM; ++j) f[j] = TA::fragment(la, wm + 32 * j, kk, lane);
  };
  auto readB = [&](auto& f, const u16* lb, int kk) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < FN; ++i) f[i] = TB::fragment(lb, wn + 32 * i, kk, lane);
  };
  auto multiply = [&](const s16x8 (&f)[FM], const auto& g) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < FM; ++j)
#pragma unroll
      for (int i = 0; i < FN; ++i) acc[i][j] = mfma<H>(g[i], f[j], acc[i][j]);
  };
  // LDS reads and loads between the products: all waves ask at the same time, and a wave whose requests wait their turn in
  // front of its products would start those late.
  constexpr int kReadA = FM * (AKC ? 1 : 2), kReadB = FN * (BKC ? 1 : 2);
  auto mixed = [&](auto reads, auto loads) __attribute__((always_inline)) {
    constexpr int kReads = decltype(reads)::value, kProducts = FM * FN, kV = decltype(loads)::value;
    constexpr int kEach = (kReads + kProducts - 1) / kProducts;
#pragma unroll
    for (int i = 0; i < kProducts; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);                               // a product
      if (i * kEach < kReads) __builtin_amdgcn_sched_group_barrier(0x100, kEach, 0);   // LDS reads
#pragma unroll
      for (int v = i * kV / kProducts; v < (i + 1) * kV / kProducts; ++v)
        __builtin_amdgcn_sched_group_barrier(0x010, 1, 0);   // a load
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  // The loads of a tile: the first part right after the barrier that frees its buffer, the rest over the next two steps, so
  // that the last of them has a step's time or more until the barrier that waits for it.
  constexpr int kL0 = (kLoads + 2) / 3, kL1 = kL0 + (kLoads - kL0 + 1) / 2;
  using N0 = std::integral_constant<int, kL0>;
  using N1 = std::integral_constant<int, kL1 - kL0>;
  using N2 = std::integral_constant<int, kLoads - kL1>;
  using None = std::integral_constant<int, 0>;
  using RA = std::integral_constant<int, kReadA>;
  using RB = std::integral_constant<int, kReadB>;
  using RAB = std::integral_constant<int, kReadA + kReadB>;
  // Tile s in (la, lb), its first fragments in set 0; tile s + 1 is on its way to (na, nb), whose first fragments are read at
  // the end (behind the last tile, for nothing), when the loads of tile s + 2 into (la, lb) begin.
  auto tile = [&](u16* la, u16* lb, u16* na, u16* nb, int s) __attribute__((always_inline)) {
    if constexpr (!f32) {
      load(kL0, kL1, na, nb);
      readA(fa[1], la, 16);
      readB(fb[1], lb, 16);
      multiply(fa[0], fb[0]);
      mixed(RAB{}, N1{});
      load(kL1, kLoads, na, nb);
      readA(fa[0], la, 32);
      readB(fb[0], lb, 32);
      multiply(fa[1], fb[1]);
      mixed(RAB{}, N2{});
      readA(fa[1], la, 48);
      readB(fb[1], lb, 48);
      multiply(fa[0], fb[0]);
      mixed(RAB{}, None{});
    } else {   // hi of k 0 and 16 at 0 and 16, lo at 32 and 48; fa[0] and fb hold hi, fa[1] and fl lo
      load(kL0, kL1, na, nb);
      readB(fl, lb, 32);
      multiply(fa[0], fb[0]);
      mixed(RB{}, N1{});
      load(kL1, kLoads, na, nb);
      readA(fa[1], la, 32);
      multiply(fa[0], fl);
      mixed(RA{}, N2{});
      readA(fa[0], la, 16);
      readB(fb[1], lb, 16);
      multiply(fa[1], fb[0]);
      mixed(RAB{}, None{});
      readB(fl, lb, 48);
      multiply(fa[0], fb[1]);
      mixed(RB{}, None{});
      readA(fa[1], la, 48);
      multiply(fa[0], fl);
      mixed(RA{}, None{});
    }
    aim(s + 2);
    __syncthreads();
    load(0, kL0, la, lb);
    readA(fa[0], na, 0);
    readB(fb[0], nb, 0);
    multiply(fa[1], fb[1]);
    mixed(RAB{}, N0{});
  };

  // two buffers of their own names, so that the compiler sees that a tile's loads do not touch the one being read
  aim(s0);
  load(0, kLoads, sA0, sB0);
  aim(s0 + 1);
  load(0, kL0, sA1, sB1);
  __syncthreads();
  readA(fa[0], sA0, 0);
  readB(fb[0], sB0, 0);
  for (int s = s0; s < s1; s += 2) {   // the tile behind an odd number of them is zeros
    tile(sA0, sB0, sA1, sB1, s);
    tile(sA1, sB1, sA0, sB0, s + 1);
  }
  __syncthreads();

  // The accumulators of block (i, j) hold, in lane l, row m = l & 31 and four consecutive n in each of four groups. Each wave
  // turns 32 rows at a time through the LDS that the tiles no longer need, so that a row's columns leave side by side:
  // 16 bytes a lane (a 16-bit row of 64 columns is one 128-byte line) where the rows are aligned for it.
  constexpr int kPitch = TN + 4, kPer = NW / 4;   // waves to each of the four buffers
  static_assert(kPer * 32 * kPitch * 4 <= (BM < BN ? BM : BN) * kBK * 2, "the turned rows fit");
  const int which = wave / kPer;
  float* turn = reinterpret_cast<float*>(which == 0 ? sA0 : which == 1 ? sB0 : which == 2 ? sA1 : sB1) + (wave % kPer) * 32 * kPitch;
  float* slab = a.slab ? a.slab + (long long)blockIdx.y * a.M * a.N : nullptr;
  const int wide = a.slab ? (a.N % 8 == 0 ? 8 : a.N % 2 == 0 ? 2 : 1) : vec_of<S, 8>(a.e, a.N) ? 8 : vec_of<S, 2>(a.e, a.N) ? 2 : 1;
#pragma unroll 1
  for (int j = 0; j < FM; ++j) {
    auto put = [&](auto at) __attribute__((always_inline)) {
      constexpr int J = decltype(at)::value;
#pragma unroll
      for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *reinterpret_cast<f32x4*>(turn + (lane & 31) * kPitch + 32 * i + 8 * q + 4 * (lane >> 5)) =
              (f32x4){acc[i][J][4 * q], acc[i][J][4 * q + 1], acc[i][J][4 * q + 2], acc[i][J][4 * q + 3]};
    };
    static_assert(FM == 1 || FM == 2 || FM == 4, "the blocks below");
    if (j == 0) put(std::integral_constant<int, 0>{});
    if constexpr (FM > 1) if (j == 1) put(std::integral_constant<int, 1>{});
    if constexpr (FM > 2) {
      if (j == 2) put(std::integral_constant<int, 2>{});
      if (j == 3) put(std::integral_constant<int, 3>{});
    }
    __builtin_amdgcn_wave_barrier();   // a wave's LDS accesses are in order; the compiler's must be too
    const int mb = m0 + wm + 32 * j;
    if (wide == 8) drain<S, 8, RES, TN, kPitch>(a, slab, turn, lane, mb, n0 + wn, sBias + wn, sEb + wn, sEa + mb - m0);
    else if (wide == 2) drain<S, 2, RES, TN, kPitch>(a, slab, turn, lane, mb, n0 + wn, sBias + wn, sEb + wn, sEa + mb - m0);
    else drain<S, 1, RES, TN, kPitch>(a, slab, turn, lane, mb, n0 + wn, sBias + wn, sEb + wn, sEa + mb - m0);
    __builtin_amdgcn_wave_barrier();
  }
}

// the slabs of a split product, added in order, and the epilogue: V columns a thread
template <typename S, int V>
__global__ void __launch_bounds__(256) linear_join_kernel(const GemmArgs a) {
  const int NV = a.N / V;
  const long long total = (long long)a.M * NV, mn = (long long)a.M * a.N;
  for (long long i = blockIdx.x * 256LL + threadIdx.x; i < total; i += gridDim.x * 256LL) {
    const long long m = i / NV;
    const int n = (int)(i - m * NV) * V;
    const float* p = a.slab + m * a.N + n;
    float v[V];
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = 0.f;
#pragma unroll 4
    for (int s = 0; s < a.splits; ++s) {
      float t[V];
      load_pack<float, V>(p + s * mn, t);
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] += t[j];
    }
    Cols<S, V> cols;
    cols.load(a.e, n);
    float res[V];
#pragma unroll
    for (int j = 0; j < V; ++j) res[j] = 0.f;
    if (a.e.res) load_pack<S, V>(static_cast<const S*>(a.e.res) + m * a.e.ldr + n, res);
    epilogue<S, V>(a.e, cols, m, n, v, res, a.e.ea ? a.e.ea[m] : 0);
  }
}

// ------------------------------------------------------------------ fp32 as it lies
// fp32 operands without the split: v_mfma_f32_32x32x2_f32 multiplies at a sixteenth of the 16-bit rate, a fifth of what the
// planes' three products reach, but reads what the caller holds, in one launch where the planes and their powers of
// two take up to seven: for small products, by the rule at plain_shape_of. 64 x 64 tiles of four waves, 32 k a step; the next step's values are fetched
// into registers while this one's are multiplied out of the other half of LDS, where k is the row, so that both
// forms are read at 32 neighbouring words.
constexpr int kPlainTile = 64, kPlainK = 32;

// eight values of a thread's row from k on: (row, k + j), zeros outside
template <bool KC>
__device__ __forceinline__ void plain_load(const float* p, long long ld, int row, int R, int k, int K, bool vec, float (&v)[8]) {
  if constexpr (KC) {
    const float* q = p + row * ld + k;
    if (vec && row < R && k + 8 <= K) {
      const f32x4 a = *reinterpret_cast<const f32x4*>(q), b = *reinterpret_cast<const f32x4*>(q + 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[j] = a[j];
        v[4 + j] = b[j];
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = row < R && k + j < K ? q[j] : 0.f;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = row < R && k + j < K ? p[(k + j) * ld + row] : 0.f;
  }
}

template <bool AKC, bool BKC>
__global__ void __launch_bounds__(256) linear_plain_kernel(const GemmArgs a, bool avec, bool bvec) {
  __shared__ float sA[2][kPlainK][kPlainTile], sB[2][kPlainK][kPlainTile];
  const int NT = (a.N + kPlainTile - 1) / kPlainTile;
  const int m0 = blockIdx.x / NT * kPlainTile, n0 = blockIdx.x % NT * kPlainTile;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wm = (wave >> 1) * 32, wn = (wave & 1) * 32, r = lane & 31, half = lane >> 5;
  const float* A = reinterpret_cast<const float*>(a.A);
  const float* B = reinterpret_cast<const float*>(a.B);
  const int s0 = blockIdx.y * a.per, s1 = min(a.steps, s0 + a.per);
  f32x16 acc = {};
  float va[8], vb[8];
  auto fetch = [&](int s) __attribute__((always_inline)) {
    const int k = s * kPlainK + wave * 8;
    plain_load<AKC>(A, a.lda, m0 + lane, a.M, k, a.K, avec, va);
    plain_load<BKC>(B, a.ldb, n0 + lane, a.N, k, a.K, bvec, vb);
  };
  fetch(s0);
  for (int s = s0; s < s1; ++s) {
    const int b = (s - s0) & 1;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      sA[b][wave * 8 + j][lane] = va[j];
      sB[b][wave * 8 + j][lane] = vb[j];
    }
    __syncthreads();   // the half written before last is read by nobody any more
    if (s + 1 < s1) fetch(s + 1);
#pragma unroll
    for (int k = 0; k < kPlainK; k += 2)
      acc = __builtin_amdgcn_mfma_f32_32x32x2f32(sA[b][k + half][wm + r], sB[b][k + half][wn + r], acc, 0, 0, 0);
  }
  const int n = n0 + wn + r;
  if (n >= a.N) return;
  float* slab = a.splits > 1 ? a.slab + (long long)blockIdx.y * a.M * a.N : nullptr;
  Cols<float, 1> cols;
  if (!slab) cols.load(a.e, n);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const long long m = m0 + wm + (i >> 2) * 8 + half * 4 + (i & 3);
    if (m >= a.M) continue;
    if (slab) {
      slab[m * a.N + n] = acc[i];
    } else {
      float v[1] = {acc[i]}, res[1] = {0.f};
      if (a.e.res) res[0] = static_cast<const float*>(a.e.res)[m * a.e.ldr + n];
      epilogue<float, 1>(a.e, cols, m, n, v, res, 0);
    }
  }
}

// ------------------------------------------------------------------ few rows
// Up to 64 rows of x: bound by the one read of W. A workgroup takes 16 rows of W (columns of y), its waves a slice of K each;
// a lane fetches 16 bytes of its row of W and of its rows of x straight into the fragments of v_mfma_f32_16x16x32 (fp32: four
// v_mfma_f32_16x16x4_f32, exact products, lane group g and element j standing for k = 16 s + 4 g + j in both operands), and the
// slices are added in order through LDS: one launch, no workspace. 1 x 1024 -> 4096 bf16: 4.1 us, 16 x 4096 -> 1024 fp16: 10 us
// (the tiled product and its join took 12.5 for the first); in fp32 6.4 and 18 us. Rows off 16 bytes are read an element at a
// time: 16 x 4095 -> 1024 bf16 33 us.
template <typename S> struct Frag { typedef f32x4 T; };
template <> struct Frag<__bf16> { typedef bf16x8 T; };
template <> struct Frag<_Float16> { typedef f16x8 T; };

template <typename S>
__device__ __forceinline__ f32x4 mfma16(typename Frag<S>::T a, typename Frag<S>::T b, f32x4 c) {
  if constexpr (__is_same(S, __bf16)) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  else if constexpr (__is_same(S, _Float16)) return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  else {
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
    return c;
  }
}

// the 16 bytes of a row from k on; zeros behind K
template <typename S, bool VEC>
__device__ __forceinline__ typename Frag<S>::T few_load(const S* row, int k, int K) {
  constexpr int E = 16 / sizeof(S);
  typename Frag<S>::T v = {};
  if constexpr (VEC) {
    if (k < K) v = *reinterpret_cast<const typename Frag<S>::T*>(row + k);
  } else {
#pragma unroll
    for (int j = 0; j < E; ++j)
      if (k + j < K) v[j] = row[k + j];
  }
  return v;
}

template <typename S, bool VEC, int MT>
__global__ void __launch_bounds__(1024) linear_few_kernel(const S* __restrict__ x, long long ldx, const S* __restrict__ w,
                                                          long long ldw, int M, int N, int K, Epi e) {
  constexpr int E = 16 / sizeof(S), KS = 4 * E, U = MT == 1 ? 8 : 4;
  extern __shared__ float part[];   // [waves][MT][16 m][16 n]
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const int r = lane & 15, g = lane >> 4, n0 = blockIdx.x * 16;
  const int steps = (K + KS - 1) / KS, per = (steps + waves - 1) / waves;
  const int s0 = wave * per, s1 = min(steps, s0 + per);
  // rows behind the end repeat the last one: their products are not used
  const S* wr = w + min(n0 + r, N - 1) * ldw;
  const S* xr[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) xr[t] = x + min(16 * t + r, M - 1) * ldx;
  f32x4 acc[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) acc[t] = (f32x4){0.f, 0.f, 0.f, 0.f};
  for (int s = s0; s < s1; s += U) {
    typename Frag<S>::T fw[U], fx[U][MT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = s + u < s1 ? (s + u) * KS + g * E : K;
      fw[u] = few_load<S, VEC>(wr, k, K);
#pragma unroll
      for (int t = 0; t < MT; ++t) fx[u][t] = few_load<S, VEC>(xr[t], k, K);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int t = 0; t < MT; ++t) acc[t] = mfma16<S>(fw[u], fx[u][t], acc[t]);
  }
#pragma unroll
  for (int t = 0; t < MT; ++t) *reinterpret_cast<f32x4*>(part + ((wave * MT + t) * 16 + r) * 16 + 4 * g) = acc[t];
  __syncthreads();
  for (int i = threadIdx.x; i < MT * 256; i += blockDim.x) {
    const int m = i >> 4, n = n0 + (i & 15);
    if (m >= M || n >= N) continue;
    float v[1] = {0.f}, res[1] = {0.f};
    for (int k = 0; k < waves; ++k) v[0] += part[k * MT * 256 + i];
    Cols<S, 1> cols;
    cols.load(e, n);
    if (e.res) res[0] = (float)static_cast<const S*>(e.res)[m * e.ldr + n];
    epilogue<S, 1>(e, cols, m, n, v, res, 0);
  }
}

// ------------------------------------------------------------------ operands laid out
// [R][C] at ld -> rows of Cp = C rounded up to 8, zeros behind C (a matrix whose rows do not start on 16 bytes). A launch
// takes the operands of a pass side by side (blockIdx.z), since alone the small ones take what a launch takes.
constexpr int kMostJobs = 3;
struct PackJob {
  const u16* x;
  u16* out;
  long long ld;
  int R, C, Cp;
};
struct PackJobs {
  PackJob j[kMostJobs];
};
__global__ void __launch_bounds__(256) linear_pack_kernel(const PackJobs jobs) {
  const PackJob& t = jobs.j[blockIdx.z];
  const int per = t.Cp / 8, C = t.C;
  const long long total = (long long)t.R * per;
  for (long long i = blockIdx.x * 256LL + threadIdx.x; i < total; i += gridDim.x * 256LL) {
    const int r = (int)(i / per), c = (int)(i - (long long)r * per) * 8;
    const u16* p = t.x + r * t.ld + c;
    s16x8 v;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = c + j < C ? (short)p[j] : (short)0;
    *reinterpret_cast<s16x8*>(t.out + (long long)r * t.Cp + c) = v;
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

// fp32 [R][C] at ld -> rows of 64 to each 32 columns (hi, then lo; zeros behind C), one power of two a row. A wave takes
// a row, a lane pairs of columns; rows of up to 2048 stay in registers, longer ones are read again. Bound by memory:
// 9002 x 1030 in 17 us, 4.4 TB/s.
constexpr int kSplitKeep = 16;
__device__ __forceinline__ void load_two(bool two, const float* p, int c, int C, float& a, float& b) {
  a = b = 0.f;
  if (two && c + 1 < C) {
    const float2 t = *reinterpret_cast<const float2*>(p + c);
    a = t.x;
    b = t.y;
  } else {
    if (c < C) a = p[c];
    if (c + 1 < C) b = p[c + 1];
  }
}
__device__ __forceinline__ void split_two(float a, float b, int ea, int eb, unsigned& hi, unsigned& lo) {
  typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
  _Float16 h0, l0, h1, l1;
  split(a, ea, h0, l0);
  split(b, eb, h1, l1);
  hi = __builtin_bit_cast(unsigned, (f16x2){h0, h1});
  lo = __builtin_bit_cast(unsigned, (f16x2){l0, l1});
}
// an operand to be laid out, of a launch's several (blockIdx.z)
struct SplitJob {
  const float* x;   // [R][C] at ld
  long long ld;
  unsigned* out;
  short* ex;        // the powers of two
  float* part;      // by columns: [parts][C] largest magnitudes of chunks of `rows` rows
  int R, C, width;  // width: C32 (by rows) or Cp (by columns)
  int rows, parts;
  bool two, known;  // two: pairs are aligned; known: `part` is there
};
struct SplitJobs {
  SplitJob j[kMostJobs];
};
__global__ void __launch_bounds__(256) linear_split_rows_kernel(const SplitJobs jobs) {
  const SplitJob& t = jobs.j[blockIdx.z];
  const float* __restrict__ x = t.x;
  unsigned* __restrict__ out = t.out;
  const long long ld = t.ld;
  const int R = t.R, C = t.C, C32 = t.width;
  const bool two = t.two;
  const int lane = threadIdx.x & 63;
  for (long long r = blockIdx.x * 4LL + (threadIdx.x >> 6); r < R; r += gridDim.x * 4LL) {
    const float* p = x + r * ld;
    unsigned* o = out + r * C32;   // C32 pairs of words: 2 C32 halves
    float v[kSplitKeep][2], m = 0.f;
#pragma unroll
    for (int i = 0; i < kSplitKeep; ++i) {
      v[i][0] = v[i][1] = 0.f;
      if (i * 128 < C) load_two(two, p, i * 128 + 2 * lane, C, v[i][0], v[i][1]);
      m = fmaxf(m, fmaxf(finite_abs(v[i][0]), finite_abs(v[i][1])));
    }
    for (int c = kSplitKeep * 128 + 2 * lane; c < C; c += 128) {
      float a, b;
      load_two(two, p, c, C, a, b);
      m = fmaxf(m, fmaxf(finite_abs(a), finite_abs(b)));
    }
    const int e = exp_of(se::wave_max(m));
    if (lane == 0) t.ex[r] = (short)e;
    auto put = [&](int c, float a, float b) __attribute__((always_inline)) {
      unsigned hi, lo;
      split_two(a, b, e, e, hi, lo);
      const int at = (c >> 5) * 32 + (c & 31) / 2;
      o[at] = hi;
      o[at + 16] = lo;
    };
#pragma unroll
    for (int i = 0; i < kSplitKeep; ++i)
      if (i * 128 + 2 * lane < C32) put(i * 128 + 2 * lane, v[i][0], v[i][1]);
    for (int c = kSplitKeep * 128 + 2 * lane; c < C32; c += 128) {
      float a, b;
      load_two(two, p, c, C, a, b);
      put(c, a, b);
    }
  }
}

// the same with one power of two a column, 32 rows of hi, then the 32 of lo: the columns' largest magnitudes over chunks
// of rows, their powers, then the halves in rows of Cp
__global__ void __launch_bounds__(256) linear_col_max_kernel(const SplitJobs jobs) {
  const SplitJob& t = jobs.j[blockIdx.z];
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= t.C || (int)blockIdx.y >= t.parts || t.known) return;
  const float* __restrict__ x = t.x + c;
  const int r0 = blockIdx.y * t.rows, r1 = min(t.R, r0 + t.rows);
  float m = 0.f;
#pragma unroll 8
  for (int r = r0; r < r1; ++r) m = fmaxf(m, finite_abs(x[r * t.ld]));
  t.part[(long long)blockIdx.y * t.C + c] = m;
}
__global__ void __launch_bounds__(1024) linear_col_exp_kernel(const SplitJobs jobs) {
  __shared__ float s[16][64];
  const SplitJob& t = jobs.j[blockIdx.z];
  const int l = threadIdx.x & 63, k = threadIdx.x >> 6, c = blockIdx.x * 64 + l;
  float m = 0.f;
  if (c < t.C)
#pragma unroll 8
    for (int i = k; i < t.parts; i += 16) m = fmaxf(m, t.part[(long long)i * t.C + c]);
  s[k][l] = m;
  __syncthreads();
  if (k || c >= t.C) return;
  for (int i = 1; i < 16; ++i) m = fmaxf(m, s[i][l]);
  t.ex[c] = (short)exp_of(m);
}
__global__ void __launch_bounds__(256) linear_split_cols_kernel(const SplitJobs jobs) {
  const SplitJob& t = jobs.j[blockIdx.z];
  const float* __restrict__ x = t.x;
  const short* __restrict__ ex = t.ex;
  unsigned* __restrict__ out = t.out;
  const int per = t.width / 2, R = t.R, C = t.C;
  const bool two = t.two;
  const long long total = (R + 31LL) / 32 * 32 * per;
  for (long long i = blockIdx.x * 256LL + threadIdx.x; i < total; i += gridDim.x * 256LL) {
    const int r = (int)(i / per), c = (int)(i - (long long)r * per) * 2;
    float a = 0.f, b = 0.f;
    if (r < R) load_two(two, x + r * t.ld, c, C, a, b);
    unsigned hi, lo;
    split_two(a, b, c < C ? ex[c] : 0, c + 1 < C ? ex[c + 1] : 0, hi, lo);
    const long long at = ((long long)(r >> 5) * 64 + (r & 31)) * per + c / 2;
    out[at] = hi;
    out[at + 32LL * per] = lo;
  }
}

// g = dy act'(z) in rows of Np (zeros behind N), and each chunk of rows' column sums of g. z NULL: g = dy; g NULL: the
// sums alone. A lane takes eight columns, cg lanes (a power of two) a row, 256 / cg rows at a time; the block's sums
// of a column are added in a fixed order through LDS; top (fp32, or NULL): and their largest finite magnitudes, for the
// powers of two of g's columns. Bound by memory: 16384 x 8192 bf16 in 163 us, 4.9 TB/s, 190 behind
// large products (a column a lane: 367).
template <typename S, bool VEC>
__global__ void __launch_bounds__(256) linear_slope_kernel(const S* __restrict__ dy, long long ld, const S* __restrict__ z,
                                                           int act, int M, int N, int Np, int cg, int rows,
                                                           S* __restrict__ g, float* __restrict__ part,
                                                           float* __restrict__ top) {
  __shared__ float sum[256][9];
  const int c = threadIdx.x % cg, n = (blockIdx.x * cg + c) * 8, step = 256 / cg;
  const long long r0 = (long long)blockIdx.y * rows;
  const int r1 = (int)min((long long)M - r0, (long long)rows);
  constexpr bool f32 = sizeof(S) == 4;
  float s[8], t8[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) s[j] = t8[j] = 0.f;
  if (n < Np)
#pragma unroll 2
    for (int r = threadIdx.x / cg; r < r1; r += step) {
      const long long m = r0 + r;
      float v[8], t[8];
      if constexpr (VEC) {
        load_pack<S, 8>(dy + m * ld + n, v);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = n + j < N ? (float)dy[m * ld + n + j] : 0.f;
      }
      if (z) {
        load_pack<S, 8>(z + m * Np + n, t);
        slope_of<sizeof(S) == 2, 8>(act, t, v);
        if constexpr (!VEC)   // z's rows are not filled behind N
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = n + j < N ? v[j] : 0.f;
      }
      if (g) store_pack<S, 8>(g + m * Np + n, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) s[j] += v[j];
      if constexpr (f32)
#pragma unroll
        for (int j = 0; j < 8; ++j) t8[j] = fmaxf(t8[j], finite_abs(v[j]));
    }
  if (part) {
#pragma unroll
    for (int j = 0; j < 8; ++j) sum[threadIdx.x][j] = s[j];
    __syncthreads();
    for (int i = threadIdx.x; i < cg * 8; i += 256) {
      const int at = blockIdx.x * cg * 8 + i;
      if (at >= N) continue;
      float v = 0.f;
      for (int k = 0; k < step; ++k) v += sum[k * cg + i / 8][i & 7];
      part[(long long)blockIdx.y * N + at] = v;
    }
  }
  if constexpr (f32) {
    if (!top) return;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 8; ++j) sum[threadIdx.x][j] = t8[j];
    __syncthreads();
    for (int i = threadIdx.x; i < cg * 8; i += 256) {
      const int at = blockIdx.x * cg * 8 + i;
      if (at >= N) continue;
      float v = 0.f;
      for (int k = 0; k < step; ++k) v = fmaxf(v, sum[k * cg + i / 8][i & 7]);
      top[(long long)blockIdx.y * N + at] = v;
    }
  }
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
  const u16* p;
  const short* ex;
  long long ld, bytes;
};

inline int up8(int n) { return (n + 7) / 8 * 8; }
inline unsigned blocks_for(long long n) { return (unsigned)std::min<long long>((n + 255) / 256, 8192); }

// Tile and split of a product by what a round of workgroups costs, measured on 16384 x 8192 outputs over 2 to 128 steps of 64 k:
// 256 x 256 tiles, one workgroup a CU, 12 us + 1.52 us a step; 128 x 128, two a CU, 4.2 us + 0.97 us a step, alone on it 0.55 us. So large
// tiles for long sums over many tiles (8192^3: 0.83 ms against 1.02), small ones for short sums and where their rounds fit
// better (25792 x 2048 over 512: 75 us against 94). A split's slabs are written and read at 4 bytes a sum.
struct Shape {
  int tile, per;
  long long tiles;
  double us;
};
inline Shape shape_of(int M, int N, int steps, double products) {   // products: of a step, against 16 bits
  Shape best{};
  double least = 1e300;
  for (int t : {128, 256}) {
    const long long tiles = (long long)((M + t - 1) / t) * ((N + t - 1) / t);
    const double fixed = (t == 256 ? 12 : 4.2) * products, each = (t == 256 ? 1.52 : 0.97) * products;
    const long long slots = t == 256 ? 256 : 512;
    for (int p = 1; p <= 64; p = p < 8 ? p + 1 : p + p / 4) {
      const int per = ((steps + p - 1) / p + 1) / 2 * 2;   // the kernel takes steps in pairs
      const int splits = (steps + per - 1) / per;
      if (p > 1 && (per < 4 || splits < 2)) break;
      const long long blocks = tiles * splits, rounds = blocks / slots, rest = blocks - rounds * slots;
      // a last round that leaves every small tile a CU of its own steps faster
      const double last = rest == 0 ? 0 : fixed + per * (t == 128 && rest <= 256 ? 0.55 * products : each);
      double us = rounds * (fixed + each * per) + last;
      if (splits > 1) us += 3 + (double)M * N * (6.0 * splits + 2) / 4.5e6;
      if (us < least) {
        least = us;
        best = Shape{t, per, tiles, us};
      }
    }
  }
  return best;
}

// The same for fp32 operands as they lie, 64 x 64 tiles and 32 k a step: four workgroups a CU take 2.6 us a step, 0.5 more for
// each operand read across its rows and 1.4 for rows off 16 bytes, two and one a CU 0.55 and 0.4 of it. Measured on
// 17 sizes in each direction, laid-out planes against this: 1365 x 83 x 76: 14, 23 and 21 us against 9, 9 and 10;
// 1000^3: 29, 40 and 35 against 35, 38 and 39; 2048 x 1024 x 1024: 36, 46 and 45 against 47, 59 and 65.
inline Shape plain_shape_of(int M, int N, int steps, double each) {
  Shape best{};
  double least = 1e300;
  const long long tiles = (long long)((M + kPlainTile - 1) / kPlainTile) * ((N + kPlainTile - 1) / kPlainTile);
  for (int p = 1; p <= 64; p = p < 8 ? p + 1 : p + p / 4) {
    const int per = (steps + p - 1) / p, splits = (steps + per - 1) / per;
    if (p > 1 && (per < 2 || splits < 2)) break;
    const long long blocks = tiles * splits, slots = 1024, rounds = blocks / slots, rest = blocks - rounds * slots;
    const double last = rest == 0 ? 0 : 3 + per * (rest <= 256 ? 0.4 : rest <= 512 ? 0.55 : 1) * each;
    double us = rounds * (4.5 + each * per) + last;
    if (splits > 1) us += 4 + (double)M * N * (6.0 * splits + 2) / 4.5e6;
    if (us < least) {
      least = us;
      best = Shape{kPlainTile, per, tiles, us};
    }
  }
  return best;
}

// A pass of the product: lays its operands out, multiplies, joins. `run` false: takes the workspace, launches nothing.
struct Pass {
  Carve ws;
  bool run;
  hipStream_t st;
  int rc = SE_OK;
  int tile = 0, splits = 1;   // of the last product; tile 0: none was chosen
  void launched() {
    if (rc == SE_OK && hipGetLastError() != hipSuccess) rc = SE_E_LAUNCH;
  }

  // 16-bit [R][C] at ld, as it is or packed (by lay()): off 16 bytes, or rows further apart than a tile's offsets reach
  PackJobs packs{};
  int n_packs = 0;
  Mat half(const void* x, long long ld, int R, int C) {
    Mat m{};
    if (ld % 8 == 0 && C % 8 == 0 && ((uintptr_t)x & 15) == 0 && ld <= kMostLd) {
      m.p = static_cast<const u16*>(x);
      m.ld = ld;
      m.bytes = ((long long)(R - 1) * ld + C) * 2;
      return m;
    }
    const int Cp = up8(C);
    u16* out = ws.take<u16>((long long)R * Cp);
    packs.j[n_packs++] = PackJob{static_cast<const u16*>(x), out, ld, R, C, Cp};
    m.p = out;
    m.ld = Cp;
    m.bytes = (long long)R * Cp * 2;
    return m;
  }
  // fp32 [R][C] at ld as hi and lo, powers of two by row (reduced along the row) or by column (along the column); what is
  // registered is laid out by lay(). top: the columns' largest magnitudes over `parts` chunks of rows, if they are known
  SplitJobs by_rows{}, by_cols{};
  int n_rows = 0, n_cols = 0;
  Mat planes(const void* xv, long long ld, int R, int C, bool by_row, float* top = nullptr, int parts = 0) {
    SplitJob t{};
    t.x = static_cast<const float*>(xv);
    t.ld = ld;
    t.R = R; t.C = C;
    t.width = by_row ? (C + 31) / 32 * 32 : up8(C);
    t.two = ld % 2 == 0 && ((uintptr_t)xv & 7) == 0;
    Mat m{};
    m.ld = by_row ? 2LL * t.width : t.width;
    m.bytes = (by_row ? (long long)R : 2LL * ((R + 31) / 32 * 32)) * m.ld * 2;
    u16* out = ws.take<u16>(m.bytes / 2);
    m.p = out;
    m.ex = t.ex = ws.take<short>(by_row ? R : C);
    t.out = reinterpret_cast<unsigned*>(out);
    if (!by_row) {
      t.known = parts > 0;
      t.rows = std::max(64, (R + 255) / 256);
      t.parts = t.known ? parts : (R + t.rows - 1) / t.rows;
      t.part = t.known ? top : ws.take<float>((long long)t.parts * C);
    }
    if (by_row) by_rows.j[n_rows++] = t;
    else by_cols.j[n_cols++] = t;
    return m;
  }
  void lay() {
    if (!run || rc != SE_OK) return;
    if (n_packs) {
      unsigned blocks = 0;
      for (int i = 0; i < n_packs; ++i) blocks = std::max(blocks, blocks_for((long long)packs.j[i].R * packs.j[i].Cp / 8));
      hipLaunchKernelGGL(linear_pack_kernel, dim3(blocks, 1, n_packs), dim3(256), 0, st, packs);
    }
    if (n_rows) {
      long long most = 0;
      for (int i = 0; i < n_rows; ++i) most = std::max(most, (by_rows.j[i].R + 3LL) / 4);
      const dim3 grid((unsigned)std::min<long long>(most, 1 << 20), 1, n_rows);
      hipLaunchKernelGGL(linear_split_rows_kernel, grid, dim3(256), 0, st, by_rows);
    }
    if (n_cols) {
      int C = 0, parts = 0;
      unsigned blocks = 0;
      for (int i = 0; i < n_cols; ++i) {
        const SplitJob& t = by_cols.j[i];
        C = std::max(C, t.C);
        if (!t.known) parts = std::max(parts, t.parts);
        blocks = std::max(blocks, blocks_for((t.R + 31LL) / 32 * 32 * t.width / 2));
      }
      if (parts) hipLaunchKernelGGL(linear_col_max_kernel, dim3((C + 255) / 256, parts, n_cols), dim3(256), 0, st, by_cols);
      hipLaunchKernelGGL(linear_col_exp_kernel, dim3((C + 63) / 64, 1, n_cols), dim3(1024), 0, st, by_cols);
      hipLaunchKernelGGL(linear_split_cols_kernel, dim3(blocks, 1, n_cols), dim3(256), 0, st, by_cols);
    }
    n_packs = n_rows = n_cols = 0;
    launched();
  }

  template <typename H, typename S, bool AKC, bool BKC, bool RES>
  void start(const GemmArgs& a, const Shape& c) {
    const dim3 grid((unsigned)c.tiles, a.splits);
    if (c.tile == 256)
      hipLaunchKernelGGL((linear_gemm_kernel<H, S, AKC, BKC, RES, 256, 256, 2, 2>), grid, dim3(256), 0, st, a);
    else
      hipLaunchKernelGGL((linear_gemm_kernel<H, S, AKC, BKC, RES, 128, 128, 2, 2>), grid, dim3(256), 0, st, a);
  }
  // fp32: the operands as they lie, where that is estimated to be faster than laying planes out (tiles 0: it is not)
  template <bool AKC, bool BKC>
  Shape plain_of(const void* A, long long lda, const void* B, long long ldb, int M, int N, int K) {
    const bool avec = lda % 4 == 0 && ((uintptr_t)A & 15) == 0, bvec = ldb % 4 == 0 && ((uintptr_t)B & 15) == 0;
    auto slow = [](bool kc, bool vec) { return kc ? (vec ? 0 : 1.4) : 0.5; };
    const Shape c = plain_shape_of(M, N, (K + kPlainK - 1) / kPlainK, 2.6 + slow(AKC, avec) + slow(BKC, bvec));
    // planes: a launch and one pass over an operand by rows, three and two by columns, two of a kind in the same launches
    auto laid = [](bool kc, double n) { return kc ? 4 + n * 8 / 4.5e6 : 9 + n * 12 / 4.5e6; };
    const double planes = shape_of(M, N, (2 * ((K + 31) / 32 * 32) + kBK - 1) / kBK, 1.5).us + laid(AKC, (double)M * K) +
                          laid(BKC, (double)N * K) - (AKC != BKC ? 0 : AKC ? 2 : 6);
    return c.us > planes || c.tiles > 0xffffff ? Shape{} : c;
  }
  template <bool AKC, bool BKC>
  void plain(const void* A, long long lda, const void* B, long long ldb, int M, int N, int K, const Epi& e, const Shape& c) {
    GemmArgs a{};
    a.M = M; a.N = N; a.K = K;
    a.A = static_cast<const u16*>(A); a.B = static_cast<const u16*>(B);
    a.lda = lda; a.ldb = ldb;
    a.e = e;
    a.steps = (K + kPlainK - 1) / kPlainK;
    const bool avec = lda % 4 == 0 && ((uintptr_t)A & 15) == 0, bvec = ldb % 4 == 0 && ((uintptr_t)B & 15) == 0;
    a.per = c.per;
    a.splits = splits = (a.steps + a.per - 1) / a.per;
    tile = c.tile;
    if (a.splits > 1) a.slab = ws.take<float>((long long)a.splits * M * N);
    if (!run || rc != SE_OK) return;
    hipLaunchKernelGGL((linear_plain_kernel<AKC, BKC>), dim3((unsigned)c.tiles, a.splits), dim3(256), 0, st, a, avec, bvec);
    launched();
    if (a.splits > 1) join<float>(a);
  }
  template <typename H, typename S, bool AKC, bool BKC>
  void product(const Mat& A, const Mat& B, int M, int N, int K, const Epi& e) {
    GemmArgs a{};
    a.M = M; a.N = N; a.K = K;
    a.lda = A.ld; a.ldb = B.ld; a.a_bytes = A.bytes; a.b_bytes = B.bytes;
    a.A = A.p; a.B = B.p;
    a.e = e;
    a.e.ea = A.ex; a.e.eb = B.ex;
    if (__is_same(S, float)) a.K = 2 * ((K + 31) / 32 * 32);   // 32 k of hi and of lo to a tile
    if (A.ld > 2 * kMostLd || B.ld > 2 * kMostLd) { rc = SE_E_UNSUPPORTED; return; }   // hi and lo side by side
    a.steps = (a.K + kBK - 1) / kBK;
    const Shape c = shape_of(M, N, a.steps, sizeof(S) == 4 ? 1.5 : 1);
    a.per = c.per;
    a.splits = splits = (a.steps + a.per - 1) / a.per;
    tile = c.tile;
    if (a.splits > 1) a.slab = ws.take<float>((long long)a.splits * M * N);
    if (!run || rc != SE_OK) return;
    const bool res = e.res && a.splits == 1;
    if constexpr (AKC && BKC) {   // the forward alone has one
      if (res) start<H, S, AKC, BKC, true>(a, c);
      else start<H, S, AKC, BKC, false>(a, c);
    } else {
      start<H, S, AKC, BKC, false>(a, c);
    }
    launched();
    if (a.splits > 1) join<S>(a);
  }
  template <typename S>
  void join(const GemmArgs& a) {
    const Epi& e = a.e;
    const int N = a.N;
    // 4 columns a thread where the rows of everything are aligned for it
    auto ok = [&](int v) {
      const uintptr_t al = std::min<int>(16, v * sizeof(S)) - 1;
      return N % v == 0 && (((uintptr_t)e.C | (uintptr_t)e.bias | (uintptr_t)e.res) & al) == 0 && e.ldc % v == 0 &&
             (!e.res || e.ldr % v == 0);
    };
    const long long mn = (long long)a.M * N;
    if (ok(4)) hipLaunchKernelGGL((linear_join_kernel<S, 4>), dim3(blocks_for(mn / 4)), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((linear_join_kernel<S, 1>), dim3(blocks_for(mn)), dim3(256), 0, st, a);
    launched();
  }
};

constexpr int kFewRows = SE_LINEAR_FEW_ROWS;

template <typename S, int MT>
void launch_few(const S* x, long long ldx, const S* w, long long ldw, int M, int N, int K, const Epi& e, bool vec,
                hipStream_t st) {
  const int ks = 64 / sizeof(S), most = MT == 4 ? 8 : 16;
  int waves = 1;
  while (waves < most && waves * 8 * ks < K) waves *= 2;   // eight fetches of 16 bytes a lane are under way at once
  const dim3 grid((N + 15) / 16), block(waves * 64);
  const size_t lds = (size_t)waves * MT * 256 * sizeof(float);
  if (vec) hipLaunchKernelGGL((linear_few_kernel<S, true, MT>), grid, block, lds, st, x, ldx, w, ldw, M, N, K, e);
  else hipLaunchKernelGGL((linear_few_kernel<S, false, MT>), grid, block, lds, st, x, ldx, w, ldw, M, N, K, e);
}

template <typename S> struct Product { using H = S; };
template <> struct Product<float> { using H = _Float16; };

template <typename S>
int forward(const se_linear_desc* d, const void* x, const void* w, const void* bias, const void* res, void* y, void* z,
            Pass& p) {
  using H = typename Product<S>::H;
  constexpr bool f32 = __is_same(S, float);
  Epi e{};
  e.C = y; e.z = z; e.bias = bias; e.res = res; e.ldc = d->N; e.ldr = d->ldr; e.ldz = up8(d->N); e.act = d->act;
  if (d->M <= kFewRows) {
    if (!p.run) return p.rc;
    const int v = 16 / sizeof(S);
    const bool vec = d->K % v == 0 && d->ldx % v == 0 && d->ldw % v == 0 && (((uintptr_t)x | (uintptr_t)w) & 15) == 0;
    const S* xs = static_cast<const S*>(x);
    const S* ws = static_cast<const S*>(w);
    if (d->M <= 16) launch_few<S, 1>(xs, d->ldx, ws, d->ldw, d->M, d->N, d->K, e, vec, p.st);
    else if (d->M <= 32) launch_few<S, 2>(xs, d->ldx, ws, d->ldw, d->M, d->N, d->K, e, vec, p.st);
    else launch_few<S, 4>(xs, d->ldx, ws, d->ldw, d->M, d->N, d->K, e, vec, p.st);
    p.launched();
    return p.rc;
  }
  if constexpr (f32) {
    const Shape c = p.template plain_of<true, true>(x, d->ldx, w, d->ldw, d->M, d->N, d->K);
    if (c.tiles) {
      p.template plain<true, true>(x, d->ldx, w, d->ldw, d->M, d->N, d->K, e, c);
      return p.rc;
    }
  }
  const Mat A = f32 ? p.planes(x, d->ldx, d->M, d->K, true) : p.half(x, d->ldx, d->M, d->K);
  const Mat B = f32 ? p.planes(w, d->ldw, d->N, d->K, true) : p.half(w, d->ldw, d->N, d->K);
  p.lay();
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
  const int Np = up8(N);
  S* g = prod && !as_is ? p.ws.template take<S>((long long)M * Np) : nullptr;
  int cg = 1;
  while (cg < 64 && cg * 8 < Np) cg *= 2;
  // chunks of rows: about 2048 workgroups, each of at least four turns
  const int across = (Np + cg * 8 - 1) / (cg * 8), turn = 256 / cg;
  const long long chunks = std::max(1, std::min(512, 2048 / across));
  const int rows = (int)std::max<long long>(4 * turn, (M + chunks - 1) / chunks), parts = (M + rows - 1) / rows;
  float* part = db ? p.ws.template take<float>((long long)parts * N) : nullptr;
  const void* gp = as_is ? dy : g;
  const long long ldg = as_is ? d->ldr : Np;
  Shape cx{}, cw{};
  if constexpr (f32) {
    if (dx) cx = p.template plain_of<true, false>(gp, ldg, w, d->ldw, M, K, N);
    if (dw) cw = p.template plain_of<false, false>(gp, ldg, x, d->ldx, N, K, M);
  }
  // the pass over dy leaves the largest magnitudes of g's columns where dW's planes need them
  const bool passes = db || (prod && !as_is), tops = f32 && dw && !cw.tiles && passes;
  float* top = tops ? p.ws.template take<float>((long long)parts * N) : nullptr;
  if (p.run && passes) {
    const bool vec = N % 8 == 0 && ((uintptr_t)dy & 15) == 0 && d->ldr % (16 / sizeof(S)) == 0;
    const S* zs = sloped ? static_cast<const S*>(z) : nullptr;
    const S* dys = static_cast<const S*>(dy);
    if (vec)
      hipLaunchKernelGGL((linear_slope_kernel<S, true>), dim3(across, parts), dim3(256), 0, p.st, dys, d->ldr, zs, d->act,
                         M, N, Np, cg, rows, g, part, top);
    else
      hipLaunchKernelGGL((linear_slope_kernel<S, false>), dim3(across, parts), dim3(256), 0, p.st, dys, d->ldr, zs, d->act,
                         M, N, Np, cg, rows, g, part, top);
    p.launched();
    if (part) {
      hipLaunchKernelGGL(linear_bias_kernel<S>, dim3((N + 63) / 64), dim3(1024), 0, p.st, part, parts, N,
                         static_cast<S*>(db));
      p.launched();
    }
  }
  Epi ex{}, ew{};
  ex.C = dx; ex.ldc = K;
  ew.C = dw; ew.ldc = K;
  Mat A{}, B{}, Aw{}, Bw{};
  if (dx && !cx.tiles) {
    A = f32 ? p.planes(gp, ldg, M, N, true) : p.half(gp, ldg, M, as_is ? N : Np);
    B = f32 ? p.planes(w, d->ldw, N, K, false) : p.half(w, d->ldw, N, K);
  }
  if (dw && !cw.tiles) {
    Aw = f32 ? p.planes(gp, ldg, M, N, false, top, tops ? parts : 0) : dx ? A : p.half(gp, ldg, M, as_is ? N : Np);
    Bw = f32 ? p.planes(x, d->ldx, M, K, false) : p.half(x, d->ldx, M, K);
  }
  p.lay();
  if (dx) {
    if constexpr (f32)
      if (cx.tiles) p.template plain<true, false>(gp, ldg, w, d->ldw, M, K, N, ex, cx);
    if (!cx.tiles) p.template product<H, S, true, false>(A, B, M, K, N, ex);
  }
  if (dw) {
    if constexpr (f32)
      if (cw.tiles) p.template plain<false, false>(gp, ldg, x, d->ldx, N, K, M, ew, cw);
    if (!cw.tiles) p.template product<H, S, false, false>(Aw, Bw, N, K, M, ew);
  }
  return p.rc;
}

int check(const se_linear_desc* d) {
  if (!d || d->M <= 0 || d->N <= 0 || d->K <= 0) return SE_E_ARG;
  if (d->dtype != SE_DTYPE_F32 && d->dtype != SE_DTYPE_BF16 && d->dtype != SE_DTYPE_F16) return SE_E_ARG;
  if (d->act < SE_LINACT_NONE || d->act > SE_LINACT_SILU) return SE_E_ARG;
  if (d->ldw < d->K || d->ldx < 0 || (d->M > 1 && d->ldx < d->K) || d->ldr < 0 || (d->M > 1 && d->ldr && d->ldr < d->N))
    return SE_E_ARG;
  if (d->N > kMostLd || d->K > kMostLd) return SE_E_UNSUPPORTED;
  // indexes of rows are 32-bit, of fp32's hi and lo rows too; a launch has less than 2^32 threads
  const long long most = 1LL << 37, M = d->M, N = d->N, K = d->K;
  if (M > (1 << 28) || M * N > most || M * K > most || N * K > most) return SE_E_UNSUPPORTED;
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
  if (!x || !w || !y || ((uintptr_t)z & 15) || ((uintptr_t)ws & 15)) return SE_E_ARG;
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

extern "C" int se_linear_tile(const se_linear_desc* d, int product, int* splits) {
  const int rc = check(d);
  if (rc != SE_OK) return rc;
  if (product < 0 || product > 2) return SE_E_ARG;
  Pass p{Carve{nullptr}, false, nullptr};
  char* some = reinterpret_cast<char*>(256);   // on 16 bytes, never read
  if (product == 0) forward_any(d, some, some, nullptr, nullptr, nullptr, nullptr, p);
  else backward_any(d, some, some, some, nullptr, product == 1 ? some : nullptr, product == 2 ? some : nullptr, nullptr, p);
  if (p.rc != SE_OK) return p.rc;
  if (splits) *splits = p.splits;
  return p.tile;
}

extern "C" int se_linear_bwd(const se_linear_desc* d, const void* dy, const void* x, const void* w, const void* z, void* dx,
                             void* dw, void* db, void* ws, size_t ws_bytes, void* stream) {
  const int rc = check(d);
  if (rc != SE_OK) return rc;
  if (!dy || (dx && !w) || (dw && !x) || (!dx && !dw && !db) || (d->act != SE_LINACT_NONE && !z)) return SE_E_ARG;
  if ((d->M > 1 && d->ldr < d->N) || ((uintptr_t)z & 15) || ((uintptr_t)ws & 15)) return SE_E_ARG;
  const size_t need = se_linear_bwd_workspace_size(d, dy, x, w, dx != nullptr, dw != nullptr, db != nullptr);
  if (need && (!ws || ws_bytes < need)) return SE_E_WORKSPACE;
  Pass p{Carve{static_cast<char*>(ws)}, true, se::as_stream(stream)};
  return backward_any(d, dy, x, w, z, dx, dw, db, p);
}
