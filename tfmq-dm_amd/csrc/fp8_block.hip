// Linears on e4m3 operands with one fp32 scale per block of 128 (activations: a row x 128 channels; weights: 128 x 128; both gradients' operands:
// 128 tokens down a column).
//
// A block whose largest magnitude is a (at least 2^-100) has the scale s = fl32(a / 448) and the stored values q = e4m3(fl32(x fl32(448 / a))),
// round half even; a NaN or an infinity makes its whole block NaN.  The product of two quantised rows is
//     y[m, n] = sum_b s_x[m, b] s_w[n, b] (sum_{k in block b} q_x[m, k] q_w[n, k])
// -- the inner sum is what two v_mfma_f32_32x32x64_f8f6f4 (K = 128) return in fp32 from a zero accumulator, the outer one an fp32 FMA per
// output and block.  The hardware's own block scales are powers of two, so fp32 scales have to be applied by the VALU.
//
// The 8-bit MFMA aligns each group of 8 products to the group's largest and drops what lies below 2^-13 of it (measured; the groups meet in
// fp32): 1.4e-5 of a 64-term sum of normal values, 1 / 15 of fp16's own rounding of the result and 1 / 120 of bf16's.  Outputs of 16 bits take
// it.  fp32 outputs (a weight's gradient among them) do not: their fragments are widened in registers to fp16, which holds every e4m3 value,
// and multiplied by v_mfma_f32_32x32x16_f16 (6e-9 in the same measurement), at half the matrix rate and two conversions per four bytes.
#include "conv_common.hpp"
#include <type_traits>

typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));

namespace {

constexpr float F8_MAX = 448.0f;
constexpr float AMAX_MIN = 7.888609052210118e-31f;      // 2^-100: keeps both the scale and its reciprocal normal numbers

enum { DT_F32 = 0, DT_F16 = 1, DT_BF16 = 2 };
template <int DT> struct Elem;
template <> struct Elem<DT_F32> { using type = float; };
template <> struct Elem<DT_F16> { using type = _Float16; };
template <> struct Elem<DT_BF16> { using type = __bf16; };

// magnitudes compare as integers: a NaN is larger than an infinity, so the maximum carries it
__device__ __forceinline__ unsigned mag_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }
__device__ __forceinline__ float2 block_scale(unsigned amax_bits) {      // {reciprocal, scale}
  const unsigned lo = __float_as_uint(AMAX_MIN);
  const float a = __uint_as_float(amax_bits < lo ? lo : amax_bits);
  return make_float2(F8_MAX / a, a / F8_MAX);
}
// four values -> four e4m3 bytes (v_cvt_pk_fp8_f32 rounds half to even; |x r| <= 448 (1 + 2^-23) rounds to 448, never past it)
__device__ __forceinline__ unsigned pack4_f8(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return static_cast<unsigned>(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true));
}

// 8 consecutive elements of a row from column c (zeros from column K on)
template <int DT, bool VEC>
__device__ __forceinline__ void load8(const typename Elem<DT>::type* row, int c, int K, float (&v)[8]) {
  using T = typename Elem<DT>::type;
  if (VEC) {          // row 16-byte aligned, K % 8 == 0
    if (c < K) {
      if constexpr (DT == DT_F32) {
        const float4 a = *reinterpret_cast<const float4*>(row + c), b = *reinterpret_cast<const float4*>(row + c + 4);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
      } else {
        typedef T v8t __attribute__((ext_vector_type(8)));
        const v8t a = *reinterpret_cast<const v8t*>(row + c);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = static_cast<float>(a[i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = 0.0f;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c + i < K ? static_cast<float>(row[c + i]) : 0.0f;
  }
}

// ---- rows: q [M][Kp], s [Kb][M].  16 lanes hold one block of one row (8 values each); a workgroup takes 16 rows of one block column, so the
// scales leave as 64 contiguous bytes.  HBM-bound: 2 (4) bytes read and 1 written per element.
template <int DT, bool VEC>
__global__ __launch_bounds__(256) void k_quant_rows(const typename Elem<DT>::type* __restrict__ x, long M, int K, long ld, uint8_t* __restrict__ q,
                                                    float* __restrict__ s, int Kb) {
  const int lane16 = threadIdx.x & 15, sub = threadIdx.x >> 4;
  const long nrow = (M + 15) / 16, nt = nrow * Kb;
  for (long t = blockIdx.x; t < nt; t += gridDim.x) {
    const long m = (t / Kb) * 16 + sub;
    const int kb = static_cast<int>(t % Kb);
    if (m >= M) continue;
    float v[8];
    load8<DT, VEC>(x + m * ld, kb * 128 + lane16 * 8, K, v);
    unsigned a = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) a = max(a, mag_bits(v[i]));
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) a = max(a, static_cast<unsigned>(__shfl_xor(static_cast<int>(a), o, 16)));
    const float2 sc = block_scale(a);
    uint2 w;
    w.x = pack4_f8(v[0] * sc.x, v[1] * sc.x, v[2] * sc.x, v[3] * sc.x);
    w.y = pack4_f8(v[4] * sc.x, v[5] * sc.x, v[6] * sc.x, v[7] * sc.x);
    *reinterpret_cast<uint2*>(q + (m * Kb + kb) * 128 + lane16 * 8) = w;
    if (lane16 == 0) s[static_cast<long>(kb) * M + m] = sc.y;
  }
}

// ---- columns: x [M][K] -> q [K][Mp] with one scale per column and block of 128 rows, s [Mb][K].  A workgroup takes 128 rows x 64 columns:
// thread (column c = tid & 63, row quarter tid >> 6) holds 32 values, the column's maximum meets in LDS, the bytes are transposed through LDS
// and leave as 128-byte rows.
template <int DT>
__global__ __launch_bounds__(256) void k_quant_cols(const typename Elem<DT>::type* __restrict__ x, long M, int K, long ld, uint8_t* __restrict__ q,
                                                    float* __restrict__ s, long Mp) {
  __shared__ unsigned amax[4][64];
  __shared__ __attribute__((aligned(16))) unsigned bytes[64][33];
  const int nkt = (K + 63) / 64;
  const long mb = blockIdx.x / nkt;
  const int k0 = static_cast<int>(blockIdx.x % nkt) * 64;
  const int c = threadIdx.x & 63, qr = threadIdx.x >> 6;
  const int k = k0 + c;
  float v[32];
  unsigned a = 0;
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    const long m = mb * 128 + qr * 32 + i;
    v[i] = (k < K && m < M) ? static_cast<float>(x[m * ld + k]) : 0.0f;
    a = max(a, mag_bits(v[i]));
  }
  amax[qr][c] = a;
  __syncthreads();
  a = max(max(amax[0][c], amax[1][c]), max(amax[2][c], amax[3][c]));
  const float2 sc = block_scale(a);
  if (qr == 0 && k < K) s[mb * K + k] = sc.y;
#pragma unroll
  for (int i = 0; i < 8; ++i) bytes[c][qr * 8 + i] = pack4_f8(v[4 * i] * sc.x, v[4 * i + 1] * sc.x, v[4 * i + 2] * sc.x, v[4 * i + 3] * sc.x);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int idx = threadIdx.x + i * 256, row = idx >> 5, w = idx & 31;
    if (k0 + row < K) *reinterpret_cast<unsigned*>(q + static_cast<long>(k0 + row) * Mp + mb * 128 + w * 4) = bytes[row][w];
  }
}

// ---- weights: w fp32 [N][K] -> q [N][Kp] and its transpose qt [K][Np], s [Nb][Kb]; one workgroup per 128 x 128 block, run once per layer
__global__ __launch_bounds__(256) void k_pack_w_f8(const float* __restrict__ w, int N, int K, uint8_t* __restrict__ q, uint8_t* __restrict__ qt,
                                                   float* __restrict__ s) {
  __shared__ unsigned red[256];
  __shared__ uint8_t tile[128][132];
  const int Kb = (K + 127) / 128, Nb = (N + 127) / 128;
  const int nb = blockIdx.x / Kb, kb = blockIdx.x % Kb;
  const int kk = threadIdx.x & 127, half = threadIdx.x >> 7, k = kb * 128 + kk;
  unsigned a = 0;
  for (int r = half; r < 128; r += 2) {
    const int n = nb * 128 + r;
    if (n < N && k < K) a = max(a, mag_bits(w[static_cast<long>(n) * K + k]));
  }
  red[threadIdx.x] = a;
  __syncthreads();
  for (int o = 128; o > 0; o >>= 1) {
    if (static_cast<int>(threadIdx.x) < o) red[threadIdx.x] = max(red[threadIdx.x], red[threadIdx.x + o]);
    __syncthreads();
  }
  const float2 sc = block_scale(red[0]);
  if (threadIdx.x == 0) s[nb * Kb + kb] = sc.y;
  for (int r = half; r < 128; r += 2) {
    const int n = nb * 128 + r;
    const float v = (n < N && k < K) ? w[static_cast<long>(n) * K + k] * sc.x : 0.0f;
    const uint8_t b = static_cast<uint8_t>(pack4_f8(v, 0.0f, 0.0f, 0.0f) & 0xff);
    tile[r][kk] = b;
    if (n < N) q[(static_cast<long>(n) * Kb + kb) * 128 + kk] = b;
  }
  __syncthreads();
  for (int r = half; r < 128; r += 2)
    if (kb * 128 + r < K) qt[(static_cast<long>(kb * 128 + r) * Nb + nb) * 128 + kk] = tile[kk][r];
}

// ---- a lane's 32 bytes of one 64-channel half of a block, as the two matrix instructions take them
template <bool WIDE> struct Frag;
template <> struct Frag<false> {
  v8i b;
  __device__ __forceinline__ void set(int i, unsigned w) { b[i] = static_cast<int>(w); }
  __device__ __forceinline__ void done() {}
  static __device__ __forceinline__ v16f mul(const Frag& w, const Frag& x, v16f d) {
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w.b, x.b, d, 0, 0, 0, 0, 0, 0);
  }
};
template <> struct Frag<true> {
  v8i b;
  v8h f[4];
  __device__ __forceinline__ void set(int i, unsigned w) { b[i] = static_cast<int>(w); }
  __device__ __forceinline__ void done() {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const v2h lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b[i], 1.0f, false), hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b[i], 1.0f, true);
      f[i >> 1][(i & 1) * 4] = lo[0]; f[i >> 1][(i & 1) * 4 + 1] = lo[1]; f[i >> 1][(i & 1) * 4 + 2] = hi[0]; f[i >> 1][(i & 1) * 4 + 3] = hi[1];
    }
  }
  static __device__ __forceinline__ v16f mul(const Frag& w, const Frag& x, v16f d) {
#pragma unroll
    for (int c = 0; c < 4; ++c) d = __builtin_amdgcn_mfma_f32_32x32x16_f16(w.f[c], x.f[c], d, 0, 0, 0);
    return d;
  }
};

struct GemmF8P {
  const uint8_t *a, *b;        // a: [M][Kp] (the output's rows), b: [N][Kp] (its columns)
  const float *sa, *sb;        // sa [Kb][M]; sb: [(n / 128) * sbn + kb * sbk] per block of columns, or (SBROW) [Kb][N] per column
  long sbn, sbk;
  const float* bias;
  void* y;
  long M;
  int N, Kb;
  int tm, tn;                  // tiles along M, N
};

// one 16-byte piece of a 128-byte operand row lives at slot (piece ^ key(row)): 8 consecutive lanes of a fragment read hit 8 different slots
__device__ __forceinline__ int key_x(int r) { return r & 7; }
__device__ __forceinline__ int key_w(int r) { return (r & 3) | ((r >> 2) & 4); }

template <int YDT>
__device__ __forceinline__ void store_run(typename Elem<YDT>::type* p, const float* v, int n, bool vec) {
  // up to 16 consecutive outputs of one row
  using T = typename Elem<YDT>::type;
  if (vec && n == 16) {
    if constexpr (YDT == DT_F32) {
#pragma unroll
      for (int i = 0; i < 4; ++i) reinterpret_cast<float4*>(p)[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
    } else {
      typedef T v8t __attribute__((ext_vector_type(8)));
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        v8t o;
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = static_cast<T>(v[8 * i + e]);
        reinterpret_cast<v8t*>(p)[i] = o;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (i < n) p[i] = static_cast<T>(v[i]);
  }
}

// The product.  The MFMA computes W_tile X_tile^T, so a lane owns ONE row m of the output (its scale is one register) and its 16 accumulators are
// columns n; the rows of W enter the fragment in the order n = 16 h + 4 a + c for fragment row 8 a + 4 h + c, so those 16 columns are consecutive.
// Operand tiles of one block (128 bytes a row) travel by LDS-DMA into two stages, the next one in flight while this one is multiplied.
template <int BM, int BN, int WM, int WN, int YDT, bool SBROW>
__global__ __launch_bounds__(64 * (BM / WM) * (BN / WN), 2) void k_gemm_f8(GemmF8P p) {
  constexpr int NWM = BM / WM, NWN = BN / WN, NW = NWM * NWN, TM = WM / 32, TN = WN / 32;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  constexpr int STAGE = (BM + BN) * 128;
  using YT = typename Elem<YDT>::type;
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  const int j = lane & 31, hh = lane >> 5;
  const int wm = wid % NWM, wn = wid / NWM;
  const int tile = xcd_tile_id();
  const long m0 = static_cast<long>(tile % p.tm) * BM;
  const int n0 = (tile / p.tm) * BN;
  const long Kp = static_cast<long>(p.Kb) * 128;

  // ---- LDS-DMA plan: instruction i of a wave moves 8 rows x 128 bytes; rows [0, BN) of a stage are W, [BN, BN + BM) X
  constexpr int NI = (BM + BN) / 8 / NW;
  static_assert((BM + BN) % (8 * NW) == 0 && BN % 8 == 0, "whole rows per wave instruction");
  const uint8_t* src[NI];
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int row = (wid * NI + i) * 8 + (lane >> 3), slot = lane & 7;
    if (row < BN) {
      const int n = min(n0 + row, p.N - 1);
      src[i] = p.b + static_cast<long>(n) * Kp + ((slot ^ key_w(row)) << 4);
    } else {
      const int r = row - BN;
      const long m = min(m0 + r, p.M - 1);
      src[i] = p.a + m * Kp + ((slot ^ key_x(r)) << 4);
    }
  }
  const unsigned lds0 = static_cast<unsigned>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) unsigned char*)smem));
  auto fetch = [&](int kb, int st) {
#pragma unroll
    for (int i = 0; i < NI; ++i) glds16(src[i] + static_cast<long>(kb) * 128, __builtin_amdgcn_readfirstlane(lds0 + st * STAGE + (wid * NI + i) * 1024));
  };
  long mrow[TM];
#pragma unroll
  for (int t = 0; t < TM; ++t) mrow[t] = min(m0 + wm * WM + t * 32 + j, p.M - 1);
  const int nbase = n0 + wn * WN;

  v16f acc[TN][TM];
#pragma unroll
  for (int u = 0; u < TN; ++u)
#pragma unroll
    for (int t = 0; t < TM; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[u][t][r] = 0.0f;

  float sx[TM], sxn[TM] = {};
  const int nb_last = (p.N - 1) >> 7;
#pragma unroll
  for (int t = 0; t < TM; ++t) sx[t] = p.sa[mrow[t]];
  fetch(0, 0);
  for (int kb = 0; kb < p.Kb; ++kb) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();                 // this stage has arrived for every wave, and every wave is through with the other one
    if (kb + 1 < p.Kb) {
#pragma unroll
      for (int t = 0; t < TM; ++t) sxn[t] = p.sa[static_cast<long>(kb + 1) * p.M + mrow[t]];
      fetch(kb + 1, (kb + 1) & 1);
    }
    const unsigned char* sW = smem + (kb & 1) * STAGE;
    const unsigned char* sX = sW + BN * 128;
    using F = Frag<YDT == DT_F32>;
    F xf[TM][2];
#pragma unroll
    for (int t = 0; t < TM; ++t) {
      const int r = wm * WM + t * 32 + j;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint4 w = *reinterpret_cast<const uint4*>(sX + r * 128 + (((s * 4 + hh * 2 + e) ^ key_x(r)) << 4));
          xf[t][s].set(4 * e, w.x); xf[t][s].set(4 * e + 1, w.y); xf[t][s].set(4 * e + 2, w.z); xf[t][s].set(4 * e + 3, w.w);
        }
        xf[t][s].done();
      }
    }
#pragma unroll
    for (int u = 0; u < TN; ++u) {
      const int i = 16 * ((j >> 2) & 1) + 4 * (j >> 3) + (j & 3);          // fragment row j holds this row of the 32
      const int r = wn * WN + u * 32 + i;
      F wf[2];
#pragma unroll
      for (int s = 0; s < 2; ++s) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint4 w = *reinterpret_cast<const uint4*>(sW + r * 128 + (((s * 4 + hh * 2 + e) ^ key_w(r)) << 4));
          wf[s].set(4 * e, w.x); wf[s].set(4 * e + 1, w.y); wf[s].set(4 * e + 2, w.z); wf[s].set(4 * e + 3, w.w);
        }
        wf[s].done();
      }
      float sw = 0.0f, swr[16];
      if constexpr (SBROW) {
#pragma unroll
        for (int r2 = 0; r2 < 16; ++r2) swr[r2] = p.sb[static_cast<long>(kb) * p.N + min(nbase + u * 32 + 16 * hh + r2, p.N - 1)];
      } else {
        sw = p.sb[static_cast<long>(min((nbase + u * 32) >> 7, nb_last)) * p.sbn + kb * p.sbk];
      }
#pragma unroll
      for (int t = 0; t < TM; ++t) {
        v16f z;
#pragma unroll
        for (int r2 = 0; r2 < 16; ++r2) z[r2] = 0.0f;
        const v16f d = F::mul(wf[1], xf[t][1], F::mul(wf[0], xf[t][0], z));
        if constexpr (SBROW) {
#pragma unroll
          for (int r2 = 0; r2 < 16; ++r2) acc[u][t][r2] = __builtin_fmaf(d[r2], sx[t] * swr[r2], acc[u][t][r2]);
        } else {
          const float f = sx[t] * sw;
#pragma unroll
          for (int r2 = 0; r2 < 16; ++r2) acc[u][t][r2] = __builtin_fmaf(d[r2], f, acc[u][t][r2]);
        }
      }
    }
#pragma unroll
    for (int t = 0; t < TM; ++t) sx[t] = sxn[t];
  }
  // ---- lane (row m, half hh) holds columns u * 32 + 16 hh + (0 .. 15)
  const bool vec = (p.N * sizeof(YT)) % 16 == 0;
#pragma unroll
  for (int t = 0; t < TM; ++t) {
    const long m = m0 + wm * WM + t * 32 + j;
    if (m >= p.M) continue;
#pragma unroll
    for (int u = 0; u < TN; ++u) {
      const int n = nbase + u * 32 + 16 * hh;
      const int cnt = min(16, p.N - n);
      if (cnt <= 0) continue;
      float v[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) v[r] = acc[u][t][r] + ((p.bias && r < cnt) ? p.bias[n + r] : 0.0f);
      store_run<YDT>(reinterpret_cast<YT*>(p.y) + m * p.N + n, v, cnt, vec);
    }
  }
}

template <int BM, int BN, int WM, int WN, int YDT, bool SBROW>
int launch_gemm(tfmq_handle h, GemmF8P p, hipStream_t st) {
  constexpr int smem = 2 * (BM + BN) * 128;
  auto kern = &k_gemm_f8<BM, BN, WM, WN, YDT, SBROW>;
  TFMQ_HIP(h, hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, smem));
  p.tm = ceil_div(p.M, BM);
  p.tn = ceil_div(p.N, BN);
  const long nb = static_cast<long>(p.tm) * p.tn;
  TFMQ_CHECK_ARG(h, nb < (1L << 31), "gemm_fp8: too many tiles");
  hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>(nb)), dim3(64 * (BM / WM) * (BN / WN)), smem, st, p);
  TFMQ_LAUNCH_CHECK(h);
  return TFMQ_OK;
}

template <int DT>
int launch_quant_rows(tfmq_handle h, const void* x, long M, int K, long ld, uint8_t* q, float* s, hipStream_t st) {
  using T = typename Elem<DT>::type;
  const int Kb = (K + 127) / 128;
  const long nt = (M + 15) / 16 * Kb;
  const unsigned grid = static_cast<unsigned>(nt < 65536 ? nt : 65536);
  const bool vec = K % 8 == 0 && (ld * sizeof(T)) % 16 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0;
  if (vec) hipLaunchKernelGGL((k_quant_rows<DT, true>), dim3(grid), dim3(256), 0, st, static_cast<const T*>(x), M, K, ld, q, s, Kb);
  else hipLaunchKernelGGL((k_quant_rows<DT, false>), dim3(grid), dim3(256), 0, st, static_cast<const T*>(x), M, K, ld, q, s, Kb);
  TFMQ_LAUNCH_CHECK(h);
  return TFMQ_OK;
}

template <int DT>
int launch_quant_cols(tfmq_handle h, const void* x, long M, int K, long ld, uint8_t* q, float* s, hipStream_t st) {
  using T = typename Elem<DT>::type;
  const long Mb = (M + 127) / 128, nb = Mb * ((K + 63) / 64);
  TFMQ_CHECK_ARG(h, nb < (1L << 31), "quantize_fp8: too many blocks");
  hipLaunchKernelGGL((k_quant_cols<DT>), dim3(static_cast<unsigned>(nb)), dim3(256), 0, st, static_cast<const T*>(x), M, K, ld, q, s, Mb * 128);
  TFMQ_LAUNCH_CHECK(h);
  return TFMQ_OK;
}

// ---- few rows (M <= 32 a workgroup): one launch, W read once straight into the fragments, the activations quantised on the way in.  Eight waves
// share the K blocks of 32 columns; a lane holds row j's elements [32 hh, +32) of each 64-channel half of a block, so a block's largest magnitude
// is 64 values and one exchange between the two half waves.  The partial sums meet in LDS in the waves' order (no atomics).
struct SmallF8P {
  const void* x;
  long ld;
  int M, K;
  const uint8_t* w;
  const float* ws;             // [Nb][Kb]
  const float* bias;
  void* y;
  int N, Kb;
};
template <int DT, bool VEC, int YDT>
__global__ __launch_bounds__(512) void k_linear_f8_small(SmallF8P p) {
  constexpr int NW = 8;
  using T = typename Elem<DT>::type;
  using YT = typename Elem<YDT>::type;
  __shared__ float part[NW][32][33];
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6, j = lane & 31, hh = lane >> 5;
  const int n0 = blockIdx.x * 32, m0 = blockIdx.y * 32;
  const T* xrow = static_cast<const T*>(p.x) + static_cast<long>(min(m0 + j, p.M - 1)) * p.ld;
  const uint8_t* wrow = p.w + static_cast<long>(min(n0 + j, p.N - 1)) * p.Kb * 128;
  const float* wsc = p.ws + static_cast<long>(n0 >> 7) * p.Kb;
  v16f acc;
#pragma unroll
  for (int r = 0; r < 16; ++r) acc[r] = 0.0f;
  for (int kb = wid; kb < p.Kb; kb += NW) {
    uint4 wv[4];
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int e = 0; e < 2; ++e) wv[2 * s + e] = *reinterpret_cast<const uint4*>(wrow + kb * 128 + s * 64 + hh * 32 + e * 16);
    const float sw = wsc[kb];
    float v[2][4][8];
    unsigned a = 0;
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        load8<DT, VEC>(xrow, kb * 128 + s * 64 + hh * 32 + g * 8, p.K, v[s][g]);
#pragma unroll
        for (int i = 0; i < 8; ++i) a = max(a, mag_bits(v[s][g][i]));
      }
    a = max(a, static_cast<unsigned>(__shfl_xor(static_cast<int>(a), 32, 64)));
    const float2 sc = block_scale(a);
    v16f d;
#pragma unroll
    for (int r = 0; r < 16; ++r) d[r] = 0.0f;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      Frag<YDT == DT_F32> xf, wf;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const float(&e)[8] = v[s][g];
        xf.set(2 * g, pack4_f8(e[0] * sc.x, e[1] * sc.x, e[2] * sc.x, e[3] * sc.x));
        xf.set(2 * g + 1, pack4_f8(e[4] * sc.x, e[5] * sc.x, e[6] * sc.x, e[7] * sc.x));
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint4 w = wv[2 * s + e];
        wf.set(4 * e, w.x); wf.set(4 * e + 1, w.y); wf.set(4 * e + 2, w.z); wf.set(4 * e + 3, w.w);
      }
      xf.done();
      wf.done();
      d = Frag<YDT == DT_F32>::mul(wf, xf, d);
    }
    const float f = sc.y * sw;
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[r] = __builtin_fmaf(d[r], f, acc[r]);
  }
#pragma unroll
  for (int r = 0; r < 16; ++r) part[wid][j][8 * (r >> 2) + 4 * hh + (r & 3)] = acc[r];
  __syncthreads();
#pragma unroll
  for (int it = 0; it < 2; ++it) {
    const int idx = tid + it * 512, m = idx >> 5, n = idx & 31;
    if (m0 + m >= p.M || n0 + n >= p.N) continue;
    float t = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; ++w) t += part[w][m][n];
    if (p.bias) t += p.bias[n0 + n];
    static_cast<YT*>(p.y)[static_cast<long>(m0 + m) * p.N + n0 + n] = static_cast<YT>(t);
  }
}

template <int DT>
int launch_small(tfmq_handle h, const SmallF8P& p, int y_dtype, hipStream_t st) {
  using T = typename Elem<DT>::type;
  const dim3 grid(static_cast<unsigned>((p.N + 31) / 32), static_cast<unsigned>((p.M + 31) / 32));
  const bool vec = p.K % 8 == 0 && (p.ld * sizeof(T)) % 16 == 0 && reinterpret_cast<uintptr_t>(p.x) % 16 == 0;
  auto go = [&](auto v, auto y) { hipLaunchKernelGGL((k_linear_f8_small<DT, decltype(v)::value, decltype(y)::value>), grid, dim3(512), 0, st, p); };
  auto pick = [&](auto y) { vec ? go(std::true_type{}, y) : go(std::false_type{}, y); };
  if (y_dtype == DT_F32) pick(std::integral_constant<int, DT_F32>{});
  else if (y_dtype == DT_F16) pick(std::integral_constant<int, DT_F16>{});
  else pick(std::integral_constant<int, DT_BF16>{});
  TFMQ_LAUNCH_CHECK(h);
  return TFMQ_OK;
}

}  // namespace

extern "C" int tfmq_quantize_fp8(tfmq_handle h, const void* x, int dtype, long M, int K, long ld, int by_column, uint8_t* q, float* s, void* stream) {
  DeviceGuard guard(h);
  TFMQ_CHECK_ARG(h, h && x && q && s, "quantize_fp8: null pointer");
  TFMQ_CHECK_ARG(h, M > 0 && K > 0 && ld >= K && dtype >= 0 && dtype <= 2, "quantize_fp8: bad shape or type");
  hipStream_t st = as_stream(stream);
  if (by_column) {
    if (dtype == DT_F32) return launch_quant_cols<DT_F32>(h, x, M, K, ld, q, s, st);
    return dtype == DT_F16 ? launch_quant_cols<DT_F16>(h, x, M, K, ld, q, s, st) : launch_quant_cols<DT_BF16>(h, x, M, K, ld, q, s, st);
  }
  if (dtype == DT_F32) return launch_quant_rows<DT_F32>(h, x, M, K, ld, q, s, st);
  return dtype == DT_F16 ? launch_quant_rows<DT_F16>(h, x, M, K, ld, q, s, st) : launch_quant_rows<DT_BF16>(h, x, M, K, ld, q, s, st);
}

extern "C" int tfmq_pack_w_fp8(tfmq_handle h, const float* w, int N, int K, uint8_t* q, uint8_t* qt, float* s, void* stream) {
  DeviceGuard guard(h);
  TFMQ_CHECK_ARG(h, h && w && q && qt && s && N > 0 && K > 0, "pack_w_fp8: bad argument");
  const long nb = static_cast<long>((N + 127) / 128) * ((K + 127) / 128);
  TFMQ_CHECK_ARG(h, nb < (1L << 31), "pack_w_fp8: too many blocks");
  hipLaunchKernelGGL(k_pack_w_f8, dim3(static_cast<unsigned>(nb)), dim3(256), 0, as_stream(stream), w, N, K, q, qt, s);
  TFMQ_LAUNCH_CHECK(h);
  return TFMQ_OK;
}

extern "C" int tfmq_gemm_fp8(tfmq_handle h, const uint8_t* a, const float* sa, const uint8_t* b, const float* sb, long sbn, long sbk, int sb_row,
                             const float* bias, void* y, int y_dtype, long M, int N, int Kb, void* stream) {
  DeviceGuard guard(h);
  TFMQ_CHECK_ARG(h, h && a && sa && b && sb && y, "gemm_fp8: null pointer");
  TFMQ_CHECK_ARG(h, M > 0 && N > 0 && Kb > 0 && y_dtype >= 0 && y_dtype <= 2, "gemm_fp8: bad shape or type");
  TFMQ_CHECK_ARG(h, !sb_row || y_dtype == DT_F32, "gemm_fp8: a scale per column comes with an fp32 output");
  TFMQ_CHECK_ARG(h, reinterpret_cast<uintptr_t>(a) % 16 == 0 && reinterpret_cast<uintptr_t>(b) % 16 == 0 && reinterpret_cast<uintptr_t>(y) % 16 == 0,
                 "gemm_fp8: operands and output must be 16-byte aligned");
  GemmF8P p{a, b, sa, sb, sbn, sbk, bias, y, M, N, Kb, 0, 0};
  hipStream_t st = as_stream(stream);
  if (sb_row) return launch_gemm<128, 128, 64, 64, DT_F32, true>(h, p, st);
  if (y_dtype == DT_F32) return launch_gemm<128, 128, 64, 64, DT_F32, false>(h, p, st);
  if (y_dtype == DT_F16) return launch_gemm<128, 128, 64, 64, DT_F16, false>(h, p, st);
  return launch_gemm<128, 128, 64, 64, DT_BF16, false>(h, p, st);
}

extern "C" int tfmq_linear_fp8_small(tfmq_handle h, const void* x, int dtype, long M, int K, long ld, const uint8_t* w, const float* ws, const float* bias,
                                     void* y, int y_dtype, int N, void* stream) {
  DeviceGuard guard(h);
  TFMQ_CHECK_ARG(h, h && x && w && ws && y, "linear_fp8_small: null pointer");
  TFMQ_CHECK_ARG(h, M > 0 && M <= 1024 && N > 0 && K > 0 && ld >= K && dtype >= 0 && dtype <= 2 && y_dtype >= 0 && y_dtype <= 2,
                 "linear_fp8_small: bad shape (at most 1024 rows) or type");
  TFMQ_CHECK_ARG(h, reinterpret_cast<uintptr_t>(w) % 16 == 0, "linear_fp8_small: weights must be 16-byte aligned");
  const SmallF8P p{x, ld, static_cast<int>(M), K, w, ws, bias, y, N, (K + 127) / 128};
  if (dtype == DT_F32) return launch_small<DT_F32>(h, p, y_dtype, as_stream(stream));
  return dtype == DT_F16 ? launch_small<DT_F16>(h, p, y_dtype, as_stream(stream)) : launch_small<DT_BF16>(h, p, y_dtype, as_stream(stream));
}
