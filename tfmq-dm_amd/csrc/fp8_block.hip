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
#include <algorithm>
#include <type_traits>

typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));

namespace {

constexpr float F8_MAX = 448.0f;
constexpr float AMAX_MIN = 7.888609052210118e-31f;      // 2^-100: keeps both the scale and its reciprocal normal numbers

enum { DT_F32 = 0, DT_F16 = 1, DT_BF16 = 2, DT_PART = 3 };          // DT_PART: fp32 partial sums of a 16-bit result (its products)
template <int DT> struct Elem;
template <> struct Elem<DT_F32> { using type = float; };
template <> struct Elem<DT_F16> { using type = _Float16; };
template <> struct Elem<DT_BF16> { using type = __bf16; };
template <> struct Elem<DT_PART> { using type = float; };

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

// 8 consecutive elements of a row from column c (zeros from column K on).  Inside the row they are one 16-byte load (fp32: two) at any alignment of
// the elements; VEC: rows are 16-byte aligned and K % 8 == 0, so that a group is inside or outside as a whole.
struct Raw8 {
  uint4 a, b;          // 16-bit types: a
};
template <int ES, bool VEC>
__device__ __forceinline__ Raw8 raw8(const char* row, int c, int K) {
  Raw8 r{make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
  const char* p = row + static_cast<long>(c) * ES;
  if (VEC ? c < K : c + 8 <= K) {
    __builtin_memcpy(&r.a, p, 16);
    if (ES == 4) __builtin_memcpy(&r.b, p + 16, 16);
  } else if (!VEC && c < K) {
    unsigned w[8] = {};
    unsigned short h[8] = {};
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < K) {
        if (ES == 4) __builtin_memcpy(&w[i], p + i * 4, 4);
        else __builtin_memcpy(&h[i], p + i * 2, 2);
      }
    if (ES == 4) {
      r.a = make_uint4(w[0], w[1], w[2], w[3]);
      r.b = make_uint4(w[4], w[5], w[6], w[7]);
    } else {
      r.a = make_uint4(h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16);
    }
  }
  return r;
}
template <int DT>
__device__ __forceinline__ void widen8(const Raw8& r, float (&v)[8]) {
  if constexpr (DT == DT_F32) {
    v[0] = __uint_as_float(r.a.x); v[1] = __uint_as_float(r.a.y); v[2] = __uint_as_float(r.a.z); v[3] = __uint_as_float(r.a.w);
    v[4] = __uint_as_float(r.b.x); v[5] = __uint_as_float(r.b.y); v[6] = __uint_as_float(r.b.z); v[7] = __uint_as_float(r.b.w);
  } else {
    typedef typename Elem<DT>::type v8t __attribute__((ext_vector_type(8)));
    const v8t t = __builtin_bit_cast(v8t, r.a);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = static_cast<float>(t[i]);
  }
}
template <int DT, bool VEC>
__device__ __forceinline__ void load8(const typename Elem<DT>::type* row, int c, int K, float (&v)[8]) {
  widen8<DT>(raw8<DT == DT_F32 ? 4 : 2, VEC>(reinterpret_cast<const char*>(row), c, K), v);
}

// ---- rows: q [M][Kp], s [Kb][M].  16 lanes hold one block of one row (8 values each); a workgroup takes 16 rows of one block column, so the
// scales leave as 64 contiguous bytes.  HBM-bound: 2 (4) bytes read and 1 written per element; 16384 x 1280 fp16: 14 us (4.5 TB/s).
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

// ---- columns: x [M][K] -> qc [K][Mp] with one scale per column and block of 128 rows, sc [Mb][K]; the row form (q, s as above) from the same
// values where it is wanted too, so that an upstream gradient, which both products read, is read once.  A workgroup takes 128 rows x 128 columns, a
// thread 4 x 8 of them; the columns' maxima meet in LDS, the bytes are transposed through LDS and leave as 128-byte rows.  HBM-bound: 8192 x (640 + 640)
// bf16, the first 640 in both forms: 12 us (3.1 TB/s; four waves a tile and conflicts in the transposition: 14.4).
struct QuantTileP {
  const void* x;
  int dt, vec;                 // type code; rows 16-byte aligned and K % 8 == 0
  long M, ld;
  int K, Kb;
  uint8_t *q, *qc;
  float *s, *sc;               // q, s null: columns only
};
// the thread's 4 rows of 8: all loads before the first conversion
template <int ES, bool VEC>
__device__ __forceinline__ void tile_raw(const QuantTileP& p, long m0, int k, Raw8 (&r)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    r[i] = Raw8{make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
    if (m0 + i < p.M) r[i] = raw8<ES, VEC>(static_cast<const char*>(p.x) + (m0 + i) * p.ld * ES, k, p.K);
  }
}
struct QuantLds {
  unsigned amax[8][128];          // per wave and column
  float scale[128];               // reciprocals
  unsigned bytes[128][36];        // 16-byte pieces of a column's 128 bytes at piece ^ (column >> 4): the writes, four bytes of 16 columns 8 apart, spread over the banks
};
template <int DT>
__device__ __forceinline__ void quant_tile_of(const QuantTileP& p, int t, QuantLds& L) {
  constexpr int ES = DT == DT_F32 ? 4 : 2;
  const long mb = t / p.Kb, Mp = (p.M + 127) / 128 * 128;
  const int kb = t % p.Kb;
  const int cg = threadIdx.x & 15, rg = threadIdx.x >> 4, k = kb * 128 + cg * 8;
  const long m0 = mb * 128 + rg * 4;
  Raw8 raw[4];
  if (p.vec) tile_raw<ES, true>(p, m0, k, raw);
  else tile_raw<ES, false>(p, m0, k, raw);
  float v[4][8];
  unsigned cm[8] = {};
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    widen8<DT>(raw[r], v[r]);
#pragma unroll
    for (int e = 0; e < 8; ++e) cm[e] = max(cm[e], mag_bits(v[r][e]));
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    cm[e] = max(cm[e], static_cast<unsigned>(__shfl_xor(static_cast<int>(cm[e]), 16, 64)));
    cm[e] = max(cm[e], static_cast<unsigned>(__shfl_xor(static_cast<int>(cm[e]), 32, 64)));
  }
  if ((threadIdx.x & 63) < 16) {
    *reinterpret_cast<uint4*>(&L.amax[threadIdx.x >> 6][cg * 8]) = make_uint4(cm[0], cm[1], cm[2], cm[3]);
    *reinterpret_cast<uint4*>(&L.amax[threadIdx.x >> 6][cg * 8 + 4]) = make_uint4(cm[4], cm[5], cm[6], cm[7]);
  }
  if (p.q) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      unsigned a = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) a = max(a, mag_bits(v[r][e]));
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) a = max(a, static_cast<unsigned>(__shfl_xor(static_cast<int>(a), o, 16)));
      const float2 sc = block_scale(a);
      if (m0 + r < p.M) {
        uint2 w;
        w.x = pack4_f8(v[r][0] * sc.x, v[r][1] * sc.x, v[r][2] * sc.x, v[r][3] * sc.x);
        w.y = pack4_f8(v[r][4] * sc.x, v[r][5] * sc.x, v[r][6] * sc.x, v[r][7] * sc.x);
        *reinterpret_cast<uint2*>(p.q + ((m0 + r) * p.Kb + kb) * 128 + cg * 8) = w;
        if (cg == 0) p.s[static_cast<long>(kb) * p.M + m0 + r] = sc.y;
      }
    }
  }
  __syncthreads();
  if (threadIdx.x < 128) {
    unsigned a = 0;
#pragma unroll
    for (int w = 0; w < 8; ++w) a = max(a, L.amax[w][threadIdx.x]);
    const float2 sc = block_scale(a);
    L.scale[threadIdx.x] = sc.x;
    if (kb * 128 + static_cast<int>(threadIdx.x) < p.K) p.sc[mb * p.K + kb * 128 + threadIdx.x] = sc.y;
  }
  __syncthreads();
  const float4 s0 = *reinterpret_cast<const float4*>(&L.scale[cg * 8]), s1 = *reinterpret_cast<const float4*>(&L.scale[cg * 8 + 4]);
  const float sr[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
#pragma unroll
  for (int e = 0; e < 8; ++e) L.bytes[cg * 8 + e][rg ^ ((cg >> 1) << 2)] = pack4_f8(v[0][e] * sr[e], v[1][e] * sr[e], v[2][e] * sr[e], v[3][e] * sr[e]);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int idx = threadIdx.x + i * 512, row = idx >> 3, pc = idx & 7;
    if (kb * 128 + row < p.K)
      *reinterpret_cast<uint4*>(p.qc + static_cast<long>(kb * 128 + row) * Mp + mb * 128 + pc * 16) = *reinterpret_cast<const uint4*>(&L.bytes[row][(pc ^ (row >> 4)) * 4]);
  }
}
// one launch for up to two tensors (n0 tiles of the first)
struct QuantPairP {
  QuantTileP t[2];
};
__global__ __launch_bounds__(512) void k_quant_cols(QuantPairP pr, int n0) {
  __shared__ __attribute__((aligned(16))) QuantLds L;
  const int second = static_cast<int>(blockIdx.x) >= n0, t = blockIdx.x - (second ? n0 : 0);
  const QuantTileP& p = pr.t[second];
  if (p.dt == DT_F32) quant_tile_of<DT_F32>(p, t, L);
  else if (p.dt == DT_F16) quant_tile_of<DT_F16>(p, t, L);
  else quant_tile_of<DT_BF16>(p, t, L);
}

// ---- weights: w fp32 [N][K] -> q [N][Kp] and its transpose qt [K][Np], s [Nb][Kb]; one workgroup per 128 x 128 block, run once per layer (640 x 640: 38 us)
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
  int nslice;                  // slices of the Kb blocks: slice s writes fp32 partials at y + s * M * N
};

// one 16-byte piece of a 128-byte operand row lives at slot (piece ^ key(row)): 8 consecutive lanes of a fragment read hit 8 different slots
__device__ __forceinline__ int key_x(int r) { return r & 7; }
__device__ __forceinline__ int key_w(int r) { return (r & 3) | ((r >> 2) & 4); }

// The product.  The MFMA computes W_tile X_tile^T, so a lane owns ONE row m of the output (its scale is one register) and its 16 accumulators are
// columns n; the rows of W enter the fragment in the order n = 16 h + 4 a + c for fragment row 8 a + 4 h + c, so those 16 columns are consecutive.
// Operand tiles of one block (128 bytes a row) and its scales travel by LDS-DMA into S stages, S - 1 of them in flight while one is multiplied.
// Everything that a block needs comes this way: a compiler-counted load would wait for all LDS-DMA behind it.  A workgroup walks over its tiles (or,
// sliced, one K range of a tile) as one sequence of blocks: the next tile's first stages are under way while the results of this one are rounded and
// stored.
// What bounds it: the LDS-DMA of the operands, the fragment reads, the matrix instructions and the VALU that scales every block's result take about as long as
// each other, and the barrier of a stage lets them overlap only between the two waves of a SIMD.  16384 x 1280 x 10240 fp16 out (256 x 256 tiles, half the
// operand bytes of 128 x 128): 262 us, 1.6 PFLOP/s, MFMA busy 38 %, VALU 37 %,
// LDS 32 % and 14 % conflicts of the LDS-DMA's writes with the reads (nothing is full: the steps of a block follow each other).  Fragments of block b + 1 in registers under the products of
// b: 256 x 128 tiles spill 68 bytes, 177 against 134 us at 8192 x 1280 x 10240; without spills (eight waves of 32 x 64) 44.7 against 41.6 us at
// 1024 x 5120 x 1280.  8192 x 320 x 2560 (three blocks a tile): 24 us, 42 MB of stores.
template <int BM, int BN, int WM, int WN, int YDT, bool SBROW, int S>
struct GemmF8 {
  static constexpr int NWM = BM / WM, NWN = BN / WN, NW = NWM * NWN;
  static constexpr int STAGE = (BM + BN) * 128, NSC = BM / 64 + (SBROW ? BN / 64 : 1), SCALES = NSC * 256;
  static constexpr int LDS = S * (STAGE + SCALES);
};
template <int BM, int BN, int WM, int WN, int YDT, bool SBROW, int S>
__device__ __forceinline__ void gemm_f8(const GemmF8P& p, unsigned char* smem, int bid, int nblocks, int first) {
  using G = GemmF8<BM, BN, WM, WN, YDT, SBROW, S>;
  constexpr int NWM = G::NWM, NW = G::NW, TM = WM / 32, TN = WN / 32, STAGE = G::STAGE;
  using YT = typename Elem<YDT>::type;
  using F = Frag<YDT == DT_F32>;
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int j = lane & 31, hh = lane >> 5;
  const int wm = wid % NWM, wn = wid / NWM;
  const long Kp = static_cast<long>(p.Kb) * 128;
  const int ntile = p.tm * p.tn;

  // ---- LDS-DMA plan: instruction i of a wave moves 8 rows x 128 bytes; rows [0, BN) of a stage are W, [BN, BN + BM) X; a wave moves one of them.
  // One more instruction a wave moves 64 scales: rows of X first, then (SBROW) columns or the column blocks' (surplus waves repeat a piece).
  constexpr int NI = (BM + BN) / 8 / NW, PER = NI + 1;
  static_assert((BM + BN) % (8 * NW) == 0 && BN % (8 * NI) == 0, "whole rows per wave instruction, one operand per wave");
  static_assert(G::NSC <= NW && BN % 128 == 0 && 128 % WN == 0, "a wave per 64 scales; a wave's columns share a block");
  const unsigned lds0 = static_cast<unsigned>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) unsigned char*)smem));
  const bool is_w = wid * NI * 8 < BN;
  const int sc = wid % G::NSC;
  const bool sc_x = sc < BM / 64;
  const int nb_last = (p.N - 1) >> 7;
  // neighbouring workgroups of an XCD share rows and columns: groups of 8 row tiles walk the columns
  auto origin = [&](int tile, long& m, int& n) {
    const int gsz = 8 * p.tn, grp = tile / gsz, first = grp * 8, rows = min(p.tm - first, 8), in = tile - grp * gsz;
    m = static_cast<long>(first + in % rows) * BM;
    n = (in / rows) * BN;
  };
  unsigned voff[NI], soff = 0;
  const uint8_t* src = nullptr;
  const float* ssrc = nullptr;
  auto place = [&](int tile) {
    long m0;
    int n0;
    origin(tile, m0, n0);
    src = uniform_ptr(is_w ? p.b + n0 * Kp : p.a + m0 * Kp);
    const int last_m = __builtin_amdgcn_readfirstlane(static_cast<int>(min(static_cast<long>(BM), p.M - m0) - 1)), last_n = p.N - 1 - n0;
    const unsigned last = is_w ? last_n : last_m;
    const int r0 = (is_w ? wid : wid - BN / (8 * NI)) * NI * 8 + (lane >> 3);
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int r = r0 + 8 * i;
      voff[i] = min(static_cast<unsigned>(r), last) * static_cast<unsigned>(Kp) + (((lane & 7) ^ (is_w ? key_w(r) : key_x(r))) << 4);
      asm volatile("" : "+v"(voff[i]));          // kept, not recomputed for every block
    }
    if (sc_x) {
      ssrc = p.sa + m0;
      soff = 4 * min(sc * 64 + lane, last_m);
    } else if (SBROW) {
      ssrc = p.sb + n0;
      soff = 4 * min((sc - BM / 64) * 64 + lane, last_n);
    } else {
      ssrc = p.sb + static_cast<long>(n0 >> 7) * p.sbn;
      soff = 4 * static_cast<unsigned>(min(min(lane, BN / 128 - 1), nb_last - (n0 >> 7))) * static_cast<unsigned>(p.sbn);
    }
    ssrc = uniform_ptr(ssrc);
    asm volatile("" : "+v"(soff));
  };
  const long sstep = sc_x ? p.M : SBROW ? p.N : p.sbk;
  auto fetch = [&](int kb, int st) {
    const uint8_t* base = uniform_ptr(src + static_cast<long>(kb) * 128);
    const unsigned dst = __builtin_amdgcn_readfirstlane(lds0 + st * STAGE + wid * NI * 1024);
#pragma unroll
    for (int i = 0; i < NI; ++i)
      asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(voff[i]), "s"(base), "s"(dst + i * 1024) : "memory", "m0");
    const float* sbase = uniform_ptr(ssrc + kb * sstep);
    const unsigned sdst = __builtin_amdgcn_readfirstlane(lds0 + S * STAGE + st * G::SCALES + sc * 256);
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1" ::"v"(soff), "s"(sbase), "s"(sdst) : "memory", "m0");
  };
  // this workgroup's slice of the blocks, and its tiles
  const int sl = p.nslice > 1 ? bid % p.nslice : 0;
  const int per = (p.Kb + p.nslice - 1) / p.nslice, k_lo = sl * per, k_hi = min(p.Kb, k_lo + per);
  int tile = p.nslice > 1 ? bid / p.nslice : first;
  const int stride = p.nslice > 1 ? ntile : nblocks;
  if (tile >= ntile) return;

  // fragment addresses inside a stage: four 16-byte pieces of a row (the sub-tiles are immediates)
  const int rw = wn * WN + 16 * ((j >> 2) & 1) + 4 * (j >> 3) + (j & 3), rx = wm * WM + j;          // fragment row j of W holds row rw
  unsigned pw[4], px[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int piece = (q >> 1) * 4 + hh * 2 + (q & 1);
    pw[q] = rw * 128 + ((piece ^ key_w(rw)) << 4);
    px[q] = BN * 128 + rx * 128 + ((piece ^ key_x(rx)) << 4);
  }
  v16f acc[TN][TM];
  // one block of a stage: products into acc
  auto block = [&](int st) {
    const unsigned char* D = smem + st * STAGE;
    const float* sS = reinterpret_cast<const float*>(smem + S * STAGE + st * G::SCALES);
    float sx[TM];
#pragma unroll
    for (int t = 0; t < TM; ++t) sx[t] = sS[rx + t * 32];
    if constexpr (!SBROW) {
      const float sb = sS[BM + ((wn * WN) >> 7)];
#pragma unroll
      for (int t = 0; t < TM; ++t) sx[t] *= sb;
    }
    F wf[TN][2];
    float swr[SBROW ? TN : 1][16];
#pragma unroll
    for (int u = 0; u < TN; ++u) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const uint4 w = *reinterpret_cast<const uint4*>(D + pw[q] + u * 32 * 128);
        F& f = wf[u][q >> 1];
        f.set(4 * (q & 1), w.x); f.set(4 * (q & 1) + 1, w.y); f.set(4 * (q & 1) + 2, w.z); f.set(4 * (q & 1) + 3, w.w);
      }
      wf[u][0].done();
      wf[u][1].done();
      if constexpr (SBROW) {
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) {
          const float4 v = *reinterpret_cast<const float4*>(sS + BM + wn * WN + u * 32 + 16 * hh + 4 * q4);
          swr[u][4 * q4] = v.x; swr[u][4 * q4 + 1] = v.y; swr[u][4 * q4 + 2] = v.z; swr[u][4 * q4 + 3] = v.w;
        }
      }
    }
#pragma unroll
    for (int t = 0; t < TM; ++t) {
      F xf[2];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const uint4 w = *reinterpret_cast<const uint4*>(D + px[q] + t * 32 * 128);
        F& f = xf[q >> 1];
        f.set(4 * (q & 1), w.x); f.set(4 * (q & 1) + 1, w.y); f.set(4 * (q & 1) + 2, w.z); f.set(4 * (q & 1) + 3, w.w);
      }
      xf[0].done();
      xf[1].done();
#pragma unroll
      for (int u = 0; u < TN; ++u) {
        const v16f z = {};
        // (a wave that has its operands goes first: 8192 x 1280 x 10240 135 -> 131 us.  With two workgroups a CU it gains nothing, the gradients' launch loses 2)
        if constexpr (BM == 256) __builtin_amdgcn_s_setprio(1);
        const v16f d = F::mul(wf[u][1], xf[1], F::mul(wf[u][0], xf[0], z));
        if constexpr (BM == 256) __builtin_amdgcn_s_setprio(0);
        if constexpr (SBROW) {
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[u][t][r] = __builtin_fmaf(d[r], sx[t] * swr[u][r], acc[u][t][r]);
        } else {
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[u][t][r] = __builtin_fmaf(d[r], sx[t], acc[u][t][r]);
        }
      }
    }
  };

  // the fetches run S - 1 blocks ahead of the products, over the tiles' ends: (ft, fk) is the next one, `ahead` stages are under way or have arrived
  int ft = k_lo < k_hi ? tile : ntile, fk = k_lo, ahead = 0;
  auto fetch_next = [&](int st) {
    if (ft >= ntile) return;
    if (fk == k_lo) place(ft);
    fetch(fk, st);
    ++ahead;
    if (++fk == k_hi) {
      fk = k_lo;
      ft += stride;
    }
  };
#pragma unroll
  for (int s = 0; s < S - 1; ++s) fetch_next(s);
  // waits for the oldest stage: what was issued behind it may be under way -- `ahead` - 1 stages and, for S - 1 blocks behind a tile whose stores are
  // known (every lane, whole lines), those
  constexpr int NST = TM * TN * static_cast<int>(sizeof(YT));
  static_assert((S - 2) * PER + NST < 64, "the counter's range");
  auto arrive = [&](bool stores) {
    if (stores) {
      if (S >= 4 && ahead == 3) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * PER + NST) : "memory");
      else if (S >= 3 && ahead == 2) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(PER + NST) : "memory");
      else asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NST) : "memory");
    } else {
      if (S >= 4 && ahead == 3) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * PER) : "memory");
      else if (S >= 3 && ahead == 2) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(PER) : "memory");
      else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    --ahead;
  };
  static_assert(S >= 2 && S <= 4, "the waits above");
  int st = 0, stores = 0;
  for (; tile < ntile; tile += stride) {
#pragma unroll
    for (int u = 0; u < TN; ++u)
#pragma unroll
      for (int t = 0; t < TM; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[u][t][r] = 0.0f;
    for (int kb = k_lo; kb < k_hi; ++kb) {
      arrive(stores > 0);
      --stores;
      LDS_BARRIER();                   // this stage has arrived for every wave, and every wave is through with the one before it
      const int before = st == 0 ? S - 1 : st - 1;
      fetch_next(before);
      block(st);
      st = st == S - 1 ? 0 : st + 1;
    }
    // ---- lane (row m, half hh) holds columns u * 32 + 16 hh + (0 .. 15): out through LDS (this wave's part of the stage just multiplied), 32 rows x
    // 128 bytes at a time, so that the stores are whole lines; 16-byte piece c of row r at c ^ (r & 7)
    long mt;
    int n0;
    origin(tile, mt, n0);
    const int nbase = n0 + wn * WN;
    const bool full = (p.N * sizeof(YT)) % 16 == 0 && mt + BM <= p.M && n0 + BN <= p.N;
    YT* out = reinterpret_cast<YT*>(p.y) + (p.nslice > 1 ? static_cast<long>(sl) * p.M * p.N : 0);
    constexpr int CW = 128 / static_cast<int>(sizeof(YT)), UC = CW / 32, PE = 16 / static_cast<int>(sizeof(YT));
    static_assert(NW * 32 * 128 <= STAGE && WN % CW == 0, "the waves' store buffers fit a stage");
    const bool vec = (p.N * sizeof(YT)) % 16 == 0;
    LDS_BARRIER();                     // every wave is through with that stage
    unsigned char* sO = smem + (st == 0 ? S - 1 : st - 1) * STAGE + wid * 32 * 128;
#pragma unroll
    for (int c = 0; c < WN / CW; ++c) {
      const int nc = nbase + c * CW;
#pragma unroll
      for (int t = 0; t < TM; ++t) {
#pragma unroll
        for (int u = 0; u < UC; ++u) {
          float v[16];
#pragma unroll
          for (int r = 0; r < 16; ++r) v[r] = acc[c * UC + u][t][r];
          if (p.bias) {
            const int nl = nc + u * 32 + 16 * hh;
#pragma unroll
            for (int r = 0; r < 16; ++r) v[r] += p.bias[min(nl + r, p.N - 1)];
          }
          typedef YT vt __attribute__((ext_vector_type(PE)));
#pragma unroll
          for (int i = 0; i < 16 / PE; ++i) {
            vt o;
#pragma unroll
            for (int e = 0; e < PE; ++e) o[e] = static_cast<YT>(v[i * PE + e]);
            *reinterpret_cast<vt*>(sO + j * 128 + ((((u * 32 + 16 * hh) / PE + i) ^ (j & 7)) << 4)) = o;
          }
        }
        const long mb = mt + wm * WM + t * 32;
        if (vec) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int r = i * 8 + (lane >> 3), pc = lane & 7;
            const uint4 w = *reinterpret_cast<const uint4*>(sO + r * 128 + ((pc ^ (r & 7)) << 4));
            if (full || (mb + r < p.M && nc + pc * PE < p.N)) *reinterpret_cast<uint4*>(out + (mb + r) * p.N + nc + pc * PE) = w;
          }
        } else {
#pragma unroll 1
          for (int e = lane; e < 32 * CW; e += 64) {
            const int r = e / CW, n = e % CW;
            if (mb + r < p.M && nc + n < p.N) out[(mb + r) * p.N + nc + n] = reinterpret_cast<const YT*>(sO + r * 128 + (((n / PE) ^ (r & 7)) << 4))[n % PE];
          }
        }
      }
    }
    stores = full ? S - 1 : 0;
  }
}

template <int BM, int BN, int WM, int WN, int YDT, bool SBROW, int S>
__global__ __launch_bounds__(64 * (BM / WM) * (BN / WN), 2) void k_gemm_f8(GemmF8P p) {
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  gemm_f8<BM, BN, WM, WN, YDT, SBROW, S>(p, smem, blockIdx.x, gridDim.x, xcd_tile_id());
}
// a weight gradient's slices (the longer workgroups, first) and the other gradient's tiles in one launch: either alone leaves CUs idle.  8192 x 640 x 640
// bf16: 22 us (the weight's alone 17.7); eight waves and four stages (one workgroup a CU, every fragment widened twice) 30.
template <int YDT>
__global__ __launch_bounds__(256, 2) void k_gemm_f8_grads(GemmF8P gw, GemmF8P gx, int nw) {
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int q = blockIdx.x;
  if (q < nw) gemm_f8<128, 128, 64, 64, DT_F32, true, 2>(gw, smem, q, nw, q);
  else gemm_f8<128, 128, 64, 64, YDT, false, 2>(gx, smem, q - nw, gridDim.x - nw, q - nw);
}

// slices of the K axis, added in order (and the bias), rounded once; four outputs a thread (640 x 640 fp32, ten slices: 4.5 us)
template <int YDT>
__global__ __launch_bounds__(256) void k_sum_slices(const float* __restrict__ part, const float* __restrict__ bias, typename Elem<YDT>::type* __restrict__ y, long n, int N,
                                                    int nslice) {
  using YT = typename Elem<YDT>::type;
  const long i = (static_cast<long>(blockIdx.x) * 256 + threadIdx.x) * 4;
  if (i >= n) return;
  if (n % 4 == 0 && N % 4 == 0) {
    float4 a = make_float4(0, 0, 0, 0);
    for (int s = 0; s < nslice; ++s) {
      const float4 v = *reinterpret_cast<const float4*>(part + s * n + i);
      a.x += v.x; a.y += v.y; a.z += v.z; a.w += v.w;
    }
    if (bias) {
      const int c = static_cast<int>(i % N);
      a.x += bias[c]; a.y += bias[c + 1]; a.z += bias[c + 2]; a.w += bias[c + 3];
    }
    typedef YT v4t __attribute__((ext_vector_type(4)));
    v4t o;
    o[0] = static_cast<YT>(a.x); o[1] = static_cast<YT>(a.y); o[2] = static_cast<YT>(a.z); o[3] = static_cast<YT>(a.w);
    *reinterpret_cast<v4t*>(y + i) = o;
  } else {
    for (long e = i; e < min(n, i + 4); ++e) {
      float a = 0.0f;
      for (int s = 0; s < nslice; ++s) a += part[s * n + e];
      if (bias) a += bias[e % N];
      y[e] = static_cast<YT>(a);
    }
  }
}

template <int BM, int BN, int WM, int WN, int YDT, bool SBROW, int S>
int launch_gemm(tfmq_handle h, GemmF8P p, hipStream_t st) {
  using G = GemmF8<BM, BN, WM, WN, YDT, SBROW, S>;
  constexpr int NW = G::NW, smem = G::LDS;
  auto kern = &k_gemm_f8<BM, BN, WM, WN, YDT, SBROW, S>;
  static LdsRoom room_kern;
  TFMQ_HIP(h, room_kern.ask(h, reinterpret_cast<const void*>(kern), smem));
  p.tm = ceil_div(p.M, BM);
  p.tn = ceil_div(p.N, BN);
  const long nt = static_cast<long>(p.tm) * p.tn;
  TFMQ_CHECK_ARG(h, nt * 8 < (1L << 31), "gemm_fp8: too many tiles");
  const long room = static_cast<long>(h->cu_count) * (8 / NW);          // resident workgroups
  const long nb = p.nslice > 1 ? nt * p.nslice : (nt < room ? nt : room);
  hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>(nb)), dim3(64 * NW), smem, st, p);
  TFMQ_LAUNCH_CHECK(h);
  return TFMQ_OK;
}

// 128 x 128 tiles: with at most one a CU, eight waves of 32 x 64 and four stages; else two workgroups a CU, four waves of 64 x 64 and two stages.  us,
// the latter against the former, quantiser included: 1024 x 5120 x 1280 46.7 / 41.6, 512 x 1280 x 1280 15.3 / 14.1, 2048 x 768 x 1280 13.4 / 12.7.
// Eight waves at two workgroups a CU (126 registers, four waves a SIMD) gain nothing on full cards: 8192 x 320 x 2560 25.5 / 24.6,
// 16384 x 5120 x 1280 146 / 152.
template <int YDT, bool SBROW>
int launch_128(tfmq_handle h, const GemmF8P& p, hipStream_t st) {
  const long nb = static_cast<long>(ceil_div(p.M, 128)) * ceil_div(p.N, 128) * p.nslice;
  return nb <= h->cu_count ? launch_gemm<128, 128, 32, 64, YDT, SBROW, 4>(h, p, st) : launch_gemm<128, 128, 64, 64, YDT, SBROW, 2>(h, p, st);
}

bool rows_aligned(const void* x, int dtype, int K, long ld) {
  return K % 8 == 0 && (ld * (dtype == DT_F32 ? 4 : 2)) % 16 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0;
}
// by type code and alignment: f(integral_constant<dtype>, bool_constant<vec>)
template <typename F>
int for_input(const void* x, int dtype, int K, long ld, F f) {
  const bool vec = rows_aligned(x, dtype, K, ld);
  auto pick = [&](auto d) { return vec ? f(d, std::true_type{}) : f(d, std::false_type{}); };
  if (dtype == DT_F32) return pick(std::integral_constant<int, DT_F32>{});
  return dtype == DT_F16 ? pick(std::integral_constant<int, DT_F16>{}) : pick(std::integral_constant<int, DT_BF16>{});
}
QuantTileP quant_tiles(const void* x, int dtype, long M, int K, long ld, uint8_t* q, float* s, uint8_t* qc, float* sc) {
  return QuantTileP{x, dtype, rows_aligned(x, dtype, K, ld), M, ld, K, (K + 127) / 128, q, qc, s, sc};
}

int launch_quant_cols(tfmq_handle h, const QuantTileP& a, const QuantTileP* b, hipStream_t st) {
  auto tiles = [](const QuantTileP& p) { return (p.M + 127) / 128 * p.Kb; };
  const long na = tiles(a), n = na + (b ? tiles(*b) : 0);
  TFMQ_CHECK_ARG(h, n < (1L << 31), "quantize_fp8: too many blocks");
  hipLaunchKernelGGL(k_quant_cols, dim3(static_cast<unsigned>(n)), dim3(512), 0, st, QuantPairP{{a, b ? *b : a}}, static_cast<int>(na));
  TFMQ_LAUNCH_CHECK(h);
  return TFMQ_OK;
}

int launch_quant_rows(tfmq_handle h, const void* x, int dtype, long M, int K, long ld, uint8_t* q, float* s, hipStream_t st) {
  const int Kb = (K + 127) / 128;
  const long nt = (M + 15) / 16 * Kb;
  const unsigned grid = static_cast<unsigned>(nt < 65536 ? nt : 65536);
  return for_input(x, dtype, K, ld, [&](auto d, auto v) {
    using T = typename Elem<decltype(d)::value>::type;
    hipLaunchKernelGGL((k_quant_rows<decltype(d)::value, decltype(v)::value>), dim3(grid), dim3(256), 0, st, static_cast<const T*>(x), M, K, ld, q, s, Kb);
    TFMQ_LAUNCH_CHECK(h);
    return TFMQ_OK;
  });
}

// ---- few rows (M <= 32 a workgroup): one launch, W read once straight into the fragments, the activations quantised on the way in.  Eight waves
// share the K blocks of 32 columns; a lane holds row j's elements [32 hh, +32) of each 64-channel half of a block, so a block's largest magnitude
// is 64 values and one exchange between the two half waves.  The partial sums meet in LDS in the waves' order (no atomics).  Bound by two dependent trips to
// memory per wave and launch: 2 x 1280 x 1280 4.9 us, 154 x 768 x 1280 4.9, 32 x 1280 x 10240 9.7 (1.4 TB/s of W).
struct SmallF8P {
  const void* x;
  long ld;
  int M, K;
  const uint8_t* w;
  const float* ws;             // scale of (column block, k block) at ws[n * ws_n + k * ws_k]
  long ws_n, ws_k;
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
  const float* wsc = p.ws + static_cast<long>(n0 >> 7) * p.ws_n;
  v16f acc;
#pragma unroll
  for (int r = 0; r < 16; ++r) acc[r] = 0.0f;
  for (int kb = wid; kb < p.Kb; kb += NW) {
    uint4 wv[4];
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int e = 0; e < 2; ++e) wv[2 * s + e] = *reinterpret_cast<const uint4*>(wrow + kb * 128 + s * 64 + hh * 32 + e * 16);
    const float sw = wsc[kb * p.ws_k];
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

int launch_small(tfmq_handle h, const SmallF8P& p, int dtype, int y_dtype, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>((p.N + 31) / 32), static_cast<unsigned>((p.M + 31) / 32));
  return for_input(p.x, dtype, p.K, p.ld, [&](auto d, auto v) {
    auto go = [&](auto y) { hipLaunchKernelGGL((k_linear_f8_small<decltype(d)::value, decltype(v)::value, decltype(y)::value>), grid, dim3(512), 0, st, p); };
    if (y_dtype == DT_F32) go(std::integral_constant<int, DT_F32>{});
    else if (y_dtype == DT_F16) go(std::integral_constant<int, DT_F16>{});
    else go(std::integral_constant<int, DT_BF16>{});
    TFMQ_LAUNCH_CHECK(h);
    return TFMQ_OK;
  });
}

template <int YDT>
int launch_grads(tfmq_handle h, GemmF8P gw, GemmF8P gx, hipStream_t st) {
  constexpr int smem = GemmF8<128, 128, 64, 64, DT_F32, true, 2>::LDS;
  auto kern = &k_gemm_f8_grads<YDT>;
  static LdsRoom room;
  TFMQ_HIP(h, room.ask(h, reinterpret_cast<const void*>(kern), smem));
  gw.tm = ceil_div(gw.M, 128), gw.tn = ceil_div(gw.N, 128);
  gx.tm = ceil_div(gx.M, 128), gx.tn = ceil_div(gx.N, 128);
  const long nw = static_cast<long>(gw.tm) * gw.tn * gw.nslice, nx = static_cast<long>(gx.tm) * gx.tn;
  TFMQ_CHECK_ARG(h, (nw + nx) * 8 < (1L << 31), "linear_fp8_bwd: too many tiles");
  hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>(nw + nx)), dim3(256), smem, st, gw, gx, static_cast<int>(nw));
  TFMQ_LAUNCH_CHECK(h);
  return TFMQ_OK;
}

// ---- which kernel multiplies.  Tiles of 256 x 256 where they fill the card in whole rounds (at least three quarters of all), else 128 x 128.  us of the
// product alone, 128^2 / 256^2 in turn on one box, fastest of six, normal values: 16384 x 1280 x 10240 (10 rounds, full) 280 / 242; 8192 x 1280 x 10240 (five,
// full) 138 / 122; 6144 x 1280 x 3840 (360 tiles, 70 %) 43 / 50; 8192 x 320 x 2560 (320 tiles, 62 %) 19.6 / 23.1; 4096 x 1280 x 1280 (80 tiles, 31 %)
// 14.6 / 22.3.
bool big_tiles(tfmq_handle h, long M, int N) {
  const long nt = static_cast<long>(ceil_div(M, 256)) * ceil_div(N, 256), cu = h->cu_count;
  return nt >= cu && nt * 4 >= (nt + cu - 1) / cu * cu * 3;
}
// One launch that quantises on the way in (tiles of 32 x 32, eight ways along K) instead of two: for few rows, and while its workgroups are at most two
// per CU -- from there the 128 x 128 tiles' reuse counts for more than their idle CUs.  us, one launch against two: 154 x 1280 x 1280 6.2 / 14.5,
// 256 x 1280 x 1280 9.9 / 14.6, 256 x 5120 x 1280 31 / 42, 512 x 1280 x 1280 (2.5 per CU) 13.6 / 15.3, 512 x 5120 x 1280 45.6 / 44.5,
// 1024 x 1280 x 1280 21 / 16.5, 154 x 1280 x 10240 (6 per CU) 26.7 / 15.4.
// From 20 blocks on the slices below beat it earlier: 256 x 5120 x 1280 31 / 19.
bool one_launch(tfmq_handle h, long M, int N, int K) {
  return M <= 32 || static_cast<long>(ceil_div(M, 32)) * ceil_div(N, 32) <= (K > 19 * 128 ? 1L : 2L) * h->cu_count;
}
// slices of the K axis of a product whose tiles leave half the CUs idle: at least ten blocks each, a slice costs a write and a read of the result in fp32
// and all of them a launch.  us, whole against sliced: 1024 x 5120 x 1280 (80 tiles, 40 blocks) 41.6 / 28.7, 512 x 5120 x 1280 40.5 / 21.6; with three
// blocks a slice 1024 x 1280 x 1280 15.3 / 20.7, 512 x 768 x 1280 10.6 / 12.8.
int product_slices(tfmq_handle h, long M, int N, int K) {
  if (one_launch(h, M, N, K)) return 1;
  const long nt = static_cast<long>(ceil_div(M, 128)) * ceil_div(N, 128), Kb = (K + 127) / 128;
  const long n = std::min(h->cu_count / nt, Kb / 10);
  return static_cast<int>(n < 1 ? 1 : n);
}
template <int YDT>
int launch_sum(tfmq_handle h, const float* part, const float* bias, void* y, long n, int N, int nslice, hipStream_t st) {
  hipLaunchKernelGGL((k_sum_slices<YDT>), dim3(static_cast<unsigned>((n + 1023) / 1024)), dim3(256), 0, st, part, bias, static_cast<typename Elem<YDT>::type*>(y), n, N, nslice);
  TFMQ_LAUNCH_CHECK(h);
  return TFMQ_OK;
}
// part: room for p.nslice partial results, or null (one slice)
int launch_product(tfmq_handle h, const GemmF8P& p, int y_dtype, float* part, hipStream_t st) {
  if (p.nslice > 1) {
    GemmF8P q = p;
    q.y = part;
    q.bias = nullptr;
    const int rc = y_dtype == DT_F32 ? launch_128<DT_F32, false>(h, q, st) : launch_128<DT_PART, false>(h, q, st);
    if (rc != TFMQ_OK) return rc;
    const long n = p.M * p.N;
    if (y_dtype == DT_F32) return launch_sum<DT_F32>(h, part, p.bias, p.y, n, p.N, p.nslice, st);
    return y_dtype == DT_F16 ? launch_sum<DT_F16>(h, part, p.bias, p.y, n, p.N, p.nslice, st) : launch_sum<DT_BF16>(h, part, p.bias, p.y, n, p.N, p.nslice, st);
  }
  if (y_dtype == DT_F32) return launch_128<DT_F32, false>(h, p, st);
  if (big_tiles(h, p.M, p.N))
    return y_dtype == DT_F16 ? launch_gemm<256, 256, 128, 64, DT_F16, false, 2>(h, p, st) : launch_gemm<256, 256, 128, 64, DT_BF16, false, 2>(h, p, st);
  return y_dtype == DT_F16 ? launch_128<DT_F16, false>(h, p, st) : launch_128<DT_BF16, false>(h, p, st);
}
// slices of the token axis of a weight gradient [N][K]: its tiles alone leave CUs idle, every slice costs a write and a read of the result in fp32.
// 8192 x 640 x 640 (25 tiles): one slice 305 us, ten (one workgroup a CU) 22 with the other gradient, twice and three times as many slower again.
int grad_slices(tfmq_handle h, long M, int N, int K) {
  const long nt = static_cast<long>(ceil_div(N, 128)) * ceil_div(K, 128), Mb = (M + 127) / 128;
  const long n = h->cu_count / nt;
  return static_cast<int>(n < 1 ? 1 : n < Mb ? n : Mb);
}
size_t up256(size_t n) { return (n + 255) / 256 * 256; }

// the buffers of a call inside its workspace; sizes in bytes
struct Carve {
  char* p;
  size_t at = 0;
  template <typename T>
  T* take(size_t n) {
    T* r = reinterpret_cast<T*>(p + at);
    at += up256(n * sizeof(T));
    return r;
  }
};
struct LinWs {
  uint8_t* q = nullptr;
  float *s = nullptr, *part = nullptr;
  int slices;
  LinWs(Carve& c, tfmq_handle h, long M, int N, int K, bool quantise) {
    const long Kb = (K + 127) / 128;
    slices = product_slices(h, M, N, K);
    if (quantise && !one_launch(h, M, N, K)) {
      q = c.take<uint8_t>(static_cast<size_t>(M) * Kb * 128);
      s = c.take<float>(static_cast<size_t>(M) * Kb);
    }
    if (slices > 1) part = c.take<float>(static_cast<size_t>(slices) * M * N);
  }
};
struct BwdWs {
  uint8_t *gq = nullptr, *gc, *xc;
  float *gs = nullptr, *gcs, *xcs, *part = nullptr;
  int slices;
  BwdWs(Carve& c, tfmq_handle h, long M, int N, int K, bool gx, bool gw) {
    const long Mb = (M + 127) / 128, Nb = (N + 127) / 128;
    if (gx && !one_launch(h, M, K, N)) {
      gq = c.take<uint8_t>(static_cast<size_t>(M) * Nb * 128);
      gs = c.take<float>(static_cast<size_t>(M) * Nb);
    }
    if (!gw) return;
    gc = c.take<uint8_t>(static_cast<size_t>(N) * Mb * 128);
    gcs = c.take<float>(static_cast<size_t>(N) * Mb);
    xc = c.take<uint8_t>(static_cast<size_t>(K) * Mb * 128);
    xcs = c.take<float>(static_cast<size_t>(K) * Mb);
    slices = grad_slices(h, M, N, K);
    if (slices > 1) part = c.take<float>(static_cast<size_t>(slices) * N * K);
  }
};
bool shape_ok(long M, int N, int K) { return M > 0 && N > 0 && K > 0 && K <= (1 << 22) && N <= (1 << 22) && M <= (1L << 30); }
bool type_ok(int t) { return t >= 0 && t <= 2; }
bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

}  // namespace

extern "C" int tfmq_quantize_fp8(tfmq_handle h, const void* x, int dtype, long M, int K, long ld, int by_column, uint8_t* q, float* s, void* stream) {
  DeviceGuard guard(h);
  TFMQ_CHECK_ARG(h, h && x && q && s, "quantize_fp8: null pointer");
  TFMQ_CHECK_ARG(h, shape_ok(M, 1, K) && ld >= K && type_ok(dtype), "quantize_fp8: bad shape or type");
  TFMQ_CHECK_ARG(h, aligned16(q), "quantize_fp8: q must be 16-byte aligned");
  if (!by_column) return launch_quant_rows(h, x, dtype, M, K, ld, q, s, as_stream(stream));
  return launch_quant_cols(h, quant_tiles(x, dtype, M, K, ld, nullptr, nullptr, q, s), nullptr, as_stream(stream));
}

extern "C" int tfmq_pack_w_fp8(tfmq_handle h, const float* w, int N, int K, uint8_t* q, uint8_t* qt, float* s, void* stream) {
  DeviceGuard guard(h);
  TFMQ_CHECK_ARG(h, h && w && q && qt && s && shape_ok(1, N, K), "pack_w_fp8: bad argument");
  const long nb = static_cast<long>((N + 127) / 128) * ((K + 127) / 128);
  TFMQ_CHECK_ARG(h, nb < (1L << 31), "pack_w_fp8: too many blocks");
  hipLaunchKernelGGL(k_pack_w_f8, dim3(static_cast<unsigned>(nb)), dim3(256), 0, as_stream(stream), w, N, K, q, qt, s);
  TFMQ_LAUNCH_CHECK(h);
  return TFMQ_OK;
}

extern "C" size_t tfmq_linear_fp8_ws_bytes(tfmq_handle h, long M, int N, int K, int quantised) {
  if (!h || !shape_ok(M, N, K)) return 0;
  Carve c{nullptr};
  LinWs w(c, h, M, N, K, !quantised);
  return c.at;
}

extern "C" int tfmq_linear_fp8(tfmq_handle h, const void* x, int dtype, long M, int K, long ld, const uint8_t* xq, const float* xs, const uint8_t* w,
                               const float* ws, long ws_n, long ws_k, const float* bias, void* y, int y_dtype, int N, void* work, void* stream) {
  DeviceGuard guard(h);
  TFMQ_CHECK_ARG(h, h && (x || (xq && xs)) && w && ws && y, "linear_fp8: null pointer");
  TFMQ_CHECK_ARG(h, shape_ok(M, N, K) && type_ok(y_dtype) && (!x || (ld >= K && type_ok(dtype))), "linear_fp8: bad shape or type");
  TFMQ_CHECK_ARG(h, aligned16(w) && aligned16(xq) && aligned16(y) && aligned16(work), "linear_fp8: operands, output and workspace must be 16-byte aligned");
  hipStream_t st = as_stream(stream);
  const int Kb = (K + 127) / 128;
  if (x && one_launch(h, M, N, K)) return launch_small(h, SmallF8P{x, ld, static_cast<int>(M), K, w, ws, ws_n, ws_k, bias, y, N, Kb}, dtype, y_dtype, st);
  Carve c{static_cast<char*>(work)};
  const LinWs b(c, h, M, N, K, x != nullptr);
  TFMQ_CHECK_ARG(h, c.at == 0 || work, "linear_fp8: null workspace");
  if (x) {
    const int rc = launch_quant_rows(h, x, dtype, M, K, ld, b.q, b.s, st);
    if (rc != TFMQ_OK) return rc;
    xq = b.q;
    xs = b.s;
  }
  return launch_product(h, GemmF8P{xq, w, xs, ws, ws_n, ws_k, bias, y, M, N, Kb, 0, 0, b.slices}, y_dtype, b.part, st);
}

extern "C" size_t tfmq_linear_fp8_bwd_ws_bytes(tfmq_handle h, long M, int N, int K, int want_gx, int want_gw) {
  if (!h || !shape_ok(M, N, K)) return 0;
  Carve c{nullptr};
  BwdWs w(c, h, M, N, K, want_gx != 0, want_gw != 0);
  return c.at;
}

extern "C" int tfmq_linear_fp8_bwd(tfmq_handle h, const void* x, int x_dtype, long x_ld, const void* gy, int gy_dtype, long gy_ld, long M, int N, int K,
                                   const uint8_t* wt, const float* ws, void* gx, float* gw, void* work, void* stream) {
  DeviceGuard guard(h);
  TFMQ_CHECK_ARG(h, h && gy && (gx || gw) && (!gx || (wt && ws)) && (!gw || x), "linear_fp8_bwd: null pointer");
  TFMQ_CHECK_ARG(h, shape_ok(M, N, K) && gy_ld >= N && type_ok(gy_dtype) && (!gw || (x_ld >= K && type_ok(x_dtype))), "linear_fp8_bwd: bad shape or type");
  TFMQ_CHECK_ARG(h, aligned16(wt) && aligned16(gx) && aligned16(gw) && aligned16(work), "linear_fp8_bwd: operands, outputs and workspace must be 16-byte aligned");
  hipStream_t st = as_stream(stream);
  const int Nb = (N + 127) / 128, Kb = (K + 127) / 128;
  Carve c{static_cast<char*>(work)};
  const BwdWs b(c, h, M, N, K, gx != nullptr, gw != nullptr);
  TFMQ_CHECK_ARG(h, c.at == 0 || work, "linear_fp8_bwd: null workspace");
  int rc = TFMQ_OK;
  if (gw) {
    const QuantTileP qx = quant_tiles(x, x_dtype, M, K, x_ld, nullptr, nullptr, b.xc, b.xcs);
    rc = launch_quant_cols(h, quant_tiles(gy, gy_dtype, M, N, gy_ld, b.gq, b.gs, b.gc, b.gcs), &qx, st);
  } else if (b.gq) {
    rc = launch_quant_rows(h, gy, gy_dtype, M, N, gy_ld, b.gq, b.gs, st);
  }
  if (rc != TFMQ_OK) return rc;
  // the weight's blocks seen from its columns: scale (n block, k block) at ws[n block][k block]
  const GemmF8P px{b.gq, wt, b.gs, ws, 1, Kb, nullptr, gx, M, K, Nb, 0, 0, 1};
  const int Mb = static_cast<int>((M + 127) / 128);
  const GemmF8P pw{b.gc, b.xc, b.gcs, b.xcs, 0, 0, nullptr, gw ? (b.part ? b.part : gw) : nullptr, N, K, Mb, 0, 0, gw ? b.slices : 1};
  if (b.gq && gw && !big_tiles(h, M, K)) {
    if (gy_dtype == DT_F32) rc = launch_grads<DT_F32>(h, pw, px, st);
    else rc = gy_dtype == DT_F16 ? launch_grads<DT_F16>(h, pw, px, st) : launch_grads<DT_BF16>(h, pw, px, st);
  } else {
    if (gx)
      rc = b.gq ? launch_product(h, px, gy_dtype, nullptr, st)
                : launch_small(h, SmallF8P{gy, gy_ld, static_cast<int>(M), N, wt, ws, 1, Kb, nullptr, gx, K, Nb}, gy_dtype, gy_dtype, st);
    if (rc == TFMQ_OK && gw) rc = launch_128<DT_F32, true>(h, pw, st);
  }
  if (rc != TFMQ_OK) return rc;
  if (gw && b.part) rc = launch_sum<DT_F32>(h, b.part, nullptr, gw, static_cast<long>(N) * K, K, b.slices, st);
  return rc;
}
