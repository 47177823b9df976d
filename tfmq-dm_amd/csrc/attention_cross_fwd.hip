// Cross attention of Tq query tokens to Tk states of an encoder, per-item lengths, a key mask and shared key heads (CrossAttention.forward with
// `context` and `mask`, ldm/modules/attention.py:168-194; there a fully masked row attends to everything evenly, here it is zero):
//     o_i = sum_j p_ij v_j,  p_ij = exp(scale q_i k_j - lse_i),  lse_i = log sum_j exp(scale q_i k_j)   over the kept keys j.
//
// One pass over the keys with the running maximum and sum.  A wave owns 32 rows as the COLUMNS of S^T = K Q^T: a lane has one row, its maximum and
// sum are registers, and the probabilities are already the operand that O^T = V^T P^T wants.  K and V tiles of 64 keys are loaded into registers
// while the previous tile is multiplied, and stored to LDS row-major; V is read transposed by ds_read_b64_tr_b16.  Scores, statistics and sums are fp32;
// the probabilities are rounded to the operand type for the second product (the sum takes them unrounded).  They are taken against a reference below the
// maximum: fp16 ones lie up to 2^15, so that a long tail of small ones beside one large counts down to 2^-32 of it and not 2^-25.
#include "attention_cross.hpp"

using namespace xattn;

namespace {

// A score costs an FMA, an exponential, half a maximum, an addition and half a conversion beside 4 d / 64 matrix cycles per 64 of them: the VALU is the busier
// pipe.  2 x 4096 x 4096, 16 heads of 64, lengths drawn: 130 us (mean over six draws); VALU 52 % and MFMA 30 % busy, 2.0 waves a SIMD of the three that
// fit (the workgroups run in the items' order, whatever their lengths); four (128 registers) took 127 -> 127 - 130, two LDS buffers spill.  4 x 1000 x 1500, 16 heads on 4 of 128, lengths and mask drawn: 39 us.
template <typename T, int D>
__global__ __launch_bounds__(256, 2) void k_xattn_fwd(XattnP p) {
  constexpr int NKS = nks(D), NRT = nrt(D), KS = stride_rows(D), VS = stride_cols(D);
  using V8 = typename Vec8<T>::type;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  unsigned char* sK = smem;
  unsigned char* sV = smem + 64 * KS;
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6, j = lane & 31, hh = lane >> 5;
  int b, g, blk;
  pair_block(p.G, p.nrb * p.nsplit, b, g, blk);
  const int sp = blk % p.nsplit, rb = blk / p.nsplit;
  const int qlen = clamp_len(p.q_lens, b, p.Tq), klen = clamp_len(p.kv_lens, b, p.Tk);

  const long row = static_cast<long>(rb) * 128 + wid * 32 + j;
  const int hi = static_cast<int>(row / p.Tq), i = static_cast<int>(row - static_cast<long>(hi) * p.Tq);
  const bool ok = row < p.R && i < qlen;
  const int head = g * p.rep + hi;
  V8 qf[NKS];
  {
    const T* qrow = static_cast<const T*>(p.q.p) + b * p.q.bs + i * p.q.ts + static_cast<long>(head) * p.d;
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks) {
      const int c = ks * 16 + hh * 8;
      uint4 w = make_uint4(0, 0, 0, 0);
      if (ok && c < p.d) w = *reinterpret_cast<const uint4*>(qrow + c);
      qf[ks] = __builtin_bit_cast(V8, w);
    }
  }
  const T* kb = static_cast<const T*>(p.k.p) + b * p.k.bs + static_cast<long>(g) * p.d;
  const T* vb = static_cast<const T*>(p.v.p) + b * p.v.bs + static_cast<long>(g) * p.d;
  const uint8_t* mb = p.mask ? p.mask + b * p.mask_bs : nullptr;
  auto keep_bit = [&](int t) { const int key = t * 64 + lane; return key < klen && (!mb || mb[key] != 0); };

  const int nt = (klen + 63) / 64, per = (nt + p.nsplit - 1) / p.nsplit;
  const int t0 = sp * per, t1 = min(nt, t0 + per);
  KeyTile<T, D, 64, KS> tk;
  KeyTile<T, D, 64, VS> tv;
  unsigned long long cur = 0, nxt = 0;
  auto fetch = [&](int t) {
    tk.load(kb, p.k.ts, t * 64, p.Tk, p.d);
    tv.load(vb, p.v.ts, t * 64, p.Tk, p.d);
  };
  const float c2 = p.scale * LOG2E;
  constexpr float BELOW = std::is_same<T, _Float16>::value ? 7.0f : 0.0f;          // (with the late rescaling's 2^8 below fp16's largest)
  float m = -INFINITY, l = 0.0f;          // the reference, 2^BELOW under the maximum, and the sum against it
  v16f o[NRT];
#pragma unroll
  for (int t = 0; t < NRT; ++t) o[t] = zero16();

  if (t0 < t1) {
    cur = __ballot(keep_bit(t0));
    fetch(t0);
  }
  for (int t = t0; t < t1; ++t) {
    __syncthreads();                   // every wave is through with the previous tile
    tk.store(sK, cur, ~0ull, p.d);
    tv.store(sV, cur, ~0ull, p.d);
    __syncthreads();
    nxt = 0;
    if (t + 1 < t1) {
      nxt = __ballot(keep_bit(t + 1));
      fetch(t + 1);
    }
    if (cur != 0) {
      v16f s[2];
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        s[kt] = zero16();
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks) s[kt] = mfma16(frag_rows<T>(sK, KS, kt * 32 + j, ks, hh), qf[ks], s[kt]);
      }
      if (cur != ~0ull) drop_keys(s, cur, hh);
      float mx = -INFINITY;
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[kt][r]);
      mx = fmaxf(mx, __shfl_xor(mx, 32, 64)) * c2;          // (scale > 0)
      mx -= BELOW;
      // the sums move to a new maximum only where one has risen by more than 2^8 since (or there was none): probabilities up to 256 times those of the
      // maximum are as exact as those, and past the first tile this is rare
      if (__any(mx > m + 8.0f)) {
        const float mn = fmaxf(m, mx), alpha = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.0f : mn));
        m = mn;
        l *= alpha;
#pragma unroll
        for (int t2 = 0; t2 < NRT; ++t2)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[t2][r] *= alpha;
      }
      const float mu = m == -INFINITY ? 0.0f : m;
      float rs[2] = {0.0f, 0.0f};
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          s[kt][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kt][r], c2, -mu));
          rs[r & 1] += s[kt][r];
        }
      l += rs[0] + rs[1];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const V8 pf = frag_regs<T>(s[u >> 1], u & 1);
#pragma unroll
        for (int t2 = 0; t2 < NRT; ++t2) o[t2] = mfma16(frag_cols<T>(sV, VS, u * 16, t2, lane), pf, o[t2]);
      }
    }
    cur = nxt;
  }
  l += __shfl_xor(l, 32, 64);
  if (row >= p.R) return;
  zero_unless(ok, o);
  const long orow = (static_cast<long>(b) * p.H + head) * p.Tq + i;          // row of [B][H][Tq]
  if (p.nsplit > 1) {
    // slice sp's sums against its own maximum: [slice][row][d] and {m, l} behind them
    float* po = p.part + (static_cast<long>(sp) * p.B * p.H * p.Tq + orow) * p.d;
#pragma unroll
    for (int t = 0; t < NRT; ++t) store16_f32(po, t * 32, hh, p.d, o[t], 1.0f);
    if (hh == 0) {
      float* ml = p.part + static_cast<long>(p.nsplit) * p.B * p.H * p.Tq * p.d + (static_cast<long>(sp) * p.B * p.H * p.Tq + orow) * 2;
      ml[0] = ok ? m : -INFINITY;
      ml[1] = ok ? l : 0.0f;
    }
    return;
  }
  const float inv = ok && l != 0.0f ? 1.0f / l : 0.0f;
  T* yrow = static_cast<T*>(p.y) + (static_cast<long>(b) * p.Tq + i) * p.H * p.d + static_cast<long>(head) * p.d;
#pragma unroll
  for (int t = 0; t < NRT; ++t) store16<T>(yrow, t * 32, hh, p.d, o[t], inv);
  if (p.lse && hh == 0) p.lse[orow] = ok && l != 0.0f ? (m + __builtin_amdgcn_logf(l)) * LN2 : -INFINITY;
}

// ---- up to 128 states (a text encoder's): K and V of one (item, key head) stay in LDS, the waves walk over rows on their own, without barriers, the next
// rows' queries under way.  All keys are in the accumulators at once: one maximum, no running rescale.  Bound by HBM (4 bytes of q and o per 2 x 77 products
// and exponentials): the tiled kernel above needed 156 us for 128 x 1024 x 77, 8 heads of 80; 8 x 4096 x 77, 8 heads of 40: 16.5 us (2.5 TB/s).
// waves per SIMD that the registers allow without spilling (the walk waits for memory: 4 against 2 took the 128 x 1024 x 77 call, 8 heads of 80, from 114 to
// 112 us; reading and writing rows through buffer descriptors then to 105, 3.4 TB/s)
constexpr int short_waves(int D, int NKT) { return D <= 64 || (D <= 96 && NKT <= 3) ? 4 : D <= 128 || NKT <= 2 ? 3 : 2; }

template <typename T, int D, int NKT>
__global__ __launch_bounds__(256, short_waves(D, NKT)) void k_xattn_short(XattnP p) {
  constexpr int NKS = nks(D), NRT = nrt(D), KS = stride_rows(D), VS = stride_cols(D), NK = NKT * 32;
  using V8 = typename Vec8<T>::type;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  unsigned char* sK = smem;
  unsigned char* sV = smem + NK * KS;
  float* sB = reinterpret_cast<float*>(smem + NK * (KS + VS));
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6, j = lane & 31, hh = lane >> 5;
  const int id = xcd_tile_id();
  const int rb = id % p.nrb, bg = id / p.nrb, b = bg / p.G, g = bg - b * p.G;
  const int qlen = clamp_len(p.q_lens, b, p.Tq), klen = clamp_len(p.kv_lens, b, p.Tk);
  const long hc = static_cast<long>(g) * p.rep * p.d, C = static_cast<long>(p.H) * p.d;
  const Rsrc rq = buffer_of(static_cast<const T*>(p.q.p) + b * p.q.bs + hc, ((p.Tq - 1) * p.q.ts + static_cast<long>(p.rep) * p.d) * 2);
  const Rsrc ry = buffer_of(static_cast<T*>(p.y) + b * p.Tq * C + hc, (p.Tq * C - hc) * 2);
  const Rsrc rl = buffer_of(p.lse ? p.lse + (static_cast<long>(b) * p.H + g * p.rep) * p.Tq : nullptr, p.lse ? p.R * 4 : 0);
  const unsigned qts = static_cast<unsigned>(p.q.ts) * 2, yts = static_cast<unsigned>(C) * 2, hs = static_cast<unsigned>(p.d) * 2;

  const long r_end = min(p.R, (static_cast<long>(rb) + 1) * p.rows_per);
  RowWalk w(static_cast<long>(rb) * p.rows_per + wid * 32 + j, p.Tq);
  V8 qf[NKS];
  auto load_q = [&]() {
    const unsigned off = w.row < r_end && w.i < qlen ? w.i * qts + w.hi * hs : NOWHERE;
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks) {
      const int c = ks * 16 + hh * 8;
      qf[ks] = load8<V8>(rq, off != NOWHERE && c < p.d ? off + c * 2 : NOWHERE);
    }
  };
  load_q();
  const bool any = stage_short<T, D, NKT, KS, VS, false>(p, b, g, klen, sK, sV, sB);          // (an item that keeps nothing: zeros, whatever its rows hold)
  const float c2 = p.scale * LOG2E;
  while (w.row - j < r_end) {
    const bool in = w.row < r_end, ok = any && in && w.i < qlen;
    const unsigned yoff = w.i * yts + w.hi * hs, loff = in && hh == 0 ? static_cast<unsigned>(w.row) * 4 : NOWHERE;
    v16f s[NKT];
#pragma unroll
    for (int kt = 0; kt < NKT; ++kt) {
      s[kt] = start_scores(sB + kt * 32, hh);
#pragma unroll
      for (int ks = 0; ks < NKS; ++ks) s[kt] = mfma16(frag_rows<T>(sK, KS, kt * 32 + j, ks, hh), qf[ks], s[kt]);
    }
    hold_order();
    w.step();
    load_q();
    float mx = -INFINITY;
#pragma unroll
    for (int kt = 0; kt < NKT; ++kt)
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[kt][r]);
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64)) * c2;
    const float mu = mx == -INFINITY ? 0.0f : mx;
    float rs[2] = {0.0f, 0.0f};
#pragma unroll
    for (int kt = 0; kt < NKT; ++kt)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[kt][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kt][r], c2, -mu));
        rs[r & 1] += s[kt][r];
      }
    float l = rs[0] + rs[1];
    l += __shfl_xor(l, 32, 64);
    V8 pf[2 * NKT];
#pragma unroll
    for (int u = 0; u < 2 * NKT; ++u) pf[u] = frag_regs<T>(s[u >> 1], u & 1);
    hold_order();                        // (the scores' registers are free from here on)
    v16f o[NRT];
#pragma unroll
    for (int t = 0; t < NRT; ++t) o[t] = zero16();
#pragma unroll
    for (int u = 0; u < 2 * NKT; ++u)
#pragma unroll
      for (int t = 0; t < NRT; ++t) o[t] = mfma16(frag_cols<T>(sV, VS, u * 16, t, lane), pf[u], o[t]);
    zero_unless(ok, o);
    const float inv = ok && l != 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
    for (int t = 0; t < NRT; ++t) store16<T>(ry, yoff, in, t * 32, hh, p.d, o[t], inv);
    const float lse = ok && l != 0.0f ? (mx + __builtin_amdgcn_logf(l)) * LN2 : -INFINITY;
    __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(lse), rl, static_cast<int>(loff), 0, 0);
  }
}

// joins the slices of a row: a wave a row, 16 lanes of 8 channels for each of four slices at a time (a longer walk per lane waits for memory at every
// step: 512 slices of one row took 250 us with one lane per 8 channels).  The four partial sums meet in a fixed order.
template <typename T>
__global__ __launch_bounds__(256) void k_xattn_join(XattnP p) {
  const long rows = static_cast<long>(p.B) * p.H * p.Tq;
  const long r = static_cast<long>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, c16 = lane & 15, s4 = lane >> 4;
  if (r >= rows) return;
  const float* ml = p.part + static_cast<long>(p.nsplit) * rows * p.d;
  float M = -INFINITY;
  for (int s = lane; s < p.nsplit; s += 64) M = fmaxf(M, ml[(s * rows + r) * 2]);
  M = wave_reduce_max(M);
  const float mu = M == -INFINITY ? 0.0f : M;
  float l = 0.0f;
  for (int s = lane; s < p.nsplit; s += 64) l = __builtin_fmaf(ml[(s * rows + r) * 2 + 1], __builtin_amdgcn_exp2f(ml[(s * rows + r) * 2] - mu), l);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) l += __shfl_xor(l, o, 64);
  const float inv = l != 0.0f ? 1.0f / l : 0.0f;
  const long bh = r / p.Tq;
  const int i = static_cast<int>(r - bh * p.Tq), b = static_cast<int>(bh / p.H), head = static_cast<int>(bh - static_cast<long>(b) * p.H);
  T* y = static_cast<T*>(p.y) + (static_cast<long>(b) * p.Tq + i) * p.H * p.d + static_cast<long>(head) * p.d;
  for (int c0 = 0; c0 < p.d; c0 += 128) {
    const int c = min(c0 + c16 * 8, p.d - 8);          // (lanes past the head read its last channels)
    float a[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) a[e] = 0.0f;
#pragma unroll 4
    for (int s = s4; s < p.nsplit; s += 4) {
      const float w = __builtin_amdgcn_exp2f(ml[(s * rows + r) * 2] - mu);
      const float4* po = reinterpret_cast<const float4*>(p.part + (s * rows + r) * p.d + c);
      const float4 x = po[0], z = po[1];
      a[0] = __builtin_fmaf(x.x, w, a[0]); a[1] = __builtin_fmaf(x.y, w, a[1]); a[2] = __builtin_fmaf(x.z, w, a[2]); a[3] = __builtin_fmaf(x.w, w, a[3]);
      a[4] = __builtin_fmaf(z.x, w, a[4]); a[5] = __builtin_fmaf(z.y, w, a[5]); a[6] = __builtin_fmaf(z.z, w, a[6]); a[7] = __builtin_fmaf(z.w, w, a[7]);
    }
    typename Vec8<T>::type w8;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      a[e] += __shfl_xor(a[e], 16, 64);
      a[e] += __shfl_xor(a[e], 32, 64);
      w8[e] = static_cast<T>(a[e] * inv);
    }
    if (s4 == 0 && c0 + c16 * 8 < p.d) *reinterpret_cast<typename Vec8<T>::type*>(y + c) = w8;
  }
  if (p.lse && lane == 0) p.lse[r] = l != 0.0f ? (M + __builtin_amdgcn_logf(l)) * LN2 : -INFINITY;
}

template <typename T, int D, int NKT>
int launch_short(tfmq_handle h, XattnP p, hipStream_t st) {
  auto kern = &k_xattn_short<T, D, NKT>;
  constexpr int smem = NKT * 32 * (stride_rows(D) + stride_cols(D) + 4);
  static LdsRoom room_kern;
  TFMQ_HIP(h, room_kern.ask(h, reinterpret_cast<const void*>(kern), smem));
  const long pairs = static_cast<long>(p.B) * p.G;
  p.rows_per = short_rows(h, pairs, p.R, short_waves(D, NKT));
  p.nrb = ceil_div(p.R, p.rows_per);
  TFMQ_CHECK_ARG(h, pairs * p.nrb < MAX_BLOCKS, "xattn_fwd: too many workgroups");
  hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>(pairs * p.nrb)), dim3(256), smem, st, p);
  TFMQ_LAUNCH_CHECK(h);
  return TFMQ_OK;
}

template <typename T>
int launch_fwd(tfmq_handle h, XattnP p, hipStream_t st) {
  return for_head_dim(p.d, [&](auto dc) {
    constexpr int D = decltype(dc)::value;
    const int nkt = (p.Tk + 31) / 32;
    if (p.nsplit == 1 && nkt >= 1 && nkt <= 4 && rows_fit(p)) {          // (no states at all: the tiled kernel reads none)
      if (nkt == 1) return launch_short<T, D, 1>(h, p, st);
      if (nkt == 2) return launch_short<T, D, 2>(h, p, st);
      if (nkt == 3) return launch_short<T, D, 3>(h, p, st);
      return launch_short<T, D, 4>(h, p, st);
    }
    auto kern = &k_xattn_fwd<T, D>;
    constexpr int smem = 64 * (stride_rows(D) + stride_cols(D));
    static LdsRoom room_kern;
    TFMQ_HIP(h, room_kern.ask(h, reinterpret_cast<const void*>(kern), smem));
    p.nrb = ceil_div(p.R, 128);
    const long nb = static_cast<long>(p.B) * p.G * p.nrb * p.nsplit;
    TFMQ_CHECK_ARG(h, nb < MAX_BLOCKS, "xattn_fwd: too many workgroups");
    hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>(nb)), dim3(256), smem, st, p);
    TFMQ_LAUNCH_CHECK(h);
    if (p.nsplit > 1) {
      hipLaunchKernelGGL((k_xattn_join<T>), dim3(static_cast<unsigned>((static_cast<long>(p.B) * p.H * p.Tq + 3) / 4)), dim3(256), 0, st, p);
      TFMQ_LAUNCH_CHECK(h);
    }
    return TFMQ_OK;
  });
}

}  // namespace

// Slices of the key axis of a forward call, where the rows alone leave CUs idle.  Few rows (at most a wave's 32 of a workgroup's 128: single tokens with
// shared key heads): four workgroups a CU, so that items of different lengths even out; us at 16 x 1 x 4095, 32 heads on 8 of 128, for 1 / 4 / 6 / 8 / 16
// slices: lengths drawn 92 / 39 / 32 / 31 / 33, all full 91 / 47 / 55 / 50 / 52.  Full tiles write and join as much as they read: two a CU and none from one
// a CU on; 2 x 512 x 4096, 16 heads of 64 (128 workgroups), 1 / 2 / 4 / 8 slices 62 / 45 / 34 / 37; 2 x 1000 x 1500, 16 heads on 4 of 128 (256 workgroups)
// 1 / 2 slices 16 / 35.  A slice has four tiles of 64 keys (1 x 64 x 4096, 16 heads: 16 / 32 slices 13.9 / 16.2; 65536 keys of one head: 256 / 512 slices
// 36 / 57), two where that leaves fewer than four slices (8 x 16 x 500, 8 heads of 40: 2 / 4 slices 11.6 / 9.3).
extern "C" int tfmq_xattn_splits(tfmq_handle h, int B, int H, int G, int Tq, int Tk) {
  if (!h || B <= 0 || H <= 0 || G <= 0 || H % G || Tq <= 0 || Tk <= 128) return 1;
  const long R = static_cast<long>(H / G) * Tq, blocks = static_cast<long>(B) * G * ceil_div(R, 128);
  if (R > 32 && blocks >= h->cu_count) return 1;
  const long n = (R > 32 ? 2L : 4L) * h->cu_count / blocks, most = std::max<long>(ceil_div(Tk, 256), std::min<long>(4, ceil_div(Tk, 128)));
  return static_cast<int>(n < 1 ? 1 : n < most ? n : most);
}

extern "C" int tfmq_xattn_fwd(tfmq_handle h, const tfmq_xattn_desc* a, void* stream) {
  TFMQ_CHECK_ARG(h, h && a, "xattn_fwd: null pointer");
  DeviceGuard guard(h);
  TFMQ_CHECK_ARG(h, a->B > 0 && a->H > 0 && a->G > 0 && a->H % a->G == 0 && a->Tq > 0 && a->Tk >= 0 && a->d > 0 && a->d <= 160 && a->d % 8 == 0,
                 "xattn_fwd: bad shape");
  TFMQ_CHECK_ARG(h, a->dtype == 1 || a->dtype == 2, "xattn_fwd: fp16 or bf16");
  TFMQ_CHECK_ARG(h, a->q && (a->Tk == 0 || (a->k && a->v)) && a->o, "xattn_fwd: null tensor");
  TFMQ_CHECK_ARG(h, a->nsplit >= 1 && (a->nsplit == 1 || a->ws), "xattn_fwd: slices need a workspace");
  TFMQ_CHECK_ARG(h, a->k_ts < (1 << 23) && a->v_ts < (1 << 23) && a->k_ts >= 0 && a->v_ts >= 0, "xattn_fwd: token strides of k and v must lie in [0, 2^23)");
  XattnP p{};
  p.q = {a->q, a->q_bs, a->q_ts};
  p.k = {a->k, a->k_bs, a->k_ts};
  p.v = {a->v, a->v_bs, a->v_ts};
  p.y = a->o;
  p.lse = a->lse;
  p.part = a->ws;
  p.q_lens = a->q_lens;
  p.kv_lens = a->kv_lens;
  p.mask = a->mask;
  p.mask_bs = a->mask_bs;
  p.B = a->B; p.H = a->H; p.G = a->G; p.rep = a->H / a->G; p.Tq = a->Tq; p.Tk = a->Tk; p.d = a->d;
  p.R = static_cast<long>(p.rep) * p.Tq;
  p.scale = a->scale;
  p.nsplit = a->nsplit;
  return a->dtype == 1 ? launch_fwd<_Float16>(h, p, as_stream(stream)) : launch_fwd<__bf16>(h, p, as_stream(stream));
}
