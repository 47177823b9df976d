// Gradients of the cross attention (attention_cross_fwd.hip): with p_ij = exp(scale q_i k_j - lse_i), dp_ij = go_i v_j and
// D_i = sum_j p_ij dp_ij = sum_c o_ic go_ic,
//     ds_ij = p_ij (dp_ij - D_i),   dq_i = scale sum_j ds_ij k_j,   dk_j = scale sum_i ds_ij q_i,   dv_j = sum_i p_ij go_i.
//
// Two kernels recompute p from the saved lse, each with its sums in registers and no atomics: k_xattn_dq walks the keys of 128 rows (a lane owns a row,
// as in the forward), k_xattn_dkv walks the rows of 128 keys (a lane owns a key; shared key heads sum over their query heads because those are
// further rows).  Seven products (eight over more than 128 states) instead of the five of a fused pass, for results that are the same bits every
// time.  Where few key blocks face many rows -- 77 states under 4096 tokens -- the rows are cut into slices whose fp32 sums are added in order.
//
// fp16 range: ds has the size of p go v, which may lie far below fp16's normal numbers (a loss averaged over many tokens, small states) or above its largest
// (states of thousands).  The ds operand is therefore carried with a power of two by the largest |dp - D| itself -- of the row in dq, of the slice's rows in
// dkv -- so that it stays below 2^15 and what underflows below 2^-33 of that largest; and p in dv with 2^12.  All are exact and taken out of the fp32
// sums.  bf16 has the range.
#include "attention_cross.hpp"

using namespace xattn;

namespace {

template <typename T> constexpr bool is_f16() { return std::is_same<T, _Float16>::value; }

// the power of two that brings a magnitude to 1 ... 2 (2^0 for zero; within 2^+-72 for every input: products of fp16 values lie in that)
__device__ __forceinline__ int inv_exponent(float a) {
  const int e = static_cast<int>((__float_as_uint(a) >> 23) & 255);
  return e == 0 ? 0 : 127 - min(max(e, 55), 199);
}
constexpr int DS_TOP = 13;          // where the operand's largest |dp - D| is put when it is known beforehand: 2^13 ... 2^14

// Four products and the exponentials per score; operand reads run ahead of the products (dealt between them; at d = 160 the registers hold the rows or the
// transposed tiles).  One wave a SIMD from d = 72 on (d = 128: 409 registers; at two waves 80 and 96 spill 144 - 220 bytes).  4 x 1000 x 1500, 16 heads on 4 of
// 128, lengths and mask drawn: 75 us, MFMA 16 % busy, 0.66 waves a SIMD on average.
//
// D comes from the row's own p dp, as over few states (below), without a walk of its own: the walk starts from the D0 of the rounded o, sums
// delta = sum_j ds_j = D - D0 in fp32 and B = sum_j p_j k_j beside sum_j ds_j k_j, and dq loses delta B at its end.  (D0's rounding is small against
// D but not against p (dp - D) where few states hold a row's weight: two kept of 1500, bf16, dq 2.5 times its roundings' bound.)  The fourth product took this
// kernel from 67 to 75 us; the whole backward pass of 4 x 1000 x 1500 and 16 heads on 4, bf16, from 113 to 121 at d = 40, 198 to 227 at 80 (two waves a SIMD
// before), 273 to 291 at 128 and 380 to 417 at 160.
template <typename T, int D>
__global__ __launch_bounds__(256, D <= 64 ? 2 : 1) void k_xattn_dq(XattnP p) {
  constexpr float PSHIFT = is_f16<T>() ? 12.0f : 0.0f, UNSHIFT = is_f16<T>() ? 1.0f / 4096.0f : 1.0f;          // p carries 2^PSHIFT
  constexpr int NKS = nks(D), NRT = nrt(D), KS = stride_both(D), VS = stride_rows(D);
  using V8 = typename Vec8<T>::type;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  unsigned char* sK = smem;
  unsigned char* sV = smem + 64 * KS;
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6, j = lane & 31, hh = lane >> 5;
  int b, g, rb;
  pair_block(p.G, p.nrb, b, g, rb);
  const int qlen = clamp_len(p.q_lens, b, p.Tq), klen = clamp_len(p.kv_lens, b, p.Tk);
  const long row = static_cast<long>(rb) * 128 + wid * 32 + j;
  const int hi = static_cast<int>(row / p.Tq), i = static_cast<int>(row - static_cast<long>(hi) * p.Tq);
  const long brow = (static_cast<long>(b) * p.H + g * p.rep) * p.Tq + row;          // row of [B][H][Tq]
  const bool in = row < p.R, ok = in && i < qlen;
  const int head = g * p.rep + hi;

  V8 qf[NKS], gf[NKS];
  float dl = 0.0f;
  {
    const long hc = static_cast<long>(head) * p.d;
    const T* qrow = static_cast<const T*>(p.q.p) + b * p.q.bs + i * p.q.ts + hc;
    const T* grow = static_cast<const T*>(p.go.p) + b * p.go.bs + i * p.go.ts + hc;
    const T* orow = static_cast<const T*>(p.o.p) + b * p.o.bs + i * p.o.ts + hc;
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks) {
      const int c = ks * 16 + hh * 8;
      uint4 a = make_uint4(0, 0, 0, 0), w = a, z = a;
      if (ok && c < p.d) {
        a = *reinterpret_cast<const uint4*>(qrow + c);
        w = *reinterpret_cast<const uint4*>(grow + c);
        z = *reinterpret_cast<const uint4*>(orow + c);
      }
      qf[ks] = __builtin_bit_cast(V8, a);
      gf[ks] = __builtin_bit_cast(V8, w);
      const V8 of = __builtin_bit_cast(V8, z);
#pragma unroll
      for (int e = 0; e < 8; ++e) dl = __builtin_fmaf(static_cast<float>(of[e]), static_cast<float>(gf[ks][e]), dl);
    }
  }
  dl += __shfl_xor(dl, 32, 64);
  float lse2 = INFINITY;
  if (ok) {
    const float v = p.lse_in[brow];
    lse2 = v == -INFINITY ? INFINITY : v * LOG2E;
  }
  lse2 -= PSHIFT;
  // fp16: the operand's power of two, by the largest |dp - D0| so far: 2^8 ... 2^9 (with p's) in the first tile that has one; a larger one moves it down
  // only past 2^15 (and the sums with it: exact, and rare)
  float f = 1.0f, dlf = dl, top = 0.0f, lim = 0.0f, dsum[2] = {0.0f, 0.0f};

  const T* kb = static_cast<const T*>(p.k.p) + b * p.k.bs + static_cast<long>(g) * p.d;
  const T* vb = static_cast<const T*>(p.v.p) + b * p.v.bs + static_cast<long>(g) * p.d;
  const uint8_t* mb = p.mask ? p.mask + b * p.mask_bs : nullptr;
  auto keep_bit = [&](int t) { const int key = t * 64 + lane; return key < klen && (!mb || mb[key] != 0); };
  const int nt = (klen + 63) / 64;
  KeyTile<T, D, 64, KS> tk;
  KeyTile<T, D, 64, VS> tv;
  unsigned long long cur = 0, nxt = 0;
  auto fetch = [&](int t) {
    tk.load(kb, p.k.ts, t * 64, p.Tk, p.d);
    tv.load(vb, p.v.ts, t * 64, p.Tk, p.d);
  };
  const float c2 = p.scale * LOG2E;
  v16f acc[NRT], pk[NRT];
#pragma unroll
  for (int t = 0; t < NRT; ++t) acc[t] = zero16(), pk[t] = zero16();
  if (nt > 0) {
    cur = __ballot(keep_bit(0));
    fetch(0);
  }
  for (int t = 0; t < nt; ++t) {
    __syncthreads();
    tk.store(sK, cur, ~0ull, p.d);
    tv.store(sV, cur, ~0ull, p.d);
    __syncthreads();
    nxt = 0;
    if (t + 1 < nt) {
      nxt = __ballot(keep_bit(t + 1));
      fetch(t + 1);
    }
    if (cur != 0) {
      // (operand reads run ahead of the products, as in k_xattn_dkv)
      V8 kr[NKS], vr[NKS];
      auto read_rows = [&](int kt) {
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks) {
          kr[ks] = frag_rows<T>(sK, KS, kt * 32 + j, ks, hh);
          vr[ks] = frag_rows<T>(sV, VS, kt * 32 + j, ks, hh);
        }
      };
      read_rows(0);
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        if (kt == 1 && D > 128) read_rows(1);          // (at 160 the registers hold the rows or the transposed tiles, not both)
        hold_order();
        v16f s = zero16(), dp = zero16();
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks) {
          s = mfma16(kr[ks], qf[ks], s);
          dp = mfma16(vr[ks], gf[ks], dp);
        }
        V8 ct[2][NRT];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int t2 = 0; t2 < NRT; ++t2) ct[u][t2] = frag_cols<T>(sK, KS, kt * 32 + u * 16, t2, lane);
        deal_reads<2 * NKS, 1>();
        hold_order();
        const unsigned bits = static_cast<unsigned>(cur >> (32 * kt)) >> (4 * hh);
        if (cur != ~0ull) {
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const bool kept = (bits >> crow(r, 0)) & 1;
            s[r] = kept ? s[r] : -INFINITY;
            if (is_f16<T>()) dp[r] = kept ? dp[r] : dl;
          }
        }
        if constexpr (is_f16<T>()) {
          float mx = 0.0f;
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            dp[r] = __builtin_fmaf(dp[r], f, -dlf);
            mx = fmaxf(mx, fabsf(dp[r]));
          }
          if (__any(mx > lim)) {
            const float row = fmaxf(mx, __shfl_xor(mx, 32, 64));
            const float ratio = row > lim ? __builtin_amdgcn_exp2f(static_cast<float>(inv_exponent(row) + 8) - PSHIFT) : 1.0f;
            lim = row > lim ? 32768.0f * UNSHIFT : lim;
            f *= ratio, dlf *= ratio, top *= ratio, mx *= ratio, dsum[0] *= ratio, dsum[1] *= ratio;
#pragma unroll
            for (int r = 0; r < 16; ++r) dp[r] *= ratio;
#pragma unroll
            for (int t2 = 0; t2 < NRT; ++t2)
#pragma unroll
              for (int r = 0; r < 16; ++r) acc[t2][r] *= ratio;
          }
          top = fmaxf(top, mx);
        } else {
#pragma unroll
          for (int r = 0; r < 16; ++r) dp[r] -= dl;
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          s[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], c2, -lse2));
          dp[r] *= s[r];
          dsum[r & 1] += dp[r];
        }
        V8 pf[2], df[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) pf[u] = frag_regs<T>(s, u), df[u] = frag_regs<T>(dp, u);
        hold_order();
        if (kt == 0 && D <= 128) read_rows(1);
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int t2 = 0; t2 < NRT; ++t2) {
            acc[t2] = mfma16(ct[u][t2], df[u], acc[t2]);
            pk[t2] = mfma16(ct[u][t2], pf[u], pk[t2]);
          }
        if (kt == 0 && D <= 128) deal_reads<4 * NRT, 1>();
      }
    }
    cur = nxt;
  }
  top = fmaxf(top, __shfl_xor(top, 32, 64));
  float dd = dsum[0] + dsum[1];
  dd = (dd + __shfl_xor(dd, 32, 64)) * UNSHIFT;
  if (!in) return;
#pragma unroll
  for (int t = 0; t < NRT; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[t][r] = __builtin_fmaf(-dd, pk[t][r], acc[t][r]);
  zero_unless(ok, acc);
  if (hh == 0) {
    p.delta[brow] = dl + dd / f;
    if (is_f16<T>()) p.delta[static_cast<long>(p.B) * p.H * p.Tq + brow] = ok ? (top + fabsf(dd)) / f : 0.0f;          // (k_xattn_dkv's range)
  }
  T* yrow = static_cast<T*>(p.y) + (static_cast<long>(b) * p.Tq + i) * p.H * p.d + static_cast<long>(head) * p.d;
#pragma unroll
  for (int t = 0; t < NRT; ++t) store16<T>(yrow, t * 32, hh, p.d, acc[t], p.scale * UNSHIFT / f);
}

// ---- dq against up to 128 states: K and V stay in LDS, the waves walk over rows without barriers (k_xattn_short's form).  A row's probabilities and dp all
// stay in registers and D is their own mean of dp.  From o, which the forward has rounded, D is off by that rounding, and few states leave
// ds = p (dp - D) small against D: bf16 gradients of q and k at 18 states, of which a mask and lengths kept about three, were 1.9 times as far from the exact
// ones as from one rounding, now 1.4 (the ds operand's and the result's).  8 x 4096 x 77, 8 heads of 40: 26 us for 63 MB of q, go and dq, VALU 33 % busy, 1.5
// waves a SIMD.
constexpr int dq_short_waves(int D, int NKT) { return D <= 64 && NKT <= 2 ? 4 : NKT <= (D <= 32 ? 4 : D <= 64 ? 3 : D <= 96 ? 2 : 0) ? 3 : 2; }
template <typename T, int D, int NKT>
__global__ __launch_bounds__(256, dq_short_waves(D, NKT)) void k_xattn_dq_short(XattnP p) {
  constexpr int NKS = nks(D), NRT = nrt(D), KS = stride_both(D), VS = stride_rows(D), NK = NKT * 32;
  using V8 = typename Vec8<T>::type;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  unsigned char* sK = smem;
  unsigned char* sV = smem + NK * KS;
  float* sB = reinterpret_cast<float*>(smem + NK * (KS + VS));
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6, j = lane & 31, hh = lane >> 5;
  const int id = xcd_tile_id();
  const int rb = id % p.nrb, bg = id / p.nrb, b = bg / p.G, g = bg - b * p.G;
  const int qlen = clamp_len(p.q_lens, b, p.Tq), klen = clamp_len(p.kv_lens, b, p.Tk);
  const long hc = static_cast<long>(g) * p.rep * p.d, C = static_cast<long>(p.H) * p.d, rd = static_cast<long>(p.rep) * p.d;
  const long brow0 = (static_cast<long>(b) * p.H + g * p.rep) * p.Tq, rows = static_cast<long>(p.B) * p.H * p.Tq;
  const Rsrc rq = buffer_of(static_cast<const T*>(p.q.p) + b * p.q.bs + hc, ((p.Tq - 1) * p.q.ts + rd) * 2);
  const Rsrc rg = buffer_of(static_cast<const T*>(p.go.p) + b * p.go.bs + hc, ((p.Tq - 1) * p.go.ts + rd) * 2);
  const Rsrc ry = buffer_of(static_cast<T*>(p.y) + b * p.Tq * C + hc, (p.Tq * C - hc) * 2);
  const Rsrc rl = buffer_of(p.lse_in + brow0, p.R * 4), rdl = buffer_of(p.delta + brow0, p.R * 4), rmx = buffer_of(p.delta + rows + brow0, p.R * 4);
  const unsigned qts = static_cast<unsigned>(p.q.ts) * 2, gts = static_cast<unsigned>(p.go.ts) * 2;
  const unsigned yts = static_cast<unsigned>(C) * 2, hs = static_cast<unsigned>(p.d) * 2;

  const long r_end = min(p.R, (static_cast<long>(rb) + 1) * p.rows_per);
  RowWalk w(static_cast<long>(rb) * p.rows_per + wid * 32 + j, p.Tq);
  V8 qf[NKS], gf[NKS];
  float lse = 0.0f;
  auto load_rows = [&]() {
    const bool ok = w.row < r_end && w.i < qlen;
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks) {
      const int c = ks * 16 + hh * 8;
      const bool there = ok && c < p.d;
      const unsigned col = w.hi * hs + c * 2;
      qf[ks] = load8<V8>(rq, there ? w.i * qts + col : NOWHERE);
      gf[ks] = load8<V8>(rg, there ? w.i * gts + col : NOWHERE);
    }
    lse = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rl, static_cast<int>(ok ? static_cast<unsigned>(w.row) * 4 : NOWHERE), 0, 0));
  };
  load_rows();
  const bool any = stage_short<T, D, NKT, KS, VS, true>(p, b, g, klen, sK, sV, sB);
  const float c2 = p.scale * LOG2E;
  while (w.row - j < r_end) {
    const bool in = w.row < r_end, ok = any && in && w.i < qlen;
    const unsigned yoff = w.i * yts + w.hi * hs, loff = in && hh == 0 ? static_cast<unsigned>(w.row) * 4 : NOWHERE;
    const float lse2 = ok && lse != -INFINITY ? lse * LOG2E : INFINITY;
    float dl = 0.0f, sum = 0.0f, hi = -INFINITY, lo = INFINITY;
    V8 df[2 * NKT];
    v16f ps[NKT], dps[NKT];
#pragma unroll
    for (int kt = 0; kt < NKT; ++kt) {
      hold_order();                      // (one key tile's operands at a time)
      v16f s = start_scores(sB + kt * 32, hh), dp = zero16();
#pragma unroll
      for (int ks = 0; ks < NKS; ++ks) {
        s = mfma16(frag_rows<T>(sK, KS, kt * 32 + j, ks, hh), qf[ks], s);
        dp = mfma16(frag_rows<T>(sV, VS, kt * 32 + j, ks, hh), gf[ks], dp);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float pr = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], c2, -lse2));
        dl = __builtin_fmaf(pr, dp[r], dl);
        sum += pr;
        if (is_f16<T>()) hi = fmaxf(hi, dp[r]), lo = fminf(lo, dp[r]);          // (a dropped key's dp is a kept one's)
        s[r] = pr;
      }
      ps[kt] = s;
      dps[kt] = dp;
    }
    // (the p sum to 1 up to the rounding of lse, 2^-23 |lse|; times D that is not small against ds where a row is nearly one key)
    sum += __shfl_xor(sum, 32, 64);
    dl += __shfl_xor(dl, 32, 64);
    dl = sum != 0.0f ? dl / sum : 0.0f;
    float f = 1.0f, inv_f = 1.0f;
    if (is_f16<T>()) {
      const float mx = fmaxf(fmaxf(hi, __shfl_xor(hi, 32, 64)) - dl, dl - fminf(lo, __shfl_xor(lo, 32, 64)));
      const float fe = static_cast<float>(inv_exponent(mx) + DS_TOP);
      f = __builtin_amdgcn_exp2f(fe);
      inv_f = __builtin_amdgcn_exp2f(-fe);
      __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(ok ? mx : 0.0f), rmx, static_cast<int>(loff), 0, 0);          // (k_xattn_dkv's range)
    }
#pragma unroll
    for (int kt = 0; kt < NKT; ++kt) {
#pragma unroll
      for (int r = 0; r < 16; ++r) ps[kt][r] *= is_f16<T>() ? __builtin_fmaf(dps[kt][r], f, -dl * f) : dps[kt][r] - dl;
#pragma unroll
      for (int u = 0; u < 2; ++u) df[2 * kt + u] = frag_regs<T>(ps[kt], u);
    }
    __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(dl), rdl, static_cast<int>(loff), 0, 0);
    hold_order();
    w.step();
    load_rows();
    v16f acc[NRT];
#pragma unroll
    for (int t = 0; t < NRT; ++t) acc[t] = zero16();
#pragma unroll
    for (int u = 0; u < 2 * NKT; ++u)
#pragma unroll
      for (int t = 0; t < NRT; ++t) acc[t] = mfma16(frag_cols<T>(sK, KS, u * 16, t, lane), df[u], acc[t]);
    zero_unless(ok, acc);
#pragma unroll
    for (int t = 0; t < NRT; ++t) store16<T>(ry, yoff, in, t * 32, hh, p.d, acc[t], p.scale * inv_f);
  }
}

// ---- dk and dv: four products per score, both sums in registers (2 x d fp32 a key).  Staging the next tile costs registers that d = 128 does not have twice:
// one wave a SIMD (436 registers), two LDS buffers spill (120 -> 400 us).  4 x 1000 x 1500, 16 heads on 4 of 128, lengths and mask drawn: 91 us, MFMA 12 % busy,
// 0.42 waves a SIMD on average (key blocks behind an item's length leave at once, and the slices are chosen by the stored length); 8 x 4096 x 77, 8 heads
// of 40: 27 us, of whose 128 keys a workgroup 77 are there.
template <int D> constexpr int dkv_rows() { return D <= 128 ? 64 : 32; }

template <typename T, int D>
__global__ __launch_bounds__(256, D <= 64 ? 2 : 1) void k_xattn_dkv(XattnP p) {
  constexpr int NKS = nks(D), NRT = nrt(D), S = stride_both(D), NR = dkv_rows<D>();
  using V8 = typename Vec8<T>::type;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  unsigned char* sQ = smem;
  unsigned char* sG = smem + NR * S;
  float* sL = reinterpret_cast<float*>(smem + 2 * NR * S);          // lse (base 2) of the tile's rows, +inf: not a row; -D of them
  float* sD = sL + NR;
  float* sM = sD + NR;                                              // 4 floats: the waves' maxima
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6, j = lane & 31, hh = lane >> 5;
  int b, g, blk;
  pair_block(p.G, p.nrb * p.nsplit, b, g, blk);
  const int sp = blk % p.nsplit, kbk = blk / p.nsplit;
  const int qlen = clamp_len(p.q_lens, b, p.Tq), klen = clamp_len(p.kv_lens, b, p.Tk);
  const int key = kbk * 128 + wid * 32 + j;
  const bool keep = key < klen && (!p.mask || p.mask[b * p.mask_bs + key] != 0);
  const bool work = __any(keep);
  const long brow0 = (static_cast<long>(b) * p.H + g * p.rep) * p.Tq;          // the row space of (b, g) inside [B][H][Tq]
  const float* dmax = p.delta + static_cast<long>(p.B) * p.H * p.Tq + brow0;          // fp16: the rows' largest |dp - D|

  const int nt = static_cast<int>((p.R + NR - 1) / NR), per = (nt + p.nsplit - 1) / p.nsplit;
  const int t0 = sp * per;
  int t1 = min(nt, t0 + per);
  if (kbk * 128 >= klen || qlen == 0) t1 = t0;          // nothing to sum: zeros are written below
  if (p.nsplit > 1 && kbk * 128 >= klen) return;          // (k_xattn_sum knows)

  V8 kf[NKS], vf[NKS];
  {
    const T* krow = static_cast<const T*>(p.k.p) + b * p.k.bs + key * p.k.ts + static_cast<long>(g) * p.d;
    const T* vrow = static_cast<const T*>(p.v.p) + b * p.v.bs + key * p.v.ts + static_cast<long>(g) * p.d;
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks) {
      const int c = ks * 16 + hh * 8;
      uint4 a = make_uint4(0, 0, 0, 0), w = a;
      if (keep && c < p.d) {
        a = *reinterpret_cast<const uint4*>(krow + c);
        w = *reinterpret_cast<const uint4*>(vrow + c);
      }
      kf[ks] = __builtin_bit_cast(V8, a);
      vf[ks] = __builtin_bit_cast(V8, w);
    }
  }
  constexpr float PSHIFT = is_f16<T>() ? 12.0f : 0.0f;
  float ff = 1.0f, unf = 1.0f;          // the power of two in ds, relative to the one in p, and what takes it out again
  if (is_f16<T>() && t0 < t1) {
    float mx = 0.0f;
    for (long r = static_cast<long>(t0) * NR + tid; r < min(p.R, static_cast<long>(t1) * NR); r += 256) mx = fmaxf(mx, dmax[r]);
    mx = wave_reduce_max(mx);
    if (lane == 0) sM[wid] = mx;
    __syncthreads();
    const int fe = inv_exponent(fmaxf(fmaxf(sM[0], sM[1]), fmaxf(sM[2], sM[3]))) + DS_TOP;
    ff = __builtin_amdgcn_exp2f(static_cast<float>(fe) - PSHIFT);
    unf = __builtin_amdgcn_exp2f(static_cast<float>(-fe));
  }
  const T* qb = static_cast<const T*>(p.q.p) + b * p.q.bs + static_cast<long>(g) * p.rep * p.d;
  const T* gb = static_cast<const T*>(p.go.p) + b * p.go.bs + static_cast<long>(g) * p.rep * p.d;
  RowTile2<T, D, NR, S> tile;
  tile.start(static_cast<long>(t0) * NR, p.R, p.Tq, p.d, p.q.ts, p.go.ts);
  long srow = static_cast<long>(t0) * NR + tid;          // threads below NR: the row whose statistics this one brings
  int si = static_cast<int>(srow % p.Tq);
  float rl = INFINITY, rd = 0.0f;
  auto fetch = [&]() {
    tile.load(qb, gb, p.Tq, qlen, p.d);
    if (tid < NR) {
      rl = INFINITY;
      rd = 0.0f;
      if (srow < p.R && si < qlen) {
        const float v = p.lse_in[brow0 + srow];
        rl = v == -INFINITY ? INFINITY : v * LOG2E;
        rd = p.delta[brow0 + srow];
      }
      srow += NR;
      si += tile.di;
      si -= si >= p.Tq ? p.Tq : 0;
    }
  };
  const float c2 = p.scale * LOG2E;
  v16f bias;
#pragma unroll
  for (int r = 0; r < 16; ++r) bias[r] = keep ? 0.0f : -INFINITY;
  v16f ak[NRT], av[NRT];
#pragma unroll
  for (int t = 0; t < NRT; ++t) ak[t] = zero16(), av[t] = zero16();
  if (t0 < t1) fetch();
  for (int t = t0; t < t1; ++t) {
    __syncthreads();
    tile.store(sQ, sG);
    if (tid < NR) sL[tid] = rl - PSHIFT, sD[tid] = -rd;
    __syncthreads();
    if (t + 1 < t1) fetch();
    if (work) {
      // operand reads run ahead of the products: the rows of the next half, and the transposed tiles while the exponentials are taken
      V8 qr[NKS], gr[NKS];
      auto read_rows = [&](int half) {
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks) {
          qr[ks] = frag_rows<T>(sQ, S, half * 32 + j, ks, hh);
          gr[ks] = frag_rows<T>(sG, S, half * 32 + j, ks, hh);
        }
      };
      read_rows(0);
#pragma unroll
      for (int half = 0; half < NR / 32; ++half) {
        hold_order();
        v16f s = bias, dp = start_scores(sD + half * 32, hh);          // (-inf for a dropped key; dp - D)
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks) {
          s = mfma16(qr[ks], kf[ks], s);
          dp = mfma16(gr[ks], vf[ks], dp);
        }
        V8 gt[2][NRT], qt[2][NRT];
        auto read_cols = [&](int u) {
#pragma unroll
          for (int t2 = 0; t2 < NRT; ++t2) {
            gt[u][t2] = frag_cols<T>(sG, S, half * 32 + u * 16, t2, lane);
            qt[u][t2] = frag_cols<T>(sQ, S, half * 32 + u * 16, t2, lane);
          }
        };
        read_cols(0);
        if (D <= 128) read_cols(1);          // (at 160 the registers hold one of the two)
        deal_reads<2 * NKS, 2>();
        hold_order();
#pragma unroll
        for (int a = 0; a < 4; ++a) {
          const float4 L = *reinterpret_cast<const float4*>(sL + half * 32 + 8 * a + 4 * hh);
          const float lv[4] = {L.x, L.y, L.z, L.w};
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int r = 4 * a + c;
            const float pr = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], c2, -lv[c]));
            s[r] = pr;
            dp[r] = is_f16<T>() ? pr * dp[r] * ff : pr * dp[r];
          }
        }
        V8 pf[2], df[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) pf[u] = frag_regs<T>(s, u), df[u] = frag_regs<T>(dp, u);
        hold_order();
        if (half + 1 < NR / 32) read_rows(half + 1);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          if (u == 1 && D > 128) {
            hold_order();
            read_cols(1);
          }
#pragma unroll
          for (int t2 = 0; t2 < NRT; ++t2) {
            av[t2] = mfma16(gt[u][t2], pf[u], av[t2]);
            ak[t2] = mfma16(qt[u][t2], df[u], ak[t2]);
          }
        }
        if (half + 1 < NR / 32) deal_reads<4 * NRT, 1>();
      }
    }
  }
  if (key >= (p.nsplit > 1 ? klen : p.Tk)) return;
  zero_unless(keep, ak);          // (a live row that is not finite makes 0 * inf of a dropped key's zeros)
  zero_unless(keep, av);
  const float fk = p.scale * unf, fv = is_f16<T>() ? 1.0f / 4096.0f : 1.0f;
  const long krow = (static_cast<long>(b) * p.Tk + key) * p.G + g;
  if (p.nsplit > 1) {
    const long n = static_cast<long>(p.B) * p.Tk * p.G * p.d;
    float* pk = p.part + 2 * sp * n + krow * p.d;
#pragma unroll
    for (int t = 0; t < NRT; ++t) {
      store16_f32(pk, t * 32, hh, p.d, ak[t], fk);
      store16_f32(pk + n, t * 32, hh, p.d, av[t], fv);
    }
    return;
  }
#pragma unroll
  for (int t = 0; t < NRT; ++t) {
    store16<T>(static_cast<T*>(p.dk) + krow * p.d, t * 32, hh, p.d, ak[t], fk);
    store16<T>(static_cast<T*>(p.dv) + krow * p.d, t * 32, hh, p.d, av[t], fv);
  }
}

// dk and dv: the slices' sums in order; 8 channels a thread.  HBM: 4 x 1500 x 512, two slices: 6 us
template <typename T>
__global__ __launch_bounds__(256) void k_xattn_sum(XattnP p, long n) {
  const long i = (static_cast<long>(blockIdx.x) * 256 + threadIdx.x) * 8;
  if (i >= 2 * n) return;
  float a[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) a[e] = 0.0f;
  const long key = (i < n ? i : i - n) / (static_cast<long>(p.G) * p.d);          // of [B][Tk]
  const int b = static_cast<int>(key / p.Tk);
  const int slices = key - static_cast<long>(b) * p.Tk < clamp_len(p.kv_lens, b, p.Tk) ? p.nsplit : 0;          // (nothing was written behind the length)
  for (int s = 0; s < slices; ++s) {
    const float4* q = reinterpret_cast<const float4*>(p.part + 2 * s * n + i);
    const float4 x = q[0], y = q[1];
    a[0] += x.x; a[1] += x.y; a[2] += x.z; a[3] += x.w; a[4] += y.x; a[5] += y.y; a[6] += y.z; a[7] += y.w;
  }
  typename Vec8<T>::type w;
#pragma unroll
  for (int e = 0; e < 8; ++e) w[e] = static_cast<T>(a[e]);
  T* out = i < n ? static_cast<T*>(p.dk) + i : static_cast<T*>(p.dv) + (i - n);
  *reinterpret_cast<typename Vec8<T>::type*>(out) = w;
}

template <typename T, int D, int NKT>
int launch_dq_short(tfmq_handle h, XattnP p, hipStream_t st) {
  auto kern = &k_xattn_dq_short<T, D, NKT>;
  constexpr int smem = NKT * 32 * (stride_both(D) + stride_rows(D) + 4);
  static LdsRoom room_kern;
  TFMQ_HIP(h, room_kern.ask(h, reinterpret_cast<const void*>(kern), smem));
  const long pairs = static_cast<long>(p.B) * p.G;
  p.rows_per = short_rows(h, pairs, p.R, dq_short_waves(D, NKT));
  p.nrb = ceil_div(p.R, p.rows_per);
  TFMQ_CHECK_ARG(h, pairs * p.nrb < MAX_BLOCKS, "xattn_bwd: too many workgroups");
  hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>(pairs * p.nrb)), dim3(256), smem, st, p);
  TFMQ_LAUNCH_CHECK(h);
  return TFMQ_OK;
}
template <typename T, int D>
int launch_dq(tfmq_handle h, XattnP p, hipStream_t st) {
  const int nkt = rows_fit(p) ? (p.Tk + 31) / 32 : 5;
  if (nkt == 1) return launch_dq_short<T, D, 1>(h, p, st);
  if (nkt == 2) return launch_dq_short<T, D, 2>(h, p, st);
  if (nkt == 3) return launch_dq_short<T, D, 3>(h, p, st);
  if (nkt == 4) return launch_dq_short<T, D, 4>(h, p, st);
  auto kern = &k_xattn_dq<T, D>;
  constexpr int smem = 64 * (stride_both(D) + stride_rows(D));
  static LdsRoom room_kern;
  TFMQ_HIP(h, room_kern.ask(h, reinterpret_cast<const void*>(kern), smem));
  p.nrb = ceil_div(p.R, 128);
  const long n = static_cast<long>(p.B) * p.G * p.nrb;
  TFMQ_CHECK_ARG(h, n < MAX_BLOCKS, "xattn_bwd: too many workgroups");
  hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>(n)), dim3(256), smem, st, p);
  TFMQ_LAUNCH_CHECK(h);
  return TFMQ_OK;
}

template <typename T>
int launch_bwd(tfmq_handle h, XattnP p, hipStream_t st) {
  return for_head_dim(p.d, [&](auto dc) {
    constexpr int D = decltype(dc)::value;
    auto kk = &k_xattn_dkv<T, D>;
    constexpr int sk = 2 * dkv_rows<D>() * (stride_both(D) + 4) + 16;
    static LdsRoom room_kk;
    TFMQ_HIP(h, room_kk.ask(h, reinterpret_cast<const void*>(kk), sk));
    const int rc = launch_dq<T, D>(h, p, st);
    if (rc != TFMQ_OK) return rc;
    XattnP c = p;
    c.nrb = ceil_div(p.Tk, 128);
    const long nk = static_cast<long>(p.B) * p.G * c.nrb * p.nsplit;
    TFMQ_CHECK_ARG(h, nk < MAX_BLOCKS, "xattn_bwd: too many workgroups");
    hipLaunchKernelGGL(kk, dim3(static_cast<unsigned>(nk)), dim3(256), sk, st, c);
    TFMQ_LAUNCH_CHECK(h);
    if (p.nsplit > 1) {
      const long n = static_cast<long>(p.B) * p.Tk * p.G * p.d;
      hipLaunchKernelGGL((k_xattn_sum<T>), dim3(static_cast<unsigned>((2 * n / 8 + 255) / 256)), dim3(256), 0, st, p, n);
      TFMQ_LAUNCH_CHECK(h);
    }
    return TFMQ_OK;
  });
}

}  // namespace

// Slices of the rows in the dk / dv kernel: only where its key blocks leave CUs idle; at least two row tiles a slice.  Two workgroups a CU; us for
// 1 / 2 / 4 / 8 / 16 slices of the whole backward pass: 8 x 4096 x 77, 8 heads of 40 (64 key blocks) 139 / 88 / 62 / 53 / 59; 4 x 1000 x 1500, 16 heads on
// 4 of 128 (192 key blocks), mean over three draws of the lengths, 239 / 177 / 171 / 181 / 220.
extern "C" int tfmq_xattn_bwd_splits(tfmq_handle h, int B, int H, int G, int Tq, int Tk) {
  if (!h || B <= 0 || H <= 0 || G <= 0 || H % G || Tq <= 0 || Tk <= 0) return 1;
  const long blocks = static_cast<long>(B) * G * ceil_div(Tk, 128), R = static_cast<long>(H / G) * Tq;
  const long want = 2L * h->cu_count;
  if (blocks * 2 > want) return 1;
  const long most = (R + 127) / 128, n = want / blocks;
  return static_cast<int>(n < 1 ? 1 : n < most ? n : most);
}

extern "C" int tfmq_xattn_bwd(tfmq_handle h, const tfmq_xattn_desc* a, void* stream) {
  TFMQ_CHECK_ARG(h, h && a, "xattn_bwd: null pointer");
  DeviceGuard guard(h);
  TFMQ_CHECK_ARG(h, a->B > 0 && a->H > 0 && a->G > 0 && a->H % a->G == 0 && a->Tq > 0 && a->Tk > 0 && a->d > 0 && a->d <= 160 && a->d % 8 == 0,
                 "xattn_bwd: bad shape");
  TFMQ_CHECK_ARG(h, a->dtype == 1 || a->dtype == 2, "xattn_bwd: fp16 or bf16");
  TFMQ_CHECK_ARG(h, a->q && a->k && a->v && a->o && a->go && a->lse && a->dq && a->dk && a->dv && a->ws, "xattn_bwd: null tensor");
  TFMQ_CHECK_ARG(h, a->nsplit >= 1, "xattn_bwd: bad slice count");
  TFMQ_CHECK_ARG(h, a->k_ts < (1 << 23) && a->v_ts < (1 << 23) && a->k_ts >= 0 && a->v_ts >= 0, "xattn_bwd: token strides of k and v must lie in [0, 2^23)");
  XattnP p{};
  p.q = {a->q, a->q_bs, a->q_ts};
  p.k = {a->k, a->k_bs, a->k_ts};
  p.v = {a->v, a->v_bs, a->v_ts};
  p.o = {a->o, a->o_bs, a->o_ts};
  p.go = {a->go, a->go_bs, a->go_ts};
  p.lse_in = a->lse;
  p.y = a->dq;
  p.dk = a->dk;
  p.dv = a->dv;
  p.q_lens = a->q_lens;
  p.kv_lens = a->kv_lens;
  p.mask = a->mask;
  p.mask_bs = a->mask_bs;
  p.B = a->B; p.H = a->H; p.G = a->G; p.rep = a->H / a->G; p.Tq = a->Tq; p.Tk = a->Tk; p.d = a->d;
  p.R = static_cast<long>(p.rep) * p.Tq;
  p.scale = a->scale;
  p.nsplit = a->nsplit;
  const long rows = static_cast<long>(p.B) * p.H * p.Tq;
  p.delta = a->ws;
  p.part = a->ws + (2 * rows + 3) / 4 * 4;
  return a->dtype == 1 ? launch_bwd<_Float16>(h, p, as_stream(stream)) : launch_bwd<__bf16>(h, p, as_stream(stream));
}
