// Shared pieces of the cross attention kernels (attention_cross_fwd.hip, attention_cross_bwd.hip): operand types, the tile staging and the
// transposed fragment reads.
//
// Rows and heads: the R = (H / G) Tq query rows that share key head g of item b are one row space, row r = query r % Tq of head g H / G + r / Tq,
// so shared key heads cost nothing extra and a one-token call still fills a fragment with its H / G heads.
#pragma once
#include "conv_common.hpp"
#include <algorithm>
#include <type_traits>

namespace xattn {

typedef float v16f __attribute__((ext_vector_type(16)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef short v8s __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));

template <typename T> struct Vec8;
template <> struct Vec8<_Float16> { using type = v8h; };
template <> struct Vec8<__bf16> { using type = v8b; };

__device__ __forceinline__ v16f mfma16(v8h a, v8h b, v16f c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ v16f mfma16(v8b a, v8b b, v16f c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ v16f zero16() {
  v16f z;
#pragma unroll
  for (int r = 0; r < 16; ++r) z[r] = 0.0f;
  return z;
}

constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;
constexpr long MAX_BLOCKS = (1L << 32) / 256;          // of a launch: its threads (256 a workgroup) are counted in 32 bits

struct View {          // [B][T][heads * d] with unit channel stride; element strides
  const void* p;
  long bs, ts;
};

struct XattnP {
  View q, k, v, o, go;
  const float* lse_in;
  void *y, *dk, *dv;                 // forward: o; backward: dq, dk, dv; contiguous
  float *lse, *delta, *part;         // [B][H][Tq] each; split partials
  const int32_t *q_lens, *kv_lens;   // [B] or null
  const uint8_t* mask;               // [B][Tk] (row stride mask_bs) or null
  long mask_bs;
  int B, H, G, rep, Tq, Tk, d;
  long R;                            // rep * Tq
  float scale;
  int nrb, nsplit;                   // row (or key) blocks, slices of the other axis
  int rows_per;                      // short states: rows a workgroup walks
};

__device__ __forceinline__ int clamp_len(const int32_t* lens, int b, int T) { return lens ? min(max(lens[b], 0), T) : T; }

// (item, key head, block of the pair) of this workgroup, `nb` blocks a pair.  Workgroups go to the 8 XCDs in turn: with the heads running fastest a
// head's blocks, which read the same K and V, share an XCD (or few), and an item's blocks spread over all of them, so that items of different
// lengths load the XCDs evenly.  (Placement is a matter of speed only.)
__device__ __forceinline__ void pair_block(int G, int nb, int& b, int& g, int& blk) {
  const int q = blockIdx.x, r = q / G;
  g = q - r * G;
  b = r / nb;
  blk = r - b * nb;
}

// a fragment register r of half hh holds row 8 (r >> 2) + 4 hh + (r & 3) of a 32-row product
__device__ __forceinline__ constexpr int crow(int r, int hh) { return 8 * (r >> 2) + 4 * hh + (r & 3); }

// scores S^T of 64 keys (two products): those of dropped keys become -inf
__device__ __forceinline__ void drop_keys(v16f (&s)[2], unsigned long long keep, int hh) {
#pragma unroll
  for (int kt = 0; kt < 2; ++kt) {
    const unsigned bits = static_cast<unsigned>(keep >> (32 * kt)) >> (4 * hh);
#pragma unroll
    for (int r = 0; r < 16; ++r) s[kt][r] = ((bits >> crow(r, 0)) & 1) ? s[kt][r] : -INFINITY;
  }
}

// ---- a tile of NROW consecutive keys x D channels: global -> registers -> LDS (rows of STRIDE bytes).  The loads are unconditional (a scalar base,
// one 32-bit offset per piece for the whole walk; past the last stored key the last one is read again) and asynchronous; keys that are not kept,
// and channels from d on, become zeros on the way into LDS, so what a dropped place holds (NaN included) never reaches a product.
template <typename T, int D, int NROW, int STRIDE, int NT = 256>
struct KeyTile {
  static constexpr int DP = D / 8, N = NROW * DP, PT = (N + NT - 1) / NT;
  uint4 reg[PT];
  __device__ __forceinline__ static int row_of(int it) { return min((static_cast<int>(threadIdx.x) + it * NT) / DP, NROW - 1); }
  __device__ __forceinline__ static int piece_of(int it) { return (static_cast<int>(threadIdx.x) + it * NT) % DP; }
  // keys [k0, k0 + NROW) of a tensor with Tk stored keys, token stride ts (elements, NROW * ts * 2 < 2^31)
  __device__ __forceinline__ void load(const T* base, long ts, int k0, int Tk, int d) {
    const char* p = reinterpret_cast<const char*>(base + k0 * ts);
    const int last = Tk - 1 - k0;
#pragma unroll
    for (int it = 0; it < PT; ++it) reg[it] = *reinterpret_cast<const uint4*>(p + offset(it, min(row_of(it), last), ts, d));
  }
  // the same keys, those not kept (bits of `keep`) read from key `kept` of the tensor instead
  __device__ __forceinline__ void load_kept(const T* base, long ts, int k0, int kept, unsigned keep, int d) {
    const char *p = reinterpret_cast<const char*>(base + k0 * ts), *q = reinterpret_cast<const char*>(base + kept * ts);
#pragma unroll
    for (int it = 0; it < PT; ++it) {
      const bool own = (keep >> row_of(it)) & 1;
      reg[it] = *reinterpret_cast<const uint4*>((own ? p : q) + offset(it, own ? row_of(it) : 0, ts, d));
    }
  }
  __device__ __forceinline__ static unsigned offset(int it, int row, long ts, int d) {
    return static_cast<unsigned>(row) * static_cast<unsigned>(ts * 2) + static_cast<unsigned>(min(piece_of(it) * 8, d - 8) * 2);
  }
  __device__ __forceinline__ void store(unsigned char* lds, unsigned long long keep, unsigned long long all, int d) {
    if (keep != all || d != D) {
#pragma unroll
      for (int it = 0; it < PT; ++it)
        if (!((keep >> row_of(it)) & 1) || piece_of(it) * 8 >= d) reg[it] = make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int it = 0; it < PT; ++it)
      if (N % NT == 0 || static_cast<int>(threadIdx.x) + it * NT < N) *reinterpret_cast<uint4*>(lds + row_of(it) * STRIDE + piece_of(it) * 16) = reg[it];
  }
};

// ---- tiles of NROW rows of the row space, walked in order, of two tensors at once (queries and upstream gradients).  A thread keeps where its rows are
// and steps NROW rows ahead (no division in the loop); rows past the end, or behind q_lens, are read from the item's first row and become zeros.
template <typename T, int D, int NROW, int STRIDE, int NT = 256>
struct RowTile2 {
  static constexpr int DP = D / 8, N = NROW * DP, PT = (N + NT - 1) / NT;
  uint4 a[PT], b[PT];
  long oa[PT], ob[PT];          // element offsets of the rows
  int i[PT];                    // their query index
  long left;                    // rows from the tile's first on
  unsigned live;
  int di;
  long da, db, wa, wb;          // a step of NROW rows, and of a wrap to the next head
  __device__ __forceinline__ static int row_of(int it) { return min((static_cast<int>(threadIdx.x) + it * NT) / DP, NROW - 1); }
  __device__ __forceinline__ static int piece_of(int it) { return (static_cast<int>(threadIdx.x) + it * NT) % DP; }
  __device__ __forceinline__ void start(long row0, long R, int Tq, int d, long ats, long bts) {
    const int dh = NROW / Tq;
    di = NROW - dh * Tq;
    da = di * ats + static_cast<long>(dh) * d;
    db = di * bts + static_cast<long>(dh) * d;
    wa = d - Tq * ats;
    wb = d - Tq * bts;
    left = R - row0;
#pragma unroll
    for (int it = 0; it < PT; ++it) {
      const long row = row0 + row_of(it), h = row / Tq;
      i[it] = static_cast<int>(row - h * Tq);
      oa[it] = i[it] * ats + h * d;
      ob[it] = i[it] * bts + h * d;
    }
  }
  // the tile at hand into registers, and a step ahead
  __device__ __forceinline__ void load(const T* pa, const T* pb, int Tq, int qlen, int d) {
    live = 0;
#pragma unroll
    for (int it = 0; it < PT; ++it) {
      const bool ok = row_of(it) < left && i[it] < qlen;
      const int c = min(piece_of(it) * 8, d - 8);
      a[it] = *reinterpret_cast<const uint4*>(pa + (ok ? oa[it] : 0) + c);
      b[it] = *reinterpret_cast<const uint4*>(pb + (ok ? ob[it] : 0) + c);
      live |= (ok && piece_of(it) * 8 < d ? 1u : 0u) << it;
      i[it] += di;
      const bool wrap = i[it] >= Tq;
      i[it] -= wrap ? Tq : 0;
      oa[it] += da + (wrap ? wa : 0);
      ob[it] += db + (wrap ? wb : 0);
    }
    left -= NROW;
  }
  __device__ __forceinline__ void store(unsigned char* la, unsigned char* lb) {
    if (__any(live != (1u << PT) - 1)) {
#pragma unroll
      for (int it = 0; it < PT; ++it)
        if (!((live >> it) & 1)) a[it] = b[it] = make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int it = 0; it < PT; ++it)
      if (N % NT == 0 || static_cast<int>(threadIdx.x) + it * NT < N) {
        *reinterpret_cast<uint4*>(la + row_of(it) * STRIDE + piece_of(it) * 16) = a[it];
        *reinterpret_cast<uint4*>(lb + row_of(it) * STRIDE + piece_of(it) * 16) = b[it];
      }
  }
};

// keeps the order of what stands before and behind it: operand reads asked for early stay early
__device__ __forceinline__ void hold_order() { __builtin_amdgcn_sched_barrier(0); }
// N matrix instructions with R LDS reads behind each: the LDS counter holds 15 reads, a burst of more would stall the wave behind them
template <int N, int R>
__device__ __forceinline__ void deal_reads() {
  if constexpr (N > 0) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    __builtin_amdgcn_sched_group_barrier(0x100, R, 0);
    deal_reads<N - 1, R>();
  }
}

// rows [row0, row0 + 32) of a tile as an operand, channels [16 ks, +16): lane j = row, half hh = 8 of the 16 channels
template <typename T>
__device__ __forceinline__ typename Vec8<T>::type frag_rows(const unsigned char* lds, int stride, int row, int ks, int hh) {
  return *reinterpret_cast<const typename Vec8<T>::type*>(lds + row * stride + (ks * 16 + hh * 8) * 2);
}

// The tile transposed: channels [32 t, +32) as the operand's rows, tile rows [r0, +16) as its 16 reduction steps, in the order in which a lane
// of the other operand holds a product's registers (half hh: rows r0 + 4 hh + (0 .. 3), then r0 + 8 + 4 hh + (0 .. 3)).  ds_read_b64_tr_b16 hands lane
// i of 16 the i-th of 16 channels of four rows; the channel groups are dealt so that register r of half hh of the result is channel
// 32 t + 16 (r >> 3) + 8 hh + (r & 7): eight consecutive ones, and the two halves of a wave side by side, so that a store covers 32 bytes of a row.
template <typename T>
__device__ __forceinline__ typename Vec8<T>::type frag_cols(const unsigned char* lds, int stride, int r0, int t, int lane) {
  const int L = lane & 15, gg = (lane >> 4) & 1, hh = lane >> 5, cg = L & 3;
  const unsigned char* p = lds + (r0 + 4 * hh + (L >> 2)) * stride + (t * 32 + 16 * gg + 8 * (cg & 1) + 4 * (cg >> 1)) * 2;
  using P = __attribute__((address_space(3))) v4s*;
  const v4s a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(p));
  const v4s b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(p + 8 * stride));
  v8s w;
  w[0] = a[0]; w[1] = a[1]; w[2] = a[2]; w[3] = a[3]; w[4] = b[0]; w[5] = b[1]; w[6] = b[2]; w[7] = b[3];
  return __builtin_bit_cast(typename Vec8<T>::type, w);
}

// registers 8 u .. 8 u + 7 of a product, rounded, as the operand of the reduction step that frag_cols feeds with rows 16 u ...
template <typename T>
__device__ __forceinline__ typename Vec8<T>::type frag_regs(const v16f& s, int u) {
  typename Vec8<T>::type f;
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = static_cast<T>(s[8 * u + e]);
  return f;
}

// ---- buffers whose reads past the end give zeros and whose writes past it are dropped: rows and channels that are not there need no branches, and
// without branches around them the compiler can count stores and loads apart (a wait for the next rows does not wait for the last stores)
typedef unsigned v4u __attribute__((ext_vector_type(4)));
using Rsrc = __amdgpu_buffer_rsrc_t;
constexpr unsigned NOWHERE = 0xfffffff0u;
__device__ __forceinline__ Rsrc buffer_of(const void* p, long bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(uniform_ptr(static_cast<const char*>(p))), 0, __builtin_amdgcn_readfirstlane(static_cast<int>(bytes)), 0x00027000);
}
template <typename V8>
__device__ __forceinline__ V8 load8(Rsrc r, unsigned off) {
  return __builtin_bit_cast(V8, __builtin_amdgcn_raw_buffer_load_b128(r, static_cast<int>(off), 0, 0));
}
// a lane's 16 channels (of 32 from c0 on) of the row at byte `row`
template <typename T>
__device__ __forceinline__ void store16(Rsrc r, unsigned row, bool ok, int c0, int hh, int d, const v16f& v, float f) {
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    const int c = c0 + 16 * g + 8 * hh;
    typename Vec8<T>::type w;
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = static_cast<T>(v[8 * g + e] * f);
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(v4u, w), r, static_cast<int>(ok && c < d ? row + 2 * c : NOWHERE), 0, 0);
  }
}

// a lane's place in the row space of one (item, key head), 128 rows further each step
struct RowWalk {
  long row;
  int hi, i, dh, di, Tq;
  __device__ __forceinline__ RowWalk(long r, int tq) : row(r), Tq(tq) {
    hi = static_cast<int>(r / Tq);
    i = static_cast<int>(r - static_cast<long>(hi) * Tq);
    dh = 128 / Tq;
    di = 128 - dh * Tq;
  }
  __device__ __forceinline__ void step() {
    row += 128;
    hi += dh;
    i += di;
    if (i >= Tq) {
      i -= Tq;
      ++hi;
    }
  }
};

// all of up to 128 states into LDS and 0 / -inf per key; a barrier behind it.  -> whether any key is kept.  Channels from d on are zeros.  A dropped key's
// row of K is a kept one's: its score is -inf plus a finite number or what that key's is, so a query that is not finite (0 * inf with zeros) gives what it
// gives over the kept keys alone.  Its row of V is zeros in the forward (p v adds nothing whatever the kept ones hold), a kept one's in the gradients
// (VKEPT: go v then has no value that no kept key has).
template <typename T, int D, int NKT, int KS, int VS, bool VKEPT>
__device__ __forceinline__ bool stage_short(const XattnP& p, int b, int g, int klen, unsigned char* sK, unsigned char* sV, float* sB) {
  const int lane = threadIdx.x & 63;
  const T* kb = static_cast<const T*>(p.k.p) + b * p.k.bs + static_cast<long>(g) * p.d;
  const T* vb = static_cast<const T*>(p.v.p) + b * p.v.bs + static_cast<long>(g) * p.d;
  const uint8_t* mb = p.mask ? p.mask + b * p.mask_bs : nullptr;
  unsigned long long keep[2] = {0, 0};
#pragma unroll
  for (int w = 0; w < (NKT + 1) / 2; ++w) {
    const int key = w * 64 + lane;
    const bool kept = key < klen && (!mb || mb[min(key, p.Tk - 1)] != 0);
    keep[w] = __ballot(kept);
    if (threadIdx.x < 64 && key < NKT * 32) sB[key] = kept ? 0.0f : -INFINITY;
  }
  const int first = keep[0] ? __ffsll(keep[0]) - 1 : keep[1] ? 63 + __ffsll(keep[1]) : 0;
#pragma unroll
  for (int t = 0; t < NKT; ++t) {
    KeyTile<T, D, 32, KS> tk;
    KeyTile<T, D, 32, VS> tv;
    const int k0 = min(t * 32, p.Tk - 1);
    const unsigned kk = static_cast<unsigned>(keep[t >> 1] >> (32 * (t & 1)));
    tk.load_kept(kb, p.k.ts, k0, first, kk, p.d);
    if (VKEPT) tv.load_kept(vb, p.v.ts, k0, first, kk, p.d);
    else tv.load(vb, p.v.ts, k0, p.Tk, p.d);
    tk.store(sK + t * 32 * KS, 0xffffffffull, 0xffffffffull, p.d);
    tv.store(sV + t * 32 * VS, VKEPT ? 0xffffffffull : kk, 0xffffffffull, p.d);
  }
  __syncthreads();
  return (keep[0] | keep[1]) != 0;
}

// scores start from 0 for kept keys and from -inf for dropped ones: a mask costs no arithmetic
__device__ __forceinline__ v16f start_scores(const float* bias, int hh) {
  v16f s;
#pragma unroll
  for (int a = 0; a < 4; ++a) {
    const float4 b = *reinterpret_cast<const float4*>(bias + 8 * a + 4 * hh);
    s[4 * a] = b.x; s[4 * a + 1] = b.y; s[4 * a + 2] = b.z; s[4 * a + 3] = b.w;
  }
  return s;
}

// what a row that is not there (or has no query), or a dropped key, leaves: zeros, whatever its lanes computed
template <int N>
__device__ __forceinline__ void zero_unless(bool ok, v16f (&a)[N]) {
  if (!ok) {
#pragma unroll
    for (int t = 0; t < N; ++t) a[t] = zero16();
  }
}

// a lane's 16 channels (of 32 from c0 on) of one row; those below d, d % 8 == 0
template <typename T>
__device__ __forceinline__ void store16(T* row, int c0, int hh, int d, const v16f& v, float f) {
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    const int c = c0 + 16 * g + 8 * hh;
    if (c >= d) continue;
    typename Vec8<T>::type w;
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = static_cast<T>(v[8 * g + e] * f);
    *reinterpret_cast<typename Vec8<T>::type*>(row + c) = w;
  }
}
__device__ __forceinline__ void store16_f32(float* row, int c0, int hh, int d, const v16f& v, float f) {
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int c = c0 + 16 * (q >> 1) + 8 * hh + 4 * (q & 1);
    if (c < d) *reinterpret_cast<float4*>(row + c) = make_float4(v[4 * q] * f, v[4 * q + 1] * f, v[4 * q + 2] * f, v[4 * q + 3] * f);
  }
}

constexpr int nks(int D) { return (D + 15) / 16; }
constexpr int nrt(int D) { return (D + 31) / 32; }
// LDS row strides (bytes).  Row fragments want an odd number of 16-byte units, transposed ones four rows 64 bytes apart modulo the 256 bytes of the
// banks; where a tile is read both ways the stride is the next odd multiple of 16 whose bank step is within 4 of that.
constexpr int stride_rows(int D) { return D * 2 + 16; }
constexpr int stride_cols(int D) { return (nrt(D) | 1) * 64; }
constexpr int stride_both(int D) {
  int s = D * 2;
  for (;; s += 16) {
    const int m = (s / 4) % 64;
    if ((s / 16) % 2 == 1 && s >= nrt(D) * 64 && (m == 12 || m == 20 || m == 44 || m == 52)) return s;
  }
}

// short states are staged once per workgroup: as many rows each (of pairs x R) as leave `per_cu` workgroups per CU
inline int short_rows(tfmq_handle h, long pairs, long R, int per_cu) {
  const long tiles = (R + 127) / 128;
  return static_cast<int>(std::min<long>(tiles, std::max<long>(1, pairs * tiles / (static_cast<long>(per_cu) * h->cu_count)))) * 128;
}

// the row walks address an item's rows with 32 bits (2 GiB a tensor and item); longer ones take the tiled kernels
inline bool rows_fit(const XattnP& p) {
  const long m = 1L << 30, C = static_cast<long>(p.H) * p.d;
  return p.Tq * C < m && p.q.ts >= 0 && p.q.ts * p.Tq + C < m && (!p.go.p || (p.go.ts >= 0 && p.go.ts * p.Tq + C < m && p.o.ts >= 0 && p.o.ts * p.Tq + C < m));
}

// head dims run in the smallest of these that holds them
template <typename F>
int for_head_dim(int d, F f) {
  if (d <= 32) return f(std::integral_constant<int, 32>{});
  if (d <= 48) return f(std::integral_constant<int, 48>{});
  if (d <= 64) return f(std::integral_constant<int, 64>{});
  if (d <= 80) return f(std::integral_constant<int, 80>{});
  if (d <= 96) return f(std::integral_constant<int, 96>{});
  if (d <= 128) return f(std::integral_constant<int, 128>{});
  return f(std::integral_constant<int, 160>{});
}

}  // namespace xattn
