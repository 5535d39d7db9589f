// Attention over packed sequences: the tokens of many requests stand behind one another without padding,
//
//     o[i, h] = sum_j p_ij v[j, h / G],   p_i = softmax_j( scale q[i, h] . k[j, h / G] + bias[h, clamp(j - pos_i, -R, R)] ),
//     pos_i = i + k_len - q_len  (the queries are the LAST q_len positions of their sequence),  j <= pos_i when causal,
//
// with G = heads / kv_heads query heads per key / value head, D = 64 or 128, bf16 or f16.  A row with nothing to attend to is 0.
//
// One pass over the keys with a running maximum and sum per row (fp32, exp2 domain).  Rows: the G query heads that share a key
// head are rows of ONE tile (row r of a sequence = query r / G, head kvh * G + r % G), so a key tile is read once for all of
// them and a single new token still fills G rows.  Both products are issued transposed, S^T = K Q^T and O^T = V^T P^T: a lane
// owns one row, its maximum / sum / rescale are lane-local but for one exchange with lane ^ 32.  The K rows enter the first MFMA
// in the order (bits 2 and 3 of the row swapped) in which its result registers are the second one's B operand: P never leaves
// the registers.  V^T fragments come from the row-major V tile by the transposing LDS read.
//
// Two kernels, by the rows of a batch's sequences:
//   tile  128 rows per workgroup, 32 per wave, key tiles of 32 shared by the four waves (LDS-DMA, two stages);
//   few   <= 32 rows each, some over more than 128 keys (new tokens): eight waves take different keys, each with its own LDS stage and no
//         barrier in the loop, and join at the end through LDS.
// Where there are too few workgroups for the chip the key range is split over several and joined by a third kernel.
// P is rounded to the operands' 16-bit type for the second product (half a step, relative, of every weight: the errors of
// independent weights average out below the output's own rounding); sums and statistics stay fp32.
#include "td_common.h"
#include <algorithm>
#include <math.h>
#include <type_traits>
#include <vector>

typedef __attribute__((address_space(3))) void* ap_lptr_t;
typedef short ap_v4s __attribute__((ext_vector_type(4)));
typedef unsigned ap_u4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) ap_v4s* ap_trptr_t;

#define AP_ROWS 128        // rows of a tile item
#define AP_FEW 32          // rows of a few item
#define AP_FEW_KEYS 128    // ... of batches with more keys for some than this, where all workgroups run at once (one token over 200 keys, 12 heads
                           // of 128: 5.5 against 7.5 us).  Where they do not, the tile kernel has three a CU, which pays up to
#define AP_MANY_KEYS 384   // ... this many (128 tokens over 150 keys each 39.9 against 26.1 us, 400: 68.7 against 60.0, 777: 116 against 127)
#define AP_PAD 96          // the bias table repeats its ends: distances within a key tile of the range need no clamp
#define AP_TAU 8.0f        // a row's reference moves when a score exceeds it by 8 (a weight of 2^8),
#define AP_LOOK 4096.0f    // looked for when a lane's weights of a tile add up to more than this (16; few kernel, D = 64: 32)
#define AP_STEP 4194304.0f // from here on a reference's own rounding (2^-24 of it) is a matter of weights: 2^22, where that is 2^0.25

// One workgroup's work per key head: `rows` rows from head `head0` of query token `token`, which stands at position `pos` of its
// sequence, over keys [key0, key1) of the sequence whose first key token is k_begin.  slot: row in the partial buffer, -1 = writes o
struct ApItem { int32_t token, head0, rows, pos, k_begin, key0, key1, slot; };
struct ApJoin { int32_t token, head0, rows, slot, splits, tile_rows, pad0, pad1; };
#define AP_GRID_Y 32768    // items per grid.z

struct ApParams {
  const uint16_t *q, *k, *v; uint16_t* o;
  int64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs, o_ts, o_hs;   // token / head strides, elements
  const float* bias; int R;                                  // [H, 2R + 1] or null
  const ApItem* items; int n_items;
  float* po; float* pml; int64_t ws_rows;                    // partials [Hkv][ws_rows][D], [Hkv][ws_rows][2] (max, sum)
  int Hkv, G, causal;
  uint32_t gmagic;                                           // ceil(2^32 / G): x / G = mulhi(x, gmagic) for x G < 2^32 (G > 1)
  float c;                                                   // scale * log2(e)
};

template <int DT> struct ap_mma;
template <> struct ap_mma<TD_F16> {
  __device__ static __forceinline__ v16f run(v4i a, v4i b, v16f c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
  }
};
template <> struct ap_mma<TD_BF16> {
  __device__ static __forceinline__ v16f run(v4i a, v4i b, v16f c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
  }
};

__device__ __forceinline__ float ap_other_half(float x, bool mx) {   // x of this lane (+ | max) x of lane ^ 32
  const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  const float a = __uint_as_float(s[0]), b = __uint_as_float(s[1]);
  return mx ? fmaxf(a, b) : a + b;
}

// Tiles in LDS: row-major, rows of 2 D bytes, the 16-byte chunks of a row permuted by an XOR so that the reads touch every
// bank once (K: ds_read_b128 by 16 lanes of 16 different rows; V: 4 rows x 64 bytes twice per transposing read)
template <int D> __device__ __forceinline__ uint32_t ap_kx(uint32_t row) { return D == 128 ? (row & 15u) : ((row >> 1) & 7u); }
template <int D> __device__ __forceinline__ uint32_t ap_vx(uint32_t row) { return D == 128 ? 4u * (row & 3u) : 4u * ((row >> 1) & 1u); }

// 64 lanes x 16 bytes from base + off (a lane each) to LDS, lane after lane; `bytes` bounds the offsets
__device__ __forceinline__ void ap_dma(const void* base, uint32_t bytes, char* lds, uint32_t off) {
  const auto r = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, (int)bytes, 0x00020000);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (ap_lptr_t)lds, 16, off, 0, 0, 0);
}

__device__ __forceinline__ void ap_store(void* base, uint32_t bytes, v4i v, uint32_t off) {   // an offset of `bytes` or more is not stored
  const auto r = __builtin_amdgcn_make_buffer_rsrc(base, 0, (int)bytes, 0x00020000);
  __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(ap_u4, v), r, off, 0, 0);
}
__device__ __forceinline__ void ap_dma_ptr(const void* src, char* lds) {   // the same from an address per lane
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src, (ap_lptr_t)lds, 16, 0, 0);
}

// query token (from the item's) and head of a row: rows run over the heads of a token first; x is less than a tile, so the
// division is one multiplication
__device__ __forceinline__ void ap_split(const ApParams& p, const ApItem& it, int x, int& q, int& h) {
  const int y = it.head0 + x;
  q = p.G > 1 ? (int)__umulhi((uint32_t)y, p.gmagic) : y;
  h = y - q * p.G;
}
// Whole rows between memory and LDS, 16 bytes a lane: lane / (ROWB / 16) of each group of rows.  The pointer steps from group to
// group: a step is a fixed number of tokens and heads, but for the carry from the last head to the next token.
template <int D> struct ApRowWalk {
  static constexpr int LPR = D / 8, RP = 64 / LPR;          // lanes per row, rows per group
  int64_t at; int h;                                        // element offset from the item's first token and this key head's first head
  int64_t step, carry; int dh, G;
  __device__ __forceinline__ ApRowWalk(const ApParams& p, const ApItem& it, int x, int64_t ts, int64_t hs) : G(p.G) {
    int q;
    ap_split(p, it, x, q, h);
    at = q * ts + h * hs;
    const int dq = G > 1 ? (int)__umulhi((uint32_t)RP, p.gmagic) : RP;
    dh = RP - dq * G;
    step = dq * ts + dh * hs;
    carry = ts - G * hs;
  }
  __device__ __forceinline__ void next() {
    at += step;
    h += dh;
    if (h >= G) { h -= G; at += carry; }
  }
};

// exp2 domain; finite values whose product with log2 e is past fp32 (from 2.36e38 on, the type's lowest among them) stay finite: a row of
// nothing else is a uniform row, and the order of the values is kept
template <int THREADS>
__device__ __forceinline__ void ap_load_bias(const ApParams& p, int kvh, int bn, float* lbias) {
  const float* b = p.bias + (int64_t)kvh * p.G * (2 * p.R + 1);
  for (int h = 0; h < p.G; ++h)
    for (int i = threadIdx.x; i < bn; i += THREADS) {
      const float x = b[h * (2 * p.R + 1) + max(0, min(2 * p.R, i - AP_PAD))];
      const float y = x * 1.4426950408889634f;
      lbias[h * bn + i] = fabsf(x) < INFINITY && fabsf(y) == INFINITY ? copysignf(3.4028235e38f, x) : y;
    }
}

// Scores of 32 N keys from kb, registers s[b][r] = key kb + 32 b + 16 (r >> 3) + 8 half + (r & 7) of this lane's row: bias and mask.
// Afterwards the score in the exp2 domain is mul * s + base.
struct ApScore {
  float c; int R; const float* lb;          // lb[key - position]
  float far_past, far_next;
  int pos, kmax, half;                      // this row's position and end
  int wfirst, wlast, wmin, wmax;            // the wave's first and last position, smallest and largest end
  template <bool BIAS, int N> __device__ __forceinline__ void finish(v16f (&s)[N], int kb, float& mul, float& base) const {
    mul = c;
    base = 0.f;
    if constexpr (BIAS) {
      const bool next = kb - wlast >= R, past = kb + 32 * N - 1 - wfirst <= -R;
      if (next || past) {                                     // all of it lies beyond the range: one value a row
        base = next ? far_next : far_past;
      } else {                                                // |key - position| < R + 96 everywhere
        const float* d = lb + (kb + 8 * half - pos);
#pragma unroll
        for (int b = 0; b < N; ++b)
#pragma unroll
          for (int r = 0; r < 16; ++r) s[b][r] = fmaf(s[b][r], c, d[32 * b + 16 * (r >> 3) + (r & 7)]);
        mul = 1.f;
      }
    }
    if (kb + 32 * N > wmin) {
      asm volatile("");                     // a branch: as selects the mask would cost every block three instructions a score
      const int lim = kmax - kb - 8 * half;
#pragma unroll
      for (int b = 0; b < N; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[b][r] = 32 * b + 16 * (r >> 3) + (r & 7) < lim ? s[b][r] : -INFINITY;
    }
  }
  template <int N> __device__ __forceinline__ float maximum(const v16f (&s)[N], float mul, float base) const {   // of the row
    float mx = s[0][0];
#pragma unroll
    for (int b = 0; b < N; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[b][r]);
    return fmaf(ap_other_half(mx, true), mul, base);
  }
};

// x0: the wave's first row within the item; this lane's row is x0 + (lane & 31), past the end the last one
template <bool BIAS>
__device__ __forceinline__ ApScore ap_score(const ApParams& p, const ApItem& it, int x0, int lane, const float* lbias, int bn) {
  ApScore sc;
  int q, h;
  ap_split(p, it, min(x0, it.rows - 1), q, h);
  sc.wfirst = it.pos + q;
  ap_split(p, it, min(x0 + 31, it.rows - 1), q, h);
  sc.wlast = it.pos + q;
  ap_split(p, it, min(x0 + (lane & 31), it.rows - 1), q, h);
  sc.c = p.c; sc.R = p.R; sc.half = lane >> 5;
  sc.pos = it.pos + q;
  sc.kmax = p.causal ? min(it.key1, sc.pos + 1) : it.key1;             // keys [key0, kmax) of this row
  sc.wmin = p.causal ? min(it.key1, sc.wfirst + 1) : it.key1;
  sc.wmax = p.causal ? min(it.key1, sc.wlast + 1) : it.key1;
  sc.lb = lbias + (BIAS ? h * bn + p.R + AP_PAD : 0);
  sc.far_past = BIAS ? sc.lb[-p.R] : 0.f;
  sc.far_next = BIAS ? sc.lb[p.R] : 0.f;
  return sc;
}

// Running state of a wave's rows: weights are exp2(score - ref).  ref is a row's maximum when it was last looked at, not its
// running maximum: the maximum of a tile is taken only when a lane's weights of it add up to more than 2^12 (of 60 vector instructions a
// block 24 less: 32 760 causal tokens 3.06 -> 2.85 ms).  Of 16 weights one must then be above 2^8, and the row moves; of 32 all may lie
// between 2^7 and 2^8, and the row is looked at again in the next such tile.  Weights up to 2^12 fit f16, bf16 and the fp32 sums.
//
// score = mul * s + base is fused into the exponent, so it is never rounded by itself, while ref is.  Where a score is large (a far tile
// under a bias of -1e9, products of 1e9) that rounding is many powers of two: a weight against ref could be anything.  Rows whose ref
// reaches AP_STEP take their scores rounded as ref was, so the largest weighs 1; they alone, for a row's bits are its own.
struct ApState {
  float m, ref, l;          // m: ref, or -infinity while the row has seen nothing
  bool look;                // a row of the wave has, or its ref is that large: the maximum of every tile is taken
};

// Scores of 32 NB keys from kt to weights, packed, and their sum into st.  FIRST: nothing to add to or to rescale, acc and st come in undefined.
template <int DT, int D, int NB, bool BIAS, bool FIRST>
__device__ __forceinline__ void ap_weights(const ApScore& score, int kt, v16f (&s)[NB], v16f (&acc)[D / 32], ApState& st, uint32_t (&pk)[NB][8]) {
  float mul, base;
  score.template finish<BIAS>(s, kt, mul, base);
  auto settle = [&]() {
    const bool own = fabsf(st.ref) >= AP_STEP;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[b][r] = own ? fmaf(s[b][r], mul, base) : s[b][r];
    mul = own ? 1.f : mul;
    base = own ? 0.f : base;
  };
  auto weights = [&]() {
    const float off = base - st.ref;
    float sum = 0.f;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int r = 0; r < 16; r += 2) {
        const float e0 = __builtin_amdgcn_exp2f(fmaf(s[b][r], mul, off)), e1 = __builtin_amdgcn_exp2f(fmaf(s[b][r + 1], mul, off));
        sum += e0 + e1;
        pk[b][r >> 1] = pack2<DT>(e0, e1);
      }
    return sum;
  };
  if constexpr (FIRST) {
    st.m = score.maximum(s, mul, base);
    st.ref = st.m == -INFINITY ? 0.f : st.m;
    st.look = __any(fabsf(st.m) >= AP_STEP);           // -infinity too
    if (st.look) settle();
    st.l = weights();
  } else {
    float sum = weights();
    if (st.look || __any(sum > AP_LOOK)) {
      // a row moves for its own sum only: its bits do not depend on its neighbours (nor on what stands in rows past the end)
      const bool own = ap_other_half(sum, true) > AP_LOOK || fabsf(st.m) >= AP_STEP;
      const float mx = score.maximum(s, mul, base);
      const float mn = own && mx > st.m + AP_TAU ? mx : st.m;
      st.ref = mn == -INFINITY ? 0.f : mn;
      const float alpha = __builtin_amdgcn_exp2f(st.m - st.ref);
      st.m = mn;
      st.l *= alpha;
#pragma unroll
      for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[d][r] *= alpha;
      st.look = __any(fabsf(st.m) >= AP_STEP);
      if (st.look) settle();
      sum = weights();
    }
    st.l += sum;
  }
}

// A whole tile of 32 keys: scores, weights, P V.
template <int DT, int D, bool BIAS, bool FIRST>
__device__ __forceinline__ void ap_tile(const ApScore& score, const char* sk, const char* sv, uint32_t krow, uint32_t kxor,
                                        uint32_t vrow, uint32_t vxor, int kt, const v4i (&qf)[D / 16], v16f (&acc)[D / 32], ApState& st) {
  constexpr int ROWB = 2 * D;
  v16f s[1];
#pragma unroll
  for (int r = 0; r < 16; ++r) s[0][r] = 0.f;
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk) s[0] = ap_mma<DT>::run(*reinterpret_cast<const v4i*>(sk + krow + (kxor ^ (kk << 5))), qf[kk], s[0]);
  uint32_t pk[1][8];
  ap_weights<DT, D, 1, BIAS, FIRST>(score, kt, s, acc, st, pk);
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const uint32_t* w = &pk[0][4 * t];
    const v4i pf = {(int)w[0], (int)w[1], (int)w[2], (int)w[3]};
#pragma unroll
    for (int d = 0; d < D / 32; ++d) {
      const char* a = sv + t * 16 * ROWB + vrow + ((d << 6) ^ vxor);
      const v8s vf = __builtin_shufflevector(__builtin_amdgcn_ds_read_tr16_b64_v4i16((ap_trptr_t)a),
                                             __builtin_amdgcn_ds_read_tr16_b64_v4i16((ap_trptr_t)(a + 4 * ROWB)), 0, 1, 2, 3, 4, 5, 6, 7);
      if (FIRST && t == 0) {
        v16f zero;
#pragma unroll
        for (int r = 0; r < 16; ++r) zero[r] = 0.f;
        acc[d] = ap_mma<DT>::run(__builtin_bit_cast(v4i, vf), pf, zero);
      } else acc[d] = ap_mma<DT>::run(__builtin_bit_cast(v4i, vf), pf, acc[d]);
    }
  }
}

// ---- 128 rows, 32 per wave; key tiles of 32 shared by the waves, two LDS stages, one barrier a tile ----
// What bounds it.  Long ranges: the matrix pipe at the clock that the power limit leaves (causal, 32 760 tokens, 12 heads of 128: 2.79
// to 2.86 ms, 1.15 to 1.18 PFLOP/s, 0.84 of a large library product on the same card; with the softmax arithmetic taken out 2.72 ms).  Short
// ranges: the latency of a workgroup's first loads and the vector instructions around the loop.  Hence tiles of 32 keys - three
// (D = 64: four) workgroups a CU instead of two: 226 keys under 50 960 rows of 12 heads 91 us (94 against 100 when tried), prompts
// of 1 to 512 tokens, 64 heads of 64, 35.2 (35.3 against 36.7 when tried), the long range 1 % slower - and pointers that step instead of
// addresses computed row by row (1250 -> 950 vector instructions a wave at 226 keys, 107 -> 100 us).
template <int DT, int D, bool BIAS>
__global__ __launch_bounds__(256, D == 128 ? 3 : 4) void attn_packed_tile_kernel(const ApParams p) {
  constexpr int BK = 32, ROWB = 2 * D, TILE = BK * ROWB, STAGE = 2 * TILE, PIECES = TILE / 4096, RPP = 1024 / ROWB, KK = D / 16, DB = D / 32;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int item = blockIdx.z * AP_GRID_Y + blockIdx.y, kvh = blockIdx.x;
  if (item >= p.n_items) return;
  const ApItem it = p.items[item];
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int x0 = 32 * wave, bn = 2 * p.R + 1 + 2 * AP_PAD;
  float* const lbias = reinterpret_cast<float*>(smem + STAGE + AP_ROWS * ROWB);       // stage 1 and behind: Q, at the end O
  const int drow = lane / (ROWB / 16), dchunk = lane & (ROWB / 16 - 1);

  // ---- Q: whole rows (memory likes full lines) into LDS from stage 1 on, until tile 1 comes; rows past the end are not
  //      read (zeros below, never stored).  One head per key head: the rows are evenly spaced, a bounds-checked buffer needs
  //      no comparison, and the permutation of a row's chunks has a period of PER groups ----
  char* const qstage = smem + STAGE + x0 * ROWB;
  constexpr int PER = D == 128 ? 4 : 2;
  static_assert(D == 128 || D == 64, "ap_kx of row RPP t + r is ap_kx of row RPP (t mod PER) + r");
  if (p.G == 1) {
    const uint16_t* const qhead = p.q + (int64_t)it.token * p.q_ts + (int64_t)kvh * p.q_hs;
    const uint32_t bytes = (uint32_t)((it.rows - 1) * 2 * p.q_ts + ROWB), row = (uint32_t)(2 * p.q_ts);
#pragma unroll
    for (int t = 0; t < 32 / RPP; ++t)
      ap_dma(qhead, bytes, qstage + t * 1024, (x0 + drow) * row + ((dchunk ^ ap_kx<D>(RPP * (t % PER) + drow)) << 4) + t * RPP * row);
  } else {
    const uint16_t* const qhead = p.q + (int64_t)it.token * p.q_ts + (int64_t)kvh * p.G * p.q_hs;
    ApRowWalk<D> w(p, it, x0 + drow, p.q_ts, p.q_hs);
#pragma unroll
    for (int t = 0; t < 32 / RPP; ++t, w.next()) {
      const int x = RPP * t + drow;
      if (x0 + x < it.rows) ap_dma_ptr(qhead + w.at + 8 * (dchunk ^ ap_kx<D>(x)), qstage + t * 1024);
    }
  }
  // ---- K, V: piece i of this wave is rows RPP (wave + 4 i) ..; rows past the range re-read the last one (finite, masked) ----
  const uint32_t r0 = RPP * wave + drow;
  const uint32_t koff = r0 * (uint32_t)(2 * p.k_ts) + ((dchunk ^ ap_kx<D>(r0)) << 4);      // the same permutation in every piece
  const uint32_t voff = r0 * (uint32_t)(2 * p.v_ts) + ((dchunk ^ ap_vx<D>(r0)) << 4);
  const uint16_t* const kbase = p.k + (int64_t)it.k_begin * p.k_ts + (int64_t)kvh * p.k_hs;
  const uint16_t* const vbase = p.v + (int64_t)it.k_begin * p.v_ts + (int64_t)kvh * p.v_hs;
  auto fetch = [&](int kt, int buf) {
    const int nv = min(it.key1 - kt, BK);
    const uint16_t* kp = kbase + (int64_t)kt * p.k_ts;
    const uint16_t* vp = vbase + (int64_t)kt * p.v_ts;
    const uint32_t kbytes = (uint32_t)((nv - 1) * 2 * p.k_ts + ROWB), vbytes = (uint32_t)((nv - 1) * 2 * p.v_ts + ROWB);
    char* st = smem + buf * STAGE + wave * 1024;
    if (nv == BK) {
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        ap_dma(kp, kbytes, st + i * 4096, koff + i * (uint32_t)(8 * RPP * p.k_ts));
        ap_dma(vp, vbytes, st + TILE + i * 4096, voff + i * (uint32_t)(8 * RPP * p.v_ts));
      }
    } else {
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        const uint32_t r = min((int)r0 + 4 * RPP * i, nv - 1);
        ap_dma(kp, kbytes, st + i * 4096, r * (uint32_t)(2 * p.k_ts) + ((dchunk ^ ap_kx<D>(r0)) << 4));
        ap_dma(vp, vbytes, st + TILE + i * 4096, r * (uint32_t)(2 * p.v_ts) + ((dchunk ^ ap_vx<D>(r0)) << 4));
      }
    }
  };
  // the item's last row sees most keys
  int q_last, h_last;
  ap_split(p, it, it.rows - 1, q_last, h_last);
  const int kend = p.causal ? min(it.key1, it.pos + q_last + 1) : it.key1;
  int kt = it.key0;
  if (kt < kend) fetch(kt, 0);
  if constexpr (BIAS) ap_load_bias<256>(p, kvh, bn, lbias);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  v4i qf[KK];                                                          // Q^T fragments: B operand, lane = row, 8 consecutive d each
  {
    const uint32_t r = lane & 31;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) qf[kk] = *reinterpret_cast<const v4i*>(qstage + r * ROWB + (((half ^ ap_kx<D>(r)) << 4) ^ (kk << 5)));
    if (x0 + 32 > it.rows) {         // what LDS held would send the whole wave after its maxima
      const int keep = x0 + (int)r < it.rows ? -1 : 0;
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) qf[kk] &= (v4i){keep, keep, keep, keep};
    }
  }
  __syncthreads();
  const ApScore score = ap_score<BIAS>(p, it, x0, lane, lbias, bn);
  const int wend = x0 < it.rows ? score.wmax : 0;

  // ---- fragment addresses ----
  const uint32_t kr = (lane & 19) | ((lane & 4) << 1) | ((lane & 8) >> 1);      // bits 2 and 3 of the row swapped
  const uint32_t krow = kr * ROWB, kxor = (half ^ ap_kx<D>(kr)) << 4;
  const uint32_t i16 = lane & 15;
  const uint32_t vkey = 8 * half + (i16 >> 2);
  const uint32_t vrow = vkey * ROWB + ((((lane >> 4) & 1) * 2 + ((i16 & 3) >> 1)) << 4) + (i16 & 1) * 8;
  const uint32_t vxor = ap_vx<D>(vkey) << 4;                                    // a multiple of 64: moves whole 32-d blocks

  v16f acc[DB];
  ApState st;
  auto tile = [&](auto first, int buf) {
    if (kt + BK < kend) fetch(kt + BK, buf ^ 1);
    if (kt < wend)
      ap_tile<DT, D, BIAS, decltype(first)::value>(score, smem + buf * STAGE, smem + buf * STAGE + TILE, krow, kxor, vrow, vxor, kt, qf, acc, st);
    // this tile's reads have returned and the next tile has landed
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __syncthreads();
    kt += BK;
  };
  if (kt >= wend) {                 // rows that see nothing
    st.m = -INFINITY; st.l = 0.f;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[d][r] = 0.f;
  }
  if (kt < kend) tile(std::true_type{}, 0);
  for (int buf = 1; kt < kend; buf ^= 1) tile(std::false_type{}, buf);
  if (x0 >= it.rows) return;        // no barrier behind this
  const float l = ap_other_half(st.l, false);

  // ---- results.  acc[d][r] is d = 32 d + 8 (r >> 2) + 4 half + (r & 3) of this lane's row ----
  const int x = x0 + (lane & 31);
  if (it.slot >= 0) {
    if (x >= it.rows) return;
    const int64_t pr = (int64_t)kvh * p.ws_rows + it.slot + x;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int r = 0; r < 16; r += 4)
        *reinterpret_cast<float4*>(p.po + pr * D + 32 * d + 2 * r + 4 * half) = make_float4(acc[d][r], acc[d][r + 1], acc[d][r + 2], acc[d][r + 3]);
    if (half == 0) { p.pml[pr * 2] = st.m; p.pml[pr * 2 + 1] = l; }
    return;
  }
  // through the wave's own 32 rows of LDS (every wave is done with the stages): whole rows go out
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  char* const ost = smem + STAGE + x0 * ROWB;
  const uint32_t r32 = lane & 31;
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int r = 8 * j;
      const uint32_t a0 = pack2<DT>(acc[d][r] * inv, acc[d][r + 1] * inv), a1 = pack2<DT>(acc[d][r + 2] * inv, acc[d][r + 3] * inv);
      const uint32_t b0 = pack2<DT>(acc[d][r + 4] * inv, acc[d][r + 5] * inv), b1 = pack2<DT>(acc[d][r + 6] * inv, acc[d][r + 7] * inv);
      const auto s0 = __builtin_amdgcn_permlane32_swap(a0, b0, false, false);
      const auto s1 = __builtin_amdgcn_permlane32_swap(a1, b1, false, false);
      *reinterpret_cast<uint4*>(ost + r32 * ROWB + (((4 * d + 2 * j + half) ^ ap_kx<D>(r32)) << 4)) = make_uint4(s0[0], s1[0], s0[1], s1[1]);
    }
  __builtin_amdgcn_wave_barrier();
  if (p.G == 1) {
    uint16_t* const ohead = p.o + (int64_t)it.token * p.o_ts + (int64_t)kvh * p.o_hs;
    const uint32_t bytes = (uint32_t)((it.rows - 1) * 2 * p.o_ts + ROWB), row = (uint32_t)(2 * p.o_ts);
#pragma unroll
    for (int t = 0; t < 32 / RPP; ++t) {
      const uint32_t y = RPP * (t % PER) + drow;
      const v4i v = *reinterpret_cast<const v4i*>(ost + (y + RPP * (t - t % PER)) * ROWB + ((dchunk ^ ap_kx<D>(y)) << 4));
      ap_store(ohead, bytes, v, (x0 + drow) * row + 16 * dchunk + t * RPP * row);
    }
  } else {
    uint16_t* const ohead = p.o + (int64_t)it.token * p.o_ts + (int64_t)kvh * p.G * p.o_hs + 8 * dchunk;
    ApRowWalk<D> w(p, it, x0 + drow, p.o_ts, p.o_hs);
#pragma unroll
    for (int t = 0; t < 32 / RPP; ++t, w.next()) {
      const uint32_t y = RPP * t + drow;
      const uint4 v = *reinterpret_cast<const uint4*>(ost + y * ROWB + ((dchunk ^ ap_kx<D>(y)) << 4));
      if (x0 + (int)y < it.rows) *reinterpret_cast<uint4*>(ohead + w.at) = v;
    }
  }
}

// The 16 transposing reads of a wave's V tile (8 KB), all in flight: vf[4 u + i] is the fragment at a[i] + 16 u rows.
template <int ROWB>
__device__ __forceinline__ void ap_read_v(const uint32_t (&a)[4], v4i (&vf)[8]) {
  v2i x[16];
  asm volatile(
      "ds_read_b64_tr_b16 %0, %16\n ds_read_b64_tr_b16 %1, %16 offset:%20\n ds_read_b64_tr_b16 %2, %17\n ds_read_b64_tr_b16 %3, %17 offset:%20\n"
      "ds_read_b64_tr_b16 %4, %18\n ds_read_b64_tr_b16 %5, %18 offset:%20\n ds_read_b64_tr_b16 %6, %19\n ds_read_b64_tr_b16 %7, %19 offset:%20\n"
      "ds_read_b64_tr_b16 %8, %16 offset:%21\n ds_read_b64_tr_b16 %9, %16 offset:%22\n ds_read_b64_tr_b16 %10, %17 offset:%21\n"
      "ds_read_b64_tr_b16 %11, %17 offset:%22\n ds_read_b64_tr_b16 %12, %18 offset:%21\n ds_read_b64_tr_b16 %13, %18 offset:%22\n"
      "ds_read_b64_tr_b16 %14, %19 offset:%21\n ds_read_b64_tr_b16 %15, %19 offset:%22\n s_waitcnt lgkmcnt(0)"
      : "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3]), "=&v"(x[4]), "=&v"(x[5]), "=&v"(x[6]), "=&v"(x[7]), "=&v"(x[8]), "=&v"(x[9]),
        "=&v"(x[10]), "=&v"(x[11]), "=&v"(x[12]), "=&v"(x[13]), "=&v"(x[14]), "=&v"(x[15])
      : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), "n"(4 * ROWB), "n"(16 * ROWB), "n"(20 * ROWB)
      : "memory");
#pragma unroll
  for (int i = 0; i < 8; ++i) vf[i] = v4i{x[2 * i][0], x[2 * i][1], x[2 * i + 1][0], x[2 * i + 1][1]};
}

// ---- up to 32 rows; the waves take different keys, each with a K and a V stage of its own, and join at the end ----
// What bounds it: memory, K and V once: 16 sequences of up to 32 760 keys, 40 heads of 128 over 8 key heads, 702 MB in 135 us, 5.2
// TB/s (a large copy moves 4.9).  One workgroup a CU with up to 128 KB in flight; 32 rows of the MFMA for G = 5 valid ones cost nothing
// beside that.  A wave fetches its next K tile once this one is in registers and its next V tile likewise, so that 16 KB hold what
// two stages did and eight waves fit where four did: a range of 777 keys of 12 heads 8.7 against 11.4 us.
#define AP_FEW_WAVES 8
template <int DT, int D, bool BIAS>
__global__ __launch_bounds__(64 * AP_FEW_WAVES, 1) void attn_packed_few_kernel(const ApParams p) {
  constexpr int NB = D == 128 ? 1 : 2, BK = 32 * NB;        // keys per tile
  constexpr int ROWB = 2 * D, TILE = BK * ROWB, STAGE = 2 * TILE, PIECES = TILE / 1024, RPP = 1024 / ROWB, KK = D / 16, DB = D / 32;
  constexpr int NW = AP_FEW_WAVES;
  static_assert(TILE == 8192 && PIECES == 8, "the waits below count pieces");
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int item = blockIdx.z * AP_GRID_Y + blockIdx.y, kvh = blockIdx.x;
  if (item >= p.n_items) return;
  const ApItem it = p.items[item];
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int bn = 2 * p.R + 1 + 2 * AP_PAD;
  float* const lbias = reinterpret_cast<float*>(smem + NW * STAGE);
  v4i qf[KK];
  {
    int q, h;
    ap_split(p, it, min(lane & 31, it.rows - 1), q, h);
    const uint16_t* qp = p.q + (int64_t)(it.token + q) * p.q_ts + (int64_t)(kvh * p.G + h) * p.q_hs + 8 * half;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) qf[kk] = *reinterpret_cast<const v4i*>(qp + 16 * kk);
  }
  if constexpr (BIAS) {
    ap_load_bias<64 * NW>(p, kvh, bn, lbias);
    __syncthreads();
  }
  const ApScore score = ap_score<BIAS>(p, it, 0, lane, lbias, bn);
  const int kend = score.wmax;

  const int drow = lane / (ROWB / 16), dchunk = lane & (ROWB / 16 - 1);
  char* const stage = smem + wave * STAGE;
  // a tile of K (V) from key kt; rows past the range re-read the last one (finite, masked)
  const uint16_t* const kbase = p.k + (int64_t)it.k_begin * p.k_ts + (int64_t)kvh * p.k_hs;
  const uint16_t* const vbase = p.v + (int64_t)it.k_begin * p.v_ts + (int64_t)kvh * p.v_hs;
  auto fetch = [&](const uint16_t* b0, int64_t ts, char* dst, auto isv, int kt) {
    const int nv = min(it.key1 - kt, BK);
    const uint16_t* b = b0 + (int64_t)kt * ts;
    const uint32_t bytes = (uint32_t)((nv - 1) * 2 * ts + ROWB);
#pragma unroll
    for (int t = 0; t < PIECES; ++t) {
      const uint32_t r = RPP * t + drow, rc = min((int)r, nv - 1), x = decltype(isv)::value ? ap_vx<D>(r) : ap_kx<D>(r);
      ap_dma(b, bytes, dst + t * 1024, rc * (uint32_t)(2 * ts) + ((dchunk ^ x) << 4));
    }
    asm volatile("" ::: "memory");       // the waits count these in order
  };
  const uint32_t kr = (lane & 19) | ((lane & 4) << 1) | ((lane & 8) >> 1);      // bits 2 and 3 of the row swapped
  const uint32_t krow = kr * ROWB, kxor = (half ^ ap_kx<D>(kr)) << 4;
  const uint32_t i16 = lane & 15;
  const uint32_t vkey = 8 * half + (i16 >> 2);
  const uint32_t vrow = vkey * ROWB + ((((lane >> 4) & 1) * 2 + ((i16 & 3) >> 1)) << 4) + (i16 & 1) * 8;
  const uint32_t vxor = ap_vx<D>(vkey) << 4;
  uint32_t va[4];                        // fragment i: d block i % DB, 32 keys further for i >= DB
#pragma unroll
  for (int i = 0; i < 4; ++i)
    va[i] = (uint32_t)(uintptr_t)(ap_trptr_t)(stage + TILE) + vrow + (((i % DB) << 6) ^ vxor) + (i / DB) * 32 * ROWB;

  v16f acc[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[d][r] = 0.f;
  ApState st = {-INFINITY, 0.f, 0.f, true};
  int kt = it.key0 + wave * BK;
  if (kt < kend) {
    fetch(kbase, p.k_ts, stage, std::false_type{}, kt);
    fetch(vbase, p.v_ts, stage + TILE, std::true_type{}, kt);
  }
  for (; kt < kend; kt += NW * BK) {
    const bool more = kt + NW * BK < kend;
    asm volatile("s_waitcnt vmcnt(8)" ::: "memory");                  // K has landed (V's 8 pieces came after it)
    v4i kf[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) kf[i] = *reinterpret_cast<const v4i*>(stage + (i / KK) * 32 * ROWB + krow + (kxor ^ ((i % KK) << 5)));
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");                // and has been read: its stage is free (it is this wave's own)
    if (more) fetch(kbase, p.k_ts, stage, std::false_type{}, kt + NW * BK);
    v16f s[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[b][r] = 0.f;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk)
#pragma unroll
      for (int b = 0; b < NB; ++b) s[b] = ap_mma<DT>::run(kf[b * KK + kk], qf[kk], s[b]);
    uint32_t pk[NB][8];
    ap_weights<DT, D, NB, BIAS, false>(score, kt, s, acc, st, pk);
    if (more) asm volatile("s_waitcnt vmcnt(8)" ::: "memory");        // V has landed
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    v4i vf[8];
    ap_read_v<ROWB>(va, vf);
    if (more) fetch(vbase, p.v_ts, stage + TILE, std::true_type{}, kt + NW * BK);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int t = (i >> 2) + 2 * ((i & 3) / DB);
      const uint32_t* w = &pk[t >> 1][4 * (t & 1)];
      acc[i % DB] = ap_mma<DT>::run(vf[i], v4i{(int)w[0], (int)w[1], (int)w[2], (int)w[3]}, acc[i % DB]);
    }
  }
  const float l = ap_other_half(st.l, false), m = st.m;

  // acc[d][r] is d = 32 d + 8 (r >> 2) + 4 half + (r & 3) of this lane's row
  // ---- join the waves through LDS ----
  constexpr int LD = D + 4;
  float* jo = reinterpret_cast<float*>(smem);                 // [NW][32][LD]
  float* jm = jo + NW * 32 * LD;                              // [NW][32][2]
  __syncthreads();
  const int row = lane & 31;
  if (row < it.rows) {
    float* mo = jo + (wave * 32 + row) * LD;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int r = 0; r < 16; r += 4)
        *reinterpret_cast<float4*>(mo + 32 * d + 2 * r + 4 * half) = make_float4(acc[d][r], acc[d][r + 1], acc[d][r + 2], acc[d][r + 3]);
    if (half == 0) { jm[(wave * 32 + row) * 2] = m; jm[(wave * 32 + row) * 2 + 1] = l; }
  }
  __syncthreads();
  constexpr int W = D / (2 * NW);                             // d per thread
  const int jr = tid / (2 * NW), d0 = (tid % (2 * NW)) * W;
  if (jr < it.rows) {
    float mm = -INFINITY, ll = 0.f, oo[W];
#pragma unroll
    for (int w = 0; w < NW; ++w) mm = fmaxf(mm, jm[(w * 32 + jr) * 2]);
    const float mr = mm == -INFINITY ? 0.f : mm;
#pragma unroll
    for (int e = 0; e < W; ++e) oo[e] = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float a = __builtin_amdgcn_exp2f(jm[(w * 32 + jr) * 2] - mr);
      ll += a * jm[(w * 32 + jr) * 2 + 1];
#pragma unroll
      for (int e = 0; e < W; e += 4) {
        const float4 x = *reinterpret_cast<const float4*>(jo + (w * 32 + jr) * LD + d0 + e);
        oo[e] += a * x.x; oo[e + 1] += a * x.y; oo[e + 2] += a * x.z; oo[e + 3] += a * x.w;
      }
    }
    if (it.slot >= 0) {
      const int64_t pr = (int64_t)kvh * p.ws_rows + it.slot + jr;
#pragma unroll
      for (int e = 0; e < W; e += 4)
        *reinterpret_cast<float4*>(p.po + pr * D + d0 + e) = make_float4(oo[e], oo[e + 1], oo[e + 2], oo[e + 3]);
      if (d0 == 0) { p.pml[pr * 2] = mm; p.pml[pr * 2 + 1] = ll; }
    } else {
      const float inv = ll == 0.f ? 0.f : 1.0f / ll;
      int q2, g2;
      ap_split(p, it, jr, q2, g2);
      uint16_t* op = p.o + (int64_t)(it.token + q2) * p.o_ts + (int64_t)(kvh * p.G + g2) * p.o_hs + d0;
#pragma unroll
      for (int e = 0; e < W; e += 4)
        *reinterpret_cast<uint2*>(op + e) = make_uint2(pack2<DT>(oo[e] * inv, oo[e + 1] * inv), pack2<DT>(oo[e + 2] * inv, oo[e + 3] * inv));
    }
  }
}

// One wave per row: the parts of a row, weighted by exp2(maximum - common maximum).  Lane i knows part i's maximum and sum; the
// parts themselves are read eight at a time.  What bounds it: memory latency; one after the other 25 parts took 12.8 us, so 5.1.
template <int DT, int D>
__global__ __launch_bounds__(256) void attn_packed_join_kernel(const ApParams p, const ApJoin* joins) {
  constexpr int E = D / 64;
  const ApJoin j = joins[blockIdx.x];
  const int kvh = blockIdx.y, lane = threadIdx.x & 63;
  const int r = blockIdx.z * 4 + (threadIdx.x >> 6);
  if (r >= j.rows) return;
  const int64_t base = (int64_t)kvh * p.ws_rows + j.slot + r;
  float mm = -INFINITY;
  for (int s = lane; s < j.splits; s += 64) mm = fmaxf(mm, p.pml[(base + (int64_t)s * j.tile_rows) * 2]);
  mm = wave_max(mm);
  const float mr = mm == -INFINITY ? 0.f : mm;
  float ll = 0.f, o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.f;
  for (int s0 = 0; s0 < j.splits; s0 += 64) {
    const int n = min(64, j.splits - s0);
    float a = 0.f;
    if (lane < n) {
      const float2 ml = *reinterpret_cast<const float2*>(p.pml + (base + (int64_t)(s0 + lane) * j.tile_rows) * 2);
      a = __builtin_amdgcn_exp2f(ml.x - mr);
      ll += a * ml.y;
    }
    for (int s = 0; s < n; s += 8) {
      float v[8][E];
#pragma unroll
      for (int u = 0; u < 8; ++u)
#pragma unroll
        for (int e = 0; e < E; ++e) v[u][e] = p.po[(base + (int64_t)(s0 + min(s + u, n - 1)) * j.tile_rows) * D + lane * E + e];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const float w = s + u < n ? __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(a), s + u)) : 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (s + u < n) o[e] += w * v[u][e];
      }
    }
  }
  ll = wave_sum(ll);
  const float inv = ll == 0.f ? 0.f : 1.0f / ll;
  const int y = j.head0 + r, qi = p.G > 1 ? (int)__umulhi((uint32_t)y, p.gmagic) : y, g = y - qi * p.G;
  uint16_t* op = p.o + (int64_t)(j.token + qi) * p.o_ts + (int64_t)(kvh * p.G + g) * p.o_hs + lane * E;
  if constexpr (E == 2) *reinterpret_cast<uint32_t*>(op) = pack2<DT>(o[0] * inv, o[1] * inv);
  else *op = (uint16_t)pack2<DT>(o[0] * inv, 0.f);
}

// ---- the plan: which workgroup does what (host) --------------------------------------------------------------------
// Table of 8-word records: items (all for one of the two kernels), then joins.  counts = {tile items, few items, joins, partial rows,
// query tokens, key tokens}; one of the first two is 0.

// Keys a few workgroup takes.  One has a CU to itself and needs 2.5 us beside its keys; all 256 read 39 keys a us each (D = 128), one
// alone 150.  W keys in parts of L take W / (39 * 256) + 2.5 W / (256 L) and, while the last ones run without the others, L / 150:
// least at L = sqrt(1.5 W) (D = 64: sqrt(3 W)).  Or all run at once, if as many as there are CUs share W evenly.
static int64_t ap_few_chunk(const std::vector<int64_t>& keys, int64_t total, int64_t kv_heads) {
  const int64_t w = total * kv_heads;
  const auto up = [](int64_t x) { return td_cdiv(std::max<int64_t>(x, 256), 128) * 128; };
  const int64_t many = up((int64_t)std::sqrt(2.0 * (double)w));
  // Not split: up to 1024 keys, where a workgroup is done before a second launch and the join would be (5 us), or little more than a part.
  const int64_t longest = keys.empty() ? 0 : *std::max_element(keys.begin(), keys.end());
  if (longest <= std::max<int64_t>(1024, many + many / 2)) return up(longest);
  if ((int64_t)keys.size() * kv_heads > 256) return many;
  for (int64_t one = up(w / 256);; one += up(one / 32) - 128) {
    one = std::min(one, up(longest));
    int64_t n = 0;
    for (int64_t x : keys) n += kv_heads * std::max<int64_t>(1, td_cdiv(x, one));
    if (n <= 256 && (one <= many / 4 * 7 || (n >= 224 && w >= n * one / 8 * 7))) return one;
    if (n <= 256 || one >= longest) return many;
  }
}

extern "C" int td_attn_packed_plan(const int64_t* lens_q, const int64_t* lens_k, int64_t nseq, int heads, int kv_heads, int causal,
                                   int32_t* table, int64_t capacity, int64_t* counts) {
  TD_REQUIRE(lens_q && lens_k && counts && nseq >= 0, TD_ERR_INVALID, "td_attn_packed_plan: null pointer or %lld sequences", (long long)nseq);
  TD_REQUIRE(kv_heads > 0 && heads > 0 && heads % kv_heads == 0, TD_ERR_INVALID, "td_attn_packed_plan: %d heads over %d key heads", heads, kv_heads);
  const int64_t G = heads / kv_heads, MAXT = 1ll << 30;
  int64_t tq = 0, tk = 0;
  for (int64_t s = 0; s < nseq; ++s) {
    TD_REQUIRE(lens_q[s] >= 0 && lens_k[s] >= 0 && lens_q[s] <= MAXT && lens_k[s] <= MAXT, TD_ERR_INVALID,
               "td_attn_packed_plan: sequence %lld has lengths %lld, %lld", (long long)s, (long long)lens_q[s], (long long)lens_k[s]);
    tq += lens_q[s]; tk += lens_k[s];
    TD_REQUIRE(tq <= MAXT && tk <= MAXT && tq * G <= MAXT, TD_ERR_UNSUPPORTED, "td_attn_packed_plan: more than 2^30 rows");
  }
  try {
    struct Work { ApItem it; int64_t keys; };
    std::vector<Work> work;
    std::vector<ApJoin> joins;
    // One kernel for the whole batch (a second launch costs more than the better kernel saves: a prompt of 512 tokens and 8 tokens over
    // 900 keys each, 40 heads of 128 over 8, 21 us by the tile kernel, 28 by both; 8000 keys 58 against 75).
    bool few = true;
    int64_t n_few = 0, few_longest = 0;
    for (int64_t s = 0; s < nseq; ++s) {
      few &= lens_q[s] * G <= AP_FEW;
      if (lens_q[s] == 0) continue;
      n_few += lens_k[s] > AP_FEW_KEYS;
      few_longest = std::max(few_longest, lens_k[s]);
    }
    few &= few_longest > (n_few * kv_heads > 256 ? AP_MANY_KEYS : AP_FEW_KEYS);
    const int64_t tr = few ? AP_FEW : AP_ROWS;
    // pass 0 counts the keys, pass 1 emits items of at most `chunk` keys
    std::vector<int64_t> ranges;
    int64_t chunk = 0, total = 0, ws_rows = 0;
    for (int pass = 0; pass < 2; ++pass) {
      int64_t q0 = 0, k0 = 0;
      for (int64_t s = 0; s < nseq; ++s) {
        const int64_t ql = lens_q[s], kl = lens_k[s], rows = ql * G;
        for (int64_t r0 = 0; r0 < rows; r0 += tr) {
          const int64_t last = std::min(r0 + tr, rows) - 1;
          const int64_t end = causal ? std::max<int64_t>(0, std::min(kl, last / G + kl - ql + 1)) : kl;
          if (pass == 0) {
            total += end;
            if (few) ranges.push_back(end);
            continue;
          }
          int64_t per = chunk;               // few: the rest of a range makes a short part, which runs last
          if (!few) per = td_cdiv(td_cdiv(std::max<int64_t>(end, 1), std::max<int64_t>(1, td_cdiv(end, per))), 64) * 64;
          const int64_t n = std::max<int64_t>(1, td_cdiv(end, per));
          const int32_t token = (int32_t)(q0 + r0 / G), head0 = (int32_t)(r0 % G), nr = (int32_t)(last - r0 + 1), pos = (int32_t)(r0 / G + kl - ql);
          if (n > 1) joins.push_back({token, head0, nr, (int32_t)ws_rows, (int32_t)n, (int32_t)tr, 0, 0});
          for (int64_t i = 0; i < n; ++i) {
            const int64_t a = i * per, b = std::min(end, a + per);
            work.push_back({{token, head0, nr, pos, (int32_t)k0, (int32_t)a, (int32_t)b, n > 1 ? (int32_t)(ws_rows + i * tr) : -1}, b - a});
          }
          if (n > 1) ws_rows += n * tr;
          TD_REQUIRE(ws_rows <= MAXT, TD_ERR_UNSUPPORTED, "td_attn_packed_plan: more than 2^30 partial rows");
        }
        q0 += ql; k0 += kl;
      }
      if (pass == 0) {
        // A tile range is cut when it is longer than one of 512 even shares of all keys; a part is at least 512 keys, below which writing
        // and joining partials costs more than it saves.  The chip holds more workgroups (256 CUs, three or for D = 64 four each), but
        // shares for 768 (1024) of them are slower, as more partials are written and joined: causal, 10 heads of 128 over 2,
        // 4000 tokens 65 us against 70 (72), 8000 175 against 190 (185); 40 over 8, 4000 tokens 164 against 180 (188).
        chunk = few ? ap_few_chunk(ranges, total, kv_heads) : std::max<int64_t>(512, td_cdiv(total * kv_heads, 512));
      }
    }
    // longest first: the short ones fill the tail
    std::stable_sort(work.begin(), work.end(), [](const Work& a, const Work& b) { return a.keys > b.keys; });
    counts[few ? 1 : 0] = (int64_t)work.size(); counts[few ? 0 : 1] = 0; counts[2] = (int64_t)joins.size();
    counts[3] = ws_rows; counts[4] = tq; counts[5] = tk;
    const int64_t n = counts[0] + counts[1] + counts[2];
    if (table) {
      TD_REQUIRE(capacity >= n, TD_ERR_INVALID, "td_attn_packed_plan: table of %lld records, %lld needed", (long long)capacity, (long long)n);
      ApItem* t = reinterpret_cast<ApItem*>(table);
      for (auto& x : work) *t++ = x.it;
      for (auto& j : joins) *reinterpret_cast<ApJoin*>(t++) = j;
    }
  } catch (const std::bad_alloc&) {
    td_set_error("td_attn_packed_plan: out of host memory");
    return TD_ERR_INVALID;
  }
  return TD_OK;
}

template <int DT, int D, bool FEW, bool BIAS>
static void ap_launch(const ApParams& p, int64_t n, int bias_bytes, hipStream_t st) {
  static std::atomic<uint64_t> mask{0};
  // a stage of K + V and the rows; few: 16 KB for each wave, at the end the waves' sums, maxima and rows over them
  constexpr int tiles = FEW ? AP_FEW_WAVES * 16384 : (64 + AP_ROWS) * 2 * D, join = FEW ? AP_FEW_WAVES * 32 * (D + 4 + 2) * 4 : 0;
  const auto kernel = FEW ? attn_packed_few_kernel<DT, D, BIAS> : attn_packed_tile_kernel<DT, D, BIAS>;
  td_ensure_dyn_lds((const void*)kernel, std::max(tiles + 32768, join), mask);
  const dim3 grid((unsigned)p.Hkv, (unsigned)std::min<int64_t>(n, AP_GRID_Y), (unsigned)td_cdiv(n, AP_GRID_Y));
  kernel<<<grid, FEW ? 64 * AP_FEW_WAVES : 256, std::max(tiles + bias_bytes, join), st>>>(p);
}

extern "C" int td_attn_packed(const void* q, const void* k, const void* v, void* o, const int64_t* strides, int dtype, int heads, int kv_heads,
                              int head_dim, float scale, int causal, const float* bias, int bias_range, const int32_t* table,
                              const int64_t* counts, float* ws, td_stream_t stream) {
  TD_REQUIRE(q && o && counts && table && strides, TD_ERR_INVALID, "td_attn_packed: null pointer");
  TD_REQUIRE(dtype == TD_BF16 || dtype == TD_F16, TD_ERR_UNSUPPORTED, "td_attn_packed: dtype %d", dtype);
  TD_REQUIRE(head_dim == 64 || head_dim == 128, TD_ERR_UNSUPPORTED, "td_attn_packed: head_dim = %d (64 or 128)", head_dim);
  TD_REQUIRE(kv_heads > 0 && heads > 0 && heads % kv_heads == 0, TD_ERR_INVALID, "td_attn_packed: %d heads over %d key heads", heads, kv_heads);
  for (int i = 0; i < 8; ++i)
    TD_REQUIRE(strides[i] >= 0 && strides[i] % 8 == 0, TD_ERR_UNSUPPORTED, "td_attn_packed: stride %lld (a multiple of 8 elements)", (long long)strides[i]);
  for (int i = 0; i < 8; i += 2)
    TD_REQUIRE(strides[i] < (1 << 24), TD_ERR_UNSUPPORTED, "td_attn_packed: token stride %lld (less than 2^24 elements)", (long long)strides[i]);
  TD_REQUIRE((((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)o | (uintptr_t)ws) & 15) == 0, TD_ERR_UNSUPPORTED,
             "td_attn_packed: pointers must be 16-byte aligned");
  TD_REQUIRE(counts[4] <= 1 || strides[6] >= head_dim, TD_ERR_INVALID, "td_attn_packed: the tokens of o overlap");
  TD_REQUIRE(scale > 0.f && scale <= 1e38f, TD_ERR_INVALID, "td_attn_packed: scale must be positive, at most 1e38");
  const int64_t nt = counts[0], nf = counts[1], nj = counts[2], wr = counts[3];
  TD_REQUIRE(nt >= 0 && nf >= 0 && (nt == 0 || nf == 0) && nj >= 0 && wr >= 0 && (nj == 0 || ws), TD_ERR_INVALID, "td_attn_packed: counts / workspace");
  TD_REQUIRE(counts[5] == 0 || (k && v), TD_ERR_INVALID, "td_attn_packed: null keys or values");
  TD_REQUIRE(nt < (1ll << 31) && nf < (1ll << 31) && nj < (1ll << 31) && kv_heads <= 65535, TD_ERR_UNSUPPORTED,
             "td_attn_packed: too many workgroups");
  const int G = heads / kv_heads;
  TD_REQUIRE(G <= 16384, TD_ERR_UNSUPPORTED, "td_attn_packed: %d heads share a key head", G);
  int bias_bytes = 0;
  if (bias) {
    TD_REQUIRE(bias_range >= 0 && bias_range < 8192 && (int64_t)G * (2 * bias_range + 1 + 2 * AP_PAD) * 4 <= 32768, TD_ERR_UNSUPPORTED,
               "td_attn_packed: bias of range %d for %d heads per key head exceeds 32 KB", bias_range, G);
    bias_bytes = G * (2 * bias_range + 1 + 2 * AP_PAD) * 4;
  }
  ApParams p;
  p.q = (const uint16_t*)q; p.k = (const uint16_t*)k; p.v = (const uint16_t*)v; p.o = (uint16_t*)o;
  p.q_ts = strides[0]; p.q_hs = strides[1]; p.k_ts = strides[2]; p.k_hs = strides[3];
  p.v_ts = strides[4]; p.v_hs = strides[5]; p.o_ts = strides[6]; p.o_hs = strides[7];
  if (counts[4] <= 1) p.o_ts = head_dim;         // the rows past a sequence's end lie behind the end of its last one
  p.bias = bias; p.R = bias_range;
  p.po = ws; p.pml = ws ? ws + (int64_t)kv_heads * wr * head_dim : nullptr; p.ws_rows = wr;
  p.Hkv = kv_heads; p.G = G; p.causal = causal ? 1 : 0;
  p.gmagic = G > 1 ? (uint32_t)(((1ull << 32) + G - 1) / G) : 0;
  p.c = scale * 1.4426950408889634f;
  hipStream_t st = (hipStream_t)stream;
  const int64_t n = nt + nf;
  p.items = reinterpret_cast<const ApItem*>(table);
  p.n_items = (int)n;
  if (n == 0) return TD_OK;
#define AP_GO2(DT_, D_, F_) { if (bias) ap_launch<DT_, D_, F_, true>(p, n, bias_bytes, st); else ap_launch<DT_, D_, F_, false>(p, n, 0, st); }
#define AP_GO1(DT_, D_) { if (nf > 0) AP_GO2(DT_, D_, true) else AP_GO2(DT_, D_, false) }
  if (dtype == TD_BF16) { if (head_dim == 64) AP_GO1(TD_BF16, 64) else AP_GO1(TD_BF16, 128) }
  else { if (head_dim == 64) AP_GO1(TD_F16, 64) else AP_GO1(TD_F16, 128) }
#undef AP_GO1
#undef AP_GO2
  TD_CHECK_LAUNCH();
  if (nj > 0) {
    const ApJoin* joins = reinterpret_cast<const ApJoin*>(table) + n;
    const dim3 grid((unsigned)nj, (unsigned)kv_heads, (nt > 0 ? AP_ROWS : AP_FEW) / 4);
    if (dtype == TD_BF16) { if (head_dim == 64) attn_packed_join_kernel<TD_BF16, 64><<<grid, 256, 0, st>>>(p, joins); else attn_packed_join_kernel<TD_BF16, 128><<<grid, 256, 0, st>>>(p, joins); }
    else { if (head_dim == 64) attn_packed_join_kernel<TD_F16, 64><<<grid, 256, 0, st>>>(p, joins); else attn_packed_join_kernel<TD_F16, 128><<<grid, 256, 0, st>>>(p, joins); }
    TD_CHECK_LAUNCH();
  }
  return TD_OK;
}
