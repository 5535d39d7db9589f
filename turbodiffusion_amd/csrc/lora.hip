// Low-rank adapters of many requests beside a shared projection:
//
//     out[r] = y[r] + s_i B_i (A_i x[r]),    i = the adapter of row r's request;  rows without one: out[r] = y[r]
//
// x [rows, K], y / out [rows, N], A_i [rank_i, K], B_i [N, rank_i], 16-bit.  The rows are taken adapter by adapter (a permutation
// made by the plan), in tiles of 64 of one adapter, so an adapter is read for all of its rows at once however its requests lie.
//
//   shrink   S = A_i x:  fp32, MFMA 16x16x32 straight from global memory (x streams; A_i comes from L2).
//            Many tiles: a wave owns 16 rows.  Few tiles: the four waves of a workgroup share 16 rows and split K, and K is split
//            over workgroups too; expand adds the parts in order.
//   expand   out = y + B_i (s_i S): S is scaled in fp32 and rounded once to the operands' type (half a step of the update only:
//            it stays below the rounding of the output wherever the update is not many times larger than the output itself).
//            A lane ends with 8 consecutive columns of one row: 16-byte reads of y and writes of out, 64 bytes of a row together.
// Memory-bound: y and out dominate, then x; 2 rank flops per byte of them.
#include "td_common.h"
#include <algorithm>
#include <new>
#include <vector>

#define LR_TILE 64
#define LR_MAX_RANK 256

struct LoraTile { int32_t perm0, rows, adapter, pad; };
struct LoraAdapter { int64_t a_off, b_off; int32_t rank8; float scale; };   // offsets in elements; rank rounded up to 8 (zero rows / columns)

struct LoraParams {
  const uint16_t *x, *y; uint16_t* out;
  int64_t ldx, ldy, ldo;
  const uint16_t* bank; const LoraAdapter* adapters;
  const LoraTile* tiles; const int32_t* perm;
  float* s;                 // [splits][rows][RS]
  int64_t rows, K, N;
  int splits, steps;        // K splits over workgroups, K steps of 32 per split
  int ntile;                // columns per workgroup of expand
};

template <int DT> struct lr_mma;
template <> struct lr_mma<TD_F16> {
  __device__ static __forceinline__ v4f run(v4i a, v4i b, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
  }
};
template <> struct lr_mma<TD_BF16> {
  __device__ static __forceinline__ v4f run(v4i a, v4i b, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
  }
};

// RJ: 16-rank blocks of the largest adapter; KS: the waves split K
template <int DT, int RJ, bool KS>
__global__ __launch_bounds__(256) void lora_shrink_kernel(const LoraParams p) {
  constexpr int RS = 16 * RJ;
  const int lane = threadIdx.x & 63, l16 = lane & 15, lq = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const LoraTile t = p.tiles[KS ? blockIdx.x >> 2 : blockIdx.x];
  const int group = KS ? (blockIdx.x & 3) : wave;
  if (16 * group >= t.rows) return;                               // KS: the whole workgroup
  const LoraAdapter ad = p.adapters[t.adapter];
  const int prow = t.perm0 + min(16 * group + l16, t.rows - 1);   // rows past the tile repeat its last one
  const uint16_t* xp = p.x + (int64_t)p.perm[prow] * p.ldx + 8 * lq;
  const uint16_t* ap = p.bank + ad.a_off + (int64_t)l16 * p.K + 8 * lq;
  const int nsteps = (int)((p.K + 31) / 32);
  int s0 = blockIdx.y * p.steps, s1 = min(nsteps, s0 + p.steps);
  if constexpr (KS) {
    const int per = (p.steps + 3) / 4;
    s0 += wave * per;
    s1 = min(s1, s0 + per);
  }
  v4f acc[RJ];
#pragma unroll
  for (int j = 0; j < RJ; ++j) acc[j] = (v4f){0.f, 0.f, 0.f, 0.f};
  const v4i zero = {0, 0, 0, 0};
#pragma unroll 4
  for (int s = s0; s < s1; ++s) {
    const int64_t k = 32 * (int64_t)s;
    const bool in = k + 8 * lq < p.K;
    const v4i xf = in ? *reinterpret_cast<const v4i*>(xp + k) : zero;
#pragma unroll
    for (int j = 0; j < RJ; ++j) {
      if (16 * j < ad.rank8) {
        const v4i af = in && 16 * j + l16 < ad.rank8 ? *reinterpret_cast<const v4i*>(ap + (int64_t)(16 * j) * p.K + k) : zero;
        acc[j] = lr_mma<DT>::run(xf, af, acc[j]);
      }
    }
  }
  // acc[j][r] is row 4 lq + r, rank 16 j + l16
  float* sp = p.s + ((int64_t)blockIdx.y * p.rows + t.perm0 + 16 * group) * RS;
  const int nr = min(16, t.rows - 16 * group);
  if constexpr (KS) {
    __shared__ float red[3][16 * RS];
    if (wave > 0) {
#pragma unroll
      for (int j = 0; j < RJ; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) red[wave - 1][(4 * lq + r) * RS + 16 * j + l16] = acc[j][r];
    }
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int j = 0; j < RJ; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int w = 0; w < 3; ++w) acc[j][r] += red[w][(4 * lq + r) * RS + 16 * j + l16];
  }
#pragma unroll
  for (int j = 0; j < RJ; ++j)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (4 * lq + r < nr) sp[(4 * lq + r) * RS + 16 * j + l16] = acc[j][r];
}

template <int DT, int RJ>
__global__ __launch_bounds__(256) void lora_expand_kernel(const LoraParams p) {
  constexpr int RS = 16 * RJ, KK = (RJ + 1) / 2;
  const int lane = threadIdx.x & 63, l16 = lane & 15, lq = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const LoraTile t = p.tiles[blockIdx.x];
  const int64_t n0 = (int64_t)blockIdx.y * p.ntile, n1 = min(p.N, n0 + p.ntile);
  if (t.adapter < 0) {            // rows without an adapter: copy
    for (int r = wave; r < t.rows; r += 4) {
      const int64_t row = p.perm[t.perm0 + r];
      for (int64_t n = n0 + 8 * lane; n < n1; n += 512)
        *reinterpret_cast<uint4*>(p.out + row * p.ldo + n) = *reinterpret_cast<const uint4*>(p.y + row * p.ldy + n);
    }
    return;
  }
  const LoraAdapter ad = p.adapters[t.adapter];
  const v4i zero = {0, 0, 0, 0};
  // S fragments: B operand, lane = row l16 of group g, 8 ranks from 32 kk + 8 lq
  v4i sf[4][KK];
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    if (16 * g < t.rows) {
      const int pr = t.perm0 + min(16 * g + l16, t.rows - 1);
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        const int r0 = 32 * kk + 8 * lq;
        if (r0 < ad.rank8) {
          float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
          for (int s = 0; s < p.splits; ++s) {
            const float* sp = p.s + ((int64_t)s * p.rows + pr) * RS + r0;
            const float4 a = *reinterpret_cast<const float4*>(sp), b = *reinterpret_cast<const float4*>(sp + 4);
            f[0] += a.x; f[1] += a.y; f[2] += a.z; f[3] += a.w; f[4] += b.x; f[5] += b.y; f[6] += b.z; f[7] += b.w;
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) f[e] *= ad.scale;
          sf[g][kk] = __builtin_bit_cast(v4i, pack8<DT>(f));
        } else sf[g][kk] = zero;
      }
    }
  }
  int64_t yo[4], oo[4];
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const int64_t row = p.perm[t.perm0 + min(16 * g + l16, t.rows - 1)];
    yo[g] = row * p.ldy + 8 * lq;
    oo[g] = row * p.ldo + 8 * lq;
  }
  const int nl = 8 * (l16 >> 2) + (l16 & 3);      // A operand row -> column: lane ends with 8 consecutive columns
  for (int64_t n = n0 + 32 * wave; n < n1; n += 128) {
    v4f acc[4][2];
#pragma unroll
    for (int g = 0; g < 4; ++g) acc[g][0] = acc[g][1] = (v4f){0.f, 0.f, 0.f, 0.f};
    v4i bf[2][KK];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const int64_t nn = n + nl + 4 * b;
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        const int r0 = 32 * kk + 8 * lq;
        bf[b][kk] = nn < n1 && r0 < ad.rank8 ? *reinterpret_cast<const v4i*>(p.bank + ad.b_off + nn * ad.rank8 + r0) : zero;
      }
    }
    const bool in = n + 8 * lq < n1;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      if (16 * g < t.rows) {
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
          if (32 * kk < ad.rank8) {
            acc[g][0] = lr_mma<DT>::run(bf[0][kk], sf[g][kk], acc[g][0]);
            acc[g][1] = lr_mma<DT>::run(bf[1][kk], sf[g][kk], acc[g][1]);
          }
        }
        if (in && 16 * g + l16 < t.rows) {
          float f[8];
          unpack8<DT>(*reinterpret_cast<const uint4*>(p.y + yo[g] + n), f);
#pragma unroll
          for (int e = 0; e < 8; ++e) f[e] += acc[g][e >> 2][e & 3];
          *reinterpret_cast<uint4*>(p.out + oo[g] + n) = pack8<DT>(f);
        }
      }
    }
  }
}

// ---- the plan (host): rows by adapter, tiles of up to 64 of one adapter, rows without one last --------------------------
// counts = {tiles with an adapter, tiles without, rows, rows with an adapter, largest id + 1}; table = tiles (4 words each), then
// the row permutation
extern "C" int td_lora_plan(const int64_t* lens, const int64_t* ids, int64_t nseq, int32_t* table, int64_t capacity, int64_t* counts) {
  TD_REQUIRE(counts && nseq >= 0 && (nseq == 0 || (lens && ids)), TD_ERR_INVALID, "td_lora_plan: null pointer or %lld sequences", (long long)nseq);
  int64_t rows = 0, nid = 0;
  for (int64_t s = 0; s < nseq; ++s) {
    TD_REQUIRE(lens[s] >= 0 && lens[s] <= (1ll << 30), TD_ERR_INVALID, "td_lora_plan: sequence %lld has length %lld", (long long)s, (long long)lens[s]);
    TD_REQUIRE(ids[s] >= -1 && ids[s] < (1 << 20), TD_ERR_INVALID, "td_lora_plan: sequence %lld has adapter %lld", (long long)s, (long long)ids[s]);
    rows += lens[s];
    nid = std::max(nid, ids[s] + 1);
    TD_REQUIRE(rows <= (1ll << 30), TD_ERR_UNSUPPORTED, "td_lora_plan: more than 2^30 rows");
  }
  try {
    std::vector<int64_t> count(nid + 1, 0), at(nid + 1, 0);      // slot nid: no adapter
    for (int64_t s = 0; s < nseq; ++s) count[ids[s] < 0 ? nid : ids[s]] += lens[s];
    int64_t tiles[2] = {0, 0};
    for (int64_t i = 0, pos = 0; i <= nid; ++i) {
      at[i] = pos; pos += count[i];
      tiles[i == nid] += td_cdiv(count[i], LR_TILE);
    }
    counts[0] = tiles[0]; counts[1] = tiles[1]; counts[2] = rows; counts[3] = rows - count[nid]; counts[4] = nid;
    if (table) {
      TD_REQUIRE(capacity >= 4 * (tiles[0] + tiles[1]) + rows, TD_ERR_INVALID, "td_lora_plan: table of %lld words", (long long)capacity);
      LoraTile* t = reinterpret_cast<LoraTile*>(table);
      for (int64_t i = 0; i <= nid; ++i)
        for (int64_t r = 0; r < count[i]; r += LR_TILE)
          *t++ = {(int32_t)(at[i] + r), (int32_t)std::min<int64_t>(LR_TILE, count[i] - r), i == nid ? -1 : (int32_t)i, 0};
      int32_t* perm = reinterpret_cast<int32_t*>(t);
      for (int64_t s = 0, row = 0; s < nseq; ++s) {
        int64_t& pos = at[ids[s] < 0 ? nid : ids[s]];
        for (int64_t r = 0; r < lens[s]; ++r) perm[pos++] = (int32_t)row++;
      }
    }
  } catch (const std::bad_alloc&) {
    td_set_error("td_lora_plan: out of host memory");
    return TD_ERR_INVALID;
  }
  return TD_OK;
}

struct LoraShape { int rj, splits, steps; bool ks; };
// 256 CUs: with 512 tiles or more every wave owns 16 rows and walks the whole of K; below that the workgroups are 16 rows
// each, their waves split K, and K is split further until there are about 512 workgroups (at least 512 of K each)
static LoraShape lora_shape(int64_t tiles, int64_t rows, int64_t k, int max_rank) {
  LoraShape s;
  s.rj = max_rank <= 16 ? 1 : max_rank <= 32 ? 2 : max_rank <= 64 ? 4 : max_rank <= 128 ? 8 : 16;
  const int nsteps = (int)td_cdiv(k, 32);
  s.ks = tiles < 512;
  int64_t want = 1;
  if (s.ks) {
    const int64_t groups = std::max<int64_t>(std::max<int64_t>(tiles, 1), td_cdiv(rows, 16));
    want = std::max<int64_t>(1, std::min<int64_t>(td_cdiv(512, groups), nsteps / 16));
  }
  s.steps = (int)td_cdiv(nsteps, want);
  s.splits = (int)td_cdiv(nsteps, s.steps);
  return s;
}

extern "C" int td_lora_workspace(const int64_t* counts, int64_t k, int max_rank, int64_t* floats) {
  TD_REQUIRE(counts && floats && k > 0 && max_rank > 0 && max_rank <= LR_MAX_RANK, TD_ERR_INVALID, "td_lora_workspace: k = %lld, rank %d",
             (long long)k, max_rank);
  const LoraShape s = lora_shape(counts[0], counts[3], k, max_rank);
  *floats = (int64_t)s.splits * counts[3] * 16 * s.rj;
  return TD_OK;
}

extern "C" int td_lora_add(const void* x, int64_t ldx, const void* y, int64_t ldy, void* out, int64_t ldo, int dtype, int64_t k, int64_t n,
                           const void* bank, const void* adapters, int num_adapters, int max_rank, const int32_t* table,
                           const int64_t* counts, float* ws, td_stream_t stream) {
  TD_REQUIRE(x && y && out && bank && adapters && table && counts, TD_ERR_INVALID, "td_lora_add: null pointer");
  TD_REQUIRE(dtype == TD_BF16 || dtype == TD_F16, TD_ERR_UNSUPPORTED, "td_lora_add: dtype %d", dtype);
  TD_REQUIRE(k > 0 && n > 0 && k % 8 == 0 && n % 8 == 0 && k < (1 << 30) && n < (1 << 30), TD_ERR_UNSUPPORTED,
             "td_lora_add: k = %lld, n = %lld (multiples of 8)", (long long)k, (long long)n);
  TD_REQUIRE(ldx >= 0 && ldy >= 0 && ldo >= 0 && ldx % 8 == 0 && ldy % 8 == 0 && ldo % 8 == 0, TD_ERR_UNSUPPORTED,
             "td_lora_add: row strides must be multiples of 8 elements");
  TD_REQUIRE((((uintptr_t)x | (uintptr_t)y | (uintptr_t)out | (uintptr_t)bank | (uintptr_t)ws) & 15) == 0, TD_ERR_UNSUPPORTED,
             "td_lora_add: pointers must be 16-byte aligned");
  TD_REQUIRE(max_rank > 0 && max_rank <= LR_MAX_RANK, TD_ERR_UNSUPPORTED, "td_lora_add: rank %d (at most %d)", max_rank, LR_MAX_RANK);
  TD_REQUIRE(counts[4] <= num_adapters, TD_ERR_INVALID, "td_lora_add: the plan names adapter %lld of %d", (long long)counts[4] - 1, num_adapters);
  TD_REQUIRE(counts[0] >= 0 && counts[1] >= 0 && counts[0] + counts[1] < (1 << 28), TD_ERR_INVALID, "td_lora_add: counts");
  TD_REQUIRE(counts[3] == 0 || ws, TD_ERR_INVALID, "td_lora_add: null workspace");
  const LoraShape sh = lora_shape(counts[0], counts[3], k, max_rank);
  LoraParams p;
  p.x = (const uint16_t*)x; p.y = (const uint16_t*)y; p.out = (uint16_t*)out;
  p.ldx = ldx; p.ldy = ldy; p.ldo = ldo;
  p.bank = (const uint16_t*)bank; p.adapters = (const LoraAdapter*)adapters;
  p.tiles = reinterpret_cast<const LoraTile*>(table);
  p.perm = table + 4 * (counts[0] + counts[1]);
  p.s = ws; p.rows = counts[3]; p.K = k; p.N = n;
  p.splits = sh.splits; p.steps = sh.steps;
  const int64_t tiles = counts[0] + (out == y ? 0 : counts[1]);
  if (tiles == 0) return TD_OK;
  p.ntile = tiles >= 512 ? 1024 : tiles >= 32 ? 512 : 128;
  hipStream_t st = (hipStream_t)stream;
  const dim3 gs((unsigned)(counts[0] * (sh.ks ? 4 : 1)), (unsigned)sh.splits), ge((unsigned)tiles, (unsigned)td_cdiv(n, p.ntile));
  TD_REQUIRE(ge.y <= 65535, TD_ERR_UNSUPPORTED, "td_lora_add: n = %lld", (long long)n);
#define LR_GO(DT_, RJ_)                                                                        \
  {                                                                                            \
    if (counts[0] > 0) {                                                                       \
      if (sh.ks) lora_shrink_kernel<DT_, RJ_, true><<<gs, 256, 0, st>>>(p);                    \
      else lora_shrink_kernel<DT_, RJ_, false><<<gs, 256, 0, st>>>(p);                         \
    }                                                                                          \
    lora_expand_kernel<DT_, RJ_><<<ge, 256, 0, st>>>(p);                                       \
  }
#define LR_GO_DT(DT_)                                                                          \
  switch (sh.rj) {                                                                             \
    case 1: LR_GO(DT_, 1) break;                                                               \
    case 2: LR_GO(DT_, 2) break;                                                               \
    case 4: LR_GO(DT_, 4) break;                                                               \
    case 8: LR_GO(DT_, 8) break;                                                               \
    default: LR_GO(DT_, 16) break;                                                             \
  }
  if (dtype == TD_BF16) { LR_GO_DT(TD_BF16) } else { LR_GO_DT(TD_F16) }
#undef LR_GO_DT
#undef LR_GO
  TD_CHECK_LAUNCH();
  return TD_OK;
}
