// Low-rank adapters of many requests beside a shared projection:
//
//     out[r] = y[r] + s_i B_i (A_i x[r]),    i = the adapter of row r's request;  rows without one: out[r] = y[r]
//
// x [rows, K], y / out [rows, N], A_i [rank_i, K], B_i [N, rank_i], 16-bit.  The rows are taken adapter by adapter (a permutation
// made by the plan), in tiles of one adapter, so an adapter is read for all of its rows at once however its requests lie.
//
//   shrink   S = A_i x by MFMA 16x16x32, fp32.  A workgroup takes 32 rows, its four waves split K; with few rows K is split over
//            workgroups too and expand adds the fp32 parts in order.
//   expand   out = y + s_i B_i S: S is rounded once to the operands' type (half a step of the update only: it stays below the
//            rounding of the output wherever the update is not many times larger than the output itself), the scale multiplies
//            the update in fp32.  f16 ends at 65 504, which S passes long before the update does: each row of S is brought to
//            2^14 .. 2^15 by the power of two that its largest finite value asks for, and the update is brought back, both
//            exactly.  A wave keeps B_i of 64 columns in registers and walks the tile's rows, 16 at a time.
// The bank holds A and B in fragment order (td_lora_pack): every load of them is a contiguous kilobyte, ranks are padded to 8 only.
//
// What bounds it: memory; y and out dominate, then x, at 2 rank flops per byte.  MFMA fragments want 64 bytes from each of 16 rows;
// memory wants whole 128-byte lines, so x, y and out pass through LDS on their way (50 960 rows, 1536 -> 8960, ranks 128 and 64:
// expand 506 -> 419 us, 4.4 TB/s, shrink 85 -> 65 us, 423 and 70 with f16's powers of two, both 452 -> 455 in a graph; 32 760 rows,
// 5120 -> 5120, rank 32: 162 -> 122 us, 5.5 TB/s, and 103 -> 98, where shrink also waits for the previous pass's writes).  A large copy moves 4.9 TB/s.  With B_i read again for every 64 rows expand
// took 639 us; non-temporal loads and stores cost 2 to 15 %.
#include "td_common.h"
#include <algorithm>
#include <new>
#include <vector>

#define LR_WIDE 256       // rows per tile: many rows (B_i is read once per tile and column set) ...
#define LR_NARROW 32      // ... and few
#define LR_TURN 68        // floats per row of a wave's 16 x 64 update in LDS
#define LR_MAX_RANK 256

struct LoraTile { int32_t perm0, rows, adapter, pad; };
struct LoraAdapter {
  int64_t a_off, b_off;       // elements
  int32_t rank; float scale;
  __device__ int rank8() const { return (rank + 7) & ~7; }      // as laid out: rounded up to 8 (zeros)
};
// S past the rank is zero, whatever an infinite row of x or what lies behind A in the bank made of it: B is zero there, and only
// zero times zero is
__device__ __forceinline__ float4 lr_within(const float4& v, int r0, int rank) {
  return make_float4(r0 < rank ? v.x : 0.f, r0 + 1 < rank ? v.y : 0.f, r0 + 2 < rank ? v.z : 0.f, r0 + 3 < rank ? v.w : 0.f);
}
__device__ __forceinline__ float lr_largest(const float4& v) {        // of the finite magnitudes
  const auto f = [](float x) { return fabsf(x) < INFINITY ? fabsf(x) : 0.f; };
  return fmaxf(fmaxf(f(v.x), f(v.y)), fmaxf(f(v.z), f(v.w)));
}
// the power of two that brings a row of S with this largest value to [2^14, 2^15) (bf16 has the range of fp32: 1), and its inverse
template <int DT> __device__ __forceinline__ int lr_shift(float largest) {
  if constexpr (DT == TD_BF16) return 0;
  return max(-100, min(100, 15 - __builtin_amdgcn_frexp_expf(largest)));
}
__device__ __forceinline__ float lr_power(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }
template <int DT> __device__ __forceinline__ uint2 lr_round(const float4& v, int shift) {
  if constexpr (DT == TD_BF16) return make_uint2(pack2<DT>(v.x, v.y), pack2<DT>(v.z, v.w));
  const float f = lr_power(shift);
  return make_uint2(pack2<DT>(v.x * f, v.y * f), pack2<DT>(v.z * f, v.w * f));
}

struct LoraParams {
  const uint16_t *x, *y; uint16_t* out;
  int64_t ldx, ldy, ldo;
  const uint16_t* bank; const LoraAdapter* adapters;
  const LoraTile* tiles; const int32_t* perm;
  void* s;                  // splits == 1: 16-bit [rows][RS]; else f32 parts [splits][rows][RS]
  float* back;              // splits == 1, f16: what brings a row's update back [rows]
  int64_t rows, K, N;
  int splits, chunks;       // K splits over workgroups, K chunks of 64 per split
  int subs;                 // 32-row groups of a full tile
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

// Fragment order of one adapter, r8 = its padded rank:
//   A: [K / 32][rank][4 k-quads][8 k]: the fragment of ranks 16 j .. and K step s is the kilobyte at 32 r8 s + 512 j
//   B: [N / 32][rank / 32][2 column sets b][rank quads (4, fewer in the last)][16 rows i][8 ranks], row i of set b = column
//      8 (i >> 2) + 4 b + (i & 3): after both sets a lane holds 8 consecutive columns of one x row
__global__ __launch_bounds__(256) void lora_pack_kernel(const uint16_t* a, int64_t lda, const uint16_t* b, int64_t ldb, int rank, int r8,
                                                        int64_t K, int64_t N, uint16_t* da, uint16_t* db) {
  const int64_t na = (K + 31) / 32 * 4 * r8, nb = (N + 31) / 32 * 4 * r8;       // 16-byte pieces
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < na + nb; i += (int64_t)gridDim.x * 256) {
    uint16_t* d; const uint16_t* src = nullptr; int valid = 0;
    if (i < na) {
      const int64_t s = i / (4 * r8);
      const int w = (int)(i - s * 4 * r8), r = w >> 2;
      const int64_t k = 32 * s + 8 * (w & 3);
      d = da + 8 * i;
      if (r < rank && k < K) { src = a + r * lda + k; valid = 8; }
    } else {
      const int64_t j = i - na, pb = j / (4 * r8);
      int w = (int)(j - pb * 4 * r8);
      const int kk = w / 128;
      w -= kk * 128;
      const int nq = min(4, r8 / 8 - 4 * kk), bs = w / (16 * nq);
      w -= bs * 16 * nq;
      const int q = w >> 4, l = w & 15;
      const int64_t n = 32 * pb + 8 * (l >> 2) + 4 * bs + (l & 3);
      const int r0 = 32 * kk + 8 * q;
      d = db + 8 * j;
      if (n < N && r0 < rank) { src = b + n * ldb + r0; valid = min(8, rank - r0); }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) d[e] = e < valid ? src[e] : (uint16_t)0;
  }
}

// K chunks [c0, c1) of 64 of 32 rows, ranks [0, 16 NJ) of one adapter.  x: 8 lanes take a row's 128 bytes (a full line) and hand
// them over as fragments through the wave's own LDS (4 KB a chunk, 16-byte pieces XOR-permuted against bank conflicts).  No load
// sits behind a branch: the last fragment of a rank that is no multiple of 16 brings ranks of whatever lies behind it in the
// bank (it ends with spare elements), which nothing reads.
template <int DT, int NJ, int RJ>
__device__ __forceinline__ void lr_shrink(v4f (&acc)[2][RJ], const uint16_t* const (&x)[4], const uint16_t* ap, int64_t astep, int c0, int c1,
                                          int64_t K, char* turn, int lane) {
  const int l16 = lane & 15, lq = lane >> 4, lr = lane >> 3, lc = lane & 7;
  const int last = (int)((K + 31) / 32) - 1;
  const v4i zero = {0, 0, 0, 0};
  for (int c = c0; c < c1; ++c) {
    const int64_t k = 64 * (int64_t)c + 8 * lc;
    v4i xv[4], af[2][NJ];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const v4i v = *reinterpret_cast<const v4i*>(x[i] + min(k, K - 8));
      xv[i] = k < K ? v : zero;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < NJ; ++j) af[h][j] = *reinterpret_cast<const v4i*>(ap + min(2 * c + h, last) * astep + 512 * j);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 8 * i + lr;
      *reinterpret_cast<v4i*>(turn + r * 128 + ((lc ^ ((r >> 1) & 7)) << 4)) = xv[i];
    }
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (h && 2 * c + 1 > last) break;           // x is zero there and A another step's, which may be infinite
      const char* f = turn + l16 * 128 + (((4 * h + lq) ^ ((l16 >> 1) & 7)) << 4);
      const v4i x0 = *reinterpret_cast<const v4i*>(f), x1 = *reinterpret_cast<const v4i*>(f + 2048);
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        acc[0][j] = lr_mma<DT>::run(af[h][j], x0, acc[0][j]);
        acc[1][j] = lr_mma<DT>::run(af[h][j], x1, acc[1][j]);
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// RJ: 16-rank blocks of the largest adapter (1, 2, 4, 8, 16); an adapter takes the smallest of these that holds its rank
template <int DT, int RJ>
__global__ __launch_bounds__(256, RJ <= 8 ? 2 : 1) void lora_shrink_kernel(const LoraParams p) {
  constexpr int RS = 16 * RJ;
  const int lane = threadIdx.x & 63, l16 = lane & 15, lq = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const LoraTile t = p.tiles[blockIdx.x / p.subs];
  const int row0 = 32 * (blockIdx.x % p.subs);
  if (row0 >= t.rows) return;
  const LoraAdapter ad = p.adapters[t.adapter];
  const uint16_t* xp[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)                                     // rows past the tile repeat its last one
    xp[i] = p.x + (int64_t)p.perm[t.perm0 + min(row0 + 8 * i + (lane >> 3), t.rows - 1)] * p.ldx;
  const uint16_t* ap = p.bank + ad.a_off + (l16 * 4 + lq) * 8;
  const int64_t astep = 32 * ad.rank8();
  const int nchunks = (int)((p.K + 63) / 64);
  const int per = (p.chunks + 3) / 4;
  const int c0 = blockIdx.y * p.chunks + wave * per, c1 = min(min(nchunks, (int)(blockIdx.y + 1) * p.chunks), c0 + per);
  constexpr int RED = 4 * 2 * RJ * 64 * 16;
  __shared__ __attribute__((aligned(16))) char smem[RED > 16384 ? RED : 16384];
  v4f acc[2][RJ];
#pragma unroll
  for (int g = 0; g < 2; ++g)
#pragma unroll
    for (int j = 0; j < RJ; ++j) acc[g][j] = (v4f){0.f, 0.f, 0.f, 0.f};
#define LR_SHRINK(NJ_) lr_shrink<DT, NJ_, RJ>(acc, xp, ap, astep, c0, c1, p.K, smem + wave * 4096, lane)
  if (ad.rank8() <= 16) LR_SHRINK(1);
  else if constexpr (RJ > 1) {
    if (ad.rank8() <= 32) LR_SHRINK(2);
    else if constexpr (RJ > 2) {
      if (ad.rank8() <= 64) LR_SHRINK(4);
      else if constexpr (RJ > 4) {
        if (ad.rank8() <= 128) LR_SHRINK(8);
        else if constexpr (RJ > 8) LR_SHRINK(16);
      }
    }
  }
#undef LR_SHRINK
  // acc[g][j][r] is row 16 g + l16, rank 16 j + 4 lq + r; the four waves' parts are added in order, each wave a share of them
  float4 (*red)[2 * RJ][64] = reinterpret_cast<float4 (*)[2 * RJ][64]>(smem);
  __syncthreads();
#pragma unroll
  for (int g = 0; g < 2; ++g)
#pragma unroll
    for (int j = 0; j < RJ; ++j) red[wave][g * RJ + j][lane] = make_float4(acc[g][j][0], acc[g][j][1], acc[g][j][2], acc[g][j][3]);
  __syncthreads();
  const auto total = [&](int i) {
    float4 v = red[0][i][lane];
#pragma unroll
    for (int w = 1; w < 4; ++w) {
      const float4 o = red[w][i][lane];
      v.x += o.x; v.y += o.y; v.z += o.z; v.w += o.w;
    }
    return v;
  };
  if (p.splits > 1) {
    for (int i = wave; i < 2 * RJ; i += 4) {
      const int g = i / RJ, j = i % RJ, r = row0 + 16 * g + l16;
      if (16 * j >= ad.rank8() || r >= t.rows) continue;
      *reinterpret_cast<float4*>(reinterpret_cast<float*>(p.s) + ((int64_t)blockIdx.y * p.rows + t.perm0 + r) * RS + 16 * j + 4 * lq) = total(i);
    }
    return;
  }
  // f16: the largest value of each row first, block by block
  __shared__ float largest[2 * RJ][16];
  constexpr int PER = (2 * RJ + 3) / 4;
  float4 v[PER];
#pragma unroll
  for (int n = 0; n < PER; ++n) {
    const int i = wave + 4 * n, j = i % RJ;
    if (i >= 2 * RJ || 16 * j >= ad.rank8()) continue;
    v[n] = lr_within(total(i), 16 * j + 4 * lq, ad.rank);
    if constexpr (DT == TD_F16) {
      float m = lr_largest(v[n]);
      m = fmaxf(m, __shfl_xor(m, 16, 64));
      m = fmaxf(m, __shfl_xor(m, 32, 64));
      if (lq == 0) largest[i][l16] = m;
    }
  }
  if constexpr (DT == TD_F16) __syncthreads();
#pragma unroll
  for (int n = 0; n < PER; ++n) {
    const int i = wave + 4 * n, g = i / RJ, j = i % RJ, r = row0 + 16 * g + l16;
    if (i >= 2 * RJ || 16 * j >= ad.rank8() || r >= t.rows) continue;
    int shift = 0;
    if constexpr (DT == TD_F16) {
      float m = largest[g * RJ][l16];
#pragma unroll
      for (int k = 1; k < RJ; ++k)
        if (16 * k < ad.rank8()) m = fmaxf(m, largest[g * RJ + k][l16]);
      shift = lr_shift<DT>(m);
      if (j == 0 && lq == 0) p.back[t.perm0 + r] = lr_power(-shift);
    }
    *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(p.s) + (t.perm0 + r) * (int64_t)RS + 16 * j + 4 * lq) = lr_round<DT>(v[n], shift);
  }
}

// 64 columns from n of the tile's rows, ranks [0, 32 NK): B stays in registers, y and S of the next 16 rows are on their way
// while these multiply.  sb / srs: the tile's S (16-bit) and its row stride; prow: its rows' numbers, back: f16, what brings their
// updates back (both LDS); turn: the wave's own 16 x 64 floats of LDS.
template <int DT, int NK>
__device__ __forceinline__ void lr_expand(const LoraParams& p, const uint16_t* sb, int srs, const int32_t* prow, const float* back, int rows,
                                          const uint16_t* bp, int rank8, float scale, int64_t n, int l16, int lq, float* turn) {
  v4i bf[2][2][NK];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint16_t* bh = bp + min(n / 32 + h, (p.N - 1) / 32) * 32 * rank8;
#pragma unroll
    for (int kk = 0; kk < NK; ++kk)
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const int quads = min(4, max(0, rank8 / 8 - 4 * kk));
        v4i f = *reinterpret_cast<const v4i*>(bh + kk * 1024 + b * quads * 128);
        const int keep = lq < quads ? -1 : 0;                   // what lies behind the rank's last quad is not B's
        bf[h][b][kk] = f & (v4i){keep, keep, keep, keep};
      }
  }
  // y and out: 8 lanes take a row's 128 bytes (a full line), two sets of 8 rows; the update comes to them through LDS
  const int lr = (threadIdx.x & 63) >> 3;
  const int64_t col = n + 8 * (threadIdx.x & 7);
  const bool cin = col < p.N;
  const uint16_t* yb = p.y + min(col, p.N - 8);                 // columns past the end: re-read the last ones, not stored
  uint16_t* ob = p.out + col;
  uint4 yv[2];
  v4i sf[NK];
  int64_t row[2];
  float bk[2] = {1.f, 1.f};
  auto load = [&](int g) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      row[i] = prow[min(g + 8 * i + lr, rows - 1)];
      if constexpr (DT == TD_F16) bk[i] = back[min(g + 8 * i + lr, rows - 1)];
      yv[i] = *reinterpret_cast<const uint4*>(yb + row[i] * p.ldy);
    }
#pragma unroll
    for (int kk = 0; kk < NK; ++kk) {
      const int r0 = 32 * kk + 8 * lq, keep = r0 < rank8 ? -1 : 0;               // zero past the rank, like B
      sf[kk] = *reinterpret_cast<const v4i*>(sb + (int64_t)min(g + l16, rows - 1) * srs + min(r0, rank8 - 8)) & (v4i){keep, keep, keep, keep};
    }
  };
  load(0);
  for (int g = 0; g < rows; g += 16) {
    v4f acc[2][2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        acc[h][b] = (v4f){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kk = 0; kk < NK; ++kk) acc[h][b] = lr_mma<DT>::run(bf[h][b][kk], sf[kk], acc[h][b]);
        *reinterpret_cast<v4f*>(turn + l16 * LR_TURN + 32 * h + 8 * lq + 4 * b) = acc[h][b];
      }
    __builtin_amdgcn_wave_barrier();
    const uint4 v[2] = {yv[0], yv[1]};
    const int64_t r[2] = {row[0], row[1]};
    const float b[2] = {bk[0], bk[1]};
    if (g + 16 < rows) load(g + 16);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float f[8];
      unpack8<DT>(v[i], f);
      const v4f* d = reinterpret_cast<const v4f*>(turn + (8 * i + lr) * LR_TURN + 8 * (threadIdx.x & 7));
      const v4f d0 = d[0], d1 = d[1];
#pragma unroll
      for (int e = 0; e < 4; ++e) {        // two factors: their product alone may be past fp32
        f[e] = fmaf(DT == TD_F16 ? d0[e] * b[i] : d0[e], scale, f[e]);
        f[4 + e] = fmaf(DT == TD_F16 ? d1[e] * b[i] : d1[e], scale, f[4 + e]);
      }
      if (cin && g + 8 * i + lr < rows) *reinterpret_cast<uint4*>(ob + r[i] * p.ldo) = pack8<DT>(f);
    }
  }
}

template <int DT, int RJ>
__global__ __launch_bounds__(256, RJ <= 8 ? 2 : 1) void lora_expand_kernel(const LoraParams p) {
  constexpr int RS = 16 * RJ, KK = (RJ + 1) / 2;
  const int lane = threadIdx.x & 63, l16 = lane & 15, lq = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const LoraTile t = p.tiles[blockIdx.x];
  const int64_t n = (int64_t)blockIdx.y * 256 + 64 * wave;
  __shared__ int32_t prow[LR_WIDE];
  __shared__ __attribute__((aligned(16))) float turn[4][16 * LR_TURN];
  __shared__ float back[DT == TD_F16 ? LR_WIDE : 1];
  if (threadIdx.x < t.rows) prow[threadIdx.x] = p.perm[t.perm0 + threadIdx.x];
  if (t.adapter < 0) {            // rows without an adapter: copy
    __syncthreads();
    const int64_t c = (int64_t)blockIdx.y * 256 + 8 * (lane & 31);
    if (c < p.N)
      for (int r = 2 * wave + (lane >> 5); r < t.rows; r += 8)
        *reinterpret_cast<uint4*>(p.out + prow[r] * p.ldo + c) = *reinterpret_cast<const uint4*>(p.y + prow[r] * p.ldy + c);
    return;
  }
  const LoraAdapter ad = p.adapters[t.adapter];
  const uint16_t* sb = reinterpret_cast<const uint16_t*>(p.s) + (int64_t)t.perm0 * RS;
  int srs = RS;
  __shared__ __attribute__((aligned(16))) uint16_t ssum[LR_NARROW * (RS + 8)];
  if (p.splits > 1) {             // add the parts of S, round (narrow tiles only); 2^lw neighbouring lanes take a row
    const float* sp = reinterpret_cast<const float*>(p.s) + (int64_t)t.perm0 * RS;
    const int quads = ad.rank8() / 4, lw = 32 - __builtin_clz(quads - 1), q = threadIdx.x & ((1 << lw) - 1), c = 4 * q;
    for (int r = threadIdx.x >> lw; r < t.rows; r += 256 >> lw) {
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      if (q < quads) {
#pragma unroll 8
        for (int s = 0; s < p.splits; ++s) {
          const float4 o = *reinterpret_cast<const float4*>(sp + (s * p.rows + r) * RS + c);
          v.x += o.x; v.y += o.y; v.z += o.z; v.w += o.w;
        }
        v = lr_within(v, c, ad.rank);
      }
      int shift = 0;
      if constexpr (DT == TD_F16) {
        float m = lr_largest(v);
        for (int o = (1 << lw) / 2; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
        shift = lr_shift<DT>(m);
        if (q == 0) back[r] = lr_power(-shift);
      }
      if (q < quads) *reinterpret_cast<uint2*>(ssum + r * (RS + 8) + c) = lr_round<DT>(v, shift);
    }
    sb = ssum;
    srs = RS + 8;
  } else if (DT == TD_F16 && threadIdx.x < t.rows) {
    back[threadIdx.x] = p.back[t.perm0 + threadIdx.x];
  }
  __syncthreads();
  if (n >= p.N) return;
  const uint16_t* bp = p.bank + ad.b_off + lane * 8;
#define LR_EXPAND(NK_) lr_expand<DT, NK_>(p, sb, srs, prow, back, t.rows, bp, ad.rank8(), ad.scale, n, l16, lq, turn[wave])
  if (ad.rank8() <= 32) LR_EXPAND(1);
  else if constexpr (KK > 1) {
    if (ad.rank8() <= 64) LR_EXPAND(2);
    else if constexpr (KK > 2) {
      if (ad.rank8() <= 128) LR_EXPAND(4);
      else if constexpr (KK > 4) LR_EXPAND(8);
    }
  }
#undef LR_EXPAND
}

// Both steps in one launch, for a few rows: every workgroup of 256 columns forms the tile's S itself, its 8 waves splitting K, and
// the first four expand.  A_i is read once per workgroup (from L2), which pays while there are few of them.  One row, K = N =
// 4096, rank 16: 8.0 us a call instead of 11.8 (a second launch costs the host 3 us); replayed from a graph, where launches are
// cheap, 6.9 instead of 6.2.
template <int DT, int RJ>
__global__ __launch_bounds__(512) void lora_few_kernel(const LoraParams p) {
  constexpr int RS = 16 * RJ, KK = (RJ + 1) / 2, W = 8;
  const int lane = threadIdx.x & 63, l16 = lane & 15, lq = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const LoraTile t = p.tiles[blockIdx.x];
  constexpr int RED = W * 2 * RJ * 64 * 16;                       // bytes: the waves' parts of S; before that 4 KB a wave to turn x
  __shared__ __attribute__((aligned(16))) char smem[RED > W * 4096 ? RED : W * 4096];
  __shared__ __attribute__((aligned(16))) uint16_t ssum[LR_NARROW * (RS + 8)];
  __shared__ int32_t prow[LR_NARROW];
  __shared__ float back[LR_NARROW], largest[2 * RJ][16];
  if ((int)threadIdx.x < t.rows) prow[threadIdx.x] = p.perm[t.perm0 + threadIdx.x];
  __syncthreads();
  if (t.adapter < 0) {            // rows without an adapter: copy
    const int64_t c = (int64_t)blockIdx.y * 256 + 8 * (lane & 31);
    if (c < p.N)
      for (int r = 2 * wave + (lane >> 5); r < t.rows; r += 2 * W) *reinterpret_cast<uint4*>(p.out + prow[r] * p.ldo + c) = *reinterpret_cast<const uint4*>(p.y + prow[r] * p.ldy + c);
    return;
  }
  const LoraAdapter ad = p.adapters[t.adapter];
  {
    const uint16_t* xp[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) xp[i] = p.x + (int64_t)prow[min(8 * i + (lane >> 3), t.rows - 1)] * p.ldx;
    const uint16_t* ap = p.bank + ad.a_off + (l16 * 4 + lq) * 8;
    const int64_t astep = 32 * ad.rank8();
    const int nchunks = (int)((p.K + 63) / 64), per = (nchunks + W - 1) / W;
    v4f acc[2][RJ];
#pragma unroll
    for (int g = 0; g < 2; ++g)
#pragma unroll
      for (int j = 0; j < RJ; ++j) acc[g][j] = (v4f){0.f, 0.f, 0.f, 0.f};
#define LR_SHRINK(NJ_) lr_shrink<DT, NJ_, RJ>(acc, xp, ap, astep, wave * per, min(nchunks, (wave + 1) * per), p.K, smem + wave * 4096, lane)
    if (ad.rank8() <= 16) LR_SHRINK(1);
    else if constexpr (RJ > 1) {
      if (ad.rank8() <= 32) LR_SHRINK(2);
      else if constexpr (RJ > 2) LR_SHRINK(4);
    }
#undef LR_SHRINK
    float4 (*red)[2 * RJ][64] = reinterpret_cast<float4 (*)[2 * RJ][64]>(smem);
    __syncthreads();
#pragma unroll
    for (int g = 0; g < 2; ++g)
#pragma unroll
      for (int j = 0; j < RJ; ++j) red[wave][g * RJ + j][lane] = make_float4(acc[g][j][0], acc[g][j][1], acc[g][j][2], acc[g][j][3]);
    __syncthreads();
    const int g = wave / RJ, j = wave % RJ, r = 16 * g + l16;
    float4 v;
    if (wave < 2 * RJ) {
      v = red[0][wave][lane];
#pragma unroll
      for (int w = 1; w < W; ++w) {
        const float4 o = red[w][wave][lane];
        v.x += o.x; v.y += o.y; v.z += o.z; v.w += o.w;
      }
      v = lr_within(v, 16 * j + 4 * lq, ad.rank);
      if constexpr (DT == TD_F16) {
        float m = lr_largest(v);
        m = fmaxf(m, __shfl_xor(m, 16, 64));
        m = fmaxf(m, __shfl_xor(m, 32, 64));
        if (lq == 0) largest[wave][l16] = m;
      }
    }
    if constexpr (DT == TD_F16) __syncthreads();
    if (wave < 2 * RJ) {
      int shift = 0;
      if constexpr (DT == TD_F16) {
        float m = largest[g * RJ][l16];
#pragma unroll
        for (int k = 1; k < RJ; ++k) m = fmaxf(m, largest[g * RJ + k][l16]);
        shift = lr_shift<DT>(m);
        if (j == 0 && lq == 0) back[r] = lr_power(-shift);
      }
      *reinterpret_cast<uint2*>(ssum + r * (RS + 8) + 16 * j + 4 * lq) = lr_round<DT>(v, shift);
    }
    __syncthreads();
  }
  const int64_t n = (int64_t)blockIdx.y * 256 + 64 * wave;
  if (wave >= 4 || n >= p.N) return;
  const uint16_t* bp = p.bank + ad.b_off + lane * 8;
  float* const turn = reinterpret_cast<float*>(smem) + wave * 16 * LR_TURN;
#define LR_EXPAND(NK_) lr_expand<DT, NK_>(p, ssum, RS + 8, prow, back, t.rows, bp, ad.rank8(), ad.scale, n, l16, lq, turn)
  if (ad.rank8() <= 32) LR_EXPAND(1);
  else if constexpr (KK > 1) LR_EXPAND(2);
#undef LR_EXPAND
}

// ---- the plan (host): rows by adapter, tiles of one adapter, rows without one last -----------------------------------------
// counts = {tiles with an adapter, tiles without, rows, rows with an adapter, largest id + 1, rows per tile}; table = tiles (4
// words each), then the row permutation
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
    const int64_t tile = rows - count[nid] >= 8192 ? LR_WIDE : LR_NARROW;
    int64_t tiles[2] = {0, 0};
    for (int64_t i = 0, pos = 0; i <= nid; ++i) {
      at[i] = pos; pos += count[i];
      tiles[i == nid] += td_cdiv(count[i], tile);
    }
    counts[0] = tiles[0]; counts[1] = tiles[1]; counts[2] = rows; counts[3] = rows - count[nid]; counts[4] = nid; counts[5] = tile;
    if (table) {
      TD_REQUIRE(capacity >= 4 * (tiles[0] + tiles[1]) + rows, TD_ERR_INVALID, "td_lora_plan: table of %lld words", (long long)capacity);
      LoraTile* t = reinterpret_cast<LoraTile*>(table);
      for (int64_t i = 0; i <= nid; ++i)
        for (int64_t r = 0; r < count[i]; r += tile)
          *t++ = {(int32_t)(at[i] + r), (int32_t)std::min<int64_t>(tile, count[i] - r), i == nid ? -1 : (int32_t)i, 0};
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

struct LoraShape { int rj, splits, chunks; bool few; };
// 256 CUs: K is split over workgroups until there are about 256 of them (at most 8 parts, 512 of K each or more)
// few: one launch (lora_few_kernel) while its workgroups all run at once and a wave has at most 8 chunks of K (0.5 us each) to walk
static LoraShape lora_shape(const int64_t* counts, int64_t k, int64_t n, int max_rank) {
  LoraShape s;
  s.rj = max_rank <= 16 ? 1 : max_rank <= 32 ? 2 : max_rank <= 64 ? 4 : max_rank <= 128 ? 8 : 16;
  const int64_t nch = td_cdiv(k, 64), tiles = std::max<int64_t>(counts[0], 1);
  const int64_t want = counts[5] == LR_WIDE ? 1 : std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(8, td_cdiv(256, tiles)), nch / 8));
  s.chunks = (int)td_cdiv(nch, want);
  s.splits = (int)td_cdiv(nch, s.chunks);
  s.few = counts[5] == LR_NARROW && s.rj <= 4 && k <= 4096 && (counts[0] + counts[1]) * td_cdiv(n, 256) <= 256;
  return s;
}

extern "C" int td_lora_workspace(const int64_t* counts, int64_t k, int64_t n, int max_rank, int64_t* floats) {
  TD_REQUIRE(counts && floats && k > 0 && n > 0 && max_rank > 0 && max_rank <= LR_MAX_RANK, TD_ERR_INVALID, "td_lora_workspace: k = %lld, rank %d",
             (long long)k, max_rank);
  const LoraShape s = lora_shape(counts, k, n, max_rank);
  *floats = s.few ? 0 : s.splits == 1 ? counts[3] * (8 * s.rj + 1) : s.splits * counts[3] * 16 * s.rj;       // 16-bit S and a factor a row; parts of S
  return TD_OK;
}

extern "C" int td_lora_pack(const void* a, int64_t lda, const void* b, int64_t ldb, int rank, int64_t k, int64_t n, void* bank_a, void* bank_b,
                            td_stream_t stream) {
  TD_REQUIRE(a && b && bank_a && bank_b, TD_ERR_INVALID, "td_lora_pack: null pointer");
  TD_REQUIRE(rank > 0 && rank <= LR_MAX_RANK && k > 0 && n > 0 && k % 8 == 0 && n % 8 == 0 && k < (1 << 30) && n < (1 << 30), TD_ERR_UNSUPPORTED,
             "td_lora_pack: rank %d (at most %d), k = %lld, n = %lld (multiples of 8)", rank, LR_MAX_RANK, (long long)k, (long long)n);
  TD_REQUIRE(((uintptr_t)bank_a & 15) == 0 && ((uintptr_t)bank_b & 15) == 0, TD_ERR_UNSUPPORTED, "td_lora_pack: the bank must be 16-byte aligned");
  const int r8 = (rank + 7) / 8 * 8;
  const int64_t pieces = (td_cdiv(k, 32) + td_cdiv(n, 32)) * 4 * r8;
  lora_pack_kernel<<<(unsigned)std::min<int64_t>(td_cdiv(pieces, 256), 1024), 256, 0, (hipStream_t)stream>>>(
      (const uint16_t*)a, lda, (const uint16_t*)b, ldb, rank, r8, k, n, (uint16_t*)bank_a, (uint16_t*)bank_b);
  TD_CHECK_LAUNCH();
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
  TD_REQUIRE(counts[5] == LR_WIDE || counts[5] == LR_NARROW, TD_ERR_INVALID, "td_lora_add: counts");
  TD_REQUIRE(counts[2] <= 1 || ldo >= n, TD_ERR_INVALID, "td_lora_add: the rows of out overlap");
  TD_REQUIRE(out != y || ldo == ldy || counts[2] <= 1, TD_ERR_INVALID, "td_lora_add: out = y with another row stride");
  const LoraShape sh = lora_shape(counts, k, n, max_rank);
  TD_REQUIRE(counts[3] == 0 || sh.few || ws, TD_ERR_INVALID, "td_lora_add: null workspace");
  LoraParams p;
  p.x = (const uint16_t*)x; p.y = (const uint16_t*)y; p.out = (uint16_t*)out;
  p.ldx = ldx; p.ldy = ldy; p.ldo = ldo;
  p.bank = (const uint16_t*)bank; p.adapters = (const LoraAdapter*)adapters;
  p.tiles = reinterpret_cast<const LoraTile*>(table);
  p.perm = table + 4 * (counts[0] + counts[1]);
  p.s = ws; p.rows = counts[3]; p.K = k; p.N = n;
  p.back = ws ? ws + counts[3] * 8 * sh.rj : nullptr;
  p.splits = sh.splits; p.chunks = sh.chunks;
  const int64_t tiles = counts[0] + (out == y ? 0 : counts[1]);
  if (tiles == 0) return TD_OK;
  p.subs = (int)(counts[5] / 32);
  hipStream_t st = (hipStream_t)stream;
  const dim3 gs((unsigned)(counts[0] * p.subs), (unsigned)sh.splits), ge((unsigned)tiles, (unsigned)td_cdiv(n, 256));
  TD_REQUIRE(ge.y <= 65535, TD_ERR_UNSUPPORTED, "td_lora_add: n = %lld", (long long)n);
#define LR_GO(DT_, RJ_)                                                                        \
  {                                                                                            \
    if (counts[0] > 0) lora_shrink_kernel<DT_, RJ_><<<gs, 256, 0, st>>>(p);                    \
    lora_expand_kernel<DT_, RJ_><<<ge, 256, 0, st>>>(p);                                       \
  }
  if (sh.few) {
#define LR_FEW(DT_)                                                       \
    if (sh.rj == 1) lora_few_kernel<DT_, 1><<<ge, 512, 0, st>>>(p);        \
    else if (sh.rj == 2) lora_few_kernel<DT_, 2><<<ge, 512, 0, st>>>(p);   \
    else lora_few_kernel<DT_, 4><<<ge, 512, 0, st>>>(p);
    if (dtype == TD_BF16) { LR_FEW(TD_BF16) } else { LR_FEW(TD_F16) }
#undef LR_FEW
    TD_CHECK_LAUNCH();
    return TD_OK;
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
