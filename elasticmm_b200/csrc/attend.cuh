// Decode attention over a 4-bit paged cache (sm_100a): one query token per sequence.
//
//   l[t] = scale * q . k[t]      p = softmax(l) over the sequence's tokens      out = sum_t p[t] v[t]
//   weights (optional): score[block of t][kv head][place of t] += sum of p[t] over the query heads of the kv head
//
// The work is one pass over the cached rows (160 bytes per token and KV head at D = 128), so HBM bounds it; what the
// layout below is for is to spend few enough instructions per row to keep up (about 40 16-bit elements per clock and SM).
//
// Products. A warp owns one KV head and up to eight of its query heads, and takes 16 tokens at a time through
// mma.m16n8k16 with the CACHE as the 16-row operand: S^T = K Q^T (rows tokens, columns heads), O^T = V^T P^T (rows
// channels, columns heads). A tcgen05 tile has 64 rows at least, of which a decode step could fill eight, and takes
// its operands from shared memory, where the codes would first have to be written out as 16-bit values.
//
// Codes are never converted. A nibble masked in place in a 16-bit lane IS a floating-point number: c * 2^-24 from bits
// 0..3 and c * 2^-20 from bits 4..7 as fp16 (keys), c * 2^-133 and c * 2^-129 as bf16 (values; bit 7 belongs to the
// exponent there, but the smallest normal numbers have the subnormals' step), exact, and the tensor cores take
// subnormals at full rate. One AND (and half a shift) makes two operand elements. The powers of two are undone in q
// (keys) or when the result is written (values).
//
// Scales and offsets, x = o + s (c - 8), group r of 32 channels:
//   l[t]   = sum_r s_r[t] (sum_d q_d c_d) + sum_r (o_r[t] - 8 s_r[t]) Q_r,      Q_r = sum of q over the group
//            the first bracket is two MMAs per group; the last sum is one MMA (two at D = 256) with a token's scales and
//            offsets, which lie side by side in its row, as the row operand and Q in two fp16 halves (22 bits).
//   out[d] = sum_t (p s_r) c_d + sum_t p (o_r - 8 s_r)
//            p s_r is formed in 32 bits and enters as two bf16 parts (below); the last sum has scales and offsets as rows.
// p is held relative to a reference that only follows the running maximum when that outgrows it by 2^6, so the
// accumulators are rarely rescaled and no maximum is taken across lanes in between.
// Rounding. p stays in 32 bits (its fragment is transposed in two halves of 16). p s_r is cut to its first 8 bits, and
// what is left is rounded to 8 more: two MMAs on the same codes, off by 2^-16 of p s_r at most. bf16 has the range of 32
// bits, so no scale, however large, takes bits from a smaller one or from a lesser weight. One part would be 2^-8, more
// than a result's own rounding; fp16 parts run out of range: with p held below 2^14 for the sake of scales of 2^13, p s_r
// of thousands of tokens with a small scale and a small weight each was 0. Against the offsets p enters as two 11-bit
// parts, the second times 2^12 into sums of its own: 2^-22, down to 2^-45 of the largest p.
// Logits, sums and accumulators are 32 bits. Against 64 bits the result is off by its own rounding: 1.7e-3 (bf16) and
// 2.1e-4 (fp16), as where all of it is computed in 32 bits.
//
// Work. A unit is 16 (x token subsets) tokens of one sequence for the KV heads of a CTA, one warp per head, tile of
// query heads and subset. The units of the whole batch, counted on the device, are split evenly over the CTAs, whatever
// the lengths: a CTA finishes the sequences that lie in its share and leaves a partial result (in the workspace) of
// the at most two that do not; attend_join adds those.
// Every warp fetches its own rows into a ring of its own with 16-byte cp.async, so that warps never wait for one another
// inside a segment. Bulk copies of a token's heads (640 bytes; 1280 per head of head-major pages) were measured first: an
// SM completed one in 28 (38) ns whatever was in flight, which held the loads alone to 3.4 (4.7) TB/s; tensor boxes of 16
// rows of 80 bytes came to 3.7 TB/s. The 16-byte copies alone reach 6 TB/s.
//
// Measured, D = 128, 8 KV heads, 8 query heads each, bf16: one sequence of 131 071 tokens 61 us (168 MB: 2.75 TB/s), 64 of
// 128 to 8 191 tokens 65 us, with weights 81 (the first kernel, scalar: 288 ms and 14 ms). With one 16-bit part for p s_r
// these took 53, 58 and 71. 49 us of the 61 are the loop, whose loads alone take 28 and whose arithmetic alone 39: no unit
// is full (issue 43 % of cycles, ALU 40 %, tensor cores 24 %), two warps a scheduler do not hide all of one another's
// chain from codes to products. The rest is the share, the first loads, the queries and the join.
// More than eight query heads on a KV head are several tiles, each of whose warps fetches and unpacks the rows for itself
// (131 071 tokens, 8 KV heads: 16 query heads each 109 us, 64 each 433).
#pragma once
#include "q4.cuh"

namespace emm {

constexpr int kStatusLength = 3;

// Geometry of the split, chosen on the host (attend_shape in cache_ops.cuh).
struct AttendShape {
  uint32_t heads_cta;    // KV heads per CTA
  uint32_t head_groups;  // CTAs' worth of heads: ceil(H / heads_cta)
  uint32_t ntiles;       // tiles of eight query heads per KV head
  uint32_t subsets;      // token subsets of a unit, one warp each
  uint32_t tokens;       // tokens per unit: 16 * attend_tiles(D) * subsets
  uint32_t warps;        // heads_cta * ntiles * subsets
  uint32_t stages;       // tiles in a warp's ring
  int32_t block_shift;   // log2 of the block size where it is a power of two, else -1
  uint32_t grid;         // CTAs
  uint32_t items;        // num_seqs * head_groups
};

// What an item costs besides its units, in units: queries, the subsets' meeting, the result (measured: 3 us against
// 1.8 us for a unit of 32 tokens and 8 heads). 64 sequences of 128-8 191 tokens 80.6 us, 160 of up to 1 500 31.4; with 1
// 81.7 and 32.5, with 3 81.6 and 32.1.
constexpr uint32_t kItemCost = 2;

constexpr uint32_t kScoreTokens = 128;  // tokens of a warp's turn in attend_scores

struct AttendArgs {
  TokenSide pool;
  uint64_t layer_base;        // this layer's base address
  uint64_t query;             // [B, Hq, D], heads dense
  uint64_t out;               // the same
  uint64_t query_seq_stride;  // bytes
  uint64_t out_seq_stride;
  const int32_t *tables;
  uint64_t table_stride;      // entries
  const int32_t *lens;
  uint32_t num_seqs;
  uint32_t kv_heads;
  uint32_t group;             // query heads per kv head
  uint32_t max_len;
  float scale_log2;           // softmax scale * log2(e)
  uint32_t align;             // common alignment of query and out
  uint64_t score_base;        // [NB, H, BS] fp32, or 0
  uint64_t score_block_stride;
  AttendShape sh;
  // workspace
  float *part_o;              // [2 * grid][heads_cta * group][D]
  float2 *part_ml;            // [2 * grid][heads_cta * group]: reference, sum
  int2 *item_span;            // [items]: first and last CTA of an item
  int *cta_item;              // [grid]: the split item that this CTA finished, or -1
  float *lse;                 // [B, Hq], with scores
  float *logits;              // [B, Hq, logit_stride], with scores
  uint32_t *turns;            // [B + 1], with scores: turns of kScoreTokens tokens in all sequences before this one
  uint64_t logit_stride;
  int *status;
};

__device__ __forceinline__ uint32_t seq_length(const AttendArgs &a, uint32_t b, bool reporter) {
  const int32_t n = a.lens[b];
  if (n < 0 || (uint32_t)n > a.max_len) {
    if (reporter) report(a.status, kStatusLength, n);
    return n < 0 ? 0u : a.max_len;
  }
  return (uint32_t)n;
}

__device__ __forceinline__ uint32_t seq_units(const AttendArgs &a, uint32_t n) {
  return n == 0 ? 1u : (n + a.sh.tokens - 1) / a.sh.tokens;  // an empty sequence has one empty unit: its zeros
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void mma_k16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1, const float (&c)[4]) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}

__device__ __forceinline__ void mma_bf16_k16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                             uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  uint32_t y;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(y) : "f"(hi), "f"(lo));
  return y;
}
__device__ __forceinline__ uint32_t mul_half2(uint32_t a, uint32_t b) {
  uint32_t y;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(y) : "r"(a), "r"(b));
  return y;
}
// Two 32-bit values of lanes (row, 2 columns) of an 8x8 tile -> those of its transpose.
__device__ __forceinline__ void transpose8(float &x, float &y) {
  const uint32_t a = __float_as_uint(x), b = __float_as_uint(y);
  const uint32_t lo = transpose8(__byte_perm(a, b, 0x5410)), hi = transpose8(__byte_perm(a, b, 0x7632));
  x = __uint_as_float(__byte_perm(lo, hi, 0x5410));
  y = __uint_as_float(__byte_perm(lo, hi, 0x7632));
}
// Two 32-bit values as bf16 pairs whose sum they are to 2^-16: the first cut, the second what is left, rounded.
__device__ __forceinline__ void split_bf16(uint64_t x, uint32_t &hi, uint32_t &lo) {
  uint32_t a, b;
  split(x, a, b);
  hi = __byte_perm(a, b, 0x7632);
  split(add_pair(x, pair(__uint_as_float((a & 0xffff0000u) ^ 0x80000000u), __uint_as_float((b & 0xffff0000u) ^ 0x80000000u))), a, b);
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(lo) : "f"(__uint_as_float(b)), "f"(__uint_as_float(a)));
}
// N words from shared memory at a + kOff (aligned to N words, as the row format guarantees).
template <int N, int kOff>
__device__ __forceinline__ void lds_words(uint32_t (&w)[N], uint32_t a) {
  if constexpr (N == 1) {
    asm volatile("ld.shared.u32 %0, [%1+%2];" : "=r"(w[0]) : "r"(a), "n"(kOff));
  } else if constexpr (N == 2) {
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2+%3];" : "=r"(w[0]), "=r"(w[1]) : "r"(a), "n"(kOff));
  } else {
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4+%5];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                 : "r"(a), "n"(kOff));
    if constexpr (N == 8)
      asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4+%5];"
                   : "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                   : "r"(a), "n"(kOff + 16));
  }
}
// Four 8x8 matrices of 16-bit values, lane i giving the address of row i % 8 of matrix i / 8; kTrans: transposed.
template <bool kTrans, int kOff>
__device__ __forceinline__ void lds_matrices(uint32_t (&m)[4], uint32_t a) {
  if constexpr (kTrans)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4+%5];"
                 : "=r"(m[0]), "=r"(m[1]), "=r"(m[2]), "=r"(m[3])
                 : "r"(a), "n"(kOff));
  else
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4+%5];"
                 : "=r"(m[0]), "=r"(m[1]), "=r"(m[2]), "=r"(m[3])
                 : "r"(a), "n"(kOff));
}

// 16 bytes from global to shared memory, past L1.
__device__ __forceinline__ void copy16(uint32_t dst, uint64_t src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// Two of them, if `on` is not 0, without a branch.
template <int kOff0, int kOff1>
__device__ __forceinline__ void copy16_pair(uint32_t dst, uint64_t src0, uint64_t src1, uint32_t on) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.u32 p, %3, 0;\n"
      "@p cp.async.cg.shared.global [%0+%4], [%1], 16;\n"
      "@p cp.async.cg.shared.global [%0+%5], [%2], 16;\n"
      "}\n" ::"r"(dst), "l"(src0), "l"(src1), "r"(on), "n"(kOff0), "n"(kOff1)
      : "memory");
}
// A lane's share of a tile of 16 key and 16 value rows of R bytes: one chunk of 16 bytes in 32 of each plane.
template <int R, int J>
__device__ __forceinline__ void copy_tile(uint32_t dst, uint64_t k, uint64_t v, const uint32_t (&row_off)[(R + 31) / 32], uint32_t tail_lane) {
  copy16_pair<512 * J, 16 * R + 512 * J>(dst, k + row_off[J], v + row_off[J], (J + 1) * 32 <= R ? 1u : tail_lane);
  if constexpr (J + 1 < (R + 31) / 32) copy_tile<R, J + 1>(dst, k, v, row_off, tail_lane);
}
template <int kOff>
__device__ __forceinline__ void sts_word(uint32_t a, uint32_t v) {
  asm volatile("st.shared.u32 [%0+%1], %2;" ::"r"(a), "n"(kOff), "r"(v) : "memory");
}
template <int kOff>
__device__ __forceinline__ uint32_t lds_word(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1+%2];" : "=r"(v) : "r"(a), "n"(kOff));
  return v;
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

constexpr uint32_t kNib0 = 0x000f000fu, kNib1 = 0x00f000f0u;
// prmt selectors, from two words: their low (high) halves; those halves shifted down by eight bits, with bits above that
// the nibble masks drop
constexpr uint32_t kLoHalves = 0x5410u, kHiHalves = 0x7632u, kLoUpper = 0x5511u, kHiUpper = 0x7733u;
constexpr float kFirstRef = -3.40282347e38f;                  // reference before any token: no finite logit is less
constexpr float kLift = 8.f;            // p is held times 2^kLift, and is at most 2^6 of that: in fp16's range
constexpr float kWeightUnit = 0x1p96f;  // and times this in the products p s of the values
// What undoes the units of the value sums: a masked nibble is c * 2^-133 or c * 2^-129 as a bf16 subnormal.
constexpr float kUnitLo = 0x1p37f, kUnitHi = 0x1p33f;

// A CTA's share. The batch is a line on which every item takes kItemCost and then one place per unit; a CTA has the units
// whose places lie in its piece of the line.
struct Share {
  uint32_t b, hg, unit;  // first item and unit
  uint32_t place, end;   // place of that item's unit 0; end of the share
  uint32_t each, extra;  // the first `extra` CTAs have each + 1 places, the others each
};

// One CTA of eight warps per SM. A warp takes two tiles of 16 tokens at a time (one at D = 256, where its accumulators and
// queries fill the registers): their products, which depend on nothing of one another's, hide each other's latency
// better than twice the warps with half the registers did, and the loop around them is paid once.
constexpr int kAttendWarps = 8;
__host__ __device__ constexpr int attend_tiles(int D) { return D == 256 ? 1 : 2; }
// Slots of attend_tiles() tiles in a warp's ring: about 150 KB of an SM's shared memory.
__host__ __device__ constexpr int attend_stages(int D) { return D == 64 ? 6 : 4; }
__host__ __device__ constexpr int attend_slot_bytes(int D) { return attend_tiles(D) * 32 * q4_row_bytes(D) + 16; }

// Decode attention; see the top of the file.
template <typename T, int D, bool kScores>
__global__ void __launch_bounds__(kAttendWarps * 32, 1) attend_q4(const __grid_constant__ AttendArgs a) {
  constexpr int G = q4_groups(D), R = q4_row_bytes(D);
  constexpr int KW = D / 32;  // words of codes per lane and token, keys (two units of every group)
  constexpr int VW = D / 64;  // words of codes per lane and token, values (one unit of every group)
  constexpr int SW = (G + 1) / 2;  // words of a token's scales
  constexpr int kT = attend_tiles(D), kSlotBytes = attend_slot_bytes(D), kAttendStages = attend_stages(D);
  constexpr int kTile = 32 * R, kWords = kT * kTile;  // bytes of a tile; where a slot's words begin
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ Share share;
  __shared__ uint32_t scan[kAttendWarps];

  const AttendShape &sh = a.sh;
  const uint32_t tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  grid_launch_dependents();
  grid_dependency_wait();
  if (tid == 0) a.cta_item[blockIdx.x] = -1;
  // The line's length and this CTA's piece. A thread takes a run of consecutive sequences.
  {
    const uint32_t per = (a.num_seqs + blockDim.x - 1) / blockDim.x;
    const uint32_t b0 = min(a.num_seqs, tid * per), b1 = min(a.num_seqs, b0 + per);
    uint32_t mine = 0, n0 = 0;
    for (uint32_t b = b0; b < b1; ++b) {
      const uint32_t n = seq_length(a, b, blockIdx.x == 0);
      if (b == b0) n0 = n;
      mine += (seq_units(a, n) + kItemCost) * sh.head_groups;
    }
    uint32_t upto = mine;
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
      const uint32_t other = __shfl_up_sync(0xffffffffu, upto, m);
      if (lane >= m) upto += other;
    }
    if (lane == 31) scan[warp] = upto;
    __syncthreads();
    uint32_t before = 0, total = 0;
    for (uint32_t w = 0; w < blockDim.x / 32; ++w) {
      if (w < warp) before += scan[w];
      total += scan[w];
    }
    before += upto - mine;
    const uint32_t each = total / gridDim.x, extra = total - each * gridDim.x;
    const uint32_t first = each * blockIdx.x + min(blockIdx.x, extra);
    if (first >= total && tid == 0) share = Share{0, 0, 0, 0, 0, 0, 0};  // more CTAs than places
    if (before <= first && first < before + mine) {
      uint32_t at = before, n = n0, b = b0;
      for (;;) {
        const uint32_t u = (seq_units(a, n) + kItemCost) * sh.head_groups;
        if (first < at + u) break;
        at += u;
        n = seq_length(a, ++b, false);
      }
      const uint32_t one = seq_units(a, n) + kItemCost, r = (first - at) / one, rest = first - at - r * one;
      share.b = b;
      share.hg = r;
      share.unit = rest > kItemCost ? rest - kItemCost : 0;
      share.place = at + r * one + kItemCost;
      share.end = first + each + (blockIdx.x < extra ? 1 : 0);
      share.each = each;
      share.extra = extra;
    }
    __syncthreads();
    if (kScores && blockIdx.x == 0) {  // the same count for attend_scores
      uint32_t turns = 0;
      for (uint32_t b = b0; b < b1; ++b) turns += (seq_length(a, b, false) + kScoreTokens - 1) / kScoreTokens;
      uint32_t at = turns;
#pragma unroll
      for (int m = 1; m < 32; m <<= 1) {
        const uint32_t other = __shfl_up_sync(0xffffffffu, at, m);
        if (lane >= m) at += other;
      }
      if (lane == 31) scan[warp] = at;
      __syncthreads();
      at -= turns;
      for (uint32_t w = 0; w < warp; ++w) at += scan[w];
      if (tid == 0) a.turns[0] = 0;
      for (uint32_t b = b0; b < b1; ++b) a.turns[b + 1] = at += (seq_length(a, b, false) + kScoreTokens - 1) / kScoreTokens;
    }
  }
  const uint32_t end = share.end;
  uint32_t b = share.b, hg = share.hg, unit = share.unit, place = share.place;
  if (place + unit >= end) return;  // no unit of its own

  const uint32_t hl = warp % sh.heads_cta;                 // KV head within the CTA
  const uint32_t nt = warp / sh.heads_cta % sh.ntiles;     // tile of query heads
  const uint32_t sub = warp / (sh.heads_cta * sh.ntiles);  // token subset
  const uint32_t g = lane / 4, q4 = lane % 4, t_sub = sub * 16 * kT;

  // ---- loads: a ring of slots of kT tiles, 16 key rows and 16 value rows each, and a word per tile that says which tokens
  // count: kByLength, or a mask where a block lies outside the pool (read only once such a block was met)
  constexpr uint32_t kByLength = 0x10000u;
  constexpr int kChunks = R / 16, kCopies = (R + 31) / 32;  // 16-byte chunks of a row; per lane and plane of a tile
  const uint32_t ring = smem_u32(smem) + warp * kAttendStages * kSlotBytes, ring_end = ring + kAttendStages * kSlotBytes;
  uint32_t row_off[kCopies];  // chunk lane + 32 j of a plane: offset from its first row
#pragma unroll
  for (int j = 0; j < kCopies; ++j) {
    const uint32_t c = lane + 32 * j;
    row_off[j] = c / kChunks * (uint32_t)a.pool.token_stride + c % kChunks * 16;
  }
  const uint32_t tail_lane = R % 32 == 0 || lane < R % 32;  // has a chunk in the last, partial round
  const uint32_t shift = (uint32_t)sh.block_shift & 31u, block_mask = (1u << shift) - 1u;
  const bool paged = sh.block_shift >= 0;
  bool holes = false;              // a block outside the pool was met
  // Where the next slot's tokens lie. `run` slots from here on hold whole tiles of one block each, their blocks at hand
  // in `ids`; `after` more units of the item follow in the share.
  uint32_t ib = b, ihg = hg, iplace = place;
  uint32_t it = unit * sh.tokens + t_sub, in = seq_length(a, b, false), run = 0;
  uint32_t after = min(seq_units(a, in), end - place) - unit;
  uint64_t ibase = 0;              // this head's rows of block 0
  const int32_t *itab = nullptr;   // the sequence's table
  uint32_t window = 0;             // and its entries window + lane, window + 32 + lane
  int32_t ids = 0, ids_next = 0;
  bool ireal = false;              // whether this warp has a head there
  auto entry = [&](uint32_t i) { return itab[min(i + lane, (in - 1) >> shift)]; };
  auto enter = [&]() {
    const uint32_t h = ihg * sh.heads_cta + hl;
    ireal = h < a.kv_heads;
    ibase = a.layer_base + h * a.pool.head_stride;
    itab = a.tables + ib * a.table_stride;
    window = it >> shift;
    if (paged && in > 0) {
      ids = entry(window);
      ids_next = entry(window + 32);
    }
  };
  auto next_item = [&]() {
    iplace += seq_units(a, in) + kItemCost;
    if (iplace >= end) return;
    if (++ihg == sh.head_groups) {
      ihg = 0;
      in = seq_length(a, ++ib, false);
    }
    after = min(seq_units(a, in), end - iplace);
    it = t_sub;
    enter();
  };
  bool small = false;              // the next slot's tiles are whole, of blocks of less than 16 tokens in `ids`
  auto begin_run = [&]() {
    small = false;
    if (!paged || !ireal || it + 16 * kT > in) return;
    const uint32_t far = (it >> shift) - window;
    if (far >= 32) {
      if (far < 64) {  // a unit has at most 256 tokens: 32 blocks of 8
        window += 32;
        ids = ids_next;
      } else {
        window = it >> shift;
        ids = entry(window);
      }
      ids_next = entry(window + 32);
    }
    if (__any_sync(0xffffffffu, (uint32_t)ids >= a.pool.num_blocks)) return;
    // slots begin at multiples of 16 kT tokens, so a slot's blocks (32 at most) lie in one window
    if (shift < 4) {
      small = true;
      return;
    }
    const uint32_t whole = (in - it - 16 * kT) / sh.tokens + 1;
    const uint32_t known = (uint32_t)((((uint64_t)window + 32) << shift) - it + sh.tokens - 1) / sh.tokens;
    run = min(min(whole, known), after);
    after -= run;
  };
  // Tiles of smaller blocks, and those that are not 16 tokens, not all inside the pool or of blocks of no 2^k tokens.
  auto load_rest = [&](uint32_t slot) {
#pragma unroll 1
    for (uint32_t i = 0; i < kT; ++i) {
      const uint32_t t = it + 16 * i, to = slot + i * kTile;
      uint32_t word = kByLength;
      if (small) {
#pragma unroll
        for (int j = 0; j < kCopies; ++j) {
          const uint32_t c = min(lane + 32 * j, (uint32_t)(16 * kChunks - 1)), at = t + c / kChunks;
          const uint32_t id = (uint32_t)__shfl_sync(0xffffffffu, ids, (at >> shift) - window);
          const uint64_t k = ibase + (uint64_t)id * (uint32_t)a.pool.block_stride +
                             (uint64_t)(at & block_mask) * (uint32_t)a.pool.token_stride + c % kChunks * 16;
          if (lane + 32 * j < 16 * kChunks) {
            copy16(to + 16 * c, k);
            copy16(to + 16 * R + 16 * c, k + a.pool.plane_stride);
          }
        }
      } else if (t < in && ireal) {
        const uint32_t count = min(16u, in - t);
        auto row_at = [&](uint32_t row) -> uint64_t {
          const uint32_t blk = paged ? (t + row) >> shift : (t + row) / a.pool.block_size;
          const int32_t id = itab[blk];
          if ((uint32_t)id >= a.pool.num_blocks) {
            report(a.status, kStatusIdRange, id);
            return 0;
          }
          return ibase + (uint64_t)(uint32_t)id * a.pool.block_stride + (t + row - blk * a.pool.block_size) * a.pool.token_stride;
        };
        const uint32_t mask = __ballot_sync(0xffffffffu, lane < count && row_at(lane) != 0);
        if (mask != (1u << count) - 1u) {
          holes = true;
          word = mask;
        }
#pragma unroll 1
        for (uint32_t c = lane; c < count * kChunks; c += 32) {
          const uint64_t src = row_at(c / kChunks);
          if (src == 0) continue;
          copy16(to + 16 * c, src + c % kChunks * 16);
          copy16(to + 16 * R + 16 * c, src + a.pool.plane_stride + c % kChunks * 16);
        }
      }
      sts_word<kWords>(slot + 4 * i, word);
    }
    it += sh.tokens;
    if (--after == 0) next_item();
  };
  auto by_length = [&](uint32_t slot) {
#pragma unroll
    for (int i = 0; i < kT; ++i) sts_word<kWords>(slot + 4 * i, kByLength);
  };
  auto load = [&](uint32_t slot) {
    if (__builtin_expect(run == 0 && after > 0, 0)) {
      begin_run();
      if (run == 0) load_rest(slot);
    }
    if (run > 0) {
      if (__builtin_expect(holes, 0)) by_length(slot);  // the words may be an earlier tile's masks
#pragma unroll
      for (int i = 0; i < kT; ++i) {
        const uint32_t t = it + 16 * i;
        const uint32_t id = (uint32_t)__shfl_sync(0xffffffffu, ids, (t >> shift) - window);
        const uint64_t k = ibase + (uint64_t)id * (uint32_t)a.pool.block_stride +
                           (uint64_t)(t & block_mask) * (uint32_t)a.pool.token_stride;
        copy_tile<R, 0>(slot + i * kTile + 16 * lane, k, k + a.pool.plane_stride, row_off, tail_lane);
      }
      it += sh.tokens;
      if (__builtin_expect(--run == 0, 0) && after == 0) next_item();
    }
    copies_commit();  // an empty group at the end keeps the count
  };
  enter();
#pragma unroll 1
  for (uint32_t s = ring; s < ring_end; s += kSlotBytes) by_length(s);
  uint4 q_raw[G];  // eight channels of every group of the query row of this lane
  auto fetch_query = [&]() {
    const uint32_t h = hg * sh.heads_cta + hl, j = nt * 8 + g;
    const bool mine = h < a.kv_heads && j < a.group;
    const uint64_t src = a.query + b * a.query_seq_stride + ((uint64_t)(h * a.group + j) * D + 8 * q4) * 2;
#pragma unroll
    for (int r = 0; r < G; ++r) {
      q_raw[r] = make_uint4(0, 0, 0, 0);
      if (mine && a.align >= 16) {
        q_raw[r] = *reinterpret_cast<const uint4 *>(src + r * 64);
      } else if (mine) {
        const uint16_t *e = reinterpret_cast<const uint16_t *>(src + r * 64);
        q_raw[r] = make_uint4(e[0] | (uint32_t)e[1] << 16, e[2] | (uint32_t)e[3] << 16, e[4] | (uint32_t)e[5] << 16,
                              e[6] | (uint32_t)e[7] << 16);
      }
    }
  };
#pragma unroll 1
  for (uint32_t s = ring; s < ring_end - kSlotBytes; s += kSlotBytes) load(s);

  // Tokens are fragment rows in their order. Rows are R apart, an odd multiple of 16 bytes at D = 64 and 128: the value
  // loads and the matrix loads touch every bank once.
  const uint32_t tk = g;                             // key rows g and g + 8
  const uint32_t tv0 = 2 * q4, tv1 = 2 * q4 + 1;     // value rows: tokens tv0, tv1, tv0 + 8, tv1 + 8
  const uint32_t k_at = tk * R, v_at = (16 + tv0) * R;
  // Scales and offsets as 8x8 matrices. Keys: rows tokens; the two token halves, at D = 256 scales then offsets, else
  // the same columns twice (for the high and the low half of Q). Values: columns tokens; likewise by token half.
  const uint32_t mi = lane / 8, mt = lane % 8;
  const uint32_t km_at = (mt + 8 * (mi & 1)) * R + (G == 8 && mi >= 2 ? 2 * G : 0);
  const uint32_t vm_at = (16 + mt + 8 * (mi >> 1)) * R + (G == 8 && (mi & 1) ? 2 * G : 0);
  uint32_t slot = ring, slot_before = ring_end - kSlotBytes;  // the slot to compute on, and the one before it

  float *merge = reinterpret_cast<float *>(smem + sh.warps * kAttendStages * kSlotBytes);  // [(warps - warps/subsets)][8][D + 2]

  while (place < end) {
    const uint32_t n = seq_length(a, b, false), units = seq_units(a, n);
    const uint32_t unit0 = unit, count = min(units, end - place) - unit;
    const uint32_t h = hg * sh.heads_cta + hl;
    const bool active = h < a.kv_heads;
    const uint32_t j0 = nt * 8;  // first query head of the tile, within the group
    fetch_query();

    // ---- the queries of this tile as B fragments
    uint32_t qf[G][4];
    uint32_t qo[4];     // Q_r (offsets) and -8 Q_r (scales) as two halves: B fragments
    float c0, c1;       // logit factors of heads 2 q4, 2 q4 + 1
    {
      auto load8 = [&](float (&x)[8], int r) {
        const uint32_t w[4] = {q_raw[r].x, q_raw[r].y, q_raw[r].z, q_raw[r].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) unpack2<T>(w[i], x[2 * i], x[2 * i + 1]);
      };
      float top = 0.f;
#pragma unroll
      for (int r = 0; r < G; ++r) {
        float x[8];
        load8(x, r);
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(x[i]));
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // A power of two brings the head's largest |q| into [2^5, 2^6): 16 q (for the low nibbles) and 8 times a sum of 32
      // stay below fp16's largest, and smaller ones keep 11 bits down to 2^-19 of it.
      int ex = (int)((__float_as_uint(top) >> 23) & 255u) - 127 - 5;
      ex = top == 0.f ? 0 : (ex < -110 ? -110 : (ex > 123 ? 123 : ex));
      const float down = __uint_as_float((uint32_t)(127 - ex) << 23), up = __uint_as_float((uint32_t)(127 + ex) << 23);
      // k index of that product: scales of groups 0 .. G-1, then their offsets (G = 8: each 0 .. 7)
      const int r0 = G == 8 ? 2 * (int)q4 : (G == 4 ? 2 * (int)(q4 & 1) : 0);
      const bool scales = G == 4 ? q4 < 2 : q4 == 0;
      float pick0 = 0.f, pick1 = 0.f;
#pragma unroll
      for (int r = 0; r < G; ++r) {
        float x[8], sum = 0.f;
        load8(x, r);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          x[i] = __half2float(__float2half_rn(x[i] * down));
          sum += x[i];
        }
        qf[r][0] = pack_half2(16.f * x[0], 16.f * x[4]);
        qf[r][1] = pack_half2(x[1], x[5]);
        qf[r][2] = pack_half2(16.f * x[2], 16.f * x[6]);
        qf[r][3] = pack_half2(x[3], x[7]);
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        if (r == r0) pick0 = sum;
        if (r == r0 + 1) pick1 = sum;
      }
      const uint32_t hi = pack_half2(pick0, pick1);
      const float2 rounded = unpack_half2(hi);
      const uint32_t rest = pack_half2(pick0 - rounded.x, pick1 - rounded.y);
      const uint32_t eight = 0xc800c800u;  // -8, -8
      if constexpr (G == 8) {
        qo[0] = mul_half2(hi, eight);
        qo[1] = hi;
        qo[2] = mul_half2(rest, eight);
        qo[3] = rest;
      } else {
        const bool none = G == 2 && q4 >= 2;  // the row's padding
        qo[0] = none ? 0u : (scales ? mul_half2(hi, eight) : hi);
        qo[1] = none ? 0u : (scales ? mul_half2(rest, eight) : rest);
        qo[2] = qo[3] = 0;
      }
      const float c = up * a.scale_log2;
      c0 = __shfl_sync(0xffffffffu, c, 8 * q4);
      c1 = __shfl_sync(0xffffffffu, c, 8 * q4 + 4);
    }

    float acc[G][2][4], accx[4] = {0.f, 0.f, 0.f, 0.f}, accy[4] = {0.f, 0.f, 0.f, 0.f};  // accy: times 2^12
#pragma unroll
    for (int r = 0; r < G; ++r)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[r][i][k] = 0.f;
    float ref0 = kFirstRef, ref1 = kFirstRef, sum0 = 0.f, sum1 = 0.f;
    float *lg = nullptr;  // logits of head 2 q4; head 2 q4 + 1 lies one row further
    if constexpr (kScores)
      lg = a.logits + ((uint64_t)b * a.kv_heads * a.group + (uint64_t)h * a.group + j0 + 2 * q4) * a.logit_stride;
    const bool store0 = active && j0 + 2 * q4 < a.group, store1 = active && j0 + 2 * q4 + 1 < a.group;

    // Moves the references of this lane's two heads and everything held relative to them.
    auto rescale = [&](float to0, float to1) {
      const float f0 = ex2(ref0 - to0), f1 = ex2(ref1 - to1);
      ref0 = to0;
      ref1 = to1;
      sum0 *= f0;
      sum1 *= f1;
#pragma unroll
      for (int r = 0; r < G; ++r)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          acc[r][i][0] *= f0;
          acc[r][i][1] *= f1;
          acc[r][i][2] *= f0;
          acc[r][i][3] *= f1;
        }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        accx[i] *= i % 2 ? f1 : f0;
        accy[i] *= i % 2 ? f1 : f0;
      }
    };
    // Row r of accx holds the sums of p s_r, the offsets' row those of p o_r.
    auto side_sum = [&](int i) { return fmaf(accy[i], 0x1p-12f, accx[i]); };

    // Takes the -8 s of x = o + s (c - 8) out of the value sums so far. The tensor cores cut each sum of theirs short
    // rather than round it, by a share of its size, and sum p s c alone is much larger than what is left of it when the
    // values have no common sign: with a fixed number of tiles between two calls the loss stays below 2^-20 of sum p s c
    // however long the sequence. Every 64 tokens: one sequence of 131 071 tokens is off what 32-bit sums give by 2.4e-4
    // (two bf16 results that round a few values apart; every 256 tokens 4.9e-4, and 60.3 instead of 61.0 us).
    auto recentre = [&]() {
      const float s0 = -8.f * side_sum(0), s1 = -8.f * side_sum(1);
#pragma unroll
      for (int r = 0; r < G; ++r) {
        const float x0 = __shfl_sync(0xffffffffu, s0, 4 * r + q4), x1 = __shfl_sync(0xffffffffu, s1, 4 * r + q4);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          acc[r][i][0] = fmaf(x0, 1.f / kUnitLo, acc[r][i][0]);
          acc[r][i][1] = fmaf(x1, 1.f / kUnitLo, acc[r][i][1]);
          acc[r][i][2] = fmaf(x0, 1.f / kUnitHi, acc[r][i][2]);
          acc[r][i][3] = fmaf(x1, 1.f / kUnitHi, acc[r][i][3]);
        }
      }
      if (g < (uint32_t)G) accx[0] = accx[1] = accy[0] = accy[1] = 0.f;  // the scales' rows
    };
    constexpr uint32_t kRecentre = 4 / kT;  // slots between two calls

    int left = active ? (int)n - (int)(unit0 * sh.tokens + t_sub) : 0;  // tokens from this warp's next tile on
    // N tiles, the first at position n - left. kWhole: all their tokens count (mask is not read; else N = 1).
    auto tiles = [&](auto whole_tag, auto count_tag, const uint32_t base, const uint32_t mask) {
      constexpr bool kWhole = decltype(whole_tag)::value;
      constexpr int N = decltype(count_tag)::value;
      // ---- logits of 16 tokens each
      float l[N][4];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        uint32_t w0[KW], w1[KW], s0[SW], s1[SW], m[4];
        const uint32_t ka = base + i * kTile + k_at, kc = ka + q4 * (D / 8);
        lds_matrices<false, D / 2>(m, base + i * kTile + km_at);
        lds_words<KW, 0>(w0, kc);
        lds_words<KW, 8 * R>(w1, kc);
        lds_words<SW, D / 2>(s0, ka);
        lds_words<SW, 8 * R + D / 2>(s1, ka);
        float d0[4] = {0.f, 0.f, 0.f, 0.f};
        mma_k16(d0, m[0], m[1], m[2], m[3], qo[0], qo[1], d0);
        if constexpr (G == 8) mma_k16(d0, m[0], m[1], m[2], m[3], qo[2], qo[3], d0);
        float x[4];
#pragma unroll
        for (int r = 0; r < G; ++r) {
          const uint32_t sel = r % 2 ? kHiHalves : kLoHalves, up = r % 2 ? kHiUpper : kLoUpper;
          const uint32_t u0 = __byte_perm(w0[r / 2], w0[KW / 2 + r / 2], sel), u1 = __byte_perm(w1[r / 2], w1[KW / 2 + r / 2], sel);
          const uint32_t y0 = __byte_perm(w0[r / 2], w0[KW / 2 + r / 2], up), y1 = __byte_perm(w1[r / 2], w1[KW / 2 + r / 2], up);
          float d[4] = {0.f, 0.f, 0.f, 0.f};
          mma_k16(d, u0 & kNib0, u1 & kNib0, u0 & kNib1, u1 & kNib1, qf[r][0], qf[r][1], d);
          mma_k16(d, y0 & kNib0, y1 & kNib0, y0 & kNib1, y1 & kNib1, qf[r][2], qf[r][3], d);
          const float2 f0 = unpack_half2(s0[r / 2]), f1 = unpack_half2(s1[r / 2]);
          const float e0 = r % 2 ? f0.y : f0.x, e1 = r % 2 ? f1.y : f1.x;
          x[0] = r ? fmaf(e0, d[0], x[0]) : e0 * d[0];
          x[1] = r ? fmaf(e0, d[1], x[1]) : e0 * d[1];
          x[2] = r ? fmaf(e1, d[2], x[2]) : e1 * d[2];
          x[3] = r ? fmaf(e1, d[3], x[3]) : e1 * d[3];
        }
        l[i][0] = c0 * fmaf(x[0], 0x1p20f, d0[0]);
        l[i][1] = c1 * fmaf(x[1], 0x1p20f, d0[1]);
        l[i][2] = c0 * fmaf(x[2], 0x1p20f, d0[2]);
        l[i][3] = c1 * fmaf(x[3], 0x1p20f, d0[3]);
      }
      // ---- scales, offsets and codes of the value rows: tokens tv0, tv1, tv0 + 8, tv1 + 8
      uint32_t sv[N][4][SW], m[N][4], w[N][4][VW];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const uint32_t va = base + i * kTile + v_at, vc = va + g * (D / 16);
        lds_matrices<true, D / 2>(m[i], base + i * kTile + vm_at);
        lds_words<SW, D / 2>(sv[i][0], va);
        lds_words<SW, R + D / 2>(sv[i][1], va);
        lds_words<SW, 8 * R + D / 2>(sv[i][2], va);
        lds_words<SW, 9 * R + D / 2>(sv[i][3], va);
        lds_words<VW, 0>(w[i][0], vc);
        lds_words<VW, R>(w[i][1], vc);
        lds_words<VW, 8 * R>(w[i][2], vc);
        lds_words<VW, 9 * R>(w[i][3], vc);
      }
      if constexpr (!kWhole) {
        // Tokens that do not count: no weight, and no scale or offset that could be anything (0 * NaN).
        if (!(mask >> tk & 1)) l[0][0] = l[0][1] = -INFINITY;
        if (!(mask >> (tk + 8) & 1)) l[0][2] = l[0][3] = -INFINITY;
        const uint32_t t[4] = {tv0, tv1, tv0 + 8, tv1 + 8};
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (!(mask >> t[i] & 1)) {
            const uint32_t stay = i % 2 ? 0x0000ffffu : 0xffff0000u;
            m[0][i / 2 * 2] &= stay;
            m[0][i / 2 * 2 + 1] &= stay;
#pragma unroll
            for (int k = 0; k < SW; ++k) sv[0][i][k] = 0;
          }
      }
      if constexpr (kScores) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const uint32_t t = n - (uint32_t)left + 16 * i + tk;
          if (kWhole || (mask >> tk & 1)) {
            if (store0) lg[t] = l[i][0];
            if (store1) lg[a.logit_stride + t] = l[i][1];
          }
          if (kWhole || (mask >> (tk + 8) & 1)) {
            if (store0) lg[t + 8] = l[i][2];
            if (store1) lg[a.logit_stride + t + 8] = l[i][3];
          }
        }
      }
      // ---- weights; the reference follows the maximum only when it is left 2^6 behind
      float p[N][4], most = kFirstRef;
#pragma unroll
      for (int i = 0; i < N; ++i) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          p[i][k] = l[i][k] - (k % 2 ? ref1 : ref0);
          most = fmaxf(most, p[i][k]);
        }
      }
      if (__builtin_expect(__any_sync(0xffffffffu, most > kLift + 6.f), 0)) {
        float m0 = l[0][0], m1 = l[0][1];
#pragma unroll
        for (int i = 0; i < N; ++i) {
          m0 = fmaxf(m0, fmaxf(l[i][0], l[i][2]));
          m1 = fmaxf(m1, fmaxf(l[i][1], l[i][3]));
        }
#pragma unroll
        for (int s = 4; s < 32; s <<= 1) {
          m0 = fmaxf(m0, __shfl_xor_sync(0xffffffffu, m0, s));
          m1 = fmaxf(m1, __shfl_xor_sync(0xffffffffu, m1, s));
        }
        rescale(fmaxf(ref0, m0 - kLift), fmaxf(ref1, m1 - kLift));
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
          for (int k = 0; k < 4; ++k) p[i][k] = l[i][k] - (k % 2 ? ref1 : ref0);
      }
#pragma unroll
      for (int i = 0; i < N; ++i) {
#pragma unroll
        for (int k = 0; k < 4; ++k) p[i][k] = ex2(p[i][k]);
        sum0 += p[i][0] + p[i][2];
        sum1 += p[i][1] + p[i][3];
        transpose8(p[i][0], p[i][1]);  // from here on tokens tv0, tv1, tv0 + 8, tv1 + 8 of head g
        transpose8(p[i][2], p[i][3]);
      }
#pragma unroll
      for (int i = 0; i < N; ++i) {
        // ---- sums of p s_r and p o_r: rows r and G + r of accx and accy, p in two 11-bit parts
        {
          const uint32_t h01 = pack_half2(p[i][0], p[i][1]), h23 = pack_half2(p[i][2], p[i][3]);
          const float2 r01 = unpack_half2(h01), r23 = unpack_half2(h23);
          const uint32_t l01 = pack_half2((p[i][0] - r01.x) * 0x1p12f, (p[i][1] - r01.y) * 0x1p12f);
          const uint32_t l23 = pack_half2((p[i][2] - r23.x) * 0x1p12f, (p[i][3] - r23.y) * 0x1p12f);
          mma_k16(accx, m[i][0], m[i][1], m[i][2], m[i][3], h01, h23, accx);
          mma_k16(accy, m[i][0], m[i][1], m[i][2], m[i][3], l01, l23, accy);
        }
        // ---- values
        const uint64_t p01 = mul_pair(pair(p[i][0], p[i][1]), pair(kWeightUnit, kWeightUnit));
        const uint64_t p23 = mul_pair(pair(p[i][2], p[i][3]), pair(kWeightUnit, kWeightUnit));
#pragma unroll
        for (int r = 0; r < G; ++r) {
          const uint32_t sel = r % 2 ? kHiHalves : kLoHalves, up = r % 2 ? kHiUpper : kLoUpper;
          float sc[4];
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            const float2 f = unpack_half2(sv[i][t][r / 2]);
            sc[t] = r % 2 ? f.y : f.x;
          }
          uint32_t e0, e1, f0, f1;
          split_bf16(mul_pair(p01, pair(sc[0], sc[1])), e0, f0);
          split_bf16(mul_pair(p23, pair(sc[2], sc[3])), e1, f1);
          const uint32_t u01 = __byte_perm(w[i][0][r / 2], w[i][1][r / 2], sel), u23 = __byte_perm(w[i][2][r / 2], w[i][3][r / 2], sel);
          const uint32_t y01 = __byte_perm(w[i][0][r / 2], w[i][1][r / 2], up), y23 = __byte_perm(w[i][2][r / 2], w[i][3][r / 2], up);
          mma_bf16_k16(acc[r][0], u01 & kNib0, u01 & kNib1, u23 & kNib0, u23 & kNib1, e0, e1);
          mma_bf16_k16(acc[r][1], y01 & kNib0, y01 & kNib1, y23 & kNib0, y23 & kNib1, e0, e1);
          mma_bf16_k16(acc[r][0], u01 & kNib0, u01 & kNib1, u23 & kNib0, u23 & kNib1, f0, f1);
          mma_bf16_k16(acc[r][1], y01 & kNib0, y01 & kNib1, y23 & kNib0, y23 & kNib1, f0, f1);
        }
      }
    };

    for (uint32_t k = 0; k < count; ++k) {
      copies_wait<kAttendStages - 2>();
      __syncwarp();  // this slot's rows are there for every lane, and every lane has left the slot before
      load(slot_before);
      if (__builtin_expect(left >= 16 * kT && !holes, 1)) {
        tiles(std::true_type{}, std::integral_constant<int, kT>{}, slot, 0xffffu);
        left -= (int)sh.tokens;
      } else {
        const int next = left - (int)sh.tokens;
#pragma unroll 1
        for (uint32_t i = 0; i < kT && left > 0; ++i, left -= 16) {
          uint32_t mask = left >= 16 ? 0xffffu : (1u << left) - 1u;
          const uint32_t word = lds_word<kWords>(slot + 4 * i);
          if (word != kByLength) mask = word;
          if (mask) tiles(std::false_type{}, std::integral_constant<int, 1>{}, slot + i * kTile, mask);
        }
        left = next;
      }
      if (k % kRecentre == kRecentre - 1) recentre();
      slot_before = slot;
      slot += kSlotBytes;
      if (slot == ring_end) slot = ring;
    }

    // ---- the segment's result: o[r][i] of channel 32 r + 4 g + i, heads 2 q4 and 2 q4 + 1
#pragma unroll
    for (int s = 4; s < 32; s <<= 1) {
      sum0 += __shfl_xor_sync(0xffffffffu, sum0, s);
      sum1 += __shfl_xor_sync(0xffffffffu, sum1, s);
    }
#pragma unroll
    for (int r = 0; r < G; ++r) {
      const int so = G == 8 ? 4 * r : 4 * (G + r);  // lanes that hold the offsets' sums
      const float x0 = __shfl_sync(0xffffffffu, side_sum(G == 8 ? 2 : 0), so + q4) - 8.f * __shfl_sync(0xffffffffu, side_sum(0), 4 * r + q4);
      const float x1 = __shfl_sync(0xffffffffu, side_sum(G == 8 ? 3 : 1), so + q4) - 8.f * __shfl_sync(0xffffffffu, side_sum(1), 4 * r + q4);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        acc[r][i][0] = fmaf(acc[r][i][0], kUnitLo, x0);
        acc[r][i][1] = fmaf(acc[r][i][1], kUnitLo, x1);
        acc[r][i][2] = fmaf(acc[r][i][2], kUnitHi, x0);
        acc[r][i][3] = fmaf(acc[r][i][3], kUnitHi, x1);
      }
    }
    if (sh.subsets > 1) {
      // The subsets' results meet in the first subset's warp, through shared memory, one after the other.
      const uint32_t per = sh.heads_cta * sh.ntiles;
      float *slot = merge + (uint64_t)(warp % per + (sub ? sub - 1 : 0) * per) * 8 * (D + 2);
      if (sub) {
#pragma unroll
        for (int r = 0; r < G; ++r) {
          float *o0 = slot + (2 * q4) * (D + 2) + 32 * r + 4 * g, *o1 = o0 + (D + 2);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            *reinterpret_cast<float2 *>(o0 + 2 * i) = make_float2(acc[r][i][0], acc[r][i][2]);
            *reinterpret_cast<float2 *>(o1 + 2 * i) = make_float2(acc[r][i][1], acc[r][i][3]);
          }
        }
        if (g == 0) {
          *reinterpret_cast<float2 *>(slot + (2 * q4) * (D + 2) + D) = make_float2(ref0, sum0);
          *reinterpret_cast<float2 *>(slot + (2 * q4 + 1) * (D + 2) + D) = make_float2(ref1, sum1);
        }
      }
      __syncthreads();
      if (sub == 0) {
        for (uint32_t s = 1; s < sh.subsets; ++s) {
          const float *from = merge + (uint64_t)(warp % per + (s - 1) * per) * 8 * (D + 2);
          const float2 ml0 = *reinterpret_cast<const float2 *>(from + (2 * q4) * (D + 2) + D);
          const float2 ml1 = *reinterpret_cast<const float2 *>(from + (2 * q4 + 1) * (D + 2) + D);
          const float to0 = fmaxf(ref0, ml0.x), to1 = fmaxf(ref1, ml1.x);
          const float a0 = ex2(ref0 - to0), a1 = ex2(ref1 - to1), f0 = ex2(ml0.x - to0), f1 = ex2(ml1.x - to1);
          ref0 = to0;
          ref1 = to1;
          sum0 = sum0 * a0 + ml0.y * f0;
          sum1 = sum1 * a1 + ml1.y * f1;
#pragma unroll
          for (int r = 0; r < G; ++r) {
            const float *o0 = from + (2 * q4) * (D + 2) + 32 * r + 4 * g, *o1 = o0 + (D + 2);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const float2 v0 = *reinterpret_cast<const float2 *>(o0 + 2 * i), v1 = *reinterpret_cast<const float2 *>(o1 + 2 * i);
              acc[r][i][0] = acc[r][i][0] * a0 + v0.x * f0;
              acc[r][i][2] = acc[r][i][2] * a0 + v0.y * f0;
              acc[r][i][1] = acc[r][i][1] * a1 + v1.x * f1;
              acc[r][i][3] = acc[r][i][3] * a1 + v1.y * f1;
            }
          }
        }
      }
      __syncthreads();  // the buffer is free for the next segment
    }
    const bool whole = count == units;
    if (sub == 0 && active) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const uint32_t j = j0 + 2 * q4 + c;
        if (j >= a.group) continue;
        const float sum = c ? sum1 : sum0, ref = c ? ref1 : ref0;
        const uint64_t head = (uint64_t)h * a.group + j;
        if (whole) {
          const float inv = sum == 0.f ? 0.f : 1.f / sum;  // no token counts: zeros
          T *out = reinterpret_cast<T *>(a.out + b * a.out_seq_stride) + head * D + 4 * g;
#pragma unroll
          for (int r = 0; r < G; ++r) {
            if (a.align >= 8) {
              *reinterpret_cast<uint2 *>(out + 32 * r) = make_uint2(pack2<T>(acc[r][0][c] * inv, acc[r][0][2 + c] * inv),
                                                                    pack2<T>(acc[r][1][c] * inv, acc[r][1][2 + c] * inv));
            } else {
#pragma unroll
              for (int i = 0; i < 4; ++i) out[32 * r + i] = from_f32<T>(acc[r][i / 2][2 * (i % 2) + c] * inv);
            }
          }
          if (kScores && g == 0) a.lse[(uint64_t)b * a.kv_heads * a.group + head] = sum == 0.f ? INFINITY : ref + lg2(sum);
        } else {
          const uint64_t slot = 2ull * blockIdx.x + (unit0 == 0 ? 1 : 0);
          const uint64_t row = slot * sh.heads_cta * a.group + hl * a.group + j;
          float *o = a.part_o + row * D + 4 * g;
#pragma unroll
          for (int r = 0; r < G; ++r)
            *reinterpret_cast<float4 *>(o + 32 * r) = make_float4(acc[r][0][c], acc[r][0][2 + c], acc[r][1][c], acc[r][1][2 + c]);
          if (g == 0) a.part_ml[row] = make_float2(ref, sum);
        }
      }
    }
    if (tid == 0 && unit0 + count == units) {
      // This CTA ends the item: say which CTA has its first unit.
      const uint32_t long_ones = share.extra * (share.each + 1);
      const uint32_t from = place < long_ones ? place / (share.each + 1) : share.extra + (place - long_ones) / share.each;
      const uint32_t item = b * sh.head_groups + hg;
      a.item_span[item] = make_int2((int)from, (int)blockIdx.x);
      if (!whole) a.cta_item[blockIdx.x] = (int)item;
    }
    unit = 0;
    place += units + kItemCost;
    if (++hg == sh.head_groups) {
      hg = 0;
      ++b;
    }
  }
  copies_wait<0>();
}

// Adds the partial results of the items that several CTAs worked on. grid.x: items, or (by_cta) the CTAs that finished
// one; grid.y x kHeads: the query heads of an item. kJoinWarps / kHeads warps share a head's parts, all 16 where few items
// have many parts (131 071 tokens: the whole call 61.4 us, with two warps 69.5), two where many have few (64 sequences: 81
// us, with 16 warps 110.5). One round of loads each: latency bounds it.
constexpr int kJoinWarps = 16;

template <typename T, int D, int kHeads>
__global__ void __launch_bounds__(kJoinWarps * 32) attend_join(const __grid_constant__ AttendArgs a, const uint32_t by_cta) {
  constexpr int C = D / 32;                // channels per lane
  constexpr int W = kJoinWarps / kHeads;   // warps per head
  __shared__ float red[kJoinWarps][2];
  __shared__ float o[kJoinWarps][D];
  grid_launch_dependents();
  grid_dependency_wait();
  const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32, mine = warp % W;
  const uint32_t rows = a.sh.heads_cta * a.group, y = blockIdx.y * kHeads + warp / W;
  int item = (int)blockIdx.x;
  if (by_cta) item = a.cta_item[blockIdx.x];
  if (item < 0) return;
  const int2 span = a.item_span[item];
  if (span.x == span.y) return;
  const uint32_t b = item / a.sh.head_groups, hg = item % a.sh.head_groups;
  const uint32_t h = hg * a.sh.heads_cta + y / a.group;
  const bool real = y < rows && h < a.kv_heads;
  const uint32_t parts = real ? (uint32_t)(span.y - span.x) + 1 : 0;
  auto row_of = [&](uint32_t i) { return (2ull * (span.x + i) + (i == 0 ? 1 : 0)) * rows + y; };
  // Each warp runs through its parts with a maximum of its own; the warps' results meet in shared memory.
  float acc[C], sum = 0.f, top = kFirstRef;
#pragma unroll
  for (int c = 0; c < C; ++c) acc[c] = 0.f;
  constexpr int kAhead = D == 256 ? 5 : 10;  // parts whose loads are in flight together: all of 148 CTAs'
  for (uint32_t i0 = mine; i0 < parts; i0 += W * kAhead) {
    float v[kAhead][C];
    float2 ml[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const uint32_t i = i0 + u * W;
      ml[u] = make_float2(kFirstRef, 0.f);
#pragma unroll
      for (int c = 0; c < C; ++c) v[u][c] = 0.f;
      if (i < parts) {
        const uint64_t row = row_of(i);
        ml[u] = a.part_ml[row];
        const float *src = a.part_o + row * D + lane * C;
        if constexpr (C == 2) {
          *reinterpret_cast<float2 *>(v[u]) = *reinterpret_cast<const float2 *>(src);
        } else {
#pragma unroll
          for (int c = 0; c < C; c += 4) *reinterpret_cast<float4 *>(v[u] + c) = *reinterpret_cast<const float4 *>(src + c);
        }
      }
    }
    float to = top;
#pragma unroll
    for (int u = 0; u < kAhead; ++u) to = fmaxf(to, ml[u].x);
    const float f = ex2(top - to);
    top = to;
    sum *= f;
#pragma unroll
    for (int c = 0; c < C; ++c) acc[c] *= f;
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const float e = ex2(ml[u].x - to);
      sum = fmaf(ml[u].y, e, sum);
#pragma unroll
      for (int c = 0; c < C; ++c) acc[c] = fmaf(v[u][c], e, acc[c]);
    }
  }
  if constexpr (W > 1) {
#pragma unroll
    for (int c = 0; c < C; ++c) o[warp][lane * C + c] = acc[c];
    if (lane == 0) {
      red[warp][0] = top;
      red[warp][1] = sum;
    }
    __syncthreads();
    if (mine != 0) return;
    float to = top;
    for (int w = 0; w < W; ++w) to = fmaxf(to, red[warp + w][0]);
    sum = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c) acc[c] = 0.f;
    for (int w = 0; w < W; ++w) {
      const float e = ex2(red[warp + w][0] - to);
      sum = fmaf(red[warp + w][1], e, sum);
#pragma unroll
      for (int c = 0; c < C; ++c) acc[c] = fmaf(o[warp + w][lane * C + c], e, acc[c]);
    }
    top = to;
  }
  if (!real) return;
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const uint64_t head = (uint64_t)h * a.group + y % a.group;
  T *out = reinterpret_cast<T *>(a.out + b * a.out_seq_stride) + head * D + lane * C;
  if (a.align >= 4) {
#pragma unroll
    for (int c = 0; c < C; c += 2) reinterpret_cast<uint32_t *>(out)[c / 2] = pack2<T>(acc[c] * inv, acc[c + 1] * inv);
  } else {
#pragma unroll
    for (int c = 0; c < C; ++c) out[c] = from_f32<T>(acc[c] * inv);
  }
  if (lane == 0 && a.score_base)
    a.lse[(uint64_t)b * a.kv_heads * a.group + head] = sum == 0.f ? INFINITY : top + lg2(sum);
}

// Adds every token's weight to its score. A warp's turn is 128 tokens of a (sequence, KV head) pair, four a lane. Turns are
// counted over the tokens that there are (max_len may be far more), so every warp has the same number, give or take one: one
// or two of them at 131 K tokens and 8 heads, whose latencies are what the kernel costs.
// Six blocks an SM: with eight (32 registers) 160 sequences of up to 1 500 tokens take 35.1 instead of 32.1 us.
__global__ void __launch_bounds__(256, 6) attend_scores(const __grid_constant__ AttendArgs a) {
  grid_launch_dependents();
  grid_dependency_wait();
  const uint32_t lane = threadIdx.x % 32;
  const uint64_t total = (uint64_t)a.turns[a.num_seqs] * a.kv_heads, step = (uint64_t)gridDim.x * 8;
  for (uint64_t i = (uint64_t)blockIdx.x * 8 + threadIdx.x / 32; i < total; i += step) {
    const uint32_t turn = (uint32_t)(i / a.kv_heads), h = (uint32_t)(i - (uint64_t)turn * a.kv_heads);
    // The last sequence that begins at or before this turn: 32 are looked at together, then the 32 within a step of those.
    uint32_t b = 0;
    for (uint32_t width = a.num_seqs; width > 1;) {
      const uint32_t each = (width + 31) / 32, from = min(b + lane * each, a.num_seqs);
      const uint32_t below = __ballot_sync(0xffffffffu, lane * each < width && a.turns[from] <= turn);
      b += (31 - __clz(below)) * each;
      width = min(each, a.num_seqs - b);
    }
    const uint32_t n = seq_length(a, b, false), t = (turn - a.turns[b]) * kScoreTokens + lane * 4;
    if (t >= n) continue;
    const uint32_t bh = b * a.kv_heads + h;
    const uint64_t head = (uint64_t)bh * a.group;
    float *sc[4];
    float old[4], w[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < 4; ++k) {  // the entries' addresses and old values, while the logits come
      sc[k] = nullptr;
      old[k] = 0.f;
      if (t + k >= n) continue;
      const uint32_t blk = a.pool.block_shift >= 0 ? (t + k) >> a.pool.block_shift : (t + k) / a.pool.block_size;
      const int32_t id = a.tables[b * a.table_stride + blk];
      if ((uint32_t)id >= a.pool.num_blocks) continue;
      sc[k] = reinterpret_cast<float *>(a.score_base + (uint64_t)id * a.score_block_stride) + (uint64_t)h * a.pool.block_size +
              (t + k - blk * a.pool.block_size);
      old[k] = *sc[k];
    }
#pragma unroll 4
    for (uint32_t j = 0; j < a.group; ++j) {
      const float lse = a.lse[head + j];
      const float4 l = *reinterpret_cast<const float4 *>(a.logits + (head + j) * a.logit_stride + t);
      w[0] += ex2(l.x - lse);
      w[1] += ex2(l.y - lse);
      w[2] += ex2(l.z - lse);
      w[3] += ex2(l.w - lse);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (sc[k]) *sc[k] = old[k] + w[k];
  }
}

}  // namespace emm
