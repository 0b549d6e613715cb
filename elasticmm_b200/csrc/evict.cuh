// Eviction of tokens inside a request (sm_100a): which tokens stay, and their rows' move to the sequence's first places.
//
//   select_tokens  per (layer, sequence, kv head) of n > keep tokens: the first `sink`, the last `recent`, and of the
//                  others the keep - sink - recent with the largest accumulated weight; equal weights: the lower
//                  position; a NaN counts as -infinity. The index is ascending. n <= keep: 0 .. n-1, then -1.
//   keep_rows      position j of the sequence receives the row of position index[j]. index[j] >= j and ascending, so a
//                  chunk of destinations is free once the sources of all earlier chunks and its own have been read:
//                  one CTA walks its sequence in chunks, loads chunk i, waits for all its threads, then stores chunk i.
#pragma once
#include "q4.cuh"

namespace emm {

struct SelectArgs {
  const uint64_t *layers;       // score layers, [NB, H, BS] fp32 with dense blocks
  uint64_t block_stride;        // bytes
  uint32_t num_blocks;
  uint32_t block_size;
  int32_t block_shift;          // log2(block_size), or -1
  const int32_t *tables;
  uint64_t table_stride;
  uint32_t table_width;
  const int32_t *lens;
  uint32_t num_seqs;
  uint32_t heads;
  uint32_t keep, recent, sink;
  int32_t *index;               // [L, B, H, keep]
  int32_t *new_lens;            // [B]
  int *status;
};

// A float's order as an unsigned integer; -0 and 0 are equal, NaN is -infinity.
__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) x = -INFINITY;
  const uint32_t u = __float_as_uint(x + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// One CTA per (layer, sequence, head). The keys are read once into shared memory (kShared; a sequence that does not fit
// there reads its weights again in every pass, which L2 serves). The want-th largest is found by at most four radix passes
// of eight bits, fewer where a digit's bin is taken whole. What bounds it is latency: the table, the weights, the passes'
// barriers. So a digit is found by one warp, bins are cleared a pass ahead, and the index leaves after one more barrier.
// 2 048 CTAs of 3 000-4 096 tokens take 61 us, 336 of 9 000-20 001 take 43.
template <int kThreads, bool kShared>
__global__ void __launch_bounds__(kThreads) select_tokens(const __grid_constant__ SelectArgs a) {
  grid_launch_dependents();
  grid_dependency_wait();
  constexpr int kWarps = kThreads / 32, kAhead = 8;
  extern __shared__ uint32_t keys[];  // kShared: one per position
  __shared__ uint32_t hist[2][256];
  __shared__ uint32_t part[2][32];
  __shared__ uint32_t pick[3];
  const uint32_t h = blockIdx.x % a.heads, b = blockIdx.x / a.heads, l = blockIdx.y;
  const uint32_t tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  int32_t len = a.lens[b];
  if (len < 0 || (uint64_t)len > (uint64_t)a.table_width * a.block_size) {
    if (tid == 0 && h == 0) report(a.status, 3, len);
    len = 0;
  }
  const uint32_t n = (uint32_t)len;
  int32_t *out = a.index + (((uint64_t)l * a.num_seqs + b) * a.heads + h) * a.keep;
  if (l == 0 && h == 0 && tid == 0) a.new_lens[b] = (int32_t)min(n, a.keep);
  if (n <= a.keep) {
    for (uint32_t j = tid; j < a.keep; j += kThreads) out[j] = j < n ? (int32_t)j : -1;
    return;
  }
  const uint64_t base = a.layers[l] + (uint64_t)h * a.block_size * 4;
  const int32_t *table = a.tables + b * a.table_stride;
  const uint32_t first = a.sink, last = n - a.recent;  // candidates [first, last)
  uint32_t want = a.keep - a.sink - a.recent;           // of them

  auto block_at = [&](uint32_t t) -> int32_t { return table[a.block_shift >= 0 ? t >> a.block_shift : t / a.block_size]; };
  auto key_in = [&](uint32_t t, int32_t id) -> uint32_t {
    if ((uint32_t)id >= a.num_blocks) {
      report(a.status, kStatusIdRange, id);
      return 0;
    }
    const uint32_t place = a.block_shift >= 0 ? t & ((1u << a.block_shift) - 1u) : t % a.block_size;
    return order_key(reinterpret_cast<const float *>(base + (uint64_t)(uint32_t)id * a.block_stride)[place]);
  };
  auto key_at = [&](uint32_t t) -> uint32_t {
    if constexpr (kShared) return keys[t];
    return key_in(t, block_at(t));
  };
  if (tid < 256) hist[0][tid] = 0;
  if constexpr (kShared) {
    for (uint32_t t0 = tid; t0 < n; t0 += kThreads * kAhead) {
      int32_t id[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) id[u] = t0 + u * kThreads < n ? block_at(t0 + u * kThreads) : 0;
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (t0 + u * kThreads < n) keys[t0 + u * kThreads] = key_in(t0 + u * kThreads, id[u]);
    }
  }
  __syncthreads();
  uint32_t prefix = 0, mask = 0;  // the digits found, and where they stand
  const bool none = want == 0;
  for (int pass = 0; pass < 4 && !none; ++pass) {
    const int shift = 24 - 8 * pass;
    uint32_t *bins = hist[pass & 1];
    if (tid < 256) hist[~pass & 1][tid] = 0;
#pragma unroll 4
    for (uint32_t t = first + tid; t < last; t += kThreads) {
      const uint32_t k = key_at(t);
      if ((k & mask) == prefix) atomicAdd(&bins[k >> shift & 255u], 1u);
    }
    __syncthreads();
    if (warp == 0) {  // lane i has bins 255 - 8 i and the seven below: a scan from the largest digit down
      uint32_t c[8], mine = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) mine += c[i] = bins[255 - 8 * lane - i];
      uint32_t upto = mine;
#pragma unroll
      for (int m = 1; m < 32; m <<= 1) {
        const uint32_t other = __shfl_up_sync(0xffffffffu, upto, m);
        if (lane >= m) upto += other;
      }
      uint32_t above = upto - mine;
      if (above < want && want <= upto) {
        int i = 0;
#pragma unroll
        for (int k = 0; k < 7; ++k)
          if (i == k && above + c[k] < want) {
            above += c[k];
            i = k + 1;
          }
        uint32_t in_bin = c[0];
#pragma unroll
        for (int k = 1; k < 8; ++k)
          if (i == k) in_bin = c[k];
        pick[0] = 255 - 8 * lane - i;
        pick[1] = want - above;
        pick[2] = in_bin;
      }
    }
    __syncthreads();
    prefix |= pick[0] << shift;
    mask |= 255u << shift;
    want = pick[1];
    if (pick[2] == want) break;  // the whole bin is taken
  }
  // Taken: the ends, keys above the one found (as far as its digits go), and the `want` earliest equal to it. Warp w has a
  // run of positions, counts both kinds, and after a barrier knows where its part of the index begins.
  const uint32_t run = (n + kWarps * 32 - 1) / (kWarps * 32) * 32, begin = min(n, warp * run), end = min(n, begin + run);
  auto kinds = [&](uint32_t t, bool &sure, bool &tie) {
    sure = tie = false;
    if (t >= end) return;
    if (t < first || t >= last) {
      sure = true;
    } else if (!none) {
      const uint32_t k = key_at(t) & mask;
      sure = k > prefix;
      tie = k == prefix;
    }
  };
  uint32_t n_sure = 0, n_tie = 0;
  for (uint32_t t0 = begin; t0 < end; t0 += 32) {
    bool sure, tie;
    kinds(t0 + lane, sure, tie);
    n_sure += __popc(__ballot_sync(0xffffffffu, sure));
    n_tie += __popc(__ballot_sync(0xffffffffu, tie));
  }
  if (lane == 0) {
    part[0][warp] = n_sure;
    part[1][warp] = n_tie;
  }
  __syncthreads();
  uint32_t s_before = lane < warp ? part[0][lane] : 0, t_before = lane < warp ? part[1][lane] : 0;
  s_before = __reduce_add_sync(0xffffffffu, s_before);
  t_before = __reduce_add_sync(0xffffffffu, t_before);
  uint32_t at = s_before + min(t_before, want);
  for (uint32_t t0 = begin; t0 < end; t0 += 32) {
    const uint32_t below = (1u << lane) - 1u;
    bool sure, tie;
    kinds(t0 + lane, sure, tie);
    const uint32_t tb = __ballot_sync(0xffffffffu, tie);
    const bool take = sure || (tie && t_before + __popc(tb & below) < want);
    const uint32_t kb = __ballot_sync(0xffffffffu, take);
    const uint32_t j = at + __popc(kb & below);
    if (take && j < a.keep) out[j] = (int32_t)(t0 + lane);
    at += __popc(kb);
    t_before += __popc(tb);
  }
}

struct KeepArgs {
  TokenSide pool;
  uint32_t planes;
  uint32_t heads;
  uint32_t splits;     // CTAs that share a row's bytes
  uint32_t row_bytes;  // of one of them
  const int32_t *tables;
  uint64_t table_stride;
  uint32_t table_width;
  const int32_t *lens;
  uint32_t num_seqs;
  uint32_t keep;
  const int32_t *index;
  int *status;
};

// One CTA per (layer, sequence, head, plane), several where those are few; every kept row is read and written once, so HBM
// bounds it, and what counts is how many rows are in flight and how few instructions a row takes. 8 sequences of 3 000-4 096
// tokens cut to 2 048 in 32 layers of 8 heads of 128: 684 us (6.2 TB/s read and written; with the rows' blocks looked up in
// front of the copies 740). A ring of chunks in shared memory is filled by asynchronous copies. A thread has one vector of
// type V at a fixed place of a row and kKeepAhead rows of a chunk, and stores what it loaded itself.
// Before chunk i is stored, a barrier: every thread's loads up to chunk i have landed; those of later chunks, some still
// under way, read behind every destination so far.
// kPlain: rows of at most 256 vectors, blocks of 2^k tokens, strides below 2^32. Else positions are counted in segments of
// 256 vectors and everything is 64 bits wide.
constexpr int kKeepThreads = 256, kKeepAhead = 4, kKeepStages = 3;

template <typename V, bool kPlain>
__global__ void __launch_bounds__(kKeepThreads) keep_rows(const __grid_constant__ KeepArgs a) {
  grid_launch_dependents();
  grid_dependency_wait();
  using Pos = typename std::conditional<kPlain, uint32_t, uint64_t>::type;
  __shared__ __align__(16) V ring[kKeepStages][kKeepAhead][kKeepThreads];
  const uint32_t piece = blockIdx.x % a.splits, pbh = blockIdx.x / a.splits;
  const uint32_t p = pbh % a.planes, bh = pbh / a.planes;
  const uint32_t h = bh % a.heads, b = bh / a.heads, l = blockIdx.y;
  const int32_t len = a.lens[b];
  if (len < 0 || (uint64_t)len > (uint64_t)a.table_width * a.pool.block_size) {
    if (threadIdx.x == 0 && h == 0) report(a.status, 3, len);
    return;
  }
  if ((uint32_t)len <= a.keep) return;
  const int32_t *index = a.index + (((uint64_t)l * a.num_seqs + b) * a.heads + h) * a.keep;
  const int32_t *table = a.tables + b * a.table_stride;
  const uint32_t vecs = a.row_bytes / (uint32_t)sizeof(V);
  const uint32_t segments = kPlain ? 1u : (vecs + kKeepThreads - 1) / kKeepThreads, wide = min(vecs, (uint32_t)kKeepThreads);
  const uint32_t rows = kKeepThreads / wide;  // rows (or segments) side by side
  const uint32_t mine = threadIdx.x / wide, part = threadIdx.x % wide;
  const uint64_t base = a.pool.layers[l] + p * a.pool.plane_stride + h * a.pool.head_stride + piece * a.row_bytes + part * sizeof(V);
  // Row segments in order; a thread that has none counts from behind the end.
  const Pos total = (Pos)a.keep * segments, step = (Pos)rows * kKeepAhead, own = mine < rows ? (Pos)mine : total;
  auto block_of = [&](uint32_t t) -> int32_t { return table[kPlain ? t >> a.pool.block_shift : t / a.pool.block_size]; };
  auto row_in = [&](uint32_t t, int32_t entry) -> uint64_t {
    const uint32_t id = (uint32_t)entry;
    if (id >= a.pool.num_blocks) {
      report(a.status, kStatusIdRange, entry);
      return 0;
    }
    if constexpr (kPlain)
      return base + (uint64_t)id * (uint32_t)a.pool.block_stride +
             (uint64_t)(t & ((1u << a.pool.block_shift) - 1u)) * (uint32_t)a.pool.token_stride;
    else
      return base + (uint64_t)id * a.pool.block_stride + (uint64_t)(t % a.pool.block_size) * a.pool.token_stride;
  };
  // Bytes from a row's first segment to segment i's, or -1 where this thread has no vector in it.
  auto segment = [&](Pos i) -> int64_t {
    if constexpr (kPlain) return 0;
    const uint32_t seg = (uint32_t)(i % segments) * kKeepThreads;
    return part + seg < vecs ? (int64_t)seg * (int64_t)sizeof(V) : -1;
  };
  // What a row needs is fetched a chunk ahead of its use: its position, then the block of that, then its bytes.
  int32_t next[kKeepAhead];                      // positions of the chunk after the next to load
  int32_t from[kKeepAhead], from_block[kKeepAhead];  // the next to load: positions (-1: does not move) and blocks
  auto positions = [&](Pos first) {
#pragma unroll
    for (int u = 0; u < kKeepAhead; ++u) {
      const Pos i = first + u * rows;
      next[u] = i < total ? index[kPlain ? i : i / segments] : -1;
    }
  };
  auto blocks = [&](Pos first) {
#pragma unroll
    for (int u = 0; u < kKeepAhead; ++u) {
      const Pos i = first + u * rows;
      // a row that stays, or that the index does not put behind its place and inside the sequence, is left alone
      const bool on = next[u] > (int64_t)(kPlain ? i : i / segments) && next[u] < len && segment(i) >= 0;
      from[u] = on ? next[u] : -1;
      from_block[u] = on ? block_of((uint32_t)next[u]) : 0;
    }
  };
  uint32_t moves = 0;  // bit kKeepAhead s + u: row u of the chunk in stage s moves
  auto load = [&](Pos first, int s) {
    moves &= ~(((1u << kKeepAhead) - 1u) << (s * kKeepAhead));
#pragma unroll
    for (int u = 0; u < kKeepAhead; ++u) {
      if (from[u] >= 0) {
        const uint64_t src = row_in((uint32_t)from[u], from_block[u]);
        if (src) {
          const Pos i = first + u * rows;
          V *to = &ring[s][u][threadIdx.x];
          if constexpr (sizeof(V) >= 4)
            asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(smem_u32(to)), "l"(src + segment(i)), "n"((int)sizeof(V)) : "memory");
          else *to = *reinterpret_cast<const V *>(src + segment(i));
          moves |= 1u << (s * kKeepAhead + u);
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  auto ahead_of = [&](Pos first) {  // from here on `from` is of the chunk at first
    blocks(first);
    positions(first + step);
  };
  int32_t to_block[kKeepAhead];  // of the chunk to store
  auto places = [&](Pos first) {
#pragma unroll
    for (int u = 0; u < kKeepAhead; ++u) {
      const Pos i = first + u * rows;
      to_block[u] = i < total ? block_of((uint32_t)(kPlain ? i : i / segments)) : 0;
    }
  };
  positions(own);
  ahead_of(own);
  places(own);
#pragma unroll
  for (int s = 0; s < kKeepStages - 1; ++s) {
    load(own + s * step, s);
    ahead_of(own + (s + 1) * step);
  }
  int stage = 0, ahead = kKeepStages - 1;
  const Pos chunks = (total + step - 1) / step;
  Pos first = own;
#pragma unroll 1
  for (Pos c = 0; c < chunks; ++c, first += step) {
    load(first + (kKeepStages - 1) * step, ahead);
    ahead_of(first + kKeepStages * step);
    uint64_t dst[kKeepAhead];
#pragma unroll
    for (int u = 0; u < kKeepAhead; ++u) {
      const Pos i = first + u * rows;
      dst[u] = 0;
      if (moves >> (stage * kKeepAhead + u) & 1) {
        dst[u] = row_in((uint32_t)(kPlain ? i : i / segments), to_block[u]);
        if (!kPlain && dst[u]) dst[u] += segment(i);
      }
    }
    places(first + step);
    asm volatile("cp.async.wait_group %0;" ::"n"(kKeepStages - 1) : "memory");
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kKeepAhead; ++u)
      if (dst[u]) *reinterpret_cast<V *>(dst[u]) = ring[stage][u][threadIdx.x];
    stage = stage + 1 == kKeepStages ? 0 : stage + 1;
    ahead = ahead + 1 == kKeepStages ? 0 : ahead + 1;
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// Sets the weights of newly written tokens to zero in all layers (grid.y) and heads: a slot that held an evicted or
// freed token starts over. Padding slots are skipped, slots outside the pool recorded.
__global__ void __launch_bounds__(256)
reset_scores(const uint64_t *layers, uint64_t block_stride, uint32_t num_blocks, uint32_t block_size, uint32_t heads,
             const int64_t *slots, uint64_t num_tokens, int *status) {
  grid_launch_dependents();
  grid_dependency_wait();
  const uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= num_tokens * heads) return;
  const uint64_t t = i / heads;
  const uint32_t h = (uint32_t)(i - t * heads);
  const int64_t slot = slots[t];
  if (slot < 0) return;
  const uint64_t blk = (uint64_t)slot / block_size;
  if (blk >= num_blocks) {
    if (h == 0) report(status, kStatusIdRange, slot);
    return;
  }
  reinterpret_cast<float *>(layers[blockIdx.y] + blk * block_stride)[h * block_size + ((uint64_t)slot - blk * block_size)] = 0.f;
}

}  // namespace emm
