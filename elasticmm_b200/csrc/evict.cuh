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

// One CTA per (layer, sequence, head). Warp w of a tile of 16 * kThreads positions has positions w * 512 .. + 511, 16 keys
// in each lane's registers; the want-th largest key is found by three radix passes of 11, 11 and 10 bits over
// histograms in shared memory. A sequence of one tile reads its weights once; a longer one reads them again in every
// pass, which L2 serves. What bounds it is latency (table, weight, three passes), so the host takes as few
// threads as hold the longest sequence, and as many CTAs share an SM.
constexpr int kSelectKeys = 16, kSelectBins = 2048;

template <int kThreads>
__global__ void __launch_bounds__(kThreads, kThreads == 1024 ? 1 : 1536 / kThreads) select_tokens(const __grid_constant__ SelectArgs a) {
  constexpr int kWarps = kThreads / 32, kBins = kSelectBins / kThreads, kTile = kThreads * kSelectKeys;
  __shared__ uint32_t hist[kSelectBins];
  __shared__ uint32_t part[2][kWarps];
  __shared__ uint32_t pick[2];
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
  const bool none = want == 0;

  uint32_t keys[kSelectKeys];
  auto load = [&](uint32_t tile) {
    int32_t id[kSelectKeys];
#pragma unroll
    for (int u = 0; u < kSelectKeys; ++u) {
      const uint32_t t = tile + warp * (32 * kSelectKeys) + u * 32 + lane;
      id[u] = -1;
      if (t < n) id[u] = table[a.block_shift >= 0 ? t >> a.block_shift : t / a.block_size];
    }
#pragma unroll
    for (int u = 0; u < kSelectKeys; ++u) {
      const uint32_t t = tile + warp * (32 * kSelectKeys) + u * 32 + lane;
      keys[u] = 0;
      if (t >= n) continue;
      if ((uint32_t)id[u] >= a.num_blocks) {
        report(a.status, kStatusIdRange, id[u]);
        continue;
      }
      const uint32_t place = a.block_shift >= 0 ? t & ((1u << a.block_shift) - 1u) : t % a.block_size;
      keys[u] = order_key(reinterpret_cast<const float *>(base + (uint64_t)(uint32_t)id[u] * a.block_stride)[place]);
    }
  };
  const bool one_tile = n <= kTile;
  load(0);
  uint32_t prefix = 0, mask = 0;  // the digits found, and where they stand
  for (int pass = 0; pass < 3 && !none; ++pass) {
    const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0), bits = pass == 2 ? 10 : 11;
#pragma unroll
    for (int i = 0; i < kBins; ++i) hist[i * kThreads + tid] = 0;
    __syncthreads();
    for (uint32_t tile = 0; tile < n; tile += kTile) {
      if (!one_tile) load(tile);
#pragma unroll
      for (int u = 0; u < kSelectKeys; ++u) {
        const uint32_t t = tile + warp * (32 * kSelectKeys) + u * 32 + lane;
        if (t >= first && t < last && (keys[u] & mask) == prefix) atomicAdd(&hist[keys[u] >> shift & ((1u << bits) - 1u)], 1u);
      }
    }
    __syncthreads();
    // Thread t has bins 2047 - kBins t and the ones below it: a scan from the largest digit down.
    uint32_t mine = 0;
#pragma unroll
    for (int i = 0; i < kBins; ++i) mine += hist[kSelectBins - 1 - (tid * kBins + i)];
    uint32_t upto = mine;
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
      const uint32_t other = __shfl_up_sync(0xffffffffu, upto, m);
      if (lane >= m) upto += other;
    }
    if (lane == 31) part[0][warp] = upto;
    __syncthreads();
    uint32_t above = upto - mine;
    for (uint32_t w = 0; w < warp; ++w) above += part[0][w];
    if (above < want && want <= above + mine) {
      uint32_t d = kSelectBins - 1 - tid * kBins;
      while (above + hist[d] < want) above += hist[d--];
      pick[0] = d;
      pick[1] = want - above;
    }
    __syncthreads();
    prefix |= pick[0] << shift;
    mask |= ((1u << bits) - 1u) << shift;
    want = pick[1];
  }
  // Taken: the ends, keys above the one found, and the `want` earliest equal to it.
  uint32_t done = 0, ties = 0;  // in the tiles before
  for (uint32_t tile = 0; tile < n; tile += kTile) {
    if (!one_tile) load(tile);
    uint32_t sure = 0, tie = 0;  // bit u: this lane's key u
    uint32_t n_sure = 0, n_tie = 0;
#pragma unroll
    for (int u = 0; u < kSelectKeys; ++u) {
      const uint32_t t = tile + warp * (32 * kSelectKeys) + u * 32 + lane;
      const bool in = t < n, end = in && (t < first || t >= last), mid = in && !end && !none;
      if (end || (mid && keys[u] > prefix)) sure |= 1u << u;
      if (mid && keys[u] == prefix) tie |= 1u << u;
      n_sure += __popc(__ballot_sync(0xffffffffu, sure >> u & 1));
      n_tie += __popc(__ballot_sync(0xffffffffu, tie >> u & 1));
    }
    __syncthreads();
    if (lane == 0) {
      part[0][warp] = n_sure;
      part[1][warp] = n_tie;
    }
    __syncthreads();
    uint32_t s_before = 0, t_before = ties, s_all = 0, t_all = 0;
    for (uint32_t w = 0; w < kWarps; ++w) {
      if (w < warp) {
        s_before += part[0][w];
        t_before += part[1][w];
      }
      s_all += part[0][w];
      t_all += part[1][w];
    }
    // Of the ties before this warp, the first `want` are taken; done counts what earlier tiles took.
    uint32_t at = done + s_before + min(t_before, want) - min(ties, want);
#pragma unroll
    for (int u = 0; u < kSelectKeys; ++u) {
      const uint32_t below = (1u << lane) - 1u;
      const uint32_t tb = __ballot_sync(0xffffffffu, tie >> u & 1);
      const bool take = (sure >> u & 1) || ((tie >> u & 1) && t_before + __popc(tb & below) < want);
      const uint32_t kb = __ballot_sync(0xffffffffu, take);
      const uint32_t j = at + __popc(kb & below);
      if (take && j < a.keep) out[j] = (int32_t)(tile + warp * (32 * kSelectKeys) + u * 32 + lane);
      at += __popc(kb);
      t_before += __popc(tb);
    }
    done += s_all + min(ties + t_all, want) - min(ties, want);
    ties += t_all;
  }
}

struct KeepArgs {
  TokenSide pool;
  uint32_t planes;
  uint32_t heads;
  uint32_t row_bytes;
  const int32_t *tables;
  uint64_t table_stride;
  uint32_t table_width;
  const int32_t *lens;
  uint32_t num_seqs;
  uint32_t keep;
  const int32_t *index;
  int *status;
};

// One CTA per (layer, sequence, head, plane); every kept row is read and written once, so HBM bounds it, and what counts is
// how many rows are in flight and how few instructions a row takes (300 for two vectors, with 64-bit positions and
// divisions, held the kernel to 3.6 TB/s). A ring of chunks in shared memory is filled by asynchronous copies. A thread has
// one vector of type V at a fixed place of a row and kKeepAhead rows of a chunk, and stores what it loaded itself.
// Before chunk i is stored, a barrier: every thread's loads up to chunk i have landed; those of later chunks, some still
// under way, read behind every destination so far.
// kPlain: rows of at most 256 vectors, blocks of 2^k tokens, strides below 2^32. Else positions are counted in segments of
// 256 vectors and everything is 64 bits wide.
constexpr int kKeepThreads = 256, kKeepAhead = 4, kKeepStages = 3;

template <typename V, bool kPlain>
__global__ void __launch_bounds__(kKeepThreads) keep_rows(const __grid_constant__ KeepArgs a) {
  using Pos = typename std::conditional<kPlain, uint32_t, uint64_t>::type;
  __shared__ __align__(16) V ring[kKeepStages][kKeepAhead][kKeepThreads];
  const uint32_t p = blockIdx.x % a.planes, bh = blockIdx.x / a.planes;
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
  const uint64_t base = a.pool.layers[l] + p * a.pool.plane_stride + h * a.pool.head_stride + part * sizeof(V);
  // Row segments in order; a thread that has none counts from behind the end.
  const Pos total = (Pos)a.keep * segments, step = (Pos)rows * kKeepAhead, own = mine < rows ? (Pos)mine : total;
  auto row_at = [&](uint32_t t) -> uint64_t {
    const uint32_t blk = kPlain ? t >> a.pool.block_shift : t / a.pool.block_size;
    const uint32_t id = (uint32_t)table[blk];
    if (id >= a.pool.num_blocks) {
      report(a.status, kStatusIdRange, (int32_t)id);
      return 0;
    }
    if constexpr (kPlain)
      return base + (uint64_t)id * (uint32_t)a.pool.block_stride +
             (uint64_t)(t & ((1u << a.pool.block_shift) - 1u)) * (uint32_t)a.pool.token_stride;
    else
      return base + (uint64_t)id * a.pool.block_stride + (uint64_t)(t - blk * a.pool.block_size) * a.pool.token_stride;
  };
  // Bytes from a row's first segment to segment i's, or -1 where this thread has no vector in it.
  auto segment = [&](Pos i) -> int64_t {
    if constexpr (kPlain) return 0;
    const uint32_t seg = (uint32_t)(i % segments) * kKeepThreads;
    return part + seg < vecs ? (int64_t)seg * (int64_t)sizeof(V) : -1;
  };
  int32_t from[kKeepAhead];  // positions of the next chunk to load
  auto positions = [&](Pos first) {
#pragma unroll
    for (int u = 0; u < kKeepAhead; ++u) {
      const Pos i = first + u * rows;
      from[u] = i < total ? index[kPlain ? i : i / segments] : -1;
    }
  };
  uint32_t moves = 0;  // bit kKeepAhead s + u: row u of the chunk in stage s moves
  auto load = [&](Pos first, int s) {
    moves &= ~(((1u << kKeepAhead) - 1u) << (s * kKeepAhead));
#pragma unroll
    for (int u = 0; u < kKeepAhead; ++u) {
      const Pos i = first + u * rows;
      const uint32_t j = (uint32_t)(kPlain ? i : i / segments);
      // a row that stays, or that the index does not put behind its place and inside the sequence, is left alone
      if (from[u] > (int64_t)j && from[u] < len && segment(i) >= 0) {
        const uint64_t src = row_at((uint32_t)from[u]);
        if (src) {
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
  positions(own);
#pragma unroll
  for (int s = 0; s < kKeepStages - 1; ++s) {
    load(own + s * step, s);
    positions(own + (s + 1) * step);
  }
  int stage = 0, ahead = kKeepStages - 1;
  const Pos chunks = (total + step - 1) / step;
  Pos first = own;
#pragma unroll 1
  for (Pos c = 0; c < chunks; ++c, first += step) {
    load(first + (kKeepStages - 1) * step, ahead);
    positions(first + kKeepStages * step);
    uint64_t dst[kKeepAhead];
#pragma unroll
    for (int u = 0; u < kKeepAhead; ++u) {
      const Pos i = first + u * rows;
      dst[u] = 0;
      if (moves >> (stage * kKeepAhead + u) & 1) {
        dst[u] = row_at((uint32_t)(kPlain ? i : i / segments));
        if (!kPlain && dst[u]) dst[u] += segment(i);
      }
    }
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
