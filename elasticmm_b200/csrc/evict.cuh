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

constexpr int kSelectThreads = 256;

__global__ void __launch_bounds__(kSelectThreads) select_tokens(const __grid_constant__ SelectArgs a) {
  __shared__ uint32_t hist[256];
  __shared__ uint32_t pick[2];
  __shared__ uint32_t part[2][kSelectThreads / 32];
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
    for (uint32_t j = tid; j < a.keep; j += kSelectThreads) out[j] = j < n ? (int32_t)j : -1;
    return;
  }
  const uint64_t base = a.layers[l];
  auto key_at = [&](uint32_t t) -> uint32_t {
    const int32_t id = a.tables[b * a.table_stride + t / a.block_size];
    if ((uint32_t)id >= a.num_blocks) {
      report(a.status, kStatusIdRange, id);
      return 0;
    }
    return order_key(reinterpret_cast<const float *>(base + (uint64_t)id * a.block_stride)[h * a.block_size + t % a.block_size]);
  };
  const uint32_t first = a.sink, last = n - a.recent;  // candidates [first, last)
  uint32_t want = a.keep - a.sink - a.recent;           // of them
  // The want-th largest key, digit by digit from the top.
  uint32_t prefix = 0, mask = 0;
  for (int shift = 24; shift >= 0 && want > 0; shift -= 8) {
    hist[tid] = 0;
    __syncthreads();
    for (uint32_t t = first + tid; t < last; t += kSelectThreads) {
      const uint32_t k = key_at(t);
      if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & 255u], 1u);
    }
    __syncthreads();
    if (tid == 0) {
      uint32_t left = want, d = 255;
      while (d > 0 && hist[d] < left) left -= hist[d--];
      pick[0] = d;
      pick[1] = left;
    }
    __syncthreads();
    prefix |= pick[0] << shift;
    mask |= 255u << shift;
    want = pick[1];
    __syncthreads();
  }
  // Now `want` keys equal to prefix are taken, the earliest, and all keys above it.
  const bool none = a.keep == a.sink + a.recent;
  uint32_t done = 0, ties = 0;  // taken so far, equal keys met so far
  for (uint32_t t0 = 0; t0 < n; t0 += kSelectThreads) {
    const uint32_t t = t0 + tid;
    bool sure = false, tie = false;
    if (t < n) {
      if (t < first || t >= last) {
        sure = true;
      } else if (!none) {
        const uint32_t k = key_at(t);
        sure = k > prefix;
        tie = k == prefix;
      }
    }
    const uint32_t tb = __ballot_sync(0xffffffffu, tie);
    if (lane == 0) part[0][warp] = __popc(tb);
    __syncthreads();
    uint32_t before = ties, all = 0;
    for (uint32_t w = 0; w < kSelectThreads / 32; ++w) {
      if (w < warp) before += part[0][w];
      all += part[0][w];
    }
    const bool take = sure || (tie && before + __popc(tb & ((1u << lane) - 1)) < want);
    const uint32_t kb = __ballot_sync(0xffffffffu, take);
    if (lane == 0) part[1][warp] = __popc(kb);
    __syncthreads();
    uint32_t at = done, taken = 0;
    for (uint32_t w = 0; w < kSelectThreads / 32; ++w) {
      if (w < warp) at += part[1][w];
      taken += part[1][w];
    }
    at += __popc(kb & ((1u << lane) - 1));
    if (take && at < a.keep) out[at] = (int32_t)t;
    done += taken;
    ties += all;
    __syncthreads();
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

constexpr int kKeepThreads = 256;

// One CTA per (layer, sequence, head, plane). A chunk is as many rows as its threads hold vectors of type V.
template <typename V>
__global__ void __launch_bounds__(kKeepThreads) keep_rows(const __grid_constant__ KeepArgs a) {
  const uint32_t p = blockIdx.x % a.planes, bh = blockIdx.x / a.planes;
  const uint32_t h = bh % a.heads, b = bh / a.heads, l = blockIdx.y;
  const int32_t len = a.lens[b];
  if (len < 0 || (uint64_t)len > (uint64_t)a.table_width * a.pool.block_size) {
    if (threadIdx.x == 0 && h == 0) report(a.status, 3, len);
    return;
  }
  if ((uint32_t)len <= a.keep) return;
  const int32_t *index = a.index + (((uint64_t)l * a.num_seqs + b) * a.heads + h) * a.keep;
  const uint64_t base = a.pool.layers[l] + p * a.pool.plane_stride + h * a.pool.head_stride;
  auto row_at = [&](uint32_t t) -> uint64_t {
    const int32_t id = a.tables[b * a.table_stride + t / a.pool.block_size];
    if ((uint32_t)id >= a.pool.num_blocks) {
      report(a.status, kStatusIdRange, id);
      return 0;
    }
    return base + (uint64_t)id * a.pool.block_stride + (t % a.pool.block_size) * a.pool.token_stride;
  };
  const uint32_t vecs = a.row_bytes / (uint32_t)sizeof(V);
  const uint64_t total = (uint64_t)a.keep * vecs;
  for (uint64_t c = 0; c < total; c += kKeepThreads) {
    const uint64_t i = c + threadIdx.x;
    V v;
    uint64_t dst = 0;
    if (i < total) {
      const uint32_t j = (uint32_t)(i / vecs), part = (uint32_t)(i % vecs);
      const int32_t t = index[j];
      if (t > (int32_t)j && t < len) {
        const uint64_t src = row_at((uint32_t)t);
        dst = row_at(j);
        if (src && dst) {
          v = *reinterpret_cast<const V *>(src + part * sizeof(V));
          dst += part * sizeof(V);
        } else {
          dst = 0;
        }
      }
    }
    __syncthreads();
    if (dst) *reinterpret_cast<V *>(dst) = v;
    __syncthreads();
  }
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
