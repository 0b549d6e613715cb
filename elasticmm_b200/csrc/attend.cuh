// Decode attention over a 4-bit paged cache (sm_100a): one query token per sequence.
//
//   l[t] = scale * q . k[t]      p = softmax(l) over the sequence's tokens      out = sum_t p[t] v[t]
//   weights (optional): score[block of t][kv head][place of t] += sum of p[t] over the query heads of the kv head
#pragma once
#include "q4.cuh"

namespace emm {

constexpr int kStatusLength = 3;

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
  uint64_t score_base;        // [NB, H, BS] fp32, or 0
  uint64_t score_block_stride;
  float *logits;              // workspace [B, Hq, max_len]
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

// Block of position t, or -1 (reported) for an id outside the pool.
__device__ __forceinline__ int32_t block_of(const AttendArgs &a, uint32_t b, uint32_t t, bool reporter) {
  const int32_t id = a.tables[b * a.table_stride + t / a.pool.block_size];
  if ((uint32_t)id >= a.pool.num_blocks) {
    if (reporter) report(a.status, kStatusIdRange, id);
    return -1;
  }
  return id;
}

template <int D>
__device__ __forceinline__ float q4_value(const uint8_t *row, uint32_t d) {
  constexpr uint32_t G = q4_groups(D);
  const uint32_t r = d / 32, u = d % 32 / 4, i = d % 4;
  const uint32_t code = *reinterpret_cast<const uint16_t *>(row + 2 * (u * G + r));
  const float s = __half2float(*reinterpret_cast<const __half *>(row + D / 2 + 2 * r));
  const float o = __half2float(*reinterpret_cast<const __half *>(row + D / 2 + 2 * G + 2 * r));
  return o + s * ((float)(int)((code >> (4 * i)) & 15u) - 8.f);
}

// One CTA per (sequence, kv head): logits into the workspace, then the weights, then the weighted sum by channel.
template <typename T, int D>
__global__ void __launch_bounds__(256) attend_q4(const __grid_constant__ AttendArgs a) {
  __shared__ float qs[64 * 256 / 4];  // 16 heads of 256 channels at a time
  __shared__ float red[8], stat[2 * 64];
  const uint32_t b = blockIdx.x / a.kv_heads, h = blockIdx.x % a.kv_heads;
  const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint32_t n = seq_length(a, b, threadIdx.x == 0 && h == 0);
  const uint32_t heads = a.kv_heads * a.group;
  float *lg = a.logits + ((uint64_t)b * heads + h * a.group) * a.max_len;
  auto row_of = [&](uint32_t t, int32_t id, uint32_t plane) {
    return reinterpret_cast<const uint8_t *>(a.layer_base + plane * a.pool.plane_stride + (uint64_t)id * a.pool.block_stride +
                                             (t % a.pool.block_size) * a.pool.token_stride + h * a.pool.head_stride);
  };
  for (uint32_t j0 = 0; j0 < a.group; j0 += 16) {
    const uint32_t nj = min(16u, a.group - j0);
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < nj * D; i += 256)
      qs[i] = to_f32<T>(reinterpret_cast<const T *>(a.query + b * a.query_seq_stride)[(h * a.group + j0) * D + i]);
    __syncthreads();
    for (uint32_t t = warp; t < n; t += 8) {
      const int32_t id = block_of(a, b, t, lane == 0);
      float k[D / 32];
      if (id >= 0)
        for (uint32_t i = 0; i < D / 32; ++i) k[i] = q4_value<D>(row_of(t, id, 0), i * 32 + lane);
      for (uint32_t j = 0; j < nj; ++j) {
        float s = 0.f;
        if (id >= 0)
          for (uint32_t i = 0; i < D / 32; ++i) s += k[i] * qs[j * D + i * 32 + lane];
        for (int m = 16; m; m >>= 1) s += __shfl_xor_sync(0xffffffffu, s, m);
        if (lane == 0) lg[(uint64_t)(j0 + j) * a.max_len + t] = id < 0 ? -INFINITY : s * a.scale_log2;
      }
    }
  }
  __syncthreads();
  for (uint32_t j = 0; j < a.group; ++j) {
    float m = -1e30f, z = 0.f;
    for (uint32_t t = threadIdx.x; t < n; t += 256) m = fmaxf(m, lg[(uint64_t)j * a.max_len + t]);
    for (int k = 16; k; k >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, k));
    if (lane == 0) red[warp] = m;
    __syncthreads();
    for (int k = 0; k < 8; ++k) m = fmaxf(m, red[k]);
    __syncthreads();
    for (uint32_t t = threadIdx.x; t < n; t += 256) z += exp2f(lg[(uint64_t)j * a.max_len + t] - m);
    for (int k = 16; k; k >>= 1) z += __shfl_xor_sync(0xffffffffu, z, k);
    if (lane == 0) red[warp] = z;
    __syncthreads();
    if (threadIdx.x == 0) {
      z = 0.f;
      for (int k = 0; k < 8; ++k) z += red[k];
      stat[2 * j] = m;
      stat[2 * j + 1] = z > 0.f ? 1.f / z : (z == 0.f ? 0.f : z);
    }
    __syncthreads();
    for (uint32_t t = threadIdx.x; t < n; t += 256) {
      float &l = lg[(uint64_t)j * a.max_len + t];
      l = exp2f(l - stat[2 * j]) * stat[2 * j + 1];
    }
  }
  __syncthreads();
  if (a.score_base) {
    for (uint32_t t = threadIdx.x; t < n; t += 256) {
      const int32_t id = block_of(a, b, t, false);
      if (id < 0) continue;
      float w = 0.f;
      for (uint32_t j = 0; j < a.group; ++j) w += lg[(uint64_t)j * a.max_len + t];
      float *sc = reinterpret_cast<float *>(a.score_base + (uint64_t)id * a.score_block_stride) + h * a.pool.block_size +
                  t % a.pool.block_size;
      *sc += w;
    }
  }
  for (uint32_t i = threadIdx.x; i < a.group * D; i += 256) {
    const uint32_t j = i / D, d = i % D;
    float acc = 0.f;
    for (uint32_t t = 0; t < n; ++t) {
      const int32_t id = block_of(a, b, t, false);
      if (id >= 0) acc += lg[(uint64_t)j * a.max_len + t] * q4_value<D>(row_of(t, id, 1), d);
    }
    reinterpret_cast<T *>(a.out + b * a.out_seq_stride)[(h * a.group + j) * D + d] = from_f32<T>(acc);
  }
}

}  // namespace emm
