// The 4-bit cache row and the kernels that write it from 16-bit keys/values and read it back (sm_100a).
//
// A row holds one token of one KV head: D channels (64, 128 or 256) in D/32 groups of 32. Group r has a scale s and an
// offset o, both fp16, and channel x is the code c in 0..15 that stands for o + s * (c - 8):
//
//   lo, hi = min, max of the group, clamped to +-65504       s = fp16((hi - lo) / 15)       o = fp16(lo + 8 s)
//   c = clamp(rint((x - o) / s) + 8, 0, 15), rint to even;  s == 0: c = 8;  a NaN in the group: o = NaN, s = 0, c = 8
//
// The arithmetic is IEEE fp32 (one rounding per operation, no contraction), so a row's bytes do not depend on how the
// kernel splits the work. s and o are rounded to fp16 because they are read for every group in every decode step
// (32 of 160 bits per group in fp32 would be 64); c is taken with the rounded s and o, so the rounding adds at most
// half an fp16 step of |o| to the half step s/2 of the code.
//
// Bytes of a row: the codes, then D/32 scales, then D/32 offsets, then zeros up to a multiple of 16. A unit of two
// bytes holds four channels (lower nibble first); the unit of channels 32 r + 4 u .. + 3 lies at byte 2 (u D/32 + r).
// So the D/16 bytes from byte u D/16 on hold four channels of EVERY group, which is what one lane of the attention's
// matrix fragments needs: it loads them at once (attend.cuh).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "page_copy.cuh"

namespace emm {

constexpr int kQ4Group = 32;

__host__ __device__ constexpr int q4_groups(int D) { return D / kQ4Group; }
__host__ __device__ constexpr int q4_row_bytes(int D) { return (D / 2 + 4 * q4_groups(D) + 15) / 16 * 16; }

// Geometry of a pool as the token kernels address it: address(l, p, slot, h) =
// layers[l] + p * plane_stride + block * block_stride + token * token_stride + h * head_stride.
struct TokenSide {
  const uint64_t *layers;
  uint64_t plane_stride;
  uint64_t block_stride;
  uint64_t token_stride;
  uint64_t head_stride;
  uint32_t num_blocks;
  uint32_t block_size;
};

struct Q4RowsArgs {
  TokenSide pool;
  uint32_t layer_begin;
  uint32_t num_tokens;
  uint32_t heads;
  uint64_t key;  // append reads these, read writes them: [layers, T, H, D], heads dense
  uint64_t value;
  uint64_t key_layer_stride;  // bytes
  uint64_t key_token_stride;
  uint64_t value_layer_stride;
  uint64_t value_token_stride;
  const int64_t *slots;
  int *status;
};

template <typename T>
__device__ __forceinline__ float to_f32(T x);
template <>
__device__ __forceinline__ float to_f32<__half>(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
// One rounding; an fp16 result saturates (o + 7 s of a group that reaches 65504 can exceed it by s's rounding).
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) {
  x = x > 65504.f ? 65504.f : (x < -65504.f ? -65504.f : x);
  return __float2half_rn(x);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// Address of a token's row of head 0, or 0 when the slot is padding or outside the pool (reported).
__device__ __forceinline__ uint64_t slot_address(const TokenSide &s, uint32_t layer, uint32_t plane, int64_t slot,
                                                 bool reporter, int *status) {
  if (slot < 0) return 0;
  const uint64_t blk = (uint64_t)slot / s.block_size;
  if (blk >= s.num_blocks) {
    if (reporter) report(status, kStatusIdRange, slot);
    return 0;
  }
  const uint64_t tok = (uint64_t)slot - blk * s.block_size;
  return s.layers[layer] + plane * s.plane_stride + blk * s.block_stride + tok * s.token_stride;
}

struct __align__(8) Quad {
  uint16_t v[4];
};

// One thread per unit of four channels; the eight threads of a group find its smallest and largest value by shuffles.
// grid.x * 256 threads cover T * H * D/4 units, grid.y the layers and planes. kWide: 8-byte loads.
template <typename T, int D, bool kWide>
__global__ void __launch_bounds__(256) q4_append(const __grid_constant__ Q4RowsArgs a) {
  constexpr uint32_t kUnits = D / 4, G = q4_groups(D);
  const uint64_t idx = (uint64_t)blockIdx.x * 256 + threadIdx.x;
  const uint32_t unit = (uint32_t)(idx % kUnits);
  const uint64_t th = idx / kUnits;
  const uint32_t t = (uint32_t)(th / a.heads), h = (uint32_t)(th % a.heads);
  const uint32_t lrel = blockIdx.y >> 1, p = blockIdx.y & 1;
  const bool mine = t < a.num_tokens;

  float x[4] = {0.f, 0.f, 0.f, 0.f};
  uint64_t row = 0;
  if (mine) {
    const uint64_t src = (p ? a.value + lrel * a.value_layer_stride + t * a.value_token_stride
                            : a.key + lrel * a.key_layer_stride + t * a.key_token_stride) +
                         ((uint64_t)h * D + unit * 4) * 2;
    T e[4];
    if (kWide) {
      *reinterpret_cast<Quad *>(e) = *reinterpret_cast<const Quad *>(src);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) e[i] = reinterpret_cast<const T *>(src)[i];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = to_f32<T>(e[i]);
    row = slot_address(a.pool, a.layer_begin + lrel, p, a.slots[t], unit == 0 && h == 0, a.status);
  }
  bool nan = false;
  float lo = 65504.f, hi = -65504.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    nan |= x[i] != x[i];
    x[i] = fminf(fmaxf(x[i], -65504.f), 65504.f);
    lo = fminf(lo, x[i]);
    hi = fmaxf(hi, x[i]);
  }
#pragma unroll
  for (int m = 1; m < 8; m <<= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, m));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, m));
    nan |= __shfl_xor_sync(0xffffffffu, (int)nan, m) != 0;
  }
  if (row == 0) return;
  __half s = __float2half_rn(__fdiv_rn(__fsub_rn(hi, lo), 15.f));
  const float sf = __half2float(s);
  __half o = __float2half_rn(__fadd_rn(lo, __fmul_rn(8.f, sf)));
  const float of = __half2float(o);
  uint32_t code = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    int c = 8;
    if (!nan && sf != 0.f) c = 8 + __float2int_rn(__fdiv_rn(__fsub_rn(x[i], of), sf));
    c = c < 0 ? 0 : (c > 15 ? 15 : c);
    code |= (uint32_t)c << (4 * i);
  }
  if (nan) {
    s = __ushort_as_half((unsigned short)0);
    o = __ushort_as_half((unsigned short)0x7fff);
  }
  const uint32_t r = unit / 8, u = unit % 8;
  uint8_t *dst = reinterpret_cast<uint8_t *>(row + (uint64_t)h * a.pool.head_stride);
  *reinterpret_cast<uint16_t *>(dst + 2 * (u * G + r)) = (uint16_t)code;
  if (u == 0) {
    *reinterpret_cast<__half *>(dst + D / 2 + 2 * r) = s;
    *reinterpret_cast<__half *>(dst + D / 2 + 2 * G + 2 * r) = o;
  }
  if (D == 64 && u == 1 && r == 0) *reinterpret_cast<uint2 *>(dst + 40) = make_uint2(0, 0);  // the row's padding
}

// The inverse: o + s * (c - 8), rounded once to T. A padding or reported slot gives a row of zeros.
template <typename T, int D, bool kWide>
__global__ void __launch_bounds__(256) q4_read(const __grid_constant__ Q4RowsArgs a) {
  constexpr uint32_t kUnits = D / 4, G = q4_groups(D);
  const uint64_t idx = (uint64_t)blockIdx.x * 256 + threadIdx.x;
  const uint32_t unit = (uint32_t)(idx % kUnits);
  const uint64_t th = idx / kUnits;
  const uint32_t t = (uint32_t)(th / a.heads), h = (uint32_t)(th % a.heads);
  const uint32_t lrel = blockIdx.y >> 1, p = blockIdx.y & 1;
  if (t >= a.num_tokens) return;
  const uint64_t row = slot_address(a.pool, a.layer_begin + lrel, p, a.slots[t], unit == 0 && h == 0, a.status);
  T e[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) e[i] = from_f32<T>(0.f);
  if (row) {
    const uint32_t r = unit / 8, u = unit % 8;
    const uint8_t *src = reinterpret_cast<const uint8_t *>(row + (uint64_t)h * a.pool.head_stride);
    const uint32_t code = *reinterpret_cast<const uint16_t *>(src + 2 * (u * G + r));
    const float s = __half2float(*reinterpret_cast<const __half *>(src + D / 2 + 2 * r));
    const float o = __half2float(*reinterpret_cast<const __half *>(src + D / 2 + 2 * G + 2 * r));
#pragma unroll
    for (int i = 0; i < 4; ++i)
      e[i] = from_f32<T>(__fadd_rn(o, __fmul_rn(s, (float)(int)((code >> (4 * i)) & 15u) - 8.f)));
  }
  const uint64_t dst = (p ? a.value + lrel * a.value_layer_stride + t * a.value_token_stride
                          : a.key + lrel * a.key_layer_stride + t * a.key_token_stride) +
                       ((uint64_t)h * D + unit * 4) * 2;
  if (kWide) {
    *reinterpret_cast<Quad *>(dst) = *reinterpret_cast<const Quad *>(e);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) reinterpret_cast<T *>(dst)[i] = e[i];
  }
}

}  // namespace emm
