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

#include <type_traits>

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
  int32_t block_shift;  // log2(block_size), or -1
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

__device__ __forceinline__ float2 unpack_half2(uint32_t x) {
  return __half22float2(*reinterpret_cast<const __half2 *>(&x));
}

// Two 16-bit values of a word.
template <typename T>
__device__ __forceinline__ void unpack2(uint32_t w, float &lo, float &hi) {
  if constexpr (std::is_same<T, __half>::value) {
    const float2 f = unpack_half2(w);
    lo = f.x;
    hi = f.y;
  } else {
    lo = __uint_as_float(w << 16);
    hi = __uint_as_float(w & 0xffff0000u);
  }
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (std::is_same<T, __half>::value) {
    uint32_t y;
    asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(y) : "f"(hi), "f"(lo));
    return y;
  } else {
    uint32_t y;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(y) : "f"(hi), "f"(lo));
    return y;
  }
}

// Two 32-bit values in one register pair, an operation on both in one instruction, each rounded as the single one is.
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
  uint64_t y;
  asm("mov.b64 %0, {%1, %2};" : "=l"(y) : "f"(lo), "f"(hi));
  return y;
}
__device__ __forceinline__ void split(uint64_t x, uint32_t &lo, uint32_t &hi) { asm("mov.b64 {%0, %1}, %2;" : "=r"(lo), "=r"(hi) : "l"(x)); }
__device__ __forceinline__ uint64_t add_pair(uint64_t a, uint64_t b) {
  uint64_t y;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(y) : "l"(a), "l"(b));
  return y;
}
__device__ __forceinline__ uint64_t mul_pair(uint64_t a, uint64_t b) {
  uint64_t y;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(y) : "l"(a), "l"(b));
  return y;
}
__device__ __forceinline__ uint64_t fma_pair(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t y;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(y) : "l"(a), "l"(b), "l"(c));
  return y;
}

// Address of a token's row of head 0, or 0 when the slot is padding or outside the pool (reported).
__device__ __forceinline__ uint64_t slot_address(const TokenSide &s, uint32_t layer, uint32_t plane, int64_t slot,
                                                 bool reporter, int *status) {
  if (slot < 0) return 0;
  const uint64_t blk = s.block_shift >= 0 ? (uint64_t)slot >> s.block_shift : (uint64_t)slot / s.block_size;
  if (blk >= s.num_blocks) {
    if (reporter) report(status, kStatusIdRange, slot);
    return 0;
  }
  const uint64_t tok = (uint64_t)slot - blk * s.block_size;
  return s.layers[layer] + plane * s.plane_stride + blk * s.block_stride + tok * s.token_stride;
}

// ---- one thread per group of 32 channels (64 bytes), where keys and values lie on 32-byte boundaries
//
// Append, 32 channels per thread: 64 bytes in, 20 out. At HBM's rate an SM has about 470 issue slots per warp for that, so
// the bound is how few instructions a thread takes (393 here, 12 a channel) and that enough warps wait for their loads
// (six blocks an SM; with the five that 43 registers allow the kernel below takes 5 us longer):
//   * smallest and largest value on packed 16-bit pairs;
//   * the quotient d / s, d = x - o, as d times an approximate 1/s and one step of correction with the fma's remainder:
//     that is within 2^-45 of d / s before its rounding. It rounds to the same integer as the division does: a half-integer
//     h times s is exact (5 and 11 bits), so d / s is h itself, which the corrected quotient then is too, or d is at least
//     one unit in its last place away from h s, which is over half a unit of h (by 2^-11 of it or more). Every 50th
//     group of bf16 values has such an exact half, so a test with divisions behind it would run in half of all warps;
//   * these in instructions on pairs of channels, which round each half as the single ones do (7 us of 141);
//   * rounding by adding 1.5 * 2^23 + 8, which leaves the code in the low bits; four make a unit by integer fma;
//   * a group with a code outside 0..15 before the clamp (an offset much larger than its range), with s = 0, infinities or
//     NaN goes through the definition step by step.
// Rows are put together in shared memory and leave in 16-byte pieces. 4 099 tokens x 32 layers x 8 heads of 128, bf16: 134 us
// (5.3 TB/s).
constexpr int kRowWarps = 8;

template <typename T>
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
  uint32_t d;
  if constexpr (std::is_same<T, __half>::value) asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  else asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
template <typename T>
__device__ __forceinline__ uint32_t min2(uint32_t a, uint32_t b) {
  uint32_t d;
  if constexpr (std::is_same<T, __half>::value) asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  else asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ void load32(uint32_t (&w)[16], int i, uint64_t src) {
  asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(w[i]), "=r"(w[i + 1]), "=r"(w[i + 2]), "=r"(w[i + 3]), "=r"(w[i + 4]), "=r"(w[i + 5]), "=r"(w[i + 6]), "=r"(w[i + 7])
               : "l"(src));
}
__device__ __forceinline__ void store32(uint64_t dst, const uint32_t (&w)[16], int i) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(dst), "r"(w[i]), "r"(w[i + 1]), "r"(w[i + 2]), "r"(w[i + 3]),
               "r"(w[i + 4]), "r"(w[i + 5]), "r"(w[i + 6]), "r"(w[i + 7])
               : "memory");
}

// The group's codes by the definition, from its channels in memory; `step` is the distance of its units in the row.
template <typename T>
__device__ __noinline__ void encode_exact(uint64_t src, float s, float o, uint8_t *row, int step) {
#pragma unroll 1
  for (int u = 0; u < 8; ++u) {
    uint32_t code = 0;
#pragma unroll 1
    for (int i = 0; i < 4; ++i) {
      const float x = fminf(fmaxf(to_f32<T>(reinterpret_cast<const T *>(src)[4 * u + i]), -65504.f), 65504.f);
      const int c = s == 0.f ? 8 : 8 + __float2int_rn(__fdiv_rn(__fsub_rn(x, o), s));
      code |= (uint32_t)(c < 0 ? 0 : (c > 15 ? 15 : c)) << (4 * i);
    }
    *reinterpret_cast<uint16_t *>(row + u * step) = (uint16_t)code;
  }
}

// grid.x * kRowWarps warps cover the T * H rows, 32 / (D/32) of them each; grid.y the layers and planes.
template <typename T, int D>
__global__ void __launch_bounds__(kRowWarps * 32, 6) q4_append_rows(const __grid_constant__ Q4RowsArgs a) {
  grid_launch_dependents();
  grid_dependency_wait();
  constexpr int G = q4_groups(D), R = q4_row_bytes(D), kRows = 32 / G, kPieces = kRows * R / 16;
  __shared__ __align__(16) uint8_t stage[kRowWarps][kRows * R];
  const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32, r = lane % G;
  const uint64_t rows = (uint64_t)a.num_tokens * a.heads, row = ((uint64_t)blockIdx.x * kRowWarps + warp) * kRows + lane / G;
  const uint32_t lrel = blockIdx.y >> 1, p = blockIdx.y & 1;
  const bool mine = row < rows;
  const uint32_t t = mine ? (uint32_t)row / a.heads : 0u, h = mine ? (uint32_t)row - t * a.heads : 0u;
  const uint64_t src = (p ? a.value + lrel * a.value_layer_stride + t * a.value_token_stride
                          : a.key + lrel * a.key_layer_stride + t * a.key_token_stride) +
                       ((uint64_t)h * D + 32 * r) * 2;
  uint32_t w[16];
  load32(w, 0, src);
  load32(w, 8, src + 32);
  const int64_t slot = mine ? a.slots[t] : -1;

  uint32_t big = w[0], small = w[0];
#pragma unroll
  for (int i = 1; i < 16; ++i) {
    big = max2<T>(big, w[i]);
    small = min2<T>(small, w[i]);
  }
  float hi, hi2, lo, lo2;
  unpack2<T>(big, hi, hi2);
  unpack2<T>(small, lo, lo2);
  const bool nan = hi != hi || hi2 != hi2;
  hi = fmaxf(hi, hi2);
  lo = fminf(lo, lo2);
  bool exact = hi > 65504.f || lo < -65504.f;  // infinities too
  hi = fminf(fmaxf(hi, -65504.f), 65504.f);
  lo = fminf(fmaxf(lo, -65504.f), 65504.f);
  __half s = __float2half_rn(__fdiv_rn(__fsub_rn(hi, lo), 15.f));
  const float sf = __half2float(s);
  __half o = __float2half_rn(__fadd_rn(lo, __fmul_rn(8.f, sf)));
  const float of = __half2float(o);

  float inv;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(sf));
  exact = exact || !((lo - of) * inv > -8.25f && (hi - of) * inv < 7.25f);  // also for s = 0 and NaN
  const uint64_t inv2 = pair(inv, inv), minus_s = pair(-sf, -sf), minus_o = pair(-of, -of);
  uint32_t unit[8];
#pragma unroll
  for (int u = 0; u < 8; ++u) {
    uint32_t k[4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float x0, x1;
      unpack2<T>(w[2 * u + i], x0, x1);
      const uint64_t d = add_pair(pair(x0, x1), minus_o), q = mul_pair(d, inv2);
      split(add_pair(fma_pair(fma_pair(q, minus_s, d), inv2, q), pair(12582920.f, 12582920.f)), k[2 * i], k[2 * i + 1]);
    }
    unit[u] = ((k[3] * 16u + k[2]) * 16u + k[1]) * 16u + k[0];  // its low 16 bits: the constant's are zero but for the 8
  }
  if (nan) {
    s = __ushort_as_half((unsigned short)0);
    o = __ushort_as_half((unsigned short)0x7fff);
#pragma unroll
    for (int u = 0; u < 8; ++u) unit[u] = 0x8888u;
  }
  uint8_t *mem = stage[warp] + lane / G * R;
#pragma unroll
  for (int u = 0; u < 8; ++u) *reinterpret_cast<uint16_t *>(mem + 2 * (u * G + r)) = (uint16_t)unit[u];
  if (exact && !nan) encode_exact<T>(src, sf, of, mem + 2 * r, 2 * G);
  *reinterpret_cast<__half *>(mem + D / 2 + 2 * r) = s;
  *reinterpret_cast<__half *>(mem + D / 2 + 2 * G + 2 * r) = o;
  if (D == 64 && r == 0) *reinterpret_cast<uint2 *>(mem + 40) = make_uint2(0, 0);  // the row's padding
  uint64_t dst = slot_address(a.pool, a.layer_begin + lrel, p, slot, r == 0 && h == 0, a.status);
  if (dst) dst += (uint64_t)h * a.pool.head_stride;
  __syncwarp();
#pragma unroll
  for (int c0 = 0; c0 < kPieces; c0 += 32) {
    const uint32_t c = c0 + lane, from = min(c / (R / 16), (uint32_t)kRows - 1);
    const uint64_t to = __shfl_sync(0xffffffffu, dst, from * G);
    if (to && c < kPieces)
      *reinterpret_cast<uint4 *>(to + c % (R / 16) * 16) = *reinterpret_cast<const uint4 *>(stage[warp] + c * 16);
  }
}

// The inverse: o + s * (c - 8), rounded once to T. HBM's writes bound it: 16 383 tokens x 28 layers x 4 heads of 128 in 206 us
// (6.0 TB/s). A padding or reported slot gives a row of zeros.
template <typename T, int D>
__global__ void __launch_bounds__(kRowWarps * 32) q4_read_rows(const __grid_constant__ Q4RowsArgs a) {
  grid_launch_dependents();
  grid_dependency_wait();
  constexpr int G = q4_groups(D), R = q4_row_bytes(D), kRows = 32 / G, kPieces = kRows * R / 16;
  __shared__ __align__(16) uint8_t stage[kRowWarps][kRows * R];
  const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32, r = lane % G;
  const uint64_t rows = (uint64_t)a.num_tokens * a.heads, row = ((uint64_t)blockIdx.x * kRowWarps + warp) * kRows + lane / G;
  const uint32_t lrel = blockIdx.y >> 1, p = blockIdx.y & 1;
  const bool mine = row < rows;
  const uint32_t t = mine ? (uint32_t)row / a.heads : 0u, h = mine ? (uint32_t)row - t * a.heads : 0u;
  uint64_t src = slot_address(a.pool, a.layer_begin + lrel, p, mine ? a.slots[t] : -1, r == 0 && h == 0, a.status);
  if (src) src += (uint64_t)h * a.pool.head_stride;
#pragma unroll
  for (int c0 = 0; c0 < kPieces; c0 += 32) {
    const uint32_t c = c0 + lane, from = min(c / (R / 16), (uint32_t)kRows - 1);
    const uint64_t at = __shfl_sync(0xffffffffu, src, from * G);
    if (c < kPieces) {
      uint4 v = make_uint4(0, 0, 0, 0);  // codes, scale and offset 0 stand for 0
      if (at) v = *reinterpret_cast<const uint4 *>(at + c % (R / 16) * 16);
      *reinterpret_cast<uint4 *>(stage[warp] + c * 16) = v;
    }
  }
  __syncwarp();
  const uint8_t *mem = stage[warp] + lane / G * R;
  const float s = __half2float(*reinterpret_cast<const __half *>(mem + D / 2 + 2 * r));
  const float o = __half2float(*reinterpret_cast<const __half *>(mem + D / 2 + 2 * G + 2 * r));
  const uint64_t s2 = pair(s, s), o2 = pair(o, o);
  uint32_t w[16];
#pragma unroll
  for (int u = 0; u < 8; ++u) {
    const uint32_t unit = *reinterpret_cast<const uint16_t *>(mem + 2 * (u * G + r));
#pragma unroll
    for (int i = 0; i < 2; ++i) {  // 2^23 + c less 2^23 + 8: exact
      const uint64_t c = pair(__uint_as_float(0x4b000000u | (unit >> (8 * i) & 15u)), __uint_as_float(0x4b000000u | (unit >> (8 * i + 4) & 15u)));
      uint32_t v0, v1;
      split(fma_pair(s2, add_pair(c, pair(-8388616.f, -8388616.f)), o2), v0, v1);
      w[2 * u + i] = pack2<T>(__uint_as_float(v0), __uint_as_float(v1));
    }
  }
  if (!mine) return;
  const uint64_t dst = (p ? a.value + lrel * a.value_layer_stride + t * a.value_token_stride
                          : a.key + lrel * a.key_layer_stride + t * a.key_token_stride) +
                       ((uint64_t)h * D + 32 * r) * 2;
  store32(dst, w, 0);
  store32(dst + 32, w, 8);
}

// ---- keys and values on other boundaries: one thread per unit of four channels, element by element; the eight threads
// of a group find its smallest and largest value by shuffles. grid.x * 256 threads cover T * H * D/4 units.
template <typename T, int D>
__global__ void __launch_bounds__(256) q4_append_units(const __grid_constant__ Q4RowsArgs a) {
  grid_launch_dependents();
  grid_dependency_wait();
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
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = to_f32<T>(reinterpret_cast<const T *>(src)[i]);
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

template <typename T, int D>
__global__ void __launch_bounds__(256) q4_read_units(const __grid_constant__ Q4RowsArgs a) {
  grid_launch_dependents();
  grid_dependency_wait();
  constexpr uint32_t kUnits = D / 4, G = q4_groups(D);
  const uint64_t idx = (uint64_t)blockIdx.x * 256 + threadIdx.x;
  const uint32_t unit = (uint32_t)(idx % kUnits);
  const uint64_t th = idx / kUnits;
  const uint32_t t = (uint32_t)(th / a.heads), h = (uint32_t)(th % a.heads);
  const uint32_t lrel = blockIdx.y >> 1, p = blockIdx.y & 1;
  if (t >= a.num_tokens) return;
  const uint64_t row = slot_address(a.pool, a.layer_begin + lrel, p, a.slots[t], unit == 0 && h == 0, a.status);
  T *dst = reinterpret_cast<T *>((p ? a.value + lrel * a.value_layer_stride + t * a.value_token_stride
                                    : a.key + lrel * a.key_layer_stride + t * a.key_token_stride) +
                                 ((uint64_t)h * D + unit * 4) * 2);
  float s = 0.f, o = 0.f;
  uint32_t code = 0;
  if (row) {
    const uint32_t r = unit / 8, u = unit % 8;
    const uint8_t *src = reinterpret_cast<const uint8_t *>(row + (uint64_t)h * a.pool.head_stride);
    code = *reinterpret_cast<const uint16_t *>(src + 2 * (u * G + r));
    s = __half2float(*reinterpret_cast<const __half *>(src + D / 2 + 2 * r));
    o = __half2float(*reinterpret_cast<const __half *>(src + D / 2 + 2 * G + 2 * r));
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) dst[i] = from_f32<T>(__fadd_rn(o, __fmul_rn(s, (float)(int)((code >> (4 * i)) & 15u) - 8.f)));
}

}  // namespace emm
