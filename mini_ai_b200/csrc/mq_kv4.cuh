// The paged 4-bit key/value cache: its layout, and the kernels that pack rows
// into it and read them back.
//
// A row's head is head_dim / 32 blocks (c, d) of 32 elements, each standing
// for c * d, c in [-8, 7] (the Q4_0 block, w = d * (q - 8) with q = c + 8).
// With s the block's first element of largest |x|:
//   d = fp16(bf16(s / -8)), c = clamp(rint(x / d), -8, 7).
// Rounding d to bf16's 8 significant bits is the one liberty taken with the
// Q4_0 block: c has at most 3 bits beside its power of two, so that every
// c * d is an fp16 number exactly, and one fp16 tensor-core operand holds the
// cache without error. It costs at most 2^-9 of d, against a step of d. x / d
// is a true division: fp32 then gives the nearest code of the real quotient,
// since d * (k + 1/2) is an fp32 number and no x beside it divides to k + 1/2.
// A block with a non-finite element, or whose |d| passes 8160 (8 d would pass
// the fp16 range), is stored as NaN: the attention that sees it answers NaN.
//
// Layout. Tokens are grouped by 16 into units, one contiguous piece per
// (layer, page, KV head, 16 tokens):
//   [K codes 16 x 16 NB | K scales 16 x NB fp16 | V codes | V scales],
// NB = head_dim / 32 blocks, 576 NB bytes, so a page's head is one contiguous
// range and a unit one bulk copy. Inside a token's 16 NB bytes the codes lie
// as the lanes of an m16n8k16 fragment take them, so a lane reads its part of
// a token with one vector load and no lane moves data:
//   K: chunk t (of 4) = for each block j the word of elements 32j + 8t + 0..7;
//   V: chunk g (of 8) = for each block j the half-word of 32j + 4g + 0..3;
// element i of a word is its nibble i.
#pragma once

#include <cuda_bf16.h>

#include <climits>

#include "mq_common.cuh"

namespace mq {

constexpr int kKv4Unit = 16;  // tokens

struct Kv4View {
  uint8_t *base;
  int layers, pages, page, kv, hd, nb;
  int64_t page_head_bytes;  // one head of one page
};

__host__ __device__ constexpr int kv4_unit_bytes(int nb) { return 576 * nb; }
__host__ __device__ constexpr int kv4_k_scale_off(int nb) { return 256 * nb; }
__host__ __device__ constexpr int kv4_v_off(int nb) { return 288 * nb; }
__host__ __device__ constexpr int kv4_v_scale_off(int nb) { return 544 * nb; }

// The unit of tokens [16 u, 16 u + 16) of a page's head.
__host__ __device__ __forceinline__ uint8_t *kv4_unit(const Kv4View &c, int layer, int page_id, int head, int u) {
  return c.base + (((int64_t)layer * c.pages + page_id) * c.kv + head) * c.page_head_bytes +
         (int64_t)u * kv4_unit_bytes(c.nb);
}

// 32 elements over 4 neighbouring lanes, 8 each (lane t: elements 8t..8t+7):
// this lane's nibbles and the block's scale.
__device__ __forceinline__ uint32_t kv4_pack(const float (&x)[8], uint16_t &scale) {
  const int t = threadIdx.x & 3;
  float s = x[0];
  int at = 0;
  bool bad = !isfinite(x[0]);
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    bad |= !isfinite(x[i]);
    if (fabsf(x[i]) > fabsf(s)) s = x[i], at = i;
  }
  at += 8 * t;
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {  // ties go to the lower place
    const float s2 = __shfl_xor_sync(0xffffffffu, s, o);
    const int at2 = __shfl_xor_sync(0xffffffffu, at, o);
    bad |= (bool)__shfl_xor_sync(0xffffffffu, (int)bad, o);
    if (fabsf(s2) > fabsf(s) || (fabsf(s2) == fabsf(s) && at2 < at)) s = s2, at = at2;
  }
  const float d8 = __bfloat162float(__float2bfloat16_rn(s * -0.125f));
  bad |= fabsf(d8) > 8160.0f;
  const __half dh = __float2half_rn(d8);
  const float d = __half2float(dh);
  scale = bad ? (uint16_t)0x7e00u : __half_as_ushort(dh);
  if (bad || d == 0.0f) return 0x88888888u;  // all codes 0
  // Nearest integers by x times 1 / d, rounded by adding 1.5 * 2^23: right wherever the remainder (which fma gives
  // exactly) stays below d / 2; where it does not, a tie or a quotient next to one, by the division.
  constexpr float kRound = 12582912.0f;
  const float inv = __frcp_rn(d);
  uint32_t w = 0;
  float far = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float t = fmaf(x[i], inv, kRound);
    far = fmaxf(far, fabsf(fmaf(kRound - t, d, x[i])));
    w |= (__float_as_uint(fminf(fmaxf(t, kRound - 8.0f), kRound + 7.0f)) & 15u) << (4 * i);
  }
  if (!(far < 0.5f * fabsf(d))) {
    w = 0;
#pragma unroll 1
    for (int i = 0; i < 8; ++i) {
      float v = x[0];
#pragma unroll
      for (int j = 1; j < 8; ++j) v = i == j ? x[j] : v;
      w |= ((uint32_t)(int)fminf(fmaxf(rintf(__fdiv_rn(v, d)), -8.0f), 7.0f) & 15u) << (4 * i);
    }
  }
  return w ^ 0x88888888u;  // c + 8
}

struct Kv4Rows {  // rows [rows][kv][hd] with strides in elements
  const float *p;
  int64_t ld, hs;
};

constexpr int kKv4Threads = 256;

// One quad of lanes per block of a row: reads 32 floats, writes 16 bytes of
// codes and a scale. Rows of no valid slot are skipped.
// Index: 32 bits where the call's blocks fit (a 64-bit division costs as much as the packing).
template <bool VEC, typename Index>
__global__ void __launch_bounds__(kKv4Threads)
    kv4_store_kernel(const Kv4View c, int layer, const Kv4Rows k, const Kv4Rows v, const int *__restrict__ slots,
                     int rows) {
  const int per_row = 2 * c.kv * c.nb;  // blocks of a row: K heads, then V heads
  const Index total = (Index)rows * per_row;
  const Index i0 = (Index)blockIdx.x * (kKv4Threads / 4) + (threadIdx.x >> 2);
  const bool inside = i0 < total;
  const Index idx = inside ? i0 : total - 1;  // whole warps: kv4_pack shuffles
  const int row = (int)(idx / per_row), in_row = (int)(idx - (Index)row * per_row);
  const bool is_v = in_row >= c.kv * c.nb;
  const int hb = is_v ? in_row - c.kv * c.nb : in_row, head = hb / c.nb, j = hb % c.nb, t = threadIdx.x & 3;
  const int slot = slots[row];
  const Kv4Rows &src = is_v ? v : k;
  const float *p = src.p + row * src.ld + head * src.hs + 32 * j + 8 * t;
  float x[8];
  if (VEC) {
    const float4 a = __ldg(reinterpret_cast<const float4 *>(p)), b = __ldg(reinterpret_cast<const float4 *>(p) + 1);
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __ldg(p + i);
  }
  uint16_t scale;
  const uint32_t w = kv4_pack(x, scale);
  if (!inside || slot < 0 || slot >= c.pages * c.page) return;
  const int page_id = slot / c.page, in_page = slot % c.page, tok = in_page % kKv4Unit;
  uint8_t *unit = kv4_unit(c, layer, page_id, head, in_page / kKv4Unit);
  if (!is_v) {
    *reinterpret_cast<uint32_t *>(unit + tok * 16 * c.nb + t * 4 * c.nb + 4 * j) = w;
    if (t == 0) *reinterpret_cast<uint16_t *>(unit + kv4_k_scale_off(c.nb) + 2 * (tok * c.nb + j)) = scale;
  } else {
    uint8_t *vr = unit + kv4_v_off(c.nb) + tok * 16 * c.nb + 2 * j;
    *reinterpret_cast<uint16_t *>(vr + (2 * t) * 2 * c.nb) = (uint16_t)w;
    *reinterpret_cast<uint16_t *>(vr + (2 * t + 1) * 2 * c.nb) = (uint16_t)(w >> 16);
    if (t == 0) *reinterpret_cast<uint16_t *>(unit + kv4_v_scale_off(c.nb) + 2 * (tok * c.nb + j)) = scale;
  }
}

// The values at `slots`, k and v [rows][kv][hd]; rows of no valid slot are 0.
// Threads as in the store.
template <bool VEC, typename Index>
__global__ void __launch_bounds__(kKv4Threads)
    kv4_load_kernel(const Kv4View c, int layer, const int *__restrict__ slots, int rows, float *__restrict__ k,
                    float *__restrict__ v) {
  const int per_row = 2 * c.kv * c.nb;
  const Index idx = (Index)blockIdx.x * (kKv4Threads / 4) + (threadIdx.x >> 2);
  if (idx >= (Index)rows * per_row) return;
  const int row = (int)(idx / per_row), in_row = (int)(idx - (Index)row * per_row);
  const bool is_v = in_row >= c.kv * c.nb;
  const int hb = is_v ? in_row - c.kv * c.nb : in_row, head = hb / c.nb, j = hb % c.nb, t = threadIdx.x & 3;
  const int slot = slots[row];
  float x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = 0.0f;
  if (slot >= 0 && slot < c.pages * c.page) {
    const int page_id = slot / c.page, in_page = slot % c.page, tok = in_page % kKv4Unit;
    const uint8_t *unit = kv4_unit(c, layer, page_id, head, in_page / kKv4Unit);
    uint32_t w;
    uint16_t scale;
    if (!is_v) {
      w = __ldg(reinterpret_cast<const uint32_t *>(unit + tok * 16 * c.nb + t * 4 * c.nb + 4 * j));
      scale = __ldg(reinterpret_cast<const uint16_t *>(unit + kv4_k_scale_off(c.nb) + 2 * (tok * c.nb + j)));
    } else {
      const uint8_t *vr = unit + kv4_v_off(c.nb) + tok * 16 * c.nb + 2 * j;
      w = __ldg(reinterpret_cast<const uint16_t *>(vr + (2 * t) * 2 * c.nb)) |
          (uint32_t)__ldg(reinterpret_cast<const uint16_t *>(vr + (2 * t + 1) * 2 * c.nb)) << 16;
      scale = __ldg(reinterpret_cast<const uint16_t *>(unit + kv4_v_scale_off(c.nb) + 2 * (tok * c.nb + j)));
    }
    const float d = __half2float(__ushort_as_half(scale));
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = d * (float)((int)((w >> (4 * i)) & 15u) - 8);
  }
  float *o = (is_v ? v : k) + ((int64_t)row * c.kv + head) * c.hd + 32 * j + 8 * t;
  if (VEC) {
    reinterpret_cast<float4 *>(o)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4 *>(o)[1] = make_float4(x[4], x[5], x[6], x[7]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = x[i];
  }
}

}  // namespace mq

// Opaque handle behind mq_kv4*.
struct mq_kv4 {
  int device = 0;
  mq::Kv4View v{};
  size_t bytes = 0;
  int sms = 0;
  void *owned = nullptr;  // the allocation, where the caller gave no memory
};
