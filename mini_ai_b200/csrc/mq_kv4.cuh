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

constexpr int kKv4Each = 2;                                   // blocks a quad of lanes
constexpr int kKv4Blocks = kKv4Threads / 4 * kKv4Each;         // blocks a CTA

// A block's place: row, head and block of the head, K or V.
struct Kv4Place {
  int row, head, j;
  bool v;
};
template <typename Index>
__device__ __forceinline__ Kv4Place kv4_place(const Kv4View &c, Index idx, int per_row) {
  Kv4Place p;
  p.row = (int)(idx / per_row);
  const int in_row = (int)(idx - (Index)p.row * per_row), half = c.kv * c.nb;
  p.v = in_row >= half;
  const int hb = p.v ? in_row - half : in_row;
  p.head = hb / c.nb, p.j = hb % c.nb;
  return p;
}
// Where lane t's 8 elements of the block lie in `unit`: K one word, V two half-words 2 nb bytes apart; and its scale.
__device__ __forceinline__ uint8_t *kv4_codes(const Kv4View &c, uint8_t *unit, const Kv4Place &p, int tok, int t) {
  if (p.v) return unit + kv4_v_off(c.nb) + tok * 16 * c.nb + 4 * t * c.nb + 2 * p.j;
  return unit + tok * 16 * c.nb + t * 4 * c.nb + 4 * p.j;
}
__device__ __forceinline__ uint16_t *kv4_scale(const Kv4View &c, uint8_t *unit, const Kv4Place &p, int tok) {
  return reinterpret_cast<uint16_t *>(unit + (p.v ? kv4_v_scale_off(c.nb) : kv4_k_scale_off(c.nb))) + tok * c.nb + p.j;
}

// One quad of lanes per block of a row, two blocks each: reads 32 floats,
// writes 16 bytes of codes and a scale. Rows of no valid slot are skipped.
// Index: 32 bits where the call's blocks fit (a 64-bit division costs as much as the packing).
template <bool VEC, typename Index>
__global__ void __launch_bounds__(kKv4Threads)
    kv4_store_kernel(const Kv4View c, int layer, const Kv4Rows k, const Kv4Rows v, const int *__restrict__ slots,
                     int rows) {
  const int per_row = 2 * c.kv * c.nb, t = threadIdx.x & 3;  // blocks of a row: K heads, then V heads
  const Index total = (Index)rows * per_row, i0 = (Index)blockIdx.x * kKv4Blocks + (threadIdx.x >> 2);
  Kv4Place at[kKv4Each];
  int slot[kKv4Each];
  float x[kKv4Each][8];
#pragma unroll
  for (int n = 0; n < kKv4Each; ++n) {
    const Index idx = i0 + n * (kKv4Threads / 4);
    at[n] = kv4_place(c, idx < total ? idx : total - 1, per_row);  // whole warps: kv4_pack shuffles
    slot[n] = idx < total ? slots[at[n].row] : -1;
    const Kv4Rows &src = at[n].v ? v : k;
    const float *p = src.p + at[n].row * src.ld + at[n].head * src.hs + 32 * at[n].j + 8 * t;
    if (VEC) {
      const float4 a = __ldg(reinterpret_cast<const float4 *>(p)), b = __ldg(reinterpret_cast<const float4 *>(p) + 1);
      x[n][0] = a.x, x[n][1] = a.y, x[n][2] = a.z, x[n][3] = a.w;
      x[n][4] = b.x, x[n][5] = b.y, x[n][6] = b.z, x[n][7] = b.w;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[n][i] = __ldg(p + i);
    }
  }
#pragma unroll
  for (int n = 0; n < kKv4Each; ++n) {
    uint16_t scale;
    const uint32_t w = kv4_pack(x[n], scale);
    if (slot[n] < 0 || slot[n] >= c.pages * c.page) continue;
    const int page_id = slot[n] / c.page, in_page = slot[n] - page_id * c.page, tok = in_page % kKv4Unit;
    uint8_t *unit = kv4_unit(c, layer, page_id, at[n].head, in_page / kKv4Unit);
    uint8_t *codes = kv4_codes(c, unit, at[n], tok, t);
    if (at[n].v) {
      *reinterpret_cast<uint16_t *>(codes) = (uint16_t)w;
      *reinterpret_cast<uint16_t *>(codes + 2 * c.nb) = (uint16_t)(w >> 16);
    } else {
      *reinterpret_cast<uint32_t *>(codes) = w;
    }
    if (t == 0) *kv4_scale(c, unit, at[n], tok) = scale;
  }
}

// The values at `slots`, k and v [rows][kv][hd]; rows of no valid slot are 0.
// Threads as in the store.
template <bool VEC, typename Index>
__global__ void __launch_bounds__(kKv4Threads)
    kv4_load_kernel(const Kv4View c, int layer, const int *__restrict__ slots, int rows, float *__restrict__ k,
                    float *__restrict__ v) {
  const int per_row = 2 * c.kv * c.nb, t = threadIdx.x & 3;
  const Index total = (Index)rows * per_row, i0 = (Index)blockIdx.x * kKv4Blocks + (threadIdx.x >> 2);
  Kv4Place at[kKv4Each];
  uint32_t w[kKv4Each];
  float d[kKv4Each];
#pragma unroll
  for (int n = 0; n < kKv4Each; ++n) {
    const Index idx = i0 + n * (kKv4Threads / 4);
    if (idx >= total) continue;
    at[n] = kv4_place(c, idx, per_row);
    const int slot = slots[at[n].row];
    w[n] = 0x88888888u, d[n] = 0.0f;
    if (slot < 0 || slot >= c.pages * c.page) continue;
    const int page_id = slot / c.page, in_page = slot - page_id * c.page, tok = in_page % kKv4Unit;
    uint8_t *unit = kv4_unit(c, layer, page_id, at[n].head, in_page / kKv4Unit);
    const uint8_t *codes = kv4_codes(c, unit, at[n], tok, t);
    if (at[n].v)
      w[n] = __ldg(reinterpret_cast<const uint16_t *>(codes)) |
             (uint32_t)__ldg(reinterpret_cast<const uint16_t *>(codes + 2 * c.nb)) << 16;
    else
      w[n] = __ldg(reinterpret_cast<const uint32_t *>(codes));
    d[n] = __half2float(__ushort_as_half(__ldg(kv4_scale(c, unit, at[n], tok))));
  }
#pragma unroll
  for (int n = 0; n < kKv4Each; ++n) {
    if (i0 + n * (kKv4Threads / 4) >= total) continue;
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = d[n] * (float)((int)((w[n] >> (4 * i)) & 15u) - 8);
    float *o = (at[n].v ? v : k) + ((int64_t)at[n].row * c.kv + at[n].head) * c.hd + 32 * at[n].j + 8 * t;
    if (VEC) {
      reinterpret_cast<float4 *>(o)[0] = make_float4(x[0], x[1], x[2], x[3]);
      reinterpret_cast<float4 *>(o)[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = x[i];
    }
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
