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
// cache without error. It costs at most 2^-8 of d, against a step of d (and
// 2^-25 more below 2^-14, where fp16's numbers stand 2^-24 apart), and it makes
// values differ from those of a Q4_0 block with its full fp16 scale. x / d
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

__device__ __forceinline__ float max_nan(float x, float y) {  // NaN if either is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float min_nan(float x, float y) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
  return r;
}

// 32 elements over 4 neighbouring lanes, 8 each (lane t: elements 8t..8t+7):
// this lane's nibbles and the block's scale. Its instructions are about half of
// the time of a store of many rows (8192 rows of 8 heads of 128: 26 us, 15.4
// million warp instructions, 13 us of issue slots, against 11 us of memory
// traffic); the rest is the latency of slots, rows and codes one after another.
// With the extreme's place carried along and every code clamped at both ends
// they were 18.3 million, 28 us.
__device__ __forceinline__ uint32_t kv4_pack(const float (&x)[8], uint16_t &scale) {
  float hi = x[0], lo = x[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) hi = max_nan(hi, x[i]), lo = min_nan(lo, x[i]);
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
  }
  float s = hi > -lo ? hi : lo;  // the element of largest |x|
  if (__any_sync(0xffffffffu, hi == -lo)) {  // of both signs: the first one
    int at = 32;
#pragma unroll
    for (int i = 7; i >= 0; --i)
      if (fabsf(x[i]) == hi) at = 8 * (threadIdx.x & 3) + i;
    float mine = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i == (at & 7)) mine = x[i];
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      const int at2 = __shfl_xor_sync(0xffffffffu, at, o);
      const float mine2 = __shfl_xor_sync(0xffffffffu, mine, o);
      if (at2 < at) at = at2, mine = mine2;
    }
    if (hi == -lo) s = mine;
  }
  const float d8 = __bfloat162float(__float2bfloat16_rn(s * -0.125f));
  const __half dh = __float2half_rn(d8);
  const float d = __half2float(dh);
  const bool bad = !(fabsf(d8) <= 8160.0f);  // or not finite
  scale = bad ? (uint16_t)0x7e00u : __half_as_ushort(dh);
  if (bad || d == 0.0f) return 0x88888888u;  // all codes 0
  // Nearest integers by x times 1 / d, rounded by adding 1.5 * 2^23: right wherever the remainder (which fma gives
  // exactly) stays below d / 2; where it does not, a tie or a quotient next to one, by the division. So too below
  // fp16's normal scales, where d may be far enough off for codes below -8.
  constexpr float kRound = 12582912.0f;
  const float inv = __frcp_rn(d);
  float far = 0.0f, sum0 = 34952.0f, sum1 = 34952.0f;  // four codes in base 16, each with 8 added
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float minus = kRound - fmaf(x[i], inv, kRound);  // -c
    far = fmaxf(far, fabsf(fmaf(minus, d, x[i])));
    const float place = -(float)(1 << (4 * (i & 3))), c = fmaxf(minus, -7.0f);
    if (i < 4) sum0 = fmaf(c, place, sum0);
    else sum1 = fmaf(c, place, sum1);
  }
  uint32_t w = __float_as_uint(sum0 + 8388608.0f) & 0xffffu | __float_as_uint(sum1 + 8388608.0f) << 16;
  if (!(far < 0.5f * fabsf(d)) || fabsf(d) < 6.103515625e-5f) {
    w = 0;
#pragma unroll 1
    for (int i = 0; i < 8; ++i) {
      float v = x[0];
#pragma unroll
      for (int j = 1; j < 8; ++j) v = i == j ? x[j] : v;
      w |= (uint32_t)((int)fminf(fmaxf(rintf(__fdiv_rn(v, d)), -8.0f), 7.0f) + 8) << (4 * i);
    }
  }
  return w;
}

struct Kv4Rows {  // rows [rows][kv][hd] with strides in elements
  const float *p;
  int64_t ld, hs;
};

constexpr int kKv4Threads = 256;

constexpr int kKv4Quads = kKv4Threads / 4;  // quads of lanes: blocks that a CTA packs at a time
constexpr int kKv4Each = 2;                // rows in flight a thread (4 made the load slower: 25 -> 27 us)

// A thread's place in every row that it takes: the same head and block of K or
// V. A CTA holds `whole` rows of `per_row` blocks at a time, or (rows of more
// blocks than quads) its blockIdx.y-th part of one; CTAs stride over the rows,
// so that the divisions are paid once.
struct Kv4Place {
  int row;   // of those that the CTA holds
  int head, j;
  bool v, inside;
  int codes;  // bytes from a token's place 0 in the unit to this lane's codes, and to the scale
  int scale;
};
__host__ __device__ __forceinline__ int kv4_whole(int per_row) { return per_row < kKv4Quads ? kKv4Quads / per_row : 1; }
__device__ __forceinline__ Kv4Place kv4_place(const Kv4View &c) {
  const int per_row = 2 * c.kv * c.nb, half = c.kv * c.nb, quad = threadIdx.x >> 2, t = threadIdx.x & 3;
  Kv4Place p;
  p.row = per_row < kKv4Quads ? quad / per_row : 0;
  int in_row = per_row < kKv4Quads ? quad % per_row : blockIdx.y * kKv4Quads + quad;
  p.inside = in_row < per_row && p.row < kv4_whole(per_row);
  in_row = min(in_row, per_row - 1);
  p.v = in_row >= half;
  const int hb = p.v ? in_row - half : in_row;
  p.head = hb / c.nb, p.j = hb % c.nb;
  p.codes = p.v ? kv4_v_off(c.nb) + 4 * t * c.nb + 2 * p.j : t * 4 * c.nb + 4 * p.j;
  p.scale = (p.v ? kv4_v_scale_off(c.nb) : kv4_k_scale_off(c.nb)) + 2 * p.j;
  return p;
}
// The token of `slot` in the place's head: its unit, and its number there.
__device__ __forceinline__ uint8_t *kv4_slot(const Kv4View &c, int layer, int head, int slot, int &tok) {
  const int page_id = slot / c.page, in_page = slot - page_id * c.page;
  tok = in_page % kKv4Unit;
  return kv4_unit(c, layer, page_id, head, in_page / kKv4Unit);
}

// One quad of lanes per block of a row: reads 32 floats, writes 16 bytes of
// codes and a scale. Rows of no valid slot are skipped.
template <bool VEC>
__global__ void __launch_bounds__(kKv4Threads)
    kv4_store_kernel(const Kv4View c, int layer, const Kv4Rows k, const Kv4Rows v, const int *__restrict__ slots,
                     int rows) {
  const Kv4Place at = kv4_place(c);
  const int64_t step = (int64_t)gridDim.x * kv4_whole(2 * c.kv * c.nb);
  const Kv4Rows &src = at.v ? v : k;
  const float *p = src.p + at.head * src.hs + 32 * at.j + 8 * (threadIdx.x & 3);
  // Every warp goes around together (kv4_pack shuffles): the bound is on the CTA's first row.
  for (int64_t first = (int64_t)blockIdx.x * kv4_whole(2 * c.kv * c.nb); first < rows; first += kKv4Each * step) {
    int slot[kKv4Each];
    float x[kKv4Each][8];
#pragma unroll
    for (int n = 0; n < kKv4Each; ++n) {
      const int64_t row = first + n * step + at.row;
      const bool real = at.inside && row < rows;
      slot[n] = real ? slots[row] : -1;
      const float *q = p + (real ? row : 0) * src.ld;
      if (VEC) {
        const float4 a = __ldg(reinterpret_cast<const float4 *>(q)), b = __ldg(reinterpret_cast<const float4 *>(q) + 1);
        x[n][0] = a.x, x[n][1] = a.y, x[n][2] = a.z, x[n][3] = a.w;
        x[n][4] = b.x, x[n][5] = b.y, x[n][6] = b.z, x[n][7] = b.w;
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[n][i] = __ldg(q + i);
      }
    }
#pragma unroll
    for (int n = 0; n < kKv4Each; ++n) {
      uint16_t scale;
      const uint32_t w = kv4_pack(x[n], scale);
      if (slot[n] < 0 || slot[n] >= c.pages * c.page) continue;
      int tok;
      uint8_t *unit = kv4_slot(c, layer, at.head, slot[n], tok);
      uint8_t *codes = unit + at.codes + tok * 16 * c.nb;
      if (at.v) {  // two half-words
        *reinterpret_cast<uint16_t *>(codes) = (uint16_t)w;
        *reinterpret_cast<uint16_t *>(codes + 2 * c.nb) = (uint16_t)(w >> 16);
      } else {
        *reinterpret_cast<uint32_t *>(codes) = w;
      }
      if ((threadIdx.x & 3) == 0) *reinterpret_cast<uint16_t *>(unit + at.scale + 2 * tok * c.nb) = scale;
    }
  }
}

// The values at `slots`, k and v [rows][kv][hd]; rows of no valid slot are 0.
// Threads as in the store.
template <bool VEC>
__global__ void __launch_bounds__(kKv4Threads)
    kv4_load_kernel(const Kv4View c, int layer, const int *__restrict__ slots, int rows, float *__restrict__ k,
                    float *__restrict__ v) {
  const Kv4Place at = kv4_place(c);
  const int64_t step = (int64_t)gridDim.x * kv4_whole(2 * c.kv * c.nb);
  float *out = (at.v ? v : k) + at.head * c.hd + 32 * at.j + 8 * (threadIdx.x & 3);
  if (!at.inside) return;
  for (int64_t first = (int64_t)blockIdx.x * kv4_whole(2 * c.kv * c.nb); first < rows; first += kKv4Each * step) {
    uint32_t w[kKv4Each];
    float d[kKv4Each];
#pragma unroll
    for (int n = 0; n < kKv4Each; ++n) {
      const int64_t row = first + n * step + at.row;
      const int slot = row < rows ? slots[row] : -1;
      w[n] = 0x88888888u, d[n] = 0.0f;
      if (slot < 0 || slot >= c.pages * c.page) continue;
      int tok;
      const uint8_t *unit = kv4_slot(c, layer, at.head, slot, tok), *codes = unit + at.codes + tok * 16 * c.nb;
      if (at.v)
        w[n] = __ldg(reinterpret_cast<const uint16_t *>(codes)) |
               (uint32_t)__ldg(reinterpret_cast<const uint16_t *>(codes + 2 * c.nb)) << 16;
      else
        w[n] = __ldg(reinterpret_cast<const uint32_t *>(codes));
      d[n] = __half2float(__ushort_as_half(__ldg(reinterpret_cast<const uint16_t *>(unit + at.scale + 2 * tok * c.nb))));
    }
#pragma unroll
    for (int n = 0; n < kKv4Each; ++n) {
      const int64_t row = first + n * step + at.row;
      if (row >= rows) continue;
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i)  // 2^23 + q, less 2^23 + 8
        x[i] = d[n] * (__uint_as_float((w[n] >> (4 * i) & 15u) | 0x4B000000u) - 8388616.0f);
      float *o = out + row * ((int64_t)c.kv * c.hd);
      if (VEC) {
        reinterpret_cast<float4 *>(o)[0] = make_float4(x[0], x[1], x[2], x[3]);
        reinterpret_cast<float4 *>(o)[1] = make_float4(x[4], x[5], x[6], x[7]);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = x[i];
      }
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
  int *err_dev = nullptr, *err_host = nullptr;  // the device's bounded-wait flag
  uint64_t wait_ns = 0;                         // limit of a kernel's waits
  uint32_t lost = 0;                            // bytes that a copy is waited for beside its own
};
