// Causal attention of a ragged batch's query rows over the paged 4-bit cache.
//
// Row i of request r (new_r rows, len_r cached tokens, its own among them)
// stands at position len_r - new_r + i and sees the tokens 0..position:
//   out = sum_s p_s v_s / sum_s p_s, p_s = exp(scale q . k_s - max).
// A row that sees nothing is 0.
#pragma once

#include "mq_kv4.cuh"

namespace mq {

struct Kv4AttnArgs {
  Kv4View c;
  int layer;
  const float *q;
  int64_t ld_q, hs_q;
  float *out;
  int64_t ld_o, hs_o;
  const int *offsets, *lens, *tables;
  int n, width, rows, heads;
  float scale;
};

// One warp per (row, head): lanes along the elements of a block.
__global__ void __launch_bounds__(32) kv4_attention_kernel(const Kv4AttnArgs a) {
  const int row = blockIdx.x, h = blockIdx.y, lane = threadIdx.x, nb = a.c.nb;
  int lo = 0, hi = a.n;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (a.offsets[mid + 1] > row) hi = mid;
    else lo = mid + 1;
  }
  if (lo >= a.n || row < a.offsets[lo]) return;
  const int len = (int)min((int64_t)max(a.lens[lo], 0), (int64_t)a.width * a.c.page);
  const int last = min(len - (a.offsets[lo + 1] - a.offsets[lo]) + row - a.offsets[lo], len - 1);
  const int kh = h / (a.heads / a.c.kv);
  float q[4], acc[4] = {0, 0, 0, 0}, m = -INFINITY, l = 0.0f;
  for (int j = 0; j < nb; ++j) q[j] = a.q[row * a.ld_q + h * a.hs_q + 32 * j + lane];
  for (int s = 0; s <= last; ++s) {
    const int id = a.tables[(int64_t)lo * a.width + s / a.c.page];
    if (id < 0 || id >= a.c.pages) continue;
    const int in_page = s % a.c.page, tok = in_page % kKv4Unit;
    const uint8_t *u = kv4_unit(a.c, a.layer, id, kh, in_page / kKv4Unit);
    float dot = 0.0f, v[4];
    for (int j = 0; j < nb; ++j) {
      const uint32_t kw = *reinterpret_cast<const uint32_t *>(u + tok * 16 * nb + (lane >> 3) * 4 * nb + 4 * j);
      const uint16_t vw =
          *reinterpret_cast<const uint16_t *>(u + kv4_v_off(nb) + tok * 16 * nb + (lane >> 2) * 2 * nb + 2 * j);
      const float dk = __half2float(*reinterpret_cast<const __half *>(u + kv4_k_scale_off(nb) + 2 * (tok * nb + j)));
      const float dv = __half2float(*reinterpret_cast<const __half *>(u + kv4_v_scale_off(nb) + 2 * (tok * nb + j)));
      dot += q[j] * (dk * (float)((int)((kw >> (4 * (lane & 7))) & 15u) - 8));
      v[j] = dv * (float)((int)((vw >> (4 * (lane & 3))) & 15u) - 8);
    }
    for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
    dot *= a.scale;
    const float m2 = fmaxf(m, dot), shift = m2 == -INFINITY ? 0.0f : m2;
    const float old = expf(m - shift), p = expf(dot - shift);
    l = l * old + p;
    for (int j = 0; j < nb; ++j) acc[j] = acc[j] * old + p * v[j];
    m = m2;
  }
  for (int j = 0; j < nb; ++j) a.out[row * a.ld_o + h * a.hs_o + 32 * j + lane] = l == 0.0f ? 0.0f : acc[j] / l;
}

}  // namespace mq
