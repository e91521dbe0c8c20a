// Causal attention of a ragged batch's query rows over the paged 4-bit cache:
// the work's division over CTAs, and the kernel for few rows a request.
//
// Row i of request r (new_r rows, len_r cached tokens, its own among them)
// stands at position len_r - new_r + i and sees the tokens 0..position:
//   out = sum_s p_s v_s / sum_s p_s, p_s = exp(scale q . k_s - max).
// A row that sees nothing is 0. The G = heads / kv query heads that share a KV
// head are rows of one matrix: "flat row" f = i G + g of (request, KV head).
//
// Division (stream-K). An item is a tile of RT flat rows of one (request, KV
// head); its work is the number of BN-token tiles that its last row sees. All
// items in order (request, KV head, row tile) form one line of work, cut into
// equal pieces, one a CTA, whatever the lengths. A CTA thus has at most one
// item that began in an earlier CTA and one that it leaves unfinished; the
// partial results of those (reference, sum and unscaled output per row) go to
// its two workspace slots, and a second kernel joins them in order. The
// kernels read all lengths from device memory, so that a captured launch
// serves any batch.
#pragma once

#include "mq_kv4.cuh"
#include "mq_pages.cuh"
#include "mq_sm100.cuh"

namespace mq {

struct Kv4AttnArgs {
  Kv4View c;
  int layer;
  const float *q;
  int64_t ld_q, hs_q;
  float *out;
  int64_t ld_o, hs_o;
  const int *offsets, *lens, *tables;
  int n, width, rows, group;
  int min_rows, max_rows;  // requests of min_rows..max_rows flat rows are this kernel's
  bool cut;                // items may be cut (and joined)
  float scale;             // times log2(e): the softmax is in powers of two
  float *parts;            // [grid][2] partial items
  int4 *meta;              // [grid][2]: the item that a CTA leaves unfinished; the CTAs that it is spread over, and
                           // whether the CTA gave up (many rows)
  bool vec_q, vec_o;
  int *err;          // raised when a wait ran out
  uint64_t wait_ns;  // limit of a wait
  uint32_t lost;     // bytes that a copy's barrier waits for and that never come: 0, or 16 where all waits shall run out
};

constexpr int kManyTile = 128;  // rows and tokens of a tile of the many-row kernel

// ------------------------------------------------------------ division of the work
struct Kv4Request {
  int row0;      // first row in q and out
  int flat;      // flat rows
  int base;      // position of the first row (negative: it sees nothing)
  int len;       // cached tokens
  int tiles;     // row tiles
  int64_t work;  // of one KV head
};

// Quotients of two non-negative 64-bit numbers that are nearly always small:
// a 64-bit division costs about 100 instructions.
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
  if (((a | b) >> 32) == 0) return (uint32_t)a / (uint32_t)b;
  return a / b;
}

// What beginning and ending an item costs, in steps of BN tokens. Without it
// the CTAs with many short items end last: a 4096-token prompt took 561 us
// instead of 372. 4 for the many-row kernel (299 us with the queries in L2; 3:
// 301, 6: 310), 1 for the other (48 ragged chats 90.5 us; 2: 91.1, 4: 96.7).
template <int RT>
constexpr int kv4_setup() { return RT == kManyTile ? 4 : 1; }

// Work of the first n row tiles of a request: for each its setup, then its steps. With `period` = G BN / RT row
// tiles to a step of BN tokens, and the tokens before the request's rows
// rounded up to whole steps, tile i counts floor(i / period) + 1 steps more:
// never fewer than its last row sees, and at most one more.
template <int RT, int BN>
__device__ __forceinline__ int64_t kv4_work(int base, int group, int n) {
  const int64_t before = (max(base, 0) + BN - 1) / BN + 1 + kv4_setup<RT>();
  if (n <= 1) return n ? before : 0;
  const int period = group * (BN / RT), full = n / period, rest = n % period;
  return n * before + (int64_t)period * full * (full - 1) / 2 + (int64_t)rest * full;
}

template <int RT, int BN>
__device__ __forceinline__ Kv4Request kv4_request(const Kv4AttnArgs &a, int r) {
  static_assert(BN % RT == 0, "");
  Kv4Request q;
  const int first = __ldg(a.offsets + r), end = __ldg(a.offsets + r + 1);
  const int64_t fresh = (int64_t)end - first;
  q.row0 = first;
  q.len = (int)min((int64_t)max(__ldg(a.lens + r), 0), (int64_t)a.width * a.c.page);
  q.base = (int)max((int64_t)q.len - fresh, (int64_t)INT_MIN);
  const int n = first >= 0 ? max(min(end, a.rows) - first, 0) : 0;
  q.flat = n * a.group;
  if (q.flat < a.min_rows || q.flat > a.max_rows) q.flat = 0;
  q.tiles = (q.flat + RT - 1) / RT;
  q.work = kv4_work<RT, BN>(q.base, a.group, q.tiles);
  return q;
}

// Work of row tile i.
template <int RT, int BN>
__device__ __forceinline__ int kv4_tile_work(const Kv4Request &q, int group, int i) {
  return (max(q.base, 0) + BN - 1) / BN + 1 + kv4_setup<RT>() + i / (group * (BN / RT));
}

// A walk along this CTA's piece of the line: the item it stands in, and what is left.
struct Kv4Walk {
  Kv4Request q;
  int r, head, tile;    // request, KV head, row tile
  int t, whole;         // BN-token tiles of the item behind this place, and all of them
  int64_t left;         // work left to this CTA
  int64_t line, place;  // the whole line, and the current place on it
  int ctas;             // pieces
};

// CTA `cta` of `grid`. All threads; a block-wide scan. false: no work for it.
template <int RT, int BN>
__device__ __forceinline__ bool kv4_walk(const Kv4AttnArgs &a, Kv4Walk &w, int cta, int grid) {
  __shared__ int64_t sums[32], s_at;
  __shared__ int s_r;
  const int per = (a.n + blockDim.x - 1) / blockDim.x;
  const int r0 = threadIdx.x * per, r1 = min(r0 + per, a.n);
  int64_t mine = 0;
  for (int r = r0; r < r1; ++r) mine += a.c.kv * kv4_request<RT, BN>(a, r).work;
  const int64_t upto = block_scan(mine, sums, w.line);
  if (w.line == 0) return false;
  w.ctas = (int)min((int64_t)grid, w.line);
  if (cta >= w.ctas) return false;
  w.place = quotient(cta * w.line, w.ctas);
  w.left = quotient((cta + 1) * w.line, w.ctas) - w.place;
  if (w.place >= upto - mine && w.place < upto) {
    int64_t at = w.place - (upto - mine);
    int r = r0;
    for (;; ++r) {
      const int64_t here = a.c.kv * kv4_request<RT, BN>(a, r).work;
      if (at < here) break;
      at -= here;
    }
    s_r = r, s_at = at;
  }
  __syncthreads();
  w.r = s_r;
  w.q = kv4_request<RT, BN>(a, w.r);
  w.head = (int)quotient(s_at, w.q.work);
  const int64_t in_head = s_at - w.head * w.q.work;
  int lo = 0, hi = w.q.tiles - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (kv4_work<RT, BN>(w.q.base, a.group, mid + 1) > in_head) hi = mid;
    else lo = mid + 1;
  }
  w.tile = lo;
  w.t = (int)(in_head - kv4_work<RT, BN>(w.q.base, a.group, lo));
  w.whole = kv4_tile_work<RT, BN>(w.q, a.group, lo);
  if (!a.cut || w.t <= kv4_setup<RT>()) w.left += w.t, w.place -= w.t, w.t = 0;  // no item is cut in its setup: see kv4_next
  return true;
}

struct Kv4Segment {
  Kv4Request q;
  int r, head, tile;  // request, KV head, row tile
  int t0, t1;         // BN-token tiles of this CTA
  int whole;          // of the item
};

// The next item's part of this CTA; advances the walk. false: done.
template <int RT, int BN>
__device__ __forceinline__ bool kv4_next(const Kv4AttnArgs &a, Kv4Walk &w, Kv4Segment &s) {
  if (w.left == 0) return false;
  if (w.t == w.whole) {
    w.t = 0;
    if (++w.tile == w.q.tiles) {
      w.tile = 0;
      if (++w.head == a.c.kv) {
        w.head = 0;
        do w.q = kv4_request<RT, BN>(a, ++w.r);
        while (w.q.work == 0);
      }
    }
    w.whole = kv4_tile_work<RT, BN>(w.q, a.group, w.tile);
  }
  const int setup = kv4_setup<RT>(), end = (int)min((int64_t)w.whole, w.t + w.left);
  if (end < w.whole && (!a.cut || end <= setup)) {  // a later CTA does this item
    w.left = 0;
    return false;
  }
  s.q = w.q;
  s.r = w.r, s.head = w.head, s.tile = w.tile;
  s.t0 = max(w.t - setup, 0), s.t1 = end - setup, s.whole = w.whole - setup;
  w.left -= end - w.t, w.place += end - w.t;
  w.t = end;
  return true;
}

// The CTAs from this one on that an item which ends at place `end` is spread over.
__device__ __forceinline__ int kv4_spread(const Kv4Walk &w, int64_t end) {
  return (int)quotient(end * w.ctas - 1, w.line) - (int)blockIdx.x + 1;
}

// ------------------------------------------------------------ fragments
__device__ __forceinline__ float ex2(float x) {  // 2^x, off by at most 2^-22 of it
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint32_t h2_bits(__half2 h) { return *reinterpret_cast<const uint32_t *>(&h); }
__device__ __forceinline__ __half2 bits_h2(uint32_t u) { return *reinterpret_cast<const __half2 *>(&u); }

// (x, y) as fp16 hi + lo pairs: 22 bits of each.
__device__ __forceinline__ void split_f16(float x, float y, uint32_t &hi, uint32_t &lo) {
  hi = h2_bits(__floats2half2_rn(x, y));
  float a, b;  // x and y less their hi parts, in one mixed-precision instruction each
  asm("{\n\t.reg .f16 h0, h1, m;\n\t"
      "mov.b32 {h0, h1}, %2;\n\t"
      "mov.b16 m, 0xBC00;\n\t"
      "fma.rn.f32.f16 %0, h0, m, %3;\n\t"
      "fma.rn.f32.f16 %1, h1, m, %4;\n\t}"
      : "=f"(a), "=f"(b)
      : "r"(hi), "f"(x), "f"(y));
  lo = h2_bits(__floats2half2_rn(a, b));
}

// Pairs of floats in one instruction.
__device__ __forceinline__ uint64_t two(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float2 of_two(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t add_two(uint64_t x, uint64_t y) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
  return r;
}
__device__ __forceinline__ uint64_t mul_two(uint64_t x, uint64_t y) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
  return r;
}
__device__ __forceinline__ uint64_t fma_two(uint64_t x, uint64_t y, uint64_t z) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(x), "l"(y), "l"(z));
  return r;
}

// D = A B + D: A 16 x 16 row-major, B 16 x 8 column-major, fp16; D fp32.
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// 2 nibbles of each half-word as codes c = q - 8: 1024 + q and 64 + q are fp16
// numbers that hold q in their low and in their next four bits.
__device__ __forceinline__ __half2 code_lo(uint32_t x) {
  return __hsub2(bits_h2((x & 0x000F000Fu) | 0x64006400u), __float2half2_rn(1032.0f));
}
__device__ __forceinline__ __half2 code_hi(uint32_t x) {
  return __hsub2(bits_h2((x & 0x00F000F0u) | 0x54005400u), __float2half2_rn(72.0f));
}

// N consecutive half-words of shared memory (aligned to the whole where N is even).
template <int N>
__device__ __forceinline__ void lds_halves(const uint8_t *p, uint32_t (&w)[(N + 1) / 2]) {
  if constexpr (N == 4) {
    const uint2 v = *reinterpret_cast<const uint2 *>(p);
    w[0] = v.x, w[1] = v.y;
  } else if constexpr (N == 2) {
    w[0] = *reinterpret_cast<const uint32_t *>(p);
  } else {
    const uint16_t *h = reinterpret_cast<const uint16_t *>(p);
    w[0] = h[0];
    if constexpr (N == 3) w[0] |= (uint32_t)h[1] << 16, w[1] = h[2];
  }
}

// Half-word j of a and of b side by side.
template <int W>
__device__ __forceinline__ uint32_t pair_halves(const uint32_t (&a)[W], const uint32_t (&b)[W], int j) {
  return __byte_perm(a[j >> 1], b[j >> 1], j & 1 ? 0x7632 : 0x5410);
}
template <int W>
__device__ __forceinline__ float half_at(const uint32_t (&a)[W], int j) {
  return __half2float(__ushort_as_half((uint16_t)(a[j >> 1] >> (j & 1 ? 16 : 0))));
}

// acc and total, in units of 2^top, joined with another sum; all -inf: nothing was seen.
__device__ __forceinline__ void kv4_add_part(float &top, float &total, float4 &acc, float ref, float sum, float4 v) {
  const float now = fmaxf(top, ref), shift = now == -INFINITY ? 0.0f : now;
  const float old = ex2(top - shift), k = ex2(ref - shift);
  top = now;
  total = total * old + k * sum;
  acc.x = acc.x * old + k * v.x, acc.y = acc.y * old + k * v.y;
  acc.z = acc.z * old + k * v.z, acc.w = acc.w * old + k * v.w;
}

// ------------------------------------------------------------ few rows
// One CTA, 4 warps, 8 flat rows an item. Every warp streams its own 16-token
// units through a ring of bulk copies in shared memory, without a barrier to
// the other warps, and keeps a softmax of its own; the four are joined at the
// item's end.
//
// m16n8k16 products with the query side as A: its 16 rows are the 8 rows' hi
// parts and their lo parts, so that both halves of a score land in one
// thread's accumulators. The weights of a score fragment are, in place, the A
// fragment of the product with V, again as hi and lo rows.
//   Scores: K enters as its codes c, and the block's scale is applied to its
//   32-element sum. (Codes q = c + 8, one operation an element pair cheaper,
//   with -8 sum(query) as the accumulator's start: the difference of large
//   sums put outputs 3e-6 off.)
//   Output: V is c d, exact in fp16.
// Tokens of a unit are taken in the order that keeps shared memory free of
// bank conflicts: column n of score tile i is token (n >> 1) + 4 (n & 1) + 8 i.
//
// Bound: latency of dependent instructions. A unit of 16 tokens x 8 rows x 128
// elements costs 524 instructions (measured), most of them decoding; 12 warps an
// SM (168 registers a thread) issue in 57 % of the slots, and that is 2.4 TB/s
// of cache on 48 ragged chats (89 us; the slots alone would take 43, the bytes
// 33). Three CTAs an SM: four had to spill (114 us). Two units a step: one took
// 99 us, four 104.
constexpr int kDecWarps = 4;
constexpr int kDecRowTile = 8;
constexpr int kDecUnits = 2;   // per warp and step
constexpr int kDecTokens = kDecWarps * kDecUnits * kKv4Unit;  // BN
constexpr int kDecStages = 3;
// Steps that one accumulator sums, two products each: a product truncates what
// it adds to, by up to 2^-23 of it and always towards 0, and equal weights added
// one by one round the same way every time (131072 tokens a CTA put outputs
// 1.9e-4 off in one chain). Chains are joined in F32, in the place of the item's
// part; up to 4096 tokens are one. 32 requests of 32768 tokens, 8 KV heads of
// 128: 412 us (64 steps: 409, no bound: 408).
constexpr int kDecChain = 32;
constexpr uint64_t kKv4WaitNs = 1000000000ull;  // limit of a wait, unless the cache was made with another
constexpr uint64_t kKv4DrainNs = 20000000ull;   // for what a CTA that gave up still has in flight

template <int NB>
struct DecSmem {
  static constexpr int kUnit = kv4_unit_bytes(NB);
  static constexpr int kRing = kDecStages * kDecUnits * kUnit;  // of a warp
  static constexpr int kRowStride = 32 * NB + 4;                // floats; rows 4 banks apart
  static constexpr int kBars = kDecWarps * kRing;
  static constexpr int kBytes = kBars + kDecWarps * kDecStages * 8;
  static_assert((kDecRowTile * (kRowStride + 2)) * 4 <= kRing, "a warp's result fits its ring");
};

__host__ __device__ constexpr int kv4_part_floats(int row_tile, int hd) { return row_tile * (hd + 2); }

template <int NB>
__global__ void __launch_bounds__(kDecWarps * 32, 3) kv4_decode_kernel(const Kv4AttnArgs a) {
  using L = DecSmem<NB>;
  constexpr int HD = 32 * NB, W = (NB + 1) / 2;
  constexpr int kPer = 32 / kDecUnits;  // steps a lookup
  constexpr uint32_t kAll = (1u << kDecUnits) - 1;
  extern __shared__ __align__(128) uint8_t sm[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  uint8_t *ring = sm + warp * L::kRing;
  uint64_t *bars = reinterpret_cast<uint64_t *>(sm + L::kBars) + warp * kDecStages;
  if (lane == 0) {
    for (int s = 0; s < kDecStages; ++s) sm100::mbar_init(&bars[s], 1);
    sm100::fence_mbar_init();
  }
  __shared__ int s_gone;  // a wait of this CTA ran out: all its rows from here on are NaN
  __shared__ float s_kept[2][2][kDecRowTile];  // of even and odd chains: references and sums
  if (threadIdx.x == 0) s_gone = 0;
  sm100::griddep_wait();
  sm100::griddep_launch_dependents();
  if (a.cut && threadIdx.x == 0) a.meta[2 * blockIdx.x + 1].x = 0;
  Kv4Walk walk;
  if (!kv4_walk<kDecRowTile, kDecTokens>(a, walk, blockIdx.x, gridDim.x)) return;
  __syncwarp();

  const int upp = a.c.page / kKv4Unit;  // units of a page
  const int64_t unit_page = a.c.page_head_bytes * a.c.kv;
  uint32_t steps_done = 0;  // of this warp, over all segments: the ring's place
  volatile int *gave_up = &s_gone;
  bool gone = false;
  Kv4Segment s;
  while (kv4_next<kDecRowTile, kDecTokens>(a, walk, s)) {
    // This thread's row of the tile: flat row f, and the last token that it sees.
    const int f = s.tile * kDecRowTile + g;
    const bool real = f < s.q.flat;
    const int qi = f / a.group;
    const int last = min(s.q.base + qi, s.q.len - 1);
    const int last_min = min(s.q.base + s.tile * kDecRowTile / a.group, s.q.len - 1);
    const int last_max = min(s.q.base + (min((s.tile + 1) * kDecRowTile, s.q.flat) - 1) / a.group, s.q.len - 1);
    const int *table = a.tables + (int64_t)s.r * a.width;
    const uint8_t *slice = kv4_unit(a.c, a.layer, 0, s.head, 0);

    // Queries as A fragments, scaled so that the row's largest element is in [2^14, 2^15).
    uint32_t qa[2 * NB][4];
    float fscale;
    {
      float x[NB][8];
      float mx = 0.0f;
      bool bad = false;
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        if (real) {
          const float *p = a.q + (s.q.row0 + qi) * a.ld_q + (s.head * a.group + f % a.group) * a.hs_q + 32 * j + 8 * t;
          if (a.vec_q) {
            const float4 u = *reinterpret_cast<const float4 *>(p), v = *reinterpret_cast<const float4 *>(p + 4);
            x[j][0] = u.x, x[j][1] = u.y, x[j][2] = u.z, x[j][3] = u.w;
            x[j][4] = v.x, x[j][5] = v.y, x[j][6] = v.z, x[j][7] = v.w;
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[j][i] = p[i];
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) x[j][i] = 0.0f;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) mx = fmaxf(mx, fabsf(x[j][i])), bad |= !isfinite(x[j][i]);
      }
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      bad = __shfl_xor_sync(0xffffffffu, (int)bad, 1) | bad;
      bad = __shfl_xor_sync(0xffffffffu, (int)bad, 2) | bad;
      const int e = min(141 - (int)(__float_as_uint(mx) >> 23), 126);  // 2^e mx in [2^14, 2^15)
      const float up = __uint_as_float((uint32_t)(127 + e) << 23);
      fscale = bad ? __uint_as_float(0x7fc00000u) : ldexpf(a.scale, -e);
#pragma unroll
      for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int p = 0; p < 2; ++p) {  // the element pairs of nibbles 2p and 2p + 1
          uint32_t(&A)[4] = qa[2 * j + p];
          split_f16(x[j][2 * p] * up, x[j][2 * p + 4] * up, A[0], A[1]);
          split_f16(x[j][2 * p + 1] * up, x[j][2 * p + 5] * up, A[2], A[3]);
        }
    }

    int from = s.t0;  // of the chain
    do {
      const int to = min(from + kDecChain, s.t1);
      const int first_unit = from * (kDecTokens / kKv4Unit);
      const int end_unit = min(to * (kDecTokens / kKv4Unit), (last_max + kKv4Unit) / kKv4Unit);
      const int steps =
          gone ? 0 : max(0, (end_unit - first_unit + kDecWarps * kDecUnits - 1) / (kDecWarps * kDecUnits));
      float o[4 * NB][4];
      float ref, sum;       // weights are 2^(score - ref): at most 2^15; their sum over this thread's tokens
      uint32_t poison = 0;  // blocks of this row with a NaN value that it sees
      // A row that does not see a token weighs it 0, which a NaN value would not
      // respect: a segment whose output has a NaN is done again with such values
      // set to 0 and the rows that see them marked.
      for (int careful = 0; careful < 2; ++careful) {
#pragma unroll
        for (int i = 0; i < 4 * NB; ++i)
#pragma unroll
          for (int c = 0; c < 4; ++c) o[i][c] = 0.0f;
        ref = -INFINITY, sum = 0.0f;

        // The ring: step k of this warp is units first_unit + (k * 4 + warp) * 2 + {0, 1}.
        uint32_t held = 0;  // kDecUnits bits a stage: units that were fetched
        // Every kPer steps each lane looks up one unit of the next kPer, and copies it when its step comes.
        const uint8_t *unit_at = nullptr;
        uint32_t there = 0;  // lanes whose unit is in the cache
        auto fetch = [&](int k) {
          if (k % kPer == 0) {
            const int u = first_unit + ((k + lane / kDecUnits) * kDecWarps + warp) * kDecUnits + lane % kDecUnits;
            const int id = u < end_unit ? __ldg(table + u / upp) : -1;
            const bool in = id >= 0 && id < a.c.pages;
            unit_at = slice + id * unit_page + (int64_t)(u % upp) * L::kUnit;
            there = __ballot_sync(0xffffffffu, in);
          }
          const uint32_t stage = (steps_done + k) % kDecStages, have = there >> (kDecUnits * (k % kPer)) & kAll;
          held = (held & ~(kAll << (kDecUnits * stage))) | have << (kDecUnits * stage);
          if (lane == 0) sm100::mbar_arrive_expect_tx(&bars[stage], __popc(have) * L::kUnit + a.lost);
          __syncwarp();
          if (lane / kDecUnits == k % kPer && (there >> lane & 1u))
            sm100::bulk_load(ring + (stage * kDecUnits + lane % kDecUnits) * L::kUnit, unit_at, L::kUnit, &bars[stage]);
        };
        for (int k = 0; k < min(kDecStages - 1, steps); ++k) fetch(k);

        for (int k = 0; k < steps; ++k) {
          if (k + kDecStages - 1 < steps) fetch(k + kDecStages - 1);
          const uint32_t stage = (steps_done + k) % kDecStages;
          if (!__all_sync(0xffffffffu, sm100::mbar_wait(&bars[stage], ((steps_done + k) / kDecStages) & 1u, a.err,
                                                        gave_up, a.wait_ns))) {
            gone = true;  // the copies in flight land before their places are used for anything else
            for (uint32_t i = steps_done + k; i < steps_done + min(k + kDecStages, steps); ++i)
              sm100::mbar_wait(&bars[i % kDecStages], (i / kDecStages) & 1u, nullptr, nullptr, kKv4DrainNs);
            break;
          }
          const uint32_t have = held >> (kDecUnits * stage) & kAll;
          const int u0 = first_unit + (k * kDecWarps + warp) * kDecUnits;
          const uint8_t *buf = ring + stage * kDecUnits * L::kUnit;

          // ---- scores: sc[unit][tile i][b] of token t + 4 b + 8 i
          float sc[kDecUnits][2][2];
          float mx = -INFINITY;
#pragma unroll
          for (int j = 0; j < kDecUnits; ++j) {
            const uint8_t *unit = buf + j * L::kUnit;
            if (!(have >> j & 1u)) {
#pragma unroll
              for (int i = 0; i < 4; ++i) sc[j][i >> 1][i & 1] = -INFINITY;
              continue;
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              uint32_t kw[NB];
              const uint8_t *kp = unit + ((g >> 1) + 4 * (g & 1) + 8 * i) * (16 * NB) + t * (4 * NB);
              if constexpr (NB == 4) {
                const uint4 v = *reinterpret_cast<const uint4 *>(kp);
                kw[0] = v.x, kw[1] = v.y, kw[2] = v.z, kw[3] = v.w;
              } else if constexpr (NB == 2) {
                const uint2 v = *reinterpret_cast<const uint2 *>(kp);
                kw[0] = v.x, kw[1] = v.y;
              } else {
#pragma unroll
                for (int b = 0; b < NB; ++b) kw[b] = reinterpret_cast<const uint32_t *>(kp)[b];
              }
              uint32_t d0[W], d1[W];
              lds_halves<NB>(unit + kv4_k_scale_off(NB) + (t + 8 * i) * (2 * NB), d0);
              lds_halves<NB>(unit + kv4_k_scale_off(NB) + (t + 4 + 8 * i) * (2 * NB), d1);
              uint64_t s01 = 0;  // the two tokens' scores
#pragma unroll
              for (int b = 0; b < NB; ++b) {
                float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                const uint32_t w = kw[b], w8 = w >> 8;
                mma16816(c, qa[2 * b], h2_bits(code_lo(w)), h2_bits(code_hi(w)));
                mma16816(c, qa[2 * b + 1], h2_bits(code_lo(w8)), h2_bits(code_hi(w8)));
                const uint64_t dd = two(half_at(d0, b), half_at(d1, b));
                s01 = fma_two(dd, two(c[0], c[1]), s01);
                s01 = fma_two(dd, two(c[2], c[3]), s01);
              }
              const float2 s2 = of_two(mul_two(s01, two(fscale, fscale)));
              sc[j][i][0] = s2.x, sc[j][i][1] = s2.y;
            }
            if ((u0 + j) * kKv4Unit + kKv4Unit - 1 > last_min) {  // some row's end
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if ((u0 + j) * kKv4Unit + t + 4 * (i & 1) + 8 * (i >> 1) > last) sc[j][i >> 1][i & 1] = -INFINITY;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) mx = fmaxf(mx, sc[j][i >> 1][i & 1]);
          }

          // ---- the weights' reference: moved only when a weight would pass 2^15
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          const bool grow = mx > ref + 15.0f || (ref == -INFINITY && mx > -INFINITY);
          if (__any_sync(0xffffffffu, grow)) {
            const float to = grow ? mx - 8.0f : ref;
            const float old = grow ? ex2(ref - to) : 1.0f;
            ref = to;
            sum *= old;
#pragma unroll
            for (int i = 0; i < 4 * NB; ++i)
#pragma unroll
              for (int c = 0; c < 4; ++c) o[i][c] *= old;
          }
          const float shift = ref == -INFINITY ? 0.0f : ref;

          // ---- weights and output
#pragma unroll
          for (int j = 0; j < kDecUnits; ++j) {
            if (!(have >> j & 1u)) continue;
            const uint8_t *unit = buf + j * L::kUnit;
            float p[4];  // tokens t, t + 4, t + 8, t + 12
#pragma unroll
            for (int i = 0; i < 4; ++i) p[i] = ex2(sc[j][i >> 1][i & 1] - shift), sum += p[i];
            uint32_t pa[4];
            split_f16(p[0], p[1], pa[0], pa[1]);
            split_f16(p[2], p[3], pa[2], pa[3]);
            uint32_t vw[4][W], vd[4][W];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int tok = t + 4 * i;
              lds_halves<NB>(unit + kv4_v_off(NB) + tok * (16 * NB) + g * (2 * NB), vw[i]);
              lds_halves<NB>(unit + kv4_v_scale_off(NB) + tok * (2 * NB), vd[i]);
            }
            const int tok0 = (u0 + j) * kKv4Unit + t;
            if ((u0 + j) * kKv4Unit + kKv4Unit - 1 > last_max) {  // tokens that no row sees may hold anything
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (tok0 + 4 * i > last_max)
#pragma unroll
                  for (int w = 0; w < W; ++w) vd[i][w] = 0u;
            }
            if (careful) {
#pragma unroll
              for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                  const int sh = b & 1 ? 16 : 0;
                  if ((vd[i][b >> 1] >> sh & 0x7fffu) > 0x7c00u) {
                    if (tok0 + 4 * i <= last) poison |= 1u << b;
                    vd[i][b >> 1] &= ~(0xffffu << sh);
                  }
                }
            }
#pragma unroll
            for (int b = 0; b < NB; ++b) {
              const uint32_t x0 = pair_halves(vw[0], vw[1], b), x1 = pair_halves(vw[2], vw[3], b);
              const __half2 e0 = bits_h2(pair_halves(vd[0], vd[1], b)), e1 = bits_h2(pair_halves(vd[2], vd[3], b));
              const uint32_t y0 = x0 >> 8, y1 = x1 >> 8;
              mma16816(o[4 * b], pa, h2_bits(__hmul2(code_lo(x0), e0)), h2_bits(__hmul2(code_lo(x1), e1)));
              mma16816(o[4 * b + 1], pa, h2_bits(__hmul2(code_hi(x0), e0)), h2_bits(__hmul2(code_hi(x1), e1)));
              mma16816(o[4 * b + 2], pa, h2_bits(__hmul2(code_lo(y0), e0)), h2_bits(__hmul2(code_lo(y1), e1)));
              mma16816(o[4 * b + 3], pa, h2_bits(__hmul2(code_hi(y0), e0)), h2_bits(__hmul2(code_hi(y1), e1)));
            }
          }
          __syncwarp();  // the stage's readers are done before lane 0 refills it
        }
        steps_done += steps;
        bool nan = false;
#pragma unroll
        for (int i = 0; i < 4 * NB; ++i)
#pragma unroll
          for (int c = 0; c < 4; ++c) nan |= isnan(o[i][c]);
        if (gone || !__any_sync(0xffffffffu, nan)) break;
      }
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      poison |= __shfl_xor_sync(0xffffffffu, poison, 1);
      poison |= __shfl_xor_sync(0xffffffffu, poison, 2);

      // ---- join the warps through their rings
      float *mine = reinterpret_cast<float *>(ring);
      if (t == 0) {
        mine[kDecRowTile * L::kRowStride + g] = ref;
        mine[kDecRowTile * L::kRowStride + kDecRowTile + g] = sum;
      }
#pragma unroll
      for (int b = 0; b < NB; ++b) {  // n8-tile i of block b, column n is element 32 b + 4 n + i
        float4 lo = make_float4(o[4 * b][0] + o[4 * b][2], o[4 * b + 1][0] + o[4 * b + 1][2],
                                o[4 * b + 2][0] + o[4 * b + 2][2], o[4 * b + 3][0] + o[4 * b + 3][2]);
        float4 hi = make_float4(o[4 * b][1] + o[4 * b][3], o[4 * b + 1][1] + o[4 * b + 1][3],
                                o[4 * b + 2][1] + o[4 * b + 2][3], o[4 * b + 3][1] + o[4 * b + 3][3]);
        if (poison >> b & 1u) {
          const float x = __uint_as_float(0x7fc00000u);
          lo = hi = make_float4(x, x, x, x);
        }
        float4 *dst = reinterpret_cast<float4 *>(mine + g * L::kRowStride + 32 * b + 8 * t);
        dst[0] = lo, dst[1] = hi;
      }
      __syncthreads();
      gone = *gave_up;  // (no warp goes on before all have read it)
      const bool done = to == s.t1, whole = s.t0 == 0 && s.t1 == s.whole;
      float *part = a.parts + (int64_t)(2 * blockIdx.x + (s.t0 == 0)) * kv4_part_floats(kDecRowTile, HD);
      const int now = (from - s.t0) / kDecChain & 1;
      for (int i = threadIdx.x; i < kDecRowTile * HD / 4; i += kDecWarps * 32) {
        const int row = i / (HD / 4), e = 4 * (i % (HD / 4)), fr = s.tile * kDecRowTile + row;
        if (fr >= s.q.flat) continue;
        float rw[kDecWarps], top = -INFINITY;
#pragma unroll
        for (int w = 0; w < kDecWarps; ++w) {
          rw[w] = reinterpret_cast<const float *>(sm + w * L::kRing)[kDecRowTile * L::kRowStride + row];
          top = fmaxf(top, rw[w]);
        }
        const float shift = top == -INFINITY ? 0.0f : top;
        float total = gone ? __uint_as_float(0x7fc00000u) : 0.0f;
        float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < kDecWarps; ++w) {
          const float *src = reinterpret_cast<const float *>(sm + w * L::kRing);
          const float k = ex2(rw[w] - shift);
          const float4 v = *reinterpret_cast<const float4 *>(src + row * L::kRowStride + e);
          total += k * src[kDecRowTile * L::kRowStride + kDecRowTile + row];
          acc.x += k * v.x, acc.y += k * v.y, acc.z += k * v.z, acc.w += k * v.w;
        }
        if (from > s.t0)  // the chains before, kept where the item's part has its place
          kv4_add_part(top, total, acc, s_kept[now ^ 1][0][row], s_kept[now ^ 1][1][row],
                       *reinterpret_cast<const float4 *>(part + 2 * kDecRowTile + row * HD + e));
        if (done && whole) {
          const float inv = total == 0.0f ? 0.0f : 1.0f / total;
          acc.x *= inv, acc.y *= inv, acc.z *= inv, acc.w *= inv;
          float *dst = a.out + (int64_t)(s.q.row0 + fr / a.group) * a.ld_o +
                       (int64_t)(s.head * a.group + fr % a.group) * a.hs_o + e;
          if (a.vec_o) *reinterpret_cast<float4 *>(dst) = acc;
          else dst[0] = acc.x, dst[1] = acc.y, dst[2] = acc.z, dst[3] = acc.w;
        } else {
          *reinterpret_cast<float4 *>(part + 2 * kDecRowTile + row * HD + e) = acc;
          if (e == 0 && done) part[row] = top, part[kDecRowTile + row] = total;
          if (e == 0 && !done) s_kept[now][0][row] = top, s_kept[now][1][row] = total;
        }
      }
      if (threadIdx.x == 0 && s.t0 == 0 && !whole && done) {  // the item goes on in the next CTAs
        a.meta[2 * blockIdx.x] = make_int4(s.q.row0, s.tile, s.head, s.q.flat);
        a.meta[2 * blockIdx.x + 1].x = kv4_spread(walk, walk.place - s.t1 + s.whole);
      }
      __syncthreads();
      sm100::fence_proxy_async_smem();  // the rings' next writers are bulk copies
      from = to;
    } while (from < s.t1);
  }
}

// Joins the parts of the items that their first CTA left unfinished. Items of
// 8 rows, which may have many parts: one a block, 4 elements a thread, every
// kJoinSlices-th part a slice, eight parts' loads in flight together. Items of
// 128 rows, mostly of two parts: 64 rows a block, 4 rows a thread. Parts are
// added in order, and slices in order. Blocks are few and large enough that all
// are resident at once: their latency (two dependent loads) is the time.
struct Kv4Join {
  const int4 *meta[2];
  const float *parts[2];
  int ctas[2];
};
constexpr int kJoinRows = 8;
constexpr int kJoinSlices = 2;
constexpr int kJoinBatch = 8;
constexpr int kJoinEach = 4;                                    // rows a thread of the large items
constexpr int kJoinMany = kJoinRows * kJoinSlices * kJoinEach;  // rows a block of them

// `parts0`: the two places of the item's first CTA; its own part is the second.
__device__ __forceinline__ const float *kv4_part(const float *parts0, int i, int64_t stride) {
  return parts0 + (2 * i + (i == 0)) * stride;
}

// Row fr of the item `m` (Kv4AttnArgs::meta): acc / total to elements e..e + 3.
__device__ __forceinline__ void kv4_write(const Kv4AttnArgs &a, int4 m, int fr, int e, float total, float4 acc) {
  const float inv = total == 0.0f ? 0.0f : 1.0f / total;
  acc.x *= inv, acc.y *= inv, acc.z *= inv, acc.w *= inv;
  float *dst =
      a.out + (int64_t)(m.x + fr / a.group) * a.ld_o + (int64_t)(m.z * a.group + fr % a.group) * a.hs_o + e;
  if (a.vec_o) *reinterpret_cast<float4 *>(dst) = acc;
  else dst[0] = acc.x, dst[1] = acc.y, dst[2] = acc.z, dst[3] = acc.w;
}

// NaN to all rows of the items that CTA `cta` of the many-row kernel had, or began. (A call, so that its registers are
// no matter to the join.)
template <int NB>
__device__ __noinline__ void kv4_void(const Kv4AttnArgs &a, int cta, int grid) {
  constexpr int HD = 32 * NB;
  Kv4Walk w;
  Kv4Segment s;
  if (!kv4_walk<kManyTile, kManyTile>(a, w, cta, grid)) return;
  while (kv4_next<kManyTile, kManyTile>(a, w, s)) {
    if (s.t0) continue;  // begun by an earlier CTA, whose join looks at this one's state
    for (int i = threadIdx.x; i < kManyTile * HD; i += blockDim.x) {
      const int f = s.tile * kManyTile + i / HD;
      if (f < s.q.flat)
        a.out[(int64_t)(s.q.row0 + f / a.group) * a.ld_o + (int64_t)(s.head * a.group + f % a.group) * a.hs_o + i % HD] =
            __uint_as_float(0x7fc00000u);
    }
  }
}

template <int NB>
__global__ void __launch_bounds__(kJoinRows * 8 * NB * kJoinSlices)
    kv4_join_kernel(const __grid_constant__ Kv4AttnArgs a, const Kv4Join j) {
  constexpr int HD = 32 * NB, kQuads = HD / 4, kLanes = kJoinRows * kQuads;
  __shared__ float4 s_acc[kJoinSlices][kLanes];
  __shared__ float s_top[kJoinSlices][kJoinRows], s_sum[kJoinSlices][kJoinRows];
  sm100::griddep_wait();
  if ((int)blockIdx.x >= j.ctas[0]) {
    constexpr int kRows = kManyTile, kChunks = kRows / kJoinMany;
    const int at = blockIdx.x - j.ctas[0], b = at / kChunks;
    const int4 m = j.meta[1][2 * b], state = j.meta[1][2 * b + 1];
    if (state.y) {
      if (at % kChunks == 0) kv4_void<NB>(a, b, j.ctas[1]);
      return;
    }
    const int parts = state.x;
    if (parts == 0) return;
    constexpr int64_t kStride = kv4_part_floats(kRows, HD);
    const float *parts0 = j.parts[1] + 2 * b * kStride;
    const int row0 = at % kChunks * kJoinMany + threadIdx.x / kQuads, e = 4 * (threadIdx.x % kQuads);
    float top[kJoinEach], total[kJoinEach];
    float4 acc[kJoinEach];
#pragma unroll
    for (int n = 0; n < kJoinEach; ++n) top[n] = -INFINITY, total[n] = 0.0f, acc[n] = make_float4(0, 0, 0, 0);
    for (int i = 0; i < parts; ++i) {
      const float *p = kv4_part(parts0, i, kStride);
      const bool gone = j.meta[1][2 * (b + i) + 1].y;  // the CTA gave up: its part may be anything
      float ref[kJoinEach], sum[kJoinEach];
      float4 v[kJoinEach];
#pragma unroll
      for (int n = 0; n < kJoinEach; ++n) {
        const int row = row0 + n * (kJoinRows * kJoinSlices);
        ref[n] = -INFINITY, sum[n] = 0.0f, v[n] = make_float4(0, 0, 0, 0);
        if (m.y * kRows + row < m.w) {  // rows past the item's have no parts
          ref[n] = p[row], sum[n] = p[kRows + row];
          v[n] = *reinterpret_cast<const float4 *>(p + 2 * kRows + row * HD + e);
        }
        if (gone) ref[n] = 0.0f, sum[n] = __uint_as_float(0x7fc00000u);
      }
#pragma unroll
      for (int n = 0; n < kJoinEach; ++n) kv4_add_part(top[n], total[n], acc[n], ref[n], sum[n], v[n]);
    }
#pragma unroll
    for (int n = 0; n < kJoinEach; ++n) {
      const int fr = m.y * kRows + row0 + n * (kJoinRows * kJoinSlices);
      if (fr < m.w) kv4_write(a, m, fr, e, total[n], acc[n]);
    }
    return;
  }
  const int b = blockIdx.x;
  const int4 m = j.meta[0][2 * b];
  const int parts = j.meta[0][2 * b + 1].x;
  if (parts == 0) return;
  constexpr int64_t kStride = kv4_part_floats(kDecRowTile, HD);
  const float *parts0 = j.parts[0] + 2 * b * kStride;
  const int lane = threadIdx.x % kLanes, slice = threadIdx.x / kLanes, row = lane / kQuads, e = 4 * (lane % kQuads);
  const int fr = m.y * kDecRowTile + row;
  const bool real = fr < m.w;
  float top = -INFINITY, total = 0.0f;
  float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int i0 = slice; real && i0 < parts; i0 += kJoinSlices * kJoinBatch) {
    float ref[kJoinBatch], sum[kJoinBatch];
    float4 v[kJoinBatch];
#pragma unroll
    for (int n = 0; n < kJoinBatch; ++n) {
      const int i = i0 + n * kJoinSlices;
      ref[n] = -INFINITY, sum[n] = 0.0f, v[n] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (i < parts) {
        const float *p = kv4_part(parts0, i, kStride);
        ref[n] = p[row], sum[n] = p[kDecRowTile + row];
        v[n] = *reinterpret_cast<const float4 *>(p + 2 * kDecRowTile + row * HD + e);
      }
    }
#pragma unroll
    for (int n = 0; n < kJoinBatch; ++n) kv4_add_part(top, total, acc, ref[n], sum[n], v[n]);
  }
  if (slice) s_acc[slice][lane] = acc;
  if (e == 0) s_top[slice][row] = top, s_sum[slice][row] = total;
  __syncthreads();
  if (slice || !real) return;
#pragma unroll
  for (int i = 1; i < kJoinSlices; ++i) kv4_add_part(top, total, acc, s_top[i][row], s_sum[i][row], s_acc[i][lane]);
  kv4_write(a, m, fr, e, total, acc);
}

}  // namespace mq
