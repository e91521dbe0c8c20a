// Causal attention over the paged 4-bit cache for many rows a request
// (prompts and their chunks): 128 flat rows an item, 128 tokens a step, on
// tcgen05. Work division and row semantics as in mq_kv4_attn.cuh.
//
// Per step, with Q and P as fp16 hi + lo pairs (22 bits) in TMEM and the
// cache's values, exact in fp16, in shared memory:
//   S = Qhi K^T + Qlo K^T            [128 rows, 128 tokens], fp32 in TMEM
//   P = 2^(S f - ref) -> Phi, Plo    one thread a row and half of the columns
//   O = Phi V + Plo V                [128 rows, hd], fp32 in TMEM
// and the running output of a row is in a thread's registers: adding one
// step's O there costs hd additions a row, keeps every tensor-core sum at 16
// additions (they truncate), and lets a moved reference scale registers.
// All lo products come before the hi ones: an addition truncates the sum that it
// makes, so the small terms go where sums are small. With them last, scores lost
// up to 8 more steps of 2^-23, and the outputs of four chunks of 300-700 rows
// were 1.07e-6 off instead of 0.47e-6.
// Both A operands come from TMEM, so shared memory feeds the tensor cores
// with B alone (64 of its 128 bytes a clock).
//
// Warps: 0-7 softmax (a thread: one row, half of a step's tokens), 8-11 the
// running output (a thread: one row), 12-15 decode K and 16-19 V (packed units
// -> swizzled tiles), 20 issues the MMAs, 21 the copies of the packed units, 22
// walks the items and hands their segments to the others through a ring.
// S of step i + 1 is computed while the softmax of step i runs, O of step i
// during the softmax of step i + 1; and an item is written out while the next
// one's queries are read.
//
// Bound: the tensor cores' 2048 clocks a step (twice 4 hd operations a (row,
// token) pair), and nearly as much the softmax chain of a step, which is longer
// by a quarter. Measured: a 4096-token prompt of 32 heads of 128 in 334 us, 0.82
// PFLOP/s of MMAs, where every pass has new queries, and 307 us with the queries
// in L2 (there 372 with the running output in the softmax warps).
//
// A wait that runs out makes the CTA's roles leave, whatever they have before
// them; the join then writes NaN for all that the CTA had (kv4_void).
#pragma once

#include "mq_kv4_attn.cuh"

namespace mq {

constexpr int kPreRows = kManyTile;    // RT
constexpr int kPreTokens = kManyTile;  // BN
constexpr int kPreSoft = 256;      // softmax threads
constexpr int kPreThreads = kPreSoft + 512;
constexpr int kPreGroups = kPreSoft / kPreRows;      // threads of a row
constexpr int kPreCols = kPreTokens / kPreGroups;    // of S a thread
constexpr int kWarpOut = kPreSoft / 32, kWarpK = kWarpOut + 4, kWarpV = kWarpK + 4, kWarpMma = kWarpV + 4, kWarpCopy = kWarpMma + 1,
              kWarpWalk = kWarpMma + 2;
constexpr int kPreRaw = 3;       // packed steps in flight
constexpr int kPreStages = 2;    // K and V tiles
constexpr int kPreMasks = 4;
constexpr int kPreSegs = 4;
constexpr int kStageRow = 80;  // bytes: 16 floats; 8 rows meet all banks once
constexpr int kPreUnits = kPreTokens / kKv4Unit;

// A segment as the roles need it.
enum { kSegEnd = 0, kSegWhole = 1, kSegTail = 2, kSegHead = 3 };  // of an item: all, a later part, its first part
struct PreSegment {
  int kind;
  int row0, flat, base, len;  // Kv4Request
  int request, head, tile;
  int t0, steps;              // first step, and the steps that some row sees
};

template <int NB>
struct PreSmem {
  static constexpr int HD = 32 * NB;
  static constexpr int kPanel = kPreTokens * 128;           // 64 head elements of every token
  static constexpr int kK = (NB + 1) / 2 * kPanel;
  static constexpr int kVPanel = HD * 128;                  // 64 tokens of every head element
  static constexpr int kV = 2 * kVPanel;
  static constexpr int kRaw = kPreUnits * kv4_unit_bytes(NB);
  static constexpr int kKOff = 0;
  static constexpr int kVOff = kPreStages * kK;
  static constexpr int kRawOff = kVOff + kPreStages * kV;
  static constexpr int kXchOff = kRawOff + kPreRaw * kRaw;  // floats [2 parities][groups][128 rows]
  static constexpr int kOldOff = kXchOff + 2 * kPreGroups * kPreRows * 4;  // floats [masks][128]: a step's factor
  static constexpr int kEndOff = kOldOff + kPreMasks * kPreRows * 4;       // floats [2 segments][sum, ref][128]
  static constexpr int kNanOff = kEndOff + 4 * kPreRows * 4;  // bytes [masks][NB][16 token groups]
  static constexpr int kStageOff = kNanOff + kPreMasks * NB * 16;  // 32 rows x 16 elements a warp
  static constexpr int kBarOff = kStageOff + (kPreSoft / 32 + 4) * 32 * kStageRow;
  static constexpr int kBars = 2 * kPreRaw + 4 * kPreStages + 12 + 2 * kPreSegs;
  static constexpr int kBytes = kBarOff + 8 * kBars + 64 + 16 * kPreSegs / 4 + kPreSegs * (int)sizeof(PreSegment);
  static constexpr int kAlloc = kBytes + 1024;  // slack for 1024-byte alignment
  static_assert(kAlloc <= 227 * 1024, "shared memory");
  static_assert(kK % 1024 == 0 && kVPanel % 1024 == 0 && kBarOff % 8 == 0, "swizzle atoms and barriers");
};

// TMEM columns. P replaces S in place: the 16 columns of 16 tokens' scores
// become 8 of their weights' hi parts and 8 of the lo parts; Q likewise
// replaces its own fp32 elements.
constexpr uint32_t kTmQ = 0;    // hd
constexpr uint32_t kTmS = 128;  // 2 x 128: even and odd steps
constexpr uint32_t kTmO = 384;  // hd

// Instruction descriptor, kind::f16: F16 x F16 -> F32, both K-major.
__host__ __device__ constexpr uint32_t idesc_half_f32(int M, int N) {
  return (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

__device__ __forceinline__ void umma_f16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
      "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void tm_ld16(uint32_t addr, uint32_t *r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
}
__device__ __forceinline__ void tm_st16(uint32_t addr, const uint32_t *r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
          addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tm_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float max_three(float x, float y, float z) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
  return r;
}

// One lane of a converged warp, the same one every time.
__device__ __forceinline__ bool elect_one() {
  uint32_t leader;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(leader));
  return leader != 0;
}

template <int N>
__device__ __forceinline__ void set_regs_up() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void set_regs_down() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
__device__ __forceinline__ void softmax_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kPreSoft) : "memory"); }

// A place in a ring of N barriers, and the parity of its current pass.
template <int N>
struct Ring {
  int i = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next() {
    if (++i == N) i = 0, phase ^= 1u;
  }
};

template <int NB>
__global__ void __launch_bounds__(kPreThreads, 1) kv4_prefill_kernel(const Kv4AttnArgs a) {
  using L = PreSmem<NB>;
  constexpr int HD = L::HD, W = (NB + 1) / 2, UB = kv4_unit_bytes(NB);
  extern __shared__ uint8_t pre_raw[];
  uint8_t *sm = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(pre_raw) + 1023) & ~uintptr_t(1023));
  uint64_t *raw_full = reinterpret_cast<uint64_t *>(sm + L::kBarOff), *raw_empty = raw_full + kPreRaw;
  uint64_t *k_full = raw_empty + kPreRaw, *k_empty = k_full + kPreStages;
  uint64_t *v_full = k_empty + kPreStages, *v_empty = v_full + kPreStages;
  uint64_t *q_full = v_empty + kPreStages, *s_full = q_full + 1, *p_full = s_full + 2, *o_full = p_full + 2,
           *fin = o_full + 1, *o_free = fin + 1, *end_full = o_free + 1, *end_empty = end_full + 2,
           *seg_full = end_empty + 2, *seg_empty = seg_full + kPreSegs;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(seg_empty + kPreSegs);
  volatile int *abort = reinterpret_cast<volatile int *>(tmem_slot + 1);
  uint32_t *raw_valid = tmem_slot + 2;   // [kPreRaw]: the packed units that were copied
  uint32_t *unit_mask = raw_valid + kPreRaw;  // [kPreMasks]: the same, for the softmax
  volatile uint32_t *nan_step = unit_mask + kPreMasks;  // [kPreMasks]: the last step in this place that had NaN values
  volatile int *soft_kind = reinterpret_cast<volatile int *>(const_cast<uint32_t *>(nan_step) + kPreMasks);
  PreSegment *segs = reinterpret_cast<PreSegment *>(const_cast<int *>(soft_kind) + 1);
  float *xch = reinterpret_cast<float *>(sm + L::kXchOff);
  float *olds = reinterpret_cast<float *>(sm + L::kOldOff), *ends = reinterpret_cast<float *>(sm + L::kEndOff);
  uint8_t *nan_bits = sm + L::kNanOff;

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kPreRaw; ++i) sm100::mbar_init(&raw_full[i], 1), sm100::mbar_init(&raw_empty[i], 256);
    for (int i = 0; i < kPreStages; ++i) {
      sm100::mbar_init(&k_full[i], 128), sm100::mbar_init(&k_empty[i], 1);
      sm100::mbar_init(&v_full[i], 128), sm100::mbar_init(&v_empty[i], 1);
    }
    sm100::mbar_init(q_full, kPreSoft);
    sm100::mbar_init(&s_full[0], 1), sm100::mbar_init(&s_full[1], 1);
    // (two of each: the softmax may be a step ahead of the MMAs, and a parity tells only neighbouring phases apart)
    sm100::mbar_init(&p_full[0], kPreSoft), sm100::mbar_init(&p_full[1], kPreSoft);
    sm100::mbar_init(o_full, 1);
    sm100::mbar_init(fin, 1);
    sm100::mbar_init(o_free, 128);
    for (int i = 0; i < 2; ++i) sm100::mbar_init(&end_full[i], 128), sm100::mbar_init(&end_empty[i], 128);
    for (int i = 0; i < kPreSegs; ++i) sm100::mbar_init(&seg_full[i], 1), sm100::mbar_init(&seg_empty[i], 15);
    *abort = 0;
    for (int i = 0; i < kPreMasks; ++i) nan_step[i] = ~0u;
    sm100::fence_mbar_init();
  }
  sm100::griddep_wait();
  sm100::griddep_launch_dependents();
  if (threadIdx.x == kWarpWalk * 32) a.meta[2 * blockIdx.x + 1] = make_int4(0, 0, 0, 0);  // the walker's
  Kv4Walk walk;
  const bool work = kv4_walk<kPreRows, kPreTokens>(a, walk, blockIdx.x, gridDim.x);
  if (work) {
    if (warp == kWarpMma) {
      sm100::tmem_alloc(tmem_slot, 512);
      sm100::tmem_relinquish();
    }
    sm100::tc_fence_before();
    __syncthreads();
    sm100::tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
    // Waits sleep in the barrier: polling took as many issue slots as the work.
    auto wait = [&](uint64_t *bar, uint32_t parity) {
      return sm100::mbar_wait_sleep(bar, parity, nullptr, abort, a.wait_ns);
    };
    // What is still in flight at the end. (Looked at once more when the time is up: it may have passed while another
    // process had the device.)
    auto drain = [&](uint64_t *bar, uint32_t parity) {
      if (!sm100::mbar_wait(bar, parity, nullptr, nullptr, kKv4DrainNs) && !sm100::mbar_try_wait(bar, parity)) *abort = 1;
    };
    Ring<kPreSegs> sg;
    // The next segment of a role's warp; false at the end. seg_done() lets the walker reuse its place.
    auto seg_next = [&]() {
      return __all_sync(0xffffffffu, wait(&seg_full[sg.i], sg.phase)) && segs[sg.i].kind != kSegEnd;
    };
    auto seg_done = [&]() {
      __syncwarp();
      if (lane == 0) sm100::mbar_arrive(&seg_empty[sg.i]);
      sg.next();
    };

    if (warp < kWarpOut) {
      // -------------------------------------------------------- softmax
      const int grp = warp >> 2, row = 32 * (warp & 3) + lane;
      const uint32_t lanes = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
      uint8_t *stage = sm + L::kStageOff + warp * 32 * kStageRow;
      Ring<2> score, end;
      Ring<kPreMasks> mask;
      int parity = 0;  // of the exchange buffers
      bool ok = true;
      // The values of this row's threads, by `join`.
      auto exchange = [&](float mine, auto join) {
        float *x = xch + parity * kPreGroups * kPreRows + row;
        x[grp * kPreRows] = mine;
        softmax_sync();
        parity ^= 1;
        return join(x[0], x[kPreRows]);
      };
      auto larger = [](float x, float y) { return fmaxf(x, y); };
      auto plus = [](float x, float y) { return x + y; };
      constexpr int QC = HD / kPreGroups;  // query elements of a thread
      static_assert(kPreGroups == 2, "");
      for (;;) {
        // One warp waits for the segment and decides for all, whatever comes: they share barriers.
        if (warp == 0) {
          const bool got = wait(&seg_full[sg.i], sg.phase);
          if (lane == 0) *soft_kind = got ? segs[sg.i].kind : (int)kSegEnd;
        }
        softmax_sync();
        if (*soft_kind == kSegEnd) break;
        const PreSegment &s = segs[sg.i];
        const int steps = s.steps, f = s.tile * kPreRows + row, qi = f / a.group;
        const bool real = f < s.flat;
        // The last token that the row sees, from the first of this thread's.
        int see = (real ? min(s.base + qi, s.len - 1) : -1) - s.t0 * kPreTokens - kPreCols * grp;
        uint64_t sums = 0;  // of the weights, two
        float ref = -INFINITY;
        if (steps > 0) {
          // ---- the thread's half of the row's elements, scaled so that the row's largest is in [2^14, 2^15). They are
          // read along the rows, handed out by row through shared memory, and kept in Q's place until the row's
          // largest is known. (The scores of the segment before are complete, so no MMA reads Q.)
          const bool sees = real && min(s.base + qi, s.len - 1) >= 0;
          const float *p = real ? a.q + (int64_t)(s.row0 + qi) * a.ld_q +
                                      (int64_t)(s.head * a.group + f % a.group) * a.hs_q + grp * QC
                                : nullptr;
          const uint32_t keep = lanes + kTmQ + QC * grp;
          const float *src[4];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            src[i] = reinterpret_cast<const float *>(
                __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(p), 8 * i + (lane >> 2)));
          auto load = [&](int c, float4 (&v)[4]) {
            const int e = 16 * c + 4 * (lane & 3);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              v[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
              if (src[i]) {
                if (a.vec_q) v[i] = *reinterpret_cast<const float4 *>(src[i] + e);
                else v[i] = make_float4(src[i][e], src[i][e + 1], src[i][e + 2], src[i][e + 3]);
              }
            }
          };
          float4 v[4], next[4];
          load(0, v);
          float mx = 0.0f;
          bool bad = false;
#pragma unroll 1
          for (int c = 0; c < QC / 16; ++c) {
            if (c + 1 < QC / 16) load(c + 1, next);
#pragma unroll
            for (int i = 0; i < 4; ++i)
              *reinterpret_cast<float4 *>(stage + (8 * i + (lane >> 2)) * kStageRow + 16 * (lane & 3)) = v[i];
            __syncwarp();
            uint32_t r[16];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint4 u = *reinterpret_cast<const uint4 *>(stage + lane * kStageRow + 16 * i);
              r[4 * i] = u.x, r[4 * i + 1] = u.y, r[4 * i + 2] = u.z, r[4 * i + 3] = u.w;
              v[i] = next[i];
            }
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float x = __uint_as_float(r[i]);
              mx = fmaxf(mx, fabsf(x)), bad |= !isfinite(x);
            }
            tm_st16(keep + 16 * c, r);
          }
          tm_st_wait();
          mx = exchange(bad ? INFINITY : mx, larger);
          bad = mx == INFINITY;
          const int e = min(141 - (int)(__float_as_uint(mx) >> 23), 126);
          float up = __uint_as_float((uint32_t)(127 + e) << 23);
          if (a.scale < 0.0f) up = -up;  // f is positive: the largest S is the largest score
          // (never 0, so that f * -inf is -inf; a row that sees nothing is 0 whatever its query)
          const float scale = bad && sees ? __uint_as_float(0x7fc00000u) : fmaxf(ldexpf(fabsf(a.scale), -e), 1.2e-38f);
#pragma unroll 1
          for (int c = 0; c < QC / 16; ++c) {
            uint32_t r[16], w[16];
            tm_ld16(keep + 16 * c, r);
            sm100::tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 8; ++i) {  // in the order of a decoded word: elements 0, 4, 1, 5, ... of every 8
              const int x = 8 * (i >> 2) + (i & 3);
              split_f16(__uint_as_float(r[x]) * up, __uint_as_float(r[x + 4]) * up, w[i], w[8 + i]);
            }
            tm_st16(keep + 16 * c, w);
          }
          tm_st_wait();
          sm100::tc_fence_before();
          sm100::mbar_arrive(q_full);

          for (int k = 0; k < steps; ++k) {
            ok = wait(&s_full[score.i], score.phase) && ok;
            const uint32_t cols = lanes + kTmS + 128 * score.i + kPreCols * grp;
            uint64_t *done = &p_full[score.i];
            score.next();
            sm100::tc_fence_after();
            const uint32_t units = unit_mask[mask.i] >> (4 * grp) & 15u;
            // (Loops of 16 columns keep the instruction cache: unrolled further, the roles' code evicted itself and a
            // step took up to three times as long.)
            // Hide what the row does not see (TMEM is read and written by whole warps).
            if (__any_sync(0xffffffffu, see < 63 || units != 15u)) {
#pragma unroll 1
              for (int c = 0; c < kPreCols; c += 16) {
                uint32_t r[16];
                tm_ld16(cols + c, r);
                sm100::tmem_ld_wait();
                const int seen = units >> (c >> 4) & 1u ? see - c : -1;
#pragma unroll
                for (int i = 0; i < 16; ++i)
                  if (i > seen) r[i] = 0xff800000u;
                tm_st16(cols + c, r);
              }
              tm_st_wait();
            }
            float top = -INFINITY;
#pragma unroll
            for (int c = 0; c < kPreCols; c += 32) {
              uint32_t r[32];
              tm_ld16(cols + c, r);
              tm_ld16(cols + c + 16, r + 16);
              sm100::tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 32; i += 2) top = max_three(top, __uint_as_float(r[i]), __uint_as_float(r[i + 1]));
            }
            top = exchange(top, larger) * scale;
            float old = 1.0f;
            if (top > ref + 15.0f || (ref == -INFINITY && top > -INFINITY)) {
              const float to = top - 8.0f;
              old = ex2(ref - to);
              ref = to;
            }
            if (grp == 0) olds[mask.i * kPreRows + row] = old;
            mask.next();
            const float shift = ref == -INFINITY ? 0.0f : ref;
            const uint64_t shifts = two(-shift, -shift), scales = two(scale, scale);
            uint64_t here = 0;  // the weights of the step (thousands of equal ones, added one by one, round one way)
#pragma unroll 1
            for (int c = 0; c < kPreCols; c += 16) {
              uint32_t r[16], w[16];
              tm_ld16(cols + c, r);
              sm100::tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 16; i += 2) {
                const float2 z = of_two(fma_two(two(__uint_as_float(r[i]), __uint_as_float(r[i + 1])), scales, shifts));
                const float p0 = ex2(z.x), p1 = ex2(z.y);
                here = add_two(here, two(p0, p1));
                split_f16(p0, p1, w[i >> 1], w[8 + (i >> 1)]);
              }
              tm_st16(cols + c, w);
            }
            sums = fma_two(sums, two(old, old), here);
            tm_st_wait();
            sm100::tc_fence_before();
            sm100::mbar_arrive(done);
            see -= kPreTokens;
          }
        }
        // ---- the rows' ends, for the output's warps
        const float2 halves = of_two(sums);
        const float total = exchange(halves.x + halves.y, plus);
        if (threadIdx.x == 0) sm100::mbar_arrive(&seg_empty[sg.i]);  // all have read it
        sg.next();
        if (grp == 0) {
          ok = wait(&end_empty[end.i], end.phase ^ 1u) && ok;
          ends[2 * end.i * kPreRows + row] = ok ? total : __uint_as_float(0x7fc00000u);
          ends[(2 * end.i + 1) * kPreRows + row] = ref;
          sm100::mbar_arrive(&end_full[end.i]);
          end.next();
        }
      }
    } else if (warp < kWarpK) {
      // -------------------------------------------------------- the running output
      set_regs_up<160>();
      const int row = 32 * (warp & 3) + lane;
      const uint32_t lanes = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
      uint8_t *stage = sm + L::kStageOff + warp * 32 * kStageRow;
      uint32_t o_phase = 0, step = 0;  // steps of this CTA, counted by the decode warps alike
      Ring<kPreMasks> mask;
      Ring<2> end;
      bool ok = true;
      auto all_wait = [&](uint64_t *bar, uint32_t phase) { return __all_sync(0xffffffffu, wait(bar, phase)) != 0; };
      for (; ok && seg_next(); seg_done()) {
        const PreSegment &s = segs[sg.i];
        const int steps = s.steps, f = s.tile * kPreRows + row, qi = f / a.group;
        const bool real = f < s.flat;
        int see = (real ? min(s.base + qi, s.len - 1) : -1) - s.t0 * kPreTokens;  // the last token that the row sees
        uint64_t acc[HD / 2];  // pairs
#pragma unroll
        for (int i = 0; i < HD / 2; ++i) acc[i] = 0;
        uint32_t poison = 0;
        for (int k = 0; ok && k < steps; ++k) {
          ok = all_wait(o_full, o_phase);
          o_phase ^= 1u;
          sm100::tc_fence_after();
          const float old = olds[mask.i * kPreRows + row];
          if (__any_sync(0xffffffffu, old != 1.0f)) {
#pragma unroll
            for (int i = 0; i < HD / 2; ++i) acc[i] = mul_two(acc[i], two(old, old));
          }
#pragma unroll
          for (int c = 0; c < HD; c += 16) {
            uint32_t r[16];
            tm_ld16(lanes + kTmO + c, r);
            sm100::tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 16; i += 2)
              acc[(c + i) / 2] = add_two(acc[(c + i) / 2], two(__uint_as_float(r[i]), __uint_as_float(r[i + 1])));
          }
          sm100::tc_fence_before();
          sm100::mbar_arrive(o_free);
          // NaN values of the step entered as 0: the rows that see them are marked.
          if (nan_step[mask.i] == step) {
            const uint64_t *bits = reinterpret_cast<const uint64_t *>(nan_bits + mask.i * NB * 16);
            auto upto = [](int n) { return n < 0 ? 0 : n >= 63 ? ~0ull : (2ull << n) - 1; };
            const uint64_t m0 = upto(see), m1 = upto(see - 64);
#pragma unroll
            for (int b = 0; b < NB; ++b)
              if ((bits[2 * b] & m0) | (bits[2 * b + 1] & m1)) poison |= 1u << b;
          }
          ++step;
          mask.next();
          see -= kPreTokens;
        }
        ok = all_wait(&end_full[end.i], end.phase) && ok;
        const float total = ok ? ends[2 * end.i * kPreRows + row] : __uint_as_float(0x7fc00000u);
        const float ref = ends[(2 * end.i + 1) * kPreRows + row];
        sm100::mbar_arrive(&end_empty[end.i]);
        end.next();
        const bool whole = s.kind == kSegWhole;
        float *dst = nullptr;
        float inv = 1.0f;
        if (!ok) poison = ~0u;
        if (real && whole) {
          dst = a.out + (int64_t)(s.row0 + qi) * a.ld_o + (int64_t)(s.head * a.group + f % a.group) * a.hs_o;
          inv = total == 0.0f ? 0.0f : 1.0f / total;
        } else if (real) {
          float *part = a.parts + (int64_t)(2 * blockIdx.x + (s.kind == kSegHead)) * kv4_part_floats(kPreRows, HD);
          dst = part + 2 * kPreRows + row * HD;
          part[row] = ref, part[kPreRows + row] = total;
        }
        const bool vec = a.vec_o || !whole;
        float *to[4];  // of the rows that this lane writes parts of
#pragma unroll
        for (int i = 0; i < 4; ++i)
          to[i] = reinterpret_cast<float *>(
              __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(dst), 8 * i + (lane >> 2)));
#pragma unroll
        for (int c = 0; c < HD; c += 16) {
          const float nan = __uint_as_float(0x7fc00000u);
          const bool dead = poison >> (c / 32) & 1u;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 u = of_two(mul_two(acc[(c + 4 * i) / 2], two(inv, inv)));
            const float2 v = of_two(mul_two(acc[(c + 4 * i) / 2 + 1], two(inv, inv)));
            *reinterpret_cast<float4 *>(stage + lane * kStageRow + 16 * i) =
                dead ? make_float4(nan, nan, nan, nan) : make_float4(u.x, u.y, v.x, v.y);
          }
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float4 o = *reinterpret_cast<const float4 *>(stage + (8 * i + (lane >> 2)) * kStageRow + 16 * (lane & 3));
            if (to[i]) {
              float *d = to[i] + c + 4 * (lane & 3);
              if (vec) *reinterpret_cast<float4 *>(d) = o;
              else d[0] = o.x, d[1] = o.y, d[2] = o.z, d[3] = o.w;
            }
          }
          __syncwarp();
        }
      }
    } else if (warp < kWarpV) {
      // -------------------------------------------------------- packed units -> K tiles
      // A warp takes 8 tokens x 4 chunks at a time, paired so that neither the loads nor the stores meet a bank
      // twice. Token: 32 it + tk0, whose unit is 2 it + half a warp pair's.
      const int dw = warp - kWarpK, tk0 = 8 * dw + (lane & 7), t = (lane >> 3) ^ ((lane & 7) >> 1), tk = tk0 & 15;
      const int u0 = tk0 >> 4;
      const uint32_t src0 = L::kRawOff + u0 * UB + tk * (16 * NB) + t * (4 * NB);
      const uint32_t scale0 = L::kRawOff + u0 * UB + kv4_k_scale_off(NB) + tk * (2 * NB);
      const uint32_t dst0 = L::kKOff + tk0 * 128 + ((t ^ (lane & 7)) << 4);  // even blocks; odd ones are 64 bytes away
      set_regs_down<56>();
      Ring<kPreRaw> raw;
      Ring<kPreStages> st;
      Ring<kPreMasks> mask;
      bool ok = true;
      for (; ok && seg_next(); seg_done()) {
        const int steps = segs[sg.i].steps;
        for (int k = 0; k < steps; ++k) {
          if (!(ok = wait(&raw_full[raw.i], raw.phase))) break;
          if (!(ok = wait(&k_empty[st.i], st.phase ^ 1u))) break;
          const uint32_t valid = raw_valid[raw.i];
          if (threadIdx.x == kWarpK * 32) unit_mask[mask.i] = valid;
          const uint8_t *src = sm + src0 + raw.i * L::kRaw, *scale = sm + scale0 + raw.i * L::kRaw;
          uint8_t *dst = sm + dst0 + st.i * L::kK;
#pragma unroll 1
          for (int it = 0; it < 4; ++it) {
            uint32_t kw[NB], d[W];
            const uint8_t *kp = src + it * 2 * UB;
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
            lds_halves<NB>(scale + it * 2 * UB, d);
            if (!(valid >> (2 * it + u0) & 1u)) {
#pragma unroll
              for (int i = 0; i < W; ++i) d[i] = 0u;
            }
#pragma unroll
            for (int b = 0; b < NB; ++b) {
              const __half2 dd = bits_h2(pair_halves(d, d, b));
              const uint32_t w = kw[b], w8 = w >> 8;
              uint4 o;
              o.x = h2_bits(__hmul2(code_lo(w), dd)), o.y = h2_bits(__hmul2(code_hi(w), dd));
              o.z = h2_bits(__hmul2(code_lo(w8), dd)), o.w = h2_bits(__hmul2(code_hi(w8), dd));
              uint8_t *p = b & 1 ? sm + ((uint32_t)(dst - sm) ^ 64u) : dst;
              *reinterpret_cast<uint4 *>(p + (b >> 1) * L::kPanel + it * 32 * 128) = o;
            }
          }
          sm100::fence_proxy_async_smem();
          sm100::mbar_arrive(&k_full[st.i]);
          sm100::mbar_arrive(&raw_empty[raw.i]);
          raw.next(), st.next(), mask.next();
        }
      }
    } else if (warp < kWarpMma) {
      // -------------------------------------------------------- packed units -> V tiles
      // A thread takes 8 tokens and 4 elements of every block, two blocks at a time. Odd token groups read their
      // tokens in pairs swapped, which spares half of the bank conflicts.
      const int dw = warp - kWarpV, m = 4 * dw + (lane & 3), g = lane >> 2, odd = m & 1;
      const uint32_t src0 = L::kRawOff + (m >> 1) * UB + kv4_v_off(NB) + (8 * odd) * (16 * NB) + g * (2 * NB);
      const uint32_t scale0 = L::kRawOff + (m >> 1) * UB + kv4_v_scale_off(NB) + (8 * odd) * (2 * NB);
      const uint32_t dst0 = L::kVOff + (m >> 3) * L::kVPanel + 4 * g * 128;
      uint32_t step = 0;
      set_regs_down<56>();
      Ring<kPreRaw> raw;
      Ring<kPreStages> st;
      Ring<kPreMasks> mask;
      bool ok = true;
      for (; ok && seg_next(); seg_done()) {
        const int steps = segs[sg.i].steps;
        for (int k = 0; k < steps; ++k) {
          if (!(ok = wait(&raw_full[raw.i], raw.phase))) break;
          if (!(ok = wait(&v_empty[st.i], st.phase ^ 1u))) break;
          const bool have = raw_valid[raw.i] >> (m >> 1) & 1u;
          // tokens 0, 2, 4, 6 and 1, 3, 5, 7 of the group, or the other way round
          const uint8_t *w0 = sm + src0 + raw.i * L::kRaw + odd * (16 * NB), *w1 = w0 + (1 - 2 * odd) * (16 * NB);
          const uint8_t *d0 = sm + scale0 + raw.i * L::kRaw + odd * (2 * NB), *d1 = d0 + (1 - 2 * odd) * (2 * NB);
          uint8_t *dst = sm + dst0 + st.i * L::kV;
#pragma unroll 1
          for (int b2 = 0; b2 < W; ++b2) {
            uint32_t vw[8], vd[8];
            __half2 check = __float2half2_rn(0.0f);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const uint8_t *pw = (i & 1 ? w1 : w0) + (i & ~1) * (16 * NB) + 4 * b2;
              const uint8_t *pd = (i & 1 ? d1 : d0) + (i & ~1) * (2 * NB) + 4 * b2;
              if constexpr (NB % 2 == 0) {
                vw[i] = *reinterpret_cast<const uint32_t *>(pw), vd[i] = *reinterpret_cast<const uint32_t *>(pd);
              } else {  // half-words; a row's last block stands alone
                vw[i] = *reinterpret_cast<const uint16_t *>(pw), vd[i] = *reinterpret_cast<const uint16_t *>(pd);
                if (2 * b2 + 1 < NB) {
                  vw[i] |= (uint32_t)reinterpret_cast<const uint16_t *>(pw)[1] << 16;
                  vd[i] |= (uint32_t)reinterpret_cast<const uint16_t *>(pd)[1] << 16;
                }
              }
              if (!have) vd[i] = 0u;
              check = __hadd2(check, __habs2(bits_h2(vd[i])));
            }
            uint32_t bad[2] = {0u, 0u};
            const uint32_t cb = h2_bits(check);
            if ((cb & 0x7c00u) == 0x7c00u || (cb & 0x7c000000u) == 0x7c000000u) {  // a NaN scale, or large ones
#pragma unroll
              for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                  if ((vd[i] >> (16 * h) & 0x7fffu) >= 0x7c00u) {
                    bad[h] |= 1u << (i ^ odd);
                    vd[i] &= ~(0xffffu << (16 * h));
                  }
              if (bad[0] | bad[1]) nan_step[mask.i] = step;
            }
#pragma unroll 1
            for (int h = 0; h < (NB == 1 ? 1 : 2); ++h) {
              const int b = 2 * b2 + h;
              if (b >= NB) break;
              if (g == 0) nan_bits[(mask.i * NB + b) * 16 + m] = (uint8_t)(h ? bad[1] : bad[0]);
              const uint32_t sel = odd ? (h ? 0x3276u : 0x1054u) : (h ? 0x7632u : 0x5410u);
              uint32_t o[4][4];
#pragma unroll
              for (int p = 0; p < 4; ++p) {
                const uint32_t x = __byte_perm(vw[2 * p], vw[2 * p + 1], sel), y = x >> 8;
                const __half2 dd = bits_h2(__byte_perm(vd[2 * p], vd[2 * p + 1], sel));
                o[0][p] = h2_bits(__hmul2(code_lo(x), dd)), o[1][p] = h2_bits(__hmul2(code_hi(x), dd));
                o[2][p] = h2_bits(__hmul2(code_lo(y), dd)), o[3][p] = h2_bits(__hmul2(code_hi(y), dd));
              }
#pragma unroll
              for (int i = 0; i < 4; ++i)  // element 32 b + 4 g + i
                *reinterpret_cast<uint4 *>(dst + (32 * b + i) * 128 + (((m & 7) ^ (4 * (g & 1) + i)) << 4)) =
                    make_uint4(o[i][0], o[i][1], o[i][2], o[i][3]);
            }
          }
          sm100::fence_proxy_async_smem();
          sm100::mbar_arrive(&v_full[st.i]);
          sm100::mbar_arrive(&raw_empty[raw.i]);
          raw.next(), st.next(), mask.next();
          ++step;
        }
      }
    } else {
      set_regs_down<48>();
      if (warp == kWarpMma) {
        // ------------------------------------------------------ MMA issue
        // The whole warp walks and waits, one lane issues: operands computed by whole warps stay in uniform
        // registers, where the instruction wants them (from one lane's registers an MMA took 95 clocks to issue,
        // and 64 to run).
        constexpr uint32_t id_s = idesc_half_f32(kPreRows, kPreTokens), id_o = idesc_half_f32(kPreRows, HD);
        const uint64_t k_desc = sm100::umma_desc_sw128(sm100::smem_u32(sm + L::kKOff));
        const uint64_t v_desc = sm100::umma_desc_sw128(sm100::smem_u32(sm + L::kVOff));
        Ring<kPreStages> ks, vs;
        uint32_t q_phase = 0, free_phase = 1;  // O is free at first
        int sb = 0;     // S buffer of the next scores
        Ring<2> pbuf;  // of the next output
        bool ok = true;
        auto all_wait = [&](uint64_t *bar, uint32_t parity) {
          return __all_sync(0xffffffffu, sm100::mbar_wait(bar, parity, nullptr, abort, a.wait_ns)) != 0;
        };
        for (; ok && seg_next(); seg_done()) {
          const int steps = segs[sg.i].steps;
          if (steps == 0) continue;
          if (!(ok = all_wait(q_full, q_phase))) break;
          q_phase ^= 1u;
          // S of a step may replace the P of two steps before: the MMAs of one thread run in order.
          auto scores = [&]() {
            if (!all_wait(&k_full[ks.i], ks.phase)) return false;
            sm100::tc_fence_after();
            const uint64_t desc = k_desc + (uint64_t)(ks.i * (L::kK >> 4));
            const uint32_t d = tmem + kTmS + 128 * sb;
            if (elect_one()) {
#pragma unroll
              for (int part = 1; part >= 0; --part)
#pragma unroll
                for (int kk = 0; kk < 2 * NB; ++kk)
                  umma_f16_ts(d, tmem + kTmQ + 16 * kk + 8 * part, desc + (kk >> 2) * (L::kPanel >> 4) + 2 * (kk & 3),
                              id_s, !part || kk);
              sm100::umma_commit(&s_full[sb]);
              sm100::umma_commit(&k_empty[ks.i]);
            }
            __syncwarp();
            ks.next();
            sb ^= 1;
            return true;
          };
          if (!(ok = scores())) break;
          for (int k = 0; k < steps; ++k) {
            if (k + 1 < steps && !(ok = scores())) break;
            if (!(ok = all_wait(&v_full[vs.i], vs.phase) && all_wait(&p_full[pbuf.i], pbuf.phase) && all_wait(o_free, free_phase)))
              break;
            free_phase ^= 1u;
            sm100::tc_fence_after();
            const uint64_t desc = v_desc + (uint64_t)(vs.i * (L::kV >> 4));
            const uint32_t p = tmem + kTmS + 128 * pbuf.i;
            if (elect_one()) {
#pragma unroll
              for (int part = 1; part >= 0; --part)
#pragma unroll
                for (int kk = 0; kk < kPreTokens / 16; ++kk)
                  umma_f16_ts(tmem + kTmO, p + 16 * kk + 8 * part,
                              desc + (kk >> 2) * (L::kVPanel >> 4) + 2 * (kk & 3), id_o, !part || kk);
              sm100::umma_commit(o_full);
              sm100::umma_commit(&v_empty[vs.i]);
            }
            __syncwarp();
            vs.next();
            pbuf.next();
          }
        }
        if (elect_one()) {  // every MMA has completed before the TMEM is released
          sm100::umma_commit(fin);
          drain(fin, 0u);
        }
      } else if (warp == kWarpCopy) {
        // ------------------------------------------------------ copies of the packed units
        const int upp = a.c.page / kKv4Unit;
        const int64_t unit_page = a.c.page_head_bytes * a.c.kv;
        Ring<kPreRaw> raw;
        bool ok = true;
        int issued = 0;
        for (; ok && seg_next(); seg_done()) {
          const PreSegment s = segs[sg.i];
          const int steps = s.steps, end_unit = (s.len + kKv4Unit - 1) / kKv4Unit;
          const int *table = a.tables + (int64_t)s.request * a.width;
          const uint8_t *slice = kv4_unit(a.c, a.layer, 0, s.head, 0);
          for (int k = 0; k < steps; ++k) {
            const int u = (s.t0 + k) * kPreUnits + lane;
            int id = lane < kPreUnits && u < end_unit ? __ldg(table + u / upp) : -1;
            if (id >= a.c.pages) id = -1;
            const uint32_t have = __ballot_sync(0xffffffffu, id >= 0);
            ok = __all_sync(0xffffffffu, wait(&raw_empty[raw.i], raw.phase ^ 1u));
            if (!ok) break;
            if (lane == 0) {
              raw_valid[raw.i] = have;
              sm100::mbar_arrive_expect_tx(&raw_full[raw.i], __popc(have) * UB + a.lost);
            }
            __syncwarp();
            if (id >= 0)
              sm100::bulk_load(sm + L::kRawOff + raw.i * L::kRaw + lane * UB,
                               slice + id * unit_page + (int64_t)(u % upp) * UB, UB, &raw_full[raw.i]);
            raw.next();
            ++issued;
          }
        }
        // the last copies have landed before the CTA can exit
        for (int i = max(0, issued - kPreRaw); i < issued; ++i)
          drain(&raw_full[i % kPreRaw], (uint32_t)(i / kPreRaw) & 1u);
      } else if (warp == kWarpWalk && lane == 0) {
        // ------------------------------------------------------ the walk over the items
        Kv4Segment s;
        for (bool more = true; more; sg.next()) {
          more = kv4_next<kPreRows, kPreTokens>(a, walk, s);
          if (!wait(&seg_empty[sg.i], sg.phase ^ 1u)) break;
          PreSegment &d = segs[sg.i];
          if (more) {
            const bool whole = s.t0 == 0 && s.t1 == s.whole;
            const int f = min((s.tile + 1) * kPreRows, s.q.flat) - 1, last = min(s.q.base + f / a.group, s.q.len - 1);
            d.kind = whole ? kSegWhole : s.t0 == 0 ? kSegHead : kSegTail;
            d.row0 = s.q.row0, d.flat = s.q.flat, d.base = s.q.base, d.len = s.q.len;
            d.request = s.r, d.head = s.head, d.tile = s.tile, d.t0 = s.t0;
            d.steps = max(0, min(s.t1, (last + kPreTokens) / kPreTokens) - s.t0);
            if (d.kind == kSegHead) {  // the item goes on in the next CTAs
              a.meta[2 * blockIdx.x] = make_int4(s.q.row0, s.tile, s.head, s.q.flat);
              a.meta[2 * blockIdx.x + 1].x = kv4_spread(walk, walk.place - s.t1 + s.whole);
            }
          } else {
            d.kind = kSegEnd;
          }
          sm100::mbar_arrive(&seg_full[sg.i]);
        }
      }
    }
    __syncwarp();
    sm100::tc_fence_before();
    __syncthreads();
    if (threadIdx.x == 0 && *abort) {  // the roles have left the items that were still to come: the join sees to them
      a.meta[2 * blockIdx.x + 1].y = 1;
      atomicExch(a.err, 1);
    }
    if (warp == kWarpMma) {
      sm100::tc_fence_after();
      sm100::tmem_dealloc(tmem, 512);
    }
  }
}

}  // namespace mq
