// Block tables and slot maps of a ragged batch, built on the GPU.
//
// A cache page holds `page` consecutive tokens of one request; a request's
// block table lists its pages, and token p of it lives in slot
// table[p / page] * page + p % page. A step brings new_r rows to request r,
// which holds ctx_r tokens: the plan appends the pages that they need, taken
// from the top of a stack of free pages in request order, and writes every
// row's slot and position.
//
//   held_r = ceil(ctx_r / page), need_r = ceil((ctx_r + new_r) / page)
//   offset_r = sum of new over the requests before r, first_r = sum of
//   need - held over them; page i >= held_r of request r is
//   free[n_free - 1 - (first_r + i - held_r)].
//
// The bytes are few (a thousand requests with 64k rows: 0.5 MB), so latency
// bounds it: one launch, in which every CTA computes the two prefix sums itself
// (R loads, no exchange) and writes its share of the rows. Where outputs replace
// inputs (the lengths, the stack's size) the CTAs are one cluster and wait once
// for one another, between reading and writing. 8 requests: 4.9 us in a graph;
// 1000 requests and 65 k rows: 12.3 us as a cluster of 8, 8.7 as 17 CTAs.
#pragma once

#include "mq_common.cuh"
#include "mq_sm100.cuh"

namespace mq {

constexpr int kPagesThreads = 1024;
constexpr int kPagesMaxSeqs = 8192;  // shared memory: 12 bytes a request
constexpr int kPagesCluster = 8;     // CTAs of a large batch planned in place
constexpr int kPagesCtas = 64;       // and otherwise, at most

struct PagesArgs {
  const int *ctx, *fresh;  // tokens held and tokens brought, per request
  int n, page;
  int *tables;
  int width;  // pages per table row
  const int *stack;
  int capacity;
  const int *n_free;
  int rows;
  int *offsets, *lens, *slots, *positions, *n_free_out, *refused;
  bool vec;       // slots and positions are aligned to 16 bytes
  bool in_place;  // seq_lens is ctx_lens, or n_free_out is n_free
};

__host__ __device__ constexpr size_t pages_smem(int n) { return (size_t)(3 * n + 1) * sizeof(int); }

__device__ __forceinline__ int64_t warp_scan(int64_t v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  return v;
}

// Inclusive sum over the CTA's threads (whole warps); `total` the CTA's sum. Two barriers.
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t *warp_sums, int64_t &total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nwarps = blockDim.x >> 5;
  v = warp_scan(v);
  if (lane == 31) warp_sums[warp] = v;
  __syncthreads();
  const int64_t sums = warp_scan(lane < nwarps ? warp_sums[lane] : 0);
  total = __shfl_sync(0xffffffffu, sums, 31);
  const int64_t before = __shfl_sync(0xffffffffu, sums, warp ? warp - 1 : 0);
  __syncthreads();
  return v + (warp ? before : 0);
}

// Pages of n tokens, 0 <= n <= INT_MAX, in 32 bits (64-bit divisions were half of the kernel's time).
__device__ __forceinline__ int pages_of(int n, int page) { return (int)(((uint32_t)n + page - 1) / (uint32_t)page); }

__global__ void __launch_bounds__(kPagesThreads) pages_plan_kernel(const PagesArgs a) {
  extern __shared__ int pages_sm[];
  __shared__ int64_t warp_sums[kPagesThreads / 32];
  int *off = pages_sm, *ctx = off + a.n + 1, *first = ctx + a.n;  // first: -1 of a refused request
  const int ncta = gridDim.x, cta = blockIdx.x;
  const int n_free = min(max(*a.n_free, 0), a.capacity);
  const int64_t room = (int64_t)a.width * a.page;
  int64_t rows_before = 0, pages_before = 0;  // over earlier chunks of requests
  int refused = 0, taken = 0;                 // this thread's
  for (int r0 = 0; r0 < a.n; r0 += blockDim.x) {
    const int r = r0 + threadIdx.x;
    const bool real = r < a.n;
    const int c = real ? a.ctx[r] : 0, m = real ? a.fresh[r] : 0;
    int64_t sum;
    const int64_t end = rows_before + block_scan(max(m, 0), warp_sums, sum);
    rows_before += sum;
    const bool fits = real && c >= 0 && m >= 0 && (int64_t)c + m <= room && end <= a.rows;
    const int more = fits ? pages_of(c + m, a.page) - pages_of(c, a.page) : 0;
    const int64_t upto = pages_before + block_scan(more, warp_sums, sum);
    pages_before += sum;
    if (real) {
      const bool served = fits && (more == 0 || upto <= n_free);
      off[r + 1] = (int)min(end, (int64_t)INT_MAX);
      ctx[r] = c;
      first[r] = served ? (int)min(upto - more, (int64_t)INT_MAX) : -1;
      refused += !served;
      taken += served ? more : 0;
    }
  }
  if (threadIdx.x == 0) off[0] = 0;
  int64_t both;  // refused requests and, below them, taken pages; the barriers order the writes of off, ctx and first
  block_scan((int64_t)refused << 40 | taken, warp_sums, both);
  if (ncta > 1 && a.in_place) sm100::cluster_sync();  // every CTA has read what is replaced
  if (cta == 0) {
    for (int r = threadIdx.x; r < a.n; r += blockDim.x) {
      a.offsets[r + 1] = off[r + 1];
      a.lens[r] = first[r] < 0 ? ctx[r] : ctx[r] + off[r + 1] - off[r];
    }
    if (threadIdx.x == 0) {
      a.offsets[0] = 0;
      *a.n_free_out = n_free - (int)(both & ((1ll << 40) - 1));
      *a.refused = (int)(both >> 40);
    }
  }
  // Four neighbouring rows a thread: one search, mostly one page.
  const int total = off[a.n];
  for (int64_t row0 = 4 * ((int64_t)cta * blockDim.x + threadIdx.x); row0 < a.rows;
       row0 += 4 * (int64_t)ncta * blockDim.x) {
    int slot[4], pos[4], r = 0, known = -1, id = 0;  // `id`: page `known` of request r
    if (row0 < total) {
      int lo = 0, hi = a.n - 1;  // the first request that ends behind the row
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (off[mid + 1] > row0) hi = mid;
        else lo = mid + 1;
      }
      r = lo;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t row = row0 + i;
      slot[i] = pos[i] = -1;
      if (row >= total) continue;
      while (off[r + 1] <= row) ++r, known = -1;
      if (first[r] < 0) continue;
      const int p = ctx[r] + (int)(row - off[r]), page = (uint32_t)p / (uint32_t)a.page, in = p - page * a.page;
      if (page != known) {
        const int held = pages_of(ctx[r], a.page);
        int *entry = a.tables + (int64_t)r * a.width + page;
        id = page < held ? *entry : a.stack[n_free - 1 - (first[r] + page - held)];
        if (page >= held && in == 0) *entry = id;  // a new page's first token is one of the new rows
        known = page;
      }
      const int64_t s = (int64_t)id * a.page + in;
      slot[i] = id >= 0 && s <= INT_MAX ? (int)s : -1;
      pos[i] = p;
    }
    if (a.vec && row0 + 4 <= a.rows) {
      *reinterpret_cast<int4 *>(a.slots + row0) = make_int4(slot[0], slot[1], slot[2], slot[3]);
      *reinterpret_cast<int4 *>(a.positions + row0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (row0 + i < a.rows) a.slots[row0 + i] = slot[i], a.positions[row0 + i] = pos[i];
    }
  }
}

// Returns the pages of `requests` to the stack, in the order given (a request
// named twice counts once), and sets their lengths to 0. One CTA; each thread
// compares its request with those before it in the chunk of 1024. 1 of 8
// requests 3.3 us, 16 of 1000 4.4 us, all of 1000 (64 pages each) 91 us.
__global__ void __launch_bounds__(kPagesThreads)
    pages_release_kernel(const int *requests, int n, int n_seqs, int page, int *lens, const int *tables, int width,
                         int *stack, int capacity, int *n_free) {
  __shared__ int64_t warp_sums[kPagesThreads / 32];
  __shared__ int s_first[kPagesThreads + 1], s_req[kPagesThreads];
  int64_t top = min(max(*n_free, 0), capacity);
  __syncthreads();
  for (int i0 = 0; i0 < n; i0 += blockDim.x) {
    const int i = i0 + threadIdx.x;
    int r = i < n ? requests[i] : -1;
    if (r < 0 || r >= n_seqs) r = -1;
    s_req[threadIdx.x] = r;
    __syncthreads();
    for (int j = 0; j < (int)threadIdx.x && r >= 0; ++j)
      if (s_req[j] == r) r = -1;  // of earlier chunks' requests the lengths are 0 already
    const int64_t len = r >= 0 ? min((int64_t)max(lens[r], 0), (int64_t)width * page) : 0;
    const int pages = (int)((len + page - 1) / page);
    int64_t sum;
    const int64_t upto = block_scan(pages, warp_sums, sum);
    s_first[threadIdx.x + 1] = (int)min(upto, (int64_t)INT_MAX);
    s_req[threadIdx.x] = r;
    if (threadIdx.x == 0) s_first[0] = 0;
    __syncthreads();
    const int64_t fit = min(sum, (int64_t)capacity - top);  // a full stack keeps its size: lengths were not the tables'
    for (int64_t p = threadIdx.x; p < fit; p += blockDim.x) {
      int lo = 0, hi = (int)blockDim.x - 1;
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (s_first[mid + 1] > p) hi = mid;
        else lo = mid + 1;
      }
      stack[top + p] = tables[(int64_t)s_req[lo] * width + (p - s_first[lo])];
    }
    if (r >= 0) lens[r] = 0;
    top += fit;
    __syncthreads();
  }
  if (threadIdx.x == 0) *n_free = (int)top;
}

}  // namespace mq
