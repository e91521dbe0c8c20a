// C-ABI entry points of the paged 4-bit key/value cache and of the block
// tables that address it (declared in include/mq_b200.h).
//
// No call here allocates or synchronises except creation and destruction of a
// cache: all of them may be captured in a CUDA graph, and what a call needs
// beside its arguments is the caller's workspace, so graphs share nothing.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdlib>
#include <new>

#include "mq_kv4.cuh"
#include "mq_kv4_attn.cuh"
#include "mq_kv4_prefill.cuh"
#include "mq_pages.cuh"
#include "mq_tcdec_api.h"

using namespace mq;

namespace {

// Switches the calling thread to `device` for the scope and restores it.
struct OnDevice {
  int prev = -1;
  cudaError_t err = cudaSuccess;
  explicit OnDevice(int device) {
    err = cudaGetDevice(&prev);
    if (err == cudaSuccess && prev != device) err = cudaSetDevice(device);
    else if (err == cudaSuccess) prev = -1;
  }
  ~OnDevice() {
    if (prev >= 0) cudaSetDevice(prev);
  }
};

// An error that is reported is not left behind for the calls that look for their own with cudaGetLastError.
int report(cudaError_t e, const char *what) {
  cudaGetLastError();
  return cuda_fail(e, what);
}

int check_device(int device) {
  int count = 0;
  const cudaError_t e = cudaGetDeviceCount(&count);
  if (e != cudaSuccess) return report(e, "cudaGetDeviceCount");
  if (device < 0 || device >= count) return fail(MQ_ERR_INVALID, "CUDA device id %d out of range", device);
  if (!gemm_supported(device)) return fail(MQ_ERR_UNSUPPORTED, "the kernels need an sm_100 device (device %d)", device);
  return MQ_OK;
}

bool valid_page(int page) { return page >= kKv4Unit && page <= 1024 && page % kKv4Unit == 0; }

// Rows [rows][heads][hd] of floats, heads of one row not overlapping.
int check_rows(const char *what, const float *p, int64_t ld, int64_t hs, int heads, int hd) {
  if (!p) return fail(MQ_ERR_INVALID, "null %s pointer", what);
  if (reinterpret_cast<uintptr_t>(p) % sizeof(float)) return fail(MQ_ERR_INVALID, "%s is not aligned to a float", what);
  if (ld < 0 || hs < 0 || (heads > 1 && hs < hd))
    return fail(MQ_ERR_INVALID, "%s strides (%lld, %lld) do not hold heads of %d", what, (long long)ld, (long long)hs,
                hd);
  return MQ_OK;
}

// Whether heads of hd elements at i * ld + h * hs (hs >= hd) share memory.
bool heads_overlap(int rows, int64_t ld, int heads, int64_t hs, int hd) {
  using wide = __int128;
  if (rows < 2) return false;
  if (ld < hd) return true;
  if (heads < 2 || ld >= (wide)(heads - 1) * hs + hd || hs >= (wide)(rows - 1) * ld + hd) return false;
  for (int h = 1; h < heads; ++h) {  // rows between heads: the two rows on either side of each head's distance
    const wide at = (wide)h * hs, i = at / ld;
    if ((i < rows && at - i * ld < hd) || (i + 1 < rows && (i + 1) * ld - at < hd)) return true;
  }
  return false;
}

bool vector16(const void *p, int64_t ld, int64_t hs) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 4 == 0 && hs % 4 == 0;
}

// CTAs of a store or load: one for the rows that it holds at a time, or as many as the device takes at once.
dim3 row_grid(const mq_kv4 *c, int rows) {
  const int per_row = 2 * c->v.kv * c->v.nb, parts = (per_row + kKv4Quads - 1) / kKv4Quads;
  const int64_t want = ((int64_t)rows + kv4_whole(per_row) - 1) / kv4_whole(per_row);
  return dim3((unsigned)std::min<int64_t>(want, std::max(1, 8 * c->sms / std::min(parts, 8))), (unsigned)parts);
}

int check_cache(const mq_kv4 *c, int layer) {
  if (!c) return fail(MQ_ERR_INVALID, "null cache handle");
  if (layer < 0 || layer >= c->v.layers) return fail(MQ_ERR_INVALID, "layer %d of %d", layer, c->v.layers);
  return MQ_OK;
}

int cache_shape(int layers, int pages, int page_size, int kv_heads, int head_dim, Kv4View &v, size_t &bytes) {
  if (layers < 1 || pages < 1 || kv_heads < 1 || kv_heads > 65536)
    return fail(MQ_ERR_INVALID, "invalid cache shape: %d layers, %d pages, %d heads", layers, pages, kv_heads);
  if (!valid_page(page_size))
    return fail(MQ_ERR_INVALID, "page size %d: a multiple of %d up to 1024 is needed", page_size, kKv4Unit);
  if (head_dim < 32 || head_dim > 128 || head_dim % 32)
    return fail(MQ_ERR_INVALID, "head size %d: 32, 64, 96 or 128 is needed", head_dim);
  if ((int64_t)pages * page_size > INT_MAX)
    return fail(MQ_ERR_INVALID, "%d pages of %d tokens: slots must stay below 2^31", pages, page_size);
  const int nb = head_dim / 32;
  const int64_t page_head = (int64_t)(page_size / kKv4Unit) * kv4_unit_bytes(nb);
  const int64_t slices = (int64_t)layers * pages;  // both below 2^31
  if (slices > INT64_MAX / page_head / kv_heads) return fail(MQ_ERR_INVALID, "cache size overflow");
  v = Kv4View{nullptr, layers, pages, page_size, kv_heads, head_dim, nb, page_head};
  bytes = (size_t)(slices * kv_heads * page_head);
  return MQ_OK;
}

bool env_set(const char *name) {
  const char *e = std::getenv(name);
  return e && *e && std::atoi(e) != 0;
}

uint64_t wait_limit() {
  const char *e = std::getenv("MQ_KV4_WAIT_NS");
  const unsigned long long ns = e ? std::strtoull(e, nullptr, 10) : 0;
  return ns ? std::min<uint64_t>(ns, 10 * kKv4WaitNs) : kKv4WaitNs;  // (never without a bound)
}

// The launch's own status decides: an error that an earlier call of the thread left behind is none of this one's.
template <typename... KArgs, typename... Args>
int launch(const char *what, cudaLaunchAttribute attr, void (*kernel)(KArgs...), dim3 grid, int threads, size_t smem,
           cudaStream_t s, const Args &...args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
  if (e != cudaSuccess) return report(e, what);
  count_launch();
  return MQ_OK;
}

// Launched behind the previous kernel of the stream with programmatic
// serialization, where that is allowed: it may start early and waits where it
// depends on that one.
cudaLaunchAttribute early(bool allowed) {
  cudaLaunchAttribute a = {};
  a.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  a.val.programmaticStreamSerializationAllowed = allowed;
  return a;
}

// MQ_PDL=0 launches normally, as for the linears.
template <typename... KArgs, typename... Args>
int launch_after(const char *what, void (*kernel)(KArgs...), const Args &...args) {
  static const bool on = [] {
    const char *e = std::getenv("MQ_PDL");
    return !e || !*e || std::atoi(e) != 0;
  }();
  return launch(what, early(on), kernel, args...);
}

// A kernel's workspace: its CTAs' notes on unfinished items, then the parts.
size_t parts_bytes(int ctas, int row_tile, int hd) {
  return (size_t)ctas * 2 * (sizeof(int4) + sizeof(float) * kv4_part_floats(row_tile, hd));
}
int dec_ctas(int sms) { return 3 * sms; }

// Flat rows (rows of a request times the query heads of a KV head) up to which
// the few-row kernel takes a request: it runs 8 of them at a time, and its time
// grows with every 8. 16 requests of 4000 tokens, 8 KV heads of 128: 91 us
// against the many-row kernel's 96 at 24 rows, 114 against 97 at 28.
constexpr int kFewRows = 24;
// Requests that cannot be longer are not cut, which spares the joining kernel.
// One request (8, 64) of 256 tokens: 8.7 us (9.9, 18.6) whole, 9.5 (11.2, 20.4)
// cut; of 512 tokens: 12.0 (14.1, 28.0) whole, 9.2 (11.7, 27.2) cut.
constexpr int kShortTokens = 256;
bool many_rows(int group, int max_new) { return (int64_t)group * max_new > kFewRows; }

void use_workspace(Kv4AttnArgs &a, uint8_t *ws, int ctas) {
  a.meta = reinterpret_cast<int4 *>(ws);
  a.parts = reinterpret_cast<float *>(ws + (size_t)ctas * 2 * sizeof(int4));
}

// Lets `kernel` use `bytes` of shared memory on `device`; once per device.
template <typename Kernel>
int allow_smem(Kernel kernel, int bytes, int device, std::atomic<uint64_t> &ready) {
  const uint64_t bit = 1ull << (device & 63);
  if (device < 64 && (ready.load(std::memory_order_relaxed) & bit)) return MQ_OK;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return report(e, "cudaFuncSetAttribute");
  if (device < 64) ready.fetch_or(bit, std::memory_order_relaxed);
  return MQ_OK;
}

template <int NB>
int run_attention(Kv4AttnArgs a, const mq_kv4 *c, uint8_t *ws, bool many, cudaStream_t s) {
  static std::atomic<uint64_t> dec_ready{0}, pre_ready{0};
  if (int rc = allow_smem(kv4_decode_kernel<NB>, DecSmem<NB>::kBytes, c->device, dec_ready)) return rc;
  Kv4Join j{};
  j.ctas[0] = dec_ctas(c->sms);
  use_workspace(a, ws, j.ctas[0]);
  a.min_rows = 1, a.max_rows = many ? kFewRows : INT_MAX;
  a.cut = many || (int64_t)a.width * a.c.page > kShortTokens;
  j.meta[0] = a.meta, j.parts[0] = a.parts;
  if (int rc = launch_after("cache attention", kv4_decode_kernel<NB>, dim3(j.ctas[0]), kDecWarps * 32,
                            DecSmem<NB>::kBytes, s, a))
    return rc;
  if (many) {
    if (int rc = allow_smem(kv4_prefill_kernel<NB>, PreSmem<NB>::kAlloc, c->device, pre_ready)) return rc;
    j.ctas[1] = c->sms;
    use_workspace(a, ws + parts_bytes(j.ctas[0], kDecRowTile, a.c.hd), j.ctas[1]);
    a.min_rows = kFewRows + 1, a.max_rows = INT_MAX;
    j.meta[1] = a.meta, j.parts[1] = a.parts;
    if (int rc = launch_after("cache attention", kv4_prefill_kernel<NB>, dim3(j.ctas[1]), kPreThreads,
                              PreSmem<NB>::kAlloc, s, a))
      return rc;
  }
  if (!a.cut) return MQ_OK;
  return launch_after("join attention parts", kv4_join_kernel<NB>,
                      dim3(j.ctas[0] + j.ctas[1] * (kPreRows / kJoinMany)), kJoinRows * 8 * NB * kJoinSlices, 0, s, a, j);
}

}  // namespace

extern "C" {

size_t mq_kv4_bytes(int layers, int pages, int page_size, int kv_heads, int head_dim) {
  Kv4View v;
  size_t bytes = 0;
  last_error().clear();
  return cache_shape(layers, pages, page_size, kv_heads, head_dim, v, bytes) == MQ_OK ? bytes : 0;
}

int mq_kv4_create(int device, int layers, int pages, int page_size, int kv_heads, int head_dim, void *memory,
                  size_t memory_bytes, void *stream, mq_kv4 **out) {
  last_error().clear();
  if (!out) return fail(MQ_ERR_INVALID, "null output handle");
  *out = nullptr;
  Kv4View v;
  size_t bytes = 0;
  if (int rc = cache_shape(layers, pages, page_size, kv_heads, head_dim, v, bytes)) return rc;
  if (memory && memory_bytes < bytes)
    return fail(MQ_ERR_SIZE, "cache memory: %zu bytes, %zu are needed", memory_bytes, bytes);
  if (reinterpret_cast<uintptr_t>(memory) % 16) return fail(MQ_ERR_INVALID, "cache memory is not aligned to 16 bytes");
  if (int rc = check_device(device)) return rc;
  OnDevice g(device);
  if (g.err != cudaSuccess) return report(g.err, "cudaSetDevice");
  auto *c = new (std::nothrow) mq_kv4;
  if (!c) return fail(MQ_ERR_INVALID, "out of host memory");
  // (The flag is allocated with the device's first handle, which may be made while a stream is captured.)
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  cudaThreadExchangeStreamCaptureMode(&mode);
  const int rc = device_err_flag(device, &c->err_dev, &c->err_host);
  cudaThreadExchangeStreamCaptureMode(&mode);
  if (rc) {
    cudaGetLastError();
    delete c;
    return rc;
  }
  c->wait_ns = wait_limit();
  c->lost = env_set("MQ_KV4_LOSE_COPIES") ? 16 : 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaSuccess;
  void *base = memory;
  if (!base) e = cudaMalloc(&base, bytes);
  if (e != cudaSuccess) {
    delete c;
    return report(e, "cudaMalloc cache");
  }
  e = cudaMemsetAsync(base, 0, bytes, s);
  if (e == cudaSuccess && !memory) e = cudaStreamSynchronize(s);
  if (e != cudaSuccess) {
    if (!memory) cudaFree(base);
    delete c;
    return report(e, "clear cache");
  }
  v.base = static_cast<uint8_t *>(base);
  c->device = device;
  c->v = v;
  c->bytes = bytes;
  c->owned = memory ? nullptr : base;
  cudaDeviceGetAttribute(&c->sms, cudaDevAttrMultiProcessorCount, device);
  *out = c;
  return MQ_OK;
}

void mq_kv4_destroy(mq_kv4 *c) {
  if (!c) return;
  if (c->owned) {
    OnDevice g(c->device);
    cudaFree(c->owned);
  }
  delete c;
}

int mq_kv4_info(const mq_kv4 *c, int *device, int *layers, int *pages, int *page_size, int *kv_heads, int *head_dim,
                size_t *device_bytes) {
  last_error().clear();
  if (!c) return fail(MQ_ERR_INVALID, "null cache handle");
  if (device) *device = c->device;
  if (layers) *layers = c->v.layers;
  if (pages) *pages = c->v.pages;
  if (page_size) *page_size = c->v.page;
  if (kv_heads) *kv_heads = c->v.kv;
  if (head_dim) *head_dim = c->v.hd;
  if (device_bytes) *device_bytes = c->bytes;
  return MQ_OK;
}

int mq_kv4_store(const mq_kv4 *c, int layer, const float *k, int64_t ld_k, int64_t hs_k, const float *v, int64_t ld_v,
                 int64_t hs_v, const int *slots, int rows, void *stream) {
  last_error().clear();
  if (int rc = check_cache(c, layer)) return rc;
  if (rows < 0) return fail(MQ_ERR_INVALID, "negative row count %d", rows);
  if (rows == 0) return MQ_OK;
  if (int rc = check_rows("key", k, ld_k, hs_k, c->v.kv, c->v.hd)) return rc;
  if (int rc = check_rows("value", v, ld_v, hs_v, c->v.kv, c->v.hd)) return rc;
  if (!slots) return fail(MQ_ERR_INVALID, "null slot map");
  OnDevice g(c->device);
  if (g.err != cudaSuccess) return report(g.err, "cudaSetDevice");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const Kv4Rows kr{k, ld_k, hs_k}, vr{v, ld_v, hs_v};
  auto *kernel = vector16(k, ld_k, hs_k) && vector16(v, ld_v, hs_v) ? kv4_store_kernel<true> : kv4_store_kernel<false>;
  return launch("cache store", early(false), kernel, row_grid(c, rows), kKv4Threads, 0, s, c->v, layer, kr, vr, slots,
                rows);
}

int mq_kv4_load(const mq_kv4 *c, int layer, const int *slots, int rows, float *k, float *v, void *stream) {
  last_error().clear();
  if (int rc = check_cache(c, layer)) return rc;
  if (rows < 0) return fail(MQ_ERR_INVALID, "negative row count %d", rows);
  if (rows == 0) return MQ_OK;
  const int64_t ld = (int64_t)c->v.kv * c->v.hd;
  if (int rc = check_rows("key", k, ld, c->v.hd, c->v.kv, c->v.hd)) return rc;
  if (int rc = check_rows("value", v, ld, c->v.hd, c->v.kv, c->v.hd)) return rc;
  if (!slots) return fail(MQ_ERR_INVALID, "null slot map");
  OnDevice g(c->device);
  if (g.err != cudaSuccess) return report(g.err, "cudaSetDevice");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  auto *kernel = vector16(k, 0, 0) && vector16(v, 0, 0) ? kv4_load_kernel<true> : kv4_load_kernel<false>;
  return launch("cache load", early(false), kernel, row_grid(c, rows), kKv4Threads, 0, s, c->v, layer, slots, rows, k,
                v);
}

size_t mq_kv4_attention_workspace(const mq_kv4 *c, int heads, int max_new) {
  if (!c || heads < 1) return 0;
  size_t n = parts_bytes(dec_ctas(c->sms), kDecRowTile, c->v.hd);
  if (many_rows(heads / c->v.kv, max_new)) n += parts_bytes(c->sms, kPreRows, c->v.hd);
  return n;
}

int mq_kv4_attention(const mq_kv4 *c, int layer, const float *q, int64_t ld_q, int64_t hs_q, int rows, int heads,
                     const int *offsets, const int *seq_lens, const int *block_tables, int n_seqs, int max_pages,
                     int max_new, float scale, float *out, int64_t ld_out, int64_t hs_out, void *workspace,
                     size_t workspace_bytes, void *stream) {
  last_error().clear();
  if (int rc = check_cache(c, layer)) return rc;
  if (rows < 0 || n_seqs < 0) return fail(MQ_ERR_INVALID, "negative count: %d rows, %d requests", rows, n_seqs);
  if (heads < 1 || heads % c->v.kv)
    return fail(MQ_ERR_INVALID, "%d query heads do not share %d key/value heads evenly", heads, c->v.kv);
  if ((int64_t)rows * heads > INT_MAX) return fail(MQ_ERR_INVALID, "%d rows of %d heads are too many", rows, heads);
  if ((int64_t)max_pages * c->v.page > INT_MAX - 4096)
    return fail(MQ_ERR_INVALID, "%d pages a request: tokens must stay below 2^31 - 4096", max_pages);
  if (max_pages < 1 || max_new < 0) return fail(MQ_ERR_INVALID, "%d pages a request, %d new rows", max_pages, max_new);
  if (!std::isfinite(scale)) return fail(MQ_ERR_INVALID, "the score scale is not finite");
  if (rows == 0 || n_seqs == 0) return MQ_OK;
  if (int rc = check_rows("query", q, ld_q, hs_q, heads, c->v.hd)) return rc;
  if (int rc = check_rows("output", out, ld_out, hs_out, heads, c->v.hd)) return rc;
  if (heads_overlap(rows, ld_out, heads, hs_out, c->v.hd))
    return fail(MQ_ERR_INVALID, "heads of the output overlap (strides %lld, %lld)", (long long)ld_out,
                (long long)hs_out);
  if (!offsets || !seq_lens || !block_tables) return fail(MQ_ERR_INVALID, "null offsets, lengths or block tables");
  const size_t need = mq_kv4_attention_workspace(c, heads, max_new);
  if (!workspace || workspace_bytes < need)
    return fail(MQ_ERR_SIZE, "attention workspace: %zu bytes, %zu are needed", workspace ? workspace_bytes : 0, need);
  if (reinterpret_cast<uintptr_t>(workspace) % 16)
    return fail(MQ_ERR_INVALID, "the attention workspace is not aligned to 16 bytes");
  if (*(volatile int *)c->err_host) {
    *(volatile int *)c->err_host = 0;
    return fail(MQ_ERR_TIMEOUT, "an earlier tensor-core launch on device %d ran out of a bounded wait", c->device);
  }
  OnDevice g(c->device);
  if (g.err != cudaSuccess) return report(g.err, "cudaSetDevice");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  Kv4AttnArgs a{};
  a.c = c->v;
  a.layer = layer;
  a.q = q, a.ld_q = ld_q, a.hs_q = hs_q;
  a.out = out, a.ld_o = ld_out, a.hs_o = hs_out;
  a.offsets = offsets, a.lens = seq_lens, a.tables = block_tables;
  a.n = n_seqs, a.width = max_pages, a.rows = rows, a.group = heads / c->v.kv;
  a.scale = scale * 1.44269504088896341f;
  a.vec_q = vector16(q, ld_q, hs_q);
  a.vec_o = vector16(out, ld_out, hs_out);
  a.err = c->err_dev, a.wait_ns = c->wait_ns, a.lost = c->lost;
  uint8_t *ws = static_cast<uint8_t *>(workspace);
  const bool many = many_rows(a.group, max_new);
  switch (c->v.nb) {
  case 1: return run_attention<1>(a, c, ws, many, s);
  case 2: return run_attention<2>(a, c, ws, many, s);
  case 3: return run_attention<3>(a, c, ws, many, s);
  default: return run_attention<4>(a, c, ws, many, s);
  }
}

int mq_pages_plan(int device, const int *ctx_lens, const int *new_lens, int n_seqs, int page_size, int *block_tables,
                  int max_pages, const int *free_pages, int n_pages, const int *n_free, int rows, int *offsets,
                  int *seq_lens, int *slots, int *positions, int *n_free_out, int *refused, void *stream) {
  last_error().clear();
  if (n_seqs < 0 || n_seqs > kPagesMaxSeqs)
    return fail(MQ_ERR_INVALID, "%d requests: at most %d are planned in one call", n_seqs, kPagesMaxSeqs);
  if (rows < 0) return fail(MQ_ERR_INVALID, "negative row count %d", rows);
  if (!valid_page(page_size))
    return fail(MQ_ERR_INVALID, "page size %d: a multiple of %d up to 1024 is needed", page_size, kKv4Unit);
  if (max_pages < 1 || n_pages < 0 || (int64_t)max_pages * page_size > INT_MAX)
    return fail(MQ_ERR_INVALID, "%d pages a request, %d free pages", max_pages, n_pages);
  if ((n_seqs && (!ctx_lens || !new_lens || !block_tables || !seq_lens)) || (rows && (!slots || !positions)) ||
      (n_pages && !free_pages) || !n_free || !offsets || !n_free_out || !refused)
    return fail(MQ_ERR_INVALID, "null pointer");
  if (seq_lens == new_lens && n_seqs) return fail(MQ_ERR_INVALID, "the lengths may not replace the new row counts");
  if (int rc = check_device(device)) return rc;
  OnDevice g(device);
  if (g.err != cudaSuccess) return report(g.err, "cudaSetDevice");
  const PagesArgs a{ctx_lens, new_lens, n_seqs, page_size, block_tables, max_pages, free_pages, n_pages,
                    n_free, rows, offsets, seq_lens, slots, positions, n_free_out, refused,
                    vector16(slots, 0, 0) && vector16(positions, 0, 0), seq_lens == ctx_lens || n_free_out == n_free};
  // (The 48 KB that need no permission count the kernel's static part too.)
  static std::atomic<uint64_t> ready{0};
  if (int rc = allow_smem(pages_plan_kernel, (int)pages_smem(kPagesMaxSeqs), device, ready)) return rc;
  // A thread for each request and for every four rows, in one CTA while that is enough: a decode step of 8
  // requests took 7.7 us with 1024 threads.
  const int want = std::max(n_seqs, rows / 4);
  const int ctas = (int)std::min<int64_t>(kPagesCtas, ((int64_t)rows + 4 * kPagesThreads - 1) / (4 * kPagesThreads));
  const dim3 grid(ctas <= 1 ? 1 : a.in_place ? kPagesCluster : ctas);
  cudaLaunchAttribute cluster = {};
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim.x = a.in_place ? grid.x : 1;
  cluster.val.clusterDim.y = 1;
  cluster.val.clusterDim.z = 1;
  return launch("plan pages", cluster, pages_plan_kernel, grid,
                std::min(kPagesThreads, std::max(64, (want + 31) / 32 * 32)), pages_smem(n_seqs),
                static_cast<cudaStream_t>(stream), a);
}

int mq_pages_release(int device, const int *requests, int n, int n_seqs, int page_size, int *seq_lens,
                     const int *block_tables, int max_pages, int *free_pages, int n_pages, int *n_free, void *stream) {
  last_error().clear();
  if (n < 0 || n_seqs < 0) return fail(MQ_ERR_INVALID, "negative count: %d of %d requests", n, n_seqs);
  if (!valid_page(page_size))
    return fail(MQ_ERR_INVALID, "page size %d: a multiple of %d up to 1024 is needed", page_size, kKv4Unit);
  if (max_pages < 1 || n_pages < 0 || (int64_t)max_pages * page_size > INT_MAX)
    return fail(MQ_ERR_INVALID, "%d pages a request, %d free pages", max_pages, n_pages);
  if (n == 0 || n_seqs == 0) return MQ_OK;
  if (!requests || !seq_lens || !block_tables || (n_pages && !free_pages) || !n_free)
    return fail(MQ_ERR_INVALID, "null pointer");
  if (int rc = check_device(device)) return rc;
  OnDevice g(device);
  if (g.err != cudaSuccess) return report(g.err, "cudaSetDevice");
  return launch("release pages", early(false), pages_release_kernel, dim3(1), kPagesThreads, 0,
                static_cast<cudaStream_t>(stream), requests, n, n_seqs, page_size, seq_lens, block_tables, max_pages,
                free_pages, n_pages, n_free);
}

}  // extern "C"
