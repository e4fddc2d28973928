// serving.cu — the C ABI of the drafted-decoding operators: the quantised
// key/value cache, the shared-prefix attention and the verification of drafts.
#include <algorithm>
#include <climits>
#include <string>

#include "../../include/needle_b200_debug.h"
#include "failure.h"
#include "serving.h"

using namespace nbk;
using nbr::fail;
using nbr::guard;

struct nb_kv_cache {
  KvCacheDev dev;
  int device = 0;
  void* pool = nullptr;
};

namespace nbr {
namespace {

// Makes `device` current for a call and puts the caller's back.
struct OnDevice {
  int before = -1;
  explicit OnDevice(int device) {
    int now = -1;
    NB_CUDA(cudaGetDevice(&now));
    if (now != device) {
      NB_CUDA(cudaSetDevice(device));
      before = now;
    }
  }
  ~OnDevice() {
    if (before >= 0) cudaSetDevice(before);
  }
};

int device_or_current(int32_t device) {
  int count = 0;
  if (cudaGetDeviceCount(&count) != cudaSuccess || count == 0) {
    cudaGetLastError();
    fail(NB_ERR_NO_DEVICE, "no CUDA device");
  }
  if (device >= count || device < -1) fail(NB_ERR_ARGUMENT, "no CUDA device " + std::to_string(device));
  int d = device;
  if (d < 0) NB_CUDA(cudaGetDevice(&d));
  return d;
}

KvBatchDev batch_of(const nb_kv_batch& b) {
  if (b.sequences > (1u << 24) || b.rows > (1u << 26) || b.max_rows > (1u << 26) || b.max_length > (1u << 30))
    fail(NB_ERR_ARGUMENT, "a batch holds at most 2^24 sequences, 2^26 rows and 2^30 positions of a sequence");
  if (b.sequences && (!b.row_start || !b.lengths)) fail(NB_ERR_ARGUMENT, "row_start and lengths are needed");
  if (b.sequences && b.max_length && (!b.pages || b.page_stride == 0)) fail(NB_ERR_ARGUMENT, "a batch with positions needs its pages");
  if (reinterpret_cast<uintptr_t>(b.row_start) % 4 || reinterpret_cast<uintptr_t>(b.lengths) % 4 || reinterpret_cast<uintptr_t>(b.pages) % 4)
    fail(NB_ERR_ARGUMENT, "row_start, lengths and pages must be 4-byte aligned");
  KvBatchDev d;
  d.sequences = (int)b.sequences;
  d.rows = (int)b.rows;
  // more rows than the batch has are no sequence's; the attention's tiles of a
  // sequence, rows x query heads of a kv head, then stay within 32 bits
  d.max_rows = (int)std::min(b.max_rows, b.rows);
  d.max_length = (int)b.max_length;
  d.page_stride = b.page_stride;
  d.row_start = b.row_start;
  d.lengths = b.lengths;
  d.pages = b.pages;
  return d;
}

RowsDev rows_of(const nb_rows& r, const char* name, const nb_kv_batch& b, uint32_t heads, uint32_t dim, bool output) {
  if (r.dtype < NB_F32 || r.dtype > NB_BF16) fail(NB_ERR_ARGUMENT, std::string(name) + ": unknown dtype " + std::to_string(r.dtype));
  if (b.sequences && b.rows && !r.data) fail(NB_ERR_ARGUMENT, std::string(name) + " is needed");
  if (reinterpret_cast<uintptr_t>(r.data) % (r.dtype == NB_F32 ? 4 : 2)) fail(NB_ERR_ARGUMENT, std::string(name) + " is not aligned to its type");
  if (r.row_stride < 0 || r.head_stride < 0 || r.row_stride > (1ll << 40) || r.head_stride > (1ll << 40))
    fail(NB_ERR_ARGUMENT, std::string(name) + ": strides must lie in [0, 2^40]");
  if (output) {
    // rows within heads or heads within rows, neither reaching into the next
    const int64_t rows = b.rows, hs = r.head_stride, rs = r.row_stride, d = dim, n = heads;
    const bool heads_inside = (n == 1 || hs >= d) && (rows <= 1 || rs >= (n - 1) * hs + d);
    const bool rows_inside = (rows <= 1 || rs >= d) && (n == 1 || hs >= (rows - 1) * rs + d);
    if (!heads_inside && !rows_inside) fail(NB_ERR_ARGUMENT, std::string(name) + ": rows or heads of an output overlap");
  }
  RowsDev d;
  d.data = r.data;
  d.dtype = r.dtype;
  d.row_stride = r.row_stride;
  d.head_stride = r.head_stride;
  return d;
}

void attend_sizes(const nb_kv_cache& c, const KvBatchDev& b, uint32_t prefix_length, uint32_t heads) {
  if (heads == 0 || heads % c.dev.kv_heads || heads / c.dev.kv_heads > (uint32_t)KV_MAX_GROUP)
    fail(NB_ERR_ARGUMENT, "heads must be a multiple of the cache's kv_heads, at most 64 for each");
  if (prefix_length > (1u << 30)) fail(NB_ERR_ARGUMENT, "prefix_length is above 2^30");
  const uint64_t group = heads / c.dev.kv_heads;
  if ((uint64_t)b.rows * heads > (1ull << 30) || (uint64_t)b.sequences * (((uint64_t)b.max_rows * group + 15) / 16) > (uint64_t)INT_MAX)
    fail(NB_ERR_ARGUMENT, "too many rows for one call");
}

}  // namespace
}  // namespace nbr

using namespace nbr;

extern "C" {

nb_status nb_kv_cache_create(int32_t device, int32_t format, uint32_t kv_heads, uint32_t head_dim, uint32_t pages, nb_kv_cache** out) {
  if (!out) return NB_ERR_ARGUMENT;
  *out = nullptr;
  return guard([&] {
    if (format != NB_KV_INT8 && format != NB_KV_E4M3) fail(NB_ERR_ARGUMENT, "unknown cache format " + std::to_string(format));
    if (head_dim != 64 && head_dim != 128) fail(NB_ERR_ARGUMENT, "head_dim must be 64 or 128");
    if (kv_heads == 0 || kv_heads > 256) fail(NB_ERR_ARGUMENT, "kv_heads must lie in [1, 256]");
    if (pages == 0) fail(NB_ERR_ARGUMENT, "a cache has at least one page");
    const int d = device_or_current(device);
    OnDevice on(d);
    const size_t blocks = (size_t)pages * kv_heads, codes = blocks * KV_PAGE * head_dim, scales = blocks * KV_PAGE * sizeof(float);
    auto* c = new nb_kv_cache;
    c->device = d;
    cudaError_t e = cudaMalloc(&c->pool, 2 * codes + 2 * scales + 256);
    if (e != cudaSuccess) {
      cudaGetLastError();
      delete c;
      fail(NB_ERR_CUDA, std::string("cudaMalloc of the page pool: ") + cudaGetErrorString(e));
    }
    auto* p = static_cast<uint8_t*>(c->pool);
    c->dev.k = p;
    c->dev.v = p + codes;
    c->dev.ks = reinterpret_cast<float*>(p + 2 * codes);
    c->dev.vs = reinterpret_cast<float*>(p + 2 * codes + scales);
    c->dev.error = reinterpret_cast<uint32_t*>(p + 2 * codes + 2 * scales);
    c->dev.kv_heads = (int)kv_heads;
    c->dev.dim = (int)head_dim;
    c->dev.pages = pages;
    c->dev.e4m3 = format == NB_KV_E4M3;
    e = kv_pool_clear(c->dev, cudaStreamPerThread);
    if (e == cudaSuccess) e = cudaStreamSynchronize(cudaStreamPerThread);
    if (e != cudaSuccess) {
      cudaFree(c->pool);
      delete c;
      fail(NB_ERR_CUDA, std::string("clearing the page pool: ") + cudaGetErrorString(e));
    }
    *out = c;
  });
}

void nb_kv_cache_release(nb_kv_cache* cache) {
  if (!cache) return;
  guard([&] {
    OnDevice on(cache->device);
    cudaFree(cache->pool);  // waits for the device
  });
  delete cache;
}

nb_status nb_kv_cache_append(nb_kv_cache* cache, const nb_kv_batch* batch, const nb_rows* keys, const nb_rows* values, void* stream) {
  if (!cache || !batch || !keys || !values) return NB_ERR_ARGUMENT;
  return guard([&] {
    const KvBatchDev b = batch_of(*batch);
    const RowsDev k = rows_of(*keys, "keys", *batch, cache->dev.kv_heads, cache->dev.dim, false);
    const RowsDev v = rows_of(*values, "values", *batch, cache->dev.kv_heads, cache->dev.dim, false);
    if (k.dtype != v.dtype) fail(NB_ERR_ARGUMENT, "keys and values must have one dtype");
    OnDevice on(cache->device);
    NB_CUDA(kv_append(cache->dev, b, k, v, static_cast<cudaStream_t>(stream)));
  });
}

nb_status nb_kv_cache_read(const nb_kv_cache* cache, const nb_kv_batch* batch, const nb_rows* keys, const nb_rows* values, void* stream) {
  if (!cache || !batch || !keys || !values) return NB_ERR_ARGUMENT;
  return guard([&] {
    const KvBatchDev b = batch_of(*batch);
    const RowsDev k = rows_of(*keys, "keys", *batch, cache->dev.kv_heads, cache->dev.dim, true);
    const RowsDev v = rows_of(*values, "values", *batch, cache->dev.kv_heads, cache->dev.dim, true);
    if (k.dtype != v.dtype) fail(NB_ERR_ARGUMENT, "keys and values must have one dtype");
    OnDevice on(cache->device);
    NB_CUDA(kv_read(cache->dev, b, k, v, static_cast<cudaStream_t>(stream)));
  });
}

nb_status nb_kv_cache_attend_workspace(const nb_kv_cache* cache, const nb_kv_batch* batch, uint32_t prefix_length, uint32_t heads,
                                       size_t* bytes) {
  if (!cache || !batch || !bytes) return NB_ERR_ARGUMENT;
  return guard([&] {
    const KvBatchDev b = batch_of(*batch);
    attend_sizes(*cache, b, prefix_length, heads);
    *bytes = kv_attend_workspace(cache->dev, b, (int)prefix_length, (int)heads);
  });
}

nb_status nb_kv_cache_attend(const nb_kv_cache* cache, const nb_kv_batch* batch, const uint32_t* prefix_pages, uint32_t prefix_length,
                             const nb_rows* query, const nb_rows* out, uint32_t heads, float scale, void* workspace,
                             size_t workspace_bytes, void* stream) {
  if (!cache || !batch || !query || !out) return NB_ERR_ARGUMENT;
  return guard([&] {
    const KvBatchDev b = batch_of(*batch);
    attend_sizes(*cache, b, prefix_length, heads);
    KvAttend a;
    a.query = rows_of(*query, "query", *batch, heads, cache->dev.dim, false);
    a.out = rows_of(*out, "out", *batch, heads, cache->dev.dim, true);
    if (a.query.dtype == DTYPE_F32 || a.query.dtype != a.out.dtype) fail(NB_ERR_ARGUMENT, "query and out must both be NB_F16 or both NB_BF16");
    if (prefix_length && !prefix_pages) fail(NB_ERR_ARGUMENT, "a prefix needs its pages");
    if (reinterpret_cast<uintptr_t>(prefix_pages) % 4) fail(NB_ERR_ARGUMENT, "prefix_pages must be 4-byte aligned");
    a.prefix_pages = prefix_pages;
    a.prefix = (int)prefix_length;
    a.heads = (int)heads;
    a.scale = scale;
    if (b.sequences && b.rows) {
      const size_t need = kv_attend_workspace(cache->dev, b, a.prefix, a.heads);
      if (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 16)
        fail(NB_ERR_ARGUMENT, "the workspace must be 16-byte aligned and hold " + std::to_string(need) + " bytes");
    }
    a.workspace = workspace;
    OnDevice on(cache->device);
    NB_CUDA(kv_attend(cache->dev, b, a, static_cast<cudaStream_t>(stream)));
  });
}

nb_status nb_kv_cache_check(nb_kv_cache* cache, void* stream) {
  if (!cache) return NB_ERR_ARGUMENT;
  return guard([&] {
    OnDevice on(cache->device);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    uint32_t error = 0;
    NB_CUDA(cudaMemcpyAsync(&error, cache->dev.error, sizeof error, cudaMemcpyDeviceToHost, st));
    NB_CUDA(cudaStreamSynchronize(st));
    if (!error) return;
    NB_CUDA(kv_clear_report(cache->dev, error, st));
    NB_CUDA(cudaStreamSynchronize(st));
    std::string message;
    auto say = [&](uint32_t bit, const char* what) {
      if (error & bit) message += (message.empty() ? "" : "; ") + std::string(what);
    };
    say(KV_WAIT_FAILED, "a bounded device wait of the shared-prefix attention gave up");
    say(KV_BAD_SEQUENCE, "a sequence's rows or length were outside the batch's bounds, it was left out");
    say(KV_BAD_PAGE, "a page number was outside the pool, its positions were masked or not written");
    fail(error & KV_WAIT_FAILED ? NB_ERR_TIMEOUT : NB_ERR_ARGUMENT, message);
  });
}

nb_status nb_debug_expire_attention(nb_kv_cache* cache, uint32_t on) {
  if (!cache) return NB_ERR_ARGUMENT;
  cache->dev.expire = on != 0;
  return NB_OK;
}

nb_status nb_verify_drafts(int32_t device, const nb_verify* a, void* stream) {
  if (!a) return NB_ERR_ARGUMENT;
  return guard([&] {
    if (a->dtype < NB_F32 || a->dtype > NB_BF16) fail(NB_ERR_ARGUMENT, "logits: unknown dtype " + std::to_string(a->dtype));
    if (a->vocab == 0 || a->vocab > (1u << 24)) fail(NB_ERR_ARGUMENT, "vocab must lie in [1, 2^24]");
    if (a->sequences > (1u << 20) || a->drafts > 1024) fail(NB_ERR_ARGUMENT, "at most 2^20 sequences and 1024 drafts of each");
    if (!(a->temperature >= 0.0f) || a->temperature > 1e30f) fail(NB_ERR_ARGUMENT, "temperature must lie in [0, 1e30]");
    if (a->temperature > 0.0f && a->temperature < 1e-30f) fail(NB_ERR_ARGUMENT, "a temperature above 0 must be at least 1e-30");
    if (a->row_stride < (int64_t)a->vocab || a->row_stride > (1ll << 40)) fail(NB_ERR_ARGUMENT, "row_stride must be at least vocab");
    if (a->sequences) {
      if (!a->logits || !a->tokens || !a->accepted) fail(NB_ERR_ARGUMENT, "logits, tokens and accepted are needed");
      if (a->drafts && !a->draft_tokens) fail(NB_ERR_ARGUMENT, "draft_tokens are needed");
      if (a->temperature > 0.0f && (!a->sample_uniforms || (a->drafts && !a->accept_uniforms)))
        fail(NB_ERR_ARGUMENT, "a temperature above 0 needs accept_uniforms and sample_uniforms");
    }
    const void* words[] = {a->draft_probabilities, a->draft_tokens, a->draft_counts, a->mask_bits, a->accept_uniforms, a->sample_uniforms, a->tokens,
                           a->accepted};
    for (const void* p : words)
      if (reinterpret_cast<uintptr_t>(p) % 4) fail(NB_ERR_ARGUMENT, "the arrays must be 4-byte aligned");
    if (reinterpret_cast<uintptr_t>(a->logits) % (a->dtype == NB_F32 ? 4 : 2)) fail(NB_ERR_ARGUMENT, "logits are not aligned to their type");
    VerifyDev v;
    v.sequences = (int)a->sequences;
    v.drafts = (int)a->drafts;
    v.vocab = (int)a->vocab;
    v.dtype = a->dtype;
    v.row_stride = a->row_stride;
    v.logits = a->logits;
    v.q = a->draft_probabilities;
    v.draft_tokens = a->draft_tokens;
    v.draft_counts = a->draft_counts;
    v.mask = a->mask_bits;
    v.accept = a->accept_uniforms;
    v.sample = a->sample_uniforms;
    v.temperature = a->temperature;
    v.tokens = a->tokens;
    v.accepted = a->accepted;
    OnDevice on(device_or_current(device));
    NB_CUDA(verify_drafts(v, static_cast<cudaStream_t>(stream)));
  });
}

}  // extern "C"
