// serving.h — parameters and launchers of the drafted-decoding operators
// (kv_cache.cu, kv_attend.cu, verify.cu); the C ABI over them is serving.cu.
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace nbk {

constexpr int KV_PAGE = 64;
constexpr float KV_SCALE_MIN = 0x1p-60f, KV_PEAK_MAX = 0x1p40f;
constexpr uint32_t KV_BAD_SEQUENCE = 1u, KV_BAD_PAGE = 2u, KV_WAIT_FAILED = 4u;
constexpr int KV_MAX_GROUP = 64;  // query heads of one kv head

enum Dtype { DTYPE_F32 = 0, DTYPE_F16 = 1, DTYPE_BF16 = 2 };

// The pool: codes [pages][kv_heads][64 · dim] and scales [pages][kv_heads][64]
// for keys and values. Within a page and head, the key code of position p and
// dimension d is byte key_byte(p, d) below, the value code byte value_byte(p,
// d): the orders in which a warp's lanes feed them to matrix instructions.
struct KvCacheDev {
  uint8_t *k = nullptr, *v = nullptr;
  float *ks = nullptr, *vs = nullptr;
  uint32_t* error = nullptr;
  int kv_heads = 0, dim = 0;
  uint32_t pages = 0;
  bool e4m3 = false;
  bool expire = false;  // a test's: a wait of the first block of every attention launch runs out
};

// Rows of 64 codes: eight lanes that read 16 bytes each of two neighbouring
// rows meet in no bank of shared memory.
__host__ __device__ constexpr int key_byte(int p, int d) { return (d / 64) * (KV_PAGE * 64) + p * 64 + d % 64; }

// 16 positions × 32 dimensions make a 512-byte block of 32 lanes × 16 bytes:
// lane 4·(d % 8) + (p % 16) / 4 holds four dimensions d % 32 / 8 of four
// neighbouring positions each.
__host__ __device__ constexpr int value_byte(int p, int d, int dim) {
  return (p / 16) * 16 * dim + (d / 32) * 512 + (d % 8) * 64 + (p % 16 / 4) * 16 + (d % 32 / 8) * 4 + p % 4;
}

struct KvBatchDev {
  int sequences = 0, rows = 0, max_rows = 0, max_length = 0;
  uint32_t page_stride = 0;
  const int32_t* row_start = nullptr;
  const int32_t* lengths = nullptr;
  const uint32_t* pages = nullptr;
};

struct RowsDev {
  void* data = nullptr;
  int dtype = DTYPE_F32;
  long long row_stride = 0, head_stride = 0;
};

cudaError_t kv_pool_clear(const KvCacheDev& c, cudaStream_t st);
cudaError_t kv_clear_report(const KvCacheDev& c, uint32_t reported, cudaStream_t st);
cudaError_t kv_check_spans(const KvCacheDev& c, const KvBatchDev& b, cudaStream_t st);  // for calls without rows
cudaError_t kv_append(const KvCacheDev& c, const KvBatchDev& b, const RowsDev& keys, const RowsDev& values, cudaStream_t st);
cudaError_t kv_read(const KvCacheDev& c, const KvBatchDev& b, const RowsDev& keys, const RowsDev& values, cudaStream_t st);

struct KvAttend {
  const uint32_t* prefix_pages = nullptr;
  int prefix = 0, heads = 0;
  float scale = 1.0f;
  RowsDev query, out;
  void* workspace = nullptr;
};
size_t kv_attend_workspace(const KvCacheDev& c, const KvBatchDev& b, int prefix, int heads);
cudaError_t kv_attend(const KvCacheDev& c, const KvBatchDev& b, const KvAttend& a, cudaStream_t st);

struct VerifyDev {
  int sequences = 0, drafts = 0, vocab = 0, dtype = DTYPE_F32;
  long long row_stride = 0;
  const void* logits = nullptr;
  const float* q = nullptr;
  const uint32_t* draft_tokens = nullptr;
  const int32_t* draft_counts = nullptr;
  const uint32_t* mask = nullptr;
  const float* accept = nullptr;
  const float* sample = nullptr;
  float temperature = 1.0f;
  uint32_t* tokens = nullptr;
  int32_t* accepted = nullptr;
};
cudaError_t verify_drafts(const VerifyDev& v, cudaStream_t st);

}  // namespace nbk
