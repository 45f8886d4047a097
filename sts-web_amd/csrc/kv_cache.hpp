// kv_cache.hpp -- the RoPE table and K/V cache handles behind the C ABI, and what
// their entry points share (host code).
#pragma once

#include <hip/hip_runtime.h>

#include "common.hpp"
#include "window.hpp"

struct sts_rope {
  uint32_t head_dim = 0;
  uint32_t max_seq_len = 0;
  float* cos_t = nullptr;  // device [max_seq_len][head_dim/2]
  float* sin_t = nullptr;
};

struct sts_kv_cache {
  uint64_t max_len = 0, heads = 0, head_dim = 0;
  uint64_t q_heads = 0;  // query heads of q/out (a multiple of heads: GQA)
  uint64_t offset = 0, len = 0, write_pos = 0;
  uint64_t batch = 0;
  uint32_t flags = 0;
  float* k = nullptr;
  float* v = nullptr;
  uint16_t* k16 = nullptr;      // bf16 mirror (STS_KV_BF16_MIRROR)
  uint16_t* v16 = nullptr;
  float* weights = nullptr;  // [batch][heads][max_len] (STS_KV_WEIGHTS), and the
  float* scores = nullptr;   // scratch of the decodes that keep them
};

namespace sts {
namespace kv {

inline hipStream_t as_stream(void* s) { return reinterpret_cast<hipStream_t>(s); }

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Any multiple of 4 up to 128 (shader_attention.wgsl:36 takes head_dim <= 128);
// 64 and 128 have their own kernels, the others run padded ones.
inline int check_head_dim(uint64_t d) {
  if (d == 0 || d > 128 || d % 4 != 0)
    return ::sts::fail(STS_ERR_INVALID, "head_dim %llu not supported (a multiple of 4 up to 128)",
                (unsigned long long)d);
  return STS_OK;
}

// KVCache::advance (model.rs:293-298), n steps of the one-step update.
inline void kv_advance(sts_kv_cache* c, uint64_t n) {
  if (n >= c->max_len) {
    // Whole-ring advance: the same end state as n single steps.
    c->write_pos = (c->write_pos + n) % c->max_len;
    c->offset += n;
    c->len = c->max_len;
    return;
  }
  c->write_pos = (c->write_pos + n) % c->max_len;
  c->offset += n;
  c->len = (c->len + n < c->max_len) ? c->len + n : c->max_len;
}

// Oldest valid slot of the logical window.
inline uint64_t kv_start(const sts_kv_cache* c) {
  return (c->write_pos + c->max_len - c->len) % c->max_len;
}

inline void kv_free(sts_kv_cache* c) {
  for (void* ptr : {(void*)c->k, (void*)c->v, (void*)c->k16, (void*)c->v16,
                    (void*)c->weights, (void*)c->scores})
    if (ptr) (void)hipFree(ptr);
  c->k = c->v = nullptr;
  c->k16 = c->v16 = nullptr;
  c->weights = c->scores = nullptr;
}

// Floats that a decode which keeps the weights needs: the scores of every query
// head's window rows (whole tiles of 16), then each head's maximum and sum.
inline uint64_t score_stride(uint64_t max_len) { return (max_len + 15) / 16 * 16; }
inline uint64_t weights_scratch(uint64_t batch, uint64_t heads, uint64_t max_len) {
  return batch * heads * (score_stride(max_len) + 2);
}

inline int kv_ensure(sts_kv_cache* c, uint64_t batch, hipStream_t stream) {
  if (c->k) {
    if (batch != c->batch)
      return ::sts::fail(STS_ERR_STATE, "cache allocated for batch %llu, called with batch %llu",
                  (unsigned long long)c->batch, (unsigned long long)batch);
    return STS_OK;
  }
  if (batch == 0) return fail(STS_ERR_INVALID, "batch must be >= 1");
  // The lazy allocation must not be recorded into a HIP graph (its zero fill
  // would be a memset node, and the graph would own nothing it addresses).
  hipStreamCaptureStatus cap = hipStreamCaptureStatusNone;
  STS_HIP(hipStreamIsCapturing(stream, &cap));
  if (cap != hipStreamCaptureStatusNone)
    return ::sts::fail(STS_ERR_STATE,
                "the cache's first use allocates its buffers, which cannot happen while the "
                "stream is being captured; allocate it first (sts_kv_ensure_allocated)");
  const uint64_t n = batch * c->heads * c->max_len * c->head_dim;
  if (hipMalloc(&c->k, n * sizeof(float)) != hipSuccess) {
    c->k = nullptr;
    return ::sts::fail(STS_ERR_NOMEM, "K cache allocation of %llu bytes failed",
                (unsigned long long)(n * sizeof(float)));
  }
  if (hipMalloc(&c->v, n * sizeof(float)) != hipSuccess) {
    (void)hipFree(c->k);
    c->k = nullptr;
    c->v = nullptr;
    return ::sts::fail(STS_ERR_NOMEM, "V cache allocation of %llu bytes failed",
                (unsigned long long)(n * sizeof(float)));
  }
  if (c->flags & STS_KV_BF16_MIRROR) {
    if (hipMalloc(&c->k16, n * sizeof(uint16_t)) != hipSuccess ||
        hipMalloc(&c->v16, n * sizeof(uint16_t)) != hipSuccess) {
      for (void* ptr : {(void*)c->k, (void*)c->v, (void*)c->k16, (void*)c->v16})
        if (ptr) (void)hipFree(ptr);
      c->k = c->v = nullptr;
      c->k16 = c->v16 = nullptr;
      return ::sts::fail(STS_ERR_NOMEM, "bf16 mirror allocation of %llu bytes failed",
                  (unsigned long long)(2 * n * sizeof(uint16_t)));
    }
    STS_HIP(hipMemsetAsync(c->k16, 0, n * sizeof(uint16_t), stream));
    STS_HIP(hipMemsetAsync(c->v16, 0, n * sizeof(uint16_t), stream));
  }
  if (c->flags & STS_KV_WEIGHTS) {
    const uint64_t nw = batch * c->heads * c->max_len;
    if (hipMalloc(&c->weights, nw * sizeof(float)) != hipSuccess ||
        hipMalloc(&c->scores, weights_scratch(batch, c->q_heads, c->max_len) * sizeof(float)) != hipSuccess) {
      kv_free(c);
      return ::sts::fail(STS_ERR_NOMEM, "attention weights allocation of %llu bytes failed",
                         (unsigned long long)(nw * sizeof(float)));
    }
    if (int rc = launch_clear_weights(c->weights, batch * c->heads, (uint32_t)c->max_len, 0,
                                      (uint32_t)c->max_len, stream)) {
      kv_free(c);
      return rc;
    }
  }
  // Zero-filled like Tensor::zeros (model.rs:272-279).
  STS_HIP(hipMemsetAsync(c->k, 0, n * sizeof(float), stream));
  STS_HIP(hipMemsetAsync(c->v, 0, n * sizeof(float), stream));
  c->batch = batch;
  return STS_OK;
}

// The decode of a cache that keeps attention weights (STS_KV_WEIGHTS): attention of
// q over the window and the account of it; with k_new / v_new, their row is
// appended (rotated at the cache's offset with `rope`, as q is) and counted in
// `next`, the handle's state after the call.  Everything that can be refused is
// refused before anything is written.
int decode_keeping_weights(const sts_kv_cache* c, const sts_kv_cache* next, const sts_rope* rope,
                           const float* q, const float* k_new, const float* v_new, float* out,
                           float scale, hipStream_t stream);

}  // namespace kv
}  // namespace sts
