// window_api.cpp -- the entry points of include/sts_attn.h over drafts, masks and
// kept attention weights: argument checks and the K/V handle's part.
#include <hip/hip_runtime.h>

#include <cmath>

#include "append.hpp"
#include "common.hpp"
#include "decode.hpp"
#include "kv_cache.hpp"
#include "window.hpp"

using sts::fail;
using namespace sts::kv;

namespace {

int check_rows_type(int rows) {
  STS_CHECK(rows == STS_ROWS_F32 || rows == STS_ROWS_BF16, "unknown K/V row type %d", rows);
  return STS_OK;
}

sts::WindowParams window_params(const float* q, const void* k, const void* v, float* out,
                                const int32_t* lens, const int32_t* starts, uint32_t T, uint32_t heads,
                                uint32_t kv_heads, uint32_t head_dim, uint32_t max_len) {
  sts::WindowParams p;
  p.q = q;
  p.k = k;
  p.v = v;
  p.out = out;
  p.lens = lens;
  p.starts = starts;
  p.T = T;
  p.H = heads;
  p.KH = kv_heads;
  p.group = kv_heads ? heads / kv_heads : 0;
  p.dh = head_dim;
  p.M = max_len;
  return p;
}

// The same over a handle's cache (f32 rows) in the state `c`.
sts::WindowParams handle_params(const sts_kv_cache* c, const float* q, float* out, uint32_t T) {
  sts::WindowParams p = window_params(q, c->k, c->v, out, nullptr, nullptr, T, (uint32_t)c->q_heads,
                                      (uint32_t)c->heads, (uint32_t)c->head_dim, (uint32_t)c->max_len);
  p.len = (uint32_t)c->len;
  p.start = (uint32_t)kv_start(c);
  return p;
}

int check_rope(const sts_rope* rope, const sts_kv_cache* c, uint64_t rows) {
  if (!rope) return STS_OK;
  STS_CHECK(rope->head_dim == c->head_dim, "RoPE head_dim %u != cache head_dim %llu", rope->head_dim,
            (unsigned long long)c->head_dim);
  STS_CHECK(c->offset + rows <= rope->max_seq_len, "positions %llu..%llu beyond the RoPE table (%u rows)",
            (unsigned long long)c->offset, (unsigned long long)(c->offset + rows), rope->max_seq_len);
  return STS_OK;
}

}  // namespace

namespace sts {
namespace kv {

// One token a stream, with the scores kept or under a range: where every head has K
// and V rows of its own, in f32, the decode kernel, which has no matrix tile to leave
// 15/16 empty (kept, the account included, 32 heads of 3000 rows 22 us against 27, 64
// streams of 128 to 3000 rows 559 against 592, and on a handle it also rotates and
// appends the token's rows, a launch less; under a range, 2777 rows 17.5 us against
// 22.5, 64 streams over 300 rows of 3000 99 against 112); else the window kernel,
// which reads the rows of a group of heads, or bf16 rows, once.
static bool by_decode(const WindowParams& p, bool bf16) { return p.group == 1 && !bf16; }

static DecodeParams decode_params(const WindowParams& p) {
  DecodeParams d;
  d.q = p.q;
  d.k = static_cast<const float*>(p.k);
  d.v = static_cast<const float*>(p.v);
  d.out = p.out;
  d.rope_cos = p.rope_cos;
  d.rope_sin = p.rope_sin;
  d.rope_pos = p.rope_pos;
  d.lens = p.lens;
  d.starts = p.starts;
  d.len = p.len;
  d.start = p.start;
  d.H = p.H;
  d.M = p.M;
  d.q_bstride = d.out_bstride = d.kn_bstride = (uint64_t)p.H * p.dh;
  d.kv_hstride = (uint64_t)p.M * p.dh;
  d.kv_bstride = (uint64_t)p.H * p.M * p.dh;
  d.scale_log2 = p.qscale;
  d.scores = p.scores;
  d.stats = p.stats;
  d.score_stride = p.score_stride;
  d.lo = p.lo;
  d.hi = p.hi;
  d.counts = p.counts;
  d.slopes = p.slopes;
  d.cap_log2 = p.cap_log2;
  return d;
}

int decode_keeping_weights(const sts_kv_cache* c, const sts_kv_cache* next, const sts_rope* rope,
                           const float* q, const float* k_new, const float* v_new, float* out,
                           float scale, hipStream_t stream) {
  WindowParams p = handle_params(next, q, out, 1);
  const uint32_t batch = (uint32_t)c->batch, max_len = (uint32_t)c->max_len;
  if (int rc = check_window(p, batch, false)) return rc;
  if (rope) {
    p.rope_cos = rope->cos_t;
    p.rope_sin = rope->sin_t;
    p.rope_pos = (uint32_t)c->offset;
  }
  p.qscale = softmax_scale_log2(scale);
  p.score_stride = (uint32_t)score_stride(max_len);
  p.scores = c->scores;
  p.stats = c->scores + (uint64_t)batch * p.H * p.score_stride;
  if (by_decode(p, false)) {
    DecodeParams d = decode_params(p);
    if (k_new) {
      d.k_new = k_new;
      d.v_new = v_new;
      d.k_wr = c->k;
      d.v_wr = c->v;
      d.k16_wr = c->k16;
      d.v16_wr = c->v16;
    }
    if (int rc = launch_decode(d, batch, p.dh, p.len, stream)) return rc;
  } else {
    if (int rc = reserve_window(p, kWindowWeights, batch, false, p.len, stream)) return rc;
    if (k_new) {
      const uint32_t pos = (uint32_t)(c->offset % c->max_len);
      if (int rc = launch_kv_append(k_new, v_new, c->k, c->v, pos, batch, 1, p.KH, p.dh, max_len,
                                    rope ? rope->cos_t : nullptr, rope ? rope->sin_t : nullptr,
                                    (uint32_t)c->offset, c->k16, c->v16, stream))
        return rc;
    }
    if (int rc = launch_window(p, kWindowWeights, batch, false, p.len, stream)) return rc;
  }
  return launch_account(p, c->weights, batch, p.len, k_new != nullptr, stream);
}

}  // namespace kv
}  // namespace sts

extern "C" {

int sts_tree_attention(const float* q, const void* k_cache, const void* v_cache, float* out,
                       const int32_t* parents, const int32_t* counts, const int32_t* lens,
                       const int32_t* starts, uint32_t batch, uint32_t nodes, uint32_t heads,
                       uint32_t kv_heads, uint32_t head_dim, uint32_t max_len, float scale,
                       int row_type, void* stream) {
  sts::clear_error();
  STS_CHECK(q && k_cache && v_cache && out && parents && lens && starts, "null pointer argument");
  if (int rc = check_rows_type(row_type)) return rc;
  STS_CHECK(nodes >= 1 && nodes <= STS_TREE_MAX_NODES, "nodes %u must be in 1..%u", nodes,
            STS_TREE_MAX_NODES);
  STS_CHECK(aligned16(q) && aligned16(k_cache) && aligned16(v_cache) && aligned16(out),
            "q, k_cache, v_cache, out must be 16-byte aligned");
  STS_CHECK(std::isfinite(scale), "scale must be finite");
  sts::WindowParams p = window_params(q, k_cache, v_cache, out, lens, starts, nodes, heads, kv_heads,
                                      head_dim, max_len);
  p.parents = parents;
  p.counts = counts;
  p.qscale = sts::softmax_scale_log2(scale);
  return sts::launch_window(p, sts::kWindowTree, batch, row_type == STS_ROWS_BF16, max_len,
                            as_stream(stream));
}

int sts_tree_commit(void* k_cache, void* v_cache, const int32_t* path, const int32_t* accepted,
                    const int32_t* counts, const int32_t* lens, const int32_t* starts, uint32_t batch,
                    uint32_t nodes, uint32_t kv_heads, uint32_t head_dim, uint32_t max_len,
                    int row_type, void* stream) {
  sts::clear_error();
  STS_CHECK(k_cache && v_cache && path && accepted && lens && starts, "null pointer argument");
  if (int rc = check_rows_type(row_type)) return rc;
  STS_CHECK(nodes >= 1 && nodes <= STS_TREE_MAX_NODES, "nodes %u must be in 1..%u", nodes,
            STS_TREE_MAX_NODES);
  const bool bf16 = row_type == STS_ROWS_BF16;
  sts::WindowParams shape = window_params(nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nodes,
                                          kv_heads, kv_heads, head_dim, max_len);
  if (int rc = sts::check_window(shape, batch, bf16)) return rc;
  STS_CHECK(batch <= 65535 / 3, "batch %u too large for a commit", batch);
  STS_CHECK(aligned16(k_cache) && aligned16(v_cache), "k_cache, v_cache must be 16-byte aligned");
  sts::TreeCommit c;
  c.buf[0] = k_cache;
  c.buf[1] = v_cache;
  c.size[0] = c.size[1] = bf16 ? 2 : 4;
  c.nbuf = 2;
  c.lens = lens;
  c.starts = starts;
  c.counts = counts;
  c.path = path;
  c.accepted = accepted;
  c.T = nodes;
  c.KH = kv_heads;
  c.dh = head_dim;
  c.M = max_len;
  return sts::launch_tree_commit(c, batch, as_stream(stream));
}

int sts_masked_attention(const float* q, const void* k_cache, const void* v_cache, float* out,
                         const int32_t* lo, const int32_t* hi, const float* slopes,
                         const int32_t* counts, const int32_t* lens, const int32_t* starts,
                         uint32_t batch, uint32_t seq, uint32_t heads, uint32_t kv_heads,
                         uint32_t head_dim, uint32_t max_len, float scale, float softcap, int row_type,
                         void* stream) {
  sts::clear_error();
  STS_CHECK(q && k_cache && v_cache && out && lens && starts, "null pointer argument");
  if (int rc = check_rows_type(row_type)) return rc;
  STS_CHECK(aligned16(q) && aligned16(k_cache) && aligned16(v_cache) && aligned16(out),
            "q, k_cache, v_cache, out must be 16-byte aligned");
  STS_CHECK(std::isfinite(scale), "scale must be finite");
  STS_CHECK(std::isfinite(softcap) && softcap >= 0.f, "softcap must be finite and not negative");
  sts::WindowParams p = window_params(q, k_cache, v_cache, out, lens, starts, seq, heads, kv_heads,
                                      head_dim, max_len);
  p.lo = lo;
  p.hi = hi;
  p.slopes = slopes;
  p.counts = counts;
  p.qscale = sts::softmax_scale_log2(scale);
  if (softcap > 0.f) {
    p.qscale = scale / softcap;
    p.cap_log2 = sts::softmax_scale_log2(softcap);
    STS_CHECK(std::isfinite(p.qscale) && std::isfinite(p.cap_log2) && p.cap_log2 > 0.f,
              "scale / softcap out of range");
    // Below, terms of q . k in units of the cap would fall under f32's range.
    STS_CHECK(scale == 0.f || std::fabs(p.qscale) >= 0x1p-100f,
              "softcap %g too large for the scale %g (2^100 times at most)", softcap, scale);
  }
  const bool bf16 = row_type == STS_ROWS_BF16;
  if (int rc = sts::check_window(p, batch, bf16)) return rc;
  if (seq == 1 && sts::kv::by_decode(p, bf16)) {
    sts::DecodeParams d = sts::kv::decode_params(p);
    d.masked = true;
    return sts::launch_decode(d, batch, head_dim, max_len, as_stream(stream));
  }
  return sts::launch_window(p, sts::kWindowMasked, batch, bf16, max_len, as_stream(stream));
}

uint64_t sts_decode_ring_weights_scratch(uint32_t batch, uint32_t heads, uint32_t max_len) {
  return weights_scratch(batch, heads, max_len);
}

int sts_decode_ring_weights(const float* q, const void* k_cache, const void* v_cache, float* out,
                            float* weights, float* scratch, const int32_t* lens,
                            const int32_t* starts, uint32_t batch, uint32_t heads, uint32_t kv_heads,
                            uint32_t head_dim, uint32_t max_len, float scale, int row_type,
                            void* stream) {
  sts::clear_error();
  STS_CHECK(q && k_cache && v_cache && out && weights && scratch && lens && starts,
            "null pointer argument");
  if (int rc = check_rows_type(row_type)) return rc;
  STS_CHECK(aligned16(q) && aligned16(k_cache) && aligned16(v_cache) && aligned16(out) &&
                aligned16(scratch),
            "q, k_cache, v_cache, out, scratch must be 16-byte aligned");
  STS_CHECK(std::isfinite(scale), "scale must be finite");
  sts::WindowParams p = window_params(q, k_cache, v_cache, out, lens, starts, 1, heads, kv_heads,
                                      head_dim, max_len);
  p.qscale = sts::softmax_scale_log2(scale);
  p.score_stride = (uint32_t)score_stride(max_len);
  p.scores = scratch;
  p.stats = scratch + (uint64_t)batch * heads * p.score_stride;
  const bool bf16 = row_type == STS_ROWS_BF16;
  if (int rc = sts::check_window(p, batch, bf16)) return rc;
  if (sts::kv::by_decode(p, bf16)) {
    if (int rc = sts::launch_decode(sts::kv::decode_params(p), batch, head_dim, max_len, as_stream(stream)))
      return rc;
  } else if (int rc = sts::launch_window(p, sts::kWindowWeights, batch, bf16, max_len, as_stream(stream))) {
    return rc;
  }
  return sts::launch_account(p, weights, batch, max_len, false, as_stream(stream));
}

int sts_evict_ring(void* k_cache, void* v_cache, float* weights, int32_t* kept, const int32_t* lens,
                   const int32_t* starts, uint32_t batch, uint32_t kv_heads, uint32_t head_dim,
                   uint32_t max_len, uint32_t keep, uint32_t recent, int row_type, void* stream) {
  sts::clear_error();
  STS_CHECK(k_cache && v_cache && weights && kept && lens && starts, "null pointer argument");
  if (int rc = check_rows_type(row_type)) return rc;
  const bool bf16 = row_type == STS_ROWS_BF16;
  sts::WindowParams shape = window_params(nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, 1,
                                          kv_heads, kv_heads, head_dim, max_len);
  if (int rc = sts::check_window(shape, batch, bf16)) return rc;
  STS_CHECK(keep >= 1 && keep <= max_len, "keep %u must be in 1..max_len", keep);
  STS_CHECK(recent <= keep, "recent %u must be at most keep %u", recent, keep);
  STS_CHECK(aligned16(k_cache) && aligned16(v_cache), "k_cache, v_cache must be 16-byte aligned");
  sts::Evict e;
  e.buf[0] = k_cache;
  e.buf[1] = v_cache;
  e.size[0] = e.size[1] = bf16 ? 2 : 4;
  e.nbuf = 2;
  e.weights = weights;
  e.kept = kept;
  e.lens = lens;
  e.starts = starts;
  e.keep = keep;
  e.recent = recent;
  e.KH = kv_heads;
  e.dh = head_dim;
  e.M = max_len;
  return sts::launch_evict(e, batch, as_stream(stream));
}

/* ---------------------------------------------------------------------- */
/* The K/V handle                                                           */
/* ---------------------------------------------------------------------- */

int sts_kv_weights(const sts_kv_cache* cache, float** weights) {
  sts::clear_error();
  STS_CHECK(cache && weights, "null pointer argument");
  *weights = cache->weights;
  return STS_OK;
}

int sts_kv_tree_step(sts_kv_cache* cache, const sts_rope* rope, const float* q, const float* k_new,
                     const float* v_new, const int32_t* parents, float* out, uint64_t nodes,
                     float scale, void* stream) {
  sts::clear_error();
  // Every check runs before anything is written or the counters move, so a
  // rejected call leaves the cache as it was.
  STS_CHECK(cache && q && k_new && v_new && parents && out, "null pointer argument");
  STS_CHECK(nodes >= 1 && nodes <= STS_TREE_MAX_NODES && nodes <= cache->max_len,
            "nodes %llu must be in 1..%u and at most max_len", (unsigned long long)nodes,
            STS_TREE_MAX_NODES);
  if (cache->k && cache->batch != 1)
    return fail(STS_ERR_STATE, "a draft needs a batch-1 cache (allocated with batch %llu)",
                (unsigned long long)cache->batch);
  STS_CHECK(aligned16(q) && aligned16(k_new) && aligned16(v_new) && aligned16(out),
            "q, k_new, v_new, out must be 16-byte aligned");
  STS_CHECK(std::isfinite(scale), "scale must be finite");
  if (int rc = check_rope(rope, cache, nodes)) return rc;
  hipStream_t s = as_stream(stream);
  sts_kv_cache next = *cache;
  kv_advance(&next, nodes);
  const uint32_t n = (uint32_t)nodes;
  if (int rc = sts::check_window(handle_params(&next, q, out, n), 1, false)) return rc;
  if (int rc = sts::reserve_window(handle_params(&next, q, out, n), sts::kWindowTree, 1, false,
                                (uint32_t)next.len, s)) return rc;
  if (int rc = kv_ensure(cache, 1, s)) return rc;
  const uint64_t offset = cache->offset;
  const uint32_t pos = (uint32_t)(offset % cache->max_len);
  if (int rc = sts::launch_tree_append(k_new, v_new, parents, cache->k, cache->v, cache->k16,
                                       cache->v16, rope ? rope->cos_t : nullptr,
                                       rope ? rope->sin_t : nullptr, (uint32_t)offset, pos, n,
                                       (uint32_t)cache->heads, (uint32_t)cache->head_dim,
                                       (uint32_t)cache->max_len, s))
    return rc;
  if (cache->weights) {
    if (int rc = sts::launch_clear_weights(cache->weights, cache->heads, (uint32_t)cache->max_len, pos, n, s))
      return rc;
  }
  kv_advance(cache, nodes);
  sts::WindowParams p = handle_params(cache, q, out, n);
  p.parents = parents;
  p.qscale = sts::softmax_scale_log2(scale);
  if (rope) {
    p.rope_cos = rope->cos_t;
    p.rope_sin = rope->sin_t;
    p.rope_pos = (uint32_t)offset;
  }
  return sts::launch_window(p, sts::kWindowTree, 1, false, p.len, s);
}

int sts_kv_tree_commit(sts_kv_cache* cache, uint64_t nodes, const uint32_t* path, uint64_t accepted,
                       void* stream) {
  sts::clear_error();
  STS_CHECK(cache && (path || accepted == 0), "null pointer argument");
  STS_CHECK(nodes >= 1 && nodes <= STS_TREE_MAX_NODES && nodes <= cache->len,
            "nodes %llu must be in 1..%u and at most the window's %llu rows",
            (unsigned long long)nodes, STS_TREE_MAX_NODES, (unsigned long long)cache->len);
  STS_CHECK(accepted <= nodes, "accepted %llu must be at most nodes %llu", (unsigned long long)accepted,
            (unsigned long long)nodes);
  if (cache->k && cache->batch != 1)
    return fail(STS_ERR_STATE, "a draft needs a batch-1 cache (allocated with batch %llu)",
                (unsigned long long)cache->batch);
  sts::TreeCommit c;
  bool moves = false;
  for (uint64_t j = 0; j < accepted; ++j) {
    STS_CHECK(path[j] < nodes && (j == 0 || path[j] > path[j - 1]),
              "path must name nodes in ascending order (entry %llu is %u of %llu)",
              (unsigned long long)j, path[j], (unsigned long long)nodes);
    c.path_host[j] = (uint8_t)path[j];
    moves |= path[j] != j;
  }
  if (moves && cache->k) {
    c.buf[0] = cache->k;
    c.buf[1] = cache->v;
    c.size[0] = c.size[1] = 4;
    c.nbuf = 2;
    if (cache->k16) {
      c.buf[2] = cache->k16;
      c.buf[3] = cache->v16;
      c.size[2] = c.size[3] = 2;
      c.nbuf = 4;
    }
    c.weights = cache->weights;
    c.len = (uint32_t)cache->len;
    c.start = (uint32_t)kv_start(cache);
    c.n = (uint32_t)accepted;
    c.T = (uint32_t)nodes;
    c.KH = (uint32_t)cache->heads;
    c.dh = (uint32_t)cache->head_dim;
    c.M = (uint32_t)cache->max_len;
    if (int rc = sts::launch_tree_commit(c, 1, as_stream(stream))) return rc;
  }
  return sts_kv_rollback(cache, nodes - accepted);
}

int sts_kv_evict(sts_kv_cache* cache, uint64_t keep, uint64_t recent, int32_t* kept, void* stream) {
  sts::clear_error();
  STS_CHECK(cache, "null cache handle");
  if (!(cache->flags & STS_KV_WEIGHTS))
    return fail(STS_ERR_STATE, "the cache keeps no attention weights (STS_KV_WEIGHTS)");
  STS_CHECK(keep >= 1 && keep <= cache->max_len, "keep %llu must be in 1..max_len",
            (unsigned long long)keep);
  STS_CHECK(recent <= keep, "recent %llu must be at most keep %llu", (unsigned long long)recent,
            (unsigned long long)keep);
  if (!cache->k) return fail(STS_ERR_STATE, "cache has no buffers yet (nothing appended)");
  if (int rc = sts::check_window(handle_params(cache, nullptr, nullptr, 1), (uint32_t)cache->batch, false))
    return rc;
  if (cache->len <= keep && !kept) return STS_OK;
  sts::Evict e;
  e.buf[0] = cache->k;
  e.buf[1] = cache->v;
  e.size[0] = e.size[1] = 4;
  e.nbuf = 2;
  if (cache->k16) {
    e.buf[2] = cache->k16;
    e.buf[3] = cache->v16;
    e.size[2] = e.size[3] = 2;
    e.nbuf = 4;
  }
  e.weights = cache->weights;
  // The decodes' scratch holds batch * query heads * max_len words or more.
  e.kept = kept ? kept : reinterpret_cast<int32_t*>(cache->scores);
  e.len = (uint32_t)cache->len;
  e.start = (uint32_t)kv_start(cache);
  e.keep = (uint32_t)keep;
  e.recent = (uint32_t)recent;
  e.KH = (uint32_t)cache->heads;
  e.dh = (uint32_t)cache->head_dim;
  e.M = (uint32_t)cache->max_len;
  if (int rc = sts::launch_evict(e, (uint32_t)cache->batch, as_stream(stream))) return rc;
  if (cache->len > keep) cache->len = keep;
  return STS_OK;
}

}  // extern "C"
