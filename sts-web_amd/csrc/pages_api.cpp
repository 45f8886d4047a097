// pages_api.cpp -- the entry points of include/sts_attn.h over K/V rows in pages and
// the verdict on a draft: argument checks.
#include <hip/hip_runtime.h>

#include <cmath>

#include "common.hpp"
#include "decode.hpp"
#include "kv_cache.hpp"
#include "pages.hpp"
#include "verify.hpp"

using sts::fail;
using namespace sts::kv;

namespace {

// The pool, table and rope of a call over `batch` streams, checked.
int paged_rows(const sts_pages* pages, const sts_rope* rope, const int32_t* table, const int32_t* lens,
               uint32_t batch, uint32_t max_pages, uint32_t max_rows, sts::PagedRows* out) {
  STS_CHECK(pages && table && lens && pages->k && pages->v, "null pointer argument");
  const int type = pages->row_type;
  STS_CHECK(type == STS_PAGES_F32 || type == STS_PAGES_BF16 || type == STS_PAGES_INT8,
            "unknown page row type %d", type);
  const bool int8 = type == STS_PAGES_INT8;
  STS_CHECK(!int8 || (pages->k_scale && pages->v_scale), "8-bit rows need k_scale and v_scale");
  STS_CHECK(aligned16(pages->k) && aligned16(pages->v) &&
                (!int8 || (aligned16(pages->k_scale) && aligned16(pages->v_scale))),
            "k, v and their scales must be 16-byte aligned");
  STS_CHECK(batch >= 1 && pages->pages >= 1 && pages->kv_heads >= 1 && max_pages >= 1 && max_rows >= 1,
            "empty shape");
  const uint32_t dh = pages->head_dim, unit = int8 ? 16 : type == STS_PAGES_BF16 ? 8 : 4;
  STS_CHECK(dh >= unit && dh <= 128 && dh % unit == 0,
            "head_dim %u not supported (a multiple of %u up to 128 for these rows)", dh, unit);
  const uint32_t R = pages->page_rows;
  STS_CHECK(R >= 16 && R <= 4096 && (R & (R - 1)) == 0, "page_rows %u must be a power of two in 16..4096", R);
  STS_CHECK(batch <= 65535 && pages->kv_heads <= 65535, "batch (%u) and kv_heads (%u) must be <= 65535", batch,
            pages->kv_heads);
  STS_CHECK(pages->pages <= 0x7FFFFFFFu && (uint64_t)max_pages * R <= 0x7FFFFFFFull,
            "too many pages (%u in the pool, %u of %u rows a stream)", pages->pages, max_pages, R);
  STS_CHECK(max_rows <= (uint64_t)max_pages * R, "max_rows %u must be at most the table's %u pages of %u rows",
            max_rows, max_pages, R);
  out->k = pages->k;
  out->v = pages->v;
  out->ks = pages->k_scale;
  out->vs = pages->v_scale;
  out->table = table;
  out->lens = lens;
  out->pages = pages->pages;
  out->max_pages = max_pages;
  out->max_rows = max_rows;
  out->shift = (uint32_t)__builtin_ctz(R);
  out->KH = pages->kv_heads;
  out->dh = dh;
  out->type = type;
  if (rope) {
    STS_CHECK(rope->head_dim == dh, "RoPE head_dim %u != pages' head_dim %u", rope->head_dim, dh);
    STS_CHECK(max_rows <= rope->max_seq_len, "max_rows %u beyond the RoPE table (%u rows)", max_rows,
              rope->max_seq_len);
    out->rope_cos = rope->cos_t;
    out->rope_sin = rope->sin_t;
  }
  return STS_OK;
}

int check_append(const sts::PagedAppend& a, uint32_t batch) {
  STS_CHECK(a.k_new && a.v_new, "null pointer argument");
  STS_CHECK(aligned16(a.k_new) && aligned16(a.v_new), "k_new, v_new must be 16-byte aligned");
  STS_CHECK(a.stride >= (uint64_t)a.rows.KH * a.rows.dh && a.stride % 4 == 0,
            "new_stride must be at least kv_heads * head_dim and a multiple of 4");
  STS_CHECK(a.T >= 1 && a.T <= a.rows.max_rows, "seq %u must be in 1..max_rows", a.T);
  // (The launch counts its threads in 32 bits: 32 a row.)
  STS_CHECK((uint64_t)batch * a.T * a.rows.KH <= (1u << 26), "too many new rows (%u streams x %u x %u heads)",
            batch, a.T, a.rows.KH);
  return STS_OK;
}

}  // namespace

extern "C" {

int sts_paged_append(const sts_pages* pages, const sts_rope* rope, const float* k_new, const float* v_new,
                     uint64_t new_stride, const int32_t* table, const int32_t* counts, const int32_t* lens,
                     uint32_t batch, uint32_t seq, uint32_t max_pages, uint32_t max_rows, void* stream) {
  sts::clear_error();
  sts::PagedAppend a;
  if (int rc = paged_rows(pages, rope, table, lens, batch, max_pages, max_rows, &a.rows)) return rc;
  a.k_new = k_new;
  a.v_new = v_new;
  a.stride = new_stride;
  a.counts = counts;
  a.T = seq;
  if (int rc = check_append(a, batch)) return rc;
  return sts::launch_paged_append(a, batch, as_stream(stream));
}

int sts_paged_decode(const sts_pages* pages, const sts_rope* rope, const float* q, uint64_t q_stride,
                     const float* k_new, const float* v_new, uint64_t new_stride, float* out,
                     const int32_t* table, const int32_t* lens, uint32_t batch, uint32_t heads,
                     uint32_t max_pages, uint32_t max_rows, float scale, void* stream) {
  sts::clear_error();
  sts::PagedDecode d;
  if (int rc = paged_rows(pages, rope, table, lens, batch, max_pages, max_rows, &d.rows)) return rc;
  STS_CHECK(q && out, "null pointer argument");
  STS_CHECK(!k_new == !v_new, "k_new and v_new must both be given or both be null");
  STS_CHECK(aligned16(q) && aligned16(out), "q, out must be 16-byte aligned");
  STS_CHECK(heads >= 1 && heads % d.rows.KH == 0, "query heads %u not a multiple of the %u K/V heads", heads,
            d.rows.KH);
  STS_CHECK(q_stride >= (uint64_t)heads * d.rows.dh && q_stride % 4 == 0,
            "q_stride must be at least heads * head_dim and a multiple of 4");
  STS_CHECK(std::isfinite(scale), "scale must be finite");
  d.group = heads / d.rows.KH;
  // (The launch counts its threads in 32 bits: a workgroup of 256 for 16 query heads of
  // a K/V head and split.)
  STS_CHECK(((uint64_t)d.group / 16 + 1) * batch * d.rows.KH <= (1u << 22), "too many heads (%u streams x %u)",
            batch, heads);
  d.q = q;
  d.q_stride = q_stride;
  d.out = out;
  d.H = heads;
  d.qscale = sts::softmax_scale_log2(scale);
  if (k_new) {
    sts::PagedAppend a;
    a.rows = d.rows;
    a.k_new = k_new;
    a.v_new = v_new;
    a.stride = new_stride;
    a.T = 1;
    if (int rc = check_append(a, batch)) return rc;
    d.k_new = k_new;
    d.v_new = v_new;
    d.new_stride = new_stride;
  }
  return sts::launch_paged_decode(d, batch, as_stream(stream));
}

int sts_paged_gather(const sts_pages* pages, void* k_out, void* v_out, const int32_t* table, const int32_t* first,
                     const int32_t* lens, uint32_t batch, uint32_t max_pages, uint32_t max_rows, uint32_t max_len,
                     int out_type, void* stream) {
  sts::clear_error();
  sts::PagedGather g;
  if (int rc = paged_rows(pages, nullptr, table, lens, batch, max_pages, max_rows, &g.rows)) return rc;
  STS_CHECK(k_out && v_out, "null pointer argument");
  STS_CHECK(out_type == STS_ROWS_F32 || out_type == STS_ROWS_BF16, "unknown K/V row type %d", out_type);
  STS_CHECK(aligned16(k_out) && aligned16(v_out), "k_out, v_out must be 16-byte aligned");
  STS_CHECK(max_len >= 1 && max_len <= 0x7FFFFFFFu, "max_len %u must be in 1..2^31-1", max_len);
  // (The launch counts its threads in 32 bits: a workgroup of 256 for 32 rows of a head.)
  const uint64_t blocks = (uint64_t)(max_len < max_rows ? max_len : max_rows) / 32 + 2;
  STS_CHECK(blocks * batch * g.rows.KH <= (1u << 23), "too many rows (%u streams x %u heads x %u)", batch,
            g.rows.KH, max_len < max_rows ? max_len : max_rows);
  g.k_out = k_out;
  g.v_out = v_out;
  g.first = first;
  g.M = max_len;
  g.bf16 = out_type == STS_ROWS_BF16;
  return sts::launch_paged_gather(g, batch, as_stream(stream));
}

int sts_verify_draft(const float* target, const float* draft, const int32_t* tokens, const int32_t* parents,
                     const int32_t* counts, const float* rand, int32_t* path, int32_t* accepted, int32_t* next,
                     uint32_t batch, uint32_t nodes, uint32_t vocab, void* stream) {
  sts::clear_error();
  STS_CHECK(target && tokens && parents && rand && path && accepted && next, "null pointer argument");
  STS_CHECK(nodes >= 1 && nodes <= STS_TREE_MAX_NODES, "nodes %u must be in 1..%u", nodes, STS_TREE_MAX_NODES);
  STS_CHECK(batch >= 1 && vocab >= 1, "empty shape");
  STS_CHECK(batch <= 65535 && vocab <= (1u << 28), "batch (%u) must be <= 65535 and vocab (%u) <= 2^28", batch,
            vocab);
  sts::VerifyDraft v;
  v.target = target;
  v.draft = draft;
  v.tokens = tokens;
  v.parents = parents;
  v.counts = counts;
  v.rand = rand;
  v.path = path;
  v.accepted = accepted;
  v.next = next;
  v.T = nodes;
  v.V = vocab;
  return sts::launch_verify_draft(v, batch, as_stream(stream));
}

}  // extern "C"
