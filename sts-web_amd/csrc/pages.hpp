// pages.hpp -- K/V rows kept in pages: append, read back, decode attention.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace sts {

// The rows of one launch's streams.  Row r of stream b, K/V head j, is row
// (page * KH + j) * R + r % R of k and v (rows of dh elements), where
// page = table[b * max_pages + r / R]; an entry outside [0, pages) is no page.
struct PagedRows {
  void* k = nullptr;
  void* v = nullptr;
  float* ks = nullptr;  // the rows' scales (int8 rows)
  float* vs = nullptr;
  const int32_t* table = nullptr;
  const int32_t* lens = nullptr;  // rows of each stream, taken as at most max_rows
  uint32_t pages = 0, max_pages = 0, max_rows = 0;
  uint32_t shift = 0;  // R = 1 << shift
  uint32_t KH = 0, dh = 0;
  int type = 0;  // sts_page_type
  const float* rope_cos = nullptr;  // [at least max_rows][dh/2], or null
  const float* rope_sin = nullptr;
};

// Rows lens[b] - counts[b] + i of each stream, i < counts[b] (null: T; at most T and
// lens[b]), written from token i of stream b at k_new + (b*T + i)*stride + j*dh.
struct PagedAppend {
  PagedRows rows;
  const float* k_new = nullptr;
  const float* v_new = nullptr;
  uint64_t stride = 0;
  const int32_t* counts = nullptr;
  uint32_t T = 0;
};
int launch_paged_append(const PagedAppend& p, uint32_t batch, hipStream_t stream);

// Row first[b] + i (null: 0) of stream b to row i of k_out, v_out [B][KH][M][dh],
// i < M; bf16: rounded to nearest even, else f32.
struct PagedGather {
  PagedRows rows;
  void* k_out = nullptr;
  void* v_out = nullptr;
  const int32_t* first = nullptr;
  uint32_t M = 0;
  bool bf16 = false;
};
int launch_paged_gather(const PagedGather& p, uint32_t batch, hipStream_t stream);

// One query of each stream over all of its rows.
struct PagedDecode {
  PagedRows rows;
  const float* q = nullptr;  // stream b, head h at q + b*q_stride + h*dh
  uint64_t q_stride = 0;
  // The newest row of stream b, written first: K/V head j at k_new + b*new_stride + j*dh;
  // or null.
  const float* k_new = nullptr;
  const float* v_new = nullptr;
  uint64_t new_stride = 0;
  float* out = nullptr;      // [B][H][dh]
  uint32_t H = 0, group = 1;
  float qscale = 0.f;        // scale * log2(e)
  // Set by launch_paged_decode.
  uint32_t rblocks = 1, nsplit = 1, batch = 0;
  float rows_factor = 0.f;   // rows of a split for each row there is; 0: nsplit for every stream
  uint32_t record = 0;       // floats of a split's record
  float* part = nullptr;
  uint32_t* counters = nullptr;
};
int launch_paged_decode(PagedDecode p, uint32_t batch, hipStream_t stream);

}  // namespace sts
