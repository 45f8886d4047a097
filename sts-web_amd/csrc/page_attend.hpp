// page_attend.hpp -- what the decode kernels over paged rows share: loads, the deal of
// the rows to workgroups, and the merge of their splits.
#pragma once

#include "coherent.hpp"
#include "common.hpp"
#include "lane.hpp"
#include "page_rows.hpp"
#include "rope.hpp"
#include "score.hpp"

namespace sts {
namespace paged {

constexpr int kWaves = 4;
constexpr int kNt = 2;  // cache policy: nontemporal, each row is read once
constexpr uint32_t kOutside = 0x80000000u;  // past every buffer resource: loads zeros
constexpr int kMaxSplits = 128;

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template <int WORDS>
struct Words {
  uint32_t w[WORDS];
  __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t rs, uint32_t off) {
    if constexpr (WORDS == 4) {
      const u32x4 x = __builtin_amdgcn_raw_buffer_load_b128(rs, off, 0, kNt);
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = x[i];
    } else if constexpr (WORDS == 2) {
      const u32x2 x = __builtin_amdgcn_raw_buffer_load_b64(rs, off, 0, kNt);
      w[0] = x[0];
      w[1] = x[1];
    } else {
      w[0] = __builtin_amdgcn_raw_buffer_load_b32(rs, off, 0, kNt);
    }
  }
};

// Over all 64 lanes.
__device__ __forceinline__ float lanes_max(float x) {
  x = fmaxf(x, xchg<0>(x));
  x = fmaxf(x, xchg<1>(x));
  x = fmaxf(x, xchg<2>(x));
  x = fmaxf(x, xchg<3>(x));
  return max_xor32(max_xor16(x));
}
__device__ __forceinline__ float lanes_sum(float x) {
  x += xchg<0>(x);
  x += xchg<1>(x);
  x += xchg<2>(x);
  x += xchg<3>(x);
  return sum_xor32(sum_xor16(x));
}

// What a workgroup has to do: one split of one stream and K/V head.
struct Share {
  uint32_t b, kvh, split, splits;
  uint32_t first;  // splits of the streams before, each counted once for all heads
  uint32_t len;    // the stream's rows
};

// The share of that number; false past the last.  unit: the rows below which no split
// goes.  Everything found is uniform.
__device__ __forceinline__ bool find_share(const PagedDecode& p, uint32_t share, uint32_t unit, Share& s) {
  const PagedRows& rows = p.rows;
  if (p.rows_factor > 0.f) {
    // Streams of different lengths are cut into splits of about the same length: lane
    // x looks at stream x, and the share's stream is the last whose streams before take
    // no more shares.
    const int lane = threadIdx.x & 63;
    const uint32_t mine_len = lane < (int)p.batch ? paged_len(rows, lane) : 0u;
    const float total = lanes_sum((float)mine_len);
    const uint32_t chunk = max((uint32_t)min(total * p.rows_factor, 0x1p31f) + 1, unit);
    const uint32_t mine = lane < (int)p.batch ? min(max((mine_len + chunk - 1) / chunk, 1u), p.nsplit) : 0;
    uint32_t before = lanes_upto(mine);
    if (share >= (uint32_t)__builtin_amdgcn_readlane((int)before, 63) * rows.KH) return false;
    before -= mine;
    s.b = 63 - __builtin_clzll(__ballot(lane < (int)p.batch && before * rows.KH <= share));
    s.splits = (uint32_t)__builtin_amdgcn_readlane((int)mine, s.b);
    s.first = (uint32_t)__builtin_amdgcn_readlane((int)before, s.b);
    const uint32_t at = share - s.first * rows.KH;
    s.kvh = at % rows.KH;
    s.split = at / rows.KH;
    s.len = (uint32_t)__builtin_amdgcn_readlane((int)mine_len, s.b);
  } else {
    s.splits = p.nsplit;
    s.split = share % s.splits;
    s.kvh = share / s.splits % rows.KH;
    s.b = share / s.splits / rows.KH;
    s.first = s.b * s.splits;
    s.len = __builtin_amdgcn_readfirstlane(paged_len(rows, s.b));
  }
  return true;
}

// ---- merge of the splits ------------------------------------------------------
//
// Record sp of a block of `live` query heads holds its split's O [live][D], then (m, l)
// [live]; a workgroup that has published its own takes a ticket, and the last to arrive
// merges them, always in the same order.  A thread has kAhead columns of records
// requested at once.  Where that would be more than two round trips (one workgroup of 128
// splits of 8 heads: 17 us), clusters of about the root of their number are merged first,
// each by its own last, and the clusters' records after that.
constexpr int kAhead = 8;
constexpr int kClusters = 16;  // at most: of kMaxSplits, 11
constexpr uint32_t kCounters = 1 + kClusters;  // arrival counters of a block
constexpr int kMergeBytes = kMaxSplits * 16 * 4 + 128 + kWaves * 64 * 16;

struct Records {
  __amdgpu_buffer_rsrc_t rs;
  uint32_t size;  // floats of a record
  uint32_t live;
};

// Whether this workgroup, whose stores it waits for, is the last of n to get here.
__device__ __forceinline__ bool last_of(uint32_t* counter, uint32_t n, uint32_t& s_last) {
  __builtin_amdgcn_s_waitcnt(0);
  __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "workgroup");
  __syncthreads();
  if (threadIdx.x == 0) {
    const uint32_t ticket = atomicAdd(counter, 1u);
    s_last = ticket == n - 1;
    if (ticket == n - 1) atomicExch(counter, 0u);
  }
  __syncthreads();
  const bool last = s_last;
  __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "workgroup");
  return last;
}

// Records from, from + step, ... (n of them): put(x, a, m, l) gets float4 column x of
// their merged O and its head's m and l.  mem: kMergeBytes of LDS that every thread is
// done with.
template <int D, class Put>
__device__ __forceinline__ void merge_records(const Records& r, uint32_t from, uint32_t step, uint32_t n, char* mem,
                                              Put put) {
  constexpr int C4 = D / 4;
  const int tid = threadIdx.x;
  const uint32_t live = r.live, slots = live * C4;
  auto& s_f = *reinterpret_cast<float(*)[kMaxSplits][16]>(mem);  // the records' factors 2^(m_s - m)
  auto& s_ml = *reinterpret_cast<float(*)[2][16]>(mem + kMaxSplits * 16 * 4);
  auto& s_sum = *reinterpret_cast<f32x4(*)[kWaves * 64]>(mem + kMaxSplits * 16 * 4 + 128);
  coh_f4 y[kAhead];
  // Groups of threads, one for each column, take the records in turn.
  auto request = [&](uint32_t sp, uint32_t groups, uint32_t x) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      y[u] = ld_coherent4(r.rs, sp + u * groups < n ? ((from + (sp + u * groups) * step) * r.size + x * 4) * 4 : kOutside);
  };
  const uint32_t n0 = min(slots, (uint32_t)(kWaves * 64)), g0 = kWaves * 64 / n0;
  // A wave looks after every fourth head, its lanes after two records each.
  const uint32_t lane = tid & 63, wave = tid >> 6;
  u32x2 ml[16 / kWaves][2];
#pragma unroll
  for (int i = 0; i < 16 / kWaves; ++i)
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const uint32_t sp = lane + 64 * u, row = wave + kWaves * i;
      ml[i][u] = __builtin_amdgcn_raw_buffer_load_b64(
          r.rs, sp < n && row < live ? ((from + sp * step) * r.size + live * D + row * 2) * 4 : kOutside, 0, kSc1);
    }
  if (tid / n0 < g0) request(tid / n0, g0, tid % n0);
#pragma unroll
  for (int i = 0; i < 16 / kWaves; ++i) {
    const uint32_t row = wave + kWaves * i;
    if (row >= live) break;
    float m[2], mt = -FLT_MAX;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      m[u] = lane + 64 * u < n ? __uint_as_float(ml[i][u][0]) : -FLT_MAX;
      mt = fmaxf(mt, m[u]);
    }
    mt = lanes_max(mt);
    float lt = 0.f;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const float f = exp2_hw(m[u] - mt);
      if (lane + 64 * u < n) s_f[lane + 64 * u][row] = f;
      lt += f * __uint_as_float(ml[i][u][1]);  // (0 past the records)
    }
    lt = lanes_sum(lt);
    if (lane == 0) {
      s_ml[0][row] = mt;
      s_ml[1][row] = lt;
    }
  }
  __syncthreads();
  for (uint32_t x0 = 0; x0 < slots; x0 += kWaves * 64) {
    const uint32_t cols = min(slots - x0, (uint32_t)(kWaves * 64)), groups = kWaves * 64 / cols;
    const uint32_t x = x0 + tid % cols, grp = tid / cols;
    f32x4 a = f32x4{0.f, 0.f, 0.f, 0.f};
    if (grp < groups) {
      for (uint32_t sp = grp; sp < n; sp += kAhead * groups) {
        if (x0 > 0 || sp != grp) request(sp, groups, x);
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
          if (sp + u * groups < n) a += y[u] * s_f[sp + u * groups][x / C4];
      }
    }
    if (groups > 1) {
      s_sum[tid] = a;
      __syncthreads();
      if (grp == 0)
        for (uint32_t u = 1; u < groups; ++u) a += s_sum[tid + u * cols];
    }
    if (grp == 0) put(x, make_float4(a[0], a[1], a[2], a[3]), s_ml[0][x / C4], s_ml[1][x / C4]);
  }
}

// Column x of a record, and its head's (m, l).
template <int D>
__device__ __forceinline__ void put_record(const Records& r, uint32_t sp, uint32_t x, float4 a, float m, float l) {
  constexpr int C4 = D / 4;
  st_coherent4(r.rs, (sp * r.size + x * 4) * 4, coh_f4{a.x, a.y, a.z, a.w});
  if (x % C4 == 0)
    __builtin_amdgcn_raw_buffer_store_b64(u32x2{__float_as_uint(m), __float_as_uint(l)}, r.rs,
                                          (sp * r.size + r.live * D + x / C4 * 2) * 4, 0, kSc1);
}

// Records of `slots` columns that are read in one round trip.
__host__ __device__ constexpr uint32_t read_at_once(uint32_t slots) {
  return slots <= kWaves * 64 ? kWaves * 64 / slots * kAhead : kAhead / 2;
}

// What follows a split's put_record: its part in the merge, whose outcome goes to put.
// HEADS: a block's at most (of one head no splits are too many for one merge).
template <int D, int HEADS, class Put>
__device__ __forceinline__ void merge_splits(const Records& r, uint32_t* counters, uint32_t split, uint32_t nsplit,
                                             char* mem, uint32_t& s_last, Put put) {
  uint32_t from = 0, step = 1, n = nsplit;
  if constexpr (kMaxSplits > 2 * read_at_once(HEADS * (D / 4))) {
    if (nsplit > 2 * read_at_once(r.live * (D / 4))) {
      uint32_t size = 1;
      while (size * size < nsplit) ++size;
      const uint32_t cluster = split / size, first = cluster * size, some = min(size, nsplit - first);
      if (!last_of(counters + 1 + cluster, some, s_last)) return;
      // (A column's first record is read by the thread that then writes it.)
      merge_records<D>(r, first, 1, some, mem,
                       [&](uint32_t x, float4 a, float m, float l) { put_record<D>(r, first, x, a, m, l); });
      step = size;
      n = (nsplit + size - 1) / size;
    }
  }
  if (!last_of(counters, n, s_last)) return;
  merge_records<D>(r, from, step, n, mem, put);
}

}  // namespace paged

// The kernels' launches: p is planned.
int launch_paged_lone(const PagedDecode& p, dim3 grid, hipStream_t stream);

}  // namespace sts
