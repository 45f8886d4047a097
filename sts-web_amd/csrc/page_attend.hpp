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
    float total = (float)mine_len;
#pragma unroll
    for (int x = 1; x < 64; x *= 2) total += __shfl_xor(total, x, 64);
    const uint32_t chunk = max((uint32_t)min(total * p.rows_factor, 0x1p31f) + 1, unit);
    const uint32_t mine = lane < (int)p.batch ? min(max((mine_len + chunk - 1) / chunk, 1u), p.nsplit) : 0;
    uint32_t before = mine;
#pragma unroll
    for (int x = 1; x < 64; x *= 2) {
      const uint32_t y = (uint32_t)__shfl_up((int)before, x, 64);
      before += lane >= x ? y : 0;
    }
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

// The splits of a block of `live` query heads merged by the last of its workgroups to
// arrive, always in the same order: record sp of prs holds O [live][D], then (m, l)
// [live].  mem: kMergeBytes of LDS that every thread is done with; sums [16][2];
// finish(x, a, l) gets float4 column x of the unnormalised outputs and its head's l.
constexpr int kMergeBytes = 2 * kMaxSplits * 16 * 4 + kWaves * 64 * 16;
template <int D, bool PAD, class Finish>
__device__ __forceinline__ void merge_splits(const PagedDecode& p, __amdgpu_buffer_rsrc_t prs, char* mem,
                                             float (*sums)[2], uint32_t& s_last, uint32_t live, uint32_t nsplit,
                                             uint64_t unit, Finish finish) {
  constexpr int C4 = D / 4;
  const int tid = threadIdx.x;
  const uint32_t REC = p.record, slots = live * C4;
  // Every thread's records are acknowledged before the workgroup takes its arrival
  // ticket; the last one merges the splits, always in the same order.
  __builtin_amdgcn_s_waitcnt(0);
  __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "workgroup");
  __syncthreads();
  if (tid == 0) {
    const uint32_t ticket = atomicAdd(p.counters + unit, 1u);
    s_last = ticket == nsplit - 1;
    if (ticket == nsplit - 1) atomicExch(p.counters + unit, 0u);
  }
  __syncthreads();
  if (!s_last) return;
  __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "workgroup");
  // The splits' (m, l) of every head; m gives way to the split's factor 2^(m_s - m).
  auto& s_f = *reinterpret_cast<float(*)[kMaxSplits][16]>(mem);
  auto& s_l = *reinterpret_cast<float(*)[kMaxSplits][16]>(mem + kMaxSplits * 16 * 4);
  auto& s_sum = *reinterpret_cast<f32x4(*)[kWaves * 64]>(mem + 2 * kMaxSplits * 16 * 4);
  for (uint32_t x = tid; x < nsplit * live; x += kWaves * 64) {
    const uint32_t sp = x / live, row = x % live;
    const u32x2 y = __builtin_amdgcn_raw_buffer_load_b64(prs, (sp * REC + live * D + row * 2) * 4, 0, kSc1);
    s_f[sp][row] = __uint_as_float(y[0]);
    s_l[sp][row] = __uint_as_float(y[1]);
  }
  __syncthreads();
  if (tid < (int)live) {
    float mt = -FLT_MAX, lt = 0.f;
    for (uint32_t sp = 0; sp < nsplit; ++sp) mt = fmaxf(mt, s_f[sp][tid]);
    for (uint32_t sp = 0; sp < nsplit; ++sp) {
      const float f = exp2_hw(s_f[sp][tid] - mt);
      s_f[sp][tid] = f;
      lt += f * s_l[sp][tid];
    }
    sums[tid][1] = lt;
  }
  __syncthreads();
  // Groups of threads, one for each column, take the splits in turn.
  constexpr int AT = 8;
  for (uint32_t x0 = 0; x0 < slots; x0 += kWaves * 64) {
    const uint32_t n = min(slots - x0, (uint32_t)(kWaves * 64)), groups = kWaves * 64 / n;
    const uint32_t x = x0 + tid % n, grp = tid / n;
    f32x4 a = f32x4{0.f, 0.f, 0.f, 0.f};
    if (grp < groups) {
      for (uint32_t sp = grp; sp < nsplit; sp += AT * groups) {
        coh_f4 y[AT];
#pragma unroll
        for (int u = 0; u < AT; ++u)
          y[u] = ld_coherent4(prs, sp + u * groups < nsplit ? ((sp + u * groups) * REC + x * 4) * 4 : kOutside);
#pragma unroll
        for (int u = 0; u < AT; ++u)
          if (sp + u * groups < nsplit) a += y[u] * s_f[sp + u * groups][x / C4];
      }
    }
    __syncthreads();
    s_sum[tid] = a;
    __syncthreads();
    if (grp == 0) {
      for (uint32_t u = 1; u < groups; ++u) a += s_sum[tid + u * n];
      finish(x, make_float4(a[0], a[1], a[2], a[3]), sums[x / C4][1]);
    }
  }
}

}  // namespace paged

// The kernels' launches: p is planned, nsplit and shares set.
int launch_paged_lone(const PagedDecode& p, dim3 grid, hipStream_t stream);

}  // namespace sts
