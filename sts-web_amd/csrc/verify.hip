// verify.hip -- the verdict on a draft (gfx950).  No counterpart in the reference, which
// samples one token a step (crates/sts-wasm/src/wgsl/shader_sample_topk.wgsl).
//
// Speculative sampling down a tree.  At a place (a kept node) let p be the target's
// probabilities there and q those that its children were drawn from; r = p and m = 1 at
// first.  Each child in turn, of token x:
//   kept      if u q(x) m < r(x): the walk goes on at the child
//   rejected  otherwise: r <- max(0, r / m - q), m <- sum r (unless that is zero)
// and where no child is kept a token is drawn from r / m.  The tokens are then distributed
// as the target's.  Children taken without chance (no q) stand for q = 1 at their own
// token: r(x) <- 0 instead, m <- sum r.
//
// r is never stored: a word's r follows from p, q and the masses of the rejections
// before.  Without q, one sum over the words that are no child's token serves all of a
// place's rejections: the children's own are added to it.  Sums and comparisons are in
// f64, so that the verdict is that of exact arithmetic but where a random number lies
// within 2^-45 of a border.
//
// One workgroup a stream.  The numbers at the drafted tokens are read once, all
// together; whole rows only where something is rejected and for the last draw, each wave
// a stretch of the words, so that the draw finds its wave from sixteen sums.  What bounds
// it is the latency of these steps, not the bytes.
#include "common.hpp"
#include "verify.hpp"
#include "window.hpp"

namespace sts {

namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kBatch = 8;
typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));  // rows start anywhere

__device__ __forceinline__ double wave_total(double x) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) x += __shfl_xor(x, d, 64);
  return x;
}

// CH: 64 nodes each.
template <bool DRAWN, int CH>
__global__ __launch_bounds__(kThreads) void verify_kernel(const VerifyDraft p) {
  __shared__ int32_t s_token[CH * 64], s_parent[CH * 64];
  __shared__ float s_rand[CH * 64], s_p[CH * 64], s_q[CH * 64];
  __shared__ double s_mass[DRAWN ? CH * 64 : 1];  // the masses that rejections divided by
  __shared__ int32_t s_out[DRAWN ? 1 : CH * 64];  // the words that a sum leaves out
  __shared__ double s_sum[kWaves];
  __shared__ int32_t s_last[kWaves];

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t b = blockIdx.x, V = p.V;
  const uint64_t base = (uint64_t)b * p.T;
  int count_at = (int)p.T;
  if (p.counts) count_at = p.counts[b];
  if (tid < CH * 64) {
    int token_at = -1, parent_at = -1;
    float u_at = 0.f, at_p = 0.f, at_q = DRAWN ? 0.f : 1.f;
    if (tid < (int)p.T) {
      token_at = p.tokens[base + tid];
      parent_at = p.parents[base + tid];
      u_at = p.rand[base + tid];
    }
    parent_at = tid < count_at && parent_at >= 0 && parent_at < tid ? parent_at : -1;
    token_at = (uint32_t)token_at < V ? token_at : -1;
    if (parent_at >= 0 && token_at >= 0) {
      at_p = p.target[(base + parent_at) * V + token_at];
      if constexpr (DRAWN) at_q = p.draft[(base + parent_at) * V + token_at];
    }
    s_token[tid] = token_at;
    s_parent[tid] = parent_at;
    s_rand[tid] = u_at;
    s_p[tid] = at_p > 0.f ? at_p : 0.f;
    s_q[tid] = at_q > 0.f ? at_q : 0.f;
  }
  const int n = min(max(count_at, 0), (int)p.T);
  if (n == 0) {
    if (tid < (int)p.T) p.path[base + tid] = -1;
    if (tid == 0) {
      p.accepted[b] = 0;
      p.next[b] = -1;
    }
    return;
  }
  __syncthreads();
  // Every wave keeps the nodes in its lanes, node c*64 + lane in element c.
  int token[CH], parent[CH], path[CH];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    token[c] = s_token[c * 64 + lane];
    parent[c] = s_parent[c * 64 + lane];
    path[c] = -1;
  }

  // The wave's stretch of the words: whole steps of 256.
  const uint32_t steps = ((V + 255) / 256 + kWaves - 1) / kWaves;
  const uint32_t from = wave * steps * 256 + lane * 4;
  auto word4 = [&](const float* row, uint32_t x) {  // words x .. x+3 of a row, zeros past its end
    f4 y = {0.f, 0.f, 0.f, 0.f};
    if (x + 4 <= V) {
      y = *reinterpret_cast<const f4*>(row + x);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (x + e < V) y[e] = row[x + e];
    }
    return y;
  };
  // The words of steps step .. step + kBatch - 1 of place cur, requested together.
  struct Batch {
    f4 p[kBatch], q[DRAWN ? kBatch : 1];
  };
  auto load = [&](int cur, uint32_t step, Batch& x) {
    const float* row = p.target + (base + cur) * V;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) x.p[i] = word4(row, step + i < steps ? from + (step + i) * 256 : V);
    if constexpr (DRAWN) {
      row = p.draft + (base + cur) * V;
#pragma unroll
      for (int i = 0; i < kBatch; ++i) x.q[i] = word4(row, step + i < steps ? from + (step + i) * 256 : V);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  // What is left of N words after k rejections.
  auto left_of = [&](const float* at_p, const float* at_q, int k, auto& r) {
    constexpr int N = sizeof(r) / sizeof(double);
#pragma unroll
    for (int e = 0; e < N; ++e) r[e] = at_p[e] > 0.f ? (double)at_p[e] : 0.0;
    if constexpr (DRAWN) {
      if (k > 0) {
#pragma unroll
        for (int e = 0; e < N; ++e) r[e] = fmax(r[e] - (at_q[e] > 0.f ? (double)at_q[e] : 0.0), 0.0);
#pragma unroll 1
        for (int j = 1; j < k; ++j) {
          const double m = s_mass[j];
#pragma unroll
          for (int e = 0; e < N; ++e) r[e] = fmax(r[e] / m - (at_q[e] > 0.f ? (double)at_q[e] : 0.0), 0.0);
        }
      }
    }
  };
  // The same of words x .. x+3 of step i of a batch (without draft: without the k words of
  // s_out).
  auto left4 = [&](const Batch& y, int i, uint32_t x, int k, double (&r)[4]) {
    const float at_p[4] = {y.p[i][0], y.p[i][1], y.p[i][2], y.p[i][3]};
    float at_q[4] = {0.f, 0.f, 0.f, 0.f};
    if constexpr (DRAWN) {
#pragma unroll
      for (int e = 0; e < 4; ++e) at_q[e] = y.q[i][e];
    }
    left_of(at_p, at_q, k, r);
    if constexpr (!DRAWN) {
      for (int j = 0; j < k; ++j) {
        const uint32_t d = (uint32_t)s_out[j] - x;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (d == (uint32_t)e) r[e] = 0.0;
      }
    }
  };
  // Its sum over all words, the waves' sums in s_sum.
  auto sum_left = [&](int cur, int k) {
    double sum = 0.0;
#pragma unroll 1
    for (uint32_t step = 0; step < steps; step += kBatch) {
      Batch y;
      load(cur, step, y);
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        double r[4];
        left4(y, i, from + (step + i) * 256, k, r);
        sum += (r[0] + r[1]) + (r[2] + r[3]);
        __builtin_amdgcn_sched_barrier(0);  // (registers)
      }
    }
    sum = wave_total(sum);
    __syncthreads();
    if (lane == 0) s_sum[wave] = sum;
    __syncthreads();
    double total = 0.0;
    for (int w = 0; w < kWaves; ++w) total += s_sum[w];
    return total;
  };

  // The walk, the same on every wave: a node's children come after it, and once one is
  // kept its own come next.
  int cur = 0, k = 0, len = 1;
  double mass = 1.0;
  bool summed = false;  // s_sum holds the sums of r as it is
  // Without draft: the sum over the words that are no child's, once there is one (else
  // -1); the words out are those of the children up to node `cut`.
  double others = -1.0;
  int cut = 0;
  // The first child of cur behind node i, or n.
  auto next_child = [&](int i) {
    int found = n;
#pragma unroll
    for (int c = CH - 1; c >= 0; --c) {
      const uint64_t m = __ballot(parent[c] == cur && c * 64 + lane > i);
      if (m) found = c * 64 + __builtin_ctzll(m);
    }
    return found;
  };
  // Lists the words that are out, of the children up to node `last`, and counts them.
  auto list_out = [&](int last) {
    __syncthreads();  // (every thread is past its last look at them)
    int count = 0;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const bool out = parent[c] == cur && c * 64 + lane <= last && token[c] >= 0;
      const uint64_t m = __ballot(out);
      if (out && wave == 0) s_out[count + __builtin_popcountll(m & ((1ull << lane) - 1))] = token[c];
      count += __builtin_popcountll(m);
    }
    __syncthreads();
    return count;
  };
  if (lane == 0) path[0] = 0;
  for (int i = next_child(0); i < n; i = next_child(i)) {
    double left[1];
    left_of(&s_p[i], &s_q[i], k, left);
    double r = left[0];
    const int word = s_token[i];
    if constexpr (!DRAWN) {
#pragma unroll
      for (int c = 0; c < CH; ++c)
        if (__any(parent[c] == cur && c * 64 + lane <= cut && token[c] == word)) r = 0.0;
    }
    if ((double)s_rand[i] * (double)s_q[i] * mass < r) {
      cur = i;
      k = 0;
      cut = i;
      mass = 1.0;
      others = -1.0;
      summed = false;
#pragma unroll
      for (int c = 0; c < CH; ++c)
        if (c * 64 + lane == len) path[c] = i;
      ++len;
      continue;
    }
    if constexpr (DRAWN) {
      __syncthreads();
      if (tid == 0) s_mass[k] = mass;
      __syncthreads();
      const double total = sum_left(cur, k + 1);
      summed = total > 0.0;
      if (summed) {
        mass = total;
        ++k;
      }
    } else {
      if (others < 0.0) {
        k = list_out(n - 1);
        others = sum_left(cur, k);
      }
      // And the words of the children behind, each once, but those of children before.
      bool counts[CH];
#pragma unroll
      for (int c = 0; c < CH; ++c) counts[c] = parent[c] == cur && c * 64 + lane > i && token[c] >= 0;
      for (int j = next_child(cur); j < n; j = next_child(j)) {
        const int word = s_token[j];
#pragma unroll
        for (int c = 0; c < CH; ++c) counts[c] &= c * 64 + lane <= j || token[c] != word;
      }
      double behind = 0.0;
      bool more = false;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        behind += counts[c] ? (double)s_p[c * 64 + lane] : 0.0;
        more |= __any(counts[c]);
      }
      double total = others;
      if (more) total += wave_total(behind);
      summed = total > 0.0 && !more;
      if (total > 0.0) {
        mass = total;
        cut = i;
      }
    }
  }
  double total = mass;
  if (!summed) {
    if constexpr (!DRAWN) k = list_out(cut);
    total = sum_left(cur, k);
  }

  // The draw: the first word at which the running sum passes its share of the whole.
  const double point = (double)s_rand[0] * total;
  int at = -1;  // the wave
  double below = 0.0;
  for (int w = 0; w < kWaves && at < 0; ++w) {
    if (below + s_sum[w] > point) at = w;
    else below += s_sum[w];
  }
  if (wave == 0) {
#pragma unroll
    for (int c = 0; c < CH; ++c)
      if (c * 64 + lane < (int)p.T) p.path[base + c * 64 + lane] = path[c];
    if (lane == 0) p.accepted[b] = len;
  }
  // Of the wave's stretch, the first word whose running sum from `below` passes the point,
  // or else (rounding) the last of which anything is left.
  auto search = [&](double below, double point) {
    int found = -1, some = -1;
#pragma unroll 1
    for (uint32_t step = 0; step < steps && found < 0; step += kBatch) {
      Batch y;
      load(cur, step, y);
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        __builtin_amdgcn_sched_barrier(0);
        if (found >= 0) continue;
        const uint32_t x = from + (step + i) * 256;
        double r[4];
        left4(y, i, x, k, r);
        const double four = (r[0] + r[1]) + (r[2] + r[3]);
        double upto = four;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
          const double y = __shfl_up(upto, d, 64);
          if (lane >= d) upto += y;
        }
        double run = below + (upto - four);
        int mine = -1;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          run += r[e];
          if (r[e] > 0.0) {
            some = (int)(x + e);
            if (mine < 0 && run > point) mine = (int)(x + e);
          }
        }
        const uint64_t who = __ballot(mine >= 0);
        if (who) found = __shfl(mine, __builtin_ctzll(who), 64);
        below += __shfl(upto, 63, 64);
      }
    }
    if (found >= 0) return found;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) some = max(some, __shfl_xor(some, d, 64));
    return some;
  };
  if (at >= 0) {
    if (wave == at) {
      const int word = search(below, point);
      if (lane == 0) p.next[b] = word;
    }
    return;
  }
  // Rounding, or nothing left anywhere (-1): the last word of which anything is.
  const int word = search(0.0, __builtin_inf());
  if (lane == 0) s_last[wave] = word;
  __syncthreads();
  if (tid == 0) {
    int last = -1;
    for (int w = 0; w < kWaves; ++w) last = max(last, s_last[w]);
    p.next[b] = last;
  }
}

}  // namespace

int launch_verify_draft(const VerifyDraft& p, uint32_t batch, hipStream_t stream) {
  const dim3 grid(batch), block(kThreads);
  if (p.T <= 64) {
    if (p.draft)
      hipLaunchKernelGGL((verify_kernel<true, 1>), grid, block, 0, stream, p);
    else
      hipLaunchKernelGGL((verify_kernel<false, 1>), grid, block, 0, stream, p);
  } else {
    if (p.draft)
      hipLaunchKernelGGL((verify_kernel<true, kMaxTreeNodes / 64>), grid, block, 0, stream, p);
    else
      hipLaunchKernelGGL((verify_kernel<false, kMaxTreeNodes / 64>), grid, block, 0, stream, p);
  }
  STS_HIP(hipGetLastError());
  return STS_OK;
}

}  // namespace sts
