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
// before.  Sums and comparisons are in f64, so that the verdict is that of exact
// arithmetic but where a random number lies within 2^-45 of a border.
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
typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));  // rows start anywhere

__device__ __forceinline__ double wave_total(double x) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) x += __shfl_xor(x, d, 64);
  return x;
}

template <bool DRAWN>
__global__ __launch_bounds__(kThreads) void verify_kernel(const VerifyDraft p) {
  __shared__ int32_t s_token[kMaxTreeNodes], s_parent[kMaxTreeNodes], s_path[kMaxTreeNodes];
  __shared__ float s_rand[kMaxTreeNodes], s_p[kMaxTreeNodes], s_q[kMaxTreeNodes];
  __shared__ double s_mass[kMaxTreeNodes];   // DRAWN: the masses that rejections divided by
  __shared__ int32_t s_cut[kMaxTreeNodes];   // else the tokens that are out
  __shared__ double s_sum[kWaves];
  __shared__ int32_t s_last[kWaves];

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t b = blockIdx.x, V = p.V;
  const uint64_t base = (uint64_t)b * p.T;
  const int count_at = p.counts ? p.counts[b] : (int)p.T;
  const int n = min(max(count_at, 0), (int)p.T);
  if (tid < (int)p.T) {
    int token = -1, parent = -1;
    float u = 0.f, at_p = 0.f, at_q = DRAWN ? 0.f : 1.f;
    if (tid < n) {
      token = p.tokens[base + tid];
      parent = p.parents[base + tid];
      u = p.rand[base + tid];
      parent = parent >= 0 && parent < tid ? parent : -1;
      token = (uint32_t)token < V ? token : -1;
      if (parent >= 0 && token >= 0) {
        at_p = p.target[(base + parent) * V + token];
        if constexpr (DRAWN) at_q = p.draft[(base + parent) * V + token];
      }
    }
    s_token[tid] = token;
    s_parent[tid] = tid > 0 ? parent : -1;
    s_rand[tid] = u;
    s_p[tid] = at_p > 0.f ? at_p : 0.f;
    s_q[tid] = at_q > 0.f ? at_q : 0.f;
  }
  __syncthreads();
  if (n == 0) {
    if (tid < (int)p.T) p.path[base + tid] = -1;
    if (tid == 0) {
      p.accepted[b] = 0;
      p.next[b] = -1;
    }
    return;
  }

  // Stretch of this wave: whole steps of 256 words.
  const uint32_t steps = ((V + 255) / 256 + kWaves - 1) / kWaves;
  const uint32_t from = wave * steps * 256;
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
  // What is left of word x after k rejections.
  auto left_of = [&](float at_p, float at_q, int k) {
    double r = at_p > 0.f ? (double)at_p : 0.0;
    if constexpr (DRAWN) {
      const double q = at_q > 0.f ? (double)at_q : 0.0;
      for (int j = 0; j < k; ++j) r = fmax((j ? r / s_mass[j] : r) - q, 0.0);
    }
    return r;
  };
  // What is left of words x .. x+3 at node `cur` after k rejections (else: without the k
  // tokens of s_cut).
  auto left4 = [&](int cur, int k, uint32_t x, double (&r)[4]) {
    const float* row = p.target + (base + cur) * V;
    const f4 a = word4(row, x);
    f4 z = {0.f, 0.f, 0.f, 0.f};
    if constexpr (DRAWN) {
      if (k > 0) z = word4(p.draft + (base + cur) * V, x);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) r[e] = left_of(a[e], z[e], k);
    if constexpr (!DRAWN) {
      for (int j = 0; j < k; ++j) {
        const uint32_t d = (uint32_t)s_cut[j] - x;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (d == (uint32_t)e) r[e] = 0.0;
      }
    }
  };
  // Its sum over all words, the waves' sums in s_sum and their last word with anything
  // left in s_last.
  auto sum_left = [&](int cur, int k) {
    double sum = 0.0;
    int last = -1;
    for (uint32_t i = 0; i < steps; ++i) {
      const uint32_t x = from + i * 256 + lane * 4;
      if (x >= V) break;
      double r[4];
      left4(cur, k, x, r);
      sum += (r[0] + r[1]) + (r[2] + r[3]);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (r[e] > 0.0) last = (int)(x + e);
    }
    sum = wave_total(sum);
#pragma unroll
    for (int d = 1; d < 64; d *= 2) last = max(last, __shfl_xor(last, d, 64));
    __syncthreads();
    if (lane == 0) {
      s_sum[wave] = sum;
      s_last[wave] = last;
    }
    __syncthreads();
    double total = 0.0;
    for (int w = 0; w < kWaves; ++w) total += s_sum[w];
    return total;
  };

  // The walk, the same on every thread: a node's children come after it, and once one is
  // kept its own come next.
  int cur = 0, k = 0, len = 1;
  double mass = 1.0;
  bool summed = false;  // s_sum holds the sums of r as it is
  if (tid == 0) s_path[0] = 0;
  for (int i = 1; i < n; ++i) {
    if (s_parent[i] != cur) continue;
    double r = left_of(s_p[i], s_q[i], k);
    if constexpr (!DRAWN) {
      for (int j = 0; j < k; ++j)
        if (s_cut[j] == s_token[i]) r = 0.0;
    }
    if ((double)s_rand[i] * (double)s_q[i] * mass < r) {
      cur = i;
      k = 0;
      mass = 1.0;
      summed = false;
      if (tid == 0) s_path[len] = i;
      ++len;
      continue;
    }
    // (Every thread is past its last look at these.)
    __syncthreads();
    if (tid == 0) {
      if (DRAWN) s_mass[k] = mass;
      else s_cut[k] = s_token[i];
    }
    __syncthreads();
    const double total = sum_left(cur, k + 1);
    summed = total > 0.0;
    if (summed) {
      mass = total;
      ++k;
    }
  }
  double total = mass;
  if (!summed) total = sum_left(cur, k);

  // The draw: the first word at which the running sum passes its share of the whole.
  const double point = (double)s_rand[0] * total;
  int at = -1;      // the wave
  double below = 0.0;
  int last = -1;
  for (int w = 0; w < kWaves; ++w) {
    last = max(last, s_last[w]);
    if (at < 0) {
      if (below + s_sum[w] > point) at = w;
      else below += s_sum[w];
    }
  }
  if (tid < (int)p.T) p.path[base + tid] = tid < len ? s_path[tid] : -1;
  if (tid == 0) {
    p.accepted[b] = len;
    if (at < 0) p.next[b] = last;  // (rounding, or nothing left anywhere: -1)
  }
  if (wave != at) return;
  int found = -1, some = -1;
  for (uint32_t i = 0; i < steps && found < 0; ++i) {
    const uint32_t x = from + i * 256 + lane * 4;
    double r[4] = {0.0, 0.0, 0.0, 0.0};
    if (x < V) left4(cur, k, x, r);
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
  if (found < 0) {  // (rounding: the stretch's last)
#pragma unroll
    for (int d = 1; d < 64; d *= 2) some = max(some, __shfl_xor(some, d, 64));
    found = some;
  }
  if (lane == 0) p.next[b] = found;
}

}  // namespace

int launch_verify_draft(const VerifyDraft& p, uint32_t batch, hipStream_t stream) {
  const dim3 grid(batch), block(kThreads);
  if (p.draft)
    hipLaunchKernelGGL((verify_kernel<true>), grid, block, 0, stream, p);
  else
    hipLaunchKernelGGL((verify_kernel<false>), grid, block, 0, stream, p);
  STS_HIP(hipGetLastError());
  return STS_OK;
}

}  // namespace sts
