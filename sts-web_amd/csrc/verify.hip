// verify.hip -- the verdict on a draft (gfx950).  No counterpart in the reference, which
// samples one token a step (crates/sts-wasm/src/wgsl/shader_sample_topk.wgsl).
//
// Speculative sampling down a tree.  At a place (a kept node) let p be the target's
// probabilities there and q those that its children were drawn from; r = p and m = 1 at
// first.  Each child in turn, of token x:
//   kept      if u q(x) m < r(x): the walk goes on at the child
//   rejected  otherwise: r <- max(0, r / m - q), m <- sum r (unless that is zero)
// and where no child is kept a token is drawn from r / m.  The tokens are then distributed
// as the target's if each child was drawn from q independently of the others (with
// replacement).  Children taken without chance (no q) stand for q = 1 at their own
// token: r(x) <- 0 instead, m <- sum r.
//
// r is never stored: a word's r follows from p, q and the masses of the rejections
// before.  Without q, one sum over the words that are no child's token serves all of a
// place's rejections: the children's own are added to it.  Sums and comparisons are in
// f64, so that the verdict is that of exact arithmetic but where a random number lies
// within 2^-45 of a border (rows of up to 2^23 words, whose running sum and total pass
// through 180 roundings at most; 2^-41 up to 2^28 words, 3200).  With q a place's second and later
// rejections each make that distance up to 4 / m times as large: the errors of r and of m
// before, relative to what was left, come to twice themselves and a rounding in r / m,
// and are then relative to the smaller m that max(0, r / m - q) leaves.
//
// One workgroup a stream.  The numbers at the drafted tokens are read once, all
// together; whole rows only where something is rejected and for the last draw, each wave
// a stretch of the words, so that the draw finds its wave from sixteen sums.  What bounds
// it is the latency of these steps, not the bytes.
#include "coherent.hpp"
#include "common.hpp"
#include "lane.hpp"
#include "verify.hpp"
#include "window.hpp"

namespace sts {

namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kBatch = 8;
constexpr uint32_t kOutside = 0x80000000u;  // past every row: loads zeros
typedef float f4 __attribute__((ext_vector_type(4)));

constexpr int kPieces = 64;  // sums that a wave keeps of its stretch of the words

// The value of the lane whose index differs in bit LEVEL (and, for 2 and 3, in the bits
// below).
template <int LEVEL>
__device__ __forceinline__ double xchg64(double x) {
  const uint2 y = __builtin_bit_cast(uint2, x);
  float lo = __uint_as_float(y.x), hi = __uint_as_float(y.y);
  if constexpr (LEVEL == 5) {
    lo = xor32(lo);
    hi = xor32(hi);
  } else {
    lo = xchg<LEVEL>(lo);
    hi = xchg<LEVEL>(hi);
  }
  return __builtin_bit_cast(double, make_uint2(__float_as_uint(lo), __float_as_uint(hi)));
}
template <int LEVELS = 6>
__device__ __forceinline__ double lanes_total(double x) {
  if constexpr (LEVELS > 0) {
    x += xchg64<LEVELS - 1>(x);
    return lanes_total<LEVELS - 1>(x);
  }
  return x;
}
// kBatch values summed over the lanes: the lane ends with value lane / 8.
template <int N = kBatch, int LEVEL = 5>
__device__ __forceinline__ double batch_totals(double* x, int lane) {
  if constexpr (N > 1) {
    const bool up = (lane >> LEVEL) & 1;
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const double keep = up ? x[i + N / 2] : x[i], give = up ? x[i] : x[i + N / 2];
      x[i] = keep + xchg64<LEVEL>(give);
    }
    return batch_totals<N / 2, LEVEL - 1>(x, lane);
  }
  return lanes_total<LEVEL + 1>(x[0]);
}
static_assert(kBatch == 8, "eight values leave three levels of single ones");

// CH: 64 nodes each.
template <bool DRAWN, int CH>
__global__ __launch_bounds__(kThreads) void verify_kernel(const VerifyDraft p) {
  // What the first wave asks the others for: the place, the words out, whether to sum, whether
  // to draw then; and the mass of r, where it has that.
  __shared__ int32_t s_ask[4];
  __shared__ double s_mass_of;
  __shared__ float s_rand[CH * 64], s_p[CH * 64], s_q[DRAWN ? CH * 64 : 1];
  // The masses that a place's second and later rejections divide by, and 1 / them.  Every wave
  // writes the same; an entry changes only behind a barrier of the place's first sum.
  __shared__ double s_mass[DRAWN ? CH * 64 : 1][2];
  __shared__ int32_t s_out[DRAWN ? 1 : CH * 64];  // the words that a sum leaves out
  __shared__ double s_sum[2][kWaves];             // the waves' sums of r, by turns
  __shared__ double s_piece[kWaves][kPieces];     // and those of their pieces
  __shared__ int32_t s_last[kWaves];
  __shared__ int32_t s_path[CH * 64];  // the kept nodes (a barrier of the sum behind the last is before they are read)

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t b = blockIdx.x, V = p.V;
  const uint64_t base = (uint64_t)b * p.T;
  int count = (int)p.T;
  if (p.counts) count = p.counts[b];
  // A wave that walks keeps the nodes in its lanes, node c*64 + lane in element c; the numbers
  // at their tokens are the first wave's to fetch.
  const bool walks = DRAWN || wave == 0;
  int token[CH], parent[CH];
  bool fresh[CH];  // without draft: no earlier child of the place has the word
  float u[CH];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int i = c * 64 + lane;
    token[c] = parent[c] = -1;
    u[c] = 0.f;
    if (walks && i < (int)p.T) {
      parent[c] = p.parents[base + i];
      if (wave == 0) {
        token[c] = p.tokens[base + i];
        u[c] = p.rand[base + i];
      }
    }
  }
  const int n = min(max(count, 0), (int)p.T);
  if (n == 0) {
    if (tid < (int)p.T) p.path[base + tid] = -1;
    if (tid == 0) {
      p.accepted[b] = 0;
      p.next[b] = -1;
    }
    return;
  }
  if (walks) {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int i = c * 64 + lane;
      if (i >= n || parent[c] >= i || parent[c] < 0) parent[c] = -1;
    }
    if (tid == 0) s_path[0] = 0;
    if (wave == 0) {
      float at_p[CH], at_q[CH];
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        at_p[c] = at_q[c] = 0.f;
        if ((uint32_t)token[c] >= V) token[c] = -1;
        if (parent[c] >= 0 && token[c] >= 0) {
          at_p[c] = p.target[(base + parent[c]) * V + token[c]];
          if constexpr (DRAWN) at_q[c] = p.draft[(base + parent[c]) * V + token[c]];
        }
      }
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        s_rand[c * 64 + lane] = u[c];
        s_p[c * 64 + lane] = fmaxf(at_p[c], 0.f);  // (of NaN, too)
        if constexpr (DRAWN) s_q[c * 64 + lane] = fmaxf(at_q[c], 0.f);
      }
    }
    if constexpr (DRAWN) {
      __syncthreads();
    } else {
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
  }

  // The wave's stretch of the words: steps of 256, in at most kPieces pieces of `rounds`.
  const uint32_t steps = ((V + 255) / 256 + kWaves - 1) / kWaves;
  const uint32_t rounds = (steps + kPieces - 1) / kPieces;  // a piece's steps
  const uint32_t from = wave * steps * 256 + lane * 4;
  // The words of steps step, step + stride, ... (kBatch of them) of place cur, requested
  // together.
  struct Batch {
    f4 p[kBatch], q[DRAWN ? kBatch : 1];
  };
  // (Buffer loads: words past the row's end are zeros, without a branch.)
  auto row_of = [&](const float* x, int cur) { return coherent_rsrc(x + (base + cur) * V, V * 4); };
  auto word4 = [&](__amdgpu_buffer_rsrc_t row, uint32_t step) {
    return __builtin_bit_cast(f4, __builtin_amdgcn_raw_buffer_load_b128(
                                      row, step < steps ? (from + step * 256) * 4 : kOutside, 0, 0));
  };
  auto load = [&](auto many, int cur, uint32_t step, uint32_t stride, Batch& x) {
    const __amdgpu_buffer_rsrc_t target = row_of(p.target, cur);
#pragma unroll
    for (int i = 0; i < kBatch; ++i) x.p[i] = word4(target, step + i * stride);
    if constexpr (DRAWN && decltype(many)::value > 0) {
      const __amdgpu_buffer_rsrc_t draft = row_of(p.draft, cur);
#pragma unroll
      for (int i = 0; i < kBatch; ++i) x.q[i] = word4(draft, step + i * stride);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  // Takes the k words of s_out out of a batch (without draft).
  auto take_out = [&](uint32_t step, uint32_t stride, int k, Batch& x) {
    uint32_t out = 0;  // bit 4 i + e: word e of the lane's four of step i
    for (int j = 0; j < k; ++j) {
      const uint32_t rel = __builtin_amdgcn_readfirstlane((uint32_t)s_out[j] - wave * steps * 256);
      if (rel >= steps * 256) continue;  // another wave's
#pragma unroll
      for (int i = 0; i < kBatch; ++i)
        if (rel >> 8 == step + i * stride && (rel & 255) >> 2 == (uint32_t)lane) out |= 1u << (4 * i + (rel & 3));
    }
    if (__any(out)) {
#pragma unroll
      for (int i = 0; i < kBatch; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) x.p[i][e] = out >> (4 * i + e) & 1 ? 0.f : x.p[i][e];
    }
  };
  // What is left of a word after k rejections.  max(p, q) - q is max(0, p - q), exactly;
  // a quotient is the product with the inverse and one correction, which rounds it right.
  auto left_of = [&](float at_p, float at_q, int k) {
    const float p0 = fmaxf(at_p, 0.f);  // (of NaN, too)
    if constexpr (!DRAWN) return (double)p0;
    if (k == 0) return (double)p0;
    const float q0 = fmaxf(at_q, 0.f);
    const double q = (double)q0;
    double r = (double)fmaxf(p0, q0) - q;
#pragma unroll 1
    for (int j = 1; j < k; ++j) {
      const double m = s_mass[j][0], by = s_mass[j][1];
      const double t = r * by, d = fma(fma(-t, m, r), by, t) - q;
      r = d > 0.0 ? d : 0.0;
    }
    return r;
  };
  // Words of step i of a batch, after no rejection (MANY 0), one (1) or k of them (2).
  auto left4 = [&](auto many, const Batch& y, int i, int k, double (&r)[4]) {
    constexpr int MANY = decltype(many)::value;
    if constexpr (DRAWN && MANY > 0) {
      float q0[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        q0[e] = MANY == 1 || k > 0 ? fmaxf(y.q[i][e], 0.f) : 0.f;
        r[e] = (double)fmaxf(fmaxf(y.p[i][e], 0.f), q0[e]) - (double)q0[e];
      }
      if constexpr (MANY > 1) {
        // (left_of's loop over the rejections outside.)
#pragma unroll 1
        for (int j = 1; j < k; ++j) {
          const double m = s_mass[j][0], by = s_mass[j][1];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const double t = r[e] * by, d = fma(fma(-t, m, r[e]), by, t) - (double)q0[e];
            r[e] = d > 0.0 ? d : 0.0;
          }
        }
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) r[e] = (double)fmaxf(y.p[i][e], 0.f);
    }
  };
  // Its sum over all words; the waves' sums in s_sum[turn], and of their pieces in s_piece.
  int turn = 0;
  auto sum_left = [&](int cur, int k) {
    double sum = 0.0;
    auto words = [&](auto many) {
#pragma unroll 1
      for (uint32_t piece = 0; piece * rounds < steps; piece += kBatch) {
        double part[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) part[i] = 0.0;
#pragma unroll 1
        for (uint32_t round = 0; round < rounds; ++round) {
          Batch y;
          load(many, cur, piece * rounds + round, rounds, y);
          if constexpr (!DRAWN) take_out(piece * rounds + round, rounds, k, y);
#pragma unroll
          for (int i = 0; i < kBatch; ++i) {
            double r[4];
            left4(many, y, i, k, r);
            part[i] += (r[0] + r[1]) + (r[2] + r[3]);
            __builtin_amdgcn_sched_barrier(0);  // (registers)
          }
        }
        const double mine = batch_totals(part, lane);
        if ((lane & 7) == 0) s_piece[wave][piece + lane / 8] = mine;
        sum += (lane & 7) == 0 ? mine : 0.0;
      }
    };
    // (Loops of their own: one for all costs the place without rejections a microsecond, and
    // branches inside it the registers.)
    if (!DRAWN || k == 0) words(std::integral_constant<int, 0>{});
    else if (k == 1) words(std::integral_constant<int, 1>{});
    else words(std::integral_constant<int, 2>{});
    sum = lanes_total(sum);
    turn ^= 1;
    if (lane == 0) s_sum[turn][wave] = sum;
    __syncthreads();
    double total = 0.0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) total += s_sum[turn][w];
    return total;
  };

  // The walk: a node's children come after it, and once one is kept its own come next.
  // Without draft the first wave walks and the others wait for rows to sum: 64 streams' trees
  // with two places of rejections 13.9 us, 16.5 where every wave walks, for whose instructions
  // the four waves of a SIMD wait in turn.  With draft each rejection needs a sum, and telling
  // the others costs what it saves (20.7 and 19.9 us for three).
  int cur = 0, k = 0, len = 1;
  double mass = 1.0;
  bool summed = false;  // s_sum holds the sums of r as it is
  // Without draft: the sum over the words that are no child's, once there is one (else
  // -1); the words out are those of the children up to node `cut`.
  double others = -1.0;
  int cut = 0;
  // Node i's element of x.
  auto of_node = [&](const int (&x)[CH], int i) {
    int y = __builtin_amdgcn_readlane(x[0], i & 63);
#pragma unroll
    for (int c = 1; c < CH; ++c)
      if (i >> 6 == c) y = __builtin_amdgcn_readlane(x[c], i & 63);
    return y;
  };
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
    int count = 0;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const bool out = parent[c] == cur && c * 64 + lane <= last && token[c] >= 0;
      const uint64_t m = __ballot(out);
      if (out) s_out[count + __builtin_popcountll(m & ((1ull << lane) - 1))] = token[c];
      count += __builtin_popcountll(m);
    }
    return count;
  };
  // Without draft: child i is rejected, and no words but the children's have anything left: what
  // is left are the words of the children past `cut`, each counted where it comes first.  Where
  // only the child's own has, it stays, with the mass as it was, and the cut, which would take
  // it out, goes no further.
  auto reject = [&](int i) {
    const int word = of_node(token, i);
    double rest = 0.0;
    bool before = false;  // a word that stayed
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int at = c * 64 + lane;
      const double x = fresh[c] && at > cut && token[c] != word ? (double)s_p[at] : 0.0;
      rest += x;
      before |= __any(x > 0.0 && at < i);
    }
    rest = lanes_total(rest);
    if (rest > 0.0) {
      mass = rest;
      if (!before) cut = i;
    }
  };
  auto keep = [&](int i) {
    cur = i;
    k = 0;
    cut = i;
    mass = 1.0;
    others = -1.0;
    summed = false;
    if (tid == 0) s_path[len] = i;
    ++len;
  };
  // Without draft: all the children behind i at once, `others` known and more than nothing.
  // The mass that a child divides by is that of the words which no child before it has: the
  // others and, summed from the last child on, its own and those behind.  Returns the child
  // that is kept, or n.
  auto decide = [&](int i) {
    double behind = 0.0;
    int found = n;
#pragma unroll
    for (int c = CH - 1; c >= 0; --c) {
      const int at = 63 - lane;  // the lanes in reverse
      const bool on = __ballot(fresh[c] && c * 64 + lane > i) >> at & 1;
      const double p_at = on ? (double)s_p[c * 64 + at] : 0.0, upto = behind + lanes_upto(p_at);
      const uint64_t kept = __ballot(on && (double)s_rand[c * 64 + at] * (others + upto) < p_at);
      if (kept) found = c * 64 + __builtin_clzll(kept);
      behind = __shfl(upto, 63, 64);
    }
    return found;
  };
  int i = 0;          // the last node looked at
  bool asked = false; // for a sum that i's rejection needs
  double total = 0.0; // of the last row summed
  for (;;) {
    if (walks) {
      if (asked) {
        if constexpr (DRAWN) {
          summed = total > 0.0;
          if (summed) {
            mass = total;
            ++k;
          }
        } else {
          others = total;
          if (others > 0.0) {
            i = decide(i);
            if (i < n) {
              keep(i);
            } else {
              mass = others;
              summed = true;
            }
          } else {
            reject(i);
          }
        }
        asked = false;
      }
      while (!asked && (i = next_child(i)) < n) {
        const double p_at = (double)s_p[i];
        double r = p_at, q_at = 1.0;
        if constexpr (DRAWN) {
          q_at = (double)s_q[i];
          r = left_of(s_p[i], s_q[i], k);
        } else {
          const int word = of_node(token, i);
#pragma unroll
          for (int c = 0; c < CH; ++c)
            if (__any(parent[c] == cur && c * 64 + lane <= cut && token[c] == word)) r = 0.0;
        }
        if ((double)s_rand[i] * q_at * mass < r) {
          keep(i);
        } else if constexpr (DRAWN) {
          if (k > 0 && lane < 2) s_mass[k][lane] = lane ? 1.0 / mass : mass;
          __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
          __builtin_amdgcn_wave_barrier();
          __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
          asked = true;
        } else if (others < 0.0) {
#pragma unroll
          for (int c = 0; c < CH; ++c) fresh[c] = parent[c] == cur && token[c] >= 0;
          for (int j = next_child(cur); j < n; j = next_child(j)) {
            const int word = of_node(token, j);
#pragma unroll
            for (int c = 0; c < CH; ++c) fresh[c] &= c * 64 + lane <= j || token[c] != word;
          }
          k = list_out(n - 1);
          asked = true;
        } else {
          reject(i);
        }
      }
      if (!DRAWN && !asked && !summed) k = list_out(cut);
      if (!DRAWN && lane == 0) {
        s_ask[0] = cur;
        s_ask[1] = k;
        s_ask[2] = asked || !summed;
        s_ask[3] = !asked;
        s_mass_of = mass;
      }
    }
    bool sums = asked || !summed, last = !asked;
    if constexpr (!DRAWN) {
      __syncthreads();
      cur = __builtin_amdgcn_readfirstlane(s_ask[0]);
      k = __builtin_amdgcn_readfirstlane(s_ask[1]);
      sums = __builtin_amdgcn_readfirstlane(s_ask[2]);
      last = __builtin_amdgcn_readfirstlane(s_ask[3]);
      mass = s_mass_of;
    }
    total = sums ? sum_left(cur, DRAWN && asked ? k + 1 : k) : mass;
    if (last) break;
  }

  // The draw: the first word at which the running sum passes its share of the whole.  The
  // wave, then its piece, then the word; where rounding leaves none, the last with anything
  // left.
  const double point = (double)s_rand[0] * total;
  if (wave == 0) {
#pragma unroll
    for (int c = 0; c < CH; ++c)
      if (c * 64 + lane < (int)p.T) p.path[base + c * 64 + lane] = c * 64 + lane < len ? s_path[c * 64 + lane] : -1;
    if (lane == 0) p.accepted[b] = len;
  }
  int at = -1;
  double below = 0.0;
  for (int w = 0; w < kWaves && at < 0; ++w) {
    const double sum = s_sum[turn][w];
    if (below + sum > point) at = w;
    else below += sum;
  }
  // Running sums over the lanes, from `below` on.
  auto running = [&](double x) { return below + lanes_upto(x); };
  // The first word of piece `piece` of this wave whose running sum passes `point`, or -1;
  // `some`: the last with anything left.
  int some = -1;
  auto search = [&](uint32_t piece, double point) {
    int found = -1;
#pragma unroll 1
    for (uint32_t step = piece * rounds; step < min((piece + 1) * rounds, steps) && found < 0; ++step) {
      Batch y;
      const uint32_t x = from + step * 256;
      y.p[0] = word4(row_of(p.target, cur), step);
      if constexpr (DRAWN) y.q[0] = word4(row_of(p.draft, cur), step);
      if constexpr (!DRAWN) {
#pragma unroll
        for (int i = 1; i < kBatch; ++i) y.p[i] = f4{0.f, 0.f, 0.f, 0.f};
        take_out(step, 1, k, y);
      }
      double r[4];
      left4(std::integral_constant<int, 2>{}, y, 0, k, r);
      const double four = (r[0] + r[1]) + (r[2] + r[3]), upto = running(four);
      double run = upto - four;
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
      below = __shfl(upto, 63, 64);
    }
    return found;
  };
  if (at >= 0) {
    if (wave != at) return;
    const uint32_t pieces = (steps + rounds - 1) / rounds;
    const double mine = (uint32_t)lane < pieces ? s_piece[wave][lane] : 0.0, upto = running(mine);
    const uint64_t who = __ballot((uint32_t)lane < pieces && mine > 0.0 && upto > point);
    // (Rounding: the last piece with anything left.)
    const uint64_t any = __ballot((uint32_t)lane < pieces && mine > 0.0);
    const int piece = who ? __builtin_ctzll(who) : 63 - __builtin_clzll(any);
    below = __shfl(upto - mine, piece, 64);
    int word = search(piece, point);
    if (word < 0) {
#pragma unroll
      for (int d = 1; d < 64; d *= 2) some = max(some, __shfl_xor(some, d, 64));
      word = some;
    }
    if (lane == 0) p.next[b] = word;
    return;
  }
  // Nothing passes the point: the last word of all with anything left, -1 if there is none.
  for (uint32_t piece = 0; piece * rounds < steps; ++piece) search(piece, __builtin_inf());
#pragma unroll
  for (int d = 1; d < 64; d *= 2) some = max(some, __shfl_xor(some, d, 64));
  if (lane == 0) s_last[wave] = some;
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
