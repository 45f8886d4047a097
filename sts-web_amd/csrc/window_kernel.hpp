// window_kernel.hpp -- attention of up to 64 query rows per K/V head over a
// ring window on the f32 matrix cores (gfx950): the kernel behind
// sts_tree_attention, sts_masked_attention and sts_decode_ring_weights.
//
// For query row i and window row r
//   x_ir = scale q_i.k_r, capped and biased where asked; -inf where r is not seen
//   out_i = sum_r 2^(x_ir log2 e - m_i) v_r / sum_r 2^(x_ir log2 e - m_i)
// with the running maximum m_i and the sum kept in f32 over one pass.
//
// A workgroup takes 16*R query rows of one (stream, K/V head) -- the nodes or
// queries times the heads of the group, so that a K/V row is read once for all
// of them -- and one split of the window.  Its four waves share the query rows
// and deal the split's 16-row tiles among themselves; nothing goes through LDS
// until the end:
//   S^T = K Q^T    A = K tile: lane (m, g) = (lane & 15, lane >> 4) holds row m,
//                  dims (4c + g)*CW + e; B = Q in the same dims.  The lane then
//                  has the scores of query m for rows 4g .. 4g+3
//   O^T += V^T P^T A = V^T: step i of 4 takes rows 4g + i, and the lane holds of
//                  row 4g + i the dims (16 tc + m)*VW + e; B = the scores'
//                  exponentials as they stand, register i
// Both tiles are 16-byte loads straight from the cache, and the exponentials
// never leave their registers.  The waves' (m, l, O) are merged through LDS, the
// splits' through records in the stream's workspace by the last to arrive.
#pragma once

#include <cfloat>

#include "coherent.hpp"
#include "common.hpp"
#include "lane.hpp"
#include "rope.hpp"
#include "window.hpp"

namespace sts {
namespace window {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kWaves = 4;
constexpr int kTile = 16;             // window rows a wave takes at once
constexpr int kMaxSplits = 64;
constexpr uint32_t kOutside = 0x80000000u;  // past every buffer resource: loads zeros

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// tanh to a few units in the last place relative to itself, also for small
// arguments: x P(x^2) below 0.6 (P fitted to tanh(x)/x at Chebyshev nodes, 9e-11),
// where 1 - 2/(e^2x + 1) would cancel; that form above.
__device__ __forceinline__ float tanh_rel(float x) {
  const float a = fabsf(x), z = x * x;
  float pz = 0.0022146995f;
  pz = fmaf(pz, z, -0.0082483031f);
  pz = fmaf(pz, z, 0.0217261855f);
  pz = fmaf(pz, z, -0.0539507493f);
  pz = fmaf(pz, z, 0.1333322972f);
  pz = fmaf(pz, z, -0.3333333135f);
  const float small = fmaf(x * z, pz, x);
  const float t = exp2_hw(a * (2.f * kLog2e));  // inf for large a: 2 / inf = 0
  const float big = copysignf(1.f - 2.f * __builtin_amdgcn_rcpf(t + 1.f), x);
  return a < 0.6f ? small : big;
}

__device__ __forceinline__ float wave_max(float x) {
  x = fmaxf(x, xchg<0>(x));
  x = fmaxf(x, xchg<1>(x));
  x = fmaxf(x, xchg<2>(x));
  x = fmaxf(x, xchg<3>(x));
  return max_xor32(max_xor16(x));
}

// W elements loaded at a byte offset of a cache head, as f32 (bf16 is widened).
template <bool BF, int W>
struct Piece {
  static constexpr int kWords = BF ? W / 2 : W;
  uint32_t w[kWords];
  __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t rs, uint32_t off) {
    if constexpr (kWords == 4) {
      const u32x4 x = __builtin_amdgcn_raw_buffer_load_b128(rs, off, 0, 0);
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = x[i];
    } else {
      static_assert(kWords == 2, "8 or 16 bytes a lane");
      const u32x2 x = __builtin_amdgcn_raw_buffer_load_b64(rs, off, 0, 0);
      w[0] = x[0];
      w[1] = x[1];
    }
  }
  __device__ __forceinline__ float operator[](int e) const {
    if constexpr (BF) {
      const uint32_t x = w[e >> 1];
      return __uint_as_float((e & 1) ? x & 0xffff0000u : x << 16);
    } else {
      return __uint_as_float(w[e]);
    }
  }
};

__device__ __forceinline__ bool not_finite(float x) {
  return (__float_as_uint(x) & 0x7f800000u) == 0x7f800000u;
}

template <int D, int R, bool BF, WindowMode MODE, bool PAD>
__global__ __launch_bounds__(kWaves * 64) void window_kernel(const WindowParams p) {
  constexpr int CW = BF ? 8 : 4;                    // dims of K a lane loads at once
  constexpr int NC = D / (4 * CW);                  // loads per K row tile
  constexpr int VW = CW < D / 16 ? CW : D / 16;     // dims of V a lane loads at once
  constexpr int NV = D / (16 * VW);                 // loads per V row
  constexpr int ES = BF ? 2 : 4;                    // bytes per element
  constexpr int ROWS = 16 * R;
  constexpr int LDO = D + 4;                        // LDS row of a partial output
  constexpr int C4 = D / 4;

  __shared__ __align__(16) float s_o[kWaves][16][LDO];
  __shared__ float s_ml[kWaves][ROWS][2];
  __shared__ uint32_t s_last;
  __shared__ uint32_t s_anc[MODE == kWindowTree ? kMaxTreeNodes : 1][kMaxTreeNodes / 32];
  __shared__ int s_jump[MODE == kWindowTree ? kMaxTreeNodes : 1];
  __shared__ int s_depth[MODE == kWindowTree ? kMaxTreeNodes : 1];

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int m16 = lane & 15, g = lane >> 4;
  const uint32_t split = blockIdx.x % p.nsplit, rb = blockIdx.x / p.nsplit;
  const uint32_t kvh = blockIdx.y, b = blockIdx.z;
  const uint32_t dh = PAD ? p.dh : (uint32_t)D;

  uint32_t len = p.len, start = p.start;
  if (p.lens) {
    const int32_t L = p.lens[b];
    len = L <= 0 ? 0u : min((uint32_t)L, p.M);
    const int32_t st = p.starts[b] % (int32_t)p.M;
    start = (uint32_t)(st < 0 ? st + (int32_t)p.M : st);
  }
  uint32_t n = min(p.T, len);
  if (p.counts) {
    const int32_t c = p.counts[b];
    n = c <= 0 ? 0u : min((uint32_t)c, n);
  }
  const uint32_t base = len - n;  // window row of query 0

  // Row rr of the block is query rr / group, head kvh*group + rr % group.
  const uint32_t row0 = rb * ROWS, nrows = n * p.group, all = p.T * p.group;
  auto out_row = [&](uint32_t rr) {
    return p.out + (((size_t)b * p.T + rr / p.group) * p.H + kvh * p.group + rr % p.group) * dh;
  };
  auto zero_rows = [&](uint32_t from, uint32_t to) {
    const uint32_t d4 = dh / 4;
    for (uint32_t t = tid; t < (to - from) * d4; t += kWaves * 64)
      *reinterpret_cast<float4*>(out_row(from + t / d4) + t % d4 * 4) = make_float4(0.f, 0.f, 0.f, 0.f);
  };
  const uint32_t end = min(row0 + ROWS, all);  // rows of out that this block owns
  const uint32_t live = min(max(nrows, row0), end);
  if (split == 0 && live < end) zero_rows(live, end);
  if (live == row0) return;

  // The rows that each query sees, and their union over the block.  Rows of the
  // block past the queries see everything, so that they never make a tile
  // partly seen; their results go nowhere.
  uint32_t lo[R], hi[R], ulo = 0, uhi = len;
  bool real[R];
  if constexpr (MODE == kWindowMasked) {
    ulo = len;
    uhi = 0;
  }
#pragma unroll
  for (int rt = 0; rt < R; ++rt) {
    const uint32_t rr = row0 + rt * 16 + m16;
    real[rt] = rr < nrows;
    lo[rt] = 0;
    hi[rt] = len;
    if constexpr (MODE == kWindowMasked) {
      if (real[rt]) {
        const uint32_t i = rr / p.group;
        const size_t at = (size_t)b * p.T + i;
        hi[rt] = base + i + 1;
        if (p.lo) lo[rt] = (uint32_t)max(p.lo[at], 0);
        if (p.hi) hi[rt] = min((uint32_t)max(p.hi[at], 0), len);
        if (lo[rt] < hi[rt]) {
          ulo = min(ulo, lo[rt]);
          uhi = max(uhi, hi[rt]);
        }
      }
    }
  }
  if constexpr (MODE == kWindowMasked) {
#pragma unroll
    for (int x = 1; x < 16; x *= 2) {  // the four lane groups hold the same rows
      ulo = min(ulo, (uint32_t)__shfl_xor((int)ulo, x, 64));
      uhi = max(uhi, (uint32_t)__shfl_xor((int)uhi, x, 64));
    }
    ulo = __builtin_amdgcn_readfirstlane(ulo);
    uhi = __builtin_amdgcn_readfirstlane(uhi);
    if (ulo >= uhi) {  // no query of the block sees anything
      if (split == 0) zero_rows(row0, live);
      return;
    }
  }

  // Tiles of 16 window rows, dealt to the splits and waves in turn; a split gets
  // at least a tile for each wave.
  const uint32_t t0 = ulo / kTile, t1 = (uhi + kTile - 1) / kTile;
  const uint32_t nsplit = min(p.nsplit, (t1 - t0 + kWaves - 1) / kWaves);
  if (split >= nsplit) return;

  const size_t head = ((size_t)b * p.KH + kvh) * p.M * dh * ES;
  const __amdgpu_buffer_rsrc_t krs = coherent_rsrc(static_cast<const char*>(p.k) + head, p.M * dh * ES);
  const __amdgpu_buffer_rsrc_t vrs = coherent_rsrc(static_cast<const char*>(p.v) + head, p.M * dh * ES);
  auto row_off = [&](uint32_t r) {
    uint32_t slot = start + r;
    slot = slot >= p.M ? slot - p.M : slot;
    return r < uhi ? slot * (dh * ES) : kOutside;
  };
  Piece<BF, CW> kk[NC];
  Piece<BF, VW> vv[4][NV];
  auto load_k = [&](uint32_t r0) {
    const uint32_t off = row_off(r0 + m16) + g * (CW * ES);
#pragma unroll
    for (int c = 0; c < NC; ++c)
      kk[c].load(krs, !PAD || (uint32_t)(c * 4 + g) * CW < dh ? off + c * (4 * CW * ES) : kOutside);
  };
  auto load_v = [&](uint32_t r0) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t off = row_off(r0 + 4 * g + i) + m16 * (VW * ES);
#pragma unroll
      for (int c = 0; c < NV; ++c)
        vv[i][c].load(vrs, !PAD || (uint32_t)(c * 16 + m16) * VW < dh ? off + c * (16 * VW * ES) : kOutside);
    }
  };
  const uint32_t tstep = nsplit * kWaves;
  uint32_t t = t0 + split + nsplit * wave;
  load_k(t * kTile);
  load_v(t * kTile);

  // The draft's relation "is above or is", a bit per node, and the nodes'
  // depths: each node takes over what its jump target knows and jumps twice as
  // far, log2 of the nodes' number times.
  if constexpr (MODE == kWindowTree) {
    const uint32_t words = (n + 31) / 32;
    if (tid < (int)n) {
      int up = p.parents[(size_t)b * p.T + tid];
      up = up < 0 || up >= tid ? -1 : up;
#pragma unroll
      for (int w = 0; w < (int)kMaxTreeNodes / 32; ++w) s_anc[tid][w] = 0;
      s_anc[tid][tid >> 5] = 1u << (tid & 31);
      s_jump[tid] = up;
      s_depth[tid] = up >= 0;
    }
    __syncthreads();
    for (uint32_t reach = 1; reach < n; reach *= 2) {
      const int to = tid < (int)n ? s_jump[tid] : -1;
      uint32_t above[kMaxTreeNodes / 32];
      int next = -1, deeper = 0;
      if (to >= 0) {
        for (uint32_t w = 0; w < kMaxTreeNodes / 32; ++w) above[w] = w < words ? s_anc[to][w] : 0;
        next = s_jump[to];
        deeper = s_depth[to];
      }
      __syncthreads();
      if (to >= 0) {
        for (uint32_t w = 0; w < kMaxTreeNodes / 32; ++w)
          if (w < words) s_anc[tid][w] |= above[w];
        s_jump[tid] = next;
        s_depth[tid] += deeper;
      }
      __syncthreads();
    }
  }

  // The query rows: rotated, scaled, in the matrix operand's layout.
  float qf[R][NC][CW];
  uint32_t node[R];
#pragma unroll
  for (int rt = 0; rt < R; ++rt) {
    const uint32_t rr = row0 + rt * 16 + m16;
    node[rt] = real[rt] ? rr / p.group : 0;
    const float* src = p.q + (((size_t)b * p.T + node[rt]) * p.H + kvh * p.group + rr % p.group) * dh;
    uint32_t pos = p.rope_pos;
    if constexpr (MODE == kWindowTree) pos += s_depth[node[rt]];
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int e = 0; e < CW; e += 4) {
        const uint32_t d = (c * 4 + g) * CW + e;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        if (real[rt] && (!PAD || d < dh)) {
          x = *reinterpret_cast<const float4*>(src + d);
          if (p.rope_cos) {
            const size_t ro = (size_t)pos * (dh / 2) + d / 2;
            x = rope4(x, *reinterpret_cast<const float2*>(p.rope_cos + ro),
                      *reinterpret_cast<const float2*>(p.rope_sin + ro));
          }
        }
        qf[rt][c][e] = x.x * p.qscale;
        qf[rt][c][e + 1] = x.y * p.qscale;
        qf[rt][c][e + 2] = x.z * p.qscale;
        qf[rt][c][e + 3] = x.w * p.qscale;
      }
  }
  float slope[R];
  if constexpr (MODE == kWindowMasked) {
#pragma unroll
    for (int rt = 0; rt < R; ++rt)
      slope[rt] = p.slopes && real[rt]
                      ? p.slopes[kvh * p.group + (row0 + rt * 16 + m16) % p.group] * kLog2e
                      : 0.f;
  }

  float m[R], l[R];
  f32x4 o[R][NV * VW];
#pragma unroll
  for (int rt = 0; rt < R; ++rt) {
    m[rt] = -FLT_MAX;
    l[rt] = 0.f;
#pragma unroll
    for (int x = 0; x < NV * VW; ++x) o[rt][x] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  for (; t < t1; t += tstep) {
    const uint32_t r0 = t * kTile;
    f32x4 s[R];
#pragma unroll
    for (int rt = 0; rt < R; ++rt) s[rt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int e = 0; e < CW; ++e)
#pragma unroll
        for (int rt = 0; rt < R; ++rt)
          s[rt] = __builtin_amdgcn_mfma_f32_16x16x4f32(kk[c][e], qf[rt][c][e], s[rt], 0, 0, 0);
    load_k((t + tstep) * kTile);

    // A tile that some query does not see, or that the window's end cuts.
    bool partly = false;
    if constexpr (MODE == kWindowMasked) {
#pragma unroll
      for (int rt = 0; rt < R; ++rt)
        partly |= real[rt] && (lo[rt] > r0 || hi[rt] < r0 + kTile);
      partly = __any(partly);
    } else {
      partly = r0 + kTile > (MODE == kWindowTree ? base : len);
    }
#pragma unroll
    for (int rt = 0; rt < R; ++rt) {
      if constexpr (MODE == kWindowMasked) {
        if (p.cap_log2 > 0.f) {
#pragma unroll
          for (int i = 0; i < 4; ++i) s[rt][i] = p.cap_log2 * tanh_rel(s[rt][i]);
        }
        if (p.slopes) {
          const int away = (int)(base + node[rt]) - (int)(r0 + 4 * g);
#pragma unroll
          for (int i = 0; i < 4; ++i) s[rt][i] -= slope[rt] * fabsf((float)(away - i));
        }
      }
      if constexpr (MODE == kWindowWeights) {
        if (real[rt]) {
          float* to = p.scores + ((size_t)b * p.H + kvh * p.group + row0 + rt * 16 + m16) * p.score_stride + r0 + 4 * g;
          *reinterpret_cast<f32x4*>(to) = s[rt];  // the stride covers whole tiles
        }
      }
      if (partly) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t r = r0 + 4 * g + i;
          bool seen = r >= lo[rt] && r < hi[rt];
          if constexpr (MODE == kWindowTree) {
            if (seen && r >= base && real[rt]) {
              const uint32_t j = r - base;
              seen = (s_anc[node[rt]][j >> 5] >> (j & 31)) & 1u;
            }
          }
          s[rt][i] = seen ? s[rt][i] : -INFINITY;
        }
      }
      float top = fmaxf(fmaxf(s[rt][0], s[rt][1]), fmaxf(s[rt][2], s[rt][3]));
      top = fmaxf(m[rt], max_xor32(max_xor16(top)));
      const float alpha = exp2_hw(m[rt] - top);
      m[rt] = top;
#pragma unroll
      for (int i = 0; i < 4; ++i) s[rt][i] = exp2_hw(s[rt][i] - top);
      l[rt] = l[rt] * alpha + ((s[rt][0] + s[rt][1]) + (s[rt][2] + s[rt][3]));
      if (__any(alpha != 1.f)) {
#pragma unroll
        for (int x = 0; x < NV * VW; ++x) o[rt][x] *= alpha;
      }
    }

    float vf[4][NV * VW];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int c = 0; c < NV; ++c)
#pragma unroll
        for (int e = 0; e < VW; ++e) vf[i][c * VW + e] = vv[i][c][e];
    // A value that is not finite, in a row that some query does not see: the
    // product would carry it to that query as 0 * inf.  It is taken out of the
    // operand and added by hand to the queries that see its row.
    if (partly) {
      bool bad = false;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int x = 0; x < NV * VW; ++x) {
          bad |= not_finite(vf[i][x]);
          vf[i][x] = not_finite(vf[i][x]) ? 0.f : vf[i][x];
        }
      if (__any(bad)) {
        for (int key = 0; key < kTile; ++key) {
          const uint32_t off = row_off(r0 + key);
          const int from = (key >> 2) * 16 + m16;
          float w[R];
#pragma unroll
          for (int rt = 0; rt < R; ++rt) {
            const float a = (key & 1) ? s[rt][1] : s[rt][0], z = (key & 1) ? s[rt][3] : s[rt][2];
            w[rt] = __shfl((key & 2) ? z : a, from, 64);
          }
#pragma unroll
          for (int c = 0; c < NV; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t d = (c * 16 + 4 * g + i) * VW;
              Piece<BF, VW> x;
              x.load(vrs, !PAD || d < dh ? off + d * ES : kOutside);
#pragma unroll
              for (int e = 0; e < VW; ++e)
#pragma unroll
                for (int rt = 0; rt < R; ++rt)
                  if (not_finite(x[e]) && !(w[rt] == 0.f)) o[rt][c * VW + e][i] += w[rt] * x[e];
            }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int x = 0; x < NV * VW; ++x)
#pragma unroll
        for (int rt = 0; rt < R; ++rt)
          o[rt][x] = __builtin_amdgcn_mfma_f32_16x16x4f32(vf[i][x], s[rt][i], o[rt][x], 0, 0, 0);
    load_v((t + tstep) * kTile);
  }

  // The waves' states merged through LDS, a row tile at a time.
#pragma unroll
  for (int rt = 0; rt < R; ++rt) {
    l[rt] = sum_xor32(sum_xor16(l[rt]));
    if (g == 0) {
      s_ml[wave][rt * 16 + m16][0] = m[rt];
      s_ml[wave][rt * 16 + m16][1] = l[rt];
    }
  }
  constexpr uint32_t REC = ROWS * (D + 2);  // floats of a split's record: O, then (m, l)
  const size_t unit = ((size_t)b * p.KH + kvh) * p.rblocks + rb;
  const __amdgpu_buffer_rsrc_t prs =
      coherent_rsrc(p.part + unit * p.nsplit * REC, nsplit > 1 ? p.nsplit * REC * 4 : 0);
  auto finish = [&](uint32_t row, int col, float4 a, float mt, float lt) {
    const uint32_t rr = row0 + row;
    if (rr >= nrows) return;
    const float f = lt > 0.f || lt != lt ? 1.f / lt : 0.f;  // a row that sees nothing: zeros
    if (!PAD || (uint32_t)col * 4 < dh)
      *reinterpret_cast<float4*>(out_row(rr) + col * 4) = make_float4(a.x * f, a.y * f, a.z * f, a.w * f);
    if (MODE == kWindowWeights && col == 0) {
      float* st = p.stats + ((size_t)b * p.H + kvh * p.group + rr) * 2;
      st[0] = mt;
      st[1] = lt;
    }
  };
#pragma unroll
  for (int rt = 0; rt < R; ++rt) {
    if (rt > 0) __syncthreads();
#pragma unroll
    for (int c = 0; c < NV; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < VW; ++e) s_o[wave][m16][(c * 16 + 4 * g + i) * VW + e] = o[rt][c * VW + e][i];
    __syncthreads();
    for (int x = tid; x < 16 * C4; x += kWaves * 64) {
      const int row = x / C4, col = x % C4;
      float mt = s_ml[0][rt * 16 + row][0];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) mt = fmaxf(mt, s_ml[w][rt * 16 + row][0]);
      float lt = 0.f;
      float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float f = exp2_hw(s_ml[w][rt * 16 + row][0] - mt);
        lt += f * s_ml[w][rt * 16 + row][1];
        const float4 y = *reinterpret_cast<const float4*>(&s_o[w][row][col * 4]);
        a.x += f * y.x;
        a.y += f * y.y;
        a.z += f * y.z;
        a.w += f * y.w;
      }
      if (nsplit == 1) {
        finish(rt * 16 + row, col, a, mt, lt);
      } else {
        const uint32_t rec = split * REC * 4;
        st_coherent4(prs, rec + ((rt * 16 + row) * D + col * 4) * 4, coh_f4{a.x, a.y, a.z, a.w});
        if (col == 0) {
          st_coherent(prs, rec + (ROWS * D + (rt * 16 + row) * 2) * 4, mt);
          st_coherent(prs, rec + (ROWS * D + (rt * 16 + row) * 2 + 1) * 4, lt);
        }
      }
    }
  }
  if (nsplit == 1) return;

  // Every thread's records are acknowledged before the workgroup takes its
  // arrival ticket; the last one merges the splits, always in their order.
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
  // Each split's factor 2^(m_s - m) and the rows' (m, l), in the LDS of the
  // partial outputs, which every thread is done with.
  float* s_f = &s_o[0][0][0];  // [split][ROWS]
  static_assert(kMaxSplits * ROWS <= kWaves * 16 * LDO, "the factors fit");
  if (tid < ROWS) {
    float mt = -FLT_MAX;
    for (uint32_t sp = 0; sp < nsplit; ++sp) {
      const float x = ld_coherent(prs, (sp * REC + ROWS * D + tid * 2) * 4);
      s_f[sp * ROWS + tid] = x;
      mt = fmaxf(mt, x);
    }
    float lt = 0.f;
    for (uint32_t sp = 0; sp < nsplit; ++sp) {
      const float f = exp2_hw(s_f[sp * ROWS + tid] - mt);
      s_f[sp * ROWS + tid] = f;
      lt += f * ld_coherent(prs, (sp * REC + ROWS * D + tid * 2 + 1) * 4);
    }
    s_ml[0][tid][0] = mt;
    s_ml[0][tid][1] = lt;
  }
  __syncthreads();
  for (int x = tid; x < ROWS * C4; x += kWaves * 64) {
    const int row = x / C4, col = x % C4;
    if (row0 + row >= nrows) break;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    for (uint32_t sp = 0; sp < nsplit; sp += 4) {
      coh_f4 y[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        y[k] = coh_f4{0.f, 0.f, 0.f, 0.f};
        if (sp + k < nsplit) y[k] = ld_coherent4(prs, ((sp + k) * REC + row * D + col * 4) * 4);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float f = sp + k < nsplit ? s_f[(sp + k) * ROWS + row] : 0.f;
        a.x += f * y[k].x;
        a.y += f * y[k].y;
        a.z += f * y[k].z;
        a.w += f * y[k].w;
      }
    }
    finish(row, col, a, s_ml[0][row][0], s_ml[0][row][1]);
  }
}

// The launch of one mode: the instances for the head dim and the K/V type.
template <WindowMode MODE, int R, bool BF>
void launch_rows(const WindowParams& p, dim3 grid, hipStream_t stream) {
  const dim3 block(kWaves * 64);
  if (p.dh == 128)
    hipLaunchKernelGGL((window_kernel<128, R, BF, MODE, false>), grid, block, 0, stream, p);
  else if (p.dh == 64)
    hipLaunchKernelGGL((window_kernel<64, R, BF, MODE, false>), grid, block, 0, stream, p);
  else if (p.dh > 64)
    hipLaunchKernelGGL((window_kernel<128, R, BF, MODE, true>), grid, block, 0, stream, p);
  else
    hipLaunchKernelGGL((window_kernel<64, R, BF, MODE, true>), grid, block, 0, stream, p);
}

template <WindowMode MODE>
int launch_mode(const WindowParams& p, int row_tiles, bool bf16, dim3 grid, hipStream_t stream) {
  if (row_tiles == 1)
    bf16 ? launch_rows<MODE, 1, true>(p, grid, stream) : launch_rows<MODE, 1, false>(p, grid, stream);
  else if (row_tiles == 2)
    bf16 ? launch_rows<MODE, 2, true>(p, grid, stream) : launch_rows<MODE, 2, false>(p, grid, stream);
  else
    bf16 ? launch_rows<MODE, 4, true>(p, grid, stream) : launch_rows<MODE, 4, false>(p, grid, stream);
  STS_HIP(hipGetLastError());
  return STS_OK;
}

}  // namespace window

// One translation unit each.
int launch_window_tree(const WindowParams& p, int row_tiles, bool bf16, dim3 grid, hipStream_t stream);
int launch_window_masked(const WindowParams& p, int row_tiles, bool bf16, dim3 grid, hipStream_t stream);
int launch_window_weights(const WindowParams& p, int row_tiles, bool bf16, dim3 grid, hipStream_t stream);

}  // namespace sts
