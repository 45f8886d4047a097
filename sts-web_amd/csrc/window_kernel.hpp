// window_kernel.hpp -- attention of up to 32 query rows per K/V head over a
// ring window on the matrix cores (gfx950): the kernel behind
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
// and deal the split's tiles among themselves:
//   S^T = K Q^T    A = K tile: lane (m, g) = (lane & 15, lane >> 4) holds row m,
//                  dims (4c + g)*CW + e; B = Q in the same dims.  The lane then
//                  has the scores of query m for rows 4g .. 4g+3
//   O^T += V^T P^T A = V^T: the lane holds of rows 4g + i the dims
//                  (16 tc + m)*VW + e; B = the scores' exponentials as they stand
// Both tiles are 16-byte loads straight from the cache, and the exponentials
// never leave their registers; in LDS stand the queries' operands and, at the end,
// the waves' (m, l, O), which are merged there.  The splits are merged through
// records in the stream's workspace by the last to arrive.
//
// One row tile (R = 1) over f32 rows multiplies in f32 (16x16x4): its 64 products of
// a 16 KB tile take a quarter of the time that HBM takes to deliver it.  Two (R = 2),
// or bf16 rows, would be bound by those products and multiply bf16 parts instead
// (16x16x32): an f32 value is the exact sum of three, so that f32 rows take six
// products for one (those of parts below 2^-26 of the whole are left out), and bf16
// rows, as they are against the parts of Q and of the weights, three.  Parts have
// f32's exponents: every element is held to f32's grade by itself, whatever stands in
// its row, tile or channel.  (Two f16 parts of each value under a common scale take
// half the products, but hold small elements only relative to the largest; 24 drafts
// of 40 nodes took 174 us with them.)  At 1000 queries of 32 heads over 2600 bf16 rows
// of 8 K/V heads that is 110 us against 488 in f32; at 24 drafts of 40 nodes over f32
// rows 203 against 513.
#pragma once

#include <cfloat>

#include "coherent.hpp"
#include "common.hpp"
#include "lane.hpp"
#include "rope.hpp"
#include "score.hpp"
#include "window.hpp"

namespace sts {
namespace window {

constexpr int kWaves = 4;
constexpr uint32_t kXcds = 8;
constexpr int kNt = 2;                // cache policy: nontemporal
// Splits of a block of 16 * row_tiles query rows at most: the merge holds two
// numbers for each split and row in LDS.
constexpr int max_splits(int row_tiles) { return 128 / row_tiles; }
constexpr uint32_t kOutside = 0x80000000u;  // past every buffer resource: loads zeros

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// W elements loaded at a byte offset of a cache head, as f32 (bf16 is widened).
// AUX: the cache policy of the load.
template <bool BF, int W, int AUX>
struct Piece {
  static constexpr int kWords = BF ? W / 2 : W;
  uint32_t w[kWords];
  __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t rs, uint32_t off) {
    if constexpr (kWords == 4) {
      const u32x4 x = __builtin_amdgcn_raw_buffer_load_b128(rs, off, 0, AUX);
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = x[i];
    } else {
      static_assert(kWords == 2, "8 or 16 bytes a lane");
      const u32x2 x = __builtin_amdgcn_raw_buffer_load_b64(rs, off, 0, AUX);
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

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// x[8] as matrix operands: three bf16 values each, the nearest to what is left, whose
// sum is x exactly (24 bits; bf16 has f32's exponents, and subnormals from 2^-133 on).
// x is finite and at most kMostParts in magnitude, above which the first would be rounded
// to infinity.
constexpr int kParts = 3;
constexpr float kMostParts = 0x1.FEp127f;
__device__ __forceinline__ void split_parts(const float* x, bf16x8 (&y)[kParts]) {
  typedef __bf16 b2 __attribute__((ext_vector_type(2)));
  typedef float f2 __attribute__((ext_vector_type(2)));
  u32x4 w[kParts];  // pairs put together as words: no half moves on its own
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    float a = x[e], z = x[e + 1];
#pragma unroll
    for (int n = 0; n < kParts; ++n) {
      w[n][e / 2] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f2){a, z}, b2));
      a -= __uint_as_float(w[n][e / 2] << 16);
      z -= __uint_as_float(w[n][e / 2] & 0xffff0000u);
    }
  }
#pragma unroll
  for (int n = 0; n < kParts; ++n) y[n] = __builtin_bit_cast(bf16x8, w[n]);
}

__device__ __forceinline__ f32x4 multiply(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// The lane's number, found anew: kept through the loops it, and what is derived from
// it, would cost registers that the tiles need.
__device__ __forceinline__ int fresh_lane() {
  int x = (int)__builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u));
  asm volatile("" : "+v"(x));
  return x;
}

template <int D, int R, bool BF, WindowMode MODE, bool PAD>
__global__ __launch_bounds__(kWaves * 64, 2) void window_kernel(const WindowParams p) {
  constexpr int CW = BF ? 8 : 4;                    // dims of K a lane loads at once
  constexpr int NC = D / (4 * CW);                  // loads per K row tile
  constexpr int VW = CW < D / 16 ? CW : D / 16;     // dims of V a lane loads at once
  constexpr int NV = D / (16 * VW);                 // loads per V row
  constexpr int ES = BF ? 2 : 4;                    // bytes per element
  constexpr bool PARTS = R > 1 || BF;               // products of parts
  constexpr int KT = PARTS ? 2 : 1;                 // 16-row tiles a wave takes at once
  constexpr int TILE = 16 * KT;
  constexpr int NP = NC * CW / 8;                   // 32-dim steps of K Q^T in parts
  constexpr int NX = NV * VW;                       // 16-dim tiles of the output
  constexpr int ROWS = 16 * R;
  constexpr int LDO = D + 4;                        // LDS row of a partial output
  constexpr int C4 = D / 4;

  // The queries' parts while the tiles are read, partial outputs after that.
  typedef bf16x8 Frag;
  constexpr int kPartBytes = PARTS ? R * NP * kParts * 64 * 16 : 0;
  constexpr int kOutBytes = kWaves * ROWS * LDO * 4;
  __shared__ __align__(16) char s_mem[kPartBytes > kOutBytes ? kPartBytes : kOutBytes];
  auto& s_q = *reinterpret_cast<Frag(*)[PARTS ? R : 1][NP][kParts][64]>(s_mem);
  auto& s_o = *reinterpret_cast<float(*)[kWaves][ROWS][LDO]>(s_mem);
  struct Row {
    uint32_t lo, hi;
    int at;       // window row of the query
    float slope;  // in units of log2(e)
  };
  __shared__ Row s_row[MODE == kWindowMasked ? ROWS : 1];
  __shared__ float s_ml[kWaves][ROWS][2];
  __shared__ uint32_t s_last;
  __shared__ uint32_t s_anc[MODE == kWindowTree ? kMaxTreeNodes : 1][kMaxTreeNodes / 32];
  __shared__ int s_jump[MODE == kWindowTree ? kMaxTreeNodes : 1];
  __shared__ int s_depth[MODE == kWindowTree ? kMaxTreeNodes : 1];

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int m16 = lane & 15, g = lane >> 4;
  // Workgroups go round the XCDs: the row blocks of one (stream, K/V head, split),
  // which read the same rows, take turns on one of them, next to one another, so that
  // its L2 serves all but the first.
  const uint32_t turn = blockIdx.x / kXcds, rb = turn % p.rblocks;
  const uint32_t share = turn / p.rblocks * kXcds + blockIdx.x % kXcds;
  uint32_t b, kvh, split, splits;
  uint32_t first;  // splits of the streams before, each counted once for all heads
  int32_t len_at = (int32_t)p.len, start_at = (int32_t)p.start, count_at = (int32_t)p.T;  // the stream's
  if (p.rows_factor > 0.f) {
    // Windows of different lengths are cut into splits of about the same length:
    // lane x looks at stream x, and the share's stream is the last whose streams
    // before take no more shares.
    uint32_t rows = 0;
    if (lane < (int)p.batch) {
      if (p.lens) {
        len_at = p.lens[lane];
        start_at = p.starts[lane];
      }
      if (p.counts) count_at = p.counts[lane];
      rows = (uint32_t)min(max(len_at, 0), (int32_t)p.M);
      if constexpr (MODE == kWindowMasked) {  // (one query a stream: the rows that it sees)
        const uint32_t hi = p.hi ? min((uint32_t)max(p.hi[lane], 0), rows) : rows;
        const uint32_t lo = p.lo ? (uint32_t)max(p.lo[lane], 0) : 0;
        rows = lo < hi ? hi - lo : 0;
      }
    }
    uint32_t total = rows;
#pragma unroll
    for (int x = 1; x < 64; x *= 2) total += (uint32_t)__shfl_xor((int)total, x, 64);
    const uint32_t chunk = max((uint32_t)((float)total * p.rows_factor) + 1, (uint32_t)(kWaves * TILE));
    const uint32_t mine = lane < (int)p.batch ? min(max((rows + chunk - 1) / chunk, 1u), p.nsplit) : 0;
    uint32_t before = mine;
#pragma unroll
    for (int x = 1; x < 64; x *= 2) {
      const uint32_t y = (uint32_t)__shfl_up((int)before, x, 64);
      before += lane >= x ? y : 0;
    }
    if (share >= (uint32_t)__builtin_amdgcn_readlane((int)before, 63) * p.KH) return;
    before -= mine;
    b = 63 - __builtin_clzll(__ballot(lane < (int)p.batch && before * p.KH <= share));
    splits = (uint32_t)__builtin_amdgcn_readlane((int)mine, b);
    first = (uint32_t)__builtin_amdgcn_readlane((int)before, b);
    const uint32_t at = share - first * p.KH;
    kvh = at % p.KH;
    split = at / p.KH;
    len_at = __builtin_amdgcn_readlane(len_at, b);
    start_at = __builtin_amdgcn_readlane(start_at, b);
    count_at = __builtin_amdgcn_readlane(count_at, b);
  } else {
    if (share >= p.shares) return;
    splits = p.nsplit;
    split = share % splits;
    kvh = share / splits % p.KH;
    b = share / splits / p.KH;
    first = b * splits;
    if (p.lens) {
      len_at = p.lens[b];
      start_at = p.starts[b];
    }
    if (p.counts) count_at = p.counts[b];
  }
  const uint32_t dh = PAD ? p.dh : (uint32_t)D;

  // What does not depend on the window's length is requested first: the queries of
  // the wave's row tile (dims (4c + g)*CW + e of row m16 in this lane), the draft.
  const uint32_t all = p.T * p.group;
  const uint32_t qrow = rb * ROWS + (PARTS ? wave % R * 16 : 0) + m16;
  float4 qraw[NC * CW / 4];
  {
    const float* src = p.q + (((size_t)b * p.T + qrow / p.group) * p.H + kvh * p.group + qrow % p.group) * dh;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int e = 0; e < CW; e += 4) {
        const uint32_t d = (c * 4 + g) * CW + e;
        qraw[(c * CW + e) / 4] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (qrow < all && (!PAD || d < dh)) qraw[(c * CW + e) / 4] = *reinterpret_cast<const float4*>(src + d);
      }
  }
  const bool narrow = MODE == kWindowTree && p.T <= 64;
  const int me = narrow ? lane : tid;  // the node that this lane looks after
  int up = -1;
  if (MODE == kWindowTree && me < (int)p.T) up = p.parents[(size_t)b * p.T + me];

  int32_t lo_at = 0, hi_at = 0;  // of the block's row tid
  float slope_at = 0.f;
  if (MODE == kWindowMasked && tid < ROWS && rb * ROWS + tid < all) {
    const uint32_t rr = rb * ROWS + tid;
    const size_t at = (size_t)b * p.T + rr / p.group;
    if (p.lo) lo_at = p.lo[at];
    if (p.hi) hi_at = p.hi[at];
    if (p.slopes) slope_at = p.slopes[kvh * p.group + rr % p.group];
  }

  const uint32_t len = __builtin_amdgcn_readfirstlane(len_at <= 0 ? 0u : min((uint32_t)len_at, p.M));
  start_at %= (int32_t)p.M;
  const uint32_t start =
      __builtin_amdgcn_readfirstlane((uint32_t)(start_at < 0 ? start_at + (int32_t)p.M : start_at));
  const uint32_t n = __builtin_amdgcn_readfirstlane(count_at <= 0 ? 0u : min(min((uint32_t)count_at, p.T), len));
  const uint32_t base = len - n;  // window row of query 0

  // Row rr of the block is query rr / group, head kvh*group + rr % group.
  const uint32_t row0 = rb * ROWS, nrows = n * p.group;
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

  // The rows that each query sees, their union over the block, and the rows that
  // all of its queries see.  Rows of the block past the queries see everything, so
  // that they never make a tile partly seen; their results go nowhere.
  uint32_t ulo = 0, uhi = len, alo = 0, ahi = MODE == kWindowTree ? base : len;
  if constexpr (MODE == kWindowMasked) {
    ulo = len;
    uhi = 0;
    if (tid < ROWS) {
      const uint32_t rr = row0 + tid, i = rr / p.group;
      uint32_t lo = 0, hi = len;
      if (rr < nrows) {
        lo = (uint32_t)max(lo_at, 0);
        hi = p.hi ? min((uint32_t)max(hi_at, 0), len) : base + i + 1;
      }
      s_row[tid] = Row{lo, hi, (int)(base + i), slope_at * kLog2e};
    }
    __syncthreads();
    const int last = (int)(live - row0);  // (the last rows of a block may be missing)
    const Row mine = s_row[min(lane, last - 1)];
    if (mine.lo < mine.hi) {
      ulo = mine.lo;
      uhi = mine.hi;
    }
    alo = mine.lo;
    ahi = mine.lo < mine.hi ? mine.hi : 0;
#pragma unroll
    for (int x = 1; x < 64; x *= 2) {
      ulo = min(ulo, (uint32_t)__shfl_xor((int)ulo, x, 64));
      uhi = max(uhi, (uint32_t)__shfl_xor((int)uhi, x, 64));
      alo = max(alo, (uint32_t)__shfl_xor((int)alo, x, 64));
      ahi = min(ahi, (uint32_t)__shfl_xor((int)ahi, x, 64));
    }
    ulo = __builtin_amdgcn_readfirstlane(ulo);
    uhi = __builtin_amdgcn_readfirstlane(uhi);
    alo = __builtin_amdgcn_readfirstlane(alo);
    ahi = __builtin_amdgcn_readfirstlane(ahi);
    if (ulo >= uhi) {  // no query of the block sees anything
      if (split == 0) zero_rows(row0, live);
      return;
    }
  }

  // Tiles of TILE window rows, dealt to the splits and waves in turn; a split gets
  // at least a tile for each wave.
  const uint32_t t0 = ulo / TILE, t1 = (uhi + TILE - 1) / TILE;
  const uint32_t nsplit = min(splits, (t1 - t0 + kWaves - 1) / kWaves);
  if (split >= nsplit) return;

  const size_t head = ((size_t)b * p.KH + kvh) * p.M * dh * ES;
  const __amdgpu_buffer_rsrc_t krs = coherent_rsrc(static_cast<const char*>(p.k) + head, p.M * dh * ES);
  const __amdgpu_buffer_rsrc_t vrs = coherent_rsrc(static_cast<const char*>(p.v) + head, p.M * dh * ES);
  auto row_off = [&](uint32_t r) {
    uint32_t slot = start + r;
    slot = slot >= p.M ? slot - p.M : slot;
    return r < uhi ? slot * (dh * ES) : kOutside;
  };
  // One row tile is all the query rows there are: nothing is read twice.
  constexpr int AUX = R > 1 ? 0 : kNt;
  typedef Piece<BF, CW, AUX> KRow[NC];  // a lane's part of 16 rows of K, and of V
  typedef Piece<BF, VW, AUX> VRow[4][NV];
  auto load_k = [&](uint32_t r0, KRow& k, int lane) {
    const int m16 = lane & 15, g = lane >> 4;
    const uint32_t off = row_off(r0 + m16) + g * (CW * ES);
#pragma unroll
    for (int c = 0; c < NC; ++c)
      k[c].load(krs, !PAD || (uint32_t)(c * 4 + g) * CW < dh ? off + c * (4 * CW * ES) : kOutside);
  };
  auto load_v = [&](uint32_t r0, VRow& v, int lane) {
    const int m16 = lane & 15, g = lane >> 4;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t off = row_off(r0 + 4 * g + i) + m16 * (VW * ES);
#pragma unroll
      for (int c = 0; c < NV; ++c)
        v[i][c].load(vrs, !PAD || (uint32_t)(c * 16 + m16) * VW < dh ? off + c * (16 * VW * ES) : kOutside);
    }
  };
  KRow kk[KT];
  VRow vv[KT];
  const uint32_t tstep = nsplit * kWaves;
  uint32_t t = t0 + split + nsplit * wave;
#pragma unroll
  for (int kt = 0; kt < KT; ++kt) load_k(t * TILE + kt * 16, kk[kt], lane);
  if constexpr (!PARTS) load_v(t * TILE, vv[0], lane);

  // The draft's relation "is above or is", a bit per node, and the nodes' depths:
  // each node takes over what its jump target knows and jumps as far as that one
  // does, until none has anywhere left to go.  Up to 64 nodes a wave does it for
  // itself, in registers, if it comes to any of the draft's rows; larger drafts go
  // through LDS.
  auto narrow_tree = [&]() __attribute__((always_inline)) {
    uint32_t a0 = lane < 32 ? 1u << lane : 0u, a1 = lane < 32 ? 0u : 1u << (lane - 32);
    int depth = up >= 0;
    while (__any(up >= 0)) {
      const int from = up >= 0 ? up : lane;
      const uint32_t b0 = __shfl((int)a0, from, 64), b1 = __shfl((int)a1, from, 64);
      const int deeper = __shfl(depth, from, 64), next = __shfl(up, from, 64);
      if (up >= 0) {
        a0 |= b0;
        a1 |= b1;
        depth += deeper;
        up = next;
      }
    }
    s_anc[lane][0] = a0;  // (the waves write the same)
    s_anc[lane][1] = a1;
    s_depth[lane] = depth;
  };
  if constexpr (MODE == kWindowTree) {
    up = me < (int)n && up >= 0 && up < me ? up : -1;
    if (narrow) {
      if (p.rope_cos) narrow_tree();  // (for the depths)
    } else {
      const uint32_t words = (n + 31) / 32;
#pragma unroll
      for (int w = 0; w < (int)kMaxTreeNodes / 32; ++w) s_anc[tid][w] = 0;
      s_anc[tid][tid >> 5] = 1u << (tid & 31);
      s_depth[tid] = up >= 0;
      s_jump[tid] = up;
      for (uint32_t reach = 1; reach < n; reach *= 2) {
        __syncthreads();
        uint32_t above[kMaxTreeNodes / 32];
        int next = -1, deeper = 0;
        if (up >= 0) {
#pragma unroll
          for (int w = 0; w < (int)kMaxTreeNodes / 32; ++w) above[w] = w < (int)words ? s_anc[up][w] : 0;
          next = s_jump[up];
          deeper = s_depth[up];
        }
        __syncthreads();
        if (up >= 0) {
#pragma unroll
          for (int w = 0; w < (int)kMaxTreeNodes / 32; ++w)
            if (w < (int)words) s_anc[tid][w] |= above[w];
          s_depth[tid] += deeper;
          s_jump[tid] = up = next;
        }
      }
      __syncthreads();
    }
  }

  // The query rows, rotated.
  auto turn_q = [&](float (&x)[NC][CW]) {
    uint32_t pos = p.rope_pos;
    if constexpr (MODE == kWindowTree) pos += s_depth[qrow < nrows ? qrow / p.group : 0];
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int e = 0; e < CW; e += 4) {
        const uint32_t d = (c * 4 + g) * CW + e;
        float4 y = qraw[(c * CW + e) / 4];
        if (p.rope_cos && (!PAD || d < dh)) {
          const size_t ro = (size_t)pos * (dh / 2) + d / 2;
          y = rope4(y, *reinterpret_cast<const float2*>(p.rope_cos + ro),
                    *reinterpret_cast<const float2*>(p.rope_sin + ro));
        }
        const bool on = qrow < nrows;
        x[c][e] = on ? y.x : 0.f;
        x[c][e + 1] = on ? y.y : 0.f;
        x[c][e + 2] = on ? y.z : 0.f;
        x[c][e + 3] = on ? y.w : 0.f;
      }
  };
  float qf[PARTS ? 1 : NC][CW];  // one row tile: in registers, scaled
  if constexpr (PARTS) {
    // In LDS as operand parts, scaled.
    if (wave < R) {
      float x[NC][CW];
      turn_q(x);
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int e = 0; e < CW; ++e) x[c][e] *= p.qscale;
#pragma unroll
      for (int c = 0; c < NP; ++c) {
        Frag y[kParts];
        split_parts(&x[0][0] + 8 * c, y);
#pragma unroll
        for (int n = 0; n < kParts; ++n) s_q[wave][c][n][lane] = y[n];
      }
    }
    __syncthreads();
  } else {
    turn_q(qf);
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int e = 0; e < CW; ++e) qf[c][e] *= p.qscale;
  }

  if constexpr (MODE == kWindowTree) {
    if (narrow && !p.rope_cos && t < t1 && (t + (t1 - 1 - t) / tstep * tstep + 1) * TILE > base) narrow_tree();
  }

  // The weights are taken relative to m, which follows the scores' maximum only when
  // they pass it, and then to 2^kRoom above it: the outputs are seldom rescaled, and no
  // weight is above 1, so that sums over a whole window of values of 1e30 stay in
  // range.  (A weight below 2^-118 of the largest may be lost.)
  constexpr float kRoom = 8.f;
  float m[R], l[R];
  f32x4 o[R][NX];
#pragma unroll
  for (int rt = 0; rt < R; ++rt) {
    m[rt] = -FLT_MAX;
    l[rt] = 0.f;
#pragma unroll
    for (int x = 0; x < NX; ++x) o[rt][x] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  // Whether some query does not see all of n rows from r0, or the window ends there.
  auto partly_seen = [&](uint32_t r0, uint32_t n) { return r0 < alo || r0 + n > ahi; };

  // What follows the scores of rows r0 .. (16 for each of s's tiles): cap, bias,
  // mask, and the weights they turn into, relative to m.
  auto weigh = [&](uint32_t r0, auto& s, bool partly, int lane) __attribute__((always_inline)) {
    const int m16 = lane & 15, g = lane >> 4;
    constexpr int K = sizeof(s[0]) / sizeof(f32x4);
    if constexpr (MODE == kWindowMasked) {
      if (p.cap_log2 > 0.f) {
#pragma unroll
        for (int rt = 0; rt < R; ++rt)
#pragma unroll
          for (int kt = 0; kt < K; ++kt)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[rt][kt][i] = p.cap_log2 * tanh_rel(s[rt][kt][i]);
      }
      if (p.slopes) {
#pragma unroll
        for (int rt = 0; rt < R; ++rt) {
          const int away = s_row[rt * 16 + m16].at - (int)(r0 + 4 * g);
          const float slope = s_row[rt * 16 + m16].slope;
#pragma unroll
          for (int kt = 0; kt < K; ++kt)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[rt][kt][i] -= slope * fabsf((float)(away - kt * 16 - i));
        }
      }
    }
    if constexpr (MODE == kWindowWeights) {
#pragma unroll
      for (int rt = 0; rt < R; ++rt)
        if (row0 + rt * 16 + m16 < nrows) {
          float* to = p.scores + ((size_t)b * p.H + kvh * p.group + row0 + rt * 16 + m16) * p.score_stride + r0 + 4 * g;
          // The stride covers whole tiles of 16 rows.
#pragma unroll
          for (int kt = 0; kt < K; ++kt)
            if (kt == 0 || r0 + kt * 16 < len) *reinterpret_cast<f32x4*>(to + kt * 16) = s[rt][kt];
        }
    }
    if (partly) {
#pragma unroll
      for (int rt = 0; rt < R; ++rt) {
        const uint32_t rr = row0 + rt * 16 + m16;
        uint32_t lo = 0, hi = len, node = 0;
        if constexpr (MODE == kWindowMasked) {
          lo = s_row[rt * 16 + m16].lo;
          hi = s_row[rt * 16 + m16].hi;
        }
        if constexpr (MODE == kWindowTree) node = rr < nrows ? rr / p.group : 0;
#pragma unroll
        for (int kt = 0; kt < K; ++kt)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t r = r0 + kt * 16 + 4 * g + i;
            bool seen = r >= lo && r < hi;
            if constexpr (MODE == kWindowTree) {
              if (seen && r >= base && rr < nrows) {
                const uint32_t j = r - base;
                seen = (s_anc[node][j >> 5] >> (j & 31)) & 1u;
              }
            }
            s[rt][kt][i] = seen ? s[rt][kt][i] : -INFINITY;
          }
      }
    }
    float top[R];
    bool passed = false;
#pragma unroll
    for (int rt = 0; rt < R; ++rt) {
      float x = -INFINITY;
#pragma unroll
      for (int kt = 0; kt < K; ++kt)
        x = fmaxf(x, fmaxf(fmaxf(s[rt][kt][0], s[rt][kt][1]), fmaxf(s[rt][kt][2], s[rt][kt][3])));
      top[rt] = max_xor32(max_xor16(x));
      passed |= top[rt] > m[rt];
    }
    if (__any(passed)) {
#pragma unroll
      for (int rt = 0; rt < R; ++rt) {
        const float now = top[rt] > m[rt] ? top[rt] + kRoom : m[rt], alpha = exp2_hw(m[rt] - now);
        m[rt] = now;
        l[rt] *= alpha;
#pragma unroll
        for (int x = 0; x < NX; ++x) o[rt][x] *= alpha;
      }
    }
#pragma unroll
    for (int rt = 0; rt < R; ++rt)
#pragma unroll
      for (int kt = 0; kt < K; ++kt) {
#pragma unroll
        for (int i = 0; i < 4; ++i) s[rt][kt][i] = exp2_hw(s[rt][kt][i] - m[rt]);
        l[rt] += (s[rt][kt][0] + s[rt][kt][1]) + (s[rt][kt][2] + s[rt][kt][3]);
      }
  };

  // The products of 16 rows of V in f32, with the weights w(rt) of the lane's four
  // rows.  A value that is not finite, in a row that some query does not see, would
  // be carried to that query as 0 * inf: it is taken out of the operand and added by
  // hand to the queries that see its row.
  auto add_values = [&](uint32_t r0, const VRow& v, auto w, bool partly, int lane)
      __attribute__((always_inline)) {
    const int m16 = lane & 15, g = lane >> 4;
    if (partly) {
      bool bad = false;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int x = 0; x < NX; ++x) bad |= not_finite(v[i][x / VW][x % VW]);
      if (__any(bad)) {
        for (int key = 0; key < 16; ++key) {
          const uint32_t off = row_off(r0 + key);
          const int from = (key >> 2) * 16 + m16;
          float u[R];
#pragma unroll
          for (int rt = 0; rt < R; ++rt) {
            const f32x4 y = w(rt);
            const float a = (key & 1) ? y[1] : y[0], z = (key & 1) ? y[3] : y[2];
            u[rt] = __shfl((key & 2) ? z : a, from, 64);
          }
#pragma unroll
          for (int c = 0; c < NV; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t d = (c * 16 + 4 * g + i) * VW;
              Piece<BF, VW, AUX> x;
              x.load(vrs, !PAD || d < dh ? off + d * ES : kOutside);
#pragma unroll
              for (int e = 0; e < VW; ++e) {
                const float y = x[e];
#pragma unroll
                for (int rt = 0; rt < R; ++rt)
                  if (not_finite(y) && !(u[rt] == 0.f)) o[rt][c * VW + e][i] += u[rt] * y;
              }
              __builtin_amdgcn_sched_barrier(0);
            }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int x = 0; x < NX; ++x) {
        float y = v[i][x / VW][x % VW];
        y = partly && not_finite(y) ? 0.f : y;
#pragma unroll
        for (int rt = 0; rt < R; ++rt)
          o[rt][x] = __builtin_amdgcn_mfma_f32_16x16x4f32(y, w(rt)[i], o[rt][x], 0, 0, 0);
      }
  };

  // 16 rows in f32, of which K and V stand in kk[0] and vv[0]; `next` runs when K is
  // no longer needed.
  auto in_f32 = [&](uint32_t r0, int at, auto next) __attribute__((always_inline)) {
    const bool partly = partly_seen(r0, 16);
    // Each score as kSums sums, of the dims in turn: shorter sums round less (outputs of
    // 32 heads on 4 over 30 to 1200 rows off by 8.5e-7 with one, by 3.5e-7 with four).
    constexpr int kSums = PARTS ? 1 : 4;
    f32x4 s[R][1];
#pragma unroll
    for (int rt = 0; rt < R; ++rt) {
      f32x4 sum[kSums];
#pragma unroll
      for (int n = 0; n < kSums; ++n) sum[n] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < NP; ++c) {
        float x[8];
        if constexpr (PARTS) {
          Frag qq[kParts];
#pragma unroll
          for (int n = 0; n < kParts; ++n) qq[n] = s_q[rt][c][n][at];
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = (float)qq[0][e] + ((float)qq[1][e] + (float)qq[2][e]);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = qf[(c * 8 + e) / CW][(c * 8 + e) % CW];
        }
#pragma unroll
        for (int e = 0; e < 8; ++e)
          sum[e % kSums] = __builtin_amdgcn_mfma_f32_16x16x4f32(kk[0][(c * 8 + e) / CW][(c * 8 + e) % CW], x[e],
                                                                sum[e % kSums], 0, 0, 0);
        if constexpr (PARTS) __builtin_amdgcn_sched_barrier(0);
      }
      s[rt][0] = kSums == 1 ? sum[0] : (sum[0] + sum[1 % kSums]) + (sum[2 % kSums] + sum[3 % kSums]);
    }
    next();
    weigh(r0, s, partly, at);
    add_values(r0, vv[0], [&](int rt) { return s[rt][0]; }, partly, at);
  };

  // Products of parts.  A tile of f32 rows with a value that is not finite, or too
  // near the end of f32's range to be split, is multiplied in f32, so that what sees
  // it follows f32; so are V rows of either type that hold such a value where some
  // query does not see them (0 * inf).
  // V is requested while K is consumed and the next tile's K while V is: a tile and
  // a half in registers in all, so that two waves fit a SIMD, which measured faster
  // than one wave with 64 query rows and both tiles ahead.  f32 rows 16 at a time,
  // which takes fewer registers, measured 222 us where 24 drafts of 40 nodes take 203.
  if constexpr (PARTS) {
    f32x4 s[R][KT];
    for (;;) {
    bool weighed = false;  // the tile's weights stand in s
    for (; t < t1; t += tstep) {
      const uint32_t r0 = t * TILE;
      const bool partly = partly_seen(r0, TILE);
      const int at = fresh_lane();
      float top = 0.f;  // K's largest (NaN stays)
#pragma unroll
      for (int rt = 0; rt < R; ++rt)
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) s[rt][kt] = f32x4{0.f, 0.f, 0.f, 0.f};
      // The queries' parts are read anew for every tile: kept in registers (the
      // compiler lifts the loads out of the loop) they would push others out.
#pragma unroll
      for (int c = 0; c < NP; ++c) {
        Frag kf[KT][BF ? 1 : kParts];
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
          if constexpr (BF) {
            kf[kt][0] = __builtin_bit_cast(Frag, kk[kt][c]);
          } else {
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              x[e] = kk[kt][(c * 8 + e) / CW][(c * 8 + e) % CW];
              top = __builtin_elementwise_maximum(top, fabsf(x[e]));
            }
            split_parts(x, kf[kt]);
          }
        }
        // The products below 2^-26 of the whole are left out.
#pragma unroll
        for (int n = kParts - 1; n >= 0; --n) {
          Frag qq[R];
#pragma unroll
          for (int rt = 0; rt < R; ++rt) qq[rt] = s_q[rt][c][n][at];
#pragma unroll
          for (int j = BF ? 0 : kParts - 1 - n; j >= 0; --j)
#pragma unroll
            for (int rt = 0; rt < R; ++rt)
#pragma unroll
              for (int kt = 0; kt < KT; ++kt) s[rt][kt] = multiply(kf[kt][j], qq[rt], s[rt][kt]);
        }
        if (c == NP / 2 - 1) load_v(r0, vv[0], at);
      }
      if (!BF && !__all(top <= kMostParts)) break;
      load_v(r0 + 16, vv[1], at);
      weigh(r0, s, partly, at);
      if constexpr (!BF) {
        top = 0.f;
#pragma unroll
        for (int i = 0; i < 4 * KT; ++i)
#pragma unroll
          for (int c = 0; c < NV; ++c)
#pragma unroll
            for (int e = 0; e < VW; ++e) top = __builtin_elementwise_maximum(top, fabsf(vv[i / 4][i % 4][c][e]));
        weighed = !__all(top <= kMostParts);
      } else if (partly) {
        bool bad = false;
#pragma unroll
        for (int i = 0; i < 4 * KT; ++i)
#pragma unroll
          for (int x = 0; x < NX; ++x) bad |= not_finite(vv[i / 4][i % 4][x / VW][x % VW]);
        weighed = __any(bad);
      }
      if (weighed) break;
      Frag pp[R][kParts];
#pragma unroll
      for (int rt = 0; rt < R; ++rt) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = s[rt][e >> 2][e & 3];
        split_parts(x, pp[rt]);
      }
#pragma unroll
      for (int x = 0; x < NX; ++x) {
        Frag vf[BF ? 1 : kParts];
        if constexpr (BF) {
          // The halves of the rows' words, paired along the rows.
          u32x4 y;
#pragma unroll
          for (int k = 0; k < 4; ++k)
            y[k] = __builtin_amdgcn_perm(vv[k / 2][k % 2 * 2 + 1][x / VW].w[x % VW / 2],
                                         vv[k / 2][k % 2 * 2][x / VW].w[x % VW / 2], x & 1 ? 0x07060302 : 0x05040100);
          vf[0] = __builtin_bit_cast(Frag, y);
        } else {
          float y[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) y[k] = vv[k / 4][k % 4][x / VW][x % VW];
          split_parts(y, vf);
        }
#pragma unroll
        for (int n = kParts - 1; n >= 0; --n)
#pragma unroll
          for (int j = BF ? 0 : n; j >= 0; --j)
#pragma unroll
            for (int rt = 0; rt < R; ++rt) o[rt][x] = multiply(vf[j], pp[rt][n - j], o[rt][x]);
        if (x == NX / 2 - 1) load_k((t + tstep) * TILE, kk[0], at);
      }
      load_k((t + tstep) * TILE + 16, kk[1], at);
    }
    if (t >= t1) break;
    const int at = fresh_lane();
    if (weighed) {
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
        const uint32_t r0 = t * TILE + kt * 16;
        load_v(r0, vv[0], at);
        add_values(r0, vv[0], [&](int rt) { return s[rt][kt]; }, partly_seen(r0, 16), at);
      }
    } else {
      for (uint32_t r0 = t * TILE; r0 < (t + 1) * TILE; r0 += 16) {
        load_k(r0, kk[0], at);
        load_v(r0, vv[0], at);
        in_f32(r0, at, [] {});
      }
    }
    t += tstep;
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) load_k(t * TILE + kt * 16, kk[kt], at);
    }
  } else {
    for (; t < t1; t += tstep) {
      const int at = fresh_lane();
      in_f32(t * TILE, at, [&] { load_k((t + tstep) * TILE, kk[0], at); });
      load_v((t + tstep) * TILE, vv[0], at);
    }
  }
  if constexpr (PARTS) __syncthreads();  // every wave is done with the queries' parts

  // The waves' states merged through LDS.
  const int lane1 = fresh_lane(), tid1 = wave * 64 + lane1;
#pragma unroll
  for (int rt = 0; rt < R; ++rt) {
    l[rt] = sum_xor32(sum_xor16(l[rt]));
    if ((lane1 >> 4) == 0) {
      s_ml[wave][rt * 16 + (lane1 & 15)][0] = m[rt];
      s_ml[wave][rt * 16 + (lane1 & 15)][1] = l[rt];
    }
#pragma unroll
    for (int c = 0; c < NV; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < VW; e += 4)
          *reinterpret_cast<f32x4*>(&s_o[wave][rt * 16 + (lane1 & 15)][(c * 16 + 4 * (lane1 >> 4) + i) * VW + e]) =
              f32x4{o[rt][c * VW + e][i], o[rt][c * VW + e + 1][i], o[rt][c * VW + e + 2][i], o[rt][c * VW + e + 3][i]};
  }
  __syncthreads();
  constexpr uint32_t REC = ROWS * (D + 2);  // floats of a split's record: O, then (m, l)
  const size_t unit = ((size_t)b * p.KH + kvh) * p.rblocks + rb;
  const __amdgpu_buffer_rsrc_t prs =
      coherent_rsrc(p.part + (((size_t)first * p.KH + kvh * splits) * p.rblocks + rb * splits) * REC,
                    nsplit > 1 ? splits * REC * 4 : 0);
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
  constexpr int NXT = ROWS * C4 / (kWaves * 64);  // float4 columns of a thread
#pragma unroll
  for (int k = 0; k < NXT; ++k) {
    const int x = tid1 + k * kWaves * 64, row = x / C4, col = x % C4;
    float mt = s_ml[0][row][0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) mt = fmaxf(mt, s_ml[w][row][0]);
    float lt = 0.f;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float f = exp2_hw(s_ml[w][row][0] - mt);
      lt += f * s_ml[w][row][1];
      const float4 y = *reinterpret_cast<const float4*>(&s_o[w][row][col * 4]);
      a.x += f * y.x;
      a.y += f * y.y;
      a.z += f * y.z;
      a.w += f * y.w;
    }
    if (nsplit == 1) {
      finish(row, col, a, mt, lt);
    } else {
      const uint32_t rec = split * REC * 4;
      st_coherent4(prs, rec + x * 16, coh_f4{a.x, a.y, a.z, a.w});
      if (col == 0) __builtin_amdgcn_raw_buffer_store_b64(u32x2{__float_as_uint(mt), __float_as_uint(lt)}, prs,
                                                          rec + (ROWS * D + row * 2) * 4, 0, kSc1);
    }
  }
  if (nsplit == 1) return;

  // Every thread's records are acknowledged before the workgroup takes its
  // arrival ticket; the last one merges the splits, always in their order.
  __builtin_amdgcn_s_waitcnt(0);
  __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "workgroup");
  __syncthreads();
  if (tid1 == 0) {
    const uint32_t ticket = atomicAdd(p.counters + unit, 1u);
    s_last = ticket == nsplit - 1;
    if (ticket == nsplit - 1) atomicExch(p.counters + unit, 0u);
  }
  __syncthreads();
  if (!s_last) return;
  __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "workgroup");
  // Each thread's columns of the first splits, requested before anything else.
  constexpr int AT = R == 1 ? 8 : 4;
  coh_f4 y[AT][NXT];
  auto request = [&](uint32_t sp) {
#pragma unroll
    for (int u = 0; u < AT; ++u)
#pragma unroll
      for (int k = 0; k < NXT; ++k)  // (past the record: zeros)
        y[u][k] = ld_coherent4(prs, sp + u < nsplit ? (sp + u) * REC * 4 + (tid1 + k * kWaves * 64) * 16 : kOutside);
  };
  // The splits' (m, l) of every row, all requested at once, in the LDS of the
  // partial outputs, which every thread is done with; m then gives way to the
  // split's factor 2^(m_s - m).
  constexpr int MS = max_splits(R);
  auto& s_f = *reinterpret_cast<float(*)[MS][ROWS]>(s_mem);
  auto& s_l = *reinterpret_cast<float(*)[MS][ROWS]>(s_mem + MS * ROWS * 4);
  static_assert(2 * MS * ROWS * 4 <= kOutBytes, "the splits' numbers fit");
  constexpr int NML = MS * ROWS / (kWaves * 64);
  u32x2 ml[NML];
  request(0);
#pragma unroll
  for (int k = 0; k < NML; ++k) {
    const uint32_t x = tid1 + k * kWaves * 64;
    if (x < nsplit * ROWS)
      ml[k] = __builtin_amdgcn_raw_buffer_load_b64(prs, (x / ROWS * REC + ROWS * D + x % ROWS * 2) * 4, 0, kSc1);
  }
#pragma unroll
  for (int k = 0; k < NML; ++k) {
    const uint32_t x = tid1 + k * kWaves * 64;
    if (x < nsplit * ROWS) {
      s_f[x / ROWS][x % ROWS] = __uint_as_float(ml[k][0]);
      s_l[x / ROWS][x % ROWS] = __uint_as_float(ml[k][1]);
    }
  }
  __syncthreads();
  if (tid1 < ROWS) {
    float mt = -FLT_MAX, lt = 0.f;
    for (uint32_t sp = 0; sp < nsplit; ++sp) mt = fmaxf(mt, s_f[sp][tid1]);
    for (uint32_t sp = 0; sp < nsplit; ++sp) {
      const float f = exp2_hw(s_f[sp][tid1] - mt);
      s_f[sp][tid1] = f;
      lt += f * s_l[sp][tid1];
    }
    s_ml[0][tid1][0] = mt;
    s_ml[0][tid1][1] = lt;
  }
  __syncthreads();
  float4 a[NXT];
#pragma unroll
  for (int k = 0; k < NXT; ++k) a[k] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (uint32_t sp = 0; sp < nsplit; sp += AT) {
    if (sp > 0) request(sp);
#pragma unroll
    for (int u = 0; u < AT; ++u)
#pragma unroll
      for (int k = 0; k < NXT; ++k) {
        const float f = sp + u < nsplit ? s_f[sp + u][(tid1 + k * kWaves * 64) / C4] : 0.f;
        a[k].x += f * y[u][k].x;
        a[k].y += f * y[u][k].y;
        a[k].z += f * y[u][k].z;
        a[k].w += f * y[u][k].w;
      }
  }
#pragma unroll
  for (int k = 0; k < NXT; ++k) {
    const int row = (tid1 + k * kWaves * 64) / C4;
    finish(row, (tid1 + k * kWaves * 64) % C4, a[k], s_ml[0][row][0], s_ml[0][row][1]);
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
  else
    bf16 ? launch_rows<MODE, 2, true>(p, grid, stream) : launch_rows<MODE, 2, false>(p, grid, stream);
  STS_HIP(hipGetLastError());
  return STS_OK;
}

}  // namespace window

// One translation unit each.
int launch_window_tree(const WindowParams& p, int row_tiles, bool bf16, dim3 grid, hipStream_t stream);
int launch_window_masked(const WindowParams& p, int row_tiles, bool bf16, dim3 grid, hipStream_t stream);
int launch_window_weights(const WindowParams& p, int row_tiles, bool bf16, dim3 grid, hipStream_t stream);

}  // namespace sts
