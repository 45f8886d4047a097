// paged_decode.hip -- attention of one query a stream over K/V rows in pages (gfx950).
// No counterpart in the reference, whose decode reads one ring a stream
// (crates/sts-wasm/src/model.rs:598-668).
//
// For query head h over the rows r of its stream
//   out_h = sum_r 2^(x_r - m) v_r / sum_r 2^(x_r - m),  x_r = scale log2(e) q_h.k_r
// in one pass with a running maximum m and sum in f32.
//
// A workgroup takes up to 16 query heads of one (stream, K/V head) and one split of
// the stream's rows; its four waves deal the split's tiles among themselves.  A tile is
// 16 rows of f32, 32 of the others, requested while the last is worked on.  A tile, or
// each sixteen of its rows, lies in one page and has a buffer resource of its own, ending
// with the stream's rows or empty where no page holds them: a lane's offsets are the same
// for all tiles, rows that are not there read as zeros, and pools may pass 4 GB.
//   S^T = K Q^T     A = K: lane (m, g) = (lane & 15, lane >> 4) holds row m; B = Q
//   O^T += V^T P^T  A = V^T: the lane holds of rows 4g + i the dims (16 c + m) VW + e;
//                   B = the weights as the first product leaves them in the lane
// f32 rows multiply in f32 (16x16x4).  bf16 rows are operands as they stand, against Q
// and the weights as three bf16 parts each, which add up to the f32 values; int8 codes
// are whole numbers that bf16 holds, and their rows' scales go into the scores and the
// weights.  Every product is therefore of f32's grade.
#include <algorithm>

#include "page_attend.hpp"

namespace sts {

namespace {

using namespace paged;

constexpr int kParts = 3;
constexpr uint32_t kSplitRows = 128;  // rows that a split is worth its record from
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// x[8] as three operands of bf16 values, each the nearest to what the ones before
// leave: their sum is x to 2^-26 of it (bf16 has f32's exponents).
__device__ __forceinline__ void parts_of(const float* x, bf16x8 (&y)[kParts]) {
  typedef __bf16 b2 __attribute__((ext_vector_type(2)));
  typedef float f2 __attribute__((ext_vector_type(2)));
  u32x4 w[kParts];
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

// The code in byte B of w as a float; whole numbers up to 127 are bf16 values, the
// upper half of the float's bits.
template <int B>
__device__ __forceinline__ uint32_t code_bits(uint32_t w) {
  return __float_as_uint((float)(int)(int8_t)(w >> (8 * B)));
}
__device__ __forceinline__ uint32_t pair_up(uint32_t hi, uint32_t lo) {
  return __builtin_amdgcn_perm(hi, lo, 0x07060302);
}

// WHOLE: a tile never passes the end of a page.
template <int D, int TYPE, bool PAD, bool WHOLE>
__global__ __launch_bounds__(kWaves * 64, TYPE == STS_PAGES_F32 ? 2 : 3) void paged_decode_kernel(const PagedDecode p) {
  constexpr bool F32 = TYPE == STS_PAGES_F32, I8 = TYPE == STS_PAGES_INT8;
  constexpr int ES = F32 ? 4 : I8 ? 1 : 2;
  constexpr int CW = 16 / ES;                     // dims of K a lane loads at once
  constexpr int NC = D / (4 * CW);                // loads per K row
  constexpr int VW = CW < D / 16 ? CW : D / 16;   // dims of V a lane loads at once
  constexpr int NV = D / (16 * VW);               // loads per V row
  constexpr int KT = F32 ? 1 : 2;                 // 16-row tiles a wave takes at once
  constexpr int TILE = 16 * KT;
  constexpr int NS = WHOLE ? 1 : KT;              // pieces of a tile that lie in one page
  constexpr int PIECE = TILE / NS;
  constexpr int NX = NV * VW;                     // 16-dim tiles of the output
  constexpr int NP = D / 32;                      // 32-dim steps of K Q^T
  constexpr int LDO = D + 4;                      // LDS row of a partial output
  constexpr int C4 = D / 4;

  constexpr int kPartBytes = F32 ? 0 : NP * kParts * 64 * 16;
  constexpr int kOutBytes = kWaves * 16 * LDO * 4;
  constexpr int kMostBytes = kPartBytes > kOutBytes ? kPartBytes : kOutBytes;
  __shared__ __align__(16) char s_mem[kMostBytes > kMergeBytes ? kMostBytes : kMergeBytes];
  auto& s_q = *reinterpret_cast<bf16x8(*)[NP][kParts][64]>(s_mem);
  auto& s_o = *reinterpret_cast<float(*)[kWaves][16][LDO]>(s_mem);
  __shared__ float s_ml[kWaves][16][2];
  __shared__ __align__(16) char s_new[2][D * ES];  // the appended row, K and V, as the page holds it
  __shared__ float s_scale[2];
  __shared__ uint32_t s_last;

  const PagedRows& rows = p.rows;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int m16 = lane & 15, g = lane >> 4;
  const uint32_t rb = blockIdx.x % p.rblocks, share = blockIdx.x / p.rblocks;
  Share at;
  if (!find_share(p, share, kSplitRows, at)) return;
  const uint32_t b = at.b, kvh = at.kvh, split = at.split, splits = at.splits, first = at.first, len = at.len;
  const uint32_t dh = PAD ? rows.dh : (uint32_t)D;
  const uint32_t h0 = kvh * p.group + rb * 16;           // the block's first query head
  const uint32_t live = min(p.group - rb * 16, 16u);     // its heads
  float* out = p.out + ((uint64_t)b * p.H + h0) * dh;
  if (len == 0) {
    if (split == 0)
      for (uint32_t t = tid; t < live * dh; t += kWaves * 64) out[t] = 0.f;
    return;
  }
  // Tiles of TILE rows, dealt to the splits and waves in turn.
  const uint32_t tiles = (len + TILE - 1) / TILE;
  const uint32_t nsplit = min(splits, (len + kSplitRows - 1) / kSplitRows);
  if (split >= nsplit) return;
  const uint32_t tstep = nsplit * kWaves;
  uint32_t t = split + nsplit * wave;

  // The pages of a tile: lane x asks for piece x.
  const __amdgpu_buffer_rsrc_t trs =
      coherent_rsrc(rows.table + (uint64_t)b * rows.max_pages, rows.max_pages * 4);
  auto ask_pages = [&](uint32_t t) {
    const uint32_t r = t * TILE + (lane & (NS - 1)) * PIECE;
    return __builtin_amdgcn_raw_buffer_load_b32(trs, r < len ? (r >> rows.shift) * 4 : kOutside, 0, 0);
  };
  // Where the rows of a tile's pieces are.  Uniform.
  struct Where {
    uint64_t at[NS];    // row index of the first
    uint32_t rows[NS];  // how many there are
  };
  const uint32_t in_page = (1u << rows.shift) - 1, page_heads = rows.KH << rows.shift, head = kvh << rows.shift;
  auto find = [&](uint32_t t, uint32_t asked, Where& w) {
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      const uint32_t page = (uint32_t)__builtin_amdgcn_readlane((int)asked, n);
      const uint32_t r0 = t * TILE + n * PIECE;
      const bool there = r0 < len && page < rows.pages;
      w.at[n] = there ? (uint64_t)page * page_heads + (head + (r0 & in_page)) : 0;
      w.rows[n] = there ? min(len - r0, (uint32_t)PIECE) : 0u;
    }
  };
  typedef Words<CW * ES / 4> KRow[NC];
  typedef Words<VW * ES / 4> VRow[4][NV];
  KRow kk[KT];
  VRow vv[KT];
  f32x4 ks[I8 ? KT : 1], vs[I8 ? KT : 1];
  const uint32_t rowb = dh * ES;
  const uint32_t koff = m16 * rowb + g * (CW * ES);
  // rows of 16-row tile kt, which begin at row `from` of its piece's resource
  auto scales = [&](const float* s, const Where& w, f32x4 (&x)[I8 ? KT : 1]) {
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      const __amdgpu_buffer_rsrc_t rs = coherent_rsrc(s + w.at[n], w.rows[n] * 4);
#pragma unroll
      for (int k = 0; k < KT / NS; ++k)
        x[n * (KT / NS) + k] =
            __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, g * 16 + k * 64, 0, kNt));
    }
  };
  auto load_k = [&](const Where& w) {
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      const __amdgpu_buffer_rsrc_t rs =
          coherent_rsrc(static_cast<const char*>(rows.k) + w.at[n] * rowb, w.rows[n] * rowb);
#pragma unroll
      for (int k = 0; k < KT / NS; ++k)
#pragma unroll
        for (int c = 0; c < NC; ++c)
          kk[n * (KT / NS) + k][c].load(rs, !PAD || (uint32_t)(c * 4 + g) * CW < dh
                                                ? koff + k * 16 * rowb + c * (4 * CW * ES) : kOutside);
    }
    if constexpr (I8) scales(rows.ks, w, ks);
  };
  auto load_v = [&](const Where& w) {
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      const __amdgpu_buffer_rsrc_t rs =
          coherent_rsrc(static_cast<const char*>(rows.v) + w.at[n] * rowb, w.rows[n] * rowb);
#pragma unroll
      for (int k = 0; k < KT / NS; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int c = 0; c < NV; ++c)
            vv[n * (KT / NS) + k][i][c].load(
                rs, !PAD || (uint32_t)(c * 16 + m16) * VW < dh
                        ? (k * 16 + 4 * g + i) * rowb + m16 * (VW * ES) + c * (16 * VW * ES) : kOutside);
    }
    if constexpr (I8) scales(rows.vs, w, vs);
  };

  // The pages are asked for two tiles ahead, so that no rows wait for them but the first.
  // The queries come last: four dims a load, each behind a test of its own and a wait for
  // what was requested before it (the first K and V rows, its cosines and sines), so that
  // they lengthen the prologue: f32 rows of 128 dims have eight such loads, the others two.
  const bool mine = (uint32_t)m16 < live;  // this lane's column is a query head
  const float* qsrc = p.q + b * p.q_stride + (uint64_t)(h0 + (mine ? m16 : 0)) * dh;
  // Dims of the lane's elements in 32-dim step c (f32: of its 4-dim load c).
  auto q_dim = [&](int c) {
    return F32 ? (c * 4 + g) * 4 : I8 ? c / 2 * 64 + g * 16 + c % 2 * 8 : (c * 4 + g) * 8;
  };
  auto get_q = [&](uint32_t d) {  // four of them, rotated and scaled
    if (!mine || (PAD && d >= dh)) return make_float4(0.f, 0.f, 0.f, 0.f);
    float4 y = *reinterpret_cast<const float4*>(qsrc + d);
    if (rows.rope_cos) {
      const uint64_t ro = (uint64_t)(len - 1) * (dh / 2) + d / 2;
      y = rope4(y, *reinterpret_cast<const float2*>(rows.rope_cos + ro),
                *reinterpret_cast<const float2*>(rows.rope_sin + ro));
    }
    return make_float4(y.x * p.qscale, y.y * p.qscale, y.z * p.qscale, y.w * p.qscale);
  };
  uint32_t asked = ask_pages(t);
  uint32_t asked_next = ask_pages(t + tstep);
  Where now;
  find(t, asked, now);
  load_k(now);
  load_v(now);
  float qf[F32 ? NC : 1][4];
  if constexpr (F32) {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const float4 y = get_q(q_dim(c));
      qf[c][0] = y.x;
      qf[c][1] = y.y;
      qf[c][2] = y.z;
      qf[c][3] = y.w;
    }
  } else {
    for (int c = wave; c < NP; c += kWaves) {
      const float4 y = get_q(q_dim(c)), z = get_q(q_dim(c) + 4);
      const float x[8] = {y.x, y.y, y.z, y.w, z.x, z.y, z.z, z.w};
      bf16x8 f[kParts];
      parts_of(x, f);
#pragma unroll
      for (int n = 0; n < kParts; ++n) s_q[c][n][lane] = f[n];
    }
    __syncthreads();
  }

  // A row to append is made by the wave that comes to its tile, K by the first D / 4 lanes
  // and V by the next: rotated, rounded, stored (by the first block of the group's heads)
  // and left in LDS, from where it takes its place among the loaded rows.
  const uint32_t new_row = len - 1, new_tile = new_row / TILE;
  bool appended = false;
  if (p.k_new && new_tile % nsplit == split && new_tile / nsplit % kWaves == (uint32_t)wave) {
    const uint32_t page = (uint32_t)rows.table[(uint64_t)b * rows.max_pages + (new_row >> rows.shift)];
    appended = page < rows.pages;
    constexpr int G = D / 4;
    const int which = lane / G;
    const uint32_t d = lane % G * 4;
    const bool on = which < 2 && (!PAD || d < dh);
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    if (on) {
      x = *reinterpret_cast<const float4*>((which ? p.v_new : p.k_new) + b * p.new_stride + (uint64_t)kvh * dh + d);
      if (rows.rope_cos && !which) {
        const uint64_t ro = (uint64_t)new_row * (dh / 2) + d / 2;
        x = rope4(x, *reinterpret_cast<const float2*>(rows.rope_cos + ro),
                  *reinterpret_cast<const float2*>(rows.rope_sin + ro));
      }
    }
    float scale = 1.f;
    if constexpr (I8) scale = row_scale(lanes_largest<G>(largest(x)));
    uint32_t words[ES];  // four values of ES bytes
    if constexpr (I8) {
      words[0] = row_codes(x, scale);
    } else if constexpr (F32) {
      words[0] = __float_as_uint(x.x);
      words[1] = __float_as_uint(x.y);
      words[2] = __float_as_uint(x.z);
      words[3] = __float_as_uint(x.w);
    } else {
      const uint2 y = bf16x4(x);
      words[0] = y.x;
      words[1] = y.y;
    }
    if (on) {
      uint32_t* to = reinterpret_cast<uint32_t*>(&s_new[which][d * ES]);
#pragma unroll
      for (int i = 0; i < ES; ++i) to[i] = words[i];
      if (I8 && d == 0) s_scale[which] = scale;
      if (appended && rb == 0) {
        const uint64_t at = (uint64_t)page * page_heads + (head + (new_row & in_page));
        to = reinterpret_cast<uint32_t*>(static_cast<char*>(which ? rows.v : rows.k) + at * rowb + d * ES);
#pragma unroll
        for (int i = 0; i < ES; ++i) to[i] = words[i];
        if (I8 && d == 0) (which ? rows.vs : rows.ks)[at] = scale;
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  }

  // The weights are relative to m, which follows the scores' maximum only when they
  // pass it, and then to 2^kRoom above it: the outputs are seldom rescaled.  (A weight
  // below 2^-118 of the largest may be lost.)
  constexpr float kRoom = 8.f;
  float m = -FLT_MAX, l = 0.f;
  f32x4 o[NX];
#pragma unroll
  for (int x = 0; x < NX; ++x) o[x] = f32x4{0.f, 0.f, 0.f, 0.f};

  for (; t < tiles; t += tstep) {
    if (appended && t == new_tile) {
      const uint32_t r = new_row % TILE;
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
#pragma unroll
        for (int c = 0; c < NC; ++c)
          if (r == (uint32_t)(kt * 16 + m16) && (!PAD || (uint32_t)(c * 4 + g) * CW < dh))
            kk[kt][c] = *reinterpret_cast<const Words<CW * ES / 4>*>(&s_new[0][(c * 4 + g) * (CW * ES)]);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (r == (uint32_t)(kt * 16 + 4 * g + i)) {
#pragma unroll
            for (int c = 0; c < NV; ++c)
              if (!PAD || (uint32_t)(c * 16 + m16) * VW < dh)
                vv[kt][i][c] = *reinterpret_cast<const Words<VW * ES / 4>*>(&s_new[1][(c * 16 + m16) * (VW * ES)]);
            if constexpr (I8) {
              ks[kt][i] = s_scale[0];
              vs[kt][i] = s_scale[1];
            }
          }
      }
    }
    f32x4 s[KT];
    // The queries' parts are read anew for every tile: kept in registers (the compiler
    // lifts the loads out of the loop) they would take a third workgroup's.
    int at_lane = lane;
    asm volatile("" : "+v"(at_lane));
    if constexpr (F32) {
      // Four sums of the dims in turn: shorter sums round less.
      f32x4 sum[4];
#pragma unroll
      for (int n = 0; n < 4; ++n) sum[n] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          sum[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kk[0][c].w[e]), qf[c][e], sum[e], 0, 0, 0);
      s[0] = (sum[0] + sum[1]) + (sum[2] + sum[3]);
    } else {
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) s[kt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < NP; ++c) {
        bf16x8 kf[KT];
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
          if constexpr (I8) {
            u32x4 y;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const uint32_t w = kk[kt][c / 2].w[c % 2 * 2 + i];
              y[i * 2] = pair_up(code_bits<1>(w), code_bits<0>(w));
              y[i * 2 + 1] = pair_up(code_bits<3>(w), code_bits<2>(w));
            }
            kf[kt] = __builtin_bit_cast(bf16x8, y);
          } else {
            kf[kt] = __builtin_bit_cast(bf16x8, kk[kt][c]);
          }
        }
#pragma unroll
        for (int n = kParts - 1; n >= 0; --n) {
          const bf16x8 q = s_q[c][n][at_lane];
#pragma unroll
          for (int kt = 0; kt < KT; ++kt) s[kt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[kt], q, s[kt], 0, 0, 0);
        }
      }
      if constexpr (I8) {
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) s[kt] *= ks[kt];
      }
    }
    // Rows that are not there.
    uint32_t there = 0;
#pragma unroll
    for (int n = 0; n < NS; ++n) there += now.rows[n];
    if (there < TILE) {
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if ((uint32_t)(kt % (KT / NS) * 16 + 4 * g + i) >= now.rows[kt / (KT / NS)]) {
            s[kt][i] = -INFINITY;
            if constexpr (I8) vs[kt][i] = 0.f;  // (what lies behind the rows may not be a number)
          }
    }
    // The next tile's K, now that this one's is used up.
    Where next;
    find(t + tstep, asked_next, next);
    asked_next = ask_pages(t + 2 * tstep);
    load_k(next);

    float top = -INFINITY;
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) top = fmaxf(top, fmaxf(fmaxf(s[kt][0], s[kt][1]), fmaxf(s[kt][2], s[kt][3])));
    top = max_xor32(max_xor16(top));
    if (__any(top > m)) {
      const float to = top > m ? top + kRoom : m, alpha = exp2_hw(m - to);
      m = to;
      l *= alpha;
#pragma unroll
      for (int x = 0; x < NX; ++x) o[x] *= alpha;
    }
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
#pragma unroll
      for (int i = 0; i < 4; ++i) s[kt][i] = exp2_hw(s[kt][i] - m);
      l += (s[kt][0] + s[kt][1]) + (s[kt][2] + s[kt][3]);
    }
    if constexpr (F32) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int x = 0; x < NX; ++x)
          o[x] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(vv[0][i][x / VW].w[x % VW]), s[0][i], o[x], 0, 0, 0);
    } else {
      if constexpr (I8) {
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) s[kt] *= vs[kt];
      }
#pragma unroll
      for (int k2 = 0; k2 < KT; k2 += 2) {
        bf16x8 pp[kParts];
        const float w[8] = {s[k2][0], s[k2][1], s[k2][2], s[k2][3],
                            s[k2 + 1][0], s[k2 + 1][1], s[k2 + 1][2], s[k2 + 1][3]};
        parts_of(w, pp);
#pragma unroll
        for (int x = 0; x < NX; ++x) {
          u32x4 y;  // the rows' values of dim x, paired along the rows
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t a = vv[k2 + k / 2][k % 2 * 2][x / VW].w[x % VW * ES / 4];
            const uint32_t z = vv[k2 + k / 2][k % 2 * 2 + 1][x / VW].w[x % VW * ES / 4];
            if constexpr (I8) {
              const int sh = x % 4 * 8;
              y[k] = pair_up(__float_as_uint((float)(int)(int8_t)(z >> sh)), __float_as_uint((float)(int)(int8_t)(a >> sh)));
            } else {
              y[k] = __builtin_amdgcn_perm(z, a, x & 1 ? 0x07060302 : 0x05040100);
            }
          }
          const bf16x8 vf = __builtin_bit_cast(bf16x8, y);
#pragma unroll
          for (int n = kParts - 1; n >= 0; --n) o[x] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pp[n], o[x], 0, 0, 0);
        }
      }
    }
    load_v(next);
    now = next;
  }
  if constexpr (!F32) __syncthreads();  // every wave is done with the queries' parts

  // The waves' states merged through LDS.
  l = sum_xor32(sum_xor16(l));
  if (g == 0) {
    s_ml[wave][m16][0] = m;
    s_ml[wave][m16][1] = l;
  }
  if (mine) {
#pragma unroll
    for (int c = 0; c < NV; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < VW; e += 4)
          *reinterpret_cast<f32x4*>(&s_o[wave][m16][(c * 16 + 4 * g + i) * VW + e]) =
              f32x4{o[c * VW + e][i], o[c * VW + e + 1][i], o[c * VW + e + 2][i], o[c * VW + e + 3][i]};
  }
  __syncthreads();
  const uint32_t slots = live * C4;  // float4 columns of the block's outputs
  auto finish = [&](uint32_t x, float4 a, float, float lt) {
    const uint32_t row = x / C4, col = x % C4;
    const float f = lt > 0.f || lt != lt ? 1.f / lt : 0.f;  // nothing seen: zeros
    if (!PAD || col * 4 < dh)
      *reinterpret_cast<float4*>(out + (uint64_t)row * dh + col * 4) = make_float4(a.x * f, a.y * f, a.z * f, a.w * f);
  };
  const Records rec{coherent_rsrc(p.part + (((uint64_t)first * rows.KH + kvh * splits) * p.rblocks + rb * splits) * p.record,
                                  nsplit > 1 ? splits * p.record * 4 : 0),
                    p.record, live};
  for (uint32_t x = tid; x < slots; x += kWaves * 64) {
    const uint32_t row = x / C4, col = x % C4;
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
    if (nsplit == 1) finish(x, a, mt, lt);
    else put_record<D>(rec, split, x, a, mt, lt);
  }
  if (nsplit == 1) return;
  const uint64_t unit = ((uint64_t)b * rows.KH + kvh) * p.rblocks + rb;
  merge_splits<D, 16>(rec, p.counters + unit * kCounters, split, nsplit, s_mem, s_last, finish);
}

struct PagedPlan {
  uint32_t rblocks = 1, nsplit = 1, shares = 0, record = 0;
  float rows_factor = 0.f;
};

PagedPlan plan_paged(const PagedDecode& p, uint32_t batch) {
  PagedPlan pl;
  const PagedRows& rows = p.rows;
  pl.rblocks = (p.group + 15) / 16;
  const uint64_t units = (uint64_t)batch * rows.KH * pl.rblocks;
  // Two workgroups a CU, which between them even out what streams of different lengths
  // leave uneven (24 streams of 900 to 4099 bf16 rows of 8 heads 47 us, with one a CU 59;
  // 9 of 31 to 2777 f32 rows 70.1 and 73.1); one for a single stream, whose splits are
  // alike and whose merge is then shorter (3000 8-bit rows of 32 heads 10.7 us for 11.8,
  // 30000 of 4 heads 16.3 for 18.7).
  const uint64_t target = (uint64_t)device_cu_count() * (batch > 1 ? 2 : 1);
  // A split is worth its record from 128 rows of a group's head on (30 streams of 20 to 500
  // f32 rows of 6 heads 15.7 us, from 64 on 19.7, from 256 on 18.4), of a lone head from a unit
  // for each of its waves on.
  const uint32_t least = p.group == 1 ? 64 : kSplitRows;
  const uint64_t most = std::min<uint64_t>((rows.max_rows + least - 1) / least, kMaxSplits);
  if (batch > 1 && batch <= 64) {
    // Streams of different ages: splits of about equal length whatever their stream,
    // not more than fit at once where one round can hold them (rounding up gives each
    // stream half a split more).  A wave looks at a stream a lane, so more of them are cut
    // into as many splits each whatever their length (64 streams of 31 to 3000 bf16 rows of
    // 8 heads 74 us, 65 of them 89).
    const uint64_t heads = (uint64_t)rows.KH * pl.rblocks;
    const uint64_t fit = 2 * units <= target ? target - units / 2 : target;
    pl.rows_factor = (float)heads / (float)fit;
    pl.nsplit = (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>(fit / heads + 1, most));
    pl.shares = (uint32_t)(rows.KH * (fit / heads + batch + 1));
  } else {
    const uint64_t want = std::max<uint64_t>(1, (target + units - 1) / units);
    pl.nsplit = (uint32_t)std::max<uint64_t>(1, std::min(want, most));
    pl.shares = batch * rows.KH * pl.nsplit;
  }
  const uint32_t live = std::min(p.group, 16u), wide = rows.dh <= 64 ? 64 : 128;
  pl.record = live * wide + (2 * live + 3) / 4 * 4;
  return pl;
}

int paged_workspace(const PagedDecode& p, const PagedPlan& pl, uint32_t batch, hipStream_t stream, Workspace** out) {
  *out = nullptr;
  if (pl.nsplit <= 1) return STS_OK;
  return get_workspace(stream, (size_t)pl.shares * pl.rblocks * pl.record,
                       (size_t)batch * p.rows.KH * pl.rblocks * kCounters, out);
}

template <int TYPE, bool WHOLE>
void launch_type(const PagedDecode& p, dim3 grid, hipStream_t stream) {
  const dim3 block(kWaves * 64);
  if (p.rows.dh == 128)
    hipLaunchKernelGGL((paged_decode_kernel<128, TYPE, false, WHOLE>), grid, block, 0, stream, p);
  else if (p.rows.dh == 64)
    hipLaunchKernelGGL((paged_decode_kernel<64, TYPE, false, WHOLE>), grid, block, 0, stream, p);
  else if (p.rows.dh > 64)
    hipLaunchKernelGGL((paged_decode_kernel<128, TYPE, true, WHOLE>), grid, block, 0, stream, p);
  else
    hipLaunchKernelGGL((paged_decode_kernel<64, TYPE, true, WHOLE>), grid, block, 0, stream, p);
}

}  // namespace

int launch_paged_decode(PagedDecode p, uint32_t batch, hipStream_t stream) {
  const PagedPlan pl = plan_paged(p, batch);
  Workspace* ws = nullptr;
  if (int rc = paged_workspace(p, pl, batch, stream, &ws)) return rc;
  if (ws) {
    p.part = ws->part;
    p.counters = ws->counters;
  }
  p.rblocks = pl.rblocks;
  p.nsplit = pl.nsplit;
  p.batch = batch;
  p.rows_factor = pl.rows_factor;
  p.record = pl.record;
  const dim3 grid(pl.shares * pl.rblocks);
  if (p.group == 1) return launch_paged_lone(p, grid, stream);
  const bool whole = p.rows.shift > 4;  // pages of 32 rows or more hold whole tiles
  if (p.rows.type == STS_PAGES_F32) launch_type<STS_PAGES_F32, true>(p, grid, stream);
  else if (p.rows.type == STS_PAGES_BF16)
    whole ? launch_type<STS_PAGES_BF16, true>(p, grid, stream) : launch_type<STS_PAGES_BF16, false>(p, grid, stream);
  else
    whole ? launch_type<STS_PAGES_INT8, true>(p, grid, stream) : launch_type<STS_PAGES_INT8, false>(p, grid, stream);
  STS_HIP(hipGetLastError());
  return STS_OK;
}

}  // namespace sts
