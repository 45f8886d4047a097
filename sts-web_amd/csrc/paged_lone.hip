// paged_lone.hip -- attention of one query a stream over K/V rows in pages where every
// query head has rows of its own (gfx950).  The formula is paged_decode.hip's; a matrix
// tile would leave 15 of its 16 columns empty, and the work on the weights would be done
// sixteen times over, so the products run on the vector units in f32.
//
// A lane holds 16 bytes of a row, G lanes a row, 64 / G rows a load; a unit is eight
// loads of K and of V (at most; sixteen rows at least), 16 KB at most, which a wave has
// requested while it works on the last.  The dot products are summed over the G lanes by
// a butterfly that leaves each lane one row's score, so that scales, masks and
// exponentials are done once a row, and the weights go to the row's lanes through LDS.
// Sixteen rows lie in one page and have a buffer resource of their own, as there.
//
// A row to be appended is made by the wave that comes to its unit: rotated, rounded,
// stored, and used from registers.
#include "page_attend.hpp"

namespace sts {

namespace {

using namespace paged;

// Element e of a lane's 16 bytes, as f32.
template <int TYPE>
__device__ __forceinline__ float element(const Words<4>& x, int e) {
  if constexpr (TYPE == STS_PAGES_F32) return __uint_as_float(x.w[e]);
  else if constexpr (TYPE == STS_PAGES_BF16)
    return __uint_as_float((e & 1) ? x.w[e >> 1] & 0xffff0000u : x.w[e >> 1] << 16);
  else return (float)(int)(int8_t)(x.w[e >> 2] >> (8 * (e & 3)));
}

// One level of the butterfly: N values in, N / 2 out; the lane whose bit LEVEL is set
// keeps the upper half.
template <int LEVEL, int N>
__device__ __forceinline__ void fold(float* s, int c) {
  const bool hi = (c >> LEVEL) & 1;
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    const float a = s[i], z = s[i + N / 2];
    s[i] = (hi ? z : a) + xchg<LEVEL>(hi ? a : z);
  }
}
// N values summed over lanes whose index differs in bits 0 .. LEVELS-1: the lane ends
// with value (c >> (LEVELS - log2 N)) & (N - 1).
template <int LEVELS, int N>
__device__ __forceinline__ float fold_all(float* s, int c) {
  if constexpr (LEVELS > 0) {
    if constexpr (N > 1) fold<LEVELS - 1, N>(s, c);
    else s[0] += xchg<LEVELS - 1>(s[0]);
    return fold_all<LEVELS - 1, (N > 1 ? N / 2 : 1)>(s, c);
  }
  return s[0];
}
// The same over lanes whose index differs in bits FROM .. FROM + log2 N - 1 alone: N
// values in, of which each lane ends with N / M (those from (lane >> FROM) N / M on), M the
// number of lanes.
template <int LEVEL>
__device__ __forceinline__ float xor_lane(float x) {
  if constexpr (LEVEL == 5) return xor32(x);
  else return __int_as_float(__builtin_amdgcn_ds_swizzle(__float_as_int(x), 0x1F | 1 << (LEVEL + 10)));
}
template <int FROM, int LEVEL, int N>
__device__ __forceinline__ void fold_groups(float* s, int lane) {
  if constexpr (LEVEL >= FROM) {
    static_assert(N > 1, "a value for each lane at least");
    const bool hi = (lane >> LEVEL) & 1;
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const float a = s[i], z = s[i + N / 2];
      s[i] = (hi ? z : a) + xor_lane<LEVEL>(hi ? a : z);
    }
    fold_groups<FROM, LEVEL - 1, N / 2>(s, lane);
  }
}
// An operation over lanes whose index differs in bits FROM .. TO-1.
template <int FROM, int TO, class Op>
__device__ __forceinline__ float over(float x, Op op) {
  if constexpr (FROM < TO) return over<FROM + 1, TO>(op(x, xchg<FROM>(x)), op);
  return x;
}
constexpr int log2_of(int n) { return n <= 1 ? 0 : 1 + log2_of(n / 2); }

template <int D, int TYPE, bool PAD>
__global__ __launch_bounds__(kWaves * 64) __attribute__((amdgpu_waves_per_eu(1, 8)))
void paged_lone_kernel(const PagedDecode p) {
  constexpr bool I8 = TYPE == STS_PAGES_INT8;
  constexpr int ES = TYPE == STS_PAGES_F32 ? 4 : I8 ? 1 : 2;
  constexpr int CW = 16 / ES;                // a lane's dims
  constexpr int G = D / CW, LG = log2_of(G); // lanes a row
  constexpr int NG = 64 / G;                 // rows a load
  constexpr int RPG = G < 8 ? G : 8, LR = log2_of(RPG);  // loads of a unit
  constexpr int UNIT = NG * RPG;
  constexpr int NSUB = UNIT / 16;
  constexpr int C4 = D / 4;
  static_assert(UNIT >= 16, "whole sixteens");

  constexpr int kAccBytes = kWaves * D * 4;
  __shared__ __align__(16) char s_mem[kAccBytes > kMergeBytes ? kAccBytes : kMergeBytes];
  auto& s_acc = *reinterpret_cast<float(*)[kWaves][D]>(s_mem);
  __shared__ __align__(16) float s_p[kWaves][UNIT];
  __shared__ float s_ml[kWaves][2];
  __shared__ uint32_t s_last;

  const PagedRows& rows = p.rows;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane / G, c = lane % G;
  const int jj = (c >> (LG - LR)) & (RPG - 1);  // the lane's row of its group, once summed
  Share at;
  if (!find_share(p, blockIdx.x, kWaves * UNIT, at)) return;
  const uint32_t b = at.b, h = at.kvh, len = at.len;
  const uint32_t dh = PAD ? rows.dh : (uint32_t)D;
  float* out = p.out + ((uint64_t)b * p.H + h) * dh;
  if (len == 0) {
    if (at.split == 0)
      for (uint32_t t = tid; t < dh; t += kWaves * 64) out[t] = 0.f;
    return;
  }
  const uint32_t units = (len + UNIT - 1) / UNIT;
  const uint32_t nsplit = min(at.splits, (units + kWaves - 1) / kWaves);
  if (at.split >= nsplit) return;
  const uint32_t step = nsplit * kWaves;
  uint32_t u = at.split + nsplit * wave;

  // Each lane asks for the page of the row whose score it will have.
  const uint32_t my_row = jj * NG + g;  // of a unit
  const __amdgpu_buffer_rsrc_t trs =
      coherent_rsrc(rows.table + (uint64_t)b * rows.max_pages, rows.max_pages * 4);
  auto ask_pages = [&](uint32_t u) {
    const uint32_t r = u * UNIT + my_row;
    return (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(trs, r < len ? (r >> rows.shift) * 4 : kOutside, 0, 0);
  };
  const uint32_t in_page = (1u << rows.shift) - 1;
  const uint32_t rowb = dh * ES;
  auto row_at = [&](uint32_t page, uint32_t r) {
    return (((uint64_t)page * rows.KH + h) << rows.shift) + (r & in_page);
  };
  // Where a unit's rows are: for each sixteen its first (uniform) and how many there are,
  // and whether the lane's own row is there.
  struct Where {
    uint64_t at[NSUB];
    uint32_t rows[NSUB];
    uint64_t mine;
    bool seen;
  };
  auto find = [&](uint32_t u, uint32_t asked, Where& w) {
#pragma unroll
    for (int s = 0; s < NSUB; ++s) {
      const uint32_t page = (uint32_t)__builtin_amdgcn_readlane((int)asked, (s * 16 / NG) << (LG - LR));
      const uint32_t r0 = u * UNIT + s * 16;
      const bool there = r0 < len && page < rows.pages;
      w.at[s] = there ? row_at(page, r0) : 0;
      w.rows[s] = there ? min(len - r0, 16u) : 0u;
    }
    const uint32_t r = u * UNIT + my_row;
    w.seen = r < len && asked < rows.pages;
    w.mine = w.seen ? row_at(asked, r) : 0;
  };
  const bool lane_on = !PAD || (uint32_t)c * CW < dh;
  const uint32_t lane_off = lane_on ? g * rowb + c * 16 : kOutside;
  auto load = [&](const void* from, const Where& w, Words<4> (&x)[RPG]) {
#pragma unroll
    for (int s = 0; s < NSUB; ++s) {
      const __amdgpu_buffer_rsrc_t rs =
          coherent_rsrc(static_cast<const char*>(from) + w.at[s] * rowb, w.rows[s] * rowb);
#pragma unroll
      for (int j = 0; j < RPG; ++j)
        if (j * NG / 16 == s) x[j].load(rs, lane_off + j * NG % 16 * rowb);
    }
  };

  uint32_t asked = ask_pages(u);
  uint32_t asked_next = ask_pages(u + step);
  // The query, rotated and scaled, and the row to append.
  float q[CW];
  float4 kn4[CW / 4], vn4[CW / 4];
  const bool append = p.k_new != nullptr;
  const uint32_t new_row = len - 1, new_unit = new_row / UNIT;
  const bool owner = append && new_unit % nsplit == at.split && new_unit / nsplit % kWaves == (uint32_t)wave;
#pragma unroll
  for (int e = 0; e < CW / 4; ++e) {
    const uint32_t d = c * CW + e * 4;
    float4 q4 = make_float4(0.f, 0.f, 0.f, 0.f);
    kn4[e] = vn4[e] = q4;
    if (lane_on) {
      q4 = *reinterpret_cast<const float4*>(p.q + b * p.q_stride + (uint64_t)h * dh + d);
      if (owner) {
        kn4[e] = *reinterpret_cast<const float4*>(p.k_new + b * p.new_stride + (uint64_t)h * dh + d);
        vn4[e] = *reinterpret_cast<const float4*>(p.v_new + b * p.new_stride + (uint64_t)h * dh + d);
      }
      if (rows.rope_cos) {
        const uint64_t ro = (uint64_t)new_row * (dh / 2) + d / 2;
        const float2 cs = *reinterpret_cast<const float2*>(rows.rope_cos + ro);
        const float2 sn = *reinterpret_cast<const float2*>(rows.rope_sin + ro);
        q4 = rope4(q4, cs, sn);
        kn4[e] = rope4(kn4[e], cs, sn);
      }
    }
    q[e * 4] = q4.x * p.qscale;
    q[e * 4 + 1] = q4.y * p.qscale;
    q[e * 4 + 2] = q4.z * p.qscale;
    q[e * 4 + 3] = q4.w * p.qscale;
  }

  Words<4> kk[RPG], vv[RPG];
  float ks = 1.f, vs = 1.f;
  Where now;
  find(u, asked, now);
  load(rows.k, now, kk);
  __builtin_amdgcn_sched_barrier(0);
  load(rows.v, now, vv);
  if constexpr (I8) {
    ks = rows.ks[now.mine];
    vs = rows.vs[now.mine];
  }

  // The new row as the page holds it, in the lanes of every row group.
  Words<4> kn, vn;
  float kns = 1.f, vns = 1.f;
  const int new_g = (int)(new_row % UNIT % NG), new_j = (int)(new_row % UNIT / NG);
  bool appended = false;
  if (owner) {
    const uint32_t page = (uint32_t)rows.table[(uint64_t)b * rows.max_pages + (new_row >> rows.shift)];
    appended = page < rows.pages;
    auto make = [&](const float4* x, Words<4>& y, float& scale) {
      float top = 0.f;
#pragma unroll
      for (int e = 0; e < CW / 4; ++e) {
        if constexpr (I8) top = __builtin_elementwise_maximum(top, largest(x[e]));
      }
      if constexpr (I8) {
        top = over<0, LG>(top, [](float a, float z) { return __builtin_elementwise_maximum(a, z); });
        scale = row_scale(top);
      }
#pragma unroll
      for (int e = 0; e < CW / 4; ++e) {
        if constexpr (I8) {
          y.w[e] = row_codes(x[e], scale);
        } else if constexpr (TYPE == STS_PAGES_BF16) {
          const uint2 t = bf16x4(x[e]);
          y.w[e * 2] = t.x;
          y.w[e * 2 + 1] = t.y;
        } else {
          y.w[0] = __float_as_uint(x[e].x);
          y.w[1] = __float_as_uint(x[e].y);
          y.w[2] = __float_as_uint(x[e].z);
          y.w[3] = __float_as_uint(x[e].w);
        }
      }
    };
    make(kn4, kn, kns);
    make(vn4, vn, vns);
    if (appended && g == new_g && lane_on) {
      const uint64_t to = row_at(page, new_row);
      *reinterpret_cast<u32x4*>(static_cast<char*>(rows.k) + to * rowb + c * 16) = u32x4{kn.w[0], kn.w[1], kn.w[2], kn.w[3]};
      *reinterpret_cast<u32x4*>(static_cast<char*>(rows.v) + to * rowb + c * 16) = u32x4{vn.w[0], vn.w[1], vn.w[2], vn.w[3]};
      if (I8 && c == 0) {
        rows.ks[to] = kns;
        rows.vs[to] = vns;
      }
    }
  }

  constexpr float kRoom = 8.f;  // as in paged_decode.hip
  float m = -FLT_MAX, l = 0.f, acc[CW];
#pragma unroll
  for (int e = 0; e < CW; ++e) acc[e] = 0.f;

  while (u < units) {
    if (appended && u == new_unit) {
#pragma unroll
      for (int j = 0; j < RPG; ++j)
        if (g == new_g && j == new_j) {
          kk[j] = kn;
          vv[j] = vn;
        }
      if (my_row == new_row % UNIT) {
        ks = kns;
        vs = vns;
      }
    }
    float s[RPG];
#pragma unroll
    for (int j = 0; j < RPG; ++j) {
      s[j] = q[0] * element<TYPE>(kk[j], 0);
#pragma unroll
      for (int e = 1; e < CW; ++e) s[j] = fmaf(q[e], element<TYPE>(kk[j], e), s[j]);
    }
    float sc = fold_all<LG, RPG>(s, c);
    if constexpr (I8) sc *= ks;
    sc = now.seen ? sc : -INFINITY;
    // (One maximum for the wave, so that its rows' sums add up without factors.)
    float top = over<LG - LR, 4>(sc, [](float a, float z) { return fmaxf(a, z); });
    top = max_xor32(max_xor16(top));
    if (__any(top > m)) {
      const float to = top > m ? top + kRoom : m, alpha = exp2_hw(m - to);
      m = to;
      l *= alpha;
#pragma unroll
      for (int e = 0; e < CW; ++e) acc[e] *= alpha;
    }
    const float w = exp2_hw(sc - m);
    l += w;
    if ((c & ((1 << (LG - LR)) - 1)) == 0) s_p[wave][g * RPG + jj] = I8 ? (now.seen ? w * vs : 0.f) : w;
    // The next unit's K, now that this one's is used up.
    find(u + step, asked_next, now);
    asked_next = ask_pages(u + 2 * step);
    load(rows.k, now, kk);
    if constexpr (I8) {
      ks = rows.ks[now.mine];
      vs = rows.vs[now.mine];
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    float pp[RPG];
#pragma unroll
    for (int j = 0; j < RPG; j += 4) {
      const float4 y = *reinterpret_cast<const float4*>(&s_p[wave][g * RPG + j]);
      pp[j] = y.x;
      pp[j + 1] = y.y;
      pp[j + 2] = y.z;
      pp[j + 3] = y.w;
    }
#pragma unroll
    for (int j = 0; j < RPG; ++j)
#pragma unroll
      for (int e = 0; e < CW; ++e) acc[e] = fmaf(pp[j], element<TYPE>(vv[j], e), acc[e]);
    load(rows.v, now, vv);
    u += step;
  }

  // The row groups' sums added up, and the waves' states merged through LDS.  (A row's weight
  // is in the 2^(LG - LR) lanes that share it.)
  l = sum_xor32(sum_xor16(over<LG - LR, 4>(l, [](float a, float z) { return a + z; })));
  fold_groups<LG, 5, CW>(acc, lane);
  constexpr int PER = CW / NG;
#pragma unroll
  for (int e = 0; e < PER; ++e) s_acc[wave][c * CW + g * PER + e] = acc[e];
  if (lane == 0) {
    s_ml[wave][0] = m;
    s_ml[wave][1] = l;
  }
  __syncthreads();
  auto finish = [&](uint32_t x, float4 a, float, float lt) {
    const float f = lt > 0.f || lt != lt ? 1.f / lt : 0.f;  // nothing seen: zeros
    if (!PAD || x * 4 < dh)
      *reinterpret_cast<float4*>(out + x * 4) = make_float4(a.x * f, a.y * f, a.z * f, a.w * f);
  };
  const Records rec{coherent_rsrc(p.part + ((uint64_t)at.first * rows.KH + h * at.splits) * p.record,
                                  nsplit > 1 ? at.splits * p.record * 4 : 0),
                    p.record, 1};
  if (tid < C4) {
    float mt = s_ml[0][0], lt = 0.f;
#pragma unroll
    for (int w = 1; w < kWaves; ++w) mt = fmaxf(mt, s_ml[w][0]);
    f32x4 a = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float f = exp2_hw(s_ml[w][0] - mt);
      lt = fmaf(f, s_ml[w][1], lt);
      a += *reinterpret_cast<const f32x4*>(&s_acc[w][tid * 4]) * f;
    }
    const float4 y = make_float4(a[0], a[1], a[2], a[3]);
    if (nsplit == 1) finish(tid, y, mt, lt);
    else put_record<D>(rec, at.split, tid, y, mt, lt);
  }
  if (nsplit == 1) return;
  merge_splits<D, 1>(rec, p.counters + ((uint64_t)b * rows.KH + h) * kCounters, at.split, nsplit, s_mem, s_last, finish);
}

// Of 8-bit rows a CU holds three or four workgroups, by their registers, or two, by LDS that
// the launch asks for and nobody uses.  Four heads a CU or more, over long rows, gain by two
// (64 streams of 32 heads of 128 to 3000 rows of 128 dims 134 us for 138, 100 of 150 to 3000
// rows of 64 dims 105 for 110); fewer or shorter ones lose (100 streams of 8 heads of 150 to
// 3000 rows of 128 dims 64 for 60, 64 of 32 heads of 25 to 500 rows 32 for 29, 100 of 64 dims
// 33 for 25).
constexpr uint32_t kTwoACu = 48 * 1024;
uint32_t spare_lds(const PagedDecode& p) {
  if (p.rows.type != STS_PAGES_INT8) return 0;
  const bool many = (uint64_t)p.batch * p.rows.KH >= 4ull * device_cu_count();
  const bool longs = (uint64_t)p.rows.max_rows * p.rows.dh >= 128 * 1024;
  return many && longs ? kTwoACu : 0;
}

template <int TYPE>
void launch_type(const PagedDecode& p, dim3 grid, hipStream_t stream) {
  const dim3 block(kWaves * 64);
  const uint32_t lds = spare_lds(p);
  if (p.rows.dh == 128)
    hipLaunchKernelGGL((paged_lone_kernel<128, TYPE, false>), grid, block, lds, stream, p);
  else if (p.rows.dh == 64)
    hipLaunchKernelGGL((paged_lone_kernel<64, TYPE, false>), grid, block, lds, stream, p);
  else if (p.rows.dh > 64)
    hipLaunchKernelGGL((paged_lone_kernel<128, TYPE, true>), grid, block, lds, stream, p);
  else
    hipLaunchKernelGGL((paged_lone_kernel<64, TYPE, true>), grid, block, lds, stream, p);
}

}  // namespace

int launch_paged_lone(const PagedDecode& p, dim3 grid, hipStream_t stream) {
  if (p.rows.type == STS_PAGES_F32) launch_type<STS_PAGES_F32>(p, grid, stream);
  else if (p.rows.type == STS_PAGES_BF16) launch_type<STS_PAGES_BF16>(p, grid, stream);
  else launch_type<STS_PAGES_INT8>(p, grid, stream);
  STS_HIP(hipGetLastError());
  return STS_OK;
}

}  // namespace sts
