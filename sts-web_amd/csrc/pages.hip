// pages.hip -- K/V rows into pages and out of them (gfx950).  No counterpart in the
// reference, whose caches are one ring a stream (crates/sts-wasm/src/model.rs:195-363).
//
// Both are copies that round, bound by HBM for many rows and by their launch for few.
#include "common.hpp"
#include "page_rows.hpp"
#include "rope.hpp"

namespace sts {

namespace {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));

// Four values of a row, of which lane c of G holds dims 4c .. 4c+3, to row `at`.
template <int TYPE, int G>
__device__ __forceinline__ void store_row(void* rows, float* scales, uint64_t at, uint32_t dh, int c, float4 x,
                                          bool on) {
  const uint64_t to = at * dh + c * 4;
  if constexpr (TYPE == STS_PAGES_F32) {
    if (on) *reinterpret_cast<float4*>(static_cast<float*>(rows) + to) = x;
  } else if constexpr (TYPE == STS_PAGES_BF16) {
    if (on) *reinterpret_cast<uint2*>(static_cast<uint16_t*>(rows) + to) = bf16x4(x);
  } else {
    const float s = row_scale(lanes_largest<G>(largest(x)));
    const uint32_t codes = row_codes(x, s);
    if (on) *reinterpret_cast<uint32_t*>(static_cast<int8_t*>(rows) + to) = codes;
    if (on && c == 0) scales[at] = s;
  }
}

// G lanes a row (K and V of it), 256 / G rows a workgroup.  A token is read before its
// stream's count is known, the tokens past it for nothing: one round trip less.  The 8-bit rows' instructions
// count: with the codes' corrections behind a test 512 rows of 32 heads take 7.5 us (9.7
// without).  (Measured slower: two or four rows for a group of lanes; half the lanes with
// eight values each, 2048 f32 rows of 32 heads 26.0 us for 23.3.)
template <int TYPE, int G>
__global__ __launch_bounds__(256) void paged_append_kernel(const PagedAppend p, uint32_t total) {
  const PagedRows& rows = p.rows;
  const int c = threadIdx.x % G;
  const uint32_t n = blockIdx.x * (256 / G) + threadIdx.x / G;
  if (n >= total) return;  // (whole groups of G lanes)
  const uint32_t bt = n / rows.KH, j = n - bt * rows.KH, b = bt / p.T, i = bt - b * p.T;
  const bool mine = (uint32_t)c * 4 < rows.dh;
  float4 k = make_float4(0.f, 0.f, 0.f, 0.f), v = k;
  if (mine) {
    const uint64_t from = bt * p.stride + (uint64_t)j * rows.dh + c * 4;
    k = *reinterpret_cast<const float4*>(p.k_new + from);
    v = *reinterpret_cast<const float4*>(p.v_new + from);
  }
  const uint32_t len = paged_len(rows, b);
  uint32_t count = min(p.T, len);
  if (p.counts) count = (uint32_t)min(max(p.counts[b], 0), (int32_t)count);
  if (i >= count) return;
  const uint32_t r = len - count + i;
  uint64_t at;
  if (!paged_row(rows, b, j, r, at)) return;
  if (rows.rope_cos && mine) {
    const uint64_t ro = (uint64_t)r * (rows.dh / 2) + c * 2;
    k = rope4(k, *reinterpret_cast<const float2*>(rows.rope_cos + ro),
              *reinterpret_cast<const float2*>(rows.rope_sin + ro));
  }
  store_row<TYPE, G>(rows.k, rows.ks, at, rows.dh, c, k, mine);
  store_row<TYPE, G>(rows.v, rows.vs, at, rows.dh, c, v, mine);
}

// Four values of a row.
template <int TYPE>
struct Four {
  float4 x;
  uint2 h;
  uint32_t w;
  __device__ __forceinline__ void load(const void* rows, uint64_t at) {
    if constexpr (TYPE == STS_PAGES_F32) {
      const f4 y = *reinterpret_cast<const f4*>(static_cast<const float*>(rows) + at);
      x = make_float4(y[0], y[1], y[2], y[3]);
    } else if constexpr (TYPE == STS_PAGES_BF16) {
      const u2 y = *reinterpret_cast<const u2*>(static_cast<const uint16_t*>(rows) + at);
      h = make_uint2(y[0], y[1]);
    } else {
      w = *reinterpret_cast<const uint32_t*>(static_cast<const int8_t*>(rows) + at);
    }
  }
  __device__ __forceinline__ float4 value(float s) const {
    if constexpr (TYPE == STS_PAGES_F32) return x;
    else if constexpr (TYPE == STS_PAGES_BF16)
      return make_float4(__uint_as_float(h.x << 16), __uint_as_float(h.x & 0xffff0000u), __uint_as_float(h.y << 16),
                         __uint_as_float(h.y & 0xffff0000u));
    else
      return make_float4((float)(int8_t)w * s, (float)(int8_t)(w >> 8) * s, (float)(int8_t)(w >> 16) * s,
                         (float)(int8_t)(w >> 24) * s);
  }
};

// A wave takes the sixteen rows of a page from r0 on (r0 a multiple of 16) of one stream and
// head, K or V: at most eight times 64 lanes of four values, all requested before the first
// is stored.  With streaming stores, which leave the caches to the pages: 3000 bf16 rows of
// 32 heads 24.7 us, 6.0 TB/s (30.8 with plain ones; torch's copy of a large tensor moves 4.8).
template <int TYPE, bool BF>
__global__ __launch_bounds__(256) void paged_gather_kernel(const PagedGather p) {
  constexpr int N = 8;
  const PagedRows& rows = p.rows;
  const uint32_t b = blockIdx.z, j = blockIdx.y, lane = threadIdx.x & 63;
  const uint32_t sixteen = __builtin_amdgcn_readfirstlane(blockIdx.x * 2 + (threadIdx.x >> 7));
  const bool second = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6 & 1);  // V
  const uint32_t first = __builtin_amdgcn_readfirstlane(p.first ? (uint32_t)max(p.first[b], 0) : 0u);
  const uint32_t len = __builtin_amdgcn_readfirstlane(paged_len(rows, b));
  const uint32_t r0 = sixteen * 16 + (first & ~15u);
  if (r0 >= len) return;
  uint64_t at;
  const bool there = paged_row(rows, b, j, r0, at);
  const uint32_t d4 = rows.dh / 4, last = min(min(len, first + p.M), r0 + 16);
  // Where row r0 would go; the rows before `first` in its sixteen go nowhere.
  const int64_t out = ((int64_t)(((uint64_t)b * rows.KH + j) * p.M) + r0 - first) * rows.dh;
  uint32_t row[N];
  bool on[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const uint32_t t = i * 64 + lane;
    row[i] = t / d4;
    on[i] = t < 16 * d4 && r0 + row[i] >= first && r0 + row[i] < last;
  }
  auto move = [&](const void* from, const float* scales, void* to) {
    Four<TYPE> x[N];
    float s[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      s[i] = 0.f;
      if (on[i] && there) {
        x[i].load(from, at * rows.dh + (i * 64 + lane) * 4);
        if constexpr (TYPE == STS_PAGES_INT8) s[i] = scales[at + row[i]];
      }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (!on[i]) continue;
      const float4 y = there ? x[i].value(s[i]) : make_float4(0.f, 0.f, 0.f, 0.f);
      const int64_t e = out + (i * 64 + lane) * 4;
      if constexpr (BF) {
        const uint2 z = bf16x4(y);
        __builtin_nontemporal_store(u2{z.x, z.y}, reinterpret_cast<u2*>(static_cast<uint16_t*>(to) + e));
      } else {
        __builtin_nontemporal_store(f4{y.x, y.y, y.z, y.w}, reinterpret_cast<f4*>(static_cast<float*>(to) + e));
      }
    }
  };
  move(second ? rows.v : rows.k, second ? rows.vs : rows.ks, second ? p.v_out : p.k_out);
}

}  // namespace

int launch_paged_append(const PagedAppend& p, uint32_t batch, hipStream_t stream) {
  const uint32_t total = batch * p.T * p.rows.KH;
  const bool narrow = p.rows.dh <= 64;
  const uint32_t per = narrow ? 16 : 8;
  const dim3 grid((total + per - 1) / per), block(256);
  auto go = [&](auto type) {
    constexpr int TYPE = decltype(type)::value;
    if (narrow)
      hipLaunchKernelGGL((paged_append_kernel<TYPE, 16>), grid, block, 0, stream, p, total);
    else
      hipLaunchKernelGGL((paged_append_kernel<TYPE, 32>), grid, block, 0, stream, p, total);
  };
  if (p.rows.type == STS_PAGES_F32) go(std::integral_constant<int, STS_PAGES_F32>{});
  else if (p.rows.type == STS_PAGES_BF16) go(std::integral_constant<int, STS_PAGES_BF16>{});
  else go(std::integral_constant<int, STS_PAGES_INT8>{});
  STS_HIP(hipGetLastError());
  return STS_OK;
}

int launch_paged_gather(const PagedGather& p, uint32_t batch, hipStream_t stream) {
  // Sixteens of the longest stream, or of the caches where those are shorter (one more where
  // a stream's first row lies inside one).
  const uint32_t most = p.rows.max_rows < p.M ? p.rows.max_rows : p.M;
  const dim3 grid(((most + 15) / 16 + (p.first ? 1 : 0) + 1) / 2, p.rows.KH, batch), block(256);
  auto go = [&](auto type) {
    constexpr int TYPE = decltype(type)::value;
    if (p.bf16)
      hipLaunchKernelGGL((paged_gather_kernel<TYPE, true>), grid, block, 0, stream, p);
    else
      hipLaunchKernelGGL((paged_gather_kernel<TYPE, false>), grid, block, 0, stream, p);
  };
  if (p.rows.type == STS_PAGES_F32) go(std::integral_constant<int, STS_PAGES_F32>{});
  else if (p.rows.type == STS_PAGES_BF16) go(std::integral_constant<int, STS_PAGES_BF16>{});
  else go(std::integral_constant<int, STS_PAGES_INT8>{});
  STS_HIP(hipGetLastError());
  return STS_OK;
}

}  // namespace sts
