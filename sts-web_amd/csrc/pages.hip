// pages.hip -- K/V rows into pages and out of them (gfx950).  No counterpart in the
// reference, whose caches are one ring a stream (crates/sts-wasm/src/model.rs:195-363).
//
// Both are copies that round, bound by HBM for many rows and by their launch for few.
#include "common.hpp"
#include "page_rows.hpp"
#include "rope.hpp"

namespace sts {

namespace {

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
    float top = largest(x);
#pragma unroll
    for (int d = 1; d < G; d *= 2) top = __builtin_elementwise_maximum(top, __shfl_xor(top, d, G));
    const float s = row_scale(top);
    const uint32_t codes = row_codes(x, s);
    if (on) *reinterpret_cast<uint32_t*>(static_cast<int8_t*>(rows) + to) = codes;
    if (on && c == 0) scales[at] = s;
  }
}

// G lanes a row (K and V of it), 256 / G rows a workgroup.
template <int TYPE, int G>
__global__ __launch_bounds__(256) void paged_append_kernel(const PagedAppend p, uint64_t total) {
  const PagedRows& rows = p.rows;
  const int c = threadIdx.x % G;
  const uint64_t n = (uint64_t)blockIdx.x * (256 / G) + threadIdx.x / G;
  if (n >= total) return;  // (whole groups of G lanes)
  const uint32_t j = (uint32_t)(n % rows.KH);
  const uint64_t bt = n / rows.KH;
  const uint32_t i = (uint32_t)(bt % p.T), b = (uint32_t)(bt / p.T);
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

// Four values of row `at` from dim d on.
template <int TYPE>
struct Four {
  float4 x;
  uint2 h;
  uint32_t w;
  float s;
  __device__ __forceinline__ void load(const void* rows, const float* scales, uint64_t at, uint32_t dh, uint32_t d) {
    if constexpr (TYPE == STS_PAGES_F32) x = *reinterpret_cast<const float4*>(static_cast<const float*>(rows) + at * dh + d);
    else if constexpr (TYPE == STS_PAGES_BF16)
      h = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(rows) + at * dh + d);
    else {
      w = *reinterpret_cast<const uint32_t*>(static_cast<const int8_t*>(rows) + at * dh + d);
      s = scales[at];
    }
  }
  __device__ __forceinline__ float4 value() const {
    if constexpr (TYPE == STS_PAGES_F32) return x;
    else if constexpr (TYPE == STS_PAGES_BF16)
      return make_float4(__uint_as_float(h.x << 16), __uint_as_float(h.x & 0xffff0000u), __uint_as_float(h.y << 16),
                         __uint_as_float(h.y & 0xffff0000u));
    else
      return make_float4((float)(int8_t)w * s, (float)(int8_t)(w >> 8) * s, (float)(int8_t)(w >> 16) * s,
                         (float)(int8_t)(w >> 24) * s);
  }
};

constexpr uint32_t kGatherRows = 32;  // rows of a workgroup

// One workgroup takes kGatherRows rows of one stream and head.
template <int TYPE, bool BF>
__global__ __launch_bounds__(256) void paged_gather_kernel(const PagedGather p) {
  const PagedRows& rows = p.rows;
  const uint32_t b = blockIdx.z, j = blockIdx.y;
  const uint32_t len = paged_len(rows, b);
  const uint32_t first = p.first ? (uint32_t)max(p.first[b], 0) : 0u;
  const uint32_t r0 = blockIdx.x * kGatherRows + (first & ~(kGatherRows - 1));
  if (r0 >= len) return;
  const uint32_t d4 = rows.dh / 4;
  const uint64_t out = ((uint64_t)b * rows.KH + j) * p.M;
  for (uint32_t t = threadIdx.x; t < kGatherRows * d4; t += 256) {
    const uint32_t r = r0 + t / d4, d = t % d4 * 4;
    if (r < first || r >= len || r - first >= p.M) continue;
    uint64_t at;
    float4 k = make_float4(0.f, 0.f, 0.f, 0.f), v = k;
    if (paged_row(rows, b, j, r, at)) {
      Four<TYPE> a, z;
      a.load(rows.k, rows.ks, at, rows.dh, d);
      z.load(rows.v, rows.vs, at, rows.dh, d);
      k = a.value();
      v = z.value();
    }
    const uint64_t to = (out + (r - first)) * rows.dh + d;
    if constexpr (BF) {
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.k_out) + to) = bf16x4(k);
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.v_out) + to) = bf16x4(v);
    } else {
      *reinterpret_cast<float4*>(static_cast<float*>(p.k_out) + to) = k;
      *reinterpret_cast<float4*>(static_cast<float*>(p.v_out) + to) = v;
    }
  }
}

}  // namespace

int launch_paged_append(const PagedAppend& p, uint32_t batch, hipStream_t stream) {
  const uint64_t total = (uint64_t)batch * p.T * p.rows.KH;
  const bool narrow = p.rows.dh <= 64;
  const dim3 grid((uint32_t)((total + (narrow ? 15 : 7)) / (narrow ? 16 : 8))), block(256);
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
  // Rows of the longest stream, or of the caches where those are shorter (a block more
  // where a stream's first row lies inside one).
  const uint32_t most = p.rows.max_rows < p.M ? p.rows.max_rows : p.M;
  const dim3 grid((most + kGatherRows - 1) / kGatherRows + (p.first ? 1 : 0), p.rows.KH, batch), block(256);
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
