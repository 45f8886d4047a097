// window.hip -- launch plans of the window attention kernels, and the account of
// the attention weights that sts_decode_ring_weights keeps.
#include <algorithm>

#include "window_kernel.hpp"

namespace sts {

namespace {


// The rows' weights under every query head of a K/V head's group, from their kept
// scores, added to their accounts: a thread takes kAccountRows rows, 256 apart, so
// that its requests go out together (64 streams of 32 heads over 128 to 3000 rows: one
// row a thread 23 us, four 10).
constexpr int kAccountRows = 4;
__global__ __launch_bounds__(256) void account_kernel(const WindowParams p, float* __restrict__ weights,
                                                      bool fresh) {
  const uint32_t r0 = blockIdx.x * (256 * kAccountRows) + threadIdx.x;
  const uint32_t b = blockIdx.z;
  uint32_t len = p.len, start = p.start;
  if (p.lens) {
    const int32_t L = p.lens[b];
    len = L <= 0 ? 0u : min((uint32_t)L, p.M);
    const int32_t st = p.starts[b] % (int32_t)p.M;
    start = (uint32_t)(st < 0 ? st + (int32_t)p.M : st);
  }
  if (r0 >= len) return;
  const size_t h0 = (size_t)b * p.H + blockIdx.y * p.group;
  float* w = weights + ((size_t)b * p.KH + blockIdx.y) * p.M;
  uint32_t slot[kAccountRows];
  float had[kAccountRows], sum[kAccountRows];
#pragma unroll
  for (int k = 0; k < kAccountRows; ++k) {
    const uint32_t r = r0 + 256 * k;
    slot[k] = start + r;
    slot[k] = slot[k] >= p.M ? slot[k] - p.M : slot[k];
    had[k] = r < len ? w[slot[k]] : 0.f;
    sum[k] = 0.f;
  }
  for (uint32_t h = 0; h < p.group; ++h) {
    const float m = p.stats[(h0 + h) * 2], l = p.stats[(h0 + h) * 2 + 1];
#pragma unroll
    for (int k = 0; k < kAccountRows; ++k) {
      const uint32_t r = r0 + 256 * k;
      if (r < len) sum[k] += exp2_hw(p.scores[(h0 + h) * p.score_stride + r] - m) / l;
    }
  }
#pragma unroll
  for (int k = 0; k < kAccountRows; ++k) {
    const uint32_t r = r0 + 256 * k;
    if (r < len) w[slot[k]] = fresh && r == len - 1 ? sum[k] : had[k] + sum[k];
  }
}

__global__ __launch_bounds__(256) void clear_weights_kernel(float* weights, uint64_t units, uint32_t M,
                                                            uint32_t pos, uint32_t n) {
  const uint32_t s = blockIdx.x * 256 + threadIdx.x;
  if (s >= n) return;
  const uint32_t slot = (uint32_t)(((uint64_t)pos + s) % M);
  for (uint64_t u = blockIdx.y; u < units; u += gridDim.y) weights[u * M + slot] = 0.f;
}

struct WindowPlan {
  int row_tiles = 1;
  uint32_t rblocks = 1, nsplit = 1;
  size_t record = 0;  // floats of a split's record
  uint32_t shares = 0;
  float rows_factor = 0.f;
};

WindowPlan plan_window(const WindowParams& p, WindowMode mode, uint32_t batch, bool bf16, uint32_t max_rows) {
  WindowPlan pl;
  const uint32_t rows = p.T * p.group;
  pl.row_tiles = rows <= 16 ? 1 : 2;
  const uint32_t per = 16u * pl.row_tiles;
  pl.rblocks = (rows + per - 1) / per;
  const uint64_t units = (uint64_t)batch * p.KH * pl.rblocks;
  // One row tile is bound by the reads: as many workgroups as keep 64 KB of rows
  // requested on each CU (f32 rows of 128 one, bf16 rows of 64 four; at 7 streams of
  // 20011 such rows 52 us against 102 with one).  Two are bound by their products:
  // two workgroups, what a CU holds at once (a draft of 60 over 3000 rows 37 us, with
  // four 54; 24 drafts of 40 nodes 202 and 200).
  const uint32_t tile = pl.row_tiles > 1 || bf16 ? 32 : 16;
  const uint32_t wide = p.dh <= 64 ? 64 : 128;
  const uint32_t tile_bytes = 2 * tile * wide * (bf16 ? 2 : 4) * window::kWaves;
  const uint32_t per_cu = pl.row_tiles > 1 ? 2 : std::min(4u, std::max(1u, 65536 / tile_bytes));
  const uint64_t target = (uint64_t)device_cu_count() * per_cu;
  // A split is worth its record from a tile for each of its waves on.
  const uint64_t most = std::min<uint64_t>((max_rows + tile * window::kWaves - 1) / (tile * window::kWaves),
                                           window::max_splits(pl.row_tiles));
  // (The kernel adds up the streams' rows in 32 bits.)
  if ((mode != kWindowMasked || p.T == 1) && batch > 1 && batch <= 64 && (uint64_t)batch * p.M >> 32 == 0) {
    // Streams of different ages: splits of about equal length whatever their stream,
    // not more than fit at once where one round can hold them (rounding up gives each
    // window half a split more).  Products in several rounds end more evenly with
    // splits of half the length (24 streams of 900 to 3000 rows 202 us for 213), reads
    // do not (9 tokens over 700 rows 40 us, with half 49).
    const uint64_t rounds = pl.row_tiles > 1 ? 2 : 1;
    const uint64_t fit = 2 * units <= target ? target - units / 2 : rounds * target;
    const uint64_t heads = (uint64_t)p.KH * pl.rblocks;
    pl.rows_factor = (float)heads / (float)fit;
    pl.nsplit = (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>(fit / heads + 1, most));
    pl.shares = (uint32_t)(p.KH * (fit / heads + batch + 1));
  } else {
    const uint64_t want = std::max<uint64_t>(1, (target + units - 1) / units);
    pl.nsplit = (uint32_t)std::max<uint64_t>(1, std::min(want, most));
    pl.shares = batch * p.KH * pl.nsplit;
  }
  pl.record = (size_t)per * ((p.dh <= 64 ? 64 : 128) + 2);
  return pl;
}

int window_workspace(const WindowParams& p, const WindowPlan& pl, uint32_t batch, hipStream_t stream,
                     Workspace** out) {
  *out = nullptr;
  if (pl.nsplit <= 1) return STS_OK;
  const size_t units = (size_t)batch * p.KH * pl.rblocks;
  return get_workspace(stream, (size_t)pl.shares * pl.rblocks * pl.record, units, out);
}

}  // namespace

int check_window(const WindowParams& p, uint32_t batch, bool bf16) {
  STS_CHECK(batch >= 1 && p.T >= 1 && p.H >= 1 && p.KH >= 1 && p.M >= 1, "empty shape");
  STS_CHECK(p.dh >= 4 && p.dh <= 128 && p.dh % 4 == 0,
            "head_dim %u not supported (a multiple of 4 up to 128)", p.dh);
  STS_CHECK(!bf16 || p.dh % 8 == 0, "bf16 K/V rows need a head_dim that is a multiple of 8 (got %u)", p.dh);
  STS_CHECK(p.H % p.KH == 0, "query heads %u not a multiple of the %u K/V heads", p.H, p.KH);
  STS_CHECK((uint64_t)p.M * p.dh * (bf16 ? 2 : 4) <= 0x7FFFFFF0ull,
            "max_len %u too large for one head's buffer resource", p.M);
  STS_CHECK(batch <= 65535 && p.KH <= 65535, "batch (%u) and kv_heads (%u) must be <= 65535", batch, p.KH);
  // (The launch counts its threads in 32 bits: 16 rows of a K/V head and up to 128
  // splits make a workgroup of 256.)
  STS_CHECK((uint64_t)p.T * p.H <= 0x7FFFFFFull &&
                ((uint64_t)p.T * (p.H / p.KH) / 16 + 1) * batch * p.KH <= (1u << 23),
            "too many query rows (%u streams x %u x %u heads)", batch, p.T, p.H);
  return STS_OK;
}

int reserve_window(const WindowParams& p, WindowMode mode, uint32_t batch, bool bf16,
                   uint32_t max_rows, hipStream_t stream) {
  Workspace* ws = nullptr;
  return window_workspace(p, plan_window(p, mode, batch, bf16, max_rows), batch, stream, &ws);
}

int launch_window(WindowParams p, WindowMode mode, uint32_t batch, bool bf16, uint32_t max_rows,
                  hipStream_t stream) {
  if (int rc = check_window(p, batch, bf16)) return rc;
  const WindowPlan pl = plan_window(p, mode, batch, bf16, max_rows);
  Workspace* ws = nullptr;
  if (int rc = window_workspace(p, pl, batch, stream, &ws)) return rc;
  p.rblocks = pl.rblocks;
  p.nsplit = pl.nsplit;
  if (ws) {
    p.part = ws->part;
    p.counters = ws->counters;
  }
  p.shares = pl.shares;
  p.batch = batch;
  p.rows_factor = pl.rows_factor;
  const uint64_t blocks =
      ((uint64_t)p.shares + window::kXcds - 1) / window::kXcds * window::kXcds * (uint64_t)pl.rblocks;
  const dim3 grid((uint32_t)blocks);
  if (mode == kWindowTree) return launch_window_tree(p, pl.row_tiles, bf16, grid, stream);
  if (mode == kWindowMasked) return launch_window_masked(p, pl.row_tiles, bf16, grid, stream);
  return launch_window_weights(p, pl.row_tiles, bf16, grid, stream);
}

int launch_account(const WindowParams& p, float* weights, uint32_t batch, uint32_t max_rows,
                   bool fresh, hipStream_t stream) {
  const dim3 grid((max_rows + 256 * kAccountRows - 1) / (256 * kAccountRows), p.KH, batch);
  hipLaunchKernelGGL(account_kernel, grid, dim3(256), 0, stream, p, weights, fresh);
  STS_HIP(hipGetLastError());
  return STS_OK;
}

int launch_clear_weights(float* weights, uint64_t units, uint32_t M, uint32_t pos, uint32_t n,
                         hipStream_t stream) {
  if (n == 0) return STS_OK;
  const dim3 grid((n + 255) / 256, (uint32_t)std::min<uint64_t>(units, 4096));
  hipLaunchKernelGGL(clear_weights_kernel, grid, dim3(256), 0, stream, weights, units, M, pos, n);
  STS_HIP(hipGetLastError());
  return STS_OK;
}

}  // namespace sts
