// ring_rows.hip -- rows of the K/V ring moved about: the rows of a draft written,
// its accepted path made the window's end, and windows cut down to the rows that
// got most of the attention.  HBM-bound copies; the eviction's choice of rows is
// a radix selection per (stream, K/V head).
#include <algorithm>

#include "coherent.hpp"
#include "common.hpp"
#include "rope.hpp"
#include "window.hpp"

namespace sts {

namespace {

// A window's length and first slot: device arrays, clamped, or uniform values.
struct Span {
  uint32_t len, start;
};
__device__ __forceinline__ Span span_of(const int32_t* lens, const int32_t* starts, uint32_t len,
                                        uint32_t start, uint32_t M, uint32_t b) {
  Span s{len, start};
  if (lens) {
    const int32_t L = lens[b];
    s.len = L <= 0 ? 0u : min((uint32_t)L, M);
    const int32_t st = starts[b] % (int32_t)M;
    s.start = (uint32_t)(st < 0 ? st + (int32_t)M : st);
  }
  return s;
}

__device__ __forceinline__ uint32_t slot_of(Span s, uint32_t row, uint32_t M) {
  const uint32_t x = s.start + row;
  return x >= M ? x - M : x;
}

// Four floats rounded to bf16 (nearest even), packed as 8 bytes.
__device__ __forceinline__ uint2 bf16x4(float4 x) {
  typedef __bf16 b4 __attribute__((ext_vector_type(4)));
  const b4 y = {(__bf16)x.x, (__bf16)x.y, (__bf16)x.z, (__bf16)x.w};
  return __builtin_bit_cast(uint2, y);
}

// One thread per 4 elements of k_new / v_new [n][KH][4*D4]: the row of node i to
// slot (pos + i) % M, K rotated at the node's depth below the window's end.
__global__ __launch_bounds__(256) void tree_append_kernel(
    const float4* __restrict__ k_in, const float4* __restrict__ v_in,
    const int32_t* __restrict__ parents, float4* __restrict__ k, float4* __restrict__ v,
    uint2* __restrict__ k16, uint2* __restrict__ v16, const float2* __restrict__ cos_t,
    const float2* __restrict__ sin_t, uint32_t rope_pos, uint32_t pos, uint32_t n, uint32_t KH,
    uint32_t D4, uint32_t M) {
  __shared__ int s_up[kMaxTreeNodes];
  for (uint32_t i = threadIdx.x; i < n; i += 256) {
    const int up = parents[i];
    s_up[i] = up < 0 || up >= (int)i ? -1 : up;
  }
  __syncthreads();
  const uint32_t x = blockIdx.x * 256 + threadIdx.x;
  if (x >= n * KH * D4) return;
  const uint32_t d4 = x % D4, h = x / D4 % KH, i = x / D4 / KH;
  const uint32_t slot = (uint32_t)(((uint64_t)pos + i) % M);
  const size_t dst = ((size_t)h * M + slot) * D4 + d4;
  float4 kr = k_in[x];
  const float4 vr = v_in[x];
  if (cos_t) {
    uint32_t at = rope_pos;
    for (int j = s_up[i]; j >= 0; j = s_up[j]) ++at;  // parents come first: the walk ends
    const size_t row = (size_t)at * D4 + d4;
    kr = rope4(kr, cos_t[row], sin_t[row]);
  }
  k[dst] = kr;
  v[dst] = vr;
  if (k16) {
    k16[dst] = bf16x4(kr);
    v16[dst] = bf16x4(vr);
  }
}

// Row base + path[j] to row base + j for every accepted j with j < path[j] < n,
// of one column of the rows, eight rows at a time.  A row is read before
// anything is written over it: the rows written so far lie below every row still
// to be read.
template <typename T>
__device__ __forceinline__ void commit_column(const TreeCommit& p, T* rows, uint32_t cols, uint32_t b) {
  const Span s = span_of(p.lens, p.starts, p.len, p.start, p.M, b);
  uint32_t n = min(p.T, s.len);
  if (p.counts) n = p.counts[b] <= 0 ? 0u : min((uint32_t)p.counts[b], n);
  uint32_t take = p.n;
  if (p.accepted) take = p.accepted[b] <= 0 ? 0u : (uint32_t)p.accepted[b];
  take = min(take, n);
  const uint32_t base = s.len - n;
  for (uint32_t j0 = 0; j0 < take; j0 += 8) {
    T x[8];
    bool move[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t j = j0 + k;
      move[k] = false;
      if (j < take) {
        const int from = p.path ? p.path[(size_t)b * p.T + j] : (int)p.path_host[j];
        move[k] = from > (int)j && from < (int)n;
        if (move[k]) x[k] = rows[(size_t)slot_of(s, base + (uint32_t)from, p.M) * cols];
      }
    }
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (move[k]) rows[(size_t)slot_of(s, base + j0 + k, p.M) * cols] = x[k];
  }
}

// A thread per 8-byte column of a (stream, K/V head, buffer), and one for the
// head's weights.
__global__ __launch_bounds__(64) void tree_commit_kernel(const TreeCommit p) {
  const uint32_t nbuf = p.nbuf + (p.weights != nullptr);
  const uint32_t which = blockIdx.z % nbuf, b = blockIdx.z / nbuf;
  const size_t unit = (size_t)b * p.KH + blockIdx.y;
  const uint32_t c = blockIdx.x * 64 + threadIdx.x;
  if (which == p.nbuf) {
    if (c == 0) commit_column(p, p.weights + unit * p.M, 1, b);
    return;
  }
  const uint32_t cols = p.dh * p.size[which] / 8;
  if (c < cols) commit_column(p, static_cast<uint2*>(p.buf[which]) + unit * p.M * cols + c, cols, b);
}

// ---- eviction ----------------------------------------------------------------

constexpr int kSelThreads = 1024;

// Weights as integers in their order, the largest first in descending order: NaN
// above all, both zeros the same.
__device__ __forceinline__ uint32_t order_key(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t x = __float_as_uint(w + 0.f);
  return x & 0x80000000u ? ~x : x | 0x80000000u;
}

// Sum of `x` over the workgroup's lower threads, and over all of them.
__device__ __forceinline__ uint32_t scan(uint32_t x, uint32_t* s_wave, uint32_t& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t upto = x;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const uint32_t y = __shfl_up(upto, d, 64);
    upto += lane >= d ? y : 0;
  }
  if (lane == 63) s_wave[wave] = upto;
  __syncthreads();
  uint32_t before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kSelThreads / 64; ++w) {
    const uint32_t c = s_wave[w];
    before += w < wave ? c : 0;
    total += c;
  }
  __syncthreads();
  return before + upto - x;
}

// Which window rows stay, for one (stream, K/V head): the `recent` newest, and of
// the others the `keep - recent` of largest weight, the oldest first among equals.
// The least key that stays is found a byte at a time from the top.  A thread looks
// after kPer rows in a row of each run of kSelThreads * kPer; windows of one run
// (SMALL: max_len 4096 or less) keep their keys in registers, and their weights are
// moved here, all of them having been read: at 3000 rows of 32 heads that and the
// scans over runs instead of single rows take 9 us, reading them for every byte 11.
template <bool SMALL>
__global__ __launch_bounds__(kSelThreads) void evict_select_kernel(const Evict p) {
  constexpr int kPer = 4, kRun = kSelThreads * kPer;
  __shared__ uint32_t s_hist[4][256];  // one for each byte
  __shared__ uint32_t s_pick[4][2];    // the byte taken, and how many of it are wanted
  __shared__ uint32_t s_wave[kSelThreads / 64];
  const uint32_t h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  const Span s = span_of(p.lens, p.starts, p.len, p.start, p.M, b);
  int32_t* kept = p.kept + ((size_t)b * p.KH + h) * p.keep;
  if (s.len <= p.keep) {
    for (uint32_t j = tid; j < p.keep; j += kSelThreads) kept[j] = j < s.len ? (int32_t)j : -1;
    return;
  }
  const uint32_t old = s.len - p.recent;
  uint32_t want = p.keep - p.recent;  // < old
  const uint32_t total_want = want;
  for (uint32_t j = tid; j < p.recent; j += kSelThreads) kept[want + j] = (int32_t)(old + j);
  if (want == 0) return;
  float* w = p.weights + ((size_t)b * p.KH + h) * p.M;
  float mine[kPer];  // the weights of rows r0 + kPer*tid .. of a run
  auto read_run = [&](uint32_t r0) {
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const uint32_t r = r0 + tid * kPer + k;
      mine[k] = r < old ? w[slot_of(s, r, p.M)] : 0.f;
    }
  };
  if (SMALL) read_run(0);
  s_hist[tid >> 8][tid & 255] = 0;
  __syncthreads();
  uint32_t prefix = 0;
#pragma unroll
  for (int byte = 0; byte < 4; ++byte) {
    const int shift = 24 - 8 * byte;
    const uint32_t above = shift == 24 ? 0 : 0xffffffffu << (shift + 8);
    for (uint32_t r0 = 0; r0 < (SMALL ? 1 : old); r0 += kRun) {
      if (!SMALL) read_run(r0);
#pragma unroll
      for (int k = 0; k < kPer; ++k) {
        const uint32_t key = order_key(mine[k]);
        if (r0 + tid * kPer + k < old && (key & above) == prefix) atomicAdd(&s_hist[byte][key >> shift & 255], 1u);
      }
    }
    __syncthreads();
    if (tid < 64) {
      // Lane x holds the bins 255-4x .. 252-4x, largest first; the bin in which
      // the running count reaches `want` is taken.
      uint32_t c[4], sum = 0;
      for (int k = 0; k < 4; ++k) sum += c[k] = s_hist[byte][255 - 4 * tid - k];
      uint32_t upto = sum;
      for (int x = 1; x < 64; x *= 2) {
        const uint32_t y = __shfl_up(upto, x, 64);
        upto += (int)tid >= x ? y : 0;
      }
      uint32_t run = upto - sum;
      for (int k = 0; k < 4; ++k) {
        if (run < want && run + c[k] >= want) {
          s_pick[byte][0] = 255 - 4 * tid - k;
          s_pick[byte][1] = want - run;
        }
        run += c[k];
      }
    }
    __syncthreads();
    prefix |= s_pick[byte][0] << shift;
    want = s_pick[byte][1];
  }
  // Rows above the least key stay, and the oldest `want` rows that equal it.
  uint32_t placed = 0, equal = 0;
  for (uint32_t r0 = 0; r0 < old && placed < total_want; r0 += kRun) {
    if (!SMALL) read_run(r0);
    uint32_t total, same = 0;
#pragma unroll
    for (int k = 0; k < kPer; ++k) same += r0 + tid * kPer + k < old && order_key(mine[k]) == prefix;
    uint32_t rank = equal + scan(same, s_wave, total);
    equal += total;
    bool stays[kPer];
    uint32_t count = 0;
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const bool in = r0 + tid * kPer + k < old;
      const uint32_t key = order_key(mine[k]);
      stays[k] = in && (key > prefix || (key == prefix && rank < want));
      rank += in && key == prefix;
      count += stays[k];
    }
    uint32_t at = placed + scan(count, s_wave, total);
    placed += total;
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      if (!stays[k]) continue;
      kept[at] = (int32_t)(r0 + tid * kPer + k);
      if (SMALL) w[slot_of(s, s.len - p.keep + at, p.M)] = mine[k];
      ++at;
    }
  }
}

constexpr int kMoveThreads = 256;
constexpr int kMoveDeep = 8;  // loads of a wave in a batch, two batches in flight (16: 33 us for 29)

// The kept rows moved to the window's end, the last ones first: row kept[j] to row
// len - keep + j, for one slice of the rows (LANES lanes of T), by one wave.  A load
// instruction takes 64 / LANES rows from the highest j down, the stores follow in
// the loads' order.  Nothing is read after it was overwritten: a row lies at or
// below the place it goes to, so the rows that a store overwrites are those of the
// same or of earlier loads, which have returned.  Waves need nothing of one another.
template <typename T>
__device__ __forceinline__ void move_rows(char* head, uint32_t row_bytes, uint32_t lanes, uint32_t slice, Span s,
                                          const int32_t* kept, uint32_t keep, uint32_t moved, uint32_t M) {
  constexpr uint32_t kNone = 0x80000000u;  // past the buffer: loads zeros, stores nothing
  const uint32_t lane = threadIdx.x & 63, per = 64 / lanes;
  const uint32_t col = (slice * lanes + lane % lanes) * sizeof(T), sub = lane / lanes;
  const bool on = col < row_bytes;
  const uint32_t gone = s.len - keep;
  const __amdgpu_buffer_rsrc_t rs = coherent_rsrc(head, M * row_bytes);
  struct Batch {
    T x[kMoveDeep];
    uint32_t to[kMoveDeep];
  } one, two;
  int from[kMoveDeep];
  auto indices = [&](uint32_t done) {
#pragma unroll
    for (int k = 0; k < kMoveDeep; ++k) {
      const uint32_t back = done + k * per + sub;  // counted from the last row that moves
      from[k] = back < moved ? kept[moved - 1 - back] : -1;
    }
  };
  auto load = [&](Batch& b, uint32_t done) {
#pragma unroll
    for (int k = 0; k < kMoveDeep; ++k) {
      const uint32_t back = done + k * per + sub;
      const bool move = on && from[k] >= 0;
      const uint32_t off = move ? slot_of(s, (uint32_t)from[k], M) * row_bytes + col : kNone;
      b.to[k] = move ? slot_of(s, gone + moved - 1 - back, M) * row_bytes + col : kNone;
      if constexpr (sizeof(T) == 16)
        b.x[k] = __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b128(rs, off, 0, 0));
      else if constexpr (sizeof(T) == 8)
        b.x[k] = __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b64(rs, off, 0, 0));
      else
        b.x[k] = __builtin_amdgcn_raw_buffer_load_b32(rs, off, 0, 0);
    }
  };
  auto store = [&](const Batch& b) {
#pragma unroll
    for (int k = 0; k < kMoveDeep; ++k) {
      if constexpr (sizeof(T) == 16)
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(coh_u4, b.x[k]), rs, b.to[k], 0, 0);
      else if constexpr (sizeof(T) == 8)
        __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(coh_u2, b.x[k]), rs, b.to[k], 0, 0);
      else
        __builtin_amdgcn_raw_buffer_store_b32(b.x[k], rs, b.to[k], 0, 0);
    }
  };
  const uint32_t step = per * kMoveDeep;
  indices(0);
  load(one, 0);
  indices(step);
  for (uint32_t done = 0; done < moved; done += 2 * step) {
    load(two, done + step);
    indices(done + 2 * step);
    __builtin_amdgcn_sched_barrier(0);
    store(one);
    __builtin_amdgcn_sched_barrier(0);
    load(one, done + 2 * step);
    indices(done + 3 * step);
    __builtin_amdgcn_sched_barrier(0);
    store(two);
    __builtin_amdgcn_sched_barrier(0);
  }
}

// A wave per slice of a (stream, K/V head, buffer), and one for the head's weights
// where the selection left them (with_weights).
__global__ __launch_bounds__(kMoveThreads) void evict_move_kernel(const Evict p, uint32_t slices, uint32_t lanes,
                                                                  bool with_weights) {
  const uint32_t job = blockIdx.x * (kMoveThreads / 64) + threadIdx.x / 64;
  const uint32_t which = job / slices, slice = job % slices;
  const uint32_t h = blockIdx.y, b = blockIdx.z;
  const Span s = span_of(p.lens, p.starts, p.len, p.start, p.M, b);
  if (s.len <= p.keep) return;
  const uint32_t moved = p.keep - p.recent;  // the newest rows are in place
  const size_t unit = (size_t)b * p.KH + h;
  const int32_t* kept = p.kept + unit * p.keep;
  if (which >= p.nbuf) {
    if (which == p.nbuf && slice == 0 && with_weights)
      move_rows<uint32_t>(reinterpret_cast<char*>(p.weights + unit * p.M), 4, 1, 0, s, kept, p.keep, moved, p.M);
    return;
  }
  const uint32_t bytes = p.dh * p.size[which];
  char* head = static_cast<char*>(p.buf[which]) + unit * p.M * bytes;
  if (bytes % 16 == 0)
    move_rows<uint4>(head, bytes, lanes, slice, s, kept, p.keep, moved, p.M);
  else  // (the bf16 copy of an odd head dim: twice the lanes, at most 32)
    move_rows<uint2>(head, bytes, 2 * lanes, slice, s, kept, p.keep, moved, p.M);
}

}  // namespace

int launch_tree_append(const float* k_new, const float* v_new, const int32_t* parents, float* k,
                       float* v, uint16_t* k16, uint16_t* v16, const float* cos_t,
                       const float* sin_t, uint32_t rope_pos, uint32_t pos, uint32_t n,
                       uint32_t KH, uint32_t dh, uint32_t M, hipStream_t stream) {
  const uint32_t total = n * KH * (dh / 4);
  hipLaunchKernelGGL(tree_append_kernel, dim3((total + 255) / 256), dim3(256), 0, stream,
                     reinterpret_cast<const float4*>(k_new), reinterpret_cast<const float4*>(v_new),
                     parents, reinterpret_cast<float4*>(k), reinterpret_cast<float4*>(v),
                     reinterpret_cast<uint2*>(k16), reinterpret_cast<uint2*>(v16),
                     reinterpret_cast<const float2*>(cos_t), reinterpret_cast<const float2*>(sin_t),
                     rope_pos, pos, n, KH, dh / 4, M);
  STS_HIP(hipGetLastError());
  return STS_OK;
}

int launch_tree_commit(const TreeCommit& p, uint32_t batch, hipStream_t stream) {
  uint32_t cols = 0;
  for (uint32_t i = 0; i < p.nbuf; ++i) cols = std::max(cols, p.dh * p.size[i] / 8);
  const dim3 grid((cols + 63) / 64, p.KH, batch * (p.nbuf + (p.weights != nullptr)));
  hipLaunchKernelGGL(tree_commit_kernel, grid, dim3(64), 0, stream, p);
  STS_HIP(hipGetLastError());
  return STS_OK;
}

int launch_evict(const Evict& p, uint32_t batch, hipStream_t stream) {
  const bool small = p.M <= 4 * kSelThreads;
  if (small)
    hipLaunchKernelGGL(evict_select_kernel<true>, dim3(p.KH, batch), dim3(kSelThreads), 0, stream, p);
  else
    hipLaunchKernelGGL(evict_select_kernel<false>, dim3(p.KH, batch), dim3(kSelThreads), 0, stream, p);
  STS_HIP(hipGetLastError());
  if (p.keep == p.recent) return STS_OK;  // only the newest rows stay, and they are in place
  // Slices of a row of 64 (4 lanes of 16 bytes) to 256 bytes, the wider while there
  // are two waves for every CU (20 streams of 8 heads 83 us, with eight 94; one of 32
  // takes 64 bytes either way, 29 us, with 128 41).
  uint32_t bytes = 0;
  for (uint32_t i = 0; i < p.nbuf; ++i) bytes = std::max(bytes, p.dh * p.size[i]);
  const uint64_t units = (uint64_t)batch * p.KH * p.nbuf;
  uint32_t lanes = 16;
  auto slices_of = [&](uint32_t l) { return (bytes + 16 * l - 1) / (16 * l); };
  while (lanes > 4 && units * slices_of(lanes) < 2 * (uint64_t)device_cu_count()) lanes /= 2;
  const uint32_t slices = slices_of(lanes), jobs = p.nbuf * slices + !small;
  hipLaunchKernelGGL(evict_move_kernel, dim3((jobs + 3) / 4, p.KH, batch), dim3(kMoveThreads), 0, stream, p, slices,
                     lanes, !small);
  STS_HIP(hipGetLastError());
  return STS_OK;
}

}  // namespace sts
