// window.hpp -- attention of several query rows per K/V head over a ring
// window: drafted trees, masked chunks, and single tokens whose weights are kept.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace sts {

constexpr uint32_t kMaxTreeNodes = 256;

// Which rows of the window a query sees.
enum WindowMode {
  kWindowTree,    // the committed rows, its ancestors among the drafted ones, itself
  kWindowMasked,  // rows lo..hi-1; capped scores, distance bias
  kWindowWeights  // all of them; the scores are kept
};

// One launch.  Stream b's window has lens[b] rows, row r in slot
// (starts[b] + r) % M of k + (b*KH + j)*M*dh for K/V head j (f32, or bf16 bits);
// query i of its counts[b] (at most T) is window row lens[b] - counts[b] + i,
// and its head h uses K/V head h / group.
struct WindowParams {
  const float* q = nullptr;  // [B][T][H][dh]
  const void* k = nullptr;
  const void* v = nullptr;
  float* out = nullptr;             // [B][T][H][dh]; rows past counts[b] get zeros
  const int32_t* lens = nullptr;    // per-stream device arrays, or null for the
  const int32_t* starts = nullptr;  // uniform len / start below
  const int32_t* counts = nullptr;  // or null: T of every stream
  const int32_t* parents = nullptr; // [B][T] (tree)
  const int32_t* lo = nullptr;      // [B][T] or null (masked)
  const int32_t* hi = nullptr;
  const float* slopes = nullptr;    // [H] or null (masked)
  const float* rope_cos = nullptr;  // [max_pos][dh/2]: query i is rotated at rope_pos
  const float* rope_sin = nullptr;  // (tree: plus its depth) before it is scaled
  uint32_t rope_pos = 0;
  uint32_t len = 0, start = 0;
  uint32_t T = 0, H = 0, KH = 0, M = 0, dh = 0;
  uint32_t group = 1;      // H / KH
  float qscale = 0.f;      // folded into q: scale * log2(e), or scale / cap
  float cap_log2 = 0.f;    // cap * log2(e), 0: no cap
  float* scores = nullptr; // [B][H][score_stride] row scores in units of log2(e) (weights)
  float* stats = nullptr;  // [B][H][2] their maximum and sum of 2^(score - maximum)
  uint32_t score_stride = 0;
  // Set by launch_window.
  uint32_t rblocks = 1, nsplit = 1;
  uint32_t shares = 0;  // streams x K/V heads x splits
  uint32_t batch = 0;
  float rows_factor = 0.f;  // rows of a split for each row there is; 0: nsplit for every stream
  float* part = nullptr;
  uint32_t* counters = nullptr;
};

// Refuses what launch_window cannot run, without launching.
int check_window(const WindowParams& p, uint32_t batch, bool bf16);

// max_rows: the longest window there can be (M, or the uniform length).
int launch_window(WindowParams p, WindowMode mode, uint32_t batch, bool bf16, uint32_t max_rows,
                  hipStream_t stream);

// Makes sure the split workspace launch_window needs for these sizes exists, so
// that a caller can fail before it changes any state.
int reserve_window(const WindowParams& p, WindowMode mode, uint32_t batch, bool bf16,
                   uint32_t max_rows, hipStream_t stream);

// weights[b][j][slot of row r] += sum over the group's heads of
// 2^(score - max) / sum, for the rows of each window; with `fresh` the newest
// row's weight is set instead (its slot held another row before).
int launch_account(const WindowParams& p, float* weights, uint32_t batch, uint32_t max_rows,
                   bool fresh, hipStream_t stream);

// Sets the weights of slots (pos + s) % M, s < n, to zero: [units][M].
int launch_clear_weights(float* weights, uint64_t units, uint32_t M, uint32_t pos, uint32_t n,
                         hipStream_t stream);

// ---- draft rows and eviction (ring_rows.hip) --------------------------------

// Writes the drafted K and V rows [n][KH][dh] to slots (pos + i) % M, K rotated
// at table row rope_pos + depth of node i when cos_t is set, and to the bf16
// copies when k16 is set (batch 1).
int launch_tree_append(const float* k_new, const float* v_new, const int32_t* parents, float* k,
                       float* v, uint16_t* k16, uint16_t* v16, const float* cos_t,
                       const float* sin_t, uint32_t rope_pos, uint32_t pos, uint32_t n,
                       uint32_t KH, uint32_t dh, uint32_t M, hipStream_t stream);

// The accepted path of each stream's draft, moved to the draft's first rows.
struct TreeCommit {
  void* buf[4] = {};               // caches [B][KH][M][dh] of elements of `size` bytes
  uint32_t size[4] = {};
  uint32_t nbuf = 0;
  float* weights = nullptr;        // [B][KH][M], moved along, or null
  const int32_t* lens = nullptr;   // device arrays, or null for the values below
  const int32_t* starts = nullptr;
  const int32_t* counts = nullptr;    // null: T
  const int32_t* path = nullptr;      // [B][T], or null: path_host
  const int32_t* accepted = nullptr;  // [B], or null: n
  uint32_t len = 0, start = 0, n = 0;
  uint8_t path_host[kMaxTreeNodes] = {};
  uint32_t T = 0, KH = 0, dh = 0, M = 0;
};
int launch_tree_commit(const TreeCommit& p, uint32_t batch, hipStream_t stream);

// Eviction by weight: each stream's window cut to `keep` rows.
struct Evict {
  void* buf[4] = {};
  uint32_t size[4] = {};
  uint32_t nbuf = 0;
  float* weights = nullptr;  // [B][KH][M]
  int32_t* kept = nullptr;   // [B][KH][keep] window rows kept, ascending; -1 past a shorter window
  const int32_t* lens = nullptr;
  const int32_t* starts = nullptr;
  uint32_t len = 0, start = 0;
  uint32_t keep = 0, recent = 0, KH = 0, dh = 0, M = 0;
};
int launch_evict(const Evict& p, uint32_t batch, hipStream_t stream);

}  // namespace sts
