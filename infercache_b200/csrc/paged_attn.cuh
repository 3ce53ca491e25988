// What the two paged-attention kernels share: the call's parameters, the
// sessions' row counts, tensor maps over 8-bit pages.
#pragma once

#include <algorithm>

#include "common.cuh"
#include "q8.cuh"

namespace ic {
namespace paged {

constexpr int MAX_SESSIONS = 4096;  // the sessions' prefix sums fit in 16 KB of shared memory
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;

struct Params {
  const void* q;
  const void* k;              // codes of the layer
  const void* v;
  void* out;
  float* lse;                 // may be null
  const int32_t* table;
  const int32_t* lens;
  const int32_t* q_start;
  const float* k_scale;
  const float* v_scale;
  float* ws;
  int32_t* status;
  int64_t q_stride_t, q_stride_h;
  int32_t S, width, Hq, H, G, n_pages;
  int32_t n_q;                // rows of q: sessions are clipped to them
  int32_t few_rows;           // sessions with at most this many rows are the streaming kernel's, the others the tile kernel's
  int32_t cluster;            // streaming kernel: CTAs per group where each has a cluster
  float sl2;                  // scale * log2(e)
};

// Query tokens of session s and where they begin, clipped to the rows of q.
__device__ __forceinline__ int query_tokens(const Params& p, int s, int& begin) {
  begin = min(max(p.q_start[s], 0), p.n_q);
  return max(0, min(p.q_start[s + 1], p.n_q) - begin);
}
// Tokens that session s holds, clipped to its table row.
__device__ __forceinline__ int held_tokens(const Params& p, int s) {
  const int64_t cap = static_cast<int64_t>(p.width) * q8::PAGE;
  return static_cast<int>(min(static_cast<int64_t>(max(p.lens[s], 0)), cap));
}

// Tensor map of codes [H, pool_tokens, D] as 128-byte lines, one box per page
// (D = 64: two tokens per line; D = 256: two boxes per page), 128-byte swizzle:
// 16-byte chunk c of line r is stored at chunk c ^ (r % 8).
int page_map(CUtensorMap* m, const void* codes, int64_t pool_tokens, int heads, int D);

// What Params::few_rows is for a call; ALL_ROWS: everything is the streaming kernel's.
constexpr int ALL_ROWS = 0x7fffffff;
int few_rows(const ic_paged_attn_args& a);

int launch_stream(const Params& p, const ic_paged_attn_args& a, cudaStream_t st);
int launch_tile(const Params& p, const ic_paged_attn_args& a, cudaStream_t st);
// Rows per tile of the streaming kernel, 8 or 16.  16 read the pages half as
// often but cost registers, hence warps, so they pay where they halve the number
// of tiles: not up to 8 rows a session, nor, up to 128 dims, for 17 to 24, which
// make three tiles or two.  Measured with 8 and with 16: 24 sessions x up to 4k
// tokens x 2 heads, 24 rows, 128 dims 22.8 / 24.8 us, 24 x 1400 x 4 heads 19.2 /
// 25.2 (64 dims 15.5 / 18.4, but 64 sessions of 8k 102 / 90); at 256 dims 24 rows
// of 64 sessions of 8k 296 / 253; 16 rows of those at 128 dims 112 / 92.
inline int stream_rows(int64_t max_rows, int head_dim) {
  return max_rows <= 8 || (max_rows > 16 && max_rows <= 24 && head_dim <= 128) ? 8 : 16;
}
int64_t stream_workspace(const ic_paged_attn_args& a);  // bytes, 0 when the call needs none

}  // namespace paged
}  // namespace ic
