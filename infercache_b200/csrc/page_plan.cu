// Block tables and slot maps from request lengths, and the release of
// sessions' pages: the page bookkeeping of a serving tick on the device, so
// that a tick needs no host round trip and can be captured in a graph.
//
// The plan is two prefix sums over the sessions (new tokens, new pages)
// followed by one independent computation per new token.  The sums are one
// CTA's block scans (a few thousand sessions at most take a few passes);
// because that CTA reads every length before anything is written, lens_out may
// alias lens.  Tokens: 12 bytes are written for each and next to nothing is
// read, so a large admission is bound by HBM writes and spreads over the GPU
// in a second kernel, while a decode tick's few tokens are finished by the
// scanning CTA itself (a second launch would cost more than the work).
#include "common.cuh"
#include "launch.cuh"
#include "q8.cuh"

namespace ic {
namespace {

constexpr int PT = 1024;            // threads of the scanning CTA
constexpr int TPT = 8;              // consecutive tokens per thread
// Tokens that the scanning CTA finishes itself: one pass of its threads.
constexpr int FUSED_TOKENS = PT * TPT;

// Inclusive block scan of one int64 per thread; `total` gets the block's sum.
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t* warp_sums, int64_t& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t u = __shfl_up_sync(FULL_MASK, v, o);
    if (lane >= o) v += u;
  }
  if (lane == 31) warp_sums[warp] = v;
  __syncthreads();
  if (warp == 0) {
    int64_t w = lane < static_cast<int>(blockDim.x >> 5) ? warp_sums[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t u = __shfl_up_sync(FULL_MASK, w, o);
      if (lane >= o) w += u;
    }
    warp_sums[lane] = w;
  }
  __syncthreads();
  total = warp_sums[31];
  const int64_t r = v + (warp > 0 ? warp_sums[warp - 1] : 0);
  __syncthreads();  // warp_sums may be written again
  return r;
}

__device__ __forceinline__ int32_t pages_of(int64_t tokens) {
  return static_cast<int32_t>((tokens + q8::PAGE - 1) / q8::PAGE);
}

// One thread's TPT tokens.  work[2s] is session s's length before the call (-1
// when it was denied), work[2s + 1] its first new page's rank, work[2S] the
// stack's height before the call.
__device__ __forceinline__ void plan_tokens(const ic_page_plan_args& a, const int32_t* q_start, const int32_t* work,
                                            int64_t i0) {
  const int S = a.num_sessions;
  const int64_t n = a.total;
  if (i0 >= n) return;
  // the last session with q_start[s] <= i0 (empty sessions before it are skipped)
  int lo = 0, hi = S;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (q_start[mid] <= i0) lo = mid; else hi = mid;
  }
  int s = lo;
  const int32_t top = work[2 * S];
  int32_t slot[TPT];
  int64_t pos[TPT];
  int32_t begin = q_start[s], end = q_start[s + 1], held_len = work[2 * s], rank = work[2 * s + 1];
  int32_t page_at = -1, page = -1;  // the page id last looked up, and its index in the session
#pragma unroll
  for (int j = 0; j < TPT; ++j) {
    const int64_t i = i0 + j;
    while (i >= end && s + 1 < S) {
      ++s;
      begin = end;
      end = q_start[s + 1];
      held_len = work[2 * s];
      rank = work[2 * s + 1];
      page_at = -1;
    }
    slot[j] = -1;
    pos[j] = -1;
    if (i < n && i < end && held_len >= 0) {
      const int64_t p = held_len + (i - begin);
      const int32_t idx = static_cast<int32_t>(p / q8::PAGE), held = pages_of(held_len);
      int32_t* row = a.block_table + static_cast<int64_t>(s) * a.width;
      if (idx != page_at) {
        page = idx < held ? row[idx] : a.free_pages[top - 1 - (rank + idx - held)];
        page_at = idx;
      }
      if (idx >= held && p % q8::PAGE == 0) row[idx] = page;  // a new page's first token enters it
      slot[j] = page < 0 ? -1 : page * q8::PAGE + static_cast<int32_t>(p % q8::PAGE);
      pos[j] = p;
    }
  }
  if (i0 + TPT <= n && (reinterpret_cast<uintptr_t>(a.slots) & 15) == 0 &&
      (reinterpret_cast<uintptr_t>(a.positions) & 15) == 0) {
#pragma unroll
    for (int j = 0; j < TPT; j += 4)
      *reinterpret_cast<int4*>(a.slots + i0 + j) = make_int4(slot[j], slot[j + 1], slot[j + 2], slot[j + 3]);
#pragma unroll
    for (int j = 0; j < TPT; j += 2)
      *reinterpret_cast<longlong2*>(a.positions + i0 + j) = make_longlong2(pos[j], pos[j + 1]);
  } else {
#pragma unroll
    for (int j = 0; j < TPT; ++j)
      if (i0 + j < n) {
        a.slots[i0 + j] = slot[j];
        a.positions[i0 + j] = pos[j];
      }
  }
}

__global__ void __launch_bounds__(PT) plan_rows_kernel(const ic_page_plan_args a, int fused) {
  __shared__ int64_t warp_sums[32];
  grid_dependency_wait();
  grid_launch_dependents();
  const int S = a.num_sessions;
  int32_t top = *a.free_count;
  bool bad = false;
  if (top < 0 || top > a.free_capacity) {
    bad = true;
    top = 0;
  }
  int64_t tokens = 0, pages = 0, taken = 0;
  for (int s0 = 0; s0 < S; s0 += PT) {
    const int s = s0 + threadIdx.x;
    const int64_t len = s < S ? a.lens[s] : 0;
    const int64_t c = s < S ? a.counts[s] : 0;
    int64_t sum;
    const int64_t q_end = tokens + block_scan(c > 0 ? c : 0, warp_sums, sum);
    tokens += sum;
    const bool fits = c >= 0 && len >= 0 && len + c <= static_cast<int64_t>(a.width) * q8::PAGE && q_end <= a.total;
    const int64_t need = fits ? pages_of(len + c) - pages_of(len) : 0;
    const int64_t upto = pages + block_scan(need, warp_sums, sum);
    pages += sum;
    const bool granted = fits && (need == 0 || upto <= top);
    block_scan(granted ? need : 0, warp_sums, sum);
    taken += sum;
    if (s < S) {
      a.q_start[s + 1] = static_cast<int32_t>(q_end < 0x7fffffff ? q_end : 0x7fffffff);
      a.workspace[2 * s] = granted ? static_cast<int32_t>(len) : -1;
      a.workspace[2 * s + 1] = static_cast<int32_t>(upto - need);
      a.lens_out[s] = static_cast<int32_t>(granted ? len + c : len);
      bad |= !granted;
    }
  }
  if (threadIdx.x == 0) {
    a.q_start[0] = 0;
    a.workspace[2 * S] = top;
    *a.free_count_out = top - static_cast<int32_t>(taken);
  }
  if (__syncthreads_or(bad) && threadIdx.x == 0 && a.dev_status) atomicOr(a.dev_status, IC_DEVFLAG_NO_PAGES);
  if (fused) plan_tokens(a, a.q_start, a.workspace, static_cast<int64_t>(threadIdx.x) * TPT);
}

__global__ void __launch_bounds__(256) plan_tokens_kernel(const ic_page_plan_args a) {
  extern __shared__ int32_t qs[];  // q_start, when it fits
  grid_dependency_wait();
  grid_launch_dependents();
  const int S = a.num_sessions;
  for (int s = threadIdx.x; s <= S; s += blockDim.x) qs[s] = a.q_start[s];
  __syncthreads();
  plan_tokens(a, qs, a.workspace, (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) * TPT);
}

__global__ void __launch_bounds__(PT) release_kernel(const ic_page_release_args a) {
  __shared__ int64_t warp_sums[32];
  grid_dependency_wait();
  grid_launch_dependents();
  const int S = a.num_sessions, lane = threadIdx.x & 31;
  // how many pages in all: the first one goes to the top of the stack
  int64_t total = 0, sum;
  bool bad = false;
  for (int s0 = 0; s0 < S; s0 += PT) {
    const int s = s0 + threadIdx.x;
    const int64_t len = s < S ? a.lens[s] : 0, keep = s < S ? a.keep[s] : 0;
    const bool drops = keep >= 0 && keep < len;
    const bool ok = !drops || len <= static_cast<int64_t>(a.width) * q8::PAGE;
    bad |= !ok;
    block_scan(ok && drops ? pages_of(len) - pages_of(keep) : 0, warp_sums, sum);
    total += sum;
  }
  const int32_t top = *a.free_count;
  if (top < 0 || top + total > a.free_capacity) bad = true;
  if (__syncthreads_or(bad)) {  // nothing is given back from corrupt lengths, or past the stack's end
    if (threadIdx.x == 0 && a.dev_status) atomicOr(a.dev_status, IC_DEVFLAG_BAD_ROW);
    return;
  }
  int64_t before = 0;
  for (int s0 = 0; s0 < S; s0 += PT) {
    const int s = s0 + threadIdx.x;
    const int32_t len = s < S ? a.lens[s] : 0, keep = s < S ? a.keep[s] : 0;
    const bool drops = keep >= 0 && keep < len;
    const int32_t kept = drops ? pages_of(keep) : 0, mine = drops ? pages_of(len) - kept : 0;
    const int64_t first = before + block_scan(mine, warp_sums, sum) - mine;
    before += sum;
    // a warp walks its 32 sessions' pages together
    for (int r = 0; r < 32; ++r) {
      const int32_t n = __shfl_sync(FULL_MASK, mine, r);
      if (n == 0) continue;
      const int64_t f = __shfl_sync(FULL_MASK, first, r);
      int32_t* row = a.block_table + static_cast<int64_t>(s - lane + r) * a.width + __shfl_sync(FULL_MASK, kept, r);
      for (int p = lane; p < n; p += 32) {
        a.free_pages[top + total - 1 - (f + p)] = row[p];
        row[p] = -1;
      }
    }
    if (drops) a.lens[s] = keep;
  }
  __syncthreads();
  if (threadIdx.x == 0) *a.free_count = top + static_cast<int32_t>(total);
}

constexpr int PLAN_MAX_SESSIONS = 8192;  // q_start in 32 KB of shared memory

}  // namespace
}  // namespace ic

extern "C" int ic_page_plan(const ic_page_plan_args* a, void* stream) {
  if (!a || !a->lens || !a->counts || !a->block_table || !a->free_pages || !a->free_count || !a->q_start ||
      !a->lens_out || !a->free_count_out || !a->workspace || (a->total > 0 && (!a->slots || !a->positions)) ||
      a->num_sessions < 1 || a->width < 1 || a->total < 0 || a->free_capacity < 0) {
    ic::set_last_error("page_plan: bad arguments");
    return IC_ERR_INVALID_ARG;
  }
  if (a->num_sessions > ic::PLAN_MAX_SESSIONS || a->width > (1 << 26)) {
    ic::set_last_error("page_plan: at most 8192 sessions and 2^26 pages per session");
    return IC_ERR_UNSUPPORTED;
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  ic_page_plan_args args = *a;
  int fused = a->total <= ic::FUSED_TOKENS ? 1 : 0;
  void* p1[] = {&args, &fused};
  int rc = ic::launch_pdl(reinterpret_cast<const void*>(ic::plan_rows_kernel), dim3(1), dim3(ic::PT), 0, st, p1,
                          "page_plan (sessions)");
  if (rc != IC_OK || fused) return rc;
  const int64_t threads = (static_cast<int64_t>(a->total) + ic::TPT - 1) / ic::TPT;
  void* p2[] = {&args};
  return ic::launch_pdl(reinterpret_cast<const void*>(ic::plan_tokens_kernel),
                        dim3(static_cast<unsigned>((threads + 255) / 256)), dim3(256), (a->num_sessions + 1) * 4, st, p2,
                        "page_plan (tokens)");
}

extern "C" int ic_page_release(const ic_page_release_args* a, void* stream) {
  if (!a || !a->lens || !a->keep || !a->block_table || !a->free_pages || !a->free_count || a->num_sessions < 1 ||
      a->width < 1 || a->free_capacity < 0) {
    ic::set_last_error("page_release: bad arguments");
    return IC_ERR_INVALID_ARG;
  }
  ic_page_release_args args = *a;
  void* p[] = {&args};
  return ic::launch_pdl(reinterpret_cast<const void*>(ic::release_kernel), dim3(1), dim3(ic::PT), 0,
                        static_cast<cudaStream_t>(stream), p, "page_release");
}
