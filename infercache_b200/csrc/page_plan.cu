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
// Measured (B200): 16 sessions of one token 7.1 us (host time), 1000 as much; 512
// prompts of 256 to 32768 tokens, 8.5 million in all, 25 us, 4.2 TB/s of stores
// and some 4 us for the two kernels to begin; the rest is the search at each warp's
// begin and the stores' address work.  Release: one CTA, each warp its 32 sessions'
// pages one session after another, bound by those chains of loads: all 2300 pages of
// 16 sessions 27 us, all 515 thousand of 512 sessions 344 us.
#include "common.cuh"
#include "launch.cuh"
#include "q8.cuh"

namespace ic {
namespace {

constexpr int PT = 1024;            // most threads of the scanning CTA
constexpr int TPT = 8;              // tokens per thread
constexpr int WT = 32 * TPT;        // consecutive tokens per warp
// Tokens that the scanning CTA finishes itself: one pass of its threads.
constexpr int FUSED_TOKENS = PT * TPT;

// Inclusive block scan of one int64 per thread; `total` gets the block's sum.
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t* warp_sums, int64_t& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t u = __shfl_up_sync(FULL_MASK, v, o);
    if (lane >= o) v += u;
  }
  if (warps == 1) {
    total = __shfl_sync(FULL_MASK, v, 31);
    return v;
  }
  if (lane == 31) warp_sums[warp] = v;
  __syncthreads();
  int64_t w = lane < warps ? warp_sums[lane] : 0;  // every warp scans the warps' sums for itself
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t u = __shfl_up_sync(FULL_MASK, w, o);
    if (lane >= o) w += u;
  }
  total = __shfl_sync(FULL_MASK, w, 31);
  const int64_t before = __shfl_sync(FULL_MASK, w, warp > 0 ? warp - 1 : 0);
  __syncthreads();  // warp_sums may be written again
  return v + (warp > 0 ? before : 0);
}

// Pool row of a page's slot; -1 for a page that no pool has (its rows fit 31 bits).
__device__ __forceinline__ int32_t row_of(int32_t page, int32_t slot) {
  return static_cast<uint32_t>(page) > 0x7fffffffu / q8::PAGE ? -1 : page * q8::PAGE + slot;
}

__device__ __forceinline__ int32_t pages_of(int64_t tokens) {
  return static_cast<int32_t>((tokens + q8::PAGE - 1) / q8::PAGE);
}

// A warp's tokens [i0, i1), i0 a multiple of 32.  len[s] is session s's length
// before the call (-1 when it was denied), rank[s] its first new page's rank,
// `top` the stack's height before the call.
__device__ __forceinline__ void plan_tokens(const ic_page_plan_args& a, const int32_t* q_start, const int32_t* len,
                                            const int32_t* rank, int stride, int32_t top, int64_t i0, int64_t i1) {
  const int S = a.num_sessions, lane = threadIdx.x & 31;
  if (i0 >= i1) return;
  int lo = 0, hi = S;  // the last session with q_start[s] <= i0
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (q_start[mid] <= i0) lo = mid; else hi = mid;
  }
  int s = lo;
  int64_t begin = q_start[s], end = q_start[s + 1];
  const bool vec = ((reinterpret_cast<uintptr_t>(a.slots) & 7) | (reinterpret_cast<uintptr_t>(a.positions) & 15)) == 0;
  const auto held_of = [&](int x) { return len[static_cast<int64_t>(x) * stride]; };
  const auto rank_of = [&](int x) { return rank[static_cast<int64_t>(x) * stride]; };
#pragma unroll 1
  for (; i0 < i1; i0 += WT) {
    while (i0 >= end && s + 1 < S) {
      ++s;
      begin = end;
      end = q_start[s + 1];
    }
    const int32_t had = held_of(s);
    if (vec && had >= 0 && i0 >= begin && i0 + WT <= end && i0 + WT <= i1) {
      // all of them are one session's: everything but the token's number is uniform
      const uint32_t held = static_cast<uint32_t>(pages_of(had));
      int32_t* row = a.block_table + static_cast<int64_t>(s) * a.width;
      const int32_t* fresh = a.free_pages + (top - 1 - rank_of(s)) + static_cast<int64_t>(held);  // page idx: fresh[-idx]
      const uint32_t p0 = static_cast<uint32_t>(had) + static_cast<uint32_t>(i0 - begin) + 2 * lane;
      int32_t page[TPT];
#pragma unroll
      for (int j = 0; j < TPT; ++j) {
        const uint32_t p = p0 + 64 * (j >> 1) + (j & 1), idx = p / q8::PAGE;
        if ((j & 1) && p % q8::PAGE != 0)
          page[j] = page[j - 1];
        else
          page[j] = idx < held ? row[idx] : fresh[-static_cast<int64_t>(idx)];
      }
#pragma unroll
      for (int j = 0; j < TPT; j += 2) {
        int32_t slot[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const uint32_t p = p0 + 64 * (j >> 1) + k;
          if (p % q8::PAGE == 0 && p / q8::PAGE >= held) row[p / q8::PAGE] = page[j + k];
          slot[k] = row_of(page[j + k], static_cast<int32_t>(p % q8::PAGE));
        }
        const int64_t i = i0 + 64 * (j >> 1) + 2 * lane, p = p0 + 64 * (j >> 1);
        *reinterpret_cast<int2*>(a.slots + i) = make_int2(slot[0], slot[1]);
        *reinterpret_cast<longlong2*>(a.positions + i) = make_longlong2(p, p + 1);
      }
      continue;
    }
    int x = s;  // this lane's session
    int64_t xb = begin, xe = end;
#pragma unroll 1
    for (int j = 0; j < TPT; ++j) {
      const int64_t i = i0 + 32 * j + lane;
      if (i >= i1) break;
      if (i >= xe && x + 1 < S) {  // the next session, mostly; else the last that begins at or before i
        int a0 = x + 1, a1 = S;
        if (q_start[a0 + 1] > i) a1 = a0 + 1;
        while (a1 - a0 > 1) {
          const int mid = (a0 + a1) >> 1;
          if (q_start[mid] <= i) a0 = mid; else a1 = mid;
        }
        x = a0;
        xb = q_start[x];
        xe = q_start[x + 1];
      }
      int32_t slot = -1, pos = -1;  // positions fit: a table row holds fewer than 2^31 tokens
      const int32_t have = held_of(x);
      if (i < xe && have >= 0) {
        pos = have + static_cast<int32_t>(i - xb);
        const int32_t idx = pos / q8::PAGE, held = pages_of(have);
        int32_t* row = a.block_table + static_cast<int64_t>(x) * a.width;
        const int32_t page = idx < held ? row[idx] : a.free_pages[top - 1 - (rank_of(x) + idx - held)];
        if (idx >= held && pos % q8::PAGE == 0) row[idx] = page;  // a new page's first token enters it
        slot = row_of(page, pos % q8::PAGE);
      }
      a.slots[i] = slot;
      a.positions[i] = pos;
    }
  }
}

// `fused`: the sessions fit one pass of the threads and the tokens are
// finished here, from shared memory, `per_warp` consecutive ones by each warp.
__global__ void __launch_bounds__(PT) plan_rows_kernel(const ic_page_plan_args a, int fused, int per_warp) {
  __shared__ int64_t warp_sums[32];
  __shared__ int32_t taken_s;
  __shared__ int32_t qs[PT + 1], len_s[PT], rank_s[PT];
  if (threadIdx.x == 0) taken_s = 0;
  grid_dependency_wait();
  grid_launch_dependents();
  const int S = a.num_sessions;
  int32_t top = *a.free_count;
  bool bad = false;
  if (top < 0 || top > a.free_capacity) {
    bad = true;
    top = 0;
  }
  int64_t tokens = 0, pages = 0;
  int32_t taken = 0;  // pages up to the last granted one: grants are a prefix of the needs
  for (int s0 = 0; s0 < S; s0 += blockDim.x) {
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
    if (granted && need > 0) taken = static_cast<int32_t>(upto);
    if (s < S) {
      const int32_t q_to = static_cast<int32_t>(q_end < 0x7fffffff ? q_end : 0x7fffffff);
      const int32_t had = granted ? static_cast<int32_t>(len) : -1, rank = static_cast<int32_t>(upto - need);
      a.q_start[s + 1] = q_to;
      if (fused) {
        qs[s + 1] = q_to;
        len_s[s] = had;
        rank_s[s] = rank;
      } else {
        a.workspace[2 * s] = had;
        a.workspace[2 * s + 1] = rank;
      }
      a.lens_out[s] = static_cast<int32_t>(granted ? len + c : len);
      bad |= !granted;
    }
  }
  if (threadIdx.x == 0) {
    a.q_start[0] = 0;
    qs[0] = 0;
    a.workspace[2 * S] = top;
  }
  taken = __reduce_max_sync(FULL_MASK, taken);
  if ((threadIdx.x & 31) == 0 && taken > 0) atomicMax(&taken_s, taken);
  if (__syncthreads_or(bad) && threadIdx.x == 0 && a.dev_status) atomicOr(a.dev_status, IC_DEVFLAG_NO_PAGES);
  if (threadIdx.x == 0) *a.free_count_out = top - taken_s;
  if (fused) {
    const int64_t i0 = static_cast<int64_t>(threadIdx.x >> 5) * per_warp;
    plan_tokens(a, qs, len_s, rank_s, 1, top, i0, min(i0 + per_warp, static_cast<int64_t>(a.total)));
  }
}

// Each warp takes `per_warp` consecutive tokens (a multiple of 32).
__global__ void __launch_bounds__(256) plan_tokens_kernel(const ic_page_plan_args a, int64_t per_warp) {
  extern __shared__ int32_t qs[];
  grid_dependency_wait();
  grid_launch_dependents();
  const int S = a.num_sessions;
  for (int s = threadIdx.x; s <= S; s += blockDim.x) qs[s] = a.q_start[s];
  __syncthreads();
  const int64_t i0 = (static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5)) * per_warp;
  plan_tokens(a, qs, a.workspace, a.workspace + 1, 2, a.workspace[2 * S], i0,
              min(i0 + per_warp, static_cast<int64_t>(a.total)));
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
  int fused = a->total <= ic::FUSED_TOKENS && a->num_sessions <= ic::PT ? 1 : 0;
  // no more warps than the sessions and, when fused, the tokens need: barriers
  // and scans over idle warps would be most of a decode tick's plan
  int threads = a->num_sessions < ic::PT ? (a->num_sessions + 31) / 32 * 32 : ic::PT;
  if (fused) threads = max(threads, (a->total + ic::WT - 1) / ic::WT * 32);
  // A warp walks its tokens 32 at a time and waits for each step's loads: spread
  // them over the warps there are (a token each of 1000 sessions: 7.2 us; 256
  // tokens to a warp: 14.5), but keep the 256 that are taken at once where
  // sessions bring long runs.
  const auto spread = [](int64_t each) {
    return each <= ic::WT / 2 ? (each + 31) / 32 * 32 : (each + ic::WT - 1) / ic::WT * ic::WT;
  };
  int fused_per_warp = static_cast<int>(spread((a->total + threads / 32 - 1) / (threads / 32)));
  void* p1[] = {&args, &fused, &fused_per_warp};
  int rc = ic::launch_pdl(reinterpret_cast<const void*>(ic::plan_rows_kernel), dim3(1), dim3(threads), 0, st, p1,
                          "page_plan (sessions)");
  if (rc != IC_OK || fused) return rc;
  // one wave of 8 CTAs per SM at most: a CTA copies q_start before it begins
  const int64_t warps = static_cast<int64_t>(148) * 8 * 8;
  int64_t per_warp = spread((a->total + warps - 1) / warps);
  const int64_t per_cta = 8 * per_warp;
  void* p2[] = {&args, &per_warp};
  return ic::launch_pdl(reinterpret_cast<const void*>(ic::plan_tokens_kernel),
                        dim3(static_cast<unsigned>((a->total + per_cta - 1) / per_cta)), dim3(256), (a->num_sessions + 1) * 4, st, p2,
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
