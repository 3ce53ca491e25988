// Attention of a few query tokens per session over 8-bit pages: the streaming
// kernel, bound by HBM (every page is read once: 2 * D + 8/16 bytes per token
// and KV head).
//
// Work.  A session's query rows (its new tokens x the query heads of a KV
// head) are cut into tiles of 8 or 16 rows; a (session, KV head, tile) is a
// group, its pages a run of units.  Two ways to deal them out (cluster_size):
//  * a cluster of 1 to 8 CTAs per group, joined through distributed shared
//    memory, while the table's width bounds what a CTA gets;
//  * for wide tables, all groups' pages on one line, OVERHEAD units before each
//    group's first, cut into equal shares, one per CTA, so that ragged lengths
//    and a single long session balance alike.  A CTA walks its share group by
//    group; a group that ends up in several shares leaves partial (max, sum, O)
//    per share, which a second small kernel joins in share order.
// Nothing depends on an order of atomics.
//
// Measured (B200, 128 dims): 64 sessions of 1k to 8k tokens, 4 KV heads of 7 query
// heads, 57 to 60 us: 5.2 TB/s of codes and scales, 78 to 80 % of a plain copy's
// rate; 16 of 2k, 2 heads of 8, 12.2 us (clusters of 8; 15.4 under a table of 2048
// columns); one of 128k, as many heads, 23.8 us, of which the join is 4; one of 300
// tokens 6.7 us (launch and dependent loads: q, table, scales, pages; 9.3 under
// 2048 columns).
//
// Inside a CTA each warp streams its own pages (every 8th of the segment)
// through a ring of its own: one elected lane issues two TMA box copies per
// page (16 tokens of K, 16 of V), completion on the stage's mbarrier, no block
// barrier while streaming.  Per page, on the tensor cores (mma.sync m16n8k16,
// fp16 operands: both code formats are exact in fp16):
//   S^T = K Q^T     K's codes become the A operand straight from 16-byte
//                   shared-memory loads: the contraction's order is free, so
//                   lane (g, t) takes 16 consecutive codes of tokens g and
//                   g + 8 and q is laid out to match;
//   u = S^T * (k scale * softmax scale) + log2(v scale)
//   P' = 2^(u - M + 7)   M: a running maximum, replaced only when some u
//                   passes it by 8, so P' <= 2^15 and small weights stay
//                   normal in fp16 down to 2^-21 of M;
//   O^T += V^T P'^T  V's codes paired over tokens by byte permutes;
//   l += sum P' / v scale.
// Folding the page's V scale into the exponent makes every page's codes add to
// one accumulator without a multiplication per output element, and the weight
// of a page never under- or overflows however far the pages' scales lie apart:
// M follows the scaled weights themselves.
#include <cuda.h>
#include <math.h>

#include <type_traits>

#include "common.cuh"
#include "launch.cuh"
#include "mma_helpers.cuh"
#include "paged_attn.cuh"
#include "q8.cuh"
#include "tc05.cuh"

namespace ic {
namespace paged {
namespace {

constexpr int SMS = 148;
constexpr int NW = 8;                 // warps per CTA
// What a group costs a CTA besides its pages, in pages: about 2.5 us to begin and
// to join its warps, against 0.1 us a page.  (Counting pages alone gave one CTA 16
// groups of one page: 83 sessions of 6 tokens, 4 heads of 16: 98 us, now 25; the 64
// sessions of up to 8k tokens: 62 us, now 58.)
constexpr int OVERHEAD = 24;
// The fewest units a CTA takes; more than OVERHEAD, so that a share holds a page.
constexpr int MIN_SHARE = 32;
static_assert(MIN_SHARE > OVERHEAD, "a share that begins before a group's first page reaches it");
constexpr float TINY = 7.8886090522101181e-31f;  // 2^-100
constexpr float SLACK = 8.f;          // u may pass M by this much
constexpr float LIFT = 7.f;           // P' = 2^(u - M + LIFT): at most 2^15

// CTAs per SM: two where 128 registers a thread hold O and the rest with hardly a
// spill.  With 16 rows of 128 dims that is the cluster form (52 bytes of spills;
// 83 sessions of 12 rows, 4 heads, 80 keys: 18.2 us, one CTA per SM 23.1); shares
// of the line would spill 228 bytes (3 sessions of up to 29k: 26 us, one CTA 20).
// Ring stages per warp: what their shared memory leaves beside the merge rows.
__host__ __device__ constexpr int ctas_per_sm(int D, int NG, bool grouped) { return D * NG > (grouped ? 256 : 128) || D == 256 ? 1 : 2; }
__host__ __device__ constexpr int stages(int D, int NG, bool grouped) { return D == 64 ? 5 : ctas_per_sm(D, NG, grouped) == 1 && D == 128 ? 5 : 2; }

struct Task {  // the group that continues past a CTA's share, when it begins there
  int32_t valid, s, h, tile, last_cta, first_slot;
};

template <int D, int NG, bool GROUPED>
struct Layout {
  static constexpr int PAGE_B = 16 * D;                      // codes of a page of one head
  static constexpr int ST = stages(D, NG, GROUPED);
  static constexpr int RING = NW * ST * 2 * PAGE_B;
  static constexpr int ROWS = 8 * NG;
  static constexpr int PITCH = D + 4;                        // floats per row of a warp's O
  static constexpr int MERGE = RING;                         // 8 rows of every warp's O
  static constexpr int BARS = MERGE + NW * 8 * PITCH * 4;
  static constexpr int STAT = BARS + NW * ST * 8;            // M, l per warp and row
  static constexpr int QS = STAT + NW * ROWS * 8;            // NG = 2: q as B operands, 16 bytes per lane
  static constexpr int QB = QS + (NG == 2 ? NG * D * 16 : 0);  // and its rows' scales
  static constexpr int SCAN = QB + ROWS * 4;
  static constexpr int PREFIX = SCAN + 64;
  static int bytes(int S) { return PREFIX + (S + 1) * 4 + 1024; }  // + alignment
};

// Byte offset of 16-byte chunk c of token t in a swizzled page.
template <int D>
__device__ __forceinline__ int page_off(int t, int c) {
  if (D == 64) {
    const int line = t >> 1;
    return line * 128 + (((((t & 1) << 2) | c) ^ (line & 7)) << 4);
  }
  return (c >> 3) * 2048 + t * 128 + (((c & 7) ^ (t & 7)) << 4);
}

__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t half2_bits(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// 16 query elements (two 16-byte vectors) as fp16 pairs; bf16 values times `f`.
__device__ __forceinline__ void q_pairs(const uint4& a, const uint4& b, float, uint32_t* o, __half*) {
  o[0] = a.x; o[1] = a.y; o[2] = a.z; o[3] = a.w; o[4] = b.x; o[5] = b.y; o[6] = b.z; o[7] = b.w;
}
__device__ __forceinline__ void q_pairs(const uint4& a, const uint4& b, float f, uint32_t* o, __nv_bfloat16*) {
  const uint32_t u[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
  for (int i = 0; i < 8; ++i)
    o[i] = half2_bits(__uint_as_float(u[i] << 16) * f, __uint_as_float(u[i] & 0xffff0000u) * f);
}
__device__ __forceinline__ uint32_t max_magnitude(uint32_t m, const uint4& v) {  // finite bf16 pairs, as float bits
  const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t lo = (u[i] << 16) & 0x7fffffffu, hi = u[i] & 0x7fff0000u;
    m = max(m, lo < 0x7f800000u ? lo : 0u);
    m = max(m, hi < 0x7f800000u ? hi : 0u);
  }
  return m;
}

__device__ __forceinline__ float2 ld_cluster2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

// Four finished elements x / l; no key at all gives zeros, NaN stays NaN.
template <typename QT>
__device__ __forceinline__ void store_row(QT* dst, const float4& x, float l) {
  const float inv = l > 0.f ? 1.f / l : l == l ? 0.f : l;
  const auto pair = [&](float a, float b) {
    return static_cast<uint32_t>(Mma<QT>::bits(a * inv)) | (static_cast<uint32_t>(Mma<QT>::bits(b * inv)) << 16);
  };
  *reinterpret_cast<uint2*>(dst) = make_uint2(pair(x.x, x.y), pair(x.z, x.w));
}
__device__ __forceinline__ float lse_of(float m, float l) {
  return l > 0.f ? (m - LIFT + log2f(l)) * LN2 : l == l ? -INFINITY : l;
}

// GROUPED: one cluster of CTAs per group instead of shares of the line.
template <typename QT, int D, int CODE, int NG, bool GROUPED>
__global__ void __launch_bounds__(NW * 32, ctas_per_sm(D, NG, GROUPED))
    stream_kernel(const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv, const Params p) {
  using L = Layout<D, NG, GROUPED>;
  constexpr int ST = L::ST, ROWS = L::ROWS, MT = D / 16, NC = D / 64, W4 = D / 32;
  constexpr bool SCALE_Q = std::is_same<QT, __nv_bfloat16>::value;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = smem_raw + ((1024 - (smem_addr(smem_raw) & 1023)) & 1023);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::BARS);
  float* stat = reinterpret_cast<float*>(smem + L::STAT);     // [NW][ROWS][2]
  // Tiles of 16 rows: q stays in shared memory for all warps, which leaves its
  // registers to O (in registers: 64 sessions of 8k at 256 dims 155 us instead of
  // 123, with 300 bytes of spills); warp nt lays out n-tile nt.
  constexpr bool Q_SHARED = NG == 2;
  uint4* qs = reinterpret_cast<uint4*>(smem + L::QS);         // [NG][NC * 2][32]
  const uint32_t qs_lane = smem_addr(smem + L::QS) + (threadIdx.x & 31) * 16;
  float* q_back = reinterpret_cast<float*>(smem + L::QB);     // [ROWS]
  int32_t* scan = reinterpret_cast<int32_t*>(smem + L::SCAN);
  int32_t* prefix = reinterpret_cast<int32_t*>(smem + L::PREFIX);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, tq = lane & 3;
  const int CL = GROUPED ? p.cluster : 1, rank = GROUPED ? static_cast<int>(cluster_ctarank()) : 0;
  const int gw = rank * NW + warp, stride = NW * CL;  // this warp among those of a segment

  if (tid < NW * ST) {
    mbar_init(bars + tid, 1);
    fence_barrier_init();
  }
  if (tid == 0) prefix[0] = 0;
  grid_dependency_wait();
  grid_launch_dependents();

  // ---- the line of all groups' pages: prefix sums over the sessions -----------
  // Up to 32 sessions live in the lanes of every warp; more, in shared memory.
  const bool lanes = p.S <= 32;
  int l_begin = 0, l_tok = 0, l_len = 0, l_upto = 0, total;
  const auto units_of = [&](int x, int& begin, int& tok, int& len) {
    tok = query_tokens(p, x, begin);
    len = held_tokens(p, x);
    const int rows = tok * p.G;
    const int units = GROUPED ? 1 : OVERHEAD + max(1, (len + q8::PAGE - 1) / q8::PAGE);
    return rows <= p.few_rows ? (rows + ROWS - 1) / ROWS * p.H * units : 0;
  };
  // One session's units fit 31 bits, and so do all while q_start ascends; where it
  // does not, the sums stop at 2^31 - 1 and every index still stays in its range.
  const auto add = [](int x, int y) {
    return static_cast<int>(min(static_cast<uint32_t>(x) + static_cast<uint32_t>(y), 0x7fffffffu));
  };
  if (lanes) {
    if (lane < p.S) l_upto = units_of(lane, l_begin, l_tok, l_len);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(FULL_MASK, l_upto, o);
      if (lane >= o) l_upto = add(l_upto, u);
    }
    total = __shfl_sync(FULL_MASK, l_upto, 31);
    __syncthreads();  // the barriers are initialised
  } else {
    int carry = 0;
    for (int s0 = 0; s0 < p.S; s0 += NW * 32) {
      const int s = s0 + tid;
      int w = 0, x, y, z;
      if (s < p.S) w = units_of(s, x, y, z);
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(FULL_MASK, w, o);
        if (lane >= o) w = add(w, u);
      }
      if (lane == 31) scan[warp] = w;
      __syncthreads();
      int before = carry;
#pragma unroll
      for (int i = 0; i < NW; ++i) {
        if (i < warp) before = add(before, scan[i]);
        carry = add(carry, scan[i]);
      }
      if (s < p.S) prefix[s + 1] = add(before, w);
      __syncthreads();
    }
    total = prefix[p.S];
  }
  constexpr uint32_t CTAS = SMS * ctas_per_sm(D, NG, false);
  const int share = GROUPED ? 1 : max(static_cast<int>((static_cast<uint32_t>(total) + CTAS - 1) / CTAS), MIN_SHARE);
  const int cta = GROUPED ? blockIdx.x / CL : blockIdx.x;
  const int64_t pos0 = static_cast<int64_t>(cta) * share;
  const int end = static_cast<int>(min(pos0 + share, static_cast<int64_t>(total)));
  float* part = p.ws;                                                  // [2 * CTAS][ROWS][D]
  float* part_stat = part + static_cast<size_t>(2) * CTAS * ROWS * D;  // [2 * CTAS][ROWS][2]
  Task* tasks = reinterpret_cast<Task*>(part_stat + static_cast<size_t>(2) * CTAS * ROWS * 2);
  if (!GROUPED && tid == 0) tasks[cta].valid = 0;
  if (pos0 >= end) return;  // GROUPED: a whole cluster

  const uint32_t ring = smem_addr(smem) + warp * (ST * 2 * L::PAGE_B);
  uint64_t* wbar = bars + warp * ST;
  uint32_t phases = 0;   // bit i: parity of the next wait on stage i
  bool dead = false;     // a wait gave up: nothing more is loaded
  int st = 0;            // stage of the next page to be consumed

  // A segment: session s, KV head h, row tile, pages p0 .. p1 of the group (at
  // least one); this warp's are p0 + gw + stride * i, i < mine.
  struct Seg {
    int s, h, q_begin, n_tok, len, row0, pages, p0, p1, mine, end;  // end: of the group, on the line
  };
  const auto find = [&](int pos, int from) {
    Seg g;
    int before;
    if (lanes) {
      g.s = __popc(__ballot_sync(FULL_MASK, l_upto <= pos));
      before = __shfl_sync(FULL_MASK, l_upto, max(g.s - 1, 0));
      if (g.s == 0) before = 0;
      g.q_begin = __shfl_sync(FULL_MASK, l_begin, g.s);
      g.n_tok = __shfl_sync(FULL_MASK, l_tok, g.s);
      g.len = __shfl_sync(FULL_MASK, l_len, g.s);
    } else {
      int lo = from, hi = p.S;  // the last session whose first unit is <= pos
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (prefix[mid] <= pos) lo = mid; else hi = mid;
      }
      g.s = lo;
      before = prefix[lo];
      g.n_tok = query_tokens(p, lo, g.q_begin);
      g.len = held_tokens(p, lo);
    }
    g.pages = max(1, (g.len + q8::PAGE - 1) / q8::PAGE);
    const uint32_t tiles = static_cast<uint32_t>(g.n_tok * p.G + ROWS - 1) / ROWS, at = pos - before;
    const uint32_t units = OVERHEAD + g.pages, gi = GROUPED ? at : at / units, hh = tiles == 1 ? gi : gi / tiles;
    const int off = at - gi * units - OVERHEAD;  // units before the first page are negative
    g.p0 = GROUPED ? 0 : max(off, 0);
    g.p1 = GROUPED ? g.pages : min(g.pages, off + (end - pos));
    g.end = static_cast<int>(min(static_cast<uint32_t>(pos - off) + g.pages, 0x7fffffffu));
    g.h = hh;
    g.row0 = (gi - hh * tiles) * ROWS;
    g.mine = g.p1 - g.p0 > gw ? static_cast<uint32_t>(g.p1 - g.p0 - gw + stride - 1) / static_cast<uint32_t>(stride) : 0;
    return g;
  };
  // Lane j holds page base + j of this warp: its id, then its K scale and the
  // logarithm and reciprocal of its V scale (both at least 2^-100, so a zero
  // scale stays harmless).
  const auto fetch_id = [&](const Seg& g, int base) {
    const int i = base + lane, pg = g.p0 + gw + stride * i;
    int id = -1;
    if (i < g.mine && pg * q8::PAGE < g.len) {
      id = p.table[static_cast<int64_t>(g.s) * p.width + pg];
      if (static_cast<unsigned>(id) >= static_cast<unsigned>(p.n_pages)) {
        id = -1;
        if (p.status) atomicOr(p.status, IC_DEVFLAG_BAD_ROW);
      }
    }
    return id;
  };
  const auto fetch_scales = [&](const Seg& g, int id, float& ks, float& vs) {
    ks = vs = 1.f;
    if (id >= 0) {
      ks = p.k_scale[static_cast<int64_t>(g.h) * p.n_pages + id];
      vs = p.v_scale[static_cast<int64_t>(g.h) * p.n_pages + id];
    }
  };
  const auto issue = [&](const Seg& g, int stage, int page) {
    if (lane == 0 && page >= 0 && !dead) {
      unsigned char* dst = smem + warp * (ST * 2 * L::PAGE_B) + stage * 2 * L::PAGE_B;
      mbar_arrive_expect_tx(wbar + stage, 2 * L::PAGE_B);
      const int y = D == 64 ? page * 8 : page * 16;
#pragma unroll
      for (int x = 0; x < (D == 256 ? 2 : 1); ++x) {
        tc::tma_load_3d(dst + x * 2048, &mk, x * 128, y, g.h, wbar + stage);
        tc::tma_load_3d(dst + L::PAGE_B + x * 2048, &mv, x * 128, y, g.h, wbar + stage);
      }
    }
  };
  const auto wrap = [](int x) { return x >= ST ? x - ST : x; };
  // The first ST pages of a segment; the ring is empty when this is called.
  const auto begin_pages = [&](const Seg& g, int id) {
#pragma unroll
    for (int i = 0; i < ST; ++i) {
      const int page = __shfl_sync(FULL_MASK, id, i);
      if (i < g.mine) issue(g, wrap(st + i), page);
    }
  };

  int pos = static_cast<int>(pos0);
  Seg seg = find(pos, 0);
  int id_c = fetch_id(seg, 0);
  begin_pages(seg, id_c);
  for (;;) {
    const int s = seg.s, h = seg.h, len = seg.len, rows = seg.n_tok * p.G, row0 = seg.row0, mine = seg.mine;
    float ks_c, vs_c, ks_n = 1.f, vs_n = 1.f;
    int id_n = -1;
    fetch_scales(seg, id_c, ks_c, vs_c);
    if (mine > 32) id_n = fetch_id(seg, 32);

    // ---- q as the B operand; head rows past the session's are zero ---------------
    uint32_t qb[Q_SHARED ? 1 : NG][NC * 4][2];
    float qmul[NG][2];
    int lim[NG][2];      // keys that rows 2 tq, 2 tq + 1 of each n-tile see
#pragma unroll
    for (int n = 0; n < (Q_SHARED ? 1 : NG); ++n) {
      const int nt = Q_SHARED ? warp : n;
      if (Q_SHARED && warp >= NG) break;
      const int r = row0 + nt * 8 + g;
      const bool ok = r < rows;
      const QT* src = static_cast<const QT*>(p.q);
      if (ok) src += (seg.q_begin + r / p.G) * p.q_stride_t + (h * p.G + r % p.G) * p.q_stride_h;
      uint4 va[NC], vb[NC];
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int chunk = D == 64 ? tq : (c >> 1) * 8 + 2 * tq + (c & 1);
        va[c] = vb[c] = make_uint4(0, 0, 0, 0);
        if (ok) {
          va[c] = reinterpret_cast<const uint4*>(src + chunk * 16)[0];
          vb[c] = reinterpret_cast<const uint4*>(src + chunk * 16)[1];
        }
      }
      float f = 1.f, back = 1.f;
      if (SCALE_Q) {
        // bf16 to fp16: a power of two brings the row's largest finite value
        // into [2^13, 2^14), so that nothing overflows and elements down to
        // 2^-27 of it convert exactly
        uint32_t m = 0;
#pragma unroll
        for (int c = 0; c < NC; ++c) m = max_magnitude(max_magnitude(m, va[c]), vb[c]);
        m = max(m, __shfl_xor_sync(FULL_MASK, m, 1));
        m = max(m, __shfl_xor_sync(FULL_MASK, m, 2));
        const int x = max(static_cast<int>(m >> 23) - 126, -100);
        f = q8::two_to(14 - x);
        back = q8::two_to(x - 14);
      }
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        uint32_t o[8];
        q_pairs(va[c], vb[c], f, o, static_cast<QT*>(nullptr));
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          qb[n][c * 4 + j][0] = o[2 * j];
          qb[n][c * 4 + j][1] = o[2 * j + 1];
        }
        if (Q_SHARED) {
          qs[(nt * NC * 2 + 2 * c) * 32 + lane] = make_uint4(o[0], o[1], o[2], o[3]);
          qs[(nt * NC * 2 + 2 * c + 1) * 32 + lane] = make_uint4(o[4], o[5], o[6], o[7]);
        }
      }
      if (Q_SHARED) {
        if (tq == 0) q_back[nt * 8 + g] = back;
      } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) qmul[n][i] = __shfl_sync(FULL_MASK, back, (2 * tq + i) * 4) * p.sl2;
      }
    }
    if (Q_SHARED) __syncthreads();
#pragma unroll
    for (int nt = 0; nt < NG; ++nt) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (Q_SHARED) qmul[nt][i] = q_back[nt * 8 + 2 * tq + i] * p.sl2;
        const int ri = row0 + nt * 8 + 2 * tq + i;
        lim[nt][i] = ri < rows ? len - seg.n_tok + ri / p.G + 1 : 0;
      }
    }
    const int lim_all = len - seg.n_tok + row0 / p.G + 1;  // keys that every row of the tile sees
    ks_c = fmaxf(ks_c, TINY);
    vs_c = fmaxf(vs_c, TINY);
    float lv_c = log2f(vs_c), iv_c = 1.f / vs_c;

    float M[NG][2], l[NG][2], o[NG][MT][4];
#pragma unroll
    for (int nt = 0; nt < NG; ++nt) {
      M[nt][0] = M[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) o[nt][mt][0] = o[nt][mt][1] = o[nt][mt][2] = o[nt][mt][3] = 0.f;
    }

    // ---- stream ---------------------------------------------------------------------
#pragma unroll 1
    for (int i = 0; i < mine; ++i) {
      if ((i & 31) == 0) {
        if (i > 0) {
          id_c = id_n;
          ks_c = fmaxf(ks_n, TINY);
          vs_c = fmaxf(vs_n, TINY);
          lv_c = log2f(vs_c);
          iv_c = 1.f / vs_c;
          id_n = i + 32 < mine ? fetch_id(seg, i + 32) : -1;
        }
        fetch_scales(seg, id_n, ks_n, vs_n);
      }
      const int page = __shfl_sync(FULL_MASK, id_c, i & 31);
      const float ks = __shfl_sync(FULL_MASK, ks_c, i & 31);
      const float lv = __shfl_sync(FULL_MASK, lv_c, i & 31), inv_vs = __shfl_sync(FULL_MASK, iv_c, i & 31);
      const int nx = i + ST;  // the page that takes this one's stage
      const int next_c = __shfl_sync(FULL_MASK, id_c, nx & 31), next_n = __shfl_sync(FULL_MASK, id_n, nx & 31);
      const int next = nx < mine ? ((nx >> 5) == (i >> 5) ? next_c : next_n) : -1;
      if (page >= 0 && !dead) {
        const bool ok = mbar_wait_bounded(wbar + st, (phases >> st) & 1, p.status);
        dead = !__all_sync(FULL_MASK, ok);
        phases ^= 1u << st;
      }
      if (page >= 0 && !dead) {
        const uint32_t kp = ring + st * 2 * L::PAGE_B, vp = kp + L::PAGE_B;
        const int tok0 = (seg.p0 + gw + stride * i) * q8::PAGE;
        float acc[NG][4];
#pragma unroll
        for (int nt = 0; nt < NG; ++nt) acc[nt][0] = acc[nt][1] = acc[nt][2] = acc[nt][3] = 0.f;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const int chunk = D == 64 ? tq : (c >> 1) * 8 + 2 * tq + (c & 1);
          const uint4 k0 = lds128(kp + page_off<D>(g, chunk)), k1 = lds128(kp + page_off<D>(g + 8, chunk));
          const uint32_t w0[4] = {k0.x, k0.y, k0.z, k0.w}, w1[4] = {k1.x, k1.y, k1.z, k1.w};
#pragma unroll
          for (int j2 = 0; j2 < 2; ++j2) {
            uint4 qv[NG];
            if (Q_SHARED) {
#pragma unroll
              for (int nt = 0; nt < NG; ++nt) qv[nt] = lds128(qs_lane + (nt * NC * 2 + 2 * c + j2) * 512);
            }
#pragma unroll
            for (int j = 2 * j2; j < 2 * j2 + 2; ++j) {
              uint32_t a0, a1, a2, a3;
              q8::decode4_h2<CODE>(w0[j], a0, a2);
              q8::decode4_h2<CODE>(w1[j], a1, a3);
#pragma unroll
              for (int nt = 0; nt < NG; ++nt)
                Mma<__half>::run(acc[nt], a0, a1, a2, a3,
                                 Q_SHARED ? (j & 1 ? qv[nt].z : qv[nt].x) : qb[Q_SHARED ? 0 : nt][c * 4 + j][0],
                                 Q_SHARED ? (j & 1 ? qv[nt].w : qv[nt].y) : qb[Q_SHARED ? 0 : nt][c * 4 + j][1]);
            }
          }
        }
        // V: tokens 2 tq, 2 tq + 1, 2 tq + 8, 2 tq + 9; this lane's D / 8 dims from D / 8 * g
        uint32_t t[4][W4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int tok = 2 * tq + (x & 1) + (x >> 1) * 8;
          if (D == 64) {
            const uint2 v = lds64(vp + page_off<D>(tok, g >> 1) + (g & 1) * 8);
            t[x][0] = v.x;
            t[x][1] = v.y;
          } else {
#pragma unroll
            for (int c = 0; c < W4 / 4; ++c) {
              const uint4 v = lds128(vp + page_off<D>(tok, g * (W4 / 4) + c));
              t[x][4 * c] = v.x;
              t[x][4 * c + 1] = v.y;
              t[x][4 * c + 2] = v.z;
              t[x][4 * c + 3] = v.w;
            }
          }
          if (tok0 + q8::PAGE > len && tok0 + tok >= len) {  // nothing of an earlier owner's rows
#pragma unroll
            for (int c = 0; c < W4; ++c) t[x][c] = 0;
          }
        }
        const bool edge = tok0 + q8::PAGE > lim_all;
        bool over = false;
#pragma unroll
        for (int nt = 0; nt < NG; ++nt) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float u = fmaf(acc[nt][e], ks * qmul[nt][e & 1], lv);
            if (edge && tok0 + g + (e >> 1) * 8 >= lim[nt][e & 1]) u = -INFINITY;
            acc[nt][e] = u;
            over |= u > M[nt][e & 1] + SLACK;
          }
        }
        if (__any_sync(FULL_MASK, over)) {
#pragma unroll
          for (int nt = 0; nt < NG; ++nt) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float m = fmaxf(acc[nt][e], acc[nt][e + 2]);
#pragma unroll
              for (int x = 4; x < 32; x <<= 1) m = fmaxf(m, __shfl_xor_sync(FULL_MASK, m, x));
              m = fmaxf(m, M[nt][e]);
              const float f = m == -INFINITY ? 1.f : tc::ex2(M[nt][e] - m);
              M[nt][e] = m;
              l[nt][e] *= f;
#pragma unroll
              for (int mt = 0; mt < MT; ++mt) {
                o[nt][mt][e] *= f;
                o[nt][mt][e + 2] *= f;
              }
            }
          }
        }
        uint32_t pb[NG][2];
#pragma unroll
        for (int nt = 0; nt < NG; ++nt) {
          float pr[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float m = M[nt][e & 1];
            pr[e] = tc::ex2(acc[nt][e] - (m == -INFINITY ? 0.f : m - LIFT));
          }
          l[nt][0] = fmaf(pr[0] + pr[2], inv_vs, l[nt][0]);
          l[nt][1] = fmaf(pr[1] + pr[3], inv_vs, l[nt][1]);
          pb[nt][0] = transpose8(half2_bits(pr[0], pr[1]));
          pb[nt][1] = transpose8(half2_bits(pr[2], pr[3]));
        }
#pragma unroll
        for (int c = 0; c < W4; ++c) {
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            uint32_t a0, a1, a2, a3;
            q8::decode4_h2<CODE>(__byte_perm(t[0][c], t[1][c], half ? 0x7362 : 0x5140), a0, a1);
            q8::decode4_h2<CODE>(__byte_perm(t[2][c], t[3][c], half ? 0x7362 : 0x5140), a2, a3);
#pragma unroll
            for (int nt = 0; nt < NG; ++nt)
              Mma<__half>::run(o[nt][2 * c + half], a0, a1, a2, a3, pb[nt][0], pb[nt][1]);
          }
        }
      }
      // Not before the products have consumed what was loaded from the page: a load
      // that is merely issued may still be under way when the next page's copy
      // begins to land in this stage.
      __syncwarp();
      issue(seg, st, next);
      st = wrap(st + 1);
    }
    if (dead) {  // copies in flight land before their buffers are given up (short waits)
      for (int x = 0; x < ST; ++x) mbar_wait_bounded(wbar + x, (phases >> x) & 1, nullptr, 200000000ull);
    }

    // ---- the next segment's first pages are on their way while this one is joined ------
    // (a share that ends before the next group's first page has no part of it)
    const int next_pos = seg.end;
    const bool more = !GROUPED && next_pos < end - OVERHEAD;
    Seg nseg;
    int nid = -1;
    if (more) {
      nseg = find(next_pos, s);
      nid = fetch_id(nseg, 0);
      begin_pages(nseg, nid);
    }
#pragma unroll
    for (int nt = 0; nt < NG; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) l[nt][e] += __shfl_xor_sync(FULL_MASK, l[nt][e], x);

    // ---- join the warps, 8 rows at a time ----------------------------------------------
    float* wo = reinterpret_cast<float*>(smem + L::MERGE);
    float* cx = reinterpret_cast<float*>(smem);  // GROUPED: [ROWS][D] in the ring, which is done, and [ROWS][2] behind it
    float* cs = cx + ROWS * D;
    const bool whole = seg.p0 == 0 && seg.p1 == seg.pages;
    const int slot = 2 * cta + (pos == pos0 ? 0 : 1);
#pragma unroll
    for (int nt = 0; nt < NG; ++nt) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = 2 * tq + e;
        float* dst = wo + (warp * 8 + row) * L::PITCH + (D / 8) * g;
        // elements 2 mt + {0, 1} of this lane's dims are o[mt][e], o[mt][e + 2]
#pragma unroll
        for (int c = 0; c < MT / 2; ++c)
          reinterpret_cast<float4*>(dst)[c] =
              make_float4(o[nt][2 * c][e], o[nt][2 * c][e + 2], o[nt][2 * c + 1][e], o[nt][2 * c + 1][e + 2]);
        if (g == 0) *reinterpret_cast<float2*>(stat + (warp * 8 + row) * 2) = make_float2(M[nt][e], l[nt][e]);
      }
      __syncthreads();
      for (int e = tid; e < 8 * (D / 4); e += NW * 32) {
        const int row = e / (D / 4), d0 = e % (D / 4) * 4, r = row0 + nt * 8 + row;
        float2 ml[NW];
        float m = -INFINITY, lsum = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
          ml[w] = *reinterpret_cast<const float2*>(stat + (w * 8 + row) * 2);
          m = fmaxf(m, ml[w].x);
        }
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < NW; ++w) {
          const float f = ml[w].x == -INFINITY ? 0.f : tc::ex2(ml[w].x - m);
          lsum = fmaf(ml[w].y, f, lsum);
          const float4 u = *reinterpret_cast<const float4*>(wo + (w * 8 + row) * L::PITCH + d0);
          x.x = fmaf(u.x, f, x.x); x.y = fmaf(u.y, f, x.y); x.z = fmaf(u.z, f, x.z); x.w = fmaf(u.w, f, x.w);
        }
        const size_t prow = static_cast<size_t>(slot) * ROWS + nt * 8 + row;
        if (GROUPED) {  // this CTA's part, for the cluster to read
          *reinterpret_cast<float4*>(cx + (nt * 8 + row) * D + d0) = x;
          if (d0 == 0) *reinterpret_cast<float2*>(cs + (nt * 8 + row) * 2) = make_float2(m, lsum);
        } else if (!whole) {
          *reinterpret_cast<float4*>(part + prow * D + d0) = x;
          if (d0 == 0) *reinterpret_cast<float2*>(part_stat + prow * 2) = make_float2(m, lsum);
        } else if (r < rows) {
          const int64_t orow = static_cast<int64_t>(seg.q_begin + r / p.G) * p.Hq + h * p.G + r % p.G;
          store_row<QT>(static_cast<QT*>(p.out) + orow * D + d0, x, lsum);
          if (d0 == 0 && p.lse) p.lse[orow] = lse_of(m, lsum);
        }
      }
      __syncthreads();
    }
    if (GROUPED) {
      // Every CTA's rows lie in its shared memory; CTA j finishes rows j, j + CL,
      // ..., a warp each, adding the parts in the CTAs' order.
      cluster_arrive_release();
      cluster_wait_acquire();
      for (int row = rank + warp * CL; row < ROWS && row0 + row < rows; row += NW * CL) {
        const int r = row0 + row;
        const uint32_t sa = smem_addr(cs + row * 2), xa = smem_addr(cx + row * D);
        // lane j holds part j's maximum and sum
        const float2 ml = lane < CL ? ld_cluster2(map_shared(sa, lane)) : make_float2(-INFINITY, 0.f);
        const float m = warp_max(ml.x), f = ml.x == -INFINITY ? 0.f : tc::ex2(ml.x - m);
        float lsum = 0.f;
        for (int j = 0; j < CL; ++j) lsum = fmaf(__shfl_sync(FULL_MASK, ml.y, j), __shfl_sync(FULL_MASK, f, j), lsum);
        const int64_t orow = static_cast<int64_t>(seg.q_begin + r / p.G) * p.Hq + h * p.G + r % p.G;
#pragma unroll
        for (int d1 = 0; d1 < D; d1 += 128) {
          const int d0 = d1 + lane * 4;
          float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
          for (int j = 0; j < CL; ++j) {
            const float fj = __shfl_sync(FULL_MASK, f, j);
            if (d0 < D) {
              const float4 u = ld_cluster4(map_shared(xa + d0 * 4, j));
              x.x = fmaf(u.x, fj, x.x); x.y = fmaf(u.y, fj, x.y); x.z = fmaf(u.z, fj, x.z); x.w = fmaf(u.w, fj, x.w);
            }
          }
          if (d0 < D) store_row<QT>(static_cast<QT*>(p.out) + orow * D + d0, x, lsum);
        }
        if (lane == 0 && p.lse) p.lse[orow] = lse_of(m, lsum);
      }
      cluster_arrive_release();  // nobody leaves while its rows are read
      cluster_wait_acquire();
      break;
    }
    if (tid == 0 && seg.p0 == 0 && seg.p1 < seg.pages) {  // this CTA holds the group's first page, not its last
      Task t;
      t.valid = 1;
      t.s = s;
      t.h = h;
      t.tile = row0 / ROWS;
      t.last_cta = (min(seg.end, total) - 1) / share;
      t.first_slot = slot;
      tasks[cta] = t;
    }
    if (!more) break;
    pos = next_pos;
    seg = nseg;
    id_c = nid;
  }
}

// Joins the partials of the groups that lie in several shares: for every CTA of
// the streaming kernel (most have nothing to do and leave) one CTA, or several
// with RPC rows of the tile each.  The weights of all partials first, a warp per
// row; then the rows' elements, SUBS subgroups of threads with every SUBS-th
// partial each, joined in order.
constexpr int JT = 512;
template <typename QT, int D, int NG, int RPC>
__global__ void __launch_bounds__(JT) join_kernel(const Params p) {
  constexpr int ROWS = 8 * NG, LN = D / 4, ITEMS = RPC * LN, SUBS = ITEMS >= JT ? 1 : JT / ITEMS;
  constexpr int CTAS = SMS * ctas_per_sm(D, NG, false), PER = (CTAS + 31) / 32;
  __shared__ float weight[RPC][CTAS + 1];
  __shared__ float lsums[RPC], tops[RPC];
  __shared__ float4 sx[SUBS > 1 ? JT : 1];
  grid_dependency_wait();
  grid_launch_dependents();
  const float* part = p.ws;
  const float* part_stat = part + static_cast<size_t>(2) * CTAS * ROWS * D;
  const Task* tasks = reinterpret_cast<const Task*>(part_stat + static_cast<size_t>(2) * CTAS * ROWS * 2);
  const int cta = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, row0 = blockIdx.y * RPC;
  // partial i of the group that begins here: slot 0 or 1 of this CTA, then slot 0
  // of each later one; lane i of a row's warp looks at partial i without waiting
  // to hear how many there are
  const auto stat_at = [&](int slot) {
    return *reinterpret_cast<const float2*>(part_stat + (static_cast<size_t>(slot) * ROWS + row0 + warp) * 2);
  };
  float2 ml[PER], other = make_float2(0.f, 0.f);
#pragma unroll
  for (int k = 0; k < PER; ++k) ml[k] = make_float2(-INFINITY, 0.f);
  if (warp < RPC && cta + lane < CTAS) ml[0] = stat_at(2 * (cta + lane));
  if (warp < RPC && lane == 0) other = stat_at(2 * cta + 1);
  const Task t = tasks[cta];
  if (!t.valid) return;
  int q_begin;
  const int rows = query_tokens(p, t.s, q_begin) * p.G;
  const int n = t.last_cta - cta + 1;
  if (warp < RPC) {
    if (lane == 0 && t.first_slot != 2 * cta) ml[0] = other;
    if (lane >= n) ml[0].x = -INFINITY;
    float m = -INFINITY, lsum = 0.f;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      if (k > 0 && lane + 32 * k < n) ml[k] = stat_at(2 * (cta + lane + 32 * k));
    }
#pragma unroll
    for (int k = 0; k < PER; ++k) m = fmaxf(m, ml[k].x);
    m = warp_max(m);
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      if (lane + 32 * k < n) {
        const float f = ml[k].x == -INFINITY ? 0.f : tc::ex2(ml[k].x - m);
        weight[warp][lane + 32 * k] = f;
        lsum = fmaf(ml[k].y, f, lsum);
      }
    }
    lsum = warp_sum(lsum);
    if (lane == 0) {
      lsums[warp] = lsum;
      tops[warp] = m;
    }
  }
  __syncthreads();
  for (int e = tid; e < ITEMS * SUBS; e += JT) {
    const int sub = e / ITEMS, er = e % ITEMS / LN, d0 = e % LN * 4, r = t.tile * ROWS + row0 + er;
    const auto load = [&](int i) {
      const size_t at = static_cast<size_t>(i == 0 ? t.first_slot : 2 * (cta + i)) * ROWS + row0 + er;
      return *reinterpret_cast<const float4*>(part + at * D + d0);
    };
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (int i = sub; i < n; i += SUBS) {
      const float4 u = load(i);
      const float f = weight[er][i];
      x.x = fmaf(u.x, f, x.x); x.y = fmaf(u.y, f, x.y); x.z = fmaf(u.z, f, x.z); x.w = fmaf(u.w, f, x.w);
    }
    if (SUBS > 1) {
      sx[tid] = x;
      __syncthreads();  // ITEMS * SUBS = JT: every thread comes here once
      if (sub != 0) return;
#pragma unroll
      for (int i = 1; i < SUBS; ++i) {
        const float4 u = sx[tid + i * ITEMS];
        x.x += u.x; x.y += u.y; x.z += u.z; x.w += u.w;
      }
    }
    if (r < rows) {
      const int64_t orow = static_cast<int64_t>(q_begin + r / p.G) * p.Hq + t.h * p.G + r % p.G;
      store_row<QT>(static_cast<QT*>(p.out) + orow * D + d0, x, lsums[er]);
      if (d0 == 0 && p.lse) p.lse[orow] = lse_of(tops[er], lsums[er]);
    }
  }
}

// At most this many groups of `rows` rows, whatever the sessions' counts.
int64_t group_bound(const ic_paged_attn_args& a, int rows) {
  const int64_t G = a.num_q_heads / a.num_kv_heads, n = a.num_q_tokens;
  return std::min<int64_t>(n * ((G + rows - 1) / rows), n * G / rows + std::min<int64_t>(a.num_sessions, n)) * a.num_kv_heads;
}
// CTAs per group when each group gets a cluster of its own, 0 for shares of the
// line.  A cluster joins its parts through distributed shared memory, without
// the 3 to 4 us of a second kernel, but a group is then split over no more than
// 8 CTAs, or left whole when there are many groups: so only while the table's
// width leaves a CTA at most MAX_CTA_PAGES pages.  (33 sessions x 19 tokens x 8
// heads of 8 at 256 dims: shares of the line 859 us, a CTA per group 264 at the
// time, 232 now.)
// Powers of two: clusters of 3 and 6 do not fill the processor groups (96 groups
// of 16 rows at 128 dims over 1400 keys: 21.1 us in 3s, 17.0 in 2s).
constexpr int MAX_CTA_PAGES = 96;
int cluster_size(const ic_paged_attn_args& a, int rows) {
  const int64_t groups = group_bound(a, rows), slots = SMS * ctas_per_sm(a.head_dim, rows / 8, true);
  int64_t cl = 1;
  while (cl < 8 && 2 * cl * groups <= slots) cl *= 2;
  return a.table_width <= MAX_CTA_PAGES * cl && groups * cl <= 0x7fffffff ? static_cast<int>(cl) : 0;
}

template <typename QT, int D, int CODE, int NG>
int launch(const Params& p, const ic_paged_attn_args& a, cudaStream_t st) {
  CUtensorMap mk, mv;
  int rc;
  if ((rc = page_map(&mk, a.k, a.pool_tokens, p.H, D)) != IC_OK) return rc;
  if ((rc = page_map(&mv, a.v, a.pool_tokens, p.H, D)) != IC_OK) return rc;
  Params params = p;
  if (const int cl = p.few_rows == ALL_ROWS ? cluster_size(a, 8 * NG) : 0) {
    static PerDeviceLimit grouped_limit;
    const int smem = Layout<D, NG, true>::bytes(p.S);
    auto kern = stream_kernel<QT, D, CODE, NG, true>;
    if ((rc = ensure_dynamic_smem(kern, smem, &grouped_limit)) != IC_OK) return rc;
    params.cluster = cl;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(group_bound(a, 8 * NG) * cl));
    cfg.blockDim = dim3(NW * 32);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cl;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    cudaLaunchKernelEx(&cfg, kern, mk, mv, params);
    return launch_status("paged_attention (stream, grouped)");
  }
  auto kern = stream_kernel<QT, D, CODE, NG, false>;
  static PerDeviceLimit limit;
  const int smem = Layout<D, NG, false>::bytes(p.S);
  if ((rc = ensure_dynamic_smem(kern, smem, &limit)) != IC_OK) return rc;
  constexpr int ctas = SMS * ctas_per_sm(D, NG, false);
  void* args[] = {&mk, &mv, &params};
  if ((rc = launch_pdl(reinterpret_cast<const void*>(kern), dim3(ctas), dim3(NW * 32), smem, st, args,
                       "paged_attention (stream)")) != IC_OK)
    return rc;
  // Few groups mean many partials each: then two rows per CTA.
  void* jargs[] = {&params};
  const bool few = p.S * p.H <= 16;
  const void* join = few ? reinterpret_cast<const void*>(join_kernel<QT, D, NG, 2>)
                         : reinterpret_cast<const void*>(join_kernel<QT, D, NG, 8 * NG>);
  return launch_pdl(join, dim3(ctas, few ? 4 * NG : 1), dim3(JT), 0, st, jargs, "paged_attention (join)");
}

template <typename QT, int D, int CODE>
int launch_ng(const Params& p, const ic_paged_attn_args& a, cudaStream_t st, bool one) {
  return one ? launch<QT, D, CODE, 1>(p, a, st) : launch<QT, D, CODE, 2>(p, a, st);
}
template <typename QT, int D>
int launch_code(const Params& p, const ic_paged_attn_args& a, cudaStream_t st, bool one) {
  return a.code_dtype == IC_E4M3 ? launch_ng<QT, D, IC_E4M3>(p, a, st, one) : launch_ng<QT, D, IC_I8>(p, a, st, one);
}
template <typename QT>
int launch_dim(const Params& p, const ic_paged_attn_args& a, cudaStream_t st, bool one) {
  switch (a.head_dim) {
    case 64: return launch_code<QT, 64>(p, a, st, one);
    case 128: return launch_code<QT, 128>(p, a, st, one);
    default: return launch_code<QT, 256>(p, a, st, one);
  }
}

}  // namespace

int64_t stream_workspace(const ic_paged_attn_args& a) {
  const int rows = stream_rows(static_cast<int64_t>(a.max_count) * (a.num_q_heads / a.num_kv_heads), a.head_dim);
  if (few_rows(a) == ALL_ROWS && cluster_size(a, rows) > 0) return 0;
  const int64_t ctas = SMS * ctas_per_sm(a.head_dim, rows / 8, false);
  return 2 * ctas * rows * (a.head_dim + 2) * 4 + ctas * static_cast<int64_t>(sizeof(Task));
}

int launch_stream(const Params& p, const ic_paged_attn_args& a, cudaStream_t st) {
  const bool one = stream_rows(static_cast<int64_t>(a.max_count) * p.G, a.head_dim) == 8;
  return a.q_dtype == IC_F16 ? launch_dim<__half>(p, a, st, one) : launch_dim<__nv_bfloat16>(p, a, st, one);
}

}  // namespace paged
}  // namespace ic
