// Attention of a few query tokens per session over 8-bit pages: the streaming
// kernel, bound by HBM (every page is read once: 2 * D + 8/16 bytes per token
// and KV head).
//
// Work.  A session's query rows (its new tokens x the query heads of a KV
// head) are cut into tiles of 8 or 16 rows; a (session, KV head, tile) is a
// group, its pages a run of units.  All groups' pages form one line, cut into
// equal shares, one per CTA, so that ragged lengths and a single long session
// balance alike.  A CTA walks its share group by group; a group that ends up in
// several shares leaves partial (max, sum, O) per share, which a second small
// kernel joins in share order.  Nothing depends on an order of atomics.
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

constexpr int NW = 8;                 // warps per CTA
constexpr float SLACK = 8.f;          // u may pass M by this much
constexpr float LIFT = 7.f;           // P' = 2^(u - M + LIFT): at most 2^15

// CTAs per SM (two where 128 registers a thread hold q and O without spills)
// and ring stages per warp: 96 KB of pages in flight per CTA, twice that where
// it has the SM to itself.
__host__ __device__ constexpr int ctas_per_sm(int D, int NG) { return D * NG > 128 ? 1 : 2; }
__host__ __device__ constexpr int stages(int D, int NG) { return (ctas_per_sm(D, NG) == 1 ? 192 : 96) * 1024 / (NW * 32 * D); }

struct Task {  // the group that continues past a CTA's share, when it begins there
  int32_t valid, s, h, tile, last_cta, first_slot;
};

template <int D, int NG>
struct Layout {
  static constexpr int PAGE_B = 16 * D;                      // codes of a page of one head
  static constexpr int ST = stages(D, NG);
  static constexpr int RING = NW * ST * 2 * PAGE_B;
  static constexpr int ROWS = 8 * NG;
  static constexpr int PITCH = D + 4;                        // floats per row of a warp's O
  static constexpr int MERGE = NW * ROWS * PITCH * 4;        // aliases the ring
  static constexpr int BUF = RING > MERGE ? RING : MERGE;
  static constexpr int BARS = BUF;
  static constexpr int STAT = BARS + NW * ST * 8;            // M, l per warp and row
  static constexpr int SCAN = STAT + NW * ROWS * 8;
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

template <typename QT, int D, int CODE, int NG>
__global__ void __launch_bounds__(NW * 32, ctas_per_sm(D, NG))
    stream_kernel(const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv, const Params p) {
  using L = Layout<D, NG>;
  constexpr int ST = L::ST, ROWS = L::ROWS, MT = D / 16, NC = D / 64, W4 = D / 32;
  constexpr bool SCALE_Q = std::is_same<QT, __nv_bfloat16>::value;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = smem_raw + ((1024 - (smem_addr(smem_raw) & 1023)) & 1023);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::BARS);
  float* stat = reinterpret_cast<float*>(smem + L::STAT);     // [NW][ROWS][2]
  int32_t* scan = reinterpret_cast<int32_t*>(smem + L::SCAN);
  int32_t* prefix = reinterpret_cast<int32_t*>(smem + L::PREFIX);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, tq = lane & 3;

  if (tid < NW * ST) {
    mbar_init(bars + tid, 1);
    fence_barrier_init();
  }
  if (tid == 0) prefix[0] = 0;
  grid_dependency_wait();
  grid_launch_dependents();

  // ---- the line of all groups' pages: prefix sums over the sessions -----------
  {
    int carry = 0;
    for (int s0 = 0; s0 < p.S; s0 += NW * 32) {
      const int s = s0 + tid;
      int w = 0;
      if (s < p.S) {
        int begin;
        const int rows = query_tokens(p, s, begin) * p.G;
        const int pages = max(1, (held_tokens(p, s) + q8::PAGE - 1) / q8::PAGE);
        if (rows <= p.few_rows) w = (rows + ROWS - 1) / ROWS * p.H * pages;
      }
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(FULL_MASK, w, o);
        if (lane >= o) w += u;
      }
      if (lane == 31) scan[warp] = w;
      __syncthreads();
      int before = carry;
#pragma unroll
      for (int i = 0; i < NW; ++i) {
        if (i < warp) before += scan[i];
        carry += scan[i];
      }
      if (s < p.S) prefix[s + 1] = before + w;
      __syncthreads();
    }
  }
  const int total = prefix[p.S];
  const int share = max((total + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x), p.min_share);
  const int cta = blockIdx.x;
  const int64_t pos0 = static_cast<int64_t>(cta) * share;
  const int end = static_cast<int>(min(pos0 + share, static_cast<int64_t>(total)));
  float* part = p.ws;                                                    // [2 * ctas][ROWS][D]
  float* part_stat = part + static_cast<size_t>(2) * gridDim.x * ROWS * D;  // [2 * ctas][ROWS][2]
  Task* tasks = reinterpret_cast<Task*>(part_stat + static_cast<size_t>(2) * gridDim.x * ROWS * 2);
  if (tid == 0) tasks[cta].valid = 0;
  if (pos0 >= end) return;

  const uint32_t ring = smem_addr(smem) + warp * (ST * 2 * L::PAGE_B);
  uint64_t* wbar = bars + warp * ST;
  uint32_t phases = 0;   // bit i: parity of the next wait on stage i
  bool dead = false;     // a wait gave up: nothing more is loaded
  int s = 0;
  int pos = static_cast<int>(pos0);
  while (pos < end) {
    // ---- the segment: session s, KV head h, row tile, pages p0 .. p1 ------------
    {
      int lo = s, hi = p.S;  // the last session whose first unit is <= pos
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (prefix[mid] <= pos) lo = mid; else hi = mid;
      }
      s = lo;
    }
    int q_begin;
    const int n_tok = query_tokens(p, s, q_begin), rows = n_tok * p.G, len = held_tokens(p, s);
    const int pages = max(1, (len + q8::PAGE - 1) / q8::PAGE), tiles = (rows + ROWS - 1) / ROWS;
    const int gi = (pos - prefix[s]) / pages, p0 = (pos - prefix[s]) % pages;
    const int p1 = min(pages, p0 + (end - pos));
    const int h = gi / tiles, row0 = gi % tiles * ROWS;
    const int group_begin = pos - p0, group_end = group_begin + pages;
    const int mine = max(0, (p1 - p0 - warp + NW - 1) / NW);   // this warp's pages: p0 + warp + NW * i
    const int32_t* trow = p.table + static_cast<int64_t>(s) * p.width + p0 + warp;
    const float* ksh = p.k_scale + static_cast<int64_t>(h) * p.n_pages;
    const float* vsh = p.v_scale + static_cast<int64_t>(h) * p.n_pages;

    // lane j holds page 32 * batch + j of this warp: id, K scale, log2 and
    // reciprocal of the V scale (at least 2^-100, so a zero scale stays harmless);
    // the next batch beside it
    int id_c, id_n = -1;
    float ks_c, lv_c, iv_c, ks_n = 0.f, lv_n = 0.f, iv_n = 1.f;
    const auto fetch = [&](int base, int& id, float& ks, float& lv, float& iv) {
      id = -1;
      ks = 0.f;
      float vs = 1.f;
      const int i = base + lane;
      if (i < mine && (p0 + warp + NW * i) * q8::PAGE < len) {
        const int x = trow[NW * i];
        if (static_cast<unsigned>(x) < static_cast<unsigned>(p.n_pages)) {
          id = x;
          ks = ksh[x];
          vs = fmaxf(vsh[x], 7.8886090522101181e-31f);
        } else if (p.status) {
          atomicOr(p.status, IC_DEVFLAG_BAD_ROW);
        }
      }
      lv = log2f(vs);
      iv = 1.f / vs;
    };
    const auto issue = [&](int i, int page) {
      const int st = i % ST;
      if (lane == 0 && page >= 0 && !dead) {
        unsigned char* dst = smem + warp * (ST * 2 * L::PAGE_B) + st * 2 * L::PAGE_B;
        mbar_arrive_expect_tx(wbar + st, 2 * L::PAGE_B);
        const int y = D == 64 ? page * 8 : page * 16;
#pragma unroll
        for (int x = 0; x < (D == 256 ? 2 : 1); ++x) {
          tc::tma_load_3d(dst + x * 2048, &mk, x * 128, y, h, wbar + st);
          tc::tma_load_3d(dst + L::PAGE_B + x * 2048, &mv, x * 128, y, h, wbar + st);
        }
      }
    };
    fetch(0, id_c, ks_c, lv_c, iv_c);
#pragma unroll
    for (int i = 0; i < ST; ++i) {
      const int page = __shfl_sync(FULL_MASK, id_c, i);
      if (i < mine) issue(i, page);
    }
    if (mine > 32) fetch(32, id_n, ks_n, lv_n, iv_n);

    // ---- q as the B operand; head rows past the session's are zero ---------------
    uint32_t qb[NG][NC * 4][2];
    float qmul[NG][2];
    int lim[NG][2];      // keys that rows 2 tq, 2 tq + 1 of each n-tile see
#pragma unroll
    for (int nt = 0; nt < NG; ++nt) {
      const int r = row0 + nt * 8 + g;
      const bool ok = r < rows;
      const QT* src = static_cast<const QT*>(p.q);
      if (ok) src += (q_begin + r / p.G) * p.q_stride_t + (h * p.G + r % p.G) * p.q_stride_h;
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
          qb[nt][c * 4 + j][0] = o[2 * j];
          qb[nt][c * 4 + j][1] = o[2 * j + 1];
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        qmul[nt][i] = __shfl_sync(FULL_MASK, back, (2 * tq + i) * 4) * p.sl2;
        const int ri = row0 + nt * 8 + 2 * tq + i;
        lim[nt][i] = ri < rows ? len - n_tok + ri / p.G + 1 : 0;
      }
    }
    const int lim_all = len - n_tok + row0 / p.G + 1;  // keys that every row of the tile sees

    float M[NG][2], l[NG][2], o[NG][MT][4];
#pragma unroll
    for (int nt = 0; nt < NG; ++nt) {
      M[nt][0] = M[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) o[nt][mt][0] = o[nt][mt][1] = o[nt][mt][2] = o[nt][mt][3] = 0.f;
    }

    // ---- stream ---------------------------------------------------------------------
    for (int i = 0; i < mine; ++i) {
      if (i > 0 && (i & 31) == 0) {
        id_c = id_n;
        ks_c = ks_n;
        lv_c = lv_n;
        iv_c = iv_n;
        if (i + 32 < mine) fetch(i + 32, id_n, ks_n, lv_n, iv_n);
      }
      const int page = __shfl_sync(FULL_MASK, id_c, i & 31);
      const float ks = __shfl_sync(FULL_MASK, ks_c, i & 31);
      const float lv = __shfl_sync(FULL_MASK, lv_c, i & 31), inv_vs = __shfl_sync(FULL_MASK, iv_c, i & 31);
      const int st = i % ST;
      if (page >= 0 && !dead) {
        const bool ok = mbar_wait_bounded(wbar + st, (phases >> st) & 1, p.status);
        dead = !__all_sync(FULL_MASK, ok);
        phases ^= 1u << st;
      }
      if (page >= 0 && !dead) {
        const uint32_t kp = ring + st * 2 * L::PAGE_B, vp = kp + L::PAGE_B;
        const int tok0 = (p0 + warp + NW * i) * q8::PAGE;
        float acc[NG][4];
#pragma unroll
        for (int nt = 0; nt < NG; ++nt) acc[nt][0] = acc[nt][1] = acc[nt][2] = acc[nt][3] = 0.f;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const int chunk = D == 64 ? tq : (c >> 1) * 8 + 2 * tq + (c & 1);
          const uint4 k0 = lds128(kp + page_off<D>(g, chunk)), k1 = lds128(kp + page_off<D>(g + 8, chunk));
          const uint32_t w0[4] = {k0.x, k0.y, k0.z, k0.w}, w1[4] = {k1.x, k1.y, k1.z, k1.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint32_t a0, a1, a2, a3;
            q8::decode4_h2<CODE>(w0[j], a0, a2);
            q8::decode4_h2<CODE>(w1[j], a1, a3);
#pragma unroll
            for (int nt = 0; nt < NG; ++nt)
              Mma<__half>::run(acc[nt], a0, a1, a2, a3, qb[nt][c * 4 + j][0], qb[nt][c * 4 + j][1]);
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
      __syncwarp();
      {
        const int nx = i + ST;
        const int from_c = __shfl_sync(FULL_MASK, id_c, nx & 31), from_n = __shfl_sync(FULL_MASK, id_n, nx & 31);
        if (nx < mine) issue(nx, (nx >> 5) == (i >> 5) ? from_c : from_n);
      }
    }
    if (dead) {  // copies in flight land before their buffers are given up (short waits)
      for (int st = 0; st < ST; ++st) mbar_wait_bounded(wbar + st, (phases >> st) & 1, nullptr, 200000000ull);
    }
#pragma unroll
    for (int nt = 0; nt < NG; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) l[nt][e] += __shfl_xor_sync(FULL_MASK, l[nt][e], x);

    // ---- join the warps ---------------------------------------------------------------
    __syncthreads();  // every warp is done with its ring, which the O rows alias
    float* wo = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int nt = 0; nt < NG; ++nt) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = nt * 8 + 2 * tq + e;
        float* dst = wo + (warp * ROWS + row) * L::PITCH + (D / 8) * g;
        // elements 2 mt + {0, 1} of this lane's dims are o[mt][e], o[mt][e + 2]
#pragma unroll
        for (int c = 0; c < MT / 2; ++c)
          reinterpret_cast<float4*>(dst)[c] =
              make_float4(o[nt][2 * c][e], o[nt][2 * c][e + 2], o[nt][2 * c + 1][e], o[nt][2 * c + 1][e + 2]);
        if (g == 0) {
          stat[(warp * ROWS + row) * 2] = M[nt][e];
          stat[(warp * ROWS + row) * 2 + 1] = l[nt][e];
        }
      }
    }
    __syncthreads();
    const bool whole = p0 == 0 && p1 == pages;
    const int slot = 2 * cta + (pos == pos0 ? 0 : 1);
    for (int e = tid; e < ROWS * (D / 4); e += NW * 32) {
      const int row = e / (D / 4), d0 = e % (D / 4) * 4, r = row0 + row;
      float m = -INFINITY, lsum = 0.f;
#pragma unroll
      for (int w = 0; w < NW; ++w) m = fmaxf(m, stat[(w * ROWS + row) * 2]);
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const float mw = stat[(w * ROWS + row) * 2];
        const float f = mw == -INFINITY ? 0.f : tc::ex2(mw - m);
        lsum = fmaf(stat[(w * ROWS + row) * 2 + 1], f, lsum);
        const float4 u = *reinterpret_cast<const float4*>(wo + (w * ROWS + row) * L::PITCH + d0);
        x.x = fmaf(u.x, f, x.x); x.y = fmaf(u.y, f, x.y); x.z = fmaf(u.z, f, x.z); x.w = fmaf(u.w, f, x.w);
      }
      if (!whole) {
        *reinterpret_cast<float4*>(part + (static_cast<size_t>(slot) * ROWS + row) * D + d0) = x;
        if (d0 == 0) {
          part_stat[(static_cast<size_t>(slot) * ROWS + row) * 2] = m;
          part_stat[(static_cast<size_t>(slot) * ROWS + row) * 2 + 1] = lsum;
        }
      } else if (r < rows) {
        const float inv = lsum > 0.f ? 1.f / lsum : lsum == lsum ? 0.f : lsum;  // NaN stays NaN
        const int64_t orow = static_cast<int64_t>(q_begin + r / p.G) * p.Hq + h * p.G + r % p.G;
        QT* dst = static_cast<QT*>(p.out) + orow * D + d0;
        const uint32_t lo = static_cast<uint32_t>(Mma<QT>::bits(x.x * inv)) | (static_cast<uint32_t>(Mma<QT>::bits(x.y * inv)) << 16);
        const uint32_t hi = static_cast<uint32_t>(Mma<QT>::bits(x.z * inv)) | (static_cast<uint32_t>(Mma<QT>::bits(x.w * inv)) << 16);
        *reinterpret_cast<uint2*>(dst) = make_uint2(lo, hi);
        if (d0 == 0 && p.lse) p.lse[orow] = lsum > 0.f ? (m - LIFT + log2f(lsum)) * LN2 : lsum == lsum ? -INFINITY : lsum;
      }
    }
    if (tid == 0 && !whole && p1 < pages && group_begin >= pos0) {  // this CTA holds the group's first page, not its last
      Task t;
      t.valid = 1;
      t.s = s;
      t.h = h;
      t.tile = row0 / ROWS;
      t.last_cta = (group_end - 1) / share;
      t.first_slot = slot;
      tasks[cta] = t;
    }
    pos += p1 - p0;
    fence_proxy_async_smem();  // the O rows were written through the generic proxy; copies follow
    __syncthreads();
  }
}

// Joins the partials of the groups that lie in several shares: one CTA per
// (CTA where such a group begins, row).  Eight subgroups of lanes take every
// eighth partial each; their sums are joined in order.
template <typename QT, int D, int NG>
__global__ void __launch_bounds__(8 * (D / 4)) join_kernel(const Params p, int ctas) {
  constexpr int ROWS = 8 * NG, LN = D / 4;
  __shared__ float4 sx[8][LN];
  __shared__ float sl[8];
  grid_dependency_wait();
  grid_launch_dependents();
  const float* part = p.ws;
  const float* part_stat = part + static_cast<size_t>(2) * ctas * ROWS * D;
  const Task* tasks = reinterpret_cast<const Task*>(part_stat + static_cast<size_t>(2) * ctas * ROWS * 2);
  const Task t = tasks[blockIdx.x];
  if (!t.valid) return;
  int q_begin;
  const int rows = query_tokens(p, t.s, q_begin) * p.G;
  const int row = blockIdx.y, r = t.tile * ROWS + row;
  if (r >= rows) return;
  const int sub = threadIdx.x / LN, ln = threadIdx.x % LN;
  const int n = t.last_cta - static_cast<int>(blockIdx.x) + 1;
  // partial i: the first share's, then slot 0 of each later one
  const auto at = [&](int i) {
    return (static_cast<size_t>(i == 0 ? t.first_slot : 2 * (blockIdx.x + i)) * ROWS + row);
  };
  float m = -INFINITY;
  for (int i = sub; i < n; i += 8) m = fmaxf(m, part_stat[at(i) * 2]);
  if (ln == 0) sl[sub] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) m = fmaxf(m, sl[i]);
  __syncthreads();
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
  float lsum = 0.f;
#pragma unroll 4
  for (int i = sub; i < n; i += 8) {
    const float mi = part_stat[at(i) * 2], li = part_stat[at(i) * 2 + 1];
    const float4 u = *reinterpret_cast<const float4*>(part + at(i) * D + 4 * ln);
    const float f = mi == -INFINITY ? 0.f : tc::ex2(mi - m);
    lsum = fmaf(li, f, lsum);
    x.x = fmaf(u.x, f, x.x); x.y = fmaf(u.y, f, x.y); x.z = fmaf(u.z, f, x.z); x.w = fmaf(u.w, f, x.w);
  }
  sx[sub][ln] = x;
  if (ln == 0) sl[sub] = lsum;
  __syncthreads();
  if (sub != 0) return;
  lsum = 0.f;
  x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float4 u = sx[i][ln];
    x.x += u.x; x.y += u.y; x.z += u.z; x.w += u.w;
    lsum += sl[i];
  }
  const float inv = lsum > 0.f ? 1.f / lsum : lsum == lsum ? 0.f : lsum;
  const int64_t orow = static_cast<int64_t>(q_begin + r / p.G) * p.Hq + t.h * p.G + r % p.G;
  QT* dst = static_cast<QT*>(p.out) + orow * D + 4 * ln;
  const uint32_t lo = static_cast<uint32_t>(Mma<QT>::bits(x.x * inv)) | (static_cast<uint32_t>(Mma<QT>::bits(x.y * inv)) << 16);
  const uint32_t hi = static_cast<uint32_t>(Mma<QT>::bits(x.z * inv)) | (static_cast<uint32_t>(Mma<QT>::bits(x.w * inv)) << 16);
  *reinterpret_cast<uint2*>(dst) = make_uint2(lo, hi);
  if (ln == 0 && p.lse) p.lse[orow] = lsum > 0.f ? (m - LIFT + log2f(lsum)) * LN2 : lsum == lsum ? -INFINITY : lsum;
}

constexpr int SMS = 148;

template <typename QT, int D, int CODE, int NG>
int launch(const Params& p, const ic_paged_attn_args& a, cudaStream_t st) {
  CUtensorMap mk, mv;
  int rc;
  if ((rc = page_map(&mk, a.k, a.pool_tokens, p.H, D)) != IC_OK) return rc;
  if ((rc = page_map(&mv, a.v, a.pool_tokens, p.H, D)) != IC_OK) return rc;
  auto kern = stream_kernel<QT, D, CODE, NG>;
  static PerDeviceLimit limit;
  const int smem = Layout<D, NG>::bytes(p.S);
  if ((rc = ensure_dynamic_smem(kern, smem, &limit)) != IC_OK) return rc;
  Params params = p;
  int ctas = SMS * ctas_per_sm(D, NG);
  void* args[] = {&mk, &mv, &params};
  if ((rc = launch_pdl(reinterpret_cast<const void*>(kern), dim3(ctas), dim3(NW * 32), smem, st, args,
                       "paged_attention (stream)")) != IC_OK)
    return rc;
  void* jargs[] = {&params, &ctas};
  return launch_pdl(reinterpret_cast<const void*>(join_kernel<QT, D, NG>), dim3(ctas, 8 * NG), dim3(8 * (D / 4)), 0, st,
                    jargs, "paged_attention (join)");
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

int64_t stream_workspace(int head_dim, int rows_per_tile) {
  const int64_t ctas = SMS * ctas_per_sm(head_dim, rows_per_tile / 8);
  return 2 * ctas * rows_per_tile * (head_dim + 2) * 4 + ctas * static_cast<int64_t>(sizeof(Task));
}

int launch_stream(const Params& p, const ic_paged_attn_args& a, cudaStream_t st) {
  const bool one = stream_rows(static_cast<int64_t>(a.max_count) * p.G) == 8;
  return a.q_dtype == IC_F16 ? launch_dim<__half>(p, a, st, one) : launch_dim<__nv_bfloat16>(p, a, st, one);
}

}  // namespace paged
}  // namespace ic
