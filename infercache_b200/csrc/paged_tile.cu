// Attention of many query tokens per session over 8-bit pages (prompts in
// chunks on top of what the cache holds): the tile kernel, bound by the tensor
// cores (4 * D operations per query row and key).
//
// A session's query rows (its new tokens x the query heads of a KV head) are
// cut into tiles of 128; one CTA per (session, KV head, pair of tiles), the
// latest rows (the longest key ranges) first.  Both tiles share every 128-key
// tile, so a key's codes are converted once per 256 rows.  Roles:
//   warpgroup 0  warp 0 issues S = Q K^T (tcgen05.mma, fp16 operands in shared
//                memory, fp32 in TMEM), warp 1 issues O += P V (P read from TMEM);
//   warpgroup 1  loads the pages' codes (16 bytes a lane, two tiles ahead in
//                registers), converts them to fp16 -- exact for both formats --
//                and stores them as 128-byte-swizzled operand tiles into a ring,
//                in consumption order K0 K1 V0 K2 V1 ..., with the pages' scales
//                beside them; rows behind the session's last token become zero;
//   warpgroups 2, 3  one thread per query row of tile a, b: q into shared memory
//                as fp16 (bf16 rows times a power of two), then per key tile
//                u = S * (k scale * softmax scale) + log2(v scale),
//                P' = 2^(u - M + 7) as fp16 into TMEM, l += sum P' / v scale,
//                O rescaled only when u passes M by more than 8.
// The V scales sit in the exponent for the reason given in paged_stream.cu.
// The score tiles take turns in one TMEM buffer: each row copies its scores to
// registers at once, so the next Q K^T overlaps its exponentials.  P is handed
// over in two halves of 64 keys.
// Measured (4 sessions x 1500-2048 tokens x 16 heads over 4096-8192 keys, D =
// 128, e4m3): 1.9 us per step of two query tiles x 128 keys, of which the tensor
// cores need 1.1, plus about 10 us per CTA to begin and end.  Codes loaded one
// tile ahead instead of two, 325 us a call instead of 285; a pass of its own
// for the scores' scaling, no change; two score buffers with P in the scores'
// place, 337 us against 327 at the time.
// 256 dims: O takes half of TMEM, so a CTA has one query tile; warpgroup 3 is a
// second pair of hands for the codes, and the ring holds two key tiles.  Chunks of
// 1500 to 2048 tokens of 4 sessions over 4-8k keys: 560 us, 0.66 of the measured
// bf16 rate (3831 in the streaming kernel).
// TMEM columns: S 0, P_a 128, P_b 192, O_a 256, O_b 384.  Registers: 512
// threads start with 128 each; warpgroups 0 and 1 give theirs to the softmax
// (56 + 96 + 176 + 176 = 504 of 512; 256 dims: 56 + 96 + 176 + 96).
#include <cuda.h>
#include <math.h>

#include <type_traits>

#include "common.cuh"
#include "exp2_poly.cuh"
#include "launch.cuh"
#include "mma_helpers.cuh"
#include "paged_attn.cuh"
#include "q8.cuh"
#include "tc05.cuh"

namespace ic {
namespace paged {
namespace {

constexpr int TB = 128;                // query rows and keys per tile
constexpr int SUB = TB * 64 * 2;       // one 64-column swizzled sub-tile: 16 KB
constexpr int THREADS = 512;
// Query tiles per CTA, warps that convert codes, K / V ring slots.
template <int D> constexpr int TILES = D == 256 ? 1 : 2;
template <int D> constexpr int CONVERTERS = D == 256 ? 8 : 4;
template <int D> constexpr int SLOTS = D == 256 ? 2 : 5;
constexpr int NSC = 8;                 // key tiles whose scales are kept: the ring runs at most 3 ahead of the softmax
constexpr int SORTED = 128;            // up to this many sessions are taken longest first
constexpr float SLACK = 8.f, LIFT = 7.f;
constexpr float MIN_FACTOR = 1.17549435e-38f;  // 2^-126

template <int D>
struct Lay {
  static constexpr int TILE = D / 64 * SUB;
  static constexpr int RS = SLOTS<D>;
  static constexpr int RING = TILES<D> * TILE;
  static constexpr int SCALES = RING + RS * TILE;      // [NSC][3][8]: k scale, log2 v scale, 1 / v scale
  static constexpr int BARS = SCALES + NSC * 24 * 4;   // 16-byte aligned rows of 8
  static constexpr int NBAR = 22;
  static constexpr int MISC = BARS + NBAR * 8;         // TMEM address, abort, session, pair; the scan's 16 sums
  static constexpr int BYTES = MISC + 16 + 64 + 1024;  // + alignment
};

__device__ __forceinline__ uint64_t kdesc(uint32_t tile, int kk) {
  return tc::sw128_desc(tile + (kk >> 2) * SUB + (kk & 3) * 32, 16, 1024);
}
__device__ __forceinline__ uint64_t mndesc(uint32_t tile, int kk) { return tc::sw128_desc(tile + kk * 2048, SUB, 1024); }

__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int32_t* status, volatile int* abort) {
  int ok = *abort ? 0 : (mbar_wait_bounded(bar, parity, status) ? 1 : 0);
  ok = __all_sync(FULL_MASK, ok);
  if (!ok) *abort = 1;
  return ok != 0;
}
__device__ __forceinline__ bool one_wait(uint64_t* bar, uint32_t parity, int32_t* status, volatile int* abort) {
  if (*abort) return false;
  if (mbar_wait_bounded(bar, parity, status)) return true;
  *abort = 1;
  return false;
}
__device__ __forceinline__ uint32_t half2_bits(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void sts128(uint32_t addr, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

template <typename QT, int D, int CODE>
__global__ void __launch_bounds__(THREADS, 1) tile_kernel(const Params p) {
  using L = Lay<D>;
  constexpr int NS = D / 64;  // 64-column sub-tiles of an operand row
  constexpr int NT = TILES<D>, CW = CONVERTERS<D>, RS = L::RS;
  constexpr int PW = 8 / CW;  // pages of a key tile that a converting warp takes
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = smem_raw + ((1024 - (smem_addr(smem_raw) & 1023)) & 1023);
  const uint32_t sbase = smem_addr(smem);
  float* scales = reinterpret_cast<float*>(smem + L::SCALES);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::BARS);
  uint64_t* q_full = bars + 0;
  uint64_t* r_full = bars + 1;    // [RS]
  uint64_t* r_empty = bars + 6;   // [RS]
  uint64_t* s_full = bars + 11;   // [2]
  uint64_t* s_free = bars + 13;
  uint64_t* p_full = bars + 14;   // [2][2]: tile, half of its keys
  uint64_t* pv_done = bars + 18;  // [2]
  uint64_t* mma_done = bars + 20;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::MISC);
  volatile int* abort = reinterpret_cast<volatile int*>(smem + L::MISC + 4);
  volatile int* found = reinterpret_cast<volatile int*>(smem + L::MISC + 8);  // session, pair
  int* sums = reinterpret_cast<int*>(smem + L::MISC + 16);
  int2* sorted = reinterpret_cast<int2*>(smem + L::RING);  // before the ring is written
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (tid == 0) {
    *abort = 0;
    found[0] = -1;
    mbar_init(q_full, NT * 128);
    for (int i = 0; i < RS; ++i) {
      mbar_init(r_full + i, CW * 32);
      mbar_init(r_empty + i, 1);
    }
    for (int x = 0; x < 2; ++x) {
      mbar_init(s_full + x, 1);
      mbar_init(p_full + 2 * x, 128);
      mbar_init(p_full + 2 * x + 1, 128);
      mbar_init(pv_done + x, 1);
    }
    mbar_init(s_free, 128);
    mbar_init(mma_done, 2);
    fence_barrier_init();
  }
  if (warp == 0) tc::tmem_alloc(tmem_slot, 512);
  grid_dependency_wait();
  grid_launch_dependents();

  // ---- which session and pair of tiles -------------------------------------------
  // A few sessions are taken longest first (the CTAs that run last then are the
  // short ones), many in their order.
  const int h = blockIdx.x % p.H, unit = blockIdx.x / p.H;
  const auto pairs_of = [&](int x) {
    int begin;
    const int rows = query_tokens(p, x, begin) * p.G;
    return rows > p.few_rows ? (rows + NT * TB - 1) / (NT * TB) : 0;
  };
  if (p.S <= SORTED) {
    int own = 0, held = 0;
    if (tid < p.S) {
      own = pairs_of(tid);
      held = held_tokens(p, tid);
      sorted[tid] = make_int2(held, own);
    }
    __syncthreads();
    int before = 0;
    for (int t = 0; t < p.S; ++t) {
      const int2 o = sorted[t];
      if (o.x > held || (o.x == held && t < tid)) before += o.y;
    }
    const int at = unit - before;
    if (tid < p.S && at >= 0 && at < own) {
      found[0] = tid;
      found[1] = own - 1 - at;
    }
    __syncthreads();
  } else {
    int carry = 0;
    for (int s0 = 0; s0 < p.S; s0 += THREADS) {
      const int s = s0 + tid;
      const int own = s < p.S ? pairs_of(s) : 0;
      int upto = own;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(FULL_MASK, upto, o);
        if (lane >= o) upto += x;
      }
      if (lane == 31) sums[warp] = upto;
      __syncthreads();
      int before = carry;
      for (int i = 0; i < THREADS / 32; ++i) {
        if (i < warp) before += sums[i];
        carry += sums[i];
      }
      const int at = unit - (before + upto - own);
      if (at >= 0 && at < own) {
        found[0] = s;
        found[1] = own - 1 - at;
      }
      __syncthreads();
      if (found[0] >= 0) break;
    }
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = *tmem_slot;
  const int s = found[0], pair = found[1];
  if (s < 0) {  // more CTAs than units: the launch counts with the most that there can be
    if (warp == 0) tc::tmem_dealloc(tmem, 512);
    return;
  }
  int q_begin;
  const int n_tok = query_tokens(p, s, q_begin), rows = n_tok * p.G, len = held_tokens(p, s);
  const int row_a = pair * NT * TB;
  const bool has_b = NT == 2 && row_a + TB < rows;
  // keys that row r sees: len - n_tok + r / G + 1; a tile's last row sets its range
  const auto tiles_of = [&](int row0) {
    const int last = min(row0 + TB, rows) - 1;
    return max(1, (len - n_tok + last / p.G + 1 + TB - 1) / TB);
  };
  const int na = tiles_of(row_a), nb = has_b ? tiles_of(row_a + TB) : 0;
  const int n = has_b ? nb : na;
  const auto u_k = [&](int j) { return j == 0 ? 0 : 2 * j - 1; };
  const auto u_v = [&](int j) { return j == n - 1 ? 2 * n - 1 : 2 * j + 2; };

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    constexpr uint32_t IDESC = tc::idesc_f16(0, TB, TB, 0, 0);
    constexpr uint32_t IDESC_PV = tc::idesc_f16(0, TB, D, 0, 1);
    if (warp == 0 && lane == 0) {
      // ---- S_a(j), S_b(j) in turn through the one score buffer ---------------------
      int n_s = 0;
      auto issue_s = [&](int x, int j) -> bool {
        if (n_s >= 1 && !one_wait(s_free, (n_s - 1) & 1, p.status, abort)) return false;
        tc::fence_after();
        const uint32_t sk = sbase + L::RING + (u_k(j) % RS) * L::TILE;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
          tc::mma_ss(tmem, kdesc(sbase + x * L::TILE, kk), kdesc(sk, kk), IDESC, kk > 0 ? 1u : 0u);
        tc::commit(s_full + x);
        ++n_s;
        return true;
      };
      bool ok = one_wait(q_full, 0, p.status, abort);
      for (int j = 0; ok && j < n; ++j) {
        const int u = u_k(j);
        if (!(ok = one_wait(r_full + u % RS, (u / RS) & 1, p.status, abort))) break;
        if (j < na && !(ok = issue_s(0, j))) break;
        if (j < nb && !(ok = issue_s(1, j))) break;
        tc::commit(r_empty + u % RS);
      }
      tc::commit(mma_done);
      mbar_wait_bounded(mma_done, 0, p.status);
    } else if (warp == 1 && lane == 0) {
      // ---- O_a += P_a V(j), O_b += P_b V(j) -------------------------------------------
      bool ok = true;
      for (int j = 0; ok && j < n; ++j) {
        // P first: it shows that S(j) is done, hence that the slot's last tenant was
        // there; without that a parity alone cannot tell this phase from the one before
        const int u = u_v(j);
        bool here = false;
        const uint32_t sv = sbase + L::RING + (u % RS) * L::TILE;
        for (int x = 0; x < 2; ++x) {
          if (j >= (x ? nb : na)) continue;
          for (int half = 0; half < 2; ++half) {
            if (!(ok = one_wait(p_full + 2 * x + half, j & 1, p.status, abort))) break;
            if (!here && !(ok = one_wait(r_full + u % RS, (u / RS) & 1, p.status, abort))) break;
            here = true;
            tc::fence_after();
#pragma unroll
            for (int kk = 0; kk < TB / 32; ++kk)
              tc::mma_ts(tmem + 256 + x * 128, tmem + 128 + x * 64 + half * 32 + kk * 8, mndesc(sv, 4 * half + kk), IDESC_PV,
                         (j > 0 || half > 0 || kk > 0) ? 1u : 0u);
          }
          if (!ok) break;
          tc::commit(pv_done + x);
        }
        if (ok) tc::commit(r_empty + u % RS);
      }
      tc::commit(mma_done);
      mbar_wait_bounded(mma_done, 0, p.status);
    }
  } else if (warp < 8 || (CW == 8 && warp >= 12)) {
    // ---- codes to operand tiles -----------------------------------------------------
    asm volatile("setmaxnreg.dec.sync.aligned.u32 96;");
    const int cw = warp < 8 ? warp - 4 : warp - 8, t8 = lane >> 2, c4 = lane & 3;
    const int32_t* trow = p.table + static_cast<int64_t>(s) * p.width;
    const int64_t plane = static_cast<int64_t>(h) * p.n_pages;
    const uint8_t* kc = static_cast<const uint8_t*>(p.k) + plane * q8::PAGE * D;
    const uint8_t* vc = static_cast<const uint8_t*>(p.v) + plane * q8::PAGE * D;
    const int total = 2 * n;
    const auto what = [&](int u, int& j) -> bool {  // ring position to key tile; whether it is V
      const bool is_v = u > 0 && (u == total - 1 || (u & 1) == 0);
      j = is_v ? (u == total - 1 ? n - 1 : u / 2 - 1) : (u + 1) / 2;
      return is_v;
    };
    // this warp's tokens of a key tile are pages PW cw .. PW cw + PW - 1 of its eight
    const auto pages_at = [&](int u, int* id) {
      int j;
      what(u, j);
#pragma unroll
      for (int i = 0; i < PW; ++i) {
        const int pg = j * 8 + cw * PW + i;
        id[i] = -1;
        if (u < total && pg * q8::PAGE < len) {
          const int x = trow[pg];
          if (static_cast<unsigned>(x) < static_cast<unsigned>(p.n_pages))
            id[i] = x;
          else if (p.status && lane == 0)
            atomicOr(p.status, IC_DEVFLAG_BAD_ROW);
        }
      }
    };
    // Two ring positions' codes stay in registers (positions alternate between
    // them); as soon as a vector is stored, the one two positions on is loaded in
    // its place, so a load has two tiles' time to arrive.
    struct Held {
      uint4 reg[2 * PW][NS];
      float ks, vs;   // lane i < PW: the scales of this warp's page i ...
      bool mine;      // ... and whether there is such a page
    };
    const uint32_t lane_codes = t8 * D + c4 * 16;
    // One page's four vectors (two groups of 8 tokens): where this lane's part of
    // it begins, and whether every token of it is held.
    struct At {
      const uint8_t* ptr;
      int tokens;   // of the page that are held: 16 but for the last page, 0 for none
    };
    const auto page_at = [&](int u, const int* id, int i) -> At {
      int j;
      const uint8_t* codes = what(u, j) ? vc : kc;
      const int left = len - (j * 8 + cw * PW + i) * q8::PAGE;
      return At{codes + static_cast<int64_t>(max(id[i], 0)) * (q8::PAGE * D) + lane_codes, id[i] < 0 ? 0 : min(left, q8::PAGE)};
    };
    const auto load_one = [&](const At& at, int g, int sub) -> uint4 {
      if (at.tokens < q8::PAGE && (g & 1) * 8 + t8 >= at.tokens) return make_uint4(0, 0, 0, 0);
      return *reinterpret_cast<const uint4*>(at.ptr + (g & 1) * 8 * D + sub * 64);
    };
    const auto load_scales = [&](const int* id, Held& b) {
      const int page = id[PW == 1 ? 0 : lane & 1];
      b.mine = lane < PW && page >= 0;
      b.ks = b.vs = 1.f;
      if (b.mine) {
        b.ks = p.k_scale[plane + page];
        b.vs = p.v_scale[plane + page];
      }
    };
    int next[PW], later[PW];  // page ids two and three positions on
    const auto step = [&](int u, Held& b) -> bool {
      pages_at(u + 3, later);
      const int st = u % RS;
      if (u >= RS && !warp_wait(r_empty + st, ((u / RS) - 1) & 1, p.status, abort)) return false;
      int j;
      const bool is_v = what(u, j);
      if (!is_v && lane < PW) {
        float* sc = scales + (j % NSC) * 24 + cw * PW + lane;
        const float k1 = fmaxf(b.ks, 7.8886090522101181e-31f), v1 = fmaxf(b.vs, 7.8886090522101181e-31f);
        sc[0] = k1;                                   // at least 2^-100: a zero scale stays harmless
        sc[8] = b.mine ? log2f(v1) : -INFINITY;       // no page: no weight
        sc[16] = b.mine ? 1.f / v1 : 0.f;
      }
      load_scales(next, b);
      const At at[2] = {page_at(u + 2, next, 0), page_at(u + 2, next, PW - 1)};
      const uint32_t dst = sbase + L::RING + st * L::TILE + (cw * PW * 16 + t8) * 128 + (((2 * c4) ^ t8) << 4);
#pragma unroll
      for (int g = 0; g < 2 * PW; ++g) {
#pragma unroll
        for (int sub = 0; sub < NS; ++sub) {
          const uint4 w = b.reg[g][sub];
          uint32_t x[8];
          q8::decode4_h2<CODE>(w.x, x[0], x[1]);
          q8::decode4_h2<CODE>(w.y, x[2], x[3]);
          q8::decode4_h2<CODE>(w.z, x[4], x[5]);
          q8::decode4_h2<CODE>(w.w, x[6], x[7]);
          sts128(dst + sub * SUB + g * 1024, x[0], x[1], x[2], x[3]);
          sts128((dst ^ 16) + sub * SUB + g * 1024, x[4], x[5], x[6], x[7]);
          b.reg[g][sub] = load_one(at[g >> 1], g, sub);
        }
      }
      fence_proxy_async_smem();
      tc::mbar_arrive(r_full + st);
#pragma unroll
      for (int i = 0; i < PW; ++i) next[i] = later[i];
      return true;
    };
    Held even, odd;
    const auto fill = [&](int u, Held& b) {
      pages_at(u, next);
      load_scales(next, b);
      const At at[2] = {page_at(u, next, 0), page_at(u, next, PW - 1)};
#pragma unroll
      for (int g = 0; g < 2 * PW; ++g)
#pragma unroll
        for (int sub = 0; sub < NS; ++sub) b.reg[g][sub] = load_one(at[g >> 1], g, sub);
    };
    fill(0, even);
    fill(1, odd);
    pages_at(2, next);
    for (int u = 0; u < total; u += 2) {  // total is even
      if (!step(u, even) || !step(u + 1, odd)) break;
    }
  } else {
    // ---- softmax: one thread per query row of tile x -----------------------------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 176;");
    const int x = (warp - 8) >> 2;
    const int nx = x ? nb : na;
    const int quarter = warp & 3, r = quarter * 32 + lane;
    const int row0 = row_a + x * TB, qr = row0 + r;
    const bool valid = nx > 0 && qr < rows;
    const int64_t tok = q_begin + (valid ? qr / p.G : 0), head = h * p.G + (valid ? qr % p.G : 0);
    // a negative softmax scale goes into q's sign: f below stays positive
    const uint32_t flip = p.sl2 < 0.f ? 0x80008000u : 0u;
    float qmul = fabsf(p.sl2);
    if (nx > 0) {
      const QT* src = static_cast<const QT*>(p.q) + tok * p.q_stride_t + head * p.q_stride_h;
      // at most 16 vectors at a time; two passes where the row has more (256 dims)
      constexpr int QC = D / 8 < 16 ? D / 8 : 16;
      uint4 w[QC];
      const auto load_q = [&](int c0) {
#pragma unroll
        for (int c = 0; c < QC; ++c) w[c] = valid ? reinterpret_cast<const uint4*>(src)[c0 + c] : make_uint4(0, 0, 0, 0);
      };
      constexpr bool SCALE_Q = std::is_same<QT, __nv_bfloat16>::value;
      float f = 1.f;
      if (SCALE_Q) {
        // bf16 to fp16: a power of two brings the row's largest finite value into [2^13, 2^14)
        uint32_t m = 0;
        for (int c0 = D / 8 - QC; c0 >= 0; c0 -= QC) {
          load_q(c0);
#pragma unroll
          for (int c = 0; c < QC; ++c) {
            const uint32_t* u = reinterpret_cast<const uint32_t*>(&w[c]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t lo = (u[i] << 16) & 0x7fffffffu, hi = u[i] & 0x7fff0000u;
              m = max(m, lo < 0x7f800000u ? lo : 0u);
              m = max(m, hi < 0x7f800000u ? hi : 0u);
            }
          }
        }
        const int e = max(static_cast<int>(m >> 23) - 126, -100);
        f = q8::two_to(14 - e);
        qmul *= q8::two_to(e - 14);
      } else {
        load_q(0);
      }
#pragma unroll
      for (int c0 = 0; c0 < D / 8; c0 += QC) {
        if (c0 > 0) load_q(c0);
        if (SCALE_Q) {
#pragma unroll
          for (int c = 0; c < QC; ++c) {
            uint32_t* u = reinterpret_cast<uint32_t*>(&w[c]);
#pragma unroll
            for (int i = 0; i < 4; ++i)
              u[i] = half2_bits(__uint_as_float(u[i] << 16) * f, __uint_as_float(u[i] & 0xffff0000u) * f);
          }
        }
#pragma unroll
        for (int c = 0; c < QC; ++c)
          sts128(sbase + x * L::TILE + ((c0 + c) >> 3) * SUB + r * 128 + (((c & 7) ^ (r & 7)) << 4), w[c].x ^ flip,
                 w[c].y ^ flip, w[c].z ^ flip, w[c].w ^ flip);
      }
    }
    fence_proxy_async_smem();
    tc::mbar_arrive(q_full);
    const int lim = valid ? len - n_tok + qr / p.G + 1 : 0;   // keys that this row sees
    const int lim_all = len - n_tok + row0 / p.G + 1;         // keys that every row of the tile sees
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t ts = tmem + lane_off, tp = tmem + lane_off + 128 + x * 64, to = tmem + lane_off + 256 + x * 128;
    const auto factor = [&](float k) {  // a NaN softmax scale stays NaN
      const float x = k * qmul;
      return x < MIN_FACTOR ? MIN_FACTOR : x;
    };
    float m_used = -INFINITY, l = 0.f;
    float sc[TB];
    bool ok = true;
    for (int j = 0; j < nx; ++j) {
      if (!(ok = warp_wait(s_full + x, j & 1, p.status, abort))) break;
      tc::fence_after();
#pragma unroll
      for (int c = 0; c < TB; c += 32) tc::tmem_ld32(ts + c, sc + c);
      tc::tmem_wait_ld();
      tc::fence_before();
      tc::mbar_arrive(s_free);
      if (j * TB + TB > lim_all) {
        const int end = lim - j * TB;
#pragma unroll
        for (int c = 0; c < TB; ++c) sc[c] = c < end ? sc[c] : -INFINITY;
      }
      // u = s * f + lv with f > 0: a page's largest u is its largest s's, and a masked
      // score stays -inf.  The product may underflow (queries of zeros, a softmax
      // scale of 0 or near it, pages of tiny values), so it is the smallest normal
      // number at least: scores, 2^33 at most, times 2^-126 move no weight.
      const float4* page = reinterpret_cast<const float4*>(scales + (j % NSC) * 24);
      float f[8], lv[8];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float4 a = page[i], b = page[2 + i];
        f[4 * i] = factor(a.x); f[4 * i + 1] = factor(a.y); f[4 * i + 2] = factor(a.z); f[4 * i + 3] = factor(a.w);
        lv[4 * i] = b.x; lv[4 * i + 1] = b.y; lv[4 * i + 2] = b.z; lv[4 * i + 3] = b.w;
      }
      float mx = -INFINITY;
#pragma unroll
      for (int g = 0; g < 8; ++g) {
        const float* v = sc + 16 * g;
        float m0 = max3(v[0], v[1], v[2]), m1 = max3(v[3], v[4], v[5]);
        m0 = max3(m0, v[6], v[7]);
        m1 = max3(m1, v[8], v[9]);
        m0 = max3(m0, v[10], v[11]);
        m1 = max3(m1, v[12], v[13]);
        mx = fmaxf(mx, fmaf(max3(max3(m0, v[14], v[15]), m1, m1), f[g], lv[g]));
      }
      const float m_new = mx > m_used + SLACK ? mx : m_used;
      const float alpha = m_new == m_used ? 1.f : tc::ex2(m_used - m_new);
      const float off = m_new == -INFINITY ? 0.f : LIFT - m_new;
#pragma unroll
      for (int g = 0; g < 8; ++g) lv[g] += off;
      if (j >= 1) {  // P V(j - 1) has read P and written O
        if (!(ok = warp_wait(pv_done + x, (j - 1) & 1, p.status, abort))) break;
        tc::fence_after();
        if (__any_sync(FULL_MASK, m_new != m_used)) {
#pragma unroll 1
          for (int c = 0; c < D; c += 16) {
            float o[16];
            tc::tmem_ld16(to + c, o);
            tc::tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] *= alpha;
            tc::tmem_st16(to + c, o);
          }
        }
      }
      float sum = 0.f;
      const float* iv = reinterpret_cast<const float*>(page + 4);
#pragma unroll
      for (int g = 0; g < 8; ++g) {
        float pk[8];
        const poly::f2 f2 = poly::splat(f[g]), c2 = poly::splat(lv[g]);
        poly::f2 r2[2] = {poly::splat(0.f), poly::splat(0.f)};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float e0, e1;
          poly::unpack(poly::fma2(poly::pack(sc[16 * g + 2 * i], sc[16 * g + 2 * i + 1]), f2, c2), e0, e1);
          e0 = tc::ex2(e0);
          e1 = tc::ex2(e1);
          r2[i & 1] = poly::add2(r2[i & 1], poly::pack(e0, e1));
          pk[i] = __uint_as_float(half2_bits(e0, e1));
        }
        tc::tmem_st8(tp + 8 * g, pk);
        if (g == 3 || g == 7) {
          tc::tmem_wait_st();
          tc::fence_before();
          tc::mbar_arrive(p_full + 2 * x + (g >> 2));
        }
        float r4[4];
        poly::unpack(poly::add2(r2[0], r2[1]), r4[0], r4[1]);
        sum = fmaf(r4[0] + r4[1], iv[g], sum);
      }
      l = fmaf(l, alpha, sum);
      m_used = m_new;
    }
    if (nx > 0 && ok) ok = warp_wait(pv_done + x, (nx - 1) & 1, p.status, abort);
    if (nx > 0 && ok) {
      tc::fence_after();
      const int64_t orow = tok * p.Hq + head;
      const float inv = l > 0.f ? 1.f / l : l == l ? 0.f : l;  // no key: zeros; NaN stays NaN
      if (valid && p.lse) p.lse[orow] = l > 0.f ? (m_used - LIFT + log2f(l)) * LN2 : l == l ? -INFINITY : l;
      QT* dst = static_cast<QT*>(p.out) + orow * D;
#pragma unroll 1
      for (int c = 0; c < D; c += 32) {
        float o[32];
        tc::tmem_ld32(to + c, o);
        tc::tmem_wait_ld();
        if (valid) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
              w[k] = static_cast<uint32_t>(Mma<QT>::bits(o[8 * i + 2 * k] * inv)) |
                     (static_cast<uint32_t>(Mma<QT>::bits(o[8 * i + 2 * k + 1] * inv)) << 16);
            *reinterpret_cast<uint4*>(dst + c + 8 * i) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
      }
    }
  }
  tc::fence_before();
  __syncthreads();
  if (warp == 0) {
    tc::fence_after();
    tc::tmem_dealloc(tmem, 512);
  }
}

template <typename QT, int D, int CODE>
int launch(const Params& p, const ic_paged_attn_args& a, cudaStream_t st) {
  auto kern = tile_kernel<QT, D, CODE>;
  static PerDeviceLimit limit;
  int rc;
  if ((rc = ensure_dynamic_smem(kern, Lay<D>::BYTES, &limit)) != IC_OK) return rc;
  // at most this many (session, pair) units, whatever the sessions' counts
  const int64_t units = static_cast<int64_t>(a.num_q_tokens) * p.G / (TILES<D> * TB) + std::min<int64_t>(p.S, a.num_q_tokens);
  Params params = p;
  void* args[] = {&params};
  return launch_pdl(reinterpret_cast<const void*>(kern), dim3(static_cast<unsigned>(units * p.H)), dim3(THREADS),
                    Lay<D>::BYTES, st, args, "paged_attention (tile)");
}

template <typename QT>
int launch_q(const Params& p, const ic_paged_attn_args& a, cudaStream_t st) {
  if (a.head_dim == 64)
    return a.code_dtype == IC_E4M3 ? launch<QT, 64, IC_E4M3>(p, a, st) : launch<QT, 64, IC_I8>(p, a, st);
  if (a.head_dim == 128)
    return a.code_dtype == IC_E4M3 ? launch<QT, 128, IC_E4M3>(p, a, st) : launch<QT, 128, IC_I8>(p, a, st);
  return a.code_dtype == IC_E4M3 ? launch<QT, 256, IC_E4M3>(p, a, st) : launch<QT, 256, IC_I8>(p, a, st);
}

}  // namespace

int launch_tile(const Params& p, const ic_paged_attn_args& a, cudaStream_t st) {
  return a.q_dtype == IC_F16 ? launch_q<__half>(p, a, st) : launch_q<__nv_bfloat16>(p, a, st);
}

}  // namespace paged
}  // namespace ic
