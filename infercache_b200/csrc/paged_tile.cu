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
//   warpgroup 1  loads the pages' codes (16 bytes a lane, one key tile ahead in
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
// registers at once, so the next Q K^T overlaps its exponentials.
// TMEM columns: S 0, P_a 128, P_b 192, O_a 256, O_b 384.  Registers: 512
// threads start with 128 each; warpgroups 0 and 1 give theirs to the softmax
// (56 + 96 + 176 + 176 = 504 of 512).
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
constexpr int RS = 5;                  // K / V ring slots
constexpr int NSC = 8;                 // key tiles whose scales are kept: the ring runs at most 3 ahead of the softmax
constexpr float SLACK = 8.f, LIFT = 7.f;

template <int D>
struct Lay {
  static constexpr int TILE = D / 64 * SUB;
  static constexpr int RING = 2 * TILE;
  static constexpr int SCALES = RING + RS * TILE;      // [NSC][3][8]: k scale, log2 v scale, 1 / v scale
  static constexpr int BARS = SCALES + NSC * 24 * 4;
  static constexpr int NBAR = 20;
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

template <typename QT, int D, int CODE>
__global__ void __launch_bounds__(THREADS, 1) tile_kernel(const Params p) {
  using L = Lay<D>;
  constexpr int NS = D / 64;  // 64-column sub-tiles of an operand row
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
  uint64_t* p_full = bars + 14;   // [2]
  uint64_t* pv_done = bars + 16;  // [2]
  uint64_t* mma_done = bars + 18;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::MISC);
  volatile int* abort = reinterpret_cast<volatile int*>(smem + L::MISC + 4);
  volatile int* found = reinterpret_cast<volatile int*>(smem + L::MISC + 8);  // session, pair
  int* sums = reinterpret_cast<int*>(smem + L::MISC + 16);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (tid == 0) {
    *abort = 0;
    found[0] = -1;
  }
  grid_dependency_wait();
  grid_launch_dependents();

  // ---- which session and pair of tiles -------------------------------------------
  const int h = blockIdx.x % p.H, unit = blockIdx.x / p.H;
  {
    int carry = 0;
    for (int s0 = 0; s0 < p.S; s0 += THREADS) {
      const int s = s0 + tid;
      int own = 0;
      if (s < p.S) {
        int begin;
        const int rows = query_tokens(p, s, begin) * p.G;
        own = rows > p.few_rows ? (rows + 2 * TB - 1) / (2 * TB) : 0;
      }
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
  const int s = found[0], pair = found[1];
  if (s < 0) return;
  int q_begin;
  const int n_tok = query_tokens(p, s, q_begin), rows = n_tok * p.G, len = held_tokens(p, s);
  const int row_a = pair * 2 * TB;
  const bool has_b = row_a + TB < rows;
  // keys that row r sees: len - n_tok + r / G + 1; a tile's last row sets its range
  const auto tiles_of = [&](int row0) {
    const int last = min(row0 + TB, rows) - 1;
    return max(1, (len - n_tok + last / p.G + 1 + TB - 1) / TB);
  };
  const int na = tiles_of(row_a), nb = has_b ? tiles_of(row_a + TB) : 0;
  const int n = has_b ? nb : na;
  const auto u_k = [&](int j) { return j == 0 ? 0 : 2 * j - 1; };
  const auto u_v = [&](int j) { return j == n - 1 ? 2 * n - 1 : 2 * j + 2; };

  if (tid == 0) {
    mbar_init(q_full, has_b ? 256 : 128);
    for (int i = 0; i < RS; ++i) {
      mbar_init(r_full + i, 128);
      mbar_init(r_empty + i, 1);
    }
    for (int x = 0; x < 2; ++x) {
      mbar_init(s_full + x, 1);
      mbar_init(p_full + x, 128);
      mbar_init(pv_done + x, 1);
    }
    mbar_init(s_free, 128);
    mbar_init(mma_done, 2);
    fence_barrier_init();
  }
  if (warp == 0) tc::tmem_alloc(tmem_slot, 512);
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = *tmem_slot;

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
        const int u = u_v(j);
        if (!(ok = one_wait(r_full + u % RS, (u / RS) & 1, p.status, abort))) break;
        const uint32_t sv = sbase + L::RING + (u % RS) * L::TILE;
        for (int x = 0; x < 2; ++x) {
          if (j >= (x ? nb : na)) continue;
          if (!(ok = one_wait(p_full + x, j & 1, p.status, abort))) break;
          tc::fence_after();
#pragma unroll
          for (int kk = 0; kk < TB / 16; ++kk)
            tc::mma_ts(tmem + 256 + x * 128, tmem + 128 + x * 64 + kk * 8, mndesc(sv, kk), IDESC_PV,
                       (j > 0 || kk > 0) ? 1u : 0u);
          tc::commit(pv_done + x);
        }
        if (ok) tc::commit(r_empty + u % RS);
      }
      tc::commit(mma_done);
      mbar_wait_bounded(mma_done, 0, p.status);
    }
  } else if (warp < 8) {
    // ---- codes to operand tiles -----------------------------------------------------
    asm volatile("setmaxnreg.dec.sync.aligned.u32 96;");
    const int cw = warp - 4, t8 = lane >> 2, c4 = lane & 3;
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
    // this warp's 32 tokens of a key tile are pages 2 cw and 2 cw + 1 of its eight
    const auto pages_at = [&](int u, int* id) {
      int j;
      what(u, j);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int pg = j * 8 + cw * 2 + i;
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
    const auto load = [&](int u, const int* id, uint4 (*reg)[NS], float& ks, float& vs) {
      int j;
      const uint8_t* codes = what(u, j) ? vc : kc;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int page = id[g >> 1], tok = (g & 1) * 8 + t8;
        const bool ok = page >= 0 && (j * 8 + cw * 2 + (g >> 1)) * q8::PAGE + tok < len;
#pragma unroll
        for (int sub = 0; sub < NS; ++sub) {
          reg[g][sub] = make_uint4(0, 0, 0, 0);
          if (ok)
            reg[g][sub] = *reinterpret_cast<const uint4*>(codes + (static_cast<int64_t>(page) * q8::PAGE + tok) * D +
                                                          sub * 64 + c4 * 16);
        }
      }
      ks = 0.f;
      vs = 0.f;
      if (lane < 2 && id[lane & 1] >= 0) {
        ks = p.k_scale[plane + id[lane & 1]];
        vs = p.v_scale[plane + id[lane & 1]];
      }
    };
    uint4 cur[4][NS], nxt[4][NS];
    int id1[2], id2[2];
    float ks, vs, ksn, vsn;
    bool mine;   // whether this lane's page (lanes 0, 1) can be attended
    bool mine_n;
    pages_at(0, id1);
    load(0, id1, cur, ks, vs);
    mine = lane < 2 && id1[lane & 1] >= 0;
    pages_at(1, id1);
    for (int u = 0; u < total; ++u) {
      pages_at(u + 2, id2);
      if (u + 1 < total) load(u + 1, id1, nxt, ksn, vsn);
      mine_n = lane < 2 && id1[lane & 1] >= 0;
      const int st = u % RS;
      if (u >= RS && !warp_wait(r_empty + st, ((u / RS) - 1) & 1, p.status, abort)) break;
      int j;
      const bool is_v = what(u, j);
      const uint32_t dst = sbase + L::RING + st * L::TILE;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int tok = cw * 32 + g * 8 + t8;
#pragma unroll
        for (int sub = 0; sub < NS; ++sub) {
          const uint4 w = cur[g][sub];
          uint32_t x[8];
          q8::decode4_h2<CODE>(w.x, x[0], x[1]);
          q8::decode4_h2<CODE>(w.y, x[2], x[3]);
          q8::decode4_h2<CODE>(w.z, x[4], x[5]);
          q8::decode4_h2<CODE>(w.w, x[6], x[7]);
          const uint32_t row = dst + sub * SUB + tok * 128;
          sts128(row + (((2 * c4) ^ t8) << 4), x[0], x[1], x[2], x[3]);
          sts128(row + (((2 * c4 + 1) ^ t8) << 4), x[4], x[5], x[6], x[7]);
        }
      }
      if (!is_v && lane < 2) {
        float* sc = scales + (j % NSC) * 24 + cw * 2 + lane;
        const float v1 = fmaxf(vs, 7.8886090522101181e-31f);  // 2^-100: a zero scale stays harmless
        sc[0] = ks;
        sc[8] = mine ? log2f(v1) : -INFINITY;                 // no page: no weight
        sc[16] = mine ? 1.f / v1 : 0.f;
      }
      fence_proxy_async_smem();
      tc::mbar_arrive(r_full + st);
#pragma unroll
      for (int g = 0; g < 4; ++g)
#pragma unroll
        for (int sub = 0; sub < NS; ++sub) cur[g][sub] = nxt[g][sub];
      ks = ksn;
      vs = vsn;
      mine = mine_n;
      id1[0] = id2[0];
      id1[1] = id2[1];
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
    float qmul = p.sl2;
    if (nx > 0) {
      const QT* src = static_cast<const QT*>(p.q) + tok * p.q_stride_t + head * p.q_stride_h;
      float f = 1.f;
      if (std::is_same<QT, __nv_bfloat16>::value) {
        // bf16 to fp16: a power of two brings the row's largest finite value into [2^13, 2^14)
        uint32_t m = 0;
        if (valid) {
#pragma unroll 8
          for (int c = 0; c < D / 8; ++c) {
            const uint4 w = reinterpret_cast<const uint4*>(src)[c];
            const uint32_t u[4] = {w.x, w.y, w.z, w.w};
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
        qmul = q8::two_to(e - 14) * p.sl2;
      }
#pragma unroll 8
      for (int c = 0; c < D / 8; ++c) {
        uint4 w = make_uint4(0, 0, 0, 0);
        if (valid) w = reinterpret_cast<const uint4*>(src)[c];
        if (std::is_same<QT, __nv_bfloat16>::value) {
          uint32_t* u = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            u[i] = half2_bits(__uint_as_float(u[i] << 16) * f, __uint_as_float(u[i] & 0xffff0000u) * f);
        }
        sts128(sbase + x * L::TILE + (c >> 3) * SUB + r * 128 + (((c & 7) ^ (r & 7)) << 4), w.x, w.y, w.z, w.w);
      }
      fence_proxy_async_smem();
      tc::mbar_arrive(q_full);
    }
    const int lim = valid ? len - n_tok + qr / p.G + 1 : 0;   // keys that this row sees
    const int lim_all = len - n_tok + row0 / p.G + 1;         // keys that every row of the tile sees
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t ts = tmem + lane_off, tp = tmem + lane_off + 128 + x * 64, to = tmem + lane_off + 256 + x * 128;
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
      const float* page = scales + (j % NSC) * 24;
#pragma unroll
      for (int g = 0; g < 8; ++g) {
        const poly::f2 f = poly::splat(page[g] * qmul), lv = poly::splat(page[8 + g]);
#pragma unroll
        for (int c = 16 * g; c < 16 * g + 16; c += 2)
          poly::unpack(poly::fma2(poly::pack(sc[c], sc[c + 1]), f, lv), sc[c], sc[c + 1]);
      }
      if (j * TB + TB > lim_all) {
        const int end = lim - j * TB;
#pragma unroll
        for (int c = 0; c < TB; ++c) sc[c] = c < end ? sc[c] : -INFINITY;
      }
      float m8[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) m8[i] = sc[i];
#pragma unroll
      for (int c = 8; c < TB; ++c) m8[c & 7] = fmaxf(m8[c & 7], sc[c]);
      const float mx = fmaxf(fmaxf(fmaxf(m8[0], m8[1]), fmaxf(m8[2], m8[3])), fmaxf(fmaxf(m8[4], m8[5]), fmaxf(m8[6], m8[7])));
      const float m_new = mx > m_used + SLACK ? mx : m_used;
      const float alpha = m_new == m_used ? 1.f : tc::ex2(m_used - m_new);
      const poly::f2 neg = poly::splat(m_new == -INFINITY ? 0.f : LIFT - m_new);
      float sum = 0.f;
#pragma unroll
      for (int g = 0; g < 8; ++g) {
        float pk[8];
        poly::f2 r2[2] = {poly::splat(0.f), poly::splat(0.f)};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float e0, e1;
          poly::unpack(poly::add2(poly::pack(sc[16 * g + 2 * i], sc[16 * g + 2 * i + 1]), neg), e0, e1);
          e0 = tc::ex2(e0);
          e1 = tc::ex2(e1);
          r2[i & 1] = poly::add2(r2[i & 1], poly::pack(e0, e1));
          pk[i] = __uint_as_float(half2_bits(e0, e1));
        }
        float r4[4];
        poly::unpack(r2[0], r4[0], r4[1]);
        poly::unpack(r2[1], r4[2], r4[3]);
        sum = fmaf((r4[0] + r4[1]) + (r4[2] + r4[3]), page[16 + g], sum);
        if (g == 0 && j >= 1) {
          if (!(ok = warp_wait(pv_done + x, (j - 1) & 1, p.status, abort))) break;
          tc::fence_after();
        }
        tc::tmem_st8(tp + 8 * g, pk);
      }
      if (!ok) break;
      l = fmaf(l, alpha, sum);
      if (j >= 1 && __any_sync(FULL_MASK, m_new != m_used)) {
        const float f = m_new != m_used ? alpha : 1.f;
#pragma unroll 1
        for (int c = 0; c < D; c += 16) {
          float o[16];
          tc::tmem_ld16(to + c, o);
          tc::tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 16; ++i) o[i] *= f;
          tc::tmem_st16(to + c, o);
        }
      }
      tc::tmem_wait_st();
      tc::fence_before();
      tc::mbar_arrive(p_full + x);
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
  const int64_t units = static_cast<int64_t>(a.num_q_tokens) * p.G / (2 * TB) + std::min<int64_t>(p.S, a.num_q_tokens);
  Params params = p;
  void* args[] = {&params};
  return launch_pdl(reinterpret_cast<const void*>(kern), dim3(static_cast<unsigned>(units * p.H)), dim3(THREADS),
                    Lay<D>::BYTES, st, args, "paged_attention (tile)");
}

template <typename QT>
int launch_q(const Params& p, const ic_paged_attn_args& a, cudaStream_t st) {
  if (a.head_dim == 64)
    return a.code_dtype == IC_E4M3 ? launch<QT, 64, IC_E4M3>(p, a, st) : launch<QT, 64, IC_I8>(p, a, st);
  return a.code_dtype == IC_E4M3 ? launch<QT, 128, IC_E4M3>(p, a, st) : launch<QT, 128, IC_I8>(p, a, st);
}

}  // namespace

int launch_tile(const Params& p, const ic_paged_attn_args& a, cudaStream_t st) {
  return a.q_dtype == IC_F16 ? launch_q<__half>(p, a, st) : launch_q<__nv_bfloat16>(p, a, st);
}

}  // namespace paged
}  // namespace ic
