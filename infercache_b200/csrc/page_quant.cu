// Rows into and out of 8-bit pages.
//
// Write: one warp per (page run, layer and head, K or V) -- a run is the
// tokens of one call in consecutive slots of one page.  The run's rows pass through
// a few vectors per lane: their largest magnitude gives the page scale's exponent,
// then the codes are stored; a run that does not start its page and needs a larger
// scale first rounds the page's other codes again.  Read: one thread per
// 8 codes of RT tokens.  Both are bound by HBM (a write moves size + 1 bytes per
// element, a read 1 + size) as long as an element costs few instructions, which
// is why maxima and fp16 codes are taken two at a time.  Measured (B200): 16
// prompts of 2048 fp16 tokens, 36 layers, 2 heads, 128 dims, written as int8 and
// read back: 600 to 636 us for 3.62 GB, 87 to 92 % of a plain copy's rate (the read
// alone 339); one token of 64 sessions, 4 heads, written and read back: 8 to 9 us, the
// calls' host time.
#include <stdio.h>

#include <type_traits>

#include "common.cuh"
#include "launch.cuh"
#include "q8.cuh"

namespace ic {
namespace {

constexpr int WARPS = 4;  // warps per CTA (write)

struct Range {
  const int32_t* slots;
  const int32_t* page_ids;
  char* k_buf;
  char* v_buf;
  int64_t start, n, stride_l, stride_h, stride_t;
  int64_t n_pages;
};

struct Batch {
  uint8_t* k;
  uint8_t* v;
  float* k_scale;
  float* v_scale;
  int32_t* status;
  int64_t pool_tokens;
  int32_t heads, layer_begin, count;
  int32_t window;                        // slots form of a write: tokens whose pages one warp looks after
  int64_t first[IC_PAGE_BATCH_MAX + 1];  // work items (warps or threads) before each range
  Range r[IC_PAGE_BATCH_MAX];
};

__device__ __forceinline__ int64_t slot_of(const Range& r, int64_t t) {
  if (r.slots) return r.slots[t];
  const int64_t lt = r.start + t;
  if (lt >= r.n_pages * q8::PAGE) return -1;
  const int32_t page = r.page_ids[lt / q8::PAGE];
  return page < 0 ? -1 : static_cast<int64_t>(page) * q8::PAGE + lt % q8::PAGE;
}

// A lane's vector of a source row: 16 bytes.
template <typename T> constexpr int VE = 16 / sizeof(T);

__device__ __forceinline__ void vec_floats(const uint4& u, float* o, const float*) {
  o[0] = __uint_as_float(u.x); o[1] = __uint_as_float(u.y); o[2] = __uint_as_float(u.z); o[3] = __uint_as_float(u.w);
}
template <typename T>
__device__ __forceinline__ void vec_floats(const uint4& u, float* o, const T*) {
  const uint2 lo = make_uint2(u.x, u.y), hi = make_uint2(u.z, u.w);
  load4(reinterpret_cast<const T*>(&lo), o);
  load4(reinterpret_cast<const T*>(&hi), o + 4);
}

// The largest magnitude among vectors, kept as the type's own bits (two 16-bit
// maxima per register): as unsigned integers they order like the magnitudes,
// with infinities and NaN above every finite value.
template <typename T>
__device__ __forceinline__ uint32_t max_bits(uint32_t m, const uint4& u) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    m = sizeof(T) == 4 ? max(m, w[i] & 0x7fffffffu) : __vmaxu2(m, w[i] & 0x7fff7fffu);
  return m;
}
// The warp's maximum as the bits of a float (>= 0x7f800000: not finite).
__device__ __forceinline__ uint32_t warp_max_bits(uint32_t m, const float*) { return __reduce_max_sync(FULL_MASK, m); }
__device__ __forceinline__ uint32_t warp_max_bits(uint32_t m, const __nv_bfloat16*) {
  return __reduce_max_sync(FULL_MASK, max(m & 0xffffu, m >> 16)) << 16;
}
__device__ __forceinline__ uint32_t warp_max_bits(uint32_t m, const __half*) {
  const uint32_t h = __reduce_max_sync(FULL_MASK, max(m & 0xffffu, m >> 16));
  return __float_as_uint(__half2float(__ushort_as_half(static_cast<uint16_t>(h))));
}

// Codes of one vector whose values are finite and at most QMAX * 2^e, four per
// word.  int8: adding 1.5 * 2^23 rounds to nearest even and leaves the integer
// in the low byte; e4m3: the conversion instruction.
template <int CODE, typename T>
__device__ __forceinline__ void encode_vec(const uint4& u, int e, uint32_t* o, const T* type) {
  const float unit = q8::two_to(-e);
  float x[VE<T>];
  vec_floats(u, x, type);
#pragma unroll
  for (int i = 0; i < VE<T> / 4; ++i) {
    if (CODE == IC_E4M3) {
      uint16_t lo, hi;
      asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(x[4 * i + 1] * unit), "f"(x[4 * i] * unit));
      asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(x[4 * i + 3] * unit), "f"(x[4 * i + 2] * unit));
      o[i] = static_cast<uint32_t>(lo) | (static_cast<uint32_t>(hi) << 16);
    } else {
      uint32_t r[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) r[k] = __float_as_uint(fmaf(x[4 * i + k], unit, 12582912.f));
      o[i] = __byte_perm(__byte_perm(r[0], r[1], 0x0040), __byte_perm(r[2], r[3], 0x0040), 0x5410);
    }
  }
}
// fp16 sources whose unit is an fp16 number stay in fp16, two values an
// instruction: the product with a power of two and the addition of 1.5 * 2^10
// round once (a product that turns subnormal lies far under half a code step).
template <int CODE>
__device__ __forceinline__ void encode_half(const uint4& u, __half2 unit, uint32_t* o) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const __half2 a = *reinterpret_cast<const __half2*>(&w[2 * i]), b = *reinterpret_cast<const __half2*>(&w[2 * i + 1]);
    if (CODE == IC_E4M3) {
      __half2 x = __hmul2(a, unit), y = __hmul2(b, unit);
      uint16_t lo, hi;
      asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(lo) : "r"(*reinterpret_cast<uint32_t*>(&x)));
      asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(hi) : "r"(*reinterpret_cast<uint32_t*>(&y)));
      o[i] = static_cast<uint32_t>(lo) | (static_cast<uint32_t>(hi) << 16);
    } else {
      const __half2 off = __float2half2_rn(1536.f);
      __half2 x = __hfma2(a, unit, off), y = __hfma2(b, unit, off);
      o[i] = __byte_perm(*reinterpret_cast<uint32_t*>(&x), *reinterpret_cast<uint32_t*>(&y), 0x6420);
    }
  }
}

template <int N>
__device__ __forceinline__ void store_codes(uint32_t* dst, const uint32_t* o) {
  if (N == 2)
    *reinterpret_cast<uint2*>(dst) = make_uint2(o[0], o[1]);
  else
    *dst = o[0];
}

// A page's source rows pass through CHUNK vectors per lane twice, for the
// maximum and for the codes; the second reading hits the cache and a run that
// fits needs none.  4 leave more loads of short runs in flight: one token of 149
// sessions in 28 layers 65 us (8: 78), 4 to 10 of 108 in 36 44 (51); 8 take a
// 16-bit page of 128 dims whole: 16 prompts of 2k tokens in 36 layers, written and
// read back, 596 us (4: 616), 4 of 1024 x 4 heads 150 (161).  Both with 64
// registers a thread (80: 652 us for the prompts).
constexpr int64_t BIG_WRITE = 1 << 18;  // tokens x layers x heads from which it is 8

// `cnt` tokens, source rows src + t * stride (elements), into slots off ..
// off + cnt - 1 of the page at `page` (16 rows of D codes).
template <typename T, int D, int CODE, int CHUNK>
__device__ __forceinline__ void write_run(const T* src, int64_t stride, int cnt, int off, uint8_t* page, float* scale_p,
                                          int32_t* status, int lane) {
  constexpr int E = VE<T>, W = E / 4;         // elements and code words per vector
  constexpr int VR = D / E;                   // vectors per row
  constexpr int NV = q8::PAGE * VR / 32;      // vectors per lane for a whole page
  constexpr int CH = NV < CHUNK ? NV : CHUNK; // of which so many are held at a time
  const T* type = nullptr;
  const int chunks = (cnt * VR + 32 * CH - 1) / (32 * CH);
  uint4 raw[CH];
  const auto load_chunk = [&](int c) {
#pragma unroll
    for (int j = 0; j < CH; ++j) {
      const int it = lane + 32 * (c * CH + j), t = it / VR;
      raw[j] = make_uint4(0, 0, 0, 0);
      if (t < cnt) raw[j] = reinterpret_cast<const uint4*>(src + t * stride)[it % VR];
    }
  };
  const float held = off > 0 ? *scale_p : 0.f;
  uint32_t m = 0;
#pragma unroll 1
  for (int c = chunks - 1; c >= 0; --c) {     // ends with chunk 0 in registers
    load_chunk(c);
#pragma unroll
    for (int j = 0; j < CH; ++j) m = max_bits<T>(m, raw[j]);
  }
  uint32_t amax = warp_max_bits(m, type);
  bool plain = amax < 0x7f800000u;            // every value finite
  if (!plain) {
    amax = 0;
#pragma unroll 1
    for (int it = lane; it < cnt * VR; it += 32) {
      float x[E];
      vec_floats(reinterpret_cast<const uint4*>(src + it / VR * stride)[it % VR], x, type);
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const uint32_t b = __float_as_uint(x[i]) & 0x7fffffffu;
        amax = max(amax, b < 0x7f800000u ? b : 0u);
      }
    }
    amax = __reduce_max_sync(FULL_MASK, amax);
    if (lane == 0 && status) atomicOr(status, IC_DEVFLAG_NONFINITE);
  }
  int e = q8::exponent_for<CODE>(amax);
  if (e == q8::E_MAX) plain = false;          // the values may pass the largest code
  if (off > 0) {
    const int e_old = static_cast<int>((__float_as_uint(held) >> 23) & 255u) - 127;
    if (e > e_old) {  // round the page's other codes again to the larger unit
      const float f = q8::two_to(max(e_old - e, -126));
      for (int it = lane; it < q8::PAGE * D / 4; it += 32) {
        const int t = it / (D / 4);
        if (t >= off && t < off + cnt) continue;
        uint32_t* p = reinterpret_cast<uint32_t*>(page) + it;
        float x[4];
        q8::decode4<CODE>(*p, x);
        *p = q8::encode4<CODE>(x[0] * f, x[1] * f, x[2] * f, x[3] * f);
      }
    } else {
      e = q8::clamp_exp(e_old);
    }
  }
  uint32_t* dst = reinterpret_cast<uint32_t*>(page + off * D);
  if (plain) {
    const bool in_half = std::is_same<T, __half>::value && e >= -15 && e <= 24;
    const __half2 unit = __float2half2_rn(q8::two_to(-e));
#pragma unroll 1
    for (int c = 0;;) {
      if (in_half) {
#pragma unroll
        for (int j = 0; j < CH; ++j) {
          const int it = lane + 32 * (c * CH + j);
          uint32_t o[2];
          encode_half<CODE>(raw[j], unit, o);
          if (it / VR < cnt) store_codes<W>(dst + it * W, o);
        }
      } else {
#pragma unroll
        for (int j = 0; j < CH; ++j) {
          const int it = lane + 32 * (c * CH + j);
          uint32_t o[W];
          encode_vec<CODE>(raw[j], e, o, type);
          if (it / VR < cnt) store_codes<W>(dst + it * W, o);
        }
      }
      if (++c >= chunks) break;
      load_chunk(c);                          // again, from the cache
    }
  } else {
    const float unit = q8::two_to(-e);
#pragma unroll 1
    for (int it = lane; it < cnt * VR; it += 32) {
      const uint4 u = reinterpret_cast<const uint4*>(src + it / VR * stride)[it % VR];
      float x[E];
      vec_floats(u, x, type);
#pragma unroll
      for (int i = 0; i < W; ++i)
        dst[it * W + i] = q8::encode4<CODE>(x[4 * i] * unit, x[4 * i + 1] * unit, x[4 * i + 2] * unit, x[4 * i + 3] * unit);
    }
  }
  __syncwarp();  // every lane has read the old scale
  if (lane == 0) *scale_p = q8::two_to(e);
}

template <typename T, int D, int CODE, int CHUNK>
__global__ void __launch_bounds__(WARPS * 32, 8) write_kernel(const __grid_constant__ Batch b) {
  grid_dependency_wait();
  grid_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * WARPS + (threadIdx.x >> 5);
  if (item >= b.first[b.count]) return;
  int i = 0;
  while (b.first[i + 1] <= item) ++i;
  const Range& r = b.r[i];
  const int64_t w = item - b.first[i];
  const int lh = blockIdx.y, l = lh / b.heads, h = lh % b.heads;
  const bool is_v = blockIdx.z != 0;
  const int64_t plane = static_cast<int64_t>(b.layer_begin + l) * b.heads + h;
  uint8_t* codes = (is_v ? b.v : b.k) + plane * b.pool_tokens * D;
  float* scales = (is_v ? b.v_scale : b.k_scale) + plane * (b.pool_tokens / q8::PAGE);
  const T* buf = reinterpret_cast<const T*>(is_v ? r.v_buf : r.k_buf) + l * r.stride_l + h * r.stride_h;

  if (!r.slots) {  // work item w is the w-th page that the range touches
    const int64_t page0 = (r.start / q8::PAGE + w) * q8::PAGE;
    const int64_t t0 = max(page0 - r.start, int64_t{0}), t1 = min(page0 + q8::PAGE - r.start, r.n);
    const int64_t slot = slot_of(r, t0);
    if (slot < 0 || slot >= b.pool_tokens) return;
    write_run<T, D, CODE, CHUNK>(buf + t0 * r.stride_t, r.stride_t, static_cast<int>(t1 - t0),
                          static_cast<int>(slot % q8::PAGE), codes + slot / q8::PAGE * (q8::PAGE * D),
                          scales + slot / q8::PAGE, b.status, lane);
    return;
  }
  // the pages whose first token is among tokens w0 .. w0 + window - 1 (window <=
  // 16): lane j holds token w0 - 1 + j's slot.  A page's tokens are one warp's, run
  // after run where they leave slots out: two runs raise one scale.
  const int64_t w0 = w * b.window, tj = w0 - 1 + lane;
  const int32_t slot = tj >= 0 && tj < r.n ? r.slots[tj] : -1;
  const int32_t prev = __shfl_up_sync(FULL_MASK, slot, 1);
  const bool valid = slot >= 0 && slot < b.pool_tokens;
  const bool same = lane > 0 && valid && prev >= 0 && slot / q8::PAGE == prev / q8::PAGE;
  const uint32_t page_goes_on = __ballot_sync(FULL_MASK, same);
  const uint32_t cont = __ballot_sync(FULL_MASK, same && slot == prev + 1);  // the next slot: the same run
  uint32_t heads = __ballot_sync(FULL_MASK, valid && !same && lane >= 1 && lane <= b.window);
  while (heads) {
    int j = __ffs(heads) - 1;
    heads &= heads - 1;
    do {
      const int32_t s0 = __shfl_sync(FULL_MASK, slot, j);
      const uint32_t rest = ~(cont >> j >> 1);  // bit k: token j + 1 + k does not go on
      const int cnt = min(__ffs(rest), q8::PAGE - s0 % q8::PAGE);
      write_run<T, D, CODE, CHUNK>(buf + (w0 - 1 + j) * r.stride_t, r.stride_t, cnt, s0 % q8::PAGE,
                            codes + static_cast<int64_t>(s0 / q8::PAGE) * (q8::PAGE * D), scales + s0 / q8::PAGE, b.status,
                            lane);
      __syncwarp();
      j += cnt;
    } while (j < 32 && (page_goes_on >> j & 1));
  }
}

// 8 codes times their scale 2^e, rounded once to T.
__device__ __forceinline__ uint32_t pack_pair(float a, float b, const __half*) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack_pair(float a, float b, const __nv_bfloat16*) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <int CODE, typename T>
__device__ __forceinline__ void store8(T* p, const uint2& u, float s) {
  uint32_t h[4];
  q8::decode4_h2<CODE>(u.x, h[0], h[1]);
  q8::decode4_h2<CODE>(u.y, h[2], h[3]);
  if (std::is_same<T, __half>::value && s >= 6.103515625e-05f && s <= 32768.f) {  // the scale is a normal fp16 number
    const __half2 s2 = __float2half2_rn(s);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 v = __hmul2(*reinterpret_cast<__half2*>(&h[i]), s2);
      h[i] = *reinterpret_cast<const uint32_t*>(&v);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 v = __half22float2(*reinterpret_cast<__half2*>(&h[i]));
      h[i] = pack_pair(v.x * s, v.y * s, p);
    }
  }
  *reinterpret_cast<uint4*>(p) = make_uint4(h[0], h[1], h[2], h[3]);
}
template <int CODE>
__device__ __forceinline__ void store8(float* p, const uint2& u, float s) {
  float x[8];
  q8::decode4<CODE>(u.x, x);
  q8::decode4<CODE>(u.y, x + 4);
  *reinterpret_cast<float4*>(p) = make_float4(x[0] * s, x[1] * s, x[2] * s, x[3] * s);
  *reinterpret_cast<float4*>(p + 4) = make_float4(x[4] * s, x[5] * s, x[6] * s, x[7] * s);
}

constexpr int RT = 4;  // tokens per thread (read): their loads are in flight together

template <int D> constexpr int READ_TOKENS = RT * 256 / (D / 8);  // tokens per CTA

template <typename T, int D, int CODE>
__global__ void __launch_bounds__(256) read_kernel(const __grid_constant__ Batch b) {
  constexpr int V8 = D / 8, STEP = 256 / V8;
  grid_dependency_wait();
  grid_launch_dependents();
  int i = 0;
  while (b.first[i + 1] <= blockIdx.x) ++i;
  const Range& r = b.r[i];
  const int64_t t0 = (blockIdx.x - b.first[i]) * READ_TOKENS<D> + threadIdx.x / V8;
  const int c = threadIdx.x % V8;
  const int lh = blockIdx.y, l = lh / b.heads, h = lh % b.heads;
  const bool is_v = blockIdx.z != 0;
  const int64_t plane = static_cast<int64_t>(b.layer_begin + l) * b.heads + h;
  const uint8_t* codes = (is_v ? b.v : b.k) + plane * b.pool_tokens * D;
  const float* scales = (is_v ? b.v_scale : b.k_scale) + plane * (b.pool_tokens / q8::PAGE);
  T* out = reinterpret_cast<T*>(is_v ? r.v_buf : r.k_buf) + l * r.stride_l + h * r.stride_h + 8 * c;
  uint2 u[RT];
  float s[RT];
  int64_t slot[RT];
#pragma unroll
  for (int j = 0; j < RT; ++j) slot[j] = t0 + j * STEP < r.n ? slot_of(r, t0 + j * STEP) : -1;
#pragma unroll
  for (int j = 0; j < RT; ++j) {
    u[j] = make_uint2(0, 0);
    s[j] = 0.f;
    if (slot[j] >= 0 && slot[j] < b.pool_tokens) {
      u[j] = reinterpret_cast<const uint2*>(codes + slot[j] * D)[c];
      s[j] = scales[slot[j] / q8::PAGE];
    }
  }
#pragma unroll
  for (int j = 0; j < RT; ++j)
    if (t0 + j * STEP < r.n) store8<CODE>(out + (t0 + j * STEP) * r.stride_t, u[j], s[j]);
}

bool q8_args_ok(const ic_page_q8_args* a, const char* name) {
  char msg[160];
  const auto fail = [&](const char* why) {
    snprintf(msg, sizeof(msg), "%s: %s", name, why);
    set_last_error(msg);
    return false;
  };
  if (!a || !a->rows || !a->pool.k || !a->pool.v || !a->k_scale || !a->v_scale) return fail("null argument");
  if (a->pool.dtype != IC_E4M3 && a->pool.dtype != IC_I8) return fail("the pool must hold 8-bit codes");
  if (a->count < 1 || a->count > IC_PAGE_BATCH_MAX) return fail("1 <= count <= IC_PAGE_BATCH_MAX ranges");
  if (a->pool.num_layers < 1 || a->pool.num_kv_heads < 1 || a->pool.pool_tokens < q8::PAGE ||
      a->pool.pool_tokens % q8::PAGE || a->pool.pool_tokens > 0x7fffffff || a->layer_begin < 0 ||
      a->layer_end > a->pool.num_layers || a->layer_begin > a->layer_end)
    return fail("bad pool or layer range");
  if (static_cast<int64_t>(a->layer_end - a->layer_begin) * a->pool.num_kv_heads > 65535)
    return fail("more than 65535 layers times heads");
  if (a->buf_dtype != IC_F32 && a->buf_dtype != IC_F16 && a->buf_dtype != IC_BF16) return fail("bad buffer dtype");
  if ((reinterpret_cast<uintptr_t>(a->pool.k) & 15) || (reinterpret_cast<uintptr_t>(a->pool.v) & 15))
    return fail("the pool must be 16-byte aligned");
  const int esz = a->buf_dtype == IC_F32 ? 4 : 2;
  for (int i = 0; i < a->count; ++i) {
    const ic_page_q8_rows& r = a->rows[i];
    if (r.n_tokens < 0 || r.n_tokens > 0x7fffffff) return fail("bad token count");
    if (r.n_tokens == 0) continue;
    if (!r.k_buf || !r.v_buf || (!r.slots && !r.page_ids)) return fail("null buffer, slots or pages");
    if (!r.slots && (r.start_token < 0 || r.start_token + r.n_tokens > static_cast<int64_t>(r.n_page_ids) * q8::PAGE))
      return fail("tokens past the page list");
    if ((r.stride_l * esz) % 16 || (r.stride_h * esz) % 16 || (r.stride_t * esz) % 16 ||
        (reinterpret_cast<uintptr_t>(r.k_buf) & 15) || (reinterpret_cast<uintptr_t>(r.v_buf) & 15))
      return fail("buffer rows must be 16-byte aligned");
  }
  return true;
}

int q8_dim_error(const char* name) {
  char msg[96];
  snprintf(msg, sizeof(msg), "%s: head_dim must be 64, 128 or 256", name);
  set_last_error(msg);
  return IC_ERR_UNSUPPORTED;
}

void fill_batch(const ic_page_q8_args* a, Batch& b) {
  b.k = static_cast<uint8_t*>(a->pool.k);
  b.v = static_cast<uint8_t*>(a->pool.v);
  b.k_scale = a->k_scale;
  b.v_scale = a->v_scale;
  b.status = a->dev_status;
  b.pool_tokens = a->pool.pool_tokens;
  b.heads = a->pool.num_kv_heads;
  b.layer_begin = a->layer_begin;
  b.count = a->count;
  for (int i = 0; i < a->count; ++i) {
    const ic_page_q8_rows& r = a->rows[i];
    b.r[i] = Range{r.slots, r.page_ids, static_cast<char*>(r.k_buf), static_cast<char*>(r.v_buf), r.start_token,
                   r.n_tokens, r.stride_l, r.stride_h, r.stride_t, r.n_page_ids};
  }
}

template <typename T, int D, int CHUNK>
const void* write_fn(int code) {
  return code == IC_E4M3 ? reinterpret_cast<const void*>(write_kernel<T, D, IC_E4M3, CHUNK>)
                         : reinterpret_cast<const void*>(write_kernel<T, D, IC_I8, CHUNK>);
}
template <typename T, int CHUNK>
const void* write_fn_c(int d, int code) {
  return d == 64 ? write_fn<T, 64, CHUNK>(code) : d == 128 ? write_fn<T, 128, CHUNK>(code) : write_fn<T, 256, CHUNK>(code);
}
template <typename T>
const void* write_fn_d(int d, int code, bool big) {
  return big ? write_fn_c<T, 8>(d, code) : write_fn_c<T, 4>(d, code);
}
template <typename T, int D>
const void* read_fn(int code) {
  return code == IC_E4M3 ? reinterpret_cast<const void*>(read_kernel<T, D, IC_E4M3>)
                         : reinterpret_cast<const void*>(read_kernel<T, D, IC_I8>);
}
template <typename T>
const void* read_fn_d(int d, int code) {
  return d == 64 ? read_fn<T, 64>(code) : d == 128 ? read_fn<T, 128>(code) : read_fn<T, 256>(code);
}

}  // namespace
}  // namespace ic

extern "C" int ic_page_write_q8(const ic_page_q8_args* a, void* stream) {
  using namespace ic;
  if (!q8_args_ok(a, "page_write_q8")) return IC_ERR_INVALID_ARG;
  const int D = a->pool.head_dim;
  if (D != 64 && D != 128 && D != 256) return q8_dim_error("page_write_q8");
  const int planes = (a->layer_end - a->layer_begin) * a->pool.num_kv_heads;
  if (planes == 0) return IC_OK;
  Batch b = {};
  fill_batch(a, b);
  // Slots form: a warp looks after the pages whose first token is among `window` tokens.
  // One while that leaves few warps (a decode tick: every run is one token and
  // all run side by side); with many, 4 and then 16, so that a prompt's warps
  // have a page each instead of most of them finding nothing to do.
  int64_t tokens = 0;
  for (int i = 0; i < a->count; ++i) tokens += a->rows[i].n_tokens;
  b.window = tokens * planes <= 8192 ? 1 : tokens * planes <= 65536 ? 4 : 16;
  for (int i = 0; i < a->count; ++i) {
    const ic_page_q8_rows& r = a->rows[i];
    const int64_t items = r.n_tokens == 0 ? 0
                          : r.slots      ? (r.n_tokens + b.window - 1) / b.window
                                         : (r.start_token + r.n_tokens - 1) / q8::PAGE - r.start_token / q8::PAGE + 1;
    b.first[i + 1] = b.first[i] + items;
  }
  const int64_t blocks = (b.first[b.count] + WARPS - 1) / WARPS;
  if (blocks == 0) return IC_OK;
  if (blocks > 0x7fffffff) {
    set_last_error("page_write_q8: too many tokens for one launch");
    return IC_ERR_UNSUPPORTED;
  }
  const bool big = tokens * planes > BIG_WRITE;
  const void* fn = a->buf_dtype == IC_F32   ? write_fn_d<float>(D, a->pool.dtype, big)
                   : a->buf_dtype == IC_F16 ? write_fn_d<__half>(D, a->pool.dtype, big)
                                            : write_fn_d<__nv_bfloat16>(D, a->pool.dtype, big);
  void* p[] = {&b};
  return launch_pdl(fn, dim3(static_cast<unsigned>(blocks), planes, 2), dim3(WARPS * 32), 0,
                    static_cast<cudaStream_t>(stream), p, "page_write_q8");
}

extern "C" int ic_page_read_q8(const ic_page_q8_args* a, void* stream) {
  using namespace ic;
  if (!q8_args_ok(a, "page_read_q8")) return IC_ERR_INVALID_ARG;
  const int D = a->pool.head_dim;
  if (D != 64 && D != 128 && D != 256) return q8_dim_error("page_read_q8");
  const int planes = (a->layer_end - a->layer_begin) * a->pool.num_kv_heads;
  if (planes == 0) return IC_OK;
  Batch b = {};
  fill_batch(a, b);
  const int per_cta = RT * 256 / (D / 8);
  for (int i = 0; i < a->count; ++i) b.first[i + 1] = b.first[i] + (a->rows[i].n_tokens + per_cta - 1) / per_cta;
  const int64_t blocks = b.first[b.count];
  if (blocks == 0) return IC_OK;
  if (blocks > 0x7fffffff) {
    set_last_error("page_read_q8: too many tokens for one launch");
    return IC_ERR_UNSUPPORTED;
  }
  const void* fn = a->buf_dtype == IC_F32   ? read_fn_d<float>(D, a->pool.dtype)
                   : a->buf_dtype == IC_F16 ? read_fn_d<__half>(D, a->pool.dtype)
                                            : read_fn_d<__nv_bfloat16>(D, a->pool.dtype);
  void* p[] = {&b};
  return launch_pdl(fn, dim3(static_cast<unsigned>(blocks), planes, 2), dim3(256), 0, static_cast<cudaStream_t>(stream),
                    p, "page_read_q8");
}
