// Penalties for repeated tokens, biases and grammar masks on logits, in one
// pass: each CTA takes a chunk of one row's vocabulary.  It counts in shared
// memory which of its ids the row's tokens and biases name (integer atomics, so
// the result does not depend on their order) while it streams the chunk --
// convert, mask, store -- and then writes the few ids that are named a second
// time, finished.  The stream never waits for the counts, and the row's tokens
// arrive while it runs.  Bound by HBM: every
// logit is read once and written once; the row's tokens (a few KB) are read by
// each of its chunks from L2.  Measured (B200): 64 bf16 rows of 152k ids with all
// parts 19 to 22 us, 2.8 TB/s (the second visit of the named ids waits for the
// counts); one row with a repetition penalty 4.8 us, the call's host time.
#include <math.h>

#include "common.cuh"
#include "launch.cuh"

namespace ic {
namespace {

constexpr int LT = 256;
constexpr int AHEAD = 8;  // of the row's tokens, how many per thread are loaded before anything is waited for

constexpr int LIST = 2048;  // named ids that a chunk keeps a list of

// A word per id of the chunk: the answer's occurrences, the last bias entry + 1,
// and whether the id stands in the prompt.  Rows with more tokens or biases
// than the fields hold (WIDE) keep the bias entries in words of their own.
constexpr uint32_t SEEN = 0x80000000u;
constexpr int COUNT_BITS = 16, MAX_COUNT = (1 << COUNT_BITS) - 1, MAX_BIAS = 0x7fff - 1;

template <typename T> struct Vec4;
template <> struct Vec4<float> { using type = uint4; };
template <> struct Vec4<__half> { using type = uint2; };
template <> struct Vec4<__nv_bfloat16> { using type = uint2; };

__device__ __forceinline__ void vec_floats(const uint4& u, float* o, float*) {
  o[0] = __uint_as_float(u.x); o[1] = __uint_as_float(u.y); o[2] = __uint_as_float(u.z); o[3] = __uint_as_float(u.w);
}
__device__ __forceinline__ void vec_floats(const uint2& u, float* o, __half*) { load4(reinterpret_cast<const __half*>(&u), o); }
__device__ __forceinline__ void vec_floats(const uint2& u, float* o, __nv_bfloat16*) {
  load4(reinterpret_cast<const __nv_bfloat16*>(&u), o);
}

// NV vectors of 4 ids per thread: the chunk is LT * 4 * NV ids.  VEC: rows are
// aligned for vector accesses; otherwise (an odd vocabulary) element by element.
template <typename T, int NV, bool VEC, bool WIDE>
__global__ void __launch_bounds__(LT) logits_kernel(const ic_logits_args a) {
  constexpr int CHUNK = LT * 4 * NV, U = NV < 4 ? NV : 4;
  constexpr uint32_t COUNT = WIDE ? ~SEEN : MAX_COUNT;
  extern __shared__ uint4 words4[];               // [CHUNK] words; WIDE: then the biases' entries [CHUNK]
  uint32_t* words = reinterpret_cast<uint32_t*>(words4);
  uint32_t* entry = WIDE ? words + CHUNK : words;
  const int tid = threadIdx.x, row = blockIdx.y;
  const int base = blockIdx.x * CHUNK, n = min(CHUNK, a.vocab - base);
  const bool with_tokens = a.tokens != nullptr, with_bias = a.bias_ids != nullptr;
  const T* in = static_cast<const T*>(a.logits) + row * a.logits_stride + base;
  float* out = a.out + row * a.out_stride + base;
  const uint32_t* mask = a.mask ? reinterpret_cast<const uint32_t*>(a.mask) + row * a.mask_stride : nullptr;
  const int32_t* tok = a.tokens + row * a.tokens_stride;
  const int32_t* ids = a.bias_ids + row * a.bias_stride;
  __shared__ uint16_t list[LIST];                 // ids of the chunk that are named
  __shared__ int n_list;
  int32_t ahead[AHEAD];
  int len = 0, prompt = 0, n_bias = 0;
  if (with_tokens || with_bias)
    for (int i = tid; i < CHUNK / 4 * (WIDE ? 2 : 1); i += LT) words4[i] = make_uint4(0, 0, 0, 0);
  if (tid == 0) n_list = 0;
  grid_dependency_wait();
  grid_launch_dependents();

  if (with_tokens) {  // on their way while the chunk streams
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) ahead[j] = tid + LT * j < a.max_tokens ? tok[tid + LT * j] - base : -1;
    len = a.token_lens ? min(a.token_lens[row], a.max_tokens) : a.max_tokens;
    prompt = a.prompt_lens ? a.prompt_lens[row] : 0;
  }
  if (with_bias) n_bias = a.bias_lens ? min(a.bias_lens[row], a.bias_width) : a.bias_width;

  // ---- stream ------------------------------------------------------------------
  const auto masked = [&](int e) { return mask && !((mask[(base + e) >> 5] >> ((base + e) & 31)) & 1u); };
#pragma unroll 1
  for (int j0 = 0; j0 < NV; j0 += U) {
    if (VEC) {
      using V = typename Vec4<T>::type;
      V vec[U];
      uint32_t allowed[U];
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const int e = 4 * (tid + LT * (j0 + j));
        vec[j] = V{};
        allowed[j] = 0xffffffffu;
        if (e < n) {
          vec[j] = *reinterpret_cast<const V*>(in + e);
          if (mask) allowed[j] = mask[(base + e) >> 5] >> ((base + e) & 31);
        }
      }
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const int e = 4 * (tid + LT * (j0 + j));
        if (e < n) {
          float x[4];
          vec_floats(vec[j], x, static_cast<T*>(nullptr));
#pragma unroll
          for (int i = 0; i < 4; ++i) x[i] = (allowed[j] >> i) & 1u ? x[i] : -INFINITY;
          *reinterpret_cast<float4*>(out + e) = make_float4(x[0], x[1], x[2], x[3]);
        }
      }
    } else {
      T one[4 * U];
#pragma unroll
      for (int j = 0; j < 4 * U; ++j) {
        const int e = tid + LT * (4 * j0 + j);
        one[j] = T{};
        if (e < n) one[j] = in[e];
      }
#pragma unroll
      for (int j = 0; j < 4 * U; ++j) {
        const int e = tid + LT * (4 * j0 + j);
        if (e < n) out[e] = masked(e) ? -INFINITY : DT<T>::to_f(one[j]);
      }
    }
  }
  if (!with_tokens && !with_bias) return;

  // ---- count; whoever names an id first puts it on the list -------------------------
  __syncthreads();
  const auto push = [&](int rel) {
    const int at = atomicAdd(&n_list, 1);
    if (at < LIST) list[at] = static_cast<uint16_t>(rel);
  };
  for (int t = tid; t < n_bias; t += LT) {
    const int rel = ids[t] - base;
    if (rel >= 0 && rel < n && atomicMax(entry + rel, static_cast<uint32_t>(t + 1) << (WIDE ? 0 : COUNT_BITS)) == 0) push(rel);
  }
  if (with_bias) __syncthreads();  // the counts go into the same words, or look at the entries
  if (with_tokens) {
    const auto count = [&](int t, int rel) -> bool {
      if (t >= len || rel < 0 || rel >= n) return false;
      const uint32_t old = t < prompt ? atomicOr(words + rel, SEEN) : atomicAdd(words + rel, 1u);
      return old == 0 && !(WIDE && with_bias && entry[rel] != 0);
    };
    uint32_t first = 0;
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) first |= static_cast<uint32_t>(count(tid + LT * j, ahead[j])) << j;
    // one place on the list's end per warp, not per id: the ends' counter would
    // serialise the CTA
    int upto = __popc(first);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(FULL_MASK, upto, o);
      if ((tid & 31) >= o) upto += u;
    }
    int at = 0;
    if ((tid & 31) == 31 && upto > 0) at = atomicAdd(&n_list, upto);
    at = __shfl_sync(FULL_MASK, at, 31) + upto - __popc(first);
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      if ((first >> j) & 1u) {
        if (at < LIST) list[at] = static_cast<uint16_t>(ahead[j]);
        ++at;
      }
    }
    for (int t = tid + LT * AHEAD; t < len; t += LT) {
      const int rel = tok[t] - base;
      if (count(t, rel)) push(rel);
    }
  }
  __syncthreads();

  // ---- the ids that are named ---------------------------------------------------
  const float rep = a.repetition ? a.repetition[row] : a.repetition_all;
  const float freq = a.frequency ? a.frequency[row] : a.frequency_all;
  const float pres = a.presence ? a.presence[row] : a.presence_all;
  const float* bias = a.bias_values + row * a.bias_stride;
  // With out = logits, in[rel] holds what the stream stored: the logit, or -inf
  // for a masked id.
  const auto finish = [&](int rel, uint32_t w, uint32_t b) {
    if (masked(rel)) return;
    float x = DT<T>::to_f(in[rel]);
    const uint32_t c = w & COUNT;
    if (c != 0 || (w & SEEN)) {
      // a row's own penalty divides, rounding once; a number's reciprocal comes from
      // the caller, as torch divides by a number
      x = !(x > 0.f) ? x * rep : a.repetition ? __fdiv_rn(x, rep) : x * a.repetition_all_inv;
      if (c != 0) x = __fsub_rn(x, __fadd_rn(__fmul_rn(freq, static_cast<float>(c)), pres));
    }
    if (b != 0) x += bias[b - 1];
    out[rel] = x;
  };
  const auto entry_of = [&](int rel, uint32_t w) -> uint32_t {
    return WIDE ? (with_bias ? entry[rel] : 0u) : (w & ~SEEN) >> COUNT_BITS;
  };
  const int listed = n_list;
  if (listed <= LIST) {
    for (int i = tid; i < listed; i += LT) {
      const int rel = list[i];
      finish(rel, words[rel], entry_of(rel, words[rel]));
    }
  } else {  // more ids than the list holds: look at every word
    for (int rel = tid; rel < n; rel += LT) {
      const uint32_t w = words[rel], b = entry_of(rel, w);
      if ((w | b) != 0) finish(rel, w, b);
    }
  }
}

template <typename T, int NV, bool WIDE>
int launch_logits(const ic_logits_args& a, cudaStream_t st, bool vec) {
  constexpr int CHUNK = LT * 4 * NV, SMEM = CHUNK * 4 * (WIDE ? 2 : 1);  // at most 48 KB
  static_assert(SMEM + LIST * 2 + 64 <= 48 * 1024, "the default shared-memory limit");
  ic_logits_args args = a;
  void* p[] = {&args};
  const void* fn = vec ? reinterpret_cast<const void*>(logits_kernel<T, NV, true, WIDE>)
                       : reinterpret_cast<const void*>(logits_kernel<T, NV, false, WIDE>);
  return launch_pdl(fn, dim3((a.vocab + CHUNK - 1) / CHUNK, a.rows), dim3(LT), SMEM, st, p, "process_logits");
}

template <typename T>
int logits_dispatch(const ic_logits_args& a, cudaStream_t st) {
  // Vector accesses need every row's start aligned and whole vectors at its end.
  const bool vec = a.vocab % 4 == 0 && a.logits_stride % 4 == 0 && a.out_stride % 4 == 0 &&
                   (reinterpret_cast<uintptr_t>(a.logits) & (4 * sizeof(T) - 1)) == 0 &&
                   (reinterpret_cast<uintptr_t>(a.out) & 15) == 0;
  if (a.max_tokens > MAX_COUNT || a.bias_width > MAX_BIAS) return launch_logits<T, 4, true>(a, st, vec);
  // Chunk: the largest that still gives 4 CTAs per SM; every chunk of a row
  // reads the row's tokens again.
  const int64_t total = static_cast<int64_t>(a.vocab) * a.rows, want = 4 * 148;
  if (total >= want * LT * 32) return launch_logits<T, 8, false>(a, st, vec);
  if (total >= want * LT * 16) return launch_logits<T, 4, false>(a, st, vec);
  if (total >= want * LT * 8) return launch_logits<T, 2, false>(a, st, vec);
  return launch_logits<T, 1, false>(a, st, vec);
}

}  // namespace
}  // namespace ic

extern "C" int ic_process_logits(const ic_logits_args* a, void* stream) {
  if (!a || !a->logits || !a->out || a->rows < 0 || a->vocab < 1 || a->max_tokens < 0 || a->bias_width < 0 ||
      (a->bias_ids && !a->bias_values) || a->logits_stride < a->vocab || a->out_stride < a->vocab) {
    ic::set_last_error("process_logits: bad arguments");
    return IC_ERR_INVALID_ARG;
  }
  if ((a->tokens && a->tokens_stride < a->max_tokens) || (a->bias_ids && a->bias_stride < a->bias_width) ||
      (a->mask && a->mask_stride < (static_cast<int64_t>(a->vocab) + 31) / 32)) {
    ic::set_last_error("process_logits: a row stride is shorter than its row");
    return IC_ERR_INVALID_ARG;
  }
  if (a->rows > 65535) {
    ic::set_last_error("process_logits: at most 65535 rows");
    return IC_ERR_UNSUPPORTED;
  }
  if (a->rows == 0) return IC_OK;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (a->dtype) {
    case IC_F32: return ic::logits_dispatch<float>(*a, st);
    case IC_F16: return ic::logits_dispatch<__half>(*a, st);
    case IC_BF16: return ic::logits_dispatch<__nv_bfloat16>(*a, st);
    default:
      ic::set_last_error("process_logits: logits must be fp32, fp16 or bf16");
      return IC_ERR_INVALID_ARG;
  }
}
