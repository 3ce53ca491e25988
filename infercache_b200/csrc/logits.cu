// Penalties for repeated tokens, biases and grammar masks on logits, in one
// pass: each CTA takes a chunk of one row's vocabulary, loads its logits into
// registers, counts in shared memory which of its ids the row's tokens name
// (integer atomics, so the result does not depend on their order), and writes
// the finished 32-bit logits.  Bound by HBM: every logit is read once and
// written once; the row's tokens (a few KB) are read by each of its chunks
// from L2.
#include <math.h>

#include "common.cuh"
#include "launch.cuh"

namespace ic {
namespace {

constexpr int LT = 256;
constexpr uint32_t SEEN = 0x80000000u;  // the id stands in the prompt; the low bits count the answer's occurrences

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
template <typename T, int NV, bool VEC>
__global__ void __launch_bounds__(LT) logits_kernel(const ic_logits_args a) {
  constexpr int CHUNK = LT * 4 * NV;
  extern __shared__ uint32_t words[];             // [CHUNK], then the biases' entries [CHUNK]
  uint32_t* entry = words + CHUNK;
  const int tid = threadIdx.x, row = blockIdx.y;
  const int base = blockIdx.x * CHUNK, n = min(CHUNK, a.vocab - base);
  const bool with_tokens = a.tokens != nullptr, with_bias = a.bias_ids != nullptr;
  grid_dependency_wait();
  grid_launch_dependents();

  const T* in = static_cast<const T*>(a.logits) + row * a.logits_stride + base;
  float* out = a.out + row * a.out_stride + base;
  using V = typename Vec4<T>::type;
  V vec[VEC ? NV : 1];
  T one[VEC ? 1 : NV * 4];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    if (VEC) {
      const int e = 4 * (tid + LT * j);
      vec[j] = V{};
      if (e < n) vec[j] = *reinterpret_cast<const V*>(in + e);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int e = tid + LT * (4 * j + i);
        one[4 * j + i] = T{};
        if (e < n) one[4 * j + i] = in[e];
      }
    }
  }

  if (with_tokens || with_bias) {
    const int n_words = CHUNK * (with_bias ? 2 : 1);
    for (int i = tid; i < n_words / 4; i += LT) reinterpret_cast<uint4*>(words)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    if (with_tokens) {
      const int32_t* tok = a.tokens + row * a.tokens_stride;
      const int len = a.token_lens ? min(a.token_lens[row], a.max_tokens) : a.max_tokens;
      const int prompt = a.prompt_lens ? a.prompt_lens[row] : 0;
#pragma unroll 4
      for (int t = tid; t < len; t += LT) {
        const int rel = tok[t] - base;
        if (rel >= 0 && rel < n) {
          if (t < prompt) atomicOr(words + rel, SEEN); else atomicAdd(words + rel, 1u);
        }
      }
    }
    if (with_bias) {
      const int32_t* ids = a.bias_ids + row * a.bias_stride;
      const int len = a.bias_lens ? min(a.bias_lens[row], a.bias_width) : a.bias_width;
      for (int t = tid; t < len; t += LT) {
        const int rel = ids[t] - base;
        if (rel >= 0 && rel < n) atomicMax(entry + rel, static_cast<uint32_t>(t + 1));
      }
    }
    __syncthreads();
  }

  const float rep = a.repetition ? a.repetition[row] : a.repetition_all;
  const float inv_rep = a.repetition ? 1.f / rep : a.repetition_all_inv;
  const float freq = a.frequency ? a.frequency[row] : a.frequency_all;
  const float pres = a.presence ? a.presence[row] : a.presence_all;
  const float* bias = with_bias ? a.bias_values + row * a.bias_stride : nullptr;
  const uint32_t* mask = a.mask ? reinterpret_cast<const uint32_t*>(a.mask) + row * a.mask_stride : nullptr;
  const auto finish = [&](float x, int e) {
    if (with_tokens) {
      const uint32_t w = words[e];
      if (w != 0) {
        x = x > 0.f ? x * inv_rep : x * rep;
        const uint32_t c = w & ~SEEN;
        if (c != 0) x = __fsub_rn(x, __fadd_rn(__fmul_rn(freq, static_cast<float>(c)), pres));
      }
    }
    if (with_bias) {
      const uint32_t b = entry[e];
      if (b != 0) x += bias[b - 1];
    }
    if (mask && !((mask[(base + e) >> 5] >> ((base + e) & 31)) & 1u)) x = -INFINITY;
    return x;
  };
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    if (VEC) {
      const int e = 4 * (tid + LT * j);
      if (e < n) {
        float x[4];
        vec_floats(vec[j], x, static_cast<T*>(nullptr));
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = finish(x[i], e + i);
        *reinterpret_cast<float4*>(out + e) = make_float4(x[0], x[1], x[2], x[3]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int e = tid + LT * (4 * j + i);
        if (e < n) out[e] = finish(DT<T>::to_f(one[4 * j + i]), e);
      }
    }
  }
}

template <typename T, int NV>
int launch_logits(const ic_logits_args& a, cudaStream_t st, bool vec) {
  constexpr int CHUNK = LT * 4 * NV;
  const int smem = CHUNK * 4 * (a.bias_ids ? 2 : 1);
  ic_logits_args args = a;
  void* p[] = {&args};
  static PerDeviceLimit lim_vec, lim_one;
  int rc;
  const dim3 grid((a.vocab + CHUNK - 1) / CHUNK, a.rows);
  if (vec) {
    if ((rc = ensure_dynamic_smem(logits_kernel<T, NV, true>, smem, &lim_vec)) != IC_OK) return rc;
    return launch_pdl(reinterpret_cast<const void*>(logits_kernel<T, NV, true>), grid, dim3(LT), smem, st, p,
                      "process_logits");
  }
  if ((rc = ensure_dynamic_smem(logits_kernel<T, NV, false>, smem, &lim_one)) != IC_OK) return rc;
  return launch_pdl(reinterpret_cast<const void*>(logits_kernel<T, NV, false>), grid, dim3(LT), smem, st, p,
                    "process_logits");
}

template <typename T>
int logits_dispatch(const ic_logits_args& a, cudaStream_t st) {
  // Vector accesses need every row's start aligned and whole vectors at its end.
  const bool vec = a.vocab % 4 == 0 && (a.logits_stride * sizeof(T)) % (4 * sizeof(T)) == 0 && a.out_stride % 4 == 0 &&
                   (reinterpret_cast<uintptr_t>(a.logits) & (4 * sizeof(T) - 1)) == 0 &&
                   (reinterpret_cast<uintptr_t>(a.out) & 15) == 0;
  // Chunk: the largest that still gives 4 CTAs per SM; every chunk of a row
  // reads the row's tokens again.
  const int64_t total = static_cast<int64_t>(a.vocab) * a.rows, want = 4 * 148;
  if (total >= want * LT * 32) return launch_logits<T, 8>(a, st, vec);
  if (total >= want * LT * 16) return launch_logits<T, 4>(a, st, vec);
  if (total >= want * LT * 8) return launch_logits<T, 2>(a, st, vec);
  return launch_logits<T, 1>(a, st, vec);
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
