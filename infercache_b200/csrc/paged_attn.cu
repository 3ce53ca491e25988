// Attention over 8-bit pages: argument checks and the choice between the
// streaming kernel (paged_stream.cu: few query rows per session, HBM-bound) and
// the tile kernel (paged_tile.cu: many, tensor-core-bound).
#include <cuda.h>

#include "common.cuh"
#include "paged_attn.cuh"
#include "q8.cuh"

namespace ic {
namespace paged {

namespace {

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn find_encode() {
  void* f = nullptr;
  cudaDriverEntryPointQueryResult q;
  if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess ||
      q != cudaDriverEntryPointSuccess) {
    cudaGetLastError();
    return nullptr;
  }
  return reinterpret_cast<EncodeTiledFn>(f);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// IC_OK, or the refusal (with its reason as the last error).
int check(const ic_paged_attn_args* a) {
  if (!a || !a->q || !a->out || !a->k || !a->v || !a->k_scale || !a->v_scale || !a->block_table || !a->lens ||
      !a->q_start) {
    set_last_error("paged_attention: null argument");
    return IC_ERR_INVALID_ARG;
  }
  if (a->num_sessions < 1 || a->table_width < 0 || a->table_width > (1 << 26) || a->num_q_tokens < 1 || a->max_count < 0 || a->num_kv_heads < 1 ||
      a->num_q_heads < 1 || a->num_q_heads % a->num_kv_heads || a->pool_tokens < q8::PAGE ||
      a->pool_tokens % q8::PAGE || a->pool_tokens > 0x7fffffff || a->q_stride_t < 0 || a->q_stride_h < 0) {
    set_last_error("paged_attention: bad shape");
    return IC_ERR_INVALID_ARG;
  }
  if ((a->q_dtype != IC_F16 && a->q_dtype != IC_BF16) || (a->code_dtype != IC_E4M3 && a->code_dtype != IC_I8)) {
    set_last_error("paged_attention: q must be fp16 or bf16 and the cache e4m3 or int8");
    return IC_ERR_INVALID_ARG;
  }
  if (a->head_dim != 64 && a->head_dim != 128 && a->head_dim != 256) {
    set_last_error("paged_attention: head_dim must be 64, 128 or 256");
    return IC_ERR_UNSUPPORTED;
  }
  if (!aligned16(a->q) || !aligned16(a->out) || !aligned16(a->k) || !aligned16(a->v) || a->q_stride_t % 8 ||
      a->q_stride_h % 8) {
    set_last_error("paged_attention: q, out and the cache must have 16-byte aligned rows");
    return IC_ERR_INVALID_ARG;
  }
  if (a->num_sessions > MAX_SESSIONS) {
    set_last_error("paged_attention: at most 4096 sessions");
    return IC_ERR_UNSUPPORTED;
  }
  // The tile kernel's grid and a session's rows fit 31 bits.
  const int64_t G = a->num_q_heads / a->num_kv_heads, rows = a->num_q_tokens * G;
  if (rows > (1 << 30) || (rows / 128 + a->num_sessions) * a->num_kv_heads > 0x7fffffff) {
    set_last_error("paged_attention: more than 2^30 query rows per KV head, or 2^31 tiles of them in all");
    return IC_ERR_UNSUPPORTED;
  }
  // The streaming kernel numbers its groups' pages, and its overhead for each
  // group, with 32 bits.  Its groups: tiles of 8 rows or more, and no more than
  // few_rows of a session where the tile kernel has the others.
  const int few = few_rows(*a);
  int64_t tiles = rows / 8 + a->num_sessions;
  if (few != ALL_ROWS) tiles = std::min(tiles, static_cast<int64_t>(a->num_sessions) * ((few + 7) / 8));
  if (tiles * a->num_kv_heads > 0x7fffffffLL / (a->table_width + 32)) {
    set_last_error("paged_attention: the streaming kernel's query tiles x KV heads x table width exceed 2^31");
    return IC_ERR_UNSUPPORTED;
  }
  return IC_OK;
}

}  // namespace

// Sessions with at most this many query rows per KV head are the streaming
// kernel's.  It reads a session's pages once per 8 or 16 rows, the tile kernel
// converts them once per 256 (128 at 256 dims) but gives each (session, KV head,
// that many rows) to one CTA.  Two conditions follow: the call's rows have to
// amount to enough CTAs (below some 16 the streaming kernel's even shares win
// although it does the work several times over), and the session's to three or
// more of its row tiles.  Measured, streaming / tiles, in us:
//   rows in all, one session of 8192 tokens, 2 heads of 8:
//     128 dims: 4096 119 / 133, 6144 172 / 134; 256 dims: 2048 104 / 138, 4096 196 / 139
//   rows per session, 64 sessions of 4000 tokens, 2 to 4 heads:
//     128 dims: 36 102 / 96, 48 103 / 95, 64 132 / 94 (40 sessions of 3000 tokens,
//     35 rows, a second wave of tiles: 100 / 127); 256 dims: 16 117 / 164, 24 213 /
//     165, 36 164 / 90, 64 214 / 91
// Short tiles also want more of them, lest a long session's CTA runs alone: 24
// sessions of 1400 tokens, 4 heads, 48 rows (4608 in all) 26 / 30 at 128 dims, 20 /
// 26 at 64; 24 of 256 to 4096, 2 heads, 48 rows (2304) 47 / 76 at 256 dims.
int few_rows(const ic_paged_attn_args& a) {
  const int64_t G = a.num_q_heads / a.num_kv_heads, rows = a.num_q_tokens * static_cast<int64_t>(a.num_q_heads);
  const int few = a.head_dim == 256 ? (rows > 4096 ? 16 : 128) : rows > 6144 ? 40 : 64;
  return a.max_count * G <= few || rows <= (a.head_dim == 256 ? 2048 : 4096) ? ALL_ROWS : few;
}

int page_map(CUtensorMap* m, const void* codes, int64_t pool_tokens, int heads, int D) {
  static const EncodeTiledFn fn = find_encode();
  if (!fn) {
    set_last_error("paged_attention: cuTensorMapEncodeTiled unavailable");
    return IC_ERR_CUDA;
  }
  const cuuint64_t line = D == 64 ? 128 : D, lines = D == 64 ? pool_tokens / 2 : pool_tokens;
  const cuuint64_t dims[3] = {line, lines, static_cast<cuuint64_t>(heads)};
  const cuuint64_t strides[2] = {line, line * lines};
  const cuuint32_t box[3] = {128, D == 64 ? 8u : 16u, 1};
  const cuuint32_t estr[3] = {1, 1, 1};
  if (fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(codes), dims, strides, box, estr,
         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS) {
    set_last_error("paged_attention: tensor map encoding failed");
    return IC_ERR_INVALID_ARG;
  }
  return IC_OK;
}

}  // namespace paged
}  // namespace ic

extern "C" int64_t ic_paged_attention_workspace(const ic_paged_attn_args* a) {
  return ic::paged::check(a) == IC_OK ? ic::paged::stream_workspace(*a) : 0;
}

extern "C" int ic_paged_attention(const ic_paged_attn_args* a, void* stream) {
  using namespace ic;
  int rc = paged::check(a);
  if (rc != IC_OK) return rc;
  const int64_t need = paged::stream_workspace(*a);
  if (need > 0 && (!a->workspace || !paged::aligned16(a->workspace) || a->workspace_bytes < need)) {
    set_last_error("paged_attention: workspace missing, misaligned or too small");
    return IC_ERR_INVALID_ARG;
  }
  paged::Params p;
  p.q = a->q;
  p.k = a->k;
  p.v = a->v;
  p.out = a->out;
  p.lse = a->lse;
  p.table = a->block_table;
  p.lens = a->lens;
  p.q_start = a->q_start;
  p.k_scale = a->k_scale;
  p.v_scale = a->v_scale;
  p.ws = static_cast<float*>(a->workspace);
  p.status = a->dev_status;
  p.q_stride_t = a->q_stride_t;
  p.q_stride_h = a->q_stride_h;
  p.S = a->num_sessions;
  p.width = a->table_width;
  p.Hq = a->num_q_heads;
  p.H = a->num_kv_heads;
  p.G = a->num_q_heads / a->num_kv_heads;
  p.n_pages = static_cast<int32_t>(a->pool_tokens / q8::PAGE);
  p.n_q = a->num_q_tokens;
  p.few_rows = paged::few_rows(*a);
  p.sl2 = a->scale * paged::LOG2E;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (p.few_rows != paged::ALL_ROWS && (rc = paged::launch_tile(p, *a, st)) != IC_OK) return rc;
  return paged::launch_stream(p, *a, st);
}
