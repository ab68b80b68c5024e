// prompt.cu -- causal attention of packed prompts over their own K and V
// (sm_100a): o_i = sum_{j <= i} softmax_j(scale q_i k_j) v_j within each
// request, grouped heads.
//
// Simple form: one warp per (row, query head) with the online softmax's
// running maximum, sum and output in registers.
#include "internal.h"
#include "ptx.cuh"

namespace slmt {

namespace {

struct PromptParams {
  const void* q;
  const void* k;
  const void* v;
  void* out;
  const int32_t* qsl;
  const int32_t* seq_lens;
  int32_t* err;
  int64_t q_tok, q_head, k_tok, k_head, v_tok, v_head, o_tok, o_head;
  float scale;
  int num_tokens, num_reqs, max_query, hq, kv, bf16, out_dtype;
};

__device__ __forceinline__ float get16(const void* p, int64_t i, int bf16) {
  return bf16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i])
              : __half2float(reinterpret_cast<const __half*>(p)[i]);
}

template <int D>
__global__ void __launch_bounds__(128) prompt_simple_kernel(const PromptParams p) {
  constexpr int VEC = (D + 31) / 32;
  const int lane = threadIdx.x & 31;
  const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int i = (int)(item / p.hq), h = (int)(item % p.hq);
  const int r = blockIdx.y;
  const int a = p.qsl[r], b = p.qsl[r + 1];
  if (a < 0 || b < a || b > p.num_tokens || b - a > p.max_query) {
    if (item == 0 && lane == 0 && p.err) atomicOr(reinterpret_cast<unsigned int*>(p.err), SLMT_DEVERR_SEQ_LEN);
  }
  const int lo = max(a, 0), hi = min(b, p.num_tokens);
  if (i >= hi - lo || i >= p.max_query) return;
  if (p.seq_lens && p.seq_lens[r] != b - a) return;
  const int hk = h / (p.hq / p.kv);
  float q[VEC], o[VEC], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int d = 0; d < VEC; ++d) {
    const int c = lane + 32 * d;
    q[d] = c < D ? get16(p.q, (int64_t)(lo + i) * p.q_tok + (int64_t)h * p.q_head + c, p.bf16) : 0.f;
    o[d] = 0.f;
  }
  for (int j = 0; j <= i; ++j) {
    float s = 0.f;
#pragma unroll
    for (int d = 0; d < VEC; ++d) {
      const int c = lane + 32 * d;
      if (c < D) s += q[d] * get16(p.k, (int64_t)(lo + j) * p.k_tok + (int64_t)hk * p.k_head + c, p.bf16);
    }
#pragma unroll
    for (int w = 16; w > 0; w >>= 1) s += __shfl_xor_sync(0xffffffffu, s, w);
    s *= p.scale;
    const float mn = fmaxf(m, s);
    const float base = mn == -INFINITY ? 0.f : mn;
    const float f = expf(m - base), e = expf(s - base);
    l = l * f + e;
#pragma unroll
    for (int d = 0; d < VEC; ++d) {
      const int c = lane + 32 * d;
      if (c < D) o[d] = o[d] * f + e * get16(p.v, (int64_t)(lo + j) * p.v_tok + (int64_t)hk * p.v_head + c, p.bf16);
    }
    m = mn;
  }
#pragma unroll
  for (int d = 0; d < VEC; ++d) {
    const int c = lane + 32 * d;
    if (c >= D) continue;
    const int64_t at = (int64_t)(lo + i) * p.o_tok + (int64_t)h * p.o_head + c;
    const float x = o[d] / l;
    if (p.out_dtype == SLMT_DTYPE_F32) reinterpret_cast<float*>(p.out)[at] = x;
    else if (p.out_dtype == SLMT_DTYPE_F16) reinterpret_cast<__half*>(p.out)[at] = __float2half_rn(x);
    else reinterpret_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(x);
  }
}

}  // namespace
}  // namespace slmt

using namespace slmt;

extern "C" int slmt_prompt_attention(const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* k,
                                     int64_t k_token_stride, int64_t k_head_stride, const void* v,
                                     int64_t v_token_stride, int64_t v_head_stride, int dtype,
                                     const int32_t* query_start_loc, const int32_t* seq_lens, int64_t num_reqs,
                                     int64_t max_query_len, int64_t num_tokens, int64_t num_q_heads,
                                     int64_t num_kv_heads, int64_t head_dim, float sm_scale, void* out, int out_dtype,
                                     int64_t out_token_stride, int64_t out_head_stride, int32_t* err_flag,
                                     void* stream) {
  if (!valid_head_dim(head_dim)) return SLMT_ERR_HEAD_DIM;
  if (num_reqs < 0 || max_query_len < 0 || num_tokens < 0 || num_tokens > INT32_MAX / 2) return SLMT_ERR_SHAPE;
  if (num_kv_heads <= 0 || num_q_heads <= 0 || num_q_heads % num_kv_heads != 0) return SLMT_ERR_SHAPE;
  if (num_q_heads > 65535 || num_q_heads / num_kv_heads > 128) return SLMT_ERR_UNSUPPORTED;
  if (dtype != SLMT_DTYPE_F16 && dtype != SLMT_DTYPE_BF16) return SLMT_ERR_DTYPE;
  if (out_dtype != SLMT_DTYPE_F32 && out_dtype != SLMT_DTYPE_F16 && out_dtype != SLMT_DTYPE_BF16)
    return SLMT_ERR_DTYPE;
  if (!(sm_scale > 0.f) || !(sm_scale - sm_scale == 0.f)) return SLMT_ERR_SHAPE;
  if (num_reqs == 0 || max_query_len == 0 || num_tokens == 0) return SLMT_OK;
  if (!q || !k || !v || !out || !query_start_loc) return SLMT_ERR_NULL;
  if (rows_overlap(num_tokens, num_q_heads, out_token_stride, out_head_stride)) return SLMT_ERR_SHAPE;
  const uintptr_t any = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) |
                        reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(out);
  if (any % 16 != 0) return SLMT_ERR_ALIGN;
  if ((q_token_stride | q_head_stride | k_token_stride | k_head_stride | v_token_stride | v_head_stride) % 8 != 0)
    return SLMT_ERR_ALIGN;
  if ((out_token_stride | out_head_stride) % (out_dtype == SLMT_DTYPE_F32 ? 4 : 8) != 0) return SLMT_ERR_ALIGN;
  PromptParams p = {q, k, v, out, query_start_loc, seq_lens, err_flag, q_token_stride, q_head_stride,
                    k_token_stride, k_head_stride, v_token_stride, v_head_stride, out_token_stride, out_head_stride,
                    sm_scale, (int)num_tokens, (int)num_reqs, (int)std::min<int64_t>(max_query_len, num_tokens),
                    (int)num_q_heads, (int)num_kv_heads, dtype == SLMT_DTYPE_BF16, out_dtype};
  const dim3 grid((unsigned)(((int64_t)p.max_query * p.hq + 3) / 4), (unsigned)num_reqs);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (head_dim == 64) prompt_simple_kernel<64><<<grid, 128, 0, st>>>(p);
  else if (head_dim == 80) prompt_simple_kernel<80><<<grid, 128, 0, st>>>(p);
  else prompt_simple_kernel<128><<<grid, 128, 0, st>>>(p);
  return launch_status();
}
