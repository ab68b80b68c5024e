// rotary.cu -- rotary positions of q and k rows, alone or together with the
// quantize-on-write of k and v into the 4-bit paged cache (sm_100a).
//
// Pair i of a row (dims i and i + rot/2, or 2i and 2i+1 interleaved) of a
// token at position p turns by theta = p * inv_freq[i]:
//     y1 = x1 c - x2 s,   y2 = x2 c + x1 s,
// c = a cos(theta), s = a sin(theta) (a: attention scaling); dims past rot
// pass through.  theta is taken in 64 bits -- p * inv_freq is exact there for
// positions below 2^29, where fp32 products are off by radians' worth of
// error at far positions -- and c, s are rounded to fp32; products, the sum
// and the final rounding to the 16-bit type are one fp32 rounding each, so
// the rows are those of the plain formula bit for bit, and the cache gets the
// bytes that the store kernel writes for them.
#include "internal.h"
#include "ptx.cuh"
#include "quant_store.cuh"

namespace slmt {

namespace {

constexpr int kRotThreads = 256;
constexpr int kRotTokens = 4;  // tokens of one CTA

struct RotaryParams {
  const void* q;
  const void* k;
  const void* v;  // null: no store
  void* q_out;
  void* k_out;  // null: the rotated k rows go to the cache only
  const void* positions;
  const float* inv_freq;
  uint8_t* cache;
  const int64_t* slot_mapping;
  int32_t* err;
  int64_t num_slots;
  int64_t q_tok, q_head, k_tok, k_head, v_tok, v_head, qo_tok, qo_head, ko_tok, ko_head;  // strides, elements
  float scaling;
  int num_tokens, hq, kv, half, interleaved, pos_i64, bf16;
};

__device__ __forceinline__ float load16(const void* p, int64_t i, int bf16) {
  return bf16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i])
              : __half2float(reinterpret_cast<const __half*>(p)[i]);
}

// cos and sin of p * f, in turns: the product is exact in 64 bits, its whole
// turns are taken off with the rest of the multiplication by 1/(2 pi) kept.
__device__ __forceinline__ float2 turn(int64_t pos, float f) {
  const double x = (double)pos * (double)f;
  const double hi = 0.15915494309189535, lo = -9.839338337591243e-18;  // 1/(2 pi) in two doubles
  const double n = rint(x * hi);
  const double r = fma(x, lo, fma(x, hi, -n));
  double s, c;
  sincospi(2.0 * r, &s, &c);
  return make_float2((float)c, (float)s);
}

template <int D>
__global__ void __launch_bounds__(kRotThreads) rotary_kernel(const RotaryParams p) {
  constexpr int VEC = SlotGeom<D>::VEC;
  __shared__ float2 s_cs[kRotTokens][D / 2];
  const int t0 = blockIdx.x * kRotTokens;
  const int nt = min(kRotTokens, p.num_tokens - t0);
  for (int i = threadIdx.x; i < nt * p.half; i += kRotThreads) {
    const int t = i / p.half, f = i - t * p.half;
    const int64_t pos = p.pos_i64 ? reinterpret_cast<const int64_t*>(p.positions)[t0 + t]
                                  : (int64_t) reinterpret_cast<const int32_t*>(p.positions)[t0 + t];
    const float2 cs = turn(pos, p.inv_freq[f]);
    s_cs[t][f] = make_float2(__fmul_rn(cs.x, p.scaling), __fmul_rn(cs.y, p.scaling));
  }
  __syncthreads();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int heads = p.hq + p.kv;
  for (int row = warp; row < nt * heads; row += kRotThreads / 32) {
    const int t = row / heads, h = row - t * heads;
    const int64_t tok = t0 + t;
    const bool is_k = h >= p.hq;
    const int hh = is_k ? h - p.hq : h;
    const int64_t in = is_k ? tok * p.k_tok + hh * p.k_head : tok * p.q_tok + hh * p.q_head;
    const void* src = is_k ? p.k : p.q;
    float y[VEC];
    const bool act = lane < SlotGeom<D>::LANES;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const int i = lane * VEC + j;
      y[j] = 0.f;
      if (act) {
        const float x = load16(src, in + i, p.bf16);
        y[j] = x;
        if (i < 2 * p.half) {
          bool second;
          int pair, other;
          if (p.interleaved) {
            second = i & 1, pair = i >> 1, other = i ^ 1;
          } else {
            second = i >= p.half, pair = second ? i - p.half : i, other = second ? i - p.half : i + p.half;
          }
          const float o = load16(src, in + other, p.bf16);
          const float2 cs = s_cs[t][pair];
          const float a = __fmul_rn(x, cs.x), b = __fmul_rn(o, cs.y);
          y[j] = second ? __fadd_rn(a, b) : __fsub_rn(a, b);
        }
        y[j] = p.bf16 ? __bfloat162float(__float2bfloat16_rn(y[j])) : __half2float(__float2half_rn(y[j]));
      }
    }
    __syncwarp();  // in place: the whole row is read before any of it is written
    void* dst = is_k ? p.k_out : p.q_out;
    if (dst && act) {
      const int64_t out = is_k ? tok * p.ko_tok + hh * p.ko_head : tok * p.qo_tok + hh * p.qo_head;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        if (p.bf16) reinterpret_cast<__nv_bfloat16*>(dst)[out + lane * VEC + j] = __float2bfloat16_rn(y[j]);
        else reinterpret_cast<__half*>(dst)[out + lane * VEC + j] = __float2half_rn(y[j]);
      }
    }
    if (is_k && p.cache) {
      const int64_t slot = p.slot_mapping[tok];
      if (slot >= p.num_slots) {
        if (lane == 0 && p.err) atomicOr(reinterpret_cast<unsigned int*>(p.err), SLMT_DEVERR_SLOT);
      } else if (slot >= 0) {
        float xv[VEC];
        const size_t esz = 2;
        load_row_vals<D>(reinterpret_cast<const uint8_t*>(p.v) + (tok * p.v_tok + hh * p.v_head) * esz, p.bf16, xv);
        const SlotRow r = quantize_slot_vals<D>(y, xv);
        write_slot_row<D>(p.cache + (slot * p.kv + hh) * (D + 8), r);
      }
    }
  }
}

int rotary_launch(const RotaryParams& p, int64_t head_dim, cudaStream_t st) {
  const dim3 grid((unsigned)((p.num_tokens + kRotTokens - 1) / kRotTokens));
  switch (head_dim) {
    case 64:
      rotary_kernel<64><<<grid, kRotThreads, 0, st>>>(p);
      break;
    case 80:
      rotary_kernel<80><<<grid, kRotThreads, 0, st>>>(p);
      break;
    default:
      rotary_kernel<128><<<grid, kRotThreads, 0, st>>>(p);
  }
  return launch_status();
}

// Checks shared by both entries; SLMT_OK and *empty for a call with no rows.
int rotary_check(const void* q, const void* k, int dtype, const void* positions, int pos_dtype, const float* inv_freq,
                 int64_t rotary_dim, float scaling, int64_t num_tokens, int64_t hq, int64_t kv, int64_t head_dim,
                 bool* empty) {
  *empty = false;
  if (!valid_head_dim(head_dim)) return SLMT_ERR_HEAD_DIM;
  if (num_tokens < 0 || num_tokens > INT32_MAX / 2 || hq < 0 || kv < 0 || hq > 65535 || kv > 65535)
    return SLMT_ERR_SHAPE;
  if (rotary_dim < 0 || rotary_dim > head_dim || rotary_dim % 2 != 0) return SLMT_ERR_SHAPE;
  if (dtype != SLMT_DTYPE_F16 && dtype != SLMT_DTYPE_BF16) return SLMT_ERR_DTYPE;
  if (pos_dtype != SLMT_DTYPE_I32 && pos_dtype != SLMT_DTYPE_I64) return SLMT_ERR_DTYPE;
  if (!(scaling - scaling == 0.0f)) return SLMT_ERR_SHAPE;  // not finite
  if (num_tokens == 0 || hq + kv == 0) {
    *empty = true;
    return SLMT_OK;
  }
  if ((hq > 0 && !q) || (kv > 0 && !k) || !positions || (rotary_dim > 0 && !inv_freq)) return SLMT_ERR_NULL;
  return SLMT_OK;
}

}  // namespace
}  // namespace slmt

using namespace slmt;

extern "C" int slmt_rotary(const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* k,
                           int64_t k_token_stride, int64_t k_head_stride, int dtype, const void* positions,
                           int pos_dtype, const float* inv_freq, int64_t rotary_dim, int interleaved, float scaling,
                           int64_t num_tokens, int64_t num_q_heads, int64_t num_kv_heads, int64_t head_dim,
                           void* q_out, int64_t qo_token_stride, int64_t qo_head_stride, void* k_out,
                           int64_t ko_token_stride, int64_t ko_head_stride, void* stream) {
  bool empty;
  const int rc = rotary_check(q, k, dtype, positions, pos_dtype, inv_freq, rotary_dim, scaling, num_tokens,
                              num_q_heads, num_kv_heads, head_dim, &empty);
  if (rc != SLMT_OK || empty) return rc;
  if ((num_q_heads > 0 && !q_out) || (num_kv_heads > 0 && !k_out)) return SLMT_ERR_NULL;
  if (rows_overlap(num_tokens, num_q_heads, qo_token_stride, qo_head_stride) ||
      rows_overlap(num_tokens, num_kv_heads, ko_token_stride, ko_head_stride))
    return SLMT_ERR_SHAPE;
  const RotaryParams p = {q, k, nullptr, q_out, k_out, positions, inv_freq, nullptr, nullptr, nullptr, 0,
                          q_token_stride, q_head_stride, k_token_stride, k_head_stride, 0, 0, qo_token_stride,
                          qo_head_stride, ko_token_stride, ko_head_stride, scaling, (int)num_tokens,
                          (int)num_q_heads, (int)num_kv_heads, (int)(rotary_dim / 2), interleaved != 0,
                          pos_dtype == SLMT_DTYPE_I64, dtype == SLMT_DTYPE_BF16};
  return rotary_launch(p, head_dim, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int slmt_rotary_store(const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* k,
                                 int64_t k_token_stride, int64_t k_head_stride, const void* v, int64_t v_token_stride,
                                 int64_t v_head_stride, int dtype, const void* positions, int pos_dtype,
                                 const float* inv_freq, int64_t rotary_dim, int interleaved, float scaling,
                                 int64_t num_tokens, int64_t num_q_heads, int64_t num_kv_heads, int64_t head_dim,
                                 void* q_out, int64_t qo_token_stride, int64_t qo_head_stride, void* k_out,
                                 int64_t ko_token_stride, int64_t ko_head_stride, uint8_t* kv_cache,
                                 int64_t num_blocks, int64_t block_size, const int64_t* slot_mapping,
                                 int32_t* err_flag, void* stream) {
  bool empty;
  const int rc = rotary_check(q, k, dtype, positions, pos_dtype, inv_freq, rotary_dim, scaling, num_tokens,
                              num_q_heads, num_kv_heads, head_dim, &empty);
  if (rc != SLMT_OK || empty) return rc;
  if (num_kv_heads <= 0 || num_blocks < 0 || block_size <= 0) return SLMT_ERR_SHAPE;
  if ((num_q_heads > 0 && !q_out) || !v || !kv_cache || !slot_mapping) return SLMT_ERR_NULL;
  if (rows_overlap(num_tokens, num_q_heads, qo_token_stride, qo_head_stride) ||
      (k_out && rows_overlap(num_tokens, num_kv_heads, ko_token_stride, ko_head_stride)))
    return SLMT_ERR_SHAPE;
  if (reinterpret_cast<uintptr_t>(kv_cache) % 8 != 0) return SLMT_ERR_ALIGN;
  const RotaryParams p = {q, k, v, q_out, k_out, positions, inv_freq, kv_cache, slot_mapping, err_flag,
                          num_blocks * block_size, q_token_stride, q_head_stride, k_token_stride, k_head_stride,
                          v_token_stride, v_head_stride, qo_token_stride, qo_head_stride, ko_token_stride,
                          ko_head_stride, scaling, (int)num_tokens, (int)num_q_heads, (int)num_kv_heads,
                          (int)(rotary_dim / 2), interleaved != 0, pos_dtype == SLMT_DTYPE_I64,
                          dtype == SLMT_DTYPE_BF16};
  return rotary_launch(p, head_dim, reinterpret_cast<cudaStream_t>(stream));
}
