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
constexpr int kRotRows = 4;  // rows of a thread in flight

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

// How a thread's 8 dims of a row lie.
enum RotaryLayout {
  ROT_HALF = 0,         // 4 pairs as dims 4i.. and rot/2 + 4i.., or 8 dims past rot: half % 4 == 0, aligned rows
  ROT_INTERLEAVED = 1,  // 4 pairs, 8 dims next to one another, aligned rows
  ROT_ANY = 2           // 8 dims next to one another, partners fetched one by one
};

__device__ __forceinline__ float from16(uint32_t bits, int bf16) {
  return bf16 ? __bfloat162float(__ushort_as_bfloat16((uint16_t)bits)) : __half2float(__ushort_as_half((uint16_t)bits));
}
__device__ __forceinline__ uint32_t to16(float x, int bf16) {
  return bf16 ? (uint32_t)__bfloat16_as_ushort(__float2bfloat16_rn(x)) : (uint32_t)__half_as_ushort(__float2half_rn(x));
}

// One CTA per token: D / 8 lanes to a row (D 80: 10 of 16), so a thread's
// pairs are the same in every row and their cos and sin stay in registers.
// The rows' loads are issued before the CTA works out the token's angles (64
// double-precision sincos at most, a thread each), which hides one behind the
// other.
template <int D, int LAYOUT, bool STORE>
__global__ void __launch_bounds__(kRotThreads) rotary_kernel(const RotaryParams p) {
  constexpr int ACTIVE = D / 8, LANES = D == 64 ? 8 : 16, SLOTS = kRotThreads / LANES;
  constexpr int ROWS = LAYOUT == ROT_ANY ? 1 : kRotRows;
  __shared__ float2 s_cs[D / 2];
  const int64_t tok = blockIdx.x;
  const int li = threadIdx.x % LANES, slot0 = threadIdx.x / LANES;
  const bool act = li < ACTIVE;
  const int heads = p.hq + p.kv, half = p.half;
  // dims of the thread: 4 from d0 on and 4 from d1 on; pairs from pair0 on
  int d0 = 8 * li, d1 = d0 + 4, pair0 = 4 * li;
  bool turns = false;  // HALF: all 4 pairs turn, or none
  if (LAYOUT == ROT_HALF) {
    turns = li < half / 4;
    d0 = turns ? 4 * li : 2 * half + 8 * (li - half / 4);
    d1 = turns ? half + 4 * li : d0 + 4;
  }
  float2 cs[4];
  const uint16_t* q = reinterpret_cast<const uint16_t*>(p.q);
  const uint16_t* k = reinterpret_cast<const uint16_t*>(p.k);
  const uint16_t* v = reinterpret_cast<const uint16_t*>(p.v);
  int64_t cache_slot = -1;
  if (STORE) {
    cache_slot = p.slot_mapping[tok];
    if (cache_slot >= p.num_slots) {
      if (threadIdx.x == 0 && p.err) atomicOr(reinterpret_cast<unsigned int*>(p.err), SLMT_DEVERR_SLOT);
      cache_slot = -1;
    }
  }
  bool first = true;
  for (int h0 = 0; h0 < heads; h0 += SLOTS * ROWS) {
    uint2 lo[ROWS], hi[ROWS], vlo[ROWS], vhi[ROWS];
    float other[8];  // ROT_ANY: the partners
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const int h = h0 + slot0 + r * SLOTS;
      lo[r] = hi[r] = vlo[r] = vhi[r] = make_uint2(0u, 0u);
      if (!act || h >= heads) continue;
      const bool is_k = h >= p.hq;
      const uint16_t* row = is_k ? k + tok * p.k_tok + (int64_t)(h - p.hq) * p.k_head
                                 : q + tok * p.q_tok + (int64_t)h * p.q_head;
      if (LAYOUT == ROT_HALF) {
        lo[r] = *reinterpret_cast<const uint2*>(row + d0);
        hi[r] = *reinterpret_cast<const uint2*>(row + d1);
      } else if (LAYOUT == ROT_INTERLEAVED) {
        const uint4 x = *reinterpret_cast<const uint4*>(row + d0);
        lo[r] = make_uint2(x.x, x.y), hi[r] = make_uint2(x.z, x.w);
      } else {
        uint32_t e[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int i = d0 + j;
          e[j] = row[i];
          int o = i;
          if (i < 2 * half) o = p.interleaved ? i ^ 1 : (i < half ? i + half : i - half);
          other[j] = from16(row[o], p.bf16);
        }
        lo[r] = make_uint2(e[0] | e[1] << 16, e[2] | e[3] << 16);
        hi[r] = make_uint2(e[4] | e[5] << 16, e[6] | e[7] << 16);
      }
      if (STORE && is_k && cache_slot >= 0) {
        const uint16_t* vr = v + tok * p.v_tok + (int64_t)(h - p.hq) * p.v_head;
        if (LAYOUT == ROT_HALF) {
          vlo[r] = *reinterpret_cast<const uint2*>(vr + d0);
          vhi[r] = *reinterpret_cast<const uint2*>(vr + d1);
        } else if (LAYOUT == ROT_INTERLEAVED) {
          const uint4 x = *reinterpret_cast<const uint4*>(vr + d0);
          vlo[r] = make_uint2(x.x, x.y), vhi[r] = make_uint2(x.z, x.w);
        } else {
          vlo[r] = make_uint2(vr[d0] | (uint32_t)vr[d0 + 1] << 16, vr[d0 + 2] | (uint32_t)vr[d0 + 3] << 16);
          vhi[r] = make_uint2(vr[d1] | (uint32_t)vr[d1 + 1] << 16, vr[d1 + 2] | (uint32_t)vr[d1 + 3] << 16);
        }
      }
    }
    if (first) {
      for (int i = threadIdx.x; i < half; i += kRotThreads) {
        const int64_t pos = p.pos_i64 ? reinterpret_cast<const int64_t*>(p.positions)[tok]
                                      : (int64_t) reinterpret_cast<const int32_t*>(p.positions)[tok];
        const float2 t = turn(pos, p.inv_freq[i]);
        s_cs[i] = make_float2(__fmul_rn(t.x, p.scaling), __fmul_rn(t.y, p.scaling));
      }
    }
    // the angles; and, where partners are other threads' dims, every row is
    // read before any of it is written (in-place calls)
    if (first || LAYOUT == ROT_ANY) __syncthreads();
    if (first && LAYOUT != ROT_ANY) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bool on = act && (LAYOUT == ROT_HALF ? turns : pair0 + j < half);
        cs[j] = on ? s_cs[pair0 + j] : make_float2(0.f, 0.f);
      }
    }
    first = false;
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const int h = h0 + slot0 + r * SLOTS;
      const bool live = act && h < heads;
      const bool is_k = h >= p.hq;
      // x: dims d0..d0+3, d1..d1+3
      float x[8];
      const uint32_t w[4] = {lo[r].x, lo[r].y, hi[r].x, hi[r].y};
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = from16(j & 1 ? w[j >> 1] >> 16 : w[j >> 1] & 0xFFFFu, p.bf16);
      uint32_t y[8];
      if (LAYOUT == ROT_HALF) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float a = x[j], b = x[4 + j];
          y[j] = to16(turns ? __fsub_rn(__fmul_rn(a, cs[j].x), __fmul_rn(b, cs[j].y)) : a, p.bf16);
          y[4 + j] = to16(turns ? __fadd_rn(__fmul_rn(b, cs[j].x), __fmul_rn(a, cs[j].y)) : b, p.bf16);
        }
      } else if (LAYOUT == ROT_INTERLEAVED) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float a = x[2 * j], b = x[2 * j + 1];
          const bool on = pair0 + j < half;
          y[2 * j] = to16(on ? __fsub_rn(__fmul_rn(a, cs[j].x), __fmul_rn(b, cs[j].y)) : a, p.bf16);
          y[2 * j + 1] = to16(on ? __fadd_rn(__fmul_rn(b, cs[j].x), __fmul_rn(a, cs[j].y)) : b, p.bf16);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int i = d0 + j;
          float z = x[j];
          if (live && i < 2 * half) {
            const bool second = p.interleaved ? i & 1 : i >= half;
            const float2 t = s_cs[p.interleaved ? i >> 1 : second ? i - half : i];
            const float a = __fmul_rn(z, t.x), b = __fmul_rn(other[j], t.y);
            z = second ? __fadd_rn(a, b) : __fsub_rn(a, b);
          }
          y[j] = to16(z, p.bf16);
        }
      }
      uint16_t* dst = reinterpret_cast<uint16_t*>(is_k ? p.k_out : p.q_out);
      if (live && dst) {
        dst += is_k ? tok * p.ko_tok + (int64_t)(h - p.hq) * p.ko_head : tok * p.qo_tok + (int64_t)h * p.qo_head;
        const uint2 a = make_uint2(y[0] | y[1] << 16, y[2] | y[3] << 16);
        const uint2 b = make_uint2(y[4] | y[5] << 16, y[6] | y[7] << 16);
        if (LAYOUT == ROT_HALF) {
          *reinterpret_cast<uint2*>(dst + d0) = a;
          *reinterpret_cast<uint2*>(dst + d1) = b;
        } else if (LAYOUT == ROT_INTERLEAVED) {
          *reinterpret_cast<uint4*>(dst + d0) = make_uint4(a.x, a.y, b.x, b.y);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) dst[d0 + j] = (uint16_t)y[j];
        }
      }
      // the cache: the whole warp takes part where a row of it is a k row
      if (STORE && cache_slot >= 0 && __any_sync(0xffffffffu, h < heads && is_k)) {
        float mn[2] = {INFINITY, INFINITY}, mx[2] = {-INFINITY, -INFINITY}, vx[8], kx[8];
        const uint32_t vw[4] = {vlo[r].x, vlo[r].y, vhi[r].x, vhi[r].y};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          vx[j] = from16(j & 1 ? vw[j >> 1] >> 16 : vw[j >> 1] & 0xFFFFu, p.bf16);
          kx[j] = from16(y[j], p.bf16);
          if (act) {
            mn[0] = fminf(mn[0], kx[j]), mx[0] = fmaxf(mx[0], kx[j]);
            mn[1] = fminf(mn[1], vx[j]), mx[1] = fmaxf(mx[1], vx[j]);
          }
        }
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            mn[i] = fminf(mn[i], __shfl_xor_sync(0xffffffffu, mn[i], o));
            mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], o));
          }
        }
        if (live && is_k) {
          const SlotScale ks = slot_scale(mn[0], mx[0]), vs = slot_scale(mn[1], mx[1]);
          uint32_t kc = 0u, vc = 0u;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            kc |= slot_code(kx[j], ks) << (4 * j);
            vc |= slot_code(vx[j], vs) << (4 * j);
          }
          uint8_t* row = p.cache + (cache_slot * p.kv + (h - p.hq)) * (D + 8);
          if (LAYOUT == ROT_HALF) {
            *reinterpret_cast<uint16_t*>(row + d0 / 2) = (uint16_t)kc;
            *reinterpret_cast<uint16_t*>(row + d1 / 2) = (uint16_t)(kc >> 16);
            *reinterpret_cast<uint16_t*>(row + D / 2 + d0 / 2) = (uint16_t)vc;
            *reinterpret_cast<uint16_t*>(row + D / 2 + d1 / 2) = (uint16_t)(vc >> 16);
          } else {
            *reinterpret_cast<uint32_t*>(row + d0 / 2) = kc;
            *reinterpret_cast<uint32_t*>(row + D / 2 + d0 / 2) = vc;
          }
          if (li == 0) *reinterpret_cast<uint2*>(row + D) = make_uint2(slot_rulers(ks), slot_rulers(vs));
        }
      }
    }
    if (LAYOUT == ROT_ANY && h0 + SLOTS * ROWS < heads) __syncthreads();
  }
}

template <int D, bool STORE>
int rotary_launch_d(const RotaryParams& p, int layout, cudaStream_t st) {
  const dim3 grid((unsigned)p.num_tokens);
  if (layout == ROT_HALF)
    rotary_kernel<D, ROT_HALF, STORE><<<grid, kRotThreads, 0, st>>>(p);
  else if (layout == ROT_INTERLEAVED)
    rotary_kernel<D, ROT_INTERLEAVED, STORE><<<grid, kRotThreads, 0, st>>>(p);
  else
    rotary_kernel<D, ROT_ANY, STORE><<<grid, kRotThreads, 0, st>>>(p);
  return launch_status();
}

// Whether rows at these strides can be read and written `bytes` at a time.
bool rows_aligned(const void* base, int64_t tok, int64_t head, int64_t bytes) {
  return reinterpret_cast<uintptr_t>(base) % bytes == 0 && (2 * tok) % bytes == 0 && (2 * head) % bytes == 0;
}

int rotary_launch(const RotaryParams& p, int64_t head_dim, cudaStream_t st) {
  const int64_t bytes = p.interleaved ? 16 : 8;
  const bool aligned = rows_aligned(p.q, p.q_tok, p.q_head, bytes) && rows_aligned(p.k, p.k_tok, p.k_head, bytes) &&
                       rows_aligned(p.v, p.v_tok, p.v_head, bytes) && rows_aligned(p.q_out, p.qo_tok, p.qo_head, bytes) &&
                       rows_aligned(p.k_out, p.ko_tok, p.ko_head, bytes);
  const int layout = !aligned ? ROT_ANY : p.interleaved ? ROT_INTERLEAVED : p.half % 4 == 0 ? ROT_HALF : ROT_ANY;
  const bool store = p.cache != nullptr;
  switch (head_dim) {
    case 64:
      return store ? rotary_launch_d<64, true>(p, layout, st) : rotary_launch_d<64, false>(p, layout, st);
    case 80:
      return store ? rotary_launch_d<80, true>(p, layout, st) : rotary_launch_d<80, false>(p, layout, st);
    default:
      return store ? rotary_launch_d<128, true>(p, layout, st) : rotary_launch_d<128, false>(p, layout, st);
  }
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
