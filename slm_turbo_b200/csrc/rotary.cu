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
constexpr int kRotRows = 4;   // q rows of a thread in flight
constexpr int kRotKRows = 2;  // k rows of a thread in flight, with their v rows

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

template <bool BF16>
__device__ __forceinline__ float from16(uint32_t bits) {
  return BF16 ? __bfloat162float(__ushort_as_bfloat16((uint16_t)bits)) : __half2float(__ushort_as_half((uint16_t)bits));
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (BF16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  return pack_half2(lo, hi);
}
__device__ __forceinline__ int64_t position_of(const RotaryParams& p, int64_t tok) {
  return p.pos_i64 ? reinterpret_cast<const int64_t*>(p.positions)[tok]
                   : (int64_t) reinterpret_cast<const int32_t*>(p.positions)[tok];
}

// D / 8 lanes to a row; D 80: 10 of 16.
template <int D>
struct RotGeom {
  static constexpr int ACTIVE = D / 8, LANES = D == 64 ? 8 : 16, SLOTS = kRotThreads / LANES;
};

// 8 of a row's values, dims d0..d0+3 and d1..d1+3, two to a word.
template <int LAYOUT>
__device__ __forceinline__ uint4 load8(const uint16_t* row, int d0, int d1) {
  if (LAYOUT == ROT_INTERLEAVED) return *reinterpret_cast<const uint4*>(row + d0);
  if (LAYOUT == ROT_ANY)
    return make_uint4(row[d0] | (uint32_t)row[d0 + 1] << 16, row[d0 + 2] | (uint32_t)row[d0 + 3] << 16,
                      row[d1] | (uint32_t)row[d1 + 1] << 16, row[d1 + 2] | (uint32_t)row[d1 + 3] << 16);
  const uint2 a = *reinterpret_cast<const uint2*>(row + d0), b = *reinterpret_cast<const uint2*>(row + d1);
  return make_uint4(a.x, a.y, b.x, b.y);
}
template <int LAYOUT>
__device__ __forceinline__ void store8(uint16_t* row, int d0, int d1, const uint4& w) {
  if (LAYOUT == ROT_INTERLEAVED) {
    *reinterpret_cast<uint4*>(row + d0) = w;
  } else if (LAYOUT == ROT_HALF) {
    *reinterpret_cast<uint2*>(row + d0) = make_uint2(w.x, w.y);
    *reinterpret_cast<uint2*>(row + d1) = make_uint2(w.z, w.w);
  } else {
    const uint32_t a[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int j = 0; j < 8; ++j) row[d0 + j] = (uint16_t)(j & 1 ? a[j >> 1] >> 16 : a[j >> 1]);
  }
}
template <bool BF16>
__device__ __forceinline__ void unpack8(const uint4& w, float (&x)[8]) {
  const uint32_t a[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = from16<BF16>(j & 1 ? a[j >> 1] >> 16 : a[j >> 1] & 0xFFFFu);
}
template <bool BF16>
__device__ __forceinline__ uint4 pack8(const float (&y)[8]) {
  return make_uint4(pack2<BF16>(y[0], y[1]), pack2<BF16>(y[2], y[3]), pack2<BF16>(y[4], y[5]), pack2<BF16>(y[6], y[7]));
}

// The turned row's 8 values.  cs: cos and sin of pairs pair0..pair0+3, of
// which the first `on` turn.  Every product and sum is rounded by itself.
template <int LAYOUT, bool BF16>
__device__ __forceinline__ uint4 turn8(const uint4& w, const float4 (&cs)[2], int on) {
  if (on <= 0) return w;
  float x[8], y[8];
  unpack8<BF16>(w, x);
  const float c[4] = {cs[0].x, cs[0].z, cs[1].x, cs[1].z}, s[4] = {cs[0].y, cs[0].w, cs[1].y, cs[1].w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int i1 = LAYOUT == ROT_HALF ? j : 2 * j, i2 = LAYOUT == ROT_HALF ? 4 + j : 2 * j + 1;
    // scalar: packed multiplies and adds were seen contracted into one rounding
    y[i1] = __fsub_rn(__fmul_rn(x[i1], c[j]), __fmul_rn(x[i2], s[j]));
    y[i2] = __fadd_rn(__fmul_rn(x[i2], c[j]), __fmul_rn(x[i1], s[j]));
  }
  if (on < 4) {
#pragma unroll
    for (int j = 1; j < 4; ++j)
      if (j >= on) y[2 * j] = x[2 * j], y[2 * j + 1] = x[2 * j + 1];
  }
  return pack8<BF16>(y);
}

// Smallest and largest of two packed 16-bit values each.
template <bool BF16>
__device__ __forceinline__ uint32_t min2(uint32_t a, uint32_t b) {
  if constexpr (BF16) {
    const __nv_bfloat162 r = __hmin2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  } else {
    const __half2 r = __hmin2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
}
template <bool BF16>
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
  if constexpr (BF16) {
    const __nv_bfloat162 r = __hmax2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  } else {
    const __half2 r = __hmax2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
}

// One row of k (turned) and v into its slot: the lanes of the row are
// neighbours in the warp, and the whole warp takes part in the exchange.  The
// rows hold 16-bit values, so their extremes are found on packed ones: k's in
// the lower half of a word, v's in the upper.  They start from the infinities
// as the store kernel's do: a row of NaN has a minimum of +infinity.
template <int D, int LAYOUT, bool BF16>
__device__ __forceinline__ void quantize8(const uint4& kw, const uint4& vw, uint8_t* row, bool act, bool write, int li,
                                          int d0, int d1) {
  constexpr uint32_t INF = BF16 ? 0x7F807F80u : 0x7C007C00u, NEG_INF = INF | 0x80008000u;
  const uint32_t k_lo = min2<BF16>(min2<BF16>(kw.x, kw.y), min2<BF16>(kw.z, kw.w));
  const uint32_t k_hi = max2<BF16>(max2<BF16>(kw.x, kw.y), max2<BF16>(kw.z, kw.w));
  const uint32_t v_lo = min2<BF16>(min2<BF16>(vw.x, vw.y), min2<BF16>(vw.z, vw.w));
  const uint32_t v_hi = max2<BF16>(max2<BF16>(vw.x, vw.y), max2<BF16>(vw.z, vw.w));
  uint32_t lo = min2<BF16>(__byte_perm(k_lo, v_lo, 0x5410), __byte_perm(k_lo, v_lo, 0x7632));
  uint32_t hi = max2<BF16>(__byte_perm(k_hi, v_hi, 0x5410), __byte_perm(k_hi, v_hi, 0x7632));
  lo = act ? min2<BF16>(lo, INF) : INF, hi = act ? max2<BF16>(hi, NEG_INF) : NEG_INF;
#pragma unroll
  for (int o = RotGeom<D>::LANES / 2; o > 0; o >>= 1) {
    lo = min2<BF16>(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = max2<BF16>(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  if (!write) return;
  const SlotScale ks = slot_scale(from16<BF16>(lo & 0xFFFFu), from16<BF16>(hi & 0xFFFFu));
  const SlotScale vs = slot_scale(from16<BF16>(lo >> 16), from16<BF16>(hi >> 16));
  float x[8];
  unpack8<BF16>(kw, x);
  const uint32_t kc = slot_codes8(x, ks);
  unpack8<BF16>(vw, x);
  const uint32_t vc = slot_codes8(x, vs);
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

// A token's slot in the cache, -1 if it has none.
__device__ __forceinline__ int64_t slot_of(const RotaryParams& p, int64_t tok, bool report) {
  const int64_t s = p.slot_mapping[tok];
  if (s < p.num_slots) return s;
  if (report && p.err) atomicOr(reinterpret_cast<unsigned int*>(p.err), SLMT_DEVERR_SLOT);
  return -1;
}

// TOKENS tokens per CTA.  The k rows come first (they are stored and
// quantized, which takes longest), then the q rows, kRotRows of a thread in
// flight.  The first rows' loads are issued before the CTA works out its
// tokens' angles -- double-precision sincos, a long chain -- which hides one
// behind the other; four tokens share that wait when there are enough of them
// to fill the GPU, and one token per CTA spreads few tokens over more SMs.
template <int D, int LAYOUT, bool STORE, bool BF16, int TOKENS>
__global__ void __launch_bounds__(kRotThreads, 4) rotary_kernel(const RotaryParams p) {
  using G = RotGeom<D>;
  constexpr int SLOTS = G::SLOTS;
  __shared__ float4 s_cs4[TOKENS][D / 4];  // pairs of (cos, sin): read two at a time
  const int64_t tok0 = (int64_t)blockIdx.x * TOKENS;
  const int nt = (int)min((int64_t)TOKENS, p.num_tokens - tok0);
  const int li = threadIdx.x % G::LANES, slot0 = threadIdx.x / G::LANES;
  const bool act = li < G::ACTIVE;
  const int half = p.half;
  // dims of the thread: 4 from d0 on and 4 from d1 on; pairs from pair0 on
  int d0 = 8 * li, d1 = d0 + 4, on;
  const int pair0 = 4 * li;
  if (LAYOUT == ROT_HALF) {
    on = li < half / 4 ? 4 : 0;
    d0 = on ? 4 * li : 2 * half + 8 * (li - half / 4);
    d1 = on ? half + 4 * li : d0 + 4;
  } else {
    on = half - pair0;
  }
  const uint16_t* q = reinterpret_cast<const uint16_t*>(p.q);
  const uint16_t* k = reinterpret_cast<const uint16_t*>(p.k);
  const uint16_t* v = reinterpret_cast<const uint16_t*>(p.v);
  uint16_t* q_out = reinterpret_cast<uint16_t*>(p.q_out);
  uint16_t* k_out = reinterpret_cast<uint16_t*>(p.k_out);

  auto angles = [&] {
    float2* s_cs = reinterpret_cast<float2*>(s_cs4);
    for (int i = threadIdx.x; i < nt * half; i += kRotThreads) {
      const int t = TOKENS == 1 ? 0 : i / half, f = TOKENS == 1 ? i : i - t * half;
      const float2 c = turn(position_of(p, tok0 + t), p.inv_freq[f]);
      s_cs[t * (D / 2) + f] = make_float2(__fmul_rn(c.x, p.scaling), __fmul_rn(c.y, p.scaling));
    }
    __syncthreads();
  };
  auto pairs_of = [&](int t, float4 (&cs)[2]) {
    if (act) cs[0] = s_cs4[t][pair0 / 2], cs[1] = s_cs4[t][pair0 / 2 + 1];
  };

  bool first = true;
  if (STORE) {  // k rows, two of a thread in flight
    constexpr int ROWS = kRotKRows;
    const int rows = nt * p.kv;
    int t = slot0 / p.kv, h = slot0 - t * p.kv;
    for (int base = 0; base < rows; base += SLOTS * ROWS) {
      uint4 x[ROWS], vx[ROWS];
      int tt[ROWS], hh[ROWS];
      int64_t slot[ROWS];
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        tt[r] = t, hh[r] = h;
        x[r] = vx[r] = make_uint4(0u, 0u, 0u, 0u);
        slot[r] = -1;
        if (t < nt) {
          const int64_t tok = tok0 + t;
          if (STORE) slot[r] = slot_of(p, tok, li == 0 && h == 0);
          if (act) {
            x[r] = load8<LAYOUT>(k + tok * p.k_tok + (int64_t)h * p.k_head, d0, d1);
            if (STORE && slot[r] >= 0) vx[r] = load8<LAYOUT>(v + tok * p.v_tok + (int64_t)h * p.v_head, d0, d1);
          }
        }
        h += SLOTS;
        while (h >= p.kv && t < nt) h -= p.kv, ++t;
      }
      if (first) angles();
      first = false;
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        const bool live = tt[r] < nt;
        float4 cs[2] = {};
        pairs_of(live ? tt[r] : 0, cs);
        const uint4 y = turn8<LAYOUT, BF16>(x[r], cs, on);
        if (live && act && k_out)
          store8<LAYOUT>(k_out + (tok0 + tt[r]) * p.ko_tok + (int64_t)hh[r] * p.ko_head, d0, d1, y);
        if (STORE && __any_sync(0xffffffffu, slot[r] >= 0))
          quantize8<D, LAYOUT, BF16>(y, vx[r], p.cache + (slot[r] * p.kv + hh[r]) * (D + 8), act, act && slot[r] >= 0,
                                     li, d0, d1);
      }
    }
  }
  {  // q rows, and k rows that are not stored
    const int heads = STORE ? p.hq : p.hq + p.kv, rows = nt * heads;
    int t = heads ? slot0 / heads : 0, h = slot0 - t * heads;
    for (int base = 0; base < rows; base += SLOTS * kRotRows) {
      uint4 x[kRotRows];
      uint16_t* out[kRotRows];
      int tt[kRotRows];
#pragma unroll
      for (int r = 0; r < kRotRows; ++r) {
        tt[r] = t;
        x[r] = make_uint4(0u, 0u, 0u, 0u);
        if (act && t < nt) {
          const int64_t tok = tok0 + t;
          if (STORE || h < p.hq) {
            x[r] = load8<LAYOUT>(q + tok * p.q_tok + (int64_t)h * p.q_head, d0, d1);
            out[r] = q_out + tok * p.qo_tok + (int64_t)h * p.qo_head;
          } else {
            x[r] = load8<LAYOUT>(k + tok * p.k_tok + (int64_t)(h - p.hq) * p.k_head, d0, d1);
            out[r] = k_out + tok * p.ko_tok + (int64_t)(h - p.hq) * p.ko_head;
          }
        }
        h += SLOTS;
        while (h >= heads && t < nt) h -= heads, ++t;
      }
      if (first) angles();
      first = false;
#pragma unroll
      for (int r = 0; r < kRotRows; ++r) {
        if (!act || tt[r] >= nt) continue;
        float4 cs[2] = {};
        pairs_of(tt[r], cs);
        store8<LAYOUT>(out[r], d0, d1, turn8<LAYOUT, BF16>(x[r], cs, on));
      }
    }
  }
}

// Rows at any alignment and any rot: a CTA per token, partners fetched one by
// one, a row of a thread at a time.  Partners are other threads' dims, so
// every row of a pass is read before any of it is written (in-place calls).
template <int D, bool STORE, bool BF16>
__global__ void __launch_bounds__(kRotThreads) rotary_any_kernel(const RotaryParams p) {
  using G = RotGeom<D>;
  __shared__ float2 s_cs[D / 2];
  const int64_t tok = blockIdx.x;
  const int li = threadIdx.x % G::LANES, slot0 = threadIdx.x / G::LANES;
  const bool act = li < G::ACTIVE;
  const int heads = p.hq + p.kv, half = p.half, d0 = 8 * li;
  for (int i = threadIdx.x; i < half; i += kRotThreads) {
    const float2 c = turn(position_of(p, tok), p.inv_freq[i]);
    s_cs[i] = make_float2(__fmul_rn(c.x, p.scaling), __fmul_rn(c.y, p.scaling));
  }
  const int64_t slot = STORE ? slot_of(p, tok, threadIdx.x == 0) : -1;
  for (int h0 = 0; h0 < heads; h0 += G::SLOTS) {
    const int h = h0 + slot0;
    const bool live = act && h < heads, is_k = h >= p.hq;
    const uint16_t* row = reinterpret_cast<const uint16_t*>(is_k ? p.k : p.q) +
                          (is_k ? tok * p.k_tok + (int64_t)(h - p.hq) * p.k_head : tok * p.q_tok + (int64_t)h * p.q_head);
    float x[8], other[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int i = d0 + j;
      const int o = i >= 2 * half ? i : p.interleaved ? i ^ 1 : i < half ? i + half : i - half;
      x[j] = live ? from16<BF16>(row[i]) : 0.f;
      other[j] = live ? from16<BF16>(row[o]) : 0.f;
    }
    __syncthreads();  // the angles; rows read
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int i = d0 + j;
      if (live && i < 2 * half) {
        const bool second = p.interleaved ? i & 1 : i >= half;
        const float2 c = s_cs[p.interleaved ? i >> 1 : second ? i - half : i];
        const float a = __fmul_rn(x[j], c.x), b = __fmul_rn(other[j], c.y);
        x[j] = second ? __fadd_rn(a, b) : __fsub_rn(a, b);
      }
    }
    const uint4 y = pack8<BF16>(x);
    uint16_t* dst = reinterpret_cast<uint16_t*>(is_k ? p.k_out : p.q_out);
    if (live && dst)
      store8<ROT_ANY>(dst + (is_k ? tok * p.ko_tok + (int64_t)(h - p.hq) * p.ko_head
                                  : tok * p.qo_tok + (int64_t)h * p.qo_head), d0, d0 + 4, y);
    if (STORE && slot >= 0 && __any_sync(0xffffffffu, h < heads && is_k)) {
      uint4 vw = make_uint4(0u, 0u, 0u, 0u);
      if (live && is_k)
        vw = load8<ROT_ANY>(reinterpret_cast<const uint16_t*>(p.v) + tok * p.v_tok + (int64_t)(h - p.hq) * p.v_head, d0,
                            d0 + 4);
      quantize8<D, ROT_ANY, BF16>(y, vw, p.cache + (slot * p.kv + (is_k ? h - p.hq : 0)) * (D + 8), act, live && is_k,
                                  li, d0, d0 + 4);
    }
    __syncthreads();  // before the next pass's rows are written
  }
}

template <int D, int LAYOUT, bool STORE, bool BF16>
int rotary_launch_tokens(const RotaryParams& p, cudaStream_t st) {
  // four tokens per CTA from two CTAs per SM on, one below
  if (p.num_tokens >= 8 * 148)
    rotary_kernel<D, LAYOUT, STORE, BF16, 4><<<(p.num_tokens + 3) / 4, kRotThreads, 0, st>>>(p);
  else
    rotary_kernel<D, LAYOUT, STORE, BF16, 1><<<p.num_tokens, kRotThreads, 0, st>>>(p);
  return launch_status();
}

template <int D, bool STORE, bool BF16>
int rotary_launch_typed(const RotaryParams& p, int layout, cudaStream_t st) {
  if (layout == ROT_HALF) return rotary_launch_tokens<D, ROT_HALF, STORE, BF16>(p, st);
  if (layout == ROT_INTERLEAVED) return rotary_launch_tokens<D, ROT_INTERLEAVED, STORE, BF16>(p, st);
  rotary_any_kernel<D, STORE, BF16><<<p.num_tokens, kRotThreads, 0, st>>>(p);
  return launch_status();
}

template <int D, bool STORE>
int rotary_launch_d(const RotaryParams& p, int layout, cudaStream_t st) {
  return p.bf16 ? rotary_launch_typed<D, STORE, true>(p, layout, st) : rotary_launch_typed<D, STORE, false>(p, layout, st);
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
