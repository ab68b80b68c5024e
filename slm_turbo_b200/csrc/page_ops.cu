// page_ops.cu -- page bookkeeping around the 4-bit paged cache (sm_100a).
//
//  * page_plan_kernel: block tables, slot ids and positions of one serving
//    step, from the requests' lengths alone.
//  * load_kernel: packed slots back to 16- or 32-bit K and V rows.
#include "internal.h"
#include "ptx.cuh"

namespace slmt {

namespace {

// ------------------------------------------------------------- page plan --
// Request r brings the n_r = qsl[r+1] - qsl[r] last of its seq_lens[r]
// tokens, the first of them at position ctx_r = seq_lens[r] - n_r.  It owns
// have_r = ceil(ctx_r / bs) pages and needs need_r = ceil(seq_lens[r] / bs);
// page have_r + i is free_blocks[cursor + off_r + i] with the exclusive sum
// off_r = sum_{r' < r} (need_r' - have_r').  Every CTA sums the requests for
// itself (a tile of kPlanTile at a time), so one launch does all of it with
// no exchange between CTAs and no atomics: the plan is the same every time.
// A new page's first token is always one of the step's new tokens
// (have_r * bs >= ctx_r), so the thread of that token writes the table entry;
// entries of new pages are never read here, only computed.
// Bound by latency: the reads of the lengths, the sum, the search and the
// page's read follow one another.  64 prompts of 270 K tokens 5.4 us (7.6 with
// a thread's four tokens one after another and 32-bit divisions by the block
// size), 256 requests of one token 4.1 us (4.6), a launch alone 2.2.
constexpr int kPlanThreads = 256;
constexpr int kPlanTile = 1024;              // requests summed at a time
constexpr int kPlanTokens = 4 * kPlanThreads;  // tokens of one CTA

struct PlanParams {
  const int32_t* qsl;
  const int32_t* seq_lens;
  int32_t* tables;
  int64_t table_stride;
  const int32_t* free_blocks;  // null: the tables are complete already
  int64_t num_free;
  const int32_t* cursor_in;  // null: 0
  int64_t* slots;
  int64_t* positions;
  int32_t* cursor_out;
  int32_t* err;
  int num_reqs, num_tokens, block_size, max_blocks;
  int shift;  // log2 of the block size, -1 if it is no power of two

  __device__ __forceinline__ int pages(int tokens) const {  // rounded down
    return shift >= 0 ? tokens >> shift : (int)((unsigned)tokens / (unsigned)block_size);
  }
  __device__ __forceinline__ int pages_up(int tokens) const {
    const unsigned x = (unsigned)tokens + (unsigned)block_size - 1u;
    return (int)(shift >= 0 ? x >> shift : x / (unsigned)block_size);
  }
};

__device__ __forceinline__ void set_error(int32_t* err, unsigned bit) {
  if (err) atomicOr(reinterpret_cast<unsigned int*>(err), bit);
}

__global__ void __launch_bounds__(kPlanThreads) page_plan_kernel(const PlanParams p) {
  __shared__ int s_start[kPlanTile + 1];  // query_start_loc of the tile
  __shared__ int s_ctx[kPlanTile];        // tokens before the step's, -1: lengths that do not fit
  __shared__ int64_t s_off[kPlanTile];    // place of the request's first new page in the free list
  __shared__ int64_t s_warp[kPlanThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int t0 = blockIdx.x * kPlanTokens;
  const int t1 = min(t0 + kPlanTokens, p.num_tokens);
  unsigned bad = 0u;

  const int first = p.num_reqs ? p.qsl[0] : 0, last = p.num_reqs ? p.qsl[p.num_reqs] : 0;
  int64_t base = p.cursor_in ? (int64_t)*p.cursor_in : 0;
  for (int r0 = 0; r0 < p.num_reqs; r0 += kPlanTile) {
    const int nr = min(kPlanTile, p.num_reqs - r0);
    constexpr int PER = kPlanTile / kPlanThreads;
    // thread t sums the requests PER*t .. PER*t+PER-1 of the tile
    int grow[PER];
    int64_t sum = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int r = PER * tid + i;
      grow[i] = 0;
      if (r < nr) {
        const int a = p.qsl[r0 + r], b = p.qsl[r0 + r + 1], len = p.seq_lens[r0 + r];
        int ctx = len - (b - a);
        if (b < a || ctx < 0 || a < 0) {
          ctx = -1;
          bad |= SLMT_DEVERR_SEQ_LEN;
        } else {
          const int need = min(p.pages_up(len), p.max_blocks), have = min(p.pages_up(ctx), p.max_blocks);
          grow[i] = p.free_blocks ? need - have : 0;
        }
        s_start[r] = a;
        s_ctx[r] = ctx;
        if (r == nr - 1) s_start[nr] = b;
      }
      sum += grow[i];
    }
    int64_t incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t x = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += x;
    }
    if (lane == 31) s_warp[warp] = incl;
    __syncthreads();
    int64_t before = base, total = 0;
#pragma unroll
    for (int w = 0; w < kPlanThreads / 32; ++w) {
      if (w < warp) before += s_warp[w];
      total += s_warp[w];
    }
    before += incl - sum;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int r = PER * tid + i;
      if (r < nr) s_off[r] = before;
      before += grow[i];
    }
    base += total;
    __syncthreads();

    // four tokens of a thread at a time: their searches and their pages' reads
    // are under way together
    constexpr int U = kPlanTokens / kPlanThreads;
    const int lo_t = max(t0, s_start[0]), hi_t = min(t1, s_start[nr]);
    if (lo_t < hi_t) {
      int req[U] = {};
      for (int step = 1 << (31 - __clz(nr)); step > 0; step >>= 1) {
#pragma unroll
        for (int u = 0; u < U; ++u) {  // the last request of the tile that starts at or before the token
          const int r = req[u] + step;
          if (r < nr && s_start[r] <= t0 + u * kPlanThreads + tid) req[u] = r;
        }
      }
      int pos[U], in_page[U];
      int32_t* entry[U];
      const int32_t* from[U];
      bool own[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int t = t0 + u * kPlanThreads + tid, r = req[u], ctx = s_ctx[r];
        pos[u] = in_page[u] = 0;
        entry[u] = nullptr, from[u] = nullptr;
        own[u] = t >= lo_t && t < hi_t;
        if (!own[u] || ctx < 0 || t < s_start[r] || t >= s_start[r + 1]) continue;
        pos[u] = ctx + (t - s_start[r]);
        const int page = p.pages(pos[u]);
        in_page[u] = pos[u] - page * p.block_size;
        if (page >= p.max_blocks) {
          bad |= SLMT_DEVERR_SEQ_LEN;
          continue;
        }
        int32_t* e = p.tables + (int64_t)(r0 + r) * p.table_stride + page;
        const int have = p.pages_up(ctx);
        if (p.free_blocks && page >= have) {
          const int64_t at = s_off[r] + (page - have);
          if (at >= 0 && at < p.num_free) from[u] = p.free_blocks + at;
          else bad |= SLMT_DEVERR_FREE_BLOCKS;
          if (in_page[u] == 0) entry[u] = e;
        } else {
          from[u] = e;
        }
      }
      int block[U];
#pragma unroll
      for (int u = 0; u < U; ++u) block[u] = from[u] ? *from[u] : -1;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int t = t0 + u * kPlanThreads + tid;
        if (from[u] && block[u] < 0) bad |= SLMT_DEVERR_BLOCK_ID;
        if (entry[u]) *entry[u] = block[u];
        if (!own[u]) continue;
        p.slots[t] = block[u] < 0 ? -1 : (int64_t)block[u] * p.block_size + in_page[u];
        p.positions[t] = pos[u];
      }
    }
    __syncthreads();  // the tile's arrays are filled again
  }
  // rows of no request: the padding behind the last token (and anything
  // before the first request's rows)
  for (int t = t0 + tid; t < t1; t += kPlanThreads) {
    if (t < first || t >= last) {
      p.slots[t] = -1;
      p.positions[t] = 0;
    }
  }
  if (last > p.num_tokens || first < 0) bad |= SLMT_DEVERR_SEQ_LEN;
  if (blockIdx.x == 0 && tid == 0 && p.cursor_out) {
    if (p.free_blocks && base > p.num_free) {
      bad |= SLMT_DEVERR_FREE_BLOCKS;
      base = p.num_free;
    }
    *p.cursor_out = (int32_t)base;
  }
  if (bad) set_error(p.err, bad);
}

// ------------------------------------------------------------------- load --
// x = code * step + min in fp32 (code * step is exact: 4 by 11 bits), rounded
// once.  A thread turns 4 code bytes into 8 values: D/8 threads for a row's
// K, D/8 for its V, so a warp's reads and 16-byte writes are contiguous.
template <typename T>
struct Vec8;
template <>
struct Vec8<__half> {
  static __device__ __forceinline__ void store(void* p, const float (&x)[8]) {
    uint4 v;
    v.x = pack_half2(x[0], x[1]), v.y = pack_half2(x[2], x[3]);
    v.z = pack_half2(x[4], x[5]), v.w = pack_half2(x[6], x[7]);
    *reinterpret_cast<uint4*>(p) = v;
  }
};
__device__ __forceinline__ uint32_t pack_bf162(float lo, float hi) {
  __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&h);
}
template <>
struct Vec8<__nv_bfloat16> {
  static __device__ __forceinline__ void store(void* p, const float (&x)[8]) {
    uint4 v;
    v.x = pack_bf162(x[0], x[1]), v.y = pack_bf162(x[2], x[3]);
    v.z = pack_bf162(x[4], x[5]), v.w = pack_bf162(x[6], x[7]);
    *reinterpret_cast<uint4*>(p) = v;
  }
};
template <>
struct Vec8<float> {
  static __device__ __forceinline__ void store(void* p, const float (&x)[8]) {
    reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
  }
};

// A thread keeps its place in a token's slots (head, K or V, piece) and walks
// over tokens, four at a time; places are found once, with 32-bit arithmetic.
// The next four tokens' slot ids are fetched two steps ahead and their code
// words one step ahead of their conversion.
constexpr int kLoadThreads = 256;
constexpr int kLoadUnroll = 4;

template <int D, typename T>
__global__ void __launch_bounds__(kLoadThreads)
    load_kernel(const uint8_t* __restrict__ cache, int64_t num_slots, const int64_t* __restrict__ slot_mapping,
                int64_t num_tokens, int kv, int places, int sub_tokens, int steps, T* __restrict__ key,
                T* __restrict__ value, int32_t* err) {
  constexpr int PIECES = D / 4, U = kLoadUnroll;  // 8-value pieces of a row's K and V
  // `places` pieces of a token in this block's pass (kv * PIECES when a block
  // holds whole tokens, sub_tokens of them; else a part, by blockIdx.y)
  const int sub = threadIdx.x / places;
  const int place = threadIdx.x - sub * places + blockIdx.y * kLoadThreads;
  if (sub >= sub_tokens || place >= kv * PIECES) return;
  const int h = place / PIECES, piece = place - h * PIECES;
  const int which = piece >= PIECES / 2, c = piece - which * (PIECES / 2);
  const int64_t slot_bytes = (int64_t)kv * (D + 8);
  const uint8_t* code_base = cache + (int64_t)h * (D + 8) + which * (D / 2) + 4 * c;
  const int to_ruler = D + 4 * which - which * (D / 2) - 4 * c;
  T* out = (which ? value : key) + (int64_t)h * D + 8 * c;
  int64_t t = (int64_t)blockIdx.x * (sub_tokens * U) * steps + sub;  // first token of this step
  int64_t slot[U];
  uint32_t codes[U], rulers[U];
  auto fetch_slots = [&](int64_t from) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t tok = from + u * sub_tokens;
      slot[u] = tok < num_tokens ? slot_mapping[tok] : -1;
    }
  };
  auto fetch_codes = [&] {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      codes[u] = rulers[u] = 0u;  // code 0, min 0: a row of zeros
      if ((uint64_t)slot[u] < (uint64_t)num_slots) {
        const uint8_t* s = code_base + slot[u] * slot_bytes;
        codes[u] = *reinterpret_cast<const uint32_t*>(s);
        rulers[u] = *reinterpret_cast<const uint32_t*>(s + to_ruler);
      } else if (slot[u] >= 0 && place == 0) {
        set_error(err, SLMT_DEVERR_SLOT);
      }
    }
  };
  fetch_slots(t);
  fetch_codes();
  if (steps > 1) fetch_slots(t + U * sub_tokens);
#pragma unroll 1
  for (int step = 0; step < steps; ++step) {
    uint32_t now_codes[U], now_rulers[U];
#pragma unroll
    for (int u = 0; u < U; ++u) now_codes[u] = codes[u], now_rulers[u] = rulers[u];
    if (step + 1 < steps) {
      fetch_codes();
      if (step + 2 < steps) fetch_slots(t + 2 * U * sub_tokens);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t tok = t + u * sub_tokens;
      if (tok >= num_tokens) return;
      const float mn = half_bits_to_float((uint16_t)(now_rulers[u] & 0xFFFFu));
      const float st = half_bits_to_float((uint16_t)(now_rulers[u] >> 16));
      // A nibble left where it is under the bits of 2^23 is the float 2^23 +
      // code * 16^j: one multiply-add with 16^-j and -2^23 16^-j gives the
      // code, exactly, without shifts or integer conversions.  Five nibbles
      // fit below bit 23; four are taken from the word as it is, four shifted.
      const uint64_t st2 = f2_pack(st, st), mn2 = f2_pack(mn, mn);
      const uint32_t w0 = now_codes[u], w1 = w0 >> 16;
      float x[8];
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        const uint32_t w = j < 4 ? w0 : w1;
        const int k = j & 3;  // nibbles k and k + 1 of w
        const float s0 = 1.f / (float)(1 << (4 * k)), s1 = s0 / 16.f;
        const uint64_t biased = f2_pack(__uint_as_float((w & (15u << (4 * k))) | 0x4B000000u),
                                        __uint_as_float((w & (15u << (4 * k + 4))) | 0x4B000000u));
        const uint64_t code = f2_fma(biased, f2_pack(s0, s1), f2_pack(-8388608.f * s0, -8388608.f * s1));
        f2_unpack(f2_fma(code, st2, mn2), x[j], x[j + 1]);
      }
      Vec8<T>::store(out + tok * kv * D, x);
    }
    t += U * sub_tokens;
  }
}

template <int D, typename T>
int load_launch_typed(const uint8_t* cache, int64_t num_slots, const int64_t* slot_mapping, int64_t tokens, int kv,
                      void* key, void* value, int32_t* err, cudaStream_t st) {
  const int64_t all = (int64_t)kv * (D / 4);  // pieces of a token
  const int places = (int)std::min<int64_t>(all, kLoadThreads);
  const int sub_tokens = kLoadThreads / places;
  const int64_t parts = (all + kLoadThreads - 1) / kLoadThreads;
  const int64_t per_step = (int64_t)sub_tokens * kLoadUnroll, all_steps = (tokens + per_step - 1) / per_step;
  // several steps per block once every SM has its 6 blocks of a step each
  const int64_t steps = std::max<int64_t>(1, std::min<int64_t>(8, all_steps * parts / (148 * 6)));
  const int64_t blocks = (all_steps + steps - 1) / steps;
  if (blocks > INT32_MAX || parts > 65535) return SLMT_ERR_UNSUPPORTED;
  load_kernel<D, T><<<dim3((unsigned)blocks, (unsigned)parts), kLoadThreads, 0, st>>>(
      cache, num_slots, slot_mapping, tokens, kv, places, sub_tokens, (int)steps, (T*)key, (T*)value, err);
  return launch_status();
}

template <int D>
int load_launch(const uint8_t* cache, int64_t num_slots, const int64_t* slot_mapping, int64_t tokens, int kv,
                void* key, void* value, int dtype, int32_t* err, cudaStream_t st) {
  if (dtype == SLMT_DTYPE_F16)
    return load_launch_typed<D, __half>(cache, num_slots, slot_mapping, tokens, kv, key, value, err, st);
  if (dtype == SLMT_DTYPE_BF16)
    return load_launch_typed<D, __nv_bfloat16>(cache, num_slots, slot_mapping, tokens, kv, key, value, err, st);
  return load_launch_typed<D, float>(cache, num_slots, slot_mapping, tokens, kv, key, value, err, st);
}

}  // namespace
}  // namespace slmt

using namespace slmt;

extern "C" int slmt_page_plan(const int32_t* query_start_loc, const int32_t* seq_lens, int64_t num_reqs,
                              int32_t* block_tables, int64_t bt_seq_stride, int64_t max_blocks_per_seq,
                              int64_t block_size, const int32_t* free_blocks, int64_t num_free,
                              const int32_t* free_cursor, int64_t num_tokens, int64_t* slot_mapping,
                              int64_t* positions, int32_t* cursor_out, int32_t* err_flag, void* stream) {
  if (num_reqs < 0 || num_tokens < 0 || max_blocks_per_seq < 0 || block_size <= 0 || num_free < 0)
    return SLMT_ERR_SHAPE;
  if (num_reqs > 1 && bt_seq_stride < max_blocks_per_seq) return SLMT_ERR_SHAPE;
  // positions, token and page numbers are 32-bit in the kernel
  if (num_tokens > INT32_MAX / 2 || num_reqs > INT32_MAX / 2 || num_free > INT32_MAX || block_size > INT32_MAX / 2 ||
      max_blocks_per_seq > INT32_MAX / 2)
    return SLMT_ERR_SHAPE;
  if (num_reqs > 0 && (!query_start_loc || !seq_lens || (!block_tables && max_blocks_per_seq > 0)))
    return SLMT_ERR_NULL;
  if (num_tokens > 0 && (!slot_mapping || !positions)) return SLMT_ERR_NULL;
  if (cursor_out && cursor_out == free_cursor) return SLMT_ERR_SHAPE;  // every CTA reads one, CTA 0 writes the other
  if (ranges_overlap(slot_mapping, 8 * num_tokens, positions, 8 * num_tokens)) return SLMT_ERR_SHAPE;
  if (num_tokens == 0 && !cursor_out) return SLMT_OK;
  PlanParams p;
  p.qsl = query_start_loc;
  p.seq_lens = seq_lens;
  p.tables = block_tables;
  p.table_stride = bt_seq_stride;
  p.free_blocks = free_blocks;
  p.num_free = free_blocks ? num_free : 0;
  p.cursor_in = free_cursor;
  p.slots = slot_mapping;
  p.positions = positions;
  p.cursor_out = cursor_out;
  p.err = err_flag;
  p.num_reqs = (int)num_reqs;
  p.num_tokens = (int)num_tokens;
  p.block_size = (int)block_size;
  p.shift = (block_size & (block_size - 1)) == 0 ? __builtin_ctzll((unsigned long long)block_size) : -1;
  p.max_blocks = (int)max_blocks_per_seq;
  const int64_t grid = std::max<int64_t>(1, (num_tokens + kPlanTokens - 1) / kPlanTokens);
  page_plan_kernel<<<(unsigned)grid, kPlanThreads, 0, reinterpret_cast<cudaStream_t>(stream)>>>(p);
  return launch_status();
}

extern "C" int slmt_kv_dequantize_load(const uint8_t* kv_cache, int64_t num_blocks, int64_t block_size,
                                       int64_t num_kv_heads, int64_t head_dim, const int64_t* slot_mapping,
                                       int64_t num_tokens, void* key, void* value, int out_dtype, int32_t* err_flag,
                                       void* stream) {
  if (!valid_head_dim(head_dim)) return SLMT_ERR_HEAD_DIM;
  if (num_tokens < 0 || num_kv_heads <= 0 || num_kv_heads > INT32_MAX / 2 || num_blocks < 0 || block_size <= 0)
    return SLMT_ERR_SHAPE;
  if (out_dtype != SLMT_DTYPE_F32 && out_dtype != SLMT_DTYPE_F16 && out_dtype != SLMT_DTYPE_BF16)
    return SLMT_ERR_DTYPE;
  if (num_tokens == 0) return SLMT_OK;
  if (!kv_cache || !slot_mapping || !key || !value) return SLMT_ERR_NULL;
  // 4-byte code words and ruler pairs in, 16-byte pieces out
  if (reinterpret_cast<uintptr_t>(kv_cache) % 8 != 0 || reinterpret_cast<uintptr_t>(key) % 16 != 0 ||
      reinterpret_cast<uintptr_t>(value) % 16 != 0)
    return SLMT_ERR_ALIGN;
  const int64_t slots = num_blocks * block_size;
  const int64_t out_bytes = num_tokens * num_kv_heads * head_dim * (out_dtype == SLMT_DTYPE_F32 ? 4 : 2);
  const int64_t cache_bytes = slots * num_kv_heads * (head_dim + 8);
  if (ranges_overlap(key, out_bytes, value, out_bytes) || ranges_overlap(key, out_bytes, kv_cache, cache_bytes) ||
      ranges_overlap(value, out_bytes, kv_cache, cache_bytes))
    return SLMT_ERR_SHAPE;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int kv = (int)num_kv_heads;
  switch (head_dim) {
    case 64:
      return load_launch<64>(kv_cache, slots, slot_mapping, num_tokens, kv, key, value, out_dtype, err_flag, st);
    case 80:
      return load_launch<80>(kv_cache, slots, slot_mapping, num_tokens, kv, key, value, out_dtype, err_flag, st);
    default:
      return load_launch<128>(kv_cache, slots, slot_mapping, num_tokens, kv, key, value, out_dtype, err_flag, st);
  }
}
