// prompt.cu -- causal attention of packed prompts over their own K and V
// (sm_100a): o_i = sum_{j <= i} softmax_j(scale q_i k_j) v_j within each
// request, grouped heads.
//
// One persistent CTA per SM, tiles of 128 query rows by 128 keys.  The rows of
// a tile are (token, query head of one kv head's group), token by token, so a
// group shares its K and V tiles and a prompt of a few tokens still fills
// rows.  A work item is two such tiles of consecutive tokens (A and B) of one
// request and kv head.
//
//   S = Q K^T   tcgen05.mma, both operands in shared memory, S in TMEM
//   P = exp2((S - m) scale log2 e)   rounded to the inputs' type, over S in TMEM
//   O += P V    tcgen05.mma, P from TMEM, V in shared memory as it was copied
//
// Warps 0-3 and 4-7 are the softmax of tile A and of tile B, a row per thread;
// while one of them works on its scores, the tensor core computes the other
// tile's products.  Warp 8 issues the products, warp 9 the tiled copies into
// a ring of K and V tiles, warps 10 and 11 look at the V tiles on the
// diagonal (below).  Warp 9 also walks the list of items and hands them to the
// other roles through a ring.
//
// What bounds it, per step of 256 rows by 128 keys at D 128 (cycles of an SM):
// the products need 4 * 512, the exponentials 2 * 1024 of the 16-a-clock unit;
// a tile's softmax (1950) and its products (950 with their signals) take turns,
// so a step takes about 2900.  Long prompts run into the power cap before that
// counts: one of 16384 tokens (32/8 heads, bf16) takes 1.72 ms, 1280 TFLOP/s,
// in a short run and about 2.0 ms, 1100 TFLOP/s, with the clock held at 1.7
// GHz.  Short ones are bound by their chain: products, softmax, products,
// output (a prompt of 130 tokens beside three shorter ones: 9.5 us).
// Measured and dropped, in turn on one GPU: scores of 64 keys at a time into
// alternating halves (the softmax then never waits, but S costs 768 cycles in
// place of 512 and its products change accumulators twice as often), one
// product warp per tile (products into different accumulators interleave), two
// warps to a row, and a part of the exponentials by a polynomial on the FMA
// pipe (12 instructions in place of 2): 2.0-2.4 ms, 2.2-2.4 ms, 2.2 ms and
// 1.93 against 1.95 ms.
//
// A tile's first scores of the next item go out behind its own last products,
// before the other tile's: what it does then falls beside the other's end, and
// the two do not run into the next item in step.  An item's output is written
// behind the next one's first weights; at D 64 tensor memory has room for two
// accumulators per tile, so those weights need not wait for it (48 prompts of
// 5 to 393 tokens, 32/4 heads: 42 us; with one accumulator and the tiles
// starting together 3.4 more).
//
// P is held in the inputs' 16 bits because the tensor core takes both operands
// of a product in one type; each weight is off by half a step of it (bf16 2^-8,
// fp16 2^-11, relative), the output's error as a norm goes from 0.0016 to
// 0.0022 (bf16) and from 0.0002 to 0.00025 (fp16).
//
// Running maximum: the reference m of a row moves only when a score passes it
// by more than 2^8 in weight; until then old weights stay on their scale, and
// O is rescaled in TMEM only then.  Sums are fp32, of the unrounded weights.
//
// What is not attended to is not seen: hidden scores are replaced, not added
// to.  For V that is not enough -- a hidden key's weight is 0, but 0 times a
// NaN or an infinity is a NaN -- so V tiles with a hidden key are searched for
// such values; where there are some they are taken out of the tile, and added
// to the rows that do attend to them at the end, read from global memory.
#include <atomic>
#include <type_traits>

#include "internal.h"
#include "tcgen05.cuh"

namespace slmt {

namespace {

// mbar_wait in fewer instructions.  The roles' code between two items runs once
// and has left the instruction cache when it is needed again, so short items
// pay for its length: with mbar_wait at every wait, the items walked by every
// role, and the copies and products written out at each of their places, 1000
// short requests took 132 us instead of 105, 48 of 5 to 393 tokens 44.8 instead
// of 41.8.
__device__ __forceinline__ bool wait_short(uint64_t* bar, uint32_t parity, uint64_t limit_ns) {
  uint64_t t0 = 0;
#pragma unroll 1
  while (!mbar_try_wait(bar, parity)) {
    const uint64_t now = global_timer_ns();
    if (t0 == 0) t0 = now;
    if (now - t0 > limit_ns) return false;
  }
  return true;
}

constexpr int kThreads = 384;
constexpr int kMaxReqs = 1024;    // requests of one launch (sorted in shared memory)
constexpr int kReqBits = 10;
constexpr uint32_t kTmemCols = 512;
constexpr int kMaxStages = 6;
constexpr int kItems = 8;          // ring of work items

struct PromptParams {
  const void* v;
  void* out;
  const int32_t* qsl;
  const int32_t* seq_lens;
  int32_t* err;
  int64_t v_tok, v_head, o_tok, o_head;
  uint64_t wait_limit_ns;
  float scale_log2;
  bool out_wide;  // every output row starts on 32 bytes
  int num_tokens, num_reqs, max_query, kv, group, tile_tokens, out_dtype, stall;
  uint32_t kv_recip;  // 2^32 / kv, rounded up
};

// One work item, as every role sees it.
struct Item {
  int head;          // kv head
  int start, rows;   // the request's first row and its number of rows
  int tok[2];        // first token of tile A and of tile B
  int steps[2];      // 64-key steps of each (0: no rows in the tile)
  int nk;            // 128-key tiles loaded (0: no more items)
  int guard;         // first of these that some row of A or B does not see whole
};

struct PromptCtl {
  uint64_t q_full[2], q_empty[2], o_full[2][2], drain, never;  // o_full: [tile][accumulator]
  uint64_t s_full[2], p_ready[2][2];  // [tile], [tile][first or second 64 keys]
  uint64_t kv_full[kMaxStages], kv_empty[kMaxStages], v_ok[kMaxStages];
  uint64_t item_full[kItems], item_empty[kItems];
  uint32_t tmem;
  uint32_t tile_bad[2][2];
  uint32_t slot_bad[kMaxStages][2];
  alignas(16) uint32_t sort_key[kMaxReqs];  // (pairs of tiles << kReqBits) | request, descending
  int start[kMaxReqs], rows[kMaxReqs];
  Item items[kItems];
};

template <int D>
struct PromptGeom {
  static constexpr int PANELS = (D + 63) / 64;        // 128-byte wide panels of a tile
  static constexpr int TILE = PANELS * 128 * 128;     // bytes
  static constexpr int STAGES = D == 64 ? 6 : 4;      // K and V take turns: an even number
  static constexpr int OUTS = D == 64 ? 2 : 1;        // accumulators of a tile: what tensor memory has room for
  static constexpr int SMEM = 1024 + (2 + STAGES) * TILE + (int)sizeof(PromptCtl);
  static_assert(SMEM <= 227 * 1024 && STAGES % 2 == 0 && STAGES <= kMaxStages, "");
};

// The items in the order of falling cost -- requests' last tiles first -- dealt
// to the CTAs in rows, each row in the direction that gives its longer items to
// the end with the smaller sum so far (1999 + 777 + 63 tokens of 32 heads, D 80:
// 50.4 us; back and forth in turn 54.5, the longest CTA has 24 steps instead of
// 22).  Level t holds the items of tile pair t of every request that has one:
// those are the first `count` of the requests sorted by length.
// A whole warp walks together.
struct Walk {
  int row, level, count, base;  // deal, tile pair, requests of the level, items before it
  int longest;                  // pairs of the longest request that is not among them
  int first, lead;              // cost of the row's first item; first CTA's sum less the last one's
  int back;                     // -1: the row runs from the last CTA to the first, else 0
  __device__ __forceinline__ void begin(const PromptCtl* c) {
    row = 0, count = 0, base = 0, lead = 0, back = 0;
    level = longest = (int)(c->sort_key[0] >> kReqBits);
    first = level - 1;
  }
  __device__ __forceinline__ bool next(const PromptCtl* c, const PromptParams& p, Item& it) {
    const int nc = gridDim.x, me = blockIdx.x;
    int at = row == 0 ? me : row * nc;
#pragma unroll 1
    for (int pass = row == 0;; ++pass) {  // to the row's first item, then to this CTA's
      int in_level = count * p.kv;
      while (at - base >= in_level) {
        base += in_level;
        if (--level < 0) return false;
        while (longest > level) {  // requests join: 32 looked at together
          const int i = count + (int)(threadIdx.x & 31);
          const int pairs = i < p.num_reqs ? (int)(c->sort_key[i] >> kReqBits) : 0;
          const uint32_t in = __ballot_sync(0xffffffffu, pairs > level);
          count += __popc(in);
          longest = in == 0xffffffffu ? (count < p.num_reqs ? (int)(c->sort_key[count] >> kReqBits) : 0)
                                      : __shfl_sync(0xffffffffu, pairs, __ffs(~in) - 1);
        }
        in_level = count * p.kv;
      }
      if (pass) break;
      // an item costs about its last key, in tile pairs; the last item of a row
      // costs about what the first of the next does
      lead += ((first - level) ^ back) - back;
      first = level;
      back = lead > 0 ? -1 : 0;
      at += back ? nc - 1 - me : me;
    }
    ++row;
    // rem / kv by 2^32 / kv rounded up (which kv 1 has no room for): at most one too large
    const int rem = at - base;
    int rank = p.kv == 1 ? rem : (int)__umulhi((uint32_t)rem, p.kv_recip);
    it.head = rem - rank * p.kv;
    if (it.head < 0) --rank, it.head += p.kv;
    const int req = (int)(c->sort_key[rank] & ((1u << kReqBits) - 1));
    it.start = c->start[req];
    it.rows = c->rows[req];
    const int lo = level * 2 * p.tile_tokens, hi = lo + p.tile_tokens;
    const int steps_lo = (min(hi, it.rows) + 63) >> 6;
    const int steps_hi = hi < it.rows ? (min(hi + p.tile_tokens, it.rows) + 63) >> 6 : 0;
    const bool turn = (row & 1) == 0;  // A and B take the longer tile in turn, and the only one
    it.tok[0] = turn ? hi : lo, it.tok[1] = turn ? lo : hi;
    it.steps[0] = turn ? steps_hi : steps_lo, it.steps[1] = turn ? steps_lo : steps_hi;
    it.nk = (max(steps_lo, steps_hi) + 1) >> 1;
    it.guard = (lo + 1) >> 7;
    return true;
  }
};

template <bool BF16>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  if constexpr (BF16) {
    __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&h);
  } else {
    return pack_half2(lo, hi);
  }
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
template <bool BF16>
__device__ __forceinline__ uint4 pack8(const float* x) {
  return make_uint4(pack16<BF16>(x[0], x[1]), pack16<BF16>(x[2], x[3]), pack16<BF16>(x[4], x[5]),
                    pack16<BF16>(x[6], x[7]));
}

template <int D, bool BF16>
__global__ void __launch_bounds__(kThreads, 1)
    prompt_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                  const __grid_constant__ CUtensorMap map_v, const PromptParams p) {
  using G = PromptGeom<D>;
  constexpr int TILE = G::TILE, STAGES = G::STAGES, PANELS = G::PANELS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  PromptCtl* c = reinterpret_cast<PromptCtl*>(smem + (2 + STAGES) * TILE);
  uint8_t* ring = smem + 2 * TILE;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint64_t limit = p.wait_limit_ns;
  const uint64_t drain_limit = max(limit, (uint64_t)1000000000);  // of the last waits, for what is in flight

  // ---- set-up: barriers, tensor memory, the requests sorted by length
  if (tid == 0) {
    for (int x = 0; x < 2; ++x) {
      mbar_init(&c->q_full[x], 1), mbar_init(&c->q_empty[x], 1);
      mbar_init(&c->s_full[x], 1);
      for (int h = 0; h < 2; ++h) mbar_init(&c->p_ready[x][h], 128);
      for (int o = 0; o < 2; ++o) mbar_init(&c->o_full[x][o], 2);  // the commit, and the thread that set tile_bad
    }
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&c->kv_full[s], 1);
      mbar_init(&c->kv_empty[s], s & 1 ? 3 : 1);  // the products; V tiles: and both guard warps
      mbar_init(&c->v_ok[s], 2);
    }
    for (int i = 0; i < kItems; ++i) {
      mbar_init(&c->item_full[i], 1);
      mbar_init(&c->item_empty[i], 11);  // the warps but the one that makes them
    }
    mbar_init(&c->drain, 1), mbar_init(&c->never, 1);
    fence_mbar_init();
  }
  if (warp == 8) tmem_alloc(&c->tmem, kTmemCols);
  if (tid == 32 * 9) prefetch_map(&map_q), prefetch_map(&map_k), prefetch_map(&map_v);
  constexpr int COUNTED = 256;  // requests ranked by counting, more are sorted
  int padded = (p.num_reqs + 3) & ~3;
  if (padded > COUNTED) padded = kMaxReqs;
  unsigned bad_len = 0u;
  for (int r = tid; r < padded; r += kThreads) {
    int n = 0, a = 0;
    if (r < p.num_reqs) {
      const int qa = p.qsl[r], qb = p.qsl[r + 1];
      if (!(p.seq_lens && p.seq_lens[r] != qb - qa)) {
        a = max(qa, 0);
        n = max(min(qb, p.num_tokens) - a, 0);
        if (qa < 0 || qb < qa || qb > p.num_tokens || n > p.max_query) bad_len = SLMT_DEVERR_SEQ_LEN;
        n = min(n, p.max_query);
      }
      c->start[r] = a;
      c->rows[r] = n;
    }
    const int pairs = (n + 2 * p.tile_tokens - 1) / (2 * p.tile_tokens);
    c->sort_key[r] = ((uint32_t)pairs << kReqBits) | (uint32_t)r;
  }
  if (bad_len && blockIdx.x == 0 && p.err) atomicOr(reinterpret_cast<unsigned int*>(p.err), bad_len);
  __syncthreads();
  if (padded <= COUNTED) {
    // A thread counts the keys above its own (all differ).  200 requests are
    // 1.7 us sooner this way than sorted, 500 are 2 us later.
    static_assert(COUNTED <= kThreads, "");
    const uint32_t own = tid < padded ? c->sort_key[tid] : 0u;
    int rank = 0;
#pragma unroll 4
    for (int r = 0; r < padded; r += 4) {
      const uint4 k = *reinterpret_cast<const uint4*>(c->sort_key + r);
      rank += (k.x > own) + (k.y > own) + (k.z > own) + (k.w > own);
    }
    __syncthreads();
    if (tid < padded) c->sort_key[rank] = own;
  } else {
    // Bitonic, four keys to a thread of the first eight warps: of the 55 passes
    // 6 go through shared memory, the others stay within a warp or a thread.
    static_assert(kMaxReqs == 8 * 128, "");
    uint4* keys = reinterpret_cast<uint4*>(c->sort_key);
    const bool mine = warp < 8;
    const int e = 4 * tid;  // of the first of them
    uint32_t v[4] = {};
    if (mine) {
      const uint4 x = keys[tid];
      v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
    }
    auto keep = [&](uint32_t& a, uint32_t other, bool larger) { a = larger ? max(a, other) : min(a, other); };
    for (int k = 2; k <= kMaxReqs; k <<= 1) {
      const bool falling = (e & k) == 0;
      int j = k >> 1;
      for (; j >= 128; j >>= 1) {
        if (mine) keys[tid] = make_uint4(v[0], v[1], v[2], v[3]);
        __syncthreads();
        if (mine) {
          const uint4 y = keys[tid ^ (j >> 2)];
          const bool larger = ((e & j) == 0) == falling;
          keep(v[0], y.x, larger), keep(v[1], y.y, larger), keep(v[2], y.z, larger), keep(v[3], y.w, larger);
        }
        __syncthreads();
      }
      for (; j >= 4; j >>= 1) {
        const bool larger = ((e & j) == 0) == falling;
#pragma unroll
        for (int i = 0; i < 4; ++i) keep(v[i], __shfl_xor_sync(0xffffffffu, v[i], j >> 2), larger);
      }
      auto order = [&](uint32_t& a, uint32_t& b, bool fall) {
        const uint32_t hi = max(a, b), lo = min(a, b);
        a = fall ? hi : lo, b = fall ? lo : hi;
      };
      if (j == 2) order(v[0], v[2], falling), order(v[1], v[3], falling);
      order(v[0], v[1], k == 2 ? true : falling), order(v[2], v[3], k == 2 ? false : falling);
    }
    if (mine) keys[tid] = make_uint4(v[0], v[1], v[2], v[3]);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = c->tmem;
  // columns: S of A and B (128 each; P takes the first 64 of each), O of A and B
  const uint32_t col_s = 0, col_o = 256;

  bool failed = false;
  // the next item, for a warp that takes all of them in their order
  uint32_t item_at = 0;
  auto next_item = [&](Item& it) {
    const uint32_t s = item_at % kItems;
    if (!__all_sync(0xffffffffu, wait_short(&c->item_full[s], (item_at / kItems) & 1u, limit))) {
      failed = true;
      return false;
    }
    it = c->items[s];
    ++item_at;
    __syncwarp();
    if (lane == 0) mbar_arrive(&c->item_empty[s]);
    return it.nk != 0;
  };
  if (warp >= 8) {
    regs_lower<88>();
    if (warp == 9) {
      // ------------------------------------------------------------ copies
      {
        const bool leader = elect_one();
        uint32_t fill = 0, queries = 0;  // bit x: parity of tile x's copies, bit 2 + x: whether there was one
        // a tile of the ring or of the queries, once it is free; false: nothing is under way
        auto load = [&](const CUtensorMap* map, uint64_t* empty, uint32_t phase, uint64_t* full, uint32_t bytes,
                        uint8_t* to, int head, int row) {
          if (!__all_sync(0xffffffffu, wait_short(empty, (phase & 1u) ^ 1u, limit))) {
            failed = true;
          } else if (leader) {
            mbar_arrive_expect_tx(full, bytes);
            for (int d = 0; d < PANELS; ++d) tma_load_3d(to + d * 16384, map, d * 64, head, row, full);
          }
          return !failed;
        };
        // The products look one item ahead: the next one is made known behind
        // this one's first keys, queries and values.
        Walk w;
        Item it, nxt;
        uint32_t at = 0;
        int i = 2;
        it.nk = 0;
        w.begin(c);
        while (!failed) {
          if (i == 2) {
            if (!w.next(c, p, nxt)) nxt.nk = 0;
            const uint32_t s = at % kItems;
            if (!__all_sync(0xffffffffu, wait_short(&c->item_empty[s], ((at / kItems) & 1u) ^ 1u, limit))) {
              failed = true;
            } else if (leader) {
              c->items[s] = nxt;
              mbar_arrive(&c->item_full[s]);
            }
            ++at;
          }
          if (i >= 2 * it.nk) {
            if (nxt.nk == 0) break;
            it = nxt, i = 0;
          }
          const uint32_t s = fill % STAGES;  // K and V in turn
          if (failed || !load(i & 1 ? &map_v : &map_k, &c->kv_empty[s], fill / STAGES, &c->kv_full[s], TILE,
                              ring + s * TILE, it.head, it.start + 64 * (i & ~1)))
            break;
          ++fill;
          if (i++ == 0) {
#pragma unroll 1
            for (int x = 0; x < 2; ++x)
              if (!failed && (x ? it.steps[1] : it.steps[0]) &&
                  load(&map_q, &c->q_empty[x], queries >> x, &c->q_full[x],
                       (uint32_t)(PANELS * 128 * p.tile_tokens * p.group), smem + x * TILE, it.head * p.group,
                       it.start + (x ? it.tok[1] : it.tok[0])))
                queries = (queries ^ (1u << x)) | (4u << x);
          }
        }
        // no copy is in flight when this warp is done, whatever happened
        for (uint32_t f = fill > (uint32_t)STAGES ? fill - STAGES : 0; f < fill; ++f)
          if (!wait_short(&c->kv_full[f % STAGES], (f / STAGES) & 1u, drain_limit)) failed = true;
        for (int x = 0; x < 2; ++x)
          if ((queries >> (2 + x) & 1u) && !wait_short(&c->q_full[x], (queries >> x & 1u) ^ 1u, drain_limit)) failed = true;
      }
    } else if (warp == 8) {
      // ----------------------------------------------------------- products
      // The whole warp walks and waits, so that what the products need is the
      // same in every lane and stays in uniform registers; one lane issues.
      constexpr uint32_t idesc_s = mma_idesc(BF16, 128, 128, false), idesc_s64 = mma_idesc(BF16, 128, 64, false),
                         idesc_o = mma_idesc(BF16, 128, D, true);
      constexpr uint32_t HI = desc_hi(1024);
      const bool leader = elect_one();
      const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
      const uint32_t q_lo = desc_lo(smem_addr(smem), 16), k_lo = desc_lo(smem_addr(ring), 16),
                     v_lo = desc_lo(smem_addr(ring), 16384);
      // bit x: tile x's phases of its queries and weights, its accumulator
      uint32_t fill = 0, q_phase = 0, p_phase = 0, out = 0, ok_phase = 0;
      auto wait = [&](uint64_t* bar, uint32_t phase) {
        const bool ok = __all_sync(0xffffffffu, wait_short(bar, phase & 1u, limit));
        failed |= !ok;
        return ok;
      };
      auto full = [&](uint32_t f) { return wait(&c->kv_full[f % STAGES], f / STAGES); };
      auto release = [&](uint32_t f) {  // once the products issued so far are done
        if (leader) mma_commit(&c->kv_empty[f % STAGES]);
      };
      // scores of tile x with the keys of fill f, or the first 64 of them
      auto scores = [&](int x, uint32_t f, bool two, bool last) {
        const uint32_t a = q_lo + x * (TILE >> 4), b = k_lo + (f % STAGES) * (TILE >> 4);
        const uint32_t idesc = two ? idesc_s : idesc_s64;
        if (leader) {
#pragma unroll
          for (int u = 0; u < D / 16; ++u) {
            const uint32_t off = ((u >> 2) * 16384 + (u & 3) * 32) >> 4;
            mma_ss(tm + col_s + 128 * x, a + off, HI, b + off, HI, idesc, u > 0);
          }
          mma_commit(&c->s_full[x]);
          if (last) mma_commit(&c->q_empty[x]);
        }
      };
      // half the keys at a time: the first half's weights are there while the
      // second half's are still being computed
      auto weigh = [&](int x, int h, uint32_t f, bool first) {
        const uint32_t b = v_lo + (f % STAGES) * (TILE >> 4) + h * (8192 >> 4);
        const uint32_t d = tm + col_o + D * (G::OUTS * x + (out >> x & 1u));
        if (leader) {
#pragma unroll
          for (int u = 0; u < 4; ++u)
            mma_ts(d, tm + col_s + 128 * x + 32 * h + 8 * u, b + u * (2048 >> 4), HI, idesc_o, u > 0 || !first);
        }
      };
      struct Next {
        int steps[2], nk, guard;
      };
      auto fetch = [&](Next& n) {
        Item it;
        const bool more = next_item(it);
        n.steps[0] = __shfl_sync(0xffffffffu, more ? it.steps[0] : 0, 0);
        n.steps[1] = __shfl_sync(0xffffffffu, more ? it.steps[1] : 0, 0);
        n.nk = __shfl_sync(0xffffffffu, more ? it.nk : 0, 0);
        n.guard = __shfl_sync(0xffffffffu, more ? it.guard : 0, 0);
      };
      // Half the code, with the tiles and halves as loops, is 2 us less for the
      // ragged batch above and up to 10% more for long prompts: where a tile's
      // operands lie is then worked out at every product.
      Next cur = {}, nxt;
      do {
        fetch(nxt);
        const uint32_t next_fill = fill + 2 * cur.nk;
        uint32_t bad = 0, begun = 0;  // bit x: tile x, with the next item
#pragma unroll 1
        for (int j = 0; j <= cur.nk && !failed; ++j) {  // the last pass begins what has not begun
          const uint32_t fv = fill + 2 * j + 1, fk = fv + 1;
          const bool more_keys = j + 1 < cur.nk;
          if (j < cur.nk) {
            if (j >= cur.guard) {  // looked at: there, too
              const uint32_t s = fv % STAGES;
              if (!wait(&c->v_ok[s], ok_phase >> s)) break;
              ok_phase ^= 1u << s;
              bad |= c->slot_bad[s][0] | c->slot_bad[s][1];
            } else if (!full(fv)) {
              break;
            }
            if (more_keys && !full(fk)) break;
          }
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const int next_steps = nxt.steps[x];
            int left = cur.steps[x] - 2 * j - 2;
            uint32_t keys = fk;
            if (left > -2) {
              if (wait(&c->p_ready[x][0], p_phase >> x)) {
                tc_fence_after();
                weigh(x, 0, fv, j == 0);
              }
              if (left > -1 && !failed && wait(&c->p_ready[x][1], p_phase >> x)) {
                tc_fence_after();
                weigh(x, 1, fv, false);
              }
              if (failed) break;
              p_phase ^= 1u << x;
              if (left <= 0) {
                const uint32_t o = G::OUTS == 2 ? out >> x & 1u : 0u;
                if (leader) {
                  c->tile_bad[x][o] = bad;
                  mbar_arrive(&c->o_full[x][o]);
                  mma_commit(&c->o_full[x][o]);
                }
                if (G::OUTS == 2) out ^= 1u << x;
              }
            }
            if (left <= 0) {
              // The next item's first scores, if they can go out without a wait
              // or nothing is left to do here.  (The queries are asked for behind
              // the keys: once they are there, the keys' barrier is in the phase
              // that is looked at.)
              if (next_steps == 0 || (begun >> x & 1u)) continue;
              if (j < cur.nk) {
                if (!__all_sync(0xffffffffu, mbar_test(&c->q_full[x], q_phase >> x & 1u)) ||
                    !__all_sync(0xffffffffu, mbar_test(&c->kv_full[next_fill % STAGES], (next_fill / STAGES) & 1u)))
                  continue;
              } else if (!wait(&c->q_full[x], q_phase >> x) || !full(next_fill)) {
                break;
              }
              tc_fence_after();
              q_phase ^= 1u << x;
              begun |= 1u << x;
              keys = next_fill, left = next_steps;
            }
            scores(x, keys, left > 1, left <= 2);
          }
          if (failed) break;
          if (j < cur.nk) release(fv);
          if (more_keys) release(fk);
        }
        if (nxt.nk && !failed) release(next_fill);
        fill = next_fill;
        cur = nxt;
      } while (!failed && cur.nk);
      // products in flight read shared and tensor memory
      if (leader) mma_commit(&c->drain);
      if (!wait_short(&c->drain, 0, drain_limit)) failed = true;
    } else {
      // ------------------------------------------- non-finite values in V
      constexpr uint32_t EXP = BF16 ? 0x7F80u : 0x7C00u;
      const int half = warp - 10;
      uint32_t fill = 0;
      Item it;
      while (!failed && next_item(it)) {
        for (int j = 0; j < it.nk; ++j) {
          const uint32_t f = fill + 2 * j + 1, s = f % STAGES;
          if (!__all_sync(0xffffffffu, wait_short(&c->kv_full[s], (f / STAGES) & 1u, limit))) {
            failed = true;
            break;
          }
          if (j >= it.guard) {
            uint4* tile = reinterpret_cast<uint4*>(ring + s * TILE + half * (TILE / 2));
            uint32_t top = 0;
#pragma unroll 8
            for (int i = lane; i < TILE / 32; i += 32) {
              const uint4 x = tile[i];
              top = __vmaxu2(top, x.x & 0x7FFF7FFFu);
              top = __vmaxu2(top, x.y & 0x7FFF7FFFu);
              top = __vmaxu2(top, x.z & 0x7FFF7FFFu);
              top = __vmaxu2(top, x.w & 0x7FFF7FFFu);
            }
            const bool found = __any_sync(0xffffffffu, (top & 0xFFFFu) >= EXP || (top >> 16) >= EXP);
            if (found) {
              uint16_t* v = reinterpret_cast<uint16_t*>(tile);
              for (int i = lane; i < TILE / 4; i += 32)
                if ((v[i] & EXP) == EXP) v[i] = 0;
              fence_proxy_async_shared();  // before the tensor core reads them
            }
            __syncwarp();
            if (lane == 0) {
              c->slot_bad[s][half] = found;
              mbar_arrive(&c->v_ok[s]);
            }
          }
          if (lane == 0) mbar_arrive(&c->kv_empty[s]);
        }
        fill += 2 * it.nk;
      }
    }
  } else {
    // ---------------------------------------------------------------- softmax
    regs_raise<208>();
    constexpr float SHIFT = BF16 ? 0.f : 6.f;  // fp16 weights lie in [2^-24, 2^14]: a row's largest is 2^6 or more
    constexpr float MOVE = 8.f;
    constexpr int OUT = D == 80 ? 80 : 32;                    // output columns at a time
    const int x = warp >> 2, row = tid & 127;
    const int row_tok = row / p.group, row_head = row - row_tok * p.group;
    const uint32_t lane_base = (uint32_t)(warp & 3) << 21;
    const uint32_t ts = tmem + lane_base + col_s + 128 * x, outs = tmem + lane_base + col_o + D * G::OUTS * x;
    uint32_t to = outs;  // the accumulator of the item at hand
    const float sc = p.scale_log2;
    uint32_t ns = 0, no = 0;
    // A finished item's output is written after the next item's first weights
    // are computed: the wait for the item's last product is then over.  With two
    // accumulators the weights are announced before it, with one after it (that
    // product overwrites O).
    struct Pending {
      int64_t at;
      float sum;
      int start, head, tok, guard;
      bool any, valid;
    } last;
    last.any = false;
    auto finish = [&] {
      last.any = false;
      const uint32_t buf = no % G::OUTS, from = outs + D * buf;
      if (!__all_sync(0xffffffffu, wait_short(&c->o_full[x][buf], (no++ / G::OUTS) & 1u, limit))) {
        failed = true;
        return;
      }
      tc_fence_after();
      const float inv = 1.f / last.sum;
      const bool bad = c->tile_bad[x][buf] != 0;
      // A thread writes its own row, a 32-byte sector at a time.  Turning the
      // rows in shared memory first, so that a warp's store covers whole lines,
      // cost more than the lines do (1000 short requests 169 us for 155, 48 of
      // 5 to 393 tokens 48.8 for 48.0).
#pragma unroll 1
      for (int i = 0; i < D; i += OUT) {
        float o[OUT];
        __syncwarp();
#pragma unroll
        for (int k = 0; k < OUT; k += 16) tmem_ld16(o + k, from + i + k);
        tmem_wait_ld();
        if (!last.valid) continue;
        if (bad) {
          // the values taken out of the V tiles, for the rows that attend to them
          for (int j = 128 * last.guard; j <= last.tok; ++j) {
            const uint16_t* v = reinterpret_cast<const uint16_t*>(p.v) + (int64_t)(last.start + j) * p.v_tok +
                                (int64_t)last.head * p.v_head + i;
#pragma unroll
            for (int k = 0; k < OUT; ++k) {
              const float y = BF16 ? __bfloat162float(__ushort_as_bfloat16(v[k])) : __half2float(__ushort_as_half(v[k]));
              if (!(y - y == 0.f)) o[k] += y;
            }
          }
        }
#pragma unroll
        for (int k = 0; k < OUT; ++k) o[k] *= inv;
        auto put = [&](void* to, const uint4& lo, const uint4& hi) {
          if (p.out_wide) {
            st_global_256(to, lo, hi);
          } else {
            reinterpret_cast<uint4*>(to)[0] = lo;
            reinterpret_cast<uint4*>(to)[1] = hi;
          }
        };
        if (p.out_dtype == SLMT_DTYPE_F32) {
          float* to_row = reinterpret_cast<float*>(p.out) + last.at + i;
#pragma unroll
          for (int k = 0; k < OUT; k += 8) {
            const uint32_t* b = reinterpret_cast<const uint32_t*>(o + k);
            put(to_row + k, make_uint4(b[0], b[1], b[2], b[3]), make_uint4(b[4], b[5], b[6], b[7]));
          }
          continue;
        }
        uint16_t* to_row = reinterpret_cast<uint16_t*>(p.out) + last.at + i;
        if (p.out_dtype == SLMT_DTYPE_BF16) {
#pragma unroll
          for (int k = 0; k < OUT; k += 16) put(to_row + k, pack8<true>(o + k), pack8<true>(o + k + 8));
        } else {
#pragma unroll
          for (int k = 0; k < OUT; k += 16) put(to_row + k, pack8<false>(o + k), pack8<false>(o + k + 8));
        }
      }
    };
    // test hook: a wait that runs out
    if (p.stall && blockIdx.x == 0 && x == 0 && !__all_sync(0xffffffffu, wait_short(&c->never, 0, limit))) failed = true;
    int tok = 0, first_hidden = 0;
    float m = 0.f, sum = 0.f;
    // The softmax of one step over KEYS keys: 128, or 64 where the others are
    // hidden from all of the tile.  False if a wait ran out.
    auto step = [&](auto keys, int j) {
      constexpr int KEYS = decltype(keys)::value;
      if (!__all_sync(0xffffffffu, wait_short(&c->s_full[x], ns++ & 1u, limit))) return false;
      tc_fence_after();
      float s[KEYS];
#pragma unroll
      for (int k = 0; k < KEYS; k += 32) tmem_ld32(s + k, ts + k);
      tmem_wait_ld();
      if (j >= first_hidden) {
        const int seen = tok - 128 * j;  // columns 0..seen are attended to
#pragma unroll
        for (int k = 0; k < KEYS; k += 32) {
          const uint32_t word = seen >= k + 31 ? 0xFFFFFFFFu : seen < k ? 0u : (2u << (seen - k)) - 1u;
#pragma unroll
          for (int l = 0; l < 32; ++l) s[k + l] = word & (1u << l) ? s[k + l] : -INFINITY;
        }
      }
      float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
      for (int k = 4; k < KEYS - 4; k += 8) {
#pragma unroll
        for (int l = 0; l < 4; ++l) mx[l] = max3(mx[l], s[k + l], s[k + 4 + l]);
      }
#pragma unroll
      for (int l = 0; l < 4; ++l) mx[l] = fmaxf(mx[l], s[KEYS - 4 + l]);
      const float top = max3(m, max3(mx[0], mx[1], mx[2]), mx[3]);
      if (j == 0) {
        m = top;
      } else {
        const bool move = (top - m) * sc > MOVE;
        if (__any_sync(0xffffffffu, move)) {
          // products up to the last step's are done: this step's scores, issued after them, are
          const float f = move ? exp2_approx((m - top) * sc) : 1.f;
          if (move) m = top;
          sum *= f;
#pragma unroll 1
          for (int k = 0; k < D; k += 16) {
            float o[16];
            tmem_ld16(o, to + k);
            tmem_wait_ld();
#pragma unroll
            for (int l = 0; l < 16; ++l) o[l] *= f;
            tmem_st16(to + k, reinterpret_cast<uint32_t*>(o));
          }
        }
      }
      const float ref = m == -INFINITY ? 0.f : m;
      // exponents s * sc - ref * sc in one rounding: that of ref * sc is the
      // same for the whole row and cancels, as long as it stays below one
      float offset = fmaf(-ref, sc, SHIFT);
      const bool far = !(fabsf(ref * sc) < 0x1p20f);
      if (__any_sync(0xffffffffu, far)) {
        // for such a row the difference first: exact near the maximum, whatever
        // its size (the other rows keep their bits)
        const float base = far ? ref : 0.f;
#pragma unroll
        for (int k = 0; k < KEYS; ++k) s[k] -= base;
        if (far) offset = SHIFT;
      }
      const bool pending = j == 0 && last.any, hold = G::OUTS == 1 && pending;  // the last item's output
      const uint64_t scale2 = f2_pack(sc, sc), offset2 = f2_pack(offset, offset);
      uint64_t acc0 = f2_pack(0.f, 0.f), acc1 = acc0;
#pragma unroll
      for (int k0 = 0; k0 < KEYS / 2; k0 += 16) {
        uint32_t w16[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          float lo, hi;
          f2_unpack(f2_fma(f2_pack(s[2 * (k0 + k)], s[2 * (k0 + k) + 1]), scale2, offset2), lo, hi);
          lo = exp2_approx(lo), hi = exp2_approx(hi);
          if (k & 1) acc1 = f2_add(acc1, f2_pack(lo, hi));
          else acc0 = f2_add(acc0, f2_pack(lo, hi));
          w16[k] = pack16<BF16>(lo, hi);
        }
        tmem_st16(ts + k0, w16);
        if (k0 == 16 && KEYS == 128) {
          tmem_wait_st();
          tc_fence_before();
          if (!hold) mbar_arrive(&c->p_ready[x][0]);
        }
      }
      float a0, a1;
      f2_unpack(f2_add(acc0, acc1), a0, a1);
      sum += a0 + a1;
      tmem_wait_st();
      if (hold) {
        const float keep = sum;
        finish();
        __syncwarp();
        sum = keep;
        if (failed) return false;
      }
      tc_fence_before();
      if (hold || KEYS == 64) mbar_arrive(&c->p_ready[x][0]);
      mbar_arrive(&c->p_ready[x][1]);
      if (pending && !hold) {
        const float keep = sum;
        finish();
        __syncwarp();
        sum = keep;
        if (failed) return false;
      }
      return true;
    };
    Item it;
    while (!failed && next_item(it)) {
      const int steps = it.steps[x];
      if (steps == 0) continue;
      tok = min(it.tok[x] + row_tok, it.rows - 1);
      first_hidden = (it.tok[x] + 1) >> 7;  // first key tile that a row of this tile does not see whole
      m = -INFINITY, sum = 0.f;
      for (int j = 0; 2 * j < steps && !failed; ++j) {
        const bool ok = 2 * j + 1 < steps ? step(std::integral_constant<int, 128>(), j)
                                          : step(std::integral_constant<int, 64>(), j);
        failed |= !ok;
      }
      if (failed) break;
      const int h = it.head * p.group + row_head;
      last.at = (int64_t)(it.start + tok) * p.o_tok + (int64_t)h * p.o_head;
      last.sum = sum;
      last.start = it.start, last.head = it.head, last.tok = tok, last.guard = it.guard;
      if (G::OUTS == 2) to = to == outs ? outs + D : outs;
      last.any = true, last.valid = row_tok < p.tile_tokens && it.tok[x] + row_tok < it.rows;
    }
    if (!failed && last.any) finish();
  }
  if (failed && p.err) atomicOr(reinterpret_cast<unsigned int*>(p.err), SLMT_DEVERR_TIMEOUT);
  __syncthreads();
  if (warp == 8) tmem_dealloc(tmem, kTmemCols);
}

// Tensor map of rows [tokens, heads, D] of a 16-bit type: the box is 64 dims
// (a 128-byte swizzled panel; dims past D read as zero) of box_heads heads of
// box_tokens tokens.
bool encode_rows(CUtensorMap* m, const void* base, bool bf16, int64_t d, int64_t heads, int64_t tokens,
                 int64_t head_stride, int64_t token_stride, int box_heads, int box_tokens) {
  auto enc = tensor_map_encoder();
  if (!enc) return false;
  if (heads == 1) head_stride = d;  // not used
  if (tokens == 1) token_stride = d;
  const cuuint64_t dims[3] = {(cuuint64_t)d, (cuuint64_t)heads, (cuuint64_t)tokens};
  const cuuint64_t strides[2] = {(cuuint64_t)(2 * head_stride), (cuuint64_t)(2 * token_stride)};
  const cuuint32_t box[3] = {64, (cuuint32_t)box_heads, (cuuint32_t)box_tokens};
  const cuuint32_t one[3] = {1, 1, 1};
  return enc(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(base),
             dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, bool BF16>
int prompt_launch(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const PromptParams& p, int grid,
                  int device, cudaStream_t st) {
  // once per device: the attribute belongs to the device's context
  static std::atomic<uint64_t> ready{0};
  const uint64_t bit = device < 64 ? 1ull << device : 0ull;
  if (!(ready.load(std::memory_order_relaxed) & bit)) {
    if (cudaFuncSetAttribute(prompt_kernel<D, BF16>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             PromptGeom<D>::SMEM) != cudaSuccess) {
      launch_status();  // clears it
      return SLMT_ERR_CUDA;
    }
    ready.fetch_or(bit, std::memory_order_relaxed);
  }
  prompt_kernel<D, BF16><<<grid, kThreads, PromptGeom<D>::SMEM, st>>>(mq, mk, mv, p);
  return launch_status();
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
  const float scale_log2 = sm_scale * 1.4426950408889634f;
  if (!(sm_scale > 0.f) || !(scale_log2 - scale_log2 == 0.f)) return SLMT_ERR_SHAPE;
  if (num_reqs == 0 || max_query_len == 0 || num_tokens == 0) return SLMT_OK;
  if (!q || !k || !v || !out || !query_start_loc) return SLMT_ERR_NULL;
  if (rows_overlap(num_tokens, num_q_heads, out_token_stride, out_head_stride)) return SLMT_ERR_SHAPE;
  // the tiled copies: 16-byte aligned rows, strides positive and below 2^40 bytes
  const uintptr_t any = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) |
                        reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(out);
  if (any % 16 != 0) return SLMT_ERR_ALIGN;
  for (const int64_t s : {q_token_stride, k_token_stride, v_token_stride})
    if (num_tokens > 1 && (s % 8 != 0 || s <= 0 || s >= (1ll << 39))) return SLMT_ERR_ALIGN;
  if (num_q_heads > 1 && (q_head_stride % 8 != 0 || q_head_stride <= 0 || q_head_stride >= (1ll << 39)))
    return SLMT_ERR_ALIGN;
  for (const int64_t s : {k_head_stride, v_head_stride})
    if (num_kv_heads > 1 && (s % 8 != 0 || s <= 0 || s >= (1ll << 39))) return SLMT_ERR_ALIGN;
  const int out_unit = out_dtype == SLMT_DTYPE_F32 ? 4 : 8;
  if ((num_tokens > 1 && out_token_stride % out_unit != 0) || (num_q_heads > 1 && out_head_stride % out_unit != 0))
    return SLMT_ERR_ALIGN;

  const bool bf16 = dtype == SLMT_DTYPE_BF16;
  const int group = (int)(num_q_heads / num_kv_heads);
  const int tile_tokens = 128 / group;
  const int64_t max_query = std::min(max_query_len, num_tokens);
  if ((max_query + 2 * tile_tokens - 1) / (2 * tile_tokens) >= (1 << (32 - kReqBits))) return SLMT_ERR_UNSUPPORTED;
  CUtensorMap mq, mk, mv;
  if (!encode_rows(&mq, q, bf16, head_dim, num_q_heads, num_tokens, q_head_stride, q_token_stride, group,
                   tile_tokens) ||
      !encode_rows(&mk, k, bf16, head_dim, num_kv_heads, num_tokens, k_head_stride, k_token_stride, 1, 128) ||
      !encode_rows(&mv, v, bf16, head_dim, num_kv_heads, num_tokens, v_head_stride, v_token_stride, 1, 128))
    return SLMT_ERR_CUDA;
  PromptParams p;
  p.v = v;
  p.out = out;
  p.err = err_flag;
  p.v_tok = v_token_stride, p.v_head = v_head_stride;
  p.o_tok = out_token_stride, p.o_head = out_head_stride;
  p.wait_limit_ns = wait_limit_ns();
  p.stall = debug_stall();
  p.scale_log2 = scale_log2;
  p.num_tokens = (int)num_tokens;
  p.max_query = (int)max_query;
  p.kv = (int)num_kv_heads;
  p.kv_recip = (uint32_t)(((1ull << 32) + num_kv_heads - 1) / num_kv_heads);
  p.group = group;
  p.tile_tokens = tile_tokens;
  p.out_dtype = out_dtype;
  const int sector = 2 * out_unit;
  p.out_wide = reinterpret_cast<uintptr_t>(out) % 32 == 0 && (num_tokens == 1 || out_token_stride % sector == 0) &&
               (num_q_heads == 1 || out_head_stride % sector == 0);
  int dev = 0;
  const int sms = current_device_sms(&dev);
  if (sms <= 0) return SLMT_ERR_CUDA;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  for (int64_t r = 0; r < num_reqs; r += kMaxReqs) {
    const int64_t nr = std::min<int64_t>(kMaxReqs, num_reqs - r);
    p.qsl = query_start_loc + r;
    p.seq_lens = seq_lens ? seq_lens + r : nullptr;
    p.num_reqs = (int)nr;
    // no more CTAs than there can be items
    const int64_t pairs = std::min(nr * ((max_query + 2 * tile_tokens - 1) / (2 * tile_tokens)),
                                   num_tokens / (2 * tile_tokens) + nr);
    if (pairs * num_kv_heads >= INT32_MAX / 2) return SLMT_ERR_UNSUPPORTED;  // items are numbered in 32 bits
    const int grid = (int)std::min<int64_t>(sms, pairs * num_kv_heads);
    int rc;
    if (head_dim == 64)
      rc = bf16 ? prompt_launch<64, true>(mq, mk, mv, p, grid, dev, st) : prompt_launch<64, false>(mq, mk, mv, p, grid, dev, st);
    else if (head_dim == 80)
      rc = bf16 ? prompt_launch<80, true>(mq, mk, mv, p, grid, dev, st) : prompt_launch<80, false>(mq, mk, mv, p, grid, dev, st);
    else
      rc = bf16 ? prompt_launch<128, true>(mq, mk, mv, p, grid, dev, st)
                : prompt_launch<128, false>(mq, mk, mv, p, grid, dev, st);
    if (rc != SLMT_OK) return rc;
  }
  return SLMT_OK;
}
