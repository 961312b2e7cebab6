// Causal attention of packed whole prompts over the BF16 keys and values at
// hand, for sm_100a.
//
//   o_i = sum_{j <= i} p_ij v_j / sum_{j <= i} p_ij,   p_ij = exp(scale q_i . k_j - m_i)
//
// An item is two tiles of 128 query rows of one KV head (a row is a token and a
// query head of the group: 128 / G tokens x G heads).  It walks the prompt's
// keys in tiles of kKeys and runs both products on the tensor cores:
//
//   S = Q K^T      A = Q tile, B = K tile, both [rows, 128 dims], K-major
//   O += P V       A = P in tensor memory, B = V tile [kKeys tokens, 128 dims], MN-major
//
// Every tile is brought by TMA (128-byte swizzle) straight from the packed
// projection, whatever its strides.  Running maximum and sum of the softmax are
// FP32; P is rounded to BF16 for the second product (a tensor-core operand) and
// the denominator sums the unrounded values, as in decode attention.
//
// Tensor memory holds two O tiles (256 columns), two S tiles (2 kKeys) and two P
// tiles.  P has columns of its own, so that the next scores of a tile are made
// while the softmax works on these; a tile's chain is then the softmax alone, and
// the tensor cores follow.  That is why a key tile is narrower than 128: with 128
// keys P has to lie over its S, every tile waits for softmax, O product and S
// product in turn, and an earlier form of this kernel took 23 % longer on one
// prompt of 32,768 tokens (8 + 1 heads).
//
// What bounds it: an S product of 128 rows takes eight steps of 52 cycles (32 +
// 80 / 4 each, the 32 whatever the width), an O product five of 64; that is 736
// cycles where the arithmetic alone is 640.  That prompt has 420,455 such steps of a
// key tile and a query tile, 1,064 us of products on 148 SMs at 1.965 GHz, and takes
// 1,600 us in short runs (1,375 TFLOP/s, 0.84 of 1,643): nothing is saturated.
// 8,192 tokens (32 + 8 heads) under counters: tensor pipe active 67 %, issue slots
// 44 %, special-function unit about half, 103 MB read from DRAM and 33 MB written
// (the results stay in L2 for the next reader); a tile's S product, softmax and O
// product follow one another, and two tiles do not fill the gaps.  Without a pause
// the power limit holds the clock near 1.4 GHz: 1,160 to 1,210 TFLOP/s (0.83 to 0.86
// of the 1,400 that plain products keep up).  16 prompts of 1,000 to 4,096 tokens
// (32 + 8 heads) 702 us, 1,136 TFLOP/s; 64 prompts of up to 300 tokens 48.5 us, where
// an item is too short to hide its own start.  (Figures here and below are short
// runs of the present kernel, within 1.5 % from card to card, where nothing else is
// said.)
//
// One CTA per SM at a time, which goes from item to item; its warps meet only
// through mbarriers, and every wait is bounded and reports through the status
// word:
//   softmax warps  those of query tile 0, then those of tile 1 (a warp reaches
//                  the tensor-memory lanes 32 (warp % 4) ..)
//   result warps   divide an item's O by the sums and store it
//   score warp     issues S products, value warp O products (one elected lane;
//                  two warps, so that neither waits behind the other's barriers;
//                  four, one per tile too, polled so much that an earlier form
//                  took 11 % longer)
//   load warp      loads the items' tiles
//   item warp      picks the CTA's items, up to two ahead of the others
//
// The code is kept short (waits with a small way out, loops over the two tiles
// rolled in the result warps): sixteen warps in seven roles share the instruction
// caches, and 64 short prompts take 56.7 us with the loops of the result warps
// unrolled and 48.5 without.
#include <cuda.h>
#include <math.h>

#include <algorithm>
#include <cfloat>
#include <climits>

#include "fp_api.h"
#include "fp_common.cuh"
#include "fp_pipe.cuh"
#include "fp_tensor.cuh"

namespace fpb {
namespace {

constexpr int kQTiles = 2;
constexpr int kKeys = 80;                  // keys of a tile
constexpr int kStages = 3;                 // K tiles and V tiles in flight, each
constexpr int kKeyTileBytes = kKeys * 256;
constexpr int kKeyHalf = kKeys * 128;      // one 64-dim half of a K or V tile
constexpr int kSoftmaxWarps = 8, kResultWarps = 4;
constexpr int kScoreWarp = kSoftmaxWarps + kResultWarps, kValueWarp = kScoreWarp + 1, kLoadWarp = kScoreWarp + 2,
              kItemWarp = kScoreWarp + 3;
constexpr int kPromptThreads = 32 * (kSoftmaxWarps + kResultWarps + 4);  // whole warpgroups
constexpr int kItemReaders = kLoadWarp + 1;  // warps that read an item's description
// Tensor memory columns: O tiles, S tiles, P tiles.
constexpr int64_t kChunkBytes = 64 << 20;     // see head_chunk
constexpr int kKeptPrompts = 512;             // kept in shared memory, further ones are read again
constexpr uint32_t kTmemColumns = 512, kTmemS = kQTiles * kTile, kTmemP = kTmemS + kQTiles * kKeys;
static_assert(kTmemP + kQTiles * kKeys / 2 <= kTmemColumns && kKeys % 16 == 0, "tensor memory is full");
// Registers of the softmax warps, of the result warps and of the rest: 256 x 184
// + 128 x 88 + 128 x 56 = 512 x 128, what the block is launched with.
constexpr int kSoftmaxRegs = 184, kResultRegs = 88, kOtherRegs = 56;
// How far (log2 units) a row's maximum may rise above the reference point of its
// exponentials before the reference follows and O is rescaled: the caller's choice,
// up to this.  Nothing is lost in range, but the largest weights, rounded to BF16,
// no longer include the exact 1 of a row's maximum.  RMS error against 64 bits,
// relative to that of attention in FP32 with one rounding (five sets of prompts of 1
// to 16,384 tokens), and times of 16 ragged prompts / of one of 32,768 tokens: 8:
// 1.16 to 1.34, 705 / 1,612 us; 4: 1.15 to 1.22, 782 / 1,672; 1: 1.12 to 1.14, 830 /
// 1,739; 0: 1.08 to 1.12, 844 / 1,814 (a rescale waits for the O product before it).
// Largest error at 8: up to 1.9 times that of FP32, at 0 up to 1.2 times.
constexpr float kLongestLag = 8.f;

__device__ int32_t g_prompt_status;

// What every role needs to know about an item.
struct Item {
  int head, row0, length;  // KV head, first row and rows (tokens) of the prompt
  int tok0;                // first token of query tile 0
  int last[kQTiles];       // last key tile of each query tile; -1: it has no rows
};

// A wait that ran out raises `abort`, and every later one gives up at once.
struct PromptWait {
  volatile int abort;
  uint32_t limit;  // cycles
};

struct PromptSmem {
  __align__(1024) uint8_t q[kQTiles][kTileBytes];
  __align__(1024) uint8_t o[kTileBytes];  // results on their way out
  __align__(1024) uint8_t k[kStages][kKeyTileBytes];
  __align__(1024) uint8_t v[kStages][kKeyTileBytes];
  float sum[kQTiles][kTile];  // of the probabilities of each row
  int stray[3][kTile];        // see screen_values
  int stray_item;             // the item that they belong to
  Item item[2];
  int2 prompts[kKeptPrompts];  // first row and rows of the first prompts
  __align__(16) uint8_t block[16];  // answer to the request for a block
  __align__(8) uint64_t block_full;
  uint64_t item_full[2], item_empty[2], item_wanted;
  uint64_t q_full[kQTiles], q_empty[kQTiles];
  uint64_t k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages];
  uint64_t s_ready[kQTiles], s_free[kQTiles];         // S product done; S read
  uint64_t p_ready[kQTiles], p_free[kQTiles];         // P written and O rescaled; O product done
  uint64_t turn[kQTiles][4];                          // a tile's turn at the exponentials, per 32 rows
  uint64_t sum_full[kQTiles], sum_empty[kQTiles];
  uint64_t o_done[kQTiles], o_free[kQTiles];          // the item's last O product done; O read
  uint64_t drained[2];
  uint32_t tmem_base;
  PromptWait wait;
};

struct PromptParams {
  CUtensorMap q_map, k_map, v_map;
  __nv_bfloat16* out;
  int64_t o_token, o_head;
  const int32_t* starts;
  int prompts, tokens, kv_heads;
  int head_chunk;  // KV heads whose items come before the next ones'
  int group, group_log2;
  float scale_log2, lag;
  uint32_t wait_limit;
  int skip_tile;  // test hook: this K tile of an item is not loaded (-1: none)
  int falling_blocks;  // test hook: blocks are numbered from the last one down
};

__device__ __forceinline__ uint32_t clock32() {
  uint32_t c;
  asm volatile("mov.u32 %0, %clock;" : "=r"(c));
  return c;
}

// As bounded_wait, inlined whole (a call would keep the register split from
// taking effect) and without a suspend-time hint: with hints of 2 and 20
// microseconds the waits woke later and the kernel took a tenth longer.
__device__ __forceinline__ bool arrived(uint64_t* bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(smem_addr(bar)), "r"(parity)
      : "memory");
  return done != 0;
}
// What runs out is reported once, at the end of the kernel.
__device__ __forceinline__ bool await(uint64_t* bar, uint32_t parity, PromptWait* ws) {
  if (arrived(bar, parity)) return true;
  const uint32_t t0 = clock32();
#pragma unroll 1
  do {
    if (ws->abort) return false;
    if (clock32() - t0 > ws->limit) ws->abort = 1;
  } while (!arrived(bar, parity));
  return true;
}

// The same with one answer for all lanes of a warp, so that none leaves a loop alone
// when a wait gives up.  Once per item: with votes in all waits one prompt of 32,768
// tokens (8 + 1 heads) takes 13 % longer.
__device__ __forceinline__ bool await_all(uint64_t* bar, uint32_t parity, PromptWait* ws) {
  return __all_sync(0xffffffffu, await(bar, parity, ws));
}

// One arrival for the whole warp.
__device__ __forceinline__ void arrive_warp(uint64_t* bar, int lane) {
  __syncwarp();
  if (lane == 0) mbar_arrive(bar);
}

__device__ __forceinline__ void tmem_acquire() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_release() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }

// Tile coordinates: {dim, head, token}.
__device__ __forceinline__ void tma_load(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
      ::"r"(smem_addr(dst)), "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_addr(bar))
      : "memory");
}
template <int kRows>
__device__ __forceinline__ void tma_load_tile(uint8_t* dst, const CUtensorMap* map, int head, int row, uint64_t* bar) {
  mbar_expect_tx(bar, kRows * 256);
#pragma unroll
  for (int h = 0; h < 2; ++h) tma_load(dst + h * kRows * 128, map, 64 * h, head, row, bar);
}

// The low words of the operand descriptors (address / 16); the rest is constant.
// K-major (Q, K): groups of 8 rows 1024 bytes apart, as tile_desc.  MN-major
// (V: rows are the contraction, 64 dims side by side): groups of 8 tokens 1024
// bytes apart, the two halves of the dims kKeyHalf apart.
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t key_desc_low(uint32_t addr) { return ((addr & 0x3ffffu) >> 4) | (1u << 16); }
__device__ __forceinline__ uint32_t value_desc_low(uint32_t addr) {
  return ((addr & 0x3ffffu) >> 4) | ((uint32_t)(kKeyHalf >> 4) << 16);
}
constexpr uint32_t kScoreInstr = (kInstrDesc & ~(63u << 17)) | ((uint32_t)(kKeys >> 3) << 17);  // N = kKeys
constexpr uint32_t kValueInstr = kInstrDesc | (1u << 16);  // B is MN-major

// The products of one pair of tiles, in steps of 16, by one elected lane
// (the whole warp calls).  One block of assembly: written instruction by
// instruction, moving each descriptor to the uniform registers that the
// instruction reads took longer (90 cycles) than the product itself (64).
#define FP_STEP(a_off, b_off, acc)            \
  "add.u32 a, %1, " #a_off ";\n\t"            \
  "add.u32 b, %2, " #b_off ";\n\t"            \
  "mov.b64 da, {a, %3};\n\t"                  \
  "mov.b64 db, {b, %3};\n\t"                  \
  "@q tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %4, " acc ";\n\t"

// S = Q K^T: the 128-deep rows are two halves of four steps of 32 bytes.
__device__ __forceinline__ void score_product(uint32_t d_tmem, uint32_t q_low, uint32_t k_low) {
  asm volatile(
      "{\n\t.reg .pred q, no, yes;\n\t.reg .b32 a, b;\n\t.reg .b64 da, db;\n\t"
      "elect.sync _|q, 0xffffffff;\n\tsetp.ne.b32 no, 0, 0;\n\tsetp.eq.b32 yes, 0, 0;\n\t"
      FP_STEP(0, 0, "no") FP_STEP(2, 2, "yes") FP_STEP(4, 4, "yes") FP_STEP(6, 6, "yes")
      "add.u32 %2, %2, %5;\n\t"
      FP_STEP(1024, 0, "yes") FP_STEP(1026, 2, "yes") FP_STEP(1028, 4, "yes") FP_STEP(1030, 6, "yes")
      "}"
      : "+r"(d_tmem), "+r"(q_low), "+r"(k_low)
      : "n"(kDescHigh), "r"(kScoreInstr), "n"(kKeyHalf / 16)
      : "memory");
}
#undef FP_STEP

// O (+)= P V over kKeys tokens: steps of 16 tokens, 2048 bytes apart in V and
// eight tensor-memory columns apart in P.
#define FP_STEP(a_off, b_off, acc)            \
  "add.u32 a, %1, " #a_off ";\n\t"            \
  "add.u32 b, %2, " #b_off ";\n\t"            \
  "mov.b64 db, {b, %3};\n\t"                  \
  "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [a], db, %4, " acc ";\n\t"
__device__ __forceinline__ void value_product(uint32_t d_tmem, uint32_t p_tmem, uint32_t v_low, bool accumulate) {
  static_assert(kKeys == 80, "the steps below");
  asm volatile(
      "{\n\t.reg .pred q, acc, yes;\n\t.reg .b32 a, b;\n\t.reg .b64 db;\n\t"
      "elect.sync _|q, 0xffffffff;\n\tsetp.ne.b32 acc, %5, 0;\n\tsetp.eq.b32 yes, 0, 0;\n\t"
      FP_STEP(0, 0, "acc") FP_STEP(8, 128, "yes") FP_STEP(16, 256, "yes") FP_STEP(24, 384, "yes")
      FP_STEP(32, 512, "yes")
      "}"
      ::"r"(d_tmem), "r"(p_tmem), "r"(v_low), "n"(kDescHigh), "r"(kValueInstr), "r"((uint32_t)accumulate)
      : "memory");
}
#undef FP_STEP

// Arrives on `bar` when everything issued so far is done; one elected lane, the
// same as above, where `wanted`.
__device__ __forceinline__ void commit(uint64_t* bar, bool wanted = true) {
  asm volatile(
      "{\n\t.reg .pred q, w;\n\telect.sync _|q, 0xffffffff;\n\tsetp.ne.b32 w, %1, 0;\n\tand.pred q, q, w;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}"
      ::"r"(smem_addr(bar)), "r"((uint32_t)wanted)
      : "memory");
}

// ---------------------------------------------------------------------------
// Items.  An item is a pair of query tiles of some prompt and a KV head; pair i
// of a prompt costs the more the larger i is, and the same in every prompt.

// Finds items by their number, one warp.  They are numbered head_chunk KV heads
// after head_chunk KV heads and within those in the order "all prompts' pairs i,
// from the largest i down", so that the longest are under way first; the warp
// walks down the levels i, and within one through the prompts, and begins again
// should a number fall from call to call (see ask_for_block).
struct ItemPicker {
  const PromptParams& p;
  PromptSmem& sm;
  const int lane;
  int levels, level = -1;
  uint32_t in_chunk = 0, first = 0;  // items of a chunk of heads; number of the first one of the present chunk
  int head0 = 0;                   // its first head
  uint32_t above = 0, here = 0;    // pairs of the levels done; prompts that have one of this level
  int group = 0;                   // prompts 32 group .. are next,
  uint32_t before = 0;             // and so many before them have a pair of this level
  uint32_t latest = 0;             // number of the last call

  __device__ __forceinline__ int2 read_prompt(int r) const {  // first row and rows
    int2 x = make_int2(0, 0);
    if (r < p.prompts) {
      x.x = max(0, min(p.starts[r], p.tokens));
      x.y = max(0, min(p.starts[r + 1], p.tokens) - x.x);
    }
    return x;
  }
  __device__ __forceinline__ int2 prompt(int r) const { return r < kKeptPrompts ? sm.prompts[r] : read_prompt(r); }
  __device__ __forceinline__ int pairs(int rows) const {
    return (rows + (kQTiles * kTile >> p.group_log2) - 1) >> (8 - p.group_log2);
  }
  __device__ __forceinline__ bool reaches(int r) const { return pairs(prompt(r).y) > level; }

  __device__ __forceinline__ void enter_level() {
    here = 0;
    group = 0;
    before = 0;
    for (int r = 0; r < p.prompts; r += 32) here += (uint32_t)__popc(__ballot_sync(0xffffffffu, reaches(r + lane)));
  }
  __device__ __forceinline__ ItemPicker(const PromptParams& params, PromptSmem& smem, int lane_)
      : p(params), sm(smem), lane(lane_) {
    int most = 0, sum = 0;
    for (int r = lane; r < (p.prompts + 31 & ~31); r += 32) {
      const int2 x = read_prompt(r);
      if (r < kKeptPrompts) sm.prompts[r] = x;
      most = max(most, pairs(x.y));
      sum += pairs(x.y);
    }
    levels = (int)__reduce_max_sync(0xffffffffu, (unsigned)most);
    in_chunk = __reduce_add_sync(0xffffffffu, (unsigned)sum) * (uint32_t)p.head_chunk;
    level = levels;  // above every pair
    __syncwarp();
  }
  // Item number `at`; head -1: there are fewer.
  __device__ __forceinline__ Item item(uint32_t at) {
    if (at < latest) {
      level = levels;
      head0 = 0;
      first = above = here = 0;
    }
    latest = at;
    while (head0 < p.kv_heads && at - first >= in_chunk) {
      first += in_chunk;
      head0 += p.head_chunk;
      level = head0 < p.kv_heads ? levels : -1;
      above = here = 0;
    }
    const uint32_t heads = (uint32_t)max(1, min(p.head_chunk, p.kv_heads - head0));
    const uint32_t x = (at - first) / heads;  // pair of every head of the chunk
    while (level >= 0 && x >= above + here) {
      above += here;
      if (--level >= 0) enter_level();
    }
    const int tile_tokens = kTile >> p.group_log2;
    Item w;
    w.head = -1;
    w.row0 = w.length = 0;
    w.tok0 = max(level, 0) * kQTiles * tile_tokens;
    w.last[0] = w.last[1] = -1;
    if (level < 0) return w;
    w.head = head0 + (int)(at - first - x * heads);
    const uint32_t rank = x - above;  // of the prompts of this level
    for (; 32 * group < p.prompts; ++group) {
      const int2 mine = prompt(32 * group + lane);
      uint32_t have = __ballot_sync(0xffffffffu, pairs(mine.y) > level);
      if (rank >= before + (uint32_t)__popc(have)) {
        before += (uint32_t)__popc(have);
        continue;
      }
      for (uint32_t skip = rank - before; skip > 0; --skip) have &= have - 1;
      const int src = __ffs(have) - 1;
      w.row0 = __shfl_sync(0xffffffffu, mine.x, src);
      w.length = __shfl_sync(0xffffffffu, mine.y, src);
      break;
    }
#pragma unroll
    for (int t = 0; t < kQTiles; ++t) {
      const int t0 = w.tok0 + t * tile_tokens;
      if (t0 < w.length) w.last[t] = (min(t0 + tile_tokens, w.length) - 1) / kKeys;
    }
    return w;
  }
};

// Every item has a block of the grid.  A CTA does its own and then takes over
// blocks that have not started yet (cluster launch control), in their order, so
// that whoever is done first goes on first.  The next block is asked for once the
// load warp has begun with the last one taken and the result warps with the one
// before: asked for earlier, it would be bound to a CTA that may be late (two
// prompts of 8,192 tokens, 32 + 32 heads: 914 us without the wait for the load
// warp, 888 with it).  Blocks come in rising order as a rule, but nothing promises
// it: whatever order they come in, every one is looked at, also behind one that has
// no item.
__device__ __forceinline__ void ask_for_block(PromptSmem& sm, int lane) {
  if (lane == 0) {
    mbar_expect_tx(&sm.block_full, 16);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the answer before was read
    asm volatile(
        "clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(
            smem_addr(sm.block)),
        "r"(smem_addr(&sm.block_full))
        : "memory");
  }
  __syncwarp();
}
// The block's number; false: none is left.
__device__ __forceinline__ bool block_taken(PromptSmem& sm, uint32_t& number) {
  uint32_t taken;
  asm volatile(
      "{\n\t.reg .b128 answer;\n\t.reg .pred p;\n\tld.shared.b128 answer, [%2];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, answer;\n\tselp.u32 %0, 1, 0, p;\n\tmov.u32 %1, 0;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, answer;\n\t}"
      : "=r"(taken), "=r"(number)
      : "r"(smem_addr(sm.block))
      : "memory");
  __syncwarp();
  return taken != 0;
}

__device__ __forceinline__ void prompt_items(const PromptParams& p, PromptSmem& sm, int lane) {
  ItemPicker picker(p, sm, lane);
  uint32_t number = blockIdx.x, asked = 0;
  bool more = true, answered = true;  // `number` is a block of this CTA's
  int n = 0;                          // items so far
  const auto publish = [&](const Item& w) {
    if (lane == 0) {
      sm.item[n & 1] = w;
      mbar_arrive(&sm.item_full[n & 1]);
    }
    __syncwarp();
    ++n;
  };
  while (more) {
    const Item w = picker.item(p.falling_blocks ? gridDim.x - 1 - number : number);
    if (w.head >= 0) {
      publish(w);
      if (n >= 2 && !await_all(&sm.item_empty[n & 1], (uint32_t)((n >> 1) - 1) & 1u, &sm.wait)) break;
      if (!await_all(&sm.item_wanted, (uint32_t)(n - 1) & 1u, &sm.wait)) break;
    }
    ask_for_block(sm, lane);
    answered = await_all(&sm.block_full, asked++ & 1u, &sm.wait);
    if (!answered) break;
    more = block_taken(sm, number);
  }
  if (!more) {
    Item none;
    none.head = -1;
    publish(none);
  }
  // A wait ran out, and the call is invalid: the blocks that are left are taken all
  // the same, so that none of them has to start.
  while (more) {
    if (answered) {
      ask_for_block(sm, lane);
      ++asked;
    }
    answered = false;
    for (int tries = 0; tries < 1000 && !answered; ++tries) answered = mbar_try(&sm.block_full, (asked - 1) & 1u, 1000u);
    answered = __all_sync(0xffffffffu, answered);
    if (!answered) return;
    more = block_taken(sm, number);
  }
}

// Takes the next item; false: none is left (or a wait ran out).
__device__ __forceinline__ bool next_item(PromptSmem& sm, int n, int lane, Item& w) {
  const int slot = n & 1;
  if (!await_all(&sm.item_full[slot], (uint32_t)(n >> 1) & 1u, &sm.wait)) return false;
  w = sm.item[slot];
  arrive_warp(&sm.item_empty[slot], lane);
  return w.head >= 0;
}

__device__ __forceinline__ void prompt_load(const PromptParams& p, PromptSmem& sm, int lane) {
  const int tile_tokens = kTile >> p.group_log2;
  uint32_t q_used[kQTiles] = {0, 0};
  uint32_t tile = 0;  // key tiles so far
  bool ok = true;
  Item w;
  for (int n = 0; ok && next_item(sm, n, lane, w); ++n) {
    const int last_any = max(w.last[0], w.last[1]);
    if (lane == 0) {
      mbar_arrive(&sm.item_wanted);
      const auto load_q = [&](int t) {
        if (!ok || w.last[t] < 0) return;
        uint64_t* const full = &sm.q_full[t];
        const uint32_t used = q_used[t]++;
        if (used > 0) ok = await(&sm.q_empty[t], (used - 1) & 1u, &sm.wait);
        if (ok)
          tma_load_tile<kTile>(sm.q[t], &p.q_map, w.head * p.group, w.row0 + w.tok0 + t * tile_tokens, full);
      };
      for (int j = 0; ok && j <= last_any; ++j, ++tile) {
        const uint32_t stage = tile % kStages, use = tile / kStages;
        const int row = w.row0 + j * kKeys;
        if (use > 0) ok = await(&sm.k_empty[stage], (use - 1) & 1u, &sm.wait);
        if (ok && j != p.skip_tile) tma_load_tile<kKeys>(sm.k[stage], &p.k_map, w.head, row, &sm.k_full[stage]);
        if (j == 0) {
          load_q(0);
          load_q(1);
        }
        if (ok && use > 0) ok = await(&sm.v_empty[stage], (use - 1) & 1u, &sm.wait);
        if (ok) tma_load_tile<kKeys>(sm.v[stage], &p.v_map, w.head, row, &sm.v_full[stage]);
      }
    }
    ok = __shfl_sync(0xffffffffu, (int)ok, 0);
  }
  if (lane != 0 || !sm.wait.abort) return;
  // A wait ran out somewhere.  Shared memory is given back at the end of the
  // kernel, so this thread stays until its own copies have landed (bounded: a
  // tile that was left out never lands).
  for (int b = 0; b < 2 * kStages + kQTiles; ++b) {
    uint64_t* bar = b < kStages       ? &sm.k_full[b]
                    : b < 2 * kStages ? &sm.v_full[b - kStages]
                                      : &sm.q_full[b - 2 * kStages];
    for (int parity = 0; parity < 2; ++parity)
      for (int tries = 0; tries < 100 && !mbar_try(bar, (uint32_t)parity, 1000u); ++tries) {
      }
  }
}

// Rows (tokens) from .. of a V tile become zero: no row of the item sees them (they
// come later, belong to another prompt or to nothing), and whatever they hold must
// not meet a zero probability.
__device__ __forceinline__ void clear_value_rows(uint8_t* tile, int from, int lane) {
#pragma unroll 1
  for (int x = from * 8 + lane; x < kKeys * 8; x += 32) {
    reinterpret_cast<uint4*>(tile)[x] = make_uint4(0u, 0u, 0u, 0u);
    reinterpret_cast<uint4*>(tile + kKeyHalf)[x] = make_uint4(0u, 0u, 0u, 0u);
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

// The same goes for tokens that only some of an item's rows see: their zero
// probabilities must not meet an infinity or a NaN.  Do rows from .. to - 1 of a V
// tile hold one?
__device__ __forceinline__ bool has_stray_values(const uint8_t* tile, int from, int to, int lane) {
  uint32_t sum[4] = {0, 0, 0, 0};  // 0 * x of everything, as pairs
#pragma unroll 1
  for (int i = 8 * from + lane; i < 8 * to; i += 32)
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const uint4 x = reinterpret_cast<const uint4*>(tile + half * kKeyHalf)[i];
      asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(sum[0]) : "r"(x.x), "r"(0u));
      asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(sum[1]) : "r"(x.y), "r"(0u));
      asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(sum[2]) : "r"(x.z), "r"(0u));
      asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(sum[3]) : "r"(x.w), "r"(0u));
    }
  return __any_sync(0xffffffffu, (sum[0] | sum[1] | sum[2] | sum[3]) != 0);
}

// Takes all of the tile's out of it (they become zero) and notes in sm.stray, per
// dim, the first token of the prompt that holds an infinity of either sign and the
// first that holds a NaN; the result warps bring them back into the rows that see
// these tokens.  So such values take no time beside the search, which costs 64 short
// prompts 1 us (47.5 to 48.4) and 16 ragged ones 1 %; rows that came out NaN computed
// again one by one took 600 times as long where a prompt of 4,096 tokens held an
// infinity in its first token.  `fresh`: the first time in this item.
__device__ __forceinline__ void screen_values(PromptSmem& sm, uint8_t* tile, int token0, bool fresh, int lane) {
  if (fresh)
    for (int x = lane; x < 3 * kTile; x += 32) sm.stray[x / kTile][x % kTile] = INT_MAX;
  __syncwarp();
#pragma unroll 1
  for (int x = lane; x < kKeyTileBytes / 2; x += 32) {
    uint16_t* const at = reinterpret_cast<uint16_t*>(tile) + x;
    const uint32_t bits = *at;
    if ((bits & 0x7f80u) != 0x7f80u) continue;
    const int row = x % (kKeyHalf / 2) / 64, chunk = (x % 64 >> 3) ^ (row & 7);
    const int dim = x / (kKeyHalf / 2) * 64 + chunk * 8 + (x & 7);
    atomicMin(&sm.stray[(bits & 0x7fu) ? 2 : bits >> 15][dim], token0 + row);
    *at = 0;
  }
  __threadfence_block();
  __syncwarp();
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

// Nothing that this warp issued may still be running when tensor memory is given
// back, also when a wait gave up and the roles ran ahead.
__device__ __forceinline__ void drain(uint64_t* bar) {
  __syncwarp();
  commit(bar);
#pragma unroll 1
  for (int tries = 0; tries < (1 << 20); ++tries)
    if (mbar_try(bar, 0u, 1000u)) break;
  __syncwarp();
}

// The warp that issues the score products, key tile by key tile for both query
// tiles: S_t(j) as soon as the softmax has taken S_t(j - 1).
__device__ __forceinline__ void issue_scores(PromptSmem& sm, uint32_t tmem, int lane) {
  uint32_t q_used[kQTiles] = {0, 0}, issued[kQTiles] = {0, 0};
  uint32_t tile = 0;  // key tiles so far
  Item w;
  for (int n = 0; next_item(sm, n, lane, w); ++n) {
    const int last_any = max(w.last[0], w.last[1]);
#pragma unroll 1
    for (int j = 0; j <= last_any; ++j, ++tile) {
      const uint32_t stage = tile % kStages;
      await(&sm.k_full[stage], (tile / kStages) & 1u, &sm.wait);
#pragma unroll
      for (int t = 0; t < kQTiles; ++t) {
        if (j > w.last[t]) continue;
        if (j == 0) await(&sm.q_full[t], q_used[t]++ & 1u, &sm.wait);
        if (issued[t] > 0) await(&sm.s_free[t], (issued[t] - 1) & 1u, &sm.wait);
        ++issued[t];
        __syncwarp();
        tmem_acquire();
        score_product(tmem + kTmemS + (uint32_t)(t * kKeys), key_desc_low(smem_addr(sm.q[t])),
                      key_desc_low(smem_addr(sm.k[stage])));
        commit(&sm.s_ready[t]);
        if (j == w.last[t]) commit(&sm.q_empty[t]);
      }
      commit(&sm.k_empty[stage]);
    }
  }
  drain(&sm.drained[0]);
}

// The warp that issues the value products: O_t(j) as soon as P_t(j) is written.
__device__ __forceinline__ void issue_values(PromptSmem& sm, uint32_t tmem, int lane, int group_log2) {
  uint32_t items[kQTiles] = {0, 0}, issued[kQTiles] = {0, 0};
  uint32_t tile = 0;  // key tiles so far
  Item w;
  for (int n = 0; next_item(sm, n, lane, w); ++n) {
    const int last_any = max(w.last[0], w.last[1]);
    // Tokens up to tok0 are seen by every row of the item, those from `end` on by none.
    const int end = min(w.tok0 + (kQTiles * kTile >> group_log2), w.length);
    bool screened = false;
#pragma unroll 1
    for (int j = 0; j <= last_any; ++j, ++tile) {
      const uint32_t stage = tile % kStages;
      await(&sm.v_full[stage], (tile / kStages) & 1u, &sm.wait);
      const int to = min(end - j * kKeys, kKeys), from = max(w.tok0 + 1 - j * kKeys, 0);
      if (to < kKeys) clear_value_rows(sm.v[stage], to, lane);
      if (from < to && has_stray_values(sm.v[stage], from, to, lane)) {
        // What is noted of an earlier item has been read once its O has been: of the
        // tiles that this item has, that is so from its second key tile on.
#pragma unroll 1
        for (int t = 0; t < kQTiles; ++t)
          if ((j == 0 || w.last[t] < 0) && items[t] > 0) await(&sm.o_free[t], (items[t] - 1) & 1u, &sm.wait);
        screen_values(sm, sm.v[stage], j * kKeys, !screened, lane);
        screened = true;
        if (lane == 0) *reinterpret_cast<volatile int*>(&sm.stray_item) = n;
      }
#pragma unroll
      for (int t = 0; t < kQTiles; ++t) {
        if (j > w.last[t]) continue;
        // The result warps have read the item before's O.
        if (j == 0 && items[t]++ > 0) await(&sm.o_free[t], items[t] & 1u, &sm.wait);
        await(&sm.p_ready[t], issued[t]++ & 1u, &sm.wait);
        __syncwarp();
        tmem_acquire();
        value_product(tmem + (uint32_t)(t * kTile), tmem + kTmemP + (uint32_t)(t * kKeys / 2),
                      value_desc_low(smem_addr(sm.v[stage])), j > 0);
        commit(&sm.p_free[t]);
        if (j == w.last[t]) {
          commit(&sm.o_done[t]);
          arrive_warp(&sm.o_done[t], lane);  // for what screen_values wrote
        }
      }
      commit(&sm.v_empty[stage]);
    }
  }
  drain(&sm.drained[1]);
}

// ---------------------------------------------------------------------------
// Softmax.

__device__ __forceinline__ uint64_t pack2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack2(uint64_t x, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.ftz.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.ftz.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// Largest of three, NaN if one is.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ uint32_t bf16_pair(float low, float high) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(high), "f"(low));
  return r;
}

// Loads or stores kCount 32-bit columns of this thread's lane; the caller waits.
template <int kCount>
__device__ __forceinline__ void tmem_load(uint32_t at, uint32_t* r) {
  if constexpr (kCount >= 32) {
    tmem_load32_async(at, *reinterpret_cast<uint32_t(*)[32]>(r));
    tmem_load<kCount - 32>(at + 32, r + 32);
  } else if constexpr (kCount >= 16) {
    tmem_load16_async(at, *reinterpret_cast<uint32_t(*)[16]>(r));
    tmem_load<kCount - 16>(at + 16, r + 16);
  } else {
    static_assert(kCount == 0, "columns come in sixteens");
  }
}
template <int kCount>
__device__ __forceinline__ void tmem_store(uint32_t at, const uint32_t* r) {
  if constexpr (kCount >= 16) {
    tmem_store16(at, *reinterpret_cast<const uint32_t(*)[16]>(r));
    tmem_store<kCount - 16>(at + 16, r + 16);
  } else if constexpr (kCount >= 8) {
    tmem_store8(at, *reinterpret_cast<const uint32_t(*)[8]>(r));
    tmem_store<kCount - 8>(at + 8, r + 8);
  } else {
    static_assert(kCount == 0, "columns come in eights");
  }
}

// Scores of the columns behind `visible` become -inf, in place.  Rolled loops over
// the few pieces that the diagonal crosses and those behind it, in front of the
// one copy of the softmax: a second, masked copy of that was fetched anew by every
// item and its steps took twice as long; the mask in registers, behind the load,
// made 128 prompts of 128 tokens (32 + 32 heads) 7 % slower, reading the pieces
// behind the diagonal too 4 %.
__device__ __forceinline__ void hide_later(uint32_t tmem_s, int visible) {
  // A warp's rows are in the order of their tokens.
  const int lowest = __shfl_sync(0xffffffffu, visible, 0), highest = __shfl_sync(0xffffffffu, visible, 31);
  int c = max(0, (lowest + 1) & ~15);
#pragma unroll 1
  for (; c <= min(highest, kKeys - 1); c += 16) {
    uint32_t s[16];
    tmem_load16_async(tmem_s + (uint32_t)c, s);
    tmem_wait_loads();
#pragma unroll
    for (int x = 0; x < 16; ++x)
      if (c + x > visible) s[x] = 0xff800000u;
    tmem_store16(tmem_s + (uint32_t)c, s);
  }
#pragma unroll 1
  for (; c < kKeys; c += 16) {
    uint32_t s[16];
#pragma unroll
    for (int x = 0; x < 16; ++x) s[x] = 0xff800000u;
    tmem_store16(tmem_s + (uint32_t)c, s);
  }
  tmem_wait_stores();
}

// Softmax warps of query tile `mine`: thread = query row.
__device__ __forceinline__ void prompt_softmax(const PromptParams& p, PromptSmem& sm, uint32_t tmem, int mine, int row) {
  const int lane = row & 31, rows = row >> 5;
  const uint32_t lanes = (uint32_t)(32 * rows) << 16;
  const uint32_t tmem_s = tmem + lanes + kTmemS + (uint32_t)(mine * kKeys);
  const uint32_t tmem_p = tmem + lanes + kTmemP + (uint32_t)(mine * (kKeys / 2));
  const uint32_t tmem_o = tmem + lanes + (uint32_t)(mine * kTile);
  const uint64_t scale2 = pack2(p.scale_log2, p.scale_log2);
  uint32_t s_used = 0, sums = 0;
  // Tile 0's warp and tile 1's of the same rows sit on one scheduler and take
  // turns at the exponentials, tile 0 first: side by side both would be slow,
  // and the tensor cores would wait for both.  The turn is passed on at half of
  // them, so that the other's are there when these end (one prompt of 32,768
  // tokens, 8 + 1 heads: 1,601 us, at the end or at a third 1,613).
  uint32_t turns = 0;
  const auto take_turn = [&] {
    await(&sm.turn[mine][rows], (turns + (uint32_t)mine + 1) & 1u, &sm.wait);  // tile 0's first passes at once
    // Lane 0 passes the turn on alone.  Without this, a lane still polling could find
    // that the turn had come back, its barrier's parity where it was, and poll on.
    // (The other waits are followed by a meeting of the warp before it arrives
    // anywhere.)
    __syncwarp();
    ++turns;
  };
  Item w;
  for (int n = 0; next_item(sm, n, lane, w); ++n) {
    const int my_last = w.last[mine];
    // Rows past the prompt compute like its last token.
    const int position = min(w.tok0 + ((mine * kTile + row) >> p.group_log2), w.length - 1);
    // Key tiles below this one are seen whole by every row.
    const int first_masked = (w.tok0 + (mine * kTile >> p.group_log2) + 1) / kKeys;
    // Weights are 2^-shift smaller, so that they sum to less than a half (each is
    // below 2^lag otherwise) and no sum of finite values overflows.  What that takes
    // from the other end: of one prompt of 32,768 tokens, values of 2^-90 come out
    // to 2^-19, of 2^-96 to 2^-9, and below 2^-104 as zero.
    const float shift = p.lag + 1.f + (float)(32 - __clz(w.length));
    float ref = 0.f;  // reference point of the exponentials
    uint64_t row_sum[2] = {0, 0};
#pragma unroll 1
    for (int j = 0; j <= my_last; ++j) {
      await(&sm.s_ready[mine], s_used & 1u, &sm.wait);
      ++s_used;
      tmem_acquire();
      if (j >= first_masked) hide_later(tmem_s, position - j * kKeys);
      uint32_t s[kKeys];
      tmem_load<kKeys>(tmem_s, s);
      tmem_wait_loads();
      tmem_release();
      arrive_warp(&sm.s_free[mine], lane);
      float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int x = 0; x < kKeys; x += 2)
        top[(x >> 1) & 3] = max3(top[(x >> 1) & 3], __uint_as_float(s[x]), __uint_as_float(s[x + 1]));
      // The scale is positive, so the largest raw score gives the largest scaled one.
      float tile_max = max3(max3(top[0], top[1], top[2]), top[3], top[3]) * p.scale_log2;
      // The reference follows the running maximum once that is p.lag above it.
      if (__any_sync(0xffffffffu, j == 0 || !(tile_max <= ref + p.lag))) {
        // An infinite or NaN maximum makes the whole row NaN.
        if (!(tile_max < INFINITY)) tile_max = NAN;
        if (j == 0) {
          ref = tile_max == -INFINITY ? -FLT_MAX : tile_max;  // below every score to come
        } else {
          float keep = 1.f;
          if (!(tile_max <= ref + p.lag)) {
            keep = ex2(ref - tile_max);
            ref = tile_max;
            row_sum[0] = fma2(row_sum[0], pack2(keep, keep), 0);
            row_sum[1] = fma2(row_sum[1], pack2(keep, keep), 0);
          }
          await(&sm.p_free[mine], s_used & 1u, &sm.wait);  // the O product before this one is done
          tmem_acquire();
#pragma unroll 1
          for (int c = 0; c < kTile; c += 16) {
            uint32_t o[16];
            tmem_load16_async(tmem_o + (uint32_t)c, o);
            tmem_wait_loads();
#pragma unroll
            for (int x = 0; x < 16; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * keep);
            tmem_store16(tmem_o + (uint32_t)c, o);
          }
        }
      }
      const uint64_t minus_ref = pack2(-ref - shift, -ref - shift);
      take_turn();
      uint32_t packed[kKeys / 2];
#pragma unroll
      for (int i = 0; i < kKeys / 2; ++i) {  // pairs of columns
        if (i == kKeys / 4 && lane == 0) mbar_arrive(&sm.turn[mine ^ 1][rows]);
        float a, b;
        unpack2(fma2(pack2(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1])), scale2, minus_ref), a, b);
        a = ex2(a);
        b = ex2(b);
        row_sum[i & 1] = add2(row_sum[i & 1], pack2(a, b));
        packed[i] = bf16_pair(a, b);
      }
      if (s_used > 1) await(&sm.p_free[mine], s_used & 1u, &sm.wait);
      tmem_acquire();
      tmem_store<kKeys / 2>(tmem_p, packed);
      tmem_wait_stores();
      tmem_release();
      arrive_warp(&sm.p_ready[mine], lane);
    }
    for (int j = my_last + 1; j <= w.last[mine ^ 1]; ++j) {  // the other tile goes on alone
      take_turn();
      arrive_warp(&sm.turn[mine ^ 1][rows], lane);
    }
    if (my_last < 0) continue;
    float a, b;
    unpack2(add2(row_sum[0], row_sum[1]), a, b);
    if (sums > 0) await(&sm.sum_empty[mine], (sums - 1) & 1u, &sm.wait);
    ++sums;
    sm.sum[mine][row] = a + b;
    arrive_warp(&sm.sum_full[mine], lane);
  }
}

// ---------------------------------------------------------------------------
// Results.

// Result warps: thread = query row of both tiles.
__device__ __forceinline__ void prompt_results(const PromptParams& p, PromptSmem& sm, uint32_t tmem, int row) {
  const int lane = row & 31;
  const uint32_t tmem_o = tmem + ((uint32_t)(row & ~31) << 16);
  uint32_t used = 0;  // bit t: parity of tile t's uses
  Item w;
  for (int n = 0; next_item(sm, n, lane, w); ++n) {
#pragma unroll 1
    for (int t = 0; t < kQTiles; ++t) {
      if ((t == 0 ? w.last[0] : w.last[1]) < 0) continue;
      await(&sm.sum_full[t], (used >> t) & 1u, &sm.wait);
      const float sum = sm.sum[t][row];
      arrive_warp(&sm.sum_empty[t], lane);
      await(&sm.o_done[t], (used >> t) & 1u, &sm.wait);
      used ^= 1u << t;
      tmem_acquire();
      const float inv = 1.f / sum;  // sum 0: every score is -inf, and the row NaN
      // Rows go out through shared memory, so that they leave in whole lines; a
      // warp keeps to its 32 rows.
      const uint64_t inv2 = pack2(inv, inv);
#pragma unroll 1
      for (int c = 0; c < kTile; c += 32) {
        uint32_t o[32];
        tmem_load32(tmem_o + (uint32_t)(t * kTile + c), o);
#pragma unroll
        for (int ch = 0; ch < 4; ++ch) {
          uint32_t packed[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const uint64_t y = fma2(pack2(__uint_as_float(o[8 * ch + 2 * x]), __uint_as_float(o[8 * ch + 2 * x + 1])), inv2, 0);
            float a, b;
            unpack2(y, a, b);
            packed[x] = bf16_pair(a, b);
          }
          *reinterpret_cast<uint4*>(sm.o + tile_chunk(row, c + 8 * ch)) = make_uint4(packed[0], packed[1], packed[2], packed[3]);
        }
      }
      if (*reinterpret_cast<volatile int*>(&sm.stray_item) == n) {
        // The infinities and NaN that were taken out of the values, for the rows
        // that see them: there every weight is positive.
        __threadfence_block();
        const int token = w.tok0 + ((t * kTile + row) >> p.group_log2);
#pragma unroll 1
        for (int d = 0; d < kTile; ++d) {
          const bool up = sm.stray[0][d] <= token, down = sm.stray[1][d] <= token;
          float add = up ? INFINITY : down ? -INFINITY : 0.f;
          if (sm.stray[2][d] <= token || (up && down)) add = NAN;
          if (add == 0.f) continue;
          uint16_t* const at = reinterpret_cast<uint16_t*>(sm.o + tile_chunk(row, d)) + (d & 7);
          const float y = __uint_as_float((uint32_t)*at << 16) + add;
          *at = (uint16_t)bf16_pair(y, y);
        }
      }
      tmem_release();
      arrive_warp(&sm.o_free[t], lane);
      // Two rows at a time, 16 bytes a lane; the next two are two heads on, or in
      // the next token (the second next with one head).
      const int first_row = t * kTile + (row & ~31), mine = first_row + (lane >> 4);
      int tok = w.tok0 + (mine >> p.group_log2), g = mine & (p.group - 1);
      const uint8_t* line[4];  // rows of a swizzled group of eight
#pragma unroll
      for (int i = 0; i < 4; ++i) line[i] = sm.o + tile_chunk((row & ~31) + 2 * i + (lane >> 4), 8 * (lane & 15));
      __nv_bfloat16* dst =
          p.out + (int64_t)(w.row0 + tok) * p.o_token + (int64_t)(w.head * p.group + g) * p.o_head + 8 * (lane & 15);
      const int64_t to_head = 2 * p.o_head, to_token = p.group == 1 ? 2 * p.o_token : p.o_token - (p.group - 2) * p.o_head;
      const int tokens = p.group == 1 ? 2 : 1;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        if (tok < w.length)
          *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(line[i & 3] + (i >> 2) * 1024);
        g += 2;
        const bool on = g >= p.group;
        dst += on ? to_token : to_head;
        tok += on ? tokens : 0;
        g = on ? g & (p.group - 1) : g;
      }
      __syncwarp();
    }
  }
}

__global__ void __launch_bounds__(kPromptThreads, 1) prompt_attn_kernel(const __grid_constant__ PromptParams p) {
  // The operand tiles start on 1024-byte boundaries (the swizzle is a function
  // of the address); the launch reserves the slack for this.
  extern __shared__ uint8_t dyn[];
  PromptSmem& sm = *reinterpret_cast<PromptSmem*>(dyn + ((1024u - (smem_addr(dyn) & 1023u)) & 1023u));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sm.item_full[i], 1);
      mbar_init(&sm.item_empty[i], kItemReaders);
    }
#pragma unroll
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&sm.k_full[i], 1);
      mbar_init(&sm.k_empty[i], 1);
      mbar_init(&sm.v_full[i], 1);
      mbar_init(&sm.v_empty[i], 1);
    }
#pragma unroll
    for (int t = 0; t < kQTiles; ++t) {
      mbar_init(&sm.q_full[t], 1);
      mbar_init(&sm.q_empty[t], 1);
      mbar_init(&sm.s_ready[t], 1);
      mbar_init(&sm.s_free[t], 4);  // warps, as all counts below
      mbar_init(&sm.p_ready[t], 4);
      mbar_init(&sm.p_free[t], 1);
      for (int i = 0; i < 4; ++i) mbar_init(&sm.turn[t][i], 1);
      mbar_init(&sm.sum_full[t], 4);
      mbar_init(&sm.sum_empty[t], kResultWarps);
      mbar_init(&sm.o_done[t], 2);  // the products and the value warp
      mbar_init(&sm.o_free[t], kResultWarps);
    }
    mbar_init(&sm.item_wanted, 1);
    mbar_init(&sm.block_full, 1);
    mbar_init(&sm.drained[0], 1);
    mbar_init(&sm.drained[1], 1);
    sm.stray_item = -1;
    sm.wait.abort = 0;
    sm.wait.limit = p.wait_limit;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  __syncwarp();
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&sm.tmem_base)),
                 "r"(kTmemColumns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (warp == kLoadWarp && lane < 3)
    asm volatile("prefetch.tensormap [%0];" ::"l"(lane == 0 ? &p.q_map : lane == 1 ? &p.k_map : &p.v_map) : "memory");
  tmem_release();
  __syncthreads();
  tmem_acquire();
  const uint32_t tmem = sm.tmem_base;

  if (warp < kSoftmaxWarps) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    prompt_softmax(p, sm, tmem, warp >> 2, tid & (kTile - 1));
  } else if (warp < kScoreWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kResultRegs));
    prompt_results(p, sm, tmem, tid & (kTile - 1));
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    if (warp == kScoreWarp) issue_scores(sm, tmem, lane);
    if (warp == kValueWarp) issue_values(sm, tmem, lane, p.group_log2);
    if (warp == kLoadWarp) prompt_load(p, sm, lane);
    if (warp == kItemWarp) prompt_items(p, sm, lane);
  }
  tmem_release();
  __syncthreads();
  if (tid == 0 && sm.wait.abort) atomicOr(&g_prompt_status, FP_DECODE_WAIT_TIMEOUT);
  if (warp == 0) {
    tmem_acquire();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemColumns) : "memory");
  }
}

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                 const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// The driver's tensor map encoder, looked up once (no link against libcuda).
int encode_tiled(EncodeTiled& fn) {
  static std::atomic<void*> known{nullptr};
  void* at = known.load(std::memory_order_acquire);
  if (at == nullptr) {
    cudaDriverEntryPointQueryResult found = cudaDriverEntryPointSymbolNotFound;
    if (int rc = cuda_status(cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &at, 12000, cudaEnableDefault, &found),
                             "cudaGetDriverEntryPointByVersion(cuTensorMapEncodeTiled)"))
      return rc;
    if (found != cudaDriverEntryPointSuccess || at == nullptr)
      return fail(FP_ERR_CUDA, "the driver has no cuTensorMapEncodeTiled");
    known.store(at, std::memory_order_release);
  }
  fn = reinterpret_cast<EncodeTiled>(at);
  return FP_OK;
}

// Map of BF16 [tokens, heads, 128] with boxes of 64 dims x box_heads x
// box_tokens (rows of 128 bytes, swizzled; rows outside the tensor read zero).
// The stride of a dimension of size one is never used and may be anything.
int head_map(CUtensorMap& map, const char* name, const void* base, int64_t tokens, int64_t heads, int64_t token_stride,
             int64_t head_stride, uint32_t box_heads, uint32_t box_tokens) {
  EncodeTiled fn = nullptr;
  if (int rc = encode_tiled(fn)) return rc;
  if (heads == 1) head_stride = 128;
  if (tokens == 1) token_stride = heads * head_stride;
  const cuuint64_t sizes[3] = {128, (cuuint64_t)heads, (cuuint64_t)tokens};
  const cuuint64_t strides[2] = {(cuuint64_t)head_stride * 2, (cuuint64_t)token_stride * 2};
  const cuuint32_t box[3] = {64, box_heads, box_tokens}, step[3] = {1, 1, 1};
  const CUresult rc =
      fn(&map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), sizes, strides, box, step,
         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (rc != CUDA_SUCCESS) return fail(FP_ERR_ARGUMENT, "no tensor map for %s (driver error %d)", name, (int)rc);
  return FP_OK;
}

// KV heads whose keys and values (512 bytes a token) are walked together: as many
// as kChunkBytes hold, so that they stay in L2 while every pair of query tiles
// reads them; rather fewer than chunks of different sizes, whose last one would
// leave SMs without work.  All heads at a time / 20 / 32 / 48 / 64 / 96 MB: 16
// prompts of 1,000 to 4,096 tokens (32 + 8 heads, 168 MB) 748 / 710 / 709 / 700 /
// 701 / 706 us, two of 8,192 (32 + 32 heads, 268 MB) 953 / 924 / 897 / 897 / 888
// / 889 us.
int head_chunk(int64_t tokens, int kv_heads) {
  const int most = (int)std::max<int64_t>(1, std::min<int64_t>(kv_heads, kChunkBytes / (tokens * 512)));
  for (int n = most; 2 * n > most; --n)
    if (kv_heads % n == 0) return n;
  return most;
}

std::atomic<int>& falling_blocks() {
  static std::atomic<int> on{0};
  return on;
}

bool strides_fit(const void* base, int64_t tokens, int64_t heads, int64_t token_stride, int64_t head_stride) {
  const auto fits = [](int64_t n, int64_t stride) {
    return n == 1 || (stride > 0 && stride % 8 == 0 && stride < (1LL << 38));
  };
  return reinterpret_cast<uintptr_t>(base) % 16 == 0 && fits(tokens, token_stride) && fits(heads, head_stride);
}

}  // namespace
}  // namespace fpb

using namespace fpb;

extern "C" {

int fp_prompt_attention(const void* q, int64_t q_token, int64_t q_head, const void* k, int64_t k_token, int64_t k_head,
                        const void* v, int64_t v_token, int64_t v_head, const int32_t* starts, int32_t prompts,
                        int64_t tokens, void* out, int64_t o_token, int64_t o_head, int32_t kv_heads, int32_t group,
                        float scale, void* stream) {
  return fp_prompt_attention_lag(q, q_token, q_head, k, k_token, k_head, v, v_token, v_head, starts, prompts, tokens, out,
                                 o_token, o_head, kv_heads, group, scale, kLongestLag, stream);
}

int fp_prompt_attention_lag(const void* q, int64_t q_token, int64_t q_head, const void* k, int64_t k_token,
                            int64_t k_head, const void* v, int64_t v_token, int64_t v_head, const int32_t* starts,
                            int32_t prompts, int64_t tokens, void* out, int64_t o_token, int64_t o_head,
                            int32_t kv_heads, int32_t group, float scale, float lag, void* stream) {
  if (prompts == 0 || tokens == 0) return FP_OK;
  FP_REQUIRE(prompts > 0 && tokens > 0 && tokens < (1LL << 30) && kv_heads > 0 && kv_heads <= 65535,
             "bad prompt geometry (%d prompts, %lld tokens, %d KV heads)", prompts, (long long)tokens, kv_heads);
  FP_REQUIRE(group == 1 || group == 2 || group == 4 || group == 8, "query group %d must be 1, 2, 4 or 8", group);
  const float scale_log2 = scale * 1.4426950408889634f;
  FP_REQUIRE(scale_log2 >= FLT_MIN && scale_log2 < INFINITY,
             "the softmax scale must be positive and finite, and so must its product with log2(e) in normal FP32");
  FP_REQUIRE(lag >= 0.f && lag <= kLongestLag, "the lag must be within 0 .. %g", kLongestLag);
  FP_REQUIRE(q && k && v && starts && out, "null prompt attention argument");
  const int q_heads = kv_heads * group;
  FP_REQUIRE(strides_fit(q, tokens, q_heads, q_token, q_head) && strides_fit(k, tokens, kv_heads, k_token, k_head) &&
                 strides_fit(v, tokens, kv_heads, v_token, v_head) &&
                 strides_fit(out, tokens, q_heads, o_token, o_head),
             "q / k / v / out rows must be 16-byte aligned with positive strides");
  PromptParams p;
  const uint32_t tile_tokens = (uint32_t)(kTile / group);
  if (int rc = head_map(p.q_map, "q", q, tokens, q_heads, q_token, q_head, (uint32_t)group, tile_tokens)) return rc;
  if (int rc = head_map(p.k_map, "k", k, tokens, kv_heads, k_token, k_head, 1, kKeys)) return rc;
  if (int rc = head_map(p.v_map, "v", v, tokens, kv_heads, v_token, v_head, 1, kKeys)) return rc;
  static std::atomic<uint64_t> smem_allowed;
  const int smem = (int)sizeof(PromptSmem) + 1024;
  if (int rc = allow_dynamic_smem(prompt_attn_kernel, smem, smem_allowed)) return rc;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.o_token = o_token;
  p.o_head = o_head;
  p.starts = starts;
  p.prompts = prompts;
  p.tokens = (int)tokens;
  p.kv_heads = kv_heads;
  p.head_chunk = head_chunk(tokens, kv_heads);
  p.group = group;
  p.group_log2 = group == 1 ? 0 : group == 2 ? 1 : group == 4 ? 2 : 3;
  p.scale_log2 = scale_log2;
  p.lag = lag;
  p.wait_limit = (uint32_t)std::min<long long>(wait_debug().limit, 0xf0000000LL);
  p.skip_tile = (int)std::max<long long>(-1, std::min<long long>(wait_debug().skip_record, 1 << 20));
  p.falling_blocks = falling_blocks().load(std::memory_order_relaxed);
  // Every prompt has at most one pair of tiles that is not full.
  const int64_t items = (tokens / (kQTiles * tile_tokens) + prompts) * kv_heads;
  FP_REQUIRE(items < (1LL << 31), "too much work for one call (%lld tokens, %d prompts, %d KV heads)", (long long)tokens,
             prompts, kv_heads);
  prompt_attn_kernel<<<(unsigned)items, kPromptThreads, smem, (cudaStream_t)stream>>>(p);
  FP_LAUNCH_CHECK("prompt_attn_kernel");
  return FP_OK;
}

int fp_debug_falling_blocks(int32_t on) {
  falling_blocks().store(on != 0, std::memory_order_relaxed);
  return FP_OK;
}

int fp_prompt_status(int32_t* status) {
  FP_REQUIRE(status, "null status");
  // The copies below go by the legacy stream, which non-blocking streams do not wait for.
  if (int rc = cuda_status(cudaDeviceSynchronize(), "cudaDeviceSynchronize")) return rc;
  if (int rc = cuda_status(cudaMemcpyFromSymbol(status, g_prompt_status, sizeof(int32_t)),
                           "cudaMemcpyFromSymbol(g_prompt_status)"))
    return rc;
  const int32_t zero = 0;
  return cuda_status(cudaMemcpyToSymbol(g_prompt_status, &zero, sizeof(int32_t)),
                     "cudaMemcpyToSymbol(g_prompt_status)");
}

}  // extern "C"
