// Causal attention of packed whole prompts over the BF16 keys and values at
// hand, for sm_100a.
//
//   o_i = sum_{j <= i} p_ij v_j / sum_{j <= i} p_ij,   p_ij = exp(scale q_i . k_j - m_i)
//
// A CTA takes two tiles of 128 query rows of one KV head (a row is a token and
// a query head of the group: 128 / G tokens x G heads), walks the prompt's keys
// in tiles of 128 and runs both products on the tensor cores (tcgen05.mma):
//
//   S = Q K^T      A = Q tile, B = K tile, both [rows, 128 dims], K-major
//   O += P V       A = P in tensor memory, B = V tile [128 tokens, 128 dims], MN-major
//
// Every tile is brought by TMA (128-byte swizzle) straight from the packed
// projection, whatever its strides.  Running maximum and sum of the softmax are
// FP32, one thread per query row; P is rounded to BF16 for the second product
// and the denominator sums the unrounded values, as in decode attention.
//
//   warps 0-3   softmax of query tile 0, warps 4-7 of query tile 1
//   warp 8      issues every tcgen05.mma
//   warp 9      TMA loads
#include <cuda.h>
#include <math.h>

#include "fp_api.h"
#include "fp_common.cuh"
#include "fp_pipe.cuh"
#include "fp_tensor.cuh"

namespace fpb {
namespace {

constexpr int kQTiles = 2;
constexpr int kStages = 2;            // K tiles and V tiles in flight, each
constexpr int kSoftmaxThreads = 256;  // one warpgroup per query tile, thread = row
constexpr int kIssueWarp = 8, kLoadWarp = 9;
constexpr int kPromptThreads = kSoftmaxThreads + 64;
constexpr uint32_t kTmemColumns = 512;  // S tiles: 0..255, O tiles: 256..511

__device__ int32_t g_prompt_status;

struct PromptSmem {
  __align__(1024) uint8_t q[kQTiles][kTileBytes];
  __align__(1024) uint8_t k[kStages][kTileBytes];
  __align__(1024) uint8_t v[kStages][kTileBytes];
  __align__(8) uint64_t q_full;
  uint64_t k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages];
  uint64_t s_ready[kQTiles], p_ready[kQTiles], o_done[kQTiles];
  uint64_t drained;
  uint32_t tmem_base;
  int row0, length, tile;  // of the CTA's work; tile -1: none
  WaitState wait;
};

// BF16 [tokens, heads, 128], strides in scalars.
struct Heads {
  const __nv_bfloat16* at;
  int64_t token, head;
};

struct PromptParams {
  CUtensorMap q_map, k_map, v_map;
  Heads q, k, v;
  __nv_bfloat16* out;
  int64_t o_token, o_head;
  const int32_t* starts;
  int prompts, tokens, group;
  float scale_log2;
  long long wait_limit;
  int skip_tile;  // test hook: this K tile is not loaded (-1: none)
};

// What every role needs to know about the CTA's work.
struct PromptWork {
  int head, row0, length;  // KV head, first row and rows (tokens) of the prompt
  int tok0, tile_tokens;   // first token of tile 0, tokens per tile
  int last[kQTiles];       // last key tile of each query tile; -1: it has no rows
  int last_any;
};

// Key tile coordinates: {dim, head, token}.
__device__ __forceinline__ void tma_load(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
      ::"r"(smem_addr(dst)), "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_addr(bar))
      : "memory");
}

// V tile as the B operand: rows are the contraction (tokens), 64 dims side by
// side: groups of 8 tokens 1024 bytes apart, the two halves of the dims
// kHalfTile apart (MN-major, 128-byte swizzle).
__device__ __forceinline__ uint64_t value_desc(uint32_t addr) {
  return (uint64_t)((addr & 0x3ffffu) >> 4) | ((uint64_t)(kHalfTile >> 4) << 16) |
         ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
constexpr uint32_t kValueInstr = kInstrDesc | (1u << 16);  // B is MN-major

// O (+)= P V over 128 tokens: eight steps of 16 tokens, 2048 bytes apart in V
// and eight tensor-memory columns apart in P.
__device__ __forceinline__ void value_product(uint32_t d_tmem, uint32_t p_tmem, uint32_t v_addr, bool accumulate) {
#pragma unroll
  for (int j = 0; j < 8; ++j)
    umma_tmem_a(d_tmem, p_tmem + 8u * (uint32_t)j, value_desc(v_addr + 2048u * (uint32_t)j), accumulate || j > 0,
                kValueInstr);
}

// One warp finds the CTA's prompt: item x of the list of all prompts' pairs of
// query tiles, the last (longest) pair of each prompt first.
__device__ __forceinline__ void find_work(const PromptParams& p, PromptSmem& sm, int lane) {
  const int pair_tokens = kQTiles * kTile / p.group;
  int left = (int)blockIdx.x;
  for (int base = 0; base < p.prompts; base += 32) {
    const int r = base + lane;
    int row0 = 0, length = 0;
    if (r < p.prompts) {
      row0 = max(0, min(p.starts[r], p.tokens));
      length = max(0, min(p.starts[r + 1], p.tokens) - row0);
    }
    const int pairs = (length + pair_tokens - 1) / pair_tokens;
    int upto = pairs;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int other = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane >= d) upto += other;
    }
    const uint32_t beyond = __ballot_sync(0xffffffffu, upto > left);
    if (beyond) {
      if (lane == __ffs(beyond) - 1) {
        sm.row0 = row0;
        sm.length = length;
        sm.tile = pairs - 1 - (left - (upto - pairs));
      }
      return;
    }
    left -= __shfl_sync(0xffffffffu, upto, 31);
  }
  if (lane == 0) sm.tile = -1;
}

__device__ __forceinline__ void prompt_load(const PromptParams& p, PromptSmem& sm, const PromptWork& w) {
  mbar_expect_tx(&sm.q_full, kQTiles * kTileBytes);
#pragma unroll
  for (int t = 0; t < kQTiles; ++t)
#pragma unroll
    for (int h = 0; h < 2; ++h)
      tma_load(sm.q[t] + h * kHalfTile, &p.q_map, 64 * h, w.head * p.group, w.row0 + w.tok0 + t * w.tile_tokens, &sm.q_full);
  int loaded = 0;
  for (; loaded <= w.last_any; ++loaded) {
    const int stage = loaded % kStages, use = loaded / kStages, row = w.row0 + loaded * kTile;
    if (use > 0 && !bounded_wait(&sm.k_empty[stage], (use - 1) & 1u, &sm.wait)) break;
    if (loaded != p.skip_tile) {
      mbar_expect_tx(&sm.k_full[stage], kTileBytes);
#pragma unroll
      for (int h = 0; h < 2; ++h)
        tma_load(sm.k[stage] + h * kHalfTile, &p.k_map, 64 * h, w.head, row, &sm.k_full[stage]);
    }
    if (use > 0 && !bounded_wait(&sm.v_empty[stage], (use - 1) & 1u, &sm.wait)) break;
    mbar_expect_tx(&sm.v_full[stage], kTileBytes);
#pragma unroll
    for (int h = 0; h < 2; ++h)
      tma_load(sm.v[stage] + h * kHalfTile, &p.v_map, 64 * h, w.head, row, &sm.v_full[stage]);
  }
  if (!*(volatile int*)&sm.wait.abort) return;
  // A wait ran out somewhere: shared memory is given back at the end of the
  // kernel, so this thread stays until its own copies have landed.
  for (int tile = max(0, loaded - kStages); tile <= min(loaded, w.last_any); ++tile) {
    const int stage = tile % kStages;
    const uint32_t parity = (uint32_t)(tile / kStages) & 1u;
    for (int tries = 0; tries < 1000 && tile != p.skip_tile && !mbar_try(&sm.k_full[stage], parity, 1000u); ++tries) {
    }
    for (int tries = 0; tries < 1000 && tile < loaded && !mbar_try(&sm.v_full[stage], parity, 1000u); ++tries) {
    }
  }
}

// Rows (tokens) valid .. 127 of a V tile become zero: they belong to another
// prompt or to nothing, and whatever they hold must not meet a zero probability.
__device__ __forceinline__ void clear_value_rows(uint8_t* tile, int valid, int lane) {
  for (int x = valid * 16 + lane; x < kTile * 16; x += 32) {
    const int row = x >> 4, chunk = x & 15;
    *reinterpret_cast<uint4*>(tile + (chunk >> 3) * kHalfTile + row * 128 + (chunk & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

// The warp that issues the products: S_t(0); then per key tile j and query tile
// t: O_t(j), S_t(j + 1).
__device__ __forceinline__ void prompt_issue(PromptSmem& sm, const PromptWork& w, uint32_t tmem, int lane) {
  const auto after_wait = [] { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); };
  const auto scores = [&](int t, int j) {
    if (lane == 0) {
      tile_product(tmem + (uint32_t)(t * kTile), smem_addr(sm.q[t]), smem_addr(sm.k[j % kStages]), false);
      umma_commit(&sm.s_ready[t]);
    }
  };
  const auto last_tile = [&](int j) { return j <= w.last[kQTiles - 1] ? kQTiles - 1 : 0; };
  bounded_wait(&sm.q_full, 0u, &sm.wait);
  bounded_wait(&sm.k_full[0], 0u, &sm.wait);
  after_wait();
#pragma unroll
  for (int t = 0; t < kQTiles; ++t)
    if (w.last[t] >= 0) scores(t, 0);
  if (lane == 0) umma_commit(&sm.k_empty[0]);
  for (int j = 0; j <= w.last_any; ++j) {
    const int stage = j % kStages, next = (j + 1) % kStages;
    const uint32_t parity = (uint32_t)(j / kStages) & 1u, next_parity = (uint32_t)((j + 1) / kStages) & 1u;
    bool v_seen = false, k_seen = false;
#pragma unroll
    for (int t = 0; t < kQTiles; ++t) {
      if (j <= w.last[t]) {
        if (!v_seen) {
          bounded_wait(&sm.v_full[stage], parity, &sm.wait);
          const int valid = w.length - j * kTile;
          if (valid < kTile) clear_value_rows(sm.v[stage], valid, lane);
          __syncwarp();
        }
        v_seen = true;
        bounded_wait(&sm.p_ready[t], (uint32_t)j & 1u, &sm.wait);
        after_wait();
        if (lane == 0) {
          // P_t sits in the first half of S_t's columns.
          value_product(tmem + (uint32_t)((kQTiles + t) * kTile), tmem + (uint32_t)(t * kTile),
                        smem_addr(sm.v[stage]), j > 0);
          umma_commit(&sm.o_done[t]);
          if (t == last_tile(j)) umma_commit(&sm.v_empty[stage]);
        }
      }
      if (j + 1 <= w.last[t]) {
        if (!k_seen) bounded_wait(&sm.k_full[next], next_parity, &sm.wait);
        k_seen = true;
        after_wait();
        scores(t, j + 1);
        if (lane == 0 && t == last_tile(j + 1)) umma_commit(&sm.k_empty[next]);
      }
      __syncwarp();
    }
  }
  // Nothing may still be running when tensor memory is given back, also when a
  // wait above gave up and the roles ran ahead.
  if (lane == 0) {
    umma_commit(&sm.drained);
#pragma unroll 1
    for (int tries = 0; tries < (1 << 20); ++tries)
      if (mbar_try(&sm.drained, 0u, 1000u)) break;
  }
  __syncwarp();
}

template <bool kMasked>
__device__ __forceinline__ float chunk_max(const uint32_t (&s)[32], int first, int visible, float m) {
#pragma unroll
  for (int x = 0; x < 32; ++x)
    if (!kMasked || first + x <= visible) m = fmaxf(m, __uint_as_float(s[x]));
  return m;
}

// exp2(score * scale - ref) of 32 scores as 16 BF16 pairs; returns their sum
// (of the unrounded values).
template <bool kMasked>
__device__ __forceinline__ float chunk_probabilities(const uint32_t (&s)[32], int first, int visible, float scale,
                                                     float ref, uint32_t (&packed)[16]) {
  float sum = 0.f;
#pragma unroll
  for (int x = 0; x < 32; x += 2) {
    float a = ex2(fmaf(__uint_as_float(s[x]), scale, -ref));
    float b = ex2(fmaf(__uint_as_float(s[x + 1]), scale, -ref));
    if (kMasked && first + x > visible) a = 0.f;
    if (kMasked && first + x + 1 > visible) b = 0.f;
    sum += a + b;
    const __nv_bfloat162 pair = __floats2bfloat162_rn(a, b);
    packed[x >> 1] = *reinterpret_cast<const uint32_t*>(&pair);
  }
  return sum;
}

// One query row by one warp, key by key over the keys that it sees, lane l
// carrying dims 4 l .. 4 l + 3.  The tensor cores also multiply the values of
// later tokens (by zero probabilities), so a row that came out NaN or infinite
// is computed again here: what it then shows is its own.
__device__ __noinline__ void prompt_row(const PromptParams& p, int row0, int tok, int kv_head, int q_head, int lane) {
  const auto load = [&](const Heads& h, int row, int head, float (&x)[4]) {
    const uint2 two = *reinterpret_cast<const uint2*>(h.at + row * h.token + head * h.head + 4 * lane);
    x[0] = __uint_as_float(two.x << 16);
    x[1] = __uint_as_float(two.x & 0xffff0000u);
    x[2] = __uint_as_float(two.y << 16);
    x[3] = __uint_as_float(two.y & 0xffff0000u);
  };
  float q[4], k[4], v[4], o[4] = {0.f, 0.f, 0.f, 0.f}, top = -INFINITY, sum = 0.f;
  load(p.q, row0 + tok, q_head, q);
  for (int j = 0; j <= tok; ++j) {
    load(p.k, row0 + j, kv_head, k);
    load(p.v, row0 + j, kv_head, v);
    float score = q[0] * k[0] + q[1] * k[1] + q[2] * k[2] + q[3] * k[3];
#pragma unroll
    for (int d = 16; d; d >>= 1) score += __shfl_xor_sync(0xffffffffu, score, d);
    score *= p.scale_log2;
    const float new_top = fmaxf(top, score), ref = new_top == -INFINITY ? 0.f : new_top;
    const float keep = ex2(top - ref), weight = ex2(score - ref);
    sum = sum * keep + weight;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      if (new_top > top) o[x] *= keep;
      if (weight != 0.f) o[x] += weight * v[x];  // also for NaN
    }
    top = new_top;
  }
  const float inv = sum > 0.f ? 1.f / sum : sum;
  const __nv_bfloat162 a = __floats2bfloat162_rn(o[0] * inv, o[1] * inv), b = __floats2bfloat162_rn(o[2] * inv, o[3] * inv);
  *reinterpret_cast<uint2*>(p.out + (row0 + tok) * p.o_token + q_head * p.o_head + 4 * lane) =
      make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}

// Softmax warpgroup of query tile `mine`: thread = query row.
__device__ __forceinline__ void prompt_softmax(const PromptParams& p, PromptSmem& sm, const PromptWork& w,
                                               uint32_t tmem, int mine, int row, int warp) {
  const int my_last = w.last[mine];
  if (my_last < 0) return;
  const int tok = w.tok0 + mine * w.tile_tokens + row / p.group;
  const int position = min(tok, w.length - 1);  // rows past the prompt compute like its last token
  float row_max = -INFINITY, row_sum = 0.f;
  const uint32_t lane_base = (uint32_t)(32 * (warp & 3)) << 16;  // this warp's tensor-memory lanes
  const uint32_t tmem_s = tmem + (uint32_t)(mine * kTile) + lane_base;
  const uint32_t tmem_o = tmem + (uint32_t)((kQTiles + mine) * kTile) + lane_base;
  uint32_t s[32];
  for (int j = 0; j <= my_last; ++j) {
    const uint32_t parity = (uint32_t)j & 1u;
    bounded_wait(&sm.s_ready[mine], parity, &sm.wait);
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const int visible = position - j * kTile;  // columns 0..visible of this tile count
    const bool masked = __any_sync(0xffffffffu, visible < kTile - 1);
    float raw_max = -INFINITY;
#pragma unroll 1
    for (int c = 0; c < 4; ++c) {
      tmem_load32(tmem_s + (uint32_t)(32 * c), s);
      raw_max = masked ? chunk_max<true>(s, 32 * c, visible, raw_max) : chunk_max<false>(s, 32 * c, visible, raw_max);
    }
    const float new_max = fmaxf(row_max, raw_max * p.scale_log2);  // the scale is positive
    const float ref = new_max == -INFINITY ? 0.f : new_max;
    const bool rise = new_max > row_max;
    const float keep = rise ? ex2(row_max - ref) : 1.f;
    if (j > 0) {
      bounded_wait(&sm.o_done[mine], parity ^ 1u, &sm.wait);
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      if (__any_sync(0xffffffffu, rise)) {
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          tmem_load32(tmem_o + (uint32_t)(32 * c), s);
#pragma unroll
          for (int x = 0; x < 32; ++x) s[x] = __float_as_uint(__uint_as_float(s[x]) * keep);
          tmem_store32(tmem_o + (uint32_t)(32 * c), s);
        }
      }
    }
    row_sum *= keep;
    row_max = new_max;
#pragma unroll 1
    for (int c = 0; c < 4; ++c) {
      tmem_load32(tmem_s + (uint32_t)(32 * c), s);
      uint32_t packed[16];
      row_sum += masked ? chunk_probabilities<true>(s, 32 * c, visible, p.scale_log2, ref, packed)
                        : chunk_probabilities<false>(s, 32 * c, visible, p.scale_log2, ref, packed);
      tmem_store16(tmem_s + (uint32_t)(16 * c), packed);  // over scores already read
    }
    tmem_wait_stores();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    mbar_arrive(&sm.p_ready[mine]);
  }

  bounded_wait(&sm.o_done[mine], (uint32_t)my_last & 1u, &sm.wait);
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const float inv = row_sum > 0.f ? 1.f / row_sum : row_sum;  // NaN stays NaN
  __nv_bfloat16* dst = p.out + (int64_t)(w.row0 + tok) * p.o_token + (int64_t)(w.head * p.group + row % p.group) * p.o_head;
  bool finite = true;
#pragma unroll 1
  for (int c = 0; c < 4; ++c) {
    tmem_load32(tmem_o + (uint32_t)(32 * c), s);
    if (tok < w.length) {
#pragma unroll
      for (int ch = 0; ch < 4; ++ch) {
        uint32_t o[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const float a = __uint_as_float(s[8 * ch + 2 * x]) * inv, b = __uint_as_float(s[8 * ch + 2 * x + 1]) * inv;
          finite &= fabsf(a) < INFINITY && fabsf(b) < INFINITY;
          const __nv_bfloat162 pair = __floats2bfloat162_rn(a, b);
          o[x] = *reinterpret_cast<const uint32_t*>(&pair);
        }
        *reinterpret_cast<uint4*>(dst + 32 * c + 8 * ch) = make_uint4(o[0], o[1], o[2], o[3]);
      }
    }
  }
  __syncwarp();
  for (uint32_t again = __ballot_sync(0xffffffffu, !finite); again; again &= again - 1) {
    const int r = row - (row & 31) + __ffs(again) - 1;
    prompt_row(p, w.row0, w.tok0 + mine * w.tile_tokens + r / p.group, w.head, w.head * p.group + r % p.group, row & 31);
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}

__global__ void __launch_bounds__(kPromptThreads, 1) prompt_attn_kernel(const __grid_constant__ PromptParams p) {
  // The operand tiles start on 1024-byte boundaries (the swizzle is a function
  // of the address); the launch reserves the slack for this.
  extern __shared__ uint8_t dyn[];
  PromptSmem& sm = *reinterpret_cast<PromptSmem*>(dyn + ((1024u - (smem_addr(dyn) & 1023u)) & 1023u));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (warp == 0) find_work(p, sm, lane);
  __syncthreads();
  PromptWork w;
  if (sm.tile < 0) return;
  w.head = blockIdx.y;
  w.row0 = sm.row0;
  w.length = sm.length;
  w.tile_tokens = kTile / p.group;
  w.tok0 = sm.tile * kQTiles * w.tile_tokens;
#pragma unroll
  for (int t = 0; t < kQTiles; ++t) {
    const int t0 = w.tok0 + t * w.tile_tokens;
    w.last[t] = t0 < w.length ? (min(t0 + w.tile_tokens, w.length) - 1) >> 7 : -1;
  }
  w.last_any = max(w.last[0], w.last[kQTiles - 1]);

  if (tid == 0) {
    mbar_init(&sm.q_full, 1);
    mbar_init(&sm.drained, 1);
#pragma unroll
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&sm.k_full[i], 1);
      mbar_init(&sm.k_empty[i], 1);
      mbar_init(&sm.v_full[i], 1);
      mbar_init(&sm.v_empty[i], 1);
    }
#pragma unroll
    for (int t = 0; t < kQTiles; ++t) {
      mbar_init(&sm.s_ready[t], 1);
      mbar_init(&sm.o_done[t], 1);
      mbar_init(&sm.p_ready[t], kTile);
    }
    sm.wait.abort = 0;
    sm.wait.status = &g_prompt_status;
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
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = sm.tmem_base;

  if (tid < kSoftmaxThreads) {
    prompt_softmax(p, sm, w, tmem, tid / kTile, tid & (kTile - 1), warp);
  } else if (warp == kIssueWarp) {
    prompt_issue(sm, w, tmem, lane);
  } else if (warp == kLoadWarp && lane == 0) {
    prompt_load(p, sm, w);
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 0) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
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
  if (prompts == 0 || tokens == 0) return FP_OK;
  FP_REQUIRE(prompts > 0 && tokens > 0 && tokens < (1LL << 30) && kv_heads > 0 && kv_heads <= 65535,
             "bad prompt geometry (%d prompts, %lld tokens, %d KV heads)", prompts, (long long)tokens, kv_heads);
  FP_REQUIRE(group == 1 || group == 2 || group == 4 || group == 8, "query group %d must be 1, 2, 4 or 8", group);
  FP_REQUIRE(scale > 0.f && scale < INFINITY, "the softmax scale must be positive and finite");
  FP_REQUIRE(q && k && v && starts && out, "null prompt attention argument");
  const int q_heads = kv_heads * group;
  FP_REQUIRE(strides_fit(q, tokens, q_heads, q_token, q_head) && strides_fit(k, tokens, kv_heads, k_token, k_head) &&
                 strides_fit(v, tokens, kv_heads, v_token, v_head) &&
                 strides_fit(out, tokens, q_heads, o_token, o_head),
             "q / k / v / out rows must be 16-byte aligned with positive strides");
  PromptParams p;
  const uint32_t tile_tokens = (uint32_t)(kTile / group);
  if (int rc = head_map(p.q_map, "q", q, tokens, q_heads, q_token, q_head, (uint32_t)group, tile_tokens)) return rc;
  if (int rc = head_map(p.k_map, "k", k, tokens, kv_heads, k_token, k_head, 1, kTile)) return rc;
  if (int rc = head_map(p.v_map, "v", v, tokens, kv_heads, v_token, v_head, 1, kTile)) return rc;
  static std::atomic<uint64_t> smem_allowed;
  const int smem = (int)sizeof(PromptSmem) + 1024;
  if (int rc = allow_dynamic_smem(prompt_attn_kernel, smem, smem_allowed)) return rc;
  p.q = Heads{static_cast<const __nv_bfloat16*>(q), q_token, q_head};
  p.k = Heads{static_cast<const __nv_bfloat16*>(k), k_token, k_head};
  p.v = Heads{static_cast<const __nv_bfloat16*>(v), v_token, v_head};
  p.out = static_cast<__nv_bfloat16*>(out);
  p.o_token = o_token;
  p.o_head = o_head;
  p.starts = starts;
  p.prompts = prompts;
  p.tokens = (int)tokens;
  p.group = group;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.wait_limit = wait_debug().limit;
  p.skip_tile = (int)std::max<long long>(-1, std::min<long long>(wait_debug().skip_record, 1 << 20));
  // Every prompt has at most one pair of tiles that is not full.
  const int64_t pairs = tokens / (kQTiles * tile_tokens) + prompts;
  prompt_attn_kernel<<<dim3((unsigned)pairs, (unsigned)kv_heads), kPromptThreads, smem, (cudaStream_t)stream>>>(p);
  FP_LAUNCH_CHECK("prompt_attn_kernel");
  return FP_OK;
}

int fp_prompt_status(int32_t* status) {
  FP_REQUIRE(status, "null status");
  if (int rc = cuda_status(cudaMemcpyFromSymbol(status, g_prompt_status, sizeof(int32_t)),
                           "cudaMemcpyFromSymbol(g_prompt_status)"))
    return rc;
  const int32_t zero = 0;
  return cuda_status(cudaMemcpyToSymbol(g_prompt_status, &zero, sizeof(int32_t)),
                     "cudaMemcpyToSymbol(g_prompt_status)");
}

}  // extern "C"
