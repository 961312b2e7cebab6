// RMS norm of query and key heads with the position rotation in the same pass,
// alone (fp_norm_rotary) and on the way into the store (fp_hbm_append), for
// sm_100a.
//
//   y      = x * rsqrt(mean(x^2) + eps) * w            (per head; left out without weights)
//   (a, b) = pair (y_i, y_(i + rot/2)) or (y_2i, y_(2i+1)) of the first `rot` dims
//   (a, b) -> factor * (a cos t - b sin t, b cos t + a sin t),  t = position * frequency_i
//
// Everything between the load and the one rounding of the result to BF16 is
// FP32.  The angle is reduced in 64 bits: a frequency is held in turns per token
// as a 64-bit binary fraction, so position * frequency modulo one turn is one
// wrapping 64-bit multiplication, which adds no error.  The fraction itself is as
// good as the double that it comes from (within 2^-54 turns per token for up to
// one radian per token: 2^-37 turns at position 131,072).  Sine and cosine of the
// remaining half turn come from the special-function unit, whose absolute error
// of about 2^-21 there is a 4000th of the half step of the BF16 result.  No table
// of angles is read.
//
// A head's 128 values are held by half a warp: a lane has two pieces of four
// neighbouring dims, half a rotated range apart, so that both members of every
// pair are in one lane in either layout and nothing is exchanged for the
// rotation (see piece_dims).  Memory bound: 256 bytes in and out per head.
#include <cuda_bf16.h>

#include "fp_api.h"
#include "fp_common.cuh"
#include "fp_store.cuh"

namespace fpb {
namespace {

constexpr int kRowThreads = 256;
constexpr int64_t kManyRows = 65536;  // heads x tokens (see launch_rows)

// A set of heads [tokens, heads, 128] and where their results go (strides in scalars).
struct HeadSet {
  const uint16_t* in;
  uint16_t* out;  // null: no token-major result
  int64_t in_token, in_head, out_token, out_head;
  const void* weight;  // null: no norm
  int heads;
};

struct RotaryParams {
  HeadSet q, k;
  const uint16_t* value;  // append only
  int64_t v_token, v_head;
  const int64_t* slots;  // append only
  const void* positions;
  const uint64_t* turns;
  int64_t tokens;
  int positions_64, weights_f32, rot_lanes, layer, unit;
  float factor, eps;
};

// 16 bytes global -> shared without a register in between.
__device__ __forceinline__ void async_copy16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_addr(dst)), "l"(src) : "memory");
}

// First dims of the two pieces of lane l (0..15) of a half warp.  Lanes below
// rot / 8 hold rotated dims: 4 l .. and, half the rotated range further, rot / 2
// + 4 l ..; the others share the rest in the same manner.
__device__ __forceinline__ void piece_dims(int l, int rot_lanes, int& a, int& b) {
  if (l < rot_lanes) {
    a = 4 * l;
    b = 4 * (rot_lanes + l);
  } else {
    a = 4 * (rot_lanes + l);
    b = 4 * (16 + l);
  }
}

__device__ __forceinline__ float bf16_low(uint32_t x) { return __uint_as_float(x << 16); }
__device__ __forceinline__ float bf16_high(uint32_t x) { return __uint_as_float(x & 0xffff0000u); }
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  const __nv_bfloat162 pair = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&pair);
}

// factor * (cos, sin) of the four angles of this lane.
struct Angles {
  float c[4], s[4];
};

template <bool kInterleaved>
__device__ __forceinline__ Angles lane_angles(const RotaryParams& p, int64_t position, int l, int a, int b) {
  Angles t;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    t.c[i] = 1.f;
    t.s[i] = 0.f;
  }
  if (l >= p.rot_lanes) return t;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    // Half layout: the pairs are (a + i, b + i).  Interleaved: (a, a + 1),
    // (a + 2, a + 3), (b, b + 1), (b + 2, b + 3).
    const int f = kInterleaved ? ((i & 2) ? b : a) / 2 + (i & 1) : a + i;
    const uint64_t phase = (uint64_t)position * p.turns[f];  // turns modulo 1, as a fraction of 2^64
    const float radians = (float)(int32_t)(phase >> 32) * 1.46291807926715968e-9f;  // 2 pi / 2^32
    t.c[i] = p.factor * __cosf(radians);
    t.s[i] = p.factor * __sinf(radians);
  }
  return t;
}

__device__ __forceinline__ void lane_weights(const RotaryParams& p, const void* weight, int a, int b,
                                             float (&w)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int d = (i < 4 ? a : b - 4) + i;
    w[i] = weight == nullptr ? 1.f
           : p.weights_f32   ? static_cast<const float*>(weight)[d]
                             : bf16_low(static_cast<const uint16_t*>(weight)[d]);
  }
}

// One head of a half warp: `x` holds the lane's two pieces as BF16 pairs.
template <bool kInterleaved>
__device__ __forceinline__ void norm_rotate(const RotaryParams& p, uint32_t half_mask, bool norm,
                                            const float (&w)[8], const Angles& t, bool rotated,
                                            uint2 (&x)[2]) {
  if (!norm && !rotated) return;  // such dims keep their bits
  float y[8] = {bf16_low(x[0].x), bf16_high(x[0].x), bf16_low(x[0].y), bf16_high(x[0].y),
                bf16_low(x[1].x), bf16_high(x[1].x), bf16_low(x[1].y), bf16_high(x[1].y)};
  if (norm) {
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum = fmaf(y[i], y[i], sum);
#pragma unroll
    for (int d = 8; d; d >>= 1) sum += __shfl_xor_sync(half_mask, sum, d);
    const float inv = rsqrtf(fmaf(sum, 1.f / 128.f, p.eps));
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] *= inv * w[i];
  }
  if (rotated) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int m = kInterleaved ? 2 * i : i, n = kInterleaved ? 2 * i + 1 : i + 4;
      const float first = y[m], second = y[n];
      y[m] = first * t.c[i] - second * t.s[i];
      y[n] = second * t.c[i] + first * t.s[i];
    }
  }
  x[0] = make_uint2(pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3]));
  x[1] = make_uint2(pack_bf16(y[4], y[5]), pack_bf16(y[6], y[7]));
}

// Dims d .. d + 3 of token `off` into a raw K record (fp_common.cuh: pairs 2 and
// 2 of one half of a word, in two neighbouring owners).
__device__ __forceinline__ void scatter_key_piece(uint8_t* rec, int off, int d, uint2 x) {
  const int owner = 32 * (off >> 4) + 4 * (off & 7) + ((d >> 1) & 3);
  uint8_t* at = rec + 16 * (kOwners * (d >> 4) + owner) + 4 * (2 * ((off >> 3) & 1) + ((d >> 3) & 1));
  *reinterpret_cast<uint32_t*>(at) = x.x;
  *reinterpret_cast<uint32_t*>(at + 16) = x.y;
}

// The same for a V record: every dim is a scalar of another owner's word.
__device__ __forceinline__ void scatter_value_piece(uint8_t* rec, int off, int d, uint2 x) {
  const int within = 2 * ((off >> 3) & 1) + (off & 1), c = (off >> 1) & 3;
  const uint32_t v[4] = {x.x & 0xffffu, x.x >> 16, x.y & 0xffffu, x.y >> 16};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int dim = d + i, owner = 32 * (dim >> 4) + 4 * (dim & 7) + c;
    uint8_t* at = rec + 16 * (kOwners * (off >> 4) + owner) + 2 * (4 * ((dim >> 3) & 1) + within);
    *reinterpret_cast<uint16_t*>(at) = (uint16_t)v[i];
  }
}

__device__ __forceinline__ int64_t token_position(const RotaryParams& p, int64_t token) {
  return p.positions_64 ? static_cast<const int64_t*>(p.positions)[token]
                        : (int64_t)static_cast<const int32_t*>(p.positions)[token];
}

// Up to kRows heads (head0 .. head0 + count - 1) of one token by a half warp, all
// loaded before the first is worked on.  `keep(r, x)` gets each result's pieces.
template <bool kInterleaved, int kRows, typename Keep>
__device__ __forceinline__ void rotate_rows(const RotaryParams& p, const HeadSet& set, int64_t token, int head0,
                                            int count, int a, int b, uint32_t half_mask, bool rotated,
                                            const Angles& t, const float (&w)[8], Keep&& keep) {
  const uint16_t* src = set.in + token * set.in_token + head0 * set.in_head;
  uint2 x[kRows][2];
#pragma unroll
  for (int r = 0; r < kRows; ++r)
    if (r < count) {
      x[r][0] = *reinterpret_cast<const uint2*>(src + r * set.in_head + a);
      x[r][1] = *reinterpret_cast<const uint2*>(src + r * set.in_head + b);
    }
#pragma unroll
  for (int r = 0; r < kRows; ++r)
    if (r < count) {
      norm_rotate<kInterleaved>(p, half_mask, set.weight != nullptr, w, t, rotated, x[r]);
      if (set.out != nullptr) {
        uint16_t* dst = set.out + token * set.out_token + (head0 + r) * set.out_head;
        *reinterpret_cast<uint2*>(dst + a) = x[r][0];
        *reinterpret_cast<uint2*>(dst + b) = x[r][1];
      }
      keep(r, x[r]);
    }
}

// A CTA takes sixteen consecutive tokens, one per half warp, and p.unit heads of
// one kind (query, key or, for an append, value) of each (blockIdx.y), kRows at
// a time.
template <bool kAppend, bool kInterleaved, int kRows>
__global__ void __launch_bounds__(kRowThreads, kRows == 4 ? 4 : 1) rotary_rows_kernel(RotaryParams p, StoreView v) {
  const int q_units = (p.q.heads + p.unit - 1) / p.unit, k_units = (p.k.heads + p.unit - 1) / p.unit;
  const int64_t token = (int64_t)blockIdx.x * (kRowThreads / 16) + (threadIdx.x >> 4);
  if (token >= p.tokens) return;  // uniform over the half warp
  const int unit = blockIdx.y;
  const int l = threadIdx.x & 15;
  const uint32_t half_mask = 0xffffu << (threadIdx.x & 16);
  const int kind = unit < q_units ? 0 : unit < q_units + k_units ? 1 : 2;
  const int head0 = p.unit * (unit - (kind == 0 ? 0 : kind == 1 ? q_units : q_units + k_units));
  const HeadSet& set = kind == 0 ? p.q : p.k;
  const int end = min(head0 + p.unit, set.heads);
  int a, b;
  piece_dims(l, p.rot_lanes, a, b);

  // Where the token's records are staged; -1: it has no place in the store.
  int staged = -1, off = 0;
  if (kAppend && kind != 0) {
    const int64_t slot = p.slots[token];
    if (slot >= 0 && (slot >> 7) < v.s.NB) {
      staged = v.s.wslot[slot >> 7];
      off = (int)(slot & 127);
    }
  }
  if (kAppend && kind == 2) {
    if (staged < 0) return;
    const uint16_t* src = p.value + token * p.v_token;
    for (int head = head0; head < end; ++head) {
      uint8_t* rec = v.staging(staged, p.layer, v.s.H + head);
      scatter_value_piece(rec, off, a, *reinterpret_cast<const uint2*>(src + head * p.v_head + a));
      scatter_value_piece(rec, off, b, *reinterpret_cast<const uint2*>(src + head * p.v_head + b));
    }
    return;
  }
  const Angles t = lane_angles<kInterleaved>(p, token_position(p, token), l, a, b);
  float w[8];
  lane_weights(p, set.weight, a, b, w);
  for (int head = head0; head < end; head += kRows)
    rotate_rows<kInterleaved, kRows>(p, set, token, head, end - head, a, b, half_mask, l < p.rot_lanes, t, w,
                                           [&](int r, const uint2(&x)[2]) {
                                             if (!kAppend || kind != 1 || staged < 0) return;
                                             uint8_t* rec = v.staging(staged, p.layer, head + r);
                                             scatter_key_piece(rec, off, a, x[0]);
                                             scatter_key_piece(rec, off, b, x[1]);
                                           });
}

// Append of many tokens.  A CTA takes sixteen consecutive input tokens, one per
// half warp, and either kQuerySlice query heads or kKvSlice KV heads of each
// (blockIdx.y).  Sixteen tokens at offsets 16 i .. 16 i + 15 of one block are a
// complete piece of its records (see hbm_kv.cu's token writer): such a group,
// where it starts at one of the CTA's tokens and is contiguous in the input, is
// normed and rotated into shared memory and leaves in 16-byte pieces of whole
// lines.  Tokens outside every such group go to their places one by one, by the
// CTA that has them among its sixteen.
// Slices of eight query heads against sixteen, 32 + 8 heads: prompts of 512 tokens
// 5.7 / 8.0 us, of 1,000 tokens 6.9 / 8.5 us, of 8,192 tokens 44.8 / 45.1 us; with
// four, two prompts of 8,192 tokens (32 + 32 heads) take 176 us against 164.
constexpr int kKvSlice = 4, kQuerySlice = 8;
// Up to here rotary_rows_kernel.  Rows against groups: 256 decode tokens (64 + 8
// heads) 7.8 / 9.6 us, 512 of them 14.9 / 12.3 us; one prompt of 256 tokens (32 +
// 8 heads) 4.2 / 5.1 us, of 400 tokens 6.4 / 5.8 us.  Two prompts of 8,192 tokens
// with 32 + 32 heads: 418 / 164 us, 0.89 of the measured copy bandwidth.
constexpr int kFewTokens = 384;
constexpr int kTileRow = 272;  // bytes of a staged token row (256 + pad)

template <bool kInterleaved>
__global__ void __launch_bounds__(kRowThreads, 4) append_kernel(RotaryParams p, StoreView v, int kv_slices) {
  __shared__ __align__(16) uint8_t tile[kKvSlice][2][16][kTileRow];
  __shared__ int tok_slot[16];  // staging slot of each token, -1: not stored
  __shared__ int tok_off[16];   // offset in its block
  __shared__ int tok_whole[16];  // covered by a complete group
  __shared__ int group_start;    // token (of the sixteen) at which a complete group starts, -1: none
  const int tid = threadIdx.x, mine = tid >> 4, l = tid & 15;
  const int64_t t0 = (int64_t)blockIdx.x * 16;
  const uint32_t half_mask = 0xffffu << (tid & 16);
  int a, b;
  piece_dims(l, p.rot_lanes, a, b);

  if ((int)blockIdx.y >= kv_slices) {
    const int64_t token = t0 + mine;
    if (token >= p.tokens) return;
    const Angles t = lane_angles<kInterleaved>(p, token_position(p, token), l, a, b);
    float w[8];
    lane_weights(p, p.q.weight, a, b, w);
    const int head0 = ((int)blockIdx.y - kv_slices) * kQuerySlice, end = min(head0 + kQuerySlice, p.q.heads);
    for (int head = head0; head < end; head += 4)
      rotate_rows<kInterleaved, 4>(p, p.q, token, head, end - head, a, b, half_mask, l < p.rot_lanes, t, w,
                                             [](int, const uint2(&)[2]) {});
    return;
  }

  const int head0 = (int)blockIdx.y * kKvSlice, heads = min(kKvSlice, v.s.H - head0);
  if (tid < 32) {
    // Slots of the inputs t0 - 16 .. t0 + 31; bit i of `follows`: input t0 - 16 + i
    // is the next slot of the same group of sixteen as the one before it.
    const auto slot_at = [&](int64_t t) { return t >= 0 && t < p.tokens ? p.slots[t] : (int64_t)-2; };
    const int64_t early = slot_at(t0 - 16 + tid), late = slot_at(t0 + 16 + (tid & 15));
    int64_t before_early = __shfl_up_sync(0xffffffffu, early, 1);
    int64_t before_late = __shfl_up_sync(0xffffffffu, late, 1);
    const int64_t last_early = __shfl_sync(0xffffffffu, early, 31);
    if (tid == 0) {
      before_early = -2;
      before_late = last_early;
    }
    const auto next = [](int64_t slot, int64_t before) { return before >= 0 && slot == before + 1 && (slot & 15) != 0; };
    const uint64_t follows = (uint64_t)__ballot_sync(0xffffffffu, next(early, before_early)) |
                             ((uint64_t)__ballot_sync(0xffffffffu, tid < 16 && next(late, before_late)) << 32);
    const int64_t slot = __shfl_sync(0xffffffffu, early, 16 + (tid & 15));  // of token tid
    const int off = (int)(slot & 127);
    int w = -1;
    bool whole = false;
    if (slot >= 0 && (slot >> 7) < v.s.NB) {
      w = v.s.wslot[slot >> 7];
      const int first = 16 + (tid & 15) - (off & 15);  // the group's first input, in the window
      whole = w >= 0 && first >= 0 && ((follows >> first) & 0xfffeu) == 0xfffeu;
    }
    const uint32_t starts = __ballot_sync(0xffffffffu, tid < 16 && whole && (off & 15) == 0);
    if (tid < 16) {
      tok_slot[tid] = w;
      tok_off[tid] = off;
      tok_whole[tid] = whole;
    }
    if (tid == 0) group_start = __ffs(starts) - 1;
  }
  __syncthreads();

  float w[8];
  lane_weights(p, p.k.weight, a, b, w);
  if (tok_slot[mine] >= 0 ? !tok_whole[mine] : t0 + mine < p.tokens) {
    // Keys of tokens that are not stored are rotated all the same.
    const int64_t token = t0 + mine;
    const int staged = tok_slot[mine], off = tok_off[mine];
    const Angles t = lane_angles<kInterleaved>(p, token_position(p, token), l, a, b);
    const uint16_t* src = p.value + token * p.v_token;
    uint2 val[kKvSlice][2];
#pragma unroll
    for (int h = 0; h < kKvSlice; ++h)
      if (h < heads) {
        val[h][0] = *reinterpret_cast<const uint2*>(src + (head0 + h) * p.v_head + a);
        val[h][1] = *reinterpret_cast<const uint2*>(src + (head0 + h) * p.v_head + b);
      }
    rotate_rows<kInterleaved, kKvSlice>(p, p.k, token, head0, heads, a, b, half_mask, l < p.rot_lanes, t, w,
                                        [&](int h, const uint2(&x)[2]) {
                                          if (staged < 0) return;
                                          uint8_t* rec = v.staging(staged, p.layer, head0 + h);
                                          scatter_key_piece(rec, off, a, x[0]);
                                          scatter_key_piece(rec, off, b, x[1]);
                                          rec = v.staging(staged, p.layer, v.s.H + head0 + h);
                                          scatter_value_piece(rec, off, a, val[h][0]);
                                          scatter_value_piece(rec, off, b, val[h][1]);
                                        });
  }
  if (group_start < 0) return;

  // The group's tokens are first .. first + 15, one per half warp.
  const int64_t token = t0 + group_start + mine;
  const int staged = tok_slot[group_start], group = tok_off[group_start] >> 4;
#pragma unroll
  for (int h = 0; h < kKvSlice; ++h)
    if (h < heads)
      async_copy16(&tile[h][1][mine][16 * l], p.value + token * p.v_token + (head0 + h) * p.v_head + 8 * l);
  const Angles t = lane_angles<kInterleaved>(p, token_position(p, token), l, a, b);
  rotate_rows<kInterleaved, kKvSlice>(p, p.k, token, head0, heads, a, b, half_mask, l < p.rot_lanes, t, w,
                                      [&](int h, const uint2(&x)[2]) {
                                        *reinterpret_cast<uint2*>(&tile[h][0][mine][2 * a]) = x[0];
                                        *reinterpret_cast<uint2*>(&tile[h][0][mine][2 * b]) = x[1];
                                      });
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();
#pragma unroll
  for (int h = 0; h < kKvSlice; ++h) {
    if (h >= heads) break;
    // K: thread (st, g, c) owns word st of owner 32 group + 4 g + c: tokens g and
    // g + 8, dim pairs 16 st + 2 c and + 8.
    // V: thread = owner (st, g, c) of word plane `group`: dims 16 st + g and + 8,
    // tokens 2 c, 2 c + 1 and + 8.
    const int st = tid >> 5, g = (tid >> 2) & 7, c = tid & 3;
    const auto k_pair = [&](int tok, int dim) { return *reinterpret_cast<const uint32_t*>(&tile[h][0][tok][2 * dim]); };
    const auto v_one = [&](int tok, int dim) { return (uint32_t) * reinterpret_cast<const uint16_t*>(&tile[h][1][tok][2 * dim]); };
    const auto v_pair = [&](int tok, int dim) { return v_one(tok, dim) | (v_one(tok + 1, dim) << 16); };
    *reinterpret_cast<uint4*>(v.staging(staged, p.layer, head0 + h) + 16 * (kOwners * st + 32 * group + (tid & 31))) =
        make_uint4(k_pair(g, 16 * st + 2 * c), k_pair(g, 16 * st + 8 + 2 * c), k_pair(g + 8, 16 * st + 2 * c),
                   k_pair(g + 8, 16 * st + 8 + 2 * c));
    *reinterpret_cast<uint4*>(v.staging(staged, p.layer, v.s.H + head0 + h) + 16 * (kOwners * group + tid)) =
        make_uint4(v_pair(2 * c, 16 * st + g), v_pair(8 + 2 * c, 16 * st + g), v_pair(2 * c, 16 * st + 8 + g),
                   v_pair(8 + 2 * c, 16 * st + 8 + g));
  }
}

bool rows_aligned(const void* base, int64_t token_stride, int64_t head_stride) {
  return reinterpret_cast<uintptr_t>(base) % 16 == 0 && token_stride % 8 == 0 && head_stride % 8 == 0;
}

// Checks what both entry points take and fills the shared parameters.
int rotary_params(RotaryParams& p, const fp_heads* q, const fp_heads* k, const void* q_weight,
                  const void* k_weight, int32_t weights_f32, const void* positions, int32_t positions_64,
                  int64_t tokens, const fp_rotary* rotary, float eps) {
  FP_REQUIRE(q && k && rotary && rotary->turns && positions, "null rotary argument");
  FP_REQUIRE(tokens > 0 && tokens < (1LL << 31), "bad token count %lld", (long long)tokens);
  FP_REQUIRE(rotary->rot_dim >= 0 && rotary->rot_dim <= 128 && rotary->rot_dim % 8 == 0,
             "rotated dims %d must be a multiple of 8 up to 128", rotary->rot_dim);
  FP_REQUIRE(q->heads >= 0 && k->heads >= 0 && q->heads <= 65535 && k->heads <= 65535,
             "bad head counts %d / %d", q->heads, k->heads);
  const fp_heads* const sets[2] = {q, k};
  for (const fp_heads* s : sets) {
    if (s->heads == 0) continue;
    FP_REQUIRE(s->in, "null query / key");
    FP_REQUIRE(rows_aligned(s->in, s->in_token, s->in_head) &&
                   (!s->out || rows_aligned(s->out, s->out_token, s->out_head)),
               "query / key rows must be 16-byte aligned");
  }
  const auto fill = [](HeadSet& to, const fp_heads* s, const void* weight) {
    to.in = static_cast<const uint16_t*>(s->in);
    to.out = static_cast<uint16_t*>(s->out);
    to.in_token = s->in_token;
    to.in_head = s->in_head;
    to.out_token = s->out_token;
    to.out_head = s->out_head;
    to.weight = weight;
    to.heads = s->heads;
  };
  fill(p.q, q, q_weight);
  fill(p.k, k, k_weight);
  p.value = nullptr;
  p.v_token = p.v_head = 0;
  p.slots = nullptr;
  p.positions = positions;
  p.turns = rotary->turns;
  p.tokens = tokens;
  p.positions_64 = positions_64;
  p.weights_f32 = weights_f32;
  p.rot_lanes = rotary->rot_dim / 8;
  p.layer = 0;
  p.factor = rotary->factor;
  p.eps = eps;
  return FP_OK;
}

// Launches rotary_rows_kernel: two heads per half warp where latency counts,
// sixteen (a token's angles are made once for all of them) from kManyRows on.
// With 40 heads, two against sixteen: 1,024 tokens 7.7 / 9.5 us, 2,048 tokens 15.1
// / 14.6 us, 4,096 tokens 26.4 / 21.8 us, 16,384 tokens (72 heads) 149 / 102 us,
// which is 0.91 of the measured copy bandwidth.
template <bool kAppend>
int launch_rows(RotaryParams& p, const StoreView& v, bool interleaved, cudaStream_t stream) {
  // An append has too few tokens here (kFewTokens) for the second form.
  const bool many = !kAppend && p.tokens * (p.q.heads + p.k.heads) >= kManyRows;
  p.unit = many ? 16 : 2;
  const int64_t units = (p.q.heads + p.unit - 1) / p.unit + (kAppend ? 2LL : 1LL) * ((p.k.heads + p.unit - 1) / p.unit);
  FP_REQUIRE(units <= 65535, "too many heads (%d + %d)", p.q.heads, p.k.heads);
  auto kernel = interleaved ? rotary_rows_kernel<kAppend, true, 2> : rotary_rows_kernel<kAppend, false, 2>;
  if constexpr (!kAppend)
    if (many) kernel = interleaved ? rotary_rows_kernel<false, true, 4> : rotary_rows_kernel<false, false, 4>;
  constexpr int per_block = kRowThreads / 16;
  kernel<<<dim3((unsigned)((p.tokens + per_block - 1) / per_block), (unsigned)units), kRowThreads, 0, stream>>>(p, v);
  FP_LAUNCH_CHECK("rotary_rows_kernel");
  return FP_OK;
}

}  // namespace
}  // namespace fpb

using namespace fpb;

extern "C" {

int fp_norm_rotary(const fp_heads* q, const fp_heads* k, const void* q_weight, const void* k_weight,
                   int32_t weights_f32, const void* positions, int32_t positions_64, int64_t tokens,
                   const fp_rotary* rotary, float eps, void* stream) {
  if (tokens == 0) return FP_OK;
  RotaryParams p;
  if (int rc = rotary_params(p, q, k, q_weight, k_weight, weights_f32, positions, positions_64, tokens,
                             rotary, eps))
    return rc;
  FP_REQUIRE((p.q.heads == 0 || p.q.out) && (p.k.heads == 0 || p.k.out), "null query / key result");
  if (p.q.heads + p.k.heads == 0) return FP_OK;
  return launch_rows<false>(p, StoreView{}, rotary->interleaved != 0, (cudaStream_t)stream);
}

int fp_hbm_append(const fp_store* store, const fp_heads* q, const fp_heads* k, const void* value,
                  int64_t v_stride0, int64_t v_stride1, const void* q_weight, const void* k_weight,
                  int32_t weights_f32, const void* positions, int32_t positions_64,
                  const int64_t* slot_mapping, int64_t tokens, const fp_rotary* rotary, float eps,
                  int32_t layer, void* stream) {
  if (int rc = check_store(store)) return rc;
  if (tokens == 0) return FP_OK;
  RotaryParams p;
  if (int rc = rotary_params(p, q, k, q_weight, k_weight, weights_f32, positions, positions_64, tokens,
                             rotary, eps))
    return rc;
  FP_REQUIRE(value && slot_mapping, "null value / slot_mapping");
  FP_REQUIRE(layer >= 0 && layer < store->L, "layer %d out of range", layer);
  FP_REQUIRE(k->heads == store->H, "%d key heads for a store of %d", k->heads, store->H);
  FP_REQUIRE(p.q.heads == 0 || p.q.out, "null query result");
  FP_REQUIRE(rows_aligned(value, v_stride0, v_stride1), "value rows must be 16-byte aligned");
  p.value = static_cast<const uint16_t*>(value);
  p.v_token = v_stride0;
  p.v_head = v_stride1;
  p.slots = slot_mapping;
  p.layer = layer;
  if (tokens > kFewTokens) {
    const int kv_slices = (store->H + kKvSlice - 1) / kKvSlice, q_slices = (p.q.heads + kQuerySlice - 1) / kQuerySlice;
    const auto kernel = rotary->interleaved ? append_kernel<true> : append_kernel<false>;
    kernel<<<dim3((unsigned)((tokens + 15) / 16), (unsigned)(kv_slices + q_slices)), kRowThreads, 0,
             (cudaStream_t)stream>>>(p, StoreView{*store}, kv_slices);
    FP_LAUNCH_CHECK("append_kernel");
    return FP_OK;
  }
  return launch_rows<true>(p, StoreView{*store}, rotary->interleaved != 0, (cudaStream_t)stream);
}

}  // extern "C"
