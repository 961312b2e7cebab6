// RMS norm of query and key heads with the position rotation in the same pass,
// alone (fp_norm_rotary) and on the way into the store (fp_hbm_append), for
// sm_100a.
//
//   y      = x * rsqrt(mean(x^2) + eps) * w            (per head; left out without weights)
//   (a, b) = pair (y_i, y_(i + rot/2)) or (y_2i, y_(2i+1)) of the first `rot` dims
//   (a, b) -> factor * (a cos t - b sin t, b cos t + a sin t),  t = position * frequency_i
//
// Everything between the load and the one rounding of the result to BF16 is
// FP32.  The angle is reduced exactly: a frequency is held in turns per token
// as a 64-bit binary fraction, so position * frequency modulo one turn is one
// wrapping 64-bit multiplication (error: position * 2^-65 turns, at any
// position), and sine and cosine of the remaining half turn come from the
// special-function unit, whose absolute error of about 2^-21 there is a 4000th
// of the half step of the BF16 result.  No table of angles is read.
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
constexpr int kRowsPerUnit = 4;  // heads of one token that a half warp loads together

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
  int positions_64, weights_f32, rot_lanes, layer;
  float factor, eps;
};

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

// One half warp per unit: up to kRowsPerUnit heads of one kind (query, key or,
// for an append, value) of one token.
template <bool kAppend, bool kInterleaved>
__global__ void __launch_bounds__(kRowThreads) rotary_rows_kernel(RotaryParams p, StoreView v) {
  const int q_units = (p.q.heads + kRowsPerUnit - 1) / kRowsPerUnit;
  const int k_units = (p.k.heads + kRowsPerUnit - 1) / kRowsPerUnit;
  const int units = q_units + k_units * (kAppend ? 2 : 1);
  const int64_t at = (int64_t)blockIdx.x * (kRowThreads / 16) + (threadIdx.x >> 4);
  const int64_t token = at / units;
  if (token >= p.tokens) return;  // uniform over the half warp
  const int unit = (int)(at % units);
  const int l = threadIdx.x & 15;
  const uint32_t half_mask = 0xffffu << (threadIdx.x & 16);
  const int kind = unit < q_units ? 0 : unit < q_units + k_units ? 1 : 2;
  const int head0 = kRowsPerUnit * (unit - (kind == 0 ? 0 : kind == 1 ? q_units : q_units + k_units));
  const HeadSet& set = kind == 0 ? p.q : p.k;
  const int count = min(kRowsPerUnit, set.heads - head0);
  int a, b;
  piece_dims(l, p.rot_lanes, a, b);

  const uint16_t* src = kind == 2 ? p.value + token * p.v_token + head0 * p.v_head
                                  : set.in + token * set.in_token + head0 * set.in_head;
  const int64_t step = kind == 2 ? p.v_head : set.in_head;
  uint2 x[kRowsPerUnit][2];
#pragma unroll
  for (int r = 0; r < kRowsPerUnit; ++r)
    if (r < count) {
      x[r][0] = *reinterpret_cast<const uint2*>(src + r * step + a);
      x[r][1] = *reinterpret_cast<const uint2*>(src + r * step + b);
    }

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
    if (staged >= 0) {
#pragma unroll
      for (int r = 0; r < kRowsPerUnit; ++r)
        if (r < count) {
          uint8_t* rec = v.staging(staged, p.layer, v.s.H + head0 + r);
          scatter_value_piece(rec, off, a, x[r][0]);
          scatter_value_piece(rec, off, b, x[r][1]);
        }
    }
    return;
  }
  const int64_t position = p.positions_64 ? static_cast<const int64_t*>(p.positions)[token]
                                          : (int64_t)static_cast<const int32_t*>(p.positions)[token];
  const Angles t = lane_angles<kInterleaved>(p, position, l, a, b);
  const bool norm = set.weight != nullptr, rotated = l < p.rot_lanes;
  float w[8];
  lane_weights(p, set.weight, a, b, w);
#pragma unroll
  for (int r = 0; r < kRowsPerUnit; ++r)
    if (r < count) {
      norm_rotate<kInterleaved>(p, half_mask, norm, w, t, rotated, x[r]);
      if (set.out != nullptr) {
        uint16_t* dst = set.out + token * set.out_token + (head0 + r) * set.out_head;
        *reinterpret_cast<uint2*>(dst + a) = x[r][0];
        *reinterpret_cast<uint2*>(dst + b) = x[r][1];
      }
      if (kAppend && kind == 1 && staged >= 0) {
        uint8_t* rec = v.staging(staged, p.layer, head0 + r);
        scatter_key_piece(rec, off, a, x[r][0]);
        scatter_key_piece(rec, off, b, x[r][1]);
      }
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

// Blocks of rotary_rows_kernel, refused beyond the grid's limit.
int row_blocks(const RotaryParams& p, int kinds_of_k, unsigned& blocks) {
  const int64_t units = (p.q.heads + kRowsPerUnit - 1) / kRowsPerUnit +
                        (int64_t)kinds_of_k * ((p.k.heads + kRowsPerUnit - 1) / kRowsPerUnit);
  const int64_t n = (p.tokens * units + kRowThreads / 16 - 1) / (kRowThreads / 16);
  FP_REQUIRE(n < (1LL << 31), "too many heads (%lld tokens)", (long long)p.tokens);
  blocks = (unsigned)n;
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
  unsigned blocks = 0;
  if (int rc = row_blocks(p, 1, blocks)) return rc;
  const auto kernel = rotary->interleaved ? rotary_rows_kernel<false, true> : rotary_rows_kernel<false, false>;
  kernel<<<blocks, kRowThreads, 0, (cudaStream_t)stream>>>(p, StoreView{});
  FP_LAUNCH_CHECK("rotary_rows_kernel");
  return FP_OK;
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
  unsigned blocks = 0;
  if (int rc = row_blocks(p, 2, blocks)) return rc;
  const auto kernel = rotary->interleaved ? rotary_rows_kernel<true, true> : rotary_rows_kernel<true, false>;
  kernel<<<blocks, kRowThreads, 0, (cudaStream_t)stream>>>(p, StoreView{*store});
  FP_LAUNCH_CHECK("rotary_rows_kernel");
  return FP_OK;
}

}  // extern "C"
