// The per-head norm and rotation of a decoder's queries and keys on gfx950, to rows in 16 bits or with the keys and
// values into the 4-bit cache of kv4.hip.
//
// Per row and head, x of D channels, with norm: y = x r w, r = 1 / sqrt(mean(x^2) + eps). Then the pairs (a, b)
// of the first `rotary` channels, (c, c + rotary / 2) or interleaved (2 c, 2 c + 1), turn by the row's
// position: (a cos - b sin, b cos + a sin). With x' the other channel of a pair, w' its weight and s = -sin for
// the first and sin for the second channel of one, the result is r (x (w cos) + x' (w' s)): the two factors are a
// token's for all its heads, and what passes between lanes is x as it was read, two channels to a register.
//
// Queries are computed in f32 and rounded once, but for rows whose squares f32 does not hold, which are as the keys.
// Keys are computed in f64, so that the 16 bits that they are rounded to are the definition's, whatever the order of
// its sums: a bit of one of them is a step of a code or of a whole row's scale in the cache. It costs nothing that is
// seen: there are few key heads and memory bounds the kernel.
//
// D/8 lanes of 8 channels hold a row, so a wave holds one head of 512/D tokens and takes `per` heads of the same
// tokens one after the other.
#include <algorithm>
#include <type_traits>

#include "kv4_row.hpp"

namespace h3 {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;

struct QkArgs {
  const void *q, *k, *v;
  const float *q_weight, *k_weight, *cos_t, *sin_t;
  const int32_t *positions, *slots;
  void *q_out, *k_out;
  uint8_t* cache;
  uint32_t tokens, heads, kv_heads, rotary, position_limit;
  uint32_t q_stride, k_stride, v_stride, q_out_stride, k_out_stride;
  uint32_t page_shift;
  uint32_t units, per;  // heads of q, of k and (cached) of v, one after the other; how many a wave takes
  uint64_t slot_limit;
  float eps;
};

// The lane's place: its token's row, and 8 channels of every head.
struct Lane {
  uint32_t token, first;   // first of the channels
  int32_t position, slot;  // -1: none
  int other;               // the lane that holds the pairs' other channels, in bytes for a permutation
};

__device__ __forceinline__ float channel(const uint32_t (&w)[4], int i, bool bf16) {
  const uint32_t bits = i & 1 ? w[i / 2] >> 16 : w[i / 2] & 0xffffu;
  return bf16 ? widen<true>(bits) : widen<false>(bits);
}

// The other channels of the pairs that eight channels belong to.
template <bool kPairs>
__device__ __forceinline__ void others(const uint32_t (&w)[4], int lane, uint32_t (&o)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    o[i] = kPairs ? (w[i] >> 16) | (w[i] << 16) : (uint32_t)__builtin_amdgcn_ds_bpermute(lane, (int)w[i]);
}

template <int kCtrl>
__device__ __forceinline__ double dpp64(double v) {
  const uint2 x = __builtin_bit_cast(uint2, v);
  const uint2 y = {(uint32_t)__builtin_amdgcn_mov_dpp((int)x.x, kCtrl, 0xF, 0xF, true),
                   (uint32_t)__builtin_amdgcn_mov_dpp((int)x.y, kCtrl, 0xF, 0xF, true)};
  return __builtin_bit_cast(double, y);
}
// The sum over the D/8 lanes of a row.
template <int D>
__device__ __forceinline__ float row_sum(float v) {
  v += dpp<0xB1>(v);
  v += dpp<0x4E>(v);
  v += dpp<0x141>(v);
  if constexpr (D == 128) v += dpp<0x140>(v);
  return v;
}
template <int D>
__device__ __forceinline__ double row_sum(double v) {
  v += dpp64<0xB1>(v);
  v += dpp64<0x4E>(v);
  v += dpp64<0x141>(v);
  if constexpr (D == 128) v += dpp64<0x140>(v);
  return v;
}

// 1 / sqrt(x): the instruction's, to an ulp; in f64 with two steps of Newton's from its 2^-23 or so. The f32 one takes
// subnormal numbers for 0: they count as the least normal one, since such a row is zeros (f16), of which any finite
// root makes zeros, or is normed again in 64 bits (bf16).
__device__ __forceinline__ float inverse_root(float x) {
  return __builtin_amdgcn_rsqf(x > 0.0f ? fmaxf(x, 0x1p-126f) : x);
}
__device__ __forceinline__ double inverse_root(double x) {
  const double first = __builtin_amdgcn_rsq(x);
  double r = first;
#pragma unroll
  for (int i = 0; i < 2; ++i) r = fma(r * 0.5, fma(-x * r, r, 1.0), r);
  return first == 0.0 ? 0.0 : r;  // x infinite
}

// An f64 value rounded once to the element type: to odd in f32 first (toward zero, the last bit set where that lost
// something), which the second rounding, of at least two bits fewer, cannot mistake for a tie.
template <bool kBf16>
__device__ __forceinline__ uint32_t narrow64(double x) {
  const float f = (float)x;
  const double back = f;
  uint32_t bits = __float_as_uint(f);
  if (back != x) bits = (bits - (fabs(back) > fabs(x) ? 1u : 0u)) | 1u;
  return narrow<kBf16>(__uint_as_float(bits));
}

// Eight f32, 32 bytes on: of a weight, or of a token's cos or sin.
struct Eight {
  float v[8];
};
__device__ __forceinline__ Eight eight(const float* p) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  return {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
}

// What a token's rows of one weight are multiplied by: own = w cos, other = w' (-sin or sin); past the rotated
// channels w and -0, which the other channel is not to meet (an infinity would make a NaN of it): adding
// 0 times -0 changes nothing, not a zero's sign either.
template <typename T>
struct Factors {
  T own[8], other[8];
  bool turned;
};
template <bool kPairs, bool kNorm, typename T>
__device__ __forceinline__ Factors<T> factors(const QkArgs& a, const Lane& l, const float* weight) {
  Factors<T> f;
  const uint32_t half = a.rotary / 2;
  const bool turned = f.turned = l.first < a.rotary, second = !kPairs && turned && l.first >= half;
  Eight w, v;
  if constexpr (kNorm) {
    w = eight(weight + l.first);
    v = kPairs || !turned ? w : eight(weight + (second ? l.first - half : l.first + half));
  }
  const size_t at = (size_t)(uint32_t)max(l.position, 0) * half;
  Eight c = {}, s = {};
  if constexpr (kPairs) {
    if (turned) {
      const float4 x = *reinterpret_cast<const float4*>(a.cos_t + at + l.first / 2);
      const float4 y = *reinterpret_cast<const float4*>(a.sin_t + at + l.first / 2);
      c = {x.x, x.x, x.y, x.y, x.z, x.z, x.w, x.w};
      s = {-y.x, y.x, -y.y, y.y, -y.z, y.z, -y.w, y.w};
    }
  } else if (turned) {
    c = eight(a.cos_t + at + (second ? l.first - half : l.first));
    s = eight(a.sin_t + at + (second ? l.first - half : l.first));
#pragma unroll
    for (int i = 0; i < 8; ++i) s.v[i] = second ? s.v[i] : -s.v[i];
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const T x = kNorm ? (T)w.v[i] : (T)1, y = kNorm ? (T)v.v[kPairs ? i ^ 1 : i] : (T)1;
    f.own[i] = turned ? x * (T)c.v[i] : x;
    f.other[i] = turned ? y * (T)s.v[i] : (T)-0.0f;
  }
  return f;
}

// mean(x^2) + eps of a row, in T.
template <int D, bool kBf16, typename T>
__device__ __forceinline__ T mean_square(const uint32_t (&w)[4], float eps) {
  T sum = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const T x = channel(w, i, kBf16);
    sum = fma(x, x, sum);
  }
  return fma(row_sum<D>(sum), (T)(1.0 / D), (T)eps);
}

// A channel before its rounding, and rounded.
template <bool kBf16, typename T, typename F>
__device__ __forceinline__ uint32_t turned_channel(const uint32_t (&w)[4], const uint32_t (&o)[4], int i,
                                                   const Factors<F>& f, T r) {
  const T y = fma((T)channel(w, i, kBf16), (T)f.own[i], (T)channel(o, i, kBf16) * (T)f.other[i]) * r;
  if constexpr (sizeof(T) == 8)
    return narrow64<kBf16>(y);
  else
    return narrow<kBf16>(y);
}

// Mean squares that f32's sums are exact enough for: what is lost of smaller squares is below 2^-119, and none of these
// overflows.
constexpr float kLeastSquare = 0x1p-80f, kMostSquare = 0x1p120f;

// A row's eight channels in 16 bits.
template <int D, bool kBf16, bool kPairs, bool kNorm, typename T>
__device__ __forceinline__ uint4 turn(const QkArgs& a, const Lane& l, const Factors<T>& f, uint4 raw) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  uint32_t o[4];
  others<kPairs>(w, l.other, o);
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = f.turned ? o[i] : 0;
  T square = 1, r = 1;
  if constexpr (kNorm) {
    square = mean_square<D, kBf16, T>(w, a.eps);
    r = inverse_root(square);
  }
  uint32_t out[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) out[i] = turned_channel<kBf16>(w, o, i, f, r);
  if constexpr (kNorm && kBf16 && sizeof(T) == 4) {
    if (!(square >= kLeastSquare && square < kMostSquare)) {  // (a row's lanes are of one mind)
      const double r64 = inverse_root(mean_square<D, kBf16, double>(w, a.eps));
#pragma unroll
      for (int i = 0; i < 8; ++i) out[i] = turned_channel<kBf16>(w, o, i, f, r64);
    }
  }
  return {out[0] | out[1] << 16, out[2] | out[3] << 16, out[4] | out[5] << 16, out[6] | out[7] << 16};
}

// Eight channels of a row of K (part 0) or V into their slot.
template <int D, bool kBf16>
__device__ __forceinline__ void put(const QkArgs& a, const Lane& l, uint32_t head, uint32_t part, uint4 x) {
  const uint2 row = quantize<D, kBf16>(x);
  if (l.slot < 0) return;
  const Slot<D> at = slot_at<D>(a.page_shift, a.kv_heads, (uint32_t)l.slot, head);
  *reinterpret_cast<uint32_t*>(a.cache + at.codes + part * at.half + l.first / 2) = row.y;
  if (l.first == 0) *reinterpret_cast<uint32_t*>(a.cache + at.words + part * 4 * at.tokens) = row.x;
}

// Heads from .. to - 1 (to may be less) of the token's queries, keys or values, kHeads at a time: the next ones'
// rows are under way while these are computed.
enum Kind { kQuery, kKey, kValue };
constexpr uint32_t kHeads = 4;
template <int D, bool kBf16, bool kPairs, bool kNorm, bool kCached, bool kOnce, Kind kKind>
__device__ __forceinline__ void units(const QkArgs& a, const Lane& l, uint32_t from, uint32_t to) {
  if ((int)from >= (int)to) return;
  const void* rows = kKind == kQuery ? a.q : kKind == kKey ? a.k : a.v;
  const uint32_t stride = kKind == kQuery ? a.q_stride : kKind == kKey ? a.k_stride : a.v_stride;
  const size_t row = (size_t)l.token * stride + l.first;
  uint4 x[kHeads], next[kHeads];
  const auto load = [&](uint32_t u, uint4 (&to_x)[kHeads]) {
#pragma unroll
    for (uint32_t i = 0; i < kHeads; ++i) to_x[i] = load_row<kOnce>(rows, row + min(u + i, to - 1) * D);
  };
  load(from, x);
  using T = std::conditional_t<kKind == kKey, double, float>;
  Factors<T> f;
  if constexpr (kKind != kValue)
    f = factors<kPairs, kNorm, T>(a, l, kKind == kQuery ? a.q_weight : a.k_weight);
  for (uint32_t u = from; u < to; u += kHeads) {
    if (u + kHeads < to) load(u + kHeads, next);
#pragma unroll
    for (uint32_t i = 0; i < kHeads; ++i) {
      if (u + i >= to) break;
      uint4 y = x[i];
      if constexpr (kKind != kValue) y = turn<D, kBf16, kPairs, kNorm>(a, l, f, y);
      const uint32_t head = u + i;
      if constexpr (kKind == kQuery) {
        if (l.position >= 0) store_row<kOnce>(a.q_out, (size_t)l.token * a.q_out_stride + head * D + l.first, y);
      } else if constexpr (kCached) {
        put<D, kBf16>(a, l, head, kKind == kKey ? 0 : 1, y);
      } else {
        if (l.position >= 0) store_row<kOnce>(a.k_out, (size_t)l.token * a.k_out_stride + head * D + l.first, y);
      }
    }
#pragma unroll
    for (uint32_t i = 0; i < kHeads; ++i) x[i] = next[i];
  }
}

template <int D, bool kBf16, bool kPairs, bool kNorm, bool kCached, bool kOnce>
__global__ __launch_bounds__(kThreads) void k_qk_norm_rope(QkArgs a) {
  constexpr uint32_t kLanes = D / 8, kTokens = 64 / kLanes;
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t from = (blockIdx.y * kWaves + wave) * a.per, to = min(from + a.per, a.units);
  if (from >= a.units) return;
  Lane l;
  const uint32_t at = blockIdx.x * kTokens + lane / kLanes;
  l.token = min(at, a.tokens - 1);  // the last row stands for the rows past it: their loads need no branch
  l.first = lane % kLanes * 8;
  const int32_t position = at < a.tokens ? a.positions[at] : -1;
  l.position = (uint32_t)position < a.position_limit ? position : -1;
  l.slot = -1;
  if constexpr (kCached) {
    const int32_t slot = a.slots[l.token];
    if (l.position >= 0 && (uint64_t)(uint32_t)slot < a.slot_limit) l.slot = slot;
  }
  const uint32_t half = a.rotary / 16;  // lanes of the pairs' first channels
  const uint32_t in_row = lane % kLanes;
  l.other = 4 * (int)(in_row < half ? lane + half : in_row < 2 * half ? lane - half : lane);

  const uint32_t k_end = a.heads + a.kv_heads;
  units<D, kBf16, kPairs, kNorm, kCached, kOnce, kQuery>(a, l, from, min(to, a.heads));
  units<D, kBf16, kPairs, kNorm, kCached, kOnce, kKey>(a, l, max(from, a.heads) - a.heads, min(to, k_end) - a.heads);
  if constexpr (kCached)
    units<D, kBf16, kPairs, kNorm, kCached, kOnce, kValue>(a, l, max(from, k_end) - k_end, to - k_end);
}

template <int D, bool kBf16, bool kPairs, bool kNorm, bool kOnce>
void launch_once(const QkArgs& a, dim3 grid, hipStream_t stream) {
  if (a.cache)
    hipLaunchKernelGGL((k_qk_norm_rope<D, kBf16, kPairs, kNorm, true, kOnce>), grid, dim3(kThreads), 0, stream, a);
  else
    hipLaunchKernelGGL((k_qk_norm_rope<D, kBf16, kPairs, kNorm, false, kOnce>), grid, dim3(kThreads), 0, stream, a);
}

// As many heads a wave as leave 16 waves to each compute unit: a token's factors and position serve them all, and their
// rows are under way together, while few rows want all the waves that there are. One head, as many, and a
// quarter of a token's (32 + 8 + 8 heads of 128 channels, into the cache): 256 tokens 4.3, 4.3 and 9.6 us,
// 1,024 9.2, 7.7 and 10.4, 4,096 31, 20 and 20, 31,104 311, 118 and 118 (705 MB: 6.0 TB/s, where a copy reaches 5.2).
// More than one (from 683 tokens of those heads on): past the caches, where the rows of such a call are seldom met again.
// Through them and past, alone | behind the write of its rows | and before a prompt's attention that reads q_out: 768
// tokens 8.1 and 7.4 | 12.5 and 11.7 | 32.8 and 31.9 us; 1,024 9.5 and 9.1 | 14.5 and 13.5 | 42.5 and 41.7; 4,096 21.7
// and 21.5 | 43.6 and 34.5 | 201 and 200; 8,192 43 and 38 | 83 and 77 | 655 and 655; 31,104 132 and 118. Before the
// attention of as many single tokens of 512 keys it loses (1,024: 125 and 129), a batch that is rarer than such prompts.
// Below, where each wave has one head: 512 tokens 7.3 and 7.7 alone.
template <int D, bool kBf16, bool kPairs, bool kNorm>
hipError_t launch(QkArgs a, hipStream_t stream) {
  constexpr uint32_t kTokens = 512 / D;
  const uint32_t groups = (a.tokens + kTokens - 1) / kTokens;
  const uint64_t waves = (uint64_t)groups * a.units;  // if each took one head
  a.per = (uint32_t)std::min<uint64_t>(std::max<uint64_t>(waves / (16 * device_cus()), 1),
                                       (a.units + kWaves - 1) / kWaves);
  const dim3 grid(groups, (a.units + kWaves * a.per - 1) / (kWaves * a.per));
  if (a.per > 1)
    launch_once<D, kBf16, kPairs, kNorm, true>(a, grid, stream);
  else
    launch_once<D, kBf16, kPairs, kNorm, false>(a, grid, stream);
  return hipGetLastError();
}

template <int D, bool kBf16>
hipError_t launch_kind(const QkArgs& a, const h3_qk_cfg& cfg, hipStream_t stream) {
  if (cfg.interleaved)
    return cfg.norm ? launch<D, kBf16, true, true>(a, stream) : launch<D, kBf16, true, false>(a, stream);
  return cfg.norm ? launch<D, kBf16, false, true>(a, stream) : launch<D, kBf16, false, false>(a, stream);
}

}  // namespace

hipError_t launch_qk_norm_rope(const h3_qk_cfg& cfg, const h3_kv4_cfg* kv, uint32_t tokens,
                               const QkBindings& x, hipStream_t stream) {
  QkArgs a{};
  a.q = x.q;
  a.k = x.k;
  a.v = x.v;
  a.q_weight = x.q_weight;
  a.k_weight = x.k_weight;
  a.cos_t = x.cos_t;
  a.sin_t = x.sin_t;
  a.positions = x.positions;
  a.slots = x.slots;
  a.q_out = x.q_out;
  a.k_out = x.k_out;
  a.tokens = tokens;
  a.heads = cfg.heads;
  a.kv_heads = cfg.kv_heads;
  a.rotary = cfg.rotary;
  a.position_limit = cfg.positions;
  a.q_stride = cfg.q_stride;
  a.k_stride = cfg.k_stride;
  a.v_stride = cfg.v_stride;
  a.q_out_stride = cfg.q_out_stride;
  a.k_out_stride = cfg.k_out_stride;
  a.eps = cfg.eps;
  a.units = cfg.heads + cfg.kv_heads * (kv ? 2 : 1);
  if (kv) {
    a.cache = static_cast<uint8_t*>(x.cache);
    a.page_shift = __builtin_ctz(kv->page_tokens);
    a.slot_limit = (uint64_t)kv->pages * kv->page_tokens;
  }
  const bool bf16 = cfg.elem == H3_ELEM_BF16;
  if (cfg.head_dim == 128)
    return bf16 ? launch_kind<128, true>(a, cfg, stream) : launch_kind<128, false>(a, cfg, stream);
  return bf16 ? launch_kind<64, true>(a, cfg, stream) : launch_kind<64, false>(a, cfg, stream);
}

}  // namespace h3
