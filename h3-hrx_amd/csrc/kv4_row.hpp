// A row of the 4-bit key/value cache on gfx950: where its slot lies and how D/8 lanes of 8 channels quantize it
// (kv4.hip has the format).
#pragma once

#include "internal.hpp"

namespace h3 {
namespace {

// Byte offsets of a slot's K codes and K word of one head. `half`: the bytes of a page's K codes.
template <int D>
struct Slot {
  uint64_t codes, words;
  uint32_t half, tokens;
};
template <int D>
__device__ __forceinline__ Slot<D> slot_at(uint32_t page_shift, uint32_t heads, uint32_t slot, uint32_t head) {
  const uint32_t tokens = 1u << page_shift;
  const uint32_t in_page = slot & (tokens - 1);
  const uint64_t block = (uint64_t)tokens * (D + 8);
  const uint64_t base = ((uint64_t)(slot >> page_shift) * heads + head) * block;
  return {base + in_page * (D / 2), base + (uint64_t)tokens * D + in_page * 4, tokens * (D / 2),
          tokens};
}

template <int kCtrl>
__device__ __forceinline__ float dpp(float v) {
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), kCtrl, 0xF, 0xF, true));
}

// Minimum (or maximum) over the D/8 lanes of a row on the vector pipe: quad_perm [1,0,3,2] and
// [2,3,0,1], row_half_mirror (8 lanes), row_mirror (16 lanes).
template <int D, bool kMax>
__device__ __forceinline__ float row_reduce(float v) {
  auto op = [](float a, float b) { return kMax ? fmaxf(a, b) : fminf(a, b); };
  v = op(v, dpp<0xB1>(v));
  v = op(v, dpp<0x4E>(v));
  v = op(v, dpp<0x141>(v));
  if constexpr (D == 128) v = op(v, dpp<0x140>(v));
  return v;
}

template <bool kBf16>
__device__ __forceinline__ float widen(uint32_t bits) {
  if constexpr (kBf16) return __uint_as_float(bits << 16);
  return (float)__builtin_bit_cast(_Float16, (uint16_t)bits);
}
template <bool kBf16>
__device__ __forceinline__ uint32_t narrow(float v) {  // to nearest, ties to even
  if constexpr (kBf16) return __builtin_bit_cast(uint16_t, (__bf16)v);
  return __builtin_bit_cast(uint16_t, (_Float16)v);
}
// A finite v >= 0 rounded toward zero.
template <bool kBf16>
__device__ __forceinline__ uint32_t narrow_down(float v) {
  if constexpr (kBf16) return __float_as_uint(v) >> 16;
  const uint32_t h = narrow<false>(v);
  return widen<false>(h) > v ? h - 1 : h;
}

// a / b by r, the reciprocal of b to an ulp or so: q = a r, then q + (a - q b) r. The remainder is exact
// (b is a short number, or a quotient near a whole one), so the error before the last rounding is some
// 2^-45 of the quotient: every quotient that 24 bits hold comes out exactly, the borders k + 1/2 of
// the codes and the values of the element type among them.
__device__ __forceinline__ float quotient(float a, float b, float r) {
  const float q = a * r;
  return fmaf(fmaf(-q, b, a), r, q);
}

// Sixteen bytes of a row in 16 bits. Long calls (kOnce) pass the caches by: such rows are more than L2
// holds, and what stays there is the codes. 31,104 rows written and read back took 79 us without, 61 with;
// with the codes past the caches too, 70.
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
template <bool kOnce>
__device__ __forceinline__ uint4 load_row(const void* rows, size_t at) {
  const v4u* p = reinterpret_cast<const v4u*>(static_cast<const uint16_t*>(rows) + at);
  const v4u x = kOnce ? __builtin_nontemporal_load(p) : *p;
  return {x.x, x.y, x.z, x.w};
}
template <bool kOnce>
__device__ __forceinline__ void store_row(const void* rows, size_t at, uint4 x) {
  v4u* p = reinterpret_cast<v4u*>(static_cast<uint16_t*>(const_cast<void*>(rows)) + at);
  if constexpr (kOnce)
    __builtin_nontemporal_store(v4u{x.x, x.y, x.z, x.w}, p);
  else
    *p = {x.x, x.y, x.z, x.w};
}

// The row's word and this lane's eight codes, low nibble first. Few vector instructions a channel are
// what keeps the kernel near HBM's rate: with a correctly rounded division by the step for every channel
// 31,104 rows took 51 us for 44 (before their loads passed the caches by).
template <int D, bool kBf16>
__device__ __forceinline__ uint2 quantize(uint4 raw) {
  typedef uint16_t v2us __attribute__((ext_vector_type(2)));
  constexpr uint32_t kTop = kBf16 ? 0x7f80u : 0x7c00u;  // magnitudes from here on are no numbers
  uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  float x[8];
  v2us top = {0, 0};
#pragma unroll
  for (int i = 0; i < 4; ++i) top = __builtin_elementwise_max(top, __builtin_bit_cast(v2us, w[i] & 0x7fff7fffu));
  const bool bad = top[0] >= kTop || top[1] >= kTop;
  if (bad) {  // zeros in their place: no NaN meets the arithmetic, which kv4.hip's flags let assume none
    asm volatile("");
    w[0] = w[1] = w[2] = w[3] = 0;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = widen<kBf16>(w[i] & 0xffffu);
    x[2 * i + 1] = kBf16 ? __uint_as_float(w[i] & 0xffff0000u) : widen<kBf16>(w[i] >> 16);
  }
  float lo = x[0], hi = x[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    lo = fminf(lo, x[i]);
    hi = fmaxf(hi, x[i]);
  }
  // A lane with a NaN or an infinity makes the row's maximum infinite, whatever its others are.
  if (bad) hi = __builtin_inff();
  lo = row_reduce<D, false>(lo);
  hi = row_reduce<D, true>(hi);
  if (__float_as_uint(hi) == 0x7f800000u) return {0x7fffu, 0u};
  float part = kBf16 ? 0.5f : 1.0f;  // exact on every bf16 value, subnormal ones too
  const float from = hi * part, less = lo * part, wide = from - less;
  uint32_t s = narrow_down<kBf16>(quotient(wide, 15.0f * part, (1.0f / 15.0f) / (kBf16 ? 0.5f : 1.0f)));
  // max - min may have more bits than f32. The scale is another then only where 15 s is what f32 holds of it: there the
  // sign of the exact rounding error (a two-sum) decides.
  if (widen<kBf16>(s) * (15.0f * part) == wide) {
    asm volatile("");  // a branch: one row in some hundred
    const float back = wide - from;
    s -= (from - (wide - back)) - (less + back) < 0.0f ? 1 : 0;
  }
  if (kBf16 && widen<kBf16>(s) < 0x1p-60f) part = 0x1p99f;  // the reciprocal stays finite
  const float low = lo * part, step = widen<kBf16>(s) * part;
  uint32_t codes = 0;
  if (step > 0.0f) {
    const float r = __builtin_amdgcn_rcpf(step);
    float u[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      u[i] = fminf(rintf(quotient(fmaf(x[i], part, -low), step, r)), 15.0f);
    // Four codes a whole number of 16 bits, exact in f32.
    const float first = fmaf(fmaf(fmaf(u[3], 16.0f, u[2]), 16.0f, u[1]), 16.0f, u[0]);
    const float second = fmaf(fmaf(fmaf(u[7], 16.0f, u[6]), 16.0f, u[5]), 16.0f, u[4]);
    codes = (uint32_t)first | ((uint32_t)second << 16);
  }
  return {narrow<kBf16>(lo) | (s << 16), codes};
}

}  // namespace
}  // namespace h3
