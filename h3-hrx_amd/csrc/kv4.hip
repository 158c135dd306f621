// The 4-bit key/value cache on gfx950: rows of K and V quantized into their slots as they are
// written, and read back.
//
// A row is one token's channels of one cache head, x_0 .. x_{D-1}. It is held as its minimum m, a
// scale s and D codes u_c of 4 bits, m and s in the element type of the rows:
//   s = (max x - m) / 15, rounded toward zero to the element type,
//   u_c = clamp(rne((x_c - m) / s), 0, 15), 0 where s is 0,
// and stands for m + s u_c. m is one of the row's own values, so it is held exactly; s is rounded
// toward zero so that m + 15 s never passes max x (rounded to nearest it can overflow f16, and the
// top code would read back as infinity). The codes come from a division in f32 that decides every code
// as exact arithmetic does wherever x - m is exact; bf16 rows are halved for it, which changes no
// quotient and keeps max - min below f32's largest. A row that holds a NaN or an infinity
// has m = NaN and reads back as NaN throughout.
//
// Layout (h3attn.h): one block per (page, cache head): K codes [page_tokens][D/2] bytes, V codes
// the same, K words [page_tokens], V words [page_tokens]; a word holds m low, s high.
//
// Both kernels move every byte once (HBM-bound): D/8 lanes of 8 channels hold a row, so a wave
// takes 512/D consecutive tokens of one head (their codes are 256 contiguous bytes where the slots
// are), and the four waves of a workgroup four heads of the same tokens, which lie side by side in
// the input rows. 129,024 rows of 8 heads of 128 channels are read back in 123 us (669 MB, 5.4 TB/s: a
// copy reaches 5.1); 31,104 rows are written in 31 us (161 MB, 5.2 TB/s) and read back in 25; one row takes
// 2.2 us each way, which is a launch.
#include "internal.hpp"

namespace h3 {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;

struct RowArgs {
  const void* k;
  const void* v;
  const int32_t* slots;
  uint8_t* cache;
  uint32_t tokens, heads, k_stride, v_stride;  // strides in elements
  uint32_t page_shift;
  uint64_t slot_limit;  // slots at or past it name no row
};

// The lane's places: head, the N tokens kApart from each other, and its 8 channels' position in a row.
template <int D, int N>
struct Place {
  static constexpr uint32_t kLanes = D / 8, kApart = 64 / kLanes;
  uint32_t token, head, lane;
};
template <int D, int N>
__device__ __forceinline__ Place<D, N> place(const RowArgs& a) {
  using P = Place<D, N>;
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  return {blockIdx.x * (N * P::kApart) + lane / P::kLanes, blockIdx.y * kWaves + wave,
          lane % P::kLanes};
}

// The slot of row `token`, or -1 if there is no such row or it names none.
__device__ __forceinline__ int32_t slot_of(const RowArgs& a, uint32_t token) {
  const int32_t slot = token < a.tokens ? a.slots[token] : -1;
  return (uint64_t)(uint32_t)slot < a.slot_limit ? slot : -1;
}

// Byte offsets of a slot's K codes and K word of one head. `half`: the bytes of a page's K codes.
template <int D>
struct Slot {
  uint64_t codes, words;
  uint32_t half, tokens;
};
template <int D>
__device__ __forceinline__ Slot<D> slot_at(const RowArgs& a, uint32_t slot, uint32_t head) {
  const uint32_t tokens = 1u << a.page_shift;
  const uint32_t in_page = slot & (tokens - 1);
  const uint64_t block = (uint64_t)tokens * (D + 8);
  const uint64_t base = ((uint64_t)(slot >> a.page_shift) * a.heads + head) * block;
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
  if (bad) {  // zeros in their place: no NaN meets the arithmetic, which this file's flags let assume none
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

// Quantizes rows [tokens][heads][D] of K and V into their slots.
template <int D, bool kBf16, int N>
__global__ __launch_bounds__(kThreads) void k_kv4_write(RowArgs a) {
  const Place<D, N> p = place<D, N>(a);
  if (p.head >= a.heads) return;
  const uint32_t col = p.head * D + 8 * p.lane;
  int32_t slot[N];
  uint4 k[N], v[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const uint32_t token = p.token + i * p.kApart;
    slot[i] = slot_of(a, token);
    // The last row stands for the rows past it: their loads need no branch.
    const size_t row = min(token, a.tokens - 1);
    k[i] = load_row<(N > 1)>(a.k, row * a.k_stride + col);
    v[i] = load_row<(N > 1)>(a.v, row * a.v_stride + col);
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const uint2 qk = quantize<D, kBf16>(k[i]), qv = quantize<D, kBf16>(v[i]);
    if (slot[i] < 0) continue;
    const Slot<D> at = slot_at<D>(a, slot[i], p.head);
    uint8_t* codes = a.cache + at.codes + 4 * p.lane;
    *reinterpret_cast<uint32_t*>(codes) = qk.y;
    *reinterpret_cast<uint32_t*>(codes + at.half) = qv.y;
    if (p.lane == 0) {
      uint8_t* words = a.cache + at.words;
      *reinterpret_cast<uint32_t*>(words) = qk.x;
      *reinterpret_cast<uint32_t*>(words + 4 * at.tokens) = qv.x;
    }
  }
}

// Eight channels m + s u, rounded to the element type. (NaN by its bits: this file is compiled to
// assume none in its arithmetic.)
template <bool kBf16>
__device__ __forceinline__ uint4 dequantize(uint32_t codes, uint32_t word) {
  constexpr uint32_t kTop = kBf16 ? 0x7f80u : 0x7c00u;
  if ((word & kTop) == kTop || ((word >> 16) & kTop) == kTop)
    return {0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu};
  const float m = widen<kBf16>(word & 0xffffu), s = widen<kBf16>(word >> 16);
  uint32_t out[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float lo = fmaf((float)((codes >> (8 * i)) & 15u), s, m);
    const float hi = fmaf((float)((codes >> (8 * i + 4)) & 15u), s, m);
    out[i] = narrow<kBf16>(lo) | (narrow<kBf16>(hi) << 16);
  }
  return {out[0], out[1], out[2], out[3]};
}

// Reads rows of K and V back from their slots; a slot that names no row gives zeros.
template <int D, bool kBf16, int N>
__global__ __launch_bounds__(kThreads) void k_kv4_read(RowArgs a) {
  const Place<D, N> p = place<D, N>(a);
  if (p.head >= a.heads) return;
  const uint32_t col = p.head * D + 8 * p.lane;
  int32_t slot[N];
  uint32_t ck[N], cv[N], wk[N], wv[N];
#pragma unroll
  for (int i = 0; i < N; ++i) slot[i] = slot_of(a, p.token + i * p.kApart);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const Slot<D> at = slot_at<D>(a, max(slot[i], 0), p.head);  // slot 0 is there to read
    const uint8_t* codes = a.cache + at.codes + 4 * p.lane;
    const uint8_t* words = a.cache + at.words;
    ck[i] = *reinterpret_cast<const uint32_t*>(codes);
    cv[i] = *reinterpret_cast<const uint32_t*>(codes + at.half);
    wk[i] = *reinterpret_cast<const uint32_t*>(words);
    wv[i] = *reinterpret_cast<const uint32_t*>(words + 4 * at.tokens);
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const uint32_t token = p.token + i * p.kApart;
    if (token >= a.tokens) continue;
    const bool live = slot[i] >= 0;
    const uint4 k = dequantize<kBf16>(live ? ck[i] : 0u, live ? wk[i] : 0u);
    const uint4 v = dequantize<kBf16>(live ? cv[i] : 0u, live ? wv[i] : 0u);
    store_row<(N > 1)>(a.k, (size_t)token * a.k_stride + col, k);
    store_row<(N > 1)>(a.v, (size_t)token * a.v_stride + col, v);
  }
}

template <int D, bool kBf16, int N>
hipError_t launch(const RowArgs& a, bool write, hipStream_t stream) {
  constexpr uint32_t kTokens = N * Place<D, N>::kApart;
  const dim3 grid((a.tokens + kTokens - 1) / kTokens, (a.heads + kWaves - 1) / kWaves);
  if (write)
    hipLaunchKernelGGL((k_kv4_write<D, kBf16, N>), grid, dim3(kThreads), 0, stream, a);
  else
    hipLaunchKernelGGL((k_kv4_read<D, kBf16, N>), grid, dim3(kThreads), 0, stream, a);
  return hipGetLastError();
}

// One row a lane where the rows are few (256 in 2.7 us); more, and past the caches, where that still leaves
// every compute unit workgroups to choose from: more loads in flight, and a head's parameters of 8 or 16
// tokens in one line from one wave. Two or four, written and read back: 10,000 rows 23.6 and 24.6 us, 31,104
// 57 and 60, 100,000 199 and 192 (219 with one).
template <int D, bool kBf16>
hipError_t launch_n(const RowArgs& a, bool write, hipStream_t stream) {
  const uint64_t fours = (uint64_t)a.tokens * D / 2048 * ((a.heads + kWaves - 1) / kWaves);
  const uint64_t cus = device_cus();
  return fours >= 32 * cus  ? launch<D, kBf16, 4>(a, write, stream)
         : fours >= 4 * cus ? launch<D, kBf16, 2>(a, write, stream)
                            : launch<D, kBf16, 1>(a, write, stream);
}

hipError_t rows(const h3_kv4_cfg& cfg, uint32_t tokens, uint32_t k_stride, uint32_t v_stride,
                const void* k, const void* v, const int32_t* slots, void* cache, bool write,
                hipStream_t stream) {
  RowArgs a;
  a.k = k;
  a.v = v;
  a.slots = slots;
  a.cache = static_cast<uint8_t*>(cache);
  a.tokens = tokens;
  a.heads = cfg.kv_heads;
  a.k_stride = k_stride;
  a.v_stride = v_stride;
  a.page_shift = __builtin_ctz(cfg.page_tokens);
  a.slot_limit = (uint64_t)cfg.pages * cfg.page_tokens;
  const bool bf16 = cfg.elem == H3_ELEM_BF16;
  if (cfg.head_dim == 128)
    return bf16 ? launch_n<128, true>(a, write, stream) : launch_n<128, false>(a, write, stream);
  return bf16 ? launch_n<64, true>(a, write, stream) : launch_n<64, false>(a, write, stream);
}

}  // namespace

hipError_t launch_kv4_write(const h3_kv4_cfg& cfg, uint32_t tokens, uint32_t k_stride,
                            uint32_t v_stride, const void* k, const void* v, const int32_t* slots,
                            void* cache, hipStream_t stream) {
  return rows(cfg, tokens, k_stride, v_stride, k, v, slots, cache, true, stream);
}

hipError_t launch_kv4_read(const h3_kv4_cfg& cfg, uint32_t tokens, uint32_t k_stride,
                           uint32_t v_stride, const int32_t* slots, const void* cache, void* k,
                           void* v, hipStream_t stream) {
  return rows(cfg, tokens, k_stride, v_stride, k, v, slots, const_cast<void*>(cache), false,
              stream);
}

}  // namespace h3
