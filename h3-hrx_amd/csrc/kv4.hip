// The 4-bit key/value cache on gfx950: rows of K and V quantized into their slots as they are
// written, and read back.
//
// A row is one token's channels of one cache head, x_0 .. x_{D-1}. It is held as its minimum m, a
// scale s and D codes u_c of 4 bits, m and s in the element type of the rows:
//   s = (max x - m) / 15, rounded toward zero to the element type,
//   u_c = clamp(rne((x_c - m) / s), 0, 15), 0 where s is 0,
// and stands for m + s u_c. m is one of the row's own values, so it is held exactly; s is rounded
// toward zero so that m + 15 s never passes max x (rounded to nearest it can overflow f16, and the
// top code would read back as infinity). The codes come from an IEEE division in f32, which decides
// every code as exact arithmetic does wherever x - m is exact; bf16 rows are halved for it, which
// changes no quotient and keeps max - min below f32's largest. A row that holds a NaN or an infinity
// has m = NaN and reads back as NaN throughout.
//
// Layout (h3attn.h): one block per (page, cache head): K codes [page_tokens][D/2] bytes, V codes
// the same, K words [page_tokens], V words [page_tokens]; a word holds m low, s high.
//
// Both kernels move every byte once (HBM-bound): D/8 lanes of 8 channels hold a row, so a wave
// takes 512/D consecutive tokens of one head (their codes are 256 contiguous bytes where the slots
// are), and the four waves of a workgroup four heads of the same tokens, which lie side by side in
// the input rows.
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

// The lane's place: token, head, and its 8 channels' position in the row.
template <int D>
struct Place {
  uint32_t token, head, lane;
  bool live;
};
template <int D>
__device__ __forceinline__ Place<D> place(const RowArgs& a) {
  constexpr uint32_t kLanes = D / 8, kRows = 64 / kLanes;
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  Place<D> p;
  p.head = blockIdx.y * kWaves + wave;
  p.token = blockIdx.x * kRows + lane / kLanes;
  p.lane = lane % kLanes;
  p.live = p.head < a.heads && p.token < a.tokens;
  return p;
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

// The row's word and this lane's eight codes, low nibble first.
template <int D, bool kBf16>
__device__ __forceinline__ uint2 quantize(uint4 raw) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  float x[8];
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t h = (w[i / 2] >> (16 * (i & 1))) & 0xffffu;
    x[i] = widen<kBf16>(h);
    bad |= (h & 0x7fffu) >= (kBf16 ? 0x7f80u : 0x7c00u);
  }
  float lo = x[0], hi = x[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    lo = fminf(lo, x[i]);
    hi = fmaxf(hi, x[i]);
  }
  lo = row_reduce<D, false>(lo);
  hi = row_reduce<D, true>(hi);
  if (row_reduce<D, true>(bad ? 1.0f : 0.0f) > 0.0f) return {0x7fffu, 0u};
  constexpr float kPart = kBf16 ? 0.5f : 1.0f;  // exact on every bf16 value, subnormal ones too
  const float low = lo * kPart;
  const uint32_t s = narrow_down<kBf16>((hi * kPart - low) / (15.0f * kPart));
  const float step = widen<kBf16>(s) * kPart;
  uint32_t codes = 0;
  if (step > 0.0f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float u = fminf(rintf((x[i] * kPart - low) / step), 15.0f);
      codes |= (uint32_t)u << (4 * i);
    }
  }
  return {narrow<kBf16>(lo) | (s << 16), codes};
}

// Quantizes rows [tokens][heads][D] of K and V into their slots.
template <int D, bool kBf16>
__global__ __launch_bounds__(kThreads) void k_kv4_write(RowArgs a) {
  const Place<D> p = place<D>(a);
  if (!p.live) return;  // whole rows leave: a row's lanes share token and head
  const int32_t slot = a.slots[p.token];
  if (slot < 0 || (uint64_t)slot >= a.slot_limit) return;
  const uint32_t col = p.head * D + 8 * p.lane;
  const uint4 k = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.k) +
                                                  (size_t)p.token * a.k_stride + col);
  const uint4 v = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.v) +
                                                  (size_t)p.token * a.v_stride + col);
  const Slot<D> at = slot_at<D>(a, slot, p.head);
  const uint2 qk = quantize<D, kBf16>(k), qv = quantize<D, kBf16>(v);
  uint8_t* codes = a.cache + at.codes + 4 * p.lane;
  *reinterpret_cast<uint32_t*>(codes) = qk.y;
  *reinterpret_cast<uint32_t*>(codes + at.half) = qv.y;
  if (p.lane == 0) {
    uint8_t* words = a.cache + at.words;
    *reinterpret_cast<uint32_t*>(words) = qk.x;
    *reinterpret_cast<uint32_t*>(words + 4 * at.tokens) = qv.x;
  }
}

// Eight channels m + s u, rounded to the element type.
template <bool kBf16>
__device__ __forceinline__ uint4 dequantize(uint32_t codes, uint32_t word) {
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
template <int D, bool kBf16>
__global__ __launch_bounds__(kThreads) void k_kv4_read(RowArgs a) {
  const Place<D> p = place<D>(a);
  if (!p.live) return;
  const int32_t slot = a.slots[p.token];
  uint4 k = {0, 0, 0, 0}, v = k;
  if (slot >= 0 && (uint64_t)slot < a.slot_limit) {
    const Slot<D> at = slot_at<D>(a, slot, p.head);
    const uint8_t* codes = a.cache + at.codes + 4 * p.lane;
    const uint8_t* words = a.cache + at.words;
    const uint32_t ck = *reinterpret_cast<const uint32_t*>(codes);
    const uint32_t cv = *reinterpret_cast<const uint32_t*>(codes + at.half);
    k = dequantize<kBf16>(ck, *reinterpret_cast<const uint32_t*>(words));
    v = dequantize<kBf16>(cv, *reinterpret_cast<const uint32_t*>(words + 4 * at.tokens));
  }
  const uint32_t col = p.head * D + 8 * p.lane;
  *reinterpret_cast<uint4*>(static_cast<uint16_t*>(const_cast<void*>(a.k)) +
                            (size_t)p.token * a.k_stride + col) = k;
  *reinterpret_cast<uint4*>(static_cast<uint16_t*>(const_cast<void*>(a.v)) +
                            (size_t)p.token * a.v_stride + col) = v;
}

template <int D, bool kBf16>
hipError_t launch(const RowArgs& a, bool write, hipStream_t stream) {
  const dim3 grid((a.tokens + 512 / D - 1) / (512 / D), (a.heads + kWaves - 1) / kWaves);
  if (write)
    hipLaunchKernelGGL((k_kv4_write<D, kBf16>), grid, dim3(kThreads), 0, stream, a);
  else
    hipLaunchKernelGGL((k_kv4_read<D, kBf16>), grid, dim3(kThreads), 0, stream, a);
  return hipGetLastError();
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
    return bf16 ? launch<128, true>(a, write, stream) : launch<128, false>(a, write, stream);
  return bf16 ? launch<64, true>(a, write, stream) : launch<64, false>(a, write, stream);
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
