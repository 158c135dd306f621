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
#include "kv4_row.hpp"

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
    const Slot<D> at = slot_at<D>(a.page_shift, a.heads, slot[i], p.head);
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
    const Slot<D> at = slot_at<D>(a.page_shift, a.heads, max(slot[i], 0), p.head);  // slot 0 is there to read
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
