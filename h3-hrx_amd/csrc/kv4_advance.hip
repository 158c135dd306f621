// The bookkeeping of a step over the 4-bit cache on gfx950: page tables, slots and positions from the rows that each
// sequence asks for, so that a captured step needs nothing from the host but those numbers.
//
// Sequence b holds ceil(length_b / P) pages of P tokens and asks for n_b rows, hence for
// ceil((length_b + n_b) / P) - ceil(length_b / P) pages. Everything is sums over the sequences before b: of the
// ended sequences' pages, where they go on the stack of free pages; of pages and rows asked for, who is
// granted; of those granted, whose page is which and whose rows are where. No atomics: the same numbers give the
// same pages.
//
// One workgroup makes the sums, 1,024 sequences at a time, and hands out pages by their number in the step (a search
// in the sums per page: a prompt's hundreds are as quick as a token's one). Rows are slots and positions by
// the same search.
#include "internal.hpp"

namespace h3 {
namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr uint32_t kMost = 1u << 30;  // sums stop here: past every number of rows or pages that can be granted

struct AdvanceArgs {
  AdvanceBindings x;
  uint32_t batch, columns, rows, pages, page_shift;
};

// Sums of two numbers at once.
struct Two {
  uint32_t a, b;
};
__device__ __forceinline__ uint32_t add(uint32_t x, uint32_t y) { return min(x + y, kMost); }

// The sums over the threads up to this one. `scratch`: a Two per wave.
__device__ __forceinline__ Two sum_to_here(Two v, Two* scratch) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const Two x = {__shfl_up(v.a, d), __shfl_up(v.b, d)};
    if (lane >= d) v = {add(v.a, x.a), add(v.b, x.b)};
  }
  __syncthreads();  // the scratch of the call before is read
  if (lane == 63) scratch[wave] = v;
  __syncthreads();
  for (int w = 0; w < wave; ++w) v = {add(v.a, scratch[w].a), add(v.b, scratch[w].b)};
  return v;
}

// The first of n sums, which do not decrease, that is past i.
__device__ __forceinline__ int find(const uint32_t* sums, int n, uint32_t i) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (sums[mid] > i) hi = mid; else lo = mid + 1;
  }
  return lo;
}

__device__ __forceinline__ uint32_t tokens_of(const AdvanceArgs& a, uint32_t b) {
  return (uint32_t)min(max(a.x.lengths[b], 0), (int)(a.columns << a.page_shift));
}

__device__ __forceinline__ int slot_of(const AdvanceArgs& a, int page, uint32_t position) {
  return (uint32_t)page < a.pages ? (page << a.page_shift) + (int)(position & ((1u << a.page_shift) - 1)) : -1;
}

__global__ __launch_bounds__(kThreads) void k_kv4_advance(AdvanceArgs a) {
  __shared__ Two scratch[kWaves];
  __shared__ uint32_t page_sums[kThreads], row_sums[kThreads], first_column[kThreads], first_token[kThreads];
  __shared__ Two carry_s, granted_s;
  const uint32_t t = threadIdx.x, up = (1u << a.page_shift) - 1;
  const uint32_t before = (uint32_t)min(max(*a.x.free_count, 0), (int)a.pages);
  const uint32_t prefix = a.x.prefix_length ? (uint32_t)max(*a.x.prefix_length, 0) : 0;

  // The pages of the sequences that end, onto the stack.
  uint32_t count = before;
  for (uint32_t b0 = 0; b0 < a.batch; b0 += kThreads) {
    const uint32_t b = b0 + t;
    uint32_t held = 0;
    if (b < a.batch && a.x.asked[b] < 0) held = (tokens_of(a, b) + up) >> a.page_shift;
    const Two sums = sum_to_here({held, 0}, scratch);
    page_sums[t] = sums.a;
    __syncthreads();
    const uint32_t all = page_sums[kThreads - 1];
    for (uint32_t i = t; i < all; i += kThreads) {
      const int s = find(page_sums, kThreads, i);
      const uint32_t column = i - (s ? page_sums[s - 1] : 0);
      if (count + i < a.pages) a.x.free_pages[count + i] = a.x.table[(size_t)(b0 + s) * a.columns + column];
    }
    count = min(count + all, a.pages);
  }
  __syncthreads();

  // Who gets rows and pages, and which.
  Two asked = {0, 0}, granted = {0, 0};  // pages and rows of the sequences before these
  if (t == 0) a.x.q_starts[0] = 0;
  for (uint32_t b0 = 0; b0 < a.batch; b0 += kThreads) {
    const uint32_t b = b0 + t;
    uint32_t have = 0, rows = 0, held = 0, need = 0;
    if (b < a.batch) {
      const int n = a.x.asked[b];
      if (n >= 0) {
        have = tokens_of(a, b);
        if ((uint64_t)have + (uint32_t)n <= (uint64_t)a.columns << a.page_shift) rows = (uint32_t)n;
        held = (have + up) >> a.page_shift;
        need = ((have + rows + up) >> a.page_shift) - held;
      }
    }
    Two sums = sum_to_here({need, rows}, scratch);
    sums = {add(sums.a, asked.a), add(sums.b, asked.b)};
    if ((need != 0 && sums.a > count) || sums.b > a.rows) rows = need = 0;
    const Two mine = sum_to_here({need, rows}, scratch);
    page_sums[t] = mine.a;
    row_sums[t] = mine.b;
    first_column[t] = held;
    first_token[t] = have;
    if (t == kThreads - 1) {
      carry_s = sums;
      granted_s = mine;
    }
    __syncthreads();
    asked = carry_s;
    const Two all = granted_s;
    for (uint32_t i = t; i < all.a; i += kThreads) {
      const int s = find(page_sums, kThreads, i);
      const uint32_t column = first_column[s] + i - (s ? page_sums[s - 1] : 0);
      a.x.table[(size_t)(b0 + s) * a.columns + column] = a.x.free_pages[count - 1 - (granted.a + i)];
    }
    if (b < a.batch) {
      a.x.lengths_out[b] = (int)(have + rows);
      a.x.q_starts[b + 1] = (int)(granted.b + mine.b);
    }
    __syncthreads();
    for (uint32_t i = t; i < all.b; i += kThreads) {
      const int s = find(row_sums, kThreads, i);
      const uint32_t position = first_token[s] + i - (s ? row_sums[s - 1] : 0);
      const int page = a.x.table[(size_t)(b0 + s) * a.columns + (position >> a.page_shift)];
      a.x.slots[granted.b + i] = slot_of(a, page, position);
      a.x.positions[granted.b + i] = (int)(prefix + position);
    }
    granted = {granted.a + all.a, granted.b + all.b};
  }
  for (uint32_t i = granted.b + t; i < a.rows; i += kThreads) a.x.slots[i] = a.x.positions[i] = -1;
  if (t == 0) *a.x.free_count_out = (int)(count - granted.a);
}

}  // namespace

hipError_t launch_kv4_advance(const h3_kv4_cfg& cfg, uint32_t batch, uint32_t table_stride, uint32_t rows,
                              const AdvanceBindings& x, hipStream_t stream) {
  AdvanceArgs a{x, batch, table_stride, rows, cfg.pages, (uint32_t)__builtin_ctz(cfg.page_tokens)};
  hipLaunchKernelGGL(k_kv4_advance, dim3(1), dim3(kThreads), 0, stream, a);
  return hipGetLastError();
}

}  // namespace h3
