// The bookkeeping of a step over the 4-bit cache on gfx950: page tables, slots and positions from the rows that each
// sequence asks for, so that a captured step needs nothing from the host but those numbers.
//
// Sequence b holds ceil(length_b / P) pages of P tokens and asks for n_b rows, hence for
// ceil((length_b + n_b) / P) - ceil(length_b / P) pages. Everything is sums over the sequences before b: of the
// ended sequences' pages, where they go on the stack of free pages; of pages and rows asked for, who is
// granted; of those granted, whose page is which and whose rows are where. No atomics: the same numbers give the
// same pages.
//
// One workgroup makes the sums, a sequence to a thread, and hands out pages by their number in the step (a search in
// the sums per page: a prompt's hundreds are as quick as a token's one). Where nobody asks for more than one row a
// thread finishes its own sequence. Long calls' slots and positions are a launch of their own. Latency bounds
// both: 64 sequences of a token each, of which three end, 5.1 us (one alone 3.4); 512 with prompts among them,
// 129,024 rows, 6.9 and 5.5 (61 with the rows in the first, a search after another).
#include "internal.hpp"

namespace h3 {
namespace {

// More rows than this have a launch of their own: 512 sequences with prompts among them, 9.0 us for 2,048 rows in one
// launch and 12.8 for 2,049 in two, 12.8 for 16,384; in one, 61 for 129,024.
constexpr uint32_t kRowsApart = 2048;
constexpr uint32_t kGiven = 4;  // entries of ended sequences under way in a thread
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

// The sum of v over the wave's lanes up to this one, on the vector pipe: row_shr by 1, 2, 4 and 8, then the last lane
// of 16 (row_bcast15) and of 32 (row_bcast31) to the lanes after them.
template <int kCtrl, int kRows>
__device__ __forceinline__ uint32_t add_from(uint32_t v) {
  return add(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, kCtrl, kRows, 0xF, false));
}
__device__ __forceinline__ uint32_t wave_sum(uint32_t v) {
  v = add_from<0x111, 0xF>(v);
  v = add_from<0x112, 0xF>(v);
  v = add_from<0x114, 0xF>(v);
  v = add_from<0x118, 0xF>(v);
  v = add_from<0x142, 0xA>(v);
  return add_from<0x143, 0xC>(v);
}

// The sums over the workgroup's threads up to this one, and over all of them. `scratch`: a Two per wave.
template <int kThreads>
__device__ __forceinline__ Two sum_to_here(Two v, Two* scratch, Two* all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  v = {wave_sum(v.a), wave_sum(v.b)};
  __syncthreads();  // the scratch of the call before is read
  if (lane == 63) scratch[wave] = v;
  __syncthreads();
  Two before = {0, 0}, sum = {0, 0};
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) {
    if (w == wave) before = sum;
    sum = {add(sum.a, scratch[w].a), add(sum.b, scratch[w].b)};
  }
  *all = sum;
  return {add(v.a, before.a), add(v.b, before.b)};
}

// The first of kN sums (a power of two, of which none is below the one before it) that is past i; the last one if
// none is.
template <int kN>
__device__ __forceinline__ uint32_t find(const uint32_t* sums, uint32_t i) {
  uint32_t at = 0;
#pragma unroll
  for (uint32_t step = kN / 2; step; step /= 2) at += sums[at + step - 1] <= i ? step : 0;
  return at;
}

__device__ __forceinline__ uint32_t tokens_of(const AdvanceArgs& a, uint32_t b) {
  return (uint32_t)min(max(a.x.lengths[b], 0), (int)(a.columns << a.page_shift));
}

__device__ __forceinline__ int slot_of(const AdvanceArgs& a, int page, uint32_t position) {
  return (uint32_t)page < a.pages ? (page << a.page_shift) + (int)(position & ((1u << a.page_shift) - 1)) : -1;
}

// take(i) and then put(i, what it gave) for i in t, t + kThreads, .. below n: four under way at a time.
template <int kThreads, typename Take, typename Put>
__device__ __forceinline__ void each(uint32_t t, uint32_t n, Take take, Put put) {
  for (uint32_t i = t; i < n; i += 4 * kThreads) {
    decltype(take(i)) got[4];
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k)
      if (i + k * kThreads < n) got[k] = take(i + k * kThreads);
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k)
      if (i + k * kThreads < n) put(i + k * kThreads, got[k]);
  }
}

// places: whether slots and positions are written here.
template <int kThreads>
__global__ __launch_bounds__(kThreads) void k_kv4_advance(AdvanceArgs a, bool places) {
  __shared__ Two scratch[kThreads / 64];
  __shared__ uint32_t page_sums[kThreads], row_sums[kThreads], first_column[kThreads], first_token[kThreads];
  __shared__ uint32_t some_none[2];
  const uint32_t t = threadIdx.x, up = (1u << a.page_shift) - 1;
  const uint32_t before = (uint32_t)min(max(*a.x.free_count, 0), (int)a.pages);
  const uint32_t prefix = a.x.prefix_length ? (uint32_t)max(*a.x.prefix_length, 0) : 0;

  // The pages of the sequences that end, onto the stack. An entry that is no page (-1 where the program has taken the
  // page back, as behind a window) is not pushed: it would be granted as one, and what is written there lost.
  uint32_t count = before, turn = 0;
  if (t < 2) some_none[t] = 0;
  for (uint32_t b0 = 0; b0 < a.batch; b0 += kThreads) {
    const uint32_t b = b0 + t;
    uint32_t held = 0;
    if (b < a.batch && a.x.asked[b] < 0) held = (tokens_of(a, b) + up) >> a.page_shift;
    if (!__syncthreads_or(held != 0)) continue;
    Two all;
    page_sums[t] = sum_to_here<kThreads>({held, 0}, scratch, &all).a;
    __syncthreads();
    for (uint32_t i0 = 0; i0 < all.a; i0 += kGiven * kThreads, turn ^= 1) {
      int page[kGiven];
#pragma unroll
      for (uint32_t k = 0; k < kGiven; ++k) {
        const uint32_t i = i0 + k * kThreads + t;
        page[k] = -1;
        if (i >= all.a) continue;
        const uint32_t s = find<kThreads>(page_sums, i);
        page[k] = a.x.table[(size_t)(b0 + s) * a.columns + i - (s ? page_sums[s - 1] : 0)];
        if ((uint32_t)page[k] >= a.pages) some_none[turn] = 1;
      }
      // Places on the stack by the entries' numbers, or, from a turn with an entry that is no page on, by the pages'
      // sums. Two flags in turn: a thread that is ahead sets the other one until all have read this.
      __syncthreads();
      if (some_none[turn] == 0) {
#pragma unroll
        for (uint32_t k = 0; k < kGiven; ++k) {
          const uint32_t i = k * kThreads + t;
          if (i0 + i < all.a && count + i < a.pages) a.x.free_pages[count + i] = page[k];
        }
        count = min(count + min(all.a - i0, kGiven * kThreads), a.pages);
      } else {
#pragma unroll
        for (uint32_t k = 0; k < kGiven; ++k) {
          const bool is = (uint32_t)page[k] < a.pages;
          Two sum;
          const uint32_t place = count + sum_to_here<kThreads>({is, 0}, scratch, &sum).a - 1;
          if (is && place < a.pages) a.x.free_pages[place] = page[k];
          count = min(count + sum.a, a.pages);
        }
      }
    }
  }
  __syncthreads();

  // Who gets rows and pages, and which.
  Two asked = {0, 0}, granted = {0, 0};  // pages and rows of the sequences before these
  if (t == 0) a.x.q_starts[0] = 0;
  for (uint32_t b0 = 0; b0 < a.batch; b0 += kThreads) {
    const uint32_t b = b0 + t;
    uint32_t have = 0, rows = 0, held = 0, need = 0;
    int last_page = -1;  // where a single row goes if it needs no page
    if (b < a.batch) {
      const int n = a.x.asked[b];
      if (n >= 0) {
        have = tokens_of(a, b);
        if ((uint64_t)have + (uint32_t)n <= (uint64_t)a.columns << a.page_shift) rows = (uint32_t)n;
        held = (have + up) >> a.page_shift;
        need = ((have + rows + up) >> a.page_shift) - held;
        if (held) last_page = a.x.table[(size_t)b * a.columns + held - 1];
      }
    }
    Two all;
    Two mine = sum_to_here<kThreads>({need, rows}, scratch, &all);
    const Two sums = {add(mine.a, asked.a), add(mine.b, asked.b)};
    asked = {add(asked.a, all.a), add(asked.b, all.b)};
    const bool refused = (need != 0 && sums.a > count) || sums.b > a.rows;
    if (__syncthreads_or(refused)) {
      if (refused) rows = need = 0;
      mine = sum_to_here<kThreads>({need, rows}, scratch, &all);
    }
    if (b < a.batch) {
      a.x.lengths_out[b] = (int)(have + rows);
      a.x.q_starts[b + 1] = (int)(granted.b + mine.b);
    }
    if (!__syncthreads_or(rows > 1)) {
      const uint32_t at = granted.b + mine.b - 1;
      if (rows) {
        if (need) {
          last_page = a.x.free_pages[count - granted.a - mine.a];
          a.x.table[(size_t)b * a.columns + held] = last_page;
        }
        if (places) {
          a.x.slots[at] = slot_of(a, last_page, have);
          a.x.positions[at] = (int)(prefix + have);
        }
      }
    } else {
      page_sums[t] = mine.a;
      row_sums[t] = mine.b;
      first_column[t] = held;
      first_token[t] = have;
      __syncthreads();
      each<kThreads>(t, all.a,
                     [&](uint32_t i) { return a.x.free_pages[count - 1 - (granted.a + i)]; },
                     [&](uint32_t i, int page) {
                       const uint32_t s = find<kThreads>(page_sums, i);
                       const uint32_t column = first_column[s] + i - (s ? page_sums[s - 1] : 0);
                       a.x.table[(size_t)(b0 + s) * a.columns + column] = page;
                     });
      if (places) {
        __syncthreads();
        const auto position = [&](uint32_t i, uint32_t s) { return first_token[s] + i - (s ? row_sums[s - 1] : 0); };
        each<kThreads>(t, all.b,
                       [&](uint32_t i) {
                         const uint32_t s = find<kThreads>(row_sums, i), at = position(i, s);
                         const int page = a.x.table[(size_t)(b0 + s) * a.columns + (at >> a.page_shift)];
                         return int2{slot_of(a, page, at), (int)(prefix + at)};
                       },
                       [&](uint32_t i, int2 place) {
                         a.x.slots[granted.b + i] = place.x;
                         a.x.positions[granted.b + i] = place.y;
                       });
      }
    }
    granted = {granted.a + all.a, granted.b + all.b};
  }
  if (places)
    for (uint32_t i = granted.b + t; i < a.rows; i += kThreads) a.x.slots[i] = a.x.positions[i] = -1;
  if (t == 0) *a.x.free_count_out = (int)(count - granted.a);
}

// Slots and positions from q_starts, lengths_out and the table: four rows a thread. Where the starts fit LDS the
// searches for the rows' sequences are there. A row behind its sequence's end is most often the next one's; if not (idle
// sequences between them, 65,534 behind the last row at most) it is searched for: passing those one after
// another cost a thread 8.2 ms there, and 51 us where 411 are idle.
constexpr int kPlaceThreads = 256, kPlaceRows = 4, kPlaceStarts = 2048;
__global__ __launch_bounds__(kPlaceThreads) void k_kv4_places(AdvanceArgs a) {
  __shared__ uint32_t ends[kPlaceStarts];
  const uint32_t first = (blockIdx.x * kPlaceThreads + threadIdx.x) * kPlaceRows;
  const int* starts = a.x.q_starts;
  const uint32_t prefix = a.x.prefix_length ? (uint32_t)max(*a.x.prefix_length, 0) : 0;
  const bool in_lds = a.batch < kPlaceStarts;
  if (in_lds) {
    for (uint32_t i = threadIdx.x; i < kPlaceStarts; i += kPlaceThreads)
      ends[i] = i < a.batch ? (uint32_t)starts[i + 1] : ~0u;
    __syncthreads();
  }
  const auto end_of = [&](uint32_t s) { return in_lds ? ends[s] : (uint32_t)starts[s + 1]; };
  // The first sequence from `from` on whose end is past the row; a.batch if there is none.
  const auto search = [&](uint32_t from, uint32_t row) {
    if (in_lds) return find<kPlaceStarts>(ends, row);
    for (uint32_t hi = a.batch; from < hi;) {
      const uint32_t mid = (from + hi) / 2;
      if ((uint32_t)starts[mid + 1] > row) hi = mid; else from = mid + 1;
    }
    return from;
  };
  uint32_t b = search(0, first), end = 0, length = 0;
  const auto take = [&] {
    if (b < a.batch) end = end_of(b), length = (uint32_t)a.x.lengths_out[b];
  };
  take();
  int slot[kPlaceRows], position[kPlaceRows];
#pragma unroll
  for (uint32_t i = 0; i < kPlaceRows; ++i) {
    const uint32_t row = first + i;
    if (b < a.batch && row >= end) {
      if (++b < a.batch && end_of(b) <= row) b = search(b + 1, row);
      take();
    }
    slot[i] = position[i] = -1;
    if (b < a.batch) {
      const uint32_t at = length - (end - row);
      slot[i] = slot_of(a, a.x.table[(size_t)b * a.columns + (at >> a.page_shift)], at);
      position[i] = (int)(prefix + at);
    }
  }
#pragma unroll
  for (uint32_t i = 0; i < kPlaceRows; ++i)
    if (first + i < a.rows) {
      a.x.slots[first + i] = slot[i];
      a.x.positions[first + i] = position[i];
    }
}

}  // namespace

hipError_t launch_kv4_advance(const h3_kv4_cfg& cfg, uint32_t batch, uint32_t table_stride, uint32_t rows,
                              const AdvanceBindings& x, hipStream_t stream) {
  AdvanceArgs a{x, batch, table_stride, rows, cfg.pages, (uint32_t)__builtin_ctz(cfg.page_tokens)};
  const bool apart = rows > kRowsApart;
  if (batch <= 64)
    hipLaunchKernelGGL(k_kv4_advance<256>, dim3(1), dim3(256), 0, stream, a, !apart);
  else
    hipLaunchKernelGGL(k_kv4_advance<1024>, dim3(1), dim3(1024), 0, stream, a, !apart);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || !apart) return e;
  constexpr uint32_t kRows = kPlaceThreads * kPlaceRows;
  hipLaunchKernelGGL(k_kv4_places, dim3((rows + kRows - 1) / kRows), dim3(kPlaceThreads), 0, stream, a);
  return hipGetLastError();
}

}  // namespace h3
