// Attention over the 4-bit cache behind a prefix that all sequences share, out of the kernels of attention_kv4.hpp.
//
// The softmax over a row's keys, the prefix's F and its own O, is that of two partial ones: with m the largest
// score, l = sum e^(s - m) and o = sum e^(s - m) v over each,
//   out = (e^(m_F - m) o_F + e^(m_O - m) o_O) / (e^(m_F - m) l_F + e^(m_O - m) l_O),  m = max(m_F, m_O).
// Where sequences have few rows, all rows of the call are one matrix against the prefix (F), in tiles of 32 rows
// or of 256, so that each of its keys is unpacked once for as many rows; their own keys (O) are
// attention_kv4's. Both leave m, l and o in the workspace and a join ends the rows. Calls that gain nothing by that
// (few rows in all, or sequences that fill tiles by themselves) take every row over F and then O in one pass.
//
// 4 query heads to each of 8 cache heads of 128 channels: 64 sequences of up to 700 keys of their own behind 8,192,
// 29 us and 5 for the join (79 in one pass), bound by what starts a workgroup and by vector issue beside the products
// (43 and 14 % busy); 8 times 257 rows behind 31,104, 1,137 us, 39 for their own keys and 31 for the join (1,400),
// bound as k_attention_kv4_rows is, whose loop it runs (vector pipe 53 and matrix pipe 48 % busy).
#include "attention_kv4.hpp"

namespace h3 {
namespace {

// All rows over the prefix in tiles of 256: the tiles' steps of every cache head are one line, as
// k_attention_kv4_line's, of which each workgroup takes an equal range. The tiles are alike, so that a tile's pieces
// follow from its number: piece i of it is the prefix's part i. The line is of the rows that there are: where a call has
// places for more (a captured step's padding) their sums have room for more pieces, and the line is divided
// as finely: 64 tokens of 2,056 places behind 31,104 keys 99 us (all places' rows multiplied 1,001). A tile of n steps
// in ranges of n / (most - 1) and more has `most` pieces at most; without padding those of the plan's.
struct FrontLine {
  int rows, each, steps, range;  // of a cache head, its tiles; of a tile; of a workgroup
};
__device__ __forceinline__ FrontLine front_line(const Args& a, int tokens, int length) {
  const int rows = tokens * (int)a.group, each = (rows + kTileRows - 1) / kTileRows, groups = (int)a.front_groups;
  const int steps = max((length + kTileKeys - 1) / kTileKeys, 1);
  int range = max((steps * each * (int)a.kv_heads + groups - 1) / groups, kLeastSteps);
  if (rows < (int)a.part_rows) {
    const int most = (int)min(a.front_places / (uint32_t)max(rows, 1), kJoinParts - 1);
    range = max(range, (steps + most - 2) / (most - 1));
  }
  return {rows, each, steps, range};
}

template <int D, bool kBf16>
__global__ __launch_bounds__(kRowsThreads, 2) void k_attention_kv4_front(Args a) {
  __shared__ __attribute__((aligned(16))) RowsLds<D> lds;
  const Sequence seq = sequence<kFrontPart>(a, 0);
  const FrontLine line = front_line(a, seq.rows, seq.length);
  const int each = line.each, tiles = each * (int)a.kv_heads;
  const int begin = (int)blockIdx.x * line.range, stop = min(begin + line.range, line.steps * tiles);
  for (int at = begin; at < stop;) {
    const int tile = at / line.steps, start = tile * line.steps, first = at - start;
    const int last = min(line.steps, first + stop - at);
    const int head = tile / each, piece = (int)blockIdx.x - start / line.range;
    attend_rows<D, kBf16, kFrontPart>(a, lds, seq, 0, head, (tile - head * each) * kTileRows, {first, last}, piece);
    __syncthreads();  // LDS is free again
    at += last - first;
  }
}

// The first workgroups take all rows over the prefix in tiles of 32, the others the sequences' own keys, in
// tiles of R rows or (0) of 32; kShare: see attend_few.
template <int D, bool kBf16, int R, int kShare>
__global__ __launch_bounds__(kThreads, 2) void k_attention_kv4_shared(Args own, Args front) {
  union Lds {
    MidLds<D> mid;
    FewLds<D, R ? R : 4> few;
  };
  __shared__ Lds lds;
  uint32_t x = blockIdx.x;
  if (x < front.front_groups) {
    const uint32_t y = x / front.parts;
    attend_mid<D, kBf16, false, kFrontPart>(front, lds.mid, x - y * front.parts, y, 0);
    return;
  }
  x -= front.front_groups;
  if constexpr (kShare == 1) {
    const uint32_t each = (own.kv_heads + kWaves - 1) / kWaves, b = x / each;
    const uint32_t head = (x - b * each) * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (head < own.kv_heads) attend_few<D, kBf16, R, false, kOwnPart, 1>(own, lds.few, 0, head, b);
    return;
  }
  const uint32_t tiles = own.kv_heads * own.row_tiles, b = x / tiles;
  if constexpr (R == 0)
    attend_mid<D, kBf16, false, kOwnPart>(own, lds.mid, 0, x - b * tiles, b);
  else
    attend_few<D, kBf16, R, false, kOwnPart>(own, lds.few, 0, x - b * tiles, b);
}

template <int D, bool kBf16, int R>
void launch_tiles_shared(const Args& own, const Args& front, bool heads_apart, hipStream_t stream) {
  if constexpr (R != 0) {
    if (heads_apart) {
      const uint32_t groups = front.front_groups + (own.kv_heads + kWaves - 1) / kWaves * own.batch;
      hipLaunchKernelGGL((k_attention_kv4_shared<D, kBf16, R, 1>), dim3(groups), dim3(kThreads), 0, stream, own, front);
      return;
    }
  }
  const uint32_t groups = front.front_groups + own.kv_heads * own.row_tiles * own.batch;
  hipLaunchKernelGGL((k_attention_kv4_shared<D, kBf16, R, kWaves>), dim3(groups), dim3(kThreads), 0, stream, own,
                     front);
}

// Whether a token's row is one that its sequence takes. 64 ends at a time, a lane each: the first past the token is
// the sequence's. (No row from the last sequence's end on has sums over the prefix.)
__device__ __forceinline__ bool taken(const Args& a, int token, int lane) {
  const int end = a.q_starts[a.batch];
  int b = 0;
  for (int span = (int)a.batch; span > 0;) {  // the sequence is one of b .. b + span - 1, or there is none
    const int each = (span + 63) / 64, last = min(b + (lane + 1) * each, b + span) - 1;
    const uint64_t past = __ballot(a.q_starts[last + 1] > token);
    if (past == 0) return false;
    const int chunk = __builtin_ctzll(past) * each;
    if (each == 1) {
      b += chunk;
      break;
    }
    span = min(each, span - chunk);
    b += chunk;
  }
  const int start = max(a.q_starts[b], 0);
  return token >= start && token - start < (int)a.max_q && token < end;
}

// Joins a row's parts, its own and then the prefix's: W waves per (row, query head), wave w the parts w, w + W, ..;
// lane p of a wave holds part p's weight.
template <int D, bool kBf16, int W>
__global__ __launch_bounds__(kThreads) void k_attention_kv4_shared_join(Args a) {
  constexpr int kPer = D / 64;
  __shared__ float lds_sum[W == 1 ? 1 : W][D];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t at = blockIdx.x * (kWaves / W) + wave / W;
  if (at >= a.part_rows) return;
  const uint32_t token = at / a.group, g = at - token * a.group;
  int front = (int)a.front_parts;
  uint32_t pitch = a.part_rows;
  if (front == 0) {
    const int length = min(max(*a.prefix_length, 0), (int)(a.prefix_stride << a.page_shift));
    const FrontLine line = front_line(a, min(max(a.q_starts[a.batch], 0), (int)a.q_rows), length);
    if ((int)at >= line.rows) return;
    const int tile = (int)blockIdx.y * line.each + (int)at / kTileRows;
    front = (tile * line.steps + line.steps - 1) / line.range - tile * line.steps / line.range + 1;
    pitch = (uint32_t)line.rows;
  }
  const int parts = 1 + front;
  // Of the row's part p: in 32 bits, as the workspace is 200 MB at most. Part p - 1 of the prefix's is pitch * (p - 1) on.
  const uint32_t own = at * a.kv_heads + blockIdx.y, step = pitch * a.kv_heads;
  const uint32_t behind = own + (a.part_rows - pitch) * a.kv_heads;
  const auto place = [&](uint32_t p) { return p ? behind + p * step : own; };
  const float2 ml = lane < parts ? a.part_ml[place(lane)] : float2{-kInf, 0.0f};
  float x[4][kPer];
  const auto load = [&](int p0) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float* from = a.part_o + (size_t)place(p0 + i * W) * D + lane * kPer;
#pragma unroll
      for (int d = 0; d < kPer; ++d) x[i][d] = p0 + i * W < parts ? from[d] : 0.0f;
    }
  };
  load(wave % W);  // under way before the row is known to be one
  if (!taken(a, (int)token, lane)) return;  // whole workgroups where W waves share a row
  const float top = across32<true>(across16<true>(over16<true>(ml.x)));
  const float f = __builtin_amdgcn_exp2f(ml.x - (top == -kInf ? 0.0f : top));
  const float total = across32<false>(across16<false>(over16<false>(f * ml.y)));
  const uint64_t live = __ballot(!(ml.y == 0.0f));  // the parts with sums: those with a weight or a NaN
  float sum[kPer];
#pragma unroll
  for (int d = 0; d < kPer; ++d) sum[d] = 0.0f;
  for (int p0 = wave % W; p0 < parts; p0 += 4 * W) {
    if (p0 >= 4 * W) load(p0);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int p = p0 + i * W;
      if (p >= parts || !((live >> p) & 1)) continue;
      const float w = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(f), p));
#pragma unroll
      for (int d = 0; d < kPer; ++d) sum[d] = fmaf(w, x[i][d], sum[d]);
    }
  }
  if constexpr (W > 1) {
#pragma unroll
    for (int d = 0; d < kPer; ++d) lds_sum[wave][lane * kPer + d] = sum[d];
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int d = 0; d < kPer; ++d) {
      sum[d] = 0.0f;
#pragma unroll
      for (int w = 0; w < W; ++w) sum[d] += lds_sum[w][lane * kPer + d];
    }
  }
  write_row<D, kBf16>(a, token, blockIdx.y * a.group + g, lane, top, total, sum);
}

template <int D, bool kBf16>
hipError_t launch_shared(const Args& all, const Kv4PrefixPlan& plan, hipStream_t stream) {
  const uint32_t rows = all.q_rows * all.group;
  Args own = all;  // part_ml is the same for every launch: behind all parts' sums
  own.part_rows = rows;
  own.part_ml = reinterpret_cast<float2*>(all.part_o + (size_t)plan.parts * rows * all.kv_heads * D);
  own.parts = 1;
  Args front = own;
  front.batch = 1;
  front.max_q = front.q_rows;
  front.table = all.prefix_table;
  front.table_stride = all.prefix_stride;
  front.q_starts = all.q_starts + all.batch;
  front.parts = plan.front_parts;
  front.front_parts = plan.front_parts;
  front.front_groups = plan.front_groups;
  front.front_places = (plan.parts - 1) * rows;
  front.rows_from = 0;
  front.rows_to = rows;
  Args few = own;
  few.row_tiles = plan.own.few.row_tiles;
  few.rows_from = plan.own.few.rows_from;
  few.rows_to = plan.own.few.rows_to;
  const dim3 block(kThreads);
  if (plan.front_parts) {
    front.row_tiles = (rows + kMidRows - 1) / kMidRows;
    switch (plan.own.few.tile_rows) {
      case 4: launch_tiles_shared<D, kBf16, 4>(few, front, plan.heads_apart, stream); break;
      case 8: launch_tiles_shared<D, kBf16, 8>(few, front, plan.heads_apart, stream); break;
      case 16: launch_tiles_shared<D, kBf16, 16>(few, front, plan.heads_apart, stream); break;
      default: launch_tiles_shared<D, kBf16, 0>(few, front, false, stream);
    }
  } else {
    hipLaunchKernelGGL((k_attention_kv4_front<D, kBf16>), dim3(front.front_groups), dim3(kRowsThreads), 0, stream,
                       front);
    if (plan.own.many.row_tiles) {
      Args many = own;
      many.row_tiles = plan.own.many.row_tiles;
      many.rows_from = plan.own.many.rows_from;
      many.rows_to = plan.own.many.rows_to;
      hipLaunchKernelGGL((k_attention_kv4_rows<D, kBf16, kOwnPart>), dim3(all.kv_heads * many.row_tiles, 1, all.batch),
                         dim3(kRowsThreads), 0, stream, many);
    }
    if (few.row_tiles) launch_tiles<D, kBf16, false, kOwnPart>(few, plan.own.few, stream);
  }
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  Args join = own;
  join.front_parts = plan.front_parts;
  join.front_groups = plan.front_groups;
  join.front_places = front.front_places;
  if (plan.parts > 8)
    hipLaunchKernelGGL((k_attention_kv4_shared_join<D, kBf16, kWaves>), dim3(rows, all.kv_heads), block, 0, stream,
                       join);
  else
    hipLaunchKernelGGL((k_attention_kv4_shared_join<D, kBf16, 1>), dim3((rows + kWaves - 1) / kWaves, all.kv_heads),
                       block, 0, stream, join);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_attention_kv4_prefix(const h3_kv4_cfg& cfg, const h3_kv4_attention_cfg& acfg,
                                       uint32_t prefix_stride, const Kv4PrefixPlan& plan, uint32_t batch,
                                       uint32_t q_rows, uint32_t max_q, const Kv4Bindings& x,
                                       hipStream_t stream) {
  Args a = make_args(cfg, acfg, batch, q_rows, max_q, x);
  a.prefix_stride = prefix_stride;
  if (!plan.shared) return launch_keys<kPrefix>(cfg, a, plan.one, stream);
  const bool bf16 = cfg.elem == H3_ELEM_BF16;
  if (cfg.head_dim == 128)
    return bf16 ? launch_shared<128, true>(a, plan, stream) : launch_shared<128, false>(a, plan, stream);
  return bf16 ? launch_shared<64, true>(a, plan, stream) : launch_shared<64, false>(a, plan, stream);
}

}  // namespace h3
