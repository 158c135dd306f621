// Grouped-query attention over the 4-bit paged cache: how a call is cut, and its launches (the kernels are in
// attention_kv4.hpp).
#include "attention_kv4.hpp"

namespace h3 {

// How a call is cut. The host knows no sequence's rows or keys, only that none has more than max_q rows
// and more keys than the table holds (or a window shows); it estimates times, in us from one MI355X's
// figures, and takes the least.
//
// The kernel: up to 32 rows a sequence k_attention_kv4_few or _mid, in tiles of 4, 8, 16 or 32 rows. Beyond,
// tiles of 32 rows there or of 256 in k_attention_kv4_rows: the small ones fill the chip and divide the
// keys where the large ones would leave it idle, the large ones unpack a key once for 256 rows. In us,
// small and large, 4 query heads to each of 8 cache heads: one sequence of 1,000 keys 12 and 26 (64 rows),
// 12 and 39 (256 rows); 64 sequences of 5,000 keys 163 and 253 (48 rows), 630 and 400 (256 rows).
// A call with longer sequences that are not all alike may hold single tokens too (prompts beside
// decoding): beside large tiles those have a launch of their own, in tiles of their heads; a launch's
// workgroups for sequences of the other kind leave at once. A prompt of 300 tokens beside single tokens of up to 2,000 keys, in small tiles
// alone and in both: 33 and 74 us (8 of them), 51 and 75 (32); up to 500 keys, 168 and 95 (512).
namespace {

constexpr double kLeave = 0.6e-3;  // us for a workgroup that has no rows, where sequences differ in length

// k_attention_kv4_few or _mid for sequences of up to `rows` rows, and its time (all_rows: of all
// sequences; keys: of a tile, of which its rows see the part `seen` on average). The keys are divided in
// the number of parts for which that is least: rounds * (start + steps of a workgroup * step) + the
// join's, with 6 or 7 to start a workgroup and join its waves; per four waves' step 1.2 to 1.8 (256 keys,
// 4 to 16 rows), or 0.95 for each workgroup on a compute unit (128 keys, 32 rows), or what HBM takes for
// the resident workgroups' bytes where that is more (5.0 TB/s, 4.4 with one workgroup a compute unit). The
// join is a launch (5) and writes and reads every part's sums in f32.
// Timed: 16 groups of 129,024 keys 73, 58 and 66 us in 16, 32 and 64 parts; 128 groups of 25 rows over a
// window of 4,096 keys 40, 28, 30 and 28 us in 1, 2, 3 and 4; 512 groups of up to 8,192 keys 78, 83, 84
// and 86 us; 8 groups of 1,000 keys 10.0, 10.4, 10.5 and 9.1 us, where the second launch costs the host more
// than the split gains.
Kv4Launch plan_few(const h3_kv4_cfg& cfg, uint32_t rows, uint32_t batch, double all_rows, uint64_t keys,
                   double seen, uint32_t cus, bool divide, double* time) {
  const uint32_t tile = rows <= 4 ? 4 : rows <= 8 ? 8 : rows <= 16 ? 16 : kMidRows;
  const uint32_t tiles = (rows + tile - 1) / tile;
  const int step_keys = kWaves * (tile == kMidRows ? kMidKeys : kStepKeys);
  const double step = tile <= 4 ? 1.2 : tile <= 8 ? 1.3 : tile <= 16 ? 1.8 : 0.95;
  const double groups = cfg.kv_heads * std::min((double)batch * tiles, all_rows / tile + batch);
  const double slots = 2.0 * cus, start = tile == kMidRows ? 7 : 6;
  const uint64_t steps = (keys + step_keys - 1) / step_keys;
  Kv4Launch p = {tile, tiles, 1, 0, rows};
  const double part_bytes = (double)batch * rows * cfg.kv_heads * (cfg.head_dim + 2) * 4;
  for (uint32_t n = 1; n <= (divide ? kMaxParts : 1) && (n == 1 || n <= steps); ++n) {
    if (n > 1 && n * part_bytes > kFewBytes) break;
    const double wgs = groups * n;
    const double each = std::ceil(std::min(wgs, slots) / cus);  // on the fullest compute units
    const double hbm = (each > 1 ? each * cus : wgs) * step_keys * (cfg.head_dim + 8) /
                       (each > 1 ? 5.0e6 : 4.4e6);
    const double one = std::max(tile == kMidRows ? step * each : step, hbm);
    const double longest = (double)((steps + n - 1) / n), usual = longest * seen;
    const double t = std::max(std::ceil(wgs / slots) * (start + usual * one), start + longest * one) +
                     (n > 1 ? 5 + wgs * std::min(rows, tile) * (cfg.head_dim + 2) * 8 / 4e6 : 0) +
                     kLeave * n * ((double)cfg.kv_heads * batch * tiles - groups);
    if (n == 1 || t < *time) {
      p.parts = n;
      *time = t;
    }
  }
  return p;
}

// k_attention_kv4_rows or _line for sequences of up to `rows` rows, and its time: a workgroup per row tile
// and cache head, or (parts: how many workgroups) one line of all their keys where the workgroups would
// fill the chip badly: 1.1 us (one wave with rows) to 2.3 (eight) per 64 keys and 8 to start a row tile,
// and for the line 12 to find it, a tenth more a step, and the join's traffic, two row tiles' sums a
// workgroup. In us, apart and along a line, 4 query heads to each of 8 cache heads: 1,025 tokens of 8,192
// keys 255 and 200; 512 of 65,536 1,950 and 640; 8,192 of 8,192 620 and 820; 12 times 700 of 5,000 784
// and 787.
Kv4Launch plan_many(const h3_kv4_cfg& cfg, const h3_kv4_attention_cfg& acfg, uint32_t rows, uint32_t batch,
                    uint32_t q_rows, uint32_t max_q, uint64_t keys, double seen, uint32_t cus,
                    bool divide, double* time) {
  const uint32_t group = acfg.heads / cfg.kv_heads;
  Kv4Launch p = {(uint32_t)kTileRows, (rows + kTileRows - 1) / kTileRows, 1, 1, rows};
  const double step = 0.9 + 0.175 * std::min(8u, (rows + 31) / 32);  // by the waves that have rows
  const uint32_t tiles = line_tiles(batch, q_rows, max_q, group);
  const double most = (double)((keys + kTileKeys - 1) / kTileKeys);  // steps of a row tile
  const bool alike = (uint64_t)batch * max_q == q_rows;
  const double wgs =
      cfg.kv_heads * (alike ? tiles : std::min<double>(tiles, (double)q_rows * group / kTileRows + 1));
  const double all = wgs * most * seen;
  const double apart = wgs <= cus ? most : std::max<double>(most, all / cus + most * 0.5 * cus / wgs);
  *time = 4 + 8 * std::max(1.0, wgs / cus) + apart * step +
          kLeave * std::max(0.0, (double)cfg.kv_heads * batch * p.row_tiles - wgs);
  if (divide && tiles <= (uint32_t)kLineTiles && batch <= (uint32_t)kLineTiles &&
      tiles * (most + 2) * cfg.kv_heads < (1u << 30)) {
    const double lines = std::min<double>(cus, std::max(1.0, all / kLeastSteps));
    const double sums = 2 * lines * std::min(rows, (uint32_t)kTileRows) * (cfg.head_dim + 2) * 4;
    const double line = 12 + 8 * (wgs / lines + 1) + 1.1 * all / lines * step + 2 * sums / 4e6;
    if (line < *time) {
      p.parts = std::max(2u, (uint32_t)lines);
      *time = line;
    }
  }
  return p;
}

}  // namespace

Kv4Plan kv4_plan(const h3_kv4_cfg& cfg, const h3_kv4_attention_cfg& acfg, uint32_t batch,
                 uint32_t q_rows, uint32_t max_q, uint32_t cus, bool divide) {
  return kv4_front_plan(cfg, acfg, 0, batch, q_rows, max_q, cus, divide);
}

Kv4Plan kv4_front_plan(const h3_kv4_cfg& cfg, const h3_kv4_attention_cfg& acfg, uint64_t front_keys,
                       uint32_t batch, uint32_t q_rows, uint32_t max_q, uint32_t cus, bool divide,
                       double* time) {
  const uint32_t group = acfg.heads / cfg.kv_heads, rows = max_q * group;
  const bool alike = (uint64_t)batch * max_q == q_rows;  // every sequence has max_q rows
  const uint64_t all_keys = (uint64_t)acfg.table_stride * cfg.page_tokens + (acfg.window ? 0 : front_keys);
  const auto tile_keys = [&](uint32_t tile) {  // what the rows of a tile see at most
    return acfg.window ? std::min<uint64_t>(all_keys, acfg.window + front_keys + tile / group + 1)
                       : all_keys;
  };
  // A causal prompt's rows see half of its own keys on average.
  const double seen =
      acfg.causal && !acfg.window ? 1 - std::min<uint64_t>(all_keys, max_q) / 2.0 / all_keys : 1;
  Kv4Plan p{};
  double least = 1e30;
  const auto take = [&](const Kv4Launch& many, const Kv4Launch& few, double t) {
    if (t < least) p = {many, few}, least = t;
    if (time) *time = least;
  };
  double small = 0, large = 0, singles = 0;
  if (rows <= kFewMost) {
    const Kv4Launch all = plan_few(cfg, rows, batch, (double)q_rows * group, tile_keys(kMidRows), seen, cus,
                                   divide, &small);
    take(Kv4Launch{}, all, small);
  }
  if (rows <= kFewRows) return p;
  Kv4Launch many = plan_many(cfg, acfg, rows, batch, q_rows, max_q, tile_keys(kTileRows), seen, cus, divide,
                             &large);
  if (alike || group > kFewRows) {
    take(many, Kv4Launch{}, large);
    return p;
  }
  const Kv4Launch few = plan_few(cfg, group, batch, (double)batch * group, tile_keys(0), 1, cus, divide,
                                 &singles);
  many.rows_from = group + 1;
  take(many, few, large + singles);
  return p;
}

namespace {

constexpr double kSharedBytes = 200e6;  // of the sums of a shared call

// Workgroups of k_attention_kv4_few or _mid with `steps` of their four waves' steps each, over keys that many of them
// share: us alone on a compute unit, and of one of 512 beside another (`each`: its part of the launch's time). Per
// step 1.2 alone and 2.3 beside another (4 rows, 256 keys), 1.0 and 1.4 (32 rows, 128 keys).
struct Work {
  double alone, each;
};
Work few_work(uint32_t tile, double steps, uint32_t cus) {
  const double one = tile <= 4 ? 1.2 : tile <= 8 ? 1.3 : tile <= 16 ? 1.8 : 1.03;
  const double two = tile <= 4 ? 2.3 : tile <= 8 ? 2.5 : tile <= 16 ? 3.4 : 1.4;
  return tile == kMidRows ? Work{7 + steps * one, (3 + steps * two) / (2 * cus)}
                          : Work{5 + steps * one, (4 + steps * two) / (2 * cus)};
}
double few_steps(uint32_t tile, double keys) { return keys / (kWaves * (tile == kMidRows ? kMidKeys : kStepKeys)); }

}  // namespace

// Estimated as above, by the workgroups' work rather than HBM's rate, since the prefix comes from the caches. In us, in
// one pass, shared in tiles of 32 (in parts) and along a line of tiles of 256, 4 query heads to each of 8 cache heads:
//   rows (sequences x new tokens)     keys: prefix, own   one pass   tiles of 32    of 256
//   64 x 1                            8,192, 700 at most   79         33 (4)         54
//   16 x 1                            2,000, 300           17         12 (8)         30
//   64 x 1                            1,000, 700           22         22 (1)         49
//   32 x 1                            30,000, 300          118        39 (16)        59
//   400 x 1                           3,000, 300           173        70 (1, apart)  112
//   32 x 9                            10,000, 500          129        92 (4)         112
//   4 x 130                           20,000, 130          303                       241
//   8 x 257                           31,104, 257          1,400                     1,149
//   8 x 257                           2,000, 257           155                       168
// and with long keys of their own, which a shared call does not divide:
//   2 x 1                             31,104, 31,104       26         151 (3)        186
//   8 x 1                             31,104, 8,192        49         47 (8)         82
//   8 x 1                             8,192, 8,192         27         47 (2)         65
//   64 x 1                            8,192, 8,192         142        98 (1)         131
// (a captured run, three caches in turn). It takes the least of a line, or one 2 us from it.
Kv4PrefixPlan kv4_prefix_plan(const h3_kv4_cfg& cfg, const h3_kv4_attention_cfg& acfg, uint32_t prefix_stride,
                              uint32_t batch, uint32_t q_rows, uint32_t max_q, uint32_t cus, bool divide) {
  const uint64_t prefix = (uint64_t)prefix_stride * cfg.page_tokens;
  const uint64_t own_keys = (uint64_t)acfg.table_stride * cfg.page_tokens;
  const uint32_t group = acfg.heads / cfg.kv_heads;
  const uint64_t rows = (uint64_t)q_rows * group;  // of a cache head
  Kv4PrefixPlan p{};
  double least = 0, own_time = 0;
  p.one = kv4_front_plan(cfg, acfg, prefix, batch, q_rows, max_q, cus, divide, &least);
  const double row_bytes = (double)rows * cfg.kv_heads * (cfg.head_dim + 2) * 4;
  if (!divide || row_bytes > kSharedBytes) return p;
  const auto groups_of = [&](const Kv4Launch& few) {  // workgroups of a part of few rows
    return cfg.kv_heads * std::min((double)batch * few.row_tiles, (double)rows / few.tile_rows + batch);
  };
  const auto join = [&](uint32_t parts) { return 3.5 + 0.15 * parts + parts * row_bytes * 2 / 4e6; };
  if (p.one.many.row_tiles == 0) {
    const Kv4Launch& few = p.one.few;
    const Work w = few_work(few.tile_rows, few_steps(few.tile_rows, (double)(prefix + own_keys)) / few.parts, cus);
    const double wgs = groups_of(few) * few.parts;
    least = (wgs <= cus ? w.alone : std::max(w.alone, 2 + wgs * w.each)) + (few.parts > 1 ? join(few.parts) : 0);
  }
  p.own = kv4_front_plan(cfg, acfg, 0, batch, q_rows, max_q, cus, false, &own_time);
  const bool small = p.own.many.row_tiles == 0;
  const Work own = few_work(p.own.few.tile_rows, few_steps(p.own.few.tile_rows, (double)own_keys), cus);
  const double own_each = small ? groups_of(p.own.few) * own.each : 0;
  if (small) own_time = std::max(own.alone, 2 + own_each);
  const auto take = [&](double time, uint32_t front_parts, uint32_t front_groups, uint32_t parts, bool apart) {
    if (parts > kJoinParts || parts * row_bytes > kSharedBytes || time >= least) return;
    least = time;
    p.shared = true;
    p.heads_apart = apart;
    p.front_parts = front_parts;
    p.front_groups = front_groups;
    p.parts = parts;
  };
  // Tiles of 32 rows, in one launch with the sequences' own where those are few. It has all workgroups in one dimension
  // of the grid, which holds 2^32 threads at most.
  const auto fits = [](uint64_t groups) { return groups * kThreads < (1ull << 32); };
  if (rows <= kFewMost && small) {
    const uint32_t tiles = (uint32_t)(rows + kMidRows - 1) / kMidRows * cfg.kv_heads;
    const double steps = std::max(1.0, few_steps(kMidRows, (double)prefix));
    // Own keys of a head by one wave: a workgroup for four heads, each step of which takes four times as long.
    const double each_keys = few_steps(p.own.few.tile_rows, (double)own_keys) * kWaves;
    const Work wide = few_work(p.own.few.tile_rows, each_keys, cus);
    const double wide_each = (double)batch * ((cfg.kv_heads + kWaves - 1) / kWaves) * wide.each;
    for (uint32_t n = 1; n <= steps && n < kJoinParts; n += 1 + n / 8) {  // (the estimate is flat between)
      const Work w = few_work(kMidRows, steps / n, cus);
      // More of them than find room: the last ones leave the chip partly idle.
      const double tail = tiles * n > 2 * cus ? 0.4 * w.each * 2 * cus : 0;
      const double front = 6 + (double)tiles * n * w.each + tail;
      // The longest of them, one to a compute unit slower by a third while `beside` us of the sequences' own run there
      // too, or two beside each other.
      const auto longest = [&](double beside) {
        const double walk = steps / n * 1.03;
        return 7 + (tiles * n <= cus ? walk + 0.33 * std::min(walk, beside) : 2 * walk);
      };
      if (fits((uint64_t)batch * cfg.kv_heads * p.own.few.row_tiles + n * tiles))
        take(std::max({longest(2 * own_each), own.alone, front + own_each}) + join(1 + n), n, n * tiles, 1 + n, false);
      if (p.own.few.tile_rows < kMidRows && fits((uint64_t)batch * ((cfg.kv_heads + kWaves - 1) / kWaves) + n * tiles))
        take(std::max({longest(2 * wide_each), 5 + wide.each * 2 * cus, front + wide_each}) + join(1 + n), n,
             n * tiles, 1 + n, true);
    }
  }
  // Tiles of 256 rows along one line.
  const uint64_t tiles = (rows + kTileRows - 1) / kTileRows * cfg.kv_heads;
  const double steps = (double)((prefix + kTileKeys - 1) / kTileKeys), all = tiles * steps;
  if (all < (1u << 30)) {
    const uint32_t groups = (uint32_t)std::min<double>(cus, std::max(1.0, all / kLeastSteps));
    const uint32_t pieces = (uint32_t)((groups + tiles - 1) / tiles) + 1;
    const double step = 0.9 + 0.175 * std::min<double>(8, (rows + 31) / 32);
    take(own_time + 12 + 8 * (tiles / (double)groups + 1) + all / groups * step + join(1 + pieces), 0, groups,
         1 + pieces, false);
  }
  return p;
}

size_t kv4_prefix_workspace_bytes(const h3_kv4_cfg& cfg, const h3_kv4_attention_cfg& acfg, uint32_t batch,
                                  uint32_t q_rows, const Kv4PrefixPlan& plan) {
  if (!plan.shared) return kv4_workspace_bytes(cfg, batch, plan.one);
  return (size_t)plan.parts * q_rows * acfg.heads * (cfg.head_dim + 2) * 4;
}

size_t kv4_workspace_bytes(const h3_kv4_cfg& cfg, uint32_t batch, const Kv4Plan& plan) {
  const size_t row = (cfg.head_dim + 2) * 4;
  size_t bytes = 0;
  if (plan.few.parts > 1)
    bytes = (size_t)plan.few.parts * batch * plan.few.rows_to * cfg.kv_heads * row;
  if (plan.many.parts > 1)
    bytes = std::max(bytes, (size_t)2 * plan.many.parts * kTileRows * row + sizeof(Line));
  return bytes;
}

hipError_t launch_attention_kv4(const h3_kv4_cfg& cfg, const h3_kv4_attention_cfg& acfg,
                                const Kv4Plan& plan, uint32_t batch, uint32_t q_rows,
                                uint32_t max_q, const Kv4Bindings& x, hipStream_t stream) {
  return launch_keys<kOwn>(cfg, make_args(cfg, acfg, batch, q_rows, max_q, x), plan, stream);
}

}  // namespace h3
