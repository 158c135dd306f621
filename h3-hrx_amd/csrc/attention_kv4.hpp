// Grouped-query attention over the 4-bit paged cache of kv4.hip, on gfx950.
//
// The codes go into the matrix instructions as they are. With k_j = m_j + s_j u_j (u whole numbers
// 0..15) a score is
//   q . k_j = s_j (q . (16 + u_j)) + (m_j - 16 s_j) sum(q),
// exact products of q with small integers, and one multiplication and one FMA in f32 per score.
// 16 + u is a 16-bit float by one shift and one AND-OR (v_and_or_b32) per pair of codes: the code's
// bits are the top four mantissa bits under the exponent of 16, in f16 and in bf16. The values,
//   sum_j p_j v_j = sum_j (p_j s_j) (u_j - 8) + sum_j p_j (m_j + 8 s_j),
// take the scale into the probability. The first sum is the MFMA's over 16 + u less 24 times the
// sum of the same rounded p s, which one more MFMA with a row of ones gives, so what p s loses in
// rounding to 16 bits multiplies u - 8, as in an attention over centred 16-bit values; the second
// sum is kept in f32. In f16, p s is held relative to the largest scale so far (a power of two,
// raised as the running maximum is), times 2^8: weights down to 2^-22 of the largest stay normal.
// (With 256 rows to a tile of keys the values are formed once for all of them instead, in LDS.)
//
// A query row is one (token, query head) pair; the G = heads / kv_heads heads of one cache head
// are rows of the same matrix, row = token * G + g, so that a key is read once for all of them.
#pragma once

#include <algorithm>
#include <cmath>

#include "internal.hpp"

namespace h3 {
namespace {

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kInf = __builtin_inff();

// The keys that a launch's rows see: their own sequence's; with its first tokens outside the window too; behind a
// prefix that all sequences share; their own sequence's alone, or that prefix alone, of the rows of all sequences as
// one's, their sums left in the workspace for the join of the two.
enum Keys { kOwn, kSinks, kPrefix, kOwnPart, kFrontPart };
template <Keys K> constexpr bool kPart = K == kOwnPart || K == kFrontPart;
template <Keys K> constexpr bool kPlain = K != kSinks && K != kPrefix;  // nothing lies before span(i)

constexpr uint32_t kJoinParts = 64;  // parts of a row behind a prefix at most: the lanes of the join's wave

struct Args {
  const void* q;
  const uint8_t* cache;
  const int32_t* table;
  const int32_t* prefix_table;   // kPrefix
  const int32_t* prefix_length;  // kPrefix, kFrontPart: one
  const int32_t* lengths;
  const int32_t* q_starts;       // kFrontPart: the end of the last sequence's rows, one
  void* out;
  float* lse;  // null: not wanted
  float* part_o;
  float2* part_ml;
  struct Line* line;
  uint32_t kv_heads, group, q_stride, out_stride, table_stride;
  uint32_t pages, page_shift;
  uint32_t batch, q_rows, max_q;
  uint32_t parts, row_tiles;    // row_tiles: a sequence's at most; of a line, all sequences'
  uint32_t rows_from, rows_to;  // the sequences a launch takes: those of rows_from .. rows_to rows
  uint32_t causal, window;
  uint32_t sinks;          // kSinks: the first tokens
  uint32_t prefix_stride;  // kPrefix: pages that prefix_table holds
  uint32_t part_rows;    // kPart: the call's rows (tokens times group), places of the own keys' sums
  uint32_t front_parts;  // kPart: the parts that the prefix's sums are in (0: pieces of a line, front_groups long)
  uint32_t front_groups, front_places;  // front_places: rows of the prefix's sums that the workspace holds
  float scale;  // the softmax scale times log2(e)
};

// A sequence's rows and keys, from device memory and so checked here: rows that q does not have,
// or past max_q, are not computed, keys past the table's columns not read.
// Keys are counted from the sequence's first token, behind a prefix from `base` on: the least multiple of
// a page and of kFrontUnit that the prefix's keys 0 .. front - 1 lie before, so that a step's or a page's keys are all
// the prefix's or all the sequence's. Row i sees the keys of span(i) and, before them, all below `front`.
constexpr int kFrontUnit = 64;
struct Sequence {
  int start, n, rows, length;  // first row of q, its rows, the rows computed, keys
  int front, base;             // (kOwn: not looked at)
};
template <Keys K>
__device__ __forceinline__ Sequence sequence(const Args& a, uint32_t b) {
  Sequence s;
  s.front = s.base = 0;
  if constexpr (K == kFrontPart) {
    s.start = 0;
    s.n = s.rows = min(max(*a.q_starts, 0), (int)a.q_rows);
    s.length = min(max(*a.prefix_length, 0), (int)(a.table_stride << a.page_shift));
    return s;
  }
  if constexpr (K == kSinks) s.front = (int)a.sinks;
  if constexpr (K == kPrefix) {
    const int unit = max(1 << a.page_shift, kFrontUnit);
    s.front = min(max(*a.prefix_length, 0), (int)(a.prefix_stride << a.page_shift));
    s.base = (s.front + unit - 1) & -unit;
  }
  const int total = (int)a.q_rows;
  s.start = min(max(a.q_starts[b], 0), total);
  const int end = min(max(a.q_starts[b + 1], s.start), total);
  s.n = end - s.start;
  s.rows = min(s.n, (int)a.max_q);
  s.length = min(max(a.lengths[b], 0), (int)(a.table_stride << a.page_shift));
  return s;
}

__device__ __forceinline__ bool takes(const Args& a, int rows) {
  return rows >= (int)a.rows_from && rows <= (int)a.rows_to;
}

// The keys [lo, hi) that a sequence's token i sees.
template <Keys K>
__device__ __forceinline__ int2 span(const Args& a, const Sequence& s, int i) {
  const int base = K == kPrefix ? s.base : 0;
  if (K == kFrontPart || !a.causal) return {base, base + s.length};
  const int p = s.length - s.n + i;
  const int hi = min(max(p + 1, 0), s.length);
  const int lo = a.window ? (int)max((int64_t)p + 1 - a.window, (int64_t)0) : 0;
  return {base + min(lo, hi), base + hi};
}

// Whether a row that sees [seen.x, seen.y) and what lies below `front` before it does not see key `key`.
template <Keys K>
__device__ __forceinline__ bool unseen(const Sequence& s, int2 seen, int key) {
  if constexpr (kPlain<K>) return (key < seen.x) | (key >= seen.y);
  return ((key < seen.x) & (key >= s.front)) | (key >= seen.y);
}
// Whether rows of which each sees all of [lo, hi) see all the `keys` keys from key0 on.
template <Keys K>
__device__ __forceinline__ bool all_seen(const Sequence& s, int lo, int hi, int key0, int keys) {
  if constexpr (kPlain<K>) return key0 >= lo && key0 + keys <= hi;
  return (key0 >= lo || key0 + keys <= s.front) && key0 + keys <= hi;
}

// Steps first .. last - 1 of a row's keys.
struct Steps {
  int first, last;
};

// The steps of kKeys keys that rows with keys [lo, hi) take, counted without those between the front's and
// lo's: step v begins at key key(v).
template <Keys K, int kKeys>
struct Walk {
  int front, gap, first, last;
  __device__ __forceinline__ int key(int v) const {
    if constexpr (kPlain<K>) return v * kKeys;
    return (v < front ? v : v + gap) * kKeys;
  }
};
template <Keys K, int kKeys>
__device__ __forceinline__ Walk<K, kKeys> walk(const Sequence& s, int lo, int hi) {
  const int first = lo / kKeys, end = (hi + kKeys - 1) / kKeys;
  if constexpr (kPlain<K>) return {0, 0, first, end};
  const int front = (min(s.front, hi) + kKeys - 1) / kKeys, gap = max(first - front, 0);
  return {front, gap, 0, max(end - gap, front)};
}

template <bool kBf16>
__device__ __forceinline__ float widen(uint32_t bits) {
  if constexpr (kBf16) return __uint_as_float(bits << 16);
  return (float)__builtin_bit_cast(_Float16, (uint16_t)bits);
}
// Whether either half of a parameter word is a NaN or an infinity.
template <bool kBf16>
__device__ __forceinline__ bool has_nan(uint32_t word) {
  constexpr uint32_t kTop = kBf16 ? 0x7f80u : 0x7c00u;
  return (word & kTop) == kTop || ((word >> 16) & kTop) == kTop;
}
template <bool kBf16>
__device__ __forceinline__ uint32_t narrow(float v) {
  if constexpr (kBf16) return __builtin_bit_cast(uint16_t, (__bf16)v);
  return __builtin_bit_cast(uint16_t, (_Float16)v);
}
template <bool kBf16>
__device__ __forceinline__ uint32_t narrow2(float lo, float hi) {  // one v_cvt_pk
  typedef float v2f __attribute__((ext_vector_type(2)));
  typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
  if constexpr (kBf16)
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v2f{lo, hi}, v2bf));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v2f{lo, hi}, v2h));
}

// The constants that make 16-bit floats of codes, the mask in a scalar and the exponent of 16 in a
// vector register: as literals they would split every AND-OR in two.
struct Codes {
  uint32_t mask, bias;
};
template <bool kBf16>
__device__ __forceinline__ Codes make_codes() {
  Codes c{kBf16 ? 0x00780078u : 0x03C003C0u, kBf16 ? 0x41804180u : 0x4C004C00u};
  asm("" : "+s"(c.mask));
  asm("" : "+v"(c.bias));
  return c;
}

// Nibble n of both halves of w as a pair of 16 + u.
template <bool kBf16>
__device__ __forceinline__ uint32_t code_pair(uint32_t w, int n, const Codes& c) {
  const int shift = (kBf16 ? 3 : 6) - 4 * n;  // to the top of the mantissa
  return ((shift >= 0 ? w << shift : w >> -shift) & c.mask) | c.bias;
}

template <bool kBf16>
__device__ __forceinline__ v4f mfma16(uint4 a, uint4 b, v4f c) {
  if constexpr (kBf16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a),
                                                   __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a),
                                                __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}

template <Keys K>
__device__ __forceinline__ int page_of(const Args& a, const int32_t* table, const Sequence& s, int key) {
  if constexpr (K == kPrefix) {
    const bool front = key < s.base;
    const uint32_t col = (uint32_t)(front ? key : key - s.base) >> a.page_shift;
    const int id = col < (front ? a.prefix_stride : a.table_stride) ? (front ? a.prefix_table : table)[col] : -1;
    return (uint32_t)id < a.pages ? id : -1;
  }
  const uint32_t col = (uint32_t)key >> a.page_shift;
  const int id = col < a.table_stride ? table[col] : -1;
  return (uint32_t)id < a.pages ? id : -1;
}

// Up to 16 rows: a workgroup's four waves hold the same R rows of one cache head and take every
// fourth 64 keys; their results are joined in LDS. Loads of the next 64 keys are in flight over the
// work on these, so the kernel is bound by HBM as long as that work is short, and most of it is
// vector instructions: the unpacking of the codes (one shift and one AND-OR a pair, fixed), then the
// softmax. A 16 x 16 x 32 score tile S = Q K^T of R < 16 rows would leave 16 - R of its rows idle in
// every softmax instruction, so T = 16 / R groups of 16 keys share one: group t meets a copy of Q
// that holds its R rows at rows R t .. and zeros elsewhere, all accumulating into the same tile. A
// lane (n = lane % 16, h = lane / 16) then has rows (4 h + i) % R of key 16 ((4 h) / R) + n: its
// own key's factors, and no copies. Probabilities pass through LDS, [key][R] in 16 bits, and come
// back through the transposed read as the operand of O^T = V^T P^T.
// 64 sequences of up to 8,192 tokens, 4 query heads to each of 8 cache heads: 353 MB in 76 us, 4.7 TB/s
// (more while all of them last; the vector pipe is 37 % busy); two of 129,024, 7 to each, in 32 parts: 281
// MB in 54 us, the join's 5 with it. About 6 us go to the launch, the first loads' chain (length, table, codes)
// and the join of the waves.
constexpr int kStepKeys = 64;
constexpr float kRaise = 7.0f;     // scores may pass m by this (p up to 2^7) before m is raised
constexpr float kHeld = 256.0f;    // f16: p s is held times this over the largest scale

template <int D, int R>
struct Step {
  uint32_t k[4][D / 32];          // key n of each 16: channels D/4 h and on
  uint32_t v[16];                 // keys 32 (e / 8) + 8 h + e % 8: channels D/16 n and on
  uint32_t kw[R / 4], vw[R / 4];  // the words of the lane's key in each score tile
  uint64_t hidden;                // a bit per key: its page is none of the cache's
};

__device__ __forceinline__ const uint8_t* lane_pointer(const uint8_t* p, int lane) {
  const uint64_t x = reinterpret_cast<uint64_t>(p);
  const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)x, lane);
  const uint32_t hi = __builtin_amdgcn_readlane((uint32_t)(x >> 32), lane);
  return reinterpret_cast<const uint8_t*>((uint64_t)hi << 32 | lo);
}

// A load of codes; kOnce: past the caches, where they would not be met again (see reads_once).
template <bool kOnce, typename T>
__device__ __forceinline__ T load_codes(const uint8_t* p) {
  const T* from = reinterpret_cast<const T*>(p);
  return kOnce ? __builtin_nontemporal_load(from) : *from;
}

// `ids`: lane l's is the page of key `key` + l. Sixteen keys lie side by side in a page; each lane
// finds its own key's K codes, and the first lanes of the sixteens lend theirs to all.
template <int D, int R, bool kOnce>
__device__ __forceinline__ void load_step(const Args& a, int ids, uint32_t head, int key, int lane,
                                          Step<D, R>& s) {
  const int n = lane & 15, h = lane >> 4;
  const uint32_t page_tokens = 1u << a.page_shift, mask = page_tokens - 1;
  const uint32_t block = page_tokens * (D + 8);
  // Keys of no page are masked; page 0 is there to read.
  const uint8_t* page = a.cache + (uint64_t)head * block +
                        (uint64_t)(uint32_t)max(ids, 0) * (block * a.kv_heads);
  s.hidden = __ballot(ids < 0);
  const uint8_t* mine = page + (((uint32_t)key + lane) & mask) * (D / 2);
  const uint8_t* at[4];
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    at[t] = lane_pointer(mine, 16 * t);
    typedef uint32_t Row __attribute__((ext_vector_type(D / 32)));
    const Row k = load_codes<kOnce, Row>(at[t] + (n * (D / 2) + (D / 8) * h));
#pragma unroll
    for (int i = 0; i < D / 32; ++i) s.k[t][i] = k[i];
  }
#pragma unroll
  for (int c = 0; c < R / 4; ++c) {
    const int t = c * (16 / R) + 4 * h / R;
    const uint32_t in_page = ((uint32_t)key + 16 * t) & mask;
    const uint8_t* codes = at[0];
    if constexpr (R == 4) codes = mine - n * (D / 2);
    if constexpr (R == 8) {
      const uint8_t *even = at[2 * c], *odd = at[2 * c + 1];
      codes = h >> 1 ? odd : even;
    }
    if constexpr (R == 16) codes = at[c];
    const uint8_t* kw = codes + (page_tokens * D - in_page * (D / 2 - 4) + 4 * n);
    s.kw[c] = *reinterpret_cast<const uint32_t*>(kw);
    s.vw[c] = *reinterpret_cast<const uint32_t*>(kw + page_tokens * 4);
  }
#pragma unroll
  for (int st = 0; st < 2; ++st) {
    const uint8_t *even = at[2 * st], *odd = at[2 * st + 1];
    const uint8_t* vc = (h >> 1 ? odd : even) +
                        (page_tokens * (D / 2) + 8 * (h & 1) * (D / 2) + n * (D / 32));
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if constexpr (D == 128)
        s.v[8 * st + e] = load_codes<kOnce, uint32_t>(vc + e * 64);
      else
        s.v[8 * st + e] = load_codes<kOnce, uint16_t>(vc + e * 32);
    }
  }
}

typedef short v4s __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4s lds_v4s;

// Maximum or sum over 16, 32 or 64 lanes, on the vector pipe: quad_perm [1,0,3,2] and [2,3,0,1],
// row_half_mirror, row_mirror, then the swaps of 16 and of 32 lanes.
template <bool kMax>
__device__ __forceinline__ float both(float x, float y) {
  return kMax ? fmaxf(x, y) : x + y;
}
template <int kCtrl>
__device__ __forceinline__ float dpp(float v) {
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), kCtrl, 0xF, 0xF, true));
}
template <bool kMax>
__device__ __forceinline__ float over16(float v) {
  v = both<kMax>(v, dpp<0xB1>(v));
  v = both<kMax>(v, dpp<0x4E>(v));
  v = both<kMax>(v, dpp<0x141>(v));
  return both<kMax>(v, dpp<0x140>(v));
}
template <bool kMax>
__device__ __forceinline__ float across16(float v) {  // with lane ^ 16
  const auto r =
      __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return both<kMax>(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
template <bool kMax>
__device__ __forceinline__ float across32(float v) {  // with lane ^ 32
  const auto r =
      __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return both<kMax>(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// Over the lanes that hold the same rows: the 16 of a group, and the groups whose 4 h % R is the same.
template <int R, bool kMax>
__device__ __forceinline__ float row_lanes(float v) {
  v = over16<kMax>(v);
  if constexpr (R == 4) v = across16<kMax>(v);
  if constexpr (R <= 8) v = across32<kMax>(v);
  return v;
}

// The sum l of a row's weights: NaN where its sum over values is. A key whose row of V is no number counts as one whose
// score is none (in blocks at a mask's edge it is made one), so that out and lse say so wherever the key lies.
__device__ __forceinline__ float or_nan(float l, float sum) { return sum != sum ? sum : l; }

// A row's results in the element type, from its sums and the sum of its weights. In f16 they are means of finite
// values: rounding the weights to 16 bits (2^-11) may carry a mean of values near 65504 past it, and is not to make it
// infinite. A row whose l is NaN stays NaN.
struct Mean {
  float inv, most;
};
template <bool kBf16>
__device__ __forceinline__ Mean make_mean(float l) {
  return {l == 0.0f ? 0.0f : 1.0f / l, or_nan(kBf16 ? kInf : 65504.0f, l)};
}
template <bool kBf16>
__device__ __forceinline__ float mean(float sum, const Mean& m) {
  const float x = sum * m.inv;
  return kBf16 ? x : fminf(fmaxf(x, -m.most), m.most);
}

// Where part `part` of a row's keys leaves its sums: row `row` (of at most rows_to) of sequence b. Behind a prefix the
// rows' own sums come first, the parts over the prefix after them: of all the call's rows, or along a line of those
// that there are.
template <Keys K>
__device__ __forceinline__ size_t few_place(const Args& a, const Sequence& s, uint32_t part, uint32_t b,
                                            uint32_t row, uint32_t head) {
  if constexpr (K == kOwnPart) return ((size_t)((uint32_t)s.start * a.group) + row) * a.kv_heads + head;
  if constexpr (K == kFrontPart) {
    const uint32_t pitch = a.front_parts ? a.part_rows : (uint32_t)s.rows * a.group;
    return (a.part_rows + (size_t)part * pitch + row) * a.kv_heads + head;
  }
  return (((size_t)part * a.batch + b) * a.rows_to + row) * a.kv_heads + head;
}

template <int D, int R>
struct FewLds {
  __attribute__((aligned(16))) uint16_t p[kWaves][kStepKeys * R];
  __attribute__((aligned(16))) float o[kWaves][R][D + 4];
  float row[kWaves][R];  // a factor per row, from its lanes to its column
  float2 ml[kWaves][R];
};

// kShare: the waves that share a head's keys, all four or (1) each wave a head of its own.
template <int D, bool kBf16, int R, bool kOnce, Keys K, int kShare = kWaves>
__device__ __forceinline__ void attend_few(const Args& a, FewLds<D, R>& lds, uint32_t part, uint32_t head,
                                           uint32_t b) {
  constexpr int T = 16 / R, kTiles = R / 4, kSteps = D / 32, kDimTiles = D / 16;
  auto &lds_p = lds.p;
  auto &lds_o = lds.o;
  auto &lds_row = lds.row;
  auto &lds_ml = lds.ml;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, h = lane >> 4;
  const int32_t* table = a.table + (size_t)b * a.table_stride;
  // Step `part` * 4 + wave of the sequence and every 4 * parts-th after it. Without a window the first
  // is known before the sequence is, and its loads go ahead: where the sequence ends before it, they
  // read what the table holds, and nothing comes of them.
  const Sequence seq = sequence<K>(a, b);
  const int group = (int)a.group, rows = seq.rows * group, stride = (int)a.parts * kShare;
  const int mine = kShare == kWaves ? wave : 0, thread = kShare == kWaves ? (int)threadIdx.x : lane;
  int step = (int)part * kShare + mine;
  Walk<K, kStepKeys> way{};
  if constexpr (kPlain<K>) {
    if (a.window) step += span<K>(a, seq, 0).x / kStepKeys;
  } else {
    way = walk<K, kStepKeys>(seq, span<K>(a, seq, 0).x, span<K>(a, seq, (rows - 1) / group).y);
  }
  int ids = page_of<K>(a, table, seq, way.key(step) + lane);
  Step<D, R> tiles[2];
  load_step<D, R, kOnce>(a, ids, head, way.key(step), lane, tiles[0]);
  ids = page_of<K>(a, table, seq, way.key(step + stride) + lane);
  if (rows == 0 || !takes(a, rows)) return;
  const int2 first_span = span<K>(a, seq, 0), last_span = span<K>(a, seq, (rows - 1) / group);
  const int key_lo = first_span.x, key_hi = last_span.y;  // seen by some row
  const int all_lo = last_span.x, all_hi = first_span.y;  // seen by every row
  const int last = kPlain<K> ? (key_hi + kStepKeys - 1) / kStepKeys : way.last;
  const uint32_t heads = a.kv_heads * a.group;
  if (part > 0 && step - mine >= last) {  // no keys: part 0 stands for an empty row
    if (thread < rows) a.part_ml[few_place<K>(a, seq, part, b, thread, head)] = {-kInf, 0};
    return;
  }

  // Q operands: channel D/4 h + 8 s + {0,4,1,5,2,6,3,7} in k slot 8 h + 0..7 of step s, the order in
  // which the codes of a word come out in pairs. Rows past the last are zeros.
  uint4 qf[T][kSteps];
  float q_sum[4], m[4], l[4], mid[4];  // row (4 h + i) % R; mid: sum p (m + 8 s)
  v4f o[kDimTiles], ones = {0, 0, 0, 0};
  const int q_token = n % R / group, q_g = n % R - q_token * group;
  float q_total = 0.0f;
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    uint4 x = {0, 0, 0, 0};
    if (n % R < rows)
      x = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.q) +
                                          (size_t)(seq.start + q_token) * a.q_stride +
                                          (head * group + q_g) * D + (D / 4) * h + 8 * s);
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) q_total += widen<kBf16>(w[i] & 0xffffu) + widen<kBf16>(w[i] >> 16);
    x = {(x.x & 0xffffu) | (x.z << 16), (x.x >> 16) | (x.z & 0xffff0000u),
         (x.y & 0xffffu) | (x.w << 16), (x.y >> 16) | (x.w & 0xffff0000u)};
#pragma unroll
    for (int u = 0; u < T; ++u) qf[u][s] = n / R == u ? x : uint4{0, 0, 0, 0};
  }
  q_total = across32<false>(across16<false>(q_total));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    q_sum[i] = __shfl(q_total, (4 * h + i) % R);
    m[i] = -kInf;
    l[i] = mid[i] = 0.0f;
  }
#pragma unroll
  for (int d = 0; d < kDimTiles; ++d) o[d] = {0, 0, 0, 0};
  float s_top = 0.0f, s_factor = 0.0f;  // f16: a power of two no scale passes, and kHeld over it
  const uint32_t one2 = kBf16 ? 0x3F803F80u : 0x3C003C00u;
  const uint4 one8 = {one2, one2, one2, one2};
  const Codes codes = make_codes<kBf16>();

  auto attend = [&](const Step<D, R>& cur, Step<D, R>& next) {
    const int key0 = way.key(step);
    if (step + stride < last) {
      const int now = ids;
      ids = page_of<K>(a, table, seq, (kPlain<K> ? key0 + 2 * kStepKeys * stride : way.key(step + 2 * stride)) + lane);
      load_step<D, R, kOnce>(a, now, head, kPlain<K> ? key0 + kStepKeys * stride : way.key(step + stride), lane, next);
    }
    // Scores.
    v4f acc[kTiles];
#pragma unroll
    for (int c = 0; c < kTiles; ++c) {
      acc[c] = {0, 0, 0, 0};
#pragma unroll
      for (int u = 0; u < T; ++u)
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
          const uint32_t w = cur.k[c * T + u][s];
          const uint4 kf = {code_pair<kBf16>(w, 0, codes), code_pair<kBf16>(w, 1, codes),
                            code_pair<kBf16>(w, 2, codes), code_pair<kBf16>(w, 3, codes)};
          acc[c] = mfma16<kBf16>(qf[u][s], kf, acc[c]);
        }
    }
    float ks[kTiles], km[kTiles], vs[kTiles], vm[kTiles];
#pragma unroll
    for (int c = 0; c < kTiles; ++c) {
      ks[c] = widen<kBf16>(cur.kw[c] >> 16) * a.scale;
      km[c] = fmaf(-16.0f, ks[c], widen<kBf16>(cur.kw[c] & 0xffffu) * a.scale);
      vs[c] = widen<kBf16>(cur.vw[c] >> 16);
      vm[c] = fmaf(8.0f, vs[c], widen<kBf16>(cur.vw[c] & 0xffffu));
    }
    const bool whole = all_seen<K>(seq, all_lo, all_hi, key0, kStepKeys) && cur.hidden == 0;
    if (!whole) {
      // A key whose V words hold a NaN gives NaN through its score, where only the rows that see it
      // look; the words of keys that no row sees may hold anything.
#pragma unroll
      for (int c = 0; c < kTiles; ++c) {
        const int sub = c * T + 4 * h / R, key = key0 + 16 * sub + n;
        const bool none = unseen<K>(seq, {key_lo, key_hi}, key) || (cur.hidden >> (16 * sub)) & 1;
        const bool nan = has_nan<kBf16>(cur.vw[c]);
        if (nan) km[c] = __uint_as_float(0x7fc00000u);
        if (none || nan) vs[c] = vm[c] = 0.0f;
      }
    }
    bool raise = false;
    float x[kTiles][4];  // scores less m, base 2
#pragma unroll
    for (int c = 0; c < kTiles; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        x[c][i] = fmaf(ks[c], acc[c][i], fmaf(km[c], q_sum[i], -m[i]));
    if (!whole) {
#pragma unroll
      for (int c = 0; c < kTiles; ++c) {
        const int sub = c * T + 4 * h / R, key = key0 + 16 * sub + n;
        const bool hidden = (cur.hidden >> (16 * sub)) & 1;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = (4 * h + i) % R;
          const int2 seen = row < rows ? span<K>(a, seq, row / group) : int2{0, 0};
          if (hidden || unseen<K>(seq, seen, key)) x[c][i] = -kInf;
        }
      }
    }
#pragma unroll
    for (int c = 0; c < kTiles; ++c)
      raise |= fmaxf(fmaxf(x[c][0], x[c][1]), fmaxf(x[c][2], x[c][3])) > kRaise;
    if constexpr (!kBf16) {
#pragma unroll
      for (int c = 0; c < kTiles; ++c) raise |= vs[c] > s_top;
    }
    if (__any(raise)) {
      float ratio = 1.0f;
      if constexpr (!kBf16) {
        float s = vs[0];
#pragma unroll
        for (int c = 1; c < kTiles; ++c) s = fmaxf(s, vs[c]);
        s = across32<true>(across16<true>(over16<true>(s)));
        if (s > s_top) {
          const float up = __uint_as_float((__float_as_uint(s) + 0x7fffffu) & 0x7f800000u);
          ratio = s_top / up;
          s_top = up;
          s_factor = kHeld / up;
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // The scores themselves again: x is infinite while m is.
        float y[kTiles], top = -kInf;
#pragma unroll
        for (int c = 0; c < kTiles; ++c) {
          y[c] = fmaf(ks[c], acc[c][i], km[c] * q_sum[i]);
          if (!whole && x[c][i] == -kInf) y[c] = -kInf;
          top = fmaxf(top, y[c]);
        }
        const float up = fmaxf(m[i], row_lanes<R, true>(top));
        const float base = up == -kInf ? 0.0f : up;
        const float alpha = __builtin_amdgcn_exp2f(m[i] - base);
        m[i] = up;
        l[i] *= alpha;
        mid[i] *= alpha;
        if (n == 0 && 4 * h < R) lds_row[wave][4 * h + i] = alpha * ratio;
#pragma unroll
        for (int c = 0; c < kTiles; ++c) x[c][i] = y[c] - base;
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      const float both = lds_row[wave][n % R];
#pragma unroll
      for (int d = 0; d < kDimTiles; ++d) o[d] *= both;
      ones *= both;
    }
    // Probabilities, and p s in 16 bits (one rounding, of a weight of u - 8) on their way to columns.
#pragma unroll
    for (int c = 0; c < kTiles; ++c) {
      const float f = kBf16 ? vs[c] : vs[c] * s_factor;
      const int key = 16 * (c * T + 4 * h / R) + n;
      float ps[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float p = __builtin_amdgcn_exp2f(x[c][i]);
        l[i] += p;
        mid[i] = fmaf(p, vm[c], mid[i]);
        ps[i] = p * f;
      }
      *reinterpret_cast<uint2*>(&lds_p[wave][key * R + 4 * h % R]) = {
          narrow2<kBf16>(ps[0], ps[1]), narrow2<kBf16>(ps[2], ps[3])};
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    // O^T: dim tile d holds channel D/16 n + d in row n; keys pair up across words.
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int at = (32 * s + 8 * h + (n >> 2)) * R + 4 * (n & 3) % R;
      uint16_t* p = &lds_p[wave][at];
      const v4s p0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)p);
      const v4s p1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(p + 4 * R));
      const uint2 w0 = __builtin_bit_cast(uint2, p0), w1 = __builtin_bit_cast(uint2, p1);
      const uint4 pf = {w0.x, w0.y, w1.x, w1.y};
      ones = mfma16<kBf16>(one8, pf, ones);
      uint32_t lo[4], hi[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t v0 = cur.v[8 * s + 2 * i], v1 = cur.v[8 * s + 2 * i + 1];
        lo[i] = (v0 & 0xffffu) | (v1 << 16);
        hi[i] = (v0 >> 16) | (v1 & 0xffff0000u);
      }
#pragma unroll
      for (int d = 0; d < kDimTiles; ++d) {
        const uint32_t* w = d < 4 ? lo : hi;
        const uint4 vf = {code_pair<kBf16>(w[0], d & 3, codes), code_pair<kBf16>(w[1], d & 3, codes),
                          code_pair<kBf16>(w[2], d & 3, codes), code_pair<kBf16>(w[3], d & 3, codes)};
        o[d] = mfma16<kBf16>(vf, pf, o[d]);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  };
  // Two sets of registers in turn, so that the next step's loads land in their place; with 16 rows
  // there are not enough for both, and the loads are moved.
  for (; step < last; step += stride) {
    attend(tiles[0], tiles[1]);
    if constexpr (R <= 8) {
      step += stride;
      if (step >= last) break;
      attend(tiles[1], tiles[0]);
    } else {
      tiles[0] = tiles[1];
    }
  }

  // Join the four waves: every wave's sums relative to the common maximum.
  const float unit = kBf16 ? 1.0f : s_top * (1.0f / kHeld);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float ls = row_lanes<R, false>(l[i]), ms = row_lanes<R, false>(mid[i]);
    if (n == 0 && 4 * h < R) {
      lds_ml[wave][4 * h + i] = {m[i], ls};
      lds_row[wave][4 * h + i] = ms;
    }
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  const float ms = lds_row[wave][n % R];
  if (n < R) {
    // Row i of dim tile d: channel (D/16) (4h + i) + d.
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int d = 0; d < kDimTiles; d += 4) {
        float4 f;
        f.x = fmaf(unit, fmaf(-24.0f, ones[i], o[d][i]), ms);
        f.y = fmaf(unit, fmaf(-24.0f, ones[i], o[d + 1][i]), ms);
        f.z = fmaf(unit, fmaf(-24.0f, ones[i], o[d + 2][i]), ms);
        f.w = fmaf(unit, fmaf(-24.0f, ones[i], o[d + 3][i]), ms);
        *reinterpret_cast<float4*>(&lds_o[wave][n][kDimTiles * (4 * h + i) + d]) = f;
      }
  }
  if constexpr (kShare == kWaves) {
    __syncthreads();
  } else {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
  constexpr int kJoiners = kShare * 64, kPer = R * D / kJoiners;  // channels a thread; kJoiners / R threads a row
  const int row = thread / (kJoiners / R), ch = (thread % (kJoiners / R)) * kPer, wave0 = wave - mine;
  if (row < rows) {
    float2 ml[kShare];
    float top = -kInf;
#pragma unroll
    for (int w = 0; w < kShare; ++w) {
      ml[w] = lds_ml[wave0 + w][row];
      top = fmaxf(top, ml[w].x);
    }
    const float base = top == -kInf ? 0.0f : top;
    float total = 0.0f, sum[kPer];
#pragma unroll
    for (int d = 0; d < kPer; ++d) sum[d] = 0.0f;
#pragma unroll
    for (int w = 0; w < kShare; ++w) {
      const float f = __builtin_amdgcn_exp2f(ml[w].x - base);
      total = fmaf(f, ml[w].y, total);
#pragma unroll
      for (int d = 0; d < kPer; ++d) sum[d] = fmaf(f, lds_o[wave0 + w][row][ch + d], sum[d]);
    }
    total = or_nan(total, sum[0]);
    const int token = row / group, g = row - token * group;
    const size_t q_row = (size_t)(seq.start + token);
    const uint32_t q_head = head * group + g;
    if (kPart<K> || a.parts > 1) {
      const size_t place = few_place<K>(a, seq, part, b, row, head);
#pragma unroll
      for (int d = 0; d < kPer; ++d) a.part_o[place * D + ch + d] = sum[d];
      if (ch == 0) a.part_ml[place] = {top, total};
    } else {
      const bool none = total == 0.0f;  // a NaN among the scores or values leaves total NaN
      const Mean by = make_mean<kBf16>(total);
      uint16_t* out = static_cast<uint16_t*>(a.out) + q_row * a.out_stride + q_head * D + ch;
#pragma unroll
      for (int d = 0; d < kPer; ++d) out[d] = (uint16_t)narrow<kBf16>(mean<kBf16>(sum[d], by));
      if (a.lse && ch == 0)
        a.lse[q_row * heads + q_head] = none ? -kInf : (top + __log2f(total)) * kLn2;
    }
  }
}

template <int D, bool kBf16, int R, bool kOnce, Keys K>
__global__ __launch_bounds__(kThreads, 2) void k_attention_kv4_few(Args a) {
  __shared__ FewLds<D, R> lds;
  attend_few<D, kBf16, R, kOnce, K>(a, lds, blockIdx.x, blockIdx.y, blockIdx.z);
}

// Many rows: eight waves of 32 rows share tiles of 64 keys in LDS, unpacked once for all of them:
// K as 16 + u, V as m + s u rounded to the element type (the one rounding beside p's). S^T = K Q^T and
// O^T = V^T P^T on 32 x 32 x 16. LDS row m of 32 K rows holds key swap23(m), so the score registers
// of a lane (one row of q, half = lane / 32) are keys 8 half + 0..7 and 16 + 8 half + 0..7: the B
// operands of the PV product's two steps, as they are. V stays token-major and its operand comes
// through the transposed LDS read. 8,192 causal tokens of 32 heads on 8 (128 channels): 599 to 605 us, 0.91 to
// 0.92 PFLOP/s of the 1.14 to 1.32 that a library product of 8,192^3 reaches; the matrix pipe is busy for 45 % of the
// time and the vector pipe for 50 %.
constexpr int kRowsThreads = 512;
constexpr int kTileRows = 256, kTileKeys = 64;
constexpr float kPTop = 32768.0f;  // a lane's probabilities of 32 keys sum to no more, or m is raised
constexpr float kPLog = 7.0f;      // the largest score gives p = 2^7: f16 stays normal to 2^-21 of it

__device__ __forceinline__ uint32_t swap23(uint32_t m) {
  return (m & ~12u) | ((m & 4) << 1) | ((m & 8) >> 1);
}

template <bool kBf16>
__device__ __forceinline__ v16f mfma32(uint4 a, uint4 b, v16f c) {
  if constexpr (kBf16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf, a),
                                                   __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, a),
                                                __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}

// Lane kLane of each 16 lanes, to all of them.
template <int kLane>
__device__ __forceinline__ float spread(float v) {
  return __int_as_float(
      __builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x150 + kLane, 0xF, 0xF, true));
}

// Row pitches in LDS. The rows that a K read of eight lanes takes start 16 bytes apart modulo 256, the
// four keys of a transposed V read 64 apart, so that no two fall on the same banks.
template <int D> constexpr int kKPitch = 2 * D + 16;
template <int D> constexpr int kVPitch = 2 * D + 64;

template <int D>
struct RowsLds {
  uint8_t k[3][kTileKeys * kKPitch<D>];
  uint8_t v[3][kTileKeys * kVPitch<D>];
  float ks[3][kTileKeys], km[3][kTileKeys];  // times the scale: s, and m - 16 s
  float vn[3][kTileKeys];                    // NaN for a key whose V words hold one, else 0
  uint8_t dead[3][kTileKeys];                // the key's page is none of the cache's
};

// Waves 0..3 bring a tile's keys to LDS, waves 4..7 its values: a thread one key's (tid / 4 % 64)
// channels D/4 (tid % 4) and on. Their D/32 words go to 16-byte chunks 4 i + tid % 4, so that the
// lanes of a store lie side by side: chunk c of an LDS row holds channels 8 chunk_word(c) and on, an
// order that Q is read in and the results are written in.
template <int D>
struct Staged {
  uint32_t codes[D / 32];
  uint32_t word;
  int page;
};
template <int D>
__device__ __forceinline__ constexpr int chunk_word(int c) {
  return (D / 32) * (c & 3) + (c >> 2);
}

template <int D>
__device__ __forceinline__ void fetch(const Args& a, uint32_t head, int key, int page, Staged<D>& s) {
  const uint32_t page_tokens = 1u << a.page_shift, in_page = (uint32_t)key & (page_tokens - 1);
  const uint32_t block = page_tokens * (D + 8), v = threadIdx.x >> 8;
  const uint8_t* at = a.cache + (uint64_t)head * block +
                      (uint64_t)(uint32_t)max(page, 0) * (block * a.kv_heads);
  const uint8_t* codes = at + (v * page_tokens * (D / 2) + in_page * (D / 2) + (threadIdx.x & 3) * (D / 8));
  const uint8_t* word = at + (page_tokens * D + v * page_tokens * 4 + in_page * 4);
  if constexpr (D == 128) {
    const uint4 x = *reinterpret_cast<const uint4*>(codes);
    s.codes[0] = x.x, s.codes[1] = x.y, s.codes[2] = x.z, s.codes[3] = x.w;
  } else {
    const uint2 x = *reinterpret_cast<const uint2*>(codes);
    s.codes[0] = x.x, s.codes[1] = x.y;
  }
  s.word = *reinterpret_cast<const uint32_t*>(word);
  s.page = page;
}

// A key's s and m as its values are made of them: bf16 in f32 (m16: m - 16 s), f16 twice in a pair each.
template <bool kBf16>
struct Factors {
  float s, m16;
  uint32_t s2, m2;
};
template <bool kBf16>
__device__ __forceinline__ Factors<kBf16> factors(uint32_t word) {
  const float s = widen<kBf16>(word >> 16);
  return {s, fmaf(-16.0f, s, widen<kBf16>(word & 0xffffu)), (word >> 16) | (word & 0xffff0000u),
          (word & 0xffffu) | (word << 16)};
}

// A pair of values m + s u, u as 16 + u in `code`, rounded once to the element type: in f16 u is exact, and one packed
// FMA is the value. (Never past the row's own extremes, as m + 15 s is not; a rounded midpoint m + 8 s plus (u - 8) s
// was infinite for some rows that end near 65504.)
template <bool kBf16>
__device__ __forceinline__ uint32_t value_pair(uint32_t code, const Factors<kBf16>& f) {
  if constexpr (kBf16)
    return narrow2<true>(fmaf(__uint_as_float(code << 16), f.s, f.m16),
                         fmaf(__uint_as_float(code & 0xffff0000u), f.s, f.m16));
  const v2h u = __builtin_bit_cast(v2h, code) - v2h{(_Float16)16.0f, (_Float16)16.0f};
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(u, __builtin_bit_cast(v2h, f.s2),
                                                                __builtin_bit_cast(v2h, f.m2)));
}

template <int D, bool kBf16, Keys K>
__device__ __forceinline__ void unpack(const Args& a, RowsLds<D>& lds, int buf, int key0, const Sequence& seq,
                                       int key_lo, int key_hi, const Codes& codes, const Staged<D>& s) {
  const uint32_t at = (threadIdx.x >> 2) & 63, part = threadIdx.x & 3;
  if (__builtin_amdgcn_readfirstlane(threadIdx.x >> 8) == 0) {
    const uint32_t m = (at & 32) + swap23(at & 31);
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
      *reinterpret_cast<uint4*>(&lds.k[buf][m * kKPitch<D> + 16 * (4 * i + part)]) = {
          code_pair<kBf16>(s.codes[i], 0, codes), code_pair<kBf16>(s.codes[i], 1, codes),
          code_pair<kBf16>(s.codes[i], 2, codes), code_pair<kBf16>(s.codes[i], 3, codes)};
    if (part == 0) {
      const float ks = widen<kBf16>(s.word >> 16) * a.scale;
      lds.ks[buf][at] = ks;
      lds.km[buf][at] = fmaf(-16.0f, ks, widen<kBf16>(s.word & 0xffffu) * a.scale);
      lds.dead[buf][at] = s.page < 0;
    }
    return;
  }
  // A key whose V words hold a NaN gives NaN through its score, where only the rows that see it
  // look; its V rows, and those of keys that no row sees, are zeros.
  const int key = key0 + (int)at;
  const bool nan = has_nan<kBf16>(s.word);
  const bool keep = s.page >= 0 && !unseen<K>(seq, {key_lo, key_hi}, key) && !nan;
  const Factors<kBf16> f = factors<kBf16>(keep ? s.word : 0u);
#pragma unroll
  for (int i = 0; i < D / 32; ++i) {
    uint4 x;
    x.x = value_pair<kBf16>(code_pair<kBf16>(s.codes[i], 0, codes), f);
    x.y = value_pair<kBf16>(code_pair<kBf16>(s.codes[i], 1, codes), f);
    x.z = value_pair<kBf16>(code_pair<kBf16>(s.codes[i], 2, codes), f);
    x.w = value_pair<kBf16>(code_pair<kBf16>(s.codes[i], 3, codes), f);
    *reinterpret_cast<uint4*>(&lds.v[buf][at * kVPitch<D> + 16 * (4 * i + part)]) = x;
  }
  if (part == 0) lds.vn[buf][at] = nan ? __uint_as_float(0x7fc00000u) : 0.0f;
}

// acc times the keys' factors: lane r of 16 holds register r's.
template <int R = 0>
__device__ __forceinline__ void scale_scores(float ks, v16f& acc) {
  if constexpr (R < 16) {
    acc[R] *= spread<R>(ks);
    scale_scores<R + 1>(ks, acc);
  }
}

// A wave's sums over the keys so far: O^T, and per lane (of its row) l, relative to m; m is -inf until
// the row has met a key, and exponents are relative to 0 until then.
template <int D>
struct RowSums {
  v16f o[D / 32];
  float m, l;
  __device__ __forceinline__ float base() const { return m == -kInf ? 0.0f : m; }
};

// What a wave reads of a 32-key block (block blk of buffer buf) before its products: the first half
// of the K operands. The reads run a phase ahead of their use, here and below: two waves a SIMD do not
// hide an LDS read's latency.
template <int D>
struct KeyOps {
  uint4 k[D / 32];
};
template <int D, int kFrom>
__device__ __forceinline__ KeyOps<D> read_keys(const RowsLds<D>& lds, int buf, int blk, int lane) {
  const int n = lane & 31, half = lane >> 5;
  KeyOps<D> x;
#pragma unroll
  for (int s = 0; s < D / 32; ++s)
    x.k[s] = *reinterpret_cast<const uint4*>(
        &lds.k[buf][(32 * blk + n) * kKPitch<D> + 16 * (2 * (kFrom + s) + half)]);
  return x;
}

// V^T operands of step s of a block, channels of chunks 4 d .. 4 d + 3, keys 8 half + 0..7: lane j of 16
// points at key j / 4, channels 4 (j % 4) and on, and receives channel j of four keys.
template <int D>
struct ValueOps {
  uint4 v[D / 32];
};
template <int D>
__device__ __forceinline__ ValueOps<D> read_values(const RowsLds<D>& lds, int buf, int blk, int s,
                                                   int lane) {
  const int j = lane & 15, quad = lane >> 4;
  const int key = 32 * blk + 16 * s + 8 * (quad >> 1) + (j >> 2);
  ValueOps<D> x;
#pragma unroll
  for (int d = 0; d < D / 32; ++d) {
    const uint32_t chunk = 4 * d + 2 * (quad & 1) + ((j & 3) >> 1);
    const uint8_t* v = &lds.v[buf][key * kVPitch<D> + 16 * chunk + 8 * (j & 1)];
    const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)v);
    const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(v + 4 * kVPitch<D>));
    const uint2 l2 = __builtin_bit_cast(uint2, lo), h2 = __builtin_bit_cast(uint2, hi);
    x.v[d] = {l2.x, l2.y, h2.x, h2.y};
  }
  return x;
}

// Which keys of a 32-key block a lane's row sees: [lo, hi), and before lo those below front, counted from its first key
// (8 half).
struct Seen {
  int lo, hi, front;
  bool pages;  // some page of the workgroup's keys is none of the cache's: `dead` says which keys
};

// One 32-key block (blk of buf) of a wave, from its products x = q (16 + u): probabilities and the sum
// over values. s_k x + (m_k - 16 s_k) sum(q) - m is a multiplication on the vector unit and two products
// added to it in f32 on the matrix unit, (km, 1) (sum(q), -m). Where a row meets its first keys, or a
// lane's probabilities pass kPTop, m is raised. The products of the next block run among the vector
// instructions: its first operands are in `keys`, the others' block is next_blk of next_buf; they are
// returned.
template <int D, bool kBf16, Keys K>
__device__ __forceinline__ v16f attend_block(const RowsLds<D>& lds, int buf, int blk, int next_buf,
                                             int next_blk, v16f x, const uint4 (&qf)[D / 16],
                                             const KeyOps<D>& keys, bool whole, const Seen& seen,
                                             float q_sum, int lane, RowSums<D>& r) {
  const int n = lane & 31, half = lane >> 5;
  const float ks = lds.ks[buf][32 * blk + (lane & 7) + 8 * half + 2 * (lane & 8)];
  const float kv = lds.km[buf][32 * blk + swap23(n)] + lds.vn[buf][32 * blk + swap23(n)];
  const KeyOps<D> rest = read_keys<D, D / 32>(lds, next_buf, next_blk, lane);
  const float km = half ? -1.0f : kv;
  v16f next = v16f{};
#pragma unroll
  for (int s = 0; s < D / 32; ++s) next = mfma32<kBf16>(keys.k[s], qf[s], next);
  scale_scores(ks, x);
  v16f y = __builtin_amdgcn_mfma_f32_32x32x2f32(km, half ? r.base() : q_sum, x, 0, 0, 0);
  if (!whole) {
    asm volatile("");  // a branch, not 16 selects in every block
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int k = (i & 7) + 2 * (i & 8);
      if ((k < seen.lo && (kPlain<K> || k >= seen.front)) || k >= seen.hi) y[i] = -kInf;
    }
    if (seen.pages) {
      asm volatile("");
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (lds.dead[buf][32 * blk + 8 * half + (i & 7) + 2 * (i & 8)]) y[i] = -kInf;
    }
  }
  // The softmax goes before the SIMD's other wave's products, which wait for nothing: 8,224 rows behind a prefix of
  // 31,104 keys 1,194 us with this priority and 1,236 without.
  __builtin_amdgcn_s_setprio(1);
  const ValueOps<D> v0 = read_values<D>(lds, buf, blk, 0, lane);
  float p[16], ts = 0.0f;
#pragma unroll
  for (int s = 0; s < D / 32; ++s) next = mfma32<kBf16>(rest.k[s], qf[D / 32 + s], next);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    p[i] = __builtin_amdgcn_exp2f(y[i]);
    ts += p[i];
  }
  // Matrix and vector instructions in turn, so that the matrix unit works under the vector ones
  // whatever the SIMD's other wave is at.
  __builtin_amdgcn_sched_group_barrier(0x100, D / 16, 0);
#pragma unroll
  for (int i = 0; i < D / 32; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    __builtin_amdgcn_sched_group_barrier(0x002, 32 / (D / 32), 0);
  }
  if (__builtin_expect(__any(!(ts <= kPTop) || r.m == -kInf), 0)) {
    const float was = r.base();
    float top = y[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) top = fmaxf(top, y[i]);
    top = across32<true>(top) + (was - kPLog);
    const float up = fmaxf(r.m, top);
    const float alpha = __builtin_amdgcn_exp2f(r.m - (up == -kInf ? 0.0f : up));
    r.m = up;
    const float by = was - r.base();
    r.l *= alpha;
#pragma unroll
    for (int d = 0; d < D / 32; ++d) r.o[d] *= alpha;
    ts = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      p[i] = __builtin_amdgcn_exp2f(y[i] + by);
      ts += p[i];
    }
  }
  const ValueOps<D> v1 = read_values<D>(lds, buf, blk, 1, lane);
  r.l += ts;
  uint4 pf[2];
#pragma unroll
  for (int s = 0; s < 2; ++s)
    pf[s] = {narrow2<kBf16>(p[8 * s], p[8 * s + 1]), narrow2<kBf16>(p[8 * s + 2], p[8 * s + 3]),
             narrow2<kBf16>(p[8 * s + 4], p[8 * s + 5]), narrow2<kBf16>(p[8 * s + 6], p[8 * s + 7])};
  __builtin_amdgcn_s_setprio(0);
#pragma unroll
  for (int d = 0; d < D / 32; ++d) r.o[d] = mfma32<kBf16>(v0.v[d], pf[0], r.o[d]);
#pragma unroll
  for (int d = 0; d < D / 32; ++d) r.o[d] = mfma32<kBf16>(v1.v[d], pf[1], r.o[d]);
  return next;
}

// Steps st (tiles of keys) of rows row0 .. row0 + 255 of sequence b for one cache head. Results go to out
// and lse, or (slot >= 0) as sums relative to m to that slot of the workspace.
template <int D, bool kBf16, Keys K>
__device__ __forceinline__ void attend_rows(const Args& a, RowsLds<D>& lds, const Sequence& seq,
                                            uint32_t b, uint32_t head, int row0, Steps st, int slot) {
  constexpr int kSteps = D / 16, kBlocks = D / 32;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 31, half = lane >> 5;
  const int group = (int)a.group, rows = seq.rows * group;
  const int key_lo = span<K>(a, seq, row0 / group).x;
  const int key_hi = span<K>(a, seq, (min(row0 + kTileRows, rows) - 1) / group).y;
  const auto way = walk<K, kTileKeys>(seq, key_lo, key_hi);
  const uint32_t heads = a.kv_heads * a.group;

  // The wave's rows, the keys that some and that all of them see, and the tiles it takes.
  const int wave_row0 = row0 + 32 * wave, row = wave_row0 + n;
  const int2 wave_first = span<K>(a, seq, min(wave_row0, rows - 1) / group);
  const int2 wave_last = span<K>(a, seq, min(wave_row0 + 31, rows - 1) / group);
  const int token = row / group, g = row - token * group;
  const int2 seen = row < rows ? span<K>(a, seq, token) : int2{0, 0};
  const bool active = wave_row0 < rows;
  const int from = max(st.first, wave_first.x / kTileKeys);
  const int to = active ? min(st.last, (wave_last.y + kTileKeys - 1) / kTileKeys) : from;

  // Q^T operands: chunk 2 s + half's channels, in the order {0,4,1,5,2,6,3,7} of the codes' pairs.
  uint4 qf[kSteps];
  float sum = 0.0f;
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    uint4 x = {0, 0, 0, 0};
    if (row < rows)
      x = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.q) +
                                          (size_t)(seq.start + token) * a.q_stride +
                                          (head * a.group + g) * D + 8 * chunk_word<D>(2 * s + half));
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) sum += widen<kBf16>(w[i] & 0xffffu) + widen<kBf16>(w[i] >> 16);
    qf[s] = {(x.x & 0xffffu) | (x.z << 16), (x.x >> 16) | (x.z & 0xffff0000u),
             (x.y & 0xffffu) | (x.w << 16), (x.y >> 16) | (x.w & 0xffff0000u)};
  }
  const float q_sum = across32<false>(sum);

  RowSums<D> sums;
#pragma unroll
  for (int d = 0; d < kBlocks; ++d) sums.o[d] = v16f{};
  sums.m = row < rows ? -kInf : 0.0f;
  sums.l = 0.0f;
  const int32_t* table = a.table + (size_t)b * a.table_stride;
  const int at = (int)(threadIdx.x >> 2) & 63;
  const Codes codes = make_codes<kBf16>();

  Staged<D> staged;
  int page = -1;
  bool hidden = false;
  if (st.first < st.last) {
    const int key = way.key(st.first) + at;
    fetch<D>(a, head, key, page_of<K>(a, table, seq, key), staged);
    page = page_of<K>(a, table, seq, way.key(st.first + 1) + at);
    if constexpr (kPlain<K>) {
      for (int k = max(st.first * kTileKeys, key_lo & ~15) + 16 * (int)threadIdx.x;
           k < min(st.last * kTileKeys, key_hi); k += 16 * kRowsThreads)
        hidden |= page_of<K>(a, table, seq, k) < 0;
    } else {
      for (int i = (int)threadIdx.x; i < 4 * (st.last - st.first); i += kRowsThreads) {
        const int k = way.key(st.first + i / 4) + 16 * (i % 4);
        if (k < key_hi && (k < seq.front || k + 16 > key_lo)) hidden |= page_of<K>(a, table, seq, k) < 0;
      }
    }
    unpack<D, kBf16, K>(a, lds, 0, way.key(st.first), seq, key_lo, key_hi, codes, staged);
    fetch<D>(a, head, way.key(st.first + 1) + at, page, staged);
    page = page_of<K>(a, table, seq, way.key(st.first + 2) + at);
  }
  hidden = __syncthreads_or(hidden);  // some seen key's page is none of the cache's
  // Three buffers and one barrier a tile: while a wave is at tile t, another may still read t - 1's
  // values, and the tile written is t + 1. Tiles past the last are fetched and unpacked like the
  // others (their keys are seen by no row, and page -1 reads page 0), so that the loop has no tail.
  v16f x = v16f{};
  KeyOps<D> keys;
  int buf = 0;
  bool under_way = false;  // x holds this tile's first products
  for (int step = st.first; step < st.last; ++step) {
    const int next = buf == 2 ? 0 : buf + 1, key0 = way.key(step), key1 = way.key(step + 1);
    const bool takes_tile = kPlain<K> ? step >= from && step < to
                                      : active && key0 < wave_last.y &&
                                            (key0 < seq.front || key0 + kTileKeys > wave_first.x);
    if (takes_tile) {
      const bool whole = all_seen<K>(seq, wave_last.x, wave_first.y, key0, kTileKeys) && !hidden;
      if (kPlain<K> ? step == from : !under_way) {
        const KeyOps<D> k0 = read_keys<D, 0>(lds, buf, 0, lane), k1 = read_keys<D, D / 32>(lds, buf, 0, lane);
        if constexpr (!kPlain<K>) x = v16f{};  // between the front's tiles and its own the wave let some pass
#pragma unroll
        for (int s = 0; s < kSteps / 2; ++s) x = mfma32<kBf16>(k0.k[s], qf[s], x);
#pragma unroll
        for (int s = 0; s < kSteps / 2; ++s) x = mfma32<kBf16>(k1.k[s], qf[kSteps / 2 + s], x);
      }
      keys = read_keys<D, 0>(lds, buf, 1, lane);
      const Seen see = {seen.x - key0 - 8 * half, seen.y - key0 - 8 * half,
                        kPlain<K> ? 0 : seq.front - key0 - 8 * half, hidden};
      x = attend_block<D, kBf16, K>(lds, buf, 0, buf, 1, x, qf, keys, whole, see, q_sum, lane, sums);
      unpack<D, kBf16, K>(a, lds, next, key1, seq, key_lo, key_hi, codes, staged);
      __syncthreads();
      keys = read_keys<D, 0>(lds, next, 0, lane);
      fetch<D>(a, head, way.key(step + 2) + at, page, staged);
      page = page_of<K>(a, table, seq, way.key(step + 3) + at);
      x = attend_block<D, kBf16, K>(lds, buf, 1, next, 0, x, qf, keys, whole,
                                    {see.lo - 32, see.hi - 32, see.front - 32, hidden}, q_sum, lane, sums);
    } else {
      unpack<D, kBf16, K>(a, lds, next, key1, seq, key_lo, key_hi, codes, staged);
      fetch<D>(a, head, way.key(step + 2) + at, page, staged);
      page = page_of<K>(a, table, seq, way.key(step + 3) + at);
      __syncthreads();
    }
    under_way = takes_tile;
    buf = next;
  }

  __syncthreads();  // the tiles are done with: LDS is free for the results
  // Register 4 i + b of block d holds channel 8 w + 2 half + {0, 4, 1, 5}[b] of the lane's row, w the
  // word of chunk 4 d + i.
  const v16f(&o)[kBlocks] = sums.o;
  const float m = sums.m, total = across32<false>(sums.l);
  const bool none = total == 0.0f;
  const size_t q_row = (size_t)(seq.start + token);
  const uint32_t q_head = head * a.group + g;
  if (slot >= 0) {
    if (row < rows) {
      const size_t place = kPart<K> ? few_place<K>(a, seq, (uint32_t)slot, b, (uint32_t)row, head)
                                    : (size_t)slot * kTileRows + (row - row0);
#pragma unroll
      for (int d = 0; d < kBlocks; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float* to = a.part_o + place * D + 8 * chunk_word<D>(4 * d + i) + 2 * half;
          *reinterpret_cast<float2*>(to) = {o[d][4 * i], o[d][4 * i + 2]};
          *reinterpret_cast<float2*>(to + 4) = {o[d][4 * i + 1], o[d][4 * i + 3]};
        }
      if (half == 0) a.part_ml[place] = {m, total};
    }
    return;
  }
  if (!active) return;
  const Mean by = make_mean<kBf16>(total);
  // Through LDS (each wave its own 32 rows) so that whole rows leave together.
  uint8_t* rows_lds = reinterpret_cast<uint8_t*>(&lds) + wave * 32 * 2 * D;
  static_assert(sizeof(lds.k) + sizeof(lds.v) >= 8 * 32 * 2 * D && offsetof(RowsLds<D>, k) == 0 &&
                    offsetof(RowsLds<D>, v) == sizeof(lds.k),
                "the tiles hold the rows");
#pragma unroll
  for (int d = 0; d < kBlocks; ++d)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint8_t* to = rows_lds + n * (2 * D) + 16 * (chunk_word<D>(4 * d + i) ^ (n & (D / 8 - 1))) + 4 * half;
      *reinterpret_cast<uint32_t*>(to) =
          narrow2<kBf16>(mean<kBf16>(o[d][4 * i], by), mean<kBf16>(o[d][4 * i + 2], by));
      *reinterpret_cast<uint32_t*>(to + 8) =
          narrow2<kBf16>(mean<kBf16>(o[d][4 * i + 1], by), mean<kBf16>(o[d][4 * i + 3], by));
    }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  constexpr int kLanes = D / 8;  // lanes of 16 bytes a row
#pragma unroll
  for (int i = 0; i < 32 * kLanes / 64; ++i) {
    const int r = i * (64 / kLanes) + lane / kLanes, chunk = lane % kLanes;
    const uint4 x = *reinterpret_cast<const uint4*>(rows_lds + r * (2 * D) +
                                                    16 * (chunk ^ (r & (D / 8 - 1))));
    const int to = wave_row0 + r, t = to / group;
    if (to < rows)
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) +
                                (size_t)(seq.start + t) * a.out_stride +
                                (head * a.group + (to - t * group)) * D + 8 * chunk) = x;
  }
  if (a.lse && half == 0 && row < rows)
    a.lse[q_row * heads + q_head] = none ? -kInf : (m + __log2f(total)) * kLn2;
}

// 17 rows and more, in tiles of 32: as k_attention_kv4_few, with score tiles S^T = K Q^T of 32 keys and 32
// rows (32 x 32 x 16), so that a code unpacked serves 32 rows, and a lane holds 16 keys of one row. K row
// m of a tile is key swap23(m), so that the score registers (half = lane / 32) are keys 8 half + 0..7 and
// 16 + 8 half + 0..7, the B operands of O^T = V^T P^T as they are: no probability passes through LDS, and
// a row's sums and factors stay in its lanes. The keys' factors reach their registers by a broadcast within
// 16 lanes, lane r holding register r's. Some 325 vector instructions and 19 MFMAs a wave's step of 32
// keys, where two 16-row tiles of k_attention_kv4_few take 540: 0.92 us a step with one wave a SIMD. 128
// groups of 25 rows over a window of 4,096 keys 28 us (36 in two tiles of 16 rows); 512 groups of 64 rows
// over 8,192 keys 251 us (373).
constexpr int kMidRows = 32, kMidKeys = 32;
constexpr float kMidTop = 128.0f;  // a lane's 16 probabilities sum to no more, or m is raised

template <int D>
struct MidStep {
  uint32_t k[D / 16];  // key swap23(lane % 32): channels D/2 half and on
  uint32_t v[16];      // keys 16 (e / 8) + 8 half + e % 8: channels D/32 (lane % 32) and on
  uint32_t kw, ks, vs;  // words: the K word of that key, and K's and V's of register lane % 16's key
  uint64_t hidden;     // a bit per lane: the key's page is none of the cache's
};

// `ids`: the page of key `key` + swap23(lane % 32).
template <int D, bool kOnce>
__device__ __forceinline__ void load_mid(const Args& a, int ids, uint32_t head, int key, int lane,
                                         MidStep<D>& s) {
  const uint32_t n = lane & 31, half = lane >> 5;
  const uint32_t page_tokens = 1u << a.page_shift, mask = page_tokens - 1;
  const uint32_t block = page_tokens * (D + 8), in_page = ((uint32_t)key + swap23(n)) & mask;
  // Keys of no page are masked; page 0 is there to read.
  const uint8_t* page = a.cache + (uint64_t)head * block +
                        (uint64_t)(uint32_t)max(ids, 0) * (block * a.kv_heads);
  s.hidden = __ballot(ids < 0);
  const uint8_t *lo = lane_pointer(page, 0), *hi = lane_pointer(page, 16);  // of each 16 keys
  const uint8_t* mine = page + (in_page * (D / 2) + half * (D / 4));
#pragma unroll
  for (int i = 0; i < D / 64; ++i) {
    typedef uint32_t Words __attribute__((ext_vector_type(4)));
    const Words x = load_codes<kOnce, Words>(mine + 16 * i);
    s.k[4 * i] = x.x, s.k[4 * i + 1] = x.y, s.k[4 * i + 2] = x.z, s.k[4 * i + 3] = x.w;
  }
  s.kw = *reinterpret_cast<const uint32_t*>(page + (page_tokens * D + 4 * in_page));
  const uint32_t at[2] = {(uint32_t)key & mask, ((uint32_t)key + 16) & mask};
  const uint8_t* words = lane & 8 ? hi + 4 * at[1] : lo + 4 * at[0];
  words += page_tokens * D + 4 * ((lane & 7) + 8 * half);
  s.ks = *reinterpret_cast<const uint32_t*>(words);
  s.vs = *reinterpret_cast<const uint32_t*>(words + page_tokens * 4);
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const uint8_t* v = (t ? hi : lo) + (page_tokens + at[t]) * (D / 2) + (8 * half * (D / 2) + n * (D / 64));
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if constexpr (D == 128)
        s.v[8 * t + e] = load_codes<kOnce, uint16_t>(v + e * 64);
      else
        s.v[8 * t + e] = v[e * 32];
    }
  }
}

// p times their keys' factors f.
template <int R = 0>
__device__ __forceinline__ void weigh(float f, const float (&p)[16], float (&ps)[16]) {
  if constexpr (R < 16) {
    ps[R] = p[R] * spread<R>(f);
    weigh<R + 1>(f, p, ps);
  }
}
// sum plus the products of p with their keys' `add`. One block of instructions: the compiler would move each
// broadcast to a register first; the wait is what a broadcast's source and p, fresh from exp, ask for.
__device__ __forceinline__ float add_weighed(float sum, float add, const float (&p)[16]) {
  asm("s_nop 1\n"
      "v_fmac_f32_dpp %0, %1, %2 row_newbcast:0 row_mask:0xf bank_mask:0xf\n"
      "v_fmac_f32_dpp %0, %1, %3 row_newbcast:1 row_mask:0xf bank_mask:0xf\n"
      "v_fmac_f32_dpp %0, %1, %4 row_newbcast:2 row_mask:0xf bank_mask:0xf\n"
      "v_fmac_f32_dpp %0, %1, %5 row_newbcast:3 row_mask:0xf bank_mask:0xf\n"
      "v_fmac_f32_dpp %0, %1, %6 row_newbcast:4 row_mask:0xf bank_mask:0xf\n"
      "v_fmac_f32_dpp %0, %1, %7 row_newbcast:5 row_mask:0xf bank_mask:0xf\n"
      "v_fmac_f32_dpp %0, %1, %8 row_newbcast:6 row_mask:0xf bank_mask:0xf\n"
      "v_fmac_f32_dpp %0, %1, %9 row_newbcast:7 row_mask:0xf bank_mask:0xf\n"
      "v_fmac_f32_dpp %0, %1, %10 row_newbcast:8 row_mask:0xf bank_mask:0xf\n"
      "v_fmac_f32_dpp %0, %1, %11 row_newbcast:9 row_mask:0xf bank_mask:0xf\n"
      "v_fmac_f32_dpp %0, %1, %12 row_newbcast:10 row_mask:0xf bank_mask:0xf\n"
      "v_fmac_f32_dpp %0, %1, %13 row_newbcast:11 row_mask:0xf bank_mask:0xf\n"
      "v_fmac_f32_dpp %0, %1, %14 row_newbcast:12 row_mask:0xf bank_mask:0xf\n"
      "v_fmac_f32_dpp %0, %1, %15 row_newbcast:13 row_mask:0xf bank_mask:0xf\n"
      "v_fmac_f32_dpp %0, %1, %16 row_newbcast:14 row_mask:0xf bank_mask:0xf\n"
      "v_fmac_f32_dpp %0, %1, %17 row_newbcast:15 row_mask:0xf bank_mask:0xf\n"
      : "+&v"(sum)
      : "v"(add), "v"(p[0]), "v"(p[1]), "v"(p[2]), "v"(p[3]), "v"(p[4]), "v"(p[5]), "v"(p[6]), "v"(p[7]),
        "v"(p[8]), "v"(p[9]), "v"(p[10]), "v"(p[11]), "v"(p[12]), "v"(p[13]), "v"(p[14]), "v"(p[15]));
  return sum;
}

template <int D>
struct MidLds {
  __attribute__((aligned(16))) float o[kWaves][kMidRows][D + 4];
  float2 ml[kWaves][kMidRows];
};

template <int D, bool kBf16, bool kOnce, Keys K>
__device__ __forceinline__ void attend_mid(const Args& a, MidLds<D>& lds, uint32_t part, uint32_t y, uint32_t b) {
  constexpr int kSteps = D / 16, kBlocks = D / 32;
  auto &lds_o = lds.o;
  auto &lds_ml = lds.ml;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 31, half = lane >> 5;
  const uint32_t at_y = y / a.kv_heads, head = y - at_y * a.kv_heads;
  // A sequence's tiles begin at a place of its own: with the first tiles, all that short sequences have, a fixed
  // number of workgroups apart, one shader engine in four would get them (129 sequences, one of them of 30
  // tokens in four tiles, 102 us for 42).
  uint32_t tile = at_y + __umulhi(b * 0x9E3779B1u, a.row_tiles);
  tile -= tile >= a.row_tiles ? a.row_tiles : 0;
  const int32_t* table = a.table + (size_t)b * a.table_stride;
  const Sequence seq = sequence<K>(a, b);
  const int group = (int)a.group, rows = seq.rows * group, stride = (int)a.parts * kWaves;
  const int row0 = (int)tile * kMidRows, mine = (int)swap23(n);
  // Before the loads: most workgroups of a ragged call end here. (Over a prefix most have rows, and whether they do is
  // a load away: 64 tokens behind 8,192 keys 35.6 us with the loads first, 35.8 so.)
  if (K != kFrontPart && tile > 0 && row0 >= rows) return;
  int step = (int)part * kWaves + wave;
  Walk<K, kMidKeys> way{};
  if constexpr (kPlain<K>) {
    if (a.window) step += span<K>(a, seq, row0 / group).x / kMidKeys;
  } else {
    way = walk<K, kMidKeys>(seq, span<K>(a, seq, row0 / group).x,
                            span<K>(a, seq, (min(row0 + kMidRows, rows) - 1) / group).y);
  }
  int ids = page_of<K>(a, table, seq, way.key(step) + mine);
  MidStep<D> tiles[2];
  load_mid<D, kOnce>(a, ids, head, way.key(step), lane, tiles[0]);
  ids = page_of<K>(a, table, seq, way.key(step + stride) + mine);
  if (row0 >= rows || !takes(a, rows)) return;
  const int2 first_span = span<K>(a, seq, row0 / group);
  const int2 last_span = span<K>(a, seq, (min(row0 + kMidRows, rows) - 1) / group);
  const int key_lo = first_span.x, key_hi = last_span.y;  // seen by some row
  const int all_lo = last_span.x, all_hi = first_span.y;  // seen by every row
  const int last = kPlain<K> ? (key_hi + kMidKeys - 1) / kMidKeys : way.last;
  const uint32_t heads = a.kv_heads * a.group;
  const int row = row0 + n, token = row / group, g = row - token * group;
  if (part > 0 && step - wave >= last) {  // no keys: part 0 stands for an empty row
    if (threadIdx.x < kMidRows && row < rows) a.part_ml[few_place<K>(a, seq, part, b, row, head)] = {-kInf, 0};
    return;
  }

  // Q operands: channels D/2 half + 8 s + {0,4,1,5,2,6,3,7}. Rows past the last are zeros.
  uint4 qf[kSteps];
  float sum = 0.0f;
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    uint4 x = {0, 0, 0, 0};
    if (row < rows)
      x = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.q) +
                                          (size_t)(seq.start + token) * a.q_stride +
                                          (head * group + g) * D + (D / 2) * half + 8 * s);
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) sum += widen<kBf16>(w[i] & 0xffffu) + widen<kBf16>(w[i] >> 16);
    qf[s] = {(x.x & 0xffffu) | (x.z << 16), (x.x >> 16) | (x.z & 0xffff0000u),
             (x.y & 0xffffu) | (x.w << 16), (x.y >> 16) | (x.w & 0xffff0000u)};
  }
  const float q_sum = across32<false>(sum);
  const int2 seen = row < rows ? span<K>(a, seq, token) : int2{0, 0};

  RowSums<D> r;
#pragma unroll
  for (int d = 0; d < kBlocks; ++d) r.o[d] = v16f{};
  r.m = row < rows ? -kInf : 0.0f;
  r.l = 0.0f;
  float mid = 0.0f;                    // sum p (m + 8 s)
  float s_top = 0.0f, s_factor = 0.0f;  // f16: a power of two no scale passes, and kHeld over it
  // The sum of a row's p s, by a 16 x 16 x 32 product of the same operands: its columns are rows n % 16,
  // lanes 16 and on of each half bringing the keys of rows 16 and on, and its rows 4 (lane / 16) and on
  // take the ones of the lane's own kind.
  v4f ones = {0, 0, 0, 0};
  const uint32_t one2 = ((lane >> 2) & 1) == ((lane >> 4) & 1) ? (kBf16 ? 0x3F803F80u : 0x3C003C00u) : 0u;
  const uint4 one8 = {one2, one2, one2, one2};
  const Codes codes = make_codes<kBf16>();

  auto attend = [&](const MidStep<D>& cur, MidStep<D>& next) {
    const int key0 = way.key(step);
    if (step + stride < last) {
      const int now = ids;
      ids = page_of<K>(a, table, seq, (kPlain<K> ? key0 + 2 * kMidKeys * stride : way.key(step + 2 * stride)) + mine);
      load_mid<D, kOnce>(a, now, head, kPlain<K> ? key0 + kMidKeys * stride : way.key(step + stride), lane, next);
    }
    v16f x = v16f{};
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const uint4 kf = {code_pair<kBf16>(cur.k[s], 0, codes), code_pair<kBf16>(cur.k[s], 1, codes),
                        code_pair<kBf16>(cur.k[s], 2, codes), code_pair<kBf16>(cur.k[s], 3, codes)};
      x = mfma32<kBf16>(kf, qf[s], x);
    }
    const float ks = widen<kBf16>(cur.ks >> 16) * a.scale;
    float km = widen<kBf16>(cur.kw & 0xffffu) * a.scale;
    km = fmaf(-16.0f, widen<kBf16>(cur.kw >> 16) * a.scale, km);
    float vs = widen<kBf16>(cur.vs >> 16), vm = fmaf(8.0f, vs, widen<kBf16>(cur.vs & 0xffffu));
    const bool whole = all_seen<K>(seq, all_lo, all_hi, key0, kMidKeys) && cur.hidden == 0;
    if (!whole) {
      // A key whose V words hold a NaN gives NaN through its score, where only the rows that see it
      // look; the words of keys that no row sees may hold anything.
      const bool nan = has_nan<kBf16>(cur.vs);
      const uint64_t nans = __ballot(nan);  // of register lane % 16's keys
      if ((nans >> ((mine & 7) | (mine & 8) << 2 | (mine & 16) >> 1)) & 1) km = __uint_as_float(0x7fc00000u);
      const int key = key0 + (lane & 7) + 8 * half + 2 * (lane & 8);
      const bool none = unseen<K>(seq, {key_lo, key_hi}, key) || (cur.hidden >> (2 * (lane & 8))) & 1;
      if (none || nan) vs = vm = 0.0f;
    }
    scale_scores(ks, x);
    const v16f y = [&] {
      v16f y = __builtin_amdgcn_mfma_f32_32x32x2f32(half ? -1.0f : km, half ? r.base() : q_sum, x, 0, 0, 0);
      if (!whole) {
        asm volatile("");  // a branch, not 16 selects in every step
        const int lo = seen.x - key0 - 8 * half, hi = seen.y - key0 - 8 * half;
        const int front = kPlain<K> ? 0 : seq.front - key0 - 8 * half;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int k = (i & 7) + 2 * (i & 8);
          if ((k < lo && (kPlain<K> || k >= front)) || k >= hi || (cur.hidden >> (2 * (i & 8))) & 1)
            y[i] = -kInf;
        }
      }
      return y;
    }();
    float p[16], ts = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      p[i] = __builtin_amdgcn_exp2f(y[i]);
      ts += p[i];
    }
    bool raise = !(ts <= kMidTop) || r.m == -kInf;
    if constexpr (!kBf16) raise |= vs > s_top;
    if (__any(raise)) {
      float ratio = 1.0f;
      if constexpr (!kBf16) {
        const float s = across32<true>(across16<true>(over16<true>(vs)));
        if (s > s_top) {
          const float up = __uint_as_float((__float_as_uint(s) + 0x7fffffu) & 0x7f800000u);
          ratio = s_top / up;
          s_top = up;
          s_factor = kHeld / up;
        }
      }
      const float was = r.base();
      float top = y[0];
#pragma unroll
      for (int i = 1; i < 16; ++i) top = fmaxf(top, y[i]);
      top = across32<true>(top) + was;
      const float up = fmaxf(r.m, top);
      const float alpha = __builtin_amdgcn_exp2f(r.m - (up == -kInf ? 0.0f : up));
      r.m = up;
      const float by = was - r.base();
      r.l *= alpha;
      mid *= alpha;
      ones *= alpha * ratio;
#pragma unroll
      for (int d = 0; d < kBlocks; ++d) r.o[d] *= alpha * ratio;
      ts = 0.0f;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        p[i] = __builtin_amdgcn_exp2f(y[i] + by);
        ts += p[i];
      }
    }
    r.l += ts;
    float ps[16];
    weigh(kBf16 ? vs : vs * s_factor, p, ps);
    mid = add_weighed(mid, vm, p);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const float* w = ps + 8 * t;
      const uint4 pf = {narrow2<kBf16>(w[0], w[1]), narrow2<kBf16>(w[2], w[3]), narrow2<kBf16>(w[4], w[5]),
                        narrow2<kBf16>(w[6], w[7])};
      ones = mfma16<kBf16>(one8, pf, ones);
      uint32_t v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = cur.v[8 * t + 2 * i] | (cur.v[8 * t + 2 * i + 1] << 16);
#pragma unroll
      for (int d = 0; d < kBlocks; ++d)
        r.o[d] = mfma32<kBf16>({code_pair<kBf16>(v[0], d, codes), code_pair<kBf16>(v[1], d, codes),
                                code_pair<kBf16>(v[2], d, codes), code_pair<kBf16>(v[3], d, codes)},
                               pf, r.o[d]);
    }
  };
  for (; step < last; step += stride) {
    attend(tiles[0], tiles[1]);
    step += stride;
    if (step >= last) break;
    attend(tiles[1], tiles[0]);
  }

  // Join the four waves. Register i of block d holds channel (D/32) (8 (i / 4) + 4 half + i % 4) + d.
  const float unit = kBf16 ? 1.0f : s_top * (1.0f / kHeld);
  const float l = across32<false>(r.l), add = across32<false>(mid);
  if (half == 0) lds_ml[wave][n] = {r.m, l};
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    float* to = &lds_o[wave][n][kBlocks * (8 * (i / 4) + 4 * half + i % 4)];
#pragma unroll
    for (int d = 0; d < kBlocks; ++d) to[d] = fmaf(unit, fmaf(-24.0f, ones[0], r.o[d][i]), add);
  }
  __syncthreads();
  const int at = (int)threadIdx.x / 8, ch = 4 * ((int)threadIdx.x % 8);  // channels ch + 32 j + 0..3
  const int out_row = row0 + at;
  if (out_row >= rows) return;
  float2 ml[kWaves];
  float top = -kInf, total = 0.0f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    ml[w] = lds_ml[w][at];
    top = fmaxf(top, ml[w].x);
  }
  const float base = top == -kInf ? 0.0f : top;
  float4 sums[kBlocks];
#pragma unroll
  for (int j = 0; j < kBlocks; ++j) sums[j] = {0, 0, 0, 0};
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const float f = __builtin_amdgcn_exp2f(ml[w].x - base);
    total = fmaf(f, ml[w].y, total);
#pragma unroll
    for (int j = 0; j < kBlocks; ++j) {
      const float4 x = *reinterpret_cast<const float4*>(&lds_o[w][at][ch + 32 * j]);
      sums[j] = {fmaf(f, x.x, sums[j].x), fmaf(f, x.y, sums[j].y), fmaf(f, x.z, sums[j].z),
                 fmaf(f, x.w, sums[j].w)};
    }
  }
  total = or_nan(total, sums[0].x);
  const int out_token = out_row / group, out_g = out_row - out_token * group;
  const size_t q_row = (size_t)(seq.start + out_token);
  const uint32_t q_head = head * group + out_g;
  if (kPart<K> || a.parts > 1) {
    const size_t place = few_place<K>(a, seq, part, b, out_row, head);
#pragma unroll
    for (int j = 0; j < kBlocks; ++j)
      *reinterpret_cast<float4*>(a.part_o + place * D + ch + 32 * j) = sums[j];
    if (ch == 0) a.part_ml[place] = {top, total};
  } else {
    const bool none = total == 0.0f;  // a NaN among the scores or values leaves total NaN
    const Mean by = make_mean<kBf16>(total);
    uint16_t* out = static_cast<uint16_t*>(a.out) + q_row * a.out_stride + q_head * D + ch;
#pragma unroll
    for (int j = 0; j < kBlocks; ++j)
      *reinterpret_cast<uint2*>(out + 32 * j) = {
          narrow2<kBf16>(mean<kBf16>(sums[j].x, by), mean<kBf16>(sums[j].y, by)),
          narrow2<kBf16>(mean<kBf16>(sums[j].z, by), mean<kBf16>(sums[j].w, by))};
    if (a.lse && ch == 0) a.lse[q_row * heads + q_head] = none ? -kInf : (top + __log2f(total)) * kLn2;
  }
}

template <int D, bool kBf16, bool kOnce, Keys K>
__global__ __launch_bounds__(kThreads, 2) void k_attention_kv4_mid(Args a) {
  __shared__ MidLds<D> lds;
  attend_mid<D, kBf16, kOnce, K>(a, lds, blockIdx.x, blockIdx.y, blockIdx.z);
}

// One wave's joined row: D/64 channels a lane.
template <int D, bool kBf16>
__device__ __forceinline__ void write_row(const Args& a, size_t q_row, uint32_t q_head, int lane,
                                          float m, float l, const float (&sum)[D / 64]) {
  const bool none = l == 0.0f;
  const Mean by = make_mean<kBf16>(l);
  uint16_t* out = static_cast<uint16_t*>(a.out) + q_row * a.out_stride + q_head * D + lane * (D / 64);
  if constexpr (D == 128)
    *reinterpret_cast<uint32_t*>(out) = narrow2<kBf16>(mean<kBf16>(sum[0], by), mean<kBf16>(sum[1], by));
  else
    *out = (uint16_t)narrow<kBf16>(mean<kBf16>(sum[0], by));
  if (a.lse && lane == 0)
    a.lse[q_row * (a.kv_heads * a.group) + q_head] = none ? -kInf : (m + __log2f(l)) * kLn2;
}

// The tiles of keys that the rows from row0 on see.
template <Keys K>
__device__ __forceinline__ Steps row_steps(const Args& a, const Sequence& seq, int row0) {
  const int group = (int)a.group, rows = seq.rows * group;
  const int lo = span<K>(a, seq, row0 / group).x;
  const int hi = span<K>(a, seq, (min(row0 + kTileRows, rows) - 1) / group).y;
  const auto way = walk<K, kTileKeys>(seq, lo, hi);
  return {way.first, max(way.last, way.first)};
}

template <int D, bool kBf16, Keys K>
__global__ __launch_bounds__(kRowsThreads, 2) void k_attention_kv4_rows(Args a) {
  __shared__ __attribute__((aligned(16))) RowsLds<D> lds;
  const Sequence seq = sequence<K>(a, blockIdx.z);
  const int rows = seq.rows * (int)a.group;
  // A row tile's heads side by side; the last rows see the most keys: they start first.
  const uint32_t tile = blockIdx.x / a.kv_heads, head = blockIdx.x - tile * a.kv_heads;
  const int row0 = (int)(a.row_tiles - 1 - tile) * kTileRows;
  if (row0 >= rows || !takes(a, rows)) return;
  attend_rows<D, kBf16, K>(a, lds, seq, blockIdx.z, head, row0, row_steps<K>(a, seq, row0), kPart<K> ? 0 : -1);
}

// The same row tiles where they would leave the chip partly idle: the tiles of keys of all of them (of
// every cache head) are one line, of which each workgroup takes an equal range. A range that holds a
// row tile's keys whole finishes it; one that ends or begins inside leaves its sums in the workspace,
// in slot 2 w if it is workgroup w's first and 2 w + 1 if its last, for k_attention_kv4_rows_join. Every
// workgroup finds the line from the sequences by itself (at most kLineTiles row tiles and sequences;
// rows that q_starts counts twice may have none), and the first leaves it in the workspace for the join.
// 1,025 tokens of 32 heads on 8 over 8,192 keys: 172 us and 15 for the join, 255 apart.
constexpr int kLineTiles = 512;  // one per thread
constexpr int kLeastSteps = 8;   // of a range: a shorter one is mostly start and join

struct Line {
  int tiles, steps, range;  // row tiles, their steps (of one head), a workgroup's steps
  int unused;
  int b[kLineTiles], row0[kLineTiles], first[kLineTiles];
  int end[kLineTiles];  // of a row tile's steps in the line of one head
};

// The sum of v over the threads up to this one, of kRowsThreads. `scratch`: eight ints.
__device__ __forceinline__ int sum_to_here(int v, int* scratch) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int x = __shfl_up(v, d);
    if (lane >= d) v += x;
  }
  if (lane == 63) scratch[wave] = v;
  __syncthreads();
  for (int w = 0; w < wave; ++w) v += scratch[w];
  __syncthreads();
  return v;
}

template <Keys K>
__device__ __forceinline__ void make_line(const Args& a, Line& line, int* scratch) {
  const int t = (int)threadIdx.x;
  int tiles = 0;
  if (t < (int)a.batch) {
    const int rows = sequence<K>(a, t).rows * (int)a.group;
    if (takes(a, rows)) tiles = (rows + kTileRows - 1) / kTileRows;
  }
  const int after = sum_to_here(tiles, scratch);
  for (int i = 0, at = after - tiles; i < tiles && at < (int)a.row_tiles; ++i, ++at) {
    line.b[at] = t;
    line.row0[at] = i * kTileRows;
  }
  if (t == kRowsThreads - 1) line.tiles = min(after, (int)a.row_tiles);
  __syncthreads();
  int count = 0;
  if (t < line.tiles) {
    const Steps st = row_steps<K>(a, sequence<K>(a, line.b[t]), line.row0[t]);
    line.first[t] = st.first;
    count = max(st.last - st.first, 1);  // a tile that sees no key still has its rows to write
  }
  const int end = sum_to_here(count, scratch);
  if (t < kLineTiles) line.end[t] = end;
  if (t == kRowsThreads - 1) {
    line.steps = end;
    const int all = end * (int)a.kv_heads;
    line.range = max((all + (int)gridDim.x - 1) / (int)gridDim.x, kLeastSteps);
  }
  __syncthreads();
}

template <int D, bool kBf16, Keys K>
__global__ __launch_bounds__(kRowsThreads, 2) void k_attention_kv4_line(Args a) {
  __shared__ __attribute__((aligned(16))) RowsLds<D> lds;
  __shared__ Line line;
  __shared__ int scratch[8];
  make_line<K>(a, line, scratch);
  if (blockIdx.x == 0)
    for (int i = threadIdx.x; i < (int)(sizeof(Line) / 4); i += kRowsThreads)
      reinterpret_cast<int*>(a.line)[i] = reinterpret_cast<const int*>(&line)[i];
  const int steps = __builtin_amdgcn_readfirstlane(line.steps);
  const int range = __builtin_amdgcn_readfirstlane(line.range);
  const int begin = (int)blockIdx.x * range, stop = min(begin + range, steps * (int)a.kv_heads);
  for (int at = begin; at < stop;) {
    const int head = at / steps, off = at - head * steps;
    int lo = 0, hi = line.tiles - 1;  // the first row tile that ends past off
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (line.end[mid] > off) hi = mid; else lo = mid + 1;
    }
    const int tile = __builtin_amdgcn_readfirstlane(lo);
    const int start = __builtin_amdgcn_readfirstlane(tile ? line.end[tile - 1] : 0);
    const int count = __builtin_amdgcn_readfirstlane(line.end[tile]) - start;
    const int first = __builtin_amdgcn_readfirstlane(line.first[tile]);
    const int b = __builtin_amdgcn_readfirstlane(line.b[tile]);
    const int row0 = __builtin_amdgcn_readfirstlane(line.row0[tile]);
    const int s0 = off - start, s1 = min(count, s0 + stop - at);
    const int slot = s1 - s0 == count ? -1 : 2 * (int)blockIdx.x + (at == begin ? 0 : 1);
    attend_rows<D, kBf16, K>(a, lds, sequence<K>(a, b), b, head, row0, {first + s0, first + s1}, slot);
    __syncthreads();  // LDS is free again
    at += s1 - s0;
  }
}

// Joins the ranges of the row tiles that more than one workgroup took: W waves per row, wave w the ranges
// w, w + W, ..
template <int D, bool kBf16, int W>
__global__ __launch_bounds__(kThreads) void k_attention_kv4_rows_join(Args a) {
  constexpr int kPer = D / 64, kTileGroups = kTileRows * W / kWaves;
  __shared__ float lds_sum[W][D];
  __shared__ float2 lds_ml[W];
  const Line& line = *a.line;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tile = blockIdx.x / kTileGroups;
  if (tile >= line.tiles) return;
  const int start = (int)blockIdx.y * line.steps + (tile ? line.end[tile - 1] : 0);
  const int end = (int)blockIdx.y * line.steps + line.end[tile];
  const int w0 = start / line.range, w1 = (end - 1) / line.range;
  if (w0 == w1) return;
  const Sequence seq = sequence<kOwn>(a, line.b[tile]);
  const int in_tile = (int)(blockIdx.x % kTileGroups) * (kWaves / W) + wave / W;
  const int row = line.row0[tile] + in_tile, group = (int)a.group;
  if (row >= seq.rows * group) return;  // whole workgroups leave where W waves share a row
  float m = -kInf, l = 0.0f, sum[kPer];
#pragma unroll
  for (int d = 0; d < kPer; ++d) sum[d] = 0.0f;
  for (int w = w0 + wave % W; w <= w1; w += W) {
    const size_t place = (size_t)(2 * w + (w * line.range >= start ? 0 : 1)) * kTileRows + in_tile;
    const float2 ml = a.part_ml[place];
    const float* x = a.part_o + place * D + lane * kPer;
    const float up = fmaxf(m, ml.x), base = up == -kInf ? 0.0f : up;
    const float was = __builtin_amdgcn_exp2f(m - base), f = __builtin_amdgcn_exp2f(ml.x - base);
    m = up;
    l = l * was + f * ml.y;
#pragma unroll
    for (int d = 0; d < kPer; ++d) sum[d] = sum[d] * was + f * x[d];
  }
  if constexpr (W > 1) {
    if (lane == 0) lds_ml[wave] = {m, l};
#pragma unroll
    for (int d = 0; d < kPer; ++d) lds_sum[wave][lane * kPer + d] = sum[d];
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int w = 1; w < W; ++w) {
      const float2 ml = lds_ml[w];
      const float up = fmaxf(m, ml.x), base = up == -kInf ? 0.0f : up;
      const float was = __builtin_amdgcn_exp2f(m - base), f = __builtin_amdgcn_exp2f(ml.x - base);
      m = up;
      l = l * was + f * ml.y;
#pragma unroll
      for (int d = 0; d < kPer; ++d) sum[d] = sum[d] * was + f * lds_sum[w][lane * kPer + d];
    }
  }
  const int token = row / group, g = row - token * group;
  const size_t q_row = (size_t)(seq.start + token);
  write_row<D, kBf16>(a, q_row, blockIdx.y * a.group + g, lane, m, l, sum);
}

// Joins the parts of a row: W waves per (row, query head), wave w the parts w, w + W, ..; lane p of a
// wave holds part p's weight (kMaxParts lanes at most). A part without keys has no sums to read.
constexpr uint32_t kMaxParts = 64;
constexpr uint32_t kFewRows = 32;    // rows in one tile of k_attention_kv4_few or _mid
constexpr uint32_t kFewMost = 4096;  // rows of a sequence that they take
constexpr double kFewBytes = 64e6;   // of their parts' sums

// At least the row tiles of a call's sequences: a sequence of r rows has r / 256 and a part of one.
uint32_t line_tiles(uint32_t batch, uint32_t q_rows, uint32_t max_q, uint32_t group) {
  const uint64_t all = (uint64_t)q_rows * group / kTileRows + batch;
  const uint64_t each = ((uint64_t)max_q * group + kTileRows - 1) / kTileRows;
  return (uint32_t)std::min(all, each * batch);
}

template <int D, bool kBf16, int W>
__global__ __launch_bounds__(kThreads) void k_attention_kv4_join(Args a) {
  constexpr int kPer = D / 64;
  __shared__ float lds_sum[W == 1 ? 1 : W][D];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int parts = (int)a.parts;
  const uint32_t row = blockIdx.x * (kWaves / W) + wave / W;
  const size_t place = few_place<kOwn>(a, {}, 0, blockIdx.z, min(row, a.rows_to - 1), blockIdx.y);
  const size_t pitch = (size_t)a.batch * a.rows_to * a.kv_heads;
  const float* from = a.part_o + place * D + lane * kPer;
  auto load = [&](int p, float (&x)[4][kPer]) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int d = 0; d < kPer; ++d) x[i][d] = p + i * W < parts ? from[(p + i * W) * pitch * D + d] : 0.0f;
  };
  // The weights and the first four parts' sums are under way before the row is known to be there.
  const float2 ml = lane < parts ? a.part_ml[lane * pitch + place] : float2{-kInf, 0.0f};
  float x[4][kPer], sum[kPer];
  load(wave % W, x);
  const Sequence seq = sequence<kOwn>(a, blockIdx.z);
  const uint32_t token = row / a.group, g = row - token * a.group;
  if ((int)token >= seq.rows || !takes(a, seq.rows * (int)a.group)) return;
  const size_t q_row = (size_t)(seq.start + token);
  const uint32_t q_head = blockIdx.y * a.group + g;
  const float top = across32<true>(across16<true>(over16<true>(ml.x)));
  const float f = __builtin_amdgcn_exp2f(ml.x - (top == -kInf ? 0.0f : top));
  const float total = across32<false>(across16<false>(over16<false>(f * ml.y)));
  const uint64_t live = __ballot(!(ml.y == 0.0f));  // the parts with sums: those with a weight or a NaN
#pragma unroll
  for (int d = 0; d < kPer; ++d) sum[d] = 0.0f;
  for (int p = wave % W; p < parts; p += 4 * W) {
    if (p >= 4 * W) {
      if (live >> p == 0) break;
      load(p, x);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int part = p + i * W;
      if (part >= parts || !((live >> part) & 1)) continue;
      const float w = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(f), part));
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
  write_row<D, kBf16>(a, q_row, q_head, lane, top, total, sum);
}

template <int D, bool kBf16, bool kOnce, Keys K>
void launch_tiles(const Args& a, const Kv4Launch& plan, hipStream_t stream) {
  const dim3 grid(plan.parts, a.kv_heads * plan.row_tiles, a.batch), block(kThreads);
  if (plan.tile_rows == 4)
    hipLaunchKernelGGL((k_attention_kv4_few<D, kBf16, 4, kOnce, K>), grid, block, 0, stream, a);
  else if (plan.tile_rows == 8)
    hipLaunchKernelGGL((k_attention_kv4_few<D, kBf16, 8, kOnce, K>), grid, block, 0, stream, a);
  else if (plan.tile_rows == 16)
    hipLaunchKernelGGL((k_attention_kv4_few<D, kBf16, 16, kOnce, K>), grid, block, 0, stream, a);
  else
    hipLaunchKernelGGL((k_attention_kv4_mid<D, kBf16, kOnce, K>), grid, block, 0, stream, a);
}

// Whether codes go past the caches: where one row tile reads them and the call may read more than half of
// the 256 MB of the last cache, so that the next call would not meet them there. 32 sequences of 4,096 keys
// (142 MB, 8 cache heads of 128 channels) 46 us in the caches and 41 past them, two of 129,024 63 and 58;
// 16 of 4,096, called again and again, 27 and 31. Rows of 64 channels are a quarter of a line each and gain
// nothing (64 sequences of 8,192 keys 53 and 58 us). In one pass behind a prefix they go through them, since the prefix's
// come to every sequence and one kernel reads both: 64 sequences of 8,192 keys of their own 86 us behind 64 shared ones
// (82 past the caches) and 103 behind 2,000 (101).
bool reads_once(const Args& a, const Kv4Launch& plan, int dim) {
  const double keys = (double)((uint64_t)a.table_stride << a.page_shift);
  const double seen = a.window ? std::min(keys, (double)a.window + a.sinks + a.max_q) : keys;
  return dim == 128 && plan.row_tiles == 1 && seen * a.batch * a.kv_heads * (dim + 8) > 128e6;
}

template <int D, bool kBf16, Keys K>
hipError_t launch_few(Args a, const Kv4Launch& plan, hipStream_t stream) {
  if (plan.row_tiles == 0) return hipSuccess;
  a.parts = plan.parts;
  a.row_tiles = plan.row_tiles;
  a.rows_from = plan.rows_from;
  a.rows_to = plan.rows_to;
  a.part_ml = reinterpret_cast<float2*>(a.part_o + (size_t)plan.parts * a.batch * plan.rows_to *
                                                       a.kv_heads * D);
  if constexpr (D == 128 && K != kPrefix) {
    if (reads_once(a, plan, D))
      launch_tiles<D, kBf16, true, K>(a, plan, stream);
    else
      launch_tiles<D, kBf16, false, K>(a, plan, stream);
  } else {
    launch_tiles<D, kBf16, false, K>(a, plan, stream);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || plan.parts == 1) return e;
  const uint32_t rows = std::min(a.max_q * a.group, plan.rows_to);
  if (plan.parts > 8)
    hipLaunchKernelGGL((k_attention_kv4_join<D, kBf16, kWaves>), dim3(rows, a.kv_heads, a.batch),
                       dim3(kThreads), 0, stream, a);
  else
    hipLaunchKernelGGL((k_attention_kv4_join<D, kBf16, 1>),
                       dim3((rows + kWaves - 1) / kWaves, a.kv_heads, a.batch), dim3(kThreads), 0,
                       stream, a);
  return hipGetLastError();
}

template <int D, bool kBf16, Keys K>
hipError_t launch_many(Args a, const Kv4Launch& plan, hipStream_t stream) {
  if (plan.row_tiles == 0) return hipSuccess;
  a.row_tiles = plan.row_tiles;
  a.rows_from = plan.rows_from;
  a.rows_to = plan.rows_to;
  if (plan.parts == 1) {
    hipLaunchKernelGGL((k_attention_kv4_rows<D, kBf16, K>), dim3(a.kv_heads * plan.row_tiles, 1, a.batch),
                       dim3(kRowsThreads), 0, stream, a);
    return hipGetLastError();
  }
  a.part_ml = reinterpret_cast<float2*>(a.part_o + (size_t)2 * plan.parts * kTileRows * D);
  a.line = reinterpret_cast<Line*>(a.part_ml + (size_t)2 * plan.parts * kTileRows);
  const uint32_t tiles = line_tiles(a.batch, a.q_rows, a.max_q, a.group);
  a.row_tiles = tiles;
  hipLaunchKernelGGL((k_attention_kv4_line<D, kBf16, K>), dim3(plan.parts), dim3(kRowsThreads), 0, stream,
                     a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  // A workgroup a row where the rows alone would leave the chip idle.
  if (tiles * a.kv_heads <= 64)
    hipLaunchKernelGGL((k_attention_kv4_rows_join<D, kBf16, kWaves>),
                       dim3(tiles * kTileRows, a.kv_heads), dim3(kThreads), 0, stream, a);
  else
    hipLaunchKernelGGL((k_attention_kv4_rows_join<D, kBf16, 1>),
                       dim3(tiles * kTileRows / kWaves, a.kv_heads), dim3(kThreads), 0, stream, a);
  return hipGetLastError();
}

template <int D, bool kBf16, Keys K>
hipError_t launch_both(const Args& a, const Kv4Plan& plan, hipStream_t stream) {
  const hipError_t e = launch_many<D, kBf16, K>(a, plan.many, stream);
  return e != hipSuccess ? e : launch_few<D, kBf16, K>(a, plan.few, stream);
}

template <Keys K>
hipError_t launch_keys(const h3_kv4_cfg& cfg, const Args& a, const Kv4Plan& plan, hipStream_t stream) {
  const bool bf16 = cfg.elem == H3_ELEM_BF16;
  if (cfg.head_dim == 128)
    return bf16 ? launch_both<128, true, K>(a, plan, stream) : launch_both<128, false, K>(a, plan, stream);
  return bf16 ? launch_both<64, true, K>(a, plan, stream) : launch_both<64, false, K>(a, plan, stream);
}

// What every launch of a call has; the parts' places and numbers are the launch's own.
Args make_args(const h3_kv4_cfg& cfg, const h3_kv4_attention_cfg& acfg, uint32_t batch, uint32_t q_rows,
               uint32_t max_q, const Kv4Bindings& x) {
  Args a{};
  a.q = x.q;
  a.cache = static_cast<const uint8_t*>(x.cache);
  a.table = x.table;
  a.prefix_table = x.prefix_table;
  a.prefix_length = x.prefix_length;
  a.lengths = x.lengths;
  a.q_starts = x.q_starts;
  a.out = x.out;
  a.lse = x.lse;
  a.part_o = static_cast<float*>(x.workspace);
  a.kv_heads = cfg.kv_heads;
  a.group = acfg.heads / cfg.kv_heads;
  a.q_stride = acfg.q_stride;
  a.out_stride = acfg.out_stride;
  a.table_stride = acfg.table_stride;
  a.pages = cfg.pages;
  a.page_shift = __builtin_ctz(cfg.page_tokens);
  a.batch = batch;
  a.q_rows = q_rows;
  a.max_q = max_q;
  a.causal = acfg.causal;
  a.window = acfg.window;
  a.scale = acfg.scale * kLog2e;
  return a;
}

}  // namespace

}  // namespace h3
