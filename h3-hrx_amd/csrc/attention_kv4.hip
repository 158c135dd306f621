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
// raised as the running maximum is), times 2^14: weights down to 2^-28 of the largest stay normal.
//
// A query row is one (token, query head) pair; the G = heads / kv_heads heads of one cache head
// are rows of the same matrix, row = token * G + g, so that a key is read once for all of them.
#include <algorithm>

#include "internal.hpp"

namespace h3 {
namespace {

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kKeys = 32;  // keys of a wave's step: two 16-key score tiles, one PV step
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kInf = __builtin_inff();

struct Args {
  const void* q;
  const uint8_t* cache;
  const int32_t* table;
  const int32_t* lengths;
  const int32_t* q_starts;
  void* out;
  float* lse;  // null: not wanted
  float* part_o;
  float2* part_ml;
  uint32_t kv_heads, group, q_stride, out_stride, table_stride;
  uint32_t pages, page_shift;
  uint32_t q_rows, max_q;
  uint32_t parts, row_tiles;
  uint32_t rows_from, rows_to;  // the sequences a launch takes: those of rows_from .. rows_to rows
  uint32_t causal, window;
  float scale;  // the softmax scale times log2(e)
};

// A sequence's rows and keys, from device memory and so checked here: rows that q does not have,
// or past max_q, are not computed, keys past the table's columns not read.
struct Sequence {
  int start, n, rows, length;  // first row of q, its rows, the rows computed, keys
};
__device__ __forceinline__ Sequence sequence(const Args& a, uint32_t b) {
  Sequence s;
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
__device__ __forceinline__ int2 span(const Args& a, const Sequence& s, int i) {
  if (!a.causal) return {0, s.length};
  const int p = s.length - s.n + i;
  const int hi = min(max(p + 1, 0), s.length);
  const int lo = a.window ? (int)max((int64_t)p + 1 - a.window, (int64_t)0) : 0;
  return {min(lo, hi), hi};
}

// The steps of `keys` keys that a tile of rows takes, and the ones of them part `part` takes.
struct Steps {
  int first, last;
};
__device__ __forceinline__ Steps steps(int lo, int hi, uint32_t parts, uint32_t part, int keys) {
  const int t0 = lo / keys, t1 = (hi + keys - 1) / keys;
  const int n = max(t1 - t0, 0);
  const int per = (n + (int)parts - 1) / (int)parts;
  return {t0 + min((int)part * per, n), t0 + min(((int)part + 1) * per, n)};
}

template <bool kBf16>
__device__ __forceinline__ float widen(uint32_t bits) {
  if constexpr (kBf16) return __uint_as_float(bits << 16);
  return (float)__builtin_bit_cast(_Float16, (uint16_t)bits);
}
template <bool kBf16>
__device__ __forceinline__ uint32_t narrow(float v) {
  if constexpr (kBf16) return __builtin_bit_cast(uint16_t, (__bf16)v);
  return __builtin_bit_cast(uint16_t, (_Float16)v);
}
template <bool kBf16>
__device__ __forceinline__ uint32_t narrow2(float lo, float hi) {
  return narrow<kBf16>(lo) | (narrow<kBf16>(hi) << 16);
}

// Nibble n of both halves of w as a pair of 16 + u.
template <bool kBf16>
__device__ __forceinline__ uint32_t code_pair(uint32_t w, int n) {
  constexpr int kAt = kBf16 ? 3 : 6;  // the code's lowest bit in the mantissa
  const int shift = kAt - 4 * n;
  const uint32_t at = shift >= 0 ? w << shift : w >> -shift;
  return (at & (kBf16 ? 0x00780078u : 0x03C003C0u)) | (kBf16 ? 0x41804180u : 0x4C004C00u);
}

template <bool kBf16>
__device__ __forceinline__ v4f mfma16(uint4 a, uint4 b, v4f c) {
  if constexpr (kBf16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a),
                                                   __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a),
                                                __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}

// What one lane loads of a wave's 32 keys: lane (n = lane % 16, h = lane / 16) the K codes of key n
// of either 16-key half, channels D/4 h and on; the V codes of keys 4h + e of either half, channels
// D/16 n and on; and those keys' K and V words.
template <int D>
struct Tile {
  uint32_t k[2][D / 32];
  uint32_t v[8];
  uint4 kw[2], vw[2];
};

template <int D>
__device__ __forceinline__ void load_half(const uint8_t* block, uint32_t in_page,
                                          uint32_t page_tokens, int half, int n, int h,
                                          Tile<D>& t) {
  const uint8_t* kc = block + in_page * (D / 2);
  const uint8_t* vc = kc + page_tokens * (D / 2);
  const uint8_t* kw = block + page_tokens * D + in_page * 4;
  const uint8_t* vw = kw + page_tokens * 4;
  if constexpr (D == 128) {
    const uint4 k = *reinterpret_cast<const uint4*>(kc + n * 64 + 16 * h);
    t.k[half][0] = k.x, t.k[half][1] = k.y, t.k[half][2] = k.z, t.k[half][3] = k.w;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      t.v[4 * half + e] = *reinterpret_cast<const uint32_t*>(vc + (4 * h + e) * 64 + 4 * n);
  } else {
    const uint2 k = *reinterpret_cast<const uint2*>(kc + n * 32 + 8 * h);
    t.k[half][0] = k.x, t.k[half][1] = k.y;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      t.v[4 * half + e] = *reinterpret_cast<const uint16_t*>(vc + (4 * h + e) * 32 + 2 * n);
  }
  t.kw[half] = *reinterpret_cast<const uint4*>(kw + 16 * h);
  t.vw[half] = *reinterpret_cast<const uint4*>(vw + 16 * h);
}

// The pages of a step's two halves; -1 where the table names none that the cache has.
struct Pages {
  int id[2];
};
__device__ __forceinline__ Pages pages_of(const Args& a, const int32_t* table, int key) {
  Pages p;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const uint32_t col = (uint32_t)(key + 16 * half) >> a.page_shift;
    const int id = col < a.table_stride ? table[col] : -1;
    p.id[half] = (uint32_t)id < a.pages ? id : -1;
  }
  return p;
}

template <int D>
__device__ __forceinline__ void load_tile(const Args& a, const Pages& p, uint32_t head, int key,
                                          int n, int h, Tile<D>& t) {
  const uint32_t page_tokens = 1u << a.page_shift;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const uint64_t page = max(p.id[half], 0);  // keys of no page are masked; page 0 is there to read
    const uint8_t* block =
        a.cache + (page * a.kv_heads + head) * ((uint64_t)page_tokens * (D + 8));
    load_half<D>(block, (uint32_t)(key + 16 * half) & (page_tokens - 1), page_tokens, half, n, h, t);
  }
}

__device__ __forceinline__ float quarter_max(float v) {  // over the lanes with the same lane % 16
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float quarter_sum(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}

// Few rows: a workgroup's four waves hold the same QT * 16 rows of one cache head and take every
// fourth step of its keys; their results are joined in LDS. S^T = K Q^T and O^T = V^T P^T, both
// 16 x 16 x 32: a lane's score registers are four keys of one row, and they are the lane's own part
// of the next product's operand, so no probability crosses lanes.
template <int D, bool kBf16, int QT>
__global__ __launch_bounds__(kThreads) void k_attention_kv4_few(Args a) {
  constexpr int kRows = 16 * QT, kSteps = D / 32, kDimTiles = D / 16;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, h = lane >> 4;
  const uint32_t head = blockIdx.y, b = blockIdx.z;
  const uint32_t part = blockIdx.x % a.parts;
  const Sequence seq = sequence(a, b);
  const int rows = seq.rows * (int)a.group;
  const int row0 = (int)(blockIdx.x / a.parts) * kRows;
  if (row0 >= rows || !takes(a, rows)) return;
  const int token0 = row0 / (int)a.group;
  const int token1 = min(row0 + kRows, rows) - 1;
  const int2 first_span = span(a, seq, token0), last_span = span(a, seq, token1 / (int)a.group);
  const int key_lo = first_span.x, key_hi = last_span.y;     // seen by some row
  const int all_lo = last_span.x, all_hi = first_span.y;     // seen by every row
  const Steps st = steps(key_lo, key_hi, a.parts, part, kKeys);
  const uint32_t heads = a.kv_heads * a.group;

  // Q^T operands: channel D/4 h + 8 s + {0,4,1,5,2,6,3,7} in k slot 8 h + 0..7 of step s, the order
  // in which the codes of a K word come out in pairs. Rows past the last are zeros.
  uint4 qf[QT][kSteps];
  float q_sum[QT];
  int2 seen[QT];
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const int row = row0 + 16 * t + n;
    const int token = row / (int)a.group, g = row - token * (int)a.group;
    seen[t] = row < rows ? span(a, seq, token) : int2{0, 0};
    float sum = 0.0f;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      uint4 x = {0, 0, 0, 0};
      if (row < rows)
        x = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.q) +
                                            (size_t)(seq.start + token) * a.q_stride +
                                            (head * a.group + g) * D + (D / 4) * h + 8 * s);
      const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) sum += widen<kBf16>(w[i] & 0xffffu) + widen<kBf16>(w[i] >> 16);
      qf[t][s] = {(x.x & 0xffffu) | (x.z << 16), (x.x >> 16) | (x.z & 0xffff0000u),
                  (x.y & 0xffffu) | (x.w << 16), (x.y >> 16) | (x.w & 0xffff0000u)};
    }
    q_sum[t] = quarter_sum(sum);
  }

  v4f o[QT][kDimTiles], ones[QT];
  float m[QT], base[QT], l[QT], mid[QT];  // base: m, or 0 while no key was seen; mid: sum p (m + 8 s)
#pragma unroll
  for (int t = 0; t < QT; ++t) {
#pragma unroll
    for (int d = 0; d < kDimTiles; ++d) o[t][d] = {0, 0, 0, 0};
    ones[t] = {0, 0, 0, 0};
    m[t] = -kInf;
    base[t] = l[t] = mid[t] = 0.0f;
  }
  float s_top = 0.0f;            // f16: the power of two that p s is held relative to
  float s_factor = 1.0f;         // what p is multiplied by beside s
  const uint32_t one2 = kBf16 ? 0x3F803F80u : 0x3C003C00u;
  const uint4 one8 = {one2, one2, one2, one2};
  const int32_t* table = a.table + (size_t)b * a.table_stride;

  Tile<D> tile;
  int step = st.first + wave;
  Pages pg{{-1, -1}};
  if (step < st.last) {
    pg = pages_of(a, table, step * kKeys);
    load_tile<D>(a, pg, head, step * kKeys, n, h, tile);
  }
  for (; step < st.last; step += kWaves) {
    const Tile<D> cur = tile;
    const Pages at = pg;
    const int key0 = step * kKeys;
    if (step + kWaves < st.last) {
      pg = pages_of(a, table, key0 + kKeys * kWaves);
      load_tile<D>(a, pg, head, key0 + kKeys * kWaves, n, h, tile);
    }
    // Scores.
    v4f acc[QT][2];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
#pragma unroll
      for (int t = 0; t < QT; ++t) acc[t][half] = {0, 0, 0, 0};
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const uint32_t w = cur.k[half][s];
        const uint4 kf = {code_pair<kBf16>(w, 0), code_pair<kBf16>(w, 1), code_pair<kBf16>(w, 2),
                          code_pair<kBf16>(w, 3)};
#pragma unroll
        for (int t = 0; t < QT; ++t) acc[t][half] = mfma16<kBf16>(kf, qf[t][s], acc[t][half]);
      }
    }
    // This lane's eight keys: score factors and value factors.
    float ks[8], km[8], vs[8], vm[8], s_max = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint4 kw4 = cur.kw[e / 4], vw4 = cur.vw[e / 4];
      const uint32_t kw = e % 4 == 0 ? kw4.x : e % 4 == 1 ? kw4.y : e % 4 == 2 ? kw4.z : kw4.w;
      const uint32_t vw = e % 4 == 0 ? vw4.x : e % 4 == 1 ? vw4.y : e % 4 == 2 ? vw4.z : vw4.w;
      const float s = widen<kBf16>(kw >> 16) * a.scale;
      ks[e] = s;
      km[e] = fmaf(-16.0f, s, widen<kBf16>(kw & 0xffffu) * a.scale);
      vs[e] = widen<kBf16>(vw >> 16);
      vm[e] = fmaf(8.0f, vs[e], widen<kBf16>(vw & 0xffffu));
    }
    const bool whole = key0 >= all_lo && key0 + kKeys <= all_hi && at.id[0] >= 0 && at.id[1] >= 0;
    float x[QT][8];
    bool raise = false;
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      float top = -kInf;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[t][e] = fmaf(ks[e], acc[t][e / 4][e % 4], km[e] * q_sum[t]);
        if (!whole) {
          const int key = key0 + 16 * (e / 4) + 4 * h + e % 4;
          if (key < seen[t].x || key >= seen[t].y || at.id[e / 4] < 0) x[t][e] = -kInf;
        }
        top = fmaxf(top, x[t][e]);
      }
      raise |= top > m[t];
    }
    if constexpr (!kBf16) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int key = key0 + 16 * (e / 4) + 4 * h + e % 4;
        if (whole || (key >= key_lo && key < key_hi && at.id[e / 4] >= 0)) s_max = fmaxf(s_max, vs[e]);
      }
      raise |= s_max > s_top;
    }
    if (__any(raise)) {
      float ratio = 1.0f;
      if constexpr (!kBf16) {
        // The least power of two that no scale so far passes; s_top stays 0 while all are 0.
        float s = s_max;
#pragma unroll
        for (int x2 = 32; x2 >= 1; x2 >>= 1) s = fmaxf(s, __shfl_xor(s, x2));
        if (s > s_top) {
          const float up = __uint_as_float((__float_as_uint(s) + 0x7fffffu) & 0x7f800000u);
          ratio = s_top / up;
          s_top = up;
          s_factor = 16384.0f / up;
        }
      }
#pragma unroll
      for (int t = 0; t < QT; ++t) {
        float top = x[t][0];
#pragma unroll
        for (int e = 1; e < 8; ++e) top = fmaxf(top, x[t][e]);
        const float up = fmaxf(m[t], quarter_max(top));
        const float at0 = up == -kInf ? 0.0f : up;
        const float alpha = __builtin_amdgcn_exp2f(m[t] - at0);
        m[t] = up;
        base[t] = at0;
        l[t] *= alpha;
        mid[t] *= alpha;
        const float both = alpha * ratio;
#pragma unroll
        for (int d = 0; d < kDimTiles; ++d) o[t][d] *= both;
        ones[t] *= both;
      }
    }
    // Probabilities, and the operand p s in 16 bits (f16: relative to s_top, times 2^14; one
    // rounding, of a weight of u - 8).
    uint4 pf[QT];
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      float ps[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float p = __builtin_amdgcn_exp2f(x[t][e] - base[t]);
        const bool off = !whole && x[t][e] == -kInf;  // its words may hold anything
        l[t] += p;
        mid[t] += off ? 0.0f : p * vm[e];
        ps[e] = off ? 0.0f : p * (kBf16 ? vs[e] : vs[e] * s_factor);
      }
      pf[t] = {narrow2<kBf16>(ps[0], ps[1]), narrow2<kBf16>(ps[2], ps[3]),
               narrow2<kBf16>(ps[4], ps[5]), narrow2<kBf16>(ps[6], ps[7])};
      ones[t] = mfma16<kBf16>(one8, pf[t], ones[t]);
    }
    // O^T: dim tile d holds channel D/16 n + d in row n; keys pair up across words.
    uint32_t lo[4], hi[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      lo[i] = (cur.v[2 * i] & 0xffffu) | (cur.v[2 * i + 1] << 16);
      hi[i] = (cur.v[2 * i] >> 16) | (cur.v[2 * i + 1] & 0xffff0000u);
    }
#pragma unroll
    for (int d = 0; d < kDimTiles; ++d) {
      const uint32_t* w = d < 4 ? lo : hi;
      const uint4 vf = {code_pair<kBf16>(w[0], d & 3), code_pair<kBf16>(w[1], d & 3),
                        code_pair<kBf16>(w[2], d & 3), code_pair<kBf16>(w[3], d & 3)};
#pragma unroll
      for (int t = 0; t < QT; ++t) o[t][d] = mfma16<kBf16>(vf, pf[t], o[t][d]);
    }
  }

  // Join the four waves: per 16-row tile, every wave's sums relative to the common maximum.
  __shared__ float lds_o[kWaves][16][D + 4];
  __shared__ float2 lds_ml[kWaves][16];
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const float lsum = quarter_sum(l[t]), msum = quarter_sum(mid[t]);
    const float unit = kBf16 ? 1.0f : s_top * (1.0f / 16384.0f);
    if (t) __syncthreads();
    if (h == 0) lds_ml[wave][n] = {m[t], lsum};
    // Row i of dim tile d: channel (D/16) (4h + i) + d.
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int d = 0; d < kDimTiles; d += 4) {
        float4 f;
        f.x = fmaf(unit, fmaf(-24.0f, ones[t][i], o[t][d][i]), msum);
        f.y = fmaf(unit, fmaf(-24.0f, ones[t][i], o[t][d + 1][i]), msum);
        f.z = fmaf(unit, fmaf(-24.0f, ones[t][i], o[t][d + 2][i]), msum);
        f.w = fmaf(unit, fmaf(-24.0f, ones[t][i], o[t][d + 3][i]), msum);
        *reinterpret_cast<float4*>(&lds_o[wave][n][kDimTiles * (4 * h + i) + d]) = f;
      }
    __syncthreads();
    // 16 threads a row, D/16 channels each.
    const int r = threadIdx.x >> 4, c = (threadIdx.x & 15) * (D / 16);
    const int row = row0 + 16 * t + r;
    if (row < rows) {
      float2 ml[kWaves];
      float top = -kInf;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        ml[w] = lds_ml[w][r];
        top = fmaxf(top, ml[w].x);
      }
      const float at0 = top == -kInf ? 0.0f : top;
      float total = 0.0f, sum[D / 16];
#pragma unroll
      for (int d = 0; d < D / 16; ++d) sum[d] = 0.0f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float f = __builtin_amdgcn_exp2f(ml[w].x - at0);
        total = fmaf(f, ml[w].y, total);
#pragma unroll
        for (int d = 0; d < D / 16; ++d) sum[d] = fmaf(f, lds_o[w][r][c + d], sum[d]);
      }
      const int token = row / (int)a.group, g = row - token * (int)a.group;
      const size_t q_row = (size_t)(seq.start + token);
      const uint32_t q_head = head * a.group + g;
      if (a.parts > 1) {
        const size_t at = ((size_t)part * a.q_rows + q_row) * heads + q_head;
#pragma unroll
        for (int d = 0; d < D / 16; ++d) a.part_o[at * D + c + d] = sum[d];
        if (c == 0) a.part_ml[at] = {top, total};
      } else {
        const bool none = total == 0.0f;  // a NaN among the scores leaves total NaN
        const float inv = none ? 0.0f : 1.0f / total;
        uint16_t* out = static_cast<uint16_t*>(a.out) + q_row * a.out_stride + q_head * D + c;
#pragma unroll
        for (int d = 0; d < D / 16; d += 2)
          *reinterpret_cast<uint32_t*>(out + d) = narrow2<kBf16>(sum[d] * inv, sum[d + 1] * inv);
        if (a.lse && c == 0)
          a.lse[q_row * heads + q_head] = none ? -kInf : (top + __log2f(total)) * kLn2;
      }
    }
  }
}

// Many rows: eight waves of 32 rows share tiles of 64 keys in LDS, unpacked once for all of them:
// K as 16 + u, V as m + s u rounded to the element type (the one rounding beside p's). S^T = K Q^T and
// O^T = V^T P^T on 32 x 32 x 16. LDS row m of 32 K rows holds key swap23(m), so the score registers
// of a lane (one row of q, half = lane / 32) are keys 8 half + 0..7 and 16 + 8 half + 0..7: the B
// operands of the PV product's two steps, as they are. V stays token-major and its operand comes
// through the transposed LDS read.
constexpr int kRowsThreads = 512;
constexpr int kTileKeys = 64;
constexpr float kPTop = 32768.0f;  // a lane's probabilities of 32 keys sum to no more, or m is raised
constexpr float kPLog = 7.0f;      // the largest score gives p = 2^7: f16 stays normal to 2^-21 of it

typedef short v4s __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4s lds_v4s;

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

template <int D>
struct RowsLds {
  uint8_t k[2][kTileKeys * D * 2];
  uint8_t v[2][kTileKeys * D * 2];
  float ks[2][kTileKeys], km[2][kTileKeys];  // times the scale: s, and m - 16 s
  uint8_t live[2][8];                        // a bit per key: its page is one
};

// A thread's share of a tile on the way to LDS: key tid / 8, channels D/8 (tid % 8) and on.
template <int D>
struct Staged {
  uint32_t k[D / 64], v[D / 64];
  uint32_t kw, vw;
  int page;
};

template <int D>
__device__ __forceinline__ void fetch(const Args& a, uint32_t head, int key, int page, Staged<D>& s) {
  const uint32_t page_tokens = 1u << a.page_shift, in_page = (uint32_t)key & (page_tokens - 1);
  const uint8_t* block = a.cache + ((uint64_t)max(page, 0) * a.kv_heads + head) *
                                       ((uint64_t)page_tokens * (D + 8));
  const uint8_t* kc = block + in_page * (D / 2) + (threadIdx.x & 7) * (D / 16);
  const uint8_t* kw = block + page_tokens * D + in_page * 4;
#pragma unroll
  for (int i = 0; i < D / 64; ++i) {
    s.k[i] = reinterpret_cast<const uint32_t*>(kc)[i];
    s.v[i] = reinterpret_cast<const uint32_t*>(kc + page_tokens * (D / 2))[i];
  }
  s.kw = *reinterpret_cast<const uint32_t*>(kw);
  s.vw = *reinterpret_cast<const uint32_t*>(kw + page_tokens * 4);
  s.page = page;
}

__device__ __forceinline__ int page_of(const Args& a, const int32_t* table, int key) {
  const uint32_t col = (uint32_t)key >> a.page_shift;
  const int id = col < a.table_stride ? table[col] : -1;
  return (uint32_t)id < a.pages ? id : -1;
}

// A pair of values m + s u, u as 16 + u in `code`, in the element type. f16: (u - 8) s + (m + 8 s) in
// packed f16, exact but for the midpoint's rounding and the result's.
template <bool kBf16>
__device__ __forceinline__ uint32_t value_pair(uint32_t code, float s, float m16, uint32_t s2,
                                               uint32_t mid2) {
  if constexpr (kBf16)
    return narrow2<true>(fmaf(__uint_as_float(code << 16), s, m16),
                         fmaf(__uint_as_float(code & 0xffff0000u), s, m16));
  const v2h u = __builtin_bit_cast(v2h, code) - v2h{(_Float16)24.0f, (_Float16)24.0f};
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(u, __builtin_bit_cast(v2h, s2),
                                                                __builtin_bit_cast(v2h, mid2)));
}

// Chunk (16 bytes) swizzles of the LDS rows of 2 D bytes, which spread the rows that one read takes
// over the banks.
template <int D>
__device__ __forceinline__ uint32_t v_swizzle(uint32_t key) {
  return (D == 128 ? 4 : 2) * (key & 3);
}

template <int D, bool kBf16>
__device__ __forceinline__ void unpack(const Args& a, RowsLds<D>& lds, int buf, int key0, int key_lo,
                                       int key_hi, const Staged<D>& s) {
  const uint32_t at = threadIdx.x >> 3, part = threadIdx.x & 7;
  const uint32_t m = (at & 32) + swap23(at & 31);
  const int key = key0 + (int)at;
  constexpr uint32_t kNan = kBf16 ? 0x7f80u : 0x7c00u;
  const bool live = s.page >= 0;
  const bool seen = live && key >= key_lo && key < key_hi;
  // A key whose V words hold a NaN gives NaN through its score, where only the rows that see it
  // look; its V rows, and those of keys that no row sees, are zeros.
  const bool nan = (s.vw & 0x7fffu) >= kNan || ((s.vw >> 16) & 0x7fffu) >= kNan;
  const bool keep = seen && !nan;
  const float vs = keep ? widen<kBf16>(s.vw >> 16) : 0.0f;
  const float vm = keep ? widen<kBf16>(s.vw & 0xffffu) : 0.0f;
  const float m16 = fmaf(-16.0f, vs, vm);
  const uint32_t s2 = narrow2<kBf16>(vs, vs), mid = narrow<kBf16>(fmaf(8.0f, vs, vm));
  const uint32_t mid2 = mid | (mid << 16);
#pragma unroll
  for (int i = 0; i < D / 64; ++i) {
    const uint32_t chunk = part * (D / 64) + i;
    uint4 x;
    x.x = code_pair<kBf16>(s.k[i], 0), x.y = code_pair<kBf16>(s.k[i], 1);
    x.z = code_pair<kBf16>(s.k[i], 2), x.w = code_pair<kBf16>(s.k[i], 3);
    *reinterpret_cast<uint4*>(&lds.k[buf][m * (2 * D) + 16 * (chunk ^ (m & (D / 8 - 1)))]) = x;
    x.x = value_pair<kBf16>(code_pair<kBf16>(s.v[i], 0), vs, m16, s2, mid2);
    x.y = value_pair<kBf16>(code_pair<kBf16>(s.v[i], 1), vs, m16, s2, mid2);
    x.z = value_pair<kBf16>(code_pair<kBf16>(s.v[i], 2), vs, m16, s2, mid2);
    x.w = value_pair<kBf16>(code_pair<kBf16>(s.v[i], 3), vs, m16, s2, mid2);
    *reinterpret_cast<uint4*>(&lds.v[buf][at * (2 * D) + 16 * (chunk ^ v_swizzle<D>(at))]) = x;
  }
  if (part == 0) {
    const float ks = widen<kBf16>(s.kw >> 16) * a.scale;
    const float km = fmaf(-16.0f, ks, widen<kBf16>(s.kw & 0xffffu) * a.scale);
    lds.ks[buf][at] = ks;
    lds.km[buf][at] = seen && nan ? __uint_as_float(0x7fc00000u) : km;
  }
  const uint64_t bits = __ballot(live && part == 0);  // key 8 w + i of wave w at bit 8 i
  if ((threadIdx.x & 63) == 0) {
    uint32_t byte = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) byte |= (uint32_t)((bits >> (8 * i)) & 1) << i;
    lds.live[buf][threadIdx.x >> 6] = (uint8_t)byte;
  }
}

// The 16 scores of a lane in a 32-key block, less m (base 2): acc times the keys' factors (lane r of
// 16 holds register r's) plus c.
template <int R = 0>
__device__ __forceinline__ void scores(float ks, const v16f& acc, const v16f& c, float (&y)[16]) {
  if constexpr (R < 16) {
    y[R] = spread<R>(ks) * acc[R] + c[R];
    scores<R + 1>(ks, acc, c, y);
  }
}

template <int D, bool kBf16>
__global__ __launch_bounds__(kRowsThreads, 2) void k_attention_kv4_rows(Args a) {
  constexpr int kRows = 256, kSteps = D / 16, kBlocks = D / 32;
  __shared__ __attribute__((aligned(16))) RowsLds<D> lds;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 31, half = lane >> 5;
  const uint32_t head = blockIdx.x, b = blockIdx.z;
  const uint32_t part = blockIdx.y % a.parts;
  const Sequence seq = sequence(a, b);
  const int rows = seq.rows * (int)a.group;
  // The last rows see the most keys: they start first.
  const int row0 = (int)(a.row_tiles - 1 - blockIdx.y / a.parts) * kRows;
  if (row0 >= rows || !takes(a, rows)) return;
  const int group = (int)a.group;
  const int2 first_span = span(a, seq, row0 / group);
  const int2 last_span = span(a, seq, (min(row0 + kRows, rows) - 1) / group);
  const int key_lo = first_span.x, key_hi = last_span.y;
  const Steps st = steps(key_lo, key_hi, a.parts, part, kTileKeys);
  const uint32_t heads = a.kv_heads * a.group;

  // The wave's rows, and the keys that some and that all of them see.
  const int wave_row0 = row0 + 32 * wave, row = wave_row0 + n;
  const bool active = wave_row0 < rows;
  const int2 wave_first = span(a, seq, min(wave_row0, rows - 1) / group);
  const int2 wave_last = span(a, seq, min(wave_row0 + 31, rows - 1) / group);
  const int token = row / group, g = row - token * group;
  const int2 seen = row < rows ? span(a, seq, token) : int2{0, 0};

  // Q^T operands: channels 8 (2 s + half) + {0,4,1,5,2,6,3,7}, the order of the codes' pairs.
  uint4 qf[kSteps];
  float sum = 0.0f;
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    uint4 x = {0, 0, 0, 0};
    if (row < rows)
      x = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.q) +
                                          (size_t)(seq.start + token) * a.q_stride +
                                          (head * a.group + g) * D + 8 * (2 * s + half));
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) sum += widen<kBf16>(w[i] & 0xffffu) + widen<kBf16>(w[i] >> 16);
    qf[s] = {(x.x & 0xffffu) | (x.z << 16), (x.x >> 16) | (x.z & 0xffff0000u),
             (x.y & 0xffffu) | (x.w << 16), (x.y >> 16) | (x.w & 0xffff0000u)};
  }
  const float q_sum = sum + __shfl_xor(sum, 32);

  v16f o[kBlocks];
#pragma unroll
  for (int d = 0; d < kBlocks; ++d) o[d] = v16f{};
  float m = -kInf, l = 0.0f;  // m: what exponents are relative to, the largest score less kPLog
  const int32_t* table = a.table + (size_t)b * a.table_stride;
  const int at = (int)(threadIdx.x >> 3);

  Staged<D> staged;
  int page = -1;
  if (st.first < st.last) {
    fetch<D>(a, head, st.first * kTileKeys + at, page_of(a, table, st.first * kTileKeys + at), staged);
    unpack<D, kBf16>(a, lds, 0, st.first * kTileKeys, key_lo, key_hi, staged);
    if (st.first + 1 < st.last) {
      const int key = (st.first + 1) * kTileKeys + at;
      fetch<D>(a, head, key, page_of(a, table, key), staged);
      page = page_of(a, table, key + kTileKeys);
    }
    __syncthreads();
  }
  for (int step = st.first; step < st.last; ++step) {
    const int buf = (step - st.first) & 1, key0 = step * kTileKeys;
    if (step + 1 < st.last) {
      unpack<D, kBf16>(a, lds, buf ^ 1, key0 + kTileKeys, key_lo, key_hi, staged);
      if (step + 2 < st.last) {
        const int key = key0 + 2 * kTileKeys + at;
        fetch<D>(a, head, key, page, staged);
        page = page_of(a, table, key + kTileKeys);
      }
    }
    if (active && key0 < wave_last.y && key0 + kTileKeys > wave_first.x) {
      const uint64_t live = *reinterpret_cast<const uint64_t*>(lds.live[buf]);
      const bool whole = key0 >= wave_last.x && key0 + kTileKeys <= wave_first.y && live == ~0ull;
#pragma unroll
      for (int blk = 0; blk < 2; ++blk) {
        const float ks = lds.ks[buf][32 * blk + (lane & 7) + 8 * half + 2 * (lane & 8)];
        const float km = half ? -1.0f : lds.km[buf][32 * blk + swap23(n)];
        // c = (m - 16 s) sum(q) - m of the row, in f32 on the matrix unit.
        const v16f c = __builtin_amdgcn_mfma_f32_32x32x2f32(km, half ? m : q_sum, v16f{}, 0, 0, 0);
        v16f acc = v16f{};
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
          const uint4 kf = *reinterpret_cast<const uint4*>(
              &lds.k[buf][(32 * blk + n) * (2 * D) + 16 * ((2 * s + half) ^ (n & (D / 8 - 1)))]);
          acc = mfma32<kBf16>(kf, qf[s], acc);
        }
        float y[16], ts = 0.0f;
        scores(ks, acc, c, y);
        if (!whole) {
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int k = 32 * blk + 8 * half + (r & 7) + 2 * (r & 8);
            if (key0 + k < seen.x || key0 + k >= seen.y || !((live >> k) & 1)) y[r] = -kInf;
          }
        }
        float p[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          p[r] = __builtin_amdgcn_exp2f(y[r]);
          ts += p[r];
        }
        if (__any(!(ts <= kPTop))) {
          // The first keys, or scores far past m: the block's maximum, and everything relative to it.
          float top = -kInf;
          const v16f c0 =
              __builtin_amdgcn_mfma_f32_32x32x2f32(km, half ? 0.0f : q_sum, v16f{}, 0, 0, 0);
          float x[16];
          scores(ks, acc, c0, x);
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            if (!whole && y[r] == -kInf) x[r] = -kInf;
            top = fmaxf(top, x[r]);
          }
          top = fmaxf(top, __shfl_xor(top, 32)) - kPLog;
          const float up = fmaxf(m, top), base = up == -kInf ? 0.0f : up;
          const float alpha = __builtin_amdgcn_exp2f(m - base);
          m = up;
          l *= alpha;
#pragma unroll
          for (int d = 0; d < kBlocks; ++d) o[d] *= alpha;
          ts = 0.0f;
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            p[r] = __builtin_amdgcn_exp2f(x[r] - base);
            ts += p[r];
          }
        }
        l += ts;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const uint4 pf = {narrow2<kBf16>(p[8 * s], p[8 * s + 1]),
                            narrow2<kBf16>(p[8 * s + 2], p[8 * s + 3]),
                            narrow2<kBf16>(p[8 * s + 4], p[8 * s + 5]),
                            narrow2<kBf16>(p[8 * s + 6], p[8 * s + 7])};
          // V^T operand: row 32 d + n, keys 8 half + 0..7 of the step. Lane j of 16 points at key j / 4,
          // channels 4 (j % 4) and on, and receives channel j of four keys.
          const int j = lane & 15, quad = lane >> 4;
          const int key = 32 * blk + 16 * s + 8 * (quad >> 1) + (j >> 2);
#pragma unroll
          for (int d = 0; d < kBlocks; ++d) {
            const uint32_t chunk = 4 * d + 2 * (quad & 1) + ((j & 3) >> 1);
            const uint8_t* v =
                &lds.v[buf][key * (2 * D) + 16 * (chunk ^ v_swizzle<D>(j >> 2)) + 8 * (j & 1)];
            const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)v);
            const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(v + 4 * 2 * D));
            const uint2 l2 = __builtin_bit_cast(uint2, lo), h2 = __builtin_bit_cast(uint2, hi);
            o[d] = mfma32<kBf16>(uint4{l2.x, l2.y, h2.x, h2.y}, pf, o[d]);
          }
        }
      }
    }
    __syncthreads();
  }

  // Register 4 i + b of block d holds channel 32 d + 8 i + 2 half + {0, 4, 1, 5}[b] of the lane's row.
  if (!active) return;
  const float total = l + __shfl_xor(l, 32);
  const bool none = total == 0.0f;
  const size_t q_row = (size_t)(seq.start + token);
  const uint32_t q_head = head * a.group + g;
  if (a.parts > 1) {
    if (row < rows) {
      const size_t place = ((size_t)part * a.q_rows + q_row) * heads + q_head;
#pragma unroll
      for (int d = 0; d < kBlocks; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float* to = a.part_o + place * D + 32 * d + 8 * i + 2 * half;
          *reinterpret_cast<float2*>(to) = {o[d][4 * i], o[d][4 * i + 2]};
          *reinterpret_cast<float2*>(to + 4) = {o[d][4 * i + 1], o[d][4 * i + 3]};
        }
      if (half == 0) a.part_ml[place] = {m, total};
    }
    return;
  }
  const float inv = none ? 0.0f : 1.0f / total;
  // Through LDS (each wave its own 32 rows; the tiles are done) so that whole rows leave together.
  uint8_t* rows_lds = &lds.k[0][0] + wave * 32 * 2 * D;
  static_assert(sizeof(lds.k) + sizeof(lds.v) >= 8 * 32 * 2 * D, "the tiles hold the rows");
#pragma unroll
  for (int d = 0; d < kBlocks; ++d)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint8_t* to = rows_lds + n * (2 * D) + 16 * ((4 * d + i) ^ (n & (D / 8 - 1))) + 4 * half;
      *reinterpret_cast<uint32_t*>(to) = narrow2<kBf16>(o[d][4 * i] * inv, o[d][4 * i + 2] * inv);
      *reinterpret_cast<uint32_t*>(to + 8) =
          narrow2<kBf16>(o[d][4 * i + 1] * inv, o[d][4 * i + 3] * inv);
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

// Joins the parts of a row: one wave per (row, query head), D/64 channels a lane.
template <int D, bool kBf16>
__global__ __launch_bounds__(kThreads) void k_attention_kv4_join(Args a) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t heads = a.kv_heads * a.group;
  const Sequence seq = sequence(a, blockIdx.z);
  const uint32_t row = blockIdx.x * kWaves + wave;
  const uint32_t token = row / a.group, g = row - token * a.group;
  if ((int)token >= seq.rows || !takes(a, seq.rows * (int)a.group)) return;
  const size_t q_row = (size_t)(seq.start + token);
  const uint32_t q_head = blockIdx.y * a.group + g;
  float top = -kInf;
  for (uint32_t p = 0; p < a.parts; ++p)
    top = fmaxf(top, a.part_ml[((size_t)p * a.q_rows + q_row) * heads + q_head].x);
  const float at0 = top == -kInf ? 0.0f : top;
  float total = 0.0f, sum[D / 64];
#pragma unroll
  for (int d = 0; d < D / 64; ++d) sum[d] = 0.0f;
  for (uint32_t p = 0; p < a.parts; ++p) {
    const size_t at = ((size_t)p * a.q_rows + q_row) * heads + q_head;
    const float2 ml = a.part_ml[at];
    const float f = __builtin_amdgcn_exp2f(ml.x - at0);
    total = fmaf(f, ml.y, total);
#pragma unroll
    for (int d = 0; d < D / 64; ++d) sum[d] = fmaf(f, a.part_o[at * D + lane * (D / 64) + d], sum[d]);
  }
  const bool none = total == 0.0f;
  const float inv = none ? 0.0f : 1.0f / total;
  uint16_t* out = static_cast<uint16_t*>(a.out) + q_row * a.out_stride + q_head * D + lane * (D / 64);
#pragma unroll
  for (int d = 0; d < D / 64; ++d) out[d] = (uint16_t)narrow<kBf16>(sum[d] * inv);
  if (a.lse && lane == 0)
    a.lse[q_row * heads + q_head] = none ? -kInf : (top + __log2f(total)) * kLn2;
}

// One launch over the sequences of `plan`'s row counts, and the join of its parts.
template <int D, bool kBf16>
hipError_t launch(Args a, uint32_t batch, const Kv4Launch& plan, hipStream_t stream) {
  if (plan.row_tiles == 0) return hipSuccess;
  a.parts = plan.parts;
  a.row_tiles = plan.row_tiles;
  a.rows_from = plan.rows_from;
  a.rows_to = plan.rows_to;
  a.part_ml = reinterpret_cast<float2*>(a.part_o + (size_t)plan.parts * a.q_rows * a.kv_heads *
                                                       a.group * D);
  const uint32_t tiles = plan.row_tiles * plan.parts;
  const dim3 few(tiles, a.kv_heads, batch);
  if (plan.tile_rows == 16)
    hipLaunchKernelGGL((k_attention_kv4_few<D, kBf16, 1>), few, dim3(kThreads), 0, stream, a);
  else if (plan.tile_rows == 32)
    hipLaunchKernelGGL((k_attention_kv4_few<D, kBf16, 2>), few, dim3(kThreads), 0, stream, a);
  else
    hipLaunchKernelGGL((k_attention_kv4_rows<D, kBf16>), dim3(a.kv_heads, tiles, batch),
                       dim3(kRowsThreads), 0, stream, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || plan.parts == 1) return e;
  const uint32_t rows = std::min(a.max_q * a.group, plan.rows_to);
  const dim3 join((rows + kWaves - 1) / kWaves, a.kv_heads, batch);
  hipLaunchKernelGGL((k_attention_kv4_join<D, kBf16>), join, dim3(kThreads), 0, stream, a);
  return hipGetLastError();
}

template <int D, bool kBf16>
hipError_t launch_both(const Args& a, uint32_t batch, const Kv4Plan& plan, hipStream_t stream) {
  const hipError_t e = launch<D, kBf16>(a, batch, plan.many, stream);
  return e != hipSuccess ? e : launch<D, kBf16>(a, batch, plan.few, stream);
}

constexpr uint32_t kFewRows = 32;  // what k_attention_kv4_few holds

}  // namespace

// Sequences of up to kFewRows rows are k_attention_kv4_few's, the others k_attention_kv4_rows', a call
// with both kinds one launch of each (the host knows no sequence's rows, only that none has more than
// max_q; the workgroups of the other kind leave at once). The keys of a row tile are divided while the
// chip has room for more workgroups and a part keeps 512 keys.
Kv4Plan kv4_plan(const h3_kv4_cfg& cfg, const h3_kv4_attention_cfg& acfg, uint32_t batch,
                 uint32_t max_q, uint32_t cus) {
  Kv4Plan p{};
  const uint32_t group = acfg.heads / cfg.kv_heads, rows = max_q * group;
  const uint64_t most = ((uint64_t)acfg.table_stride * cfg.page_tokens + 511) / 512;
  auto parts = [&](uint32_t row_tiles, uint32_t resident) {
    const uint64_t groups = (uint64_t)batch * cfg.kv_heads * row_tiles;
    const uint64_t room = ((uint64_t)resident * cus + groups - 1) / groups;
    return (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>({room, most, 128}));
  };
  if (rows > kFewRows) {
    p.many = {256, (rows + 255) / 256, 1, kFewRows + 1, rows};
    p.many.parts = parts(p.many.row_tiles, 1);
  }
  if (rows <= kFewRows || batch > 1) {
    const uint32_t few = std::min(rows, kFewRows);
    p.few = {few <= 16 ? 16u : 32u, 1, 1, 0, few};
    p.few.parts = parts(1, 4);
  }
  return p;
}

size_t kv4_workspace_bytes(const h3_kv4_cfg& cfg, const h3_kv4_attention_cfg& acfg, uint32_t q_rows,
                           const Kv4Plan& plan) {
  const uint32_t parts = std::max(plan.many.parts, plan.few.parts);
  if (parts <= 1) return 0;
  return (size_t)parts * q_rows * acfg.heads * (cfg.head_dim + 2) * 4;
}

hipError_t launch_attention_kv4(const h3_kv4_cfg& cfg, const h3_kv4_attention_cfg& acfg,
                                uint32_t batch, uint32_t q_rows, uint32_t max_q, const void* q,
                                const void* cache, const int32_t* table, const int32_t* lengths,
                                const int32_t* q_starts, void* out, float* lse, void* workspace,
                                hipStream_t stream) {
  Kv4Plan plan = kv4_plan(cfg, acfg, batch, max_q, device_cus());
  if (!workspace) plan.many.parts = plan.few.parts = 1;
  Args a{};
  a.q = q;
  a.cache = static_cast<const uint8_t*>(cache);
  a.table = table;
  a.lengths = lengths;
  a.q_starts = q_starts;
  a.out = out;
  a.lse = lse;
  a.part_o = static_cast<float*>(workspace);
  a.kv_heads = cfg.kv_heads;
  a.group = acfg.heads / cfg.kv_heads;
  a.q_stride = acfg.q_stride;
  a.out_stride = acfg.out_stride;
  a.table_stride = acfg.table_stride;
  a.pages = cfg.pages;
  a.page_shift = __builtin_ctz(cfg.page_tokens);
  a.q_rows = q_rows;
  a.max_q = max_q;
  a.causal = acfg.causal;
  a.window = acfg.window;
  a.scale = acfg.scale * kLog2e;
  const bool bf16 = cfg.elem == H3_ELEM_BF16;
  if (cfg.head_dim == 128)
    return bf16 ? launch_both<128, true>(a, batch, plan, stream)
                : launch_both<128, false>(a, batch, plan, stream);
  return bf16 ? launch_both<64, true>(a, batch, plan, stream)
              : launch_both<64, false>(a, batch, plan, stream);
}

}  // namespace h3
