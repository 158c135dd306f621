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
  if (row0 >= rows) return;
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

// Joins the parts of a row: one wave per (row, query head), D/64 channels a lane.
template <int D, bool kBf16>
__global__ __launch_bounds__(kThreads) void k_attention_kv4_join(Args a) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t heads = a.kv_heads * a.group;
  const Sequence seq = sequence(a, blockIdx.z);
  const uint32_t row = blockIdx.x * kWaves + wave;
  const uint32_t token = row / a.group, g = row - token * a.group;
  if ((int)token >= seq.rows) return;
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

template <int D, bool kBf16>
hipError_t launch(Args a, uint32_t batch, const Kv4Plan& plan, hipStream_t stream) {
  a.parts = plan.parts;
  const dim3 grid(plan.row_tiles * plan.parts, a.kv_heads, batch);
  if (plan.tile_rows == 16)
    hipLaunchKernelGGL((k_attention_kv4_few<D, kBf16, 1>), grid, dim3(kThreads), 0, stream, a);
  else if (plan.tile_rows == 32)
    hipLaunchKernelGGL((k_attention_kv4_few<D, kBf16, 2>), grid, dim3(kThreads), 0, stream, a);
  else
    hipLaunchKernelGGL((k_attention_kv4_few<D, kBf16, 4>), grid, dim3(kThreads), 0, stream, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || plan.parts == 1) return e;
  const dim3 join((a.max_q * a.group + kWaves - 1) / kWaves, a.kv_heads, batch);
  hipLaunchKernelGGL((k_attention_kv4_join<D, kBf16>), join, dim3(kThreads), 0, stream, a);
  return hipGetLastError();
}

}  // namespace

// Row tiles of 16, 32 or 64 rows, and the keys of a tile in parts while the chip has room for four
// workgroups a compute unit and a part keeps 512 keys.
Kv4Plan kv4_plan(const h3_kv4_cfg& cfg, const h3_kv4_attention_cfg& acfg, uint32_t batch,
                 uint32_t max_q, uint32_t cus) {
  Kv4Plan p;
  const uint64_t rows = (uint64_t)max_q * (acfg.heads / cfg.kv_heads);
  p.tile_rows = rows <= 16 ? 16 : rows <= 32 ? 32 : 64;
  p.row_tiles = (uint32_t)((rows + p.tile_rows - 1) / p.tile_rows);
  const uint64_t keys = (uint64_t)acfg.table_stride * cfg.page_tokens;
  const uint64_t groups = (uint64_t)batch * cfg.kv_heads * p.row_tiles;
  const uint64_t room = (4ull * cus + groups - 1) / groups, most = (keys + 511) / 512;
  p.parts = (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>({room, most, 128}));
  return p;
}

size_t kv4_workspace_bytes(const h3_kv4_cfg& cfg, const h3_kv4_attention_cfg& acfg, uint32_t q_rows,
                           const Kv4Plan& plan) {
  if (plan.parts <= 1) return 0;
  return (size_t)plan.parts * q_rows * acfg.heads * (cfg.head_dim + 2) * 4;
}

hipError_t launch_attention_kv4(const h3_kv4_cfg& cfg, const h3_kv4_attention_cfg& acfg,
                                uint32_t batch, uint32_t q_rows, uint32_t max_q, const void* q,
                                const void* cache, const int32_t* table, const int32_t* lengths,
                                const int32_t* q_starts, void* out, float* lse, void* workspace,
                                hipStream_t stream) {
  Kv4Plan plan = kv4_plan(cfg, acfg, batch, max_q, device_cus());
  if (!workspace) plan.parts = 1;
  Args a;
  a.q = q;
  a.cache = static_cast<const uint8_t*>(cache);
  a.table = table;
  a.lengths = lengths;
  a.q_starts = q_starts;
  a.out = out;
  a.lse = lse;
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = reinterpret_cast<float2*>(a.part_o +
                                        (size_t)plan.parts * q_rows * acfg.heads * cfg.head_dim);
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
    return bf16 ? launch<128, true>(a, batch, plan, stream)
                : launch<128, false>(a, batch, plan, stream);
  return bf16 ? launch<64, true>(a, batch, plan, stream) : launch<64, false>(a, batch, plan, stream);
}

}  // namespace h3
