// Attention over pages of keys and values in 4 bits (fp4.h), for one head size (LS_HEAD_DIM, a multiple of 32).
//
// Query rows of request b are the packed rows offsets[b] .. offsets[b + 1] - 1; the last of them stands at position
// lengths[b] - 1.  A row at position p attends to the keys 0 .. p of its request, with a window w to p - w + 1 .. p:
//   out = sum_t e^(c q.k_t - m) v_t / sum_t e^(c q.k_t - m),   m = max_t c q.k_t.
// The g query heads of a key/value head are rows of one product: row r of a request is head r % g of its token r / g.
//
// A wave holds NT tiles of 16 query rows and walks the keys in tiles of 32.  It computes S^T = K Q^T and then
// O^T += V^T P^T, both on the matrix units (16x16x32, bfloat16 operands, sums in 32 bits): the scores of S^T lie in the
// registers of just the lane that has to bring them to the second product, so neither the keys and values nor the
// weights pass through LDS.  Codes become bfloat16 operands exactly, two an instruction with their scale.  The
// softmax keeps a reference instead of the maximum: a row's reference moves only when a score passes it by more than 8
// (powers of two: weights up to 256), so most tiles do not touch the sums; weights are held in 32 bits, added up as they
// are and rounded to bfloat16 for the product (half a step of 2^-8 each, as the queries' own type has it).
// The float32 path has queries and weights as three bfloat16 terms each (24 bits together): every product of a term with
// a key or value is exact, so the sums are those of 32-bit operands.
//
// Requests of at most 16 rows a head (decoded tokens): a workgroup's four waves take the key tiles of one split in turn
// and fold at the end through LDS.  Others (prompts): every wave has a block of rows of its own, and the four waves of a
// workgroup share the operands of tiles of 64 keys through LDS.  In both a request's keys are cut into splits by a rule of its
// own length (and rows) and of the heads alone; where there are several, they leave sums that a second launch folds.  So a
// row's result does not depend on what else is in the step.
//
// What bounds it: decoding, the bytes (17/32 a key element): 4 requests of 131,071 keys (32 heads over 8, 570 MB) are read in
// 105 us, 5.4 TB/s, and their splits folded in 7; 64 of 1 to 8,192 (367 MB) take 79 and 4.5, 64 of 4,608 each (321 MB) 64 to 67 in all.
// Some 6 vector instructions a key and lane column are two thirds of what that leaves room for.  Prompts, the vector unit next
// to the matrix units: a tile of 16 rows by 32 keys has 16 products of 16 cycles and some 60 vector instructions of 4, of them
// 8 exponentials of 16, and two waves a SIMD overlap them in part (6,660 rows of 32 heads behind up to 8,192 keys in pages of 16:
// 780 us, 870 TFLOP/s, where a large product of the library reaches 1,190).  Two groups of waves a barrier apart, one at the matrix and
// one at the vector units, were slower (885 us for 770: alone on its SIMD, a wave waits for its own results).  The float32 path
// is at the matrix units' rate there (4 times 2,048 rows behind 8,192 keys 2,450 us, 393 TFLOP/s of three products each); decoding,
// its three products and two waves a SIMD take 95 us for 64 requests of 4,608 keys and 152 for 4 of 131,071.

#include "fp4.h"
#include "fp4_attention_api.h"

#include <algorithm>
#include <type_traits>

#ifndef LS_HEAD_DIM
#error "LS_HEAD_DIM must be defined"
#endif

namespace ls {

constexpr int D = LS_HEAD_DIM;
static_assert(D % 32 == 0 && D >= 32 && D <= 256, "head sizes are multiples of 32 up to 256");

// A head is cut into sections of 128, 64 and 32 elements: section s has E(s) elements a lane column (16 columns).
constexpr int kSections = D / 128 + (D % 128 >= 64) + (D % 64 >= 32);
__host__ __device__ constexpr int section_elems(int s) { return s < D / 128 ? 8 : (s == D / 128 && D % 128 >= 64) ? 4 : 2; }
__host__ __device__ constexpr int section_dim(int s) {
  int at = 0;
  for (int i = 0; i < s; ++i) at += 16 * section_elems(i);
  return at;
}

constexpr int kTileKeys = 32;
constexpr int kSharedKeys = 64;  // where a workgroup shares the tiles
constexpr int kThreads = 256;
constexpr float kSlack = 8.f;  // how far a score may pass the reference, in powers of two
constexpr float kToLog2 = 1.4426950408889634f;
constexpr float kLargestBf16 = 3.38953139e38f;

template <typename T> constexpr int kTerms = std::is_same_v<T, float> ? 3 : 1;
// Row tiles a wave holds where every wave has rows of its own: what its registers allow (2 of 2,048 rows a head of 160 behind
// 4,096 keys: one tile 752 us, two 498; heads of 128 with three or four tiles spill or leave one wave a SIMD).
template <typename T> constexpr int kPromptTiles = std::is_same_v<T, float> ? 1 : (D <= 160 ? 2 : 1);

// Waves a SIMD of the prompt kernel.
template <typename T> constexpr int kPromptWaves = D <= 128 ? 2 : 1;

// Keys a split of a request of few rows covers, by how many keys its rows see and how many heads do so: some 512 workgroups
// a request at most, and no split too short to be worth its launch.  One split leaves out the second launch.  (32 heads over 8,
// shortest splits of 512 keys / of 512 up to 4,096 keys and 1,024 behind / of 512 and 2,048, us: 64 requests of 1 to 8,192 keys
// 65.6 / 62.8 / 62.1, 64 of 8,192 122 / 116 / 111, 128 of 1 to 16,384 264 / 238 / 226, 8 of 8,192 21.2 / 19.4 / 20.1, one of 8,192
// 10.6 / 12.6 / 18.3, one of 32,768 16.2 / 16.1 / 20.0: longer ones would gain 5 % where requests fill the card and lose a quarter
// to a half where they do not.  8 of 532, 16 heads: one split 7.4, two 9.7.)
constexpr int kOneSplit = 768, kDecodeGroups = 512;
__host__ __device__ inline int shortest_split(int span, int kv_heads) { return kv_heads < 4 ? 256 : span <= 4096 ? 512 : 1024; }
__host__ __device__ inline int decode_split(int span, int kv_heads) {
  if (span <= kOneSplit || kv_heads >= kDecodeGroups) return max(span, kOneSplit);
  const int even = (int)(((long)span * kv_heads + kDecodeGroups - 1) / kDecodeGroups);
  return max(shortest_split(span, kv_heads), (even + 127) / 128 * 128);
}
// The same for prompts, by how many workgroups its rows fill.  A split leaves 4 (D + 2) bytes a row, written and read again, and
// reads 17/16 D a key: with bfloat16 operands one is no shorter than four keys a row, so that many portions of a few tokens
// behind long contexts do not move more sums than keys, up to 1,024 keys, from where on the products take longer.  (32 heads over
// 8 of 128, all splits down to 256 keys / by rows: 64 requests of 33 tokens behind 8,192 keys 1,260 us and 1.1 GB for sums / 875
// and 0.6; 16 of 64 behind 4,096 229 / 119, 4 of 128 106 / 67; one of 33 behind 8,192 36 / 33, behind 1,000 21 / 28.)  The float32
// path has three products for one, so its sums weigh a third: 7 requests of up to 129 tokens of 12 heads over 4 of 64 with a
// window of 500 34 / 41 to 47.
constexpr int kPromptGroups = 512, kPromptShortest = 256, kPromptShortMost = 1024;
template <typename T> __host__ __device__ inline int shortest_prompt_split(int rows) {
  if (sizeof(T) == 4 || rows <= kPromptShortest / 4) return kPromptShortest;
  return rows >= kPromptShortMost / 4 ? kPromptShortMost : (4 * rows + 63) / 64 * 64;
}
__host__ __device__ inline int prompt_splits_wanted(int groups, int kv_heads) { return max(1, kPromptGroups / (max(1, groups) * kv_heads)); }
template <typename T> __host__ __device__ inline int prompt_split(int span, int groups, int kv_heads, int rows) {
  const int want = prompt_splits_wanted(groups, kv_heads);
  return max(shortest_prompt_split<T>(rows), ((span + want - 1) / want + 63) / 64 * 64);  // whole tiles of 64
}

// How a request of `rows` rows a head whose rows see `span` keys is cut: the same in the kernels and on the host.
constexpr int kFewRows = 16;  // rows a head up to which a request belongs to the decoding part
template <typename T> constexpr int kGroupRows = 64 * kPromptTiles<T>;  // rows of a prompt's workgroup
struct Cut {
  int groups, len, splits;  // workgroups of rows (0: few rows), keys a split, splits
};
template <typename T>
__host__ __device__ inline Cut cut_request(int rows, int span, int kv_heads) {
  Cut c;
  c.groups = rows <= kFewRows ? 0 : (rows + kGroupRows<T> - 1) / kGroupRows<T>;
  c.len = c.groups == 0 ? decode_split(span, kv_heads) : prompt_split<T>(span, c.groups, kv_heads, rows);
  c.splits = max(1, (span + c.len - 1) / c.len);
  return c;
}
// The first key that a row at `position` sees, and the first tile of the rows from there on.
__host__ __device__ inline int first_seen(int position, int window) { return window > 0 && position >= window ? position - window + 1 : 0; }
__host__ __device__ inline int first_tile(int position, int window) { return first_seen(position, window) & ~(kSharedKeys - 1); }

struct Fp4Args {
  const void* q;
  long ldq;
  void* out;
  long ldo;
  Fp4Pool pool;
  const int* table;
  int columns;
  const int* offsets;
  const int* lengths;
  int requests, rows;      // rows: of q and out
  int most, longest;       // what the launches are sized for: a request of more rows is left out, a length counts as no more
  int group;               // query heads a key/value head
  float factor;            // |scale| * log2(e)
  bool negative;           // the scale is: queries change their sign
  int window;
  float* part_acc;         // [entries][D]: the sums of a row's split (see split_entry)
  float* part_ml;          // [entries][2]: reference, sum of the weights
  long per_row, per_request, head_entries;  // room for entries that a row of q and a request have, and a head in all
};

// One request as all kernels see it.
struct Request {
  int first, tokens, rows, start, base, end;  // first packed row, rows, rows a head, first position, keys that are seen: base .. end - 1
  __device__ __forceinline__ Request(const Fp4Args& a, int b) {
    const int from = a.offsets[b], to = a.offsets[b + 1];
    const bool ok = from >= 0 && to >= from && to <= a.rows && to - from <= a.most;
    first = ok ? from : 0;
    tokens = ok ? to - from : 0;
    rows = tokens * a.group;
    const int room = (int)min((long)a.columns << a.pool.page_shift, (long)a.longest);  // (a few tiles on stay below 2^31)
    end = min(max(a.lengths[b], 0), room);
    start = end - tokens;
    base = first_tile(start, a.window);
  }
};

// Where the sums of a split of row r of a head lie, -1 where there is no room.  The entries of a request of n tokens lie between
// those of the requests before it and after it: `per_row` n + `per_request` are its own, which is never less than what it leaves.
__device__ __forceinline__ long split_entry(const Fp4Args& a, const Request& rq, int b, int head, int split, int r) {
  const long entry = (long)split * rq.rows + r;
  if (entry >= a.per_row * rq.tokens + a.per_request) return -1;
  return head * a.head_entries + a.per_row * rq.first + a.per_request * b + entry;
}

struct KeyTile {  // what a lane has of 32 keys and values, as they lie in the pages
  unsigned int k[2][D / 32];
  unsigned int v[2][kSections][4];
  unsigned int ks[2][kSections], vs[2][kSections];
  bool good[2];  // the block of four tokens of this lane's values has a page
};

__device__ __forceinline__ void load_words(unsigned int* to, const unsigned char* from, int n) {
  if (n == 4) {
    const auto w = *reinterpret_cast<const __attribute__((ext_vector_type(4))) unsigned int*>(from);
    to[0] = w[0]; to[1] = w[1]; to[2] = w[2]; to[3] = w[3];
  } else if (n == 2) {
    const auto w = *reinterpret_cast<const __attribute__((ext_vector_type(2))) unsigned int*>(from);
    to[0] = w[0]; to[1] = w[1];
  } else {
    to[0] = *reinterpret_cast<const unsigned int*>(from);
  }
}

struct PageIds {
  int k[2], v[2];
};

__device__ __forceinline__ PageIds load_ids(const Fp4Args& a, const int* __restrict__ row, int t0, int lane) {
  PageIds ids;
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const int k_at = (t0 + 16 * s + (lane & 15)) >> a.pool.page_shift, v_at = (t0 + 16 * s + 4 * (lane >> 4)) >> a.pool.page_shift;
    ids.k[s] = row[min(k_at, a.columns - 1)];
    ids.v[s] = row[min(v_at, a.columns - 1)];
  }
  return ids;
}

__device__ __forceinline__ void load_tile(KeyTile& tile, const Fp4Args& a, const PageIds& ids, int head, int t0, int lane) {
  const int n = lane & 15, j = lane >> 4, mask = (1 << a.pool.page_shift) - 1;
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const bool k_ok = ids.k[s] >= 0 && ids.k[s] < a.pool.pages, v_ok = ids.v[s] >= 0 && ids.v[s] < a.pool.pages;
    const long k_row = (((long)(k_ok ? ids.k[s] : 0) * a.pool.kv_heads + head) << a.pool.page_shift) + ((t0 + 16 * s + n) & mask);
    const long v_blk = ((((long)(v_ok ? ids.v[s] : 0) * a.pool.kv_heads + head) << a.pool.page_shift) + ((t0 + 16 * s + 4 * j) & mask)) >> 2;
    tile.good[s] = v_ok;
    const unsigned char* kc = a.pool.k_codes + k_row * (D / 2);
    const unsigned char* ks = a.pool.k_scales + k_row * (D / 32);
    const unsigned char* vc = a.pool.v_codes + v_blk * (2 * D);
    const unsigned char* vs = a.pool.v_scales + v_blk * (D / 8);
#pragma unroll
    for (int c = 0; c < kSections; ++c) {
      const int e = section_elems(c), dim = section_dim(c);
      load_words(&tile.k[s][dim / 32], kc + dim / 2 + j * 2 * e, e / 2);
      tile.ks[s][c] = ks[(dim + j * 4 * e) / 32];
      load_words(tile.v[s][c], vc + (dim + n * e) / 8 * 16, 4);
      load_words(&tile.vs[s][c], vs + (dim + n * e) / 32 * 4, 1);
    }
  }
}

template <typename T> __device__ __forceinline__ float weight_exp2(float x);
template <> __device__ __forceinline__ float weight_exp2<float>(float x) { return exp2f(x); }
template <> __device__ __forceinline__ float weight_exp2<bf16_t>(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ bf16x8 as_operand(unsigned int a, unsigned int b, unsigned int c, unsigned int d) {
  typedef __attribute__((ext_vector_type(4))) unsigned int u32x4;
  return __builtin_bit_cast(bf16x8, u32x4{a, b, c, d});
}

// The rows of a wave: NT tiles of 16, a lane has column lane % 16 of each.
template <typename T, int NT>
struct Rows {
  bf16x8 q[kTerms<T>][NT][D / 32];
  f32x4 acc[NT][D / 16];
  float m[NT], l[NT];
  int last[NT], low[NT];       // the keys low .. last are seen by the lane's row (last < low: none)
  int any_last, all_last;      // uniform: the largest and the smallest `last` of the rows there are
  int any_low, all_low;        // the smallest and the largest `low`

  __device__ __forceinline__ void init(const Fp4Args& a, const Request& rq, int head, int row0, int lane) {
    any_last = -1; all_last = 0x7fffffff; any_low = 0x7fffffff; all_low = 0;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int r = row0 + 16 * t + (lane & 15);
      const bool there = r < rq.rows;
      const int token = there ? r / a.group : 0, sub = there ? r - token * a.group : 0;
      last[t] = there ? rq.start + token : -1;
      low[t] = there ? first_seen(last[t], a.window) : 0;
      // (a row that is not there has row 0's queries: no branch, and its sums are nobody's)
      const T* from = static_cast<const T*>(a.q) + (long)(rq.first + token) * a.ldq + (long)(head * a.group + sub) * D;
#pragma unroll
      for (int c = 0; c < kSections; ++c) {
        const int e = section_elems(c), dim = section_dim(c);
#pragma unroll
        for (int i = 0; i < e / 2; ++i) {
          const T* p = from + dim + (lane >> 4) * 4 * e + 8 * i;
          float x[8];
          if constexpr (sizeof(T) == 2) {
            typedef unsigned int any4 __attribute__((ext_vector_type(4), aligned(2)));
            any4 w = *reinterpret_cast<const any4*>(p);
            if (a.negative) w ^= any4{0x80008000u, 0x80008000u, 0x80008000u, 0x80008000u};
            q[0][t][dim / 32 + i] = as_operand(w[0], w[1], w[2], w[3]);
          } else {
            typedef float any4 __attribute__((ext_vector_type(4), aligned(4)));
            const any4 u = *reinterpret_cast<const any4*>(p), w = *reinterpret_cast<const any4*>(reinterpret_cast<const float*>(p) + 4);
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              x[y] = a.negative ? -u[y] : u[y];
              x[4 + y] = a.negative ? -w[y] : w[y];
            }
          }
          if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int y = 0; y < 8; ++y) {
              float rest = x[y];
#pragma unroll
              for (int term = 0; term < 3; ++term) {
                // (the numbers between bfloat16's largest and float32's would round to an infinity)
                const bf16_t part = static_cast<bf16_t>(term == 0 ? fminf(fmaxf(rest, -kLargestBf16), kLargestBf16) : rest);
                q[term][t][dim / 32 + i][y] = part;
                rest = rest - static_cast<float>(part);
              }
            }
          }
        }
      }
#pragma unroll
      for (int i = 0; i < D / 16; ++i) acc[t][i] = f32x4{0.f, 0.f, 0.f, 0.f};
      m[t] = -INFINITY;
      l[t] = 0.f;
    }
    // uniform bounds: rows are in the order of their positions
    const int row_end = min(row0 + 16 * NT, rq.rows);
    if (row0 < row_end) {
      all_last = rq.start + row0 / a.group;
      any_last = rq.start + (row_end - 1) / a.group;
      any_low = first_seen(all_last, a.window);
      all_low = first_seen(any_last, a.window);
    }
  }

  // The weights of the lane's scores (before their factor) of every row tile, and what they add to the sums.
  template <int H>
  __device__ __forceinline__ void weigh(const Fp4Args& a, const float (&x)[NT][8 * H], bf16x8 (&p)[kTerms<T>][NT][H]) {
    float top[NT];
    bool far = false;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      top[t] = x[t][0];
#pragma unroll
      for (int i = 1; i < 8 * H; ++i) top[t] = fmaxf(top[t], x[t][i]);
      top[t] = top[t] * a.factor;
      far = far || top[t] > m[t] + kSlack;  // (-inf + 8 is -inf: any score moves the first reference)
    }
    if (__ballot(far) != 0ull) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const float next = fmaxf(m[t], quad16_max(top[t]));
        const float f = m[t] == -INFINITY ? 0.f : weight_exp2<T>(m[t] - next);
        m[t] = next;
        l[t] = l[t] * f;
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
#pragma unroll
          for (int y = 0; y < 4; ++y) acc[t][i][y] = acc[t][i][y] * f;
      }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const float ref = m[t] == -INFINITY ? 0.f : m[t];
#pragma unroll
      for (int i = 0; i < 8 * H; ++i) {
        const float w = weight_exp2<T>(fmaf(x[t][i], a.factor, -ref));
        l[t] = l[t] + w;
        float rest = w;
#pragma unroll
        for (int term = 0; term < kTerms<T>; ++term) {
          const bf16_t part = static_cast<bf16_t>(rest);
          p[term][t][i / 8][i % 8] = part;
          if constexpr (kTerms<T> > 1) rest = rest - static_cast<float>(part);
        }
      }
    }
  }

  // 32 keys from t0 on.
  __device__ __forceinline__ void step(const Fp4Args& a, KeyTile& tile, int t0, int lane) {
    const int n = lane & 15, j = lane >> 4;
    const bool whole = t0 >= all_low && t0 + kTileKeys - 1 <= all_last && __ballot(!(tile.good[0] && tile.good[1])) == 0ull;
    if (!whole) {
      // what lies where no row looks may be anything: its values become zeros
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const int key = t0 + 16 * s + 4 * j + y;
          const bool seen = tile.good[s] && key >= any_low && key <= any_last;
#pragma unroll
          for (int c = 0; c < kSections; ++c) {
            tile.v[s][c][y] = seen ? tile.v[s][c][y] : 0u;
            tile.vs[s][c] = seen ? tile.vs[s][c] : ((tile.vs[s][c] & ~(255u << (8 * y))) | (127u << (8 * y)));
          }
        }
    }
    // groups that are not finite (rare): which keys, and which values
    bool k_nan[2] = {false, false}, v_nan = false;
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int c = 0; c < kSections; ++c) {
        k_nan[s] = k_nan[s] || tile.ks[s][c] == kFp4Nan;
        const unsigned int w = tile.vs[s][c];
        v_nan = v_nan || (((w & 0x7f7f7f7fu) + 0x01010101u) & w & 0x80808080u) != 0u;
      }
    unsigned int nan_keys = 0u;
    const bool bad_keys = __ballot(k_nan[0] || k_nan[1]) != 0ull;
    const bool bad_values = __ballot(v_nan) != 0ull;
    if (bad_keys) {
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const unsigned long long b = __ballot(k_nan[s]);
        const unsigned int f = (unsigned int)(b | (b >> 32));
        nan_keys |= ((f | (f >> 16)) & 0xffffu) << (16 * s);
      }
    }
    if (bad_values) mark_values(tile, t0, lane);

    // S^T = K Q^T
    f32x4 sc[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) sc[t][0] = sc[t][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int c = 0; c < kSections; ++c) {
        const float scale = fp4_scale(tile.ks[s][c]);
        const int base = section_dim(c) / 32;
#pragma unroll
        for (int i = 0; i < section_elems(c) / 2; ++i) {
          const unsigned int w = tile.k[s][base + i];
          const bf16x8 k = as_operand(fp4_pair<0>(w, scale), fp4_pair<1>(w, scale), fp4_pair<2>(w, scale), fp4_pair<3>(w, scale));
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int term = kTerms<T> - 1; term >= 0; --term)  // the small terms first
              sc[t][s] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, q[term][t][base + i], sc[t][s], 0, 0, 0);
        }
      }
    bf16x8 p[kTerms<T>][NT][1];
    float x[NT][8];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[t][i] = sc[t][i >> 2][i & 3];
      if (bad_keys) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          x[t][i] = ((nan_keys >> (16 * (i >> 2) + 4 * j + (i & 3))) & 1u) ? __uint_as_float(0x7fc00000u) : x[t][i];
      }
      if (!whole) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int key = t0 + 16 * (i >> 2) + 4 * j + (i & 3);
          const bool seen = key >= low[t] && key <= last[t] && tile.good[i >> 2];
          x[t][i] = seen ? x[t][i] : -INFINITY;
        }
      }
    }
    weigh<1>(a, x, p);
    // O^T += V^T P^T
#pragma unroll
    for (int c = 0; c < kSections; ++c) {
      const int e = section_elems(c), at = section_dim(c) / 16;
      float scale[2][4];
      unsigned int w[2][4];
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          scale[s][y] = fp4_scale((tile.vs[s][c] >> (8 * y)) & 255u);
          w[s][y] = e == 8 ? tile.v[s][c][y] : e == 4 ? tile.v[s][c][y] >> (16 * (n & 1)) : tile.v[s][c][y] >> (8 * (n & 3));
        }
#pragma unroll
      for (int pair = 0; pair < e / 2; ++pair) {
        unsigned int both[2][4];
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int y = 0; y < 4; ++y)
            both[s][y] = pair == 0 ? fp4_pair<0>(w[s][y], scale[s][y]) : pair == 1 ? fp4_pair<1>(w[s][y], scale[s][y])
                         : pair == 2 ? fp4_pair<2>(w[s][y], scale[s][y]) : fp4_pair<3>(w[s][y], scale[s][y]);
        const bf16x8 even = as_operand(__builtin_amdgcn_perm(both[0][1], both[0][0], 0x05040100u), __builtin_amdgcn_perm(both[0][3], both[0][2], 0x05040100u),
                                       __builtin_amdgcn_perm(both[1][1], both[1][0], 0x05040100u), __builtin_amdgcn_perm(both[1][3], both[1][2], 0x05040100u));
        const bf16x8 odd = as_operand(__builtin_amdgcn_perm(both[0][1], both[0][0], 0x07060302u), __builtin_amdgcn_perm(both[0][3], both[0][2], 0x07060302u),
                                      __builtin_amdgcn_perm(both[1][1], both[1][0], 0x07060302u), __builtin_amdgcn_perm(both[1][3], both[1][2], 0x07060302u));
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int term = kTerms<T> - 1; term >= 0; --term) {
            acc[t][at + 2 * pair] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(even, p[term][t][0], acc[t][at + 2 * pair], 0, 0, 0);
            acc[t][at + 2 * pair + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(odd, p[term][t][0], acc[t][at + 2 * pair + 1], 0, 0, 0);
          }
      }
    }
  }

  // Values of groups that are not finite: zeros for the product, and NaN in the sums of the rows that see them.
  __device__ __forceinline__ void mark_values(KeyTile& tile, int t0, int lane) {
    const int j = lane >> 4;
#pragma unroll
    for (int c = 0; c < kSections; ++c)
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int y = 0; y < 4; ++y) {  // (registers are not indexed by a loop's variable: unrolled)
          const bool here = ((tile.vs[s][c] >> (8 * y)) & 255u) == kFp4Nan;
          const unsigned long long b = __ballot(here);
          tile.v[s][c][y] = here ? 0u : tile.v[s][c][y];
          tile.vs[s][c] = here ? ((tile.vs[s][c] & ~(255u << (8 * y))) | (127u << (8 * y))) : tile.vs[s][c];
          if (b == 0ull) continue;
#pragma unroll 1
          for (int block = 0; block < 4; ++block) {
            // the lane's sums are of the columns 4 j .. 4 j + 3, which lie in one group; lane 4 j of the block tells
            const bool mine = (b >> (4 * j + 16 * block)) & 1ull;
            const int key = t0 + 16 * s + 4 * block + y;
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              const float add = mine && key >= low[t] && key <= last[t] ? __uint_as_float(0x7fc00000u) : 0.f;
#pragma unroll
              for (int i = 0; i < section_elems(c); ++i)
#pragma unroll
                for (int z = 0; z < 4; ++z) acc[t][section_dim(c) / 16 + i][z] += add;
            }
          }
        }
  }
};

// Walk the key tiles first, first + stride, ... below end.
template <typename T, int NT>
__device__ __forceinline__ void walk_keys(Rows<T, NT>& rows, const Fp4Args& a, const int* __restrict__ table_row, int head,
                                          int first, int end, int stride, int lane) {
  if (first >= end) return;
  PageIds ids = load_ids(a, table_row, first, lane);
  KeyTile tile;
  load_tile(tile, a, ids, head, first, lane);
  ids = load_ids(a, table_row, first + stride < end ? first + stride : first, lane);
  for (int t0 = first; t0 < end; t0 += stride) {
    KeyTile next;
    const int t1 = t0 + stride < end ? t0 + stride : t0;  // (behind the last tile the same one again: within bounds)
    load_tile(next, a, ids, head, t1, lane);
    ids = load_ids(a, table_row, t1 + stride < end ? t1 + stride : t1, lane);
    rows.step(a, tile, t0, lane);
    tile = next;
  }
}

// The same for pages of at least 16 tokens: 16 keys lie in one page, so a tile's addresses are two scalars and the lane's own
// offsets, which never change.  The block table's entries come 64 at a time, one a lane, a run ahead.
template <typename T, int NT>
__device__ __forceinline__ void walk_keys_by_pages(Rows<T, NT>& rows, const Fp4Args& a, const int* __restrict__ table_row, int head,
                                                   int first, int end, int stride, int lane) {
  if (first >= end) return;
  const int n = lane & 15, j = lane >> 4, shift = a.pool.page_shift, mask = (1 << shift) - 1;
  const int final = first + (end - 1 - first) / stride * stride;
  int base = first >> shift;  // the entry that lane 0 has
  int now = table_row[min(base + lane, a.columns - 1)], later = table_row[min(base + 64 + lane, a.columns - 1)];
  const auto load = [&](KeyTile& tile, int t0) LS_INLINED {
    // (uniform.  Tiles begin at multiples of 32, and so does the first run: both halves of a tile lie in one run.  A step is eight
    // entries at most: never more than one run ahead.)
    if (__builtin_expect(((t0 + 16) >> shift) - base >= 64, 0)) {  // (said to be rare: without it heads of 128 spill two registers)
      base += 64;
      now = later;
      later = table_row[min(base + 64 + lane, a.columns - 1)];
    }
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int at = t0 + 16 * s;
      const int page = __builtin_amdgcn_readlane(now, (at >> shift) - base);
      tile.good[s] = (unsigned int)page < (unsigned int)a.pool.pages;
      const long row = (((long)(tile.good[s] ? page : 0) * a.pool.kv_heads + head) << shift) + (at & mask);
      const unsigned char* kc = a.pool.k_codes + row * (D / 2);
      const unsigned char* ks = a.pool.k_scales + row * (D / 32);
      const unsigned char* vc = a.pool.v_codes + row * (D / 2);
      const unsigned char* vs = a.pool.v_scales + row * (D / 32);
#pragma unroll
      for (int c = 0; c < kSections; ++c) {
        const int e = section_elems(c), dim = section_dim(c);
        load_words(&tile.k[s][dim / 32], kc + (unsigned int)(n * (D / 2) + dim / 2 + j * 2 * e), e / 2);
        tile.ks[s][c] = ks[(unsigned int)(n * (D / 32) + (dim + j * 4 * e) / 32)];
        load_words(tile.v[s][c], vc + (unsigned int)(j * (2 * D) + (dim + n * e) / 8 * 16), 4);
        load_words(&tile.vs[s][c], vs + (unsigned int)(j * (D / 8) + (dim + n * e) / 32 * 4), 1);
      }
    }
  };
  KeyTile tile;
  load(tile, first);
  for (int t0 = first; t0 <= final; t0 += stride) {
    KeyTile next;
    load(next, min(t0 + stride, final));
    rows.step(a, tile, t0, lane);
    tile = next;
  }
}

template <typename T> __device__ __forceinline__ void store_run(T* to, const float* x, int n);
template <> __device__ __forceinline__ void store_run<float>(float* to, const float* x, int n) {
  typedef float any2 __attribute__((ext_vector_type(2), aligned(4)));
  typedef float any4 __attribute__((ext_vector_type(4), aligned(4)));
  if (n == 8) {
    *reinterpret_cast<any4*>(to) = any4{x[0], x[1], x[2], x[3]};
    *reinterpret_cast<any4*>(to + 4) = any4{x[4], x[5], x[6], x[7]};
  } else if (n == 4) {
    *reinterpret_cast<any4*>(to) = any4{x[0], x[1], x[2], x[3]};
  } else {
    *reinterpret_cast<any2*>(to) = any2{x[0], x[1]};
  }
}
template <> __device__ __forceinline__ void store_run<bf16_t>(bf16_t* to, const float* x, int n) {
  typedef __bf16 any2 __attribute__((ext_vector_type(2), aligned(2)));
  typedef __bf16 any4 __attribute__((ext_vector_type(4), aligned(2)));
  typedef __bf16 any8 __attribute__((ext_vector_type(8), aligned(2)));
  if (n == 8) {
    *reinterpret_cast<any8*>(to) = any8{(bf16_t)x[0], (bf16_t)x[1], (bf16_t)x[2], (bf16_t)x[3], (bf16_t)x[4], (bf16_t)x[5], (bf16_t)x[6], (bf16_t)x[7]};
  } else if (n == 4) {
    *reinterpret_cast<any4*>(to) = any4{(bf16_t)x[0], (bf16_t)x[1], (bf16_t)x[2], (bf16_t)x[3]};
  } else {
    *reinterpret_cast<any2*>(to) = any2{(bf16_t)x[0], (bf16_t)x[1]};
  }
}

// Waves a SIMD: what is in flight is what the waves ask for, a tile each (64 requests of up to 8,192 keys: three waves
// 108 us, four 101; a second tile ahead in two waves 124).
template <typename T> constexpr int kDecodeWaves = std::is_same_v<T, float> ? (D > 160 ? 1 : 2) : kSections == 1 ? 4 : D <= 96 ? 3 : 2;

// Decoded tokens: a workgroup has one split of one head of one request.
constexpr int kFoldPad = D + 4;
struct FoldShared {
  float acc[4][16][kFoldPad];
  float m[4][16], l[4][16];
};
template <typename T, bool kWholePages>
__device__ __forceinline__ void decode_part(const Fp4Args& a, FoldShared& fold, int split, int head, int b) {
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Request rq(a, b);
  if (rq.rows == 0 || rq.rows > kFewRows) return;
  const Cut cut = cut_request<T>(rq.rows, rq.end - rq.base, a.pool.kv_heads);
  const int splits = cut.splits, len = cut.len;
  if (split >= splits) return;
  const int begin = rq.base + split * len, end = min(rq.end, begin + len);
  Rows<T, 1> rows;
  rows.init(a, rq, head, 0, lane);
  const int* row = a.table + (long)b * a.columns;
  if constexpr (kWholePages)
    walk_keys_by_pages<T, 1>(rows, a, row, head, begin + kTileKeys * w, end, 4 * kTileKeys, lane);
  else
    walk_keys<T, 1>(rows, a, row, head, begin + kTileKeys * w, end, 4 * kTileKeys, lane);
  const int n = lane & 15, j = lane >> 4;
  const float l = quad16_sum(rows.l[0]);
  if (j == 0) {
    fold.m[w][n] = rows.m[0];
    fold.l[w][n] = l;
  }
#pragma unroll
  for (int c = 0; c < kSections; ++c)
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      const int e = section_elems(c);
      float x[8];
#pragma unroll
      for (int i = 0; i < e; ++i) x[i] = rows.acc[0][section_dim(c) / 16 + i][y];
      float* to = &fold.acc[w][n][section_dim(c) + e * (4 * j + y)];
#pragma unroll
      for (int i = 0; i < e; ++i) to[i] = x[i];
    }
  __syncthreads();
  const int there = min(rq.rows, 16);
  for (int i = threadIdx.x; i < there * (D / 4); i += kThreads) {
    const int r = i / (D / 4), d = 4 * (i % (D / 4));
    float top = fold.m[0][r];
#pragma unroll
    for (int k = 1; k < 4; ++k) top = fmaxf(top, fold.m[k][r]);
    float sum = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float f = fold.m[k][r] == -INFINITY ? fold.l[k][r] : weight_exp2<T>(fold.m[k][r] - top);  // (no score: 0, or NaN)
      sum = fmaf(fold.l[k][r], f, sum);
#pragma unroll
      for (int y = 0; y < 4; ++y) x[y] = fmaf(fold.acc[k][r][d + y], f, x[y]);
    }
    if (splits == 1) {
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
      for (int y = 0; y < 4; ++y) x[y] = x[y] * inv;
      const int token = r / a.group, sub = r - token * a.group;
      store_run<T>(static_cast<T*>(a.out) + (long)(rq.first + token) * a.ldo + (long)(head * a.group + sub) * D + d, x, 4);
    } else {
      const long at = split_entry(a, rq, b, head, split, r);
      if (at >= 0) {
        store_run<float>(a.part_acc + at * D + d, x, 4);
        if (d == 0) {
          a.part_ml[2 * at] = top;
          a.part_ml[2 * at + 1] = sum;
        }
      }
    }
  }
}

template <typename T, bool kWholePages>
__global__ __launch_bounds__(kThreads, kDecodeWaves<T>) void fp4_decode_kernel(Fp4Args a) {
  __shared__ FoldShared fold;
  // Grid (kv heads, requests, splits): neighbours in x go to one XCD after the other, so with heads there every XCD has as
  // much to do, and the workgroups of splits that a request does not have come last.  (With splits in x the XCDs of the last
  // ones had nothing: 64 requests of 4,608 keys in five of eight places 95 us, now 75.)
  decode_part<T, kWholePages>(a, fold, blockIdx.z, blockIdx.x, blockIdx.y);
}

// Prompts: a workgroup's four waves share the tiles of 64 keys, as operands in LDS.  Wave w makes the operands of the
// keys 16 w .. 16 w + 15, and of half of the values of the 32 keys from 32 (w / 2) on; an operand is 1 KiB, 16 bytes a lane,
// written and read in one piece.  Two buffers: while one is read, the codes of the next tile are on their way to registers.
constexpr int kOperands = 4 * (D / 32) + 2 * (D / 16);  // operands of a tile: keys, then values
struct SharedFlags {  // what is out of the ordinary in a tile (rare); `any` says whether there is something
  unsigned int any[4], k_nan[4], k_bad[4];
  unsigned long long v_nan[2][kSections][2][4];  // by half of the tile, section, 16 keys, place in a block: a bit a lane
};

struct Staged {  // the codes a wave turns into operands
  unsigned int k[D / 32], ks[kSections];
  unsigned int v[2][kSections][4], vs[2][kSections];
  bool k_ok, v_ok[2];
};
struct StagedIds {
  int k, v[2];
};

__device__ __forceinline__ StagedIds staged_ids(const Fp4Args& a, const int* __restrict__ row, int t0, int lane, int w) {
  StagedIds ids;
  ids.k = row[min((t0 + 16 * w + (lane & 15)) >> a.pool.page_shift, a.columns - 1)];
#pragma unroll
  for (int s = 0; s < 2; ++s)
    ids.v[s] = row[min((t0 + 32 * (w >> 1) + 16 * s + 4 * (lane >> 4)) >> a.pool.page_shift, a.columns - 1)];
  return ids;
}

// Where a lane's codes lie in a page that begins at a tile (or holds a part of one): page 0's addresses.  A row of a pool is a
// token of a head of a page; value blocks are of four rows, so rows times the bytes of one row are their addresses too.
struct StagedFrom {
  const unsigned char *kc, *ks, *vc[2], *vs[2];
  unsigned int code_page, scale_page;  // bytes of a page
  int mask;
  __device__ __forceinline__ void init(const Fp4Args& a, int head, int lane, int w) {
    const int n = lane & 15, j = lane >> 4;
    mask = (1 << a.pool.page_shift) - 1;
    const long head_row = (long)head << a.pool.page_shift;
    const long k_row = head_row + ((16 * w + n) & mask);
    kc = a.pool.k_codes + k_row * (D / 2);
    ks = a.pool.k_scales + k_row * (D / 32);
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const long v_row = head_row + ((32 * (w >> 1) + 16 * s + 4 * j) & mask);
      vc[s] = a.pool.v_codes + v_row * (D / 2);
      vs[s] = a.pool.v_scales + v_row * (D / 32);
    }
    code_page = (unsigned int)(a.pool.kv_heads << a.pool.page_shift) * (D / 2);
    scale_page = code_page / 16;
  }
};

// The codes of the tile at t0, a multiple of 64.
__device__ __forceinline__ void stage_tile(Staged& st, const Fp4Args& a, const StagedFrom& from, const StagedIds& ids, int t0, int lane) {
  const int n = lane & 15, j = lane >> 4;
  const long row = t0 & from.mask & ~(kSharedKeys - 1);  // (uniform) in pages of more than a tile
  st.k_ok = (unsigned int)ids.k < (unsigned int)a.pool.pages;
  const unsigned int k_page = st.k_ok ? ids.k : 0;
  const unsigned char* kc = from.kc + row * (D / 2) + (unsigned long)k_page * from.code_page;
  const unsigned char* ks = from.ks + row * (D / 32) + (unsigned long)k_page * from.scale_page;
#pragma unroll
  for (int c = 0; c < kSections; ++c) {
    const int e = section_elems(c), dim = section_dim(c);
    load_words(&st.k[dim / 32], kc + (dim / 2 + j * 2 * e), e / 2);
    st.ks[c] = ks[(dim + j * 4 * e) / 32];
  }
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    st.v_ok[s] = (unsigned int)ids.v[s] < (unsigned int)a.pool.pages;
    const unsigned int v_page = st.v_ok[s] ? ids.v[s] : 0;
    const unsigned char* vc = from.vc[s] + row * (D / 2) + (unsigned long)v_page * from.code_page;
    const unsigned char* vs = from.vs[s] + row * (D / 32) + (unsigned long)v_page * from.scale_page;
#pragma unroll
    for (int c = 0; c < kSections; ++c) {
      const int e = section_elems(c), dim = section_dim(c);
      load_words(st.v[s][c], vc + (dim + n * e) / 8 * 16, 4);
      load_words(&st.vs[s][c], vs + (dim + n * e) / 32 * 4, 1);
    }
  }
}

// What is out of the ordinary in the codes of a tile: keys that no row of the workgroup sees (outside low .. last) and pages
// that are not there become zeros, groups that are not finite zeros and flags.
__device__ __forceinline__ void check_tile(Staged& st, SharedFlags& flags, int t0, int low, int last, int lane, int w) {
  const int j = lane >> 4, v0 = t0 + 32 * (w >> 1);
  bool odd = !(st.k_ok && st.v_ok[0] && st.v_ok[1]);
#pragma unroll
  for (int c = 0; c < kSections; ++c) odd = odd || st.ks[c] == kFp4Nan;
#pragma unroll
  for (int s = 0; s < 2; ++s)
#pragma unroll
    for (int c = 0; c < kSections; ++c) {
      const unsigned int b = st.vs[s][c];
      odd = odd || (((b & 0x7f7f7f7fu) + 0x01010101u) & b & 0x80808080u) != 0u;
    }
  const bool any = __ballot(odd) != 0ull;
  if (lane == 0) flags.any[w] = any ? 1u : 0u;
  if (!any && v0 >= low && v0 + 31 <= last) return;  // (uniform)
#pragma unroll
  for (int s = 0; s < 2; ++s)
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      const int key = v0 + 16 * s + 4 * j + y;
      const bool seen = st.v_ok[s] && key >= low && key <= last;
#pragma unroll
      for (int c = 0; c < kSections; ++c) {
        st.v[s][c][y] = seen ? st.v[s][c][y] : 0u;
        st.vs[s][c] = seen ? st.vs[s][c] : ((st.vs[s][c] & ~(255u << (8 * y))) | (127u << (8 * y)));
      }
    }
  if (!any) return;
  bool k_nan = false;
#pragma unroll
  for (int c = 0; c < kSections; ++c) k_nan = k_nan || st.ks[c] == kFp4Nan;
  const unsigned long long nan = __ballot(k_nan), bad = __ballot(!st.k_ok);
  const unsigned int f = (unsigned int)(nan | (nan >> 32)), g = (unsigned int)(bad | (bad >> 32));
  if (lane == 0) {
    flags.k_nan[w] = (f | (f >> 16)) & 0xffffu;
    flags.k_bad[w] = (g | (g >> 16)) & 0xffffu;
  }
#pragma unroll
  for (int c = 0; c < kSections; ++c)
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const bool here = ((st.vs[s][c] >> (8 * y)) & 255u) == kFp4Nan;
        const unsigned long long b = __ballot(here);
        if (lane == 0 && (w & 1) == 0) flags.v_nan[w >> 1][c][s][y] = b;
        st.v[s][c][y] = here ? 0u : st.v[s][c][y];
        st.vs[s][c] = here ? ((st.vs[s][c] & ~(255u << (8 * y))) | (127u << (8 * y))) : st.vs[s][c];
      }
}

// Codes to operands: the keys'.
__device__ __forceinline__ void share_keys(const Staged& st, bf16x8* __restrict__ operands, int lane, int w) {
#pragma unroll
  for (int c = 0; c < kSections; ++c) {
    const float scale = fp4_scale(st.ks[c]);
    const int base = section_dim(c) / 32;
#pragma unroll
    for (int i = 0; i < section_elems(c) / 2; ++i) {
      const unsigned int x = st.k[base + i];
      operands[(w * (D / 32) + base + i) * 64 + lane] =
          as_operand(fp4_pair<0>(x, scale), fp4_pair<1>(x, scale), fp4_pair<2>(x, scale), fp4_pair<3>(x, scale));
    }
  }
}

// The values': of the pairs of elements that a lane column has, the wave's half (of a section of one pair, the even wave's).
__device__ __forceinline__ void share_values(const Staged& st, bf16x8* __restrict__ operands, int lane, int w) {
  const int n = lane & 15;
#pragma unroll
  for (int c = 0; c < kSections; ++c) {
    const int e = section_elems(c), at = section_dim(c) / 16;
    const int mine = e == 8 ? 2 : 1;
    if (e == 2 && (w & 1)) continue;  // (uniform)
    const int from = e == 2 ? 0 : mine * (w & 1);
    unsigned int x[2][4];
    float scale[2][4];
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        scale[s][y] = fp4_scale((st.vs[s][c] >> (8 * y)) & 255u);
        x[s][y] = st.v[s][c][y] >> ((e == 8 ? 0 : e == 4 ? 16 * (n & 1) : 8 * (n & 3)) + 8 * from);
      }
#pragma unroll
    for (int pair = 0; pair < mine; ++pair) {
      unsigned int both[2][4];
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int y = 0; y < 4; ++y) both[s][y] = pair == 0 ? fp4_pair<0>(x[s][y], scale[s][y]) : fp4_pair<1>(x[s][y], scale[s][y]);
      bf16x8* to = operands + (4 * (D / 32) + (w >> 1) * (D / 16) + at + 2 * (from + pair)) * 64 + lane;
      to[0] = as_operand(__builtin_amdgcn_perm(both[0][1], both[0][0], 0x05040100u), __builtin_amdgcn_perm(both[0][3], both[0][2], 0x05040100u),
                         __builtin_amdgcn_perm(both[1][1], both[1][0], 0x05040100u), __builtin_amdgcn_perm(both[1][3], both[1][2], 0x05040100u));
      to[64] = as_operand(__builtin_amdgcn_perm(both[0][1], both[0][0], 0x07060302u), __builtin_amdgcn_perm(both[0][3], both[0][2], 0x07060302u),
                          __builtin_amdgcn_perm(both[1][1], both[1][0], 0x07060302u), __builtin_amdgcn_perm(both[1][3], both[1][2], 0x07060302u));
    }
  }
}

// Scores of a shared tile's 64 keys.
template <typename T, int NT>
__device__ __forceinline__ void score_shared(const Rows<T, NT>& rows, f32x4 (&sc)[NT][4], const bf16x8* __restrict__ operands, int lane) {
#pragma unroll
  for (int s = 0; s < 4; ++s)
#pragma unroll
    for (int t = 0; t < NT; ++t) sc[t][s] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int s = 0; s < 4; ++s)
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      const bf16x8 k = operands[(s * (D / 32) + i) * 64 + lane];
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int term = kTerms<T> - 1; term >= 0; --term)
          sc[t][s] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, rows.q[term][t][i], sc[t][s], 0, 0, 0);
    }
}

// Weights of the scores of the keys t0 .. t0 + 63, and the sums of the values.
template <typename T, int NT>
__device__ __forceinline__ void sum_shared(Rows<T, NT>& rows, const Fp4Args& a, const f32x4 (&sc)[NT][4], const bf16x8* __restrict__ operands,
                                           const SharedFlags& flags, bool odd, int t0, int lane) {
  const int j = lane >> 4;
  const bool whole = t0 >= rows.all_low && t0 + kSharedKeys - 1 <= rows.all_last;
  bf16x8 p[kTerms<T>][NT][2];
  float x[NT][16];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) x[t][i] = sc[t][i >> 2][i & 3];
  if (odd) {  // (uniform, rare)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int w = i >> 2, bit = 4 * j + (i & 3);
      const bool nan = flags.any[w] != 0u && ((flags.k_nan[w] >> bit) & 1u), bad = flags.any[w] != 0u && ((flags.k_bad[w] >> bit) & 1u);
#pragma unroll
      for (int t = 0; t < NT; ++t) x[t][i] = bad ? -INFINITY : nan ? __uint_as_float(0x7fc00000u) : x[t][i];
    }
  }
  if (!whole) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int key = t0 + 16 * (i >> 2) + 4 * j + (i & 3);
#pragma unroll
      for (int t = 0; t < NT; ++t) x[t][i] = key >= rows.low[t] && key <= rows.last[t] ? x[t][i] : -INFINITY;
    }
  }
  rows.template weigh<2>(a, x, p);
  if (odd) {  // values that are not finite (those of pages that are not there are zeros)
    for (int u = 0; u < 2; ++u)
      if (flags.any[2 * u] != 0u)
        for (int s = 0; s < 2; ++s)
          for (int y = 0; y < 4; ++y)
            for (int block = 0; block < 4; ++block) {
              const int key = t0 + 32 * u + 16 * s + 4 * block + y;
#pragma unroll
              for (int c = 0; c < kSections; ++c) {
                const bool here = (flags.v_nan[u][c][s][y] >> (4 * j + 16 * block)) & 1ull;
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                  const float add = here && key >= rows.low[t] && key <= rows.last[t] ? __uint_as_float(0x7fc00000u) : 0.f;
#pragma unroll
                  for (int i = 0; i < section_elems(c); ++i)
#pragma unroll
                    for (int z = 0; z < 4; ++z) rows.acc[t][section_dim(c) / 16 + i][z] += add;
                }
              }
            }
  }
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      const bf16x8 v = operands[(4 * (D / 32) + u * (D / 16) + i) * 64 + lane];
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int term = kTerms<T> - 1; term >= 0; --term)
          rows.acc[t][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, p[term][t][u], rows.acc[t][i], 0, 0, 0);
    }
}

struct PromptShared {
  bf16x8 operands[2][kOperands * 64];
  SharedFlags flags[2];
};
// A workgroup has four row blocks of a head of a request, and one split of its keys.
template <typename T>
__device__ __forceinline__ void prompt_part(const Fp4Args& a, PromptShared& shared, int place, int head, int b) {
  constexpr int NT = kPromptTiles<T>, kBlock = 16 * NT;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  auto& operands = shared.operands;
  auto& flags = shared.flags;
  const Request rq(a, b);
  if (rq.rows <= kFewRows) return;
  const Cut cut = cut_request<T>(rq.rows, rq.end - rq.base, a.pool.kv_heads);
  const int groups = cut.groups, splits = cut.splits, len = cut.len;
  if (place >= groups * splits) return;
  const int split = place / groups, group = groups - 1 - (place - split * groups);  // the rows that see most keys first
  const int row0 = (4 * group + w) * kBlock;
  Rows<T, NT> rows;
  rows.init(a, rq, head, row0, lane);
  // the keys that the workgroup's rows see
  const int first_token = 4 * group * kBlock / a.group, last_token = (min((4 * group + 4) * kBlock, rq.rows) - 1) / a.group;
  const int low = first_seen(rq.start + first_token, a.window), last = rq.start + last_token;
  const int split_begin = rq.base + split * len;
  const int begin = low > split_begin ? split_begin + (low - split_begin) / kSharedKeys * kSharedKeys : split_begin;
  const int end = min(min(rq.end, split_begin + len), last + 1);
  const int* row = a.table + (long)b * a.columns;
  if (begin < end) {  // (uniform)
    StagedFrom from;
    from.init(a, head, lane, w);
    Staged st;
    // tiles behind the last are asked for as the last one again: within bounds, and not used
    const int final = begin + (end - 1 - begin) / kSharedKeys * kSharedKeys;
    StagedIds ids = staged_ids(a, row, begin, lane, w);
    stage_tile(st, a, from, ids, begin, lane);
    ids = staged_ids(a, row, min(begin + kSharedKeys, final), lane, w);
    check_tile(st, flags[0], begin, low, last, lane, w);
    share_keys(st, operands[0], lane, w);
    share_values(st, operands[0], lane, w);
    stage_tile(st, a, from, ids, min(begin + kSharedKeys, final), lane);
    ids = staged_ids(a, row, min(begin + 2 * kSharedKeys, final), lane, w);
    __syncthreads();
    int buffer = 0;
    for (int t0 = begin; t0 <= final; t0 += kSharedKeys, buffer ^= 1) {
      const SharedFlags& f = flags[buffer];
      check_tile(st, flags[buffer ^ 1], min(t0 + kSharedKeys, final), low, last, lane, w);
      // the products of the keys, and beside them the next tile's operands
      f32x4 sc[NT][4];
      share_keys(st, operands[buffer ^ 1], lane, w);
      score_shared<T, NT>(rows, sc, operands[buffer], lane);
      share_values(st, operands[buffer ^ 1], lane, w);
      stage_tile(st, a, from, ids, min(t0 + 2 * kSharedKeys, final), lane);
      ids = staged_ids(a, row, min(t0 + 3 * kSharedKeys, final), lane, w);
      const bool odd = __builtin_amdgcn_readfirstlane(f.any[0] | f.any[1] | f.any[2] | f.any[3]) != 0;
      sum_shared<T, NT>(rows, a, sc, operands[buffer], f, odd, t0, lane);
      __syncthreads();
    }
  }
  const int n = lane & 15, j = lane >> 4;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int r = row0 + 16 * t + n;
    const float l = quad16_sum(rows.l[t]);
    const bool there = r < rq.rows;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int token = there ? r / a.group : 0, sub = there ? r - token * a.group : 0;
    T* out = static_cast<T*>(a.out) + (long)(rq.first + token) * a.ldo + (long)(head * a.group + sub) * D;
    const long at = there ? split_entry(a, rq, b, head, split, r) : -1;
    const bool keep = at >= 0;
    if (splits > 1 && keep && j == 0) {
      a.part_ml[2 * at] = rows.m[t];
      a.part_ml[2 * at + 1] = l;
    }
#pragma unroll
    for (int c = 0; c < kSections; ++c)
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const int e = section_elems(c), dim = section_dim(c) + e * (4 * j + y);
        float x[8];
#pragma unroll
        for (int i = 0; i < e; ++i) x[i] = rows.acc[t][section_dim(c) / 16 + i][y];
        if (splits == 1) {
#pragma unroll
          for (int i = 0; i < e; ++i) x[i] = x[i] * inv;
          if (there) store_run<T>(out + dim, x, e);
        } else if (keep) {
          store_run<float>(a.part_acc + at * D + dim, x, e);
        }
      }
  }
}

// Steps with prompts: grid (kv heads, places + splits, requests); a request has as many places as row blocks of a workgroup
// times splits, and with the heads in x an XCD reads few heads' pages again and again.  Behind them in y is the decoding part, for the requests of few rows among them (only the device knows which; a
// launch of its own cost 4.5 us with nothing to do).
template <typename T, bool kWholePages>
__global__ __launch_bounds__(kThreads, kPromptWaves<T>) void fp4_prompt_kernel(Fp4Args a, int places) {
  __shared__ union Shared {
    PromptShared prompt;
    FoldShared fold;
    __device__ Shared() {}
  } shared;
  const int at = blockIdx.y, head = blockIdx.x;
  if (at < places) prompt_part<T>(a, shared.prompt, at, head, blockIdx.z);
  else decode_part<T, kWholePages>(a, shared.fold, at - places, head, blockIdx.z);
}

// Fold the splits of a (row, head): the sums of the splits 0, 4, 8, ..., those of 1, 5, ..., and so on, then the four in order.
// Few of them: a workgroup each, a wave a sum, the factors of all splits first so that the sums' loads do not wait for one
// another (4 requests of 131,071 keys in 64 splits: 12 -> 5.4 us).  Many: a wave each, the same sums (bits) in its registers.
constexpr int kMostSplits = kDecodeGroups;
static_assert(kPromptGroups <= kMostSplits, "the combine kernel keeps a factor a split");
template <typename T, bool kWaveEach>
__global__ __launch_bounds__(kThreads) void fp4_combine_kernel(Fp4Args a) {  // grid ((row, head) pairs of a request, requests)
  __shared__ float factor[kWaveEach ? 1 : kMostSplits];
  __shared__ float part[kWaveEach ? 1 : 4][D];
  const int t = threadIdx.x, lane = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6);
  const int heads = a.group * a.pool.kv_heads, b = blockIdx.y;
  const Request rq(a, b);
  const int splits = cut_request<T>(rq.rows, rq.end - rq.base, a.pool.kv_heads).splits;
  if (splits <= 1 || splits > kMostSplits) return;
  const int pairs = rq.rows * a.pool.kv_heads, stride_pairs = kWaveEach ? 4 * gridDim.x : gridDim.x;
  constexpr int kEach = (D + 63) / 64;
  const int d0 = kEach * lane;
  for (int place = kWaveEach ? 4 * blockIdx.x + w : blockIdx.x; place < pairs; place += stride_pairs) {
    const int token = place / heads, query_head = place - token * heads, row = rq.first + token;
    const int head = query_head / a.group, r = token * a.group + (query_head - head * a.group);
    const long base = split_entry(a, rq, b, head, 0, r), apart = rq.rows;
    if (split_entry(a, rq, b, head, splits - 1, r) < 0) return;
    T* out = static_cast<T*>(a.out) + (long)row * a.ldo + (long)query_head * D;
    const auto sum_at = [&](int s, int y) LS_INLINED -> float { return a.part_acc[(base + s * apart) * D + min(d0 + y, D - 1)]; };
    // (asked for before the factors are known)
    float ahead[kWaveEach ? 4 : 1][kEach];
#pragma unroll
    for (int k = 0; k < (kWaveEach ? 4 : 1); ++k)
#pragma unroll
      for (int y = 0; y < kEach; ++y) ahead[k][y] = sum_at(min(kWaveEach ? k : w, splits - 1), y);
    // every wave the same: the largest reference, the factors, the sum of the weights
    float top = -INFINITY;
    for (int s = lane; s < splits; s += 64) top = fmaxf(top, a.part_ml[2 * (base + s * apart)]);
    top = wave_max(top);
    const auto factor_of = [&](int s, float& l) LS_INLINED -> float {
      const float m = a.part_ml[2 * (base + s * apart)];
      l = a.part_ml[2 * (base + s * apart) + 1];
      return m == -INFINITY ? l : weight_exp2<T>(m - top);  // (no score: 0, or NaN)
    };
    float sum = 0.f, l;
    for (int s = lane; s < splits; s += 64) {
      const float f = factor_of(s, l);
      sum = fmaf(l, f, sum);
      if (!kWaveEach && w == 0) factor[s] = f;
    }
    sum = wave_sum(sum);
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    if constexpr (kWaveEach) {
      float x[4][kEach];
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int y = 0; y < kEach; ++y) x[k][y] = 0.f;
      for (int s0 = 0; s0 < splits; s0 += 4)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int s = min(s0 + k, splits - 1);
          const float f = factor_of(s, l);
#pragma unroll
          for (int y = 0; y < kEach; ++y) {
            const float v = fmaf(s0 == 0 ? ahead[k][y] : sum_at(s, y), f, x[k][y]);
            x[k][y] = s0 + k < splits ? v : x[k][y];
          }
        }
#pragma unroll
      for (int y = 0; y < kEach; ++y)
        if (d0 + y < D) out[d0 + y] = from_f32<T>((((x[0][y] + x[1][y]) + x[2][y]) + x[3][y]) * inv);
    } else {
      __syncthreads();
      float x[kEach];
#pragma unroll
      for (int y = 0; y < kEach; ++y) x[y] = w < splits ? fmaf(ahead[0][y], factor[min(w, splits - 1)], 0.f) : 0.f;
#pragma unroll 8
      for (int s = w + 4; s < splits; s += 4) {
        const float f = factor[s];
#pragma unroll
        for (int y = 0; y < kEach; ++y) x[y] = fmaf(sum_at(s, y), f, x[y]);
      }
#pragma unroll
      for (int y = 0; y < kEach; ++y)
        if (d0 + y < D) part[w][d0 + y] = x[y];
      __syncthreads();
      if (t < D) out[t] = from_f32<T>((((part[0][t] + part[1][t]) + part[2][t]) + part[3][t]) * inv);
      __syncthreads();
    }
  }
}

struct Plan {
  int decode_splits = 1, prompt_places = 0;  // places: row blocks of a workgroup times splits, of a request's head
  bool fold = false;                         // a request may have more than one split
  long per_row = 0, per_request = 0, head_entries = 0;
};

// What is launched for `requests` requests with `rows` rows, of at most `most` tokens and `longest` keys: bounds for every such step.
// (In host code the plain min and max are those of int: what may pass 31 bits takes the standard library's.)
template <typename T>
Plan make_plan(int kv_heads, int group, int rows, int requests, int most, int longest, int window) {
  Plan p;
  // What requests of so many tokens leave a head at most, at both ends of every run of lengths (behind its first a sixth more: 17 to
  // 32,768 tokens are 49 runs): between them it is no more than on the straight line, and where it reaches `most_entries`, which
  // no prompt passes, it stays there.
  struct End {
    long tokens, entries;
  } ends[128];
  int used = 0;
  const auto run_of = [&](long first, long last, int splits, long most_entries) {
    ends[used++] = {first, std::min<long>(first * group * splits, most_entries)};
    ends[used++] = {std::min<long>(last, std::max<long>(first, most_entries / ((long)group * splits))), std::min<long>(last * group * splits, most_entries)};
  };
  // the keys that a request's rows see, at most: with a window those of its tokens and the window before, in whole tiles
  const auto seen = [&](int n) { return window > 0 ? (int)std::min<long>(longest, (long)n + window - 1 + kSharedKeys) : longest; };
  const int few = kFewRows / group, span = seen(min(max(1, few), most));
  if (span > kOneSplit) {
    const auto most_of = [&](int n) { return (n + shortest_split(n, kv_heads) - 1) / shortest_split(n, kv_heads); };
    p.decode_splits = min(max(most_of(span), most_of(min(span, 4096))), (kDecodeGroups + kv_heads - 1) / kv_heads);
    if (p.decode_splits > 1 && few > 0) run_of(1, min(few, most), p.decode_splits, kFewRows * (long)p.decode_splits);
  }
  if (most > few) {
    const auto groups_of = [&](int n) { return (int)(((long)n * group + kGroupRows<T> - 1) / kGroupRows<T>); };
    p.prompt_places = groups_of(most);
    // (a run's first length has most splits)
    for (int n = few + 1, last; n <= most; n = last + 1) {
      const int groups = groups_of(n), want = prompt_splits_wanted(groups, kv_heads);
      if (want == 1) break;  // nor has any longer one more than one split
      last = min(most, n + n / 6);
      const int shortest = shortest_prompt_split<T>((int)std::min<long>((long)n * group, kPromptShortMost));
      const int splits = min(want, (seen(last) + shortest - 1) / shortest);
      if (splits > 1) {
        const int places = prompt_splits_wanted(1, kv_heads);  // of a request with more than one split, at most
        run_of(n, last, splits, (long)places * kGroupRows<T>);
        p.prompt_places = max(p.prompt_places, min(places, groups_of(last) * splits));
      }
    }
  }
  p.fold = used > 0;
  // Room by rows, by requests or some of each, whichever takes least: with so much a row, a request has what it may still lack.
  for (long splits = 0; p.fold && splits <= kDecodeGroups; splits = splits ? 2 * splits : 1)
    for (const long per_row : {splits * group, (long)p.decode_splits * group}) {
      long lacks = 0;
      for (int i = 0; i < used; ++i) lacks = std::max<long>(lacks, ends[i].entries - per_row * ends[i].tokens);
      const long all = per_row * rows + lacks * requests;
      if (p.head_entries == 0 || all < p.head_entries) {
        p.per_row = per_row;
        p.per_request = lacks;
        p.head_entries = all;
      }
    }
  return p;
}

// Bytes of the splits' sums that a step may leave.
inline long bytes_of(const Plan& p, int kv_heads) { return p.head_entries * kv_heads * (D + 2) * (long)sizeof(float); }

template <typename T, bool kWholePages>
void launch_parts(const Fp4Args& a, const Plan& p, hipStream_t stream) {
  const int heads = a.pool.kv_heads;
  if (p.prompt_places == 0)
    fp4_decode_kernel<T, kWholePages><<<dim3(heads, a.requests, p.decode_splits), kThreads, 0, stream>>>(a);
  else
    fp4_prompt_kernel<T, kWholePages><<<dim3(heads, p.prompt_places + p.decode_splits, a.requests), kThreads, 0, stream>>>(a, p.prompt_places);
}

template <typename T>
int run_fp4(Fp4Args& a, int most, int longest, void* scratch, long scratch_bytes, hipStream_t stream) {
  const int heads = a.pool.kv_heads;
  const Plan p = make_plan<T>(heads, a.group, a.rows, a.requests, most, longest, a.window);
  a.per_row = p.per_row; a.per_request = p.per_request; a.head_entries = p.head_entries;
  LS_REQUIRE((long)p.prompt_places + p.decode_splits <= 65535, "fp4_attention: %d rows a request", most);
  LS_REQUIRE(scratch_bytes >= bytes_of(p, heads), "fp4_attention: %ld bytes of scratch, %ld needed", scratch_bytes, bytes_of(p, heads));
  a.part_acc = static_cast<float*>(scratch);
  a.part_ml = a.part_acc + p.head_entries * heads * D;
  if (a.pool.page_shift >= 4) launch_parts<T, true>(a, p, stream);
  else launch_parts<T, false>(a, p, stream);
  if (p.fold) {
    const long pairs = (long)most * a.group * heads;  // of the request with most
    LS_REQUIRE(pairs <= 0x7ffffff0l, "fp4_attention: %d rows of %d heads", most, a.group * heads);
    if (pairs * a.requests >= 2048)
      fp4_combine_kernel<T, true><<<dim3((unsigned)std::min<long>((pairs + 3) / 4, 1024), a.requests), kThreads, 0, stream>>>(a);
    else
      fp4_combine_kernel<T, false><<<dim3((unsigned)pairs, a.requests), kThreads, 0, stream>>>(a);
  }
  return check_launch("fp4_attention");
}

}  // namespace ls

LS_DEFINE_ERROR_API

extern "C" int ls_fp4_attention_head_dim() { return ls::D; }

extern "C" long ls_fp4_attention_scratch_bytes(int dtype, int rows, int requests, int kv_heads, int group, int most, int longest, int window) {
  using namespace ls;
  if (rows <= 0 || requests <= 0 || kv_heads <= 0 || group <= 0 || most <= 0) return 0;
  return bytes_of(dtype == kF32 ? make_plan<float>(kv_heads, group, rows, requests, most, longest, window)
                                : make_plan<bf16_t>(kv_heads, group, rows, requests, most, longest, window), kv_heads);
}

namespace ls {
template <typename T>
void plan_of(int rows, int requests, int kv_heads, int group, int most, int longest, int window, int tokens, int length, long* out) {
  const Plan p = make_plan<T>(kv_heads, group, rows, requests, most, longest, window);
  const Cut c = cut_request<T>(tokens * group, length - first_tile(length - tokens, window), kv_heads);
  out[0] = c.splits;
  out[1] = c.groups == 0 ? c.splits : (long)c.groups * c.splits;
  out[2] = c.groups == 0 ? p.decode_splits : p.prompt_places;
  out[3] = c.splits == 1 ? 0 : (long)c.splits * tokens * group;
  out[4] = p.per_row * tokens + p.per_request;
  out[5] = p.head_entries;
}
}  // namespace ls

extern "C" int ls_fp4_attention_plan(int dtype, int rows, int requests, int kv_heads, int group, int most, int longest, int window,
                                     int tokens, int length, long* out) {
  using namespace ls;
  LS_REQUIRE((dtype == kF32 || dtype == kBF16) && rows >= 1 && requests >= 1 && kv_heads >= 1 && group >= 1 && tokens >= 1 &&
                 tokens <= most && most <= rows && length >= tokens && length <= longest && window >= 0 && (long)most * group <= 0x7fffff00l,
             "fp4_attention: no plan for a request of %d tokens and %d keys among %d rows", tokens, length, rows);
  if (dtype == kF32) plan_of<float>(rows, requests, kv_heads, group, most, longest, window, tokens, length, out);
  else plan_of<bf16_t>(rows, requests, kv_heads, group, most, longest, window, tokens, length, out);
  return 0;
}

extern "C" int ls_fp4_attention(int dtype, const void* q, long ldq, void* out, long ldo, int rows, const void* k_codes,
                                const void* k_scales, const void* v_codes, const void* v_scales, int pages, int page_size,
                                int kv_heads, int group, const int* table, int columns, const int* offsets,
                                const int* lengths, int requests, int most, int longest, float scale, int window,
                                void* scratch, long scratch_bytes, void* stream) {
  using namespace ls;
  LS_REQUIRE(dtype == kF32 || dtype == kBF16, "fp4_attention: dtype %d", dtype);
  LS_REQUIRE(rows >= 0 && pages >= 1 && kv_heads >= 1 && kv_heads <= 32767 && group >= 1 && columns >= 1 && requests >= 1 &&
                 requests <= 65535 && most >= 0 && longest >= 0 && window >= 0 && ldq >= 0 && ldo >= 0,
             "fp4_attention: %d rows of %d requests, %d heads by %d, %d pages, %d columns", rows, requests, kv_heads, group,
             pages, columns);
  LS_REQUIRE(page_size >= 4 && (page_size & (page_size - 1)) == 0, "fp4_attention: pages of %d tokens", page_size);
  LS_REQUIRE((long)kv_heads * page_size * (D / 2) <= 0x7fffffffl, "fp4_attention: pages of %d heads of %d tokens", kv_heads, page_size);
  LS_REQUIRE(most <= rows && (long)most * group <= 0x7fffff00l && longest <= 0x7fff0000, "fp4_attention: %d rows a request, %d keys", most, longest);
  if (rows == 0 || most == 0) return 0;
  Fp4Args a;
  a.q = q; a.ldq = ldq; a.out = out; a.ldo = ldo;
  a.pool = Fp4Pool{static_cast<const unsigned char*>(k_codes), static_cast<const unsigned char*>(k_scales),
                   static_cast<const unsigned char*>(v_codes), static_cast<const unsigned char*>(v_scales), pages,
                   __builtin_ctz((unsigned)page_size), kv_heads};
  a.table = table; a.columns = columns; a.offsets = offsets; a.lengths = lengths; a.requests = requests; a.rows = rows;
  a.group = group; a.window = window; a.most = most; a.longest = longest;
  a.factor = fmaxf(fabsf(scale) * kToLog2, 1.1754944e-38f);  // (never 0: a masked score stays -inf times it)
  a.negative = scale < 0.f;
  return dtype == kF32 ? run_fp4<float>(a, most, longest, scratch, scratch_bytes, (hipStream_t)stream)
                       : run_fp4<bf16_t>(a, most, longest, scratch, scratch_bytes, (hipStream_t)stream);
}
