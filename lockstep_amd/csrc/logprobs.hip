// Log probabilities of given tokens, with the entropy of the distribution, the token's rank and the first alternatives.
//
// For a row x of `vocab` logits and a token t, with m = max x, S = sum e^(x - m), T = sum e^(x - m) (x - m):
//   logprob = (x_t - m) - log S,   entropy = log S - T / S,
//   rank    = how many tokens come before t in the order "larger logit first, then lower id",
//   top     = the first k tokens of that order, each with its log probability.
//
// What bounds it: reading the row once.  A row is cut into pieces of 2,048 neighbouring logits, a piece is a wave's: a
// lane takes vectors of 16 bytes, 64 vectors apart, and has its 32 logits in registers for the maximum first and the sums
// then, so a piece costs one maximum and one rescaling a lane and the row is read once.  Everything is held a lane (m, S,
// T) and a lane's pieces are folded in the order of a stream: piece i belongs to stream i mod 8.  Only at the end are a
// stream's lanes folded and the streams after one another.  So the order of every sum depends on the row's
// length alone: with many rows a workgroup of eight waves takes a row, a wave a stream; with few rows every piece is a
// wave of its own that leaves its lanes' (m, S, T), and a second launch folds them; rows of one or two pieces, and many rows of
// up to eight, go to a wave each -- the same bits.
//
// The alternatives come without a sort.  The lanes' maxima of every piece are kept; the k-th largest of 128 maxima over
// disjoint parts of the row is a bound that the k first tokens reach (each of those parts holds one that does), and only
// the lanes that reach it, some k of them, are read again.  Where more tokens reach it than there is room for, those above it
// are taken and then the equal ones from the row's start on (rows that are masked but for a few tokens); rows where that is
// no use either (ascending logits) and rows with an infinity or a NaN go by the digits of the k-th key, which reads the row
// a dozen times.  A NaN counts as larger than all numbers, -0 as 0.

#include "common.h"
#include "serving_api.h"

#include <algorithm>

namespace ls {

constexpr int kPiece = 2048;
constexpr int kLaneElems = kPiece / 64;
constexpr int kStreams = 8;
constexpr int kRowThreads = kStreams * 64;
constexpr int kMaxPieces = 256;
constexpr int kMaxVocab = kPiece * kMaxPieces;
constexpr int kMaxTop = 32;
constexpr int kParts = 128;       // disjoint parts of the row whose maxima give the bound
constexpr int kMaxSets = 64;      // a wave's lanes of pieces that are read again
constexpr int kMaxFound = 64;     // a wave's tokens that reach the bound

constexpr float kLog2e = 1.4426950408889634f;

struct LaneSums {
  float m, s, t;
};

__device__ __forceinline__ unsigned int logit_key(float f) {  // ascending; -0 counts as 0, every NaN as the largest
  const unsigned int b = __float_as_uint(f + 0.0f);
  if (f != f) return 0xffffffffu;
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

__device__ __forceinline__ float key_logit(unsigned int key) {  // (0 for -0)
  return __uint_as_float((key & 0x80000000u) ? key & 0x7fffffffu : ~key);
}

__device__ __forceinline__ LaneSums fold_sums(const LaneSums& a, const LaneSums& b) {
  const float m = fmaxf(a.m, b.m);
  LaneSums r{m, 0.f, 0.f};
  // a side without any weight (nothing yet, or only logits of -inf) adds nothing; NaN weights do.  (Behind a distance of
  // 1e4 nothing is left of a side, and a greater one would make 0 times an infinity of it.)
  if (a.s != 0.f) {
    const float d = fmaxf(a.m - m, -1e4f), f = __builtin_amdgcn_exp2f(d * kLog2e);
    r.s = a.s * f;
    r.t = f * fmaf(a.s, d, a.t);
  }
  if (b.s != 0.f) {
    const float d = fmaxf(b.m - m, -1e4f), f = __builtin_amdgcn_exp2f(d * kLog2e);
    r.s = fmaf(b.s, f, r.s);
    r.t = fmaf(f, fmaf(b.s, d, b.t), r.t);
  }
  return r;
}

template <typename T> struct Row;
template <> struct Row<float> {
  static constexpr int VEC = 4;
  typedef float vec_t __attribute__((ext_vector_type(4), aligned(4)));
};
template <> struct Row<bf16_t> {
  static constexpr int VEC = 8;
  typedef unsigned int vec_t __attribute__((ext_vector_type(4), aligned(2)));
};

// The lane's 32 logits of a piece as floats; -inf behind the row's end.
// VEC: neighbouring logits a lane has (1 where rows are so short that vectors would leave lanes without any); kElems: how many in all.
template <typename T, int VEC = Row<T>::VEC, int kElems = kLaneElems>
__device__ __forceinline__ void load_piece(float (&x)[kElems], const T* __restrict__ row, int piece, int vocab, int lane) {
  const int base = piece * kPiece;
  if (VEC > 1 && base + kPiece <= vocab) {  // uniform
    typename Row<T>::vec_t raw[kLaneElems / Row<T>::VEC];
#pragma unroll
    for (int i = 0; i < kLaneElems / Row<T>::VEC; ++i)
      raw[i] = *reinterpret_cast<const typename Row<T>::vec_t*>(row + base + (i * 64 + lane) * Row<T>::VEC);
#pragma unroll
    for (int i = 0; i < kLaneElems / Row<T>::VEC; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (sizeof(T) == 4) {
          x[i * 4 + e] = raw[i][e];
        } else {
          x[i * 8 + 2 * e] = __uint_as_float(raw[i][e] << 16);
          x[i * 8 + 2 * e + 1] = __uint_as_float(raw[i][e] & 0xffff0000u);
        }
      }
  } else {
#pragma unroll
    for (int i = 0; i < kElems / VEC; ++i)
      if (base + i * 64 * VEC < vocab) {  // (uniform)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const int at = base + (i * 64 + lane) * VEC + e;
          const float v = to_f32(row[min(at, vocab - 1)]);
          x[i * VEC + e] = at < vocab ? v : -INFINITY;
        }
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) x[i * VEC + e] = -INFINITY;
      }
  }
}

// The piece's sums of a lane, and (uniform) how many of the piece's tokens come before the token `given` of logit `mine`.
// kWhole: the piece ends inside the row; else vectors behind the row's end are left out.
template <typename T, bool kWhole, int VEC = Row<T>::VEC, int kElems = kLaneElems>
__device__ __forceinline__ LaneSums piece_sums(const float (&x)[kElems], int piece, int vocab, int given, float mine, int& before, int lane) {
  constexpr int kVecs = kElems / VEC;
  const int base = piece * kPiece;
  const auto here = [&](int v) LS_INLINED -> bool { return kWhole || base + v * 64 * VEC < vocab; };  // (uniform)
  LaneSums r;
  r.m = x[0];
#pragma unroll
  for (int v = 0; v < kVecs; ++v)
    if (here(v)) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) r.m = fmaxf(r.m, x[v * VEC + e]);
    }
  const float ref = r.m == -INFINITY ? 0.f : r.m;
  r.s = 0.f;
  r.t = 0.f;
#pragma unroll
  for (int v = 0; v < kVecs; ++v)
    if (here(v)) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float d = x[v * VEC + e] - ref;
        const float w = __builtin_amdgcn_exp2f(d * kLog2e);
        r.s = r.s + w;
        r.t = fmaf(w, fmaxf(d, -1e4f), r.t);  // (a logit of -inf: 0 times a number)
      }
    }
  // A NaN compares false with everything, so "not smaller" counts it as larger.
  const auto count = [&](auto comes_before) LS_INLINED {
#pragma unroll
    for (int v = 0; v < kVecs; ++v)
      if (here(v)) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) before += __popcll(__ballot(comes_before(x[v * VEC + e], base + (v * 64 + lane) * VEC + e)));
      }
  };
  if (base > given) count([&](float l, int) LS_INLINED { return !(l <= mine); });  // (uniform) equal logits of this piece come later
  else if (base + kPiece <= given) count([&](float l, int) LS_INLINED { return !(l < mine); });  // or before
  else count([&](float l, int at) LS_INLINED { return at < given ? !(l < mine) : !(l <= mine); });
  return r;
}

template <typename T>
__device__ __forceinline__ LaneSums sums_of_piece(const float (&x)[kLaneElems], int piece, int vocab, int given, float mine, int& before, int lane) {
  if ((piece + 1) * kPiece <= vocab) return piece_sums<T, true>(x, piece, vocab, given, mine, before, lane);  // (uniform)
  return piece_sums<T, false>(x, piece, vocab, given, mine, before, lane);
}

// The sums of the wave's lanes, the same in every lane.
__device__ __forceinline__ LaneSums fold_lanes(const LaneSums& mine) {
  const float m = wave_max(mine.m);
  const float d = fmaxf(mine.m - m, -1e4f), f = __builtin_amdgcn_exp2f(d * kLog2e);  // (no logit yet: 0 times a number)
  return LaneSums{m, wave_sum(mine.s * f), wave_sum(f * fmaf(mine.s, d, mine.t))};
}

struct FinishShared {
  float m[kStreams], s[kStreams], t[kStreams];
  int before[kStreams];
  alignas(16) unsigned int part[kParts];
  int smaller[4][kParts];
  unsigned int bound;
  int set_list[kStreams][kMaxSets];
  int found[kStreams];              // a wave's tokens that reach the bound; more than kMaxFound: too many
  unsigned int key[kStreams * kMaxFound];
  int id[kStreams * kMaxFound];
  int digits[kStreams][16];
  int wave_count[kStreams];
};

// What the wave's lanes have written to LDS is there for its other lanes.
__device__ __forceinline__ void wave_handover() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Exclusive sum over the workgroup's threads; `total` gets the whole sum.
__device__ __forceinline__ int row_scan(int v, int* __restrict__ wave_sums, int& total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  int inclusive = v;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int other = __shfl_up(inclusive, off);
    if (lane >= off) inclusive += other;
  }
  __syncthreads();  // wave_sums may still be read from the call before
  if (lane == 63) wave_sums[w] = inclusive;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int k = 0; k < kStreams; ++k) {
    if (k < w) before += wave_sums[k];
    total += wave_sums[k];
  }
  return before + inclusive - v;
}

// The first k tokens of the row in sh.key / sh.id by the digits of the k-th key: a workgroup of kRowThreads.
template <typename T>
__device__ __forceinline__ int find_by_digits(FinishShared& sh, const T* __restrict__ row, int vocab, int top) {
  const int t = threadIdx.x;
  unsigned int prefix = 0;
  int want = top;  // the place of the key looked for among the keys with this prefix
  for (int shift = 28; shift >= 0; shift -= 4) {
    int count[16];
#pragma unroll
    for (int d = 0; d < 16; ++d) count[d] = 0;
    for (int i = t; i < vocab; i += kRowThreads) {
      const unsigned int key = logit_key(to_f32(row[i]));
      const unsigned int digit = shift == 28 || (key >> (shift + 4)) == prefix ? (key >> shift) & 15u : 16u;
#pragma unroll
      for (int d = 0; d < 16; ++d) count[d] += digit == (unsigned int)d ? 1 : 0;
    }
#pragma unroll
    for (int d = 0; d < 16; ++d) {
      const int n = wave_sum(count[d]);
      if ((t & 63) == 0) sh.digits[t >> 6][d] = n;
    }
    __syncthreads();
    int digit = 15, above = 0;
    for (; digit >= 0; --digit) {  // (every thread comes to the same digit)
      int n = 0;
#pragma unroll
      for (int w = 0; w < kStreams; ++w) n += sh.digits[w][digit];
      if (digit == 0 || above + n >= want) break;
      above += n;
    }
    prefix = (prefix << 4) | (unsigned int)digit;
    want -= above;
    __syncthreads();
  }
  // the keys above it, fewer than `top`, and the first `want` equal ones in the order of their ids
  int mine = 0, all;
  for (int i = t; i < vocab; i += kRowThreads) mine += logit_key(to_f32(row[i])) > prefix ? 1 : 0;
  int at = row_scan(mine, sh.wave_count, all);
  if (mine > 0)
    for (int i = t; i < vocab; i += kRowThreads) {
      const unsigned int key = logit_key(to_f32(row[i]));
      if (key > prefix && at < top) {
        sh.key[at] = key;
        sh.id[at++] = i;
      }
    }
  int ties = 0;
  for (int base = 0; base < vocab && ties < want; base += kRowThreads) {
    const int i = base + t;
    const bool tie = i < vocab && logit_key(to_f32(row[i])) == prefix;
    const int place = ties + row_scan(tie ? 1 : 0, sh.wave_count, all);
    if (tie && place < want) {
      sh.key[top - want + place] = prefix;
      sh.id[top - want + place] = i;
    }
    ties += all;
  }
  __syncthreads();
  return top;
}

// A wave lists the sets (lanes of pieces) of its own stream that reach the bound, then its tokens that do (sh.found: how many,
// kMaxFound + 1 where there are more).  `lane_key`: the key of the lane's largest logit.
template <typename T>
__device__ __forceinline__ void list_tokens(FinishShared& sh, const float* __restrict__ set_max, unsigned int lane_key, unsigned int bound,
                                            const T* __restrict__ row, int vocab, int pieces) {
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned long long below = (1ull << lane) - 1ull;
  int listed = 0, reached = 0;  // (uniform in the wave)
  if (__ballot(lane_key >= bound) != 0ull)
#pragma unroll 4
    for (int p = w; p < pieces; p += kStreams) {
      const unsigned long long hit = __ballot(logit_key(set_max[p * 64 + lane]) >= bound);
      const int at = listed + __popcll(hit & below);
      if (((hit >> lane) & 1ull) && at < kMaxSets) sh.set_list[w][at] = p * 64 + lane;
      listed += __popcll(hit);
    }
  if (listed <= kMaxSets) {
    constexpr int VEC = Row<T>::VEC;
    wave_handover();
#pragma unroll 4
    for (int i = 0; i < listed * kLaneElems; i += 64) {
      const int j = i + lane, set = sh.set_list[w][min(j / kLaneElems, listed - 1)], e = j % kLaneElems;
      const int id = (set >> 6) * kPiece + ((e / VEC) * 64 + (set & 63)) * VEC + e % VEC;
      const unsigned int key = logit_key(to_f32(row[min(id, vocab - 1)]));
      const unsigned long long hit = __ballot(j < listed * kLaneElems && id < vocab && key >= bound);
      const int at = reached + __popcll(hit & below);
      if (((hit >> lane) & 1ull) && at < kMaxFound) {
        sh.key[w * kMaxFound + at] = key;
        sh.id[w * kMaxFound + at] = id;
      }
      reached += __popcll(hit);
    }
  } else {
    reached = kMaxFound + 1;
  }
  if (lane == 0) sh.found[w] = min(reached, kMaxFound + 1);
}

// The first `want` tokens (at most 32) whose key is `key`, in the order of their ids, behind what the last list holds.  All
// lists are short of their room by that much, or this leaves them alone.
template <typename T>
__device__ __forceinline__ void first_equal(FinishShared& sh, const T* __restrict__ row, int vocab, unsigned int key, int want) {
  const int t = threadIdx.x, at = sh.found[kStreams - 1];
  __syncthreads();
  if (at + want > kMaxFound) return;  // (uniform)
  int ties = 0, all;
  for (int base = 0; base < vocab && ties < want; base += kRowThreads) {
    const int i = base + t;
    const bool tie = i < vocab && logit_key(to_f32(row[min(i, vocab - 1)])) == key;
    const int place = ties + row_scan(tie ? 1 : 0, sh.wave_count, all);
    if (tie && place < want) {
      sh.key[(kStreams - 1) * kMaxFound + at + place] = key;
      sh.id[(kStreams - 1) * kMaxFound + at + place] = i;
    }
    ties += all;
  }
  __syncthreads();
  if (t == 0) sh.found[kStreams - 1] = at + min(ties, want);
  __syncthreads();
}

// What is left when every stream's lanes have their sums: a workgroup of kRowThreads, wave w with stream w.  Rows have three pieces
// at least (shorter ones are a wave's), of which two are whole: 32 parts have logits, as many as may be wanted.
template <typename T>
__device__ __forceinline__ void finish_row(FinishShared& sh, const float* __restrict__ set_max, LaneSums mine, int before,
                                           const T* __restrict__ row, int vocab, int pieces, int given, float given_logit,
                                           int top, int r, float* __restrict__ logprob, float* __restrict__ entropy,
                                           int* __restrict__ rank, int* __restrict__ top_ids,
                                           float* __restrict__ top_logprobs) {
  const int t = threadIdx.x, lane = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6);
  const float stream_max = mine.m;
  mine = fold_lanes(mine);
  if (lane == 0) {
    sh.m[w] = mine.m; sh.s[w] = mine.s; sh.t[w] = mine.t;
    sh.before[w] = before;
  }
  __syncthreads();
  LaneSums all{sh.m[0], sh.s[0], sh.t[0]};
  int ahead = sh.before[0];
#pragma unroll
  for (int s = 1; s < kStreams; ++s) {
    all = fold_sums(all, LaneSums{sh.m[s], sh.s[s], sh.t[s]});
    ahead += sh.before[s];
  }
  const float log_sum = logf(all.s);
  const bool valid = given >= 0 && given < vocab;
  if (valid && given_logit != given_logit) {  // (uniform) before a NaN come only the NaN of lower ids
    int nan = 0;
    for (int i = t; i < given; i += kRowThreads) {
      const float x = to_f32(row[i]);
      nan += x != x ? 1 : 0;
    }
    nan = wave_sum(nan);
    __syncthreads();
    if (lane == 0) sh.before[w] = nan;
    __syncthreads();
    ahead = 0;
#pragma unroll
    for (int s = 0; s < kStreams; ++s) ahead += sh.before[s];
  }
  if (t == 0) {
    logprob[r] = valid ? (given_logit - all.m) - log_sum : __uint_as_float(0x7fc00000u);
    entropy[r] = log_sum - all.t / all.s;
    rank[r] = valid ? ahead : -1;
  }
  if (top == 0) return;

  if (all.s == all.s && all.s != 0.f) {  // finite logits but for -inf
    unsigned int part = logit_key(stream_max);  // of all the lane's sets
    const unsigned int lane_key = part;
    {
      const auto x = __builtin_amdgcn_permlane16_swap(part, part, false, false);
      part = max((unsigned int)x[0], (unsigned int)x[1]);
      const auto y = __builtin_amdgcn_permlane32_swap(part, part, false, false);
      part = max((unsigned int)y[0], (unsigned int)y[1]);
    }
    if (lane < 16) sh.part[w * 16 + lane] = part;
    __syncthreads();
    {  // how many parts are larger: a quarter of the comparisons a thread
      const int mine = t & (kParts - 1), from = (t / kParts) * (kParts / 4);
      const unsigned int key = sh.part[mine];
      int larger = 0;
#pragma unroll
      for (int i = 0; i < kParts / 4; i += 4) {
        const uint4 other = *reinterpret_cast<const uint4*>(&sh.part[from + i]);
        larger += other.x > key || (other.x == key && from + i < mine) ? 1 : 0;
        larger += other.y > key || (other.y == key && from + i + 1 < mine) ? 1 : 0;
        larger += other.z > key || (other.z == key && from + i + 2 < mine) ? 1 : 0;
        larger += other.w > key || (other.w == key && from + i + 3 < mine) ? 1 : 0;
      }
      sh.smaller[t / kParts][mine] = larger;
      __syncthreads();
      if (t < kParts && sh.smaller[0][t] + sh.smaller[1][t] + sh.smaller[2][t] + sh.smaller[3][t] == top - 1) sh.bound = key;
    }
    __syncthreads();
    const unsigned int bound = sh.bound;
    list_tokens<T>(sh, set_max, lane_key, bound, row, vocab, pieces);
  } else if (lane == 0) {
    sh.found[w] = kMaxFound + 1;
    sh.bound = 0xffffffffu;
  }
  __syncthreads();
  int found[kStreams], most = 0, listed = 0;
  const auto take_lists = [&]() LS_INLINED {
    most = listed = 0;
#pragma unroll
    for (int k = 0; k < kStreams; ++k) {
      found[k] = sh.found[k];
      most = max(most, found[k]);
      listed += found[k];
    }
  };
  take_lists();
  if (most > kMaxFound) {  // (uniform) many tokens at the bound?  Those above it, and the first of the equal ones
    const unsigned int bound = sh.bound;
    if (bound < 0xffffffffu) {
      __syncthreads();
      list_tokens<T>(sh, set_max, logit_key(stream_max), bound + 1u, row, vocab, pieces);
      __syncthreads();
      take_lists();
    }
    if (most <= kMaxFound && listed < top) {
      first_equal<T>(sh, row, vocab, bound, top - listed);
      take_lists();
    }
    if (most > kMaxFound || listed < top) {
      find_by_digits<T>(sh, row, vocab, top);
      found[0] = top;
#pragma unroll
      for (int k = 1; k < kStreams; ++k) found[k] = 0;
      most = top;
    }
  }
  // Their order: a token's place is how many of the others come before it.  Eight lanes a token, a list each.
  const int list = lane & 7;
  for (int c0 = 0; c0 < kStreams * most; c0 += kRowThreads / 8) {  // (uniform)
    const int c = c0 + (t >> 3), from = c / most, i = c - from * most;
    int limit = 0, mine = 0;
#pragma unroll
    for (int k = 0; k < kStreams; ++k) {
      limit = from == k ? found[k] : limit;
      mine = list == k ? found[k] : mine;
    }
    const bool there = from < kStreams && i < limit;
    const int at = there ? from * kMaxFound + i : 0;
    const unsigned int key = sh.key[at];
    const int id = sh.id[at];
    int place = 0;
#pragma unroll 4
    for (int k = 0; k < mine; ++k) {
      const unsigned int other = sh.key[list * kMaxFound + k];
      place += other > key || (other == key && sh.id[list * kMaxFound + k] < id) ? 1 : 0;
    }
    place += __shfl_xor(place, 1);
    place += __shfl_xor(place, 2);
    place += __shfl_xor(place, 4);
    if (there && list == 0 && place < top) {
      top_ids[(long)r * top + place] = id;
      top_logprobs[(long)r * top + place] = (key_logit(key) - all.m) - log_sum;
    }
  }
}

// A workgroup a row (many rows).
template <typename T>
__global__ __launch_bounds__(kRowThreads, 8) void logprobs_rows_kernel(const T* __restrict__ logits, long ld,
                                                                    const int* __restrict__ tokens, int vocab, int top,
                                                                    float* __restrict__ logprob, float* __restrict__ entropy,
                                                                    int* __restrict__ rank, int* __restrict__ top_ids,
                                                                    float* __restrict__ top_logprobs) {
  extern __shared__ float set_max[];  // [pieces * 64] where alternatives are asked for
  __shared__ FinishShared sh;
  const int r = blockIdx.x, lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const T* row = logits + (long)r * ld;
  const int pieces = (vocab + kPiece - 1) / kPiece;
  const int given = tokens[r];
  const float mine = given >= 0 && given < vocab ? to_f32(row[given]) : 0.f;
  LaneSums sums{-INFINITY, 0.f, 0.f};
  int before = 0;
  for (int p = w; p < pieces; p += kStreams) {
    float x[kLaneElems];
    load_piece<T>(x, row, p, vocab, lane);
    const LaneSums here = piece_sums<T, true>(x, p, vocab, given, mine, before, lane);  // (-inf behind the row's end adds nothing)
    if (top > 0) set_max[p * 64 + lane] = here.m;
    sums = fold_sums(sums, here);
  }
  finish_row<T>(sh, set_max, sums, before, row, vocab, pieces, given, mine, top, r, logprob, entropy, rank, top_ids,
                top_logprobs);
}

// A wave a piece (few rows): the lanes' sums to part[row][piece][3][64], the count to count[row][piece].
constexpr int kPieceThreads = 256;
template <typename T>
__global__ __launch_bounds__(kPieceThreads) void logprobs_pieces_kernel(const T* __restrict__ logits, long ld,
                                                                        const int* __restrict__ tokens, int vocab,
                                                                        int pieces, float* __restrict__ part,
                                                                        int* __restrict__ count) {
  const int r = blockIdx.y, lane = threadIdx.x & 63;
  const int p = blockIdx.x * (kPieceThreads / 64) + (threadIdx.x >> 6);
  if (p >= pieces) return;  // (no wave waits for another)
  const T* row = logits + (long)r * ld;
  float x[kLaneElems];
  load_piece<T>(x, row, p, vocab, lane);
  const int given = tokens[r];
  const float mine = given >= 0 && given < vocab ? to_f32(row[given]) : 0.f;
  int before = 0;
  const LaneSums here = sums_of_piece<T>(x, p, vocab, given, mine, before, lane);
  const long at = (long)r * pieces + p;
  part[at * 192 + lane] = here.m;
  part[at * 192 + 64 + lane] = here.s;
  part[at * 192 + 128 + lane] = here.t;
  if (lane == 0) count[at] = before;
}

template <typename T>
__global__ __launch_bounds__(kRowThreads, 4) void logprobs_fold_kernel(const T* __restrict__ logits, long ld,
                                                                    const int* __restrict__ tokens, int vocab, int pieces,
                                                                    const float* __restrict__ part, const int* __restrict__ count,
                                                                    int top, float* __restrict__ logprob,
                                                                    float* __restrict__ entropy, int* __restrict__ rank,
                                                                    int* __restrict__ top_ids, float* __restrict__ top_logprobs) {
  extern __shared__ float set_max[];
  __shared__ FinishShared sh;
  const int r = blockIdx.x, lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const T* row = logits + (long)r * ld;
  const int given = tokens[r];
  const float mine = given >= 0 && given < vocab ? to_f32(row[given]) : 0.f;
  LaneSums sums{-INFINITY, 0.f, 0.f};
  int before = 0;
  constexpr int kBatch = 10;  // pieces whose sums are asked for together
  for (int p0 = w; p0 < pieces; p0 += kBatch * kStreams) {
    LaneSums here[kBatch];
    int counts[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const long at = (long)r * pieces + min(p0 + k * kStreams, pieces - 1);
      here[k] = LaneSums{part[at * 192 + lane], part[at * 192 + 64 + lane], part[at * 192 + 128 + lane]};
      counts[k] = count[at];
    }
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int p = p0 + k * kStreams;
      if (p < pieces) {  // (uniform)
        before += counts[k];
        if (top > 0) set_max[p * 64 + lane] = here[k].m;
        sums = fold_sums(sums, here[k]);
      }
    }
  }
  finish_row<T>(sh, set_max, sums, before, row, vocab, pieces, given, mine, top, r, logprob, entropy, rank, top_ids,
                top_logprobs);
}

// Short rows: a wave a row, four a workgroup; no wave waits for another.  The same sums (bits) as a workgroup a row, whose streams
// have one piece at most there.  The bound is the k-th largest of the 64 lanes' maxima; the tokens that reach it are listed in
// LDS, and a lane orders two of them.  (75,000 rows of 2,000 logits in float32: 526 us a workgroup each, 155 a wave each.)
constexpr int kShortPieces = kStreams, kShortThreads = 256;
constexpr int kNarrowVocab = 512;  // up to here a lane has single logits: vectors would leave lanes without any
constexpr int kShortList = 128;
struct ShortShared {
  unsigned int key[kShortThreads / 64][kShortList];
  int id[kShortThreads / 64][kShortList];
  int sets[kShortThreads / 64][kShortList];
};

// Appends the tokens (in the order of their ids) for which `wanted(key)` holds to the wave's list; returns how many there are then,
// kShortList + 1 where there are more than room.  `most`: how many are to be taken.
template <typename T, typename F>
__device__ __forceinline__ int list_in_order(ShortShared& sh, int w, int lane, const T* __restrict__ row, int vocab, int listed, int most, F wanted) {
  const unsigned long long below = (1ull << lane) - 1ull;
  const int until = listed + most;
  for (int base = 0; base < vocab && listed < until; base += 64) {
    const int id = base + lane;
    const unsigned int key = logit_key(to_f32(row[min(id, vocab - 1)]));
    const unsigned long long hit = __ballot(id < vocab && wanted(key));
    const int at = listed + __popcll(hit & below);
    if (((hit >> lane) & 1ull) && at < until && at < kShortList) {
      sh.key[w][at] = key;
      sh.id[w][at] = id;
    }
    listed = min(until, listed + __popcll(hit));
  }
  return min(listed, kShortList + 1);
}

// kPieces: the most pieces of a row (their lanes' maxima stay in registers).  kNarrow: logits a lane has of a narrow row, or 0 (a
// million rows of 150 logits: with four 0.31 ms; with 32, most of them behind the row's end, 0.80, spent on branches over those).
template <typename T, int kNarrow, int kPieces>
__global__ __launch_bounds__(kShortThreads) void logprobs_short_kernel(const T* __restrict__ logits, long ld, const int* __restrict__ tokens,
                                                                       int rows, int vocab, int top, float* __restrict__ logprob,
                                                                       float* __restrict__ entropy, int* __restrict__ rank,
                                                                       int* __restrict__ top_ids, float* __restrict__ top_logprobs) {
  __shared__ ShortShared sh;
  constexpr int VEC = kNarrow ? 1 : Row<T>::VEC, kElems = kNarrow ? kNarrow : kLaneElems;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = blockIdx.x * (kShortThreads / 64) + w;
  if (r >= rows) return;
  const T* row = logits + (long)r * ld;
  const int pieces = (vocab + kPiece - 1) / kPiece;
  const int given = tokens[r];
  const bool valid = given >= 0 && given < vocab;
  const float given_logit = valid ? to_f32(row[given]) : 0.f;
  LaneSums all{-INFINITY, 0.f, 0.f};
  float set_max[kPieces], lane_max = -INFINITY;
  int before = 0;
#pragma unroll
  for (int p = 0; p < kPieces; ++p) {
    set_max[p] = -INFINITY;
    if (p < pieces) {  // (uniform)
      float x[kElems];
      load_piece<T, VEC, kElems>(x, row, p, vocab, lane);
      LaneSums here;
      if constexpr (kNarrow) here = piece_sums<T, false, VEC, kElems>(x, p, vocab, given, given_logit, before, lane);
      else here = sums_of_piece<T>(x, p, vocab, given, given_logit, before, lane);
      set_max[p] = here.m;
      lane_max = fmaxf(lane_max, here.m);
      all = fold_sums(all, fold_lanes(here));
    }
  }
  const float log_sum = logf(all.s);
  if (valid && given_logit != given_logit) {  // (uniform) before a NaN come only the NaN of lower ids
    before = 0;
    for (int base = 0; base < given; base += 64) {
      const float x = to_f32(row[min(base + lane, vocab - 1)]);
      before += __popcll(__ballot(base + lane < given && x != x));
    }
  }
  if (lane == 0) {
    logprob[r] = valid ? (given_logit - all.m) - log_sum : __uint_as_float(0x7fc00000u);
    entropy[r] = log_sum - all.t / all.s;
    rank[r] = valid ? before : -1;
  }
  if (top == 0) return;

  int listed = kShortList + 1;
  unsigned int bound = 0u;
  if (all.s == all.s && all.s != 0.f) {  // (uniform) finite logits but for -inf
    if (top <= 12) {  // the largest again and again
      float rest = lane_max;
      for (int got = 0; got < top;) {
        const float m = wave_max(rest);
        const unsigned long long at = __ballot(rest == m);
        got += __popcll(at);
        bound = logit_key(m);
        rest = rest == m ? -INFINITY : rest;
        if (m == -INFINITY) break;
      }
    } else {
      const unsigned int mine = logit_key(lane_max);
      int larger = 0;
#pragma unroll
      for (int i = 0; i < 64; ++i) {
        const unsigned int other = (unsigned int)__builtin_amdgcn_readlane((int)mine, i);
        larger += other > mine || (other == mine && i < lane) ? 1 : 0;
      }
      bound = (unsigned int)__builtin_amdgcn_readlane((int)mine, __ffsll((long long)__ballot(larger == top - 1)) - 1);
    }
    const unsigned long long below = (1ull << lane) - 1ull;
    int sets = 0;
#pragma unroll
    for (int p = 0; p < kPieces; ++p)
      if (p < pieces) {
        const unsigned long long hit = __ballot(logit_key(set_max[p]) >= bound);
        const int at = sets + __popcll(hit & below);
        if (((hit >> lane) & 1ull) && at < kShortList) sh.sets[w][at] = p * 64 + lane;
        sets += __popcll(hit);
      }
    if (sets <= kShortList) {
      wave_handover();
      listed = 0;
      // two sets of 32 at a time (or more of fewer); vectors behind the row's end do not count
      for (int i = 0; i < sets * kElems; i += 64) {
        const int j = i + lane, set = sh.sets[w][min(j / kElems, sets - 1)], e = j % kElems;
        const int id = (set >> 6) * kPiece + ((e / VEC) * 64 + (set & 63)) * VEC + e % VEC;
        const bool inside = j < sets * kElems && id < vocab;
        if (__ballot(inside) == 0ull) continue;
        const unsigned int key = logit_key(to_f32(row[inside ? id : 0]));
        const unsigned long long hit = __ballot(inside && key >= bound);
        const int at = listed + __popcll(hit & below);
        if (((hit >> lane) & 1ull) && at < kShortList) {
          sh.key[w][at] = key;
          sh.id[w][at] = id;
        }
        listed += __popcll(hit);
      }
    }
  }
  if (listed > kShortList) {
    // many tokens at the bound?  Those above it, and the first of the equal ones
    const int above = bound == 0u ? kShortList + 1 : list_in_order<T>(sh, w, lane, row, vocab, 0, kShortList + 1, [&](unsigned int key) LS_INLINED { return key > bound; });
    if (above > kShortList) {
      // the k-th key bit by bit: the largest value that k keys reach
      unsigned int value = 0u;
      for (int bit = 31; bit >= 0; --bit) {
        const unsigned int next = value | (1u << bit);
        int n = 0;
        for (int base = 0; base < vocab; base += 64) {
          const int id = base + lane;
          n += __popcll(__ballot(id < vocab && logit_key(to_f32(row[min(id, vocab - 1)])) >= next));
        }
        if (n >= top) value = next;
      }
      bound = value;
      listed = list_in_order<T>(sh, w, lane, row, vocab, 0, kShortList + 1, [&](unsigned int key) LS_INLINED { return key > bound; });
    } else {
      listed = above;
    }
    if (listed < top)
      listed = list_in_order<T>(sh, w, lane, row, vocab, listed, top - listed, [&](unsigned int key) LS_INLINED { return key == bound; });
  }
  wave_handover();
  // their order: a token's place is how many of the others come before it
  for (int c0 = 0; c0 < listed; c0 += 64) {  // (uniform)
    const int c = min(c0 + lane, listed - 1);
    const unsigned int key = sh.key[w][c];
    const int id = sh.id[w][c];
    int place = 0;
#pragma unroll 8
    for (int i = 0; i < listed; ++i) {
      const unsigned int other = sh.key[w][i];
      place += other > key || (other == key && sh.id[w][i] < id) ? 1 : 0;
    }
    if (c0 + lane < listed && place < top) {
      top_ids[(long)r * top + place] = id;
      top_logprobs[(long)r * top + place] = (key_logit(key) - all.m) - log_sum;
    }
  }
}

inline int logprob_pieces(int vocab) { return (vocab + kPiece - 1) / kPiece; }
// Where a wave takes a row: always those of one or two pieces; of up to eight where the rows are many (10,000 logits in float32, 20
// wanted: 512 rows 14.4 us a workgroup each, 20.9 a wave each; 1,024 rows 20.1 and 25.5, 2,048 rows 36.4 and 30.1, 15,000 rows 223
// and 150).
inline bool logprobs_short(int rows, int vocab) {
  const int pieces = logprob_pieces(vocab);
  return pieces <= 2 || (pieces <= kShortPieces && rows >= 1536);
}
// With fewer rows than compute units a workgroup a row leaves units idle; a wave a piece pays for its second launch once the
// streams have more than two pieces (8 rows of 15,000 logits: 6.5 us by rows, 7.8 by pieces; of 60,000: 9.9 and 8.4).
// (Fewer rows than that fit a grid's y.)
inline bool logprobs_by_pieces(int rows, int vocab) { return rows < compute_units() && logprob_pieces(vocab) > 2 * kStreams; }

template <typename T>
int run_logprobs(const void* logits, long ld, const int* tokens, int rows, int vocab, int top, float* logprob, float* entropy,
                 int* rank, int* top_ids, float* top_logprobs, void* scratch, hipStream_t stream) {
  const int pieces = logprob_pieces(vocab);
  const size_t lds = top > 0 ? sizeof(float) * 64 * (size_t)pieces : 0;
  const T* x = static_cast<const T*>(logits);
  // (a grid has less than 2^32 threads: rows in runs, of which all but absurd calls have one)
  const auto in_runs = [&](int run, auto launch) {
    for (long from = 0; from < rows; from += run)
      launch(x + from * ld, tokens + from, (int)std::min<long>(run, rows - from), logprob + from, entropy + from, rank + from,
             top_ids + from * top, top_logprobs + from * top);
  };
  if (logprobs_short(rows, vocab)) {
    in_runs(1 << 24, [&](const T* x, const int* tokens, int rows, float* logprob, float* entropy, int* rank, int* top_ids, float* top_logprobs) {
      const int waves = kShortThreads / 64;
      auto* kernel = vocab <= kNarrowVocab / 2 ? logprobs_short_kernel<T, kNarrowVocab / 128, 1>
                     : vocab <= kNarrowVocab   ? logprobs_short_kernel<T, kNarrowVocab / 64, 1>
                     : pieces <= 2             ? logprobs_short_kernel<T, 0, 2>
                                               : logprobs_short_kernel<T, 0, kShortPieces>;
      kernel<<<(rows + waves - 1) / waves, kShortThreads, 0, stream>>>(x, ld, tokens, rows, vocab, top, logprob, entropy, rank, top_ids,
                                                                       top_logprobs);
    });
  } else if (logprobs_by_pieces(rows, vocab)) {
    if (lds > 48 * 1024) {
      const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(logprobs_fold_kernel<T>),
                                               hipFuncAttributeMaxDynamicSharedMemorySize, 64 * 1024 + 1024);
      LS_REQUIRE(e == hipSuccess, "token_logprobs: %s", hipGetErrorString(e));
    }
    float* part = static_cast<float*>(scratch);
    int* count = reinterpret_cast<int*>(part + (size_t)rows * pieces * 192);
    const int waves = kPieceThreads / 64;
    logprobs_pieces_kernel<T><<<dim3((pieces + waves - 1) / waves, rows), kPieceThreads, 0, stream>>>(x, ld, tokens, vocab,
                                                                                                 pieces, part, count);
    logprobs_fold_kernel<T><<<rows, kRowThreads, lds, stream>>>(x, ld, tokens, vocab, pieces, part, count, top, logprob,
                                                               entropy, rank, top_ids, top_logprobs);
  } else {
    if (lds > 48 * 1024) {
      const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(logprobs_rows_kernel<T>),
                                               hipFuncAttributeMaxDynamicSharedMemorySize, 64 * 1024 + 1024);
      LS_REQUIRE(e == hipSuccess, "token_logprobs: %s", hipGetErrorString(e));
    }
    in_runs(1 << 22, [&](const T* x, const int* tokens, int rows, float* logprob, float* entropy, int* rank, int* top_ids, float* top_logprobs) {
      logprobs_rows_kernel<T><<<rows, kRowThreads, lds, stream>>>(x, ld, tokens, vocab, top, logprob, entropy, rank, top_ids, top_logprobs);
    });
  }
  return check_launch("token_logprobs");
}

}  // namespace ls

extern "C" int ls_logprobs_max_vocab() { return ls::kMaxVocab; }
extern "C" int ls_logprobs_max_top() { return ls::kMaxTop; }

extern "C" long ls_logprobs_scratch_bytes(int rows, int vocab) {
  if (rows <= 0 || vocab <= 0 || !ls::logprobs_by_pieces(rows, vocab)) return 0;
  return (long)rows * ls::logprob_pieces(vocab) * (192 + 1) * (long)sizeof(float);
}

extern "C" int ls_token_logprobs(int dtype, const void* logits, long ld, const int* tokens, int rows, int vocab, int top,
                                 float* logprob, float* entropy, int* rank, int* top_ids, float* top_logprobs,
                                 void* scratch, long scratch_bytes, void* stream) {
  using namespace ls;
  LS_REQUIRE(dtype == kF32 || dtype == kBF16, "token_logprobs: dtype %d", dtype);
  LS_REQUIRE(rows >= 1 && vocab >= 1 && vocab <= kMaxVocab && top >= 0 && top <= kMaxTop && top <= vocab && ld >= 0,
             "token_logprobs: %d rows of %d logits, %d alternatives", rows, vocab, top);
  LS_REQUIRE(scratch_bytes >= ls_logprobs_scratch_bytes(rows, vocab), "token_logprobs: %ld bytes of scratch", scratch_bytes);
  if (dtype == kF32)
    return run_logprobs<float>(logits, ld, tokens, rows, vocab, top, logprob, entropy, rank, top_ids, top_logprobs, scratch,
                               (hipStream_t)stream);
  return run_logprobs<bf16_t>(logits, ld, tokens, rows, vocab, top, logprob, entropy, rank, top_ids, top_logprobs, scratch,
                              (hipStream_t)stream);
}
