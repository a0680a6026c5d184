// Block tables and slot maps of a step, built on the device from what every request holds and brings.
//
// For request i with h_i tokens held and n_i new ones (page size p, block tables of `columns` entries):
//   need_i  = ceil((h_i + n_i) / p) - ceil(h_i / p)             pages it has to be given
//   first_i = cursor + need_0 + ... + need_(i-1)                where they begin in the free list
// It is taken into the step if 0 <= h_i, 0 <= n_i, h_i + n_i <= columns * p, need_i = 0 or first_i + need_i <= free
// pages, and its tokens end within the room of the outputs.  Both limits are reached for good: behind the first request
// that does not fit, none that needs a page (a row) is taken, so the pages that are given out are a run of the free
// list.  Then, offsets_i = n_0 + ... + n_(i-1) over the requests taken, and token t of request i
//   position = h_i + t - offsets_i,   slot = page * p + position % p  (-1 where the table has no page there).
//
// What bounds it: nothing but latency; the bytes are those of a few rows.  Every workgroup adds up all requests by
// itself (two sums over at most kMaxRequests numbers that stay in LDS), so there is one launch and no workgroup waits
// for another; then it takes its run of tokens, each of which finds its request by bisection in LDS.  A token that is
// the first of a page writes that page's entry of the block table, and no token reads an entry that this call writes:
// the pages given out are found from the free list.  Sums are held in 64 bits.  64 requests of a token take 4.7 us, 256 that
// bring 48,600 tokens 5.6, of which the smallest launch is 2.4.

#include "common.h"
#include "serving_api.h"

namespace ls {

constexpr int kTableThreads = 256;
constexpr int kTableWaves = kTableThreads / 64;
constexpr int kMaxRequests = 8192;  // two 32-bit numbers a request in LDS

__device__ __forceinline__ long long wave_scan(long long v) {  // inclusive, over the 64 lanes
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const long long other = __shfl_up(v, off);
    if ((int)(threadIdx.x & 63) >= off) v += other;
  }
  return v;
}

// Exclusive sum over the workgroup's threads; `total` gets the whole sum.
__device__ __forceinline__ long long block_scan(long long v, long long* __restrict__ wave_sums, long long& total) {
  const long long inclusive = wave_scan(v);
  __syncthreads();  // wave_sums may still be read from the call before
  if ((threadIdx.x & 63) == 63) wave_sums[threadIdx.x >> 6] = inclusive;
  __syncthreads();
  long long before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kTableWaves; ++w) {
    if (w < (int)(threadIdx.x >> 6)) before += wave_sums[w];
    total += wave_sums[w];
  }
  return before + inclusive - v;
}

// kEach: requests a thread adds up, their numbers in registers; 0: any, read again in every loop.
template <int kEach>
__global__ __launch_bounds__(kTableThreads) void step_tables_kernel(
    const int* __restrict__ lengths, const int* __restrict__ news, int requests, int* table, int columns, int page_shift,
    const int* __restrict__ free_pages, int free_count, const int* __restrict__ cursor, int* __restrict__ slots,
    int* __restrict__ tok_seq, int* __restrict__ tok_pos, int tokens, int* __restrict__ offsets,
    int* __restrict__ new_lengths, int* __restrict__ progress) {
  extern __shared__ int held_in_lds[];
  int* begin = held_in_lds;                 // [requests + 1] first row of every request
  int* first_page = begin + requests + 1;   // [requests] where its new pages begin in the free list
  __shared__ long long wave_sums[kTableWaves];
  __shared__ int4 totals[kTableWaves];
  const int t = threadIdx.x;
  const int each = kEach ? kEach : (requests + kTableThreads - 1) / kTableThreads;  // neighbouring requests a thread adds up
  const int lo = min(requests, t * each), hi = min(requests, lo + each);
  const long long room = (long long)columns << page_shift;
  const long long round = (1ll << page_shift) - 1;
  int kept_have[kEach ? kEach : 1], kept_fresh[kEach ? kEach : 1];
  if constexpr (kEach > 0) {
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      kept_have[k] = lo + k < hi ? lengths[lo + k] : -1;
      kept_fresh[k] = lo + k < hi ? news[lo + k] : 0;
    }
  }
  const long long start = cursor[0];

  // body(request, tokens held, new ones, pages needed; -1 where it does not fit its block table)
  const auto each_request = [&](auto body) LS_INLINED {
    const auto one = [&](int i, long long have, long long fresh) LS_INLINED {
      const bool fits = have >= 0 && fresh >= 0 && have + fresh <= room;
      body(i, have, fresh, fits ? ((have + fresh + round) >> page_shift) - ((have + round) >> page_shift) : -1ll);
    };
    if constexpr (kEach > 0) {
#pragma unroll
      for (int k = 0; k < kEach; ++k)
        if (lo + k < hi) one(lo + k, kept_have[k], kept_fresh[k]);
    } else {
      for (int i = lo; i < hi; ++i) one(i, lengths[i], news[i]);
    }
  };
  long long mine = 0, all;
  each_request([&](int, long long, long long, long long need) LS_INLINED { mine += need > 0 ? need : 0; });
  long long at = start + block_scan(mine, wave_sums, all);
  // which requests get their pages, and how many rows those bring
  mine = 0;
  each_request([&](int i, long long, long long fresh, long long need) LS_INLINED {
    const bool taken = need == 0 || (need > 0 && start >= 0 && at + need <= free_count);
    begin[i] = taken ? (int)fresh : -1;
    first_page[i] = taken && need > 0 ? (int)at : 0;
    if (need > 0) at += need;
    if (taken) mine += fresh;
  });
  long long row = block_scan(mine, wave_sums, all);
  long long pages = 0, refused = 0, rows = 0;
  each_request([&](int i, long long have, long long, long long need) LS_INLINED {
    const long long n = begin[i];
    const bool taken = n == 0 || (n > 0 && row + n <= tokens);
    begin[i] = (int)min(row, (long long)tokens);
    if (n > 0) row += n;
    if (taken) {
      pages += need > 0 ? need : 0;
      rows += n;
    } else {
      ++refused;
    }
    if (blockIdx.x == 0) new_lengths[i] = (int)have + (taken ? (int)n : 0);
  });
  // The rows of the requests taken are one run from row 0 on, so the rows behind them are where that run ends; a request
  // that is refused for its rows begins and ends there.  (What is taken fits 31 bits: it fits the outputs and the list.)
  {
    const int r = wave_sum((int)rows), p = wave_sum((int)pages), f = wave_sum((int)refused);
    if ((t & 63) == 0) totals[t >> 6] = make_int4(r, p, f, 0);
  }
  __syncthreads();
  int used = 0, pages_all = 0, refused_all = 0;
#pragma unroll
  for (int w = 0; w < kTableWaves; ++w) {
    used += totals[w].x;
    pages_all += totals[w].y;
    refused_all += totals[w].z;
  }
  for (int i = lo; i < hi; ++i) begin[i] = min(begin[i], used);
  if (t == 0) begin[requests] = used;
  if (blockIdx.x == 0) {
    if (t == 0) {
      progress[0] = (int)start + pages_all;
      progress[1] = refused_all;
      offsets[requests] = used;
    }
    for (int i = lo; i < hi; ++i) offsets[i] = begin[i];
  }
  __syncthreads();

  for (long long j = (long long)blockIdx.x * kTableThreads + t; j < tokens; j += (long long)gridDim.x * kTableThreads) {
    if (j >= used) {
      slots[j] = -1; tok_seq[j] = -1; tok_pos[j] = -1;
      continue;
    }
    int a = 0, b = requests;  // begin[a] <= j < begin[b]: the last request that begins at or before row j
    while (b - a > 1) {
      const int m = (a + b) >> 1;
      if (begin[m] <= j) a = m; else b = m;
    }
    const int have = lengths[a];
    const int position = have + ((int)j - begin[a]);
    const int held_pages = (int)(((long long)have + round) >> page_shift);
    const int column = position >> page_shift;
    int page;
    if (column >= held_pages) {
      page = free_pages[first_page[a] + (column - held_pages)];
      if ((position & (int)round) == 0) table[(long)a * columns + column] = page;
    } else {
      page = table[(long)a * columns + column];
    }
    const long long slot = ((long long)page << page_shift) + (position & (int)round);
    slots[j] = page >= 0 && slot <= 0x7fffffffll ? (int)slot : -1;
    tok_seq[j] = a;
    tok_pos[j] = position;
  }
}

}  // namespace ls

LS_DEFINE_ERROR_API

extern "C" int ls_step_tables_max_requests() { return ls::kMaxRequests; }

extern "C" int ls_step_tables(const int* lengths, const int* news, int requests, int* table, int columns, int page_size,
                              const int* free_pages, int free_count, const int* cursor, int* slots, int* tok_seq,
                              int* tok_pos, int tokens, int* offsets, int* new_lengths, int* progress, void* stream) {
  using namespace ls;
  LS_REQUIRE(requests >= 0 && requests <= kMaxRequests && columns >= 1 && free_count >= 0 && tokens >= 0,
             "step_tables: %d requests, %d columns, %d free pages, %d tokens", requests, columns, free_count, tokens);
  LS_REQUIRE(page_size >= 4 && (page_size & (page_size - 1)) == 0, "step_tables: pages of %d tokens", page_size);
  LS_REQUIRE((long)columns * page_size <= 0x7fffffffl, "step_tables: positions beyond 31 bits");
  const int shift = __builtin_ctz((unsigned)page_size);
  // a workgroup adds up all requests before its first token: with many requests it takes more tokens
  const int run = requests > 1024 ? 4 * kTableThreads : kTableThreads;
  const int groups = tokens > run ? (tokens + run - 1) / run : 1;
  const size_t lds = sizeof(int) * (2 * (size_t)requests + 1);
  auto* kernel = requests <= kTableThreads ? step_tables_kernel<1> : requests <= 4 * kTableThreads ? step_tables_kernel<4> : step_tables_kernel<0>;
  if (lds + 128 > 64 * 1024) {
    hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024 - 1024);
    LS_REQUIRE(e == hipSuccess, "step_tables: %s", hipGetErrorString(e));
  }
  kernel<<<groups < 1024 ? groups : 1024, kTableThreads, lds, (hipStream_t)stream>>>(
      lengths, news, requests, table, columns, shift, free_pages, free_count, cursor, slots, tok_seq, tok_pos, tokens,
      offsets, new_lengths, progress);
  return check_launch("step_tables");
}
