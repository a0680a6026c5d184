// Keys and values into pages of 4 bits and back (layout and number format: fp4.h).
//
// What bounds both: the bytes, once in and once out.  A thread has eight neighbouring elements of one head of one token (16
// or 32 bytes), four threads a group of 32, whose largest magnitude goes round by register exchanges.  The order of the
// threads puts four neighbouring tokens of a head into one wave: their values share blocks of four tokens, so where the
// slots are neighbours too a wave stores whole runs of 256 bytes.  Slots may come in any order; what a slot holds does not
// depend on what else is written (two rows of one call with the same slot: either may stay, element by element).
// 8,209 tokens of 8 heads of 128 in float32 (76 MB in and out): written in 13 us, 5.8 TB/s, read back in 9.4.

#include "fp4.h"
#include "serving_api.h"

namespace ls {

constexpr int kPagesThreads = 256;

typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned int u32x4_any __attribute__((ext_vector_type(4), aligned(2)));

__device__ __forceinline__ void load8(float (&x)[8], const float* __restrict__ p) {
  const f32x4_any a = *reinterpret_cast<const f32x4_any*>(p), b = *reinterpret_cast<const f32x4_any*>(p + 4);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    x[e] = a[e];
    x[4 + e] = b[e];
  }
}
__device__ __forceinline__ void load8(float (&x)[8], const bf16_t* __restrict__ p) {
  const u32x4_any a = *reinterpret_cast<const u32x4_any*>(p);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    x[2 * e] = __uint_as_float(a[e] << 16);
    x[2 * e + 1] = __uint_as_float(a[e] & 0xffff0000u);
  }
}
__device__ __forceinline__ void store8(float* p, const float (&x)[8]) {
  *reinterpret_cast<f32x4_any*>(p) = f32x4_any{x[0], x[1], x[2], x[3]};
  *reinterpret_cast<f32x4_any*>(p + 4) = f32x4_any{x[4], x[5], x[6], x[7]};
}
__device__ __forceinline__ void store8(bf16_t* p, const float (&x)[8]) {
  u32x4_any a;
#pragma unroll
  for (int e = 0; e < 4; ++e)  // every value but NaN is exact in bfloat16, and the NaN's upper half is one too
    a[e] = (__float_as_uint(x[2 * e]) >> 16) | (__float_as_uint(x[2 * e + 1]) & 0xffff0000u);
  *reinterpret_cast<u32x4_any*>(p) = a;
}

struct Where {  // a thread's octet of a head of a token
  int token, head, octet;
};

// Threads in the order [block of four tokens][head][token][octet]; false behind the last token.
__device__ __forceinline__ bool find_octet(Where& w, long i, int tokens, int heads, int octets) {
  w.octet = (int)(i % octets);
  i /= octets;
  const int sub = (int)(i & 3);
  i >>= 2;
  w.head = (int)(i % heads);
  i /= heads;
  const long token = 4 * i + sub;
  w.token = (int)min(token, (long)tokens - 1);
  return token < tokens;
}

struct Place {  // where an octet lies in the pool
  long k_code, k_scale, v_code, v_scale;
};
__device__ __forceinline__ Place find_place(int slot, int page_shift, int head, int octet, int heads, int octets) {
  const long row = ((long)(slot >> page_shift) * heads + head) << page_shift;  // the head's first token of the page
  const int token = slot & ((1 << page_shift) - 1), groups = octets / 4;
  const long block = (row + token) >> 2;
  Place p;
  p.k_code = ((row + token) * octets + octet) * 4;
  p.k_scale = (row + token) * groups + octet / 4;
  p.v_code = (block * octets + octet) * 16 + (token & 3) * 4;
  p.v_scale = (block * groups + octet / 4) * 4 + (token & 3);
  return p;
}

// The codes of eight elements of a group and the group's scale byte; all four lanes of the group together.
__device__ __forceinline__ unsigned int quantise(const float (&x)[8], unsigned int& byte) {
  // magnitudes as whole numbers: their order is the same, and infinities and NaN are the largest
  unsigned int largest = 0u;
#pragma unroll
  for (int e = 0; e < 8; ++e) largest = max(largest, __float_as_uint(x[e]) & 0x7fffffffu);
  largest = max(largest, (unsigned int)__builtin_amdgcn_update_dpp(0, (int)largest, 0xB1, 0xf, 0xf, true));
  largest = max(largest, (unsigned int)__builtin_amdgcn_update_dpp(0, (int)largest, 0x4E, 0xf, 0xf, true));
  const int exponent = (int)(largest >> 23);  // floor(log2) + 127; 0 for the numbers below 2^-126
  byte = (unsigned int)max(exponent - 2, 2);
  if (exponent == 255) {
    byte = kFp4Nan;
    return 0u;
  }
  const float scale = fp4_scale(byte);
  unsigned int codes = 0u;
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[0], x[1], scale, 0);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[2], x[3], scale, 1);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[4], x[5], scale, 2);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[6], x[7], scale, 3);
  return codes;
}

template <typename T>
__global__ __launch_bounds__(kPagesThreads) void fp4_write_kernel(const T* __restrict__ k, long ldk, const T* __restrict__ v,
                                                                  long ldv, const int* __restrict__ slots, int tokens,
                                                                  int heads, int octets, unsigned char* k_codes,
                                                                  unsigned char* k_scales, unsigned char* v_codes,
                                                                  unsigned char* v_scales, long room, int page_shift) {
  Where w;
  const bool inside = find_octet(w, (long)blockIdx.x * kPagesThreads + threadIdx.x, tokens, heads, octets);
  const int slot = slots[w.token];
  // the four threads of a group agree on this: they have the same token
  if (!inside || slot < 0 || slot >= room) return;
  const long from = (long)w.head * octets * 8 + w.octet * 8;
  float x[8], y[8];
  load8(x, k + w.token * ldk + from);
  load8(y, v + w.token * ldv + from);
  unsigned int k_byte, v_byte;
  const unsigned int k_word = quantise(x, k_byte), v_word = quantise(y, v_byte);
  const Place p = find_place(slot, page_shift, w.head, w.octet, heads, octets);
  *reinterpret_cast<unsigned int*>(k_codes + p.k_code) = k_word;
  *reinterpret_cast<unsigned int*>(v_codes + p.v_code) = v_word;
  if ((w.octet & 3) == 0) {
    k_scales[p.k_scale] = (unsigned char)k_byte;
    v_scales[p.v_scale] = (unsigned char)v_byte;
  }
}

__device__ __forceinline__ void values_of(float (&x)[8], unsigned int codes, unsigned int byte) {
  const float scale = fp4_scale(byte);
  const unsigned int pair[4] = {fp4_pair<0>(codes, scale), fp4_pair<1>(codes, scale), fp4_pair<2>(codes, scale),
                                fp4_pair<3>(codes, scale)};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    x[2 * e] = byte == kFp4Nan ? __uint_as_float(0x7fc00000u) : __uint_as_float(pair[e] << 16);
    x[2 * e + 1] = byte == kFp4Nan ? __uint_as_float(0x7fc00000u) : __uint_as_float(pair[e] & 0xffff0000u);
  }
}

template <typename T>
__global__ __launch_bounds__(kPagesThreads) void fp4_read_kernel(T* __restrict__ k, long ldk, T* __restrict__ v, long ldv,
                                                                 const int* __restrict__ slots, int tokens, int heads,
                                                                 int octets, const unsigned char* __restrict__ k_codes,
                                                                 const unsigned char* __restrict__ k_scales,
                                                                 const unsigned char* __restrict__ v_codes,
                                                                 const unsigned char* __restrict__ v_scales, long room,
                                                                 int page_shift) {
  Where w;
  const bool inside = find_octet(w, (long)blockIdx.x * kPagesThreads + threadIdx.x, tokens, heads, octets);
  const int slot = slots[w.token];
  if (!inside || slot < 0 || slot >= room) return;
  const long to = (long)w.head * octets * 8 + w.octet * 8;
  const Place p = find_place(slot, page_shift, w.head, w.octet, heads, octets);
  float x[8];
  values_of(x, *reinterpret_cast<const unsigned int*>(k_codes + p.k_code), k_scales[p.k_scale]);
  store8(k + w.token * ldk + to, x);
  values_of(x, *reinterpret_cast<const unsigned int*>(v_codes + p.v_code), v_scales[p.v_scale]);
  store8(v + w.token * ldv + to, x);
}

inline int check_pages(const char* what, int dtype, int tokens, int kv_heads, int dim, int pages, int page_size, long ldk, long ldv) {
  LS_REQUIRE(dtype == kF32 || dtype == kBF16, "%s: dtype %d", what, dtype);
  LS_REQUIRE(dim >= 32 && dim % 32 == 0 && dim <= 256 && kv_heads >= 1 && kv_heads <= 65536 && tokens >= 0 && pages >= 1,
             "%s: %d tokens, %d heads of %d, %d pages", what, tokens, kv_heads, dim, pages);
  LS_REQUIRE(page_size >= 4 && (page_size & (page_size - 1)) == 0, "%s: pages of %d tokens", what, page_size);
  LS_REQUIRE(ldk >= 0 && ldv >= 0, "%s: row strides %ld, %ld", what, ldk, ldv);
  const long groups = ((tokens + 3l) / 4 * 4 * kv_heads * (dim / 8) + kPagesThreads - 1) / kPagesThreads;
  LS_REQUIRE(groups * kPagesThreads <= 0xffffffffl, "%s: %d tokens of %d heads", what, tokens, kv_heads);  // (a grid's limit)
  return 0;
}

}  // namespace ls

extern "C" int ls_fp4_write(int dtype, const void* k, long ldk, const void* v, long ldv, const int* slots, int tokens,
                            int kv_heads, int dim, void* k_codes, void* k_scales, void* v_codes, void* v_scales, int pages,
                            int page_size, void* stream) {
  using namespace ls;
  const int bad = check_pages("fp4_write", dtype, tokens, kv_heads, dim, pages, page_size, ldk, ldv);
  if (bad || tokens == 0) return bad;
  const int octets = dim / 8, shift = __builtin_ctz((unsigned)page_size);
  const unsigned groups = (unsigned)(((tokens + 3l) / 4 * 4 * kv_heads * octets + kPagesThreads - 1) / kPagesThreads);
  const long room = (long)pages << shift;
  auto* kc = static_cast<unsigned char*>(k_codes);
  auto* ks = static_cast<unsigned char*>(k_scales);
  auto* vc = static_cast<unsigned char*>(v_codes);
  auto* vs = static_cast<unsigned char*>(v_scales);
  if (dtype == kF32)
    fp4_write_kernel<float><<<groups, kPagesThreads, 0, (hipStream_t)stream>>>(
        static_cast<const float*>(k), ldk, static_cast<const float*>(v), ldv, slots, tokens, kv_heads, octets, kc, ks, vc, vs,
        room, shift);
  else
    fp4_write_kernel<bf16_t><<<groups, kPagesThreads, 0, (hipStream_t)stream>>>(
        static_cast<const bf16_t*>(k), ldk, static_cast<const bf16_t*>(v), ldv, slots, tokens, kv_heads, octets, kc, ks, vc,
        vs, room, shift);
  return check_launch("fp4_write");
}

extern "C" int ls_fp4_read(int dtype, void* k, long ldk, void* v, long ldv, const int* slots, int tokens, int kv_heads,
                           int dim, const void* k_codes, const void* k_scales, const void* v_codes, const void* v_scales,
                           int pages, int page_size, void* stream) {
  using namespace ls;
  const int bad = check_pages("fp4_read", dtype, tokens, kv_heads, dim, pages, page_size, ldk, ldv);
  if (bad || tokens == 0) return bad;
  const int octets = dim / 8, shift = __builtin_ctz((unsigned)page_size);
  const unsigned groups = (unsigned)(((tokens + 3l) / 4 * 4 * kv_heads * octets + kPagesThreads - 1) / kPagesThreads);
  const long room = (long)pages << shift;
  const auto* kc = static_cast<const unsigned char*>(k_codes);
  const auto* ks = static_cast<const unsigned char*>(k_scales);
  const auto* vc = static_cast<const unsigned char*>(v_codes);
  const auto* vs = static_cast<const unsigned char*>(v_scales);
  if (dtype == kF32)
    fp4_read_kernel<float><<<groups, kPagesThreads, 0, (hipStream_t)stream>>>(
        static_cast<float*>(k), ldk, static_cast<float*>(v), ldv, slots, tokens, kv_heads, octets, kc, ks, vc, vs, room, shift);
  else
    fp4_read_kernel<bf16_t><<<groups, kPagesThreads, 0, (hipStream_t)stream>>>(
        static_cast<bf16_t*>(k), ldk, static_cast<bf16_t*>(v), ldv, slots, tokens, kv_heads, octets, kc, ks, vc, vs, room,
        shift);
  return check_launch("fp4_read");
}
