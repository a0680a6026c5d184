// The C interface of the library of attention over pages in 4 bits, one library a head size (fp4_attention.hip).
// Conventions as in core_api.h.
#pragma once

#ifdef __cplusplus
extern "C" {
#endif

const char* ls_last_error();
int ls_fp4_attention_head_dim();

// most, longest: the most rows and the most keys of any request (a request of more rows is left out, more keys count as the most).
// scratch: ls_fp4_attention_scratch_bytes(...) bytes.
long ls_fp4_attention_scratch_bytes(int dtype, int rows, int requests, int kv_heads, int group, int most, int longest, int window);
// How a request of `tokens` rows and `length` keys is cut in such a step, and what the launch has for it (host code, nothing is
// launched): out[0] its splits; its workgroups a head [1] and how many there are at most [2]; splits' sums a head that it
// leaves [3], how many have room [4], and how many the scratch holds a head [5].
int ls_fp4_attention_plan(int dtype, int rows, int requests, int kv_heads, int group, int most, int longest, int window, int tokens,
                          int length, long* out);
int ls_fp4_attention(int dtype, const void* q, long ldq, void* out, long ldo, int rows, const void* k_codes,
                     const void* k_scales, const void* v_codes, const void* v_scales, int pages, int page_size, int kv_heads,
                     int group, const int* table, int columns, const int* offsets, const int* lengths, int requests,
                     int most, int longest, float scale, int window, void* scratch, long scratch_bytes, void* stream);

#ifdef __cplusplus
}
#endif
