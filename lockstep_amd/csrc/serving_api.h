// The C interface of the serving library (tables.hip, logprobs.hip, fp4_pages.hip).  Conventions as in core_api.h.
#pragma once

#ifdef __cplusplus
extern "C" {
#endif

const char* ls_last_error();

// Block tables and slot maps of one step (tables.hip).
int ls_step_tables_max_requests();
int ls_step_tables(const int* lengths, const int* news, int requests, int* table, int columns, int page_size,
                   const int* free_pages, int free_count, const int* cursor, int* slots, int* tok_seq, int* tok_pos,
                   int tokens, int* offsets, int* new_lengths, int* progress, void* stream);

// Log probabilities of given tokens (logprobs.hip).  scratch: ls_logprobs_scratch_bytes(...) bytes.
int ls_logprobs_max_vocab();
int ls_logprobs_max_top();
long ls_logprobs_scratch_bytes(int rows, int vocab);
int ls_token_logprobs(int dtype, const void* logits, long ld, const int* tokens, int rows, int vocab, int top,
                      float* logprob, float* entropy, int* rank, int* top_ids, float* top_logprobs, void* scratch,
                      long scratch_bytes, void* stream);

// Keys and values into pages of 4 bits and back (fp4_pages.hip).
int ls_fp4_write(int dtype, const void* k, long ldk, const void* v, long ldv, const int* slots, int tokens, int kv_heads,
                 int dim, void* k_codes, void* k_scales, void* v_codes, void* v_scales, int pages, int page_size,
                 void* stream);
int ls_fp4_read(int dtype, void* k, long ldk, void* v, long ldv, const int* slots, int tokens, int kv_heads, int dim,
                const void* k_codes, const void* k_scales, const void* v_codes, const void* v_scales, int pages,
                int page_size, void* stream);

#ifdef __cplusplus
}
#endif
