// Prototypes of the kernel launchers that the native prompt-step executor (prompt_exec.cu) and the host's
// calls (host_calls.cpp) call through pointers, and the codes that launchers take.  The libraries that define them
// include this file as well, so that a definition that drifts from its prototype does not compile.
#pragma once
#include <cuda_runtime.h>

// element types
#define QD_F32 0
#define QD_BF16 1
// returned by launchers for arguments a kernel refuses (never a wrong result)
#define QD_ERR_UNSUPPORTED 10001
// gated activations
#define QD_ACT_SILU 0
#define QD_ACT_GELU_TANH 2
// rows in 8 bits: features to a scale; what becomes of a product's sums; tokens that ``qd_gemm_fp8_few`` takes
#define QD_FP8_BLOCK 128
#define QD_FP8_STORE 0
#define QD_FP8_GATED 2
#define QD_FP8_FEW_TOKENS 16
// log probabilities
#define QD_LOGPROBS_MAX_TOP 32
#define QD_LOGPROBS_MAX_VOCABULARY (1 << 22)

extern "C" {
int qd_add_rmsnorm(float* x, const void* delta, int delta_dtype, const float* w, void* out, int out_dtype,
                   const int* rows, int n_rows, int D, float eps, int write_back, int n_parts,
                   long long part_stride, cudaStream_t stream);
int qd_rope_kv_write_biased(void* qkv, const float* bias, int T, int H, int G, int d, int rotary_dim, int pairing,
                            const float* cos_t, const float* sin_t, const int* positions, void* kv,
                            const int* slot_map, int page_size, int write_kv, cudaStream_t stream);
int qd_rope_kv_write_partial(const float* part, int n_parts, const float* bias, void* q_out, int T, int H, int G, int d, int rotary_dim,
                             int pairing, const float* cos_t, const float* sin_t, const int* positions, void* kv, const int* slot_map,
                             int page_size, int write_kv, cudaStream_t stream);
int qd_rows_fp8(const void* x, int dtype, long long ldx, int n_parts, long long part_stride, int gated, int act, const float* bias, void* q,
                long long ldq, void* s, long long lds, int T, int K, cudaStream_t stream);
int qd_add_rmsnorm_fp8(float* x, const void* delta, int delta_dtype, const float* dscale, const float* w, void* q, long long ldq, void* s,
                       long long lds, const int* rows, int n_rows, int D, float eps, int write_back, int n_parts, long long part_stride,
                       cudaStream_t stream);
int qd_gemm_fp8(const void* W, long long ldw, const void* sw, long long ldsw, const void* X, long long ldx, const void* sx, long long ldsx,
                const float* bias, void* out, int out_dtype, long long ldo, void* s_out, long long lds_out, int T, int N, int K, int cg,
                int bn, int splits, int epi, int resident, int sms, cudaStream_t stream);
int qd_gemm_fp8_plan(int T, int N, int K, int epi, int out_dtype, int sms, int* cg_out, int* bn_out, int* splits_out);
int qd_gemm_fp8_few_wanted(int T, int N, int K, int sms);
int qd_token_logprobs(const void* logits, int dtype, long long ld, const int* tokens, float* logprob, float* entropy, int* top_ids,
                      float* top_logprobs, int R, int V, int top, int sms, cudaStream_t stream);
int qd_gemm_fp8_few(const void* W, long long ldw, const void* sw, long long ldsw, const void* X, long long ldx, const void* sx,
                    long long ldsx, const float* bias, void* out, int out_dtype, long long ldo, int T, int N, int K, int resident,
                    int sms, cudaStream_t stream);
int qd_gemm_pair(const void* W, const void* X, long long ldx, const float* bias, void* out, int out_dtype, long long ldo, int T,
                 int N, int K, int cg, int bn, int splits, int epi, int sms, cudaStream_t stream);
int qd_gemm_pair_plan(int T, int N, int K, int epi, int sms, int* cg_out, int* bn_out, int* splits_out);
int qd_swiglu(const void* gate_up, void* out, int dtype, int T, int F, cudaStream_t stream);
void qd_elementwise_plain_next();
int qd_decode_attention(const void* q, long long q_stride, void* out, const void* kv, const int* block_table,
                        int max_blocks, const int* token_req, const int* positions, int T, int H, int G, int d,
                        int page_size, float scale, int window, int splits, float* part_o, float* part_ml,
                        unsigned* tickets, cudaStream_t stream);
int qd_decode_attention_tma(const void* q, long long q_stride, void* out, const void* kv, long long n_pages,
                            const int* block_table, int max_blocks, const int* token_req, const int* positions, int T,
                            int H, int G, int d, int page_size, float scale, int window, int splits, float* part_o,
                            float* part_ml, unsigned* tickets, cudaStream_t stream);
int qd_decode_shares(const int* positions, const int* slot_map, int scratch_row, int T, int n_list, void* list, cudaStream_t stream);
int qd_decode_attention_shares(const void* q, long long q_stride, void* out, const void* kv, long long n_pages,
                               const int* block_table, int max_blocks, int T, int H, int G, int d, int page_size, float scale,
                               const void* shares, int n_list, int fresh, float* part_o, float* part_ml, unsigned* tickets,
                               cudaStream_t stream);
int qd_prefill_attention(const void* q, long long q_stride, void* out, const void* kv, const int* block_table,
                         int max_blocks, const int* cu_tokens, const int* start_pos, int R, int T, int H, int G,
                         int d, int page_size, float scale, int window, cudaStream_t stream);
int qd_prefill_attention_tc5(const void* q, long long q_stride, void* out, const void* kv, long long n_pages,
                             const int* block_table, int max_blocks, const int* cu_tokens, const int* start_pos,
                             int R, int T, int H, int G, int d, int page_size, float scale, int window,
                             long long* timeline, cudaStream_t stream);
}
