// C ABI of the language-model operators: the part of api.h that needs no CUDA header, so that torch_binding.cpp, which an
// ordinary C++ compiler builds, has the same declarations as the kernels' files.  All return MGW_OK (0) or an MGW_ERR_* code.
#pragma once
#include <stddef.h>

enum { MGW_F32 = 0, MGW_F16 = 1, MGW_BF16 = 2 };

#ifdef __cplusplus
extern "C" {
#endif

// ---- embedding lookup and its gradient (embedding.cu) -------------------------------------------------
// dtype: MGW_F32 / MGW_F16 / MGW_BF16; tokens: int32 (wide = 0) or int64 (wide = 1).  A token outside
// [0, vocab) is recorded in `status` (mgw_token_status) and gives a row of NaN, or no contribution to the gradient.
int mgw_token_status(int** words_out);                               // 8 pinned words, one block per process
// order: null, or memory of mgw_embedding_order_bytes() (0: not for these sizes) in which the tokens are left sorted for the
// gradient, without the token `padding`.
size_t mgw_embedding_order_bytes(long long n, long long vocab, int dim, int dtype);
int mgw_embedding_fwd(const void* tokens, int wide, long long n, const void* weight, long long ld, long long vocab, int dim, int dtype,
                      float scale, void* out, void* order, long long padding, int* status, void* stream);
size_t mgw_embedding_grad_bytes(long long n, long long vocab, int dim, int dtype);      // scratch memory of the call below
// dw [vocab, dim] is written whole; rows of the token `padding` (-1: none) stay zero.  order: null, or what the lookup left.
int mgw_embedding_grad(const void* dy, long long dy_ld, const void* tokens, int wide, long long n, long long vocab, int dim, int dtype,
                       float scale, long long padding, const void* order, void* dw, void* work, size_t work_bytes, int* status,
                       void* stream);

// ---- log probabilities, entropy, likeliest tokens, cross entropy (logprob.cu) -------------------------
// stats: [rows][2] largest logit m and log2 of the sum of exp(z - m), for the backward pass (may be null).
int mgw_logprob_fwd(const void* z, long long ld, long long rows, int vocab, int dtype, const void* tokens, int wide, long long ignore,
                    float* logprob, float* entropy, float* stats, int top, float* top_logprob, long long* top_tokens, int* status,
                    void* stream);
// Gradient for given gradients of log probability and entropy (either may be null), or of the loss (g_loss, one value).
// written: dz already holds the gradient for g_loss == expected (mgw_cross_entropy_fwd), nothing is done in that case.
int mgw_logprob_bwd(const void* z, long long ld, long long rows, int vocab, int dtype, const void* tokens, int wide, long long ignore,
                    const float* stats, const float* entropy, const float* g_logprob, const float* g_entropy, const float* g_loss,
                    const int* count, int written, float expected, void* dz, long long dz_ld, void* stream);
// Mean (or sum) of the negative log probabilities, and with dz its gradient times `expected`.  work: 2 ints, the first is
// `count` for mgw_logprob_bwd.
int mgw_cross_entropy_fwd(const void* z, long long ld, long long rows, int vocab, int dtype, const void* tokens, int wide,
                          long long ignore, int mean, float expected, float* logprob, float* stats, float* loss, void* dz, long long dz_ld,
                          int* work, int* status, void* stream);

// ---- global gradient norm and clipping (grad_clip.cu) -------------------------------------------------
// norm: 0 two-norm, 1 sum of magnitudes, 2 largest magnitude; clip = 0 only measures.  work: mgw_grad_clip_bytes(n).
size_t mgw_grad_clip_bytes(int n);
int mgw_grad_clip(const unsigned long long* ptrs, const long long* numels, const unsigned char* dtypes, int n, int norm, double scale,
                  double max_norm, int clip, void* work, size_t work_bytes, float* norm_out, void* stream);

#ifdef __cplusplus
}
#endif
