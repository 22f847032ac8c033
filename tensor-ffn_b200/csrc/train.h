// Launchers of the training operators of include/tffn.h: what a trainer of expert deltas needs of the frozen base next to
// expert_forward. Every pointer is a device pointer of the current device; nothing is allocated and nothing waits.
// Each returns a cudaError, or -1000 if a tensor map could not be encoded.
#pragma once
#include "kernels.h"
#include "launch.h"
#include <atomic>
#include <cstddef>
#include <cstdint>

namespace tffn {

// the status word that the bounded waits of these kernels write, one per device (train.cu); nullptr if it cannot be found
int* train_status_word(int device);

// opts a kernel into `bytes` of shared memory, once per device
template <auto K>
cudaError_t allow_shared(int bytes) {
    static std::atomic<uint64_t> done{0};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const uint64_t bit = 1ull << (dev & 63);
    if (done.load(std::memory_order_acquire) & bit) return cudaSuccess;
    e = cudaFuncSetAttribute(K, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) e = prefer_max_shared(K);
    if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
    return e;
}

// y = (x - mean) * rstd * weight + bias per row; without `layer` the mean is zero and there is no bias
struct NormCall {
    bool layer, f32;  // f32: x, y, weight, bias, dy, skip and dx are fp32, else bf16
    const void *x, *weight, *bias;
    int64_t rows;
    int width;
    float eps;
    void* y;
    float *mean, *rstd;
    // backward
    const void *dy, *skip;  // skip: added to dx, or nullptr
    void* dx;
    float *dweight, *dbias;  // or nullptr
    float* workspace;        // norm_workspace_floats, unless dweight and dbias are nullptr
    int* status;
};
constexpr int kNormMaxWidth = 16384;
int64_t norm_workspace_floats(int64_t rows, int width);
[[nodiscard]] int launch_norm_forward(const NormCall& c, int num_sms, cudaStream_t s);
[[nodiscard]] int launch_norm_backward(const NormCall& c, int num_sms, cudaStream_t s);

// log-probability of one token per row of logits, and the clipped policy loss on it
constexpr int kLossMaxVocab = INT32_MAX - 4096;  // an index a block's threads past the end of a row fits an int
struct LossCall {
    bool f32;
    const void* logits;  // [rows][stride]
    int64_t rows, stride;
    int vocab;
    const int32_t* targets;
    float* logprob;
    const float *old_logprob, *ref_logprob, *advantage, *weight;
    float clip_low, clip_high, kl_coef;
    float *loss, *row_loss, *kl;  // each may be nullptr; loss needs row_loss
    int* status;
    void* d_logits;               // [rows][stride], may be logits itself
};
bool policy_loss_supported(bool f32, int vocab);
[[nodiscard]] int launch_token_logprobs(const LossCall& c, int num_sms, cudaStream_t s);
[[nodiscard]] int launch_policy_loss(const LossCall& c, int num_sms, cudaStream_t s);

// attention of packed sequences; rows of a tensor are `stride` elements apart, its heads hd apart
struct AttnCall {
    int n_seqs, heads, kv_heads, hd;  // hd: a multiple of 8, at most 128
    int64_t rows_q, rows_k;
    int max_q, max_k;
    int64_t q_stride, k_stride, v_stride, out_stride;  // multiples of 8
    float scale;
    int causal, chunk;
    const int32_t *cu_q, *cu_k;
    const bf16 *q, *k, *v;
    bf16* out;
    float* lse;
    // backward: dq, dk, dv have the strides of q, k, v; d_out that of out
    const bf16* d_out;
    bf16 *dq, *dk, *dv;
    void* workspace;
    int* status;
};
int64_t attention_workspace_bytes(const AttnCall& c);
// Whether a pass has fewer than 2^30 units of work, by what its packed rows can hold; the launchers count on it.
bool attention_forward_fits(const AttnCall& c);
bool attention_backward_fits(const AttnCall& c);
[[nodiscard]] int launch_attention_train_forward(const AttnCall& c, int num_sms, cudaStream_t s);
[[nodiscard]] int launch_attention_train_backward(const AttnCall& c, int num_sms, cudaStream_t s);

}  // namespace tffn
