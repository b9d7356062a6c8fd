// train_ops.cuh -- host interface of the training operators beside the
// aggregation: embedding.cu, group_norm.cu(h), clip.cu.
#pragma once

#include "common.cuh"

namespace tcc {

// `rows` are the looked-up rows (forward) or their gradient (backward), `table`
// the table or its gradient; `padding` is INT64_MIN when there is none.
struct EmbeddingArgs {
    void* table;
    int table_type;
    uint64_t ldt, num_rows;
    const void* idx;
    int idx_type;
    uint64_t n;
    int64_t padding;
    float scale;
    void* rows;
    int row_type;
    uint64_t ldr;
    uint32_t F;
    uint32_t* bad;
};
void embedding_forward(const EmbeddingArgs& a, cudaStream_t s);
size_t embedding_backward_scratch_bytes(uint64_t n, uint64_t num_rows, uint32_t F);
void embedding_backward(const EmbeddingArgs& a, void* scratch, size_t scratch_bytes, cudaStream_t s);

// x is [N, S, C] with rows of C contiguous channels, ldx apart; mean and rstd
// are fp32 [N, G].
struct GroupNormArgs {
    const void* x;
    uint64_t ldx;
    int type;
    const void* weight;
    const void* bias;
    int param_type;
    void* y;  // forward
    uint64_t ldy;
    const void* dy;  // backward
    uint64_t lddy;
    void* dx;
    uint64_t lddx;
    void* dweight;
    void* dbias;
    float* mean;
    float* rstd;
    uint64_t N, S;
    uint32_t C, G;
    float eps;
    int act;
};
size_t group_norm_scratch_bytes(uint64_t N, uint64_t S, uint32_t C, uint32_t G, bool backward);
void group_norm_forward(const GroupNormArgs& a, void* scratch, size_t scratch_bytes, cudaStream_t s);
void group_norm_backward(const GroupNormArgs& a, void* scratch, size_t scratch_bytes, cudaStream_t s);

size_t grad_norm_scratch_bytes();
// norm: written by grad_norm and clip_grad_norm, read by clip_grads_with_norm.
void grad_norm(const tcc_tensor* t, uint32_t count, float* norm, void* scratch, size_t scratch_bytes,
               cudaStream_t s);
void clip_grads_with_norm(const tcc_tensor* t, uint32_t count, const float* norm, float max_norm,
                          float eps, cudaStream_t s);
void clip_grad_norm(const tcc_tensor* t, uint32_t count, float max_norm, float eps, float* norm,
                    void* scratch, size_t scratch_bytes, cudaStream_t s);

}  // namespace tcc
