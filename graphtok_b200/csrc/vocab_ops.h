// Operators between token ids and a model's vocabulary-wide tables (vocab_rows.cu, vocab_loss.cu); the C entries are in vocab_abi.cc.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include <string>

namespace gtok {

enum { kF32 = 0, kBF16 = 1, kF16 = 2 };

struct Matrix {                  // rows of `cols` elements, `stride` elements from one to the next
    const void* data = nullptr;
    int64_t rows = 0, cols = 0, stride = 0;
    int type = kF32;
};
struct Ids {                     // signed integers of 32 or 64 bits; `stride` elements between rows where there are several in a row
    const void* data = nullptr;
    int bits = 32;
    int64_t stride = 1;
};

struct LossCall {
    Matrix hidden, weight;       // [n, width], [vocab, width]; both bf16 or both fp16
    Ids targets;                 // one id a row; or, with `entries` > 0:
    int entries = 0;             // ids of a teacher's top logits, a row of `entries` each,
    Matrix teacher;              // and the logits
    int64_t ignore = -100;
    float temperature = 1.f;
    float* losses = nullptr;     // forward: [n]
    float* lse = nullptr;        // forward, written; backward, read: [n]
    float* total = nullptr;      // forward, optional: their sum,
    bool mean = false;           // or the mean over the rows that have a loss; backward: `grad` is of that mean
    const float* grad = nullptr; // backward: of `losses`, grad_stride apart, or of their sum or mean (grad_stride 0)
    int64_t grad_stride = 1;
    Matrix d_hidden, d_weight;   // backward, either may have no data
    void* kept = nullptr;        // optional: what the forward pass leaves there the backward one does not do again
    void* workspace = nullptr;
    uint64_t workspace_bytes = 0;
    cudaStream_t stream = nullptr;
};

constexpr int kMaxEntries = 1024;

// NULL or an error message.  Arguments are checked by the caller; `stream` must belong to the current device.
uint64_t loss_workspace(const LossCall& c, bool backward);
uint64_t loss_kept(const LossCall& c);
const char* loss_forward(const LossCall& c);
const char* loss_backward(const LossCall& c);

const char* embed(const Ids& ids, int64_t n, const Matrix& table, float scale, const Matrix& out, cudaStream_t stream);
uint64_t embed_grad_workspace(int64_t n, int64_t vocab, int64_t width);
const char* embed_grad(const Ids& ids, int64_t n, const Matrix& grad, float scale, const Matrix& out, bool accumulate, void* workspace, uint64_t workspace_bytes,
                       cudaStream_t stream);
const char* next_targets(const int32_t* ids, int64_t n, const int32_t* offsets, int64_t n_docs, const uint8_t* loss_mask, int32_t ignore, int32_t* out,
                         cudaStream_t stream);

}  // namespace gtok
