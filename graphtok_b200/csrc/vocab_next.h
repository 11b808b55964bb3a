// Operators from a model's last hidden states to the next ids: products with a table in 4 bits (vocab_quant.cu), changes to logits and
// sampling (vocab_next.cu); the C entries are in vocab_abi.cc.
#pragma once
#include "vocab_ops.h"

namespace gtok {

// A table of 4-bit codes as pack_table and quantize_table lay it out in one piece of memory: codes, scales, zeros.
struct Table4 {
    void* data = nullptr;
    int64_t vocab = 0, width = 0, group = 128;
    int type = kBF16;            // of the scales and of the hidden states that it is multiplied with
    bool zeros = false;
};

// Where the parts lie.  Codes: units of 16 rows x 64 columns, 512 bytes, two units (32 rows) beside one another, along the width, then down
// the vocabulary.  A unit is 32 lots of 16 bytes, one for each lane of the warp that multiplies with it; a lane's four words are its operand
// of m16n8k16 products of 16 columns each (vocab_quant.cu).  Scales and zeros: for every 32 rows and group 32 values, row 8 j + i at 4 i + j.
struct Table4Plan {
    int64_t tiles, units, groups;              // of 32 rows; of 64 columns; groups of a row, counted over whole units
    uint64_t scales, zeros, bytes;             // places of the parts, and the size
};
inline Table4Plan table4_plan(int64_t vocab, int64_t width, int64_t group, bool zeros) {
    Table4Plan p;
    p.tiles = (vocab + 31) / 32;
    p.units = (width + 63) / 64;
    p.groups = group == 32 ? p.units * 2 : (width + group - 1) / group;
    p.scales = static_cast<uint64_t>(p.tiles) * p.units * 1024;
    p.zeros = (p.scales + static_cast<uint64_t>(p.tiles) * p.groups * 64 + 255) / 256 * 256;
    p.bytes = p.zeros + (zeros ? static_cast<uint64_t>(p.tiles) * p.groups * 32 : 0);
    p.bytes = (p.bytes + 255) / 256 * 256;
    return p;
}

struct AdjustCall {
    Matrix logits, out;          // [n, vocab], of one type; may be the same memory
    Ids ids;                     // histories, one row's after another's
    int64_t n_ids = 0;
    const int32_t* offsets = nullptr;          // n + 1 places
    const int32_t* prompt_lengths = nullptr;   // of each row, optional
    const float* repetition = nullptr;         // of each row; without one, the number
    const float* presence = nullptr;
    const float* frequency = nullptr;
    float one_repetition = 1.f, one_presence = 0.f, one_frequency = 0.f;
    int entries = 0;             // biases a row
    const int32_t* bias_ids = nullptr;
    const float* bias = nullptr;
    int64_t bias_stride = 0;     // from a row's list to the next, 0: all rows have one
    const int32_t* allowed = nullptr;          // bits
    int64_t allowed_count = 0, allowed_stride = 0;
    const int32_t* allowed_rows = nullptr;     // which of them a row has; without it, its own
    cudaStream_t stream = nullptr;
};

struct SampleCall {
    Matrix logits;
    const void* u = nullptr;     // random numbers, fp32 or fp64
    bool wide_u = false;
    const float* temperature = nullptr;        // of each row; without one, the number
    const int32_t* top_k = nullptr;
    const float* top_p = nullptr;
    const float* min_p = nullptr;
    float one_temperature = 1.f, one_top_p = 1.f, one_min_p = 0.f;
    int32_t one_top_k = 0;
    int32_t* ids = nullptr;
    float* logprobs = nullptr;
    cudaStream_t stream = nullptr;
};

constexpr int kMaxBiases = 1024;

const char* pack_table(const Table4& t, const uint8_t* codes, int64_t codes_stride, const Matrix& scales, const uint8_t* zeros, int64_t zeros_stride, cudaStream_t stream);
const char* quantize_table(const Table4& t, const Matrix& weight, cudaStream_t stream);
const char* table_logits(const Matrix& hidden, const Table4& t, const Matrix& out, cudaStream_t stream);
const char* adjust_logits(const AdjustCall& c);
const char* sample(const SampleCall& c);

}  // namespace gtok
