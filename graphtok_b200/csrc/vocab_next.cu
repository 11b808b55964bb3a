// What happens to logits before an id is drawn, and the draw: penalties, biases and grammar masks; temperature, top-k, top-p, min-p.
#include "sm100.cuh"
#include "vocab_launch.cuh"
#include "vocab_next.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>

namespace gtok {
namespace {

__host__ __device__ constexpr int64_t div_up(int64_t a, int64_t b) { return (a + b - 1) / b; }
__host__ __device__ constexpr int64_t round_up(int64_t a, int64_t b) { return div_up(a, b) * b; }

template <typename T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

// `N` elements that are read and written together: 16 bytes.
template <typename T, int N>
struct alignas(sizeof(T) * N) Lump {
    T v[N];
};

// ---- penalties, biases, masks -------------------------------------------------------
// A block takes a slice of a row.  It counts the row's history into shared memory, as far as it lies in the slice, and then passes over
// the slice once, the logits of which are on their way meanwhile.  Bound by memory: a logit read and written, a bit of a mask; in place, only what changes.
// 251 rows of 128,256 bf16 with histories of 12,500 ids, 300 biases and masks: 109 us (22 at the rate of a copy); 44 of it with short histories and nothing else, the rest counting, masks and
// biases.  A cluster that goes over a history once, each block a part, and counts into one another's shared memory waits for the block with the frequent ids: 266 us, when counting by
// each block took 220.  Slices of half the size, four blocks to an SM: 173 us where 145.  At the 40 registers that three blocks to an SM leave, whole lumps spill 50 to 108 bytes; with two
// blocks, 64 registers and next to no spills it is 117 us, 47 rows of 151,665 fp32 25.2 where 25.8.  One row of 128,256 with 911 ids: 3.7 us, all latency.
constexpr int kAdjustThreads = 512, kMostSlice = 16384;
constexpr int kSpare = 8;                        // ids of the lump in front of a slice
constexpr uint32_t kSaid = 0x80000000u;          // of a count: the id is in the prompt

struct AdjustArgs {
    const void* logits;
    void* out;
    int64_t stride, out_stride;
    int vocab, slice, slices;
    bool in_place, history;
    const void* ids;
    int id_bits;
    int64_t n_ids;
    const int32_t *offsets, *prompt_lengths;
    const float *repetition, *presence, *frequency;
    float one_repetition, one_presence, one_frequency;
    int entries;
    const int32_t* bias_ids;
    const float* bias;
    int64_t bias_stride;
    const int32_t *allowed, *allowed_rows;
    int64_t allowed_count, allowed_stride;
};

template <typename T, int N>
__global__ void __launch_bounds__(kAdjustThreads, 3) adjust_kernel(const __grid_constant__ AdjustArgs a) {
    extern __shared__ uint4 smem[];
    uint32_t* count = reinterpret_cast<uint32_t*>(smem);                       // [slice + kSpare]
    uint32_t* biased = count + a.slice + kSpare;                               // [kMostSlice / 32 + 1]: a bit for each id that has a bias
    float* bias = reinterpret_cast<float*>(biased + kMostSlice / 32 + 1);      // [entries]
    int32_t* listed = reinterpret_cast<int32_t*>(bias + a.entries);            // [entries]
    __shared__ int twice;                                                      // an id comes more than once
    const int tid = threadIdx.x;
    after_previous();
    let_next_begin();
    const int64_t row = blockIdx.x / a.slices;
    const int s = static_cast<int>(blockIdx.x - row * a.slices);
    const T* in = static_cast<const T*>(a.logits) + row * a.stride;
    T* out = static_cast<T*>(a.out) + row * a.out_stride;
    // Lumps lie on 16 bytes of the input, whatever the row begins at; the first one of the row is no whole one.
    const int off = N == 1 ? 0 : static_cast<int>((16 - reinterpret_cast<uintptr_t>(in) % 16) % 16 / sizeof(T));
    const int base = off + s * a.slice - N;                                    // id of count[0]
    const int begin = s == 0 ? 0 : base + N, end = min(base + N + a.slice, a.vocab);
    const int v_first = base + (s == 0 ? 0 : N) + tid * N;                     // this thread's first lump

    const float rho = a.repetition ? a.repetition[row] : a.one_repetition, presence = a.presence ? a.presence[row] : a.one_presence,
                frequency = a.frequency ? a.frequency[row] : a.one_frequency;
    const uint32_t* words = nullptr;
    bool nothing = false;                              // a mask that is not there allows nothing
    if (a.allowed) {
        const int64_t which = a.allowed_rows ? a.allowed_rows[row] : row;
        if (which >= a.allowed_count) nothing = true;
        else if (which >= 0) words = reinterpret_cast<const uint32_t*>(a.allowed) + which * a.allowed_stride;
    }
    // The first logits and their bits of the mask are fetched while ids are counted; in place most logits are not needed.
    constexpr int kFetch = 2;
    Lump<T, N> ahead[kFetch];
    uint32_t bits[kFetch];
    const auto whole = [&](int v) { return v >= 0 && v < end && v + N <= a.vocab; };
    const auto allowed_at = [&](int v) {
        uint32_t b = nothing ? 0 : ~0u;
        if (words) b = __funnelshift_r(words[v >> 5], words[(v + N - 1) >> 5], v & 31);
        return b | ~((1u << N) - 1);
    };
#pragma unroll
    for (int q = 0; q < kFetch; ++q) {
        const int v = v_first + q * kAdjustThreads * N;
        if (!whole(v)) continue;
        if (!a.in_place) ahead[q] = *reinterpret_cast<const Lump<T, N>*>(in + v);
        bits[q] = allowed_at(v);
    }

    for (int i = tid; i < (a.slice + kSpare) / 4; i += kAdjustThreads) reinterpret_cast<uint4*>(count)[i] = make_uint4(0, 0, 0, 0);
    if (a.entries) {
        for (int i = tid; i < kMostSlice / 32 + 1; i += kAdjustThreads) biased[i] = 0;
        for (int i = tid; i < a.entries; i += kAdjustThreads) {
            listed[i] = a.bias_ids[row * a.bias_stride + i];
            bias[i] = a.bias[row * a.bias_stride + i];
        }
        if (tid == 0) twice = 0;
    }
    __syncthreads();
    if (a.history) {
        int64_t from = a.offsets[row], to = a.offsets[row + 1];
        from = from < 0 ? 0 : from;
        to = to > a.n_ids ? a.n_ids : to;
        const int64_t behind = from + (a.prompt_lengths ? a.prompt_lengths[row] : 0);
        constexpr int kIds = 4;                // under way a thread
        for (int64_t i = from + tid; i < to; i += kAdjustThreads * kIds) {
            int64_t id[kIds];
#pragma unroll
            for (int q = 0; q < kIds; ++q) {
                const int64_t at = i + q * kAdjustThreads;
                id[q] = at >= to ? -1 : a.id_bits == 64 ? static_cast<const int64_t*>(a.ids)[at] : static_cast<const int32_t*>(a.ids)[at];
            }
#pragma unroll
            for (int q = 0; q < kIds; ++q) {
                if (id[q] < begin || id[q] >= end) continue;
                if (i + q * kAdjustThreads < behind) atomicOr(&count[id[q] - base], kSaid);
                else atomicAdd(&count[id[q] - base], 1u);
            }
        }
    }
    // Ids with a bias are changed by themselves in the end, by the thread of their first entry to come, which takes their logit before it is written.
    constexpr int kBiases = (kMaxBiases + kAdjustThreads - 1) / kAdjustThreads;
    T biased_logit[kBiases];
    bool mine[kBiases];
#pragma unroll
    for (int q = 0; q < kBiases; ++q) {
        const int i = tid + q * kAdjustThreads, id = i < a.entries ? listed[i] : -1;
        mine[q] = false;
        if (id < begin || id >= end) continue;
        const uint32_t bit = 1u << (id & 31);
        mine[q] = !(atomicOr(&biased[(id >> 5) - (begin >> 5)], bit) & bit);
        if (mine[q]) biased_logit[q] = in[id];
        else twice = 1;
    }
    __syncthreads();

    const auto changed = [&](float x, uint32_t c, float b, bool allowed) {
        if (c) {
            x = x > 0.f ? x / rho : x * rho;
            const uint32_t times = c & ~kSaid;
            if (times) x = x - frequency * static_cast<float>(times) - presence;
        }
        return allowed ? x + b : -INFINITY;
    };
    const auto allowed_one = [&](int v) { return !nothing && (!words || (words[v >> 5] >> (v & 31) & 1)); };
    const auto lump = [&](int v0, bool fetched, Lump<T, N> x, uint32_t allowed) {
        if (whole(v0)) {
            if (!fetched) allowed = allowed_at(v0);
            uint32_t c[N], any = 0;
            if constexpr (N == 1) {
                c[0] = count[v0 - base];
            } else {                           // 16 bytes at a time
#pragma unroll
                for (int i = 0; i < N; i += 4) {
                    const uint4 four = *reinterpret_cast<const uint4*>(count + (v0 - base) + i);
                    c[i] = four.x; c[i + 1] = four.y; c[i + 2] = four.z; c[i + 3] = four.w;
                }
            }
#pragma unroll
            for (int i = 0; i < N; ++i) any |= c[i];
            if (a.in_place && !any && allowed == ~0u) return;
            if (!fetched || a.in_place) x = *reinterpret_cast<const Lump<T, N>*>(in + v0);
            if (any || allowed != ~0u)
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (c[i] || !(allowed >> i & 1)) x.v[i] = from_float<T>(changed(to_float<T>(x.v[i]), c[i], -0.f, allowed >> i & 1));
            *reinterpret_cast<Lump<T, N>*>(out + v0) = x;
        } else if (N > 1) {
            for (int i = 0; i < N; ++i) {
                const int v = v0 + i;
                if (v < 0 || v >= end) continue;
                const bool allowed = allowed_one(v);
                const uint32_t c = count[v - base];
                T one = in[v];
                if (c || !allowed) one = from_float<T>(changed(to_float<T>(one), c, -0.f, allowed));
                out[v] = one;
            }
        }
    };
#pragma unroll
    for (int q = 0; q < kFetch; ++q)
        if (v_first + q * kAdjustThreads * N < end) lump(v_first + q * kAdjustThreads * N, true, ahead[q], bits[q]);
    for (int v = v_first + kFetch * kAdjustThreads * N; v < end; v += kAdjustThreads * N) lump(v, false, ahead[0], 0);
    if (!a.entries) return;
    __syncthreads();
#pragma unroll
    for (int q = 0; q < kBiases; ++q) {
        if (!mine[q]) continue;
        const int i = tid + q * kAdjustThreads, id = listed[i];
        float sum = bias[i];
        if (twice) {                           // in the order of the list, whichever entry this is
            sum = 0.f;
            for (int j = 0; j < a.entries; ++j)
                if (listed[j] == id) sum += bias[j];
        }
        out[id] = from_float<T>(changed(to_float<T>(biased_logit[q]), count[id - base], sum, allowed_one(id)));
    }
}

template <typename T, int N>
cudaError_t adjust(AdjustArgs a, int64_t rows, cudaStream_t stream) {
    // Slices of 16,384 ids count a long history least often; of fewer where that leaves SMs without work.
    a.slice = kMostSlice;
    while (a.slice > 2048 && rows * div_up(a.vocab, a.slice) < 148) a.slice /= 2;
    a.slices = static_cast<int>(div_up(a.vocab, a.slice));
    a.slice = static_cast<int>(round_up(div_up(a.vocab, a.slices), 64));
    const int smem = (a.slice + kSpare) * 4 + (a.entries ? (kMostSlice / 32 + 1) * 4 + a.entries * 8 : 0);
    auto* kernel = adjust_kernel<T, N>;
    if (cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 128 * 1024)) return e;
    return launch(kernel, rows * a.slices, kAdjustThreads, smem, stream, a);
}

// ---- an id a row ------------------------------------------------------------------------
// With d = l - max and m = exp(d / T) for each id, in order of falling logits and, among equal ones, of rising ids: the first top_k are kept; of these
// the shortest stretch whose mass is at least top_p of theirs; of these the ones with m >= min_p; the first id at least.  The id is the first one, in the order of
// the ids, at which the running sum of kept masses is more than u times their sum.
//
// A cluster of blocks takes a row.  Where it fits they hold it in shared memory and it is read from memory once; where rows are many, fewer blocks take longer shares,
// which they read again from L2, and wait for one another less.  Masses are whole numbers, 2^F for the largest, computed in 64 bits, off by 2^-43
// relative and rounded to a unit: their sums are exact and do not depend on the order of summation, nor on how many blocks take a row.  F is 46 for up to 2^16 ids, one less for
// each doubling up to 43 at 2^19, so that sums have 62 bits: all roundings together are 2^-25 of a row's total at most (2^-29 for 128,256 ids).  With more ids F goes by the row, which takes one pass
// more: as fine as its total allows, up to 50, and the roundings are 2^-27 of it at most.  All three cuts are
// stretches from the top of one order and so is what they have in common; a cut is the last id that is kept.
//
// What a row costs is the exponentials: 11 operations in 64 bits an id, of which an SM does two warps' in a clock.  One pass over all ids gives the total; most rows
// need no other one.  The same pass counts the ids "near" the largest, some hundreds, into bins.  Where the cut lies among them, they are picked, and one block
// ranks them one by one and draws.  Otherwise (a flat distribution of which much is kept) the rest's bins say about where the cut lies, a second pass sums
// what is above exactly and lists the ids around, and bins of these alone find it.  Where the guess was wrong, or too many ids are alike, bins over ever narrower intervals of
// all ids do.  What is near, and the guess, go by the logits' mean and deviation; they decide how long it takes and not what comes out.
//
// 251 rows of 128,256 bf16 with top_p 0.9 of a flat distribution: 223 us (10 at the rate of a copy): 146 instructions an id in a pass that fetches and two of exponentials and bins, with issue slots in use 64 % of the time by
// six to seven warps a scheduler.  64 rows of 151,665 fp32 as they are: 33 us, 57 instructions an id in two passes, slots in use 51 %.  47 rows of their own wishes: 61.  One row of 50,256 with top_k 50
// and top_p 0.95: 14.6 us, a chain of steps of which each waits for the one before; its four barriers of the cluster are 0.9 of it (0.23 each, by themselves).  With 32 warps a block, where a
// block has an SM to itself, 17.  One row of 2^20 ids as they are: 68 us, 45 without the pass that looks for its unit.
// What it took: sums of 64 bits in shared memory by pieces of 32 (as one addition of 64, a loop of comparisons and exchanges, 23,900 us); one thread a place and no branch in the
// exponential; places found by all warps of a block (by the one whose ids they are among: 60 us more); no conversions and no moving of bits between keys and logits.
constexpr int kMostBlocks = 8, kDrawThreads = 512, kDrawWarps = kDrawThreads / 32, kBins = 256, kGuessBins = 512, kRanked = 512, kPieces = 5;
constexpr uint32_t kLowest = 0x007FFFFFu;        // key of -infinity
constexpr uint32_t kHighest = 0xFF800000u;       // key of +infinity
constexpr uint32_t kNone = 0xFFFFFFFFu;          // of a NaN
constexpr int64_t kWholeBits = 0x4338000000000000ll;             // 1.5 * 2^52: behind sums with it whole numbers stand in the lower bits
constexpr int kOneUnit = 1 << 19;                // ids of a row up to which F goes by their number alone
constexpr int kFinest = 50;                      // F at most
constexpr int kMostShare = 1 << 21;              // ids of a block at most: kPieces pieces make a mass of kFinest bits

struct DrawArgs {
    const void* logits;
    int64_t stride;
    int vocab, segment;            // ids; ids of a warp, a multiple of 32
    int blocks;                    // of a row
    int fixed;                     // F, in a row of more than kOneUnit ids at least
    int piece;                     // bits of a mass that are added up at a time, in 32: share of a block times 2^piece is no more than 2^32
    int listed;                    // ids that a block can list
    bool held;                     // in shared memory
    const void* u;
    bool wide_u;
    const float* temperature;
    const int32_t* top_k;
    const float *top_p, *min_p;
    float one_temperature, one_top_p, one_min_p;
    int32_t one_top_k;
    int32_t* ids;
    float* logprobs;
    double power[32];              // 2^(F + i / 32)
};

struct Cut {                       // the last of the ids that are kept
    uint32_t key;
    int id;
};

struct DrawShared {
    union {                                    // (ids are ranked when bins have been told)
        struct {
            uint32_t pieces[kPieces][kBins];   // masses of the bins, as they are added up
            uint32_t count[kBins];
            uint32_t guess[kGuessBins];
        };
        struct {
            uint64_t rank_mass[kRanked];
            uint32_t rank_key[kRanked];
            int rank_id[kRanked];
        };
    };
    uint64_t bin_mass[2][kBins];               // what this block tells the others, in two places in turn
    uint32_t bin_count[2][kBins];
    uint64_t said[2][4];
    uint64_t told[4];                          // what the cluster says
    uint64_t all_mass[kBins];                  // of the cluster
    uint32_t all_count[kBins];
    float all_guess[kGuessBins];
    uint64_t red[kDrawWarps];
    float4 seen[kDrawWarps], seen_by_block;    // key of the largest, sum, squares, count; key, mean and deviation of the row
    uint64_t warp_mass[kDrawWarps];
    double power[32];
    uint32_t pick_key[kRanked];                // ids to be ranked
    int pick_id[kRanked];
    uint32_t list_n, pick_n;
    uint64_t word[4];                          // from one thread to the block
    Cut cut;
};
struct Placed {                    // of the ids that are ranked, where lists are not in use
    uint64_t in_front[kRanked];
    int place[kRanked];
};

__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.f);               // one zero
    return x == x ? b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u) : kNone;
}
__device__ __forceinline__ float value_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key); }
// Of an interval's upper end: the key of -0, which no logit has, is that of the number below.
__device__ __forceinline__ float upper_value(uint32_t key) { return value_of(key == 0x7FFFFFFFu ? key - 1 : key); }

__device__ __forceinline__ uint64_t peer_u64(const uint64_t* p, int block) {
    uint64_t v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(sm100::in_block(sm100::smem_addr(p), block)));
    return v;
}
__device__ __forceinline__ uint32_t peer_u32(const void* p, int block) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(sm100::in_block(sm100::smem_addr(p), block)));
    return v;
}

__device__ __forceinline__ uint64_t warp_sum(uint64_t v) {
#pragma unroll
    for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(~0u, v, d);
    return v;
}
__device__ __forceinline__ uint64_t warp_scan(uint64_t v) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const uint64_t o = __shfl_up_sync(~0u, v, d);
        if (lane >= d) v += o;
    }
    return v;
}
__device__ __forceinline__ uint64_t larger(uint64_t a, uint64_t b) { return a > b ? a : b; }
__device__ __forceinline__ uint64_t warp_max(uint64_t v) {
#pragma unroll
    for (int d = 16; d; d >>= 1) v = larger(v, __shfl_xor_sync(~0u, v, d));
    return v;
}

template <typename T>
struct Row {                       // a block's share of a row
    DrawShared& s;
    const float* held;             // NULL: in memory
    const T* in;
    int first, count, segment;     // first id, ids, ids of a warp
    int blocks, piece;
    uint32_t* list_key;
    int* list_id;
    uint32_t top;                  // key of the largest
    uint64_t largest;              // its mass
    double top_value, steps;       // 32 log2(e) / T
    double least;                  // exponents of less have no mass
    float floor;                   // logits of less have no mass, where `plain`
    bool plain;
    int exchanges;

    __device__ __forceinline__ float value(int i) const { return held ? held[i] : to_float<T>(in[i]); }

    // 2^(y / 32) = 2^(j / 32) * 2^(r / 32) with j the whole number next to y: the first factor from a table and j's upper bits; the second, for r from -1/2 to 1/2, from the
    // polynomial 1 + r q(r), q of degree 3, whose largest error is the least there is: 7.8e-14 (found by exchange).  The bits of kWholeBits' number are still on it.
    __device__ __forceinline__ int64_t mass_at(double y) const {
        constexpr double kWhole = 6755399441055744.0;
        const double shifted = y + kWhole;
        const int j = __double2loint(shifted);
        const double r = y - (shifted - kWhole);
        double p = fma(r, 9.1725896167412903e-9, 1.6938633992759381e-6);
        p = fma(p, r, 2.3459619820168606e-4);
        p = fma(p, r, 2.1660849391721052e-2);
        p = fma(p, r, 1.0);
        const double t = s.power[j & 31];
        const double scaled = __hiloint2double(__double2hiint(t) + (j >> 5) * (1 << 20), __double2loint(t));
        return __double_as_longlong(fma(scaled, p, kWhole));
    }
    __device__ __forceinline__ uint64_t mass(float x) const {
        if (top == kHighest) return x == INFINITY ? largest : 0;
        const double y = (static_cast<double>(x) - top_value) * steps;
        return y > least && x > -INFINITY ? static_cast<uint64_t>(mass_at(y) - kWholeBits) : 0;
    }
    // Several, NaN (where there is no logit) among them; without branches, so that they run at once.  A logit below `floor` is brought up to it: its mass rounds to 0.
    template <int N>
    __device__ __forceinline__ void masses(const float (&x)[N], int64_t (&m)[N]) const {
        if (plain) {
#pragma unroll
            for (int q = 0; q < N; ++q) m[q] = mass_at((static_cast<double>(fmaxf(x[q], floor)) - top_value) * steps);
        } else {
#pragma unroll
            for (int q = 0; q < N; ++q) m[q] = static_cast<int64_t>(mass(x[q])) + kWholeBits;
        }
    }

    // f(logits, place of the first) for this thread's share, in which a warp's ids follow one another, kAtOnce of them at a time; NaN behind the last.
    static constexpr int kAtOnce = 4;
    template <typename F>
    __device__ __forceinline__ void some(F f) const {
        const int from = (threadIdx.x >> 5) * segment, to = from + segment < count ? from + segment : count;
        const bool together = held || reinterpret_cast<uintptr_t>(in) % (kAtOnce * sizeof(T)) == 0;    // (segments are whole lots)
        float next[kAtOnce];                   // a step ahead: from memory they take longer than a step
        const auto fetch = [&](int i) {
            if (together && i + kAtOnce <= to) {
                if (held) {
                    const float4 v = *reinterpret_cast<const float4*>(held + i);
                    next[0] = v.x; next[1] = v.y; next[2] = v.z; next[3] = v.w;
                } else {
                    const Lump<T, kAtOnce> v = *reinterpret_cast<const Lump<T, kAtOnce>*>(in + i);
#pragma unroll
                    for (int q = 0; q < kAtOnce; ++q) next[q] = to_float<T>(v.v[q]);
                }
            } else {
#pragma unroll
                for (int q = 0; q < kAtOnce; ++q) next[q] = i + q < to ? value(i + q) : __int_as_float(0x7FC00000);
            }
        };
        const int first_place = from + (threadIdx.x & 31) * kAtOnce;
        fetch(first_place);
        for (int i = first_place; i < to; i += 32 * kAtOnce) {
            float x[kAtOnce];
#pragma unroll
            for (int q = 0; q < kAtOnce; ++q) x[q] = next[q];
            fetch(i + 32 * kAtOnce);
            f(x, i);
        }
    }
    // f(logit, place), one by one.
    template <typename F>
    __device__ __forceinline__ void each(F f) const {
        some([&](const float (&x)[kAtOnce], int i) {
#pragma unroll
            for (int q = 0; q < kAtOnce; ++q) f(x[q], i + q);
        });
    }
    // The sum of the masses of what f(logit, place) holds for.
    template <typename F>
    __device__ __forceinline__ uint64_t mass_of(F f) const {
        uint64_t all = 0;
        some([&](const float (&x)[kAtOnce], int i) {
            bool in[kAtOnce], any = false;
#pragma unroll
            for (int q = 0; q < kAtOnce; ++q) any |= in[q] = f(x[q], i + q);
            if (!__any_sync(__activemask(), any)) return;
            int64_t m[kAtOnce];
            masses(x, m);
#pragma unroll
            for (int q = 0; q < kAtOnce; ++q) all += in[q] ? static_cast<uint64_t>(m[q] - kWholeBits) : 0;
        });
        return all;
    }

    // What a block tells lies in one of two places in turn: when one is written again all have been at a barrier since they read it.
    __device__ __forceinline__ uint64_t* tell() { return s.said[exchanges++ & 1]; }
    // Sum (or maximum) over the block, in its first warp.
    template <bool MAX>
    __device__ uint64_t over_warps(uint64_t v) {
        v = MAX ? warp_max(v) : warp_sum(v);
        __syncthreads();
        if ((threadIdx.x & 31) == 0) s.red[threadIdx.x >> 5] = v;
        __syncthreads();
        if (threadIdx.x >= 32) return 0;
        v = threadIdx.x < kDrawWarps ? s.red[threadIdx.x] : 0;
        return MAX ? warp_max(v) : warp_sum(v);
    }
    // The same over the cluster, in all threads; `before`: over the blocks in front of this one.
    template <bool MAX>
    __device__ uint64_t over_cluster(uint64_t v, uint64_t* before = nullptr) {
        v = over_warps<MAX>(v);
        uint64_t* said = tell();
        if (threadIdx.x == 0) said[0] = v;
        sm100::cluster_sync();
        if (threadIdx.x < 32) heard<MAX>(said, 0);
        __syncthreads();
        if (before) *before = s.told[1];
        return s.told[0];
    }
    // (the first warp) what the blocks have said, into told[at], and of a sum what the blocks in front of this one have, behind it
    template <bool MAX>
    __device__ __forceinline__ void heard(const uint64_t* said, int at) {
        const int self = static_cast<int>(sm100::cluster_rank()), lane = threadIdx.x;
        const uint64_t o = lane < blocks ? peer_u64(said, lane) : 0;
        const uint64_t all = MAX ? warp_max(o) : warp_sum(o);
        if (lane == 0) s.told[at] = all;
        if (!MAX) {
            const uint64_t front = warp_sum(lane < self ? o : 0);
            if (lane == 0) s.told[at + 1] = front;
        }
    }

    // The sum of a variable of all blocks, all of them fetched at once.
    __device__ __forceinline__ uint64_t over_blocks(const uint64_t* p) const {
        uint64_t v[kMostBlocks], sum = 0;
#pragma unroll
        for (int o = 0; o < kMostBlocks; ++o) v[o] = o < blocks ? peer_u64(p, o) : 0;
#pragma unroll
        for (int o = 0; o < kMostBlocks; ++o) sum += v[o];
        return sum;
    }
    __device__ __forceinline__ uint32_t over_blocks(const uint32_t* p) const {
        uint32_t v[kMostBlocks], sum = 0;
#pragma unroll
        for (int o = 0; o < kMostBlocks; ++o) v[o] = o < blocks ? peer_u32(p, o) : 0;
#pragma unroll
        for (int o = 0; o < kMostBlocks; ++o) sum += v[o];
        return sum;
    }

    // ---- bins: cleared, added to, told to the cluster, gathered
    __device__ void clear_bins() {
        for (int b = threadIdx.x; b < kBins; b += kDrawThreads) {
            s.count[b] = 0;
#pragma unroll
            for (int i = 0; i < kPieces; ++i) s.pieces[i][b] = 0;
        }
    }
    // Sums of 64 bits by additions of 32, which shared memory does by itself: a mass is cut into pieces so short that no sum of them overflows.
    __device__ __forceinline__ void add_mass(int b, uint64_t m) {
        for (int i = 0; m; ++i, m >>= piece) atomicAdd(&s.pieces[i][b], static_cast<uint32_t>(m) & ((1u << piece) - 1));
    }
    // (behind a barrier)
    __device__ void tell_bins(int buffer, bool masses) {
        for (int b = threadIdx.x; b < kBins; b += kDrawThreads) {
            s.bin_count[buffer][b] = s.count[b];
            if (!masses) continue;
            uint64_t m = 0;
#pragma unroll
            for (int i = kPieces - 1; i >= 0; --i) m = (m << piece) + s.pieces[i][b];
            s.bin_mass[buffer][b] = m;
        }
    }
    // (behind the cluster's barrier)
    __device__ void gather_bins(int buffer, bool masses) {
        for (int b = threadIdx.x; b < 2 * kBins; b += kDrawThreads) {
            if (b < kBins) {
                if (masses) s.all_mass[b] = over_blocks(&s.bin_mass[buffer][b]);
            } else {
                s.all_count[b - kBins] = over_blocks(&s.bin_count[buffer][b - kBins]);
            }
        }
        __syncthreads();
    }
};

// The least key from lo to hi for which in(key) holds, which does for hi and for all keys above one for which it does; asked by whole warps.
template <typename F>
__device__ __forceinline__ uint32_t least_key(uint32_t lo, uint32_t hi, F in) {
    while (lo < hi) {                                          // a lane a place: a 32nd of what is left
        const uint32_t step = ((hi - lo) >> 5) + 1, mine = static_cast<uint32_t>(min(static_cast<uint64_t>(hi), lo + static_cast<uint64_t>(threadIdx.x & 31) * step));
        const uint32_t found = __ballot_sync(~0u, in(mine));
        const int at = found ? __ffs(found) - 1 : 32;          // the first of the lanes; `hi` if there is none
        const uint32_t up = at < 32 ? __shfl_sync(~0u, mine, at & 31) : hi, down = at ? __shfl_sync(~0u, mine, (at - 1) & 31) + 1 : lo;
        hi = up;
        lo = at ? down : up;
    }
    return lo;
}

// Bins of an interval of keys [low, high], the highest first.  Even in the logits where it is wide, in the keys where it is not or `by_key` says so.
template <int N>
struct Bins {
    uint32_t low, high;
    bool by_key;
    int shift;
    float top, per;                // half the highest logit, bins for half a unit

    // `end`: the logit that the bins reach down to; what is lower is in the last one
    __device__ Bins(uint32_t low_, uint32_t high_, bool keys, float end) : low(low_), high(high_), shift(0), top(0.f), per(0.f) {
        const uint32_t range = high - low;
        by_key = keys || range < (1u << 24) || high >= kHighest;
        if (by_key) shift = max(0, 32 - __clz(range) - (31 - __clz(N)));       // range >> shift < N
        else {
            top = 0.5f * value_of(high);
            per = fminf(N / (top - 0.5f * end), 3.0e38f);
        }
    }
    __device__ Bins(uint32_t low_, uint32_t high_, bool keys) : Bins(low_, high_, keys, value_of(low_)) {}
    __device__ __forceinline__ int operator()(float x) const {           // never rises with the logit
        if (by_key) return static_cast<int>((high - key_of(x)) >> shift);
        // (cut off to a whole number by a sum whose lower bits are it: a conversion goes at a quarter of the rate)
        return static_cast<int>(__float_as_uint(__fadd_rd(fminf((top - 0.5f * x) * per, N - 1.f), 8388608.f)) & (N - 1));
    }
    // The least key of bin b or a higher one; asked by whole warps.
    __device__ uint32_t least(int b) const {
        if (by_key) {
            const uint64_t down = (static_cast<uint64_t>(b + 1) << shift) - 1;
            return down >= high - low ? low : high - static_cast<uint32_t>(down);
        }
        return least_key(low, high, [&](uint32_t k) { return (*this)(value_of(k)) <= b; });      // `high` is in bin 0
    }
};

// The first bin at which `above` and the weights (masses, or counts) of the bins from the highest on reach `target`, kBins where they do not; `above` becomes what is
// above that bin.
__device__ int locate(DrawShared& s, bool by_mass, uint64_t target, uint64_t& above) {
    constexpr int kEach = kBins / 32;
    const int tid = threadIdx.x;
    if (tid < 32) {
        uint64_t w[kEach], mine = 0;
#pragma unroll
        for (int b = 0; b < kEach; ++b) {
            w[b] = by_mass ? s.all_mass[tid * kEach + b] : s.all_count[tid * kEach + b];
            mine += w[b];
        }
        const uint64_t run = above + warp_scan(mine);
        const uint32_t reached = __ballot_sync(~0u, run >= target);
        if (tid == (reached ? __ffs(reached) - 1 : 31)) {
            uint64_t at = reached ? run - mine : run;
            int b = reached ? 0 : kEach;
#pragma unroll
            for (int i = 0; i < kEach; ++i)
                if (b == i && at + w[i] < target) {
                    at += w[i];
                    ++b;
                }
            s.word[0] = reached ? tid * kEach + b : kBins;
            s.word[1] = at;
        }
    }
    __syncthreads();
    const int bin = static_cast<int>(s.word[0]);
    above = s.word[1];
    __syncthreads();
    return bin;
}

// The ids from `low` to `high`, down to `last`; from all blocks of the cluster there are kRanked at most.
template <typename T>
__device__ __forceinline__ void pick_ids(Row<T>& row, uint32_t low, uint32_t high, Cut last, bool listed) {
    DrawShared& s = row.s;
    const float from = value_of(low), to = upper_value(high), end = value_of(last.key);
    if (threadIdx.x == 0) s.pick_n = 0;
    __syncthreads();
    const auto pick = [&](float x, int id) {
        if (!(x >= from && x <= to) || (x == end && id > last.id)) return;
        const uint32_t at = atomicAdd(&s.pick_n, 1u);
        s.pick_key[at] = key_of(x);
        s.pick_id[at] = id;
    };
    if (listed)
        for (int i = threadIdx.x; i < static_cast<int>(s.list_n); i += kDrawThreads) pick(value_of(row.list_key[i]), row.list_id[i]);
    else
        row.each([&](float x, int i) { pick(x, row.first + i); });
}
// (behind the cluster's barrier)
template <typename T>
__device__ void gather_picked(Row<T>& row) {
    DrawShared& s = row.s;
    static_assert(kRanked <= kDrawThreads, "a thread an id");
    if (threadIdx.x >= kRanked) return;
    int n[kMostBlocks], at = threadIdx.x, b = -1;
#pragma unroll
    for (int o = 0; o < kMostBlocks; ++o) n[o] = o < row.blocks ? static_cast<int>(peer_u32(&s.pick_n, o)) : 0;
#pragma unroll
    for (int o = 0; o < kMostBlocks; ++o)
        if (b < 0) {
            if (at < n[o]) b = o;
            else at -= n[o];
        }
    if (b >= 0) {
        const uint32_t k = peer_u32(&s.pick_key[at], b);
        s.rank_key[threadIdx.x] = k;
        s.rank_id[threadIdx.x] = static_cast<int>(peer_u32(&s.pick_id[at], b));
        s.rank_mass[threadIdx.x] = row.mass(value_of(k));
    }
}

// f(i, how many come first, their mass) once for each of the n ids in rank_key and so on, in one lane: eight lanes an id at a time.
template <typename F>
__device__ __forceinline__ void rank_ids(DrawShared& s, int n, F f) {
    const int part = threadIdx.x & 7;
    for (int base = 0; base < n; base += kDrawThreads / 8) {
        const int c = base + (threadIdx.x >> 3);
        const bool here = c < n;
        const uint32_t k = here ? s.rank_key[c] : 0;
        const int id = here ? s.rank_id[c] : 0;
        int higher = 0;
        uint64_t above = 0;
        for (int o = part; o < n; o += 8) {
            const uint32_t other = s.rank_key[o];
            const bool first = other > k || (other == k && s.rank_id[o] < id);
            higher += first;
            above += first ? s.rank_mass[o] : 0;
        }
#pragma unroll
        for (int d = 4; d; d >>= 1) {
            higher += __shfl_xor_sync(~0u, higher, d);
            above += __shfl_xor_sync(~0u, above, d);
        }
        if (part == 0 && here) f(c, higher, above);
    }
}

// The id at which the running weight (ids, or their masses), from the top down to `last`, reaches `target`; `last` where it never does.  What is above `high`
// weighs `above`, and `low` is how far to look first.  `listed`: ids from `low` to `high` are in the blocks' lists, and it is among them.
template <typename T>
__device__ __forceinline__ Cut find_cut(Row<T> row, bool by_mass, uint64_t target, Cut last, uint32_t low, uint32_t high, uint64_t above, bool listed) {
    // (exchanges are made twice or not at all; bins are told from the second place on, which is free)
    DrawShared& s = row.s;
    int buffer = 1;
    bool far = false;                          // below what was looked at first, where logits of any size may lie
    const int tid = threadIdx.x;
    const float end = value_of(last.key);
    const auto among = [&](float x, int i) { return x > end || (x == end && row.first + i <= last.id); };
    for (int round = 0;; ++round) {
        const Bins<kBins> bins(low, high, far || round >= 6);
        const float from = value_of(low), to = upper_value(high);
        row.clear_bins();
        __syncthreads();
        if (listed) {
            for (int i = tid; i < static_cast<int>(s.list_n); i += kDrawThreads) {
                const float x = value_of(row.list_key[i]);
                if (!(x >= from && x <= to)) continue;
                const int b = bins(x);
                atomicAdd(&s.count[b], 1u);
                if (by_mass) row.add_mass(b, row.mass(x));
            }
        } else {
            row.each([&](float x, int i) {
                if (!(x >= from && x <= to) || !among(x, i)) return;
                const int b = bins(x);
                atomicAdd(&s.count[b], 1u);
                if (by_mass) row.add_mass(b, row.mass(x));
            });
        }
        __syncthreads();
        row.tell_bins(buffer, by_mass);
        sm100::cluster_sync();
        row.gather_bins(buffer, by_mass);
        buffer ^= 1;
        const int bin = locate(s, by_mass, target, above);
        if (bin == kBins) {
            if (low <= last.key) {
                sm100::cluster_sync();                         // (bins may be told again)
                return last;
            }
            high = low - 1;
            low = last.key;
            far = true;
            continue;
        }
        const uint32_t in_bin = s.all_count[bin], next_low = bins.least(bin);
        if (bin > 0) high = bins.least(bin - 1) - 1;
        low = next_low;
        if (in_bin <= kRanked) {
            // Few: each is ranked among all.
            pick_ids(row, low, high, last, listed);
            sm100::cluster_sync();
            gather_picked(row);
            __syncthreads();
            rank_ids(s, static_cast<int>(in_bin), [&](int i, int higher, uint64_t mass_above) {
                const uint64_t before = above + (by_mass ? mass_above : higher);
                if (before < target && target <= before + (by_mass ? s.rank_mass[i] : 1)) s.cut = Cut{s.rank_key[i], s.rank_id[i]};
            });
            __syncthreads();
            const Cut cut = s.cut;
            sm100::cluster_sync();                             // (what has been picked may be written again)
            return cut;
        }
        if (low < high) continue;
        // Equal logits: of the ids in their order as many as it takes.
        const float x0 = value_of(low);
        const uint64_t one = by_mass ? row.mass(x0) : 1, want = (target - above + one - 1) / one;
        if (want >= in_bin) {
            sm100::cluster_sync();
            return low == last.key ? last : Cut{low, 0x7FFFFFFF};
        }
        uint64_t mine = 0, before = 0;
        row.each([&](float x, int i) { mine += x == x0 && among(x, i); });
        mine = warp_sum(mine);
        if (tid == 0) s.word[2] = 0;
        row.template over_cluster<false>((tid & 31) == 0 ? mine : 0, &before);
        for (int w = 0; w < tid >> 5; ++w) before += s.red[w];             // (as over_cluster left them)
        __syncthreads();
        if (before < want && want <= before + mine) {          // one warp of one block; the others' word stays 0
            const int begin = (tid >> 5) * row.segment, stop = min(begin + row.segment, row.count);
            for (int j = begin; j < stop; j += 32) {
                const int i = j + (tid & 31);
                const bool one_of = i < stop && row.value(i) == x0 && among(x0, i);
                const uint32_t ballot = __ballot_sync(~0u, one_of);
                const uint64_t upto = before + __popc(ballot & (~0u >> (31 - (tid & 31))));
                if (one_of && upto == want) s.word[2] = static_cast<uint64_t>(row.first + i) + 1;
                before += __popc(ballot);
            }
        }
        __syncthreads();
        const uint64_t id = row.template over_cluster<true>(tid == 0 ? s.word[2] : 0);
        return Cut{low, static_cast<int>(id) - 1};
    }
}

__device__ __forceinline__ uint64_t place_of(double u, uint64_t kept) {
    const uint64_t at = static_cast<uint64_t>(u * static_cast<double>(kept));
    return at < kept ? at : kept - 1;
}

// FINE: rows of more than kOneUnit ids, each with a unit of its own.
template <typename T, bool FINE>
__global__ void __launch_bounds__(kDrawThreads, 2) draw_kernel(const __grid_constant__ DrawArgs a) {
    extern __shared__ uint4 smem[];
    DrawShared& s = *reinterpret_cast<DrawShared*>(smem);
    uint32_t* lists = reinterpret_cast<uint32_t*>(&s + 1);
    Placed& placed = *reinterpret_cast<Placed*>(lists);
    float* held = reinterpret_cast<float*>(lists + 2 * a.listed);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    after_previous();
    let_next_begin();
    const int64_t r = blockIdx.x / a.blocks;
    const int block = static_cast<int>(sm100::cluster_rank());
    const int share = a.segment * kDrawWarps, first = block * share;
    const float heat = a.temperature ? a.temperature[r] : a.one_temperature, top_p = a.top_p ? a.top_p[r] : a.one_top_p, min_p = a.min_p ? a.min_p[r] : a.one_min_p;
    const int top_k = a.top_k ? a.top_k[r] : a.one_top_k;
    const double u = a.wide_u ? static_cast<const double*>(a.u)[r] : static_cast<double>(static_cast<const float*>(a.u)[r]);

    Row<T> row{s, a.held ? held : nullptr, static_cast<const T*>(a.logits) + r * a.stride + first, first, max(0, min(share, a.vocab - first)), a.segment, a.blocks, a.piece,
               lists, reinterpret_cast<int*>(lists + a.listed), 0, uint64_t{1} << a.fixed, 0.0, 46.166241308446829 / static_cast<double>(heat), -32.0 * (a.fixed + 1),
               0.f, true, 0};
    if (tid < 32) s.power[tid] = a.power[tid];
    if (tid == 0) s.list_n = 0;
    row.clear_bins();
    for (int b = tid; b < kGuessBins; b += kDrawThreads) s.guess[b] = 0;

    // ---- The row is fetched; its largest logit and, for guesses, mean and deviation.
    float most = -INFINITY, sum = 0.f, squares = 0.f, finite = 0.f;
    bool nan = false;
    {
        constexpr int N = 16 / sizeof(T), kFetch = 32 / N;                     // 128 bytes under way a thread
        const auto take = [&](float x, int i) {
            if (a.held) held[i] = x;
            most = fmaxf(most, x);
            nan |= x != x;
        };
        // 16 bytes at a time from the first whole ones on, ids in front of these and behind by themselves
        const int head = min(row.count, static_cast<int>((16 - reinterpret_cast<uintptr_t>(row.in) % 16) % 16 / sizeof(T))), lumps = (row.count - head) / N;
        const Lump<T, N>* body = reinterpret_cast<const Lump<T, N>*>(row.in + head);
        for (int l = tid; l < lumps; l += kDrawThreads * kFetch) {
            Lump<T, N> v[kFetch];
#pragma unroll
            for (int q = 0; q < kFetch; ++q)
                if (l + q * kDrawThreads < lumps) v[q] = body[l + q * kDrawThreads];
#pragma unroll
            for (int q = 0; q < kFetch; ++q)
                if (l + q * kDrawThreads < lumps) {
#pragma unroll
                    for (int e = 0; e < N; ++e) take(to_float<T>(v[q].v[e]), head + (l + q * kDrawThreads) * N + e);
                    const float x = to_float<T>(v[q].v[0]), in = x > -INFINITY ? x : 0.f;      // a part of the ids is enough for a guess
                    sum += in;
                    squares = fmaf(in, in, squares);
                    finite += x > -INFINITY ? 1.f : 0.f;
                }
        }
        if (tid < head) take(to_float<T>(row.in[tid]), tid);
        if (tid < row.count - head - lumps * N) take(to_float<T>(row.in[head + lumps * N + tid]), head + lumps * N + tid);
    }
    {
        // to the first warp, to the cluster: key of the largest (kNone for a NaN), sum, squares, count
        const uint32_t key = __reduce_max_sync(~0u, nan ? kNone : key_of(most));
#pragma unroll
        for (int d = 16; d; d >>= 1) {
            sum += __shfl_xor_sync(~0u, sum, d);
            squares += __shfl_xor_sync(~0u, squares, d);
            finite += __shfl_xor_sync(~0u, finite, d);
        }
        if (lane == 0) s.seen[warp] = make_float4(__uint_as_float(key), sum, squares, finite);
        __syncthreads();
        const auto join = [&](float4 v, int n) {
            const uint32_t k = __reduce_max_sync(~0u, lane < n ? __float_as_uint(v.x) : 0);
            if (lane >= n) v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int d = 8; d; d >>= 1) {
                v.y += __shfl_xor_sync(~0u, v.y, d);
                v.z += __shfl_xor_sync(~0u, v.z, d);
                v.w += __shfl_xor_sync(~0u, v.w, d);
            }
            return make_float4(__uint_as_float(k), v.y, v.z, v.w);
        };
        if (warp == 0) {
            const float4 v = join(s.seen[lane & (kDrawWarps - 1)], kDrawWarps);
            if (lane == 0) s.seen_by_block = v;
        }
        sm100::cluster_sync();
        if (warp == 0) {
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            if (lane < a.blocks) {
                const uint32_t* p = reinterpret_cast<const uint32_t*>(&s.seen_by_block);
                v = make_float4(__uint_as_float(peer_u32(p, lane)), __uint_as_float(peer_u32(p + 1, lane)), __uint_as_float(peer_u32(p + 2, lane)),
                                __uint_as_float(peer_u32(p + 3, lane)));
            }
            v = join(v, a.blocks);
            const float mean = v.y / v.w;
            if (lane == 0) s.seen[0] = make_float4(v.x, mean, sqrtf(fmaxf(v.z / v.w - mean * mean, 0.f)), v.w * (16 / sizeof(T)));
        }
        __syncthreads();
    }
    row.top = __float_as_uint(s.seen[0].x);
    const float mean = s.seen[0].y, deviation = s.seen[0].z, finite_ids = s.seen[0].w;
    const bool bad = row.top == kNone || !(heat >= 0.f && heat <= 3.402823466e38f) || !(u >= 0.0 && u < 1.0) || top_p != top_p || min_p != min_p;
    if (bad || row.top <= kLowest) {
        if (block == 0 && tid == 0) {
            a.ids[r] = -1;
            a.logprobs[r] = bad ? __int_as_float(0x7FC00000) : -INFINITY;
        }
        return sm100::cluster_sync();
    }
    const float most_value = value_of(row.top);
    const bool one = top_k == 1 || min_p > 1.f || top_p <= 0.f || heat == 0.f;  // the first one only
    int best = 0;
    if (one) {
        uint32_t left = 0;                     // ids from the first one on, at most
        row.each([&](float x, int i) {
            if (x == most_value) left = max(left, static_cast<uint32_t>(a.vocab - row.first - i));
        });
        best = a.vocab - static_cast<int>(row.template over_cluster<true>(left));
        if (heat == 0.f) {
            if (block == 0 && tid == 0) {
                a.ids[r] = best;
                a.logprobs[r] = 0.f;
            }
            return sm100::cluster_sync();
        }
    }
    row.top_value = static_cast<double>(most_value);
    int fixed = a.fixed;
    const auto set_floor = [&] {
        // a logit whose mass is a quarter of a unit, and that it is one that the table's exponents go down to
        const double down = row.top_value - (fixed + 2) * 0.69314718055994531 * static_cast<double>(heat);
        row.floor = __double2float_rd(down);
        const double y = (static_cast<double>(row.floor) - row.top_value) * row.steps;
        row.plain = row.top < kHighest && down > -3.4e38 && y <= row.least && y > -32.0 * 900;
    };
    set_floor();
    if constexpr (FINE) {
        // So many ids that units for all of them alike would be coarse: the total says how fine they may be (it is the same whatever the blocks are).
        uint64_t mine = 0;
        row.some([&](const float (&x)[Row<T>::kAtOnce], int) {
            int64_t m[Row<T>::kAtOnce];
            row.masses(x, m);
#pragma unroll
            for (int q = 0; q < Row<T>::kAtOnce; ++q) mine += static_cast<uint64_t>(m[q] - kWholeBits);
        });
        const uint64_t coarse = row.template over_cluster<false>(mine) + a.vocab;
        int finer = 0;
        while (fixed + finer < kFinest && coarse << (finer + 1) <= 1ull << 61) ++finer;
        fixed += finer;
        row.largest <<= finer;
        row.least = -32.0 * (fixed + 1);
        if (tid < 32) s.power[tid] *= static_cast<double>(1 << finer);
        __syncthreads();
        set_floor();
    }

    const bool by_k = !one && top_k > 0 && top_k < a.vocab, by_p = !one && top_p < 1.f, by_min = !one && min_p > 0.f && row.top < kHighest;
    const Cut all{kLowest + 1, 0x7FFFFFFF};
    Cut cut = all;
    // the least key with d / T >= log(min_p)
    uint32_t min_key = kLowest + 1;
    if (by_min) {
        const double depth = log(static_cast<double>(min_p)) * static_cast<double>(heat);
        min_key = least_key(min_key, row.top, [&](uint32_t k) { return static_cast<double>(value_of(k)) - row.top_value >= depth; });
    }
    // What is near: some 400 ids, more than top_k in any case, if logits were distributed normally (the quantile by Abramowitz and Stegun's 26.2.22), and nothing that is
    // more than 12 below the largest where that may leave out no id of the top_k.
    const float part = fminf(fmaxf(by_k ? 1.5f * top_k + 100.f : 400.f, 1.f) / fmaxf(finite_ids, 1.f), 0.5f), t = sqrtf(-2.f * logf(part));
    const float above_mean = part < 0.5f ? t - (2.30753f + 0.27061f * t) / (1.f + t * (0.99229f + 0.04481f * t)) : -8.f;
    uint32_t near = row.top < kHighest ? key_of(fminf(fmaxf(mean + above_mean * deviation, by_k ? -INFINITY : most_value - 12.f), most_value)) : row.top;
    if (near > row.top || near <= kLowest) near = row.top;
    const float near_value = value_of(near);
    float rest_end = fmaxf(mean - 3.f * deviation, near_value - 64.f * fmaxf(1.f, heat));
    if (!(rest_end < near_value)) rest_end = near_value - 1.f;
    const bool weigh = by_p && !by_k;          // the first cut goes by masses, not by numbers
    const bool cuts = by_k || by_p || by_min, guess = by_p && !by_k && near > kLowest + 1 && near < kHighest;
    const Bins<kBins> near_bins(near, row.top, false);
    const Bins<kGuessBins> rest_bins(kLowest + 1, guess ? near - 1 : kLowest + 1, false, rest_end);

    // ---- The total, and bins of what is near.
    uint64_t mine = 0;
    if (!cuts) {
        row.some([&](const float (&x)[Row<T>::kAtOnce], int) {
            int64_t m[Row<T>::kAtOnce];
            row.masses(x, m);
#pragma unroll
            for (int q = 0; q < Row<T>::kAtOnce; ++q) mine += static_cast<uint64_t>(m[q]);
            mine -= Row<T>::kAtOnce * static_cast<uint64_t>(kWholeBits);
        });
    } else {
        row.some([&](const float (&x)[Row<T>::kAtOnce], int) {
            int64_t m[Row<T>::kAtOnce];
            row.masses(x, m);
            bool any = false;
#pragma unroll
            for (int q = 0; q < Row<T>::kAtOnce; ++q) {
                mine += static_cast<uint64_t>(m[q]);
                any |= x[q] >= near_value;
            }
            mine -= Row<T>::kAtOnce * static_cast<uint64_t>(kWholeBits);
            if (guess) {
                int b[Row<T>::kAtOnce];
#pragma unroll
                for (int q = 0; q < Row<T>::kAtOnce; ++q) b[q] = rest_bins(x[q]);
#pragma unroll
                for (int q = 0; q < Row<T>::kAtOnce; ++q)
                    if (x[q] < near_value && x[q] > -INFINITY) atomicAdd(&s.guess[b[q]], 1u);
            }
            // (few and far between: they are listed, and added up together afterwards)
            if (any)
                for (int q = 0; q < Row<T>::kAtOnce; ++q) {
                    if (!(x[q] >= near_value)) continue;
                    const uint32_t at = atomicAdd(&s.list_n, 1u);
                    if (at < a.listed) row.list_key[at] = __float_as_uint(x[q]);
                    else {
                        atomicAdd(&s.count[near_bins(x[q])], 1u);
                        if (weigh) row.add_mass(near_bins(x[q]), static_cast<uint64_t>(m[q] - kWholeBits));
                    }
                }
        });
        __syncthreads();
        for (int i = tid; i < min(static_cast<int>(s.list_n), a.listed); i += kDrawThreads) {
            const float x = __uint_as_float(row.list_key[i]);
            const int b = near_bins(x);
            atomicAdd(&s.count[b], 1u);
            if (weigh) row.add_mass(b, row.mass(x));
        }
    }
    mine = warp_sum(mine);
    if (lane == 0) s.warp_mass[warp] = mine;
    uint64_t before = 0;
    if (cuts) {
        __syncthreads();
        row.tell_bins(0, weigh);
    }
    const uint64_t total = row.template over_cluster<false>(lane == 0 ? mine : 0, &before);
    if (cuts) {
        row.gather_bins(0, weigh);
    }

    const auto logprob = [&](float x) {
        const double down = row.top == kHighest ? 0.0 : (static_cast<double>(x) - row.top_value) / static_cast<double>(heat);
        // (the total in parts of the largest, which is exact and 1 at least: an id that has all of it gets 0, and none more)
        return static_cast<float>(down - log(static_cast<double>(total) * __hiloint2double((1023 - fixed) << 20, 0)));
    };
    if (one) {
        if (block == 0 && tid == 0) {
            a.ids[r] = best;
            a.logprobs[r] = logprob(most_value);
        }
        return sm100::cluster_sync();
    }

    uint64_t kept = total;
    const auto p_target = [&] {
        const uint64_t want = static_cast<uint64_t>(ceil(static_cast<double>(top_p) * static_cast<double>(kept)));
        return larger(1, want < kept ? want : kept);
    };
    bool summed = true;                        // warp_mass and `before` hold what is kept
    if (cuts) {
        // The bin of what is near in which the first cut lies, kBins if it lies lower.
        uint64_t above = 0, target = 0;
        int bin = kBins;
        if (by_k || by_p) {
            target = by_k ? static_cast<uint64_t>(top_k) : p_target();
            bin = locate(s, !by_k, target, above);
        }
        // The last bin of which ids may be kept, and how many there are down to its end.  (Of both top_k and top_p it takes all of the top_k to say where the latter cuts.)
        const int end_bin = by_min && min_key >= near && !(by_k && by_p) ? min(bin, near_bins(value_of(min_key))) : bin;
        uint32_t ids = 0;
        for (int b = lane; b < kBins; b += 32)
            if (b <= end_bin) ids += s.all_count[b];
        ids = __reduce_add_sync(~0u, ids);
        if (end_bin < kBins && ids <= kRanked) {
            // ---- Few candidates: the first block ranks them, cuts and draws.
            pick_ids(row, near_bins.least(end_bin), row.top, all, false);
            sm100::cluster_sync();
            if (block == 0) {
                gather_picked(row);
                __syncthreads();
                const int n = static_cast<int>(ids);
                rank_ids(s, n, [&](int i, int higher, uint64_t mass_above) {
                    placed.place[i] = higher;
                    placed.in_front[i] = mass_above;
                });
                __syncthreads();
                const bool here = tid < n;
                const uint32_t k = here ? s.rank_key[tid] : 0;
                const uint64_t m = here ? s.rank_mass[tid] : 0;
                bool keep = here;
                if (by_k) {
                    keep = keep && placed.place[tid] < top_k;
                    if (here && placed.place[tid] == min(top_k, n) - 1) s.word[2] = placed.in_front[tid] + m;
                    __syncthreads();
                    kept = s.word[2];
                }
                if (by_p) keep = keep && placed.in_front[tid] < p_target();
                if (by_min) keep = keep && k >= min_key;
                const uint64_t some = row.template over_warps<false>(keep ? m : 0);
                if (tid == 0) s.word[2] = some;
                if (here && !keep) s.rank_mass[tid] = 0;
                __syncthreads();
                const uint64_t at = place_of(u, s.word[2]);
                for (int base = 0; base < n; base += kDrawThreads / 8) {
                    const int c = base + (tid >> 3);
                    const int id = c < n ? s.rank_id[c] : 0;
                    const uint64_t own = c < n ? s.rank_mass[c] : 0;
                    uint64_t run = 0;
                    for (int o = tid & 7; o < n; o += 8) run += s.rank_id[o] < id ? s.rank_mass[o] : 0;
#pragma unroll
                    for (int d = 4; d; d >>= 1) run += __shfl_xor_sync(~0u, run, d);
                    if ((tid & 7) == 0 && run <= at && at < run + own) {
                        a.ids[r] = id;
                        a.logprobs[r] = logprob(value_of(s.rank_key[c]));
                    }
                }
            }
            return sm100::cluster_sync();
        }
        // ---- The cuts one after another.
        summed = false;
        bool done = false;
        if (by_p && !by_k && bin == kBins && guess) {
            // About where the cut lies, from the counts of the rest's bins: a bin's ids at its middle.
            for (int b = tid; b < kGuessBins; b += kDrawThreads) {
                const uint32_t c = row.over_blocks(&s.guess[b]);
                const float middle = rest_bins.by_key ? near_value : 2.f * (rest_bins.top - (b + 0.5f) / rest_bins.per);
                s.all_guess[b] = static_cast<float>(c) * expf((middle - most_value) / heat);
            }
            __syncthreads();
            if (tid < 32) {
                constexpr int kEach = kGuessBins / 32;
                float part = 0.f;
                for (int b = 0; b < kEach; ++b) part += s.all_guess[tid * kEach + b];
                float run = part;
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) {
                    const float o = __shfl_up_sync(~0u, run, d);
                    if (tid >= d) run += o;
                }
                const float want = static_cast<float>(static_cast<double>(target - above) * exp2(-static_cast<double>(fixed)));
                const uint32_t reached = __ballot_sync(~0u, run >= want);
                if (tid == (reached ? __ffs(reached) - 1 : 31)) {
                    float at = run - part;
                    int b = 0;
                    while (b < kEach - 1 && at + s.all_guess[tid * kEach + b] < want) at += s.all_guess[tid * kEach + b++];
                    s.word[2] = tid * kEach + b;
                }
            }
            if (tid == 0) s.list_n = 0;                        // (what was near has been added up)
            __syncthreads();
            const int around = static_cast<int>(s.word[2]);
            const uint32_t high = around > 1 ? rest_bins.least(around - 2) - 1 : near - 1, low = rest_bins.least(around + 1);
            const float from = value_of(low), to = upper_value(high);
            mine = row.mass_of([&](float x, int i) {
                if (x >= from && x <= to) {
                    const uint32_t at = atomicAdd(&s.list_n, 1u);
                    if (at < a.listed) {
                        row.list_key[at] = key_of(x);
                        row.list_id[at] = row.first + i;
                    }
                }
                return x > to;
            });
            mine = warp_sum(mine);
            if (lane == 0) s.warp_mass[warp] = mine;
            __syncthreads();
            constexpr uint64_t kTooMany = 1ull << 59;          // more than the lists can weigh
            const int listed = static_cast<int>(s.list_n);
            uint64_t in_list = 0;
            for (int i = tid; i < min(listed, a.listed); i += kDrawThreads) in_list += row.mass(value_of(row.list_key[i]));
            in_list = row.template over_warps<false>(in_list);
            const uint64_t sum_above = row.template over_warps<false>(lane == 0 ? mine : 0);
            uint64_t* said = row.tell();
            if (tid == 0) {
                said[0] = sum_above;
                said[1] = listed > a.listed ? kTooMany : in_list;
            }
            sm100::cluster_sync();
            if (warp == 0) {
                row.template heard<false>(said, 0);
                row.template heard<false>(said + 1, 2);
            }
            __syncthreads();
            const uint64_t over = s.told[0], listed_mass = s.told[2];
            if (listed_mass < kTooMany && over < target && target <= over + listed_mass) {
                cut = find_cut(row, true, target, all, low, high, over, true);
                done = true;
                if (!(by_min && min_key > cut.key)) {
                    for (int i = tid; i < listed; i += kDrawThreads) {
                        const uint32_t k = row.list_key[i];
                        const int id = row.list_id[i];
                        if (k > cut.key || (k == cut.key && id <= cut.id))
                            atomicAdd(reinterpret_cast<unsigned long long*>(&s.warp_mass[(id - first) / a.segment]), static_cast<unsigned long long>(row.mass(value_of(k))));
                    }
                    __syncthreads();
                    summed = true;
                    kept = row.template over_cluster<false>(lane == 0 ? s.warp_mass[warp] : 0, &before);
                }
            }
        }
        if (!done && (by_k || by_p)) {
            const bool among_near = bin < kBins;
            if (among_near || near > all.key)
                cut = find_cut(row, !by_k, target, all, among_near ? near_bins.least(bin) : min(near - 1, max(all.key, key_of(rest_end))), !among_near ? near - 1 : bin ? near_bins.least(bin - 1) - 1 : row.top, above,
                               false);
            if (by_k && by_p) {
                const float end = value_of(cut.key);
                kept = row.template over_cluster<false>(row.mass_of([&](float x, int i) { return x > end || (x == end && row.first + i <= cut.id); }));
                cut = find_cut(row, true, p_target(), cut, cut.key, row.top, 0, false);
            }
        }
        if (by_min && min_key > cut.key) cut = Cut{min_key, 0x7FFFFFFF};
    }

    // ---- The draw: the block, the warp and the place at which the running sum of what is kept passes u times the whole.
    const float end = value_of(cut.key);
    const auto in = [&](float x, int i) { return x > end || (x == end && row.first + i <= cut.id); };
    if (!summed) {
        mine = warp_sum(row.mass_of(in));
        __syncthreads();
        if (lane == 0) s.warp_mass[warp] = mine;
        kept = row.template over_cluster<false>(lane == 0 ? mine : 0, &before);
    }
    const uint64_t at = place_of(u, kept);
    int owner = 0;                             // the warp whose ids it is among, in one block
    while (owner < kDrawWarps && at >= before + s.warp_mass[owner]) before += s.warp_mass[owner++];
    // (in the other blocks `before` is more than `at` from the beginning, or the warps run out)
    if (owner < kDrawWarps && at >= before) {
        // The block's warps share that warp's ids, and the one that has it walks through its part.
        const int begin = owner * a.segment, stop = min(begin + a.segment, row.count), part = (a.segment / 32 + kDrawWarps - 1) / kDrawWarps * 32;
        const int from = begin + warp * part, to = min(from + part, stop);
        mine = 0;
        for (int j = from; j < to; j += 32) {
            const int i = j + lane;
            const float x = i < to ? row.value(i) : __int_as_float(0x7FC00000);
            mine += in(x, i) ? row.mass(x) : 0;
        }
        mine = warp_sum(mine);
        if (lane == 0) s.red[warp] = mine;
        __syncthreads();
        for (int w = 0; w < warp; ++w) before += s.red[w];
        if (before <= at && at < before + mine)
            for (int j = from; j < to; j += 32) {
                const int i = j + lane;
                const float x = i < to ? row.value(i) : __int_as_float(0x7FC00000);
                const uint64_t run = warp_scan(in(x, i) ? row.mass(x) : 0);
                const uint32_t passed = __ballot_sync(~0u, before + run > at);
                if (passed) {
                    if (lane == __ffs(passed) - 1) {
                        a.ids[r] = row.first + i;
                        a.logprobs[r] = logprob(x);
                    }
                    break;
                }
                before += __shfl_sync(~0u, run, 31);
            }
    }
    sm100::cluster_sync();                                     // (no block leaves while another may read from it)
}

// Blocks that find an SM each, in clusters of so many: the SMs of a processing cluster (18 or so) that are left over when they are more than two stay idle.
constexpr int alone(int blocks) { return blocks > 2 ? 128 : 148; }

template <typename T>
cudaError_t draw(const DrawArgs& a, int64_t rows, cudaStream_t stream) {
    // Blocks that find an SM each are to have one: no two of them fit.
    int smem = static_cast<int>(sizeof(DrawShared)) + a.listed * 8 + (a.held ? a.segment * kDrawWarps * 4 : 0);
    if (rows * a.blocks <= alone(a.blocks)) smem = std::max(smem, 116 * 1024);
    auto* kernel = a.vocab > kOneUnit ? draw_kernel<T, true> : draw_kernel<T, false>;
    if (cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024)) return e;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(static_cast<unsigned>(rows * a.blocks));
    config.blockDim = dim3(kDrawThreads);
    config.dynamicSmemBytes = smem;
    config.stream = stream;
    cudaLaunchAttribute attrs[2]{};
    attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[0].val.programmaticStreamSerializationAllowed = 1;
    attrs[1].id = cudaLaunchAttributeClusterDimension;
    attrs[1].val.clusterDim.x = a.blocks;
    attrs[1].val.clusterDim.y = attrs[1].val.clusterDim.z = 1;
    config.attrs = attrs;
    config.numAttrs = 2;
    return cudaLaunchKernelEx(&config, kernel, a);
}

const char* said(cudaError_t e) { return e == cudaSuccess ? nullptr : cudaGetErrorString(e); }

}  // namespace

const char* adjust_logits(const AdjustCall& c) {
    const int64_t n = c.logits.rows;
    if (!n) return nullptr;
    AdjustArgs a{};
    a.logits = c.logits.data;
    a.out = const_cast<void*>(c.out.data);
    a.stride = c.logits.stride;
    a.out_stride = c.out.stride;
    a.vocab = static_cast<int>(c.logits.cols);
    a.in_place = a.logits == a.out;
    a.history = c.offsets != nullptr;
    a.ids = c.ids.data;
    a.id_bits = c.ids.bits;
    a.n_ids = c.n_ids;
    a.offsets = c.offsets;
    a.prompt_lengths = c.prompt_lengths;
    a.repetition = c.repetition;
    a.presence = c.presence;
    a.frequency = c.frequency;
    a.one_repetition = c.one_repetition;
    a.one_presence = c.one_presence;
    a.one_frequency = c.one_frequency;
    a.entries = c.entries;
    a.bias_ids = c.bias_ids;
    a.bias = c.bias;
    a.bias_stride = c.bias_stride;
    a.allowed = c.allowed;
    a.allowed_rows = c.allowed_rows;
    a.allowed_count = c.allowed_count;
    a.allowed_stride = c.allowed_stride;
    // 16 bytes at a time where rows of both begin at the same place in them
    const int size = c.logits.type == kF32 ? 4 : 2;
    const auto place = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16; };
    const bool lumps = place(a.logits) == place(a.out) && (n == 1 || (a.stride - a.out_stride) * size % 16 == 0);
    switch (c.logits.type) {
        case kF32: return said(lumps ? adjust<float, 4>(a, n, c.stream) : adjust<float, 1>(a, n, c.stream));
        case kBF16: return said(lumps ? adjust<__nv_bfloat16, 8>(a, n, c.stream) : adjust<__nv_bfloat16, 1>(a, n, c.stream));
        default: return said(lumps ? adjust<__half, 8>(a, n, c.stream) : adjust<__half, 1>(a, n, c.stream));
    }
}

const char* sample(const SampleCall& c) {
    if (!c.logits.rows) return nullptr;
    DrawArgs a{};
    a.logits = c.logits.data;
    a.stride = c.logits.stride;
    a.vocab = static_cast<int>(c.logits.cols);
    // Blocks of a row, by what was measured for 128,256 ids in fp32 without cuts: 8 us and 35 over the blocks where each block has an SM to itself, 1.5 times that where two share
    // one (1.75 for rows in one block), in as many rounds as it takes.  (47 rows with top-k, top-p and min-p: 76, 49, 42 and 55 us in 1, 2, 4 and 8 blocks; 1 row 75, 45, 31
    // and 24; 251 rows 134, 131, 156 and 221.)
    a.blocks = 1;
    while (div_up(a.vocab, a.blocks) > kMostShare) a.blocks *= 2;
    const auto cost = [&](int blocks) {
        const int64_t all = c.logits.rows * blocks;
        return (8 + 35 * (a.vocab / 128256.0) / blocks) * (all <= alone(blocks) ? 1 : (blocks == 1 ? 1.75 : 1.5) * div_up(all, 296));
    };
    for (int blocks = 2 * a.blocks; blocks <= kMostBlocks; blocks *= 2)
        if (cost(blocks) < cost(a.blocks)) a.blocks = blocks;
    a.segment = static_cast<int>(round_up(div_up(a.vocab, a.blocks * kDrawWarps), 32));
    const auto bits = [](int64_t n) {
        int b = 0;
        while ((1ll << b) < n) ++b;
        return b;
    };
    // Sums of a row's masses have at most 62 bits, and a mass no more than kPieces pieces; F depends on the ids alone, not on how many blocks take them.
    a.piece = std::min(16, 32 - bits(a.segment * kDrawWarps));
    a.fixed = std::min(46, 62 - bits(a.vocab));
    for (int i = 0; i < 32; ++i) a.power[i] = std::exp2(a.fixed + i / 32.0);
    // Two blocks to an SM.
    constexpr int64_t kRoom = 113 * 1024 - sizeof(DrawShared);
    a.held = a.segment * kDrawWarps * 4ll + 1024 * 8 <= kRoom;
    a.listed = a.held ? 1024 : 8192;
    a.u = c.u;
    a.wide_u = c.wide_u;
    a.temperature = c.temperature;
    a.top_k = c.top_k;
    a.top_p = c.top_p;
    a.min_p = c.min_p;
    a.one_temperature = c.one_temperature;
    a.one_top_k = c.one_top_k;
    a.one_top_p = c.one_top_p;
    a.one_min_p = c.one_min_p;
    a.ids = c.ids;
    a.logprobs = c.logprobs;
    switch (c.logits.type) {
        case kF32: return said(draw<float>(a, c.logits.rows, c.stream));
        case kBF16: return said(draw<__nv_bfloat16>(a, c.logits.rows, c.stream));
        default: return said(draw<__half>(a, c.logits.rows, c.stream));
    }
}

}  // namespace gtok
