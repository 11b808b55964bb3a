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
// the slice once.  Bound by memory: a logit read and written, a bit of a mask; in place, only what changes.
constexpr int kAdjustThreads = 512;
constexpr int kSpare = 8;                        // ids of the lump in front of a slice
constexpr uint32_t kSaid = 0x80000000u;          // of a count: the id is in the prompt

struct AdjustArgs {
    const void* logits;
    void* out;
    int64_t stride, out_stride, vocab, slices;
    int slice;
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
__global__ void __launch_bounds__(kAdjustThreads) adjust_kernel(const __grid_constant__ AdjustArgs a) {
    extern __shared__ uint4 smem[];
    uint32_t* count = reinterpret_cast<uint32_t*>(smem);                       // [slice + kSpare]
    uint16_t* entry = reinterpret_cast<uint16_t*>(count + a.slice + kSpare);   // [slice + kSpare]: place in the list of biases and 1, where there are any
    float* sums = reinterpret_cast<float*>(entry + a.slice + kSpare);          // [entries]
    int32_t* listed = reinterpret_cast<int32_t*>(sums + a.entries);
    const int tid = threadIdx.x;
    after_previous();
    let_next_begin();
    const int64_t row = blockIdx.x / a.slices;
    const int s = static_cast<int>(blockIdx.x - row * a.slices);
    const T* in = static_cast<const T*>(a.logits) + row * a.stride;
    T* out = static_cast<T*>(a.out) + row * a.out_stride;
    // Lumps lie on 16 bytes of the input, whatever the row begins at; the first one of the row is no whole one.
    const int64_t off = N == 1 ? 0 : static_cast<int64_t>((16 - reinterpret_cast<uintptr_t>(in) % 16) % 16 / sizeof(T));
    const int64_t base = off + static_cast<int64_t>(s) * a.slice - N;          // id of count[0]
    const int64_t begin = s == 0 ? 0 : base + N, end = base + N + a.slice < a.vocab ? base + N + a.slice : a.vocab;

    for (int i = tid; i < (a.slice + kSpare) / 4; i += kAdjustThreads) reinterpret_cast<uint4*>(count)[i] = make_uint4(0, 0, 0, 0);
    if (a.entries) {
        for (int i = tid; i < (a.slice + kSpare) / 8; i += kAdjustThreads) reinterpret_cast<uint4*>(entry)[i] = make_uint4(0, 0, 0, 0);
        for (int i = tid; i < a.entries; i += kAdjustThreads) listed[i] = a.bias_ids[row * a.bias_stride + i];
    }
    __syncthreads();
    if (a.history) {
        int64_t from = a.offsets[row], to = a.offsets[row + 1];
        from = from < 0 ? 0 : from;
        to = to > a.n_ids ? a.n_ids : to;
        const int64_t behind = from + (a.prompt_lengths ? a.prompt_lengths[row] : 0);
#pragma unroll 4
        for (int64_t i = from + tid; i < to; i += kAdjustThreads) {
            const int64_t id = a.id_bits == 64 ? static_cast<const int64_t*>(a.ids)[i] : static_cast<const int32_t*>(a.ids)[i];
            if (id < begin || id >= end) continue;
            if (i < behind) atomicOr(&count[id - base], kSaid);
            else atomicAdd(&count[id - base], 1u);
        }
    }
    // An id's biases are added up in the order of the list, at its first entry.
    for (int i = tid; i < a.entries; i += kAdjustThreads) {
        const int64_t id = listed[i];
        if (id < begin || id >= end) continue;
        bool first = true;
        for (int j = 0; j < i && first; ++j) first = listed[j] != id;
        if (!first) continue;
        float sum = 0.f;
        for (int j = i; j < a.entries; ++j)
            if (listed[j] == id) sum += a.bias[row * a.bias_stride + j];
        sums[i] = sum;
        entry[id - base] = static_cast<uint16_t>(i + 1);
    }
    __syncthreads();

    const float rho = a.repetition ? a.repetition[row] : a.one_repetition, presence = a.presence ? a.presence[row] : a.one_presence,
                frequency = a.frequency ? a.frequency[row] : a.one_frequency;
    const uint32_t* words = nullptr;
    bool nothing = false;                              // a mask that is not there allows nothing
    if (a.allowed) {
        const int64_t which = a.allowed_rows ? a.allowed_rows[row] : row;
        if (which >= a.allowed_count) nothing = true;
        else if (which >= 0) words = reinterpret_cast<const uint32_t*>(a.allowed) + which * a.allowed_stride;
    }
    const auto changed = [&](float x, uint32_t c, int e, bool allowed) {
        if (c) {
            x = x > 0.f ? x / rho : x * rho;
            const uint32_t times = c & ~kSaid;
            if (times) x = x - frequency * static_cast<float>(times) - presence;
        }
        if (e) x += sums[e - 1];
        return allowed ? x : -INFINITY;
    };
    for (int64_t v0 = base + (s == 0 ? 0 : N) + static_cast<int64_t>(tid) * N; v0 < end; v0 += kAdjustThreads * N) {
        if (N == 1 || (v0 >= 0 && v0 + N <= a.vocab)) {
            if (v0 < 0) continue;                      // (single elements: the one before the row)
            uint32_t allowed = nothing ? ~((1u << N) - 1) : ~0u;
            if (words) {
                const uint32_t low = words[v0 >> 5], high = words[(v0 + N - 1) >> 5];
                allowed = __funnelshift_r(low, high, v0 & 31) | ~((1u << N) - 1);
            }
            uint32_t c[N], e[N], any = 0;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                c[i] = count[v0 - base + i];
                e[i] = a.entries ? entry[v0 - base + i] : 0;
                any |= c[i] | e[i];
            }
            if (a.in_place && !any && allowed == ~0u) continue;
            Lump<T, N> x = *reinterpret_cast<const Lump<T, N>*>(in + v0);
            if (any || allowed != ~0u)
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (c[i] || e[i] || !(allowed >> i & 1)) x.v[i] = from_float<T>(changed(to_float<T>(x.v[i]), c[i], static_cast<int>(e[i]), allowed >> i & 1));
            *reinterpret_cast<Lump<T, N>*>(out + v0) = x;
        } else {
            for (int i = 0; i < N; ++i) {
                const int64_t v = v0 + i;
                if (v < 0 || v >= a.vocab) continue;
                const bool allowed = !nothing && (!words || (words[v >> 5] >> (v & 31) & 1));
                const uint32_t c = count[v - base];
                const int e = a.entries ? entry[v - base] : 0;
                T x = in[v];
                if (c || e || !allowed) x = from_float<T>(changed(to_float<T>(x), c, e, allowed));
                out[v] = x;
            }
        }
    }
}

template <typename T, int N>
cudaError_t adjust(AdjustArgs a, int64_t rows, cudaStream_t stream) {
    // Slices of 16,384 ids count a long history least often; of fewer where that leaves SMs without work.
    a.slice = 16384;
    while (a.slice > 2048 && rows * div_up(a.vocab, a.slice) < 148) a.slice /= 2;
    a.slices = div_up(a.vocab, a.slice);
    const int smem = (a.slice + kSpare) * (a.entries ? 6 : 4) + a.entries * 8;
    auto* kernel = adjust_kernel<T, N>;
    if (cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 128 * 1024)) return e;
    return launch(kernel, rows * a.slices, kAdjustThreads, smem, stream, a);
}

// ---- an id a row ------------------------------------------------------------------------
// With d = l - max and m = exp(d / T) for each id, in order of falling logits and, among equal ones, of rising ids: the first top_k are kept; of these
// the shortest stretch whose mass is at least top_p of theirs; of these the ones with m >= min_p; the first id at least.  The id is the first one, in the order of
// the ids, at which the running sum of kept masses is more than u times their sum.
//
// A cluster of blocks takes a row and holds it in shared memory, as keys whose order is that of the logits; it is read from memory once.  Masses
// are whole numbers, 2^F for the largest, computed in 64 bits and off by some 2^-40 relative: their sums are exact, do not depend on the order of
// summation, and where the cuts lie is what arithmetic in 64 bits says.  All three cuts are stretches from the top of one order and so is what they
// have in common; a cut is the last id that is kept.  It is searched for by histograms over ever narrower intervals of logits, until an interval holds
// one value or no more ids than can be ranked one by one.
constexpr int kCluster = 8, kDrawThreads = 512, kDrawWarps = kDrawThreads / 32, kBins = 256, kRanked = 256;
constexpr uint32_t kLowest = 0x007FFFFFu;        // key of -infinity
constexpr uint32_t kHighest = 0xFF800000u;       // key of +infinity

struct DrawArgs {
    const void* logits;
    int type;
    int64_t stride;
    int vocab, segment;            // ids; ids of a warp, a multiple of 32
    int fixed;                     // F
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
};

struct Cut {                       // the last of the ids that are kept
    uint32_t key;
    int id;
};

struct DrawShared {
    uint64_t bin_mass[2][kBins];
    uint32_t bin_count[2][kBins];
    uint64_t all_mass[kBins];
    uint32_t all_count[kBins];
    uint64_t said[2][2];           // what this block tells the others
    uint64_t red[kDrawWarps];
    uint64_t warp_sum[kDrawWarps];
    double power[16];
    uint32_t list_key[kRanked];
    int list_id[kRanked];
    uint32_t list_n;
    uint32_t rank_key[kRanked];
    int rank_id[kRanked];
    uint64_t rank_mass[kRanked];
    uint64_t word[4];              // from one thread to the block
    Cut cut;
};

__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.f);               // one zero
    return b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key); }
// To 64 bits by moving bits (conversions go at a fraction of the rate); for finite numbers.
__device__ __forceinline__ double wide(float x) {
    const uint32_t b = __float_as_uint(x);
    if (!(b & 0x7F800000u)) return x;          // 0, and numbers below the normal ones
    return __hiloint2double(static_cast<int>((b & 0x80000000u) | (((b & 0x7FFFFFFFu) >> 3) + 0x38000000u)), static_cast<int>(b << 29));
}

__device__ __forceinline__ uint64_t peer_u64(const uint64_t* p, int block) {
    uint64_t v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(sm100::in_block(sm100::smem_addr(p), block)) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t peer_u32(const void* p, int block) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(sm100::in_block(sm100::smem_addr(p), block)) : "memory");
    return v;
}

__device__ __forceinline__ uint64_t warp_sum(uint64_t v) {
#pragma unroll
    for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(~0u, v, d);
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
    const uint32_t* keys;          // NULL: in memory
    const T* in;
    int first, count, segment;     // first id, ids, ids of a warp
    uint32_t top;                  // key of the largest
    double top_value, steps;       // 16 log2(e) / T
    double least;                  // exponents below this have no mass
    int exchanges;

    __device__ __forceinline__ uint32_t key(int i) const { return keys ? keys[i] : key_of(to_float<T>(in[i])); }

    // 2^(y / 16) = 2^(j / 16) * 2^(r / 16) with j the whole number next to y: the first factor from a table and j's upper bits, the second, r ln(2) / 16 being at most
    // 0.022, from five terms of its series (the sixth is 1.4e-13).
    __device__ __forceinline__ uint64_t mass(uint32_t k) const {
        if (k == top) return static_cast<uint64_t>(__double_as_longlong(s.power[0] + 6755399441055744.0) - 0x4338000000000000ll);
        if (k <= kLowest || top == kHighest) return 0;
        const double y = (wide(value_of(k)) - top_value) * steps;
        if (!(y > least)) return 0;
        constexpr double kWhole = 6755399441055744.0, kUnit = 0.043321698784996581;      // 1.5 * 2^52; ln(2) / 16
        const double shifted = y + kWhole;
        const int j = __double2loint(shifted);
        const double r = (y - (shifted - kWhole)) * kUnit;
        double p = fma(r, 1.0 / 120, 1.0 / 24);
        p = fma(p, r, 1.0 / 6);
        p = fma(p, r, 0.5);
        p = fma(p, r, 1.0);
        p = fma(p, r, 1.0);
        const double t = s.power[j & 15];
        const double scaled = __hiloint2double(__double2hiint(t) + (j >> 4) * (1 << 20), __double2loint(t));
        return static_cast<uint64_t>(__double_as_longlong(fma(scaled, p, kWhole)) - 0x4338000000000000ll);
    }

    // f(key, place) for this thread's share, in which a warp's ids follow one another.
    template <typename F>
    __device__ __forceinline__ void each(F f) const {
        const int from = (threadIdx.x >> 5) * segment, to = from + segment < count ? from + segment : count;
#pragma unroll 4
        for (int i = from + (threadIdx.x & 31); i < to; i += 32) f(key(i), i);
    }

    // Sum (or maximum) over the block, in all threads.
    template <bool MAX>
    __device__ uint64_t over_block(uint64_t v) {
        v = MAX ? warp_max(v) : warp_sum(v);
        __syncthreads();
        if ((threadIdx.x & 31) == 0) s.red[threadIdx.x >> 5] = v;
        __syncthreads();
        v = s.red[threadIdx.x & (kDrawWarps - 1)];
        v = MAX ? warp_max(v) : warp_sum(v);
        return MAX ? v : v / (32 / kDrawWarps);
    }
    // The same over the cluster.  What a block tells lies in one of two places in turn: when one is written again all have been at a barrier since they read it.
    template <bool MAX>
    __device__ uint64_t over_cluster(uint64_t v, uint64_t* before = nullptr) {
        v = over_block<MAX>(v);
        uint64_t* said = s.said[exchanges++ & 1];
        if (threadIdx.x == 0) said[0] = v;
        sm100::cluster_sync();
        const int self = static_cast<int>(sm100::cluster_rank());
        uint64_t all = 0, front = 0;
#pragma unroll
        for (int b = 0; b < kCluster; ++b) {
            const uint64_t o = peer_u64(said, b);
            all = MAX ? larger(all, o) : all + o;
            if (b < self) front += o;
        }
        if (before) *before = front;
        return all;
    }
};

// Bins of an interval of keys [low, high], the highest first.  Even in the logits where it is wide, in the keys where it is not or `by_key` says so.
struct Bins {
    uint32_t low, high;
    bool by_key;
    int shift;
    float top, per;                // half the highest logit, bins for half a unit

    __device__ Bins(uint32_t low_, uint32_t high_, bool keys) : low(low_), high(high_), shift(0), top(0.f), per(0.f) {
        const uint32_t range = high - low;
        by_key = keys || range < (1u << 24) || high >= kHighest;
        if (by_key) {
            while ((range >> shift) >= kBins) ++shift;
        } else {
            top = 0.5f * value_of(high);
            per = fminf(kBins / (top - 0.5f * value_of(low)), 3.0e38f);
        }
    }
    __device__ __forceinline__ int operator()(uint32_t key) const {       // never rises with the key
        if (by_key) return static_cast<int>((high - key) >> shift);
        const float b = (top - 0.5f * value_of(key)) * per;
        return b < kBins - 1 ? static_cast<int>(b) : kBins - 1;
    }
    // The least key of bin b or a higher one.
    __device__ uint32_t least(int b) const {
        uint32_t lo = low, hi = high;                          // hi: in the bin or higher
        while (lo < hi) {
            const uint32_t mid = lo + ((hi - lo) >> 1);
            if ((*this)(mid) <= b) hi = mid; else lo = mid + 1;
        }
        return lo;
    }
};

// The id at which the running weight (ids, or their masses), from the top down to `floor`, reaches `target`; `floor` where it never does.
template <typename T>
__device__ Cut find_cut(Row<T>& row, bool by_mass, uint64_t target, Cut floor, int& buffer) {
    DrawShared& s = row.s;
    const int tid = threadIdx.x;
    const auto among = [&](uint32_t k, int i) { return k > floor.key || (k == floor.key && row.first + i <= floor.id); };
    uint64_t above = 0;
    uint32_t high = row.top, low = floor.key;
    // Where most of the mass and the first hundreds of ids are.
    if (row.top < kHighest && row.top > kLowest) {
        const uint32_t near = key_of(value_of(row.top) - 8.f);
        if (near > low) low = near;
    }
    for (int round = 0;; ++round) {
        const Bins bins(low, high, round >= 6);
        uint64_t* bin_mass = s.bin_mass[buffer];
        uint32_t* bin_count = s.bin_count[buffer];
        for (int b = tid; b < kBins; b += kDrawThreads) {
            bin_mass[b] = 0;
            bin_count[b] = 0;
        }
        __syncthreads();
        row.each([&](uint32_t k, int i) {
            if (k < low || k > high || !among(k, i)) return;
            const int b = bins(k);
            atomicAdd(&bin_count[b], 1u);
            if (by_mass) atomicAdd(reinterpret_cast<unsigned long long*>(&bin_mass[b]), static_cast<unsigned long long>(row.mass(k)));
        });
        sm100::cluster_sync();
        if (tid < kBins) {
            uint32_t c = 0;
            uint64_t m = 0;
            for (int b = 0; b < kCluster; ++b) {
                c += peer_u32(&bin_count[tid], b);
                if (by_mass) m += peer_u64(&bin_mass[tid], b);
            }
            s.all_count[tid] = c;
            s.all_mass[tid] = by_mass ? m : c;
        }
        buffer ^= 1;
        __syncthreads();
        if (tid < 32) {
            // the first bin in which the target is reached: a lane eight bins
            uint64_t mine = 0;
            for (int b = 0; b < kBins / 32; ++b) mine += s.all_mass[tid * (kBins / 32) + b];
            uint64_t run = mine;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const uint64_t o = __shfl_up_sync(~0u, run, d);
                if (tid >= d) run += o;
            }
            const uint64_t all = __shfl_sync(~0u, run, 31);
            const uint32_t reached = __ballot_sync(~0u, above + run >= target);
            if (!reached) {
                if (tid == 0) {
                    s.word[0] = kBins;
                    s.word[1] = above + all;
                }
            } else if (tid == __ffs(reached) - 1) {
                uint64_t at = above + run - mine;
                int b = tid * (kBins / 32);
                while (at + s.all_mass[b] < target) at += s.all_mass[b++];
                s.word[0] = b;
                s.word[1] = at;
            }
        }
        __syncthreads();
        const int bin = static_cast<int>(s.word[0]);
        above = s.word[1];
        const uint32_t in_bin = bin < kBins ? s.all_count[bin] : 0;
        if (bin == kBins) {
            if (low <= floor.key) return floor;
            high = low - 1;
            low = floor.key;
            continue;
        }
        const uint32_t next_low = bins.least(bin);
        if (bin > 0) high = bins.least(bin - 1) - 1;
        low = next_low;
        if (low == high) {
            // Equal logits: of the ids in their order as many as it takes.
            const uint64_t one = by_mass ? row.mass(low) : 1, want = (target - above + one - 1) / one;
            if (want >= in_bin) return low == floor.key ? floor : Cut{low, 0x7FFFFFFF};
            uint64_t mine = 0, before = 0;
            row.each([&](uint32_t k, int i) { mine += k == low && among(k, i); });
            mine = warp_sum(mine);
            __syncthreads();
            if ((tid & 31) == 0) s.warp_sum[tid >> 5] = mine;
            row.template over_cluster<false>((tid & 31) == 0 ? mine : 0, &before);
            // (the one block and warp in which it lies; the others' word stays 0)
            if (tid == 0) s.word[2] = 0;
            __syncthreads();
            for (int w = 0; w < tid >> 5; ++w) before += s.warp_sum[w];
            if (before < want && want <= before + mine) {
                const int from = (tid >> 5) * row.segment, to = min(from + row.segment, row.count);
                for (int j = from; j < to; j += 32) {
                    const int i = j + (tid & 31);
                    const bool one_of = i < to && row.key(i) == low && among(low, i);
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
        if (in_bin > kRanked) continue;
        // Few: each is ranked among all.
        if (tid == 0) s.list_n = 0;                            // (an earlier list has been read: all have been at this round's barrier since)
        __syncthreads();
        row.each([&](uint32_t k, int i) {
            if (k < low || k > high || !among(k, i)) return;
            const uint32_t at = atomicAdd(&s.list_n, 1u);
            s.list_key[at] = k;
            s.list_id[at] = row.first + i;
        });
        sm100::cluster_sync();
        if (tid < kRanked) {
            int at = tid, b = 0;
            for (; b < kCluster; ++b) {
                const int n = static_cast<int>(peer_u32(&s.list_n, b));
                if (at < n) break;
                at -= n;
            }
            if (b < kCluster) {
                s.rank_key[tid] = peer_u32(&s.list_key[at], b);
                s.rank_id[tid] = static_cast<int>(peer_u32(&s.list_id[at], b));
                s.rank_mass[tid] = by_mass ? row.mass(s.rank_key[tid]) : 1;
            }
        }
        __syncthreads();
        if (tid < static_cast<int>(in_bin)) {
            const uint32_t k = s.rank_key[tid];
            const int id = s.rank_id[tid];
            uint64_t before = above;
            for (int o = 0; o < static_cast<int>(in_bin); ++o)
                if (s.rank_key[o] > k || (s.rank_key[o] == k && s.rank_id[o] < id)) before += s.rank_mass[o];
            if (before < target && target <= before + s.rank_mass[tid]) s.cut = Cut{k, id};
        }
        __syncthreads();
        const Cut cut = s.cut;
        __syncthreads();
        return cut;
    }
}

template <typename T>
__global__ void __launch_bounds__(kDrawThreads) draw_kernel(const __grid_constant__ DrawArgs a) {
    extern __shared__ uint4 smem[];
    DrawShared& s = *reinterpret_cast<DrawShared*>(smem);
    uint32_t* held = reinterpret_cast<uint32_t*>(&s + 1);
    const int tid = threadIdx.x;
    after_previous();
    let_next_begin();
    const int64_t r = blockIdx.x / kCluster;
    const int block = static_cast<int>(sm100::cluster_rank());
    const int share = a.segment * kDrawWarps, first = block * share;
    const float heat = a.temperature ? a.temperature[r] : a.one_temperature, share_p = a.top_p ? a.top_p[r] : a.one_top_p, min_p = a.min_p ? a.min_p[r] : a.one_min_p;
    const int top_k = a.top_k ? a.top_k[r] : a.one_top_k;
    const double u = a.wide_u ? static_cast<const double*>(a.u)[r] : static_cast<double>(static_cast<const float*>(a.u)[r]);

    Row<T> row{s, nullptr, static_cast<const T*>(a.logits) + r * a.stride + first, first, max(0, min(share, a.vocab - first)), a.segment, 0, 0.0, 0.0, 0.0, 0};
    // the largest logit, and whether there is a NaN
    uint64_t most = 0;
    {
        const int from = (tid >> 5) * a.segment, to = min(from + a.segment, row.count);
#pragma unroll 8
        for (int i = from + (tid & 31); i < to; i += 32) {
            const float x = to_float<T>(row.in[i]);
            const uint32_t k = key_of(x);
            if (a.held) held[i] = k;
            most = larger(most, x == x ? k : uint64_t{1} << 32);
        }
    }
    if (a.held) row.keys = held;
    if (tid < 16) s.power[tid] = exp2(a.fixed + tid / 16.0);
    most = row.template over_cluster<true>(most);
    row.top = static_cast<uint32_t>(most);
    const bool bad = most >> 32 || !(heat >= 0.f && heat <= 3.402823466e38f) || !(u >= 0.0 && u < 1.0) || share_p != share_p || min_p != min_p;
    if (bad || row.top <= kLowest) {
        if (block == 0 && tid == 0) {
            a.ids[r] = -1;
            a.logprobs[r] = bad ? __int_as_float(0x7FC00000) : -INFINITY;
        }
        return sm100::cluster_sync();
    }
    if (heat == 0.f) {
        uint64_t at = 0;                                       // the first: what is left behind it, at most
        row.each([&](uint32_t k, int i) {
            if (k == row.top) at = larger(at, a.vocab - row.first - i);
        });
        at = row.template over_cluster<true>(at);
        if (block == 0 && tid == 0) {
            a.ids[r] = a.vocab - static_cast<int>(at);
            a.logprobs[r] = 0.f;
        }
        return sm100::cluster_sync();
    }
    row.top_value = wide(value_of(row.top));
    row.steps = 23.083120654223414 / static_cast<double>(heat);                // 16 log2(e) / T
    row.least = -16.0 * (a.fixed + 1);

    uint64_t mine = 0;
    row.each([&](uint32_t k, int) { mine += row.mass(k); });
    const uint64_t total = row.template over_cluster<false>(mine);

    // The cuts.
    Cut cut{kLowest + 1, 0x7FFFFFFF};
    int buffer = 0;
    uint64_t kept = total;
    const bool one = top_k == 1 || min_p > 1.f || share_p <= 0.f;
    if (one || (top_k > 0 && top_k < a.vocab)) {
        cut = find_cut(row, false, one ? 1 : top_k, cut, buffer);
        if (!one && share_p < 1.f) {
            mine = 0;
            row.each([&](uint32_t k, int i) {
                if (k > cut.key || (k == cut.key && row.first + i <= cut.id)) mine += row.mass(k);
            });
            kept = row.template over_cluster<false>(mine);
        }
    }
    if (!one && share_p < 1.f) {
        const uint64_t want = static_cast<uint64_t>(ceil(static_cast<double>(share_p) * static_cast<double>(kept)));
        cut = find_cut(row, true, larger(1, want < kept ? want : kept), cut, buffer);
    }
    if (!one && min_p > 0.f && row.top < kHighest) {
        // the least key with d / T >= log(min_p)
        const double depth = log(static_cast<double>(min_p)) * static_cast<double>(heat);
        uint32_t lo = kLowest + 1, hi = row.top;
        while (lo < hi) {
            const uint32_t mid = lo + ((hi - lo) >> 1);
            if (wide(value_of(mid)) - row.top_value >= depth) hi = mid; else lo = mid + 1;
        }
        if (lo > cut.key) cut = Cut{lo, 0x7FFFFFFF};
    }

    // The draw: the block, the warp and the place at which the running sum passes u times the whole.
    const auto weight = [&](uint32_t k, int i) -> uint64_t { return k > cut.key || (k == cut.key && row.first + i <= cut.id) ? row.mass(k) : 0; };
    mine = 0;
    row.each([&](uint32_t k, int i) { mine += weight(k, i); });
    mine = warp_sum(mine);
    __syncthreads();
    if ((tid & 31) == 0) s.warp_sum[tid >> 5] = mine;
    uint64_t before = 0;
    kept = row.template over_cluster<false>((tid & 31) == 0 ? mine : 0, &before);
    uint64_t at = static_cast<uint64_t>(u * static_cast<double>(kept));
    if (at >= kept) at = kept - 1;
    for (int w = 0; w < tid >> 5; ++w) before += s.warp_sum[w];
    if (before <= at && at < before + mine) {
        const int from = (tid >> 5) * a.segment, to = min(from + a.segment, row.count), lane = tid & 31;
        for (int j = from; j < to; j += 32) {
            const uint32_t k = j + lane < to ? row.key(j + lane) : 0;
            const uint64_t m = j + lane < to ? weight(k, j + lane) : 0;
            uint64_t run = m;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const uint64_t o = __shfl_up_sync(~0u, run, d);
                if (lane >= d) run += o;
            }
            const uint32_t passed = __ballot_sync(~0u, before + run > at);
            if (passed) {
                if (lane == __ffs(passed) - 1) {
                    a.ids[r] = row.first + j + lane;
                    const double down = row.top == kHighest ? 0.0 : (wide(value_of(k)) - row.top_value) / static_cast<double>(heat);
                    a.logprobs[r] = static_cast<float>(down - log(static_cast<double>(total)) + a.fixed * 0.69314718055994531);
                }
                break;
            }
            before += __shfl_sync(~0u, run, 31);
        }
    }
    sm100::cluster_sync();                                     // (no block leaves while another may read from it)
}

template <typename T>
cudaError_t draw(const DrawArgs& a, int64_t rows, cudaStream_t stream) {
    const int smem = static_cast<int>(sizeof(DrawShared)) + (a.held ? a.segment * kDrawWarps * 4 : 0);
    auto* kernel = draw_kernel<T>;
    if (cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024)) return e;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(static_cast<unsigned>(rows * kCluster));
    config.blockDim = dim3(kDrawThreads);
    config.dynamicSmemBytes = smem;
    config.stream = stream;
    cudaLaunchAttribute attrs[2]{};
    attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[0].val.programmaticStreamSerializationAllowed = 1;
    attrs[1].id = cudaLaunchAttributeClusterDimension;
    attrs[1].val.clusterDim.x = kCluster;
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
    a.vocab = c.logits.cols;
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
    a.type = c.logits.type;
    a.stride = c.logits.stride;
    a.vocab = static_cast<int>(c.logits.cols);
    a.segment = static_cast<int>(round_up(div_up(a.vocab, kCluster * kDrawWarps), 32));
    int bits = 0;
    while ((1ll << bits) < a.vocab) ++bits;
    a.fixed = std::min(50, 62 - bits);                         // (sums of a row's masses have 62 bits)
    a.held = sizeof(DrawShared) + a.segment * kDrawWarps * 4ll <= 227 * 1024;
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
