// A table in 4 bits: laid out for the products, made from weights, and multiplied with hidden states.
//
// z[i, v] = sum over groups g of s[v, g] * sum over k in g of (q[v, k] - b[v, g]) * h[i, k], with codes q of 0 to 15, a scale s and a zero b
// (8 where there are none) for each group of a row.  q - b is a whole number of at most 15 and exact in bf16 and fp16, so the inner sums are
// matrix products of what is stored, in fp32, and only they are scaled: no weight is rounded on the way.
#include "sm100.cuh"
#include "vocab_launch.cuh"
#include "vocab_maps.h"
#include "vocab_next.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

namespace gtok {
namespace {

__host__ __device__ constexpr int64_t div_up(int64_t a, int64_t b) { return (a + b - 1) / b; }

template <typename T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

// ---- layout -----------------------------------------------------------------------
// Lane l of a unit holds rows l / 4 and l / 4 + 8 and, of each 16 columns, 2 (l % 4) + {0, 1, 8, 9}.  Nibbles 0 to 3 of a word are the first
// codes of the lane's four operand pairs (upper row, lower row, then the same eight columns on), nibbles 4 to 7 the second ones.
__device__ __forceinline__ int nibble_row(int lane, int i) { return lane / 4 + (i & 1) * 8; }
__device__ __forceinline__ int nibble_col(int lane, int i) { return 2 * (lane % 4) + ((i >> 1) & 1) * 8 + (i >> 2); }

// What lies between the parts and behind the last is 0: equal tables are equal byte by byte.
__device__ __forceinline__ void clear_gaps(char* at, const Table4Plan& p, bool zeros) {
    if (blockIdx.x) return;
    const uint64_t scales_end = p.scales + static_cast<uint64_t>(p.tiles) * p.groups * 64, zeros_end = p.zeros + (zeros ? static_cast<uint64_t>(p.tiles) * p.groups * 32 : 0);
    for (uint64_t i = scales_end + threadIdx.x; i < p.zeros; i += blockDim.x) at[i] = 0;
    for (uint64_t i = zeros_end + threadIdx.x; i < p.bytes; i += blockDim.x) at[i] = 0;
}

struct PackArgs {
    Table4 t;
    Table4Plan p;
    const uint8_t* codes;
    int64_t codes_stride;
    const void* scales;
    int64_t scales_stride;
    const uint8_t* zeros;
    int64_t zeros_stride;
};

// A warp a pair of units, done once for a table: every byte read and written once, but codes byte by byte.
__global__ void __launch_bounds__(256) pack_kernel(const __grid_constant__ PackArgs a) {
    after_previous();
    const int lane = threadIdx.x & 31;
    const int64_t warps = static_cast<int64_t>(gridDim.x) * 8, warp = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
    char* at = static_cast<char*>(a.t.data);
    clear_gaps(at, a.p, a.t.zeros);
    for (int64_t unit = warp; unit < a.p.tiles * a.p.units; unit += warps) {
        const int64_t tile = unit / a.p.units, u = unit - tile * a.p.units;
        for (int half = 0; half < 2; ++half) {
            uint32_t w[4];
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                w[s] = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int64_t row = tile * 32 + half * 16 + nibble_row(lane, i), col = u * 64 + s * 16 + nibble_col(lane, i);
                    const uint32_t q = row < a.t.vocab && col < a.t.width ? a.codes[row * a.codes_stride + col] & 15 : 0;
                    w[s] |= q << (4 * i);
                }
            }
            reinterpret_cast<uint4*>(at)[(unit * 2 + half) * 32 + lane] = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
    const int64_t given = div_up(a.t.width, a.t.group);
    for (int64_t i = warp; i < a.p.tiles * a.p.groups; i += warps) {
        const int64_t tile = i / a.p.groups, g = i - tile * a.p.groups, row = tile * 32 + (lane & 3) * 8 + lane / 4;
        const bool here = row < a.t.vocab && g < given;
        reinterpret_cast<uint16_t*>(at + a.p.scales)[i * 32 + lane] = here ? static_cast<const uint16_t*>(a.scales)[row * a.scales_stride + g] : 0;
        if (a.t.zeros) reinterpret_cast<uint8_t*>(at + a.p.zeros)[i * 32 + lane] = here ? a.zeros[row * a.zeros_stride + g] & 15 : 0;
    }
}

// ---- from weights -------------------------------------------------------------------
// Without zeros: s = max |w| / 7, q = round(w / s) + 8 from 0 to 15.  With zeros: s = (max(w, 0) - min(w, 0)) / 15, b = round(-min(w, 0) / s),
// q = round(w / s) + b.  Ties to even.  s is rounded to the table's 16 bits first and the codes are of what was rounded; a group of zeros, or
// one whose scale rounds to 0, has scale 0.  A group with a NaN or an infinity, or whose scale is beyond the largest of the table's type (in fp16 that of weights from 7 or 15 times 65,520 on), gets
// the scale NaN.
struct QuantizeArgs {
    Table4 t;
    Table4Plan p;
    const void* weight;
    int64_t stride;
};

// A block a tile of 32 rows and a stretch of columns: its groups' scales first, in shared memory, then its codes, whose weights come from the
// caches.  Done once for a table.
constexpr int kQuantUnits = 8;             // units of a stretch; no more groups than 16 begin in one
template <typename W, typename T>
__global__ void __launch_bounds__(256) quantize_kernel(const __grid_constant__ QuantizeArgs a, int64_t stretch) {
    __shared__ float scale[32][2 * kQuantUnits];
    __shared__ int zero[32][2 * kQuantUnits];
    after_previous();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const W* weight = static_cast<const W*>(a.weight);
    char* at = static_cast<char*>(a.t.data);
    clear_gaps(at, a.p, a.t.zeros);
    const int64_t stretches = div_up(a.p.units, stretch), tile = blockIdx.x / stretches, u0 = (blockIdx.x - tile * stretches) * stretch;
    const int64_t u1 = u0 + stretch < a.p.units ? u0 + stretch : a.p.units;
    const int64_t g0 = u0 * 64 / a.t.group, g1 = a.t.group == 32 ? u1 * 2 : div_up(u1 * 64 < a.t.width ? u1 * 64 : a.t.width, a.t.group);
    for (int64_t i = warp; i < 32 * (g1 - g0); i += 8) {
        const int r = static_cast<int>(i & 31);
        const int64_t g = g0 + (i >> 5), row = tile * 32 + r;
        const int64_t from = g * a.t.group, to = from + a.t.group < a.t.width ? from + a.t.group : a.t.width;
        float low = 0.f, high = 0.f, bad = 0.f;
        if (row < a.t.vocab)
            for (int64_t c = from + lane; c < to; c += 32) {
                const float v = to_float<W>(weight[row * a.stride + c]);
                low = fminf(low, v);
                high = fmaxf(high, v);
                bad += v - v;                  // 0, or NaN for a NaN or an infinity
            }
#pragma unroll
        for (int d = 16; d; d >>= 1) {
            low = fminf(low, __shfl_xor_sync(~0u, low, d));
            high = fmaxf(high, __shfl_xor_sync(~0u, high, d));
            bad += __shfl_xor_sync(~0u, bad, d);
        }
        if (lane == 0) {
            // (in two parts, as the difference of two large numbers may be none)
            float s = to_float<T>(from_float<T>((a.t.zeros ? high / 15.f - low / 15.f : fmaxf(high, -low) / 7.f) + bad));
            s += s - s;                        // (0, or NaN for an infinite one)
            const int b = a.t.zeros ? (s > 0.f ? static_cast<int>(fminf(fmaxf(rintf(-low / s), 0.f), 15.f)) : 0) : 8;
            scale[r][g - g0] = s;
            zero[r][g - g0] = b;
            const int64_t to_meta = (tile * a.p.groups + g) * 32 + (r & 7) * 4 + r / 8;
            reinterpret_cast<T*>(at + a.p.scales)[to_meta] = from_float<T>(s);
            if (a.t.zeros) reinterpret_cast<uint8_t*>(at + a.p.zeros)[to_meta] = static_cast<uint8_t>(b);
        }
    }
    __syncthreads();
    for (int64_t i = warp; i < 2 * (u1 - u0); i += 8) {
        const int half = static_cast<int>(i & 1);
        const int64_t u = u0 + (i >> 1);
        uint32_t w[4];
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            w[s] = 0;
            for (int n = 0; n < 8; ++n) {
                const int r = half * 16 + nibble_row(lane, n);
                const int64_t row = tile * 32 + r, col = u * 64 + s * 16 + nibble_col(lane, n), g = col / a.t.group - g0;
                uint32_t q = 0;
                if (row < a.t.vocab && col < a.t.width && scale[r][g] > 0.f)
                    q = static_cast<uint32_t>(fminf(fmaxf(rintf(to_float<W>(weight[row * a.stride + col]) / scale[r][g]) + zero[r][g], 0.f), 15.f));
                w[s] |= q << (4 * n);
            }
        }
        reinterpret_cast<uint4*>(at)[((tile * a.p.units + u) * 2 + half) * 32 + lane] = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// ---- products -------------------------------------------------------------------------
constexpr int kWarps = 16, kThreads = kWarps * 32, kAhead = 2;
constexpr int kPartLine = 68;              // floats from a row of hidden states to the next among partial sums: lanes of a fragment meet no bank twice

struct LogitsArgs {
    const uint4* codes;
    const uint16_t* scales;
    const uint8_t* zeros;
    const uint16_t* hidden;
    int64_t hidden_stride;
    void* out;
    int64_t out_stride, vocab, width;
    int tiles, groups;             // (no more than 2^19 tiles of 2^10 units or 2^11 groups)
    int units;                     // of 64 columns
    uint32_t per_group;            // 2^20 / how many of them share a group, rounded up; 0: each has two groups
    int rows;                      // of hidden states, at most 8 NT
    int split, split_log;          // warps that share a tile
    bool staged;                   // hidden states fit into shared memory
    bool pairs;                    // two of them lie on 4 bytes
    int buffers;                   // of partial sums
};

template <bool BF16> struct Half16;
template <> struct Half16<true> {
    using type = __nv_bfloat16;
    static constexpr uint32_t kBase = 0x43004300u;             // 128 + code, twice
    static __device__ __forceinline__ float lower_half(uint32_t w) { return __uint_as_float(w << 16); }
    static __device__ __forceinline__ float upper_half(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }
    // What is taken from the codes of the upper and of the lower row, twice.
    static __device__ __forceinline__ uint32_t upper_zero(uint32_t zero) { return kBase + (zero << 16 | zero); }
    static __device__ __forceinline__ uint32_t lower_zero(uint32_t zero) { return upper_zero(zero); }
    // The lane's four operand pairs of a word.  A code becomes the lowest bits of 128's mantissa, which has no room for one that lies higher.
    static __device__ __forceinline__ void operands(uint32_t w, uint32_t upper, uint32_t lower, uint32_t* q) {
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            const uint32_t a = (w >> (4 * p) & 0x000F000Fu) | kBase, &b = p & 1 ? lower : upper;
            const __nv_bfloat162 r = __hsub2(reinterpret_cast<const __nv_bfloat162&>(a), reinterpret_cast<const __nv_bfloat162&>(b));
            q[p] = reinterpret_cast<const uint32_t&>(r);
        }
    }
    static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint2 b) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b.x), "r"(b.y));
    }
};
template <> struct Half16<false> {
    using type = __half;
    static constexpr uint32_t kBase = 0x64006400u;             // 1024 + code, twice
    static __device__ __forceinline__ float lower_half(uint32_t w) { return __low2float(reinterpret_cast<const __half2&>(w)); }
    static __device__ __forceinline__ float upper_half(uint32_t w) { return __high2float(reinterpret_cast<const __half2&>(w)); }
    static __device__ __forceinline__ uint32_t upper_zero(uint32_t zero) { return kBase + (zero << 16 | zero); }
    static __device__ __forceinline__ uint32_t lower_zero(uint32_t zero) { return 0xD400D400u + (zero << 20 | zero << 4); }         // -(64 + zero), twice
    // 1024's mantissa has room for a code four bits up, too: 1024 + 16 q, of which a 16th less 64 + zero is exact.  One shift in place of three.
    static __device__ __forceinline__ void operands(uint32_t w, uint32_t upper, uint32_t lower, uint32_t* q) {
        const uint32_t sixteenth = 0x2C002C00u;
#pragma unroll
        for (int p = 0; p < 4; p += 2) {
            const uint32_t v = w >> (4 * p), a = (v & 0x000F000Fu) | kBase, b = (v & 0x00F000F0u) | kBase;
            const __half2 r = __hsub2(reinterpret_cast<const __half2&>(a), reinterpret_cast<const __half2&>(upper));
            const __half2 t = __hfma2(reinterpret_cast<const __half2&>(b), reinterpret_cast<const __half2&>(sixteenth), reinterpret_cast<const __half2&>(lower));
            q[p] = reinterpret_cast<const uint32_t&>(r);
            q[p + 1] = reinterpret_cast<const uint32_t&>(t);
        }
    }
    static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint2 b) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b.x), "r"(b.y));
    }
};

// Operand pair of hidden states: row `n`, columns col and col + 1, 0 outside.
__device__ __forceinline__ uint32_t hidden_pair(const LogitsArgs& a, int n, int64_t col) {
    if (n >= a.rows) return 0;
    const uint16_t* row = a.hidden + n * a.hidden_stride;
    if (a.pairs) return col < a.width ? *reinterpret_cast<const uint32_t*>(row + col) : 0;
    const uint32_t low = col < a.width ? row[col] : 0, high = col + 1 < a.width ? row[col + 1] : 0;
    return high << 16 | low;
}

// What a lane has under way: 64 rows x 64 columns, two tiles' units.
constexpr int kHalves = 4;                 // of 16 rows
template <int SUBS, bool ZEROS>
struct Lot {
    uint4 code[kHalves];
    uint2 scale[2][SUBS];          // of a tile's four rows that are the lane's, 16 bits each
    uint32_t zero[2][ZEROS ? SUBS : 1];
};

__device__ __forceinline__ uint4 load_once(const uint4* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

// Up to 8 NT rows of hidden states.  Warps take 64 rows of the table and every `split`th unit of the width; those that share rows add up through
// shared memory when they are done with them.  Codes come from memory straight into the lanes that multiply with them, kAhead steps before they are
// needed, across the ends of rows; hidden states lie in shared memory in the order of operands.  With 32 x 64 codes an SM's quarter has to do: 56 shifts and and-ors (40 in fp16), which go at a warp
// in two clocks, 32 subtractions in the unit beside it, NT times 8 products of 16 x 8 x 16 of 8 clocks each, and waits 186 clocks for its share of memory.
// It takes 310 with one row of 128,256 x 4096 in groups of 128: 73 us, 3.7 TB/s (42 at the rate of a copy); 50,256 x 768 in fp16 10.5 us.  Four warps a quarter are too few to hide the chain from
// shift to product, and registers do not allow more (with 9 to 16 rows up to 112 bytes of a thread's are spilled as it is).  Lots of 32 rows took 88 us (addresses, scales and waits for half as much), an integer division a lot 13 more.
template <bool BF16, int NT, int SUBS, bool ZEROS, typename Out>
__global__ void __launch_bounds__(kThreads, 1) few_rows_kernel(const __grid_constant__ LogitsArgs a) {
    using H = Half16<BF16>;
    extern __shared__ uint4 smem[];
    constexpr int kPart = 8 * NT * kPartLine;                  // floats of a warp's partial sums
    float* parts = reinterpret_cast<float*>(smem);             // [buffers][kWarps][kPart]
    uint2* staged = reinterpret_cast<uint2*>(parts + a.buffers * kWarps * kPart);      // [units * 4][NT][32]
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    after_previous();
    let_next_begin();
    // of pairs of tiles
    const int pairs = (a.tiles + 1) / 2, first = static_cast<int>(static_cast<int64_t>(pairs) * blockIdx.x / gridDim.x),
              last = static_cast<int>(static_cast<int64_t>(pairs) * (blockIdx.x + 1) / gridDim.x);
    const int at_once = kWarps >> a.split_log, part = warp & (a.split - 1), slot = warp >> a.split_log;
    const int rounds = (last - first + at_once - 1) >> (4 - a.split_log);
    const int count = (a.units - part + a.split - 1) >> a.split_log;           // units of a row that are this warp's; one at least

    Lot<SUBS, ZEROS> lot[kAhead];
    int fetch_round = 0, fetch_u = part;
    const uint4* fetch_at[2];
    int fetch_tile[2];
    const auto start = [&] {
        const int pair = min(first + fetch_round * at_once + slot, last - 1);  // (behind the last: its sums are left out)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            fetch_tile[t] = min(2 * pair + t, a.tiles - 1);
            fetch_at[t] = a.codes + static_cast<int64_t>(fetch_tile[t] * a.units + part) * 64 + lane;
        }
    };
    const auto fetch = [&](Lot<SUBS, ZEROS>& l) {
        if (fetch_round >= rounds) return;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            l.code[2 * t] = load_once(fetch_at[t]);
            l.code[2 * t + 1] = load_once(fetch_at[t] + 32);
            fetch_at[t] += a.split * 64;
#pragma unroll
            for (int s = 0; s < SUBS; ++s) {
                const uint32_t g = fetch_tile[t] * a.groups + (SUBS == 2 ? fetch_u * 2 + s : fetch_u * a.per_group >> 20);
                l.scale[t][s] = __ldg(reinterpret_cast<const uint2*>(a.scales) + static_cast<uint64_t>(g) * 8 + lane / 4);
                if constexpr (ZEROS) l.zero[t][s] = __ldg(reinterpret_cast<const uint32_t*>(a.zeros) + static_cast<uint64_t>(g) * 8 + lane / 4);
            }
        }
        fetch_u += a.split;
        if (fetch_u >= a.units) {
            fetch_u = part;
            ++fetch_round;
            start();
        }
    };
    start();
#pragma unroll
    for (int s = 0; s < kAhead; ++s) fetch(lot[s]);
    if (a.staged) {
        constexpr int kAtOnce = 8;             // under way a thread
        const int all = a.units * 4 * NT * 32;
        for (int from = tid; from < all; from += kThreads * kAtOnce) {
            uint2 v[kAtOnce];
#pragma unroll
            for (int q = 0; q < kAtOnce; ++q) {
                const int i = from + q * kThreads, l = i & 31, nt = (i >> 5) % NT, step = (i >> 5) / NT;
                const int64_t col = step * 16 + 2 * (l & 3);
                if (i < all) v[q] = make_uint2(hidden_pair(a, nt * 8 + l / 4, col), hidden_pair(a, nt * 8 + l / 4, col + 8));
            }
#pragma unroll
            for (int q = 0; q < kAtOnce; ++q)
                if (from + q * kThreads < all) staged[from + q * kThreads] = v[q];
        }
        __syncthreads();
    }

    float acc[kHalves][NT][4] = {};
    int i = 0, buffer = 0, round = 0;
    while (round < rounds) {
#pragma unroll
        for (int s = 0; s < kAhead; ++s) {
            if (round >= rounds) break;
            const Lot<SUBS, ZEROS>& l = lot[s];
            const int u = part + (i << a.split_log);
            constexpr int kSteps = 4 / SUBS;                   // of 16 columns in a group's part
#pragma unroll
            for (int sub = 0; sub < SUBS; ++sub) {
                uint2 b[kSteps][NT];
#pragma unroll
                for (int k = 0; k < kSteps; ++k)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        const int step = u * 4 + sub * kSteps + k;
                        if (a.staged) b[k][nt] = staged[(step * NT + nt) * 32 + lane];
                        else {
                            const int64_t col = step * 16 + 2 * (lane & 3);
                            b[k][nt] = make_uint2(hidden_pair(a, nt * 8 + lane / 4, col), hidden_pair(a, nt * 8 + lane / 4, col + 8));
                        }
                    }
#pragma unroll
                for (int half = 0; half < kHalves; ++half) {
                    float sum[NT][4] = {};
                    const uint32_t zeros = ZEROS ? l.zero[half / 2][ZEROS ? sub : 0] >> (16 * (half & 1)) : 0x0808u, upper_zero = H::upper_zero(zeros & 15),
                                   lower_zero = H::lower_zero(zeros >> 8 & 15);
#pragma unroll
                    for (int k = 0; k < kSteps; ++k) {
                        const int word = sub * kSteps + k;
                        const uint32_t w = word == 0 ? l.code[half].x : word == 1 ? l.code[half].y : word == 2 ? l.code[half].z : l.code[half].w;
                        uint32_t q[4];
                        H::operands(w, upper_zero, lower_zero, q);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) H::mma(sum[nt], q, b[k][nt]);
                    }
                    const uint32_t w = half & 1 ? l.scale[half / 2][sub].y : l.scale[half / 2][sub].x;
                    const float upper = H::lower_half(w), lower = H::upper_half(w);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        acc[half][nt][0] = fmaf(upper, sum[nt][0], acc[half][nt][0]);
                        acc[half][nt][1] = fmaf(upper, sum[nt][1], acc[half][nt][1]);
                        acc[half][nt][2] = fmaf(lower, sum[nt][2], acc[half][nt][2]);
                        acc[half][nt][3] = fmaf(lower, sum[nt][3], acc[half][nt][3]);
                    }
                }
            }
            fetch(lot[s]);
            if (++i < count) continue;
            // The rows of a round are done: partial sums of the warps that share some are added in their order.
            i = 0;
            float* mine = parts + (buffer * kWarps + warp) * kPart;
#pragma unroll
            for (int half = 0; half < kHalves; ++half)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        mine[(nt * 8 + 2 * (lane & 3) + (e & 1)) * kPartLine + half * 16 + lane / 4 + (e >> 1) * 8] = acc[half][nt][e];
                        acc[half][nt][e] = 0.f;
                    }
            asm volatile("bar.sync 1, %0;" ::"n"(kThreads) : "memory");        // (warps come here from different places of the unrolled loop)
            for (int o = tid; o < at_once * a.rows * 64; o += kThreads) {
                const int r = o & 63, n = (o >> 6) % a.rows, t = (o >> 6) / a.rows;
                const int pair = first + round * at_once + t;
                const int64_t v = static_cast<int64_t>(pair) * 64 + r;
                if (pair >= last || v >= a.vocab) continue;
                const float* from = parts + (buffer * kWarps + (t << a.split_log)) * kPart + n * kPartLine + r;
                float total = from[0];
                for (int p = 1; p < a.split; ++p) total += from[p * kPart];
                static_cast<Out*>(a.out)[n * a.out_stride + v] = from_float<Out>(total);
            }
            if (a.buffers > 1) buffer ^= 1;
            else asm volatile("bar.sync 1, %0;" ::"n"(kThreads) : "memory");
            ++round;
        }
    }
}

int few_smem(int nt, int units, bool staged, int buffers) { return buffers * kWarps * 8 * nt * kPartLine * 4 + (staged ? units * 4 * nt * 32 * 8 : 0); }
constexpr int kMostSmem = 227 * 1024;
// More rows than 8, and in groups of less than 128 columns than these, go to the other kernel.  (In groups of 128: 128,256 x 4096, 16 rows 113 us here and 111 there; 50,256 x 768 17.8 and
// 12.3.  Of 64: 151,665 x 2560 in fp16, 13 rows 91 and 122.  Of 32, 17 rows in two passes here and there: 50,256 x 768 30 and 21, x 2048
// 54 and 48, 5,000 x 4096 37 and 31, but 128,256 x 4096 205 and 330: for 17 to 32 rows of the largest tables the rule takes the slower one.)
constexpr int kFewRows = 16;

template <bool BF16, int NT, int SUBS, bool ZEROS, typename Out>
cudaError_t few_rows(const LogitsArgs& a, int blocks, cudaStream_t stream) {
    auto* kernel = few_rows_kernel<BF16, NT, SUBS, ZEROS, Out>;
    const int smem = few_smem(NT, a.units, a.staged, a.buffers);
    if (cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostSmem)) return e;
    return launch(kernel, blocks, kThreads, smem, stream, a);
}
template <bool BF16, int NT, typename Out>
cudaError_t few_rows(const LogitsArgs& a, int blocks, cudaStream_t stream) {
    if (a.per_group == 0) return a.zeros ? few_rows<BF16, NT, 2, true, Out>(a, blocks, stream) : few_rows<BF16, NT, 2, false, Out>(a, blocks, stream);
    return a.zeros ? few_rows<BF16, NT, 1, true, Out>(a, blocks, stream) : few_rows<BF16, NT, 1, false, Out>(a, blocks, stream);
}
template <bool BF16, typename Out>
cudaError_t few_rows(const LogitsArgs& a, int nt, int blocks, cudaStream_t stream) {
    return nt == 1 ? few_rows<BF16, 1, Out>(a, blocks, stream) : few_rows<BF16, 2, Out>(a, blocks, stream);
}

// ---- products with more rows --------------------------------------------------------------
// As for few rows, with the matrix instruction that takes 256 of the table's rows at a time, two blocks of a cluster half of them each, and all hidden states as columns.
// A stage is 128 rows x 128 columns of a block.  One warp copies codes to shared memory, one hidden states (each block half of the rows, by tiled copies).  Eight warps, or four, make
// 16-bit operands of codes, in registers, and put them into tensor memory, from where the instruction takes them.  A group's product is taken out of tensor memory by eight
// more warps and added, with its scale, to sums in registers, while the next group's goes to the other half of the accumulators.
//
// Groups of 128 and 47 rows of 128,256 x 4096: 126 us (46 at the rate of a copy), 128 rows 139: what the threads hand one another costs some 550 clocks for 64 columns, whatever the rows.  Groups of 32 and
// 125 rows of 151,665 x 2048: 212 us; 17 of 128,256 x 4096: 330.  That is 0.36 us for a group of a tile whatever the rows, so neither taking out nor adding bounds it; what is left is the way from a
// product to the next one that may use its accumulator, of which there are two.  593 tiles are eight for each pair of blocks and a ninth for one.  What it took: products issued by one thread in a straight line (as a loop of
// branches, by that thread or by a whole warp that elects one for each, a stage took two to four times as long); no copy of a loaded register that waits for the load; stages of 128 columns
// (of 64: 150 us, and 307 in groups of 32).  The warps' own products of 16 x 8 x 16 for up to 64 rows, hidden states streamed through shared memory, took 381 us for 47 rows.
constexpr int kManyStages = 4, kTakers = 8, kCodeStages = 10, kAheadMeta = 8;
// Warps that make operands.  In groups of 32 columns they are not what is waited for, and more of them are in the way: 125 rows of 151,665 x 2048 236 us with eight,
// 212 with four (fewer rows were not timed); in groups of 128, 47 rows of 128,256 x 4096, 128 and 171.
__host__ __device__ constexpr int makers(bool two) { return two ? 4 : 8; }
__host__ __device__ constexpr int many_threads(bool two) { return 32 * (makers(two) + kTakers + 3); }
constexpr int kMostColumns = 128;          // of hidden states
constexpr int kManySmem = 1024 + kManyStages * (kMostColumns / 2) * 256 + kCodeStages * 8192 + 1024;

struct ManyArgs {
    const uint4* codes;
    const uint16_t* scales;
    const uint32_t* zeros;         // of eight times four rows; NULL: 8 everywhere
    void* out;
    int64_t out_stride, vocab;
    int tiles, groups;             // of 32 rows; of a row
    int units, group_units;        // of 64 columns; how many share a group (0: each has two)
    uint32_t per_group;
    int rows;
    bool wide;                     // logits are fp32
};

__device__ __forceinline__ void bar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void load_line(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ uint4 shared_uint4(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ void prefetch(const void* p) { asm volatile("prefetch.global.L1 [%0];" ::"l"(p)); }
// 16 lanes x 32 columns: register 2 i + r of lane l goes to lane l / 4 + 8 r, column 4 i + l % 4.
__device__ __forceinline__ void tmem_store(uint32_t at, const uint32_t (&v)[16]) {
    asm volatile("tcgen05.st.sync.aligned.16x128b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(at), "r"(v[0]), "r"(v[1]), "r"(v[2]),
                 "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
                 : "memory");
}
__device__ __forceinline__ void tmem_stored() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
template <int NC>
__device__ __forceinline__ void tmem_take(uint32_t at, float (&v)[NC]) {       // on their way
#pragma unroll
    for (int c = 0; c < NC; c += 8)
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                     : "=f"(v[c]), "=f"(v[c + 1]), "=f"(v[c + 2]), "=f"(v[c + 3]), "=f"(v[c + 4]), "=f"(v[c + 5]), "=f"(v[c + 6]), "=f"(v[c + 7])
                     : "r"(at + c));
}
template <int NC>
__device__ __forceinline__ void tmem_taken(float (&v)[NC]) {                   // there
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int c = 0; c < NC; c += 8)
        asm volatile("" : "+f"(v[c]), "+f"(v[c + 1]), "+f"(v[c + 2]), "+f"(v[c + 3]), "+f"(v[c + 4]), "+f"(v[c + 5]), "+f"(v[c + 6]), "+f"(v[c + 7]));
}
// s += scale * v, two at a time
__device__ __forceinline__ void add_scaled(float& s0, float& s1, float scale, float v0, float v1) {
    asm("{\n.reg .b64 s, f, v;\nmov.b64 s, {%0, %1};\nmov.b64 f, {%2, %2};\nmov.b64 v, {%3, %4};\nfma.rn.f32x2 s, f, v, s;\nmov.b64 {%0, %1}, s;\n}"
        : "+f"(s0), "+f"(s1)
        : "f"(scale), "f"(v0), "f"(v1));
}
// The left operand lies in tensor memory: a lane a row, two elements to a column.
__device__ __forceinline__ void mma_from_tmem(uint32_t acc, uint32_t a, uint64_t b, uint32_t kind, bool add) {
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(acc), "r"(a), "l"(b), "r"(kind),
                 "r"(static_cast<uint32_t>(add))
                 : "memory");
}

// NC: columns of a taking warp, half of all.  TWO: a unit has two groups, else a group has one or more units.
template <bool BF16, int NC, bool TWO>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(many_threads(TWO), 1) many_rows_kernel(const __grid_constant__ CUtensorMap map_hidden, const __grid_constant__ ManyArgs a) {
    using namespace sm100;
    using H = Half16<BF16>;
    constexpr int kMakers = makers(TWO), kTurns = kMakers / 4, kStageBytes = NC * 256, kAcc = kManyStages * 64;             // accumulators lie behind the stages
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_addr(smem_raw) + 1023) & ~1023u;
    const uint32_t codes = base + kManyStages * kStageBytes, full = codes + kCodeStages * 8192, empty = full + 8 * kManyStages, acc_full = empty + 8 * kManyStages,
                   acc_empty = acc_full + 16, code_full = acc_empty + 16, code_empty = code_full + 8 * kCodeStages, tmem_at = code_empty + 8 * kCodeStages;
    const int warp = __shfl_sync(~0u, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;           // (of which the compiler knows that it is one for all)
    const uint32_t rank = cluster_rank();
    if (threadIdx.x == 0) {
        for (int s = 0; s < kManyStages; ++s) {
            bar_init(full + 8 * s, 2 * 4 + 1);                 // four warps of each block, and the copies
            bar_init(empty + 8 * s, 1);
        }
        for (int s = 0; s < 2; ++s) {
            bar_init(acc_full + 8 * s, 1);
            bar_init(acc_empty + 8 * s, 2 * kTakers);
        }
        for (int s = 0; s < kCodeStages; ++s) {
            bar_init(code_full + 8 * s, 1);
            bar_init(code_empty + 8 * s, 4);
        }
        bar_init_fence();
    }
    if (warp == 0) tmem_alloc(tmem_at, 512);
    __syncthreads();
    fence_before();
    cluster_sync();
    fence_after();
    uint32_t tmem;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(tmem) : "r"(tmem_at));
    after_previous();
    const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1, blocks = (a.tiles + 7) / 8;        // of 256 rows
    const int stages = (a.units + 1) / 2;      // of two units; the last one of a tile may have one
    bool ok = true;

    if (warp < kMakers) {
        // Codes to operands: a warp every other unit of its 32 rows, which are its quarter of tensor memory.
        const int quarter = warp & 3, turn = warp >> 2;
        const uint32_t to = tmem + (static_cast<uint32_t>(quarter * 32) << 16), full_of_pair = in_block(full, 0);
        const int steps = (blocks - pair + pairs - 1) / pairs * stages;
        uint32_t handed = 0;                   // the barrier of a stage that is on its way to tensor memory
        const auto hand_over = [&] {
            tmem_stored();
            fence_before();
            __syncwarp();
            if (lane == 0) bar_arrive_cluster(handed);         // (what is handed over is in tensor memory, and there)
        };
        int step = turn % stages, block = pair + turn / stages * pairs;
        for (int it = turn; it < steps && ok; it += kTurns) {
            const uint32_t cs = it % kCodeStages, s = it % kManyStages;
            const int u = 2 * step, many = min(2, a.units - u);
            uint32_t z[2][2] = {{0x08080808u, 0x08080808u}, {0x08080808u, 0x08080808u}};
            if (a.zeros) {
                const int tile = min(block * 8 + static_cast<int>(rank) * 4 + quarter, a.tiles - 1);
                const uint32_t* of_tile = a.zeros + static_cast<uint64_t>(tile * a.groups) * 8 + lane / 4;
                const auto group = [&](int unit) { return TWO ? unit * 2 : static_cast<int>(unit * a.per_group >> 20); };
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    if (h < many) {
                        z[h][0] = __ldg(of_tile + group(u + h) * 8);
                        if (TWO) z[h][1] = __ldg(of_tile + group(u + h) * 8 + 8);
                    }
                if (u + kAheadMeta < a.units) prefetch(of_tile + group(u + kAheadMeta) * 8);
            }
            for (step += kTurns; step >= stages; step -= stages) block += pairs;
            ok = __all_sync(~0u, bar_wait(code_full + 8 * cs, (it / kCodeStages) & 1));
            if (!ok) break;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (h >= many) break;
                const uint32_t at = codes + cs * 8192 + quarter * 2048 + h * 1024 + lane * 16;
                const uint4 code[2] = {shared_uint4(at), shared_uint4(at + 512)};
                uint32_t q[2][16];
#pragma unroll
                for (int half = 0; half < 2; ++half)
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint32_t w = k == 0 ? code[half].x : k == 1 ? code[half].y : k == 2 ? code[half].z : code[half].w;
                        const uint32_t zeros = z[h][TWO ? k >> 1 : 0] >> (16 * half);
                        H::operands(w, H::upper_zero(zeros & 15), H::lower_zero(zeros >> 8 & 15), &q[half][4 * k]);
                    }
                if (h == 0) {
                    if (handed) hand_over();
                    ok = __all_sync(~0u, bar_wait(empty + 8 * s, ((it / kManyStages) & 1) ^ 1));
                    if (!ok) break;
                    fence_after();
                }
                tmem_store(to + s * 64 + h * 32, q[0]);
                tmem_store(to + (16u << 16) + s * 64 + h * 32, q[1]);
            }
            __syncwarp();
            if (lane == 0) bar_arrive(code_empty + 8 * cs);
            handed = full_of_pair + 8 * s;
        }
        if (handed && ok) hand_over();
        if (!ok) tmem_stored();                // (before tensor memory is given back)
    } else if (warp < kMakers + kTakers) {
        // Products to sums: a warp 32 rows and half of the columns.
        const int quarter = warp & 3, half = (warp - kMakers) >> 2;
        const int place = (lane & 7) * 4 + (lane >> 3);
        uint32_t acc = 0;
        for (int t = pair; t < blocks; t += pairs) {
            const int tile = min(t * 8 + static_cast<int>(rank) * 4 + quarter, a.tiles - 1);
            const uint16_t* scales = a.scales + static_cast<int64_t>(tile) * a.groups * 32 + place;
            float sum[NC];
#pragma unroll
            for (int c = 0; c < NC; ++c) sum[c] = 0.f;
            uint32_t next = __ldg(scales);
            for (int g = 2; g < 2 + kAheadMeta && g < a.groups; g += 2) prefetch(scales + g * 32);
            for (int g = 0; g < a.groups && ok; ++g, ++acc) {
                const float scale = H::lower_half(next);
                if (g + 1 < a.groups) next = __ldg(scales + (g + 1) * 32);
                if (g + 2 + kAheadMeta < a.groups) prefetch(scales + (g + 2 + kAheadMeta) * 32);
                ok = __all_sync(~0u, bar_wait(acc_full + 8 * (acc & 1), (acc >> 1) & 1));
                if (!ok) break;
                fence_after();
                // in parts, as registers allow; the next one comes while one is added
                constexpr int kOnce = NC <= 32 ? NC : 16, kParts = NC / kOnce;
                const uint32_t at = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + kAcc + (acc & 1) * 2 * NC + half * NC;
                float v[kParts > 1 ? 2 : 1][kOnce];
                tmem_take<kOnce>(at, v[0]);
#pragma unroll
                for (int part = 0; part < kParts; ++part) {
                    float (&w)[kOnce] = v[kParts > 1 ? part & 1 : 0];
                    tmem_taken<kOnce>(w);
                    if (part + 1 < kParts) tmem_take<kOnce>(at + (part + 1) * kOnce, v[kParts > 1 ? part + 1 & 1 : 0]);
                    else {
                        fence_before();
                        __syncwarp();
                        if (lane == 0) bar_arrive_cluster(in_block(acc_empty + 8 * (acc & 1), 0));
                    }
#pragma unroll
                    for (int c = 0; c < kOnce; c += 2) add_scaled(sum[part * kOnce + c], sum[part * kOnce + c + 1], scale, w[c], w[c + 1]);
                }
            }
            const int64_t row = static_cast<int64_t>(t) * 256 + rank * 128 + quarter * 32 + lane;
            if (row >= a.vocab) continue;
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const int n = half * NC + c;
                if (n >= a.rows) break;
                const float x = ok ? sum[c] : __int_as_float(0x7FC00000);      // (a wait that ran out: nothing that could be taken for logits)
                if (a.wide) static_cast<float*>(a.out)[n * a.out_stride + row] = x;
                else static_cast<typename H::type*>(a.out)[n * a.out_stride + row] = from_float<typename H::type>(x);
            }
        }
    } else if (warp == kMakers + kTakers) {
        // Hidden states.
        const uint32_t full_of_pair = in_block(full, 0);
        uint32_t it = 0;
        for (int t = pair; t < blocks && ok; t += pairs)
            for (int step = 0; step < stages; ++step, ++it) {
                const uint32_t s = it % kManyStages;
                ok = __all_sync(~0u, bar_wait(empty + 8 * s, ((it / kManyStages) & 1) ^ 1));
                if (!ok) break;
                const bool two = 2 * step + 1 < a.units;
                if (elect()) {
                    if (rank == 0) bar_expect(full + 8 * s, two ? 2 * kStageBytes : kStageBytes);
                    load_tile(base + s * kStageBytes, &map_hidden, step * 128, rank * NC, full_of_pair + 8 * s);
                    if (two) load_tile(base + s * kStageBytes + NC * 128, &map_hidden, step * 128 + 64, rank * NC, full_of_pair + 8 * s);
                }
                __syncwarp();
            }
        for (uint32_t i = it < kManyStages ? 0 : it - kManyStages; i < it && ok; ++i) ok = __all_sync(~0u, bar_wait(empty + 8 * (i % kManyStages), (i / kManyStages) & 1));
        if (!ok) {                             // (copies that are under way end before the block does)
            const uint64_t from = nanoseconds();
            while (nanoseconds() - from < 2000000ull) __nanosleep(1000);
        }
    } else if (warp == kMakers + kTakers + 1) {
        // Codes.
        uint32_t it = 0;
        for (int t = pair; t < blocks && ok; t += pairs) {
            const uint4* from[4];
#pragma unroll
            for (int quarter = 0; quarter < 4; ++quarter)
                from[quarter] = a.codes + static_cast<int64_t>(min(t * 8 + static_cast<int>(rank) * 4 + quarter, a.tiles - 1)) * a.units * 64;
            for (int step = 0; step < stages; ++step, ++it) {
                const uint32_t s = it % kCodeStages, bytes = 2 * step + 1 < a.units ? 2048 : 1024;
                ok = __all_sync(~0u, bar_wait(code_empty + 8 * s, ((it / kCodeStages) & 1) ^ 1));
                if (!ok) break;
                if (elect()) {
                    bar_expect(code_full + 8 * s, 4 * bytes);
#pragma unroll
                    for (int quarter = 0; quarter < 4; ++quarter) load_line(codes + s * 8192 + quarter * 2048, from[quarter] + step * 128, bytes, code_full + 8 * s);
                }
                __syncwarp();
            }
        }
        for (uint32_t i = it < kCodeStages ? 0 : it - kCodeStages; i < it && ok; ++i) ok = __all_sync(~0u, bar_wait(code_empty + 8 * (i % kCodeStages), (i / kCodeStages) & 1));
        if (!ok) {
            const uint64_t from = nanoseconds();
            while (nanoseconds() - from < 2000000ull) __nanosleep(1000);
        }
    } else if (rank == 0 && elect()) {
        // Products.
        const uint32_t kind = mma_kind(BF16, false, false, 2 * NC);
        uint32_t it = 0, acc = 0;
        int in_group = 0;
        // One unit, in one thread and without more branches than there have to be: each costs the others' way through the instruction cache.
        const auto unit = [&](uint32_t b, uint32_t from, bool last) {
            if (in_group == 0) {
                if (!bar_wait(acc_empty + 8 * (acc & 1), ((acc >> 1) & 1) ^ 1)) return false;
                fence_after();
            }
            const uint64_t b0 = operand(b, false);                     // (32 bytes on: 2 more)
            const uint32_t to = tmem + kAcc + (acc & 1) * 2 * NC;
            mma_from_tmem(to, from, b0, kind, in_group > 0);
            mma_from_tmem(to, from + 8, b0 + 2, kind, true);
            uint32_t second = to;
            if (TWO) {                         // (the unit's second group)
                mma_commit(acc_full + 8 * (acc & 1));
                ++acc;
                if (!bar_wait(acc_empty + 8 * (acc & 1), ((acc >> 1) & 1) ^ 1)) return false;
                fence_after();
                second = tmem + kAcc + (acc & 1) * 2 * NC;
            }
            mma_from_tmem(second, from + 16, b0 + 4, kind, !TWO);
            mma_from_tmem(second, from + 24, b0 + 6, kind, true);
            if (TWO || ++in_group == a.group_units || last) {
                in_group = 0;
                mma_commit(acc_full + 8 * (acc & 1));
                ++acc;
            }
            return true;
        };
        for (int t = pair; t < blocks && ok; t += pairs)
            for (int step = 0; step < stages; ++step, ++it) {
                const uint32_t s = it % kManyStages, b = base + s * kStageBytes, from = tmem + s * 64;
                if (!bar_wait(full + 8 * s, (it / kManyStages) & 1)) { ok = false; break; }
                fence_after();
                const bool two = 2 * step + 1 < a.units, last = step + 1 == stages;
                ok = unit(b, from, last && !two);
                if (ok && two) ok = unit(b + NC * 128, from + 32, last);
                if (!ok) break;
                mma_commit(empty + 8 * s);
            }
    }
    __syncwarp();
    let_next_begin();
    __syncthreads();
    fence_before();
    cluster_sync();
    fence_after();
    if (warp == 0) tmem_free(tmem, 512);
}

template <bool BF16, int NC>
cudaError_t many_rows(const CUtensorMap& map, const ManyArgs& a, int blocks, cudaStream_t stream) {
    auto* kernel = a.group_units ? many_rows_kernel<BF16, NC, false> : many_rows_kernel<BF16, NC, true>;
    if (cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kManySmem)) return e;
    return launch(kernel, blocks, many_threads(!a.group_units), kManySmem, stream, map, a);
}
template <bool BF16>
cudaError_t many_rows(const CUtensorMap& map, const ManyArgs& a, int columns, int blocks, cudaStream_t stream) {
    switch (columns) {
        case 8: return many_rows<BF16, 8>(map, a, blocks, stream);
        case 16: return many_rows<BF16, 16>(map, a, blocks, stream);
        case 24: return many_rows<BF16, 24>(map, a, blocks, stream);
        case 32: return many_rows<BF16, 32>(map, a, blocks, stream);
        case 48: return many_rows<BF16, 48>(map, a, blocks, stream);
        default: return many_rows<BF16, 64>(map, a, blocks, stream);
    }
}

const char* said(cudaError_t e) { return e == cudaSuccess ? nullptr : cudaGetErrorString(e); }

}  // namespace

const char* pack_table(const Table4& t, const uint8_t* codes, int64_t codes_stride, const Matrix& scales, const uint8_t* zeros, int64_t zeros_stride, cudaStream_t stream) {
    PackArgs a{};
    a.t = t;
    a.p = table4_plan(t.vocab, t.width, t.group, t.zeros);
    a.codes = codes;
    a.codes_stride = codes_stride;
    a.scales = scales.data;
    a.scales_stride = scales.stride;
    a.zeros = zeros;
    a.zeros_stride = zeros_stride;
    if (!a.p.tiles) return nullptr;
    return said(launch(pack_kernel, std::min<int64_t>(div_up(a.p.tiles * a.p.units, 8), 148 * 8), 256, 0, stream, a));
}

namespace {
template <typename W>
cudaError_t quantize(const QuantizeArgs& a, int64_t stretch, cudaStream_t stream) {
    const int64_t blocks = a.p.tiles * div_up(a.p.units, stretch);
    return a.t.type == kBF16 ? launch(quantize_kernel<W, __nv_bfloat16>, blocks, 256, 0, stream, a, stretch)
                             : launch(quantize_kernel<W, __half>, blocks, 256, 0, stream, a, stretch);
}
}  // namespace

const char* quantize_table(const Table4& t, const Matrix& weight, cudaStream_t stream) {
    QuantizeArgs a{};
    a.t = t;
    a.p = table4_plan(t.vocab, t.width, t.group, t.zeros);
    a.weight = weight.data;
    a.stride = weight.stride;
    if (!a.p.tiles) return nullptr;
    // whole groups, and some columns at least: a group of more than 512 columns is a stretch of its own
    const int64_t stretch = std::max<int64_t>(t.group <= 64 ? kQuantUnits : kQuantUnits / (t.group / 64) * (t.group / 64), t.group / 64);
    switch (weight.type) {
        case kF32: return said(quantize<float>(a, stretch, stream));
        case kBF16: return said(quantize<__nv_bfloat16>(a, stretch, stream));
        default: return said(quantize<__half>(a, stretch, stream));
    }
}

const char* table_logits(const Matrix& hidden, const Table4& t, const Matrix& out, cudaStream_t stream) {
    if (!hidden.rows || !t.vocab) return nullptr;
    const Table4Plan p = table4_plan(t.vocab, t.width, t.group, t.zeros);
    const char* at = static_cast<const char*>(t.data);
    LogitsArgs a{};
    a.codes = reinterpret_cast<const uint4*>(at);
    a.scales = reinterpret_cast<const uint16_t*>(at + p.scales);
    a.zeros = t.zeros ? reinterpret_cast<const uint8_t*>(at + p.zeros) : nullptr;
    a.hidden_stride = hidden.stride;
    a.out_stride = out.stride;
    a.vocab = t.vocab;
    a.width = t.width;
    a.tiles = static_cast<int>(p.tiles);
    a.groups = static_cast<int>(p.groups);
    a.units = static_cast<int>(p.units);
    // (u / d for u and d up to 1024: u times the rounding is less than 1 / d of 2^20)
    a.per_group = t.group == 32 ? 0 : static_cast<uint32_t>(div_up(1 << 20, t.group / 64));
    const int64_t pairs = div_up(p.tiles, 2);
    const int blocks = static_cast<int>(std::min<int64_t>(148, pairs));
    // Warps that share rows: so many that the slowest warp of the fullest block takes the fewest steps, of which adding up at the end of its rows is about one.
    const auto steps = [&](int log) { return div_up(div_up(pairs, blocks), kWarps >> log) * (div_up(a.units, 1 << log) + 1); };
    a.split_log = 0;
    for (int log = 1; log <= 4 && (1 << log) <= a.units; ++log)
        if (steps(log) <= steps(a.split_log)) a.split_log = log;
    a.split = 1 << a.split_log;
    const int size = out.type == kF32 ? 4 : 2;
    // Tiled copies of hidden states take lines of whole 16 bytes.
    const bool whole = reinterpret_cast<uintptr_t>(hidden.data) % 16 == 0 && hidden.stride % 8 == 0 && hidden.stride >= hidden.cols;
    ManyArgs m{};
    m.codes = a.codes;
    m.scales = a.scales;
    m.zeros = reinterpret_cast<const uint32_t*>(a.zeros);
    m.out_stride = out.stride;
    m.vocab = t.vocab;
    m.tiles = a.tiles;
    m.groups = a.groups;
    m.units = a.units;
    m.group_units = t.group == 32 ? 0 : static_cast<int>(t.group / 64);
    m.per_group = a.per_group;
    m.wide = out.type == kF32;
    for (int64_t row = 0; row < hidden.rows;) {
        const int64_t left = hidden.rows - row;
        const bool few = few_smem(2, a.units, true, 1) <= kMostSmem;           // two tiles of eight rows are at hand
        if (left > (few && t.group < 128 ? kFewRows : 8) && whole) {
            // Rows in equal parts, as a part of few rows costs about what one of many does.
            const int rows = static_cast<int>(div_up(left, div_up(left, kMostColumns))), needed = (rows + 15) / 16 * 8;
            const int columns = needed <= 32 ? needed : needed <= 48 ? 48 : 64;
            CUtensorMap map;
            if (!encode_fn()) return "the driver has no tiled copies";
            if (!tile_map(&map, hidden.type, static_cast<const uint16_t*>(hidden.data) + row * hidden.stride, rows, hidden.cols, hidden.stride, columns))
                return "a tensor map was refused";
            m.out = static_cast<char*>(const_cast<void*>(out.data)) + row * out.stride * size;
            m.rows = rows;
            const cudaError_t e = hidden.type == kBF16 ? many_rows<true>(map, m, columns, 2 * static_cast<int>(std::min<int64_t>(74, div_up(p.tiles, 8))), stream)
                                                       : many_rows<false>(map, m, columns, 2 * static_cast<int>(std::min<int64_t>(74, div_up(p.tiles, 8))), stream);
            if (e != cudaSuccess) return cudaGetErrorString(e);
            row += rows;
            continue;
        }
        const int nt = left > 8 && few ? 2 : 1;
        a.pairs = reinterpret_cast<uintptr_t>(hidden.data) % 4 == 0 && hidden.stride % 2 == 0 && hidden.cols % 2 == 0;
        a.staged = few_smem(nt, a.units, true, 1) <= kMostSmem;
        a.buffers = few_smem(nt, a.units, a.staged, 2) <= kMostSmem ? 2 : 1;
        a.rows = static_cast<int>(std::min<int64_t>(left, 8 * nt));
        a.hidden = static_cast<const uint16_t*>(hidden.data) + row * hidden.stride;
        a.out = static_cast<char*>(const_cast<void*>(out.data)) + row * out.stride * size;
        const bool wide = out.type == kF32;
        const cudaError_t e = hidden.type == kBF16 ? (wide ? few_rows<true, float>(a, nt, blocks, stream) : few_rows<true, __nv_bfloat16>(a, nt, blocks, stream))
                                                   : (wide ? few_rows<false, float>(a, nt, blocks, stream) : few_rows<false, __half>(a, nt, blocks, stream));
        if (e != cudaSuccess) return cudaGetErrorString(e);
        row += a.rows;
    }
    return nullptr;
}

}  // namespace gtok
