// A table in 4 bits: laid out for the products, made from weights, and multiplied with hidden states.
//
// z[i, v] = sum over groups g of s[v, g] * sum over k in g of (q[v, k] - b[v, g]) * h[i, k], with codes q of 0 to 15, a scale s and a zero b
// (8 where there are none) for each group of a row.  q - b is a whole number of at most 15 and exact in bf16 and fp16, so the inner sums are
// matrix products of what is stored, in fp32, and only they are scaled: no weight is rounded on the way.
#include "vocab_launch.cuh"
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

// A warp a pair of units, done once for a table: every byte read and written once, but bytes by bytes.
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
// one whose scale rounds to 0, has scale 0.  A group with a NaN or an infinity gets the scale NaN.
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
            const float s = to_float<T>(from_float<T>((a.t.zeros ? high / 15.f - low / 15.f : fmaxf(high, -low) / 7.f) + bad));
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
constexpr int kWarps = 16, kThreads = kWarps * 32, kAhead = 4;
constexpr int kPartLine = 36;              // floats from a row of hidden states to the next among partial sums: lanes of a fragment meet no bank twice

struct LogitsArgs {
    const uint4* codes;
    const uint16_t* scales;
    const uint8_t* zeros;
    const uint16_t* hidden;
    int64_t hidden_stride;
    void* out;
    int64_t out_stride, vocab, width;
    int64_t tiles, groups;
    int units, group_units;        // of 64 columns; how many share a group (0: each has two)
    int rows;                      // of hidden states, at most 8 NT
    int split, split_log;          // warps that share a tile
    bool staged;                   // hidden states fit into shared memory
};

template <bool BF16> struct Half16;
template <> struct Half16<true> {
    using type = __nv_bfloat16;
    static constexpr uint32_t kBase = 0x43004300u;             // 128 + code, twice
    static __device__ __forceinline__ uint32_t pair(uint32_t zero) { return kBase + (zero << 16 | zero); }
    static __device__ __forceinline__ uint32_t minus(uint32_t a, uint32_t b) {
        const __nv_bfloat162 r = __hsub2(reinterpret_cast<const __nv_bfloat162&>(a), reinterpret_cast<const __nv_bfloat162&>(b));
        return reinterpret_cast<const uint32_t&>(r);
    }
    static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint2 b) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b.x), "r"(b.y));
    }
};
template <> struct Half16<false> {
    using type = __half;
    static constexpr uint32_t kBase = 0x64006400u;             // 1024 + code, twice
    static __device__ __forceinline__ uint32_t pair(uint32_t zero) { return kBase + (zero << 16 | zero); }
    static __device__ __forceinline__ uint32_t minus(uint32_t a, uint32_t b) {
        const __half2 r = __hsub2(reinterpret_cast<const __half2&>(a), reinterpret_cast<const __half2&>(b));
        return reinterpret_cast<const uint32_t&>(r);
    }
    static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint2 b) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b.x), "r"(b.y));
    }
};

// Operand pair of hidden states: row `n`, columns col and col + 1, 0 outside.
__device__ __forceinline__ uint32_t hidden_pair(const LogitsArgs& a, int n, int64_t col) {
    if (n >= a.rows) return 0;
    const uint16_t* row = a.hidden + n * a.hidden_stride;
    const uint32_t low = col < a.width ? row[col] : 0, high = col + 1 < a.width ? row[col + 1] : 0;
    return high << 16 | low;
}

// What a lane has under way of one unit pair: 32 rows x 64 columns.
template <int SUBS, bool ZEROS>
struct Lot {
    uint4 code[2];
    uint2 scale[SUBS];             // of the lane's four rows, 16 bits each
    uint32_t zero[ZEROS ? SUBS : 1];
};

__device__ __forceinline__ uint4 load_once(const uint4* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

template <bool BF16, int NT, int SUBS, bool ZEROS, typename Out>
__global__ void __launch_bounds__(kThreads, 1) few_rows_kernel(const __grid_constant__ LogitsArgs a) {
    using H = Half16<BF16>;
    extern __shared__ uint4 smem[];
    constexpr int kPart = 8 * NT * kPartLine;                  // floats of a warp's partial sums
    float* parts = reinterpret_cast<float*>(smem);             // [2][kWarps][kPart]
    uint2* staged = reinterpret_cast<uint2*>(parts + 2 * kWarps * kPart);      // [units * 4][NT][32]
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    after_previous();
    let_next_begin();
    const int64_t first = a.tiles * blockIdx.x / gridDim.x, last = a.tiles * (blockIdx.x + 1) / gridDim.x;
    const int at_once = kWarps >> a.split_log, part = warp & (a.split - 1), slot = warp >> a.split_log;
    const int64_t rounds = (last - first + at_once - 1) >> (4 - a.split_log);
    const int count = (a.units - part + a.split - 1) >> a.split_log;           // units of a tile that are this warp's; one at least

    // Units are fetched kAhead before they are needed, across the ends of tiles.
    Lot<SUBS, ZEROS> lot[kAhead];
    int64_t fetch_round = 0;
    int fetch_i = 0;
    const auto fetch = [&](Lot<SUBS, ZEROS>& l) {
        if (fetch_round >= rounds) return;
        int64_t tile = first + fetch_round * at_once + slot;
        if (tile >= last) tile = last - 1;                     // (its sums are left out)
        const int u = part + (fetch_i << a.split_log);
        const uint4* p = a.codes + (tile * a.units + u) * 64 + lane;
        l.code[0] = load_once(p);
        l.code[1] = load_once(p + 32);
#pragma unroll
        for (int s = 0; s < SUBS; ++s) {
            const int64_t g = tile * a.groups + (SUBS == 2 ? u * 2 + s : u / a.group_units);
            l.scale[s] = __ldg(reinterpret_cast<const uint2*>(a.scales + g * 32) + lane / 4);
            if constexpr (ZEROS) l.zero[s] = __ldg(reinterpret_cast<const uint32_t*>(a.zeros + g * 32) + lane / 4);
        }
        if (++fetch_i == count) {
            fetch_i = 0;
            ++fetch_round;
        }
    };
#pragma unroll
    for (int s = 0; s < kAhead; ++s) fetch(lot[s]);
    if (a.staged) {
        for (int i = tid; i < a.units * 4 * NT * 32; i += kThreads) {
            const int l = i & 31, nt = (i >> 5) % NT, step = (i >> 5) / NT;
            const int64_t col = step * 16 + 2 * (l & 3);
            staged[i] = make_uint2(hidden_pair(a, nt * 8 + l / 4, col), hidden_pair(a, nt * 8 + l / 4, col + 8));
        }
        __syncthreads();
    }

    float acc[2][NT][4] = {};
    int i = 0, buffer = 0;
    int64_t round = 0;
    while (round < rounds) {
#pragma unroll
        for (int s = 0; s < kAhead; ++s) {
            if (round >= rounds) break;
            const Lot<SUBS, ZEROS>& l = lot[s];
            const int u = part + (i << a.split_log);
#pragma unroll
            for (int sub = 0; sub < SUBS; ++sub) {
                float sum[2][NT][4] = {};
                uint32_t base[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) base[r] = H::pair(ZEROS ? l.zero[ZEROS ? sub : 0] >> (8 * r) & 15 : 8);
#pragma unroll
                for (int k = 4 / SUBS * sub; k < 4 / SUBS * (sub + 1); ++k) {
                    uint2 b[NT];
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        if (a.staged) b[nt] = staged[((u * 4 + k) * NT + nt) * 32 + lane];
                        else {
                            const int64_t col = (u * 4 + k) * 16 + 2 * (lane & 3);
                            b[nt] = make_uint2(hidden_pair(a, nt * 8 + lane / 4, col), hidden_pair(a, nt * 8 + lane / 4, col + 8));
                        }
                    }
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const uint32_t w = k == 0 ? l.code[half].x : k == 1 ? l.code[half].y : k == 2 ? l.code[half].z : l.code[half].w;
                        uint32_t q[4];
#pragma unroll
                        for (int p = 0; p < 4; ++p) q[p] = H::minus((w >> (4 * p) & 0x000F000Fu) | H::kBase, base[half * 2 + (p & 1)]);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) H::mma(sum[half][nt], q, b[nt]);
                    }
                }
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    using T = typename H::type;
                    const uint32_t w = half ? l.scale[sub].y : l.scale[sub].x;
                    const float upper = to_float<T>(reinterpret_cast<const T*>(&w)[0]), lower = to_float<T>(reinterpret_cast<const T*>(&w)[1]);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        acc[half][nt][0] = fmaf(upper, sum[half][nt][0], acc[half][nt][0]);
                        acc[half][nt][1] = fmaf(upper, sum[half][nt][1], acc[half][nt][1]);
                        acc[half][nt][2] = fmaf(lower, sum[half][nt][2], acc[half][nt][2]);
                        acc[half][nt][3] = fmaf(lower, sum[half][nt][3], acc[half][nt][3]);
                    }
                }
            }
            fetch(lot[s]);
            if (++i < count) continue;
            // The tiles of a round are done: partial sums of the warps that share one are added in their order.
            i = 0;
            float* mine = parts + (buffer * kWarps + warp) * kPart;
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        mine[(nt * 8 + 2 * (lane & 3) + (e & 1)) * kPartLine + half * 16 + lane / 4 + (e >> 1) * 8] = acc[half][nt][e];
                        acc[half][nt][e] = 0.f;
                    }
            asm volatile("bar.sync 1, %0;" ::"n"(kThreads) : "memory");        // (warps come here from different places of the unrolled loop)
            for (int o = tid; o < at_once * a.rows * 32; o += kThreads) {
                const int r = o & 31, n = (o >> 5) % a.rows, t = (o >> 5) / a.rows;
                const int64_t tile = first + round * at_once + t, v = tile * 32 + r;
                if (tile >= last || v >= a.vocab) continue;
                const float* from = parts + (buffer * kWarps + (t << a.split_log)) * kPart + n * kPartLine + r;
                float total = from[0];
                for (int p = 1; p < a.split; ++p) total += from[p * kPart];
                static_cast<Out*>(a.out)[n * a.out_stride + v] = from_float<Out>(total);
            }
            buffer ^= 1;
            ++round;
        }
    }
}

int few_smem(int nt, int units, bool staged) { return 2 * kWarps * 8 * nt * kPartLine * 4 + (staged ? units * 4 * nt * 32 * 8 : 0); }
constexpr int kMostSmem = 227 * 1024;

template <bool BF16, int NT, int SUBS, bool ZEROS, typename Out>
cudaError_t few_rows(const LogitsArgs& a, int blocks, cudaStream_t stream) {
    auto* kernel = few_rows_kernel<BF16, NT, SUBS, ZEROS, Out>;
    const int smem = few_smem(NT, a.units, a.staged);
    if (cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostSmem)) return e;
    return launch(kernel, blocks, kThreads, smem, stream, a);
}
template <bool BF16, int NT, typename Out>
cudaError_t few_rows(const LogitsArgs& a, int blocks, cudaStream_t stream) {
    if (a.group_units == 0) return a.zeros ? few_rows<BF16, NT, 2, true, Out>(a, blocks, stream) : few_rows<BF16, NT, 2, false, Out>(a, blocks, stream);
    return a.zeros ? few_rows<BF16, NT, 1, true, Out>(a, blocks, stream) : few_rows<BF16, NT, 1, false, Out>(a, blocks, stream);
}
template <bool BF16, typename Out>
cudaError_t few_rows(const LogitsArgs& a, int nt, int blocks, cudaStream_t stream) {
    return nt == 1 ? few_rows<BF16, 1, Out>(a, blocks, stream) : few_rows<BF16, 2, Out>(a, blocks, stream);
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
    a.tiles = p.tiles;
    a.groups = p.groups;
    a.units = static_cast<int>(p.units);
    a.group_units = t.group == 32 ? 0 : static_cast<int>(t.group / 64);
    const int blocks = static_cast<int>(std::min<int64_t>(148, p.tiles));
    // warps that share a tile: all, or as many as there are units
    a.split_log = 4;
    while ((1 << a.split_log) > a.units) --a.split_log;
    a.split = 1 << a.split_log;
    const int size = out.type == kF32 ? 4 : 2;
    for (int64_t row = 0; row < hidden.rows;) {
        const int64_t left = hidden.rows - row;
        const int nt = left > 8 && few_smem(2, a.units, true) <= kMostSmem ? 2 : 1;
        a.staged = few_smem(nt, a.units, true) <= kMostSmem;
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
