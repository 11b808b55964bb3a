// Rows of a table by token id: the embedding lookup, its gradient, and the ids that follow in packed documents.
#include "vocab_ops.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

namespace gtok {
namespace {

__device__ __forceinline__ int64_t load_id(const void* ids, int bits, int64_t i) {
    return bits == 64 ? static_cast<const int64_t*>(ids)[i] : static_cast<const int32_t*>(ids)[i];
}

template <typename T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

// `N` elements that are read and written together: 16 bytes, or one element where rows do not allow that.
template <typename T, int N>
struct alignas(sizeof(T) * N) Lump {
    T v[N];
};

// ---- lookup ---------------------------------------------------------------------
// out[t, :] = scale * table[id_t, :]; a negative id gives a row of zeros, an id beyond the table a row of NaN.  Bound by memory: each
// thread has four lumps under way.
template <typename T, int N>
__global__ void __launch_bounds__(256) embed_kernel(const void* ids, int bits, int64_t n, const T* table, int64_t vocab, int64_t stride, int lumps, float scale, T* out,
                                                    int64_t out_stride) {
    using L = Lump<T, N>;
    for (int64_t t = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y; t < n; t += static_cast<int64_t>(gridDim.x) * blockDim.y) {
        const int64_t id = load_id(ids, bits, t);
        const bool known = id >= 0 && id < vocab;
        const L* from = reinterpret_cast<const L*>(table + (known ? id : 0) * stride);
        L* to = reinterpret_cast<L*>(out + t * out_stride);
        const T other = from_float<T>(id < 0 ? 0.f : __int_as_float(0x7FC00000));
        for (int i = threadIdx.x; i < lumps; i += 4 * blockDim.x) {
            L v[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (known && i + k * static_cast<int>(blockDim.x) < lumps) v[k] = from[i + k * blockDim.x];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (i + k * static_cast<int>(blockDim.x) >= lumps) break;
#pragma unroll
                for (int e = 0; e < N; ++e) v[k].v[e] = known ? from_float<T>(scale * to_float<T>(v[k].v[e])) : other;
                to[i + k * blockDim.x] = v[k];
            }
        }
    }
}

// ---- the ids that follow ----------------------------------------------------------
__global__ void next_kernel(const int32_t* ids, int64_t n, const int32_t* offsets, int64_t n_docs, const uint8_t* loss_mask, int32_t ignore, int32_t* out) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
    if (i >= n) return;
    int64_t lo = 0, hi = n_docs + 1;              // offsets at or before i
    while (lo < hi) {
        const int64_t mid = (lo + hi) >> 1;
        if (offsets[mid] <= i) lo = mid + 1; else hi = mid;
    }
    const bool inner = lo >= 1 && lo <= n_docs && i + 1 < offsets[lo] && i + 1 < n;
    out[i] = inner && (!loss_mask || loss_mask[i]) ? ids[i + 1] : ignore;
}

// ---- the lookup's gradient ----------------------------------------------------------
// The places of the ids are sorted by id (radix sort, stable), so that the rows to be summed for one id follow one another in the
// order of the text and their sum does not depend on how the GPU runs.  Runs of equal ids differ from one place to tens of thousands;
// the sorted places are therefore cut into chunks of 32 whatever they hold, and runs across chunks are joined from fp32 partial sums.
constexpr int kDigit = 9, kBins = 1 << kDigit;
constexpr int kSortThreads = 256, kSortEach = 8, kSortTile = kSortThreads * kSortEach;
constexpr int kChunk = 32;

struct Key { uint32_t id, place; };

// First pass: keys from the ids (those outside the table sort behind it), and which rows of the table occur.
__device__ __forceinline__ uint32_t key_of(const void* ids, int bits, int64_t i, uint32_t vocab) {
    const int64_t id = load_id(ids, bits, i);
    return id >= 0 && id < vocab ? static_cast<uint32_t>(id) : vocab;
}

template <bool FIRST>
__global__ void __launch_bounds__(kSortThreads) count_kernel(const void* ids, int bits, const Key* in, int64_t n, uint32_t vocab, int shift, uint32_t* counts,
                                                             uint32_t* seen) {
    __shared__ uint32_t bin[kBins];
    for (int b = threadIdx.x; b < kBins; b += kSortThreads) bin[b] = 0;
    __syncthreads();
    const int64_t from = static_cast<int64_t>(blockIdx.x) * kSortTile;
    for (int i = threadIdx.x; i < kSortTile && from + i < n; i += kSortThreads) {
        const uint32_t key = FIRST ? key_of(ids, bits, from + i, vocab) : in[from + i].id;
        atomicAdd(&bin[key >> shift & (kBins - 1)], 1u);
        if (FIRST && key < vocab) atomicOr(&seen[key >> 5], 1u << (key & 31));
    }
    __syncthreads();
    for (int b = threadIdx.x; b < kBins; b += kSortThreads) counts[static_cast<int64_t>(blockIdx.x) * kBins + b] = bin[b];
}

template <bool FIRST>
__global__ void __launch_bounds__(kSortThreads) scatter_kernel(const void* ids, int bits, const Key* in, int64_t n, uint32_t vocab, int shift, const uint32_t* counts,
                                                               Key* out) {
    constexpr int kWarps = kSortThreads / 32;
    __shared__ uint32_t base[kBins];
    __shared__ uint16_t warp_bin[kWarps][kBins];
    __shared__ uint32_t warp_sum[kWarps];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    for (int b = tid; b < kWarps * kBins; b += kSortThreads) (&warp_bin[0][0])[b] = 0;
    // where this tile's keys of each bin begin: all smaller bins, and the same bin in the tiles before
    uint32_t all[2], mine[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        uint32_t sum = 0, before = 0;
        for (uint32_t t = 0; t < gridDim.x; ++t) {
            const uint32_t c = counts[static_cast<int64_t>(t) * kBins + 2 * tid + k];
            before += t < blockIdx.x ? c : 0;
            sum += c;
        }
        all[k] = sum;
        mine[k] = before;
    }
    uint32_t scan = all[0] + all[1];
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const uint32_t y = __shfl_up_sync(~0u, scan, d);
        if (lane >= d) scan += y;
    }
    if (lane == 31) warp_sum[warp] = scan;
    __syncthreads();
    for (int w = 0; w < warp; ++w) scan += warp_sum[w];
    base[2 * tid] = scan - all[0] - all[1] + mine[0];
    base[2 * tid + 1] = scan - all[1] + mine[1];
    // each warp takes its 256 keys in order; a key's rank among those of its bin
    const int64_t from = static_cast<int64_t>(blockIdx.x) * kSortTile + warp * 32 * kSortEach;
    Key key[kSortEach];
    uint16_t rank[kSortEach];
#pragma unroll
    for (int i = 0; i < kSortEach; ++i) {
        const int64_t at = from + i * 32 + lane;
        key[i] = Key{0xFFFFFFFFu, 0};
        if (at < n) key[i] = FIRST ? Key{key_of(ids, bits, at, vocab), static_cast<uint32_t>(at)} : in[at];
    }
#pragma unroll
    for (int i = 0; i < kSortEach; ++i) {
        const bool here = from + i * 32 + lane < n;
        const uint32_t b = here ? key[i].id >> shift & (kBins - 1) : kBins;
        const uint32_t same = __match_any_sync(~0u, b);
        uint16_t seen = here ? warp_bin[warp][b] : 0;
        __syncwarp();
        rank[i] = seen + __popc(same & ((1u << lane) - 1));
        if (here && (same & ((1u << lane) - 1)) == 0) warp_bin[warp][b] = seen + __popc(same);
        __syncwarp();
    }
    __syncthreads();
    for (int b = tid; b < kBins; b += kSortThreads) {
        uint32_t sum = base[b];
        base[b] = sum;
        uint32_t run = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const uint32_t c = warp_bin[w][b];
            warp_bin[w][b] = static_cast<uint16_t>(run);
            run += c;
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kSortEach; ++i) {
        if (from + i * 32 + lane >= n) continue;
        const uint32_t b = key[i].id >> shift & (kBins - 1);
        out[base[b] + warp_bin[warp][b] + rank[i]] = key[i];
    }
}

template <typename T, int N>
__device__ __forceinline__ void put_row(T* out, int64_t at, const float (&sum)[N], float scale, bool accumulate) {
    using L = Lump<T, N>;
    L* to = reinterpret_cast<L*>(out + at);
    L v;
    if (accumulate) v = *to;
#pragma unroll
    for (int e = 0; e < N; ++e) v.v[e] = from_float<T>(accumulate ? to_float<T>(v.v[e]) + scale * sum[e] : scale * sum[e]);
    *to = v;
}

// Sums of the runs in a chunk, one warp a chunk and 32 lumps of columns; rows that no id asks for become 0 (unless summed onto `out`).
template <typename T, int N>
__global__ void __launch_bounds__(256) sum_kernel(const Key* keys, int64_t n, uint32_t vocab, const T* grad, int64_t stride, int lumps, float scale, T* out,
                                                  int64_t out_stride, bool accumulate, float* partial, int64_t partial_cols, int slices, const uint32_t* seen) {
    using L = Lump<T, N>;
    const int lane = threadIdx.x & 31;
    const int64_t warps = static_cast<int64_t>(gridDim.x) * (blockDim.x / 32), self = static_cast<int64_t>(blockIdx.x) * (blockDim.x / 32) + (threadIdx.x >> 5);
    const int64_t chunks = (n + kChunk - 1) / kChunk;
    for (int64_t u = self; u < chunks * slices; u += warps) {
        const int64_t chunk = u / slices;
        const int col = (static_cast<int>(u - chunk * slices) * 32 + lane);
        const bool here = col < lumps;
        const int64_t from = chunk * kChunk;
        const int count = static_cast<int>(min(static_cast<int64_t>(kChunk), n - from));
        const Key mine = lane < count ? keys[from + lane] : Key{0xFFFFFFFFu, 0};
        const uint32_t before = from > 0 ? keys[from - 1].id : 0xFFFFFFFEu, after = from + count < n ? keys[from + count].id : 0xFFFFFFFEu;
        float sum[N];
#pragma unroll
        for (int e = 0; e < N; ++e) sum[e] = 0.f;
        uint32_t run = __shfl_sync(~0u, mine.id, 0);
        bool open = run == before;                 // the run began in an earlier chunk
        bool whole_front = true;                   // it begins where the chunk does
        for (int i = 0; i < count; i += 8) {
            L v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const uint32_t id = __shfl_sync(~0u, mine.id, (i + k) & 31), place = __shfl_sync(~0u, mine.place, (i + k) & 31);
                if (here && i + k < count && id < vocab) v[k] = reinterpret_cast<const L*>(grad + static_cast<int64_t>(place) * stride)[col];
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                if (i + k >= count) break;
                const uint32_t id = __shfl_sync(~0u, mine.id, i + k);
                if (id != run) {
                    if (here && run < vocab) {
                        if (open) {
#pragma unroll
                            for (int e = 0; e < N; ++e) partial[(chunk * 2) * partial_cols + static_cast<int64_t>(col) * N + e] = sum[e];
                        } else {
                            put_row<T, N>(out, run * out_stride + static_cast<int64_t>(col) * N, sum, scale, accumulate);
                        }
                    }
#pragma unroll
                    for (int e = 0; e < N; ++e) sum[e] = 0.f;
                    run = id;
                    open = whole_front = false;
                }
                if (here && id < vocab) {
#pragma unroll
                    for (int e = 0; e < N; ++e) sum[e] += to_float<T>(v[k].v[e]);
                }
            }
        }
        if (here && run < vocab) {
            if (open || run == after) {
                const int64_t slot = chunk * 2 + (whole_front ? 0 : 1);
#pragma unroll
                for (int e = 0; e < N; ++e) partial[slot * partial_cols + static_cast<int64_t>(col) * N + e] = sum[e];
            } else {
                put_row<T, N>(out, run * out_stride + static_cast<int64_t>(col) * N, sum, scale, accumulate);
            }
        }
    }
    if (accumulate) return;
    L zero;
#pragma unroll
    for (int e = 0; e < N; ++e) zero.v[e] = from_float<T>(0.f);
    for (int64_t r = self; r < vocab; r += warps) {
        if (seen[r >> 5] >> (r & 31) & 1) continue;
        L* to = reinterpret_cast<L*>(out + r * out_stride);
        for (int i = lane; i < lumps; i += 32) to[i] = zero;
    }
}

// Runs across chunks: the warp of the chunk where one begins adds its parts up, in order.
template <typename T, int N>
__global__ void __launch_bounds__(256) join_runs_kernel(const Key* keys, int64_t n, uint32_t vocab, int lumps, float scale, T* out, int64_t out_stride, bool accumulate,
                                                        const float* partial, int64_t partial_cols, int slices) {
    const int lane = threadIdx.x & 31;
    const int64_t warps = static_cast<int64_t>(gridDim.x) * (blockDim.x / 32), self = static_cast<int64_t>(blockIdx.x) * (blockDim.x / 32) + (threadIdx.x >> 5);
    const int64_t chunks = (n + kChunk - 1) / kChunk;
    for (int64_t u = self; u < (chunks - 1) * slices; u += warps) {
        const int64_t chunk = u / slices;
        const int64_t from = chunk * kChunk, next = from + kChunk;
        const uint32_t run = keys[next - 1].id;
        if (run >= vocab || keys[next].id != run) continue;
        const bool front = keys[from].id == run;
        if (front && from > 0 && keys[from - 1].id == run) continue;       // it began earlier
        const int64_t col = static_cast<int64_t>(u - chunk * slices) * 32 + lane;
        if (col >= lumps) continue;
        float sum[N];
#pragma unroll
        for (int e = 0; e < N; ++e) sum[e] = partial[(chunk * 2 + (front ? 0 : 1)) * partial_cols + col * N + e];
        for (int64_t c = chunk + 1; c < chunks && keys[c * kChunk].id == run; ++c) {
#pragma unroll
            for (int e = 0; e < N; ++e) sum[e] += partial[(c * 2) * partial_cols + col * N + e];
        }
        put_row<T, N>(out, run * out_stride + col * N, sum, scale, accumulate);
    }
}

inline int64_t div_up(int64_t x, int64_t by) { return (x + by - 1) / by; }
inline int64_t round_up(int64_t x, int64_t to) { return div_up(x, to) * to; }
inline int element(int type) { return type == kF32 ? 4 : 2; }

// Rows whose beginnings and widths are whole multiples of 16 bytes.
bool wide_rows(const Matrix& m) {
    const int size = element(m.type);
    return reinterpret_cast<uintptr_t>(m.data) % 16 == 0 && m.stride * size % 16 == 0 && m.cols * size % 16 == 0;
}

template <typename T, int N>
const char* embed_typed(const Ids& ids, int64_t n, const Matrix& table, float scale, const Matrix& out, cudaStream_t stream) {
    const int lumps = static_cast<int>(table.cols / N);
    int x = 32;
    while (x < 256 && x * 4 < lumps) x *= 2;
    const dim3 block(x, 256 / x);
    const int64_t blocks = div_up(n, block.y);
    embed_kernel<T, N><<<static_cast<unsigned>(std::min<int64_t>(blocks, 1 << 20)), block, 0, stream>>>(ids.data, ids.bits, n, static_cast<const T*>(table.data), table.rows,
                                                                                                   table.stride, lumps, scale,
                                                                                                   static_cast<T*>(const_cast<void*>(out.data)), out.stride);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? nullptr : cudaGetErrorString(e);
}

struct GradPlan {
    int64_t tiles, chunks;
    uint64_t seen, counts, a, b, partial, bytes;
    int passes;
};
GradPlan grad_plan(int64_t n, int64_t vocab, int64_t width) {
    GradPlan p;
    p.tiles = div_up(n, kSortTile);
    p.chunks = div_up(n, kChunk);
    p.passes = 1;
    while (p.passes * kDigit < 32 && (vocab >> (p.passes * kDigit))) ++p.passes;
    uint64_t at = 0;
    auto take = [&](uint64_t bytes) {
        const uint64_t from = at;
        at += round_up(bytes, 256);
        return from;
    };
    p.seen = take(div_up(vocab, 32) * 4);
    p.counts = take(p.tiles * kBins * 4);
    p.a = take(n * sizeof(Key));
    p.b = take(n * sizeof(Key));
    p.partial = take(static_cast<uint64_t>(p.chunks) * 2 * round_up(width, 8) * 4);
    p.bytes = at;
    return p;
}

template <typename T, int N>
void sum_typed(const Key* keys, int64_t n, const Matrix& grad, float scale, const Matrix& out, bool accumulate, float* partial, const uint32_t* seen, const GradPlan& p,
               cudaStream_t stream) {
    const int lumps = static_cast<int>(grad.cols / N), slices = static_cast<int>(div_up(lumps, 32));
    const int64_t cols = round_up(grad.cols, 8);
    T* to = static_cast<T*>(const_cast<void*>(out.data));
    const int64_t units = std::max(p.chunks * slices, accumulate ? 0 : out.rows);
    const unsigned blocks = static_cast<unsigned>(std::max<int64_t>(1, std::min<int64_t>(div_up(units, 8), 148 * 8)));
    sum_kernel<T, N><<<blocks, 256, 0, stream>>>(keys, n, static_cast<uint32_t>(out.rows), static_cast<const T*>(grad.data), grad.stride, lumps, scale, to, out.stride,
                                                 accumulate, partial, cols, slices, seen);
    if (p.chunks > 1)
        join_runs_kernel<T, N><<<static_cast<unsigned>(std::min<int64_t>(div_up(p.chunks * slices, 8), 148 * 8)), 256, 0, stream>>>(
            keys, n, static_cast<uint32_t>(out.rows), lumps, scale, to, out.stride, accumulate, partial, cols, slices);
}

}  // namespace

const char* embed(const Ids& ids, int64_t n, const Matrix& table, float scale, const Matrix& out, cudaStream_t stream) {
    if (n == 0) return nullptr;
    const bool wide = wide_rows(table) && wide_rows(out);
    switch (table.type) {
        case kF32: return wide ? embed_typed<float, 4>(ids, n, table, scale, out, stream) : embed_typed<float, 1>(ids, n, table, scale, out, stream);
        case kBF16: return wide ? embed_typed<__nv_bfloat16, 8>(ids, n, table, scale, out, stream) : embed_typed<__nv_bfloat16, 1>(ids, n, table, scale, out, stream);
        default: return wide ? embed_typed<__half, 8>(ids, n, table, scale, out, stream) : embed_typed<__half, 1>(ids, n, table, scale, out, stream);
    }
}

uint64_t embed_grad_workspace(int64_t n, int64_t vocab, int64_t width) { return grad_plan(n, vocab, width).bytes; }

const char* embed_grad(const Ids& ids, int64_t n, const Matrix& grad, float scale, const Matrix& out, bool accumulate, void* workspace, uint64_t workspace_bytes,
                       cudaStream_t stream) {
    const GradPlan p = grad_plan(n, out.rows, out.cols);
    if (workspace_bytes < p.bytes) return "the workspace is too small";
    char* at = static_cast<char*>(workspace);
    uint32_t* seen = reinterpret_cast<uint32_t*>(at + p.seen);
    uint32_t* counts = reinterpret_cast<uint32_t*>(at + p.counts);
    Key *from = reinterpret_cast<Key*>(at + p.a), *to = reinterpret_cast<Key*>(at + p.b);
    float* partial = reinterpret_cast<float*>(at + p.partial);
    const uint32_t vocab = static_cast<uint32_t>(out.rows);
    cudaMemsetAsync(seen, 0, div_up(out.rows, 32) * 4, stream);
    if (n) {
        const unsigned tiles = static_cast<unsigned>(p.tiles);
        count_kernel<true><<<tiles, kSortThreads, 0, stream>>>(ids.data, ids.bits, nullptr, n, vocab, 0, counts, seen);
        scatter_kernel<true><<<tiles, kSortThreads, 0, stream>>>(ids.data, ids.bits, nullptr, n, vocab, 0, counts, from);
        for (int pass = 1; pass < p.passes; ++pass) {
            count_kernel<false><<<tiles, kSortThreads, 0, stream>>>(nullptr, 0, from, n, vocab, pass * kDigit, counts, nullptr);
            scatter_kernel<false><<<tiles, kSortThreads, 0, stream>>>(nullptr, 0, from, n, vocab, pass * kDigit, counts, to);
            std::swap(from, to);
        }
    }
    const bool wide = wide_rows(grad) && wide_rows(out);
    switch (out.type) {
        case kF32:
            wide ? sum_typed<float, 4>(from, n, grad, scale, out, accumulate, partial, seen, p, stream) : sum_typed<float, 1>(from, n, grad, scale, out, accumulate, partial, seen, p, stream);
            break;
        case kBF16:
            wide ? sum_typed<__nv_bfloat16, 8>(from, n, grad, scale, out, accumulate, partial, seen, p, stream)
                 : sum_typed<__nv_bfloat16, 1>(from, n, grad, scale, out, accumulate, partial, seen, p, stream);
            break;
        default:
            wide ? sum_typed<__half, 8>(from, n, grad, scale, out, accumulate, partial, seen, p, stream)
                 : sum_typed<__half, 1>(from, n, grad, scale, out, accumulate, partial, seen, p, stream);
    }
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? nullptr : cudaGetErrorString(e);
}

const char* next_targets(const int32_t* ids, int64_t n, const int32_t* offsets, int64_t n_docs, const uint8_t* loss_mask, int32_t ignore, int32_t* out,
                         cudaStream_t stream) {
    if (n == 0) return nullptr;
    next_kernel<<<static_cast<unsigned>(div_up(n, 256)), 256, 0, stream>>>(ids, n, offsets, n_docs, loss_mask, ignore, out);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? nullptr : cudaGetErrorString(e);
}

}  // namespace gtok
