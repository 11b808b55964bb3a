// Rows of a table by token id: the embedding lookup, its gradient, and the ids that follow in packed documents.
#include "vocab_launch.cuh"
#include "vocab_ops.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

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

// A lump as it is loaded and stored; its elements unpacked only where they are added (kept apart, eight take twice the registers).
template <typename T, int N> struct RawOf { using type = T; };
template <> struct RawOf<float, 4> { using type = uint4; };
template <> struct RawOf<__nv_bfloat16, 8> { using type = uint4; };
template <> struct RawOf<__half, 8> { using type = uint4; };
template <typename T, int N>
__device__ __forceinline__ void unpack(float (&f)[N], const typename RawOf<T, N>::type& raw) {
    if constexpr (N == 8) {
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (std::is_same_v<T, __half>) {
                const float2 p = __half22float2(reinterpret_cast<const __half2&>(w[i]));
                f[2 * i] = p.x; f[2 * i + 1] = p.y;
            } else {              // bf16 is the upper half of fp32
                f[2 * i] = __uint_as_float(w[i] << 16); f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
            }
        }
    } else if constexpr (N == 4) {
        f[0] = __uint_as_float(raw.x); f[1] = __uint_as_float(raw.y); f[2] = __uint_as_float(raw.z); f[3] = __uint_as_float(raw.w);
    } else {
        f[0] = to_float<T>(raw);
    }
}
template <typename T, int N>
__device__ __forceinline__ typename RawOf<T, N>::type pack(const float (&f)[N]) {
    if constexpr (N == 8) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (std::is_same_v<T, __half>) {
                const __half2 p = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
                w[i] = reinterpret_cast<const uint32_t&>(p);
            } else {
                const __nv_bfloat162 p = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
                w[i] = reinterpret_cast<const uint32_t&>(p);
            }
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    } else if constexpr (N == 4) {
        return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
    } else {
        return from_float<T>(f[0]);
    }
}
// ---- lookup ---------------------------------------------------------------------
// out[t, :] = scale * table[id_t, :]; a negative id gives a row of zeros, an id beyond the table a row of NaN.  Bound by memory.  The output is
// cut into lumps whatever its width, so that no lane idles at any; each thread has four of them, 256 apart, under way at once, and writes past
// the caches, which are better used for rows that are asked for again.  32,749 rows of 2560 bf16: 44 us, 7.6 TB/s of rows in and out, as
// repeated ids are read from L2 (a row a warp 41 to 47 in the same place; eight lumps 43).  47 rows of 4096: 4 us, all latency.
template <typename Raw>
__device__ __forceinline__ void write_past(Raw* to, const Raw& v) {
    if constexpr (sizeof(Raw) == 16) __stcs(to, v);
    else *to = v;
}

template <typename T, int N>
__global__ void __launch_bounds__(256) embed_kernel(const void* ids, int bits, int64_t n, const T* table, int64_t vocab, int64_t stride, uint32_t lumps, float scale, T* out,
                                                    int64_t out_stride) {
    using Raw = typename RawOf<T, N>::type;
    constexpr int kEach = 4;
    after_previous();
    let_next_begin();
    const int64_t blocks = (n * lumps + 256 * kEach - 1) / (256 * kEach);
    for (int64_t block = blockIdx.x; block < blocks; block += gridDim.x) {
        const int64_t t0 = block * (256 * kEach) / lumps;
        const uint32_t first = static_cast<uint32_t>(block * (256 * kEach) - t0 * lumps) + threadIdx.x;
        int64_t t[kEach], id[kEach];
        uint32_t col[kEach];
        Raw v[kEach];
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
            const uint32_t down = (first + 256 * k) / lumps;
            col[k] = first + 256 * k - down * lumps;
            t[k] = t0 + down;
            id[k] = t[k] < n ? load_id(ids, bits, t[k]) : -1;
        }
#pragma unroll
        for (int k = 0; k < kEach; ++k)
            if (id[k] >= 0 && id[k] < vocab) v[k] = reinterpret_cast<const Raw*>(table + id[k] * stride)[col[k]];
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
            if (t[k] >= n) continue;
            float f[N];
            if (id[k] >= 0 && id[k] < vocab) {
                unpack<T, N>(f, v[k]);
#pragma unroll
                for (int e = 0; e < N; ++e) f[e] *= scale;
            } else {
#pragma unroll
                for (int e = 0; e < N; ++e) f[e] = id[k] < 0 ? 0.f : __int_as_float(0x7FC00000);
            }
            write_past(reinterpret_cast<Raw*>(out + t[k] * out_stride) + col[k], pack<T, N>(f));
        }
    }
}

// ---- the ids that follow ----------------------------------------------------------
// A thread an id; the document is found by halving, a dozen cached reads.  A launch and two round trips to memory: 3 us for 8,192 ids.
__global__ void next_kernel(const int32_t* ids, int64_t n, const int32_t* offsets, int64_t n_docs, const uint8_t* loss_mask, int32_t ignore, int32_t* out) {
    after_previous();
    let_next_begin();
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
// the sorted places are therefore cut into chunks of 32 (8, where that makes too few warps) whatever they hold, and runs across chunks are
// joined from fp32 partial sums.
//
// Most of the gradient's bytes are rows that no id asks for.  The sort is a few short launches that leave memory idle: further blocks of
// the same launches write these zeros meanwhile (the first two, before it is known which rows are asked for, all of a share).
//
// Bound by memory: 16,384 ids of 4096 bf16 onto 128,256 rows (1.05 GB written, 0.13 GB read) take 218 us, of which the sort's four launches are
// 95 with their share of the zeros; 184 at the rate of a copy.  2,047 ids of 768 fp32 onto 50,256 rows: 34 us against 25.
constexpr int kDigit = 9, kBins = 1 << kDigit;
constexpr int kSortThreads = kBins, kSortEach = 4, kSortTile = kSortThreads * kSortEach, kSortWarps = kSortThreads / 32;
constexpr int kChunk = 32, kShortChunk = 8;

struct Key { uint32_t id, place; };

struct SortArgs {
    const void* ids;
    int bits;
    int64_t n;
    uint32_t vocab;
    int tiles, shift, passes;
    const Key* in;
    Key* out;
    uint32_t *counts, *seen;       // seen: a bit for each row that an id asks for
    // rows that a launch's further blocks clear where no id asks for them
    char* rows;
    int64_t row_bytes, row_stride;
    int64_t from, to;
    int unit;                      // bytes written together: 16, or an element
};

// Ids outside the table sort behind it.
__device__ __forceinline__ uint32_t key_of(const SortArgs& a, int64_t i) {
    const int64_t id = load_id(a.ids, a.bits, i);
    return id >= 0 && id < a.vocab ? static_cast<uint32_t>(id) : a.vocab;
}

template <typename U>
__device__ __forceinline__ void clear_row(char* row, int64_t bytes, int lane) {
    U zero;
    memset(&zero, 0, sizeof(U));
    for (int64_t i = lane; i < bytes / static_cast<int64_t>(sizeof(U)); i += 32) reinterpret_cast<U*>(row)[i] = zero;
}
// Warp `self` of `warps` clears its share of the rows [a.from, a.to).  `seen` begins at the bit of row `first`; without it, all of them.
__device__ __forceinline__ void clear_rows(const SortArgs& a, const uint32_t* seen, int64_t first, int64_t from, int64_t to, int64_t self, int64_t warps) {
    const int lane = threadIdx.x & 31;
    for (int64_t r = from + self; r < to; r += warps) {
        const int64_t bit = r - first;
        if (seen && (seen[bit >> 5] >> (bit & 31) & 1)) continue;
        char* row = a.rows + r * a.row_stride;
        if (a.unit == 16) clear_row<uint4>(row, a.row_bytes, lane);
        else if (a.unit == 4) clear_row<uint32_t>(row, a.row_bytes, lane);
        else clear_row<uint16_t>(row, a.row_bytes, lane);
    }
}
__device__ __forceinline__ void clear_share(const SortArgs& a, bool all) {
    clear_rows(a, all ? nullptr : a.seen, 0, a.from, a.to, static_cast<int64_t>(blockIdx.x - a.tiles) * kSortWarps + (threadIdx.x >> 5),
               static_cast<int64_t>(gridDim.x - a.tiles) * kSortWarps);
}

template <bool FIRST>
__global__ void __launch_bounds__(kSortThreads) count_kernel(const __grid_constant__ SortArgs a) {
    __shared__ uint32_t bin[kBins];
    after_previous();
    let_next_begin();
    if (static_cast<int>(blockIdx.x) >= a.tiles) {
        if (FIRST) {
            const int64_t threads = static_cast<int64_t>(gridDim.x - a.tiles) * kSortThreads;
            for (int64_t i = static_cast<int64_t>(blockIdx.x - a.tiles) * kSortThreads + threadIdx.x; i < (a.vocab + 31) / 32; i += threads) a.seen[i] = 0;
        }
        return clear_share(a, FIRST);
    }
    for (int b = threadIdx.x; b < kBins; b += kSortThreads) bin[b] = 0;
    __syncthreads();
    const int64_t from = static_cast<int64_t>(blockIdx.x) * kSortTile;
    uint32_t key[kSortEach];
#pragma unroll
    for (int i = 0; i < kSortEach; ++i) {
        const int64_t at = from + i * kSortThreads + threadIdx.x;
        if (at < a.n) key[i] = FIRST ? key_of(a, at) : a.in[at].id;
    }
#pragma unroll
    for (int i = 0; i < kSortEach; ++i) {
        if (from + i * kSortThreads + threadIdx.x >= a.n) continue;
        atomicAdd(&bin[key[i] >> a.shift & (kBins - 1)], 1u);
    }
    __syncthreads();
    for (int b = threadIdx.x; b < kBins; b += kSortThreads) a.counts[static_cast<int64_t>(blockIdx.x) * kBins + b] = bin[b];
}

// Many tiles: their counts of each bin become sums over the tiles before, and a row behind them the totals.  32 bins a block.
constexpr int kFewTiles = 32;           // up to here each tile adds them up by itself: 32 tiles in all 47 us, with this launch 49; 64 tiles 65 and 64, 128 tiles 110 and 84
__global__ void __launch_bounds__(1024) prefix_kernel(uint32_t* counts, int64_t tiles) {
    constexpr int kEach = 8;
    __shared__ uint32_t sums[32][33];
    after_previous();
    let_next_begin();
    const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
    uint32_t* column = counts + blockIdx.x * 32 + x;
    uint32_t done = 0;
    for (int64_t base = 0; base < tiles; base += 32 * kEach) {
        uint32_t c[kEach], mine = 0;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int64_t t = base + y * kEach + i;
            c[i] = t < tiles ? column[t * kBins] : 0;
        }
#pragma unroll
        for (int i = 0; i < kEach; ++i) mine += c[i];
        __syncthreads();
        sums[y][x] = mine;
        __syncthreads();
        uint32_t before = done;
        for (int r = 0; r < 32; ++r) {
            const uint32_t v = sums[r][x];
            if (r < y) before += v;
            done += v;
        }
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int64_t t = base + y * kEach + i;
            if (t < tiles) column[t * kBins] = before;
            before += c[i];
        }
    }
    if (y == 0) column[tiles * kBins] = done;
}

struct SortSpace {
    uint32_t base[kBins];
    uint16_t warp_bin[kSortWarps][kBins];
    uint32_t warp_sum[kSortWarps];
};

// Places of a tile's keys (128 a warp, in order) after one digit: `key` to s.base[bin] + s.warp_bin[warp][bin] + rank.  `all` and `before`: keys of this
// thread's bin in all tiles and in those before; with `alone` the tile is all there is.
__device__ __forceinline__ void rank_keys(SortSpace& s, const Key (&key)[kSortEach], const bool (&here)[kSortEach], uint16_t (&rank)[kSortEach], int shift,
                                          bool alone, uint32_t all, uint32_t before) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kSortWarps; ++w) s.warp_bin[w][tid] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kSortEach; ++i) {
        const uint32_t b = here[i] ? key[i].id >> shift & (kBins - 1) : kBins;
        const uint32_t same = __match_any_sync(~0u, b);
        const uint16_t seen = here[i] ? s.warp_bin[warp][b] : 0;
        __syncwarp();
        rank[i] = seen + __popc(same & ((1u << lane) - 1));
        if (here[i] && (same & ((1u << lane) - 1)) == 0) s.warp_bin[warp][b] = seen + __popc(same);
        __syncwarp();
    }
    __syncthreads();
    uint32_t total = 0;
#pragma unroll
    for (int w = 0; w < kSortWarps; ++w) {
        const uint32_t c = s.warp_bin[w][tid];
        s.warp_bin[w][tid] = static_cast<uint16_t>(total);
        total += c;
    }
    if (alone) all = total;
    uint32_t scan = all;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const uint32_t y = __shfl_up_sync(~0u, scan, d);
        if (lane >= d) scan += y;
    }
    if (lane == 31) s.warp_sum[warp] = scan;
    __syncthreads();
    uint32_t low = lane < warp ? s.warp_sum[lane] : 0;          // kSortWarps are no more than the lanes
#pragma unroll
    for (int d = 16; d; d >>= 1) low += __shfl_xor_sync(~0u, low, d);
    s.base[tid] = low + scan - all + before;
    __syncthreads();
}

template <bool FIRST>
__global__ void __launch_bounds__(kSortThreads) scatter_kernel(const __grid_constant__ SortArgs a) {
    __shared__ SortSpace s;
    after_previous();
    let_next_begin();
    if (static_cast<int>(blockIdx.x) >= a.tiles) return clear_share(a, FIRST);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t from = static_cast<int64_t>(blockIdx.x) * kSortTile + warp * 32 * kSortEach;
    Key key[kSortEach];
    bool here[kSortEach];
    uint16_t rank[kSortEach];
#pragma unroll
    for (int i = 0; i < kSortEach; ++i) {
        const int64_t at = from + i * 32 + lane;
        here[i] = at < a.n;
        key[i] = here[i] ? (FIRST ? Key{key_of(a, at), static_cast<uint32_t>(at)} : a.in[at]) : Key{0xFFFFFFFFu, 0};
    }
    // how many keys of this thread's bin there are: in all tiles, and in those before this one
    uint32_t all = 0, before = 0;
    if (a.tiles > kFewTiles) {
        before = a.counts[static_cast<int64_t>(blockIdx.x) * kBins + tid];
        all = a.counts[static_cast<int64_t>(a.tiles) * kBins + tid];
    }
    for (int t = 0; t < a.tiles && a.tiles <= kFewTiles; t += 8) {
        uint32_t c[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) c[k] = t + k < a.tiles ? a.counts[static_cast<int64_t>(t + k) * kBins + tid] : 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            if (t + k < static_cast<int>(blockIdx.x)) before += c[k];
            all += c[k];
        }
    }
    rank_keys(s, key, here, rank, a.shift, false, all, before);
#pragma unroll
    for (int i = 0; i < kSortEach; ++i) {
        if (!here[i]) continue;
        const uint32_t b = key[i].id >> a.shift & (kBins - 1);
        if (FIRST && key[i].id < a.vocab) atomicOr(&a.seen[key[i].id >> 5], 1u << (key[i].id & 31));
        a.out[s.base[b] + s.warp_bin[warp][b] + rank[i]] = key[i];
    }
}

// All of the sort where the ids make one tile: block 0 sorts, digit after digit, the others clear a share of the rows.  Each of those finds
// out for itself which of its rows are asked for.
constexpr int kOwnRows = 4096;          // rows whose bits a block has room for
__global__ void __launch_bounds__(kSortThreads) one_tile_kernel(const __grid_constant__ SortArgs a) {
    __shared__ union {
        struct { SortSpace space; Key key[kSortTile]; } sort;
        uint32_t seen[kOwnRows / 32];
    } s;
    after_previous();
    let_next_begin();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (blockIdx.x > 0) {
        const int64_t blocks = gridDim.x - 1, self = blockIdx.x - 1;
        const int64_t share = min((a.to - a.from + blocks - 1) / blocks, static_cast<int64_t>(kOwnRows));
        for (int64_t from = a.from + self * share; from < a.to; from += blocks * share) {
            const int64_t to = min(from + share, a.to);
            __syncthreads();
            for (int i = tid; i < kOwnRows / 32; i += kSortThreads) s.seen[i] = 0;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < kSortEach; ++i) {
                const int at = i * kSortThreads + tid;
                if (at >= a.n) continue;
                const int64_t id = key_of(a, at);
                if (id >= from && id < to) atomicOr(&s.seen[(id - from) >> 5], 1u << ((id - from) & 31));
            }
            __syncthreads();
            clear_rows(a, s.seen, from, from, to, warp, kSortWarps);
        }
        return;
    }
    for (int64_t i = tid; i < (a.vocab + 31) / 32; i += kSortThreads) a.seen[i] = 0;
    Key key[kSortEach];
    bool here[kSortEach];
    uint16_t rank[kSortEach];
#pragma unroll
    for (int i = 0; i < kSortEach; ++i) {
        const int at = warp * 32 * kSortEach + i * 32 + lane;
        here[i] = at < a.n;
        key[i] = here[i] ? Key{key_of(a, at), static_cast<uint32_t>(at)} : Key{0xFFFFFFFFu, 0};
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kSortEach; ++i)
        if (here[i] && key[i].id < a.vocab) atomicOr(&a.seen[key[i].id >> 5], 1u << (key[i].id & 31));
    for (int pass = 0; pass < a.passes; ++pass) {
        rank_keys(s.sort.space, key, here, rank, pass * kDigit, true, 0, 0);
        Key* to = pass + 1 < a.passes ? s.sort.key : a.out;
#pragma unroll
        for (int i = 0; i < kSortEach; ++i) {
            if (!here[i]) continue;
            const uint32_t b = key[i].id >> (pass * kDigit) & (kBins - 1);
            to[s.sort.space.base[b] + s.sort.space.warp_bin[warp][b] + rank[i]] = key[i];
        }
        if (pass + 1 == a.passes) break;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kSortEach; ++i)
            if (here[i]) key[i] = s.sort.key[warp * 32 * kSortEach + i * 32 + lane];
    }
}

template <typename T, int N>
__device__ __forceinline__ void put_row(T* out, int64_t at, const float (&sum)[N], float scale, bool accumulate) {
    using Raw = typename RawOf<T, N>::type;
    Raw* to = reinterpret_cast<Raw*>(out + at);
    float v[N];
    if (accumulate) {
        unpack<T, N>(v, *to);
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] += scale * sum[e];
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = scale * sum[e];
    }
    *to = pack<T, N>(v);
}

// Sums of the runs in a chunk, one warp a chunk and 32 lumps of columns; then a share of the rows to be cleared.  Sums are in fp32, one
// rounding at the end of a run.
constexpr int kFlight = 4;      // (8: more registers, fewer warps, slower by a tenth)
template <typename T, int N>
__global__ void __launch_bounds__(256, 3) sum_kernel(const Key* keys, int64_t n, uint32_t vocab, const T* grad, int64_t stride, int lumps, float scale, T* out,
                                                  int64_t out_stride, bool accumulate, float* partial, int64_t partial_cols, int slices,
                                                  int in_chunk, const __grid_constant__ SortArgs sort) {
    after_previous();
    let_next_begin();
    using Raw = typename RawOf<T, N>::type;
    const int lane = threadIdx.x & 31;
    const int64_t warps = static_cast<int64_t>(gridDim.x) * (blockDim.x / 32), self = static_cast<int64_t>(blockIdx.x) * (blockDim.x / 32) + (threadIdx.x >> 5);
    const int64_t chunks = (n + in_chunk - 1) / in_chunk;
    for (int64_t u = self; u < chunks * slices; u += warps) {
        const int64_t chunk = u / slices;
        const int col = (static_cast<int>(u - chunk * slices) * 32 + lane);
        const bool here = col < lumps;
        const int64_t from = chunk * in_chunk;
        const int count = static_cast<int>(min(static_cast<int64_t>(in_chunk), n - from));
        const Key mine = lane < count ? keys[from + lane] : Key{0xFFFFFFFFu, 0};
        const uint32_t before = from > 0 ? keys[from - 1].id : 0xFFFFFFFEu, after = from + count < n ? keys[from + count].id : 0xFFFFFFFEu;
        float sum[N];
#pragma unroll
        for (int e = 0; e < N; ++e) sum[e] = 0.f;
        uint32_t run = __shfl_sync(~0u, mine.id, 0);
        bool open = run == before;                 // the run began in an earlier chunk
        int slot = 0;                              // of its part; 1 behind the first run
        auto put = [&](bool to_partial) {
            if (!here || run >= vocab) return;
            if (to_partial) {
                float* to = partial + (chunk * 2 + slot) * partial_cols + static_cast<int64_t>(col) * N;
#pragma unroll
                for (int e = 0; e < N; ++e) to[e] = sum[e];
            } else {
                put_row<T, N>(out, run * out_stride + static_cast<int64_t>(col) * N, sum, scale, accumulate);
            }
        };
        for (int i = 0; i < count; i += kFlight) {
            Raw v[kFlight];
#pragma unroll
            for (int k = 0; k < kFlight; ++k) {
                const uint32_t id = __shfl_sync(~0u, mine.id, (i + k) & 31), place = __shfl_sync(~0u, mine.place, (i + k) & 31);
                if (here && i + k < count && id < vocab) {
                    v[k] = reinterpret_cast<const Raw*>(grad + static_cast<int64_t>(place) * stride)[col];
                    // what a run's sum will be added to comes nearer meanwhile
                    if (accumulate) asm volatile("prefetch.global.L2 [%0];" ::"l"(out + id * out_stride + static_cast<int64_t>(col) * N));
                }
            }
#pragma unroll
            for (int k = 0; k < kFlight; ++k) {
                if (i + k >= count) break;
                const uint32_t id = __shfl_sync(~0u, mine.id, i + k);
                if (id != run) {
                    put(open);
#pragma unroll
                    for (int e = 0; e < N; ++e) sum[e] = 0.f;
                    run = id;
                    open = false;
                    slot = 1;
                }
                if (here && id < vocab) {
                    float f[N];
                    unpack<T, N>(f, v[k]);
#pragma unroll
                    for (int e = 0; e < N; ++e) sum[e] += f[e];
                }
            }
        }
        put(open || run == after);
    }
    clear_rows(sort, sort.seen, 0, sort.from, sort.to, self, warps);
}

// Runs across chunks: the warp of the chunk where one begins adds its parts up, in order.
template <typename T, int N>
__global__ void __launch_bounds__(256) join_runs_kernel(const Key* keys, int64_t n, uint32_t vocab, int lumps, float scale, T* out, int64_t out_stride, bool accumulate,
                                                        const float* partial, int64_t partial_cols, int slices, int in_chunk,
                                                        const __grid_constant__ SortArgs sort) {
    using F = Lump<float, N>;
    after_previous();
    let_next_begin();
    const int lane = threadIdx.x & 31;
    const int64_t warps = static_cast<int64_t>(gridDim.x) * (blockDim.x / 32), self = static_cast<int64_t>(blockIdx.x) * (blockDim.x / 32) + (threadIdx.x >> 5);
    const int64_t chunks = (n + in_chunk - 1) / in_chunk;
    for (int64_t u = self; u < (chunks - 1) * slices; u += warps) {
        const int64_t chunk = u / slices;
        const int64_t from = chunk * in_chunk, next = from + in_chunk;
        const uint32_t run = keys[next - 1].id, behind = keys[next].id, head = keys[from].id, before = from > 0 ? keys[from - 1].id : 0xFFFFFFFEu;
        if (run >= vocab || behind != run) continue;
        const bool front = head == run;
        if (front && before == run) continue;       // it began earlier
        const int64_t col = static_cast<int64_t>(u - chunk * slices) * 32 + lane;
        const bool here = col < lumps;
        F sum{};
        if (here) sum = *reinterpret_cast<const F*>(partial + (chunk * 2 + (front ? 0 : 1)) * partial_cols + col * N);
        // 32 chunks further on at a time: how many of them the run reaches, then their parts with several loads under way
        for (int64_t c = chunk + 1;; c += 32) {
            const uint32_t begins = c + lane < chunks ? keys[(c + lane) * in_chunk].id : 0xFFFFFFFEu;
            const uint32_t other = __ballot_sync(~0u, begins != run);
            const int count = other ? __ffs(other) - 1 : 32;
            for (int i = 0; i < count; i += 8) {
                F v[8];
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    if (here && i + k < count) v[k] = *reinterpret_cast<const F*>(partial + (c + i + k) * 2 * partial_cols + col * N);
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    if (!here || i + k >= count) break;
#pragma unroll
                    for (int e = 0; e < N; ++e) sum.v[e] += v[k].v[e];
                }
            }
            if (other) break;
        }
        if (here) put_row<T, N>(out, run * out_stride + col * N, sum.v, scale, accumulate);
    }
    clear_rows(sort, sort.seen, 0, sort.from, sort.to, self, warps);
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
    const int64_t lumps = table.cols / N;
    const cudaError_t e = launch(embed_kernel<T, N>, std::min<int64_t>(div_up(n * lumps, 1024), 1 << 30), 256, 0, stream, ids.data, ids.bits, n,
                                 static_cast<const T*>(table.data), table.rows, table.stride, static_cast<uint32_t>(lumps), scale,
                                 static_cast<T*>(const_cast<void*>(out.data)), out.stride);
    return e == cudaSuccess ? nullptr : cudaGetErrorString(e);
}

struct GradPlan {
    int64_t tiles, chunks;
    int in_chunk;
    uint64_t seen, counts, a, b, partial, bytes;
    int passes;
};
GradPlan grad_plan(int64_t n, int64_t vocab, int64_t width) {
    GradPlan p;
    p.tiles = div_up(n, kSortTile);
    // Short chunks where long ones would leave the GPU with less than 32 warps an SM (256: a warp's columns of 16 bits): sums of 2,047 rows of 768
    // 14 -> 7 us; in large calls their partial sums would be memory traffic for nothing.
    p.in_chunk = div_up(n, kChunk) * div_up(width, 256) < 148 * 32 ? kShortChunk : kChunk;
    p.chunks = div_up(n, p.in_chunk);
    p.passes = 1;
    while (p.passes * kDigit < 32 && (vocab >> (p.passes * kDigit))) ++p.passes;
    uint64_t at = 0;
    auto take = [&](uint64_t bytes) {
        const uint64_t from = at;
        at += round_up(bytes, 256);
        return from;
    };
    p.seen = take(div_up(vocab, 32) * 4);
    p.counts = take((p.tiles + 1) * kBins * 4);
    p.a = take(n * sizeof(Key));
    p.b = take(n * sizeof(Key));
    p.partial = take(static_cast<uint64_t>(p.chunks) * 2 * round_up(width, 8) * 4);
    p.bytes = at;
    return p;
}

template <typename T, int N>
cudaError_t sum_typed(const Key* keys, int64_t n, const Matrix& grad, float scale, const Matrix& out, bool accumulate, float* partial, SortArgs sort, const GradPlan& p,
                      int64_t rows_at_once, int64_t all, cudaStream_t stream) {
    const int lumps = static_cast<int>(grad.cols / N), slices = static_cast<int>(div_up(lumps, 32));
    const int64_t cols = round_up(grad.cols, 8);
    T* to = static_cast<T*>(const_cast<void*>(out.data));
    const uint32_t vocab = static_cast<uint32_t>(out.rows);
    auto blocks = [&](int64_t sums) { return std::min<int64_t>(div_up(std::max<int64_t>(1, std::max(sums, sort.to - sort.from)), 8), 148 * 8); };
    sort.from = sort.to;
    sort.to = p.chunks < 2 ? all : std::max(sort.from, all - rows_at_once);
    if (cudaError_t e = launch(sum_kernel<T, N>, blocks(p.chunks * slices), 256, 0, stream, keys, n, vocab, static_cast<const T*>(grad.data), grad.stride, lumps, scale, to,
                               out.stride, accumulate, partial, cols, slices, p.in_chunk, sort))
        return e;
    if (p.chunks < 2) return cudaSuccess;
    sort.from = sort.to;
    sort.to = all;
    return launch(join_runs_kernel<T, N>, blocks((p.chunks - 1) * slices), 256, 0, stream, keys, n, vocab, lumps, scale, to, out.stride, accumulate,
                  partial, cols, slices, p.in_chunk, sort);
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
    Key *keys = reinterpret_cast<Key*>(at + p.a), *other = reinterpret_cast<Key*>(at + p.b);
    float* partial = reinterpret_cast<float*>(at + p.partial);
    const bool wide = wide_rows(grad) && wide_rows(out);
    const int size = element(out.type);
    SortArgs s{};
    s.ids = ids.data;
    s.bits = ids.bits;
    s.n = n;
    s.vocab = static_cast<uint32_t>(out.rows);
    s.tiles = static_cast<int>(p.tiles);
    s.passes = p.passes;
    s.counts = reinterpret_cast<uint32_t*>(at + p.counts);
    s.seen = reinterpret_cast<uint32_t*>(at + p.seen);
    s.rows = static_cast<char*>(const_cast<void*>(out.data));
    s.row_bytes = out.cols * size;
    s.row_stride = out.stride * size;
    s.unit = wide_rows(out) ? 16 : size;
    // Rows cleared beside the other work of a launch.  Beside the sort of many tiles 140 MB: more than fits into the sort's own time, but sums and
    // clearing together go slower than either (16,384 ids of 4096 onto 128,256 rows: 239 us with 40 MB, 220 with 140, 228 with 260).  One tile is
    // sorted in the time of 80 MB.
    const int64_t rows_at_once = std::max<int64_t>(1, ((p.tiles == 1 ? 40 : 140) << 20) / s.row_bytes), all = accumulate ? 0 : out.rows;
    auto clearing = [&](int64_t blocks) {
        s.from = s.to;
        s.to = std::min(all, s.from + rows_at_once);
        return blocks + std::min<int64_t>(div_up(s.to - s.from, kSortWarps), 148 * 4);
    };
    cudaError_t e = cudaSuccess;
    if (p.tiles == 1) {
        s.out = keys;
        s.to = std::min(all, 2 * rows_at_once);
        e = launch(one_tile_kernel, 1 + std::min<int64_t>(div_up(s.to, kSortWarps), 148 * 4), kSortThreads, 0, stream, s);
    } else {
        for (int pass = 0; pass < p.passes && p.tiles && e == cudaSuccess; ++pass) {
            s.in = keys;
            s.out = pass ? other : keys;
            s.shift = pass * kDigit;
            // (one block at least to clear `seen`)
            e = launch(pass ? count_kernel<false> : count_kernel<true>, std::max(clearing(p.tiles), p.tiles + 1), kSortThreads, 0, stream, s);
            if (e == cudaSuccess && p.tiles > kFewTiles) e = launch(prefix_kernel, kBins / 32, 1024, 0, stream, s.counts, p.tiles);
            if (e != cudaSuccess) break;
            e = launch(pass ? scatter_kernel<false> : scatter_kernel<true>, clearing(p.tiles), kSortThreads, 0, stream, s);
            if (pass) std::swap(keys, other);
        }
        if (!p.tiles) e = cudaMemsetAsync(s.seen, 0, div_up(out.rows, 32) * 4, stream);
    }
    if (e != cudaSuccess) return cudaGetErrorString(e);
    switch (out.type) {
        case kF32:
            e = (wide ? sum_typed<float, 4> : sum_typed<float, 1>)(keys, n, grad, scale, out, accumulate, partial, s, p, rows_at_once, all, stream);
            break;
        case kBF16:
            e = (wide ? sum_typed<__nv_bfloat16, 8> : sum_typed<__nv_bfloat16, 1>)(keys, n, grad, scale, out, accumulate, partial, s, p, rows_at_once, all, stream);
            break;
        default:
            e = (wide ? sum_typed<__half, 8> : sum_typed<__half, 1>)(keys, n, grad, scale, out, accumulate, partial, s, p, rows_at_once, all, stream);
    }
    return e == cudaSuccess ? nullptr : cudaGetErrorString(e);
}

const char* next_targets(const int32_t* ids, int64_t n, const int32_t* offsets, int64_t n_docs, const uint8_t* loss_mask, int32_t ignore, int32_t* out,
                         cudaStream_t stream) {
    if (n == 0) return nullptr;
    const cudaError_t e = launch(next_kernel, div_up(n, 256), 256, 0, stream, ids, n, offsets, n_docs, loss_mask, ignore, out);
    return e == cudaSuccess ? nullptr : cudaGetErrorString(e);
}

}  // namespace gtok
