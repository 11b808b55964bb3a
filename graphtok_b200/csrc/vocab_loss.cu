// Losses over a vocabulary from hidden states H [n, width] and an output table W [vocab, width], and their gradients, without ever
// holding the logits Z = H W^T as a whole.
//
//   loss_i = lse(z_i) - z_i[target_i]                                         (cross entropy)
//   loss_i = sum_k q_ik (log q_ik - z_i[t_ik] / T + lse(z_i / T))             (distillation; q = softmax of a teacher's top logits / T)
//   dZ_i   = g_i / T (softmax(z_i / T) - q_i),   dH = dZ W,   dW = dZ^T H
//
// Cross entropy is the second form with one entry of q = 1 a row, and runs as that.
//
// Forward: one matrix product whose epilogue reduces each 256 x 256 tile of Z, as it leaves the accumulators, to a running maximum and
// sum per row (and takes the entries' logits out); a small kernel joins the tiles' pairs.  Backward: per piece of the vocabulary, the
// tile of Z is computed again and becomes dZ in 16 bits, from which two more products give the piece's part of dH and its rows of dW.
// A piece's dZ is the only thing in memory that grows with n x vocab.
//
// Rows without a loss (ignored targets, no teacher entries) are left out before the products: the others are copied together, so
// neither time nor NaN of masked positions is carried along.
#include "sm100.cuh"
#include "vocab_ops.h"

#include <algorithm>
#include <climits>
#include <cmath>

namespace gtok {
namespace {

using namespace sm100;

constexpr int kTile = 256;              // rows and columns of a pair's tile
constexpr int kDepth = 64;              // elements of the summed dimension a stage holds: one 128-byte line
constexpr int kStages = 6;
constexpr int kStageBytes = 32768;      // 128 x 64 of either operand
constexpr int kEpilogueWarps = 8;
constexpr int kThreads = 128 + 32 * kEpilogueWarps;
constexpr int kStagingBytes = 4096;     // a warp's 32 lines of 128 bytes on their way out
constexpr int kSmemBytes = 1024 + kStages * kStageBytes + kEpilogueWarps * kStagingBytes + 256;
constexpr int kGroup = 16;              // row tiles that share a sweep over the vocabulary: 16 x 256 rows stay in L2

constexpr float kLog2e = 1.4426950408889634f;

// Scalars in device memory that the kernels hand to one another.
struct Shared {
    int active;          // rows with a loss
    int error;           // a wait ran out
    float row_scale;     // gradient of row i, times this, is what dZ carries of it ...
    float unscale;       // ... and the products times this are the gradients
};

enum { kForward = 0, kDelta = 1, kHiddenGrad = 2, kWeightGrad = 3 };

struct Product {
    Shared* shared;
    const int* rows;           // place of each active row
    int n_rows;                // rows of the padded arrays (a multiple of kTile)
    int vocab, width;
    int first, count;          // first column of this piece, its columns
    int entries;
    const int* entry_ids;      // [n, entries], ascending in a row, INT_MAX after the last
    const float* entry_share;  // q; NULL: 1
    float exponent;            // log2(e) / T
    float2* partial;           // forward: (maximum, sum) of [half tile of columns][row]
    float* entry_logits;       // forward: [n, entries]
    const float* lse;          // [n]
    const float* grad;
    int64_t grad_stride;
    int splits;                // hidden gradient: parts of the piece's columns that are summed apart
    bool add;                  // ... onto what earlier pieces left
    void* direct;              // weight gradient, where its rows are no lines of whole 16 bytes: written by the threads
    int64_t direct_stride;
};

struct Place { int m, n, k0, k1, split; };     // tile of the output, blocks of the summed dimension

template <int MODE>
__device__ __forceinline__ int tile_count(const Product& p, int active) {
    const int row_tiles = (active + kTile - 1) / kTile, col_tiles = (p.count + kTile - 1) / kTile, width_tiles = (p.width + kTile - 1) / kTile;
    if (MODE == kHiddenGrad) return row_tiles * width_tiles * p.splits;
    if (MODE == kWeightGrad) return active ? col_tiles * width_tiles : 0;
    return row_tiles * col_tiles;
}

template <int MODE>
__device__ __forceinline__ Place tile_place(const Product& p, int active, int t) {
    const int row_tiles = (active + kTile - 1) / kTile, col_tiles = (p.count + kTile - 1) / kTile, width_tiles = (p.width + kTile - 1) / kTile;
    Place q;
    q.k0 = 0;
    q.split = 0;
    if (MODE == kHiddenGrad) {
        const int blocks = (p.count + kDepth - 1) / kDepth;
        q.split = t / (row_tiles * width_tiles);
        t -= q.split * row_tiles * width_tiles;
        q.m = t / width_tiles;
        q.n = t - q.m * width_tiles;
        q.k0 = static_cast<int>(static_cast<int64_t>(blocks) * q.split / p.splits);
        q.k1 = static_cast<int>(static_cast<int64_t>(blocks) * (q.split + 1) / p.splits);
    } else if (MODE == kWeightGrad) {
        q.m = t / width_tiles;
        q.n = t - q.m * width_tiles;
        q.k1 = (active + kDepth - 1) / kDepth;
    } else {
        const int group = t / (kGroup * col_tiles);
        const int first = group * kGroup, rows = min(kGroup, row_tiles - first);
        t -= first * col_tiles;
        q.n = t / rows;
        q.m = first + t - q.n * rows;
        q.k1 = (p.width + kDepth - 1) / kDepth;
    }
    return q;
}

template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (BF16) {
        __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<uint32_t*>(&v);
    } else {
        __half2 v = __floats2half2_rn(a, b);
        return *reinterpret_cast<uint32_t*>(&v);
    }
}
template <bool BF16>
__device__ __forceinline__ uint16_t pack1(float a) {
    if constexpr (BF16) {
        __nv_bfloat16 v = __float2bfloat16_rn(a);
        return *reinterpret_cast<uint16_t*>(&v);
    } else {
        __half v = __float2half_rn(a);
        return *reinterpret_cast<uint16_t*>(&v);
    }
}

// A thread's way through the entries of its row, in ascending order of their ids.
struct Entries {
    int64_t at = 0, end = 0;
    int next = INT_MAX;
    __device__ __forceinline__ void begin(const Product& p, int row, int column) {
        at = static_cast<int64_t>(row) * p.entries;
        end = at + p.entries;
        int64_t lo = at, hi = end;            // first entry at or behind `column`
        while (lo < hi) {
            const int64_t mid = (lo + hi) >> 1;
            if (p.entry_ids[mid] < column) lo = mid + 1; else hi = mid;
        }
        at = lo;
        next = at < end ? p.entry_ids[at] : INT_MAX;
    }
    __device__ __forceinline__ void step(const Product& p) {
        ++at;
        next = at < end ? p.entry_ids[at] : INT_MAX;
    }
};

// A persistent product: one pair of blocks an SM pair, tiles handed out in turn.  Warp 0 of each block copies its half of the operands
// in, warp 1 of the first block issues the matrix instructions for both, eight warps of each block take the accumulators out while the
// next tile is summed into the other half of tensor memory.
template <int MODE, bool BF16>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    product_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_out,
                   const __grid_constant__ Product p) {
    constexpr bool kAcrossA = MODE == kWeightGrad, kAcrossB = MODE >= kHiddenGrad;     // operand's lines run across the summed dimension
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_addr(smem_raw) + 1023) & ~1023u;
    const uint32_t staging = base + kStages * kStageBytes;
    const uint32_t bars = staging + kEpilogueWarps * kStagingBytes;
    const uint32_t full = bars, empty = bars + 8 * kStages, acc_full = empty + 8 * kStages, acc_empty = acc_full + 16, tmem_at = acc_empty + 16;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            bar_init(full + 8 * s, 1);
            bar_init(empty + 8 * s, 1);
        }
        for (int s = 0; s < 2; ++s) {
            bar_init(acc_full + 8 * s, 1);
            bar_init(acc_empty + 8 * s, 2 * kEpilogueWarps);
        }
        bar_init_fence();
    }
    if (warp == 2) tmem_alloc(tmem_at, 512);
    __syncthreads();
    fence_before();
    cluster_sync();
    fence_after();
    uint32_t tmem;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(tmem) : "r"(tmem_at));

    const int active = p.shared->active;
    const int tiles = tile_count<MODE>(p, active);
    const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    bool ok = true;

    if (warp == 0) {
        if (elect()) {
            const uint32_t full_of_pair = in_block(full, 0);
            uint32_t it = 0;
            for (int t = pair; t < tiles && ok; t += pairs) {
                const Place q = tile_place<MODE>(p, active, t);
                const int am = q.m * kTile + rank * 128, bn = q.n * kTile + rank * 128 + ((MODE == kForward || MODE == kDelta) ? p.first : 0);
                const int bk = MODE == kHiddenGrad ? p.first : 0;
                for (int k = q.k0; k < q.k1; ++k, ++it) {
                    const uint32_t s = it % kStages;
                    if (!bar_wait(empty + 8 * s, ((it / kStages) & 1) ^ 1)) { ok = false; break; }
                    const uint32_t a = base + s * kStageBytes, b = a + kStageBytes / 2, bar = full_of_pair + 8 * s;
                    if (rank == 0) bar_expect(full + 8 * s, 2 * kStageBytes);
                    const int x = k * kDepth;
                    load_tile(a, &map_a, kAcrossA ? am : x, kAcrossA ? x : am, bar);
                    load_tile(a + 8192, &map_a, kAcrossA ? am + 64 : x, kAcrossA ? x : am + 64, bar);
                    load_tile(b, &map_b, kAcrossB ? bn : x, kAcrossB ? x + bk : bn, bar);
                    load_tile(b + 8192, &map_b, kAcrossB ? bn + 64 : x, kAcrossB ? x + bk : bn + 64, bar);
                }
            }
            if (!ok) {      // copies that are still under way land before the block may leave
                const uint64_t from = nanoseconds();
                while (nanoseconds() - from < 2000000ull) __nanosleep(1000);
            }
        }
    } else if (warp == 1) {
        if (rank == 0 && elect()) {
            constexpr uint32_t kind = mma_kind(BF16, kAcrossA, kAcrossB);
            uint32_t it = 0, acc = 0;
            for (int t = pair; t < tiles && ok; t += pairs, ++acc) {
                const Place q = tile_place<MODE>(p, active, t);
                if (!bar_wait(acc_empty + 8 * (acc & 1), ((acc >> 1) & 1) ^ 1)) { ok = false; break; }
                fence_after();
                for (int k = q.k0; k < q.k1; ++k, ++it) {
                    const uint32_t s = it % kStages;
                    if (!bar_wait(full + 8 * s, (it / kStages) & 1)) { ok = false; break; }
                    fence_after();
                    const uint32_t a = base + s * kStageBytes, b = a + kStageBytes / 2;
#pragma unroll
                    for (int j = 0; j < kDepth / 16; ++j)
                        mma(tmem + (acc & 1) * 256, operand(a + j * (kAcrossA ? 2048 : 32), kAcrossA), operand(b + j * (kAcrossB ? 2048 : 32), kAcrossB), kind,
                            k > q.k0 || j > 0);
                    mma_commit(empty + 8 * s);
                }
                if (ok) mma_commit(acc_full + 8 * (acc & 1));
            }
        }
    } else if (warp >= 4) {
        const int quarter = warp & 3, half = (warp - 4) >> 2;
        const uint32_t lines = staging + (warp - 4) * kStagingBytes;
        const uint32_t line = lines + lane * 128;
        uint32_t acc = 0;
        for (int t = pair; t < tiles; t += pairs, ++acc) {
            const Place q = tile_place<MODE>(p, active, t);
            const int m = q.m * kTile + rank * 128 + quarter * 32 + lane;       // this thread's line of the tile
            const int column = q.n * kTile + half * 128;                        // of the output; of the piece where columns are the vocabulary's
            const uint32_t from = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + (acc & 1) * 256 + half * 128;
            Entries e;
            float lse2 = 0.f, f = 0.f;
            bool live = true;
            if (MODE == kForward || MODE == kDelta) {
                live = m < active;
                if (live) {
                    const int row = p.rows[m];
                    e.begin(p, row, p.first + column);
                    if (MODE == kDelta) {
                        lse2 = p.lse[row] * kLog2e;
                        f = p.grad[row * p.grad_stride] * p.shared->row_scale;
                    }
                }
            }
            if (MODE == kWeightGrad) f = p.shared->unscale;
            ok = __all_sync(~0u, bar_wait(acc_full + 8 * (acc & 1), (acc >> 1) & 1));
            if (!ok) break;
            fence_after();
            if constexpr (MODE == kForward) {
                float high = -INFINITY, sum = 0.f;
#pragma unroll 1
                for (int c = 0; c < 128; c += 32) {
                    float v[32];
                    tmem_load(from + c, v);
                    const int at = p.first + column + c;
                    if (at + 32 > p.vocab) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) v[i] = at + i < p.vocab ? v[i] : -INFINITY;
                    }
                    float top = v[0];
#pragma unroll
                    for (int i = 1; i < 32; ++i) top = fmaxf(top, v[i]);
                    top = fmaxf(top, high);
                    const float from_top = top == -INFINITY ? 0.f : top * p.exponent;
                    sum *= exp2_fast(fmaf(high, p.exponent, -from_top));
                    high = top;
                    float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int i = 0; i < 32; ++i) part[i & 3] += exp2_fast(fmaf(v[i], p.exponent, -from_top));
                    sum += (part[0] + part[1]) + (part[2] + part[3]);
                    while (e.next < at + 32) {
                        const int j = e.next - at;
                        float z = 0.f;
#pragma unroll
                        for (int i = 0; i < 32; ++i) z = i == j ? v[i] : z;
                        p.entry_logits[e.at] = z;
                        e.step(p);
                    }
                    __syncwarp();
                }
                if (live) p.partial[static_cast<int64_t>(q.n * 2 + half) * p.n_rows + m] = make_float2(high, sum);
            } else if constexpr (MODE == kDelta || MODE == kWeightGrad) {
                // 64 columns of 16 bits make a line
#pragma unroll 1
                for (int c = 0; c < 128; c += 64) {
                    if (lane == 0) stores_read();
                    __syncwarp();
#pragma unroll 1
                    for (int d = 0; d < 64; d += 32) {
                        float v[32];
                        tmem_load(from + c + d, v);
                        if constexpr (MODE == kDelta) {
                            const int at = p.first + column + c + d;
#pragma unroll
                            for (int i = 0; i < 32; ++i) v[i] = f * exp2_fast(fmaf(v[i], p.exponent, -lse2));
                            while (e.next < at + 32) {
                                const int j = e.next - at;
                                const float share = p.entry_share ? p.entry_share[e.at] * f : f;
#pragma unroll
                                for (int i = 0; i < 32; ++i) v[i] -= i == j ? share : 0.f;
                                e.step(p);
                            }
                            __syncwarp();
                            if (!live || at + 32 > p.vocab) {
#pragma unroll
                                for (int i = 0; i < 32; ++i) v[i] = live && at + i < p.vocab ? v[i] : 0.f;
                            }
                        } else {
#pragma unroll
                            for (int i = 0; i < 32; ++i) v[i] *= f;
                            if (p.direct) {
                                const int row = q.m * kTile + static_cast<int>(rank) * 128 + quarter * 32 + lane;
                                if (row < p.count) {
                                    uint16_t* to = static_cast<uint16_t*>(p.direct) + static_cast<int64_t>(p.first + row) * p.direct_stride;
#pragma unroll
                                    for (int i = 0; i < 32; ++i)
                                        if (column + c + d + i < p.width) to[column + c + d + i] = pack1<BF16>(v[i]);
                                }
                                continue;
                            }
                        }
#pragma unroll
                        for (int g = 0; g < 4; ++g) {
                            const uint32_t to = line + (((d >> 3) + g) ^ (lane & 7)) * 16;
                            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(pack2<BF16>(v[8 * g], v[8 * g + 1])),
                                         "r"(pack2<BF16>(v[8 * g + 2], v[8 * g + 3])), "r"(pack2<BF16>(v[8 * g + 4], v[8 * g + 5])),
                                         "r"(pack2<BF16>(v[8 * g + 6], v[8 * g + 7]))
                                         : "memory");
                        }
                    }
                    if (MODE == kWeightGrad && p.direct) continue;
                    smem_to_async();
                    __syncwarp();
                    if (lane == 0) {
                        const int row = q.m * kTile + static_cast<int>(rank) * 128 + quarter * 32;
                        if (MODE == kDelta) store_tile(&map_out, lines, column + c, row);
                        else if (column + c < p.width && row < p.count) store_tile(&map_out, lines, column + c, p.first + row);
                        stores_commit();
                    }
                }
            } else {
                // 32 columns of fp32 make a line
#pragma unroll 1
                for (int c = 0; c < 128; c += 32) {
                    if (column + c >= p.width) break;
                    float v[32];
                    tmem_load(from + c, v);
                    if (lane == 0) stores_read();
                    __syncwarp();
#pragma unroll
                    for (int g = 0; g < 8; ++g) {
                        const uint32_t to = line + (g ^ (lane & 7)) * 16;
                        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(__float_as_uint(v[4 * g])), "r"(__float_as_uint(v[4 * g + 1])),
                                     "r"(__float_as_uint(v[4 * g + 2])), "r"(__float_as_uint(v[4 * g + 3]))
                                     : "memory");
                    }
                    smem_to_async();
                    __syncwarp();
                    if (lane == 0) {
                        const int row = q.split * p.n_rows + q.m * kTile + static_cast<int>(rank) * 128 + quarter * 32;
                        if (p.add) add_tile(&map_out, lines, column + c, row); else store_tile(&map_out, lines, column + c, row);
                        stores_commit();
                    }
                }
            }
            fence_before();
            __syncwarp();
            if (lane == 0) bar_arrive_cluster(in_block(acc_empty + 8 * (acc & 1), 0));
        }
        if (lane == 0) stores_done();
    }
    if (!ok) atomicExch(&p.shared->error, 1);
    __syncwarp();
    __syncthreads();
    fence_before();
    cluster_sync();
    fence_after();
    if (warp == 2) tmem_free(tmem, 512);
}

// ---- what the products need beforehand ------------------------------------------

__device__ __forceinline__ int64_t load_id(const void* ids, int bits, int64_t i) {
    return bits == 64 ? static_cast<const int64_t*>(ids)[i] : static_cast<const int32_t*>(ids)[i];
}
__device__ __forceinline__ float load_value(const void* data, int type, int64_t i) {
    if (type == kBF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(data)[i]);
    if (type == kF16) return __half2float(static_cast<const __half*>(data)[i]);
    return static_cast<const float*>(data)[i];
}

constexpr int kNone = -1, kBad = -2;      // what a row without a loss has in place of its first entry

// A teacher's rows: entries sorted by id (ties by place), their softmax beside them.  One block a row.
__global__ void teacher_kernel(Ids ids, Matrix logits, int entries, int room, int vocab, float inv_temperature, int* entry_ids, float* entry_share, int* first) {
    extern __shared__ uint8_t smem_raw[];
    uint64_t* key = reinterpret_cast<uint64_t*>(smem_raw);
    float* share = reinterpret_cast<float*>(key + room);
    __shared__ float red[32];
    __shared__ int bad;
    const int64_t row = blockIdx.x;
    const int tid = threadIdx.x, threads = blockDim.x;
    if (tid == 0) bad = 0;
    __syncthreads();
    float top = -INFINITY;
    for (int k = tid; k < room; k += threads) {
        int64_t id = -1;
        float l = -INFINITY;
        if (k < entries) {
            id = load_id(ids.data, ids.bits, row * ids.stride + k);
            if (id >= vocab) bad = 1;
            if (id >= 0) l = load_value(logits.data, logits.type, row * logits.stride + k) * inv_temperature;
        }
        key[k] = (static_cast<uint64_t>(id >= 0 && id < vocab ? static_cast<uint32_t>(id) : 0x7FFFFFFFu) << 32) | static_cast<uint32_t>(k);
        share[k] = l;
        top = l != l ? l : fmaxf(top, l);
    }
    // maximum, then sum, over the block
    auto over_block = [&](float x, bool max_of) {
#pragma unroll
        for (int d = 16; d; d >>= 1) {
            const float y = __shfl_xor_sync(~0u, x, d);
            x = max_of ? (x != x || y != y ? x + y : fmaxf(x, y)) : x + y;
        }
        __syncthreads();
        if ((tid & 31) == 0) red[tid >> 5] = x;
        __syncthreads();
        x = red[0];
        for (int w = 1; w < (threads >> 5); ++w) x = max_of ? (x != x || red[w] != red[w] ? x + red[w] : fmaxf(x, red[w])) : x + red[w];
        return x;
    };
    top = over_block(top, true);
    float sum = 0.f;
    const bool none = top == -INFINITY;
    for (int k = tid; k < room; k += threads) {
        share[k] = none ? 0.f : expf(share[k] - top);
        sum += share[k];
    }
    sum = over_block(sum, false);
    for (int size = 2; size <= room; size <<= 1)
        for (int step = size >> 1; step; step >>= 1) {
            __syncthreads();
            for (int i = tid; i < room / 2; i += threads) {
                const int a = ((i & ~(step - 1)) << 1) | (i & (step - 1)), b = a | step;
                const uint64_t x = key[a], y = key[b];
                if ((x > y) == ((a & size) == 0)) { key[a] = y; key[b] = x; }
            }
        }
    __syncthreads();
    for (int k = tid; k < entries; k += threads) {
        entry_ids[row * entries + k] = static_cast<int>(key[k] >> 32);
        entry_share[row * entries + k] = share[static_cast<uint32_t>(key[k])] / sum;
    }
    if (tid == 0) first[row] = bad ? kBad : none ? kNone : 0;
}

// Which rows have a loss: their places in order, behind them those of the others; and the scale of the gradients.  One block.
__global__ void __launch_bounds__(1024) rows_kernel(Ids targets, int64_t ignore, int vocab, int n, const int* first, int* entry_ids, int* rows, Shared* shared,
                                                    float* losses, float* lse, const float* grad, int64_t grad_stride, bool grad_of_mean, float inv_temperature,
                                                    bool half) {
    constexpr int kEach = 8;
    __shared__ int warp_sum[32];
    __shared__ float warp_top[32];
    __shared__ int done;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) done = 0;
    __syncthreads();
    float top = 0.f;
    for (int base = 0; base < n; base += 1024 * kEach) {
        const int at = base + tid * kEach;
        uint32_t bits = 0;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            if (at + i >= n) break;
            int state;
            if (first) {
                state = first[at + i];
            } else {
                const int64_t id = load_id(targets.data, targets.bits, at + i);
                state = id < 0 || id == ignore ? kNone : id >= vocab ? kBad : 0;
                entry_ids[at + i] = state < 0 ? INT_MAX : static_cast<int>(id);
            }
            if (state >= 0) {
                bits |= 1u << i;
                if (grad) {
                    const float g = fabsf(grad[(at + i) * grad_stride]);
                    top = g != g || top != top ? g + top : fmaxf(top, g);
                }
            } else if (losses) {
                losses[at + i] = state == kBad ? __int_as_float(0x7FC00000) : 0.f;
                lse[at + i] = 0.f;
            }
        }
        const int mine = __popc(bits);
        int before = mine;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int y = __shfl_up_sync(~0u, before, d);
            if (lane >= d) before += y;
        }
        if (lane == 31) warp_sum[warp] = before;
        __syncthreads();
        if (warp == 0) {
            int x = warp_sum[lane];
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int y = __shfl_up_sync(~0u, x, d);
                if (lane >= d) x += y;
            }
            warp_sum[lane] = x;
        }
        __syncthreads();
        int to = done + before - mine + (warp ? warp_sum[warp - 1] : 0);
        int out = at - to;                    // rows without a loss before this thread's
        for (int i = 0; i < kEach && at + i < n; ++i) {
            if (bits >> i & 1) rows[to++] = at + i; else rows[n - 1 - out++] = at + i;
        }
        __syncthreads();
        if (tid == 0) done += warp_sum[31];
        __syncthreads();
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) {
        const float y = __shfl_xor_sync(~0u, top, d);
        top = top != top || y != y ? top + y : fmaxf(top, y);
    }
    if (lane == 0) warp_top[warp] = top;
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < 32; ++w) top = top != top || warp_top[w] != warp_top[w] ? top + warp_top[w] : fmaxf(top, warp_top[w]);
        shared->active = done;
        shared->error = 0;
        if (grad) {
            // dZ is kept with the largest row gradient as 1 (bf16: its range is fp32's) or as 2^15, so that fp16 holds probabilities
            // down to 2^-29 in full precision and nothing above 2^16.
            const float unit = half ? 32768.f : 1.f;
            shared->row_scale = top == 0.f ? 0.f : unit / top;
            shared->unscale = top / unit * inv_temperature / (grad_of_mean ? fmaxf(static_cast<float>(done), 1.f) : 1.f);
        }
    }
}

// Rows `rows[0 .. active)` (all `n` where rows is NULL) copied together, lines of `cols` rounded up to whole 16 bytes; lines up to the next whole tile become 0.
__global__ void gather_kernel(const uint16_t* src, int64_t stride, int cols, const int* rows, const Shared* shared, int n, uint16_t* dst, int dst_cols, bool wide) {
    const int active = rows ? shared->active : n;
    const int end = rows ? (active + kTile - 1) / kTile * kTile : n;
    const int lines = dst_cols / 8;
    for (int64_t j = blockIdx.x; j < end; j += gridDim.x) {
        const uint16_t* from = j < active ? src + (rows ? rows[j] : j) * stride : nullptr;
        uint4* to = reinterpret_cast<uint4*>(dst + j * dst_cols);
        for (int i = threadIdx.x; i < lines; i += blockDim.x) {
            uint4 v = make_uint4(0, 0, 0, 0);
            if (from && wide) {
                v = __ldg(reinterpret_cast<const uint4*>(from) + i);
            } else if (from) {
                uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    if (8 * i + k < cols) w[k >> 1] |= static_cast<uint32_t>(from[8 * i + k]) << (16 * (k & 1));
                v = make_uint4(w[0], w[1], w[2], w[3]);
            }
            to[i] = v;
        }
    }
}

// ---- and afterwards ---------------------------------------------------------------

// Joins the half tiles' maxima and sums of 32 rows a block and takes the losses.
__global__ void __launch_bounds__(512) join_kernel(const float2* partial, int parts, int n_rows, const Shared* shared, const int* rows, int entries,
                                                   const int* entry_ids, const float* entry_share, const float* entry_logits, float exponent,
                                                   float inv_temperature, float* losses, float* lse) {
    __shared__ float2 piece[16][32];
    const int active = shared->active;
    const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
    for (int base = blockIdx.x * 32; base < active; base += gridDim.x * 32) {
        const int m = base + x;
        float high = -INFINITY, sum = 0.f;
        if (m < active)
            for (int k = y; k < parts; k += 16) {
                const float2 v = partial[static_cast<int64_t>(k) * n_rows + m];
                const float top = fmaxf(high, v.x), ref = top == -INFINITY ? 0.f : top;
                sum = sum * exp2_fast((high - ref) * exponent) + v.y * exp2_fast((v.x - ref) * exponent);
                high = top;
            }
        __syncthreads();
        piece[y][x] = make_float2(high, sum);
        __syncthreads();
        // 16 threads a row again, now beside one another
        const int row_of = threadIdx.x >> 4, k = threadIdx.x & 15;
        float2 v = piece[k][row_of];
        float top = v.x;
#pragma unroll
        for (int d = 8; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
        const float ref = top == -INFINITY ? 0.f : top;
        float total = v.y * exp2_fast((v.x - ref) * exponent);
#pragma unroll
        for (int d = 8; d; d >>= 1) total += __shfl_xor_sync(~0u, total, d);
        const float row_lse = ref * inv_temperature + logf(total);
        if (base + row_of < active) {
            const int row = rows[base + row_of];
            float loss = 0.f;
            for (int i = k; i < entries; i += 16) {
                const int64_t at = static_cast<int64_t>(row) * entries + i;
                if (entry_ids[at] == INT_MAX) continue;
                const float q = entry_share ? entry_share[at] : 1.f;
                if (q != 0.f) loss += q * ((entry_share ? logf(q) : 0.f) + (row_lse - entry_logits[at] * inv_temperature));
            }
#pragma unroll
            for (int d = 8; d; d >>= 1) loss += __shfl_xor_sync(0xFFFFu << (threadIdx.x & 16), loss, d);
            if (k == 0) {
                const bool failed = shared->error != 0;
                losses[row] = failed ? __int_as_float(0x7FC00000) : loss;
                lse[row] = row_lse;
            }
        }
    }
}

// Sum or mean of the losses, one block: sums of every 1024th, then over the block, always in the same order.
__global__ void __launch_bounds__(1024) total_kernel(const float* losses, int n, const Shared* shared, bool mean, float* total) {
    __shared__ float red[32];
    float sum = 0.f;
    for (int i = threadIdx.x; i < n; i += 1024) sum += losses[i];
#pragma unroll
    for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(~0u, sum, d);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = sum;
    __syncthreads();
    if (threadIdx.x < 32) {
        sum = red[threadIdx.x];
#pragma unroll
        for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(~0u, sum, d);
        if (threadIdx.x == 0) *total = mean ? sum / fmaxf(static_cast<float>(shared->active), 1.f) : sum;
    }
}

// Hidden gradient: the splits' sums in order, scaled, each row back at its place; rows without a loss get 0.
template <bool BF16>
__global__ void hidden_grad_kernel(const float* part, int splits, int n_rows, int part_cols, const Shared* shared, const int* rows, int n, int cols, uint16_t* out,
                                   int64_t stride, bool wide) {
    const int active = shared->active;
    const float unscale = shared->error ? __int_as_float(0x7FC00000) : shared->unscale;
    for (int64_t j = blockIdx.x; j < n; j += gridDim.x) {
        uint16_t* to = out + rows[j] * stride;
        for (int i = threadIdx.x * 4; i < cols; i += blockDim.x * 4) {
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            if (j < active) {
                for (int s = 0; s < splits; ++s) {
                    const float4 w = *reinterpret_cast<const float4*>(part + (static_cast<int64_t>(s) * n_rows + j) * part_cols + i);
                    v.x += w.x; v.y += w.y; v.z += w.z; v.w += w.w;
                }
                v.x *= unscale; v.y *= unscale; v.z *= unscale; v.w *= unscale;
            }
            if (wide) {
                *reinterpret_cast<uint2*>(to + i) = make_uint2(pack2<BF16>(v.x, v.y), pack2<BF16>(v.z, v.w));
            } else {
                const float each[4] = {v.x, v.y, v.z, v.w};
                for (int k = 0; k < 4 && i + k < cols; ++k) to[i + k] = pack1<BF16>(each[k]);
            }
        }
    }
}

// The table's gradient where no row has a loss (the products have nothing to do then), and NaN in it after a wait that ran out.
__global__ void no_rows_kernel(const Shared* shared, uint16_t* out, int64_t rows, int cols, int64_t stride, uint16_t nan) {
    if (shared->error && blockIdx.x == 0 && threadIdx.x == 0) out[0] = nan;
    if (shared->active) return;
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x)
        for (int i = threadIdx.x; i < cols; i += blockDim.x) out[r * stride + i] = 0;
}

// ---- host -------------------------------------------------------------------------

inline int64_t round_up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }
inline int64_t div_up(int64_t x, int64_t by) { return (x + by - 1) / by; }

struct Plan {
    int n, n_rows, vocab, width, cols, entries;     // cols: width in whole 16 bytes
    bool copy_weight;
    int piece, splits;                              // backward: columns a piece, parts of a piece summed apart
    uint64_t shared, rows, entry_ids, entry_share, first, entry_logits, hidden, weight, partial, delta, sums, bytes;
};

int multiprocessors() {
    int device = 0, count = 148;
    if (cudaGetDevice(&device) == cudaSuccess) cudaDeviceGetAttribute(&count, cudaDevAttrMultiProcessorCount, device);
    return count;
}

constexpr int64_t kDeltaBytes = 256 << 20;          // of a piece's dZ

Plan make_plan(const LossCall& c, bool backward) {
    Plan p{};
    p.n = static_cast<int>(c.hidden.rows);
    p.n_rows = static_cast<int>(round_up(std::max<int64_t>(c.hidden.rows, 1), kTile));
    p.vocab = static_cast<int>(c.weight.rows);
    p.width = static_cast<int>(c.hidden.cols);
    p.cols = static_cast<int>(round_up(p.width, 8));
    p.entries = c.entries ? c.entries : 1;
    p.copy_weight = p.width % 8 || c.weight.stride % 8 || reinterpret_cast<uintptr_t>(c.weight.data) % 16;
    uint64_t at = 0;
    auto take = [&](uint64_t bytes) {
        const uint64_t from = at;
        at += round_up(bytes, 1024);
        return from;
    };
    const int64_t listed = static_cast<int64_t>(p.n) * p.entries;
    p.shared = take(sizeof(Shared));
    p.rows = take(4ull * p.n);
    p.entry_ids = take(4ull * listed);
    if (c.entries) {
        p.entry_share = take(4ull * listed);
        p.first = take(4ull * p.n);
    }
    p.hidden = take(2ull * p.n_rows * p.cols);
    if (p.copy_weight) p.weight = take(2ull * p.vocab * p.cols);
    if (!backward) {
        p.entry_logits = take(4ull * listed);
        p.partial = take(8ull * 2 * div_up(p.vocab, kTile) * p.n_rows);
    } else {
        const int64_t tiles = div_up(p.vocab, kTile), room = std::max<int64_t>(1, kDeltaBytes / (2ll * kTile * p.n_rows));
        const int64_t pieces = div_up(tiles, room);
        p.piece = static_cast<int>(div_up(tiles, pieces) * kTile);
        const int64_t outs = static_cast<int64_t>(p.n_rows / kTile) * div_up(p.width, kTile), pairs = 74;
        p.splits = 1;
        double best = 1e30;
        for (int s = 1; s <= 32 && s * 512 <= p.piece; ++s) {
            const double waves = static_cast<double>(div_up(outs * s, pairs)) / s + 0.01 * s;
            if (waves < best - 1e-9) { best = waves; p.splits = s; }
        }
        p.delta = take(2ull * p.n_rows * p.piece);
        p.sums = take(4ull * p.splits * p.n_rows * p.cols);
    }
    p.bytes = at;
    return p;
}

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                              CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn encode_fn() {
    static const EncodeFn fn = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult got;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &got) != cudaSuccess || got != cudaDriverEntryPointSuccess) f = nullptr;
        return reinterpret_cast<EncodeFn>(f);
    }();
    return fn;
}

// Lines of 128 bytes, `height` of them a box, swizzled.
bool tile_map(CUtensorMap* map, int type, const void* data, int64_t rows, int64_t cols, int64_t stride, int height) {
    const int size = type == kF32 ? 4 : 2;
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)}, strides[1] = {static_cast<cuuint64_t>(stride * size)};
    const cuuint32_t box[2] = {static_cast<cuuint32_t>(128 / size), static_cast<cuuint32_t>(height)}, steps[2] = {1, 1};
    const CUtensorMapDataType kind = type == kF32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : type == kBF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    return encode_fn()(map, kind, 2, const_cast<void*>(data), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                       CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int MODE>
cudaError_t launch_product(bool bf16, const CUtensorMap& a, const CUtensorMap& b, const CUtensorMap& out, const Product& p, cudaStream_t stream) {
    auto* kernel = bf16 ? product_kernel<MODE, true> : product_kernel<MODE, false>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes);
    if (e != cudaSuccess) return e;
    kernel<<<multiprocessors() / 2 * 2, kThreads, kSmemBytes, stream>>>(a, b, out, p);
    return cudaGetLastError();
}

struct Prepared {
    Plan plan;
    char* at;
    Shared* shared;
    int* rows;
    const uint16_t* weight;
    int64_t weight_stride;
    Product product;
    CUtensorMap hidden_map, weight_map;
};

const char* cuda_error(cudaError_t e) { return e == cudaSuccess ? nullptr : cudaGetErrorString(e); }

const char* prepare(const LossCall& c, bool backward, Prepared& w) {
    w.plan = make_plan(c, backward);
    const Plan& p = w.plan;
    if (c.workspace_bytes < p.bytes) return "the workspace is too small";
    if (!encode_fn()) return "the driver has no tiled copies";
    w.at = static_cast<char*>(c.workspace);
    w.shared = reinterpret_cast<Shared*>(w.at + p.shared);
    w.rows = reinterpret_cast<int*>(w.at + p.rows);
    int* entry_ids = reinterpret_cast<int*>(w.at + p.entry_ids);
    float* entry_share = c.entries ? reinterpret_cast<float*>(w.at + p.entry_share) : nullptr;
    int* first = c.entries ? reinterpret_cast<int*>(w.at + p.first) : nullptr;
    const float inv_temperature = 1.f / c.temperature;
    if (c.entries) {
        int room = 2;
        while (room < c.entries) room *= 2;
        teacher_kernel<<<p.n, std::min(256, std::max(32, room / 2)), room * 12, c.stream>>>(c.targets, c.teacher, c.entries, room, p.vocab, inv_temperature, entry_ids,
                                                                                             entry_share, first);
    }
    rows_kernel<<<1, 1024, 0, c.stream>>>(c.targets, c.ignore, p.vocab, p.n, first, entry_ids, w.rows, w.shared, backward ? nullptr : c.losses,
                                          backward ? nullptr : c.lse, backward ? c.grad : nullptr, c.grad_stride, c.grad_of_mean, inv_temperature,
                                          c.hidden.type == kF16);
    uint16_t* hidden = reinterpret_cast<uint16_t*>(w.at + p.hidden);
    const bool wide = p.width % 8 == 0 && c.hidden.stride % 8 == 0 && reinterpret_cast<uintptr_t>(c.hidden.data) % 16 == 0;
    gather_kernel<<<std::min(p.n_rows, 148 * 16), 128, 0, c.stream>>>(static_cast<const uint16_t*>(c.hidden.data), c.hidden.stride, p.width, w.rows, w.shared, p.n, hidden,
                                                                      p.cols, wide);
    w.weight = static_cast<const uint16_t*>(c.weight.data);
    w.weight_stride = c.weight.stride;
    if (p.copy_weight) {
        uint16_t* copy = reinterpret_cast<uint16_t*>(w.at + p.weight);
        gather_kernel<<<148 * 16, 128, 0, c.stream>>>(w.weight, c.weight.stride, p.width, nullptr, w.shared, p.vocab, copy, p.cols, false);
        w.weight = copy;
        w.weight_stride = p.cols;
    }
    if (!tile_map(&w.hidden_map, c.hidden.type, hidden, p.n_rows, p.cols, p.cols, 64) ||
        !tile_map(&w.weight_map, c.hidden.type, w.weight, p.vocab, p.cols, w.weight_stride, 64))
        return "a tensor map was refused";
    Product& q = w.product;
    q = Product{};
    q.shared = w.shared;
    q.rows = w.rows;
    q.n_rows = p.n_rows;
    q.vocab = p.vocab;
    q.width = p.cols;
    q.count = p.vocab;
    q.entries = p.entries;
    q.entry_ids = entry_ids;
    q.entry_share = entry_share;
    q.exponent = kLog2e / c.temperature;
    q.splits = 1;
    return cuda_error(cudaGetLastError());
}

}  // namespace

uint64_t loss_workspace(const LossCall& c, bool backward) { return c.hidden.rows ? make_plan(c, backward).bytes : 0; }

const char* loss_forward(const LossCall& c) {
    if (c.hidden.rows == 0) return c.total ? cuda_error(cudaMemsetAsync(c.total, 0, 4, c.stream)) : nullptr;
    Prepared w;
    if (const char* e = prepare(c, false, w)) return e;
    const Plan& p = w.plan;
    Product& q = w.product;
    q.partial = reinterpret_cast<float2*>(w.at + p.partial);
    q.entry_logits = reinterpret_cast<float*>(w.at + p.entry_logits);
    if (cudaError_t e = launch_product<kForward>(c.hidden.type == kBF16, w.hidden_map, w.weight_map, w.hidden_map, q, c.stream)) return cuda_error(e);
    join_kernel<<<static_cast<int>(std::min<int64_t>(div_up(p.n, 32), 148 * 4)), 512, 0, c.stream>>>(
        q.partial, static_cast<int>(2 * div_up(p.vocab, kTile)), p.n_rows, w.shared, w.rows, p.entries, q.entry_ids, q.entry_share, q.entry_logits, q.exponent,
        1.f / c.temperature, c.losses, c.lse);
    if (c.total) total_kernel<<<1, 1024, 0, c.stream>>>(c.losses, p.n, w.shared, c.mean, c.total);
    return cuda_error(cudaGetLastError());
}

const char* loss_backward(const LossCall& c) {
    const bool bf16 = c.hidden.type == kBF16;
    if (c.hidden.rows == 0) {
        if (!c.d_weight.data) return nullptr;
        return cuda_error(cudaMemset2DAsync(const_cast<void*>(c.d_weight.data), c.d_weight.stride * 2, 0, c.d_weight.cols * 2, c.d_weight.rows, c.stream));
    }
    Prepared w;
    if (const char* e = prepare(c, true, w)) return e;
    const Plan& p = w.plan;
    uint16_t* delta = reinterpret_cast<uint16_t*>(w.at + p.delta);
    float* sums = reinterpret_cast<float*>(w.at + p.sums);
    CUtensorMap delta_map, delta_out, sums_out, weight_out;
    if (!tile_map(&delta_map, c.hidden.type, delta, p.n_rows, p.piece, p.piece, 64) || !tile_map(&delta_out, c.hidden.type, delta, p.n_rows, p.piece, p.piece, 32) ||
        !tile_map(&sums_out, kF32, sums, static_cast<int64_t>(p.splits) * p.n_rows, p.cols, p.cols, 32))
        return "a tensor map was refused";
    uint16_t* d_weight = static_cast<uint16_t*>(const_cast<void*>(c.d_weight.data));
    const bool direct = d_weight && (p.width % 8 || c.d_weight.stride % 8 || reinterpret_cast<uintptr_t>(d_weight) % 16);
    if (d_weight && !direct) {
        if (!tile_map(&weight_out, c.hidden.type, d_weight, p.vocab, p.width, c.d_weight.stride, 32)) return "a tensor map was refused";
    } else {
        weight_out = delta_out;
    }
    for (int first = 0; first < p.vocab; first += p.piece) {
        Product q = w.product;
        q.first = first;
        q.count = std::min(p.piece, p.vocab - first);
        q.lse = c.lse;
        q.grad = c.grad;
        q.grad_stride = c.grad_stride;
        if (cudaError_t e = launch_product<kDelta>(bf16, w.hidden_map, w.weight_map, delta_out, q, c.stream)) return cuda_error(e);
        if (c.d_hidden.data) {
            q.splits = p.splits;
            q.add = first > 0;
            if (cudaError_t e = launch_product<kHiddenGrad>(bf16, delta_map, w.weight_map, sums_out, q, c.stream)) return cuda_error(e);
        }
        if (d_weight) {
            q.splits = 1;
            q.add = false;
            q.direct = direct ? d_weight : nullptr;
            q.direct_stride = c.d_weight.stride;
            if (direct) q.width = p.width;
            if (cudaError_t e = launch_product<kWeightGrad>(bf16, delta_map, w.hidden_map, weight_out, q, c.stream)) return cuda_error(e);
        }
    }
    if (c.d_hidden.data) {
        uint16_t* out = static_cast<uint16_t*>(const_cast<void*>(c.d_hidden.data));
        const bool wide = p.width % 4 == 0 && c.d_hidden.stride % 4 == 0 && reinterpret_cast<uintptr_t>(out) % 8 == 0;
        auto* kernel = bf16 ? hidden_grad_kernel<true> : hidden_grad_kernel<false>;
        kernel<<<std::min(p.n, 148 * 16), 256, 0, c.stream>>>(sums, p.splits, p.n_rows, p.cols, w.shared, w.rows, p.n, p.width, out, c.d_hidden.stride, wide);
    }
    if (d_weight) no_rows_kernel<<<148 * 4, 256, 0, c.stream>>>(w.shared, d_weight, p.vocab, p.width, c.d_weight.stride, bf16 ? 0x7FC0 : 0x7E00);
    return cuda_error(cudaGetLastError());
}

}  // namespace gtok
