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
// sum per row (and takes the entries' logits out); a small kernel joins the tiles' pairs.  Up to 64 rows have a form of their own (few_kernel).  Backward: per piece of the vocabulary, the
// tile of Z is computed again and becomes dZ in 16 bits, from which two more products give the piece's part of dH and its rows of dW.
// Nothing in memory grows with n x vocab as the logits do: of dZ there is a piece at a time, 512 MiB or one tile of the vocabulary, and the
// forward pass keeps a maximum and a sum for each row and 128 ids, 8 bytes, a 32nd of the logits in 16 bits (65 MB for 8,192 rows of 128,256).
//
// Rows without a loss (ignored targets, no teacher entries) are left out before the products: the others are copied together, so
// neither time nor NaN of masked positions is carried along.
#include "sm100.cuh"
#include "vocab_launch.cuh"
#include "vocab_ops.h"

#include <algorithm>
#include <climits>
#include <cmath>

namespace gtok {
namespace {

using namespace sm100;

constexpr int kTile = 256;              // rows and columns of a pair's tile
constexpr int kDepth = 64;              // elements of the summed dimension a stage holds: one 128-byte line
constexpr int kStageBytes = 32768;      // 128 x 64 of either operand
constexpr int kEpilogueWarps = 8;
constexpr int kThreads = 128 + 32 * kEpilogueWarps;
constexpr int kStagingBytes = 4096;     // a warp's 32 lines of 128 bytes on their way out
// Row tiles that share a sweep over the vocabulary: 16 x 256 rows, which stay in L2 up to a width of some 12,000 (100 of 126 MB).  Measured at 4096 only:
// 4,093 rows in 2.52 ms, with 8 tiles 2.60, with 32 2.53.
constexpr int kGroup = 16;

constexpr float kLog2e = 1.4426950408889634f;

// The matrix instruction's sums are cut off, not rounded: each step of 16 elements takes the logit towards 0, by 2^-26 of its final
// value on average (measured on random and on coherent rows alike: 1.9e-6 to 2.1e-6 of it at a width of 2048, 4.0e-6 to 4.2e-6 at
// 4096).  Logits are scaled up by that much.  Where nothing is cut off, as in rows of one element or of small whole numbers, they are too large
// by it instead: the error of such rows is what that of all others would be without (losses of 4,093 rows of width 4096 against 64 bits: 6e-7 with, 2.6e-6 without).
inline float cut_off(int width) { return 1.f + static_cast<float>((width + 15) / 16) * 0x1p-26f; }

// Scalars in device memory that the kernels hand to one another.
struct Shared {
    int active;          // rows with a loss
    int error;           // a wait ran out
    unsigned joined;     // blocks of join_kernel, or of the last product of a backward pass, that are done
    int splits;          // hidden gradient: parts of a piece's columns that are summed apart
    float unscale;       // gradients are the products times this
};

enum { kForward = 0, kDelta = 1, kHiddenGrad = 2, kWeightGrad = 3 };

// The forward pass writes no tiles and has its room for another stage.
__host__ __device__ constexpr int stages(int mode) { return mode == kForward ? 7 : 6; }
__host__ __device__ constexpr int smem_bytes(int mode) { return 1024 + stages(mode) * kStageBytes + (mode == kForward ? 0 : kEpilogueWarps * kStagingBytes) + 256; }

struct Entry { int id; float share; };        // what a row's softmax should be at `id`; ascending in a row, INT_MAX after the last
struct RowInfo { float lse2, factor; };       // of an active row: lse in powers of 2; what dZ is multiplied by

// The hidden gradient's parts and where their sums go.
struct HiddenOut {
    const float* part;         // NULL: nothing to do
    int part_cols;
    const int* rows;
    int n, cols;
    uint16_t* out;
    int64_t stride;
    bool wide;                 // rows of `out` are lines of whole 16 bytes
};

struct Product {
    Shared* shared;
    int n_rows;                // rows of the padded arrays (a multiple of kTile)
    int vocab, width;
    int first, count;          // first column of this piece, its columns
    int entries;
    const Entry* entry;        // [active][entries]
    const RowInfo* info;       // backward: [active]
    float exponent;            // log2(e) / T
    float2* partial;           // forward: (maximum, sum) of [half tile of columns][row]
    float* entry_logits;       // forward: [active][entries]
    bool add;                  // hidden gradient: onto what earlier pieces left
    bool direct;               // weight gradient, where its rows are no lines of whole 16 bytes: written by the threads
    uint16_t* out;             // weight gradient
    int64_t out_stride;
    bool last;                 // weight gradient: of the last piece
    HiddenOut hidden_out;      // and what its idle warps may finish meanwhile
};

struct Place { int m, n, k0, k1, split; };     // tile of the output, blocks of the summed dimension

// How one product is cut into tiles.
template <int MODE>
struct Tiling {
    int row_tiles, col_tiles, width_tiles, splits, blocks, tiles;
    __device__ __forceinline__ Tiling(const Product& p, int active, int splits_) : splits(splits_) {
        row_tiles = (active + kTile - 1) / kTile;
        width_tiles = (p.width + kTile - 1) / kTile;
        col_tiles = (p.count + kTile - 1) / kTile;
        if (MODE == kHiddenGrad) {
            blocks = (p.count + kDepth - 1) / kDepth;        // fewer in the last piece; a split may then be left without any
            tiles = row_tiles * width_tiles * splits;
        } else if (MODE == kWeightGrad) {
            blocks = (active + kDepth - 1) / kDepth;
            tiles = active ? col_tiles * width_tiles : 0;
        } else {
            blocks = (p.width + kDepth - 1) / kDepth;
            tiles = row_tiles * col_tiles;
        }
    }
    __device__ __forceinline__ Place place(int t) const {
        Place q;
        q.k0 = 0;
        q.k1 = blocks;
        q.split = 0;
        if (MODE == kHiddenGrad) {
            q.split = t / (row_tiles * width_tiles);
            t -= q.split * row_tiles * width_tiles;
            q.m = t / width_tiles;
            q.n = t - q.m * width_tiles;
            q.k0 = static_cast<int>(static_cast<int64_t>(blocks) * q.split / splits);
            q.k1 = static_cast<int>(static_cast<int64_t>(blocks) * (q.split + 1) / splits);
        } else if (MODE == kWeightGrad) {
            q.m = t / width_tiles;
            q.n = t - q.m * width_tiles;
        } else {
            const int group = t / (kGroup * col_tiles);
            const int first = group * kGroup, rows = min(kGroup, row_tiles - first);
            t -= first * col_tiles;
            q.n = t / rows;
            q.m = first + t - q.n * rows;
        }
        return q;
    }
};

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

// A sum in units of 2^unit, in those of the power of a maximum of logits as it is (rounded once, with what it differs by).
__device__ __forceinline__ float in_units(float sum, float unit, float high, float exponent) {
    return sum * exp2_fast(fmaf(high == -INFINITY ? 0.f : -high, exponent, unit));
}

// A row's entries from a column on.  The first of them is searched for while the tile before is worked on, a step at a time, so that
// the loads' latency is not waited for: each step looks at seven entries at once, and four steps do for kMaxEntries.
struct Ahead {
    const Entry* list;
    int lo, hi, column;
    bool there;
    Entry next, then;          // the entry that comes next, and the one after it
    RowInfo info;
    __device__ __forceinline__ Entry get(const Product& p, int i) const { return i < p.entries ? list[i] : Entry{INT_MAX, 0.f}; }
    __device__ __forceinline__ void begin(const Product& p, int m, bool live, int from, bool with_info) {
        list = p.entry + static_cast<int64_t>(m) * p.entries;
        lo = 0;
        hi = live ? p.entries : 0;
        column = from;
        there = !live;
        next = then = Entry{INT_MAX, 0.f};
        info = RowInfo{0.f, 0.f};
        if (with_info && live) info = p.info[m];
    }
    __device__ __forceinline__ void step(const Product& p) {
        if (there) return;
        if (lo < hi) {
            const int s = (hi - lo + 8) >> 3;          // hi - lo + 1 places are possible, and seven probes leave eight parts of them
            int c = 0;
#pragma unroll
            for (int k = 1; k < 8; ++k) {
                const int at = lo + k * s - 1;
                c += at < hi && list[at].id < column;
            }
            lo += c * s;
            hi = min(hi, lo + s - 1);
            if (lo < hi) return;
        }
        next = get(p, lo);
        then = get(p, lo + 1);
        there = true;
    }
    __device__ __forceinline__ void advance(const Product& p) {
        ++lo;
        next = then;
        then = get(p, lo + 1);
    }
};

// Hidden gradient: the splits' sums in order, scaled, each row back at its place; rows without a loss get 0.  Eight columns a thread.
template <bool BF16>
__device__ __forceinline__ void finish_hidden(const HiddenOut& h, const Shared* shared, int64_t self, int64_t threads) {
    const int active = shared->active, splits = shared->splits;
    const int64_t apart = static_cast<int64_t>((active + kTile - 1) / kTile * kTile) * h.part_cols;
    const float unscale = shared->error ? __int_as_float(0x7FC00000) : shared->unscale;
    const int lines = (h.cols + 7) / 8;
    const int64_t units = static_cast<int64_t>(h.n) * lines;
    constexpr int kUnits = 2, kParts = 4;             // on their way at once
    for (int64_t u = self; u < units; u += kUnits * threads) {
        float v[kUnits][8];
        const float* from[kUnits];
        bool sums[kUnits];
        int j[kUnits], i[kUnits];
#pragma unroll
        for (int k = 0; k < kUnits; ++k) {
            const int64_t at = min(u + k * threads, units - 1);
            j[k] = static_cast<int>(at / lines);
            i[k] = static_cast<int>(at - static_cast<int64_t>(j[k]) * lines) * 8;
            sums[k] = u + k * threads < units && j[k] < active;
            from[k] = h.part + static_cast<int64_t>(j[k]) * h.part_cols + i[k];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[k][e] = 0.f;
        }
        for (int s = 0; s < splits; s += kParts) {
            float4 a[kUnits][kParts], b[kUnits][kParts];
#pragma unroll
            for (int k = 0; k < kUnits; ++k)
#pragma unroll
                for (int d = 0; d < kParts; ++d)
                    if (sums[k] && s + d < splits) {
                        a[k][d] = *reinterpret_cast<const float4*>(from[k] + (s + d) * apart);
                        b[k][d] = *reinterpret_cast<const float4*>(from[k] + (s + d) * apart + 4);
                    }
#pragma unroll
            for (int k = 0; k < kUnits; ++k)
#pragma unroll
                for (int d = 0; d < kParts; ++d)
                    if (sums[k] && s + d < splits) {
                        v[k][0] += a[k][d].x; v[k][1] += a[k][d].y; v[k][2] += a[k][d].z; v[k][3] += a[k][d].w;
                        v[k][4] += b[k][d].x; v[k][5] += b[k][d].y; v[k][6] += b[k][d].z; v[k][7] += b[k][d].w;
                    }
        }
#pragma unroll
        for (int k = 0; k < kUnits; ++k) {
            if (u + k * threads >= units) break;
            if (sums[k]) {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[k][e] *= unscale;
            }
            uint16_t* to = h.out + h.rows[j[k]] * h.stride + i[k];
            if (h.wide) {
                *reinterpret_cast<uint4*>(to) =
                    make_uint4(pack2<BF16>(v[k][0], v[k][1]), pack2<BF16>(v[k][2], v[k][3]), pack2<BF16>(v[k][4], v[k][5]), pack2<BF16>(v[k][6], v[k][7]));
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (i[k] + e < h.cols) to[e] = pack1<BF16>(v[k][e]);
            }
        }
    }
}

// A persistent product: one pair of blocks an SM pair, tiles handed out in turn.  Warp 0 of each block copies its half of the operands
// in, warp 1 of the first block issues the matrix instructions for both, eight warps of each block take the accumulators out while the
// next tile is summed into the other half of tensor memory.
//
//   forward        A = H, B = W (lines along the width)      -> maximum, sum and the entries' logits of each row
//   delta          the same                                  -> dZ = factor (2^(z log2(e) / T - lse2) - q), 16 bits
//   hidden grad    A = dZ (along the vocabulary), B = W (across)   -> parts of dH, fp32
//   weight grad    A = dZ (across), B = H (across)           -> rows of dW
//
// Bound by the tensor cores, and in long calls by the power that they may take.  256 x 256 a pair, because a tile then takes 64 KB of operands from
// L2 for each 8.4 MFLOP, which L2 just gives at the full rate (13 TB/s); both operands come through TMA in 128-byte lines, whichever way they
// run, so nothing is ever transposed in memory.  Epilogues work from registers: 32 columns of a row a thread and step, the next 32 on their way.
// Tensor pipe in use (2,048 rows, 128,256 x 1024): forward 97 %, the others 93 to 96.  Forward of 4,093 rows against
// 128,256 x 4096 in 2.5 to 2.6 ms: 1.6 to 1.7 PFLOP/s, 1.00 to 1.04 of what a library product of 8192^3 measured.
template <int MODE, bool BF16>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    product_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_out,
                   const __grid_constant__ Product p) {
    constexpr bool kAcrossA = MODE == kWeightGrad, kAcrossB = MODE >= kHiddenGrad;     // operand's lines run across the summed dimension
    constexpr bool kRows = MODE == kForward || MODE == kDelta;                          // the tile is one of logits
    constexpr int kStages = stages(MODE);
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_addr(smem_raw) + 1023) & ~1023u;
    const uint32_t staging = base + kStages * kStageBytes;
    const uint32_t bars = staging + (MODE == kForward ? 0 : kEpilogueWarps * kStagingBytes);
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

    after_previous();
    const int active = p.shared->active, splits = MODE == kHiddenGrad ? p.shared->splits : 1;
    const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    const Tiling<MODE> tiling(p, active, splits);
    const int tiles = tiling.tiles;
    bool ok = true;

    if (warp == 0) {
        if (elect()) {
            const uint32_t full_of_pair = in_block(full, 0);
            uint32_t it = 0;
            for (int t = pair; t < tiles && ok; t += pairs) {
                const Place q = tiling.place(t);
                const int am = q.m * kTile + rank * 128, bn = q.n * kTile + rank * 128 + (kRows ? p.first : 0);
                const int bk = MODE == kHiddenGrad ? p.first : 0;
                // Boxes of 64 rows that hold no active row are taken from beyond the array, which gives zeros: nothing is read for them, and products
                // with zeros take less power.
                const int am0 = MODE == kWeightGrad || am < active ? am : p.n_rows, am1 = MODE == kWeightGrad || am + 64 < active ? am + 64 : p.n_rows;
                for (int k = q.k0; k < q.k1; ++k, ++it) {
                    const uint32_t s = it % kStages;
                    if (!bar_wait(empty + 8 * s, ((it / kStages) & 1) ^ 1)) { ok = false; break; }
                    const uint32_t a = base + s * kStageBytes, b = a + kStageBytes / 2, bar = full_of_pair + 8 * s;
                    if (rank == 0) bar_expect(full + 8 * s, 2 * kStageBytes);
                    const int x = k * kDepth;
                    load_tile(a, &map_a, kAcrossA ? am0 : x, kAcrossA ? x : am0, bar);
                    load_tile(a + 8192, &map_a, kAcrossA ? am1 : x, kAcrossA ? x : am1, bar);
                    load_tile(b, &map_b, kAcrossB ? bn : x, kAcrossB ? x + bk : bn, bar);
                    load_tile(b + 8192, &map_b, kAcrossB ? bn + 64 : x, kAcrossB ? x + bk : bn + 64, bar);
                }
            }
            // The other block's arrivals for the last stages come before this one may leave ...
            for (uint32_t i = it < kStages ? 0 : it - kStages; i < it && ok; ++i) ok = bar_wait(empty + 8 * (i % kStages), (i / kStages) & 1);
            if (!ok) {      // ... and, after a wait that ran out, copies that are still under way
                const uint64_t from = nanoseconds();
                while (nanoseconds() - from < 2000000ull) __nanosleep(1000);
            }
        }
    } else if (warp == 1) {
        if (rank == 0 && elect()) {
            const uint32_t kind = mma_kind(BF16, kAcrossA, kAcrossB, kTile);
            uint32_t it = 0, acc = 0;
            for (int t = pair; t < tiles && ok; t += pairs) {
                const Place q = tiling.place(t);
                if (q.k0 >= q.k1) continue;
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
                ++acc;
            }
        }
    } else if (warp < 4) {
        if (MODE == kWeightGrad && p.hidden_out.part)
            finish_hidden<BF16>(p.hidden_out, p.shared, static_cast<int64_t>(blockIdx.x) * 64 + threadIdx.x - 64, static_cast<int64_t>(gridDim.x) * 64);
    } else {
        const int quarter = warp & 3, half = (warp - 4) >> 2;
        const uint32_t lines = staging + (warp - 4) * kStagingBytes;
        const uint32_t line = lines + lane * 128;
        const float unscale = MODE == kWeightGrad ? p.shared->unscale : 0.f;
        Ahead ahead;
        auto look_ahead = [&](int t) {
            if (t >= tiles) t = pair;                  // (no further tile: anything that is in bounds)
            const Place q = tiling.place(t);
            const int m = q.m * kTile + rank * 128 + quarter * 32 + lane;
            ahead.begin(p, m, m < active, p.first + q.n * kTile + half * 128, MODE == kDelta);
        };
        if (kRows && pair < tiles) look_ahead(pair);
        uint32_t acc = 0;
        // Forward: maximum and sum of a row in this tile; where all tiles are of the same rows, in all so far.  The sum is in units of 2^unit, the
        // maximum's power as it is rounded, so that a step at which the maximum stays multiplies by exactly 1.  (By the power that is not rounded, the
        // sum took that rounding anew at every step: with 200 rows of 151,665 ids and logits of 40 to 100 in front, lse was off by up to 1.6e-4, and is by 5e-7.)
        float high = -INFINITY, unit = -INFINITY, sum = 0.f;
        for (int t = pair; t < tiles; t += pairs) {
            const Place q = tiling.place(t);
            if (q.k0 >= q.k1) continue;
            const int m = q.m * kTile + rank * 128 + quarter * 32 + lane;       // this thread's line of the tile
            const int column = q.n * kTile + half * 128;                        // of the output; of the piece where columns are the vocabulary's
            const uint32_t from = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + (acc & 1) * 256 + half * 128;
            const bool live = m < active;
            Ahead e;
            if (kRows) {
                while (!ahead.there) ahead.step(p);
                e = ahead;
                look_ahead(t + pairs);
            }
            ok = __all_sync(~0u, bar_wait(acc_full + 8 * (acc & 1), (acc >> 1) & 1));
            if (!ok) break;
            fence_after();
            float va[32], vb[32];
            if (tiling.row_tiles > 1) {
                high = unit = -INFINITY;
                sum = 0.f;
            }
            // What becomes of 32 columns from `c` on.
            auto work = [&](float (&v)[32], int c) {
                const int at = p.first + column + c;
                if constexpr (MODE == kForward) {
                    if (at + 32 > p.vocab) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) v[i] = at + i < p.vocab ? v[i] : -INFINITY;
                    }
                    float top = v[0];
#pragma unroll
                    for (int i = 1; i < 32; ++i) top = fmaxf(top, v[i]);
                    top = fmaxf(top, high);
                    const float at_top = __fmul_rn(top, p.exponent), from_top = top == -INFINITY ? 0.f : at_top;
                    sum *= exp2_fast(unit - from_top);
                    high = top;
                    unit = at_top;
                    float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int i = 0; i < 32; ++i) part[i & 3] += exp2_fast(fmaf(v[i], p.exponent, -from_top));
                    sum += (part[0] + part[1]) + (part[2] + part[3]);
                    while (e.next.id < at + 32) {
                        const int j = e.next.id - at;
                        float z = 0.f;
#pragma unroll
                        for (int i = 0; i < 32; ++i) z = i == j ? v[i] : z;
                        p.entry_logits[static_cast<int64_t>(m) * p.entries + e.lo] = z;
                        e.advance(p);
                    }
                    ahead.step(p);
                    __syncwarp();
                } else if constexpr (MODE == kDelta || MODE == kWeightGrad) {
                    // 64 columns of 16 bits make a line
                    if (MODE == kDelta) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) v[i] = e.info.factor * exp2_fast(fmaf(v[i], p.exponent, -e.info.lse2));
                        while (e.next.id < at + 32) {
                            const int j = e.next.id - at;
                            const float share = e.next.share * e.info.factor;
#pragma unroll
                            for (int i = 0; i < 32; ++i) v[i] -= i == j ? share : 0.f;
                            e.advance(p);
                        }
                        ahead.step(p);
                        __syncwarp();
                        if (!live || at + 32 > p.vocab) {
#pragma unroll
                            for (int i = 0; i < 32; ++i) v[i] = live && at + i < p.vocab ? v[i] : 0.f;
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; ++i) v[i] *= unscale;
                        if (p.direct) {
                            if (m < p.count) {
                                uint16_t* to = p.out + static_cast<int64_t>(p.first + m) * p.out_stride;
#pragma unroll
                                for (int i = 0; i < 32; ++i)
                                    if (column + c + i < p.width) to[column + c + i] = pack1<BF16>(v[i]);
                            }
                            __syncwarp();
                            return;
                        }
                    }
                    if ((c & 32) == 0) {
                        if (lane == 0) stores_read();
                        __syncwarp();
                    }
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const uint32_t to = line + ((((c & 32) >> 3) + g) ^ (lane & 7)) * 16;
                        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(pack2<BF16>(v[8 * g], v[8 * g + 1])),
                                     "r"(pack2<BF16>(v[8 * g + 2], v[8 * g + 3])), "r"(pack2<BF16>(v[8 * g + 4], v[8 * g + 5])),
                                     "r"(pack2<BF16>(v[8 * g + 6], v[8 * g + 7]))
                                     : "memory");
                    }
                    if (c & 32) {
                        smem_to_async();
                        __syncwarp();
                        if (lane == 0) {
                            const int x = column + c - 32, row = m - lane;
                            if (MODE == kDelta) store_tile(&map_out, lines, x, row);
                            else if (x < p.width && row < p.count) store_tile(&map_out, lines, x, p.first + row);
                            stores_commit();
                        }
                    }
                } else {
                    // 32 columns of fp32 make a line
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
                        const int row = q.split * ((active + kTile - 1) / kTile * kTile) + m;
                        if (column + c < p.width) {
                            if (p.add) add_tile(&map_out, lines, column + c, row); else store_tile(&map_out, lines, column + c, row);
                        }
                        stores_commit();
                    }
                }
            };
            // Lines without an active row, of which nothing is asked; dZ is read in steps of 64 rows, and they are 0 up to there.
            const bool idle = MODE == kDelta ? m - lane >= (active + kDepth - 1) / kDepth * kDepth : MODE != kWeightGrad && m - lane >= active;
            if (idle) {
                if (lane == 0) bar_arrive_cluster(in_block(acc_empty + 8 * (acc & 1), 0));
                ++acc;
                continue;
            }
            tmem_load(from, va);
#pragma unroll 1
            for (int c = 0; c < 128; c += 64) {
                tmem_wait(va);
                tmem_load(from + c + 32, vb);
                work(va, c);
                tmem_wait(vb);
                if (c == 0) {
                    tmem_load(from + 64, va);
                } else {              // all taken out: the next tile but one may be summed there
                    fence_before();
                    __syncwarp();
                    if (lane == 0) bar_arrive_cluster(in_block(acc_empty + 8 * (acc & 1), 0));
                }
                work(vb, c + 32);
            }
            if (MODE == kForward && live && tiling.row_tiles > 1)
                p.partial[static_cast<int64_t>(q.n * 2 + half) * p.n_rows + m] = make_float2(high, in_units(sum, unit, high, p.exponent));
            ++acc;
        }
        if (MODE == kForward && tiling.row_tiles == 1 && pair < tiles) {
            const int m = rank * 128 + quarter * 32 + lane;
            if (m < active) p.partial[static_cast<int64_t>(pair * 2 + half) * p.n_rows + m] = make_float2(high, in_units(sum, unit, high, p.exponent));
        }
        if (lane == 0) stores_done();
    }
    if (!ok) atomicExch(&p.shared->error, 1);
    __syncwarp();
    let_next_begin();
    __syncthreads();
    if (MODE == kWeightGrad) {
        if (active == 0) {       // no product, no gradient
            for (int64_t r = p.first + blockIdx.x; r < p.first + p.count; r += gridDim.x)
                for (int i = threadIdx.x; i < p.width; i += kThreads) p.out[r * p.out_stride + i] = 0;
        }
        // Behind everything else, a wait may have run out here or in any product before: then no gradient is left that looks like one.
        if (p.last) {
            bool behind = false;
            if (threadIdx.x == 0) {
                __threadfence();
                behind = atomicAdd(&p.shared->joined, 1u) == gridDim.x - 1;
                __threadfence();
            }
            if (__syncthreads_or(behind) && *static_cast<volatile int*>(&p.shared->error)) {
                const uint16_t nan = BF16 ? 0x7FC0 : 0x7E00;
                for (int64_t r = warp; r < p.vocab; r += kThreads / 32)
                    for (int i = lane; i < p.width; i += 32) p.out[r * p.out_stride + i] = nan;
                for (int j = warp; p.hidden_out.part && j < active; j += kThreads / 32)
                    for (int i = lane; i < p.hidden_out.cols; i += 32) p.hidden_out.out[p.hidden_out.rows[j] * p.hidden_out.stride + i] = nan;
            }
        }
    }
    fence_before();
    cluster_sync();
    fence_after();
    if (warp == 2) tmem_free(tmem, 512);
}

// Forward of a few rows (cross entropy): the table's rows are the ones that go down the tile, 256 of them a pair, and the hidden states the columns,
// as many as there are, so that the matrix instructions cost what the rows ask for and not 256 of them.  A thread keeps maximum and sum of
// each of its columns over all its tiles and joins them with its warp's at the end.
//
// Bound by reading the table; stages of 20 KB leave room for ten of them on their way.  37 rows against 151,665 x 2048: 98 us, 6.4 TB/s, as a copy.
// With the rows down the tile it was 105 alone, and 130 in a loop, where 256 rows of products for 37 asked for more power than there is.
constexpr int kFewRows = 64, kFewStages = 10, kFewStageBytes = 16384 + kFewRows / 2 * 128;
constexpr int kFewSmem = 1024 + kFewStages * kFewStageBytes + 256;

struct Few {
    Shared* shared;
    int vocab, width, columns;       // columns: a multiple of 16
    int n_rows;
    const Entry* entry;
    float exponent;
    float2* partial;                 // of [pair, block, quarter of lanes][row]
    float* entry_logits;
};

template <bool BF16>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    few_kernel(const __grid_constant__ CUtensorMap map_weight, const __grid_constant__ CUtensorMap map_hidden, const __grid_constant__ Few p) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_addr(smem_raw) + 1023) & ~1023u;
    const uint32_t full = base + kFewStages * kFewStageBytes, empty = full + 8 * kFewStages, acc_full = empty + 8 * kFewStages, acc_empty = acc_full + 16,
                   tmem_at = acc_empty + 16;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    if (threadIdx.x == 0) {
        for (int s = 0; s < kFewStages; ++s) {
            bar_init(full + 8 * s, 1);
            bar_init(empty + 8 * s, 1);
        }
        for (int s = 0; s < 2; ++s) {
            bar_init(acc_full + 8 * s, 1);
            bar_init(acc_empty + 8 * s, 2 * kEpilogueWarps);
        }
        bar_init_fence();
    }
    if (warp == 2) tmem_alloc(tmem_at, 2 * kFewRows);
    __syncthreads();
    fence_before();
    cluster_sync();
    fence_after();
    uint32_t tmem;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(tmem) : "r"(tmem_at));
    after_previous();
    const int active = p.shared->active, pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    const int tiles = active ? (p.vocab + kTile - 1) / kTile : 0, blocks = (p.width + kDepth - 1) / kDepth;
    const int mine = p.columns / 2;          // of the columns: the rows of the hidden states that a block copies, and those that a warp takes out
    bool ok = true;

    if (warp == 0) {
        if (elect()) {
            const uint32_t full_of_pair = in_block(full, 0);
            uint32_t it = 0;
            for (int t = pair; t < tiles && ok; t += pairs) {
                const int row = t * kTile + rank * 128;
                for (int k = 0; k < blocks; ++k, ++it) {
                    const uint32_t s = it % kFewStages;
                    if (!bar_wait(empty + 8 * s, ((it / kFewStages) & 1) ^ 1)) { ok = false; break; }
                    const uint32_t a = base + s * kFewStageBytes, bar = full_of_pair + 8 * s;
                    if (rank == 0) bar_expect(full + 8 * s, 2 * 16384 + p.columns * 128);
                    load_tile(a, &map_weight, k * kDepth, row, bar);
                    load_tile(a + 8192, &map_weight, k * kDepth, row + 64, bar);
                    load_tile(a + 16384, &map_hidden, k * kDepth, rank * mine, bar);
                }
            }
            for (uint32_t i = it < kFewStages ? 0 : it - kFewStages; i < it && ok; ++i) ok = bar_wait(empty + 8 * (i % kFewStages), (i / kFewStages) & 1);
            if (!ok) {
                const uint64_t from = nanoseconds();
                while (nanoseconds() - from < 2000000ull) __nanosleep(1000);
            }
        }
    } else if (warp == 1) {
        if (rank == 0 && elect()) {
            const uint32_t kind = mma_kind(BF16, false, false, p.columns);
            uint32_t it = 0, acc = 0;
            for (int t = pair; t < tiles && ok; t += pairs, ++acc) {
                if (!bar_wait(acc_empty + 8 * (acc & 1), ((acc >> 1) & 1) ^ 1)) { ok = false; break; }
                fence_after();
                for (int k = 0; k < blocks; ++k, ++it) {
                    const uint32_t s = it % kFewStages;
                    if (!bar_wait(full + 8 * s, (it / kFewStages) & 1)) { ok = false; break; }
                    fence_after();
                    const uint32_t a = base + s * kFewStageBytes, b = a + 16384;
#pragma unroll
                    for (int j = 0; j < kDepth / 16; ++j)
                        mma(tmem + (acc & 1) * kFewRows, operand(a + j * 32, false), operand(b + j * 32, false), kind, k > 0 || j > 0);
                    mma_commit(empty + 8 * s);
                }
                if (ok) mma_commit(acc_full + 8 * (acc & 1));
            }
        }
    } else if (warp >= 4) {
        const int quarter = warp & 3, half = (warp - 4) >> 2, first = half * mine;
        float high[32], sum[32];
        int target[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            high[i] = -INFINITY;
            sum[i] = 0.f;
            target[i] = i < mine && first + i < active ? p.entry[first + i].id : INT_MAX;
        }
        uint32_t acc = 0;
        for (int t = pair; t < tiles; t += pairs, ++acc) {
            ok = __all_sync(~0u, bar_wait(acc_full + 8 * (acc & 1), (acc >> 1) & 1));
            if (!ok) break;
            fence_after();
            float v[32];
            tmem_load(tmem + (static_cast<uint32_t>(quarter * 32) << 16) + (acc & 1) * kFewRows + first, v);
            tmem_wait(v);
            fence_before();
            __syncwarp();
            if (lane == 0) bar_arrive_cluster(in_block(acc_empty + 8 * (acc & 1), 0));
            const int id = t * kTile + rank * 128 + quarter * 32 + lane;
            if (id < p.vocab) {
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    if (i >= mine) break;
                    if (target[i] == id) p.entry_logits[first + i] = v[i];
                    // in units of the maximum's rounded power, as in product_kernel
                    const float top = fmaxf(high[i], v[i]), from_top = top == -INFINITY ? 0.f : __fmul_rn(top, p.exponent);
                    sum[i] = sum[i] * exp2_fast(__fmul_rn(high[i], p.exponent) - from_top) + exp2_fast(fmaf(v[i], p.exponent, -from_top));
                    high[i] = top;
                }
            }
            __syncwarp();
        }
        if (pair < tiles) {
            float2* to = p.partial + static_cast<int64_t>((pair * 2 + rank) * 4 + quarter) * p.n_rows + first;
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                if (i >= mine) break;
                float top = high[i];
#pragma unroll
                for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
                float all = in_units(sum[i], __fmul_rn(high[i], p.exponent), top, p.exponent);
#pragma unroll
                for (int d = 16; d; d >>= 1) all += __shfl_xor_sync(~0u, all, d);
                if (lane == i) to[i] = make_float2(top, all);
            }
        }
    }
    if (!ok) atomicExch(&p.shared->error, 1);
    __syncwarp();
    let_next_begin();
    __syncthreads();
    fence_before();
    cluster_sync();
    fence_after();
    if (warp == 2) tmem_free(tmem, 2 * kFewRows);
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
// Maximum that keeps NaN.
__device__ __forceinline__ float max_nan(float a, float b) { return a != a || b != b ? a + b : fmaxf(a, b); }

constexpr int kNone = -1, kBad = -2;      // a row without a loss: nothing wanted of it; something beyond the vocabulary

// A teacher's rows: entries sorted by id (ties by place) with their softmax.  One block a row, a bitonic sort of id and place in shared memory; all
// latency: 301 rows of 20 entries 6 us, 2,048 of 64 9 us.
__global__ void teacher_kernel(Ids ids, Matrix logits, int entries, int room, int vocab, float inv_temperature, Entry* entry, int* state) {
    extern __shared__ uint8_t smem_raw[];
    uint64_t* key = reinterpret_cast<uint64_t*>(smem_raw);
    float* share = reinterpret_cast<float*>(key + room);
    __shared__ float red[32];
    __shared__ int bad;
    after_previous();
    let_next_begin();
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
        top = max_nan(top, l);
    }
    auto over_block = [&](float x, bool max_of) {
#pragma unroll
        for (int d = 16; d; d >>= 1) {
            const float y = __shfl_xor_sync(~0u, x, d);
            x = max_of ? max_nan(x, y) : x + y;
        }
        __syncthreads();
        if ((tid & 31) == 0) red[tid >> 5] = x;
        __syncthreads();
        x = red[0];
        for (int w = 1; w < (threads >> 5); ++w) x = max_of ? max_nan(x, red[w]) : x + red[w];
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
    for (int k = tid; k < entries; k += threads)
        entry[row * entries + k] = Entry{static_cast<int>(key[k] >> 32), share[static_cast<uint32_t>(key[k])] / sum};
    if (tid == 0) state[row] = bad ? kBad : none ? kNone : 0;
}

// Time in ns of the hidden gradient's part of a piece in `s` splits: `outs` tiles of it over `blocks` steps of the summed dimension.  A step
// of a tile takes 270, beginning and ending one 700, and each split costs its way to memory and back.  No more splits than make eight rounds of
// the pairs, and eight steps each: they would gain nothing, and their sums take room.  (The best of 32 is looked for, by a lane each.)
constexpr int kSplitRounds = 8;
__host__ __device__ inline int64_t split_time(int s, int64_t outs, int blocks, int pairs) {
    if (s > 1 && (s * 8 > blocks || outs * s > kSplitRounds * pairs)) return INT64_MAX;
    return (outs * s + pairs - 1) / pairs * (270 * blocks / s + 700) + 90 * s * outs;
}

// Lines of `cols` elements, eight at a time by the lanes of a warp; elements up to the next whole 16 bytes become 0, and all of them without `from`.
// `wide`: `from` begins at whole 16 bytes, and so do its lines.
__device__ __forceinline__ void copy_line(const uint16_t* from, int cols, bool wide, uint16_t* to, int to_cols) {
    const int lane = threadIdx.x & 31, lines = to_cols / 8;
    if (from && wide) {
        for (int i = lane; i < lines; i += 8 * 32) {
            uint4 v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (i + 32 * k < lines) v[k] = __ldg(reinterpret_cast<const uint4*>(from) + i + 32 * k);
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (i + 32 * k < lines) reinterpret_cast<uint4*>(to)[i + 32 * k] = v[k];
        }
        return;
    }
    for (int i = lane; i < lines; i += 32) {
        uint32_t w[4] = {0, 0, 0, 0};
        if (from)
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (8 * i + k < cols) w[k >> 1] |= static_cast<uint32_t>(from[8 * i + k]) << (16 * (k & 1));
        reinterpret_cast<uint4*>(to)[i] = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

struct RowsArgs {
    Ids targets;
    int64_t ignore;
    int vocab, n;
    int each;                    // rows a block
    const int* state;            // of a teacher's rows; NULL: from the targets
    const Entry* entry_from;     // of a teacher
    int entries;
    Entry* entry;                // the active rows' together
    int* rows;
    Shared* shared;
    float *losses, *lse;         // forward
    const uint16_t* src;         // hidden states
    int64_t stride;
    int cols;
    bool wide;
    uint16_t* dst;
    int dst_cols;

    // Target, 0 for a teacher's row, or what it has in place of a loss.
    __device__ __forceinline__ int of(int row) const {
        if (state) return state[row];
        const int64_t t = load_id(targets.data, targets.bits, row);
        return t < 0 || t == ignore ? kNone : t >= vocab ? kBad : static_cast<int>(t);
    }
};

// The rows that have a loss, together and in order, with their entries and places; behind their places those of the others.  Up to the next
// multiple of 64, in which they are read, there are lines of 0 behind them.  Each block counts the active rows before its own (at most kRowBlocks
// blocks do that, so it is never much), which takes less than a launch that counts for all: 37 rows, 9 -> 5 us.
constexpr int kRowBlocks = 2048;
__global__ void __launch_bounds__(256) rows_kernel(const __grid_constant__ RowsArgs a) {
    __shared__ int part[2][8];
    after_previous();
    let_next_begin();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int first = blockIdx.x * a.each, last = min(first + a.each, a.n);
    int before = 0, active = 0;
    for (int base = 0; base < a.n; base += 8 * 256) {
        int id[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) id[k] = base + k * 256 + tid < a.n ? a.of(base + k * 256 + tid) : kNone;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            active += id[k] >= 0;
            before += id[k] >= 0 && base + k * 256 + tid < first;
        }
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) {
        before += __shfl_xor_sync(~0u, before, d);
        active += __shfl_xor_sync(~0u, active, d);
    }
    if (lane == 0) {
        part[0][warp] = before;
        part[1][warp] = active;
    }
    __syncthreads();
    before = active = 0;
#pragma unroll
    for (int w = 0; w < 8; ++w) {
        before += part[0][w];
        active += part[1][w];
    }
    if (blockIdx.x == 0 && tid == 0) {
        Shared s{};
        s.active = active;
        *a.shared = s;
    }
    for (int base = first; base < last; base += 32) {
        const int own = base + lane < last ? a.of(base + lane) : kNone;
        const uint32_t live = __ballot_sync(~0u, own >= 0);
        for (int i = warp; i < 32 && base + i < last; i += 8) {
            const int row = base + i, id = __shfl_sync(~0u, own, i), to = before + __popc(live & ((1u << i) - 1));
            if (id >= 0) {
                copy_line(a.src + row * a.stride, a.cols, a.wide, a.dst + static_cast<int64_t>(to) * a.dst_cols, a.dst_cols);
                for (int k = lane; k < a.entries; k += 32) a.entry[static_cast<int64_t>(to) * a.entries + k] = a.entry_from[static_cast<int64_t>(row) * a.entries + k];
                if (lane == 0) {
                    a.rows[to] = row;
                    if (!a.state) a.entry[to] = Entry{id, 1.f};
                }
            } else if (lane == 0) {
                a.rows[a.n - 1 - (row - to)] = row;
                if (a.losses) {
                    a.losses[row] = id == kBad ? __int_as_float(0x7FC00000) : 0.f;
                    a.lse[row] = 0.f;
                }
            }
        }
        before += __popc(live);
    }
    for (int j = active + blockIdx.x * 8 + warp; j < (active + kDepth - 1) / kDepth * kDepth; j += gridDim.x * 8)
        copy_line(nullptr, a.cols, a.wide, a.dst + static_cast<int64_t>(j) * a.dst_cols, a.dst_cols);
}

// A table whose rows are no lines of whole 16 bytes, as such.  A warp a row.
__global__ void __launch_bounds__(256) table_kernel(const uint16_t* src, int64_t stride, int rows, int cols, uint16_t* dst, int dst_cols) {
    after_previous();
    let_next_begin();
    for (int64_t r = blockIdx.x * 8 + (threadIdx.x >> 5); r < rows; r += gridDim.x * 8) copy_line(src + r * stride, cols, false, dst + r * dst_cols, dst_cols);
}

struct ScaleArgs {
    const Shared* from;          // of the forward pass, or of what has just been prepared
    Shared* shared;
    const int* rows;
    RowInfo* info;
    const float *lse, *grad;
    int64_t grad_stride;
    bool grad_of_mean, half;
    float inv_temperature;
    int width_tiles, blocks, pairs;
    int entries;                 // of a teacher
    const Entry* entry;
};

constexpr int kScales = 8;

// The scale of the gradients, each active row's part of it, and the number of the hidden gradient's splits.  One block: 4 us for 1,021 rows, 9 for
// 8,192, a dozen reads one after the other.
__global__ void __launch_bounds__(1024) scale_kernel(const __grid_constant__ ScaleArgs a) {
    __shared__ float warp_top[32], warp_off[kScales][33], best_scale;
    after_previous();
    let_next_begin();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int active = a.from->active;
    float top = 0.f;
    for (int base = tid; base < active; base += 8 * 1024) {
        float g[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) g[i] = base + 1024 * i < active ? fabsf(a.grad[a.rows[base + 1024 * i] * a.grad_stride]) : 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, g[i] < INFINITY ? g[i] : 0.f);
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
    if (lane == 0) warp_top[warp] = top;
    __syncthreads();
    top = warp_top[lane];
#pragma unroll
    for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
    // dZ is kept with the largest row gradient as 1 (bf16: its range is fp32's) or as 2^15 (and less than twice that, see below), so that fp16
    // holds probabilities down to 2^-29 in full precision and nothing of 2^16 and more.  The largest of the finite ones: one that is not finite
    // is a matter of its own row, whose dZ it makes infinite or NaN.
    float unit = a.half ? 32768.f : 1.f;
    top = top < 0x1p-100f ? 0x1p-100f : top;
    if (a.entries) {
        // A teacher's large probabilities are much of dZ and often alike in all rows.  Of eight scales within a factor of 2 the one is taken
        // at which the first two thousand are rounded by the smallest steps (error of the gradients against
        // rounding them once: 1.3 to 1.6 times, then 1.2 to 1.4).
        const int some = static_cast<int>(min(static_cast<int64_t>(active) * a.entries, static_cast<int64_t>(2 * 1024)));
        float x[2], off[kScales] = {};
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int i = tid + 1024 * k;
            x[k] = i < some ? fabsf(a.grad[a.grad_stride ? a.rows[i / a.entries] * a.grad_stride : 0]) / top * a.entry[i].share : 0.f;
            x[k] = x[k] < INFINITY ? x[k] : 0.f;
        }
#pragma unroll
        for (int j = 0; j < kScales; ++j) {
            const float scale = exp2f(static_cast<float>(j) / kScales);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const float step = __uint_as_float(__float_as_uint(x[k] * scale) & 0x7F800000u) / scale;          // the power of 2 below, as the step's size goes
                off[j] += step * step;
            }
        }
#pragma unroll
        for (int j = 0; j < kScales; ++j) {
#pragma unroll
            for (int d = 16; d; d >>= 1) off[j] += __shfl_xor_sync(~0u, off[j], d);
            if (lane == 0) warp_off[j][warp] = off[j];
        }
        __syncthreads();
        if (warp == 0) {
            float all = INFINITY;
            if (lane < kScales) {
                all = 0.f;
                for (int w = 0; w < 32; ++w) all += warp_off[lane][w];
            }
            float least = all;
#pragma unroll
            for (int d = 16; d; d >>= 1) least = fminf(least, __shfl_xor_sync(~0u, least, d));
            const uint32_t which = __ballot_sync(~0u, all == least);
            if (lane == 0) best_scale = which ? exp2f(static_cast<float>(__ffs(which) - 1) / kScales) : 1.f;
        }
        __syncthreads();
        unit *= best_scale;
    }
    const float row_scale = unit / top;
    for (int base = tid; base < active; base += 8 * 1024) {
        RowInfo r[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (base + 1024 * i >= active) break;
            const int row = a.rows[base + 1024 * i];
            r[i] = RowInfo{a.lse[row] * kLog2e, a.grad[row * a.grad_stride] * row_scale};
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (base + 1024 * i < active) a.info[base + 1024 * i] = r[i];
    }
    if (warp) return;
    // each lane the time of one number of splits
    const int64_t time = split_time(lane + 1, static_cast<int64_t>((active + kTile - 1) / kTile) * a.width_tiles, a.blocks, a.pairs);
    int64_t least = time;
#pragma unroll
    for (int d = 16; d; d >>= 1) least = min(least, __shfl_xor_sync(~0u, least, d));
    const int splits = __ffs(__ballot_sync(~0u, time == least));
    if (lane == 0) {
        Shared s{};
        s.active = active;
        s.error = a.from->error;
        s.splits = splits;
        s.unscale = top / unit * a.inv_temperature / (a.grad_of_mean ? fmaxf(static_cast<float>(active), 1.f) : 1.f);
        *a.shared = s;
    }
}

// ---- and afterwards ---------------------------------------------------------------

struct JoinArgs {
    const float2* partial;
    int vocab, pairs, n_rows;
    bool few;                    // of few_kernel
    Shared* shared;
    const int* rows;
    int n, entries;
    const Entry* entry;
    const float* entry_logits;
    float exponent, inv_temperature;
    float *losses, *lse, *total;
    bool mean;
};

// Joins the half tiles' maxima and sums of 32 rows a block and takes the losses; the last block to end adds them up, in the same order always.
// Reads 16 bytes a tile and row: 25 us for 8,192 rows and 501 tiles, of 2.5 ms; 4 us behind the product for 37 rows.
__global__ void __launch_bounds__(1024) join_kernel(const __grid_constant__ JoinArgs a) {
    __shared__ float2 piece[32][33];
    __shared__ float red[32];
    __shared__ bool last;
    after_previous();
    let_next_begin();
    const int active = a.shared->active;
    const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
    const int tiles = (a.vocab + kTile - 1) / kTile, parts = a.few ? 8 * min(tiles, a.pairs) : 2 * (active > kTile ? tiles : min(tiles, a.pairs));
    for (int base = blockIdx.x * 32; base < active; base += gridDim.x * 32) {
        const int m = base + x, j = base + y;
        // what the second half of the work needs, on its way during the first
        Entry e{INT_MAX, 0.f};
        float logit = 0.f;
        int row = 0;
        if (j < active) {
            row = a.rows[j];
            if (x < a.entries) {
                e = a.entry[static_cast<int64_t>(j) * a.entries + x];
                logit = a.entry_logits[static_cast<int64_t>(j) * a.entries + x];
            }
        }
        float high = -INFINITY, sum = 0.f;
        if (m < active) {
            for (int k = y; k < parts; k += 32 * 8) {
                float2 v[8];
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    v[i] = k + 32 * i < parts ? a.partial[static_cast<int64_t>(k + 32 * i) * a.n_rows + m] : make_float2(-INFINITY, 0.f);
                float top = high;
#pragma unroll
                for (int i = 0; i < 8; ++i) top = fmaxf(top, v[i].x);
                const float ref = top == -INFINITY ? 0.f : top;
                sum *= exp2_fast((high - ref) * a.exponent);
#pragma unroll
                for (int i = 0; i < 8; ++i) sum += v[i].y * exp2_fast((v[i].x - ref) * a.exponent);
                high = top;
            }
        }
        __syncthreads();
        piece[y][x] = make_float2(high, sum);
        __syncthreads();
        // a warp a row, its 32 parts beside one another
        const float2 v = piece[x][y];
        float top = v.x;
#pragma unroll
        for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
        const float ref = top == -INFINITY ? 0.f : top;
        float total = v.y * exp2_fast((v.x - ref) * a.exponent);
#pragma unroll
        for (int d = 16; d; d >>= 1) total += __shfl_xor_sync(~0u, total, d);
        const float row_lse = ref * a.inv_temperature + logf(total);
        if (j < active) {
            float loss = 0.f;
            for (int i = x; i < a.entries; i += 32) {
                if (i >= 32) {
                    e = a.entry[static_cast<int64_t>(j) * a.entries + i];
                    logit = a.entry_logits[static_cast<int64_t>(j) * a.entries + i];
                }
                if (e.id != INT_MAX && e.share != 0.f) loss += e.share * (logf(e.share) + (row_lse - logit * a.inv_temperature));
            }
#pragma unroll
            for (int d = 16; d; d >>= 1) loss += __shfl_xor_sync(~0u, loss, d);
            if (x == 0) {
                a.losses[row] = a.shared->error ? __int_as_float(0x7FC00000) : loss;
                a.lse[row] = a.shared->error ? __int_as_float(0x7FC00000) : row_lse;
            }
        }
    }
    if (!a.total) return;
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) last = atomicAdd(&a.shared->joined, 1u) == gridDim.x - 1;
    __syncthreads();
    if (!last) return;
    __threadfence();
    float sum = 0.f;
    for (int i = threadIdx.x; i < a.n; i += 1024) sum += __ldcg(a.losses + i);
#pragma unroll
    for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(~0u, sum, d);
    if (x == 0) red[y] = sum;
    __syncthreads();
    if (y) return;
    sum = red[x];
#pragma unroll
    for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(~0u, sum, d);
    if (x == 0) *a.total = a.mean ? sum / fmaxf(static_cast<float>(active), 1.f) : sum;
}

// The hidden gradient where the table's product does not finish it.
template <bool BF16>
__global__ void __launch_bounds__(256) hidden_grad_kernel(const __grid_constant__ HiddenOut h, const Shared* shared) {
    after_previous();
    finish_hidden<BF16>(h, shared, static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x, static_cast<int64_t>(gridDim.x) * 256);
}

// ---- host -------------------------------------------------------------------------

inline int64_t round_up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }
inline int64_t div_up(int64_t x, int64_t by) { return (x + by - 1) / by; }

int multiprocessors() {
    int device = 0, count = 148;
    if (cudaGetDevice(&device) == cudaSuccess) cudaDeviceGetAttribute(&count, cudaDevAttrMultiProcessorCount, device);
    return count;
}

struct Plan {
    int n, n_rows, vocab, width, cols, entries;     // cols: width in whole 16 bytes
    int pairs;
    bool copy_weight;
    int piece;                                      // backward: columns a piece
    int64_t sum_rows;                               // rows of the hidden gradient's parts, however many rows are active
    // what a forward pass may leave for the backward one
    uint64_t shared, rows, entry, hidden, kept_bytes;
    // and the rest of the workspace
    uint64_t entry_raw, state, info, own_shared, entry_logits, weight, partial, delta, sums, bytes;
};

// Of a piece's dZ.  Each piece adds its part to the hidden gradient's sums, and at its ends pairs wait for the last: 8,192 rows against 128,256 x
// 2048 take 12.0 ms with 64 MiB, 11.9 with 128, 11.0 with 256, 10.8 with 512.
constexpr int64_t kDeltaBytes = 512 << 20;

Plan make_plan(const LossCall& c, bool backward) {
    Plan p{};
    p.n = static_cast<int>(c.hidden.rows);
    p.n_rows = static_cast<int>(round_up(c.hidden.rows, kTile));
    p.vocab = static_cast<int>(c.weight.rows);
    p.width = static_cast<int>(c.hidden.cols);
    p.cols = static_cast<int>(round_up(p.width, 8));
    p.entries = c.entries ? c.entries : 1;
    p.pairs = multiprocessors() / 2;
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
    p.entry = take(sizeof(Entry) * listed);
    p.hidden = take(2ull * p.n_rows * p.cols);
    p.kept_bytes = at;
    if (c.kept) at = 0;
    if (c.entries && !(backward && c.kept)) {
        p.entry_raw = take(sizeof(Entry) * listed);
        p.state = take(4ull * p.n);
    }
    if (p.copy_weight) p.weight = take(2ull * p.vocab * p.cols);
    const int64_t tiles = div_up(p.vocab, kTile);
    if (!backward) {
        p.entry_logits = take(4ull * listed);
        p.partial = take(8ull * std::max<int64_t>(2 * tiles, 8 * p.pairs) * p.n_rows);
    } else {
        p.own_shared = take(sizeof(Shared));
        p.info = take(sizeof(RowInfo) * p.n);
        const int64_t room = std::max<int64_t>(1, kDeltaBytes / (2ll * kTile * p.n_rows));
        p.piece = static_cast<int>(div_up(tiles, div_up(tiles, room)) * kTile);
        const int64_t width_tiles = div_up(p.cols, kTile);
        p.sum_rows = std::max<int64_t>(p.n_rows, kSplitRounds * p.pairs / width_tiles * kTile);
        p.delta = take(2ull * p.n_rows * p.piece);
        p.sums = take(4ull * p.sum_rows * p.cols);
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
cudaError_t launch_product(bool bf16, int pairs, const CUtensorMap& a, const CUtensorMap& b, const CUtensorMap& out, const Product& p, cudaStream_t stream) {
    auto* kernel = bf16 ? product_kernel<MODE, true> : product_kernel<MODE, false>;
    if (cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes(MODE))) return e;
    return launch(kernel, 2 * pairs, kThreads, smem_bytes(MODE), stream, a, b, out, p);
}

struct Prepared {
    Plan plan;
    char *at, *kept;
    Shared* shared;
    int* rows;
    Entry* entry;
    uint16_t* hidden;
    const void* weight;
    int64_t weight_stride;
};

const char* cuda_error(cudaError_t e) { return e == cudaSuccess ? nullptr : cudaGetErrorString(e); }

// Addresses in the workspace; the table copied where its rows are no lines of whole 16 bytes; and, unless `given`, the active rows.
cudaError_t prepare(const LossCall& c, bool backward, bool given, Prepared& w) {
    const Plan& p = w.plan;
    w.at = static_cast<char*>(c.workspace);
    w.kept = c.kept ? static_cast<char*>(c.kept) : w.at;
    w.shared = reinterpret_cast<Shared*>(w.kept + p.shared);
    w.rows = reinterpret_cast<int*>(w.kept + p.rows);
    w.entry = reinterpret_cast<Entry*>(w.kept + p.entry);
    w.hidden = reinterpret_cast<uint16_t*>(w.kept + p.hidden);
    w.weight = c.weight.data;
    w.weight_stride = c.weight.stride;
    if (p.copy_weight) {
        uint16_t* copy = reinterpret_cast<uint16_t*>(w.at + p.weight);
        if (cudaError_t e = launch(table_kernel, std::min<int64_t>(div_up(p.vocab, 8), 148 * 8), 256, 0, c.stream, static_cast<const uint16_t*>(w.weight), w.weight_stride,
                                   p.vocab, p.width, copy, p.cols))
            return e;
        w.weight = copy;
        w.weight_stride = p.cols;
    }
    if (given) return cudaSuccess;
    Entry* entry_raw = reinterpret_cast<Entry*>(w.at + p.entry_raw);
    int* state = reinterpret_cast<int*>(w.at + p.state);
    if (c.entries) {
        int room = 2;
        while (room < c.entries) room *= 2;
        if (cudaError_t e = launch(teacher_kernel, p.n, std::min(256, std::max(32, room / 2)), room * 12, c.stream, c.targets, c.teacher, c.entries, room, p.vocab,
                                   1.f / c.temperature, entry_raw, state))
            return e;
    }
    RowsArgs r{};
    r.targets = c.targets;
    r.ignore = c.ignore;
    r.vocab = p.vocab;
    r.n = p.n;
    r.each = static_cast<int>(std::max<int64_t>(8, div_up(p.n, kRowBlocks)));
    r.state = c.entries ? state : nullptr;
    r.entry_from = entry_raw;
    r.entries = c.entries;
    r.entry = w.entry;
    r.rows = w.rows;
    r.shared = w.shared;
    r.losses = backward ? nullptr : c.losses;
    r.lse = backward ? nullptr : c.lse;
    r.src = static_cast<const uint16_t*>(c.hidden.data);
    r.stride = c.hidden.stride;
    r.cols = p.width;
    r.wide = p.width % 8 == 0 && c.hidden.stride % 8 == 0 && reinterpret_cast<uintptr_t>(c.hidden.data) % 16 == 0;
    r.dst = w.hidden;
    r.dst_cols = p.cols;
    return launch(rows_kernel, div_up(p.n, r.each), 256, 0, c.stream, r);
}

Product product_of(const LossCall& c, const Prepared& w) {
    Product q{};
    q.shared = w.shared;
    q.n_rows = w.plan.n_rows;
    q.vocab = w.plan.vocab;
    q.width = w.plan.cols;
    q.count = w.plan.vocab;
    q.entries = w.plan.entries;
    q.entry = w.entry;
    q.exponent = kLog2e / c.temperature * cut_off(w.plan.width);
    return q;
}

}  // namespace

uint64_t loss_workspace(const LossCall& c, bool backward) { return c.hidden.rows ? make_plan(c, backward).bytes : 0; }
uint64_t loss_kept(const LossCall& c) { return c.hidden.rows ? make_plan(c, false).kept_bytes : 0; }

const char* loss_forward(const LossCall& c) {
    if (c.hidden.rows == 0) return c.total ? cuda_error(cudaMemsetAsync(c.total, 0, 4, c.stream)) : nullptr;
    if (!encode_fn()) return "the driver has no tiled copies";
    Prepared w;
    w.plan = make_plan(c, false);
    const Plan& p = w.plan;
    if (cudaError_t e = prepare(c, false, false, w)) return cuda_error(e);
    Product q = product_of(c, w);
    q.partial = reinterpret_cast<float2*>(w.at + p.partial);
    q.entry_logits = reinterpret_cast<float*>(w.at + p.entry_logits);
    const bool bf16 = c.hidden.type == kBF16, few = p.n <= kFewRows && !c.entries;
    const int columns = static_cast<int>(round_up(p.n, 16));
    CUtensorMap hidden_map, weight_map;
    if (!tile_map(&hidden_map, c.hidden.type, w.hidden, p.n_rows, p.cols, p.cols, few ? columns / 2 : 64) ||
        !tile_map(&weight_map, c.hidden.type, w.weight, p.vocab, p.cols, w.weight_stride, 64))
        return "a tensor map was refused";
    if (few) {
        Few f{};
        f.shared = q.shared;
        f.vocab = q.vocab;
        f.width = q.width;
        f.columns = columns;
        f.n_rows = q.n_rows;
        f.entry = q.entry;
        f.exponent = q.exponent;
        f.partial = q.partial;
        f.entry_logits = q.entry_logits;
        auto* kernel = bf16 ? few_kernel<true> : few_kernel<false>;
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kFewSmem);
        if (e == cudaSuccess) e = launch(kernel, 2 * p.pairs, kThreads, kFewSmem, c.stream, weight_map, hidden_map, f);
        if (e != cudaSuccess) return cuda_error(e);
    } else if (cudaError_t e = launch_product<kForward>(bf16, p.pairs, hidden_map, weight_map, hidden_map, q, c.stream)) {
        return cuda_error(e);
    }
    JoinArgs j{};
    j.partial = q.partial;
    j.vocab = p.vocab;
    j.pairs = p.pairs;
    j.few = few;
    j.n_rows = p.n_rows;
    j.shared = w.shared;
    j.rows = w.rows;
    j.n = p.n;
    j.entries = p.entries;
    j.entry = q.entry;
    j.entry_logits = q.entry_logits;
    j.exponent = q.exponent;
    j.inv_temperature = 1.f / c.temperature * cut_off(p.width);
    j.losses = c.losses;
    j.lse = c.lse;
    j.total = c.total;
    j.mean = c.mean;
    return cuda_error(launch(join_kernel, std::min<int64_t>(div_up(p.n, 32), 148 * 2), 1024, 0, c.stream, j));
}

const char* loss_backward(const LossCall& c) {
    const bool bf16 = c.hidden.type == kBF16;
    if (c.hidden.rows == 0) {
        if (!c.d_weight.data) return nullptr;
        return cuda_error(cudaMemset2DAsync(const_cast<void*>(c.d_weight.data), c.d_weight.stride * 2, 0, c.d_weight.cols * 2, c.d_weight.rows, c.stream));
    }
    if (!encode_fn()) return "the driver has no tiled copies";
    Prepared w;
    w.plan = make_plan(c, true);
    const Plan& p = w.plan;
    if (cudaError_t e = prepare(c, true, c.kept != nullptr, w)) return cuda_error(e);
    uint16_t* delta = reinterpret_cast<uint16_t*>(w.at + p.delta);
    float* sums = reinterpret_cast<float*>(w.at + p.sums);
    uint16_t* d_weight = static_cast<uint16_t*>(const_cast<void*>(c.d_weight.data));
    const bool direct = d_weight && (p.width % 8 || c.d_weight.stride % 8 || reinterpret_cast<uintptr_t>(d_weight) % 16);
    // operands come in boxes of 64 lines, results leave in boxes of 32
    CUtensorMap hidden_map, weight_map, delta_map, delta_out, sums_out, weight_out;
    if (!tile_map(&hidden_map, c.hidden.type, w.hidden, p.n_rows, p.cols, p.cols, 64) ||
        !tile_map(&weight_map, c.hidden.type, w.weight, p.vocab, p.cols, w.weight_stride, 64) ||
        !tile_map(&delta_map, c.hidden.type, delta, p.n_rows, p.piece, p.piece, 64) || !tile_map(&delta_out, c.hidden.type, delta, p.n_rows, p.piece, p.piece, 32) ||
        !tile_map(&sums_out, kF32, sums, p.sum_rows, p.cols, p.cols, 32))
        return "a tensor map was refused";
    if (d_weight && !direct) {
        if (!tile_map(&weight_out, c.hidden.type, d_weight, p.vocab, p.width, c.d_weight.stride, 32)) return "a tensor map was refused";
    } else {
        weight_out = delta_out;
    }
    ScaleArgs a{};
    a.from = w.shared;
    a.shared = reinterpret_cast<Shared*>(w.at + p.own_shared);
    a.rows = w.rows;
    a.info = reinterpret_cast<RowInfo*>(w.at + p.info);
    a.lse = c.lse;
    a.grad = c.grad;
    a.grad_stride = c.grad_stride;
    a.grad_of_mean = c.mean;
    a.half = !bf16;
    a.inv_temperature = 1.f / c.temperature;
    a.width_tiles = static_cast<int>(div_up(p.cols, kTile));
    a.blocks = p.piece / kDepth;
    a.pairs = p.pairs;
    a.entries = c.entries;
    a.entry = w.entry;
    if (cudaError_t e = launch(scale_kernel, 1, 1024, 0, c.stream, a)) return cuda_error(e);
    HiddenOut h{};
    if (c.d_hidden.data) {
        h.part = sums;
        h.part_cols = p.cols;
        h.rows = w.rows;
        h.n = p.n;
        h.cols = p.width;
        h.out = static_cast<uint16_t*>(const_cast<void*>(c.d_hidden.data));
        h.stride = c.d_hidden.stride;
        h.wide = p.width % 8 == 0 && h.stride % 8 == 0 && reinterpret_cast<uintptr_t>(h.out) % 16 == 0;
    }
    // A small hidden gradient is finished by idle warps of the last product, which hides it (6 to 8 us of 280); a large one takes those few
    // warps longer than the product (4,099 x 1024 in 5 splits: 40 us more than the kernel of its own, which takes 8).
    const int64_t lines = static_cast<int64_t>(p.n) * div_up(p.width, 8);
    const bool within = d_weight && lines <= 16ll * 64 * 2 * p.pairs;
    for (int first = 0; first < p.vocab; first += p.piece) {
        Product q = product_of(c, w);
        q.shared = a.shared;
        q.info = a.info;
        q.first = first;
        q.count = std::min(p.piece, p.vocab - first);
        if (cudaError_t e = launch_product<kDelta>(bf16, p.pairs, hidden_map, weight_map, delta_out, q, c.stream)) return cuda_error(e);
        if (c.d_hidden.data) {
            q.add = first > 0;
            if (cudaError_t e = launch_product<kHiddenGrad>(bf16, p.pairs, delta_map, weight_map, sums_out, q, c.stream)) return cuda_error(e);
        }
        if (d_weight) {
            q.direct = direct;
            q.out = d_weight;
            q.out_stride = c.d_weight.stride;
            q.width = p.width;
            q.last = first + p.piece >= p.vocab;
            if (within && q.last) q.hidden_out = h;
            if (cudaError_t e = launch_product<kWeightGrad>(bf16, p.pairs, delta_map, hidden_map, weight_out, q, c.stream)) return cuda_error(e);
        }
    }
    if (!c.d_hidden.data || within) return nullptr;
    return cuda_error(launch(bf16 ? hidden_grad_kernel<true> : hidden_grad_kernel<false>, std::min<int64_t>(div_up(lines, 512), 148 * 16), 256, 0, c.stream, h, a.shared));
}

}  // namespace gtok
