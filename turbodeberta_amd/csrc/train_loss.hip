// Softmax cross entropy over a vocabulary, from hidden states and the output layer's weights, with its gradient; the logits are never in memory.
//
//   s_rv = x_r . W_v + b_v,  loss_r = log sum_v exp s_rv - s_r,label
//   D_rv = exp(s_rv) / sum_v exp s_rv - [v = label],  dx_r = g_r sum_v D_rv W_v,  dW_v = sum_r g_r D_rv x_r,  db_v = sum_r g_r D_rv
//
// Only rows that have a label count (15 % of them in masked language modelling).  The first kernel gathers them, in order; how many they are is known on the device only, so
// the others have a workgroup for each CU, which takes tile after tile of what there is.  Forward, a tile's logits leave as a maximum and a sum of exponentials
// for each row; backward they are made again, and D goes to a workspace in the type of the matrix instructions, at most 2 GiB of it at a time (a piece of the
// vocabulary): both gradients read it.  Sums of dx over the vocabulary are split over the workgroups and added up in a fixed order: no atomics, the same bits every time.
#include <algorithm>
#include <atomic>
#include <cfloat>
#include <cmath>

#include "tdb_error.h"
#include "train_product.h"

namespace tdb_train {

constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.693147180559945309417f;
constexpr int TILE = 256;           // what rows and columns of the buffers are rounded up to
constexpr int FINISH_ROWS = 32;     // rows of a workgroup of the last forward kernel
constexpr int FEW = 1024;           // rows up to which tiles may be lower than 256; all of them where there are few tiles

// Rows of a tile where n count: the height by which the busiest of `blocks` workgroups has least to do, tiles at their price; `wide` tiles lie beside each other.  16 bits, 128100 x 768: a tile's
// logits and their gradient took 125 us for 256 rows, 70 to 77 for 128, 48 for 64, 31 for 32 (lower tiles load more for their products).  float32, bound by products, 765 for 256, 514 for 160,
// 414 for 128, 336 for 96, 240 for 64, 135 for 32: 96 rows 382 us in one tile and 529 in two of 64, 160 rows 524 in one and 667 in five of 32; up to 16 rows have a tile
// of their own: 1, 43175 x 1060, 67 + 56 us in 32 rows, 67 + 43 in 16.  Where tiles are few, low ones share out better:
// 141 rows, 18134 classes, 704 columns of bfloat16 take 51 us in 71 tiles of 256 rows and 31 in 213 of 64.  (No tiles past the rows' multiple of 256, which the buffers have.)
template <int DT>
__device__ __forceinline__ int tile_rows(int n, int least, uint32_t wide, uint32_t blocks, int64_t few) {
    if (n > few) return TILE;
    auto cost = [&](int h, int dear) { return float((uint32_t(n + h - 1) / uint32_t(h) * wide + blocks - 1) / blocks) * float(h * dear); };
    constexpr int HEIGHTS[] = {160, 128, 96, 64, 32, 16}, DEAR[] = {DT == TDB_F32 ? 34 : 0, DT == TDB_F32 ? 35 : 40, DT == TDB_F32 ? 37 : 0, DT == TDB_F32 ? 40 : 52, DT == TDB_F32 ? 45 : 64, DT == TDB_F32 ? 60 : 0};
    int best = TILE;
    float least_cost = cost(TILE, 32);
#pragma unroll
    for (int i = 0; i < 6; ++i) {
        const int h = HEIGHTS[i];
        const float c = cost(h, DEAR[i]);
        if (DEAR[i] && h >= least && (h > 16 || n <= 16) && (n + h - 1) / h * h <= (n + TILE - 1) / TILE * TILE && c < least_cost) best = h, least_cost = c;
    }
    return best;
}

// float16: D lies in [-2^14, 2^14] (twice that with gradients of the rows' own), so that probabilities down to 2^-38 are told from 0 (2^-24 without).
template <int DT>
constexpr float D_SCALE = DT == TDB_F16 ? 16384.f : 1.f;

struct Loss {
    const char *x, *w;
    const void* bias;
    const int64_t* labels;
    int64_t rows, vocab, ignore, x_stride, w_pitch;
    int32_t hidden, reduction, bias_kind;       // 0: none, 1: as x, 2: float32
    float* loss;
    // state: count[0] rows that count, count[1] workgroups that are done
    int32_t *count, *index, *place, *label;     // of the gathered rows: row, label; of the rows: their place among the gathered ones
    float* biases;                              // of all classes, -inf behind them up to a multiple of TILE
    float *top, *inverse, *right;               // largest logit, 1 / sum of exponentials relative to it, the label's logit
    char* gathered;
    int64_t pitch;                              // of a gathered row, bytes
    // workspace
    float *maxima, *sums;                       // [groups of column tiles][rows]
    double* block_sums;
    int64_t padded;                             // rows, rounded up
    int32_t group, few_width;                   // column tiles that a workgroup of the kernel for many rows takes together; columns of the tiles of the one for few
    int32_t blocks;                             // workgroups of the kernel for many rows
    int64_t few_rows;                           // rows up to which tiles may be lower than 256
    __device__ __forceinline__ int64_t dw_rows() const { return (vocab + TILE - 1) / TILE * TILE; }
    template <int DT>
    __device__ __forceinline__ int rows_of(int n) const { return tile_rows<DT>(n, 16, uint32_t(vocab + few_width - 1) / uint32_t(few_width), blocks, few_rows); }       // of a tile of logits
};

// How the logits' maxima and sums lie: groups of column tiles, rows `pitch` to each.
struct Partials {
    int64_t groups, tiles, group, pitch;
    __device__ __forceinline__ Partials(const Loss& p, bool many) : tiles(many ? (p.vocab + TILE - 1) / TILE : (p.vocab + p.few_width - 1) / p.few_width), group(many ? p.group : 1), pitch(many ? p.padded : p.few_rows) {
        groups = (tiles + group - 1) / group;
    }
};

// The bias of a class, -inf past the vocabulary.  As it is, a mask of float32's lowest value among them: logits are subtracted before they are scaled to base 2, so a difference of two of them is 0, one from an
// ordinary logit the mask itself, whose exponential is 0, and a label's loss there the mask's size.
template <int DT>
__device__ __forceinline__ float bias_of(const Loss& p, int64_t v) {
    if (v >= p.vocab) return -INFINITY;
    if (!p.bias_kind) return 0.f;
    return p.bias_kind == 2 ? static_cast<const float*>(p.bias)[v] : float(static_cast<const typename Matrix<DT>::T*>(p.bias)[v]);
}

template <int WAVES>
__device__ __forceinline__ int block_count(int x, int* scratch) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) x += __shfl_xor(x, d);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = x;
    __syncthreads();
    int all = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) all += scratch[w];
    return all;
}

constexpr int GATHER_WAVES = 8, GATHER_ROWS = 4;       // rows that a wave copies at once

// Rows that count, in order: where they come from, their labels, and they themselves, dense, zeros behind them up to a multiple of the steps' 128 bytes.
// A workgroup has `chunk` rows and counts for itself what lies in front of them.  Workgroups from row_blocks on write the biases as the other kernels take them.
template <int DT>
__global__ __launch_bounds__(64 * GATHER_WAVES) void loss_gather_kernel(Loss p, int64_t chunk, int row_blocks, bool wide) {
    using T = typename Matrix<DT>::T;
    constexpr int THREADS = 64 * GATHER_WAVES, U = 8;
    if (int(blockIdx.x) >= row_blocks) {
        const int64_t v = (int64_t(blockIdx.x) - row_blocks) * (4 * THREADS) + 4 * threadIdx.x;
        if (v < (p.vocab + TILE - 1) / TILE * TILE) *reinterpret_cast<f32x4*>(p.biases + v) = f32x4{bias_of<DT>(p, v), bias_of<DT>(p, v + 1), bias_of<DT>(p, v + 2), bias_of<DT>(p, v + 3)};
        return;
    }
    __shared__ int scratch[GATHER_WAVES];
    const int wave = threadIdx.x >> 6, l = threadIdx.x & 63;
    const int64_t first = blockIdx.x * chunk, end = min(p.rows, first + chunk);
    int seen = 0;
    for (int64_t i = threadIdx.x; i < first; i += THREADS * U) {
        int64_t label[U];
#pragma unroll
        for (int u = 0; u < U; ++u) label[u] = p.labels[min(i + THREADS * u, first - 1)];
#pragma unroll
        for (int u = 0; u < U; ++u) seen += i + THREADS * u < first && label[u] != p.ignore;
    }
    const int before = block_count<GATHER_WAVES>(seen, scratch);
    int at = before;
    for (int64_t i0 = first; i0 < end; i0 += THREADS) {
        const int64_t i = i0 + threadIdx.x;
        const int64_t label = i < end ? p.labels[i] : p.ignore;
        const bool counts = label != p.ignore;
        const uint64_t who = __builtin_amdgcn_ballot_w64(counts);
        __syncthreads();
        if (l == 0) scratch[wave] = __popcll(who);
        __syncthreads();
        int place = at + __popcll(who & ((uint64_t(1) << l) - 1)), all = 0;
#pragma unroll
        for (int v = 0; v < GATHER_WAVES; ++v) place += v < wave ? scratch[v] : 0, all += scratch[v];
        at += all;
        if (i < end) {
            p.place[i] = counts ? place : -1;
            if (counts) {
                p.index[place] = int32_t(i);
                p.label[place] = label >= 0 && label < p.vocab ? int32_t(label) : -1;
                p.right[place] = __builtin_nanf("");        // (stays for a label that is none)
            } else if (p.reduction == 0) {
                p.loss[i] = 0.f;
            }
        }
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) p.count[1] = 0;
    if (int(blockIdx.x) == row_blocks - 1 && threadIdx.x == 0) p.count[0] = at;
    __syncthreads();
    const int columns = int(p.pitch / sizeof(T));
    for (int r0 = before + wave * GATHER_ROWS; r0 < at; r0 += GATHER_WAVES * GATHER_ROWS) {
        const T* from[GATHER_ROWS];
#pragma unroll
        for (int u = 0; u < GATHER_ROWS; ++u) from[u] = reinterpret_cast<const T*>(p.x) + p.index[min(r0 + u, at - 1)] * p.x_stride;
        if (wide) {
            constexpr int PER = 16 / sizeof(T);
            for (int c = l; c < columns / PER; c += 64) {
                uint4 v[GATHER_ROWS];
#pragma unroll
                for (int u = 0; u < GATHER_ROWS; ++u) v[u] = c * PER < p.hidden ? reinterpret_cast<const uint4*>(from[u])[c] : uint4{0, 0, 0, 0};
#pragma unroll
                for (int u = 0; u < GATHER_ROWS; ++u)
                    if (r0 + u < at) reinterpret_cast<uint4*>(p.gathered + (r0 + u) * p.pitch)[c] = v[u];
            }
        } else {
            for (int c0 = l; c0 < columns; c0 += 64 * U) {
                T v[U][GATHER_ROWS];
#pragma unroll
                for (int k = 0; k < U; ++k)
#pragma unroll
                    for (int u = 0; u < GATHER_ROWS; ++u) v[k][u] = c0 + 64 * k < p.hidden ? from[u][c0 + 64 * k] : T(0.f);
#pragma unroll
                for (int k = 0; k < U; ++k)
#pragma unroll
                    for (int u = 0; u < GATHER_ROWS; ++u)
                        if (r0 + u < at && c0 + 64 * k < columns) reinterpret_cast<T*>(p.gathered + (r0 + u) * p.pitch)[c0 + 64 * k] = v[k][u];
            }
        }
    }
}

// The operands of a tile's logits.
template <int DT>
__device__ __forceinline__ Rows hidden_rows(const Loss& p, int n) { return {p.gathered, p.pitch, n, uint32_t(p.pitch)}; }
template <int DT>
__device__ __forceinline__ Rows weight_rows(const Loss& p) { return {p.w, p.w_pitch, p.vocab, uint32_t(p.hidden * sizeof(typename Matrix<DT>::T))}; }

// A tile's logits: the sums start from the biases.
template <int DT, class P>
__device__ __forceinline__ void logits_of(const Loss& p, typename P::Flow& flow, float* s_bias, int64_t m0, int64_t n0, typename P::Acc& acc) {
    __syncthreads();                        // (the biases of the tile before have been read)
    if (threadIdx.x < P::BN) s_bias[threadIdx.x] = p.biases[n0 + threadIdx.x];
    __syncthreads();
    P::run(flow, {m0, n0, 0, p.pitch / P::LINE_BYTES}, acc,
           [&](int j, int q) { return *reinterpret_cast<const f32x4*>(s_bias + P::wave_n() + j * Matrix<DT>::SIDE + quad_n<DT>(q)); });
}

// Forward: of each gathered row and group of column tiles the largest logit and the sum of exponentials relative to it.
template <int DT, class P>
struct Running {
    using M = Matrix<DT>;
    float top[P::TM], sum[P::TM];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < P::TM; ++i) top[i] = -FLT_MAX, sum[i] = 0.f;
    }
    // labels: of the tile's rows
    __device__ __forceinline__ void add(const Loss& p, int n, const typename P::Acc& acc, int64_t m0, int64_t n0, const int32_t* labels) {
#pragma unroll
        for (int i = 0; i < P::TM; ++i) {
            float most = top[i];
#pragma unroll
            for (int j = 0; j < P::TN; ++j)
#pragma unroll
                for (int e = 0; e < 4 * M::QUADS; ++e) most = fmaxf(most, acc[i][j][e]);
            float more[2] = {0.f, 0.f};
#pragma unroll
            for (int j = 0; j < P::TN; ++j)
#pragma unroll
                for (int e = 0; e < 4 * M::QUADS; ++e) more[e & 1] += __builtin_amdgcn_exp2f((acc[i][j][e] - most) * LOG2E);
            sum[i] = sum[i] * __builtin_amdgcn_exp2f((top[i] - most) * LOG2E) + (more[0] + more[1]);
            top[i] = most;
            // The label's own logit, in the one tile that has it: row after row, the value's place is the same for all lanes.
            const int at = P::wave_m() + i * M::SIDE + lane_m<DT>();
            const int rel = m0 + at < n ? labels[at] - int(n0) - P::wave_n() : -1;
            const bool here = rel >= 0 && rel < P::COLUMNS && n0 + P::wave_n() + rel < p.vocab;
            for (uint64_t who = __builtin_amdgcn_ballot_w64(here) & (~uint64_t(0) >> (64 - M::SIDE)); who; who &= who - 1) {
                const int lane = __builtin_ctzll(who), c = __builtin_amdgcn_readlane(rel, lane);
#pragma unroll
                for (int j = 0; j < P::TN; ++j)
#pragma unroll
                    for (int e = 0; e < 4 * M::QUADS; ++e)
                        if ((threadIdx.x & (M::SIDE - 1)) == lane && c == j * M::SIDE + quad_n<DT>(e / 4) + e % 4) p.right[m0 + at] = acc[i][j][e];
            }
        }
    }
    // All waves' together, to memory.  s_top, s_sum: WN * BM each.
    __device__ __forceinline__ void finish(float* s_top, float* s_sum, float* maxima, float* sums) {
#pragma unroll
        for (int i = 0; i < P::TM; ++i) {
            const float most = over_quads<DT>(top[i], [](float x, float y) { return fmaxf(x, y); });
            const float s = over_quads<DT>(sum[i] * __builtin_amdgcn_exp2f((top[i] - most) * LOG2E), [](float x, float y) { return x + y; });
            const int at = P::wave_n() / P::COLUMNS * P::BM + P::wave_m() + i * M::SIDE + lane_m<DT>();
            s_top[at] = most, s_sum[at] = s;
        }
        step_barrier();
        if (threadIdx.x < P::BM) {
            float most = s_top[threadIdx.x], s = 0.f;
#pragma unroll
            for (int w = 1; w < P::WN; ++w) most = fmaxf(most, s_top[w * P::BM + threadIdx.x]);
#pragma unroll
            for (int w = 0; w < P::WN; ++w) s += s_sum[w * P::BM + threadIdx.x] * __builtin_amdgcn_exp2f((s_top[w * P::BM + threadIdx.x] - most) * LOG2E);
            maxima[threadIdx.x] = most, sums[threadIdx.x] = s;
        }
    }
};

template <int DT, class P>
__device__ __forceinline__ void logits_body(const Loss& p, int n, char* smem, float* s_bias, int32_t* s_label, float* s_top, float* s_sum) {
    const Partials parts(p, false);
    typename P::Flow flow(smem, hidden_rows<DT>(p, n), weight_rows<DT>(p));
    const int64_t row_tiles = (n + P::BM - 1) / P::BM, all = row_tiles * parts.groups;
    for (int64_t block = blockIdx.x; block < all; block += gridDim.x) {
        int64_t row, g, split;
        tile_of(block, row_tiles, parts.groups, 1, row, g, split);
        const int64_t m0 = row * P::BM, n0 = g * P::BN;
        typename P::Acc acc;
        if (threadIdx.x < P::BM) s_label[threadIdx.x] = m0 + threadIdx.x < n ? p.label[m0 + threadIdx.x] : -1;
        logits_of<DT, P>(p, flow, s_bias, m0, n0, acc);
        Running<DT, P> running;
        running.clear();
        running.add(p, n, acc, m0, n0, s_label);
        running.finish(s_top, s_sum, p.maxima + g * parts.pitch + m0, p.sums + g * parts.pitch + m0);
    }
}

// What a tile needs beside its operands, 1 KB of each of several arrays: of float32 or labels, of the tile's columns (number 0) or rows (the others).  A wave brings one of them.
template <class P, int ARRAYS>
struct TileArrays {
    static constexpr int BYTES = 2 * ARRAYS * 1024;
    const char* from = nullptr;     // the wave's own
    int64_t bytes = 0;
    bool columns = false;
    char* smem;
    int set = 1;                    // of the two in LDS that holds the present tile's; the other one is filled
    static __device__ __forceinline__ int own() { return int(uniform(threadIdx.x >> 6)) % ARRAYS; }
    __device__ __forceinline__ void array(int k, const void* p, int64_t values) {
        if (own() == k) from = static_cast<const char*>(p), bytes = 4 * values, columns = k == 0;
    }
    __device__ __forceinline__ void load(const typename P::Tile& t) {
        const int64_t at = 4 * (columns ? t.n0 : t.m0);
        const uint32_t lds = uniform(uint32_t(reinterpret_cast<uintptr_t>(TDB_SHARED(char, smem))));
        load_shared(lds + ((set ^ 1) * ARRAYS + own()) * 1024, buffer_of(from + at, bytes - at), (threadIdx.x & 63) * 16);
    }
    __device__ __forceinline__ const char* of(int k) const { return smem + (set * ARRAYS + k) * 1024; }
};

// Many rows: a workgroup of eight waves to a CU.  Few: tiles of as many rows as there are.  (Two kernels, of which one ends at once: with all heights in one the compiler kept
// some 100 scalar and a few vector registers in memory, and 8192 rows took 2520 us instead of 2120.)  The next tile's first step is on its way while a tile's exponentials are made.
template <int DT>
using Logits256 = Product<DT, 256, 256, 2, 4, 2, false, false>;
constexpr int MANY_SHARED = Logits256<TDB_BF16>::SHARED;
// Few rows: eight waves to a CU in 16 bits, with steps as deep as LDS holds; of float32, which has the more to multiply, twice four, or twice eight for tiles of 128 columns.  (31 rows, 91214 classes,
// 1024 columns of float32: 156 + 119 us with eight waves, 139 + 103 with twice four; 55, 128100, 1024 of float16: 76 + 49 and 81 + 51.)
template <int DT, int BN>
struct Few {
    static constexpr int THREADS = DT != TDB_F32 || BN == 128 ? 512 : 256, WAVES = THREADS / 64, WM = WAVES / 4, LINE = WM * 64, PER_CU = DT != TDB_F32 ? 1 : 2;
    using Logits128 = Product<DT, 128, BN, WM, 4, BN == 128 ? 2 : 3, false, false, LINE>;
    using Logits64 = Product<DT, 64, BN, WM, 4, 3, false, false, LINE>;
    using Logits32 = Product<DT, 32, BN, 1, WAVES, DT != TDB_F32 ? 4 : BN == 128 ? 3 : 2, false, false>;
    using Logits16 = Product<DT, 16, BN, 1, WAVES, BN == 128 ? 3 : 2, false, false>;
    using Logits160 = Product<DT, 160, BN, WM, 4, 2, false, false, LINE>;       // (float32)
    using Logits96 = Product<DT, 96, BN, WM, 4, BN == 128 ? 2 : 3, false, false, LINE>;
    static constexpr int SHARED = std::max({Logits128::SHARED, Logits64::SHARED, Logits32::SHARED, DT == TDB_F32 ? Logits160::SHARED : 0, DT == TDB_F32 ? Logits96::SHARED : 0});
};

template <int DT>
__global__ __launch_bounds__(512, 2) void loss_logits_many_kernel(Loss p) {
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    __shared__ float s_top[1024], s_sum[1024];
    using P = Logits256<DT>;
    const int n = p.count[0];
    if (p.template rows_of<DT>(n) != 256) return;
    const Partials parts(p, true);
    const int64_t row_tiles = (n + P::BM - 1) / P::BM, all = row_tiles * parts.groups;
    typename P::Flow flow(smem, hidden_rows<DT>(p, n), weight_rows<DT>(p));
    TileArrays<P, 2> arrays;
    arrays.smem = smem + P::SHARED;
    arrays.array(0, p.biases, (p.vocab + TILE - 1) / TILE * TILE), arrays.array(1, p.label, n);
    // The tile after the t-th of a group: of the same group, or the first of the workgroup's next one.
    int64_t row, g, split;
    auto tile = [&](int64_t r, int64_t t) { return typename P::Tile{r * P::BM, t * P::BN, 0, p.pitch / P::LINE_BYTES}; };
    int64_t block = blockIdx.x;
    if (block >= all) return;
    tile_of(block, row_tiles, parts.groups, 1, row, g, split);
    int64_t t = g * parts.group;
    typename P::Tile now = tile(row, t);
    P::open(flow, now, arrays);
    int stage = 0;
    Running<DT, P> running;
    running.clear();
    while (true) {
        const bool last = t + 1 == min(parts.tiles, (g + 1) * parts.group);
        int64_t next_row = row, next_g = g;
        if (last && block + gridDim.x < all) tile_of(block + gridDim.x, row_tiles, parts.groups, 1, next_row, next_g, split);
        const int64_t next_t = last ? next_g * parts.group : t + 1;
        const typename P::Tile next = tile(next_row, next_t);
        const bool more = !last || block + gridDim.x < all;
        arrays.set ^= 1;
        typename P::Acc acc;
        P::template run_on<0>(flow, now, next, more, stage, true, acc, [&](int j, int q) { return *reinterpret_cast<const f32x4*>(arrays.of(0) + 4 * (P::wave_n() + j * Matrix<DT>::SIDE + quad_n<DT>(q))); }, arrays);
        running.add(p, n, acc, now.m0, now.n0, reinterpret_cast<const int32_t*>(arrays.of(1)));
        if (last) {
            running.finish(s_top, s_sum, p.maxima + g * parts.pitch + now.m0, p.sums + g * parts.pitch + now.m0);
            running.clear();
            block += gridDim.x;
        }
        if (!more) break;
        row = next_row, g = next_g, t = next_t, now = next;
    }
}
template <int DT, int BN>
__global__ __launch_bounds__((Few<DT, BN>::THREADS), 2) void loss_logits_few_kernel(Loss p) {
    using F = Few<DT, BN>;
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    __shared__ __attribute__((aligned(16))) float s_bias[BN];
    __shared__ int32_t s_label[160];
    __shared__ float s_top[640], s_sum[640];
    const int n = p.count[0];
    const int height = p.template rows_of<DT>(n);
    if constexpr (DT == TDB_F32) {
        if (height == 16) return logits_body<DT, typename F::Logits16>(p, n, smem, s_bias, s_label, s_top, s_sum);
        if (height == 96) return logits_body<DT, typename F::Logits96>(p, n, smem, s_bias, s_label, s_top, s_sum);
        if constexpr (BN == 256)        // (the narrow tiles are for 128 rows at most)
            if (height == 160) return logits_body<DT, typename F::Logits160>(p, n, smem, s_bias, s_label, s_top, s_sum);
    }
    switch (height) {
        case 32: return logits_body<DT, typename F::Logits32>(p, n, smem, s_bias, s_label, s_top, s_sum);
        case 64: return logits_body<DT, typename F::Logits64>(p, n, smem, s_bias, s_label, s_top, s_sum);
        case 128: return logits_body<DT, typename F::Logits128>(p, n, smem, s_bias, s_label, s_top, s_sum);
    }
}

// The rows' losses and what the gradient needs of them; their sum by the workgroup that ends last.  A workgroup has 32 rows, 32 groups of threads share the parts of each.
template <int DT>
__global__ __launch_bounds__(1024) void loss_finish_kernel(Loss p) {
    __shared__ float s_top[32][33], s_sum[32][33];
    __shared__ double s_all[32];
    const int n = p.count[0], l = threadIdx.x & 31, w = threadIdx.x >> 5;
    const Partials parts(p, p.template rows_of<DT>(n) == 256);
    const int groups = int(parts.groups);
    double mine = 0.0;
    for (int64_t r0 = int64_t(blockIdx.x) * FINISH_ROWS; r0 < n; r0 += int64_t(gridDim.x) * FINISH_ROWS) {
        const int64_t r = min(r0 + l, int64_t(n - 1));
        float top = -FLT_MAX, sum = 0.f;
        for (int g = w; g < groups; g += 32 * 8) {
            float t[8], s[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int64_t at = min(g + 32 * u, groups - 1) * parts.pitch + r;
                t[u] = g + 32 * u < groups ? p.maxima[at] : -FLT_MAX, s[u] = g + 32 * u < groups ? p.sums[at] : 0.f;
            }
            float most = top;
#pragma unroll
            for (int u = 0; u < 8; ++u) most = fmaxf(most, t[u]);
            sum *= __builtin_amdgcn_exp2f((top - most) * LOG2E);
#pragma unroll
            for (int u = 0; u < 8; ++u) sum += s[u] * __builtin_amdgcn_exp2f((t[u] - most) * LOG2E);
            top = most;
        }
        __syncthreads();
        s_top[l][w] = top, s_sum[l][w] = sum;
        __syncthreads();
        // A row for each half wave.
        top = s_top[w][l], sum = s_sum[w][l];
        float most = top;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) most = fmaxf(most, __shfl_xor(most, d));
        sum *= __builtin_amdgcn_exp2f((top - most) * LOG2E);
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor(sum, d);
        const int64_t row = r0 + w;
        if (l == 0 && row < n) {
            const float loss = (most - p.right[row]) + log2f(sum) * LN2;
            p.top[row] = p.label[row] < 0 ? __builtin_nanf("") : most;
            p.inverse[row] = D_SCALE<DT> / sum;
            if (p.reduction == 0) p.loss[p.index[row]] = loss;
            mine += loss;
        }
    }
    if (p.reduction == 0) return;
    // (only workgroups that have rows, or the first one, take part)
    const int taking_part = max(1, min(int(gridDim.x), (n + FINISH_ROWS - 1) / FINISH_ROWS));
    if (int(blockIdx.x) >= taking_part) return;
    if (l == 0) s_all[w] = mine;
    __syncthreads();
    if (threadIdx.x >= 64) return;
    double sum = threadIdx.x < 32 ? s_all[threadIdx.x] : 0.0;
    auto over_wave = [](double x) {
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) x += __shfl_xor(x, d);
        return x;
    };
    sum = over_wave(sum);
    bool last = false;
    if (threadIdx.x == 0) {
        __hip_atomic_store(p.block_sums + blockIdx.x, sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        last = __hip_atomic_fetch_add(p.count + 1, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == taking_part - 1;
    }
    if (!__builtin_amdgcn_readfirstlane(int(last))) return;
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
    sum = 0.0;
    for (int i = threadIdx.x; i < taking_part; i += 64) sum += __hip_atomic_load(p.block_sums + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    sum = over_wave(sum);
    if (threadIdx.x == 0) p.loss[0] = float(p.reduction == 2 ? sum / double(n) : sum);
}

// What the gradient needs beside Loss.
struct Gradient {
    const float* dloss;
    int64_t dloss_stride;
    void *dx, *dbias;
    char* dweight;
    int64_t dx_stride, dweight_pitch;
    // D, [padded rows][columns of a piece], of x's type: a matrix instruction takes both operands in one.  So it is rounded, by half a step of the type at most, and that is the largest error of 16-bit gradients
    // beside their own rounding.  Against 64 bits, relative to the norm, bfloat16: 2458 rows x 768, 128100 classes, dx and dW 1.9e-3, from D in float32 1.7e-3; 512 rows with gradients of their own, 30011 classes,
    // 2.3e-3 and 1.7e-3; float16 2.5e-4 to 4.1e-4, and 2.0e-4 to 3.7e-4.  What that saves: D as a sum of two values takes both products twice (8192 x 1024, 128100 classes: 3.8 ms on 7.9) and twice the workspace, in
    // float32 instructions a tenth of the rate.  Sums over D, of dx, dW and dbias, are of float32, dbias from D before it is rounded.
    char* d;
    int64_t d_pitch;
    int64_t first, columns;     // of the piece (columns a multiple of TILE)
    float* parts;               // of dx, [splits][rows that count, rounded up to tiles][part_pitch]
    int64_t part_pitch;
    float* dw_parts;            // of dW, where its tiles' contraction is split: [dw_splits][vocabulary][part_pitch]
    int64_t dw_splits;
    // Where every row has a gradient g of its own, it goes into D (g <- g / common), in float16 without its power of two, which the row itself takes (x <- x shift).
    int32_t* reach;             // float16: power of two of the row's g and of its largest value
    char* shifted;              // gathered rows times shift; the gathered rows themselves otherwise
    float *scale, *share, *shift, *common;      // inverse times g; g; 1 but in float16, there the row's power of two relative to common; a power of two
    float* column_sums;         // of D, [tiles of rows][columns]
    bool wide_dweight, later;   // later: a piece that is not the first
};

// What the gradient of a tile needs of its rows, in LDS.
struct RowArrays {
    const float *top, *scale, *right, *share, *shift;
    const int32_t* label;
};

// D of a tile, to memory, and its sums over the tile's rows.  s_column: WM * BN.
template <int DT, class P, bool WEIGHTED>
__device__ __forceinline__ void difference_of(const Loss& p, const Gradient& g, int n, const typename P::Acc& acc, int64_t row, int64_t n0, const RowArrays& of, char* scratch, float* s_column) {
    using M = Matrix<DT>;
    using T = typename M::T;
    constexpr int N = P::TN * M::QUADS * 4;     // values of a lane in a row
    const int64_t m0 = row * P::BM;
    const int first = P::wave_m() + lane_m<DT>();
    // (rows that are not there: zeros)
    auto relative = [&](int i) { return m0 + first + i * M::SIDE < n ? of.label[first + i * M::SIDE] - int(n0) - P::wave_n() : -1; };
    auto share_of = [&](int i) { return WEIGHTED ? of.share[first + i * M::SIDE] : D_SCALE<DT>; };
    auto shift_of = [&](int i) { return WEIGHTED && DT == TDB_F16 ? of.shift[first + i * M::SIDE] : 1.f; };
    float sums[N];
#pragma unroll
    for (int c = 0; c < N; ++c) sums[c] = 0.f;
    float top = 0.f, scale = 0.f, shift = 1.f;
    P::store(
        scratch, g.d + m0 * g.d_pitch + (n0 - g.first) * int64_t(sizeof(T)), g.d_pitch, P::BM, P::BN, true,
        [&](int i, int j, int q) {
            if (j == 0 && q == 0) {
                const bool there = m0 + first + i * M::SIDE < n;
                top = there ? of.top[first + i * M::SIDE] : INFINITY, scale = there ? of.scale[first + i * M::SIDE] : 0.f, shift = there ? shift_of(i) : 0.f;
            }
            const f32x4 v = P::quad(acc, i, j, q);
            f32x4 d;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                d[e] = __builtin_amdgcn_exp2f((v[e] - top) * LOG2E) * scale;
                sums[(j * M::QUADS + q) * 4 + e] += WEIGHTED && DT == TDB_F16 ? d[e] * shift : d[e];
            }
            return d;
        },
        [&](int i, char* rows) {    // the label's own value
            const int rel = relative(i);
            if (rel >= 0 && rel < P::COLUMNS && (threadIdx.x & 63) < M::SIDE) {
                const float right = of.right[first + i * M::SIDE];
                *reinterpret_cast<T*>(rows + P::lies_at(lane_m<DT>(), rel * int(sizeof(T)))) = T(__builtin_amdgcn_exp2f((right - top) * LOG2E) * scale - share_of(i));
            }
        });
    if (!g.dbias) return;
    float sum = over_m<DT>(sums);
    const int c = lane_m<DT>() % N, mine = c / (4 * M::QUADS) * M::SIDE + quad_n<DT>(c / 4 % M::QUADS) + c % 4;     // the lane's column
#pragma unroll
    for (int i = 0; i < P::TM; ++i) {
        const int rel = relative(i);
        for (uint64_t who = __builtin_amdgcn_ballot_w64(rel >= 0 && rel < P::COLUMNS) & (~uint64_t(0) >> (64 - M::SIDE)); who; who &= who - 1) {
            const int lane = __builtin_ctzll(who);
            const float less = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, share_of(i) * shift_of(i)), lane));
            sum -= __builtin_amdgcn_readlane(rel, lane) == mine ? less : 0.f;
        }
    }
    if (lane_m<DT>() < N) s_column[P::wave_m() / (P::TM * M::SIDE) * P::BN + P::wave_n() + mine] = sum;
    step_barrier();
    if (threadIdx.x < P::BN) {
        float all = 0.f;
#pragma unroll
        for (int w = 0; w < P::WM; ++w) all += s_column[w * P::BN + threadIdx.x];
        g.column_sums[row * g.columns + n0 - g.first + threadIdx.x] = all;
    }
}

// D of a piece of the vocabulary.
template <int DT, class P, bool WEIGHTED>
__device__ __forceinline__ void difference_body(const Loss& p, const Gradient& g, int n, char* smem, float* s_bias, float (&s_rows)[6][160], float* s_column) {
    typename P::Flow flow(smem, hidden_rows<DT>(p, n), weight_rows<DT>(p));
    const int64_t row_tiles = (n + P::BM - 1) / P::BM, column_tiles = g.columns / P::BN, all = row_tiles * column_tiles;
    for (int64_t block = blockIdx.x; block < all; block += gridDim.x) {
        int64_t row, column, split;
        tile_of(block, row_tiles, column_tiles, 1, row, column, split);
        const int64_t m0 = row * P::BM, n0 = g.first + column * P::BN;
        typename P::Acc acc;
        __syncthreads();
        if (const int64_t m = m0 + threadIdx.x; threadIdx.x < P::BM && m < n) {
            s_rows[0][threadIdx.x] = p.top[m], s_rows[1][threadIdx.x] = WEIGHTED ? g.scale[m] : p.inverse[m], s_rows[2][threadIdx.x] = p.right[m];
            s_rows[3][threadIdx.x] = __builtin_bit_cast(float, p.label[m]);
            if (WEIGHTED) s_rows[4][threadIdx.x] = g.share[m], s_rows[5][threadIdx.x] = g.shift[m];
        }
        logits_of<DT, P>(p, flow, s_bias, m0, n0, acc);
        const RowArrays rows{s_rows[0], s_rows[1], s_rows[2], s_rows[4], s_rows[5], reinterpret_cast<const int32_t*>(s_rows[3])};
        difference_of<DT, P, WEIGHTED>(p, g, n, acc, row, n0, rows, smem, s_column);
    }
}

template <int DT, bool WEIGHTED>
__global__ __launch_bounds__(512, 2) void loss_difference_many_kernel(Loss p, Gradient g) {
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    __shared__ float s_column[512];
    using P = Logits256<DT>;
    const int n = p.count[0];
    if (p.template rows_of<DT>(n) != 256) return;
    const int64_t row_tiles = (n + P::BM - 1) / P::BM, column_tiles = g.columns / P::BN, all = row_tiles * column_tiles;
    typename P::Flow flow(smem, hidden_rows<DT>(p, n), weight_rows<DT>(p));
    constexpr int ARRAYS = WEIGHTED ? 7 : 5;
    TileArrays<P, ARRAYS> arrays;
    arrays.smem = smem + P::SHARED;
    arrays.array(0, p.biases, (p.vocab + TILE - 1) / TILE * TILE), arrays.array(1, p.top, n), arrays.array(2, WEIGHTED ? g.scale : p.inverse, n), arrays.array(3, p.right, n);
    arrays.array(4, p.label, n);
    if constexpr (WEIGHTED) arrays.array(5, g.share, n), arrays.array(6, g.shift, n);
    auto tile = [&](int64_t block, int64_t& row) {
        int64_t column, split;
        tile_of(block < all ? block : 0, row_tiles, column_tiles, 1, row, column, split);
        return typename P::Tile{row * P::BM, g.first + column * P::BN, 0, p.pitch / P::LINE_BYTES};
    };
    if (blockIdx.x >= all) return;
    int64_t row, next_row;
    typename P::Tile now = tile(blockIdx.x, row);
    P::open(flow, now, arrays);
    int stage = 0;
    for (int64_t block = blockIdx.x; block < all; block += gridDim.x) {
        const typename P::Tile next = tile(block + gridDim.x, next_row);
        arrays.set ^= 1;
        typename P::Acc acc;
        auto start = [&](int j, int q) { return *reinterpret_cast<const f32x4*>(arrays.of(0) + 4 * (P::wave_n() + j * Matrix<DT>::SIDE + quad_n<DT>(q))); };
        P::template run_on<P::STORES>(flow, now, next, block + gridDim.x < all, stage, block == blockIdx.x, acc, start, arrays);
        auto floats = [&](int k) { return reinterpret_cast<const float*>(arrays.of(k)); };
        const RowArrays rows{floats(1), floats(2), floats(3), floats(ARRAYS - 2), floats(ARRAYS - 1), reinterpret_cast<const int32_t*>(arrays.of(4))};
        difference_of<DT, P, WEIGHTED>(p, g, n, acc, row, now.n0, rows, P::scratch(smem, stage), s_column);
        row = next_row, now = next;
    }
}
template <int DT, bool WEIGHTED, int BN>
__global__ __launch_bounds__((Few<DT, BN>::THREADS), 2) void loss_difference_few_kernel(Loss p, Gradient g) {
    using F = Few<DT, BN>;
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    __shared__ __attribute__((aligned(16))) float s_bias[BN];
    __shared__ float s_column[2 * BN], s_rows[6][160];
    const int n = p.count[0];
    const int height = p.template rows_of<DT>(n);
    if constexpr (DT == TDB_F32) {
        if (height == 16) return difference_body<DT, typename F::Logits16, WEIGHTED>(p, g, n, smem, s_bias, s_rows, s_column);
        if (height == 96) return difference_body<DT, typename F::Logits96, WEIGHTED>(p, g, n, smem, s_bias, s_rows, s_column);
        if constexpr (BN == 256)        // (the narrow tiles are for 128 rows at most)
            if (height == 160) return difference_body<DT, typename F::Logits160, WEIGHTED>(p, g, n, smem, s_bias, s_rows, s_column);
    }
    switch (height) {
        case 32: return difference_body<DT, typename F::Logits32, WEIGHTED>(p, g, n, smem, s_bias, s_rows, s_column);
        case 64: return difference_body<DT, typename F::Logits64, WEIGHTED>(p, g, n, smem, s_bias, s_rows, s_column);
        case 128: return difference_body<DT, typename F::Logits128, WEIGHTED>(p, g, n, smem, s_bias, s_rows, s_column);
    }
}

// How the workgroups of a launch share out the product of dx: over the tiles of rows and columns, and where they are more than tiles, over the contraction.
template <int DT>
struct Shares {
    int height;
    int64_t row_tiles, column_tiles, splits;
    __device__ __forceinline__ Shares(const Loss& p, const Gradient& g, int n, int64_t blocks, int width) {
        // (Up to 192 rows in 16 bits the product waits for the weights whatever its tiles' height, and low ones make fewer parts to be added up: 154 x 768, tiles of 256 rows 56 + 27 us, of
        // 64 57 + 10.)
        // float32 is bound by products: 8 rows, 128100 x 768, 121 us in 64 rows, 75 in 32.
        height = DT == TDB_F32 ? tile_rows<DT>(n, 32, 1, 1, FEW) : n <= 192 ? 64 : tile_rows<DT>(n, 128, 1, 1, FEW);
        if (height <= 64 && width == 192) width = 256;
        row_tiles = (n + height - 1) / height, column_tiles = (p.hidden + width - 1) / width;
        const int64_t tiles = row_tiles * column_tiles;
        splits = tiles ? max(int64_t(1), min(blocks / tiles, g.columns * int64_t(sizeof(typename Matrix<DT>::T)) / 128)) : 0;
    }
};

// A tile's part of a sum, in float32, to the rows that there are; more: added to what is there.
template <int DT, class P>
__device__ __forceinline__ void store_part(const typename P::Acc& acc, float* parts, int64_t pitch, int64_t m0, int64_t n0, int64_t rows, bool more) {
    using M = Matrix<DT>;
#pragma unroll
    for (int i = 0; i < P::TM; ++i) {
        const int64_t m = m0 + P::wave_m() + i * M::SIDE + lane_m<DT>();
        float* const to = parts + m * pitch;
#pragma unroll
        for (int j = 0; j < P::TN; ++j)
#pragma unroll
            for (int q = 0; q < M::QUADS; ++q) {
                const int64_t c = n0 + P::wave_n() + j * M::SIDE + quad_n<DT>(q);
                if (m < rows && c < pitch) {
                    f32x4 v = P::quad(acc, i, j, q);
                    if (more) v += *reinterpret_cast<const f32x4*>(to + c);
                    *reinterpret_cast<f32x4*>(to + c) = v;
                }
            }
    }
}

// Parts of dx: D W over a share of the piece's columns.
template <int DT, class P>
__device__ __forceinline__ void dx_body(const Loss& p, const Gradient& g, int n, const Shares<DT>& share, char* smem) {
    using M = Matrix<DT>;
    const int64_t all = share.row_tiles * share.column_tiles * share.splits, steps = g.columns / P::STEP;
    const Rows a{g.d, g.d_pitch, n, uint32_t(g.d_pitch)};
    const Rows b{p.w + g.first * p.w_pitch, p.w_pitch, min(g.columns, p.vocab - g.first), weight_rows<DT>(p).width};
    typename P::Flow flow(smem, a, b);
    for (int64_t block = blockIdx.x; block < all; block += gridDim.x) {
        int64_t row, column, split;
        tile_of(block, share.row_tiles, share.column_tiles, share.splits, row, column, split);
        const int64_t m0 = row * P::BM, n0 = column * P::BN;
        typename P::Acc acc;
        P::run(flow, {m0, n0, steps * split / share.splits, steps * (split + 1) / share.splits}, acc, P::ZEROS);
        store_part<DT, P>(acc, g.parts + split * share.row_tiles * P::BM * g.part_pitch, g.part_pitch, m0, n0, n, g.later);
    }
}

// Tiles of dx and dW are 256, 192 or 128 columns wide.
template <int DT, int BN>
using Dx256 = Product<DT, 256, BN, BN == 256 ? 2 : 4, BN == 256 ? 4 : 2, 2, false, true>;
template <int DT, int BN>
using Dx128 = Product<DT, 128, BN, BN == 256 ? 2 : 4, BN == 256 ? 4 : 2, 3, false, true>;
template <int DT, int BN>
using Dx64 = Product<DT, 64, BN == 192 ? 256 : BN, BN == 128 ? 2 : 1, BN == 128 ? 4 : 8, 3, false, true>;
template <int BN>
using Dx160 = Product<TDB_F32, 160, BN, 2, 4, 2, false, true>;
template <int BN>
using Dx32 = Product<TDB_F32, 32, BN == 192 ? 256 : BN, 1, 8, 4, false, true>;
template <int BN>
using Dx96 = Product<TDB_F32, 96, BN, 2, 4, 3, false, true>;
constexpr int DX_SHARED = Dx128<TDB_BF16, 256>::SHARED;
static_assert(Dx256<TDB_BF16, 256>::SHARED <= DX_SHARED && Dx64<TDB_BF16, 256>::SHARED <= DX_SHARED && Dx32<256>::SHARED <= DX_SHARED && Dx160<256>::SHARED <= DX_SHARED && Dx96<256>::SHARED <= DX_SHARED, "");

template <int DT, int BN>
__global__ __launch_bounds__(512, 2) void loss_dx_kernel(Loss p, Gradient g) {
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    const int n = p.count[0];
    const Shares<DT> share(p, g, n, gridDim.x, BN);
    if constexpr (DT == TDB_F32) {
        if (share.height == 32) return dx_body<DT, Dx32<BN>>(p, g, n, share, smem);
        if (share.height == 96) return dx_body<DT, Dx96<BN>>(p, g, n, share, smem);
        if (share.height == 160) return dx_body<DT, Dx160<BN>>(p, g, n, share, smem);
    }
    switch (share.height) {
        case 64: return dx_body<DT, Dx64<DT, BN>>(p, g, n, share, smem);
        case 128: return dx_body<DT, Dx128<DT, BN>>(p, g, n, share, smem);
        default: return dx_body<DT, Dx256<DT, BN>>(p, g, n, share, smem);
    }
}

// What the gradient of a sum or mean makes of every row.
__device__ __forceinline__ float row_factor(const Loss& p, const Gradient& g, int n) { return p.reduction == 2 ? g.dloss[0] / float(n) : g.dloss[0]; }

// dx, zeros where a row does not count.  Where few rows are split over many parts a workgroup has 256 columns of a row and its waves share out the parts, otherwise each wave has a row.
// blocks, width: workgroups of the launch before and its tiles' columns.
template <int DT>
__global__ __launch_bounds__(256) void loss_dx_sum_kernel(Loss p, Gradient g, int blocks, int width) {
    using T = typename Matrix<DT>::T;
    __shared__ float s_sum[4][256];
    const int n = p.count[0], l = threadIdx.x & 63, w = threadIdx.x >> 6;
    const Shares<DT> share(p, g, n, blocks, width);
    const int64_t apart = share.row_tiles * share.height * g.part_pitch;
    auto factor_of = [&](int place) { return (p.reduction ? row_factor(p, g, n) : *g.common * g.shift[place]) * (1.f / D_SCALE<DT>); };
    // parts first, first + step, ... of columns c ..
    auto sum_of = [&](int place, int64_t c, int64_t first, int64_t step) {
        const float* const from = g.parts + place * g.part_pitch + min(c, g.part_pitch - 4);
        f32x4 sum = {0.f, 0.f, 0.f, 0.f};
        for (int64_t s = first; s < share.splits; s += 8 * step) {
            f32x4 x[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) x[u] = *reinterpret_cast<const f32x4*>(from + min(s + u * step, share.splits - 1) * apart);
#pragma unroll
            for (int u = 0; u < 8; ++u)
                if (s + u * step < share.splits) sum += x[u];
        }
        return sum;
    };
    if (share.splits <= 16) {
        const bool wide = reinterpret_cast<uintptr_t>(g.dx) % (4 * sizeof(T)) == 0 && g.dx_stride % 4 == 0 && p.hidden % 4 == 0;
        for (int64_t row = int64_t(blockIdx.x) * 4 + w; row < p.rows; row += int64_t(gridDim.x) * 4) {
            const int place = p.place[row];
            T* const to = static_cast<T*>(g.dx) + row * g.dx_stride;
            const float factor = place < 0 ? 0.f : factor_of(place);
            for (int c = 4 * l; c < p.hidden; c += 256) {
                f32x4 sum = {0.f, 0.f, 0.f, 0.f};
                if (place >= 0) sum = sum_of(place, c, 0, 1) * factor;
                if (wide) {
                    typedef __attribute__((ext_vector_type(4))) T T4;
                    *reinterpret_cast<T4*>(to + c) = T4{T(sum[0]), T(sum[1]), T(sum[2]), T(sum[3])};
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (c + e < p.hidden) to[c + e] = T(sum[e]);
                }
            }
        }
        return;
    }
    const int chunks = (p.hidden + 255) / 256;
    for (int64_t item = blockIdx.x; item < p.rows * chunks; item += gridDim.x) {
        const int64_t row = item / chunks;
        const int c0 = int(item - row * chunks) * 256, at = c0 + threadIdx.x, place = p.place[row];
        T* const to = static_cast<T*>(g.dx) + row * g.dx_stride;
        if (place < 0) {
            if (at < p.hidden) to[at] = T(0.f);
            continue;
        }
        const f32x4 sum = sum_of(place, c0 + 4 * l, w, 4);
        __syncthreads();
        *reinterpret_cast<f32x4*>(&s_sum[w][4 * l]) = sum;
        __syncthreads();
        if (at < p.hidden) to[at] = T((((s_sum[0][threadIdx.x] + s_sum[1][threadIdx.x]) + s_sum[2][threadIdx.x]) + s_sum[3][threadIdx.x]) * factor_of(place));
    }
}

// float16: of each row the power of two of its gradient and of its largest value together, or NO_REACH where the gradient is 0, infinite or NaN.  (Of a value: -24 for the smallest and for rows of
// zeros, 15 for the largest and where one is infinite or NaN.)  A wave to a row; bound by the launch at 154 x 768 (4.7 us), 8192 x 1024 take 8.8.
constexpr int NO_REACH = -(1 << 20);
__global__ __launch_bounds__(256) void loss_reach_kernel(Loss p, Gradient g) {
    const int n = p.count[0], l = threadIdx.x & 63, w = threadIdx.x >> 6;
    for (int r = blockIdx.x * 4 + w; r < n; r += gridDim.x * 4) {
        const float weight = g.dloss[p.index[r] * g.dloss_stride];
        const uint4* const from = reinterpret_cast<const uint4*>(p.gathered + r * p.pitch);
        uint32_t most = 0;
        for (int c = l; c < int(p.pitch / 16); c += 64) {
            const uint4 v = from[c];
            for (const uint32_t pair : {v.x, v.y, v.z, v.w}) most = max(most, max(pair & 0x7fff, pair >> 16 & 0x7fff));
        }
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) most = max(most, uint32_t(__shfl_xor(int(most), d)));
        const int value = most >= 0x7c00 ? 15 : most ? ilogbf(float(__builtin_bit_cast(_Float16, uint16_t(most)))) : -24;
        if (l == 0) g.reach[r] = weight != 0.f && fabsf(weight) < INFINITY ? ilogbf(weight) + value : NO_REACH;
    }
}

// Rows with gradients of their own.  float32, bfloat16: common is the power of two of the largest.  float16: a row's own power of two goes to x instead of D, relative to a common one by which the largest of all
// g x comes to lie in [2^15, 2^16).  Up to there a power of two takes no bits; what x loses at the other end is half of float16's smallest step, 2^-25, so 2^-40 of the largest g x, where dW, in float16
// too, holds no more than 2^-41 of float16's largest value.  (With g alone made common, x of ordinary size lost bits from 2^-14 of the largest g on and was gone at 2^-24.)  The common one is not below 2^-100, where
// all of dx and dW are float16's 0, so that float32 holds its products for dbias.
template <int DT>
__global__ __launch_bounds__(256) void loss_weigh_kernel(Loss p, Gradient g) {
    using T = typename Matrix<DT>::T;
    __shared__ int s_most[4];
    const int n = p.count[0], l = threadIdx.x & 63, w = threadIdx.x >> 6;
    int most = NO_REACH;
    float largest = 0.f;
    for (int r = threadIdx.x; r < n; r += 256) {
        if (DT == TDB_F16) most = max(most, g.reach[r]);
        else largest = fmaxf(largest, fabsf(g.dloss[p.index[r] * g.dloss_stride]));
    }
    if (DT != TDB_F16) most = __builtin_bit_cast(int, largest);         // (of positive values the larger has the larger bits)
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) most = max(most, __shfl_xor(most, d));
    if (l == 0) s_most[w] = most;
    __syncthreads();
    most = max(max(s_most[0], s_most[1]), max(s_most[2], s_most[3]));
    largest = __builtin_bit_cast(float, most);
    const int common = DT == TDB_F16 ? (most == NO_REACH ? 0 : max(most - 15, -100)) : largest > 0.f && largest < INFINITY ? ilogbf(largest) : 0;
    if (blockIdx.x == 0 && threadIdx.x == 0) *g.common = ldexpf(1.f, common);
    for (int r = blockIdx.x * 4 + w; r < n; r += gridDim.x * 4) {
        const float weight = g.dloss[p.index[r] * g.dloss_stride];
        const int own = DT == TDB_F16 && weight != 0.f && fabsf(weight) < INFINITY ? ilogbf(weight) : common;
        const float share = ldexpf(weight, -own), shift = ldexpf(1.f, own - common);
        if (l == 0) g.scale[r] = p.inverse[r] * share, g.share[r] = D_SCALE<DT> * share, g.shift[r] = shift;
        if constexpr (DT == TDB_F16) {
            const T* const from = reinterpret_cast<const T*>(p.gathered + r * p.pitch);
            T* const to = reinterpret_cast<T*>(g.shifted + r * p.pitch);
            for (int c = l; c < int(p.pitch / sizeof(T)); c += 64) to[c] = T(float(from[c]) * shift);
        }
    }
}

// dW and dbias of a piece.
template <int DT, int BN>
using Dweight = Product<DT, 256, BN, BN == 256 ? 2 : 4, BN == 256 ? 4 : 2, 2, true, true>;

// (SPLIT, several workgroups to a tile's rows, as a kernel of its own: as an argument it cost the others 2 of 41 us at 7 rows, 128100 x 768.)
template <int DT, int BN, bool SPLIT>
__global__ __launch_bounds__(512, 2) void loss_dweight_kernel(Loss p, Gradient g) {
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    using P = Dweight<DT, BN>;
    using T = typename Matrix<DT>::T;
    constexpr int BM = P::BM;
    const int n = p.count[0];
    const int64_t columns = min(g.columns, p.vocab - g.first), row_tiles = (columns + BM - 1) / BM, column_tiles = g.dweight ? (p.hidden + BN - 1) / BN : 1, splits = SPLIT ? g.dw_splits : 1, all = row_tiles * column_tiles * splits;
    const int64_t steps = (n + P::STEP - 1) / P::STEP;
    const Rows a{g.d, g.d_pitch, n, uint32_t(g.d_pitch)}, b{g.shifted, p.pitch, n, uint32_t(p.pitch)};
    typename P::Flow flow(smem, a, b);
    const int heights = n ? (n + p.template rows_of<DT>(n) - 1) / p.template rows_of<DT>(n) : 0;
    const float factor = n == 0 ? 0.f : (p.reduction ? row_factor(p, g, n) : *g.common) * (1.f / D_SCALE<DT>);
    int64_t split, next_split;
    auto tile = [&](int64_t block, int64_t& part) {
        int64_t row, column;
        tile_of(block < all ? block : 0, row_tiles, column_tiles, splits, row, column, part);
        return typename P::Tile{row * BM, column * BN, steps * part / splits, steps * (part + 1) / splits};
    };
    if (blockIdx.x >= all) return;
    typename P::Tile now = tile(blockIdx.x, split);
    typename P::Alone alone;
    if (g.dweight) P::open(flow, now, alone);
    int stage = 0;
    for (int64_t block = blockIdx.x; block < all; block += gridDim.x) {
        const typename P::Tile next = tile(block + gridDim.x, next_split);
        if (const int64_t m = now.m0 + threadIdx.x; g.dbias && now.n0 == 0 && split == 0 && threadIdx.x < BM && m < columns) {
            float sum = 0.f;
            for (int t = 0; t < heights; ++t) sum += g.column_sums[t * g.columns + m];
            if (p.bias_kind == 2) static_cast<float*>(g.dbias)[g.first + m] = sum * factor;
            else static_cast<T*>(g.dbias)[g.first + m] = T(sum * factor);
        }
        if (g.dweight) {
            typename P::Acc acc;
            P::template run_on<P::STORES>(flow, now, next, block + gridDim.x < all, stage, SPLIT || !g.wide_dweight || block == blockIdx.x, acc, P::ZEROS, alone);
            if constexpr (SPLIT) store_part<DT, P>(acc, g.dw_parts + split * p.dw_rows() * g.part_pitch, g.part_pitch, now.m0, now.n0, columns, false);
            else P::store(
                P::scratch(smem, stage), g.dweight + (g.first + now.m0) * g.dweight_pitch + now.n0 * int64_t(sizeof(T)), g.dweight_pitch, columns - now.m0, p.hidden - now.n0, g.wide_dweight,
                [&](int i, int j, int q) {
                    f32x4 v = P::quad(acc, i, j, q);
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] *= factor;
                    return v;
                },
                [](int, char*) {});
        }
        now = next, split = next_split;
    }
}
// dW of parts.
template <int DT>
__global__ __launch_bounds__(256) void loss_dweight_sum_kernel(Loss p, Gradient g) {
    using T = typename Matrix<DT>::T;
    const int n = p.count[0];
    const float factor = n == 0 ? 0.f : (p.reduction ? row_factor(p, g, n) : *g.common) * (1.f / D_SCALE<DT>);
    const int64_t quads = g.part_pitch / 4, apart = p.dw_rows() * g.part_pitch;
    for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < p.vocab * quads; i += int64_t(gridDim.x) * 256) {
        const int64_t v = i / quads;
        const int c = int(i - v * quads) * 4;
        f32x4 sum = {0.f, 0.f, 0.f, 0.f};
        for (int64_t s = 0; s < g.dw_splits; ++s) sum += *reinterpret_cast<const f32x4*>(g.dw_parts + s * apart + i * 4);
        T* const to = reinterpret_cast<T*>(g.dweight + v * g.dweight_pitch) + c;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (c + e < p.hidden) to[e] = T(sum[e] * factor);
    }
}

// ------------------------------------------------------------------------------------------------------------------- host

constexpr int64_t D_BYTES = int64_t(1) << 31;       // of the workspace that holds D, unless 256 columns take more
constexpr int64_t PARTIAL_BYTES = int64_t(1) << 27;
constexpr int64_t SPLIT_ROWS = 512, PART_BYTES = int64_t(1) << 28;

int64_t round_up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }

constexpr int WIDTHS[] = {256, 192, 128};
constexpr int dear(int dtype, int i) { return i == 0 ? 64 : dtype == TDB_F32 ? i == 1 ? 66 : 67 : i == 1 ? 72 : 88; }        // what a column of such tiles costs

// The width of tiles of dx, which is split along its contraction: that of the least work, tiles at their price for each column.  dx and dW of 2500 x 768, 128100 classes, in tiles of 256, 192 and
// 128 columns: bfloat16 926, 1044 and 1269 us, float32 7.37, 7.57 and 7.70 ms; 384 wide 649, 575 and 704 us, 4.92, 3.79 and 3.86 ms.
int dx_columns(int hidden, int dtype) {
    int best = 0;
    auto cost = [&](int i) { return (hidden + WIDTHS[i] - 1) / WIDTHS[i] * WIDTHS[i] * dear(dtype, i); };
    for (int i = 1; i < 3; ++i)
        if (cost(i) < cost(best)) best = i;
    return WIDTHS[best];
}

// The width of tiles of dW, `high` of them below each other, and how many workgroups share the rows of each, SPLIT_ROWS of them at least: the least work of the busiest workgroup.  Parts are
// written and read: of half of the rows' products 1 / 216 for each 1 / rows in float32, 1 / 1666 in 16 bits, and PART_BYTES hold them.  4199 rows, 2010 classes, 1024 columns of float32 whole and
// by eight workgroups 537 and 159 + 15 us; 16055, 5157, 816 2030 and, by five, 1254 + 23.
void dweight_tiles(int hidden, int dtype, int64_t high, int64_t rows, bool whole, int blocks, int32_t& width, int32_t& splits) {
    double least = 0.0;
    width = 0;
    for (int i = 0; i < 3; ++i) {
        const int64_t tiles = high * ((hidden + WIDTHS[i] - 1) / WIDTHS[i]);
        for (int64_t s = 1; s == 1 || (!whole && s <= 16 && s * SPLIT_ROWS <= rows && s * high * TILE * hidden * 4 <= PART_BYTES); ++s) {
            const double part = s == 1 ? 0.0 : double(s) * (dtype == TDB_F32 ? 216 : 1666) / double(rows) * double(high * hidden * 64) / blocks;
            const double cost = double((tiles * s + blocks - 1) / blocks) / double(s) * WIDTHS[i] * dear(dtype, i) + part;
            if (!width || cost < least) least = cost, width = WIDTHS[i], splits = int32_t(s);
        }
    }
}

struct Plan {
    int size;                               // of a value
    int64_t padded, pitch, vocab;           // rows and bytes of the gathered rows, vocabulary, rounded up
    int32_t group, few_width, dx_width, dw_width;       // columns of the tiles of few rows' logits, dx and dW
    int32_t dw_splits;                      // workgroups that share the rows of a tile of dW
    int64_t few_rows;
    bool many, few;                         // whether there may be as many or as few rows as the kernels are for
    int64_t columns;                        // of a piece
    int blocks, finish_blocks;
    // offsets
    int64_t index, place, label, top, inverse, right, biases, gathered, state;
    int64_t maxima, sums, block_sums, forward;
    int64_t d, parts, part_pitch, column_sums, dw_parts, shifted, reach, scale, share, shift, common, backward;
};

Plan plan_of(const tdb_loss_args& a) {
    Plan p;
    p.size = a.dtype == TDB_F32 ? 4 : 2;
    p.padded = round_up(std::max<int64_t>(a.rows, 1), TILE);
    p.pitch = round_up(int64_t(a.hidden) * p.size, 128);
    p.vocab = round_up(a.vocab, TILE);
    const int64_t wide = p.vocab / TILE;
    p.group = int32_t((wide * p.padded * 8 + PARTIAL_BYTES - 1) / PARTIAL_BYTES);
    p.many = a.rows > 128, p.few = a.rows > 0;
    const int64_t most = std::min<int64_t>(std::max<int64_t>(D_BYTES / (p.padded * p.size) / TILE, 1), (int64_t(1) << 22) / p.size / TILE), pieces = (wide + most - 1) / most;
    p.columns = (wide + pieces - 1) / pieces * TILE;
    p.blocks = std::max(8, tdb_compute_units(-1) & -8);
    // Few rows of float32: tiles of 128 columns where those share out better over the CUs.  The two passes over the weights in tiles of 256 and 128 columns: one row (of 32), 32510 classes, 768 columns
    // 37 + 39 and 27 + 29 us; 42, 73329, 928 148 + 145 and 125 + 125; 16, 128100, 1232 187 + 138 and 201 + 163.  (In 16 bits tiles of 128 are no faster: 20, 73329, 768 27 + 29 and 28 + 30.)
    auto rounds = [&](int64_t tiles) { return (tiles + p.blocks - 1) / p.blocks; };
    p.few_width = a.dtype == TDB_F32 && a.rows <= 128 && rounds(2 * wide) < 2 * rounds(wide) ? 128 : 256;
    p.few_rows = p.padded / TILE * wide <= 2 * p.blocks ? p.padded : std::min<int64_t>(p.padded, FEW);
    p.dx_width = dx_columns(a.hidden, a.dtype);
    dweight_tiles(a.hidden, a.dtype, p.columns / TILE, a.rows, p.columns != p.vocab, p.blocks, p.dw_width, p.dw_splits);
    p.finish_blocks = int(std::min<int64_t>((std::max<int64_t>(a.rows, 1) + FINISH_ROWS - 1) / FINISH_ROWS, 256));
    int64_t at = 256;
    auto take = [&](int64_t bytes) {
        const int64_t here = at;
        at += round_up(bytes, 256);
        return here;
    };
    p.index = take(p.padded * 4), p.place = take(p.padded * 4), p.label = take(p.padded * 4), p.top = take(p.padded * 4), p.inverse = take(p.padded * 4), p.right = take(p.padded * 4), p.biases = take(p.vocab * 4);
    p.gathered = take(p.padded * p.pitch);
    p.state = at;
    at = 0;
    const int64_t partials = std::max((wide + p.group - 1) / p.group * p.padded, p.vocab / p.few_width * p.few_rows) * 4;
    p.maxima = take(partials), p.sums = take(partials), p.block_sums = take(p.finish_blocks * 8);
    p.forward = at;
    at = 0;
    p.part_pitch = round_up(a.hidden, 4);
    // As many parts of dx as workgroups share its tiles, or one.
    p.d = take(p.padded * p.columns * p.size);
    p.parts = take(std::max(p.padded, int64_t(p.blocks) * TILE) * std::max<int64_t>(p.part_pitch, 1) * 4);
    p.column_sums = take(std::max<int64_t>(p.padded / TILE, p.few_rows / 32) * p.columns * 4);
    p.dw_parts = take(p.dw_splits > 1 ? p.dw_splits * p.vocab * p.part_pitch * 4 : 0);
    const bool weighted = a.reduction == 0;
    p.shifted = take(weighted && a.dtype == TDB_F16 ? p.padded * p.pitch : 0);
    p.reach = take(weighted && a.dtype == TDB_F16 ? p.padded * 4 : 0);
    p.scale = take(weighted ? p.padded * 4 : 0), p.share = take(weighted ? p.padded * 4 : 0), p.shift = take(weighted ? p.padded * 4 : 0), p.common = take(4);
    p.backward = at;
    return p;
}

int check_sizes(const tdb_loss_args* a) {
    if (!a) return tdb_fail(TDB_ERR_NULL, "args is NULL");
    if (a->dtype != TDB_F32 && a->dtype != TDB_BF16 && a->dtype != TDB_F16) return tdb_fail(TDB_ERR_DTYPE, "unknown dtype %d", a->dtype);
    if (a->bias && a->bias_dtype != a->dtype && a->bias_dtype != TDB_F32) return tdb_fail(TDB_ERR_DTYPE, "bias_dtype %d: need that of x, or float32", a->bias_dtype);
    if (a->rows < 0 || a->rows > (1 << 27) || a->vocab < 1 || a->vocab > (1 << 27) || a->hidden < 1 || a->hidden > 32768)
        return tdb_fail(TDB_ERR_SHAPE, "%lld rows, %d columns, %lld classes: need up to 2^27, 1 to 32768, 1 to 2^27", (long long)a->rows, a->hidden, (long long)a->vocab);
    if (a->reduction < 0 || a->reduction > 2) return tdb_fail(TDB_ERR_SHAPE, "reduction %d: need 0 (none), 1 (sum) or 2 (mean)", a->reduction);
    return TDB_OK;
}

int check(const tdb_loss_args* a, bool backward) {
    if (const int rc = check_sizes(a); rc != TDB_OK) return rc;
    const int size = a->dtype == TDB_F32 ? 4 : 2;
    if (!a->weight || !a->state || !a->workspace) return tdb_fail(TDB_ERR_NULL, "weight, state and workspace must be non-NULL");
    if (a->weight_stride % (4 / size) || a->weight_stride < a->hidden || a->weight_stride > (1 << 22) / size)
        return tdb_fail(TDB_ERR_STRIDE, "weight_stride %lld: need a multiple of 4 bytes, at least a row and at most 4 MiB", (long long)a->weight_stride);
    if (reinterpret_cast<uintptr_t>(a->weight) % 4) return tdb_fail(TDB_ERR_ALIGN, "weight must be 4-byte aligned");
    for (const void* t : {static_cast<const void*>(a->state), static_cast<const void*>(a->workspace)})
        if (reinterpret_cast<uintptr_t>(t) % 16) return tdb_fail(TDB_ERR_ALIGN, "state and workspace must be 16-byte aligned");
    if (!backward) {
        if (a->rows && (!a->x || !a->labels)) return tdb_fail(TDB_ERR_NULL, "x and labels must be non-NULL");
        if (a->x_stride < 0) return tdb_fail(TDB_ERR_STRIDE, "negative row stride");
        if (!a->loss && (a->rows || a->reduction)) return tdb_fail(TDB_ERR_NULL, "loss must be non-NULL");
    } else {
        if (a->rows && !a->dloss) return tdb_fail(TDB_ERR_NULL, "dloss must be non-NULL");
        if (a->dbias && !a->bias) return tdb_fail(TDB_ERR_NULL, "dbias needs a bias");
        if (a->dloss_stride < 0 || (a->dx && a->rows > 1 && a->dx_stride < a->hidden) || (a->dweight && a->dweight_stride < a->hidden))
            return tdb_fail(TDB_ERR_STRIDE, "rows of a result overlap");
        if (a->dweight && a->dweight_stride > (1 << 22) / size)        // (a tile's rows are written through one buffer, whose offsets have 32 bits)
            return tdb_fail(TDB_ERR_STRIDE, "dweight_stride %lld: need at most 4 MiB", (long long)a->dweight_stride);
    }
    const Plan p = plan_of(*a);
    if (a->state_bytes < p.state || a->workspace_bytes < (backward ? p.backward : p.forward)) return tdb_fail(TDB_ERR_SHAPE, "state or workspace is too small");
    return TDB_OK;
}

Loss loss_of(const tdb_loss_args& a, const Plan& p) {
    Loss k{};
    char *state = static_cast<char*>(a.state), *work = static_cast<char*>(a.workspace);
    k.x = static_cast<const char*>(a.x), k.w = static_cast<const char*>(a.weight), k.bias = a.bias, k.labels = a.labels;
    k.rows = a.rows, k.vocab = a.vocab, k.ignore = a.ignore_index, k.x_stride = a.x_stride, k.w_pitch = a.weight_stride * p.size;
    k.hidden = a.hidden, k.reduction = a.reduction, k.bias_kind = !a.bias ? 0 : a.bias_dtype == a.dtype ? 1 : 2, k.loss = a.loss;
    k.count = reinterpret_cast<int32_t*>(state), k.index = reinterpret_cast<int32_t*>(state + p.index), k.place = reinterpret_cast<int32_t*>(state + p.place);
    k.label = reinterpret_cast<int32_t*>(state + p.label), k.top = reinterpret_cast<float*>(state + p.top), k.inverse = reinterpret_cast<float*>(state + p.inverse);
    k.biases = reinterpret_cast<float*>(state + p.biases), k.gathered = state + p.gathered, k.pitch = p.pitch, k.padded = p.padded, k.group = p.group, k.few_width = p.few_width, k.blocks = p.blocks, k.few_rows = p.few_rows;
    k.right = reinterpret_cast<float*>(state + p.right), k.maxima = reinterpret_cast<float*>(work + p.maxima), k.sums = reinterpret_cast<float*>(work + p.sums);
    k.block_sums = reinterpret_cast<double*>(work + p.block_sums);
    return k;
}

template <auto KERNEL, class... ARGS>
hipError_t launch(int64_t grid, int threads, int shared, hipStream_t s, const ARGS&... args) {
    if (shared > 65536) {
        static std::atomic<uint64_t> raised;        // devices where the kernel may have that much
        int dev = 0;
        if (const hipError_t e = hipGetDevice(&dev); e != hipSuccess) return e;
        if (!(raised.load(std::memory_order_acquire) >> dev & 1)) {
            if (const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(KERNEL), hipFuncAttributeMaxDynamicSharedMemorySize, shared); e != hipSuccess) return e;
            raised.fetch_or(uint64_t(1) << dev, std::memory_order_release);
        }
    }
    KERNEL<<<unsigned(grid), threads, shared, s>>>(args...);
    return hipGetLastError();
}

// go(the width of the tiles of few rows' logits, a constant)
template <int DT, class GO>
hipError_t few_rows(const Plan& p, GO go) {
    if constexpr (DT == TDB_F32)
        if (p.few_width == 128) return go(std::integral_constant<int, 128>());
    return go(std::integral_constant<int, 256>());
}

#define TDB_TRY(...) \
    do { \
        if (const hipError_t e = (__VA_ARGS__); e != hipSuccess) return e; \
    } while (0)

template <int DT>
hipError_t forward(const tdb_loss_args& a, hipStream_t s) {
    const Plan p = plan_of(a);
    const Loss k = loss_of(a, p);
    const int64_t chunk = round_up(std::max<int64_t>(64, (a.rows + 511) / 512), 64);
    const bool wide = reinterpret_cast<uintptr_t>(a.x) % 16 == 0 && a.x_stride * p.size % 16 == 0 && int64_t(a.hidden) * p.size % 16 == 0;
    const int64_t row_blocks = std::max<int64_t>(1, (a.rows + chunk - 1) / chunk), bias_blocks = (p.vocab + 256 * GATHER_WAVES - 1) / (256 * GATHER_WAVES);
    TDB_TRY(launch<loss_gather_kernel<DT>>(row_blocks + bias_blocks, 64 * GATHER_WAVES, 0, s, k, chunk, int(row_blocks), wide));
    if (p.few) TDB_TRY(few_rows<DT>(p, [&](auto f) { return launch<loss_logits_few_kernel<DT, f()>>(Few<DT, f()>::PER_CU * p.blocks, Few<DT, f()>::THREADS, Few<DT, f()>::SHARED, s, k); }));
    if (p.many) TDB_TRY(launch<loss_logits_many_kernel<DT>>(p.blocks, 512, MANY_SHARED + TileArrays<Logits256<DT>, 2>::BYTES, s, k));
    return launch<loss_finish_kernel<DT>>(p.finish_blocks, 1024, 0, s, k);
}

template <int DT>
hipError_t backward(const tdb_loss_args& a, hipStream_t s) {
    const Plan p = plan_of(a);
    const Loss k = loss_of(a, p);
    Gradient g{};
    char* const work = static_cast<char*>(a.workspace);
    g.dloss = a.dloss, g.dloss_stride = a.dloss_stride, g.dx = a.dx, g.dbias = a.dbias, g.dweight = static_cast<char*>(a.dweight);
    g.dx_stride = a.dx_stride, g.dweight_pitch = a.dweight_stride * p.size;
    g.d = work + p.d, g.d_pitch = p.columns * p.size, g.parts = reinterpret_cast<float*>(work + p.parts), g.part_pitch = p.part_pitch;
    const bool weighted = a.reduction == 0;
    auto floats = [&](int64_t at) { return reinterpret_cast<float*>(work + at); };
    g.shifted = weighted && a.dtype == TDB_F16 ? work + p.shifted : k.gathered;
    g.reach = reinterpret_cast<int32_t*>(work + p.reach), g.scale = floats(p.scale), g.share = floats(p.share), g.shift = floats(p.shift), g.common = floats(p.common), g.column_sums = floats(p.column_sums), g.dw_parts = floats(p.dw_parts), g.dw_splits = a.dweight ? p.dw_splits : 1;
    g.wide_dweight = reinterpret_cast<uintptr_t>(a.dweight) % 4 == 0 && g.dweight_pitch % 4 == 0;
    if (weighted && a.rows && a.dtype == TDB_F16) TDB_TRY(launch<loss_reach_kernel>(std::min<int64_t>(p.padded / 16, 1024), 256, 0, s, k, g));
    if (weighted && a.rows) TDB_TRY(launch<loss_weigh_kernel<DT>>(std::min<int64_t>(p.padded / 16, 1024), 256, 0, s, k, g));
    for (g.first = 0; g.first < a.vocab; g.first += p.columns) {
        g.columns = std::min(p.columns, p.vocab - g.first), g.later = g.first > 0;
        if (weighted) {
            if (p.few) TDB_TRY(few_rows<DT>(p, [&](auto f) { return launch<loss_difference_few_kernel<DT, true, f()>>(Few<DT, f()>::PER_CU * p.blocks, Few<DT, f()>::THREADS, Few<DT, f()>::SHARED, s, k, g); }));
            if (p.many) TDB_TRY(launch<loss_difference_many_kernel<DT, true>>(p.blocks, 512, MANY_SHARED + TileArrays<Logits256<DT>, 7>::BYTES, s, k, g));
        } else {
            if (p.few) TDB_TRY(few_rows<DT>(p, [&](auto f) { return launch<loss_difference_few_kernel<DT, false, f()>>(Few<DT, f()>::PER_CU * p.blocks, Few<DT, f()>::THREADS, Few<DT, f()>::SHARED, s, k, g); }));
            if (p.many) TDB_TRY(launch<loss_difference_many_kernel<DT, false>>(p.blocks, 512, MANY_SHARED + TileArrays<Logits256<DT>, 5>::BYTES, s, k, g));
        }
        if (a.rows && a.dx) {
            if (p.dx_width == 256) TDB_TRY(launch<loss_dx_kernel<DT, 256>>(p.blocks, 512, DX_SHARED, s, k, g));
            else if (p.dx_width == 192) TDB_TRY(launch<loss_dx_kernel<DT, 192>>(p.blocks, 512, DX_SHARED, s, k, g));
            else TDB_TRY(launch<loss_dx_kernel<DT, 128>>(p.blocks, 512, DX_SHARED, s, k, g));
        }
        if (a.dweight || a.dbias) {
            auto dweight = [&](auto width) {
                constexpr int BN = width();
                return g.dw_splits > 1 ? launch<loss_dweight_kernel<DT, BN, true>>(p.blocks, 512, Dweight<DT, BN>::SHARED, s, k, g)
                                       : launch<loss_dweight_kernel<DT, BN, false>>(p.blocks, 512, Dweight<DT, BN>::SHARED, s, k, g);
            };
            if (p.dw_width == 256) TDB_TRY(dweight(std::integral_constant<int, 256>()));
            else if (p.dw_width == 192) TDB_TRY(dweight(std::integral_constant<int, 192>()));
            else TDB_TRY(dweight(std::integral_constant<int, 128>()));
            if (g.dw_splits > 1) TDB_TRY(launch<loss_dweight_sum_kernel<DT>>(std::min<int64_t>((a.vocab * (p.part_pitch / 4) + 255) / 256, 4096), 256, 0, s, k, g));
        }
    }
    if (a.rows && a.dx) {
        g.columns = p.columns;              // (what the parts of dx were shared out by: the first piece's)
        TDB_TRY(launch<loss_dx_sum_kernel<DT>>(std::min<int64_t>(a.rows * ((a.hidden + 255) / 256), 2048), 256, 0, s, k, g, p.blocks, int(p.dx_width)));
    }
    return hipSuccess;
}

int run(const tdb_loss_args* a, bool back, void* stream) {
    if (const int rc = check(a, back); rc != TDB_OK) return rc;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    auto one = [&](auto dt) { return back ? backward<decltype(dt)::value>(*a, s) : forward<decltype(dt)::value>(*a, s); };
    const hipError_t e = a->dtype == TDB_F32 ? one(std::integral_constant<int, TDB_F32>{}) : a->dtype == TDB_BF16 ? one(std::integral_constant<int, TDB_BF16>{}) : one(std::integral_constant<int, TDB_F16>{});
    if (e != hipSuccess) return tdb_fail(TDB_ERR_LAUNCH, "kernel launch failed: %s", hipGetErrorString(e));
    return TDB_OK;
}

}  // namespace tdb_train

extern "C" {

int tdb_loss_fwd(const tdb_loss_args* args, void* stream) { return tdb_train::run(args, false, stream); }
int tdb_loss_bwd(const tdb_loss_args* args, void* stream) { return tdb_train::run(args, true, stream); }
int64_t tdb_loss_state(const tdb_loss_args* args) { return tdb_train::check_sizes(args) == TDB_OK ? tdb_train::plan_of(*args).state : 0; }
int64_t tdb_loss_workspace(const tdb_loss_args* args, int32_t backward) {
    if (tdb_train::check_sizes(args) != TDB_OK) return 0;
    const tdb_train::Plan p = tdb_train::plan_of(*args);
    return backward ? p.backward : p.forward;
}

}  // extern "C"
