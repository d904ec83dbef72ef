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
constexpr int TILE = 256;           // rows that the gathered ones are filled up to with zeros, columns of D
constexpr int FINISH_ROWS = 64;     // rows of a workgroup of the last forward kernel

// float16: D lies in [-2^14, 2^14], so that probabilities down to 2^-38 are told from 0 (2^-24 without).
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
    float *top, *inverse;                       // largest logit (base 2), 1 / sum of exponentials
    char* gathered;
    int64_t pitch;                              // of a gathered row, bytes
    // workspace
    float *right, *maxima, *sums;               // the label's logit; [groups of column tiles][rows]
    double* block_sums;
    int64_t padded;                             // rows, rounded up
    int32_t column_tiles, group;                // of the vocabulary, those that one workgroup takes together
};

template <int DT>
__device__ __forceinline__ float bias_of(const Loss& p, int64_t v) {
    if (v >= p.vocab) return -INFINITY;
    if (!p.bias_kind) return 0.f;
    const float b = p.bias_kind == 2 ? static_cast<const float*>(p.bias)[v] : float(static_cast<const typename Matrix<DT>::T*>(p.bias)[v]);
    const float t = b * LOG2E;
    return fabsf(t) == INFINITY && fabsf(b) != INFINITY ? copysignf(FLT_MAX, b) : t;        // (a mask of the type's lowest value stays a number)
}

__device__ __forceinline__ int block_count(int x, int* scratch) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) x += __shfl_xor(x, d);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = x;
    __syncthreads();
    return scratch[0] + scratch[1] + scratch[2] + scratch[3];
}

// Rows that count, in order: where they come from, their labels, and they themselves, dense, zeros behind them up to a multiple of TILE rows and of the steps' 128 bytes.
// A workgroup has `chunk` rows and counts for itself what lies in front of them.
template <int DT>
__global__ __launch_bounds__(256) void loss_gather_kernel(Loss p, int64_t chunk, bool wide) {
    using T = typename Matrix<DT>::T;
    __shared__ int scratch[4];
    const int wave = threadIdx.x >> 6, l = threadIdx.x & 63;
    const int64_t first = blockIdx.x * chunk, end = min(p.rows, first + chunk);
    int seen = 0;
    for (int64_t i = threadIdx.x; i < first; i += 256) seen += p.labels[i] != p.ignore;
    const int before = block_count(seen, scratch);
    int at = before;
    for (int64_t i0 = first; i0 < end; i0 += 256) {
        const int64_t i = i0 + threadIdx.x;
        const int64_t label = i < end ? p.labels[i] : p.ignore;
        const bool counts = label != p.ignore;
        const uint64_t who = __builtin_amdgcn_ballot_w64(counts);
        __syncthreads();
        if (l == 0) scratch[wave] = __popcll(who);
        __syncthreads();
        int place = at + __popcll(who & ((uint64_t(1) << l) - 1)), all = 0;
#pragma unroll
        for (int v = 0; v < 4; ++v) place += v < wave ? scratch[v] : 0, all += scratch[v];
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
    int fill = at;
    if (blockIdx.x == gridDim.x - 1) {
        if (threadIdx.x == 0) p.count[0] = at;
        fill = (at + TILE - 1) / TILE * TILE;
    }
    __syncthreads();
    const int columns = int(p.pitch / sizeof(T));
    for (int r = before + wave; r < fill; r += 4) {
        char* const to = p.gathered + r * p.pitch;
        const T* const from = reinterpret_cast<const T*>(p.x) + (r < at ? p.index[r] : 0) * p.x_stride;
        if (wide) {
            constexpr int PER = 16 / sizeof(T);
            for (int c = l; c < columns / PER; c += 64) {
                uint4 v = {0, 0, 0, 0};
                if (r < at && c * PER < p.hidden) v = reinterpret_cast<const uint4*>(from)[c];
                reinterpret_cast<uint4*>(to)[c] = v;
            }
        } else {
            for (int c = l; c < columns; c += 64) reinterpret_cast<T*>(to)[c] = r < at && c < p.hidden ? from[c] : T(0.f);
        }
    }
}

// The biases of a tile's columns, in base 2; -inf past the vocabulary.
template <int DT, int BN>
__device__ __forceinline__ void stage_bias(const Loss& p, int64_t n0, float* s_bias) {
    if (threadIdx.x < BN) s_bias[threadIdx.x] = bias_of<DT>(p, n0 + threadIdx.x);
}

// Forward: of each gathered row and group of column tiles the largest logit and the sum of exponentials relative to it.
template <int DT, class P, int BM, int BN, int WN>
__global__ __launch_bounds__(P::WAVES * 64, 2) void loss_logits_kernel(Loss p) {
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    __shared__ float s_bias[BN], s_top[WN][BM], s_sum[WN][BM];
    using M = Matrix<DT>;
    const int n = p.count[0];
    const int64_t row_tiles = (n + BM - 1) / BM, groups = (p.column_tiles + p.group - 1) / p.group, all = row_tiles * groups;
    const Rows a{p.gathered, p.pitch, p.padded, uint32_t(p.pitch)}, b{p.w, p.w_pitch, p.vocab, uint32_t((p.hidden * sizeof(typename M::T) + 15) / 16 * 16)};
    for (int64_t block = blockIdx.x; block < all; block += gridDim.x) {
        int64_t row, g, split;
        tile_of(block, row_tiles, groups, 1, row, g, split);
        const int64_t m0 = row * BM;
        float top[P::TM], sum[P::TM];
#pragma unroll
        for (int i = 0; i < P::TM; ++i) top[i] = -FLT_MAX, sum[i] = 0.f;
        for (int64_t t = g * p.group; t < min(int64_t(p.column_tiles), (g + 1) * p.group); ++t) {
            const int64_t n0 = t * BN;
            typename P::Acc acc;
            P::run(smem, a, b, m0, n0, 0, p.pitch / 128, acc);
            stage_bias<DT, BN>(p, n0, s_bias);
            __syncthreads();
#pragma unroll
            for (int i = 0; i < P::TM; ++i) {
                const int64_t m = m0 + P::wave_m() + i * M::SIDE + lane_m<DT>();
                float most = top[i];
                f32x4 s[P::TN][M::QUADS];
#pragma unroll
                for (int j = 0; j < P::TN; ++j)
#pragma unroll
                    for (int q = 0; q < M::QUADS; ++q) {
                        const f32x4 v = P::quad(acc, i, j, q), bias = *reinterpret_cast<const f32x4*>(s_bias + P::wave_n() + j * M::SIDE + quad_n<DT>(q));
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            s[j][q][e] = fmaf(v[e], LOG2E, bias[e]);
                            most = fmaxf(most, s[j][q][e]);
                        }
                    }
                float more = 0.f;
#pragma unroll
                for (int j = 0; j < P::TN; ++j)
#pragma unroll
                    for (int q = 0; q < M::QUADS; ++q)
#pragma unroll
                        for (int e = 0; e < 4; ++e) more += __builtin_amdgcn_exp2f(s[j][q][e] - most);
                sum[i] = sum[i] * __builtin_amdgcn_exp2f(top[i] - most) + more;
                top[i] = most;
                // The label's own logit, in the one tile that has it.
                const int64_t label = m < n ? p.label[m] : -1, rel = label - n0 - P::wave_n();
                const bool here = label >= 0 && rel >= 0 && rel < P::TN * M::SIDE;
                if (__builtin_amdgcn_ballot_w64(here)) {
#pragma unroll
                    for (int j = 0; j < P::TN; ++j)
#pragma unroll
                        for (int q = 0; q < M::QUADS; ++q)
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                if (here && rel == j * M::SIDE + quad_n<DT>(q) + e) p.right[m] = s[j][q][e];
                }
            }
        }
#pragma unroll
        for (int i = 0; i < P::TM; ++i) {
            const float most = over_quads<DT>(top[i], [](float x, float y) { return fmaxf(x, y); });
            const float s = over_quads<DT>(sum[i] * __builtin_amdgcn_exp2f(top[i] - most), [](float x, float y) { return x + y; });
            const int at = P::wave_m() + i * M::SIDE + lane_m<DT>(), w = P::wave_n() / (P::TN * M::SIDE);
            s_top[w][at] = most, s_sum[w][at] = s;
        }
        __syncthreads();
        if (threadIdx.x < BM) {
            float most = s_top[0][threadIdx.x], s = 0.f;
#pragma unroll
            for (int w = 1; w < WN; ++w) most = fmaxf(most, s_top[w][threadIdx.x]);
#pragma unroll
            for (int w = 0; w < WN; ++w) s += s_sum[w][threadIdx.x] * __builtin_amdgcn_exp2f(s_top[w][threadIdx.x] - most);
            p.maxima[g * p.padded + m0 + threadIdx.x] = most;
            p.sums[g * p.padded + m0 + threadIdx.x] = s;
        }
    }
}

// The rows' losses and what the gradient needs of them; their sum by the workgroup that ends last.  A workgroup has 64 rows, its waves share the groups of columns out.
template <int DT>
__global__ __launch_bounds__(256) void loss_finish_kernel(Loss p) {
    __shared__ float s_top[4][64], s_sum[4][64];
    __shared__ double s_all[256];
    __shared__ bool s_last;
    const int n = p.count[0], l = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int groups = (p.column_tiles + p.group - 1) / p.group, fill = (n + TILE - 1) / TILE * TILE;
    double mine = 0.0;
    for (int64_t r0 = int64_t(blockIdx.x) * FINISH_ROWS; r0 < fill; r0 += int64_t(gridDim.x) * FINISH_ROWS) {
        const int64_t r = r0 + l;
        float top = -FLT_MAX, sum = 0.f;
        if (r < n)
            for (int g = w; g < groups; g += 16) {
                float t[4], s[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int at = min(g + 4 * u, groups - 1);
                    t[u] = p.maxima[at * p.padded + r], s[u] = p.sums[at * p.padded + r];
                }
                float most = top;
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    if (g + 4 * u < groups) most = fmaxf(most, t[u]);
                sum *= __builtin_amdgcn_exp2f(top - most);
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    if (g + 4 * u < groups) sum += s[u] * __builtin_amdgcn_exp2f(t[u] - most);
                top = most;
            }
        __syncthreads();
        s_top[w][l] = top, s_sum[w][l] = sum;
        __syncthreads();
        if (w == 0) {
#pragma unroll
            for (int v = 0; v < 4; ++v) top = fmaxf(top, s_top[v][l]);
            sum = 0.f;
#pragma unroll
            for (int v = 0; v < 4; ++v) sum += s_sum[v][l] * __builtin_amdgcn_exp2f(s_top[v][l] - top);
            if (r < n) {
                const float loss = ((top - p.right[r]) + log2f(sum)) * LN2;
                p.top[r] = p.label[r] < 0 ? __builtin_nanf("") : top;
                p.inverse[r] = D_SCALE<DT> / sum;
                if (p.reduction == 0) p.loss[p.index[r]] = loss;
                mine += loss;
            } else if (r < fill) {
                p.top[r] = 0.f, p.inverse[r] = 0.f;
            }
        }
    }
    if (p.reduction == 0) return;
    s_all[threadIdx.x] = mine;
    __syncthreads();
    for (int d = 32; d > 0; d >>= 1) {
        if (threadIdx.x < d) s_all[threadIdx.x] += s_all[threadIdx.x + d];
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        __hip_atomic_store(p.block_sums + blockIdx.x, s_all[0], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        s_last = __hip_atomic_fetch_add(p.count + 1, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == int(gridDim.x) - 1;
    }
    __syncthreads();
    if (!s_last) return;
    double sum = 0.0;
    for (unsigned i = threadIdx.x; i < gridDim.x; i += 256) sum += __hip_atomic_load(p.block_sums + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    s_all[threadIdx.x] = sum;
    __syncthreads();
    for (int d = 128; d > 0; d >>= 1) {
        if (threadIdx.x < d) s_all[threadIdx.x] += s_all[threadIdx.x + d];
        __syncthreads();
    }
    if (threadIdx.x == 0) p.loss[0] = float(p.reduction == 2 ? s_all[0] / double(n) : s_all[0]);
}

// What the gradient needs beside Loss.
struct Gradient {
    const float* dloss;
    int64_t dloss_stride;
    void *dx, *dbias;
    char* dweight;
    int64_t dx_stride, dweight_pitch;
    char* d;                    // [padded rows][columns of a piece]
    int64_t d_pitch;
    int64_t first, columns;     // of the piece (columns a multiple of TILE)
    float* parts;               // of dx, [splits][rows that count, rounded up to tiles][part_pitch]
    int64_t part_pitch;
    // Where every row has a gradient g of its own, it goes into D (g <- g / common), in float16 without its power of two, which the row itself takes (x <- x shift).
    char* shifted;              // gathered rows times shift; the gathered rows themselves otherwise
    float *scale, *share, *shift, *common;      // inverse times g; g; 1 but in float16; a power of two
    float* column_sums;         // of D, [tiles of rows][columns]
    bool wide_dweight, later;   // later: a piece that is not the first
};

// D of a piece of the vocabulary.
template <int DT, class P, int BM, int BN, int WM, bool WEIGHTED>
__global__ __launch_bounds__(P::WAVES * 64, 2) void loss_difference_kernel(Loss p, Gradient g) {
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    __shared__ float s_bias[BN], s_column[WM][BN];
    using M = Matrix<DT>;
    const int n = p.count[0];
    const int64_t row_tiles = (n + BM - 1) / BM, column_tiles = g.columns / BN, all = row_tiles * column_tiles;
    const Rows a{p.gathered, p.pitch, p.padded, uint32_t(p.pitch)}, b{p.w, p.w_pitch, p.vocab, uint32_t((p.hidden * sizeof(typename M::T) + 15) / 16 * 16)};
    for (int64_t block = blockIdx.x; block < all; block += gridDim.x) {
        int64_t row, column, split;
        tile_of(block, row_tiles, column_tiles, 1, row, column, split);
        const int64_t m0 = row * BM, n0 = g.first + column * BN;
        typename P::Acc acc;
        P::run(smem, a, b, m0, n0, 0, p.pitch / 128, acc);
        stage_bias<DT, BN>(p, n0, s_bias);
        float top[P::TM], scale[P::TM], share[P::TM], shift[P::TM];
        int rel[P::TM];
#pragma unroll
        for (int i = 0; i < P::TM; ++i) {
            const int64_t m = m0 + P::wave_m() + i * M::SIDE + lane_m<DT>();
            top[i] = p.top[m], scale[i] = WEIGHTED ? g.scale[m] : p.inverse[m];
            share[i] = WEIGHTED ? g.share[m] : D_SCALE<DT>, shift[i] = WEIGHTED && DT == TDB_F16 ? g.shift[m] : 1.f;
            rel[i] = m < n ? p.label[m] - int(n0) - P::wave_n() : -1;
        }
        __syncthreads();
        float sums[P::TN * M::QUADS * 4];
#pragma unroll
        for (int c = 0; c < P::TN * M::QUADS * 4; ++c) sums[c] = 0.f;
        P::store(smem, g.d, g.d_pitch, m0, p.padded, n0 - g.first, g.columns, true, [&](int i, int j, int q) {
            const f32x4 v = P::quad(acc, i, j, q), bias = *reinterpret_cast<const f32x4*>(s_bias + P::wave_n() + j * M::SIDE + quad_n<DT>(q));
            f32x4 d;
#pragma unroll
            for (int e = 0; e < 4; ++e) d[e] = __builtin_amdgcn_exp2f(fmaf(v[e], LOG2E, bias[e]) - top[i]) * scale[i];
            const int at = rel[i] - j * M::SIDE - quad_n<DT>(q);
            if (__builtin_amdgcn_ballot_w64(at >= 0 && at < 4)) {
#pragma unroll
                for (int e = 0; e < 4; ++e) d[e] -= at == e ? share[i] : 0.f;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) sums[(j * M::QUADS + q) * 4 + e] += d[e] * shift[i];
            return d;
        });
        if (g.dbias) {
            const float sum = over_m<DT>(sums);
            constexpr int N = P::TN * M::QUADS * 4;
            const int c = lane_m<DT>() % N;     // the value that the lane has
            if (lane_m<DT>() < N) s_column[P::wave_m() / (P::TM * M::SIDE)][P::wave_n() + c / (4 * M::QUADS) * M::SIDE + quad_n<DT>(c / 4 % M::QUADS) + c % 4] = sum;
            __syncthreads();
            if (threadIdx.x < BN) {
                float all = 0.f;
#pragma unroll
                for (int w = 0; w < WM; ++w) all += s_column[w][threadIdx.x];
                g.column_sums[row * g.columns + n0 - g.first + threadIdx.x] = all;
            }
        }
    }
}

// Parts of dx: D W over a share of the piece's columns.
template <int DT, class P, int BM, int BN>
__global__ __launch_bounds__(P::WAVES * 64, 2) void loss_dx_kernel(Loss p, Gradient g) {
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    using M = Matrix<DT>;
    const int n = p.count[0];
    const int64_t row_tiles = (n + BM - 1) / BM, column_tiles = (p.hidden + BN - 1) / BN, tiles = row_tiles * column_tiles, steps = g.columns / P::STEP;
    const int64_t splits = tiles ? max(int64_t(1), min(int64_t(gridDim.x) / tiles, steps)) : 0, all = tiles * splits;
    const Rows a{g.d, g.d_pitch, p.padded, uint32_t(g.d_pitch)};
    const Rows b{p.w + g.first * p.w_pitch, p.w_pitch, min(g.columns, p.vocab - g.first), uint32_t((p.hidden * sizeof(typename M::T) + 15) / 16 * 16)};
    for (int64_t block = blockIdx.x; block < all; block += gridDim.x) {
        int64_t row, column, split;
        tile_of(block, row_tiles, column_tiles, splits, row, column, split);
        const int64_t m0 = row * BM, n0 = column * BN;
        typename P::Acc acc;
        P::run(smem, a, b, m0, n0, steps * split / splits, steps * (split + 1) / splits, acc);
#pragma unroll
        for (int i = 0; i < P::TM; ++i) {
            const int64_t m = m0 + P::wave_m() + i * M::SIDE + lane_m<DT>();
            float* const to = g.parts + (split * row_tiles * BM + m) * g.part_pitch;
#pragma unroll
            for (int j = 0; j < P::TN; ++j)
#pragma unroll
                for (int q = 0; q < M::QUADS; ++q) {
                    const int64_t c = n0 + P::wave_n() + j * M::SIDE + quad_n<DT>(q);
                    if (m < n && c < g.part_pitch) {
                        f32x4 v = P::quad(acc, i, j, q);
                        if (g.later) v += *reinterpret_cast<const f32x4*>(to + c);
                        *reinterpret_cast<f32x4*>(to + c) = v;
                    }
                }
        }
    }
}

// What the gradient of a sum or mean makes of every row.
__device__ __forceinline__ float row_factor(const Loss& p, const Gradient& g, int n) { return p.reduction == 2 ? g.dloss[0] / float(n) : g.dloss[0]; }

// dx: a workgroup for each row, zeros where it does not count.  blocks, tiles: of the launch before.
template <int DT>
__global__ __launch_bounds__(256) void loss_dx_sum_kernel(Loss p, Gradient g, int blocks, int bm, int bn) {
    using T = typename Matrix<DT>::T;
    constexpr int STEP = 128 / sizeof(T);
    const int n = p.count[0];
    const int64_t high = int64_t((n + bm - 1) / bm), tiles = high * ((p.hidden + bn - 1) / bn);
    const int64_t splits = tiles ? max(int64_t(1), min(int64_t(blocks) / tiles, g.columns / STEP)) : 0;
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const int place = p.place[row];
        T* const to = static_cast<T*>(g.dx) + row * g.dx_stride;
        if (place < 0) {
            for (int c = threadIdx.x; c < p.hidden; c += 256) to[c] = T(0.f);
            continue;
        }
        const float factor = (p.reduction ? row_factor(p, g, n) : *g.common * g.shift[place]) * (1.f / D_SCALE<DT>);
        for (int c = threadIdx.x; c < p.hidden; c += 256) {
            float sum = 0.f;
#pragma unroll 8
            for (int64_t s = 0; s < splits; ++s) sum += g.parts[(s * high * bm + place) * g.part_pitch + c];
            to[c] = T(sum * factor);
        }
    }
}

// Rows with gradients of their own.  common is the power of two of the largest; float16: a row's own power of two, relative to that, goes to x, which takes it without rounding.
template <int DT>
__global__ __launch_bounds__(256) void loss_weigh_kernel(Loss p, Gradient g) {
    using T = typename Matrix<DT>::T;
    __shared__ float s_most[4];
    const int n = p.count[0], l = threadIdx.x & 63, w = threadIdx.x >> 6, fill = (n + TILE - 1) / TILE * TILE;
    float most = 0.f;
    for (int r = threadIdx.x; r < n; r += 256) most = fmaxf(most, fabsf(g.dloss[p.index[r] * g.dloss_stride]));
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) most = fmaxf(most, __shfl_xor(most, d));
    if (l == 0) s_most[w] = most;
    __syncthreads();
    most = fmaxf(fmaxf(s_most[0], s_most[1]), fmaxf(s_most[2], s_most[3]));
    const int common = most > 0.f && most < INFINITY ? ilogbf(most) : 0;
    if (blockIdx.x == 0 && threadIdx.x == 0) *g.common = ldexpf(1.f, common);
    for (int r = blockIdx.x * 4 + w; r < fill; r += gridDim.x * 4) {
        const float weight = r < n ? g.dloss[p.index[r] * g.dloss_stride] : 0.f;
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
template <int DT, class P, int BM, int BN>
__global__ __launch_bounds__(P::WAVES * 64, 2) void loss_dweight_kernel(Loss p, Gradient g) {
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    using M = Matrix<DT>;
    using T = typename M::T;
    const int n = p.count[0];
    const int64_t columns = min(g.columns, p.vocab - g.first), row_tiles = (columns + BM - 1) / BM, column_tiles = g.dweight ? (p.hidden + BN - 1) / BN : 1, all = row_tiles * column_tiles;
    const int64_t steps = (n + P::STEP - 1) / P::STEP;
    const Rows a{g.d, g.d_pitch, p.padded, uint32_t(g.d_pitch)}, b{g.shifted, p.pitch, p.padded, uint32_t(p.pitch)};
    const float factor = n == 0 ? 0.f : (p.reduction ? row_factor(p, g, n) : *g.common) * (1.f / D_SCALE<DT>);
    for (int64_t block = blockIdx.x; block < all; block += gridDim.x) {
        int64_t row, column, split;
        tile_of(block, row_tiles, column_tiles, 1, row, column, split);
        const int64_t m0 = row * BM, n0 = column * BN, m = m0 + threadIdx.x;
        if (g.dbias && column == 0 && threadIdx.x < BM && m < columns) {
            float sum = 0.f;
            for (int t = 0; t < (n + TILE - 1) / TILE; ++t) sum += g.column_sums[t * g.columns + m];
            if (p.bias_kind == 2) static_cast<float*>(g.dbias)[g.first + m] = sum * factor;
            else static_cast<T*>(g.dbias)[g.first + m] = T(sum * factor);
        }
        if (!g.dweight) continue;
        typename P::Acc acc;
        P::run(smem, a, b, m0, n0, 0, steps, acc);
        P::store(smem, g.dweight + g.first * g.dweight_pitch, g.dweight_pitch, m0, columns, n0, p.hidden, g.wide_dweight, [&](int i, int j, int q) {
            f32x4 v = P::quad(acc, i, j, q);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] *= factor;
            return v;
        });
    }
}

// ------------------------------------------------------------------------------------------------------------------- host

constexpr int64_t D_BYTES = int64_t(1) << 31;       // of the workspace that holds D, unless 256 columns take more
constexpr int64_t PARTIAL_BYTES = int64_t(1) << 27;

int64_t round_up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }

struct Plan {
    int size;                               // of a value
    int64_t padded, pitch, vocab;           // rows and bytes of the gathered rows, vocabulary, rounded up
    int32_t column_tiles, group, groups;
    int64_t columns;                        // of a piece
    int blocks, finish_blocks;
    // offsets
    int64_t index, place, label, top, inverse, gathered, state;
    int64_t right, maxima, sums, block_sums, forward;
    int64_t d, parts, part_pitch, column_sums, shifted, scale, share, shift, common, backward;
};

Plan plan_of(const tdb_loss_args& a) {
    Plan p;
    p.size = a.dtype == TDB_F32 ? 4 : 2;
    p.padded = round_up(std::max<int64_t>(a.rows, 1), TILE);
    p.pitch = round_up(int64_t(a.hidden) * p.size, 128);
    p.vocab = round_up(a.vocab, TILE);
    p.column_tiles = int32_t(p.vocab / TILE);
    p.group = int32_t((int64_t(p.column_tiles) * p.padded * 8 + PARTIAL_BYTES - 1) / PARTIAL_BYTES);
    p.groups = (p.column_tiles + p.group - 1) / p.group;
    const int64_t most = std::min<int64_t>(std::max<int64_t>(D_BYTES / (p.padded * p.size) / TILE, 1), (int64_t(1) << 22) / p.size / TILE), pieces = (p.column_tiles + most - 1) / most;
    p.columns = (p.column_tiles + pieces - 1) / pieces * TILE;
    p.blocks = std::max(8, tdb_compute_units(-1) & -8);
    p.finish_blocks = int(std::min<int64_t>(p.padded / FINISH_ROWS, 1024));
    int64_t at = 256;
    auto take = [&](int64_t bytes) {
        const int64_t here = at;
        at += round_up(bytes, 256);
        return here;
    };
    p.index = take(p.padded * 4), p.place = take(p.padded * 4), p.label = take(p.padded * 4), p.top = take(p.padded * 4), p.inverse = take(p.padded * 4);
    p.gathered = take(p.padded * p.pitch);
    p.state = at;
    at = 0;
    p.right = take(p.padded * 4), p.maxima = take(p.groups * p.padded * 4), p.sums = take(p.groups * p.padded * 4), p.block_sums = take(p.finish_blocks * 8);
    p.forward = at;
    at = 0;
    p.part_pitch = round_up(a.hidden, 4);
    // As many parts of dx as workgroups share its tiles, or one.
    p.d = take(p.padded * p.columns * p.size);
    p.parts = take(std::max(p.padded, int64_t(p.blocks) * TILE) * std::max<int64_t>(p.part_pitch, 1) * 4);
    p.column_sums = take(p.padded / TILE * p.columns * 4);
    const bool weighted = a.reduction == 0;
    p.shifted = take(weighted && a.dtype == TDB_F16 ? p.padded * p.pitch : 0);
    p.scale = take(weighted ? p.padded * 4 : 0), p.share = take(weighted ? p.padded * 4 : 0), p.shift = take(weighted ? p.padded * 4 : 0), p.common = take(4);
    p.backward = at;
    return p;
}

int check(const tdb_loss_args* a, bool backward) {
    if (!a) return tdb_fail(TDB_ERR_NULL, "args is NULL");
    if (a->dtype != TDB_F32 && a->dtype != TDB_BF16 && a->dtype != TDB_F16) return tdb_fail(TDB_ERR_DTYPE, "unknown dtype %d", a->dtype);
    if (a->bias && a->bias_dtype != a->dtype && a->bias_dtype != TDB_F32) return tdb_fail(TDB_ERR_DTYPE, "bias_dtype %d: need that of x, or float32", a->bias_dtype);
    if (a->rows < 0 || a->rows > (1 << 27) || a->vocab < 1 || a->vocab > (1 << 27) || a->hidden < 1 || a->hidden > 32768)
        return tdb_fail(TDB_ERR_SHAPE, "%lld rows, %d columns, %lld classes: need up to 2^27, 1 to 32768, 1 to 2^27", (long long)a->rows, a->hidden, (long long)a->vocab);
    if (a->reduction < 0 || a->reduction > 2) return tdb_fail(TDB_ERR_SHAPE, "reduction %d: need 0 (none), 1 (sum) or 2 (mean)", a->reduction);
    const int size = a->dtype == TDB_F32 ? 4 : 2;
    if (!a->weight || !a->state || !a->workspace) return tdb_fail(TDB_ERR_NULL, "weight, state and workspace must be non-NULL");
    if (a->weight_stride * size % 16 || a->weight_stride * size < round_up(int64_t(a->hidden) * size, 16) || a->weight_stride * size > (1 << 22))
        return tdb_fail(TDB_ERR_STRIDE, "weight_stride %lld: need whole 16 bytes, at least a row and at most 4 MiB", (long long)a->weight_stride);
    for (const void* t : {a->weight, static_cast<const void*>(a->state), static_cast<const void*>(a->workspace)})
        if (reinterpret_cast<uintptr_t>(t) % 16) return tdb_fail(TDB_ERR_ALIGN, "weight, state and workspace must be 16-byte aligned");
    if (!backward) {
        if (a->rows && (!a->x || !a->labels)) return tdb_fail(TDB_ERR_NULL, "x and labels must be non-NULL");
        if (a->x_stride < 0) return tdb_fail(TDB_ERR_STRIDE, "negative row stride");
        if (!a->loss && (a->rows || a->reduction)) return tdb_fail(TDB_ERR_NULL, "loss must be non-NULL");
    } else {
        if (a->rows && !a->dloss) return tdb_fail(TDB_ERR_NULL, "dloss must be non-NULL");
        if (a->dbias && !a->bias) return tdb_fail(TDB_ERR_NULL, "dbias needs a bias");
        if (a->dloss_stride < 0 || (a->dx && a->rows > 1 && a->dx_stride < a->hidden) || (a->dweight && a->dweight_stride < a->hidden))
            return tdb_fail(TDB_ERR_STRIDE, "rows of a result overlap");
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
    k.gathered = state + p.gathered, k.pitch = p.pitch, k.padded = p.padded, k.column_tiles = p.column_tiles, k.group = p.group;
    k.right = reinterpret_cast<float*>(work + p.right), k.maxima = reinterpret_cast<float*>(work + p.maxima), k.sums = reinterpret_cast<float*>(work + p.sums);
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
    TDB_TRY(launch<loss_gather_kernel<DT>>(std::max<int64_t>(1, (a.rows + chunk - 1) / chunk), 256, 0, s, k, chunk, wide));
    using P = Product<DT, 256, 256, 2, 4, 2, false, false>;
    if (a.rows) TDB_TRY(launch<loss_logits_kernel<DT, P, 256, 256, 4>>(p.blocks, P::WAVES * 64, P::SHARED, s, k));
    return launch<loss_finish_kernel<DT>>(p.finish_blocks, 256, 0, s, k);
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
    g.scale = floats(p.scale), g.share = floats(p.share), g.shift = floats(p.shift), g.common = floats(p.common), g.column_sums = floats(p.column_sums);
    g.wide_dweight = reinterpret_cast<uintptr_t>(a.dweight) % 16 == 0 && g.dweight_pitch % 16 == 0 && int64_t(a.hidden) * p.size % 16 == 0;
    if (weighted && a.rows) TDB_TRY(launch<loss_weigh_kernel<DT>>(std::min<int64_t>(p.padded / 16, 1024), 256, 0, s, k, g));
    using Lined = Product<DT, 256, 256, 2, 4, 2, false, false>;
    using Across = Product<DT, 256, 256, 2, 4, 2, false, true>;
    using Turned = Product<DT, 256, 256, 2, 4, 2, true, true>;
    for (g.first = 0; g.first < a.vocab; g.first += p.columns) {
        g.columns = std::min(p.columns, p.vocab - g.first), g.later = g.first > 0;
        if (a.rows && weighted) TDB_TRY(launch<loss_difference_kernel<DT, Lined, 256, 256, 2, true>>(p.blocks, Lined::WAVES * 64, Lined::SHARED, s, k, g));
        else if (a.rows) TDB_TRY(launch<loss_difference_kernel<DT, Lined, 256, 256, 2, false>>(p.blocks, Lined::WAVES * 64, Lined::SHARED, s, k, g));
        if (a.rows && a.dx) TDB_TRY(launch<loss_dx_kernel<DT, Across, 256, 256>>(p.blocks, Across::WAVES * 64, Across::SHARED, s, k, g));
        if (a.dweight || a.dbias) TDB_TRY(launch<loss_dweight_kernel<DT, Turned, 256, 256>>(p.blocks, Turned::WAVES * 64, Turned::SHARED, s, k, g));
    }
    if (a.rows && a.dx) {
        g.columns = p.columns;              // (what the parts of dx were shared out by: the first piece's)
        TDB_TRY(launch<loss_dx_sum_kernel<DT>>(std::min<int64_t>(a.rows, 1 << 16), 256, 0, s, k, g, p.blocks, 256, 256));
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
int64_t tdb_loss_state(const tdb_loss_args* args) { return args ? tdb_train::plan_of(*args).state : 0; }
int64_t tdb_loss_workspace(const tdb_loss_args* args, int32_t backward) {
    if (!args) return 0;
    const tdb_train::Plan p = tdb_train::plan_of(*args);
    return backward ? p.backward : p.forward;
}

}  // extern "C"
