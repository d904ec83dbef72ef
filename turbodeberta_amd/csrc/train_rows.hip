// Dropout, and LayerNorm with dropout and a residual in front of it, forward and backward.  All of it is bound by memory: a pass reads its inputs and
// writes its results once, and what lies between (masks, sums, statistics) is computed again rather than stored.
//   * A wave has a row in registers, 8 columns a lane at a time, so mean and variance are taken from the row itself in two passes (no difference of large
//     sums) and reduce inside the wave.
//   * The generator makes the numbers of 8 neighbouring columns at once: one call for each chunk of 8.
//   * Backward: the workgroups share the rows out among themselves, each wave keeps its rows' part of the weight's and bias's gradient in registers;
//     the waves of a workgroup are added up in LDS, the workgroups by a second launch in a fixed order: no atomics, the same bits every time.
//   * Rows of other widths than multiples of 8, wider than 2048 or not aligned to 16 bytes: a workgroup per row, a column a lane at a time, the row in LDS.
// Measured, with what a pass reads and writes: dropout of 16384 x 1024 float32 22 us (134 MB, 6.0 TB/s); LayerNorm of 16384 x 768 bfloat16 forward 11.5 us (50 MB, 4.4 TB/s),
// backward 20.1 (76 MB, 3.8 TB/s) and the sum of the parts 3.8; with dropout and residual, 16384 x 1024 forward 18.1 (101 MB, 5.6 TB/s), backward 31.6 (168 MB, 5.3 TB/s) and 4.1. A
// large copy makes 5.0 TB/s; what was written just before is still in the last cache.
#include <algorithm>

#include "philox.h"
#include "tdb_error.h"
#include "tdb_internal.h"
#include "tdb_train.h"

namespace {

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;

template <int DT>
struct Elem;
template <>
struct Elem<TDB_BF16> {
    using T = __bf16;
};
template <>
struct Elem<TDB_F16> {
    using T = _Float16;
};
template <>
struct Elem<TDB_F32> {
    using T = float;
};

template <int DT>
__device__ __forceinline__ void load8(const void* p, int64_t at, float (&v)[8]) {
    using T = typename Elem<DT>::T;
    typedef __attribute__((ext_vector_type(8))) T T8;
    const T8 x = *reinterpret_cast<const T8*>(static_cast<const T*>(p) + at);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = float(x[i]);
}
template <int DT>
__device__ __forceinline__ void store8(void* p, int64_t at, const float (&v)[8]) {
    using T = typename Elem<DT>::T;
    typedef __attribute__((ext_vector_type(8))) T T8;
    T8 x;
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = T(v[i]);
    *reinterpret_cast<T8*>(static_cast<T*>(p) + at) = x;
}
// Weights are of the rows' type or float32.
template <int DT>
__device__ __forceinline__ void load_weight8(const void* p, bool wide, int64_t at, float (&v)[8]) {
    if (wide) load8<TDB_F32>(p, at, v);
    else load8<DT>(p, at, v);
}
template <int DT>
__device__ __forceinline__ float load1(const void* p, int64_t at) {
    return float(static_cast<const typename Elem<DT>::T*>(p)[at]);
}
template <int DT>
__device__ __forceinline__ void store1(void* p, int64_t at, float v) {
    static_cast<typename Elem<DT>::T*>(p)[at] = typename Elem<DT>::T(v);
}
template <int DT>
__device__ __forceinline__ float load_weight1(const void* p, bool wide, int64_t at) {
    return wide ? load1<TDB_F32>(p, at) : load1<DT>(p, at);
}

// Sum over the wave, in every lane: four steps inside the rows of 16 lanes, then the swaps of rows.
__device__ __forceinline__ float wave_sum(float x) {
    auto turn = [](float v, auto ctrl) {
        return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), decltype(ctrl)::value, 0xf, 0xf, true));
    };
    x += turn(x, std::integral_constant<int, 0x128>{});     // row_ror:8
    x += turn(x, std::integral_constant<int, 0x124>{});
    x += turn(x, std::integral_constant<int, 0x122>{});
    x += turn(x, std::integral_constant<int, 0x121>{});
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const uint32_t w = __builtin_bit_cast(uint32_t, __builtin_bit_cast(float, uint32_t(r[0])) + __builtin_bit_cast(float, uint32_t(r[1])));
    const auto s = __builtin_amdgcn_permlane32_swap(w, w, false, false);
    return __builtin_bit_cast(float, uint32_t(s[0])) + __builtin_bit_cast(float, uint32_t(s[1]));
}

// Kept values of chunk `chunk` (8 values) of the numbering.
__device__ __forceinline__ uint32_t kept8(uint64_t chunk, uint32_t threshold, TdbKey key) {
    return tdb_kept(tdb_philox(uint32_t(chunk), uint32_t(chunk >> 32), 0, 0, key), threshold);
}
__device__ __forceinline__ bool kept1(uint64_t at, uint32_t threshold, TdbKey key) { return kept8(at >> 3, threshold, key) >> (at & 7) & 1; }

__device__ __forceinline__ void drop8(float (&v)[8], uint32_t kept, float factor) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (kept >> i & 1) ? v[i] * factor : 0.f;
}

template <int DT, bool ALIGNED>
__global__ __launch_bounds__(256) void dropout_kernel(const void* x, void* y, int64_t n, uint32_t threshold, float factor, const int64_t* seed) {
    const TdbKey key = threshold ? tdb_key(seed) : TdbKey{0, 0};
    const int64_t chunks = (n + 7) / 8, step = int64_t(gridDim.x) * 256;
    for (int64_t c = int64_t(blockIdx.x) * 256 + threadIdx.x; c < chunks; c += step) {
        if (ALIGNED && 8 * c + 8 <= n) {
            float v[8];
            load8<DT>(x, 8 * c, v);
            drop8(v, kept8(c, threshold, key), factor);
            store8<DT>(y, 8 * c, v);
        } else {
            const uint32_t kept = kept8(c, threshold, key);
            const int64_t end = min(n, 8 * c + 8);
            for (int64_t i = 8 * c; i < end; ++i) store1<DT>(y, i, (kept >> (i & 7) & 1) ? load1<DT>(x, i) * factor : 0.f);
        }
    }
}

struct Norm {
    const void *x, *residual, *weight, *bias, *dy;
    void *y, *dx, *dresidual;
    float* partial;
    const int64_t* seed;
    int64_t xs, rs, dys, ys, dxs, drs, rows;
    uint32_t threshold;
    float factor, eps;
    int hidden;
    bool wide;              // weights in float32
};

// What a wave has of a row: chunks l, l + 64, ... of 8 columns; zeros past the row.
template <int CH>
using Row = float[CH][8];

// A row as it lies in memory, on its way: x, the residual, dy.
template <int DT, int CH, bool RES, bool DY>
struct Raw {
    using T = typename Elem<DT>::T;
    typedef __attribute__((ext_vector_type(8))) T T8;
    T8 x[CH], r[RES ? CH : 1], dy[DY ? CH : 1];
    __device__ __forceinline__ void load(const Norm& p, int64_t t) {
        const int l = threadIdx.x & 63, chunks = p.hidden / 8;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int at = 8 * min(l + 64 * c, chunks - 1);         // (past the row: read, not used)
            x[c] = *reinterpret_cast<const T8*>(static_cast<const T*>(p.x) + t * p.xs + at);
            if constexpr (RES) r[c] = *reinterpret_cast<const T8*>(static_cast<const T*>(p.residual) + t * p.rs + at);
            if constexpr (DY) dy[c] = *reinterpret_cast<const T8*>(static_cast<const T*>(p.dy) + t * p.dys + at);
        }
    }
    // z of row t, zeros past the row
    __device__ __forceinline__ void z_of(const Norm& p, int64_t t, TdbKey key, Row<CH>& z, uint32_t (&kept)[CH]) const {
        const int l = threadIdx.x & 63, chunks = p.hidden / 8;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            kept[c] = 0xff;
#pragma unroll
            for (int i = 0; i < 8; ++i) z[c][i] = float(x[c][i]);
            if (p.threshold) {
                kept[c] = kept8(uint64_t(t) * chunks + l + 64 * c, p.threshold, key);
                drop8(z[c], kept[c], p.factor);
            }
            if constexpr (RES) {
#pragma unroll
                for (int i = 0; i < 8; ++i) z[c][i] += float(r[c][i]);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) z[c][i] = l + 64 * c < chunks ? z[c][i] : 0.f;
        }
    }
};
// Whether a wave has registers for the next row while it works on one.
template <int DT, int CH>
constexpr bool AHEAD = CH <= 2;

// z -> z - mean, zeros past the row; returns 1 / standard deviation
template <int CH>
__device__ __forceinline__ float centre(Row<CH>& z, int hidden, float eps) {
    const int l = threadIdx.x & 63, chunks = hidden / 8;
    float sum = 0.f, sq = 0.f;
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) sum += z[c][i];
    const float mean = wave_sum(sum) / float(hidden);
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            z[c][i] = l + 64 * c < chunks ? z[c][i] - mean : 0.f;
            sq += z[c][i] * z[c][i];
        }
    return rsqrtf(wave_sum(sq) / float(hidden) + eps);
}

template <int DT, int CH, bool RES>
__global__ __launch_bounds__(256) void norm_fwd_kernel(Norm p) {
    const int l = threadIdx.x & 63, chunks = p.hidden / 8;
    const TdbKey key = p.threshold ? tdb_key(p.seed) : TdbKey{0, 0};
    float z[CH][8], w[CH][8], b[CH][8];
    uint32_t kept[CH];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int at = 8 * min(l + 64 * c, chunks - 1);
#pragma unroll
        for (int i = 0; i < 8; ++i) w[c][i] = 1.f, b[c][i] = 0.f;
        if (p.weight) load_weight8<DT>(p.weight, p.wide, at, w[c]), load_weight8<DT>(p.bias, p.wide, at, b[c]);
    }
    Raw<DT, CH, RES, false> row;
    int64_t t = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6);
    const int64_t step = int64_t(gridDim.x) * 4;
    if (t < p.rows) row.load(p, t);
    for (; t < p.rows; t += step) {
        row.z_of(p, t, key, z, kept);
        if (t + step < p.rows) row.load(p, t + step);
        const float rstd = centre<CH>(z, p.hidden, p.eps);
#pragma unroll
        for (int c = 0; c < CH; ++c)
            if (l + 64 * c < chunks) {
                float y[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = z[c][i] * rstd * w[c][i] + b[c][i];
                store8<DT>(p.y, t * p.ys + 8 * (l + 64 * c), y);
            }
    }
}

constexpr int BWD_WAVES = 8;

// partial: [gridDim.x][2][hidden], the workgroups' sums of dy xhat and of dy.
template <int DT, int CH, bool RES>
__global__ __launch_bounds__(64 * BWD_WAVES) void norm_bwd_kernel(Norm p) {
    __shared__ float s_sum[BWD_WAVES][64 * 8];
    const int wave = threadIdx.x >> 6, l = threadIdx.x & 63, chunks = p.hidden / 8;
    const TdbKey key = p.threshold ? tdb_key(p.seed) : TdbKey{0, 0};
    float w[CH][8], dw[CH][8], db[CH][8];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
#pragma unroll
        for (int i = 0; i < 8; ++i) w[c][i] = 1.f, dw[c][i] = db[c][i] = 0.f;
        if (p.weight) load_weight8<DT>(p.weight, p.wide, 8 * min(l + 64 * c, chunks - 1), w[c]);
    }
    Raw<DT, CH, RES, true> row;
    int64_t t = int64_t(blockIdx.x) * BWD_WAVES + wave;
    const int64_t step = int64_t(gridDim.x) * BWD_WAVES;
    if (AHEAD<DT, CH> && t < p.rows) row.load(p, t);
    for (; t < p.rows; t += step) {
        float z[CH][8], g[CH][8];
        uint32_t kept[CH];
        if (!AHEAD<DT, CH>) row.load(p, t);
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i) g[c][i] = l + 64 * c < chunks ? float(row.dy[c][i]) : 0.f;
        row.z_of(p, t, key, z, kept);
        if (AHEAD<DT, CH> && t + step < p.rows) row.load(p, t + step);
        const float rstd = centre<CH>(z, p.hidden, p.eps);
        float sum = 0.f, dot = 0.f;
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                z[c][i] *= rstd;
                dw[c][i] += g[c][i] * z[c][i];
                db[c][i] += g[c][i];
                g[c][i] *= w[c][i];
                sum += g[c][i];
                dot += g[c][i] * z[c][i];
            }
        sum = wave_sum(sum) / float(p.hidden), dot = wave_sum(dot) / float(p.hidden);
#pragma unroll
        for (int c = 0; c < CH; ++c)
            if (l + 64 * c < chunks) {
#pragma unroll
                for (int i = 0; i < 8; ++i) g[c][i] = rstd * (g[c][i] - sum - z[c][i] * dot);
                const int at = 8 * (l + 64 * c);
                if constexpr (RES) {
                    if (p.dresidual) store8<DT>(p.dresidual, t * p.drs + at, g[c]);
                }
                if (p.dx) {
                    if (p.threshold) drop8(g[c], kept[c], p.factor);
                    store8<DT>(p.dx, t * p.dxs + at, g[c]);
                }
            }
    }
    if (!p.partial) return;
#pragma unroll
    for (int which = 0; which < 2; ++which)
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 8; ++i) s_sum[wave][i * 64 + l] = which ? db[c][i] : dw[c][i];
            __syncthreads();
            for (int at = threadIdx.x; at < 512; at += 64 * BWD_WAVES) {
                float sum = 0.f;
#pragma unroll
                for (int v = 0; v < BWD_WAVES; ++v) sum += s_sum[v][(at & 7) * 64 + (at >> 3)];
                if (512 * c + at < p.hidden) p.partial[(int64_t(blockIdx.x) * 2 + which) * p.hidden + 512 * c + at] = sum;
            }
        }
}

// Any width, any alignment: a workgroup per row.  LDS: the row, and a word for each wave.
template <int N>
__device__ __forceinline__ float block_sum(float x, float* scratch) {
    x = wave_sum(x);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = x;
    __syncthreads();
    float sum = 0.f;
#pragma unroll
    for (int v = 0; v < N; ++v) sum += scratch[v];
    return sum;
}

// z - mean of row t into s_z; returns 1 / standard deviation.  (A thread reads back only what it has written itself.)
template <int DT>
__device__ __forceinline__ float any_centre(const Norm& p, int64_t t, TdbKey key, float* s_z, float* scratch) {
    float sum = 0.f, sq = 0.f;
    for (int c = threadIdx.x; c < p.hidden; c += 256) {
        float z = load1<DT>(p.x, t * p.xs + c);
        if (p.threshold) z = kept1(uint64_t(t) * p.hidden + c, p.threshold, key) ? z * p.factor : 0.f;
        if (p.residual) z += load1<DT>(p.residual, t * p.rs + c);
        s_z[c] = z;
        sum += z;
    }
    const float mean = block_sum<4>(sum, scratch) / float(p.hidden);
    for (int c = threadIdx.x; c < p.hidden; c += 256) {
        const float z = s_z[c] - mean;
        s_z[c] = z;
        sq += z * z;
    }
    return rsqrtf(block_sum<4>(sq, scratch) / float(p.hidden) + p.eps);
}

template <int DT>
__global__ __launch_bounds__(256) void norm_fwd_any_kernel(Norm p) {
    extern __shared__ float s_z[];
    __shared__ float scratch[4];
    const TdbKey key = p.threshold ? tdb_key(p.seed) : TdbKey{0, 0};
    for (int64_t t = blockIdx.x; t < p.rows; t += gridDim.x) {
        const float rstd = any_centre<DT>(p, t, key, s_z, scratch);
        for (int c = threadIdx.x; c < p.hidden; c += 256) {
            float y = s_z[c] * rstd;
            if (p.weight) y = y * load_weight1<DT>(p.weight, p.wide, c) + load_weight1<DT>(p.bias, p.wide, c);
            store1<DT>(p.y, t * p.ys + c, y);
        }
    }
}

// The columns' sums are in the workgroup's own part of the workspace, each column with one thread.
template <int DT>
__global__ __launch_bounds__(256) void norm_bwd_any_kernel(Norm p) {
    extern __shared__ float s_z[];
    __shared__ float scratch[4];
    const TdbKey key = p.threshold ? tdb_key(p.seed) : TdbKey{0, 0};
    float* const mine = p.partial ? p.partial + int64_t(blockIdx.x) * 2 * p.hidden : nullptr;
    bool first = p.rows > blockIdx.x;
    if (mine && !first)
        for (int c = threadIdx.x; c < 2 * p.hidden; c += 256) mine[c] = 0.f;
    for (int64_t t = blockIdx.x; t < p.rows; t += gridDim.x) {
        const float rstd = any_centre<DT>(p, t, key, s_z, scratch);
        float sum = 0.f, dot = 0.f;
        for (int c = threadIdx.x; c < p.hidden; c += 256) {
            const float dy = load1<DT>(p.dy, t * p.dys + c), z = s_z[c] * rstd;
            const float g = p.weight ? dy * load_weight1<DT>(p.weight, p.wide, c) : dy;
            sum += g;
            dot += g * z;
            if (mine) {
                mine[c] = first ? dy * z : mine[c] + dy * z;
                mine[p.hidden + c] = first ? dy : mine[p.hidden + c] + dy;
            }
        }
        first = false;
        sum = block_sum<4>(sum, scratch) / float(p.hidden);
        dot = block_sum<4>(dot, scratch) / float(p.hidden);
        for (int c = threadIdx.x; c < p.hidden; c += 256) {
            const float dy = load1<DT>(p.dy, t * p.dys + c);
            const float g = p.weight ? dy * load_weight1<DT>(p.weight, p.wide, c) : dy;
            const float dz = rstd * (g - sum - s_z[c] * rstd * dot);
            if (p.dresidual) store1<DT>(p.dresidual, t * p.drs + c, dz);
            if (p.dx) store1<DT>(p.dx, t * p.dxs + c, !p.threshold ? dz : kept1(uint64_t(t) * p.hidden + c, p.threshold, key) ? dz * p.factor : 0.f);
        }
    }
}

// dweight, dbias: column sums of the workgroups' parts.  A workgroup has 16 columns; its 32 groups of 16 lanes share out the parts and ask for eight at a time.
template <int DT>
__global__ __launch_bounds__(512) void norm_sum_kernel(const float* partial, int parts, int hidden, void* dweight, void* dbias) {
    __shared__ float s_sum[32][17];
    const int group = threadIdx.x >> 4, l = threadIdx.x & 15, c = blockIdx.x * 16 + l;
    const float* at = partial + int64_t(blockIdx.y) * hidden + min(c, hidden - 1);
    float sum = 0.f;
    for (int g = group; g < parts; g += 32 * 8) {
        float x[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) x[u] = at[int64_t(min(g + 32 * u, parts - 1)) * 2 * hidden];
#pragma unroll
        for (int u = 0; u < 8; ++u) sum += g + 32 * u < parts ? x[u] : 0.f;
    }
    s_sum[group][l] = sum;
    __syncthreads();
    if (threadIdx.x < 16 && c < hidden) {
#pragma unroll
        for (int v = 1; v < 32; ++v) sum += s_sum[v][l];
        store1<DT>(blockIdx.y ? dbias : dweight, c, sum);
    }
}

// Workgroups of a launch, at most.  Waves with a row each walk on and ask for the next row ahead: forward 4 workgroups of 4 waves to a CU (16384 x 768 with residual: 17.7 us, with a
// wave for each row 19.5), backward one of 8 waves (31 us; two 37, four 48: each ends by adding up its waves).  Workgroups with a row each, backward: two to a CU
// (1013 x 771: 13 us, one 19).
constexpr int MAX_GRID = 1 << 20, FWD_GRID = 1024, BWD_PARTS = 256, BWD_ANY_PARTS = 512;
int parts_of(int64_t rows, int at_once) { return int(std::min<int64_t>(at_once > 1 ? BWD_PARTS : BWD_ANY_PARTS, std::max<int64_t>(1, (rows + at_once - 1) / at_once))); }

bool aligned(const void* p, int64_t stride, int size) { return !p || (reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride * size % 16 == 0); }

int check_norm(const tdb_norm_args* a, bool backward) {
    if (!a) return tdb_fail(TDB_ERR_NULL, "args is NULL");
    if (a->dtype != TDB_F32 && a->dtype != TDB_BF16 && a->dtype != TDB_F16) return tdb_fail(TDB_ERR_DTYPE, "unknown dtype %d", a->dtype);
    if (a->weight_dtype != a->dtype && a->weight_dtype != TDB_F32) return tdb_fail(TDB_ERR_DTYPE, "weight_dtype %d: need that of x, or float32", a->weight_dtype);
    if (a->rows < 0 || a->rows > (int64_t(1) << 40) || a->hidden < 1 || a->hidden > 32768)
        return tdb_fail(TDB_ERR_SHAPE, "%lld rows of %d: need 1 to 32768 columns", (long long)a->rows, a->hidden);
    if (a->threshold < 0 || a->threshold > 65536) return tdb_fail(TDB_ERR_SHAPE, "threshold %d: need 0 to 65536", a->threshold);
    if (!(a->eps >= 0.f)) return tdb_fail(TDB_ERR_SHAPE, "eps must not be negative");
    if (a->rows == 0 && !backward) return TDB_OK;
    if (a->threshold && !a->seed) return tdb_fail(TDB_ERR_NULL, "dropout needs a seed");
    if (!a->weight != !a->bias) return tdb_fail(TDB_ERR_NULL, "weight and bias: both or neither");
    if (!a->dweight != !a->dbias) return tdb_fail(TDB_ERR_NULL, "dweight and dbias: both or neither");
    if (backward && a->dweight && !a->workspace) return tdb_fail(TDB_ERR_NULL, "dweight needs a workspace");
    if (a->rows && (!a->x || (backward ? !a->dy : !a->y))) return tdb_fail(TDB_ERR_NULL, "x and y (or dy) must be non-NULL");
    const int64_t strides[] = {a->x_stride, a->residual_stride, a->dy_stride, a->y_stride, a->dx_stride, a->dresidual_stride};
    for (int64_t s : strides)
        if (s < 0) return tdb_fail(TDB_ERR_STRIDE, "negative row stride");
    const void* written[] = {a->y, a->dx, a->dresidual};
    const int64_t apart[] = {a->y_stride, a->dx_stride, a->dresidual_stride};
    for (int i = 0; i < 3; ++i)
        if (written[i] && a->rows > 1 && apart[i] < a->hidden) return tdb_fail(TDB_ERR_STRIDE, "rows of a result overlap");
    return TDB_OK;
}

template <int DT, int CH, bool RES>
void launch_rows(const Norm& n, int parts, hipStream_t s) {
    if (parts) norm_bwd_kernel<DT, CH, RES><<<parts, 64 * BWD_WAVES, 0, s>>>(n);
    else norm_fwd_kernel<DT, CH, RES><<<unsigned(std::min<int64_t>((n.rows + 3) / 4, FWD_GRID)), 256, 0, s>>>(n);
}

template <int DT>
hipError_t launch_norm(const tdb_norm_args& a, bool backward, hipStream_t s) {
    Norm n;
    n.x = a.x, n.residual = a.residual, n.weight = a.weight, n.bias = a.bias, n.dy = a.dy;
    n.y = a.y, n.dx = a.dx, n.dresidual = a.residual ? a.dresidual : nullptr;
    n.partial = a.dweight ? a.workspace : nullptr;
    n.seed = a.seed;
    n.xs = a.x_stride, n.rs = a.residual_stride, n.dys = a.dy_stride, n.ys = a.y_stride, n.dxs = a.dx_stride, n.drs = a.dresidual_stride;
    n.rows = a.rows, n.hidden = a.hidden, n.threshold = uint32_t(a.threshold), n.factor = tdb_kept_factor(a.threshold), n.eps = a.eps;
    n.wide = a.weight_dtype == TDB_F32;
    constexpr int size = DT == TDB_F32 ? 4 : 2;
    const bool rows = a.hidden % 8 == 0 && a.hidden <= 2048 && aligned(a.x, a.x_stride, size) && aligned(a.residual, a.residual_stride, size) &&
                      aligned(a.weight, 0, size) && aligned(a.bias, 0, size) &&
                      (backward ? aligned(a.dy, a.dy_stride, size) && aligned(a.dx, a.dx_stride, size) && aligned(n.dresidual, a.dresidual_stride, size)
                                : aligned(a.y, a.y_stride, size));
    const int parts = backward ? parts_of(a.rows, rows ? BWD_WAVES : 1) : 0;
    const size_t lds = size_t(a.hidden) * 4;
    if (rows) {
        const int ch = a.hidden <= 512 ? 1 : a.hidden <= 1024 ? 2 : 4;
        if (a.residual) {
            if (ch == 1) launch_rows<DT, 1, true>(n, parts, s);
            else if (ch == 2) launch_rows<DT, 2, true>(n, parts, s);
            else launch_rows<DT, 4, true>(n, parts, s);
        } else {
            if (ch == 1) launch_rows<DT, 1, false>(n, parts, s);
            else if (ch == 2) launch_rows<DT, 2, false>(n, parts, s);
            else launch_rows<DT, 4, false>(n, parts, s);
        }
    } else if (backward) {
        if (lds > 65536)
            if (const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(norm_bwd_any_kernel<DT>), hipFuncAttributeMaxDynamicSharedMemorySize, int(lds)); e != hipSuccess) return e;
        norm_bwd_any_kernel<DT><<<parts, 256, lds, s>>>(n);
    } else {
        if (lds > 65536)
            if (const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(norm_fwd_any_kernel<DT>), hipFuncAttributeMaxDynamicSharedMemorySize, int(lds)); e != hipSuccess) return e;
        norm_fwd_any_kernel<DT><<<unsigned(std::min<int64_t>(a.rows, MAX_GRID)), 256, lds, s>>>(n);
    }
    if (n.partial) {
        const dim3 grid((a.hidden + 15) / 16, 2);
        if (n.wide) norm_sum_kernel<TDB_F32><<<grid, 512, 0, s>>>(n.partial, parts, a.hidden, a.dweight, a.dbias);
        else norm_sum_kernel<DT><<<grid, 512, 0, s>>>(n.partial, parts, a.hidden, a.dweight, a.dbias);
    }
    return hipGetLastError();
}

int norm(const tdb_norm_args* a, bool backward, void* stream) {
    if (const int rc = check_norm(a, backward); rc != TDB_OK) return rc;
    if (a->rows == 0 && !(backward && a->dweight)) return TDB_OK;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const hipError_t e = a->dtype == TDB_F32 ? launch_norm<TDB_F32>(*a, backward, s) : a->dtype == TDB_BF16 ? launch_norm<TDB_BF16>(*a, backward, s) : launch_norm<TDB_F16>(*a, backward, s);
    if (e != hipSuccess) return tdb_fail(TDB_ERR_LAUNCH, "kernel launch failed: %s", hipGetErrorString(e));
    return TDB_OK;
}

template <int DT>
void launch_dropout(const void* x, void* y, int64_t n, int threshold, const int64_t* seed, hipStream_t s) {
    const unsigned grid = unsigned(std::min<int64_t>((n + 2047) / 2048, MAX_GRID));
    const float factor = tdb_kept_factor(threshold);
    if (aligned(x, 0, 1) && aligned(y, 0, 1)) dropout_kernel<DT, true><<<grid, 256, 0, s>>>(x, y, n, threshold, factor, seed);
    else dropout_kernel<DT, false><<<grid, 256, 0, s>>>(x, y, n, threshold, factor, seed);
}

}  // namespace

extern "C" {

int tdb_dropout(const void* x, void* y, int64_t n, int32_t dtype, int32_t threshold, const int64_t* seed, void* stream) {
    if (dtype != TDB_F32 && dtype != TDB_BF16 && dtype != TDB_F16) return tdb_fail(TDB_ERR_DTYPE, "unknown dtype %d", dtype);
    if (n < 0) return tdb_fail(TDB_ERR_SHAPE, "negative number of values");
    if (threshold < 0 || threshold > 65536) return tdb_fail(TDB_ERR_SHAPE, "threshold %d: need 0 to 65536", threshold);
    if (n == 0) return TDB_OK;
    if (!x || !y) return tdb_fail(TDB_ERR_NULL, "x and y must be non-NULL");
    if (threshold && !seed) return tdb_fail(TDB_ERR_NULL, "dropout needs a seed");
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (dtype == TDB_F32) launch_dropout<TDB_F32>(x, y, n, threshold, seed, s);
    else if (dtype == TDB_BF16) launch_dropout<TDB_BF16>(x, y, n, threshold, seed, s);
    else launch_dropout<TDB_F16>(x, y, n, threshold, seed, s);
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return tdb_fail(TDB_ERR_LAUNCH, "kernel launch failed: %s", hipGetErrorString(e));
    return TDB_OK;
}

int tdb_norm_fwd(const tdb_norm_args* args, void* stream) { return norm(args, false, stream); }
int tdb_norm_bwd(const tdb_norm_args* args, void* stream) { return norm(args, true, stream); }
int64_t tdb_norm_workspace(int64_t rows, int32_t hidden) { return rows < 0 || hidden < 1 ? 0 : int64_t(parts_of(rows, 1)) * 2 * hidden; }

}  // extern "C"
