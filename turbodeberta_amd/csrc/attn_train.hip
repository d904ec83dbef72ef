// Disentangled attention for training: forward with dropout on the probabilities and the rows' log sums, and the gradients of q, k, v and of both position tables.
//
//   S_ij = scale (q_i . k_j + q_i . K_r[d(i-j)] + k_j . Q_r[d(i-j)]),  P = softmax_j S,  P' = dropout(P),  O = P' V
//   dP = dropout'(dO V^T),  dS = P (dP - D),  D_i = dO_i . O_i,  dV = P'^T dO
//   dq_i = scale sum_j dS_ij (k_j + K_r[d(i-j)]),  dk_j = scale sum_i dS_ij (q_i + Q_r[d(i-j)])
//   dK_r[x] = scale sum_{d(i-j) = x} dS_ij q_i,  dQ_r[x] = scale sum_{d(i-j) = x} dS_ij k_j
//
// Backward in four launches for a number of heads at a time.  The costly part, scores, exponentials, random numbers, is done once: attn_bwd_kv_kernel owns keys, sums up
// their gradients and writes dS, rounded to the type, tile by tile to a workspace; attn_bwd_q_kernel owns queries and reads dS; attn_bwd_tables_kernel owns relative
// positions (a diagonal of tiles) and reads dS; tables_sum_kernel adds its parts up by table row.  No atomics: every sum has one owner and one order.
// Positions are handled as offsets i - j everywhere; d() is looked up where a table row is fetched, and where the sums of the offsets that share a row are added up.
#include <algorithm>
#include <cstring>
#include <mutex>

#include "attn_train.h"

namespace tdb_train {

// ---------------------------------------------------------------------------------------------------------------- forward

template <int DT, int NX>
constexpr int RING = 64 * NX + 64;

template <int DT, int NX>
struct FwdLds {
    using T = typename Elem<DT>::T;
    alignas(16) T k[TILE * ROW<DT>], v[TILE * ROW<DT>], pk[RING<DT, NX> * ROW<DT>], pq[RING<DT, NX> * ROW<DT>];
    alignas(16) float scratch[4][TERMS<NX>];
};

template <int DT, int NX>
__global__ __launch_bounds__(THREADS, 1) void attn_fwd_kernel(Args a) {
    using E = Elem<DT>;
    using T = typename E::T;
    using X8 = typename E::X8;
    constexpr int ring = RING<DT, NX>;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    FwdLds<DT, NX>& sm = *reinterpret_cast<FwdLds<DT, NX>*>(smem);
    if (a.cu && threadIdx.x < 64)
        tdb_fill_gaps(a.cu, a.B, a.L, a.total, static_cast<char*>(a.o.p), a.o.l * sizeof(T), a.o.h * sizeof(T), a.H, a.D * sizeof(T), blockIdx.x, gridDim.x);
    int h;
    Where w;
    if (!locate<64 * NX>(a, h, w)) return;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane_c(), g = lane_g();
    const int row = w.row0 + 16 * NX * wave;        // the wave's first query
    f32x4 o[NX][4];
#pragma unroll
    for (int x = 0; x < NX; ++x)
#pragma unroll
        for (int d = 0; d < 4; ++d) o[x][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (w.row0 >= w.len) {
#pragma unroll
        for (int x = 0; x < NX; ++x) store_rows<DT>(a.o, a, w, h, row + 16 * x, o[x], 0.f);
        return;
    }
    const T *const kp = rows_of<DT>(a.k, a, w, h), *const vp = rows_of<DT>(a.v, a, w, h);
    const T *const pk = static_cast<const T*>(a.pk.p) + h * a.pk.h, *const pq = static_cast<const T*>(a.pq.p) + h * a.pq.h;
    const bool has_pk = a.pk.p, has_pq = a.pq.p;
    const TdbKey key = a.threshold ? tdb_key(a.seed) : TdbKey{0, 0};
    X8 q[NX][2];
    load_own<DT, NX>(q, a.q, a, w, h, row);

    Stage<DT> k_next, v_next, pk_next, pq_next;
    int which[LOADS<DT>];
    auto tables = [&](Stage<DT>& s1, Stage<DT>& s2) {
        if (has_pk) s1.load(pk, a.pk.l, which, a.D);
        if (has_pq) s2.load(pq, a.pq.l, which, a.D);
    };
    if (has_pk || has_pq) {
#pragma unroll
        for (int n = 1; n <= NX; ++n) {
            table_rows<DT, 1>(a, 64 * n, w.row0, 0, which);
            tables(pk_next, pq_next);
            if (has_pk) pk_next.store(sm.pk + 64 * n * ROW<DT>);
            if (has_pq) pq_next.store(sm.pq + 64 * n * ROW<DT>);
        }
        table_rows<DT, 1>(a, 0, w.row0, 0, which);
    }
    auto fetch = [&](int y0) {
        k_next.load(kp, a.k.l, y0, w.len, a.D);
        v_next.load(vp, a.v.l, y0, w.len, a.D);
        if (has_pk || has_pq) {
            tables(pk_next, pq_next);
            table_rows<DT, 1>(a, 0, w.row0, y0 + TILE, which);
        }
    };
    fetch(0);

    const float c1 = a.scale * LOG2E;
    float most[NX], sum[NX];
#pragma unroll
    for (int x = 0; x < NX; ++x) most[x] = -__builtin_inff(), sum[x] = 0.f;
    int base = 0;
    for (int y0 = 0; y0 < w.len; y0 += TILE, base = base == 0 ? ring - 64 : base - 64) {
        __syncthreads();
        k_next.store(sm.k);
        v_next.store(sm.v);
        if (has_pk) pk_next.store(sm.pk + base * ROW<DT>);
        if (has_pq) pq_next.store(sm.pq + base * ROW<DT>);
        __syncthreads();
        if (y0 + TILE < w.len) fetch(y0 + TILE);

        f32x4 s[NX][4];
        scores<DT, NX, ring>(s, q, sm.k, sm.pk, sm.pq, has_pk, has_pq, base, NX * wave, sm.scratch[wave]);
        if (y0 + TILE > w.len) {
#pragma unroll
            for (int x = 0; x < NX; ++x)
#pragma unroll
                for (int m = 0; m < 4; ++m)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (y0 + 16 * m + 4 * g + e >= w.len) s[x][m][e] = -__builtin_inff();
        }
        X8 p[NX][2];
#pragma unroll
        for (int x = 0; x < NX; ++x) {
            float mx = s[x][0][0];
#pragma unroll
            for (int m = 0; m < 4; ++m)
#pragma unroll
                for (int e = 0; e < 4; ++e) mx = fmaxf(mx, s[x][m][e]);
            mx = fmaxf(most[x], column_max(mx) * c1);
            const float from = mx == -__builtin_inff() ? 0.f : mx;       // (a row of nothing but -inf)
            const float again = __builtin_amdgcn_exp2f(most[x] - from);
            most[x] = mx;
            sum[x] *= again;
#pragma unroll
            for (int d = 0; d < 4; ++d) o[x][d] *= again;
            float part = 0.f;
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                uint32_t kept = 0xff;
                if (a.threshold) kept = tdb_kept(tdb_philox(4 * ((y0 >> 5) + u) + g, row + 16 * x + c, w.b * a.H + h, 1, key), a.threshold);
#pragma unroll
                for (int n = 0; n < 8; ++n) {
                    const float v = __builtin_amdgcn_exp2f(fmaf(s[x][2 * u + (n >> 2)][n & 3], c1, -from));
                    part += v;
                    p[x][u][n] = T((kept >> n & 1) ? v : 0.f);
                }
            }
            sum[x] += part;
        }
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                const X8 v = pair_frag<DT>(sm.v, ROW<DT>, 32 * u, 16 * d);
#pragma unroll
                for (int x = 0; x < NX; ++x) o[x][d] = E::mma(v, p[x][u], o[x][d]);
            }
    }
#pragma unroll
    for (int x = 0; x < NX; ++x) {
        const float all = column_sum(sum[x]);
        store_rows<DT>(a.o, a, w, h, row + 16 * x, o[x], all > 0.f ? a.factor / all : all == 0.f ? 0.f : all);      // (NaN stays)
        const int r = row + 16 * x + c;
        if (g == 0 && r < w.len) a.lse[h * a.lines + w.line + r] = all == 0.f ? __builtin_inff() : most[x] + __builtin_amdgcn_logf(all);
    }
}

// --------------------------------------------------------------------------------------------------------------- backward

// D_i = dO_i . O_i for every row and head: 8 lanes each.  float16: the largest squares of the norms of rows of dO and V as well.
template <int DT>
__global__ __launch_bounds__(THREADS) void attn_delta_kernel(Args a, uint32_t* largest) {
    const int64_t unit = (int64_t(blockIdx.x) * THREADS + threadIdx.x) >> 3;
    const int64_t row = unit / a.H;
    const int h = int(unit - row * a.H), d = 8 * (threadIdx.x & 7);
    bool mine = row < a.lines;
    if (mine) {
        if (!a.cu) {
            const int b = int(row / a.L);
            mine = !a.seqlens || row - int64_t(b) * a.L < a.seqlens[b];
        } else if (DT == TDB_F16) {         // rows of no sequence may hold anything
            int lo = 0, hi = a.B;
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (a.cu[mid] <= row) lo = mid;
                else hi = mid;
            }
            int64_t first;
            const int len = valid_rows(a, lo, first);
            mine = row >= first && row < first + len;
        }
    }
    float dot = 0.f, sq = 0.f, sv = 0.f;
    if (mine && d < a.D) {
        using T = typename Elem<DT>::T;
        const int64_t b = a.cu ? 0 : row / a.L, r = a.cu ? row : row - b * a.L;
        const auto o = read8<DT>(static_cast<const T*>(a.o.p) + b * a.o.b + h * a.o.h + r * a.o.l + d);
        const auto x = read8<DT>(static_cast<const T*>(a.dout.p) + b * a.dout.b + h * a.dout.h + r * a.dout.l + d);
#pragma unroll
        for (int i = 0; i < 8; ++i) dot += float(o[i]) * float(x[i]), sq += float(x[i]) * float(x[i]);
        if constexpr (DT == TDB_F16) {
            const auto v = read8<DT>(static_cast<const T*>(a.v.p) + b * a.v.b + h * a.v.h + r * a.v.l + d);
#pragma unroll
            for (int i = 0; i < 8; ++i) sv += float(v[i]) * float(v[i]);
        }
    }
#pragma unroll
    for (int n = 1; n < 8; n <<= 1) dot += __shfl_xor(dot, n), sq += __shfl_xor(sq, n), sv += __shfl_xor(sv, n);
    if (mine && (threadIdx.x & 7) == 0) a.delta[h * a.lines + row] = dot;
    if constexpr (DT == TDB_F16) {
#pragma unroll
        for (int n = 8; n < 64; n <<= 1) sq = fmaxf(sq, __shfl_xor(sq, n)), sv = fmaxf(sv, __shfl_xor(sv, n));
        if ((threadIdx.x & 63) == 0) {      // (squares: their bits are in their order; the largest does not depend on theirs)
            atomicMax(largest, __builtin_bit_cast(uint32_t, sq));
            atomicMax(largest + 1, __builtin_bit_cast(uint32_t, sv));
        }
    }
}

__global__ void clear_kernel(uint32_t* x) { x[threadIdx.x] = 0; }

// A skewed tile: row x has the values of y at index 79 - y, zeros on both sides.  A row is 97 values apart from the next, so that
// index 16 + r - x of row x, r = x - y + 63, lies at 96 x + 16 + r: eight neighbouring r at a multiple of 8.
constexpr int SKEW = 97, SKEWED = 16 * SKEW + 32;

template <int DT, int NX>
struct KvLds {
    using T = typename Elem<DT>::T;
    alignas(16) T q[TILE * ROW<DT>], dout[TILE * ROW<DT>], pk[RING<DT, NX> * ROW<DT>], pq[RING<DT, NX> * ROW<DT>];
    alignas(16) T skewed[4][NX * SKEWED];
    alignas(16) float lse[TILE], delta[TILE];
    alignas(16) uint32_t kept[4][TILE];
    alignas(16) float scratch[4][TERMS<NX>];
};

template <int DT, int NX>
__global__ __launch_bounds__(THREADS, 1) void attn_bwd_kv_kernel(Args a) {
    using E = Elem<DT>;
    using T = typename E::T;
    using X8 = typename E::X8;
    constexpr int ring = RING<DT, NX>;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    KvLds<DT, NX>& sm = *reinterpret_cast<KvLds<DT, NX>*>(smem);
    int h;
    Where w;
    if (!locate<64 * NX>(a, h, w)) return;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, c = lane_c(), g = lane_g();
    const int row = w.row0 + 16 * NX * wave;        // the wave's first key
    f32x4 dk[NX][4], dv[NX][4];
#pragma unroll
    for (int x = 0; x < NX; ++x)
#pragma unroll
        for (int d = 0; d < 4; ++d) dk[x][d] = dv[x][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (w.row0 >= w.len) {
#pragma unroll
        for (int x = 0; x < NX; ++x) store_rows<DT>(a.dk, a, w, h, row + 16 * x, dk[x], 0.f), store_rows<DT>(a.dv, a, w, h, row + 16 * x, dv[x], 0.f);
        return;
    }
    const T *const qp = rows_of<DT>(a.q, a, w, h), *const dop = rows_of<DT>(a.dout, a, w, h);
    const T *const pk = static_cast<const T*>(a.pk.p) + h * a.pk.h, *const pq = static_cast<const T*>(a.pq.p) + h * a.pq.h;
    const bool has_pk = a.pk.p, has_pq = a.pq.p;
    const TdbKey key = a.threshold ? tdb_key(a.seed) : TdbKey{0, 0};
    const float power = score_power<DT>(a), rounded = w.len > 1 ? power : 0.f;      // (the softmax of one key is a constant)
    X8 k[NX][2], v[NX][2];
    load_own<DT, NX>(k, a.k, a, w, h, row);
    load_own<DT, NX>(v, a.v, a, w, h, row);
    T* const skewed = sm.skewed[wave];
    for (int n = lane; n < NX * SKEWED; n += 64) skewed[n] = T(0.f);

    Stage<DT> q_next, do_next, pk_next, pq_next;
    float line_next = 0.f;
    int which[LOADS<DT>];
    auto tables = [&](Stage<DT>& s1, Stage<DT>& s2) {
        if (has_pk) s1.load(pk, a.pk.l, which, a.D);
        if (has_pq) s2.load(pq, a.pq.l, which, a.D);
    };
    if (has_pk || has_pq) {
#pragma unroll
        for (int n = 1; n <= NX; ++n) {
            table_rows<DT, -1>(a, 64 * n, w.row0, 0, which);
            tables(pk_next, pq_next);
            if (has_pk) pk_next.store(sm.pk + 64 * n * ROW<DT>);
            if (has_pq) pq_next.store(sm.pq + 64 * n * ROW<DT>);
        }
        table_rows<DT, -1>(a, 0, w.row0, 0, which);
    }
    const float* const lines = (threadIdx.x < TILE ? a.lse : a.delta) + h * a.lines + w.line;
    auto fetch = [&](int y0) {
        q_next.load(qp, a.q.l, y0, w.len, a.D);
        do_next.load(dop, a.dout.l, y0, w.len, a.D);
        if (threadIdx.x < 2 * TILE) {
            const int r = y0 + (threadIdx.x & (TILE - 1));
            line_next = r < w.len ? lines[r] : threadIdx.x < TILE ? __builtin_inff() : 0.f;
        }
        if (has_pk || has_pq) {
            tables(pk_next, pq_next);
            table_rows<DT, -1>(a, 0, w.row0, y0 + TILE, which);
        }
    };
    fetch(0);

    const float c1 = a.scale * LOG2E, shift = DT == TDB_F16 ? float(a.p_shift) : 0.f, unshift = DT == TDB_F16 ? ldexpf(1.f, -a.p_shift) : 1.f;
    const bool edge = w.row0 + 64 * NX > w.len;
    const int tile_col = row / TILE, block = row / 16 % 4;
    T* const ds = static_cast<T*>(a.ds) + ((int64_t(h - a.head0) * a.row_tiles + w.row_tile) * a.tiles + tile_col) * TILE_VALUES + (block * 128 + lane) * 8;
    int base = 0;
    for (int y0 = 0; y0 < w.len; y0 += TILE, base = base == 0 ? ring - 64 : base - 64) {
        __syncthreads();
        q_next.store(sm.q);
        do_next.store(sm.dout);
        if (has_pk) pk_next.store(sm.pk + base * ROW<DT>);
        if (has_pq) pq_next.store(sm.pq + base * ROW<DT>);
        if (threadIdx.x < 2 * TILE) (threadIdx.x < TILE ? sm.lse : sm.delta)[threadIdx.x & (TILE - 1)] = line_next;
        __syncthreads();
        if (y0 + TILE < w.len) fetch(y0 + TILE);

        if (a.threshold) {      // a lane has a query: whether each of the wave's keys is kept
            uint32_t bits = 0;
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                const uint32_t kept = tdb_kept(tdb_philox(4 * (row >> 5) + n, y0 + lane, w.b * a.H + h, 1, key), a.threshold);
                if constexpr (NX == 2) bits |= (kept & 15) << (4 * n) | (kept >> 4) << (16 + 4 * n);
                else bits |= (kept >> (row & 16 ? 4 : 0) & 15) << (4 * n);
            }
            sm.kept[wave][lane] = bits;
            wave_fence();
        }
        f32x4 s[NX][4], dp[NX][4];
        scores<DT, NX, ring>(s, k, sm.q, sm.pq, sm.pk, has_pq, has_pk, base, NX * wave, sm.scratch[wave]);
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            const X8 d0 = row_frag<DT>(sm.dout, 16 * m, 0), d1 = row_frag<DT>(sm.dout, 16 * m, 32);
#pragma unroll
            for (int x = 0; x < NX; ++x) dp[x][m] = E::mma(d1, v[x][1], E::mma(d0, v[x][0], f32x4{0.f, 0.f, 0.f, 0.f}));
        }
        const bool some = edge || y0 + TILE > w.len;
        X8 p[NX][2], dsx[NX][2];
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            const f32x4 lse = *reinterpret_cast<const f32x4*>(sm.lse + 16 * m + 4 * g), delta = *reinterpret_cast<const f32x4*>(sm.delta + 16 * m + 4 * g);
            uint32_t kept[4] = {~0u, ~0u, ~0u, ~0u};
            if (a.threshold) {
                const u32x4 words = *reinterpret_cast<const u32x4*>(sm.kept[wave] + 16 * m + 4 * g);
#pragma unroll
                for (int e = 0; e < 4; ++e) kept[e] = words[e];
            }
#pragma unroll
            for (int x = 0; x < NX; ++x)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float pr = __builtin_amdgcn_exp2f(fmaf(s[x][m][e], c1, shift - lse[e]));
                    float grad = dp[x][m][e];
                    if (some && (y0 + 16 * m + 4 * g + e >= w.len || row + 16 * x + c >= w.len)) pr = 0.f, grad = 0.f;
                    const bool in = kept[e] >> (16 * x + c) & 1;
                    p[x][m >> 1][4 * (m & 1) + e] = T(in ? pr : 0.f);
                    dsx[x][m >> 1][4 * (m & 1) + e] = T(pr * unshift * ((in ? grad * a.factor : 0.f) - delta[e]) * rounded);
                }
        }
        if (tile_col * TILE < w.len) {
            T* const to = ds + int64_t(y0 / TILE) * a.tiles * TILE_VALUES;
#pragma unroll
            for (int x = 0; x < NX; ++x)
#pragma unroll
                for (int u = 0; u < 2; ++u) *reinterpret_cast<X8*>(to + (x * 128 + u * 64) * 8) = dsx[x][u];
        }
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                const X8 o = pair_frag<DT>(sm.dout, ROW<DT>, 32 * u, 16 * d), q = pair_frag<DT>(sm.q, ROW<DT>, 32 * u, 16 * d);
#pragma unroll
                for (int x = 0; x < NX; ++x) dv[x][d] = E::mma(o, p[x][u], dv[x][d]), dk[x][d] = E::mma(q, dsx[x][u], dk[x][d]);
            }
        if (has_pq) {
            wave_fence();
#pragma unroll
            for (int x = 0; x < NX; ++x)
#pragma unroll
                for (int n = 0; n < 16; ++n) skewed[x * SKEWED + c * SKEW + 79 - 16 * (n >> 2) - 4 * g - (n & 3)] = dsx[x][n >> 3][n & 7];
            wave_fence();
#pragma unroll
            for (int x = 0; x < NX; ++x)
#pragma unroll
                for (int n = 0; n < 3; ++n) {
                    const X8 b = read8<DT>(skewed + x * SKEWED + c * (SKEW - 1) + 16 + 32 * n + 8 * g);
                    const int at = wrapped<ring>(16 * (NX * wave + x) + 32 * n + 8 * g + base);
#pragma unroll
                    for (int d = 0; d < 4; ++d) dk[x][d] = E::mma(turned_frag<DT>(sm.pq, ROW<DT>, at, at + 4, 16 * d), b, dk[x][d]);
                }
            wave_fence();
        }
    }
#pragma unroll
    for (int x = 0; x < NX; ++x) {
        store_rows<DT>(a.dk, a, w, h, row + 16 * x, dk[x], a.scale / power);
        store_rows<DT>(a.dv, a, w, h, row + 16 * x, dv[x], a.factor * unshift);
    }
}

// A tile of dS as bwd_kv leaves it: 8 values each of 512 lanes: key 16 blk + c, queries 32 u + 4 g + e and 32 u + 16 + 4 g + e.
template <int DT>
struct Scores {
    using X8 = typename Elem<DT>::X8;
    X8 x[2];
    __device__ __forceinline__ void load(const typename Elem<DT>::T* tile) {
#pragma unroll
        for (int n = 0; n < 2; ++n) x[n] = read8<DT>(tile + (n * THREADS + threadIdx.x) * 8);
    }
    static __device__ __forceinline__ int key(int n) { return 16 * ((n * THREADS + threadIdx.x) >> 7) + lane_c(); }
    static __device__ __forceinline__ int query(int i) { return 32 * (threadIdx.x >> 6 & 1) + 16 * (i >> 2) + 4 * lane_g() + (i & 3); }
};

template <int DT>
struct QLds {
    using T = typename Elem<DT>::T;
    alignas(16) T k[TILE * ROW<DT>], pk[128 * ROW<DT>], ds[TILE * ROW<DT>], skewed[4][SKEWED];
};

// dq: a workgroup has 64 queries, a wave 16.
template <int DT>
__global__ __launch_bounds__(THREADS, DT == TDB_F32 ? 1 : 2) void attn_bwd_q_kernel(Args a) {
    using E = Elem<DT>;
    using T = typename E::T;
    using X8 = typename E::X8;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    QLds<DT>& sm = *reinterpret_cast<QLds<DT>*>(smem);
    if (a.cu && threadIdx.x < 64) {
        const Tensor* const all[] = {&a.dq, &a.dk, &a.dv};
        if (a.head0 == 0)
            for (const Tensor* t : all)
                tdb_fill_gaps(a.cu, a.B, a.L, a.total, static_cast<char*>(t->p), t->l * sizeof(T), t->h * sizeof(T), a.H, a.D * sizeof(T), blockIdx.x, gridDim.x);
    }
    int h;
    Where w;
    if (!locate<TILE>(a, h, w)) return;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane_c(), g = lane_g();
    f32x4 dq[4];
#pragma unroll
    for (int d = 0; d < 4; ++d) dq[d] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (w.row0 >= w.len) {
        store_rows<DT>(a.dq, a, w, h, w.row0 + 16 * wave, dq, 0.f);
        return;
    }
    const T* const kp = rows_of<DT>(a.k, a, w, h);
    const T* const pk = static_cast<const T*>(a.pk.p) + h * a.pk.h;
    const bool has_pk = a.pk.p;
    const T* const tiles = static_cast<const T*>(a.ds) + (int64_t(h - a.head0) * a.row_tiles + w.row_tile + w.row0 / TILE) * a.tiles * TILE_VALUES;
    for (int n = threadIdx.x; n < 4 * SKEWED; n += THREADS) sm.skewed[0][n] = T(0.f);
    Stage<DT> k_next, pk_next;
    Scores<DT> ds_next;
    int which[LOADS<DT>];
    if (has_pk) {
        table_rows<DT, 1>(a, 64, w.row0, 0, which);
        pk_next.load(pk, a.pk.l, which, a.D);
        pk_next.store(sm.pk + 64 * ROW<DT>);
        table_rows<DT, 1>(a, 0, w.row0, 0, which);
    }
    auto fetch = [&](int y0) {
        k_next.load(kp, a.k.l, y0, w.len, a.D);
        ds_next.load(tiles + int64_t(y0 / TILE) * TILE_VALUES);
        if (has_pk) {
            pk_next.load(pk, a.pk.l, which, a.D);
            table_rows<DT, 1>(a, 0, w.row0, y0 + TILE, which);
        }
    };
    fetch(0);
    int base = 0;
    for (int y0 = 0; y0 < w.len; y0 += TILE, base ^= 64) {
        __syncthreads();
        k_next.store(sm.k);
        if (has_pk) pk_next.store(sm.pk + base * ROW<DT>);
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            const int j = Scores<DT>::key(n), i = Scores<DT>::query(0);
            typedef __attribute__((ext_vector_type(4))) T T4;
            *reinterpret_cast<T4*>(sm.ds + j * ROW<DT> + i) = __builtin_shufflevector(ds_next.x[n], ds_next.x[n], 0, 1, 2, 3);
            *reinterpret_cast<T4*>(sm.ds + j * ROW<DT> + i + 16) = __builtin_shufflevector(ds_next.x[n], ds_next.x[n], 4, 5, 6, 7);
            if (has_pk) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int q = Scores<DT>::query(e);
                    sm.skewed[q >> 4][(q & 15) * SKEW + 79 - j] = ds_next.x[n][e];
                }
            }
        }
        __syncthreads();
        if (y0 + TILE < w.len) fetch(y0 + TILE);
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            const X8 b = line_frag<DT>(sm.ds, ROW<DT>, 32 * n, 16 * wave);
#pragma unroll
            for (int d = 0; d < 4; ++d) dq[d] = E::mma(line_frag<DT>(sm.k, ROW<DT>, 32 * n, 16 * d), b, dq[d]);
        }
        if (has_pk) {
#pragma unroll
            for (int n = 0; n < 3; ++n) {
                const X8 b = read8<DT>(sm.skewed[wave] + c * (SKEW - 1) + 16 + 32 * n + 8 * g);
                const int at = (16 * wave + 32 * n + 8 * g + base) & 127;
#pragma unroll
                for (int d = 0; d < 4; ++d) dq[d] = E::mma(turned_frag<DT>(sm.pk, ROW<DT>, at, at + 4, 16 * d), b, dq[d]);
            }
        }
    }
    store_rows<DT>(a.dq, a, w, h, w.row0 + 16 * wave, dq, a.scale / score_power<DT>(a));
}

// Tables: a workgroup has a diagonal of tiles (query tile - key tile = t) of every `splits`-th sequence, a wave 32 of its 128 offsets r = i - j + 63.
constexpr int BY_OFFSET = 128;
template <int DT>
constexpr int OFFSET_ROW = DT == TDB_F32 ? BY_OFFSET + 4 : BY_OFFSET + 8;

template <int DT>
struct TablesLds {
    using T = typename Elem<DT>::T;
    alignas(16) T q[TILE * ROW<DT>], k[TILE * ROW<DT>], by_query[TILE * OFFSET_ROW<DT>], by_key[TILE * OFFSET_ROW<DT>];
};

template <int DT>
__global__ __launch_bounds__(THREADS, DT == TDB_F32 ? 1 : 2) void attn_bwd_tables_kernel(Args a) {
    using E = Elem<DT>;
    using T = typename E::T;
    using X8 = typename E::X8;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    TablesLds<DT>& sm = *reinterpret_cast<TablesLds<DT>*>(smem);
    const int diagonals = 2 * a.tiles - 1, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane_c(), g = lane_g();
    const int split = blockIdx.x % a.splits, at = blockIdx.x / a.splits, t = at % diagonals - (a.tiles - 1), h = a.head0 + at / diagonals;
    const bool has_pk = a.pk.p, has_pq = a.pq.p;
    f32x4 dpk[2][4], dpq[2][4];
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int d = 0; d < 4; ++d) dpk[n][d] = dpq[n][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int n = threadIdx.x; n < TILE * OFFSET_ROW<DT>; n += THREADS) sm.by_query[n] = sm.by_key[n] = T(0.f);

    Stage<DT> q_next, k_next;
    Scores<DT> ds_next;
    Where w;
    int it = 0, end = 0;
    w.b = split - a.splits;
    auto advance = [&]() {              // to the next tile; false: none is left
        for (++it; it >= end;) {
            w.b += a.splits;
            if (w.b >= a.B) return false;
            w.len = valid_rows(a, w.b, w.first);
            w.row_tile = a.cu ? w.first / TILE + w.b : int64_t(w.b) * a.tiles;
            const int n = (w.len + TILE - 1) / TILE;
            it = max(0, t), end = min(n, n + t);
        }
        return true;
    };
    auto fetch = [&]() {
        q_next.load(rows_of<DT>(a.q, a, w, h), a.q.l, it * TILE, w.len, a.D);
        k_next.load(rows_of<DT>(a.k, a, w, h), a.k.l, (it - t) * TILE, w.len, a.D);
        ds_next.load(static_cast<const T*>(a.ds) + ((int64_t(h - a.head0) * a.row_tiles + w.row_tile + it) * a.tiles + it - t) * TILE_VALUES);
    };
    bool more = advance();
    if (more) fetch();
    while (more) {
        __syncthreads();
        q_next.store(sm.q);
        k_next.store(sm.k);
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            const int j = Scores<DT>::key(n);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int i = Scores<DT>::query(e);
                if (has_pk) sm.by_query[i * OFFSET_ROW<DT> + i - j + 63] = ds_next.x[n][e];
                if (has_pq) sm.by_key[j * OFFSET_ROW<DT> + i - j + 63] = ds_next.x[n][e];
            }
        }
        __syncthreads();
        more = advance();
        if (more) fetch();
        auto add = [&](f32x4 (&acc)[2][4], const T* rows, const T* by) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                X8 b[2];
#pragma unroll
                for (int n = 0; n < 2; ++n) b[n] = line_frag<DT>(by, OFFSET_ROW<DT>, 32 * u, 32 * wave + 16 * n);
#pragma unroll
                for (int d = 0; d < 4; ++d) {
                    const X8 x = line_frag<DT>(rows, ROW<DT>, 32 * u, 16 * d);
#pragma unroll
                    for (int n = 0; n < 2; ++n) acc[n][d] = E::mma(x, b[n], acc[n][d]);
                }
            }
        };
        if (has_pk) add(dpk, sm.q, sm.by_query);
        if (has_pq) add(dpq, sm.k, sm.by_key);
    }
    float* const part = a.partial + int64_t(blockIdx.x) * 2 * BY_OFFSET * 64;
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            const int to = (32 * wave + 16 * n + c) * 64 + 16 * d + 4 * g;
            if (has_pk) *reinterpret_cast<f32x4*>(part + to) = dpk[n][d];
            if (has_pq) *reinterpret_cast<f32x4*>(part + BY_OFFSET * 64 + to) = dpq[n][d];
        }
}

// The first offset in [-(L - 1), L) whose table row is `row` or a later one (the lookup table does not decrease): 64 places at a time.
__device__ __forceinline__ int first_offset(const Args& a, int row) {
    int lo = 1 - a.L, hi = a.L;             // the answer lies in [lo, hi]
    while (lo < hi) {
        const int step = (hi - lo + 63) / 64, at = lo + (threadIdx.x & 63) * step;
        const uint64_t less = __builtin_amdgcn_ballot_w64(at < hi && a.lut[at + a.lut_half] < row);
        const int n = __builtin_popcountll(less);
        if (n == 0) return lo;
        hi = min(hi, lo + n * step);
        lo = lo + (n - 1) * step + 1;
    }
    return lo;
}

// A table row's gradient: the offsets that share it, each in the one or two diagonals whose tiles have it, and their splits.  Four waves share the offsets.
template <int DT>
__global__ __launch_bounds__(THREADS) void tables_sum_kernel(Args a) {
    __shared__ float s_sum[4][64];
    const int which = blockIdx.z, h = a.head0 + blockIdx.y, row = blockIdx.x, wave = threadIdx.x >> 6, d = threadIdx.x & 63, diagonals = 2 * a.tiles - 1;
    if (!(which ? a.pq.p : a.pk.p)) return;
    const int lo = first_offset(a, row), hi = first_offset(a, row + 1);
    float sum = 0.f;
    for (int off = lo + ((wave - lo) & 3); off < hi; off += 4) {        // (a wave's offsets do not depend on the longest length)
        const int n0 = off + 63 + 64 * a.tiles, last = n0 / 64 - a.tiles, r = off + 63 - 64 * last;         // (rounded down: 64 last <= off + 63)
        for (int n = 0; n < 2; ++n) {
            const int t = last - n, at = r + 64 * n;        // offset `at` of diagonal t
            if (at > 126 || t <= -a.tiles || t >= a.tiles) continue;
            const float* p = a.partial + (((int64_t(blockIdx.y) * diagonals + t + a.tiles - 1) * a.splits * 2 + which) * BY_OFFSET + at) * 64 + d;
            for (int s = 0; s < a.splits; ++s) sum += p[int64_t(s) * 2 * BY_OFFSET * 64];
        }
    }
    s_sum[wave][d] = sum;
    __syncthreads();
    if (wave == 0 && d < a.D) {
        using T = typename Elem<DT>::T;
        for (int n = 1; n < 4; ++n) sum += s_sum[n][d];
        T* const to = static_cast<T*>(which ? a.dpq : a.dpk) + h * (which ? a.dpq_h : a.dpk_h) + int64_t(row) * a.D + d;
        *to = T(sum * a.scale / score_power<DT>(a));
    }
}

// ---------------------------------------------------------------------------------------------------------------- host

size_t elem(int dtype) { return dtype == TDB_F32 ? 4 : 2; }
int64_t up(int64_t x) { return (x + 255) / 256 * 256; }

constexpr int64_t MOST_SCORES = int64_t(512) << 20;      // bytes of dS at a time, unless one head has more

// What a backward call needs, and how many heads it takes at a time.
struct Plan {
    int tiles, row_tiles, splits, heads;
    int64_t lines, delta, partial, ds, bytes;       // offsets of the parts, and the sum
};
Plan plan_of(const tdb_train_attn_args& a) {
    Plan p;
    p.tiles = (a.max_seqlen + TILE - 1) / TILE;
    p.row_tiles = a.cu_seqlens ? a.total_tokens / TILE + a.batch : a.batch * p.tiles;
    p.lines = a.cu_seqlens ? a.total_tokens : int64_t(a.batch) * a.max_seqlen;
    const int64_t each = int64_t(p.row_tiles) * p.tiles * TILE_VALUES * int64_t(elem(a.dtype));
    p.heads = int(std::max<int64_t>(1, std::min<int64_t>(a.heads, MOST_SCORES / std::max<int64_t>(each, 1))));
    const int diagonals = 2 * p.tiles - 1;
    p.splits = int(std::max<int64_t>(1, std::min<int64_t>(a.batch, 1024 / (int64_t(p.heads) * diagonals))));
    p.delta = 256;                                  // in front: the two maxima
    p.partial = p.delta + up(p.lines * a.heads * 4);
    p.ds = p.partial + ((a.pos_key || a.pos_query) ? int64_t(p.heads) * diagonals * p.splits * 2 * BY_OFFSET * 64 * 4 : 0);
    p.bytes = p.ds + p.heads * each;
    return p;
}

bool aligned(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

int check(const tdb_train_attn_args* a, bool backward) {
    if (!a) return tdb_fail(TDB_ERR_NULL, "args is NULL");
    if (a->dtype != TDB_F32 && a->dtype != TDB_BF16 && a->dtype != TDB_F16) return tdb_fail(TDB_ERR_DTYPE, "unknown dtype %d", a->dtype);
    if (a->batch < 0 || a->heads < 1 || a->heads > 65535) return tdb_fail(TDB_ERR_SHAPE, "bad batch %d / heads %d", a->batch, a->heads);
    if (a->head_dim < 8 || a->head_dim > 64 || a->head_dim % 8) return tdb_fail(TDB_ERR_SHAPE, "head_dim %d: need a multiple of 8 in [8, 64]", a->head_dim);
    if (a->max_seqlen < 1 || a->max_seqlen > (1 << 20)) return tdb_fail(TDB_ERR_SHAPE, "sequence length %d out of range [1, %d]", a->max_seqlen, 1 << 20);
    if (a->total_tokens < 0) return tdb_fail(TDB_ERR_SHAPE, "negative total_tokens");
    if (a->threshold < 0 || a->threshold > 65536) return tdb_fail(TDB_ERR_SHAPE, "threshold %d: need 0 to 65536", a->threshold);
    if (!(a->sm_scale > 0.f) || !(a->sm_scale < 1e30f)) return tdb_fail(TDB_ERR_SHAPE, "sm_scale must be positive");
    const int64_t lines = a->cu_seqlens ? a->total_tokens : int64_t(a->batch) * a->max_seqlen;
    if (lines * a->heads > (1 << 28) || (lines / TILE + a->batch) * a->heads >= (1 << 24))       // (of the launches' sizes)
        return tdb_fail(TDB_ERR_SHAPE, "%lld rows of %d heads: need 2^28 at most", (long long)lines, a->heads);
    if (a->batch == 0 || lines == 0) return TDB_OK;
    if (!a->q || !a->k || !a->v || !a->o || !a->lse || (backward && (!a->dout || !a->dq || !a->dk || !a->dv || !a->workspace)))
        return tdb_fail(TDB_ERR_NULL, "a required pointer is NULL");
    if (a->threshold && !a->seed) return tdb_fail(TDB_ERR_NULL, "dropout needs a seed");
    const void* ptrs[] = {a->q, a->k, a->v, a->o, a->dout, a->dq, a->dk, a->dv, a->pos_key, a->pos_query, a->workspace};
    for (const void* p : ptrs)
        if (!aligned(p)) return tdb_fail(TDB_ERR_ALIGN, "tensors must be 16-byte aligned");
    for (int n = 0; n < 24; ++n) {
        const int64_t s = (&a->q_stride_b)[n];
        if (s < 0 || s * int64_t(elem(a->dtype)) % 16) return tdb_fail(TDB_ERR_STRIDE, "strides must be non-negative multiples of 16 bytes");
    }
    const int64_t rows[] = {a->o_stride_l, a->dq_stride_l, a->dk_stride_l, a->dv_stride_l};
    for (int n = 0; n < (backward ? 4 : 1); ++n)
        if (rows[n] < a->head_dim) return tdb_fail(TDB_ERR_STRIDE, "rows of a result overlap");
    const int64_t table[] = {a->pos_key_stride_h, a->pos_key_stride_r, a->pos_query_stride_h, a->pos_query_stride_r};
    for (int64_t s : table)
        if (s < 0 || s * int64_t(elem(a->dtype)) % 16) return tdb_fail(TDB_ERR_STRIDE, "strides of the tables must be non-negative multiples of 16 bytes");
    if (a->pos_key || a->pos_query) {
        if (a->span < 1 || a->span > (1 << 20)) return tdb_fail(TDB_ERR_POSITION, "span %d out of range", a->span);
        if (!a->delta_lut || a->lut_half < a->max_seqlen - 1) return tdb_fail(TDB_ERR_POSITION, "delta_lut is missing or shorter than the sequences");
        if (backward && ((a->pos_key && !a->dpos_key) || (a->pos_query && !a->dpos_query))) return tdb_fail(TDB_ERR_NULL, "a table's gradient has no place");
    }
    if (backward && a->workspace_bytes < plan_of(*a).bytes) return tdb_fail(TDB_ERR_SHAPE, "the workspace is too small");
    return TDB_OK;
}

Args args_of(const tdb_train_attn_args& a, const Plan& p) {
    Args k;
    memset(&k, 0, sizeof(k));
    k.q = {const_cast<void*>(a.q), a.q_stride_b, a.q_stride_h, a.q_stride_l};
    k.k = {const_cast<void*>(a.k), a.k_stride_b, a.k_stride_h, a.k_stride_l};
    k.v = {const_cast<void*>(a.v), a.v_stride_b, a.v_stride_h, a.v_stride_l};
    k.o = {a.o, a.o_stride_b, a.o_stride_h, a.o_stride_l};
    k.dout = {const_cast<void*>(a.dout), a.dout_stride_b, a.dout_stride_h, a.dout_stride_l};
    k.dq = {a.dq, a.dq_stride_b, a.dq_stride_h, a.dq_stride_l};
    k.dk = {a.dk, a.dk_stride_b, a.dk_stride_h, a.dk_stride_l};
    k.dv = {a.dv, a.dv_stride_b, a.dv_stride_h, a.dv_stride_l};
    k.pk = {const_cast<void*>(a.pos_key), 0, a.pos_key_stride_h, a.pos_key_stride_r};
    k.pq = {const_cast<void*>(a.pos_query), 0, a.pos_query_stride_h, a.pos_query_stride_r};
    k.lut = a.delta_lut, k.lut_half = a.lut_half, k.span = a.span;
    k.seqlens = a.seqlens_k, k.cu = a.cu_seqlens;
    k.B = a.batch, k.H = a.heads, k.D = a.head_dim, k.L = a.max_seqlen, k.total = a.total_tokens;
    k.head0 = 0, k.heads = a.heads;
    k.lines = p.lines, k.lse = a.lse;
    k.tiles = p.tiles, k.row_tiles = p.row_tiles, k.splits = p.splits;
    k.dpk = a.dpos_key, k.dpq = a.dpos_query, k.dpk_h = a.dpos_key_stride_h, k.dpq_h = a.dpos_query_stride_h;
    k.seed = a.seed, k.threshold = uint32_t(a.threshold), k.factor = tdb_kept_factor(a.threshold), k.scale = a.sm_scale;
    while (k.p_shift < 15 && (2 << k.p_shift) <= a.max_seqlen) ++k.p_shift;
    if (a.workspace) {
        char* const at = static_cast<char*>(a.workspace);
        k.largest = reinterpret_cast<const uint32_t*>(at);
        k.delta = reinterpret_cast<float*>(at + p.delta);
        k.partial = reinterpret_cast<float*>(at + p.partial);
        k.ds = at + p.ds;
    }
    return k;
}

int blocks_of(const Args& k, int rows) { return k.cu ? k.total / rows + k.B : k.B * ((k.L + rows - 1) / rows); }

// The kernels' LDS lies above what a launch has without asking, once per device and kernel.
template <auto kernel>
hipError_t launch(size_t lds, int64_t grid, hipStream_t s, const Args& k) {
    static std::mutex mutex;
    static bool raised[64];
    int device = 0;
    hipError_t e = hipGetDevice(&device);
    if (e != hipSuccess) return e;
    if (device < 0 || device >= 64) return hipErrorInvalidDevice;
    {
        const std::lock_guard<std::mutex> guard(mutex);
        if (!raised[device]) {
            e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, int(lds));
            if (e != hipSuccess) return e;
            raised[device] = true;
        }
    }
    kernel<<<unsigned(grid), THREADS, lds, s>>>(k);
    return hipGetLastError();
}

template <int DT, int NX>
hipError_t forward(Args k, hipStream_t s) {
    static_assert(sizeof(FwdLds<DT, NX>) <= 163840 && sizeof(KvLds<DT, NX>) <= 163840, "LDS of a CU");
    k.blocks = blocks_of(k, 64 * NX);
    return launch<attn_fwd_kernel<DT, NX>>(sizeof(FwdLds<DT, NX>), int64_t(k.blocks) * k.heads, s, k);
}

template <int DT, int NX>
hipError_t backward(Args k, int heads, hipStream_t s) {
    if (DT == TDB_F16) clear_kernel<<<1, 2, 0, s>>>(const_cast<uint32_t*>(k.largest));
    attn_delta_kernel<DT><<<unsigned((k.lines * k.H * 8 + THREADS - 1) / THREADS), THREADS, 0, s>>>(k, const_cast<uint32_t*>(k.largest));
    hipError_t e = hipGetLastError();
    for (k.head0 = 0; e == hipSuccess && k.head0 < k.H; k.head0 += heads) {
        k.heads = std::min(heads, k.H - k.head0);
        k.blocks = blocks_of(k, 64 * NX);
        e = launch<attn_bwd_kv_kernel<DT, NX>>(sizeof(KvLds<DT, NX>), int64_t(k.blocks) * k.heads, s, k);
        if (e != hipSuccess) break;
        k.blocks = blocks_of(k, TILE);
        e = launch<attn_bwd_q_kernel<DT>>(sizeof(QLds<DT>), int64_t(k.blocks) * k.heads, s, k);
        if (e != hipSuccess || (!k.pk.p && !k.pq.p)) continue;
        e = launch<attn_bwd_tables_kernel<DT>>(sizeof(TablesLds<DT>), int64_t(k.heads) * (2 * k.tiles - 1) * k.splits, s, k);
        if (e != hipSuccess) break;
        tables_sum_kernel<DT><<<dim3(2 * k.span, k.heads, 2), THREADS, 0, s>>>(k);
        e = hipGetLastError();
    }
    return e;
}

int run(const tdb_train_attn_args* a, bool back, void* stream) {
    if (const int rc = check(a, back); rc != TDB_OK) return rc;
    const Plan p = plan_of(*a);
    if (a->batch == 0 || p.lines == 0) return TDB_OK;
    const Args k = args_of(*a, p);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    hipError_t e;
    if (a->dtype == TDB_F32) e = back ? backward<TDB_F32, 1>(k, p.heads, s) : forward<TDB_F32, 1>(k, s);
    else if (a->dtype == TDB_BF16) e = back ? backward<TDB_BF16, 2>(k, p.heads, s) : forward<TDB_BF16, 2>(k, s);
    else e = back ? backward<TDB_F16, 2>(k, p.heads, s) : forward<TDB_F16, 2>(k, s);
    if (e != hipSuccess) return tdb_fail(TDB_ERR_LAUNCH, "kernel launch failed: %s", hipGetErrorString(e));
    return TDB_OK;
}

}  // namespace tdb_train

extern "C" {

int tdb_attn_train_fwd(const tdb_train_attn_args* args, void* stream) { return tdb_train::run(args, false, stream); }
int tdb_attn_train_bwd(const tdb_train_attn_args* args, void* stream) { return tdb_train::run(args, true, stream); }
int64_t tdb_attn_train_workspace(const tdb_train_attn_args* args) { return args ? tdb_train::plan_of(*args).bytes : 0; }

}  // extern "C"
