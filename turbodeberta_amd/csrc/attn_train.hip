// Disentangled attention for training: forward with dropout on the probabilities and the rows' log sums, and the gradients of q, k, v and of both position tables.
//
//   S_ij = scale (q_i . k_j + q_i . K_r[d(i-j)] + k_j . Q_r[d(i-j)]),  P = softmax_j S,  P' = dropout(P),  O = P' V
//   dP = dropout'(dO V^T),  dS = P (dP - D),  D_i = dO_i . O_i,  dV = P'^T dO
//   dq_i = scale sum_j dS_ij (k_j + K_r[d(i-j)]),  dk_j = scale sum_i dS_ij (q_i + Q_r[d(i-j)])
//   dK_r[x] = scale sum_{d(i-j) = x} dS_ij q_i,  dQ_r[x] = scale sum_{d(i-j) = x} dS_ij k_j
//
// Roundings to the type, each where a matrix instruction of it takes its operand: P' (in 16 bits as the sum of two values in the forward pass), dS, and what is stored.  A
// gradient's error is that of dS's rounding and its own, 1.4 times its own (bfloat16 2.3e-3 of its norm, 1.7e-3 for its own alone); sums are float32.  float16: P' and dS are
// scaled by powers of two to the top of its range, dS by one for each sequence and head, so that no sequence's gradients depend on the others'.
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

// Workgroups of four waves, 64 rows x; in 16 bits two of them fit a CU's LDS.
constexpr int THREADS = 256, WAVES = THREADS / 64;
template <int DT>
constexpr int PER_CU = DT == TDB_F32 ? 1 : 2;

template <int DT>
struct FwdLds {
    using T = typename Elem<DT>::T;
    alignas(16) T k[TILE * ROW<DT>], v[TILE * ROW<DT>], pk[RING * ROW<DT>], pq[RING * ROW<DT>];
    alignas(16) float scratch[WAVES][TERMS<DT>];
};

// Forward: one pass over the keys with the running maximum and sum of each row.  A wave has 16 queries, a lane one of them, so the transposed scores S^T come out of the products
// with a query's keys in a lane's registers, and the probabilities go into the next product as they are.  A step's keys, values and the 64 table rows that the ring
// of the tables lacks are on their way while the step before is worked on.
// Batch 32 x 512, lengths 384 .. 512, 12 heads, bfloat16: 170 us for 42 GFLOP.  Bound by the waits of one wave's chain (scores, their turn
// through LDS, maximum, exponentials, product), of which two waves of a SIMD hide a part: vector instructions take 49 % of the time, LDS 45, products 20.  Two workgroups to a CU
// are what LDS holds; one takes 240 us.
template <int DT, bool PK, bool PQ>
__global__ __launch_bounds__(THREADS, PER_CU<DT>) void attn_fwd_kernel(Args a) {
    using E = Elem<DT>;
    using T = typename E::T;
    using X8 = typename E::X8;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    FwdLds<DT>& sm = *reinterpret_cast<FwdLds<DT>*>(smem);
    if (a.cu && threadIdx.x < 64)
        tdb_fill_gaps(a.cu, a.B, a.L, a.total, static_cast<char*>(a.o.p), a.o.l * sizeof(T), a.o.h * sizeof(T), a.H, a.D * sizeof(T), blockIdx.x, gridDim.x);
    int h;
    Where w;
    if (!locate<TILE>(a, h, w)) return;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane_c(), g = lane_g();
    const int row = w.row0 + 16 * wave;             // the wave's first query
    f32x4 o[4];
#pragma unroll
    for (int d = 0; d < 4; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (w.row0 >= w.len) {
        store_rows<DT>(a.o, a, w, h, row, o, 0.f);
        return;
    }
    const TdbKey key = a.threshold ? tdb_key(a.seed) : TdbKey{0, 0};
    Source<DT, THREADS> keys(a.k, a, w, h), values(a.v, a, w, h);
    Stage<DT, THREADS> k_next, v_next;
    Tables<DT, 1, THREADS, PK, PQ> tables(a, h);
    X8 q[2];
    load_own<DT>(q, a.q, a, w, h, row);
    tables.fill(sm.pk, sm.pq, w.row0);
    bool far = false;
    auto fetch = [&](int y0) {
        keys.load(k_next);
        values.load(v_next);
        tables.load();
        tables.look(0, w.row0 - y0 - TILE);
        tables.look_at_ends(w.row0 - y0);
    };
    fetch(0);

    const float c1 = a.scale * LOG2E;
    float most = -__builtin_inff(), sum = 0.f;
    int base = 0;
    for (int y0 = 0; y0 < w.len; y0 += TILE, base ^= 64) {
        __syncthreads();
        k_next.store(sm.k);
        v_next.store(sm.v);
        tables.store(sm.pk, sm.pq, base);
        far = tables.far();
        __syncthreads();
        if (y0 + TILE < w.len) fetch(y0 + TILE);

        f32x4 s[4];
        scores<DT, PK, PQ>(s, q, sm.k, sm.pk, sm.pq, base, wave, sm.scratch[wave], far);
        X8 v[2][4];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int d = 0; d < 4; ++d) v[u][d] = pair_frag<DT>(sm.v, 32 * u, 16 * d);
        ahead<DT>();
        if (y0 + TILE > w.len) {
#pragma unroll
            for (int m = 0; m < 4; ++m)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (y0 + 16 * m + 4 * g + e >= w.len) s[m][e] = -__builtin_inff();
        }
        float mx = s[0][0];
#pragma unroll
        for (int m = 0; m < 4; ++m)
#pragma unroll
            for (int e = 0; e < 4; ++e) mx = fmaxf(mx, s[m][e]);
        mx = fmaxf(most, column_max(mx) * c1);
        const float from = mx == -__builtin_inff() ? 0.f : mx;       // (a row of nothing but -inf)
        const float again = __builtin_amdgcn_exp2f(most - from);
        most = mx;
        sum *= again;
#pragma unroll
        for (int d = 0; d < 4; ++d) o[d] *= again;
        X8 p[2], rest[2];                   // 16 bits: a probability is the sum of two values, as D (see store_rest) takes the result for exact
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            float z[8];
#pragma unroll
            for (int n = 0; n < 8; ++n) {
                z[n] = __builtin_amdgcn_exp2f(fmaf(s[2 * u + (n >> 2)][n & 3], c1, -from));
                sum += z[n];
            }
            if (a.threshold) {
                const uint4 r = tdb_philox(4 * ((y0 >> 5) + u) + g, row + c, w.b * a.H + h, 1, key);
#pragma unroll
                for (int n = 0; n < 8; ++n) z[n] = tdb_number(r, n) >= a.threshold ? z[n] : 0.f;
            }
#pragma unroll
            for (int n = 0; n < 8; ++n) {
                p[u][n] = T(z[n]);
                if constexpr (DT != TDB_F32) rest[u][n] = T(z[n] - float(p[u][n]));
            }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                o[d] = E::mma(v[u][d], p[u], o[d]);
                if constexpr (DT != TDB_F32) o[d] = E::mma(v[u][d], rest[u], o[d]);
            }
    }
    const float all = column_sum(sum);
    const float whole = all > 0.f ? a.factor / all : all == 0.f ? 0.f : all;                       // (NaN stays)
    store_rows<DT>(a.o, a, w, h, row, o, whole);
    if constexpr (DT != TDB_F32) store_rest<DT>(a.rest, a, w, h, row, o, whole);
    const float lse = all == 0.f ? __builtin_inff() : most + __builtin_amdgcn_logf(all);
    __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, lse), buffer(a.lse + h * a.lines + w.line, int64_t(w.len) * 4), g == 0 ? (row + c) * 4 : int(NOWHERE), 0, 0);
}

// --------------------------------------------------------------------------------------------------------------- backward

// Rounded to a tile, up and down: |x| < 64 tiles.
__device__ __forceinline__ int tile_up(const Args& a, int x) { return (x + TILE * a.tiles + TILE - 1) / TILE - a.tiles; }
__device__ __forceinline__ int tile_down(const Args& a, int x) { return (x + TILE * a.tiles) / TILE - a.tiles; }

// D_i = dO_i . O_i for every row and head, without dropout's factor: 8 lanes each, a workgroup for 64 rows.  float16: the largest squares of the norms of the sequence's rows of dO
// and V as well.  And the offsets at which the rows of the tables start, and the diagonals of tiles that lie in the last or in the first of these rows altogether.
template <int DT>
__global__ __launch_bounds__(THREADS) void attn_delta_kernel(Args a) {
    using T = typename Elem<DT>::T;
    const int d = 8 * (threadIdx.x & 7);
    if (a.lut) {
        const int id = blockIdx.x * THREADS + threadIdx.x, all = gridDim.x * THREADS;
        const int first = a.lut[1 - a.L + a.lut_half], last = a.lut[a.L - 1 + a.lut_half];
        for (int r = id; r <= 2 * a.span; r += all)
            if (r <= first || r > last) a.starts[r] = r <= first ? 1 - a.L : a.L;
        if (id == 0 && first == last) a.level[0] = 1 - a.tiles, a.level[1] = -a.tiles;
        for (int off = id + 2 - a.L; off < a.L; off += all) {
            const int before = a.lut[off - 1 + a.lut_half], row = a.lut[off + a.lut_half];
            for (int r = max(before, 0) + 1; r <= min(row, 2 * a.span); ++r) a.starts[r] = off;
            if (row != before && row == last) a.level[0] = tile_up(a, off + 63);
            if (row != before && before == first) a.level[1] = tile_down(a, off - 64);
        }
    }
    int h;
    Where w;
    if (!locate<TILE>(a, h, w)) return;
    const T *const o = rows_of<DT>(a.o, a, w, h), *const dout = rows_of<DT>(a.dout, a, w, h), *const v = rows_of<DT>(a.v, a, w, h);
    const T* const rest = static_cast<const T*>(a.rest) + (h * a.lines + w.line) * a.D;
    float most_do = 0.f, most_v = 0.f;
#pragma unroll
    for (int n = 0; n < 8 * TILE / THREADS; ++n) {
        const int row = w.row0 + n * (THREADS / 8) + (threadIdx.x >> 3);
        const bool mine = row < w.len;
        float dot = 0.f, sq = 0.f, sv = 0.f;
        if (mine && d < a.D) {
            const auto y = read8<DT>(o + row * a.o.l + d);
            const auto x = read8<DT>(dout + row * a.dout.l + d);
#pragma unroll
            for (int i = 0; i < 8; ++i) dot += float(y[i]) * float(x[i]), sq += float(x[i]) * float(x[i]);
            if (DT != TDB_F32 && a.rest) {
                const auto y = read8<DT>(rest + int64_t(row) * a.D + d);
#pragma unroll
                for (int i = 0; i < 8; ++i) dot += float(y[i]) * float(x[i]);
            }
            if constexpr (DT == TDB_F16) {
                const auto z = read8<DT>(v + row * a.v.l + d);
#pragma unroll
                for (int i = 0; i < 8; ++i) sv += float(z[i]) * float(z[i]);
            }
        }
#pragma unroll
        for (int n = 1; n < 8; n <<= 1) dot += __shfl_xor(dot, n), sq += __shfl_xor(sq, n), sv += __shfl_xor(sv, n);
        if (mine && (threadIdx.x & 7) == 0) a.delta[h * a.lines + w.line + row] = a.factor > 0.f ? dot / a.factor : 0.f;
        most_do = fmaxf(most_do, sq), most_v = fmaxf(most_v, sv);
    }
    if constexpr (DT == TDB_F16) {
        __shared__ float s_most[2][WAVES];
#pragma unroll
        for (int n = 8; n < 64; n <<= 1) most_do = fmaxf(most_do, __shfl_xor(most_do, n)), most_v = fmaxf(most_v, __shfl_xor(most_v, n));
        if ((threadIdx.x & 63) == 0) s_most[0][threadIdx.x >> 6] = most_do, s_most[1][threadIdx.x >> 6] = most_v;
        __syncthreads();
        if (threadIdx.x < 2) {              // (squares: their bits are in their order; the largest does not depend on it)
            const float* const m = s_most[threadIdx.x];
            atomicMax(a.largest + (int64_t(h) * a.B + w.b) * 2 + threadIdx.x, __builtin_bit_cast(uint32_t, fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]))));
        }
    }
}

__global__ __launch_bounds__(THREADS) void clear_kernel(uint32_t* x, int64_t n) {
    for (int64_t i = int64_t(blockIdx.x) * THREADS + threadIdx.x; i < n; i += int64_t(gridDim.x) * THREADS) x[i] = 0;
}

// Level tiles: those of the diagonals from hi on and up to lo, whose offsets all have the last or the first row of the tables.  They come in runs, and all that the
// positions add to a gradient there is a row of a table times a sum of scores' gradients: kept in float32, from before they are rounded, for the owner's row of keys or
// queries, and multiplied when its walk has ended.  4 x 4096, 256 buckets: of 127 diagonals 112.
struct Level {
    int hi, lo;
    __device__ __forceinline__ Level(const Args& a) {
        hi = 1 << 24, lo = -(1 << 24);
        if (a.lut) hi = a.level[0], lo = a.level[1];
    }
    __device__ __forceinline__ void ready() { hi = __builtin_amdgcn_readfirstlane(hi), lo = __builtin_amdgcn_readfirstlane(lo); }
    __device__ __forceinline__ bool has(int t) const { return t >= hi || t <= lo; }
    __device__ __forceinline__ bool any(int first, int last) const { return last >= hi || first <= lo; }        // of first .. last
};
constexpr int ROW_SUMS = WAVES * TILE;          // of a tile: each query's over 16 keys at a time

// Sums over the 16 lanes of a row of a result, for 16 values at once: lane c has that of value c.  (In each step a lane gives half of its values away and keeps the others;
// the partners are c ^ 8, c ^ 7, c ^ 2, c ^ 1.)
__device__ __forceinline__ float sums_of_16(float (&x)[16]) {
    const int c = lane_c();
    auto turn = [](float v, auto ctrl) { return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), decltype(ctrl)::value, 0xf, 0xf, true)); };
    auto step = [&](auto half, auto ctrl) {
        constexpr int N = decltype(half)::value;
        const bool upper = c & N;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const float keep = upper ? x[n + N] : x[n], give = upper ? x[n] : x[n + N];
            x[n] = keep + turn(give, ctrl);
        }
    };
    step(std::integral_constant<int, 8>{}, std::integral_constant<int, 0x128>{});      // rotated by 8
    step(std::integral_constant<int, 4>{}, std::integral_constant<int, 0x141>{});      // eight lanes mirrored
    step(std::integral_constant<int, 2>{}, std::integral_constant<int, 0x4e>{});       // quads: 2 3 0 1
    step(std::integral_constant<int, 1>{}, std::integral_constant<int, 0xb1>{});       // 1 0 3 2
    return x[0];
}

__device__ __forceinline__ float* level_part(const Args& a, int which, int h, int block) { return a.level_parts + (int64_t(which * a.heads + h - a.head0) * a.blocks + block) * 2 * 64; }
__device__ __forceinline__ void level_none(const Args& a, int which, int h, int block) {
    if (threadIdx.x < 128) level_part(a, which, h, block)[threadIdx.x] = 0.f;
}

// An owner's share of level tiles.  sum[0], sum[1]: over the tiles of hi and lo, for row c.  Adds the two table rows times the sums to acc, and leaves the workgroup's two
// sums of own rows times the sums, without the sequence's power, for the table's gradient.  lds: 2 KiB.
template <int DT>
__device__ __forceinline__ void level_end(const Args& a, const Tensor& table, int which, int h, int block, const typename Elem<DT>::X8 (&own)[2], const float (&sum)[2], f32x4 (&acc)[4],
                                          void* lds, int wave, float power) {
    using T = typename Elem<DT>::T;
    const int c = lane_c(), g = lane_g();
    float(*const part)[2][64] = static_cast<float(*)[2][64]>(lds);
    __syncthreads();                    // (what was in it has been read)
#pragma unroll
    for (int n = 0; n < 2; ++n) {
        const int row = a.lut[(n ? 1 - a.L : a.L - 1) + a.lut_half];
        const __amdgpu_buffer_rsrc_t from = buffer(static_cast<const T*>(table.p) + h * table.h + int64_t(row) * table.l, a.D * sizeof(T));
        typedef __attribute__((ext_vector_type(4))) T T4;
        typedef __attribute__((ext_vector_type(2))) uint32_t u32x2;
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            const int at = (16 * d + 4 * g) * int(sizeof(T));
            T4 t;
            if constexpr (DT == TDB_F32) t = __builtin_bit_cast(T4, __builtin_amdgcn_raw_buffer_load_b128(from, at, 0, 0));
            else t = __builtin_bit_cast(T4, __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(from, at, 0, 0)));
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[d][e] += float(t[e]) * sum[n];
        }
        float x[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] = float(own[e >> 3][e & 7]) * (sum[n] / power);
        const float total = sums_of_16(x);
        part[wave][n][32 * (c >> 3) + 8 * g + (c & 7)] = total;
    }
    __syncthreads();
    if (threadIdx.x < 128) {
        const int n = threadIdx.x >> 6, d = threadIdx.x & 63;
        level_part(a, which, h, block)[threadIdx.x] = (part[0][n][d] + part[1][n][d]) + (part[2][n][d] + part[3][n][d]);
    }
}

// A skewed tile: row x has the values of y at index 79 - y.  A row is 113 values apart from the next, so that index 16 + r - x of row x, r = x - y + 63, lies at
// 112 x + 16 + r: eight neighbouring r at a multiple of 8, and 16 x on distinct banks (14 chunks of 16 bytes).  r runs to 95: what lies outside of 0 <= y < 64 is not the
// row's.
template <int DT>
constexpr int SKEW = DT == TDB_F32 ? 97 : 113;
template <int DT>
constexpr int SKEWED = 16 * SKEW<DT>;
// A value of LDS by itself.  (Left alone, the compiler writes neighbours together, eight bytes at odd addresses: 60 clocks for each of four.)
template <class T>
__device__ __forceinline__ void put(T* to, T x) { *TDB_SHARED(volatile T, to) = x; }

// The eight r = 32 n + 8 g .. of the lane's row, zeros outside (ZEROS: these are in LDS already).
template <int DT, bool ZEROS>
__device__ __forceinline__ typename Elem<DT>::X8 skew_frag(const typename Elem<DT>::T* skewed, int n) {
    const int c = lane_c(), r = 32 * n + 8 * lane_g();
    typename Elem<DT>::X8 x = read8<DT>(skewed + c * (SKEW<DT> - 1) + 16 + r);
    if (ZEROS || n == 1) return x;      // (c <= r <= c + 63)
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (n == 0 ? r + i < c : r + i > c + 63) x[i] = typename Elem<DT>::T(0.f);
    return x;
}

template <int DT>
struct KvLds {
    using T = typename Elem<DT>::T;
    alignas(16) T q[TILE * ROW<DT>], dout[TILE * ROW<DT>], pk[RING * ROW<DT>], pq[RING * ROW<DT>];
    alignas(16) float lse[TILE], delta[TILE];
    alignas(16) uint32_t kept[2][WAVES / 2][TILE];       // a bit for each of 32 keys
    alignas(16) float scratch[WAVES][TERMS<DT>];             // of the scores; then the skewed gradients of scores
    static_assert(SKEWED<DT> * sizeof(T) <= TERMS<DT> * sizeof(float), "");
};

// dk, dv: a workgroup has 64 keys, a wave 16, a lane one of them; it walks over the queries.  Here scores, exponentials and random numbers are made again, once for the whole
// backward pass.  (Each owner making its own scores, without a workspace, needs them three times.)  Which keys are dropped is drawn a step ahead, a bit each.
// The batch above: 260 us, bound like the forward pass (vector instructions 48 % of the time, LDS 45, products 19).  Registers are full: 256, two waves to a SIMD; with both tables 128 scalar and 2 vector registers are spilled (float16 132 and 6).
template <int DT, bool PK, bool PQ>
__global__ __launch_bounds__(THREADS, PER_CU<DT>) void attn_bwd_kv_kernel(Args a) {
    using E = Elem<DT>;
    using T = typename E::T;
    using X8 = typename E::X8;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    KvLds<DT>& sm = *reinterpret_cast<KvLds<DT>*>(smem);
    int h;
    Where w;
    if (!locate<TILE>(a, h, w)) return;
    Level level(a);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, c = lane_c(), g = lane_g();
    const int row = w.row0 + 16 * wave;             // the wave's first key
    f32x4 dk[4], dv[4];
#pragma unroll
    for (int d = 0; d < 4; ++d) dk[d] = dv[d] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (w.row0 >= w.len) {
        store_rows<DT>(a.dk, a, w, h, row, dk, 0.f);
        store_rows<DT>(a.dv, a, w, h, row, dv, 0.f);
        return;
    }
    Source<DT, THREADS> queries(a.q, a, w, h), douts(a.dout, a, w, h);
    Stage<DT, THREADS> q_next, do_next;
    Tables<DT, -1, THREADS, PK, PQ> tables(a, h);
    X8 k[2], v[2];
    load_own<DT>(k, a.k, a, w, h, row);
    load_own<DT>(v, a.v, a, w, h, row);
    tables.fill(sm.pk, sm.pq, w.row0);
    const TdbKey key = a.threshold ? tdb_key(a.seed) : TdbKey{0, 0};
    const float power = score_power<DT>(a, h, w.b);
    const __amdgpu_buffer_rsrc_t lines = buffer((wave == 0 ? a.lse : a.delta) + h * a.lines + w.line, int64_t(w.len) * 4);      // of the waves that load them
    float line_next = 0.f;
    bool far = false;
    auto fetch = [&](int y0) {
        queries.load(q_next);
        douts.load(do_next);
        if (wave < 2) line_next = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(lines, lane * 4, y0 * 4, 0));
        tables.load();
        tables.look(0, w.row0 - y0 - TILE);
        tables.look_at_ends(w.row0 - y0);
    };
    fetch(0);
    // Which of 32 keys are kept for the queries of a step: the two waves that have the keys share the work, a step ahead.  A lane has a query and two of the four counters
    // whose numbers are those of the keys: 4 neighbouring ones of each half.
    auto draw = [&](int y0, int to) {
        const int query = 32 * (wave & 1) + (lane & 31), n = lane >> 5;
        uint32_t low = 0, high = 0;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t kept = tdb_kept(tdb_philox(4 * (row >> 5) + 2 * n + i, y0 + query, w.b * a.H + h, 1, key), a.threshold);
            low |= (kept & 15) << (4 * i), high |= (kept >> 4) << (4 * i);
        }
        uint8_t* const bytes = reinterpret_cast<uint8_t*>(&sm.kept[to][wave >> 1][query]);
        bytes[n] = uint8_t(low), bytes[2 + n] = uint8_t(high);
    };
    if (a.threshold) draw(0, 0);

    const float c1 = a.scale * LOG2E, shift = DT == TDB_F16 ? float(a.p_shift) : 0.f, unshift = DT == TDB_F16 ? ldexpf(1.f, -a.p_shift) : 1.f;
    const float down = unshift * power;         // (1 but in float16)
    const bool edge = w.row0 + TILE > w.len;
    const int tile_col = row / TILE, bit = (row & 16) + c;
    T* ds = static_cast<T*>(a.ds) + ((int64_t(h - a.head0) * a.row_tiles + w.row_tile) * a.tiles + tile_col) * TILE_VALUES + row / 16 % 4 * 1024;
    T* const skewed = reinterpret_cast<T*>(sm.scratch[wave]);
    int base = 0, odd = 0;
    float by_key[2] = {0.f, 0.f};
    float* row_sums = a.row_sums + ((int64_t(h - a.head0) * a.row_tiles + w.row_tile) * a.tiles + tile_col) * ROW_SUMS;
    level.ready();
    for (int y0 = 0; y0 < w.len; y0 += TILE, base ^= 64, ds += int64_t(a.tiles) * TILE_VALUES, row_sums += int64_t(a.tiles) * ROW_SUMS, odd ^= 1) {
        const bool is_level = (PK || PQ) && level.has((y0 - w.row0) / TILE);
        __syncthreads();
        q_next.store(sm.q);
        do_next.store(sm.dout);
        tables.store(sm.pk, sm.pq, base);
        if (wave < 2) (wave == 0 ? sm.lse : sm.delta)[lane] = line_next;
        far = tables.far();
        __syncthreads();
        if (y0 + TILE < w.len) {
            fetch(y0 + TILE);
            if (a.threshold) draw(y0 + TILE, odd ^ 1);
        }
        f32x4 s[4], dp[4];
        scores<DT, PQ, PK>(s, k, sm.q, sm.pq, sm.pk, base, wave, sm.scratch[wave], far);
        {
            X8 y[4][2];
#pragma unroll
            for (int m = 0; m < 4; ++m)
#pragma unroll
                for (int n = 0; n < 2; ++n) y[m][n] = row_frag<DT>(sm.dout, 16 * m, 32 * n);
            ahead<DT>();
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int m = 0; m < 4; ++m) dp[m] = E::mma(y[m][n], v[n], n == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : dp[m]);
        }
        X8 turned[2][4];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int d = 0; d < 4; ++d) turned[u][d] = pair_frag<DT>(sm.dout, 32 * u, 16 * d);
        ahead<DT>();
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            const f32x4 lse = *reinterpret_cast<const f32x4*>(sm.lse + 16 * m + 4 * g);
#pragma unroll
            for (int e = 0; e < 4; ++e) s[m][e] = __builtin_amdgcn_exp2f(fmaf(s[m][e], c1, shift - lse[e]));
        }
        if (edge || y0 + TILE > w.len) {        // rows and keys behind the sequence, whatever they have given
#pragma unroll
            for (int m = 0; m < 4; ++m)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (y0 + 16 * m + 4 * g + e >= w.len || row + c >= w.len) s[m][e] = 0.f, dp[m][e] = 0.f;
        }
        X8 p[2], dsx[2];
        float grads[16];
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            const f32x4 delta = *reinterpret_cast<const f32x4*>(sm.delta + 16 * m + 4 * g);
            f32x4 pr = s[m], grad = dp[m];
            if (a.threshold) {
                const u32x4 words = *reinterpret_cast<const u32x4*>(sm.kept[odd][wave >> 1] + 16 * m + 4 * g);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const bool in = words[e] >> bit & 1;
                    pr[e] = in ? pr[e] : 0.f;
                    grad[e] = in ? grad[e] : 0.f;
                }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                p[m >> 1][4 * (m & 1) + e] = T(pr[e]);
                grads[4 * m + e] = DT == TDB_F16 ? s[m][e] * ((grad[e] - delta[e]) * down) : s[m][e] * (grad[e] - delta[e]);
                dsx[m >> 1][4 * (m & 1) + e] = T(grads[4 * m + e]);
            }
        }
        if (w.len == 1) {               // the softmax of one key is a constant
#pragma unroll
            for (int n = 0; n < 16; ++n) grads[n] = 0.f, dsx[n >> 3][n & 7] = T(0.f);
        }
        if (is_level) {
            if constexpr (PQ) {
                float all = 0.f;
#pragma unroll
                for (int n = 0; n < 16; ++n) all += grads[n];
                by_key[y0 - w.row0 >= TILE * level.hi ? 0 : 1] += all;
            }
            if constexpr (PK) {
                const float of_query = sums_of_16(grads);
                __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, of_query), buffer(row_sums, ROW_SUMS * 4), (16 * (c >> 2) + 4 * g + (c & 3)) * 16, wave * 4, 0);
            }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const __amdgpu_buffer_rsrc_t to = buffer(ds, 1024 * sizeof(T));
            if constexpr (DT == TDB_F32) {
                const f32x8 x = __builtin_bit_cast(f32x8, dsx[u]);
                __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, __builtin_shufflevector(x, x, 0, 1, 2, 3)), to, lane * 32, u * 2048, 0);
                __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, __builtin_shufflevector(x, x, 4, 5, 6, 7)), to, lane * 32 + 16, u * 2048, 0);
            } else {
                __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, dsx[u]), to, lane * 16, u * 1024, 0);
            }
        }
        if (PQ && !far && !is_level) {
#pragma unroll
            for (int n = 0; n < 16; ++n) put(skewed + c * SKEW<DT> + 79 - 16 * (n >> 2) - 4 * g - (n & 3), T(dsx[n >> 3][n & 7]));
        }
        X8 q[2][4];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int d = 0; d < 4; ++d) q[u][d] = pair_frag<DT>(sm.q, 32 * u, 16 * d);
        ahead<DT>();
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int d = 0; d < 4; ++d) dv[d] = E::mma(turned[u][d], p[u], dv[d]);
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int d = 0; d < 4; ++d) dk[d] = E::mma(q[u][d], dsx[u], dk[d]);
        if (PQ && !is_level) {
            if (far) {
#pragma unroll
                for (int d = 0; d < 4; ++d) {
                    const X8 t = level_frag<DT>(sm.pq, wrapped(63 + base), 16 * d);
#pragma unroll
                    for (int u = 0; u < 2; ++u) dk[d] = E::mma(t, dsx[u], dk[d]);
                }
            } else {
                wave_fence();
                X8 t[3][4], b[3];
#pragma unroll
                for (int n = 0; n < 3; ++n) {
                    b[n] = skew_frag<DT, false>(skewed, n);
#pragma unroll
                    for (int d = 0; d < 4; ++d) t[n][d] = ring_frag<DT>(sm.pq, 16 * wave + 32 * n + base, 16 * d);
                }
                ahead<DT>();
#pragma unroll
                for (int n = 0; n < 3; ++n)
#pragma unroll
                    for (int d = 0; d < 4; ++d) dk[d] = E::mma(t[n][d], b[n], dk[d]);
                wave_fence();
            }
        }
    }
    if (PQ && level.any(-w.row0 / TILE, (w.len - 1) / TILE - w.row0 / TILE)) {
        by_key[0] = column_sum(by_key[0]), by_key[1] = column_sum(by_key[1]);
        level_end<DT>(a, a.pq, 1, h, w.block, k, by_key, dk, sm.pq, wave, power);
    } else if (PQ) {
        level_none(a, 1, h, w.block);
    }
    store_rows<DT>(a.dk, a, w, h, row, dk, a.scale * a.factor / power);
    store_rows<DT>(a.dv, a, w, h, row, dv, a.factor * unshift);
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
    // as rows of keys, columns of queries
    __device__ __forceinline__ void store(typename Elem<DT>::T* rows) const {
        typedef __attribute__((ext_vector_type(4))) typename Elem<DT>::T T4;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            *reinterpret_cast<T4*>(rows + place<DT>(key(n), query(0))) = __builtin_shufflevector(x[n], x[n], 0, 1, 2, 3);
            *reinterpret_cast<T4*>(rows + place<DT>(key(n), query(4))) = __builtin_shufflevector(x[n], x[n], 4, 5, 6, 7);
        }
    }
    static __device__ __forceinline__ int key(int n) { return 16 * ((n * THREADS + threadIdx.x) >> 7) + lane_c(); }
    static __device__ __forceinline__ int query(int i) { return 32 * (threadIdx.x >> 6 & 1) + 16 * (i >> 2) + 4 * lane_g() + (i & 3); }
};

template <int DT>
struct QLds {
    using T = typename Elem<DT>::T;
    alignas(16) T k[TILE * ROW<DT>], pk[RING * ROW<DT>], ds[TILE * ROW<DT>], skewed[4][SKEWED<DT>];
};

// dq: a workgroup has 64 queries, a wave 16; the next step's rows and tile of dS are on their way.  The batch above: 88 us, of which the tiles, 154 MB, need 31; 4 x 4096: 490
// for 1.6 GB, 320 at the rate of a large copy.  (Two steps ahead took 104 and 540: registers for two waves to a SIMD, not three.)
template <int DT, bool PK>
__global__ __launch_bounds__(THREADS, PER_CU<DT>) void attn_bwd_q_kernel(Args a) {
    using E = Elem<DT>;
    using T = typename E::T;
    using X8 = typename E::X8;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    QLds<DT>& sm = *reinterpret_cast<QLds<DT>*>(smem);
    if (a.cu && threadIdx.x < 64 && a.head0 == 0) {
        const Tensor* const all[] = {&a.dq, &a.dk, &a.dv};
        for (const Tensor* t : all)
            tdb_fill_gaps(a.cu, a.B, a.L, a.total, static_cast<char*>(t->p), t->l * sizeof(T), t->h * sizeof(T), a.H, a.D * sizeof(T), blockIdx.x, gridDim.x);
    }
    int h;
    Where w;
    if (!locate<TILE>(a, h, w)) return;
    Level level(a);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), row = w.row0 + 16 * wave;
    f32x4 dq[4];
#pragma unroll
    for (int d = 0; d < 4; ++d) dq[d] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (w.row0 >= w.len) {
        store_rows<DT>(a.dq, a, w, h, row, dq, 0.f);
        return;
    }
    const T* tile = static_cast<const T*>(a.ds) + (int64_t(h - a.head0) * a.row_tiles + w.row_tile + w.row0 / TILE) * a.tiles * TILE_VALUES;
    Source<DT, THREADS> keys(a.k, a, w, h);
    struct Next {                       // a step's rows on their way
        Stage<DT, THREADS> k, pk;
        Scores<DT> ds;
        int ends[2];
        u32x4 sums;
    } next;
    Tables<DT, 1, THREADS, PK, false> tables(a, h);
    tables.fill(sm.pk, nullptr, w.row0);
    if constexpr (PK) {                 // what no step writes: an index below 16 or above 79 of a row
        for (int n = threadIdx.x; n < 4 * SKEWED<DT>; n += THREADS) (&sm.skewed[0][0])[n] = T(0.f);
    }
    int y_next = 0;
    const float* row_sums = a.row_sums + (int64_t(h - a.head0) * a.row_tiles + w.row_tile + w.row0 / TILE) * a.tiles * ROW_SUMS;
    float by_query[2] = {0.f, 0.f};
    level.ready();
    auto fetch = [&]() {
        if constexpr (PK) {             // (zeros for other tiles)
            const __amdgpu_buffer_rsrc_t from = buffer(row_sums, level.has((w.row0 - y_next) / TILE) ? ROW_SUMS * 4 : 0);
            next.sums = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(from, (16 * wave + lane_c()) * 16, 0, 0));
            row_sums += ROW_SUMS;
        }
        keys.load(next.k);
        next.ds.load(tile);
        tile += TILE_VALUES;
        tables.load();
        next.pk = tables.k;
        tables.look_at_ends(w.row0 - y_next);
        next.ends[0] = tables.ends[0], next.ends[1] = tables.ends[1];
        y_next += TILE;
        tables.look(0, w.row0 - y_next);
    };
    int base = 0;
    auto step = [&](int y0) {
        const int t = (w.row0 - y0) / TILE;
        const bool is_level = PK && level.has(t);
        __syncthreads();
        next.k.store(sm.k);
        if constexpr (PK) {
            const f32x4 x = __builtin_bit_cast(f32x4, next.sums);
            const float all = (x[0] + x[1]) + (x[2] + x[3]);
            by_query[0] += t >= level.hi ? all : 0.f, by_query[1] += t >= level.hi ? 0.f : all;
        }
        if constexpr (PK) next.pk.store(sm.pk + base * ROW<DT>);
        next.ds.store(sm.ds);
        const bool far = PK && __builtin_amdgcn_readfirstlane(next.ends[0]) == __builtin_amdgcn_readfirstlane(next.ends[1]);
        if (PK && !far && !is_level) {
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                const int q = Scores<DT>::query(0);
                T* const to = sm.skewed[q >> 4] + (q & 15) * SKEW<DT> + 79 - Scores<DT>::key(n);
#pragma unroll
                for (int e = 0; e < 8; ++e) to[(e >> 2) * SKEWED<DT> + (e & 3) * SKEW<DT>] = next.ds.x[n][e];
            }
        }
        __syncthreads();
        if (y_next < w.len) fetch();
        X8 b[2], k[2][4];
        auto own = [&]() {
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                b[n] = line_frag<DT>(sm.ds, 32 * n, 16 * wave);
#pragma unroll
                for (int d = 0; d < 4; ++d) k[n][d] = line_frag<DT>(sm.k, 32 * n, 16 * d);
            }
        };
        if (PK && !far && !is_level) {
            X8 by[3], t[3][4];
#pragma unroll
            for (int n = 0; n < 3; ++n) {
                by[n] = skew_frag<DT, true>(sm.skewed[wave], n);
#pragma unroll
                for (int d = 0; d < 4; ++d) t[n][d] = ring_frag<DT>(sm.pk, 16 * wave + 32 * n + base, 16 * d);
            }
            ahead<DT>();
            own();
#pragma unroll
            for (int n = 0; n < 3; ++n)
#pragma unroll
                for (int d = 0; d < 4; ++d) dq[d] = E::mma(t[n][d], by[n], dq[d]);
        } else {
            own();
        }
        if (PK && far && !is_level) {
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                const X8 t = level_frag<DT>(sm.pk, wrapped(63 + base), 16 * d);
#pragma unroll
                for (int n = 0; n < 2; ++n) dq[d] = E::mma(t, b[n], dq[d]);
            }
        }
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int d = 0; d < 4; ++d) dq[d] = E::mma(k[n][d], b[n], dq[d]);
        base ^= 64;
    };
    fetch();
    for (int y0 = 0; y0 < w.len; y0 += TILE) step(y0);
    const float power = score_power<DT>(a, h, w.b);
    if (PK && level.any(w.row0 / TILE - (w.len - 1) / TILE, w.row0 / TILE)) {
        X8 q[2];
        load_own<DT>(q, a.q, a, w, h, row);
        level_end<DT>(a, a.pk, 0, h, w.block, q, by_query, dq, sm.pk, wave, power);
    } else if (PK) {
        level_none(a, 0, h, w.block);
    }
    store_rows<DT>(a.dq, a, w, h, row, dq, a.scale * a.factor / power);
}

// Parts that the sequences of a diagonal are dealt to, as many as it has tiles, next to the longest one; each is 2^seg_bits, to which a sequence's tiles are dealt in turn.
__device__ __forceinline__ int splits_of(const Args& a, int t) { return min(max(1, (((a.tiles - abs(t)) << a.split_bits) * a.per_tile) >> 16), 1 << a.split_bits); }

// Tables: a workgroup has a diagonal of tiles (query tile - key tile = t) of every `splits`-th sequence.  Its waves share the two tables and the 128 offsets r = i - j + 63 of
// a tile: in blocks of 16, dealt in turn, so that each has as many of those that 32 queries (or keys) reach.  Where all offsets of a diagonal have one table row ("far")
// their sum is all that is wanted: Q^T dS and K^T dS^T, whose columns are added up at the end.
constexpr int BY_OFFSET = 128;
template <int DT>
constexpr int OFFSET_ROW = DT == TDB_F32 ? BY_OFFSET + 4 : BY_OFFSET + 8;
template <int DT>
__device__ __forceinline__ typename Elem<DT>::X8 offset_frag(const typename Elem<DT>::T* rows, int k0, int col) {
    return turned_frag<DT>(rows, k0 + 8 * lane_g(), k0 + 8 * lane_g() + 4, col, [](int r, int c) { return r * OFFSET_ROW<DT> + c; });
}

template <int DT>
struct TablesLds {
    using T = typename Elem<DT>::T;
    alignas(16) T q[TILE * ROW<DT>], k[TILE * ROW<DT>], by_query[TILE * OFFSET_ROW<DT>], by_key[TILE * OFFSET_ROW<DT>];
};

// Sum over the 16 lanes of a row of a result.
__device__ __forceinline__ float row_sum(float x) {
    auto turn = [](float v, auto ctrl) {
        return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), decltype(ctrl)::value, 0xf, 0xf, true));
    };
    x += turn(x, std::integral_constant<int, 0x128>{});
    x += turn(x, std::integral_constant<int, 0x124>{});
    x += turn(x, std::integral_constant<int, 0x122>{});
    x += turn(x, std::integral_constant<int, 0x121>{});
    return x;
}

// The tiles of a diagonal in the sequences first, first + step, ...; a sequence's length is read while the one before it is walked through.
struct Diagonal {
    int t, step, it, end, b_next, seg, segs;
    int b, first, len;                  // of the sequence
    int from, to;                       // of the one to come, as they stand in memory
    __device__ __forceinline__ void start(const Args& a, int diagonal, int sequence, int seg, int splits) {
        this->seg = seg;
        t = diagonal, step = splits, b_next = sequence, segs = 1 << a.seg_bits, it = end = 0;
        peek(a);
    }
    __device__ __forceinline__ void peek(const Args& a) {
        const int n = min(b_next, a.B - 1);
        const int32_t* const ends = a.cu ? a.cu + 1 : a.seqlens;
        from = 0, to = a.L;
        if (a.cu) from = a.cu[n];
        if (ends) to = ends[n];
    }
    __device__ __forceinline__ bool advance(const Args& a) {             // to the next tile; false: none is left
        it += segs;
        while (it >= end) {
            if (b_next >= a.B) return false;
            b = b_next, first = __builtin_amdgcn_readfirstlane(from);
            const int last = __builtin_amdgcn_readfirstlane(to);
            len = first < 0 || last < first || (a.cu && last > a.total) ? 0 : min(last - first, a.L);
            b_next += step;
            peek(a);
            const int n = (len + TILE - 1) / TILE;
            it = max(0, t) + seg, end = min(n, n + t);
        }
        return true;
    }
};

template <int DT, bool PK, bool PQ>
struct TablesNext {
    Stage<DT, THREADS> q, k;
    Scores<DT> ds;
    __device__ __forceinline__ void load(const Diagonal& d, const Args& a, int h) {
        Where w;
        w.b = d.b, w.first = d.first, w.len = d.len;
        const int64_t row_tile = a.cu ? d.first / TILE + d.b : int64_t(d.b) * a.tiles;
        if constexpr (PK) Source<DT, THREADS>(a.q, a, w, h, d.it * TILE).load(q);
        if constexpr (PQ) Source<DT, THREADS>(a.k, a, w, h, (d.it - d.t) * TILE).load(k);
        ds.load(static_cast<const typename Elem<DT>::T*>(a.ds) + ((int64_t(h - a.head0) * a.row_tiles + row_tile + d.it) * a.tiles + d.it - d.t) * TILE_VALUES);
    }
};

// What a wave does, for each of the roles that waves have: every one of them passes the same barriers.  KEYS: it sums up for the table of queries (from keys).
template <int DT, bool PK, bool PQ, bool KEYS, bool FAR>
__device__ __forceinline__ void sum_tables(const Args& a, TablesLds<DT>& sm, Diagonal diagonal, int h, int split, int wave) {
    using E = Elem<DT>;
    using T = typename E::T;
    using X8 = typename E::X8;
    constexpr int SHARE = PK && PQ ? 2 : 4, BLOCKS = 8 / SHARE, SOME = BLOCKS == 4 ? 3 : 2;         // waves of a table, blocks of a wave, those that 32 rows reach
    const int share = wave % SHARE, c = lane_c(), g = lane_g();
    f32x4 acc[FAR ? 1 : BLOCKS][4];
#pragma unroll
    for (int n = 0; n < (FAR ? 1 : BLOCKS); ++n)
#pragma unroll
        for (int d = 0; d < 4; ++d) acc[n][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    const T* const rows = KEYS ? sm.k : sm.q;
    TablesNext<DT, PK, PQ> next;
    float power = 1.f, coming = 1.f;            // float16: of the sums, and of the next tile's sequence
    int of = -1;
    auto fetch = [&]() {
        next.load(diagonal, a, h);
        if (DT == TDB_F16 && diagonal.b != of) coming = score_power<DT>(a, h, diagonal.b), of = diagonal.b;
    };
    bool more = diagonal.advance(a);
    if (more) fetch();
    while (more) {
        if (DT == TDB_F16 && coming != power) {
#pragma unroll
            for (int n = 0; n < (FAR ? 1 : BLOCKS); ++n)
#pragma unroll
                for (int d = 0; d < 4; ++d) acc[n][d] *= coming / power;
            power = coming;
        }
        __syncthreads();
        if constexpr (PK) next.q.store(sm.q);
        if constexpr (PQ) next.k.store(sm.k);
        if constexpr (FAR) {
            next.ds.store(sm.by_key);
        } else {
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                const int j = Scores<DT>::key(n), i0 = Scores<DT>::query(0);
                T* const by_query = sm.by_query + i0 * (OFFSET_ROW<DT> + 1) - j + 63;
                T* const by_key = sm.by_key + j * (OFFSET_ROW<DT> - 1) + i0 + 63;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int i = 16 * (e >> 2) + (e & 3);
                    if constexpr (PK) by_query[i * (OFFSET_ROW<DT> + 1)] = next.ds.x[n][e];
                    if constexpr (PQ) by_key[i] = next.ds.x[n][e];
                }
            }
        }
        __syncthreads();
        more = diagonal.advance(a);
        if (more) fetch();
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            // far: 16 keys of the queries' sum, or 16 queries of the keys'; twice as many for half as many waves.  Else: 32 queries reach the blocks 2 u .. 2 u + 5, 32 keys
            // 2 - 2 u .. 7 - 2 u: of a wave's four all but the first or the last.
            constexpr int N = FAR ? 4 / SHARE : SOME;
            const int late = BLOCKS == 4 && (KEYS ? u == 0 : u == 1);
            X8 b[N];
#pragma unroll
            for (int n = 0; n < N; ++n) {
                if constexpr (!FAR) b[n] = offset_frag<DT>(KEYS ? sm.by_key : sm.by_query, 32 * u, 16 * (share + SHARE * (n + late)));
                else if constexpr (KEYS) b[n] = line_frag<DT>(sm.by_key, 32 * u, 16 * (share + SHARE * n));
                else b[n] = row_frag<DT>(sm.by_key, 16 * (share + SHARE * n), 32 * u);
            }
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                const X8 x = line_frag<DT>(rows, 32 * u, 16 * d);
#pragma unroll
                for (int n = 0; n < N; ++n) acc[FAR ? 0 : n + late][d] = E::mma(x, b[n], acc[FAR ? 0 : n + late][d]);
            }
        }
    }
    float* const part = a.partial + ((((int64_t(h - a.head0) * (2 * a.tiles - 1) + diagonal.t + a.tiles - 1) << (a.split_bits + a.seg_bits)) + split) * 2 + (KEYS ? 1 : 0)) * (BY_OFFSET * 64);
#pragma unroll
    for (int n = 0; n < (FAR ? 1 : BLOCKS); ++n)
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            if constexpr (DT == TDB_F16) acc[n][d] *= 1.f / power;
            if constexpr (FAR) {            // a row for each wave of a table
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[n][d][e] = row_sum(acc[n][d][e]);
                if (c == 0) *reinterpret_cast<f32x4*>(part + share * 64 + 16 * d + 4 * g) = acc[n][d];
            } else {
                *reinterpret_cast<f32x4*>(part + (16 * (share + SHARE * n) + c) * 64 + 16 * d + 4 * g) = acc[n][d];
            }
        }
}

// The batch above: 104 us.  A step asks for a tile of dS, of Q and of K, 450 MB in all, of which 225 come from beyond the XCDs' caches; 50 are written: 2.6 TB/s, half of what a
// large copy makes.  LDS is busy 45 % of the time, products 20, vector instructions 10: no unit is its bound, a step's chain of loads, LDS and two barriers is.  4 x 4096, where
// 15 of 127 diagonals are its: 280 us.
// (Each head's workgroups on one XCD, for its cache: equal, and 107 and 380 us in packed and long batches, whose diagonals are less alike.)
template <int DT, bool PK, bool PQ>
__global__ __launch_bounds__(THREADS, DT == TDB_F32 ? 1 : 3) void attn_bwd_tables_kernel(Args a) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    TablesLds<DT>& sm = *reinterpret_cast<TablesLds<DT>*>(smem);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // Long diagonals first.  A short one has no use for its last parts: which of eight neighbours, one for each XCD, these are changes from diagonal to diagonal.
    const int bits = a.split_bits + a.seg_bits, at = blockIdx.x >> bits, split = (blockIdx.x + at) & ((1 << bits) - 1), n = at / a.heads, t = n & 1 ? (n + 1) / 2 : -(n / 2);
    const int h = a.head0 + at - n * a.heads;
    const int splits = splits_of(a, t);
    Level level(a);
    level.ready();
    if ((split >> a.seg_bits) >= splits || level.has(t)) return;
    Diagonal diagonal;
    diagonal.start(a, t, split >> a.seg_bits, split & ((1 << a.seg_bits) - 1), splits);
    const bool keys = PQ && (!PK || wave >= 2);
    if (one_row(a, TILE * t - 63, TILE * t + 63)) {
        if (keys) sum_tables<DT, PK, PQ, PQ, true>(a, sm, diagonal, h, split, wave);
        else sum_tables<DT, PK, PQ, !PK, true>(a, sm, diagonal, h, split, wave);
        return;
    }
    for (int n = threadIdx.x; n < TILE * OFFSET_ROW<DT>; n += THREADS) sm.by_query[n] = sm.by_key[n] = typename Elem<DT>::T(0.f);
    if (keys) sum_tables<DT, PK, PQ, PQ, false>(a, sm, diagonal, h, split, wave);
    else sum_tables<DT, PK, PQ, !PK, false>(a, sm, diagonal, h, split, wave);
}

// A table row's gradient, offsets lo .. hi - 1: those of far diagonals come as one row for each wave of a table; the others, fewer than 128 at either end, from the one or
// two diagonals whose tiles have them.  A wave for each row, parts dealt to its four groups of 16 lanes and asked for four at a time; the outermost rows, which have
// hundreds of offsets, take the workgroup's waves together.  (A wave for each row, one part after the other, took 290 us at 4 x 4096, this 32; batch 32 x 512 18.)  Which group has a part does not depend on
// the longest length, and a sum's bits do not either.
template <int DT>
__global__ __launch_bounds__(THREADS) void tables_sum_kernel(Args a) {
    constexpr int MANY = 32, MOST_GROUPS = THREADS / 16;
    __shared__ f32x4 s_sum[MOST_GROUPS][16];
    const int which = blockIdx.z, h = a.head0 + blockIdx.y, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), d = threadIdx.x & 15;
    const int diagonals = 2 * a.tiles - 1, share_bits = a.pk.p && a.pq.p ? 1 : 2, split_bits = a.split_bits + a.seg_bits;
    if (!(which ? a.pq.p : a.pk.p)) return;
    const float* const parts = a.partial + (((int64_t(blockIdx.y) * diagonals) << (split_bits + 1)) + which) * (BY_OFFSET * 64) + 4 * d;
    const int row0 = blockIdx.x * WAVES, mine = a.starts[min(row0 + min(int(threadIdx.x & 63), WAVES), 2 * a.span)];       // lane n: where row row0 + n starts
    auto range = [&](int n, int& lo, int& hi) {         // (no offsets past the last row)
        lo = min(max(__builtin_amdgcn_readlane(mine, n), 1 - a.L), a.L), hi = min(max(__builtin_amdgcn_readlane(mine, n + 1), lo), a.L);
    };
    // the sum of the row's parts that group `group` of `groups` (a power of two) has
    auto sum_of = [&](int lo, int hi, int group, int groups) {
        // diagonals whose offsets all lie in the row's
        const int t0 = lo == 1 - a.L ? 1 - a.tiles : tile_up(a, lo + 63), t1 = hi == a.L ? a.tiles - 1 : tile_down(a, hi - 64);
        f32x4 sum = {0.f, 0.f, 0.f, 0.f};
        // where(n, t, at, s): part n is row `at` of part s of diagonal t; false: there is none
        auto add = [&](int from, int to, auto where) {
            constexpr int AHEAD = 4;
            for (int n = from + ((group - from) & (groups - 1)); n < to; n += AHEAD * groups) {
                f32x4 x[AHEAD];
#pragma unroll
                for (int u = 0; u < AHEAD; ++u) {
                    int t = 0, at = 0, s = 0;
                    const bool any = n + u * groups < to && where(n + u * groups, t, at, s) && (s >> a.seg_bits) < splits_of(a, t);
                    const int64_t tile = ((int64_t(t + a.tiles - 1) << split_bits) + s) * (2 * BY_OFFSET * 64);
                    const f32x4 y = *reinterpret_cast<const f32x4*>(parts + (any ? tile + at * 64 : 0));
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[u][e] = any ? y[e] : 0.f;
                }
#pragma unroll
                for (int u = 0; u < AHEAD; ++u) sum += x[u];
            }
        };
        const int zero = (a.L + MOST_GROUPS - 1) / MOST_GROUPS * MOST_GROUPS;           // offset `off` has the numbers (off + zero) << (split_bits + 1) ...
        auto offsets = [&](int from, int to) {
            add((from + zero) << (split_bits + 1), (to + zero) << (split_bits + 1), [&](int n, int& t, int& at, int& s) {
                const int off = (n >> (split_bits + 1)) - zero;
                t = ((off + 63) >> 6) - ((n >> split_bits) & 1), at = off + 63 - TILE * t, s = n & ((1 << split_bits) - 1);
                return at <= 126 && t > -a.tiles && t < a.tiles && !(t0 <= t && t <= t1);
            });
        };
        if (t0 > t1) {
            offsets(lo, hi);
        } else {                        // what diagonals t0 - 1 and t1 + 1 have, where there are such
            if (t0 > 1 - a.tiles) offsets(lo, min(TILE * t0, hi));
            if (t1 < a.tiles - 1) offsets(max(TILE * t1 + 1, lo), hi);
        }
        if (t0 <= t1 && (lo == 1 - a.L || hi == a.L)) {      // level tiles: a sum of each workgroup that has met one, which stands for them all
            const float* const from = a.level_parts + (int64_t(which * a.heads + blockIdx.y) * a.blocks * 2 + (hi == a.L ? 0 : 1)) * 64 + 4 * d;
            const int share = min(groups, 4), mine = group & (share - 1);           // groups that share a sequence
            for (int b = group / share; b < a.B; b += groups / share) {
                int64_t first;
                const int len = valid_rows(a, b, first), tiles = (len + TILE - 1) / TILE;
                const int64_t at = a.cu ? first / TILE + b : int64_t(b) * a.tiles;
                for (int n = mine; n < tiles; n += 4 * share) {
                    f32x4 x[4];
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        const bool any = n + u * share < tiles;
                        const f32x4 y = *reinterpret_cast<const f32x4*>(from + (at + (any ? n + u * share : 0)) * 128);
#pragma unroll
                        for (int e = 0; e < 4; ++e) x[u][e] = any ? y[e] : 0.f;
                    }
#pragma unroll
                    for (int u = 0; u < 4; ++u) sum += x[u];
                }
            }
        } else if (t0 <= t1) {
            const int first = (a.tiles + MOST_GROUPS - 1) / MOST_GROUPS * MOST_GROUPS, bits = share_bits + split_bits;
            add((t0 + first) << bits, (t1 + 1 + first) << bits, [&](int n, int& t, int& at, int& s) {
                t = (n >> bits) - first, at = (n >> split_bits) & ((1 << share_bits) - 1), s = n & ((1 << split_bits) - 1);
                return true;
            });
        }
        return sum;
    };
    auto store = [&](int row, float all) {
        if (row >= 2 * a.span || int(threadIdx.x & 63) >= a.D) return;
        using T = typename Elem<DT>::T;
        T* const to = static_cast<T*>(which ? a.dpq : a.dpk) + h * (which ? a.dpq_h : a.dpk_h) + int64_t(row) * a.D + (threadIdx.x & 63);
        *to = T(all * (a.scale * a.factor));
    };
    // what lane 4 d + e of a wave adds up: value e of lane d of each group
    auto total = [&](int first, int groups) {
        float all = 0.f;
        for (int n = 0; n < groups; ++n) all += s_sum[first + n][(threadIdx.x & 63) >> 2][threadIdx.x & 3];
        return all;
    };
    int lo, hi;
    range(wave, lo, hi);
    const bool many = hi - lo > MANY;
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
    if (!many && hi > lo) sum = sum_of(lo, hi, (threadIdx.x >> 4) & 3, 4);
    s_sum[threadIdx.x >> 4][d] = sum;
    __syncthreads();
    if (!many) store(row0 + wave, total(4 * wave, 4));
    for (int n = 0; n < WAVES; ++n) {           // (the same for every wave)
        range(n, lo, hi);
        if (hi - lo <= MANY) continue;
        __syncthreads();
        s_sum[threadIdx.x >> 4][d] = sum_of(lo, hi, threadIdx.x >> 4, MOST_GROUPS);
        __syncthreads();
        if (wave == n) store(row0 + n, total(0, MOST_GROUPS));
    }
}

// ---------------------------------------------------------------------------------------------------------------- host

size_t elem(int dtype) { return dtype == TDB_F32 ? 4 : 2; }
int64_t up(int64_t x) { return (x + 255) / 256 * 256; }

constexpr int64_t MOST_STRIDE = int64_t(1) << 24;        // bytes: 64 rows' offsets fit 31 bits
constexpr int64_t MOST_SCORES = int64_t(2) << 30;        // bytes of dS, and of the positions' sums, at a time, unless one head has more (4 x 4096, 12 heads: 3.1 ms with 512 MiB, 2.8)

// Whether there are position terms; without them the table's fields mean nothing and are not looked at.
bool has_terms(const tdb_train_attn_args& a) { return a.pos_key || a.pos_query; }

// No sequence of a packing is longer than all its tokens, whatever bound the caller gives.
int longest_of(const tdb_train_attn_args& a) { return a.cu_seqlens ? std::max(1, std::min(a.max_seqlen, a.total_tokens)) : a.max_seqlen; }

// What a backward call needs, and how many heads it takes at a time.
struct Plan {
    int tiles, row_tiles, split_bits, seg_bits, heads;
    int64_t lines, largest, starts, delta, level, partial, sums, ds, bytes;       // offsets of the parts, and the sum
};
Plan plan_of(const tdb_train_attn_args& a) {
    Plan p;
    p.tiles = (longest_of(a) + TILE - 1) / TILE;
    p.row_tiles = a.cu_seqlens ? a.total_tokens / TILE + a.batch : a.batch * p.tiles;
    p.lines = a.cu_seqlens ? a.total_tokens : int64_t(a.batch) * a.max_seqlen;
    const int64_t each = int64_t(p.row_tiles) * p.tiles * TILE_VALUES * int64_t(elem(a.dtype));
    const bool terms = has_terms(a);
    const int diagonals = 2 * p.tiles - 1;
    int least = 0;                                  // parts of a long diagonal, see below
    while (least < 12 && p.row_tiles >> least > 64) ++least;
    const int64_t part = BY_OFFSET * 64 * 4, sums = terms ? ((int64_t(diagonals) << (least + 1)) * part) + int64_t(p.row_tiles) * (p.tiles * ROW_SUMS * 4 + 1024) : 0;
    p.heads = int(std::max<int64_t>(1, std::min<int64_t>(a.heads, MOST_SCORES / std::max<int64_t>({each, sums, 1}))));
    // A diagonal's parts, a power of two: three workgroups for each of 256 CUs where every diagonal has its own sums, and 64 tiles for a workgroup where most are level
    // (4 x 4096: 281 us and 32 for the sums; with 32 tiles 230 and 54, for sums of half of dS's size).
    int bits = 0;
    while ((int64_t(2) << bits) * p.heads * p.tiles <= 768 && (2 << bits) <= a.batch) ++bits;
    bits = std::max(bits, least);
    p.split_bits = 0;
    while (p.split_bits < bits && (2 << p.split_bits) <= a.batch) ++p.split_bits;
    p.seg_bits = bits - p.split_bits;
    p.largest = 256;                                // in front: the diagonals of level tiles
    p.starts = p.largest + (a.dtype == TDB_F16 ? up(int64_t(a.heads) * a.batch * 8) : 0);
    p.delta = p.starts + (terms ? up((2 * int64_t(a.span) + 1) * 4) : 0);
    p.level = p.delta + up(p.lines * a.heads * 4);
    p.partial = p.level + (terms ? int64_t(2) * p.heads * p.row_tiles * 2 * 64 * 4 : 0);
    p.sums = p.partial + (terms ? ((int64_t(p.heads) * diagonals) << (bits + 1)) * part : 0);
    p.ds = p.sums + (terms ? int64_t(p.heads) * p.row_tiles * p.tiles * ROW_SUMS * 4 : 0);
    p.bytes = p.ds + p.heads * each;
    return p;
}

bool aligned(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

int check(const tdb_train_attn_args* a, bool backward, bool sizes_only = false) {
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
    if (has_terms(*a) && (a->span < 1 || a->span > (1 << 20))) return tdb_fail(TDB_ERR_POSITION, "span %d out of range", a->span);
    if (sizes_only || a->batch == 0 || lines == 0) return TDB_OK;
    if (!a->q || !a->k || !a->v || !a->o || !a->lse || (backward && (!a->dout || !a->dq || !a->dk || !a->dv || !a->workspace)))
        return tdb_fail(TDB_ERR_NULL, "a required pointer is NULL");
    if (a->threshold && !a->seed) return tdb_fail(TDB_ERR_NULL, "dropout needs a seed");
    const void* ptrs[] = {a->q, a->k, a->v, a->o, a->dout, a->dq, a->dk, a->dv, a->pos_key, a->pos_query, a->workspace, a->o_rest};
    for (const void* p : ptrs)
        if (!aligned(p)) return tdb_fail(TDB_ERR_ALIGN, "tensors must be 16-byte aligned");
    for (int n = 0; n < 24; ++n) {
        const int64_t s = (&a->q_stride_b)[n];
        if (s < 0 || s * int64_t(elem(a->dtype)) % 16) return tdb_fail(TDB_ERR_STRIDE, "strides must be non-negative multiples of 16 bytes");
    }
    const int64_t rows[] = {a->q_stride_l, a->k_stride_l, a->v_stride_l, a->o_stride_l, a->dout_stride_l, a->dq_stride_l, a->dk_stride_l, a->dv_stride_l};
    for (int n = 0; n < (backward ? 8 : 4); ++n)
        if (rows[n] < a->head_dim || rows[n] * int64_t(elem(a->dtype)) > MOST_STRIDE)
            return tdb_fail(TDB_ERR_STRIDE, "rows must lie head_dim values to 16 MiB apart");
    const int64_t written[][2] = {{a->o_stride_h, a->o_stride_b}, {a->dq_stride_h, a->dq_stride_b}, {a->dk_stride_h, a->dk_stride_b}, {a->dv_stride_h, a->dv_stride_b}};
    for (int n = backward ? 1 : 0; n < (backward ? 4 : 1); ++n)
        if ((a->heads > 1 && written[n][0] < a->head_dim) || (!a->cu_seqlens && a->batch > 1 && written[n][1] < a->head_dim)) return tdb_fail(TDB_ERR_STRIDE, "rows of a result overlap");
    const int64_t table[] = {a->pos_key_stride_h, a->pos_key_stride_r, a->pos_query_stride_h, a->pos_query_stride_r};
    for (int64_t s : table)
        if (s < 0 || s * int64_t(elem(a->dtype)) % 16) return tdb_fail(TDB_ERR_STRIDE, "strides of the tables must be non-negative multiples of 16 bytes");
    if (has_terms(*a)) {
        if (2 * int64_t(a->span) * std::max(a->pos_key ? a->pos_key_stride_r : 0, a->pos_query ? a->pos_query_stride_r : 0) * int64_t(elem(a->dtype)) > INT32_MAX)
            return tdb_fail(TDB_ERR_STRIDE, "a head's table must lie within 2 GiB");
        if (!a->delta_lut || a->lut_half < a->max_seqlen - 1) return tdb_fail(TDB_ERR_POSITION, "delta_lut is missing or shorter than the sequences");
        if (backward && ((a->pos_key && !a->dpos_key) || (a->pos_query && !a->dpos_query))) return tdb_fail(TDB_ERR_NULL, "a table's gradient has no place");
        const int64_t least = a->heads > 1 ? 2 * int64_t(a->span) * a->head_dim : 0;
        if (backward && ((a->pos_key && a->dpos_key_stride_h < least) || (a->pos_query && a->dpos_query_stride_h < least)))
            return tdb_fail(TDB_ERR_STRIDE, "gradients of the heads' tables overlap");
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
    if (has_terms(a)) k.lut = a.delta_lut, k.lut_half = a.lut_half, k.span = a.span;
    k.seqlens = a.seqlens_k, k.cu = a.cu_seqlens;
    k.B = a.batch, k.H = a.heads, k.D = a.head_dim, k.L = longest_of(a), k.total = a.total_tokens;
    k.head0 = 0, k.heads = a.heads;
    k.lines = p.lines, k.lse = a.lse, k.rest = a.dtype == TDB_F32 ? nullptr : a.o_rest;
    k.tiles = p.tiles, k.row_tiles = p.row_tiles, k.split_bits = p.split_bits, k.seg_bits = p.seg_bits, k.per_tile = 65536 / p.tiles + 1;
    k.dpk = a.dpos_key, k.dpq = a.dpos_query, k.dpk_h = a.dpos_key_stride_h, k.dpq_h = a.dpos_query_stride_h;
    k.seed = a.seed, k.threshold = uint32_t(a.threshold), k.factor = tdb_kept_factor(a.threshold), k.scale = a.sm_scale;
    while (k.p_shift < 15 && (2 << k.p_shift) <= k.L) ++k.p_shift;
    if (a.workspace) {
        char* const at = static_cast<char*>(a.workspace);
        k.level = reinterpret_cast<int32_t*>(at), k.largest = reinterpret_cast<uint32_t*>(at + p.largest);
        k.starts = reinterpret_cast<int32_t*>(at + p.starts);
        k.level_parts = reinterpret_cast<float*>(at + p.level), k.row_sums = reinterpret_cast<float*>(at + p.sums);
        k.delta = reinterpret_cast<float*>(at + p.delta);
        k.partial = reinterpret_cast<float*>(at + p.partial);
        k.ds = at + p.ds;
    }
    return k;
}

int blocks_of(const Args& k, int rows) { return k.cu ? k.total / rows + k.B : k.B * ((k.L + rows - 1) / rows); }

// The kernels' LDS lies above what a launch has without asking, once per device and kernel.
template <auto kernel>
hipError_t launch(size_t lds, int64_t grid, int threads, hipStream_t s, const Args& k) {
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
    kernel<<<unsigned(grid), threads, lds, s>>>(k);
    return hipGetLastError();
}

// The kernel's instance for the terms that a call has.
template <template <bool, bool> class F>
hipError_t by_terms(const Args& k, hipStream_t s) {
    if (k.pk.p && k.pq.p) return F<true, true>::run(k, s);
    if (k.pk.p) return F<true, false>::run(k, s);
    if (k.pq.p) return F<false, true>::run(k, s);
    return F<false, false>::run(k, s);
}

template <int DT>
struct Launch {
    static_assert(sizeof(FwdLds<DT>) * PER_CU<DT> <= 163840 && sizeof(KvLds<DT>) * PER_CU<DT> <= 163840, "LDS of a CU");
    template <bool PK, bool PQ>
    struct Fwd {
        static hipError_t run(Args k, hipStream_t s) {
            k.blocks = blocks_of(k, TILE);
            return launch<attn_fwd_kernel<DT, PK, PQ>>(sizeof(FwdLds<DT>), int64_t(k.blocks) * k.heads, THREADS, s, k);
        }
    };
    template <bool PK, bool PQ>
    struct Heads {                      // the backward pass of a number of heads
        static hipError_t run(Args k, hipStream_t s) {
            k.blocks = blocks_of(k, TILE);
            hipError_t e = launch<attn_bwd_kv_kernel<DT, PK, PQ>>(sizeof(KvLds<DT>), int64_t(k.blocks) * k.heads, THREADS, s, k);
            if (e != hipSuccess) return e;
            k.blocks = blocks_of(k, TILE);
            e = launch<attn_bwd_q_kernel<DT, PK>>(sizeof(QLds<DT>), int64_t(k.blocks) * k.heads, THREADS, s, k);
            if constexpr (PK || PQ) {
                if (e != hipSuccess) return e;
                e = launch<attn_bwd_tables_kernel<DT, PK, PQ>>(sizeof(TablesLds<DT>), (int64_t(k.heads) * (2 * k.tiles - 1)) << (k.split_bits + k.seg_bits), THREADS, s, k);
                if (e != hipSuccess) return e;
                tables_sum_kernel<DT><<<dim3((2 * k.span + WAVES - 1) / WAVES, k.heads, 2), THREADS, 0, s>>>(k);
                e = hipGetLastError();
            }
            return e;
        }
    };
    static hipError_t forward(const Args& k, hipStream_t s) { return by_terms<Fwd>(k, s); }
    static hipError_t backward(Args k, int heads, hipStream_t s) {
        if (DT == TDB_F16) {
            const int64_t n = int64_t(k.H) * k.B * 2;
            clear_kernel<<<unsigned(std::min<int64_t>((n + THREADS - 1) / THREADS, 1024)), THREADS, 0, s>>>(k.largest, n);
        }
        k.blocks = blocks_of(k, TILE);
        attn_delta_kernel<DT><<<unsigned(int64_t(k.blocks) * k.H), THREADS, 0, s>>>(k);
        hipError_t e = hipGetLastError();
        for (k.head0 = 0; e == hipSuccess && k.head0 < k.H; k.head0 += heads) {
            k.heads = std::min(heads, k.H - k.head0);
            e = by_terms<Heads>(k, s);
        }
        return e;
    }
};

int run(const tdb_train_attn_args* a, bool back, void* stream) {
    if (const int rc = check(a, back); rc != TDB_OK) return rc;
    const Plan p = plan_of(*a);
    if (a->batch == 0 || p.lines == 0) return TDB_OK;
    const Args k = args_of(*a, p);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    hipError_t e;
    if (a->dtype == TDB_F32) e = back ? Launch<TDB_F32>::backward(k, p.heads, s) : Launch<TDB_F32>::forward(k, s);
    else if (a->dtype == TDB_BF16) e = back ? Launch<TDB_BF16>::backward(k, p.heads, s) : Launch<TDB_BF16>::forward(k, s);
    else e = back ? Launch<TDB_F16>::backward(k, p.heads, s) : Launch<TDB_F16>::forward(k, s);
    if (e != hipSuccess) return tdb_fail(TDB_ERR_LAUNCH, "kernel launch failed: %s", hipGetErrorString(e));
    return TDB_OK;
}

}  // namespace tdb_train

extern "C" {

int tdb_attn_train_fwd(const tdb_train_attn_args* args, void* stream) { return tdb_train::run(args, false, stream); }
int tdb_attn_train_bwd(const tdb_train_attn_args* args, void* stream) { return tdb_train::run(args, true, stream); }
int64_t tdb_attn_train_workspace(const tdb_train_attn_args* args) { return tdb_train::check(args, false, true) == TDB_OK ? tdb_train::plan_of(*args).bytes : 0; }

}  // extern "C"
