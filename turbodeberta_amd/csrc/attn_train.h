// Parts of the attention kernels for training: tiles in LDS, operands of the matrix instructions, scores with their position terms.
//
// Types.  A "frag" is what a lane has of an operand of 16 rows x 32 columns of the contraction: 8 values of row (or column) c = lane & 15, columns
// 8 g .. 8 g + 7, g = lane >> 4.  In 16 bits that is one matrix instruction (16x16x32), in float32 eight (16x16x4: step s contracts column
// 8 g + s of lane group g; the order of a sum is free as long as both operands have it).  A result has row 4 g + e (e = 0..3), column c in a lane.
//
// Layout of scores.  A wave owns 16 NX rows x (a lane has one of each 16) and runs over the other side's rows y, 64 a step: S[y][x], y in the
// result's rows.  Forward x are queries and y keys, so a softmax row is in a lane and the three others of its column, and the probabilities are an operand
// of the next product as they stand.  Backward x are keys and y queries: the same for the gradients of keys and values.
//
// Position terms.  Both are functions of x - y (r = x - y + 63 in a tile), with the table of x's side ("own") and of y's ("other"):
//   own:   x . T_own[r]    computed for the 80 r that 16 x and 64 y have, result columns x: stored to LDS as rows x, index y + 16 - x, a row of
//          81 floats: x * 81 + 16 - x + y is a multiple of 4 for every y that is one, so four y at once are one read of 16 bytes.
//   other: y . T_other[r]  for the 16 (NX + 1) r of 16 y and the wave's x, result columns y: stored as rows y, read back value by value, lanes
//          along x, without conflicts.
// They are held in float32.  The tables' rows lie in LDS as rings in the order of r; 64 rows are new in each step.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "philox.h"
#include "tdb_internal.h"
#include "tdb_train.h"

namespace tdb_train {

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(8))) float f32x8;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((ext_vector_type(8))) short s16x8;
typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;

#define TDB_SHARED(T, p) ((__attribute__((address_space(3))) T*)(p))

template <int DT>
struct Elem;
template <>
struct Elem<TDB_BF16> {
    using T = __bf16;
    using X8 = bf16x8;
    static __device__ __forceinline__ f32x4 mma(X8 a, X8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <>
struct Elem<TDB_F16> {
    using T = _Float16;
    using X8 = f16x8;
    static __device__ __forceinline__ f32x4 mma(X8 a, X8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
template <>
struct Elem<TDB_F32> {
    using T = float;
    using X8 = f32x8;
    static __device__ __forceinline__ f32x4 mma(X8 a, X8 b, f32x4 c) {
#pragma unroll
        for (int s = 0; s < 8; ++s) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[s], b[s], c, 0, 0, 0);
        return c;
    }
};

constexpr int TILE = 64;                        // rows y of a step, and of a tile of score gradients
constexpr int TILE_VALUES = TILE * TILE;
constexpr int THREADS = 256;
constexpr float LOG2E = 1.44269504088896340736f;

// Rows of 64 values in LDS, 16 bytes apart: 16 rows at the same column are on distinct banks.
template <int DT>
constexpr int ROW = DT == TDB_F32 ? 68 : 72;
// 16-byte pieces of a row of 64 values, and of a tile for each thread
template <int DT>
constexpr int PIECES = DT == TDB_F32 ? 16 : 8;
template <int DT>
constexpr int LOADS = TILE * PIECES<DT> / THREADS;

__device__ __forceinline__ int lane_c() { return threadIdx.x & 15; }
__device__ __forceinline__ int lane_g() { return threadIdx.x >> 4 & 3; }

// Between writes and reads of a wave's own part of LDS: the hardware keeps their order, the compiler is told to.
__device__ __forceinline__ void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

template <int DT>
__device__ __forceinline__ typename Elem<DT>::X8 zero8() {
    typename Elem<DT>::X8 x;
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = typename Elem<DT>::T(0.f);
    return x;
}

// Eight neighbouring values at a 16-byte boundary of LDS or global memory.
template <int DT>
__device__ __forceinline__ typename Elem<DT>::X8 read8(const typename Elem<DT>::T* p) {
    if constexpr (DT == TDB_F32) {
        const f32x4 lo = *reinterpret_cast<const f32x4*>(p), hi = *reinterpret_cast<const f32x4*>(p + 4);
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    } else {
        return *reinterpret_cast<const typename Elem<DT>::X8*>(p);
    }
}

// Frag of rows `row` + c, columns k0 + 8 g ..
template <int DT>
__device__ __forceinline__ typename Elem<DT>::X8 row_frag(const typename Elem<DT>::T* rows, int row, int k0) {
    return read8<DT>(rows + (row + lane_c()) * ROW<DT> + k0 + 8 * lane_g());
}

// Transposed frags: the lane's row of the operand is column col + c in LDS, the contraction runs over rows in LDS.  Each lane gives the address of four columns of
// one row; the hardware hands the lanes of a group their columns.  `lo` and `hi`: first of the four rows of the lane group's two halves.
template <int DT>
__device__ __forceinline__ typename Elem<DT>::X8 turned_frag(const typename Elem<DT>::T* rows, int stride, int lo, int hi, int col) {
    if constexpr (DT == TDB_F32) {
        f32x8 x;
#pragma unroll
        for (int s = 0; s < 4; ++s) x[s] = rows[(lo + s) * stride + col + lane_c()], x[4 + s] = rows[(hi + s) * stride + col + lane_c()];
        return x;
    } else {
        const int at = (lane_c() >> 2) * stride + col + 4 * (lane_c() & 3);
        const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16(TDB_SHARED(s16x4, rows + lo * stride + at));
        const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16(TDB_SHARED(s16x4, rows + hi * stride + at));
        return __builtin_bit_cast(typename Elem<DT>::X8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
    }
}
// Over rows k0 + 8 g + s
template <int DT>
__device__ __forceinline__ typename Elem<DT>::X8 line_frag(const typename Elem<DT>::T* rows, int stride, int k0, int col) {
    return turned_frag<DT>(rows, stride, k0 + 8 * lane_g(), k0 + 8 * lane_g() + 4, col);
}
// Over rows k0 + 4 g + s and k0 + 16 + 4 g + s, the order in which two results of 16 rows are an operand
template <int DT>
__device__ __forceinline__ typename Elem<DT>::X8 pair_frag(const typename Elem<DT>::T* rows, int stride, int k0, int col) {
    return turned_frag<DT>(rows, stride, k0 + 4 * lane_g(), k0 + 16 + 4 * lane_g(), col);
}

// Strides in elements; the last dimension is contiguous, every row starts at a multiple of 16 bytes.
struct Tensor {
    void* p;
    int64_t b, h, l;
};

struct Args {
    Tensor q, k, v, o, dout, dq, dk, dv;
    Tensor pk, pq;                      // b unused, l: row
    const int32_t* lut;
    int32_t lut_half, span;
    const int32_t *seqlens, *cu;        // packed where cu is there
    int32_t B, H, D, L, total;
    int32_t head0, heads;               // of this launch
    int32_t blocks;                     // per head
    int64_t lines;                      // rows of lse and delta for each head
    float *lse, *delta;
    void* ds;                           // [heads][tiles of rows][tiles][64 x 64]
    float* partial;
    int32_t tiles, row_tiles, splits;   // tiles: of the longest sequence; row_tiles: of all sequences
    void *dpk, *dpq;                    // [H, table rows, D]
    int64_t dpk_h, dpq_h;
    const int64_t* seed;
    uint32_t threshold;
    float factor, scale;
    int32_t p_shift;                    // float16: probabilities are multiplied by 2^p_shift where they are rounded
    const uint32_t* largest;            // float16: squares of the largest norms of a row of dout and of v
};

struct Where {
    int b, row0, len;       // sequence, first row of the tile, valid rows of the sequence
    int64_t first;          // row of the packed tensors (else 0)
    int64_t line;           // of lse and delta
    int64_t row_tile;       // number of the sequence's first row tile among all sequences'
};

__device__ __forceinline__ int valid_rows(const Args& a, int b, int64_t& first) {
    if (!a.cu) {
        first = 0;
        return a.seqlens ? min(max(a.seqlens[b], 0), a.L) : a.L;
    }
    const int s = a.cu[b], e = a.cu[b + 1];
    first = s;
    return s < 0 || e < s || e > a.total ? 0 : min(e - s, a.L);       // (a malformed entry has no rows)
}

// A workgroup's head and tile of `rows` rows (a power of two from 64 on); false where it has none.  Workgroups are started in turn on the 8 XCDs: neighbours in the
// numbering below, which read the same tensors, share one's cache.  Packed sequences have first / rows + b tiles in front of them at most.
template <int rows>
__device__ __forceinline__ bool locate(const Args& a, int& h, Where& w) {
    const uint32_t all = uint32_t(a.blocks) * a.heads, id = blockIdx.x, part = all >> 3, more = all & 7, xcd = id & 7;
    const uint32_t n = xcd * part + min(xcd, more) + (id >> 3);
    h = __builtin_amdgcn_readfirstlane(int(n / uint32_t(a.blocks)));
    const int block = int(n) - h * a.blocks;
    h += a.head0;
    if (!a.cu) {
        const int tiles = (a.L + rows - 1) / rows;
        w.b = block / tiles;
        w.row0 = (block - w.b * tiles) * rows;
        w.len = valid_rows(a, w.b, w.first);
        w.line = int64_t(w.b) * a.L;
        w.row_tile = int64_t(w.b) * a.tiles;
        return true;
    }
    int lo = 0, hi = a.B;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.cu[mid] / rows + mid <= block) lo = mid;
        else hi = mid;
    }
    w.b = __builtin_amdgcn_readfirstlane(lo);
    w.len = valid_rows(a, w.b, w.first);
    w.row0 = (block - w.b - int(w.first) / rows) * rows;
    w.line = w.first;
    w.row_tile = w.first / TILE + w.b;
    return w.row0 >= 0 && w.row0 < w.len;
}

template <int DT>
__device__ __forceinline__ const typename Elem<DT>::T* rows_of(const Tensor& t, const Args& a, const Where& w, int h) {
    return static_cast<const typename Elem<DT>::T*>(t.p) + (a.cu ? w.first * t.l : w.b * t.b) + h * t.h;
}

// A tile of 64 rows of 64 values on its way from global memory to LDS.
template <int DT>
struct Stage {
    using T = typename Elem<DT>::T;
    static constexpr int EACH = 64 / PIECES<DT>, STEP = THREADS / PIECES<DT>;      // values of a piece, rows of a pass
    u32x4 x[LOADS<DT>];
    static __device__ __forceinline__ int row(int n) { return threadIdx.x / PIECES<DT> + n * STEP; }
    static __device__ __forceinline__ int col() { return threadIdx.x % PIECES<DT> * EACH; }
    // rows row0 .., zeros from `len` on and past D columns
    __device__ __forceinline__ void load(const T* rows, int64_t stride, int row0, int len, int D) {
#pragma unroll
        for (int n = 0; n < LOADS<DT>; ++n) {
            const int r = row0 + row(n);
            x[n] = r < len && col() < D ? *reinterpret_cast<const u32x4*>(rows + r * stride + col()) : u32x4{0, 0, 0, 0};
        }
    }
    // rows of a table, given for each pass
    __device__ __forceinline__ void load(const T* rows, int64_t stride, const int (&which)[LOADS<DT>], int D) {
#pragma unroll
        for (int n = 0; n < LOADS<DT>; ++n)
            x[n] = col() < D ? *reinterpret_cast<const u32x4*>(rows + which[n] * stride + col()) : u32x4{0, 0, 0, 0};
    }
    __device__ __forceinline__ void store(T* rows) const {
#pragma unroll
        for (int n = 0; n < LOADS<DT>; ++n) *reinterpret_cast<u32x4*>(rows + row(n) * ROW<DT> + col()) = x[n];
    }
};

// The table rows of 64 neighbouring r: r = r0 + (row of the stage) of a tile whose x start at x0 and whose y start at y0.  SIGN: 1 where x are
// queries (relative position x - y), -1 where they are keys.
template <int DT, int SIGN>
__device__ __forceinline__ void table_rows(const Args& a, int r0, int x0, int y0, int (&which)[LOADS<DT>]) {
#pragma unroll
    for (int n = 0; n < LOADS<DT>; ++n) {
        const int at = SIGN * (r0 + Stage<DT>::row(n) - 63 + x0 - y0);
        which[n] = a.lut[min(max(at, -a.lut_half), a.lut_half) + a.lut_half];
    }
}

// Sum, and maximum, over the four lanes of a column.
__device__ __forceinline__ float column_sum(float x) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const uint32_t w = __builtin_bit_cast(uint32_t, __builtin_bit_cast(float, uint32_t(r[0])) + __builtin_bit_cast(float, uint32_t(r[1])));
    const auto s = __builtin_amdgcn_permlane32_swap(w, w, false, false);
    return __builtin_bit_cast(float, uint32_t(s[0])) + __builtin_bit_cast(float, uint32_t(s[1]));
}
__device__ __forceinline__ float column_max(float x) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const uint32_t w = __builtin_bit_cast(uint32_t, fmaxf(__builtin_bit_cast(float, uint32_t(r[0])), __builtin_bit_cast(float, uint32_t(r[1]))));
    const auto s = __builtin_amdgcn_permlane32_swap(w, w, false, false);
    return fmaxf(__builtin_bit_cast(float, uint32_t(s[0])), __builtin_bit_cast(float, uint32_t(s[1])));
}

constexpr int OWN_ROW = 81;                     // floats of a row of x's term, see above
template <int NX>
constexpr int OTHER_ROW = 16 * (NX + 1) + 4;    // and of y's term: 16 rows at the same column are on distinct banks
// floats of a wave's scratch for the two
template <int NX>
constexpr int TERMS = NX * 16 * OWN_ROW + 16 * OTHER_ROW<NX>;

// Place of a ring's row; at is below twice its size.
template <int ring>
__device__ __forceinline__ int wrapped(int at) {
    return at >= ring ? at - ring : at;
}

// Scores of the wave's 16 NX rows x (x blocks first .. first + NX - 1 of 16 rows) with a step's 64 rows y, without the scale.  own[a][k]: frags of x.  Rings of
// `ring` rows whose row for r is (r + base) mod ring.  scratch: the wave's own, TERMS<NX> floats.
template <int DT, int NX, int ring>
__device__ __forceinline__ void scores(f32x4 (&s)[NX][4], const typename Elem<DT>::X8 (&own)[NX][2], const typename Elem<DT>::T* y_rows,
                                       const typename Elem<DT>::T* own_ring, const typename Elem<DT>::T* other_ring, bool has_own, bool has_other, int base,
                                       int first, float* scratch) {
    using E = Elem<DT>;
    using X8 = typename E::X8;
    const int c = lane_c(), g = lane_g();
    const f32x4 none = {0.f, 0.f, 0.f, 0.f};
    if (has_own) {
#pragma unroll
        for (int n = 0; n < NX + 4; ++n) {      // r = 16 (first + n) + 15 - row of the frag
            const int at = wrapped<ring>(16 * (first + n) + base);
            const X8 t0 = read8<DT>(own_ring + (at + 15 - c) * ROW<DT> + 8 * g), t1 = read8<DT>(own_ring + (at + 15 - c) * ROW<DT> + 32 + 8 * g);
#pragma unroll
            for (int a = 0; a < NX; ++a) {
                const int b = n - a;
                if (b < 0 || b > 4) continue;
                const f32x4 w = E::mma(t1, own[a][1], E::mma(t0, own[a][0], none));
                float* const to = scratch + a * 16 * OWN_ROW + c * OWN_ROW + 64 - 16 * b + 4 * g;
#pragma unroll
                for (int e = 0; e < 4; ++e) to[e] = w[e];
            }
        }
        wave_fence();
#pragma unroll
        for (int a = 0; a < NX; ++a)
#pragma unroll
            for (int m = 0; m < 4; ++m) s[a][m] = *reinterpret_cast<const f32x4*>(scratch + a * 16 * OWN_ROW + c * (OWN_ROW - 1) + 16 + 16 * m + 4 * g);
        wave_fence();
    } else {
#pragma unroll
        for (int a = 0; a < NX; ++a)
#pragma unroll
            for (int m = 0; m < 4; ++m) s[a][m] = none;
    }
    float* const other = scratch + NX * 16 * OWN_ROW;
#pragma unroll
    for (int m = 0; m < 4; ++m) {
        const X8 y0 = row_frag<DT>(y_rows, 16 * m, 0), y1 = row_frag<DT>(y_rows, 16 * m, 32);
#pragma unroll
        for (int a = 0; a < NX; ++a) s[a][m] = E::mma(y1, own[a][1], E::mma(y0, own[a][0], s[a][m]));
        if (has_other) {
#pragma unroll
            for (int n = 0; n <= NX; ++n) {     // r = 16 (first - m + 3 + n) + row
                const int at = wrapped<ring>(16 * (first - m + 3 + n) + base);
                const X8 t0 = row_frag<DT>(other_ring, at, 0), t1 = row_frag<DT>(other_ring, at, 32);
                const f32x4 w = E::mma(t1, y1, E::mma(t0, y0, none));
                *reinterpret_cast<f32x4*>(other + c * OTHER_ROW<NX> + 16 * n + 4 * g) = w;
            }
            wave_fence();
#pragma unroll
            for (int a = 0; a < NX; ++a)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[a][m][e] += other[(4 * g + e) * OTHER_ROW<NX> + 16 * a + c + 15 - 4 * g - e];
            wave_fence();
        }
    }
}

// Four neighbouring values of a result's row, rounded to the type.
template <int DT>
__device__ __forceinline__ void store4(typename Elem<DT>::T* p, f32x4 v) {
    using T = typename Elem<DT>::T;
    typedef __attribute__((ext_vector_type(4))) T T4;
    T4 x;
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = T(v[e]);
    *reinterpret_cast<T4*>(p) = x;
}

// A result with columns x (16 of them from row `row` on) and rows d, as rows of a tensor: rows of the sequence as they are, the padding behind them as zeros.
template <int DT>
__device__ __forceinline__ void store_rows(const Tensor& t, const Args& a, const Where& w, int h, int row, const f32x4 (&acc)[4], float factor) {
    using T = typename Elem<DT>::T;
    T* const to = const_cast<T*>(rows_of<DT>(t, a, w, h));
    const int r = row + lane_c();
    if (r >= (a.cu ? w.len : a.L)) return;
#pragma unroll
    for (int d = 0; d < 4; ++d)
        if (16 * d + 4 * lane_g() < a.D) store4<DT>(to + r * t.l + 16 * d + 4 * lane_g(), r < w.len ? acc[d] * factor : f32x4{0.f, 0.f, 0.f, 0.f});
}

// The wave's own rows as frags; zeros past the sequence and past D columns.
template <int DT, int NX>
__device__ __forceinline__ void load_own(typename Elem<DT>::X8 (&own)[NX][2], const Tensor& t, const Args& a, const Where& w, int h, int row) {
    const typename Elem<DT>::T* const from = rows_of<DT>(t, a, w, h);
#pragma unroll
    for (int n = 0; n < NX; ++n)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int r = row + 16 * n + lane_c(), d = 32 * k + 8 * lane_g();
            own[n][k] = r < w.len && d < a.D ? read8<DT>(from + r * t.l + d) : zero8<DT>();
        }
}

// float16: a power of two that brings the gradients of scores near the top of the type's range: they are at most 2 |dout| |v| times dropout's factor.  Other types
// hold any size: 1.
template <int DT>
__device__ __forceinline__ float score_power(const Args& a) {
    if constexpr (DT != TDB_F16) return 1.f;
    const float most = 2.f * a.factor * sqrtf(__builtin_bit_cast(float, a.largest[0])) * sqrtf(__builtin_bit_cast(float, a.largest[1]));
    if (!(most > 0.f) || !(most < __builtin_inff())) return 1.f;
    int e;
    (void)frexpf(most, &e);             // most < 2^e
    return ldexpf(1.f, min(max(15 - e, -100), 100));
}

}  // namespace tdb_train
