// Parts of the attention kernels for training: tiles in LDS, operands of the matrix instructions, scores with their position terms.
//
// Types.  A "frag" is what a lane has of an operand of 16 rows x 32 columns of the contraction: 8 values of row (or column) c = lane & 15, columns
// 8 g .. 8 g + 7, g = lane >> 4.  In 16 bits that is one matrix instruction (16x16x32), in float32 eight (16x16x4: step s contracts column
// 8 g + s of lane group g; the order of a sum is free as long as both operands have it).  A result has row 4 g + e (e = 0..3), column c in a lane.
//
// Layout of scores.  A wave owns 16 rows x (a lane has one) and runs over the other side's rows y, 64 a step: S[y][x], y in the
// result's rows.  Forward x are queries and y keys, so a softmax row is in a lane and the three others of its column, and the probabilities are an operand
// of the next product as they stand.  Backward x are keys and y queries: the same for the gradients of keys and values.
//
// Position terms.  Both are functions of x - y (r = x - y + 63 in a tile), with the table of x's side ("own") and of y's ("other"):
//   own:   x . T_own[r]    computed for the 80 r that 16 x and 64 y have, result columns x: stored to LDS as rows x, index y + 16 - x, a row of
//          85 floats: x * 85 + 16 - x + y is a multiple of 4 for every y that is one, so four y at once are one read of 16 bytes, and 84 x for
//          16 x are on distinct banks.
//   other: y . T_other[r]  for the 32 r of 16 y and 16 x, result columns y: stored as rows y, read back value by value, lanes along x.
// They are held in float32.  The tables' rows lie in LDS as rings in the order of r; 64 rows are new in each step.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "philox.h"
#include "tdb_error.h"
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
constexpr float LOG2E = 1.44269504088896340736f;

// Rows of 64 values in LDS.  float32: 16 bytes apart.  16 bits: side by side, so that two workgroups fit a CU, their 16-byte chunks permuted.  LDS serves a read of 16 bytes a
// lane in 4 clocks if each time these 16 lanes are on distinct banks, in 8 if not (measured): rows 0 .. 3 and 12 .. 15 at one chunk with rows 4 .. 11 at the next.  A
// transposing read has 32 bytes of rows 0 .. 7, or of 0 .. 3 and 8 .. 11.  This permutation serves all of them.
template <int DT>
constexpr int ROW = DT == TDB_F32 ? 68 : 64;
template <int DT>
__device__ __forceinline__ int place(int row, int col) {
    if constexpr (DT == TDB_F32) return row * ROW<DT> + col;
    return row * ROW<DT> + (col ^ (((row & 6) ^ (row & 8 ? 5 : 0)) << 3));
}

__device__ __forceinline__ int lane_c() { return threadIdx.x & 15; }
__device__ __forceinline__ int lane_g() { return threadIdx.x >> 4 & 3; }

// Between writes and reads of a wave's own part of LDS: the hardware keeps their order, the compiler is told to.
__device__ __forceinline__ void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
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

// What is written ahead of it stays ahead.  16 bits: operands are asked for well ahead of their products (left alone, the compiler fetches them two by two, and every
// product waits for LDS).  float32 has no registers for that.
template <int DT>
__device__ __forceinline__ void ahead() {
    if constexpr (DT != TDB_F32) __builtin_amdgcn_sched_barrier(0);
}

// Frag of rows `row` + c, columns k0 + 8 g ..; row a multiple of 16
template <int DT>
__device__ __forceinline__ typename Elem<DT>::X8 row_frag(const typename Elem<DT>::T* rows, int row, int k0) {
    return read8<DT>(rows + row * ROW<DT> + place<DT>(lane_c(), k0 + 8 * lane_g()));
}

// Transposed frags: the lane's row of the operand is column col + c in LDS, the contraction runs over rows in LDS.  Each lane gives the address of four columns of
// one row; the hardware hands the lanes of a group their columns.  `lo` and `hi`: first of the four rows of the lane group's two halves, multiples of 4.  AT: where a value lies.
template <int DT, typename AT>
__device__ __forceinline__ typename Elem<DT>::X8 turned_frag(const typename Elem<DT>::T* rows, int lo, int hi, int col, AT at) {
    if constexpr (DT == TDB_F32) {
        f32x8 x;
#pragma unroll
        for (int s = 0; s < 4; ++s) x[s] = rows[at(lo + s, col + lane_c())], x[4 + s] = rows[at(hi + s, col + lane_c())];
        return x;
    } else {
        const int r = lane_c() >> 2, c = col + 4 * (lane_c() & 3);
        const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16(TDB_SHARED(s16x4, rows + at(lo + r, c)));
        const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16(TDB_SHARED(s16x4, rows + at(hi + r, c)));
        return __builtin_bit_cast(typename Elem<DT>::X8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
    }
}
// Over rows k0 + 8 g + s
template <int DT>
__device__ __forceinline__ typename Elem<DT>::X8 line_frag(const typename Elem<DT>::T* rows, int k0, int col) {
    return turned_frag<DT>(rows + k0 * ROW<DT>, 8 * lane_g(), 8 * lane_g() + 4, col, place<DT>);
}
// Over rows k0 + 4 g + s and k0 + 16 + 4 g + s, the order in which two results of 16 rows are an operand
template <int DT>
__device__ __forceinline__ typename Elem<DT>::X8 pair_frag(const typename Elem<DT>::T* rows, int k0, int col) {
    return turned_frag<DT>(rows + k0 * ROW<DT>, 4 * lane_g(), 16 + 4 * lane_g(), col, place<DT>);
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
    void* rest;                         // 16 bits: what rounding took from o
    int32_t* starts;                    // of table rows: the first offset whose row is this one or a later one
    void* ds;                           // [heads][tiles of rows][tiles][64 x 64]
    float *partial, *level_parts, *row_sums;
    int32_t* level;                     // the first and the last diagonal of tiles whose offsets all have the last, the first row
    int32_t tiles, row_tiles;           // of the longest sequence; of all sequences
    int32_t split_bits, seg_bits;       // parts of the longest diagonal: of the sequences, of each sequence
    int32_t per_tile;                   // 65536 / tiles, rounded up
    void *dpk, *dpq;                    // [H, table rows, D]
    int64_t dpk_h, dpq_h;
    const int64_t* seed;
    uint32_t threshold;
    float factor, scale;
    int32_t p_shift;                    // float16: probabilities are multiplied by 2^p_shift where they are rounded
    uint32_t* largest;                  // float16, [heads, sequences, 2]: squares of the largest norms of a row of dout and of v
};

struct Where {
    int b, row0, len;       // sequence, first row of the tile, valid rows of the sequence
    int64_t first;          // row of the packed tensors (else 0)
    int64_t line;           // of lse and delta
    int64_t row_tile;       // number of the sequence's first row tile among all sequences'
    int block;              // number of this tile, in the workspace too
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
    w.block = block;
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

// Loads go through buffer resources: what lies beyond the resource's end reads as zeros, so rows past a sequence and columns past D need no code of their own.
constexpr uint32_t NOWHERE = 0x80000000u;       // an offset past every end
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer(const void* p, int64_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, int(min(max(bytes, int64_t(0)), int64_t(0x7fffffff))), 0x00020000);
}

// A tile of 64 rows of 64 values on its way from global memory to LDS, 16 bytes a lane at a time, by `threads` threads.
template <int DT, int threads>
struct Stage {
    using T = typename Elem<DT>::T;
    static constexpr int PIECES = DT == TDB_F32 ? 16 : 8, EACH = 64 / PIECES, STEP = threads / PIECES, LOADS = TILE * PIECES / threads;
    u32x4 x[LOADS];
    static __device__ __forceinline__ int row(int n) { return threadIdx.x / PIECES + n * STEP; }
    static __device__ __forceinline__ int col() { return threadIdx.x % PIECES * EACH; }
    // of a lane's pieces, in bytes, where rows are `stride` bytes apart
    static __device__ __forceinline__ void offsets(uint32_t (&at)[LOADS], uint32_t stride, int D) {
#pragma unroll
        for (int n = 0; n < LOADS; ++n) at[n] = col() < D ? row(n) * stride + col() * sizeof(T) : NOWHERE;
    }
    __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t from, const uint32_t (&at)[LOADS]) {
#pragma unroll
        for (int n = 0; n < LOADS; ++n) x[n] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(from, int(at[n]), 0, 0));
    }
    __device__ __forceinline__ void store(T* rows) const {
#pragma unroll
        for (int n = 0; n < LOADS; ++n) *reinterpret_cast<u32x4*>(rows + place<DT>(row(n), col())) = x[n];
    }
};

// Rows of one head of one sequence, 64 at a time in order.
template <int DT, int threads>
struct Source {
    using S = Stage<DT, threads>;
    const char* next;
    uint32_t stride;                    // bytes, at most 2^24
    int left;                           // rows
    uint32_t at[S::LOADS];
    __device__ __forceinline__ Source(const Tensor& t, const Args& a, const Where& w, int h, int row = 0) {
        stride = uint32_t(t.l) * sizeof(typename S::T), left = w.len - row;
        next = reinterpret_cast<const char*>(rows_of<DT>(t, a, w, h)) + int64_t(row) * stride;
        S::offsets(at, stride, a.D);
    }
    __device__ __forceinline__ void load(S& s) {
        s.load(__builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(next), 0, int(min(left, TILE) * stride), 0x00020000), at);
        next += int64_t(TILE) * stride, left -= TILE;
    }
};

// Both tables' rows for 64 neighbouring r of a tile.  SIGN: 1 where x are queries (the relative position is x - y), -1 where they are keys.
template <int DT, int SIGN, int threads, bool PK, bool PQ>
struct Tables {
    using S = Stage<DT, threads>;
    using T = typename S::T;
    __amdgpu_buffer_rsrc_t lut, pk, pq;
    uint32_t pk_stride, pq_stride, lane;        // bytes; of the lane's column (past every end where there is none: what is added is below 2^31)
    int at, last;                               // the lane's place in the lookup table for x0 = y0 and r0 = 0, and its last one, in bytes
    S k, q;
    int which[S::LOADS], ends[2];
    int most, half;                             // the largest relative position, and its place
    __device__ __forceinline__ Tables(const Args& a, int h) {
        most = a.L - 1, half = a.lut_half, ends[0] = 0, ends[1] = 1;
        lut = buffer(a.lut, (2 * int64_t(a.lut_half) + 1) * 4);
        if constexpr (PK) pk = buffer(static_cast<const T*>(a.pk.p) + h * a.pk.h, 2 * int64_t(a.span) * a.pk.l * sizeof(T));
        if constexpr (PQ) pq = buffer(static_cast<const T*>(a.pq.p) + h * a.pq.h, 2 * int64_t(a.span) * a.pq.l * sizeof(T));
        pk_stride = uint32_t(a.pk.l) * sizeof(T), pq_stride = uint32_t(a.pq.l) * sizeof(T);
        lane = S::col() < a.D ? S::col() * sizeof(T) : NOWHERE;
        at = (SIGN * (S::row(0) - 63) + a.lut_half) * 4, last = 8 * a.lut_half;
    }
    // looks up the rows of r0 .. r0 + 63; `from`: x0 - y0 of the tile
    __device__ __forceinline__ void look(int r0, int from) {
        if constexpr (PK || PQ) {
#pragma unroll
            for (int n = 0; n < S::LOADS; ++n)
                which[n] = int(__builtin_amdgcn_raw_buffer_load_b32(lut, min(max(at + 4 * SIGN * (r0 + from + n * S::STEP), 0), last), 0, 0));
        }
    }
    // looks up the rows of the first and the last relative position of a tile of 64 x 64
    __device__ __forceinline__ void look_at_ends(int from) {
        if constexpr (PK || PQ) {
#pragma unroll
            for (int n = 0; n < 2; ++n)
                ends[n] = int(__builtin_amdgcn_raw_buffer_load_b32(lut, (min(max(SIGN * from + (n ? 63 : -63), -most), most) + half) * 4, 0, 0));
        }
    }
    // whether they are one row
    __device__ __forceinline__ bool far() const { return (PK || PQ) && __builtin_amdgcn_readfirstlane(ends[0]) == __builtin_amdgcn_readfirstlane(ends[1]); }
    // fetches the rows looked up last
    __device__ __forceinline__ void load() {
        auto one = [&](S& s, __amdgpu_buffer_rsrc_t from, uint32_t stride) {
            uint32_t to[S::LOADS];
#pragma unroll
            for (int n = 0; n < S::LOADS; ++n) to[n] = uint32_t(which[n]) * stride + lane;
            s.load(from, to);
        };
        if constexpr (PK) one(k, pk, pk_stride);
        if constexpr (PQ) one(q, pq, pq_stride);
    }
    __device__ __forceinline__ void store(T* pk_ring, T* pq_ring, int to) const {
        if constexpr (PK) k.store(pk_ring + to * ROW<DT>);
        if constexpr (PQ) q.store(pq_ring + to * ROW<DT>);
    }
    // fills the second half of the rings for a first step with x0 - y0 = from; the rows of r = 0 .. 63 are those looked up last
    __device__ __forceinline__ void fill(T* pk_ring, T* pq_ring, int from) {
        if constexpr (PK || PQ) {
            look_at_ends(from);
            look(0, from);
            int first[S::LOADS];
#pragma unroll
            for (int i = 0; i < S::LOADS; ++i) first[i] = which[i];
            look(64, from);
            load();
            store(pk_ring, pq_ring, 64);
#pragma unroll
            for (int i = 0; i < S::LOADS; ++i) which[i] = first[i];
        }
    }
};

// Whether all relative positions first .. last that occur have one table row.
__device__ __forceinline__ bool one_row(const Args& a, int first, int last) {
    const int lo = min(max(first, 1 - a.L), a.L - 1), hi = min(max(last, 1 - a.L), a.L - 1);
    return a.lut[lo + a.lut_half] == a.lut[hi + a.lut_half];
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

// Floats of a row of x's term, of which 88 (22 chunks of 16 bytes) are next to the one before in what is read: reads of 16 bytes a lane, and writes of one value a lane, are on
// distinct banks.  And of y's term, two blocks of 16 rows in the same place: 43 apart in what is read, four times that is 44 banks on.
constexpr int OWN_ROW = 89, OTHER_ROW = 44;
static_assert(2 * OTHER_ROW <= OWN_ROW, "");
template <int DT>
constexpr int TERMS = DT == TDB_F32 ? 1552 : 16 * OWN_ROW;      // floats of a wave's scratch for the two, in turn, and for a skewed tile

// A table's rows r = 0 .. 126 of a tile of 64 x and 64 y, and one more.
constexpr int RING = 128;
__device__ __forceinline__ int wrapped(int at) { return at & (RING - 1); }

// A row as both operands' frags: the same for every row or column.
template <int DT>
__device__ __forceinline__ typename Elem<DT>::X8 same_frag(const typename Elem<DT>::T* rows, int row, int k0) {
    return read8<DT>(rows + place<DT>(row, k0 + 8 * lane_g()));
}
// And as an operand whose row is column col + c and which is the same all along the contraction.
template <int DT>
__device__ __forceinline__ typename Elem<DT>::X8 level_frag(const typename Elem<DT>::T* rows, int row, int col) {
    const typename Elem<DT>::T v = rows[place<DT>(row, col + lane_c())];
    typename Elem<DT>::X8 x;
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = v;
    return x;
}
// Over the ring's rows r0 + 8 g + s
template <int DT>
__device__ __forceinline__ typename Elem<DT>::X8 ring_frag(const typename Elem<DT>::T* rows, int r0, int col) {
    const int at = wrapped(r0 + 8 * lane_g());
    return turned_frag<DT>(rows, at, at + 4, col, place<DT>);
}

// Four results behind the wait states of their products, on every path (see tdb_settled).
__device__ __forceinline__ void settle(f32x4 (&s)[4]) { asm volatile("s_nop 7\n\ts_nop 7" : "+v"(s[0]), "+v"(s[1]), "+v"(s[2]), "+v"(s[3])); }

// Scores of the wave's 16 rows x (x block `first`) with a step's 64 rows y, without the scale.  own[k]: frags of x.  Rings whose row for r is (r + base) mod RING, base a
// multiple of 64.  scratch: the wave's own, TERMS floats.  far: the step's relative positions have one table row, so the terms are one number for each x and one for
// each y.
template <int DT, bool OWN, bool OTHER>
__device__ __forceinline__ void scores(f32x4 (&s)[4], const typename Elem<DT>::X8 (&own)[2], const typename Elem<DT>::T* y_rows, const typename Elem<DT>::T* own_ring,
                                       const typename Elem<DT>::T* other_ring, int base, int first, float* scratch, bool far) {
    using E = Elem<DT>;
    using X8 = typename E::X8;
    const int c = lane_c(), g = lane_g();
    const f32x4 none = {0.f, 0.f, 0.f, 0.f};
    const int mid = wrapped(63 + base);
    if ((OWN || OTHER) && far) {
        f32x4 w = none;
        if constexpr (OWN) w = E::mma(same_frag<DT>(own_ring, mid, 32), own[1], E::mma(same_frag<DT>(own_ring, mid, 0), own[0], none));
        X8 t0, t1;
        if constexpr (OTHER) t0 = same_frag<DT>(other_ring, mid, 0), t1 = same_frag<DT>(other_ring, mid, 32);
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            const X8 y0 = row_frag<DT>(y_rows, 16 * m, 0), y1 = row_frag<DT>(y_rows, 16 * m, 32);
            s[m] = E::mma(y1, own[1], E::mma(y0, own[0], w));
            if constexpr (OTHER) s[m] = E::mma(y1, t1, E::mma(y0, t0, s[m]));
        }
        settle(s);
        return;
    }
    X8 t[5][2], y[4][2];
    if constexpr (OWN) {
#pragma unroll
        for (int n = 0; n < 5; ++n)             // r = 16 (first + n) + 15 - row of the frag
#pragma unroll
            for (int k = 0; k < 2; ++k) t[n][k] = read8<DT>(own_ring + wrapped(16 * (first + n) + base) * ROW<DT> + place<DT>(15 - c, 32 * k + 8 * g));
    }
#pragma unroll
    for (int m = 0; m < 4; ++m)
#pragma unroll
        for (int k = 0; k < 2; ++k) y[m][k] = row_frag<DT>(y_rows, 16 * m, 32 * k);
    ahead<DT>();
    f32x4 w[OTHER ? 4 : 1][2];
    if constexpr (OWN) {
        f32x4 x[5];
#pragma unroll
        for (int n = 0; n < 5; ++n) x[n] = E::mma(t[n][0], own[0], none);
#pragma unroll
        for (int n = 0; n < 5; ++n) x[n] = E::mma(t[n][1], own[1], x[n]);
#pragma unroll
        for (int n = 0; n < 5; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) scratch[c * OWN_ROW + 64 - 16 * n + 4 * g + e] = x[n][e];
    }
    if constexpr (OTHER) {
#pragma unroll
        for (int n = 0; n < 5; ++n)             // r = 16 (first + n) + row: of y blocks 3 - n and 4 - n
#pragma unroll
            for (int k = 0; k < 2; ++k) t[n][k] = row_frag<DT>(other_ring, wrapped(16 * (first + n) + base), 32 * k);
    }
    wave_fence();
#pragma unroll
    for (int m = 0; m < 4; ++m) {
        if constexpr (OWN) s[m] = *reinterpret_cast<const f32x4*>(scratch + c * (OWN_ROW - 1) + 16 + 16 * m + 4 * g);
        else s[m] = none;
    }
    ahead<DT>();
    if constexpr (OTHER) {
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int m = 0; m < 4; ++m)
#pragma unroll
                for (int n = 0; n < 2; ++n) w[m][n] = E::mma(t[3 - m + n][k], y[m][k], k == 0 ? none : w[m][n]);
    }
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int m = 0; m < 4; ++m) s[m] = E::mma(y[m][k], own[k], s[m]);
    if constexpr (OTHER) {                      // two y blocks at once, where x's term was, which has been read
        wave_fence();
#pragma unroll
        for (int two = 0; two < 4; two += 2) {
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int n = 0; n < 2; ++n) *reinterpret_cast<f32x4*>(scratch + (16 * m + c) * OTHER_ROW + 16 * n + 4 * g) = w[two + m][n];
            wave_fence();
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[two + m][e] += scratch[(16 * m + 4 * g + e) * OTHER_ROW + c + 15 - 4 * g - e];
            wave_fence();
        }
    } else {
        settle(s);
    }
    wave_fence();
}

// 16 rows of a tensor from `row` on, of which `rows` are there; offsets of a lane's row c and column d.
template <int DT>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows16(const Tensor& t, const Args& a, const Where& w, int h, int row, int rows) {
    const int stride = int(t.l) * int(sizeof(typename Elem<DT>::T));
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<typename Elem<DT>::T*>(rows_of<DT>(t, a, w, h)) + row * t.l, 0, min(max(rows - row, 0), 16) * stride, 0x00020000);
}
template <int DT>
__device__ __forceinline__ uint32_t offset16(const Tensor& t, const Args& a, int d) {
    return d < a.D ? (uint32_t(lane_c()) * uint32_t(t.l) + d) * sizeof(typename Elem<DT>::T) : NOWHERE;
}

// A result with columns x (16 of them from row `row` on) and rows d, as rows of a tensor: rows of the sequence as they are, the padding behind them as zeros.
template <int DT>
__device__ __forceinline__ void store_rows(const Tensor& t, const Args& a, const Where& w, int h, int row, const f32x4 (&acc)[4], float factor) {
    using T = typename Elem<DT>::T;
    typedef __attribute__((ext_vector_type(4))) T T4;
    typedef __attribute__((ext_vector_type(2))) uint32_t u32x2;
    const __amdgpu_buffer_rsrc_t to = rows16<DT>(t, a, w, h, row, a.cu ? w.len : a.L);
    const bool there = row + lane_c() < w.len;
#pragma unroll
    for (int d = 0; d < 4; ++d) {
        T4 x;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = T(there ? acc[d][e] * factor : 0.f);
        const int at = int(offset16<DT>(t, a, 16 * d + 4 * lane_g()));
        if constexpr (DT == TDB_F32) __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, x), to, at, 0, 0);
        else __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, x), to, at, 0, 0);
    }
}

// What rounding takes from those results, [heads, rows, D] of the type, back to back.  The sum D = dO . O of a row stands against every score's gradient of the row, the same
// error in all of them: with O as it is stored the gradients of long rows lose more to it than to their own roundings.
template <int DT>
__device__ __forceinline__ void store_rest(void* rest, const Args& a, const Where& w, int h, int row, const f32x4 (&acc)[4], float factor) {
    using T = typename Elem<DT>::T;
    typedef __attribute__((ext_vector_type(4))) T T4;
    typedef __attribute__((ext_vector_type(2))) uint32_t u32x2;
    const int stride = a.D * int(sizeof(T));
    const __amdgpu_buffer_rsrc_t to = buffer(static_cast<char*>(rest) + (h * a.lines + w.line + row) * stride, rest ? min(w.len - row, 16) * stride : 0);
#pragma unroll
    for (int d = 0; d < 4; ++d) {
        T4 x;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = T(acc[d][e] * factor - float(T(acc[d][e] * factor)));
        const int col = 16 * d + 4 * lane_g();
        __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, x), to, col < a.D ? lane_c() * stride + col * int(sizeof(T)) : int(NOWHERE), 0, 0);
    }
}

// The wave's own rows as frags; zeros past the sequence and past D columns.
template <int DT>
__device__ __forceinline__ void load_own(typename Elem<DT>::X8 (&own)[2], const Tensor& t, const Args& a, const Where& w, int h, int row) {
    const __amdgpu_buffer_rsrc_t from = rows16<DT>(t, a, w, h, row, w.len);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int at = int(offset16<DT>(t, a, 32 * k + 8 * lane_g()));
        const u32x4 lo = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(from, at, 0, 0));
        if constexpr (DT == TDB_F32) {
            const u32x4 hi = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(from, at, 16, 0));
            own[k] = __builtin_bit_cast(f32x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        } else {
            own[k] = __builtin_bit_cast(typename Elem<DT>::X8, lo);
        }
    }
}

// float16: a power of two that brings the gradients of a sequence's and head's scores, which are kept without dropout's factor, near the top of the type's range: they are at most
// 2 |dout| |v|.  2^40 at most (from 2^-24 for the type's largest rows on): sums of several sequences are scaled from one's power to the next one's.  Other types hold any size: 1.
template <int DT>
__device__ __forceinline__ float score_power(const Args& a, int h, int b) {
    if constexpr (DT != TDB_F16) return 1.f;
    const uint32_t* const of = a.largest + (int64_t(h) * a.B + b) * 2;
    const float most = 2.f * sqrtf(__builtin_bit_cast(float, of[0])) * sqrtf(__builtin_bit_cast(float, of[1]));
    if (!(most > 0.f) || !(most < __builtin_inff())) return 1.f;
    int e;
    (void)frexpf(most, &e);             // most < 2^e
    return ldexpf(1.f, min(15 - e, 40));
}

}  // namespace tdb_train
