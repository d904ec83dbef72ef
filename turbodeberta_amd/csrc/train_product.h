// Products of the loss over a vocabulary: C[m][n] = sum over k of A(m, k) B(n, k), one tile of a workgroup at a time, float32 sums.
//
// An operand lies in memory with the contraction along its rows ("lined": [m][k]) or across them ("turned": [k][m]).  Both go from memory straight into LDS, 128 bytes
// of contraction a step for lined ones (64 values of 16 bits, 32 of float32) and as many rows for turned ones; what lies past an operand's
// end is past its buffer's end and comes as zeros.  A turned operand of 16 bits is turned by the reads from LDS.
//   * 16 bits: 32x32x16 instructions.  A frag is 32 rows x 16 of the contraction: row l % 32, 8 (l / 32) ..
//   * float32: 16x16x4 instructions.   A frag is 16 rows x 16 of the contraction: row l % 16, 4 (l / 16) ..; four instructions
// The tile's m is along the lanes of a result, four neighbouring n are in a lane ("quad").
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "tdb_internal.h"
#include "tdb_train.h"

namespace tdb_train {

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;

#define TDB_SHARED(T, p) ((__attribute__((address_space(3))) T*)(p))

template <int DT>
struct Matrix;
template <>
struct Matrix<TDB_BF16> {
    using T = __bf16;
    using Frag = bf16x8;
    using Acc = f32x16;
    static constexpr int SIDE = 32, QUADS = 4;      // rows of a frag, quads of a result
    static __device__ __forceinline__ Acc mma(Frag n, Frag m, Acc c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(n, m, c, 0, 0, 0); }
};
template <>
struct Matrix<TDB_F16> {
    using T = _Float16;
    using Frag = f16x8;
    using Acc = f32x16;
    static constexpr int SIDE = 32, QUADS = 4;
    static __device__ __forceinline__ Acc mma(Frag n, Frag m, Acc c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(n, m, c, 0, 0, 0); }
};
template <>
struct Matrix<TDB_F32> {
    using T = float;
    using Frag = f32x4;
    using Acc = f32x4;
    static constexpr int SIDE = 16, QUADS = 1;
    static __device__ __forceinline__ Acc mma(Frag n, Frag m, Acc c) {
#pragma unroll
        for (int s = 0; s < 4; ++s) c = __builtin_amdgcn_mfma_f32_16x16x4f32(n[s], m[s], c, 0, 0, 0);
        return c;
    }
};

// Which m of a result a lane has, and where its quad q starts along n.
template <int DT>
__device__ __forceinline__ int lane_m() { return threadIdx.x & (Matrix<DT>::SIDE - 1); }
template <int DT>
__device__ __forceinline__ int quad_n(int q) {
    if constexpr (DT == TDB_F32) return 4 * (threadIdx.x >> 4 & 3);
    return 8 * q + 4 * (threadIdx.x >> 5 & 1);
}
// Over the lanes that have the same m.
template <int DT, class F>
__device__ __forceinline__ float over_quads(float x, F f) {
    if constexpr (DT == TDB_F32) x = f(x, __shfl_xor(x, 16));
    return f(x, __shfl_xor(x, 32));
}

// A matrix in memory: rows `pitch` bytes apart, `width` bytes of each.
struct Rows {
    const char* p;
    int64_t pitch;
    int64_t count;
    uint32_t width;         // a multiple of 16
};

__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ void load_shared(uint32_t to, u32x4 buffer, uint32_t offset) {      // (nothing else in the kernels of this header uses m0)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(to), "v"(offset), "s"(buffer) : "memory");
}
// `bytes` from p on, at most 2 GiB
__device__ __forceinline__ u32x4 buffer_of(const char* p, int64_t bytes) {
    const uint64_t a = reinterpret_cast<uint64_t>(p);
    return u32x4{uniform(uint32_t(a)), uniform(uint32_t(a >> 32) & 0xffff), uniform(uint32_t(bytes < 0 ? 0 : bytes > 0x7fffffff ? 0x7fffffff : bytes)), 0x00020000};
}
template <int N>
__device__ __forceinline__ void wait_loads() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void step_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

constexpr uint32_t PAST = 0x80000000u;      // past every buffer's end

// One operand's share of a step: EXTENT rows of the tile (m or n), LINE bytes of each along the contraction (128 or 64).
template <int DT, int EXTENT, bool TURNED, int WAVES, int LINE>
struct Side {
    using M = Matrix<DT>;
    using T = typename M::T;
    static constexpr int ES = sizeof(T), STEP = LINE / ES, BYTES = EXTENT * LINE;
    static constexpr int LOADS = BYTES / 1024 / WAVES;                 // of 1 KB, by each wave
    static constexpr int ROW = TURNED ? EXTENT * ES : LINE, CHUNKS = ROW / 16, BLOCKS = ROW / 64;
    static_assert(LOADS * 1024 * WAVES == BYTES && (LINE == 128 || LINE == 64), "");
    uint32_t from[LOADS];       // of the lane, in the step's buffer
    uint32_t column[LOADS];     // lined: bytes into the row

    // Lined: 16-byte chunk c of row r lies at c ^ swap(r), so that the 16 rows that LDS serves together (0..3, 12..15, 20..27 and the others) are on distinct banks.  Turned: 64-byte block b
    // of row k lies at b ^ turn(k), so that the four rows that a read of 16 bits takes together, or every fourth of float32, are.
    static __device__ __forceinline__ int swap(int r) { return LINE == 128 ? r >> 1 & 7 : r >> 2 & 3; }
    static __device__ __forceinline__ int turn(int k) { return (DT == TDB_F32 ? k >> 2 & 3 : (k & 3) | (k >> 1 & 4)) & (BLOCKS - 1); }

    // Tile of rows (lined) or columns (turned) first ..
    __device__ __forceinline__ void place(const Rows& a, int64_t first) {
        const int wave = threadIdx.x >> 6, l = threadIdx.x & 63;
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
            const int at = (wave * LOADS + j) * 64 + l, row = at / CHUNKS, chunk = at % CHUNKS;
            if constexpr (TURNED) {
                const uint32_t c = ((((chunk >> 2) ^ turn(row)) << 2) | (chunk & 3)) * 16;
                from[j] = c + uint32_t(first) * ES < a.width ? uint32_t(row) * uint32_t(a.pitch) + c : PAST;
            } else {
                column[j] = (chunk ^ swap(row)) * 16;
                from[j] = uint32_t(row) * uint32_t(a.pitch) + column[j];
            }
        }
    }
    // Step s of the contraction into LDS.
    __device__ __forceinline__ void load(const Rows& a, int64_t first, int64_t s, uint32_t lds) const {
        const uint32_t to = lds + uniform(threadIdx.x >> 6) * (LOADS * 1024);
        if constexpr (TURNED) {
            const int64_t k = s * STEP;
            const char* p = a.p + k * a.pitch + first * ES;
            const u32x4 buffer = buffer_of(p, (a.count - 1 - k) * a.pitch + a.width - first * ES);
#pragma unroll
            for (int j = 0; j < LOADS; ++j) load_shared(to + j * 1024, buffer, from[j]);
        } else {
            const int64_t into = s * LINE;
            const u32x4 buffer = buffer_of(a.p + first * a.pitch + into, (a.count - 1 - first) * a.pitch + a.width - into);
            const bool whole = into + LINE <= a.width;
#pragma unroll
            for (int j = 0; j < LOADS; ++j) load_shared(to + j * 1024, buffer, whole || into + column[j] < a.width ? from[j] : PAST);
        }
    }
    // Frag of rows row .. (a multiple of SIDE), part kk of the step (32 bytes, or 64 of float32)
    __device__ __forceinline__ typename M::Frag frag(const char* lds, int row, int kk) const {
        const int l = threadIdx.x & 63;
        if constexpr (!TURNED) {
            const int r = row + lane_m<DT>(), chunk = DT == TDB_F32 ? 4 * kk + (l >> 4) : 2 * kk + (l >> 5);
            return *reinterpret_cast<const typename M::Frag*>(lds + r * LINE + ((chunk ^ swap(r)) << 4));
        } else if constexpr (DT == TDB_F32) {
            f32x4 x;
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const int k = 16 * kk + 4 * (l >> 4) + s;
                x[s] = *reinterpret_cast<const float*>(lds + k * ROW + (((row >> 4) ^ turn(k)) << 6) + 4 * (l & 15));
            }
            return x;
        } else {
            const int k = 16 * kk + 8 * (l >> 5) + (l >> 2 & 3);
            const char* at = lds + k * ROW + (((row >> 5) ^ turn(k)) << 6) + 32 * (l >> 4 & 1) + 8 * (l & 3);       // (turn(k + 4) = turn(k))
            const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16(TDB_SHARED(s16x4, at));
            const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16(TDB_SHARED(s16x4, at + 4 * ROW));
            return __builtin_bit_cast(typename M::Frag, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
        }
    }
};

// BM x BN by WM x WN waves, NS stages in LDS.
template <int DT, int BM_, int BN_, int WM_, int WN_, int NS, bool TURN_A, bool TURN_B, int LINE = 128>
struct Product {
    static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, LINE_BYTES = LINE;
    using M = Matrix<DT>;
    using T = typename M::T;
    static constexpr int WAVES = WM * WN, TM = BM / WM / M::SIDE, TN = BN / WN / M::SIDE, PARTS = LINE / (DT == TDB_F32 ? 64 : 32);
    using A = Side<DT, BM, TURN_A, WAVES, LINE>;
    using B = Side<DT, BN, TURN_B, WAVES, LINE>;
    static constexpr int STEP = A::STEP, STAGE = A::BYTES + B::BYTES, SHARED = NS * STAGE;
    using Acc = typename M::Acc[TM][TN];

    static __device__ __forceinline__ int wave_m() { return int(uniform(threadIdx.x >> 6)) / WN * (BM / WM); }
    static __device__ __forceinline__ int wave_n() { return int(uniform(threadIdx.x >> 6)) % WN * (BN / WN); }

    // Steps [begin, end) of the tile at rows m0 of A and n0 of B.  The sums start from start(j, q), four neighbours along n, called behind the first step's barrier.
    template <class START>
    static __device__ __forceinline__ void run(char* smem, const Rows& a, const Rows& b, int64_t m0, int64_t n0, int64_t begin, int64_t end, Acc& acc, START start) {
        constexpr int LOADS = A::LOADS + B::LOADS;
        A side_a;
        B side_b;
        side_a.place(a, m0), side_b.place(b, n0);
        const uint32_t lds = uniform(uint32_t(reinterpret_cast<uintptr_t>(TDB_SHARED(char, smem))));
        auto load = [&](int64_t s, int stage) {
            side_a.load(a, m0, s, lds + stage * STAGE);
            side_b.load(b, n0, s, lds + stage * STAGE + A::BYTES);
        };
        const int steps = int(end - begin);
        step_barrier();                     // nobody has use for what LDS held
#pragma unroll
        for (int s = 0; s < NS - 1; ++s)
            if (s < steps) load(begin + s, s);
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int q = 0; q < M::QUADS; ++q) {
                const f32x4 v = start(j, q);
#pragma unroll
                for (int i = 0; i < TM; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[i][j][4 * q + e] = v[e];
            }
        int stage = 0, ahead = NS - 1;
        for (int s = 0; s < steps; ++s) {
            if (s + NS - 2 < steps) wait_loads<(NS - 2) * LOADS>();
            else wait_loads<0>();
            step_barrier();                 // this stage is there, and nobody reads the one before it any more
            if (s + NS - 1 < steps) load(begin + s + NS - 1, ahead);
            const char* at = smem + stage * STAGE;
#pragma unroll
            for (int kk = 0; kk < PARTS; ++kk) {
                typename M::Frag fa[TM], fb[TN];
#pragma unroll
                for (int i = 0; i < TM; ++i) fa[i] = side_a.frag(at, wave_m() + i * M::SIDE, kk);
#pragma unroll
                for (int j = 0; j < TN; ++j) fb[j] = side_b.frag(at + A::BYTES, wave_n() + j * M::SIDE, kk);
#pragma unroll
                for (int i = 0; i < TM; ++i)
#pragma unroll
                    for (int j = 0; j < TN; ++j) acc[i][j] = M::mma(fb[j], fa[i], acc[i][j]);
            }
            stage = stage == NS - 1 ? 0 : stage + 1;
            ahead = ahead == NS - 1 ? 0 : ahead + 1;
        }
        step_barrier();                     // LDS is free for what follows
    }
    static __device__ __forceinline__ void run(char* smem, const Rows& a, const Rows& b, int64_t m0, int64_t n0, int64_t begin, int64_t end, Acc& acc) {
        run(smem, a, b, m0, n0, begin, end, acc, [](int, int) { return f32x4{0.f, 0.f, 0.f, 0.f}; });
    }

    // The tile's values to rows of memory by way of LDS, SIDE rows at a time: value(i, j, q) gives four neighbours, then(i, the wave's rows in LDS) may change what lies there.
    // to: value (m0, n0); rows and columns: how many of the tile's there are.  Whole 16-byte chunks where `wide`.
    static constexpr int COLUMNS = TN * M::SIDE, PITCH = COLUMNS * int(sizeof(T)) + 16;
    template <class OF, class THEN>
    static __device__ __forceinline__ void store(char* smem, char* to, int64_t pitch, int64_t rows, int64_t columns, bool wide, OF value, THEN then) {
        constexpr int ES = sizeof(T), PER = COLUMNS * ES / 16;
        typedef __attribute__((ext_vector_type(4))) T T4;
        const int l = threadIdx.x & 63;
        char* const own = smem + uniform(threadIdx.x >> 6) * (2 * M::SIDE * PITCH);
        static_assert(WAVES * 2 * M::SIDE * PITCH <= SHARED, "");
        to += wave_m() * pitch + wave_n() * ES, rows -= wave_m(), columns -= wave_n();
#pragma unroll
        for (int i = 0; i < TM; ++i) {
            char* const mine = own + (i & 1) * (M::SIDE * PITCH);
#pragma unroll
            for (int j = 0; j < TN; ++j)
#pragma unroll
                for (int q = 0; q < M::QUADS; ++q) {
                    const f32x4 v = value(i, j, q);
                    *reinterpret_cast<T4*>(mine + lane_m<DT>() * PITCH + (j * M::SIDE + quad_n<DT>(q)) * ES) = T4{T(v[0]), T(v[1]), T(v[2]), T(v[3])};
                }
            then(i, mine);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            if (wide) {
                const auto buffer = __builtin_amdgcn_make_buffer_rsrc(to + i * M::SIDE * pitch, 0, int(rows > i * M::SIDE && columns > 0 ? min((rows - 1 - i * M::SIDE) * pitch + columns * ES, int64_t(0x7fffffff)) : 0), 0x00020000);
#pragma unroll
                for (int r = 0; r < M::SIDE * PER / 64; ++r) {
                    const int at = r * 64 + l, row = at / PER, c = at % PER;
                    const u32x4 v = *reinterpret_cast<const u32x4*>(mine + row * PITCH + c * 16);
                    __builtin_amdgcn_raw_buffer_store_b128(v, buffer, c * 16 < columns * ES ? uint32_t(row) * uint32_t(pitch) + c * 16 : PAST, 0, 0);
                }
            } else {
                for (int at = l; at < M::SIDE * COLUMNS; at += 64) {
                    const int row = at / COLUMNS, c = at % COLUMNS;
                    if (i * M::SIDE + row < rows && c < columns) *reinterpret_cast<T*>(to + (i * M::SIDE + row) * pitch + c * ES) = *reinterpret_cast<const T*>(mine + row * PITCH + c * ES);
                }
            }
        }
    }
    // Four neighbours of the sums.
    static __device__ __forceinline__ f32x4 quad(const Acc& acc, int i, int j, int q) {
        if constexpr (DT == TDB_F32) return acc[i][j];
        else return f32x4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
    }
};

// Sums of a lane's N values over the lanes that have the same n.  Each step halves the values: a lane passes on one half and keeps the other.  Value number
// (lane's m) mod N is the lane's in the end.
template <int DT, int N>
__device__ __forceinline__ float over_m(float (&x)[N]) {
    constexpr int SIDE = Matrix<DT>::SIDE;
    static_assert(N <= SIDE && (N & (N - 1)) == 0, "");
#pragma unroll
    for (int w = N / 2; w >= 1; w /= 2) {
        const bool high = threadIdx.x & w;
#pragma unroll
        for (int k = 0; k < w; ++k) {
            const float a = x[k], b = x[k + w], pass = high ? a : b, keep = high ? b : a;     // (not high ? x[k] : x[k + w], which chooses an address)
            x[k] = keep + __shfl_xor(pass, w);
        }
    }
    float sum = x[0];
#pragma unroll
    for (int w = N; w < SIDE; w *= 2) sum += __shfl_xor(sum, w);
    return sum;
}

// Tile number `block` of `rows` x `columns` tiles.  Workgroups start in turn on the 8 XCDs: blocks of one (equal mod 8) take neighbouring tiles, eight rows of tiles at a time.
__device__ __forceinline__ void tile_of(int64_t block, int64_t rows, int64_t columns, int64_t splits, int64_t& row, int64_t& column, int64_t& split) {
    const int64_t tiles = rows * columns, all = tiles * splits, part = all >> 3, more = all & 7, xcd = block & 7;
    int64_t b = xcd * part + min(xcd, more) + (block >> 3);
    split = b / tiles;
    b -= split * tiles;
    const int64_t group = b / (8 * columns), in = b - group * 8 * columns, high = min(int64_t(8), rows - 8 * group);
    column = in / high;
    row = group * 8 + in - column * high;
}

}  // namespace tdb_train
