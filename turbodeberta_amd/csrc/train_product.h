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

#include <type_traits>

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
    const char* p;          // at a multiple of 4 bytes, as is pitch
    int64_t pitch;
    int64_t count;
    uint32_t width;
};

__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ void load_shared(uint32_t to, u32x4 buffer, uint32_t offset) {      // (nothing else in the kernels of this header uses m0)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(to), "v"(offset), "s"(buffer) : "memory");
}
// `bytes` from p on, at most 2 GiB; an odd 16-bit value at their end has its four bytes read
__device__ __forceinline__ u32x4 buffer_of(const char* p, int64_t bytes) {
    const uint64_t a = reinterpret_cast<uint64_t>(p);
    return u32x4{uniform(uint32_t(a)), uniform(uint32_t(a >> 32) & 0xffff), uniform(uint32_t(bytes < 0 ? 0 : bytes > 0x7ffffffc ? 0x7ffffffc : bytes + 3 & ~3)), 0x00020000};
}
template <int N>
__device__ __forceinline__ void wait_loads() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// Behind the last products of a tile: all wait states that one of them may need (12; 16 of them), on every path.  Paths join here, and the compiler follows one of them back to the products (see tdb_settled).
__device__ __forceinline__ void settle() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_nop 7\n\ts_nop 7" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}
__device__ __forceinline__ void step_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

constexpr uint32_t PAST = 0x80000000u;      // past every buffer's end

// One operand's share of a step: EXTENT rows of the tile (m or n), LINE bytes of each along the contraction (128 or 64).
template <int DT, int EXTENT, bool TURNED, int WAVES, int LINE>
struct Side {
    using M = Matrix<DT>;
    using T = typename M::T;
    static constexpr int ES = sizeof(T), STEP = LINE / ES, BYTES = EXTENT * LINE;
    static constexpr int UNITS = BYTES / 1024, LOADS = (UNITS + WAVES - 1) / WAVES;        // loads of 1 KB, by each wave (where they do not share out evenly, some bring the same)
    static constexpr int ROW = TURNED ? EXTENT * ES : LINE, CHUNKS = ROW / 16, BLOCKS = ROW / 64;
    static_assert(UNITS * 1024 == BYTES && (LINE == 128 || LINE == 64), "");
    static __device__ __forceinline__ uint32_t unit(int j) {
        const uint32_t at = uniform(threadIdx.x >> 6) * LOADS + j;
        return UNITS % WAVES ? at % UNITS : at;
    }
    uint32_t from[LOADS];       // of the lane, in the step's buffer
    uint32_t column[LOADS];     // lined: bytes into the row

    // Lined: 16-byte chunk c of row r lies at c ^ swap(r), so that the 16 rows that LDS serves together (0..3, 12..15, 20..27 and the others) are on distinct banks.  Turned: 64-byte block b
    // of row k lies at b ^ turn(k), so that the four rows that a read of 16 bits takes together, or every fourth of float32, are.
    static __device__ __forceinline__ int swap(int r) { return LINE == 128 ? r >> 1 & 7 : r >> 2 & 3; }
    static __device__ __forceinline__ int turn(int k) {
        if constexpr (DT == TDB_F32) return k >> 2 & 3;
        else if constexpr (BLOCKS % 4) return k >> 1 & 1;       // (rows of an odd number of 128 bytes: neighbours are on distinct banks by themselves)
        else return ((k & 3) | (k >> 1 & 4)) & (BLOCKS % 8 ? 3 : 7);
    }
    static_assert(!TURNED || (DT == TDB_F32 ? BLOCKS % 4 == 0 : BLOCKS % 2 == 0), "");

    // The same for every tile.  Columns of a turned operand past its width come from its next row, or as zeros: they are sums of their own, which nobody stores.
    __device__ __forceinline__ void place(const Rows& a) {
        const int l = threadIdx.x & 63;
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
            const int at = unit(j) * 64 + l, row = at / CHUNKS, chunk = at % CHUNKS;
            if constexpr (TURNED) {
                from[j] = uint32_t(row) * uint32_t(a.pitch) + ((((chunk >> 2) ^ turn(row)) << 2) | (chunk & 3)) * 16;
            } else {
                column[j] = (chunk ^ swap(row)) * 16;
                from[j] = uint32_t(row) * uint32_t(a.pitch) + column[j];
            }
        }
    }
    // Where a step's buffer begins and how much there is of it from there on; lined: of its rows too.
    struct Cursor {
        const char* p;
        int64_t left, line;
        __device__ __forceinline__ void seek(const Rows& a, int64_t first, int64_t step) {
            if constexpr (TURNED) p = a.p + step * STEP * a.pitch + first * ES, left = (a.count - 1 - step * STEP) * a.pitch + a.width - first * ES, line = 0;
            else p = a.p + first * a.pitch + step * LINE, left = (a.count - 1 - first) * a.pitch + a.width - step * LINE, line = a.width - step * LINE;
        }
        __device__ __forceinline__ void advance(const Rows& a) {
            const int64_t by = TURNED ? STEP * a.pitch : int64_t(LINE);
            p += by, left -= by, line -= by;
        }
    };
    // Loads lo .. hi - 1 of a step into LDS.  TAIL: rows may end inside a step; 16-byte chunks behind their ends are zeros, and clear() takes out what lies behind the
    // end of a row in its last one.
    template <bool TAIL>
    __device__ __forceinline__ void load(const Cursor& c, uint32_t lds, int lo = 0, int hi = LOADS) const {
        const u32x4 buffer = buffer_of(c.p, c.left);
#pragma unroll
        for (int j = 0; j < LOADS; ++j)
            if (j >= lo && j < hi) load_shared(lds + unit(j) * 1024, buffer, TURNED || !TAIL || int(column[j]) < int(max(int64_t(0), min(c.line, int64_t(LINE)))) ? from[j] : PAST);
    }
    // Zeros behind the first `rest` bytes of a lined step's rows, to the end of their 16.
    static __device__ __forceinline__ void clear(char* lds, int rest) {
        for (int r = threadIdx.x; r < EXTENT; r += WAVES * 64)
            for (int b = rest & 15; b < 16; b += 2) *reinterpret_cast<uint16_t*>(lds + r * LINE + ((rest >> 4 ^ swap(r)) << 4) + b) = 0;
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

    // A tile: rows m0 of A, n0 of B, steps [begin, end) of the contraction.
    struct Tile {
        int64_t m0, n0, begin, end;
    };
    // The loads of step after step, of one tile after another.
    struct Flow {
        A side_a;
        B side_b;
        typename A::Cursor at_a;
        typename B::Cursor at_b;
        Rows a, b;
        char* smem;
        uint32_t lds;
        static constexpr int LOADS = A::LOADS + B::LOADS;
        __device__ __forceinline__ Flow(char* smem, const Rows& a, const Rows& b) : a(a), b(b), smem(smem) {
            side_a.place(a), side_b.place(b);
            lds = uniform(uint32_t(reinterpret_cast<uintptr_t>(TDB_SHARED(char, smem))));
        }
        __device__ __forceinline__ void seek(const Tile& t) { at_a.seek(a, t.m0, t.begin), at_b.seek(b, t.n0, t.begin); }
        __device__ __forceinline__ void nothing() { at_a.left = at_b.left = 0; }        // (zeros)
        __device__ __forceinline__ void load(int stage, int lo = 0, int hi = LOADS) {
            side_a.template load<false>(at_a, lds + stage * STAGE, lo, hi);
            side_b.template load<!TURN_A>(at_b, lds + stage * STAGE + A::BYTES, lo - A::LOADS, hi - A::LOADS);
            if (hi == LOADS) at_a.advance(a), at_b.advance(b);
        }
        __device__ __forceinline__ void frag_a(typename M::Frag& f, int stage, int i, int kk) const { f = side_a.frag(smem + stage * STAGE, wave_m() + i * M::SIDE, kk); }
        __device__ __forceinline__ void frag_b(typename M::Frag& f, int stage, int j, int kk) const { f = side_b.frag(smem + stage * STAGE + A::BYTES, wave_n() + j * M::SIDE, kk); }
    };
    // The step of a tile in which B's rows end inside 16 bytes (if there is none, one that never comes), and what lies behind their ends there taken out.
    static __device__ __forceinline__ int ragged_step(const Flow& flow, const Tile& t) { return !TURN_B && flow.b.width % 16 ? int(flow.b.width / LINE - t.begin) : -1; }
    static __device__ __forceinline__ void clear(const Flow& flow, int stage) {
        if constexpr (!TURN_B) B::clear(flow.smem + stage * STAGE + A::BYTES, int(flow.b.width % LINE));
        step_barrier();
    }
    static __device__ __forceinline__ void products(const Flow& flow, int stage, Acc& acc) {
#pragma unroll
        for (int kk = 0; kk < PARTS; ++kk) {
            typename M::Frag fa[TM], fb[TN];
#pragma unroll
            for (int i = 0; i < TM; ++i) flow.frag_a(fa[i], stage, i, kk);
#pragma unroll
            for (int j = 0; j < TN; ++j) flow.frag_b(fb[j], stage, j, kk);
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j) acc[i][j] = M::mma(fb[j], fa[i], acc[i][j]);
        }
    }
    // The sums start from start(j, q), four neighbours along n, called behind a barrier.
    template <class START>
    static __device__ __forceinline__ void begin_sums(Acc& acc, START start) {
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
    }
    static constexpr auto ZEROS = [](int, int) { return f32x4{0.f, 0.f, 0.f, 0.f}; };

    // One tile by itself.
    template <class START>
    static __device__ __forceinline__ void run(Flow& flow, const Tile& t, Acc& acc, START start) {
        const int steps = int(t.end - t.begin), ragged = ragged_step(flow, t);
        step_barrier();                     // nobody has use for what LDS held
        flow.seek(t);
#pragma unroll
        for (int s = 0; s < NS - 1; ++s)
            if (s < steps) flow.load(s);
        begin_sums(acc, start);
        int stage = 0, ahead = NS - 1;
        for (int s = 0; s < steps; ++s) {
            if (s + NS - 2 < steps) wait_loads<(NS - 2) * Flow::LOADS>();
            else wait_loads<0>();
            step_barrier();                 // this stage is there, and nobody reads the one before it any more
            if (s + NS - 1 < steps) flow.load(ahead);
            if (s == ragged) clear(flow, stage);
            products(flow, stage, acc);
            stage = stage == NS - 1 ? 0 : stage + 1;
            ahead = ahead == NS - 1 ? 0 : ahead + 1;
        }
        step_barrier();                     // LDS is free for what follows
    }

    // Tiles one after another with two stages: the first step of the next tile, and what beside.load asks for it, are on their way while this one's last steps are made.  `stage` holds the
    // first step of this tile, which open or the call before has asked for; behind the call the next one's, and scratch(smem, stage) is free.  LATER: memory
    // operations that every wave has issued since the last call asked for this tile's, unless it is the first one.
    template <class BESIDE>
    static __device__ __forceinline__ void open(Flow& flow, const Tile& t, BESIDE& beside) {
        static_assert(NS == 2, "");
        flow.seek(t);
        beside.load(t);
        if (t.begin < t.end) flow.load(0);
    }
    static __device__ __forceinline__ char* scratch(char* smem, int stage) { return smem + (stage ^ 1) * STAGE; }
    template <int LATER, class START, class BESIDE>
    static __device__ __forceinline__ void run_on(Flow& flow, const Tile& t, const Tile& next, bool more, int& stage, bool first, Acc& acc, START start, BESIDE& beside) {
        const int steps = int(t.end - t.begin), ragged = ragged_step(flow, t);
        auto go_on = [&]() {
            flow.seek(next), beside.load(next);
            flow.at_a.left = more ? flow.at_a.left : 0, flow.at_b.left = more ? flow.at_b.left : 0;
        };
        if (LATER == 0 || first) wait_loads<0>();
        else wait_loads<LATER>();
        step_barrier();
        if (steps <= 1) go_on();
        flow.load(stage ^ 1);
        begin_sums(acc, start);
        if (steps == 0) {
            stage ^= 1;
        } else if constexpr (DT == TDB_F32) {
            for (int s = 0; s < steps; ++s) {
                if (s) {
                    wait_loads<0>();
                    step_barrier();
                    if (s + 1 == steps) go_on();
                    flow.load(stage ^ 1);
                }
                if (s == ragged) clear(flow, stage);
                products(flow, stage, acc);
                stage ^= 1;
            }
            settle();
        } else {
            // The frags of a quarter of a step are read while the products of the one before it are made, each of which keeps the matrix pipe busy for 32 clk; the barrier lies in front of a
            // step's last quarter, whose frags are in registers by then, and with that quarter the loads of the step after the next one are issued.
            typename M::Frag fa[2][TM], fb[2][TN];
            auto multiply = [&](auto KK, auto READ, int from, auto LOAD, int to) {
                constexpr int kk = decltype(KK)::value, OPS = TM * TN, R = TM + TN, set = (kk + 1) & 1;
#pragma unroll
                for (int op = 0; op < OPS; ++op) {
                    acc[op / TN][op % TN] = M::mma(fb[kk & 1][op % TN], fa[kk & 1][op / TN], acc[op / TN][op % TN]);
                    __builtin_amdgcn_sched_barrier(0);
                    if constexpr (decltype(READ)::value) {
#pragma unroll
                        for (int r = R * op / OPS; r < R * (op + 1) / OPS; ++r) {
                            if (r < TN) flow.frag_b(fb[set][r < TN ? r : 0], from, r, (kk + 1) % PARTS);
                            else flow.frag_a(fa[set][r < TN ? 0 : r - TN], from, r - TN, (kk + 1) % PARTS);
                        }
                    }
                    if constexpr (decltype(LOAD)::value) flow.load(to, Flow::LOADS * op / OPS, Flow::LOADS * (op + 1) / OPS);
                    __builtin_amdgcn_sched_barrier(0);
                }
            };
            static_assert(PARTS == 4, "");
            constexpr std::true_type yes;
            constexpr std::false_type no;
            constexpr std::integral_constant<int, 0> q0;
            constexpr std::integral_constant<int, 1> q1;
            constexpr std::integral_constant<int, 2> q2;
            constexpr std::integral_constant<int, 3> q3;
            if (ragged == 0) clear(flow, stage);
#pragma unroll
            for (int i = 0; i < TM; ++i) flow.frag_a(fa[0][i], stage, i, 0);
#pragma unroll
            for (int j = 0; j < TN; ++j) flow.frag_b(fb[0][j], stage, j, 0);
            for (int s = 0; s + 1 < steps; ++s) {
                multiply(q0, yes, stage, no, 0);
                multiply(q1, yes, stage, no, 0);
                multiply(q2, yes, stage, no, 0);
                wait_loads<0>();
                step_barrier();
                if (s + 1 == ragged) clear(flow, stage ^ 1);
                if (s + 2 == steps) go_on();
                multiply(q3, yes, stage ^ 1, yes, stage);
                stage ^= 1;
            }
            multiply(q0, yes, stage, no, 0);
            multiply(q1, yes, stage, no, 0);
            multiply(q2, yes, stage, no, 0);
            multiply(q3, no, 0, no, 0);
            stage ^= 1;
        }
        step_barrier();
    }
    // Nothing beside the product's operands.
    struct Alone {
        __device__ __forceinline__ void load(const Tile&) {}
    };

    // The tile's values to rows of memory by way of LDS (SCRATCH bytes), SIDE rows at a time: value(i, j, q) gives four neighbours, then(i, the wave's rows in LDS) may change what
    // lies there.  to: value (m0, n0); rows and columns: how many of the tile's there are.  16 bytes at a time where `wide` (rows at multiples of 4 bytes), and what is less at
    // a row's end value by value: STORES memory operations of every wave at least.
    static constexpr int COLUMNS = TN * M::SIDE, ROW = COLUMNS * int(sizeof(T)), PER = ROW / 16, STORES = TM * M::SIDE * PER / 64;
    static constexpr int SETS = WAVES * 2 * M::SIDE * ROW <= STAGE ? 2 : 1, SCRATCH = WAVES * SETS * M::SIDE * ROW;       // (two where a stage holds them)
    static_assert(SCRATCH <= (NS == 2 ? STAGE : SHARED), "");
    // Where byte b of a wave's row lies: 16-byte chunks exchanged so that 16 rows' chunks are on distinct banks.
    static __device__ __forceinline__ int lies_at(int row, int b) { return row * ROW + (b ^ ((row * ROW / 256 & ((PER & -PER) - 1)) << 4)); }
    template <class OF, class THEN>
    static __device__ __forceinline__ void store(char* scratch, char* to, int64_t pitch, int64_t rows, int64_t columns, bool wide, OF value, THEN then) {
        constexpr int ES = sizeof(T);
        typedef __attribute__((ext_vector_type(4))) T T4;
        const int l = threadIdx.x & 63;
        char* const own = scratch + uniform(threadIdx.x >> 6) * (SETS * M::SIDE * ROW);
        to += wave_m() * pitch + wave_n() * ES, rows -= wave_m(), columns -= wave_n();
#pragma unroll
        for (int i = 0; i < TM; ++i) {
            char* const mine = own + i % SETS * (M::SIDE * ROW);
#pragma unroll
            for (int j = 0; j < TN; ++j)
#pragma unroll
                for (int q = 0; q < M::QUADS; ++q) {
                    const f32x4 v = value(i, j, q);
                    *reinterpret_cast<T4*>(mine + lies_at(lane_m<DT>(), (j * M::SIDE + quad_n<DT>(q)) * ES)) = T4{T(v[0]), T(v[1]), T(v[2]), T(v[3])};
                }
            then(i, mine);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            if (wide) {
                const auto buffer = __builtin_amdgcn_make_buffer_rsrc(to + i * M::SIDE * pitch, 0, int(rows > i * M::SIDE && columns > 0 ? min((rows - 1 - i * M::SIDE) * pitch + columns * ES, int64_t(0x7fffffff)) : 0), 0x00020000);
#pragma unroll
                for (int r = 0; r < M::SIDE * PER / 64; ++r) {
                    const int at = r * 64 + l, row = at / PER, c = at % PER;
                    const u32x4 v = *reinterpret_cast<const u32x4*>(mine + lies_at(row, c * 16));
                    __builtin_amdgcn_raw_buffer_store_b128(v, buffer, c * 16 + 16 <= columns * ES ? uint32_t(row) * uint32_t(pitch) + c * 16 : PAST, 0, 0);
                }
                if (const int whole = int(columns * ES / 16 * (16 / ES)), rest = int(columns) - whole; rest > 0 && columns < COLUMNS)       // a row's end: fewer than 16 bytes
                    for (int at = l; at < M::SIDE * rest; at += 64) {
                        const int row = at / rest, c = whole + at % rest;
                        if (i * M::SIDE + row < rows) *reinterpret_cast<T*>(to + (i * M::SIDE + row) * pitch + c * ES) = *reinterpret_cast<const T*>(mine + lies_at(row, c * ES));
                    }
            } else {
                for (int at = l; at < M::SIDE * COLUMNS; at += 64) {
                    const int row = at / COLUMNS, c = at % COLUMNS;
                    if (i * M::SIDE + row < rows && c < columns) *reinterpret_cast<T*>(to + (i * M::SIDE + row) * pitch + c * ES) = *reinterpret_cast<const T*>(mine + lies_at(row, c * ES));
                }
            }
            if constexpr (SETS == 1) {
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
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
