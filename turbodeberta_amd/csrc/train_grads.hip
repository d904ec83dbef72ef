// The norm of many tensors together, and all of them times min(1, max_norm / (norm + 1e-6)).
//
// Bound by memory: a pass reads everything for the norm, and reads it again and writes it where something is clipped.  Tensors are described in the kernels' arguments, a
// launch for each 176 (norm) or 128 of them, so nothing is copied to the device and a captured graph is the same calls.  A workgroup has a run of values of one tensor;
// sums are held in 64 bits (a square of a float32 is no more than that holds, and the instructions are far from binding) and added up in a fixed order: the
// same bits every time, no overflow.
#include <algorithm>
#include <cmath>
#include <new>
#include <vector>

#include "tdb_error.h"
#include "tdb_internal.h"
#include "tdb_train.h"

namespace tdb_train {

constexpr double EPS = 1e-6;
constexpr int HEAD = 2;             // of the workspace: the norm, then the workgroups' sums
constexpr int NORM_TENSORS = 176, CLIP_TENSORS = 128;

// start: the first workgroup of each tensor; kind: types of `from` and `to`
struct NormTable {
    const void* from[NORM_TENSORS];
    int64_t n[NORM_TENSORS];
    uint16_t kind[NORM_TENSORS];
    int32_t start[NORM_TENSORS + 1];
    int32_t tensors, first;         // workgroup number 0 of this launch among all launches'
    int64_t run;                    // values of a workgroup
    double* sums;
};
struct ClipTable {
    const void* from[CLIP_TENSORS];
    void* to[CLIP_TENSORS];
    int64_t n[CLIP_TENSORS];
    uint16_t kind[CLIP_TENSORS];
    int32_t start[CLIP_TENSORS + 1];
    int32_t tensors, first;
    int64_t run;
    const double* norm;
    double max_norm;
};
static_assert(sizeof(NormTable) <= 4096 && sizeof(ClipTable) <= 4096, "kernel arguments");

template <int DT>
struct Value;
template <>
struct Value<TDB_F32> {
    using T = float;
};
template <>
struct Value<TDB_BF16> {
    using T = __bf16;
};
template <>
struct Value<TDB_F16> {
    using T = _Float16;
};

// The tensor that workgroup b of a table has a run of, and where the run begins.
template <class TABLE>
__device__ __forceinline__ int tensor_of(const TABLE& t, int b, int64_t& begin) {
    int lo = 0, hi = t.tensors;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (t.start[mid] <= b) lo = mid;
        else hi = mid;
    }
    begin = (b - t.start[lo]) * t.run;
    return lo;
}

// each(value) over [begin, end), 16 bytes at a time between the first and the last aligned address.
template <int DT, class F>
__device__ __forceinline__ void over_values(const void* from, int64_t begin, int64_t end, F each) {
    using T = typename Value<DT>::T;
    constexpr int PER = 16 / sizeof(T), U = 4;
    typedef __attribute__((ext_vector_type(PER))) T V;
    const T* const p = static_cast<const T*>(from);
    const int64_t odd = (16 - (reinterpret_cast<uintptr_t>(p + begin) & 15)) / sizeof(T) % PER, lo = min(end, begin + odd), chunks = (end - lo) / PER, tail = lo + chunks * PER;
    if (begin + threadIdx.x < lo) each(float(p[begin + threadIdx.x]));
    if (tail + threadIdx.x < end) each(float(p[tail + threadIdx.x]));
    const V* const v = reinterpret_cast<const V*>(p + lo);
    int64_t c = threadIdx.x;
    for (; c + 256 * (U - 1) < chunks; c += 256 * U) {
        V x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) x[u] = v[c + 256 * u];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < PER; ++i) each(float(x[u][i]));
    }
    for (; c < chunks; c += 256) {
        const V x = v[c];
#pragma unroll
        for (int i = 0; i < PER; ++i) each(float(x[i]));
    }
}

// NORM 0: the largest magnitude, as bits, among which NaN is the largest; 1 and 2: sums of magnitudes and squares.
template <int NORM>
struct Sum {
    double sum = 0.0;
    uint32_t most = 0;
    __device__ __forceinline__ void add(float x) {
        if constexpr (NORM == 0) most = max(most, __builtin_bit_cast(uint32_t, x) & 0x7fffffff);
        else if constexpr (NORM == 1) sum += double(fabsf(x));
        else sum = fma(double(x), double(x), sum);
    }
    __device__ __forceinline__ void add(const Sum& o) { sum += o.sum, most = max(most, o.most); }
    __device__ __forceinline__ double value() const { return NORM == 0 ? double(__builtin_bit_cast(float, most)) : sum; }
    static __device__ __forceinline__ Sum of(double x) {
        Sum s;
        if (NORM == 0) s.most = __builtin_bit_cast(uint32_t, float(x)) & 0x7fffffff;
        else s.sum = x;
        return s;
    }
};
// Over the workgroup, in thread 0.
template <int NORM, int WAVES>
__device__ __forceinline__ Sum<NORM> over_block(Sum<NORM> x) {
    __shared__ double parts[WAVES];
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) {
        Sum<NORM> o;
        if (NORM == 0) o.most = __shfl_xor(x.most, d);
        else o.sum = __shfl_xor(x.sum, d);
        x.add(o);
    }
    if ((threadIdx.x & 63) == 0) parts[threadIdx.x >> 6] = x.value();
    __syncthreads();
    if (threadIdx.x == 0) {
#pragma unroll
        for (int w = 1; w < WAVES; ++w) x.add(Sum<NORM>::of(parts[w]));
    }
    return x;
}

template <int NORM>
__global__ __launch_bounds__(256) void grads_norm_kernel(const NormTable t) {
    int64_t begin;
    const int k = tensor_of(t, blockIdx.x, begin);
    const int64_t end = min(t.n[k], begin + t.run);
    Sum<NORM> sum;
    auto each = [&](float x) { sum.add(x); };
    const int kind = t.kind[k] & 3;
    if (kind == TDB_F32) over_values<TDB_F32>(t.from[k], begin, end, each);
    else if (kind == TDB_BF16) over_values<TDB_BF16>(t.from[k], begin, end, each);
    else over_values<TDB_F16>(t.from[k], begin, end, each);
    sum = over_block<NORM, 4>(sum);
    if (threadIdx.x == 0) t.sums[t.first + blockIdx.x] = sum.value();
}

template <int NORM>
__global__ __launch_bounds__(1024) void grads_total_kernel(double* work, int parts, float* total) {
    Sum<NORM> sum;
    for (int i = threadIdx.x; i < parts; i += 1024) sum.add(Sum<NORM>::of(work[HEAD + i]));
    sum = over_block<NORM, 16>(sum);
    if (threadIdx.x == 0) {
        const double norm = NORM == 2 ? sqrt(sum.value()) : sum.value();
        work[0] = norm;
        *total = float(norm);
    }
}

template <int FROM, int TO>
__device__ __forceinline__ void scale_values(const void* from, void* to, int64_t begin, int64_t end, float factor) {
    using F = typename Value<FROM>::T;
    using T = typename Value<TO>::T;
    constexpr int PER = 8, U = 4;
    typedef __attribute__((ext_vector_type(PER))) F VF;
    typedef __attribute__((ext_vector_type(PER))) T VT;
    const F* const x = static_cast<const F*>(from);
    T* const y = static_cast<T*>(to);
    // 8 values at a time where both sides can have aligned ones at once.
    const uintptr_t a = reinterpret_cast<uintptr_t>(x + begin) / sizeof(F) % PER, b = reinterpret_cast<uintptr_t>(y + begin) / sizeof(T) % PER;
    if (a != b) {
        for (int64_t i = begin + threadIdx.x; i < end; i += 256) y[i] = T(float(x[i]) * factor);
        return;
    }
    const int64_t lo = min(end, begin + int64_t((PER - a) % PER)), chunks = (end - lo) / PER, tail = lo + chunks * PER;
    if (begin + threadIdx.x < lo) y[begin + threadIdx.x] = T(float(x[begin + threadIdx.x]) * factor);
    if (tail + threadIdx.x < end) y[tail + threadIdx.x] = T(float(x[tail + threadIdx.x]) * factor);
    const VF* const v = reinterpret_cast<const VF*>(x + lo);
    VT* const w = reinterpret_cast<VT*>(y + lo);
    auto scaled = [&](VF s) {
        VT r;
#pragma unroll
        for (int i = 0; i < PER; ++i) r[i] = T(float(s[i]) * factor);
        return r;
    };
    int64_t c = threadIdx.x;
    for (; c + 256 * (U - 1) < chunks; c += 256 * U) {
        VF s[U];
#pragma unroll
        for (int u = 0; u < U; ++u) s[u] = v[c + 256 * u];
#pragma unroll
        for (int u = 0; u < U; ++u) w[c + 256 * u] = scaled(s[u]);
    }
    for (; c < chunks; c += 256) w[c] = scaled(v[c]);
}

// The last runs first: the norm's pass has read them last, and what of them the last cache holds need not come from memory again.
__global__ __launch_bounds__(256) void grads_scale_kernel(const ClipTable t) {
    const double ratio = t.max_norm / (*t.norm + EPS);
    const float factor = ratio > 1.0 ? 1.f : float(ratio);
    int64_t begin;
    const int k = tensor_of(t, int(gridDim.x - 1 - blockIdx.x), begin);
    const int64_t end = min(t.n[k], begin + t.run);
    const void* const from = t.from[k];
    void* const to = t.to[k];
    if (factor == 1.f && from == to) return;
    switch (t.kind[k]) {
        case TDB_F32 * 4 + TDB_F32: return scale_values<TDB_F32, TDB_F32>(from, to, begin, end, factor);
        case TDB_F32 * 4 + TDB_BF16: return scale_values<TDB_BF16, TDB_F32>(from, to, begin, end, factor);
        case TDB_F32 * 4 + TDB_F16: return scale_values<TDB_F16, TDB_F32>(from, to, begin, end, factor);
        case TDB_BF16 * 4 + TDB_F32: return scale_values<TDB_F32, TDB_BF16>(from, to, begin, end, factor);
        case TDB_BF16 * 4 + TDB_BF16: return scale_values<TDB_BF16, TDB_BF16>(from, to, begin, end, factor);
        case TDB_BF16 * 4 + TDB_F16: return scale_values<TDB_F16, TDB_BF16>(from, to, begin, end, factor);
        case TDB_F16 * 4 + TDB_F32: return scale_values<TDB_F32, TDB_F16>(from, to, begin, end, factor);
        case TDB_F16 * 4 + TDB_BF16: return scale_values<TDB_BF16, TDB_F16>(from, to, begin, end, factor);
        default: return scale_values<TDB_F16, TDB_F16>(from, to, begin, end, factor);
    }
}

// ------------------------------------------------------------------------------------------------------------------- host

int size_of(int dtype) { return dtype == TDB_F32 ? 4 : 2; }
bool known(int dtype) { return dtype == TDB_F32 || dtype == TDB_BF16 || dtype == TDB_F16; }

// Values of a workgroup, and workgroups in all.
int64_t run_of(const tdb_grads_args& a, int64_t& groups) {
    int64_t all = 0;
    for (int i = 0; i < a.tensors; ++i) all += a.numel[i];
    const int64_t run = std::max<int64_t>(8192, (all / 4096 + 2047) / 2048 * 2048);
    groups = 0;
    for (int i = 0; i < a.tensors; ++i) groups += (a.numel[i] + run - 1) / run;
    return run;
}

int check_grads(const tdb_grads_args* a, bool clip) {
    if (!a) return tdb_fail(TDB_ERR_NULL, "args is NULL");
    if (a->tensors < 0 || a->tensors > (1 << 20)) return tdb_fail(TDB_ERR_SHAPE, "%d tensors: need 0 to 2^20", a->tensors);
    if (a->norm < 0 || a->norm > 2) return tdb_fail(TDB_ERR_SHAPE, "norm %d: need 1, 2 or 0 (the largest magnitude)", a->norm);
    if (!a->total || !a->workspace || (a->tensors && (!a->from || !a->numel || !a->from_dtype))) return tdb_fail(TDB_ERR_NULL, "from, numel, from_dtype, total and workspace must be non-NULL");
    if (reinterpret_cast<uintptr_t>(a->workspace) % 8) return tdb_fail(TDB_ERR_ALIGN, "workspace must be 8-byte aligned");
    int64_t all = 0;
    for (int i = 0; i < a->tensors; ++i) {
        if (!known(a->from_dtype[i])) return tdb_fail(TDB_ERR_DTYPE, "tensor %d: unknown dtype %d", i, a->from_dtype[i]);
        if (a->numel[i] < 0 || a->numel[i] > int64_t(1) << 40) return tdb_fail(TDB_ERR_SHAPE, "tensor %d: %lld values", i, (long long)a->numel[i]);
        if (a->numel[i] && !a->from[i]) return tdb_fail(TDB_ERR_NULL, "tensor %d is NULL", i);
        if (reinterpret_cast<uintptr_t>(a->from[i]) % size_of(a->from_dtype[i])) return tdb_fail(TDB_ERR_ALIGN, "tensor %d is not aligned to its values", i);
        all += a->numel[i];
    }
    if (all > int64_t(1) << 42) return tdb_fail(TDB_ERR_SHAPE, "%lld values in all: need up to 2^42", (long long)all);
    if (a->workspace_bytes < tdb_grads_workspace(a)) return tdb_fail(TDB_ERR_SHAPE, "workspace is too small");
    if (!clip) return TDB_OK;
    if (!(a->max_norm >= 0.0)) return tdb_fail(TDB_ERR_SHAPE, "max_norm must not be negative");
    if (a->tensors && (!a->to || !a->to_dtype)) return tdb_fail(TDB_ERR_NULL, "to and to_dtype must be non-NULL");
    // Results may lie where their own input does, and nowhere else on an input or a result.
    struct Range {
        uintptr_t begin, end;
        int tensor;
        bool result;
    };
    std::vector<Range> ranges;
    ranges.reserve(2 * size_t(a->tensors));
    for (int i = 0; i < a->tensors; ++i) {
        if (!known(a->to_dtype[i])) return tdb_fail(TDB_ERR_DTYPE, "result %d: unknown dtype %d", i, a->to_dtype[i]);
        if (!a->numel[i]) continue;
        if (!a->to[i]) return tdb_fail(TDB_ERR_NULL, "result %d is NULL", i);
        const uintptr_t from = reinterpret_cast<uintptr_t>(a->from[i]), to = reinterpret_cast<uintptr_t>(a->to[i]);
        if (to % size_of(a->to_dtype[i])) return tdb_fail(TDB_ERR_ALIGN, "result %d is not aligned to its values", i);
        ranges.push_back({to, to + a->numel[i] * size_of(a->to_dtype[i]), i, true});
        if (to != from || a->to_dtype[i] != a->from_dtype[i]) ranges.push_back({from, from + a->numel[i] * size_of(a->from_dtype[i]), i, false});
    }
    std::sort(ranges.begin(), ranges.end(), [](const Range& x, const Range& y) { return x.begin < y.begin; });
    uintptr_t any_end = 0, result_end = 0;      // of what begins before
    for (const Range& r : ranges) {
        if (r.begin < result_end || (r.result && r.begin < any_end)) return tdb_fail(TDB_ERR_STRIDE, "tensor %d overlaps another one or its result", r.tensor);
        any_end = std::max(any_end, r.end);
        if (r.result) result_end = std::max(result_end, r.end);
    }
    return TDB_OK;
}

// Tables of up to MOST tensors each, launched one after another.
template <class TABLE, int MOST, class FILL, class LAUNCH>
void in_tables(const tdb_grads_args& a, TABLE& t, FILL fill, LAUNCH launch) {
    int64_t groups;
    t.run = run_of(a, groups);
    t.tensors = t.first = t.start[0] = 0;
    auto flush = [&]() {
        if (!t.tensors) return;
        launch(t.start[t.tensors]);
        t.first += t.start[t.tensors];
        t.tensors = 0;
    };
    for (int i = 0; i < a.tensors; ++i) {
        if (!a.numel[i]) continue;
        fill(i, t.tensors);
        t.n[t.tensors] = a.numel[i];
        t.start[t.tensors + 1] = t.start[t.tensors] + int32_t((a.numel[i] + t.run - 1) / t.run);
        if (++t.tensors == MOST) flush();
    }
    flush();
}

int launched() {
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return tdb_fail(TDB_ERR_LAUNCH, "kernel launch failed: %s", hipGetErrorString(e));
    return TDB_OK;
}

template <int NORM>
int norm_of(const tdb_grads_args& a, hipStream_t s) {
    NormTable t;
    double* const work = static_cast<double*>(a.workspace);
    t.sums = work + HEAD;
    in_tables<NormTable, NORM_TENSORS>(a, t, [&](int i, int k) { t.from[k] = a.from[i], t.kind[k] = uint16_t(a.from_dtype[i]); },
                                       [&](int groups) { grads_norm_kernel<NORM><<<groups, 256, 0, s>>>(t); });
    grads_total_kernel<NORM><<<1, 1024, 0, s>>>(work, t.first, a.total);
    return launched();
}

}  // namespace tdb_train

extern "C" {

int64_t tdb_grads_workspace(const tdb_grads_args* a) {
    if (!a || a->tensors < 0 || a->tensors > (1 << 20) || (a->tensors && !a->numel)) return 0;
    for (int i = 0; i < a->tensors; ++i)
        if (a->numel[i] < 0 || a->numel[i] > int64_t(1) << 40) return 0;
    int64_t groups;
    tdb_train::run_of(*a, groups);
    return (tdb_train::HEAD + groups) * 8;
}

int tdb_grads_norm(const tdb_grads_args* a, void* stream) {
    using namespace tdb_train;
    if (const int rc = check_grads(a, false); rc != TDB_OK) return rc;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    return a->norm == 0 ? norm_of<0>(*a, s) : a->norm == 1 ? norm_of<1>(*a, s) : norm_of<2>(*a, s);
}

int tdb_grads_clip(const tdb_grads_args* a, void* stream) try {
    using namespace tdb_train;
    if (const int rc = check_grads(a, true); rc != TDB_OK) return rc;
    ClipTable t;
    t.norm = static_cast<const double*>(a->workspace), t.max_norm = a->max_norm;
    in_tables<ClipTable, CLIP_TENSORS>(*a, t, [&](int i, int k) { t.from[k] = a->from[i], t.to[k] = a->to[i], t.kind[k] = uint16_t(a->to_dtype[i] * 4 + a->from_dtype[i]); },
                                       [&](int groups) { grads_scale_kernel<<<groups, 256, 0, static_cast<hipStream_t>(stream)>>>(t); });
    return launched();
} catch (const std::bad_alloc&) {      // (of the list that overlaps are looked for in)
    return tdb_fail(TDB_ERR_LAUNCH, "out of host memory");
}

}  // extern "C"
