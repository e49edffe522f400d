// The global norm over many gradient tensors, and clipping: g <- g min(1, max_norm / (norm + eps)).
//
// Two passes, both bound by memory: partial norms over all tensors, then every workgroup of the second
// pass adds the partials (the same order everywhere, so the same factor on every run) and scales its
// share.  Where the factor is 1 and the result goes in place, the second pass ends there: multiplying
// by 1 would change nothing.  Sums in 64 bits: squares of fp32 neither overflow nor vanish there, and a
// sum over 10^9 values keeps all its digits.
//
// Tensors come as pointers and lengths in the kernel's own arguments (4 KiB: about 120 tensors a
// launch), so nothing is copied to the device and a call can be captured into a graph.  The tensors
// are cut into chunks of 8192 elements and a workgroup takes a range of chunks, so of each tensor one
// run of elements; a chunk's loads are under way while the one before it is worked on.
#include "internal.h"

using namespace stacr;

namespace {

constexpr int kTensors = 120;           // of a launch
constexpr int kChunk = 8192;            // elements: 256 threads x 4 pieces of 8
constexpr int kPieces = kChunk / (kBlock * 8);
constexpr int kGroups = 1024;           // workgroups of a pass over all its launches, 4 a CU

struct ClipArgs {
    const void *in[kTensors];
    void *out[kTensors];
    int64_t n[kTensors];
    uint32_t first[kTensors];           // first chunk of the tensor in this launch
    uint32_t dtype[kTensors];
    int count;
    uint32_t chunks;
    int parts;                          // partial norms over all launches
    double *part;                       // the norm pass: this launch's
    double max_norm, eps;
    float *norm_out;                    // or NULL
};
static_assert(sizeof(ClipArgs) <= 4096, "kernel arguments");

struct Raw8 {  // eight elements as they lie in memory
    uint4 w[2];
};

// eight elements from p on, at any alignment
template <int DT> __device__ __forceinline__ Raw8 load8(const typename Act<DT>::T *p)
{
    Raw8 r;
    __builtin_memcpy(&r.w, p, 8 * sizeof(*p));
    return r;
}

template <int DT> __device__ __forceinline__ void widen(const Raw8 &r, float (&v)[8])
{
    typename Act<DT>::T e[8];
    __builtin_memcpy(e, &r.w, sizeof(e));
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = Act<DT>::ld(e[k]);
}

// body(values, first element's offset) over the whole chunks of elements [from, to), two chunks under way;
// returns where the rest begins
template <int DT, typename F>
__device__ __forceinline__ int64_t whole_chunks(const typename Act<DT>::T *p, int64_t from, int64_t to, F &&body)
{
    const int mine = threadIdx.x * 8;
    if (to - from < kChunk) return from;
    Raw8 r[kPieces], next[kPieces];
#pragma unroll
    for (int i = 0; i < kPieces; ++i) r[i] = load8<DT>(p + from + i * kBlock * 8 + mine);
    for (; to - from >= kChunk; from += kChunk) {
        const bool more = to - from >= 2 * kChunk;
        if (more) {
#pragma unroll
            for (int i = 0; i < kPieces; ++i) next[i] = load8<DT>(p + from + kChunk + i * kBlock * 8 + mine);
        }
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            float v[8];
            widen<DT>(r[i], v);
            body(v, from + i * kBlock * 8 + mine);
            if (more) r[i] = next[i];
        }
    }
    return from;
}

template <int NORM> __device__ __forceinline__ void take(double &sum, uint32_t &top, float v)
{
    if constexpr (NORM == 2) sum = __builtin_fma((double)v, (double)v, sum);
    else if constexpr (NORM == 1) sum += (double)__builtin_fabsf(v);
    else {  // magnitudes order as integers, NaN above infinity
        const uint32_t key = __float_as_uint(v) & 0x7fffffffu;
        top = key > top ? key : top;
    }
}

template <int DT, int NORM>
__device__ __forceinline__ void run_norm(const void *in, int64_t from, int64_t to, double &sum, uint32_t &top)
{
    const typename Act<DT>::T *p = static_cast<const typename Act<DT>::T *>(in);
    from = whole_chunks<DT>(p, from, to, [&](const float(&v)[8], int64_t) {
#pragma unroll
        for (int k = 0; k < 8; ++k) take<NORM>(sum, top, v[k]);
    });
    for (int64_t i = from + threadIdx.x * 8; i < to; i += kBlock * 8) {
        if (i + 8 <= to) {
            float v[8];
            widen<DT>(load8<DT>(p + i), v);
#pragma unroll
            for (int k = 0; k < 8; ++k) take<NORM>(sum, top, v[k]);
        } else {
            for (int64_t k = i; k < to; ++k) take<NORM>(sum, top, Act<DT>::ld(p[k]));
        }
    }
}

template <int DT>
__device__ __forceinline__ void run_scale(const void *in, void *out, int64_t from, int64_t to, float f)
{
    using T = typename Act<DT>::T;
    const T *p = static_cast<const T *>(in);
    T *q = static_cast<T *>(out);
    const auto put = [&](const float(&v)[8], int64_t at) {
        T e[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) e[k] = Act<DT>::st(v[k] * f);
        __builtin_memcpy(q + at, e, sizeof(e));
    };
    from = whole_chunks<DT>(p, from, to, put);
    for (int64_t i = from + threadIdx.x * 8; i < to; i += kBlock * 8) {
        if (i + 8 <= to) {
            float v[8];
            widen<DT>(load8<DT>(p + i), v);
            put(v, i);
        } else {
            for (int64_t k = i; k < to; ++k) q[k] = Act<DT>::st(Act<DT>::ld(p[k]) * f);
        }
    }
}

// f(tensor, first element, end) over this workgroup's runs
template <typename F> __device__ __forceinline__ void over_runs(const ClipArgs &a, F &&f)
{
    uint32_t c = (uint32_t)((uint64_t)a.chunks * blockIdx.x / gridDim.x);
    const uint32_t end = (uint32_t)((uint64_t)a.chunks * (blockIdx.x + 1) / gridDim.x);
    if (c >= end) return;
    int t = 0, hi = a.count - 1;  // the last tensor that starts at or before chunk c
    while (t < hi) {
        const int mid = (t + hi + 1) >> 1;
        if (a.first[mid] <= c) t = mid;
        else hi = mid - 1;
    }
    for (; c < end; ++t) {
        const uint32_t first = a.first[t], stop = t + 1 < a.count && a.first[t + 1] < end ? a.first[t + 1] : end;
        const int64_t to = (int64_t)(stop - first) * kChunk;
        f(t, (int64_t)(c - first) * kChunk, to < a.n[t] ? to : a.n[t]);
        c = stop;
    }
}

template <int NORM> __device__ __forceinline__ double joined(double a, double b)
{
    if constexpr (NORM == 0) return b > a || b != b ? b : a;
    else return a + b;
}

template <int NORM> __device__ __forceinline__ double block_join(double v)
{
    __shared__ double s[kWaves];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = joined<NORM>(v, __shfl_xor(v, o, 64));
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    v = s[0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) v = joined<NORM>(v, s[w]);
    __syncthreads();
    return v;
}

template <int NORM> __global__ __launch_bounds__(kBlock) void k_grad_norm(const ClipArgs a)
{
    double sum = 0.0;
    uint32_t top = 0;
    over_runs(a, [&](int t, int64_t from, int64_t to) {
        if (a.dtype[t] == STACR_DTYPE_F32) run_norm<STACR_DTYPE_F32, NORM>(a.in[t], from, to, sum, top);
        else if (a.dtype[t] == STACR_DTYPE_BF16) run_norm<STACR_DTYPE_BF16, NORM>(a.in[t], from, to, sum, top);
        else run_norm<STACR_DTYPE_F16, NORM>(a.in[t], from, to, sum, top);
    });
    const double v = block_join<NORM>(NORM == 0 ? (double)__uint_as_float(top) : sum);
    if (threadIdx.x == 0) a.part[blockIdx.x] = v;
}

template <int NORM> __global__ __launch_bounds__(kBlock) void k_grad_clip(const ClipArgs a)
{
    double v = 0.0;
#pragma unroll 8
    for (int i = threadIdx.x; i < a.parts; i += kBlock) v = joined<NORM>(v, a.part[i]);
    v = block_join<NORM>(v);
    const double norm = NORM == 2 ? sqrt(v) : v;
    if (a.norm_out && blockIdx.x == 0 && threadIdx.x == 0) *a.norm_out = (float)norm;
    if (a.count == 0) return;
    // a NaN norm makes every gradient NaN, an infinite one zero (or NaN where it was infinite)
    double f = a.max_norm / (norm + a.eps);
    if (f > 1.0) f = 1.0;
    const float factor = (float)f;
    over_runs(a, [&](int t, int64_t from, int64_t to) {
        if (factor == 1.0f && a.in[t] == a.out[t]) return;
        if (a.dtype[t] == STACR_DTYPE_F32) run_scale<STACR_DTYPE_F32>(a.in[t], a.out[t], from, to, factor);
        else if (a.dtype[t] == STACR_DTYPE_BF16) run_scale<STACR_DTYPE_BF16>(a.in[t], a.out[t], from, to, factor);
        else run_scale<STACR_DTYPE_F16>(a.in[t], a.out[t], from, to, factor);
    });
}

int64_t chunks_of(int64_t n) { return (n + kChunk - 1) / kChunk; }

int launches_for(int count) { return (count + kTensors - 1) / kTensors; }

}  // namespace

extern "C" {

int stacr_clip_workspace_bytes(int count, size_t *bytes)
{
    if (count < 0 || !bytes) return stacr_fail(STACR_ERR_INVALID, "stacr_clip_workspace_bytes: bad argument");
    *bytes = sizeof(double) * (size_t)(kGroups + launches_for(count) + 1);
    return STACR_OK;
}

int stacr_clip_gradients(int count, const void *const *in, void *const *out, const int64_t *sizes, const int *dtypes,
                         int norm_type, double max_norm, double eps, float *norm, void *workspace, size_t workspace_bytes,
                         void *stream)
{
    if (count < 0 || (count && (!in || !sizes || !dtypes)) || !norm)
        return stacr_fail(STACR_ERR_INVALID, "stacr_clip_gradients: NULL pointer argument");
    if (norm_type < 0 || norm_type > 2)
        return stacr_fail(STACR_ERR_INVALID, "stacr_clip_gradients: norm type 0 (max), 1 or 2, got %d", norm_type);
    if (out && (!(max_norm >= 0.0) || !(eps >= 0.0)))
        return stacr_fail(STACR_ERR_INVALID, "stacr_clip_gradients: max_norm and eps must not be negative");
    int64_t total = 0;
    for (int i = 0; i < count; ++i) {
        if (sizes[i] < 0 || (sizes[i] && (!in[i] || (out && !out[i]))))
            return stacr_fail(STACR_ERR_INVALID, "stacr_clip_gradients: tensor %d has a negative size or a NULL pointer", i);
        if (dtypes[i] < STACR_DTYPE_F32 || dtypes[i] > STACR_DTYPE_F16)
            return stacr_fail(STACR_ERR_INVALID, "stacr_clip_gradients: tensor %d has dtype code %d", i, dtypes[i]);
        total += chunks_of(sizes[i]);
    }
    if (total >= (int64_t)1 << 32) return stacr_fail(STACR_ERR_UNSUPPORTED, "stacr_clip_gradients: more than 2^45 elements");
    size_t need = 0;
    const int rc = stacr_clip_workspace_bytes(count, &need);
    if (rc) return rc;
    if (!workspace || workspace_bytes < need)
        return stacr_fail(STACR_ERR_WORKSPACE, "stacr_clip_gradients: workspace of %zu bytes, %zu needed", workspace_bytes, need);
    hipStream_t s = static_cast<hipStream_t>(stream);
    double *part = static_cast<double *>(workspace);

    // the launch of tensors from `first` on: at most kTensors that hold anything; returns the next first
    const auto fill = [&](ClipArgs &a, int first) {
        a.count = 0;
        a.chunks = 0;
        int i = first;
        for (; i < count && a.count < kTensors; ++i) {
            if (!sizes[i]) continue;
            a.in[a.count] = in[i];
            a.out[a.count] = out ? out[i] : nullptr;
            a.n[a.count] = sizes[i];
            a.dtype[a.count] = (uint32_t)dtypes[i];
            a.first[a.count++] = a.chunks;
            a.chunks += (uint32_t)chunks_of(sizes[i]);
        }
        return i;
    };
    const auto groups = [&](const ClipArgs &a) {
        return (int)hmax<int64_t>(1, hmin<int64_t>(a.chunks, (int64_t)kGroups * a.chunks / hmax<int64_t>(1, total)));
    };
    ClipArgs a{};
    a.max_norm = max_norm;
    a.eps = eps;
    int parts = 0;
    for (int i = 0; i < count;) {
        i = fill(a, i);
        if (!a.count) break;
        const int grid = groups(a);
        a.part = part + parts;
        parts += grid;
        stacr_launch("k_grad_norm", s, [&] {
            if (norm_type == 2) k_grad_norm<2><<<grid, kBlock, 0, s>>>(a);
            else if (norm_type == 1) k_grad_norm<1><<<grid, kBlock, 0, s>>>(a);
            else k_grad_norm<0><<<grid, kBlock, 0, s>>>(a);
        });
    }
    a.part = part;
    a.parts = parts;
    a.norm_out = norm;
    int i = 0;
    do {
        a.count = 0;
        a.chunks = 0;
        if (out) i = fill(a, i);
        const int grid = a.count ? groups(a) : 1;
        if (a.count || a.norm_out)
            stacr_launch("k_grad_clip", s, [&] {
                if (norm_type == 2) k_grad_clip<2><<<grid, kBlock, 0, s>>>(a);
                else if (norm_type == 1) k_grad_clip<1><<<grid, kBlock, 0, s>>>(a);
                else k_grad_clip<0><<<grid, kBlock, 0, s>>>(a);
            });
        a.norm_out = nullptr;
    } while (out && i < count);
    return stacr_hip_check(hipGetLastError(), "gradient clipping kernels");
}

}  // extern "C"
