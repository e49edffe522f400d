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
// are cut into chunks of 8192 elements and a workgroup takes a range of chunks.
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
    uint8_t dtype[kTensors];
    int count;
    uint32_t chunks;
    int norm;                           // 0: max, 1, 2
    int parts;                          // partial norms over all launches
    double *part;                       // the norm pass: this launch's
    double max_norm, eps;
    float *norm_out;                    // or NULL
};
static_assert(sizeof(ClipArgs) <= 4096, "kernel arguments");

// eight elements from p on, at any alignment
template <int DT> __device__ __forceinline__ void load8(const typename Act<DT>::T *p, float (&v)[8])
{
    typename Act<DT>::T e[8];
    __builtin_memcpy(e, p, sizeof(e));
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = Act<DT>::ld(e[k]);
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
__device__ __forceinline__ void chunk_norm(const void *in, int64_t n, int64_t start, double &sum, uint32_t &top)
{
    const typename Act<DT>::T *p = static_cast<const typename Act<DT>::T *>(in) + start;
    const int64_t left = n - start;
    if (left >= kChunk) {
        float v[kPieces][8];
#pragma unroll
        for (int i = 0; i < kPieces; ++i) load8<DT>(p + (i * kBlock + threadIdx.x) * 8, v[i]);
#pragma unroll
        for (int i = 0; i < kPieces; ++i)
#pragma unroll
            for (int k = 0; k < 8; ++k) take<NORM>(sum, top, v[i][k]);
    } else {
        for (int i = threadIdx.x * 8; i < left; i += kBlock * 8) {
            if (i + 8 <= left) {
                float v[8];
                load8<DT>(p + i, v);
#pragma unroll
                for (int k = 0; k < 8; ++k) take<NORM>(sum, top, v[k]);
            } else {
                for (int k = i; k < left; ++k) take<NORM>(sum, top, Act<DT>::ld(p[k]));
            }
        }
    }
}

template <int DT>
__device__ __forceinline__ void chunk_scale(const void *in, void *out, int64_t n, int64_t start, float f)
{
    using T = typename Act<DT>::T;
    const T *p = static_cast<const T *>(in) + start;
    T *q = static_cast<T *>(out) + start;
    const int64_t left = n - start;
    if (left >= kChunk) {
        float v[kPieces][8];
#pragma unroll
        for (int i = 0; i < kPieces; ++i) load8<DT>(p + (i * kBlock + threadIdx.x) * 8, v[i]);
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            T e[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) e[k] = Act<DT>::st(v[i][k] * f);
            __builtin_memcpy(q + (i * kBlock + threadIdx.x) * 8, e, sizeof(e));
        }
    } else {
        for (int64_t i = threadIdx.x; i < left; i += kBlock) q[i] = Act<DT>::st(Act<DT>::ld(p[i]) * f);
    }
}

// f(tensor, first element) over this workgroup's chunks
template <typename F> __device__ __forceinline__ void over_chunks(const ClipArgs &a, F &&f)
{
    uint32_t c = (uint32_t)((uint64_t)a.chunks * blockIdx.x / gridDim.x);
    const uint32_t end = (uint32_t)((uint64_t)a.chunks * (blockIdx.x + 1) / gridDim.x);
    if (c >= end) return;
    int lo = 0, hi = a.count - 1;  // the last tensor that starts at or before chunk c
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (a.first[mid] <= c) lo = mid;
        else hi = mid - 1;
    }
    for (; c < end; ++c) {
        while (lo + 1 < a.count && a.first[lo + 1] <= c) ++lo;
        f(lo, (int64_t)(c - a.first[lo]) * kChunk);
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
    over_chunks(a, [&](int t, int64_t start) {
        if (a.dtype[t] == STACR_DTYPE_F32) chunk_norm<STACR_DTYPE_F32, NORM>(a.in[t], a.n[t], start, sum, top);
        else if (a.dtype[t] == STACR_DTYPE_BF16) chunk_norm<STACR_DTYPE_BF16, NORM>(a.in[t], a.n[t], start, sum, top);
        else chunk_norm<STACR_DTYPE_F16, NORM>(a.in[t], a.n[t], start, sum, top);
    });
    const double v = block_join<NORM>(NORM == 0 ? (double)__uint_as_float(top) : sum);
    if (threadIdx.x == 0) a.part[blockIdx.x] = v;
}

template <int NORM> __global__ __launch_bounds__(kBlock) void k_grad_clip(const ClipArgs a)
{
    double v = 0.0;
    for (int i = threadIdx.x; i < a.parts; i += kBlock) v = joined<NORM>(v, a.part[i]);
    v = block_join<NORM>(v);
    const double norm = NORM == 2 ? sqrt(v) : v;
    if (a.norm_out && blockIdx.x == 0 && threadIdx.x == 0) *a.norm_out = (float)norm;
    if (a.count == 0) return;
    // a NaN norm makes every gradient NaN, an infinite one zero (or NaN where it was infinite)
    double f = a.max_norm / (norm + a.eps);
    if (f > 1.0) f = 1.0;
    const float factor = (float)f;
    over_chunks(a, [&](int t, int64_t start) {
        if (factor == 1.0f && a.in[t] == a.out[t]) return;
        if (a.dtype[t] == STACR_DTYPE_F32) chunk_scale<STACR_DTYPE_F32>(a.in[t], a.out[t], a.n[t], start, factor);
        else if (a.dtype[t] == STACR_DTYPE_BF16) chunk_scale<STACR_DTYPE_BF16>(a.in[t], a.out[t], a.n[t], start, factor);
        else chunk_scale<STACR_DTYPE_F16>(a.in[t], a.out[t], a.n[t], start, factor);
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
            a.dtype[a.count] = (uint8_t)dtypes[i];
            a.first[a.count++] = a.chunks;
            a.chunks += (uint32_t)chunks_of(sizes[i]);
        }
        return i;
    };
    const auto groups = [&](const ClipArgs &a) {
        return (int)hmax<int64_t>(1, hmin<int64_t>(a.chunks, (int64_t)kGroups * a.chunks / hmax<int64_t>(1, total)));
    };
    ClipArgs a{};
    a.norm = norm_type;
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
