// The global norm over many gradient tensors, and clipping: g <- g min(1, max_norm / (norm + eps)).
//
// Two passes, both bound by memory: partial norms over all tensors, then every workgroup of the second
// pass adds the partials (the same order everywhere, so the same factor on every run) and scales its
// share.  Where the factor is 1 and the result goes in place, the second pass ends there: multiplying
// by 1 would change nothing.  Sums in 64 bits: squares of fp32 neither overflow nor vanish there, and a
// sum over 10^9 values keeps all its digits.
//
// Tensors come as pointers and lengths in the kernel's own arguments (4 KiB: 272 tensors a launch, 176
// with outputs of their own), so nothing is copied to the device and a call can be captured into a graph.  The tensors
// are cut into chunks of 8192 elements and a workgroup takes a range of chunks, so of each tensor one
// run of elements; a chunk's loads are under way while the one before it is worked on.
#include "internal.h"

using namespace stacr;

namespace {

constexpr int kChunk = 8192;            // elements: 256 threads x 4 pieces of 8
constexpr int kPieces = kChunk / (kBlock * 8);
// Workgroups of a launch, 4 a CU.  (Shared out over a call's launches, a third of them each, the norm of
// 266 tensors ran at 3.6 TB/s; one launch with all of them reads at 5.6.)
constexpr int kGroups = 1024;

// The tensors of a launch, at most T, and with outputs of their own where OUT (otherwise in place).
template <int T, bool OUT> struct Table {
    static constexpr int kTensors = T;
    static constexpr bool kOut = OUT;
    const void *in[T];
    void *out[OUT ? T : 1];
    uint32_t first[T + 1];              // first chunk of each, and the end
    uint16_t tail[T];                   // elements of the last chunk (1 .. 8192) | type << 14
    int count;
    int parts;                          // partial norms over all launches
    double *part;                       // the norm pass: this launch's
    double max_norm, eps;
    float *norm_out;                    // or NULL
    bool stream;                        // results past the caches: more than they hold
};
using Alone = Table<272, false>;
using Pairs = Table<176, true>;
static_assert(sizeof(Alone) <= 4096 && sizeof(Pairs) <= 4096, "kernel arguments");

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
__device__ __forceinline__ void run_scale(const void *in, void *out, int64_t from, int64_t to, float f, bool stream)
{
    using T = typename Act<DT>::T;
    const T *p = static_cast<const T *>(in);
    T *q = static_cast<T *>(out);
    const auto put = [&](const float(&v)[8], int64_t at) {
        T e[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) e[k] = Act<DT>::st(v[k] * f);
        if (stream) {
#pragma unroll
            for (int w = 0; w < (int)sizeof(e) / 16; ++w) {
                uint4 x;
                __builtin_memcpy(&x, e + w * (16 / sizeof(T)), 16);
                store16_stream(q + at + w * (16 / sizeof(T)), x);
            }
        } else {
            __builtin_memcpy(q + at, e, sizeof(e));
        }
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

// f(tensor, its type, first element, end) over this workgroup's runs
template <typename A, typename F> __device__ __forceinline__ void over_runs(const A &a, F &&f)
{
    const uint32_t chunks = a.first[a.count];
    uint32_t c = (uint32_t)((uint64_t)chunks * blockIdx.x / gridDim.x);
    const uint32_t end = (uint32_t)((uint64_t)chunks * (blockIdx.x + 1) / gridDim.x);
    if (c >= end) return;
    int t = 0, hi = a.count - 1;  // the last tensor that starts at or before chunk c
    while (t < hi) {
        const int mid = (t + hi + 1) >> 1;
        if (a.first[mid] <= c) t = mid;
        else hi = mid - 1;
    }
    for (; c < end; ++t) {
        const uint32_t first = a.first[t], next = a.first[t + 1], stop = next < end ? next : end;
        const uint32_t tail = a.tail[t];
        const int64_t n = (int64_t)(next - first - 1) * kChunk + (tail & 0x3fffu), to = (int64_t)(stop - first) * kChunk;
        f(t, tail >> 14, (int64_t)(c - first) * kChunk, to < n ? to : n);
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

template <int NORM> __global__ __launch_bounds__(kBlock) void k_grad_norm(const Alone a)
{
    double sum = 0.0;
    uint32_t top = 0;
    over_runs(a, [&](int t, uint32_t type, int64_t from, int64_t to) {
        if (type == STACR_DTYPE_F32) run_norm<STACR_DTYPE_F32, NORM>(a.in[t], from, to, sum, top);
        else if (type == STACR_DTYPE_BF16) run_norm<STACR_DTYPE_BF16, NORM>(a.in[t], from, to, sum, top);
        else run_norm<STACR_DTYPE_F16, NORM>(a.in[t], from, to, sum, top);
    });
    const double v = block_join<NORM>(NORM == 0 ? (double)__uint_as_float(top) : sum);
    if (threadIdx.x == 0) a.part[blockIdx.x] = v;
}

template <int NORM, typename A> __global__ __launch_bounds__(kBlock) void k_grad_clip(const A a)
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
    if (!A::kOut && factor == 1.0f) return;
    over_runs(a, [&](int t, uint32_t type, int64_t from, int64_t to) {
        void *out = A::kOut ? a.out[A::kOut ? t : 0] : const_cast<void *>(a.in[t]);
        if (factor == 1.0f && a.in[t] == out) return;
        if (type == STACR_DTYPE_F32) run_scale<STACR_DTYPE_F32>(a.in[t], out, from, to, factor, a.stream);
        else if (type == STACR_DTYPE_BF16) run_scale<STACR_DTYPE_BF16>(a.in[t], out, from, to, factor, a.stream);
        else run_scale<STACR_DTYPE_F16>(a.in[t], out, from, to, factor, a.stream);
    });
}

int64_t chunks_of(int64_t n) { return (n + kChunk - 1) / kChunk; }

// the launch of tensors from `i` on, as many as fit of those that hold anything; i moves past them
template <typename A>
void fill(A &a, int &i, int count, const void *const *in, void *const *out, const int64_t *sizes, const int *dtypes)
{
    a.count = 0;
    a.first[0] = 0;
    for (; i < count && a.count < A::kTensors; ++i) {
        if (!sizes[i]) continue;
        const int64_t chunks = chunks_of(sizes[i]);
        a.in[a.count] = in[i];
        if (A::kOut) a.out[a.count] = out[i];
        a.tail[a.count] = (uint16_t)((sizes[i] - (chunks - 1) * kChunk) | dtypes[i] << 14);
        a.first[a.count + 1] = a.first[a.count] + (uint32_t)chunks;
        ++a.count;
    }
}

template <typename A> int groups(const A &a) { return (int)hmin<int64_t>(kGroups, a.first[a.count]); }

template <typename A>
void clip_launches(int norm_type, int count, const void *const *in, void *const *out, const int64_t *sizes, const int *dtypes,
                   double max_norm, double eps, double *part, int parts, float *norm, bool stream, hipStream_t s)
{
    A a{};
    a.stream = stream;
    a.max_norm = max_norm;
    a.eps = eps;
    a.part = part;
    a.parts = parts;
    a.norm_out = norm;
    int i = 0;
    do {
        if (out) fill(a, i, count, in, out, sizes, dtypes);
        const int grid = a.count ? groups(a) : 1;  // none: the norm alone
        if (a.count || a.norm_out)
            stacr_launch("k_grad_clip", s, [&] {
                if (norm_type == 2) k_grad_clip<2, A><<<grid, kBlock, 0, s>>>(a);
                else if (norm_type == 1) k_grad_clip<1, A><<<grid, kBlock, 0, s>>>(a);
                else k_grad_clip<0, A><<<grid, kBlock, 0, s>>>(a);
            });
        a.norm_out = nullptr;
    } while (out && i < count);
}

}  // namespace

extern "C" {

int stacr_clip_workspace_bytes(int count, size_t *bytes)
{
    if (count < 0 || !bytes) return stacr_fail(STACR_ERR_INVALID, "stacr_clip_workspace_bytes: bad argument");
    *bytes = sizeof(double) * (size_t)kGroups * (size_t)((count + Alone::kTensors - 1) / Alone::kTensors + 1);
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
    int64_t total = 0, bytes = 0;
    for (int i = 0; i < count; ++i) {
        if (sizes[i] < 0 || (sizes[i] && (!in[i] || (out && !out[i]))))
            return stacr_fail(STACR_ERR_INVALID, "stacr_clip_gradients: tensor %d has a negative size or a NULL pointer", i);
        if (dtypes[i] < STACR_DTYPE_F32 || dtypes[i] > STACR_DTYPE_F16)
            return stacr_fail(STACR_ERR_INVALID, "stacr_clip_gradients: tensor %d has dtype code %d", i, dtypes[i]);
        total += chunks_of(sizes[i]);
        bytes += sizes[i] * (dtypes[i] == STACR_DTYPE_F32 ? 4 : 2);
    }
    if (total >= (int64_t)1 << 32) return stacr_fail(STACR_ERR_UNSUPPORTED, "stacr_clip_gradients: more than 2^45 elements");
    size_t need = 0;
    const int rc = stacr_clip_workspace_bytes(count, &need);
    if (rc) return rc;
    if (!workspace || workspace_bytes < need)
        return stacr_fail(STACR_ERR_WORKSPACE, "stacr_clip_gradients: workspace of %zu bytes, %zu needed", workspace_bytes, need);
    hipStream_t s = static_cast<hipStream_t>(stream);
    double *part = static_cast<double *>(workspace);

    int parts = 0;
    Alone a{};
    for (int i = 0; i < count;) {
        fill(a, i, count, in, nullptr, sizes, dtypes);
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
    // 454 M elements of 16 bits with results of their own: 553 us with ordinary stores, 528 past the caches
    const bool past = bytes > kCacheBytes;
    bool place = true;
    for (int i = 0; out && i < count; ++i) place = place && out[i] == in[i];
    if (place) clip_launches<Alone>(norm_type, count, in, out, sizes, dtypes, max_norm, eps, part, parts, norm, past, s);
    else clip_launches<Pairs>(norm_type, count, in, out, sizes, dtypes, max_norm, eps, part, parts, norm, past, s);
    return stacr_hip_check(hipGetLastError(), "gradient clipping kernels");
}

}  // extern "C"
