// Rotary positions: pairs of features of each head turned by the angle of the token's position.
//
//   (a, b) -> (a cos t - b sin t, b cos t + a sin t),  t = position * frequency of the pair,
// pairs (j, j + rot / 2) or (2 j, 2 j + 1) of the head's first `rot` features, the rest as it is; the
// backward is the turn by -t.  Cosines and sines come from tables in fp32 (made in 64 bits: at position
// 2^16 an angle in fp32 is already off by 2^-9).  The kernel moves every element once and is bound by
// that; queries and keys go in one launch.  A wave takes a token: its lanes keep the table's values of
// their features in registers over all heads, so a table is read once a token and not once a head.
#include "internal.h"

using namespace stacr;

namespace {

struct RotaryArgs {
    const void *in[2];        // queries, keys
    void *out[2];
    int heads[2];
    int64_t si[2][3], so[2][3];  // strides of batch, token, head, in elements
    int64_t seq, tokens;         // tokens: batch * seq
    const float *cos_t, *sin_t;  // length x rot / 2
    int64_t length, offset;
    const void *pos;             // batch x seq, or NULL: offset + token
    int pos_bytes;
    int64_t pos_sb, pos_ss;
    int head, rot;
    int parts;                   // waves that share a token's heads
    bool copy_rest;              // the features past rot have to be written
    float sign;
};

// V elements (16 bytes, or one); STREAM: past the caches
template <int DT, int V, bool STREAM>
__device__ __forceinline__ void get_vec(const typename Act<DT>::T *p, float (&x)[V])
{
    if constexpr (V > 1 && STREAM) {
        const uint4 w = load16_stream(p);
        typename Act<DT>::T e[V];
        __builtin_memcpy(e, &w, 16);
#pragma unroll
        for (int k = 0; k < V; ++k) x[k] = Act<DT>::ld(e[k]);
    } else {
        load_vec<DT, V>(p, x);
    }
}

template <int DT, int V, bool STREAM>
__device__ __forceinline__ void put_vec(typename Act<DT>::T *p, const float (&x)[V])
{
    using A = Act<DT>;
    if constexpr (V == 1) {
        p[0] = A::st(x[0]);
    } else {
        typename A::T e[V];
#pragma unroll
        for (int k = 0; k < V; ++k) e[k] = A::st(x[k]);
        uint4 w;
        __builtin_memcpy(&w, e, 16);
        if constexpr (STREAM) store16_stream(p, w);
        else *reinterpret_cast<uint4 *>(p) = w;
    }
}

// A lane's unit of a head, V = 16 bytes of elements (V 1: rows, strides or features that do not allow
// it).  HALF: V features and their partners; else V neighbouring features (V 1: one pair either way).
// The units past the turned ones are V features to copy.
template <int DT, int V, bool HALF, bool STREAM>
__global__ __launch_bounds__(kBlock) void k_rotary(const RotaryArgs p)
{
    using T = typename Act<DT>::T;
    constexpr int W = V == 1 || HALF ? 2 * V : V;  // features of a turned unit
    constexpr int P = W / 2;                       // its pairs
    const int lane = threadIdx.x & 63;
    const int64_t wave = (int64_t)blockIdx.x * kWaves + (threadIdx.x >> 6);
    const int64_t token = wave / p.parts;
    const int part = (int)(wave - token * p.parts);
    if (token >= p.tokens) return;
    const int64_t b = token / p.seq, s = token - b * p.seq;
    int64_t at = p.offset + s;
    if (p.pos) {
        const int64_t i = b * p.pos_sb + s * p.pos_ss;
        at = p.pos_bytes == 8 ? static_cast<const int64_t *>(p.pos)[i] : static_cast<const int32_t *>(p.pos)[i];
    }
    const bool known = at >= 0 && at < p.length;
    const int half = p.rot / 2;
    const int turned = p.rot / W, units = turned + (p.copy_rest ? (p.head - p.rot) / V : 0);
    const int ul = units < 64 ? units : 64, hl = 64 / ul, h0 = lane / ul;
    if (h0 >= hl) return;
    for (int u = lane - h0 * ul; u < units; u += ul) {
        if (u < turned) {
            const int j = u * P;  // first pair
            float c[P], n[P];
#pragma unroll
            for (int e = 0; e < P; ++e) {
                // a position outside the tables has no angle
                c[e] = known ? p.cos_t[at * half + j + e] : __uint_as_float(0x7fc00000u);
                n[e] = known ? p.sign * p.sin_t[at * half + j + e] : __uint_as_float(0x7fc00000u);
            }
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const T *in = static_cast<const T *>(p.in[t]) + b * p.si[t][0] + s * p.si[t][1];
                T *out = static_cast<T *>(p.out[t]) + b * p.so[t][0] + s * p.so[t][1];
#pragma unroll 4
                for (int h = h0 + part * hl; h < p.heads[t]; h += hl * p.parts) {
                    const T *x = in + h * p.si[t][2];
                    T *y = out + h * p.so[t][2];
                    if constexpr (HALF || V == 1) {
                        const int ja = HALF ? j : 2 * j, jb = HALF ? j + half : 2 * j + 1;
                        float a[V], d[V], ra[V], rd[V];
                        get_vec<DT, V, STREAM>(x + ja, a);
                        get_vec<DT, V, STREAM>(x + jb, d);
#pragma unroll
                        for (int e = 0; e < V; ++e) {
                            ra[e] = a[e] * c[e] - d[e] * n[e];
                            rd[e] = d[e] * c[e] + a[e] * n[e];
                        }
                        put_vec<DT, V, STREAM>(y + ja, ra);
                        put_vec<DT, V, STREAM>(y + jb, rd);
                    } else {
                        float a[V], r[V];
                        get_vec<DT, V, STREAM>(x + 2 * j, a);
#pragma unroll
                        for (int e = 0; e < P; ++e) {
                            r[2 * e] = a[2 * e] * c[e] - a[2 * e + 1] * n[e];
                            r[2 * e + 1] = a[2 * e + 1] * c[e] + a[2 * e] * n[e];
                        }
                        put_vec<DT, V, STREAM>(y + 2 * j, r);
                    }
                }
            }
        } else {
            const int j = p.rot + (u - turned) * V;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const T *in = static_cast<const T *>(p.in[t]) + b * p.si[t][0] + s * p.si[t][1] + j;
                T *out = static_cast<T *>(p.out[t]) + b * p.so[t][0] + s * p.so[t][1] + j;
#pragma unroll 4
                for (int h = h0 + part * hl; h < p.heads[t]; h += hl * p.parts) {
                    const T *x = in + h * p.si[t][2];
                    T *y = out + h * p.so[t][2];
                    if constexpr (V == 1) y[0] = x[0];
                    else if constexpr (STREAM) store16_stream(y, load16_stream(x));
                    else *reinterpret_cast<uint4 *>(y) = *reinterpret_cast<const uint4 *>(x);
                }
            }
        }
    }
}

// cos and sin of position p times frequency base^(-2 j / rot), in 64 bits, rounded once.
//   linear    positions divided by the factor
//   ntk       base' = base factor^(rot / (rot - 2)): the slowest pair as under linear, the fastest as it was
//   by parts  pairs with more than beta_fast turns over the original length as they are, those with fewer
//             than beta_slow divided by the factor, a linear blend between, and both tables times
//             0.1 ln(factor) + 1
__global__ __launch_bounds__(kBlock) void k_rotary_tables(int64_t length, int half, double base, int scaling, double factor,
                                                          double low, double high, float *cos_t, float *sin_t)
{
    const int64_t n = length * half;
    for (int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x; i < n; i += (int64_t)gridDim.x * kBlock) {
        const int64_t at = i / half;
        const int j = (int)(i - at * half);
        double f = pow(base, -(double)j / half), size = 1.0;
        if (scaling == STACR_ROTARY_LINEAR) f /= factor;
        if (scaling == STACR_ROTARY_BY_PARTS) {
            double slow = (j - low) / (high - low);
            slow = slow < 0.0 ? 0.0 : slow > 1.0 ? 1.0 : slow;
            f = f * (1.0 - slow) + f / factor * slow;
            size = factor > 1.0 ? 0.1 * log(factor) + 1.0 : 1.0;
        }
        double sn, cs;
        sincos((double)at * f, &sn, &cs);
        cos_t[i] = (float)(cs * size);
        sin_t[i] = (float)(sn * size);
    }
}

bool whole(const void *p, const int64_t (&st)[3], int64_t v)
{
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && st[0] % v == 0 && st[1] % v == 0 && st[2] % v == 0;
}

template <int DT, int V, bool STREAM> void launch(const RotaryArgs &a, bool half, hipStream_t s)
{
    const int64_t waves = a.tokens * a.parts;
    const unsigned grid = (unsigned)((waves + kWaves - 1) / kWaves);
    stacr_launch("k_rotary", s, [&] {
        if (half) k_rotary<DT, V, true, STREAM><<<grid, kBlock, 0, s>>>(a);
        else k_rotary<DT, V, false, STREAM><<<grid, kBlock, 0, s>>>(a);
    });
}

// 32768 tokens of 40 heads of 128 features (671 MB in and out): 133 us with ordinary loads and stores, 119
// past the caches; what the caches hold stays in them for the attention that follows.
template <int DT> void typed(const RotaryArgs &a, bool vec, bool half, hipStream_t s)
{
    constexpr int V = Act<DT>::kVec;
    const int64_t moved = 2 * a.tokens * (a.heads[0] + a.heads[1]) * a.head * (int64_t)sizeof(typename Act<DT>::T);
    if (!vec) launch<DT, 1, false>(a, half, s);
    else if (moved > 2 * kCacheBytes) launch<DT, V, true>(a, half, s);
    else launch<DT, V, false>(a, half, s);
}

}  // namespace

extern "C" {

int stacr_rotary_tables(int64_t length, int rot, double base, int scaling, double factor, int64_t original_length,
                        double beta_fast, double beta_slow, float *cos_t, float *sin_t, void *stream)
{
    if (length < 0 || rot < 2 || rot % 2 || !(base > 1.0))
        return stacr_fail(STACR_ERR_INVALID, "stacr_rotary_tables: length >= 0, an even rot >= 2 and base > 1 are required");
    if (scaling < STACR_ROTARY_PLAIN || scaling > STACR_ROTARY_BY_PARTS)
        return stacr_fail(STACR_ERR_INVALID, "stacr_rotary_tables: unknown scaling code %d", scaling);
    if (scaling != STACR_ROTARY_PLAIN && !(factor >= 1.0))
        return stacr_fail(STACR_ERR_INVALID, "stacr_rotary_tables: a scaling factor of at least 1 is required");
    if (scaling == STACR_ROTARY_BY_PARTS && (original_length < 1 || !(beta_slow > 0.0) || !(beta_fast > beta_slow)))
        return stacr_fail(STACR_ERR_INVALID, "stacr_rotary_tables: original_length >= 1 and beta_fast > beta_slow > 0 are required");
    if (scaling == STACR_ROTARY_NTK && rot < 4)
        return stacr_fail(STACR_ERR_INVALID, "stacr_rotary_tables: ntk scaling needs rot >= 4");
    if (length == 0) return STACR_OK;
    if (!cos_t || !sin_t) return stacr_fail(STACR_ERR_INVALID, "stacr_rotary_tables: NULL pointer argument");
    hipStream_t s = static_cast<hipStream_t>(stream);
    double low = 0.0, high = 1.0;
    if (scaling == STACR_ROTARY_NTK) base *= pow(factor, (double)rot / (rot - 2));
    if (scaling == STACR_ROTARY_BY_PARTS) {
        // the pair that makes n turns over the original length
        const double scale = rot / (2.0 * log(base)), turn = original_length / 6.283185307179586;
        low = floor(scale * log(turn / beta_fast));
        high = ceil(scale * log(turn / beta_slow));
        if (low < 0.0) low = 0.0;
        if (high > rot / 2 - 1) high = rot / 2 - 1;
        if (high <= low) high = low + 0.001;
    }
    const int64_t n = length * (rot / 2);
    const int grid = (int)hmin<int64_t>((n + kBlock - 1) / kBlock, 65536);
    stacr_launch("k_rotary_tables", s, [&] {
        k_rotary_tables<<<grid, kBlock, 0, s>>>(length, rot / 2, base, scaling, factor, low, high, cos_t, sin_t);
    });
    return stacr_hip_check(hipGetLastError(), "rotary tables kernel");
}

int stacr_rotary(const void *q, const int64_t *q_strides, int q_heads, const void *k, const int64_t *k_strides, int k_heads,
                 int dtype, int64_t batch, int64_t seq, int head, int rot, int layout, const float *cos_t,
                 const float *sin_t, int64_t length, const void *positions, int position_bytes,
                 int64_t position_stride_batch, int64_t position_stride_seq, int64_t offset, int inverse, void *q_out,
                 const int64_t *q_out_strides, void *k_out, const int64_t *k_out_strides, void *stream)
{
    if (dtype != STACR_DTYPE_F32 && dtype != STACR_DTYPE_BF16 && dtype != STACR_DTYPE_F16)
        return stacr_fail(STACR_ERR_INVALID, "stacr_rotary: unsupported dtype code %d", dtype);
    if (batch < 0 || seq < 0 || q_heads < 0 || k_heads < 0 || head < 1 || rot < 2 || rot % 2 || rot > head || length < 0)
        return stacr_fail(STACR_ERR_INVALID, "stacr_rotary: sizes >= 0 and an even rot from 2 to the head are required");
    if (layout != STACR_ROTARY_HALF && layout != STACR_ROTARY_INTERLEAVED)
        return stacr_fail(STACR_ERR_INVALID, "stacr_rotary: unknown layout code %d", layout);
    if (positions && position_bytes != 4 && position_bytes != 8)
        return stacr_fail(STACR_ERR_INVALID, "stacr_rotary: positions of 4 or 8 bytes, got %d", position_bytes);
    if (head > 1 << 16 || q_heads > 1 << 20 || k_heads > 1 << 20)
        return stacr_fail(STACR_ERR_UNSUPPORTED, "stacr_rotary: more than 2^16 features a head, or 2^20 heads");
    if (batch * seq == 0 || q_heads + k_heads == 0) return STACR_OK;
    if ((q_heads && (!q || !q_out || !q_strides || !q_out_strides)) ||
        (k_heads && (!k || !k_out || !k_strides || !k_out_strides)) || !cos_t || !sin_t)
        return stacr_fail(STACR_ERR_INVALID, "stacr_rotary: NULL pointer argument");
    if (batch * seq > (int64_t)1 << 31)
        return stacr_fail(STACR_ERR_UNSUPPORTED, "stacr_rotary: more than 2^31 tokens");
    RotaryArgs a{};
    const void *in[2] = {q, k};
    void *out[2] = {q_out, k_out};
    const int64_t *si[2] = {q_strides, k_strides}, *so[2] = {q_out_strides, k_out_strides};
    const int heads[2] = {q_heads, k_heads};
    const int64_t v = dtype == STACR_DTYPE_F32 ? 4 : 8;
    const bool half = layout == STACR_ROTARY_HALF;
    bool vec = head % v == 0 && rot % v == 0 && (half ? rot / 2 % v == 0 : true), same = true;
    for (int t = 0; t < 2; ++t) {
        if (!heads[t]) continue;
        a.in[t] = in[t];
        a.out[t] = out[t];
        a.heads[t] = heads[t];
        for (int i = 0; i < 3; ++i) {
            a.si[t][i] = si[t][i];
            a.so[t][i] = so[t][i];
            same = same && si[t][i] == so[t][i];
        }
        vec = vec && whole(in[t], a.si[t], v) && whole(out[t], a.so[t], v);
        same = same && in[t] == out[t];
    }
    a.copy_rest = !same && rot < head;
    a.seq = seq;
    a.tokens = batch * seq;
    a.cos_t = cos_t;
    a.sin_t = sin_t;
    a.length = length;
    a.offset = offset;
    a.pos = positions;
    a.pos_bytes = position_bytes;
    a.pos_sb = position_stride_batch;
    a.pos_ss = position_stride_seq;
    a.head = head;
    a.rot = rot;
    a.sign = inverse ? -1.0f : 1.0f;
    // a wave a token, or where tokens are few as many as its heads have passes, up to a wave for each of
    // the chip's 1024 SIMDs
    const int width = vec ? (half ? 2 * (int)v : (int)v) : 2;
    const int units = rot / width + (a.copy_rest ? (head - rot) / (vec ? (int)v : 1) : 0);
    const int hl = units < 64 ? 64 / units : 1;
    const int passes = (int)hmax((q_heads + hl - 1) / hl, (k_heads + hl - 1) / hl);
    a.parts = (int)hmax<int64_t>(1, hmin<int64_t>(passes, 1024 / a.tokens));
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (dtype == STACR_DTYPE_F32) typed<STACR_DTYPE_F32>(a, vec, half, s);
    else if (dtype == STACR_DTYPE_BF16) typed<STACR_DTYPE_BF16>(a, vec, half, s);
    else typed<STACR_DTYPE_F16>(a, vec, half, s);
    return stacr_hip_check(hipGetLastError(), "rotary kernel");
}

}  // extern "C"
