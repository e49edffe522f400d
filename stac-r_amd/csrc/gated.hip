// The gated feed-forward block: h = act(x Wg^T + bg) * (x Wu^T + bu), and its backward pass.
//
//   forward    one product over [Wg; Wu] whose tiles hold a gate column block beside the same up
//              columns, so that a lane ends with both pre-activations of its outputs and the epilogue
//              writes h = act(g) u alone
//   backward   dg = dh u act'(g), du = dh act(g): an elementwise pass over g and u, which the forward
//              kept, or, where it kept x alone, the same product again with another epilogue; then
//              dx = dg Wg + du Wu (one product, K over both halves), [dWg; dWu] = [dg | du]^T x
//   few rows   a workgroup of four waves takes 16 outputs of both projections, each wave a quarter of
//              K: the weights are read once, straight into the operands
//
// 16-bit types multiply as they are, sums in fp32.  dg and du are rounded to the type between the
// products (they are the next product's matrix-core operands).  fp32 is split into three bf16 parts
// x = hi + mid + lo (8 + 8 + 8 significand bits by truncation, so the split is exact), and a product is
// the six part products down to 2^-16 of the leading one: the terms left out are below 2^-21 of
// |a| |b|, where fp32's own rounding of the sum is 2^-24 a step.  A fourth plane holds hi with
// infinities and NaN replaced by 0, which the five smaller products take, so that a non-finite value
// meets the other operand once, in hi * hi, as it would in fp32.
#include <type_traits>

#include "matmul_tile.h"

using namespace stacr;

namespace {

enum { kFwd = 0, kBwd = 1, kStore = 2 };  // epilogues
constexpr int kPlanes = 4;                // hi, mid, lo, finite hi
constexpr int kPairs = 6;
// (plane of A, plane of B) of the six products, the smallest first
constexpr int kPairA[kPairs] = {2, 3, 1, 1, 3, 0};
constexpr int kPairB[kPairs] = {3, 2, 1, 3, 1, 0};

struct MmArgs {
    MmOperand a, b;
    const uint16_t *b2[kMmMaxSegs];  // up weights (forward and recomputation)
    int nseg;
    int64_t M, N, K;                 // N: columns of C (of one half of it, for the gated products)
    int64_t a_half;                  // second half of C's rows: A's column offset
    int halves;
    int mt, nt, splits, tiles;       // tiles: of all halves and splits
    void *out, *out2;
    int64_t ldo;
    int out_dt;
    float *part;                     // splits > 1: fp32 partial products [split][half][M][N]
    // gated epilogues
    const void *bias_g, *bias_u, *dh;
    void *gate, *up;                 // kept pre-activations or NULL, in the type, or with the low
    uint8_t *gate_low, *up_low;      // bytes not NULL the upper 16 of 24 bits
    uint16_t *dgu;                   // [plane][M][2 * ff_pad]
    int64_t ff_pad, plane;
    int act;
};

// ------------------------------------------------------------------ activations
// fp32 takes the accurate library functions and divisions, the 16-bit types the exponential and the
// reciprocal of one instruction (about 1e-6 relative at |x| < 20, a thousandth of their rounding).
template <bool EXACT> __device__ __forceinline__ float exp_of(float x)
{
    if constexpr (EXACT) return expf(x);
    else return __expf(x);
}

template <bool EXACT> __device__ __forceinline__ float inverse(float x)
{
    if constexpr (EXACT) return 1.0f / x;
    else return __builtin_amdgcn_rcpf(x);
}

// The normal distribution below g, bell = exp(-g^2 / 2).  With x = |g| / sqrt(2) the part beyond |g| is
// erfc(x) / 2 = bell exp(x^2) erfc(x) / 2, and exp(x^2) erfc(x) is smooth and falls like 1 / x: a polynomial
// without a constant term in t = 1 / (1 + 0.51 x), fitted for the least largest relative error, 9e-7, over
// 0 <= x <= 10 (in fp32, for g above -4: 2e-6, where 1 + erf(x) in fp32 loses 1e-3).  The library's erf takes
// about 30 instructions on two paths that a wave mostly takes both.
__device__ __forceinline__ float normal_below(float g, float bell)
{
    const float t = __builtin_amdgcn_rcpf(fmaf(fabsf(g), 0.51f * 0.70710678118654752f, 1.0f));
    float p = 0.094499744f;
    p = fmaf(p, t, -0.35913408f);
    p = fmaf(p, t, 0.35844463f);
    p = fmaf(p, t, 0.055053536f);
    p = fmaf(p, t, 0.27906591f);
    p = fmaf(p, t, 0.28415236f);
    p = fmaf(p, t, 0.28791749f);
    const float beyond = 0.5f * p * t * bell;
    return g < 0.0f ? beyond : 1.0f - beyond;
}

// act(g) and act'(g)
template <bool EXACT, int ACT> __device__ __forceinline__ void activate(float g, float &a, float &slope)
{
    if constexpr (ACT == STACR_ACT_SILU) {
        const float s = inverse<EXACT>(1.0f + exp_of<EXACT>(-g));
        a = g * s;
        slope = s * (1.0f + g * (1.0f - s));
    } else if constexpr (ACT == STACR_ACT_GELU) {
        const float bell = exp_of<EXACT>(-0.5f * g * g);
        const float below = EXACT ? 0.5f * (1.0f + erff(g * 0.70710678118654752f)) : normal_below(g, bell);
        a = g * below;
        slope = below + g * 0.39894228040143268f * bell;
    } else if constexpr (ACT == STACR_ACT_GELU_TANH) {
        const float in = 0.79788456080286536f * (g + 0.044715f * g * g * g);
        const float t = 1.0f - 2.0f * inverse<EXACT>(1.0f + exp_of<EXACT>(2.0f * in));
        a = 0.5f * g * (1.0f + t);
        const float bend = 1.0f - t * t;  // 0 in the tails, where g * g may be infinite
        slope = 0.5f * (1.0f + t);
        if (bend > 0.0f) slope += 0.5f * g * bend * 0.79788456080286536f * (1.0f + 3.0f * 0.044715f * g * g);
    } else if constexpr (ACT == STACR_ACT_RELU) {
        a = g > 0.0f ? g : (g != g ? g : 0.0f);
        slope = g > 0.0f ? 1.0f : 0.0f;
    } else {
        const float s = inverse<EXACT>(1.0f + exp_of<EXACT>(-g));
        a = s;
        slope = s * (1.0f - s);
    }
}

// f(the activation's code as a constant): the choice is made once, outside the unrolled epilogues, whose
// code would not fit the instruction cache with a choice a value
template <typename F> __device__ __forceinline__ void with_activation(int act, F &&f)
{
    switch (act) {
    case STACR_ACT_SILU: f(std::integral_constant<int, STACR_ACT_SILU>()); break;
    case STACR_ACT_GELU: f(std::integral_constant<int, STACR_ACT_GELU>()); break;
    case STACR_ACT_GELU_TANH: f(std::integral_constant<int, STACR_ACT_GELU_TANH>()); break;
    case STACR_ACT_RELU: f(std::integral_constant<int, STACR_ACT_RELU>()); break;
    default: f(std::integral_constant<int, STACR_ACT_SIGMOID>());
    }
}

template <bool EXACT> __device__ __forceinline__ void activate(int act, float g, float &a, float &slope)
{
    with_activation(act, [&](auto c) { activate<EXACT, decltype(c)::value>(g, a, slope); });
}

// the three bf16 parts of v by truncation, and hi without infinities and NaN; a NaN keeps a set bit
__device__ __forceinline__ void split_f32(float v, uint16_t (&p)[kPlanes])
{
    const uint32_t u = __float_as_uint(v);
    const bool finite = (u & 0x7f800000u) != 0x7f800000u;
    const uint32_t hi = u & 0xffff0000u;
    p[0] = (uint16_t)((hi >> 16) | (!finite && (u & 0x7fffffu) ? 0x40u : 0u));
    p[3] = finite ? p[0] : (uint16_t)0;
    const float r1 = finite ? v - __uint_as_float(hi) : 0.0f;
    const uint32_t mid = __float_as_uint(r1) & 0xffff0000u;
    p[1] = (uint16_t)(mid >> 16);
    p[2] = (uint16_t)(__float_as_uint(r1 - __uint_as_float(mid)) >> 16);
}

// The 24-bit form of a kept pre-activation: fp32 rounded to its upper three bytes (2^-16 relative).  Kept in
// the 16-bit type, g and u would each put another rounding of that type into dg and du; this one is a
// hundredth of it.
__device__ __forceinline__ uint32_t to_24(float v)
{
    return v != v ? 0x7fc00000u : __float_as_uint(v) + 0x80u;  // the lowest byte is not kept
}

// ------------------------------------------------------------------ rows of a result
// Eight consecutive values at column n of a row at p: whole where all are below N, at any alignment.
// (Stores of 16 bytes a lane, 64 neighbouring bytes from four lanes.)
__device__ __forceinline__ void put8(uint16_t *p, uint4 v, int64_t n, int64_t N)
{
    if (n + 8 <= N) {
        __builtin_memcpy(p + n, &v, 16);
    } else {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (n + k < N) p[n + k] = (uint16_t)(w[k >> 1] >> (k & 1) * 16);
    }
}

__device__ __forceinline__ void put4f(float *p, const float (&v)[4], int64_t n, int64_t N)
{
    if (n + 4 <= N) {
        __builtin_memcpy(p + n, v, 16);
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (n + k < N) p[n + k] = v[k];
    }
}

template <typename T> __device__ __forceinline__ uint4 get8(const T *p, int64_t n, int64_t N)
{
    uint4 v = make_uint4(0, 0, 0, 0);
    if (n + 8 <= N) {
        __builtin_memcpy(&v, p + n, 16);
    } else {
        uint32_t w[4] = {};
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (n + k < N) w[k >> 1] |= (uint32_t)p[n + k] << (k & 1) * 16;
        v = make_uint4(w[0], w[1], w[2], w[3]);
    }
    return v;
}

template <int DT> __device__ __forceinline__ uint2 pack4(const float (&v)[4])
{
    using A = Act<DT>;
    if constexpr (DT == STACR_DTYPE_BF16) {  // one instruction a pair
        typedef float F2 __attribute__((ext_vector_type(2)));
        typedef __bf16 B2 __attribute__((ext_vector_type(2)));
        const F2 x = {v[0], v[1]}, y = {v[2], v[3]};
        return make_uint2(__builtin_bit_cast(uint32_t, __builtin_convertvector(x, B2)),
                          __builtin_bit_cast(uint32_t, __builtin_convertvector(y, B2)));
    }
    return make_uint2((uint32_t)A::st(v[0]) | (uint32_t)A::st(v[1]) << 16, (uint32_t)A::st(v[2]) | (uint32_t)A::st(v[3]) << 16);
}

__device__ __forceinline__ uint4 eights(uint2 a, uint2 b)
{
    mm_eights(a.x, b.x);
    mm_eights(a.y, b.y);
    return make_uint4(a.x, a.y, b.x, b.y);
}

// Quads of the neighbouring 16-column blocks a, b of this lane's row, to columns n .. + 31 (below N) of the
// row at p; `in`: the row is there
template <int DT>
__device__ __forceinline__ void put_blocks(void *p, int lane, const float (&a)[4], const float (&b)[4], int64_t n, int64_t N,
                                           bool in)
{
    if constexpr (DT == STACR_DTYPE_F32) {
        if (!in) return;
        put4f(static_cast<float *>(p), a, n + (lane >> 4) * 4, N);
        put4f(static_cast<float *>(p), b, n + 16 + (lane >> 4) * 4, N);
    } else {
        const uint4 v = eights(pack4<DT>(a), pack4<DT>(b));  // every lane takes part
        if (in) put8(static_cast<uint16_t *>(p), v, n + (lane >> 4) * 8, N);
    }
}

// dg or du of the same into a row of [dg | du] (fp32: of its four planes)
template <int DT>
__device__ __forceinline__ void put_slopes(uint16_t *p, int64_t plane, int lane, const float (&a)[4], const float (&b)[4],
                                           int64_t n, int64_t N, bool in)
{
    if constexpr (DT == STACR_DTYPE_F32) {
        uint16_t s[8][kPlanes];
#pragma unroll
        for (int r = 0; r < 4; ++r) split_f32(a[r], s[r]), split_f32(b[r], s[4 + r]);
#pragma unroll
        for (int t = 0; t < kPlanes; ++t) {
            const uint2 x = make_uint2((uint32_t)s[0][t] | (uint32_t)s[1][t] << 16, (uint32_t)s[2][t] | (uint32_t)s[3][t] << 16);
            const uint2 y = make_uint2((uint32_t)s[4][t] | (uint32_t)s[5][t] << 16, (uint32_t)s[6][t] | (uint32_t)s[7][t] << 16);
            const uint4 v = eights(x, y);
            if (in) put8(p + t * plane, v, n + (lane >> 4) * 8, N);
        }
    } else {
        put_blocks<DT>(p, lane, a, b, n, N, in);
    }
}

// A wave's rows, from its first on, of a result whose rows are multiples of 16 bytes: stores without a branch,
// as the buffer's range drops the rows past the last and a column past the last gets an offset past the range.
// For the forward's 8 bytes an output (32768 x 2048 x 8192: 2164 -> 2094 us against stores that each test their
// place; a plain product, with a quarter of that to write, gains nothing by it).
struct EvenRows {
    __amdgpu_buffer_rsrc_t r;
    uint32_t row;  // bytes of a row

    __device__ __forceinline__ EvenRows(void *p, int64_t first, int64_t rows, int64_t bytes)
        : r(mm_rsrc(static_cast<unsigned char *>(p) + first * bytes, (rows - first) * bytes)), row((uint32_t)bytes)
    {
    }
    // this lane's place in the wave's first 16 rows
    __device__ __forceinline__ uint32_t at(int lane, int64_t n, int64_t N, int size) const
    {
        return (lane & 15) * row + (n < N ? (uint32_t)n * size : kMmPast);
    }
    __device__ __forceinline__ void put(uint32_t at, uint4 v) const
    {
        typedef uint32_t U4 __attribute__((ext_vector_type(4)));
        __builtin_amdgcn_raw_buffer_store_b128(U4{v.x, v.y, v.z, v.w}, r, at, 0, 0);
    }
    __device__ __forceinline__ void put(uint32_t at, uint2 v) const
    {
        typedef uint32_t U2 __attribute__((ext_vector_type(2)));
        __builtin_amdgcn_raw_buffer_store_b64(U2{v.x, v.y}, r, at, 0, 0);
    }
};

// As put_blocks, for the wave's rows 16 i + lane % 16
template <int DT>
__device__ __forceinline__ void put_even(const EvenRows &rows, int i, int lane, const float (&a)[4], const float (&b)[4],
                                         int64_t n, int64_t N)
{
    const uint4 v = eights(pack4<DT>(a), pack4<DT>(b));
    rows.put(rows.at(lane, n + (lane >> 4) * 8, N, 2) + i * 16 * rows.row, v);
}

// rows of N 16-bit values, `ld` apart, that are eights of them at multiples of 16 bytes
__device__ __forceinline__ bool even_rows(const void *p, int64_t N, int64_t ld)
{
    return ((N | ld) & 7) == 0 && (reinterpret_cast<uintptr_t>(p) & 15) == 0;
}

// Upper 16 of the 24 bits of two quads of neighbouring blocks, as eights, and the lower 8 of them
__device__ __forceinline__ void to_kept(const float (&a)[4], const float (&b)[4], uint4 &high, uint2 &low)
{
    uint32_t x[4], y[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) x[r] = to_24(a[r]), y[r] = to_24(b[r]);
    // (bytes of __builtin_amdgcn_perm's result: 0 to 3 name the second operand's, 4 to 7 the first's)
    const auto upper = [](uint32_t p, uint32_t q) { return __builtin_amdgcn_perm(q, p, 0x07060302u); };
    const auto lower = [](const uint32_t (&v)[4]) {
        const uint32_t p = __builtin_amdgcn_perm(v[1], v[0], 0x0c0c0501u), q = __builtin_amdgcn_perm(v[3], v[2], 0x05010c0cu);
        return p | q;
    };
    high = eights(make_uint2(upper(x[0], x[1]), upper(x[2], x[3])), make_uint2(upper(y[0], y[1]), upper(y[2], y[3])));
    low = make_uint2(lower(x), lower(y));
    mm_eights(low.x, low.y);
}

// A workgroup takes every gridDim.x-th tile.  Consecutive logical tiles share an XCD (workgroups are dealt
// to the 8 XCDs round-robin, and gridDim.x is a multiple of 8 where there is more than one round) and
// walk `kGroup` tile rows together, so that an XCD's tiles share operands in its L2.
constexpr int kGroup = 8;

template <int DT, bool AK, bool BK, int EPI, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(WM *WN * 64, 1) void k_gated_mm(const MmArgs p)
{
    constexpr int MT = DT == STACR_DTYPE_F16 ? STACR_DTYPE_F16 : STACR_DTYPE_BF16;  // the operands' type
    constexpr int NW = WM * WN, TM = BM / WM, TN = BN / WN, MI = TM / 16, NI = TN / 16;
    constexpr uint32_t kA = BM * 128, kStage = (BM + BN) * 128;
    constexpr bool DUAL = EPI != kStore;
    static_assert(NI % 4 == 0, "results leave in eights of two blocks (of two pairs)");
    extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;

    MmLoader<AK, BM, NW> la;
    MmLoader<BK, BN, NW> lb;
    la.init(lane, wave, p.a.ld);
    lb.init(lane, wave, p.b.ld);
    if constexpr (DUAL) {  // tile rows 32 i .. + 15: gate rows n0 + 16 i .., the next 16 the same up rows
#pragma unroll
        for (int i = 0; i < lb.kPer; ++i) {
            const int row = (wave * lb.kPer + i) * 8 + (lane >> 3);
            lb.off[i] = (uint32_t)((row >> 5) * 16 + (row & 15)) * (uint32_t)p.b.ld * 2 + lb.kc[i & 1] * 2;
        }
    }
    MmReader<AK, BM, MI> ra;
    MmReader<BK, BN, NI> rb;
    ra.init(lane, wm * TM);
    rb.init(lane, wn * TN);
    const int ksteps = (int)((p.K + kMmK - 1) / kMmK), steps = ksteps * p.nseg;

    struct Tile {
        int64_t m0, n0;
        int half, split, begin, count;  // steps begin .. begin + count - 1
    };
    const auto locate = [&](int id) __attribute__((always_inline)) {
        Tile t;
        const int q = p.tiles >> 3, r = p.tiles & 7, x = id & 7;
        id = x * q + (x < r ? x : r) + (id >> 3);
        const int each = p.mt * p.nt * p.halves;
        t.split = id / each;
        id -= t.split * each;
        const int mrows = p.mt * p.halves;
        const int group = id / (kGroup * p.nt), first = group * kGroup;
        const int size = mrows - first < kGroup ? mrows - first : kGroup;
        const int in = id - group * kGroup * p.nt;
        const int mrow = first + in % size;
        t.half = mrow / p.mt;
        t.m0 = (int64_t)(mrow - t.half * p.mt) * BM;
        t.n0 = (int64_t)(in / size) * (DUAL ? BN / 2 : BN);
        t.begin = (int)((int64_t)steps * t.split / p.splits);
        t.count = (int)((int64_t)steps * (t.split + 1) / p.splits) - t.begin;
        return t;
    };

    // The step that is loaded next, and its tile (one step ahead of the one that is multiplied): bytes from
    // the operands' first values of this tile in it to their end bound the reads (rows past the last, K
    // past the last).
    const unsigned char *pa = nullptr, *pb = nullptr, *pb2 = nullptr;
    int64_t left_a = 0, left_b = 0;
    const int64_t step_a = AK ? kMmK * 2 : p.a.ld * (kMmK * 2), step_b = BK ? kMmK * 2 : p.b.ld * (kMmK * 2);
    int ahead = blockIdx.x, seg = 0, ks = 0, todo = 0;
    Tile lt{};
    const auto seek = [&](int s, int k) __attribute__((always_inline)) {
        seg = s;
        ks = k;
        const int64_t k0 = (int64_t)k * kMmK, kpad = (p.K + 7) & ~7ll;
        const int64_t at_a = AK ? lt.m0 * p.a.ld + k0 : k0 * p.a.ld + lt.m0 + lt.half * p.a_half;
        const int64_t at_b = BK ? lt.n0 * p.b.ld + k0 : k0 * p.b.ld + lt.n0;
        const int64_t end_a = AK ? (p.a.extent - 1) * p.a.ld + kpad : (p.K - 1) * p.a.ld + p.a.extent;
        const int64_t end_b = BK ? (p.b.extent - 1) * p.b.ld + kpad : (p.K - 1) * p.b.ld + p.b.extent;
        pa = reinterpret_cast<const unsigned char *>(p.a.seg[s] + at_a);
        pb = reinterpret_cast<const unsigned char *>(p.b.seg[s] + at_b);
        if constexpr (DUAL) pb2 = reinterpret_cast<const unsigned char *>(p.b2[s] + at_b);
        left_a = (end_a - at_a) * 2;
        left_b = (end_b - at_b) * 2;
    };
    const auto open = [&]() __attribute__((always_inline)) {
        lt = locate(ahead);
        todo = lt.count;
        seek(lt.begin / ksteps, lt.begin % ksteps);
    };
    const auto next = [&]() __attribute__((always_inline)) {
        if (--todo > 0) {
            if (++ks < ksteps) {
                pa += step_a;
                pb += step_b;
                if constexpr (DUAL) pb2 += step_b;
                left_a -= step_a;
                left_b -= step_b;
            } else {
                seek(seg + 1, 0);
            }
        } else if ((ahead += gridDim.x) < p.tiles) {
            open();
        } else {
            left_a = left_b = 0;  // nothing more: zeros
            todo = 1;
        }
    };
    const auto load = [&](unsigned char *at) __attribute__((always_inline)) {
        const uint32_t k = (uint32_t)ks * kMmK;
        const auto r = mm_rsrc(pa, left_a);
#pragma unroll
        for (int i = 0; i < la.kPer; ++i)
            mm_copy16(r, at + (wave * la.kPer + i) * 1024, !AK || k + la.kc[i & 1] < (uint32_t)p.K ? la.off[i] : kMmPast);
        const auto s = mm_rsrc(pb, left_b), s2 = mm_rsrc(pb2, left_b);
#pragma unroll
        for (int i = 0; i < lb.kPer; ++i) {
            const bool second = DUAL && ((wave * lb.kPer + i) & 2);  // 8 rows of one copy are of one weight
            mm_copy16(second ? s2 : s, at + kA + (wave * lb.kPer + i) * 1024,
                      !BK || k + lb.kc[i & 1] < (uint32_t)p.K ? lb.off[i] : kMmPast);
        }
    };

    mmf4 acc[MI][NI];
    // One step: the next one's copies into `to`, the products of what is in `from`.  Two pointers that do
    // not alias: without that knowledge the compiler waits for the copies before it reads.
    const auto step = [&](const unsigned char *__restrict__ from, unsigned char *__restrict__ to) {
        load(to);
        __builtin_amdgcn_sched_barrier(0);  // all copies first: among the reads they come late
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            uint4 av[MI], bv[NI];
#pragma unroll
            for (int j = 0; j < NI; ++j) bv[j] = rb.get(from + kA, j, kk, lane);
#pragma unroll
            for (int i = 0; i < MI; ++i) av[i] = ra.get(from, i, kk, lane);
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int j = 0; j < NI; ++j) acc[i][j] = mm_mfma<MT>(bv[j], av[i], acc[i][j]);
        }
        // Reads run two rows of blocks ahead of their products.  (Not where both operands come in halves and two
        // workgroups share a CU: there the compiler's own order was 12 % faster, everywhere else 5 to 12 % slower.)
        if constexpr (AK || BK || MI > 4) {
            constexpr int ra_n = AK ? 1 : 2, rb_n = BK ? 1 : 2;
            constexpr int kAll = 2 * (MI * ra_n + NI * rb_n), kFirst = NI * rb_n + 2 * ra_n;
            constexpr int kEach = (kAll - kFirst + 2 * MI - 4) / (2 * MI - 3);
            __builtin_amdgcn_sched_group_barrier(0x100, kFirst, 0);
#pragma unroll
            for (int i = 0; i < 2 * MI; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x008, NI, 0);
                __builtin_amdgcn_sched_group_barrier(0x100, kEach, 0);
            }
        }
    };

    open();
    load(lds);
    int buf = 0;
    for (int id = blockIdx.x; id < p.tiles; id += gridDim.x) {
        const Tile t = lt;  // the loader enters the next tile with this one's last step
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < NI; ++j) acc[i][j] = mmf4{0.0f, 0.0f, 0.0f, 0.0f};
        for (int it = 0; it < t.count; ++it) {
            next();
            __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0): this wave's copies of this step are in LDS
            asm volatile("s_barrier" ::: "memory");  // and everybody's; the other stage has been read
            step(lds + buf * kStage, lds + (buf ^ 1) * kStage);
            buf ^= 1;
        }

        // a lane holds, of each 16 x 16 block, columns 4 (lane / 16) .. + 3 of row lane % 16
        const int64_t mfirst = t.m0 + wm * TM + (lane & 15);
        const auto quad = [&](const mmf4 &w, float(&v)[4]) __attribute__((always_inline)) {
#pragma unroll
            for (int r = 0; r < 4; ++r) v[r] = w[r];
        };
        if constexpr (EPI == kStore) {
            void *o = t.half ? p.out2 : p.out;
            const bool wide = p.splits > 1 || p.out_dt == STACR_DTYPE_F32;
            if (p.splits > 1) o = p.part + ((int64_t)t.split * p.halves + t.half) * p.M * p.N;
#pragma unroll
            for (int i = 0; i < MI; ++i) {
                const int64_t m = mfirst + i * 16;
#pragma unroll
                for (int j = 0; j < NI; j += 2) {
                    const int64_t n = t.n0 + wn * TN + j * 16;
                    float a[4], b[4];
                    quad(acc[i][j], a);
                    quad(acc[i][j + 1], b);
                    if (wide) put_blocks<STACR_DTYPE_F32>(static_cast<float *>(o) + m * p.N, lane, a, b, n, p.N, m < p.M);
                    else put_blocks<MT>(static_cast<uint16_t *>(o) + m * p.N, lane, a, b, n, p.N, m < p.M);
                }
            }
        } else {
            constexpr bool EXACT = DT == STACR_DTYPE_F32;
            using T = typename Act<DT>::T;
            const int64_t f0 = t.n0 + wn * (TN / 2);  // blocks (0, 1) of NI: gate and up of 16 outputs from f0 on
            if (p.bias_g || p.bias_u) {
#pragma unroll
                for (int j = 0; j < NI; j += 2)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int64_t f = f0 + j * 8 + (lane >> 4) * 4 + r;
                        const float bg = p.bias_g && f < p.N ? load_any(p.bias_g, DT, f) : 0.0f;
                        const float bu = p.bias_u && f < p.N ? load_any(p.bias_u, DT, f) : 0.0f;
#pragma unroll
                        for (int i = 0; i < MI; ++i) acc[i][j][r] += bg, acc[i][j + 1][r] += bu;
                    }
            }
            if constexpr (EPI == kFwd) {
                const bool even = even_rows(p.out, p.N, p.ldo);
                const EvenRows rows(p.out, t.m0 + wm * TM, p.M, p.ldo * 2);
                with_activation(p.act, [&](auto c) __attribute__((always_inline)) {
#pragma unroll
                    for (int i = 0; i < MI; ++i) {
                        const int64_t m = mfirst + i * 16;
#pragma unroll
                        for (int j = 0; j < NI; j += 4) {
                            float h[2][4];
#pragma unroll
                            for (int b = 0; b < 2; ++b)
#pragma unroll
                                for (int r = 0; r < 4; ++r) {
                                    float a, slope;
                                    activate<EXACT, decltype(c)::value>(acc[i][j + 2 * b][r], a, slope);
                                    h[b][r] = a * acc[i][j + 2 * b + 1][r];
                                }
                            if constexpr (!EXACT) {
                                if (even) {
                                    put_even<DT>(rows, i, lane, h[0], h[1], f0 + j * 8, p.N);
                                    continue;
                                }
                            }
                            put_blocks<DT>(static_cast<T *>(p.out) + m * p.ldo, lane, h[0], h[1], f0 + j * 8, p.N, m < p.M);
                        }
                    }
                });
                if (p.gate) {  // rows of ff_pad values, a multiple of 8
                    const int64_t first = t.m0 + wm * TM;
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        void *o = u ? p.up : p.gate;
                        const EvenRows k(o, first, p.M, p.ff_pad * 2);
                        const EvenRows l(u ? p.up_low : p.gate_low, first, p.gate_low ? p.M : first, p.ff_pad);
#pragma unroll
                        for (int j = 0; j < NI; j += 4) {
                            const int64_t f = f0 + j * 8;
                            const uint32_t at = k.at(lane, f + (lane >> 4) * 8, p.ff_pad, 2);
                            const uint32_t low = l.at(lane, f + (lane >> 4) * 8, p.ff_pad, 1);
#pragma unroll
                            for (int i = 0; i < MI; ++i) {
                                float a[4], b[4];
                                quad(acc[i][j + u], a);
                                quad(acc[i][j + 2 + u], b);
                                if constexpr (EXACT) {
                                    const int64_t m = mfirst + i * 16;
                                    put_blocks<DT>(static_cast<T *>(o) + m * p.ff_pad, lane, a, b, f, p.ff_pad, m < p.M);
                                } else if (p.gate_low) {
                                    uint4 v;
                                    uint2 w;
                                    to_kept(a, b, v, w);
                                    k.put(at + i * 16 * k.row, v);
                                    l.put(low + i * 16 * l.row, w);
                                } else {
                                    k.put(at + i * 16 * k.row, eights(pack4<DT>(a), pack4<DT>(b)));
                                }
                            }
                        }
                    }
                }
            } else {
                with_activation(p.act, [&](auto c) __attribute__((always_inline)) {
#pragma unroll
                    for (int i = 0; i < MI; ++i) {
                        __builtin_amdgcn_sched_barrier(0);  // a row of blocks at a time: all at once spill
                        const int64_t m = mfirst + i * 16;
#pragma unroll
                        for (int j = 0; j < NI; j += 4) {
                            const int64_t f = f0 + j * 8;
                            float d[2][4] = {}, dg[2][4], du[2][4];
                            if constexpr (EXACT) {
#pragma unroll
                                for (int b = 0; b < 2; ++b)
#pragma unroll
                                    for (int r = 0; r < 4; ++r) {
                                        const int64_t n = f + b * 16 + (lane >> 4) * 4 + r;
                                        if (m < p.M && n < p.N) d[b][r] = static_cast<const float *>(p.dh)[m * p.ldo + n];
                                    }
                            } else {
                                uint4 w = make_uint4(0, 0, 0, 0);
                                if (m < p.M) w = get8(static_cast<const T *>(p.dh) + m * p.ldo, f + (lane >> 4) * 8, p.N);
                                mm_quads(w.x, w.z);
                                mm_quads(w.y, w.w);
                                const uint32_t q[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                                for (int e = 0; e < 8; ++e) d[e >> 2][e & 3] = Act<DT>::ld((T)(q[e >> 1] >> (e & 1) * 16));
                            }
#pragma unroll
                            for (int b = 0; b < 2; ++b)
#pragma unroll
                                for (int r = 0; r < 4; ++r) {
                                    float a, slope;
                                    activate<EXACT, decltype(c)::value>(acc[i][j + 2 * b][r], a, slope);
                                    dg[b][r] = d[b][r] * acc[i][j + 2 * b + 1][r] * slope;
                                    du[b][r] = d[b][r] * a;
                                }
                            uint16_t *row = p.dgu + m * 2 * p.ff_pad;
                            put_slopes<DT>(row, p.plane, lane, dg[0], dg[1], f, p.ff_pad, m < p.M);
                            put_slopes<DT>(row + p.ff_pad, p.plane, lane, du[0], du[1], f, p.ff_pad, m < p.M);
                        }
                    }
                });
            }
        }
    }
    __builtin_amdgcn_s_waitcnt(0x0070);  // the copies past the end
}

// sum of the partial products over the splits, in order, rounded once
template <int DT>
__global__ __launch_bounds__(kBlock) void k_gated_join(const float *__restrict__ part, int splits, int64_t size,
                                                       int64_t half_size, void *out, void *out2)
{
    for (int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x; i < size; i += (int64_t)gridDim.x * kBlock) {
        float v = 0.0f;
        for (int s = 0; s < splits; ++s) v += part[s * size + i];
        const bool second = i >= half_size;
        static_cast<typename Act<DT>::T *>(second ? out2 : out)[second ? i - half_size : i] = Act<DT>::st(v);
    }
}

// ------------------------------------------------------------------ operands that need another form
// rows x cols of `src` (row stride ld) as rows of ld_dst (a multiple of 8, zeros past cols): fp32 as its
// four bf16 planes, 16-bit types as they are; up to three matrices a launch (grid.y)
struct PackOne {
    const void *src;
    int64_t ld, rows;
    uint16_t *dst;
    bool vec;
};
struct PackArgs {
    PackOne m[3];
    int64_t cols, ld_dst;
};

template <int DT> __global__ __launch_bounds__(kBlock) void k_gated_pack(const PackArgs p)
{
    const PackOne o = p.m[blockIdx.y];
    const void *__restrict__ src = o.src;
    uint16_t *__restrict__ dst = o.dst;
    const int64_t ld = o.ld, cols = p.cols, ld_dst = p.ld_dst;
    const bool vec = o.vec;
    const int64_t chunks = ld_dst / 8, n = o.rows * chunks, plane = o.rows * ld_dst;
    for (int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x; i < n; i += (int64_t)gridDim.x * kBlock) {
        const int64_t row = i / chunks, c = (i - row * chunks) * 8;
        if constexpr (DT == STACR_DTYPE_F32) {
            const float *s = static_cast<const float *>(src) + row * ld + c;
            float v[8];
            if (vec && c + 7 < cols) {
                const float4 lo = *reinterpret_cast<const float4 *>(s), hi = *reinterpret_cast<const float4 *>(s + 4);
                v[0] = lo.x; v[1] = lo.y; v[2] = lo.z; v[3] = lo.w;
                v[4] = hi.x; v[5] = hi.y; v[6] = hi.z; v[7] = hi.w;
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = c + e < cols ? s[e] : 0.0f;
            }
            uint16_t q[8][kPlanes];
#pragma unroll
            for (int e = 0; e < 8; ++e) split_f32(v[e], q[e]);
#pragma unroll
            for (int t = 0; t < kPlanes; ++t)
                *reinterpret_cast<uint4 *>(dst + t * plane + row * ld_dst + c) =
                    make_uint4((uint32_t)q[0][t] | (uint32_t)q[1][t] << 16, (uint32_t)q[2][t] | (uint32_t)q[3][t] << 16,
                               (uint32_t)q[4][t] | (uint32_t)q[5][t] << 16, (uint32_t)q[6][t] | (uint32_t)q[7][t] << 16);
        } else {
            const uint16_t *s = static_cast<const uint16_t *>(src) + row * ld + c;
            uint32_t v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = c + e < cols ? s[e] : 0u;
            *reinterpret_cast<uint4 *>(dst + row * ld_dst + c) =
                make_uint4(v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16);
        }
    }
}

// ------------------------------------------------------------------ kept pre-activations
// [dg | du] from dh and the kept g and u, eight values a thread; LOW: g and u in 24 bits; plain: fp32
// values beside their planes, or NULL.  PAST: more than the caches hold; what the pass reads, it reads for the
// last time, and past the caches it leaves [dg | du] in them for the two products that follow (8192 x 1024 x
// 4096: the pass 89 -> 71 us, dx 167 -> 146, dW 133 -> 128).
template <int DT, bool LOW, bool PAST>
__global__ __launch_bounds__(kBlock) void k_gated_slopes(const void *__restrict__ dh, const void *__restrict__ gate,
                                                         const void *__restrict__ up, const uint8_t *__restrict__ gate_low,
                                                         const uint8_t *__restrict__ up_low, int64_t rows, int64_t ff, int act,
                                                         uint16_t *__restrict__ dgu, int64_t ff_pad, int64_t plane,
                                                         float *__restrict__ plain)
{
    using T = typename Act<DT>::T;
    typedef uint32_t u2 __attribute__((ext_vector_type(2)));
    constexpr bool EXACT = DT == STACR_DTYPE_F32;
    const int64_t eighths = ff_pad / 8, n = rows * eighths;
    const auto read16 = [](const auto *p) __attribute__((always_inline)) {
        if constexpr (PAST) return load16_stream(p);
        else return *reinterpret_cast<const uint4 *>(p);
    };
    with_activation(act, [&](auto c) __attribute__((always_inline)) {
        for (int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x; i < n; i += (int64_t)gridDim.x * kBlock) {
            const int64_t m = i / eighths, f = (i - m * eighths) * 8, at = m * ff_pad + f;
            const int have = ff - f < 8 ? (int)(ff - f) : 8;  // outputs; the rest of the padded row gets zeros
            const auto read = [&](const void *src, const uint8_t *low, float(&v)[8]) __attribute__((always_inline)) {
                if constexpr (EXACT) {
                    const float *p = static_cast<const float *>(src) + at;
                    const uint4 lo = read16(p), hi = read16(p + 4);
                    __builtin_memcpy(v, &lo, 16);
                    __builtin_memcpy(v + 4, &hi, 16);
                } else {
                    const uint4 w = read16(static_cast<const T *>(src) + at);
                    const uint32_t q[4] = {w.x, w.y, w.z, w.w};
                    u2 b = {0, 0};
                    if constexpr (LOW) b = __builtin_nontemporal_load(reinterpret_cast<const u2 *>(low + at));
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const uint32_t h = q[k >> 1] >> (k & 1) * 16 & 0xffffu;
                        if constexpr (LOW) v[k] = __uint_as_float(h << 16 | ((k < 4 ? b.x : b.y) >> (k & 3) * 8 & 255u) << 8);
                        else v[k] = Act<DT>::ld((T)h);
                    }
                }
            };
            float d[8], g[8], u[8], dg[8], du[8];
            if constexpr (EXACT) {
#pragma unroll
                for (int k = 0; k < 8; ++k) d[k] = k < have ? static_cast<const float *>(dh)[m * ff + f + k] : 0.0f;
            } else {
                const T *p = static_cast<const T *>(dh) + m * ff + f;
                const uint4 w = have == 8 && PAST ? load16_stream(p) : get8(p, 0, have);
                const uint32_t q[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int k = 0; k < 8; ++k) d[k] = Act<DT>::ld((T)(q[k >> 1] >> (k & 1) * 16));
            }
            read(gate, gate_low, g);
            read(up, up_low, u);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                float a, slope;
                activate<EXACT, decltype(c)::value>(g[k], a, slope);
                dg[k] = k < have ? d[k] * u[k] * slope : 0.0f;
                du[k] = k < have ? d[k] * a : 0.0f;
            }
            uint16_t *row = dgu + m * 2 * ff_pad + f;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const float(&v)[8] = half ? du : dg;
                uint16_t *o = row + half * ff_pad;
                if constexpr (EXACT) {
                    if (plain) __builtin_memcpy(plain + (m * 2 + half) * ff_pad + f, v, 32);
                    uint16_t s[8][kPlanes];
#pragma unroll
                    for (int k = 0; k < 8; ++k) split_f32(v[k], s[k]);
#pragma unroll
                    for (int t = 0; t < kPlanes; ++t)
                        *reinterpret_cast<uint4 *>(o + t * plane) =
                            make_uint4((uint32_t)s[0][t] | (uint32_t)s[1][t] << 16, (uint32_t)s[2][t] | (uint32_t)s[3][t] << 16,
                                       (uint32_t)s[4][t] | (uint32_t)s[5][t] << 16, (uint32_t)s[6][t] | (uint32_t)s[7][t] << 16);
                } else {
                    const float lo[4] = {v[0], v[1], v[2], v[3]}, hi[4] = {v[4], v[5], v[6], v[7]};
                    const uint2 x = pack4<DT>(lo), y = pack4<DT>(hi);
                    *reinterpret_cast<uint4 *>(o) = make_uint4(x.x, x.y, y.x, y.y);
                }
            }
        }
    });
}

// ------------------------------------------------------------------ bias gradients
// column sums of [dg | du]: partial sums over row ranges of kBiasRows, then their sum in order.  A
// workgroup takes 256 columns of a range: 32 threads of 8 columns, eight rows apart (3001 x 5464 fp16: 7.3 us,
// 4.5 TB/s; ranges of 128 rows with eight loads on the way: 8.2), and then 32 columns of the partial sums, eight
// threads each (one thread a column, whose loads wait for one another: 7.3 us, now 3.9).
constexpr int kBiasRows = 256;

template <int DT>
__global__ __launch_bounds__(kBlock) void k_gated_bias_part(const uint16_t *__restrict__ dgu, int64_t rows, int64_t ff_pad,
                                                            int64_t plane, float *__restrict__ part)
{
    __shared__ float s[8][256 + 4];
    constexpr int PL = DT == STACR_DTYPE_F32 ? 3 : 1;
    const int64_t cols = 2 * ff_pad, c = (int64_t)blockIdx.x * 256 + (threadIdx.x & 31) * 8;
    const int64_t r0 = (int64_t)blockIdx.y * kBiasRows, r1 = r0 + kBiasRows < rows ? r0 + kBiasRows : rows;
    float sum[8] = {};
    if (c < cols) {
#pragma unroll 4
        for (int64_t r = r0 + (threadIdx.x >> 5); r < r1; r += 8) {
            const uint16_t *p = dgu + r * cols + c;
            float v[PL][8];
#pragma unroll
            for (int t = 0; t < PL; ++t) load_vec<DT == STACR_DTYPE_F32 ? STACR_DTYPE_BF16 : DT, 8>(p + t * plane, v[t]);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if constexpr (PL == 3) sum[e] += v[0][e] + (v[1][e] + v[2][e]);
                else sum[e] += v[0][e];
            }
        }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) s[threadIdx.x >> 5][(threadIdx.x & 31) * 8 + e] = sum[e];
    __syncthreads();
    float v = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; ++k) v += s[k][threadIdx.x];
    const int64_t out = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (out < cols) part[(int64_t)blockIdx.y * cols + out] = v;
}

template <int DT>
__global__ __launch_bounds__(kBlock) void k_gated_bias_sum(const float *__restrict__ part, int parts, int64_t ff,
                                                           int64_t ff_pad, void *db_gate, void *db_up)
{
    __shared__ float s[8][32];
    const int half = blockIdx.y, col = threadIdx.x & 31, lane = threadIdx.x >> 5;
    const int64_t f = (int64_t)blockIdx.x * 32 + col;
    void *out = half ? db_up : db_gate;
    if (!out) return;
    float sum = 0.0f;
    if (f < ff) {
#pragma unroll 8
        for (int i = lane; i < parts; i += 8) sum += part[(int64_t)i * 2 * ff_pad + half * ff_pad + f];
    }
    s[lane][col] = sum;
    __syncthreads();
    if (lane || f >= ff) return;
    sum = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; ++k) sum += s[k][col];
    static_cast<typename Act<DT>::T *>(out)[f] = Act<DT>::st(sum);
}

// ------------------------------------------------------------------ few rows
// Eight consecutive values of a row at p (k .. k + 7, zeros from `left` on) as matrix-core operands.
template <int DT, bool VEC>
__device__ __forceinline__ void few_load(const void *base, int64_t at, int64_t left, uint4 (&o)[DT == STACR_DTYPE_F32 ? 4 : 1])
{
    if constexpr (DT == STACR_DTYPE_F32) {
        const float *p = static_cast<const float *>(base) + at;
        float v[8];
        if constexpr (VEC) {
            float4 lo = make_float4(0, 0, 0, 0), hi = lo;
            if (left > 0) lo = *reinterpret_cast<const float4 *>(p), hi = *reinterpret_cast<const float4 *>(p + 4);
            v[0] = lo.x; v[1] = lo.y; v[2] = lo.z; v[3] = lo.w;
            v[4] = hi.x; v[5] = hi.y; v[6] = hi.z; v[7] = hi.w;
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = e < left ? p[e] : 0.0f;
        }
        uint16_t q[8][kPlanes];
#pragma unroll
        for (int e = 0; e < 8; ++e) split_f32(v[e], q[e]);
#pragma unroll
        for (int t = 0; t < kPlanes; ++t)
            o[t] = make_uint4((uint32_t)q[0][t] | (uint32_t)q[1][t] << 16, (uint32_t)q[2][t] | (uint32_t)q[3][t] << 16,
                              (uint32_t)q[4][t] | (uint32_t)q[5][t] << 16, (uint32_t)q[6][t] | (uint32_t)q[7][t] << 16);
    } else {
        const uint16_t *p = static_cast<const uint16_t *>(base) + at;
        if constexpr (VEC) {
            o[0] = left > 0 ? *reinterpret_cast<const uint4 *>(p) : make_uint4(0, 0, 0, 0);
        } else {
            uint32_t v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = e < left ? p[e] : 0u;
            o[0] = make_uint4(v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16);
        }
    }
}

struct FewArgs {
    const void *x, *wg, *wu, *bias_g, *bias_u;
    int64_t rows, d, x_ld, ff;
    int act;
    void *h, *gate, *up;
    uint8_t *gate_low, *up_low;
};

// NT: blocks of 16 rows.  VEC: d and every row start are multiples of 8 values.
template <int DT, int NT, bool VEC>
__global__ __launch_bounds__(kBlock) void k_gated_few(const FewArgs p)
{
    constexpr int MT = DT == STACR_DTYPE_F16 ? STACR_DTYPE_F16 : STACR_DTYPE_BF16;
    constexpr int P = DT == STACR_DTYPE_F32 ? kPlanes : 1;
    __shared__ float red[kWaves][2 * NT][64][4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t f0 = (int64_t)blockIdx.x * 16;
    const int64_t f = f0 + (lane & 15) < p.ff ? f0 + (lane & 15) : p.ff - 1;
    int64_t xrow[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int64_t m = t * 16 + (lane & 15);
        xrow[t] = (m < p.rows ? m : p.rows - 1) * p.x_ld;
    }
    mmf4 ag[NT], au[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) ag[t] = au[t] = mmf4{0.0f, 0.0f, 0.0f, 0.0f};
    // U blocks of 32 of K a wave at a time, their loads all on the way before the first product (a loop over
    // single blocks is not unrolled: matrix instructions do not allow a remainder loop).  One token through
    // 1024 -> 4096: 7.7 us with one block at a time, 7.0 with eight, by events around the launch (the kernel itself
    // 4.9 us: 3.4 TB/s of weights that the caches may hold, so its start and its end count as much as the reads).
    constexpr int U = DT == STACR_DTYPE_F32 || !VEC ? 2 : NT == 4 ? 4 : 8;
    const int64_t d = p.d;
    const auto blocks = [&](int64_t k0, auto whole) __attribute__((always_inline)) {
        uint4 g[U][P], u[U][P], x[U][NT][P];
#pragma unroll
        for (int b = 0; b < U; ++b) {
            const int64_t k = k0 + b * 32 + (lane >> 4) * 8, left = decltype(whole)::value ? 8 : d - k;
            few_load<DT, VEC>(p.wg, f * d + k, left, g[b]);
            few_load<DT, VEC>(p.wu, f * d + k, left, u[b]);
#pragma unroll
            for (int t = 0; t < NT; ++t) few_load<DT, VEC>(p.x, xrow[t] + k, left, x[b][t]);
        }
#pragma unroll
        for (int b = 0; b < U; ++b)
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                if constexpr (DT == STACR_DTYPE_F32) {
#pragma unroll
                    for (int q = 0; q < kPairs; ++q) {
                        ag[t] = mm_mfma<MT>(g[b][kPairB[q]], x[b][t][kPairA[q]], ag[t]);
                        au[t] = mm_mfma<MT>(u[b][kPairB[q]], x[b][t][kPairA[q]], au[t]);
                    }
                } else {
                    ag[t] = mm_mfma<MT>(g[b][0], x[b][t][0], ag[t]);
                    au[t] = mm_mfma<MT>(u[b][0], x[b][t][0], au[t]);
                }
            }
    };
    for (int64_t k0 = wave * (U * 32); k0 < d; k0 += kWaves * (U * 32)) {
        if (k0 + U * 32 <= d) blocks(k0, std::true_type());
        else blocks(k0, std::false_type());
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) red[wave][2 * t][lane][r] = ag[t][r], red[wave][2 * t + 1][lane][r] = au[t][r];
    __syncthreads();
    // output (f0 + i, row m): lane (i / 4) * 16 + m % 16, value i % 4
    for (int o = threadIdx.x; o < NT * 256; o += kBlock) {
        const int i = o & 15, mm = (o >> 4) & 15, t = o >> 8;
        const int64_t m = t * 16 + mm, ff = f0 + i;
        if (m >= p.rows || ff >= p.ff) continue;
        const int l = (i >> 2) * 16 + mm, r = i & 3;
        float g = 0.0f, u = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) g += red[w][2 * t][l][r], u += red[w][2 * t + 1][l][r];
        if (p.bias_g) g += load_any(p.bias_g, DT, ff);
        if (p.bias_u) u += load_any(p.bias_u, DT, ff);
        float a, slope;
        activate<DT == STACR_DTYPE_F32>(p.act, g, a, slope);
        store_any(p.h, DT, m * p.ff + ff, a * u);
        if (p.gate) {
            const int64_t at = m * ((p.ff + 7) & ~7ll) + ff;
            if (DT != STACR_DTYPE_F32 && p.gate_low) {
                const uint32_t x = to_24(g), y = to_24(u);
                static_cast<uint16_t *>(p.gate)[at] = (uint16_t)(x >> 16);
                static_cast<uint16_t *>(p.up)[at] = (uint16_t)(y >> 16);
                p.gate_low[at] = (uint8_t)(x >> 8);
                p.up_low[at] = (uint8_t)(y >> 8);
            } else {
                store_any(p.gate, DT, at, g);
                store_any(p.up, DT, at, u);
            }
        }
    }
}

// Rows up to which the forward takes k_gated_few.
constexpr int64_t kFewRows = 64;

// ------------------------------------------------------------------ host side
constexpr int kCus = 256;
constexpr int64_t kMaxFeatures = 1 << 20;  // row strides whose tile offsets stay within 31 bits

inline int64_t up_to(int64_t n, int64_t m) { return (n + m - 1) / m * m; }
inline size_t aligned(size_t n) { return (n + 255) & ~(size_t)255; }

bool aligned_to(const void *p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

struct Problem {
    int dt;
    int64_t rows, d, ff, x_ld;
    int64_t d_pad, ff_pad;
    bool pack_x, pack_w;  // another form of x / the weights is needed
};

Problem problem(int dt, int64_t rows, int64_t d, int64_t ff, int64_t x_ld, const void *x, const void *wg, const void *wu)
{
    Problem q{dt, rows, d, ff, x_ld, up_to(d, 8), up_to(ff, 8), false, false};
    const bool wide = dt == STACR_DTYPE_F32;
    q.pack_x = wide || d % 8 || x_ld % 8 || !aligned_to(x, 16);
    q.pack_w = wide || d % 8 || !aligned_to(wg, 16) || !aligned_to(wu, 16);
    return q;
}

template <auto Kernel> void raise_lds(size_t bytes)
{
    static const hipError_t done = hipFuncSetAttribute(reinterpret_cast<const void *>(Kernel),
                                                       hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    (void)done;  // a launch that it does not allow fails by itself
}

template <int DT, bool AK, bool BK, int EPI, int BM, int BN, int WM, int WN>
void mm_run(MmArgs p, int a_cu, hipStream_t s)
{
    constexpr size_t lds = 2 * (BM + BN) * 128;
    static_assert(lds <= 160 * 1024, "LDS budget");
    p.mt = (int)((p.M + BM - 1) / BM);
    const int64_t cols = EPI == kBwd ? p.ff_pad : p.N;
    p.nt = (int)((cols + (EPI == kStore ? BN : BN / 2) - 1) / (EPI == kStore ? BN : BN / 2));
    p.tiles = p.mt * p.nt * p.halves * p.splits;
    constexpr auto kernel = k_gated_mm<DT, AK, BK, EPI, BM, BN, WM, WN>;
    raise_lds<kernel>(lds);
    const int grid = hmin(p.tiles, kCus * a_cu);
    const char *name = EPI == kFwd ? "k_gated_mm_forward" : EPI == kBwd ? "k_gated_mm_slopes"
                       : BK || AK ? "k_gated_mm_input" : "k_gated_mm_weights";
    stacr_launch(name, s, [&] { kernel<<<grid, WM * WN * 64, lds, s>>>(p); });
}

int64_t tiles(int64_t m, int64_t n, int bm, int bn) { return ((m + bm - 1) / bm) * ((n + bn - 1) / bn); }

// The tile of a product and how many workgroups share its K, by what they cost, in steps of a 256 x 256
// tile (1.7 us): a round is as many tiles as the chip holds at once, a tile costs its steps and about 6 more
// for its start and its results; partial products are written and read again (8192 x 1024 in two: 20 us).
//   256 x 256   8 waves, one workgroup a CU: 1 a step
//   256 x 128   8 waves, one workgroup a CU: 0.66 for half the work (LDS and L2 move 1.5 times as much for it)
//   128 x 128   4 waves, two workgroups a CU: 0.6 for both, half the work together
// (8192 x 1024 of K 8192, 128 tiles of 256 x 256: 130 us and 20 to join two splits; 256 of 256 x 128: 150 us;
// 512 of 128 x 128: 130 to 142 us.  Forward, the three in this order: 8192 x 1024 x 4096 187, 211 and 209 us,
// 3001 x 1000 x 2731 in fp16 83, 79 and 73 us.)
struct ProductPlan {
    int tile, splits;
};

ProductPlan product_plan(int64_t m, int64_t n, int halves, int64_t k, int nseg, bool dual)
{
    const int64_t steps = hmax<int64_t>(1, (k + kMmK - 1) / kMmK * nseg);
    const double cost[3] = {1.0, 0.66, 0.6};
    const int bm[3] = {256, 256, 128}, bn[3] = {256, 128, 128}, slots[3] = {kCus, kCus, 2 * kCus};
    ProductPlan best{0, 1};
    double least = 1e300;
    for (int t = 0; t < 3; ++t) {
        const int64_t each = tiles(m, n, bm[t], dual ? bn[t] / 2 : bn[t]) * halves;
        for (int s = 1; s <= (dual ? 1 : 16) && s * 4 <= steps + 3; ++s) {
            const int64_t rounds = (each * s + slots[t] - 1) / slots[t];
            double c = rounds * ((double)((steps + s - 1) / s) + 6.0) * cost[t];
            if (s > 1) c += 2.5 + (double)m * n * halves * 8.0 * s / 7.0e6 / 1.7;
            if (c < least) least = c, best = ProductPlan{t, s};
        }
    }
    return best;
}

template <int DT, bool AK, bool BK, int EPI> void tiled(const MmArgs &p, int tile, hipStream_t s)
{
    if (tile == 0) mm_run<DT, AK, BK, EPI, 256, 256, 2, 4>(p, 1, s);
    else if (tile == 1) mm_run<DT, AK, BK, EPI, 256, 128, 4, 2>(p, 1, s);
    else mm_run<DT, AK, BK, EPI, 128, 128, 2, 2>(p, 2, s);
}

template <int DT, int EPI> void dual(const MmArgs &p, hipStream_t s)
{
    tiled<DT, true, true, EPI>(p, product_plan(p.M, p.N, 1, p.K, p.nseg, true).tile, s);
}

size_t part_bytes(const ProductPlan &q, int64_t m, int64_t n, int halves)
{
    return q.splits > 1 ? aligned((size_t)q.splits * halves * m * n * 4) : 0;
}

// The workspace's pieces, in order; x and the weights as other forms, [dg | du], partial sums.
struct Pieces {
    size_t x, wg, wu, dgu, part, total;
};

int planes(int dt) { return dt == STACR_DTYPE_F32 ? kPlanes : 1; }
int pairs(int dt) { return dt == STACR_DTYPE_F32 ? kPairs : 1; }

Pieces pieces(const Problem &q, bool backward)
{
    Pieces w{};
    size_t at = 0;
    const int pl = planes(q.dt);
    const bool few = !backward && q.rows <= kFewRows;
    w.x = at;
    if (q.pack_x && !few) at += aligned((size_t)pl * q.rows * q.d_pad * 2);
    w.wg = at;
    if (q.pack_w && !few) at += aligned((size_t)pl * q.ff * q.d_pad * 2);
    w.wu = at;
    if (q.pack_w && !few) at += aligned((size_t)pl * q.ff * q.d_pad * 2);
    w.dgu = at;
    if (backward) at += aligned((size_t)pl * q.rows * 2 * q.ff_pad * 2);
    w.part = at;
    if (backward) {
        const size_t dx = part_bytes(product_plan(q.rows, q.d, 1, q.ff_pad, 2 * pairs(q.dt), false), q.rows, q.d, 1);
        const size_t dw = part_bytes(product_plan(q.ff, q.d, 2, q.rows, pairs(q.dt), false), q.ff, q.d, 2);
        const size_t db = aligned((size_t)((q.rows + kBiasRows - 1) / kBiasRows) * 2 * q.ff_pad * 4);
        at += hmax(hmax(dx, dw), db);
    }
    w.total = at;
    return w;
}

// One element (or piece) a thread.  (4096 workgroups that loop, each time a power of two further on, met in
// the same memory channels: 268 M slopes took 770 us, 617 without the loop.)
int blocks_for(int64_t n) { return (int)hmin<int64_t>((n + kBlock - 1) / kBlock, 1 << 30); }

template <int DT, int NT> void few_launch(const FewArgs &a, bool vec, hipStream_t s)
{
    const int grid = (int)((a.ff + 15) / 16);
    stacr_launch("k_gated_few", s, [&] {
        if (vec) k_gated_few<DT, NT, true><<<grid, kBlock, 0, s>>>(a);
        else k_gated_few<DT, NT, false><<<grid, kBlock, 0, s>>>(a);
    });
}

template <int DT> void few_typed(const FewArgs &a, bool vec, hipStream_t s)
{
    if (a.rows <= 16) few_launch<DT, 1>(a, vec, s);
    else if (a.rows <= 32) few_launch<DT, 2>(a, vec, s);
    else few_launch<DT, 4>(a, vec, s);
}

// the weights and x as the products' operands, packed where they have to be
struct Operands {
    const uint16_t *x, *wg, *wu;
    int64_t x_ld, w_ld;
    size_t x_plane, w_plane;
};

Operands operands(const Problem &q, const void *x, const void *wg, const void *wu, char *ws, const Pieces &w, bool need_x,
                  bool need_w, hipStream_t s)
{
    Operands o{};
    o.x = static_cast<const uint16_t *>(x);
    o.wg = static_cast<const uint16_t *>(wg);
    o.wu = static_cast<const uint16_t *>(wu);
    o.x_ld = q.x_ld;
    o.w_ld = q.d;
    PackArgs a{};
    a.cols = q.d;
    a.ld_dst = q.d_pad;
    int count = 0;
    int64_t most = 0;
    const auto pack = [&](const void *src, int64_t ld, int64_t rows, size_t at) {
        uint16_t *dst = reinterpret_cast<uint16_t *>(ws + at);
        a.m[count++] = PackOne{src, ld, rows, dst, aligned_to(src, 16) && ld % 4 == 0};
        most = hmax(most, rows * q.d_pad / 8);
        return dst;
    };
    if (q.pack_x && need_x) {
        o.x = pack(x, q.x_ld, q.rows, w.x);
        o.x_ld = q.d_pad;
        o.x_plane = (size_t)q.rows * q.d_pad;
    }
    if (q.pack_w && need_w) {
        o.wg = pack(wg, q.d, q.ff, w.wg);
        o.wu = pack(wu, q.d, q.ff, w.wu);
        o.w_ld = q.d_pad;
        o.w_plane = (size_t)q.ff * q.d_pad;
    }
    if (count)
        stacr_launch("k_gated_pack", s, [&] {
            const dim3 grid((unsigned)blocks_for(most), (unsigned)count);
            if (q.dt == STACR_DTYPE_F32) k_gated_pack<STACR_DTYPE_F32><<<grid, kBlock, 0, s>>>(a);
            else k_gated_pack<STACR_DTYPE_BF16><<<grid, kBlock, 0, s>>>(a);
        });
    return o;
}

// x [Wg; Wu]^T for either gated epilogue
MmArgs gated_args(const Problem &q, const Operands &o, const void *bg, const void *bu, int act)
{
    MmArgs p{};
    p.nseg = pairs(q.dt);
    for (int i = 0; i < p.nseg; ++i) {
        const int pa = p.nseg > 1 ? kPairA[i] : 0, pb = p.nseg > 1 ? kPairB[i] : 0;
        p.a.seg[i] = o.x + pa * o.x_plane;
        p.b.seg[i] = o.wg + pb * o.w_plane;
        p.b2[i] = o.wu + pb * o.w_plane;
    }
    p.a.ld = o.x_ld;
    p.a.extent = q.rows;
    p.b.ld = o.w_ld;
    p.b.extent = q.ff;
    p.M = q.rows;
    p.N = q.ff;
    p.K = q.d_pad;
    p.halves = p.splits = 1;
    p.ldo = q.ff;
    p.bias_g = bg;
    p.bias_u = bu;
    p.act = act;
    p.ff_pad = q.ff_pad;
    return p;
}

template <int EPI> void dual_typed(int dt, const MmArgs &p, hipStream_t s)
{
    if (dt == STACR_DTYPE_F32) dual<STACR_DTYPE_F32, EPI>(p, s);
    else if (dt == STACR_DTYPE_BF16) dual<STACR_DTYPE_BF16, EPI>(p, s);
    else dual<STACR_DTYPE_F16, EPI>(p, s);
}

template <bool AK>
void product_typed(int dt, MmArgs p, const ProductPlan &plan, float *part, hipStream_t s)
{
    p.splits = plan.splits;
    p.part = part;
    p.out_dt = dt;
    if (dt == STACR_DTYPE_F16) tiled<STACR_DTYPE_F16, AK, false, kStore>(p, plan.tile, s);
    else tiled<STACR_DTYPE_BF16, AK, false, kStore>(p, plan.tile, s);
    if (plan.splits > 1) {
        const int64_t half = p.M * p.N, n = half * p.halves;
        stacr_launch("k_gated_join", s, [&] {
            if (dt == STACR_DTYPE_F32)
                k_gated_join<STACR_DTYPE_F32><<<blocks_for(n), kBlock, 0, s>>>(part, plan.splits, n, half, p.out, p.out2);
            else if (dt == STACR_DTYPE_BF16)
                k_gated_join<STACR_DTYPE_BF16><<<blocks_for(n), kBlock, 0, s>>>(part, plan.splits, n, half, p.out, p.out2);
            else k_gated_join<STACR_DTYPE_F16><<<blocks_for(n), kBlock, 0, s>>>(part, plan.splits, n, half, p.out, p.out2);
        });
    }
}

template <int DT>
void slopes_launch(const void *dh, const void *gate, const void *up, const uint8_t *gate_low, const uint8_t *up_low,
                   const Problem &q, int act, uint16_t *dgu, int64_t plane, float *plain, hipStream_t s)
{
    const int grid = blocks_for(q.rows * q.ff_pad / 8);
    const int64_t each = DT == STACR_DTYPE_F32 ? 12 + 16 : (gate_low ? 8 : 6) + 4;  // bytes read and written a value
    const auto run = [&](auto low, auto past) {
        stacr_launch("k_gated_slopes", s, [&] {
            k_gated_slopes<DT, decltype(low)::value, decltype(past)::value><<<grid, kBlock, 0, s>>>(
                dh, gate, up, gate_low, up_low, q.rows, q.ff, act, dgu, q.ff_pad, plane, plain);
        });
    };
    const bool past = q.rows * q.ff_pad * each > kCacheBytes;
    if (gate_low) past ? run(std::true_type(), std::true_type()) : run(std::true_type(), std::false_type());
    else past ? run(std::false_type(), std::true_type()) : run(std::false_type(), std::false_type());
}

template <int DT>
void bias_launch(const uint16_t *dgu, const Problem &q, int64_t plane, float *part, void *dbg, void *dbu, hipStream_t s)
{
    const int parts = (int)((q.rows + kBiasRows - 1) / kBiasRows);
    if (parts)
        stacr_launch("k_gated_bias_part", s, [&] {
            k_gated_bias_part<DT><<<dim3((unsigned)((2 * q.ff_pad + 255) / 256), (unsigned)parts), kBlock, 0, s>>>(
                dgu, q.rows, q.ff_pad, plane, part);
        });
    stacr_launch("k_gated_bias_sum", s, [&] {
        k_gated_bias_sum<DT><<<dim3((unsigned)((q.ff + 31) / 32), 2), kBlock, 0, s>>>(part, parts, q.ff, q.ff_pad, dbg, dbu);
    });
}

int check_kept(const char *what, int dtype, const void *gate, const void *up, const void *gate_low, const void *up_low)
{
    if ((gate == nullptr) != (up == nullptr) || (gate_low == nullptr) != (up_low == nullptr) || (gate_low && !gate))
        return stacr_fail(STACR_ERR_INVALID, "%s: gate goes with up, gate_low with up_low, both with gate and up", what);
    if (!aligned_to(gate, 16) || !aligned_to(up, 16) || !aligned_to(gate_low, 16) || !aligned_to(up_low, 16))
        return stacr_fail(STACR_ERR_INVALID, "%s: kept pre-activations must be 16-byte aligned", what);
    if (gate_low && dtype == STACR_DTYPE_F32)
        return stacr_fail(STACR_ERR_INVALID, "%s: fp32 pre-activations have no low bytes", what);
    return STACR_OK;
}

int check_problem(const char *what, int dtype, int64_t rows, int64_t d, int64_t ff, int64_t x_ld, int act)
{
    if (dtype != STACR_DTYPE_F32 && dtype != STACR_DTYPE_BF16 && dtype != STACR_DTYPE_F16)
        return stacr_fail(STACR_ERR_INVALID, "%s: unsupported dtype code %d", what, dtype);
    if (rows < 0 || d < 1 || ff < 1 || x_ld < d)
        return stacr_fail(STACR_ERR_INVALID, "%s: rows >= 0, d >= 1, ff >= 1 and a row stride of at least d are required",
                          what);
    if (act < STACR_ACT_SILU || act > STACR_ACT_SIGMOID)
        return stacr_fail(STACR_ERR_INVALID, "%s: unknown activation code %d", what, act);
    if (d > kMaxFeatures || ff > kMaxFeatures || x_ld > kMaxFeatures || rows >= (int64_t)1 << 24)
        return stacr_fail(STACR_ERR_UNSUPPORTED, "%s: more than 2^20 features, or 2^24 rows", what);
    // the products' grids, and the bias partials' second grid dimension
    if (tiles(rows, ff, 128, 64) >= (int64_t)1 << 30 || tiles(rows, d, 128, 128) >= (int64_t)1 << 30)
        return stacr_fail(STACR_ERR_UNSUPPORTED, "%s: more than 2^30 tiles", what);
    return STACR_OK;
}

}  // namespace

extern "C" {

int stacr_gated_workspace_bytes(const void *x, int dtype, int64_t rows, int64_t d, int64_t x_ld, const void *w_gate,
                                const void *w_up, int64_t ff, int backward, size_t *bytes)
{
    const int rc = check_problem("stacr_gated_workspace_bytes", dtype, rows, d, ff, x_ld, STACR_ACT_SILU);
    if (rc) return rc;
    if (!bytes) return stacr_fail(STACR_ERR_INVALID, "stacr_gated_workspace_bytes: NULL pointer argument");
    *bytes = pieces(problem(dtype, rows, d, ff, x_ld, x, w_gate, w_up), backward != 0).total;
    return STACR_OK;
}

int stacr_gated_forward(const void *x, int dtype, int64_t rows, int64_t d, int64_t x_ld, const void *w_gate,
                        const void *w_up, int64_t ff, const void *b_gate, const void *b_up, int activation, void *h,
                        void *gate, void *up, void *gate_low, void *up_low, void *workspace, size_t workspace_bytes, void *stream)
{
    const int rc = check_problem("stacr_gated_forward", dtype, rows, d, ff, x_ld, activation);
    if (rc) return rc;
    if (rows == 0) return STACR_OK;
    if (!x || !w_gate || !w_up || !h) return stacr_fail(STACR_ERR_INVALID, "stacr_gated_forward: NULL pointer argument");
    const int kept = check_kept("stacr_gated_forward", dtype, gate, up, gate_low, up_low);
    if (kept) return kept;
    hipStream_t s = static_cast<hipStream_t>(stream);
    Problem q = problem(dtype, rows, d, ff, x_ld, x, w_gate, w_up);
    if (rows <= kFewRows) {
        const FewArgs a{x, w_gate, w_up, b_gate, b_up, rows, d, x_ld, ff, activation, h, gate, up,
                        static_cast<uint8_t *>(gate_low), static_cast<uint8_t *>(up_low)};
        const bool vec = d % 8 == 0 && x_ld % 8 == 0 && aligned_to(x, 16) && aligned_to(w_gate, 16) && aligned_to(w_up, 16);
        if (dtype == STACR_DTYPE_F32) few_typed<STACR_DTYPE_F32>(a, vec, s);
        else if (dtype == STACR_DTYPE_BF16) few_typed<STACR_DTYPE_BF16>(a, vec, s);
        else few_typed<STACR_DTYPE_F16>(a, vec, s);
        return stacr_hip_check(hipGetLastError(), "gated forward kernels");
    }
    const Pieces w = pieces(q, false);
    if (w.total && (!workspace || workspace_bytes < w.total))
        return stacr_fail(STACR_ERR_WORKSPACE, "stacr_gated_forward: workspace of %zu bytes, %zu needed", workspace_bytes,
                          w.total);
    const Operands o = operands(q, x, w_gate, w_up, static_cast<char *>(workspace), w, true, true, s);
    MmArgs p = gated_args(q, o, b_gate, b_up, activation);
    p.out = h;
    p.gate = gate;
    p.up = up;
    p.gate_low = static_cast<uint8_t *>(gate_low);
    p.up_low = static_cast<uint8_t *>(up_low);
    dual_typed<kFwd>(dtype, p, s);
    return stacr_hip_check(hipGetLastError(), "gated forward kernels");
}

int stacr_gated_backward(const void *dh, const void *x, int dtype, int64_t rows, int64_t d, int64_t x_ld,
                         const void *w_gate, const void *w_up, int64_t ff, const void *b_gate, const void *b_up,
                         int activation, const void *gate, const void *up, const void *gate_low, const void *up_low,
                         void *dx, void *dw_gate, void *dw_up,
                         void *db_gate, void *db_up, void *dgu, void *workspace, size_t workspace_bytes, void *stream)
{
    const int rc = check_problem("stacr_gated_backward", dtype, rows, d, ff, x_ld, activation);
    if (rc) return rc;
    const bool kept = gate != nullptr, weights = dw_gate != nullptr;
    if (weights != (dw_up != nullptr)) return stacr_fail(STACR_ERR_INVALID, "stacr_gated_backward: dw_gate with dw_up");
    const int bad = check_kept("stacr_gated_backward", dtype, gate, up, gate_low, up_low);
    if (bad) return bad;
    if (rows && (!dh || (!x && (!kept || weights)) || ((!w_gate || !w_up) && (!kept || dx))))
        return stacr_fail(STACR_ERR_INVALID, "stacr_gated_backward: NULL pointer argument");
    if (dgu && dtype == STACR_DTYPE_F32 && !kept)
        return stacr_fail(STACR_ERR_UNSUPPORTED, "stacr_gated_backward: fp32 [dg | du] is given out from gate and up only");
    if (dgu && !aligned_to(dgu, 16))
        return stacr_fail(STACR_ERR_INVALID, "stacr_gated_backward: [dg | du] must be 16-byte aligned");
    hipStream_t s = static_cast<hipStream_t>(stream);
    const Problem q = problem(dtype, rows, d, ff, x_ld, x, w_gate, w_up);
    const Pieces w = pieces(q, true);
    if (w.total && (!workspace || workspace_bytes < w.total))
        return stacr_fail(STACR_ERR_WORKSPACE, "stacr_gated_backward: workspace of %zu bytes, %zu needed", workspace_bytes,
                          w.total);
    char *ws = static_cast<char *>(workspace);
    const int64_t plane = rows * 2 * q.ff_pad;
    // fp32's planes are the workspace's, its values go out beside them
    float *plain = dtype == STACR_DTYPE_F32 ? static_cast<float *>(dgu) : nullptr;
    uint16_t *slopes = dgu && !plain ? static_cast<uint16_t *>(dgu) : reinterpret_cast<uint16_t *>(ws + w.dgu);
    float *part = reinterpret_cast<float *>(ws + w.part);
    const Operands o = operands(q, x, w_gate, w_up, ws, w, rows > 0 && (!kept || weights), rows > 0 && (!kept || dx), s);
    if (rows && kept) {
        const uint8_t *gl = static_cast<const uint8_t *>(gate_low), *ul = static_cast<const uint8_t *>(up_low);
        if (dtype == STACR_DTYPE_F32) slopes_launch<STACR_DTYPE_F32>(dh, gate, up, nullptr, nullptr, q, activation, slopes, plane, plain, s);
        else if (dtype == STACR_DTYPE_BF16) slopes_launch<STACR_DTYPE_BF16>(dh, gate, up, gl, ul, q, activation, slopes, plane, nullptr, s);
        else slopes_launch<STACR_DTYPE_F16>(dh, gate, up, gl, ul, q, activation, slopes, plane, nullptr, s);
    } else if (rows) {
        MmArgs p = gated_args(q, o, b_gate, b_up, activation);
        p.dh = dh;
        p.dgu = slopes;
        p.plane = plane;
        dual_typed<kBwd>(dtype, p, s);
    }
    const int np = pairs(dtype);
    if (dx && rows) {
        MmArgs p{};
        p.nseg = 2 * np;
        for (int i = 0; i < p.nseg; ++i) {
            const int j = i % np, pa = np > 1 ? kPairA[j] : 0, pb = np > 1 ? kPairB[j] : 0;
            const bool second = i >= np;
            p.a.seg[i] = slopes + pa * plane + (second ? q.ff_pad : 0);
            p.b.seg[i] = (second ? o.wu : o.wg) + pb * o.w_plane;
        }
        p.a.ld = 2 * q.ff_pad;
        p.a.extent = rows;
        p.b.ld = o.w_ld;
        p.b.extent = q.d_pad;
        p.M = rows;
        p.N = d;
        p.K = ff;
        p.halves = 1;
        p.out = dx;
        product_typed<true>(dtype, p, product_plan(rows, d, 1, q.ff_pad, p.nseg, false), part, s);
    }
    if (weights && rows == 0) {
        const int bytes = dtype == STACR_DTYPE_F32 ? 4 : 2;
        for (void *w : {dw_gate, dw_up}) {
            const int e = stacr_fill_int_launch(w, bytes, ff * d, 0, s);
            if (e) return e;
        }
    } else if (weights) {
        MmArgs p{};
        p.nseg = np;
        for (int i = 0; i < np; ++i) {
            p.a.seg[i] = slopes + (np > 1 ? kPairA[i] : 0) * plane;
            p.b.seg[i] = o.x + (np > 1 ? kPairB[i] : 0) * o.x_plane;
        }
        p.a.ld = 2 * q.ff_pad;
        p.a.extent = 2 * q.ff_pad;
        p.a_half = q.ff_pad;
        p.b.ld = o.x_ld;
        p.b.extent = q.d_pad;
        p.M = ff;
        p.N = d;
        p.K = rows;
        p.halves = 2;
        p.out = dw_gate;
        p.out2 = dw_up;
        product_typed<false>(dtype, p, product_plan(ff, d, 2, rows, np, false), part, s);
    }
    if (db_gate || db_up) {
        if (dtype == STACR_DTYPE_F32) bias_launch<STACR_DTYPE_F32>(slopes, q, plane, part, db_gate, db_up, s);
        else if (dtype == STACR_DTYPE_BF16) bias_launch<STACR_DTYPE_BF16>(slopes, q, plane, part, db_gate, db_up, s);
        else bias_launch<STACR_DTYPE_F16>(slopes, q, plane, part, db_gate, db_up, s);
    }
    return stacr_hip_check(hipGetLastError(), "gated backward kernels");
}

}  // extern "C"
