// The gated feed-forward block: h = act(x Wg^T + bg) * (x Wu^T + bu), and its backward pass.
//
//   forward    one product over [Wg; Wu] whose tiles hold a gate column block beside the same up
//              columns, so that a lane ends with both pre-activations of its outputs and the epilogue
//              writes h = act(g) u alone
//   backward   dg = dh u act'(g), du = dh act(g): the same product again with another epilogue (nothing
//              but x is kept by the forward), or an elementwise pass where g and u were kept; then
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
    int mt, nt, splits;
    void *out, *out2;
    int64_t ldo;
    int out_dt;
    bool vec;                        // rows of out (and dh) are whole, aligned 16-byte pieces
    float *part;                     // splits > 1: fp32 partial products [split][half][M][N]
    // gated epilogues
    const void *bias_g, *bias_u, *dh;
    void *gate, *up;                 // kept pre-activations or NULL
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

// act(g) and act'(g)
template <bool EXACT, int ACT> __device__ __forceinline__ void activate(float g, float &a, float &slope)
{
    if constexpr (ACT == STACR_ACT_SILU) {
        const float s = inverse<EXACT>(1.0f + exp_of<EXACT>(-g));
        a = g * s;
        slope = s * (1.0f + g * (1.0f - s));
    } else if constexpr (ACT == STACR_ACT_GELU) {
        const float below = 0.5f * (1.0f + erff(g * 0.70710678118654752f));
        a = g * below;
        slope = below + g * 0.39894228040143268f * exp_of<EXACT>(-0.5f * g * g);
    } else if constexpr (ACT == STACR_ACT_GELU_TANH) {
        const float in = 0.79788456080286536f * (g + 0.044715f * g * g * g);
        const float t = 1.0f - 2.0f * inverse<EXACT>(1.0f + exp_of<EXACT>(2.0f * in));
        a = 0.5f * g * (1.0f + t);
        slope = 0.5f * (1.0f + t) +
                0.5f * g * (1.0f - t * t) * 0.79788456080286536f * (1.0f + 3.0f * 0.044715f * g * g);
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

// four consecutive values of a row of type DT (n .. n + 3, those below N)
template <int DT>
__device__ __forceinline__ void store4(void *out, int64_t row, int64_t n, int64_t N, const float (&v)[4], bool vec)
{
    using A = Act<DT>;
    typename A::T *p = static_cast<typename A::T *>(out) + row + n;
    if (vec && n + 3 < N) {
        if constexpr (DT == STACR_DTYPE_F32) {
            *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
        } else {
            *reinterpret_cast<uint2 *>(p) = make_uint2((uint32_t)A::st(v[0]) | (uint32_t)A::st(v[1]) << 16,
                                                       (uint32_t)A::st(v[2]) | (uint32_t)A::st(v[3]) << 16);
        }
        return;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
        if (n + r < N) p[r] = A::st(v[r]);
}

template <int DT>
__device__ __forceinline__ void load4(const void *in, int64_t row, int64_t n, int64_t N, float (&v)[4], bool vec)
{
    using A = Act<DT>;
    const typename A::T *p = static_cast<const typename A::T *>(in) + row + n;
    if (vec && n + 3 < N) {
        if constexpr (DT == STACR_DTYPE_F32) {
            const float4 w = *reinterpret_cast<const float4 *>(p);
            v[0] = w.x; v[1] = w.y; v[2] = w.z; v[3] = w.w;
        } else {
            const uint2 w = *reinterpret_cast<const uint2 *>(p);
            v[0] = A::ld((typename A::T)(w.x & 0xffffu)); v[1] = A::ld((typename A::T)(w.x >> 16));
            v[2] = A::ld((typename A::T)(w.y & 0xffffu)); v[3] = A::ld((typename A::T)(w.y >> 16));
        }
        return;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = n + r < N ? A::ld(p[r]) : 0.0f;
}

// dg and du of four outputs f .. f + 3 of token m into [dg | du] (fp32: its four planes)
template <int DT>
__device__ __forceinline__ void store_dgu(uint16_t *dgu, int64_t ff_pad, int64_t plane, int64_t m, int64_t f,
                                          const float (&dg)[4], const float (&du)[4])
{
    uint16_t *p = dgu + m * 2 * ff_pad + f;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const float(&v)[4] = half ? du : dg;
        uint16_t *q = p + half * ff_pad;
        if constexpr (DT == STACR_DTYPE_F32) {
            uint16_t s[4][kPlanes];
#pragma unroll
            for (int r = 0; r < 4; ++r) split_f32(v[r], s[r]);
#pragma unroll
            for (int t = 0; t < kPlanes; ++t)
                *reinterpret_cast<uint2 *>(q + t * plane) =
                    make_uint2((uint32_t)s[0][t] | (uint32_t)s[1][t] << 16, (uint32_t)s[2][t] | (uint32_t)s[3][t] << 16);
        } else {
            using A = Act<DT>;
            *reinterpret_cast<uint2 *>(q) = make_uint2((uint32_t)A::st(v[0]) | (uint32_t)A::st(v[1]) << 16,
                                                       (uint32_t)A::st(v[2]) | (uint32_t)A::st(v[3]) << 16);
        }
    }
}

// A workgroup's results on their way out: rows of COLS values of type DT in LDS (16 bytes between rows
// against bank conflicts), then whole 16-byte pieces of rows to memory, consecutive lanes consecutive.
template <int DT, int COLS> struct Staged {
    using T = typename Act<DT>::T;
    static constexpr int kVec = 16 / sizeof(T), kPieces = COLS / kVec;
    static constexpr uint32_t pitch = COLS * sizeof(T) + 16;

    static __device__ __forceinline__ void put4(unsigned char *lds, int row, int col, const float (&v)[4])
    {
        using A = Act<DT>;
        unsigned char *p = lds + row * pitch + col * sizeof(T);
        if constexpr (DT == STACR_DTYPE_F32) *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
        else
            *reinterpret_cast<uint2 *>(p) = make_uint2((uint32_t)A::st(v[0]) | (uint32_t)A::st(v[1]) << 16,
                                                       (uint32_t)A::st(v[2]) | (uint32_t)A::st(v[3]) << 16);
    }

    static __device__ __forceinline__ void get4(const unsigned char *lds, int row, int col, float (&v)[4])
    {
        load4<DT>(lds + row * pitch, 0, col, COLS, v, true);
    }

    // rows m0 .. of `out` (those below M), columns n0 .. (below N)
    static __device__ __forceinline__ void store(const unsigned char *lds, int rows, int threads, void *out, int64_t ldo,
                                                 int64_t m0, int64_t M, int64_t n0, int64_t N, bool vec)
    {
        const int live = (int)(M - m0 < rows ? M - m0 : rows);
        T *base = static_cast<T *>(out) + m0 * ldo + n0;
        const int cols = (int)(N - n0 < COLS ? N - n0 : COLS);
        for (int i = threadIdx.x; i < live * kPieces; i += threads) {
            const int r = i / kPieces, c = (i % kPieces) * kVec;
            const uint4 v = *reinterpret_cast<const uint4 *>(lds + r * pitch + c * sizeof(T));
            T *p = base + r * ldo + c;
            if (vec && c + kVec <= cols) {
                *reinterpret_cast<uint4 *>(p) = v;
            } else {
                const T *e = reinterpret_cast<const T *>(lds + r * pitch) + c;
                for (int k = 0; k < kVec; ++k)
                    if (c + k < cols) p[k] = e[k];
            }
        }
    }

    // the same rows and columns of `in` into LDS, zeros outside
    static __device__ __forceinline__ void load(unsigned char *lds, int rows, int threads, const void *in, int64_t ld,
                                                int64_t m0, int64_t M, int64_t n0, int64_t N, bool vec)
    {
        const int live = (int)(M - m0 < rows ? M - m0 : rows);
        const T *base = static_cast<const T *>(in) + m0 * ld + n0;
        const int cols = (int)(N - n0 < COLS ? N - n0 : COLS);
#pragma unroll 4
        for (int i = threadIdx.x; i < rows * kPieces; i += threads) {
            const int r = i / kPieces, c = (i % kPieces) * kVec;
            uint4 v = make_uint4(0, 0, 0, 0);
            if (r < live) {
                const T *p = base + r * ld + c;
                if (vec && c + kVec <= cols) {
                    v = *reinterpret_cast<const uint4 *>(p);
                } else {
                    T e[kVec];
                    for (int k = 0; k < kVec; ++k) e[k] = c + k < cols ? p[k] : T(0);
                    __builtin_memcpy(&v, e, 16);
                }
            }
            *reinterpret_cast<uint4 *>(lds + r * pitch + c * sizeof(T)) = v;
        }
    }
};

// LDS of a product's workgroup: two stages, or what its epilogue stages
template <int DT, int EPI, int BM, int BN> constexpr size_t mm_lds()
{
    const size_t stages = 2 * (BM + BN) * 128;
    size_t out = 0;
    if (EPI == kFwd) out = BM * Staged<DT, BN / 2>::pitch;
    if (EPI == kBwd) out = BM * Staged<DT, BN / 2>::pitch * (DT == STACR_DTYPE_F32 ? 1 : 2);
    if (EPI == kStore) out = BM * Staged<STACR_DTYPE_BF16, BN>::pitch;
    return out > stages ? out : stages;
}

// A workgroup's tile: consecutive logical ids share an XCD (ids are dealt to the 8 XCDs round-robin)
// and walk `kGroup` tile rows together, so that an XCD's tiles share operands in its L2.
constexpr int kGroup = 8;

template <int DT, bool AK, bool BK, int EPI, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(WM *WN * 64) void k_gated_mm(const MmArgs p)
{
    constexpr int MT = DT == STACR_DTYPE_F16 ? STACR_DTYPE_F16 : STACR_DTYPE_BF16;  // the operands' type
    constexpr int NW = WM * WN, TM = BM / WM, TN = BN / WN, MI = TM / 16, NI = TN / 16;
    constexpr uint32_t kA = BM * 128, kStage = (BM + BN) * 128;
    constexpr bool DUAL = EPI != kStore;
    extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;

    // tile
    const int total = gridDim.x;
    int id = blockIdx.x;
    {
        const int q = total >> 3, r = total & 7, x = id & 7;
        id = x * q + (x < r ? x : r) + (id >> 3);
    }
    const int split = id / (p.mt * p.nt * p.halves);
    id -= split * p.mt * p.nt * p.halves;
    const int mrows = p.mt * p.halves;
    const int group = id / (kGroup * p.nt), first = group * kGroup;
    const int size = mrows - first < kGroup ? mrows - first : kGroup;
    const int in = id - group * kGroup * p.nt;
    const int mrow = first + in % size, ntile = in / size;
    const int half = mrow / p.mt;
    const int64_t m0 = (int64_t)(mrow - half * p.mt) * BM;
    const int64_t n0 = (int64_t)ntile * (DUAL ? BN / 2 : BN);

    MmLoader<AK, BM, NW> la;
    MmLoader<BK, BN, NW> lb;
    la.init(lane, wave, p.a.ld);
    lb.init(lane, wave, p.b.ld);
    if constexpr (DUAL) {  // tile rows 32 i .. + 15: gate rows n0 + 16 i .., the next 16 the same up rows
#pragma unroll
        for (int i = 0; i < lb.kPer; ++i) {
            const int row = (wave * lb.kPer + i) * 8 + (lane >> 3);
            lb.off[i] = (uint32_t)((row >> 5) * 16 + (row & 15)) * (uint32_t)p.b.ld * 2 + lb.kc * 2;
        }
    }
    MmReader<AK, BM, MI> ra;
    MmReader<BK, BN, NI> rb;
    ra.init(lane, wm * TM);
    rb.init(lane, wn * TN);

    const int ksteps = (int)((p.K + kMmK - 1) / kMmK), steps = ksteps * p.nseg;
    const int begin = (int)((int64_t)steps * split / p.splits), end = (int)((int64_t)steps * (split + 1) / p.splits);

    // The step that is loaded next: bytes from the operands' first values of this tile in it to their end
    // bound the reads (rows past the last, K past the last).
    const unsigned char *pa = nullptr, *pb = nullptr, *pb2 = nullptr;
    int64_t left_a = 0, left_b = 0;
    const int64_t step_a = AK ? kMmK * 2 : p.a.ld * (kMmK * 2), step_b = BK ? kMmK * 2 : p.b.ld * (kMmK * 2);
    int seg = 0, ks = 0;
    auto seek = [&](int s, int k) {
        seg = s;
        ks = k;
        const int64_t k0 = (int64_t)k * kMmK, kpad = (p.K + 7) & ~7ll;
        const int64_t at_a = AK ? m0 * p.a.ld + k0 : k0 * p.a.ld + m0 + half * p.a_half;
        const int64_t at_b = BK ? n0 * p.b.ld + k0 : k0 * p.b.ld + n0;
        const int64_t end_a = AK ? (p.a.extent - 1) * p.a.ld + kpad : (p.K - 1) * p.a.ld + p.a.extent;
        const int64_t end_b = BK ? (p.b.extent - 1) * p.b.ld + kpad : (p.K - 1) * p.b.ld + p.b.extent;
        pa = reinterpret_cast<const unsigned char *>(p.a.seg[s] + at_a);
        pb = reinterpret_cast<const unsigned char *>(p.b.seg[s] + at_b);
        if constexpr (DUAL) pb2 = reinterpret_cast<const unsigned char *>(p.b2[s] + at_b);
        left_a = (end_a - at_a) * 2;
        left_b = (end_b - at_b) * 2;
    };
    auto next = [&] {
        if (++ks == ksteps) {
            if (seg + 1 < p.nseg) seek(seg + 1, 0);
        } else {
            pa += step_a;
            pb += step_b;
            if constexpr (DUAL) pb2 += step_b;
            left_a -= step_a;
            left_b -= step_b;
        }
    };
    auto load = [&](unsigned char *__restrict__ at) {
        const uint32_t k = (uint32_t)ks * kMmK;
        {
            const auto r = mm_rsrc(pa, left_a);
            const bool live = !AK || k + la.kc < (uint32_t)p.K;
#pragma unroll
            for (int i = 0; i < la.kPer; ++i) mm_copy16(r, at + (wave * la.kPer + i) * 1024, live ? la.off[i] : kMmPast);
        }
        const bool live = !BK || k + lb.kc < (uint32_t)p.K;
        const auto r = mm_rsrc(pb, left_b), r2 = mm_rsrc(pb2, left_b);
#pragma unroll
        for (int i = 0; i < lb.kPer; ++i) {
            const bool second = DUAL && ((wave * lb.kPer + i) & 2);  // 8 rows of one copy are of one weight
            mm_copy16(second ? r2 : r, at + kA + (wave * lb.kPer + i) * 1024, live ? lb.off[i] : kMmPast);
        }
    };

    mmf4 acc[MI][NI];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j) acc[i][j] = mmf4{0.0f, 0.0f, 0.0f, 0.0f};

    // One step: the next one's copies into `to`, the products of what is in `from`.  Two pointers that do
    // not alias: without that knowledge the compiler waits for the copies before it reads.
    auto step = [&](const unsigned char *__restrict__ from, unsigned char *__restrict__ to, bool more) {
        if (more) load(to);
        const unsigned char *ta = from, *tb = from + kA;
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            uint4 av[MI], bv[NI];
#pragma unroll
            for (int j = 0; j < NI; ++j) bv[j] = rb.get(tb, j, kk, lane);
#pragma unroll
            for (int i = 0; i < MI; ++i) av[i] = ra.get(ta, i, kk, lane);
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int j = 0; j < NI; ++j) acc[i][j] = mm_mfma<MT>(bv[j], av[i], acc[i][j]);
        }
    };
    if (begin < end) {
        seek(begin / ksteps, begin % ksteps);
        load(lds);
        next();
    }
    for (int it = begin; it < end; ++it) {
        const int buf = (it - begin) & 1;
        __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0): this wave's copies of this step are in LDS
        asm volatile("s_barrier" ::: "memory");  // and everybody's; the other stage has been read
        step(lds + buf * kStage, lds + (buf ^ 1) * kStage, it + 1 < end);
        next();
    }

    // a lane holds, of each 16 x 16 block, columns 4 (lane / 16) .. + 3 of row lane % 16
    constexpr int NT = NW * 64;
    const int row0 = wm * TM + (lane & 15), quad = (lane >> 4) * 4;
    __syncthreads();  // the last step has been read
    if constexpr (EPI == kStore) {
        void *o = half ? p.out2 : p.out;
        if (p.splits > 1 || p.out_dt == STACR_DTYPE_F32) {
            float *out = p.splits > 1 ? p.part + ((int64_t)split * p.halves + half) * p.M * p.N : static_cast<float *>(o);
            const bool vec = p.splits > 1 ? (p.N & 3) == 0 : p.vec;
#pragma unroll
            for (int i = 0; i < MI; ++i) {
                const int64_t m = m0 + row0 + i * 16;
                if (m >= p.M) continue;
#pragma unroll
                for (int j = 0; j < NI; ++j) {
                    const float v[4] = {acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]};
                    store4<STACR_DTYPE_F32>(out, m * p.N, n0 + wn * TN + j * 16 + quad, p.N, v, vec);
                }
            }
        } else {
            using S = Staged<MT, BN>;
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int j = 0; j < NI; ++j) {
                    const float v[4] = {acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]};
                    S::put4(lds, row0 + i * 16, wn * TN + j * 16 + quad, v);
                }
            __syncthreads();
            S::store(lds, BM, NT, o, p.ldo, m0, p.M, n0, p.N, p.vec);
        }
    } else {
        constexpr bool EXACT = DT == STACR_DTYPE_F32;
        constexpr int F = BN / 2;
        using S = Staged<DT, F>;
        const int col0 = wn * (TN / 2) + quad;
        if (p.bias_g || p.bias_u) {
#pragma unroll
            for (int j = 0; j < NI; j += 2) {
                float bg[4] = {}, bu[4] = {};
                if (p.bias_g) load4<DT>(p.bias_g, 0, n0 + col0 + j * 8, p.N, bg, false);
                if (p.bias_u) load4<DT>(p.bias_u, 0, n0 + col0 + j * 8, p.N, bu, false);
#pragma unroll
                for (int i = 0; i < MI; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc[i][j][r] += bg[r], acc[i][j + 1][r] += bu[r];
            }
        }
        if constexpr (EPI == kFwd) {
            with_activation(p.act, [&](auto c) {
#pragma unroll
                for (int i = 0; i < MI; ++i)
#pragma unroll
                    for (int j = 0; j < NI; j += 2) {
                        float h[4];
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            float a, slope;
                            activate<EXACT, decltype(c)::value>(acc[i][j][r], a, slope);
                            h[r] = a * acc[i][j + 1][r];
                        }
                        S::put4(lds, row0 + i * 16, col0 + j * 8, h);
                    }
            });
            __syncthreads();
            S::store(lds, BM, NT, p.out, p.ldo, m0, p.M, n0, p.N, p.vec);
            if (p.gate) {  // the kept pre-activations
#pragma unroll
                for (int which = 0; which < 2; ++which) {
                    __syncthreads();
#pragma unroll
                    for (int i = 0; i < MI; ++i)
#pragma unroll
                        for (int j = 0; j < NI; j += 2) {
                            const mmf4 &w = acc[i][j + which];
                            const float v[4] = {w[0], w[1], w[2], w[3]};
                            S::put4(lds, row0 + i * 16, col0 + j * 8, v);
                        }
                    __syncthreads();
                    S::store(lds, BM, NT, which ? p.up : p.gate, p.ldo, m0, p.M, n0, p.N, p.vec);
                }
            }
        } else {
            // dh is staged first; a lane's dg takes the place of the dh that it read, du a second stage
            S::load(lds, BM, NT, p.dh, p.ldo, m0, p.M, n0, p.N, p.vec);
            __syncthreads();
            unsigned char *second = lds + BM * S::pitch;
            with_activation(p.act, [&](auto c) {
#pragma unroll
                for (int i = 0; i < MI; ++i) {
                    __builtin_amdgcn_sched_barrier(0);  // a row of blocks at a time: all at once spill
                    const int64_t m = m0 + row0 + i * 16;
#pragma unroll
                    for (int j = 0; j < NI; j += 2) {
                        float d[4], dg[4], du[4];
                        S::get4(lds, row0 + i * 16, col0 + j * 8, d);
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            float a, slope;
                            activate<EXACT, decltype(c)::value>(acc[i][j][r], a, slope);
                            dg[r] = d[r] * acc[i][j + 1][r] * slope;
                            du[r] = d[r] * a;
                        }
                        if constexpr (EXACT) {
                            if (m < p.M && n0 + col0 + j * 8 < p.ff_pad)
                                store_dgu<DT>(p.dgu, p.ff_pad, p.plane, m, n0 + col0 + j * 8, dg, du);
                        } else {
                            S::put4(lds, row0 + i * 16, col0 + j * 8, dg);
                            S::put4(second, row0 + i * 16, col0 + j * 8, du);
                        }
                    }
                }
            });
            if constexpr (!EXACT) {
                __syncthreads();
#pragma unroll
                for (int which = 0; which < 2; ++which)
                    S::store(which ? second : lds, BM, NT, p.dgu + which * p.ff_pad, 2 * p.ff_pad, m0, p.M, n0, p.ff_pad, true);
            }
        }
    }
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
// four bf16 planes, 16-bit types as they are
template <int DT>
__global__ __launch_bounds__(kBlock) void k_gated_pack(const void *__restrict__ src, int64_t ld, int64_t rows,
                                                       int64_t cols, uint16_t *__restrict__ dst, int64_t ld_dst, bool vec)
{
    const int64_t chunks = ld_dst / 8, n = rows * chunks, plane = rows * ld_dst;
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
template <int DT>
__global__ __launch_bounds__(kBlock) void k_gated_slopes(const void *__restrict__ dh, const void *__restrict__ gate,
                                                         const void *__restrict__ up, int64_t rows, int64_t ff, int act,
                                                         uint16_t *__restrict__ dgu, int64_t ff_pad, int64_t plane, bool vec)
{
    const int64_t quads = ff_pad / 4, n = rows * quads;
    for (int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x; i < n; i += (int64_t)gridDim.x * kBlock) {
        const int64_t m = i / quads, f = (i - m * quads) * 4;
        float d[4], g[4], u[4], dg[4], du[4];
        load4<DT>(dh, m * ff, f, ff, d, vec);
        load4<DT>(gate, m * ff, f, ff, g, vec);
        load4<DT>(up, m * ff, f, ff, u, vec);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            float a, slope;
            activate<DT == STACR_DTYPE_F32>(act, g[r], a, slope);
            dg[r] = d[r] * u[r] * slope;
            du[r] = d[r] * a;
        }
        store_dgu<DT>(dgu, ff_pad, plane, m, f, dg, du);
    }
}

// ------------------------------------------------------------------ bias gradients
// column sums of [dg | du]: `parts` row ranges of partial sums, then their sum in order
constexpr int kBiasRows = 256;

template <int DT>
__global__ __launch_bounds__(kBlock) void k_gated_bias_part(const uint16_t *__restrict__ dgu, int64_t rows, int64_t ff_pad,
                                                            int64_t plane, float *__restrict__ part)
{
    const int64_t cols = 2 * ff_pad, c = (int64_t)blockIdx.x * kBlock + threadIdx.x;
    if (c >= cols) return;
    const int64_t r0 = (int64_t)blockIdx.y * kBiasRows, r1 = r0 + kBiasRows < rows ? r0 + kBiasRows : rows;
    float sum = 0.0f;
    for (int64_t r = r0; r < r1; ++r) {
        const uint16_t *p = dgu + r * cols + c;
        if constexpr (DT == STACR_DTYPE_F32)
            sum += bf16_bits_to_f(p[0]) + (bf16_bits_to_f(p[plane]) + bf16_bits_to_f(p[2 * plane]));
        else sum += Act<DT>::ld(p[0]);
    }
    part[(int64_t)blockIdx.y * cols + c] = sum;
}

template <int DT>
__global__ __launch_bounds__(kBlock) void k_gated_bias_sum(const float *__restrict__ part, int parts, int64_t ff,
                                                           int64_t ff_pad, void *db_gate, void *db_up)
{
    const int64_t f = (int64_t)blockIdx.x * kBlock + threadIdx.x;
    if (f >= ff) return;
    for (int half = 0; half < 2; ++half) {
        void *out = half ? db_up : db_gate;
        if (!out) continue;
        float sum = 0.0f;
        for (int i = 0; i < parts; ++i) sum += part[(int64_t)i * 2 * ff_pad + half * ff_pad + f];
        static_cast<typename Act<DT>::T *>(out)[f] = Act<DT>::st(sum);
    }
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
    const int64_t d = p.d;
#pragma unroll 4
    for (int64_t k0 = wave * 32; k0 < d; k0 += kWaves * 32) {
        const int64_t k = k0 + (lane >> 4) * 8, left = d - k;
        uint4 g[P], u[P];
        few_load<DT, VEC>(p.wg, f * d + k, left, g);
        few_load<DT, VEC>(p.wu, f * d + k, left, u);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            uint4 x[P];
            few_load<DT, VEC>(p.x, xrow[t] + k, left, x);
            if constexpr (DT == STACR_DTYPE_F32) {
#pragma unroll
                for (int q = 0; q < kPairs; ++q) {
                    ag[t] = mm_mfma<MT>(g[kPairB[q]], x[kPairA[q]], ag[t]);
                    au[t] = mm_mfma<MT>(u[kPairB[q]], x[kPairA[q]], au[t]);
                }
            } else {
                ag[t] = mm_mfma<MT>(g[0], x[0], ag[t]);
                au[t] = mm_mfma<MT>(u[0], x[0], au[t]);
            }
        }
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
            store_any(p.gate, DT, m * p.ff + ff, g);
            store_any(p.up, DT, m * p.ff + ff, u);
        }
    }
}

// Rows up to which the forward takes k_gated_few.
constexpr int64_t kFewRows = 64;

// ------------------------------------------------------------------ host side
constexpr int64_t kMaxFeatures = 1 << 20;  // row strides whose tile offsets stay within 31 bits

inline int64_t up_to(int64_t n, int64_t m) { return (n + m - 1) / m * m; }
inline size_t aligned(size_t n) { return (n + 255) & ~(size_t)255; }

bool aligned_to(const void *p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

int size_of(int dt) { return dt == STACR_DTYPE_F32 ? 4 : 2; }

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

template <typename K> void raise_lds(K kernel, size_t bytes)
{
    static bool done = false;  // once per kernel instantiation
    if (!done) {
        (void)hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                                  (int)bytes);
        done = true;
    }
}

template <int DT, bool AK, bool BK, int EPI, int BM, int BN, int WM, int WN>
void mm_run(MmArgs p, hipStream_t s)
{
    constexpr size_t lds = mm_lds<DT, EPI, BM, BN>();
    static_assert(lds <= 160 * 1024, "LDS budget");
    p.mt = (int)((p.M + BM - 1) / BM);
    const int64_t cols = EPI == kBwd ? p.ff_pad : p.N;
    p.nt = (int)((cols + (EPI == kStore ? BN : BN / 2) - 1) / (EPI == kStore ? BN : BN / 2));
    auto kernel = k_gated_mm<DT, AK, BK, EPI, BM, BN, WM, WN>;
    raise_lds(kernel, lds);
    const int grid = p.mt * p.nt * p.halves * p.splits;
    const char *name = EPI == kFwd ? "k_gated_mm_forward" : EPI == kBwd ? "k_gated_mm_slopes"
                       : BK || AK ? "k_gated_mm_input" : "k_gated_mm_weights";
    stacr_launch(name, s, [&] { kernel<<<grid, WM * WN * 64, lds, s>>>(p); });
}

int64_t tiles(int64_t m, int64_t n, int bm, int bn) { return ((m + bm - 1) / bm) * ((n + bn - 1) / bn); }

// Workgroups that share K of one tile: enough to give every CU one, as long as each keeps 16 steps (its
// start and its partial product cost about that much).
int splits_for(int64_t ntiles, int64_t steps)
{
    const int64_t want = 256 / (ntiles > 0 ? ntiles : 1), most = steps / 16;
    const int64_t n = want < most ? want : most;
    return n < 1 ? 1 : (int)n;
}

template <int DT, int EPI>
void dual(const MmArgs &p, hipStream_t s)
{
    // 256 x 256 where its tiles fill the chip, else 128 x 128
    if (tiles(p.M, p.N, 256, 128) >= 256) mm_run<DT, true, true, EPI, 256, 256, 2, 4>(p, s);
    else mm_run<DT, true, true, EPI, 128, 128, 2, 2>(p, s);
}

template <int DT, bool AK>
void product(MmArgs p, hipStream_t s, bool big)
{
    if (big) mm_run<DT, AK, false, kStore, 256, 256, 2, 4>(p, s);
    else mm_run<DT, AK, false, kStore, 128, 128, 2, 2>(p, s);
}

struct ProductPlan {
    bool big;
    int splits;
};

ProductPlan product_plan(int64_t m, int64_t n, int halves, int64_t k, int nseg)
{
    const int64_t steps = (k + kMmK - 1) / kMmK * nseg;
    ProductPlan q;
    q.big = tiles(m, n, 256, 256) * halves >= 256;
    q.splits = q.big ? 1 : splits_for(tiles(m, n, 128, 128) * halves, steps);
    return q;
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
        const size_t dx = part_bytes(product_plan(q.rows, q.d, 1, q.ff_pad, 2 * pairs(q.dt)), q.rows, q.d, 1);
        const size_t dw = part_bytes(product_plan(q.ff, q.d, 2, q.rows, pairs(q.dt)), q.ff, q.d, 2);
        const size_t db = aligned((size_t)((q.rows + kBiasRows - 1) / kBiasRows) * 2 * q.ff_pad * 4);
        at += hmax(hmax(dx, dw), db);
    }
    w.total = at;
    return w;
}

int blocks_for(int64_t n) { return (int)hmin<int64_t>((n + kBlock - 1) / kBlock, 4096); }

void pack(int dt, const void *src, int64_t ld, int64_t rows, int64_t cols, uint16_t *dst, int64_t ld_dst, hipStream_t s)
{
    const int64_t n = rows * ld_dst / 8;
    if (n == 0) return;
    const bool vec = aligned_to(src, 16) && ld % 4 == 0;
    stacr_launch("k_gated_pack", s, [&] {
        if (dt == STACR_DTYPE_F32)
            k_gated_pack<STACR_DTYPE_F32><<<blocks_for(n), kBlock, 0, s>>>(src, ld, rows, cols, dst, ld_dst, vec);
        else k_gated_pack<STACR_DTYPE_BF16><<<blocks_for(n), kBlock, 0, s>>>(src, ld, rows, cols, dst, ld_dst, false);
    });
}

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
    if (q.pack_x && need_x) {
        uint16_t *dst = reinterpret_cast<uint16_t *>(ws + w.x);
        pack(q.dt, x, q.x_ld, q.rows, q.d, dst, q.d_pad, s);
        o.x = dst;
        o.x_ld = q.d_pad;
        o.x_plane = (size_t)q.rows * q.d_pad;
    }
    if (q.pack_w && need_w) {
        uint16_t *g = reinterpret_cast<uint16_t *>(ws + w.wg), *u = reinterpret_cast<uint16_t *>(ws + w.wu);
        pack(q.dt, wg, q.d, q.ff, q.d, g, q.d_pad, s);
        pack(q.dt, wu, q.d, q.ff, q.d, u, q.d_pad, s);
        o.wg = g;
        o.wu = u;
        o.w_ld = q.d_pad;
        o.w_plane = (size_t)q.ff * q.d_pad;
    }
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
    p.vec = p.N * size_of(dt) % 16 == 0 && aligned_to(p.out, 16) && aligned_to(p.out2, 16);
    p.ldo = p.N;
    if (dt == STACR_DTYPE_F16) product<STACR_DTYPE_F16, AK>(p, s, plan.big);
    else product<STACR_DTYPE_BF16, AK>(p, s, plan.big);
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
void slopes_launch(const void *dh, const void *gate, const void *up, const Problem &q, int act, uint16_t *dgu,
                   int64_t plane, bool vec, hipStream_t s)
{
    const int64_t n = q.rows * q.ff_pad / 4;
    stacr_launch("k_gated_slopes", s, [&] {
        k_gated_slopes<DT><<<blocks_for(n), kBlock, 0, s>>>(dh, gate, up, q.rows, q.ff, act, dgu, q.ff_pad, plane, vec);
    });
}

template <int DT>
void bias_launch(const uint16_t *dgu, const Problem &q, int64_t plane, float *part, void *dbg, void *dbu, hipStream_t s)
{
    const int parts = (int)((q.rows + kBiasRows - 1) / kBiasRows);
    if (parts)
        stacr_launch("k_gated_bias_part", s, [&] {
            k_gated_bias_part<DT><<<dim3((unsigned)((2 * q.ff_pad + kBlock - 1) / kBlock), (unsigned)parts), kBlock, 0, s>>>(
                dgu, q.rows, q.ff_pad, plane, part);
        });
    stacr_launch("k_gated_bias_sum", s, [&] {
        k_gated_bias_sum<DT><<<blocks_for(q.ff), kBlock, 0, s>>>(part, parts, q.ff, q.ff_pad, dbg, dbu);
    });
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
    if (tiles(rows, ff, 128, 64) >= (int64_t)1 << 30)
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
                        void *gate, void *up, void *workspace, size_t workspace_bytes, void *stream)
{
    const int rc = check_problem("stacr_gated_forward", dtype, rows, d, ff, x_ld, activation);
    if (rc) return rc;
    if (rows == 0) return STACR_OK;
    if (!x || !w_gate || !w_up || !h || (gate == nullptr) != (up == nullptr))
        return stacr_fail(STACR_ERR_INVALID, "stacr_gated_forward: NULL pointer argument");
    hipStream_t s = static_cast<hipStream_t>(stream);
    Problem q = problem(dtype, rows, d, ff, x_ld, x, w_gate, w_up);
    if (rows <= kFewRows) {
        const FewArgs a{x, w_gate, w_up, b_gate, b_up, rows, d, x_ld, ff, activation, h, gate, up};
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
    p.vec = ff * size_of(dtype) % 16 == 0 && aligned_to(h, 16) && aligned_to(gate, 16) && aligned_to(up, 16);
    dual_typed<kFwd>(dtype, p, s);
    return stacr_hip_check(hipGetLastError(), "gated forward kernels");
}

int stacr_gated_backward(const void *dh, const void *x, int dtype, int64_t rows, int64_t d, int64_t x_ld,
                         const void *w_gate, const void *w_up, int64_t ff, const void *b_gate, const void *b_up,
                         int activation, const void *gate, const void *up, void *dx, void *dw_gate, void *dw_up,
                         void *db_gate, void *db_up, void *dgu, void *workspace, size_t workspace_bytes, void *stream)
{
    const int rc = check_problem("stacr_gated_backward", dtype, rows, d, ff, x_ld, activation);
    if (rc) return rc;
    const bool kept = gate != nullptr, weights = dw_gate != nullptr;
    if ((gate == nullptr) != (up == nullptr) || weights != (dw_up != nullptr))
        return stacr_fail(STACR_ERR_INVALID, "stacr_gated_backward: gate with up and dw_gate with dw_up");
    if (rows && (!dh || (!x && (!kept || weights)) || ((!w_gate || !w_up) && (!kept || dx))))
        return stacr_fail(STACR_ERR_INVALID, "stacr_gated_backward: NULL pointer argument");
    if (dgu && dtype == STACR_DTYPE_F32)
        return stacr_fail(STACR_ERR_UNSUPPORTED, "stacr_gated_backward: [dg | du] is given out for 16-bit types only");
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
    uint16_t *slopes = dgu ? static_cast<uint16_t *>(dgu) : reinterpret_cast<uint16_t *>(ws + w.dgu);
    float *part = reinterpret_cast<float *>(ws + w.part);
    const Operands o = operands(q, x, w_gate, w_up, ws, w, rows > 0 && (!kept || weights), rows > 0 && (!kept || dx), s);
    const bool vec = ff * size_of(dtype) % 16 == 0 && aligned_to(dh, 16) && aligned_to(gate, 16) && aligned_to(up, 16);
    if (rows && kept) {
        if (dtype == STACR_DTYPE_F32) slopes_launch<STACR_DTYPE_F32>(dh, gate, up, q, activation, slopes, plane, vec, s);
        else if (dtype == STACR_DTYPE_BF16) slopes_launch<STACR_DTYPE_BF16>(dh, gate, up, q, activation, slopes, plane, vec, s);
        else slopes_launch<STACR_DTYPE_F16>(dh, gate, up, q, activation, slopes, plane, vec, s);
    } else if (rows) {
        MmArgs p = gated_args(q, o, b_gate, b_up, activation);
        p.dh = dh;
        p.dgu = slopes;
        p.plane = plane;
        p.vec = vec;
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
        product_typed<true>(dtype, p, product_plan(rows, d, 1, q.ff_pad, p.nseg), part, s);
    }
    if (weights) {
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
        product_typed<false>(dtype, p, product_plan(ff, d, 2, rows, np), part, s);
    }
    if (db_gate || db_up) {
        if (dtype == STACR_DTYPE_F32) bias_launch<STACR_DTYPE_F32>(slopes, q, plane, part, db_gate, db_up, s);
        else if (dtype == STACR_DTYPE_BF16) bias_launch<STACR_DTYPE_BF16>(slopes, q, plane, part, db_gate, db_up, s);
        else bias_launch<STACR_DTYPE_F16>(slopes, q, plane, part, db_gate, db_up, s);
    }
    return stacr_hip_check(hipGetLastError(), "gated backward kernels");
}

}  // extern "C"
