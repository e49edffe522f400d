// A tile of a matrix product on the matrix cores, for the gated feed-forward's four products.
//
// C = sum over segments s of A_s B_s, both operands 16-bit, sums in fp32.  A workgroup owns BM x BN
// of C and walks K in steps of 64.  Each operand is stored in either order:
//   K-major  row i holds K values: tile rows of 64 values (128 bytes, eight 16-byte chunks), chunk c of
//            row i kept at chunk c ^ (i >> 1 & 7) of its row: 16 lanes a cycle read one chunk column of 16
//            rows, and those lie in 16 distinct chunks of the 64 banks' 256 bytes (two rows); a lane's
//            operand is one 16-byte read
//   M-major  row k holds the tile's BM (or BN) values: chunk c of row k kept at
//            c ^ ((k & 3) << 1 | (k >> 3 & 1) << 3); operands come by ds_read_b64_tr_b16, which hands lane n of
//            16 lanes the column n of a 4 x 16 block; 32 lanes a cycle read two such blocks, eight rows apart,
//            and their eight pieces of 32 bytes lie in distinct eighths of the banks
// (A key of i & 7 puts two rows of every read into the same banks, and the reads took twice as long.)
// Tiles come straight from memory into LDS (buffer_load ... lds, 16 bytes a lane: the swizzle is in
// which chunk a lane asks for), two stages: the next step is on its way while one runs, across the
// tiles that a workgroup takes in turn.  Reads past an
// operand's end (rows past M, K past the last) give zeros by the buffer's own range check.
#pragma once

#include "internal.h"

namespace stacr {

typedef float mmf4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ __amdgpu_buffer_rsrc_t mm_rsrc(const void *p, int64_t bytes)
{
    const int n = bytes <= 0 ? 0 : bytes < 0x7fffff00ll ? (int)bytes : 0x7fffff00;
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(p), (short)0, n, 0x00020000);
}

__device__ __forceinline__ void mm_copy16(__amdgpu_buffer_rsrc_t r, void *wave_dst, uint32_t voffset)
{
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void *)wave_dst, 16, (int)voffset,
                                             0, 0, 0);
}

__device__ __forceinline__ uint2 mm_tr16(const void *p)
{
    typedef __attribute__((__vector_size__(4 * sizeof(__bf16)))) __bf16 bf16x4;
    bf16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((__attribute__((address_space(3))) bf16x4 *)(p));
    return __builtin_bit_cast(uint2, v);
}

// 16 x 16 blocks of C, K 32 an instruction.  A lane's operands are eight values, from k 8 (lane / 16) on, of
// row lane % 16 of either side; given the columns' side first, it holds of the result columns
// 4 (lane / 16) .. + 3 of row lane % 16.  (32 x 32 blocks of K 16 were 5 % slower: the card is at its power
// limit in these loops, 1.6 to 1.7 GHz, and this form draws less.)
template <int DT> __device__ __forceinline__ mmf4 mm_mfma(uint4 a, uint4 b, mmf4 c)
{
    if constexpr (DT == STACR_DTYPE_F16) {
        typedef __attribute__((ext_vector_type(8))) _Float16 v8;
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
    } else {
        typedef __attribute__((ext_vector_type(8))) __bf16 v8;
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
    }
}

// Quads to eights: a lane's columns 4 (lane / 16) .. of two neighbouring blocks become columns
// 8 (lane / 16) .. + 7 of the 32, one word at a time (and back: the exchange is its own inverse, read
// backwards).  v_permlane32_swap exchanges the first's upper half of the wave with the second's lower
// half, v_permlane16_swap the odd rows of 16 lanes of the first with the even ones of the second.
__device__ __forceinline__ void mm_eights(uint32_t &first, uint32_t &second)
{
    const auto r = __builtin_amdgcn_permlane32_swap(first, second, false, false);
    const auto s = __builtin_amdgcn_permlane16_swap(r[0], r[1], false, false);
    first = s[0];
    second = s[1];
}

__device__ __forceinline__ void mm_quads(uint32_t &first, uint32_t &second)
{
    const auto r = __builtin_amdgcn_permlane16_swap(first, second, false, false);
    const auto s = __builtin_amdgcn_permlane32_swap(r[0], r[1], false, false);
    first = s[0];
    second = s[1];
}

constexpr int kMmK = 64;          // K of a step
constexpr int kMmMaxSegs = 12;
constexpr uint32_t kMmPast = 0x7fffff00u;  // an offset past every buffer (mm_rsrc's largest)

// One operand, all its segments.  `ld`: elements between rows.  K-major: `extent` rows of K values;
// M-major: K rows of `extent` values (both the allocation's, so no read leaves it).
struct MmOperand {
    const uint16_t *seg[kMmMaxSegs];
    int64_t ld;
    int64_t extent;
};

// Per-lane byte offsets of a wave's copies of one operand tile of R rows (K-major) or columns.
template <bool KMAJOR, int R, int NW>
struct MmLoader {
    static constexpr int kCopies = R / 8;           // 1 KiB each
    static constexpr int kPer = kCopies / NW;       // of a wave
    static constexpr int kChunks = R / 8;           // M-major: chunks a row
    static_assert(kCopies % NW == 0, "copies split evenly over the waves");
    static_assert(kPer % 2 == 0, "a copy's parity is its index's");
    uint32_t off[kPer];
    uint32_t kc[2];  // K-major: this lane's k within a step, in even and odd copies

    __device__ __forceinline__ void init(int lane, int wave, int64_t ld)
    {
        const uint32_t ldb = (uint32_t)ld * 2;
        if constexpr (KMAJOR) {
#pragma unroll
            for (int i = 0; i < 2; ++i) kc[i] = (uint32_t)(((lane & 7) ^ (i * 4 + (lane >> 4))) * 8);
#pragma unroll
            for (int i = 0; i < kPer; ++i) off[i] = ((wave * kPer + i) * 8 + (lane >> 3)) * ldb + kc[i & 1] * 2;
        } else {
            kc[0] = kc[1] = 0;
            constexpr int rows = 64 / kChunks;
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                const int k = (wave * kPer + i) * rows + lane / kChunks;
                off[i] = (uint32_t)k * ldb + (uint32_t)((lane % kChunks) ^ (((k & 3) << 1) | ((k >> 3 & 1) << 3))) * 16;
            }
        }
    }
};

// Where a lane's operands lie in a tile: block b of 16 rows / columns, half kk of the step.
template <bool KMAJOR, int R, int NB>
struct MmReader {
    uint32_t at[NB];

    __device__ __forceinline__ void init(int lane, int first)
    {
        if constexpr (KMAJOR) {
#pragma unroll
            for (int b = 0; b < NB; ++b) at[b] = (uint32_t)(first + b * 16 + (lane & 15)) * 128;
        } else {
            const int high = lane >> 4;  // k in eights
            const int k = high * 8 + ((lane >> 2) & 3), f = (((lane >> 2) & 3) << 1) | ((high & 1) << 3);
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const int c = ((first + b * 16) >> 3) + ((lane >> 1) & 1);
                at[b] = (uint32_t)k * (R * 2) + (uint32_t)(c ^ f) * 16 + (lane & 1) * 8;
            }
        }
    }

    __device__ __forceinline__ uint4 get(const unsigned char *tile, int b, int kk, int lane) const
    {
        if constexpr (KMAJOR) {
            const uint32_t c = (uint32_t)(kk * 4 + (lane >> 4)) ^ (uint32_t)((lane >> 1) & 7);
            return *reinterpret_cast<const uint4 *>(tile + at[b] + c * 16);
        } else {
            const unsigned char *p = tile + at[b] + kk * 32 * (R * 2);
            const uint2 lo = mm_tr16(p), hi = mm_tr16(p + 4 * (R * 2));
            return make_uint4(lo.x, lo.y, hi.x, hi.y);
        }
    }
};

}  // namespace stacr
