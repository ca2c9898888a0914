// Device pieces that the attention kernels share (kr_attn.hip: a whole prompt,
// kr_paged.hip: new tokens over a paged cache): the MFMA, packing to 16 bits
// and the LDS layout of a block of K or V rows.
#pragma once

#include "kr_common.h"

namespace kr {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short AttnS4 __attribute__((ext_vector_type(4)));
typedef uint32_t AttnU2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) AttnS4 *LdsS4;

// two values to 16 bits (round to nearest even, as Elem<DT>::Store), packed
// low | high << 16: one v_cvt_pk_bf16_f32 for bf16
template <int DT>
__device__ __forceinline__ uint32_t Pack2(float lo, float hi)
{
    if constexpr (DT == kBF16) {
        typedef float F2 __attribute__((ext_vector_type(2)));
        typedef __bf16 B2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((F2){lo, hi}, B2));
    } else {
        return uint32_t(Elem<DT>::Store(lo)) | (uint32_t(Elem<DT>::Store(hi)) << 16);
    }
}

template <int DT>
__device__ __forceinline__ f32x16 Mfma(const uint4 &a, const uint4 &b, const f32x16 &c)
{
    if constexpr (DT == kBF16) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                       __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                      __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
}

// LDS slot of 16-byte chunk c in row r of a K / V block (an XOR, so it also
// maps a slot back to its chunk). K (D/8 chunks a row, read 16 rows x one
// chunk per 16 lanes): rows 0..15 of a pass land in 16 distinct slots of the
// 256-byte bank line. V (read by ds_read_b64_tr_b16: 4 rows x 4 chunks per
// 16 lanes): the four rows of a read land in four distinct chunk groups.
template <int D>
__device__ __forceinline__ int KSlot(int r, int c)
{
    if constexpr (D == 128) return c ^ (r & 15);
    else return c ^ ((r >> 1) & 7);
}
template <int D>
__device__ __forceinline__ int VSlot(int r, int c)
{
    if constexpr (D == 128) return c ^ (4 * (r & 3));
    else return c ^ (4 * ((r >> 1) & 1));
}

}  // namespace kr
