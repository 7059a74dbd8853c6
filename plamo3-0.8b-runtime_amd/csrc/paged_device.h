// Device helpers shared by the kernels over paged caches (paged.hip, speculate.hip, tree_attention.hip).
#pragma once

#include "device.h"
#include "paged.h"

namespace plamo {
namespace dev {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float floatx4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ uint32_t divide(uint32_t x, Divider d) { return uint32_t((uint64_t(x) * d.mul) >> d.shift); }

// v of the lane that a DPP control names, 0 where there is none (or the row is not in ROWS).
template <int CONTROL, int ROWS = 0xf>
__device__ __forceinline__ int shifted(int v) {
    return __builtin_amdgcn_update_dpp(0, v, CONTROL, ROWS, 0xf, false);
}

template <int TYPE>
__device__ __forceinline__ float from16(uint32_t h) {
    if constexpr (TYPE == TYPE_BF16) return bf(h & 0xffffu);
    return float(__builtin_bit_cast(_Float16, uint16_t(h)));
}
// Two values rounded to nearest even and packed.
template <int TYPE>
__device__ __forceinline__ uint32_t pack16(float a, float b) {
    if constexpr (TYPE == TYPE_BF16) return pack_bf16(a, b);
    const f16x2 h = {_Float16(a), _Float16(b)};
    return __builtin_bit_cast(uint32_t, h);
}

// Inclusive sum over the wave: rows of 16 lanes by shifts of 1, 2, 4 and 8, then the last lane of the row, and of the half, before.
__device__ __forceinline__ int wave_scan(int v) {
    v += shifted<0x111>(v);
    v += shifted<0x112>(v);
    v += shifted<0x114>(v);
    v += shifted<0x118>(v);
    v += shifted<0x142, 0xa>(v);
    v += shifted<0x143, 0xc>(v);
    return v;
}

}  // namespace dev
}  // namespace plamo
