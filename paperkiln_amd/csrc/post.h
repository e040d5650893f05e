// What the kernels of the post-training operators share (qk_norm_rope.hip, token_loss.hip, adamw_many.hip): element access in both storage types,
// sums over a wavefront's lanes, and the argument checks of their C entries.
#pragma once
#include <cmath>
#include <initializer_list>
#include <string>

#include "mfma_common.h"
#include "pk_internal.h"

namespace pk {

__device__ inline float elem(const float* p, int64_t i) { return p[i]; }
__device__ inline float elem(const uint16_t* p, int64_t i) { return __uint_as_float(static_cast<uint32_t>(p[i]) << 16); }
__device__ inline void put(float* p, int64_t i, float x) { p[i] = x; }
__device__ inline void put(uint16_t* p, int64_t i, float x) { p[i] = static_cast<uint16_t>(pack_bf16(x, 0.0f)); }  // nearest even, NaN stays one

// x added up over groups of G lanes (a power of two from 4 to 64), the sum in every lane of the group; all lanes are active. In registers: exchanges of
// halves, of sixteens, then inside sixteen lanes by data-parallel moves (rotation by 8, mirrored eights, lane ^ 2, lane ^ 1).
template <int G>
__device__ inline float group_sum(float x) {
    static_assert(G == 4 || G == 8 || G == 16 || G == 32 || G == 64, "lanes of a group");
    if constexpr (G >= 64) {
        const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        x = __uint_as_float(h[0]) + __uint_as_float(h[1]);
    }
    if constexpr (G >= 32) {
        const auto q = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        x = __uint_as_float(q[0]) + __uint_as_float(q[1]);
    }
    if constexpr (G >= 16) x += lane_moved<0x128>(x);
    if constexpr (G >= 8) x += lane_moved<0x141>(x);
    x += lane_moved<0x4E>(x);
    x += lane_moved<0xB1>(x);
    return x;
}

inline bool known_dtype(int dtype) { return dtype == PK_F32 || dtype == PK_BF16; }
inline int64_t elem_size(int dtype) { return dtype == PK_F32 ? 4 : 2; }
inline bool aligned(const void* p, int64_t bytes) { return reinterpret_cast<uintptr_t>(p) % static_cast<uintptr_t>(bytes) == 0; }
inline int launched() {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? PK_OK : hip_fail(e, "kernel launch");
}
inline void touch(std::initializer_list<const void*> used, void* stream) { dev_touch(used.begin(), used.size(), stream); }
// The body of a C entry: nothing thrown (a string that finds no memory) leaves it.
template <typename F>
int c_entry(F&& f) noexcept {
    try {
        return f();
    } catch (...) {
        return PK_ERR_OOM;
    }
}

}  // namespace pk
