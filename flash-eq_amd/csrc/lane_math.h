// Reductions over groups of 1, 2, 4, ... 64 neighbouring lanes, of which every lane gets the result; sums along a wave.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace feq {
namespace {

template <int CTRL>
__device__ __forceinline__ uint32_t dpp_u(uint32_t v) {
    return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, 0xF, 0xF, false));
}

// op over the lane's group of g lanes (uniform): neighbours within 16 lanes by data-parallel moves (no LDS round
// trip, which __shfl_xor takes), 16-lane rows and halves by lane swaps.  op is associative and commutative but for
// rounding, and a group's lanes all form the same sums, so the result is the same in each.
template <class Op>
__device__ __forceinline__ uint32_t group_op(uint32_t v, int g, Op op) {
    if (g > 1) v = op(v, dpp_u<0xB1>(v));      // quad_perm [1, 0, 3, 2]
    if (g > 2) v = op(v, dpp_u<0x4E>(v));      // quad_perm [2, 3, 0, 1]
    if (g > 4) v = op(v, dpp_u<0x141>(v));     // row_half_mirror: the quads of eight
    if (g > 8) v = op(v, dpp_u<0x140>(v));     // row_mirror: the eights of sixteen
    if (g > 16) {
        const auto p = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        v = op(p[0], p[1]);
    }
    if (g > 32) {
        const auto p = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        v = op(p[0], p[1]);
    }
    return v;
}

__device__ __forceinline__ float group_sum(float v, int g) {
    return __uint_as_float(group_op(__float_as_uint(v), g, [](uint32_t a, uint32_t b) {
        return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
    }));
}
__device__ __forceinline__ float group_max(float v, int g) {
    return __uint_as_float(group_op(__float_as_uint(v), g, [](uint32_t a, uint32_t b) {
        return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
    }));
}
__device__ __forceinline__ uint32_t group_max_u(uint32_t v, int g) {
    return group_op(v, g, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
}
__device__ __forceinline__ uint32_t group_min_u(uint32_t v, int g) {
    return group_op(v, g, [](uint32_t a, uint32_t b) { return a < b ? a : b; });
}

// The sum over the lanes up to this one, by a whole wave: within 16 lanes by shifts, the rows before by broadcasts of
// their last lane (masks: rows 1 and 3, then 2 and 3).
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_add(int v) {
    return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, false);
}
__device__ __forceinline__ int inclusive_sum(int v) {
    v = dpp_add<0x111, 0xF>(v);      // row_shr 1
    v = dpp_add<0x112, 0xF>(v);      // 2
    v = dpp_add<0x114, 0xF>(v);      // 4
    v = dpp_add<0x118, 0xF>(v);      // 8
    v = dpp_add<0x142, 0xA>(v);      // row_bcast 15
    return dpp_add<0x143, 0xC>(v);   // row_bcast 31
}

}  // namespace
}  // namespace feq
