// Reductions over the lanes of a wavefront: the steps within 16 lanes take their operand from another lane by DPP, as part of an ordinary instruction.
#pragma once
#include <hip/hip_runtime.h>

namespace gp {

// The largest of three; a quiet NaN loses, a signalling one becomes a quiet one, in whose place the largest of the others is forgotten.  (fmaxf makes it a quiet one
// first, an instruction more for each operand)
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}
// a value from the lane that a DPP control names
template <int CTRL> __device__ __forceinline__ float from_lane(float v) { return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xF, 0xF, true)); }
constexpr int DPP_XOR1 = 0xB1, DPP_XOR2 = 0x4E, DPP_MIRROR8 = 0x141, DPP_MIRROR16 = 0x140;
__device__ __forceinline__ float max_of_8_lanes(float v) {
    v = fmaxf(v, from_lane<DPP_XOR1>(v));
    v = fmaxf(v, from_lane<DPP_XOR2>(v));
    return fmaxf(v, from_lane<DPP_MIRROR8>(v));
}
__device__ __forceinline__ float max_of_wave(float v) {
    v = max_of_8_lanes(v);
    v = fmaxf(v, from_lane<DPP_MIRROR16>(v));
    v = fmaxf(v, __shfl_xor(v, 16, 64));
    return fmaxf(v, __shfl_xor(v, 32, 64));
}
__device__ __forceinline__ float sum_of_wave(float v) {
    v += from_lane<DPP_XOR1>(v);
    v += from_lane<DPP_XOR2>(v);
    v += from_lane<DPP_MIRROR8>(v);
    v += from_lane<DPP_MIRROR16>(v);
    v += __shfl_xor(v, 16, 64);
    return v + __shfl_xor(v, 32, 64);
}

}  // namespace gp
