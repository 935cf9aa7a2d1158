// Device arithmetic of the microscaled formats.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "mx_params.h"

namespace tlb {

// bits >= this: infinity or NaN (of a value's bits without the sign)
constexpr unsigned kInfBits = 0x7f800000u;

__device__ __forceinline__ float mx_tensor_scale(const MxRows& q) { return q.scale_dev ? __fmul_rn(q.scale, __ldg(q.scale_dev)) : q.scale; }

// e4m3 byte -> float (exact)
__device__ __forceinline__ float e4m3_value(unsigned byte) {
    unsigned h2;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"(static_cast<unsigned short>(byte)));
    return __half2float(__ushort_as_half(static_cast<unsigned short>(h2 & 0xffffu)));
}
// e8m0 byte -> float (exact; 255 is NaN, 0 is 2^-127)
__device__ __forceinline__ float e8m0_value(unsigned byte) {
    return __uint_as_float(byte == 255u ? 0x7fffffffu : byte == 0u ? 0x00400000u : byte << 23);
}
template <int FMT>
__device__ __forceinline__ float scale_value(unsigned byte) {
    return FMT == kNvfp4 ? e4m3_value(byte) : e8m0_value(byte);
}

// 8 e2m1 codes -> 8 floats (exact); the low half of a byte is the earlier value
__device__ __forceinline__ void e2m1_values(unsigned codes, float v[8]) {
    unsigned h[4];
    asm("{ .reg .b8 a, b, c, d;\n mov.b32 {a, b, c, d}, %4;\n"
        "cvt.rn.f16x2.e2m1x2 %0, a;\n cvt.rn.f16x2.e2m1x2 %1, b;\n cvt.rn.f16x2.e2m1x2 %2, c;\n cvt.rn.f16x2.e2m1x2 %3, d;\n}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3]) : "r"(codes));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}
// 4 e4m3 codes -> 4 floats (exact)
__device__ __forceinline__ void e4m3_values(unsigned codes, float v[4]) {
    unsigned h[2];
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h[0]) : "h"(static_cast<unsigned short>(codes & 0xffffu)));
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h[1]) : "h"(static_cast<unsigned short>(codes >> 16)));
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}

// 8 floats -> 8 e2m1 codes, round to nearest even, saturating at 6
__device__ __forceinline__ unsigned e2m1_codes(const float v[8]) {
    unsigned r;
    asm("{ .reg .b8 a, b, c, d;\n"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n"
        "mov.b32 %0, {a, b, c, d};\n}"
        : "=r"(r) : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return r;
}
// 4 floats -> 4 e4m3 codes, round to nearest even, saturating at 448
__device__ __forceinline__ unsigned e4m3_codes(const float v[4]) {
    unsigned short lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(lo) : "f"(v[0]), "f"(v[1]));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(hi) : "f"(v[0 + 2]), "f"(v[3]));
    return static_cast<unsigned>(lo) | (static_cast<unsigned>(hi) << 16);
}

// One value of any of the input types
template <typename T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

}  // namespace tlb
