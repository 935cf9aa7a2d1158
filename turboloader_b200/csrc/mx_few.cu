// Product of a few microscaled rows (a single token, up to four) with the rows of a matrix: reading the
// matrix bounds it, so it is read once, 16 bytes a lane, and multiplied on the ordinary cores.
//
// A warp takes two rows of the matrix and walks along them, 512 bytes of each at a step, four steps at a
// time (one row, four steps: 3.26 us for 4096 x 4096 nvfp4 codes, two rows, one step: 4.06, two and four:
// 3.07 us, 2.8 TB/s of a matrix that fits in L2; 16384 x 16384: 31.6 us, 4.8 TB/s, the decoding of the
// codes then bounds it).  4-bit codes are
// multiplied and summed in packed fp16, exactly: a half of a pair sums 8 products of at most 36 that are
// multiples of 1/4, at most 1152 quarters, and fp16 holds 2048.  Every 16 products the sum goes to fp32,
// times the two scales.  8-bit codes are multiplied in fp32.
#include <algorithm>

#include "mx_device.cuh"

namespace tlb {
namespace {

constexpr int kThreads = 128, kRows = 2;  // rows of the matrix a warp takes

__device__ __forceinline__ void e2m1_pairs(unsigned codes, __half2 v[4]) {
    unsigned h[4];
    asm("{ .reg .b8 a, b, c, d;\n mov.b32 {a, b, c, d}, %4;\n"
        "cvt.rn.f16x2.e2m1x2 %0, a;\n cvt.rn.f16x2.e2m1x2 %1, b;\n cvt.rn.f16x2.e2m1x2 %2, c;\n cvt.rn.f16x2.e2m1x2 %3, d;\n}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3]) : "r"(codes));
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = *reinterpret_cast<const __half2*>(&h[i]);
}

// The scales of a lane's 16 bytes of codes: nvfp4 two blocks of 16, mxfp4 one of 32, mxfp8 half a block of 32.
template <int FMT>
__device__ __forceinline__ unsigned scale_bits(const unsigned char* scales, int piece) {
    if (FMT == kNvfp4) return __ldg(reinterpret_cast<const unsigned short*>(scales) + piece);
    return __ldg(scales + (FMT == kMxfp4 ? piece : piece >> 1));
}

// sum * a * b for two e8m0 scales, added to acc.  The smaller scale comes first: a sum times the larger one may leave
// fp32's range though the result does not (rows near 1e35 times a weight near 1e-30).  A sum of products of codes is a
// multiple of 2^-18, so that times 2^-127 it is exact.  (1 % of the time of 4096 x 4096; adding the exponents took 5 to 10.)
__device__ __forceinline__ float add_scaled(float sum, float a, float b, float acc) {
    float larger;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(larger) : "f"(a), "f"(b));  // a NaN stays, and is the result
    return __fmaf_rn(__fmul_rn(sum, fminf(a, b)), larger, acc);
}

template <typename T, int FMT, int FEW>
__global__ void __launch_bounds__(kThreads) few_kernel(MxProduct p) {
    const int lane = threadIdx.x % 32;
    const int n_all = static_cast<int>(p.b.rows), few = static_cast<int>(p.a.rows);
    const int n0 = (blockIdx.x * (kThreads / 32) + threadIdx.x / 32) * kRows;
    if (n0 >= n_all) return;
    const int code_pitch = mx_code_pitch(FMT, p.a.cols), scale_pitch = mx_scale_pitch(FMT, p.a.cols);
    const unsigned char *codes[kRows], *scales[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {  // a row behind the last is read again in its place, and not written
        const long long row = min(n0 + r, n_all - 1);
        codes[r] = p.b.codes + row * code_pitch;
        scales[r] = p.b.scales + row * scale_pitch;
    }
    float acc[kRows][FEW] = {};
    const int pieces = code_pitch / 16;
#pragma unroll 4
    for (int piece = lane; piece < pieces; piece += 32) {
        uint4 w[kRows];
        unsigned ws[kRows];
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            w[r] = __ldg(reinterpret_cast<const uint4*>(codes[r]) + piece);
            ws[r] = scale_bits<FMT>(scales[r], piece);
        }
#pragma unroll
        for (int m = 0; m < FEW; ++m) {
            if (m >= few) break;
            const uint4 x = __ldg(reinterpret_cast<const uint4*>(p.a.codes + static_cast<long long>(m) * code_pitch) + piece);
            const unsigned xs = scale_bits<FMT>(p.a.scales + static_cast<long long>(m) * scale_pitch, piece);
            const unsigned xw[4] = {x.x, x.y, x.z, x.w};
            if constexpr (FMT == kMxfp8) {
                float xv[16];
#pragma unroll
                for (int i = 0; i < 4; ++i) e4m3_values(xw[i], xv + 4 * i);
                const float s = e8m0_value(xs);
#pragma unroll
                for (int r = 0; r < kRows; ++r) {
                    const unsigned ww[4] = {w[r].x, w[r].y, w[r].z, w[r].w};
                    float sum = 0.0f;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float v[4];
                        e4m3_values(ww[i], v);
#pragma unroll
                        for (int j = 0; j < 4; ++j) sum = __fmaf_rn(v[j], xv[4 * i + j], sum);
                    }
                    acc[r][m] = add_scaled(sum, s, e8m0_value(ws[r]), acc[r][m]);
                }
            } else {
                __half2 xv[16];
#pragma unroll
                for (int i = 0; i < 4; ++i) e2m1_pairs(xw[i], xv + 4 * i);
                const float s0 = FMT == kNvfp4 ? e4m3_value(xs & 0xffu) : e8m0_value(xs), s1 = FMT == kNvfp4 ? e4m3_value(xs >> 8) : s0;
#pragma unroll
                for (int r = 0; r < kRows; ++r) {
                    const unsigned ww[4] = {w[r].x, w[r].y, w[r].z, w[r].w};
                    float part[2];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        __half2 wv[8];
                        e2m1_pairs(ww[2 * h], wv);
                        e2m1_pairs(ww[2 * h + 1], wv + 4);
                        __half2 sum = __hmul2(wv[0], xv[8 * h]);
#pragma unroll
                        for (int i = 1; i < 8; ++i) sum = __hfma2(wv[i], xv[8 * h + i], sum);
                        const float2 f = __half22float2(sum);
                        part[h] = __fadd_rn(f.x, f.y);
                    }
                    if (FMT == kNvfp4) {
                        acc[r][m] = __fmaf_rn(__fmul_rn(part[0], s0), e4m3_value(ws[r] & 0xffu), acc[r][m]);
                        acc[r][m] = __fmaf_rn(__fmul_rn(part[1], s1), e4m3_value(ws[r] >> 8), acc[r][m]);
                    } else {
                        acc[r][m] = add_scaled(__fadd_rn(part[0], part[1]), s0, e8m0_value(ws[r]), acc[r][m]);
                    }
                }
            }
        }
    }
    const float alpha = __fmul_rn(mx_tensor_scale(p.a), mx_tensor_scale(p.b));
#pragma unroll
    for (int r = 0; r < kRows; ++r)
#pragma unroll
        for (int m = 0; m < FEW; ++m) {
            if (m >= few) break;
            float v = acc[r][m];
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) v = __fadd_rn(v, __shfl_xor_sync(0xffffffffu, v, d));
            if (lane == (r * FEW + m) % 32 && n0 + r < n_all)
                static_cast<T*>(p.out)[static_cast<long long>(m) * n_all + n0 + r] = from_float<T>(__fmul_rn(v, alpha));
        }
}

template <typename T, int FMT>
void launch(const MxProduct& p, cudaStream_t st) {
    const int n = static_cast<int>(p.b.rows);
    constexpr int cta_rows = kRows * (kThreads / 32);
    const unsigned grid = static_cast<unsigned>((n + cta_rows - 1) / cta_rows);
    if (p.a.rows == 1) few_kernel<T, FMT, 1><<<grid, kThreads, 0, st>>>(p);
    else if (p.a.rows == 2) few_kernel<T, FMT, 2><<<grid, kThreads, 0, st>>>(p);
    else few_kernel<T, FMT, 4><<<grid, kThreads, 0, st>>>(p);
}

template <typename T>
void by_format(const MxProduct& p, cudaStream_t st) {
    if (p.a.format == kNvfp4) launch<T, kNvfp4>(p, st);
    else if (p.a.format == kMxfp4) launch<T, kMxfp4>(p, st);
    else launch<T, kMxfp8>(p, st);
}

}  // namespace

// With one row reading bounds either way, and this kernel starts sooner.  With two to four its arithmetic grows
// with the rows, per byte of codes more for the smaller ones, while the tensor cores' time does not; a row of B
// costs as much as 1024 values at least.  us here and there, rows x N x K: nvfp4 2 x 8192 x 8192 12.1 / 14.8,
// 3 x 8192 x 4096 9.9 / 10.3, 4 x 8192 x 4096 12.0 / 10.3, 2 x 16384 x 8192 20.8 / 18.3; mxfp4 4 x 4096 x 4096
// 8.5 / 8.8, 3 x 8192 x 4096 12.2 / 9.4; mxfp8 3 x 4096 x 4096 10.8 / 11.3, 4 x 4096 x 4096 13.5 / 11.3.
bool mx_few(const MxProduct& p) {
    if (p.a.rows <= 1 || p.a.rows > 4) return p.a.rows <= 1;
    const long long most = p.a.format == kNvfp4 ? 3ll << 25 : p.a.format == kMxfp4 ? 1ll << 26 : 3ll << 24;
    return p.a.rows * p.b.rows * std::max(p.a.cols, 1024) <= most;
}

int launch_mx_few(const MxProduct& p, void* stream) {
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (p.out_dtype == kF32) by_format<float>(p, st);
    else if (p.out_dtype == kBf16) by_format<__nv_bfloat16>(p, st);
    else by_format<__half>(p, st);
    mx_count_launch();
    return static_cast<int>(cudaGetLastError());
}

}  // namespace tlb
