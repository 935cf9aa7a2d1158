// Gradients of the microscaled product: out = alpha * op(g) * values(q), fp32 sums.
//   transpose = 0:  out (m, cols), sums over n: the gradient of the left operand (q: the right one, n rows)
//   transpose = 1:  out (n, cols), sums over m: the gradient of the right operand (q: the left one, m rows)
#include "mx_device.cuh"

namespace tlb {
namespace {

constexpr int kTile = 64, kDepth = 32;

__device__ __forceinline__ float g_value(const MxGrad& p, long long at) {
    if (p.g_dtype == kF32) return static_cast<const float*>(p.g)[at];
    if (p.g_dtype == kBf16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p.g)[at]);
    return __half2float(static_cast<const __half*>(p.g)[at]);
}

__device__ __forceinline__ float q_value(const MxRows& q, long long row, int k) {
    const unsigned char* c = q.codes + row * mx_code_pitch(q.format, q.cols);
    const unsigned sb = q.scales[row * mx_scale_pitch(q.format, q.cols) + k / mx_block(q.format)];
    const float s = q.format == kNvfp4 ? e4m3_value(sb) : e8m0_value(sb);
    if (q.format == kMxfp8) return e4m3_value(c[k]) * s;
    float v[8];
    e2m1_values(c[k >> 1] >> ((k & 1) * 4), v);
    return v[0] * s;
}

// 64 x 64 outputs a CTA, 4 x 4 a thread.
__global__ void __launch_bounds__(256) grad_kernel(MxGrad p) {
    __shared__ float gs[kDepth][kTile + 1], qs[kDepth][kTile + 1];
    const long long rows = p.transpose ? p.n : p.m, sum = p.transpose ? p.m : p.n;
    const long long r0 = blockIdx.x * static_cast<long long>(kTile);
    const int c0 = blockIdx.y * kTile;
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    float acc[4][4] = {};
    for (long long s0 = 0; s0 < sum; s0 += kDepth) {
        for (int e = threadIdx.x; e < kTile * kDepth; e += 256) {
            const int r = p.transpose ? e % kTile : e / kDepth, s = p.transpose ? e / kTile : e % kDepth;
            gs[s][r] = r0 + r < rows && s0 + s < sum ? g_value(p, p.transpose ? (s0 + s) * p.n + r0 + r : (r0 + r) * p.n + s0 + s) : 0.0f;
            const int c = e % kTile, sq = e / kTile;
            qs[sq][c] = c0 + c < p.q.cols && s0 + sq < sum ? q_value(p.q, s0 + sq, c0 + c) : 0.0f;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kDepth; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = __fmaf_rn(gs[k][ty * 4 + i], qs[k][tx * 4 + j], acc[i][j]);
        __syncthreads();
    }
    const float alpha = mx_tensor_scale(p.q);
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) {
            const long long r = r0 + ty * 4 + i;
            const int c = c0 + tx * 4 + j;
            if (r >= rows || c >= p.q.cols) continue;
            const float v = acc[i][j] * alpha;
            const long long at = r * p.q.cols + c;
            if (p.out_dtype == kF32) static_cast<float*>(p.out)[at] = v;
            else if (p.out_dtype == kBf16) static_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(v);
            else static_cast<__half*>(p.out)[at] = __float2half_rn(v);
        }
}

}  // namespace

size_t mx_grad_workspace(const MxGrad&) { return 0; }

int launch_mx_grad(const MxGrad& p, void* stream) {
    const long long rows = p.transpose ? p.n : p.m;
    const long long gr = (rows + kTile - 1) / kTile, gc = (p.q.cols + kTile - 1) / kTile;
    if (gr > 0x7fffffffll || gc > 65535) return static_cast<int>(cudaErrorInvalidValue);
    grad_kernel<<<dim3(static_cast<unsigned>(gr), static_cast<unsigned>(gc)), 256, 0, static_cast<cudaStream_t>(stream)>>>(p);
    mx_count_launch();
    return static_cast<int>(cudaGetLastError());
}

}  // namespace tlb
