// Product of two matrices of microscaled rows: out[m][n] = tsA tsB sum_k (cA sA)(cB sB), fp32 sums.
#include "mx_device.cuh"

namespace tlb {
namespace {

constexpr int kTile = 64, kDepth = 32;

// value (row, k) without the tensor's scale
template <int FMT>
__device__ __forceinline__ float value_at(const MxRows& q, long long row, int k) {
    const unsigned char* c = q.codes + row * mx_code_pitch(FMT, q.cols);
    const float s = scale_value<FMT>(q.scales[row * mx_scale_pitch(FMT, q.cols) + k / mx_block(FMT)]);
    if (FMT == kMxfp8) return e4m3_value(c[k]) * s;
    float v[8];
    e2m1_values(c[k >> 1] >> ((k & 1) * 4), v);
    return v[0] * s;
}

// 64 x 64 outputs a CTA, 4 x 4 a thread.
template <typename T, int FMT>
__global__ void __launch_bounds__(256) product_kernel(MxProduct p) {
    __shared__ float as[kDepth][kTile + 1], bs[kDepth][kTile + 1];
    const long long m0 = blockIdx.x * static_cast<long long>(kTile);
    const int n0 = blockIdx.y * kTile, n = static_cast<int>(p.b.rows), k_all = p.a.cols;
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    float acc[4][4] = {};
    for (int k0 = 0; k0 < k_all; k0 += kDepth) {
        for (int e = threadIdx.x; e < kTile * kDepth; e += 256) {
            const int r = e / kDepth, k = e % kDepth;
            as[k][r] = m0 + r < p.a.rows && k0 + k < k_all ? value_at<FMT>(p.a, m0 + r, k0 + k) : 0.0f;
            bs[k][r] = n0 + r < n && k0 + k < k_all ? value_at<FMT>(p.b, n0 + r, k0 + k) : 0.0f;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kDepth; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = __fmaf_rn(as[k][ty * 4 + i], bs[k][tx * 4 + j], acc[i][j]);
        __syncthreads();
    }
    const float alpha = mx_tensor_scale(p.a) * mx_tensor_scale(p.b);
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) {
            const long long r = m0 + ty * 4 + i;
            const int c = n0 + tx * 4 + j;
            if (r < p.a.rows && c < n) static_cast<T*>(p.out)[r * n + c] = from_float<T>(acc[i][j] * alpha);
        }
}

template <typename T>
void by_format(const MxProduct& p, dim3 grid, cudaStream_t st) {
    if (p.a.format == kNvfp4) product_kernel<T, kNvfp4><<<grid, 256, 0, st>>>(p);
    else if (p.a.format == kMxfp4) product_kernel<T, kMxfp4><<<grid, 256, 0, st>>>(p);
    else product_kernel<T, kMxfp8><<<grid, 256, 0, st>>>(p);
}

}  // namespace

size_t mx_matmul_workspace(const MxProduct&) { return 0; }

int launch_mx_matmul(const MxProduct& p, void* stream) {
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const long long gm = (p.a.rows + kTile - 1) / kTile, gn = (p.b.rows + kTile - 1) / kTile;
    if (gm > 0x7fffffffll || gn > 65535) return static_cast<int>(cudaErrorInvalidValue);
    const dim3 grid(static_cast<unsigned>(gm), static_cast<unsigned>(gn));
    if (p.out_dtype == kF32) by_format<float>(p, grid, st);
    else if (p.out_dtype == kBf16) by_format<__nv_bfloat16>(p, grid, st);
    else by_format<__half>(p, grid, st);
    mx_count_launch();
    return static_cast<int>(cudaGetLastError());
}

}  // namespace tlb
