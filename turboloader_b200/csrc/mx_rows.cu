// Quantisation of rows to the microscaled formats and back, as a plain matrix and through the slots of
// a cache (see include/turboloader_b200.h, "microscaled rows").
//
// Arithmetic of a block (16 values for nvfp4, 32 for mxfp4 / mxfp8) with t = fp32(x / tensor scale),
// a = max |t|:
//   nvfp4  s = e4m3(a / 6),                       code = e2m1(t / s)
//   mxfp4  s = 2^max(floor(log2 a) - 2, -127),    code = e2m1(t / s)
//   mxfp8  s = 2^max(floor(log2 a) - 8, -127),    code = e4m3(t / s)
// all roundings to nearest even, saturating.  Every code is the one that exact arithmetic on t gives:
// powers of two scale exactly, and the nvfp4 quotients are rounded correctly (a quotient of t by the
// 4-bit significand of s that is not itself a rounding border of e2m1 differs from the border by more
// than half a step of fp32, so the rounded quotient never lands on the wrong side of it).
#include <atomic>

#include "../../include/turboloader_b200.h"
#include "mx_device.cuh"

namespace tlb {
namespace {

std::atomic<unsigned long long> g_mx_launches{0};

constexpr int kThreads = 256;
constexpr int kUnit = 16;  // values a thread quantises at a time (a 32-value block is two lanes)

// t / s, rounded correctly for the s used here: one step of residual correction of t * (1/s) with
// 1/s rounded to nearest (Markstein, "Computation of elementary functions on the IBM RISC System/6000
// processor", 1990).  The residual is taken as q s - t, which keeps the sign of a zero.
__device__ __forceinline__ float quotient(float t, float s, float inv) {
    const float q = __fmul_rn(t, inv);
    return __fmaf_rn(-__fmaf_rn(q, s, -t), inv, q);
}

// 16 values (t) -> codes in c[] (2 words of 4-bit codes, 4 words of 8-bit ones) and the block's scale byte.
// For the 32-value formats lanes 2i and 2i+1 hold the two halves of a block.
template <int FMT>
__device__ __forceinline__ unsigned encode16(float t[kUnit], unsigned c[4]) {
    unsigned a = 0;
#pragma unroll
    for (int i = 0; i < kUnit; ++i) a = max(a, __float_as_uint(t[i]) & 0x7fffffffu);
    if (FMT != kNvfp4) a = max(a, __shfl_xor_sync(0xffffffffu, a, 1));
    if (a >= kInfBits) {  // an infinity or a NaN: the block reads as NaN
        c[0] = c[1] = c[2] = c[3] = 0u;
        return FMT == kNvfp4 ? 0x7fu : 0xffu;
    }
    unsigned byte;
    if (FMT == kNvfp4) {
        const float six = __fdiv_rn(__uint_as_float(a), 6.0f);
        unsigned short b2;
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(b2) : "f"(0.0f), "f"(six));
        byte = b2 & 0xffu;
        if (byte == 0u) {
            c[0] = c[1] = c[2] = c[3] = 0u;
            return 0u;
        }
        const float s = e4m3_value(byte), inv = __frcp_rn(s);
#pragma unroll
        for (int i = 0; i < kUnit; ++i) t[i] = quotient(t[i], s, inv);
    } else {
        const int emax = FMT == kMxfp4 ? 2 : 8;
        byte = max(static_cast<int>(a >> 23) - emax, 0);             // biased exponent of s
        const float up = __uint_as_float((254u - byte) << 23);       // 2^-(byte - 127), exact
#pragma unroll
        for (int i = 0; i < kUnit; ++i) t[i] = __fmul_rn(t[i], up);
    }
    if (FMT == kMxfp8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) c[i] = e4m3_codes(t + 4 * i);
    } else {
        c[0] = e2m1_codes(t);
        c[1] = e2m1_codes(t + 8);
    }
    return byte;
}

template <typename T>
__device__ __forceinline__ void load16(const T* p, int left, bool aligned, float t[kUnit]) {
    if (aligned && left >= kUnit) {
        constexpr int per = 16 / sizeof(T);
#pragma unroll
        for (int j = 0; j < kUnit / per; ++j) {
            const uint4 w = __ldg(reinterpret_cast<const uint4*>(p) + j);
            T e[per];
            *reinterpret_cast<uint4*>(e) = w;
#pragma unroll
            for (int i = 0; i < per; ++i) t[j * per + i] = to_float<T>(e[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < kUnit; ++i) t[i] = i < left ? to_float<T>(p[i]) : 0.0f;
    }
}

// Claims of a write whose samples may name the same slot: the last sample wins.  owner[slot] becomes
// the largest sample number that names it; the words are -1 again after release_kernel.
__global__ void claim_kernel(const long long* index, long long n, long long slots, int* owner) {
    const long long i = blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x;
    if (i >= n) return;
    const long long s = index[i];
    if (s >= 0 && s < slots) atomicMax(owner + s, static_cast<int>(i));
}
__global__ void release_kernel(const long long* index, long long n, long long slots, int* owner) {
    const long long i = blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x;
    if (i >= n) return;
    const long long s = index[i];
    if (s >= 0 && s < slots) owner[s] = -1;
}

// One CTA quantises `rows_per_cta` consecutive rows of the call.
template <typename T, int FMT>
__global__ void __launch_bounds__(kThreads) write_kernel(MxMove p, int rows_per_cta, bool aligned) {
    const int units = mx_padded(p.q.cols) / kUnit;
    const long long total = p.n * p.tokens;
    const long long row0 = blockIdx.x * static_cast<long long>(rows_per_cta);
    const int rows = static_cast<int>(min(static_cast<long long>(rows_per_cta), total - row0));
    const float ts = mx_tensor_scale(p.q);
    __shared__ long long dest[kThreads];  // cache row of every row of this CTA, or -1
    if (p.index) {
        // Which samples of this CTA lose their slot to a later sample of the same call.
        const long long first = row0 / p.tokens, last = (row0 + rows - 1) / p.tokens;
        for (long long i = first; i <= last; ++i) {
            const long long s = p.index[i];
            bool lose = s < 0 || s >= p.slots;
            if (lose && threadIdx.x == 0 && p.status) atomicOr(p.status, TLB_DEV_BAD_INDEX);
            if (!lose && p.use_owner) lose = p.owner[s] != static_cast<int>(i);
            if (!lose && !p.use_owner) {
                bool later = false;
                for (long long j = i + 1 + threadIdx.x; j < p.n; j += kThreads) later |= p.index[j] == s;
                lose = __syncthreads_or(later);
            }
            int len = p.lengths ? p.lengths[i] : p.tokens;
            if (len < 0 || len > p.tokens) {
                len = len < 0 ? 0 : p.tokens;
                if (threadIdx.x == 0 && p.status) atomicOr(p.status, TLB_DEV_BAD_LENGTH);
            }
            for (int r = threadIdx.x; r < rows; r += kThreads) {
                const long long row = row0 + r;
                if (row / p.tokens != i) continue;
                const int token = static_cast<int>(row - i * p.tokens);
                dest[r] = lose || token >= len ? -1 : s * p.tokens + token;
                if (token == 0 && !lose && p.cache_lengths) p.cache_lengths[s] = len;
            }
        }
        __syncthreads();
    }
    for (int u0 = 0; u0 < rows * units; u0 += kThreads) {
        const int u = u0 + threadIdx.x;  // whole warps stay together: lanes 2i, 2i+1 share a block
        const bool in = u < rows * units;
        const int r = in ? u / units : 0;
        const int unit = in ? u - r * units : 0;
        const long long row = row0 + r;
        const long long to = !in ? -1 : p.index ? dest[r] : row;
        float t[kUnit];
        const int left = to >= 0 ? p.q.cols - unit * kUnit : 0;
        const long long sample = row / p.tokens;
        const T* x = static_cast<const T*>(p.in) + sample * p.sample_pitch + (row - sample * p.tokens) * p.row_pitch + unit * kUnit;
        load16<T>(x, left, aligned, t);
        if (ts != 1.0f) {
#pragma unroll
            for (int i = 0; i < kUnit; ++i) t[i] = __fdiv_rn(t[i], ts);
        }
        if (left < kUnit) {
#pragma unroll
            for (int i = 0; i < kUnit; ++i) t[i] = i < left ? t[i] : 0.0f;
        }
        unsigned c[4];
        const unsigned byte = encode16<FMT>(t, c);
        if (to >= 0) {
            unsigned char* cp = p.q.codes + to * mx_code_pitch(FMT, p.q.cols);
            if (FMT == kMxfp8)
                reinterpret_cast<uint4*>(cp)[unit] = make_uint4(c[0], c[1], c[2], c[3]);
            else
                reinterpret_cast<uint2*>(cp)[unit] = make_uint2(c[0], c[1]);
            unsigned char* sp = p.q.scales + to * mx_scale_pitch(FMT, p.q.cols);
            // a scale byte whose block lies behind the last value is a pad: zero
            if (FMT == kNvfp4)
                sp[unit] = left > 0 ? static_cast<unsigned char>(byte) : 0;
            else if ((unit & 1) == 0)
                sp[unit >> 1] = left > 0 ? static_cast<unsigned char>(byte) : 0;
        }
    }
}

// Slot and rows in use of sample i of a read; slot -1: the sample reads as zeros.
__device__ __forceinline__ long long read_slot(const MxMove& p, long long i, int& len) {
    const long long s = p.index ? p.index[i] : i;
    len = 0;
    if (s < 0 || s >= p.slots) return -1;
    len = p.cache_lengths ? min(max(p.cache_lengths[s], 0), p.tokens) : p.tokens;
    return s;
}

template <typename T, int FMT>
__global__ void __launch_bounds__(kThreads) read_kernel(MxMove p) {
    const int units = (p.q.cols + 7) / 8;
    const long long total = p.n * p.tokens * units;
    const float ts = mx_tensor_scale(p.q);
    for (long long u = blockIdx.x * static_cast<long long>(kThreads) + threadIdx.x; u < total;
         u += gridDim.x * static_cast<long long>(kThreads)) {
        const long long row = u / units;
        const int unit = static_cast<int>(u - row * units);
        const long long i = row / p.tokens;
        const int token = static_cast<int>(row - i * p.tokens);
        int len;
        const long long s = read_slot(p, i, len);
        if (unit == 0 && token == 0) {
            if (s < 0 && p.status) atomicOr(p.status, TLB_DEV_BAD_INDEX);
            if (p.lengths_out) p.lengths_out[i] = len;
        }
        float v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
        if (token < len) {
            const long long from = s * p.tokens + token;
            const unsigned char* cp = p.q.codes + from * mx_code_pitch(FMT, p.q.cols);
            const float sv = scale_value<FMT>(p.q.scales[from * mx_scale_pitch(FMT, p.q.cols) + unit * 8 / mx_block(FMT)]);
            if (FMT == kMxfp8) {
                e4m3_values(reinterpret_cast<const unsigned*>(cp)[2 * unit], v);
                e4m3_values(reinterpret_cast<const unsigned*>(cp)[2 * unit + 1], v + 4);
            } else {
                e2m1_values(reinterpret_cast<const unsigned*>(cp)[unit], v);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = __fmul_rn(__fmul_rn(v[j], sv), ts);
        }
        T* o = static_cast<T*>(p.out) + row * p.q.cols + unit * 8;
        const int left = p.q.cols - unit * 8;
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < left) o[j] = from_float<T>(v[j]);
    }
}

// Rows as they are held: codes and scales into packed buffers, zeros behind a sample's length.
__global__ void __launch_bounds__(kThreads) read_codes_kernel(MxMove p) {
    const int cw = mx_code_pitch(p.q.format, p.q.cols) / 16, sw = mx_scale_pitch(p.q.format, p.q.cols) / 4;
    const int words = cw + sw;
    const long long total = p.n * p.tokens * words;
    for (long long u = blockIdx.x * static_cast<long long>(kThreads) + threadIdx.x; u < total;
         u += gridDim.x * static_cast<long long>(kThreads)) {
        const long long row = u / words;
        const int w = static_cast<int>(u - row * words);
        const long long i = row / p.tokens;
        const int token = static_cast<int>(row - i * p.tokens);
        int len;
        const long long s = read_slot(p, i, len);
        if (w == 0 && token == 0) {
            if (s < 0 && p.status) atomicOr(p.status, TLB_DEV_BAD_INDEX);
            if (p.lengths_out) p.lengths_out[i] = len;
        }
        const bool there = token < len;
        const long long from = there ? s * p.tokens + token : 0;
        if (w < cw) {
            const uint4 z = make_uint4(0u, 0u, 0u, 0u);
            reinterpret_cast<uint4*>(p.out_codes)[row * cw + w] = there ? reinterpret_cast<const uint4*>(p.q.codes)[from * cw + w] : z;
        } else {
            reinterpret_cast<unsigned*>(p.out_scales)[row * sw + w - cw] =
                there ? reinterpret_cast<const unsigned*>(p.q.scales)[from * sw + w - cw] : 0u;
        }
    }
}

template <typename T>
void write_by_format(const MxMove& p, int grid, int rows_per_cta, bool aligned, cudaStream_t st) {
    if (p.q.format == kNvfp4) write_kernel<T, kNvfp4><<<grid, kThreads, 0, st>>>(p, rows_per_cta, aligned);
    else if (p.q.format == kMxfp4) write_kernel<T, kMxfp4><<<grid, kThreads, 0, st>>>(p, rows_per_cta, aligned);
    else write_kernel<T, kMxfp8><<<grid, kThreads, 0, st>>>(p, rows_per_cta, aligned);
}
template <typename T>
void read_by_format(const MxMove& p, int grid, cudaStream_t st) {
    if (p.q.format == kNvfp4) read_kernel<T, kNvfp4><<<grid, kThreads, 0, st>>>(p);
    else if (p.q.format == kMxfp4) read_kernel<T, kMxfp4><<<grid, kThreads, 0, st>>>(p);
    else read_kernel<T, kMxfp8><<<grid, kThreads, 0, st>>>(p);
}

int grid_for(long long threads) {
    const long long ctas = (threads + kThreads - 1) / kThreads;
    return static_cast<int>(ctas < 148 * 64 ? ctas : 148 * 64);
}

}  // namespace

void mx_count_launch() { g_mx_launches.fetch_add(1, std::memory_order_relaxed); }
unsigned long long mx_launch_count() { return g_mx_launches.load(std::memory_order_relaxed); }

int launch_mx_write(const MxMove& p0, void* stream) {
    MxMove p = p0;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int units = mx_padded(p.q.cols) / kUnit;
    const int rows_per_cta = units >= kThreads ? 1 : kThreads / units;
    const int esz = p.dtype == kF32 ? 4 : 2;
    const bool aligned = (reinterpret_cast<unsigned long long>(p.in) & 15u) == 0 && p.row_pitch * esz % 16 == 0 && p.sample_pitch * esz % 16 == 0;
    const long long grid = (p.n * p.tokens + rows_per_cta - 1) / rows_per_cta;
    if (grid > 0x7fffffffll) return static_cast<int>(cudaErrorInvalidValue);
    // Duplicates: a CTA reads the whole index per sample while that is short, else the claims are made first.
    p.use_owner = p.index && p.n > TLB_MX_SCAN_SAMPLES;
    if (p.use_owner) {
        const int ctas = static_cast<int>((p.n + kThreads - 1) / kThreads);
        claim_kernel<<<ctas, kThreads, 0, st>>>(p.index, p.n, p.slots, p.owner);
        mx_count_launch();
    }
    if (p.dtype == kF32) write_by_format<float>(p, static_cast<int>(grid), rows_per_cta, aligned, st);
    else if (p.dtype == kBf16) write_by_format<__nv_bfloat16>(p, static_cast<int>(grid), rows_per_cta, aligned, st);
    else write_by_format<__half>(p, static_cast<int>(grid), rows_per_cta, aligned, st);
    mx_count_launch();
    if (p.use_owner) {
        const int ctas = static_cast<int>((p.n + kThreads - 1) / kThreads);
        release_kernel<<<ctas, kThreads, 0, st>>>(p.index, p.n, p.slots, p.owner);
        mx_count_launch();
    }
    return static_cast<int>(cudaGetLastError());
}

int launch_mx_read(const MxMove& p, void* stream) {
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int grid = grid_for(p.n * p.tokens * ((p.q.cols + 7) / 8));
    if (p.dtype == kF32) read_by_format<float>(p, grid, st);
    else if (p.dtype == kBf16) read_by_format<__nv_bfloat16>(p, grid, st);
    else read_by_format<__half>(p, grid, st);
    mx_count_launch();
    return static_cast<int>(cudaGetLastError());
}

int launch_mx_read_codes(const MxMove& p, void* stream) {
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int words = mx_code_pitch(p.q.format, p.q.cols) / 16 + mx_scale_pitch(p.q.format, p.q.cols) / 4;
    read_codes_kernel<<<grid_for(p.n * p.tokens * words), kThreads, 0, st>>>(p);
    mx_count_launch();
    return static_cast<int>(cudaGetLastError());
}

}  // namespace tlb
