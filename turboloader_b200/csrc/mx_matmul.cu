// Product of two matrices of microscaled rows: out[m][n] = tsA tsB sum_k (cA sA)(cB sB), fp32 sums.
//
// product_kernel: one persistent CTA per SM, output tiles of 128 x tile_n (tile_n <= 224, a multiple of
// 16), the block-scaled tensor-core instructions reading codes from shared memory and scales from TMEM.
//   warp 0     copies code tiles (128 bytes of every row a stage) into a ring of kStages stages
//   warp 1     moves the stage's scales into TMEM and issues four instructions a stage
//   warps 2-3  idle (they keep the roles below on whole groups of four warps)
//   warps 4-7  turn finished accumulators into output rows, while the next tile is being summed
//   warps 8-11 read the stage's scale bytes and lay them out as the instructions want them: of a group of
//              128 rows and 4 scales, row r takes word (r % 32) * 4 + r / 32 of 512 bytes
// TMEM: two accumulators of tile_n columns, then the stage's scales: 16 columns for A (4 a group), 32 for
// B.  The moves into the scale columns and the products that read them are issued by one thread and run in
// that order, so the scales need no second buffer.
#include <atomic>
#include <mutex>

#include "mx_device.cuh"
#include "mx_tma.cuh"

namespace tlb {
namespace {

constexpr int kTileM = 128, kMaxTileN = 224;
constexpr int kStages = 4;
constexpr int kStageA = kTileM * 128, kStageB = kMaxTileN * 128, kScaleA = 2048, kScaleB = 4096;
constexpr int kStageBytes = kStageA + kStageB + kScaleA + kScaleB;
constexpr int kStagingPitch = 144, kStaging = 32 * kStagingPitch;  // an epilogue warp's 32 rows of 128 bytes
constexpr int kSmem = 1024 + kStages * kStageBytes + 4 * kStaging + 256;
constexpr int kThreads = 384;
static_assert(kSmem <= 227 * 1024, "shared memory");
constexpr unsigned kTmemColumns = 512, kTmemScaleA = 2 * kMaxTileN, kTmemScaleB = kTmemScaleA + 16;

struct TileParams {
    CUtensorMap map_a, map_b;
    MxProduct p;
    int tile_n, n_tiles;
    long long tiles;
    int k_stages;
    int vec_ok;
};

// Scale words (4 scales) of a row in one stage, and instructions' share of them.
template <int FMT> constexpr int kWords = FMT == kNvfp4 ? 4 : FMT == kMxfp4 ? 2 : 1;

template <int FMT>
__device__ __forceinline__ void mma(unsigned d, unsigned long long a, unsigned long long b, unsigned idesc, unsigned sa, unsigned sb, unsigned more) {
    if (FMT == kNvfp4)
        asm volatile(
            "{ .reg .pred p;\n setp.ne.u32 p, %6, 0;\n"
            "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n}" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(more)
            : "memory");
    else if (FMT == kMxfp4)
        asm volatile(
            "{ .reg .pred p;\n setp.ne.u32 p, %6, 0;\n"
            "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n}" ::"r"(d), "l"(a),
            "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(more)
            : "memory");
    else
        asm volatile(
            "{ .reg .pred p;\n setp.ne.u32 p, %6, 0;\n"
            "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n}" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(more)
            : "memory");
}

// 32 rows of 16 bytes -> 4 TMEM columns, for each of the four groups of 32 lanes
__device__ __forceinline__ void copy_scales(unsigned tmem, unsigned smem) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(smem_desc(smem, 0, 128, 0)) : "memory");
}

// The scale words of `row` in stage kt: zero behind the row's end and for rows behind the last.
template <int FMT>
__device__ __forceinline__ void load_scales(const MxRows& q, long long row, int kt, unsigned w[4]) {
    constexpr int words = kWords<FMT>;
    const int pitch = mx_scale_pitch(FMT, q.cols), at = kt * words * 4;
    w[0] = w[1] = w[2] = w[3] = 0u;
    if (row >= q.rows) return;
    const unsigned char* s = q.scales + row * pitch + at;
    if (FMT == kNvfp4) {  // the pitch is a multiple of 8
        const uint2 lo = __ldg(reinterpret_cast<const uint2*>(s));
        w[0] = lo.x, w[1] = lo.y;
        if (at + 8 < pitch) {
            const uint2 hi = __ldg(reinterpret_cast<const uint2*>(s) + 1);
            w[2] = hi.x, w[3] = hi.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < words; ++i)
            if (at + 4 * i < pitch) w[i] = __ldg(reinterpret_cast<const unsigned*>(s) + i);
    }
}

template <int FMT>
__device__ __forceinline__ void store_scales(unsigned base, unsigned group_bytes, int row, const unsigned w[4]) {
    const unsigned at = base + (row / 128) * 512 + (row % 32) * 16 + (row % 128) / 32 * 4;
#pragma unroll
    for (int i = 0; i < kWords<FMT>; ++i) asm volatile("st.shared.b32 [%0], %1;" ::"r"(at + i * group_bytes), "r"(w[i]) : "memory");
}

template <typename T, int FMT>
__global__ void __launch_bounds__(kThreads, 1) product_kernel(const __grid_constant__ TileParams tp) {
    extern __shared__ unsigned char raw[];
    __shared__ unsigned long long bars[4 * kStages + 4];
    __shared__ unsigned tmem_base;
    __shared__ int gave_up;
    const unsigned smem = (smem_u32(raw) + 1023u) & ~1023u;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const MxProduct& p = tp.p;
    const int tile_n = tp.tile_n;

    const unsigned codes_full = smem_u32(bars), scales_full = codes_full + 8 * kStages, empty = scales_full + 8 * kStages;
    const unsigned acc_full = empty + 8 * kStages, acc_empty = acc_full + 16;
    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(codes_full + 8 * s, 1);
            mbar_init(scales_full + 8 * s, 4);
            mbar_init(empty + 8 * s, 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(acc_full + 8 * b, 1);
            mbar_init(acc_empty + 8 * b, 4);
        }
        gave_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        tma_prefetch_map(&tp.map_a);
        tma_prefetch_map(&tp.map_b);
    }
    if (warp == 1) tmem_alloc(smem_u32(&tmem_base), kTmemColumns);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const unsigned tmem = tmem_base;
    volatile int* stop = &gave_up;

    if (warp == 0) {
        if (lane == 0) {
            unsigned it = 0;
            const unsigned bytes = kStageA + tile_n * 128;
            bool ok = true;
            for (long long tile = blockIdx.x; ok && tile < tp.tiles; tile += gridDim.x) {
                const int m0 = static_cast<int>(tile / tp.n_tiles) * kTileM, n0 = static_cast<int>(tile % tp.n_tiles) * tile_n;
                for (int kt = 0; kt < tp.k_stages; ++kt, ++it) {
                    const unsigned s = it % kStages, round = it / kStages;
                    if (!mbar_wait(empty + 8 * s, (round & 1) ^ 1, stop)) {
                        ok = false;
                        break;
                    }
                    const unsigned a = smem + s * kStageBytes, b = a + kStageA;
                    mbar_arrive_tx(codes_full + 8 * s, bytes);
                    tma_load_2d(a, &tp.map_a, kt * 128, m0, codes_full + 8 * s);
                    tma_load_2d(b, &tp.map_b, kt * 128, n0, codes_full + 8 * s);
                }
            }
            if (!ok) {  // every copy that was started lands before the CTA ends
                int none = 0;
                for (unsigned j = it > kStages ? it - kStages : 0; j < it; ++j) mbar_wait(codes_full + 8 * (j % kStages), (j / kStages) & 1, &none);
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            // bits 4-5 / 29-30 which scales of a word, 7-9 / 10-12 type of A / B, 17-22 N / 8, 23 scale type, 24-28 M / 16
            const unsigned type = FMT == kMxfp8 ? 0u : 1u;
            const unsigned idesc = type << 7 | type << 10 | static_cast<unsigned>(tile_n / 8) << 17 | (FMT == kNvfp4 ? 0u : 1u << 23) | (kTileM / 16) << 24;
            unsigned it = 0, count = 0;
            bool ok = true;
            for (long long tile = blockIdx.x; ok && tile < tp.tiles; tile += gridDim.x, ++count) {
                const unsigned buf = count & 1;
                if (!mbar_wait(acc_empty + 8 * buf, ((count >> 1) & 1) ^ 1, stop)) break;
                tc_fence_after();
                const unsigned d = tmem + buf * kMaxTileN;
                for (int kt = 0; kt < tp.k_stages; ++kt, ++it) {
                    const unsigned s = it % kStages, parity = (it / kStages) & 1;
                    if (!mbar_wait(codes_full + 8 * s, parity, stop) || !mbar_wait(scales_full + 8 * s, parity, stop)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const unsigned a = smem + s * kStageBytes, b = a + kStageA, sa = b + kStageB, sb = sa + kScaleA;
#pragma unroll
                    for (int g = 0; g < kWords<FMT>; ++g) {
                        copy_scales(tmem + kTmemScaleA + 4 * g, sa + 512 * g);
                        copy_scales(tmem + kTmemScaleB + 8 * g, sb + 1024 * g);
                        if (tile_n > 128) copy_scales(tmem + kTmemScaleB + 8 * g + 4, sb + 1024 * g + 512);
                    }
                    const unsigned long long da = smem_desc(a, 16, 1024, 2), db = smem_desc(b, 16, 1024, 2);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int g = i * kWords<FMT> / 4;                                          // group of 4 scales
                        const unsigned id = FMT == kNvfp4 ? 0u : FMT == kMxfp4 ? (i & 1) * 2u : i;  // first scale of it
                        mma<FMT>(d, da + 2 * i, db + 2 * i, idesc | id << 4 | id << 29, tmem + kTmemScaleA + 4 * g, tmem + kTmemScaleB + 8 * g,
                                 kt > 0 || i > 0);
                    }
                    tc_commit(empty + 8 * s);
                }
                if (ok) tc_commit(acc_full + 8 * buf);
            }
        }
    } else if (warp >= 8) {
        const int t = threadIdx.x - 256;
        constexpr int depth = 3;  // stages of scale words on their way
        unsigned wa[depth][4], wb0[depth][4], wb1[depth][4];
        long long ld_tile = blockIdx.x;
        int ld_kt = 0;
        auto load = [&](int d) {
            if (ld_tile >= tp.tiles) return;
            const long long m0 = ld_tile / tp.n_tiles * kTileM;
            const int n0 = static_cast<int>(ld_tile % tp.n_tiles) * tile_n;
            load_scales<FMT>(p.a, m0 + t, ld_kt, wa[d]);
            if (t < tile_n) load_scales<FMT>(p.b, n0 + t, ld_kt, wb0[d]);
            if (t + 128 < tile_n) load_scales<FMT>(p.b, n0 + t + 128, ld_kt, wb1[d]);
            if (++ld_kt == tp.k_stages) {
                ld_kt = 0;
                ld_tile += gridDim.x;
            }
        };
        const long long mine = blockIdx.x < tp.tiles ? (tp.tiles - 1 - blockIdx.x) / gridDim.x + 1 : 0;
        const long long total = mine * tp.k_stages;
#pragma unroll
        for (int d = 0; d < depth; ++d) load(d);
        bool ok = true;
        for (long long it0 = 0; ok && it0 < total; it0 += depth) {
#pragma unroll
            for (int d = 0; d < depth; ++d) {
                const long long it = it0 + d;
                if (!ok || it >= total) break;
                const unsigned s = static_cast<unsigned>(it % kStages), round = static_cast<unsigned>(it / kStages);
                ok = mbar_wait(empty + 8 * s, (round & 1) ^ 1, stop);
                if (!ok) break;
                const unsigned sa = smem + s * kStageBytes + kStageA + kStageB, sb = sa + kScaleA;
                store_scales<FMT>(sa, 512, t, wa[d]);
                if (t < tile_n) store_scales<FMT>(sb, 1024, t, wb0[d]);
                if (t + 128 < tile_n) store_scales<FMT>(sb, 1024, t + 128, wb1[d]);
                fence_async_shared();
                __syncwarp();
                if (lane == 0) mbar_arrive(scales_full + 8 * s);
                load(d);
            }
        }
    } else if (warp >= 4) {
        const int quarter = warp - 4;
        unsigned char* staging = raw + (smem - smem_u32(raw)) + kStages * kStageBytes + quarter * kStaging;
        const float alpha = __fmul_rn(mx_tensor_scale(p.a), mx_tensor_scale(p.b));
        constexpr int chunk = 128 / sizeof(T);  // columns staged at a time
        const int n = static_cast<int>(p.b.rows);
        unsigned count = 0;
        for (long long tile = blockIdx.x; tile < tp.tiles; tile += gridDim.x, ++count) {
            const unsigned buf = count & 1;
            if (!mbar_wait(acc_full + 8 * buf, (count >> 1) & 1, stop)) break;
            tc_fence_after();
            const long long m0 = tile / tp.n_tiles * kTileM + quarter * 32;
            const int n0 = static_cast<int>(tile % tp.n_tiles) * tile_n;
            const int width = min(tile_n, n - n0);
            const int rows = static_cast<int>(min(static_cast<long long>(32), p.a.rows - m0));
            const unsigned from = tmem + (static_cast<unsigned>(quarter * 32) << 16) + buf * kMaxTileN;
            for (int c0 = 0; c0 < tile_n; c0 += chunk) {
#pragma unroll
                for (int g = 0; g < chunk / 16; ++g) {
                    if (c0 + g * 16 >= tile_n) break;
                    unsigned v[16];
                    tmem_load16(from + c0 + g * 16, v);
                    tmem_load_wait();
                    T o[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[i] = from_float<T>(__fmul_rn(__uint_as_float(v[i]), alpha));
                    uint4* to = reinterpret_cast<uint4*>(staging + lane * kStagingPitch) + g * sizeof(T);
#pragma unroll
                    for (int i = 0; i < static_cast<int>(sizeof(T)); ++i) to[i] = reinterpret_cast<const uint4*>(o)[i];
                }
                if (c0 + chunk >= tile_n) {  // the accumulator is free once its last columns are in registers
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(acc_empty + 8 * buf);
                } else {
                    __syncwarp();
                }
                const int cols = min(chunk, width - c0);
                T* out = static_cast<T*>(p.out) + m0 * n + n0 + c0;
                if (tp.vec_ok) {
                    const int piece = lane % 8;
                    for (int r = lane / 8; r < rows; r += 4)
                        if (piece * static_cast<int>(16 / sizeof(T)) < cols)
                            reinterpret_cast<uint4*>(out + static_cast<long long>(r) * n)[piece] =
                                reinterpret_cast<const uint4*>(staging + r * kStagingPitch)[piece];
                } else {
                    for (int r = 0; r < rows; ++r)
                        for (int c = lane; c < cols; c += 32)
                            out[static_cast<long long>(r) * n + c] = reinterpret_cast<const T*>(staging + r * kStagingPitch)[c];
                }
                __syncwarp();
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 1) tmem_free(tmem, kTmemColumns);
}

int last_error() { return static_cast<int>(cudaGetLastError()); }

template <typename T, int FMT>
int launch_tiles(const TileParams& tp, cudaStream_t st) {
    static std::atomic<unsigned long long> prepared{0};  // one bit a device
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return last_error();
    const unsigned long long bit = 1ull << (dev & 63);
    if (!(prepared.load(std::memory_order_acquire) & bit)) {
        const cudaError_t e = cudaFuncSetAttribute(product_kernel<T, FMT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
        if (e != cudaSuccess) return static_cast<int>(e);
        prepared.fetch_or(bit, std::memory_order_release);
    }
    const long long grid = tp.tiles < kSms ? tp.tiles : kSms;
    product_kernel<T, FMT><<<static_cast<unsigned>(grid), kThreads, kSmem, st>>>(tp);
    mx_count_launch();
    return last_error();
}

template <typename T>
int by_format(const TileParams& tp, cudaStream_t st) {
    if (tp.p.a.format == kNvfp4) return launch_tiles<T, kNvfp4>(tp, st);
    if (tp.p.a.format == kMxfp4) return launch_tiles<T, kMxfp4>(tp, st);
    return launch_tiles<T, kMxfp8>(tp, st);
}

}  // namespace

// cuTensorMapEncodeTiled, reached through the runtime so that the library does not link libcuda.
int mx_encode_map(void* map, int dtype_16, const void* base, unsigned long long inner, unsigned long long rows, unsigned long long pitch,
                  unsigned box_inner, unsigned box_rows) {
    using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static std::atomic<Encode> encode{nullptr};
    Encode f = encode.load(std::memory_order_acquire);
    if (!f) {
        void* sym = nullptr;
        cudaDriverEntryPointQueryResult q;
        const cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &sym, cudaEnableDefault, &q);
        if (e != cudaSuccess) return static_cast<int>(e);
        if (q != cudaDriverEntryPointSuccess || !sym) return static_cast<int>(cudaErrorNotSupported);
        f = reinterpret_cast<Encode>(sym);
        encode.store(f, std::memory_order_release);
    }
    const cuuint64_t dims[2] = {inner, rows}, strides[1] = {pitch};
    const cuuint32_t box[2] = {box_inner, box_rows}, step[2] = {1, 1};
    const CUresult r = f(static_cast<CUtensorMap*>(map), dtype_16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8, 2,
                         const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? 0 : static_cast<int>(cudaErrorInvalidValue);
}

size_t mx_matmul_workspace(const MxProduct&) { return 0; }

int launch_mx_matmul(const MxProduct& p, void* stream) {
    TileParams tp{};
    tp.p = p;
    const int fmt = p.a.format, pitch = mx_code_pitch(fmt, p.a.cols);
    const long long m_tiles = (p.a.rows + kTileM - 1) / kTileM;
    const int n = static_cast<int>(p.b.rows);
    // The width that needs the least time: rounds of tiles over the SMs, each costing its width and a fixed part.
    long long best = 0;
    for (int w = 16; w <= kMaxTileN; w += 16) {
        const long long tiles = m_tiles * ((n + w - 1) / w), cost = (tiles + kSms - 1) / kSms * (w + 32);
        if (best == 0 || cost <= best) best = cost, tp.tile_n = w;
    }
    tp.n_tiles = (n + tp.tile_n - 1) / tp.tile_n;
    tp.tiles = m_tiles * tp.n_tiles;
    tp.k_stages = (pitch + 127) / 128;
    const int esz = p.out_dtype == kF32 ? 4 : 2;
    tp.vec_ok = static_cast<long long>(n) * esz % 16 == 0;
    if (int e = mx_encode_map(&tp.map_a, 0, p.a.codes, pitch, p.a.rows, pitch, 128, kTileM)) return e;
    if (int e = mx_encode_map(&tp.map_b, 0, p.b.codes, pitch, n, pitch, 128, tp.tile_n)) return e;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (p.out_dtype == kF32) return by_format<float>(tp, st);
    if (p.out_dtype == kBf16) return by_format<__nv_bfloat16>(tp, st);
    return by_format<__half>(tp, st);
}

}  // namespace tlb
