// Gradients of the microscaled product: out = alpha * op(g) * values(q), fp32 sums.
//   transpose = 0:  out (m, cols), sums over n: the gradient of the left operand (q: the right one, n rows)
//   transpose = 1:  out (n, cols), sums over m: the gradient of the right operand (q: the left one, m rows)
//
// Both are products of bf16 matrices on the tensor cores.  code * block scale has at most 8 significant
// bits, so widen_kernel writes q's values as bf16 without a rounding (the tensor's scale is alpha).  g enters
// whole too: bf16 as it is, fp16 as the sum of 2 and fp32 of 3 bf16 terms of 8 bits each (split_kernel),
// whose products are summed in the same accumulators, the terms being further stages of the sum.
//
// grad_kernel: a pair of CTAs (a cluster of 2) makes output tiles of 256 x tile_n, 64 of the sum a stage.
// values(q), and g where it is transposed, lie with the sum across the rows: the instructions read them so
// (the operand's other major order), 64 columns of 64 rows a box.  Roles of the warps as in the product:
//   warp 0 copies, warp 1 (leader) issues, warps 4-11 write results while the next tile is being summed.
// With few tiles and a long sum, the sum is split; the parts go to a workspace in fp32 and add_kernel adds
// them in order, so that the result does not depend on which part ends first.
#include <atomic>

#include "mx_tile.cuh"

namespace tlb {
namespace {

constexpr int kTileM = 128, kDepth = 64;  // rows of a CTA, of the sum a stage
constexpr int kStageA = kTileM * kDepth * 2, kStageB = 128 * kDepth * 2, kStageBytes = kStageA + kStageB, kStages = 6;
constexpr int kSmem = 1024 + kStages * kStageBytes + 8 * kStaging;
constexpr int kThreads = 384, kPairs = kSms / 2;
static_assert(kSmem <= 227 * 1024 - 512, "shared memory");
constexpr unsigned kTmemColumns = 512;

__device__ unsigned g_gave_up;

struct GradParams {
    CUtensorMap map_a, map_b, map_out;
    MxRows q;                 // for the tensor's scale
    void* out;                // the result, or fp32 parts [splits][rows][out_cols padded]
    long long rows, pitch;    // of the output; elements between its rows
    int cols;
    long long sum;            // length of the sum, and stages of one term of it
    int term_stages, stages;  // stages: terms * term_stages
    int tile_n, m_tiles, n_tiles, splits;
    int transpose, scaled, vec_ok;
};

__device__ __forceinline__ void mma_bf16(unsigned d, unsigned long long a, unsigned long long b, unsigned idesc, unsigned more) {
    asm volatile(
        "{ .reg .pred p;\n setp.ne.u32 p, %4, 0;\n tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d), "l"(a), "l"(b),
        "r"(idesc), "r"(more)
        : "memory");
}

// An item is a tile of one part of the sum.
struct Item {
    int m, n, split, first, last;  // stages [first, last)
    __device__ Item(const GradParams& gp, int item) {
        n = item % gp.n_tiles;
        const int rest = item / gp.n_tiles;
        m = rest % gp.m_tiles;
        split = rest / gp.m_tiles;
        first = static_cast<int>(static_cast<long long>(gp.stages) * split / gp.splits);
        last = static_cast<int>(static_cast<long long>(gp.stages) * (split + 1) / gp.splits);
    }
};

template <typename T>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1) grad_kernel(const __grid_constant__ GradParams gp) {
    extern __shared__ unsigned char raw[];
    __shared__ unsigned long long bars[2 * kStages + 4];
    __shared__ unsigned tmem_base;
    __shared__ int gave_up;
    const unsigned smem = (smem_u32(raw) + 1023u) & ~1023u;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = threadIdx.x % 32;
    const unsigned rank = __shfl_sync(0xffffffffu, cluster_rank(), 0);
    const int items = gp.m_tiles * gp.n_tiles * gp.splits, first_item = blockIdx.x / 2, step = gridDim.x / 2;

    const unsigned full = smem_u32(bars), empty = full + 8 * kStages, acc_full = empty + 8 * kStages, acc_empty = acc_full + 16;
    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(full + 8 * s, 1);
            mbar_init(empty + 8 * s, 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(acc_full + 8 * b, 1);
            mbar_init(acc_empty + 8 * b, 16);
        }
        gave_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        tma_prefetch_map(&gp.map_a);
        tma_prefetch_map(&gp.map_b);
        if (gp.vec_ok) tma_prefetch_map(&gp.map_out);
    }
    if (warp == 1) tmem_alloc(smem_u32(&tmem_base), kTmemColumns);
    tc_fence_before();
    __syncthreads();
    cluster_sync();
    tc_fence_after();
    const unsigned tmem = __shfl_sync(0xffffffffu, tmem_base, 0);
    volatile int* stop = &gave_up;
    const int b_boxes = gp.tile_n / 128;  // boxes of 64 columns that this CTA's half of B takes

    if (warp == 0) {
        const bool issue = elect_one();
        const unsigned full_at = at_leader(full), bytes = kStageA + b_boxes * 8192;
        Ring r;
        unsigned started = 0;
        bool ok = true;
        for (int it = first_item; ok && it < items; it += step) {
            const Item item(gp, it);
            const int m0 = (2 * item.m + static_cast<int>(rank)) * kTileM, n0 = item.n * gp.tile_n + static_cast<int>(rank) * (gp.tile_n / 2);
            int term = item.first / gp.term_stages, at = item.first - term * gp.term_stages;
            for (int kt = item.first; kt < item.last; ++kt) {
                ok = mbar_wait(empty + 8 * r.s, r.parity ^ 1, stop);
                if (!ok) break;
                if (issue) {
                    const unsigned a = smem + r.s * kStageBytes, b = a + kStageA, bar = full_at + 8 * r.s;
                    if (rank == 0) mbar_arrive_tx(full + 8 * r.s, 2 * bytes);
                    if (gp.transpose) {  // terms are stacked along g's rows, which the sum runs over
                        const int row = term * static_cast<int>(gp.sum) + at * kDepth;
                        tma_load_2d(a, &gp.map_a, m0, row, bar);
                        tma_load_2d(a + 8192, &gp.map_a, m0 + 64, row, bar);
                    } else {
                        tma_load_2d(a, &gp.map_a, at * kDepth, term * static_cast<int>(gp.rows) + m0, bar);
                    }
                    for (int j = 0; j < b_boxes; ++j) tma_load_2d(b + j * 8192, &gp.map_b, n0 + j * 64, at * kDepth, bar);
                }
                __syncwarp();
                r.next(kStages);
                ++started;
                if (++at == gp.term_stages) at = 0, ++term;
            }
        }
        if (*stop && rank == 0) {  // every copy that was started lands before the pair ends
            int none = 0;
            for (unsigned j = 0; j < kStages && j < started; ++j) {
                r.back(kStages);
                mbar_wait(full + 8 * r.s, r.parity, &none);
            }
        }
    } else if (warp == 1 && rank == 0) {
        const bool issue = elect_one();
        // bits 4-5 fp32 sums, 7-9 / 10-12 bf16, 15 / 16 A / B with the sum across rows, 17-22 N / 8, 24-28 M / 16
        const unsigned idesc = 1u << 4 | 1u << 7 | 1u << 10 | (gp.transpose ? 1u << 15 : 0u) | 1u << 16 | static_cast<unsigned>(gp.tile_n / 8) << 17 |
                               (2 * kTileM / 16) << 24;
        const unsigned a_step = (gp.transpose ? 2048 : 32) >> 4;  // 16 of the sum, in the descriptor's units
        Ring r;
        unsigned count = 0;
        bool ok = true;
        for (int it = first_item; ok && it < items; it += step, ++count) {
            const Item item(gp, it);
            const unsigned buf = count & 1;
            if (!mbar_wait(acc_empty + 8 * buf, ((count >> 1) & 1) ^ 1, stop)) break;
            tc_fence_after();
            const unsigned d = tmem + buf * 256;
            for (int kt = item.first; kt < item.last; ++kt) {
                ok = mbar_wait(full + 8 * r.s, r.parity, stop);
                if (!ok) break;
                tc_fence_after();
                const unsigned a = smem + r.s * kStageBytes, b = a + kStageA;
                const unsigned long long da = gp.transpose ? smem_desc(a, 8192, 1024, 2) : smem_desc(a, 16, 1024, 2), db = smem_desc(b, 8192, 1024, 2);
                if (issue) {
#pragma unroll
                    for (int i = 0; i < kDepth / 16; ++i) mma_bf16(d, da + i * a_step, db + i * (2048 >> 4), idesc, kt > item.first || i > 0);
                    tc_commit(empty + 8 * r.s);
                    if (kt == item.last - 1) tc_commit(acc_full + 8 * buf);
                }
                __syncwarp();
                r.next(kStages);
            }
        }
    } else if (warp >= 4) {
        const int quarter = warp % 4, half = (warp - 4) / 4;
        const unsigned staging = smem + kStages * kStageBytes + (warp - 4) * kStaging;
        const float alpha = gp.scaled ? mx_tensor_scale(gp.q) : 1.0f;
        const unsigned acc_empty_at = at_leader(acc_empty);
        unsigned count = 0;
        for (int it = first_item; it < items; it += step, ++count) {
            const Item item(gp, it);
            const unsigned buf = count & 1;
            if (!mbar_wait(acc_full + 8 * buf, (count >> 1) & 1, stop)) break;
            tc_fence_after();
            const long long in_part = static_cast<long long>(2 * item.m + rank) * kTileM + quarter * 32;
            const int n0 = item.n * gp.tile_n;
            const TileOut<T> to{&gp.map_out, static_cast<T*>(gp.out), gp.pitch, item.split * (static_cast<long long>(gp.m_tiles) * 2 * kTileM) + in_part,
                                gp.splits > 1 ? 32 : static_cast<int>(min(32ll, gp.rows - in_part)), n0, min(gp.tile_n, gp.cols - n0), gp.vec_ok};
            write_tile(to, tmem + (static_cast<unsigned>(quarter * 32) << 16) + buf * 256, gp.tile_n, half, lane, staging, alpha, acc_empty_at + 8 * buf);
        }
        if (lane == 0) tma_store_wait_read();
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    cluster_sync();  // neither CTA's memory or barriers are used by the other any more
    tc_fence_after();
    if (warp == 1) tmem_free(tmem, kTmemColumns);
    if (threadIdx.x == 0 && gave_up) atomicAdd(&g_gave_up, 1u);
}

// ---- operands --------------------------------------------------------------------------------------------------
// q's values without the tensor's scale, bf16, rows of `pitch` elements; 8 values a thread.
template <int FMT>
__global__ void __launch_bounds__(256) widen_kernel(MxRows q, __nv_bfloat16* out, int pitch) {
    const int units = mx_padded(q.cols) / 8;
    const long long total = q.rows * units;
    for (long long u = blockIdx.x * 256ll + threadIdx.x; u < total; u += gridDim.x * 256ll) {
        const long long row = u / units;
        const int unit = static_cast<int>(u - row * units);
        const unsigned char* cp = q.codes + row * mx_code_pitch(FMT, q.cols);
        const float s = scale_value<FMT>(q.scales[row * mx_scale_pitch(FMT, q.cols) + unit * 8 / mx_block(FMT)]);
        float v[8];
        if (FMT == kMxfp8) {
            const uint2 c = __ldg(reinterpret_cast<const uint2*>(cp) + unit);
            e4m3_values(c.x, v);
            e4m3_values(c.y, v + 4);
        } else {
            e2m1_values(__ldg(reinterpret_cast<const unsigned*>(cp) + unit), v);
        }
        __nv_bfloat162 o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = __floats2bfloat162_rn(__fmul_rn(v[2 * i], s), __fmul_rn(v[2 * i + 1], s));
        *reinterpret_cast<uint4*>(out + row * pitch + unit * 8) = *reinterpret_cast<const uint4*>(o);
    }
}

// g as TERMS matrices of bf16, rows of `pitch` elements: each term takes the 8 leading bits of what is left.
template <typename T, int TERMS>
__global__ void __launch_bounds__(256) split_kernel(const T* g, long long rows, int cols, __nv_bfloat16* out, int pitch) {
    const long long total = rows * pitch;
    for (long long i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
        const long long row = i / pitch;
        const int c = static_cast<int>(i - row * pitch);
        float left = c < cols ? to_float<T>(g[row * cols + c]) : 0.0f;
#pragma unroll
        for (int t = 0; t < TERMS; ++t) {
            unsigned bits = __float_as_uint(left);
            if ((bits & 0x7fffffffu) > kInfBits) bits |= 0x00400000u;  // a NaN stays one
            bits &= 0xffff0000u;
            reinterpret_cast<unsigned short*>(out)[t * total + i] = static_cast<unsigned short>(bits >> 16);
            // an infinity or a NaN is whole in the first term
            left = (bits & 0x7fffffffu) >= kInfBits ? 0.0f : __fsub_rn(left, __uint_as_float(bits));
        }
    }
}

// The parts of a split sum, added in order.
template <typename T>
__global__ void __launch_bounds__(256) add_kernel(GradParams gp, const float* parts, long long part, int part_pitch, T* out) {
    const float alpha = mx_tensor_scale(gp.q);
    const long long total = gp.rows * gp.cols;
    for (long long i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
        const long long row = i / gp.cols;
        const float* p = parts + row * part_pitch + (i - row * gp.cols);
        float v = p[0];
        for (int s = 1; s < gp.splits; ++s) v = __fadd_rn(v, p[s * part]);
        out[i] = from_float<T>(__fmul_rn(v, alpha));
    }
}

template <typename T>
__global__ void __launch_bounds__(256) zero_kernel(T* out, long long total) {
    for (long long i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) out[i] = from_float<T>(0.0f);
}

int last_error() { return static_cast<int>(cudaGetLastError()); }

unsigned blocks(long long threads) {
    const long long n = (threads + 255) / 256;
    return static_cast<unsigned>(n < kSms * 32 ? n : kSms * 32);
}

// ---- the host's plan, a function of sizes and types alone ---------------------------------------------------------
struct Plan {
    int terms, g_pitch, v_pitch, part_pitch;  // elements
    bool copy_g;                              // g goes through split_kernel
    size_t v_bytes, g_bytes, part_bytes;
    GradParams gp;
};

size_t round_256(size_t n) { return (n + 255) / 256 * 256; }

Plan plan(const MxGrad& p) {
    Plan pl{};
    GradParams& gp = pl.gp;
    gp.q = p.q;
    gp.rows = p.transpose ? p.n : p.m;
    gp.sum = p.transpose ? p.m : p.n;
    gp.cols = p.q.cols;
    gp.transpose = p.transpose;
    pl.terms = p.g_dtype == kBf16 ? 1 : p.g_dtype == kF16 ? 2 : 3;
    pl.copy_g = pl.terms > 1 || p.n % 8 != 0;
    pl.g_pitch = (p.n + 7) / 8 * 8;
    pl.v_pitch = mx_padded(p.q.cols);
    gp.term_stages = static_cast<int>((gp.sum + kDepth - 1) / kDepth);
    gp.stages = pl.terms * gp.term_stages;
    gp.m_tiles = static_cast<int>((gp.rows + 2 * kTileM - 1) / (2 * kTileM));
    // Two widths; the wider copies less for each product.  And the sum in as many parts as leave no pair idle, each of
    // 16 stages at least (a part costs its writing and reading again).
    long long best = 0;
    for (int w = 128; w <= 256; w += 128) {
        const long long n_tiles = (gp.cols + w - 1) / w, tiles = gp.m_tiles * n_tiles;
        const long long most = tiles >= kPairs ? 1 : kPairs / tiles, long_enough = gp.stages / 16 > 0 ? gp.stages / 16 : 1;
        const long long splits = most < long_enough ? most : long_enough;
        const long long cost = (tiles * splits + kPairs - 1) / kPairs * ((gp.stages + splits - 1) / splits) * (w + 64);
        if (best == 0 || cost < best) {
            best = cost;
            gp.tile_n = w;
            gp.n_tiles = static_cast<int>(n_tiles);
            gp.splits = static_cast<int>(splits);
        }
    }
    pl.v_bytes = round_256(static_cast<size_t>(p.q.rows) * pl.v_pitch * 2);
    pl.g_bytes = pl.copy_g ? round_256(static_cast<size_t>(pl.terms) * p.m * pl.g_pitch * 2) : 0;
    pl.part_pitch = gp.n_tiles * gp.tile_n;
    pl.part_bytes = gp.splits > 1 ? static_cast<size_t>(gp.splits) * gp.m_tiles * 2 * kTileM * pl.part_pitch * 4 : 0;
    return pl;
}

template <typename T>
int launch_grad(const GradParams& gp, cudaStream_t st) {
    static std::atomic<unsigned long long> prepared{0};  // one bit a device
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return last_error();
    const unsigned long long bit = 1ull << (dev & 63);
    if (!(prepared.load(std::memory_order_acquire) & bit)) {
        const cudaError_t e = cudaFuncSetAttribute(grad_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
        if (e != cudaSuccess) return static_cast<int>(e);
        prepared.fetch_or(bit, std::memory_order_release);
    }
    const int items = gp.m_tiles * gp.n_tiles * gp.splits;
    grad_kernel<T><<<2 * (items < kPairs ? items : kPairs), kThreads, kSmem, st>>>(gp);
    mx_count_launch();
    return last_error();
}

template <typename T>
int launch_typed(const MxGrad& p, Plan& pl, cudaStream_t st) {
    GradParams& gp = pl.gp;
    if (gp.sum == 0) {
        zero_kernel<T><<<blocks(gp.rows * gp.cols), 256, 0, st>>>(static_cast<T*>(p.out), gp.rows * gp.cols);
        mx_count_launch();
        return last_error();
    }
    unsigned char* ws = static_cast<unsigned char*>(p.workspace);
    __nv_bfloat16* v = reinterpret_cast<__nv_bfloat16*>(ws);
    const unsigned widen_blocks = blocks(p.q.rows * (pl.v_pitch / 8));
    if (p.q.format == kNvfp4) widen_kernel<kNvfp4><<<widen_blocks, 256, 0, st>>>(p.q, v, pl.v_pitch);
    else if (p.q.format == kMxfp4) widen_kernel<kMxfp4><<<widen_blocks, 256, 0, st>>>(p.q, v, pl.v_pitch);
    else widen_kernel<kMxfp8><<<widen_blocks, 256, 0, st>>>(p.q, v, pl.v_pitch);
    mx_count_launch();
    const void* g = p.g;
    if (pl.copy_g) {
        __nv_bfloat16* terms = reinterpret_cast<__nv_bfloat16*>(ws + pl.v_bytes);
        const unsigned n = blocks(p.m * pl.g_pitch);
        if (p.g_dtype == kF32) split_kernel<float, 3><<<n, 256, 0, st>>>(static_cast<const float*>(p.g), p.m, p.n, terms, pl.g_pitch);
        else if (p.g_dtype == kF16) split_kernel<__half, 2><<<n, 256, 0, st>>>(static_cast<const __half*>(p.g), p.m, p.n, terms, pl.g_pitch);
        else split_kernel<__nv_bfloat16, 1><<<n, 256, 0, st>>>(static_cast<const __nv_bfloat16*>(p.g), p.m, p.n, terms, pl.g_pitch);
        mx_count_launch();
        g = terms;
    }
    if (int e = last_error()) return e;
    const unsigned long long g_rows = static_cast<unsigned long long>(pl.terms) * p.m;
    if (int e = mx_encode_map(&gp.map_a, 2, g, p.n, g_rows, pl.g_pitch * 2ull, 64, gp.transpose ? kDepth : kTileM, 1)) return e;
    if (int e = mx_encode_map(&gp.map_b, 2, v, p.q.cols, p.q.rows, pl.v_pitch * 2ull, 64, kDepth, 1)) return e;
    if (gp.splits > 1) {
        float* parts = reinterpret_cast<float*>(ws + pl.v_bytes + pl.g_bytes);
        const unsigned long long part_rows = static_cast<unsigned long long>(gp.m_tiles) * 2 * kTileM;
        gp.out = parts;
        gp.pitch = pl.part_pitch;
        gp.scaled = 0;
        gp.vec_ok = 1;
        const unsigned long long row_bytes = static_cast<unsigned long long>(pl.part_pitch) * 4;
        if (int e = mx_encode_map(&gp.map_out, 1, parts, row_bytes, gp.splits * part_rows, row_bytes, 128, 32, 1)) return e;
        if (int e = launch_grad<float>(gp, st)) return e;
        add_kernel<T><<<blocks(gp.rows * gp.cols), 256, 0, st>>>(gp, parts, static_cast<long long>(part_rows) * pl.part_pitch, pl.part_pitch,
                                                                 static_cast<T*>(p.out));
        mx_count_launch();
        return last_error();
    }
    gp.out = p.out;
    gp.pitch = gp.cols;
    gp.scaled = 1;
    const unsigned long long row_bytes = static_cast<unsigned long long>(gp.cols) * sizeof(T);
    gp.vec_ok = row_bytes % 16 == 0;
    if (gp.vec_ok)
        if (int e = mx_encode_map(&gp.map_out, 1, p.out, row_bytes, gp.rows, row_bytes, 128, 32, 1)) return e;
    return launch_grad<T>(gp, st);
}

}  // namespace

int mx_grad_gave_up(unsigned* count) { return static_cast<int>(cudaMemcpyFromSymbol(count, g_gave_up, sizeof *count)); }

size_t mx_grad_workspace(const MxGrad& p) {
    if (p.m == 0 || p.n == 0) return 0;
    const Plan pl = plan(p);
    return pl.v_bytes + pl.g_bytes + pl.part_bytes;
}

int launch_mx_grad(const MxGrad& p, void* stream) {
    Plan pl = plan(p);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (p.out_dtype == kF32) return launch_typed<float>(p, pl, st);
    if (p.out_dtype == kBf16) return launch_typed<__nv_bfloat16>(p, pl, st);
    return launch_typed<__half>(p, pl, st);
}

}  // namespace tlb
