// Gradients of the microscaled product a * b^T, g (m, n) its result's gradient, fp32 sums:
//   of a:  out (m, cols) = g * values(b), sums over n          of b:  out (n, cols) = g^T * values(a), sums over m
//
// Both are products of bf16 matrices on the tensor cores.  code * block scale has at most 8 significant bits, so
// operands_kernel writes the values as bf16 without a rounding (the tensor's scale is alpha).  g enters whole
// too: bf16 as it is, fp16 as the sum of 2 and fp32 of 3 bf16 terms of 8 bits each, whose products are summed in
// the same accumulators, the terms being further stages of the sum.  Both as far as bf16 reaches down: its least
// subnormal is 2^-133.  What lies below it of an fp32 g (whole from 2^-110 on) is dropped, and the smallest codes of
// mxfp8 blocks whose largest value is under 2^-118 are rounded to it: less than 2^-133 a value either way.
//
// grad_kernel: a pair of CTAs (a cluster of 2) makes output tiles of 256 x tile_n, 64 of the sum a stage.
// The values, and g where it is transposed, lie with the sum across the rows: the instructions read them so
// (the operand's other major order), 64 columns of 64 rows a box.  Roles of the warps as in the product:
//   warp 0 copies, warp 1 (leader) issues, warps 4-11 write results while the next tile is being summed.
// Accumulators are taken out every hold_stages stages and added in registers, rounding to nearest (12544 x 1000 x 1024, g
// fp32: 7.4e-6 off without it, 1.6e-7 with it).
// With few tiles and a long sum, the sum is split; the parts go to a workspace in fp32 and add_kernel adds
// them in order, so that the result does not depend on which part ends first.
#include <atomic>

#include "mx_tile.cuh"

namespace tlb {
namespace {

constexpr int kTileM = 128, kDepth = 64;  // rows of a CTA, of the sum a stage
constexpr int kStageA = kTileM * kDepth * 2, kBoxB = 64 * kDepth * 2;  // bytes; kBoxB: 64 columns
constexpr int kRing = 6 * (kStageA + 2 * kBoxB), kMaxStages = kRing / (kStageA + kBoxB);  // 6 stages of 256 columns, 8 of 128
constexpr int kSmem = 1024 + kRing + 8 * kStaging;
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
    int rows_a;               // rows of a copy of g: as rows_a of the product; 64 when g is transposed, in two copies
    int hold;                 // stages that an accumulator holds: hold_stages
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
    __shared__ unsigned long long bars[2 * kMaxStages + 5];
    __shared__ unsigned tmem_base;
    __shared__ int gave_up;
    __shared__ Pair pair;
    const unsigned smem = (smem_u32(raw) + 1023u) & ~1023u;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = threadIdx.x % 32;
    const unsigned rank = __shfl_sync(0xffffffffu, cluster_rank(), 0);
    const int items = gp.m_tiles * gp.n_tiles * gp.splits, first_item = blockIdx.x / 2, step = gridDim.x / 2;

    const unsigned full = smem_u32(bars), empty = full + 8 * kMaxStages, acc_full = empty + 8 * kMaxStages, acc_empty = acc_full + 16, drained = acc_empty + 16;
    const int b_boxes = gp.tile_n / 128;  // boxes of 64 columns that this CTA's half of B takes
    const unsigned stage_bytes = kStageA + b_boxes * kBoxB, ring = kRing / stage_bytes;
    if (threadIdx.x == 0) {
        for (int s = 0; s < kMaxStages; ++s) {
            mbar_init(full + 8 * s, 1);
            mbar_init(empty + 8 * s, 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(acc_full + 8 * b, 1);
            mbar_init(acc_empty + 8 * b, 16);
        }
        mbar_init(drained, 1);
        gave_up = 0;
        pair.gave_up = 0;
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
    const unsigned copied = b_boxes * kBoxB + gp.rows_a * (gp.transpose ? 256u : 128u);  // bytes of a stage, of each CTA
    wait_for_previous();

    if (warp == 0) {
        const bool issue = elect_one();
        const unsigned full_at = at_leader(full);
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
                    const unsigned a = smem + r.s * stage_bytes, b = a + kStageA, bar = full_at + 8 * r.s;
                    if (rank == 0) mbar_arrive_tx(full + 8 * r.s, 2 * copied);
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
                r.next(ring);
                ++started;
                if (++at == gp.term_stages) at = 0, ++term;
            }
        }
        if (issue) store_at(at_leader(smem_u32(&pair.started[rank][0])), started);
    } else if (warp == 1 && rank == 0) {
        const bool issue = elect_one();
        // bits 4-5 fp32 sums, 7-9 / 10-12 bf16, 15 / 16 A / B with the sum across rows, 17-22 N / 8, 24-28 M / 16
        const unsigned idesc = 1u << 4 | 1u << 7 | 1u << 10 | (gp.transpose ? 1u << 15 : 0u) | 1u << 16 | static_cast<unsigned>(gp.tile_n / 8) << 17 |
                               (2 * kTileM / 16) << 24;
        const unsigned a_step = (gp.transpose ? 2048 : 32) >> 4;  // 16 of the sum, in the descriptor's units
        Ring r;
        unsigned count = 0;
        bool ok = true;
        for (int it = first_item; ok && it < items; it += step) {
            const Item item(gp, it);
            for (int from = item.first; ok && from < item.last; from += gp.hold, ++count) {
                const unsigned buf = count & 1;
                ok = mbar_wait(acc_empty + 8 * buf, ((count >> 1) & 1) ^ 1, stop);
                if (!ok) break;
                tc_fence_after();
                const unsigned d = tmem + buf * 256;
                const int to = min(from + gp.hold, item.last);
                for (int kt = from; kt < to; ++kt) {
                    ok = mbar_wait(full + 8 * r.s, r.parity, stop);
                    if (!ok) break;
                    tc_fence_after();
                    const unsigned a = smem + r.s * stage_bytes, b = a + kStageA;
                    const unsigned long long da = gp.transpose ? smem_desc(a, 8192, 1024, 2) : smem_desc(a, 16, 1024, 2), db = smem_desc(b, 8192, 1024, 2);
                    if (issue) {
#pragma unroll
                        for (int i = 0; i < kDepth / 16; ++i) mma_bf16(d, da + i * a_step, db + i * (2048 >> 4), idesc, kt > from || i > 0);
                        tc_commit(empty + 8 * r.s);
                        if (kt == to - 1) tc_commit(acc_full + 8 * buf);
                    }
                    __syncwarp();
                    r.next(ring);
                }
            }
        }
    } else if (warp >= 4) {
        const int quarter = warp % 4, half = (warp - 4) / 4;
        const unsigned staging = smem + kRing + (warp - 4) * kStaging;
        const float alpha = gp.scaled ? mx_tensor_scale(gp.q) : 1.0f;
        const unsigned acc_empty_at = at_leader(acc_empty);
        const unsigned long long policy = store_policy(false);
        unsigned count = 0;
        const unsigned lanes = tmem + (static_cast<unsigned>(quarter * 32) << 16);
        const auto place = [&](const Item& item) {
            const long long in_part = static_cast<long long>(2 * item.m + rank) * kTileM + quarter * 32;
            const int n0 = item.n * gp.tile_n;
            return TileOut<T>{&gp.map_out, static_cast<T*>(gp.out), gp.pitch, item.split * (static_cast<long long>(gp.m_tiles) * 2 * kTileM) + in_part,
                              gp.splits > 1 ? 32 : static_cast<int>(min(32ll, gp.rows - in_part)), n0, min(gp.tile_n, gp.cols - n0), gp.vec_ok, policy};
        };
        bool ok = true;
        int it = first_item;
        for (; it < items; it += step) {
            const Item item(gp, it);
            TileSum<T> sum;
            for (int from = item.first; from < item.last; from += gp.hold, ++count) {
                const unsigned buf = count & 1;
                ok = mbar_wait(acc_full + 8 * buf, (count >> 1) & 1, stop);
                if (!ok) break;
                tc_fence_after();
                sum.add(lanes + buf * 256, gp.tile_n, half, lane, acc_empty_at + 8 * buf);
            }
            if (!ok) break;
            sum.write(place(item), gp.tile_n, half, lane, staging, alpha);
        }
        for (; it < items; it += step) write_nan(place(Item(gp, it)), half);  // given up
        if (lane == 0) tma_store_wait_read();
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (threadIdx.x == 0 && gave_up)
        for (unsigned r = 0; r < 2; ++r) store_at(at_rank(smem_u32(&pair.gave_up), r), 1u);
    __syncwarp();
    cluster_sync();  // neither CTA's memory or barriers are used by the other any more, unless one gave up:
    if (pair.gave_up) {
        if (rank == 0 && warp == 0) wait_for_copies(full, ring, pair.started[0][0], pair.started[1][0], copied);
        if (rank == 0 && warp == 1) {  // the instructions issued so far are done before TMEM is freed
            int none = 0;
            if (elect_one()) tc_commit(drained);
            mbar_wait(drained, 0, &none);
        }
        __syncwarp();
        cluster_sync();
    }
    tc_fence_after();
    if (warp == 1) tmem_free(tmem, kTmemColumns);
    if (threadIdx.x == 0 && gave_up) atomicAdd(&g_gave_up, 1u);
}

// ---- operands --------------------------------------------------------------------------------------------------
// Values without the tensor's scale, bf16, rows of `pitch` elements (a multiple of 128); 16 values a thread.
struct Widen {
    MxRows q;
    __nv_bfloat16* out;
    int pitch;
    long long units;  // of 16 values
};
// g as `terms` matrices of bf16, rows of `pitch` elements: each term takes the 8 leading bits of what is left; 8
// values a thread.
struct Split {
    const void* g;
    int dtype, terms, cols, pitch;
    long long rows, units;
    __nv_bfloat16* out;
};

__device__ __forceinline__ long long quick_div(long long n, int d) {
    return (n >> 32) == 0 ? static_cast<long long>(static_cast<unsigned>(n) / static_cast<unsigned>(d)) : n / d;
}

template <int FMT>
__device__ __forceinline__ void widen(const Widen& w, long long u) {
    const int per_row = w.pitch / 16;
    const long long row = quick_div(u, per_row);
    const int unit = static_cast<int>(u - row * per_row);
    const unsigned char* cp = w.q.codes + row * mx_code_pitch(FMT, w.q.cols);
    const float s = scale_value<FMT>(__ldg(w.q.scales + row * mx_scale_pitch(FMT, w.q.cols) + unit / (mx_block(FMT) / 16)));
    float v[16];
    if (FMT == kMxfp8) {
        const uint4 c = __ldg(reinterpret_cast<const uint4*>(cp) + unit);
        e4m3_values(c.x, v);
        e4m3_values(c.y, v + 4);
        e4m3_values(c.z, v + 8);
        e4m3_values(c.w, v + 12);
    } else {
        const uint2 c = __ldg(reinterpret_cast<const uint2*>(cp) + unit);
        e2m1_values(c.x, v);
        e2m1_values(c.y, v + 8);
    }
    __nv_bfloat162 o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = __floats2bfloat162_rn(__fmul_rn(v[2 * i], s), __fmul_rn(v[2 * i + 1], s));
    uint4* out = reinterpret_cast<uint4*>(w.out + row * w.pitch) + unit * 2;
    out[0] = reinterpret_cast<const uint4*>(o)[0];
    out[1] = reinterpret_cast<const uint4*>(o)[1];
}

__device__ __forceinline__ void split(const Split& p, long long u) {
    const int per_row = p.pitch / 8;
    const long long row = quick_div(u, per_row);
    const int c0 = static_cast<int>(u - row * per_row) * 8;
    float left[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const long long at = row * p.cols + c0 + i;
        left[i] = c0 + i >= p.cols  ? 0.0f
                  : p.dtype == kF32 ? __ldg(static_cast<const float*>(p.g) + at)
                  : p.dtype == kF16 ? __half2float(static_cast<const __half*>(p.g)[at])
                                    : __bfloat162float(static_cast<const __nv_bfloat16*>(p.g)[at]);
    }
    for (int t = 0; t < p.terms; ++t) {
        unsigned short o[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            unsigned bits = __float_as_uint(left[i]);
            if ((bits & 0x7fffffffu) > kInfBits) bits |= 0x00400000u;  // a NaN stays one
            bits &= 0xffff0000u;
            o[i] = static_cast<unsigned short>(bits >> 16);
            // an infinity or a NaN is whole in the first term
            left[i] = (bits & 0x7fffffffu) >= kInfBits ? 0.0f : __fsub_rn(left[i], __uint_as_float(bits));
        }
        *reinterpret_cast<uint4*>(p.out + (t * p.rows + row) * p.pitch + c0) = *reinterpret_cast<const uint4*>(o);
    }
}

// All operands of a call at once: units of a, of b, of g.
template <int FMT>
__global__ void __launch_bounds__(256) operands_kernel(Widen a, Widen b, Split g) {
    let_next_start();
    const long long total = a.units + b.units + g.units;
    for (long long u = blockIdx.x * 256ll + threadIdx.x; u < total; u += gridDim.x * 256ll) {
        if (u < a.units) widen<FMT>(a, u);
        else if (u - a.units < b.units) widen<FMT>(b, u - a.units);
        else split(g, u - a.units - b.units);
    }
}

// The parts of a split sum, added in order; 4 values a thread where rows are whole pieces of 4.
template <typename T, int N>
__global__ void __launch_bounds__(256) add_kernel(GradParams gp, const float* parts, long long part, int part_pitch, T* out) {
    const float alpha = mx_tensor_scale(gp.q);
    const int per_row = gp.cols / N;
    const long long total = gp.rows * per_row;
    for (long long i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
        const long long row = quick_div(i, per_row);
        const int c = static_cast<int>(i - row * per_row) * N;
        const float* p = parts + row * part_pitch + c;
        float v[N];
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = 0.0f;
        for (int s = 0; s < gp.splits; ++s) {
            float w[N];
            if constexpr (N == 4) *reinterpret_cast<float4*>(w) = *reinterpret_cast<const float4*>(p + s * part);
            else w[0] = p[s * part];
#pragma unroll
            for (int j = 0; j < N; ++j) v[j] = s == 0 ? w[j] : __fadd_rn(v[j], w[j]);
        }
        __align__(16) T o[N];
#pragma unroll
        for (int j = 0; j < N; ++j) o[j] = from_float<T>(__fmul_rn(v[j], alpha));
        if constexpr (N == 4 && sizeof(T) == 4) *reinterpret_cast<float4*>(out + row * gp.cols + c) = *reinterpret_cast<const float4*>(o);
        else if constexpr (N == 4) *reinterpret_cast<uint2*>(out + row * gp.cols + c) = *reinterpret_cast<const uint2*>(o);
        else out[row * gp.cols + c] = o[0];
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
size_t round_256(size_t n) { return (n + 255) / 256 * 256; }

int terms_of(int dtype) { return dtype == kBf16 ? 1 : dtype == kF16 ? 2 : 3; }

struct Shared {  // what both gradients read
    int terms, g_pitch;
    bool copy_g;
    size_t g_bytes, a_bytes, b_bytes;  // 0: not needed
};

Shared shared_of(const MxGrad& p) {
    Shared s{};
    s.terms = terms_of(p.g_dtype);
    s.copy_g = s.terms > 1 || p.n % 8 != 0;
    s.g_pitch = s.copy_g ? (p.n + 63) / 64 * 64 : p.n;  // whole 128-byte lines where g is rewritten anyway
    s.g_bytes = s.copy_g ? round_256(static_cast<size_t>(s.terms) * p.m * s.g_pitch * 2) : 0;
    s.a_bytes = p.grad_b ? round_256(static_cast<size_t>(p.m) * mx_padded(p.a.cols) * 2) : 0;
    s.b_bytes = p.grad_a ? round_256(static_cast<size_t>(p.n) * mx_padded(p.b.cols) * 2) : 0;
    return s;
}

// of_b: the gradient of b, which is transposed.
GradParams plan(const MxGrad& p, const Shared& sh, bool of_b) {
    GradParams gp{};
    gp.q = of_b ? p.a : p.b;
    gp.rows = of_b ? p.n : p.m;
    gp.sum = of_b ? p.m : p.n;
    gp.cols = gp.q.cols;
    gp.transpose = of_b;
    gp.rows_a = of_b ? kDepth : mx_box_rows(gp.rows, kTileM);
    gp.term_stages = static_cast<int>((gp.sum + kDepth - 1) / kDepth);
    gp.stages = sh.terms * gp.term_stages;
    gp.m_tiles = static_cast<int>((gp.rows + 2 * kTileM - 1) / (2 * kTileM));
    // Two widths; the wider copies less for each product.  And the sum in as many parts as leave no pair idle, each of
    // 16 stages at least; writing and adding the parts costs as much as some 24 stages.
    long long best = 0;
    for (int w = 128; w <= 256; w += 128) {
        const long long n_tiles = (gp.cols + w - 1) / w, tiles = gp.m_tiles * n_tiles;
        const long long most = tiles >= kPairs ? 1 : kPairs / tiles, long_enough = gp.stages / 16 > 0 ? gp.stages / 16 : 1;
        for (long long splits = most < long_enough ? most : long_enough;; splits = 1) {
            const long long cost = (tiles * splits + kPairs - 1) / kPairs * ((gp.stages + splits - 1) / splits + (splits > 1 ? 24 : 4)) * (w + 64);
            if (best == 0 || cost < best) {
                best = cost;
                gp.tile_n = w;
                gp.n_tiles = static_cast<int>(n_tiles);
                gp.splits = static_cast<int>(splits);
            }
            if (splits == 1) break;
        }
    }
    gp.hold = hold_stages((of_b ? p.grad_b_dtype : p.grad_a_dtype) == kF32);
    return gp;
}

int part_pitch(const GradParams& gp) { return gp.n_tiles * gp.tile_n; }
size_t part_bytes(const GradParams& gp) {
    return gp.splits > 1 ? static_cast<size_t>(gp.splits) * gp.m_tiles * 2 * kTileM * part_pitch(gp) * 4 : 0;
}

template <typename T>
int launch_grad(const GradParams& gp, cudaStream_t st, bool after_operands) {
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
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(2 * (items < kPairs ? items : kPairs)));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = kSmem;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // set up while operands_kernel runs
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = after_operands ? 1 : 0;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, grad_kernel<T>, gp);
    if (e != cudaSuccess) return static_cast<int>(e);
    mx_count_launch();
    return last_error();
}

// g: its terms, rows of g_pitch elements; values: of the other operand; parts: workspace of a split sum.
template <typename T>
int one_grad(const MxGrad& p, const Shared& sh, bool of_b, const void* g, const void* values, void* parts, void* result, bool after_operands, cudaStream_t st) {
    const long long rows = of_b ? p.n : p.m, sum = of_b ? p.m : p.n;
    if (rows == 0) return 0;
    if (sum == 0) {
        const long long total = rows * (of_b ? p.a.cols : p.b.cols);
        zero_kernel<T><<<blocks(total), 256, 0, st>>>(static_cast<T*>(result), total);
        mx_count_launch();
        return last_error();
    }
    GradParams gp = plan(p, sh, of_b);
    const unsigned long long g_rows = static_cast<unsigned long long>(sh.terms) * p.m;
    if (int e = mx_encode_map(&gp.map_a, 2, g, p.n, g_rows, sh.g_pitch * 2ull, 64, gp.rows_a, 1)) return e;
    if (int e = mx_encode_map(&gp.map_b, 2, values, gp.cols, gp.q.rows, mx_padded(gp.cols) * 2ull, 64, kDepth, 1)) return e;
    if (gp.splits > 1) {
        const unsigned long long part_rows = static_cast<unsigned long long>(gp.m_tiles) * 2 * kTileM, row_bytes = static_cast<unsigned long long>(part_pitch(gp)) * 4;
        gp.out = parts;
        gp.pitch = part_pitch(gp);
        gp.scaled = 0;
        gp.vec_ok = 1;
        if (int e = mx_encode_map(&gp.map_out, 1, parts, row_bytes, gp.splits * part_rows, row_bytes, 128, 32, 1)) return e;
        if (int e = launch_grad<float>(gp, st, after_operands)) return e;
        const long long part = static_cast<long long>(part_rows) * part_pitch(gp);
        if (gp.cols % 4 == 0)
            add_kernel<T, 4><<<blocks(gp.rows * (gp.cols / 4)), 256, 0, st>>>(gp, static_cast<const float*>(parts), part, part_pitch(gp), static_cast<T*>(result));
        else
            add_kernel<T, 1><<<blocks(gp.rows * gp.cols), 256, 0, st>>>(gp, static_cast<const float*>(parts), part, part_pitch(gp), static_cast<T*>(result));
        mx_count_launch();
        return last_error();
    }
    gp.out = result;
    gp.pitch = gp.cols;
    gp.scaled = 1;
    const unsigned long long row_bytes = static_cast<unsigned long long>(gp.cols) * sizeof(T);
    gp.vec_ok = row_bytes % 16 == 0;
    if (gp.vec_ok)
        if (int e = mx_encode_map(&gp.map_out, 1, result, row_bytes, gp.rows, row_bytes, 128, 32, 1)) return e;
    return launch_grad<T>(gp, st, after_operands);
}

int typed_grad(const MxGrad& p, const Shared& sh, bool of_b, const void* g, const void* values, void* parts, bool after_operands, cudaStream_t st) {
    const int dtype = of_b ? p.grad_b_dtype : p.grad_a_dtype;
    void* result = of_b ? p.grad_b : p.grad_a;
    if (dtype == kF32) return one_grad<float>(p, sh, of_b, g, values, parts, result, after_operands, st);
    if (dtype == kBf16) return one_grad<__nv_bfloat16>(p, sh, of_b, g, values, parts, result, after_operands, st);
    return one_grad<__half>(p, sh, of_b, g, values, parts, result, after_operands, st);
}

}  // namespace

int mx_grad_gave_up(unsigned* count) { return static_cast<int>(cudaMemcpyFromSymbol(count, g_gave_up, sizeof *count)); }

size_t mx_grad_workspace(const MxGrad& p) {
    if (p.m == 0 || p.n == 0) return 0;
    const Shared sh = shared_of(p);
    // the parts of the two, which run one after the other, share their room
    const size_t of_a = p.grad_a ? part_bytes(plan(p, sh, false)) : 0, of_b = p.grad_b ? part_bytes(plan(p, sh, true)) : 0;
    return sh.g_bytes + sh.a_bytes + sh.b_bytes + (of_a > of_b ? of_a : of_b);
}

int launch_mx_grad(const MxGrad& p, void* stream) {
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const Shared sh = shared_of(p);
    unsigned char* ws = static_cast<unsigned char*>(p.workspace);
    unsigned char *a_at = ws + sh.g_bytes, *b_at = a_at + sh.a_bytes, *parts = b_at + sh.b_bytes;
    const bool any = p.m > 0 && p.n > 0;
    if (any) {
        const Widen a{p.a, reinterpret_cast<__nv_bfloat16*>(a_at), mx_padded(p.a.cols), sh.a_bytes ? p.m * (mx_padded(p.a.cols) / 16) : 0};
        const Widen b{p.b, reinterpret_cast<__nv_bfloat16*>(b_at), mx_padded(p.b.cols), sh.b_bytes ? static_cast<long long>(p.n) * (mx_padded(p.b.cols) / 16) : 0};
        const Split g{p.g, p.g_dtype, sh.terms, p.n, sh.g_pitch, p.m, sh.copy_g ? p.m * (sh.g_pitch / 8) : 0, reinterpret_cast<__nv_bfloat16*>(ws)};
        const unsigned n = blocks(a.units + b.units + g.units);
        const int format = p.grad_b ? p.a.format : p.b.format;
        if (format == kNvfp4) operands_kernel<kNvfp4><<<n, 256, 0, st>>>(a, b, g);
        else if (format == kMxfp4) operands_kernel<kMxfp4><<<n, 256, 0, st>>>(a, b, g);
        else operands_kernel<kMxfp8><<<n, 256, 0, st>>>(a, b, g);
        mx_count_launch();
        if (int e = last_error()) return e;
    }
    const void* g = sh.copy_g ? static_cast<const void*>(ws) : p.g;
    if (p.grad_a)
        if (int e = typed_grad(p, sh, false, g, b_at, parts, any, st)) return e;
    if (p.grad_b)
        if (int e = typed_grad(p, sh, true, g, a_at, parts, any && !p.grad_a, st)) return e;
    return 0;
}

}  // namespace tlb
