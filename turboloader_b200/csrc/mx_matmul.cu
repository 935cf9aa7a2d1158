// Product of two matrices of microscaled rows: out[m][n] = tsA tsB sum_k (cA sA)(cB sB), fp32 sums.
//
// arrange_kernel lays the scales of both out as the tensor cores take them: groups of 128 rows and 4
// scales, 512 bytes each, row r at word (r % 32) * 4 + r / 32.
//
// product_kernel: a pair of CTAs (a cluster of 2) makes output tiles of 256 x tile_n, tile_n <= 224 a
// multiple of 16; each CTA holds 128 rows of A, half of B's rows, and 128 rows of the result.  Per CTA:
//   warp 0      copies a stage -- 128 bytes of codes of every row, and their scales -- into a ring
//   warp 1      (leader) moves the stage's scales into TMEM and issues four instructions a stage
//   warps 4-11  turn finished accumulators into output rows, while the next tile is being summed
// TMEM: two accumulators of tile_n columns, then the stage's scales: 16 columns for A (4 a group), 32 for
// B.  The moves into the scale columns and the products that read them are issued by one thread and run in
// that order, so the scales need no second buffer.
//
// The pair exists because of shared memory: 4-bit products of 128 x 208 tiles read 10.8 kB an instruction
// and their copies write as much, more than the 128 bytes a cycle that an SM has; a pair reads and writes
// half of B (8192^3 nvfp4: 392 us -> 224).  Where all of a tile's A fits beside the ring (k_stages <=
// kSlots: 1024 values a row of 4 bits, 512 of 8), it stays in shared memory while the pair walks along its
// row of tiles, and only B is copied for each: less to copy, and the result is written row after row.
#include <atomic>

#include "mx_device.cuh"
#include "mx_tile.cuh"

namespace tlb {
namespace {

constexpr int kTileM = 128, kMaxTileN = 224;  // rows of a CTA, columns of the pair
constexpr int kCodesA = kTileM * 128, kCodesB = kMaxTileN / 2 * 128, kScaleA = 2048, kScaleB = 4096;
// The same shared memory either way: whole stages, or slots that keep A and a longer ring for B.
constexpr int kStages = 5, kStageBytes = kCodesA + kScaleA + kCodesB + kScaleB;
constexpr int kSlots = 4, kSlotBytes = kCodesA + kScaleA, kStagesB = 6, kStageBBytes = kCodesB + kScaleB;
constexpr int kRing = kSlots * kSlotBytes + kStagesB * kStageBBytes;
static_assert(kStages * kStageBytes <= kRing && kStageBytes % 1024 == 0 && kSlotBytes % 1024 == 0 && kStageBBytes % 1024 == 0, "layout");
static_assert(kSlots <= hold_stages(true) && kSlots <= hold_stages(false), "a resident tile's sum stays in one accumulator");
constexpr int kSmem = 1024 + kRing + 8 * kStaging;
constexpr int kThreads = 384;
static_assert(kSmem <= 227 * 1024 - 512, "shared memory");
constexpr unsigned kTmemColumns = 512, kTmemScaleA = 2 * kMaxTileN, kTmemScaleB = kTmemScaleA + 16;

struct TileParams {
    CUtensorMap map_a, map_b, map_sa, map_sb, map_out;
    MxProduct p;
    int tile_n, n_tiles, groups_n;  // groups_n: groups of 128 rows that a tile's B scales take (1 or 2)
    long long m_tiles, tiles;
    int k_stages;
    int rows_a;    // rows of A that a CTA copies for a stage: mx_box_rows
    int resident;  // A stays in shared memory over consecutive tiles of one row
    int vec_ok;    // output rows are multiples of 16 bytes: written by tensor-map copies
    int passing;   // the result is large for L2: its lines are the first to leave
};

// The tiles of a pair, row by row.  resident: a contiguous run, else every pairs-th.
struct Walk {
    long long tile, end, step;
    __device__ explicit Walk(const TileParams& tp) {
        const long long pair = blockIdx.x / 2, pairs = gridDim.x / 2;
        tile = tp.resident ? tp.tiles * pair / pairs : pair;
        end = tp.resident ? tp.tiles * (pair + 1) / pairs : tp.tiles;
        step = tp.resident ? 1 : pairs;
    }
    __device__ void place(const TileParams& tp, int& m, int& n) const {
        m = static_cast<int>(tile / tp.n_tiles);
        n = static_cast<int>(tile - static_cast<long long>(m) * tp.n_tiles);
    }
};

// Products that gave up a wait on this device since the library was loaded (their output is incomplete).
__device__ unsigned g_gave_up;

// Scale words (4 scales) of a row in one stage.
template <int FMT> constexpr int kWords = FMT == kNvfp4 ? 4 : FMT == kMxfp4 ? 2 : 1;

template <int FMT>
__device__ __forceinline__ void mma(unsigned d, unsigned long long a, unsigned long long b, unsigned idesc, unsigned sa, unsigned sb, unsigned more) {
    if (FMT == kNvfp4)
        asm volatile(
            "{ .reg .pred p;\n setp.ne.u32 p, %6, 0;\n"
            "tcgen05.mma.cta_group::2.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n}" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(more)
            : "memory");
    else if (FMT == kMxfp4)
        asm volatile(
            "{ .reg .pred p;\n setp.ne.u32 p, %6, 0;\n"
            "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n}" ::"r"(d), "l"(a),
            "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(more)
            : "memory");
    else
        asm volatile(
            "{ .reg .pred p;\n setp.ne.u32 p, %6, 0;\n"
            "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n}" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(more)
            : "memory");
}

// 32 rows of 16 bytes -> 4 TMEM columns, for each of the four groups of 32 lanes, in both CTAs from their own memory
__device__ __forceinline__ void copy_scales(unsigned tmem, unsigned smem) {
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(smem_desc(smem, 0, 128, 0)) : "memory");
}

// ---- scales ------------------------------------------------------------------------------------------------
struct Arrange {
    MxRows q;
    unsigned* out;
    int tile_rows;        // rows of a tile: 128 for A, tile_n for B
    int groups;           // groups of 128 rows a tile takes
    int words;            // words (4 scales) of a row, padded to whole stages
    long long threads;    // tiles * groups * 32 * words / 4 (rounded up)
};

// A thread takes 4 rows (r, r + 32, ...) and up to 4 words of each: reads along the rows, writes 16 bytes a group.
__device__ __forceinline__ void arrange(const Arrange& a, long long t) {
    const int quads = (a.words + 3) / 4;
    const int l = static_cast<int>(t % 32);
    const long long rest = t / 32;
    const int quad = static_cast<int>(rest % quads);
    const long long tile_group = rest / quads;
    const int group = static_cast<int>(tile_group % a.groups);
    const long long tile = tile_group / a.groups;
    const int pitch = mx_scale_pitch(a.q.format, a.q.cols) / 4;
    const bool whole = pitch % 4 == 0 && (reinterpret_cast<unsigned long long>(a.q.scales) & 15u) == 0;  // rows of 16-byte pieces
    unsigned w[4][4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        const int in_tile = group * 128 + c * 32 + l;
        const long long row = tile * a.tile_rows + in_tile;
        const bool there = in_tile < a.tile_rows && row < a.q.rows;
        const unsigned* s = reinterpret_cast<const unsigned*>(a.q.scales) + (there ? row : 0) * pitch;
        if (whole) {
            const uint4 v = there && quad * 4 < pitch ? __ldg(reinterpret_cast<const uint4*>(s) + quad) : make_uint4(0u, 0u, 0u, 0u);
            w[0][c] = v.x, w[1][c] = v.y, w[2][c] = v.z, w[3][c] = v.w;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i][c] = there && quad * 4 + i < pitch ? __ldg(s + quad * 4 + i) : 0u;
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (quad * 4 + i < a.words)
            reinterpret_cast<uint4*>(a.out)[((tile * a.words + quad * 4 + i) * a.groups + group) * 32 + l] = make_uint4(w[i][0], w[i][1], w[i][2], w[i][3]);
}

constexpr int kArrangeThreads = 128;
__global__ void __launch_bounds__(kArrangeThreads) arrange_kernel(Arrange a, Arrange b) {
    let_next_start();
    const long long t = blockIdx.x * static_cast<long long>(kArrangeThreads) + threadIdx.x;
    if (t < a.threads) arrange(a, t);
    else if (t - a.threads < b.threads) arrange(b, t - a.threads);
}

// ---- products ------------------------------------------------------------------------------------------------
// LONG: sums of more stages than an accumulator holds; A is then never resident.
template <typename T, int FMT, bool LONG>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1) product_kernel(const __grid_constant__ TileParams tp) {
    extern __shared__ unsigned char raw[];
    __shared__ unsigned long long bars[2 * kStagesB + 4 + 2 * kSlots + 1];
    __shared__ unsigned tmem_base;
    __shared__ int gave_up;
    __shared__ Pair pair;
    const unsigned smem = (smem_u32(raw) + 1023u) & ~1023u;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = threadIdx.x % 32;
    const unsigned rank = __shfl_sync(0xffffffffu, cluster_rank(), 0);
    const MxProduct& p = tp.p;
    const int tile_n = tp.tile_n;
    constexpr int hold = hold_stages(sizeof(T) == 4);
    const unsigned ring = tp.resident ? kStagesB : kStages;
    // Where A and its scales lie (of stage s, or of slot kt), and where stage s keeps B and its scales.
    const unsigned a_base = smem, a_step = tp.resident ? kSlotBytes : kStageBytes;
    const unsigned b_base = smem + (tp.resident ? kSlots * kSlotBytes : kCodesA + kScaleA), b_step = tp.resident ? kStageBBytes : kStageBytes;

    const unsigned full = smem_u32(bars), empty = full + 8 * kStagesB, acc_full = empty + 8 * kStagesB, acc_empty = acc_full + 16;
    const unsigned a_full = acc_empty + 16, a_empty = a_full + 8 * kSlots, drained = a_empty + 8 * kSlots;
    if (threadIdx.x == 0) {
        for (int s = 0; s < kStagesB; ++s) {
            mbar_init(full + 8 * s, 1);
            mbar_init(empty + 8 * s, 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(acc_full + 8 * b, 1);
            mbar_init(acc_empty + 8 * b, 16);
        }
        for (int s = 0; s < kSlots; ++s) {
            mbar_init(a_full + 8 * s, 1);
            mbar_init(a_empty + 8 * s, 1);
        }
        mbar_init(drained, 1);
        gave_up = 0;
        pair.gave_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        tma_prefetch_map(&tp.map_a);
        tma_prefetch_map(&tp.map_b);
        tma_prefetch_map(&tp.map_sa);
        tma_prefetch_map(&tp.map_sb);
        if (tp.vec_ok) tma_prefetch_map(&tp.map_out);
    }
    if (warp == 1) tmem_alloc(smem_u32(&tmem_base), kTmemColumns);
    tc_fence_before();
    __syncthreads();
    cluster_sync();
    tc_fence_after();
    const unsigned tmem = __shfl_sync(0xffffffffu, tmem_base, 0);
    volatile int* stop = &gave_up;
    const unsigned a_bytes = tp.rows_a * 128 + kWords<FMT> * 512;  // of a stage's A, and of what comes through the ring
    const unsigned ring_bytes = tile_n / 2 * 128 + kWords<FMT> * tp.groups_n * 512 + (tp.resident ? 0u : a_bytes);
    wait_for_previous();

    // Warps 0 and 1 walk their loops whole, so that addresses and descriptors are uniform; one lane issues.  (With a
    // loop of one lane, moving the operands to where these instructions take them bounded the product: 58 cycles for
    // each move of scales.)
    if (warp == 0) {
        const bool issue = elect_one();
        Ring r;
        unsigned rows = 0, started = 0, started_a = 0;
        const unsigned full_at = at_leader(full), a_full_at = at_leader(a_full);
        int last_m = -1;
        bool ok = true;
        for (Walk w(tp); ok && w.tile < w.end; w.tile += w.step) {
            int m, n;
            w.place(tp, m, n);
            const int m_block = 2 * m + static_cast<int>(rank);
            const bool new_row = tp.resident && m != last_m;
            if (new_row) {
                last_m = m;
                ++rows;
            }
            for (int kt = 0; kt < tp.k_stages; ++kt) {
                const int sa_row = (m_block * tp.k_stages + kt) * kWords<FMT>;
                if (new_row) {
                    ok = mbar_wait(a_empty + 8 * kt, rows & 1, stop);
                    if (!ok) break;
                    if (issue) {
                        const unsigned a = a_base + kt * a_step, bar = a_full_at + 8 * kt;
                        if (rank == 0) mbar_arrive_tx(a_full + 8 * kt, 2 * a_bytes);
                        tma_load_2d(a, &tp.map_a, kt * 128, m_block * kTileM, bar);
                        tma_load_2d(a + kCodesA, &tp.map_sa, 0, sa_row, bar);
                    }
                    __syncwarp();
                    ++started_a;
                }
                ok = mbar_wait(empty + 8 * r.s, r.parity ^ 1, stop);
                if (!ok) break;
                if (issue) {
                    const unsigned b = b_base + r.s * b_step, bar = full_at + 8 * r.s;
                    if (rank == 0) mbar_arrive_tx(full + 8 * r.s, 2 * ring_bytes);
                    tma_load_2d(b, &tp.map_b, kt * 128, n * tile_n + static_cast<int>(rank) * (tile_n / 2), bar);
                    tma_load_2d(b + kCodesB, &tp.map_sb, 0, (n * tp.k_stages + kt) * kWords<FMT> * tp.groups_n, bar);
                    if (!tp.resident) {
                        const unsigned a = a_base + r.s * a_step;
                        tma_load_2d(a, &tp.map_a, kt * 128, m_block * kTileM, bar);
                        tma_load_2d(a + kCodesA, &tp.map_sa, 0, sa_row, bar);
                    }
                }
                __syncwarp();
                r.next(ring);
                ++started;
            }
        }
        if (issue) {
            store_at(at_leader(smem_u32(&pair.started[rank][0])), started);
            store_at(at_leader(smem_u32(&pair.started[rank][1])), started_a);
        }
    } else if (warp == 1 && rank == 0) {
        const bool issue = elect_one();
        // bits 4-5 / 29-30 which scales of a word, 7-9 / 10-12 type of A / B, 17-22 N / 8, 23 scale type, 24-28 M / 16
        const unsigned type = FMT == kMxfp8 ? 0u : 1u;
        const unsigned idesc = type << 7 | type << 10 | static_cast<unsigned>(tile_n / 8) << 17 | (FMT == kNvfp4 ? 0u : 1u << 23) | (2 * kTileM / 16) << 24;
        Ring r;
        unsigned count = 0, rows = 0;
        int last_m = -1;
        bool ok = true;
        for (Walk w(tp); ok && w.tile < w.end; w.tile += w.step) {
            int m, n;
            w.place(tp, m, n);
            const bool new_row = tp.resident && m != last_m;
            // the last tile that needs this row's A frees its slots
            const bool row_ends = tp.resident && n == tp.n_tiles - 1;
            if (new_row) {
                last_m = m;
                ++rows;
            }
            for (int from = 0; ok && from < tp.k_stages; from += hold, ++count) {
                const unsigned buf = count & 1;
                ok = mbar_wait(acc_empty + 8 * buf, ((count >> 1) & 1) ^ 1, stop);
                if (!ok) break;
                tc_fence_after();
                const unsigned d = tmem + buf * kMaxTileN;
                const int to = LONG ? min(from + hold, tp.k_stages) : tp.k_stages;
                for (int kt = from; kt < to; ++kt) {
                    ok = (!new_row || mbar_wait(a_full + 8 * kt, (rows - 1) & 1, stop)) && mbar_wait(full + 8 * r.s, r.parity, stop);
                    if (!ok) break;
                    tc_fence_after();
                    const unsigned a = a_base + (tp.resident ? kt : r.s) * a_step, b = b_base + r.s * b_step;
                    const unsigned sa = a + kCodesA, sb = b + kCodesB;
                    const unsigned long long da = smem_desc(a, 16, 1024, 2), db = smem_desc(b, 16, 1024, 2);
                    if (issue) {
#pragma unroll
                        for (int g = 0; g < kWords<FMT>; ++g) {
                            copy_scales(tmem + kTmemScaleA + 4 * g, sa + 512 * g);
                            copy_scales(tmem + kTmemScaleB + 8 * g, sb + 512 * g * tp.groups_n);
                            if (tp.groups_n > 1) copy_scales(tmem + kTmemScaleB + 8 * g + 4, sb + 1024 * g + 512);
                        }
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int g = i * kWords<FMT> / 4;                                          // group of 4 scales
                            const unsigned id = FMT == kNvfp4 ? 0u : FMT == kMxfp4 ? (i & 1) * 2u : i;  // first scale of it
                            mma<FMT>(d, da + 2 * i, db + 2 * i, idesc | id << 4 | id << 29, tmem + kTmemScaleA + 4 * g, tmem + kTmemScaleB + 8 * g,
                                     kt > from || i > 0);
                        }
                        tc_commit(empty + 8 * r.s);
                        if (row_ends) tc_commit(a_empty + 8 * kt);
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
        const float alpha = __fmul_rn(mx_tensor_scale(p.a), mx_tensor_scale(p.b));
        const int n_all = static_cast<int>(p.b.rows);
        const unsigned acc_empty_at = at_leader(acc_empty);
        const unsigned long long policy = store_policy(tp.passing);
        unsigned count = 0;
        const unsigned lanes = tmem + (static_cast<unsigned>(quarter * 32) << 16);
        const auto place = [&](const Walk& w) {
            int m, n;
            w.place(tp, m, n);
            const long long m0 = static_cast<long long>(2 * m + rank) * kTileM + quarter * 32;
            const int n0 = n * tile_n;
            return TileOut<T>{&tp.map_out, static_cast<T*>(p.out), n_all, m0, static_cast<int>(min(32ll, p.a.rows - m0)), n0, min(tile_n, n_all - n0),
                              tp.vec_ok, policy};
        };
        bool ok = true;
        Walk w(tp);
        for (; w.tile < w.end; w.tile += w.step) {
            const TileOut<T> to = place(w);
            if constexpr (LONG) {
                TileSum<T> sum;
                for (int from = 0; from < tp.k_stages; from += hold, ++count) {
                    const unsigned buf = count & 1;
                    ok = mbar_wait(acc_full + 8 * buf, (count >> 1) & 1, stop);
                    if (!ok) break;
                    tc_fence_after();
                    sum.add(lanes + buf * kMaxTileN, tile_n, half, lane, acc_empty_at + 8 * buf);
                }
                if (!ok) break;
                sum.write(to, tile_n, half, lane, staging, alpha);
            } else {
                const unsigned buf = count & 1;
                ok = mbar_wait(acc_full + 8 * buf, (count >> 1) & 1, stop);
                if (!ok) break;
                tc_fence_after();
                write_tile(to, lanes + buf * kMaxTileN, tile_n, half, lane, staging, alpha, acc_empty_at + 8 * buf);
                ++count;
            }
        }
        for (; w.tile < w.end; w.tile += w.step) write_nan(place(w), half);  // given up
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
        if (rank == 0 && warp == 0) {
            wait_for_copies(full, ring, pair.started[0][0], pair.started[1][0], ring_bytes);
            if (tp.resident) wait_for_copies(a_full, tp.k_stages, pair.started[0][1], pair.started[1][1], a_bytes);
        }
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

int last_error() { return static_cast<int>(cudaGetLastError()); }

template <typename T, int FMT, bool LONG>
int launch_tiles(const TileParams& tp, cudaStream_t st) {
    static std::atomic<unsigned long long> prepared{0};  // one bit a device
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return last_error();
    const unsigned long long bit = 1ull << (dev & 63);
    if (!(prepared.load(std::memory_order_acquire) & bit)) {
        const cudaError_t e = cudaFuncSetAttribute(product_kernel<T, FMT, LONG>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
        if (e != cudaSuccess) return static_cast<int>(e);
        prepared.fetch_or(bit, std::memory_order_release);
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(2 * (tp.tiles < kSms / 2 ? tp.tiles : kSms / 2)));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = kSmem;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // set up while arrange_kernel runs
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, product_kernel<T, FMT, LONG>, tp);
    if (e != cudaSuccess) return static_cast<int>(e);
    mx_count_launch();
    return last_error();
}

template <typename T>
int by_format(const TileParams& tp, cudaStream_t st) {
    const bool more = tp.k_stages > hold_stages(sizeof(T) == 4);
    if (tp.p.a.format == kNvfp4) return more ? launch_tiles<T, kNvfp4, true>(tp, st) : launch_tiles<T, kNvfp4, false>(tp, st);
    if (tp.p.a.format == kMxfp4) return more ? launch_tiles<T, kMxfp4, true>(tp, st) : launch_tiles<T, kMxfp4, false>(tp, st);
    return more ? launch_tiles<T, kMxfp8, true>(tp, st) : launch_tiles<T, kMxfp8, false>(tp, st);
}

int words_of(int fmt) { return fmt == kNvfp4 ? 4 : fmt == kMxfp4 ? 2 : 1; }

// Sizes of a product's tiles, a function of its shape and format alone.
void plan(TileParams& tp) {
    const MxProduct& p = tp.p;
    tp.m_tiles = (p.a.rows + 2 * kTileM - 1) / (2 * kTileM);
    const int n = static_cast<int>(p.b.rows);
    // The width that needs the least time: rounds of tiles over the pairs, each costing its width and a fixed part.
    // Where the result's bytes weigh most (few stages a tile), tiles of whole 128-byte lines: two tiles that share lines
    // write them at different times (50176 x 4096 x 1024: 197 us with 208 columns, 183 with 192; 8192^3, where 224
    // columns copy less for each product: 224 us against 250 with 192).
    long long best = 0;
    const int line = p.out_dtype == kF32 ? 32 : 64;
    tp.k_stages = (mx_code_pitch(p.a.format, p.a.cols) + 127) / 128;
    tp.resident = tp.k_stages <= kSlots;
    tp.rows_a = mx_box_rows(p.a.rows, kTileM);
    for (int w = 16; w <= kMaxTileN; w += 16) {
        if (tp.resident && w % line && w < n && w > line) continue;
        const long long tiles = tp.m_tiles * ((n + w - 1) / w), cost = (tiles + kSms / 2 - 1) / (kSms / 2) * (w + 32);
        if (best == 0 || cost <= best) best = cost, tp.tile_n = w;
    }
    tp.n_tiles = (n + tp.tile_n - 1) / tp.tile_n;
    tp.groups_n = tp.tile_n > 128 ? 2 : 1;
    tp.tiles = tp.m_tiles * tp.n_tiles;
}
long long groups_a(const TileParams& tp) { return 2 * tp.m_tiles * tp.k_stages * words_of(tp.p.a.format); }
long long groups_b(const TileParams& tp) { return static_cast<long long>(tp.n_tiles) * tp.groups_n * tp.k_stages * words_of(tp.p.a.format); }

}  // namespace

// cuTensorMapEncodeTiled, reached through the runtime so that the library does not link libcuda.
int mx_encode_map(void* map, int element_bytes, const void* base, unsigned long long inner, unsigned long long rows, unsigned long long pitch,
                  unsigned box_inner, unsigned box_rows, int swizzle) {
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
    const CUtensorMapDataType type = element_bytes == 1   ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                     : element_bytes == 2 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                          : CU_TENSOR_MAP_DATA_TYPE_UINT32;
    const CUresult r = f(static_cast<CUtensorMap*>(map), type, 2, const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         swizzle ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? 0 : static_cast<int>(cudaErrorInvalidValue);
}

int mx_gave_up(unsigned* count) {
    unsigned grads = 0;
    if (const cudaError_t e = cudaMemcpyFromSymbol(count, g_gave_up, sizeof *count); e != cudaSuccess) return static_cast<int>(e);
    if (const int e = mx_grad_gave_up(&grads)) return e;
    *count += grads;
    return 0;
}

size_t mx_matmul_workspace(const MxProduct& p) {
    if (p.b.rows == 0 || mx_few(p)) return 0;
    TileParams tp{};
    tp.p = p;
    plan(tp);
    return static_cast<size_t>(groups_a(tp) + groups_b(tp)) * 512;
}

int launch_mx_matmul(const MxProduct& p, void* stream) {
    if (mx_few(p)) return launch_mx_few(p, stream);
    TileParams tp{};
    tp.p = p;
    plan(tp);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int fmt = p.a.format, pitch = mx_code_pitch(fmt, p.a.cols), words = words_of(fmt), n = static_cast<int>(p.b.rows);
    const int esz = p.out_dtype == kF32 ? 4 : 2;
    const long long out_pitch = static_cast<long long>(n) * esz, ga = groups_a(tp), gb = groups_b(tp);
    if (ga > 0x7fffffffll || gb > 0x7fffffffll) return static_cast<int>(cudaErrorInvalidValue);
    tp.vec_ok = out_pitch % 16 == 0;
    tp.passing = out_pitch * p.a.rows > 64ll << 20;  // half of L2 (50176 x 4096 x 1024: 131 us without, 125 with)
    unsigned char* sa = static_cast<unsigned char*>(p.workspace);
    unsigned char* sb = sa + ga * 512;
    if (int e = mx_encode_map(&tp.map_a, 1, p.a.codes, pitch, p.a.rows, pitch, 128, tp.rows_a, 1)) return e;
    if (int e = mx_encode_map(&tp.map_b, 1, p.b.codes, pitch, n, pitch, 128, tp.tile_n / 2, 1)) return e;
    if (int e = mx_encode_map(&tp.map_sa, 4, sa, 128, ga, 512, 128, words, 0)) return e;
    if (int e = mx_encode_map(&tp.map_sb, 4, sb, 128, gb, 512, 128, words * tp.groups_n, 0)) return e;
    if (tp.vec_ok)
        if (int e = mx_encode_map(&tp.map_out, 1, p.out, out_pitch, p.a.rows, out_pitch, 128, 32, 1)) return e;
    Arrange a{p.a, reinterpret_cast<unsigned*>(sa), kTileM, 1, tp.k_stages * words, 0}, b{p.b, reinterpret_cast<unsigned*>(sb), tp.tile_n, tp.groups_n, tp.k_stages * words, 0};
    const int quads = (a.words + 3) / 4;
    a.threads = 2 * tp.m_tiles * 32 * quads;
    b.threads = static_cast<long long>(tp.n_tiles) * tp.groups_n * 32 * quads;
    arrange_kernel<<<static_cast<unsigned>((a.threads + b.threads + kArrangeThreads - 1) / kArrangeThreads), kArrangeThreads, 0, st>>>(a, b);
    mx_count_launch();
    if (int e = last_error()) return e;
    if (p.out_dtype == kF32) return by_format<float>(tp, st);
    if (p.out_dtype == kBf16) return by_format<__nv_bfloat16>(tp, st);
    return by_format<__half>(tp, st);
}

}  // namespace tlb
