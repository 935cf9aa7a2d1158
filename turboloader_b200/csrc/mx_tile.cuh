// What the tensor-core kernels of the microscaled operators share: ring positions, and the way of a finished
// accumulator to global memory.
#pragma once
#include "mx_device.cuh"
#include "mx_tma.cuh"

namespace tlb {

// A ring position and its parity.
struct Ring {
    unsigned s = 0, parity = 0;
    __device__ void next(unsigned stages) {
        if (++s == stages) s = 0, parity ^= 1u;
    }
};

constexpr int kStaging = 32 * 128;  // an epilogue warp's 32 rows of 128 bytes

template <typename T>
struct TileOut {
    const CUtensorMap* map;  // of the whole output, boxes of 32 rows of 128 bytes, 128-byte swizzle
    T* out;
    long long pitch;         // elements between output rows
    long long m0;            // the warp's first output row, and how many of its 32 there are
    int rows;
    int n0, width;           // the tile's first output column, and how many of its columns there are
    int vec_ok;              // rows are multiples of 16 bytes
    unsigned long long policy;  // of the stores (store_policy)
};

// A chunk of 128 bytes of a warp's 32 rows, columns c0 to c0 + 128 / sizeof(T) of the tile, from registers: lane l
// holds row l.
template <typename T>
__device__ __forceinline__ void write_chunk(const TileOut<T>& to, const float* v, int c0, int tile_n, int lane, unsigned staging, float alpha) {
    constexpr int chunk = 128 / sizeof(T), per = 16 / sizeof(T);  // columns of a chunk, of 16 bytes
    const int groups = min(chunk, tile_n - c0) / 16;              // of 16 columns
    const bool whole = to.vec_ok && groups == chunk / 16;
    if (whole) {
        if (lane == 0) tma_store_wait_read();
        __syncwarp();
    }
    T o[chunk];
#pragma unroll
    for (int i = 0; i < chunk; ++i) o[i] = from_float<T>(__fmul_rn(v[i], alpha));
    const uint4* pieces = reinterpret_cast<const uint4*>(o);
    auto stage = [&]() {  // 16-byte pieces in the order of the 128-byte swizzle
#pragma unroll
        for (int i = 0; i < 8; ++i)
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(staging + lane * 128 + ((i ^ (lane & 7)) * 16)), "r"(pieces[i].x),
                         "r"(pieces[i].y), "r"(pieces[i].z), "r"(pieces[i].w)
                         : "memory");
    };
    if (whole) {
        stage();
        fence_async_shared();
        __syncwarp();
        if (lane == 0 && to.rows > 0 && c0 < to.width)
            tma_store_2d(to.map, (to.n0 + c0) * static_cast<int>(sizeof(T)), static_cast<int>(to.m0), staging, to.policy);
    } else if (to.vec_ok) {  // the tile's last, narrower chunk
        T* out = to.out + (to.m0 + lane) * to.pitch + to.n0 + c0;
        if (lane < to.rows) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i * per < groups * 16 && c0 + i * per < to.width) reinterpret_cast<uint4*>(out)[i] = pieces[i];
        }
    } else {
        __syncwarp();
        stage();
        __syncwarp();
        const int cols = min(groups * 16, to.width - c0);
        T* out = to.out + to.m0 * to.pitch + to.n0 + c0;
        for (int r = 0; r < to.rows; ++r)
            for (int c = lane; c < cols; c += 32) {
                const unsigned at = staging + r * 128 + ((c / per) ^ (r & 7)) * 16 + c % per * static_cast<int>(sizeof(T));
                if constexpr (sizeof(T) == 4) {
                    unsigned bits;
                    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(bits) : "r"(at));
                    reinterpret_cast<unsigned*>(out)[static_cast<long long>(r) * to.pitch + c] = bits;
                } else {
                    unsigned short bits;
                    asm volatile("ld.shared.b16 %0, [%1];" : "=h"(bits) : "r"(at));
                    reinterpret_cast<unsigned short*>(out)[static_cast<long long>(r) * to.pitch + c] = bits;
                }
            }
    }
}

// NaN instead of a warp's part of a tile whose sums were given up: rows x width values, every second chunk of 128 bytes of
// a row from this one on.  (A call, so that it takes no registers from the epilogue.)
template <typename T>
__device__ __noinline__ void fill_nan(T* out, long long pitch, int rows, int width) {
    constexpr int chunk = 128 / sizeof(T);
    const int lane = threadIdx.x % 32;
    for (int r = 0; r < rows; ++r)
        for (int c0 = 0; c0 < width; c0 += 2 * chunk)
            for (int c = c0 + lane; c < min(c0 + chunk, width); c += 32) out[r * pitch + c] = from_float<T>(__uint_as_float(0x7fffffffu));
}
template <typename T>
__device__ __forceinline__ void write_nan(const TileOut<T>& to, int half) {
    constexpr int chunk = 128 / sizeof(T);
    fill_nan(to.out + to.m0 * to.pitch + to.n0 + half * chunk, to.pitch, to.rows, to.width - half * chunk);
}

// The tensor cores cut where they add to an accumulator, by up to 2^-23 of the partial sum for each instruction and always
// towards zero.  So an accumulator holds this many stages (of four instructions) of a long sum, and the parts are added
// in registers, rounded to nearest.  Of a 32-bit result: 2^-18 at most, some 1e-7 of a sum of values of one sign (a plain
// fp32 sum of 20000 products: 2e-7; without this 1.2e-5, and growing with the length).  Of a 16-bit one: 2^-16, at most
// 1/32 of half a step of fp16.  Shorter parts cost time: 8192^3 nvfp4 to bf16 takes 205 us with 8 stages, 196 with 32, 198
// in one accumulator; to fp32 257 us with 4 stages, 223 with 8, 216 in one.
__host__ __device__ constexpr int hold_stages(bool result_of_32_bits) { return result_of_32_bits ? 8 : 32; }

// One warp's part of a tile of up to 256 columns whose sum comes in several accumulators: the same rows and chunks as
// write_tile's.
template <typename T>
struct TileSum {
    static constexpr int chunk = 128 / sizeof(T), chunks = 128 / chunk;
    float sum[chunks][chunk];

    __device__ __forceinline__ TileSum() {
#pragma unroll
        for (int i = 0; i < chunks; ++i)
#pragma unroll
            for (int c = 0; c < chunk; ++c) sum[i][c] = 0.0f;
    }
    __device__ __forceinline__ void add(unsigned from, int tile_n, int half, int lane, unsigned released) {
#pragma unroll
        for (int i = 0; i < chunks; ++i)
#pragma unroll
            for (int g = 0; g < chunk / 16; ++g) {
                const int c0 = (half + 2 * i) * chunk + g * 16;
                if (c0 >= tile_n) continue;
                unsigned v[16];
                tmem_load16(from + c0, v);
                tmem_load_wait();
#pragma unroll
                for (int c = 0; c < 16; ++c) sum[i][g * 16 + c] = __fadd_rn(sum[i][g * 16 + c], __uint_as_float(v[c]));
            }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_at(released);
    }
    __device__ __forceinline__ void write(const TileOut<T>& to, int tile_n, int half, int lane, unsigned staging, float alpha) {
#pragma unroll
        for (int i = 0; i < chunks; ++i)
            if ((half + 2 * i) * chunk < tile_n) write_chunk(to, sum[i], (half + 2 * i) * chunk, tile_n, lane, staging, alpha);
    }
};

// One warp's part of a tile: the 32 rows of its TMEM lanes (`from`: its lane bits and first column), every
// second chunk of 128 bytes of them, beginning with chunk `half`.  Arrives on `released` (of the leader) once
// its last columns are in registers, so that the next sums may start before the stores are done.
template <typename T>
__device__ __forceinline__ void write_tile(const TileOut<T>& to, unsigned from, int tile_n, int half, int lane, unsigned staging, float alpha,
                                           unsigned released) {
    constexpr int chunk = 128 / sizeof(T);
    auto release = [&]() {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_at(released);
    };
    if (half * chunk >= tile_n) release();
    for (int c0 = half * chunk; c0 < tile_n; c0 += 2 * chunk) {
        unsigned v[chunk];
#pragma unroll
        for (int g = 0; g < chunk / 16; ++g)
            if (c0 + g * 16 < tile_n) tmem_load16(from + c0 + g * 16, v + 16 * g);
        tmem_load_wait();
        if (c0 + 2 * chunk >= tile_n) release();
        float f[chunk];
#pragma unroll
        for (int i = 0; i < chunk; ++i) f[i] = __uint_as_float(v[i]);
        write_chunk(to, f, c0, tile_n, lane, staging, alpha);
    }
}

}  // namespace tlb
