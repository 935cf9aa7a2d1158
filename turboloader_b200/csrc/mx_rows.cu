// Quantisation of rows to the microscaled formats and back, as a plain matrix and through the slots of
// a cache (see include/turboloader_b200.h, "microscaled rows").
//
// Arithmetic of a block (16 values for nvfp4, 32 for mxfp4 / mxfp8) with t = fp32(x / tensor scale),
// a = max |t|:
//   nvfp4  s = e4m3(fp32(a * fp32(1/6))),         code = e2m1(t / s)
//   mxfp4  s = 2^max(floor(log2 a) - 2, -127),    code = e2m1(t / s)
//   mxfp8  s = 2^max(floor(log2 a) - 8, -127),    code = e4m3(t / s)
// all roundings to nearest even, saturating.  Given t and s, every code is the one that exact arithmetic gives:
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
constexpr int kWriteCtas = 148 * 8;  // CTAs of write_kernel that the GPU should have at least
constexpr int kMaxRounds = 8, kMaxRowsCta = kMaxRounds * kThreads / 4;  // rows of a CTA of write_kernel
static_assert(TLB_MX_SCAN_SAMPLES <= kThreads, "write_kernel reads the index with one load a thread");
constexpr int kUnit = 16;  // values a thread reads at a time
// Values a thread quantises at a time: 32 of 16 bits (a whole block, or two), 16 of 32 bits (of a block of 32 lanes
// 2i and 2i + 1 hold the halves): 64 bytes either way.
template <typename T> constexpr int kTake = sizeof(T) == 2 ? 32 : 16;

// t / s, rounded correctly for the s used here: one step of residual correction of t * (1/s) with
// 1/s rounded to nearest (Markstein, "Computation of elementary functions on the IBM RISC System/6000
// processor", 1990).  The residual is taken as q s - t, which keeps the sign of a zero.
__device__ __forceinline__ float quotient(float t, float s, float inv) {
    const float q = __fmul_rn(t, inv);
    return __fmaf_rn(-__fmaf_rn(q, s, -t), inv, q);
}

// max(|a|, |b|, |c|); a NaN among them is the result
__device__ __forceinline__ float max_magnitude(float a, float b, float c) {
    float r;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// N values (t) -> their codes in c[] and their scale bytes, the first block's lowest.
// few_bits: the values have at most 11 significant bits (16-bit inputs, scaled by a power of two).
// inverse (nvfp4): 1/s of every scale byte, rounded up for few_bits, else to nearest.
template <int FMT, int N>
__device__ __forceinline__ unsigned encode(float t[N], unsigned c[], bool few_bits, const float* inverse) {
    constexpr int block = FMT == kNvfp4 ? 16 : N, blocks = N / block;  // values of a block in this thread
    constexpr int words = (FMT == kMxfp8 ? block : block / 2) / 4;     // code words of them
    unsigned bytes = 0;
#pragma unroll
    for (int b = 0; b < blocks; ++b) {
        float* v = t + b * block;
        unsigned* cb = c + b * words;
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < block; i += 2) top = max_magnitude(top, v[i], v[i + 1]);
        unsigned a = __float_as_uint(top) & 0x7fffffffu;
        if (FMT != kNvfp4 && N == 16) a = max(a, __shfl_xor_sync(0xffffffffu, a, 1));
        unsigned byte;
        if (FMT == kNvfp4) {
            unsigned short b2;
            asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(b2) : "f"(0.0f), "f"(__fmul_rn(__uint_as_float(a), 1.0f / 6.0f)));
            byte = b2 & 0xffu;
            const float inv = inverse[byte];
            if (few_bits) {
                // Only a value that lies on a border, t = m s, could be rounded to the wrong side of it; all others are
                // 2^-11 away.  1/s rounded up and the product cut give m there, for each of the 8 significands of s
                // and the 7 borders m.
#pragma unroll
                for (int i = 0; i < block; ++i) v[i] = __fmul_rz(v[i], inv);
            } else {
                const float s = e4m3_value(byte);
#pragma unroll
                for (int i = 0; i < block; ++i) v[i] = quotient(v[i], s, inv);
            }
        } else {
            const int emax = FMT == kMxfp4 ? 2 : 8;
            byte = max(static_cast<int>(a >> 23) - emax, 0);        // biased exponent of s
            const float up = __uint_as_float((254u - byte) << 23);  // 2^-(byte - 127), exact
#pragma unroll
            for (int i = 0; i < block; ++i) v[i] = __fmul_rn(v[i], up);
        }
        if (FMT == kMxfp8) {
#pragma unroll
            for (int i = 0; i < words; ++i) cb[i] = e4m3_codes(v + 4 * i);
        } else {
#pragma unroll
            for (int i = 0; i < words; ++i) cb[i] = e2m1_codes(v + 8 * i);
        }
        if (a >= kInfBits) byte = FMT == kNvfp4 ? 0x7fu : 0xffu;  // an infinity or a NaN: the block reads as NaN
        if (a >= kInfBits || (FMT == kNvfp4 && byte == 0u)) {
#pragma unroll
            for (int i = 0; i < words; ++i) cb[i] = 0u;
        }
        bytes |= byte << (8 * b);
    }
    return bytes;
}

// N values from p, `left` of them there (zeros behind).  ALIGNED: p lies on a 32-byte boundary, and they come by
// 32-byte loads.  Else the words around p are read by 16-byte pieces from the boundary below it and shifted into
// place: an odd start costs one more load, and no load leaves the 16-byte pieces that hold values.
template <typename T, bool ALIGNED>
struct Raw {
    static constexpr int kVals = kTake<T>, kWords = kVals * sizeof(T) / 4;
    unsigned w[kWords + (ALIGNED ? 0 : 4)];

    __device__ __forceinline__ void load(const T* p, int left) {
        if constexpr (ALIGNED) {
#pragma unroll
            for (int j = 0; j < kWords / 8; ++j) {
                unsigned* v = w + 8 * j;
                const int have = left - j * static_cast<int>(32 / sizeof(T));
                if (have >= static_cast<int>(32 / sizeof(T))) {
                    asm volatile("ld.global.nc.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
                                 : "l"(reinterpret_cast<const unsigned char*>(p) + 32 * j));
                } else if (have <= 0) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[i] = 0u;
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {  // the row's end: value by value
                        if constexpr (sizeof(T) == 4) {
                            v[i] = i < have ? __ldg(reinterpret_cast<const unsigned*>(p) + 8 * j + i) : 0u;
                        } else {
                            const unsigned short* h = reinterpret_cast<const unsigned short*>(p) + 16 * j + 2 * i;
                            v[i] = (2 * i < have ? __ldg(h) : 0u) | (2 * i + 1 < have ? static_cast<unsigned>(__ldg(h + 1)) << 16 : 0u);
                        }
                    }
                }
            }
            return;
        }
        const unsigned shift = static_cast<unsigned>(reinterpret_cast<unsigned long long>(p)) & 15u;
        const uint4* base = reinterpret_cast<const uint4*>(reinterpret_cast<const unsigned char*>(p) - shift);
        const int bytes = left <= 0 ? 0 : static_cast<int>(shift) + min(left, kVals) * static_cast<int>(sizeof(T));
        if constexpr (!ALIGNED) {
#pragma unroll
            for (int j = 0; j <= kWords / 4; ++j) {
                uint4 v = make_uint4(0u, 0u, 0u, 0u);
                if (16 * j < bytes) v = __ldg(base + j);
                w[4 * j] = v.x, w[4 * j + 1] = v.y, w[4 * j + 2] = v.z, w[4 * j + 3] = v.w;
            }
        }
    }
    __device__ __forceinline__ void values(const T* p, int left, float t[kVals]) {
        const unsigned shift = ALIGNED ? 0u : static_cast<unsigned>(reinterpret_cast<unsigned long long>(p)) & 15u;
        if constexpr (!ALIGNED) {
            if (shift & 8u) {
#pragma unroll
                for (int i = 0; i < kWords + 2; ++i) w[i] = w[i + 2];
            }
            if (shift & 4u) {
#pragma unroll
                for (int i = 0; i < kWords + 1; ++i) w[i] = w[i + 1];
            }
            if (sizeof(T) == 2 && (shift & 2u)) {
#pragma unroll
                for (int i = 0; i < kWords; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], 16);
            }
        }
#pragma unroll
        for (int i = 0; i < kVals; ++i) {
            if constexpr (sizeof(T) == 4) {
                t[i] = __uint_as_float(w[i]);
            } else {
                const unsigned short h = static_cast<unsigned short>(w[i / 2] >> (i % 2 * 16));
                T e;
                *reinterpret_cast<unsigned short*>(&e) = h;
                t[i] = to_float<T>(e);
            }
        }
        if (!ALIGNED && left < kVals) {
#pragma unroll
            for (int i = 0; i < kVals; ++i) t[i] = i < left ? t[i] : 0.0f;
        }
    }
};

// r / d for the small numbers of one CTA: r < 2^15, or d > r / 2.  Its constants are made on the host: a division
// a thread cost a third of the time of small CTAs.
struct SmallDiv {
    unsigned d, m;
    explicit SmallDiv(unsigned d_) : d(d_), m(d_ > 1 && d_ < 32768u ? 0xffffffffu / d_ + 1u : 0u) {}
    __device__ __forceinline__ unsigned operator()(unsigned r) const { return d == 1u ? r : m ? __umulhi(r, m) : (r >= d ? 1u : 0u); }
};

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

// One CTA quantises `rows_per_cta` consecutive rows of the call, a thread kTake values at a time.  The next values
// are on their way in other warps: five CTAs an SM that load, then encode, need 23.6 us for 50176 x 1024 bf16
// values (nvfp4; 5.6 TB/s read and written), four that also load ahead in registers 28.5 us.
template <typename T, int FMT, bool ALIGNED>
__global__ void __launch_bounds__(kThreads, !ALIGNED ? 1 : sizeof(T) == 2 ? 5 : 4) write_kernel(MxMove p, int rows_per_cta, SmallDiv by_units, SmallDiv by_tokens) {
    const unsigned units = by_units.d;
    const unsigned total = static_cast<unsigned>(p.n * p.tokens);
    const unsigned row0 = blockIdx.x * static_cast<unsigned>(rows_per_cta);
    const unsigned rows = min(static_cast<unsigned>(rows_per_cta), total - row0);
    const unsigned sample0 = p.tokens == 1 ? row0 : row0 / p.tokens, token0 = row0 - sample0 * p.tokens;
    const float ts = mx_tensor_scale(p.q);
    __shared__ long long dest[kMaxRowsCta];  // cache row of every row of this CTA, or -1
    if (p.index) {
        // The CTA's samples (at most one more than its rows): their slots, their lengths, and whether a later sample of
        // the call names the same slot; by then the whole index is in shared memory, or `owner` knows.
        __shared__ long long slots[TLB_MX_SCAN_SAMPLES];
        __shared__ long long base[kMaxRowsCta + 1];  // first cache row of the sample, or -1
        __shared__ int length[kMaxRowsCta + 1];
        const unsigned last = (row0 + rows - 1) / p.tokens, samples = last - sample0 + 1;
        if (!p.use_owner && threadIdx.x < p.n) slots[threadIdx.x] = p.index[threadIdx.x];
        for (unsigned k = threadIdx.x; k < samples; k += kThreads) {
            const unsigned i = sample0 + k;
            const long long slot = p.index[i];
            const bool bad = slot < 0 || slot >= p.slots;
            int len = p.lengths ? p.lengths[i] : p.tokens;
            if (bad && p.status) atomicOr(p.status, TLB_DEV_BAD_INDEX);
            if (len < 0 || len > p.tokens) {
                len = len < 0 ? 0 : p.tokens;
                if (p.status) atomicOr(p.status, TLB_DEV_BAD_LENGTH);
            }
            base[k] = bad || (p.use_owner && p.owner[slot] != static_cast<int>(i)) ? -1 : slot * p.tokens;
            length[k] = len;
        }
        __syncthreads();
        if (!p.use_owner) {
            for (unsigned k = 0; k < samples; ++k)
                if (threadIdx.x > sample0 + k && threadIdx.x < p.n && slots[threadIdx.x] == slots[sample0 + k]) base[k] = -1;
            __syncthreads();
        }
        for (unsigned r = threadIdx.x; r < rows; r += kThreads) {
            const unsigned k = by_tokens(token0 + r), token = token0 + r - k * p.tokens;
            const bool there = base[k] >= 0;
            dest[r] = there && token < static_cast<unsigned>(length[k]) ? base[k] + token : -1;
            if (there && token == 0 && p.cache_lengths) p.cache_lengths[base[k] / p.tokens] = length[k];
        }
        __syncthreads();
    }
    const unsigned all = rows * units;
    constexpr int take = kTake<T>;
    // Power-of-two tensor scales, the usual ones, divide by an exact multiplication.
    const unsigned ts_bits = __float_as_uint(ts);
    const bool exact = (ts_bits & 0x007fffffu) == 0u && ts_bits >= 0x02000000u && ts_bits <= 0x7c000000u;
    const float inv = exact ? __uint_as_float(0x7f000000u - ts_bits) : 1.0f;
    const bool few_bits = sizeof(T) == 2 && exact;
    __shared__ float inverse[FMT == kNvfp4 ? 128 : 1];  // a division a block would cost as much as the rest of it
    if constexpr (FMT == kNvfp4) {
        if (threadIdx.x < 128) {
            const float s = e4m3_value(threadIdx.x);
            inverse[threadIdx.x] = few_bits ? __frcp_ru(s) : __frcp_rn(s);
        }
        __syncthreads();
    }
    struct Work {
        Raw<T, ALIGNED> raw;
        const T* x;
        long long to;
        int left, unit;
    };
    auto fetch = [&](Work& w, unsigned u) {  // false: the warp has no row that is written
        const bool in = u < all;
        const unsigned r = in ? by_units(u) : 0u;
        w.unit = static_cast<int>(in ? u - r * units : 0u);
        w.to = !in ? -1 : p.index ? dest[r] : static_cast<long long>(row0 + r);
        if (!__any_sync(0xffffffffu, w.to >= 0)) return false;
        const unsigned over = by_tokens(token0 + r), token = token0 + r - over * p.tokens;
        w.left = w.to >= 0 ? p.q.cols - w.unit * take : 0;
        w.x = static_cast<const T*>(p.in) + (sample0 + over) * p.sample_pitch + token * p.row_pitch + w.unit * take;
        w.raw.load(w.x, w.left);
        return true;
    };
    auto finish = [&](Work& w) {
        float t[take];
        w.raw.values(w.x, w.left, t);
        if (ts != 1.0f) {
            if (exact) {
#pragma unroll
                for (int i = 0; i < take; ++i) t[i] = __fmul_rn(t[i], inv);
            } else {
#pragma unroll
                for (int i = 0; i < take; ++i) t[i] = __fdiv_rn(t[i], ts);
            }
        }
        constexpr int words = (FMT == kMxfp8 ? take : take / 2) / 4;
        unsigned c[words];
        const unsigned bytes = encode<FMT, take>(t, c, few_bits, inverse);
        if (w.to < 0) return;
        unsigned char* cp = p.q.codes + w.to * mx_code_pitch(FMT, p.q.cols);
        if constexpr (words == 2) {
            reinterpret_cast<uint2*>(cp)[w.unit] = make_uint2(c[0], c[1]);
        } else {
#pragma unroll
            for (int i = 0; i < words / 4; ++i)
                reinterpret_cast<uint4*>(cp)[w.unit * (words / 4) + i] = make_uint4(c[4 * i], c[4 * i + 1], c[4 * i + 2], c[4 * i + 3]);
        }
        unsigned char* sp = p.q.scales + w.to * mx_scale_pitch(FMT, p.q.cols);  // blocks of zeros, pads too, have byte 0
        if constexpr (FMT == kNvfp4 && take == 32) reinterpret_cast<unsigned short*>(sp)[w.unit] = static_cast<unsigned short>(bytes);
        else if constexpr (FMT == kNvfp4 || take == 32) sp[w.unit] = static_cast<unsigned char>(bytes);
        else if ((w.unit & 1) == 0) sp[w.unit >> 1] = static_cast<unsigned char>(bytes);
    };
    for (unsigned u0 = threadIdx.x; u0 - threadIdx.x < all; u0 += kThreads) {  // whole warps stay together: lanes 2i, 2i + 1 may share a block
        Work w;
        if (fetch(w, u0)) finish(w);
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

__device__ __forceinline__ void store32(void* p, const unsigned v[8]) {  // 32 bytes, 32-byte aligned
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]),
                 "r"(v[6]), "r"(v[7])
                 : "memory");
}

// (What is wrong with a length is looked up again where a sample begins: status bits that came out of read_slot kept the
// loads of 512 x 256 x 1024 mxfp4 codes from being in flight together, 57 -> 69 us.)

// A CTA writes kReadUnits * kThreads units of 16 values, in the order of the output; a thread has the codes of all
// of its units on their way before it widens the first.  WHOLE: rows are multiples of 32 bytes, and every unit is
// stored as it is made.  Otherwise the values meet in shared memory, in the output's order, and leave it in 16-byte
// pieces; a word of padding after every 128 bytes there keeps the lanes' values, 16 apart, in different banks.
constexpr int kReadUnits = 4;
__device__ __forceinline__ unsigned spread(unsigned byte) { return byte + (byte >> 7) * 4; }
template <typename T, int FMT, bool WHOLE>
__global__ void __launch_bounds__(kThreads) read_kernel(MxMove p, SmallDiv by_units, SmallDiv by_tokens) {
    constexpr int per_thread = WHOLE ? kReadUnits : kReadUnits / 2;
    const unsigned units = by_units.d;
    const unsigned long long total = static_cast<unsigned long long>(p.n) * p.tokens * units, u0 = blockIdx.x * static_cast<unsigned long long>(per_thread * kThreads);
    const unsigned row0 = (u0 >> 32) == 0 ? static_cast<unsigned>(u0) / units : static_cast<unsigned>(u0 / units), off0 = static_cast<unsigned>(u0 - static_cast<unsigned long long>(row0) * units);
    const unsigned sample0 = p.tokens == 1 ? row0 : row0 / p.tokens, token0 = row0 - sample0 * p.tokens;
    const unsigned here = static_cast<unsigned>(min(static_cast<unsigned long long>(per_thread * kThreads), total - u0));
    const float ts = mx_tensor_scale(p.q);
    constexpr int words = FMT == kMxfp8 ? 4 : 2;
    unsigned c[per_thread][words], sb[per_thread], row[per_thread];
    int unit[per_thread];
#pragma unroll
    for (int j = 0; j < per_thread; ++j) {
        const unsigned u = j * kThreads + threadIdx.x, r = by_units(off0 + u);
        const bool in = u < here;
        unit[j] = static_cast<int>(off0 + u - r * units);
        row[j] = row0 + r;
        const unsigned over = by_tokens(token0 + r);
        const int token = static_cast<int>(token0 + r - over * p.tokens);
        sb[j] = 0u;
#pragma unroll
        for (int i = 0; i < words; ++i) c[j][i] = 0u;
        if (in) {
            const long long i = sample0 + over;
            int len;
            const long long s = read_slot(p, i, len);
            if (unit[j] == 0 && token == 0) {
                if (s < 0 && p.status) atomicOr(p.status, TLB_DEV_BAD_INDEX);
                if (s >= 0 && p.cache_lengths && p.status && p.cache_lengths[s] != len) atomicOr(p.status, TLB_DEV_BAD_LENGTH);
                if (p.lengths_out) p.lengths_out[i] = len;
            }
            if (token < len) {
                const long long from = s * p.tokens + token;
                const unsigned char* cp = p.q.codes + from * mx_code_pitch(FMT, p.q.cols);
                sb[j] = __ldg(p.q.scales + from * mx_scale_pitch(FMT, p.q.cols) + unit[j] / (mx_block(FMT) / kUnit));
                if constexpr (FMT == kMxfp8) {
                    const uint4 v = __ldg(reinterpret_cast<const uint4*>(cp) + unit[j]);
                    c[j][0] = v.x, c[j][1] = v.y, c[j][2] = v.z, c[j][3] = v.w;
                } else {
                    const uint2 v = __ldg(reinterpret_cast<const uint2*>(cp) + unit[j]);
                    c[j][0] = v.x, c[j][1] = v.y;
                }
            }
        }
    }
    extern __shared__ __align__(16) unsigned char staged[];
    const unsigned long long start = (static_cast<unsigned long long>(row0) * p.q.cols + off0 * kUnit) * sizeof(T);  // first output byte of this CTA
    const unsigned pad = static_cast<unsigned>(start) & 15u;  // the staged bytes lie like the output's, modulo 16
#pragma unroll
    for (int j = 0; j < per_thread; ++j) {
        if (j * kThreads + threadIdx.x >= here) continue;
        float v[kUnit];
        if constexpr (FMT == kMxfp8) {
#pragma unroll
            for (int i = 0; i < 4; ++i) e4m3_values(c[j][i], v + 4 * i);
        } else {
            e2m1_values(c[j][0], v);
            e2m1_values(c[j][1], v + 8);
        }
        const float s = scale_value<FMT>(sb[j]);
#pragma unroll
        for (int i = 0; i < kUnit; ++i) v[i] = __fmul_rn(v[i], s);
        if (ts != 1.0f) {
#pragma unroll
            for (int i = 0; i < kUnit; ++i) v[i] = __fmul_rn(v[i], ts);
        }
        __align__(16) T o[kUnit];
#pragma unroll
        for (int i = 0; i < kUnit; ++i) o[i] = from_float<T>(v[i]);
        if constexpr (WHOLE) {
            T* to = static_cast<T*>(p.out) + static_cast<long long>(row[j]) * p.q.cols + unit[j] * kUnit;
#pragma unroll
            for (int i = 0; i < kUnit * static_cast<int>(sizeof(T)) / 32; ++i)
                if (i == 0 || unit[j] * kUnit + i * static_cast<int>(32 / sizeof(T)) < p.q.cols)
                    store32(reinterpret_cast<unsigned char*>(to) + 32 * i, reinterpret_cast<const unsigned*>(o) + 8 * i);
        } else {
            const unsigned to = pad + ((row[j] - row0) * p.q.cols + unit[j] * kUnit - static_cast<int>(off0) * kUnit) * static_cast<unsigned>(sizeof(T));
            const int left = p.q.cols - unit[j] * kUnit;
#pragma unroll
            for (int i = 0; i < kUnit; ++i)
                if (i < left) *reinterpret_cast<T*>(staged + spread(to + i * static_cast<unsigned>(sizeof(T)))) = o[i];
        }
    }
    if constexpr (!WHOLE) {
        __syncthreads();
        // values of this CTA: whole rows but for the first one's beginning and the last one's end
        const unsigned end_off = off0 + here, end_row = by_units(end_off), rest = end_off - end_row * units;
        const unsigned count = end_row * p.q.cols + min(rest * kUnit, static_cast<unsigned>(p.q.cols)) - off0 * kUnit;
        const unsigned bytes = pad + count * static_cast<unsigned>(sizeof(T));
        unsigned char* out = static_cast<unsigned char*>(p.out) + (start - pad);
        for (unsigned b = threadIdx.x * 16; b < bytes; b += kThreads * 16) {
            if (b >= pad && b + 16 <= bytes) {
                const unsigned* w = reinterpret_cast<const unsigned*>(staged + spread(b));
                *reinterpret_cast<uint4*>(out + b) = make_uint4(w[0], w[1], w[2], w[3]);
            } else {
                for (unsigned e = max(b, pad); e < min(b + 16, bytes); e += sizeof(T)) *reinterpret_cast<T*>(out + e) = *reinterpret_cast<const T*>(staged + spread(e));
            }
        }
    }
}

// Rows as they are held: codes and scales into packed buffers, zeros behind a sample's length.  A row is `cw` words of
// 16 bytes of codes, then words of 4 bytes of scales; a thread has kReadUnits words on their way.
__global__ void __launch_bounds__(kThreads) read_codes_kernel(MxMove p, SmallDiv by_words, SmallDiv by_tokens, unsigned cw) {
    const unsigned words = by_words.d, sw = words - cw;
    const unsigned long long total = static_cast<unsigned long long>(p.n) * p.tokens * words, u0 = blockIdx.x * static_cast<unsigned long long>(kReadUnits * kThreads);
    const unsigned row0 = (u0 >> 32) == 0 ? static_cast<unsigned>(u0) / words : static_cast<unsigned>(u0 / words), off0 = static_cast<unsigned>(u0 - static_cast<unsigned long long>(row0) * words);
    const unsigned sample0 = p.tokens == 1 ? row0 : row0 / p.tokens, token0 = row0 - sample0 * p.tokens;
    const unsigned here = static_cast<unsigned>(min(static_cast<unsigned long long>(kReadUnits * kThreads), total - u0));
    uint4 v[kReadUnits];
    unsigned row[kReadUnits], word[kReadUnits];
#pragma unroll
    for (int j = 0; j < kReadUnits; ++j) {
        const unsigned u = j * kThreads + threadIdx.x, r = by_words(off0 + u), over = by_tokens(token0 + r);
        word[j] = off0 + u - r * words;
        row[j] = row0 + r;
        v[j] = make_uint4(0u, 0u, 0u, 0u);
        if (u >= here) continue;
        const long long i = sample0 + over;
        const int token = static_cast<int>(token0 + r - over * p.tokens);
        int len;
        const long long s = read_slot(p, i, len);
        if (word[j] == 0 && token == 0) {
            if (s < 0 && p.status) atomicOr(p.status, TLB_DEV_BAD_INDEX);
            if (s >= 0 && p.cache_lengths && p.status && p.cache_lengths[s] != len) atomicOr(p.status, TLB_DEV_BAD_LENGTH);
            if (p.lengths_out) p.lengths_out[i] = len;
        }
        if (token >= len) continue;
        const long long from = s * p.tokens + token;
        if (word[j] < cw) v[j] = __ldg(reinterpret_cast<const uint4*>(p.q.codes) + from * cw + word[j]);
        else v[j].x = __ldg(reinterpret_cast<const unsigned*>(p.q.scales) + from * sw + (word[j] - cw));
    }
#pragma unroll
    for (int j = 0; j < kReadUnits; ++j) {
        if (j * kThreads + threadIdx.x >= here) continue;
        if (word[j] < cw) reinterpret_cast<uint4*>(p.out_codes)[static_cast<long long>(row[j]) * cw + word[j]] = v[j];
        else reinterpret_cast<unsigned*>(p.out_scales)[static_cast<long long>(row[j]) * sw + (word[j] - cw)] = v[j].x;
    }
}

template <typename T, bool ALIGNED>
void write_by_format(const MxMove& p, int grid, int rows_per_cta, cudaStream_t st) {
    const SmallDiv by_units(mx_padded(p.q.cols) / kTake<T>), by_tokens(p.tokens);
    if (p.q.format == kNvfp4) write_kernel<T, kNvfp4, ALIGNED><<<grid, kThreads, 0, st>>>(p, rows_per_cta, by_units, by_tokens);
    else if (p.q.format == kMxfp4) write_kernel<T, kMxfp4, ALIGNED><<<grid, kThreads, 0, st>>>(p, rows_per_cta, by_units, by_tokens);
    else write_kernel<T, kMxfp8, ALIGNED><<<grid, kThreads, 0, st>>>(p, rows_per_cta, by_units, by_tokens);
}
template <typename T>
void write_by_alignment(const MxMove& p, int grid, int rows_per_cta, cudaStream_t st) {
    const auto off = [](long long elements) { return elements * static_cast<long long>(sizeof(T)) % 32 != 0; };
    const bool aligned = (reinterpret_cast<unsigned long long>(p.in) & 31u) == 0 && !off(p.row_pitch) && !off(p.sample_pitch);
    if (aligned) write_by_format<T, true>(p, grid, rows_per_cta, st);
    else write_by_format<T, false>(p, grid, rows_per_cta, st);
}
template <typename T, bool WHOLE>
void read_whole_or_not(const MxMove& p, unsigned grid, cudaStream_t st) {
    const int bytes = kReadUnits / 2 * kThreads * kUnit * static_cast<int>(sizeof(T)) + 32, smem = WHOLE ? 0 : bytes + bytes / 32 + 4;
    const SmallDiv by_units((p.q.cols + kUnit - 1) / kUnit), by_tokens(p.tokens);
    if (p.q.format == kNvfp4) read_kernel<T, kNvfp4, WHOLE><<<grid, kThreads, smem, st>>>(p, by_units, by_tokens);
    else if (p.q.format == kMxfp4) read_kernel<T, kMxfp4, WHOLE><<<grid, kThreads, smem, st>>>(p, by_units, by_tokens);
    else read_kernel<T, kMxfp8, WHOLE><<<grid, kThreads, smem, st>>>(p, by_units, by_tokens);
}
template <typename T>
int read_by_format(const MxMove& p, cudaStream_t st) {
    const bool whole = p.q.cols * sizeof(T) % 32 == 0 && (reinterpret_cast<unsigned long long>(p.out) & 31u) == 0;
    const long long units = p.n * p.tokens * ((p.q.cols + kUnit - 1) / kUnit), per_cta = (whole ? kReadUnits : kReadUnits / 2) * kThreads;
    const long long grid = (units + per_cta - 1) / per_cta;
    if (grid > 0x7fffffffll) return static_cast<int>(cudaErrorInvalidValue);
    if (whole) read_whole_or_not<T, true>(p, static_cast<unsigned>(grid), st);
    else read_whole_or_not<T, false>(p, static_cast<unsigned>(grid), st);
    return 0;
}

}  // namespace

void mx_count_launch() { g_mx_launches.fetch_add(1, std::memory_order_relaxed); }
unsigned long long mx_launch_count() { return g_mx_launches.load(std::memory_order_relaxed); }

int launch_mx_write(const MxMove& p0, void* stream) {
    MxMove p = p0;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int units = mx_padded(p.q.cols) / (p.dtype == kF32 ? kTake<float> : kTake<__half>);
    // Rounds of units a thread: more of them share a CTA's start and its look at the index (12544 CTAs of one round
    // took twice the time of 1568 of eight); fewer where they would leave SMs without work.
    const long long rounds = p.n * p.tokens * units / (static_cast<long long>(kThreads) * kWriteCtas);
    const int per_cta = static_cast<int>(rounds < 1 ? 1 : rounds > kMaxRounds ? kMaxRounds : rounds) * kThreads;
    const int rows_per_cta = units >= per_cta ? 1 : per_cta / units;
    const long long grid = (p.n * p.tokens + rows_per_cta - 1) / rows_per_cta;
    if (grid > 0x7fffffffll) return static_cast<int>(cudaErrorInvalidValue);
    // Duplicates: a CTA reads the whole index per sample while that is short, else the claims are made first.
    p.use_owner = p.index && p.n > TLB_MX_SCAN_SAMPLES;
    if (p.use_owner) {
        const int ctas = static_cast<int>((p.n + kThreads - 1) / kThreads);
        claim_kernel<<<ctas, kThreads, 0, st>>>(p.index, p.n, p.slots, p.owner);
        mx_count_launch();
    }
    if (p.dtype == kF32) write_by_alignment<float>(p, static_cast<int>(grid), rows_per_cta, st);
    else if (p.dtype == kBf16) write_by_alignment<__nv_bfloat16>(p, static_cast<int>(grid), rows_per_cta, st);
    else write_by_alignment<__half>(p, static_cast<int>(grid), rows_per_cta, st);
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
    if (int e = p.dtype == kF32 ? read_by_format<float>(p, st) : p.dtype == kBf16 ? read_by_format<__nv_bfloat16>(p, st) : read_by_format<__half>(p, st)) return e;
    mx_count_launch();
    return static_cast<int>(cudaGetLastError());
}

int launch_mx_read_codes(const MxMove& p, void* stream) {
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int cw = mx_code_pitch(p.q.format, p.q.cols) / 16, words = cw + mx_scale_pitch(p.q.format, p.q.cols) / 4;
    const long long ctas = (p.n * p.tokens * words + kReadUnits * kThreads - 1) / (kReadUnits * kThreads);
    if (ctas > 0x7fffffffll) return static_cast<int>(cudaErrorInvalidValue);
    read_codes_kernel<<<static_cast<unsigned>(ctas), kThreads, 0, st>>>(p, SmallDiv(words), SmallDiv(p.tokens), cw);
    mx_count_launch();
    return static_cast<int>(cudaGetLastError());
}

}  // namespace tlb
