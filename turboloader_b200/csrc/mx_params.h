// Launch parameters of the microscaled operators (mx_rows.cu, mx_matmul.cu, mx_grad.cu), shared with
// their host C ABI (mx_capi.cu).
#pragma once
#include <cuda_runtime.h>

namespace tlb {

enum MxFormat { kNvfp4 = 0, kMxfp4 = 1, kMxfp8 = 2 };
enum MxDtype { kF32 = 0, kBf16 = 1, kF16 = 2 };

// Rows are padded to 128 values, with zero codes and zero scale bytes, so that every row of codes
// starts on a 64-byte boundary and every row of scales on a 4-byte one.
constexpr int kMxPad = 128;
__host__ __device__ inline int mx_padded(int cols) { return (cols + kMxPad - 1) / kMxPad * kMxPad; }
__host__ __device__ inline int mx_block(int format) { return format == kNvfp4 ? 16 : 32; }
__host__ __device__ inline int mx_code_pitch(int format, int cols) { return format == kMxfp8 ? mx_padded(cols) : mx_padded(cols) / 2; }
__host__ __device__ inline int mx_scale_pitch(int format, int cols) { return mx_padded(cols) / mx_block(format); }

struct MxRows {
    unsigned char* codes;
    unsigned char* scales;
    long long rows;
    int cols, format;
    float scale;             // tensor scale = scale * (scale_dev ? *scale_dev : 1)
    const float* scale_dev;
};

// Rows of `n` samples of `tokens` rows each, quantised into or read from the slots of a cache.
struct MxMove {
    MxRows q;                // the cache (or a plain matrix: tokens = 1, index = nullptr)
    long long slots;         // samples the cache holds
    int tokens;              // rows per sample
    long long n;             // samples of this call
    const long long* index;  // slot of every sample, nullptr: slot i = i
    int* cache_lengths;      // rows in use per slot, or nullptr: all
    const int* lengths;      // write: rows of every sample, or nullptr: all
    int* lengths_out;        // read: rows in use of every sample, or nullptr
    int* owner;              // write: [slots] words, -1 between calls (see mx_rows.cu)
    int use_owner;           // write: 1 = duplicates were resolved in `owner`, 0 = look for them in `index`
    unsigned* status;
    const void* in;          // write: values, row pitch and sample pitch in elements
    long long row_pitch, sample_pitch;
    void* out;               // read: values, packed
    unsigned char* out_codes;   // read of codes: both packed
    unsigned char* out_scales;
    int dtype;
};

int launch_mx_write(const MxMove& p, void* stream);       // returns a cudaError_t value
int launch_mx_read(const MxMove& p, void* stream);
int launch_mx_read_codes(const MxMove& p, void* stream);

struct MxProduct {
    MxRows a, b;             // (m, k) and (n, k)
    void* out;               // (m, n) packed
    int out_dtype;
    void* workspace;
};
bool mx_few(const MxProduct& p);  // whether launch_mx_few takes the product
int launch_mx_few(const MxProduct& p, void* stream);
int mx_gave_up(unsigned* count);  // products and gradients on this device that gave up a bounded wait
size_t mx_matmul_workspace(const MxProduct& p);
int launch_mx_matmul(const MxProduct& p, void* stream);

// Gradients of a * b^T, g (m, n): of a, out (m, cols) = g * values(b), and of b, out (n, cols) = g^T * values(a).
// grad_a or grad_b nullptr: not wanted, and the other operand not read.
struct MxGrad {
    const void* g;           // (m, n) packed
    int g_dtype;
    long long m;
    int n;
    MxRows a, b;
    void *grad_a, *grad_b;   // packed
    int grad_a_dtype, grad_b_dtype;
    void* workspace;
};
// A 2-D tensor map (cuTensorMapEncodeTiled); a cudaError_t value.
int mx_encode_map(void* map, int element_bytes, const void* base, unsigned long long inner, unsigned long long rows, unsigned long long pitch,
                  unsigned box_inner, unsigned box_rows, int swizzle);
// Rows of a tensor-map copy of the matrix whose result rows a CTA takes, at most `most`.  A matrix with fewer is
// copied in whole groups of 8 (what lies behind them in shared memory reaches only result rows that are not
// written): copies of 128 rows of a matrix with less than 32 kept the pairs waiting (13 x 4096 x 8192 nvfp4:
// 20.0 us, 13.9 with copies of 16).
inline int mx_box_rows(long long rows, int most) { return rows >= most ? most : static_cast<int>((rows + 7) / 8 * 8); }
int mx_grad_gave_up(unsigned* count);
size_t mx_grad_workspace(const MxGrad& p);
int launch_mx_grad(const MxGrad& p, void* stream);

unsigned long long mx_launch_count();
void mx_count_launch();

}  // namespace tlb
