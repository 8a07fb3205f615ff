// Quantisation to e4m3 with one f32 scale for each block of 1 x 128 or 128 x 128 values.
//
//   a = max(max finite |x|, 2^-100),   scale = a / 448,   q = e4m3(x * (448 / a))
//
// Bound: HBM.  Each value is read once, kept in registers across the block's maximum, and written as a byte.
// Eight lanes own one row's 128 columns: lane l takes columns 64 j + 8 l .. + 7 (j = 0, 1), so a warp's load of
// 16-bit values is four full 128-byte lines and the block maximum is three shuffles.  What else bounded it was the number of
// instructions a value: with a test for infinities on each (now on a block's maximum) 16-bit rows ran at 4.1 TB/s.
// Measured: 32760 x 5120 bf16 rows 84 us (6.0 TB/s, 0.91 of the copy rate), 13824 x 5120 f32 in 128 x 128 blocks 53 us
// (6.7 TB/s), the same from bf16 or f16 51 us (4.2 TB/s, floor 32: a CTA loads, reduces and stores in turn, three to an SM, and
// values count there, not bytes).
#include "edb200_internal.h"
#include "edb200_fp8.cuh"

namespace edb {
namespace f8q {

constexpr int THREADS = 256;

// The 16 values lane l of a group holds of one row's block: columns c0 + 64 j + 8 l + e.  Columns from k on and rows that
// are not there read zero.
template <typename T, bool VEC>
__device__ __forceinline__ void load16(const T* row, int c0, int l, int k, bool live, float (&v)[16]) {
    if (VEC && live && c0 + 128 <= k) {
        load8(row + c0 + 8 * l, reinterpret_cast<float(&)[8]>(v[0]));
        load8(row + c0 + 64 + 8 * l, reinterpret_cast<float(&)[8]>(v[8]));
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int c = c0 + 64 * (i >> 3) + 8 * l + (i & 7);
            v[i] = live && c < k ? widen<T>(row[c]) : 0.0f;
        }
    }
}

template <bool VEC>
__device__ __forceinline__ void store16(uint8_t* row, int c0, int l, int k, const float (&v)[16], float inv) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int c = c0 + 64 * j + 8 * l;
        float w[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = __fmul_rn(v[8 * j + e], inv);
        const uint32_t lo = f8_pack4(w[0], w[1], w[2], w[3]), hi = f8_pack4(w[4], w[5], w[6], w[7]);
        if (VEC && c + 8 <= k) {
            *reinterpret_cast<uint2*>(row + c) = make_uint2(lo, hi);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if (c + e < k) row[c + e] = static_cast<uint8_t>((e < 4 ? lo : hi) >> (8 * (e & 3)));
            }
        }
    }
}

__device__ __forceinline__ float peak16(const float (&v)[16]) {
    float a = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) a = f8_peak(a, v[i]);
    return a;
}
__device__ __forceinline__ void no_infinities16(float (&v)[16]) {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = f8_no_infinity(v[i]);
}
__device__ __forceinline__ float group_max(float a) {
#pragma unroll
    for (int m = 4; m > 0; m >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, m));
    return a;
}

// 1 x 128: a group of eight lanes per block.  SMALL: the block's row by the product with 2^32 / kb rounded up, exact while
// blocks times kb stay below 2^32; else by division in 64 bits, which costs nothing beside the memory (372000 x 13824 bf16
// 2.58 ms, 365000 rows by the product 2.45).  VEC: whether rows are aligned is another matter than how many there are.
template <typename T, bool VEC, bool SMALL>
__global__ void __launch_bounds__(THREADS)
quantize_rows_kernel(const T* __restrict__ x, int64_t ldx, int64_t rows, int k, int kb, uint32_t inv_kb, uint8_t* __restrict__ q,
                     int64_t ldq, float* __restrict__ scale, int64_t ld_scale) {
    const int l = threadIdx.x & 7;
    int64_t row;
    int b;
    if (SMALL) {
        const uint32_t g = blockIdx.x * (THREADS / 8) + (threadIdx.x >> 3);
        const uint32_t r = kb == 1 ? g : __umulhi(g, inv_kb);
        row = r;
        b = static_cast<int>(g - r * static_cast<uint32_t>(kb));
    } else {
        const int64_t g = static_cast<int64_t>(blockIdx.x) * (THREADS / 8) + (threadIdx.x >> 3);
        row = g / kb;
        b = static_cast<int>(g - row * kb);
    }
    const bool live = row < rows;
    float v[16];
    load16<T, VEC>(x + row * ldx, b * 128, l, k, live, v);
    float a = group_max(peak16(v));
    if (__any_sync(0xffffffffu, f8_has_infinity(a))) {   // some block of the warp holds an infinity
        no_infinities16(v);
        a = group_max(peak16(v));
    }
    // f8_scale()'s two divisions as one: the group's first lane makes the scale, the others its inverse
    a = fmaxf(a, kF8Floor);
    const float quotient = __fdiv_rn(l == 0 ? a : kF8Max, l == 0 ? kF8Max : a);
    const float inv = __shfl_sync(0xffffffffu, quotient, (threadIdx.x & 24) | 1);
    if (!live) return;
    store16<VEC>(q + row * ldq, b * 128, l, k, v, inv);
    if (l == 0) scale[row * ld_scale + b] = quotient;
}

template <int N>
__device__ __forceinline__ float cta_max(float a, float* sh) {
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, m));
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = a;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) a = fmaxf(a, sh[i]);
    return a;
}

// 128 x 128: a CTA per block, 32 rows at a time, all 64 values of a thread in registers.
template <typename T, bool VEC>
__global__ void __launch_bounds__(THREADS, 3)
quantize_tiles_kernel(const T* __restrict__ x, int64_t ldx, int64_t rows, int k, uint8_t* __restrict__ q, int64_t ldq,
                      float* __restrict__ scale, int64_t ld_scale) {
    __shared__ float sh[2][THREADS / 32];
    const int l = threadIdx.x & 7;
    const int64_t row0 = static_cast<int64_t>(blockIdx.y) * 128 + (threadIdx.x >> 3);
    const int c0 = blockIdx.x * 128;
    float v[4][16];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t row = row0 + 32 * i;
        load16<T, VEC>(x + row * ldx, c0, l, k, row < rows, v[i]);
    }
    float a = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) a = fmaxf(a, peak16(v[i]));
    a = cta_max<THREADS / 32>(a, sh[0]);
    if (f8_has_infinity(a)) {   // the same in every thread
        a = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            no_infinities16(v[i]);
            a = fmaxf(a, peak16(v[i]));
        }
        a = cta_max<THREADS / 32>(a, sh[1]);
    }
    float s, inv;
    f8_scale(a, s, inv);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t row = row0 + 32 * i;
        if (row < rows) store16<VEC>(q + row * ldq, c0, l, k, v[i], inv);
    }
    if (threadIdx.x == 0) scale[static_cast<int64_t>(blockIdx.y) * ld_scale + blockIdx.x] = s;
}

template <typename T>
static edb200_status_t launch(const T* x, int64_t ldx, int64_t rows, int64_t k, int block_rows, uint8_t* q, int64_t ldq,
                              float* scale, int64_t ld_scale, cudaStream_t s) {
    const int64_t kb = (k + 127) / 128;
    // wide accesses: 16-byte loads of 8 values (two for f32), 8-byte stores
    const bool vec = (reinterpret_cast<uintptr_t>(x) & 15u) == 0 && (rows == 1 || (ldx * sizeof(T)) % 16 == 0) &&
                     (reinterpret_cast<uintptr_t>(q) & 7u) == 0 && (rows == 1 || ldq % 8 == 0);
    const int ki = static_cast<int>(k);
    if (block_rows == 1) {
        const int64_t groups = rows * kb;
        const int64_t ctas = (groups + THREADS / 8 - 1) / (THREADS / 8);
        if (ctas > 0x7fffffff) return fail(EDB200_ERR_UNSUPPORTED, "quantize_fp8: more than 2^36 blocks");
        const unsigned grid = static_cast<unsigned>(ctas);
        const int kbi = static_cast<int>(kb);
        const uint32_t inv_kb = static_cast<uint32_t>((0x100000000ull + kb - 1) / kb);
        const bool small = static_cast<double>(ctas) * (THREADS / 8) * static_cast<double>(kb) < 4294967296.0;
        auto kernel = small ? (vec ? quantize_rows_kernel<T, true, true> : quantize_rows_kernel<T, false, true>)
                            : (vec ? quantize_rows_kernel<T, true, false> : quantize_rows_kernel<T, false, false>);
        kernel<<<grid, THREADS, 0, s>>>(x, ldx, rows, ki, kbi, inv_kb, q, ldq, scale, ld_scale);
    } else {
        const int64_t rb = (rows + 127) / 128;
        if (rb > 65535) return fail(EDB200_ERR_UNSUPPORTED, "quantize_fp8: more than 65535 x 128 rows of 128 x 128 blocks");
        const dim3 grid(static_cast<unsigned>(kb), static_cast<unsigned>(rb));
        if (vec) {
            quantize_tiles_kernel<T, true><<<grid, THREADS, 0, s>>>(x, ldx, rows, ki, q, ldq, scale, ld_scale);
        } else {
            quantize_tiles_kernel<T, false><<<grid, THREADS, 0, s>>>(x, ldx, rows, ki, q, ldq, scale, ld_scale);
        }
    }
    count_launch();
    return check_cuda(cudaGetLastError(), "quantize_fp8 launch");
}

}  // namespace f8q
}  // namespace edb

extern "C" edb200_status_t edb200_quantize_fp8(const void* x, int x_dtype, int64_t ldx, int64_t rows, int64_t k, int block_rows,
                                               void* q, int64_t ldq, float* scale, int64_t ld_scale, void* stream) {
    using namespace edb;
    if (x_dtype != EDB200_TYPE_F32 && x_dtype != EDB200_TYPE_F16 && x_dtype != EDB200_TYPE_BF16) {
        return fail(EDB200_ERR_INVALID, "quantize_fp8: x_dtype must be f32, f16 or bf16");
    }
    if (block_rows != 1 && block_rows != 128) return fail(EDB200_ERR_INVALID, "quantize_fp8: block_rows must be 1 or 128");
    if (rows < 0 || k < 1 || k > 0x7fffff00ll) return fail(EDB200_ERR_INVALID, "quantize_fp8: rows >= 0 and 1 <= k < 2^31 - 256");
    if (rows == 0) return EDB200_OK;
    if (x == nullptr || q == nullptr || scale == nullptr) return fail(EDB200_ERR_INVALID, "quantize_fp8: null argument");
    if ((rows > 1 && (ldx < k || ldq < k)) || (rows > block_rows && ld_scale < (k + 127) / 128)) {
        return fail(EDB200_ERR_INVALID, "quantize_fp8: ldx and ldq must hold k columns, ld_scale ceil(k / 128)");
    }
    const uintptr_t esz = x_dtype == EDB200_TYPE_F32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(x) % esz || (reinterpret_cast<uintptr_t>(scale) & 3u)) {
        return fail(EDB200_ERR_INVALID, "quantize_fp8: x and scale must be aligned to their elements");
    }
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    uint8_t* qb = static_cast<uint8_t*>(q);
    ProfScope prof(s, PROF_ELEMENTWISE, 0.0, (double)rows * (double)k * (double)(esz + 1));
    if (x_dtype == EDB200_TYPE_F32) return f8q::launch(static_cast<const float*>(x), ldx, rows, k, block_rows, qb, ldq, scale, ld_scale, s);
    if (x_dtype == EDB200_TYPE_F16) return f8q::launch(static_cast<const __half*>(x), ldx, rows, k, block_rows, qb, ldq, scale, ld_scale, s);
    return f8q::launch(static_cast<const __nv_bfloat16*>(x), ldx, rows, k, block_rows, qb, ldq, scale, ld_scale, s);
}
