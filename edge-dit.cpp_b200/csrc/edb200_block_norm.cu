// The norms around a block fused with its gate and the residual stream:
//
//   t = post(x);   y = residual_scale * residual + gate * t;   z = pre(y) * (1 + scale) + shift
//
// with post, pre = none, LayerNorm (v - mean) * rstd or RMSNorm v * rstd, times weight plus bias, and z cast or
// quantised to e4m3 with a scale for each 128 columns.
//
// Bound: HBM.  A row's x and residual are read once, live in registers through both norms, and y and z are written
// once; the statistics are f32 sums over registers, the variance taken around the mean (two sums, no cancellation).
// A row belongs to one warp (h <= 1024, eight rows a CTA, sums by shuffles alone) or to one CTA of just as many
// threads as its chunks of eight columns need; a thread's chunk i is columns 8 (tid + i * threads) .. + 7, so 128
// columns are 16 neighbouring lanes and a quantisation block's maximum is four shuffles.
#include "edb200_internal.h"
#include "edb200_fp8.cuh"

namespace edb {
namespace bn {

struct Params {
    edb200_block_norm_t p;
};

template <bool WARP>
__device__ __forceinline__ float row_sum(float v, float* sh) {
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
    if (WARP) return v;
    const int warps = blockDim.x >> 5;
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    v = (threadIdx.x & 31) < warps ? sh[threadIdx.x & 31] : 0.0f;
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
    return v;
}

// Chunk of eight columns c .. c + 7 of a row of h; columns beyond h read `fill`.
template <bool VEC, typename T>
__device__ __forceinline__ void load_chunk(const T* row, int c, int h, float fill, float (&v)[8]) {
    if (VEC && c + 8 <= h) {
        load8(row + c, v);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = c + e < h ? widen<T>(row[c + e]) : fill;
    }
}
template <bool VEC, typename T>
__device__ __forceinline__ void store_chunk(T* row, int c, int h, const float (&v)[8]) {
    if (VEC && c + 8 <= h) {
        store8(row + c, v);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (c + e < h) row[c + e] = narrow<T>(v[e]);
        }
    }
}

// v <- norm(v) * weight + bias over the row; sh holds two reductions' worth of warp sums.
template <int CH, bool WARP, bool VEC>
__device__ __forceinline__ void norm_row(float (&v)[CH][8], int kind, const float* weight, const float* bias, float eps, int h,
                                         int tid, int step, float* sh) {
    const float n = static_cast<float>(h);
    float mean = 0.0f;
    if (kind == EDB200_NORM_LAYER) {
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < CH; ++i) {
#pragma unroll
            for (int e = 0; e < 8; ++e) s += v[i][e];   // columns beyond h are zero
        }
        mean = row_sum<WARP>(s, sh) / n;
    }
    float q = 0.0f;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        const int c = 8 * (tid + i * step);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            v[i][e] = c + e < h ? v[i][e] - mean : 0.0f;
            q = fmaf(v[i][e], v[i][e], q);
        }
    }
    const float rstd = 1.0f / sqrtf(row_sum<WARP>(q, sh + 32) / n + eps);
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        const int c = 8 * (tid + i * step);
        if (c >= h) continue;
        float w[8];
        if (weight != nullptr) {
            load_chunk<VEC>(weight, c, h, 0.0f, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[i][e] = v[i][e] * rstd * w[e];
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[i][e] *= rstd;
        }
        if (bias != nullptr) {
            load_chunk<VEC>(bias, c, h, 0.0f, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[i][e] += w[e];
        }
    }
}

template <typename TX, typename TS, int CH, bool WARP, bool VEC>
__global__ void __launch_bounds__(WARP ? 256 : 1024)
block_norm_kernel(const __grid_constant__ Params P) {
    __shared__ float sh[128];
    const edb200_block_norm_t& p = P.p;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y;
    if (WARP && row >= p.rows) return;   // a whole warp; nothing below synchronises the CTA then
    const int h = static_cast<int>(p.h);
    const int tid = threadIdx.x, step = blockDim.x;
    const int64_t mod = (p.rows_per_mod > 0 ? row / p.rows_per_mod : 0) * p.ld_mod;

    float t[CH][8], y[CH][8];
    const bool has_x = p.x != nullptr;
    if (has_x) {
        const TX* xr = static_cast<const TX*>(p.x) + row * p.ldx;
#pragma unroll
        for (int i = 0; i < CH; ++i) load_chunk<VEC>(xr, 8 * (tid + i * step), h, 0.0f, t[i]);
    }
    const TS* rr = static_cast<const TS*>(p.residual) + row * p.ld_res;
#pragma unroll
    for (int i = 0; i < CH; ++i) load_chunk<VEC>(rr, 8 * (tid + i * step), h, 0.0f, y[i]);

    if (has_x && p.post_norm != EDB200_NORM_NONE) {
        norm_row<CH, WARP, VEC>(t, p.post_norm, p.post_weight, p.post_bias, p.post_eps, h, tid, step, sh);
    }
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        const int c = 8 * (tid + i * step);
        if (c >= h) continue;
#pragma unroll
        for (int e = 0; e < 8; ++e) y[i][e] *= p.residual_scale;
        if (has_x) {
            if (p.gate != nullptr) {
                float g[8];
                load_chunk<VEC>(p.gate + mod, c, h, 0.0f, g);
#pragma unroll
                for (int e = 0; e < 8; ++e) y[i][e] = fmaf(g[e], t[i][e], y[i][e]);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) y[i][e] += t[i][e];
            }
        }
        if (p.y != nullptr) store_chunk<VEC>(static_cast<TS*>(p.y) + row * p.ldy, c, h, y[i]);
    }
    if (p.z == nullptr) return;   // uniform
    if (p.pre_norm != EDB200_NORM_NONE) {
        norm_row<CH, WARP, VEC>(y, p.pre_norm, p.pre_weight, p.pre_bias, p.pre_eps, h, tid, step, sh + 64);
    }
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        const int c = 8 * (tid + i * step);
        if (c < h) {
            float m[8];
            if (p.scale != nullptr) {
                load_chunk<VEC>(p.scale + mod, c, h, 0.0f, m);
#pragma unroll
                for (int e = 0; e < 8; ++e) y[i][e] = fmaf(y[i][e], m[e], y[i][e]);
            }
            if (p.shift != nullptr) {
                load_chunk<VEC>(p.shift + mod, c, h, 0.0f, m);
#pragma unroll
                for (int e = 0; e < 8; ++e) y[i][e] += m[e];
            }
        }
        if (p.z_dtype == EDB200_TYPE_F8_E4M3) {
            float a = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) a = fmaxf(a, c + e < h ? f8_magnitude(y[i][e]) : 0.0f);
#pragma unroll
            for (int k = 8; k > 0; k >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, k));
            if (c >= h) continue;
            float s, inv;
            f8_scale(a, s, inv);
            float w[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = f8_scaled(y[i][e], inv);
            const uint32_t lo = f8_pack4(w[0], w[1], w[2], w[3]), hi = f8_pack4(w[4], w[5], w[6], w[7]);
            uint8_t* zr = static_cast<uint8_t*>(p.z) + row * p.ldz + c;
            if (VEC && c + 8 <= h) {
                *reinterpret_cast<uint2*>(zr) = make_uint2(lo, hi);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    if (c + e < h) zr[e] = static_cast<uint8_t>((e < 4 ? lo : hi) >> (8 * (e & 3)));
                }
            }
            if ((tid & 15) == 0) p.z_scale[row * p.ld_z_scale + (c >> 7)] = s;
        } else if (c < h) {
            if (p.z_dtype == EDB200_TYPE_F32) {
                store_chunk<VEC>(static_cast<float*>(p.z) + row * p.ldz, c, h, y[i]);
            } else if (p.z_dtype == EDB200_TYPE_F16) {
                store_chunk<VEC>(static_cast<__half*>(p.z) + row * p.ldz, c, h, y[i]);
            } else {
                store_chunk<VEC>(static_cast<__nv_bfloat16*>(p.z) + row * p.ldz, c, h, y[i]);
            }
        }
    }
}

template <typename TX, typename TS, bool VEC>
static void launch_sized(const Params& P, cudaStream_t s) {
    const int64_t h = P.p.h, rows = P.p.rows;
    const int chunks = static_cast<int>((h + 7) / 8);
    if (h <= 1024) {
        const dim3 block(32, 8);
        const unsigned grid = static_cast<unsigned>((rows + 7) / 8);
        if (chunks <= 32) {
            block_norm_kernel<TX, TS, 1, true, VEC><<<grid, block, 0, s>>>(P);
        } else if (chunks <= 64) {
            block_norm_kernel<TX, TS, 2, true, VEC><<<grid, block, 0, s>>>(P);
        } else {
            block_norm_kernel<TX, TS, 4, true, VEC><<<grid, block, 0, s>>>(P);
        }
    } else {
        const unsigned grid = static_cast<unsigned>(rows);
        const unsigned threads = static_cast<unsigned>(((chunks + 1) / 2 + 31) / 32 * 32);   // <= 1024 for h <= 16384
        block_norm_kernel<TX, TS, 2, false, VEC><<<grid, threads, 0, s>>>(P);
    }
}

template <typename TX, typename TS>
static void launch_vec(const Params& P, bool vec, cudaStream_t s) {
    if (vec) {
        launch_sized<TX, TS, true>(P, s);
    } else {
        launch_sized<TX, TS, false>(P, s);
    }
}
template <typename TS>
static void launch_x(const Params& P, bool vec, cudaStream_t s) {
    if (P.p.x == nullptr || P.p.x_dtype == EDB200_TYPE_F32) {
        launch_vec<float, TS>(P, vec, s);
    } else if (P.p.x_dtype == EDB200_TYPE_F16) {
        launch_vec<__half, TS>(P, vec, s);
    } else {
        launch_vec<__nv_bfloat16, TS>(P, vec, s);
    }
}

static int esize(int dt) { return dt == EDB200_TYPE_F32 ? 4 : dt == EDB200_TYPE_F8_E4M3 ? 1 : 2; }
static bool float_type(int dt) { return dt == EDB200_TYPE_F32 || dt == EDB200_TYPE_F16 || dt == EDB200_TYPE_BF16; }

}  // namespace bn
}  // namespace edb

extern "C" edb200_status_t edb200_block_norm(const edb200_block_norm_t* pp, void* stream) {
    using namespace edb;
    if (pp == nullptr) return fail(EDB200_ERR_INVALID, "block_norm: null argument");
    const edb200_block_norm_t& p = *pp;
    if (p.rows < 0 || p.h < 1) return fail(EDB200_ERR_INVALID, "block_norm: rows >= 0 and h >= 1");
    if (p.h > 16384) return fail(EDB200_ERR_UNSUPPORTED, "block_norm: h is at most 16384");
    if (p.rows > 0x7fffffffll) return fail(EDB200_ERR_UNSUPPORTED, "block_norm: more than 2^31 - 1 rows");
    auto norm_ok = [](int k) { return k == EDB200_NORM_NONE || k == EDB200_NORM_LAYER || k == EDB200_NORM_RMS; };
    if (!norm_ok(p.post_norm) || !norm_ok(p.pre_norm)) return fail(EDB200_ERR_INVALID, "block_norm: post_norm and pre_norm must be EDB200_NORM_*");
    if (!bn::float_type(p.stream_dtype) || (p.x != nullptr && !bn::float_type(p.x_dtype)) ||
        (p.z != nullptr && !bn::float_type(p.z_dtype) && p.z_dtype != EDB200_TYPE_F8_E4M3)) {
        return fail(EDB200_ERR_INVALID, "block_norm: types are f32, f16 or bf16, and e4m3 for z alone");
    }
    if (p.rows == 0) return EDB200_OK;
    if (p.residual == nullptr || (p.y == nullptr && p.z == nullptr)) {
        return fail(EDB200_ERR_INVALID, "block_norm: residual and one of y and z must be set");
    }
    if (p.rows_per_mod < 0) return fail(EDB200_ERR_INVALID, "block_norm: rows_per_mod must not be negative");
    const bool any_mod = p.gate != nullptr || p.scale != nullptr || p.shift != nullptr;
    const int64_t n_mod = p.rows_per_mod > 0 ? (p.rows + p.rows_per_mod - 1) / p.rows_per_mod : 1;
    const bool many = p.rows > 1;   // a single row's strides are not used
    if ((many && ((p.x != nullptr && p.ldx < p.h) || p.ld_res < p.h || (p.y != nullptr && p.ldy < p.h) ||
                  (p.z != nullptr && p.ldz < p.h))) || (any_mod && n_mod > 1 && p.ld_mod < p.h)) {
        return fail(EDB200_ERR_INVALID, "block_norm: row strides must hold h columns");
    }
    const bool f8 = p.z != nullptr && p.z_dtype == EDB200_TYPE_F8_E4M3;
    if (f8 && (p.z_scale == nullptr || (many && p.ld_z_scale < (p.h + 127) / 128))) {
        return fail(EDB200_ERR_INVALID, "block_norm: e4m3 output needs z_scale with ceil(h / 128) columns");
    }
    auto at = [](const void* q) { return reinterpret_cast<uintptr_t>(q); };
    const int xs = bn::esize(p.x_dtype), ss = bn::esize(p.stream_dtype), zs = bn::esize(p.z_dtype);
    if ((p.x != nullptr && at(p.x) % xs) || at(p.residual) % ss || at(p.y) % ss || (p.z != nullptr && at(p.z) % zs) ||
        ((at(p.gate) | at(p.scale) | at(p.shift) | at(p.post_weight) | at(p.post_bias) | at(p.pre_weight) | at(p.pre_bias) |
          at(p.z_scale)) & 3u)) {
        return fail(EDB200_ERR_INVALID, "block_norm: buffers must be aligned to their elements");
    }
    // y in place: each thread reads its columns of a row before it writes them, so equal strides are safe
    if (p.y != nullptr && ((p.y == p.residual && many && p.ldy != p.ld_res) ||
                           (p.y == p.x && ((many && p.ldy != p.ldx) || p.x_dtype != p.stream_dtype)))) {
        return fail(EDB200_ERR_INVALID, "block_norm: y may alias residual or x with the same type and stride only");
    }
    // wide accesses: every row of every buffer on a 16-byte boundary (8 bytes for e4m3)
    auto wide = [&](const void* q, int64_t ld, int es, int bytes) { return q == nullptr || (at(q) % bytes == 0 && (!many || (ld * es) % bytes == 0)); };
    const int64_t ldm = n_mod > 1 ? p.ld_mod : 0;
    const bool vec = wide(p.x, p.ldx, xs, 16) && wide(p.residual, p.ld_res, ss, 16) && wide(p.y, p.ldy, ss, 16) &&
                     wide(p.z, p.ldz, zs, f8 ? 8 : 16) && wide(p.gate, ldm, 4, 16) && wide(p.scale, ldm, 4, 16) &&
                     wide(p.shift, ldm, 4, 16) && wide(p.post_weight, 0, 4, 16) && wide(p.post_bias, 0, 4, 16) &&
                     wide(p.pre_weight, 0, 4, 16) && wide(p.pre_bias, 0, 4, 16);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    double per = (double)ss;
    if (p.x != nullptr) per += xs;
    if (p.y != nullptr) per += ss;
    if (p.z != nullptr) per += zs;
    ProfScope prof(s, PROF_ELEMENTWISE, 0.0, per * (double)p.rows * (double)p.h);
    bn::Params P;
    P.p = p;
    P.p.ld_mod = ldm;
    if (p.stream_dtype == EDB200_TYPE_F32) {
        bn::launch_x<float>(P, vec, s);
    } else if (p.stream_dtype == EDB200_TYPE_F16) {
        bn::launch_x<__half>(P, vec, s);
    } else {
        bn::launch_x<__nv_bfloat16>(P, vec, s);
    }
    count_launch();
    return check_cuda(cudaGetLastError(), "block_norm launch");
}
