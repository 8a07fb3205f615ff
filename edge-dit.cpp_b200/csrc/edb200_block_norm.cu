// The norms around a block fused with its gate and the residual stream:
//
//   t = post(x);   y = residual_scale * residual + gate * t;   z = pre(y) * (1 + scale) + shift
//
// with post, pre = none, LayerNorm (v - mean) * rstd or RMSNorm v * rstd, times weight plus bias, and z cast or
// quantised to e4m3 with a scale for each 128 columns.
//
// Bound: HBM.  A row's x and residual are read once, live in registers through both norms, and y and z are written
// once; the statistics are f32 sums over registers, the variance taken around the mean (two sums, no cancellation).
// A row belongs to one warp (h <= 512, eight rows a CTA, sums by shuffles alone) or to one CTA of just as many warps as it
// needs.  A warp owns CH blocks of 128 columns, a lane four columns of each: every access of a warp is one run of memory
// (eight columns a lane took twice the f32 wavefronts), the places differ by constants, and a quantisation block's
// maximum is one reduction over the warp.  Four blocks a warp and 64 registers a thread keep three rows of 5120 under way on
// an SM (308 us at the first size below; two blocks a warp, one row: 388); where there are fewer rows than that, two blocks
// a warp finish a row sooner (1 x 5120: 3.7 against 4.0 us).
// Measured (f32 stream): 32760 x 5120 bf16 normed on both sides into e4m3 307 us back to back on the same operands (6.0 TB/s,
// 0.91 of the copy rate), 333 to 351 a call where other calls and operands come between (0.80 to 0.84); into f16 315;
// 154 x 1536 3.4 us.  Columns no multiple of four take single accesses: 32760 x 5117 739 us, so a row's h is better padded.
#include "edb200_internal.h"
#include "edb200_fp8.cuh"

namespace edb {
namespace bn {

struct Params {
    edb200_block_norm_t p;
    float inv_h;
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

// Pairs of f32: one instruction for two (each half rounded as the scalar operation's).
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
__device__ __forceinline__ uint64_t packed(float2 a) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a.x), "f"(a.y));
    return r;
}
__device__ __forceinline__ float2 apart(uint64_t a) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a));
    return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(packed(a)), "l"(packed(b)));
    return apart(r);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(packed(a)), "l"(packed(b)));
    return apart(r);
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(packed(a)), "l"(packed(b)), "l"(packed(c)));
    return apart(r);
}

// How a row is reached: ODD element by element; WIDE four columns at a time, h a multiple of four so that a piece is all
// inside or all outside; FULL the same where the warps' blocks are the row exactly and nothing is outside.
enum { ODD, WIDE, FULL };
// A vector's piece: columns from h on read zero.
template <int ACC>
__device__ __forceinline__ void load_vector(const float* row, int c, int h, float2 (&o)[2]) {
    if (ACC != ODD) {
        const float4 f = ACC == FULL || c < h ? __ldg(reinterpret_cast<const float4*>(row + c)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        o[0] = make_float2(f.x, f.y), o[1] = make_float2(f.z, f.w);
    } else {
        o[0] = make_float2(c < h ? row[c] : 0.0f, c + 1 < h ? row[c + 1] : 0.0f);
        o[1] = make_float2(c + 2 < h ? row[c + 2] : 0.0f, c + 3 < h ? row[c + 3] : 0.0f);
    }
}
template <int ACC, typename T>
__device__ __forceinline__ void store_piece(T* row, int c, int h, const float2 (&v)[2]) {
    if (ACC != ODD) {
        put4(row + c, v[0], v[1]);
    } else {
        const float w[4] = {v[0].x, v[0].y, v[1].x, v[1].y};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (c + e < h) row[c + e] = narrow<T>(w[e]);
        }
    }
}

// 1 / sqrt(a): the hardware's approximation and one Newton step, which takes its two roundings' error down to one.  An e4m3 z
// shows them wherever a value lies next to a border.  (It costs nothing measurable; the correctly rounded functions
// cost 15 % of the kernel.)
__device__ __forceinline__ float inverse_root(float a) {
    const float r = rsqrtf(a);
    const float e = fmaf(-a * r, r, 1.0f);
    return a > 0.0f && a <= 3.402823466e38f ? fmaf(0.5f * r, e, r) : r;   // 0 and infinity have no step
}

// v <- norm(v) * weight + bias over the row; the lane's columns are c0 + 128 i .. + 3, those from h on zero before and after.
// sh holds two reductions' worth of warp sums.
template <int CH, bool WARP, int ACC>
__device__ __forceinline__ void norm_row(float2 (&v)[CH][2], int kind, const float* weight, const float* bias, float eps, float inv_h,
                                         int h, int c0, float* sh) {
    if (kind == EDB200_NORM_LAYER) {
        float2 s = both(0.0f);
#pragma unroll
        for (int i = 0; i < CH; ++i) s = add2(s, add2(v[i][0], v[i][1]));
        const float2 mean = both(-row_sum<WARP>(s.x + s.y, sh) * inv_h);
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            v[i][0] = add2(v[i][0], mean);
            v[i][1] = add2(v[i][1], mean);
        }
        if (ACC != FULL && c0 + 128 * (CH - 1) + 4 > h) {   // columns beyond the row
#pragma unroll
            for (int i = 0; i < CH; ++i) {
                const int c = c0 + 128 * i;
                if (c >= h) v[i][0].x = 0.0f;
                if (c + 1 >= h) v[i][0].y = 0.0f;
                if (c + 2 >= h) v[i][1].x = 0.0f;
                if (c + 3 >= h) v[i][1].y = 0.0f;
            }
        }
    }
    float2 q = both(0.0f);
#pragma unroll
    for (int i = 0; i < CH; ++i) q = fma2(v[i][0], v[i][0], fma2(v[i][1], v[i][1], q));
    const float2 rstd = both(inverse_root(fmaf(row_sum<WARP>(q.x + q.y, sh + 32), inv_h, eps)));
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        v[i][0] = mul2(v[i][0], rstd);
        v[i][1] = mul2(v[i][1], rstd);
    }
    if (weight != nullptr) {
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            float2 w[2];
            load_vector<ACC>(weight, c0 + 128 * i, h, w);
            v[i][0] = mul2(v[i][0], w[0]);
            v[i][1] = mul2(v[i][1], w[1]);
        }
    }
    if (bias != nullptr) {
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            float2 w[2];
            load_vector<ACC>(bias, c0 + 128 * i, h, w);
            v[i][0] = add2(v[i][0], w[0]);
            v[i][1] = add2(v[i][1], w[1]);
        }
    }
}

// Largest |value| of the warp's 128 columns, by the order of the bits; NaN passes by.
__device__ __forceinline__ float warp_peak(const float2 (&v)[2]) {
    const float a = f8_peak(f8_peak(f8_peak(f8_peak(0.0f, v[0].x), v[0].y), v[1].x), v[1].y);
    return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(a)));
}

template <typename T, int CH, int ACC>
__device__ __forceinline__ void store_row(T* row, int c0, int h, const float2 (&v)[CH][2]) {
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        if (ACC == FULL || c0 + 128 * i < h) store_piece<ACC>(row, c0 + 128 * i, h, v[i]);
    }
}

template <typename TX, typename TS, int CH, bool WARP, int ACC>
__global__ void __launch_bounds__(WARP ? 256 : 1024)
block_norm_kernel(const __grid_constant__ Params P) {
    __shared__ float sh[128];
    const edb200_block_norm_t& p = P.p;
    const int64_t row = WARP ? static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5) : blockIdx.x;
    if (WARP && row >= p.rows) return;   // a whole warp; nothing below synchronises the CTA then
    const int h = static_cast<int>(p.h);
    const int lane = threadIdx.x & 31;
    const int b0 = WARP ? 0 : (threadIdx.x >> 5) * CH;   // the warp's first block of 128 columns
    const int c0 = b0 * 128 + 4 * lane;
    const int64_t mod = p.rows_per_mod > 0 ? static_cast<uint32_t>(row) / static_cast<uint32_t>(p.rows_per_mod) * p.ld_mod : 0;

    float2 t[CH][2], y[CH][2];
    const bool has_x = p.x != nullptr;
    {
        Four<TX> xs[CH];
        Four<TS> rs[CH];
        const TX* xr = static_cast<const TX*>(p.x) + (has_x ? row * p.ldx : 0);
        const TS* rr = static_cast<const TS*>(p.residual) + row * p.ld_res;
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const int c = c0 + 128 * i;
            if (ACC == FULL || (ACC == WIDE && c < h)) {
                if (has_x) xs[i].load(xr + c);
                rs[i].load(rr + c);
            } else {   // element-wise, or beyond the row: zeros
                if (has_x) xs[i].load_some(xr + c, ACC == WIDE ? 0 : h - c);
                rs[i].load_some(rr + c, ACC == WIDE ? 0 : h - c);
            }
        }
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            if (has_x) xs[i].get(t[i][0], t[i][1]);
            rs[i].get(y[i][0], y[i][1]);
        }
    }

    if (has_x && p.post_norm != EDB200_NORM_NONE) {
        norm_row<CH, WARP, ACC>(t, p.post_norm, p.post_weight, p.post_bias, p.post_eps, P.inv_h, h, c0, sh);
    }
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        y[i][0] = mul2(y[i][0], both(p.residual_scale));
        y[i][1] = mul2(y[i][1], both(p.residual_scale));
    }
    if (has_x && p.gate != nullptr) {
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            float2 g[2];
            load_vector<ACC>(p.gate + mod, c0 + 128 * i, h, g);
            y[i][0] = fma2(g[0], t[i][0], y[i][0]);
            y[i][1] = fma2(g[1], t[i][1], y[i][1]);
        }
    } else if (has_x) {
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            y[i][0] = add2(y[i][0], t[i][0]);
            y[i][1] = add2(y[i][1], t[i][1]);
        }
    }
    if (p.y != nullptr) store_row<TS, CH, ACC>(static_cast<TS*>(p.y) + row * p.ldy, c0, h, y);
    if (p.z == nullptr) return;   // uniform
    if (p.pre_norm != EDB200_NORM_NONE) {
        norm_row<CH, WARP, ACC>(y, p.pre_norm, p.pre_weight, p.pre_bias, p.pre_eps, P.inv_h, h, c0, sh + 64);
    }
    if (p.scale != nullptr) {
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            float2 m[2];
            load_vector<ACC>(p.scale + mod, c0 + 128 * i, h, m);
            y[i][0] = fma2(y[i][0], m[0], y[i][0]);
            y[i][1] = fma2(y[i][1], m[1], y[i][1]);
        }
    }
    if (p.shift != nullptr) {
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            float2 m[2];
            load_vector<ACC>(p.shift + mod, c0 + 128 * i, h, m);
            y[i][0] = add2(y[i][0], m[0]);
            y[i][1] = add2(y[i][1], m[1]);
        }
    }
    if (p.z_dtype == EDB200_TYPE_F8_E4M3) {
        // lane i makes the scale of the warp's block i; columns from h on add nothing: zero, or NaN in a row that has one
        float mine = 0.0f;
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            float a = warp_peak(y[i]);
            if (f8_has_infinity(a)) {   // the same in every lane
#pragma unroll
                for (int e = 0; e < 2; ++e) y[i][e] = make_float2(f8_no_infinity(y[i][e].x), f8_no_infinity(y[i][e].y));
                a = warp_peak(y[i]);
            }
            mine = lane == i ? a : mine;
        }
        float s, inv;
        f8_scale(mine, s, inv);
        if (lane < CH && (ACC == FULL || (b0 + lane) * 128 < h)) p.z_scale[row * p.ld_z_scale + b0 + lane] = s;
        uint8_t* zr = static_cast<uint8_t*>(p.z) + row * p.ldz;
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const float2 f = both(__shfl_sync(0xffffffffu, inv, i));
            const float2 u = mul2(y[i][0], f), v = mul2(y[i][1], f);
            const uint32_t w = f8_pack4(u.x, u.y, v.x, v.y);
            const int c = c0 + 128 * i;
            if (ACC != ODD) {
                if (ACC == FULL || c < h) __stcs(reinterpret_cast<uint32_t*>(zr + c), w);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (c + e < h) zr[c + e] = static_cast<uint8_t>(w >> (8 * e));
                }
            }
        }
    } else if (p.z_dtype == EDB200_TYPE_F32) {
        store_row<float, CH, ACC>(static_cast<float*>(p.z) + row * p.ldz, c0, h, y);
    } else if (p.z_dtype == EDB200_TYPE_F16) {
        store_row<__half, CH, ACC>(static_cast<__half*>(p.z) + row * p.ldz, c0, h, y);
    } else {
        store_row<__nv_bfloat16, CH, ACC>(static_cast<__nv_bfloat16*>(p.z) + row * p.ldz, c0, h, y);
    }
}

template <typename TX, typename TS, int CH, bool WARP>
static void launch_access(const Params& P, bool vec, unsigned grid, unsigned threads, cudaStream_t s) {
    const int64_t span = 128ll * CH * (WARP ? 1 : threads / 32);
    if (!vec) {
        block_norm_kernel<TX, TS, CH, WARP, ODD><<<grid, threads, 0, s>>>(P);
    } else if (P.p.h != span) {
        block_norm_kernel<TX, TS, CH, WARP, WIDE><<<grid, threads, 0, s>>>(P);
    } else {
        block_norm_kernel<TX, TS, CH, WARP, FULL><<<grid, threads, 0, s>>>(P);
    }
}

template <typename TX, typename TS>
static void launch_vec(const Params& P, bool vec, cudaStream_t s) {
    const int64_t rows = P.p.rows;
    const int blocks = static_cast<int>((P.p.h + 127) / 128);
    if (blocks <= 4) {
        const unsigned grid = static_cast<unsigned>((rows + 7) / 8);
        if (blocks <= 2) {
            launch_access<TX, TS, 2, true>(P, vec, grid, 256, s);
        } else {
            launch_access<TX, TS, 4, true>(P, vec, grid, 256, s);
        }
    } else if (blocks <= 64 && rows <= 2 * sm_count()) {
        launch_access<TX, TS, 2, false>(P, vec, static_cast<unsigned>(rows), 32u * ((blocks + 1) / 2), s);
    } else {
        launch_access<TX, TS, 4, false>(P, vec, static_cast<unsigned>(rows), 32u * ((blocks + 3) / 4), s);
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
    // wide accesses: four columns at a time from every buffer
    auto wide = [&](const void* q, int64_t ld, int es, int bytes) { return q == nullptr || (at(q) % bytes == 0 && (!many || (ld * es) % bytes == 0)); };
    const int64_t ldm = n_mod > 1 ? p.ld_mod : 0;
    const bool vec = p.h % 4 == 0 && wide(p.x, p.ldx, xs, 4 * xs) && wide(p.residual, p.ld_res, ss, 4 * ss) &&
                     wide(p.y, p.ldy, ss, 4 * ss) && wide(p.z, p.ldz, zs, 4 * zs) && wide(p.gate, ldm, 4, 16) && wide(p.scale, ldm, 4, 16) &&
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
    if (P.p.rows_per_mod > p.rows) P.p.rows_per_mod = p.rows;   // 32 bits hold it then
    P.inv_h = 1.0f / static_cast<float>(p.h);
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
