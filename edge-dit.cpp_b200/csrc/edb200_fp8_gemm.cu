// Matrix product over e4m3 operands with one f32 scale for each block of 128 k (edb200_mul_mat_fp8):
//
//   y[m, n] = sum_b  xs[m, b] ws[n / 128, b]  sum_{k in block b} x[m, k] w[n, k]        (+ bias, activation, ...)
//
// The inner sums run on the tensor cores (tcgen05 kind::f8f6f4, f32 accumulators in tensor memory).  A block's scale
// differs from row to row, so its sum cannot stay in one accumulator over all of k: the accumulators alternate between
// two places in tensor memory, one written by block b + 1's four MMAs while eight warps read the other, multiply by the
// block's scale and add into f32 registers ("promotion").  With tokens in the 128 lanes of tensor memory and features in
// its columns, xs[m, b] ws[n / 128, b] is one number per thread and the promotion one FMA per element.
//
// A 128 x 128-byte operand tile is exactly one block of 128 e4m3 values per row: one TMA box with 128-byte swizzle, four
// MMAs of 32 k.  Rows beyond m and n and values beyond k are zero-filled by TMA and masked in the epilogue.
#include "edb200_internal.h"
#include "edb200_ptx.cuh"
#include "edb200_fp8.cuh"

#include <atomic>
#include <cstring>

namespace edb {
namespace f8g {

// A warp waits as one, so that it also gives up as one: either a single lane runs the loop (copies and MMAs of the tile and
// few-row kernels: 256 x 5120 x 5120 17.9 us, with a vote after each wait 20.6) or each wait ends in a vote (the pair kernel,
// where the single lane was 1 to 2 % slower).

constexpr int BK = 128;                       // bytes = values of a k block
constexpr uint32_t kFmtE4M3 = 0;              // kind::f8f6f4
constexpr int SCALE_PITCH = 9;                // words between rows of eight scales in shared memory (no conflicts)

struct Params {
    const float* xs;
    const float* ws;
    long long ld_xs, ld_ws;
    const float* bias;
    const float* residual;
    const float* gate;
    void* out;
    float* out_scale;
    long long ldo, ld_res, ld_os;
    int M, N, kblocks;
    int act, out_dtype;
    int m_tiles, n_tiles, chunk;   // chunk: feature tiles walked together (pair kernel)
    int* err;
};

__device__ __forceinline__ void mma_f8_ss(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t"
        "}\n"
        ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// The same over a CTA pair: 256 tokens (128 in either CTA's tensor memory), B rows 0 .. N/2 - 1 from the leader's
// shared memory and the rest from the peer's.
__device__ __forceinline__ void mma_f8_ss_pair(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t"
        "}\n"
        ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// acc[i] += s * r[i], two elements an instruction: the packed form has the scalar one's rate (2.2 clocks for two) in half
// the issue slots.  Those matter: eight warps of back-to-back scalar FMAs left the issuing warp none, and the tensor pipe
// stood still until they were done.
template <int N, int R>
__device__ __forceinline__ void promote(float (&acc)[N], int at, const uint32_t (&r)[R], float s) {
    uint64_t ss;
    asm("mov.b64 %0, {%1, %1};" : "=l"(ss) : "f"(s));
#pragma unroll
    for (int i = 0; i < R; i += 2) {
        uint64_t a, b;
        asm("mov.b64 %0, {%1, %2};" : "=l"(a) : "f"(acc[at + i]), "f"(acc[at + i + 1]));
        asm("mov.b64 %0, {%1, %2};" : "=l"(b) : "r"(r[i]), "r"(r[i + 1]));
        asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(a) : "l"(b), "l"(ss));
        asm("mov.b64 {%0, %1}, %2;" : "=f"(acc[at + i]), "=f"(acc[at + i + 1]) : "l"(a));
    }
}

// v Phi(v), Phi the normal distribution's.  For v < 0 it is exp(-v^2 / 2) h, h = erfcx(|v| / sqrt 2) / 2 = t Q(t) with
// t = 1 / (1 + 0.305 |v|) and Q of degree 7 fitted to h / t on |v| <= 13.3, beyond which the result is 0 (weighted least
// squares towards equal relative errors; 0.305 makes them least, 1.7 u at u = 2^-24).  The relative error stays below
// (24 + 1.5 v^2) u: by 1 + erf, which cancels, it was 4 % at -5.  (The library's erfc in its place: 32760 x 5120 x 13824 into
// e4m3 4.4 ms, so 2.7.)
__device__ __forceinline__ float gelu_erf(float v) {
    const float t = __fdividef(1.0f, fmaf(0.305f, fabsf(v), 1.0f));
    float q = 0.0366991907f;
    q = fmaf(q, t, -0.1529883f);
    q = fmaf(q, t, 0.185716853f);
    q = fmaf(q, t, -0.0379767865f);
    q = fmaf(q, t, 0.121021658f);
    q = fmaf(q, t, 0.103420876f);
    q = fmaf(q, t, 0.122466817f);
    q = fmaf(q, t, 0.121639736f);
    float e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(v * v * -0.72134752f));   // -log2(e) / 2
    const float below = e * (q * t);
    return v * (v < 0.0f ? below : 1.0f - below);
}
// The others by exp and one division: gelu_tanh(v) = v / (1 + exp(-t)).  The fast exponential is off by 2 + 1.173 |argument|
// steps, so the relative error grows towards the negative tail: (9 + 2.4 |v|) u for SiLU, (9 + 8.4 |t|) u for gelu_tanh;
// where the divisor passes 2^126 the result is 0.
__device__ __forceinline__ float act_one(float v, int act) {
    if (act == EDB200_ACT_GELU_TANH) {
        const float u = 0.7978845608028654f * v * fmaf(0.044715f * v, v, 1.0f);
        return __fdividef(v, 1.0f + __expf(-2.0f * u));
    }
    if (act == EDB200_ACT_SILU) return __fdividef(v, 1.0f + __expf(-v));
    return gelu_erf(v);
}
template <int N>
__device__ __forceinline__ void bias_act(float (&v)[N], const float* bias, int act) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
        const float4 b = *reinterpret_cast<const float4*>(bias + i);
        v[i] += b.x, v[i + 1] += b.y, v[i + 2] += b.z, v[i + 3] += b.w;
    }
    if (act != EDB200_ACT_NONE) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = act_one(v[i], act);
    }
}

// Largest magnitude of a thread's columns n0 .. that lie inside N.
template <int N>
__device__ __forceinline__ float row_peak(const float (&v)[N], int n0, int n_end) {
    float a = 0.0f;
    if (n0 + N <= n_end) {
#pragma unroll
        for (int i = 0; i < N; ++i) a = f8_peak(a, v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) a = n0 + i < n_end ? f8_peak(a, v[i]) : a;
    }
    return a;
}

// Epilogue of a pair's promotion warp: lane l holds row m_first + l, columns n0 .. n0 + N - 1 (biased, activated), and memory
// wants runs of a row.  Pieces of 64 bytes a row go through the warp's staging buffer; then four lanes a row move 16 bytes
// each, eight rows an instruction.
constexpr int PITCH = 20;                     // words between staged rows (16 + 4: no conflicts)

// Rows 8 i + lane / 4 of a staged piece, this lane's four words: put(row of the warp, quarter of the 64 bytes, words).
template <typename F>
__device__ __forceinline__ void copy_out(const float* stage, int lane, const F& put) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = 8 * i + (lane >> 2);
        put(i, r, *reinterpret_cast<const uint4*>(stage + r * PITCH + 4 * (lane & 3)));
    }
}

// amax: of the row's 128 columns, none of them infinite (e4m3 output)
template <int N>
__device__ __forceinline__ void store_rows(const Params& P, const float (&v)[N], int m_first, int n0, int lane, float* stage,
                                           const float* gate, float amax) {
    const int rows = P.M - m_first;           // of the warp's, inside
    const int q = lane & 3;
    if (P.out_dtype == EDB200_TYPE_F32) {
        const long long at = static_cast<long long>(m_first + (lane >> 2)) * P.ldo;
        const long long res_at = static_cast<long long>(m_first + (lane >> 2)) * P.ld_res;
#pragma unroll
        for (int c = 0; c < N / 16; ++c) {    // 16 columns a piece
            const int n = n0 + 16 * c + 4 * q;
            float4 res[4];
            if (P.gate != nullptr) {          // on their way while the piece is staged
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (8 * i + (lane >> 2) < rows && n + 4 <= P.N) {
                        res[i] = *reinterpret_cast<const float4*>(P.residual + res_at + 8 * i * P.ld_res + n);
                    }
                }
            }
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                *reinterpret_cast<float4*>(stage + lane * PITCH + i) = make_float4(v[16 * c + i], v[16 * c + i + 1], v[16 * c + i + 2], v[16 * c + i + 3]);
            }
            __syncwarp();
            const float4 g = *reinterpret_cast<const float4*>(gate + 16 * c + 4 * q);
            copy_out(stage, lane, [&](int i, int r, uint4 u) {
                if (r >= rows || n >= P.N) return;
                float4 x = *reinterpret_cast<float4*>(&u);
                float* o = static_cast<float*>(P.out) + at + 8 * i * P.ldo + n;
                if (n + 4 <= P.N) {
                    if (P.gate != nullptr) {
                        x = make_float4(fmaf(g.x, x.x, res[i].x), fmaf(g.y, x.y, res[i].y), fmaf(g.z, x.z, res[i].z), fmaf(g.w, x.w, res[i].w));
                    }
                    *reinterpret_cast<float4*>(o) = x;
                } else {                      // the last columns of a row that does not divide
                    const float w[3] = {x.x, x.y, x.z}, h[3] = {g.x, g.y, g.z};
#pragma unroll
                    for (int e = 0; e < 3; ++e) {
                        if (n + e >= P.N) continue;
                        o[e] = P.gate != nullptr ? fmaf(h[e], w[e], P.residual[res_at + 8 * i * P.ld_res + n + e]) : w[e];
                    }
                }
            });
        }
    } else if (P.out_dtype != EDB200_TYPE_F8_E4M3) {
        const bool bf = P.out_dtype == EDB200_TYPE_BF16;
        uint16_t* base = static_cast<uint16_t*>(P.out) + static_cast<long long>(m_first + (lane >> 2)) * P.ldo;
#pragma unroll
        for (int c = 0; c < N / 32; ++c) {    // 32 columns a piece
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 32; i += 8) {
                uint32_t w[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float a = v[32 * c + i + 2 * j], b = v[32 * c + i + 2 * j + 1];
                    if (bf) {
                        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
                        w[j] = *reinterpret_cast<const uint32_t*>(&h);
                    } else {
                        const __half2 h = __floats2half2_rn(a, b);
                        w[j] = *reinterpret_cast<const uint32_t*>(&h);
                    }
                }
                *reinterpret_cast<uint4*>(stage + lane * PITCH + i / 2) = make_uint4(w[0], w[1], w[2], w[3]);
            }
            __syncwarp();
            const int n = n0 + 32 * c + 8 * q;
            copy_out(stage, lane, [&](int i, int r, uint4 u) {
                if (r >= rows || n >= P.N) return;
                uint16_t* o = base + 8 * i * P.ldo + n;
                if (n + 8 <= P.N) {
                    *reinterpret_cast<uint4*>(o) = u;
                } else {
                    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        if (n + e < P.N) o[e] = static_cast<uint16_t>(w[e >> 1] >> (16 * (e & 1)));
                    }
                }
            });
        }
    } else {
        float s, inv;
        f8_scale(amax, s, inv);
        if (lane < rows && (n0 & 127) == 0 && n0 < P.N) P.out_scale[static_cast<long long>(m_first + lane) * P.ld_os + (n0 >> 7)] = s;
        uint8_t* base = static_cast<uint8_t*>(P.out) + static_cast<long long>(m_first + (lane >> 2)) * P.ldo;
#pragma unroll
        for (int c = 0; c < N / 64; ++c) {    // 64 columns a piece
            __syncwarp();
#pragma unroll
            for (int i = 64 * c; i < 64 * c + 64; i += 16) {
                uint32_t w[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    w[j] = f8_pack4(v[i + 4 * j] * inv, v[i + 4 * j + 1] * inv, v[i + 4 * j + 2] * inv, v[i + 4 * j + 3] * inv);
                }
                *reinterpret_cast<uint4*>(stage + lane * PITCH + (i - 64 * c) / 4) = make_uint4(w[0], w[1], w[2], w[3]);
            }
            __syncwarp();
            const int n = n0 + 64 * c + 16 * q;
            copy_out(stage, lane, [&](int i, int r, uint4 u) {
                if (r >= rows || n >= P.N) return;
                uint8_t* o = base + 8 * i * P.ldo + n;
                if (n + 16 <= P.N) {
                    *reinterpret_cast<uint4*>(o) = u;
                } else {
                    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        if (n + e < P.N) o[e] = static_cast<uint8_t>(w[e >> 2] >> (8 * (e & 3)));
                    }
                }
            });
        }
    }
}

// What becomes of a token's finished features.
enum { TO_F32, TO_STREAM, TO_F16, TO_BF16, TO_F8 };   // TO_STREAM: residual + gate * y

// Four neighbouring features of token m in each lane of a warp: the 128 columns of one e4m3 block.  `whole`: all four exist.
template <int TO>
__device__ __forceinline__ void store_token(const Params& P, float (&y)[4], const float (&gate)[4], long long m, int n, bool whole,
                                            int lane) {
    if constexpr (TO == TO_F8) {
        float a = row_peak(y, n, P.N);
#pragma unroll
        for (int k = 16; k > 0; k >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, k));
        if (f8_has_infinity(a)) {   // uniform
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = f8_no_infinity(y[e]);
            a = row_peak(y, n, P.N);
#pragma unroll
            for (int k = 16; k > 0; k >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, k));
        }
        float s, inv;
        f8_scale(a, s, inv);
        const uint32_t w = f8_pack4(y[0] * inv, y[1] * inv, y[2] * inv, y[3] * inv);
        uint8_t* o = static_cast<uint8_t*>(P.out) + m * P.ldo + n;
        if (whole) {
            *reinterpret_cast<uint32_t*>(o) = w;
        } else {
            for (int e = 0; e < P.N - n; ++e) o[e] = static_cast<uint8_t>(w >> (8 * e));
        }
        if (lane == 0) P.out_scale[m * P.ld_os + (n >> 7)] = s;
    } else if constexpr (TO == TO_F32 || TO == TO_STREAM) {
        float* o = static_cast<float*>(P.out) + m * P.ldo + n;
        if (whole) {
            if (TO == TO_STREAM) {
                const float4 q = *reinterpret_cast<const float4*>(P.residual + m * P.ld_res + n);
                y[0] = fmaf(gate[0], y[0], q.x), y[1] = fmaf(gate[1], y[1], q.y);
                y[2] = fmaf(gate[2], y[2], q.z), y[3] = fmaf(gate[3], y[3], q.w);
            }
            *reinterpret_cast<float4*>(o) = make_float4(y[0], y[1], y[2], y[3]);
        } else {
            const float* q = P.residual + m * P.ld_res + n;   // read for TO_STREAM only
#pragma unroll
            for (int e = 0; e < 3; ++e) {
                if (n + e < P.N) o[e] = TO == TO_STREAM ? fmaf(gate[e], y[e], q[e]) : y[e];
            }
        }
    } else {
        uint16_t h[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            h[e] = TO == TO_BF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(y[e])) : __half_as_ushort(__float2half_rn(y[e]));
        }
        uint16_t* o = static_cast<uint16_t*>(P.out) + m * P.ldo + n;
        if (whole) {
            *reinterpret_cast<uint2*>(o) = make_uint2(h[0] | (uint32_t(h[1]) << 16), h[2] | (uint32_t(h[3]) << 16));
        } else {
#pragma unroll
            for (int e = 0; e < 3; ++e) {
                if (n + e < P.N) o[e] = h[e];
            }
        }
    }
}

// A warp's share of a finished tile: tokens first, first + step, ..., four features a lane.  PARTS: CTAs whose sums are added
// (at most), all of them asked for before the first is added.
template <int TO, int PARTS>
__device__ __forceinline__ void finish_rows(const Params& P, const float* sums, int pitch, int tokens, int m0, int n0, int first, int step,
                                            int parts, int lane) {
    const int n = n0 + 4 * lane;
    const bool whole = n + 4 <= P.N;
    float bias[4], gate[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        bias[e] = (P.bias != nullptr && n + e < P.N) ? __ldg(P.bias + n + e) : 0.0f;
        gate[e] = (TO == TO_STREAM && n + e < P.N) ? __ldg(P.gate + n + e) : 0.0f;
    }
    const int end = P.M - m0 < tokens ? P.M - m0 : tokens;
    for (int t = first; t < end; t += step) {
        float4 v;
        if constexpr (PARTS == 1) {
            v = *reinterpret_cast<const float4*>(sums + t * pitch + 4 * lane);
        } else {
            float4 q[PARTS];
#pragma unroll
            for (int p = 0; p < PARTS; ++p) {
                if (p < parts) q[p] = cluster_load4(sums + t * pitch + 4 * lane, p);
            }
            v = q[0];
#pragma unroll
            for (int p = 1; p < PARTS; ++p) {
                if (p < parts) v.x += q[p].x, v.y += q[p].y, v.z += q[p].z, v.w += q[p].w;
            }
        }
        float y[4] = {v.x + bias[0], v.y + bias[1], v.z + bias[2], v.w + bias[3]};
        if (P.act != EDB200_ACT_NONE) {
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = act_one(y[e], P.act);
        }
        store_token<TO>(P, y, gate, m0 + t, n, whole, lane);
    }
}

// The end of a tile shared by `parts` CTAs of a cluster: sums[token][128 features] lie in each one's shared memory; every
// CTA finishes each parts-th token.  One loop for each output, chosen outside it: with the choice inside, a token cost 575
// clocks.
__device__ __forceinline__ void finish_tokens(const Params& P, const float* sums, int pitch, int tokens, int m0, int n0, int part,
                                              int parts, int warp, int warps, int lane, bool bad) {
    if (parts > 1) {
        cluster_sync_all();
    } else {
        __syncthreads();
    }
    const int first = bad ? tokens : part + parts * warp, step = parts * warps;   // after a wait that gave up: nothing
    const int to = P.out_dtype == EDB200_TYPE_F32    ? (P.gate != nullptr ? TO_STREAM : TO_F32)
                   : P.out_dtype == EDB200_TYPE_F16  ? TO_F16
                   : P.out_dtype == EDB200_TYPE_BF16 ? TO_BF16
                                                     : TO_F8;
#define EDB_FINISH(TO)                                                                                \
    if (parts == 1) {                                                                                 \
        finish_rows<TO, 1>(P, sums, pitch, tokens, m0, n0, first, step, parts, lane);                 \
    } else {                                                                                          \
        finish_rows<TO, 8>(P, sums, pitch, tokens, m0, n0, first, step, parts, lane);                 \
    }
    switch (to) {
        case TO_F32: EDB_FINISH(TO_F32) break;
        case TO_STREAM: EDB_FINISH(TO_STREAM) break;
        case TO_F16: EDB_FINISH(TO_F16) break;
        case TO_BF16: EDB_FINISH(TO_BF16) break;
        default: EDB_FINISH(TO_F8) break;
    }
#undef EDB_FINISH
    if (parts > 1) cluster_sync_all();   // no CTA leaves while another reads its sums
}

// Copies of four bytes from global to shared memory that hold no register while they are under way.  `in` false: nothing is
// read, zero is written (src is any address).
__device__ __forceinline__ void copy4(float* dst, const float* src, bool in = true) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(in ? 4 : 0) : "memory");
}
// Waits for this thread's; the warp's after a __syncwarp.
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// Starts the copy of one group of scales: xs of 128 rows from m0 on, this lane's block `at`, as [row][8 of SCALE_PITCH], then
// ws of `halves` weight blocks.  Four rows of eight blocks a copy; rows past the end follow the last one.  A warp brings ROWS
// rows.  (By loads, as many under way as registers allow, a change elsewhere in the kernel that left the compiler one
// register less put them one behind the other: 600 x 1024 x 4096 17 us instead of 12.)
template <int FIRST, int ROWS>
__device__ __forceinline__ void copy_scales(const Params& P, float* dst, int m0, int at, int n_block, int halves, int lane) {
    const int nb_last = (P.N - 1) >> 7;
    if (FIRST == 0 && lane < 8 * halves) {
        const int nb = n_block + (lane >> 3);
        copy4(dst + 128 * SCALE_PITCH + lane, P.ws + static_cast<long long>(nb < nb_last ? nb : nb_last) * P.ld_ws + at);
    }
#pragma unroll 8
    for (int r = FIRST + (lane >> 3); r < FIRST + ROWS; r += 4) {
        const int m = m0 + r < P.M ? m0 + r : P.M - 1;
        copy4(dst + r * SCALE_PITCH + (lane & 7), P.xs + m * P.ld_xs + at);
    }
}

// Starts a warp's copy of a vector's 128 values from n0 on; zero where there are none.  A vector may start anywhere.
__device__ __forceinline__ void copy_vector(const Params& P, float* dst, const float* src, int n0, int lane) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int c = 32 * i + lane;
        const bool in = src != nullptr && n0 + c < P.N;
        copy4(dst + c, in ? src + n0 + c : P.xs, in);
    }
}

// ------------------------------------------------------------------ one CTA per 128 tokens x 128 features
// For products whose 256 x 256 tiles are too few or too empty for the CTA pairs below (256 x 5120 x 5120 17.9 us; pairs 25).
// Tokens in the lanes, features in the columns of four accumulators; eight promotion warps of 32 tokens x 64 features,
// warps 2 and 3 bringing the scales as in the pairs.  Where the tiles leave SMs idle a cluster of up to eight CTAs shares
// one, each a run of its k blocks; sums meet in shared memory and are added in the order of the parts.
namespace tile {
constexpr int STAGES = 5, BUFS = 4;
constexpr int A_BYTES = 128 * BK, STAGE_BYTES = 2 * A_BYTES;
constexpr int WARPS = 8;                                        // promotion warps
constexpr int CPT = 64;                                         // columns of a promotion thread
constexpr int THREADS = 32 * (WARPS + 4);                       // warp 0 TMA, 1 MMA, 2 and 3 scales, 4-11 promotion; all store
constexpr int SUM_PITCH = 132;                                  // words between rows of the sums (no conflicts)
constexpr int SCALE_WORDS = 128 * SCALE_PITCH + 8;              // a group of eight blocks: [row][8], ws [8]
constexpr int OFF_SCALE = STAGES * STAGE_BYTES;
constexpr int OFF_BAR = OFF_SCALE + 2 * SCALE_WORDS * 4;
constexpr int SMEM_BYTES = OFF_BAR + 256 + 1024;
static_assert(SMEM_BYTES <= 227 * 1024 && 128 * SUM_PITCH * 4 <= OFF_SCALE, "shared memory plan");
}  // namespace tile

__global__ void __launch_bounds__(tile::THREADS, 1)
fp8_tile_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                const __grid_constant__ Params P, const int parts) {
    using namespace tile;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + OFF_BAR);   // [STAGES]
    uint64_t* empty = full + STAGES;                                // [STAGES]
    uint64_t* acc_full = empty + STAGES;                            // [BUFS]
    uint64_t* acc_empty = acc_full + BUFS;                          // [BUFS]
    uint64_t* sc_full = acc_empty + BUFS;                           // [2]
    uint64_t* sc_empty = sc_full + 2;                               // [2]
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sc_empty + 2);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    float* scales = reinterpret_cast<float*>(smem + OFF_SCALE);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int t = blockIdx.x / parts, part = blockIdx.x - t * parts;   // a cluster is `parts` neighbours: its rank
    const int n_tile = t / P.m_tiles, m_tile = t - n_tile * P.m_tiles;
    const int n0 = n_tile * 128, m0 = m_tile * 128;
    const int b_first = static_cast<int>(static_cast<long long>(P.kblocks) * part / parts);
    const int blocks = static_cast<int>(static_cast<long long>(P.kblocks) * (part + 1) / parts) - b_first;

    if (threadIdx.x == 0) {
        for (int i = 0; i < STAGES; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < BUFS; ++i) {
            mbar_init(&acc_full[i], 1);
            mbar_init(&acc_empty[i], WARPS);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sc_full[i], 2);
            mbar_init(&sc_empty[i], WARPS);
        }
        *abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    if (warp == 0 && lane == 0) {
        tma_prefetch_desc(&map_x);
        tma_prefetch_desc(&map_w);
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem_base = *tmem_slot;
    float sum[CPT];

    if (warp == 0) {
        uint32_t s = 0, ph = 0;
        if (elect_one()) {
            for (int b = 0; b < blocks; ++b) {
                if (!mbar_wait(&empty[s], ph ^ 1u, abort_flag, P.err)) break;
                uint8_t* stage = smem + s * STAGE_BYTES;
                mbar_arrive_expect_tx(&full[s], STAGE_BYTES);
                tma_load_2d(stage, &map_x, &full[s], (b_first + b) * BK, m0);
                tma_load_2d(stage + A_BYTES, &map_w, &full[s], (b_first + b) * BK, n0);
                if (++s == STAGES) {
                    s = 0;
                    ph ^= 1u;
                }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        const uint32_t idesc = make_idesc(kDFmtF32, kFmtE4M3, kFmtE4M3, 0, 0, 128, 128);
        uint32_t s = 0, ph = 0;
        if (elect_one()) {
            for (int b = 0; b < blocks; ++b) {
                const uint32_t buf = b % BUFS, aph = (b / BUFS) & 1u;
                if (!mbar_wait(&full[s], ph, abort_flag, P.err)) break;
                if (!mbar_wait(&acc_empty[buf], aph ^ 1u, abort_flag, P.err)) break;
                tc_fence_after_sync();
                const uint32_t a_addr = smem_u32(smem + s * STAGE_BYTES), b_addr = a_addr + A_BYTES;
#pragma unroll
                for (int j = 0; j < BK / 32; ++j) {
                    mma_f8_ss(tmem_base + buf * 128, make_smem_desc_sw128(a_addr + j * 32, 16, 1024),
                              make_smem_desc_sw128(b_addr + j * 32, 16, 1024), idesc, j > 0 ? 1u : 0u);
                }
                mma_commit(&acc_full[buf]);
                mma_commit(&empty[s]);
                if (++s == STAGES) {
                    s = 0;
                    ph ^= 1u;
                }
            }
        }
        __syncwarp();
    } else if (warp == 2 || warp == 3) {   // half of the rows' scales each
        for (int b = 0; b < blocks; b += 8) {
            const int g = b >> 3;
            if (!mbar_wait_warp(&sc_empty[g & 1], ((g >> 1) & 1) ^ 1u, abort_flag, P.err)) break;
            const int at = b_first + (b + (lane & 7) < blocks ? b + (lane & 7) : blocks - 1);
            if (warp == 2) {
                copy_scales<0, 64>(P, scales + (g & 1) * SCALE_WORDS, m0, at, n_tile, 1, lane);
            } else {
                copy_scales<64, 64>(P, scales + (g & 1) * SCALE_WORDS, m0, at, n_tile, 1, lane);
            }
            copies_wait();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sc_full[g & 1]);
        }
    } else if (warp >= 4) {
        const int quarter = warp & 3, side = (warp - 4) >> 2;   // lanes of tensor memory, half of the columns
        const int row = quarter * 32 + lane;
        const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + side * CPT;
#pragma unroll
        for (int i = 0; i < CPT; ++i) sum[i] = 0.0f;
        for (int b = 0; b < blocks; ++b) {
            const uint32_t buf = b % BUFS, aph = (b / BUFS) & 1u;
            const int g = b >> 3;
            bool ok = true;
            if ((b & 7) == 0) ok = mbar_wait_warp(&sc_full[g & 1], (g >> 1) & 1, abort_flag, P.err);
            ok = ok && mbar_wait_warp(&acc_full[buf], aph, abort_flag, P.err);
            if (!ok) break;
            tc_fence_after_sync();
            uint32_t r0[32], r1[32];
            tmem_ld_32x32b_x32(taddr + buf * 128, r0);
            const float* sc = scales + (g & 1) * SCALE_WORDS;
            const float scale = sc[row * SCALE_PITCH + (b & 7)] * sc[128 * SCALE_PITCH + (b & 7)];
            tmem_wait_ld();
            tmem_ld_32x32b_x32(taddr + buf * 128 + 32, r1);
            promote(sum, 0, r0, scale);
            tmem_wait_ld();
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&acc_empty[buf]);
                if ((b & 7) == 7) mbar_arrive(&sc_empty[g & 1]);
            }
            promote(sum, 32, r1, scale);
        }
    }
    tc_fence_before_sync();
    __syncthreads();            // every block has been read: the copies and MMAs of this CTA are done
    const bool bad = *abort_flag != 0;
    if (bad) {
        for (int i = 0; i < 200; ++i) __nanosleep(1000);   // let copies and MMAs in flight land
        __syncthreads();
    }
    float* sums = reinterpret_cast<float*>(smem);   // [128][SUM_PITCH]
    if (warp >= 4) {
        const float (&v)[CPT] = sum;
        float* o = sums + ((warp & 3) * 32 + lane) * SUM_PITCH + ((warp - 4) >> 2) * CPT;
#pragma unroll
        for (int i = 0; i < CPT; i += 4) *reinterpret_cast<float4*>(o + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
    }
    finish_tokens(P, sums, SUM_PITCH, 128, m0, n0, part, parts, warp, THREADS / 32, lane, bad);
    if (warp == 1) {
        tc_fence_after_sync();
        tmem_dealloc(tmem_base, 512);
    }
}

// The residual rows of a CTA's 128 x 256 outputs into L2 while the products run (128 bytes a prefetch): the epilogue's loads
// then wait for L2, not for memory.
__device__ __forceinline__ void prefetch_residual(const Params& P, int m0, int n0, int lane) {
    const int n = n0 + 32 * (lane & 7);
    if (n >= P.N) return;
    const int rows = P.M - m0 < 128 ? P.M - m0 : 128;
    for (int r = lane >> 3; r < rows; r += 4) {
        asm volatile("prefetch.global.L2 [%0];" ::"l"(P.residual + static_cast<long long>(m0 + r) * P.ld_res + n));
    }
}

// ------------------------------------------------------ CTA pairs: 256 tokens x 256 features, one pair per two SMs
// The leader's MMAs span both CTAs (cta_group::2): each stages its own 128 tokens and half of the 256 features, so an
// SM takes in 32 KB for 512 clocks of tensor work.  The two 128-feature halves of a block are MMAs and accumulators of
// their own: all 512 tensor-memory columns hold [half][2 alternating][128].  Each of eight promotion warps owns 32 tokens x
// one half, which is one weight block and, for e4m3 output, one quantisation block; it asks for 64 columns at a time and
// gives the accumulator back before it adds the second 64.  Sixteen warps of half the columns were slower (1.63 against 1.9
// PFLOP/s), and so was one 256-column accumulator for both halves.
// Each half has an issuer of its own (warps 1 and 2 of the leader): waiting, issuing and committing are a chain of about
// 250 clocks a group for one thread, twice that per block for a common one.
// Warp 3 brings the scales, eight blocks of the CTA's 128 rows at a time, two groups in shared memory.  The promotion
// warps touch no global memory while they add: tcgen05.wait::ld waited for their loads, too, and a block took 1060 clocks
// instead of 780.  A tile's bias and gate they copy to a place of each warp's own, asynchronously, while the sums run: a
// barrier among the warps of a half, which one place for all four would need, has no limit and would wait for good for a
// warp whose wait has given up.
// Signals across the pair: the peer's warp 1 passes its full barriers on to the leader's (two arrivals there: own copies,
// peer's); acc_empty counts the promotion warps of both CTAs; the commits arrive in both.
// Measured, m x k x n, first launches on a rested GPU (1.9 GHz) and back to back under its power cap (1.4 to 1.6 GHz):
//   32760 x 5120 x 13824 into f16         2.22 ms (2.1 PFLOP/s)    2.56 ms (1.8)
//   the same, GELU into e4m3              2.33                     2.69
//   32760 x 13824 x 5120 into the stream  2.38                     2.79
// loads and MMAs alone 1.46 ms, MMAs alone 1.17.  Bound by the loop MMA - commit - reading - signal - MMA: two blocks an
// accumulator pair take about 1900 clocks, of which 512 are MMAs of the half, 550 the reading (four warps of 32 lanes, each all
// 128 columns), and the signals between the SMs the rest.  20 bytes a thread are spilled, 60 read back.
namespace pair {
constexpr int STAGES = 5;
constexpr int A_BYTES = 128 * BK, B_HALF = 64 * BK, STAGE_BYTES = A_BYTES + 2 * B_HALF;
constexpr int WARPS = 8;
constexpr int CPT = 128;
constexpr int OFF_STAGE = STAGES * STAGE_BYTES;
constexpr int OFF_VEC = OFF_STAGE + WARPS * 32 * PITCH * 4;     // [warp][bias 128, gate 128]
constexpr int SCALE_WORDS = 128 * SCALE_PITCH + 16;              // a group: [row][8 blocks], then ws [half][8]
constexpr int OFF_SCALE = OFF_VEC + WARPS * 256 * 4;
constexpr int OFF_BAR = OFF_SCALE + 2 * SCALE_WORDS * 4;
constexpr int SMEM_BYTES = OFF_BAR + 256 + 1024;
constexpr int THREADS = 32 * (WARPS + 4);                       // registers move in groups of four warps
static_assert(SMEM_BYTES <= 227 * 1024, "shared memory plan");
}  // namespace pair

__device__ __forceinline__ void pair_tile_at(const Params& P, int t, int& m_tile, int& n_tile) {
    const int per = P.m_tiles * P.chunk;
    const int c = t / per, r = t - c * per;
    const int first = c * P.chunk, width = P.n_tiles - first < P.chunk ? P.n_tiles - first : P.chunk;
    m_tile = r / width;
    n_tile = first + r - m_tile * width;
}

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(pair::THREADS, 1)
fp8_pair_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                const __grid_constant__ Params P) {
    using namespace pair;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + OFF_BAR);   // [STAGES]
    uint64_t* empty = full + STAGES;                                // [STAGES]
    uint64_t* acc_full = empty + STAGES;                            // [half][2]
    uint64_t* acc_empty = acc_full + 4;                             // [half][2]  (the leader's are used)
    uint64_t* sc_full = acc_empty + 4;                              // [2]
    uint64_t* sc_empty = sc_full + 2;                               // [2]
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sc_empty + 2);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = static_cast<int>(cluster_ctarank());
    const int first = blockIdx.x >> 1, step = gridDim.x >> 1;
    const int tiles = P.m_tiles * P.n_tiles;

    if (threadIdx.x == 0) {
        for (int i = 0; i < STAGES; ++i) {
            mbar_init(&full[i], rank == 0 ? 2 : 1);
            mbar_init(&empty[i], 2);                  // either half's MMAs have read the stage
        }
        for (int i = 0; i < 4; ++i) {
            mbar_init(&acc_full[i], 1);
            mbar_init(&acc_empty[i], WARPS);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sc_full[i], 1);
            mbar_init(&sc_empty[i], WARPS);
        }
        *abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == 1) {
        tmem_alloc_pair(tmem_slot, 512);
        tmem_relinquish_pair();
    }
    if (warp == 0 && lane == 0) {
        tma_prefetch_desc(&map_x);
        tma_prefetch_desc(&map_w);
    }
    tc_fence_before_sync();
    __syncthreads();
    cluster_sync_all();     // the peer's barriers are initialised before anything arrives on them
    tc_fence_after_sync();
    const uint32_t tmem_base = *tmem_slot;

    // 168 registers a thread at launch (384 threads); the promotion warps take what the others give up:
    // 256 x 232 + 128 x 40 = 384 x 168
    if (warp >= 4) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
        const int quarter = warp & 3, side = (warp - 4) >> 2;
        const int row = quarter * 32 + lane;
        float* stage = reinterpret_cast<float*>(smem + OFF_STAGE) + (warp - 4) * 32 * PITCH;
        const float* scales = reinterpret_cast<const float*>(smem + OFF_SCALE);
        uint32_t sg = 0;   // group of scales, over all tiles
        const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + side * 256;
        const uint32_t free0 = leader_address(&acc_empty[2 * side]), free1 = leader_address(&acc_empty[2 * side + 1]);
        float* vec = reinterpret_cast<float*>(smem + OFF_VEC) + (warp - 4) * 256;
        uint32_t g = 0;
        bool ok = true;
        for (int t = first; ok && t < tiles; t += step) {
            int m_tile, n_tile;
            pair_tile_at(P, t, m_tile, n_tile);
            const int m_first = m_tile * 256 + rank * 128 + quarter * 32;   // the warp's rows
            const int nc = n_tile * 256 + side * CPT;                       // the thread's columns
            __syncwarp();                                                   // the last tile's vectors have been read
            copy_vector(P, vec, P.bias, nc, lane);
            copy_vector(P, vec + 128, P.gate, nc, lane);
            float sum[CPT];
#pragma unroll
            for (int i = 0; i < CPT; ++i) sum[i] = 0.0f;
            // One block's reading runs into the next one's: the barrier of block b + 1 is looked at and its first columns
            // are under way before block b's last products are added.
            ok = mbar_wait_warp(&sc_full[sg & 1u], (sg >> 1) & 1u, abort_flag, P.err) &&
                 mbar_wait_warp(&acc_full[2 * side + (g & 1u)], (g >> 1) & 1u, abort_flag, P.err);
            if (!ok) break;
            const float* sc = scales + (sg & 1u) * SCALE_WORDS;
            float scale = sc[row * SCALE_PITCH] * sc[128 * SCALE_PITCH + side * 8];
            uint32_t r0[32], r1[32];
            tc_fence_after_sync();
            tmem_ld_32x32b_x32(taddr + (g & 1u) * 128, r0);
            tmem_ld_32x32b_x32(taddr + (g & 1u) * 128 + 32, r1);
            for (int b = 0; b < P.kblocks; ++b, ++g) {
                const uint32_t at = taddr + (g & 1u) * 128, next = taddr + ((g + 1) & 1u) * 128;
                const float s = scale;
                const bool more = b + 1 < P.kblocks;
                tmem_wait_ld();
                promote(sum, 0, r0, s);
                tmem_ld_32x32b_x32(at + 64, r0);
                promote(sum, 32, r1, s);
                tmem_ld_32x32b_x32(at + 96, r1);
                const bool there = mbar_test(&acc_full[2 * side + ((g + 1) & 1u)], ((g + 1) >> 1) & 1u);
                if (((b + 1) & 7) == 0 || !more) {   // the group of scales is read
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sc_empty[sg & 1u]);
                    ++sg;
                    sc = scales + (sg & 1u) * SCALE_WORDS;
                    if (more) ok = mbar_wait_warp(&sc_full[sg & 1u], (sg >> 1) & 1u, abort_flag, P.err);
                }
                const float sx = sc[row * SCALE_PITCH + ((b + 1) & 7)], sw = sc[128 * SCALE_PITCH + side * 8 + ((b + 1) & 7)];
                tmem_wait_ld();
                tc_fence_before_sync();
                if (lane == 0) mbar_arrive_relaxed((g & 1u) ? free1 : free0);
                scale = sx * sw;                                  // unused after the last block
                if (__all_sync(0xffffffffu, there) && more) {
                    tc_fence_after_sync();
                    promote(sum, 64, r0, s);
                    tmem_ld_32x32b_x32(next, r0);
                    promote(sum, 96, r1, s);
                    tmem_ld_32x32b_x32(next + 32, r1);
                } else {
                    promote(sum, 64, r0, s);
                    promote(sum, 96, r1, s);
                    if (more) {
                        ok = ok && mbar_wait_warp(&acc_full[2 * side + ((g + 1) & 1u)], ((g + 1) >> 1) & 1u, abort_flag, P.err);
                        if (!ok) break;
                        tc_fence_after_sync();
                        tmem_ld_32x32b_x32(next, r0);
                        tmem_ld_32x32b_x32(next + 32, r1);
                    }
                }
                if (!ok) break;
            }
            if (!ok) break;
            copies_wait();
            __syncwarp();
            float (&acc)[CPT] = sum;
            bias_act(acc, vec, P.act);
            float amax = 0.0f;
            if (P.out_dtype == EDB200_TYPE_F8_E4M3) {
                amax = row_peak(acc, nc, P.N);
                if (f8_has_infinity(amax)) {
#pragma unroll
                    for (int i = 0; i < CPT; ++i) acc[i] = f8_no_infinity(acc[i]);
                    amax = row_peak(acc, nc, P.N);
                }
            }
            store_rows(P, acc, m_first, nc, lane, stage, vec + 128, amax);
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
        if (warp == 0) {
            uint32_t s = 0, ph = 0;
            bool ok = true;
            for (int t = first; ok && t < tiles; t += step) {
                int m_tile, n_tile;
                pair_tile_at(P, t, m_tile, n_tile);
                const int m0 = m_tile * 256 + rank * 128, n0 = n_tile * 256 + rank * 64;
                for (int b = 0; b < P.kblocks; ++b) {
                    if (!mbar_wait_warp(&empty[s], ph ^ 1u, abort_flag, P.err)) {
                        ok = false;
                        break;
                    }
                    if (elect_one()) {
                        uint8_t* stage = smem + s * STAGE_BYTES;
                        mbar_arrive_expect_tx(&full[s], STAGE_BYTES);
                        tma_load_2d(stage, &map_x, &full[s], b * BK, m0);
                        tma_load_2d(stage + A_BYTES, &map_w, &full[s], b * BK, n0);
                        tma_load_2d(stage + A_BYTES + B_HALF, &map_w, &full[s], b * BK, n0 + 128);
                    }
                    __syncwarp();
                    if (++s == STAGES) {
                        s = 0;
                        ph ^= 1u;
                    }
                }
            }
        } else if (warp <= 2 && rank == 0) {
            const int half = warp - 1;
            const uint32_t idesc = make_idesc(kDFmtF32, kFmtE4M3, kFmtE4M3, 0, 0, 256, 128);
            const uint64_t a_desc0 = make_smem_desc_sw128(smem_u32(smem), 16, 1024);
            const uint64_t b_desc0 = make_smem_desc_sw128(smem_u32(smem) + A_BYTES + half * B_HALF, 16, 1024);
            const int blocks = first < tiles ? ((tiles - first + step - 1) / step) * P.kblocks : 0;
            uint32_t s = 0, ph = 0;
            for (int g = 0; g < blocks; ++g) {   // k blocks of all this pair's tiles
                const uint32_t buf = g & 1u, aph = (g >> 1) & 1u;
                // the stage first: it is there long before the accumulator, whose signal should find nothing left to wait for
                if (!mbar_wait_warp(&full[s], ph, abort_flag, P.err)) break;
                const uint32_t d = tmem_base + half * 256 + buf * 128;
                const uint32_t off = s * (STAGE_BYTES >> 4);   // descriptors count 16-byte units
                const uint64_t a_desc = a_desc0 + off, b_desc = b_desc0 + off;
                if (!mbar_wait_warp(&acc_empty[2 * half + buf], aph ^ 1u, abort_flag, P.err)) break;
                tc_fence_after_sync();
                if (elect_one()) {
#pragma unroll
                    for (int j = 0; j < BK / 32; ++j) {
                        mma_f8_ss_pair(d, a_desc + 2 * j, b_desc + 2 * j, idesc, j > 0 ? 1u : 0u);
                    }
                    mma_commit_pair(&acc_full[2 * half + buf]);
                    mma_commit_pair(&empty[s]);
                }
                __syncwarp();
                if (++s == STAGES) {
                    s = 0;
                    ph ^= 1u;
                }
            }
        } else if (warp == 3) {
            float* dst0 = reinterpret_cast<float*>(smem + OFF_SCALE);
            uint32_t sg = 0;
            bool ok = true;
            for (int t = first; ok && t < tiles; t += step) {
                int m_tile, n_tile;
                pair_tile_at(P, t, m_tile, n_tile);
                const int m0 = m_tile * 256 + rank * 128;
                for (int b = 0; b < P.kblocks; b += 8, ++sg) {
                    ok = mbar_wait_warp(&sc_empty[sg & 1u], ((sg >> 1) & 1u) ^ 1u, abort_flag, P.err);
                    if (!ok) break;
                    const int at = b + (lane & 7) < P.kblocks ? b + (lane & 7) : P.kblocks - 1;
                    copy_scales<0, 128>(P, dst0 + (sg & 1u) * SCALE_WORDS, m0, at, 2 * n_tile, 2, lane);
                    copies_wait();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sc_full[sg & 1u]);
                    if (b == 0 && P.gate != nullptr) prefetch_residual(P, m0, n_tile * 256, lane);
                }
            }
        } else if (warp == 1) {
            const int blocks = first < tiles ? ((tiles - first + step - 1) / step) * P.kblocks : 0;
            uint32_t s = 0, ph = 0;
            for (int g = 0; g < blocks; ++g) {
                if (!mbar_wait_warp(&full[s], ph, abort_flag, P.err)) break;
                if (elect_one()) mbar_arrive_leader(&full[s]);
                __syncwarp();
                if (++s == STAGES) {
                    s = 0;
                    ph ^= 1u;
                }
            }
        }
    }
    tc_fence_before_sync();
    __syncthreads();
    if (*abort_flag) {
        for (int i = 0; i < 200; ++i) __nanosleep(1000);   // let copies and MMAs in flight land
        __syncthreads();
    }
    cluster_sync_all();     // neither CTA leaves while the other may signal it or the pair's MMAs read its memory
    if (warp == 1) {
        tc_fence_after_sync();
        tmem_dealloc_pair(tmem_base, 512);
    }
}

// ----------------------------------------------------------- few rows: 128 features x NT tokens, k split over a cluster
// Bound: HBM, the weights read once (2 x 5120 x 30720 27.5 us, 5.7 TB/s, 0.87 of the copy rate).  The roles are turned round:
// features lie in the 128 lanes of tensor memory, tokens in its columns, so that a tile wastes nothing on tokens that are not
// there; a column's scale is then one number per token and block, laid out by warp 2 for eight blocks at a time.  Two CTAs
// share an SM and keep 160 KB of weights under way there.  Where the tiles alone leave SMs idle, a cluster of up to eight
// CTAs takes a tile, each a run of its k blocks; the partial sums meet in shared memory and are added in the order of the
// parts.
namespace few {
constexpr int THREADS = 256;                 // warp 0 TMA, 1 MMA, 2 scales, 4-7 promotion; all add up and store
constexpr int W_BYTES = 128 * BK;
template <int NT>
struct Plan {
    static constexpr int STAGES = NT >= 64 ? 4 : 5;
    static constexpr int STAGE_BYTES = W_BYTES + NT * BK;
    static constexpr int OFF_SCALE = STAGES * STAGE_BYTES;          // [2 groups][8 blocks][NT + 4]
    static constexpr int OFF_BAR = OFF_SCALE + 2 * 8 * (NT + 4) * 4;
    static constexpr int SMEM_BYTES = OFF_BAR + 256 + 1024;
    static constexpr int BUFS = 4;                                  // accumulators under way
    static constexpr int TMEM_COLS = BUFS * NT;                     // 64, 128 or 256
    static_assert(NT * 128 * 4 <= OFF_SCALE, "partial sums take the stages' place");
    static_assert(SMEM_BYTES <= 113 * 1024, "two CTAs an SM");
};
}  // namespace few

template <int NT>
__global__ void __launch_bounds__(few::THREADS, 2)
fp8_few_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
               const __grid_constant__ Params P, const int parts) {
    using namespace few;
    using L = Plan<NT>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::OFF_BAR);   // [STAGES]
    uint64_t* empty = full + L::STAGES;                                // [STAGES]
    uint64_t* acc_full = empty + L::STAGES;                            // [BUFS]
    uint64_t* acc_empty = acc_full + L::BUFS;                          // [BUFS]
    uint64_t* sc_full = acc_empty + L::BUFS;                           // [2]
    uint64_t* sc_empty = sc_full + 2;                                  // [2]
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sc_empty + 2);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    float* scales = reinterpret_cast<float*>(smem + L::OFF_SCALE);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int tile = blockIdx.x / parts, part = blockIdx.x - tile * parts;   // a cluster is `parts` neighbours: its rank
    const int n_tile = tile / P.m_tiles, m_tile = tile - n_tile * P.m_tiles;
    const int n0 = n_tile * 128, m0 = m_tile * NT;
    const int b_first = static_cast<int>(static_cast<long long>(P.kblocks) * part / parts);
    const int blocks = static_cast<int>(static_cast<long long>(P.kblocks) * (part + 1) / parts) - b_first;

    if (threadIdx.x == 0) {
        for (int i = 0; i < L::STAGES; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < L::BUFS; ++i) {
            mbar_init(&acc_full[i], 1);
            mbar_init(&acc_empty[i], 4);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sc_full[i], 1);
            mbar_init(&sc_empty[i], 4);
        }
        *abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, L::TMEM_COLS);
        tmem_relinquish();
    }
    if (warp == 0 && lane == 0) {
        tma_prefetch_desc(&map_x);
        tma_prefetch_desc(&map_w);
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem_base = *tmem_slot;
    float acc[NT];

    if (warp == 0) {
        uint32_t s = 0, ph = 0;
        if (elect_one()) {
            for (int b = 0; b < blocks; ++b) {
                if (!mbar_wait(&empty[s], ph ^ 1u, abort_flag, P.err)) break;
                uint8_t* stage = smem + s * L::STAGE_BYTES;
                mbar_arrive_expect_tx(&full[s], L::STAGE_BYTES);
                tma_load_2d(stage, &map_w, &full[s], (b_first + b) * BK, n0);
                tma_load_2d(stage + W_BYTES, &map_x, &full[s], (b_first + b) * BK, m0);
                if (++s == L::STAGES) {
                    s = 0;
                    ph ^= 1u;
                }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        const uint32_t idesc = make_idesc(kDFmtF32, kFmtE4M3, kFmtE4M3, 0, 0, 128, NT);
        uint32_t s = 0, ph = 0;
        if (elect_one()) {
            for (int b = 0; b < blocks; ++b) {
                const uint32_t buf = b % L::BUFS, aph = (b / L::BUFS) & 1u;
                if (!mbar_wait(&full[s], ph, abort_flag, P.err)) break;
                if (!mbar_wait(&acc_empty[buf], aph ^ 1u, abort_flag, P.err)) break;
                tc_fence_after_sync();
                const uint32_t a_addr = smem_u32(smem + s * L::STAGE_BYTES), b_addr = a_addr + W_BYTES;
#pragma unroll
                for (int j = 0; j < BK / 32; ++j) {
                    mma_f8_ss(tmem_base + buf * NT, make_smem_desc_sw128(a_addr + j * 32, 16, 1024),
                              make_smem_desc_sw128(b_addr + j * 32, 16, 1024), idesc, j > 0 ? 1u : 0u);
                }
                mma_commit(&acc_full[buf]);
                mma_commit(&empty[s]);
                if (++s == L::STAGES) {
                    s = 0;
                    ph ^= 1u;
                }
            }
        }
        __syncwarp();
    } else if (warp == 2) {
        const float* ws = P.ws + static_cast<long long>(n_tile) * P.ld_ws;
        for (int b = 0; b < blocks; b += 8) {
            const int g = b >> 3;
            if (!mbar_wait_warp(&sc_empty[g & 1], ((g >> 1) & 1) ^ 1u, abort_flag, P.err)) break;
            float* dst = scales + (g & 1) * 8 * (NT + 4) + (lane & 7) * (NT + 4) + (lane >> 3);
            const int at = b_first + (b + (lane & 7) < blocks ? b + (lane & 7) : blocks - 1);
            const float w = __ldg(ws + at);
#pragma unroll
            for (int i = 0; i < NT / 4; ++i) {   // four tokens of eight blocks a load; tokens past the end follow the last
                const int m = m0 + 4 * i + (lane >> 3) < P.M ? m0 + 4 * i + (lane >> 3) : P.M - 1;
                dst[4 * i] = w * __ldg(P.xs + m * P.ld_xs + at);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&sc_full[g & 1]);
        }
    } else if (warp >= 4) {
        const uint32_t taddr = tmem_base + (static_cast<uint32_t>((warp & 3) * 32) << 16);
#pragma unroll
        for (int i = 0; i < NT; ++i) acc[i] = 0.0f;
        for (int b = 0; b < blocks; ++b) {
            const uint32_t buf = b % L::BUFS, aph = (b / L::BUFS) & 1u;
            const int g = b >> 3;
            bool ok = true;
            if ((b & 7) == 0) ok = mbar_wait_warp(&sc_full[g & 1], (g >> 1) & 1, abort_flag, P.err);
            ok = ok && mbar_wait_warp(&acc_full[buf], aph, abort_flag, P.err);
            if (!ok) break;
            tc_fence_after_sync();
            const float* sc = scales + ((g & 1) * 8 + (b & 7)) * (NT + 4);
#pragma unroll
            for (int c = 0; c < NT; c += 16) {
                uint32_t r[16];
                tmem_ld_32x32b_x16(taddr + buf * NT + c, r);
                float4 f[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) f[i] = *reinterpret_cast<const float4*>(sc + c + 4 * i);
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    acc[c + 4 * i] = fmaf(__uint_as_float(r[4 * i]), f[i].x, acc[c + 4 * i]);
                    acc[c + 4 * i + 1] = fmaf(__uint_as_float(r[4 * i + 1]), f[i].y, acc[c + 4 * i + 1]);
                    acc[c + 4 * i + 2] = fmaf(__uint_as_float(r[4 * i + 2]), f[i].z, acc[c + 4 * i + 2]);
                    acc[c + 4 * i + 3] = fmaf(__uint_as_float(r[4 * i + 3]), f[i].w, acc[c + 4 * i + 3]);
                }
            }
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&acc_empty[buf]);
                if ((b & 7) == 7) mbar_arrive(&sc_empty[g & 1]);
            }
        }
    }
    tc_fence_before_sync();
    __syncthreads();            // every block has been read: the copies and MMAs of this CTA are done
    const bool bad = *abort_flag != 0;
    if (bad) {
        for (int i = 0; i < 200; ++i) __nanosleep(1000);   // let copies and MMAs in flight land
        __syncthreads();
    }
    float* sums = reinterpret_cast<float*>(smem);   // [NT][128]
    if (warp >= 4) {
        const int f = (warp & 3) * 32 + lane;
#pragma unroll
        for (int t = 0; t < NT; ++t) sums[t * 128 + f] = acc[t];
    }
    finish_tokens(P, sums, 128, NT, m0, n0, part, parts, warp, THREADS / 32, lane, bad);
    if (warp == 1) {
        tc_fence_after_sync();
        tmem_dealloc(tmem_base, L::TMEM_COLS);
    }
}

// Sets a kernel's dynamic shared memory once per device (twice where two threads make the first call at once).
using PerDevice = std::atomic<bool>[64];
template <typename K>
static edb200_status_t allow_smem(K kern, int bytes, PerDevice& done) {
    int dev = -1;
    EDB_TRY(check_cuda(cudaGetDevice(&dev), "cudaGetDevice"));
    const bool counted = dev >= 0 && dev < 64;
    if (counted && done[dev].load(std::memory_order_relaxed)) return EDB200_OK;
    EDB_TRY(check_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes), "cudaFuncSetAttribute(mul_mat_fp8)"));
    if (counted) done[dev].store(true, std::memory_order_relaxed);
    return EDB200_OK;
}

// Operand rows of k bytes as boxes of 128 bytes x box_rows (a single row's pitch may be anything).
static edb200_status_t operand_map(CUtensorMap* map, const void* base, int64_t k, int64_t rows, int64_t ld, uint32_t box_rows) {
    const uint64_t pitch = rows > 1 ? (uint64_t)ld : ((uint64_t)k + 15) / 16 * 16;
    return make_tmap_2d(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, base, (uint64_t)k, (uint64_t)rows, pitch, BK, box_rows,
                        CU_TENSOR_MAP_SWIZZLE_128B);
}

// Launches `tiles` clusters of `parts` CTAs.
template <typename K>
static edb200_status_t launch_parts(K kern, int64_t tiles, int parts, int threads, int smem, const CUtensorMap& map_x,
                                    const CUtensorMap& map_w, const Params& P, cudaStream_t s) {
    if (tiles * parts > 0x7fffffff) return fail(EDB200_ERR_UNSUPPORTED, "mul_mat_fp8: too many output tiles");
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3(static_cast<unsigned>(tiles * parts));
    cfg.blockDim = dim3(static_cast<unsigned>(threads));
    cfg.dynamicSmemBytes = static_cast<size_t>(smem);
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = static_cast<unsigned>(parts);
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    EDB_TRY(check_cuda(cudaLaunchKernelEx(&cfg, kern, map_x, map_w, P, parts), "mul_mat_fp8 launch"));
    count_launch();
    return EDB200_OK;
}

static edb200_status_t launch_tile(const edb200_fp8_weight_t& w, const void* x, int64_t m, int64_t ldx, int parts, Params& P,
                                   cudaStream_t s) {
    CUtensorMap map_x, map_w;
    EDB_TRY(operand_map(&map_x, x, w.k, m, ldx, 128));
    EDB_TRY(operand_map(&map_w, w.w, w.k, w.n, w.ldw, 128));
    static PerDevice done = {};
    EDB_TRY(allow_smem(fp8_tile_kernel, tile::SMEM_BYTES, done));
    P.m_tiles = static_cast<int>((m + 127) / 128);
    const int64_t tiles = (int64_t)P.m_tiles * ((w.n + 127) / 128);
    return launch_parts(fp8_tile_kernel, tiles, parts, tile::THREADS, tile::SMEM_BYTES, map_x, map_w, P, s);
}

template <int NT>
static edb200_status_t launch_few(const edb200_fp8_weight_t& w, const void* x, int64_t m, int64_t ldx, int parts, Params& P,
                                  cudaStream_t s) {
    CUtensorMap map_x, map_w;
    EDB_TRY(operand_map(&map_x, x, w.k, m, ldx, NT));
    EDB_TRY(operand_map(&map_w, w.w, w.k, w.n, w.ldw, 128));
    static PerDevice done = {};
    EDB_TRY(allow_smem(fp8_few_kernel<NT>, few::Plan<NT>::SMEM_BYTES, done));
    P.m_tiles = static_cast<int>((m + NT - 1) / NT);
    const int64_t tiles = (int64_t)P.m_tiles * ((w.n + 127) / 128);
    return launch_parts(fp8_few_kernel<NT>, tiles, parts, few::THREADS, few::Plan<NT>::SMEM_BYTES, map_x, map_w, P, s);
}

static edb200_status_t launch_pair(const edb200_fp8_weight_t& w, const void* x, int64_t m, int64_t ldx, int resident, Params& P,
                                   cudaStream_t s) {
    CUtensorMap map_x, map_w;
    EDB_TRY(operand_map(&map_x, x, w.k, m, ldx, 128));
    EDB_TRY(operand_map(&map_w, w.w, w.k, w.n, w.ldw, 64));
    static PerDevice done = {};
    EDB_TRY(allow_smem(fp8_pair_kernel, pair::SMEM_BYTES, done));
    P.m_tiles = static_cast<int>((m + 255) / 256);
    P.n_tiles = static_cast<int>((w.n + 255) / 256);
    // feature tiles walked together: their weights, read again for every token tile, stay within about a third of L2
    const int64_t ch = (44ll << 20) / (256 * w.k);
    P.chunk = static_cast<int>(ch < 1 ? 1 : ch < P.n_tiles ? ch : P.n_tiles);
    const int64_t tiles = (int64_t)P.m_tiles * P.n_tiles;
    if (tiles > 0x3fffffff) return fail(EDB200_ERR_UNSUPPORTED, "mul_mat_fp8: too many output tiles");
    const unsigned grid = 2u * static_cast<unsigned>(tiles < resident ? tiles : resident);
    fp8_pair_kernel<<<grid, pair::THREADS, pair::SMEM_BYTES, s>>>(map_x, map_w, P);
    count_launch();
    return check_cuda(cudaGetLastError(), "mul_mat_fp8 launch");
}

// Clusters of `parts` (1, 2, 4 or 8) CTAs, one an SM, that are resident at once: 148, 74, 33 and 15 here, fewer than SMs / parts
// because a cluster lies within one group of SMs.
static int clusters_resident(int parts) {
    static std::atomic<int> known[4] = {};
    const int i = parts == 1 ? 0 : parts == 2 ? 1 : parts == 4 ? 2 : 3;
    int n = known[i].load(std::memory_order_relaxed);
    if (n != 0) return n;
    const int most = sm_count() / parts;
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3(static_cast<unsigned>(most * parts));
    cfg.blockDim = dim3(tile::THREADS);
    cfg.dynamicSmemBytes = tile::SMEM_BYTES;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = static_cast<unsigned>(parts);
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    static PerDevice done = {};
    if (allow_smem(fp8_tile_kernel, tile::SMEM_BYTES, done) != EDB200_OK ||
        cudaOccupancyMaxActiveClusters(&n, fp8_tile_kernel, &cfg) != cudaSuccess || n <= 0 || n > most) {
        (void)cudaGetLastError();
        n = most;
    }
    known[i].store(n, std::memory_order_relaxed);
    return n;
}

// Which kernel takes a product, and into how many parts its k blocks are cut: the one whose time by the sums below is least.
// They count waves of resident CTAs; the unit is the tile kernel's block (0.31 us), and the numbers were fitted to 878 timed
// cases (m 1 to 640, n 256 to 30720, k 512 to 13824; activations and outputs at six sizes).  There the choice costs 0.2 % over
// the fastest on average and 11 % at worst, at 500 drawn sizes and epilogues besides 0.7 and 14 % (a fixed 37 pairs and parts by
// the number of SMs: 6.5 and 76 %).
// m x k x n, us:                     few rows          tiles             pairs
//   300 x 5120 x 5120 to f16          30.0              18.4              25.4
//    96 x 5120 x 10240 to f16         29.7              18.3              25.6   (tiles 75 % full, pairs 37)
//   512 x 5120 x 7168 to f16                            35.3, two waves   26.5, one wave
//   192 x 1536 x 768 to f16           6.7 in 4 parts    7.6 in 4 parts    13.1
//   154 x 1536 x 6144, GELU to e4m3   12.4 in 2 parts   13.7              15.7
//     1 x 512 x 13824 to f16          4.6, in two 6.1   6.1
enum Kernel { FEW, TILE, PAIR };
struct Choice {
    Kernel kernel;
    int parts;
};
static Choice choose(int64_t m, int64_t n, int64_t blocks, const edb200_epilogue_t& ep) {
    const auto up = [](int64_t a, int64_t b) { return (a + b - 1) / b; };
    const auto waves = [&](int64_t tiles, int64_t resident) { return static_cast<double>(up(tiles, resident)); };
    const bool act = ep.act != EDB200_ACT_NONE, gated = ep.gate != nullptr;
    const bool f8 = ep.out_dtype == EDB200_TYPE_F8_E4M3, f32 = ep.out_dtype == EDB200_TYPE_F32;
    Choice best = {FEW, 1};
    double least = 1e300;
    const auto offer = [&](Kernel kernel, int parts, double time) {
        if (time < least) {
            least = time;
            best = {kernel, parts};
        }
    };
    const int64_t rows = m <= 16 ? 16 : m <= 32 ? 32 : 64;                // of a few-row tile
    const int64_t few = up(m, rows) * up(n, 128), tiles = up(m, 128) * up(n, 128), pairs = up(m, 256) * up(n, 256);
    const double u = static_cast<double>(rows) / 64.0, full = m < 128 ? static_cast<double>(m) / 128.0 : 1.0;
    // what a tile's end takes, over f16 without activation
    const double few_end = u * ((act ? 3.5 : 0.0) + (gated ? 6.0 : 0.0) + (f8 ? 7.0 : 0.0));
    const double tile_end = full * (4.0 + (act ? 5.0 : 0.0) + (gated ? 7.0 : 0.0) + (f8 ? 9.0 : 0.0));
    const double pair_end = (act ? 9.0 : 0.0) + (gated ? 14.0 : f32 ? 7.0 : 0.0);
    for (int parts = 1; parts <= 8 && (parts == 1 || blocks >= 2 * parts); parts *= 2) {   // a part of two blocks at least
        const int64_t one = clusters_resident(parts);                      // with one CTA an SM; the few-row kernel has two,
        const double b = static_cast<double>(up(blocks, parts)), shared = few > one ? 1.7 : 1.0;   // each the slower
        offer(FEW, parts, waves(few, 2 * one) * ((parts == 1 ? 12.0 : 15.0 + 0.25 * parts) + 3.0 * u + shared * (0.55 + 0.75 * u) * b + few_end / parts));
        // up to 64 rows in one wave only: beyond it the few-row kernel's two CTAs an SM keep more of the weights under way
        if (m > 64 || (m > 32 && tiles <= one)) {
            offer(TILE, parts, 4.0 + waves(tiles, one) * (b + 10.0 + (parts == 1 ? 0.0 : 6.0 + 0.25 * parts) + tile_end / parts));
        }
    }
    if (m > 64) offer(PAIR, 1, 14.0 + waves(pairs, clusters_resident(2)) * (1.38 * static_cast<double>(blocks) + 13.0 + pair_end));
    return best;
}

}  // namespace f8g
}  // namespace edb

extern "C" edb200_status_t edb200_mul_mat_fp8(const edb200_fp8_weight_t* w, const void* x, const float* x_scale, int64_t m,
                                              int64_t ldx, int64_t ld_xs, const edb200_epilogue_t* ep, float* out_scale,
                                              int64_t ld_out_scale, void* stream) {
    using namespace edb;
    if (w == nullptr || ep == nullptr) return fail(EDB200_ERR_INVALID, "mul_mat_fp8: null argument");
    const int64_t big = 0x7fffff00ll;
    if (m < 0 || m > big || w->n < 1 || w->n > big || w->k < 1 || w->k > big) {
        return fail(EDB200_ERR_INVALID, "mul_mat_fp8: m >= 0, n >= 1 and k >= 1, each below 2^31 - 256");
    }
    if (ep->split_n != 0 || ep->pack != nullptr || ep->split_k != EDB200_SPLIT_K_NEVER) {
        return fail(EDB200_ERR_UNSUPPORTED, "mul_mat_fp8: split_n, split_k and pack belong to mul_mat_q");
    }
    if (ep->act < EDB200_ACT_NONE || ep->act > EDB200_ACT_GELU_ERF) return fail(EDB200_ERR_INVALID, "mul_mat_fp8: bad act");
    const int dt = ep->out_dtype;
    const bool f8 = dt == EDB200_TYPE_F8_E4M3;
    if (dt != EDB200_TYPE_F32 && dt != EDB200_TYPE_F16 && dt != EDB200_TYPE_BF16 && !f8) {
        return fail(EDB200_ERR_INVALID, "mul_mat_fp8: out_dtype must be f32, f16, bf16 or e4m3");
    }
    if (m == 0) return EDB200_OK;
    if (w->w == nullptr || w->scale == nullptr || x == nullptr || x_scale == nullptr || ep->out == nullptr) {
        return fail(EDB200_ERR_INVALID, "mul_mat_fp8: null argument");
    }
    const int64_t kb = (w->k + 127) / 128, nb = (w->n + 127) / 128;
    auto at = [](const void* q) { return reinterpret_cast<uintptr_t>(q); };
    // a single row's stride is not used
    if ((m > 1 && (ldx < w->k || ldx % 16)) || (at(x) & 15u) || (w->n > 1 && (w->ldw < w->k || w->ldw % 16)) || (at(w->w) & 15u)) {
        return fail(EDB200_ERR_INVALID, "mul_mat_fp8: rows of x and w must be 16-byte aligned and hold k values");
    }
    if ((m > 1 && ld_xs < kb) || (nb > 1 && w->ld_scale < kb) || ((at(x_scale) | at(w->scale)) & 3u)) {
        return fail(EDB200_ERR_INVALID, "mul_mat_fp8: scale rows must be 4-byte aligned and hold ceil(k / 128) values");
    }
    const int esz = dt == EDB200_TYPE_F32 ? 4 : f8 ? 1 : 2;
    if ((m > 1 && (ep->ldo < w->n || (ep->ldo * esz) % 16)) || (at(ep->out) & 15u)) {
        return fail(EDB200_ERR_INVALID, "mul_mat_fp8: out rows must be 16-byte aligned and ldo >= n");
    }
    if ((at(ep->bias) | at(ep->gate)) & 3u) return fail(EDB200_ERR_INVALID, "mul_mat_fp8: bias and gate must be 4-byte aligned");
    if (ep->gate != nullptr && (dt != EDB200_TYPE_F32 || ep->residual == nullptr || (m > 1 && (ep->ld_res < w->n || ep->ld_res % 4)) ||
                                (at(ep->residual) & 15u))) {
        return fail(EDB200_ERR_INVALID, "mul_mat_fp8: gated residual needs f32 out and residual rows of n values, 16-byte aligned");
    }
    if (ep->gate != nullptr && ep->out == ep->residual && m > 1 && ep->ldo != ep->ld_res) {
        return fail(EDB200_ERR_INVALID, "mul_mat_fp8: out in the residual's place needs the same stride");
    }
    if (f8 != (out_scale != nullptr) || (f8 && ((m > 1 && ld_out_scale < nb) || (at(out_scale) & 3u)))) {
        return fail(EDB200_ERR_INVALID, "mul_mat_fp8: e4m3 out, and only it, needs out_scale with ceil(n / 128) columns");
    }
    int* err = device_error_word();
    if (err == nullptr) return fail(EDB200_ERR_CUDA, "mul_mat_fp8: no CUDA device");
    f8g::Params P;
    memset(&P, 0, sizeof(P));
    P.xs = x_scale;
    P.ws = w->scale;
    P.ld_xs = ld_xs;
    P.ld_ws = w->ld_scale;
    P.bias = ep->bias;
    P.residual = ep->residual;
    P.gate = ep->gate;
    P.out = ep->out;
    P.out_scale = out_scale;
    P.ldo = ep->ldo;
    P.ld_res = ep->ld_res;
    P.ld_os = ld_out_scale;
    P.M = static_cast<int>(m);
    P.N = static_cast<int>(w->n);
    P.kblocks = static_cast<int>(kb);
    P.act = ep->act;
    P.out_dtype = dt;
    P.err = err;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    ProfScope prof(s, PROF_GEMM, 2.0 * (double)m * (double)w->n * (double)w->k,
                   (double)w->n * (double)w->k + (double)m * (double)w->k + (double)m * (double)w->n * esz);
    const f8g::Choice c = f8g::choose(m, w->n, kb, *ep);
    switch (c.kernel) {
        case f8g::PAIR: return f8g::launch_pair(*w, x, m, ldx, f8g::clusters_resident(2), P, s);
        case f8g::TILE: return f8g::launch_tile(*w, x, m, ldx, c.parts, P, s);
        default: break;
    }
    if (m <= 16) return f8g::launch_few<16>(*w, x, m, ldx, c.parts, P, s);
    if (m <= 32) return f8g::launch_few<32>(*w, x, m, ldx, c.parts, P, s);
    return f8g::launch_few<64>(*w, x, m, ldx, c.parts, P, s);
}
