// Rotary positions from position numbers (edb200_rope_apply): channels pair as neighbours or as halves, over the whole
// head or its first channels, one to four position axes, frequencies stretched for lengths beyond the trained one.
//
//   (a, b) -> m (a cos t - b sin t, a sin t + b cos t),   t = position * frequency
//
// Bound: HBM, q and k read and written once.  The angle is a product in 64 bits of which only the fraction of a turn
// goes on in 32 bits: t / 2 pi = position * (frequency / 2 pi) is off by 2^-53 of itself, 2.4e-7 rad at the largest
// 32-bit position and below f32 rounding for positions under 10^8.  A CTA makes the cosines and sines of its few
// tokens once, in shared memory, for all heads of q and k; then every thread turns 16-byte pieces.  Two pieces of a thread
// under way at once cost registers and were slower (275 against 210 us).
// Measured: 32760 tokens x 80 heads x 128 bf16 in halves 210 to 219 us (6.1 to 6.4 TB/s, 0.93 to 0.97 of the copy rate),
// neighbours 239 to 242 us (5.6);
// 154 tokens x 48 heads x 64 3.6 us.
#include "edb200_internal.h"
#include "edb200_fp8.cuh"

#include <cmath>
#include <cstring>
#include <new>

struct edb200_rope {
    int n_axes = 0;
    int pairs = 0;              // turned pairs of a head
    int layout = 0;
    float mul = 1.0f;           // multiplier of the turned channels
    double turns[128];          // turns per position, pair by pair
    unsigned char axis[128];
};

namespace edb {
namespace rope {

constexpr int THREADS = 256;
constexpr int TABLE = 1024;     // pairs of all tokens of a CTA: 8 KB of cosines and sines

struct Tensor {
    const void* in;
    void* out;
    long long in_token, in_head, out_token, out_head;
    int heads;
};
struct Params {
    Tensor t[2];
    const int32_t* positions;
    long long tokens;
    int n_axes, pairs, d_head, tokens_per_cta;
    int units_head;             // pieces of a head: turned ones first, then those that pass through
    int units_turned;
    uint32_t inv_token, inv_head;   // 2^32 / (pieces of a token, of a head), rounded up
    float mul;
    float sign;                 // -1 turns back
    double turns[128];
    unsigned char axis[128];
};

// W values of T moved as one access of W * sizeof(T) bytes (16, or one element).
template <typename T, int W>
struct Piece {
    T v[W];
};
template <typename T, int W>
__device__ __forceinline__ void load_piece(const T* p, float (&v)[W]) {
    if constexpr (W == 1) {
        v[0] = widen<T>(*p);
    } else {
        const uint4 u = *reinterpret_cast<const uint4*>(p);
        Piece<T, W> x;
        memcpy(&x, &u, 16);
#pragma unroll
        for (int i = 0; i < W; ++i) v[i] = widen<T>(x.v[i]);
    }
}
template <typename T, int W>
__device__ __forceinline__ void store_piece(T* p, const float (&v)[W]) {
    if constexpr (W == 1) {
        *p = narrow<T>(v[0]);
    } else {
        Piece<T, W> x;
#pragma unroll
        for (int i = 0; i < W; ++i) x.v[i] = narrow<T>(v[i]);
        uint4 u;
        memcpy(&u, &x, 16);
        *reinterpret_cast<uint4*>(p) = u;
    }
}

// n / d by the product with 2^32 / d rounded up: exact while n d < 2^32, which the host sees to.
__device__ __forceinline__ int divided(int n, uint32_t inverse, int d) { return d == 1 ? n : static_cast<int>(__umulhi(static_cast<uint32_t>(n), inverse)); }

template <int N>
__device__ __forceinline__ void table(const float* p, float (&v)[N]) {   // N consecutive entries at a multiple of N
    if constexpr (N >= 4) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const float4 f = *reinterpret_cast<const float4*>(p + i);
            v[i] = f.x, v[i + 1] = f.y, v[i + 2] = f.z, v[i + 3] = f.w;
        }
    } else if constexpr (N == 2) {
        const float2 f = *reinterpret_cast<const float2*>(p);
        v[0] = f.x, v[1] = f.y;
    } else {
        v[0] = *p;
    }
}

// One piece on its way: where it comes from and goes to, its values.
template <typename T, int W, bool HALF>
struct Unit {
    static constexpr int N = HALF ? W : (W == 1 ? 1 : W / 2);   // pairs
    static constexpr bool TWO = HALF || W == 1;                 // a pair's members come from two places
    const T* in;
    T* out;
    int pair, at_a, at_b;   // pair < 0: passes through
    float a[W], b[TWO ? W : 1];

    __device__ __forceinline__ void find(const Params& P, long long t0, int i, int per_token, int heads0) {
        const int t = divided(i, P.inv_token, per_token);
        const int r = i - t * per_token;
        int head = divided(r, P.inv_head, P.units_head);
        const int u = r - head * P.units_head;
        const Tensor& x = P.t[head >= heads0 ? 1 : 0];
        if (head >= heads0) head -= heads0;
        in = static_cast<const T*>(x.in) + (t0 + t) * x.in_token + head * x.in_head;
        out = static_cast<T*>(x.out) + (t0 + t) * x.out_token + head * x.out_head;
        if (u < P.units_turned) {
            const int p = u * N;
            pair = t * P.pairs + p;
            at_a = HALF ? p : 2 * p;
            at_b = HALF ? p + P.pairs : 2 * p + 1;
        } else {
            pair = -1;
            at_a = 2 * P.pairs + (u - P.units_turned) * W;
        }
    }
    __device__ __forceinline__ void load() {
        if (pair < 0 && in == out) return;   // in place already
        load_piece<T, W>(in + at_a, a);
        if (TWO && pair >= 0) load_piece<T, W>(in + at_b, reinterpret_cast<float(&)[W]>(b[0]));
    }
    __device__ __forceinline__ void turn(const float* cs, const float* sn) {
        if (pair < 0) {
            if (in != out) store_piece<T, W>(out + at_a, a);
            return;
        }
        float c[N], s[N], ya[W];
        table<N>(cs + pair, c);
        table<N>(sn + pair, s);
        if constexpr (TWO) {
            float yb[W];
#pragma unroll
            for (int e = 0; e < W; ++e) {
                ya[e] = fmaf(a[e], c[e], -__fmul_rn(b[e], s[e]));
                yb[e] = fmaf(a[e], s[e], __fmul_rn(b[e], c[e]));
            }
            store_piece<T, W>(out + at_a, ya);
            store_piece<T, W>(out + at_b, yb);
        } else {
#pragma unroll
            for (int e = 0; e < N; ++e) {
                ya[2 * e] = fmaf(a[2 * e], c[e], -__fmul_rn(a[2 * e + 1], s[e]));
                ya[2 * e + 1] = fmaf(a[2 * e], s[e], __fmul_rn(a[2 * e + 1], c[e]));
            }
            store_piece<T, W>(out + at_a, ya);
        }
    }
};

// W: values of a piece (16 bytes' worth, or 1).  A turned unit of the halves layout is two pieces, half a turned width
// apart; of the interleaved layout W values (one pair of single values where W is 1).
template <typename T, int W, bool HALF>
__global__ void __launch_bounds__(THREADS)
rope_kernel(const __grid_constant__ Params P) {
    __shared__ __align__(16) float cs[TABLE], sn[TABLE];
    const long long t0 = static_cast<long long>(blockIdx.x) * P.tokens_per_cta;
    const int nt = static_cast<int>(P.tokens - t0 < P.tokens_per_cta ? P.tokens - t0 : P.tokens_per_cta);
    for (int i = threadIdx.x; i < nt * P.pairs; i += THREADS) {
        const int t = i / P.pairs, p = i - t * P.pairs;
        const double pos = P.positions != nullptr ? static_cast<double>(P.positions[(t0 + t) * P.n_axes + P.axis[p]])
                                                  : static_cast<double>(t0 + t);
        const double turn = pos * P.turns[p];
        const float frac = static_cast<float>(turn - rint(turn));   // [-1/2, 1/2]
        float s, c;
        sincospif(2.0f * frac, &s, &c);
        cs[i] = c * P.mul;
        sn[i] = s * P.mul * P.sign;
    }
    const int heads0 = P.t[0].heads;
    const int per_token = (heads0 + P.t[1].heads) * P.units_head;
    const int total = nt * per_token;
    __syncthreads();
    for (int i = threadIdx.x; i < total; i += THREADS) {
        Unit<T, W, HALF> u;
        u.find(P, t0, i, per_token, heads0);
        u.load();
        u.turn(cs, sn);
    }
}

template <typename T>
static void launch(const Params& P, bool half, bool vec, unsigned grid, cudaStream_t s) {
    constexpr int W = 16 / sizeof(T);
    if (vec) {
        if (half) {
            rope_kernel<T, W, true><<<grid, THREADS, 0, s>>>(P);
        } else {
            rope_kernel<T, W, false><<<grid, THREADS, 0, s>>>(P);
        }
    } else if (half) {
        rope_kernel<T, 1, true><<<grid, THREADS, 0, s>>>(P);
    } else {
        rope_kernel<T, 1, false><<<grid, THREADS, 0, s>>>(P);
    }
}

static bool finite_positive(double v) { return v > 0.0 && v <= 1.7976931348623157e308; }

}  // namespace rope
}  // namespace edb

extern "C" {

edb200_status_t edb200_rope_create(const edb200_rope_config_t* cfg, edb200_rope_t** out) {
    using namespace edb;
    if (cfg == nullptr || out == nullptr) return fail(EDB200_ERR_INVALID, "rope_create: null argument");
    *out = nullptr;
    if (cfg->n_axes < 1 || cfg->n_axes > 4) return fail(EDB200_ERR_INVALID, "rope_create: n_axes must be 1..4");
    long long width = 0;
    for (int a = 0; a < cfg->n_axes; ++a) {
        if (cfg->axes_dim[a] < 2 || cfg->axes_dim[a] % 2) return fail(EDB200_ERR_INVALID, "rope_create: axes_dim must be even and positive");
        width += cfg->axes_dim[a];
    }
    if (width > 256) return fail(EDB200_ERR_UNSUPPORTED, "rope_create: at most 256 turned channels");
    if (cfg->layout != EDB200_ROPE_INTERLEAVED && cfg->layout != EDB200_ROPE_HALF) {
        return fail(EDB200_ERR_INVALID, "rope_create: layout must be EDB200_ROPE_INTERLEAVED or EDB200_ROPE_HALF");
    }
    if (cfg->scaling < EDB200_ROPE_SCALE_NONE || cfg->scaling > EDB200_ROPE_SCALE_YARN) {
        return fail(EDB200_ERR_INVALID, "rope_create: scaling must be EDB200_ROPE_SCALE_*");
    }
    if (!rope::finite_positive(cfg->theta) || cfg->theta <= 1.0) return fail(EDB200_ERR_INVALID, "rope_create: theta must be above 1");
    const bool yarn = cfg->scaling == EDB200_ROPE_SCALE_YARN;
    if (cfg->scaling != EDB200_ROPE_SCALE_NONE && (!rope::finite_positive(cfg->factor) || (yarn && cfg->factor < 1.0))) {
        return fail(EDB200_ERR_INVALID, "rope_create: factor must be positive (1 or more with YARN)");
    }
    const double fast = cfg->beta_fast == 0.0 ? 32.0 : cfg->beta_fast, slow = cfg->beta_slow == 0.0 ? 1.0 : cfg->beta_slow;
    if (yarn && (!rope::finite_positive(cfg->original_length) || !rope::finite_positive(fast) || !rope::finite_positive(slow) || fast < slow)) {
        return fail(EDB200_ERR_INVALID, "rope_create: YARN needs original_length > 0 and beta_fast >= beta_slow > 0");
    }
    if (cfg->attention_factor != 0.0 && !rope::finite_positive(cfg->attention_factor)) {
        return fail(EDB200_ERR_INVALID, "rope_create: attention_factor must be positive or 0");
    }
    edb200_rope* r = new (std::nothrow) edb200_rope();
    if (r == nullptr) return fail(EDB200_ERR_NOMEM, "rope_create: host allocation failed");
    const double two_pi = 6.283185307179586476925286766559;
    r->n_axes = cfg->n_axes;
    r->layout = cfg->layout;
    int n = 0;
    for (int a = 0; a < cfg->n_axes; ++a) {
        const int dim = cfg->axes_dim[a];
        double theta = cfg->theta;
        if (cfg->scaling == EDB200_ROPE_SCALE_NTK && dim > 2) theta *= std::pow(cfg->factor, (double)dim / (dim - 2));
        // YARN: places in the span of the frequencies that turn beta_fast and beta_slow times in original_length
        double low = 0.0, high = 0.0;
        if (yarn) {
            const auto place = [&](double turns) { return dim * std::log(cfg->original_length / (turns * two_pi)) / (2.0 * std::log(theta)); };
            low = std::fmax(std::floor(place(fast)), 0.0);
            high = std::fmin(std::ceil(place(slow)), (double)(dim - 1));
        }
        for (int j = 0; j < dim / 2; ++j) {
            double f = std::pow(theta, -2.0 * j / dim);
            if (cfg->scaling == EDB200_ROPE_SCALE_LINEAR) f /= cfg->factor;
            if (yarn) {
                const double ramp = std::fmin(std::fmax((j - low) / std::fmax(high - low, 1e-3), 0.0), 1.0);
                f = f / cfg->factor * ramp + f * (1.0 - ramp);
            }
            r->turns[n] = f / two_pi;
            r->axis[n] = static_cast<unsigned char>(a);
            ++n;
        }
    }
    r->pairs = n;
    r->mul = static_cast<float>(cfg->attention_factor != 0.0 ? cfg->attention_factor
                                                             : (yarn ? 0.1 * std::log(cfg->factor) + 1.0 : 1.0));
    *out = r;
    return EDB200_OK;
}

void edb200_rope_destroy(edb200_rope_t* r) { delete r; }

edb200_status_t edb200_rope_apply(const edb200_rope_t* r, const edb200_rope_tensor_t* q, const edb200_rope_tensor_t* k, int dtype,
                                  int d_head, int64_t tokens, const int32_t* positions, int inverse, void* stream) {
    using namespace edb;
    if (r == nullptr || q == nullptr) return fail(EDB200_ERR_INVALID, "rope_apply: null argument");
    if (dtype != EDB200_TYPE_F32 && dtype != EDB200_TYPE_F16 && dtype != EDB200_TYPE_BF16) {
        return fail(EDB200_ERR_INVALID, "rope_apply: dtype must be f32, f16 or bf16");
    }
    if (d_head < 2 * r->pairs || d_head > 65536) return fail(EDB200_ERR_INVALID, "rope_apply: d_head must hold the turned channels (and be at most 65536)");
    if (tokens < 0) return fail(EDB200_ERR_INVALID, "rope_apply: tokens must not be negative");
    if (tokens == 0) return EDB200_OK;
    const edb200_rope_tensor_t* ts[2] = {q, (k != nullptr && k->in != nullptr) ? k : nullptr};
    const int es = dtype == EDB200_TYPE_F32 ? 4 : 2, w = 16 / es;
    bool vec = d_head % w == 0 && (2 * r->pairs) % w == 0 && (r->layout != EDB200_ROPE_HALF || r->pairs % w == 0);
    rope::Params P;
    memset(&P, 0, sizeof(P));
    for (int i = 0; i < 2; ++i) {
        if (ts[i] == nullptr) continue;
        const edb200_rope_tensor_t& t = *ts[i];
        if (t.in == nullptr || t.out == nullptr || t.heads < 1 || t.heads > 65536) {
            return fail(EDB200_ERR_INVALID, "rope_apply: in and out must be set and heads be 1..65536");
        }
        if ((reinterpret_cast<uintptr_t>(t.in) | reinterpret_cast<uintptr_t>(t.out)) % es) {
            return fail(EDB200_ERR_INVALID, "rope_apply: in and out must be aligned to their elements");
        }
        const long long lim = 1ll << 46;   // token and head strides stay far inside 64-bit offsets
        const long long st[4] = {t.in_token, t.in_head, t.out_token, t.out_head};
        for (int j = 0; j < 4; ++j) {
            const bool single = (j & 1) ? t.heads == 1 : tokens == 1;   // the stride of a single one is not used
            if (!single && (st[j] < d_head || st[j] > lim)) return fail(EDB200_ERR_INVALID, "rope_apply: strides must be at least d_head");
            vec = vec && (single || st[j] % w == 0);
        }
        if (t.in == t.out && ((tokens > 1 && t.in_token != t.out_token) || (t.heads > 1 && t.in_head != t.out_head))) {
            return fail(EDB200_ERR_INVALID, "rope_apply: in place needs the same strides");
        }
        vec = vec && ((reinterpret_cast<uintptr_t>(t.in) | reinterpret_cast<uintptr_t>(t.out)) & 15u) == 0;
        P.t[i] = {t.in, t.out, t.in_token, t.in_head, t.out_token, t.out_head, t.heads};
    }
    if (ts[1] != nullptr && (q->out == k->out || q->out == k->in || k->out == q->in)) {
        return fail(EDB200_ERR_INVALID, "rope_apply: one tensor's out may not be the other's out or in");
    }
    if (reinterpret_cast<uintptr_t>(positions) & 3u) return fail(EDB200_ERR_INVALID, "rope_apply: positions must be 4-byte aligned");
    P.positions = positions;
    P.tokens = tokens;
    P.n_axes = r->n_axes;
    P.pairs = r->pairs;
    P.d_head = d_head;
    P.mul = r->mul;
    P.sign = inverse ? -1.0f : 1.0f;
    memcpy(P.turns, r->turns, sizeof(P.turns));
    memcpy(P.axis, r->axis, sizeof(P.axis));
    const int piece = vec ? w : 1;
    P.units_turned = r->layout == EDB200_ROPE_HALF || piece == 1 ? r->pairs / piece : 2 * r->pairs / piece;
    P.units_head = P.units_turned + (d_head - 2 * r->pairs) / piece;
    // tokens of a CTA: about eight pieces for each thread, their table within shared memory, and two CTAs an SM before more
    const long long per_token = (long long)(P.t[0].heads + P.t[1].heads) * P.units_head;
    long long nt = 8 * rope::THREADS / per_token;
    if (nt > rope::TABLE / r->pairs) nt = rope::TABLE / r->pairs;
    const long long even = (tokens + 2 * sm_count() - 1) / (2 * sm_count());
    if (nt > even) nt = even;
    if (nt < 1) nt = 1;
    // the kernel divides by products: pieces of a CTA times pieces of a token stay below 2^32
    if (per_token >= 65536) return fail(EDB200_ERR_UNSUPPORTED, "rope_apply: a token's heads hold more than 65535 pieces");
    P.inv_token = static_cast<uint32_t>((0x100000000ull + per_token - 1) / per_token);
    P.inv_head = static_cast<uint32_t>((0x100000000ull + P.units_head - 1) / P.units_head);
    P.tokens_per_cta = static_cast<int>(nt);
    const long long grid = (tokens + nt - 1) / nt;
    if (grid > 0x7fffffff) return fail(EDB200_ERR_UNSUPPORTED, "rope_apply: too many tokens for one launch");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    ProfScope prof(s, PROF_ELEMENTWISE, 0.0, 2.0 * es * (double)tokens * (double)(P.t[0].heads + P.t[1].heads) * (double)d_head);
    const bool half = r->layout == EDB200_ROPE_HALF;
    if (dtype == EDB200_TYPE_F32) {
        rope::launch<float>(P, half, vec, static_cast<unsigned>(grid), s);
    } else if (dtype == EDB200_TYPE_F16) {
        rope::launch<__half>(P, half, vec, static_cast<unsigned>(grid), s);
    } else {
        rope::launch<__nv_bfloat16>(P, half, vec, static_cast<unsigned>(grid), s);
    }
    count_launch();
    return check_cuda(cudaGetLastError(), "rope_apply launch");
}

}  // extern "C"
