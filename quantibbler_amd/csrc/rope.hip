// rope.hip -- heads normed and turned to their positions in one pass.
//
// Pair i of a row at position t: angle 2 pi frac(t turns_i), turns_i = f_i / 2 pi
// in units of 2^-64: an integer product modulo 2^64 is the fraction of a turn
// itself, to 2^-32 of a turn at position 2^32, where a float product has none of
// it left from 2^24 turns on.  Cos and sin of what is left of the nearest quarter
// turn are series in 64 bits (once a row, for all its heads; a f64 FMA takes what
// a f32 one does), rounded once to f32.  One pass, bound by memory (8192 rows of
// 32 and 8 heads of 128, bf16, out of wider rows: 38 us, 4.4 TB/s; where angles
// were formed head by head, 189), a few rows by the launch (one 3.6 us).
#include <math.h>

#include "kvcache_rows.h"

#pragma clang fp contract(off)

namespace qbk {

struct RotArgs {
    const void *q, *k;
    void *qo, *ko;
    const float *wq, *wk;
    const uint32_t *row_start, *pos;
    size_t qs, ks, qos, kos;  // values from one row to the next
    uint64_t before;
    uint32_t n_rows, n, per, H, Hk;
    float eps;
    uint32_t waves;  // a row's
    qbk_rope rope;
};

// cos and sin of 2 pi turns / 2^64.  |x| <= pi / 4: the series' next terms are
// below 2^-60.
__device__ __forceinline__ float2 rot_turn(uint64_t turns, double size) {
    const uint64_t quarter = (turns + (1ull << 61)) >> 62;
    const double x = (double)(int64_t)(turns - (quarter << 62)) * (6.283185307179586477 * 0x1p-64), z = x * x;
    double c = -1.0 / 87178291200.0, s = 1.0 / 6227020800.0;
    c = __builtin_fma(c, z, 1.0 / 479001600.0);
    s = __builtin_fma(s, z, -1.0 / 39916800.0);
    c = __builtin_fma(c, z, -1.0 / 3628800.0);
    s = __builtin_fma(s, z, 1.0 / 362880.0);
    c = __builtin_fma(c, z, 1.0 / 40320.0);
    s = __builtin_fma(s, z, -1.0 / 5040.0);
    c = __builtin_fma(c, z, -1.0 / 720.0);
    s = __builtin_fma(s, z, 1.0 / 120.0);
    c = __builtin_fma(c, z, 1.0 / 24.0);
    s = __builtin_fma(s, z, -1.0 / 6.0);
    c = __builtin_fma(c, z, -0.5);
    c = __builtin_fma(c, z, 1.0);
    s = __builtin_fma(s * z, x, x);
    if (quarter & 1) {
        const double t = c;
        c = -s;
        s = t;
    }
    const double by = quarter & 2 ? -size : size;
    return float2{(float)(c * by), (float)(s * by)};
}

template <typename T>
__device__ __forceinline__ float rot_in(T x) {
    if constexpr (sizeof(T) == 4) return x;
    else return bf16_to_f32(x);
}
template <typename T>
__device__ __forceinline__ T rot_out(float x) {
    if constexpr (sizeof(T) == 4) return x;
    else return f32_to_bf16(x);
}

// The row's position; false where no sequence claims it.
__device__ __forceinline__ bool rot_place(const RotArgs &a, uint32_t r, uint64_t &at) {
    uint32_t s, start, end;
    if (!kv_claim(a.row_start, a.n, a.per, r, s, start, end)) return false;
    at = a.before + a.pos[s] + (r - start);
    return true;
}

// The sum over aligned runs of LANES lanes.
template <int LANES>
__device__ __forceinline__ float rot_sum(float v) {
    auto add = [](float x, int moved) { return x + __uint_as_float((uint32_t)moved); };
    if constexpr (LANES >= 2) v = add(v, __builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), 0xB1, 0xf, 0xf, true));   // lane ^ 1
    if constexpr (LANES >= 4) v = add(v, __builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), 0x4E, 0xf, 0xf, true));   // lane ^ 2
    if constexpr (LANES >= 8) v = add(v, __builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), 0x141, 0xf, 0xf, true));  // 7 - lane
    if constexpr (LANES >= 16) v = add(v, __builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), 0x140, 0xf, 0xf, true)); // 15 - lane
    if constexpr (LANES >= 32) {
        const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    }
    return v;
}

// Four values at any alignment, one access.
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Rot4 {
    T v[4];
};

// LANES lanes a head, two runs of four channels a lane: in the half layout
// channels 4 l .. and rotary / 2 + 4 l .., the two halves of four pairs,
// interleaved and past rotary_dim 8 l .. 8 l + 7.  A wave takes 64 / LANES heads
// of a row at a time and turns all of them by the four angles it has formed
// once.
template <typename T, int LANES>
__global__ void __launch_bounds__(256) rot_quads(RotArgs a) {
    constexpr uint32_t HEADS = 64 / LANES;
    const uint64_t item = (uint64_t)blockIdx.x * 4 + (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const uint32_t r = (uint32_t)(item / a.waves), wave = (uint32_t)(item % a.waves);
    uint64_t at;
    if (r >= a.n_rows || !rot_place(a, r, at)) return;
    const uint32_t lane = threadIdx.x & 63, l = lane % LANES, hd = a.rope.head_dim, half = a.rope.rotary_dim / 2;
    const bool in = 8 * l < hd, turned = 8 * l < 2 * half, inter = a.rope.interleaved;
    const uint32_t c0 = turned && !inter ? 4 * l : 8 * l, c1 = turned && !inter ? half + 4 * l : 8 * l + 4;
    float2 t[4];
    if (turned)
#pragma unroll
        for (int i = 0; i < 4; i++) t[i] = rot_turn(a.rope.turns[4 * l + i] * at, a.rope.size);
    const uint32_t all = a.H + a.Hk;
    for (uint32_t first = wave * HEADS; first < all; first += a.waves * HEADS) {
        const uint32_t head = first + lane / LANES;
        const bool is_q = head < a.H, live = in && head < all;
        const uint32_t h = is_q ? head : head - a.H;
        const T *src = is_q ? (const T *)a.q + r * a.qs + (size_t)h * hd : (const T *)a.k + r * a.ks + (size_t)h * hd;
        T *dst = is_q ? (T *)a.qo + r * a.qos + (size_t)h * hd : (T *)a.ko + r * a.kos + (size_t)h * hd;
        const float *w = is_q ? a.wq : a.wk;
        float x[8];
        if (live) {
            const Rot4<T> lo = *(const Rot4<T> *)(src + c0), hi = *(const Rot4<T> *)(src + c1);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                x[e] = rot_in<T>(lo.v[e]);
                x[4 + e] = rot_in<T>(hi.v[e]);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = 0.0f;
        }
        float ss = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; e++) ss += x[e] * x[e];
        ss = rot_sum<LANES>(ss);
        if (!live) continue;
        if (w) {
            const float mean = ss / (float)hd + a.eps;
            const bool low = mean < 0x1p-126f;  // eps 0: the instruction takes a subnormal number for 0
            const float inv = __builtin_amdgcn_rsqf(low ? mean * 0x1p64f : mean) * (low ? 0x1p32f : 1.0f);
            const Rot4<float> lo = *(const Rot4<float> *)(w + c0), hi = *(const Rot4<float> *)(w + c1);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                x[e] = x[e] * inv * lo.v[e];
                x[4 + e] = x[4 + e] * inv * hi.v[e];
            }
        }
        if (turned) {
            if (inter) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float p = x[2 * i], q = x[2 * i + 1];
                    x[2 * i] = p * t[i].x - q * t[i].y;
                    x[2 * i + 1] = q * t[i].x + p * t[i].y;
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float p = x[i], q = x[4 + i];
                    x[i] = p * t[i].x - q * t[i].y;
                    x[4 + i] = q * t[i].x + p * t[i].y;
                }
            }
        }
        Rot4<T> lo, hi;
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int e = 0; e < 4; e++) {
                lo.v[e] = x[e];
                hi.v[e] = x[4 + e];
            }
        } else {
            const uint2 u = {f32x2_to_bf16x2(x[0], x[1]), f32x2_to_bf16x2(x[2], x[3])};
            const uint2 v = {f32x2_to_bf16x2(x[4], x[5]), f32x2_to_bf16x2(x[6], x[7])};
            lo = __builtin_bit_cast(Rot4<T>, u);
            hi = __builtin_bit_cast(Rot4<T>, v);
        }
        *(Rot4<T> *)(dst + c0) = lo;
        *(Rot4<T> *)(dst + c1) = hi;
    }
}

// A wave a row and head, a pair or a channel a lane at a time: any layout.
template <typename T>
__global__ void __launch_bounds__(256) rot_any(RotArgs a) {
    const uint64_t item = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const uint32_t all = a.H + a.Hk, r = (uint32_t)(item / all), head = (uint32_t)(item % all), lane = threadIdx.x & 63;
    uint64_t at;
    if (r >= a.n_rows || !rot_place(a, r, at)) return;
    const uint32_t hd = a.rope.head_dim, half = a.rope.rotary_dim / 2;
    const bool is_q = head < a.H;
    const uint32_t h = is_q ? head : head - a.H;
    const T *src = is_q ? (const T *)a.q + r * a.qs + (size_t)h * hd : (const T *)a.k + r * a.ks + (size_t)h * hd;
    T *dst = is_q ? (T *)a.qo + r * a.qos + (size_t)h * hd : (T *)a.ko + r * a.kos + (size_t)h * hd;
    const float *w = is_q ? a.wq : a.wk;
    float inv = 1.0f;
    if (w) {
        float ss = 0.0f;
        for (uint32_t c = lane; c < hd; c += 64) {
            const float x = rot_in<T>(src[c]);
            ss += x * x;
        }
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) ss += __shfl_xor(ss, o, 64);
        inv = 1.0f / sqrtf(ss / (float)hd + a.eps);
    }
    auto value = [&](uint32_t c) {
        const float x = rot_in<T>(src[c]);
        return w ? x * inv * w[c] : x;
    };
    for (uint32_t i = lane; i < half; i += 64) {
        const uint32_t c0 = a.rope.interleaved ? 2 * i : i, c1 = a.rope.interleaved ? 2 * i + 1 : i + half;
        const float2 t = rot_turn(a.rope.turns[i] * at, a.rope.size);
        const float x = value(c0), y = value(c1);
        dst[c0] = rot_out<T>(x * t.x - y * t.y);
        dst[c1] = rot_out<T>(y * t.x + x * t.y);
    }
    for (uint32_t c = 2 * half + lane; c < hd; c += 64) dst[c] = rot_out<T>(value(c));
}

// Whether a head falls into runs of four pairs and eight channels.  Pair by pair
// otherwise (us by runs / by pairs, 8192 rows of 32 and 8 heads of 128, bf16: 29 /
// 142, 32 rows 3.3 / 3.6).
static bool rot_by_quads(const qbk_rope &r) { return r.head_dim % 8 == 0 && r.rotary_dim % 8 == 0; }

template <typename T>
static void rot_go(RotArgs a, hipStream_t s) {
    const size_t all = a.H + a.Hk;
    if (!rot_by_quads(a.rope)) {
        hipLaunchKernelGGL(rot_any<T>, dim3((unsigned)div_ceil(a.n_rows * all, 4)), dim3(256), 0, s, a);
        return;
    }
    const uint32_t hd = a.rope.head_dim;
    const int lanes = hd <= 16 ? 2 : hd <= 32 ? 4 : hd <= 64 ? 8 : hd <= 128 ? 16 : 32;
    // Waves a row: two a SIMD, up to eight while each has five passes over heads to form its angles for (us for one wave a
    // row, two a SIMD, eight; 32 and 8 heads of 128, bf16: 1 row 7.1 / 3.5 / 3.2, 1024 rows 8.9 / 7.1 / 8.5, 4096 18.8 /
    // 18.6 / 17.0; 16 and 4 heads of 64: 32 rows 4.2 / 3.2 / 3.2, 4096 7.6 / 7.6 / 8.9; all passes apart, 8192 rows of
    // heads of 128 29 -> 48).
    const size_t passes = div_ceil(all, (size_t)(64 / lanes)), two = div_ceil((size_t)2048, (size_t)a.n_rows);
    const size_t eight = div_ceil((size_t)8192, (size_t)a.n_rows), five = div_ceil(passes, (size_t)5);
    const size_t want = eight < five ? eight : five > two ? five : two;
    a.waves = (uint32_t)(want < passes ? want : passes);
    void (*k)(RotArgs) = lanes == 2   ? rot_quads<T, 2>
                         : lanes == 4 ? rot_quads<T, 4>
                         : lanes == 8 ? rot_quads<T, 8>
                         : lanes == 16 ? rot_quads<T, 16>
                                       : rot_quads<T, 32>;
    hipLaunchKernelGGL(k, dim3((unsigned)div_ceil((size_t)a.n_rows * a.waves, 4)), dim3(256), 0, s, a);
}

static int rot_check(const qbk_rope *r) {
    if (!r) return fail(QBK_ERR_VALIDATION, "null argument");
    if (r->head_dim == 0 || r->head_dim % 2 || r->head_dim > 256 || r->rotary_dim % 2 || r->rotary_dim > r->head_dim)
        return fail(QBK_ERR_VALIDATION, fmt("rope needs an even head_dim up to 256 and an even rotary_dim up to it, got %u "
                                            "and %u", r->head_dim, r->rotary_dim));
    return QBK_OK;
}

}  // namespace qbk

using namespace qbk;

extern "C" {

int qbk_rope_init(qbk_rope *rope, size_t head_dim, size_t rotary_dim, int interleaved, double theta,
                  const qbk_rope_scaling *scaling) {
    if (!rope) return fail(QBK_ERR_VALIDATION, "null argument");
    if (head_dim == 0 || head_dim % 2 || head_dim > 256 || rotary_dim == 0 || rotary_dim % 2 || rotary_dim > head_dim)
        return fail(QBK_ERR_VALIDATION, fmt("rope needs an even head_dim up to 256 and an even rotary_dim up to it, got %zu "
                                            "and %zu", head_dim, rotary_dim));
    if (!(theta > 0.0) || !isfinite(theta)) return fail(QBK_ERR_VALIDATION, fmt("rope theta must be positive, got %g", theta));
    const int kind = scaling ? scaling->kind : QBK_ROPE_PLAIN;
    if (kind < QBK_ROPE_PLAIN || kind > QBK_ROPE_YARN) return fail(QBK_ERR_VALIDATION, fmt("unknown rope scaling %d", kind));
    const double factor = kind ? scaling->factor : 1.0;
    if (!(factor > 0.0) || !isfinite(factor))
        return fail(QBK_ERR_VALIDATION, fmt("rope scaling factor must be positive, got %g", factor));
    const bool parts = kind == QBK_ROPE_RAMP || kind == QBK_ROPE_YARN;
    if (parts && (!(scaling->original_len > 0.0) || !(scaling->low > 0.0) || !(scaling->high > scaling->low) ||
                  !isfinite(scaling->original_len) || !isfinite(scaling->high)))
        return fail(QBK_ERR_VALIDATION, fmt("rope scaling by parts needs original_len > 0 and 0 < low < high, got %g, %g and %g",
                                            scaling->original_len, scaling->low, scaling->high));
    if (kind == QBK_ROPE_YARN && !(theta > 1.0))
        return fail(QBK_ERR_VALIDATION, fmt("rope scaling by the pair's number needs theta above 1, got %g", theta));
    const long double tau = 6.28318530717958647692528676655900577L;
    long double base = theta;
    if (kind == QBK_ROPE_BASE && rotary_dim > 2)
        base *= powl((long double)factor, (long double)rotary_dim / (long double)(rotary_dim - 2));
    double first = 0.0, last = 0.0;
    if (kind == QBK_ROPE_YARN) {
        auto pair = [&](double turns) {
            return (double)rotary_dim * log(scaling->original_len / (turns * (double)tau)) / (2.0 * log(theta));
        };
        first = fmax(floor(pair(scaling->high)), 0.0);
        last = fmin(ceil(pair(scaling->low)), (double)rotary_dim - 1.0);
    }
    qbk_rope r{};
    r.head_dim = (uint32_t)head_dim;
    r.rotary_dim = (uint32_t)rotary_dim;
    r.interleaved = interleaved != 0;
    r.size = kind == QBK_ROPE_YARN && factor > 1.0 ? 0.1 * log(factor) + 1.0 : 1.0;
    for (size_t i = 0; i < rotary_dim / 2; i++) {
        long double f = powl(base, -2.0L * (long double)i / (long double)rotary_dim), keep = 1.0L;
        if (kind == QBK_ROPE_LINEAR) keep = 0.0L;
        if (kind == QBK_ROPE_RAMP)
            keep = (scaling->original_len * f / tau - scaling->low) / ((long double)scaling->high - scaling->low);
        if (kind == QBK_ROPE_YARN) keep = 1.0 - ((double)i - first) / fmax(last - first, 0.001);
        keep = keep < 0.0L ? 0.0L : keep > 1.0L ? 1.0L : keep;
        f = f * keep + f / factor * (1.0L - keep);
        if (!isfinite((double)f)) return fail(QBK_ERR_VALIDATION, fmt("rope frequencies of theta %g pass the range", theta));
        const long double part = f / tau;
        r.turns[i] = (uint64_t)((part - floorl(part)) * 0x1p64L);
    }
    *rope = r;
    return QBK_OK;
}

int qbk_rotate_heads_dev(qbk_ctx *ctx, const qbk_rope *rope, const void *q, const void *k, int dtype, size_t n_rows,
                         size_t n_heads, size_t n_kv_heads, size_t q_stride, size_t k_stride, const uint32_t *row_start,
                         const uint32_t *pos, size_t n, size_t before, const float *q_norm, const float *k_norm,
                         double eps, void *q_out, void *k_out, size_t q_out_stride, size_t k_out_stride, void *stream) {
    int rc;
    if ((rc = rot_check(rope))) return rc;
    if (dtype != QBK_F32 && dtype != QBK_BF16)
        return fail(QBK_ERR_VALIDATION, fmt("rotate_heads takes float32 or bfloat16 rows (dtype %d)", dtype));
    if (n_heads > 65536 || n_kv_heads > 65536) return fail(QBK_ERR_VALIDATION, "rotate_heads takes up to 65536 heads");
    const size_t hd = rope->head_dim, most = (size_t)1 << 40;
    const size_t strides[4] = {q_stride, q_out_stride, k_stride, k_out_stride};
    for (int i = 0; i < 4; i++) {
        const size_t width = (i < 2 ? n_heads : n_kv_heads) * hd;
        if (n_rows > 1 && width && (strides[i] < width || strides[i] > most))
            return fail(QBK_ERR_VALIDATION, fmt("a row stride of %zu does not fit a row of %zu values", strides[i], width));
    }
    if (n_rows > 0x7FFFFFFFull || before > 0xFFFFFFFFull || n > 0x7FFFFFFFull)
        return fail(QBK_ERR_VALIDATION, "rotate_heads: too many rows for one call");
    if (n_rows != 0 && n == 0) return fail(QBK_ERR_VALIDATION, "rotate_heads: rows of no sequence");
    if (n_rows != 0 && !row_start && n_rows % n != 0)
        return fail(QBK_ERR_VALIDATION, fmt("%zu rows do not split evenly over %zu sequences", n_rows, n));
    if (!(eps >= 0.0) && (q_norm || k_norm)) return fail(QBK_ERR_VALIDATION, fmt("rotate_heads: eps must not be negative, got %g", eps));
    const size_t groups = div_ceil(n_rows * (n_heads + n_kv_heads), 4);
    if (groups > 0xFFFFFF) return fail(QBK_ERR_VALIDATION, "rotate_heads: too many rows for one call");
    if (groups == 0) return QBK_OK;
    if (!pos || (n_heads && (!q || !q_out)) || (n_kv_heads && (!k || !k_out)))
        return fail(QBK_ERR_VALIDATION, "null argument");
    if ((rc = bind(ctx))) return rc;
    if (n_rows > 1 && ((n_heads && q == q_out && q_stride != q_out_stride) ||
                       (n_kv_heads && k == k_out && k_stride != k_out_stride)))
        return fail(QBK_ERR_VALIDATION, "rotate_heads in place needs one stride for rows in and out");
    RotArgs a{};
    a.q = q;
    a.k = k;
    a.qo = q_out;
    a.ko = k_out;
    a.wq = q_norm;
    a.wk = k_norm;
    a.row_start = row_start;
    a.pos = pos;
    a.qs = q_stride;
    a.ks = k_stride;
    a.qos = q_out_stride;
    a.kos = k_out_stride;
    a.before = before;
    a.n_rows = (uint32_t)n_rows;
    a.n = (uint32_t)n;
    a.per = (uint32_t)(n_rows / n ? n_rows / n : 1);
    a.H = (uint32_t)n_heads;
    a.Hk = (uint32_t)n_kv_heads;
    a.eps = (float)eps;
    a.rope = *rope;
    hipStream_t s = (hipStream_t)stream;
    if (dtype == QBK_F32) rot_go<float>(a, s);
    else rot_go<uint16_t>(a, s);
    QBK_HIP(hipGetLastError());
    return QBK_OK;
}

}  // extern "C"
