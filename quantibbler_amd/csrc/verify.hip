// verify.hip -- drafted tokens against the target's probabilities, from given
// uniform numbers.
//
// A request has n drafted tokens d_0 .. d_{n-1}, target logits x_0 .. x_n (x_j
// those that d_j was drafted for, x_n those behind the last) and the logits y_j
// that d_j was drawn from, or none, where a draft was looked up (q_j is then 1
// at d_j).  With p_j = softmax(x_j / T) and q_j = softmax(y_j / T)
//   d_j is kept while u_j q_j(d_j) < p_j(d_j);
// at the first j that is not, or at j = n, one more token is drawn,
//   with weights w = max(p_j - q_j, 0)  (all 0: p_j), at j = n w = p_n:
//   the first v of w(v) > 0 with w(0) + .. + w(v) > u_n (w(0) + .. + w(last)).
// What is emitted is then distributed as the target's own tokens are.
//
// Which v that is hangs on sums of a vocabulary's weights: off by 1e-7 of the
// whole, as f32 leaves them, one draw in a hundred over 128256 ids of like
// weight goes to a neighbour.  Exponentials and sums are 64-bit here (a f64 FMA
// takes what a f32 one does on this machine), so that an answer is the one of
// the mathematics but for one draw in 10^10.
//
//   1. statistics of every chunk of every row that a request has: largest
//      logit and sum of exponentials by it, or, T = 0, the first of the largest
//   2. (drafts with logits) which row ends a request, that row's chunks' sums of w
//   3. the chunk that holds the draw, the id in it, and the outputs
#include <math.h>

#include "qbk_internal.h"

#pragma clang fp contract(off)

namespace qbk {

#define VF_THREADS 256
#define VF_WAVES (VF_THREADS / 64)
#define VF_MAX_DRAFTS 64
#define VF_ROWS (2 * VF_MAX_DRAFTS + 1)

struct VfPart {
    float m;      // the chunk's largest logit
    uint32_t id;  // T = 0: the first that has it
    double l;     // sum of exp((x - m) / T)
};
// Where a request ends: the row, and the distributions there.
struct VfEnd {
    uint32_t row, greedy;  // greedy: the token, when T = 0
    float mp, mq;
    double lp, lq;
};

struct VfArgs {
    const void *x, *y;
    size_t xs, ys;  // values from one row to the next
    const int32_t *ids;
    const float *u, *temperature;
    const uint32_t *n_drafts;
    int32_t *tokens, *counts;
    uint32_t *pos;
    VfPart *part;  // [request][row][chunk], a request's rows: target's 0 .. k, drafts' 0 .. k - 1
    double *rest;  // [request][chunk]
    VfEnd *end;    // [request]
    uint32_t n, k, rows, vocab, chunks;
};

__device__ __forceinline__ uint32_t vf_drafts(const VfArgs &a, uint32_t i) {
    return a.n_drafts ? (a.n_drafts[i] < a.k ? a.n_drafts[i] : a.k) : a.k;
}
// log2(e) / T, 0 for T = 0 (or less, or no number): the likeliest token.
__device__ __forceinline__ double vf_heat(const VfArgs &a, uint32_t i) {
    const double log2e = 1.4426950408889634074;
    if (!a.temperature) return log2e;
    const float t = a.temperature[i];
    return t > 0.0f ? fmax(log2e / (double)t, 0x1p-500) : 0.0;  // an infinite T still masks what is -inf
}

// 2^t, t <= 0 or NaN.  t = n + f, |f| <= 1/2; the series of e^(f ln 2) up to
// the twelfth power leaves 2e-16 of it.
__device__ __forceinline__ double vf_exp2(double t) {
    t = t < -1100.0 ? -1100.0 : t;  // 0 either way
    const double n = rint(t), z = (t - n) * 0.69314718055994530942;
    double s = 1.0 / 479001600.0;
    s = __builtin_fma(s, z, 1.0 / 39916800.0);
    s = __builtin_fma(s, z, 1.0 / 3628800.0);
    s = __builtin_fma(s, z, 1.0 / 362880.0);
    s = __builtin_fma(s, z, 1.0 / 40320.0);
    s = __builtin_fma(s, z, 1.0 / 5040.0);
    s = __builtin_fma(s, z, 1.0 / 720.0);
    s = __builtin_fma(s, z, 1.0 / 120.0);
    s = __builtin_fma(s, z, 1.0 / 24.0);
    s = __builtin_fma(s, z, 1.0 / 6.0);
    s = __builtin_fma(s, z, 0.5);
    s = __builtin_fma(s, z, 1.0);
    s = __builtin_fma(s, z, 1.0);
    return __builtin_amdgcn_ldexp(s, (int)n);
}
// exp((x - m) / T) by heat; m is finite or nothing is above -inf.
__device__ __forceinline__ double vf_weight(float x, float m, double heat) {
    return vf_exp2(((double)x - (double)(m == -INFINITY ? 0.0f : m)) * heat);
}

__device__ __forceinline__ float vf_in(float x) { return x; }
__device__ __forceinline__ float vf_in(uint16_t x) { return bf16_to_f32(x); }

// Values at any alignment, 16 bytes a load.
template <typename T>
struct VfVec {
    static constexpr int N = 16 / sizeof(T);
    struct __attribute__((packed, aligned(sizeof(T)))) Load {
        T v[N];
    };
};
// N values from index at on, -inf past the vocabulary.
template <typename T>
__device__ __forceinline__ void vf_load(const T *row, uint32_t at, uint32_t vocab, float *v) {
    constexpr int N = VfVec<T>::N;
    if (at + N <= vocab) {
        const auto w = *(const typename VfVec<T>::Load *)(row + at);
#pragma unroll
        for (int e = 0; e < N; e++) v[e] = vf_in(w.v[e]);
    } else {
#pragma unroll
        for (int e = 0; e < N; e++) v[e] = at + e < vocab ? vf_in(row[at + e]) : -INFINITY;
    }
}

template <typename V, class OP>
__device__ __forceinline__ V vf_wave(V v, OP op) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v = op(v, __shfl_xor(v, o, 64));
    return v;
}
// Over the workgroup; red: a slot a wave.
template <typename V, class OP>
__device__ __forceinline__ V vf_block(V v, V *red, OP op) {
    v = vf_wave(v, op);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int w = 1; w < VF_WAVES; w++) v = op(v, red[w]);
    return v;
}
struct VfAdd {
    __device__ __forceinline__ double operator()(double a, double b) const { return a + b; }
};
struct VfMax {
    __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); }
};
struct VfMin {
    __device__ __forceinline__ uint32_t operator()(uint32_t a, uint32_t b) const { return a < b ? a : b; }
};
// The sum over the threads before this one, and over all.
__device__ __forceinline__ double vf_before(double v, double *red, double &all) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    double s = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const double t = __shfl_up(s, o, 64);
        if (lane >= o) s += t;
    }
    __syncthreads();
    if (lane == 63) red[wave] = s;
    __syncthreads();
    double base = 0.0;
    all = 0.0;
#pragma unroll
    for (int w = 0; w < VF_WAVES; w++) {
        if (w < wave) base += red[w];
        all += red[w];
    }
    const double up = __shfl_up(s, 1, 64);
    return base + (lane ? up : 0.0);
}

// A workgroup a chunk of a row.
template <typename T, int PER>
__global__ void __launch_bounds__(VF_THREADS) vf_stats(VfArgs a) {
    constexpr int N = VfVec<T>::N, LOADS = PER / N;
    __shared__ float red[VF_WAVES];
    __shared__ double red2[VF_WAVES];
    __shared__ uint32_t red3[VF_WAVES];
    const uint32_t chunk = blockIdx.x % a.chunks, row = blockIdx.x / a.chunks, i = row / a.rows, r = row % a.rows;
    const bool target = r <= a.k;
    const uint32_t j = target ? r : r - a.k - 1, drafts = vf_drafts(a, i);
    const double heat = vf_heat(a, i);
    if (j > drafts || (!target && (j == drafts || heat == 0.0))) return;
    const T *src = target ? (const T *)a.x + ((size_t)i * (a.k + 1) + j) * a.xs : (const T *)a.y + ((size_t)i * a.k + j) * a.ys;
    const uint32_t base = chunk * (VF_THREADS * PER);
    float v[PER], most = -INFINITY;
#pragma unroll
    for (int q = 0; q < LOADS; q++) vf_load<T>(src, base + (q * VF_THREADS + threadIdx.x) * N, a.vocab, v + q * N);
#pragma unroll
    for (int q = 0; q < PER; q++) most = fmaxf(most, v[q]);
    const float m = vf_block(most, red, VfMax());
    VfPart part{m, 0u, 0.0};
    if (heat == 0.0) {
        uint32_t id = ~0u;
#pragma unroll
        for (int q = PER - 1; q >= 0; q--)
            if (v[q] == m) id = base + ((q / N) * VF_THREADS + threadIdx.x) * N + q % N;
        part.id = vf_block(id, red3, VfMin());
    } else {
        double l = 0.0;
#pragma unroll
        for (int q = 0; q < PER; q++) l += vf_weight(v[q], m, heat);
        part.l = vf_block(l, red2, VfAdd());
    }
    if (threadIdx.x == 0) a.part[(size_t)row * a.chunks + chunk] = part;
}

// Where request i ends; a whole workgroup, every thread gets it.
struct VfShared {
    float m[VF_ROWS];
    double l[VF_ROWS];
    uint32_t id[VF_MAX_DRAFTS + 1];
    VfEnd end;
};
template <typename T>
__device__ __forceinline__ VfEnd vf_end(const VfArgs &a, uint32_t i, double heat, VfShared &s) {
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, drafts = vf_drafts(a, i);
    for (uint32_t r = wave; r < a.rows; r += VF_WAVES) {
        const bool target = r <= a.k;
        const uint32_t j = target ? r : r - a.k - 1;
        if (j > drafts || (!target && (j == drafts || heat == 0.0))) continue;
        const VfPart *part = a.part + ((size_t)i * a.rows + r) * a.chunks;
        float m = -INFINITY;
        uint32_t id = ~0u;
        for (uint32_t c = lane; c < a.chunks; c += 64)
            if (part[c].m > m) {  // the first chunk of a lane's that has it
                m = part[c].m;
                id = part[c].id;
            }
        const float M = vf_wave(m, VfMax());
        double l = 0.0;
        if (heat == 0.0) {
            id = vf_wave(m == M && M > -INFINITY ? id : ~0u, VfMin());
        } else {
            for (uint32_t c = lane; c < a.chunks; c += 64) l += part[c].l * vf_weight(part[c].m, M, heat);
            l = vf_wave(l, VfAdd());
        }
        if (lane == 0) {
            s.m[r] = M;
            s.l[r] = l;
            if (target) s.id[r] = id == ~0u ? 0u : id;
        }
    }
    __syncthreads();
    if (wave == 0) {
        bool kept = false;
        if (lane < drafts) {
            const int32_t d = a.ids[(size_t)i * a.k + lane];
            if (d >= 0 && (uint32_t)d < a.vocab) {
                if (heat == 0.0) {
                    kept = (uint32_t)d == s.id[lane];
                } else {
                    const float x = vf_in(((const T *)a.x)[((size_t)i * (a.k + 1) + lane) * a.xs + d]);
                    const double p = vf_weight(x, s.m[lane], heat) / s.l[lane];
                    double q = 1.0;
                    if (a.y) {
                        const uint32_t r = a.k + 1 + lane;
                        const float y = vf_in(((const T *)a.y)[((size_t)i * a.k + lane) * a.ys + d]);
                        q = vf_weight(y, s.m[r], heat) / s.l[r];
                    }
                    kept = (double)a.u[(size_t)i * (a.k + 1) + lane] * q < p;
                }
            }
        }
        const uint64_t going = __ballot(kept);
        if (lane == 0) {
            const uint64_t stop = ~going;
            uint32_t j = stop ? (uint32_t)__builtin_ctzll(stop) : 64u;
            j = j < drafts ? j : drafts;
            s.end.row = j;
            s.end.greedy = heat == 0.0 ? s.id[j] : 0u;
            s.end.mp = s.m[j];
            s.end.lp = s.l[j];
            s.end.mq = 0.0f;
            s.end.lq = 0.0;
            if (a.y && j < drafts && heat != 0.0) {
                s.end.mq = s.m[a.k + 1 + j];
                s.end.lq = s.l[a.k + 1 + j];
            }
        }
    }
    __syncthreads();
    return s.end;
}

// max(p - q, 0) at one id; 0 where either is no number.
__device__ __forceinline__ double vf_rest_of(float x, float y, const VfEnd &e, double heat) {
    const double w = vf_weight(x, e.mp, heat) / e.lp - vf_weight(y, e.mq, heat) / e.lq;
    return w > 0.0 ? w : 0.0;
}

// A workgroup a chunk of each request's last row.
template <typename T, int PER>
__global__ void __launch_bounds__(VF_THREADS) vf_rest(VfArgs a) {
    constexpr int N = VfVec<T>::N;
    __shared__ VfShared s;
    __shared__ double red[VF_WAVES];
    const uint32_t i = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks;
    const double heat = vf_heat(a, i);
    const VfEnd e = vf_end<T>(a, i, heat, s);
    if (chunk == 0 && threadIdx.x == 0) a.end[i] = e;
    if (heat == 0.0 || e.row == vf_drafts(a, i)) return;
    const T *x = (const T *)a.x + ((size_t)i * (a.k + 1) + e.row) * a.xs;
    const T *y = (const T *)a.y + ((size_t)i * a.k + e.row) * a.ys;
    double sum = 0.0;
#pragma unroll
    for (int q = 0; q < PER / N; q++) {
        const uint32_t at = chunk * (VF_THREADS * PER) + (q * VF_THREADS + threadIdx.x) * N;
        float xv[N], yv[N];
        vf_load<T>(x, at, a.vocab, xv);
        vf_load<T>(y, at, a.vocab, yv);
#pragma unroll
        for (int f = 0; f < N; f++)
            if (at + f < a.vocab) sum += vf_rest_of(xv[f], yv[f], e, heat);
    }
    sum = vf_block(sum, red, VfAdd());
    if (threadIdx.x == 0) a.rest[(size_t)i * a.chunks + chunk] = sum;
}

// A workgroup a request.
template <typename T, int PER>
__global__ void __launch_bounds__(VF_THREADS) vf_choose(VfArgs a) {
    constexpr int N = VfVec<T>::N;
    constexpr uint32_t CHUNK = VF_THREADS * PER;
    __shared__ VfShared s;
    __shared__ double red[VF_WAVES];
    __shared__ uint32_t red3[VF_WAVES];
    const uint32_t i = blockIdx.x, tid = threadIdx.x, drafts = vf_drafts(a, i);
    const double heat = vf_heat(a, i);
    const VfEnd e = a.y ? a.end[i] : vf_end<T>(a, i, heat, s);
    const T *x = (const T *)a.x + ((size_t)i * (a.k + 1) + e.row) * a.xs;
    const T *y = (const T *)a.y + ((size_t)i * a.k + e.row) * a.ys;
    int32_t token = -1;
    if (heat == 0.0) {
        token = (int32_t)e.greedy;
    } else if (e.lp > 0.0 && e.lp < INFINITY) {
        const VfPart *part = a.part + ((size_t)i * a.rows + e.row) * a.chunks;
        bool less = a.y && e.row < drafts;  // weights max(p - q, 0), otherwise p times its sum
        uint32_t skip = ~0u;                // the id that has none: a draft that was looked up
        if (!a.y && e.row < drafts) skip = (uint32_t)a.ids[(size_t)i * a.k + e.row];
        auto weight = [&](uint32_t at, float xv, float yv) {
            if (at >= a.vocab || at == skip) return 0.0;
            return less ? vf_rest_of(xv, yv, e, heat) : vf_weight(xv, e.mp, heat);
        };
        // a chunk's weights in the order of their ids, PER a thread
        auto each = [&](uint32_t chunk, double *w) {
            const uint32_t at = chunk * CHUNK + tid * PER;
#pragma unroll
            for (int q = 0; q < PER / N; q++) {
                float xv[N], yv[N] = {};
                vf_load<T>(x, at + q * N, a.vocab, xv);
                if (less) vf_load<T>(y, at + q * N, a.vocab, yv);
#pragma unroll
                for (int f = 0; f < N; f++) w[q * N + f] = weight(at + q * N + f, xv[f], yv[f]);
            }
        };
        double w[PER], skipped = 0.0, total = 0.0;
        for (int tries = 0; tries < 2; tries++) {
            if (skip < a.vocab) {  // the sum of its chunk without it
                each(skip / CHUNK, w);
                double l = 0.0;
#pragma unroll
                for (int q = 0; q < PER; q++) l += w[q];
                skipped = vf_block(l, red, VfAdd());
            }
            double t = 0.0;
            for (uint32_t c = tid; c < a.chunks; c += VF_THREADS)
                t += less ? a.rest[(size_t)i * a.chunks + c]
                          : c == skip / CHUNK && skip < a.vocab ? skipped : part[c].l * vf_weight(part[c].m, e.mp, heat);
            total = vf_block(t, red, VfAdd());
            if (total > 0.0) break;
            less = false;  // p and q are alike to the last place: p
            skip = ~0u;
        }
        const double want = (double)a.u[(size_t)i * (a.k + 1) + drafts] * total;
        // the chunk: the first whose running sum is above want, or the last with any weight
        double base = 0.0, from = 0.0;
        uint32_t chunk = ~0u;
        uint32_t last = 0;
        for (uint32_t c0 = 0; c0 < a.chunks && chunk == ~0u; c0 += VF_THREADS) {
            const uint32_t c = c0 + tid;
            double mine = 0.0;
            if (c < a.chunks)
                mine = less ? a.rest[(size_t)i * a.chunks + c]
                            : c == skip / CHUNK && skip < a.vocab ? skipped : part[c].l * vf_weight(part[c].m, e.mp, heat);
            double all;
            const double before = base + vf_before(mine, red, all);
            chunk = vf_block(mine > 0.0 && before + mine > want ? c : ~0u, red3, VfMin());
            const uint32_t some = ~vf_block(mine > 0.0 ? ~c : ~0u, red3, VfMin());
            if (some != 0u || c0 == 0) last = some != 0u ? some : last;
            from = base;
            base += all;
        }
        const bool none = chunk == ~0u;
        if (none) chunk = last;
        // what stands before it, again: the threads before it in its round
        {
            const uint32_t c = chunk / VF_THREADS * VF_THREADS + tid;
            double mine = 0.0;
            if (c < chunk)
                mine = less ? a.rest[(size_t)i * a.chunks + c]
                            : c == skip / CHUNK && skip < a.vocab ? skipped : part[c].l * vf_weight(part[c].m, e.mp, heat);
            from = (none ? 0.0 : from) + vf_block(mine, red, VfAdd());
        }
        each(chunk, w);
        double l = 0.0, all;
#pragma unroll
        for (int q = 0; q < PER; q++) l += w[q];
        double run = from + vf_before(l, red, all);
        uint32_t at = ~0u, final_ = 0u;
#pragma unroll
        for (int q = 0; q < PER; q++) {
            run += w[q];
            if (w[q] > 0.0) {
                const uint32_t id = chunk * CHUNK + tid * PER + q;
                if (run > want && at == ~0u) at = id;
                final_ = id + 1;
            }
        }
        at = vf_block(none ? ~0u : at, red3, VfMin());
        final_ = ~vf_block(~final_, red3, VfMin());
        token = (int32_t)(at != ~0u ? at : final_ - 1);
    }
    const uint32_t got = e.row + (token >= 0 ? 1u : 0u);
    for (uint32_t j = tid; j <= a.k; j += VF_THREADS)
        a.tokens[(size_t)i * (a.k + 1) + j] = j < e.row ? a.ids[(size_t)i * a.k + j] : j == e.row ? token : -1;
    if (tid == 0) {
        a.counts[i] = (int32_t)got;
        if (a.pos) a.pos[i] += got;
    }
}

// Ids a workgroup: eight a thread where the rows leave the card idle with 32.
static int vf_per(size_t n, size_t k, size_t vocab, bool given) {
    const size_t rows = n * (given ? 2 * k + 1 : k + 1);
    return rows * div_ceil(vocab, 32 * VF_THREADS) < 512 ? 8 : 32;
}
struct VfPlan {
    int per;
    size_t rows, chunks, o_rest, o_end, bytes;
};
static VfPlan vf_plan(size_t n, size_t k, size_t vocab, bool given) {
    VfPlan p;
    p.per = vf_per(n, k, vocab, given);
    p.rows = given ? 2 * k + 1 : k + 1;
    p.chunks = div_ceil(vocab, (size_t)p.per * VF_THREADS);
    p.o_rest = n * p.rows * p.chunks * sizeof(VfPart);
    p.o_end = p.o_rest + (given ? n * p.chunks * sizeof(double) : 0);
    p.bytes = round_up(p.o_end + (given ? n * sizeof(VfEnd) : 0), 256);
    return p;
}

static int vf_check(size_t n, size_t k, size_t vocab, bool given) {
    if (vocab == 0 || vocab > 0x7FFFFFFFull) return fail(QBK_ERR_VALIDATION, "verify_drafts needs 1 <= vocab < 2^31");
    if (k > VF_MAX_DRAFTS)
        return fail(QBK_ERR_VALIDATION, fmt("verify_drafts takes up to %d drafts a request, got %zu", VF_MAX_DRAFTS, k));
    if (given && k == 0) return fail(QBK_ERR_VALIDATION, "verify_drafts: draft logits without drafts");
    if (n > 0xFFFFFF || n * (2 * k + 1) > 0xFFFFFF) return fail(QBK_ERR_VALIDATION, "verify_drafts: too many rows for one launch");
    const VfPlan p = vf_plan(n, k, vocab, given);
    if (n * p.rows * p.chunks > 0xFFFFFF)  // a launch is below 2^32 threads
        return fail(QBK_ERR_VALIDATION, "verify_drafts: too many rows for one launch");
    return QBK_OK;
}

template <typename T, int PER>
static void vf_go(const VfArgs &a, hipStream_t s) {
    hipLaunchKernelGGL((vf_stats<T, PER>), dim3(a.n * a.rows * a.chunks), dim3(VF_THREADS), 0, s, a);
    if (a.y) hipLaunchKernelGGL((vf_rest<T, PER>), dim3(a.n * a.chunks), dim3(VF_THREADS), 0, s, a);
    hipLaunchKernelGGL((vf_choose<T, PER>), dim3(a.n), dim3(VF_THREADS), 0, s, a);
}

}  // namespace qbk

using namespace qbk;

extern "C" {

size_t qbk_verify_drafts_workspace_size(size_t n, size_t k, size_t vocab, int draft_logits) {
    return vf_check(n, k, vocab, draft_logits != 0) ? 0 : vf_plan(n, k, vocab, draft_logits != 0).bytes;
}

int qbk_verify_drafts_dev(qbk_ctx *ctx, const void *logits, const void *draft_logits, int dtype, size_t n, size_t k,
                          size_t vocab, size_t row_stride, size_t draft_row_stride, const int32_t *ids,
                          const uint32_t *n_drafts, const float *uniforms, const float *temperature, int32_t *tokens,
                          int32_t *counts, uint32_t *pos, void *workspace, size_t workspace_size, void *stream) {
    int rc;
    const bool given = draft_logits != nullptr;
    if ((rc = vf_check(n, k, vocab, given))) return rc;
    if (dtype != QBK_F32 && dtype != QBK_BF16)
        return fail(QBK_ERR_VALIDATION, fmt("verify_drafts takes float32 or bfloat16 logits (dtype %d)", dtype));
    const size_t most = (size_t)1 << 40;
    if ((n * (k + 1) > 1 && (row_stride < vocab || row_stride > most)) ||
        (given && n * k > 1 && (draft_row_stride < vocab || draft_row_stride > most)))
        return fail(QBK_ERR_VALIDATION, fmt("row strides of %zu and %zu do not fit rows of %zu logits", row_stride,
                                            draft_row_stride, vocab));
    if (n == 0) return QBK_OK;
    if (!logits || !uniforms || !tokens || !counts || (k && !ids)) return fail(QBK_ERR_VALIDATION, "null argument");
    const VfPlan p = vf_plan(n, k, vocab, given);
    if (!workspace || workspace_size < p.bytes)
        return fail(QBK_ERR_VALIDATION, fmt("verify_drafts workspace of %zu bytes is smaller than the %zu needed",
                                            workspace ? workspace_size : (size_t)0, p.bytes));
    if ((uintptr_t)workspace & 15) return fail(QBK_ERR_VALIDATION, "verify_drafts workspace must be 16-byte aligned");
    if ((rc = bind(ctx))) return rc;
    VfArgs a{};
    a.x = logits;
    a.y = draft_logits;
    a.xs = row_stride;
    a.ys = draft_row_stride;
    a.ids = ids;
    a.u = uniforms;
    a.temperature = temperature;
    a.n_drafts = n_drafts;
    a.tokens = tokens;
    a.counts = counts;
    a.pos = pos;
    a.part = (VfPart *)workspace;
    a.rest = (double *)((char *)workspace + p.o_rest);
    a.end = (VfEnd *)((char *)workspace + p.o_end);
    a.n = (uint32_t)n;
    a.k = (uint32_t)k;
    a.rows = (uint32_t)p.rows;
    a.vocab = (uint32_t)vocab;
    a.chunks = (uint32_t)p.chunks;
    hipStream_t s = (hipStream_t)stream;
    if (dtype == QBK_F32) p.per == 8 ? vf_go<float, 8>(a, s) : vf_go<float, 32>(a, s);
    else p.per == 8 ? vf_go<uint16_t, 8>(a, s) : vf_go<uint16_t, 32>(a, s);
    QBK_HIP(hipGetLastError());
    return QBK_OK;
}

}  // extern "C"
