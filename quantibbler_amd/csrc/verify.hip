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
// What is emitted is then distributed as the target's own tokens are.  Where a
// request's rows end, it has no more drafts than rows behind its first token, and
// without a row for that it emits nothing.
//
// Which v that is hangs on sums of a vocabulary's weights: off by 1e-7 of the
// whole, as f32 leaves them, one draw in a hundred over 128256 ids of like
// weight goes to a neighbour.  Exponentials and sums are 64-bit here (a f64 FMA
// takes what a f32 one does on this machine), so that an answer is the one of
// the mathematics but for one draw in 10^10.
//
// A unit is a wave's 512 or 2048 neighbouring ids; no wave waits for another.
//   1. every unit of every row that a request has: its largest logit and its sum
//      of exponentials by that, or, T = 0, the first of the largest
//   2. (drafts with logits) which row ends the request, that row's units' sums of w
//   3. the unit that holds the draw, the id in it, and the outputs
// 32 requests of four drafts, 128256 ids, f32 (148 MB): 33 us, 4.5 TB/s, then 13
// for two rows of each again and 8, traced launch by launch (the call 49); four
// looked-up rows of 32003 3.2 and 5.3 (the call 8.1).  Two of three launches
// depend on the one before and are bound by that; the last workgroup of 2 doing 3
// took longer (its fences, 28 us).
#include <math.h>

#include "qbk_internal.h"

#pragma clang fp contract(off)

namespace qbk {

#define VF_WAVES 4
#define VF_THREADS (64 * VF_WAVES)
#define VF_MAX_DRAFTS 64
#define VF_ROWS (2 * VF_MAX_DRAFTS + 1)

struct VfPart {
    float m;      // the unit's largest logit
    uint32_t id;  // T = 0: the first that has it
    double l;     // sum of exp((x - m) / T)
};
// Where a request ends: the row, and the distributions there.
struct VfEnd {
    uint32_t row, greedy;  // greedy: the token, when T = 0
    float mp, mq;
    double lp, op, oq;  // p's sum, and the offsets -log2 of both
};

struct VfArgs {
    const void *x, *y;
    size_t xs, ys;  // values from one row to the next
    const int32_t *ids;
    const float *u, *temperature;
    const uint32_t *n_drafts;
    int32_t *tokens, *counts;
    uint32_t *pos;
    uint64_t limit;  // of the positions; 2^32: none
    VfPart *part;  // [request][row][unit], a request's rows: target's 0 .. k, drafts' 0 .. k - 1
    double *rest;  // [request][unit]
    VfEnd *end;    // [request]
    uint32_t n, k, rows, vocab, units;
};

// Rows that request i has left where there is a limit, the drafts that it has,
// and those that are looked at.
__device__ __forceinline__ uint64_t vf_room(const VfArgs &a, uint32_t i) {
    const uint32_t at = a.pos[i];
    return a.limit > at ? a.limit - at : 0;
}
__device__ __forceinline__ uint32_t vf_given(const VfArgs &a, uint32_t i) {
    return a.n_drafts ? (a.n_drafts[i] < a.k ? a.n_drafts[i] : a.k) : a.k;
}
__device__ __forceinline__ uint32_t vf_drafts(const VfArgs &a, uint32_t i) {
    const uint32_t m = vf_given(a, i);
    if (a.limit >> 32) return m;
    const uint64_t room = vf_room(a, i);
    return m < room ? m : room ? (uint32_t)room - 1 : 0;
}
// log2(e) / T, 0 for T = 0 (or less, or no number): the likeliest token.  A T
// past 2^110 counts as that: what is -inf stays masked.
__device__ __forceinline__ double vf_heat(const VfArgs &a, uint32_t i) {
    const double log2e = 1.4426950408889634074;
    if (!a.temperature) return log2e;
    const float t = a.temperature[i];
    return t > 0.0f ? fmax(log2e / (double)t, 0x1p-110) : 0.0;
}

// 2^t for t <= 0 as s f, f a power of two; f = 0 from -1022.5 down (and for a
// NaN).  t = n + z, |z| <= 1/2 (n by adding 1.5 2^52, whose low bits then are n),
// s = 2^z = 1 + z q(z), q the polynomial that has its values at the nine
// Chebyshev nodes of that interval: off by 4e-14 of it, 1 at 0.
struct VfPower {
    double s, f;
    __device__ __forceinline__ VfPower(double t) {
        const double round = 0x1.8p52;
        t = fmax(t, -1023.0);
        const double u = t + round, z = t - (u - round);
        double q = 0x1.b63880a9fb73bp-24;
        q = __builtin_fma(q, z, 0x1.63d13636b799fp-20);
        q = __builtin_fma(q, z, 0x1.ffcb95159f368p-17);
        q = __builtin_fma(q, z, 0x1.4308ac85aa3ccp-13);
        q = __builtin_fma(q, z, 0x1.5d87fe86fe8cap-10);
        q = __builtin_fma(q, z, 0x1.3b2ab7181b759p-7);
        q = __builtin_fma(q, z, 0x1.c6b08d7047e52p-5);
        q = __builtin_fma(q, z, 0x1.ebfbdff823cedp-3);
        q = __builtin_fma(q, z, 0x1.62e42fefa39efp-1);
        s = __builtin_fma(q, z, 1.0);
        const uint32_t n = (uint32_t)__builtin_bit_cast(uint64_t, u);
        f = __builtin_bit_cast(double, (uint64_t)((n + 1023u) << 20) << 32);
    }
    __device__ __forceinline__ double value() const { return s * f; }
};
// exp((x - m) / T) by heat.
__device__ __forceinline__ VfPower vf_power(float x, float m, double heat) { return VfPower(((double)x - (double)m) * heat); }
__device__ __forceinline__ double vf_weight(float x, float m, double heat) { return vf_power(x, m, heat).value(); }
// What weights are taken by: a largest logit that is no number makes no row.
__device__ __forceinline__ float vf_by(float m) { return m == -INFINITY ? 0.0f : m; }

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
// A wave's 64 PER values of a unit, N neighbours a lane at a time, -inf past the
// vocabulary; every load is asked for before any is looked at.
template <int PER, typename T>
__device__ __forceinline__ void vf_load(const T *row, uint32_t unit, uint32_t vocab, float (&v)[PER]) {
    constexpr int N = VfVec<T>::N;
    const uint32_t at = unit * (64 * PER) + (threadIdx.x & 63) * N;
    if ((unit + 1) * (64 * PER) <= vocab) {  // the same for the whole wave
        typename VfVec<T>::Load w[PER / N];
#pragma unroll
        for (int q = 0; q < PER / N; q++) w[q] = *(const typename VfVec<T>::Load *)(row + at + q * 64 * N);
#pragma unroll
        for (int q = 0; q < PER; q++) v[q] = vf_in(w[q / N].v[q % N]);
    } else {
        T w[PER];
#pragma unroll
        for (int q = 0; q < PER; q++) {
            const uint32_t i = at + q / N * 64 * N + q % N;
            w[q] = row[i < vocab ? i : vocab - 1];
        }
#pragma unroll
        for (int q = 0; q < PER; q++) v[q] = at + q / N * 64 * N + q % N < vocab ? vf_in(w[q]) : -INFINITY;
    }
}

// Over a wave, every lane gets it: rotations within 16 lanes, then swaps of 16
// and 32.
template <int CTRL, typename V>
__device__ __forceinline__ V vf_move(V v) {
    if constexpr (sizeof(V) == 8) {
        const uint64_t b = __builtin_bit_cast(uint64_t, v);
        const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, 0xf, 0xf, true);
        const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), CTRL, 0xf, 0xf, true);
        return __builtin_bit_cast(V, (uint64_t)hi << 32 | lo);
    } else {
        return __builtin_bit_cast(V, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
    }
}
template <bool FAR, typename V>
__device__ __forceinline__ void vf_swap(V v, V &a, V &b) {
    auto swap = [](uint32_t x) {
        if constexpr (FAR) return __builtin_amdgcn_permlane32_swap(x, x, false, false);
        else return __builtin_amdgcn_permlane16_swap(x, x, false, false);
    };
    if constexpr (sizeof(V) == 8) {
        const uint64_t u = __builtin_bit_cast(uint64_t, v);
        const auto lo = swap((uint32_t)u), hi = swap((uint32_t)(u >> 32));
        a = __builtin_bit_cast(V, (uint64_t)hi[0] << 32 | lo[0]);
        b = __builtin_bit_cast(V, (uint64_t)hi[1] << 32 | lo[1]);
    } else {
        const auto w = swap(__builtin_bit_cast(uint32_t, v));
        a = __builtin_bit_cast(V, (uint32_t)w[0]);
        b = __builtin_bit_cast(V, (uint32_t)w[1]);
    }
}
template <typename V, class OP>
__device__ __forceinline__ V vf_wave(V v, OP op) {
    v = op(v, vf_move<0x128>(v));  // row_ror 8, 4, 2, 1
    v = op(v, vf_move<0x124>(v));
    v = op(v, vf_move<0x122>(v));
    v = op(v, vf_move<0x121>(v));
    V a, b;
    vf_swap<false>(v, a, b);
    v = op(a, b);
    vf_swap<true>(v, a, b);
    return op(a, b);
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
// The sum over the wave's lanes up to this one.
__device__ __forceinline__ double vf_running(double v) {
    v += vf_move<0x111>(v);  // row_shr 1, 2, 4, 8: zeros from outside the 16 lanes
    v += vf_move<0x112>(v);
    v += vf_move<0x114>(v);
    v += vf_move<0x118>(v);
    const uint32_t lane = threadIdx.x & 63;
    double before = 0.0;  // what the rows of 16 before this lane's hold
#pragma unroll
    for (int r = 0; r < 3; r++) {
        const uint64_t u = __builtin_bit_cast(uint64_t, v);
        const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)u, 16 * r + 15);
        const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), 16 * r + 15);
        before += (int)(lane >> 4) > r ? __builtin_bit_cast(double, (uint64_t)hi << 32 | lo) : 0.0;
    }
    return v + before;
}
__device__ __forceinline__ double vf_last(double v) {  // lane 63's
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)u, 63);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), 63);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// A wave a unit of a row.
template <typename T, int PER>
__global__ void __launch_bounds__(VF_THREADS) vf_stats(VfArgs a) {
    constexpr int N = VfVec<T>::N;
    const uint32_t lane = threadIdx.x & 63, wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const uint32_t groups = (a.units + VF_WAVES - 1) / VF_WAVES;
    const uint32_t unit = blockIdx.x % groups * VF_WAVES + wave, row = blockIdx.x / groups, i = row / a.rows, r = row % a.rows;
    const bool target = r <= a.k;
    const uint32_t j = target ? r : r - a.k - 1, drafts = vf_given(a, i);  // no fewer than are looked at
    const double heat = vf_heat(a, i);
    if (unit >= a.units || j > drafts || (!target && (j == drafts || heat == 0.0))) return;
    const T *src = target ? (const T *)a.x + ((size_t)i * (a.k + 1) + j) * a.xs : (const T *)a.y + ((size_t)i * a.k + j) * a.ys;
    float v[PER], most = -INFINITY;
    vf_load<PER>(src, unit, a.vocab, v);
    bool nan = false;
#pragma unroll
    for (int q = 0; q < PER; q++) {
        most = fmaxf(most, v[q]);
        nan |= v[q] != v[q];
    }
    const float m = vf_wave(most, VfMax());
    VfPart part{m, 0u, 0.0};
    if (heat == 0.0) {
        uint32_t id = ~0u;
#pragma unroll
        for (int q = PER - 1; q >= 0; q--)
            if (v[q] == m) id = unit * (64 * PER) + lane * N + (q / N) * 64 * N + q % N;
        part.id = vf_wave(id, VfMin());
    } else {
        const float by = vf_by(m);
        double l[2] = {0.0, 0.0};
#pragma unroll
        for (int q = 0; q < PER; q++) {
            const VfPower w = vf_power(v[q], by, heat);
            l[q & 1] = __builtin_fma(w.s, w.f, l[q & 1]);
        }
        part.l = vf_wave(l[0] + l[1], VfAdd());
        if (__ballot(nan) || m == INFINITY) part.l = __builtin_nan("");
    }
    if (lane == 0) a.part[(size_t)row * a.units + unit] = part;
}

// Where request i ends; a whole workgroup, every thread gets it.
struct VfShared {
    float m[VF_ROWS];
    double l[VF_ROWS];
    uint32_t id[VF_MAX_DRAFTS + 1];
};
template <typename T>
__device__ __forceinline__ VfEnd vf_end(const VfArgs &a, uint32_t i, double heat, uint32_t drafts, VfShared &s) {
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    // asked for first: each draft's own logits, a lane a draft
    const bool has = lane < drafts;
    const int32_t d = has ? a.ids[(size_t)i * a.k + lane] : -1;
    const bool known = d >= 0 && (uint32_t)d < a.vocab;
    const float xd = known ? vf_in(((const T *)a.x)[((size_t)i * (a.k + 1) + lane) * a.xs + d]) : 0.0f;
    const float yd = known && a.y ? vf_in(((const T *)a.y)[((size_t)i * a.k + lane) * a.ys + d]) : 0.0f;
    const float u = has ? a.u[(size_t)i * (a.k + 1) + lane] : 0.0f;
    for (uint32_t r = wave; r < a.rows; r += VF_WAVES) {
        const bool target = r <= a.k;
        const uint32_t j = target ? r : r - a.k - 1;
        if (j > drafts || (!target && (j == drafts || heat == 0.0))) continue;
        const VfPart *part = a.part + ((size_t)i * a.rows + r) * a.units;
        VfPart mine{-INFINITY, ~0u, 0.0};
        if (lane < a.units) mine = part[lane];
        float m = mine.m;
        uint32_t id = m > -INFINITY ? mine.id : ~0u;
        for (uint32_t c = lane + 64; c < a.units; c += 64)
            if (part[c].m > m) {  // the first unit of a lane's that has it
                m = part[c].m;
                id = part[c].id;
            }
        const float M = vf_wave(m, VfMax());
        double l = 0.0;
        if (heat == 0.0) {
            id = vf_wave(m == M && M > -INFINITY ? id : ~0u, VfMin());
        } else {
            const float by = vf_by(M);
            l = mine.l * vf_weight(mine.m, by, heat);
            for (uint32_t c = lane + 64; c < a.units; c += 64) l += part[c].l * vf_weight(part[c].m, by, heat);
            l = vf_wave(l, VfAdd());
        }
        if (lane == 0) {
            s.m[r] = M;
            s.l[r] = l;
            if (target) s.id[r] = id == ~0u ? 0u : id;
        }
    }
    __syncthreads();
    bool kept = false;
    if (known) {
        if (heat == 0.0) {
            kept = (uint32_t)d == s.id[lane];
        } else {
            const double p = vf_weight(xd, vf_by(s.m[lane]), heat) / s.l[lane];
            double q = 1.0;
            if (a.y) q = vf_weight(yd, vf_by(s.m[a.k + 1 + lane]), heat) / s.l[a.k + 1 + lane];
            kept = (double)u * q < p;
        }
    }
    const uint64_t stop = ~__ballot(kept);
    uint32_t j = stop ? (uint32_t)__builtin_ctzll(stop) : 64u;
    j = j < drafts ? j : drafts;
    const bool given = a.y && j < drafts && heat != 0.0;
    return VfEnd{j, heat == 0.0 ? s.id[j] : 0u, vf_by(s.m[j]), given ? vf_by(s.m[a.k + 1 + j]) : 0.0f, s.l[j],
                 given ? -log2(s.l[j]) : 0.0, given ? -log2(s.l[a.k + 1 + j]) : 0.0};
}

// max(p - q, 0) at one id, the logarithms of the sums as offsets; 0 where
// either is no number.
struct VfRest {
    float mp, mq;
    double heat, op, oq;
    __device__ __forceinline__ VfRest(const VfEnd &e, double heat)
        : mp(e.mp), mq(e.mq), heat(heat), op(e.op), oq(e.oq) {}
    __device__ __forceinline__ double operator()(float x, float y) const {
        const VfPower p(__builtin_fma((double)x - (double)mp, heat, op));
        const VfPower q(__builtin_fma((double)y - (double)mq, heat, oq));
        return fmax(__builtin_fma(p.s, p.f, -q.value()), 0.0);
    }
};

// A wave a unit of each request's last row.
template <typename T, int PER>
__global__ void __launch_bounds__(VF_THREADS) vf_rest(VfArgs a) {
    __shared__ VfShared s;
    const uint32_t lane = threadIdx.x & 63, groups = (a.units + VF_WAVES - 1) / VF_WAVES, i = blockIdx.x / groups;
    const uint32_t unit = blockIdx.x % groups * VF_WAVES + (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const double heat = vf_heat(a, i);
    const uint32_t drafts = vf_drafts(a, i);
    const VfEnd e = vf_end<T>(a, i, heat, drafts, s);
    if (unit == 0 && lane == 0) a.end[i] = e;
    if (heat == 0.0 || e.row == drafts || unit >= a.units) return;
    const T *x = (const T *)a.x + ((size_t)i * (a.k + 1) + e.row) * a.xs;
    const T *y = (const T *)a.y + ((size_t)i * a.k + e.row) * a.ys;
    const VfRest of(e, heat);
    float xv[PER], yv[PER];
    vf_load<PER>(x, unit, a.vocab, xv);
    vf_load<PER>(y, unit, a.vocab, yv);
    double sum = 0.0;
#pragma unroll
    for (int q = 0; q < PER; q++) sum += of(xv[q], yv[q]);
    sum = vf_wave(sum, VfAdd());
    if (lane == 0) a.rest[(size_t)i * a.units + unit] = sum;
}

// A workgroup a request: every wave looks for the unit, then each takes a
// quarter of its ids.
template <typename T, int PER>
__global__ void __launch_bounds__(VF_THREADS) vf_choose(VfArgs a) {
    constexpr int K = PER / 4;  // ids a thread
    constexpr uint32_t UNIT = 64 * PER;
    __shared__ VfShared s;
    __shared__ double sums[VF_WAVES];
    __shared__ uint32_t firsts[VF_WAVES], lasts[VF_WAVES];
    const uint32_t i = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, drafts = vf_drafts(a, i);
    const double heat = vf_heat(a, i);
    const double number = a.u[(size_t)i * (a.k + 1) + drafts];
    const VfEnd e = a.y ? a.end[i] : vf_end<T>(a, i, heat, drafts, s);
    int32_t token = -1;
    if (heat == 0.0) {
        token = (int32_t)e.greedy;
    } else if (e.lp > 0.0 && e.lp < INFINITY) {
        const T *x = (const T *)a.x + ((size_t)i * (a.k + 1) + e.row) * a.xs;
        const T *y = (const T *)a.y + ((size_t)i * a.k + e.row) * a.ys;
        const VfPart *part = a.part + ((size_t)i * a.rows + e.row) * a.units;
        const double *rest = a.rest + (size_t)i * a.units;
        const VfRest of(e, heat);
        bool less = a.y && e.row < drafts;  // weights max(p - q, 0), otherwise p times its sum
        uint32_t skip = ~0u;                // the id that has none: a draft that was looked up
        if (!a.y && e.row < drafts) skip = (uint32_t)a.ids[(size_t)i * a.k + e.row];
        skip = skip < a.vocab ? skip : ~0u;
        // this thread's weights of a unit, in the order of their ids
        double w[K];
        auto each = [&](uint32_t unit) {
            const uint32_t at = unit * UNIT + tid * K;
            double sum = 0.0;
#pragma unroll
            for (int q = 0; q < K; q++) {
                const bool in = at + q < a.vocab && at + q != skip;
                const float xv = in ? vf_in(x[at + q]) : -INFINITY;
                const float yv = in && less ? vf_in(y[at + q]) : -INFINITY;
                w[q] = less ? of(xv, yv) : vf_weight(xv, e.mp, heat);
                sum += w[q];
            }
            return sum;
        };
        double skipped = 0.0;  // the sum of the unit of skip, without it
        auto of_unit = [&](uint32_t c) {
            if (less) return rest[c];
            if (skip != ~0u && c == skip / UNIT) return skipped;
            return part[c].l * vf_weight(part[c].m, e.mp, heat);
        };
        if (skip != ~0u) {
            const VfPart p = part[skip / UNIT];
            const double all = p.l * vf_weight(p.m, e.mp, heat);
            skipped = all - vf_weight(vf_in(x[skip]), e.mp, heat);
            if (!(skipped > all * 0x1p-20)) {  // little is left, or nothing: the others' own sum
                const double mine = vf_wave(each(skip / UNIT), VfAdd());
                if (lane == 0) sums[wave] = mine;
                __syncthreads();
                skipped = (sums[0] + sums[1]) + (sums[2] + sums[3]);
                __syncthreads();
            }
        }
        double first = lane < a.units ? of_unit(lane) : 0.0, total;
        auto add_up = [&]() {
            double t = first;
            for (uint32_t c = lane + 64; c < a.units; c += 64) t += of_unit(c);
            return vf_wave(t, VfAdd());
        };
        total = add_up();
        if (!(total > 0.0)) {  // p and q are alike to the last place: p
            less = false;
            skip = ~0u;
            first = lane < a.units ? of_unit(lane) : 0.0;
            total = add_up();
        }
        const double want = number * total;
        // the unit: the first whose running sum is above want, or the last with any weight
        double base = 0.0, from = 0.0;
        uint32_t unit = 0, last = 0;
        bool found = false;
        for (uint32_t c0 = 0; c0 < a.units && !found; c0 += 64) {
            const double mine = c0 == 0 ? first : c0 + lane < a.units ? of_unit(c0 + lane) : 0.0;
            const double run = base + vf_running(mine);
            const uint64_t some = __ballot(mine > 0.0), over = __ballot(mine > 0.0 && run > want);
            if (some) last = c0 + 63 - (uint32_t)__builtin_clzll(some);
            if (over) {
                const uint32_t l = (uint32_t)__builtin_ctzll(over);
                found = true;
                unit = c0 + l;
                from = base;
                if (l > 0) {
                    const uint64_t b = __builtin_bit_cast(uint64_t, run);
                    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)b, (int)l - 1);
                    const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(b >> 32), (int)l - 1);
                    from = __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
                }
            }
            base = vf_last(run);
        }
        if (!found) unit = last;
        const double mine = each(unit), run = vf_running(mine);
        if (lane == 63) sums[wave] = run;
        __syncthreads();
        double at = from + (run - mine);
#pragma unroll
        for (uint32_t v = 0; v < VF_WAVES; v++) at += v < wave ? sums[v] : 0.0;
        uint32_t one = ~0u, end = 0u;
#pragma unroll
        for (int q = 0; q < K; q++) {
            at += w[q];
            if (w[q] > 0.0) {
                const uint32_t id = unit * UNIT + tid * K + q;
                if (found && at > want && one == ~0u) one = id;
                end = id + 1;
            }
        }
        one = vf_wave(one, VfMin());
        end = ~vf_wave(~end, VfMin());
        if (lane == 0) {
            firsts[wave] = one;
            lasts[wave] = end;
        }
        __syncthreads();
#pragma unroll
        for (uint32_t v = 0; v < VF_WAVES; v++) {
            one = firsts[v] < one ? firsts[v] : one;
            end = lasts[v] > end ? lasts[v] : end;
        }
        token = (int32_t)(one != ~0u ? one : end - 1);
    }
    if (!(a.limit >> 32)) {
        if (vf_room(a, i) == 0) token = -1;  // e.row is 0
        __syncthreads();                     // every wave has read the position
    }
    const uint32_t got = e.row + (token >= 0 ? 1u : 0u);
    for (uint32_t j = tid; j <= a.k; j += VF_THREADS)
        a.tokens[(size_t)i * (a.k + 1) + j] = j < e.row ? a.ids[(size_t)i * a.k + j] : j == e.row ? token : -1;
    if (tid == 0) {
        a.counts[i] = (int32_t)got;
        if (a.pos) a.pos[i] += got;
    }
}

// Ids a lane: 32, fewer where that leaves SIMDs idle, by the units of 2048 ids
// of all rows (us a call for 8, 16 and 32 a lane, draft logits unless said):
//   looked up, f32: 64 units 7.8 / 8.6 / 10.6, 256 8.0 / 8.8 / 10.9, 315 of one row of 128256 each 11.9 / 10.4 / 10.9
//   448, f32 12.8 / 14.0 / 18.9; 1800, f32 17.9 / 17.6 / 21.2; 2268, bf16 22.4 / 19.6 / 21.1
//   7200, rows of 50021, bf16 31.0 / 27.6 / 28.8; 7938, of 128256, bf16 37.4 / 29.6 / 28.1
//   13600, of 50021, f32 44.2 / 39.1 / 42.4; 13608, of 128256, f32 49.4 / 41.2 / 41.3; 18144, of 128256, f32 77.7 / 57.8 / 54.6
// Rows of 128256 gain from more ids a lane earlier than those of 50021 or 32003;
// the borders stand where neither loses much of what it takes (the lower one is
// late for looked-up rows: 1260 units of 128256 14.3 / 12.2 / 12.6).
static int vf_per(size_t n, size_t k, size_t vocab, bool given) {
    const size_t units = n * (given ? 2 * k + 1 : k + 1) * div_ceil(vocab, 32 * 64);
    return units < 2048 ? 8 : units < 8192 ? 16 : 32;
}
struct VfPlan {
    int per;
    size_t rows, units, o_rest, o_end, bytes;
};
static VfPlan vf_plan(size_t n, size_t k, size_t vocab, bool given) {
    VfPlan p;
    p.per = vf_per(n, k, vocab, given);
    p.rows = given ? 2 * k + 1 : k + 1;
    p.units = div_ceil(vocab, (size_t)p.per * 64);
    p.o_rest = n * p.rows * p.units * sizeof(VfPart);
    p.o_end = p.o_rest + (given ? n * p.units * sizeof(double) : 0);
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
    if (n * p.rows * div_ceil(p.units, VF_WAVES) > 0xFFFFFF)  // a launch is below 2^32 threads
        return fail(QBK_ERR_VALIDATION, "verify_drafts: too many rows for one launch");
    return QBK_OK;
}

template <typename T, int PER>
static void vf_go(const VfArgs &a, hipStream_t s) {
    const uint32_t groups = (a.units + VF_WAVES - 1) / VF_WAVES;
    hipLaunchKernelGGL((vf_stats<T, PER>), dim3(a.n * a.rows * groups), dim3(VF_THREADS), 0, s, a);
    if (a.y) hipLaunchKernelGGL((vf_rest<T, PER>), dim3(a.n * groups), dim3(VF_THREADS), 0, s, a);
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
    return qbk_verify_drafts_within_dev(ctx, logits, draft_logits, dtype, n, k, vocab, row_stride, draft_row_stride, ids,
                                        n_drafts, uniforms, temperature, tokens, counts, pos, SIZE_MAX, workspace,
                                        workspace_size, stream);
}

int qbk_verify_drafts_within_dev(qbk_ctx *ctx, const void *logits, const void *draft_logits, int dtype, size_t n,
                                 size_t k, size_t vocab, size_t row_stride, size_t draft_row_stride, const int32_t *ids,
                                 const uint32_t *n_drafts, const float *uniforms, const float *temperature,
                                 int32_t *tokens, int32_t *counts, uint32_t *pos, size_t pos_limit, void *workspace,
                                 size_t workspace_size, void *stream) {
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
    if (pos_limit >> 32 == 0 && !pos) return fail(QBK_ERR_VALIDATION, "verify_drafts: a limit of positions without positions");
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
    a.limit = pos_limit >> 32 ? 1ull << 32 : pos_limit;
    a.part = (VfPart *)workspace;
    a.rest = (double *)((char *)workspace + p.o_rest);
    a.end = (VfEnd *)((char *)workspace + p.o_end);
    a.n = (uint32_t)n;
    a.k = (uint32_t)k;
    a.rows = (uint32_t)p.rows;
    a.vocab = (uint32_t)vocab;
    a.units = (uint32_t)p.units;
    hipStream_t s = (hipStream_t)stream;
    if (dtype == QBK_F32) p.per == 8 ? vf_go<float, 8>(a, s) : p.per == 16 ? vf_go<float, 16>(a, s) : vf_go<float, 32>(a, s);
    else p.per == 8 ? vf_go<uint16_t, 8>(a, s) : p.per == 16 ? vf_go<uint16_t, 16>(a, s) : vf_go<uint16_t, 32>(a, s);
    QBK_HIP(hipGetLastError());
    return QBK_OK;
}

}  // extern "C"
