// logprobs.hip -- log probabilities of given tokens, their distribution's
// entropy and its likeliest tokens, in one pass over the logits.
//
// A row is cut into chunks of 8192 logits, a workgroup each, held in
// registers: m = max x, l = sum exp(x - m), t = sum exp(x - m) (x - m), and the
// chunk's top_k as 64-bit keys (value, then lower id first).  A second launch
// joins a row's chunks; a row of one chunk is finished by the first (32 x 8192
// 6.6 us, joined all the same 10.0; 2048 x 1000 14.2 and 19.1):
//   log p = (x - M) - log l,   entropy = log l - t / l
// (t moves from m to M as t' = f (t + (m - M) l), f = exp(m - M)).
//
// The top_k of a chunk: of the 64 threads of a wave, k hold a value at or above
// the k-th largest of their own largest values, so the largest such bound of
// the four waves is no more than the chunk's k-th largest value, and what is
// left to order is mostly little past k.  Where ties leave more than fit (a row
// of few different values) the same is done once more on keys of value and id,
// which all differ: only k threads hold keys above the k-th largest of theirs.
//
// Many rows are bound by memory: 2048 x 128256 f32, 1.05 GB in 179 us, 5.9 TB/s.
// One row of 128256 is bound by two dependent launches, 9.3 to 10.1 and 5.8 us,
// the first of sixteen workgroups: a chunk is 8192 logits whatever the call.
#include <math.h>

#include <type_traits>

#include "qbk_internal.h"

#pragma clang fp contract(off)

namespace qbk {

#define LP_THREADS 256
#define LP_PER 32
#define LP_CHUNK (LP_THREADS * LP_PER)
#define LP_MAX_TOP 64
#define LP_CAND (LP_MAX_TOP * LP_PER)  // keys that fit in LDS

struct LpArgs {
    const void *x;
    size_t stride;
    uint32_t vocab, chunks, top;
    const int32_t *targets;
    float *logprobs, *entropy;
    int32_t *top_ids;
    float *top_logprobs;
    float4 *part;     // [row][chunk] m, l, t
    uint64_t *keys;   // [row][chunk][top]
};

// A float's bits as an unsigned number of the same order, and back.
__device__ __forceinline__ uint32_t lp_rank(float x) {
    const uint32_t b = __float_as_uint(x);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float lp_unrank(uint32_t b) {
    return __uint_as_float(b ^ (b >> 31 ? 0x80000000u : 0xFFFFFFFFu));
}

// A key that orders as (value, lower id first); above 0 for every logit.
__device__ __forceinline__ uint64_t lp_key(float x, uint32_t id) {
    x = x != x ? -INFINITY : x + 0.0f;  // -0 ties with 0
    return (uint64_t)lp_rank(x) << 32 | (uint32_t)~id;
}

// exp(d), d <= 0 or NaN: d log2(e) in two parts, the second as a factor, so
// that far terms keep their last places (one rounded product is off by |d| of
// them).  Below -1000 the result is 0 and e d is 0 as well, -inf included.
__device__ __forceinline__ float lp_exp(float &d) {
    d = d < -1000.0f ? -1000.0f : d;
    const float p = d * 1.44269502f, r = __builtin_fmaf(d, 1.92596303e-8f, __builtin_fmaf(d, 1.44269502f, -p));
    const float e = __builtin_amdgcn_exp2f(p);
    return __builtin_fmaf(e, r * 0.693147182f, e);
}

template <typename T>
struct LpVec {
    struct __attribute__((packed, aligned(sizeof(T)))) Load {
        T v[16 / sizeof(T)];
    };
};
__device__ __forceinline__ float lp_in(float x) { return x; }
__device__ __forceinline__ float lp_in(uint16_t x) { return bf16_to_f32(x); }

// Over a wave, every lane gets it: rotations within 16 lanes, then swaps of 16
// and 32 (a dozen cycles each where a permute through LDS takes a hundred).
template <class OP>
__device__ __forceinline__ float lp_wave(float v, OP op) {
    auto turn = [](float x, auto ctrl) {
        return __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), decltype(ctrl)::value,
                                                                     0xf, 0xf, true));
    };
    v = op(v, turn(v, std::integral_constant<int, 0x128>{}));  // row_ror 8, 4, 2, 1
    v = op(v, turn(v, std::integral_constant<int, 0x124>{}));
    v = op(v, turn(v, std::integral_constant<int, 0x122>{}));
    v = op(v, turn(v, std::integral_constant<int, 0x121>{}));
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = op(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return op(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
// Over the workgroup; red: a float a wave, not in use by a reduction before.
__device__ __forceinline__ float lp_max(float v, float *red) {
    v = lp_wave(v, [](float p, float q) { return fmaxf(p, q); });
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int w = 1; w < LP_THREADS / 64; w++) v = fmaxf(v, red[w]);
    return v;
}
__device__ __forceinline__ float2 lp_sum(float x, float y, float2 *red) {
    auto add = [](float p, float q) { return p + q; };
    x = lp_wave(x, add);
    y = lp_wave(y, add);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = float2{x, y};
    __syncthreads();
    float2 s = red[0];
#pragma unroll
    for (int w = 1; w < LP_THREADS / 64; w++) s = float2{s.x + red[w].x, s.y + red[w].y};
    return s;
}

// The `top` largest of n distinct keys in LDS, in order, into out (0 where
// there are fewer).  The keys are followed by room for seven more.
__device__ __forceinline__ void lp_order(uint64_t *key, uint32_t n, uint32_t top, uint64_t *out) {
    if (threadIdx.x < 7) key[n + threadIdx.x] = 0;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < n; i += LP_THREADS) {
        const uint64_t mine = key[i];
        uint32_t rank = 0;
        for (uint32_t j = 0; j < n; j += 8) {
            uint64_t k[8];
#pragma unroll
            for (int e = 0; e < 8; e++) k[e] = key[j + e];
#pragma unroll
            for (int e = 0; e < 8; e++) rank += k[e] > mine;
        }
        if (rank < top) out[rank] = mine;
    }
    for (uint32_t i = n + threadIdx.x; i < top; i += LP_THREADS) out[i] = 0;
}

// The k-th largest of a wave's 64 values (k <= 64), bit by bit.
__device__ __forceinline__ uint32_t lp_kth(uint32_t v, uint32_t k) {
    uint32_t t = 0;
#pragma unroll
    for (int b = 31; b >= 0; b--) {
        const uint32_t up = t | 1u << b;
        t = (uint32_t)__popcll(__ballot(v >= up)) >= k ? up : t;
    }
    return t;
}

// The rest of a row, of its statistics (sums l and t on M), target and ordered keys; a whole workgroup.
template <typename T>
__device__ __forceinline__ void lp_finish(const LpArgs &a, uint32_t row, float M, float l, float t, bool in,
                                          float target, const uint64_t *first) {
    const float lse = logf(l), nan = __builtin_nanf("");
    const bool ok = l > 0.0f && l < INFINITY;
    if (threadIdx.x == 0) {
        if (a.entropy) a.entropy[row] = ok ? lse - t / l : nan;
        if (a.logprobs) a.logprobs[row] = ok && in ? (target - M) - lse : nan;
    }
    for (uint32_t i = threadIdx.x; i < a.top; i += LP_THREADS) {
        const uint64_t k = first[i];
        a.top_ids[(size_t)row * a.top + i] = (int32_t)~(uint32_t)k;
        a.top_logprobs[(size_t)row * a.top + i] = ok ? (lp_unrank((uint32_t)(k >> 32)) - M) - lse : nan;
    }
}
// Whether the row has a target, and its logit.
template <typename T>
__device__ __forceinline__ float lp_target(const LpArgs &a, uint32_t row, bool &in) {
    const int32_t id = a.logprobs ? a.targets[row] : -1;
    in = id >= 0 && (uint32_t)id < a.vocab;
    return lp_in(((const T *)a.x)[(size_t)row * a.stride + (in ? id : 0)]);
}

template <typename T>
__global__ void __launch_bounds__(LP_THREADS) lp_chunk(LpArgs a) {
    __shared__ float red[LP_THREADS / 64];
    __shared__ float2 red2[LP_THREADS / 64];
    __shared__ uint64_t best[LP_THREADS];
    __shared__ uint64_t cand[LP_CAND + 8];
    __shared__ uint32_t count, bounds[LP_THREADS / 64];
    __shared__ uint64_t bar;
    constexpr int V = 16 / sizeof(T), LOADS = LP_PER / V;
    const uint32_t row = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks, tid = threadIdx.x;
    const T *x = (const T *)a.x + (size_t)row * a.stride;
    const uint32_t base = chunk * LP_CHUNK;
    float v[LP_PER];
#pragma unroll
    for (int j = 0; j < LOADS; j++) {
        const uint32_t i = base + (j * LP_THREADS + tid) * V;
        if (i + V <= a.vocab) {
            const auto w = *(const typename LpVec<T>::Load *)(x + i);
#pragma unroll
            for (int e = 0; e < V; e++) v[j * V + e] = lp_in(w.v[e]);
        } else {
#pragma unroll
            for (int e = 0; e < V; e++) v[j * V + e] = i + e < a.vocab ? lp_in(x[i + e]) : -INFINITY;
        }
    }
    float most = -INFINITY;
#pragma unroll
    for (int j = 0; j < LP_PER; j++) most = fmaxf(most, v[j]);
    if (a.top > 1) {
        const uint32_t bound = lp_kth(lp_rank(most + 0.0f), a.top);
        if ((tid & 63) == 0) bounds[tid >> 6] = bound;
    }
    if (tid == 0) count = 0;
    const float m = lp_max(most, red);
    const float from = m == -INFINITY ? 0.0f : m;  // a chunk of nothing but -inf adds nothing (a NaN stays one)
    float l[2] = {0.0f, 0.0f}, t[2] = {0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < LP_PER; j++) {
        float d = v[j] - from;
        const float e = lp_exp(d);
        l[j & 1] += e;
        t[j & 1] = __builtin_fmaf(e, d, t[j & 1]);
    }
    const float2 sum = lp_sum(l[0] + l[1], t[0] + t[1], red2);
    const bool whole = a.chunks == 1;  // the row is this chunk: no second launch
    bool in = false;
    float target = 0.0f;
    if (whole) target = lp_target<T>(a, row, in);
    else if (tid == 0) a.part[blockIdx.x] = float4{m, sum.x, sum.y, 0.0f};
    if (a.top == 0) {
        if (whole) lp_finish<T>(a, row, m, sum.x, sum.y, in, target, nullptr);
        return;
    }

    auto id = [&](int j) { return base + ((j / V) * LP_THREADS + tid) * V + j % V; };
    auto take = [&](uint64_t k) {
        const uint32_t at = atomicAdd(&count, 1u);
        if (at < LP_CAND) cand[at] = k;
    };
    float least = m;
    if (a.top > 1) {
        uint32_t b = bounds[0];
#pragma unroll
        for (int w = 1; w < LP_THREADS / 64; w++) b = bounds[w] > b ? bounds[w] : b;
        least = lp_unrank(b);
    }
    // NaN counts as -inf, which is only asked for where nothing above it is left
    if (most >= least)
#pragma unroll
        for (int j = 0; j < LP_PER; j++)
            if ((v[j] >= least || least == -INFINITY) && id(j) < a.vocab) take(lp_key(v[j], id(j)));
    __syncthreads();
    if (count > LP_CAND) {
        __syncthreads();
        if (tid == 0) {
            count = 0;
            bar = 1;  // fewer threads with a logit than top: everything is above it
        }
        uint64_t mine = 0;
#pragma unroll
        for (int j = 0; j < LP_PER; j++)
            if (id(j) < a.vocab) {
                const uint64_t k = lp_key(v[j], id(j));
                mine = k > mine ? k : mine;
            }
        best[tid] = mine;
        __syncthreads();
        uint32_t rank = 0;
        for (int j = 0; j < LP_THREADS; j++) rank += best[j] > mine;
        if (mine && rank == a.top - 1) bar = mine;
        __syncthreads();
        const uint64_t floor = bar;
        if (mine >= floor)
#pragma unroll
            for (int j = 0; j < LP_PER; j++)
                if (id(j) < a.vocab) {
                    const uint64_t k = lp_key(v[j], id(j));
                    if (k >= floor) take(k);
                }
        __syncthreads();
    }
    lp_order(cand, count, a.top, whole ? best : a.keys + (size_t)blockIdx.x * a.top);
    if (!whole) return;
    __syncthreads();
    lp_finish<T>(a, row, m, sum.x, sum.y, in, target, best);
}

// A workgroup a row: the chunks' statistics and keys.
template <typename T>
__global__ void __launch_bounds__(LP_THREADS) lp_join(LpArgs a) {
    __shared__ float red[LP_THREADS / 64];
    __shared__ float2 red2[LP_THREADS / 64];
    __shared__ uint64_t cand[LP_CAND + 8];
    __shared__ uint64_t first[LP_MAX_TOP];
    __shared__ uint64_t floors[LP_THREADS / 64];
    __shared__ uint32_t count;
    const uint32_t row = blockIdx.x, tid = threadIdx.x;
    const float4 *part = a.part + (size_t)row * a.chunks;
    // asked for first: the chunks' last keys, the first four keys of every thread and the target's logit
    const uint64_t *keys = a.keys + (size_t)row * a.chunks * a.top;
    uint64_t floor = 1;  // above the zeros of a chunk short of logits
    if (a.top)
        for (uint32_t c = tid; c < a.chunks; c += LP_THREADS) {
            const uint64_t k = keys[(size_t)c * a.top + a.top - 1];
            floor = k > floor ? k : floor;
        }
    const uint64_t all = (uint64_t)a.chunks * a.top;
    uint64_t early[4];
#pragma unroll
    for (int e = 0; e < 4; e++) early[e] = tid + LP_THREADS * e < all ? keys[tid + LP_THREADS * e] : 0;
    bool in;
    const float target = lp_target<T>(a, row, in);
    float M = -INFINITY;
    for (uint32_t c = tid; c < a.chunks; c += LP_THREADS) M = fmaxf(M, part[c].x);
    M = lp_max(M, red);
    float l = 0.0f, t = 0.0f;
    for (uint32_t c = tid; c < a.chunks; c += LP_THREADS) {
        const float4 p = part[c];
        if (p.x == -INFINITY && p.y == 0.0f) continue;
        float d = p.x - M;
        const float f = lp_exp(d);
        l += p.y * f;
        t += f == 0.0f ? 0.0f : f * (p.z + d * p.y);  // d l may pass f32 where f is 0
    }
    const float2 sum = lp_sum(l, t, red2);
    l = sum.x;
    t = sum.y;
    if (a.top == 0) {
        lp_finish<T>(a, row, M, l, t, in, target, first);
        return;
    }
    // The largest last key of a chunk's list is no more than the row's last: what lies at or above it is ordered, in
    // batches where it does not fit, the best so far among them.
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
        const uint64_t k = (uint64_t)__shfl_xor((unsigned long long)floor, o, 64);
        floor = k > floor ? k : floor;
    }
    if ((tid & 63) == 0) floors[tid >> 6] = floor;
    if (tid == 0) count = 0;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < LP_THREADS / 64; w++) floor = floors[w] > floor ? floors[w] : floor;
    constexpr uint32_t BATCH = LP_CAND - LP_MAX_TOP;
    static_assert(BATCH >= 4 * LP_THREADS, "the early keys are of the first batch");
#pragma unroll
    for (int e = 0; e < 4; e++)
        if (early[e] >= floor) cand[atomicAdd(&count, 1u)] = early[e];
    for (uint64_t at = 0; at < all; at += BATCH) {
        for (uint64_t i = at + tid + (at ? 0 : 4 * LP_THREADS); i < all && i < at + BATCH; i += LP_THREADS) {
            const uint64_t k = keys[i];
            if (k >= floor) cand[atomicAdd(&count, 1u)] = k;
        }
        __syncthreads();
        lp_order(cand, count, a.top, first);
        __syncthreads();
        if (at + BATCH < all) {  // the next batch begins with the best so far
            uint32_t kept = count < a.top ? count : a.top;
            __syncthreads();
            for (uint32_t i = tid; i < kept; i += LP_THREADS) cand[i] = first[i];
            if (tid == 0) count = kept;
            __syncthreads();
        }
    }
    lp_finish<T>(a, row, M, l, t, in, target, first);
}

static size_t lp_bytes(size_t rows, size_t vocab, size_t top) {
    if (vocab <= LP_CHUNK) return 0;  // a row is one chunk, done in one launch
    return round_up(rows * div_ceil(vocab, LP_CHUNK) * (sizeof(float4) + 8 * top), 256);
}

static int lp_check(size_t rows, size_t vocab, size_t top) {
    if (vocab == 0 || vocab > 0x7FFFFFFFull) return fail(QBK_ERR_VALIDATION, "logprobs needs 1 <= vocab < 2^31");
    if (top > LP_MAX_TOP || top > vocab)
        return fail(QBK_ERR_VALIDATION, fmt("logprobs top_k must be at most %d and the vocabulary of %zu, got %zu",
                                            LP_MAX_TOP, vocab, top));
    if (rows > 0xFFFFFF || rows * div_ceil(vocab, LP_CHUNK) > 0xFFFFFF)  // a launch is below 2^32 threads
        return fail(QBK_ERR_VALIDATION, "logprobs: too many rows for one launch");
    return QBK_OK;
}

}  // namespace qbk

using namespace qbk;

extern "C" {

size_t qbk_logprobs_workspace_size(size_t rows, size_t vocab, size_t top_k) {
    return lp_check(rows, vocab, top_k) ? 0 : lp_bytes(rows, vocab, top_k);
}

int qbk_logprobs_dev(qbk_ctx *ctx, const void *logits, int dtype, size_t rows, size_t vocab, size_t row_stride,
                     const int32_t *targets, float *logprobs, float *entropy, size_t top_k, int32_t *top_ids,
                     float *top_logprobs, void *workspace, size_t workspace_size, void *stream) {
    int rc;
    if ((rc = lp_check(rows, vocab, top_k))) return rc;
    if (dtype != QBK_F32 && dtype != QBK_BF16)
        return fail(QBK_ERR_VALIDATION, fmt("logprobs takes float32 or bfloat16 logits (dtype %d)", dtype));
    if (rows > 1 && (row_stride < vocab || row_stride > ((size_t)1 << 40)))
        return fail(QBK_ERR_VALIDATION, fmt("row_stride %zu does not fit rows of %zu logits", row_stride, vocab));
    if (!targets != !logprobs) return fail(QBK_ERR_VALIDATION, "logprobs: targets and logprobs come together");
    if (top_k && (!top_ids || !top_logprobs))
        return fail(QBK_ERR_VALIDATION, "logprobs: top_k needs top_ids and top_logprobs");
    if (rows == 0) return QBK_OK;
    if (!logits) return fail(QBK_ERR_VALIDATION, "null argument");
    const size_t need = lp_bytes(rows, vocab, top_k);
    if (need && (!workspace || workspace_size < need))
        return fail(QBK_ERR_VALIDATION, fmt("logprobs workspace of %zu bytes is smaller than the %zu needed",
                                            workspace ? workspace_size : (size_t)0, need));
    if ((uintptr_t)workspace & 15) return fail(QBK_ERR_VALIDATION, "logprobs workspace must be 16-byte aligned");
    if ((rc = bind(ctx))) return rc;
    LpArgs a{};
    a.x = logits;
    a.stride = row_stride;
    a.vocab = (uint32_t)vocab;
    a.chunks = (uint32_t)div_ceil(vocab, LP_CHUNK);
    a.top = (uint32_t)top_k;
    a.targets = targets;
    a.logprobs = logprobs;
    a.entropy = entropy;
    a.top_ids = top_ids;
    a.top_logprobs = top_logprobs;
    a.part = (float4 *)workspace;
    a.keys = (uint64_t *)(a.part + rows * a.chunks);
    const dim3 grid((unsigned)(rows * a.chunks)), rgrid((unsigned)rows), block(LP_THREADS);
    hipStream_t s = (hipStream_t)stream;
    hipLaunchKernelGGL(dtype == QBK_F32 ? lp_chunk<float> : lp_chunk<uint16_t>, grid, block, 0, s, a);
    if (a.chunks > 1) hipLaunchKernelGGL(dtype == QBK_F32 ? lp_join<float> : lp_join<uint16_t>, rgrid, block, 0, s, a);
    QBK_HIP(hipGetLastError());
    return QBK_OK;
}

}  // extern "C"
