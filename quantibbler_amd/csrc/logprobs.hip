// logprobs.hip -- log probabilities of given tokens, their distribution's
// entropy and its likeliest tokens, in one pass over the logits.
//
// A row is cut into chunks of 8192 logits, a workgroup each, held in
// registers: m = max x, l = sum exp(x - m), t = sum exp(x - m) (x - m), and the
// chunk's top_k as 64-bit keys (value, then lower id first).  A second launch
// joins a row's chunks:
//   log p = (x - M) - log l,   entropy = log l - t / l
// (t moves from m to M as t' = f (t + (m - M) l), f = exp(m - M)).
//
// The top_k of a chunk: the k-th largest of the 256 threads' own largest keys
// is no larger than the chunk's k-th, and only k threads hold anything above
// it, so what is left to order is at most 32 k keys and mostly little past k.
#include <math.h>

#include "qbk_internal.h"

#pragma clang fp contract(off)

namespace qbk {

#define LP_THREADS 256
#define LP_PER 32
#define LP_CHUNK (LP_THREADS * LP_PER)
#define LP_MAX_TOP 64

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

// A key that orders as (value, lower id first); above 0 for every logit.
__device__ __forceinline__ uint64_t lp_key(float x, uint32_t id) {
    x = x != x ? -INFINITY : x + 0.0f;  // -0 ties with 0
    const uint32_t b = __float_as_uint(x);
    return (uint64_t)(b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u)) << 32 | (uint32_t)~id;
}
__device__ __forceinline__ float lp_key_value(uint64_t key) {
    const uint32_t b = (uint32_t)(key >> 32);
    return __uint_as_float(b ^ (b >> 31 ? 0x80000000u : 0xFFFFFFFFu));
}

__device__ __forceinline__ float lp_exp(float d) { return __builtin_amdgcn_exp2f(d * 1.4426950408889634f); }

template <typename T>
struct LpVec {
    struct __attribute__((packed, aligned(sizeof(T)))) Load {
        T v[16 / sizeof(T)];
    };
};
__device__ __forceinline__ float lp_in(float x) { return x; }
__device__ __forceinline__ float lp_in(uint16_t x) { return bf16_to_f32(x); }

// Sum / largest over the workgroup; every thread gets it.  red: a float a wave.
template <class OP>
__device__ __forceinline__ float lp_reduce(float v, float *red, OP op) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v = op(v, __shfl_xor(v, o, 64));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int w = 1; w < LP_THREADS / 64; w++) v = op(v, red[w]);
    return v;
}

// The `top` largest of n distinct keys in LDS, in order, into out (0 where
// there are fewer).
__device__ __forceinline__ void lp_order(const uint64_t *key, uint32_t n, uint32_t top, uint64_t *out) {
    for (uint32_t i = threadIdx.x; i < n; i += LP_THREADS) {
        const uint64_t mine = key[i];
        uint32_t rank = 0;
        for (uint32_t j = 0; j < n; j++) rank += key[j] > mine;
        if (rank < top) out[rank] = mine;
    }
    for (uint32_t i = n + threadIdx.x; i < top; i += LP_THREADS) out[i] = 0;
}

template <typename T>
__global__ void __launch_bounds__(LP_THREADS) lp_chunk(LpArgs a) {
    __shared__ float red[LP_THREADS / 64];
    __shared__ uint64_t best[LP_THREADS];
    __shared__ uint64_t cand[LP_MAX_TOP * LP_PER];
    __shared__ uint32_t count;
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
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < LP_PER; j++) m = fmaxf(m, v[j]);
    m = lp_reduce(m, red, [](float p, float q) { return fmaxf(p, q); });
    const float from = m == -INFINITY ? 0.0f : m;  // a chunk of nothing but -inf adds nothing (a NaN stays one)
    float l = 0.0f, t = 0.0f;
#pragma unroll
    for (int j = 0; j < LP_PER; j++) {
        const float d = v[j] - from, e = lp_exp(d);
        l += e;
        t += d == -INFINITY ? 0.0f : e * d;
    }
    l = lp_reduce(l, red, [](float p, float q) { return p + q; });
    t = lp_reduce(t, red, [](float p, float q) { return p + q; });
    if (tid == 0) a.part[blockIdx.x] = float4{m, l, t, 0.0f};
    if (a.top == 0) return;

    auto id = [&](int j) { return base + ((j / V) * LP_THREADS + tid) * V + j % V; };
    uint64_t mine = 0;
#pragma unroll
    for (int j = 0; j < LP_PER; j++)
        if (id(j) < a.vocab) {
            const uint64_t k = lp_key(v[j], id(j));
            mine = k > mine ? k : mine;
        }
    best[tid] = mine;
    if (tid == 0) count = 0;
    __syncthreads();
    uint32_t rank = 0;
    for (int j = 0; j < LP_THREADS; j++) rank += best[j] > mine;
    if (tid == 0) bar = 1;  // fewer threads with a logit than top: everything is above it
    __syncthreads();
    if (mine && rank == a.top - 1) bar = mine;
    __syncthreads();
    if (mine >= bar) {
        const uint64_t least = bar;
#pragma unroll
        for (int j = 0; j < LP_PER; j++)
            if (id(j) < a.vocab) {
                const uint64_t k = lp_key(v[j], id(j));
                if (k >= least) cand[atomicAdd(&count, 1u)] = k;
            }
    }
    __syncthreads();
    lp_order(cand, count, a.top, a.keys + (size_t)blockIdx.x * a.top);
}

// A workgroup a row: the chunks' statistics and keys.
template <typename T>
__global__ void __launch_bounds__(LP_THREADS) lp_join(LpArgs a) {
    __shared__ float red[LP_THREADS / 64];
    __shared__ uint64_t cand[LP_MAX_TOP * LP_PER];
    __shared__ uint64_t first[LP_MAX_TOP];
    const uint32_t row = blockIdx.x, tid = threadIdx.x;
    const float4 *part = a.part + (size_t)row * a.chunks;
    float M = -INFINITY;
    for (uint32_t c = tid; c < a.chunks; c += LP_THREADS) M = fmaxf(M, part[c].x);
    M = lp_reduce(M, red, [](float p, float q) { return fmaxf(p, q); });
    float l = 0.0f, t = 0.0f;
    for (uint32_t c = tid; c < a.chunks; c += LP_THREADS) {
        const float4 p = part[c];
        if (p.x == -INFINITY && p.y == 0.0f) continue;
        const float d = p.x - M, f = lp_exp(d);
        l += p.y * f;
        t += f == 0.0f ? 0.0f : f * (p.z + d * p.y);  // d l may pass f32 where f is 0
    }
    l = lp_reduce(l, red, [](float p, float q) { return p + q; });
    t = lp_reduce(t, red, [](float p, float q) { return p + q; });
    const float lse = logf(l);  // on M
    const float nan = __builtin_nanf("");
    const bool ok = l > 0.0f && l < INFINITY;
    if (tid == 0) {
        if (a.entropy) a.entropy[row] = ok ? lse - t / l : nan;
        if (a.logprobs) {
            const int32_t id = a.targets[row];
            const bool in = id >= 0 && (uint32_t)id < a.vocab;
            a.logprobs[row] = ok && in ? (lp_in(((const T *)a.x)[(size_t)row * a.stride + id]) - M) - lse : nan;
        }
    }
    if (a.top == 0) return;
    // batches of keys that fit, the best so far among them
    const uint64_t *keys = a.keys + (size_t)row * a.chunks * a.top;
    const uint64_t all = (uint64_t)a.chunks * a.top;
    uint32_t kept = 0;
    for (uint64_t at = 0; at < all;) {
        const uint32_t room = LP_MAX_TOP * LP_PER - kept, take = all - at < room ? (uint32_t)(all - at) : room;
        // the last chunk may be short of logits and leave zeros: the first batch holds a whole chunk's (or, of one
        // chunk, the row's) keys, so every zero ranks past `top`
        for (uint32_t i = tid; i < take; i += LP_THREADS) cand[kept + i] = keys[at + i];
        __syncthreads();
        lp_order(cand, kept + take, a.top, first);
        __syncthreads();
        at += take;
        kept = 0;
        if (at < all) {
            for (uint32_t i = tid; i < a.top; i += LP_THREADS) cand[i] = first[i];
            kept = a.top;
        }
        __syncthreads();
    }
    for (uint32_t i = tid; i < a.top; i += LP_THREADS) {
        const uint64_t k = first[i];
        const uint32_t id = ~(uint32_t)k;
        a.top_ids[(size_t)row * a.top + i] = (int32_t)id;
        a.top_logprobs[(size_t)row * a.top + i] = ok ? (lp_key_value(k) - M) - lse : nan;
    }
}

static size_t lp_bytes(size_t rows, size_t vocab, size_t top) {
    return round_up(rows * div_ceil(vocab, LP_CHUNK) * (sizeof(float4) + 8 * top), 256);
}

static int lp_check(size_t rows, size_t vocab, size_t top) {
    if (vocab == 0 || vocab > 0x7FFFFFFFull) return fail(QBK_ERR_VALIDATION, "logprobs needs 1 <= vocab < 2^31");
    if (top > LP_MAX_TOP || top > vocab)
        return fail(QBK_ERR_VALIDATION, fmt("logprobs top_k must be at most %d and the vocabulary of %zu, got %zu",
                                            LP_MAX_TOP, vocab, top));
    if (rows > 0x7FFFFFFFull || rows * div_ceil(vocab, LP_CHUNK) > 0x7FFFFFFFull)
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
    if (!workspace || workspace_size < need)
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
    if (dtype == QBK_F32) {
        hipLaunchKernelGGL((lp_chunk<float>), grid, block, 0, s, a);
        hipLaunchKernelGGL((lp_join<float>), rgrid, block, 0, s, a);
    } else {
        hipLaunchKernelGGL((lp_chunk<uint16_t>), grid, block, 0, s, a);
        hipLaunchKernelGGL((lp_join<uint16_t>), rgrid, block, 0, s, a);
    }
    QBK_HIP(hipGetLastError());
    return QBK_OK;
}

}  // extern "C"
