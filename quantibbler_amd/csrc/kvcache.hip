// kvcache.hip -- the 8-bit KV cache's rows in and out: quantised as they are
// written, one f32 scale a row and kv head, and read back as values.
//
//   A = max(max |x|, 2^-100), L = 127 (int8) or 448 (e4m3)
//   scale = A (1 / L),  code = nearest(x (L (1 / A))),  value = code * scale
//
// each product and reciprocal rounded to f32.  The floor on A keeps L / A and
// every scale a normal number.  Both kernels
// are one pass over rows and codes, bound by memory (a few rows: by the launch).
#include <math.h>

#include "kvcache.h"

#pragma clang fp contract(off)

namespace qbk {

int kv_check_shape(const qbk_kv_shape *s, size_t *bytes) {
    if (!s) return fail(QBK_ERR_VALIDATION, "null shape");
    if (s->format != QBK_KV_INT8 && s->format != QBK_KV_FP8)
        return fail(QBK_ERR_VALIDATION, fmt("kv cache format must be int8 (0) or fp8 (1), got %d", s->format));
    if (s->n_seqs == 0 || s->capacity == 0 || s->n_kv_heads == 0)
        return fail(QBK_ERR_VALIDATION, "kv cache requires non-empty sequences, capacity and heads");
    if (s->head_dim == 0 || s->head_dim % 16 != 0 || s->head_dim > 256)
        return fail(QBK_ERR_VALIDATION, fmt("kv cache head_dim must be a multiple of 16 up to 256, got %zu",
                                            s->head_dim));
    if (s->capacity > 0x7FFFFF00u || s->n_seqs > 0x7FFFFFFFu || s->n_kv_heads > 0x7FFFFFFFu)
        return fail(QBK_ERR_VALIDATION, "kv cache sizes must be below 2^31");
    // 64-bit throughout: at most 2^31 * 2^31 slabs before the check below
    const unsigned __int128 rows = (unsigned __int128)s->n_seqs * s->n_kv_heads * round_up(s->capacity, 64);
    const unsigned __int128 total = rows * (2 * (s->head_dim + 4));
    if (total > ((unsigned __int128)1 << 48)) return fail(QBK_ERR_VALIDATION, "kv cache of more than 2^48 bytes");
    *bytes = (size_t)total;
    return QBK_OK;
}

KvView kv_view(const qbk_kv_shape *s, const void *cache) {
    KvView v;
    v.cap = s->capacity;
    v.cap64 = round_up(s->capacity, 64);
    v.n_seqs = (uint32_t)s->n_seqs;
    v.Hk = (uint32_t)s->n_kv_heads;
    v.hd = (uint32_t)s->head_dim;
    const size_t rows = s->n_seqs * s->n_kv_heads * v.cap64;
    v.k = (uint8_t *)const_cast<void *>(cache);
    v.v = v.k + rows * v.hd;
    v.ks = (float *)(v.v + rows * v.hd);
    v.vs = v.ks + rows;
    return v;
}

struct KvRows {
    KvView c;
    const uint32_t *row_start, *pos;  // row_start null: `per` rows a sequence
    size_t stride;                    // values from one row to the next
    uint32_t n_rows, n, per, first;
};

// The sequence (0 .. n - 1) and position of row r; false for a row that no
// sequence claims or that lies past the capacity.  Whatever row_start holds,
// a row that passes addresses the cache in bounds.
__device__ __forceinline__ bool kv_place(const KvRows &a, uint32_t r, uint32_t &seq, size_t &at) {
    uint32_t s, start;
    if (a.row_start) {
        uint32_t lo = 0, hi = a.n;  // the last s with row_start[s] <= r
        while (hi - lo > 1) {
            const uint32_t mid = lo + (hi - lo) / 2;
            if (a.row_start[mid] <= r) lo = mid;
            else hi = mid;
        }
        s = lo;
        start = a.row_start[s];
        if (r < start || r >= a.row_start[s + 1]) return false;
    } else {
        s = r / a.per;
        start = s * a.per;
    }
    seq = a.first + s;
    at = (size_t)a.pos[s] + (r - start);
    return at < a.c.cap;
}

template <typename T>
__device__ __forceinline__ float kv_in(T x) {
    if constexpr (sizeof(T) == 4) return x;
    else return bf16_to_f32(x);
}
template <typename T>
__device__ __forceinline__ T kv_out(float x) {
    if constexpr (sizeof(T) == 4) return x;
    else return f32_to_bf16(x);
}

// A wave a row and kv head: lanes 0-31 its key, 32-63 its value, four
// channels a lane (and a second four past 128).
template <int FMT, typename T>
__global__ void __launch_bounds__(256) kv_write(KvRows a, const T *k, const T *v) {
    const size_t item = (size_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const uint32_t r = (uint32_t)(item / a.c.Hk), h = (uint32_t)(item % a.c.Hk), lane = threadIdx.x & 63;
    uint32_t seq;
    size_t at;
    if (r >= a.n_rows || !kv_place(a, r, seq, at)) return;
    const bool val = lane >= 32;
    const uint32_t hd = a.c.hd, c0 = 4 * (lane & 31);
    const T *src = (val ? v : k) + (size_t)r * a.stride + (size_t)h * hd;
    float x[8];
    uint32_t top = 0;
#pragma unroll
    for (int p = 0; p < 2; p++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const uint32_t c = c0 + 128 * p + e;
            const float f = c < hd ? kv_in<T>(src[c]) : 0.0f;
            x[4 * p + e] = f;
            const uint32_t b = __float_as_uint(f) & 0x7fffffffu;
            top = b > top ? b : top;
        }
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) {
        const uint32_t b = (uint32_t)__shfl_xor((int)top, o, 64);
        top = b > top ? b : top;
    }
    constexpr float L = FMT == QBK_KV_INT8 ? 127.0f : 448.0f;
    const bool whole = top < 0x7f800000u;
    const float A = fmaxf(__uint_as_float(whole ? top : 0u), 0x1p-100f);
    const float inv = L * (1.0f / A);
    const size_t slab = a.c.slab(seq, h);
#pragma unroll
    for (int p = 0; p < 2; p++) {
        const uint32_t c = c0 + 128 * p;
        if (c >= hd) continue;
        uint32_t w = 0;
        float y[4];
#pragma unroll
        for (int e = 0; e < 4; e++) y[e] = whole ? x[4 * p + e] * inv : 0.0f;
        if constexpr (FMT == QBK_KV_INT8) {
#pragma unroll
            for (int e = 0; e < 4; e++) w |= (uint32_t)((int)rintf(y[e]) + 128) << (8 * e);
        } else {
            w = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
            w = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], (int)w, true);
        }
        if (!val) {
            *(uint32_t *)(a.c.k + slab * hd + kv_key_at(at, c, hd)) = w;
        } else {
            uint8_t *d = a.c.v + slab * hd + kv_val_at(at, c, hd);
#pragma unroll
            for (int e = 0; e < 4; e++) d[64 * e] = (uint8_t)(w >> (8 * e));
        }
    }
    if ((lane & 31) == 0) (val ? a.c.vs : a.c.ks)[slab + at] = whole ? A * (1.0f / L) : __builtin_nanf("");
}

template <int FMT>
__device__ __forceinline__ float kv_value(uint32_t byte, float scale) {
    if constexpr (FMT == QBK_KV_INT8) return (float)((int)byte - 128) * scale;
    else return __builtin_amdgcn_cvt_f32_fp8((int)byte, 0) * scale;
}

template <int FMT, typename T>
__global__ void __launch_bounds__(256) kv_read(KvRows a, T *k, T *v) {
    const size_t item = (size_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const uint32_t r = (uint32_t)(item / a.c.Hk), h = (uint32_t)(item % a.c.Hk), lane = threadIdx.x & 63;
    if (r >= a.n_rows) return;
    uint32_t seq = 0;
    size_t at = 0;
    const bool ok = kv_place(a, r, seq, at);
    const bool val = lane >= 32;
    const uint32_t hd = a.c.hd, c0 = 4 * (lane & 31);
    T *dst = (val ? v : k) + (size_t)r * a.stride + (size_t)h * hd;
    const size_t slab = ok ? a.c.slab(seq, h) : 0;
    const float scale = ok ? (val ? a.c.vs : a.c.ks)[slab + at] : __builtin_nanf("");
#pragma unroll
    for (int p = 0; p < 2; p++) {
        const uint32_t c = c0 + 128 * p;
        if (c >= hd) continue;
        uint32_t w = 0x80808080u;  // a code that is a number in either format
        if (ok) {
            if (!val) {
                w = *(const uint32_t *)(a.c.k + slab * hd + kv_key_at(at, c, hd));
            } else {
                const uint8_t *s = a.c.v + slab * hd + kv_val_at(at, c, hd);
                w = s[0] | (uint32_t)s[64] << 8 | (uint32_t)s[128] << 16 | (uint32_t)s[192] << 24;
            }
        }
#pragma unroll
        for (int e = 0; e < 4; e++) dst[c + e] = kv_out<T>(kv_value<FMT>(w >> (8 * e) & 255u, scale));
    }
}

// Checks shared by the write and the read; *a filled for a launch, n_rows 0
// where there is nothing to do.
static int kv_rows_args(const qbk_kv_shape *shape, const void *cache, const void *k, const void *v, int dtype,
                        size_t row_stride, size_t n_rows, const uint32_t *row_start, const uint32_t *pos,
                        size_t first_seq, size_t n, KvRows *a) {
    int rc;
    size_t bytes;
    if ((rc = kv_check_shape(shape, &bytes))) return rc;
    if (dtype != QBK_F32 && dtype != QBK_BF16)
        return fail(QBK_ERR_VALIDATION, fmt("kv cache rows must be float32 or bfloat16 (dtype %d)", dtype));
    if (first_seq > shape->n_seqs || n > shape->n_seqs - first_seq)
        return fail(QBK_ERR_VALIDATION, fmt("sequences %zu .. %zu of a kv cache holding %zu", first_seq,
                                            first_seq + n, shape->n_seqs));
    const size_t width = shape->n_kv_heads * shape->head_dim;
    if (n_rows > 1 && row_stride < width)
        return fail(QBK_ERR_VALIDATION, fmt("row_stride %zu is smaller than a row of %zu values", row_stride, width));
    if (n_rows > 0x7FFFFFFFull || n_rows * shape->n_kv_heads > 0x1FFFFFFFFull || row_stride > ((size_t)1 << 40))
        return fail(QBK_ERR_VALIDATION, "kv cache: too many rows for one call");
    if (n_rows != 0 && n == 0) return fail(QBK_ERR_VALIDATION, "kv cache rows for no sequence");
    if (n_rows != 0 && !row_start && n_rows % n != 0)
        return fail(QBK_ERR_VALIDATION, fmt("%zu rows do not split evenly over %zu sequences", n_rows, n));
    if (n_rows != 0 && (!cache || !k || !v || !pos)) return fail(QBK_ERR_VALIDATION, "null argument");
    if ((uintptr_t)cache & 15) return fail(QBK_ERR_VALIDATION, "kv cache buffer must be 16-byte aligned");
    a->n_rows = (uint32_t)n_rows;
    if (n_rows == 0) return QBK_OK;
    a->c = kv_view(shape, cache);
    a->row_start = row_start;
    a->pos = pos;
    a->stride = row_stride;
    a->n = (uint32_t)n;
    a->per = (uint32_t)(n_rows / n ? n_rows / n : 1);
    a->first = (uint32_t)first_seq;
    return QBK_OK;
}

}  // namespace qbk

using namespace qbk;

extern "C" {

size_t qbk_kv_cache_size(const qbk_kv_shape *shape) {
    size_t bytes = 0;
    return kv_check_shape(shape, &bytes) ? 0 : bytes;
}

int qbk_kv_cache_write_dev(qbk_ctx *ctx, const qbk_kv_shape *shape, void *cache, const void *k, const void *v,
                           int dtype, size_t row_stride, size_t n_rows, const uint32_t *row_start,
                           const uint32_t *pos, size_t first_seq, size_t n, void *stream) {
    int rc;
    KvRows a;
    if ((rc = kv_rows_args(shape, cache, k, v, dtype, row_stride, n_rows, row_start, pos, first_seq, n, &a)))
        return rc;
    if (a.n_rows == 0) return QBK_OK;
    if ((rc = bind(ctx))) return rc;
    const dim3 grid((unsigned)div_ceil(n_rows * shape->n_kv_heads, 4));
    hipStream_t s = (hipStream_t)stream;
#define KV_GO(FMT)                                                                                                \
    if (dtype == QBK_F32)                                                                                         \
        hipLaunchKernelGGL((kv_write<FMT, float>), grid, dim3(256), 0, s, a, (const float *)k, (const float *)v); \
    else                                                                                                          \
        hipLaunchKernelGGL((kv_write<FMT, uint16_t>), grid, dim3(256), 0, s, a, (const uint16_t *)k,              \
                           (const uint16_t *)v);
    if (shape->format == QBK_KV_INT8) {
        KV_GO(QBK_KV_INT8)
    } else {
        KV_GO(QBK_KV_FP8)
    }
#undef KV_GO
    QBK_HIP(hipGetLastError());
    return QBK_OK;
}

int qbk_kv_cache_read_dev(qbk_ctx *ctx, const qbk_kv_shape *shape, const void *cache, void *k, void *v, int dtype,
                          size_t row_stride, size_t n_rows, const uint32_t *row_start, const uint32_t *pos,
                          size_t first_seq, size_t n, void *stream) {
    int rc;
    KvRows a;
    if ((rc = kv_rows_args(shape, cache, k, v, dtype, row_stride, n_rows, row_start, pos, first_seq, n, &a)))
        return rc;
    if (a.n_rows == 0) return QBK_OK;
    if ((rc = bind(ctx))) return rc;
    const dim3 grid((unsigned)div_ceil(n_rows * shape->n_kv_heads, 4));
    hipStream_t s = (hipStream_t)stream;
#define KV_GO(FMT)                                                                                          \
    if (dtype == QBK_F32)                                                                                   \
        hipLaunchKernelGGL((kv_read<FMT, float>), grid, dim3(256), 0, s, a, (float *)k, (float *)v);        \
    else                                                                                                    \
        hipLaunchKernelGGL((kv_read<FMT, uint16_t>), grid, dim3(256), 0, s, a, (uint16_t *)k, (uint16_t *)v);
    if (shape->format == QBK_KV_INT8) {
        KV_GO(QBK_KV_INT8)
    } else {
        KV_GO(QBK_KV_FP8)
    }
#undef KV_GO
    QBK_HIP(hipGetLastError());
    return QBK_OK;
}

}  // extern "C"
