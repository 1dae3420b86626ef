// kvcache.hip -- the 8-bit KV cache's rows in and out: quantised as they are
// written, one f32 scale a row and kv head, and read back as values.
//
//   A = max(max |x|, 2^-100), L = 127 (int8) or 448 (e4m3)
//   scale = A (1 / L),  code = nearest(x (L (1 / A))),  value = code * scale
//
// each product and reciprocal rounded to f32.  The floor on A keeps L / A and
// every scale a normal number.  One pass over
// rows and codes either way, bound by memory (16384 rows of 8 heads of 128 read
// as f32 28.4 us, 5.9 TB/s, as bf16 19.3, 5.2; 50584 f32 rows written 117 to 122, 4.3 to 4.5;
// a few rows are bound by the launch, 3 us).
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
    if (s->n_kv_heads > 65536) return fail(QBK_ERR_VALIDATION, "kv cache heads must be at most 65536");
    if (s->capacity > 0x7FFFFF00u || s->n_seqs > 0x7FFFFFFFu)
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
    bool tiles;  // by 64-row tiles
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

// Four values at any alignment (one access on this machine).
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Kv4 {
    T v[4];
};

// ---- many rows a sequence: a workgroup a 64-row tile of one kv head ----------

// The workgroup's tile: input rows row .. row + hi - lo - 1 stand at rows lo ..
// hi - 1 of the tile that begins at position first of sequence seq; seq -1:
// rows that no sequence claims (lo 0).
struct KvTile {
    int32_t seq;
    uint32_t row, lo, hi;
    uint64_t first;
};
// Segments of the rows: 0 those before the first sequence's, 1 .. n the
// sequences', n + 1 those behind the last one's.  Segment i's tiles are numbered
// from (its first row) / 64 + 2 i on, which leaves room for the two that its
// rows touch past those they fill, so that a tile finds its segment among 64 in
// one load and one ballot, without the other segments' counts (a running sum
// over them took 6.6 ms for 16384 sequences of four rows).
__device__ __forceinline__ bool kv_tile(const KvRows &a, uint32_t tile, KvTile *t) {
    const uint32_t lane = threadIdx.x & 63;
    auto bound = [&](uint32_t i) -> uint32_t {  // first row of segment i, 0 .. n + 2
        if (i == 0) return 0;
        if (i == a.n + 2) return a.n_rows;
        const uint32_t r = a.row_start ? a.row_start[i - 1] : (i - 1) * a.per;
        return r < a.n_rows ? r : a.n_rows;
    };
    uint32_t seg = 0, len = a.n + 2;  // seg .. seg + len - 1 hold it; the first of them begins at or before tile
    while (len > 1) {
        const uint32_t step = (len + 63) / 64, off = lane * step;
        bool below = false;
        if (off < len) below = bound(seg + off) / 64 + 2 * (seg + off) <= tile;
        const uint64_t above = ~__ballot(below);
        const uint32_t at = (above ? (uint32_t)__builtin_ctzll(above) : 64u) - 1;
        const uint32_t skip = (uint32_t)__builtin_amdgcn_readfirstlane((int)(at * step));
        seg += skip;
        len = len - skip < step ? len - skip : step;
    }
    const bool claimed = seg >= 1 && seg <= a.n;
    const uint32_t from = bound(seg), to = bound(seg + 1), k = tile - (from / 64 + 2 * seg);
    const uint32_t at = claimed ? a.pos[seg - 1] : 0, skip = at & 63;
    if (to <= from || k >= (skip + (uint64_t)(to - from) + 63) / 64) return false;
    t->seq = claimed ? (int32_t)(seg - 1) : -1;
    t->lo = k == 0 ? skip : 0;
    t->row = from + (k == 0 ? 0 : 64 * k - skip);
    t->hi = to - t->row < 64 - t->lo ? t->lo + (to - t->row) : 64;
    t->first = (uint64_t)(at - skip) + 64ull * k;
    return true;
}

// 4 x 4 bytes: out[i] = bytes i of in[0 .. 3].
__device__ __forceinline__ void kv_transpose4(const uint32_t (&in)[4], uint32_t (&out)[4]) {
    const uint32_t a = __builtin_amdgcn_perm(in[1], in[0], 0x05010400u), b = __builtin_amdgcn_perm(in[3], in[2], 0x05010400u);
    const uint32_t c = __builtin_amdgcn_perm(in[1], in[0], 0x07030602u), d = __builtin_amdgcn_perm(in[3], in[2], 0x07030602u);
    out[0] = __builtin_amdgcn_perm(b, a, 0x05040100u);
    out[1] = __builtin_amdgcn_perm(b, a, 0x07060302u);
    out[2] = __builtin_amdgcn_perm(d, c, 0x05040100u);
    out[3] = __builtin_amdgcn_perm(d, c, 0x07060302u);
}

// Largest over 16 lanes.
__device__ __forceinline__ uint32_t kv_max16(uint32_t v) {
    auto up = [](uint32_t x, uint32_t y) { return x > y ? x : y; };
    v = up(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xf, 0xf, true));  // row_ror 8, 4, 2, 1
    v = up(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x124, 0xf, 0xf, true));
    v = up(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x122, 0xf, 0xf, true));
    return up(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x121, 0xf, 0xf, true));
}

template <int FMT>
__device__ __forceinline__ uint32_t kv_codes(const float (&x)[4], float inv) {
    uint32_t w = 0;
    if constexpr (FMT == QBK_KV_INT8) {
#pragma unroll
        for (int e = 0; e < 4; e++) w |= (uint32_t)((int)rintf(x[e] * inv) + 128) << (8 * e);
    } else {
        w = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[0] * inv, x[1] * inv, 0, false);
        w = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[2] * inv, x[3] * inv, (int)w, true);
    }
    return w;
}

// Sixteen lanes a row, four channels a lane and P times 64 channels, sixteen
// rows at a time and every row's loads before the first is used; the values'
// codes go through LDS, from where 4 x 4 bytes turn round and leave as a
// channel's 16 bytes.  PADW: dwords of an LDS row.
template <int FMT, int P, typename T>
__global__ void __launch_bounds__(256) kv_write_tiles(KvRows a, const T *k, const T *v) {
    constexpr int PADW = 16 * P + 1;
    __shared__ uint32_t codes[64 * PADW];
    const uint32_t h = blockIdx.x % a.c.Hk, tid = threadIdx.x, hd = a.c.hd;
    KvTile t;
    if (!kv_tile(a, blockIdx.x / a.c.Hk, &t) || t.seq < 0 || t.first >= a.c.cap) return;
    const size_t slab = a.c.slab(a.first + t.seq, h);
    uint32_t hi = t.hi;
    if (t.first + hi > a.c.cap) hi = (uint32_t)(a.c.cap - t.first);
    const uint32_t c0 = 4 * (tid & 15);
    constexpr float L = FMT == QBK_KV_INT8 ? 127.0f : 448.0f;
#pragma unroll
    for (int val = 0; val < 2; val++) {
        Kv4<T> raw[4][P];
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const uint32_t r = 16 * q + (tid >> 4);
            const bool in = r >= t.lo && r < hi;
            const T *src = (val ? v : k) + (size_t)(t.row + (in ? r - t.lo : 0)) * a.stride + (size_t)h * hd;
#pragma unroll
            for (int p = 0; p < P; p++) raw[q][p] = *(const Kv4<T> *)(src + (c0 + 64 * p < hd ? c0 + 64 * p : 0));
        }
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const uint32_t r = 16 * q + (tid >> 4);
            float x[P][4];
            uint32_t top = 0;
#pragma unroll
            for (int p = 0; p < P; p++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    x[p][e] = kv_in<T>(raw[q][p].v[e]);  // channels past the last repeat the first four
                    const uint32_t b = __float_as_uint(x[p][e]) & 0x7fffffffu;
                    top = b > top ? b : top;
                }
            top = kv_max16(top);
            const bool whole = top < 0x7f800000u, in = r >= t.lo && r < hi;
            const float A = fmaxf(__uint_as_float(whole ? top : 0u), 0x1p-100f), inv = L * (1.0f / A);
#pragma unroll
            for (int p = 0; p < P; p++) {
                if (c0 + 64 * p >= hd) continue;
                if (!whole)
#pragma unroll
                    for (int e = 0; e < 4; e++) x[p][e] = 0.0f;
                const uint32_t w = kv_codes<FMT>(x[p], inv);
                if (val) codes[r * PADW + c0 / 4 + 16 * p] = w;
                else if (in) *(uint32_t *)(a.c.k + slab * hd + kv_key_at(t.first + r, c0 + 64 * p, hd)) = w;
            }
            if (in && (tid & 15) == 0)
                (val ? a.c.vs : a.c.ks)[slab + t.first + r] = whole ? A * (1.0f / L) : __builtin_nanf("");
        }
    }
    __syncthreads();
    uint8_t *dst = a.c.v + slab * hd + t.first * hd;
    for (uint32_t x = tid; x < hd; x += 256) {  // four channels, rows 16 i + 4 g + j of one g
        const uint32_t c4 = x >> 2, g = x & 3;
        uint32_t out[4][4];  // [i][channel]
#pragma unroll
        for (int i = 0; i < 4; i++) {
            uint32_t in[4];
#pragma unroll
            for (int j = 0; j < 4; j++) in[j] = codes[(16 * i + 4 * g + j) * PADW + c4];
            kv_transpose4(in, out[i]);
        }
#pragma unroll
        for (int e = 0; e < 4; e++) {
            uint8_t *d = dst + (size_t)(4 * c4 + e) * 64 + 16 * g;
            if (t.lo == 0 && hi == 64) {
                *(uint4 *)d = uint4{out[0][e], out[1][e], out[2][e], out[3][e]};
                continue;
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t r = 16 * i + 4 * g;
                if (r >= t.lo && r + 4 <= hi) {
                    *(uint32_t *)(d + 4 * i) = out[i][e];
                } else {
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        if (r + j >= t.lo && r + j < hi) d[4 * i + j] = (uint8_t)(out[i][e] >> (8 * j));
                }
            }
        }
    }
}

// Sixteen codes as bf16 at any alignment, 16 bytes a store.
template <int FMT>
__device__ __forceinline__ void kv_store16(uint16_t *dst, const uint4 &w, float scale) {
    struct __attribute__((packed, aligned(2))) Out {
        uint32_t v[4];
    };
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
        Out y;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const uint32_t b = (&w.x)[i + e / 2] >> (16 * (e & 1));
            y.v[e] = f32x2_to_bf16x2(kv_value<FMT>(b & 255u, scale), kv_value<FMT>(b >> 8 & 255u, scale));
        }
        *(Out *)(dst + 4 * i) = y;
    }
}

// Four codes as f32, 16 bytes a store.
template <int FMT>
__device__ __forceinline__ void kv_store4(float *dst, uint32_t w, float scale) {
    struct __attribute__((packed, aligned(4))) Out {
        float v[4];
    } y;
#pragma unroll
    for (int e = 0; e < 4; e++) y.v[e] = kv_value<FMT>(w >> (8 * e) & 255u, scale);
    *(Out *)dst = y;
}

// The other way: a lane takes 16 channels of a row, keys straight from their
// 16-byte pieces, values from LDS, where 4 x 4 bytes have been turned.  f32 has
// the keys in LDS as well and a lane four channels, so that a wave's stores lie
// behind one another.
template <int FMT, typename T>
__global__ void __launch_bounds__(256) kv_read_tiles(KvRows a, T *k, T *v) {
    __shared__ __attribute__((aligned(16))) uint32_t codes[64 * 68];
    __shared__ __attribute__((aligned(16))) uint32_t kcodes[sizeof(T) == 4 ? 64 * 68 : 4];
    __shared__ float scale[2][64];
    const uint32_t h = blockIdx.x % a.c.Hk, tid = threadIdx.x, hd = a.c.hd, nc = hd / 16;
    KvTile t;
    if (!kv_tile(a, blockIdx.x / a.c.Hk, &t)) return;
    const bool held = t.seq >= 0 && t.first < a.c.cap;
    const size_t slab = a.c.slab(a.first + (held ? t.seq : 0), h);
    const uint64_t first = held ? t.first : 0;
    const uint32_t padw = hd / 4 + 4;  // 16-byte rows
    const uint8_t *src = a.c.v + slab * hd + first * hd;
    const uint4 none = {0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u};  // numbers in either format
    const uint32_t units = (t.hi - t.lo) * nc;  // at most 64 * 16
    uint4 keys[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {  // asked for before the values are turned
        const uint32_t x = tid + 256 * i, r = t.lo + x / nc, chunk = x % nc;
        keys[i] = none;
        if (x < units && held && first + r < a.c.cap)
            keys[i] = *(const uint4 *)(a.c.k + slab * hd + kv_key_at(first + r, 16 * chunk, hd));
    }
    if (tid < 128) {
        const uint32_t r = tid & 63;
        const bool in = held && r >= t.lo && first + r < a.c.cap;
        scale[tid >> 6][r] = in ? (tid < 64 ? a.c.ks : a.c.vs)[slab + first + r] : __builtin_nanf("");
    }
    for (uint32_t x = tid; x < hd; x += 256) {
        const uint32_t c4 = x >> 2, g = x & 3;
        uint4 w[4];
#pragma unroll
        for (int e = 0; e < 4; e++) w[e] = *(const uint4 *)(src + (size_t)(4 * c4 + e) * 64 + 16 * g);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t in[4] = {(&w[0].x)[i], (&w[1].x)[i], (&w[2].x)[i], (&w[3].x)[i]};
            uint32_t out[4];
            kv_transpose4(in, out);
#pragma unroll
            for (int j = 0; j < 4; j++) codes[(16 * i + 4 * g + j) * padw + c4] = out[j];
        }
    }
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t x = tid + 256 * i, r = t.lo + x / nc, chunk = x % nc;
            if (x < units) *(uint4 *)(kcodes + r * padw + 4 * chunk) = keys[i];
        }
        __syncthreads();
        // x / words by a multiplication: x < 2^12, words <= 2^6, so that x times the factor's excess is below 2^20
        const uint32_t words = hd / 4, by = ((1u << 20) + words - 1) / words, all = (t.hi - t.lo) * words;
        for (uint32_t x = tid; x < all; x += 256) {
            const uint32_t row = x * by >> 20, c4 = x - row * words, r = t.lo + row;
            const size_t at = (size_t)(t.row + row) * a.stride + (size_t)h * hd + 4 * c4;
            kv_store4<FMT>(k + at, kcodes[r * padw + c4], scale[0][r]);  // rows not held: codes times NaN
            kv_store4<FMT>(v + at, codes[r * padw + c4], scale[1][r]);
        }
    } else {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t x = tid + 256 * i, r = t.lo + x / nc, chunk = x % nc;
            if (x >= units) continue;
            const uint4 vw = held && first + r < a.c.cap ? *(const uint4 *)(codes + r * padw + 4 * chunk) : none;
            const size_t at = (size_t)(t.row + r - t.lo) * a.stride + (size_t)h * hd + 16 * chunk;
            kv_store16<FMT>(k + at, keys[i], scale[0][r]);
            kv_store16<FMT>(v + at, vw, scale[1][r]);
        }
    }
}

// Whether a call goes by tiles.  A tile takes its transposes and barriers
// however few rows it has; rows by themselves store bytes 64 apart.  Tiles pay
// once the rows fill the chip and a sequence's are some 512 channels of a head
// (us by rows / by tiles, f32, 8 heads of 128 unless said):
//   one sequence, written: 256 rows 4.5 / 6.3, 512 6.6 / 6.3, 1024 10.1 / 6.5
//   the same read: 512 rows 4.3 / 5.1, 1024 6.2 / 5.6, 2048 9.9 / 6.8
//   1024 sequences, written: two rows each 31 / 47, four 57 / 49, sixteen 135 / 57; read 26 / 34, 49 / 35, 71 / 42
//   4096 sequences, 2 heads of 64, written: four rows 20.5 / 37, eight 37.5 / 38, sixteen 69 / 39
static bool kv_by_tiles(size_t n_rows, size_t n, const qbk_kv_shape *s) {
    return (unsigned __int128)n_rows * s->n_kv_heads > 4096 && n_rows * s->head_dim / 512 >= n;
}

// Tile numbers of a call (kv_tile): at most two a segment past the tiles that the rows fill.
static size_t kv_tiles(size_t n_rows, size_t n) { return n_rows / 64 + 2 * (n + 2); }

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
    if (n_rows > 0x7FFFFFFFull || row_stride > ((size_t)1 << 40))
        return fail(QBK_ERR_VALIDATION, "kv cache: too many rows for one call");
    if (n_rows != 0 && n == 0) return fail(QBK_ERR_VALIDATION, "kv cache rows for no sequence");
    if (n_rows != 0 && !row_start && n_rows % n != 0)
        return fail(QBK_ERR_VALIDATION, fmt("%zu rows do not split evenly over %zu sequences", n_rows, n));
    // a launch is below 2^32 threads
    a->tiles = kv_by_tiles(n_rows, n, shape);
    const size_t groups = a->tiles ? kv_tiles(n_rows, n) * shape->n_kv_heads
                                   : div_ceil(n_rows * shape->n_kv_heads, 4);
    if (groups > 0xFFFFFF) return fail(QBK_ERR_VALIDATION, "kv cache: too many rows for one call");
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

template <int FMT, typename T>
static void kv_write_go(const KvRows &a, const T *k, const T *v, hipStream_t s) {
    if (a.tiles) {
        void (*kern)(KvRows, const T *, const T *) = a.c.hd <= 64    ? kv_write_tiles<FMT, 1, T>
                                                     : a.c.hd <= 128 ? kv_write_tiles<FMT, 2, T>
                                                                     : kv_write_tiles<FMT, 4, T>;
        hipLaunchKernelGGL(kern, dim3((unsigned)(kv_tiles(a.n_rows, a.n) * a.c.Hk)), dim3(256), 0, s, a, k, v);
    } else {
        hipLaunchKernelGGL((kv_write<FMT, T>), dim3((unsigned)div_ceil((size_t)a.n_rows * a.c.Hk, 4)), dim3(256), 0, s,
                           a, k, v);
    }
}

template <int FMT, typename T>
static void kv_read_go(const KvRows &a, T *k, T *v, hipStream_t s) {
    if (a.tiles)
        hipLaunchKernelGGL((kv_read_tiles<FMT, T>), dim3((unsigned)(kv_tiles(a.n_rows, a.n) * a.c.Hk)), dim3(256), 0, s,
                           a, k, v);
    else
        hipLaunchKernelGGL((kv_read<FMT, T>), dim3((unsigned)div_ceil((size_t)a.n_rows * a.c.Hk, 4)), dim3(256), 0, s,
                           a, k, v);
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
    hipStream_t s = (hipStream_t)stream;
    if (dtype == QBK_F32)
        shape->format == QBK_KV_INT8 ? kv_write_go<QBK_KV_INT8>(a, (const float *)k, (const float *)v, s)
                                     : kv_write_go<QBK_KV_FP8>(a, (const float *)k, (const float *)v, s);
    else
        shape->format == QBK_KV_INT8 ? kv_write_go<QBK_KV_INT8>(a, (const uint16_t *)k, (const uint16_t *)v, s)
                                     : kv_write_go<QBK_KV_FP8>(a, (const uint16_t *)k, (const uint16_t *)v, s);
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
    hipStream_t s = (hipStream_t)stream;
    if (dtype == QBK_F32)
        shape->format == QBK_KV_INT8 ? kv_read_go<QBK_KV_INT8>(a, (float *)k, (float *)v, s)
                                     : kv_read_go<QBK_KV_FP8>(a, (float *)k, (float *)v, s);
    else
        shape->format == QBK_KV_INT8 ? kv_read_go<QBK_KV_INT8>(a, (uint16_t *)k, (uint16_t *)v, s)
                                     : kv_read_go<QBK_KV_FP8>(a, (uint16_t *)k, (uint16_t *)v, s);
    QBK_HIP(hipGetLastError());
    return QBK_OK;
}

}  // extern "C"
