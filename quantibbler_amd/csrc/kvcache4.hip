// kvcache4.hip -- the 4-bit KV cache's rows in and out.
//
// With A = max(max |x|, 2^-100) over a row's head and a_g the largest |x| of 32
// channels of it:
//   m_g   = e4m3(a_g (448 (1 / A)))                the group's multiplier
//   code  = e2m1((x (2688 (1 / A))) (1 / m_g))     0, 1/2, 1, 3/2, 2, 3, 4 or 6 (0 for m_g = 0)
//   scale = A (1 / 2688),  value = (code m_g) scale
// each step rounded once to f32 (to nearest, even at a tie), codes past 6 held
// at 6 (2688 = 6 448).  The multiplier of the group that holds A is 448, the
// others' follow their own largest within 2^-4.
//
// One pass over rows and codes, bound by memory where there are many (98816 f32
// rows of 8 heads of 128 written 199 us, 4.6 TB/s; 10391 written 31, read back
// 18.4, 3.1 and 5.3 TB/s; 50000 of one sequence read as bf16 33 us), by the launch
// and one row's chain of reductions where there are few (32 bf16 rows of 8 heads of
// 128 out of wider ones, from a graph, written 4.6, read 3.5).
#include <math.h>

#include "kvcache_rows.h"

#pragma clang fp contract(off)

namespace qbk {

#define KV4_MUL 448.0f
#define KV4_TOP 2688.0f

__device__ __forceinline__ uint32_t kv4_most(uint32_t a, uint32_t b) { return a > b ? a : b; }

// The largest over aligned runs of eight lanes.
__device__ __forceinline__ uint32_t kv4_max8(uint32_t v) {
    v = kv4_most(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, true));   // lane ^ 1
    v = kv4_most(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, true));   // lane ^ 2
    return kv4_most(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xf, 0xf, true));  // 7 - lane
}
// Of that, over aligned runs of 32.
__device__ __forceinline__ uint32_t kv4_max32(uint32_t v) {
    v = kv4_most(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xf, 0xf, true));  // row_ror 8
    const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return kv4_most(a[0], a[1]);
}

// What a row's values are multiplied by: per = 1 / A, 0 for a row that holds a
// NaN or an infinity (then nothing is kept but the scale, NaN).
struct Kv4Row {
    float per, scale;
    __device__ __forceinline__ Kv4Row(uint32_t top) {  // bits of the largest |x|
        const bool whole = top < 0x7f800000u;
        const float A = fmaxf(__uint_as_float(whole ? top : 0u), 0x1p-100f);
        per = whole ? 1.0f / A : 0.0f;
        scale = whole ? A * (1.0f / KV4_TOP) : __builtin_nanf("");
    }
};
// A group's multiplier, of the bits of its largest |x|, and its reciprocal.
__device__ __forceinline__ uint32_t kv4_mul(const Kv4Row &row, uint32_t top, float &by) {
    const float a = row.per == 0.0f ? 0.0f : __uint_as_float(top) * (KV4_MUL * row.per);
    const uint32_t m = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(a, a, 0, false) & 255u;
    const float f = __builtin_amdgcn_cvt_f32_fp8((int)m, 0);
    by = f > 0.0f ? 1.0f / f : 0.0f;
    return m;
}
// Four channels' codes, the first lowest.
__device__ __forceinline__ uint32_t kv4_codes(const Kv4Row &row, const float (&x)[4], float by) {
    if (row.per == 0.0f) return 0;
    float z[4];
#pragma unroll
    for (int e = 0; e < 4; e++) z[e] = (x[e] * (KV4_TOP * row.per)) * by;
    uint32_t w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, z[0], z[1], 1.0f, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, z[2], z[3], 1.0f, 1);
    return w & 0xffffu;
}

// A wave a row and kv head: lanes 0-31 its key, 32-63 its value, four channels
// a lane (and a second four past 128).  Two rows share a byte of the values: the
// even one's wave writes both where the call holds both, and a row by itself
// leaves the other half as it was.
template <typename T>
__global__ void __launch_bounds__(256) kv4_write(KvRows a, const T *k, const T *v) {
    const size_t item = (size_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const uint32_t r = (uint32_t)(item / a.c.Hk), h = (uint32_t)(item % a.c.Hk), lane = threadIdx.x & 63;
    uint32_t seq, start, end;
    size_t at;
    if (r >= a.n_rows || !kv_place(a, r, seq, at, start, end)) return;
    const bool val = lane >= 32, odd = at & 1;
    const bool both = !odd && r + 1 < end && r + 1 < a.n_rows && at + 1 < a.c.cap;  // the odd row behind is the call's too
    const bool other = odd && r > start;                                            // its even row writes this one
    const uint32_t hd = a.c.hd, ng = a.c.groups(), c0 = 4 * (lane & 31);
    const size_t slab = a.c.slab(seq, h);
    uint8_t *vc = a.c.v + slab * (16 * ng);
    uint32_t mine[2] = {0, 0};
    for (uint32_t q = 0; q < (both ? 2u : 1u); q++) {
        const T *src = (val ? v : k) + (size_t)(r + q) * a.stride + (size_t)h * hd;
        float x[2][4];
        uint32_t group[2];
#pragma unroll
        for (int p = 0; p < 2; p++) {
            group[p] = 0;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const uint32_t c = c0 + 128 * p + e;
                x[p][e] = c < hd ? kv_in<T>(src[c]) : 0.0f;
                group[p] = kv4_most(group[p], __float_as_uint(x[p][e]) & 0x7fffffffu);
            }
            group[p] = kv4_max8(group[p]);
        }
        const Kv4Row row(kv4_max32(kv4_most(group[0], group[1])));
#pragma unroll
        for (int p = 0; p < 2; p++) {
            const uint32_t c = c0 + 128 * p;
            if (c >= hd) continue;
            float by;
            const uint32_t m = kv4_mul(row, group[p], by), w = kv4_codes(row, x[p], by);
            if (q == 0 && (lane & 7) == 0) {
                if (val) a.c.vm[slab * ng + kv4_val_mul_at(at, c / 32, ng)] = (uint8_t)m;
                else a.c.km[slab * ng + kv4_key_mul_at(at, c / 32, ng)] = (uint8_t)m;
            }
            if (!val) {
                if (q == 0) *(uint16_t *)(a.c.k + slab * (hd / 2) + kv4_key_at(at, c, hd)) = (uint16_t)w;
                continue;
            }
            if (q == 0) mine[p] = w;
            if (other || (both && q == 0)) continue;
            uint8_t *d = vc + kv4_val_at(at, c, ng);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const uint32_t code = w >> (4 * e) & 15u;
                if (both) d[64 * e] = (uint8_t)((mine[p] >> (4 * e) & 15u) | code << 4);
                else if (odd) d[64 * e] = (uint8_t)((d[64 * e] & 15u) | code << 4);
                else d[64 * e] = (uint8_t)((d[64 * e] & 0xf0u) | code);
            }
        }
        if (q == 0 && (lane & 31) == 0) (val ? a.c.vs : a.c.ks)[slab + at] = row.scale;
    }
}

typedef float kv4_f2_t __attribute__((ext_vector_type(2)));

// Four codes (16 bits) as values.
__device__ __forceinline__ void kv4_values(uint32_t w, uint32_t mul, float scale, float (&x)[4]) {
    const float m = __builtin_amdgcn_cvt_f32_fp8((int)mul, 0);
    const kv4_f2_t lo = __builtin_bit_cast(kv4_f2_t, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 0));
    const kv4_f2_t hi = __builtin_bit_cast(kv4_f2_t, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 1));
    x[0] = (lo[0] * m) * scale;
    x[1] = (lo[1] * m) * scale;
    x[2] = (hi[0] * m) * scale;
    x[3] = (hi[1] * m) * scale;
}

template <typename T>
__global__ void __launch_bounds__(256) kv4_read(KvRows a, T *k, T *v) {
    const size_t item = (size_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const uint32_t r = (uint32_t)(item / a.c.Hk), h = (uint32_t)(item % a.c.Hk), lane = threadIdx.x & 63;
    if (r >= a.n_rows) return;
    uint32_t seq = 0;
    size_t at = 0;
    const bool ok = kv_place(a, r, seq, at), val = lane >= 32;
    const uint32_t hd = a.c.hd, ng = a.c.groups(), c0 = 4 * (lane & 31);
    T *dst = (val ? v : k) + (size_t)r * a.stride + (size_t)h * hd;
    const size_t slab = ok ? a.c.slab(seq, h) : 0;
    const float scale = ok ? (val ? a.c.vs : a.c.ks)[slab + at] : __builtin_nanf("");
#pragma unroll
    for (int p = 0; p < 2; p++) {
        const uint32_t c = c0 + 128 * p;
        if (c >= hd) continue;
        uint32_t w = 0, m = 0;
        if (ok && !val) {
            w = *(const uint16_t *)(a.c.k + slab * (hd / 2) + kv4_key_at(at, c, hd));
            m = a.c.km[slab * ng + kv4_key_mul_at(at, c / 32, ng)];
        } else if (ok) {
            const uint8_t *s = a.c.v + slab * (16 * ng) + kv4_val_at(at, c, ng);
            const uint32_t sh = 4 * (uint32_t)(at & 1);
#pragma unroll
            for (int e = 0; e < 4; e++) w |= (s[64 * e] >> sh & 15u) << (4 * e);
            m = a.c.vm[slab * ng + kv4_val_mul_at(at, c / 32, ng)];
        }
        float x[4];
        kv4_values(w, m, scale, x);
#pragma unroll
        for (int e = 0; e < 4; e++) dst[c + e] = kv_out<T>(x[e]);
    }
}

// ---- many rows a sequence: a workgroup a 64-row tile of one kv head ----------

// Four codes of 16 bits as four bytes, and back.
__device__ __forceinline__ uint32_t kv4_bytes(uint32_t w) {
    w = (w | w << 8) & 0x00ff00ffu;
    return (w | w << 4) & 0x0f0f0f0fu;
}
__device__ __forceinline__ uint32_t kv4_nibbles(uint32_t b) {
    b |= b >> 4;
    return __builtin_amdgcn_perm(0u, b, 0x0c0c0200u);
}
// 4 x 4 codes: out[i] = codes i of in[0 .. 3].
__device__ __forceinline__ void kv4_turn(const uint32_t (&in)[4], uint32_t (&out)[4]) {
    uint32_t b[4], t[4];
#pragma unroll
    for (int i = 0; i < 4; i++) b[i] = kv4_bytes(in[i]);
    kv_transpose4(b, t);
#pragma unroll
    for (int i = 0; i < 4; i++) out[i] = kv4_nibbles(t[i]);
}
// Bits of the codes of rows 4 k .. 4 k + 3 that lie in lo .. hi - 1.
__device__ __forceinline__ uint32_t kv4_rows_in(uint32_t row, uint32_t lo, uint32_t hi) {
    uint32_t m = 0;
#pragma unroll
    for (uint32_t j = 0; j < 4; j++) m |= row + j >= lo && row + j < hi ? 15u << (4 * j) : 0u;
    return m;
}

// Sixteen lanes a row, four channels a lane and P times 64 channels, sixteen
// rows at a time and every row's loads before the first is used; keys and values
// by workgroups of their own.  Codes go through LDS, 16 bits for four channels of
// a row: keys leave as two rows' sixteen channels, 16 bytes, values, turned by
// 4 x 4, as a channel's sixteen rows, 8 bytes; multipliers through LDS in the
// cache's order.
template <int P, typename T>
__global__ void __launch_bounds__(256) kv4_write_tiles(KvRows a, const T *k, const T *v) {
    constexpr int PAD = 16 * P + 4;  // of an LDS row, in four channels: keys are read eight bytes at a time
    __shared__ __attribute__((aligned(16))) uint16_t codes[64 * PAD];
    __shared__ __attribute__((aligned(16))) uint8_t mul[2 * P * 64];
    const uint32_t h = blockIdx.x % a.c.Hk, tid = threadIdx.x, hd = a.c.hd, ng = a.c.groups(), nc = hd / 16;
    KvTile t;
    if (!kv_tile(a, blockIdx.x / a.c.Hk, &t) || t.seq < 0 || t.first >= a.c.cap) return;
    const size_t slab = a.c.slab(a.first + t.seq, h);
    uint32_t hi = t.hi;
    if (t.first + hi > a.c.cap) hi = (uint32_t)(a.c.cap - t.first);
    const bool full = t.lo == 0 && hi == 64;
    const uint32_t c0 = 4 * (tid & 15);
    const bool val = blockIdx.y;
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
        uint32_t group[P], top = 0;
#pragma unroll
        for (int p = 0; p < P; p++) {
            group[p] = 0;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                x[p][e] = c0 + 64 * p < hd ? kv_in<T>(raw[q][p].v[e]) : 0.0f;
                group[p] = kv4_most(group[p], __float_as_uint(x[p][e]) & 0x7fffffffu);
            }
            group[p] = kv4_max8(group[p]);
            top = kv4_most(top, group[p]);
        }
        top = kv4_most(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x128, 0xf, 0xf, true));  // row_ror 8
        const Kv4Row row(top);
#pragma unroll
        for (int p = 0; p < P; p++) {
            const uint32_t c = c0 + 64 * p;
            if (c >= hd) continue;
            float by;
            const uint32_t m = kv4_mul(row, group[p], by);
            codes[r * PAD + c / 4] = (uint16_t)kv4_codes(row, x[p], by);
            if ((tid & 7) == 0)
                mul[c / 32 * 64 + (val ? (r >> 2 & 3) * 16 + (r >> 4) * 4 + (r & 3) : (r & 15) * 4 + (r >> 4))] = (uint8_t)m;
        }
        if (r >= t.lo && r < hi && (tid & 15) == 0) (val ? a.c.vs : a.c.ks)[slab + t.first + r] = row.scale;
    }
    __syncthreads();
    uint8_t *md = (val ? a.c.vm : a.c.km) + slab * ng + t.first * ng;
    for (uint32_t x = tid; x < 16 * ng; x += 256) {  // four rows of a group: key 16 i + x % 16, value 16 i + 4 g + j
        const uint32_t w = *(const uint32_t *)(mul + 4 * x);
        if (full) {
            *(uint32_t *)(md + 4 * x) = w;
            continue;
        }
#pragma unroll
        for (uint32_t i = 0; i < 4; i++) {
            const uint32_t r = val ? (x & 3) * 16 + (x >> 2 & 3) * 4 + i : 16 * i + (x & 15);
            if (r >= t.lo && r < hi) md[4 * x + i] = (uint8_t)(w >> (8 * i));
        }
    }
    if (!val) {
        uint8_t *dst = a.c.k + slab * (hd / 2) + t.first * (hd / 2);
        for (uint32_t x = tid; x < 32 * nc; x += 256) {  // rows r and r + 16, one run of 16 channels
            const uint32_t pair = x / (16 * nc), y = x - pair * 16 * nc, chunk = y >> 4, r = 32 * pair + (y & 15);
            const uint2 one = *(const uint2 *)(codes + r * PAD + 4 * chunk);
            const uint2 two = *(const uint2 *)(codes + (r + 16) * PAD + 4 * chunk);
            const bool in1 = r >= t.lo && r < hi, in2 = r + 16 >= t.lo && r + 16 < hi;
            uint8_t *d = dst + (size_t)x * 16;
            if (in1 && in2) *(uint4 *)d = uint4{one.x, one.y, two.x, two.y};
            else if (in1) *(uint2 *)d = one;
            else if (in2) *(uint2 *)(d + 8) = two;
        }
    } else {
        uint8_t *dst = a.c.v + slab * (16 * ng) + t.first * (16 * ng);
        for (uint32_t x = tid; x < 32 * ng; x += 256) {  // channels 4 q .. of one half of a group, rows of one g
            const uint32_t half = x & 1, g = x >> 1 & 3, q = x >> 3 & 3, m = x >> 5, c4 = 8 * m + 4 * half + q;
            uint32_t out[4][4];  // [i][channel]
#pragma unroll
            for (int i = 0; i < 4; i++) {
                uint32_t in[4];
#pragma unroll
                for (int j = 0; j < 4; j++) in[j] = 4 * c4 < hd ? codes[(16 * i + 4 * g + j) * PAD + c4] : 0u;
                kv4_turn(in, out[i]);
            }
            uint32_t keep[2] = {0u, 0u};  // codes that stay as they were
            if (!full) {
                keep[0] = ~(kv4_rows_in(4 * g, t.lo, hi) | kv4_rows_in(16 + 4 * g, t.lo, hi) << 16);
                keep[1] = ~(kv4_rows_in(32 + 4 * g, t.lo, hi) | kv4_rows_in(48 + 4 * g, t.lo, hi) << 16);
            }
#pragma unroll
            for (int e = 0; e < 4; e++) {
                uint2 *d = (uint2 *)(dst + m * 1024 + (4 * q + e) * 64 + g * 16 + half * 8);
                uint2 w{out[0][e] | out[1][e] << 16, out[2][e] | out[3][e] << 16};
                if (!full) {
                    const uint2 o = *d;
                    w.x = (w.x & ~keep[0]) | (o.x & keep[0]);
                    w.y = (w.y & ~keep[1]) | (o.y & keep[1]);
                }
                *d = w;
            }
        }
    }
}

// The other way: codes into LDS, 16 bits for four channels of a row, values
// turned by 4 x 4, and out as rows: four channels a lane (f32) or eight.
template <typename T>
__global__ void __launch_bounds__(256) kv4_read_tiles(KvRows a, T *k, T *v) {
    constexpr uint32_t PAD = 68, PER = sizeof(T) == 4 ? 4 : 8;  // channels a lane
    __shared__ __attribute__((aligned(16))) uint16_t codes[2][64 * PAD];
    __shared__ __attribute__((aligned(16))) uint8_t mul[2][8 * 64];
    __shared__ float scale[2][64];
    const uint32_t h = blockIdx.x % a.c.Hk, tid = threadIdx.x, hd = a.c.hd, ng = a.c.groups(), nc = hd / 16;
    KvTile t;
    if (!kv_tile(a, blockIdx.x / a.c.Hk, &t)) return;
    const bool held = t.seq >= 0 && t.first < a.c.cap;
    const size_t slab = a.c.slab(a.first + (held ? t.seq : 0), h);
    const uint64_t first = held ? t.first : 0;
    if (held) {
        const uint8_t *ks = a.c.k + slab * (hd / 2) + first * (hd / 2);
        for (uint32_t x = tid; x < 32 * nc; x += 256) {
            const uint32_t pair = x / (16 * nc), y = x - pair * 16 * nc, chunk = y >> 4, r = 32 * pair + (y & 15);
            const uint4 w = *(const uint4 *)(ks + (size_t)x * 16);
            *(uint2 *)(codes[0] + r * PAD + 4 * chunk) = uint2{w.x, w.y};
            *(uint2 *)(codes[0] + (r + 16) * PAD + 4 * chunk) = uint2{w.z, w.w};
        }
        const uint8_t *vs = a.c.v + slab * (16 * ng) + first * (16 * ng);
        for (uint32_t x = tid; x < 32 * ng; x += 256) {  // channels 4 q .. of one half of a group, rows of one g
            const uint32_t g = x & 3, q = x >> 2 & 3, half = x >> 4 & 1, m = x >> 5, c4 = 8 * m + 4 * half + q;
            if (4 * c4 >= hd) continue;
            uint2 w[4];
#pragma unroll
            for (int e = 0; e < 4; e++) w[e] = *(const uint2 *)(vs + m * 1024 + (4 * q + e) * 64 + g * 16 + half * 8);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                uint32_t in[4], out[4];
#pragma unroll
                for (int e = 0; e < 4; e++) in[e] = (i < 2 ? w[e].x : w[e].y) >> (16 * (i & 1)) & 0xffffu;
                kv4_turn(in, out);
#pragma unroll
                for (int j = 0; j < 4; j++) codes[1][(16 * i + 4 * g + j) * PAD + c4] = (uint16_t)out[j];
            }
        }
        for (uint32_t x = tid; x < 32 * ng; x += 256) {  // keys' multipliers, then values'
            const uint32_t val = x >= 16 * ng, y = x - val * 16 * ng;
            *(uint32_t *)(mul[val] + 4 * y) = *(const uint32_t *)((val ? a.c.vm : a.c.km) + slab * ng + first * ng + 4 * y);
        }
    }
    if (tid < 128) {
        const uint32_t r = tid & 63;
        const bool in = held && r >= t.lo && first + r < a.c.cap;
        scale[tid >> 6][r] = in ? (tid < 64 ? a.c.ks : a.c.vs)[slab + first + r] : __builtin_nanf("");
    }
    __syncthreads();
    // x / words by a multiplication: x < 2^12, words <= 2^6, so that x times the factor's excess is below 2^20
    const uint32_t words = hd / PER, by = ((1u << 20) + words - 1) / words, all = (t.hi - t.lo) * words;
    for (uint32_t x = tid; x < all; x += 256) {
        const uint32_t row = x * by >> 20, w = x - row * words, r = t.lo + row, c = w * PER;
        const size_t to = (size_t)(t.row + row) * a.stride + (size_t)h * hd + c;
#pragma unroll
        for (int val = 0; val < 2; val++) {
            const uint32_t m = held ? mul[val][c / 32 * 64 + (val ? (r >> 2 & 3) * 16 + (r >> 4) * 4 + (r & 3)
                                                                  : (r & 15) * 4 + (r >> 4))] : 0u;
            const float s = scale[val][r];
            float y[PER];
#pragma unroll
            for (uint32_t e = 0; e < PER; e += 4) {
                float z[4];
                kv4_values(held ? codes[val][r * PAD + (c + e) / 4] : 0u, m, s, z);
#pragma unroll
                for (int f = 0; f < 4; f++) y[e + f] = z[f];
            }
            T *d = (val ? v : k) + to;
            if constexpr (sizeof(T) == 4) {
                *(Kv4<float> *)d = Kv4<float>{{y[0], y[1], y[2], y[3]}};
            } else {
                struct __attribute__((packed, aligned(2))) Out {
                    uint32_t v[4];
                } o;
#pragma unroll
                for (int e = 0; e < 4; e++) o.v[e] = f32x2_to_bf16x2(y[2 * e], y[2 * e + 1]);
                *(Out *)d = o;
            }
        }
    }
}

template <typename T>
static void kv4_write_any(const KvRows &a, const T *k, const T *v, hipStream_t s) {
    if (a.tiles) {  // keys, then values
        void (*kern)(KvRows, const T *, const T *) = a.c.hd <= 64    ? kv4_write_tiles<1, T>
                                                     : a.c.hd <= 128 ? kv4_write_tiles<2, T>
                                                                     : kv4_write_tiles<4, T>;
        hipLaunchKernelGGL(kern, dim3((unsigned)(kv_tiles(a.n_rows, a.n) * a.c.Hk), 2), dim3(256), 0, s, a, k, v);
    } else {
        hipLaunchKernelGGL(kv4_write<T>, dim3((unsigned)div_ceil((size_t)a.n_rows * a.c.Hk, 4)), dim3(256), 0, s, a, k, v);
    }
}
void kv4_write_go(const KvRows &a, const void *k, const void *v, int dtype, hipStream_t s) {
    if (dtype == QBK_F32) kv4_write_any(a, (const float *)k, (const float *)v, s);
    else kv4_write_any(a, (const uint16_t *)k, (const uint16_t *)v, s);
}

template <typename T>
static void kv4_read_any(const KvRows &a, T *k, T *v, hipStream_t s) {
    if (a.tiles)
        hipLaunchKernelGGL(kv4_read_tiles<T>, dim3((unsigned)(kv_tiles(a.n_rows, a.n) * a.c.Hk)), dim3(256), 0, s, a, k, v);
    else
        hipLaunchKernelGGL(kv4_read<T>, dim3((unsigned)div_ceil((size_t)a.n_rows * a.c.Hk, 4)), dim3(256), 0, s, a, k, v);
}
void kv4_read_go(const KvRows &a, void *k, void *v, int dtype, hipStream_t s) {
    if (dtype == QBK_F32) kv4_read_any(a, (float *)k, (float *)v, s);
    else kv4_read_any(a, (uint16_t *)k, (uint16_t *)v, s);
}

}  // namespace qbk
