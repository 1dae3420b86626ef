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
#include <math.h>

#include "kvcache_rows.h"

#pragma clang fp contract(off)

namespace qbk {

#define KV4_MUL 448.0f
#define KV4_TOP 2688.0f

__device__ __forceinline__ uint32_t kv4_most(uint32_t a, uint32_t b) { return a > b ? a : b; }

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
#pragma unroll
            for (int o = 1; o <= 4; o <<= 1) group[p] = kv4_most(group[p], (uint32_t)__shfl_xor((int)group[p], o, 64));
        }
        uint32_t top = kv4_most(group[0], group[1]);
#pragma unroll
        for (int o = 8; o <= 16; o <<= 1) top = kv4_most(top, (uint32_t)__shfl_xor((int)top, o, 64));
        const Kv4Row row(top);
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

void kv4_write_go(const KvRows &a, const void *k, const void *v, int dtype, hipStream_t s) {
    const dim3 grid((unsigned)div_ceil((size_t)a.n_rows * a.c.Hk, 4));
    if (dtype == QBK_F32) hipLaunchKernelGGL(kv4_write<float>, grid, dim3(256), 0, s, a, (const float *)k, (const float *)v);
    else hipLaunchKernelGGL(kv4_write<uint16_t>, grid, dim3(256), 0, s, a, (const uint16_t *)k, (const uint16_t *)v);
}

void kv4_read_go(const KvRows &a, void *k, void *v, int dtype, hipStream_t s) {
    const dim3 grid((unsigned)div_ceil((size_t)a.n_rows * a.c.Hk, 4));
    if (dtype == QBK_F32) hipLaunchKernelGGL(kv4_read<float>, grid, dim3(256), 0, s, a, (float *)k, (float *)v);
    else hipLaunchKernelGGL(kv4_read<uint16_t>, grid, dim3(256), 0, s, a, (uint16_t *)k, (uint16_t *)v);
}

}  // namespace qbk
