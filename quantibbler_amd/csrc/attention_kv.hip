// attention_kv.hip -- attention of a batch over the 8-bit KV cache, behind a
// prefix that every sequence shares.
//
// Rows: query row rho = (b sq + t) G + hg of kv head hk is sequence b's query
// t, head hk G + hg.  Every row sees the prefix, so the prefix's items take 16
// NQP rows of all sequences together and read its codes once; a sequence's own
// rows are seen by its sq G rows alone.  Both kinds are items of one launch:
//   item = (kv head, tile of 16 NQ rows, run of 64-row key tiles)
// and leave a partial result (sum of weights, weighted values, reference) per
// row; a second launch joins them.  A wave takes every fourth key tile:
//   S^T = K q^T      v_mfma_f32_16x16x32_f16, codes widened to fp16 (exact)
//   p = exp2(s - M)  online, per query column; M is a whole number, so moving
//                    to another M and joining partials scale by powers of two
//   O^T += V^T p^T   p times the value row's scale, in fp16
// The score layout of the first product is the operand layout of the second
// (kvcache.h), so a tile passes through registers alone.
//
// Roundings: q is scaled by a power of two and held as fp16 (bf16 queries:
// exact but for channels 2^-28 of the row's largest) or as two fp16 halves
// (f32 queries: 22 bits); p times scale likewise, 2^12 above the reference so
// that a weight keeps its bits down to 2^-26 of the largest.  Sums are f32.
#include <math.h>

#include <atomic>

#include "kvcache.h"

#pragma clang fp contract(off)

namespace qbk {

typedef _Float16 kva_h8_t __attribute__((ext_vector_type(8)));
typedef _Float16 kva_h2_t __attribute__((ext_vector_type(2)));
typedef float kva_f4_t __attribute__((ext_vector_type(4)));
typedef uint32_t kva_u4_t __attribute__((ext_vector_type(4)));

#define KVA_WAVES 4
#define KVA_MAX_SPLITS 32  // of the prefix, and of a sequence's own rows

struct KvAttArgs {
    KvView own, pre;
    const void *q;
    void *out;
    const uint32_t *lens;
    float *po;    // [split][hk][rho][hd] weighted values
    float2 *ml;   // [split][hk][rho] reference, sum of weights
    uint32_t first_seq, prefix_seq, prefix_len, max_len;
    uint32_t n, sq, H, G, rows;      // rows = n sq G
    uint32_t sp, ss, rtp, rts;       // splits and row tiles of prefix and own items
    uint32_t n_pre;                  // prefix items
    float scale;                     // log2(e) / sqrt(hd)
};

// Own rows of sequence b that count, and the key tiles a split of them takes:
// at least one a wave, so that short sequences use few splits.
__device__ __forceinline__ uint32_t kva_len(const KvAttArgs &a, uint32_t b) {
    const uint32_t l = a.lens[b];
    return l < a.max_len ? l : a.max_len;
}
__device__ __forceinline__ uint32_t kva_run(uint32_t len, uint32_t splits) {
    const uint32_t t = (len + 63) / 64, c = (t + splits - 1) / splits;
    return c > KVA_WAVES ? c : KVA_WAVES;
}

// Eight codes (two dwords) as fp16.
template <int FMT>
__device__ __forceinline__ kva_h8_t kva_wide(uint32_t lo, uint32_t hi) {
    kva_h2_t p[4];
    if constexpr (FMT == QBK_KV_INT8) {
        const kva_h2_t bias = {(_Float16)1152.0f, (_Float16)1152.0f};
        p[0] = __builtin_bit_cast(kva_h2_t, __builtin_amdgcn_perm(0x64646464u, lo, 0x04010400u)) - bias;
        p[1] = __builtin_bit_cast(kva_h2_t, __builtin_amdgcn_perm(0x64646464u, lo, 0x04030402u)) - bias;
        p[2] = __builtin_bit_cast(kva_h2_t, __builtin_amdgcn_perm(0x64646464u, hi, 0x04010400u)) - bias;
        p[3] = __builtin_bit_cast(kva_h2_t, __builtin_amdgcn_perm(0x64646464u, hi, 0x04030402u)) - bias;
    } else {
        p[0] = __builtin_bit_cast(kva_h2_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)lo, 1.0f, false));
        p[1] = __builtin_bit_cast(kva_h2_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)lo, 1.0f, true));
        p[2] = __builtin_bit_cast(kva_h2_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)hi, 1.0f, false));
        p[3] = __builtin_bit_cast(kva_h2_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)hi, 1.0f, true));
    }
    return kva_h8_t{p[0][0], p[0][1], p[1][0], p[1][1], p[2][0], p[2][1], p[3][0], p[3][1]};
}

// The largest of a value over the four lanes of a query column (l ^ 16, l ^ 32).
__device__ __forceinline__ float kva_max4(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    const float m = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(m), __float_as_uint(m), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float kva_sum4(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    const float m = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(m), __float_as_uint(m), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// exp2 of a difference of references: a power of two, 1 where both are equal
// (two empty ones included).
__device__ __forceinline__ float kva_rescale(float from, float to) {
    return from == to ? 1.0f : __builtin_amdgcn_exp2f(from - to);
}

template <typename T>
__device__ __forceinline__ float kva_in(T x) {
    if constexpr (sizeof(T) == 4) return x;
    else return bf16_to_f32(x);
}
template <typename T>
__device__ __forceinline__ T kva_out(float x) {
    if constexpr (sizeof(T) == 4) return x;
    else return f32_to_bf16(x);
}

// LDS of a body: queries as operands, then (over them) the waves' outputs, and
// the rows' scale, references and sums.
template <int DC, int NQ, bool HI>
struct KvaLds {
    static constexpr int STEPS = 2 * DC;
    static constexpr int Q = NQ * STEPS * 1024 * (HI ? 2 : 1);
    static constexpr int OC = DC < 2 ? 64 : 128;                  // channels joined at a time
    static constexpr int O = KVA_WAVES * 16 * (OC + 4) * 4;
    static constexpr int BODY = Q > O ? Q : O;
    static constexpr int BYTES = BODY + NQ * 16 * 4 * (1 + 2 * KVA_WAVES);
};

// Rows of a body from row0 on: row r is query (b, t) = base + r's quotient by
// G, head the remainder.  The float quotient is exact: x + 1/2 is half a unit
// from every multiple of G and below 2^21 (G at most 2^20, checked on the host).
struct KvaRow {
    uint32_t base, rem, G;
    float inv;
    __device__ __forceinline__ KvaRow(const KvAttArgs &a, uint32_t row0)
        : base(row0 / a.G), rem(row0 % a.G), G(a.G), inv(1.0f / (float)a.G) {}
    __device__ __forceinline__ void at(uint32_t r, uint32_t &query, uint32_t &head) const {
        const uint32_t x = rem + r, d = (uint32_t)(((float)x + 0.5f) * inv);
        query = base + d;
        head = x - d * G;
    }
};

// Four values of a row at any alignment (one load on this machine).
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Kva4 {
    T v[4];
};

// Queries row0 .. row0 + n_rows - 1 (at most 16 NT) of kv head hk into LDS as
// the B operands of K q^T, [tile][step][lane][16 bytes], for f32 queries the
// low halves behind them; cqs[r]: the factor that scores of row r still need.
// 16 DC lanes a row, four channels a lane, every row's load before the first
// is used (a row at a time, the 128 rows of the widest body took 25 us).
template <int DC, int NT, typename T>
__device__ __forceinline__ void kva_queries(const KvAttArgs &a, char *qs, float *cqs, uint32_t row0, uint32_t n_rows,
                                            uint32_t hk) {
    constexpr int STEPS = 2 * DC, LANES = 16 * DC, AT_ONCE = KVA_WAVES * 64 / LANES, N = 16 * NT / AT_ONCE;
    const int tid = threadIdx.x, hd = (int)a.own.hd, c = 4 * (tid % LANES), r0 = tid / LANES;
    const KvaRow rows(a, row0);
    Kva4<T> raw[N];
#pragma unroll
    for (int k = 0; k < N; k++) {
        const uint32_t r = r0 + k * AT_ONCE;
        uint32_t query, head;
        rows.at(r < n_rows ? r : 0, query, head);
        const T *src = (const T *)a.q + ((size_t)query * a.H + (size_t)hk * a.G + head) * hd;
        raw[k] = *(const Kva4<T> *)(src + (c < hd ? c : 0));
    }
#pragma unroll
    for (int k = 0; k < N; k++) {
        const int r = r0 + k * AT_ONCE;
        float x[4];
        uint32_t top = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            x[e] = r < (int)n_rows && c < hd ? kva_in<T>(raw[k].v[e]) : 0.0f;
            const uint32_t b = __float_as_uint(x[e]) & 0x7fffffffu;
            top = b > top ? b : top;
        }
#pragma unroll
        for (int o = LANES / 2; o >= 1; o >>= 1) {
            const uint32_t b = (uint32_t)__shfl_xor((int)top, o, 64);
            top = b > top ? b : top;
        }
        // the largest channel to [8, 16): both halves of every channel within fp16
        const bool whole = top < 0x7f800000u;
        uint32_t ex = top >> 23;
        ex = ex < 30 ? 30 : ex > 254 ? 254 : ex;
        const float f = __uint_as_float((257 - ex) << 23);
        kva_h2_t hi[2], lo[2];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float y = whole ? x[e] * f : 0.0f;
            const _Float16 h = (_Float16)y;
            hi[e >> 1][e & 1] = h;
            lo[e >> 1][e & 1] = (_Float16)(y - (float)h);
        }
        // channel c: chunk c / 16 -> step 2 (chunk / 4) + (c % 16) / 8, operand lane (chunk % 4, column r % 16)
        const int chunk = c >> 4, step = 2 * (chunk >> 2) + ((c >> 3) & 1);
        const size_t at = (size_t)(((r >> 4) * STEPS + step) * 64 + (chunk & 3) * 16 + (r & 15)) * 16 + (c & 7) * 2;
        *(uint2 *)(qs + at) = uint2{__builtin_bit_cast(uint32_t, hi[0]), __builtin_bit_cast(uint32_t, hi[1])};
        if constexpr (sizeof(T) == 4)
            *(uint2 *)(qs + NT * STEPS * 1024 + at) =
                uint2{__builtin_bit_cast(uint32_t, lo[0]), __builtin_bit_cast(uint32_t, lo[1])};
        if (c == 0) cqs[r] = whole ? a.scale * __uint_as_float((ex - 3) << 23) : __builtin_nanf("");
    }
}

// Value scales to 2^12 over a power of two at or above every one so far
// (vref; the outputs follow when it moves).
template <int NQ, int CT>
__device__ __forceinline__ void kva_value_scales(kva_f4_t (&vs)[4], float &vref, float &vinv, kva_f4_t (&o)[NQ][CT]) {
    float vm = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; i++) vm = fmaxf(fmaxf(fmaxf(vm, vs[i][0]), fmaxf(vs[i][1], vs[i][2])), vs[i][3]);
    if (__ballot(vm > vref)) {
        vm = kva_max4(vm);
        const uint32_t e = (__float_as_uint(vm) >> 23) + 1;  // scales are 2^-107 .. 2^122
        const float to = __uint_as_float(e << 23);
        vinv = __uint_as_float((266 - e) << 23);
        const float f = vref * __uint_as_float((254 - e) << 23);
#pragma unroll
        for (int q = 0; q < NQ; q++)
#pragma unroll
            for (int ct = 0; ct < CT; ct++) o[q][ct] *= f;
        vref = to;
    }
#pragma unroll
    for (int i = 0; i < 4; i++) vs[i] *= vinv;
}

// One query tile's scores (16 keys a lane: 16 i + j past key) to weights: the
// reference moves when a score passes it eightfold, sum and outputs with it;
// p times the value scales as operands ph (and pl, the halves' rests).
template <int CT, bool HI>
__device__ __forceinline__ void kva_softmax(const kva_f4_t (&s)[4], const kva_f4_t (&vs)[4], float cq, bool masked,
                                            uint32_t key, uint32_t lim, float &ref, float &sum, kva_f4_t (&o)[CT],
                                            kva_h8_t (&ph)[2], kva_h8_t (&pl)[2]) {
    float t[4][4], tm = -INFINITY;
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            t[i][j] = s[i][j];
            if (masked && key + 16 * i + j >= lim) t[i][j] = -INFINITY;
            tm = fmaxf(tm, t[i][j]);
        }
    if (__ballot(tm * cq > ref + 3.0f)) {
        const float to = fmaxf(ref, ceilf(kva_max4(tm) * cq));
        const float f = kva_rescale(ref, to);
        sum *= f;
#pragma unroll
        for (int ct = 0; ct < CT; ct++) o[ct] *= f;
        ref = to;
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        float w[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const bool out = masked && key + 16 * i + j >= lim;
            float p = __builtin_amdgcn_exp2f(__builtin_fmaf(t[i][j], cq, -ref));
            if (out) p = 0.0f;
            sum += p;
            w[j] = p * vs[i][j];
            if (out) w[j] = 0.0f;  // whatever the scale holds
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const _Float16 h = (_Float16)w[j];
            ph[i >> 1][4 * (i & 1) + j] = h;
            if constexpr (HI) pl[i >> 1][4 * (i & 1) + j] = (_Float16)(w[j] - (float)h);
        }
    }
}

// Rows row0 .. row0 + n_rows - 1 (at most 16 NQ) of kv head hk over key tiles
// tile0 .. tile1 - 1 of the slab k, v, ks, vs.  Row r of the body sees keys
// below limit(r), none of them at or past `written`.
template <int FMT, int DC, int NQ, typename T, class Limit>
__device__ __forceinline__ void kva_body(const KvAttArgs &a, char *smem, uint32_t row0, uint32_t n_rows, uint32_t hk,
                                         const uint8_t *kcode, const uint8_t *vcode, const float *ksc,
                                         const float *vsc, uint32_t tile0, uint32_t tile1, uint32_t written,
                                         Limit limit, uint32_t split, bool last) {
    constexpr bool HI = sizeof(T) == 4;
    using L = KvaLds<DC, NQ, HI>;
    constexpr int STEPS = L::STEPS;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, col = lane & 15, g = lane >> 4;
    const int hd = (int)a.own.hd, nc = hd / 16;
    char *qs = smem;
    float *cqs = (float *)(smem + L::BODY), *refs = cqs + NQ * 16, *sums = refs + KVA_WAVES * NQ * 16;

    // A tile's codes and scales travel while the one before is worked on: keys
    // and their scales are asked for again as soon as the scores are formed,
    // values once they are added, the first of both before the queries are read.
    kva_u4_t kc[DC][4], vc[4 * DC];
    kva_f4_t ks[4], vs[4];
    const int spread = col * 16;
    auto load_k = [&](uint32_t tt) {
        const uint8_t *kt = kcode + (size_t)tt * 64 * hd + spread;
        const float *st = ksc + (size_t)tt * 64 + 4 * g;
#pragma unroll
        for (int i = 0; i < 4; i++) ks[i] = *(const kva_f4_t *)(st + 16 * i);
#pragma unroll
        for (int c = 0; c < DC; c++) {
            if (4 * c >= nc) continue;
            const int chunk = 4 * c + g < nc ? 4 * c + g : nc - 1;  // past the last chunk q is zero
#pragma unroll
            for (int i = 0; i < 4; i++) kc[c][i] = *(const kva_u4_t *)(kt + (i * nc + chunk) * 256);
        }
    };
    auto load_v = [&](uint32_t tt) {
        const uint8_t *vt = vcode + (size_t)tt * 64 * hd + col * 64 + g * 16;
        const float *st = vsc + (size_t)tt * 64 + 4 * g;
#pragma unroll
        for (int i = 0; i < 4; i++) vs[i] = *(const kva_f4_t *)(st + 16 * i);
#pragma unroll
        for (int ct = 0; ct < 4 * DC; ct++)
            if (ct < nc) vc[ct] = *(const kva_u4_t *)(vt + ct * 1024);
    };
    const uint32_t first = tile0 + wave;
    if (first < tile1) {
        load_k(first);
        load_v(first);
    }

    kva_queries<DC, NQ, T>(a, qs, cqs, row0, n_rows, hk);
    __syncthreads();

    kva_f4_t o[NQ][4 * DC];
    float ref[NQ], sum[NQ], cq[NQ];
    uint32_t lim[NQ];
    uint32_t least = 0xFFFFFFFFu;  // keys below it are seen by every row
#pragma unroll
    for (int q = 0; q < NQ; q++) {
#pragma unroll
        for (int ct = 0; ct < 4 * DC; ct++) o[q][ct] = kva_f4_t{0, 0, 0, 0};
        ref[q] = -INFINITY;
        sum[q] = 0.0f;
        cq[q] = cqs[16 * q + col];
        const uint32_t r = 16 * q + col;
        lim[q] = limit(r < n_rows ? r : n_rows - 1);
    }
    least = limit(0);
    float vref = 0.0f, vinv = 0.0f;  // a power of two at or above every value scale so far, and 2^12 over it

    for (uint32_t tt = first; tt < tile1; tt += KVA_WAVES) {
        const uint32_t key0 = tt * 64;
        const bool masked = key0 + 64 > least, more = tt + KVA_WAVES < tile1;
        if (masked) {  // what was never written takes no part, whatever it holds
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (key0 + 16 * i + 4 * g + j >= written) vs[i][j] = 0.0f;
        }
        kva_f4_t s[NQ][4];
#pragma unroll
        for (int q = 0; q < NQ; q++)
#pragma unroll
            for (int i = 0; i < 4; i++) s[q][i] = kva_f4_t{0, 0, 0, 0};
#pragma unroll
        for (int c = 0; c < DC; c++) {
            if (4 * c >= nc) continue;
#pragma unroll
            for (int u = 0; u < 2; u++) {
                kva_h8_t kf[4];
#pragma unroll
                for (int i = 0; i < 4; i++) kf[i] = kva_wide<FMT>(kc[c][i][2 * u], kc[c][i][2 * u + 1]);
#pragma unroll
                for (int q = 0; q < NQ; q++) {
                    const kva_h8_t qf = *(const kva_h8_t *)(qs + (size_t)((q * STEPS + 2 * c + u) * 64 + lane) * 16);
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        s[q][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[i], qf, s[q][i], 0, 0, 0);
                    if constexpr (HI) {
                        const kva_h8_t ql = *(const kva_h8_t *)(qs + NQ * STEPS * 1024 +
                                                                (size_t)((q * STEPS + 2 * c + u) * 64 + lane) * 16);
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            s[q][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[i], ql, s[q][i], 0, 0, 0);
                    }
                }
            }
        }
        // scores in units of 1 / cq; the key registers are free again
#pragma unroll
        for (int q = 0; q < NQ; q++)
#pragma unroll
            for (int i = 0; i < 4; i++) s[q][i] *= ks[i];
        if (more) load_k(tt + KVA_WAVES);
        kva_value_scales<NQ, 4 * DC>(vs, vref, vinv, o);

        kva_h8_t ph[NQ][2], pl[NQ][2];
#pragma unroll
        for (int q = 0; q < NQ; q++) {
            kva_softmax<4 * DC, HI>(s[q], vs, cq[q], masked, key0 + 4 * g, lim[q], ref[q], sum[q], o[q], ph[q], pl[q]);
        }
        // fp8 rows that were never written may hold NaN codes
        uint32_t keep[4] = {~0u, ~0u, ~0u, ~0u};
        if (FMT == QBK_KV_FP8 && masked) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t k0 = key0 + 16 * i + 4 * g, left = written > k0 ? written - k0 : 0;
                keep[i] = left >= 4 ? ~0u : (1u << (8 * left)) - 1u;
            }
        }
#pragma unroll
        for (int ct = 0; ct < 4 * DC; ct++) {
            if (ct >= nc) continue;
            kva_u4_t w = vc[ct];
            if (FMT == QBK_KV_FP8) {
#pragma unroll
                for (int i = 0; i < 4; i++) w[i] &= keep[i];
            }
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const kva_h8_t vf = kva_wide<FMT>(w[2 * u], w[2 * u + 1]);
#pragma unroll
                for (int q = 0; q < NQ; q++) {
                    o[q][ct] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, ph[q][u], o[q][ct], 0, 0, 0);
                    if constexpr (HI)
                        o[q][ct] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pl[q][u], o[q][ct], 0, 0, 0);
                }
            }
        }
        if (more) load_v(tt + KVA_WAVES);
    }

    // join the waves on each row's largest reference
#pragma unroll
    for (int q = 0; q < NQ; q++) {
        const float l = kva_sum4(sum[q]);
        if (g == 0) {
            refs[(wave * NQ + q) * 16 + col] = ref[q];
            sums[(wave * NQ + q) * 16 + col] = l;
        }
    }
    __syncthreads();
    auto largest = [&](int r) {  // row r of the body
        float m = refs[r];
#pragma unroll
        for (int w = 1; w < KVA_WAVES; w++) m = fmaxf(m, refs[w * NQ * 16 + r]);
        return m;
    };
    constexpr int OC = L::OC, LD = OC + 4;
    float *ob = (float *)smem;  // [wave][16 rows][LD]
    const size_t part = ((size_t)split * a.own.Hk + hk) * a.rows + row0;
#pragma unroll
    for (int q = 0; q < NQ; q++) {
        const float f = kva_rescale(ref[q], largest(16 * q + col)) * vref * 0x1p-12f;
#pragma unroll
        for (int c0 = 0; c0 < 64 * DC; c0 += OC) {
            if (c0 >= hd) continue;
            __syncthreads();  // what the region held has been read
#pragma unroll
            for (int k = 0; k < OC / 16; k++)
                *(kva_f4_t *)(ob + (wave * 16 + col) * LD + 16 * k + 4 * g) = o[q][c0 / 16 + k] * f;
            __syncthreads();
            for (int x = tid; x < 16 * OC; x += 64 * KVA_WAVES) {
                const int r = x / OC, c = x % OC;
                if (16 * q + r >= (int)n_rows || c0 + c >= hd) continue;
                float v = 0.0f;
#pragma unroll
                for (int w = 0; w < KVA_WAVES; w++) v += ob[(w * 16 + r) * LD + c];
                if (last) {
                    float l = 0.0f;
                    const float m = largest(16 * q + r);
#pragma unroll
                    for (int w = 0; w < KVA_WAVES; w++)
                        l += sums[(w * NQ + q) * 16 + r] * kva_rescale(refs[(w * NQ + q) * 16 + r], m);
                    const uint32_t rho = row0 + 16 * q + r;
                    T *dst = (T *)a.out + ((size_t)(rho / a.G) * a.H + (size_t)hk * a.G + rho % a.G) * hd;
                    dst[c0 + c] = kva_out<T>(l == 0.0f ? 0.0f : v / l);
                } else {
                    a.po[(part + 16 * q + r) * hd + c0 + c] = v;
                }
            }
        }
        if (!last && tid < 16 && 16 * q + tid < (int)n_rows) {
            const float m = largest(16 * q + tid);
            float l = 0.0f;
#pragma unroll
            for (int w = 0; w < KVA_WAVES; w++)
                l += sums[(w * NQ + q) * 16 + tid] * kva_rescale(refs[(w * NQ + q) * 16 + tid], m);
            a.ml[part + 16 * q + tid] = float2{m, l};
        }
    }
}

// The body of many rows: a wave 16 NQ rows of the 64 NQ, every wave every key
// tile.  A tile is widened once for the four of them, a quarter by each wave,
// into LDS in operand order (each 16-byte access of a wave is 1 KiB in a row),
// while the next tile's codes travel; two buffers and one barrier a tile (256
// channels: one buffer, two barriers).
template <int DC>
struct KvaStage {
    static constexpr int KEYS = 4 * 2 * DC * 1024, BYTES = 2 * KEYS + 512, BUFS = DC < 4 ? 2 : 1;
};
template <int DC, int NQ, bool HI>
struct KvaWideLds {
    static constexpr int Q = 4 * NQ * 2 * DC * 1024 * (HI ? 2 : 1);  // under the stages, read into registers first
    static constexpr int S = KvaStage<DC>::BYTES * KvaStage<DC>::BUFS;
    static constexpr int BODY = Q > S ? Q : S;
    static constexpr int BYTES = BODY + 64 * NQ * 4;
};

template <int FMT, int DC, int NQ, typename T, class Limit>
__device__ __forceinline__ void kva_wide_body(const KvAttArgs &a, char *smem, uint32_t row0, uint32_t n_rows,
                                              uint32_t hk, const uint8_t *kcode, const uint8_t *vcode,
                                              const float *ksc, const float *vsc, uint32_t tile0, uint32_t tile1,
                                              uint32_t written, Limit limit, uint32_t split, bool last) {
    constexpr bool HI = sizeof(T) == 4;
    constexpr int STEPS = 2 * DC, BUFS = KvaStage<DC>::BUFS;
    using L = KvaWideLds<DC, NQ, HI>;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, col = lane & 15, g = lane >> 4;
    const int hd = (int)a.own.hd, nc = hd / 16;
    float *cqs = (float *)(smem + L::BODY);

    kva_u4_t kc[DC], vc[DC];  // this wave's quarter: keys of block `wave`, channel tiles wave, wave + 4, ..
    float sc = 0.0f;          // threads 0 .. 63 a key's scale, 64 .. 127 a value's
    auto load = [&](uint32_t tt) {
        const uint8_t *kt = kcode + (size_t)tt * 64 * hd + (size_t)wave * 16 * hd + col * 16;
        const uint8_t *vt = vcode + (size_t)tt * 64 * hd + col * 64 + g * 16;
#pragma unroll
        for (int c = 0; c < DC; c++) {
            const int chunk = 4 * c + g < nc ? 4 * c + g : nc - 1;  // past the last chunk q is zero
            kc[c] = *(const kva_u4_t *)(kt + chunk * 256);
            if (wave + 4 * c < nc) vc[c] = *(const kva_u4_t *)(vt + (wave + 4 * c) * 1024);
        }
        if (wave < 2) sc = (wave ? vsc : ksc)[(size_t)tt * 64 + lane];
    };
    auto stage = [&](uint32_t tt, char *buf) {
        const uint32_t key0 = tt * 64;
        kva_u4_t keep = {~0u, ~0u, ~0u, ~0u};
        const bool tail = key0 + 64 > written;  // rows that were never written take no part, whatever they hold
        if (FMT == QBK_KV_FP8 && tail) {        // NaN codes
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t k0 = key0 + 16 * i + 4 * g, left = written > k0 ? written - k0 : 0;
                keep[i] = left >= 4 ? ~0u : (1u << (8 * left)) - 1u;
            }
        }
#pragma unroll
        for (int c = 0; c < DC; c++) {
#pragma unroll
            for (int u = 0; u < 2; u++)
                *(kva_h8_t *)(buf + ((wave * STEPS + 2 * c + u) * 64 + lane) * 16) =
                    kva_wide<FMT>(kc[c][2 * u], kc[c][2 * u + 1]);
            if (wave + 4 * c < nc) {
                const kva_u4_t w = vc[c] & keep;
#pragma unroll
                for (int u = 0; u < 2; u++)
                    *(kva_h8_t *)(buf + KvaStage<DC>::KEYS + ((2 * (wave + 4 * c) + u) * 64 + lane) * 16) =
                        kva_wide<FMT>(w[2 * u], w[2 * u + 1]);
            }
        }
        if (wave < 2)
            *(float *)(buf + 2 * KvaStage<DC>::KEYS + wave * 256 + lane * 4) = tail && key0 + lane >= written ? 0.0f : sc;
    };
    if (tile0 < tile1) load(tile0);
    kva_queries<DC, 4 * NQ, T>(a, smem, cqs, row0, n_rows, hk);
    __syncthreads();
    kva_h8_t qh[NQ][STEPS], ql[NQ][STEPS];
    kva_f4_t o[NQ][4 * DC];
    float ref[NQ], sum[NQ], cq[NQ], vref = 0.0f, vinv = 0.0f;
    uint32_t lim[NQ];
    const uint32_t my0 = wave * 16 * NQ;  // this wave's first row
#pragma unroll
    for (int q = 0; q < NQ; q++) {
#pragma unroll
        for (int st = 0; st < STEPS; st++) {
            const char *at = smem + (((wave * NQ + q) * STEPS + st) * 64 + lane) * 16;
            qh[q][st] = *(const kva_h8_t *)at;
            if constexpr (HI) ql[q][st] = *(const kva_h8_t *)(at + 4 * NQ * STEPS * 1024);
        }
#pragma unroll
        for (int ct = 0; ct < 4 * DC; ct++) o[q][ct] = kva_f4_t{0, 0, 0, 0};
        ref[q] = -INFINITY;
        sum[q] = 0.0f;
        cq[q] = cqs[my0 + 16 * q + col];
        const uint32_t r = my0 + 16 * q + col;
        lim[q] = limit(r < n_rows ? r : n_rows - 1);
    }
    const bool rows = my0 < n_rows;
    const uint32_t least = limit(rows ? my0 : 0), end = my0 + 16 * NQ < n_rows ? my0 + 16 * NQ : n_rows;
    const uint32_t most = rows ? limit(end - 1) : 0;  // no row of the wave sees keys from here on
    __syncthreads();  // the queries are read

    for (uint32_t tt = tile0; tt < tile1; tt++) {
        char *buf = smem + (BUFS == 2 ? ((tt - tile0) & 1) * KvaStage<DC>::BYTES : 0);
        if (BUFS == 1 && tt > tile0) __syncthreads();
        stage(tt, buf);
        __syncthreads();
        if (tt + 1 < tile1) load(tt + 1);
        const uint32_t key0 = tt * 64;
        if (key0 >= most) continue;
        const bool masked = key0 + 64 > least;
        kva_f4_t ks[4], vs[4], s[NQ][4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            ks[i] = *(const kva_f4_t *)(buf + 2 * KvaStage<DC>::KEYS + (16 * i + 4 * g) * 4);
            vs[i] = *(const kva_f4_t *)(buf + 2 * KvaStage<DC>::KEYS + 256 + (16 * i + 4 * g) * 4);
#pragma unroll
            for (int q = 0; q < NQ; q++) s[q][i] = kva_f4_t{0, 0, 0, 0};
        }
#pragma unroll
        for (int st = 0; st < STEPS; st++) {
            if (4 * (st / 2) >= nc) continue;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const kva_h8_t kf = *(const kva_h8_t *)(buf + ((i * STEPS + st) * 64 + lane) * 16);
#pragma unroll
                for (int q = 0; q < NQ; q++) {
                    s[q][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qh[q][st], s[q][i], 0, 0, 0);
                    if constexpr (HI) s[q][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, ql[q][st], s[q][i], 0, 0, 0);
                }
            }
        }
        kva_value_scales<NQ, 4 * DC>(vs, vref, vinv, o);
        kva_h8_t ph[NQ][2], pl[NQ][2];
#pragma unroll
        for (int q = 0; q < NQ; q++) {
#pragma unroll
            for (int i = 0; i < 4; i++) s[q][i] *= ks[i];
            kva_softmax<4 * DC, HI>(s[q], vs, cq[q], masked, key0 + 4 * g, lim[q], ref[q], sum[q], o[q], ph[q], pl[q]);
        }
#pragma unroll
        for (int ct = 0; ct < 4 * DC; ct++) {
            if (ct >= nc) continue;
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const kva_h8_t vf =
                    *(const kva_h8_t *)(buf + KvaStage<DC>::KEYS + ((2 * ct + u) * 64 + lane) * 16);
#pragma unroll
                for (int q = 0; q < NQ; q++) {
                    o[q][ct] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, ph[q][u], o[q][ct], 0, 0, 0);
                    if constexpr (HI) o[q][ct] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pl[q][u], o[q][ct], 0, 0, 0);
                }
            }
        }
    }
    const size_t part = ((size_t)split * a.own.Hk + hk) * a.rows + row0;
#pragma unroll
    for (int q = 0; q < NQ; q++) {
        const uint32_t r = my0 + 16 * q + col;
        const float l = kva_sum4(sum[q]), f = vref * 0x1p-12f;
        if (r >= n_rows) continue;
        if (last) {
            const uint32_t rho = row0 + r;
            T *dst = (T *)a.out + ((size_t)(rho / a.G) * a.H + (size_t)hk * a.G + rho % a.G) * hd + 4 * g;
#pragma unroll
            for (int ct = 0; ct < 4 * DC; ct++) {
                if (ct >= nc) continue;
#pragma unroll
                for (int j = 0; j < 4; j++) dst[16 * ct + j] = kva_out<T>(l == 0.0f ? 0.0f : o[q][ct][j] * f / l);
            }
        } else {
            float *dst = a.po + (part + r) * hd + 4 * g;
#pragma unroll
            for (int ct = 0; ct < 4 * DC; ct++)
                if (ct < nc) *(kva_f4_t *)(dst + 16 * ct) = o[q][ct] * f;
            if (g == 0) a.ml[part + r] = float2{ref[q], l};
        }
    }
}

// W 0: a body of up to 16 rows, each wave every fourth key tile; else one of 64 W.
template <int FMT, int DC, int W, typename T, class... ARGS>
__device__ __forceinline__ void kva_any(ARGS &&...args) {
    if constexpr (W == 0) kva_body<FMT, DC, 1, T>(args...);
    else kva_wide_body<FMT, DC, W, T>(args...);
}

template <int FMT, int DC, int NQP, int NQS, typename T>
__global__ void __launch_bounds__(64 * KVA_WAVES, DC < 4 ? 2 : 1) kva_items(KvAttArgs a) {
    extern __shared__ char smem[];
    const uint32_t Hk = a.own.Hk;
    const bool last = a.sp + a.ss == 1;
    if (blockIdx.x < a.n_pre) {
        // kv heads next to each other: with eight of them each stays on one XCD, whose L2 serves its row tiles
        const uint32_t hk = blockIdx.x % Hk, x = blockIdx.x / Hk, rt = x % a.rtp, split = x / a.rtp;
        constexpr uint32_t R = NQP ? 64 * NQP : 16;
        const uint32_t row0 = rt * R, n_rows = a.rows - row0 < R ? a.rows - row0 : R;
        const uint32_t tiles = (a.prefix_len + 63) / 64, run = (tiles + a.sp - 1) / a.sp;
        const uint32_t t0 = split * run < tiles ? split * run : tiles, t1 = t0 + run < tiles ? t0 + run : tiles;
        const size_t slab = a.pre.slab(a.prefix_seq, hk);
        const uint32_t len = a.prefix_len;
        kva_any<FMT, DC, NQP, T>(a, smem, row0, n_rows, hk, a.pre.k + slab * a.pre.hd, a.pre.v + slab * a.pre.hd,
                                  a.pre.ks + slab, a.pre.vs + slab, t0, t1, len, [&](uint32_t) { return len; }, split,
                                  last);
        return;
    }
    const uint32_t item = blockIdx.x - a.n_pre;
    const uint32_t hk = item % Hk, x = item / Hk, rt = x % a.rts, y = x / a.rts, b = y % a.n, split = y / a.n;
    const uint32_t len = kva_len(a, b), tiles = (len + 63) / 64, run = kva_run(len, a.ss);
    if (split * run >= tiles && split > 0) return;  // split 0 is there for a sequence with no rows
    constexpr uint32_t R = NQS ? 64 * NQS : 16;
    const uint32_t per = a.sq * a.G, r0 = rt * R, n_rows = per - r0 < R ? per - r0 : R;
    const uint32_t sq = a.sq;
    const KvaRow rows(a, r0);
    auto limit = [&](uint32_t r) {  // own rows seen by row r of the body: len - sq + t + 1, none where that is negative
        uint32_t t, head;
        rows.at(r, t, head);
        const uint32_t up = len + t + 1;
        return up > sq ? up - sq : 0;
    };
    const uint32_t most = (limit(n_rows - 1) + 63) / 64;
    uint32_t t1 = split * run + run;
    t1 = t1 < most ? t1 : most;
    const size_t slab = a.own.slab(a.first_seq + b, hk);
    kva_any<FMT, DC, NQS, T>(a, smem, b * per + r0, n_rows, hk, a.own.k + slab * a.own.hd, a.own.v + slab * a.own.hd,
                              a.own.ks + slab, a.own.vs + slab, split * run, t1, len, limit, a.sp + split, last);
}

// A wave a row and kv head: the partial results of its splits on their largest
// reference.
template <typename T>
__global__ void __launch_bounds__(256) kva_join(KvAttArgs a) {
    const size_t item = (size_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const uint32_t lane = threadIdx.x & 63, Hk = a.own.Hk, hd = a.own.hd;
    if (item >= (size_t)a.rows * Hk) return;
    const uint32_t hk = (uint32_t)(item / a.rows), rho = (uint32_t)(item % a.rows);
    uint32_t splits = a.sp;
    if (a.ss) {
        const uint32_t len = kva_len(a, rho / (a.sq * a.G)), run = kva_run(len, a.ss), k = ((len + 63) / 64 + run - 1) / run;
        splits += k ? k : 1;
    }
    float m = -INFINITY, l = 0.0f;
    if (lane < splits) {
        const float2 v = a.ml[((size_t)lane * Hk + hk) * a.rows + rho];
        m = v.x;
        l = v.y;
    }
    float M = m;
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) M = fmaxf(M, __shfl_xor(M, o, 64));
    const float f = kva_rescale(m, M);
    float lf = lane < splits ? l * f : 0.0f;
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) lf += __shfl_xor(lf, o, 64);
    // four channels a lane, 64 / (hd / 4) splits at a time, the loads of four such steps in flight
    const uint32_t lanes = hd <= 64 ? 16 : hd <= 128 ? 32 : 64, c = 4 * (lane % lanes), step = 64 / lanes;
    kva_f4_t v = {0, 0, 0, 0};
    const float *src = a.po + ((size_t)hk * a.rows + rho) * hd + (c < hd ? c : 0);
    const size_t apart = (size_t)Hk * a.rows * hd;
    for (uint32_t s0 = 0; s0 < splits; s0 += 4 * step) {
        kva_f4_t x[4];
        float fs[4];
#pragma unroll
        for (uint32_t k = 0; k < 4; k++) {
            const uint32_t s = s0 + k * step + lane / lanes, at = s < splits ? s : splits - 1;
            x[k] = *(const kva_f4_t *)(src + at * apart);
            fs[k] = __shfl(f, (int)at, 64);
            if (s >= splits) x[k] = kva_f4_t{0, 0, 0, 0};
        }
#pragma unroll
        for (int k = 0; k < 4; k++) v += x[k] * fs[k];
    }
#pragma unroll
    for (int o = 32; o >= 16; o >>= 1)
        if (lanes <= (uint32_t)o)
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] += __shfl_xor(v[e], o, 64);
    if (lane >= lanes || c >= hd) return;
    T *dst = (T *)a.out + ((size_t)(rho / a.G) * a.H + (size_t)hk * a.G + rho % a.G) * hd + c;
#pragma unroll
    for (int e = 0; e < 4; e++) dst[e] = kva_out<T>(lf == 0.0f ? 0.0f : v[e] / lf);
}

// How a call is cut: row tiles (16 NQ rows) and splits of the prefix and of
// the sequences' own rows.
struct KvaPlan {
    uint32_t nqp, nqs, rtp, rts, sp, ss;
    uint64_t items;
    size_t bytes;
};

static KvaPlan kva_plan(const qbk_kv_shape *s, size_t n_heads, size_t n, size_t sq, size_t max_len, size_t prefix_len) {
    KvaPlan p{};
    const size_t Hk = s->n_kv_heads, G = n_heads / Hk, rows = n * sq * G, per = sq * G;
    const uint32_t most = s->head_dim > 128 ? 1 : 2;
    auto rows_of = [](uint32_t w) { return w ? 64 * w : 16; };
    p.nqs = per > 16 && max_len ? most : 0;
    p.nqp = p.nqs ? most : rows > 16 && prefix_len ? (rows > 64 ? most : 1) : 0;
    p.rtp = (uint32_t)div_ceil(rows, rows_of(p.nqp));
    p.rts = (uint32_t)div_ceil(per, rows_of(p.nqs));
    auto splits = [](size_t tiles, uint64_t others, uint64_t target) -> uint32_t {
        uint64_t most = div_ceil(tiles, KVA_WAVES), want = div_ceil(target, others ? others : 1);
        want = want < most ? want : most;
        return (uint32_t)(want < 1 ? 1 : want > KVA_MAX_SPLITS ? KVA_MAX_SPLITS : want);
    };
    if (prefix_len) p.sp = splits(div_ceil(prefix_len, 64), (uint64_t)Hk * p.rtp, 512);
    if (max_len) p.ss = splits(div_ceil(max_len, 64), (uint64_t)n * Hk * p.rts, 1024);
    p.items = (uint64_t)Hk * p.rtp * p.sp + (uint64_t)n * Hk * p.rts * p.ss;
    p.bytes = p.sp + p.ss > 1 ? round_up((size_t)(p.sp + p.ss) * Hk * rows * (s->head_dim * 4 + 8), 256) : 0;
    return p;
}

template <int FMT, int DC, int NQP, int NQS, typename T>
static int kva_launch(const KvAttArgs &a, uint64_t items, int device, hipStream_t st) {
    constexpr bool HI = sizeof(T) == 4;
    constexpr int N = KvaLds<DC, 1, HI>::BYTES, W = KvaWideLds<DC, NQP ? NQP : 1, HI>::BYTES;
    constexpr int lds = NQP == 0 ? N : W > N ? W : N;
    void (*k)(KvAttArgs) = kva_items<FMT, DC, NQP, NQS, T>;
    if (lds > 64 * 1024) {  // once a device
        static std::atomic<uint64_t> asked{0};
        const uint64_t bit = device < 64 ? 1ull << device : 0;
        if (!bit || !(asked.load(std::memory_order_acquire) & bit)) {
            QBK_HIP(hipFuncSetAttribute((const void *)k, hipFuncAttributeMaxDynamicSharedMemorySize, lds));
            asked.fetch_or(bit, std::memory_order_release);
        }
    }
    hipLaunchKernelGGL(k, dim3((unsigned)items), dim3(64 * KVA_WAVES), lds, st, a);
    QBK_HIP(hipGetLastError());
    return QBK_OK;
}

template <int FMT, int DC, typename T>
static int kva_dispatch_dc(const KvAttArgs &a, const KvaPlan &p, int device, hipStream_t st) {
    if constexpr (DC < 4) {
        if (p.nqs == 2) return kva_launch<FMT, DC, 2, 2, T>(a, p.items, device, st);
        if (p.nqp == 2) return kva_launch<FMT, DC, 2, 0, T>(a, p.items, device, st);
    } else {
        if (p.nqs == 1) return kva_launch<FMT, DC, 1, 1, T>(a, p.items, device, st);
    }
    if (p.nqp == 1) return kva_launch<FMT, DC, 1, 0, T>(a, p.items, device, st);
    return kva_launch<FMT, DC, 0, 0, T>(a, p.items, device, st);
}

template <int FMT, typename T>
static int kva_dispatch(const KvAttArgs &a, const KvaPlan &p, int device, hipStream_t st) {
    if (a.own.hd > 128) return kva_dispatch_dc<FMT, 4, T>(a, p, device, st);
    if (a.own.hd > 64) return kva_dispatch_dc<FMT, 2, T>(a, p, device, st);
    return kva_dispatch_dc<FMT, 1, T>(a, p, device, st);
}

// The checks that need no buffers, in one place for the size and the call.
static int kva_check(const qbk_kv_shape *s, size_t n_heads, size_t n, size_t sq, size_t max_len, size_t prefix_len) {
    int rc;
    size_t bytes;
    if ((rc = kv_check_shape(s, &bytes))) return rc;
    if (n_heads == 0 || n_heads % s->n_kv_heads != 0)
        return fail(QBK_ERR_VALIDATION, fmt("n_kv_heads must divide n_heads: n_heads=%zu, n_kv_heads=%zu", n_heads,
                                            s->n_kv_heads));
    if (n_heads > (1u << 20)) return fail(QBK_ERR_VALIDATION, "kv attention takes up to 2^20 heads");
    if (sq == 0) return fail(QBK_ERR_VALIDATION, "kv attention requires at least one query a sequence");
    if (max_len > s->capacity)
        return fail(QBK_ERR_VALIDATION, fmt("max_len %zu is past the kv cache's capacity of %zu", max_len, s->capacity));
    if (n > 0x7FFFFFFFull || sq > 0x3FFFFFFFull || n_heads > 0x7FFFFFFFull || prefix_len > 0x7FFFFF00ull ||
        (n && (unsigned __int128)n * sq * (n_heads / s->n_kv_heads) > 0x7FFFFFFFull))
        return fail(QBK_ERR_VALIDATION, "kv attention: too many query rows for one launch");
    const KvaPlan p = n ? kva_plan(s, n_heads, n, sq, max_len, prefix_len) : KvaPlan{};
    if (p.items > 0x7FFFFFFFull || (unsigned __int128)n * sq * n_heads > 0x1FFFFFFFCull)
        return fail(QBK_ERR_VALIDATION, "kv attention: too many query rows for one launch");
    return QBK_OK;
}

}  // namespace qbk

using namespace qbk;

extern "C" {

size_t qbk_attention_kv_workspace_size(const qbk_kv_shape *shape, size_t n_heads, size_t n, size_t seq_q,
                                       size_t max_len, size_t prefix_len) {
    if (kva_check(shape, n_heads, n, seq_q, max_len, prefix_len) || n == 0) return 0;
    return kva_plan(shape, n_heads, n, seq_q, max_len, prefix_len).bytes;
}

int qbk_attention_kv_dev(qbk_ctx *ctx, const qbk_kv_shape *shape, const void *cache, size_t first_seq, size_t n,
                         const uint32_t *lens, size_t max_len, const qbk_kv_shape *prefix_shape,
                         const void *prefix, size_t prefix_seq, size_t prefix_len, size_t n_heads, size_t seq_q,
                         const void *q, int dtype, void *out, void *workspace, size_t workspace_size, void *stream) {
    int rc;
    if ((rc = kva_check(shape, n_heads, n, seq_q, max_len, prefix_len))) return rc;
    if (dtype != QBK_F32 && dtype != QBK_BF16)
        return fail(QBK_ERR_VALIDATION, fmt("kv attention takes float32 or bfloat16 queries (dtype %d)", dtype));
    if (first_seq > shape->n_seqs || n > shape->n_seqs - first_seq)
        return fail(QBK_ERR_VALIDATION, fmt("sequences %zu .. %zu of a kv cache holding %zu", first_seq,
                                            first_seq + n, shape->n_seqs));
    if (prefix_len) {
        size_t bytes;
        if ((rc = kv_check_shape(prefix_shape, &bytes))) return rc;
        if (prefix_shape->format != shape->format || prefix_shape->n_kv_heads != shape->n_kv_heads ||
            prefix_shape->head_dim != shape->head_dim)
            return fail(QBK_ERR_VALIDATION, "the prefix's cache must have the format, kv heads and head_dim of the "
                                            "sequences' cache");
        if (prefix_seq >= prefix_shape->n_seqs || prefix_len > prefix_shape->capacity)
            return fail(QBK_ERR_VALIDATION,
                        fmt("a prefix of %zu rows of sequence %zu in a kv cache of %zu sequences of %zu", prefix_len,
                            prefix_seq, prefix_shape->n_seqs, prefix_shape->capacity));
    }
    if (n == 0) return QBK_OK;
    if (!cache || !lens || !q || !out || (prefix_len && !prefix)) return fail(QBK_ERR_VALIDATION, "null argument");
    if (((uintptr_t)cache | (uintptr_t)(prefix_len ? prefix : nullptr)) & 15)
        return fail(QBK_ERR_VALIDATION, "kv cache buffer must be 16-byte aligned");
    const KvaPlan p = kva_plan(shape, n_heads, n, seq_q, max_len, prefix_len);
    if (p.bytes) {
        if (!workspace || workspace_size < p.bytes)
            return fail(QBK_ERR_VALIDATION, fmt("kv attention workspace of %zu bytes is smaller than the %zu needed",
                                                workspace ? workspace_size : (size_t)0, p.bytes));
        if ((uintptr_t)workspace & 15) return fail(QBK_ERR_VALIDATION, "kv attention workspace must be 16-byte aligned");
    }
    if ((rc = bind(ctx))) return rc;
    KvAttArgs a{};
    a.own = kv_view(shape, cache);
    a.pre = prefix_len ? kv_view(prefix_shape, prefix) : a.own;
    a.q = q;
    a.out = out;
    a.lens = lens;
    a.first_seq = (uint32_t)first_seq;
    a.prefix_seq = (uint32_t)prefix_seq;
    a.prefix_len = (uint32_t)prefix_len;
    a.max_len = (uint32_t)max_len;
    a.n = (uint32_t)n;
    a.sq = (uint32_t)seq_q;
    a.H = (uint32_t)n_heads;
    a.G = (uint32_t)(n_heads / shape->n_kv_heads);
    a.rows = a.n * a.sq * a.G;
    a.sp = p.sp;
    a.ss = p.ss;
    a.rtp = p.rtp;
    a.rts = p.rts;
    a.n_pre = (uint32_t)(shape->n_kv_heads * p.rtp * p.sp);
    a.scale = (float)(1.4426950408889634 / sqrt((double)shape->head_dim));
    const size_t parts = (size_t)(p.sp + p.ss) * shape->n_kv_heads * a.rows;
    a.po = (float *)workspace;
    a.ml = (float2 *)(a.po + parts * shape->head_dim);
    hipStream_t st = (hipStream_t)stream;
    if (p.items) {
        if (shape->format == QBK_KV_INT8)
            rc = dtype == QBK_F32 ? kva_dispatch<QBK_KV_INT8, float>(a, p, ctx->device, st)
                                  : kva_dispatch<QBK_KV_INT8, uint16_t>(a, p, ctx->device, st);
        else
            rc = dtype == QBK_F32 ? kva_dispatch<QBK_KV_FP8, float>(a, p, ctx->device, st)
                                  : kva_dispatch<QBK_KV_FP8, uint16_t>(a, p, ctx->device, st);
        if (rc) return rc;
    }
    if (p.sp + p.ss == 1) return QBK_OK;  // the items wrote the output
    const dim3 grid((unsigned)div_ceil((size_t)a.rows * shape->n_kv_heads, 4));
    if (dtype == QBK_F32)
        hipLaunchKernelGGL((kva_join<float>), grid, dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL((kva_join<uint16_t>), grid, dim3(256), 0, st, a);
    QBK_HIP(hipGetLastError());
    return QBK_OK;
}

}  // extern "C"
