// attention_kv.hip -- attention of a batch over the 8-bit or 4-bit KV cache,
// behind a prefix that every sequence shares.
//
// Rows: query row rho = (b sq + t) G + hg of kv head hk is sequence b's query
// t, head hk G + hg.  Every row sees the prefix, so the prefix's items take
// rows of all sequences together and read its codes for 16 or 64 of them; a
// sequence's own rows are seen by its sq G rows alone.  Both kinds are items of
// one launch:
//   item = (kv head, 16 or 64 rows, run of 64-row key tiles)
// and leave a partial result (sum of weights, mean of values, reference) per
// row; a second launch joins them.  A key tile and 16 rows, a wave:
//   S^T = K q^T      v_mfma_f32_16x16x32_f16, codes (fp4: times their multipliers) widened to fp16 (exact)
//   p = exp2(s - M)  online, per query column; M is a whole number, so moving
//                    to another M and joining partials scale by powers of two
//   O^T += V^T p^T   p times the value row's scale, in fp16
// The score layout of the first product is the operand layout of the second
// (kvcache.h), so a tile passes through registers alone.
//
// Roundings: q is scaled by a power of two and held as fp16 (bf16 queries:
// exact for channels from 2^-20 of the row's largest on, below that off by at
// most 2^-28 of it) or as two fp16 halves (f32 queries: 22 bits); p times scale
// likewise, 2^12 above a reference of its own, the row's largest of them, so
// that a weight keeps its bits down to 2^-26 of that: 11 bits where outputs are
// bf16 and hold 8 (one half more would double the second product).  Sums are
// f32.
#include <math.h>

#include <atomic>

#include "kvcache.h"

#pragma clang fp contract(off)

namespace qbk {

typedef _Float16 kva_h8_t __attribute__((ext_vector_type(8)));
typedef _Float16 kva_h2_t __attribute__((ext_vector_type(2)));
typedef float kva_f2_t __attribute__((ext_vector_type(2)));
typedef float kva_f4_t __attribute__((ext_vector_type(4)));
typedef uint32_t kva_u2_t __attribute__((ext_vector_type(2)));
typedef uint32_t kva_u4_t __attribute__((ext_vector_type(4)));

#define KVA_WAVES 4
#define KVA_MAX_SPLITS 32  // of the prefix, and of a sequence's own rows

// x / d and x % d for x below 2^31 by a multiplication (a division costs some
// 25 dependent instructions, and an item begins with five).
struct KvaDiv {
    uint32_t d, mul, shift;
    void set(uint32_t by) {
        d = by;
        shift = 0;
        while ((1ull << shift) < by) shift++;
        mul = (uint32_t)((((1ull << shift) - by) << 32) / by + 1);
    }
    __device__ __forceinline__ uint32_t split(uint32_t x, uint32_t &rest) const {
        const uint32_t q = (__umulhi(x, mul) + x) >> shift;
        rest = x - q * d;
        return q;
    }
};

struct KvAttArgs {
    KvView own, pre;
    const void *q;
    void *out;
    const uint32_t *lens;
    float *po;    // [split][hk][rho][hd] weighted means of the values
    float2 *ml;   // [split][hk][rho] reference, sum of weights
    uint32_t first_seq, prefix_seq, prefix_len, max_len;
    uint32_t plus;                   // lens are positions, so many rows behind them just written
    uint32_t n, sq, H, G, rows;      // rows = n sq G
    uint32_t sp, ss, rtp, rts;       // splits and row tiles of prefix and own items
    uint32_t n_pre;                  // prefix items
    KvaDiv by_hk, by_rtp, by_rts, by_n, by_g, by_sp, by_ss, by_sq, by_rows;
    float scale;                     // log2(e) / sqrt(hd)
};

// Own rows of sequence b that count (end: as many as there would be, had its
// last ones room), and the key tiles a split of them takes: at least one a wave,
// so that short sequences use few splits.
__device__ __forceinline__ uint32_t kva_end(const KvAttArgs &a, uint32_t b) {
    const uint32_t l = a.lens[b];
    return (l < a.max_len ? l : a.max_len) + a.plus;
}
__device__ __forceinline__ uint32_t kva_len(const KvAttArgs &a, uint32_t end) { return end < a.max_len ? end : a.max_len; }
__device__ __forceinline__ uint32_t kva_run(const KvAttArgs &a, uint32_t len) {
    uint32_t rest;
    const uint32_t c = a.by_ss.split((len + 63) / 64 + a.ss - 1, rest);
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

// The same of the 4-bit format: eight codes in one dword.
__device__ __forceinline__ void kva_wide4(uint32_t w, kva_h2_t (&p)[4]) {
    p[0] = __builtin_bit_cast(kva_h2_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.0f, 0));
    p[1] = __builtin_bit_cast(kva_h2_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.0f, 1));
    p[2] = __builtin_bit_cast(kva_h2_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.0f, 2));
    p[3] = __builtin_bit_cast(kva_h2_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.0f, 3));
}
__device__ __forceinline__ kva_h8_t kva_h8(const kva_h2_t (&p)[4]) {
    return kva_h8_t{p[0][0], p[0][1], p[1][0], p[1][1], p[2][0], p[2][1], p[3][0], p[3][1]};
}
// Two multipliers of a dword's four.
template <int HALF>
__device__ __forceinline__ kva_h2_t kva_mul4(uint32_t w) {
    return __builtin_bit_cast(kva_h2_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 1.0f, HALF));
}
// A key's eight channels of one group times the group's multiplier; a value's
// eight rows (row pairs of dwords m0 and m1) times theirs.
__device__ __forceinline__ kva_h8_t kva_key4(uint32_t w, _Float16 mul) {
    kva_h2_t p[4];
    kva_wide4(w, p);
#pragma unroll
    for (int e = 0; e < 4; e++) p[e] *= kva_h2_t{mul, mul};
    return kva_h8(p);
}
__device__ __forceinline__ kva_h8_t kva_val4(uint32_t w, uint32_t m0, uint32_t m1) {
    kva_h2_t p[4];
    kva_wide4(w, p);
    p[0] *= kva_mul4<0>(m0);
    p[1] *= kva_mul4<1>(m0);
    p[2] *= kva_mul4<0>(m1);
    p[3] *= kva_mul4<1>(m1);
    return kva_h8(p);
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

// A value that every lane holds, as a scalar.
__device__ __forceinline__ uint32_t kva_scalar(uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); }
__device__ __forceinline__ float kva_scalar(float v) { return __uint_as_float(kva_scalar(__float_as_uint(v))); }

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

// LDS of a body of up to 16 rows: queries as operands, then (over them) the
// waves' outputs; the rows' factors, references and sums.
template <int DC, bool HI>
struct KvaLds {
    static constexpr int Q = 2 * DC * 1024 * (HI ? 2 : 1);
    static constexpr int OC = DC < 2 ? 64 : 128;  // channels joined at a time
    static constexpr int O = KVA_WAVES * 16 * (OC + 4) * 4;
    static constexpr int BODY = Q > O ? Q : O;
    static constexpr int BYTES = BODY + 16 * 4 * (1 + 2 * KVA_WAVES);
};

// Rows of a body from row0 on: row r is query (b, t) = base + r's quotient by
// G, head the remainder.  The float quotient is exact: x + 1/2 is half a unit
// from every multiple of G and below 2^14 (G at most 2^13, checked on the
// host), rounding and reciprocal are within 2^-22 together.
struct KvaRow {
    uint32_t base, rem, G;
    float inv;
    __device__ __forceinline__ KvaRow(const KvAttArgs &a, uint32_t row0)
        : G(a.G), inv(__builtin_amdgcn_rcpf((float)a.G)) {
        base = a.by_g.split(row0, rem);
    }
    __device__ __forceinline__ void at(uint32_t r, uint32_t &query, uint32_t &head) const {
        const uint32_t x = rem + r, d = (uint32_t)(((float)x + 0.5f) * inv);
        query = base + d;
        head = x - d * G;
    }
};

// The largest over aligned runs of LANES (16, 32 or 64) lanes.
template <int LANES>
__device__ __forceinline__ uint32_t kva_row_max(uint32_t v) {
    auto up = [](uint32_t x, uint32_t y) { return x > y ? x : y; };
    v = up(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xf, 0xf, true));  // row_ror 8, 4, 2, 1
    v = up(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x124, 0xf, 0xf, true));
    v = up(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x122, 0xf, 0xf, true));
    v = up(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x121, 0xf, 0xf, true));
    if constexpr (LANES >= 32) {
        const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        v = up(a[0], a[1]);
    }
    if constexpr (LANES >= 64) {
        const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        v = up(b[0], b[1]);
    }
    return v;
}

// Four values of a row at any alignment (one load on this machine).
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Kva4 {
    T v[4];
};

// Queries row0 .. row0 + n_rows - 1 (at most 16 NT) of kv head hk into LDS as
// the B operands of K q^T, [tile][step][lane][16 bytes], for f32 queries the
// low halves behind them; qfs[r]: the factor that scores of row r still need,
// NaN for a row that holds a NaN or an infinity.
// 16 DC lanes a row, four channels a lane, every row's load before the first
// is used (32 requests behind 8192 rows, by a row at a time 41 us, so 29).
template <int DC, int NT, typename T>
__device__ __forceinline__ void kva_queries(const KvAttArgs &a, char *qs, float *qfs, uint32_t row0, uint32_t n_rows,
                                            uint32_t hk) {
    constexpr int STEPS = 2 * DC, LANES = 16 * DC, AT_ONCE = KVA_WAVES * 64 / LANES, N = 16 * NT / AT_ONCE;
    const int tid = threadIdx.x, hd = (int)a.own.hd, c = 4 * (tid % LANES), r0 = tid / LANES;
    const KvaRow rows(a, row0);
    // from the first row's query on; rows of a body span less than 2^32 bytes (kva_check)
    const T *q0 = (const T *)a.q + ((size_t)rows.base * a.H + (size_t)hk * a.G) * hd;
    Kva4<T> raw[N];
#pragma unroll
    for (int k = 0; k < N; k++) {
        const uint32_t r = r0 + k * AT_ONCE;
        uint32_t query, head;
        rows.at(r < n_rows ? r : 0, query, head);
        raw[k] = *(const Kva4<T> *)(q0 + (((query - rows.base) * a.H + head) * hd + (c < hd ? c : 0)));
    }
    uint32_t top[N];
#pragma unroll
    for (int k = 0; k < N; k++) {
        const bool in = r0 + k * AT_ONCE < (int)n_rows && c < hd;
        top[k] = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            raw[k].v[e] = in ? raw[k].v[e] : (T)0;
            const uint32_t b = __float_as_uint(kva_in<T>(raw[k].v[e])) & 0x7fffffffu;
            top[k] = b > top[k] ? b : top[k];
        }
    }
#pragma unroll
    for (int k = 0; k < N; k++) top[k] = kva_row_max<LANES>(top[k]);
#pragma unroll
    for (int k = 0; k < N; k++) {
        const int r = r0 + k * AT_ONCE;
        // the largest channel to [8, 16): both halves of every channel within fp16
        const bool whole = top[k] < 0x7f800000u;
        uint32_t ex = top[k] >> 23;
        ex = ex < 8 ? 8 : ex;  // rows below 2^-119 stay below 8: the factor is a normal number down to here
        const float f = __uint_as_float((257 - ex) << 23);  // NaN rows: the scores become NaN by qfs
        kva_h2_t hi[2], lo[2];
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
            const kva_f2_t y = {kva_in<T>(raw[k].v[e]) * f, kva_in<T>(raw[k].v[e + 1]) * f};
            hi[e >> 1] = __builtin_convertvector(y, kva_h2_t);
            if constexpr (sizeof(T) == 4)
                lo[e >> 1] = __builtin_convertvector(y - __builtin_convertvector(hi[e >> 1], kva_f2_t), kva_h2_t);
        }
        // channel c: chunk c / 16 -> step 2 (chunk / 4) + (c % 16) / 8, operand lane (chunk % 4, column r % 16)
        const int chunk = c >> 4, step = 2 * (chunk >> 2) + ((c >> 3) & 1);
        const int at = (((r >> 4) * STEPS + step) * 64 + (chunk & 3) * 16 + (r & 15)) * 16 + (c & 7) * 2;
        *(uint2 *)(qs + at) = uint2{__builtin_bit_cast(uint32_t, hi[0]), __builtin_bit_cast(uint32_t, hi[1])};
        if constexpr (sizeof(T) == 4)
            *(uint2 *)(qs + NT * STEPS * 1024 + at) =
                uint2{__builtin_bit_cast(uint32_t, lo[0]), __builtin_bit_cast(uint32_t, lo[1])};
        top[k] = whole ? __float_as_uint(a.scale * __uint_as_float((ex - 3) << 23)) : 0x7fc00000u;
    }
    if (c == 0)
#pragma unroll
        for (int k = 0; k < N; k++) qfs[r0 + k * AT_ONCE] = __uint_as_float(top[k]);
}

// Sums of code products to scores in base 2: times the key's scale and the
// row's factor, those two first.  Codes reach 448 (fp4: 2688) and a scaled query 16, so a
// sum by its key's scale alone would pass f32 for keys from some 2^117 on; the
// two together pass it where |q| |k| does.  From here on a score is this
// rounded number: a reference taken from it is as large as the largest, while
// of a fused product's remainders past 2^31 some are above 2^128 by themselves.
__device__ __forceinline__ void kva_scores(kva_f4_t (&s)[4], const kva_f4_t (&ks)[4], float qf) {
#pragma unroll
    for (int i = 0; i < 4; i++) s[i] *= ks[i] * qf;
}

// Scores t and value scales vs of a lane's 16 keys (16 i + j past key) that its
// row does not see: no score and no scale, whatever the cache holds there.
__device__ __forceinline__ void kva_mask(kva_f4_t (&t)[4], kva_f4_t (&vs)[4], uint32_t key, uint32_t lim) {
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const bool out = key + 16 * i + j >= lim;
            t[i][j] = out ? -INFINITY : t[i][j];
            vs[i][j] = out ? 0.0f : vs[i][j];
        }
}

// The largest of a lane's 16.
__device__ __forceinline__ float kva_most(const kva_f4_t (&t)[4]) {
    float m[4];
#pragma unroll
    for (int i = 0; i < 4; i++) m[i] = fmaxf(fmaxf(t[i][0], t[i][1]), fmaxf(t[i][2], t[i][3]));
    return fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
}

// The row's reference moves when a score passes it eightfold, its sum with it;
// what the outputs stand for stays, so wref moves the other way.
__device__ __forceinline__ void kva_reference(const kva_f4_t (&t)[4], float &ref, float &sum, float &wref) {
    const float tm = kva_most(t);
    if (__ballot(tm > ref + 3.0f)) {
        const float most = kva_max4(tm);
        const float to = most > ref + 3.0f ? ceilf(most) : ref;  // other rows' scores move no more than theirs
        const float f = kva_rescale(ref, to);
        sum *= f;
        wref *= f;
        ref = to;
    }
}

// Scores to weights: p = exp2(t - ref) into sum, t becomes p times the value's
// scale.
__device__ __forceinline__ void kva_weights(kva_f4_t (&t)[4], const kva_f4_t (&vs)[4], float ref, float &sum) {
    const float base = ref == -INFINITY ? 0.0f : ref;  // a row that has seen nothing: every p is 0
    float l[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float p = __builtin_amdgcn_exp2f(t[i][j] - base);
            l[i] += p;
            t[i][j] = p * vs[i][j];
        }
    sum += (l[0] + l[1]) + (l[2] + l[3]);
}

// Weights w = p times value scale against wref, a power of two above every one
// that the row has seen (or an eighth of it): the outputs follow when it moves.
// It is the row's own and of rows that it sees alone, and p is in it, so that
// neither a value that the mask hides nor a large one of little weight costs
// the others their bits.  A row's likeliest key has p of 1/2 and more and a
// scale of 2^-112 and more, so wref is 2^-114 and more as soon as a weight is
// not 0, and at most 2^126.
template <int CT>
__device__ __forceinline__ void kva_weight_reference(const kva_f4_t (&w)[4], float &wref, kva_f4_t (&o)[CT]) {
    const float wm = kva_most(w);
    if (__ballot(wm > 8.0f * wref)) {
        const float most = kva_max4(wm);
        if (most > 8.0f * wref) {
            uint32_t e = (__float_as_uint(most) >> 23) + 1;
            e = e < 12 ? 12 : e > 253 ? 253 : e;  // what a row that is no number has seen
            const float f = wref * __uint_as_float((254 - e) << 23);
#pragma unroll
            for (int ct = 0; ct < CT; ct++) o[ct] *= f;
            wref = __uint_as_float(e << 23);
        }
    }
}

// Weights in units of 2^-12 wref as operands ph (and pl, what the first half
// leaves).
template <bool HI>
__device__ __forceinline__ void kva_operands(const kva_f4_t (&w)[4], float wref, kva_h8_t (&ph)[2],
                                             kva_h8_t (&pl)[2]) {
    const float inv = __uint_as_float((266u << 23) - __float_as_uint(wref));  // 2^12 / wref; of 0 a number, weights are 0
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j += 2) {
            const kva_f2_t x = {w[i][j] * inv, w[i][j + 1] * inv};
            const kva_h2_t h = __builtin_convertvector(x, kva_h2_t);
            ph[i >> 1][4 * (i & 1) + j] = h[0];
            ph[i >> 1][4 * (i & 1) + j + 1] = h[1];
            if constexpr (HI) {
                const kva_h2_t r = __builtin_convertvector(x - __builtin_convertvector(h, kva_f2_t), kva_h2_t);
                pl[i >> 1][4 * (i & 1) + j] = r[0];
                pl[i >> 1][4 * (i & 1) + j + 1] = r[1];
            }
        }
}

// A wave's running state for its 16 rows: reference, sum of weights and
// weighted values (O^T, channel 16 ct + 4 g + j of row col) over wref's 2^12.
template <int DC>
struct KvaState {
    kva_f4_t o[4 * DC];
    float ref, sum, qf, wref;
    uint32_t lim;
    __device__ __forceinline__ KvaState(float qf, uint32_t lim)
        : ref(-INFINITY), sum(0.0f), qf(qf), wref(0.0f), lim(lim) {
#pragma unroll
        for (int ct = 0; ct < 4 * DC; ct++) o[ct] = kva_f4_t{0, 0, 0, 0};
    }
};

// Codes of rows at or past `written` as zero: 32 bits a 16-row block for the
// lane's four rows 4 g .. of it.
__device__ __forceinline__ kva_u4_t kva_keep(uint32_t key0, uint32_t written, int g) {
    kva_u4_t keep;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t k0 = key0 + 16 * i + 4 * g, left = written > k0 ? written - k0 : 0;
        keep[i] = left >= 4 ? ~0u : (1u << (8 * left)) - 1u;
    }
    return keep;
}

// What outputs times wref are a mean of values by (a last place of f32 off):
// sums of values may pass f32 where their mean does not, so none is formed.
__device__ __forceinline__ float kva_per(float sum) {
    return sum == 0.0f ? 0.0f : 0x1p-12f * __builtin_amdgcn_rcpf(sum);
}

// Where row rho's output goes.
template <typename T>
__device__ __forceinline__ T *kva_out_row(const KvAttArgs &a, uint32_t rho, uint32_t hk) {
    uint32_t head;
    const uint32_t query = a.by_g.split(rho, head);
    return (T *)a.out + ((size_t)query * a.H + (size_t)hk * a.G + head) * a.own.hd;
}

// A slab's codes, multipliers (fp4) and scales.
struct KvaSlab {
    const uint8_t *k, *v, *km, *vm;
    const float *ks, *vs;
    uint32_t ng;
    template <int FMT>
    static __device__ __forceinline__ KvaSlab of(const KvView &c, size_t slab) {
        KvaSlab s;
        s.ng = c.groups();
        if constexpr (FMT == QBK_KV_FP4) {
            s.k = c.k + slab * (c.hd / 2);
            s.v = c.v + slab * (16 * s.ng);
            s.km = c.km + slab * s.ng;
            s.vm = c.vm + slab * s.ng;
        } else {
            s.k = c.k + slab * c.hd;
            s.v = c.v + slab * c.hd;
            s.km = s.vm = nullptr;
        }
        s.ks = c.ks + slab;
        s.vs = c.vs + slab;
        return s;
    }
};

// A lane's scales of tile tt: of rows 16 i + 4 g .. 16 i + 4 g + 3.
__device__ __forceinline__ void kva_scales(const float *of, uint32_t tt, int g, kva_f4_t (&s)[4]) {
    const float *st = of + (size_t)tt * 64 + 4 * g;
#pragma unroll
    for (int i = 0; i < 4; i++) s[i] = *(const kva_f4_t *)(st + 16 * i);
}

// A key tile's codes on their way to a wave, and its operands.
template <int FMT, int DC>
struct KvaTile {
    kva_u4_t kc[DC][4], vc[4 * DC];
    __device__ __forceinline__ void load_k(const KvaSlab &c, uint32_t tt, int hd, int col, int g, kva_f4_t (&ks)[4]) {
        const int nc = hd / 16;
        const uint8_t *kt = c.k + (size_t)tt * 64 * hd + col * 16;
        kva_scales(c.ks, tt, g, ks);
#pragma unroll
        for (int x = 0; x < DC; x++) {
            const int chunk = 4 * x + g < nc ? 4 * x + g : nc - 1;  // past the last chunk q is zero
#pragma unroll
            for (int i = 0; i < 4; i++) kc[x][i] = *(const kva_u4_t *)(kt + (i * nc + chunk) * 256);
        }
    }
    __device__ __forceinline__ void load_v(const KvaSlab &c, uint32_t tt, int hd, int col, int g, kva_f4_t (&vs)[4]) {
        const int nc = hd / 16;
        const uint8_t *vt = c.v + (size_t)tt * 64 * hd + col * 64 + g * 16;
        kva_scales(c.vs, tt, g, vs);
#pragma unroll
        for (int ct = 0; ct < 4 * DC; ct++)
            vc[ct] = *(const kva_u4_t *)(vt + (ct < nc ? ct : nc - 1) * 1024);  // past the last tile: not stored
    }
    __device__ __forceinline__ kva_h8_t key(int x, int i) const {
        return kva_wide<FMT>(kc[x / 2][i][2 * (x & 1)], kc[x / 2][i][2 * (x & 1) + 1]);
    }
    // keep: rows that were written; fp8 rows that were not may hold NaN codes
    __device__ __forceinline__ kva_h8_t val(int ct, int u, const kva_u4_t &keep) const {
        const kva_u4_t w = FMT == QBK_KV_FP8 ? vc[ct] & keep : vc[ct];
        return kva_wide<FMT>(w[2 * u], w[2 * u + 1]);
    }
};
template <int DC>
struct KvaTile<QBK_KV_FP4, DC> {
    kva_u4_t kc[DC][2], vc[2 * DC], vm[2 * DC];
    uint32_t km[DC];
    __device__ __forceinline__ void load_k(const KvaSlab &c, uint32_t tt, int hd, int col, int g, kva_f4_t (&ks)[4]) {
        const int nc = hd / 16, ng = (int)c.ng;
        const uint8_t *kt = c.k + (size_t)tt * 32 * hd + col * 16;
        const uint8_t *mt = c.km + (size_t)tt * 64 * ng + col * 4;
        kva_scales(c.ks, tt, g, ks);
#pragma unroll
        for (int x = 0; x < DC; x++) {
            const int chunk = 4 * x + g < nc ? 4 * x + g : nc - 1;  // past the last chunk q is zero
            km[x] = *(const uint32_t *)(mt + (chunk >> 1) * 64);
#pragma unroll
            for (int p = 0; p < 2; p++) kc[x][p] = *(const kva_u4_t *)(kt + (p * nc + chunk) * 256);
        }
    }
    __device__ __forceinline__ void load_v(const KvaSlab &c, uint32_t tt, int hd, int col, int g, kva_f4_t (&vs)[4]) {
        const int ng = (int)c.ng;
        const uint8_t *vt = c.v + (size_t)tt * 1024 * ng + col * 64 + g * 16;
        const uint8_t *mt = c.vm + (size_t)tt * 64 * ng + g * 16;
        kva_scales(c.vs, tt, g, vs);
#pragma unroll
        for (int m = 0; m < 2 * DC; m++) {
            const int at = m < ng ? m : ng - 1;  // past the last tile: not stored
            vm[m] = *(const kva_u4_t *)(mt + at * 64);
            vc[m] = *(const kva_u4_t *)(vt + at * 1024);
        }
    }
    __device__ __forceinline__ kva_h8_t key(int x, int i) const {
        const kva_h2_t m = i < 2 ? kva_mul4<0>(km[x / 2]) : kva_mul4<1>(km[x / 2]);
        return kva_key4(kc[x / 2][i >> 1][2 * (i & 1) + (x & 1)], m[i & 1]);
    }
    // keep: rows that were written; those that were not may hold NaN multipliers
    __device__ __forceinline__ kva_h8_t val(int ct, int u, const kva_u4_t &keep) const {
        const kva_u4_t m = vm[ct >> 1] & keep;
        return kva_val4(vc[ct >> 1][2 * (ct & 1) + u], m[2 * u], m[2 * u + 1]);
    }
};

// Up to 16 rows, row0 .. row0 + n_rows - 1 of kv head hk, over key tiles tile0
// .. tile1 - 1 of the slab k, v, ks, vs: a wave every fourth tile, in registers
// alone (few rows are bound by the cache's bytes; 32 sequences of up to 2085
// rows, 32/8 heads of 128: 107 MB in 23.0 us, 4.7 TB/s).  Row r of the body sees
// keys below limit(r), none of them at or past `written`.
template <int FMT, int DC, typename T, class Limit>
__device__ __forceinline__ void kva_body(const KvAttArgs &a, char *smem, uint32_t row0, uint32_t n_rows, uint32_t hk,
                                         const KvaSlab &slab, uint32_t tile0, uint32_t tile1, uint32_t written,
                                         Limit limit, uint32_t split, bool last) {
    constexpr bool HI = sizeof(T) == 4;
    using L = KvaLds<DC, HI>;
    constexpr int STEPS = 2 * DC;
    const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);  // scalar: loops and addresses by it are too
    const int hd = (int)a.own.hd, nc = hd / 16;
    char *qs = smem;
    float *qfs = (float *)(smem + L::BODY), *refs = qfs + 16, *sums = refs + KVA_WAVES * 16;

    // A tile's codes and scales travel while the one before is worked on: keys
    // and their scales are asked for again as soon as the scores are formed,
    // values once they are added, the first of both before the queries are read.
    // The codes' address is formed before the scales are asked for, which come
    // first all the same: formed behind them it takes four registers more, and
    // heads of 64 lose one of three waves a SIMD (512 sequences of 500 rows, fp8,
    // f32 queries 41 / 52 us); codes asked for first cost 2 to 3 % of most calls.
    KvaTile<FMT, DC> tile;
    kva_f4_t ks[4], vs[4];
    auto load_k = [&](uint32_t tt) { tile.load_k(slab, tt, hd, col, g, ks); };
    auto load_v = [&](uint32_t tt) { tile.load_v(slab, tt, hd, col, g, vs); };
    const uint32_t first = tile0 + wave;
    if (first < tile1) {
        load_k(first);
        load_v(first);
    }
    kva_queries<DC, 1, T>(a, qs, qfs, row0, n_rows, hk);
    __syncthreads();
    KvaState<DC> st(qfs[col], limit((uint32_t)col < n_rows ? col : n_rows - 1));
    const uint32_t least = kva_scalar(limit(0));  // keys below it are seen by every row

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
        asm volatile("" ::: "memory");  // the queries are read from LDS again, not kept in registers that spill
        kva_f4_t s[4];
#pragma unroll
        for (int i = 0; i < 4; i++) s[i] = kva_f4_t{0, 0, 0, 0};
#pragma unroll
        for (int x = 0; x < STEPS; x++) {
            const kva_h8_t qf = *(const kva_h8_t *)(qs + (x * 64 + lane) * 16);
            kva_h8_t kf[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                kf[i] = tile.key(x, i);
                s[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[i], qf, s[i], 0, 0, 0);
            }
            if constexpr (HI) {
                const kva_h8_t ql = *(const kva_h8_t *)(qs + STEPS * 1024 + (x * 64 + lane) * 16);
#pragma unroll
                for (int i = 0; i < 4; i++) s[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[i], ql, s[i], 0, 0, 0);
            }
        }
        // the key registers are free again
        kva_scores(s, ks, st.qf);
        if (more) load_k(tt + KVA_WAVES);
        if (masked) kva_mask(s, vs, key0 + 4 * g, st.lim);
        kva_reference(s, st.ref, st.sum, st.wref);
        kva_weights(s, vs, st.ref, st.sum);
        kva_weight_reference(s, st.wref, st.o);
        kva_h8_t ph[2], pl[2];
        kva_operands<HI>(s, st.wref, ph, pl);
        kva_u4_t keep = {~0u, ~0u, ~0u, ~0u};
        if (FMT != QBK_KV_INT8 && masked) keep = kva_keep(key0, written, g);
#pragma unroll
        for (int ct = 0; ct < 4 * DC; ct++) {
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const kva_h8_t vf = tile.val(ct, u, keep);
                st.o[ct] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, ph[u], st.o[ct], 0, 0, 0);
                if constexpr (HI) st.o[ct] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pl[u], st.o[ct], 0, 0, 0);
            }
        }
        if (more) load_v(tt + KVA_WAVES);
    }

    // join the waves on each row's largest reference
    const float l = kva_sum4(st.sum);
    if (g == 0) {
        refs[wave * 16 + col] = st.ref;
        sums[wave * 16 + col] = l;
    }
    __syncthreads();
    float2 row = {refs[col], 0.0f};  // row col's reference and sum of weights
#pragma unroll
    for (int w = 1; w < KVA_WAVES; w++) row.x = fmaxf(row.x, refs[w * 16 + col]);
#pragma unroll
    for (int w = 0; w < KVA_WAVES; w++) row.y += sums[w * 16 + col] * kva_rescale(refs[w * 16 + col], row.x);
    constexpr int OC = L::OC, LD = OC + 4;
    float *ob = (float *)smem;  // [wave][16 rows][LD]
    const size_t part = ((size_t)split * a.own.Hk + hk) * a.rows + row0;
    const float per = kva_per(row.y), f = kva_rescale(st.ref, row.x) * st.wref;
#pragma unroll
    for (int c0 = 0; c0 < 64 * DC; c0 += OC) {
        if (c0 >= hd) continue;
        if (c0) __syncthreads();  // what the region held has been read
#pragma unroll
        for (int k = 0; k < OC / 16; k++)
            *(kva_f4_t *)(ob + (wave * 16 + col) * LD + 16 * k + 4 * g) = st.o[c0 / 16 + k] * per * f;
        __syncthreads();
        for (int x = tid; x < 16 * OC; x += 64 * KVA_WAVES) {
            const int r = x / OC, c = x % OC;
            if (r >= (int)n_rows || c0 + c >= hd) continue;
            float v = 0.0f;
#pragma unroll
            for (int w = 0; w < KVA_WAVES; w++) v += ob[(w * 16 + r) * LD + c];
            if (last) kva_out_row<T>(a, row0 + r, hk)[c0 + c] = kva_out<T>(v);
            else a.po[(part + r) * hd + c0 + c] = v;
        }
    }
    if (!last && tid < (int)n_rows) a.ml[part + tid] = row;
}

// The 4-bit cache's body of up to four rows (a step's, of four query heads a kv
// head): a wave as kva_body's, but the 16 columns of the products are the rows
// four times over, and columns 4 t .. 4 t + 3 take the keys of block t alone,
// 16 t .. 16 t + 15 of a tile.  So a lane weighs four keys, not sixteen of which
// three quarters are of columns that nobody asks for, and since it does, values
// stay codes and their multipliers go to the weights: some 340 vector operations
// a tile, in kva_body 560.  A weight times a small multiplier m is a small fp16
// number: its second half (f32 queries) is a step of 2^-24 from x = 2^-3 on, so
// that the row's largest weight, 2^11 m / 2^9 and more, is off by 2^-27 / m of
// itself where that is more than 2^-22: channels of 2^-17 of their row's largest
// keep 18 bits, those from 2^-14 on 22, of values whose codes have two;
// multipliers with the codes, as in kva_body, are 4 % slower (f32 queries, 700
// rows 8.9 / 9.3 us, 32 sequences 21.2 / 22.0).  The columns of a row are joined as
// the waves are.
// 32 sequences of up to 2085 rows, 32/8 heads of 128: 59 MB in 18.0 us, by
// kva_body 20.9, by eight waves a workgroup 17.8 (64 sequences of 600 18.2, by
// four 11.6); 128 of up to 4000 446 MB in 85.5, 5.2 TB/s.
template <int DC>
struct KvaFew {
    kva_u4_t kc[DC][2], vc[2 * DC];
    uint32_t km[DC], vm[2 * DC];
    kva_f4_t ks, vs;
    __device__ __forceinline__ void load_k(const KvaSlab &c, uint32_t tt, int hd, int col, int g) {
        const int nc = hd / 16, ng = (int)c.ng;
        const uint8_t *kt = c.k + (size_t)tt * 32 * hd + col * 16;
        const uint8_t *mt = c.km + (size_t)tt * 64 * ng + col * 4;
        ks = *(const kva_f4_t *)(c.ks + (size_t)tt * 64 + 16 * (col >> 2) + 4 * g);
#pragma unroll
        for (int x = 0; x < DC; x++) {
            const int chunk = 4 * x + g < nc ? 4 * x + g : nc - 1;  // past the last chunk q is zero
            km[x] = *(const uint32_t *)(mt + (chunk >> 1) * 64);
#pragma unroll
            for (int p = 0; p < 2; p++) kc[x][p] = *(const kva_u4_t *)(kt + (p * nc + chunk) * 256);
        }
    }
    __device__ __forceinline__ void load_v(const KvaSlab &c, uint32_t tt, int hd, int col, int g) {
        const int ng = (int)c.ng;
        const uint8_t *vt = c.v + (size_t)tt * 1024 * ng + col * 64 + g * 16;
        const uint8_t *mt = c.vm + (size_t)tt * 64 * ng + g * 16 + (col >> 2) * 4;
        vs = *(const kva_f4_t *)(c.vs + (size_t)tt * 64 + 16 * (col >> 2) + 4 * g);
#pragma unroll
        for (int m = 0; m < 2 * DC; m++) {
            const int at = m < ng ? m : ng - 1;  // past the last tile: not stored
            vm[m] = *(const uint32_t *)(mt + at * 64);
            vc[m] = *(const kva_u4_t *)(vt + at * 1024);
        }
    }
};

template <int DC, typename T, class Limit>
__device__ __forceinline__ void kva_few(const KvAttArgs &a, char *smem, uint32_t row0, uint32_t n_rows, uint32_t hk,
                                        const KvaSlab &slab, uint32_t tile0, uint32_t tile1, uint32_t written,
                                        Limit limit, uint32_t split, bool last) {
    constexpr bool HI = sizeof(T) == 4;
    using L = KvaLds<DC, HI>;
    constexpr int STEPS = 2 * DC;
    const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, g = lane >> 4;
    const int row = col & 3, block = col >> 2;  // of this lane's column
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int hd = (int)a.own.hd, nc = hd / 16;
    char *qs = smem;
    float *qfs = (float *)(smem + L::BODY), *refs = qfs + 16, *sums = refs + KVA_WAVES * 16;
    KvaFew<DC> tile;
    const uint32_t first = tile0 + wave;
    if (first < tile1) {
        tile.load_k(slab, first, hd, col, g);
        tile.load_v(slab, first, hd, col, g);
    }
    kva_queries<DC, 1, T>(a, qs, qfs, row0, n_rows, hk);
    __syncthreads();
    KvaState<DC> st(qfs[row], limit((uint32_t)row < n_rows ? row : n_rows - 1));
    const uint32_t least = kva_scalar(limit(0));  // keys below it are seen by every row
    const int qlane = (g * 16 + row) * 16;
    const uint32_t mine[4] = {block == 0 ? ~0u : 0u, block == 1 ? ~0u : 0u, block == 2 ? ~0u : 0u, block == 3 ? ~0u : 0u};

    for (uint32_t tt = first; tt < tile1; tt += KVA_WAVES) {
        const uint32_t key0 = tt * 64, key = key0 + 16 * block + 4 * g;
        const bool masked = key0 + 64 > least, more = tt + KVA_WAVES < tile1;
        kva_f4_t s[4];
#pragma unroll
        for (int i = 0; i < 4; i++) s[i] = kva_f4_t{0, 0, 0, 0};
        asm volatile("" ::: "memory");  // the queries are read from LDS again, not kept in registers that spill
#pragma unroll
        for (int x = 0; x < STEPS; x++) {
            const kva_h8_t qf = *(const kva_h8_t *)(qs + x * 1024 + qlane);
            kva_h8_t kf[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const kva_h2_t m = i < 2 ? kva_mul4<0>(tile.km[x / 2]) : kva_mul4<1>(tile.km[x / 2]);
                kf[i] = kva_key4(tile.kc[x / 2][i >> 1][2 * (i & 1) + (x & 1)], m[i & 1]);
                s[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[i], qf, s[i], 0, 0, 0);
            }
            if constexpr (HI) {
                const kva_h8_t ql = *(const kva_h8_t *)(qs + (STEPS + x) * 1024 + qlane);
#pragma unroll
                for (int i = 0; i < 4; i++) s[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[i], ql, s[i], 0, 0, 0);
            }
        }
        kva_f4_t t = s[0], vs = tile.vs;
#pragma unroll
        for (int j = 0; j < 4; j++) {  // this column's block
            const float lo = block & 1 ? s[1][j] : s[0][j], hi = block & 1 ? s[3][j] : s[2][j];
            t[j] = block & 2 ? hi : lo;
        }
        t *= tile.ks * st.qf;
        if (more) tile.load_k(slab, tt + KVA_WAVES, hd, col, g);
        uint32_t keep = ~0u;
        if (masked) {  // what was never written, or lies past the row's keys, takes no part, whatever it holds
            const uint32_t left = written > key ? written - key : 0;
            keep = left >= 4 ? ~0u : (1u << (8 * left)) - 1u;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const bool out = key + j >= st.lim;
                t[j] = out ? -INFINITY : t[j];
                vs[j] = out || key + j >= written ? 0.0f : vs[j];
            }
        }
        const float tm = fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3]));
        if (__ballot(tm > st.ref + 3.0f)) {  // as kva_reference
            const float most = kva_max4(tm);
            const float to = most > st.ref + 3.0f ? ceilf(most) : st.ref;
            const float f = kva_rescale(st.ref, to);
            st.sum *= f;
            st.wref *= f;
            st.ref = to;
        }
        const float base = st.ref == -INFINITY ? 0.0f : st.ref;
        float l = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float p = __builtin_amdgcn_exp2f(t[j] - base);
            l += p;
            t[j] = p * vs[j];
        }
        st.sum += l;
        const float wm = fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3]));
        if (__ballot(wm > 8.0f * st.wref)) {  // as kva_weight_reference
            const float most = kva_max4(wm);
            if (most > 8.0f * st.wref) {
                uint32_t e = (__float_as_uint(most) >> 23) + 1;
                e = e < 12 ? 12 : e > 253 ? 253 : e;
                const float f = st.wref * __uint_as_float((254 - e) << 23);
#pragma unroll
                for (int ct = 0; ct < 4 * DC; ct++) st.o[ct] *= f;
                st.wref = __uint_as_float(e << 23);
            }
        }
        // weights in units of 2^-12 wref, times their group's multiplier over 2^9 (at most 7 / 8, so within fp16 still)
        t *= __uint_as_float((266u << 23) - __float_as_uint(st.wref));
#pragma unroll
        for (int m = 0; m < 2 * DC; m++) {
            const uint32_t mw = tile.vm[m] & keep;
            const kva_f2_t m0 = __builtin_bit_cast(kva_f2_t, __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(mw, 0x1p-9f, false));
            const kva_f2_t m1 = __builtin_bit_cast(kva_f2_t, __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(mw, 0x1p-9f, true));
            const kva_f2_t x0 = {t[0] * m0[0], t[1] * m0[1]}, x1 = {t[2] * m1[0], t[3] * m1[1]};
            const kva_h2_t h0 = __builtin_convertvector(x0, kva_h2_t), h1 = __builtin_convertvector(x1, kva_h2_t);
            const uint32_t w0 = __builtin_bit_cast(uint32_t, h0), w1 = __builtin_bit_cast(uint32_t, h1);
            uint32_t r0 = 0, r1 = 0;
            if constexpr (HI) {
                const kva_h2_t e0 = __builtin_convertvector(x0 - __builtin_convertvector(h0, kva_f2_t), kva_h2_t);
                const kva_h2_t e1 = __builtin_convertvector(x1 - __builtin_convertvector(h1, kva_f2_t), kva_h2_t);
                r0 = __builtin_bit_cast(uint32_t, e0);
                r1 = __builtin_bit_cast(uint32_t, e1);
            }
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const kva_h8_t ph = __builtin_bit_cast(kva_h8_t, kva_u4_t{w0 & mine[2 * u], w1 & mine[2 * u], w0 & mine[2 * u + 1], w1 & mine[2 * u + 1]});
                kva_h8_t pl;
                if constexpr (HI)
                    pl = __builtin_bit_cast(kva_h8_t, kva_u4_t{r0 & mine[2 * u], r1 & mine[2 * u], r0 & mine[2 * u + 1], r1 & mine[2 * u + 1]});
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    kva_h2_t v[4];
                    kva_wide4(tile.vc[m][2 * h + u], v);
                    const kva_h8_t vf = kva_h8(v);
                    st.o[2 * m + h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, ph, st.o[2 * m + h], 0, 0, 0);
                    if constexpr (HI) st.o[2 * m + h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pl, st.o[2 * m + h], 0, 0, 0);
                }
            }
        }
        if (more) tile.load_v(slab, tt + KVA_WAVES, hd, col, g);
    }

    // join the waves' and the blocks' columns on each row's largest reference
    const float l = kva_sum4(st.sum);
    if (g == 0) {
        refs[wave * 16 + col] = st.ref;
        sums[wave * 16 + col] = l;
    }
    __syncthreads();
    float2 all = {refs[row], 0.0f};  // row's reference and sum of weights
#pragma unroll
    for (int w = 1; w < 4 * KVA_WAVES; w++) all.x = fmaxf(all.x, refs[w * 4 + row]);
#pragma unroll
    for (int w = 0; w < 4 * KVA_WAVES; w++) all.y += sums[w * 4 + row] * kva_rescale(refs[w * 4 + row], all.x);
    constexpr int OC = L::OC, LD = OC + 4;
    float *ob = (float *)smem;  // [wave][16 columns][LD]
    const size_t part = ((size_t)split * a.own.Hk + hk) * a.rows + row0;
    const float per = 512.0f * kva_per(all.y), f = kva_rescale(st.ref, all.x) * st.wref;
#pragma unroll
    for (int c0 = 0; c0 < 64 * DC; c0 += OC) {
        if (c0 >= hd) continue;
        if (c0) __syncthreads();  // what the region held has been read
#pragma unroll
        for (int k = 0; k < OC / 16; k++)
            *(kva_f4_t *)(ob + (wave * 16 + col) * LD + 16 * k + 4 * g) = st.o[c0 / 16 + k] * per * f;
        __syncthreads();
        for (int x = tid; x < 4 * OC; x += 64 * KVA_WAVES) {
            const int r = x / OC, c = x % OC;
            if (r >= (int)n_rows || c0 + c >= hd) continue;
            float v = 0.0f;
#pragma unroll
            for (int w = 0; w < 4 * KVA_WAVES; w++) v += ob[(w * 4 + r) * LD + c];
            if (last) kva_out_row<T>(a, row0 + r, hk)[c0 + c] = kva_out<T>(v);
            else a.po[(part + r) * hd + c0 + c] = v;
        }
    }
    if (!last && tid < (int)n_rows) a.ml[part + tid] = all;
}

// The body of many rows: four waves of 16 rows, every wave every key tile.  A
// tile is widened once for the four of them, a quarter by each, into LDS in
// operand order (each 16-byte access of a wave is 1 KiB in a row) while the
// codes of the two tiles behind it travel; two buffers, one barrier a tile (256
// channels: one buffer, so that a CU still holds two workgroups, two barriers
// and one tile behind).  Two workgroups a CU, so that every SIMD has two waves
// at unlike places (one alone issues a vector operation every four cycles, two
// of one workgroup stand at its barriers together); 32 rows a wave would halve
// the widening but do not fit 256 registers.  64 requests of up to 2048 rows
// behind 16384, 32/8 heads of 128: 244 MB in 60.6 us with the join, 4.0 TB/s; fp4,
// half the bytes and no fewer operations, 134 MB in 56.7.
template <int DC>
struct KvaStage {
    static constexpr int KEYS = 4 * 2 * DC * 1024, BYTES = 2 * KEYS + 512, BUFS = DC < 4 ? 2 : 1;
};
template <int DC, bool HI>
struct KvaWideLds {
    static constexpr int Q = KVA_WAVES * 2 * DC * 1024 * (HI ? 2 : 1);  // under the stages, read into registers first
    static constexpr int S = KvaStage<DC>::BYTES * KvaStage<DC>::BUFS;
    static constexpr int BODY = Q > S ? Q : S;
    static constexpr int BYTES = BODY + 16 * KVA_WAVES * 4;
};

// A wave's quarter of a tile on its way: the keys of block `wave` and every
// fourth channel tile of the values.
template <int FMT, int DC>
struct KvaPart {
    kva_u4_t kc[DC], vc[DC];
    __device__ __forceinline__ void load(const KvaSlab &c, uint32_t tt, int hd, int col, int g, int wave) {
        const int nc = hd / 16;
        const uint8_t *kt = c.k + (size_t)tt * 64 * hd + (wave * nc) * 256 + col * 16;
        const uint8_t *vt = c.v + (size_t)tt * 64 * hd + col * 64 + g * 16;
#pragma unroll
        for (int x = 0; x < DC; x++) {
            const int chunk = 4 * x + g, ct = 4 * x + wave;
            kc[x] = *(const kva_u4_t *)(kt + (chunk < nc ? chunk : nc - 1) * 256);  // past the last chunk q is zero
            vc[x] = *(const kva_u4_t *)(vt + (ct < nc ? ct : nc - 1) * 1024);       // past the last tile: not stored
        }
    }
    __device__ __forceinline__ kva_h8_t key(int x, int u) const { return kva_wide<FMT>(kc[x][2 * u], kc[x][2 * u + 1]); }
    __device__ __forceinline__ kva_h8_t val(int x, int u, const kva_u4_t &keep) const {
        const kva_u4_t w = FMT == QBK_KV_FP8 ? vc[x] & keep : vc[x];
        return kva_wide<FMT>(w[2 * u], w[2 * u + 1]);
    }
};
template <int DC>
struct KvaPart<QBK_KV_FP4, DC> {
    kva_u2_t kc[DC], vc[DC];
    kva_u4_t vm[DC];
    uint32_t km[DC];
    __device__ __forceinline__ void load(const KvaSlab &c, uint32_t tt, int hd, int col, int g, int wave) {
        const int nc = hd / 16, ng = (int)c.ng;
        const uint8_t *kt = c.k + (size_t)tt * 32 * hd + ((wave >> 1) * nc) * 256 + col * 16 + (wave & 1) * 8;
        const uint8_t *vt = c.v + (size_t)tt * 1024 * ng + col * 64 + g * 16 + (wave & 1) * 8;
        const uint8_t *kmt = c.km + (size_t)tt * 64 * ng + col * 4 + wave, *vmt = c.vm + (size_t)tt * 64 * ng + g * 16;
#pragma unroll
        for (int x = 0; x < DC; x++) {
            const int chunk = 4 * x + g < nc ? 4 * x + g : nc - 1;  // past the last chunk q is zero
            const int m = 2 * x + (wave >> 1) < ng ? 2 * x + (wave >> 1) : ng - 1;  // past the last tile: not stored
            kc[x] = *(const kva_u2_t *)(kt + chunk * 256);
            km[x] = kmt[(chunk >> 1) * 64];
            vc[x] = *(const kva_u2_t *)(vt + m * 1024);
            vm[x] = *(const kva_u4_t *)(vmt + m * 64);
        }
    }
    __device__ __forceinline__ kva_h8_t key(int x, int u) const { return kva_key4(kc[x][u], kva_mul4<0>(km[x])[0]); }
    __device__ __forceinline__ kva_h8_t val(int x, int u, const kva_u4_t &keep) const {
        const kva_u4_t m = vm[x] & keep;
        return kva_val4(vc[x][u], m[2 * u], m[2 * u + 1]);
    }
};

template <int FMT, int DC, typename T, class Limit>
__device__ __forceinline__ void kva_wide_body(const KvAttArgs &a, char *smem, uint32_t row0, uint32_t n_rows,
                                              uint32_t hk, const KvaSlab &slab, uint32_t tile0, uint32_t tile1,
                                              uint32_t written, Limit limit, uint32_t split, bool last) {
    constexpr bool HI = sizeof(T) == 4;
    constexpr int STEPS = 2 * DC, KEYS = KvaStage<DC>::KEYS, BUFS = KvaStage<DC>::BUFS;
    using L = KvaWideLds<DC, HI>;
    const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);  // scalar: loops and addresses by it are too
    const int hd = (int)a.own.hd, nc = hd / 16;
    float *qfs = (float *)(smem + L::BODY);

    // This wave's part of a tile: the keys of block `wave` and every fourth
    // channel tile of the values.
    KvaPart<FMT, DC> part[BUFS];
    float sc[BUFS];  // waves 0 and 1: a key's and a value's scale a lane
    auto load = [&](uint32_t tt, int at) {
        part[at].load(slab, tt, hd, col, g, wave);
        if (wave < 2) sc[at] = (wave ? slab.vs : slab.ks)[(size_t)tt * 64 + lane];
    };
    auto stage = [&](uint32_t tt, int at, char *buf) {
        const uint32_t key0 = tt * 64;
        const bool tail = key0 + 64 > written;  // rows that were never written take no part, whatever they hold
        kva_u4_t keep = {~0u, ~0u, ~0u, ~0u};
        if (FMT != QBK_KV_INT8 && tail) keep = kva_keep(key0, written, g);  // NaN codes or multipliers
#pragma unroll
        for (int c = 0; c < DC; c++) {
#pragma unroll
            for (int u = 0; u < 2; u++) {
                *(kva_h8_t *)(buf + ((wave * STEPS + 2 * c + u) * 64 + lane) * 16) = part[at].key(c, u);
                *(kva_h8_t *)(buf + KEYS + ((2 * (4 * c + wave) + u) * 64 + lane) * 16) = part[at].val(c, u, keep);
            }
        }
        if (wave < 2) {
            const float x = tail && key0 + lane >= written ? 0.0f : sc[at];
            *(float *)(buf + 2 * KEYS + wave * 256 + lane * 4) = x;
        }
    };
    if (tile0 < tile1) load(tile0, 0);
    if (BUFS > 1 && tile0 + 1 < tile1) load(tile0 + 1, BUFS - 1);
    kva_queries<DC, KVA_WAVES, T>(a, smem, qfs, row0, n_rows, hk);
    __syncthreads();
    kva_h8_t qh[STEPS], ql[STEPS];
#pragma unroll
    for (int x = 0; x < STEPS; x++) {
        const char *at = smem + ((wave * STEPS + x) * 64 + lane) * 16;
        qh[x] = *(const kva_h8_t *)at;
        if constexpr (HI) ql[x] = *(const kva_h8_t *)(at + KVA_WAVES * STEPS * 1024);
    }
    const uint32_t my0 = wave * 16, r = my0 + col;  // this wave's first row, this lane's
    const bool rows = my0 < n_rows;
    KvaState<DC> st(qfs[r], limit(r < n_rows ? r : n_rows - 1));
    const uint32_t least = kva_scalar(limit(rows ? my0 : 0)), end = my0 + 16 < n_rows ? my0 + 16 : n_rows;
    const uint32_t most = rows ? kva_scalar(limit(end - 1)) : 0;  // no row of the wave sees keys from here on
    __syncthreads();  // the queries are read

    auto work = [&](uint32_t tt, const char *buf) {
        const uint32_t key0 = tt * 64;
        if (key0 >= most) return;
        kva_f4_t ks[4], vs[4], s[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            ks[i] = *(const kva_f4_t *)(buf + 2 * KEYS + (16 * i + 4 * g) * 4);
            vs[i] = *(const kva_f4_t *)(buf + 2 * KEYS + 256 + (16 * i + 4 * g) * 4);
            s[i] = kva_f4_t{0, 0, 0, 0};
        }
#pragma unroll
        for (int x = 0; x < STEPS; x++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const kva_h8_t kf = *(const kva_h8_t *)(buf + ((i * STEPS + x) * 64 + lane) * 16);
                s[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qh[x], s[i], 0, 0, 0);
                if constexpr (HI) s[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, ql[x], s[i], 0, 0, 0);
            }
        kva_scores(s, ks, st.qf);
        if (key0 + 64 > least) kva_mask(s, vs, key0 + 4 * g, st.lim);
        kva_reference(s, st.ref, st.sum, st.wref);
        kva_weights(s, vs, st.ref, st.sum);
        kva_weight_reference(s, st.wref, st.o);
        kva_h8_t ph[2], pl[2];
        kva_operands<HI>(s, st.wref, ph, pl);
#pragma unroll
        for (int ct = 0; ct < 4 * DC; ct++)
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const kva_h8_t vf = *(const kva_h8_t *)(buf + KEYS + ((2 * ct + u) * 64 + lane) * 16);
                st.o[ct] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, ph[u], st.o[ct], 0, 0, 0);
                if constexpr (HI) st.o[ct] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pl[u], st.o[ct], 0, 0, 0);
            }
    };
    for (uint32_t t = tile0; t < tile1; t += BUFS)
#pragma unroll
        for (int p = 0; p < BUFS; p++) {
            const uint32_t tt = t + p;
            if (tt >= tile1) continue;
            char *buf = smem + p * KvaStage<DC>::BYTES;
            if (BUFS == 1 && tt > tile0) __syncthreads();
            stage(tt, p, buf);
            __syncthreads();  // every wave is past the tile before, so the other buffer is free as well
            if (tt + BUFS < tile1) load(tt + BUFS, p);
            work(tt, buf);
        }
    const float l = kva_sum4(st.sum), per = kva_per(l);
    if (r >= n_rows) return;
    if (last) {
        T *dst = kva_out_row<T>(a, row0 + r, hk) + 4 * g;
#pragma unroll
        for (int ct = 0; ct < 4 * DC; ct++)
            if (ct < nc)
#pragma unroll
                for (int j = 0; j < 4; j++) dst[16 * ct + j] = kva_out<T>(st.o[ct][j] * per * st.wref);
    } else {
        const size_t at = ((size_t)split * a.own.Hk + hk) * a.rows + row0 + r;
        float *dst = a.po + at * hd + 4 * g;
#pragma unroll
        for (int ct = 0; ct < 4 * DC; ct++)
            if (ct < nc) *(kva_f4_t *)(dst + 16 * ct) = st.o[ct] * per * st.wref;
        if (g == 0) a.ml[at] = float2{st.ref, l};
    }
}

enum { KVA_ROWS16 = 0, KVA_ROWS64 = 1, KVA_ROWS4 = 2 };  // a body's rows

template <int FMT, int DC, int ROWS, typename T, class... ARGS>
__device__ __forceinline__ void kva_any(ARGS &&...args) {
    if constexpr (ROWS == KVA_ROWS64) kva_wide_body<FMT, DC, T>(args...);
    else if constexpr (ROWS == KVA_ROWS4) kva_few<DC, T>(args...);
    else kva_body<FMT, DC, T>(args...);
}

template <int FMT, int DC, bool WIDEP, int OWN, typename T>
__global__ void __launch_bounds__(64 * KVA_WAVES, DC < 4 ? 2 : 1) kva_items(KvAttArgs a) {
    extern __shared__ char smem[];
    const uint32_t Hk = a.own.Hk;
    const bool last = a.sp + a.ss == 1;
    if (blockIdx.x < a.n_pre) {
        // kv heads next to each other: with eight of them each stays on one XCD, whose L2 serves its row tiles
        uint32_t hk, rt, rest;
        const uint32_t split = a.by_rtp.split(a.by_hk.split(blockIdx.x, hk), rt);
        constexpr uint32_t R = WIDEP ? 64 : 16;
        const uint32_t row0 = rt * R, n_rows = a.rows - row0 < R ? a.rows - row0 : R;
        const uint32_t tiles = (a.prefix_len + 63) / 64, run = a.by_sp.split(tiles + a.sp - 1, rest);
        const uint32_t t0 = split * run < tiles ? split * run : tiles, t1 = t0 + run < tiles ? t0 + run : tiles;
        const KvaSlab slab = KvaSlab::of<FMT>(a.pre, a.pre.slab(a.prefix_seq, hk));
        const uint32_t len = a.prefix_len;
        kva_any<FMT, DC, WIDEP ? KVA_ROWS64 : KVA_ROWS16, T>(a, smem, row0, n_rows, hk, slab, t0, t1, len, [&](uint32_t) { return len; }, split,
                                  last);
        return;
    }
    const uint32_t item = blockIdx.x - a.n_pre;
    uint32_t hk, rt, b;
    const uint32_t split = a.by_n.split(a.by_rts.split(a.by_hk.split(item, hk), rt), b);
    const uint32_t end = kva_end(a, b), len = kva_len(a, end), tiles = (len + 63) / 64, run = kva_run(a, len);
    if (split * run >= tiles && split > 0) return;  // split 0 is there for a sequence with no rows
    constexpr uint32_t R = OWN == KVA_ROWS64 ? 64 : 16;
    const uint32_t per = a.sq * a.G, r0 = rt * R, n_rows = per - r0 < R ? per - r0 : R;
    const uint32_t sq = a.sq;
    const KvaRow rows(a, r0);
    // own rows seen by row r of the body: end - sq + t + 1, none where that is negative; end is past len where a step's
    // last tokens have no room, which does not move the others
    auto limit = [&](uint32_t r) {
        uint32_t t, head;
        rows.at(r, t, head);
        const uint32_t up = end + t + 1, seen = up > sq ? up - sq : 0;
        return seen < len ? seen : len;
    };
    const uint32_t most = (kva_scalar(limit(n_rows - 1)) + 63) / 64;
    uint32_t t1 = split * run + run;
    t1 = t1 < most ? t1 : most;
    const KvaSlab slab = KvaSlab::of<FMT>(a.own, a.own.slab(a.first_seq + b, hk));
    kva_any<FMT, DC, OWN, T>(a, smem, b * per + r0, n_rows, hk, slab, split * run, t1, len, limit, a.sp + split, last);
}

// A wave a row and kv head: the partial results of its splits on their largest
// reference.  Four channels a lane and, up to 128 channels, two or four splits
// at a time; everything is asked for before anything is used, so that the
// partial rows and their references take one latency (1024 rows: 4.3 us).
template <typename T, int LANES>
__global__ void __launch_bounds__(256) kva_join(KvAttArgs a) {
    constexpr int STEP = 64 / LANES, N = (2 * KVA_MAX_SPLITS + STEP - 1) / STEP, BATCH = N < 16 ? N : 16;
    const uint32_t item = blockIdx.x * 4 + (uint32_t)__builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t lane = threadIdx.x & 63, Hk = a.own.Hk, hd = a.own.hd;
    if (item >= a.rows * Hk) return;
    uint32_t rho, head, rest;
    const uint32_t hk = a.by_rows.split(item, rho), query = a.by_g.split(rho, head);
    uint32_t splits = a.sp;
    if (a.ss) {
        const uint32_t len = kva_len(a, kva_end(a, a.by_sq.split(query, rest))), run = kva_run(a, len);
        for (uint32_t at = 0; at == 0 || (at < len && splits < a.sp + a.ss); at += 64 * run) splits++;
    }
    splits = kva_scalar(splits);
    float m = -INFINITY, l = 0.0f;
    if (lane < splits) {
        const float2 v = a.ml[((size_t)lane * Hk + hk) * a.rows + rho];
        m = v.x;
        l = v.y;
    }
    const uint32_t c = 4 * (lane % LANES), sub = lane / LANES;
    const float *src = a.po + ((size_t)hk * a.rows + rho) * hd + (c < hd ? c : 0);
    const size_t apart = (size_t)Hk * a.rows * hd;
    float share = 0.0f;  // of the row's weights, this lane's split's
    kva_f4_t v = {0, 0, 0, 0};
#pragma unroll
    for (int b = 0; b < N; b += BATCH) {
        if (b * STEP >= (int)splits) continue;
        kva_f4_t x[BATCH];
#pragma unroll
        for (int k = 0; k < BATCH; k++) {
            const uint32_t s = (b + k) * STEP + sub;
            if ((b + k) * STEP < (int)splits) x[k] = *(const kva_f4_t *)(src + (s < splits ? s : splits - 1) * apart);
        }
        if (b == 0) {
            float M = m;
#pragma unroll
            for (int o = 32; o >= 1; o >>= 1) M = fmaxf(M, __shfl_xor(M, o, 64));
            const float own = lane < splits ? l * kva_rescale(m, M) : 0.0f;
            float sum = own;
#pragma unroll
            for (int o = 32; o >= 1; o >>= 1) sum += __shfl_xor(sum, o, 64);
            share = sum == 0.0f ? 0.0f : own / sum;
        }
#pragma unroll
        for (int k = 0; k < BATCH; k++) {
            const uint32_t s = (b + k) * STEP + sub;
            const float fs = __shfl(share, (int)(s < 64 ? s : 63), 64);
            if (s < splits) v += x[k] * fs;
        }
    }
#pragma unroll
    for (int o = LANES; o < 64; o <<= 1)
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] += __shfl_xor(v[e], o, 64);
    if (lane >= LANES || c >= hd) return;
    T *dst = kva_out_row<T>(a, rho, hk) + c;
#pragma unroll
    for (int e = 0; e < 4; e++) dst[e] = kva_out<T>(v[e]);
}

// How a call is cut: row tiles (16 or 64 rows) and splits of the prefix and of
// the sequences' own rows.
struct KvaPlan {
    bool widep, wides;  // bodies of 64 rows
    bool few;           // own rows by the body of four
    uint32_t rtp, rts, sp, ss;
    uint64_t items;
    size_t bytes;
};

// fp4: splits of a prefix of tp tiles for op row tiles, `own` tiles of own rows beside it.  A workgroup takes its run of
// tiles (the body of 16 rows: four at a time) and as long as C more; two on a CU take 1.45 (16 rows: 1.65) times one's
// time, of heads past 128 twice, since one fills it.  Own rows are read by the second workgroup of a CU while the first
// computes, so that the prefix stays within one a CU where they are as many tiles (16 rows: a third; us for 256 / 512
// workgroups, 32/8 heads of 128, 64 rows: 128 row tiles of 16 behind 16384 55.0 / 48.2, with 1000 own rows each 55.9 /
// 53.2, with 2000 57.3 / 63.7; 512 tiles behind 4096 58.5 / 51.7, behind 16384 185 / 133; 16 rows: 64 tiles behind 16384
// 34.8 / 31.0, with 2000 own rows 35.8 / 40.3; 40 of heads of 80 behind 4001, 240 and 280 to 320 14.5 / 17.2, 16.0).
static uint32_t kva_prefix_splits(uint64_t op, size_t tp, bool wide, size_t dc, uint64_t own) {
    const uint64_t round = wide ? 1 : KVA_WAVES, fixed = wide ? 200 : 50, both = dc == 4 ? 40 : wide ? 29 : 33;  // by 20
    const uint64_t most = div_ceil(tp, KVA_WAVES) < KVA_MAX_SPLITS ? div_ceil(tp, KVA_WAVES) : KVA_MAX_SPLITS;
    uint64_t best = 1, least = ~0ull;
    for (uint64_t sp = 1; sp <= most; sp++) {
        const uint64_t groups = op * sp;
        if (sp > 1 && groups > (own * (wide ? 1 : 3) > op * tp ? 256 : 512)) break;
        const uint64_t rest = groups % 512, slots = groups / 512 * both + (rest > 256 ? both : rest ? 20 : 0);
        const uint64_t cost = (20 * div_ceil(div_ceil(tp, sp), round) + fixed) * slots;
        if (cost < least) {
            least = cost;
            best = sp;
        }
    }
    return (uint32_t)div_ceil(tp, div_ceil(tp, best));  // none without a tile
}

static KvaPlan kva_plan(const qbk_kv_shape *s, size_t n_heads, size_t n, size_t sq, size_t max_len, size_t prefix_len) {
    KvaPlan p{};
    const size_t Hk = s->n_kv_heads, G = n_heads / Hk, rows = n * sq * G, per = sq * G;
    const size_t dc = s->head_dim > 128 ? 4 : s->head_dim > 64 ? 2 : 1;
    // The body of 64 rows reads and widens a tile once for four of 16 rows, that of 16 rows splits a sequence's tiles
    // over its waves and is done sooner.  Own rows take the first once there are more items of 16 rows than the card
    // holds at once (us by 64 / 16 rows, 32/8 heads of 128, sequences up to 300: 512 items 13.3 / 11.3, 1024 13.8 /
    // 19.4, 2048 21 / 35; up to 1500: 27.8 / 21.1, 36.2 / 36.4, 45 / 66; heads of 64, 1024 items 9.5 / 11.7 and 24.8 /
    // 21.8; heads of 256, 256 items 24.5 / 17.6 and 41.5 / 31.3, 512 24.9 / 29.3 and 53.8 / 51.9).
    p.wides = per > 16 && max_len && (uint64_t)n * Hk * div_ceil(per, 16) > 1024 / dc;
    // fp4, whose tiles take longer to widen, past 512 keys only from more items on and where most of the 64 rows are
    // there (32/8 heads of 128, 1024 items up to 300 15.9 / 17.7, up to 700 24.8 / 23.8, up to 1500 41.9 / 34.8, with 32
    // rows a sequence 43.2 / 35.7; 2048 up to 1500 48.8 / 62.9; heads of 64, 1024 28.9 / 23.6, 2048 33.3 / 38.5; of 256,
    // 512 items up to 300 28.9 / 23.5, 1024 31 / 45 and 89 / 86).
    const bool fp4 = s->format == QBK_KV_FP4;
    if (fp4 && (max_len > 512 || dc == 4))
        p.wides = p.wides && per > 32 && (uint64_t)n * Hk * div_ceil(per, 16) > (dc == 4 ? 1023 : 1024);
    // The prefix, split over the card by either, from the row tiles on whose reading of the same codes shows (8 kv heads
    // of 128 behind 500, 8192 and 16384: 64 tiles 13.9 / 11.5, 23.7 / 20.7, 31.2 / 32.5; 128 tiles 14.9 / 15.8, 32.4 /
    // 31.4, 49.2 / 53.9; heads of 64 behind 500 and 2048: 128 tiles 12.1 / 10.3, 14.2 / 12.6, 512 24.3 / 24.8, 29.6 /
    // 32.4; heads of 256: 32 tiles 19.8 / 14.2, 21.6 / 23.2, 64 tiles 20.8 / 21.0, 24.0 / 26.8).
    // fp4 keeps to the first for heads of 256 (behind 16384: 128 tiles 122 / 101, 256 tiles 223 / 180, 512 422 / 351).
    p.widep = p.wides || (prefix_len && !(fp4 && dc == 4) &&
                          (uint64_t)Hk * div_ceil(rows, 16) >= (dc == 1 ? 512 : 256 / dc));
    p.few = fp4 && per <= 4;
    p.rtp = (uint32_t)div_ceil(rows, p.widep ? 64 : 16);
    p.rts = (uint32_t)div_ceil(per, p.wides ? 64 : 16);
    const uint64_t op = prefix_len ? (uint64_t)Hk * p.rtp : 0, os = (uint64_t)n * Hk * p.rts;
    // Splits: a workgroup a CU for the prefix, of four key tiles at least, and two for own rows where the sequences
    // alone leave CUs idle; past that a run of at most 64 tiles, so that no workgroup outlasts the rest on one long
    // sequence.  More of them write and join more partial rows (us for 128, 256 and 512 workgroups of the prefix: 32
    // requests behind 8192 30.0, 21.9, 22.8, 64 behind 16384 86.8, 54.6, 70.9; own rows of 32 sequences up to 2085: one
    // split 23.5, two 25.1, of 8 sequences for 128, 256, 512 workgroups 15.8, 13.1, 13.2; 32 sequences up to 16384,
    // runs of 16, 64 and 512 tiles: 159.8, 154.1, 161.9).
    const size_t tp = div_ceil(prefix_len, 64), ts = div_ceil(max_len, 64);
    auto splits = [](uint64_t want, size_t tiles) -> uint32_t {
        const uint64_t most = div_ceil(tiles, KVA_WAVES);
        want = want < most ? want : most;
        return (uint32_t)(want < 1 ? 1 : want > KVA_MAX_SPLITS ? KVA_MAX_SPLITS : want);
    };
    if (prefix_len) p.sp = fp4 ? kva_prefix_splits(op, tp, p.widep, dc, os * ts) : splits(div_ceil(256, op), tp);
    if (max_len) p.ss = splits(os >= 256 ? div_ceil(ts, 64) : div_ceil(512, os), ts);
    // a second launch takes longer than one more tile a wave (one sequence of 512 rows in one launch 7.9 us, split 9.2;
    // of 768 9.6 and 9.4, of 1024 11.1 and 9.4)
    // (the body of four rows, f32, in one launch and split, heads of 64: 1024 rows 7.2 and 7.9, 1500 8.8 and 8.2; of 128:
    // 768 9.0 and 9.3, 1024 10.2 and 9.5; of 256: 512 12.2 and 12.3, 600 14.7 and 12.5; bf16 6.7 and 8.1, 8.1 and 8.1;
    // 8.1 and 9.2, 9.2 and 9.2; 11.0 and 11.6, 12.9 and 11.8)
    const size_t tiles = !p.few || dc == 4 ? 2 : dc == 2 ? 3 : 4;  // a wave's
    if (!prefix_len && ts <= tiles * KVA_WAVES) p.ss = 1;
    p.items = op * p.sp + os * p.ss;
    p.bytes = p.sp + p.ss > 1 ? round_up((size_t)(p.sp + p.ss) * Hk * rows * (s->head_dim * 4 + 8), 256) : 0;
    return p;
}

template <int FMT, int DC, bool WIDEP, int OWN, typename T>
static int kva_launch(const KvAttArgs &a, uint64_t items, int device, hipStream_t st) {
    constexpr bool HI = sizeof(T) == 4;
    constexpr int N = KvaLds<DC, HI>::BYTES, WIDE = KvaWideLds<DC, HI>::BYTES;
    constexpr int lds = !WIDEP ? N : OWN == KVA_ROWS64 || WIDE > N ? WIDE : N;
    static_assert(OWN != KVA_ROWS64 || WIDEP, "own rows are no more than the prefix's");
    void (*k)(KvAttArgs) = kva_items<FMT, DC, WIDEP, OWN, T>;
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
    if (p.wides) return kva_launch<FMT, DC, true, KVA_ROWS64, T>(a, p.items, device, st);
    constexpr bool FP4 = FMT == QBK_KV_FP4;
    if constexpr (FP4) {
        if constexpr (DC < 4)
            if (p.few && p.widep) return kva_launch<FMT, DC, true, KVA_ROWS4, T>(a, p.items, device, st);
        if (p.few) return kva_launch<FMT, DC, false, KVA_ROWS4, T>(a, p.items, device, st);
    }
    if constexpr (!FP4 || DC < 4)
        if (p.widep) return kva_launch<FMT, DC, true, KVA_ROWS16, T>(a, p.items, device, st);
    return kva_launch<FMT, DC, false, KVA_ROWS16, T>(a, p.items, device, st);
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
    if (n_heads > (1u << 13)) return fail(QBK_ERR_VALIDATION, "kv attention takes up to 8192 heads");
    if (sq == 0) return fail(QBK_ERR_VALIDATION, "kv attention requires at least one query a sequence");
    if (max_len > s->capacity)
        return fail(QBK_ERR_VALIDATION, fmt("max_len %zu is past the kv cache's capacity of %zu", max_len, s->capacity));
    if (n > 0x7FFFFFFFull || sq > 0x3FFFFFFFull || n_heads > 0x7FFFFFFFull || prefix_len > 0x7FFFFF00ull ||
        (n && (unsigned __int128)n * sq * (n_heads / s->n_kv_heads) > 0x7FFFFFFFull))
        return fail(QBK_ERR_VALIDATION, "kv attention: too many query rows for one launch");
    const KvaPlan p = n ? kva_plan(s, n_heads, n, sq, max_len, prefix_len) : KvaPlan{};
    // a launch is below 2^32 threads; the join takes four rows a workgroup
    if (p.items > 0xFFFFFF || (unsigned __int128)n * sq * n_heads > (p.bytes ? 4 * 0xFFFFFFull : 0x7FFFFFFFull))
        return fail(QBK_ERR_VALIDATION, "kv attention: too many query rows for one launch");
    return QBK_OK;
}

// qbk_attention_kv_dev; plus seq_q: lens[i] counts the rows before the queries'.
int attention_kv_run(qbk_ctx *ctx, const qbk_kv_shape *shape, const void *cache, size_t first_seq, size_t n,
                     const uint32_t *lens, uint32_t plus, size_t max_len, const qbk_kv_shape *prefix_shape,
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
    a.plus = plus;
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
    a.by_hk.set((uint32_t)shape->n_kv_heads);
    a.by_rtp.set(p.rtp);
    a.by_rts.set(p.rts);
    a.by_n.set(a.n);
    a.by_g.set(a.G);
    a.by_sq.set(a.sq);
    a.by_rows.set(a.rows);
    a.by_sp.set(p.sp ? p.sp : 1);
    a.by_ss.set(p.ss ? p.ss : 1);
    a.scale = (float)(1.4426950408889634 / sqrt((double)shape->head_dim));
    const size_t parts = (size_t)(p.sp + p.ss) * shape->n_kv_heads * a.rows;
    a.po = (float *)workspace;
    a.ml = (float2 *)(a.po + parts * shape->head_dim);
    hipStream_t st = (hipStream_t)stream;
    if (p.items) {
        if (shape->format == QBK_KV_INT8)
            rc = dtype == QBK_F32 ? kva_dispatch<QBK_KV_INT8, float>(a, p, ctx->device, st)
                                  : kva_dispatch<QBK_KV_INT8, uint16_t>(a, p, ctx->device, st);
        else if (shape->format == QBK_KV_FP8)
            rc = dtype == QBK_F32 ? kva_dispatch<QBK_KV_FP8, float>(a, p, ctx->device, st)
                                  : kva_dispatch<QBK_KV_FP8, uint16_t>(a, p, ctx->device, st);
        else
            rc = dtype == QBK_F32 ? kva_dispatch<QBK_KV_FP4, float>(a, p, ctx->device, st)
                                  : kva_dispatch<QBK_KV_FP4, uint16_t>(a, p, ctx->device, st);
        if (rc) return rc;
    }
    if (p.sp + p.ss == 1) return QBK_OK;  // the items wrote the output
    const dim3 grid((unsigned)div_ceil((size_t)a.rows * shape->n_kv_heads, 4));
    void (*join)(KvAttArgs) =
        dtype == QBK_F32 ? (a.own.hd <= 64 ? kva_join<float, 16> : a.own.hd <= 128 ? kva_join<float, 32> : kva_join<float, 64>)
                         : (a.own.hd <= 64    ? kva_join<uint16_t, 16>
                            : a.own.hd <= 128 ? kva_join<uint16_t, 32>
                                              : kva_join<uint16_t, 64>);
    hipLaunchKernelGGL(join, grid, dim3(256), 0, st, a);
    QBK_HIP(hipGetLastError());
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
    return attention_kv_run(ctx, shape, cache, first_seq, n, lens, 0, max_len, prefix_shape, prefix, prefix_seq,
                            prefix_len, n_heads, seq_q, q, dtype, out, workspace, workspace_size, stream);
}

}  // extern "C"
