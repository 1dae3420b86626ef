// kvcache_rows.h -- which row of a call stands where in the cache, for the
// kernels that write and read rows (kvcache.hip, kvcache4.hip).
#pragma once

#include "kvcache.h"

namespace qbk {

struct KvRows {
    KvView c;
    const uint32_t *row_start, *pos;  // row_start null: `per` rows a sequence
    size_t stride;                    // values from one row to the next
    uint32_t n_rows, n, per, first;
    bool tiles;  // by 64-row tiles
};

// The sequence s (0 .. n - 1) that claims row r, and the call's rows start ..
// end - 1 of it; row_start null: `per` rows a sequence.
__device__ __forceinline__ bool kv_claim(const uint32_t *row_start, uint32_t n, uint32_t per, uint32_t r, uint32_t &s,
                                         uint32_t &start, uint32_t &end) {
    if (row_start) {
        uint32_t lo = 0, hi = n;  // the last s with row_start[s] <= r
        while (hi - lo > 1) {
            const uint32_t mid = lo + (hi - lo) / 2;
            if (row_start[mid] <= r) lo = mid;
            else hi = mid;
        }
        s = lo;
        start = row_start[s];
        end = row_start[s + 1];
        return r >= start && r < end;
    }
    s = r / per;
    start = s * per;
    end = start + per;
    return true;
}

// The sequence (0 .. n - 1) and position of row r; false for a row that no
// sequence claims or that lies past the capacity.  Whatever row_start holds,
// a row that passes addresses the cache in bounds.
__device__ __forceinline__ bool kv_place(const KvRows &a, uint32_t r, uint32_t &seq, size_t &at, uint32_t &start,
                                         uint32_t &end) {
    uint32_t s;
    if (!kv_claim(a.row_start, a.n, a.per, r, s, start, end)) return false;
    seq = a.first + s;
    at = (size_t)a.pos[s] + (r - start);
    return at < a.c.cap;
}
__device__ __forceinline__ bool kv_place(const KvRows &a, uint32_t r, uint32_t &seq, size_t &at) {
    uint32_t start, end;
    return kv_place(a, r, seq, at, start, end);
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

// Four values at any alignment (one access on this machine).
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Kv4 {
    T v[4];
};

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

// Tile numbers of a call (kv_tile): at most two a segment past the tiles that the rows fill.
static inline size_t kv_tiles(size_t n_rows, size_t n) { return n_rows / 64 + 2 * (n + 2); }

// The 4-bit format's rows in and out (kvcache4.hip); dtype as the call's.
void kv4_write_go(const KvRows &a, const void *k, const void *v, int dtype, hipStream_t s);
void kv4_read_go(const KvRows &a, void *k, void *v, int dtype, hipStream_t s);

}  // namespace qbk
