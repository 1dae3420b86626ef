// kvcache.h -- layouts of the 8-bit and 4-bit KV caches (kvcache.hip and
// kvcache4.hip write and read them, attention_kv.hip attends over them).
//
// A buffer holds every sequence's key codes, then value codes, then key and
// value scales; each is [n_seqs][n_kv_heads] slabs of cap64 = capacity rounded
// up to 64 rows:
//   keys    [row / 16][channel / 16][row % 16][channel % 16]
//   values  [row / 64][channel][byte 16 g + 4 i + j], row % 64 = 16 i + 4 g + j
//   scales  [row] f32
// so that 64 rows are one contiguous run of 64 hd bytes and each 16-byte load
// of a wave over either is 1 KiB in a row AND the operand of
// v_mfma_f32_16x16x32_f16 that the lane has to hold: keys as the A rows of
// K q^T (lane l: row l % 16, channels of chunk l / 16), values as the A rows
// of V^T p^T (lane l: channel l % 16, the sixteen rows whose scores the lane's
// group l / 16 holds after K q^T).  Nothing is transposed or exchanged between
// lanes when the cache is read; the writer pays, row by row with four byte-wide
// stores a value dword, by 64-row tiles with a turn of 4 x 4 bytes in LDS.
// An int8 code c is held as the byte c + 128: 0x6400 | byte is the fp16 number
// 1024 + byte, from which one packed subtraction of 1152 leaves c.
//
// The 4-bit format (fp4) has the same order with half the bytes, so that the
// same loads are the same operands: a key's 16 channels are 8 bytes, those of
// rows r and r + 16 side by side, and a channel's 16 rows are 8 bytes, those of
// channels c and c + 16 side by side:
//   keys    [row / 32][channel / 16][row % 16][row / 16 % 2][channel % 16 / 2], the even channel in the low half
//   values  [row / 64][channel / 32][channel % 16][g][channel / 16 % 2][byte 2 i + j / 2], row % 64 = 16 i + 4 g + j,
//           the even j in the low half; head_dim is filled up to a multiple of 32
//   then a byte for 32 channels of a row, the e4m3 multiplier of their codes, in the order that a lane needs them:
//   keys    [row / 64][channel / 32][4 (row % 16) + row / 16 % 4]
//   values  [row / 64][channel / 32][16 g + 4 i + j]
//   then the scales as above.
// A code (e2m1, two bits of significand) times its multiplier (four) is an fp16
// number, so that a widened operand is exact, as those of the 8-bit formats are.
#pragma once

#include "qbk_internal.h"

namespace qbk {

struct KvView {
    uint8_t *k, *v;   // codes
    float *ks, *vs;   // scales
    size_t cap, cap64;
    uint32_t n_seqs, Hk, hd;
    uint8_t *km, *vm;  // fp4: multipliers

    __host__ __device__ uint32_t groups() const { return (hd + 31) / 32; }
    __host__ __device__ size_t slab(size_t seq, size_t head) const { return (seq * Hk + head) * cap64; }
};

// Byte of a key's / value's code within its slab.
__host__ __device__ static inline size_t kv_key_at(size_t row, uint32_t ch, uint32_t hd) {
    return (row >> 4) * (16 * (size_t)hd) + (ch >> 4) * 256 + (row & 15) * 16 + (ch & 15);
}
__host__ __device__ static inline size_t kv_val_at(size_t row, uint32_t ch, uint32_t hd) {
    const uint32_t t = (uint32_t)(row & 63);
    return (row >> 6) * (64 * (size_t)hd) + (size_t)ch * 64 + ((t >> 2) & 3) * 16 + (t >> 4) * 4 + (t & 3);
}


// fp4: bytes of one code's pair within its slab (channel even for a key; row
// 4 g + j of a value with j even in the low half), and of the multipliers.
__host__ __device__ static inline size_t kv4_key_at(size_t row, uint32_t ch, uint32_t hd) {
    return (row >> 5) * (16 * (size_t)hd) + (ch >> 4) * 256 + (row & 15) * 16 + (row >> 4 & 1) * 8 + (ch & 15) / 2;
}
__host__ __device__ static inline size_t kv4_val_at(size_t row, uint32_t ch, uint32_t groups) {
    const uint32_t t = (uint32_t)(row & 63);
    return (row >> 6) * (1024 * (size_t)groups) + (ch >> 5) * 1024 + (ch & 15) * 64 + (t >> 2 & 3) * 16 +
           (ch >> 4 & 1) * 8 + (t >> 4) * 2 + (t >> 1 & 1);
}
__host__ __device__ static inline size_t kv4_key_mul_at(size_t row, uint32_t group, uint32_t groups) {
    const uint32_t t = (uint32_t)(row & 63);
    return (row >> 6) * (64 * (size_t)groups) + group * 64 + (t & 15) * 4 + (t >> 4);
}
__host__ __device__ static inline size_t kv4_val_mul_at(size_t row, uint32_t group, uint32_t groups) {
    const uint32_t t = (uint32_t)(row & 63);
    return (row >> 6) * (64 * (size_t)groups) + group * 64 + (t >> 2 & 3) * 16 + (t >> 4) * 4 + (t & 3);
}

// The shape's checks; *bytes the buffer's size.
int kv_check_shape(const qbk_kv_shape *s, size_t *bytes);
KvView kv_view(const qbk_kv_shape *s, const void *cache);

}  // namespace qbk
