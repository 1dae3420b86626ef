// kvcache.h -- layout of the 8-bit KV cache (kvcache.hip writes and reads it,
// attention_kv.hip attends over it).
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
#pragma once

#include "qbk_internal.h"

namespace qbk {

struct KvView {
    uint8_t *k, *v;   // codes
    float *ks, *vs;   // scales
    size_t cap, cap64;
    uint32_t n_seqs, Hk, hd;

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

// The shape's checks; *bytes the buffer's size.
int kv_check_shape(const qbk_kv_shape *s, size_t *bytes);
KvView kv_view(const qbk_kv_shape *s, const void *cache);

}  // namespace qbk
