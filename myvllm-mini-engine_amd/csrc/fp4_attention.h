// What decode and prefill over packed pages share: the tile of 32 keys that
// one wave scores and accumulates.
//
// Both products run on the 16x16x32 matrix instruction with the keys in its
// rows and up to 16 query rows (heads of a group, or (token, head) pairs) in
// its columns:
//   S^T[key, row]  = sum_d K[key, d] Q[row, d]
//   O^T[d, row]    = sum_key V[key, d] P[row, key]
// The result layout of the first (lane: column lane % 16, rows 4 * (lane / 16)
// .. + 3) holds for each lane 4 keys of its own query row, and two such
// results are 8 keys: exactly the lane's part of the second product's operand
// when both operands number the keys of a tile as
//   k = 8 * g + j  ->  key 4 * g + j (j < 4), 16 + 4 * g + j - 4 (j >= 4)
// So probabilities never leave their lane.  V^T comes from row-major fp16 rows
// in LDS by transposing reads (4 keys of 16 dims per 16 lanes and read).
#pragma once

#include "fp4_cache.h"

namespace mvme {
namespace fp4 {

typedef short s16x4 __attribute__((ext_vector_type(4)));

// Probabilities are exp2(x - reference) with the reference kept 8 below the
// largest score seen when it was set, and moved when a score passes it by 14:
// fp16 then holds every probability down to 2^-24 - 8 of the largest with
// full 11 bits from 2^-22 on, and none overflows.
constexpr float kRefBelow = 8.f;
constexpr float kRefSlack = 14.f;
constexpr float kRefNone = -3.0e38f;  // no score yet: below every finite one

constexpr int kTileKeys = 32;

// Byte address inside a tile of rows of 2 * D bytes.  16-byte chunks are XORed
// with a number of their row that puts these into different banks: 16 rows of
// one chunk (or rows 0-3 and 12-15 of one and 4-11 of the next: the order in
// which 16-byte reads are served), the chunk pairs of 8 consecutive rows that
// a transposing read takes, and 4 rows of every fourth chunk.  Rows whose
// length is a multiple of 256 bytes start in the same bank, of 128 bytes in
// one of two, of 64 bytes in one of four.
template <int D>
struct TileLayout {
    static constexpr int kChunks = D / 8;
    __device__ static inline constexpr int number(int row) {
        if (kChunks % 16 == 0) return 2 * (row & 7) | ((row >> 1) & 1);
        if (kChunks % 8 == 0) return 2 * ((row >> 1) & 3) | ((row >> 2) & 1);
        return 2 * ((row >> 2) & 1) | ((row >> 3) & 1);
    }
    __device__ static inline int at(int row, int chunk) { return row * 2 * D + ((chunk ^ number(row)) << 4); }
};

// A lane's place in a tile, for accesses at chunks `first + i` of its row.  For
// power-of-two rows the XOR of the layout acts on address bits of its own, so
// one register and an XOR with a constant give every address; `forget` keeps
// the compiler from holding them all in registers across a loop.
template <int D>
struct TileAddress {
    static constexpr bool kPow2 = (D & (D - 1)) == 0;
    int row, first, base;
    __device__ inline TileAddress(int row, int first, int bytes = 0) : row(row), first(first) {
        base = (kPow2 ? TileLayout<D>::at(row, first) : row * 2 * D) + bytes;
    }
    __device__ inline void forget() { asm volatile("" : "+v"(base)); }
    __device__ inline int chunk(int i) const {  // i and first have no bits in common
        if constexpr (kPow2) return base ^ (i << 4);
        return base + (((first + i) ^ TileLayout<D>::number(row)) << 4);
    }
};

// 16 dims of 8 keys for the value product: A operand of 16 dims and 32 keys of a tile in fp16.  `at` is the lane's
// address for the first 16 keys: row 4 g + r / 4, the 8 bytes r % 4 of the 16 dims.
template <int D>
__device__ inline u32x4 value_operand(const uint8_t* tile, int at) {
    typedef __attribute__((address_space(3))) s16x4* lds_ptr;
    const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(tile + at));
    const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(tile + at + 16 * 2 * D));
    const u32x2 x = __builtin_bit_cast(u32x2, a), y = __builtin_bit_cast(u32x2, b);
    return u32x4{x[0], x[1], y[0], y[1]};
}

}  // namespace fp4
}  // namespace mvme
