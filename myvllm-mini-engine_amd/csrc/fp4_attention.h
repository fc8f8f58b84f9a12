// What decode and prefill over packed pages share: tiles of keys or values in
// LDS, and the softmax's reference.
//
// Both products have the keys in the rows of the matrix instruction and query
// rows (heads of a group, or (token, head) pairs) in its columns:
//   S^T[key, row]  = sum_d K[key, d] Q[row, d]
//   O^T[d, row]    = sum_key V[key, d] P[row, key]
// Its result layout gives a lane, for its own column, four consecutive keys of
// each of several groups (16x16: keys 4 g .. 4 g + 3 with g = lane / 16; 32x32:
// 8 n + 4 h .. + 3 with h = lane / 32), and the operand layout of the second
// product wants eight keys of a lane's own column.  Since the order in which a
// product sums its keys is free, two such groups are eight keys: probabilities
// never leave their lane, if V^T is numbered the same way.  V^T comes from
// row-major fp16 rows in LDS by transposing reads, each of which gives a lane
// four keys of its dim.
#pragma once

#include "fp4_cache.h"

namespace mvme {
namespace fp4 {

typedef short s16x4 __attribute__((ext_vector_type(4)));

// Probabilities are exp2(x - reference) with the reference set 8 below the
// largest score, and moved when a score passes it by 14 (prefill looks when
// one passes fp16, at 16).  They are rounded to fp16 for the value product
// (half the products of fp32, and every value of the cache is exact in it):
// 11 bits from 2^-22 of the largest on, nothing below 2^-33 of it.  None
// overflows while scores (in log2) are below 2^24 in magnitude; beyond, a step
// of fp32 passes 1, and a weight can be as many powers of two off.  The
// accumulators and the sums that divide them are fp32, both of the
// probabilities as rounded: what a rounding adds, it adds to both.
constexpr float kRefBelow = 8.f;
constexpr float kRefSlack = 14.f;
constexpr float kRefNone = -3.0e38f;  // no score yet: below every finite one

constexpr int kTileKeys = 32;

// Byte address inside a tile of rows of 2 * D bytes.  16-byte chunks are XORed
// with a number of their row that puts these into different banks: one chunk of
// 16 consecutive rows (or of rows 0-3 and 12-15 and the chunk four on of rows
// 4-11: the order in which 16-byte accesses are served), and what 32 lanes of a
// transposing read take: two chunks of 8 consecutive rows (DIMS 16), or four of
// 4 rows (DIMS 32).  Rows whose length is a multiple of 256 bytes start in the
// same bank, of 128 bytes in one of two, of 64 bytes in one of four.
template <int D, int DIMS>
struct TileLayout {
    static constexpr int kChunks = D / 8;
    __device__ static inline constexpr int number(int row) {
        if (kChunks % 16 == 0) return DIMS == 16 ? 2 * (row & 7) | ((row >> 3) & 1) : 4 * (row & 3) | ((row >> 2) & 3);
        if (kChunks % 8 == 0)
            return DIMS == 16 ? 2 * ((row >> 1) & 3) | ((row >> 3) & 1) : 4 * ((row >> 1) & 1) | ((row >> 2) & 3);
        return DIMS == 16 ? 2 * ((row >> 2) & 1) | ((row >> 3) & 1) : (row >> 2) & 3;
    }
    __device__ static inline int at(int row, int chunk) { return row * 2 * D + ((chunk ^ number(row)) << 4); }
};

// A lane's place in a tile, for accesses at chunks `first + i` of its row.  For
// power-of-two rows the XOR of the layout acts on address bits of its own, so
// one register and an XOR with a constant give every address; `forget` keeps
// the compiler from holding them all in registers across a loop.
template <int D, int DIMS>
struct TileAddress {
    static constexpr bool kPow2 = (D & (D - 1)) == 0;
    int row, first, base;
    __device__ inline TileAddress(int row, int first, int bytes = 0) : row(row), first(first) {
        base = (kPow2 ? TileLayout<D, DIMS>::at(row, first) : row * 2 * D) + bytes;
    }
    __device__ inline void forget() { asm volatile("" : "+v"(base)); }
    // Chunk `first + i` (they have no bits in common) of the row, or of a row whose number is `flip` away.
    __device__ inline int chunk(int i, int flip = 0) const {
        if constexpr (kPow2) return base ^ ((i ^ flip) << 4);
        return base + (((first + i) ^ TileLayout<D, DIMS>::number(row) ^ flip) << 4);
    }
};

// Eight keys of a lane's dim for the value product, from two transposing reads.  For each, 16 lanes take four rows, the
// lane the 8 bytes lane % 4 of 16 dims in row lane % 16 / 4.
__device__ inline u32x4 value_operand(const uint8_t* tile, int first, int second) {
    typedef __attribute__((address_space(3))) s16x4* lds_ptr;
    const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(tile + first));
    const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(tile + second));
    const u32x2 x = __builtin_bit_cast(u32x2, a), y = __builtin_bit_cast(u32x2, b);
    return u32x4{x[0], x[1], y[0], y[1]};
}

}  // namespace fp4
}  // namespace mvme
