// The packed 4-bit cache (format: include/mvme_fp4.h) as the kernels see it:
// where a token's codes and scales are, the conversions, and the checks that
// every entry point makes of its geometry.
#pragma once

#include "../../include/mvme_fp4.h"
#include "mvme_common.h"

namespace mvme {
namespace fp4 {

constexpr int kBlockDims = 32;      // dims that share a scale
constexpr int64_t kMaxDim = 256;
constexpr int64_t kMaxCapacity = 1048576;  // tokens that one block table names

// Page of a token: token / block_size by a shift for powers of two, else by a
// product with the rounded-up reciprocal 2^32 / block_size and one correction
// (exact for tokens < 2^32: the product is at most one too large).
struct BlockDiv {
    uint32_t size, magic;
    int shift;  // >= 0: block_size = 1 << shift
    __device__ inline uint32_t page(uint32_t token) const {
        if (shift >= 0) return token >> shift;
        uint32_t q = __umulhi(token, magic);
        if (q * size > token) --q;
        return q;
    }
};

inline BlockDiv make_block_div(int64_t block_size) {
    BlockDiv d{(uint32_t)block_size, 0u, -1};
    if ((block_size & (block_size - 1)) == 0) {
        d.shift = 0;
        while ((int64_t(1) << d.shift) < block_size) ++d.shift;
    } else {
        d.magic = (uint32_t)(((uint64_t(1) << 32) + block_size - 1) / block_size);
    }
    return d;
}

inline int64_t record_bytes(int64_t block_size, int64_t head_dim) {
    return (block_size * (head_dim / 2 + head_dim / kBlockDims) + 15) / 16 * 16;
}

inline bool valid_format(int64_t block_size, int64_t head_dim) {
    return block_size > 0 && block_size <= kMaxCapacity && head_dim > 0 && head_dim <= kMaxDim &&
           head_dim % kBlockDims == 0;
}

// Head dims that the attention kernels are built for.
inline bool attention_dim(int64_t d) { return d == 32 || d == 64 || d == 96 || d == 128 || d == 192 || d == 256; }

// A load by all lanes from one address that no kernel writes meanwhile, through the scalar cache.
__device__ inline int64_t uniform_load(const int64_t* p) {
    return *(const __attribute__((address_space(4))) int64_t*)(uintptr_t)p;
}

// The f32 whose exponent is a scale byte (255: the conversions give NaN).
__device__ inline float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }

// Two values of byte SEL of `w`, times the scale: exact in both types.
template <typename T, int SEL>
__device__ inline uint32_t pair_of(uint32_t w, float scale) {
    if constexpr (T::kId == MVME_FP16)
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, SEL));
    else
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, SEL));
}
// The eight values of `w`, in order.
template <typename T>
__device__ inline u32x4 values_of(uint32_t w, float scale) {
    return u32x4{pair_of<T, 0>(w, scale), pair_of<T, 1>(w, scale), pair_of<T, 2>(w, scale), pair_of<T, 3>(w, scale)};
}

inline bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

}  // namespace fp4
}  // namespace mvme
