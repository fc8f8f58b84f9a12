// Writing rows into the packed 4-bit cache and reading them back.
//
// Both move bytes: a token and kv head is head_dim 16-bit values on one side
// and head_dim * 17 / 32 bytes on the other.  A lane owns 8 consecutive dims:
// one 16-byte access of the 16-bit row, one 4-byte access of the codes, so
// that 16 lanes cover a head of 128.  The four lanes of a 32-dim block find
// its largest magnitude with two quad exchanges on the bit patterns (integer
// order is magnitude order, with NaN above infinity).
//
// Bound by those bytes for many rows, by a launch and the chain from slot to
// store for few: 16384 tokens of 8 heads of 128 written and read back in 37.6
// us (152 MB: 4.05 TB/s, a large copy reaches 4.76), 32 tokens in 5.1 us, each
// two calls back to back in a graph (from Python 40.5 and 9.5).
#include "fp4_cache.h"

namespace mvme {
namespace fp4 {
namespace {

constexpr int kThreads = 256;
// Pieces of eight dims per lane: two, whose loads are in flight together, where there are more than the chip's lanes take at
// once, else one (16384 tokens: 39.7 us with one, 37.6 with two, 38.3 with four; 32 tokens: 5.1, 5.7 and 7.3).
constexpr uint32_t kManyLanes = 256 * 2048;

enum SlotMode { kSlots = 0, kBatch = 1, kRange = 2 };

struct RowArgs {
    uint8_t* cache[2];       // keys, values
    uint8_t* rows[2];        // 16-bit rows
    const int64_t* index;    // slots | block tables | block ids
    const int64_t* offsets;  // position per row (batch mode)
    int64_t row_stride[2];   // bytes between 16-bit rows
    int64_t num_blocks, block_size, index_width;
    int64_t record;
    int kv_heads, dim, chunks;  // chunks = dim / 8
    uint32_t lanes;             // tokens * kv_heads * chunks
};

// Page and place of row `t`; false where the metadata names none.
template <int MODE>
__device__ inline bool locate(const RowArgs& a, uint32_t t, int64_t& page, int64_t& place) {
    int64_t pos;
    if constexpr (MODE == kSlots)
        pos = a.index[t];
    else
        pos = MODE == kBatch ? a.offsets[t] : (int64_t)t;
    if (pos < 0) return false;
    int64_t block;
    if ((pos | a.block_size) >> 32) {
        block = pos / a.block_size;
        place = pos % a.block_size;
    } else {  // the common case, without a 64-bit division
        const uint32_t p = (uint32_t)pos, s = (uint32_t)a.block_size, q = p / s;
        block = q;
        place = p - q * s;
    }
    if constexpr (MODE == kSlots) {
        page = block;
    } else {
        if (block >= a.index_width) return false;
        page = a.index[MODE == kBatch ? (int64_t)t * a.index_width + block : block];
    }
    return page >= 0 && page < a.num_blocks;
}

struct Place {
    uint32_t t;
    int head, chunk;
};
__device__ inline Place place_of(const RowArgs& a, uint32_t i) {
    const uint32_t row = i / (uint32_t)a.chunks;
    Place p;
    p.chunk = (int)(i - row * (uint32_t)a.chunks);
    p.t = row / (uint32_t)a.kv_heads;
    p.head = (int)(row - p.t * (uint32_t)a.kv_heads);
    return p;
}

template <bool VEC16>
__device__ inline u32x4 load_row(const uint8_t* p) {
    if constexpr (VEC16) return *reinterpret_cast<const u32x4*>(p);
    const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = (uint32_t)h[2 * i] | (uint32_t)h[2 * i + 1] << 16;
    return w;
}

// The scale byte for a block whose largest magnitude has the 16-bit pattern `bits`.
template <typename T>
__device__ inline uint32_t scale_byte(uint32_t bits) {
    constexpr uint32_t kInf = T::kId == MVME_FP16 ? 0x7c00u : 0x7f80u;
    if (bits > kInf) return 255u;
    const uint32_t f = __float_as_uint(T::lo(bits));
    // f = 1.mantissa * 2^(e - 127): 4 * 1.mantissa <= 7 fits 2^(e - 129).
    const int e = (int)(f >> 23) - 2 + ((f & 0x7fffffu) > 0x600000u ? 1 : 0);
    return (uint32_t)min(max(e, 127 - 23), 127 + 13);
}

template <typename T, int SEL>
__device__ inline uint32_t codes_into(uint32_t w, uint32_t pair, float scale) {
    if constexpr (T::kId == MVME_FP16)
        return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, __builtin_bit_cast(f16x2, pair), scale, SEL);
    else
        return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf16x2, pair), scale, SEL);
}

template <typename T, int MODE, bool VEC16, int PIECES>
__global__ __launch_bounds__(kThreads) void fp4_write_kernel(RowArgs a) {
    const uint32_t first = blockIdx.x * (kThreads * PIECES) + threadIdx.x;
    const int plane = blockIdx.y;
    Place p[PIECES];
    u32x4 rows[PIECES];
    int64_t page[PIECES], place[PIECES];
    bool there[PIECES];
#pragma unroll
    for (int n = 0; n < PIECES; ++n) {
        // Whole quads are behind the end together: lanes is a multiple of 4.
        const uint32_t i = first + n * kThreads;
        p[n] = place_of(a, min(i, a.lanes - 1));
        // (The row is loaded beside its slot, and for nothing where that does not exist.)
        rows[n] = load_row<VEC16>(a.rows[plane] + p[n].t * a.row_stride[plane] + (p[n].head * a.dim + p[n].chunk * 8) * 2);
        there[n] = locate<MODE>(a, p[n].t, page[n], place[n]) && i < a.lanes;
    }
#pragma unroll
    for (int n = 0; n < PIECES; ++n) {
        if (!there[n]) continue;
        const u32x4 x = rows[n];
        uint32_t most = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) most = max(most, max(x[k] & 0x7fffu, (x[k] >> 16) & 0x7fffu));
        most = max(most, quad_swap<kDppQuadSwap1>(most));
        most = max(most, quad_swap<kDppQuadSwap2>(most));
        const uint32_t byte = scale_byte<T>(most);
        const float scale = scale_of(byte);
        uint32_t w = 0;
        if (byte != 255u) {
            w = codes_into<T, 0>(w, x[0], scale);
            w = codes_into<T, 1>(w, x[1], scale);
            w = codes_into<T, 2>(w, x[2], scale);
            w = codes_into<T, 3>(w, x[3], scale);
        }
        uint8_t* record = a.cache[plane] + (page[n] * a.kv_heads + p[n].head) * a.record;
        *reinterpret_cast<uint32_t*>(record + place[n] * (a.dim / 2) + p[n].chunk * 4) = w;
        if ((p[n].chunk & 3) == 0)
            record[a.block_size * (a.dim / 2) + place[n] * (a.dim / kBlockDims) + p[n].chunk / 4] = (uint8_t)byte;
    }
}

template <typename T, int MODE, bool VEC16, int PIECES>
__global__ __launch_bounds__(kThreads) void fp4_gather_kernel(RowArgs a) {
    const uint32_t first = blockIdx.x * (kThreads * PIECES) + threadIdx.x;
    const int plane = blockIdx.y;
    Place p[PIECES];
    bool there[PIECES];
    uint32_t codes[PIECES], byte[PIECES];
#pragma unroll
    for (int n = 0; n < PIECES; ++n) {
        p[n] = place_of(a, min(first + n * kThreads, a.lanes - 1));
        int64_t page, place;
        there[n] = locate<MODE>(a, p[n].t, page, place);
        const uint8_t* record = a.cache[plane] + ((there[n] ? page : 0) * a.kv_heads + p[n].head) * a.record;
        if (!there[n]) place = 0;
        codes[n] = *reinterpret_cast<const uint32_t*>(record + place * (a.dim / 2) + p[n].chunk * 4);
        byte[n] = record[a.block_size * (a.dim / 2) + place * (a.dim / kBlockDims) + p[n].chunk / 4];
    }
#pragma unroll
    for (int n = 0; n < PIECES; ++n) {
        if (first + n * kThreads >= a.lanes) return;
        u32x4 x = {0u, 0u, 0u, 0u};
        if (there[n]) x = values_of<T>(codes[n], scale_of(byte[n]));
        uint8_t* to = a.rows[plane] + p[n].t * a.row_stride[plane] + (p[n].head * a.dim + p[n].chunk * 8) * 2;
        if constexpr (VEC16) {
            *reinterpret_cast<u32x4*>(to) = x;
        } else {
            uint16_t* h = reinterpret_cast<uint16_t*>(to);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                h[2 * k] = (uint16_t)x[k];
                h[2 * k + 1] = (uint16_t)(x[k] >> 16);
            }
        }
    }
}

int check(RowArgs& a, const void* key_cache, const void* value_cache, const void* key, const void* value,
          int64_t num_blocks, int64_t block_size, int64_t kv_heads, int64_t head_dim, const int64_t* index,
          int64_t tokens, int64_t key_stride, int64_t value_stride, int dtype) {
    if (num_blocks <= 0 || kv_heads <= 0) return fail(MVME_EINVAL, "KV cache dimensions must be positive");
    if (!valid_format(block_size, head_dim))
        return fail(MVME_EINVAL, "packed KV cache requires head_dim a multiple of 32 up to 256 and block_size up to 1M");
    if (!valid_dtype(dtype)) return fail(MVME_EINVAL, "packed KV rows require FP16/BF16");
    const int64_t row = head_dim * kv_heads;
    if (kv_heads > (int64_t(1) << 24) / head_dim) return fail(MVME_EINVAL, "KV row (kv_heads*head_dim) too large");
    if (num_blocks > (int64_t(1) << 62) / (block_size * row)) return fail(MVME_EINVAL, "KV cache too large");
    // One lane per 8 dims, 256 a work-group, all lanes numbered in 32 bits.
    if (tokens < 0 || tokens > (int64_t(1) << 31) / (row / 8)) return fail(MVME_EINVAL, "too many packed KV rows");
    if (tokens == 0) return MVME_OK;
    if (!key_cache || !value_cache || !index || !key || !value)
        return fail(MVME_EINVAL, "packed KV rows: null pointer");
    if (!aligned(key_cache, 16) || !aligned(value_cache, 16))
        return fail(MVME_EINVAL, "packed KV caches must be 16-byte aligned");
    if (!aligned(key, 2) || !aligned(value, 2)) return fail(MVME_EINVAL, "packed KV rows must be 2-byte aligned");
    if (tokens > 1 && (key_stride < row || value_stride < row))
        return fail(MVME_EINVAL, "packed key/value token stride smaller than a KV row");
    a.cache[0] = static_cast<uint8_t*>(const_cast<void*>(key_cache));
    a.cache[1] = static_cast<uint8_t*>(const_cast<void*>(value_cache));
    a.rows[0] = static_cast<uint8_t*>(const_cast<void*>(key));
    a.rows[1] = static_cast<uint8_t*>(const_cast<void*>(value));
    a.index = index;
    a.row_stride[0] = key_stride * 2;
    a.row_stride[1] = value_stride * 2;
    a.num_blocks = num_blocks;
    a.block_size = block_size;
    a.record = record_bytes(block_size, head_dim);
    a.kv_heads = (int)kv_heads;
    a.dim = (int)head_dim;
    a.chunks = (int)head_dim / 8;
    a.lanes = (uint32_t)(tokens * (row / 8));
    return MVME_OK;
}

bool vector_rows(const RowArgs& a) {
    return aligned(a.rows[0], 16) && aligned(a.rows[1], 16) && a.row_stride[0] % 16 == 0 && a.row_stride[1] % 16 == 0;
}

template <int MODE, int PIECES>
int launch_write_pieces(const RowArgs& a, int dtype, void* stream) {
    const dim3 grid((a.lanes - 1) / (kThreads * PIECES) + 1, 2), block(kThreads);
    hipStream_t s = static_cast<hipStream_t>(stream);
    const bool vec = vector_rows(a);
    if (dtype == MVME_FP16) {
        if (vec) hipLaunchKernelGGL((fp4_write_kernel<Half, MODE, true, PIECES>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((fp4_write_kernel<Half, MODE, false, PIECES>), grid, block, 0, s, a);
    } else {
        if (vec) hipLaunchKernelGGL((fp4_write_kernel<BFloat16, MODE, true, PIECES>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((fp4_write_kernel<BFloat16, MODE, false, PIECES>), grid, block, 0, s, a);
    }
    return check_launch("packed KV write");
}
template <int MODE>
int launch_write(const RowArgs& a, int dtype, void* stream) {
    if (a.lanes == 0) return MVME_OK;
    return a.lanes > kManyLanes ? launch_write_pieces<MODE, 2>(a, dtype, stream)
                                : launch_write_pieces<MODE, 1>(a, dtype, stream);
}

template <int MODE, int PIECES>
int launch_gather_pieces(const RowArgs& a, int dtype, void* stream) {
    const dim3 grid((a.lanes - 1) / (kThreads * PIECES) + 1, 2), block(kThreads);
    hipStream_t s = static_cast<hipStream_t>(stream);
    const bool vec = vector_rows(a);
    if (dtype == MVME_FP16) {
        if (vec) hipLaunchKernelGGL((fp4_gather_kernel<Half, MODE, true, PIECES>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((fp4_gather_kernel<Half, MODE, false, PIECES>), grid, block, 0, s, a);
    } else {
        if (vec) hipLaunchKernelGGL((fp4_gather_kernel<BFloat16, MODE, true, PIECES>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((fp4_gather_kernel<BFloat16, MODE, false, PIECES>), grid, block, 0, s, a);
    }
    return check_launch("packed KV gather");
}
template <int MODE>
int launch_gather(const RowArgs& a, int dtype, void* stream) {
    if (a.lanes == 0) return MVME_OK;
    return a.lanes > kManyLanes ? launch_gather_pieces<MODE, 2>(a, dtype, stream)
                                : launch_gather_pieces<MODE, 1>(a, dtype, stream);
}

}  // namespace
}  // namespace fp4
}  // namespace mvme

using namespace mvme;
using namespace mvme::fp4;

extern "C" int64_t mvme_fp4_record_bytes(int64_t block_size, int64_t head_dim) {
    return valid_format(block_size, head_dim) ? record_bytes(block_size, head_dim) : 0;
}

extern "C" int mvme_fp4_write_slots(void* key_cache, void* value_cache, int64_t num_blocks, int64_t block_size,
                                    int64_t kv_heads, int64_t head_dim, const int64_t* slot_mapping,
                                    const void* key, const void* value, int64_t tokens, int64_t key_token_stride,
                                    int64_t value_token_stride, int dtype, void* stream) {
    RowArgs a{};
    if (int rc = check(a, key_cache, value_cache, key, value, num_blocks, block_size, kv_heads, head_dim,
                       slot_mapping, tokens, key_token_stride, value_token_stride, dtype))
        return rc;
    return launch_write<kSlots>(a, dtype, stream);
}

extern "C" int mvme_fp4_write_batch(void* key_cache, void* value_cache, int64_t num_blocks, int64_t block_size,
                                    int64_t kv_heads, int64_t head_dim, const int64_t* block_tables,
                                    int64_t table_width, const int64_t* token_offsets, const void* key,
                                    const void* value, int64_t batch, int64_t key_token_stride,
                                    int64_t value_token_stride, int dtype, void* stream) {
    RowArgs a{};
    if (int rc = check(a, key_cache, value_cache, key, value, num_blocks, block_size, kv_heads, head_dim,
                       block_tables, batch, key_token_stride, value_token_stride, dtype))
        return rc;
    if (table_width <= 0) return fail(MVME_EINVAL, "batch table shape mismatch");
    if (batch == 0) return MVME_OK;
    if (!token_offsets) return fail(MVME_EINVAL, "packed KV rows: null pointer");
    a.offsets = token_offsets;
    a.index_width = table_width;
    return launch_write<kBatch>(a, dtype, stream);
}

extern "C" int mvme_fp4_gather_slots(void* key_out, void* value_out, const void* key_cache, const void* value_cache,
                                     int64_t num_blocks, int64_t block_size, int64_t kv_heads, int64_t head_dim,
                                     const int64_t* slot_mapping, int64_t tokens, int dtype, void* stream) {
    RowArgs a{};
    const int64_t row = kv_heads * head_dim;
    if (int rc = check(a, key_cache, value_cache, key_out, value_out, num_blocks, block_size, kv_heads, head_dim,
                       slot_mapping, tokens, row, row, dtype))
        return rc;
    return launch_gather<kSlots>(a, dtype, stream);
}

extern "C" int mvme_fp4_gather(void* key_out, void* value_out, const void* key_cache, const void* value_cache,
                               int64_t num_blocks, int64_t block_size, int64_t kv_heads, int64_t head_dim,
                               const int64_t* block_ids, int64_t num_ids, int64_t token_count, int dtype,
                               void* stream) {
    RowArgs a{};
    const int64_t row = kv_heads * head_dim;
    if (int rc = check(a, key_cache, value_cache, key_out, value_out, num_blocks, block_size, kv_heads, head_dim,
                       block_ids, token_count, row, row, dtype))
        return rc;
    if (num_ids < 0 || (token_count > 0 && num_ids < (token_count - 1) / block_size + 1))
        return fail(MVME_EINVAL, "token_count exceeds supplied block table capacity");
    a.index_width = num_ids;
    return launch_gather<kRange>(a, dtype, stream);
}
