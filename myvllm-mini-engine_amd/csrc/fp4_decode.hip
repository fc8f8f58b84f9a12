// Decode attention over packed 4-bit pages: one query token per sequence.
//
// A work-group owns one sequence, one kv head (16 of its query heads) and one
// partition of the keys; its waves take tiles of 32 keys in turn and keep
// their own maximum, sum and accumulators, joined through LDS at the end.
// Partitions of a split sequence are joined by a second kernel.
#include "fp4_attention.h"

namespace mvme {
namespace fp4 {
namespace {

struct DecodeArgs {
    void* out;
    const void* query;
    const uint8_t* key;
    const uint8_t* value;
    const int64_t* tables;
    const int64_t* lens;
    float* partial;  // [batch, q_heads, parts, D] accumulators, then [batch, q_heads, parts, 2] (reference, sum)
    int64_t num_blocks, record;
    int64_t stats;   // offset of the (reference, sum) pairs, in floats
    int kv_heads, group, q_heads, width;
    int head_tiles;  // ceil(group / 16)
    int parts, part_tokens;
    BlockDiv div;
    float scale;     // log2(e) / sqrt(D)
};

template <int D>
struct Shape {
    static constexpr int kWaves = D <= 128 ? 8 : 4;
    static constexpr int kChunks = D / 32;           // score products per 16 keys; dwords of codes per lane
    static constexpr int kPer = D % 128 == 0 ? 4 : D == 64 || D == 192 ? 2 : 1;  // chunks that share a scale
    static constexpr int kScales = kChunks / kPer;
    static constexpr int kDimTiles = D / 16;
    static constexpr int kTileBytes = kTileKeys * 2 * D;  // fp16 rows of a tile; as large as a wave's accumulators
    static constexpr int kMinWaves = D <= 128 ? 4 : 2;
};

template <int D>
struct Row {  // a lane's part of one token: D / 4 dims
    uint32_t codes[Shape<D>::kChunks];
    uint32_t scales[Shape<D>::kScales];
};

template <int D>
__device__ inline void load_row(Row<D>& x, const uint8_t* record, uint32_t place, uint32_t block, int g) {
    const uint8_t* codes = record + place * (D / 2) + g * (D / 8);
    const uint8_t* scales = record + block * (D / 2) + place * (D / kBlockDims);
    if constexpr (Shape<D>::kChunks % 4 == 0) {
#pragma unroll
        for (int i = 0; i < Shape<D>::kChunks; i += 4) {
            const u32x4 w = *reinterpret_cast<const u32x4*>(codes + 4 * i);
#pragma unroll
            for (int j = 0; j < 4; ++j) x.codes[i + j] = w[j];
        }
    } else if constexpr (Shape<D>::kChunks % 2 == 0) {
#pragma unroll
        for (int i = 0; i < Shape<D>::kChunks; i += 2) {
            const u32x2 w = *reinterpret_cast<const u32x2*>(codes + 4 * i);
            x.codes[i] = w[0];
            x.codes[i + 1] = w[1];
        }
    } else {
#pragma unroll
        for (int i = 0; i < Shape<D>::kChunks; ++i) x.codes[i] = reinterpret_cast<const uint32_t*>(codes)[i];
    }
#pragma unroll
    for (int i = 0; i < Shape<D>::kScales; ++i)
        x.scales[i] = scales[(g * (D / 4) + 8 * i * Shape<D>::kPer) / kBlockDims];
}

template <int D>
__device__ inline void zero_row(Row<D>& x) {
#pragma unroll
    for (int i = 0; i < Shape<D>::kChunks; ++i) x.codes[i] = 0u;
#pragma unroll
    for (int i = 0; i < Shape<D>::kScales; ++i) x.scales[i] = 127u;
}

template <typename T, int D>
__global__ __launch_bounds__(64 * Shape<D>::kWaves, Shape<D>::kMinWaves) void fp4_decode_kernel(DecodeArgs a) {
    using S = Shape<D>;
    __shared__ __attribute__((aligned(16))) uint8_t tiles[S::kWaves][S::kTileBytes];
    __shared__ float stats[S::kWaves][2][16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
    const int part = blockIdx.x % a.parts, unit = blockIdx.x / a.parts;
    const int tile = unit % a.head_tiles, kv_head = unit / a.head_tiles % a.kv_heads;
    const int b = unit / a.head_tiles / a.kv_heads;
    const int64_t len = a.lens[b];
    const int heads = min(16, a.group - tile * 16);
    const int64_t first_head = (int64_t)b * a.q_heads + kv_head * a.group + tile * 16;
    const bool usable = len > 0 && len <= (int64_t)a.width * a.div.size;
    const uint32_t begin = (uint32_t)part * a.part_tokens;
    const uint32_t end = usable ? min((uint32_t)len, begin + (uint32_t)a.part_tokens) : 0u;
    if (begin >= end && (part > 0 || a.parts > 1)) return;  // no partial; an empty sequence is written by the merge

    // Query operand: head r, dims g * D / 4 + 8 c .. + 7, the order in which a lane's codes lie.
    u32x4 q[S::kChunks];
#pragma unroll
    for (int c = 0; c < S::kChunks; ++c) {
        q[c] = u32x4{0u, 0u, 0u, 0u};
        if (r < heads)
            q[c] = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(a.query) + (first_head + r) * D +
                                                   g * (D / 4) + 8 * c);
    }
    f32x4 acc[S::kDimTiles];
#pragma unroll
    for (int n = 0; n < S::kDimTiles; ++n) acc[n] = f32x4{0.f, 0.f, 0.f, 0.f};
    float ref = kRefNone, sum = 0.f;
    uint8_t* tile_lds = tiles[wave];
    const int64_t* table = a.tables + (int64_t)b * a.width;

    for (uint32_t t0 = begin + wave * kTileKeys; t0 < end; t0 += S::kWaves * kTileKeys) {
        Row<D> k[2], v[2];
        uint32_t present[2];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const uint32_t token = t0 + 16 * s + r;
            bool there = token < end;
            if (there) {
                const uint32_t block = a.div.page(token);
                const int64_t page = table[block];
                there = page >= 0 && page < a.num_blocks;
                if (there) {
                    const int64_t at = (page * a.kv_heads + kv_head) * a.record;
                    load_row<D>(k[s], a.key + at, token - block * a.div.size, a.div.size, g);
                    load_row<D>(v[s], a.value + at, token - block * a.div.size, a.div.size, g);
                }
            }
            if (!there) {
                zero_row<D>(k[s]);
                zero_row<D>(v[s]);
            }
            present[s] = (uint32_t)(__ballot(there) & 0xffffu);
        }
        // Scores.
        float x[8];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            f32x4 c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < S::kChunks; ++i)
                c = T::mfma16x16x32(values_of<T>(k[s].codes[i], scale_of(k[s].scales[i / S::kPer])), q[i], c);
#pragma unroll
            for (int j = 0; j < 4; ++j) x[4 * s + j] = (present[s] >> (4 * g + j)) & 1 ? c[j] * a.scale : kNegInf;
        }
        // Values to LDS in fp16, row-major.
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int i = 0; i < S::kChunks; ++i)
                *reinterpret_cast<u32x4*>(tile_lds + TileLayout<D>::at(16 * s + r, g * S::kChunks + i)) =
                    values_of<Half>(v[s].codes[i], scale_of(v[s].scales[i / S::kPer]));
        // Reference and probabilities.
        float top = x[0];
#pragma unroll
        for (int j = 1; j < 8; ++j) top = fmaxf(top, x[j]);
        top = row4_max(top);
        if (__any(top > ref + kRefSlack)) {
            const float moved = top > ref + kRefSlack ? top - kRefBelow : ref;
            const float by = fast_exp2(ref - moved);
            ref = moved;
            sum *= by;
#pragma unroll
            for (int n = 0; n < S::kDimTiles; ++n) acc[n] *= by;
        }
        float p[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            p[j] = fast_exp2(x[j] - ref);
            sum += p[j];
        }
        const u32x4 weights = {Half::pack(p[0], p[1]), Half::pack(p[2], p[3]), Half::pack(p[4], p[5]),
                               Half::pack(p[6], p[7])};
        // A wave reads only what it wrote: the LDS queue is in order, no barrier.
#pragma unroll
        for (int n = 0; n < S::kDimTiles; ++n) {
            const u32x4 vt = value_operand<D>(tile_lds, n, 0);
            acc[n] = Half::mfma16x16x32(vt, weights, acc[n]);
        }
    }
    sum = row4_sum(sum);

    // Join the waves: accumulators [16][D] in the tiles' LDS, each wave relative to its own reference.
    __syncthreads();
    float* mine = reinterpret_cast<float*>(tiles[wave]);
    if (r < heads) {
#pragma unroll
        for (int n = 0; n < S::kDimTiles; ++n) *reinterpret_cast<f32x4*>(mine + r * D + 16 * n + 4 * g) = acc[n];
        if (g == 0) {
            stats[wave][0][r] = ref;
            stats[wave][1][r] = sum;
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < heads * D; i += 64 * S::kWaves) {
        const int h = i / D, d = i - h * D;
        float top = stats[0][0][h];
#pragma unroll
        for (int w = 1; w < S::kWaves; ++w) top = fmaxf(top, stats[w][0][h]);
        float total = 0.f, value = 0.f;
#pragma unroll
        for (int w = 0; w < S::kWaves; ++w) {
            const float by = fast_exp2(stats[w][0][h] - top);
            total += by * stats[w][1][h];
            value += by * reinterpret_cast<const float*>(tiles[w])[i];
        }
        const int64_t head = first_head + h;
        if (a.parts == 1) {
            static_cast<uint16_t*>(a.out)[head * D + d] = T::from_float(total != 0.f ? value / total : 0.f);
        } else {
            a.partial[(head * a.parts + part) * D + d] = value;
            if (d == 0) {
                a.partial[a.stats + (head * a.parts + part) * 2] = top;
                a.partial[a.stats + (head * a.parts + part) * 2 + 1] = total;
            }
        }
    }
}

// Joins the partitions of one (sequence, query head).
template <typename T, int D>
__global__ __launch_bounds__(D < 64 ? 64 : D) void fp4_merge_kernel(DecodeArgs a) {
    const int64_t head = blockIdx.x;
    const int64_t b = head / a.q_heads;
    const int64_t len = a.lens[b];
    const bool usable = len > 0 && len <= (int64_t)a.width * a.div.size;
    const int parts = usable ? ((uint32_t)len - 1) / (uint32_t)a.part_tokens + 1 : 0;
    const float* stats = a.partial + a.stats + head * a.parts * 2;
    const float* partial = a.partial + head * a.parts * D;
    const int d = threadIdx.x;
    if (d >= D) return;
    float top = kRefNone;
    for (int p = 0; p < parts; ++p) top = fmaxf(top, stats[2 * p]);
    float total = 0.f, value = 0.f;
    for (int p = 0; p < parts; ++p) {
        const float by = fast_exp2(stats[2 * p] - top);
        total += by * stats[2 * p + 1];
        value += by * partial[(int64_t)p * D + d];
    }
    static_cast<uint16_t*>(a.out)[head * D + d] = T::from_float(total != 0.f ? value / total : 0.f);
}

struct Plan {
    int64_t parts, part_tokens;
};

bool attention_dim(int64_t d) { return d == 32 || d == 64 || d == 96 || d == 128 || d == 192 || d == 256; }

bool decode_shape(int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t block_size,
                  int64_t width) {
    return batch > 0 && q_heads > 0 && kv_heads > 0 && q_heads % kv_heads == 0 && attention_dim(head_dim) &&
           valid_format(block_size, head_dim) && width > 0 && width <= kMaxCapacity / block_size &&
           batch <= 2147483647 / q_heads;
}

// Partitions from shapes alone (lengths stay on the device).
Plan plan(int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t block_size, int64_t width,
          int64_t partition_tokens) {
    const int64_t capacity = block_size * width;
    const int64_t round = head_dim <= 128 ? 256 : 128;  // one tile for each wave
    const int64_t units = batch * kv_heads * ((q_heads / kv_heads + 15) / 16);
    int64_t tokens;
    if (partition_tokens > 0) {
        tokens = (partition_tokens + kTileKeys - 1) / kTileKeys * kTileKeys;
    } else {
        const int64_t want = units >= 1024 ? 1 : (1024 + units - 1) / units;  // two rounds of two work-groups per CU
        tokens = ((capacity + want - 1) / want + round - 1) / round * round;
    }
    if (tokens > capacity) tokens = (capacity + kTileKeys - 1) / kTileKeys * kTileKeys;
    return {(capacity - 1) / tokens + 1, tokens};
}

template <typename T, int D>
int launch(const DecodeArgs& a, int64_t units, int64_t heads, hipStream_t s) {
    hipLaunchKernelGGL((fp4_decode_kernel<T, D>), dim3((unsigned)(units * a.parts)), dim3(64 * Shape<D>::kWaves), 0, s,
                       a);
    if (int rc = check_launch("packed decode")) return rc;
    if (a.parts == 1) return MVME_OK;
    hipLaunchKernelGGL((fp4_merge_kernel<T, D>), dim3((unsigned)heads), dim3(D < 64 ? 64 : D), 0, s, a);
    return check_launch("packed decode merge");
}

template <typename T>
int launch_dim(const DecodeArgs& a, int64_t head_dim, int64_t units, int64_t heads, hipStream_t s) {
    switch (head_dim) {
        case 32: return launch<T, 32>(a, units, heads, s);
        case 64: return launch<T, 64>(a, units, heads, s);
        case 96: return launch<T, 96>(a, units, heads, s);
        case 128: return launch<T, 128>(a, units, heads, s);
        case 192: return launch<T, 192>(a, units, heads, s);
        default: return launch<T, 256>(a, units, heads, s);
    }
}

}  // namespace
}  // namespace fp4
}  // namespace mvme

using namespace mvme;
using namespace mvme::fp4;

extern "C" size_t mvme_fp4_paged_attention_workspace_size(int64_t batch, int64_t q_heads, int64_t kv_heads,
                                                          int64_t head_dim, int64_t block_size, int64_t table_width,
                                                          int64_t partition_tokens) {
    if (!decode_shape(batch, q_heads, kv_heads, head_dim, block_size, table_width)) return 0;
    const Plan p = plan(batch, q_heads, kv_heads, head_dim, block_size, table_width, partition_tokens);
    return p.parts == 1 ? 0 : (size_t)(batch * q_heads * p.parts) * (size_t)(head_dim + 2) * sizeof(float);
}

extern "C" int mvme_fp4_paged_attention(void* out, const void* query, const void* key_cache, const void* value_cache,
                                        const int64_t* block_tables, const int64_t* context_lens, int64_t batch,
                                        int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t num_blocks,
                                        int64_t block_size, int64_t table_width, int64_t partition_tokens, int dtype,
                                        void* workspace, size_t workspace_bytes, void* stream) {
    if (!valid_dtype(dtype)) return fail(MVME_EINVAL, "FP16/BF16 required");
    if (batch <= 0 || q_heads <= 0 || kv_heads <= 0 || num_blocks <= 0)
        return fail(MVME_EINVAL, "empty batch/heads/cache");
    if (q_heads % kv_heads != 0) return fail(MVME_EINVAL, "head dimension or GQA mismatch");
    if (!attention_dim(head_dim)) return fail(MVME_EINVAL, "supported head_dim: 32,64,96,128,192,256");
    if (block_size <= 0 || table_width <= 0) return fail(MVME_EINVAL, "invalid block table");
    if (block_size > kMaxCapacity || table_width > kMaxCapacity / block_size)
        return fail(MVME_EINVAL, "maximum table capacity is 1M tokens");
    if (!decode_shape(batch, q_heads, kv_heads, head_dim, block_size, table_width))
        return fail(MVME_EINVAL, "batch/head product too large");
    const int64_t record = record_bytes(block_size, head_dim);
    if (num_blocks > (int64_t(1) << 62) / record / kv_heads) return fail(MVME_EINVAL, "KV cache too large");
    if (!out || !query || !key_cache || !value_cache || !block_tables || !context_lens)
        return fail(MVME_EINVAL, "packed decode: null pointer");
    if (!aligned(query, 16) || !aligned(key_cache, 16) || !aligned(value_cache, 16) || !aligned(out, 2))
        return fail(MVME_EINVAL, "packed decode: query and caches must be 16-byte aligned");
    if (partition_tokens < 0) return fail(MVME_EINVAL, "partition_tokens must not be negative");
    const Plan p = plan(batch, q_heads, kv_heads, head_dim, block_size, table_width, partition_tokens);
    const int64_t tiles = (q_heads / kv_heads + 15) / 16, units = batch * kv_heads * tiles;
    if (p.parts > 2147483647 / units) return fail(MVME_EINVAL, "too many partitions");
    const size_t need = mvme_fp4_paged_attention_workspace_size(batch, q_heads, kv_heads, head_dim, block_size,
                                                                table_width, partition_tokens);
    if (need > 0 && (!workspace || workspace_bytes < need || !aligned(workspace, 16)))
        return fail(MVME_EWORKSPACE, "packed decode workspace too small: " + std::to_string(need) +
                                         " bytes, 16-byte aligned, are needed");
    DecodeArgs a{};
    a.out = out;
    a.query = query;
    a.key = static_cast<const uint8_t*>(key_cache);
    a.value = static_cast<const uint8_t*>(value_cache);
    a.tables = block_tables;
    a.lens = context_lens;
    a.partial = static_cast<float*>(workspace);
    a.num_blocks = num_blocks;
    a.record = record;
    a.stats = batch * q_heads * p.parts * head_dim;
    a.kv_heads = (int)kv_heads;
    a.q_heads = (int)q_heads;
    a.group = (int)(q_heads / kv_heads);
    a.width = (int)table_width;
    a.head_tiles = (int)tiles;
    a.parts = (int)p.parts;
    a.part_tokens = (int)p.part_tokens;
    a.div = make_block_div(block_size);
    a.scale = kLog2e / __builtin_sqrtf((float)head_dim);
    hipStream_t s = static_cast<hipStream_t>(stream);
    return dtype == MVME_FP16 ? launch_dim<Half>(a, head_dim, units, batch * q_heads, s)
                              : launch_dim<BFloat16>(a, head_dim, units, batch * q_heads, s);
}
