// Decode attention for batches whose sequences share prefixes: each prefix is
// read once for all query heads of its group, and every row's own keys once.
//
// Softmax sums over disjoint sets of keys join: with references m_i, sums s_i
// and outputs o_i = sum_j 2^(x_j - m_i) v_j, out = sum_i 2^(m_i - m) o_i /
// sum_i 2^(m_i - m) s_i.  So a group's prefix is attended by all its rows at
// once, each row's own keys by its heads alone, and both are cut where the
// shares end.
//
// Bounds: with few rows per key the reads (16 sequences over 1024 shared
// tokens and 64 in all, 401 MB: 77 us, of which the join is 5; 5.5 TB/s in
// the walk), with many the wide loop.  128 sequences, 32 heads on 8, over 16384
// tokens and up to 400 of their own take 82.6 us, and 72 with one token of their
// own.  Of these the prefix's keys are 45 (what 32768 more of them add, halved;
// 764 TFLOP/s, and 30 us at the rate of a large matrix product); the other 27
// do not grow with them: the join (10), two launches, what begins and ends a
// segment, and those last tokens.  In the loop a wave's tile of 32 rows and 64
// keys of 128 dims takes a SIMD about 3400 cycles (at 2.4 GHz).  By count 1024
// are matrix products and about 900 vector work, half of that exponentials, and
// the work-group's four tiles keep the LDS busy for 1250: together about what a
// tile takes, so little of it overlaps between the two waves of a SIMD.  128 rows a
// work-group are what two work-groups' registers and LDS allow; three per
// compute unit, or the next tile's scores beside this one's softmax, spill or
// were slower (88 against 85).
#include "../../include/mvme_long.h"
#include "long_attention.h"

namespace mvme {
namespace lng {
namespace {

template <typename T>
__device__ inline f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
    if constexpr (T::kId == MVME_FP16)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

template <int D>
struct WideLds {
    uint8_t tiles[2][2][Shape<D>::kWidePlane];  // [buffer][keys, values]
    uint8_t present[2][kWideKeys];              // which tokens of a tile are there,
    __attribute__((aligned(4))) uint8_t odd[2][4];  // where a wave's 16 are not all
};

// What a thread stages of a tile: 16-byte pieces 4 i + lane % 4 of one token's key and value.
template <int D>
struct Staged {
    u32x4 x[2][Shape<D>::kChunks];
    bool there;
};

// Largest weight (log2) before the reference moves: fp16 holds 65504.
constexpr float kLargest = 15.999f;

// One segment of a wide unit: 128 rows of a group, 32 per wave.  Scores are K * Q^T with 32 keys x 32 rows a product, so
// that a lane holds 32 scores of one row and its weights are at once the operand of V^T * P.
template <typename T, int D, int RUN>
__device__ inline void wide_segment(const Args& a, const Segment& seg, WideLds<D>& lds) {
    using S = Shape<D>;
    constexpr int P = S::kDim;
    const int lane = threadIdx.x & 63, column = lane & 31, h = lane >> 5;
    const int wave = uniform(threadIdx.x >> 6);
    const int64_t* table = a.tables + (int64_t)seg.seq * a.width;
    const int64_t head_at = (int64_t)seg.kv_head * (2 * D);
    // Staging: a wave has 16 consecutive tokens.  (Their order puts four that share a bank into one 16-byte access.)
    const int row = 16 * wave + 4 * ((lane >> 2) & 3) + (lane >> 4), quarter = lane & 3;
    const uint32_t looked = RUN == 16 ? 16 * wave : row;
    const auto page_of = [&](uint32_t t0) {
        const int64_t* entry = table + min(a.div.page(t0 + looked), (uint32_t)a.width - 1u);
        return RUN == 16 ? uniform_load(entry) : *entry;
    };
    uint32_t lane_at = (RUN == 16 ? (uint32_t)(row & 15) * a.row_bytes : 0u) + quarter * 16;
    const auto load = [&](Staged<D>& x, uint32_t t0, int64_t page) {
        const uint32_t token = t0 + looked;
        const bool found = token < seg.end && (uint64_t)page < (uint64_t)a.num_blocks;
        x.there = found && t0 + row < seg.end;
        const uint32_t place = found ? token - a.div.page(token) * a.div.size : 0u;
        const int64_t at = head_at + (int64_t)((uint64_t)(uint32_t)(found ? page : 0) * a.page_bytes) +
                           (int64_t)((uint64_t)place * a.row_bytes);
#pragma unroll
        for (int plane = 0; plane < 2; ++plane) {
            const uint8_t* base = (plane ? a.value : a.key) + at + lane_at;
#pragma unroll
            for (int i = 0; i < S::kChunks; ++i) {
                if (D == P || (4 * i + quarter) * 8 < D) x.x[plane][i] = *reinterpret_cast<const u32x4*>(base + 64 * i);
                else x.x[plane][i] = u32x4{0u, 0u, 0u, 0u};
            }
        }
    };
    TileAddress<P, 32> stage_at(row, quarter);
    const auto stage = [&](Staged<D>& x, int buffer) {
        const bool some = __any(!x.there);
        if (some) {
#pragma unroll
            for (int plane = 0; plane < 2; ++plane)
#pragma unroll
                for (int i = 0; i < S::kChunks; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) x.x[plane][i][j] = x.there ? x.x[plane][i][j] : 0u;
            if (quarter == 0) lds.present[buffer][row] = x.there;
        }
        if (lane == 0) lds.odd[buffer][wave] = some;
#pragma unroll
        for (int plane = 0; plane < 2; ++plane)
#pragma unroll
            for (int i = 0; i < S::kChunks; ++i)
                *reinterpret_cast<u32x4*>(lds.tiles[buffer][plane] + stage_at.chunk(4 * i)) = x.x[plane][i];
    };
    Staged<D> staged;
    load(staged, seg.begin, page_of(seg.begin));
    int64_t page = page_of(seg.begin + kWideKeys);

    const int in_tile = wave * 32 + column;
    const bool live = in_tile < seg.rows;
    const int64_t head = head_of(a, seg, live ? seg.tile * kWideRows + in_tile : 0);
    u32x4 q[S::kSteps];
#pragma unroll
    for (int i = 0; i < S::kSteps; ++i) {
        q[i] = u32x4{0u, 0u, 0u, 0u};
        if (live && (D == P || 16 * i + 8 * h < D))
            q[i] = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(a.query) + head * D + 16 * i + 8 * h);
    }
    f32x16 acc[S::kBlocks];
#pragma unroll
    for (int n = 0; n < S::kBlocks; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[n][i] = 0.f;
    float ref = kRefNone, sum = 0.f;
    TileAddress<P, 32> key_at(column, h);
    TileAddress<P, 32> value_at(4 * h + ((lane & 15) >> 2), 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1), (lane & 1) * 8);

    stage(staged, 0);
    load(staged, seg.begin + kWideKeys, page);
    page = page_of(seg.begin + 2 * kWideKeys);
    lds_barrier();
    int buffer = 0;
#pragma unroll 1
    for (uint32_t t0 = seg.begin; t0 < seg.end; t0 += kWideKeys, buffer ^= 1) {
        key_at.forget();
        value_at.forget();
        stage_at.forget();
        asm volatile("" : "+v"(lane_at));
        const uint8_t* keys = lds.tiles[buffer][0];
        const uint8_t* values = lds.tiles[buffer][1];
        f32x16 x[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
#pragma unroll
            for (int i = 0; i < 16; ++i) x[k][i] = 0.f;
#pragma unroll
            for (int i = 0; i < S::kSteps; ++i) {
                const u32x4 operand = *reinterpret_cast<const u32x4*>(keys + 32 * k * 2 * P + key_at.chunk(2 * i));
                x[k] = mfma32<T>(operand, q[i], x[k]);
            }
        }
        // The next tile (behind the last one: zeros) goes into the other buffer, and the one after it is loaded.
        stage(staged, buffer ^ 1);
        load(staged, t0 + 2 * kWideKeys, page);
        page = page_of(t0 + 3 * kWideKeys);
        const uint32_t odds = (uint32_t)uniform(*reinterpret_cast<const int*>(lds.odd[buffer]));
        if (odds) {
            const bool there = (odds >> (8 * (lane >> 4))) & 0xff ? lds.present[buffer][lane] : true;
            const uint64_t mask = __ballot(there);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const uint32_t bits = (uint32_t)(mask >> (32 * k)) >> (4 * h);
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (!((bits >> (8 * (i >> 2) + (i & 3))) & 1)) x[k][i] = kNegInf;
            }
        }
        float top = x[0][0];
#pragma unroll
        for (int i = 1; i < 32; ++i) top = fmaxf(top, x[i >> 4][i & 15]);
        if (__any(__builtin_fmaf(top, a.scale, -ref) > kLargest)) {
            top = pair32_max(top) * a.scale;
            const float moved = top > ref + kRefSlack ? top - kRefBelow : ref;
            const float by = fast_exp2(ref - moved);
            ref = moved;
            sum *= by;
#pragma unroll
            for (int n = 0; n < S::kBlocks; ++n) acc[n] *= by;
        }
        // Weights are rounded to the inputs' type for the value product, which is half of the matrix products here; the sum
        // that divides is of the rounded ones, so that what a rounding adds it adds to both.  As sums of two numbers, as
        // narrow units have them, 128 sequences over 16384 tokens take 98 us instead of 82, 20 over 4096 (16 heads) 24.8
        // instead of 22.0.  Errors against 64 bits then equal those of fp32 weights, 0.00166 (bf16, the output's rounding)
        // and 0.000207 (fp16); so they are 0.0023 and 0.00029.
        constexpr uint32_t kOnes = T::kId == MVME_FP16 ? 0x3c003c00u : 0x3f803f80u;
        u32x4 weights[4];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float p0 = fast_exp2(__builtin_fmaf(x[i >> 3][2 * (i & 7)], a.scale, -ref));
            const float p1 = fast_exp2(__builtin_fmaf(x[i >> 3][2 * (i & 7) + 1], a.scale, -ref));
            const uint32_t pair = T::pack(p0, p1);
            weights[i >> 2][i & 3] = pair;
            sum = T::dot2(pair, kOnes, sum);
        }
#pragma unroll
        for (int m = 0; m < 4; ++m)
#pragma unroll
            for (int n = 0; n < S::kBlocks; ++n) {
                // (Eight rows on, the row's number differs in bit 1.)
                const u32x4 operand = value_operand(values + 16 * m * 2 * P, value_at.chunk(4 * n), value_at.chunk(4 * n, 2) + 8 * 2 * P);
                acc[n] = mfma32<T>(operand, weights[m], acc[n]);
            }
        lds_barrier();
    }
    const float total = swap32_add(sum, sum);  // the other half of the keys is with the lane 32 away
    if (live && seg.slot < a.wide_slots) {
        const int64_t slot = (int64_t)seg.slot * kWideRows + in_tile;
#pragma unroll
        for (int n = 0; n < S::kBlocks; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int d = 32 * n + 8 * i + 4 * h;
                if (D == P || d < D)
                    *reinterpret_cast<f32x4*>(a.wide + slot * D + d) =
                        f32x4{acc[n][4 * i], acc[n][4 * i + 1], acc[n][4 * i + 2], acc[n][4 * i + 3]};
            }
        if (h == 0) {
            float* stats = a.wide + a.wide_slots * kWideRows * D + slot * 2;
            stats[0] = ref;
            stats[1] = total;
        }
    }
}

template <typename T, int D, int RUN>
__global__ __launch_bounds__(kThreads, D <= 128 ? 2 : 1) void shared_prefix_kernel(Args a) {
    __shared__ __attribute__((aligned(16))) union Lds {
        WideLds<D> wide;
        NarrowLds<D, kNoScores> narrow;
    } lds;
    Walk w;
    w.count(a);
    const int wg = w.mine();
    if (wg < 0) return;
    const int first = w.first_of(wg), stop = w.first_of(wg + 1);
#pragma unroll 1
    for (int at = first; at < stop;) {
        const Segment s = find_segment(a, w, wg, at, stop);
        at += s.rounds;
        if (s.wide) wide_segment<T, D, RUN>(a, s, lds.wide);
        else narrow_segment<T, D, RUN, kNoScores>(a, s, lds.narrow);
    }
}

template <typename T, int D>
__global__ __launch_bounds__(kThreads) void shared_prefix_join_kernel(Args a) {
    join_heads<T, D>(a, blockIdx.x / a.kv_heads, blockIdx.x % a.kv_heads);
}

int work_groups(int64_t head_dim) { return head_dim <= 128 ? 512 : 256; }

// Calls whose keys and values, each sequence's on its own, are this little are attended without regard to the groups: up
// to there reading a prefix again costs less than the pieces and their join.  Sequences of a prefix and 100 tokens more, 16
// heads on 8, alone and shared, us: 8 x 1024 9.7 and 14.3, 4 x 4096 (67 MB) 16.1 and 15.3, 16 x 1024 12.4 and 14.3, 32 x
// 1024 (134 MB) 17.7 and 18.0, 16 x 2048 17.4 and 16.0, 64 x 1024 (268 MB) 25.6 and 20.7.
constexpr int64_t kAloneBytes = 96 << 20;
bool alone(int64_t batch, int64_t kv_heads, int64_t head_dim, int64_t groups, int64_t capacity, int always) {
    if (always) return false;
    return groups == 0 || batch * capacity <= kAloneBytes / (kv_heads * head_dim * 4);
}

struct Sizes {
    int64_t shares, wide_slots, narrow_slots;
    size_t bytes;
};
Sizes sizes(int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t groups) {
    Sizes s{};
    const int64_t group = q_heads / kv_heads, tiles = (group + kColumns - 1) / kColumns;
    s.shares = work_groups(head_dim);
    // A unit's pieces are at most one more than the share boundaries in it.  Wide groups have more than 32 rows each, one
    // partial unit at most; narrow ones at least two sequences and at most two units.
    const int64_t wide = groups > 0 ? batch * group / kWideRows + std::min(groups, batch * group / (kNarrowRows + 1)) : 0;
    const int64_t narrow = groups > 0 ? 2 * std::min(groups, batch / 2) : 0;
    s.wide_slots = wide > 0 ? kv_heads * wide + s.shares : 0;
    s.narrow_slots = kv_heads * (narrow + batch * tiles) + s.shares;
    s.bytes = (size_t)(s.wide_slots * kWideRows + s.narrow_slots * kColumns) * (size_t)(head_dim + 2) * sizeof(float);
    return s;
}

template <typename T, int D>
int launch(const Args& a, hipStream_t s) {
    const dim3 grid((unsigned)a.shares), block(kThreads);
    if (a.div.size % 16 == 0) hipLaunchKernelGGL((shared_prefix_kernel<T, D, 16>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((shared_prefix_kernel<T, D, 1>), grid, block, 0, s, a);
    if (int rc = check_launch("shared-prefix attention")) return rc;
    hipLaunchKernelGGL((shared_prefix_join_kernel<T, D>), dim3((unsigned)(a.batch * a.kv_heads)), block, 0, s, a);
    return check_launch("shared-prefix join");
}

template <typename T>
int launch_dim(const Args& a, int64_t head_dim, hipStream_t s) {
    switch (head_dim) {
        case 16: return launch<T, 16>(a, s);
        case 32: return launch<T, 32>(a, s);
        case 64: return launch<T, 64>(a, s);
        case 80: return launch<T, 80>(a, s);
        case 96: return launch<T, 96>(a, s);
        case 128: return launch<T, 128>(a, s);
        case 192: return launch<T, 192>(a, s);
        default: return launch<T, 256>(a, s);
    }
}

}  // namespace
}  // namespace lng
}  // namespace mvme

using namespace mvme;
using namespace mvme::lng;

extern "C" size_t mvme_paged_attention_shared_prefix_workspace_size(int64_t batch, int64_t q_heads, int64_t kv_heads,
                                                                    int64_t head_dim, int64_t groups, int64_t block_size,
                                                                    int64_t table_width, int always) {
    Args a{};
    if (check_shape(a, batch, q_heads, kv_heads, head_dim, 1, block_size, table_width, MVME_FP16) || groups < 0 || groups > batch)
        return 0;
    if (alone(batch, kv_heads, head_dim, groups, block_size * table_width, always))
        return mvme_paged_attention_workspace_size(batch, q_heads, kv_heads, head_dim, block_size, table_width, 0);
    return sizes(batch, q_heads, kv_heads, head_dim, groups).bytes;
}

extern "C" int mvme_paged_attention_shared_prefix(void* out, const void* query, const void* key_cache,
                                                  const void* value_cache, const int64_t* block_tables,
                                                  const int64_t* context_lens, const int64_t* group_offsets,
                                                  const int64_t* prefix_lens, int64_t batch, int64_t groups,
                                                  int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                                                  int64_t num_blocks, int64_t block_size, int64_t table_width, int always,
                                                  int dtype, void* workspace, size_t workspace_bytes, void* stream) {
    Args a{};
    if (int rc = check_shape(a, batch, q_heads, kv_heads, head_dim, num_blocks, block_size, table_width, dtype)) return rc;
    if (groups < 0 || groups > batch) return fail(MVME_EINVAL, "groups must be between none and one per sequence");
    if (!out || !query || !key_cache || !value_cache || !block_tables || !context_lens || (groups > 0 && (!group_offsets || !prefix_lens)))
        return fail(MVME_EINVAL, "shared-prefix attention: null pointer");
    if (!fp4::aligned(query, 16) || !fp4::aligned(key_cache, 16) || !fp4::aligned(value_cache, 16) || !fp4::aligned(out, 8))
        return fail(MVME_EINVAL, "shared-prefix attention: queries and caches must be 16-byte, the output 8-byte aligned");
    if (alone(batch, kv_heads, head_dim, groups, block_size * table_width, always))
        return mvme_paged_attention(out, query, key_cache, value_cache, block_tables, context_lens, batch, q_heads, kv_heads,
                                    head_dim, num_blocks, block_size, table_width, 0, dtype, workspace, workspace_bytes, stream);
    const Sizes s = sizes(batch, q_heads, kv_heads, head_dim, groups);
    if (!workspace || workspace_bytes < s.bytes || !fp4::aligned(workspace, 16))
        return fail(MVME_EWORKSPACE, "shared-prefix workspace too small: " + std::to_string(s.bytes) +
                                         " bytes, 16-byte aligned, are needed");
    a.out = out;
    a.query = query;
    a.key = static_cast<const uint8_t*>(key_cache);
    a.value = static_cast<const uint8_t*>(value_cache);
    a.tables = block_tables;
    a.lens = context_lens;
    a.offsets = group_offsets;
    a.prefixes = prefix_lens;
    a.groups = (int)groups;
    a.shares = (int)s.shares;
    a.wide_slots = s.wide_slots;
    a.narrow_slots = s.narrow_slots;
    a.wide = static_cast<float*>(workspace);
    a.narrow = a.wide + s.wide_slots * kWideRows * (head_dim + 2);
    hipStream_t st = static_cast<hipStream_t>(stream);
    return dtype == MVME_FP16 ? launch_dim<Half>(a, head_dim, st) : launch_dim<BFloat16>(a, head_dim, st);
}
