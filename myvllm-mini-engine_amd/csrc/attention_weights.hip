// Decode attention that adds the weight each cached token receives to an
// account: the narrow units of the shared-prefix walk, with their dot products
// kept until the divisor is known:  w[j] += sum_h 2^(x_hj - m_h) / s_h.
//
// Bound by the reads of keys and values.  Kept dot products (4 bytes per query
// head and key, against 4 D of the caches per kv head) are written to a workspace
// and read once more by the joining kernel; recomputing them would read the
// keys again, which is D / (4 group) times as much.  4 x 65536 tokens, 32 heads on
// 4 of 128: 537 MB of caches and 34 MB of scores each way in 119 us (104 in
// the walk, 5.1 TB/s, and 16 in the join); the stores of scores are 17 to 22 of
// the walk's.  Sequences whose scores fit a work-group's LDS are taken whole, with
// no second kernel, and the longest one's work-group ends last: 32 ragged ones of
// up to 4096 tokens take 64 us, the same tokens in 32 of one length 48.5 (5.6
// TB/s), 4096 in each 90 (6.0 TB/s), and one of 4096 among 31 of 64 alone 48.7.
#include "../../include/mvme_long.h"
#include "long_attention.h"

namespace mvme {
namespace lng {
namespace {

template <typename T, int D, int RUN>
__global__ __launch_bounds__(kThreads, D <= 128 ? 2 : 1) void weighted_decode_kernel(Args a) {
    __shared__ __attribute__((aligned(16))) NarrowLds<D, kStoreScores> lds;
    Walk w;
    w.count(a);
    const int wg = blockIdx.x;
    if (wg >= w.shares) return;
    const int first = w.first_of(wg), stop = w.first_of(wg + 1);
#pragma unroll 1
    for (int at = first; at < stop;) {
        const Segment s = find_segment(a, w, wg, at, stop);
        at += s.rounds;
        narrow_segment<T, D, RUN, kStoreScores>(a, s, lds);
    }
}

// A sequence's query heads of one kv head, whole: no walk, no workspace and no second kernel.
template <typename T, int D, int RUN>
__global__ __launch_bounds__(kThreads, D <= 128 ? 2 : 1) void weighted_whole_kernel(Args a) {
    __shared__ __attribute__((aligned(16))) NarrowLds<D, kAddWeights> lds;
    Segment s{};
    s.seq = blockIdx.x / a.kv_heads;
    s.kv_head = blockIdx.x - s.seq * a.kv_heads;
    s.first_row = -1;
    s.rows = a.group;
    s.end = (uint32_t)uniform(Walk::length_from(a, uniform_load(a.lens + s.seq)));
    s.slot = -1;
    narrow_segment<T, D, RUN, kAddWeights>(a, s, lds);
}

constexpr int kAddKeys = 4 * kThreads;  // keys whose weights a work-group adds up
constexpr int kHeads = 8;               // heads whose scores are in flight

// Joins the pieces, and adds weights: work-groups 0 .. batch * kv_heads - 1 do the first, the others take kAddKeys keys of
// one sequence and kv head each, four in a row per thread.
template <typename T, int D>
__global__ __launch_bounds__(kThreads) void weighted_join_kernel(Args a, int blocks) {
    const int units = a.batch * a.kv_heads;
    if ((int)blockIdx.x < units) {
        join_heads<T, D>(a, blockIdx.x / a.kv_heads, blockIdx.x % a.kv_heads);
        return;
    }
    const int item = blockIdx.x - units, block = item % blocks, unit = item / blocks;
    const int seq = unit / a.kv_heads, kv_head = unit % a.kv_heads;
    const int len = Walk::length_from(a, a.lens[seq]);
    if (block * kAddKeys >= len) return;
    __shared__ float stats[kHeads][2];  // (reference, 1 / sum) of the heads at hand
    const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int64_t head0 = (int64_t)seq * a.q_heads + kv_head * a.group;
    const int key = block * kAddKeys + 4 * threadIdx.x;
    float* out = a.weights + ((int64_t)seq * a.kv_heads + kv_head) * a.weight_row + key;
    // The scores do not wait for the divisors.  (Keys behind the context are read where there are some, and not used.)
    const f32x4* scores = reinterpret_cast<const f32x4*>(a.scores) +
                          ((int64_t)unit * (a.score_row / 4) + (key < len ? key / 4 : 0)) * a.group;
    f32x4 s[kHeads];
    const auto load = [&](int h0) {
#pragma unroll
        for (int i = 0; i < kHeads; ++i)
            s[i] = scores[min(h0 + i, a.group - 1)];
    };
    load(0);
    float before[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) before[i] = key + i < len ? out[i] : 0.f;
    Join j;
    j.find(a, seq, kv_head);
    f32x4 add = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
    for (int h0 = 0; h0 < a.group; h0 += kHeads) {
        if (h0) load(h0);
        __syncthreads();
        for (int h = wave; h < kHeads; h += kWaves) {
            float ref = kRefNone, sum = 0.f;
            Pieces p;
            if (h0 + h >= a.group) {
            } else if (j.pieces(a, h0 + h, p)) {
                for (int i = lane; i < p.count; i += kWave) {
                    const float* of;
                    p.at(a, i, D, of);
                    const float top = fmaxf(ref, of[0]);
                    sum = sum * fast_exp2(ref - top) + of[1] * fast_exp2(of[0] - top);
                    ref = top;
                }
                float top = ref;
#pragma unroll
                for (int m = 1; m < kWave; m *= 2) top = fmaxf(top, shfl_xor(top, m));
                sum = group_sum<kWave>(sum * fast_exp2(ref - top));
                ref = top;
            } else {
                ref = a.totals[(head0 + h0 + h) * 2];
                sum = a.totals[(head0 + h0 + h) * 2 + 1];
            }
            if (lane == 0) {
                stats[h][0] = ref;
                stats[h][1] = sum != 0.f ? 1.f / sum : 0.f;
            }
        }
        __syncthreads();
#pragma unroll
        for (int h = 0; h < kHeads; ++h)
            if (h0 + h < a.group) {
                const float ref = stats[h][0], by = stats[h][1];
#pragma unroll
                for (int i = 0; i < 4; ++i) add[i] += probability(a, s[h][i], ref, by);
            }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (key + i < len) out[i] = before[i] + add[i];
}

int work_groups(int64_t head_dim) { return head_dim <= 128 ? 512 : 256; }

// Whether sequences are taken whole: their scores fit the ring, and they are short or nearly fill the chip.  Whole against
// split, us, 16 heads on 8: 1 x 512 tokens 9.2 and 11.0, 1 x 1024 14.4 and 11.9, 8 x 1024 16.3 and 15.7, 32 x 1024 25.0
// and 32.6, 64 x 4096 177 and 199; 32 heads on 4: 1 x 1024 15.3 and 13.8, 16 x 1024 17.6 and 19.2.
bool whole(int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t capacity) {
    const int64_t group = q_heads / kv_heads;
    if (group > kColumns || capacity > kRound * (kRing / (8 * group))) return false;
    return capacity <= 512 || batch * kv_heads >= 128;
}

// Whether one launch holds the join's work-groups: one per sequence and kv head, and one for each kAddKeys keys of theirs.
int64_t add_blocks(int64_t block_size, int64_t width) { return (block_size * width - 1) / kAddKeys + 1; }
bool fits_launch(int64_t batch, int64_t kv_heads, int64_t block_size, int64_t width) {
    return batch * kv_heads <= kMostThreads / kThreads / (1 + add_blocks(block_size, width));
}

struct Sizes {
    int64_t shares, slots, score_row;
    int64_t floats;
};
Sizes sizes(int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t block_size, int64_t width) {
    Sizes s{};
    if (whole(batch, q_heads, kv_heads, block_size * width)) return s;
    s.shares = work_groups(head_dim);
    s.slots = kv_heads * batch * ((q_heads / kv_heads - 1) / kColumns + 1) + s.shares;
    s.score_row = (block_size * width + 31) / 32 * 32;
    s.floats = s.slots * kColumns * (head_dim + 2) + batch * q_heads * (2 + s.score_row) + 4;
    return s;
}

template <typename T, int D>
int launch(const Args& a, int blocks, hipStream_t s) {
    const dim3 grid((unsigned)a.shares), block(kThreads), units((unsigned)(a.batch * a.kv_heads));
    if (a.shares == 0) {
        if (a.div.size % 16 == 0) hipLaunchKernelGGL((weighted_whole_kernel<T, D, 16>), units, block, 0, s, a);
        else hipLaunchKernelGGL((weighted_whole_kernel<T, D, 1>), units, block, 0, s, a);
        return check_launch("weighted attention");
    }
    if (a.div.size % 16 == 0) hipLaunchKernelGGL((weighted_decode_kernel<T, D, 16>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((weighted_decode_kernel<T, D, 1>), grid, block, 0, s, a);
    if (int rc = check_launch("weighted attention")) return rc;
    hipLaunchKernelGGL((weighted_join_kernel<T, D>), dim3((unsigned)(a.batch * a.kv_heads * (1 + blocks))), block, 0, s, a, blocks);
    return check_launch("weighted join");
}

template <typename T>
int launch_dim(const Args& a, int64_t head_dim, int blocks, hipStream_t s) {
    switch (head_dim) {
        case 16: return launch<T, 16>(a, blocks, s);
        case 32: return launch<T, 32>(a, blocks, s);
        case 64: return launch<T, 64>(a, blocks, s);
        case 80: return launch<T, 80>(a, blocks, s);
        case 96: return launch<T, 96>(a, blocks, s);
        case 128: return launch<T, 128>(a, blocks, s);
        case 192: return launch<T, 192>(a, blocks, s);
        default: return launch<T, 256>(a, blocks, s);
    }
}

}  // namespace
}  // namespace lng
}  // namespace mvme

using namespace mvme;
using namespace mvme::lng;

extern "C" size_t mvme_paged_attention_weights_workspace_size(int64_t batch, int64_t q_heads, int64_t kv_heads,
                                                              int64_t head_dim, int64_t block_size, int64_t table_width) {
    Args a{};
    if (check_shape(a, batch, q_heads, kv_heads, head_dim, 1, block_size, table_width, MVME_FP16) ||
        !fits_launch(batch, kv_heads, block_size, table_width))
        return 0;
    return (size_t)sizes(batch, q_heads, kv_heads, head_dim, block_size, table_width).floats * sizeof(float);
}

extern "C" int mvme_paged_attention_weights(void* out, const void* query, const void* key_cache, const void* value_cache,
                                            const int64_t* block_tables, const int64_t* context_lens, float* weights,
                                            int64_t weight_row, int64_t batch, int64_t q_heads, int64_t kv_heads,
                                            int64_t head_dim, int64_t num_blocks, int64_t block_size,
                                            int64_t table_width, int dtype, void* workspace, size_t workspace_bytes,
                                            void* stream) {
    Args a{};
    if (int rc = check_shape(a, batch, q_heads, kv_heads, head_dim, num_blocks, block_size, table_width, dtype)) return rc;
    if (weight_row < block_size * table_width) return fail(MVME_EINVAL, "weight rows must hold the tables' capacity");
    if (!out || !query || !key_cache || !value_cache || !block_tables || !context_lens || !weights)
        return fail(MVME_EINVAL, "weighted attention: null pointer");
    if (!fp4::aligned(query, 16) || !fp4::aligned(key_cache, 16) || !fp4::aligned(value_cache, 16) || !fp4::aligned(out, 8) ||
        !fp4::aligned(weights, 4))
        return fail(MVME_EINVAL, "weighted attention: queries and caches must be 16-byte, the output 8-byte aligned");
    const Sizes s = sizes(batch, q_heads, kv_heads, head_dim, block_size, table_width);
    const int64_t blocks = add_blocks(block_size, table_width);
    if (!fits_launch(batch, kv_heads, block_size, table_width)) return fail(MVME_EINVAL, "batch/head product too large");
    if (s.floats > 0 && (!workspace || workspace_bytes < (size_t)s.floats * sizeof(float) || !fp4::aligned(workspace, 16)))
        return fail(MVME_EWORKSPACE, "weighted attention workspace too small: " + std::to_string(s.floats * 4) +
                                         " bytes, 16-byte aligned, are needed");
    a.out = out;
    a.query = query;
    a.key = static_cast<const uint8_t*>(key_cache);
    a.value = static_cast<const uint8_t*>(value_cache);
    a.tables = block_tables;
    a.lens = context_lens;
    a.shares = (int)s.shares;
    a.narrow_slots = s.slots;
    a.weights = weights;
    a.weight_row = weight_row;
    a.score_row = s.score_row;
    a.scores = static_cast<float*>(workspace);
    a.narrow = a.scores + batch * q_heads * s.score_row;
    a.totals = a.narrow + s.slots * kColumns * (head_dim + 2);
    hipStream_t st = static_cast<hipStream_t>(stream);
    return dtype == MVME_FP16 ? launch_dim<Half>(a, head_dim, (int)blocks, st) : launch_dim<BFloat16>(a, head_dim, (int)blocks, st);
}
