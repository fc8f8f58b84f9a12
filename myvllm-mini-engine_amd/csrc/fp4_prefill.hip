// Ragged chunked prefill over packed 4-bit pages.
//
// The query rows of one sequence and kv head are its (token, head of the
// group) pairs, numbered token-major, so that any group size fills the tiles.
// A work-group takes 128 of them, 32 per wave, and one chunk of the keys.
// Tiles of 64 keys are unpacked once into LDS (keys in the query's type,
// values in fp16) and used by all rows: scores are K * Q^T, so that a lane
// holds 32 scores of one row and the softmax needs no exchange, and the
// weights are at once the operand of V^T * P.  Chunks of split calls are
// joined by a second kernel.
//
// Per tile a wave has 1024 cycles of products (128 dims), as many of vector
// work (exponentials, conversions, unpacking) and a quarter of 1300 cycles of
// LDS traffic: none alone bounds it, so the loop mixes them: the next tile is
// unpacked between the score products, and the weights of 16 keys are made
// between the value products of the 16 before.  By the counters the matrix pipe
// works for 0.445 and the vector unit for 0.50 of the SIMDs' cycles, 0.95
// together: mostly one of them at a time still.  8192 tokens, 16 heads on 8, no
// prior keys: 269-274 us, 1.0 PFLOP/s of visible pairs (a large library product
// reaches 1.40; 331 us with the scores of the next tile beside the softmax of
// this one instead, 281 us with neither); 2 x 4096 tokens 142-146 us; 8 x 128
// behind up to 4096 keys 48 us, of which the tile loop is 33.  (Calls back to
// back.)
#include <algorithm>
#include <cmath>

#include "fp4_attention.h"

namespace mvme {
namespace fp4 {
namespace {

constexpr int kThreads = 256;
constexpr int kRows = 128;   // query rows of a work-group
constexpr int kKeys = 64;    // keys of a tile

struct PrefillArgs {
    void* out;
    const void* q;
    const uint8_t* key;
    const uint8_t* value;
    const int64_t* cu;
    const int64_t* starts;
    const int64_t* tables;
    const int64_t* lens;
    float* partial;  // [total_tokens, q_heads, chunks, D], then [total_tokens, q_heads, chunks, 2]
    int64_t stats;
    int32_t* counts; // [total_tokens, q_heads]: chunks that a row sees, -1 for rows that no sequence owns
    int64_t num_blocks, record, total_tokens;
    uint64_t page_bytes;
    int num_seqs, kv_heads, q_heads, group, width;
    int items;       // work-groups per kv head and chunk; the last one clears rows that no sequence owns
    int chunks, chunk_len;
    BlockDiv div, group_div;
    float scale;     // log2(e) / sqrt(D)
};

template <int D>
struct Shape {
    static constexpr int kChunks = D / 32;
    static constexpr int kPer = D % 128 == 0 ? 4 : D == 64 || D == 192 ? 2 : 1;
    static constexpr int kScales = kChunks / kPer;
    static constexpr int kBlocks = D / 32;   // 32-dim blocks of the output
    static constexpr int kSteps = D / 16;    // score products per 32 keys
    static constexpr int kMinWaves = D <= 128 ? 2 : 1;
};

typedef float f32x16 __attribute__((ext_vector_type(16)));
template <typename T>
__device__ inline f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
    if constexpr (T::kId == MVME_FP16)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

struct Seq {
    int64_t row0, rows, start, len;
};
__device__ inline Seq sequence(const PrefillArgs& a, int s) {
    const int64_t lo = min(max(a.cu[s], (int64_t)0), a.total_tokens);
    const int64_t hi = min(max(a.cu[s + 1], lo), a.total_tokens);
    return {lo, hi - lo, a.starts[s], a.lens[s]};
}
// Keys that a sequence's rows may see: none where its start or length cannot be.
__device__ inline int64_t usable_keys(const PrefillArgs& a, const Seq& q) {
    const int64_t capacity = (int64_t)a.width * a.div.size;
    return q.start < 0 || q.start >= q.len || q.len > capacity ? 0 : q.len;
}

template <typename T, int D>
__device__ inline void store4(const PrefillArgs& a, int64_t head, int d, f32x4 v) {
    u32x2 w = {T::pack(v[0], v[1]), T::pack(v[2], v[3])};
    *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(a.out) + head * D + d) = w;
}

// Rows before the first and behind the last sequence: zeros.  Meant for few of them: one work-group per kv head, two bytes
// at a time (1024 rows, 16 heads of 128: 31 us; padded to 4096 rows: 563 us).
template <int D>
__device__ void clear_rows(const PrefillArgs& a, int kv_head) {
    const int64_t first = min(max(a.cu[0], (int64_t)0), a.total_tokens);
    const int64_t last = min(max(a.cu[a.num_seqs], first), a.total_tokens);
    const int64_t width = (int64_t)a.group * D;
    const int64_t count = (first + a.total_tokens - last) * width;
    for (int64_t i = threadIdx.x; i < count; i += kThreads) {
        const int64_t n = i / width, token = n < first ? n : last + n - first;
        static_cast<uint16_t*>(a.out)[(token * a.q_heads + (int64_t)kv_head * a.group) * D + i % width] = 0;
        if (a.chunks > 1 && i % D == 0) a.counts[token * a.q_heads + (int64_t)kv_head * a.group + i % width / D] = -1;
    }
}

// What a thread unpacks of a tile: one quarter of one token's key and value.
template <int D>
struct Staged {
    uint32_t codes[2][Shape<D>::kChunks];
    uint32_t scales[2][Shape<D>::kScales];
    bool there;
};

constexpr float kLargest = 15.999f;  // log2 of a weight that fp16 holds (65519 is the last to round down)
// Whether no score of the tile gives a weight past fp16 against the reference (a NaN does not count).
__device__ inline bool weights_fit(const f32x16 (&x)[2], float scale, float ref) {
    float top = x[0][0];
#pragma unroll
    for (int i = 1; i < 31; i += 2) top = fmaxf(fmaxf(top, x[i >> 4][i & 15]), x[(i + 1) >> 4][(i + 1) & 15]);
    top = fmaxf(top, x[1][15]);
    return __builtin_fmaf(top, scale, -ref) <= kLargest;
}
// Moves the reference to the scores; sum and accumulators follow.
template <int BLOCKS>
__device__ inline void move_reference(const f32x16 (&x)[2], float scale, float& ref, float& sum, f32x16 (&acc)[BLOCKS]) {
    float top = x[0][0];
#pragma unroll
    for (int i = 0; i < 32; ++i) top = fmaxf(top, x[i >> 4][i & 15]);
    top = pair32_max(top) * scale;
    const float moved = top > ref + kRefSlack ? top - kRefBelow : ref;
    const float by = fast_exp2(ref - moved);
    ref = moved;
    sum *= by;
#pragma unroll
    for (int n = 0; n < BLOCKS; ++n) acc[n] *= by;
}
// Pair i of a tile's scores becomes weights, as operands of four products, and adds to the sum as rounded.
__device__ inline void weigh(const f32x16 (&x)[2], int i, u32x4 (&weights)[4], float& sum, float scale, float ref) {
    const float p0 = fast_exp2(__builtin_fmaf(x[i >> 3][2 * (i & 7)], scale, -ref));
    const float p1 = fast_exp2(__builtin_fmaf(x[i >> 3][2 * (i & 7) + 1], scale, -ref));
    const uint32_t pair = Half::pack(p0, p1);
    weights[i >> 2][i & 3] = pair;
    sum = Half::dot2(pair, 0x3c003c00u, sum);
}

// Barrier of the work-group for LDS alone: loads from memory stay in flight.
__device__ inline void lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// Which of the lanes' row blocks, counted through, is `item`: its lane, and `item` from that lane's first.  -1: behind all.
__device__ inline int find_lane(int blocks, int& item) {
    const int scan = wave_incl_scan(blocks);
    const uint64_t behind = __ballot(scan > item);
    if (!behind) return -1;
    const int at = __builtin_ctzll(behind);
    item -= __builtin_amdgcn_readlane(scan - blocks, at);
    return at;
}
__device__ inline int row_blocks(const PrefillArgs& a, int s) {
    const int64_t lo = min(max(a.cu[s], (int64_t)0), a.total_tokens);
    const int64_t hi = min(max(a.cu[s + 1], lo), a.total_tokens);
    return (int)(((hi - lo) * a.group + kRows - 1) / kRows);
}
// The sequence s and its row block that `item` becomes, from sequence to sequence; a sequence's blocks from the last,
// which sees most keys.  False behind all blocks.
__device__ inline bool find_in_order(const PrefillArgs& a, int lane, int& item, int& s) {
    for (s = 0; s < a.num_seqs; s += 64) {
        const int blocks = s + lane < a.num_seqs ? row_blocks(a, s + lane) : 0;
        const int at = find_lane(blocks, item);
        if (at >= 0) {
            s += at;
            item = __builtin_amdgcn_readlane(blocks, at) - 1 - item;
            return true;
        }
        item -= __builtin_amdgcn_readlane(wave_incl_scan(blocks), 63);
    }
    return false;
}
// The same for up to 64 sequences with the blocks that see most keys first, to a tile: they take longest, and the short
// ones fill what the chip has free at the end (12 mixed sequences 42.5 us, in order 49.1; 32 x 256 tokens behind 4096 keys
// 188 and 240; equal blocks pay 1 us for the search).  One wave has a lane for each of 64 sequences; more go in order.
__device__ inline bool find_longest_first(const PrefillArgs& a, int lane, int& item, int& s) {
    const int own = min(lane, a.num_seqs - 1);
    const int blocks = lane < a.num_seqs ? row_blocks(a, own) : 0;
    const int start = (int)min(max(a.starts[own], (int64_t)0), kMaxCapacity);
    // Blocks of this lane's sequence that see keys at 64 * tile and behind; none at `top` (positions past the tables are
    // with the last tile before it).
    const int half = 1 << (31 - __builtin_clz((int)(a.width * a.div.size / kKeys) | 1)), top = 2 * half;
    const auto from = [&](int tile) {
        const uint64_t before = (uint64_t)(uint32_t)max(tile * kKeys - start, 0) * (uint32_t)a.group / kRows;
        return tile == top ? 0 : blocks - (int)min(before, (uint64_t)blocks);
    };
    const auto all = [&](int n) { return __builtin_amdgcn_readlane(wave_incl_scan(n), 63); };
    if (item >= all(blocks)) return false;
    int tile = 0;  // the last with more than `item` blocks
    for (int step = half; step > 0; step /= 2)
        if (all(from(tile + step)) > item) tile += step;
    const int longer = from(tile + 1), here = from(tile) - longer;
    item -= all(longer);
    s = find_lane(here, item);
    item = __builtin_amdgcn_readlane(blocks - longer, s) - 1 - item;
    return s >= 0;
}

template <typename T, int D, int RUN>
__global__ __launch_bounds__(kThreads, Shape<D>::kMinWaves) void fp4_prefill_kernel(PrefillArgs a) {
    using S = Shape<D>;
    constexpr int kPlane = kKeys * 2 * D;
    __shared__ __attribute__((aligned(16))) uint8_t tiles[2][2][kPlane];  // [buffer][keys, values]
    __shared__ uint8_t present[2][kKeys];       // 1: there, 2: there and its value has a NaN
    __shared__ __attribute__((aligned(4))) uint8_t odd[2][4];  // per wave's 16 tokens: whether any is not 1
    const int lane = threadIdx.x & 63, column = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int kv_head = blockIdx.x % a.kv_heads, chunk = blockIdx.x / a.kv_heads % a.chunks;
    int item = blockIdx.x / a.kv_heads / a.chunks;
    if (item == a.items - 1) {
        if (chunk == 0) clear_rows<D>(a, kv_head);
        return;
    }
    int s;
    if (!(a.num_seqs <= 64 ? find_longest_first(a, lane, item, s) : find_in_order(a, lane, item, s))) return;
    const Seq seq = sequence(a, s);
    const int64_t usable = usable_keys(a, seq);
    // (Rows are counted in 32 bits: all tokens' query heads are below 2^31.)
    const uint32_t row0 = (uint32_t)item * kRows, rows = (uint32_t)seq.rows * a.group;
    // Keys of this work-group: up to the last row's position, in its chunk.
    const uint32_t last_token = a.group_div.page(min(row0 + kRows, rows) - 1);
    const int64_t first_pos = seq.start + a.group_div.page(row0);
    const uint32_t key_end = (uint32_t)min(usable, max(seq.start + last_token + 1, (int64_t)0));
    const uint32_t begin = (uint32_t)chunk * a.chunk_len;
    const uint32_t end = min(key_end, begin + (uint32_t)a.chunk_len);
    if (chunk > 0 && begin >= end) return;

    // Staging: thread -> token `row` of a tile, quarter `quarter` of its dims; a wave has 16 consecutive tokens.  RUN 16
    // (block sizes that are multiples of 16): they lie in one page at consecutive places, looked up once per wave.
    // Codes are loaded a tile ahead of their unpacking, and pages another tile ahead of that.
    const int64_t* table = a.tables + (int64_t)s * a.width;
    // (The order of the tokens in a wave puts four that share a bank into one 16-byte access: TileLayout.)
    const int row = 16 * wave + 4 * ((lane >> 2) & 3) + (lane >> 4), quarter = lane & 3;
    const uint32_t looked = RUN == 16 ? 16 * wave : row;  // the token of the tile that is looked up
    const auto page_of = [&](uint32_t t0) {
        const int64_t* entry = table + min(a.div.page(t0 + looked), (uint32_t)a.width - 1u);
        return RUN == 16 ? uniform_load(entry) : *entry;
    };
    uint32_t code_at = (RUN == 16 ? (row & 15) * (D / 2) : 0) + quarter * (D / 8);
    uint32_t scale_at[S::kScales];
#pragma unroll
    for (int i = 0; i < S::kScales; ++i)
        scale_at[i] = (RUN == 16 ? (row & 15) * (D / kBlockDims) : 0) + (quarter * (D / 4) + 8 * i * S::kPer) / kBlockDims;
    const auto load = [&](Staged<D>& x, uint32_t t0, int64_t page) {
        const uint32_t token = t0 + looked;
        const bool found = token < end && (uint64_t)page < (uint64_t)a.num_blocks;
        x.there = found && t0 + row < end;
        const uint32_t place = found ? token - a.div.page(token) * a.div.size : 0u;
        const int64_t at = kv_head * a.record + (int64_t)((uint64_t)(uint32_t)(found ? page : 0) * a.page_bytes) + place * (D / 2);
        const uint32_t to_scales = a.div.size * (D / 2) - place * (D / 2 - D / kBlockDims);
#pragma unroll
        for (int plane = 0; plane < 2; ++plane) {
            const uint8_t* base = (plane ? a.value : a.key) + at;
            const uint8_t* from = base + code_at;
            if constexpr (S::kChunks % 4 == 0) {
#pragma unroll
                for (int i = 0; i < S::kChunks; i += 4) {
                    const u32x4 w = *reinterpret_cast<const u32x4*>(from + 4 * i);
#pragma unroll
                    for (int j = 0; j < 4; ++j) x.codes[plane][i + j] = w[j];
                }
            } else {
#pragma unroll
                for (int i = 0; i < S::kChunks; ++i) x.codes[plane][i] = reinterpret_cast<const uint32_t*>(from)[i];
            }
#pragma unroll
            for (int i = 0; i < S::kScales; ++i) x.scales[plane][i] = base[scale_at[i] + to_scales];
        }
    };
    TileAddress<D, 32> stage_at(row, quarter * S::kChunks);
    const auto prepare = [&](Staged<D>& x, int buffer) {
        // A NaN block of the values must not reach rows that do not see its key, as 0 * NaN would: it is staged as
        // zeros, and the key's score is NaN instead.  Absent tokens are zeros.
        bool nan = false;
#pragma unroll
        for (int i = 0; i < S::kScales; ++i) nan |= x.scales[1][i] == 255u;
        const bool some = __any(!x.there || nan);
        if (some) {
            nan = (__ballot(nan) >> (lane & ~3)) & 15;
#pragma unroll
            for (int plane = 0; plane < 2; ++plane) {
                const bool keep = x.there && !(plane && nan);
#pragma unroll
                for (int i = 0; i < S::kChunks; ++i) x.codes[plane][i] = keep ? x.codes[plane][i] : 0u;
#pragma unroll
                for (int i = 0; i < S::kScales; ++i) x.scales[plane][i] = keep ? x.scales[plane][i] : 127u;
            }
            if (quarter == 0) present[buffer][row] = x.there ? nan ? 2 : 1 : 0;
        }
        if (lane == 0) odd[buffer][wave] = some;
    };
    const auto unpack = [&](const Staged<D>& x, int i, int buffer) {  // eight dims, of the key or behind all of it the value
        const int plane = i / S::kChunks, n = i % S::kChunks;
        const float scale = scale_of(x.scales[plane][n / S::kPer]);
        *reinterpret_cast<u32x4*>(tiles[buffer][plane] + stage_at.chunk(n)) =
            plane ? values_of<Half>(x.codes[plane][n], scale) : values_of<T>(x.codes[plane][n], scale);
    };
    Staged<D> staged;
    int64_t page = page_of(begin);
    load(staged, begin, page);
    page = page_of(begin + kKeys);

    // This lane's row.
    const uint32_t qrow = row0 + wave * 32 + column;
    const bool live = qrow < rows;
    const uint32_t token = live ? a.group_div.page(qrow) : 0u;
    const int32_t limit = live && seq.start + token < usable ? (int32_t)(seq.start + token) : -1;  // last visible key
    const int64_t head = (seq.row0 + token) * a.q_heads + (int64_t)kv_head * a.group + (live ? qrow - token * a.group : 0u);
    u32x4 q[S::kSteps];
#pragma unroll
    for (int i = 0; i < S::kSteps; ++i)
        q[i] = live ? *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(a.q) + head * D + 16 * i + 8 * h)
                    : u32x4{0u, 0u, 0u, 0u};
    f32x16 acc[S::kBlocks];
#pragma unroll
    for (int n = 0; n < S::kBlocks; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[n][i] = 0.f;
    float ref = kRefNone, sum = 0.f;
    TileAddress<D, 32> key_at(column, h);
    TileAddress<D, 32> value_at(4 * h + ((lane & 15) >> 2), 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1), (lane & 1) * 8);

    if (begin < end) {
        prepare(staged, 0);
#pragma unroll
        for (int i = 0; i < 2 * S::kChunks; ++i) unpack(staged, i, 0);
        load(staged, begin + kKeys, page);
        page = page_of(begin + 2 * kKeys);
        lds_barrier();
    }
    int buffer = 0;
#pragma unroll 1
    for (uint32_t t0 = begin; t0 < end; t0 += kKeys, buffer ^= 1) {
        key_at.forget();
        value_at.forget();
        stage_at.forget();
        asm volatile("" : "+v"(code_at));
#pragma unroll
        for (int i = 0; i < S::kScales; ++i) asm volatile("" : "+v"(scale_at[i]));
        const uint8_t* keys = tiles[buffer][0];
        const uint8_t* values = tiles[buffer][1];
        // The scores, and the next tile's unpacking (behind the last tile: of zeros) beside them.
        prepare(staged, buffer ^ 1);
        f32x16 x[2];
        {
            constexpr int kProducts = 2 * S::kSteps, kAhead = 4, kWords = 2 * S::kChunks;
            const auto operand_of = [&](int i) {
                return *reinterpret_cast<const u32x4*>(keys + 32 * (i / S::kSteps) * 2 * D + key_at.chunk(2 * (i % S::kSteps)));
            };
#pragma unroll
            for (int i = 0; i < 16; ++i) x[0][i] = x[1][i] = 0.f;
            u32x4 operand[kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; ++i) operand[i] = operand_of(i);
#pragma unroll
            for (int i = 0; i < kProducts; ++i) {
                x[i / S::kSteps] = mfma32<T>(operand[i % kAhead], q[i % S::kSteps], x[i / S::kSteps]);
                if (i + kAhead < kProducts) operand[i % kAhead] = operand_of(i + kAhead);
#pragma unroll
                for (int n = i * kWords / kProducts; n < (i + 1) * kWords / kProducts; ++n) unpack(staged, n, buffer ^ 1);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        if (t0 + kKeys < end) {
            load(staged, t0 + 2 * kKeys, page);
            page = page_of(t0 + 3 * kKeys);
        }
        const uint32_t odds = (uint32_t)__builtin_amdgcn_readfirstlane(*reinterpret_cast<const int*>(odd[buffer]));
        uint64_t mask = ~uint64_t(0);
        if (odds) {
            // (Only waves with something odd wrote their tokens' states.)
            const int state = (odds >> (8 * (lane >> 4))) & 0xff ? present[buffer][lane] : 1;
            mask = __ballot(state != 0);
            const uint64_t nans = __ballot(state == 2);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const uint32_t bits = (uint32_t)(nans >> (32 * k)) >> (4 * h);
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if ((bits >> (8 * (i >> 2) + (i & 3))) & 1) x[k][i] = __builtin_nanf("");
            }
        }
        if (mask != ~uint64_t(0) || (int64_t)t0 + kKeys - 1 > first_pos) {
            const int32_t seen = limit - (int32_t)t0 - 4 * h;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const uint32_t bits = (uint32_t)(mask >> (32 * k)) >> (4 * h);
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int key = 8 * (i >> 2) + (i & 3);
                    if (!((bits >> key) & 1) || 32 * k + key > seen) x[k][i] = kNegInf;
                }
            }
        }
        u32x4 weights[4];
        if (__any(!weights_fit(x, a.scale, ref))) move_reference(x, a.scale, ref, sum, acc);
        // Sixteen keys at a time: their weights are made beside the products of the sixteen before them.
        const auto operand_of = [&](int i) {  // sixteen keys i / kBlocks of 32 dims i % kBlocks
            // (Eight rows on, the row's number differs in bit 1.)
            const int n = i % S::kBlocks;
            return value_operand(values + 16 * (i / S::kBlocks) * 2 * D, value_at.chunk(4 * n),
                                 value_at.chunk(4 * n, 2) + 8 * 2 * D);
        };
        constexpr int kProducts = 4 * S::kBlocks, kAhead = kProducts < 4 ? kProducts : 4;
        u32x4 operand[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) operand[i] = operand_of(i);
#pragma unroll
        for (int j = 0; j < 4; ++j) weigh(x, j, weights, sum, a.scale, ref);
#pragma unroll
        for (int i = 0; i < kProducts; ++i) {
            const int m = i / S::kBlocks, n = i % S::kBlocks;
            acc[n] = mfma32<Half>(operand[i % kAhead], weights[m], acc[n]);
            if (i + kAhead < kProducts) operand[i % kAhead] = operand_of(i + kAhead);
            if (m < 3)
#pragma unroll
                for (int j = 4 * n / S::kBlocks; j < 4 * (n + 1) / S::kBlocks; ++j)
                    weigh(x, 4 * (m + 1) + j, weights, sum, a.scale, ref);
            __builtin_amdgcn_sched_barrier(0);
        }
        lds_barrier();
    }
    const float total = swap32_add(sum, sum);  // the other half of the keys is with the lane 32 away
    if (!live) return;
    const int64_t at = head * a.chunks + chunk;
    const float by = 1.f / total;
    const bool zero = limit < 0 || total == 0.f;  // a row that sees no key
#pragma unroll
    for (int n = 0; n < S::kBlocks; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f32x4 v = {acc[n][4 * i], acc[n][4 * i + 1], acc[n][4 * i + 2], acc[n][4 * i + 3]};
            const int d = 32 * n + 8 * i + 4 * h;
            if (a.chunks == 1) store4<T, D>(a, head, d, zero ? f32x4{0.f, 0.f, 0.f, 0.f} : v * by);
            else *reinterpret_cast<f32x4*>(a.partial + at * D + d) = v;
        }
    if (a.chunks > 1 && h == 0) {
        a.partial[a.stats + at * 2] = ref;
        a.partial[a.stats + at * 2 + 1] = total;
        // (Starts that cannot be make any limit of themselves, but leave no keys.)
        if (chunk == 0) a.counts[head] = limit < 0 || end == 0 ? 0 : limit / a.chunk_len + 1;
    }
}

template <int D>
constexpr int kMergeRows = kThreads / (D / 4);
// Joins the key chunks of packed rows and query heads: four dims per thread.
template <typename T, int D>
__global__ __launch_bounds__(kThreads) void fp4_prefill_merge_kernel(PrefillArgs a) {
    const int64_t head = (int64_t)blockIdx.x * kMergeRows<D> + threadIdx.x / (D / 4);
    const int d = threadIdx.x % (D / 4) * 4;
    if ((int)threadIdx.x >= kMergeRows<D> * (D / 4) || head >= a.total_tokens * a.q_heads) return;
    // (Bounded, for rows that nothing counted: offsets that fall name more row blocks than there are work-groups.)
    const int chunks = min(a.counts[head], a.chunks);
    if (chunks < 0) return;  // cleared by the first kernel
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    const f32x2* stats = reinterpret_cast<const f32x2*>(a.partial + a.stats) + head * a.chunks;
    const float* partial = a.partial + head * a.chunks * D + d;
    float top = kRefNone, total = 0.f;
    for (int c = 0; c < chunks; ++c) top = fmaxf(top, stats[c][0]);
    f32x4 value = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int c = 0; c < chunks; ++c) {
        const float by = fast_exp2(stats[c][0] - top);
        total += by * stats[c][1];
        value += by * *reinterpret_cast<const f32x4*>(partial + (int64_t)c * D);
    }
    store4<T, D>(a, head, d, total != 0.f ? value * (1.f / total) : f32x4{0.f, 0.f, 0.f, 0.f});
}

bool prefill_shape(int64_t num_seqs, int64_t total, int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                   int64_t block_size, int64_t width) {
    return num_seqs > 0 && num_seqs <= 2147483647 / 2 && total >= 0 && q_heads > 0 && kv_heads > 0 &&
           q_heads % kv_heads == 0 && attention_dim(head_dim) && valid_format(block_size, head_dim) && width > 0 &&
           width <= kMaxCapacity / block_size && q_heads <= 2147483647 / head_dim &&
           total <= 2147483647 / (q_heads);
}

struct Plan {
    int64_t items, chunks, chunk_len;
};

// Splits the keys where the row blocks are too few for the chip, by an estimate in microseconds.  A work-group with a
// compute unit to itself takes a tile in 1.00, 1.15, 1.45, 1.5, 2.5 and 3.1 us at 32, 64, 96, 128, 192 and 256 dims, two
// on one unit in 1.4 times as long each; from 192 dims on LDS holds one.  Joining takes a launch and its traffic.
// 8 x 128 tokens behind 4096 keys (128 dims): 48 us in four pieces, 99 us whole, 67 us in sixteen; two sequences of 2048
// tokens (256 dims): 239 us whole, 363 us in pieces of 768.  Chunks are shares of the table's capacity, since the lengths
// stay on the device: in wider tables the same keys fall into fewer of them (8 x 128 in tables of 4096 tokens 48 us, 8192
// 68, 16384 and more 117: all in the first).
constexpr double kCus = 256, kMerge = 4, kMergeRate = 8e6;
double tile_time(int64_t head_dim, double fill) {  // fill: work-groups per compute unit
    const double alone = head_dim <= 128 ? 0.85 + (double)head_dim / 200 : 0.65 + (double)head_dim / 105;
    const double both = head_dim <= 128 ? 1.4 : 2;
    return alone * (fill <= 1 ? 1 : fill <= 2 ? 1 + (both - 1) * (fill - 1) : both * fill / 2);
}
constexpr int64_t kMostChunks = 64, kLeastKeys = 256;

Plan plan(int64_t num_seqs, int64_t total, int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t block_size,
          int64_t width, int64_t chunk_tokens) {
    const int64_t capacity = block_size * width, group = q_heads / kv_heads;
    // Row blocks: full ones, at most one partial per sequence, and the one that clears.
    const int64_t items = total * group / kRows + num_seqs + 1;
    int64_t len = capacity;
    if (chunk_tokens > 0) {
        len = chunk_tokens;
    } else {
        // (A quarter of the partial ones, for the estimate; a sequence has one at least.)
        const double groups = (double)(std::max(total * group / kRows + num_seqs / 4, num_seqs) * kv_heads);
        const double rows = (double)(total * q_heads), tiles = (double)((capacity + kKeys - 1) / kKeys);
        double best = 0;
        for (int64_t n = 1; n <= kMostChunks && (n - 1) * kLeastKeys < capacity; ++n) {
            const double fill = groups * n / kCus;
            if (n > 1 && fill - groups / kCus >= 2) break;  // full already
            const double time = tile_time(head_dim, fill) * std::ceil(tiles / n) +
                                (n > 1 ? kMerge + rows * n * head_dim * 8 / kMergeRate : 0);
            if (n > 1 && time >= best) continue;
            best = time;
            len = (capacity + n - 1) / n;
        }
    }
    if (len > capacity) len = capacity;
    len = (len + kKeys - 1) / kKeys * kKeys;
    return {items, (capacity - 1) / len + 1, len};
}

template <typename T, int D>
int launch(const PrefillArgs& a, hipStream_t s) {
    const dim3 grid((unsigned)((int64_t)a.items * a.chunks * a.kv_heads)), block(kThreads);
    if (a.div.size % 16 == 0) hipLaunchKernelGGL((fp4_prefill_kernel<T, D, 16>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((fp4_prefill_kernel<T, D, 1>), grid, block, 0, s, a);
    if (int rc = check_launch("packed prefill")) return rc;
    if (a.chunks == 1) return MVME_OK;
    hipLaunchKernelGGL((fp4_prefill_merge_kernel<T, D>), dim3((unsigned)((a.total_tokens * a.q_heads - 1) / kMergeRows<D> + 1)),
                       dim3(kThreads), 0, s, a);
    return check_launch("packed prefill merge");
}

template <typename T>
int launch_dim(const PrefillArgs& a, int64_t head_dim, hipStream_t s) {
    switch (head_dim) {
        case 32: return launch<T, 32>(a, s);
        case 64: return launch<T, 64>(a, s);
        case 96: return launch<T, 96>(a, s);
        case 128: return launch<T, 128>(a, s);
        case 192: return launch<T, 192>(a, s);
        default: return launch<T, 256>(a, s);
    }
}

}  // namespace
}  // namespace fp4
}  // namespace mvme

using namespace mvme;
using namespace mvme::fp4;

extern "C" size_t mvme_fp4_paged_prefill_workspace_size(int64_t num_seqs, int64_t total_tokens, int64_t q_heads,
                                                        int64_t kv_heads, int64_t head_dim, int64_t block_size,
                                                        int64_t table_width, int64_t chunk_tokens) {
    if (!prefill_shape(num_seqs, total_tokens, q_heads, kv_heads, head_dim, block_size, table_width)) return 0;
    const Plan p = plan(num_seqs, total_tokens, q_heads, kv_heads, head_dim, block_size, table_width, chunk_tokens);
    return p.chunks == 1 ? 0
                         : (size_t)(total_tokens * q_heads) * ((size_t)p.chunks * (size_t)(head_dim + 2) + 1) * sizeof(float);
}

extern "C" int mvme_fp4_paged_prefill_attention(void* out, const void* q, const void* key_cache,
                                                const void* value_cache, const int64_t* cu_seqlens_q,
                                                const int64_t* query_starts, const int64_t* block_tables,
                                                const int64_t* context_lens, int64_t num_seqs, int64_t total_tokens,
                                                int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                                                int64_t num_blocks, int64_t block_size, int64_t table_width,
                                                int64_t chunk_tokens, int dtype, void* workspace,
                                                size_t workspace_bytes, void* stream) {
    if (!valid_dtype(dtype)) return fail(MVME_EINVAL, "FP16/BF16 required");
    if (num_seqs <= 0 || total_tokens < 0 || q_heads <= 0 || kv_heads <= 0 || num_blocks <= 0)
        return fail(MVME_EINVAL, "empty batch/heads/cache");
    if (q_heads % kv_heads != 0) return fail(MVME_EINVAL, "head dimension or GQA mismatch");
    if (!attention_dim(head_dim)) return fail(MVME_EINVAL, "supported head_dim: 32,64,96,128,192,256");
    if (block_size <= 0 || table_width <= 0) return fail(MVME_EINVAL, "invalid block table");
    if (block_size > kMaxCapacity || table_width > kMaxCapacity / block_size)
        return fail(MVME_EINVAL, "maximum table capacity is 1M tokens");
    if (!prefill_shape(num_seqs, total_tokens, q_heads, kv_heads, head_dim, block_size, table_width))
        return fail(MVME_EINVAL, "too many packed query rows");
    const int64_t record = record_bytes(block_size, head_dim);
    if (num_blocks > 2147483647 || num_blocks > (int64_t(1) << 62) / record / kv_heads)
        return fail(MVME_EINVAL, "KV cache too large");
    if (chunk_tokens < 0) return fail(MVME_EINVAL, "chunk_tokens must not be negative");
    if (total_tokens == 0) return MVME_OK;
    if (!out || !q || !key_cache || !value_cache || !cu_seqlens_q || !query_starts || !block_tables || !context_lens)
        return fail(MVME_EINVAL, "packed prefill: null pointer");
    if (!aligned(q, 16) || !aligned(key_cache, 16) || !aligned(value_cache, 16) || !aligned(out, 8))
        return fail(MVME_EINVAL, "packed prefill: queries and caches must be 16-byte, the output 8-byte aligned");
    const Plan p = plan(num_seqs, total_tokens, q_heads, kv_heads, head_dim, block_size, table_width, chunk_tokens);
    if (p.chunks > kMostThreads / kThreads / kv_heads / p.items ||
        (p.chunks > 1 && (total_tokens * q_heads - 1) / (kThreads / (head_dim / 4)) >= kMostThreads / kThreads))
        return fail(MVME_EINVAL, "too many packed query rows");
    const size_t need = mvme_fp4_paged_prefill_workspace_size(num_seqs, total_tokens, q_heads, kv_heads, head_dim,
                                                              block_size, table_width, chunk_tokens);
    if (need > 0 && (!workspace || workspace_bytes < need || !aligned(workspace, 16)))
        return fail(MVME_EWORKSPACE, "packed prefill workspace too small: " + std::to_string(need) +
                                         " bytes, 16-byte aligned, are needed");
    PrefillArgs a{};
    a.out = out;
    a.q = q;
    a.key = static_cast<const uint8_t*>(key_cache);
    a.value = static_cast<const uint8_t*>(value_cache);
    a.cu = cu_seqlens_q;
    a.starts = query_starts;
    a.tables = block_tables;
    a.lens = context_lens;
    a.partial = static_cast<float*>(workspace);
    a.stats = total_tokens * q_heads * p.chunks * head_dim;
    a.counts = reinterpret_cast<int32_t*>(a.partial + a.stats + total_tokens * q_heads * p.chunks * 2);
    a.num_blocks = num_blocks;
    a.record = record;
    a.page_bytes = (uint64_t)(record * kv_heads);
    a.total_tokens = total_tokens;
    a.num_seqs = (int)num_seqs;
    a.kv_heads = (int)kv_heads;
    a.q_heads = (int)q_heads;
    a.group = (int)(q_heads / kv_heads);
    a.width = (int)table_width;
    a.items = (int)p.items;
    a.chunks = (int)p.chunks;
    a.chunk_len = (int)p.chunk_len;
    a.div = make_block_div(block_size);
    a.group_div = make_block_div(a.group);
    a.scale = kLog2e / __builtin_sqrtf((float)head_dim);
    hipStream_t s = static_cast<hipStream_t>(stream);
    return dtype == MVME_FP16 ? launch_dim<Half>(a, head_dim, s) : launch_dim<BFloat16>(a, head_dim, s);
}
