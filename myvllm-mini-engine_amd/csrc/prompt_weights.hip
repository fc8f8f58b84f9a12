// The weight that a prompt's queries give each cached token: the column sums
// of the causal softmax, without its product with the values.
//
// Two passes over the scores, since a row's divisor is known only after its
// last key.  The first takes 128 query rows (a sequence's (token, head of the
// group) pairs) and a chunk of the keys per work-group and leaves each row's
// reference and sum; the second takes 128 keys, which its waves hold in
// registers, and lets all rows that see them pass by.  Each key is added up by
// one wave, so no atomics.
//
// Bounds: the passes are two products of half an attention's size, each score
// with an exponential, so vector work (four to six instructions a score) and the
// matrix products' own cycles are of one size.  2 x 4096 queries, 16 heads on 8
// of 128: 214 us for 137 GFLOP, 640 TFLOP/s (traced alone the passes take 111
// and 131).  Keeping the first pass's scores instead would move 2 GB there, 440
// us at the rate of a large copy.  Short calls are chains of
// dependent loads: the last 32 queries of 8192 tokens take 19 us, 10 and 9.
#include "../../include/mvme_long.h"
#include "long_attention.h"

namespace mvme {
namespace lng {
namespace {

typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr int kRows = 128;     // query rows of a work-group of the first pass
constexpr int kTile = 64;      // keys (first pass) or rows (second) of a tile in LDS
constexpr int kKeys = 128;     // keys of a work-group of the second pass

struct PromptArgs {
    const void* q;
    const uint8_t* key;
    const int64_t* cu;
    const int64_t* starts;
    const int64_t* tables;
    const int64_t* lens;
    float* partial;   // [total_tokens, q_heads, chunks, 2]: (reference, sum) of a chunk's keys
    float* received;  // [parts, num_seqs, kv_heads, key_blocks, kKeys]: what the rows of a part give (several parts only)
    float* weights;   // [num_seqs, kv_heads, weight_row]
    int64_t weight_row;
    int64_t num_blocks, total_tokens;
    uint64_t page_bytes;
    uint32_t row_bytes;
    int num_seqs, kv_heads, q_heads, group, width;
    int items, chunks, chunk_len, key_blocks, parts;
    uint32_t part_rows;  // rows of a work-group of the second pass
    BlockDiv div, group_div, chunk_div;
    float scale;
};

template <typename T>
__device__ inline f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
    if constexpr (T::kId == MVME_FP16)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

struct Seq {
    int64_t row0, rows;  // packed tokens
    int64_t start;
    int usable;          // keys that rows may see: none where the start or the length cannot be
};
__device__ inline Seq sequence(const PromptArgs& a, int s) {
    const int64_t lo = min(max(a.cu[s], (int64_t)0), a.total_tokens);
    const int64_t hi = min(max(a.cu[s + 1], lo), a.total_tokens);
    const int64_t start = a.starts[s], len = a.lens[s], capacity = (int64_t)a.width * a.div.size;
    return {lo, hi - lo, start, start < 0 || start >= len || len > capacity ? 0 : (int)len};
}
__device__ inline int row_blocks(const PromptArgs& a, int s) {
    const int64_t lo = min(max(a.cu[s], (int64_t)0), a.total_tokens);
    const int64_t hi = min(max(a.cu[s + 1], lo), a.total_tokens);
    return (int)(((hi - lo) * a.group + kRows - 1) / kRows);
}
// The sequence and its row block that `item` is: all sequences' last blocks, which see most keys, then those before them, and
// so on (up to 64 sequences; more go one after the other).  False behind all.
__device__ inline bool find_rows(const PromptArgs& a, int& item, int& s) {
    const int lane = __lane_id();
    if (a.num_seqs <= kWave) {
        const int blocks = lane < a.num_seqs ? row_blocks(a, lane) : 0;
        const auto all = [&](int n) { return lane_value(wave_incl_scan(min(blocks, n)), kWave - 1); };
        int top = blocks;
#pragma unroll
        for (int m = 1; m < kWave; m *= 2) top = max(top, __shfl_xor(top, m));
        top = uniform(top);
        if (item >= all(top)) return false;
        int low = 0, high = top;  // the last number from the end with no more than `item` blocks behind it
        while (high - low > 1) {
            const int mid = (low + high) >> 1;
            if (all(mid) <= item) low = mid;
            else high = mid;
        }
        const int behind = item - all(low), scan = wave_incl_scan(blocks > low ? 1 : 0);
        s = __builtin_ctzll(__ballot(scan > behind));
        item = lane_value(blocks, s) - 1 - low;
        return true;
    }
    for (s = 0; s < a.num_seqs; s += kWave) {
        const int blocks = s + lane < a.num_seqs ? row_blocks(a, s + lane) : 0;
        const int scan = wave_incl_scan(blocks);
        const uint64_t behind = __ballot(scan > item);
        if (behind) {
            const int at = __builtin_ctzll(behind);
            s += at;
            item = lane_value(scan, at) - 1 - item;
            return true;
        }
        item -= lane_value(scan, kWave - 1);
    }
    return false;
}

template <int D>
struct Piece {
    u32x4 x[Shape<D>::kChunks];
};

template <typename T, int D, int RUN>
__global__ __launch_bounds__(kThreads, 2) void prompt_rows_kernel(PromptArgs a) {
    using S = Shape<D>;
    constexpr int P = S::kDim;
    __shared__ __attribute__((aligned(16))) uint8_t tiles[2][kTile * 2 * P];
    __shared__ uint8_t present[2][kTile];
    __shared__ __attribute__((aligned(4))) uint8_t odd[2][4];
    const int lane = threadIdx.x & 63, column = lane & 31, h = lane >> 5;
    const int wave = uniform(threadIdx.x >> 6);
    const int place = blockIdx.x, kv_head = place % a.kv_heads, chunk = place / a.kv_heads % a.chunks;
    int item = place / a.kv_heads / a.chunks, s;
    if (!find_rows(a, item, s)) return;
    s = uniform(s);
    item = uniform(item);
    const Seq seq = sequence(a, s);
    const uint32_t row0 = (uint32_t)item * kRows, rows = (uint32_t)seq.rows * a.group;
    const uint32_t last_token = a.group_div.page(min(row0 + kRows, rows) - 1);
    const int64_t first_pos = seq.start + a.group_div.page(row0);
    const uint32_t key_end = (uint32_t)min((int64_t)seq.usable, max(seq.start + last_token + 1, (int64_t)0));
    const uint32_t begin = (uint32_t)chunk * a.chunk_len, end = min(key_end, begin + (uint32_t)a.chunk_len);
    if (chunk > 0 && begin >= end) return;

    const int64_t* table = a.tables + (int64_t)s * a.width;
    const int row = 16 * wave + 4 * ((lane >> 2) & 3) + (lane >> 4), quarter = lane & 3;
    const uint32_t looked = RUN == 16 ? 16 * wave : row;
    const auto page_of = [&](uint32_t t0) {
        const int64_t* entry = table + min(a.div.page(t0 + looked), (uint32_t)a.width - 1u);
        return RUN == 16 ? uniform_load(entry) : *entry;
    };
    uint32_t lane_at = (RUN == 16 ? (uint32_t)(row & 15) * a.row_bytes : 0u) + quarter * 16;
    bool there = false;
    const auto load = [&](Piece<D>& x, uint32_t t0, int64_t page) {
        const uint32_t token = t0 + looked;
        const bool found = token < end && (uint64_t)page < (uint64_t)a.num_blocks;
        there = found && t0 + row < end;
        const uint32_t place = found ? token - a.div.page(token) * a.div.size : 0u;
        const uint8_t* base = a.key + (int64_t)kv_head * (2 * D) + (int64_t)((uint64_t)(uint32_t)(found ? page : 0) * a.page_bytes) +
                              (int64_t)((uint64_t)place * a.row_bytes) + lane_at;
#pragma unroll
        for (int i = 0; i < S::kChunks; ++i) {
            if (D == P || (4 * i + quarter) * 8 < D) x.x[i] = *reinterpret_cast<const u32x4*>(base + 64 * i);
            else x.x[i] = u32x4{0u, 0u, 0u, 0u};
        }
    };
    TileAddress<P, 32> stage_at(row, quarter), key_at(column, h);
    const auto stage = [&](Piece<D>& x, int buffer) {
        const bool some = __any(!there);
        if (some && quarter == 0) present[buffer][row] = there;
        if (lane == 0) odd[buffer][wave] = some;
#pragma unroll
        for (int i = 0; i < S::kChunks; ++i) *reinterpret_cast<u32x4*>(tiles[buffer] + stage_at.chunk(4 * i)) = x.x[i];
    };
    Piece<D> staged;
    load(staged, begin, page_of(begin));
    int64_t page = page_of(begin + kTile);

    const uint32_t qrow = row0 + wave * 32 + column;
    const bool live = qrow < rows, busy = row0 + wave * 32 < rows;
    const uint32_t token = live ? a.group_div.page(qrow) : 0u;
    const int32_t limit = live && seq.start + token < seq.usable ? (int32_t)(seq.start + token) : -1;  // last visible key
    const int64_t head = (seq.row0 + token) * a.q_heads + (int64_t)kv_head * a.group + (live ? qrow - token * a.group : 0u);
    u32x4 q[S::kSteps];
#pragma unroll
    for (int i = 0; i < S::kSteps; ++i) {
        q[i] = u32x4{0u, 0u, 0u, 0u};
        if (live && (D == P || 16 * i + 8 * h < D))
            q[i] = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(a.q) + head * D + 16 * i + 8 * h);
    }
    float ref = kRefNone, sum = 0.f;
    stage(staged, 0);
    load(staged, begin + kTile, page);
    page = page_of(begin + 2 * kTile);
    lds_barrier();
    int buffer = 0;
#pragma unroll 1
    for (uint32_t t0 = begin; t0 < end; t0 += kTile, buffer ^= 1) {
        key_at.forget();
        stage_at.forget();
        asm volatile("" : "+v"(lane_at));
        const uint8_t* keys = tiles[buffer];
        if (!busy) {  // no row: this wave only stages
            stage(staged, buffer ^ 1);
            load(staged, t0 + 2 * kTile, page);
            page = page_of(t0 + 3 * kTile);
            lds_barrier();
            continue;
        }
        f32x16 x[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
#pragma unroll
            for (int i = 0; i < 16; ++i) x[k][i] = 0.f;
#pragma unroll
            for (int i = 0; i < S::kSteps; ++i)
                x[k] = mfma32<T>(*reinterpret_cast<const u32x4*>(keys + 32 * k * 2 * P + key_at.chunk(2 * i)), q[i], x[k]);
        }
        stage(staged, buffer ^ 1);
        load(staged, t0 + 2 * kTile, page);
        page = page_of(t0 + 3 * kTile);
        const uint32_t odds = (uint32_t)uniform(*reinterpret_cast<const int*>(odd[buffer]));
        uint64_t mask = ~uint64_t(0);
        if (odds) mask = __ballot((odds >> (8 * (lane >> 4))) & 0xff ? present[buffer][lane] : true);
        if (odds || (int64_t)t0 + kTile - 1 > first_pos) {
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
        float top = x[0][0];
#pragma unroll
        for (int i = 1; i < 32; ++i) top = fmaxf(top, x[i >> 4][i & 15]);
        if (__any(__builtin_fmaf(top, a.scale, -ref) > kRefSlack)) {
            top = pair32_max(top) * a.scale;
            const float moved = top > ref + kRefSlack ? top - kRefBelow : ref;
            sum *= fast_exp2(ref - moved);
            ref = moved;
        }
        float more[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 32; ++i) more[i & 3] += fast_exp2(__builtin_fmaf(x[i >> 4][i & 15], a.scale, -ref));
        sum += (more[0] + more[1]) + (more[2] + more[3]);
        lds_barrier();
    }
    const float total = swap32_add(sum, sum);  // the other half of the keys is with the lane 32 away
    if (!live || h != 0) return;
    a.partial[(head * a.chunks + chunk) * 2] = ref;
    a.partial[(head * a.chunks + chunk) * 2 + 1] = total;
}

template <typename T, int D>
__global__ __launch_bounds__(kThreads, D <= 128 ? 2 : 1) void prompt_keys_kernel(PromptArgs a) {
    using S = Shape<D>;
    constexpr int P = S::kDim;
    __shared__ __attribute__((aligned(16))) uint8_t tiles[2][kTile * 2 * P];
    __shared__ f32x2 divisors[2][kTile];  // (reference, 1 / sum) of a tile's rows
    const int lane = threadIdx.x & 63, column = lane & 31, h = lane >> 5;
    const int wave = uniform(threadIdx.x >> 6);
    const int unit = blockIdx.x % (a.kv_heads * a.num_seqs * a.key_blocks), part = blockIdx.x / (a.kv_heads * a.num_seqs * a.key_blocks);
    const int kv_head = unit % a.kv_heads, s = unit / a.kv_heads % a.num_seqs, block = unit / a.kv_heads / a.num_seqs;
    const Seq seq = sequence(a, s);
    const int key0 = block * kKeys;
    if (key0 >= seq.usable || seq.rows == 0) return;
    const int64_t past = (int64_t)key0 - seq.start;  // tokens before this one see none of these keys
    if (past >= seq.rows) return;
    const uint32_t from_row = past > 0 ? (uint32_t)past * a.group : 0u;  // the first that sees any
    const uint32_t first_row = max(from_row, (uint32_t)part * a.part_rows);
    const uint32_t rows = (uint32_t)min(seq.rows * a.group, (int64_t)(part + 1) * a.part_rows);
    if (first_row >= rows) return;

    // This lane's key: an operand of all its wave's products.
    const uint32_t key = (uint32_t)key0 + wave * 32 + column;
    u32x4 k[S::kSteps];
    bool there;
    {
        const uint32_t page_index = a.div.page(key);
        const int64_t page = a.tables[(int64_t)s * a.width + min(page_index, (uint32_t)a.width - 1u)];
        there = (int)key < seq.usable && (uint64_t)page < (uint64_t)a.num_blocks;
        const uint32_t place = there ? key - page_index * a.div.size : 0u;
        const uint8_t* at = a.key + (int64_t)kv_head * (2 * D) + (int64_t)((uint64_t)(uint32_t)(there ? page : 0) * a.page_bytes) +
                            (int64_t)((uint64_t)place * a.row_bytes);
#pragma unroll
        for (int i = 0; i < S::kSteps; ++i) {
            if (D == P || 16 * i + 8 * h < D) k[i] = *reinterpret_cast<const u32x4*>(at + (16 * i + 8 * h) * 2);
            else k[i] = u32x4{0u, 0u, 0u, 0u};
#pragma unroll
            for (int j = 0; j < 4; ++j) k[i][j] = there ? k[i][j] : 0u;
        }
    }

    const int row = 16 * wave + 4 * ((lane >> 2) & 3) + (lane >> 4), quarter = lane & 3;
    const int64_t head0 = seq.row0 * a.q_heads + (int64_t)kv_head * a.group;
    const auto head_of_row = [&](uint32_t r) {
        const uint32_t token = a.group_div.page(r);
        return head0 + (int64_t)token * a.q_heads + (r - token * a.group);
    };
    TileAddress<P, 32> stage_at(row, quarter), query_at(column, h);
    const auto load = [&](Piece<D>& x, uint32_t r0) {
        // (Behind the last row: the last row again, without a divisor.)
        const uint8_t* from = static_cast<const uint8_t*>(a.q) + head_of_row(min(r0 + row, rows - 1)) * (2 * D) + quarter * 16;
#pragma unroll
        for (int i = 0; i < S::kChunks; ++i) {
            if (D == P || (4 * i + quarter) * 8 < D) x.x[i] = *reinterpret_cast<const u32x4*>(from + 64 * i);
            else x.x[i] = u32x4{0u, 0u, 0u, 0u};
        }
    };
    const auto stage = [&](Piece<D>& x, int buffer) {
#pragma unroll
        for (int i = 0; i < S::kChunks; ++i) *reinterpret_cast<u32x4*>(tiles[buffer] + stage_at.chunk(4 * i)) = x.x[i];
    };
    // A row's divisor: its chunks go round four lanes.  The first two of each are loaded ahead.
    const uint32_t stat_row = threadIdx.x >> 2;
    const f32x2* stats = reinterpret_cast<const f32x2*>(a.partial);
    struct Chunks {
        f32x2 x[2];
    };
    const auto first_chunks = [&](uint32_t r0) {
        const f32x2* of_row = stats + head_of_row(min(r0 + stat_row, rows - 1)) * a.chunks;
        return Chunks{of_row[min(quarter, a.chunks - 1)], of_row[min(quarter + 4, a.chunks - 1)]};
    };
    const auto divide = [&](uint32_t r0, const Chunks& ahead, f32x2* to) {
        const uint32_t r = min(r0 + stat_row, rows - 1);
        const int64_t pos = seq.start + a.group_div.page(r);
        // (A row behind the last, or that sees no key, gets no divisor.)
        const int count = r0 + stat_row < rows && pos < seq.usable ? (int)a.chunk_div.page((uint32_t)pos) + 1 : 0;
        float ref = quarter < count ? ahead.x[0][0] : kRefNone, sum = quarter < count ? ahead.x[0][1] : 0.f;
        const auto join = [&](f32x2 y) {
            const float top = fmaxf(ref, y[0]);
            sum = sum * fast_exp2(ref - top) + y[1] * fast_exp2(y[0] - top);
            ref = top;
        };
        if (a.chunks > 1) {
            if (quarter + 4 < count) join(ahead.x[1]);
            if (a.chunks > 8) {
                const f32x2* of_row = stats + head_of_row(r) * a.chunks;
                for (int c0 = quarter + 8; c0 < a.chunks; c0 += 16) {
                    f32x2 y[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) y[i] = of_row[min(c0 + 4 * i, a.chunks - 1)];
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (c0 + 4 * i < count) join(y[i]);
                }
            }
            float top = fmaxf(ref, dpp<kDppQuadSwap1>(ref));
            top = fmaxf(top, dpp<kDppQuadSwap2>(top));
            sum = group_sum<4>(sum * fast_exp2(ref - top));
            ref = top;
        }
        if (quarter == 0) to[stat_row] = f32x2{ref, sum != 0.f ? 1.f / sum : 0.f};
    };
    Piece<D> staged;
    load(staged, first_row);
    Chunks ahead = first_chunks(first_row);
    float acc[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[i] = 0.f;
    stage(staged, 0);
    load(staged, first_row + kTile);
    divide(first_row, ahead, divisors[0]);
    ahead = first_chunks(first_row + kTile);
    lds_barrier();
    int buffer = 0;
#pragma unroll 1
    for (uint32_t r0 = first_row; r0 < rows; r0 += kTile, buffer ^= 1) {
        query_at.forget();
        stage_at.forget();
        f32x16 x[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
            for (int i = 0; i < 16; ++i) x[c][i] = 0.f;
#pragma unroll
            for (int i = 0; i < S::kSteps; ++i)
                x[c] = mfma32<T>(k[i], *reinterpret_cast<const u32x4*>(tiles[buffer] + 32 * c * 2 * P + query_at.chunk(2 * i)), x[c]);
        }
        stage(staged, buffer ^ 1);
        load(staged, r0 + 2 * kTile);
        divide(r0 + kTile, ahead, divisors[buffer ^ 1]);
        ahead = first_chunks(r0 + 2 * kTile);
        const int64_t first_pos = seq.start + a.group_div.page(r0);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const f32x2 of_row = divisors[buffer][32 * c + column];
            const float ref = of_row[0], by = of_row[1];
            // (A row without a divisor sees nothing; its scores may be anything.)
            if (key0 + 32 * wave + 31 > first_pos || __any(by == 0.f)) {
                const int64_t pos = seq.start + a.group_div.page(min(r0 + 32 * c + column, rows - 1));
                const int seen = by == 0.f ? -1 : (int)(pos - (key0 + 32 * wave + 4 * h));
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float p = fast_exp2(__builtin_fmaf(x[c][i], a.scale, -ref)) * by;
                    acc[i] += 8 * (i >> 2) + (i & 3) > seen ? 0.f : p;
                }
            } else {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    acc[i] = __builtin_fmaf(fast_exp2(__builtin_fmaf(x[c][i], a.scale, -ref)), by, acc[i]);
            }
        }
        lds_barrier();
    }
    // Sums over the 32 rows side by side; lane (i, h) of the first 16 adds key 8 (i / 4) + 4 h + i % 4.
    float mine = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const float all = group_sum<32>(acc[i]);
        mine = column == i ? all : mine;
    }
    const int at = 32 * wave + 8 * (column >> 2) + 4 * h + (column & 3);
    const uint64_t keys_there = __ballot(there);
    if (column >= 16) return;
    if (a.parts > 1)
        a.received[((int64_t)part * (a.kv_heads * a.num_seqs * a.key_blocks) + unit) * kKeys + at] = mine;
    else if ((keys_there >> (at & 31)) & 1)
        a.weights[((int64_t)s * a.kv_heads + kv_head) * a.weight_row + key0 + at] += mine;
}

// Adds up the parts, from the first that has rows which see the keys; one key per thread, in the order of the parts.
__global__ __launch_bounds__(kKeys) void prompt_add_kernel(PromptArgs a) {
    const int units = a.kv_heads * a.num_seqs * a.key_blocks, unit = blockIdx.x;
    const int kv_head = unit % a.kv_heads, s = unit / a.kv_heads % a.num_seqs, block = unit / a.kv_heads / a.num_seqs;
    const Seq seq = sequence(a, s);
    const int key0 = block * kKeys, key = key0 + threadIdx.x;
    const int64_t past = max((int64_t)key0 - seq.start, (int64_t)0);
    if (key >= seq.usable || past >= seq.rows) return;
    const int64_t page = a.tables[(int64_t)s * a.width + a.div.page((uint32_t)key)];
    if ((uint64_t)page >= (uint64_t)a.num_blocks) return;
    const int first = (int)((uint32_t)past * a.group / a.part_rows), last = (int)(((uint32_t)seq.rows * a.group - 1) / a.part_rows);
    float sum = 0.f;
    for (int p = first; p <= last; ++p) sum += a.received[((int64_t)p * units + unit) * kKeys + threadIdx.x];
    a.weights[((int64_t)s * a.kv_heads + kv_head) * a.weight_row + key] += sum;
}

struct Plan {
    int64_t items, chunks, chunk_len, key_blocks, parts, part_rows;
    size_t floats;
};
Plan plan(int64_t num_seqs, int64_t total, int64_t q_heads, int64_t kv_heads, int64_t block_size, int64_t width) {
    const int64_t capacity = block_size * width, group = q_heads / kv_heads;
    Plan p{};
    p.items = total * group / kRows + num_seqs;
    // Chunks of the keys, 256 at least, until there are about three work-groups per compute unit.
    p.chunks = std::max<int64_t>(1, std::min((capacity + 255) / 256, 768 / (p.items * kv_heads)));
    p.chunks = std::min<int64_t>(p.chunks, 64);
    p.chunk_len = ((capacity + p.chunks - 1) / p.chunks + kTile - 1) / kTile * kTile;
    p.chunks = (capacity - 1) / p.chunk_len + 1;
    p.key_blocks = (capacity - 1) / kKeys + 1;
    // Parts of the rows, if sequences are alike of 1024 to 2048 rows: the first keys are seen by all rows and the last by few,
    // and the longest work-group is the last (2 x 4096 tokens, 16 heads on 8: 223 us, 257 in one part).  Where there are
    // thousands of work-groups anyhow, they balance by themselves.
    const int64_t all = total * group;
    p.parts = std::max<int64_t>(1, std::min<int64_t>(all / num_seqs / 1024, 4096 / (num_seqs * kv_heads * p.key_blocks)));
    p.part_rows = ((all - 1) / p.parts / kTile + 1) * kTile;
    p.floats = (size_t)(total * q_heads * p.chunks * 2);
    if (p.parts > 1) p.floats += (size_t)(p.parts * num_seqs * kv_heads * p.key_blocks) * kKeys;
    return p;
}

template <typename T, int D>
int launch(const PromptArgs& a, hipStream_t s) {
    const dim3 grid((unsigned)((int64_t)a.items * a.chunks * a.kv_heads)), block(kThreads);
    if (a.div.size % 16 == 0) hipLaunchKernelGGL((prompt_rows_kernel<T, D, 16>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((prompt_rows_kernel<T, D, 1>), grid, block, 0, s, a);
    if (int rc = check_launch("prompt weights, rows")) return rc;
    hipLaunchKernelGGL((prompt_keys_kernel<T, D>), dim3((unsigned)((int64_t)a.num_seqs * a.key_blocks * a.kv_heads * a.parts)), block, 0, s, a);
    if (int rc = check_launch("prompt weights, keys")) return rc;
    if (a.parts == 1) return MVME_OK;
    hipLaunchKernelGGL(prompt_add_kernel, dim3((unsigned)((int64_t)a.num_seqs * a.key_blocks * a.kv_heads)), dim3(kKeys), 0, s, a);
    return check_launch("prompt weights, parts");
}

template <typename T>
int launch_dim(const PromptArgs& a, int64_t head_dim, hipStream_t s) {
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

bool prompt_shape(int64_t num_seqs, int64_t total, int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t block_size,
                  int64_t width) {
    return num_seqs > 0 && num_seqs <= 16777216 && total >= 0 && q_heads > 0 && kv_heads > 0 && q_heads % kv_heads == 0 &&
           head_dim_built(head_dim) && block_size > 0 && block_size <= kMaxCapacity && width > 0 &&
           width <= kMaxCapacity / block_size && q_heads <= 2147483647 / head_dim && total <= 2147483647 / q_heads;
}
bool row_fits(int64_t kv_heads, int64_t head_dim) { return kv_heads * head_dim * 2 <= 65536 * 16; }
bool fits_launch(const Plan& p, int64_t num_seqs, int64_t kv_heads) {
    return p.items <= kMostThreads / kThreads / kv_heads / p.chunks &&
           num_seqs <= kMostThreads / kThreads / kv_heads / p.key_blocks / p.parts;
}

}  // namespace
}  // namespace lng
}  // namespace mvme

using namespace mvme;
using namespace mvme::lng;

extern "C" size_t mvme_prefill_attention_weights_workspace_size(int64_t num_seqs, int64_t total_tokens, int64_t q_heads,
                                                                int64_t kv_heads, int64_t head_dim, int64_t block_size,
                                                                int64_t table_width) {
    if (!prompt_shape(num_seqs, total_tokens, q_heads, kv_heads, head_dim, block_size, table_width) ||
        !row_fits(kv_heads, head_dim) || total_tokens == 0)
        return 0;
    const Plan p = plan(num_seqs, total_tokens, q_heads, kv_heads, block_size, table_width);
    return fits_launch(p, num_seqs, kv_heads) ? p.floats * sizeof(float) : 0;
}

extern "C" int mvme_prefill_attention_weights(const void* q, const void* key_cache, const int64_t* cu_seqlens_q,
                                              const int64_t* query_starts, const int64_t* block_tables,
                                              const int64_t* context_lens, float* weights, int64_t weight_row,
                                              int64_t num_seqs, int64_t total_tokens, int64_t q_heads, int64_t kv_heads,
                                              int64_t head_dim, int64_t num_blocks, int64_t block_size,
                                              int64_t table_width, int dtype, void* workspace, size_t workspace_bytes,
                                              void* stream) {
    if (!valid_dtype(dtype)) return fail(MVME_EINVAL, "FP16/BF16 required");
    if (num_seqs <= 0 || total_tokens < 0 || q_heads <= 0 || kv_heads <= 0 || num_blocks <= 0)
        return fail(MVME_EINVAL, "empty batch/heads/cache");
    if (q_heads % kv_heads != 0) return fail(MVME_EINVAL, "head dimension or GQA mismatch");
    if (!head_dim_built(head_dim)) return fail(MVME_EINVAL, "supported head_dim: 16,32,64,80,96,128,192,256");
    if (block_size <= 0 || table_width <= 0) return fail(MVME_EINVAL, "invalid block table");
    if (block_size > kMaxCapacity || table_width > kMaxCapacity / block_size)
        return fail(MVME_EINVAL, "maximum table capacity is 1M tokens");
    if (!prompt_shape(num_seqs, total_tokens, q_heads, kv_heads, head_dim, block_size, table_width))
        return fail(MVME_EINVAL, "too many packed query rows");
    const int64_t row = kv_heads * head_dim * 2;
    if (!row_fits(kv_heads, head_dim) || num_blocks > 2147483647 || num_blocks > (int64_t(1) << 62) / row / block_size)
        return fail(MVME_EINVAL, "KV cache too large");
    if (weight_row < block_size * table_width) return fail(MVME_EINVAL, "weight rows must hold the tables' capacity");
    if (total_tokens == 0) return MVME_OK;
    if (!q || !key_cache || !cu_seqlens_q || !query_starts || !block_tables || !context_lens || !weights)
        return fail(MVME_EINVAL, "prompt weights: null pointer");
    if (!fp4::aligned(q, 16) || !fp4::aligned(key_cache, 16) || !fp4::aligned(weights, 4))
        return fail(MVME_EINVAL, "prompt weights: queries and caches must be 16-byte aligned");
    const Plan p = plan(num_seqs, total_tokens, q_heads, kv_heads, block_size, table_width);
    if (!fits_launch(p, num_seqs, kv_heads)) return fail(MVME_EINVAL, "too many packed query rows");
    const size_t need = p.floats * sizeof(float);
    if (!workspace || workspace_bytes < need || !fp4::aligned(workspace, 16))
        return fail(MVME_EWORKSPACE, "prompt weights workspace too small: " + std::to_string(need) +
                                         " bytes, 16-byte aligned, are needed");
    PromptArgs a{};
    a.q = q;
    a.key = static_cast<const uint8_t*>(key_cache);
    a.cu = cu_seqlens_q;
    a.starts = query_starts;
    a.tables = block_tables;
    a.lens = context_lens;
    a.partial = static_cast<float*>(workspace);
    a.received = a.partial + total_tokens * q_heads * p.chunks * 2;
    a.weights = weights;
    a.weight_row = weight_row;
    a.num_blocks = num_blocks;
    a.total_tokens = total_tokens;
    a.page_bytes = (uint64_t)(row * block_size);
    a.row_bytes = (uint32_t)row;
    a.num_seqs = (int)num_seqs;
    a.kv_heads = (int)kv_heads;
    a.q_heads = (int)q_heads;
    a.group = (int)(q_heads / kv_heads);
    a.width = (int)table_width;
    a.items = (int)p.items;
    a.chunks = (int)p.chunks;
    a.chunk_len = (int)p.chunk_len;
    a.key_blocks = (int)p.key_blocks;
    a.parts = (int)p.parts;
    a.part_rows = (uint32_t)p.part_rows;
    a.div = fp4::make_block_div(block_size);
    a.group_div = fp4::make_block_div(a.group);
    a.chunk_div = fp4::make_block_div(p.chunk_len);
    a.scale = kLog2e / __builtin_sqrtf((float)head_dim);
    hipStream_t st = static_cast<hipStream_t>(stream);
    return dtype == MVME_FP16 ? launch_dim<Half>(a, head_dim, st) : launch_dim<BFloat16>(a, head_dim, st);
}
