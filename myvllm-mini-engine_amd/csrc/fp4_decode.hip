// Decode attention over packed 4-bit pages: one query token per sequence.
//
// A unit is one sequence and kv head (16 of its query heads).  A work-group's
// waves take the tiles of 32 keys of a unit in turn and keep their own
// maximum, sum and accumulators, joined through LDS at the end.  Units are
// handed out whole, or all units are laid end to end and cut into equal
// shares (in rounds: one tile for every wave), one per work-group, so that
// ragged and few long sequences load every CU alike; a second kernel joins the
// units that a share boundary cuts.
//
// Bound by the cache's bytes where there are enough of them: 64 ragged
// sequences of up to 4096 tokens 39 us (22 us at 6.8 TB/s; the start and drain
// of a work-group and the join are the rest), 4 x 65536 tokens 37 us (21 us),
// one of 128 tokens 4.1 us (a launch and a chain of table, page and score
// latency).  Times in this file are of calls back to back in a graph; from
// Python the smallest takes 4.9-5.1.  Matrix tiles of 16 heads x 32 keys: a
// lane's four-bit codes are its score operand as they lie in memory, only
// values go through LDS, for the transposition.
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
    float* pieces;   // [work-groups, 2, 16, D] accumulators, then [work-groups, 2, 16, 2] (reference, sum)
    int64_t num_blocks, record;
    uint64_t page_bytes;
    int64_t stats;   // offset of the (reference, sum) pairs, in floats
    int batch, kv_heads, group, q_heads, width;
    int head_tiles;  // ceil(group / 16)
    int groups;      // work-groups of the walk; 0: one per unit
    int share;       // rounds of a share; 0: as many as spread all rounds over the work-groups
    BlockDiv div;
    float scale;     // log2(e) / sqrt(D)
};

// Waves of a work-group: four work-groups fit a CU up to 128 dims and so overlap each other's joins (64 ragged sequences
// of up to 4096 tokens: 38.9 us; eight waves 47.4, two 39.1).
constexpr int kWaves = 4;
constexpr int kRound = kWaves * kTileKeys;  // keys of a round

template <int D>
struct Shape {
    static constexpr int kChunks = D / 32;           // score products per 16 keys; dwords of codes per lane
    static constexpr int kPer = D % 128 == 0 ? 4 : D == 64 || D == 192 ? 2 : 1;  // chunks that share a scale
    static constexpr int kScales = kChunks / kPer;
    static constexpr int kDimTiles = D / 16;
    static constexpr int kTileBytes = kTileKeys * 2 * D;  // fp16 rows of a tile; as large as a wave's accumulators
    static constexpr int kMinWaves = D <= 128 ? 4 : 2;
};

// The walk's order: sequences, their units, a unit's rounds.
template <int D>
__device__ inline int rounds_of(const DecodeArgs& a, int64_t len) {
    const bool usable = len > 0 && len <= (int64_t)a.width * a.div.size;
    return usable ? (int)(((uint32_t)len - 1) / kRound) + 1 : 0;
}

__device__ inline int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ inline int64_t length_of(const DecodeArgs& a, int seq) { return seq < a.batch ? a.lens[seq] : 0; }

// Shares of the walk, in rounds, have two where that still gives every CU one: more pieces cost the join more than they save
// (8192 tokens, 8 kv heads: 9.3 us in shares of two, 10.7 of one), fewer leave the CUs unevenly loaded (16 ragged sequences
// of up to 4096: 16.0 us, 19.7 in shares of four).
constexpr int kCus = 256, kLeastShare = 2;

// The walk.  Every wave computes the same, lane-parallel over the sequences; the first 64 lengths stay in registers.
template <int D>
struct Walk {
    int64_t len;  // of sequence `lane`
    int units;    // of a sequence
    int total, share;
    __device__ inline void count(const DecodeArgs& a) {
        units = a.kv_heads * a.head_tiles;
        const int lane = __lane_id();
        len = length_of(a, lane);
        total = lane_value(wave_incl_scan(rounds_of<D>(a, len)), kWave - 1);
        for (int s0 = kWave; s0 < a.batch; s0 += kWave)
            total += lane_value(wave_incl_scan(rounds_of<D>(a, length_of(a, s0 + lane))), kWave - 1);
        total *= units;
        share = a.share > 0 ? a.share : max((total + a.groups - 1) / a.groups, min((total + kCus - 1) / kCus, kLeastShare));
    }
    // The sequence that owns round `round` (< total), the round it begins at, its rounds per unit and its length.
    __device__ inline void find(const DecodeArgs& a, int round, int& seq, int& base, int& rounds, uint32_t& tokens) const {
        const int lane = __lane_id();
        int before = 0;
        for (int s0 = 0;; s0 += kWave) {
            const int64_t n = s0 == 0 ? len : length_of(a, s0 + lane);
            const int mine = rounds_of<D>(a, n) * units, incl = before + wave_incl_scan(mine);
            const uint64_t hit = __ballot(incl > round);
            if (hit || s0 + kWave >= a.batch) {
                const int at = hit ? __builtin_ctzll(hit) : 0;
                seq = s0 + at;
                rounds = lane_value(mine, at);
                base = lane_value(incl, at) - rounds;
                rounds /= units;
                tokens = (uint32_t)lane_value((int)n, at);
                return;
            }
            before = lane_value(incl, kWave - 1);
        }
    }
    // First round of sequence `seq`.
    __device__ inline int first_of(const DecodeArgs& a, int seq) const {
        const int lane = __lane_id();
        int base = 0;
        for (int s0 = 0; s0 < seq; s0 += kWave) {
            const int mine = s0 + lane < seq ? rounds_of<D>(a, s0 == 0 ? len : length_of(a, s0 + lane)) : 0;
            base += lane_value(wave_incl_scan(mine), kWave - 1);
        }
        return base * units;
    }
};

// A run of rounds of one unit: what a work-group does at a time.  Wave-uniform.
struct Segment {
    int seq, kv_head, tile;
    uint32_t begin, end;  // keys
    int slot;             // where its piece goes; -1: it is the whole unit, straight to the output
    int rounds;           // 0: none
};

template <int D>
struct Part {  // a lane's part of one token of one plane: D / 4 dims
    uint32_t codes[Shape<D>::kChunks];
    uint32_t scales[Shape<D>::kScales];
};

template <int D>
__device__ inline void clear_part(Part<D>& x, bool keep) {
#pragma unroll
    for (int i = 0; i < Shape<D>::kChunks; ++i) x.codes[i] = keep ? x.codes[i] : 0u;
#pragma unroll
    for (int i = 0; i < Shape<D>::kScales; ++i) x.scales[i] = keep ? x.scales[i] : 127u;
}

// Where a tile's tokens are.  RUN tokens (block sizes that are multiples of
// RUN) lie in one page at consecutive places: their record and first place are
// wave-uniform, and a lane's own offset never changes.  RUN 1: every lane looks
// its tokens up.
template <int D, int RUN>
struct Where {
    static constexpr int kCount = RUN == 32 ? 1 : 2;
    int64_t codes[kCount];     // byte offset of the run's first token in a plane; of a page that exists, to load without a branch
    uint32_t scales[kCount];   // from there to its scales
    bool there[kCount];
};

template <int D, int RUN>
__device__ inline Where<D, RUN> look_up(const DecodeArgs& a, const int64_t* table, int64_t head, uint32_t first,
                                        uint32_t end, int r) {
    Where<D, RUN> w;
#pragma unroll
    for (int s = 0; s < Where<D, RUN>::kCount; ++s) {
        const uint32_t token = first + 16 * s + (RUN == 1 ? r : 0), block = a.div.page(token);
        const int64_t* entry = table + min(block, (uint32_t)a.width - 1u);
        int64_t page = RUN == 1 ? *entry : uniform_load(entry);
        uint32_t place = token - block * a.div.size;
        w.there[s] = token < end && (uint64_t)page < (uint64_t)a.num_blocks;
        page = w.there[s] ? page : 0;
        place = w.there[s] ? place : 0u;
        w.codes[s] = head + (int64_t)((uint64_t)(uint32_t)page * a.page_bytes) + place * (D / 2);
        w.scales[s] = a.div.size * (D / 2) - place * (D / 2 - D / kBlockDims);
    }
    return w;
}

// A lane's offsets in a run.  Kept from being widened outside of the loop, they stay the 32-bit offset of a load.
template <int D, int RUN>
struct LaneAt {
    uint32_t codes, scales[Shape<D>::kScales];
    __device__ inline LaneAt(int r, int g) : codes((RUN == 1 ? 0 : r * (D / 2)) + g * (D / 8)) {
#pragma unroll
        for (int i = 0; i < Shape<D>::kScales; ++i)
            scales[i] = (RUN == 1 ? 0 : r * (D / kBlockDims)) + (g * (D / 4) + 8 * i * Shape<D>::kPer) / kBlockDims;
    }
    __device__ inline void forget() {
        asm volatile("" : "+v"(codes));
#pragma unroll
        for (int i = 0; i < Shape<D>::kScales; ++i) asm volatile("" : "+v"(scales[i]));
    }
};

template <int D>
__device__ inline void load_codes(Part<D>& x, const uint8_t* codes) {
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
}

template <int D, int RUN>
__device__ inline void load_tile(Part<D> (&x)[2], const uint8_t* plane, const Where<D, RUN>& w, const LaneAt<D, RUN>& at) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        const int run = RUN == 32 ? 0 : s, more = RUN == 32 ? 16 * s : 0;
        const uint8_t* base = plane + w.codes[run];
        load_codes<D>(x[s], base + at.codes + more * (D / 2));
#pragma unroll
        for (int i = 0; i < Shape<D>::kScales; ++i)
            x[s].scales[i] = (base + (at.scales[i] + w.scales[run]))[more * (D / kBlockDims)];
    }
}

template <int D>
__device__ inline void load_query(u32x4 (&q)[Shape<D>::kChunks], const DecodeArgs& a, const Segment& s, int r, int g) {
    // Head r, dims g * D / 4 + 8 c .. + 7: the order in which a lane's codes lie.
    const bool live = r < min(16, a.group - s.tile * 16);
    const int64_t head = (int64_t)s.seq * a.q_heads + s.kv_head * a.group + s.tile * 16 + r;
#pragma unroll
    for (int c = 0; c < Shape<D>::kChunks; ++c) {
        q[c] = u32x4{0u, 0u, 0u, 0u};
        if (live) q[c] = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(a.query) + head * D + g * (D / 4) + 8 * c);
    }
}

template <typename T, int D, int RUN>
__global__ __launch_bounds__(64 * kWaves, Shape<D>::kMinWaves) void fp4_decode_kernel(DecodeArgs a) {
    using S = Shape<D>;
    __shared__ __attribute__((aligned(16))) uint8_t tiles[kWaves][S::kTileBytes];
    __shared__ float stats[kWaves][2][16];
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

    Walk<D> walk;
    int first = 0, stop = 0;  // the share, in rounds
    if (a.groups) {
        walk.count(a);
        const int64_t from = (int64_t)blockIdx.x * walk.share;
        first = (int)min(from, (int64_t)walk.total);
        stop = (int)min(from + walk.share, (int64_t)walk.total);
        if (first == stop) return;
    }
    // The segment that begins at round `at` of the share (or the work-group's unit).
    const auto segment = [&](int at) {
        Segment s;
        int unit, from, n, rounds;
        uint32_t tokens;
        if (a.groups) {
            int base;
            walk.find(a, at, s.seq, base, rounds, tokens);
            unit = (at - base) / rounds;
            from = at - base - unit * rounds;
            n = min(rounds - from, stop - at);
            s.slot = n == rounds ? -1 : (int)blockIdx.x * 2 + (at > first ? 1 : 0);
        } else {
            const int units = a.kv_heads * a.head_tiles;
            s.seq = blockIdx.x / units;
            unit = blockIdx.x - s.seq * units;
            const int64_t len = a.lens[s.seq];
            rounds = rounds_of<D>(a, len);
            tokens = rounds ? (uint32_t)len : 0u;
            from = 0;
            n = max(rounds, 1);  // an empty sequence: one round without keys, which writes the zeros
            s.slot = -1;
        }
        // (Uniform all along, but only now provably so: what these address is loaded and computed once per wave.)
        s.seq = uniform(s.seq);
        s.kv_head = uniform(unit / a.head_tiles);
        s.tile = uniform(unit) - s.kv_head * a.head_tiles;
        s.begin = (uint32_t)uniform(from * kRound);
        s.end = (uint32_t)uniform((int)min(tokens, (uint32_t)(from + n) * kRound));
        s.slot = uniform(s.slot);
        s.rounds = uniform(n);
        return s;
    };

    TileAddress<D, 16> write_at(r, g * S::kChunks), read_at(4 * g + (r >> 2), (r & 3) >> 1, (r & 1) * 8);
    LaneAt<D, RUN> lane_at(r, g);
    uint8_t* tile_lds = tiles[wave];
    // A tile's registers are refilled as soon as they are used up: keys after
    // the scores, values when they are in LDS.  The lookups run a tile ahead,
    // and all of it runs on into the next segment.
    u32x4 q[S::kChunks];
    Part<D> k[2], v[2];
    Where<D, RUN> now;
    const auto find_tile = [&](const Segment& s, uint32_t t) {
        return look_up<D, RUN>(a, a.tables + (int64_t)s.seq * a.width, s.kv_head * a.record, t, s.end, r);
    };
    int at = first;
    Segment seg = segment(at);
    uint32_t t0 = seg.begin + wave * kTileKeys;
    now = find_tile(seg, t0);
    load_query<D>(q, a, seg, r, g);
    load_tile<D, RUN>(k, a.key, now, lane_at);
    load_tile<D, RUN>(v, a.value, now, lane_at);
#pragma unroll 1
    for (;;) {
        at += seg.rounds;
        Segment ahead;
        ahead.rounds = 0;
        if (at < stop) ahead = segment(at);
        f32x4 acc[S::kDimTiles];
#pragma unroll
        for (int n = 0; n < S::kDimTiles; ++n) acc[n] = f32x4{0.f, 0.f, 0.f, 0.f};
        float ref = kRefNone, sum = 0.f;
        const bool idle = t0 >= seg.end;  // no tile of this segment for this wave
#pragma unroll 1
        for (; t0 < seg.end; t0 += kRound) {
            const bool more = t0 + kRound < seg.end;
            write_at.forget();
            read_at.forget();
            lane_at.forget();
            Where<D, RUN> next = now;
            if (more) next = find_tile(seg, t0 + kRound);
            else if (ahead.rounds) next = find_tile(ahead, ahead.begin + wave * kTileKeys);
            // Scores.
            f32x4 x[2];
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                x[s] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = 0; i < S::kChunks; ++i)
                    x[s] = T::mfma16x16x32(values_of<T>(k[s].codes[i], scale_of(k[s].scales[i / S::kPer])), q[i], x[s]);
            }
            if (!more && ahead.rounds) load_query<D>(q, a, ahead, r, g);
            if (more || ahead.rounds) load_tile<D, RUN>(k, a.key, next, lane_at);
            // Keys that are not there: no weight, and zeros as values (0 * NaN is NaN).
            constexpr int kLast = Where<D, RUN>::kCount - 1;
            bool whole = t0 + kTileKeys <= seg.end && now.there[0] && now.there[kLast];
            if constexpr (RUN == 1) whole = __all(whole);
            if (!whole) {
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    const bool mine = now.there[s < kLast ? s : kLast] && t0 + 16 * s + r < seg.end;
                    const uint32_t present = (uint32_t)__ballot(mine) >> (4 * g);
                    clear_part<D>(v[s], mine);
#pragma unroll
                    for (int j = 0; j < 4; ++j) x[s][j] = (present >> j) & 1 ? x[s][j] : kNegInf;
                }
            }
            // Values to LDS in fp16, row-major.
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int i = 0; i < S::kChunks; ++i)
                    *reinterpret_cast<u32x4*>(tile_lds + write_at.chunk(i) + 16 * s * 2 * D) =
                        values_of<Half>(v[s].codes[i], scale_of(v[s].scales[i / S::kPer]));
            if (more || ahead.rounds) load_tile<D, RUN>(v, a.value, next, lane_at);
            // Reference and probabilities.
            float top = fmaxf(x[0][0], x[1][0]);
#pragma unroll
            for (int j = 1; j < 4; ++j) top = fmaxf(top, fmaxf(x[0][j], x[1][j]));
            top = row4_max(top) * a.scale;
            if (__any(top > ref + kRefSlack)) {
                const float moved = top > ref + kRefSlack ? top - kRefBelow : ref;
                const float by = fast_exp2(ref - moved);
                ref = moved;
                sum *= by;
#pragma unroll
                for (int n = 0; n < S::kDimTiles; ++n) acc[n] *= by;
            }
            u32x4 weights;
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                float p[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) p[j] = fast_exp2(__builtin_fmaf(x[s][j], a.scale, -ref));
                weights[2 * s] = Half::pack(p[0], p[1]);
                weights[2 * s + 1] = Half::pack(p[2], p[3]);
            }
            // The sum is of the weights as rounded: what a rounding adds to the values' product it adds to the divisor.
#pragma unroll
            for (int i = 0; i < 4; ++i) sum = Half::dot2(weights[i], 0x3c003c00u, sum);
            // A wave reads only what it wrote: the LDS queue is in order, no barrier.
#pragma unroll
            for (int n = 0; n < S::kDimTiles; ++n) {
                const u32x4 vt = value_operand(tile_lds, read_at.chunk(2 * n), read_at.chunk(2 * n) + 16 * 2 * D);
                acc[n] = Half::mfma16x16x32(vt, weights, acc[n]);
            }
            now = next;
        }
        if (idle && ahead.rounds) {
            now = find_tile(ahead, ahead.begin + wave * kTileKeys);
            load_query<D>(q, a, ahead, r, g);
            load_tile<D, RUN>(k, a.key, now, lane_at);
            load_tile<D, RUN>(v, a.value, now, lane_at);
        }
        sum = row4_sum(sum);

        // Join the waves: accumulators [16][D] in their tiles' LDS, each relative to its own reference.
        const int heads = min(16, a.group - seg.tile * 16);
        float* mine = reinterpret_cast<float*>(tile_lds);
        if (r < heads) {
#pragma unroll
            for (int n = 0; n < S::kDimTiles; ++n) *reinterpret_cast<f32x4*>(mine + r * D + 16 * n + 4 * g) = acc[n];
            if (g == 0) {
                stats[wave][0][r] = ref;
                stats[wave][1][r] = sum;
            }
        }
        __syncthreads();
        const int64_t first_head = (int64_t)seg.seq * a.q_heads + seg.kv_head * a.group + seg.tile * 16;
        for (int i = threadIdx.x; i < heads * D; i += 64 * kWaves) {
            const int h = i / D, d = i - h * D;
            float top = stats[0][0][h];
#pragma unroll
            for (int w = 1; w < kWaves; ++w) top = fmaxf(top, stats[w][0][h]);
            float total = 0.f, value = 0.f;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                const float by = fast_exp2(stats[w][0][h] - top);
                total += by * stats[w][1][h];
                value += by * reinterpret_cast<const float*>(tiles[w])[i];
            }
            if (seg.slot < 0) {
                static_cast<uint16_t*>(a.out)[first_head * D + i] = T::from_float(total != 0.f ? value / total : 0.f);
            } else {
                const int64_t slot = (int64_t)seg.slot * 16;
                a.pieces[slot * D + i] = value;
                if (d == 0) {
                    a.pieces[a.stats + (slot + h) * 2] = top;
                    a.pieces[a.stats + (slot + h) * 2 + 1] = total;
                }
            }
        }
        if (!ahead.rounds) return;
        __syncthreads();  // the tiles are free again
        seg = ahead;
        t0 = seg.begin + wave * kTileKeys;
    }
}

// Joins the pieces of the units that share boundaries cut, and clears what has no keys; one work-group per query head.
// The pieces go round the thread groups of D / 4 lanes; a group joins its own on the way.
constexpr int kMergeThreads = 256;

template <typename T, int D>
__global__ __launch_bounds__(kMergeThreads) void fp4_merge_kernel(DecodeArgs a) {
    constexpr int kLanes = D / 4, kGroups = kMergeThreads / kLanes;
    __shared__ __attribute__((aligned(16))) float sums[kGroups][D];
    __shared__ float stats[kGroups][2];
    const int head = blockIdx.x % a.q_heads, b = blockIdx.x / a.q_heads;
    Walk<D> walk;
    walk.count(a);
    const int rounds = rounds_of<D>(a, a.lens[b]);
    const int kv_head = head / a.group, in_group = head % a.group;
    uint16_t* out = static_cast<uint16_t*>(a.out) + (int64_t)blockIdx.x * D;
    if (rounds == 0) {
        for (int d = threadIdx.x; d < D; d += kMergeThreads) out[d] = 0;
        return;
    }
    const int at = walk.first_of(a, b) + (kv_head * a.head_tiles + in_group / 16) * rounds;
    const int first = at / walk.share, last = (at + rounds - 1) / walk.share;
    if (first == last) return;  // one share has it all
    const int group = threadIdx.x / kLanes, lane = threadIdx.x % kLanes;
    f32x4 value = {0.f, 0.f, 0.f, 0.f};
    float ref = kRefNone, sum = 0.f;
    if (group < kGroups) {
#pragma unroll 4
        for (int i = first + group; i <= last; i += kGroups) {
            // A piece that begins its share is in the share's first slot.
            const int64_t slot = (int64_t)i * 2 + (i == first && at > first * walk.share ? 1 : 0);
            const float* s = a.pieces + a.stats + (slot * 16 + in_group % 16) * 2;
            const f32x4 v = *reinterpret_cast<const f32x4*>(a.pieces + (slot * 16 + in_group % 16) * D + 4 * lane);
            const float top = fmaxf(ref, s[0]), keep = fast_exp2(ref - top), by = fast_exp2(s[0] - top);
            value = value * keep + v * by;
            sum = sum * keep + s[1] * by;
            ref = top;
        }
        *reinterpret_cast<f32x4*>(&sums[group][4 * lane]) = value;
        if (lane == 0) {
            stats[group][0] = ref;
            stats[group][1] = sum;
        }
    }
    __syncthreads();
    for (int d = threadIdx.x; d < D; d += kMergeThreads) {
        float top = stats[0][0];
#pragma unroll
        for (int i = 1; i < kGroups; ++i) top = fmaxf(top, stats[i][0]);
        float total = 0.f, v = 0.f;
#pragma unroll
        for (int i = 0; i < kGroups; ++i) {
            const float by = fast_exp2(stats[i][0] - top);
            total += by * stats[i][1];
            v += by * sums[i][d];
        }
        out[d] = T::from_float(total != 0.f ? v / total : 0.f);
    }
}

struct Plan {
    int64_t groups;  // work-groups of the walk (0: one per unit, no workspace)
    int64_t share;   // rounds of a share (0: by the lengths)
};

constexpr int64_t kWalkGroups = 1024;  // four per CU: what registers hold at once up to 128 dims
// Units go out whole where they are short: up to 512 tokens the join costs more than it shares out (64 sequences of 512: 9.6
// us whole, 13.9 shared), and where they are many for their length: up to 2048 tokens from 1024 units on (128 ragged
// sequences: 35.7 us whole, 42.3 shared), 4096 from 2048 on (256 ragged ones: 125 us, 154), and so on; 512 units of up to
// 4096 are shared (33.9 us, 45.2 whole).  The rule sees the tables' width and not the lengths.  Whole, one long sequence among
// short ones is walked alone at 1.06 us per 128 tokens: one of 2048 tokens and 127 of 16 take 21 us, where sharing takes 14
// (all 128 of 16 tokens: 5.7).  That much the rule gives up there for what it gains on batches of mostly long ones.
constexpr int64_t kShortRounds = 4, kManyUnits = 1024, kManyRounds = 16;
constexpr int64_t kMostRounds = int64_t(1) << 30;

bool decode_shape(int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t block_size,
                  int64_t width) {
    return batch > 0 && q_heads > 0 && kv_heads > 0 && q_heads % kv_heads == 0 && attention_dim(head_dim) &&
           valid_format(block_size, head_dim) && width > 0 && width <= kMaxCapacity / block_size &&
           batch <= 2147483647 / q_heads;
}

// From shapes alone (lengths stay on the device).
Plan plan(int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t block_size, int64_t width, int64_t partition_tokens) {
    const int64_t capacity = block_size * width;
    const int64_t units = batch * kv_heads * ((q_heads / kv_heads + 15) / 16);
    const int64_t rounds = (capacity - 1) / kRound + 1;  // of a unit, at most
    if (partition_tokens > 0) {
        if (partition_tokens >= capacity) return {0, 0};  // (before it is added to: it may be any number)
        const int64_t share = (partition_tokens + kRound - 1) / kRound;
        // (Rounds are counted in 32 bits; the call refuses more.)
        return {units * rounds > kMostRounds ? kMostRounds + 1 : (units * rounds - 1) / share + 1, share};
    }
    if (rounds <= kShortRounds || units * rounds > kMostRounds || rounds <= units / kManyUnits * kManyRounds)
        return {0, 0};
    return {units * rounds < kWalkGroups ? units * rounds : kWalkGroups, 0};
}

template <typename T, int D>
int launch(const DecodeArgs& a, int64_t units, hipStream_t s) {
    const dim3 grid((unsigned)(a.groups ? a.groups : units)), block(64 * kWaves);
    if (a.div.size % 32 == 0) hipLaunchKernelGGL((fp4_decode_kernel<T, D, 32>), grid, block, 0, s, a);
    else if (a.div.size % 16 == 0) hipLaunchKernelGGL((fp4_decode_kernel<T, D, 16>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((fp4_decode_kernel<T, D, 1>), grid, block, 0, s, a);
    if (int rc = check_launch("packed decode")) return rc;
    if (a.groups == 0) return MVME_OK;
    hipLaunchKernelGGL((fp4_merge_kernel<T, D>), dim3((unsigned)(a.batch * a.q_heads)), dim3(kMergeThreads), 0, s, a);
    return check_launch("packed decode merge");
}

template <typename T>
int launch_dim(const DecodeArgs& a, int64_t head_dim, int64_t units, hipStream_t s) {
    switch (head_dim) {
        case 32: return launch<T, 32>(a, units, s);
        case 64: return launch<T, 64>(a, units, s);
        case 96: return launch<T, 96>(a, units, s);
        case 128: return launch<T, 128>(a, units, s);
        case 192: return launch<T, 192>(a, units, s);
        default: return launch<T, 256>(a, units, s);
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
    const Plan p = plan(batch, q_heads, kv_heads, block_size, table_width, partition_tokens);
    // Two pieces of up to 16 heads a share.
    return (size_t)p.groups * 2 * 16 * (size_t)(head_dim + 2) * sizeof(float);
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
    if (num_blocks > 2147483647 || num_blocks > (int64_t(1) << 62) / record / kv_heads)
        return fail(MVME_EINVAL, "KV cache too large");
    if (!out || !query || !key_cache || !value_cache || !block_tables || !context_lens)
        return fail(MVME_EINVAL, "packed decode: null pointer");
    if (!aligned(query, 16) || !aligned(key_cache, 16) || !aligned(value_cache, 16) || !aligned(out, 2))
        return fail(MVME_EINVAL, "packed decode: query and caches must be 16-byte aligned");
    if (partition_tokens < 0) return fail(MVME_EINVAL, "partition_tokens must not be negative");
    const Plan p = plan(batch, q_heads, kv_heads, block_size, table_width, partition_tokens);
    const int64_t tiles = (q_heads / kv_heads + 15) / 16, units = batch * kv_heads * tiles;
    if (units > kMostThreads / (64 * kWaves)) return fail(MVME_EINVAL, "batch/head product too large");
    if (p.groups > kMostThreads / (64 * kWaves) || (p.groups && batch * q_heads > kMostThreads / kMergeThreads))
        return fail(MVME_EINVAL, "too many partitions");
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
    a.pieces = static_cast<float*>(workspace);
    a.num_blocks = num_blocks;
    a.record = record;
    a.page_bytes = (uint64_t)(record * kv_heads);
    a.stats = p.groups * 2 * 16 * head_dim;
    a.batch = (int)batch;
    a.kv_heads = (int)kv_heads;
    a.q_heads = (int)q_heads;
    a.group = (int)(q_heads / kv_heads);
    a.width = (int)table_width;
    a.head_tiles = (int)tiles;
    a.groups = (int)p.groups;
    a.share = (int)p.share;
    a.div = make_block_div(block_size);
    a.scale = kLog2e / __builtin_sqrtf((float)head_dim);
    hipStream_t s = static_cast<hipStream_t>(stream);
    return dtype == MVME_FP16 ? launch_dim<Half>(a, head_dim, units, s)
                              : launch_dim<BFloat16>(a, head_dim, units, s);
}
