// Decode attention over 16-bit pages whose prefixes may be shared, and whose
// weights may be kept: the walk that hands out the work, and the two kinds of
// tiles.  Matrix tiles and the softmax's reference are those of
// fp4_attention.h.
//
// A unit is what has the same keys: the rows of one group (its sequences'
// query heads of one kv head) over the group's prefix, or one sequence's query
// heads of one kv head over its own keys.  All units are laid end to end and
// cut into equal shares (in rounds of 128 keys), one per work-group; a second
// kernel joins the pieces.  Groups of more than kNarrowRows rows are taken 128
// rows at a time (wide: a wave has 32 rows, tiles of keys and values in LDS
// serve all four waves), everything else 16 rows at a time (narrow: the waves
// take tiles of 32 keys in turn).
#pragma once

#include <algorithm>

#include "fp4_attention.h"

namespace mvme {
namespace lng {

using fp4::BlockDiv;
using fp4::kRefBelow;
using fp4::kRefNone;
using fp4::kRefSlack;
using fp4::kTileKeys;
using fp4::TileAddress;
using fp4::uniform_load;
using fp4::value_operand;

typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kThreads = 256, kWaves = 4;
constexpr int kRound = 128;       // keys of a round: a narrow tile for every wave, or two wide tiles
constexpr int kWideRows = 128;    // rows of a wide unit
constexpr int kWideKeys = 64;     // keys of a wide tile
constexpr int kNarrowRows = 32;   // a group with more rows is wide
constexpr int kColumns = 16;      // rows of a narrow unit
constexpr int64_t kMaxCapacity = fp4::kMaxCapacity;

struct Args {
    void* out;
    const void* query;
    const uint8_t* key;
    const uint8_t* value;
    const int64_t* tables;
    const int64_t* lens;
    const int64_t* offsets;   // [groups + 1]; rows of a group
    const int64_t* prefixes;  // [groups]; tokens that they share
    float* wide;              // [wide slots, 128, D] sums, then [wide slots, 128, 2] (reference, sum)
    float* narrow;            // [narrow slots, 16, D], then [narrow slots, 16, 2]
    float* totals;            // [batch, q_heads, 2]: (reference, sum) of units that one share holds (scores only)
    float* scores;            // [batch, kv_heads, score_row / 4, group, 4] dot products (scores only)
    float* weights;           // [batch, kv_heads, weight_row]
    int64_t weight_row, score_row;  // (score rows are a multiple of 32 long)
    int64_t wide_slots, narrow_slots;
    int64_t num_blocks;
    uint64_t page_bytes;
    uint32_t row_bytes;       // of a token: kv_heads * D * 2
    int batch, groups, kv_heads, group, q_heads, width;
    int head_tiles;           // ceil(group / 16)
    int shares;               // work-groups of the walk
    BlockDiv div, group_div;
    float scale;              // log2(e) / sqrt(D)
};

template <int D>
struct Shape {
    static constexpr int kDim = (D + 31) / 32 * 32;      // padded with zeros
    static constexpr int kChunks = kDim / 32;            // 16-byte pieces of a lane's part of a token
    static constexpr int kDimTiles = kDim / 16;
    static constexpr int kTileBytes = kTileKeys * 2 * kDim;  // a narrow tile's values; as large as its 16 rows of sums
    static constexpr int kBlocks = kDim / 32;            // 32-dim blocks of a wide unit's sums
    static constexpr int kSteps = kDim / 16;
    static constexpr int kWidePlane = kWideKeys * 2 * kDim;
};

// Barrier of the work-group for LDS alone: loads from memory stay in flight.
__device__ inline void lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

__device__ inline int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// ---------------------------------------------------------------------------
// The walk.  Every wave computes the same, lane-parallel over the groups or sequences.  Order: kv heads; of each the wide
// units, the narrow units of groups, the sequences' units.
// ---------------------------------------------------------------------------
// What a lane holds of a group.
struct Group {
    int first, rows;     // sequences
    int prefix;          // tokens; 0: nothing is shared
    bool wide;           // (units take prefix_taken() of them)
    int rounds, tiles;   // of a unit, and units
};
// What a lane holds of a sequence.
struct Own {
    int len;             // 0 where the length cannot be
    int start;           // where its own keys begin: behind what its group's units take, if it has the whole prefix
    __device__ inline int rounds() const { return (len - start + kRound - 1) / kRound; }
};

struct Walk {
    bool grouped;                     // the offsets can be
    int wide_units, narrow_units;     // of a kv head, of groups
    int wide_rounds, narrow_rounds;   // the same in rounds
    int total;                        // rounds of a kv head
    int shares;                       // one per work-group, from the first on
    int share, longer;                // rounds of a share; the first `longer` shares have one more
    Group group0;                     // of group `lane`
    Own own0;                         // of sequence `lane`

    __device__ static inline int64_t capacity(const Args& a) { return (int64_t)a.width * a.div.size; }

    // How much of a prefix a group's units take.  Where pages are looked up once for 16 tokens (RUN 16) these have to lie in
    // one page, so that every segment, a sequence's own too, has to begin at a multiple of 16: the rest of the prefix is
    // among each sequence's own keys.
    __device__ static inline int prefix_taken(const Args& a, int prefix) { return a.div.size % 16 == 0 ? prefix & ~15 : prefix; }

    __device__ static inline Group group_from(const Args& a, int64_t first, int64_t next, int64_t prefix) {
        Group x{(int)first, (int)(next - first), 0, false, 0, 0};
        // (One row alone gains nothing, and needs no unit for it.)
        const int taken = x.rows >= 2 && prefix > 0 && prefix <= capacity(a) ? prefix_taken(a, (int)prefix) : 0;
        x.prefix = taken ? (int)prefix : 0;
        const int64_t rows = (int64_t)x.rows * a.group;
        x.wide = rows > kNarrowRows;
        x.rounds = (taken + kRound - 1) / kRound;
        x.tiles = x.prefix ? (int)(x.wide ? (rows + kWideRows - 1) / kWideRows : (rows + kColumns - 1) / kColumns) : 0;
        return x;
    }
    // Group g0 + lane.
    __device__ inline Group group(const Args& a, int g0) const {
        const int g = g0 + __lane_id();
        if (g0 == 0) return group0;
        if (!grouped || g >= a.groups) return Group{0, 0, 0, false, 0, 0};
        return group_from(a, a.offsets[g], a.offsets[g + 1], a.prefixes[g]);
    }
    // Group g, for every lane.
    __device__ inline Group group_at(const Args& a, int g) const {
        if (g >= kWave) return group_from(a, a.offsets[g], a.offsets[g + 1], a.prefixes[g]);
        return Group{lane_value(group0.first, g), lane_value(group0.rows, g), lane_value(group0.prefix, g),
                     (bool)lane_value((int)group0.wide, g), lane_value(group0.rounds, g), lane_value(group0.tiles, g)};
    }
    // The prefix of the group that a sequence is in, 0 without one, and that group (-1).
    __device__ inline int prefix_of(const Args& a, int seq, int& g) const {
        g = -1;
        if (!grouped) return 0;
        int prefix = 0;
        if (a.groups <= kWave) {
            for (int i = 0; i < a.groups; ++i) {
                const int behind = seq - lane_value(group0.first, i);
                if (behind >= 0 && behind < lane_value(group0.rows, i)) {
                    prefix = lane_value(group0.prefix, i);
                    g = i;
                }
            }
            return prefix;
        }
        int low = 0, high = a.groups;  // the last offset that is not above seq
        while (high - low > 1) {
            const int mid = (low + high) >> 1;
            if (a.offsets[mid] <= seq) low = mid;
            else high = mid;
        }
        const int64_t first = a.offsets[low], next = a.offsets[low + 1];
        if (first > seq || seq >= next) return 0;
        g = low;
        return group_from(a, first, next, a.prefixes[low]).prefix;
    }
    __device__ static inline int length_from(const Args& a, int64_t n) { return n > 0 && n <= capacity(a) ? (int)n : 0; }
    __device__ inline Own own_from(const Args& a, int seq, int64_t length) const {
        Own x{length_from(a, length), 0};
        int g;
        const int prefix = prefix_of(a, seq, g);
        // (By the whole prefix: who has less of it need not have even the beginning in the same pages.)
        x.start = prefix <= x.len ? prefix_taken(a, prefix) : 0;
        return x;
    }
    __device__ static inline int64_t load_length(const Args& a, int seq) { return seq < a.batch ? a.lens[seq] : 0; }
    // Sequence s0 + lane.
    __device__ inline Own own(const Args& a, int s0) const {
        return s0 == 0 ? own0 : own_from(a, s0 + __lane_id(), load_length(a, s0 + __lane_id()));
    }
    // Sequence s, for every lane.
    __device__ inline Own own_at(const Args& a, int s) const {
        if (s < kWave) return Own{lane_value(own0.len, s), lane_value(own0.start, s)};
        return own_from(a, s, a.lens[s]);
    }

    __device__ inline void count(const Args& a) {
        const int lane = __lane_id();
        wide_units = narrow_units = wide_rounds = narrow_rounds = total = 0;
        // All that is needed first, in one round trip.
        const int64_t length0 = load_length(a, lane);
        int64_t first = 0, next = 0, prefix = 0, end = 0;
        if (lane < a.groups) {
            first = a.offsets[lane];
            next = a.offsets[lane + 1];
            prefix = a.prefixes[lane];
        }
        if (a.groups > 0) end = a.offsets[a.groups];
        grouped = a.groups > 0;
        if (grouped) {
            bool good = lane >= a.groups || first <= next;
            if (lane == 0) good = good && first >= 0 && end <= a.batch;
            for (int g = kWave + lane; g < a.groups; g += kWave) good = good && a.offsets[g] <= a.offsets[g + 1];
            grouped = __all(good);
        }
        group0 = grouped && lane < a.groups ? group_from(a, first, next, prefix) : Group{0, 0, 0, false, 0, 0};
        if (grouped)
            for (int g0 = 0; g0 < a.groups; g0 += kWave) {
                const Group x = group(a, g0);
                const int w = x.wide ? x.tiles : 0, n = x.wide ? 0 : x.tiles;
                wide_units += lane_value(wave_incl_scan(w), kWave - 1);
                narrow_units += lane_value(wave_incl_scan(n), kWave - 1);
                wide_rounds += lane_value(wave_incl_scan(w * x.rounds), kWave - 1);
                narrow_rounds += lane_value(wave_incl_scan(n * x.rounds), kWave - 1);
            }
        own0 = own_from(a, lane, length0);
        int rounds = 0;
        for (int s0 = 0; s0 < a.batch; s0 += kWave) rounds += lane_value(wave_incl_scan(own(a, s0).rounds()), kWave - 1);
        total = wide_rounds + narrow_rounds + rounds * a.head_tiles;
        // Shares differ by a round at most, the first ones are longer.  They have two rounds at least where that leaves every
        // compute unit one: more pieces cost the join more than they save.
        const int all = total * a.kv_heads;
        shares = max(min(a.shares, max(all / 2, min(all, 256))), 1);
        shares = min(shares, all);  // (none where there are no rounds)
        share = shares > 0 ? all / shares : 0;
        longer = all - share * shares;
    }
    // The share of this work-group, or -1: consecutive shares are on one XCD (work-groups are dealt to these in turn), whose L2
    // then has keys that several row tiles of a group read at about the same time (128 sequences over 16384 tokens 82 us, 85
    // with shares in the order of the work-groups; where nothing is read twice that order is ahead, by one in a hundred).
    __device__ inline int mine() const {
        const int per = (shares + 7) / 8, at = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
        return (int)(blockIdx.x >> 3) < per && at < shares ? at : -1;
    }
    // First round of a work-group's share.
    __device__ inline int first_of(int wg) const { return wg * share + min(wg, longer); }
    // The work-group in whose share a round is.
    __device__ inline int owner(int round) const {
        const int until = longer * (share + 1);
        return round < until ? round / (share + 1) : longer + (round - until) / max(share, 1);
    }

    // The sequence whose table names a group's prefix: the first that reaches to its end.  (If none does, no row uses it.)
    __device__ inline int reader_of(const Args& a, const Group& x) const {
        const int lane = __lane_id();
        for (int s0 = x.first & -kWave; s0 < x.first + x.rows; s0 += kWave) {
            const int seq = s0 + lane, len = s0 == 0 ? own0.len : length_from(a, load_length(a, seq));
            const uint64_t hit = __ballot(seq >= x.first && seq < x.first + x.rows && len >= x.prefix);
            if (hit) return s0 + __builtin_ctzll(hit);
        }
        return x.first;
    }
    // The units of `group` begin at round `base` of a kv head, and number `unit` among their kind.
    __device__ inline void place_of_group(const Args& a, int g, bool wide, int& base, int& unit) const {
        const int lane = __lane_id();
        base = unit = 0;
        for (int g0 = 0; g0 < g; g0 += kWave) {
            const Group x = group(a, g0);
            const bool counts = g0 + lane < g && x.wide == wide;
            base += lane_value(wave_incl_scan(counts ? x.tiles * x.rounds : 0), kWave - 1);
            unit += lane_value(wave_incl_scan(counts ? x.tiles : 0), kWave - 1);
        }
        if (!wide) base += wide_rounds;
    }
    // First round, in its kv head, of a sequence's own units.
    __device__ inline int place_of_sequence(const Args& a, int seq) const {
        const int lane = __lane_id();
        int base = 0;
        for (int s0 = 0; s0 < seq; s0 += kWave)
            base += lane_value(wave_incl_scan(s0 + lane < seq ? own(a, s0).rounds() : 0), kWave - 1);
        return wide_rounds + narrow_rounds + base * a.head_tiles;
    }
};

// A run of rounds of one unit: what a work-group does at a time.  Wave-uniform.
struct Segment {
    int seq;              // whose pages
    int kv_head, tile;
    int first_row;        // of the group's sequences; -1: the sequence's own keys
    int rows;             // rows of the unit from the tile's first on
    uint32_t begin, end;  // keys
    int slot;             // where its piece goes; -1: it is all that its rows have
    int rounds;
    bool wide;
};

__device__ inline Segment find_segment(const Args& a, const Walk& w, int wg, int at, int stop) {
    Segment s;
    s.kv_head = at / w.total;
    int q = at - s.kv_head * w.total;
    int from, rounds, tokens, start = 0;
    const int units = w.narrow_units + a.batch * a.head_tiles;
    if (q < w.wide_rounds + w.narrow_rounds) {
        s.wide = q < w.wide_rounds;
        if (!s.wide) q -= w.wide_rounds;
        int before = 0, units_before = 0, g = 0, base = 0, unit = 0;
        for (int g0 = 0; g0 < a.groups; g0 += kWave) {
            const Group x = w.group(a, g0);
            const int tiles = x.wide == s.wide ? x.tiles : 0;
            const int incl = before + wave_incl_scan(tiles * x.rounds), incl_units = units_before + wave_incl_scan(tiles);
            const uint64_t hit = __ballot(incl > q);
            if (hit) {
                const int at_lane = __builtin_ctzll(hit);
                g = g0 + at_lane;
                base = lane_value(incl - tiles * x.rounds, at_lane);
                unit = lane_value(incl_units - tiles, at_lane);
                break;
            }
            before = lane_value(incl, kWave - 1);
            units_before = lane_value(incl_units, kWave - 1);
        }
        const Group x = w.group_at(a, g);
        rounds = max(x.rounds, 1);
        s.tile = (q - base) / rounds;
        from = q - base - s.tile * rounds;
        tokens = Walk::prefix_taken(a, x.prefix);
        s.seq = w.reader_of(a, x);
        s.first_row = x.first;
        s.rows = x.rows * a.group - s.tile * (s.wide ? kWideRows : kColumns);
        unit += s.tile;
        s.slot = (s.wide ? s.kv_head * w.wide_units : s.kv_head * units) + unit + wg;
    } else {
        q -= w.wide_rounds + w.narrow_rounds;
        s.wide = false;
        s.first_row = -1;
        int before = 0, base = 0;
        s.seq = 0;
        for (int s0 = 0; s0 < a.batch; s0 += kWave) {
            const int mine = w.own(a, s0).rounds() * a.head_tiles, incl = before + wave_incl_scan(mine);
            const uint64_t hit = __ballot(incl > q);
            if (hit) {
                const int at_lane = __builtin_ctzll(hit);
                s.seq = s0 + at_lane;
                base = lane_value(incl - mine, at_lane);
                break;
            }
            before = lane_value(incl, kWave - 1);
        }
        const Own own = w.own_at(a, uniform(s.seq));
        start = own.start;
        tokens = own.len - start;
        rounds = max(own.rounds(), 1);
        s.tile = (q - base) / rounds;
        from = q - base - s.tile * rounds;
        s.rows = a.group - s.tile * kColumns;
        s.slot = s.kv_head * units + w.narrow_units + s.seq * a.head_tiles + s.tile + wg;
    }
    const int n = min(rounds - from, stop - at);
    if (s.first_row < 0 && start == 0 && n == rounds) s.slot = -1;
    s.begin = (uint32_t)(start + from * kRound);
    s.end = (uint32_t)(start + min(tokens, (from + n) * kRound));
    s.rounds = n;
    // (Uniform all along, but only now provably so: what these address is loaded and computed once per wave.)
    s.seq = uniform(s.seq);
    s.kv_head = uniform(s.kv_head);
    s.tile = uniform(s.tile);
    s.first_row = uniform(s.first_row);
    s.rows = uniform(s.rows);
    s.begin = (uint32_t)uniform((int)s.begin);
    s.end = (uint32_t)uniform((int)s.end);
    s.slot = uniform(s.slot);
    s.rounds = uniform(s.rounds);
    s.wide = uniform(s.wide);
    return s;
}

// Query head (of all) of a unit's row: rows of a group are its (sequence, head) pairs, sequence by sequence.
__device__ inline int64_t head_of(const Args& a, const Segment& s, int row) {
    if (s.first_row < 0) return (int64_t)s.seq * a.q_heads + s.kv_head * a.group + row;
    const int seq = (int)a.group_div.page((uint32_t)row);
    return (int64_t)(s.first_row + seq) * a.q_heads + s.kv_head * a.group + (row - seq * a.group);
}

// ---------------------------------------------------------------------------
// Narrow tiles: 16 rows, 32 keys, of one wave alone.  Loads take whole rows of memory; both planes go through LDS, keys to
// become operands of the score product, values for their transposition.
// ---------------------------------------------------------------------------
// RUN tokens (block sizes that are multiples of it) lie in one page at consecutive places.  RUN 16: a tile's halves are
// looked up by the whole wave; RUN 1: lane i looks up token i of the tile.
template <int RUN>
struct Where {
    int64_t at[RUN == 16 ? 2 : 1];  // byte offset of the half's first (the lane's) token in a plane, or of one that exists
    uint32_t present;               // the tile's tokens that are there
};
template <int RUN>
struct Pages {
    int64_t page[RUN == 16 ? 2 : 1];
};
template <int RUN>
__device__ inline Pages<RUN> load_pages(const Args& a, const int64_t* table, uint32_t first) {
    Pages<RUN> p;
#pragma unroll
    for (int s = 0; s < (RUN == 16 ? 2 : 1); ++s) {
        const uint32_t token = first + (RUN == 16 ? 16 * s : (int)(threadIdx.x & 31));
        const int64_t* entry = table + min(a.div.page(token), (uint32_t)a.width - 1u);
        p.page[s] = RUN == 1 ? *entry : uniform_load(entry);
    }
    return p;
}
template <int RUN>
__device__ inline Where<RUN> look_up(const Args& a, const Pages<RUN>& p, int64_t head_at, uint32_t first, uint32_t end) {
    Where<RUN> w;
    const uint32_t left = end > first ? end - first : 0u;
    w.present = left >= 32 ? 0xffffffffu : (1u << left) - 1u;
#pragma unroll
    for (int s = 0; s < (RUN == 16 ? 2 : 1); ++s) {
        const uint32_t token = first + (RUN == 16 ? 16 * s : (int)(threadIdx.x & 31)), block = a.div.page(token);
        const bool there = token < end && (uint64_t)p.page[s] < (uint64_t)a.num_blocks;
        const uint32_t page = there ? (uint32_t)p.page[s] : 0u, place = there ? token - block * a.div.size : 0u;
        w.at[s] = head_at + (int64_t)((uint64_t)page * a.page_bytes) + (int64_t)((uint64_t)place * a.row_bytes);
        if constexpr (RUN == 16) w.present &= there ? 0xffffffffu : s ? 0x0000ffffu : 0xffff0000u;
        else w.present = (uint32_t)__ballot(there);
    }
    return w;
}

// What a lane loads of a half tile (16 tokens): pieces of 16 bytes, the i-th being number lane + 64 i of the half's.
template <int D>
struct Lines {
    using S = Shape<D>;
    static constexpr int kRow = S::kDim / 8;  // pieces of a row
    uint32_t from[S::kChunks];  // byte offset from the half's first token (RUN 1: in its row)
    int to[S::kChunks];         // in a tile
    int row[S::kChunks];
    bool real[S::kChunks];      // not padding
    __device__ inline Lines(uint32_t row_bytes) {
#pragma unroll
        for (int i = 0; i < S::kChunks; ++i) {
            const int piece = (threadIdx.x & 63) + 64 * i, chunk = piece % kRow;
            row[i] = piece / kRow;
            from[i] = row[i] * row_bytes + chunk * 16;
            to[i] = fp4::TileLayout<S::kDim, 16>::at(row[i], chunk);
            real[i] = D == S::kDim || chunk * 8 < D;
        }
    }
};

template <int D, int RUN>
__device__ inline void load_tile(u32x4 (&x)[2][Shape<D>::kChunks], const uint8_t* plane, const Where<RUN>& w,
                                 const Lines<D>& l, uint32_t row_bytes) {
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int i = 0; i < Shape<D>::kChunks; ++i) {
            const uint8_t* at;
            if constexpr (RUN == 16) {
                at = plane + w.at[s] + l.from[i];
            } else {
                const int from = (l.row[i] + 16 * s) << 2;
                const uint32_t lo = (uint32_t)__builtin_amdgcn_ds_bpermute(from, (int)(uint32_t)w.at[0]);
                const uint32_t hi = (uint32_t)__builtin_amdgcn_ds_bpermute(from, (int)(uint32_t)((uint64_t)w.at[0] >> 32));
                at = plane + (int64_t)(((uint64_t)hi << 32) | lo) + (l.from[i] - l.row[i] * row_bytes);
            }
            if (D == Shape<D>::kDim || l.real[i]) x[s][i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(at));
            else x[s][i] = u32x4{0u, 0u, 0u, 0u};
        }
}

// Two weights as sums of two numbers of the type each: the upper bits, and the rest rounded: at most 2^-15 (bf16) or 2^-21
// (fp16) of the weight is lost.  The rest is positive, the type's smallest number at least (2^-32 of the largest weight),
// so that an infinite value times a weight is infinite, as in the formula, and not NaN.
template <typename T>
__device__ inline u32x2 split_pair(float x, float y) {
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
    constexpr uint16_t kLeast = T::kId == MVME_FP16 ? 0x0001 : 0x0080;
    uint32_t high;
    if constexpr (T::kId == MVME_FP16)
        high = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(x, y));
    else
        high = __builtin_amdgcn_perm(__float_as_uint(y), __float_as_uint(x), 0x07060302u);
    const uint32_t rest = T::pack(x - T::lo(high), y - T::hi(high));
    const u16x2 low = __builtin_elementwise_max(__builtin_bit_cast(u16x2, rest), u16x2{kLeast, kLeast});
    return u32x2{high, __builtin_bit_cast(uint32_t, low)};
}

constexpr int kRing = 512;  // 16-byte pieces of scores that a wave gathers before it stores them

// The probability that a dot product stands for.  (None where there is no token, whatever the divisor is: another key's NaN
// makes that NaN.)
__device__ inline float probability(const Args& a, float score, float ref, float by) {
    return score == kNegInf ? 0.f : fast_exp2(__builtin_fmaf(score, a.scale, -ref)) * by;
}

// What becomes of a segment's dot products: nothing, they go to memory, or (the segment is a whole unit, and the ring holds
// it) they become weights at its end.
enum Scores { kNoScores, kStoreScores, kAddWeights };

template <int D, Scores SCORES>
struct NarrowLds {
    uint8_t tiles[kWaves][Shape<D>::kTileBytes];  // keys, then values
    f32x4 ring[SCORES ? kWaves : 1][SCORES ? kRing : 1];
    float stats[kWaves][2][kColumns];
    float divisors[2][kColumns];                  // (reference, 1 / sum)
};

// One segment of a narrow unit.
template <typename T, int D, int RUN, Scores SCORES>
__device__ inline void narrow_segment(const Args& a, const Segment& seg, NarrowLds<D, SCORES>& lds) {
    using S = Shape<D>;
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int wave = uniform(threadIdx.x >> 6);
    uint8_t* tile_lds = lds.tiles[wave];
    // An operand's lane (r, g) has key r of a half tile and pieces 4 c + g of 8 dims; the row's pieces likewise.
    TileAddress<S::kDim, 16> key_at(r, g), value_at(4 * g + (r >> 2), (r & 3) >> 1, (r & 1) * 8);
    Lines<D> lines(a.row_bytes);
    const int64_t* table = a.tables + (int64_t)seg.seq * a.width;
    const int64_t head_at = (int64_t)seg.kv_head * (2 * D);
    const int heads = min(kColumns, seg.rows);
    const bool live = r < heads;
    // (Columns without a row repeat the last row: what follows needs no branch for them.)
    const int64_t head = head_of(a, seg, seg.tile * kColumns + min(r, heads - 1));

    // Scores go to memory many tiles at a time: stores among the loads hold these up (a load is done only when the stores
    // before it are).  4 x 65536 tokens, 8 heads per kv head: 119 us, 123 with a store per tile.
    const int per_tile = 8 * heads, ring_tiles = kRing / per_tile;
    int ring_used = 0;
    uint32_t ring_first = 0;  // key of the first tile in the ring
    const auto flush = [&]() {
        f32x4* to = reinterpret_cast<f32x4*>(a.scores) +
                    (int64_t)(seg.seq * a.kv_heads + seg.kv_head) * (a.score_row / 4) * a.group + seg.tile * kColumns;
        for (int i = lane; i < ring_used * per_tile; i += kWave) {
            const int four = i / heads, tile = four >> 3;  // four keys, of 8 in a tile
            to[(int64_t)((ring_first + tile * kRound) / 4 + (four & 7)) * a.group + (i - four * heads)] = lds.ring[SCORES ? wave : 0][i];
        }
        ring_used = 0;
    };

    u32x4 q[S::kChunks], k[2][S::kChunks], v[2][S::kChunks];
    f32x4 acc[S::kDimTiles];
    float ref = kRefNone, sum = 0.f;
#pragma unroll
    for (int n = 0; n < S::kDimTiles; ++n) acc[n] = f32x4{0.f, 0.f, 0.f, 0.f};
    uint32_t t0 = seg.begin + wave * kTileKeys;
    Where<RUN> now;
    Pages<RUN> pages;
    if (t0 < seg.end) {
        now = look_up<RUN>(a, load_pages<RUN>(a, table, t0), head_at, t0, seg.end);
        pages = load_pages<RUN>(a, table, t0 + kRound);  // of the next tile
        load_tile<D, RUN>(k, a.key, now, lines, a.row_bytes);
        load_tile<D, RUN>(v, a.value, now, lines, a.row_bytes);
    }
#pragma unroll
    for (int c = 0; c < S::kChunks; ++c) {
        q[c] = u32x4{0u, 0u, 0u, 0u};
        if (D == S::kDim || (4 * c + g) * 8 < D)
            q[c] = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(a.query) + head * D + (4 * c + g) * 8);
    }
#pragma unroll 1
    for (; t0 < seg.end; t0 += kRound) {
        key_at.forget();
        value_at.forget();
        // (Behind the last tile the loads go on, from a page that exists: a branch around them would make every wait one
        // for all of them.)
        const Where<RUN> next = look_up<RUN>(a, pages, head_at, t0 + kRound, seg.end);
        pages = load_pages<RUN>(a, table, t0 + 2 * kRound);
        const uint32_t present = now.present;
        // A wave reads only what it wrote: the LDS queue is in order, no barrier.  Registers are refilled as soon as they
        // are in LDS.
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int i = 0; i < S::kChunks; ++i)
                *reinterpret_cast<u32x4*>(tile_lds + lines.to[i] + 16 * s * 2 * S::kDim) = k[s][i];
        load_tile<D, RUN>(k, a.key, next, lines, a.row_bytes);
        f32x4 x[2];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            x[s] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < S::kChunks; ++c)
                x[s] = T::mfma16x16x32(*reinterpret_cast<const u32x4*>(tile_lds + key_at.chunk(4 * c) + 16 * s * 2 * S::kDim),
                                       q[c], x[s]);
        }
        // Keys that are not there: no weight, and zeros as values (0 * NaN is NaN).
        if (present != 0xffffffffu) {
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int i = 0; i < S::kChunks; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[s][i][j] = (present >> (16 * s + lines.row[i])) & 1 ? v[s][i][j] : 0u;
        }
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int i = 0; i < S::kChunks; ++i)
                *reinterpret_cast<u32x4*>(tile_lds + lines.to[i] + 16 * s * 2 * S::kDim) = v[s][i];
        load_tile<D, RUN>(v, a.value, next, lines, a.row_bytes);
        if (present != 0xffffffffu) {
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int j = 0; j < 4; ++j) x[s][j] = (present >> (16 * s + 4 * g + j)) & 1 ? x[s][j] : kNegInf;
        }
        if constexpr (SCORES) {
            // Four keys of every head side by side.  (Behind the context there is room: rows are a multiple of 32.)
            if (ring_used == 0) ring_first = t0;
            f32x4* to = lds.ring[wave] + ring_used * per_tile + g * heads + r;
            if (live) {
                to[0] = x[0];
                to[4 * heads] = x[1];
            }
            ++ring_used;
            if (SCORES == kStoreScores && ring_used == ring_tiles) flush();
        }
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
        // A weight is the sum of two 16-bit numbers: the products are there anyhow, and the output's own rounding stays
        // the only one that counts.
        u32x4 high, low;
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int j = 0; j < 4; j += 2) {
                const float p0 = fast_exp2(__builtin_fmaf(x[s][j], a.scale, -ref));
                const float p1 = fast_exp2(__builtin_fmaf(x[s][j + 1], a.scale, -ref));
                const u32x2 both = split_pair<T>(p0, p1);
                high[2 * s + j / 2] = both[0];
                low[2 * s + j / 2] = both[1];
                sum += p0 + p1;
            }
#pragma unroll
        for (int n = 0; n < S::kDimTiles; ++n) {
            const u32x4 vt = value_operand(tile_lds, value_at.chunk(2 * n), value_at.chunk(2 * n) + 16 * 2 * S::kDim);
            acc[n] = T::mfma16x16x32(vt, high, acc[n]);
            acc[n] = T::mfma16x16x32(vt, low, acc[n]);
        }
        now = next;
    }
    if constexpr (SCORES == kStoreScores) flush();
    sum = row4_sum(sum);

    // Join the waves: sums [16][D] in their tiles' LDS, each relative to its own reference.
    float* mine = reinterpret_cast<float*>(tile_lds);
    if (live) {
#pragma unroll
        for (int n = 0; n < S::kDimTiles; ++n) *reinterpret_cast<f32x4*>(mine + r * S::kDim + 16 * n + 4 * g) = acc[n];
        if (g == 0) {
            lds.stats[wave][0][r] = ref;
            lds.stats[wave][1][r] = sum;
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < heads * D; i += kThreads) {
        const int h = i / D, d = i - h * D;
        float top = lds.stats[0][0][h];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) top = fmaxf(top, lds.stats[w][0][h]);
        float total = 0.f, value = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float by = fast_exp2(lds.stats[w][0][h] - top);
            total += by * lds.stats[w][1][h];
            value += by * reinterpret_cast<const float*>(lds.tiles[w])[h * S::kDim + d];
        }
        if (seg.slot < 0) {
            const int64_t to = head_of(a, seg, seg.tile * kColumns + h);
            static_cast<uint16_t*>(a.out)[to * D + d] = T::from_float(total != 0.f ? value / total : 0.f);
            if (SCORES == kStoreScores && d == 0) {
                a.totals[to * 2] = top;
                a.totals[to * 2 + 1] = total;
            }
            if (SCORES == kAddWeights && d == 0) {
                lds.divisors[0][h] = top;
                lds.divisors[1][h] = total != 0.f ? 1.f / total : 0.f;
            }
        } else if (seg.slot < a.narrow_slots) {
            const int64_t slot = (int64_t)seg.slot * kColumns + h;
            a.narrow[slot * D + d] = value;
            if (d == 0) {
                float* stats = a.narrow + a.narrow_slots * kColumns * D + slot * 2;
                stats[0] = top;
                stats[1] = total;
            }
        }
    }
    __syncthreads();  // the tiles are free again
    if constexpr (SCORES == kAddWeights) {
        float* weights = a.weights + ((int64_t)seg.seq * a.kv_heads + seg.kv_head) * a.weight_row;
        for (uint32_t key = 4 * threadIdx.x; key < seg.end; key += 4 * kThreads) {
            const uint32_t tile = key / kTileKeys;
            const f32x4* s = lds.ring[tile % kWaves] + (tile / kWaves * 8 + key / 4 % 8) * heads;
            f32x4 add = {0.f, 0.f, 0.f, 0.f};
            for (int h = 0; h < heads; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    add[i] += probability(a, s[h][i], lds.divisors[0][h], lds.divisors[1][h]);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (key + i < seg.end) weights[key + i] += add[i];
        }
    }
}

// ---------------------------------------------------------------------------
// The join: one work-group per sequence and kv head; four dims of a head per thread, the pieces dealt to what threads are
// left.  A head's pieces are those of its row of the group's unit and those of the sequence's own unit.
// ---------------------------------------------------------------------------
struct Pieces {
    int wide_slot, wide_count;      // of the unit's first piece: the others follow
    int64_t wide_row;
    int prefix_slot, prefix_count, prefix_row;  // a narrow unit of the group
    int own_slot, own_count, own_row;
    int count;
    __device__ inline const float* at(const Args& a, int i, int D, const float*& stats) const {
        if (i < wide_count) {
            const int64_t row = (int64_t)(wide_slot + i) * kWideRows + wide_row;
            stats = a.wide + a.wide_slots * kWideRows * D + row * 2;
            return a.wide + row * D;
        }
        i -= wide_count;
        int64_t row;
        if (i < prefix_count) row = (int64_t)(prefix_slot + i) * kColumns + prefix_row;
        else row = (int64_t)(own_slot + i - prefix_count) * kColumns + own_row;
        stats = a.narrow + a.narrow_slots * kColumns * D + row * 2;
        return a.narrow + row * D;
    }
};

// What all heads of a sequence and kv head have in common.
struct Join {
    Walk w;
    int kv_head, seq;
    Own own;
    int group_base, group_unit;  // of the group's units, if own.start > 0
    Group x;
    int own_base;
    __device__ inline void find(const Args& a, int s, int h) {
        w.count(a);
        seq = s;
        kv_head = h;
        own = w.own_at(a, seq);
        group_base = group_unit = 0;
        x = Group{0, 0, 0, false, 0, 0};
        if (own.start > 0) {
            int g;
            w.prefix_of(a, seq, g);
            x = w.group_at(a, uniform(g));
            w.place_of_group(a, uniform(g), x.wide, group_base, group_unit);
        }
        own_base = w.place_of_sequence(a, seq);
    }
    // False: one share had the whole unit, and wrote the output.
    __device__ inline bool pieces(const Args& a, int head, Pieces& p) const {
        p = Pieces{0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
        const int units = w.narrow_units + a.batch * a.head_tiles;
        if (own.start > 0) {
            const int64_t row = (int64_t)(seq - x.first) * a.group + head;
            const int per = x.wide ? kWideRows : kColumns, tile = (int)(row / per);
            const int at = kv_head * w.total + group_base + tile * x.rounds;
            const int first = w.owner(at), last = w.owner(at + x.rounds - 1);
            if (x.wide) {
                p.wide_slot = kv_head * w.wide_units + group_unit + tile + first;
                p.wide_count = last - first + 1;
                p.wide_row = row - (int64_t)tile * per;
            } else {
                p.prefix_slot = kv_head * units + group_unit + tile + first;
                p.prefix_count = last - first + 1;
                p.prefix_row = (int)(row - (int64_t)tile * per);
            }
        }
        const int rounds = own.rounds();
        if (rounds > 0) {
            const int tile = head / kColumns;
            const int at = kv_head * w.total + own_base + tile * rounds;
            const int first = w.owner(at), last = w.owner(at + rounds - 1);
            if (own.start == 0 && first == last) return false;
            p.own_slot = kv_head * units + w.narrow_units + seq * a.head_tiles + tile + first;
            p.own_count = last - first + 1;
            p.own_row = head - tile * kColumns;
        }
        p.count = p.wide_count + p.prefix_count + p.own_count;
        return true;
    }
};

template <typename T, int D>
__device__ inline void join_heads(const Args& a, int seq, int kv_head) {
    constexpr int kLanes = D / 4, kGroups = kThreads / kLanes;
    __shared__ __attribute__((aligned(16))) float sums[kGroups][D];
    __shared__ float stats[kGroups][2];
    Join j;
    j.find(a, seq, kv_head);
    const int heads = min(a.group, kGroups), parts = kGroups / heads;
    const int group = threadIdx.x / kLanes, lane = threadIdx.x % kLanes;
    const int part = group / heads;
    for (int h0 = 0; h0 < a.group; h0 += heads) {
        const int head = h0 + group % heads;
        const bool mine = group < kGroups && part < parts && head < a.group;
        Pieces p;
        const bool joins = mine && j.pieces(a, head, p);
        f32x4 value = {0.f, 0.f, 0.f, 0.f};
        float ref = kRefNone, sum = 0.f;
        if (joins) {
#pragma unroll 4
            for (int i = part; i < p.count; i += parts) {
                const float* s;
                const f32x4 v = *reinterpret_cast<const f32x4*>(p.at(a, i, D, s) + 4 * lane);
                const float top = fmaxf(ref, s[0]), keep = fast_exp2(ref - top), by = fast_exp2(s[0] - top);
                value = value * keep + v * by;
                sum = sum * keep + s[1] * by;
                ref = top;
            }
        }
        __syncthreads();  // (the pass before has read the sums)
        if (group < kGroups) {
            *reinterpret_cast<f32x4*>(&sums[group][4 * lane]) = value;
            if (lane == 0) {
                stats[group][0] = ref;
                stats[group][1] = sum;
            }
        }
        __syncthreads();
        if (joins && part == 0) {
            for (int i = 1; i < parts; ++i) {
                const int other = group + i * heads;
                const float top = fmaxf(ref, stats[other][0]);
                const float keep = fast_exp2(ref - top), by = fast_exp2(stats[other][0] - top);
                value = value * keep + *reinterpret_cast<const f32x4*>(&sums[other][4 * lane]) * by;
                sum = sum * keep + stats[other][1] * by;
                ref = top;
            }
            const float by = 1.f / sum;
            const f32x4 v = sum != 0.f ? value * by : f32x4{0.f, 0.f, 0.f, 0.f};
            const int64_t to = (int64_t)seq * a.q_heads + kv_head * a.group + head;
            u32x2 out = {T::pack(v[0], v[1]), T::pack(v[2], v[3])};
            *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(a.out) + to * D + 4 * lane) = out;
        }
    }
}

inline bool head_dim_built(int64_t d) {
    return d == 16 || d == 32 || d == 64 || d == 80 || d == 96 || d == 128 || d == 192 || d == 256;
}

constexpr int64_t kMostBatchHeads = kMostThreads / kThreads;

// The checks that the decode entry points make of their shapes, and what follows from these.
inline int check_shape(Args& a, int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t num_blocks,
                       int64_t block_size, int64_t table_width, int dtype) {
    if (!valid_dtype(dtype)) return fail(MVME_EINVAL, "FP16/BF16 required");
    if (batch <= 0 || q_heads <= 0 || kv_heads <= 0 || num_blocks <= 0) return fail(MVME_EINVAL, "empty batch/heads/cache");
    if (q_heads % kv_heads != 0) return fail(MVME_EINVAL, "head dimension or GQA mismatch");
    if (!head_dim_built(head_dim)) return fail(MVME_EINVAL, "supported head_dim: 16,32,64,80,96,128,192,256");
    if (block_size <= 0 || table_width <= 0) return fail(MVME_EINVAL, "invalid block table");
    if (block_size > kMaxCapacity || table_width > kMaxCapacity / block_size)
        return fail(MVME_EINVAL, "maximum table capacity is 1M tokens");
    if (q_heads > kMostBatchHeads || batch > kMostBatchHeads / q_heads) return fail(MVME_EINVAL, "batch/head product too large");
    // Positions in the walk are 32-bit: a sequence's own units, and at most as many again of its group (narrow units of
    // whose rows the last may be partial).
    const int64_t group = q_heads / kv_heads, rounds = (block_size * table_width - 1) / kRound + 1;
    if (batch * kv_heads * ((group - 1) / kColumns + 1) * 3 > (int64_t(1) << 30) / rounds)
        return fail(MVME_EINVAL, "too many cached tokens for one call");
    const int64_t row = kv_heads * head_dim * 2;
    if (row > 65536 * 16 || num_blocks > 2147483647 || num_blocks > (int64_t(1) << 62) / row / block_size)
        return fail(MVME_EINVAL, "KV cache too large");
    a.num_blocks = num_blocks;
    a.page_bytes = (uint64_t)(row * block_size);
    a.row_bytes = (uint32_t)row;
    a.batch = (int)batch;
    a.kv_heads = (int)kv_heads;
    a.q_heads = (int)q_heads;
    a.group = (int)group;
    a.width = (int)table_width;
    a.head_tiles = (int)((group - 1) / kColumns + 1);
    a.div = fp4::make_block_div(block_size);
    a.group_div = fp4::make_block_div(group);
    a.scale = kLog2e / __builtin_sqrtf((float)head_dim);
    return MVME_OK;
}

}  // namespace lng
}  // namespace mvme
