// Eviction from a paged cache: of every layer, sequence and kv head the tokens
// that are kept are chosen and their rows moved to the front, in order.
//
// The choice is a radix select, four passes over a row of weights in registers,
// then a prefix sum that ranks what is kept (read again by every pass, with a prefix
// sum per 512 tokens, one layer of 16 ragged sequences took 21.0 us, and 18.8 so).
// The moves are bound by HBM, reads and writes alike.  28 layers of 8 sequences of
// 2048 tokens, half kept, 8 heads of 128: 417 us for 0.94 GB moved, 4.5 TB/s with
// the choice, about the rate of a large copy without.
#include "../../include/mvme_long.h"
#include "fp4_cache.h"

namespace mvme {
namespace evict {
namespace {

using fp4::BlockDiv;
constexpr int64_t kMaxCapacity = fp4::kMaxCapacity;

struct Args {
    uint8_t* key;
    uint8_t* value;
    const float* weights;   // [layers, batch, kv_heads, row]
    float* new_weights;     // the same
    int64_t* kept;          // [layers, batch, kv_heads, columns]
    int64_t* new_lens;      // [batch]
    const int64_t* tables;
    const int64_t* lens;
    const int64_t* first;   // [batch], or null: none
    int64_t row, columns, keep, recent;
    int64_t num_blocks;
    uint64_t layer_bytes, page_bytes;
    uint32_t row_bytes, head_bytes;
    int batch, kv_heads, width;
    int slices, slice_bytes;   // of a head's row
    int units, rows;           // 16-byte units of a slice; rows that the threads hold at a time
    BlockDiv div;
};

__device__ inline int length(const Args& a, int seq) {
    const int64_t n = a.lens[seq];
    return n > 0 && n <= (int64_t)a.width * a.div.size ? (int)n : 0;
}

// ---------------------------------------------------------------------------
// The choice: one work-group per layer, sequence and kv head.
// ---------------------------------------------------------------------------
constexpr int kCopies = 8;  // of the histogram: weights fall into few bins, and lanes that meet in one wait for each other

// Weights in their order as unsigned numbers: NaN above all, -0 equal to +0.
__device__ inline uint32_t rank_of(float x) {
    if (x != x) return 0xffffffffu;
    const uint32_t bits = __float_as_uint(x + 0.f);
    return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}

// Exclusive prefix over the work-group of two counts, and their totals.
__device__ inline void scan_pair(int x, int y, int& before_x, int& before_y, int& all_x, int& all_y, int (*sums)[2],
                                 int waves) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int ix = wave_incl_scan(x), iy = wave_incl_scan(y);
    if (lane == kWave - 1) {
        sums[wave][0] = ix;
        sums[wave][1] = iy;
    }
    __syncthreads();
    before_x = ix - x;
    before_y = iy - y;
    all_x = all_y = 0;
    for (int w = 0; w < waves; ++w) {
        if (w < wave) {
            before_x += sums[w][0];
            before_y += sums[w][1];
        }
        all_x += sums[w][0];
        all_y += sums[w][1];
    }
    __syncthreads();
}

// kHeld > 0: weights are read once, kHeld at most per thread, and a thread's are neighbours, so that one scan ranks all.
// kHeld 0: rows of any length, read again by every pass.
template <int kSelect, int kHeld>
__global__ __launch_bounds__(kSelect) void choose_kernel(Args a) {
    constexpr int kWaves = kSelect / kWave;
    __shared__ int histogram[256][kCopies];
    __shared__ int sums[kWaves][2];
    __shared__ uint32_t chosen[2];
    const int64_t line = blockIdx.x;
    const int seq = (int)(line / a.kv_heads % a.batch);
    const int n = length(a, seq);
    const int count = (int)min((int64_t)n, a.keep);
    const float* w = a.weights + line * a.row;
    float* out = a.new_weights + line * a.row;
    int64_t* kept = a.kept + line * a.columns;
    if (line < (int64_t)a.batch * a.kv_heads && line % a.kv_heads == 0 && threadIdx.x == 0)
        a.new_lens[seq] = n > 0 ? count : a.lens[seq];
    for (int64_t i = count + threadIdx.x; i < a.row; i += kSelect) out[i] = 0.f;
    for (int64_t i = count + threadIdx.x; i < a.columns; i += kSelect) kept[i] = -1;
    if (n <= a.keep) {
        for (int i = threadIdx.x; i < n; i += kSelect) {
            out[i] = w[i];
            kept[i] = i;
        }
        return;
    }
    const int keep = (int)a.keep;
    const int first = a.first ? (int)min(max(a.first[seq], (int64_t)0), (int64_t)keep) : 0;
    const int recent = (int)min(a.recent, (int64_t)(keep - first));
    const int stop = n - recent;  // the weights decide about first .. stop - 1
    int want = keep - first - recent;
    const bool choose = want > 0;
    const int each = kHeld ? (n + kSelect - 1) / kSelect : 0, mine0 = each * (int)threadIdx.x;
    float held[kHeld ? kHeld : 1];
#pragma unroll
    for (int k = 0; k < kHeld; ++k)
        if (k < each) held[k] = w[min(mine0 + k, n - 1)];
    // The want-th largest rank, a byte at a time from the highest: `prefix` is what its upper bytes are.
    uint32_t prefix = 0, mask = 0;
    if (want > 0) {
        for (int shift = 24; shift >= 0; shift -= 8) {
            for (int i = threadIdx.x; i < 256 * kCopies; i += kSelect) histogram[i / kCopies][i % kCopies] = 0;
            __syncthreads();
            const auto count = [&](float x) {
                const uint32_t rank = rank_of(x);
                if ((rank & mask) == prefix) atomicAdd(&histogram[(rank >> shift) & 255][threadIdx.x % kCopies], 1);
            };
            if constexpr (kHeld) {
#pragma unroll
                for (int k = 0; k < kHeld; ++k)
                    if (k < each && mine0 + k >= first && mine0 + k < stop) count(held[k]);
            } else {
                for (int i = first + threadIdx.x; i < stop; i += kSelect) count(w[i]);
            }
            __syncthreads();
            // Bin 255 - t of thread t: the one in which the count from above reaches want.
            int mine = 0;
            if (threadIdx.x < 256)
#pragma unroll
                for (int i = 0; i < kCopies; ++i) mine += histogram[255 - threadIdx.x][i];
            int upto = wave_incl_scan(mine);
            if ((threadIdx.x & 63) == 63 && threadIdx.x < 256) sums[threadIdx.x >> 6][0] = upto;
            __syncthreads();
            if (threadIdx.x < 256) {
                for (int k = 0; k < (int)(threadIdx.x >> 6); ++k) upto += sums[k][0];
                if (upto >= want && upto - mine < want) {
                    chosen[0] = 255 - threadIdx.x;
                    chosen[1] = want - (upto - mine);
                }
            }
            __syncthreads();
            prefix |= chosen[0] << shift;
            mask |= 255u << shift;
            want = (int)chosen[1];
            __syncthreads();
        }
    }
    // Kept: what is protected or above that rank, and the first `want` that equal it.
    const auto sort_out = [&](int i, float x, int& is_above, int& is_level) {
        const bool decided = i < first || i >= stop;
        const uint32_t rank = rank_of(x);
        is_above = i < n && (decided || (choose && rank > prefix));
        is_level = i < n && !decided && choose && rank == prefix;
    };
    int above = 0, level = 0;
    if constexpr (kHeld) {
        int aboves = 0, levels = 0, all_above, all_level;
#pragma unroll
        for (int k = 0; k < kHeld; ++k)
            if (k < each) {
                int is_above, is_level;
                sort_out(mine0 + k, held[k], is_above, is_level);
                aboves += is_above;
                levels += is_level;
            }
        scan_pair(aboves, levels, above, level, all_above, all_level, sums, kWaves);
#pragma unroll
        for (int k = 0; k < kHeld; ++k)
            if (k < each) {
                int is_above, is_level;
                sort_out(mine0 + k, held[k], is_above, is_level);
                if (is_above || (is_level && level < want)) {
                    const int to = above + min(level, want);
                    kept[to] = mine0 + k;
                    out[to] = held[k];
                }
                above += is_above;
                level += is_level;
            }
        return;
    }
    for (int i0 = 0; i0 < n; i0 += kSelect) {
        const int i = i0 + threadIdx.x;
        const float x = w[min(i, n - 1)];
        int is_above, is_level;
        sort_out(i, x, is_above, is_level);
        int before_above, before_level, all_above, all_level;
        scan_pair(is_above, is_level, before_above, before_level, all_above, all_level, sums, kWaves);
        const int levels = level + before_level;
        if (is_above || (is_level && levels < want)) {
            const int to = above + before_above + min(levels, want);
            kept[to] = i;
            out[to] = x;
        }
        above += all_above;
        level += all_level;
    }
}

// ---------------------------------------------------------------------------
// The moves: one work-group per layer, sequence, kv head, plane and slice of the head's row, front to back.  A row never
// moves backwards and order is kept, so what a pass reads lies behind all that earlier passes wrote; within a pass every
// row is read before any is written.
// ---------------------------------------------------------------------------
constexpr int kMove = 256, kPasses = 8;

__global__ __launch_bounds__(kMove) void move_kernel(Args a) {
    __shared__ int64_t from[2][kMove], to[2][kMove];
    int64_t item = blockIdx.x;
    const int slice = (int)(item % a.slices);
    item /= a.slices;
    uint8_t* plane = item % 2 ? a.value : a.key;
    const int64_t line = item / 2;
    const int head = (int)(line % a.kv_heads), seq = (int)(line / a.kv_heads % a.batch);
    const int64_t layer = line / a.kv_heads / a.batch;
    const int n = length(a, seq);
    if (n <= a.keep) return;
    const int count = (int)a.keep;
    const int64_t* kept = a.kept + line * a.columns;
    const int64_t* table = a.tables + (int64_t)seq * a.width;
    plane += layer * a.layer_bytes + (uint64_t)head * a.head_bytes + (uint64_t)slice * a.slice_bytes;
    const int per = kMove / a.units;  // rows that the threads take side by side
    const int side = threadIdx.x / a.units, unit = threadIdx.x % a.units;
    const auto place_of = [&](uint32_t token) {
        const uint32_t block = a.div.page(token);
        const int64_t page = table[block];
        return (uint64_t)page < (uint64_t)a.num_blocks
                   ? (int64_t)((uint64_t)page * a.page_bytes + (uint64_t)(token - block * a.div.size) * a.row_bytes)
                   : (int64_t)-1;
    };
    // This thread's row of a pass: where it comes from and goes to, -1 if it does not move.
    int64_t f, t;
    const auto look_up = [&](int i0) {
        const int i = i0 + threadIdx.x;
        f = t = -1;
        if ((int)threadIdx.x < a.rows && i < count) {
            const int64_t source = kept[i];
            if (source != i) {
                f = place_of((uint32_t)source);
                t = f < 0 ? -1 : place_of((uint32_t)i);
            }
        }
    };
    look_up(0);
    for (int i0 = 0, buffer = 0; i0 < count; i0 += a.rows, buffer ^= 1) {
        if ((int)threadIdx.x < a.rows) {
            from[buffer][threadIdx.x] = f;
            to[buffer][threadIdx.x] = t;
        }
        __syncthreads();
        u32x4 x[kPasses];
#pragma unroll
        for (int p = 0; p < kPasses; ++p) {
            const int r = p * per + side;
            if (side < per && r < a.rows && to[buffer][r] >= 0)
                x[p] = *reinterpret_cast<const u32x4*>(plane + from[buffer][r] + unit * 16);
        }
        look_up(i0 + a.rows);
        __builtin_amdgcn_s_waitcnt(0);  // every row of the pass is in registers
        __syncthreads();
#pragma unroll
        for (int p = 0; p < kPasses; ++p) {
            const int r = p * per + side;
            if (side < per && r < a.rows && to[buffer][r] >= 0)
                *reinterpret_cast<u32x4*>(plane + to[buffer][r] + unit * 16) = x[p];
        }
    }
}

}  // namespace
}  // namespace evict
}  // namespace mvme

using namespace mvme;

extern "C" int mvme_evict_kv_cache(void* key_cache, void* value_cache, const float* weights, float* new_weights,
                                   int64_t weight_row, int64_t* kept, int64_t* new_lens, const int64_t* block_tables,
                                   const int64_t* context_lens, const int64_t* first, int64_t layers, int64_t batch,
                                   int64_t kv_heads, int64_t head_dim, int64_t num_blocks, int64_t block_size,
                                   int64_t table_width, int64_t keep, int64_t recent, int dtype, void* stream) {
    using namespace mvme::evict;
    if (!valid_dtype(dtype)) return fail(MVME_EINVAL, "FP16/BF16 required");
    if (layers <= 0 || batch <= 0 || kv_heads <= 0 || num_blocks <= 0) return fail(MVME_EINVAL, "empty batch/heads/cache");
    if (head_dim <= 0 || head_dim > 1024 || head_dim % 8 != 0) return fail(MVME_EINVAL, "head_dim must be a multiple of 8 up to 1024");
    if (block_size <= 0 || table_width <= 0) return fail(MVME_EINVAL, "invalid block table");
    if (block_size > kMaxCapacity || table_width > kMaxCapacity / block_size)
        return fail(MVME_EINVAL, "maximum table capacity is 1M tokens");
    if (weight_row < block_size * table_width) return fail(MVME_EINVAL, "weight rows must hold the tables' capacity");
    if (keep <= 0 || recent < 0) return fail(MVME_EINVAL, "keep must be positive and recent not negative");
    const int64_t row = kv_heads * head_dim * 2;
    if (kv_heads > 65536 || num_blocks > 2147483647 || num_blocks > (int64_t(1) << 62) / row / block_size / layers)
        return fail(MVME_EINVAL, "KV cache too large");
    if (batch > 2147483647 || layers > 2147483647) return fail(MVME_EINVAL, "batch/head product too large");
    const int64_t lines = layers * batch;  // (rows are cut, into more work-groups, only where there are few)
    if (layers > kMostThreads / 1024 / batch || lines > kMostThreads / 1024 / kv_heads)
        return fail(MVME_EINVAL, "batch/head product too large");
    if (!key_cache || !value_cache || !weights || !new_weights || !kept || !new_lens || !block_tables || !context_lens)
        return fail(MVME_EINVAL, "eviction: null pointer");
    if (!fp4::aligned(key_cache, 16) || !fp4::aligned(value_cache, 16)) return fail(MVME_EINVAL, "eviction: caches must be 16-byte aligned");
    Args a{};
    a.key = static_cast<uint8_t*>(key_cache);
    a.value = static_cast<uint8_t*>(value_cache);
    a.weights = weights;
    a.new_weights = new_weights;
    a.kept = kept;
    a.new_lens = new_lens;
    a.tables = block_tables;
    a.lens = context_lens;
    a.first = first;
    a.row = weight_row;
    a.columns = keep < weight_row ? keep : weight_row;
    a.keep = keep < weight_row ? keep : weight_row;
    a.recent = recent;
    a.num_blocks = num_blocks;
    a.page_bytes = (uint64_t)(row * block_size);
    a.layer_bytes = (uint64_t)(row * block_size) * (uint64_t)num_blocks;
    a.row_bytes = (uint32_t)row;
    a.head_bytes = (uint32_t)(head_dim * 2);
    a.batch = (int)batch;
    a.kv_heads = (int)kv_heads;
    a.width = (int)table_width;
    a.div = fp4::make_block_div(block_size);
    a.slices = 1;
    // Rows are cut where a work-group per row of a head leaves compute units without one; no further, since pieces of rows
    // are slower to move (us: 16 sequences, one layer, 20.6 in halves and 25 whole; 28 layers of one sequence 235 whole, 288
    // in halves).
    while (lines * kv_heads * 2 * a.slices < 400 && head_dim * 2 / a.slices % 128 == 0) a.slices *= 2;
    a.slice_bytes = (int)(head_dim * 2 / a.slices);
    a.units = a.slice_bytes / 16;
    const int per = kMove / a.units;
    a.rows = per * kPasses < kMove ? per * kPasses : kMove;
    hipStream_t s = static_cast<hipStream_t>(stream);
    // 512 threads choose sooner among few tokens, 1024 among many.
    const int64_t capacity = block_size * table_width;
    const dim3 grid((unsigned)(lines * kv_heads));
    if (capacity <= 512 * 4) hipLaunchKernelGGL((choose_kernel<512, 4>), grid, dim3(512), 0, s, a);
    else if (capacity <= 512 * 16) hipLaunchKernelGGL((choose_kernel<512, 16>), grid, dim3(512), 0, s, a);
    else if (capacity <= 1024 * 16) hipLaunchKernelGGL((choose_kernel<1024, 16>), grid, dim3(1024), 0, s, a);
    else hipLaunchKernelGGL((choose_kernel<1024, 0>), grid, dim3(1024), 0, s, a);
    if (int rc = check_launch("eviction choice")) return rc;
    hipLaunchKernelGGL(move_kernel, dim3((unsigned)(lines * kv_heads * 2 * a.slices)), dim3(kMove), 0, s, a);
    return check_launch("eviction moves");
}
