// Page operators of the cache: copying pages (forks, copy-on-write) and
// compacting a pool, over every layer's keys and values in one launch.
//
// Bound by bytes: each moved page is read and written once per plane.  A
// work-group takes one piece of one page in one plane; the pieces of a page
// are consecutive work-groups.  512 pages of 28 layers in bf16: 366 us, 5.15
// TB/s (a large copy reaches 4.76); 24 packed pages and a renumbered table in
// 6.0 us, of which the launch and the chain from move to store are half.
#include "fp4_cache.h"

namespace mvme {
namespace {

constexpr int kThreads = 256;
constexpr int kUnits = 8;  // units a lane moves: all its loads are in flight before the first store

struct PageArgs {
    uint8_t* planes;
    const int64_t* src;
    const int64_t* dst;
    int64_t num_planes, num_pages, page_bytes, moves;
    int64_t pieces;     // work-groups per page and plane
    int64_t copies;     // work-groups that copy; the others renumber
    int64_t first;      // work-group that a launch begins with
    int64_t* tables;
    int64_t entries;
};

template <typename Unit>
__device__ inline void copy_piece(const PageArgs& a, int64_t group) {
    const int64_t piece = group % a.pieces, rest = group / a.pieces;
    const int64_t move = rest % a.moves, plane = rest / a.moves;
    const int64_t from = a.src[move], to = a.dst[move];
    if (from < 0 || from >= a.num_pages || to < 0 || to >= a.num_pages) return;
    const int64_t units = a.page_bytes / (int64_t)sizeof(Unit);
    uint8_t* base = a.planes + plane * a.num_pages * a.page_bytes;
    const Unit* s = reinterpret_cast<const Unit*>(base + from * a.page_bytes);
    Unit* d = reinterpret_cast<Unit*>(base + to * a.page_bytes);
    const int64_t at = piece * (kThreads * kUnits) + threadIdx.x;
    Unit w[kUnits];
#pragma unroll
    for (int i = 0; i < kUnits; ++i)
        if (at + i * kThreads < units) w[i] = s[at + i * kThreads];
#pragma unroll
    for (int i = 0; i < kUnits; ++i)
        if (at + i * kThreads < units) d[at + i * kThreads] = w[i];
}

// Entries equal to src[i] become dst[i]: a binary search in the rising src.
__device__ inline void renumber(const PageArgs& a, int64_t group) {
    const int64_t at = group * kThreads + threadIdx.x;
    if (at >= a.entries) return;
    const int64_t page = a.tables[at];
    int64_t low = 0, high = a.moves;
    while (low < high) {
        const int64_t mid = (low + high) >> 1;
        if (a.src[mid] < page) low = mid + 1;
        else high = mid;
    }
    if (low < a.moves && a.src[low] == page) {
        const int64_t to = a.dst[low];
        if (page >= 0 && page < a.num_pages && to >= 0 && to < a.num_pages) a.tables[at] = to;
    }
}

template <typename Unit>
__global__ __launch_bounds__(kThreads) void move_pages_kernel(PageArgs a) {
    const int64_t group = a.first + blockIdx.x;
    if (group < a.copies) copy_piece<Unit>(a, group);
    else renumber(a, group - a.copies);
}

int move_pages(void* planes, int64_t num_planes, int64_t num_pages, int64_t page_bytes, const int64_t* src,
               const int64_t* dst, int64_t moves, int64_t* tables, int64_t entries, void* stream) {
    if (num_planes <= 0 || num_pages <= 0 || page_bytes <= 0)
        return fail(MVME_EINVAL, "page planes must have positive dimensions");
    if (page_bytes > (int64_t(1) << 62) / num_planes / num_pages) return fail(MVME_EINVAL, "page planes too large");
    if (moves < 0 || moves > num_pages) return fail(MVME_EINVAL, "more moves than pages");
    if (entries < 0) return fail(MVME_EINVAL, "negative number of table entries");
    if (moves == 0) return MVME_OK;
    if (!planes || !src || !dst || (entries > 0 && !tables)) return fail(MVME_EINVAL, "page move: null pointer");
    const uintptr_t unit = fp4::aligned(planes, 16) && page_bytes % 16 == 0  ? 16
                           : fp4::aligned(planes, 4) && page_bytes % 4 == 0 ? 4
                                                                            : 1;
    PageArgs a{};
    a.planes = static_cast<uint8_t*>(planes);
    a.src = src;
    a.dst = dst;
    a.num_planes = num_planes;
    a.num_pages = num_pages;
    a.page_bytes = page_bytes;
    a.moves = moves;
    a.pieces = (page_bytes / (int64_t)unit - 1) / (kThreads * kUnits) + 1;
    a.tables = tables;
    a.entries = entries;
    const int64_t renumbers = entries > 0 ? (entries - 1) / kThreads + 1 : 0;
    if (a.pieces > 2147483647 / num_planes / moves || num_planes * moves * a.pieces > 2147483647 - renumbers)
        return fail(MVME_EINVAL, "too many pages to move in one call");
    a.copies = num_planes * moves * a.pieces;
    // One launch, unless there are more work-groups than it can have (millions of small pages).
    constexpr int64_t kMostGroups = kMostThreads / kThreads;
    const int64_t groups = a.copies + renumbers;
    hipStream_t s = static_cast<hipStream_t>(stream);
    for (; a.first < groups; a.first += kMostGroups) {
        const dim3 grid((unsigned)(groups - a.first < kMostGroups ? groups - a.first : kMostGroups)), block(kThreads);
        if (unit == 16) hipLaunchKernelGGL((move_pages_kernel<u32x4>), grid, block, 0, s, a);
        else if (unit == 4) hipLaunchKernelGGL((move_pages_kernel<uint32_t>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((move_pages_kernel<uint8_t>), grid, block, 0, s, a);
        if (int rc = check_launch("page move")) return rc;
    }
    return MVME_OK;
}

}  // namespace
}  // namespace mvme

using namespace mvme;

extern "C" int mvme_copy_pages(void* planes, int64_t num_planes, int64_t num_pages, int64_t page_bytes,
                               const int64_t* src, const int64_t* dst, int64_t moves, void* stream) {
    return move_pages(planes, num_planes, num_pages, page_bytes, src, dst, moves, nullptr, 0, stream);
}

extern "C" int mvme_compact_pages(void* planes, int64_t num_planes, int64_t num_pages, int64_t page_bytes,
                                  const int64_t* src, const int64_t* dst, int64_t moves, int64_t* block_tables,
                                  int64_t entries, void* stream) {
    return move_pages(planes, num_planes, num_pages, page_bytes, src, dst, moves, block_tables, entries, stream);
}
