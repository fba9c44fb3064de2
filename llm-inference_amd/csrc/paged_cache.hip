// Page management of a paged KV cache, all of it on the device: copy, fork, grow
// (allocation and copy-on-write), free and compact.
//
// State: a reference count per page (0 = free), a page table row and a length per
// sequence.  A page may be named by several rows (forks share pages); its count is
// the number of rows that name it.  New pages are the lowest free ones, handed out in
// the order of the rows, so the state after a call depends on the state before it
// alone: no atomic decides a page's number.  Page numbers read from a table are
// checked against num_pages before use; entries out of range name nothing.
//
// Nothing synchronises with the host, so the calls can be captured; a pool that runs
// short is reported in a status word and leaves the state as it was.
//
// Planning kernels are one workgroup of 1024 threads, 4096 pages a round: the order of
// the free pages is a prefix sum, which ballots give within a workgroup without a second
// launch.  Pages move in a launch of their own over the whole GPU, 16 KiB a workgroup and
// turn.  Bound by HBM for the pages that move, by launches and the plan's chain of loads
// (length -> page -> count -> free pages) otherwise.  Measured (traced, pages of 16 rows of
// 512 values in 72 planes, 4096 pages): 256 forks that copy 208 pages: free 3.5 us, fork 3.8,
// plan 6.6, copy 85.5 (5.7 TB/s); a compaction that moves 283 pages: plan 5.0, copy 126
// (5.3 TB/s); four forks: 1.4, 2.0, 4.9 and 2.6.
#include "paged_internal.hpp"
#include "../../include/attn_mi355x.h"

namespace attn {
namespace {

constexpr uint32_t kPlanThreads = 1024;
constexpr uint32_t kPlanWaves = kPlanThreads / 64;
constexpr uint32_t kPlanTile = kPlanThreads * 4;  // pages per round of a plan

// 16-byte units of a page that one workgroup of a copy moves at once
constexpr uint32_t kCopyUnits = 4 * 256;

// int32 words of a planning workspace
constexpr uint32_t kHeadWords = 16;  // [0] pages to copy

struct CopyArgs {
    char* pool;
    uint64_t plane_bytes;   // between planes
    uint64_t page_bytes;
    const int32_t* src;     // [n] page numbers
    const int32_t* dst;
    const int32_t* count;   // device count of pairs, or nullptr: n
    uint32_t n;
    uint32_t num_planes;
    uint32_t num_pages;
    uint32_t chunks;        // workgroups' shares per page and plane
};

// Work items are (pair, plane, chunk), chunk innermost: neighbouring workgroups read
// neighbouring bytes.  VEC: pages and planes are 16-byte aligned; otherwise 2-byte
// elements.
template <bool VEC>
__device__ __forceinline__ void copy_items(const CopyArgs& a, uint32_t first, uint32_t step) {
    const uint32_t n = a.count ? min((uint32_t)max(*a.count, 0), a.n) : a.n;
    const uint64_t per_pair = (uint64_t)a.num_planes * a.chunks;
    const uint64_t items = n * per_pair;
    for (uint64_t w = first; w < items; w += step) {
        const uint32_t pair = (uint32_t)(w / per_pair);
        const uint32_t rem = (uint32_t)(w - pair * per_pair);
        const uint32_t plane = rem / a.chunks, chunk = rem - plane * a.chunks;
        const uint32_t s = (uint32_t)a.src[pair], d = (uint32_t)a.dst[pair];
        if (s >= a.num_pages || d >= a.num_pages || s == d) continue;
        const char* const from = a.pool + plane * a.plane_bytes + s * a.page_bytes;
        char* const to = a.pool + plane * a.plane_bytes + d * a.page_bytes;
        if constexpr (VEC) {
            const uint64_t units = a.page_bytes / 16;
            const uint64_t u0 = (uint64_t)chunk * kCopyUnits + threadIdx.x;
            u32x4 x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (u0 + 256u * i < units)
                    x[i] = __builtin_nontemporal_load(
                        reinterpret_cast<const u32x4*>(from) + u0 + 256u * i);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (u0 + 256u * i < units)
                    __builtin_nontemporal_store(x[i], reinterpret_cast<u32x4*>(to) + u0 + 256u * i);
        } else {
            const uint64_t units = a.page_bytes / 2;
            const uint64_t u0 = (uint64_t)chunk * 8u * kCopyUnits;
            for (uint32_t i = threadIdx.x; i < 8u * kCopyUnits && u0 + i < units; i += 256u)
                reinterpret_cast<f16*>(to)[u0 + i] = reinterpret_cast<const f16*>(from)[u0 + i];
        }
    }
}

template <bool VEC>
__global__ __launch_bounds__(256) void pages_copy(CopyArgs a) {
    copy_items<VEC>(a, blockIdx.x, gridDim.x);
}

// ------------------------------------------------------------------ free, fork

struct TableArgs {
    int32_t* table;       // [num_seqs][max_pages]
    int32_t* lens;        // [num_seqs]
    const int32_t* keep;  // free: [num_seqs] tokens to keep (negative: the row is left alone), or nullptr: 0
    int32_t* refs;        // [num_pages]
    // fork
    const int32_t* src_table;
    const int32_t* src_lens;
    const int32_t* parents;
    uint32_t num_src;
    uint32_t same;        // fork within one table
    uint32_t max_pages;
    uint32_t num_pages;
    uint32_t page_size;
};

// One workgroup per row: the pages past the kept tokens lose a reference.
__global__ __launch_bounds__(256) void pages_free(TableArgs a) {
    const uint32_t b = blockIdx.x;
    const int32_t keep = a.keep ? a.keep[b] : 0;
    const uint32_t n = clamp_len(a.lens[b], a.max_pages, a.page_size);
    if (keep < 0 || (uint32_t)keep >= n) return;
    __syncthreads();  // every thread has read the length
    const int32_t* const row = a.table + (uint64_t)b * a.max_pages;
    const uint32_t end = pages_for(n, a.page_size);
    for (uint32_t j = pages_for((uint32_t)keep, a.page_size) + threadIdx.x; j < end; j += 256u) {
        const uint32_t page = (uint32_t)row[j];
        if (page < a.num_pages) atomicSub(a.refs + page, 1);
    }
    if (threadIdx.x == 0) a.lens[b] = keep;
}

// One workgroup per destination row.
__global__ __launch_bounds__(256) void pages_fork(TableArgs a) {
    const uint32_t i = blockIdx.x;
    const uint32_t p = (uint32_t)a.parents[i];
    if (p >= a.num_src) return;
    if (a.same && (p == i || a.parents[p] >= 0)) return;  // the parent is written in this call
    if (a.lens[i] > 0) return;                            // the row holds a sequence
    const uint32_t n = clamp_len(a.src_lens[p], a.max_pages, a.page_size);
    __syncthreads();  // every thread has read the row's length
    const int32_t* const from = a.src_table + (uint64_t)p * a.max_pages;
    int32_t* const to = a.table + (uint64_t)i * a.max_pages;
    const uint32_t end = pages_for(n, a.page_size);
    for (uint32_t j = threadIdx.x; j < end; j += 256u) {
        const int32_t page = from[j];
        to[j] = page;
        if ((uint32_t)page < a.num_pages) atomicAdd(a.refs + page, 1);
    }
    if (threadIdx.x == 0) a.lens[i] = (int32_t)n;
}

// ------------------------------------------------------------------ grow

struct GrowArgs {
    int32_t* table;
    int32_t* lens;
    const int32_t* grow;
    int32_t* refs;
    int32_t* status;   // [2]
    int32_t* work;     // kHeadWords, then offs [B + 1], cow [B], src [B], dst [B], list [num_pages]
    uint32_t num_seqs;
    uint32_t max_pages;
    uint32_t num_pages;
    uint32_t page_size;
};

__device__ __forceinline__ int64_t wave_scan64(int64_t v, uint32_t lane) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int64_t up = __shfl_up(v, o, 64);
        if (lane >= (uint32_t)o) v += up;
    }
    return v;
}

// The counts of pages p..p+3; pages past num_pages count as -1 (neither free nor used).
__device__ __forceinline__ int4 load_refs(const int32_t* refs, uint32_t p, uint32_t num_pages) {
    struct __attribute__((packed, aligned(4))) Four { int x, y, z, w; };
    if (p + 3 < num_pages) {
        const Four f = *reinterpret_cast<const Four*>(refs + p);
        return int4{f.x, f.y, f.z, f.w};
    }
    int4 r = {-1, -1, -1, -1};
    if (p < num_pages) r.x = refs[p];
    if (p + 1 < num_pages) r.y = refs[p + 1];
    if (p + 2 < num_pages) r.z = refs[p + 2];
    if (p + 3 < num_pages) r.w = refs[p + 3];
    return r;
}

// The rank of a thread's first set flag within the workgroup, and the total of all
// flags: ballots within a wave, sums of the waves' totals through `sums` (two copies
// used in turn, so that one barrier a round is enough).
__device__ __forceinline__ uint32_t flag_rank(const bool f[4], uint32_t* sums, uint32_t& total) {
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const uint64_t below = (1ull << lane) - 1ull;
    uint32_t before = 0, mine = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint64_t m = __ballot(f[i]);
        before += (uint32_t)__popcll(m & below);
        mine += (uint32_t)__popcll(m);
    }
    if (lane == 0) sums[wave] = mine;
    __syncthreads();
    total = 0;
#pragma unroll
    for (uint32_t w = 0; w < kPlanWaves; ++w) {
        const uint32_t s = sums[w];
        if (w < wave) before += s;
        total += s;
    }
    return before;
}

// One workgroup.  First every row's need: pages for its new tokens, one more when its
// last page is partly filled and shared (that row gets a copy).  Then the lowest free
// pages, as many as all rows need; then the rows take them in order.
__global__ __launch_bounds__(kPlanThreads) void pages_grow_plan(GrowArgs a) {
    __shared__ int64_t s_scan[kPlanWaves];
    __shared__ uint32_t s_sums[2][kPlanWaves];
    __shared__ uint32_t s_short, s_copies;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
    const uint32_t B = a.num_seqs;
    int32_t* const offs = a.work + kHeadWords;  // [B + 1], saturated: only used when all fits
    int32_t* const cow = offs + B + 1;
    int32_t* const src = cow + B;
    int32_t* const dst = src + B;
    int32_t* const list = dst + B;
    if (tid == 0) s_short = s_copies = 0;
    __syncthreads();
    int64_t need_all = 0;
    for (uint32_t b0 = 0; b0 < B; b0 += kPlanThreads) {
        const uint32_t b = b0 + tid;
        int64_t need = 0;
        if (b < B) {
            const uint32_t n = clamp_len(a.lens[b], a.max_pages, a.page_size);
            const int32_t g = a.grow[b];
            uint32_t copies = 0;
            if (g > 0) {
                const uint64_t most = (uint64_t)a.max_pages * a.page_size;
                if ((uint64_t)n + (uint32_t)g > most) {
                    atomicAdd(&s_short, 1u);
                } else {
                    need = pages_for(n + (uint32_t)g, a.page_size) - pages_for(n, a.page_size);
                    if (n % a.page_size) {
                        const uint32_t page =
                            (uint32_t)a.table[(uint64_t)b * a.max_pages + n / a.page_size];
                        if (page < a.num_pages && a.refs[page] > 1) copies = 1;
                    }
                    need += copies;
                }
            }
            cow[b] = (int32_t)copies;
        }
        const int64_t incl = wave_scan64(need, lane);
        if (lane == 63) s_scan[wave] = incl;
        __syncthreads();
        int64_t before = need_all, total = 0;
#pragma unroll
        for (uint32_t w = 0; w < kPlanWaves; ++w) {
            const int64_t s = s_scan[w];
            if (w < wave) before += s;
            total += s;
        }
        if (b < B) offs[b] = (int32_t)min(before + incl - need, (int64_t)0x7fffffff);
        need_all += total;
        __syncthreads();
    }
    if (tid == 0) offs[B] = (int32_t)min(need_all, (int64_t)0x7fffffff);
    // the lowest free pages
    uint32_t found = 0;
    if (s_short == 0 && need_all > 0) {
        int4 r = load_refs(a.refs, 4u * tid, a.num_pages);
        uint32_t which = 0, looked = 0;
        for (uint32_t base = 0; base < a.num_pages && (int64_t)found < need_all; base += kPlanTile) {
            const uint32_t p = base + 4u * tid;
            const int4 next = load_refs(a.refs, p + kPlanTile, a.num_pages);  // the next round's
            const bool f[4] = {r.x == 0, r.y == 0, r.z == 0, r.w == 0};
            uint32_t total;
            uint32_t rank = found + flag_rank(f, s_sums[which], total);
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i)
                if (f[i]) {
                    if ((int64_t)rank < need_all) list[rank] = (int32_t)(p + i);
                    ++rank;
                }
            found += total;
            r = next;
            which ^= 1u;
            // After a round without a free page four rounds' pages at a time are passed over
            // while none of them is free (170000 pages, all in use but the last ones: 20.0 us
            // against 30.4 round by round), not again before the four that hold one are done.
            if (total == 0 && base >= looked) {
                const uint32_t near = base + kPlanTile;
                uint32_t far = near;
                while (far + 4u * kPlanTile <= a.num_pages) {
                    int4 q[4];
#pragma unroll
                    for (uint32_t i = 0; i < 4; ++i)
                        q[i] = load_refs(a.refs, far + i * kPlanTile + 4u * tid, a.num_pages);
                    bool any = false;
#pragma unroll
                    for (uint32_t i = 0; i < 4; ++i)
                        any |= q[i].x == 0 || q[i].y == 0 || q[i].z == 0 || q[i].w == 0;
                    if (__syncthreads_or(any)) break;
                    far += 4u * kPlanTile;
                }
                looked = far + 4u * kPlanTile;
                if (far != near) {
                    base = far - kPlanTile;
                    r = load_refs(a.refs, far + 4u * tid, a.num_pages);
                }
            }
        }
    }
    __syncthreads();
    const bool fits = s_short == 0 && (int64_t)found >= need_all;
    if (tid == 0) {
        a.status[0] = s_short ? 0 : (int32_t)(fits ? 0 : min(need_all - found, (int64_t)0x7fffffff));
        a.status[1] = (int32_t)s_short;
        if (!fits) a.work[0] = 0;
    }
    if (!fits) return;
    // need_all <= num_pages: 32 bits from here on
    for (uint32_t r = tid; r < (uint32_t)need_all; r += kPlanThreads) {
        // the last row whose pages start at or before r and that takes any
        uint32_t lo = 0, hi = B;  // offs[lo] <= r < offs[hi]
        while (hi - lo > 1) {
            const uint32_t mid = (lo + hi) >> 1;
            if ((uint32_t)offs[mid] <= r) lo = mid; else hi = mid;
        }
        const uint32_t b = lo, i = r - (uint32_t)offs[b], copies = (uint32_t)cow[b];
        const uint32_t n = clamp_len(a.lens[b], a.max_pages, a.page_size);
        int32_t* const row = a.table + (uint64_t)b * a.max_pages;
        const int32_t page = list[r];
        uint32_t column;
        if (i < copies) {  // the copy of the shared last page
            column = n / a.page_size;
            const int32_t old = row[column];
            atomicSub(a.refs + old, 1);
            const uint32_t c = atomicAdd(&s_copies, 1u);  // the order of the copies changes nothing
            src[c] = old;
            dst[c] = page;
        } else {
            column = pages_for(n, a.page_size) + i - copies;
        }
        row[column] = page;
        a.refs[page] = 1;
    }
    __syncthreads();
    if (tid == 0) a.work[0] = (int32_t)s_copies;
    for (uint32_t b = tid; b < B; b += kPlanThreads) {
        const int32_t g = a.grow[b];
        if (g > 0) a.lens[b] = (int32_t)(clamp_len(a.lens[b], a.max_pages, a.page_size) + (uint32_t)g);
    }
}

// ------------------------------------------------------------------ compact

struct CompactArgs {
    CopyArgs copy;
    const int32_t* table;
    const int32_t* lens;
    const int32_t* refs;
    int32_t* table_out;
    int32_t* refs_out;
    int32_t* used;
    int32_t* work;       // kHeadWords, then src [num_pages], dst [num_pages], map [num_pages]
    uint32_t num_seqs;
    uint32_t max_pages;
    uint32_t num_pages;
    uint32_t page_size;
    uint32_t table_blocks;  // workgroups that rewrite the table
};

// One workgroup.  With U used pages, the used pages at U and above move, in order, to
// the free pages below U, in order.
__global__ __launch_bounds__(kPlanThreads) void pages_compact_plan(CompactArgs a) {
    __shared__ uint32_t s_sums[2][kPlanWaves];
    const uint32_t tid = threadIdx.x;
    int32_t* const src = a.work + kHeadWords;
    int32_t* const dst = src + a.num_pages;
    int32_t* const map = dst + a.num_pages;
    uint32_t used = 0, which = 0;
    for (uint32_t base = 0; base < a.num_pages; base += kPlanTile) {
        const int4 r = load_refs(a.refs, base + 4u * tid, a.num_pages);
        const bool f[4] = {r.x > 0, r.y > 0, r.z > 0, r.w > 0};
        uint32_t total;
        (void)flag_rank(f, s_sums[which], total);
        used += total;
        which ^= 1u;
    }
    uint32_t holes = 0, movers = 0;
    for (uint32_t base = 0; base < a.num_pages; base += kPlanTile) {
        const uint32_t p = base + 4u * tid;
        const int4 r = load_refs(a.refs, p, a.num_pages);
        const int32_t c[4] = {r.x, r.y, r.z, r.w};
        bool hole[4], mover[4];
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            hole[i] = c[i] <= 0 && p + i < used;
            mover[i] = c[i] > 0 && p + i >= used;
        }
        uint32_t total;
        uint32_t rank = holes + flag_rank(hole, s_sums[which], total);
        holes += total;
        which ^= 1u;
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i)
            if (hole[i]) dst[rank++] = (int32_t)(p + i);
        rank = movers + flag_rank(mover, s_sums[which], total);
        movers += total;
        which ^= 1u;
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i)
            if (mover[i]) src[rank++] = (int32_t)(p + i);
            else if (p + i >= used && p + i < a.num_pages) map[p + i] = (int32_t)(p + i);
        if (a.refs_out != a.refs) {
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i)
                if (p + i < a.num_pages) a.refs_out[p + i] = c[i];
        }
    }
    __syncthreads();
    // as many free pages below U as used pages above
    for (uint32_t k = tid; k < movers; k += kPlanThreads) {
        const int32_t from = src[k], to = dst[k];
        map[from] = to;
        a.refs_out[to] = a.refs[from];
        a.refs_out[from] = 0;
    }
    if (tid == 0) {
        a.work[0] = (int32_t)movers;
        *a.used = (int32_t)used;
    }
}

// The first table_blocks workgroups rewrite the table rows, the others copy pages.
template <bool VEC>
__global__ __launch_bounds__(256) void pages_compact_move(CompactArgs a) {
    if (blockIdx.x >= a.table_blocks) {
        copy_items<VEC>(a.copy, blockIdx.x - a.table_blocks, gridDim.x - a.table_blocks);
        return;
    }
    const int32_t* const map = a.work + kHeadWords + 2u * (uint64_t)a.num_pages;
    const uint32_t used = (uint32_t)*a.used;
    for (uint32_t b = blockIdx.x; b < a.num_seqs; b += a.table_blocks) {
        const uint64_t at = (uint64_t)b * a.max_pages;
        const uint32_t end = pages_for(clamp_len(a.lens[b], a.max_pages, a.page_size), a.page_size);
        for (uint32_t j = threadIdx.x; j < end; j += 256u) {
            const uint32_t page = (uint32_t)a.table[at + j];
            a.table_out[at + j] = page >= used && page < a.num_pages ? map[page] : (int32_t)page;
        }
    }
}

// ------------------------------------------------------------------ host side

struct PoolView {
    CopyArgs c{};
    bool vec = false;
};

// false: sizes that do not describe a pool
bool pool_view(PoolView& v, attn_f16_t* pool, size_t num_planes, size_t plane_stride,
               size_t page_elems, size_t num_pages) {
    if (!paged_u31(num_planes) || !paged_u31(num_pages) || page_elems == 0) return false;
    const uint64_t plane = paged_mul(num_pages, page_elems);
    if (plane >> 62 || (plane_stride && plane_stride < plane)) return false;
    const uint64_t stride = plane_stride ? plane_stride : plane;
    if (paged_mul(paged_mul(num_planes, stride), 2) >> 62) return false;
    v.c.pool = reinterpret_cast<char*>(pool);
    v.c.plane_bytes = stride * 2;
    v.c.page_bytes = page_elems * 2;
    v.c.num_planes = (uint32_t)num_planes;
    v.c.num_pages = (uint32_t)num_pages;
    v.vec = aligned16(pool) && v.c.page_bytes % 16 == 0 && v.c.plane_bytes % 16 == 0;
    const uint64_t chunks = (v.c.page_bytes + 16ull * kCopyUnits - 1) / (16ull * kCopyUnits);
    if (paged_mul(num_planes, chunks) > 0x7fffffffull) return false;
    v.c.chunks = (uint32_t)chunks;
    return true;
}

// workgroups of a copy of up to n pages: a few per CU, each walking its share
uint32_t copy_grid(const CopyArgs& c) {
    const uint64_t items = paged_mul(c.n, (uint64_t)c.num_planes * c.chunks);
    return (uint32_t)(items < 2048 ? items : 2048);
}

hipError_t launch_copy(const CopyArgs& c, bool vec, hipStream_t stream) {
    const uint32_t grid = copy_grid(c);
    if (grid == 0) return hipSuccess;
    if (vec)
        hipLaunchKernelGGL(pages_copy<true>, dim3(grid), dim3(256), 0, stream, c);
    else
        hipLaunchKernelGGL(pages_copy<false>, dim3(grid), dim3(256), 0, stream, c);
    return hipGetLastError();
}

}  // namespace
}  // namespace attn

using namespace attn;

extern "C" {

size_t attn_pages_workspace_bytes(size_t num_seqs, size_t num_pages) {
    return 4 * (kHeadWords + 1 + 4 * num_seqs + 3 * num_pages);
}

int attn_pages_copy(attn_f16_t* pool, size_t num_planes, size_t plane_stride, size_t page_elems,
                    const int32_t* src, const int32_t* dst, size_t n, size_t num_pages,
                    hipStream_t stream) {
    if (n == 0 || num_planes == 0 || num_pages == 0) return 0;
    PoolView v;
    if (!pool_view(v, pool, num_planes, plane_stride, page_elems, num_pages) || !paged_u31(n) ||
        !pool || !src || !dst)
        return (int)hipErrorInvalidValue;
    v.c.src = src;
    v.c.dst = dst;
    v.c.n = (uint32_t)n;
    return (int)launch_copy(v.c, v.vec, stream);
}

int attn_pages_free(int32_t* page_table, int32_t* seq_lens, const int32_t* keep_lens,
                    int32_t* ref_counts, size_t num_seqs, size_t max_pages, size_t num_pages,
                    size_t page_size, hipStream_t stream) {
    if (num_seqs == 0) return 0;
    if (!paged_sizes_ok(num_seqs, max_pages, num_pages, page_size) || !page_table || !seq_lens ||
        !ref_counts)
        return (int)hipErrorInvalidValue;
    TableArgs a{};
    a.table = page_table;
    a.lens = seq_lens;
    a.keep = keep_lens;
    a.refs = ref_counts;
    a.max_pages = (uint32_t)max_pages;
    a.num_pages = (uint32_t)num_pages;
    a.page_size = (uint32_t)page_size;
    hipLaunchKernelGGL(pages_free, dim3((uint32_t)num_seqs), dim3(256), 0, stream, a);
    return (int)hipGetLastError();
}

int attn_pages_fork(const int32_t* src_table, const int32_t* src_lens, int32_t* dst_table,
                    int32_t* dst_lens, const int32_t* parents, int32_t* ref_counts, size_t num_src,
                    size_t num_dst, size_t max_pages, size_t num_pages, size_t page_size,
                    hipStream_t stream) {
    if (num_dst == 0) return 0;
    if (!paged_sizes_ok(num_src, max_pages, num_pages, page_size) || !paged_u31(num_dst) ||
        !src_table || !src_lens || !dst_table || !dst_lens || !parents || !ref_counts)
        return (int)hipErrorInvalidValue;
    const bool same = src_table == dst_table;
    // one table: its lengths and its rows are the same ones on both sides
    if (same != (src_lens == dst_lens) || (same && num_src != num_dst))
        return (int)hipErrorInvalidValue;
    TableArgs a{};
    a.table = dst_table;
    a.lens = dst_lens;
    a.refs = ref_counts;
    a.src_table = src_table;
    a.src_lens = src_lens;
    a.parents = parents;
    a.num_src = (uint32_t)num_src;
    a.same = same ? 1u : 0u;
    a.max_pages = (uint32_t)max_pages;
    a.num_pages = (uint32_t)num_pages;
    a.page_size = (uint32_t)page_size;
    hipLaunchKernelGGL(pages_fork, dim3((uint32_t)num_dst), dim3(256), 0, stream, a);
    return (int)hipGetLastError();
}

int attn_pages_grow(attn_f16_t* pool, size_t num_planes, size_t plane_stride, size_t page_elems,
                    int32_t* page_table, int32_t* seq_lens, const int32_t* grow,
                    int32_t* ref_counts, int32_t* status, size_t num_seqs, size_t max_pages,
                    size_t num_pages, size_t page_size, void* workspace, hipStream_t stream) {
    if (num_seqs == 0) return 0;
    PoolView v;
    if (!paged_sizes_ok(num_seqs, max_pages, num_pages, page_size) || !page_table || !seq_lens ||
        !grow || !ref_counts || !status || !workspace || ((uintptr_t)workspace & 3u) || !pool ||
        num_planes == 0 || !pool_view(v, pool, num_planes, plane_stride, page_elems, num_pages))
        return (int)hipErrorInvalidValue;
    GrowArgs a{};
    a.table = page_table;
    a.lens = seq_lens;
    a.grow = grow;
    a.refs = ref_counts;
    a.status = status;
    a.work = static_cast<int32_t*>(workspace);
    a.num_seqs = (uint32_t)num_seqs;
    a.max_pages = (uint32_t)max_pages;
    a.num_pages = (uint32_t)num_pages;
    a.page_size = (uint32_t)page_size;
    hipLaunchKernelGGL(pages_grow_plan, dim3(1), dim3(kPlanThreads), 0, stream, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
    v.c.count = a.work;
    v.c.src = a.work + kHeadWords + 1 + 2 * num_seqs;
    v.c.dst = v.c.src + num_seqs;
    v.c.n = (uint32_t)num_seqs;
    return (int)launch_copy(v.c, v.vec, stream);
}

int attn_pages_compact(attn_f16_t* pool, size_t num_planes, size_t plane_stride, size_t page_elems,
                       const int32_t* page_table, const int32_t* seq_lens,
                       const int32_t* ref_counts, int32_t* page_table_out,
                       int32_t* ref_counts_out, int32_t* num_used, size_t num_seqs,
                       size_t max_pages, size_t num_pages, size_t page_size, void* workspace,
                       hipStream_t stream) {
    if (num_pages == 0) return 0;
    PoolView v;
    if (!paged_sizes_ok(num_seqs, max_pages, num_pages, page_size) || !ref_counts ||
        !ref_counts_out || !num_used || !workspace || ((uintptr_t)workspace & 3u) ||
        (num_seqs && (!page_table || !seq_lens || !page_table_out)) || !pool || num_planes == 0 ||
        !pool_view(v, pool, num_planes, plane_stride, page_elems, num_pages))
        return (int)hipErrorInvalidValue;
    CompactArgs a{};
    a.table = page_table;
    a.lens = seq_lens;
    a.refs = ref_counts;
    a.table_out = page_table_out;
    a.refs_out = ref_counts_out;
    a.used = num_used;
    a.work = static_cast<int32_t*>(workspace);
    a.num_seqs = (uint32_t)num_seqs;
    a.max_pages = (uint32_t)max_pages;
    a.num_pages = (uint32_t)num_pages;
    a.page_size = (uint32_t)page_size;
    a.copy = v.c;
    a.copy.count = a.work;
    a.copy.src = a.work + kHeadWords;
    a.copy.dst = a.copy.src + num_pages;
    a.copy.n = (uint32_t)num_pages;
    a.table_blocks = (uint32_t)(num_seqs < 256 ? num_seqs : 256);
    hipLaunchKernelGGL(pages_compact_plan, dim3(1), dim3(kPlanThreads), 0, stream, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
    const dim3 grid(a.table_blocks + copy_grid(a.copy));
    if (v.vec)
        hipLaunchKernelGGL(pages_compact_move<true>, grid, dim3(256), 0, stream, a);
    else
        hipLaunchKernelGGL(pages_compact_move<false>, grid, dim3(256), 0, stream, a);
    return (int)hipGetLastError();
}

}  // extern "C"
