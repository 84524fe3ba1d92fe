// Page bookkeeping of a shared pool (nd_op_pages_fork, nd_op_pages_compact):
// what a set of sequences keeps, shares, copies, frees and gets, decided on
// the device from the tables alone, with results that do not depend on the
// order threads run in (sums, minima and prefix sums of whole numbers).
//
// Both are a handful of passes over the tables and one word a page, then the
// copies. The copies are HBM bound (each page read and written once, 16 bytes
// a thread); the rest is bound by the passes' dependent loads and the
// launches. So a fork's passes are one cluster of eight CTAs, the hardware's
// cluster barrier between them, and a second launch, issued early, writes the
// tables and copies. A compaction needs a bit a page, not a count, and its
// plan is CTAs that each have all bits and wait for nobody. Past PG_SMALL
// pages or table entries that is too few CTAs, and each pass is a launch.
// Measured (us, GPU alone, then of a Python call): 1024 sequences of 51
// columns over 14,704 pages forked 22 and 21, as launches of their own 16.5 and
// 36; 24,576 pages compacted, half live, 26, planned by a cluster 29.

#include <cooperative_groups.h>

#include "kv4_host.h"

namespace nd {

namespace cg = cooperative_groups;

constexpr int PG_BLOCK = 1024;  // pages or sequences a block of the prefix sums
constexpr int PG_CLUSTER = 8;
constexpr int PG_PLAN = 32;  // CTAs that each plan a compaction
constexpr int PG_SMALL = 1 << 17;  // pages, and table entries

__device__ __forceinline__ void after_previous() {
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    asm volatile("griddepcontrol.wait;\n" ::: "memory");
}

struct PoolView {
    uint8_t* base;
    long long page_stride, layer_stride, bytes;  // bytes of one page in one layer, a multiple of 16
    int layers;
};

struct ForkArgs {
    PoolView pool;
    const int32_t* table;
    int table_stride, seqs, cols, pages, page;
    FastDiv by_cols;
    const int32_t *src, *keep, *need;
    int n;  // new sequences
    const uint8_t* pinned;
    int32_t *table_out, *refs, *info;
    // workspace
    int32_t* writers;   // [pages] new sequences that will write on the kept page
    int32_t* first;     // [pages] n - the first of those
    int32_t* free_ids;  // [pages]
    int32_t* sums;      // [blocks of pages], [blocks of sequences], free pages, pages wanted
    int32_t* fresh;     // [n] pages a sequence gets
    int32_t* base;      // [n] how many the ones before it get
};

// What sequence d of the new set keeps: columns [0, nk) of `row`, and room
// for nn; with `writes` its last kept page is partly filled and will grow.
struct Kept {
    const int32_t* row;
    int nk, nn;
    bool writes;
};

__device__ __forceinline__ Kept kept_of(const ForkArgs& a, int d) {
    Kept k;
    const int s = __ldg(a.src + d);
    const bool has = s >= 0 && s < a.seqs;
    const long long cap = (long long)a.cols * a.page;
    const long long keep = has ? min(max((long long)__ldg(a.keep + d), 0LL), cap) : 0;
    const long long need = max(min((long long)__ldg(a.need + d), cap), keep);
    k.row = a.table + (size_t)(has ? s : 0) * a.table_stride;
    k.nk = (int)((keep + a.page - 1) / a.page);
    k.nn = (int)((need + a.page - 1) / a.page);
    k.writes = keep % a.page != 0 && need > keep;
    return k;
}

// Whether d has to copy page p, the one it will write on: not if d alone
// refers to it, nor if all that do will write on it and d is the first.
__device__ __forceinline__ bool must_copy(const ForkArgs& a, int d, int p) {
    if (a.pinned && a.pinned[p]) return true;
    const int refs = __ldcg(a.refs + p);
    return !(refs == 1 || (refs == __ldcg(a.writers + p) && __ldcg(a.first + p) == a.n - d));
}

__global__ void pages_zero_kernel(int32_t* a, int32_t* b, int n) {
    after_previous();
    for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < n; i += gridDim.x * blockDim.x) {
        a[i] = 0;
        if (b) b[i] = b[n + i] = 0;
    }
}

__device__ __forceinline__ void count_kept(const ForkArgs& a, int d, int lane) {  // by a warp
    const Kept k = kept_of(a, d);
    for (int c = lane; c < k.nk; c += 32) {
        const int p = __ldg(k.row + c);
        if (p < 0 || p >= a.pages) continue;
        atomicAdd(a.refs + p, 1);
        if (k.writes && c == k.nk - 1) {
            atomicAdd(a.writers + p, 1);
            atomicMax(a.first + p, a.n - d);
        }
    }
}

__global__ void fork_count_kernel(ForkArgs a) {
    after_previous();
    const int d = blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32;
    if (d < a.n) count_kept(a, d, threadIdx.x & 31);
}

// Fresh pages sequence d wants.
__device__ __forceinline__ int fresh_wanted(const ForkArgs& a, int d) {
    const Kept k = kept_of(a, d);
    int f = k.nn - k.nk;
    if (k.writes) {
        const int p = __ldg(k.row + k.nk - 1);
        f += p >= 0 && p < a.pages && must_copy(a, d, p);
    }
    return f;
}

// Sum of `mine` over a block of PG_BLOCK threads; `before`: of the threads before this one.
__device__ __forceinline__ int block_scan(int mine, int* before) {
    __shared__ int warp_sums[PG_BLOCK / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const int up = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += up;
    }
    __syncthreads();
    if (lane == 31) warp_sums[warp] = incl;
    __syncthreads();
    int w = warp_sums[lane];
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const int up = __shfl_up_sync(0xffffffffu, w, o);
        if (lane >= o) w += up;
    }
    *before = incl - mine + (warp ? __shfl_sync(0xffffffffu, w, warp - 1) : 0);
    return __shfl_sync(0xffffffffu, w, 31);
}

// The same of two numbers at once.
__device__ __forceinline__ int2 block_scan2(int2 mine, int2* before) {
    __shared__ int2 warp_sums[PG_BLOCK / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int2 incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const int x = __shfl_up_sync(0xffffffffu, incl.x, o), y = __shfl_up_sync(0xffffffffu, incl.y, o);
        if (lane >= o) incl.x += x, incl.y += y;
    }
    __syncthreads();
    if (lane == 31) warp_sums[warp] = incl;
    __syncthreads();
    int2 w = warp_sums[lane];
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const int x = __shfl_up_sync(0xffffffffu, w.x, o), y = __shfl_up_sync(0xffffffffu, w.y, o);
        if (lane >= o) w.x += x, w.y += y;
    }
    const int ux = __shfl_sync(0xffffffffu, w.x, max(warp - 1, 0)), uy = __shfl_sync(0xffffffffu, w.y, max(warp - 1, 0));
    *before = make_int2(incl.x - mine.x + (warp ? ux : 0), incl.y - mine.y + (warp ? uy : 0));
    return make_int2(__shfl_sync(0xffffffffu, w.x, 31), __shfl_sync(0xffffffffu, w.y, 31));
}

// Sum of sums[0 .. n) by a block.
__device__ __forceinline__ int block_total(const int32_t* sums, int n) {
    int mine = 0, before;
    for (int i = threadIdx.x; i < n; i += PG_BLOCK) mine += sums[i];
    return block_scan(mine, &before);
}

__device__ __forceinline__ bool page_free(const ForkArgs& a, int p) { return __ldcg(a.refs + p) == 0 && !(a.pinned && a.pinned[p]); }

// Blocks of pages count the free ones, blocks of sequences the new pages wanted.
__global__ void __launch_bounds__(PG_BLOCK) fork_sums_kernel(ForkArgs a, int page_blocks) {
    after_previous();
    int mine = 0, before;
    if ((int)blockIdx.x < page_blocks) {
        const int p = blockIdx.x * PG_BLOCK + threadIdx.x;
        mine = p < a.pages && page_free(a, p);
    } else {
        const int d = (blockIdx.x - page_blocks) * PG_BLOCK + threadIdx.x;
        if (d < a.n) {
            mine = fresh_wanted(a, d);
            a.fresh[d] = mine;
        }
    }
    const int sum = block_scan(mine, &before);
    if (threadIdx.x == 0) a.sums[blockIdx.x] = sum;
}

__global__ void __launch_bounds__(PG_BLOCK) fork_lists_kernel(ForkArgs a, int page_blocks) {
    after_previous();
    int before;
    if ((int)blockIdx.x < page_blocks) {
        const int p = blockIdx.x * PG_BLOCK + threadIdx.x;
        const int start = block_total(a.sums, blockIdx.x);
        const bool is = p < a.pages && page_free(a, p);
        const int sum = block_scan(is, &before);
        if (is) a.free_ids[start + before] = p;
        if ((int)blockIdx.x == page_blocks - 1 && threadIdx.x == 0) a.sums[gridDim.x] = start + sum, a.info[2] = 0;
    } else {
        const int b = blockIdx.x - page_blocks, d = b * PG_BLOCK + threadIdx.x;
        const int start = block_total(a.sums + page_blocks, b);
        const int mine = d < a.n ? a.fresh[d] : 0;
        const int sum = block_scan(mine, &before);
        if (d < a.n) a.base[d] = start + before;
        if (blockIdx.x == gridDim.x - 1 && threadIdx.x == 0) a.sums[gridDim.x + 1] = start + sum;
    }
}

// All passes of a fork but the last, by one cluster. A thread has a run of
// pages and one of sequences, so that one prefix sum places both. The totals
// go to sums[0], sums[1].
__global__ void __cluster_dims__(PG_CLUSTER, 1, 1) __launch_bounds__(PG_BLOCK) fork_plan_kernel(ForkArgs a) {
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    cg::cluster_group cluster = cg::this_cluster();
    constexpr int ALL = PG_CLUSTER * PG_BLOCK, SEQS = PG_BLOCK;
    const int rank = cluster.block_rank(), tid = threadIdx.x, all = rank * PG_BLOCK + tid;
    __shared__ int2 mine;
    __shared__ Kept kept[SEQS];
    for (int i = all; i < a.pages; i += ALL) a.refs[i] = a.writers[i] = a.first[i] = 0;
    // what this CTA's sequences keep, SEQS at a time; then their table entries
    const int each = (a.n + PG_CLUSTER - 1) / PG_CLUSTER, d0 = rank * each, d1 = min(d0 + each, a.n);
    bool zeroed = false;
    for (int base = d0; base < d1 || !zeroed; base += SEQS) {
        const int n = max(min(SEQS, d1 - base), 0);
        __syncthreads();
        if (tid < n) kept[tid] = kept_of(a, base + tid);
        if (!zeroed) cluster.sync(), zeroed = true;
        __syncthreads();
#pragma unroll 4
        for (int i = tid; i < n * a.cols; i += PG_BLOCK) {
            const int s = a.by_cols(i), c = i - s * a.cols;
            const Kept& k = kept[s];
            if (c >= k.nk) continue;
            const int p = __ldg(k.row + c);
            if (p < 0 || p >= a.pages) continue;
            atomicAdd(a.refs + p, 1);
            if (k.writes && c == k.nk - 1) {
                atomicAdd(a.writers + p, 1);
                atomicMax(a.first + p, a.n - (base + s));
            }
        }
    }
    cluster.sync();
    const int pages_each = (a.pages + ALL - 1) / ALL, seqs_each = (a.n + ALL - 1) / ALL;
    const int p0 = min(all * pages_each, a.pages), p1 = min(p0 + pages_each, a.pages);
    const int s0 = min(all * seqs_each, a.n), s1 = min(s0 + seqs_each, a.n);
    int2 own = make_int2(0, 0), before;
    for (int p = p0; p < p1; p++) own.x += page_free(a, p);
    for (int d = s0; d < s1; d++) own.y += a.fresh[d] = fresh_wanted(a, d);
    const int2 sum = block_scan2(own, &before);
    if (tid == 0) mine = sum;
    cluster.sync();
    for (int r = 0; r < rank; r++) {
        const int2 m = *cluster.map_shared_rank(&mine, r);
        before.x += m.x, before.y += m.y;
    }
    for (int p = p0; p < p1; p++)
        if (page_free(a, p)) a.free_ids[before.x++] = p;
    for (int d = s0; d < s1; d++) {
        a.base[d] = before.y;
        before.y += a.fresh[d];  // this thread's own, from above
    }
    if (all == ALL - 1) a.sums[0] = before.x, a.sums[1] = before.y, a.info[2] = 0;
    cluster.sync();  // no CTA leaves while others read its counts
}

__device__ __forceinline__ void copy_page(const PoolView& v, int from, int to, int part, int parts) {
    const long long units = v.bytes / 16;
    for (int l = 0; l < v.layers; l++) {
        const uint4* s = (const uint4*)(v.base + l * v.layer_stride + from * v.page_stride);
        uint4* t = (uint4*)(v.base + l * v.layer_stride + to * v.page_stride);
        const long long step = (long long)parts * blockDim.x;
        long long i = part * (long long)blockDim.x + threadIdx.x;
        for (; i + 3 * step < units; i += 4 * step) {
            uint4 x[4];
#pragma unroll
            for (int j = 0; j < 4; j++) x[j] = __ldcs(s + i + j * step);
#pragma unroll
            for (int j = 0; j < 4; j++) t[i + j * step] = x[j];
        }
        for (; i < units; i += step) t[i] = __ldcs(s + i);
    }
}

// A block a new sequence (and part of its copy): the row of the new table,
// references, the page it copies. Sources of copies stay referenced, so no
// copy writes what another reads.
__global__ void __launch_bounds__(128) fork_assign_kernel(ForkArgs a, int totals) {
    after_previous();
    const int d = blockIdx.x;
    const Kept k = kept_of(a, d);
    const int base = a.base[d], frees = a.sums[totals];
    auto id = [&](int rank) { return rank < frees ? a.free_ids[rank] : -1; };
    int last = -1;
    if (k.writes) {
        last = __ldg(k.row + k.nk - 1);
        if (last < 0 || last >= a.pages) last = -1;
    }
    const bool copies = last >= 0 && a.fresh[d] > k.nn - k.nk;
    const int to = copies ? id(base) : -1;
    if (to >= 0) copy_page(a.pool, last, to, blockIdx.y, gridDim.y);
    if (blockIdx.y) return;
    for (int c = threadIdx.x; c < a.cols; c += blockDim.x) {
        int p = -1;
        if (c < k.nk) {
            p = __ldg(k.row + c);
            if (p < 0 || p >= a.pages) p = -1;
            if (copies && c == k.nk - 1) p = to;
        } else if (c < k.nn) {
            p = id(base + copies + c - k.nk);
            if (p >= 0) a.refs[p] = 1;
        }
        a.table_out[(size_t)d * a.cols + c] = p;
    }
    if (threadIdx.x == 0 && d == 0) {
        const int wanted = a.sums[totals + 1], given = min(wanted, frees);
        a.info[0] = a.pages - frees + given;
        a.info[1] = given;
        a.info[3] = wanted - given;
    }
    if (threadIdx.x == 0 && copies) {
        atomicAdd(a.refs + last, -1);
        if (to >= 0) {
            a.refs[to] = 1;
            atomicAdd(a.info + 2, 1);
        }
    }
}

struct CompactArgs {
    PoolView pool;
    const int32_t* table;
    int table_stride, seqs, cols, pages;
    FastDiv by_cols;
    const uint8_t* pinned;
    int32_t *table_out, *map, *info;
    // workspace
    int32_t* refs;    // [pages]
    int2* sums;       // [blocks] live pages, those of them that may move; then the totals
    int32_t* before;  // [pages] live pages before this one that may move
    int32_t *movers, *holes;  // [pages]
};

__global__ void compact_count_kernel(CompactArgs a) {
    after_previous();
    const int s = blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32, lane = threadIdx.x & 31;
    if (s >= a.seqs) return;
    for (int c = lane; c < a.cols; c += 32) {
        const int p = __ldg(a.table + (size_t)s * a.table_stride + c);
        if (p >= 0 && p < a.pages) a.refs[p] = 1;
    }
}

// (live, live and movable)
__device__ __forceinline__ int2 page_state(const CompactArgs& a, int p) {
    if (p >= a.pages) return make_int2(0, 0);
    const bool used = __ldcg(a.refs + p) != 0, pin = a.pinned && a.pinned[p];
    return make_int2(used || pin, used && !pin);
}

__global__ void __launch_bounds__(PG_BLOCK) compact_sums_kernel(CompactArgs a) {
    after_previous();
    int before;
    const int2 st = page_state(a, blockIdx.x * PG_BLOCK + threadIdx.x);
    const int live = block_scan(st.x, &before), move = block_scan(st.y, &before);
    if (threadIdx.x == 0) a.sums[blockIdx.x] = make_int2(live, move);
}

// With n live pages: movable ones at n and after, in order, go to the holes
// before n, in order.
__global__ void __launch_bounds__(PG_BLOCK) compact_lists_kernel(CompactArgs a) {
    after_previous();
    const int blocks = gridDim.x;
    int live0 = 0, move0 = 0, n = 0, x, before_n = 0;
    for (int i = threadIdx.x; i < blocks; i += PG_BLOCK) {
        const int2 s = a.sums[i];
        n += s.x;
        if (i < (int)blockIdx.x) live0 += s.x, move0 += s.y;
    }
    n = block_scan(n, &x);
    live0 = block_scan(live0, &x);
    move0 = block_scan(move0, &x);
    // movable pages before n: whole blocks, and the part of the block n lies in
    for (int i = threadIdx.x; i < n / PG_BLOCK; i += PG_BLOCK) before_n += a.sums[i].y;
    const int q = n / PG_BLOCK * PG_BLOCK + threadIdx.x;
    if (q < n) before_n += page_state(a, q).y;
    before_n = block_scan(before_n, &x);

    const int p = blockIdx.x * PG_BLOCK + threadIdx.x;
    const int2 st = page_state(a, p);
    int live, move;
    block_scan(st.x, &live);
    const int moves = block_scan(st.y, &move);
    live += live0, move += move0;
    if (p < a.pages) {
        a.before[p] = move - before_n;  // of a mover: its place in the list
        if (p >= n && st.y) a.movers[move - before_n] = p;
        if (p < n && !st.x) a.holes[p - live] = p;
    }
    if ((int)blockIdx.x == blocks - 1 && threadIdx.x == 0) {
        a.sums[blocks] = make_int2(n, move0 + moves - before_n);
        a.info[0] = n;
        a.info[1] = move0 + moves - before_n;
    }
}

// The same where all pages' bits fit a CTA's shared memory: each of a few CTAs
// reads the whole table and counts for itself, so that none waits for
// another, and writes its share of the map. Thread t has words 4 t .. 4 t + 3.
constexpr int PG_WORDS = PG_SMALL / 32;
static_assert(PG_WORDS == 4 * PG_BLOCK, "four words a thread");

__global__ void __launch_bounds__(PG_BLOCK) compact_plan_kernel(CompactArgs a) {
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    __shared__ uint32_t live[PG_WORDS], move[PG_WORDS];  // referred to or pinned; only referred to
    __shared__ int2 count[PG_BLOCK];                     // of those, before the thread's words
    const int tid = threadIdx.x;
#pragma unroll
    for (int i = 0; i < 4; i++) live[tid + i * PG_BLOCK] = 0;
    __syncthreads();
    const int entries = a.seqs * a.cols;
#pragma unroll 8
    for (int i = tid; i < entries; i += PG_BLOCK) {
        const int s = a.by_cols(i), p = __ldg(a.table + (size_t)s * a.table_stride + (i - s * a.cols));
        if (p >= 0 && p < a.pages) atomicOr(&live[p >> 5], 1u << (p & 31));
    }
    __syncthreads();
    if (a.pinned) {
        for (int p = tid; p < (a.pages + 31) / 32 * 32; p += PG_BLOCK) {
            const uint32_t pin = __ballot_sync(0xffffffffu, p < a.pages && a.pinned[p]);
            if ((tid & 31) == 0) move[p >> 5] = live[p >> 5] & ~pin, live[p >> 5] |= pin;
        }
        __syncthreads();
    }
    const uint32_t* mv = a.pinned ? move : live;
    const int W = (a.pages + 31) / 32;
    int2 own = make_int2(0, 0), before;
#pragma unroll
    for (int i = 4 * tid; i < 4 * tid + 4; i++)
        if (i < W) own.x += __popc(live[i]), own.y += __popc(mv[i]);
    const int2 all = block_scan2(own, &before);
    count[tid] = before;
    __syncthreads();
    // movable pages before p
    auto rank = [&](int p) {
        const int w = p >> 5;
        int r = count[w >> 2].y + __popc(mv[w] & ((1u << (p & 31)) - 1));
        for (int i = w & ~3; i < w; i++) r += __popc(mv[i]);
        return r;
    };
    // the r-th page that is not live, r below their number
    auto hole = [&](int r) {
        int lo = 0, hi = PG_BLOCK;  // 128 lo - count[lo].x <= r, not so at hi
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (128 * mid - count[mid].x <= r) lo = mid;
            else hi = mid;
        }
        r -= 128 * lo - count[lo].x;
        int w = 4 * lo;
        while (w < 4 * lo + 3 && r >= 32 - __popc(live[w])) r -= 32 - __popc(live[w]), w++;
        uint32_t free = ~live[w];
        for (; r > 0; r--) free &= free - 1;
        return 32 * w + __ffs(free) - 1;
    };
    const int n = all.x, before_n = n < a.pages ? rank(n) : all.y;
    for (int p = blockIdx.x * PG_BLOCK + tid; p < a.pages; p += gridDim.x * PG_BLOCK) {
        int to = live[p >> 5] >> (p & 31) & 1 ? p : -1;
        if (p >= n && (mv[p >> 5] >> (p & 31) & 1)) {
            const int r = rank(p) - before_n;
            to = hole(r);
            a.movers[r] = p, a.holes[r] = to;
        }
        a.map[p] = to;
    }
    if (blockIdx.x == 0 && tid == 0) {
        a.sums[0] = make_int2(n, all.y - before_n);
        a.info[0] = n;
        a.info[1] = all.y - before_n;
    }
}

// Blocks of pages write the map (where the plan has not: no such blocks),
// blocks of table entries the new table, the others copy.
__global__ void __launch_bounds__(128) compact_move_kernel(CompactArgs a, int totals, int map_blocks, int table_blocks) {
    after_previous();
    const int2 tot = a.sums[totals];
    const int n = tot.x;
    auto to = [&](int p) {
        const int2 st = page_state(a, p);
        return !st.x ? -1 : p >= n && st.y ? a.holes[a.before[p]] : p;
    };
    int b = blockIdx.x;
    if (b < map_blocks) {
        const int p = b * 128 + threadIdx.x;
        if (p < a.pages) a.map[p] = to(p);
        return;
    }
    b -= map_blocks;
    if (b < table_blocks) {
        const long long i = b * 128LL + threadIdx.x;
        if (i < (long long)a.seqs * a.cols) {
            const int s = a.by_cols((int)i), p = __ldg(a.table + (size_t)s * a.table_stride + (i - (long long)s * a.cols));
            a.table_out[i] = p < 0 || p >= a.pages ? -1 : map_blocks ? to(p) : __ldcg(a.map + p);
        }
        return;
    }
    const int step = gridDim.x - map_blocks - table_blocks;
    for (int i = b - table_blocks; i < tot.y; i += step) copy_page(a.pool, a.movers[i], a.holes[i], 0, 1);
}

static PoolView pool_view(const nd_pages* p, const char* what) {
    auto fail = [&](const std::string& m) { throw std::runtime_error(std::string(what) + ": " + m); };
    if (!p) fail("null pool");
    if (!p->pool) fail("null pointer");
    if (p->num_pages < 1 || p->layers < 1 || p->page_bytes < 1) fail("sizes must be positive");
    if (p->num_pages > 1 << 28) fail("more than 2^28 pages");
    if (p->page_bytes % 16 || p->page_stride % 16 || p->layer_stride % 16 || (uintptr_t)p->pool % 16)
        fail("the pool, its pages and strides must be 16-byte aligned");
    const bool pages_in = p->page_stride >= p->page_bytes && (p->layers == 1 || p->layer_stride >= (p->num_pages - 1) * p->page_stride + p->page_bytes);
    const bool layers_in = p->layers > 1 && p->layer_stride >= p->page_bytes &&
                           (p->num_pages == 1 || p->page_stride >= (p->layers - 1) * p->layer_stride + p->page_bytes);
    if (!pages_in && !layers_in) fail("pages overlap");
    return PoolView{(uint8_t*)p->pool, p->page_stride, p->layer_stride, p->page_bytes, p->layers};
}

static void check_table(const char* what, const int* table, int stride, int seqs, int cols) {
    auto fail = [&](const std::string& m) { throw std::runtime_error(std::string(what) + ": " + m); };
    if (!table) fail("null pointer");
    if (seqs < 1 || cols < 1 || seqs > 1 << 20) fail("a table has 1 to 2^20 sequences and at least one column");
    if (stride < cols) fail("table rows overlap");
    if ((long long)seqs * cols > 0x7fffffffLL) fail("more than 2^31 - 1 table entries");
}

static int blocks_of(int n) { return (n + PG_BLOCK - 1) / PG_BLOCK; }

static unsigned long long fork_ws(int pages, int n) {
    return 4ull * (3ull * pages + 2ull * n + blocks_of(pages) + blocks_of(n) + 2);
}
static unsigned long long compact_ws(int pages) { return 8ull * (blocks_of(pages) + 1) + 16ull * pages; }

template <typename... K, typename... A>
static void launch_behind(const char* what, void (*kernel)(K...), dim3 grid, int block, cudaStream_t st, bool first, A... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(block);
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = st && !first ? 1 : 0;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, K(args)...);
    if (e != cudaSuccess) throw std::runtime_error(std::string(what) + ": " + cudaGetErrorString(e));
    add_launches(1);
}

}  // namespace nd

using namespace nd;

extern "C" {

unsigned long long nd_op_pages_fork_ws(int num_pages, int n) { return num_pages < 1 || n < 0 ? 0 : fork_ws(num_pages, n); }

int nd_op_pages_fork(const nd_pages* pool, const int* table, int table_stride, int seqs, int cols, int page, const int* src,
                     const int* keep, const int* need, int n, const unsigned char* pinned, int* table_out, int* refs, int* info,
                     void* ws, unsigned long long ws_bytes, void* stream) {
    return op_call([&] {
        const char* what = "nd_op_pages_fork";
        auto fail = [&](const std::string& m) { throw std::runtime_error(std::string(what) + ": " + m); };
        ForkArgs a{};
        a.pool = pool_view(pool, what);
        check_table(what, table, table_stride, seqs, cols);
        if (n < 1 || n > 1 << 20) fail("n must be in [1, 2^20]");
        if ((long long)n * cols > 0x7fffffffLL) fail("more than 2^31 - 1 table entries");
        if (page < 1 || (long long)page * cols > 0x7fffffffLL) fail("page must be positive, a row below 2^31 positions");
        if (!src || !keep || !need || !table_out || !refs || !info) fail("null pointer");
        if (table_out == table) fail("the new table must not be the old one");
        if (!ws || (uintptr_t)ws % 16 || ws_bytes < fork_ws(pool->num_pages, n)) fail("the workspace is too small or not 16-byte aligned");
        const int N = pool->num_pages, nb = blocks_of(N), sb = blocks_of(n);
        a.table = table, a.table_stride = table_stride, a.seqs = seqs, a.cols = cols, a.pages = N, a.page = page, a.by_cols = FastDiv(cols);
        a.src = src, a.keep = keep, a.need = need, a.n = n, a.pinned = pinned;
        a.table_out = table_out, a.refs = refs, a.info = info;
        a.writers = (int32_t*)ws, a.first = a.writers + N, a.free_ids = a.first + N, a.fresh = a.free_ids + N;
        a.base = a.fresh + n, a.sums = a.base + n;
        OnDevice on(pool->device, what);
        cudaStream_t st = (cudaStream_t)stream;
        const int sms = device_sm_count();
        int totals = 0;  // their place in sums
        if (N <= PG_SMALL && (long long)n * cols <= PG_SMALL) {
            launch_behind(what, fork_plan_kernel, PG_CLUSTER, PG_BLOCK, st, true, a);
        } else {
            totals = nb + sb;
            launch_behind(what, pages_zero_kernel, std::min((N + 255) / 256, 4 * sms), 256, st, true, a.refs, a.writers, N);
            launch_behind(what, fork_count_kernel, (n + 3) / 4, 128, st, false, a);
            launch_behind(what, fork_sums_kernel, nb + sb, PG_BLOCK, st, false, a, nb);
            launch_behind(what, fork_lists_kernel, nb + sb, PG_BLOCK, st, false, a, nb);
        }
        // 8 KB of a layer's page a block at least, 2 CTAs an SM of copies at most
        const long long parts = std::min<long long>((pool->page_bytes + 8191) / 8192, std::max(1, 2 * sms / n));
        launch_behind(what, fork_assign_kernel, dim3(n, (unsigned)parts), 128, st, false, a, totals);
    });
}

unsigned long long nd_op_pages_compact_ws(int num_pages) { return num_pages < 1 ? 0 : compact_ws(num_pages); }

int nd_op_pages_compact(const nd_pages* pool, const int* table, int table_stride, int seqs, int cols, const unsigned char* pinned,
                        int* table_out, int* map, int* info, void* ws, unsigned long long ws_bytes, void* stream) {
    return op_call([&] {
        const char* what = "nd_op_pages_compact";
        auto fail = [&](const std::string& m) { throw std::runtime_error(std::string(what) + ": " + m); };
        CompactArgs a{};
        a.pool = pool_view(pool, what);
        check_table(what, table, table_stride, seqs, cols);
        if (!table_out || !map || !info) fail("null pointer");
        if (table_out == table) fail("the new table must not be the old one");
        if (!ws || (uintptr_t)ws % 16 || ws_bytes < compact_ws(pool->num_pages)) fail("the workspace is too small or not 16-byte aligned");
        const int N = pool->num_pages, nb = blocks_of(N);
        a.table = table, a.table_stride = table_stride, a.seqs = seqs, a.cols = cols, a.pages = N, a.by_cols = FastDiv(cols), a.pinned = pinned;
        a.table_out = table_out, a.map = map, a.info = info;
        a.sums = (int2*)ws;
        a.refs = (int32_t*)(a.sums + nb + 1), a.before = a.refs + N, a.movers = a.before + N, a.holes = a.movers + N;
        OnDevice on(pool->device, what);
        cudaStream_t st = (cudaStream_t)stream;
        const int sms = device_sm_count();
        int totals = 0;  // their place in sums
        if (N <= PG_SMALL && (long long)seqs * cols <= PG_SMALL) {
            launch_behind(what, compact_plan_kernel, std::min(nb, PG_PLAN), PG_BLOCK, st, true, a);
        } else {
            totals = nb;
            launch_behind(what, pages_zero_kernel, std::min((N + 255) / 256, 4 * sms), 256, st, true, a.refs, (int32_t*)nullptr, N);
            launch_behind(what, compact_count_kernel, (seqs + 3) / 4, 128, st, false, a);
            launch_behind(what, compact_sums_kernel, nb, PG_BLOCK, st, false, a);
            launch_behind(what, compact_lists_kernel, nb, PG_BLOCK, st, false, a);
        }
        const int map_blocks = totals ? (N + 127) / 128 : 0, table_blocks = (int)(((long long)seqs * cols + 127) / 128);
        launch_behind(what, compact_move_kernel, map_blocks + table_blocks + std::min(N, 32 * sms), 128, st, false, a, totals, map_blocks, table_blocks);
    });
}

}  // extern "C"
