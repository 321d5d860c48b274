/*
 * Page operators of a paged KV cache on sm_100a (include/kvpage.h): resize,
 * copy, fork, compact.
 *
 * Two kinds of kernel.  The bookkeeping (resize, fork's plan) is integer work
 * on a few thousand table entries and bound by latency: a chain of dependent
 * loads and atomics.  It runs in one thread-block cluster, whose hardware
 * barrier separates the phases, so that a call is one launch whatever its size;
 * the rows' prefix sums are computed by every CTA for itself in shared
 * memory.  The data movers (copy, compact) are bound by HBM bandwidth, two
 * bytes of traffic per byte moved, and keep four or eight 16-byte vectors per
 * thread in flight.
 */
#include "kvpage.h"
#include "adaptor.h"
#include "device_guard.h"
#include "fastdiv.h"

#include <cuda_runtime.h>

#include <cerrno>
#include <cstdint>
#include <mutex>

namespace {

constexpr int kPlanThreads = 1024;          /* at most; 256 for small calls, whose time is barriers and loads */
constexpr uint32_t kPlanCluster = 8;
constexpr uint32_t kUnit = 128;             /* table entries that a warp takes together, four to a lane */
constexpr uint32_t kMaxUnits = 2 * KVPAGE_MAX_CALL;
constexpr int32_t kRefused = INT32_MIN;     /* in a resize of compact's: the length of a row that it has refused and reported */

/* ---- the cluster's barrier and shared memory ---- */
__device__ __forceinline__ uint32_t cluster_rank()
{
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}

__device__ __forceinline__ uint32_t cluster_size()
{
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

__device__ __forceinline__ void cluster_sync()
{
    cluster_arrive();
    cluster_wait();
}

/* store v at `p`'s place in the shared memory of CTA `rank` of the cluster */
__device__ __forceinline__ void store_cluster(int32_t *p, uint32_t rank, int32_t v)
{
    uint32_t a = (uint32_t)__cvta_generic_to_shared(p), b;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(b) : "r"(a), "r"(rank));
    asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(b), "r"(v) : "memory");
}

/* Exclusive prefix sums of K arrays of n values each in place, n <= kMaxUnits;
 * total[k] is array k's sum.  A thread sums consecutive values. */
template <int K> __device__ __noinline__ void block_scan(int32_t *const *a, uint32_t n, int32_t *total)
{
    __shared__ int32_t warp_sum[K][32];
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const uint32_t each = (n + blockDim.x - 1) / blockDim.x, i0 = min(n, threadIdx.x * each), i1 = min(n, i0 + each);
    int32_t sum[K], inc[K];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; k++) {
        sum[k] = 0;
        for (uint32_t i = i0; i < i1; i++)
            sum[k] += a[k][i];
        inc[k] = sum[k];
    }
#pragma unroll
    for (int d = 1; d < 32; d <<= 1)
#pragma unroll
        for (int k = 0; k < K; k++) {
            const int32_t o = __shfl_up_sync(~0u, inc[k], d);
            if (lane >= d)
                inc[k] += o;
        }
#pragma unroll
    for (int k = 0; k < K; k++)
        if (lane == 31)
            warp_sum[k][warp] = inc[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; k++) {
        const int32_t w = lane < warps ? warp_sum[k][lane] : 0;
        int32_t run = inc[k] - sum[k] + __reduce_add_sync(~0u, lane < warp ? w : 0);
        total[k] = __reduce_add_sync(~0u, w);
        for (uint32_t i = i0; i < i1; i++) {
            const int32_t v = a[k][i];
            a[k][i] = run;
            run += v;
        }
    }
    __syncthreads();
}

/* A call's second kernel is started while the first one runs (launch_after); it
 * waits here for the first one's results, the first one lets it start there. */
__device__ __forceinline__ void await_first() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void start_second() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

/* sets bit r; true if it was set already */
__device__ __forceinline__ bool test_and_set(uint32_t *bits, uint32_t r)
{
    const uint32_t m = 1u << (r & 31);
    return atomicOr(&bits[r >> 5], m) & m;
}

__device__ __forceinline__ bool test_bit(const uint32_t *bits, uint32_t r)
{
    return bits[r >> 5] >> (r & 31) & 1;
}

__device__ __forceinline__ uint32_t pages_of(uint32_t tokens, uint32_t bs)
{
    return tokens / bs + (tokens % bs != 0);
}

__device__ __forceinline__ int32_t free_pages(const kv_page_state &s)
{
    const int32_t c = *s.free_count;
    return min(max(c, 0), (int32_t)s.num_pages);
}

/* the row that unit u of the prefix sums `first` belongs to */
__device__ __forceinline__ uint32_t row_of(const int32_t *first, uint32_t n, int32_t u)
{
    uint32_t lo = 0, hi = n - 1;
    while (lo < hi) {
        const uint32_t mid = (lo + hi + 1) / 2;
        if (first[mid] <= u)
            lo = mid;
        else
            hi = mid - 1;
    }
    return lo;
}

/* ------------------------------------------------------------------------
 * resize.  Entry k of the call's row i has the number i * width + k, and a
 * dropped page's place in the push order is its highest number:
 *   A  every dropped entry takes one reference off its page and raises the
 *      page's mark to its number + 1 (both commute: any order, same result)
 *   B  the entry whose number the mark holds, of a page without references,
 *      stands for the page; warps count these unit by unit, the counts go to
 *      every CTA's shared memory, and each CTA scans them
 *   C  those entries push their pages
 *   D  growing rows pop, marks go back to zero, lengths and counts are written
 * with a cluster barrier between phases.  What is dropped or taken is cut into
 * units of 128 entries of a row (more where that would be too many units), so
 * that a lane has four loads or atomics in flight and long rows are shared by
 * warps: replacing 256 rows of 170 pages takes 21 us, with a warp per row and an
 * entry per lane 44; 64 rows that change by a few pages 9 us.  A reference is taken back where a page had none left, so a
 * page freed twice is neither pushed twice nor left negative.
 * ---------------------------------------------------------------------- */
__global__ void __launch_bounds__(kPlanThreads, 1)
kv_page_resize_kernel(const kv_page_state s, const int32_t *rows, const int32_t *lens, uint32_t n, int32_t *__restrict__ status,
                      bool compacted)
{
    extern __shared__ int32_t sm[];
    int32_t *row = sm, *old_p = sm + n, *new_p = sm + 2 * n, *need = sm + 3 * n;
    int32_t *drops = sm + 4 * n, *takes = sm + 5 * n;       /* units of the rows before */
    int32_t *length = sm + 6 * n;                           /* lens, which may be the state's own: read once */
    const uint32_t words = (s.num_rows + 31) / 32;
    uint32_t *seen = reinterpret_cast<uint32_t *>(sm + 7 * n), *twice = seen + words;
    int32_t *gone = sm + 7 * n + 2 * words;                 /* pages pushed by the units before */
    __shared__ int32_t served, all_drop, all_take;
    const uint32_t rank = cluster_rank(), ctas = cluster_size();
    const uint32_t lane = threadIdx.x & 31, warp0 = rank * (blockDim.x >> 5) + (threadIdx.x >> 5), warps = ctas * (blockDim.x >> 5);

    for (uint32_t i = threadIdx.x; i < 2 * words; i += blockDim.x)
        seen[i] = 0;
    if (threadIdx.x == 0)
        served = all_drop = all_take = 0;
    await_first();
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < n; i += blockDim.x) {
        const int32_t r = rows[i];
        row[i] = r;
        if (r >= 0 && (uint32_t)r < s.num_rows && test_and_set(seen, r))
            test_and_set(twice, r);
    }
    const int32_t count = free_pages(s);
    __syncthreads();
    int32_t drop = 0, take = 0;
    for (uint32_t i = threadIdx.x; i < n; i += blockDim.x) {
        const int32_t r = row[i], to = lens[i];
        bool ok = r >= 0 && (uint32_t)r < s.num_rows && to >= 0;
        uint32_t a = 0, b = 0;
        if (ok) {
            const int32_t from = s.lens[r];
            a = pages_of(max(from, 0), s.block_size);
            b = pages_of(to, s.block_size);
            ok = !test_bit(twice, r) && from >= 0 && a <= s.width && b <= s.width;
        }
        if (!ok) {
            if (rank == 0 && !(compacted && to == kRefused))
                atomicOr(s.error, KVPAGE_ERR_ROW);
            row[i] = -1;
            a = b = 0;
        }
        length[i] = to;
        old_p[i] = a;
        new_p[i] = b;
        need[i] = b > a ? b - a : 0;
        drop += a > b ? a - b : 0;
        take += need[i];
    }
    if (drop)
        atomicAdd(&all_drop, drop);
    if (take)
        atomicAdd(&all_take, take);
    __syncthreads();
    /* entries of a unit: at most as many units of n rows as kMaxUnits holds */
    uint32_t unit = kUnit;
    while ((uint32_t)max(all_drop, all_take) / unit > kMaxUnits - KVPAGE_MAX_CALL)
        unit *= 2;
    for (uint32_t i = threadIdx.x; i < n; i += blockDim.x) {
        const int32_t d = old_p[i] - new_p[i];
        drops[i] = d > 0 ? (d + unit - 1) / unit : 0;
        takes[i] = (need[i] + unit - 1) / unit;
    }
    int32_t total[3], pushed = 0;
    {
        int32_t *arrays[3] = {drops, takes, need};
        block_scan<3>(arrays, n, total);
    }
    const int32_t drop_units = total[0], take_units = total[1];
    if (drop_units > 0 && drop_units <= (int32_t)warps && unit == kUnit) {
        /* a unit per warp: its pages stay in registers from phase to phase */
        const bool mine = warp0 < (uint32_t)drop_units;
        int32_t page[4], number = 0, c = 0;
        uint32_t on = 0, stands = 0;
        if (mine) {
            const uint32_t i = row_of(drops, n, warp0);
            const int32_t k = new_p[i] + (warp0 - drops[i]) * (int32_t)kUnit + (int32_t)lane;
            const int32_t *t = s.table + (int64_t)row[i] * s.table_stride;
            number = (int32_t)(i * s.width) + k + 1;
            int32_t had[4];
#pragma unroll
            for (int j = 0; j < 4; j++)
                page[j] = k + 32 * j < old_p[i] ? t[k + 32 * j] : 0;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if (k + 32 * j >= old_p[i])
                    continue;
                if (page[j] >= 0 && (uint32_t)page[j] < s.num_pages) {
                    on |= 1u << j;
                    had[j] = atomicSub(&s.refs[page[j]], 1);
                } else {
                    atomicOr(s.error, KVPAGE_ERR_PAGE);
                }
            }
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if (!(on >> j & 1))
                    continue;
                if (had[j] >= 1) {
                    atomicMax(&s.marks[page[j]], number + 32 * j);
                } else {
                    atomicAdd(&s.refs[page[j]], 1);
                    atomicOr(s.error, KVPAGE_ERR_REFS);
                }
            }
        }
        cluster_sync();
        if (mine) {
            int32_t mark[4], refs[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                mark[j] = on >> j & 1 ? __ldcg(&s.marks[page[j]]) : 0;
                refs[j] = on >> j & 1 ? __ldcg(&s.refs[page[j]]) : 1;
            }
#pragma unroll
            for (int j = 0; j < 4; j++)
                stands |= (uint32_t)(mark[j] == number + 32 * j && refs[j] == 0) << j;
            c = __reduce_add_sync(~0u, __popc(stands));
            if (lane < ctas)
                store_cluster(&gone[warp0], lane, c);
        }
        cluster_sync();
        {
            int32_t *arrays[1] = {gone};
            block_scan<1>(arrays, drop_units, &pushed);
        }
        if (mine) {
            int32_t place = count + gone[warp0];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const uint32_t m = __ballot_sync(~0u, stands >> j & 1);
                const int32_t at = place + __popc(m & ((1u << lane) - 1));
                if ((stands >> j & 1) && (uint32_t)at < s.num_pages)
                    s.free_list[at] = page[j];
                place += __popc(m);
            }
        }
        cluster_sync();
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (on >> j & 1)
                s.marks[page[j]] = 0;
    } else if (drop_units) {
        /* the same in one loop over the warp's units for the four phases */
#pragma unroll 1
        for (int phase = 0; phase < 4; phase++) {
            if (phase)
                cluster_sync();
            if (phase == 2) {
                int32_t *arrays[1] = {gone};
                block_scan<1>(arrays, drop_units, &pushed);
            }
#pragma unroll 1
            for (int32_t u = warp0; u < drop_units; u += warps) {
                const uint32_t i = row_of(drops, n, u);
                const int32_t *t = s.table + (int64_t)row[i] * s.table_stride;
                const int32_t k0 = new_p[i] + (u - drops[i]) * (int32_t)unit, k1 = min(old_p[i], k0 + (int32_t)unit);
                int32_t c = 0;
#pragma unroll 1
                for (int32_t k = k0 + lane; k - (int32_t)lane < k1; k += kUnit) {
                    const int32_t number = (int32_t)(i * s.width) + k + 1;
                    int32_t page[4], mark[4], refs[4];
                    bool on[4];
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        page[j] = k + 32 * j < k1 ? t[k + 32 * j] : 0;
                        on[j] = k + 32 * j < k1 && page[j] >= 0 && (uint32_t)page[j] < s.num_pages;
                    }
                    if (phase == 0) {
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            if (on[j])
                                refs[j] = atomicSub(&s.refs[page[j]], 1);
                            else if (k + 32 * j < k1)
                                atomicOr(s.error, KVPAGE_ERR_PAGE);
                        }
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            if (!on[j])
                                continue;
                            if (refs[j] >= 1) {
                                atomicMax(&s.marks[page[j]], number + 32 * j);
                            } else {
                                atomicAdd(&s.refs[page[j]], 1);
                                atomicOr(s.error, KVPAGE_ERR_REFS);
                            }
                        }
                    } else if (phase == 3) {
#pragma unroll
                        for (int j = 0; j < 4; j++)
                            if (on[j])
                                s.marks[page[j]] = 0;
                    } else {
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            mark[j] = on[j] ? __ldcg(&s.marks[page[j]]) : 0;
                            refs[j] = on[j] ? __ldcg(&s.refs[page[j]]) : 1;
                        }
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            const bool stands = mark[j] == number + 32 * j && refs[j] == 0;
                            const uint32_t m = __ballot_sync(~0u, stands);
                            if (phase == 2) {
                                const int32_t place = count + gone[u] + c + __popc(m & ((1u << lane) - 1));
                                if (stands && (uint32_t)place < s.num_pages)
                                    s.free_list[place] = page[j];
                            }
                            c += __popc(m);
                        }
                    }
                }
                if (phase == 1 && lane < ctas)
                    store_cluster(&gone[u], lane, c);
            }
        }
    } else {
        cluster_sync();             /* every CTA has read the lengths and the count */
    }
    const int32_t have = min(count + pushed, (int32_t)s.num_pages);
    {
#pragma unroll 1
        for (int32_t u = warp0; u < take_units; u += warps) {
            const uint32_t i = row_of(takes, n, u);
            const int32_t want = new_p[i] - old_p[i], k0 = (u - takes[i]) * (int32_t)unit, k1 = min(want, k0 + (int32_t)unit);
            if (need[i] + want > have)
                continue;
            int32_t *t = s.table + (int64_t)row[i] * s.table_stride + old_p[i];
#pragma unroll 1
            for (int32_t k = k0 + lane; k < k1; k += kUnit) {
                int32_t page[4];
#pragma unroll
                for (int j = 0; j < 4; j++)
                    page[j] = k + 32 * j < k1 ? __ldcg(&s.free_list[have - 1 - need[i] - k - 32 * j]) : 0;
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (k + 32 * j < k1) {
                        t[k + 32 * j] = page[j];
                        if (page[j] >= 0 && (uint32_t)page[j] < s.num_pages)
                            s.refs[page[j]] = 1;
                        else
                            atomicOr(s.error, KVPAGE_ERR_PAGE);
                    }
            }
        }
    }
    if (rank)
        return;
    for (uint32_t i = threadIdx.x; i < n; i += blockDim.x) {
        const int32_t r = row[i], want = new_p[i] - old_p[i];
        const bool fits = want <= 0 || need[i] + want <= have;
        if (want > 0 && fits)
            atomicMax(&served, need[i] + want);
        if (r >= 0 && fits)
            s.lens[r] = length[i];
        if (status)
            status[i] = r < 0 ? KVPAGE_INVALID : fits ? KVPAGE_OK : KVPAGE_NO_PAGES;
    }
    __syncthreads();
    if (threadIdx.x == 0)
        *s.free_count = have - served;
}

/* ------------------------------------------------------------------------
 * fork's plan: what each child gets, the tables and the references; the pages
 * to copy go to pairs[3 * i] = (source, destination, tokens), 0 tokens where
 * there is nothing to copy.  One cluster, a warp per child.  The parents' pages
 * are looked through before any are dealt out, so that a child that would share
 * a bad one takes none; the warp that finds it tells every CTA.
 * ---------------------------------------------------------------------- */
__global__ void __launch_bounds__(kPlanThreads, 1)
kv_page_fork_kernel(const kv_page_state s, const int32_t *__restrict__ parents, const int32_t *__restrict__ children,
                    uint32_t n, int32_t *__restrict__ pairs, int32_t *__restrict__ status)
{
    extern __shared__ int32_t sm[];
    int32_t *from = sm, *child = sm + n, *length = sm + 2 * n, *need = sm + 3 * n;
    const uint32_t words = (s.num_rows + 31) / 32;
    int32_t *bad_parent = sm + 4 * n;
    uint32_t *seen = reinterpret_cast<uint32_t *>(sm + 5 * n), *twice = seen + words, *parent = seen + 2 * words;
    __shared__ int32_t served;
    const uint32_t rank = cluster_rank(), ctas = cluster_size();
    const uint32_t lane = threadIdx.x & 31, warp0 = rank * (blockDim.x >> 5) + (threadIdx.x >> 5), warps = ctas * (blockDim.x >> 5);

    start_second();
    for (uint32_t i = threadIdx.x; i < n; i += blockDim.x)
        bad_parent[i] = 0;
    cluster_arrive();
    for (uint32_t i = threadIdx.x; i < 3 * words; i += blockDim.x)
        seen[i] = 0;
    if (threadIdx.x == 0)
        served = 0;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < n; i += blockDim.x) {
        const int32_t p = parents[i], c = children[i];
        from[i] = p;
        child[i] = c;
        if (p >= 0 && (uint32_t)p < s.num_rows)
            test_and_set(parent, p);
        if (c >= 0 && (uint32_t)c < s.num_rows && test_and_set(seen, c))
            test_and_set(twice, c);
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < n; i += blockDim.x) {
        const int32_t p = from[i], c = child[i];
        bool ok = p >= 0 && (uint32_t)p < s.num_rows && c >= 0 && (uint32_t)c < s.num_rows && !test_bit(twice, c) &&
                  !test_bit(parent, c);
        int32_t len = 0;
        if (ok) {
            len = s.lens[p];
            ok = s.lens[c] == 0 && len >= 0 && pages_of(max(len, 0), s.block_size) <= s.width;
        }
        if (!ok) {
            if (rank == 0)
                atomicOr(s.error, KVPAGE_ERR_ROW);
            child[i] = -1;
            len = 0;
        }
        length[i] = len;
    }
    const int32_t have = free_pages(s);
    __syncthreads();
    cluster_wait();                 /* every CTA's bad_parent is zero */
    int32_t kept[4] = {};           /* the first pages of the warp's first child */
    for (uint32_t i = warp0; i < n; i += warps) {
        if (child[i] < 0)
            continue;
        const int32_t *tp = s.table + (int64_t)from[i] * s.table_stride;
        const int32_t held = (int32_t)pages_of(length[i], s.block_size);
        bool bad = false;
#pragma unroll 1
        for (int32_t k = lane; k - (int32_t)lane < held; k += kUnit) {
            int32_t page[4];
#pragma unroll
            for (int j = 0; j < 4; j++)
                page[j] = k + 32 * j < held ? tp[k + 32 * j] : 0;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                bad |= (uint32_t)page[j] >= s.num_pages;
                if (i == warp0 && k == (int32_t)lane)
                    kept[j] = page[j];
            }
        }
        if (__any_sync(~0u, bad) && lane < ctas)
            store_cluster(&bad_parent[i], lane, 1);
    }
    cluster_sync();                 /* every CTA has read the lengths and the count, and looked through its pages */
    for (uint32_t i = threadIdx.x; i < n; i += blockDim.x) {
        if (bad_parent[i]) {
            if (rank == 0)
                atomicOr(s.error, KVPAGE_ERR_PAGE);
            child[i] = -1;
            length[i] = 0;
        }
        need[i] = length[i] % (int32_t)s.block_size != 0;
    }
    int32_t wanted;
    int32_t *arrays[1] = {need};
    block_scan<1>(arrays, n, &wanted);
    for (uint32_t i = threadIdx.x; i < n; i += blockDim.x)
        if (length[i] % (int32_t)s.block_size && need[i] < have)
            atomicMax(&served, need[i] + 1);
    for (uint32_t i = warp0; i < n; i += warps) {
        const int32_t c = child[i], len = length[i];
        const int32_t full = len / (int32_t)s.block_size, tail = len % (int32_t)s.block_size;
        const int32_t *tp = s.table + (int64_t)(c >= 0 ? from[i] : 0) * s.table_stride;
        bool fits = c >= 0 && (!tail || need[i] < have);
        const int32_t src = fits && tail ? tp[full] : 0, dst = fits && tail ? s.free_list[have - 1 - need[i]] : 0;
        const bool lost = (uint32_t)dst >= s.num_pages;     /* not a page: nobody's from now on */
        fits = fits && !lost;
        if (fits) {
            int32_t *tc = s.table + (int64_t)c * s.table_stride;
#pragma unroll 1
            for (int32_t k = lane; k < full; k += kUnit) {
                int32_t page[4];
                const bool held = i == warp0 && k == (int32_t)lane;
#pragma unroll
                for (int j = 0; j < 4; j++)
                    page[j] = held ? kept[j] : k + 32 * j < full ? tp[k + 32 * j] : 0;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    if (k + 32 * j >= full)
                        break;
                    tc[k + 32 * j] = page[j];
                    atomicAdd(&s.refs[page[j]], 1);
                }
            }
            if (tail && lane == 0) {
                tc[full] = dst;
                s.refs[dst] = 1;
            }
        }
        if (lane == 0) {
            if (lost)
                atomicOr(s.error, KVPAGE_ERR_PAGE);
            pairs[3 * i] = src;
            pairs[3 * i + 1] = dst;
            pairs[3 * i + 2] = fits ? tail : 0;
            if (fits)
                s.lens[c] = len;
            if (status)
                status[i] = fits ? KVPAGE_OK : c < 0 || lost ? KVPAGE_INVALID : KVPAGE_NO_PAGES;
        }
    }
    __syncthreads();
    if (rank == 0 && threadIdx.x == 0)
        *s.free_count = have - served;
}

/* ---- the planes ---- */
template <int V> struct VecOf;
template <> struct VecOf<16> { using T = uint4; };
template <> struct VecOf<8> { using T = uint2; };
template <> struct VecOf<4> { using T = uint32_t; };
template <> struct VecOf<2> { using T = uint16_t; };
template <> struct VecOf<1> { using T = uint8_t; };

struct Planes {
    const uint64_t *layer_k, *layer_v;
    int32_t *error;
    uint64_t stride;        /* bytes from page to page */
    uint32_t unit, head_bytes, bs, layers, kvs, pages;
};

Planes planes_of(const kv_page_cache *c)
{
    Planes p{};
    p.layer_k = c->layer_k;
    p.layer_v = c->layer_v;
    p.error = c->error;
    p.stride = c->block_stride ? c->block_stride : (uint64_t)c->block_size * c->unit_bytes;
    p.unit = c->unit_bytes;
    p.head_bytes = c->head_bytes;
    p.bs = c->block_size;
    p.layers = c->num_layers;
    p.kvs = c->layer_v ? 2 : 1;
    p.pages = c->num_pages;
    return p;
}

/* the widest vector that no token, head, page or base of the planes splits */
int vector_of(const kv_page_cache *c)
{
    const uint64_t all = (uint64_t)c->unit_bytes | c->head_bytes | c->block_stride | (c->base_align ? c->base_align : 16) | 16;
    return (int)(all & (~all + 1));
}

bool cache_ok(const kv_page_cache *c)
{
    if (!c || !c->layer_k || !c->error || !c->unit_bytes || !c->block_size || !c->num_layers || !c->num_pages ||
        c->num_layers > INT32_MAX / 2 || c->num_pages > INT32_MAX || (c->base_align & (c->base_align - 1)))
        return false;
    const uint64_t run = (uint64_t)c->block_size * c->unit_bytes;
    return run < (1ull << 31) && (!c->block_stride || c->block_stride >= run) &&
           !(c->head_bytes && c->unit_bytes % c->head_bytes);
}

bool state_ok(const kv_page_state *s)
{
    return s && s->table && s->lens && s->refs && s->free_list && s->free_count && s->marks && s->error && s->width &&
           s->table_stride >= (int64_t)s->width && s->num_rows && s->num_pages && s->num_pages <= INT32_MAX &&
           s->block_size && s->block_size <= INT32_MAX;
}

__device__ __forceinline__ uint8_t *base_of(const Planes &p, uint32_t lk)
{
    return reinterpret_cast<uint8_t *>((p.kvs == 2 && (lk & 1) ? p.layer_v : p.layer_k)[p.kvs == 2 ? lk >> 1 : lk]);
}

template <int VEC>
__device__ __forceinline__ uint8_t *plane(const Planes &p, uint32_t lk)
{
    uint8_t *base = base_of(p, lk);
    if (!base || reinterpret_cast<uintptr_t>(base) % VEC) {
        atomicOr(p.error, KVPAGE_ERR_ALIGN);
        return nullptr;
    }
    return base;
}

/* ------------------------------------------------------------------------
 * copy.  A page in a plane is one run of vectors in every geometry.  Where a run
 * fills CTAs of 2048 vectors, a CTA moves that much of one run: four pages of 64
 * planes of 32 KiB take 3.6 us, 500 of 27 planes of 72 KiB 297 us (6.7 TB/s).
 * Shorter runs (4 KiB: one head, 16 tokens) go to a warp each, which finds its
 * page, plane and tokens once: 256 pages of 160 such planes take 53 us (6.3
 * TB/s), the first half of them 28; with a CTA per run the half took 95, with
 * CTAs of 2048 vectors that each thread places by itself 37.
 * With a token count, a token-major page stops early and a head-major one skips
 * the tokens behind it.  `pack` is the distance between the entries of the
 * lists: 1, or 3 for fork's pairs.
 * ---------------------------------------------------------------------- */
constexpr int kMoveThreads = 256;
constexpr int kMoveUnroll = 8;
constexpr uint32_t kMoveVectors = kMoveThreads * kMoveUnroll;

struct Copy {
    const int32_t *src, *dst, *tokens;
    uint32_t pack, n, planes_per_grid;  /* planes of one grid row */
    uint32_t run, per_token;            /* vectors of a page, of a token of one head */
    FastDiv per_head;                   /* of a page's head */
    FastDiv pairs;          /* pages; for long runs, CTAs of one */
};

/* grid: (pages x CTAs of a run, planes) */
template <int VEC>
__global__ void __launch_bounds__(kMoveThreads) kv_page_copy_run_kernel(const Planes p, const __grid_constant__ Copy c)
{
    using T = typename VecOf<VEC>::T;
    await_first();
    const uint32_t i = fdiv(blockIdx.x, c.pairs), x0 = (blockIdx.x - i * c.pairs.d) * kMoveVectors + threadIdx.x;
    const int32_t a = c.src[(uint64_t)i * c.pack], b = c.dst[(uint64_t)i * c.pack];
    const int32_t keep = c.tokens ? min(max(c.tokens[(uint64_t)i * c.pack], 0), (int32_t)p.bs) : (int32_t)p.bs;
    if (!keep || a == b)
        return;
    if (a < 0 || (uint32_t)a >= p.pages || b < 0 || (uint32_t)b >= p.pages) {
        if (threadIdx.x == 0)
            atomicOr(p.error, KVPAGE_ERR_PAGE);
        return;
    }
    uint8_t *base = plane<VEC>(p, blockIdx.y);
    if (!base)
        return;
    const T *from = reinterpret_cast<const T *>(base + (uint64_t)a * p.stride);
    T *to = reinterpret_cast<T *>(base + (uint64_t)b * p.stride);
    const bool part = p.head_bytes && keep < (int32_t)p.bs;
    const uint32_t all = p.head_bytes ? c.run : (uint32_t)keep * c.per_token, used = (uint32_t)keep * c.per_token;
    T v[kMoveUnroll];
    bool on[kMoveUnroll];
#pragma unroll
    for (int u = 0; u < kMoveUnroll; u++) {
        const uint32_t x = x0 + u * kMoveThreads;
        on[u] = x < all && !(part && x - fdiv(x, c.per_head) * c.per_head.d >= used);
        if (on[u])
            v[u] = from[x];
    }
#pragma unroll
    for (int u = 0; u < kMoveUnroll; u++)
        if (on[u])
            to[x0 + u * kMoveThreads] = v[u];
}

/* a warp per page and plane */
template <int VEC>
__global__ void __launch_bounds__(kMoveThreads, 8) kv_page_copy_warp_kernel(const Planes p, const __grid_constant__ Copy c)
{
    using T = typename VecOf<VEC>::T;
    constexpr int kUnroll = 4;
    const uint32_t lk0 = blockIdx.y * c.planes_per_grid, lane = threadIdx.x % 32;
    const uint32_t item = blockIdx.x * (kMoveThreads / 32) + threadIdx.x / 32;
    if (item >= min(c.planes_per_grid, p.layers * p.kvs - lk0) * c.n)
        return;
    const uint32_t plane_in = fdiv(item, c.pairs), i = item - plane_in * c.n;
    await_first();
    const int32_t a = c.src[(uint64_t)i * c.pack], b = c.dst[(uint64_t)i * c.pack];
    const int32_t keep = c.tokens ? min(max(c.tokens[(uint64_t)i * c.pack], 0), (int32_t)p.bs) : (int32_t)p.bs;
    uint8_t *base = plane<VEC>(p, lk0 + plane_in);
    if (!keep || a == b || !base)
        return;
    if (a < 0 || (uint32_t)a >= p.pages || b < 0 || (uint32_t)b >= p.pages) {
        if (lane == 0)
            atomicOr(p.error, KVPAGE_ERR_PAGE);
        return;
    }
    const T *from = reinterpret_cast<const T *>(base + (uint64_t)a * p.stride);
    T *to = reinterpret_cast<T *>(base + (uint64_t)b * p.stride);
    const uint32_t used = (uint32_t)keep * c.per_token;
    const bool part = p.head_bytes && keep < (int32_t)p.bs && c.per_head.d < c.run;
    const uint32_t all = part || keep == (int32_t)p.bs ? c.run : used;
#pragma unroll 1
    for (uint32_t x0 = lane; x0 < all; x0 += 32 * kUnroll) {
        T v[kUnroll];
        bool on[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; u++) {
            const uint32_t x = x0 + u * 32;
            on[u] = x < all && !(part && x - fdiv(x, c.per_head) * c.per_head.d >= used);
            if (on[u])
                v[u] = from[x];
        }
#pragma unroll
        for (int u = 0; u < kUnroll; u++)
            if (on[u])
                to[x0 + u * 32] = v[u];
    }
}

/* ------------------------------------------------------------------------
 * compact.  keep[j] ascends strictly from start, so token j moves from
 * keep[j] >= start + j: never up.  In one plane, a batch of tokens may be
 * stored once it and every batch before it have been loaded; the stores of a
 * batch end at or below its own highest source and so never reach the sources
 * of the next.  A CTA therefore takes one row and a few slices of planes (a
 * slice: some bytes of each token) and walks their tokens in order: load a
 * batch into registers, barrier, store it.  Slices are independent.
 *
 * Every CTA checks its row's whole list and every plane's base before it moves a
 * byte, so that all of them decide alike; 4 bytes of list against 64 bytes or
 * more of slice.
 * The first CTA of a row leaves the new length for resize, or kRefused.
 * Half of 16000 tokens of 64 planes of 2 KiB units: 305 us, 5.2 TB/s; up to 5 of
 * 24 tokens of 64 rows: 17 us, most of it the checks' dependent loads.
 * ---------------------------------------------------------------------- */
template <int VEC>
__global__ void __launch_bounds__(kMoveThreads, 4)
kv_page_compact_kernel(const Planes p, const kv_page_state s, const int32_t *__restrict__ rows,
                       const int32_t *__restrict__ start, const int32_t *__restrict__ keep,
                       const int32_t *__restrict__ offsets, uint32_t num_keep, uint32_t n,
                       uint32_t slice_vecs, uint32_t slices, uint32_t slices_per_cta, int32_t *__restrict__ new_lens)
{
    using T = typename VecOf<VEC>::T;
    __shared__ uint64_t src_off[kMoveVectors], dst_off[kMoveVectors];
    __shared__ int32_t s_first, s_bad;
    auto all_see = [&](int32_t bits) {          /* the OR of every thread's bits */
        if (bits)
            atomicOr(&s_bad, bits);
        __syncthreads();
        return s_bad;
    };
    const uint32_t i = blockIdx.y;
    const int32_t r = rows[i], st = start[i], o0 = offsets[i], o1 = offsets[i + 1];
    int32_t bad = 0;
    start_second();
    if (threadIdx.x == 0) {
        s_first = INT32_MAX;
        s_bad = 0;
    }
    __syncthreads();
    for (uint32_t k = threadIdx.x; k < n; k += kMoveThreads)
        if (k != i && rows[k] == r)
            bad = KVPAGE_ERR_ROW;
    for (uint32_t lk = threadIdx.x; lk < p.layers * p.kvs; lk += kMoveThreads)
        if (!plane<VEC>(p, lk))
            bad |= KVPAGE_ERR_ALIGN;
    int32_t len = 0;
    if (r < 0 || (uint32_t)r >= s.num_rows) {
        bad = KVPAGE_ERR_ROW;
    } else {
        len = s.lens[r];
        if (len < 0 || pages_of(max(len, 0), s.block_size) > s.width)
            bad = KVPAGE_ERR_ROW;
    }
    if (o0 < 0 || o1 < o0 || (uint32_t)o1 > num_keep || st < 0 || st > len)
        bad |= KVPAGE_ERR_KEEP;
    bad = all_see(bad);
    __syncthreads();                            /* s_bad has been read before it grows */
    const int32_t m = bad ? 0 : o1 - o0;
    const int32_t *mine = keep + (bad ? 0 : o0);
    const int32_t *t = s.table + (int64_t)(bad ? 0 : r) * s.table_stride;
    int32_t first = INT32_MAX;
    for (int32_t j = threadIdx.x; j < m; j += kMoveThreads) {
        const int32_t x = mine[j], before = j ? mine[j - 1] : st - 1;
        if (x <= before || x >= len)
            bad |= KVPAGE_ERR_KEEP;
        if (x != st + j)
            first = min(first, j);
    }
    if (first != INT32_MAX)
        atomicMin(&s_first, first);
    bad = all_see(bad);
    __syncthreads();
    first = bad ? m : min(s_first, m);
    if (first < m) {
        const int32_t b0 = (st + first) / (int32_t)p.bs, b1 = (st + m - 1) / (int32_t)p.bs;
        for (int32_t b = b0 + (int32_t)threadIdx.x; b <= b1; b += kMoveThreads) {
            const int32_t page = t[b];
            if (page < 0 || (uint32_t)page >= s.num_pages)
                bad |= KVPAGE_ERR_PAGE;
            else if (s.refs[page] != 1)
                bad |= KVPAGE_ERR_REFS;
        }
        for (int32_t j = first + (int32_t)threadIdx.x; j < m; j += kMoveThreads) {
            const int32_t page = t[mine[j] / (int32_t)p.bs];
            if (page < 0 || (uint32_t)page >= s.num_pages)
                bad |= KVPAGE_ERR_PAGE;
        }
    }
    bad = all_see(bad);
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        new_lens[i] = bad ? kRefused : st + m;
        if (bad)
            atomicOr(s.error, bad);
    }
    if (bad || first >= m)
        return;

    /* thread = (token row, vector of the slice); slices side by side in a
     * batch where the tokens are few */
    const uint32_t q0 = blockIdx.x * slices_per_cta, q1 = min(q0 + slices_per_cta, slices);
    const uint32_t per_pass = kMoveThreads / slice_vecs;
    const uint32_t tok_row = threadIdx.x / slice_vecs, vec = threadIdx.x - tok_row * slice_vecs;
    const uint32_t moved = m - first;
    const uint32_t batch = min(moved, per_pass * kMoveUnroll);      /* tokens of a batch */
    const uint32_t group = max(1u, per_pass * kMoveUnroll / batch); /* slices of a batch */
    const uint32_t slices_per_plane = p.unit / (slice_vecs * VEC);
    const uint64_t token_bytes = p.head_bytes ? p.head_bytes : p.unit;
    for (uint32_t j0 = 0; j0 < moved; j0 += batch) {
        const uint32_t tokens = min(batch, moved - j0);
        __syncthreads();
        for (uint32_t j = threadIdx.x; j < tokens; j += kMoveThreads) {
            const uint32_t to = st + first + j0 + j, x = mine[first + j0 + j];
            src_off[j] = (uint64_t)t[x / p.bs] * p.stride + (x % p.bs) * token_bytes;
            dst_off[j] = (uint64_t)t[to / p.bs] * p.stride + (to % p.bs) * token_bytes;
        }
        __syncthreads();
        for (uint32_t q = q0; q < q1; q += group) {
            T v[kMoveUnroll];
            T *to[kMoveUnroll];
#pragma unroll
            for (int u = 0; u < kMoveUnroll; u++) {
                const uint32_t slot = u * per_pass + tok_row;
                const uint32_t g = group == 1 ? 0 : slot / tokens, j = group == 1 ? slot : slot - g * tokens;
                to[u] = nullptr;
                if (tok_row < per_pass && j < tokens && g < group && q + g < q1) {
                    const uint32_t lk = (q + g) / slices_per_plane, sl = q + g - lk * slices_per_plane;
                    uint8_t *base = base_of(p, lk);
                    const uint32_t o = (sl * slice_vecs + vec) * VEC;
                    /* byte o of a token's unit: a head-major page holds head o / head_bytes apart */
                    const uint64_t at = p.head_bytes ? (uint64_t)(o / p.head_bytes) * p.bs * p.head_bytes + o % p.head_bytes : o;
                    v[u] = *reinterpret_cast<const T *>(base + src_off[j] + at);
                    to[u] = reinterpret_cast<T *>(base + dst_off[j] + at);
                }
            }
            __syncthreads();
#pragma unroll
            for (int u = 0; u < kMoveUnroll; u++)
                if (to[u])
                    *to[u] = v[u];
        }
    }
}

/* ---- launches ---- */
/* A launch; `after`: as the second kernel of a call (await_first).  Only what the
 * launch itself returns counts: the thread's last error may be that of an
 * earlier call that has nothing to do with this one, and a call that took it
 * for its own would stop between its two kernels. */
template <typename... P, typename... A>
int launch(void (*kernel)(P...), dim3 grid, uint32_t threads, uint32_t cluster, size_t smem, bool after, cudaStream_t stream, A... args)
{
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr[2];
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = attr;
    if (cluster) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
        attr[cfg.numAttrs].val.clusterDim.x = cluster;
        attr[cfg.numAttrs].val.clusterDim.y = 1;
        attr[cfg.numAttrs++].val.clusterDim.z = 1;
    }
    if (after) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (cudaLaunchKernelEx(&cfg, kernel, args...) != cudaSuccess) {
        cudaGetLastError();
        return -EIO;
    }
    g_cc_kernel_launches.fetch_add(1, std::memory_order_relaxed);
    return 0;
}

constexpr size_t kPlanSmem = (7 * KVPAGE_MAX_CALL + kMaxUnits + 3 * KVPAGE_MAX_ROWS / 32) * sizeof(int32_t);

/* one cluster; the kernels' shared memory limit is raised once per device */
template <typename... P, typename... A>
int launch_plan(void (*kernel)(P...), std::once_flag *once, cudaError_t *err, int device, uint32_t threads, size_t smem,
                bool after, cudaStream_t stream, A... args)
{
    std::call_once(once[device], [&] {
        err[device] = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kPlanSmem);
        if (err[device] != cudaSuccess)
            cudaGetLastError();
    });
    if (err[device] != cudaSuccess)
        return -EIO;
    return launch(kernel, dim3(kPlanCluster), threads, kPlanCluster, smem, after, stream, args...);
}

/* Threads of the cluster's CTAs: barriers of 8 warps are cheap, and a small
 * call's units do not need more. */
uint32_t plan_threads(const kv_page_state *s, uint32_t n)
{
    const uint64_t units = (uint64_t)n * ((s->width + kUnit - 1) / kUnit);
    return units <= kPlanCluster * 8 ? 256 : kPlanThreads;
}

/* compacted: as the second kernel of compact */
int resize_launch(const kv_page_state *s, const int32_t *rows, const int32_t *lens, uint32_t n, int32_t *status,
                  bool compacted, cudaStream_t stream)
{
    static std::once_flag once[64];
    static cudaError_t err[64];
    const uint64_t units = n + (uint64_t)n * s->width / kUnit;
    const size_t smem = (7 * (size_t)n + (units < kMaxUnits ? units : kMaxUnits) + 2 * ((s->num_rows + 31) / 32)) * sizeof(int32_t);
    return launch_plan(kv_page_resize_kernel, once, err, s->device, plan_threads(s, n), smem, compacted, stream, *s, rows, lens, n, status,
                       compacted);
}

int call_ok(const kv_page_state *s, uint32_t n)
{
    if (!state_ok(s) || s->device < 0 || s->device >= 64)
        return -EINVAL;
    if (n > KVPAGE_MAX_CALL || s->num_rows > KVPAGE_MAX_ROWS || (uint64_t)n * s->width >= (1ull << 30))
        return -E2BIG;
    return 0;
}

template <int VEC>
int copy_vec(const Planes &p, const int32_t *src, const int32_t *dst, const int32_t *tokens, uint32_t pack, uint32_t n,
             bool after, cudaStream_t stream)
{
    Copy c{};
    c.src = src;
    c.dst = dst;
    c.tokens = tokens;
    c.pack = pack;
    c.n = n;
    const uint32_t run = p.bs * (p.unit / VEC), planes = p.layers * p.kvs;
    c.run = run;
    c.per_token = (p.head_bytes ? p.head_bytes : p.unit) / VEC;
    c.per_head = make_fastdiv(p.bs * c.per_token);
    if (run >= kMoveVectors) {
        c.pairs = make_fastdiv((run + kMoveVectors - 1) / kMoveVectors);
        if ((uint64_t)n * c.pairs.d > INT32_MAX || planes > 65535)
            return -E2BIG;
        return launch(kv_page_copy_run_kernel<VEC>, dim3(n * c.pairs.d, planes), kMoveThreads, 0, 0, after, stream, p, c);
    }
    c.pairs = make_fastdiv(n);
    c.planes_per_grid = INT32_MAX / n < planes ? INT32_MAX / n : planes;    /* 31-bit numbers of page and plane */
    const uint32_t grid_y = (planes + c.planes_per_grid - 1) / c.planes_per_grid;
    if (grid_y > 65535)
        return -E2BIG;
    const uint32_t grid_x = (n * c.planes_per_grid + kMoveThreads / 32 - 1) / (kMoveThreads / 32);
    return launch(kv_page_copy_warp_kernel<VEC>, dim3(grid_x, grid_y), kMoveThreads, 0, 0, after, stream, p, c);
}

int copy_launch(const kv_page_cache *c, const int32_t *src, const int32_t *dst, const int32_t *tokens, uint32_t pack,
                uint32_t n, bool after, cudaStream_t stream)
{
    const Planes p = planes_of(c);
    switch (vector_of(c)) {
    case 16: return copy_vec<16>(p, src, dst, tokens, pack, n, after, stream);
    case 8: return copy_vec<8>(p, src, dst, tokens, pack, n, after, stream);
    case 4: return copy_vec<4>(p, src, dst, tokens, pack, n, after, stream);
    case 2: return copy_vec<2>(p, src, dst, tokens, pack, n, after, stream);
    default: return copy_vec<1>(p, src, dst, tokens, pack, n, after, stream);
    }
}

template <int VEC>
int compact_vec(const Planes &p, const kv_page_state *s, const int32_t *rows, const int32_t *start, const int32_t *keep,
                const int32_t *offsets, uint32_t num_keep, uint32_t n, int32_t *scratch, cudaStream_t stream)
{
    /* a slice: the most vectors that divide a token's piece, at most 16 (256
     * bytes of a 16-byte vector), so that a pass of the CTA covers whole tokens
     * and long rows are cut finely */
    const uint32_t piece = (p.head_bytes ? p.head_bytes : p.unit) / VEC;
    uint32_t vecs = piece < 16 ? piece : 16;
    while (piece % vecs)
        vecs--;
    const uint64_t slices = (uint64_t)(p.unit / VEC / vecs) * p.layers * p.kvs;
    if (slices > INT32_MAX)
        return -E2BIG;
    /* A CTA reads and checks its row's list before it moves anything.  Where the
     * lists are short that is most of its time, and the CTAs that the GPU holds
     * at once (592) take many slices each, side by side; for many rows twice as
     * many, so that none has too many batches.  Keeping up to 5 of 24 tokens, with
     * the resizes: 64 rows 32.7 us with 592, 36.1 with 888, 35.6 with 1184; 256
     * rows 92, 86, 81.  Long lists want many CTAs, since rows differ in length. */
    const uint32_t all = num_keep / n >= kMoveVectors / 16 ? 8192 : n <= 148 ? 592 : 1184;
    const uint32_t row_ctas = all / n ? all / n : 1;
    const uint32_t per = (uint32_t)((slices + row_ctas - 1) / row_ctas);
    const uint32_t ctas = (uint32_t)((slices + per - 1) / per);
    return launch(kv_page_compact_kernel<VEC>, dim3(ctas, n), kMoveThreads, 0, 0, false, stream, p, *s, rows, start, keep, offsets,
                  num_keep, n, vecs, (uint32_t)slices, per, scratch);
}

}  // namespace

extern "C" int kv_page_device_of(const void *ptr)
{
    cudaPointerAttributes at{};
    if (cudaPointerGetAttributes(&at, ptr) != cudaSuccess) {
        cudaGetLastError();
        return -EINVAL;
    }
    return at.type == cudaMemoryTypeDevice ? at.device : at.type == cudaMemoryTypeUnregistered ? -EINVAL : KVPAGE_ANY_DEVICE;
}

extern "C" int kv_page_resize_launch(const struct kv_page_state *s, const int32_t *rows, const int32_t *lens, uint32_t n,
                                     int32_t *status, void *stream)
{
    const int bad = call_ok(s, n);
    if (bad)
        return bad;
    if (!n)
        return 0;
    if (!rows || !lens)
        return -EINVAL;
    DeviceGuard on(s->device);
    if (!on.ok)
        return -EIO;
    return resize_launch(s, rows, lens, n, status, false, static_cast<cudaStream_t>(stream));
}

extern "C" int kv_page_copy_launch(const struct kv_page_cache *c, const int32_t *src, const int32_t *dst,
                                   const int32_t *tokens, uint32_t n, void *stream)
{
    if (!cache_ok(c) || c->device < 0 || c->device >= 64)
        return -EINVAL;
    if (!n)
        return 0;
    if (!src || !dst)
        return -EINVAL;
    if (n > INT32_MAX)
        return -E2BIG;
    DeviceGuard on(c->device);
    if (!on.ok)
        return -EIO;
    return copy_launch(c, src, dst, tokens, 1, n, false, static_cast<cudaStream_t>(stream));
}

extern "C" int kv_page_fork_launch(const struct kv_page_cache *c, const struct kv_page_state *s, const int32_t *parents,
                                   const int32_t *children, uint32_t n, int32_t *pairs, int32_t *status, void *stream)
{
    const int bad = call_ok(s, n);
    if (bad)
        return bad;
    if (!cache_ok(c) || c->device != s->device || c->block_size != s->block_size || c->num_pages != s->num_pages)
        return -EINVAL;
    if (!n)
        return 0;
    if (!parents || !children || !pairs)
        return -EINVAL;
    DeviceGuard on(s->device);
    if (!on.ok)
        return -EIO;
    static std::once_flag once[64];
    static cudaError_t err[64];
    const size_t smem = (5 * (size_t)n + 3 * ((s->num_rows + 31) / 32)) * sizeof(int32_t);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int ret = launch_plan(kv_page_fork_kernel, once, err, s->device, plan_threads(s, n), smem, false, st, *s, parents,
                                children, n, pairs, status);
    if (ret)
        return ret;
    return copy_launch(c, pairs, pairs + 1, pairs + 2, 3, n, true, st);
}

extern "C" int kv_page_compact_launch(const struct kv_page_cache *c, const struct kv_page_state *s, const int32_t *rows,
                                      const int32_t *start, const int32_t *keep, const int32_t *offsets,
                                      uint32_t num_keep, uint32_t n, int32_t *scratch, int32_t *status, void *stream)
{
    const int bad = call_ok(s, n);
    if (bad)
        return bad;
    if (!cache_ok(c) || c->device != s->device || c->block_size != s->block_size || c->num_pages != s->num_pages)
        return -EINVAL;
    if (!n)
        return 0;
    if (!rows || !start || !offsets || !scratch || (num_keep && !keep) || num_keep > INT32_MAX)
        return -EINVAL;
    DeviceGuard on(s->device);
    if (!on.ok)
        return -EIO;
    const Planes p = planes_of(c);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    int ret;
    switch (vector_of(c)) {
    case 16: ret = compact_vec<16>(p, s, rows, start, keep, offsets, num_keep, n, scratch, st); break;
    case 8: ret = compact_vec<8>(p, s, rows, start, keep, offsets, num_keep, n, scratch, st); break;
    case 4: ret = compact_vec<4>(p, s, rows, start, keep, offsets, num_keep, n, scratch, st); break;
    case 2: ret = compact_vec<2>(p, s, rows, start, keep, offsets, num_keep, n, scratch, st); break;
    default: ret = compact_vec<1>(p, s, rows, start, keep, offsets, num_keep, n, scratch, st); break;
    }
    return ret ? ret : resize_launch(s, rows, scratch, n, status, true, st);
}
