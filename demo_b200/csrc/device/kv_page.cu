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
 * bytes of traffic per byte moved, and keep eight 16-byte vectors per thread
 * in flight.
 */
#include "kvpage.h"
#include "adaptor.h"
#include "device_guard.h"

#include <cuda_runtime.h>

#include <cerrno>
#include <cstdint>
#include <mutex>

namespace {

constexpr int kPlanThreads = 1024;
constexpr int kPlanWarps = kPlanThreads / 32;
constexpr uint32_t kPlanCluster = 8;
constexpr int32_t kRefused = INT32_MIN;     /* compact's length for resize of a row that it has refused and reported */

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

__device__ __forceinline__ void cluster_sync()
{
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

/* store v at `p`'s place in the shared memory of CTA `rank` of the cluster */
__device__ __forceinline__ void store_cluster(int32_t *p, uint32_t rank, int32_t v)
{
    uint32_t a = (uint32_t)__cvta_generic_to_shared(p), b;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(b) : "r"(a), "r"(rank));
    asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(b), "r"(v) : "memory");
}

/* exclusive prefix sum of a[0 .. n) in place, n <= KVPAGE_MAX_CALL; returns
 * the total to every thread.  Each thread sums 4 consecutive values. */
__device__ int32_t block_scan(int32_t *a, uint32_t n)
{
    __shared__ int32_t warp_sum[kPlanWarps];
    static_assert(KVPAGE_MAX_CALL == 4 * kPlanThreads, "four values per thread");
    const uint32_t i0 = threadIdx.x * 4, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int32_t v[4], sum = 0;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 4; k++) {
        v[k] = i0 + k < n ? a[i0 + k] : 0;
        sum += v[k];
    }
    int32_t inc = sum;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        int32_t o = __shfl_up_sync(~0u, inc, d);
        if (lane >= d)
            inc += o;
    }
    if (lane == 31)
        warp_sum[warp] = inc;
    __syncthreads();
    if (warp == 0) {
        int32_t w = warp_sum[lane];
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            int32_t o = __shfl_up_sync(~0u, w, d);
            if (lane >= d)
                w += o;
        }
        warp_sum[lane] = w;
    }
    __syncthreads();
    int32_t run = inc - sum + (warp ? warp_sum[warp - 1] : 0);
    const int32_t total = warp_sum[kPlanWarps - 1];
#pragma unroll
    for (int k = 0; k < 4; k++) {
        if (i0 + k < n)
            a[i0 + k] = run;
        run += v[k];
    }
    __syncthreads();
    return total;
}

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

/* ------------------------------------------------------------------------
 * resize.  Entry k of the call's row i has the number i * width + k, and a
 * dropped page's place in the push order is its highest number:
 *   A  every dropped entry takes one reference off its page and raises the
 *      page's mark to its number + 1 (both commute: any order, same result)
 *   B  the entry whose number the mark holds, of a page without references,
 *      stands for the page; warps count these row by row, the counts go to
 *      every CTA's shared memory, and each CTA scans them
 *   C  those entries push their pages
 *   D  growing rows pop, marks go back to zero, lengths and counts are written
 * with a cluster barrier between phases.  A warp owns a row.  A reference is
 * taken back where a page had none left, so a page freed twice is neither
 * pushed twice nor left negative.
 * ---------------------------------------------------------------------- */
__global__ void __launch_bounds__(kPlanThreads, 1)
kv_page_resize_kernel(const kv_page_state s, const int32_t *__restrict__ rows, const int32_t *__restrict__ lens,
                      uint32_t n, int32_t *__restrict__ status)
{
    extern __shared__ int32_t sm[];
    int32_t *row = sm, *old_p = sm + n, *new_p = sm + 2 * n, *need = sm + 3 * n, *gone = sm + 4 * n;
    const uint32_t words = (s.num_rows + 31) / 32;
    uint32_t *seen = reinterpret_cast<uint32_t *>(sm + 5 * n), *twice = seen + words;
    __shared__ int32_t served;
    const uint32_t rank = cluster_rank(), ctas = cluster_size();
    const uint32_t lane = threadIdx.x & 31, warp0 = rank * kPlanWarps + (threadIdx.x >> 5), warps = ctas * kPlanWarps;

    for (uint32_t i = threadIdx.x; i < 2 * words; i += kPlanThreads)
        seen[i] = 0;
    if (threadIdx.x == 0)
        served = 0;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < n; i += kPlanThreads) {
        const int32_t r = rows[i];
        row[i] = r;
        if (r >= 0 && (uint32_t)r < s.num_rows && test_and_set(seen, r))
            test_and_set(twice, r);
    }
    __syncthreads();
    bool drop = false;
    for (uint32_t i = threadIdx.x; i < n; i += kPlanThreads) {
        const int32_t r = row[i], to = lens[i];
        bool ok = r >= 0 && (uint32_t)r < s.num_rows && !test_bit(twice, r) && to >= 0;
        uint32_t a = 0, b = 0;
        if (ok) {
            const int32_t from = s.lens[r];
            a = pages_of(max(from, 0), s.block_size);
            b = pages_of(to, s.block_size);
            ok = from >= 0 && a <= s.width && b <= s.width;
        }
        if (!ok) {
            if (rank == 0 && to != kRefused)
                atomicOr(s.error, KVPAGE_ERR_ROW);
            row[i] = -1;
            a = b = 0;
        }
        old_p[i] = a;
        new_p[i] = b;
        need[i] = b > a ? b - a : 0;
        gone[i] = 0;
        drop |= b < a;
    }
    const int32_t count = free_pages(s);
    drop = __syncthreads_or(drop);
    int32_t pushed = 0;
    if (drop) {
        for (uint32_t i = warp0; i < n; i += warps) {
            const int32_t *t = s.table + (int64_t)max(row[i], 0) * s.table_stride;
            for (int32_t k = new_p[i] + (int32_t)lane; k < old_p[i]; k += 32) {
                const int32_t p = t[k];
                if (p < 0 || (uint32_t)p >= s.num_pages) {
                    atomicOr(s.error, KVPAGE_ERR_PAGE);
                    continue;
                }
                if (atomicSub(&s.refs[p], 1) >= 1) {
                    atomicMax(&s.marks[p], (int32_t)(i * s.width) + k + 1);
                } else {
                    atomicAdd(&s.refs[p], 1);
                    atomicOr(s.error, KVPAGE_ERR_REFS);
                }
            }
        }
        cluster_sync();
        auto stands = [&](uint32_t i, int32_t k, const int32_t *t, int32_t &p) {
            if (k >= old_p[i])
                return false;
            p = t[k];
            return p >= 0 && (uint32_t)p < s.num_pages && __ldcg(&s.marks[p]) == (int32_t)(i * s.width) + k + 1 &&
                   __ldcg(&s.refs[p]) == 0;
        };
        for (uint32_t i = warp0; i < n; i += warps) {
            if (new_p[i] >= old_p[i])
                continue;
            const int32_t *t = s.table + (int64_t)row[i] * s.table_stride;
            int32_t c = 0, p;
            for (int32_t k = new_p[i] + (int32_t)lane; k - (int32_t)lane < old_p[i]; k += 32)
                c += stands(i, k, t, p);
            c = __reduce_add_sync(~0u, c);
            if (lane < ctas)
                store_cluster(&gone[i], lane, c);
        }
        cluster_sync();
        pushed = block_scan(gone, n);
        for (uint32_t i = warp0; i < n; i += warps) {
            if (new_p[i] >= old_p[i])
                continue;
            const int32_t *t = s.table + (int64_t)row[i] * s.table_stride;
            int32_t at = count + gone[i];
            for (int32_t k = new_p[i] + (int32_t)lane; k - (int32_t)lane < old_p[i]; k += 32) {
                int32_t p = 0;
                const bool mine = stands(i, k, t, p);
                const uint32_t m = __ballot_sync(~0u, mine);
                const int32_t place = at + __popc(m & ((1u << lane) - 1));
                if (mine && (uint32_t)place < s.num_pages)
                    s.free_list[place] = p;
                at += __popc(m);
            }
        }
    }
    const int32_t have = min(count + pushed, (int32_t)s.num_pages);
    block_scan(need, n);
    cluster_sync();
    for (uint32_t i = threadIdx.x; i < n; i += kPlanThreads) {
        const int32_t want = new_p[i] - old_p[i];
        if (want > 0 && need[i] + want <= have)
            atomicMax(&served, need[i] + want);
    }
    for (uint32_t i = warp0; i < n; i += warps) {
        const int32_t r = row[i];
        if (r < 0) {
            if (lane == 0 && status)
                status[i] = KVPAGE_INVALID;
            continue;
        }
        int32_t *t = s.table + (int64_t)r * s.table_stride;
        const int32_t want = new_p[i] - old_p[i];
        const bool fits = want <= 0 || need[i] + want <= have;
        for (int32_t k = new_p[i] + (int32_t)lane; k < old_p[i]; k += 32) {
            const int32_t p = t[k];
            if (p >= 0 && (uint32_t)p < s.num_pages)
                s.marks[p] = 0;
        }
        if (fits)
            for (int32_t k = lane; k < want; k += 32) {
                const int32_t p = __ldcg(&s.free_list[have - 1 - need[i] - k]);
                t[old_p[i] + k] = p;
                if (p >= 0 && (uint32_t)p < s.num_pages)
                    s.refs[p] = 1;
                else
                    atomicOr(s.error, KVPAGE_ERR_PAGE);
            }
        if (lane == 0) {
            if (fits)
                s.lens[r] = lens[i];
            if (status)
                status[i] = fits ? KVPAGE_OK : KVPAGE_NO_PAGES;
        }
    }
    __syncthreads();
    if (rank == 0 && threadIdx.x == 0)
        *s.free_count = have - served;
}

/* ------------------------------------------------------------------------
 * fork's plan: what each child gets, the tables and the references; the pages
 * to copy go to pairs[3 * i] = (source, destination, tokens), source -1 where
 * there is nothing to copy.  One cluster, a warp per child.
 * ---------------------------------------------------------------------- */
__global__ void __launch_bounds__(kPlanThreads, 1)
kv_page_fork_kernel(const kv_page_state s, const int32_t *__restrict__ parents, const int32_t *__restrict__ children,
                    uint32_t n, int32_t *__restrict__ pairs, int32_t *__restrict__ status)
{
    extern __shared__ int32_t sm[];
    int32_t *from = sm, *child = sm + n, *length = sm + 2 * n, *need = sm + 3 * n;
    const uint32_t words = (s.num_rows + 31) / 32;
    uint32_t *seen = reinterpret_cast<uint32_t *>(sm + 4 * n), *twice = seen + words, *parent = seen + 2 * words;
    __shared__ int32_t served;
    const uint32_t rank = cluster_rank(), ctas = cluster_size();
    const uint32_t lane = threadIdx.x & 31, warp0 = rank * kPlanWarps + (threadIdx.x >> 5), warps = ctas * kPlanWarps;

    for (uint32_t i = threadIdx.x; i < 3 * words; i += kPlanThreads)
        seen[i] = 0;
    if (threadIdx.x == 0)
        served = 0;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < n; i += kPlanThreads) {
        const int32_t p = parents[i], c = children[i];
        from[i] = p;
        child[i] = c;
        if (p >= 0 && (uint32_t)p < s.num_rows)
            test_and_set(parent, p);
        if (c >= 0 && (uint32_t)c < s.num_rows && test_and_set(seen, c))
            test_and_set(twice, c);
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < n; i += kPlanThreads) {
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
        need[i] = len % (int32_t)s.block_size != 0;
    }
    const int32_t have = free_pages(s);
    block_scan(need, n);
    cluster_sync();                 /* every CTA has read the lengths and the count */
    for (uint32_t i = threadIdx.x; i < n; i += kPlanThreads)
        if (length[i] % (int32_t)s.block_size && need[i] < have)
            atomicMax(&served, need[i] + 1);
    for (uint32_t i = warp0; i < n; i += warps) {
        const int32_t c = child[i], len = length[i];
        const int32_t full = len / (int32_t)s.block_size, tail = len % (int32_t)s.block_size;
        const bool fits = c >= 0 && (!tail || need[i] < have);
        int32_t src = -1, dst = -1;
        if (fits) {
            const int32_t *tp = s.table + (int64_t)from[i] * s.table_stride;
            int32_t *tc = s.table + (int64_t)c * s.table_stride;
            for (int32_t k = lane; k < full; k += 32) {
                const int32_t p = tp[k];
                tc[k] = p;
                if (p >= 0 && (uint32_t)p < s.num_pages)
                    atomicAdd(&s.refs[p], 1);
                else
                    atomicOr(s.error, KVPAGE_ERR_PAGE);
            }
            if (tail && lane == 0) {
                src = tp[full];
                dst = s.free_list[have - 1 - need[i]];
                tc[full] = dst;
                if (dst >= 0 && (uint32_t)dst < s.num_pages)
                    s.refs[dst] = 1;        /* a bad id of either: the copy sets the error bit */
            }
        }
        if (lane == 0) {
            pairs[3 * i] = fits && tail ? src : 0;
            pairs[3 * i + 1] = fits && tail ? dst : 0;
            pairs[3 * i + 2] = fits ? tail : 0;
            if (fits)
                s.lens[c] = len;
            if (status)
                status[i] = fits ? KVPAGE_OK : c < 0 ? KVPAGE_INVALID : KVPAGE_NO_PAGES;
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
        c->num_pages > INT32_MAX || (c->base_align & (c->base_align - 1)))
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

template <int VEC>
__device__ __forceinline__ uint8_t *plane(const Planes &p, uint32_t lk)
{
    const uint32_t l = p.kvs == 2 ? lk >> 1 : lk;
    uint8_t *base = reinterpret_cast<uint8_t *>((p.kvs == 2 && (lk & 1) ? p.layer_v : p.layer_k)[l]);
    if (!base || reinterpret_cast<uintptr_t>(base) % VEC) {
        atomicOr(p.error, KVPAGE_ERR_ALIGN);
        return nullptr;
    }
    return base;
}

/* ------------------------------------------------------------------------
 * copy.  A CTA moves up to kCopyVectors vectors of one page in one plane: a
 * page is one run of bytes in every geometry, so consecutive threads move
 * consecutive vectors.  With a token count, token-major pages stop early and
 * head-major ones skip the tokens behind it.  `pack` is the
 * distance between the entries of the lists: 1, or 3 for fork's pairs.
 * ---------------------------------------------------------------------- */
constexpr int kMoveThreads = 256;
constexpr int kMoveUnroll = 8;
constexpr uint32_t kMoveVectors = kMoveThreads * kMoveUnroll;

template <int VEC>
__global__ void __launch_bounds__(kMoveThreads)
kv_page_copy_kernel(const Planes p, const int32_t *__restrict__ src, const int32_t *__restrict__ dst,
                    const int32_t *__restrict__ tokens, uint32_t pack, uint32_t n, uint32_t chunks)
{
    using T = typename VecOf<VEC>::T;
    const uint32_t lk = blockIdx.y;
    const uint32_t i = blockIdx.x / chunks, chunk = blockIdx.x - i * chunks;
    const int32_t a = src[(uint64_t)i * pack], b = dst[(uint64_t)i * pack];
    int32_t keep = (int32_t)p.bs;
    if (tokens)
        keep = min(max(tokens[(uint64_t)i * pack], 0), keep);
    if (!keep || a == b)
        return;
    if (a < 0 || (uint32_t)a >= p.pages || b < 0 || (uint32_t)b >= p.pages) {
        if (threadIdx.x == 0)
            atomicOr(p.error, KVPAGE_ERR_PAGE);
        return;
    }
    uint8_t *base = plane<VEC>(p, lk);
    if (!base)
        return;
    const T *from = reinterpret_cast<const T *>(base + (uint64_t)a * p.stride);
    T *to = reinterpret_cast<T *>(base + (uint64_t)b * p.stride);
    const bool part = p.head_bytes && keep < (int32_t)p.bs;
    const uint32_t all = (p.head_bytes ? p.bs : (uint32_t)keep) * (p.unit / VEC);
    const uint32_t per_token = p.head_bytes / VEC, per_head = per_token * p.bs, used = per_token * keep;
    T v[kMoveUnroll];
    bool on[kMoveUnroll];
#pragma unroll
    for (int u = 0; u < kMoveUnroll; u++) {
        const uint32_t x = chunk * kMoveVectors + u * kMoveThreads + threadIdx.x;
        on[u] = x < all && !(part && x % per_head >= used);
        if (on[u])
            v[u] = from[x];
    }
#pragma unroll
    for (int u = 0; u < kMoveUnroll; u++)
        if (on[u])
            to[chunk * kMoveVectors + u * kMoveThreads + threadIdx.x] = v[u];
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
 * Every CTA checks its row's whole list before it moves a byte, so that all
 * of them decide alike; 4 bytes of list against 64 bytes or more of slice.
 * The first CTA of a row leaves the new length for resize, or kRefused.
 * ---------------------------------------------------------------------- */
template <int VEC>
__global__ void __launch_bounds__(kMoveThreads)
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
    if (threadIdx.x == 0) {
        s_first = INT32_MAX;
        s_bad = 0;
    }
    __syncthreads();
    for (uint32_t k = threadIdx.x; k < n; k += kMoveThreads)
        if (k != i && rows[k] == r)
            bad = KVPAGE_ERR_ROW;
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
                    uint8_t *base = plane<VEC>(p, lk);
                    const uint32_t o = (sl * slice_vecs + vec) * VEC;
                    /* byte o of a token's unit: a head-major page holds head o / head_bytes apart */
                    const uint64_t at = p.head_bytes ? (uint64_t)(o / p.head_bytes) * p.bs * p.head_bytes + o % p.head_bytes : o;
                    if (base) {
                        v[u] = *reinterpret_cast<const T *>(base + src_off[j] + at);
                        to[u] = reinterpret_cast<T *>(base + dst_off[j] + at);
                    }
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
int launched()
{
    g_cc_kernel_launches.fetch_add(1, std::memory_order_relaxed);
    return cudaPeekAtLastError() == cudaSuccess ? 0 : -EIO;
}

constexpr size_t kPlanSmem = (5 * KVPAGE_MAX_CALL + 3 * KVPAGE_MAX_ROWS / 32) * sizeof(int32_t);

/* one cluster of `ctas` CTAs; the kernels' shared memory limit is raised once per device */
template <typename... P, typename... A>
int launch_plan(void (*kernel)(P...), std::once_flag *once, cudaError_t *err, int device, uint32_t ctas, size_t smem,
                cudaStream_t stream, A... args)
{
    std::call_once(once[device], [&] {
        err[device] = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kPlanSmem);
    });
    if (err[device] != cudaSuccess)
        return -EIO;
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr[1];
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(kPlanThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ctas;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, kernel, args...) != cudaSuccess) {
        cudaGetLastError();
        return -EIO;
    }
    return launched();
}

/* a warp per row: one CTA has enough of them for a small call, whose time is
 * the barriers' and the loads'; larger calls use the cluster */
uint32_t plan_ctas(uint32_t n)
{
    return n <= kPlanWarps ? 1 : kPlanCluster;
}

int resize_launch(const kv_page_state *s, const int32_t *rows, const int32_t *lens, uint32_t n, int32_t *status,
                  cudaStream_t stream)
{
    static std::once_flag once[64];
    static cudaError_t err[64];
    const size_t smem = (5 * (size_t)n + 2 * ((s->num_rows + 31) / 32)) * sizeof(int32_t);
    return launch_plan(kv_page_resize_kernel, once, err, s->device, plan_ctas(n), smem, stream, *s, rows, lens, n, status);
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
             cudaStream_t stream)
{
    const uint32_t all = p.bs * (p.unit / VEC), chunks = (all + kMoveVectors - 1) / kMoveVectors;
    if ((uint64_t)n * chunks > INT32_MAX || p.layers * p.kvs > 65535)
        return -E2BIG;
    kv_page_copy_kernel<VEC><<<dim3(n * chunks, p.layers * p.kvs), kMoveThreads, 0, stream>>>(p, src, dst, tokens, pack,
                                                                                          n, chunks);
    return launched();
}

int copy_launch(const kv_page_cache *c, const int32_t *src, const int32_t *dst, const int32_t *tokens, uint32_t pack,
                uint32_t n, cudaStream_t stream)
{
    const Planes p = planes_of(c);
    switch (vector_of(c)) {
    case 16: return copy_vec<16>(p, src, dst, tokens, pack, n, stream);
    case 8: return copy_vec<8>(p, src, dst, tokens, pack, n, stream);
    case 4: return copy_vec<4>(p, src, dst, tokens, pack, n, stream);
    case 2: return copy_vec<2>(p, src, dst, tokens, pack, n, stream);
    default: return copy_vec<1>(p, src, dst, tokens, pack, n, stream);
    }
}

template <int VEC>
int compact_vec(const Planes &p, const kv_page_state *s, const int32_t *rows, const int32_t *start, const int32_t *keep,
                const int32_t *offsets, uint32_t num_keep, uint32_t n, int32_t *scratch, cudaStream_t stream)
{
    /* a slice: the most vectors that divide a token's piece, at most 32 (512
     * bytes of a 16-byte vector), so that a pass of the CTA covers whole tokens */
    const uint32_t piece = (p.head_bytes ? p.head_bytes : p.unit) / VEC;
    uint32_t vecs = piece < 32 ? piece : 32;
    while (piece % vecs)
        vecs--;
    const uint64_t slices = (uint64_t)(p.unit / VEC / vecs) * p.layers * p.kvs;
    if (slices > INT32_MAX)
        return -E2BIG;
    /* enough CTAs to fill the GPU a few times over, no more: each reads its row's list */
    uint32_t per = (uint32_t)((slices * n + 4095) / 4096);
    if (per > slices)
        per = (uint32_t)slices;
    const uint32_t ctas = (uint32_t)((slices + per - 1) / per);
    kv_page_compact_kernel<VEC><<<dim3(ctas, n), kMoveThreads, 0, stream>>>(p, *s, rows, start, keep, offsets, num_keep, n,
                                                                        vecs, (uint32_t)slices, per, scratch);
    return launched();
}

}  // namespace

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
    return resize_launch(s, rows, lens, n, status, static_cast<cudaStream_t>(stream));
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
    DeviceGuard on(c->device);
    if (!on.ok)
        return -EIO;
    return copy_launch(c, src, dst, tokens, 1, n, static_cast<cudaStream_t>(stream));
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
    const size_t smem = (4 * (size_t)n + 3 * ((s->num_rows + 31) / 32)) * sizeof(int32_t);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int ret = launch_plan(kv_page_fork_kernel, once, err, s->device, plan_ctas(n), smem, st, *s, parents, children, n,
                                pairs, status);
    if (ret)
        return ret;
    return copy_launch(c, pairs, pairs + 1, pairs + 2, 3, n, st);
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
    return ret ? ret : resize_launch(s, rows, scratch, n, status, st);
}
