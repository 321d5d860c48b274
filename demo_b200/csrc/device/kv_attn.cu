/*
 * Attention over a paged KV cache for drafted trees, chains and single tokens
 * (include/kvattn.h), sm_100a.
 *
 * A K/V head of a sequence serves nodes x (query heads per K/V head) query
 * rows, in tiles of whole nodes, at most 128 rows.  Per 64 positions of the
 * context a CTA computes
 *
 *   S = Q K^T        128 x 64, tcgen05.mma, Q and K in shared memory, S in TMEM
 *   P = exp2(S - m)  one thread per row, the running maximum and sum in 32 bits
 *   O += P V         128 x dim, tcgen05.mma, P in TMEM (where S was), V in shared
 *
 * Bound: with up to about 200 rows, reading K and V once from HBM: a tile of 64
 * positions is 32 KiB at 16 bits and dim 128, about 1400 cycles of an SM's
 * share of the bandwidth, while its products take some 640 cycles of the tensor
 * cores even if only one of the 128 rows is a query, and its exponentials at
 * most 512.  So one form serves single tokens and trees alike.  What is left to
 * hide is latency, from the load to the product, the softmax and the next
 * product: two CTAs share an SM, and in each S is held twice, so that S of the
 * next tile is computed under the softmax of this one.
 *
 * On a B200, 32 heads over 8 K/V heads of dim 128: one token over 2048 positions
 * takes 15.5 us (launch, line, one tile, join: latencies); a batch of 64 trees of
 * 9 to 32 nodes over 500 to 2048 positions with 344 MB of K and V 86 us (4.0 TB/s);
 * one of 32 chains of 4 nodes over 4000 to 8192 positions of e4m3 with 394 MB
 * 149 us (2.6 TB/s: the widening); 8 heads over one: a batch of 8 trees of 64
 * nodes over 32768 to 131072 positions with 173 GFLOP 210 us (0.82 PFLOP/s: the
 * chain of products and exponentials).
 *
 * Warps 0-3 are the softmax (a thread owns a TMEM lane, a row), then come the
 * loaders, a warp that issues the products, and one that finds the next pieces
 * of work for all of them.  They meet at mbarriers: pieces, a ring of tiles of
 * K and one of V, S and P, and O.  Every wait is bounded.
 *
 * The (sequence, K/V head, row tile, position tile) quadruples of a call lie on
 * one line, and each CTA takes an equal part of it, wherever that ends inside a
 * context: ragged batches and a single long row fill the GPU alike, and the
 * lengths are read on the device.  A CTA takes a piece's tiles in an order in
 * which all CTAs are at the same place of a share: row tiles of one sequence
 * then read each position together.  Pieces of a row tile are joined by a second
 * kernel, in a fixed order, so results do not depend on timing.
 */
#include "kvattn.h"
#include "adaptor.h"
#include "device_guard.h"
#include "fastdiv.h"

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <cerrno>
#include <cmath>
#include <cstdint>
#include <mutex>

namespace {

constexpr int kRows = 128;          /* query rows of a tile: TMEM lanes */
constexpr int kTile = 64;           /* positions of a tile */
constexpr int kColumn = 64;         /* Q, K and V stand in columns of 64 values: 128 bytes, the swizzle's width */
constexpr int kColumnBytes = kTile * kColumn * 2;   /* of K and V */
constexpr int kSoftmax = 128;       /* threads of the softmax */

/* how K and V come: by TMA (16-bit caches whose pages divide into boxes of 8 or
 * more rows), by 16-byte copies (16-bit caches of any other page size), or by
 * 16-byte copies that are widened (8-bit caches) */
enum Load { kTma, kCopy, kWiden };
template <Load L> struct Roles {
    static constexpr int kLoaders = L == kTma ? 64 : L == kCopy ? 128 : 256;  /* but for kCopy a half for K and one for V */
    static constexpr int kFill = L == kTma ? 1 : 128;               /* threads that arrive for a tile */
    static constexpr int kThreads = kSoftmax + kLoaders + 64;       /* a warp for the products, one that plans */
};
/* Beginning and ending a row tile (Q, the first S, O out) takes as long as about
 * 3 tiles, and counts as much: 64 sequences of up to 2048 positions, 9 to 32
 * nodes, take 83.5 us with 3, 90.3 with 0, 85.2 with 2, 82.8 with 4; 8 of up to
 * 131072 188.3, 190.8, 188.9 and 188.7. */
constexpr int kPieceCost = 3;
constexpr int kPlanned = 4;         /* pieces that the planning warp is ahead */
constexpr int kJoinThreads = 256;
constexpr int kMaxCtas = 512;       /* of the first kernel */
/* polls of a wait, at 4 us each (the hardware waits before it answers): about a
 * second; of one that a test lets run out */
constexpr uint32_t kSpinLimit = 1u << 18, kStallLimit = 1u << 12;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

/* DP: head_dim rounded up to whole columns.  K of the next tile is used a
 * softmax earlier than V of this one: where there is room its ring is longer. */
template <Load L, int DP> struct Shape {
    static constexpr int kCtas = DP <= 128 ? 2 : 1;                 /* per SM */
    static constexpr int kRaw = L == kWiden ? 4 : 0;                /* 8-bit tiles on their way */
    static constexpr int kSlotsK = DP == 64 ? 5 : kRaw ? 1 : 3;     /* kRaw, 2 for K and 1 for V: 143 us, this 140.6 (as at run_widen) */
    static constexpr int kSlotsV = DP == 64 ? 4 : 2;
    static constexpr int kSlotBytes = DP / kColumn * kColumnBytes;
    static constexpr int kQBytes = kRows * DP * 2;
    static constexpr int kTmem = DP <= 128 ? 256 : 512;             /* columns: 2 x 64 of S, then O */
    static constexpr int kShared = kQBytes + (kSlotsK + kSlotsV) * kSlotBytes + kRaw * kSlotBytes / 2;  /* of struct Shared */
    static constexpr int kSmem = kShared + 1024;
    static_assert(kCtas * (kSmem + 1024) <= 228 * 1024, "the CTAs of an SM share its shared memory");
    static_assert(2 * kTile + DP <= kTmem && kCtas * kTmem <= 512, "and its TMEM");
};

/* a row tile that lies across CTAs: its first piece is the last of CTA c (in
 * that CTA's place `slot`), the others are the first of CTAs c + 1 .. */
struct Job {
    int32_t rows, ctas, slot, q0, h;
};

struct Params {
    CUtensorMap q_map;      /* [queries][heads][dim], boxes of 64 values x the rows of a tile */
    CUtensorMap k_map, v_map;   /* kTma: [pages][kv heads][block][dim], boxes of 64 values x `box` rows */
    kv_attn_desc d;
    uint64_t stride;        /* bytes from page to page */
    FastDiv block;          /* positions of a page */
    FastDiv nodes;          /* nodes of a row tile */
    uint32_t group;         /* query heads per K/V head */
    uint32_t columns;       /* of Q, K and V */
    uint32_t box;
    uint32_t min_share;     /* tiles that a CTA takes at least */
    uint32_t wide_out;      /* rows of out start on 32 bytes */
    uint32_t stall;         /* kv_attn_launch_stalled */
    Job *jobs;              /* workspace: [CTAs] row tiles to be joined, by the CTA that has their first tiles */
    float *part_ml;         /* [2 * CTAs][128][2] maximum and sum of a piece */
    float *part_o;          /* [2 * CTAs][128][dim] */
};

/* ---- sequences and tiles ---- */
struct Seq {
    int32_t q0, nodes, ctx, row;
};

/* sequence b; false if it does not fit: nodes is then 0 where its offsets
 * are wrong, else its rows are to be voided */
__device__ bool sequence(const kv_attn_desc &d, uint32_t b, Seq &s)
{
    const int32_t o0 = d.q_offsets[b], o1 = d.q_offsets[b + 1];
    const int32_t r = d.rows ? d.rows[b] : (int32_t)b;
    s = {o0, 0, 0, 0};
    if (o0 < 0 || o1 < o0 || (uint32_t)o1 > d.total_q)
        return false;
    if (o1 == o0)
        return true;                /* nothing to do, whatever its row */
    s.nodes = o1 - o0;
    if (r < 0 || (uint32_t)r >= d.num_rows)
        return false;
    const int32_t len = d.lens[r];
    s.ctx = len - s.nodes;
    s.row = r;
    return len >= 0 && s.ctx >= 0 && (uint64_t)len <= (uint64_t)d.width * d.block_size;
}

/* a node that sees something */
__device__ __forceinline__ bool node_ok(const int32_t *parents, int32_t j)
{
    const int32_t u = parents[j];
    return u >= -1 && u < j;
}

/* positions that row tile rt's nodes may see: parents come before their nodes */
__device__ __forceinline__ int32_t visible_end(const Params &p, const Seq &s, int32_t rt)
{
    return s.ctx + min(s.nodes, (rt + 1) * (int32_t)p.nodes.d);
}

__device__ __forceinline__ uint32_t tiles_of(const Params &p, const Seq &s, int32_t rt)
{
    return ((uint32_t)visible_end(p, s, rt) + kTile - 1) / kTile;
}

/* what row tile rt is long on the line */
__device__ __forceinline__ uint32_t cost_of(const Params &p, const Seq &s, int32_t rt)
{
    return kPieceCost + tiles_of(p, s, rt);
}

/* one K/V head of the sequence, all row tiles */
__device__ __forceinline__ uint64_t head_cost(const Params &p, const Seq &s)
{
    uint64_t n = 0;
    for (int32_t rt = 0; rt * (int32_t)p.nodes.d < s.nodes; rt++)
        n += cost_of(p, s, rt);
    return n;
}

/* a run of tiles of one row tile */
struct Piece {
    int32_t q0, nodes, ctx, row;    /* the sequence's */
    int32_t h, node0, end;          /* K/V head, first node, positions that the nodes may see */
    int32_t t0, t1, n;              /* tiles t0 .. t1 of n */
    int32_t top;                    /* which come in this order: top .. t0, t1 - 1 .. top + 1 */
    __device__ __forceinline__ int32_t behind(int32_t t) const { return t == t0 ? t1 - 1 : t - 1; }
    __device__ bool whole() const { return t0 == 0 && t1 == n; }
    __device__ int32_t rows(const Params &p) const { return min(nodes - node0, (int32_t)p.nodes.d) * (int32_t)p.group; }
};

struct Line {
    int64_t x, hi, base;
    uint64_t per_head;
    uint32_t b;
    Seq s;                          /* sequence b, the length of one of its K/V heads, and what lies before it */

    /* The order of a piece's tiles: at any time the CTAs are at tiles that leave
     * the same remainder by their share, so that the row tiles of a sequence
     * read a position while it is in L2.  8 contexts of up to 131072 positions
     * with 4 row tiles each, 0.34 GB: 0.37 GB come from HBM, 1.28 GB if every
     * piece is taken from one end to the other. */
    __device__ bool next(const Params &p, int64_t share, Piece &e)
    {
        do {
            if (x >= hi)
                return false;
            while (x >= base + (int64_t)(per_head * p.d.num_kv_heads)) {
                base += (int64_t)(per_head * p.d.num_kv_heads);
                b++;
                per_head = sequence(p.d, b, s) ? head_cost(p, s) : 0;
            }
            uint64_t y = x - base;
            e.h = (int32_t)((y | per_head) >> 32 ? y / per_head : (uint32_t)y / (uint32_t)per_head);
            y -= e.h * per_head;
            int32_t rt = 0;
            uint32_t n;
            for (n = cost_of(p, s, 0); y >= n; n = cost_of(p, s, rt)) {
                y -= n;
                rt++;
            }
            e.q0 = s.q0;
            e.nodes = s.nodes;
            e.ctx = s.ctx;
            e.row = s.row;
            e.node0 = rt * (int32_t)p.nodes.d;
            e.end = visible_end(p, s, rt);
            e.n = (int32_t)n - kPieceCost;
            const int64_t upto = min((int64_t)n, (int64_t)y + (hi - x));
            e.t0 = (int32_t)max((int64_t)0, (int64_t)y - kPieceCost);
            e.t1 = (int32_t)max((int64_t)0, upto - kPieceCost);
            x += upto - (int64_t)y;
        } while (e.t1 == e.t0);
        const uint32_t past = share >> 31 ? 0 : (uint32_t)e.t1 % (uint32_t)share;
        e.top = e.t1 - 1 - (int32_t)past;
        if (e.top < e.t0)
            e.top = e.t1 - 1;
        return true;
    }
};

/* ---- mbarriers, TMEM and products ---- */
__device__ __forceinline__ uint32_t smem_u32(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void mbar_init(uint64_t *bar, uint32_t count)
{
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count) : "memory");
}

__device__ __forceinline__ void mbar_arrive(uint64_t *bar)
{
    asm volatile("mbarrier.arrive.release.cta.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

__device__ __forceinline__ bool mbar_try_wait(uint32_t bar, uint32_t parity)
{
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\t"
                 "mbarrier.try_wait.parity.acquire.cta.shared::cta.b64 p, [%1], %2;\n\t"
                 "selp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}

struct Shared {
    uint64_t k_full[5], k_empty[5], v_full[4], v_empty[4];
    uint64_t s_full[2], p_full[2];  /* of tiles in turn */
    uint64_t o_done[2], o_free;     /* O of a tile is complete; O of a piece has been read */
    uint64_t q_full, q_empty;
    uint64_t settled;               /* every product has been computed */
    uint64_t planned[kPlanned], taken[kPlanned];
    Piece pieces[kPlanned];         /* one without tiles ends the work */
    uint32_t tmem;
    uint32_t limit;                 /* polls of a wait */
    uint32_t end_at[2], end_parity[2], end_q;   /* where the loaders of K, V and Q stopped */
    volatile uint32_t dead;         /* a wait ran out: every role leaves */
    volatile uint32_t spoilt[4];    /* [piece % 4] == piece + 1: values of its fed nodes that are not finite were set aside */
    int64_t share, scan[Roles<kWiden>::kThreads / 32];
    Line line;                      /* the CTA's part of it */
};
static_assert(sizeof(Shared) <= 1024, "the last KiB of the dynamic shared memory");

/* Waits for the phase of `parity`, about a second at most.  A parity tells a
 * phase from the one before and the one after only.  Softmax does not wait for
 * every O: O is done at two barriers in turn, so that where it waits for one,
 * the one before at that barrier is known to be done (S of a tile is issued
 * behind O of the tile two before) and the one after is not yet issued. */
__device__ __noinline__ bool wait_long(Shared &sh, int32_t *error, uint32_t bar, uint32_t parity)
{
    for (uint32_t i = 0; !mbar_try_wait(bar, parity); i++) {
        if (sh.dead)
            return false;
        if (i >= sh.limit) {
            sh.dead = 1;
            atomicOr(error, KVATTN_ERR_TIMEOUT);
            return false;
        }
        if (i > 64)
            __nanosleep(32);
    }
    return true;
}

__device__ __forceinline__ bool wait(Shared &sh, int32_t *error, uint32_t bar, uint32_t parity)
{
    return mbar_try_wait(bar, parity) || wait_long(sh, error, bar, parity);
}

/* the same for what is in flight after a wait ran out, whatever comes of it */
__device__ void settle(const Shared &sh, uint32_t bar, uint32_t parity)
{
    for (uint32_t i = 0; i < sh.limit && !mbar_try_wait(bar, parity); i++)
        if (i > 64)
            __nanosleep(32);
}

/* the same for a whole warp, whose lanes go on together or not at all */
__device__ __forceinline__ bool wait_warp(Shared &sh, int32_t *error, uint32_t bar, uint32_t parity)
{
    return __all_sync(~0u, wait(sh, error, bar, parity));
}

__device__ __forceinline__ bool wait_warp(Shared &sh, int32_t *error, uint64_t *bar, uint32_t parity)
{
    return wait_warp(sh, error, smem_u32(bar), parity);
}

/* piece number `piece` of the CTA, for a whole warp; false behind the last one */
__device__ __forceinline__ bool take(const Params &p, Shared &sh, uint32_t piece, Piece &e)
{
    const uint32_t k = piece % kPlanned;
    if (!wait_warp(sh, p.d.error, &sh.planned[k], piece / kPlanned & 1))
        return false;
    e = sh.pieces[k];
    __syncwarp();
    if (threadIdx.x % 32 == 0)
        mbar_arrive(&sh.taken[k]);
    return e.t1 > e.t0;
}

/* The planning warp waits for whole pieces, which take as long as their context
 * is: a minute at most.  Where another role's wait runs out it leaves with it. */
__device__ __noinline__ bool wait_taken(Shared &sh, int32_t *error, uint32_t bar, uint32_t parity)
{
    for (uint32_t i = 0; !mbar_try_wait(bar, parity); i++) {
        if (sh.dead)
            return false;
        if (i >= 64 * sh.limit) {
            sh.dead = 1;
            atomicOr(error, KVATTN_ERR_TIMEOUT);
            return false;
        }
    }
    return true;
}

/* the planning warp: finding a piece is a chain of loads and divisions, which
 * the others would wait for (7000 cycles a piece when each did it itself) */
__device__ __forceinline__ void plan(const Params &p, Shared &sh, Line line)
{
    Piece e;
    for (uint32_t piece = 0, more = 1; more; piece++) {
        const uint32_t k = piece % kPlanned;
        more = line.next(p, sh.share, e);
        if (!more)
            e.t0 = e.t1 = 0;
        const uint32_t bar = smem_u32(&sh.taken[k]), parity = piece / kPlanned & 1 ^ 1;
        if (!__all_sync(~0u, mbar_try_wait(bar, parity) || wait_taken(sh, p.d.error, bar, parity)))
            return;
        if (threadIdx.x % 32 == 0) {
            sh.pieces[k] = e;
            mbar_arrive(&sh.planned[k]);
        }
    }
}

/* One lane of a converged warp.  What the tensor cores and the TMA are given
 * lives in uniform registers: the issuing warps run their loops as a whole and
 * leave only the instruction itself to one lane (with the whole loop in a
 * lane's branch each product took 80 cycles to issue, each load 160). */
__device__ __forceinline__ bool elect()
{
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one != 0;
}

template <typename I> __device__ __forceinline__ I uniform(I x) { return (I)__shfl_sync(~0u, (int32_t)x, 0); }

/* shared-memory matrix descriptor, 128-byte swizzle: the low word (where it
 * starts, and the bytes between 64-value columns of an operand stored row by
 * row) and the high word, which is the same for all here (1024 bytes from one
 * group of eight rows to the next) */
__device__ __forceinline__ uint32_t matrix(uint32_t addr, uint32_t lead)
{
    return (addr >> 4 & 0x3fff) | (lead >> 4 & 0x3fff) << 16;
}
constexpr uint32_t kMatrixHigh = 1024u >> 4 | 1u << 14 | 2u << 29;
constexpr uint32_t kNoLead = 16;    /* operands of one column, or stored k innermost */

/* instruction descriptor of kind::f16: 128 rows, n columns, 32-bit sums; b_rows: B is stored row by row (k outermost) */
__device__ __forceinline__ uint32_t instruction(uint32_t bf16, uint32_t n, uint32_t b_rows)
{
    return 1u << 4 | bf16 << 7 | bf16 << 10 | b_rows << 16 | (n >> 3) << 17 | (uint32_t)(kRows >> 4) << 24;
}

__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t inst, bool add)
{
    asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tsetp.ne.u32 p, %4, 0;\n\t"
                 "mov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}"
                 ::"r"(d), "r"(a), "r"(b), "r"(inst), "r"((uint32_t)add), "r"(kMatrixHigh) : "memory");
}

__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t inst, bool add)
{
    asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 b;\n\tsetp.ne.u32 p, %4, 0;\n\t"
                 "mov.b64 b, {%2, %5};\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}"
                 ::"r"(d), "r"(a), "r"(b), "r"(inst), "r"((uint32_t)add), "r"(kMatrixHigh) : "memory");
}

/* arrive at `bar` when the products issued so far are done */
__device__ __forceinline__ void mma_commit(uint64_t *bar)
{
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

__device__ __forceinline__ void tmem_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

#define R8(a, o) "=r"(a[o]), "=r"(a[o + 1]), "=r"(a[o + 2]), "=r"(a[o + 3]), "=r"(a[o + 4]), "=r"(a[o + 5]), "=r"(a[o + 6]), "=r"(a[o + 7])
#define W8(a, o) "r"(a[o]), "r"(a[o + 1]), "r"(a[o + 2]), "r"(a[o + 3]), "r"(a[o + 4]), "r"(a[o + 5]), "r"(a[o + 6]), "r"(a[o + 7])

/* loads wait in the same statement: nothing may use a register before that */
__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t *a)
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
                 "tcgen05.wait::ld.sync.aligned;"
                 : R8(a, 0), R8(a, 8) : "r"(addr) : "memory");
}

__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t *a)
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
                 "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\t"
                 "tcgen05.wait::ld.sync.aligned;"
                 : R8(a, 0), R8(a, 8), R8(a, 16), R8(a, 24) : "r"(addr) : "memory");
}

__device__ __forceinline__ void tmem_ld64(uint32_t addr, uint32_t *a)
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
                 "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, "
                 "%32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, "
                 "%48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%64];\n\t"
                 "tcgen05.wait::ld.sync.aligned;"
                 : R8(a, 0), R8(a, 8), R8(a, 16), R8(a, 24), R8(a, 32), R8(a, 40), R8(a, 48), R8(a, 56) : "r"(addr) : "memory");
}

__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t *a)
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};"
                 ::W8(a, 0), W8(a, 8), "r"(addr) : "memory");
}

__device__ __forceinline__ float exp2_approx(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

/* 32 bytes, one sector: a row's lane fills sectors of its own */
__device__ __forceinline__ void store32(void *to, const uint32_t *w)
{
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 ::"l"(to), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
}

/* ---- 16-bit types ---- */
template <typename T> struct Type;
template <> struct Type<__nv_bfloat16> {
    static constexpr uint32_t kBf16 = 1;
    /* weights are exp2(s - m) * 2^kBias with m at most kLazy behind the maximum */
    static constexpr float kLazy = 8.f, kBias = 0.f;
    static __device__ uint32_t pack(float lo, float hi)
    {
        __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<uint32_t *>(&v);
    }
    /* two e4m3 values, exactly: four conversions (there is none from 8 bits to
     * bf16, so by way of fp16 and 32 bits), where fp16 takes one */
    static __device__ uint32_t widen(uint16_t two)
    {
        const __half2 h = __half2(__nv_cvt_fp8x2_to_halfraw2(two, __NV_E4M3));
        const float2 f = __half22float2(h);
        return pack(f.x, f.y);
    }
    static __device__ bool finite(uint32_t bits16) { return (bits16 & 0x7f80) != 0x7f80; }
    static __device__ float value(uint32_t bits16) { return __uint_as_float(bits16 << 16); }
};
template <> struct Type<__half> {
    static constexpr uint32_t kBf16 = 0;
    /* fp16 has 5 exponent bits: weights up to 2^14 keep the small ones of a long context normal */
    static constexpr float kLazy = 6.f, kBias = 8.f;
    static __device__ uint32_t pack(float lo, float hi)
    {
        __half2 v = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<uint32_t *>(&v);
    }
    static __device__ uint32_t widen(uint16_t two)
    {
        const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(two, __NV_E4M3);
        return (uint32_t)h.x | (uint32_t)h.y << 16;
    }
    static __device__ bool finite(uint32_t bits16) { return (bits16 & 0x7c00) != 0x7c00; }
    static __device__ float value(uint32_t bits16) { return __half2float(__ushort_as_half((unsigned short)bits16)); }
};

__device__ __forceinline__ void copy16(uint32_t dst, const void *src, bool on)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16u : 0u) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
/* all but this thread's N last groups have landed */
template <int N> __device__ __forceinline__ void copy_wait_but() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void copy_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }
/* arrive at `bar` when this thread's copies so far have landed */
__device__ __forceinline__ void copy_arrive(uint64_t *bar)
{
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
/* what this thread has written to shared memory, or seen written, comes before the products behind it */
__device__ __forceinline__ void fence_async_proxy() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ void mbar_expect(uint32_t bar, uint32_t bytes)
{
    asm volatile("mbarrier.arrive.expect_tx.release.cta.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}

__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap *map, int32_t x, int32_t y, int32_t z, uint32_t bar)
{
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
}

__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap *map, int32_t x, int32_t y, int32_t z, int32_t w, uint32_t bar)
{
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar) : "memory");
}

/* where chunk c (16 bytes) of row r stands in a slot */
__device__ __forceinline__ uint32_t swizzled(uint32_t r, uint32_t c)
{
    return r * (kColumn * 2) + ((c ^ r) & 7) * 16;
}

/* ------------------------------------------------------------------------
 * loaders: a ring of tiles of K, one of tiles of V; a piece's last tile first.
 * ---------------------------------------------------------------------- */
/* a place in a ring, and how often the ring has been gone around */
template <int N> struct Turn {
    uint32_t slot = 0, lap = 0;
    __device__ __forceinline__ void next()
    {
        if (++slot == N) {
            slot = 0;
            lap++;
        }
    }
};

template <typename T, Load L, int DP> struct Loader {
    using S = Shape<L, DP>;
    static constexpr bool F8 = L == kWiden;
    enum : uint64_t { kNone = ~0ull };
    static constexpr int kChunks = F8 ? 4 : 8;                  /* 16-byte loads of a row of a column */
    static constexpr int kPass = 128 / kChunks;                 /* rows of one pass */
    static constexpr int kPasses = kTile / kPass;
    static constexpr int kWarpRows = kPass / 4;                 /* of them a warp's */
    static_assert(kPasses * kWarpRows == 16, "a lane of each half warp looks after one of the warp's rows");

    const Params &p;
    Shared &sh;
    uint8_t *ring;                      /* K's slots, then V's, then the 8-bit ones */
    Turn<S::kSlotsK> at_k;
    Turn<S::kSlotsV> at_v;

    __device__ Loader(const Params &p_, Shared &sh_, uint8_t *ring_) : p(p_), sh(sh_), ring(ring_) {}

    /* the slot of the next tile of V or K may be written; the lanes go on together or not at all */
    __device__ __forceinline__ bool acquire(bool v)
    {
        return wait_warp(sh, p.d.error, v ? &sh.v_empty[at_v.slot] : &sh.k_empty[at_k.slot], (v ? at_v.lap : at_k.lap) & 1 ^ 1);
    }
    __device__ __forceinline__ uint8_t *slot(bool v) const
    {
        return ring + (v ? S::kSlotsK + at_v.slot : at_k.slot) * S::kSlotBytes;
    }
    __device__ __forceinline__ uint64_t *full(bool v) const { return v ? &sh.v_full[at_v.slot] : &sh.k_full[at_k.slot]; }
    __device__ __forceinline__ void advance(bool v)
    {
        if (v)
            at_v.next();
        else
            at_k.next();
    }

    /* Boxes of a page's rows by a column; a lane looks up its box's page.  Rows
     * behind the end, and those of padding nodes, hold anything: their scores are
     * masked, and softmax makes their values finite.  A page id out of range is
     * out of the map: zeros.  One warp brings K, another V. */
    __device__ void run_tma(bool v)
    {
        const uint32_t lane = threadIdx.x % 32, boxes = kTile / p.box, box_bytes = p.box * (kColumn * 2);
        const uint32_t slots = uniform(v ? S::kSlotsV : S::kSlotsK), base = uniform(smem_u32(slot(v)));
        const uint32_t bars = uniform(smem_u32(v ? sh.v_full : sh.k_full)), frees = uniform(smem_u32(v ? sh.v_empty : sh.k_empty));
        const CUtensorMap *map = v ? &p.v_map : &p.k_map;
        uint32_t at = 0, parity = 1;
        auto stop = [&] {                   /* for land() */
            if (lane == 0)
                sh.end_at[v] = at, sh.end_parity[v] = parity;
        };
        Piece e;
        for (uint32_t piece = 0; take(p, sh, piece, e); piece++) {
            const int32_t *tab = p.d.table + (int64_t)e.row * p.d.table_stride;
            const int32_t t0 = uniform(e.t0), t1 = uniform(e.t1), end = uniform(e.end), h = uniform(e.h);
            int32_t t = uniform(e.top), pos = t * kTile + (int32_t)(lane * p.box);
            int32_t next = lane < boxes && pos < end ? tab[fdiv(pos, p.block)] : 0;
            for (int32_t left = t1 - t0; left > 0; left--) {
                const int32_t page = next;
                /* a page of more than 64 rows holds several tiles */
                const int32_t first = uniform(boxes == 1 ? pos - (int32_t)(fdiv(pos, p.block) * p.block.d) : 0);
                const uint32_t n = min(boxes, (end - t * kTile + p.box - 1) / p.box);
                if (lane < n && (uint32_t)page >= p.d.num_pages)
                    atomicOr(p.d.error, KVATTN_ERR_PAGE);
                t = t == t0 ? t1 - 1 : t - 1;
                pos = t * kTile + (int32_t)(lane * p.box);
                if (left > 1)
                    next = lane < boxes && pos < end ? tab[fdiv(pos, p.block)] : 0;     /* in flight while the tile is loaded */
                if (!wait_warp(sh, p.d.error, frees + at * 8, parity))
                    return stop();
                const uint32_t bar = bars + at * 8;
                uint32_t to = base + at * S::kSlotBytes;
                if (elect())
                    mbar_expect(bar, n * box_bytes * p.columns);
                __syncwarp();
                for (uint32_t b = 0; b < n; b++, to += box_bytes) {
                    const int32_t id = __shfl_sync(~0u, page, b);
                    if (elect())
#pragma unroll
                        for (uint32_t c = 0; c < DP / kColumn; c++)
                            if (c < p.columns)
                                tma_load(to + c * kColumnBytes, map, c * kColumn, first, h, id, bar);
                }
                if (++at == slots) {
                    at = 0;
                    parity ^= 1;
                }
            }
        }
        stop();
    }

    /* after a wait ran out: the last load of each slot, of the lap that run_tma
     * ended in, of the one before, or none (a phase that counts as over) */
    static __device__ void land(Shared &sh, bool v)
    {
        for (uint32_t k = 0; k < (v ? S::kSlotsV : S::kSlotsK); k++)
            settle(sh, smem_u32(v ? &sh.v_full[k] : &sh.k_full[k]), k < sh.end_at[v] ? sh.end_parity[v] ^ 1 : sh.end_parity[v]);
    }

    /* ---- 16 bytes at a time: pages of any size ---- */
    uint32_t chunk, row;                /* this thread's chunk, and row of a pass */
    uint32_t own_row;                   /* the row of a tile whose place this lane works out */
    uint64_t off[kPasses];              /* of this thread's rows in the planes, kNone: read as zeros */

    __device__ void take_rows()
    {
        const uint32_t t = (threadIdx.x - kSoftmax) % 128, lane = t % 32, warp = t / 32;
        chunk = t % kChunks;
        row = t / kChunks;
        own_row = lane % 16 / kWarpRows * kPass + warp * kWarpRows + lane % kWarpRows;
    }

    /* the page of this lane's row of tile t: a load that waits for nothing */
    __device__ int32_t look_up(const Piece &e, int32_t t) const
    {
        const uint32_t pos = t * kTile + own_row;
        return (int32_t)pos < e.end ? p.d.table[(int64_t)e.row * p.d.table_stride + fdiv(pos, p.block)] : -1;
    }

    /* The places of the thread's rows: each lane works out one, the threads of
     * a row take it from there. */
    __device__ void places(const Piece &e, int32_t t, int32_t page)
    {
        const kv_attn_desc &d = p.d;
        const uint32_t pos = t * kTile + own_row, j = pos - fdiv(pos, p.block) * p.block.d, esz = F8 ? 1 : 2;
        uint64_t own = kNone;
        if ((int32_t)pos < e.end) {
            if ((uint32_t)page < d.num_pages)
                own = (uint64_t)(uint32_t)page * p.stride +
                      ((uint64_t)j * (d.head_major ? 1 : d.num_kv_heads) + (uint64_t)(d.head_major ? d.block_size : 1) * e.h) *
                          (d.head_dim * esz);
            else
                atomicOr(d.error, KVATTN_ERR_PAGE);
            if (d.parents && (int32_t)pos >= e.ctx && !node_ok(d.parents + e.q0, pos - e.ctx))
                own = kNone;            /* padding nodes are not read */
        }
        const uint32_t from = threadIdx.x % 32 / kChunks;
#pragma unroll
        for (int i = 0; i < kPasses; i++)
            off[i] = __shfl_sync(~0u, own, i * kWarpRows + from);
    }

    /* this thread's share of K or V, asynchronously; chunk c's row of pass i goes to place(c, i) */
    template <typename F> __device__ __forceinline__ void copy_tile(bool v, F place)
    {
        const char *plane = static_cast<const char *>(v ? p.d.v : p.d.k);
#pragma unroll
        for (uint32_t c = 0; c < DP / kColumn; c++) {
            const uint32_t x = c * (F8 ? kColumn : kColumn * 2) + chunk * 16;
            if (x < p.d.head_dim * (F8 ? 1 : 2))
#pragma unroll
                for (int i = 0; i < kPasses; i++)
                    copy16(place(c, i), plane + (off[i] == kNone ? 0 : off[i] + x), off[i] != kNone);
        }
    }

    __device__ void run_copy()
    {
        take_rows();
        Piece e;
        for (uint32_t piece = 0; take(p, sh, piece, e); piece++) {
            int32_t t = e.top, page = look_up(e, t);
            for (int32_t left = e.t1 - e.t0; left > 0; left--) {
                places(e, t, page);
                t = e.behind(t);
                if (left > 1)
                    page = look_up(e, t);       /* in flight while the tile is copied */
                for (int v = 0; v < 2; v++) {
                    if (!acquire(v))
                        return;
                    const uint32_t to = smem_u32(slot(v));
                    copy_tile(v, [&](uint32_t c, int i) { return to + c * kColumnBytes + swizzled(row + i * kPass, chunk); });
                    copy_arrive(full(v));
                    advance(v);
                }
            }
        }
    }

    /* 8-bit caches: copied as they are, to places in shared memory that only the
     * copying thread uses, a tile ahead; that thread widens them into the rings. */
    __device__ __forceinline__ uint8_t *raw(bool v, uint32_t k, uint32_t c, int i) const
    {
        return ring + (S::kSlotsK + S::kSlotsV) * S::kSlotBytes + (2 * v + k % 2) * (S::kSlotBytes / 2) + (c * kPasses + i) * (128 * 16) +
               (threadIdx.x - kSoftmax) % 128 * 16;
    }

    __device__ bool widen(uint32_t k, bool v)
    {
        if (!acquire(v))
            return false;
#pragma unroll
        for (uint32_t c = 0; c < DP / kColumn; c++)
            if (c * kColumn + chunk * 16 < p.d.head_dim)
#pragma unroll
                for (int i = 0; i < kPasses; i++) {
                    const uint4 w = *reinterpret_cast<const uint4 *>(raw(v, k, c, i));
                    const uint32_t r = row + i * kPass;
                    uint8_t *to = slot(v) + c * kColumnBytes;
                    *reinterpret_cast<uint4 *>(to + swizzled(r, 2 * chunk)) =
                        make_uint4(Type<T>::widen((uint16_t)w.x), Type<T>::widen((uint16_t)(w.x >> 16)),
                                   Type<T>::widen((uint16_t)w.y), Type<T>::widen((uint16_t)(w.y >> 16)));
                    *reinterpret_cast<uint4 *>(to + swizzled(r, 2 * chunk + 1)) =
                        make_uint4(Type<T>::widen((uint16_t)w.z), Type<T>::widen((uint16_t)(w.z >> 16)),
                                   Type<T>::widen((uint16_t)w.w), Type<T>::widen((uint16_t)(w.w >> 16)));
                }
        mbar_arrive(full(v));
        advance(v);
        return true;
    }

    /* Four warps bring K, four V: with four for both, that widened a tile of
     * each in turn, their instructions set the pace (32 chains over up to 8192
     * positions: 150 us, 143 like this).  Fetched to registers instead of shared
     * memory the same takes 162 us a tile ahead, 185 two tiles ahead. */
    __device__ void run_widen(bool v)
    {
        take_rows();
        uint32_t k = 0;                     /* tiles fetched; all but the last are widened */
        Piece e;
        for (uint32_t piece = 0; take(p, sh, piece, e); piece++) {
            int32_t t = e.top, page = look_up(e, t);
            for (int32_t left = e.t1 - e.t0; left > 0; left--) {
                places(e, t, page);
                t = e.behind(t);
                if (left > 1)
                    page = look_up(e, t);
                copy_tile(v, [&](uint32_t c, int i) { return smem_u32(raw(v, k, c, i)); });
                copy_commit();
                if (k++) {
                    copy_wait_but<1>();
                    if (!widen(k - 2, v))
                        return;
                }
            }
        }
        copy_wait_all();
        if (k)
            widen(k - 1, v);
    }
};

/* ------------------------------------------------------------------------
 * products.  S of tile g + 1 is issued before O += P V of tile g, to be computed
 * under the softmax of g.  Those of a CTA run in the order in which they were
 * issued, so S may overwrite a buffer whose P an earlier one reads.  The same
 * warp has Q loaded: of the next piece as soon as the last S of this one is
 * done, under its softmax.
 * ---------------------------------------------------------------------- */
__device__ __forceinline__ void load_q(const Params &p, Shared &sh, uint8_t *q_smem, const Piece &e)
{
    const int32_t head = uniform(e.h * (int32_t)p.group), q = uniform(e.q0 + e.node0);
    if (elect()) {
        const uint32_t bar = smem_u32(&sh.q_full);
        mbar_expect(bar, p.columns * p.nodes.d * p.group * (kColumn * 2));
        sh.end_q++;
        for (uint32_t c = 0; c < p.columns; c++)    /* rows behind the sequence's are another's, and not used */
            tma_load(smem_u32(q_smem) + c * (kRows * kColumn * 2), &p.q_map, c * kColumn, head, q, bar);
    }
    __syncwarp();
}

template <typename T, Load L, int DP>
__device__ void products(const Params &p, Shared &sh, uint8_t *q_smem, uint8_t *ring)
{
    using S = Shape<L, DP>;
    const uint32_t dim = p.d.head_dim, s = uniform(sh.tmem), o = s + 2 * kTile;
    const uint32_t inst_s = instruction(Type<T>::kBf16, kTile, 0), inst_o = instruction(Type<T>::kBf16, dim, 1);
    const uint32_t q0 = matrix(smem_u32(q_smem), kNoLead), k0 = matrix(smem_u32(ring), kNoLead),
                   v0 = matrix(smem_u32(ring) + S::kSlotsK * S::kSlotBytes, kColumnBytes);
    Turn<S::kSlotsK> at_k;
    Turn<S::kSlotsV> at_v;
    uint32_t g = 0, piece = 0;
    Piece e;
    bool more = take(p, sh, 0, e);
    /* S of a tile; the last of its piece also releases Q */
    auto scores = [&](uint32_t tile, bool last) {
        if (!wait_warp(sh, p.d.error, &sh.k_full[at_k.slot], at_k.lap & 1))
            return false;
        if (L != kTma)
            fence_async_proxy();
        tmem_fence_after();
        const uint32_t b = k0 + at_k.slot * (S::kSlotBytes >> 4), to = s + (tile & 1) * kTile;
        if (elect()) {
#pragma unroll
            for (uint32_t x = 0; x < DP / 16; x++)
                if (x * 16 < dim)
                    mma_ss(to, q0 + ((x >> 2) * (kRows * kColumn * 2 >> 4) + (x & 3) * 2), b + ((x >> 2) * (kColumnBytes >> 4) + (x & 3) * 2),
                           inst_s, x > 0);
            mma_commit(&sh.k_empty[at_k.slot]);
            mma_commit(&sh.s_full[tile & 1]);
            if (last)
                mma_commit(&sh.q_empty);
        }
        __syncwarp();
        at_k.next();
        return true;
    };
    if (more)
        load_q(p, sh, q_smem, e);
    for (; uniform(more); piece++) {
        const int32_t n = uniform(e.t1 - e.t0);
        if (!wait_warp(sh, p.d.error, &sh.q_full, piece & 1) || !scores(g, n == 1))
            return;
        for (int32_t k = 0; k < n; k++, g++) {
            if (k + 1 < n && !scores(g + 1, k + 2 == n))
                return;
            if (k + 1 == n) {
                more = take(p, sh, piece + 1, e);
                if (!wait_warp(sh, p.d.error, &sh.q_empty, piece & 1))
                    return;
                if (uniform(more))
                    load_q(p, sh, q_smem, e);
            }
            if (k == 0 && piece && !wait_warp(sh, p.d.error, &sh.o_free, (piece - 1) & 1))
                return;
            if (!wait_warp(sh, p.d.error, &sh.v_full[at_v.slot], at_v.lap & 1) ||
                !wait_warp(sh, p.d.error, &sh.p_full[g & 1], (g >> 1) & 1))
                return;
            if (L != kTma)
                fence_async_proxy();
            tmem_fence_after();
            const uint32_t b = v0 + at_v.slot * (S::kSlotBytes >> 4), a = s + (g & 1) * kTile;
            if (elect()) {
#pragma unroll
                for (uint32_t x = 0; x < kTile / 16; x++)
                    mma_ts(o, a + x * 8, b + x * (16 * kColumn * 2 >> 4), inst_o, k > 0 || x > 0);
                mma_commit(&sh.v_empty[at_v.slot]);
                mma_commit(&sh.o_done[g & 1]);
            }
            __syncwarp();
            at_v.next();
        }
    }
}

/* ------------------------------------------------------------------------
 * softmax: thread = row.  m lags behind the true maximum by up to kLazy (in
 * powers of two), so that O, which lives in TMEM, is rescaled rarely; the
 * result is the same quotient.  The weights are rounded to the 16-bit type of
 * the products (half a step, 2^-8 of a weight in bf16, 2^-11 in fp16), which is
 * what the tensor cores take; their sum is that of the unrounded ones, and m, l
 * and O are held in 32 bits.
 * ---------------------------------------------------------------------- */
/* The positions p0 .. p0 + 64 that a node sees, a bit each.  j is the node, or
 * in a tree the nearest of its line (the node itself, its ancestors) that stands
 * before p0 + 64 or not much behind it, and on return the one before p0: tiles
 * come from the last to the first, and a piece walks a line once or twice. */
__device__ uint64_t seen(const Params &p, const Piece &e, int32_t &j, int32_t p0)
{
    const int32_t before = e.ctx - p0;
    uint64_t bits = before >= 64 ? ~0ull : before > 0 ? (1ull << before) - 1 : 0;
    if (!p.d.parents) {
        const int32_t upto = before + j + 1;
        return upto >= 64 ? ~0ull : upto > 0 ? (1ull << upto) - 1 : 0;
    }
    const int32_t *par = p.d.parents + e.q0;
    while (j >= 0 && before + j >= 0) {
        if (before + j < 64)
            bits |= 1ull << (before + j);
        const int32_t u = par[j];
        j = u >= 0 && node_ok(par, u) ? u : -1;
    }
    return bits;
}

/* Adds to O what was set aside of the values that node j sees in the piece's
 * tiles; the warp's rows that are not `active` add nothing.  Rare, and kept out
 * of the loops' way: inlined, it pushed them out of the instruction cache. */
template <typename T, bool F8>
__device__ __noinline__ void add_spoilt(const Params &p, const Piece &e, int32_t j, bool active, uint32_t o_at)
{
    const kv_attn_desc &d = p.d;
    const int32_t *par = d.parents ? d.parents + e.q0 : nullptr;
    const int32_t *tab = d.table + (int64_t)e.row * d.table_stride;
#pragma unroll 1
    for (uint32_t c = 0; c < d.head_dim; c += 16) {
        uint32_t raw[16];
        tmem_ld16(o_at + c, raw);
#pragma unroll 1
        for (int32_t a = active ? j : -1; a >= 0 && e.ctx + a >= e.t0 * kTile;) {
            const uint32_t pos = e.ctx + a, b = fdiv(pos, p.block);
            const int32_t page = tab[b];
            if (pos < (uint32_t)e.t1 * kTile && page >= 0 && (uint32_t)page < d.num_pages) {
                const uint64_t at = ((uint64_t)(pos - b * p.block.d) * (d.head_major ? 1 : d.num_kv_heads) +
                                     (uint64_t)(d.head_major ? d.block_size : 1) * e.h) * d.head_dim + c;
                const char *base = static_cast<const char *>(d.v) + (uint64_t)page * p.stride;
#pragma unroll
                for (int x = 0; x < 16; x++) {
                    const uint32_t w = F8 ? Type<T>::widen(reinterpret_cast<const uint8_t *>(base)[at + x])
                                          : reinterpret_cast<const uint16_t *>(base)[at + x];
                    if (!Type<T>::finite(w))
                        raw[x] = __float_as_uint(__uint_as_float(raw[x]) + Type<T>::value(w & 0xffff));
                }
            }
            const int32_t u = par ? par[a] : a - 1;
            a = u < 0 || (par && !node_ok(par, u)) ? -1 : u;
        }
        __syncwarp();
        tmem_st16(o_at + c, raw);
    }
    tmem_wait_st();
}

/* Rows first .. of a slot of V, behind the cached context: the softmax threads
 * set values that are not finite to 0, which would otherwise reach the rows that
 * do not see them, as 0 * value.  True if one of them is a fed node's (and not
 * what a row behind the end or a padding node's happens to hold): such values
 * are added to the rows that do see them. */
template <typename T>
__device__ bool set_aside(const Params &p, const Piece &e, int32_t t, uint8_t *slot, uint32_t values)
{
    bool any = false;
    const int32_t skip = max(0, e.ctx - t * kTile);     /* the context's */
#pragma unroll 4
    for (uint32_t x = skip * 8 + threadIdx.x; x < kColumnBytes / 16; x += kSoftmax) {
        const int32_t j = t * kTile + (int32_t)(x / 8) - e.ctx;
        if (((x ^ x >> 3) & 7) * 8 >= values)
            continue;                   /* behind the head's dimensions */
        uint4 v = *reinterpret_cast<uint4 *>(slot + x * 16);
        uint32_t *w = reinterpret_cast<uint32_t *>(&v);
        bool here = false;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            if (!Type<T>::finite(w[k])) {
                w[k] &= 0xffff0000u;
                here = true;
            }
            if (!Type<T>::finite(w[k] >> 16)) {
                w[k] &= 0x0000ffffu;
                here = true;
            }
        }
        if (here) {
            *reinterpret_cast<uint4 *>(slot + x * 16) = v;
            any |= j < e.nodes && (!p.d.parents || node_ok(p.d.parents + e.q0, j));
        }
    }
    return any;
}

/* N scores of the row, -inf where the bit is off */
template <int N> __device__ __forceinline__ void scores(uint32_t addr, uint32_t *raw, bool mask, uint64_t bits)
{
    if constexpr (N == 64)
        tmem_ld64(addr, raw);
    else
        tmem_ld32(addr, raw);
    if (mask)
#pragma unroll
        for (int c = 0; c < N; c++)
            raw[c] = bits >> c & 1 ? raw[c] : __float_as_uint(-INFINITY);
}

template <typename T, Load L, int DP>
__device__ void softmax(const Params &p, Shared &sh, uint8_t *ring)
{
    using S = Shape<L, DP>;
    const kv_attn_desc &d = p.d;
    const uint32_t tid = threadIdx.x, lanes = (tid / 32 * 32) << 16;
    const uint32_t tmem = sh.tmem + lanes, o_at = tmem + 2 * kTile;
    const float s2 = d.scale * d.k_scale * kLog2e;
    const int32_t my_node = (int32_t)(tid / p.group), sub = (int32_t)(tid % p.group);
    uint32_t g = 0, piece = 0;
    Turn<S::kSlotsV> at_v;
    Piece e;
    for (; take(p, sh, piece, e); piece++) {
        const bool valid = (int32_t)tid < e.rows(p);
        const int32_t node = valid ? e.node0 + my_node : 0;
        bool active = valid;
        if (valid && d.parents && !node_ok(d.parents + e.q0, node)) {
            active = false;
            if (d.parents[e.q0 + node] != -2)
                atomicOr(d.error, KVATTN_ERR_PARENT);
        }
        const bool work = __any_sync(~0u, active);
        const int32_t t0 = e.t0, t1 = e.t1, ctx = e.ctx;
        float m = -INFINITY, l = 0;
        int32_t line = node, t = e.top;
        for (int32_t left = t1 - t0; left > 0; left--, t = e.behind(t), g++, at_v.next()) {
            const uint32_t s_at = tmem + (g & 1) * kTile;
            const bool mask = (uint32_t)(t + 1) * kTile > (uint32_t)ctx;
            uint64_t bits = 0;
            if (t == t1 - 1)
                line = node;
            if (mask && active)
                bits = seen(p, e, line, t * kTile);
            if (!wait_warp(sh, d.error, &sh.s_full[g & 1], (g >> 1) & 1))
                return;
            if (work) {
                /* The maximum first.  Where two loading warps leave registers for
                 * all scores they stay (8 trees of 64 nodes over up to 131072
                 * positions: 180 us, 189 read twice); with four or more they are
                 * read again (64 trees on pages of 24: 89 us, 97 with spills). */
                constexpr int kHeld = L == kTma ? 64 : 32;
                uint32_t raw[kHeld];
                const float *s = reinterpret_cast<const float *>(raw);
                float now = -INFINITY;
                tmem_fence_after();
#pragma unroll 1
                for (int part = 0; part < kTile; part += kHeld) {
                    scores<kHeld>(s_at + part, raw, mask, bits >> part);
                    float top[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
                    for (int c = 4; c < kHeld; c++)
                        top[c & 3] = fmaxf(top[c & 3], s[c]);
                    now = fmaxf(now, fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])));
                }
                now *= s2;
                const bool raise = active && now > m + Type<T>::kLazy;
                if (left == t1 - t0) {
                    m = now;
                } else if (__any_sync(~0u, raise)) {
                    const float f = raise ? exp2_approx(m - now) : 1.f;
                    if (raise)
                        m = now;
                    l *= f;
                    if (!wait_warp(sh, d.error, &sh.o_done[(g - 1) & 1], ((g - 1) >> 1) & 1))
                        return;
                    tmem_fence_after();
#pragma unroll 1
                    for (uint32_t c = 0; c < d.head_dim; c += 16) {
                        uint32_t o[16];
                        tmem_ld16(o_at + c, o);
#pragma unroll
                        for (int k = 0; k < 16; k++)
                            o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
                        tmem_st16(o_at + c, o);
                    }
                }
                const float from = (m == -INFINITY ? 0.f : m) - Type<T>::kBias;
#pragma unroll 1
                for (int part = 0; part < kTile; part += kHeld) {
                    if (kHeld < kTile)
                        scores<kHeld>(s_at + part, raw, mask, bits >> part);
#pragma unroll
                    for (int half = 0; half < kHeld; half += 32) {
                        float sum[4] = {};
                        uint32_t w[16];
#pragma unroll
                        for (int c = 0; c < 32; c += 2) {
                            const float a = exp2_approx(fmaf(s[half + c], s2, -from)), b = exp2_approx(fmaf(s[half + c + 1], s2, -from));
                            sum[c & 2] += a;
                            sum[(c & 2) + 1] += b;
                            w[c / 2] = Type<T>::pack(a, b);
                        }
                        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                        tmem_st16(s_at + (part + half) / 2, w);     /* over scores that have been read */
                    }
                }
                tmem_wait_st();
                tmem_fence_before();
            }
            if (mask) {                 /* V of a tile with fed nodes */
                if (!wait_warp(sh, d.error, &sh.v_full[at_v.slot], at_v.lap & 1))
                    return;
                bool any = false;
                for (uint32_t c = 0; c < p.columns; c++)
                    any |= set_aside<T>(p, e, t, ring + (S::kSlotsK + at_v.slot) * S::kSlotBytes + c * kColumnBytes,
                                        d.head_dim - c * kColumn);
                if (any)
                    sh.spoilt[piece % 4] = piece + 1;
                fence_async_proxy();
            }
            __syncwarp();
            if (tid % 32 == 0)
                mbar_arrive(&sh.p_full[g & 1]);
        }
        /* the piece's result, or its share of it */
        if (!wait_warp(sh, d.error, &sh.o_done[(g - 1) & 1], ((g - 1) >> 1) & 1))
            return;
        tmem_fence_after();
        const bool whole = e.whole();
        const float from = (m == -INFINITY ? 0.f : m) - Type<T>::kBias;
        const uint32_t slot = 2 * blockIdx.x + (piece ? 1 : 0);
        const bool something = active && l != 0;        /* else 0, also where O is not finite: 0 * V of a weight of 0 */
        const float inv = !something ? 0.f : whole ? d.v_scale / l : 1.f;
        const bool spoilt = __any_sync(~0u, sh.spoilt[piece % 4] == piece + 1);
        if (__any_sync(~0u, valid)) {
            if (spoilt)
                add_spoilt<T, L == kWiden>(p, e, node, active, o_at);
            T *out = static_cast<T *>(d.out) + (int64_t)(e.q0 + node) * d.out_stride + (int64_t)(e.h * p.group + sub) * d.out_head_stride;
            float *part = p.part_o + ((uint64_t)slot * kRows + tid) * d.head_dim;
#pragma unroll 1
            for (uint32_t c = 0; c < d.head_dim; c += 16) {
                uint32_t raw[16], w[8];
                const float *o = reinterpret_cast<const float *>(raw);
                tmem_ld16(o_at + c, raw);
                if (whole && valid) {
#pragma unroll
                    for (int k = 0; k < 8; k++)
                        w[k] = something ? Type<T>::pack(o[2 * k] * inv, o[2 * k + 1] * inv) : 0;
                    if (p.wide_out) {
                        store32(out + c, w);
                    } else {
                        *reinterpret_cast<uint4 *>(out + c) = make_uint4(w[0], w[1], w[2], w[3]);
                        *reinterpret_cast<uint4 *>(out + c + 8) = make_uint4(w[4], w[5], w[6], w[7]);
                    }
                } else if (active) {
                    store32(part + c, raw);
                    store32(part + c + 8, raw + 8);
                }
            }
            if (tid == 0 && e.t0 == 0 && !whole)
                p.jobs[blockIdx.x] = {e.rows(p), (int32_t)(1 + (e.n - e.t1 + sh.share - 1) / sh.share), (int32_t)slot, e.q0 + e.node0, e.h};
            if (valid) {
                if (!whole) {
                    float *ml = p.part_ml + ((uint64_t)slot * kRows + tid) * 2;
                    ml[0] = active ? from : -INFINITY;
                    ml[1] = active ? l : 0.f;
                } else if (d.lse) {
                    d.lse[(int64_t)(e.q0 + node) * d.num_heads + e.h * p.group + sub] = active ? (from + log2f(l)) * kLn2 : -INFINITY;
                }
            }
        }
        tmem_fence_before();
        __syncwarp();
        if (tid % 32 == 0)
            mbar_arrive(&sh.o_free);
    }
}

/* ------------------------------------------------------------------------
 * the line: every CTA counts the call's tiles and finds its piece of them
 * ---------------------------------------------------------------------- */
template <int kThreads>
__device__ int64_t block_scan(Shared &sh, int64_t v, int64_t &total)
{
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int64_t inc = v;
#pragma unroll
    for (int k = 1; k < 32; k <<= 1) {
        const int64_t u = __shfl_up_sync(~0u, inc, k);
        if (lane >= k)
            inc += u;
    }
    __syncthreads();
    if (lane == 31)
        sh.scan[warp] = inc;
    __syncthreads();
    total = 0;
    for (int k = 0; k < kThreads / 32; k++) {
        if (k < (int)warp)
            inc += sh.scan[k];
        total += sh.scan[k];
    }
    return inc;
}

/* voids the rows of those of sequences b0 .. b1 that do not fit, with all threads of the grid */
template <typename T, int kThreads>
__device__ __noinline__ void void_rows(const Params &p, uint32_t b0, uint32_t b1)
{
    const kv_attn_desc &d = p.d;
    for (uint32_t b = b0; b < b1; b++) {
        Seq s;
        if (sequence(d, b, s))
            continue;
        if (blockIdx.x == 0 && threadIdx.x == 0)
            atomicOr(d.error, KVATTN_ERR_SEQ);
        for (int64_t x = blockIdx.x * kThreads + threadIdx.x; x < (int64_t)s.nodes * d.num_heads; x += (int64_t)gridDim.x * kThreads) {
            const int64_t i = s.q0 + x / d.num_heads, h = x % d.num_heads;
            T *out = static_cast<T *>(d.out) + i * d.out_stride + h * d.out_head_stride;
            for (uint32_t c = 0; c < d.head_dim; c += 8)
                *reinterpret_cast<uint4 *>(out + c) = make_uint4(0, 0, 0, 0);
            if (d.lse)
                d.lse[i * d.num_heads + h] = -INFINITY;
        }
    }
}

/* Adds up all sequences, kThreads at a time; the CTA's share of
 * the line, and the sequence that it begins in, go to sh.line.  With more than
 * kThreads sequences the search is a second walk. */
template <typename T, int kThreads>
__device__ void find_line(const Params &p, Shared &sh)
{
    const kv_attn_desc &d = p.d;
    const bool once = d.num_seqs <= kThreads;
    for (int walk = 0; walk < (once ? 1 : 2); walk++) {
        int64_t before = 0;
        for (uint32_t b0 = 0; b0 < d.num_seqs; b0 += kThreads) {
            const uint32_t b = b0 + threadIdx.x;
            uint64_t n = 0;
            int64_t sum;
            Seq s;
            const bool ok = b >= d.num_seqs || sequence(d, b, s);
            if (ok && b < d.num_seqs)
                n = head_cost(p, s);
            if (walk == 0 && __syncthreads_or(!ok))
                void_rows<T, kThreads>(p, b0, min(b0 + kThreads, d.num_seqs));
            const int64_t all = (int64_t)(n * d.num_kv_heads), upto = before + block_scan<kThreads>(sh, all, sum);
            before += sum;
            if (once || (walk == 0 && b0 + kThreads >= d.num_seqs)) {
                if (threadIdx.x == 0) {
                    const int64_t grid = gridDim.x, share = before >> 31 ? (before + grid - 1) / grid
                                                                         : ((uint32_t)before + gridDim.x - 1) / gridDim.x;
                    sh.share = max((int64_t)p.min_share, share);
                    sh.line.x = min(before, sh.share * blockIdx.x);
                    sh.line.hi = min(before, sh.share * (blockIdx.x + 1));
                }
                __syncthreads();
            }
            if ((once || walk == 1) && n && upto - all <= sh.line.x && sh.line.x < upto) {
                sh.line.b = b;
                sh.line.base = upto - all;
                sh.line.per_head = n;
                sh.line.s = s;
            }
        }
    }
    __syncthreads();
}

template <typename T, Load L, int DP>
__global__ void __launch_bounds__(Roles<L>::kThreads, Shape<L, DP>::kCtas) kv_attn_kernel(const __grid_constant__ Params p)
{
    using S = Shape<L, DP>;
    extern __shared__ __align__(1024) uint8_t smem[];
    constexpr int kThreads = Roles<L>::kThreads;
    uint8_t *q_smem = smem, *ring = smem + S::kQBytes;
    Shared &sh = *reinterpret_cast<Shared *>(smem + S::kShared);
    const uint32_t warp = threadIdx.x >> 5;

    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (threadIdx.x == 0) {
        const bool stall = p.stall && blockIdx.x == 0;
        sh.limit = stall ? kStallLimit : kSpinLimit;
        for (int k = 0; k < S::kSlotsK; k++) {
            mbar_init(&sh.k_full[k], Roles<L>::kFill);
            mbar_init(&sh.k_empty[k], 1);
        }
        for (int k = 0; k < S::kSlotsV; k++) {
            mbar_init(&sh.v_full[k], Roles<L>::kFill + (stall && k == 0));     /* one arrival that nobody makes */
            mbar_init(&sh.v_empty[k], 1);
        }
        for (int k = 0; k < 2; k++) {
            mbar_init(&sh.s_full[k], 1);
            mbar_init(&sh.p_full[k], kSoftmax / 32);
            mbar_init(&sh.o_done[k], 1);
        }
        for (int k = 0; k < kPlanned; k++) {
            mbar_init(&sh.planned[k], 1);
            mbar_init(&sh.taken[k], kThreads / 32 - 1);
        }
        mbar_init(&sh.o_free, kSoftmax / 32);
        mbar_init(&sh.q_full, 1);
        mbar_init(&sh.q_empty, 1);
        mbar_init(&sh.settled, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        sh.dead = 0;
        sh.end_q = 0;
        for (int k = 0; k < 4; k++)
            sh.spoilt[k] = 0;
    }
    find_line<T, kThreads>(p, sh);
    if (threadIdx.x == 0)
        p.jobs[blockIdx.x].rows = 0;
    if (sh.line.x >= sh.line.hi)
        return;
    if (warp == kThreads / 32 - 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)), "n"(S::kTmem) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    if (smem_u32(smem) % 1024 == 0) {
        if (warp < kSoftmax / 32) {
            softmax<T, L, DP>(p, sh, ring);
        } else if (warp < kThreads / 32 - 2) {
            Loader<T, L, DP> load(p, sh, ring);
            if constexpr (L == kTma) {
                load.run_tma(warp != kSoftmax / 32);
            } else if constexpr (L == kWiden)
                load.run_widen(warp >= (kSoftmax + 128) / 32);
            else
                load.run_copy();
            copy_wait_all();
        } else if (warp == kThreads / 32 - 2) {
            products<T, L, DP>(p, sh, q_smem, ring);
        } else {
            plan(p, sh, sh.line);
        }
    } else if (threadIdx.x == 0) {
        atomicOr(p.d.error, KVATTN_ERR_TIMEOUT);
    }
    tmem_fence_before();
    __syncthreads();
    if (sh.dead) {
        /* shared memory and TMEM are given up when the copies have landed and the products are done */
        if (warp == kThreads / 32 - 2) {
            if (elect())
                mma_commit(&sh.settled);
            __syncwarp();
            settle(sh, smem_u32(&sh.settled), 0);
            if (sh.end_q)
                settle(sh, smem_u32(&sh.q_full), (sh.end_q - 1) & 1);
        } else if (L == kTma && (warp == kSoftmax / 32 || warp == kSoftmax / 32 + 1)) {
            Loader<T, L, DP>::land(sh, warp != kSoftmax / 32);
        }
        for (int k = 0; L != kTma && k < 100; k++)
            __nanosleep(1000);                  /* the arrivals of 16-byte copies, which come behind the copies */
        __syncthreads();
    }
    tmem_fence_after();
    if (warp == kThreads / 32 - 1)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(sh.tmem), "n"(S::kTmem) : "memory");
}

/* ------------------------------------------------------------------------
 * join: the pieces of the row tiles that lie across CTAs, in their order.  The
 * tiles' rows, however many each has, are dealt evenly to the grid's warps; a
 * lane has four dimensions of a row, and eight loads are in flight.  Where there
 * are fewer rows than CTAs a row is a CTA's: those of a short call lie in many
 * pieces (one token's 32, of 2048 positions, in 33 each: 15.5 us instead of
 * 17.7 with a warp for a row).
 * (Joining in the first kernel, by the CTA that finishes a row tile last, takes
 * no second launch but left long joins to a few CTAs: 424 us instead of 225 for
 * 8 contexts in 37 pieces each, 118 instead of 89 for 64 in 4 or 5.)
 * ---------------------------------------------------------------------- */
/* a row's maximum and sum, and four dimensions of its result, of some pieces */
struct Partial {
    float m = -INFINITY, l = 0;
    float4 o = make_float4(0, 0, 0, 0);

    /* weighs everything for a maximum of `top` */
    __device__ __forceinline__ void raise(float top)
    {
        const float keep = exp2_approx(m - top);
        m = top;
        l *= keep;
        o = make_float4(o.x * keep, o.y * keep, o.z * keep, o.w * keep);
    }
    __device__ __forceinline__ void add(float m2, float l2, const float4 &v)
    {
        const float f = exp2_approx(m2 - m);
        l += f * l2;
        o = make_float4(o.x + f * v.x, o.y + f * v.y, o.z + f * v.z, o.w + f * v.w);
    }
};

/* pieces k0 .. k1 of rows r .. r + R, P of them in flight together; rows from r1 on are not there */
template <int R, int P>
__device__ __forceinline__ void join_pieces(const Params &p, const Job &job, uint32_t cta, int32_t r, int32_t r1, int32_t k0, int32_t k1,
                                            uint32_t c, Partial *x)
{
    /* piece k's rows: the first piece's slot, then slot 0 of the CTAs behind */
    auto at = [&](int32_t k) { return (uint64_t)(k ? 2 * (cta + k) : (uint32_t)job.slot) * kRows; };
#pragma unroll 1
    for (; k0 < k1; k0 += P) {
        float2 ml[R][P];
        float4 v[R][P];
#pragma unroll
        for (int k = 0; k < P; k++)
#pragma unroll
            for (int i = 0; i < R; i++) {
                const bool on = k0 + k < k1 && r + i < r1;
                const uint64_t row = at(k0 + k) + r + i;
                ml[i][k] = on ? *reinterpret_cast<const float2 *>(p.part_ml + row * 2) : make_float2(0, 0);
                v[i][k] = on ? *reinterpret_cast<const float4 *>(p.part_o + row * p.d.head_dim + c) : make_float4(0, 0, 0, 0);
            }
#pragma unroll
        for (int i = 0; i < R; i++) {
            float top = x[i].m;
#pragma unroll
            for (int k = 0; k < P; k++)
                if (ml[i][k].y != 0)        /* else it sees nothing there, and its sums were not written */
                    top = fmaxf(top, ml[i][k].x);
            if (top == -INFINITY)
                continue;
            x[i].raise(top);
#pragma unroll
            for (int k = 0; k < P; k++)
                if (ml[i][k].y != 0)
                    x[i].add(ml[i][k].x, ml[i][k].y, v[i][k]);
        }
    }
}

template <typename T>
__device__ __forceinline__ void join_out(const Params &p, const Job &job, int32_t r, uint32_t c, const Partial &x)
{
    const kv_attn_desc &d = p.d;
    const int32_t node = r / (int32_t)p.group, sub = r - node * (int32_t)p.group;
    const float inv = x.l == 0 ? 0.f : d.v_scale / x.l;
    T *out = static_cast<T *>(d.out) + (int64_t)(job.q0 + node) * d.out_stride + (int64_t)(job.h * p.group + sub) * d.out_head_stride;
    *reinterpret_cast<uint2 *>(out + c) = make_uint2(Type<T>::pack(x.o.x * inv, x.o.y * inv), Type<T>::pack(x.o.z * inv, x.o.w * inv));
    if (c == 0 && d.lse)
        d.lse[(int64_t)(job.q0 + node) * d.num_heads + job.h * p.group + sub] = x.l == 0 ? -INFINITY : (x.m + log2f(x.l)) * kLn2;
}

/* rows r0 .. r1 of a job, R rows and P pieces in flight together */
template <typename T, int R, int P>
__device__ __forceinline__ void join_rows(const Params &p, const Job &job, uint32_t cta, int32_t r0, int32_t r1, uint32_t lane)
{
    for (uint32_t c = lane * 4; c < p.d.head_dim; c += 128)
#pragma unroll 1
        for (int32_t r = r0; r < r1; r += R) {
            Partial x[R];
            join_pieces<R, P>(p, job, cta, r, r1, 0, job.ctas, c, x);
#pragma unroll
            for (int i = 0; i < R; i++) {
                if (r + i >= r1)
                    break;
                join_out<T>(p, job, r + i, c, x[i]);
            }
        }
}

/* one row by the whole CTA: each warp joins some of the pieces, the first one what they have */
template <typename T>
__device__ __forceinline__ void join_row(const Params &p, const Job &job, uint32_t cta, int32_t r, uint32_t lane, uint32_t warp)
{
    constexpr int kWarps = kJoinThreads / 32;
    __shared__ Partial of[kWarps][32];
    const int32_t each = (job.ctas + kWarps - 1) / kWarps, k0 = warp * each, k1 = min(job.ctas, k0 + each);
    for (uint32_t c0 = 0; c0 < p.d.head_dim; c0 += 128) {
        const uint32_t c = c0 + lane * 4;
        Partial x;
        if (c < p.d.head_dim)
            join_pieces<1, 8>(p, job, cta, r, r + 1, k0, k1, c, &x);
        of[warp][lane] = x;
        __syncthreads();
        if (warp == 0 && c < p.d.head_dim) {
            for (int w = 1; w < kWarps; w++) {
                const Partial y = of[w][lane];
                if (y.l == 0)
                    continue;
                const float top = fmaxf(x.m, y.m);
                x.raise(top);
                x.add(y.m, y.l, y.o);
            }
            join_out<T>(p, job, r, c, x);
        }
        __syncthreads();
    }
}

template <typename T>
__global__ void __launch_bounds__(kJoinThreads) kv_attn_join_kernel(const __grid_constant__ Params p, uint32_t ctas)
{
    __shared__ int32_t upto[kMaxCtas], warp_sum[kJoinThreads / 32];
    const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    /* rows before and with each job's */
    constexpr int kEach = kMaxCtas / kJoinThreads;
    int32_t rows[kEach], sum = 0;
#pragma unroll
    for (int k = 0; k < kEach; k++) {
        const uint32_t c = threadIdx.x * kEach + k;
        rows[k] = c < ctas ? p.jobs[c].rows : 0;
        sum += rows[k];
    }
    int32_t inc = sum;
#pragma unroll
    for (int k = 1; k < 32; k <<= 1) {
        const int32_t u = __shfl_up_sync(~0u, inc, k);
        if (lane >= (uint32_t)k)
            inc += u;
    }
    if (lane == 31)
        warp_sum[warp] = inc;
    __syncthreads();
    int32_t total = 0;
#pragma unroll
    for (int k = 0; k < kJoinThreads / 32; k++) {
        if (k < (int)warp)
            inc += warp_sum[k];
        total += warp_sum[k];
    }
    inc -= sum;
#pragma unroll
    for (int k = 0; k < kEach; k++)
        upto[threadIdx.x * kEach + k] = inc += rows[k];
    __syncthreads();
    const bool few = total <= (int32_t)gridDim.x;   /* then a CTA takes a row */
    const int32_t warps = gridDim.x * (kJoinThreads / 32), each = few ? 1 : (total + warps - 1) / warps;
    int32_t u = few ? blockIdx.x : (blockIdx.x * (kJoinThreads / 32) + warp) * each;
    const int32_t end = min(total, u + each);
    while (u < end) {
        uint32_t lo = 0, hi = ctas - 1;         /* the job whose rows go past u */
        while (lo < hi) {
            const uint32_t mid = (lo + hi) / 2;
            if (upto[mid] > u)
                hi = mid;
            else
                lo = mid + 1;
        }
        const Job job = p.jobs[lo];
        const int32_t r0 = u - (upto[lo] - job.rows), r1 = min(job.rows, r0 + end - u);
        /* most have two pieces: then four rows together */
        if (few)
            join_row<T>(p, job, lo, r0, lane, warp);
        else if (job.ctas == 2)
            join_rows<T, 4, 2>(p, job, lo, r0, r1, lane);
        else
            join_rows<T, 1, 8>(p, job, lo, r0, r1, lane);
        u += r1 - r0;
    }
}

/* ---- launches ---- */
bool desc_ok(const kv_attn_desc *d)
{
    if (!d || !d->num_heads || !d->num_kv_heads || d->num_heads % d->num_kv_heads || d->num_heads > 65535 ||
        !d->head_dim || d->head_dim % 16 || d->head_dim > KVATTN_MAX_HEAD_DIM || !d->block_size || d->block_size > INT32_MAX ||
        !d->num_pages || d->num_pages > INT32_MAX || d->num_heads / d->num_kv_heads > kRows || !d->width || d->table_stride < (int64_t)d->width || !d->num_rows ||
        d->total_q > INT32_MAX || (d->q_type != KVATTN_BF16 && d->q_type != KVATTN_FP16) ||
        (d->kv_type != d->q_type && d->kv_type != KVATTN_E4M3) || d->device < 0 || d->device >= 64)
        return false;
    const uint64_t run = (uint64_t)d->block_size * d->num_kv_heads * d->head_dim * (d->kv_type == KVATTN_E4M3 ? 1 : 2);
    const float s = d->scale * d->k_scale;
    return run < (1ull << 40) && (!d->block_stride || (d->block_stride >= run && d->block_stride % 16 == 0)) &&
           std::isfinite(s) && s > 0 && d->scale > 0 && std::isfinite(d->v_scale);
}

/* CTAs of a call: all that the GPU holds at once */
int grid_of(const kv_attn_desc *d)
{
    static int sms[64];
    static std::once_flag once[64];
    std::call_once(once[d->device], [&] {
        int n = 0;
        if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, d->device) != cudaSuccess)
            cudaGetLastError();
        sms[d->device] = n > 0 ? (n < kMaxCtas / 2 ? n : kMaxCtas / 2) : 148;
    });
    return sms[d->device] * (d->head_dim <= 128 ? 2 : 1);
}

struct Work {
    uint64_t jobs, ml, o, bytes;
};

Work workspace(const kv_attn_desc *d)
{
    const uint64_t slots = 2ull * grid_of(d);
    auto up = [](uint64_t n) { return (n + 255) / 256 * 256; };
    Work w;
    w.jobs = 0;
    w.ml = up(slots / 2 * sizeof(Job));
    w.o = w.ml + up(slots * kRows * 2 * sizeof(float));
    w.bytes = w.o + slots * kRows * d->head_dim * sizeof(float);
    return w;
}

/* cuTensorMapEncodeTiled, from the driver that is loaded */
using Encode = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                            const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                            CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

Encode encoder()
{
    static Encode f;
    static std::once_flag once;
    std::call_once(once, [&] {
        void *at = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &at, cudaEnableDefault, &found) == cudaSuccess &&
            found == cudaDriverEntryPointSuccess)
            f = reinterpret_cast<Encode>(at);
    });
    return f;
}

bool encode_map(const Params &p, CUtensorMap *map, int rank, const void *base, const cuuint64_t *size, const cuuint64_t *stride,
                const cuuint32_t *box)
{
    const cuuint32_t step[4] = {1, 1, 1, 1};
    const Encode encode = encoder();
    return encode && encode(map, p.d.q_type == KVATTN_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                            rank, const_cast<void *>(base), size, stride, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

/* a plane as the TMA sees it, token-major or head-major alike */
bool plane_map(const Params &p, const void *plane, CUtensorMap *map)
{
    const kv_attn_desc &d = p.d;
    const uint64_t row = d.head_dim * 2ull;
    const cuuint64_t size[4] = {d.head_dim, d.block_size, d.num_kv_heads, d.num_pages};
    const cuuint64_t stride[3] = {row * (d.head_major ? 1 : d.num_kv_heads), row * (d.head_major ? d.block_size : 1), p.stride};
    const cuuint32_t box[4] = {kColumn, p.box, 1, 1};
    return encode_map(p, map, 4, plane, size, stride, box);
}

/* the rows of a tile, whole nodes, as one box */
bool query_map(const Params &p, CUtensorMap *map)
{
    const kv_attn_desc &d = p.d;
    const cuuint64_t size[3] = {d.head_dim, d.num_heads, d.total_q};
    const cuuint64_t stride[2] = {2ull * d.q_head_stride, 2ull * d.q_stride};
    const cuuint32_t box[3] = {kColumn, p.group, p.nodes.d};
    return encode_map(p, map, 3, d.q, size, stride, box);
}

template <typename T, Load L, int DP>
int launch(const Params &p, cudaStream_t stream)
{
    static std::once_flag once[64];
    static cudaError_t err[64];
    const int dev = p.d.device;
    std::call_once(once[dev], [&] {
        err[dev] = cudaFuncSetAttribute(kv_attn_kernel<T, L, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<L, DP>::kSmem);
        if (err[dev] != cudaSuccess)
            cudaGetLastError();
    });
    if (err[dev] != cudaSuccess)
        return -EIO;
    /* what a launch returns counts, not the thread's last error: that may be an
     * earlier call's, and without the second kernel the results would be parts */
    const unsigned grid = (unsigned)grid_of(&p.d);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(Roles<L>::kThreads);
    cfg.dynamicSmemBytes = Shape<L, DP>::kSmem;
    cfg.stream = stream;
    if (cudaLaunchKernelEx(&cfg, kv_attn_kernel<T, L, DP>, p) != cudaSuccess) {
        cudaGetLastError();
        return -EIO;
    }
    g_cc_kernel_launches.fetch_add(1, std::memory_order_relaxed);
    /* started while the first kernel drains; it waits for its results on the device */
    cudaLaunchAttribute attr[1];
    cfg.gridDim = dim3(2 * grid);
    cfg.blockDim = dim3(kJoinThreads);
    cfg.dynamicSmemBytes = 0;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, kv_attn_join_kernel<T>, p, grid) != cudaSuccess) {
        cudaGetLastError();
        return -EIO;
    }
    g_cc_kernel_launches.fetch_add(1, std::memory_order_relaxed);
    return 0;
}

template <typename T, Load L>
int launch_dim(const Params &p, cudaStream_t stream)
{
    if (p.d.head_dim <= 64)
        return launch<T, L, 64>(p, stream);
    if (p.d.head_dim <= 128)
        return launch<T, L, 128>(p, stream);
    return launch<T, L, 256>(p, stream);
}

template <typename T>
int launch_load(Params &p, cudaStream_t stream)
{
    if (!query_map(p, &p.q_map))
        return -EIO;
    if (p.d.kv_type == KVATTN_E4M3)
        return launch_dim<T, kWiden>(p, stream);
    const uint32_t bs = p.d.block_size;
    p.box = bs < (uint32_t)kTile ? bs : kTile;
    /* a tile is whole boxes of one page each, which start on the swizzle's eight rows */
    if (p.box % 8 || kTile % p.box || bs % p.box)
        return launch_dim<T, kCopy>(p, stream);
    if (!plane_map(p, p.d.k, &p.k_map) || !plane_map(p, p.d.v, &p.v_map))
        return -EIO;
    return launch_dim<T, kTma>(p, stream);
}

}  // namespace

extern "C" int64_t kv_attn_workspace_bytes(const struct kv_attn_desc *d)
{
    if (!desc_ok(d))
        return -EINVAL;
    return (int64_t)workspace(d).bytes;
}

static int attn_launch(const struct kv_attn_desc *d, uint32_t stall, void *stream)
{
    if (!desc_ok(d))
        return -EINVAL;
    if (d->num_seqs > KVATTN_MAX_SEQS || (uint64_t)d->total_q * d->num_heads > KVATTN_MAX_QUERIES)
        return -E2BIG;
    if (!d->num_seqs || !d->total_q)
        return 0;
    if (!d->q || !d->out || !d->k || !d->v || !d->table || !d->lens || !d->q_offsets || !d->error || !d->workspace ||
        ((uintptr_t)d->q | (uintptr_t)d->out | (uintptr_t)d->k | (uintptr_t)d->v) % 16 || (uintptr_t)d->workspace % 256 ||
        (d->q_stride | d->q_head_stride | d->out_stride | d->out_head_stride) % 8 || d->q_stride <= 0 || d->q_head_stride <= 0 ||
        d->out_stride <= 0 || d->out_head_stride <= 0)
        return -EINVAL;
    DeviceGuard on(d->device);
    if (!on.ok)
        return -EIO;
    const Work w = workspace(d);
    if (d->workspace_bytes < w.bytes)
        return -EINVAL;
    Params p{};
    p.d = *d;
    p.stall = stall;
    p.stride = d->block_stride ? d->block_stride
                               : (uint64_t)d->block_size * d->num_kv_heads * d->head_dim * (d->kv_type == KVATTN_E4M3 ? 1 : 2);
    p.group = d->num_heads / d->num_kv_heads;
    p.nodes = make_fastdiv(kRows / p.group);
    p.columns = (d->head_dim + kColumn - 1) / kColumn;
    p.block = make_fastdiv(d->block_size);
    /* a piece's sums, written and read, are 8 bytes a row and dimension against
     * 256 bytes a dimension of a 16-bit tile: a CTA takes enough tiles to be
     * worth that */
    const uint64_t mean = ((uint64_t)d->total_q * p.group + d->num_seqs - 1) / d->num_seqs;
    const uint32_t rows = (uint32_t)(mean < kRows ? mean : kRows);
    p.min_share = 1 + rows / 32;
    p.wide_out = (uintptr_t)d->out % 32 == 0 && (d->out_stride | d->out_head_stride) % 16 == 0;
    char *base = static_cast<char *>(d->workspace);
    p.jobs = reinterpret_cast<Job *>(base + w.jobs);
    p.part_ml = reinterpret_cast<float *>(base + w.ml);
    p.part_o = reinterpret_cast<float *>(base + w.o);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return d->q_type == KVATTN_BF16 ? launch_load<__nv_bfloat16>(p, st) : launch_load<__half>(p, st);
}

extern "C" int kv_attn_launch(const struct kv_attn_desc *d, void *stream) { return attn_launch(d, 0, stream); }

extern "C" int kv_attn_launch_stalled(const struct kv_attn_desc *d, void *stream) { return attn_launch(d, 1, stream); }
