/*
 * Attention over a paged KV cache for drafted trees, chains and single tokens
 * (include/kvattn.h), sm_100a.
 *
 * A K/V head of a sequence serves rows = nodes x (query heads per K/V head)
 * query rows, in tiles of 128.  Per 64 positions of the context a CTA computes
 *
 *   S = Q K^T        128 x 64, tcgen05.mma, Q and K in shared memory, S in TMEM
 *   P = exp2(S - m)  one thread per row, the running maximum and sum in 32 bits
 *   O += P V         128 x dim, tcgen05.mma, P in TMEM (where S was), V in shared
 *
 * Bound: with up to about 200 rows, reading K and V once from HBM; a tile of
 * 64 positions is 32 KiB at 16 bits and dim 128, about 1400 cycles of an SM's
 * share of the bandwidth, and its products take 524 cycles of the tensor cores
 * even with 128 rows of which one is a query.  So one form serves single
 * tokens and trees alike.  Two CTAs share an SM: one's softmax runs beside the
 * other's products.
 *
 * A CTA has 9 warps: 0-3 softmax (a thread owns a TMEM lane, a row), 4-7
 * loaders (pages of any size and order, 16 bytes at a time, straight into the
 * 128-byte swizzle that the products read; 8-bit caches are widened on the
 * way), 8 issues the products.  They meet at mbarriers: a ring of K and V
 * slots, two S buffers (S of the next tile is computed under this tile's
 * softmax), and O.  Every wait is bounded.
 *
 * The (sequence, K/V head, row tile, position tile) quadruples of a call lie on
 * one line, and each CTA takes an equal piece of it, wherever that ends inside a
 * context: ragged batches and a single long row fill the GPU alike, and the
 * lengths are read on the device.  Pieces of a row tile are joined by a second
 * kernel, in order, so results do not depend on timing.
 */
#include "kvattn.h"
#include "adaptor.h"
#include "device_guard.h"
#include "fastdiv.h"

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
constexpr int kSoftmax = 128;       /* threads of each role */
constexpr int kLoaders = 128;
constexpr int kThreads = kSoftmax + kLoaders + 32;
constexpr int kJoinThreads = 256;
constexpr int kJoinRows = 16;       /* rows of one joining CTA */
constexpr uint32_t kSpinLimit = 1u << 20;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

/* DP: head_dim rounded up to whole 128-byte columns (64 values) */
template <int DP> struct Shape {
    static constexpr int kCtas = DP <= 128 ? 2 : 1;                 /* per SM */
    static constexpr int kSlots = DP == 64 ? 8 : DP == 128 ? 5 : 4; /* K and V tiles in the ring */
    static constexpr int kSlotBytes = kTile * DP * 2;
    static constexpr int kQBytes = kRows * DP * 2;
    static constexpr int kTmem = DP <= 128 ? 256 : 512;             /* columns: 2 x 64 of S, then O */
    static constexpr int kSmem = kQBytes + kSlots * kSlotBytes + 1024;
    static_assert(kCtas * (kSmem + 1024) <= 228 * 1024, "the CTAs of an SM share its shared memory");
    static_assert(2 * kTile + DP <= kTmem && kCtas * kTmem <= 512, "and its TMEM");
};

/* a row tile that lies across CTAs: its first piece is the last of CTA c (in
 * that CTA's place `slot`), the others are the first of CTAs c + 1 .. */
struct Job {
    int32_t rows, ctas, slot, q0, h, row0;
};

struct Params {
    kv_attn_desc d;
    uint64_t stride;        /* bytes from page to page */
    FastDiv group;          /* query heads per K/V head */
    FastDiv block;          /* positions of a page */
    uint32_t min_share;     /* tiles that a CTA takes at least */
    struct Job *jobs;       /* workspace: [CTAs] row tiles to be joined, by the CTA that has their first tiles */
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

__device__ __forceinline__ int32_t row_tiles(const Seq &s, const FastDiv &group)
{
    return (int32_t)((s.nodes * group.d + kRows - 1) / kRows);
}

/* positions that row tile rt's nodes may see: parents come before their nodes */
__device__ __forceinline__ int32_t visible_end(const Seq &s, const FastDiv &group, int32_t rt)
{
    return s.ctx + min(s.nodes, (int32_t)fdiv((uint32_t)(rt + 1) * kRows - 1, group) + 1);
}

__device__ __forceinline__ int32_t tiles_of(const Seq &s, const FastDiv &group, int32_t rt)
{
    return (visible_end(s, group, rt) + kTile - 1) / kTile;
}

/* tiles of one K/V head of the sequence, all row tiles */
__device__ __forceinline__ uint64_t head_tiles(const Seq &s, const FastDiv &group)
{
    uint64_t n = 0;
    for (int32_t rt = 0; rt < row_tiles(s, group); rt++)
        n += tiles_of(s, group, rt);
    return n;
}

/* a run of tiles of one row tile */
struct Piece {
    Seq s;
    int32_t h, rt, t0, t1, n;       /* tiles t0 .. t1 of n */
    __device__ bool whole() const { return t0 == 0 && t1 == n; }
};

struct Line {
    int64_t x, hi, base;
    uint64_t per_head;
    uint32_t b;
    Seq s;                          /* sequence b, its tiles per K/V head, and the tiles before it */

    __device__ bool next(const Params &p, Piece &e)
    {
        if (x >= hi)
            return false;
        while (x >= base + (int64_t)(per_head * p.d.num_kv_heads)) {
            base += (int64_t)(per_head * p.d.num_kv_heads);
            b++;
            per_head = sequence(p.d, b, s) ? head_tiles(s, p.group) : 0;
        }
        uint64_t y = x - base;
        e.h = (int32_t)((y | per_head) >> 32 ? y / per_head : (uint32_t)y / (uint32_t)per_head);
        y -= e.h * per_head;
        e.rt = 0;
        for (e.n = tiles_of(s, p.group, 0); y >= (uint64_t)e.n; e.n = tiles_of(s, p.group, e.rt)) {
            y -= e.n;
            e.rt++;
        }
        e.s = s;
        e.t0 = (int32_t)y;
        e.t1 = (int32_t)min((int64_t)e.n, (int64_t)y + (hi - x));
        x += e.t1 - e.t0;
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

__device__ __forceinline__ bool mbar_try_wait(uint64_t *bar, uint32_t parity)
{
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\t"
                 "mbarrier.try_wait.parity.acquire.cta.shared::cta.b64 p, [%1], %2;\n\t"
                 "selp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
    return ok != 0;
}

struct Shared {
    uint64_t full[8], empty[8], s_full[2], p_full[2], o_done[2], o_free, q_full, q_empty;
    uint32_t tmem;
    volatile uint32_t dead;         /* a wait ran out: every role leaves */
    int64_t share, scan[kThreads / 32];
    Line line;                      /* the CTA's part of it */
    volatile uint32_t spoilt[16];   /* [piece % 16] == piece + 1: values of its fed nodes that are not finite were set aside */
};
static_assert(sizeof(Shared) <= 1024, "the last KiB of the dynamic shared memory");

/* Waits for the phase of `parity`, about a second at most.  A parity tells a
 * phase from the one before and the one after only.  Softmax does not wait for
 * every O: O is done at two barriers in turn, so that where it waits for one,
 * the one before at that barrier is known to be done (S of a tile is issued
 * behind O of the tile two before) and the one after is not yet issued. */
__device__ bool wait(Shared &sh, int32_t *error, uint64_t *bar, uint32_t parity)
{
    for (uint32_t i = 0;; i++) {
        if (mbar_try_wait(bar, parity))
            return true;
        if (sh.dead)
            return false;
        if (i >= kSpinLimit) {
            sh.dead = 1;
            atomicOr(error, KVATTN_ERR_TIMEOUT);
            return false;
        }
        if (i > 256)
            __nanosleep(64);
    }
}

/* the same for a whole warp, whose lanes go on together or not at all */
__device__ __forceinline__ bool wait_warp(Shared &sh, int32_t *error, uint64_t *bar, uint32_t parity)
{
    return __all_sync(~0u, wait(sh, error, bar, parity));
}

/* shared-memory matrix descriptor, 128-byte swizzle: the low word (where it
 * starts, and the bytes between 64-value columns of an operand stored row by
 * row) and the high word, which is the same for all here (1024 bytes from one
 * group of eight rows to the next) */
__device__ __forceinline__ uint32_t matrix(uint32_t addr, uint32_t lead)
{
    return (addr >> 4 & 0x3fff) | (lead >> 4 & 0x3fff) << 16;
}
constexpr uint32_t kMatrixHigh = 1024u >> 4 | 1u << 14 | 2u << 29;

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

__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t *a)
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
                 "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};"
                 ::W8(a, 0), W8(a, 8), W8(a, 16), W8(a, 24), "r"(addr) : "memory");
}

__device__ __forceinline__ float exp2_approx(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
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
    static __device__ uint32_t widen(uint16_t two)      /* two e4m3 values, exactly */
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
__device__ __forceinline__ void copy_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }
/* arrive at `bar` when this thread's copies so far have landed */
__device__ __forceinline__ void copy_arrive(uint64_t *bar)
{
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
/* what this thread has seen written to shared memory, before the products it issues */
__device__ __forceinline__ void fence_async_proxy() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

/* where chunk c (16 bytes) of row r stands in a tile of `rows` rows: 128-byte columns, swizzled */
__device__ __forceinline__ uint32_t swizzled(uint32_t rows, uint32_t r, uint32_t c)
{
    return (c >> 3) * rows * 128 + r * 128 + ((c ^ r) & 7) * 16;
}

/* ------------------------------------------------------------------------
 * loaders: slot 2 g is K of the CTA's tile g, slot 2 g + 1 its V; Q comes with
 * the first K of a piece.
 * ---------------------------------------------------------------------- */
template <typename T, bool F8, int DP> struct Loader {
    using S = Shape<DP>;
    static constexpr int kChunks = F8 ? DP / 16 : DP / 8;       /* 16-byte loads of a cached row */
    static constexpr int kPass = kLoaders / kChunks;            /* rows of one pass */
    static constexpr int kPasses = kTile / kPass;
    static constexpr int kWarpRows = kPass / (kLoaders / 32);   /* of them a warp's */
    static constexpr int kQChunks = DP / 8, kQPass = kLoaders / kQChunks;
    static_assert(kPasses * kWarpRows == 16, "a lane of each half warp looks after one of the warp's rows");

    const Params &p;
    Shared &sh;
    uint8_t *q_smem, *ring;
    uint32_t chunk, row;                /* this thread's chunk, and row of a pass */
    uint32_t own_row;                   /* the row of a tile whose place this lane works out */
    uint32_t tok_bytes;
    bool in_dim;
    uint64_t off[kPasses];              /* of this thread's rows in the planes, kNone: read as zeros */
    bool q_due = false;                 /* Q of the piece is still to be loaded */
    static constexpr uint64_t kNone = ~0ull;

    __device__ Loader(const Params &p_, Shared &sh_, uint8_t *q_, uint8_t *ring_) : p(p_), sh(sh_), q_smem(q_), ring(ring_)
    {
        const uint32_t t = threadIdx.x - kSoftmax, lane = t % 32, warp = t / 32;
        chunk = t % kChunks;
        row = t / kChunks;
        own_row = lane % 16 / kWarpRows * kPass + warp * kWarpRows + lane % kWarpRows;
        in_dim = chunk * (F8 ? 16 : 8) < p.d.head_dim;
        tok_bytes = (p.d.head_major ? 1 : p.d.num_kv_heads) * p.d.head_dim * (F8 ? 1 : 2);
    }

    /* the page of this lane's row of tile t: a load that waits for nothing */
    __device__ int32_t look_up(const Piece &e, int32_t t) const
    {
        const uint32_t pos = t * kTile + own_row;
        const int32_t *tab = p.d.table + (int64_t)e.s.row * p.d.table_stride;
        return (int32_t)pos < visible_end(e.s, p.group, e.rt) ? tab[fdiv(pos, p.block)] : -1;
    }

    /* The places of the thread's rows: each lane works out one, the threads of
     * a row take it from there. */
    __device__ void places(const Piece &e, int32_t t, int32_t page)
    {
        const kv_attn_desc &d = p.d;
        const uint32_t pos = t * kTile + own_row, j = pos - fdiv(pos, p.block) * p.block.d;
        const bool here = (int32_t)pos < visible_end(e.s, p.group, e.rt);
        uint64_t own = kNone;
        if (here) {
            if ((uint32_t)page < d.num_pages)
                own = (uint64_t)(uint32_t)page * p.stride + (uint64_t)j * tok_bytes +
                      (uint64_t)(d.head_major ? d.block_size : 1) * d.head_dim * (F8 ? 1 : 2) * e.h;
            else
                atomicOr(d.error, KVATTN_ERR_PAGE);
            if (d.parents && (int32_t)pos >= e.s.ctx && !node_ok(d.parents + e.s.q0, pos - e.s.ctx))
                own = kNone;            /* padding nodes are not read */
        }
        const uint32_t from = threadIdx.x % 32 / kChunks;
#pragma unroll
        for (int i = 0; i < kPasses; i++)
            off[i] = __shfl_sync(~0u, own, i * kWarpRows + from);
    }

    /* pass i's address in a plane (its start, for rows that are zeros) */
    __device__ const void *address(const void *plane, int i) const
    {
        return static_cast<const char *>(plane) + (off[i] == kNone ? 0 : off[i] + chunk * 16);
    }

    /* Q of the piece, once the products of the piece before have read theirs;
     * false if that is not yet so (or, with `block`, will not be) */
    __device__ bool load_q(const Piece &e, uint32_t piece, bool block)
    {
        if (piece) {
            const uint32_t parity = (piece - 1) & 1;
            if (!(block ? wait(sh, p.d.error, &sh.q_empty, parity) : mbar_try_wait(&sh.q_empty, parity)))
                return false;
        }
        const uint32_t t = threadIdx.x - kSoftmax, c = t % kQChunks;
        const int32_t rows = (int32_t)(e.s.nodes * p.group.d) - e.rt * kRows;
        if (c * 8 < p.d.head_dim)
            for (uint32_t r = t / kQChunks; r < kRows && (int32_t)r < rows; r += kQPass) {
                const uint32_t x = e.rt * kRows + r, node = fdiv(x, p.group), g = x - node * p.group.d;
                const T *src = static_cast<const T *>(p.d.q) + (int64_t)(e.s.q0 + node) * p.d.q_stride +
                               (int64_t)(e.h * p.group.d + g) * p.d.q_head_stride + c * 8;
                copy16(smem_u32(q_smem) + swizzled(kRows, r, c), src, true);
            }
        copy_arrive(&sh.q_full);
        q_due = false;
        return true;
    }

    /* slot i for writing; Q, if due, goes first where it need not be waited
     * for, or where the ring is full */
    __device__ bool acquire(uint32_t i, const Piece &e, uint32_t piece)
    {
        uint64_t *bar = &sh.empty[i % S::kSlots];
        const uint32_t parity = ((i / S::kSlots) & 1) ^ 1;
        bool ok = true;
        if (q_due && !load_q(e, piece, false) && !mbar_try_wait(bar, parity))
            ok = load_q(e, piece, true);
        return __all_sync(~0u, ok && wait(sh, p.d.error, bar, parity));
    }

    __device__ uint8_t *slot(uint32_t i) const { return ring + (i % S::kSlots) * S::kSlotBytes; }

    /* 16-bit caches: asynchronous copies, the ring's depth in flight */
    __device__ void run16(Line line)
    {
        uint32_t i = 0, piece = 0;
        Piece e;
        for (; line.next(p, e); piece++) {
            q_due = true;
            int32_t page = look_up(e, e.t0);
            for (int32_t t = e.t0; t < e.t1; t++) {
                places(e, t, page);
                if (t + 1 < e.t1)
                    page = look_up(e, t + 1);       /* in flight while the tile is copied */
                for (int v = 0; v < 2; v++, i++) {
                    if (!acquire(i, e, piece))
                        return;
                    const void *plane = v ? p.d.v : p.d.k;
                    const uint32_t to = smem_u32(slot(i));
                    if (in_dim)
#pragma unroll
                        for (int x = 0; x < kPasses; x++)
                            copy16(to + swizzled(kTile, row + x * kPass, chunk), address(plane, x), off[x] != kNone);
                    copy_arrive(&sh.full[i % S::kSlots]);
                }
            }
            if (!__all_sync(~0u, !q_due || load_q(e, piece, true)))
                return;
        }
    }

    /* 8-bit caches: through registers, one tile ahead */
    __device__ void fetch(uint4 *k, uint4 *v)
    {
#pragma unroll
        for (int x = 0; x < kPasses; x++) {
            k[x] = v[x] = make_uint4(0, 0, 0, 0);
            if (in_dim && off[x] != kNone) {
                k[x] = __ldg(static_cast<const uint4 *>(address(p.d.k, x)));
                v[x] = __ldg(static_cast<const uint4 *>(address(p.d.v, x)));
            }
        }
    }

    __device__ void put(uint32_t i, const uint4 *raw)
    {
        if (in_dim)
#pragma unroll
            for (int x = 0; x < kPasses; x++) {
                const uint32_t *w = reinterpret_cast<const uint32_t *>(&raw[x]);
                uint32_t o[8];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    o[2 * k] = Type<T>::widen((uint16_t)w[k]);
                    o[2 * k + 1] = Type<T>::widen((uint16_t)(w[k] >> 16));
                }
                uint8_t *to = slot(i);
                *reinterpret_cast<uint4 *>(to + swizzled(kTile, row + x * kPass, 2 * chunk)) = make_uint4(o[0], o[1], o[2], o[3]);
                *reinterpret_cast<uint4 *>(to + swizzled(kTile, row + x * kPass, 2 * chunk + 1)) = make_uint4(o[4], o[5], o[6], o[7]);
            }
        mbar_arrive(&sh.full[i % S::kSlots]);
    }

    __device__ void run8(Line line)
    {
        Piece now, then;
        uint4 k[kPasses], v[kPasses], k2[kPasses], v2[kPasses];
        if (!line.next(p, now))
            return;
        int32_t t = now.t0, page = look_up(now, t);
        places(now, t, page);
        if (t + 1 < now.t1)
            page = look_up(now, t + 1);
        fetch(k, v);
        uint32_t piece = 0, i = 0;
        q_due = true;
        for (bool more = true; more;) {
            const bool last = t + 1 >= now.t1;
            bool moved = false;
            if (last)
                more = moved = line.next(p, then);
            if (more) {
                const Piece &e = moved ? then : now;
                const int32_t u = moved ? then.t0 : t + 1;
                if (moved)
                    page = look_up(e, u);
                places(e, u, page);
                if (u + 1 < e.t1)
                    page = look_up(e, u + 1);
                fetch(k2, v2);
            }
            if (!acquire(i, now, piece))
                return;
            put(i++, k);
            if (!acquire(i, now, piece))
                return;
            put(i++, v);
            if (!__all_sync(~0u, !last || !q_due || load_q(now, piece, true)))
                return;
#pragma unroll
            for (int x = 0; x < kPasses; x++) {
                k[x] = k2[x];
                v[x] = v2[x];
            }
            if (moved) {
                now = then;
                t = now.t0;
                piece++;
                q_due = true;
            } else {
                t++;
            }
        }
    }
};

/* ------------------------------------------------------------------------
 * products: S of tile g + 1 is issued before O += P V of tile g, so that it is
 * computed under the softmax of g.  Products of one CTA run in the order they
 * were issued, so S may overwrite a buffer whose P an earlier product reads.
 * ---------------------------------------------------------------------- */
template <typename T, int DP>
__device__ void products(const Params &p, Shared &sh, uint8_t *q_smem, uint8_t *ring, Line line)
{
    using S = Shape<DP>;
    const uint32_t dim = p.d.head_dim, tmem = sh.tmem, o = tmem + 2 * kTile;
    const uint32_t inst_s = instruction(Type<T>::kBf16, kTile, 0), inst_o = instruction(Type<T>::kBf16, dim, 1);
    /* one thread issues: descriptors are a constant per step on top of the slot's */
    const uint32_t q0 = matrix(smem_u32(q_smem), 16), k0 = matrix(smem_u32(ring), 16), v0 = matrix(smem_u32(ring), kTile * 128);
    uint32_t g = 0, piece = 0, slot = 0, lap = 0;       /* the slot of K of the next S, and the ring's lap */
    Piece e;
    auto scores = [&](uint32_t tile) {
        if (!wait(sh, p.d.error, &sh.full[slot], lap & 1))
            return false;
        fence_async_proxy();
        tmem_fence_after();
        const uint32_t k = k0 + slot * (S::kSlotBytes >> 4);
        const uint32_t s = tmem + (tile & 1) * kTile;
#pragma unroll
        for (uint32_t x = 0; x < DP / 16; x++)
            if (x * 16 < dim)
                mma_ss(s, q0 + ((x >> 2) * (kRows * 128) + (x & 3) * 32 >> 4), k + ((x >> 2) * (kTile * 128) + (x & 3) * 32 >> 4),
                       inst_s, x > 0);
        mma_commit(&sh.empty[slot]);
        mma_commit(&sh.s_full[tile & 1]);
        slot += 2;
        if (slot >= S::kSlots) {
            slot -= S::kSlots;
            lap++;
        }
        return true;
    };
    uint32_t v_slot = 1, v_lap = 0;
    while (line.next(p, e)) {
        const uint32_t n = e.t1 - e.t0;
        if (!wait(sh, p.d.error, &sh.q_full, piece & 1) || !scores(g))
            return;
        if (n == 1)
            mma_commit(&sh.q_empty);
        for (uint32_t k = 0; k < n; k++, g++) {
            if (k + 1 < n) {
                if (!scores(g + 1))
                    return;
                if (k + 2 == n)
                    mma_commit(&sh.q_empty);    /* every S of the piece is issued */
            }
            if (k == 0 && piece && !wait(sh, p.d.error, &sh.o_free, (piece - 1) & 1))
                return;
            if (!wait(sh, p.d.error, &sh.p_full[g & 1], (g >> 1) & 1) ||
                !wait(sh, p.d.error, &sh.full[v_slot], v_lap & 1))
                return;
            fence_async_proxy();
            tmem_fence_after();
            const uint32_t v = v0 + v_slot * (S::kSlotBytes >> 4);
#pragma unroll
            for (uint32_t x = 0; x < kTile / 16; x++)
                mma_ts(o, tmem + (g & 1) * kTile + x * 8, v + (x * 2048 >> 4), inst_o, k > 0 || x > 0);
            mma_commit(&sh.empty[v_slot]);
            mma_commit(&sh.o_done[g & 1]);
            v_slot += 2;
            if (v_slot >= S::kSlots) {
                v_slot -= S::kSlots;
                v_lap++;
            }
        }
        piece++;
    }
}

/* ------------------------------------------------------------------------
 * softmax: thread = row.  m lags behind the true maximum by up to kLazy (in
 * powers of two), so that O, which lives in TMEM, is rescaled rarely; the
 * result is the same quotient.
 * ---------------------------------------------------------------------- */
/* the positions of tile t that node j sees, a bit each */
__device__ uint64_t seen(const Params &p, const Piece &e, int32_t j, int32_t t)
{
    const int32_t p0 = t * kTile, before = e.s.ctx - p0;
    uint64_t bits = before >= 64 ? ~0ull : before > 0 ? (1ull << before) - 1 : 0;
    if (!p.d.parents) {
        const int32_t upto = before + j + 1;
        return upto >= 64 ? ~0ull : upto > 0 ? (1ull << upto) - 1 : 0;
    }
    const int32_t *par = p.d.parents + e.s.q0;
    for (int32_t a = j; before + a >= 0;) {
        if (before + a < 64)
            bits |= 1ull << (before + a);
        const int32_t u = par[a];
        if (u < 0 || !node_ok(par, u))
            break;
        a = u;
    }
    return bits;
}

/* what was set aside of the values that node j sees in tiles t0 .. t1, dims d0 .. d0 + 16 */
template <typename T, bool F8>
__device__ __noinline__ void add_spoilt(const Params &p, const Piece &e, int32_t j, uint32_t d0, float *o)
{
    const kv_attn_desc &d = p.d;
    const int32_t *par = d.parents ? d.parents + e.s.q0 : nullptr;
    const int32_t *tab = d.table + (int64_t)e.s.row * d.table_stride;
    for (int32_t a = j; a >= 0;) {
        const int32_t pos = e.s.ctx + a;
        if (pos < e.t0 * kTile)
            break;
        const int32_t page = tab[pos / (int32_t)d.block_size];
        if (pos < e.t1 * kTile && page >= 0 && (uint32_t)page < d.num_pages) {
            const uint64_t at = (uint64_t)page * p.stride +
                                ((uint64_t)(pos % (int32_t)d.block_size) * (d.head_major ? 1 : d.num_kv_heads) * d.head_dim +
                                 (uint64_t)(d.head_major ? d.block_size : 1) * d.head_dim * e.h + d0) * (F8 ? 1 : 2);
            for (int x = 0; x < 16; x++) {
                uint32_t w;
                if (F8)
                    w = Type<T>::widen(static_cast<const uint8_t *>(d.v)[at + x]);
                else
                    w = *reinterpret_cast<const uint16_t *>(static_cast<const uint8_t *>(d.v) + at + 2 * x);
                if (!Type<T>::finite(w))
                    o[x] += Type<T>::value(w & 0xffff);
            }
        }
        const int32_t u = par ? par[a] : a - 1;
        if (u < 0 || (par && !node_ok(par, u)))
            break;
        a = u;
    }
}

/* A fed node's value that is not finite would reach the rows that do not see
 * it, as 0 * value: the softmax threads set such values of a tile with fed
 * nodes to 0 before it is used, and add them to the rows that do see them. */
template <typename T, int DP>
__device__ bool set_aside(uint8_t *tile, uint32_t dim)
{
    bool any = false;
    for (uint32_t x = threadIdx.x; x < kTile * DP / 8; x += kSoftmax) {
        if (x / (kTile * 8) * 8 + ((x ^ x >> 3) & 7) >= dim / 8)
            continue;                   /* behind the head's dimensions */
        uint4 v = *reinterpret_cast<uint4 *>(tile + x * 16);
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
            *reinterpret_cast<uint4 *>(tile + x * 16) = v;
            any = true;
        }
    }
    return any;
}

template <typename T, bool F8, int DP>
__device__ void softmax(const Params &p, Shared &sh, uint8_t *ring, Line line)
{
    using S = Shape<DP>;
    const kv_attn_desc &d = p.d;
    const uint32_t tid = threadIdx.x, lanes = (tid / 32 * 32) << 16;
    const uint32_t tmem = sh.tmem + lanes, o_at = tmem + 2 * kTile;
    const float s2 = d.scale * d.k_scale * kLog2e;
    uint32_t g = 0, piece = 0;
    Piece e;
    for (; line.next(p, e); piece++) {
        const uint32_t x = e.rt * kRows + tid;
        const bool valid = x < e.s.nodes * p.group.d;
        const int32_t node = valid ? (int32_t)fdiv(x, p.group) : 0, sub = valid ? (int32_t)(x - node * p.group.d) : 0;
        bool active = valid;
        if (valid && d.parents && !node_ok(d.parents + e.s.q0, node)) {
            active = false;
            if (d.parents[e.s.q0 + node] != -2)
                atomicOr(d.error, KVATTN_ERR_PARENT);
        }
        const bool work = __any_sync(~0u, active);
        float m = -INFINITY, l = 0;
        for (int32_t t = e.t0; t < e.t1; t++, g++) {
            const uint32_t s_at = tmem + (g & 1) * kTile;
            if (!wait_warp(sh, d.error, &sh.s_full[g & 1], (g >> 1) & 1))
                return;
            if (work) {
                uint32_t raw[kTile];
                float *s = reinterpret_cast<float *>(raw);
                tmem_fence_after();
                tmem_ld64(s_at, raw);
                if ((t + 1) * kTile > e.s.ctx) {
                    const uint64_t bits = active ? seen(p, e, node, t) : 0;
#pragma unroll
                    for (int c = 0; c < kTile; c++)
                        s[c] = bits >> c & 1 ? s[c] : -INFINITY;
                }
                float top[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
                for (int c = 4; c < kTile; c++)
                    top[c & 3] = fmaxf(top[c & 3], s[c]);
                const float now = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * s2;
                const bool raise = active && now > m + Type<T>::kLazy;
                if (t == e.t0) {
                    m = now;
                } else if (__any_sync(~0u, raise)) {
                    const float f = raise ? exp2_approx(m - now) : 1.f;
                    if (raise)
                        m = now;
                    l *= f;
                    if (!wait_warp(sh, d.error, &sh.o_done[(g - 1) & 1], ((g - 1) >> 1) & 1))
                        return;
                    tmem_fence_after();
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
                float sum[4] = {};
                uint32_t w[kTile / 2];
#pragma unroll
                for (int c = 0; c < kTile; c += 2) {
                    const float a = exp2_approx(fmaf(s[c], s2, -from)), b = exp2_approx(fmaf(s[c + 1], s2, -from));
                    sum[c & 2] += a;
                    sum[(c & 2) + 1] += b;
                    w[c / 2] = Type<T>::pack(a, b);
                }
                l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                tmem_st32(s_at, w);
                tmem_wait_st();
                tmem_fence_before();
            }
            if ((t + 1) * kTile > e.s.ctx) {
                const uint32_t i = 2 * g + 1, slot = i % S::kSlots;
                if (!wait_warp(sh, d.error, &sh.full[slot], (i / S::kSlots) & 1))
                    return;
                if (set_aside<T, DP>(ring + slot * S::kSlotBytes, d.head_dim))
                    sh.spoilt[piece % 16] = piece + 1;
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
        const float inv = !active ? 0.f : whole ? d.v_scale / l : 1.f;
        T *out = static_cast<T *>(d.out) + (int64_t)(e.s.q0 + node) * d.out_stride + (int64_t)(e.h * p.group.d + sub) * d.out_head_stride;
        float *part = p.part_o + ((uint64_t)slot * kRows + tid) * d.head_dim;
        const bool spoilt = sh.spoilt[piece % 16] == piece + 1;
        if (__any_sync(~0u, valid)) {
            for (uint32_t c = 0; c < d.head_dim; c += 16) {
                uint32_t raw[16];
                float *o = reinterpret_cast<float *>(raw);
                tmem_ld16(o_at + c, raw);
                if (spoilt && active)
                    add_spoilt<T, F8>(p, e, node, c, o);
                if (!active)
#pragma unroll
                    for (int k = 0; k < 16; k++)
                        o[k] = 0.f;
                if (whole && valid) {
                    uint4 v[2];
                    uint32_t *w = reinterpret_cast<uint32_t *>(v);
#pragma unroll
                    for (int k = 0; k < 8; k++)
                        w[k] = Type<T>::pack(o[2 * k] * inv, o[2 * k + 1] * inv);
                    *reinterpret_cast<uint4 *>(out + c) = v[0];
                    *reinterpret_cast<uint4 *>(out + c + 8) = v[1];
                } else if (active) {
#pragma unroll
                    for (int k = 0; k < 4; k++)
                        *reinterpret_cast<float4 *>(part + c + 4 * k) = make_float4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
                }
            }
            if (tid == 0 && e.t0 == 0 && !whole)
                p.jobs[blockIdx.x] = {min(kRows, (int32_t)(e.s.nodes * p.group.d) - e.rt * kRows),
                                      (int32_t)(1 + (e.n - e.t1 + sh.share - 1) / sh.share), (int32_t)slot, e.s.q0, e.h, e.rt * kRows};
            if (valid) {
                if (!whole) {
                    float *ml = p.part_ml + ((uint64_t)slot * kRows + tid) * 2;
                    ml[0] = active ? from : -INFINITY;
                    ml[1] = active ? l : 0.f;
                } else if (d.lse) {
                    d.lse[(int64_t)(e.s.q0 + node) * d.num_heads + e.h * p.group.d + sub] =
                        active ? (from + log2f(l)) * kLn2 : -INFINITY;
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

template <typename T>
__device__ void void_rows(const Params &p, const Seq &s)
{
    const kv_attn_desc &d = p.d;
    for (int64_t x = 0; x < (int64_t)s.nodes * d.num_heads; x++) {
        const int64_t i = s.q0 + x / d.num_heads, h = x % d.num_heads;
        T *out = static_cast<T *>(d.out) + i * d.out_stride + h * d.out_head_stride;
        for (uint32_t c = 0; c < d.head_dim; c += 8)
            *reinterpret_cast<uint4 *>(out + c) = make_uint4(0, 0, 0, 0);
        if (d.lse)
            d.lse[i * d.num_heads + h] = -INFINITY;
    }
}

/* Counts the tiles of all sequences, kThreads at a time; the CTA's share of
 * the line, and the sequence that it begins in, go to sh.line.  With more than
 * kThreads sequences the search is a second walk. */
template <typename T>
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
            if (b < d.num_seqs) {
                if (sequence(d, b, s)) {
                    n = head_tiles(s, p.group);
                } else if (walk == 0 && blockIdx.x == b % gridDim.x) {
                    atomicOr(d.error, KVATTN_ERR_SEQ);
                    void_rows<T>(p, s);
                }
            }
            const int64_t all = (int64_t)(n * d.num_kv_heads), upto = before + block_scan(sh, all, sum);
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

template <typename T, bool F8, int DP>
__global__ void __launch_bounds__(kThreads, Shape<DP>::kCtas) kv_attn_kernel(const __grid_constant__ Params p)
{
    using S = Shape<DP>;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t *q_smem = smem, *ring = smem + S::kQBytes;
    Shared &sh = *reinterpret_cast<Shared *>(smem + S::kQBytes + S::kSlots * S::kSlotBytes);
    const uint32_t warp = threadIdx.x >> 5;

    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (threadIdx.x == 0) {
        for (int k = 0; k < S::kSlots; k++) {
            mbar_init(&sh.full[k], kLoaders);
            mbar_init(&sh.empty[k], 1);
        }
        for (int k = 0; k < 2; k++) {
            mbar_init(&sh.s_full[k], 1);
            mbar_init(&sh.o_done[k], 1);
            mbar_init(&sh.p_full[k], kSoftmax / 32);
        }
        mbar_init(&sh.o_free, kSoftmax / 32);
        mbar_init(&sh.q_full, kLoaders);
        mbar_init(&sh.q_empty, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        sh.dead = 0;
        for (int k = 0; k < 16; k++)
            sh.spoilt[k] = 0;
    }
    find_line<T>(p, sh);
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
    const Line line = sh.line;
    if (smem_u32(smem) % 1024 == 0) {
        if (warp < kSoftmax / 32) {
            softmax<T, F8, DP>(p, sh, ring, line);
        } else if (warp < (kSoftmax + kLoaders) / 32) {
            Loader<T, F8, DP> load(p, sh, q_smem, ring);
            if constexpr (F8)
                load.run8(line);
            else
                load.run16(line);
            copy_wait_all();
        } else {
            if ((threadIdx.x & 31) == 0)
                products<T, DP>(p, sh, q_smem, ring, line);
            __syncwarp();
        }
    } else if (threadIdx.x == 0) {
        atomicOr(p.d.error, KVATTN_ERR_TIMEOUT);
    }
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    if (warp == kThreads / 32 - 1)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(sh.tmem), "n"(S::kTmem) : "memory");
}

/* ------------------------------------------------------------------------
 * join: the pieces of a row tile that lies across CTAs, in their order.
 * ---------------------------------------------------------------------- */
template <typename T>
__global__ void __launch_bounds__(kJoinThreads) kv_attn_join_kernel(const __grid_constant__ Params p)
{
    const kv_attn_desc &d = p.d;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const Job job = p.jobs[blockIdx.x];
    const int32_t r0 = blockIdx.y * kJoinRows;
    if (r0 >= job.rows)
        return;
    const uint32_t quads = d.head_dim / 4;
    for (uint32_t x = threadIdx.x; x < kJoinRows * quads; x += kJoinThreads) {
        const int32_t r = r0 + (int32_t)(x / quads);
        const uint32_t c = x % quads * 4;
        if (r >= job.rows)
            return;
        /* piece k's row: the first piece's slot, then slot 0 of the CTAs behind */
        auto at = [&](int32_t k) { return (uint64_t)(k ? 2 * (blockIdx.x + k) : (uint32_t)job.slot) * kRows + r; };
        float m = -INFINITY, l = 0;
#pragma unroll 4
        for (int32_t k = 0; k < job.ctas; k++) {
            const float2 ml = *reinterpret_cast<const float2 *>(p.part_ml + at(k) * 2);
            m = fmaxf(m, ml.y == 0 ? -INFINITY : ml.x);
        }
        float4 o = make_float4(0, 0, 0, 0);
#pragma unroll 4
        for (int32_t k = 0; k < job.ctas; k++) {
            const float2 ml = *reinterpret_cast<const float2 *>(p.part_ml + at(k) * 2);
            if (ml.y == 0)
                continue;               /* sees nothing there: its sums were not written */
            const float f = exp2f(ml.x - m);
            const float4 v = *reinterpret_cast<const float4 *>(p.part_o + at(k) * d.head_dim + c);
            l += f * ml.y;
            o.x += f * v.x;
            o.y += f * v.y;
            o.z += f * v.z;
            o.w += f * v.w;
        }
        const uint32_t q = job.row0 + r;
        const int32_t node = (int32_t)fdiv(q, p.group), sub = (int32_t)(q - node * p.group.d);
        const float inv = l == 0 ? 0.f : d.v_scale / l;
        T *out = static_cast<T *>(d.out) + (int64_t)(job.q0 + node) * d.out_stride + (int64_t)(job.h * p.group.d + sub) * d.out_head_stride;
        *reinterpret_cast<uint2 *>(out + c) = make_uint2(Type<T>::pack(o.x * inv, o.y * inv), Type<T>::pack(o.z * inv, o.w * inv));
        if (c == 0 && d.lse)
            d.lse[(int64_t)(job.q0 + node) * d.num_heads + job.h * p.group.d + sub] = l == 0 ? -INFINITY : (m + log2f(l)) * kLn2;
    }
}

/* ---- launches ---- */
bool desc_ok(const kv_attn_desc *d)
{
    if (!d || !d->num_heads || !d->num_kv_heads || d->num_heads % d->num_kv_heads || d->num_heads > 65535 ||
        !d->head_dim || d->head_dim % 16 || d->head_dim > KVATTN_MAX_HEAD_DIM || !d->block_size || d->block_size > INT32_MAX ||
        !d->num_pages || d->num_pages > INT32_MAX || !d->width || d->table_stride < (int64_t)d->width || !d->num_rows ||
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
        sms[d->device] = n > 0 ? n : 148;
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

template <typename T, bool F8, int DP>
int launch(const Params &p, cudaStream_t stream)
{
    static std::once_flag once[64];
    static cudaError_t err[64];
    const int dev = p.d.device;
    std::call_once(once[dev], [&] {
        err[dev] = cudaFuncSetAttribute(kv_attn_kernel<T, F8, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<DP>::kSmem);
        if (err[dev] != cudaSuccess)
            cudaGetLastError();
    });
    if (err[dev] != cudaSuccess)
        return -EIO;
    const unsigned grid = (unsigned)grid_of(&p.d);
    kv_attn_kernel<T, F8, DP><<<grid, kThreads, Shape<DP>::kSmem, stream>>>(p);
    g_cc_kernel_launches.fetch_add(1, std::memory_order_relaxed);
    if (cudaPeekAtLastError() != cudaSuccess)
        return -EIO;
    /* started while the first kernel drains; it waits for its results on the device */
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr[1];
    cfg.gridDim = dim3(grid, kRows / kJoinRows);
    cfg.blockDim = dim3(kJoinThreads);
    cfg.stream = stream;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, kv_attn_join_kernel<T>, p) != cudaSuccess) {
        cudaGetLastError();
        return -EIO;
    }
    g_cc_kernel_launches.fetch_add(1, std::memory_order_relaxed);
    return 0;
}

template <typename T, bool F8>
int launch_dim(const Params &p, cudaStream_t stream)
{
    if (p.d.head_dim <= 64)
        return launch<T, F8, 64>(p, stream);
    if (p.d.head_dim <= 128)
        return launch<T, F8, 128>(p, stream);
    return launch<T, F8, 256>(p, stream);
}

}  // namespace

extern "C" int64_t kv_attn_workspace_bytes(const struct kv_attn_desc *d)
{
    if (!desc_ok(d))
        return -EINVAL;
    return (int64_t)workspace(d).bytes;
}

extern "C" int kv_attn_launch(const struct kv_attn_desc *d, void *stream)
{
    if (!desc_ok(d))
        return -EINVAL;
    if (d->num_seqs > KVATTN_MAX_SEQS || (uint64_t)d->total_q * d->num_heads > KVATTN_MAX_QUERIES)
        return -E2BIG;
    if (!d->num_seqs || !d->total_q)
        return 0;
    if (!d->q || !d->out || !d->k || !d->v || !d->table || !d->lens || !d->q_offsets || !d->error || !d->workspace ||
        ((uintptr_t)d->q | (uintptr_t)d->out | (uintptr_t)d->k | (uintptr_t)d->v) % 16 || (uintptr_t)d->workspace % 256 ||
        (d->q_stride | d->q_head_stride | d->out_stride | d->out_head_stride) % 8)
        return -EINVAL;
    DeviceGuard on(d->device);
    if (!on.ok)
        return -EIO;
    const Work w = workspace(d);
    if (d->workspace_bytes < w.bytes)
        return -EINVAL;
    Params p{};
    p.d = *d;
    p.stride = d->block_stride ? d->block_stride
                               : (uint64_t)d->block_size * d->num_kv_heads * d->head_dim * (d->kv_type == KVATTN_E4M3 ? 1 : 2);
    p.group = make_fastdiv(d->num_heads / d->num_kv_heads);
    p.block = make_fastdiv(d->block_size);
    /* a piece's sums, written and read, are 8 bytes a row and dimension against
     * 256 bytes a dimension of a 16-bit tile: a CTA takes enough tiles to be
     * worth that */
    const uint64_t rows = (uint64_t)d->total_q * p.group.d / d->num_seqs;
    p.min_share = 1 + (uint32_t)((rows < kRows ? rows : kRows) / 32);
    char *base = static_cast<char *>(d->workspace);
    p.jobs = reinterpret_cast<Job *>(base + w.jobs);
    p.part_ml = reinterpret_cast<float *>(base + w.ml);
    p.part_o = reinterpret_cast<float *>(base + w.o);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool e4m3 = d->kv_type == KVATTN_E4M3;
    if (d->q_type == KVATTN_BF16)
        return e4m3 ? launch_dim<__nv_bfloat16, true>(p, st) : launch_dim<__nv_bfloat16, false>(p, st);
    return e4m3 ? launch_dim<__half, true>(p, st) : launch_dim<__half, false>(p, st);
}
