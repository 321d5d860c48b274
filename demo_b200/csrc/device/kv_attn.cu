/*
 * Attention over a paged KV cache for drafted trees, chains and single tokens
 * (include/kvattn.h), sm_100a.
 *
 * One warp per (node, head): a lane scores one of 32 positions at a time, then
 * the lanes share the value rows by dimension.  One pass with the running
 * maximum and sum of the softmax, all in 32 bits.
 */
#include "kvattn.h"
#include "adaptor.h"
#include "device_guard.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <cerrno>
#include <cmath>
#include <cstdint>

namespace {

constexpr int kWarps = 4;

struct Seq {
    int32_t q0, nodes, ctx, row;
};

/* sequence b's nodes and context; false (and an error bit) if they do not fit */
__device__ bool sequence(const kv_attn_desc &d, uint32_t b, Seq &s)
{
    const int32_t o0 = d.q_offsets[b], o1 = d.q_offsets[b + 1];
    const int32_t r = d.rows ? d.rows[b] : (int32_t)b;
    if (o0 < 0 || o1 < o0 || (uint32_t)o1 > d.total_q || r < 0 || (uint32_t)r >= d.num_rows)
        return false;
    const int32_t len = d.lens[r];
    s = {o0, o1 - o0, len - (o1 - o0), r};
    return s.ctx >= 0 && (uint64_t)len <= (uint64_t)d.width * d.block_size;
}

template <typename T> __device__ __forceinline__ float to_float(T x) { return static_cast<float>(x); }

template <typename T, typename KV>
__global__ void __launch_bounds__(32 * kWarps) kv_attn_simple_kernel(const kv_attn_desc d, uint64_t stride)
{
    extern __shared__ float qs[];
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t i = blockIdx.x, h = blockIdx.y * kWarps + warp, D = d.head_dim;
    if (h >= d.num_heads)
        return;
    /* the sequence of query i: the last one that starts at or before it */
    uint32_t lo = 0, hi = d.num_seqs;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if ((uint32_t)d.q_offsets[mid] <= i)
            lo = mid;
        else
            hi = mid;
    }
    Seq s;
    const bool fits = sequence(d, lo, s);
    if ((int32_t)i < d.q_offsets[lo] || (int32_t)i >= d.q_offsets[lo + 1])
        return;
    const int32_t node = (int32_t)i - s.q0;
    T *out = static_cast<T *>(d.out) + (int64_t)i * d.out_stride + (int64_t)h * d.out_head_stride;
    bool sees = fits;
    if (!fits && lane == 0)
        atomicOr(d.error, KVATTN_ERR_SEQ);
    const int32_t *par = d.parents ? d.parents + s.q0 : nullptr;
    if (fits && par && (par[node] < -1 || par[node] >= node)) {
        sees = false;
        if (par[node] != -2 && lane == 0)
            atomicOr(d.error, KVATTN_ERR_PARENT);
    }
    float *q = qs + warp * D;
    const T *qg = static_cast<const T *>(d.q) + (int64_t)i * d.q_stride + (int64_t)h * d.q_head_stride;
    for (uint32_t x = lane; x < D; x += 32)
        q[x] = to_float(qg[x]);
    __syncwarp();
    const uint32_t kvh = h / (d.num_heads / d.num_kv_heads);
    const uint64_t tok = (d.head_major ? 1 : d.num_kv_heads) * (uint64_t)D, head = (d.head_major ? d.block_size : 1) * (uint64_t)D * kvh;
    const float scale = d.scale * d.k_scale;
    float m = -INFINITY, l = 0, acc[KVATTN_MAX_HEAD_DIM / 32] = {};
    const int32_t end = sees ? s.ctx + node + 1 : 0;
    for (int32_t p1 = end; p1 > 0; p1 -= 32) {
        const int32_t p = p1 - 1 - (int32_t)lane;
        bool on = p >= 0;
        if (on && p >= s.ctx && par) {
            int32_t a = node;
            while (a > p - s.ctx) {
                const int32_t u = par[a];
                a = u < -1 || u >= a || (u >= 0 && (par[u] < -1 || par[u] >= u)) ? -1 : u;
            }
            on = a == p - s.ctx;
        }
        const KV *k = nullptr, *v = nullptr;
        if (on) {
            const int32_t page = d.table[(int64_t)s.row * d.table_stride + p / (int32_t)d.block_size];
            if (page < 0 || (uint32_t)page >= d.num_pages) {
                atomicOr(d.error, KVATTN_ERR_PAGE);
            } else {
                const uint64_t off = page * stride + ((uint64_t)(p % (int32_t)d.block_size) * tok + head) * sizeof(KV);
                k = reinterpret_cast<const KV *>(static_cast<const char *>(d.k) + off);
                v = reinterpret_cast<const KV *>(static_cast<const char *>(d.v) + off);
            }
        }
        float x = 0;
        if (k)
            for (uint32_t e = 0; e < D; e++)
                x = fmaf(q[e], to_float(k[e]), x);
        x = on ? x * scale : -INFINITY;
        float top = x;
        for (int o = 16; o; o >>= 1)
            top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
        const float mn = fmaxf(m, top), keep = mn == -INFINITY ? 1.f : expf(m - mn);
        const float w = on ? expf(x - mn) : 0.f;
        m = mn;
        l = l * keep + w;
        for (float &a : acc)
            a *= keep;
        for (int j = 0; j < 32; j++) {
            const float wj = __shfl_sync(~0u, w, j);
            const KV *vj = reinterpret_cast<const KV *>(__shfl_sync(~0u, reinterpret_cast<unsigned long long>(v), j));
            if (vj)
#pragma unroll
                for (int e = 0; e < KVATTN_MAX_HEAD_DIM / 32; e++)
                    if (e * 32 + lane < D)
                        acc[e] = fmaf(wj, to_float(vj[e * 32 + lane]), acc[e]);
        }
    }
    for (int o = 16; o; o >>= 1)
        l += __shfl_xor_sync(~0u, l, o);
    const float inv = l > 0 ? d.v_scale / l : l == 0 ? 0.f : l;
#pragma unroll
    for (int e = 0; e < KVATTN_MAX_HEAD_DIM / 32; e++)
        if (e * 32 + lane < D)
            out[e * 32 + lane] = T(acc[e] * inv);
    if (lane == 0 && d.lse)
        d.lse[(int64_t)i * d.num_heads + h] = m + logf(l);
}

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

template <typename T, typename KV>
int launch(const kv_attn_desc *d, uint64_t stride, cudaStream_t stream)
{
    kv_attn_simple_kernel<T, KV><<<dim3(d->total_q, (d->num_heads + kWarps - 1) / kWarps), 32 * kWarps,
                                   kWarps * d->head_dim * sizeof(float), stream>>>(*d, stride);
    g_cc_kernel_launches.fetch_add(1, std::memory_order_relaxed);
    return cudaPeekAtLastError() == cudaSuccess ? 0 : -EIO;
}

}  // namespace

extern "C" int64_t kv_attn_workspace_bytes(const struct kv_attn_desc *d)
{
    if (!desc_ok(d))
        return -EINVAL;
    return 0;
}

extern "C" int kv_attn_launch(const struct kv_attn_desc *d, void *stream)
{
    if (!desc_ok(d))
        return -EINVAL;
    if (d->num_seqs > KVATTN_MAX_SEQS)
        return -E2BIG;
    if (!d->num_seqs || !d->total_q)
        return 0;
    const int64_t need = kv_attn_workspace_bytes(d);
    if (!d->q || !d->out || !d->k || !d->v || !d->table || !d->lens || !d->q_offsets || !d->error ||
        ((uintptr_t)d->q | (uintptr_t)d->out | (uintptr_t)d->k | (uintptr_t)d->v) % 16 ||
        (d->q_stride | d->q_head_stride | d->out_stride | d->out_head_stride) % 8 ||
        (int64_t)d->workspace_bytes < need || (need && (!d->workspace || (uintptr_t)d->workspace % 256)))
        return -EINVAL;
    DeviceGuard on(d->device);
    if (!on.ok)
        return -EIO;
    const bool e4m3 = d->kv_type == KVATTN_E4M3;
    const uint64_t stride = d->block_stride ? d->block_stride
                                            : (uint64_t)d->block_size * d->num_kv_heads * d->head_dim * (e4m3 ? 1 : 2);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (d->q_type == KVATTN_BF16)
        return e4m3 ? launch<__nv_bfloat16, __nv_fp8_e4m3>(d, stride, st) : launch<__nv_bfloat16, __nv_bfloat16>(d, stride, st);
    return e4m3 ? launch<__half, __nv_fp8_e4m3>(d, stride, st) : launch<__half, __half>(d, stride, st);
}
