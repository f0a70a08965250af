// Device side of a paged cache: where a slot is, which slots a query sees, and attention of one row by one warp.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "paged.h"

namespace cera {

constexpr uint32_t NO_PAGE = 0xffffffffu;
constexpr float PAGED_LOG2E = 1.44269504088896340736f;

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) {
    return x;
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) {
    return __float2half_rn(x);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) {
    return __float2bfloat16_rn(x);
}

__device__ __forceinline__ uint32_t paged_len(const PagedView &kv, uint32_t s) {
    const int32_t len = kv.lens[s], cap = (int32_t)(kv.max_pages * kv.page_size);
    return (uint32_t)min(max(len, 0), cap);
}
// The page of a slot below the capacity (NO_PAGE: not there) and its row in it.
__device__ __forceinline__ uint32_t paged_at(const PagedView &kv, uint32_t s, uint32_t slot, uint32_t &row) {
    const uint32_t i = (uint32_t)(((uint64_t)slot * kv.page_mul) >> kv.page_shift);
    row = slot - i * kv.page_size;
    const uint32_t page = (uint32_t)kv.table[(size_t)s * kv.max_pages + i];
    return page < kv.n_pages ? page : NO_PAGE;
}

// How many of the ascending starts[1..n_seqs] are at or below t: the sequence that token t belongs to, n_seqs for none.  A whole warp
// asks for one token; its loads do not wait for one another as a search by halves would.
__device__ __forceinline__ uint32_t paged_seq_of(const int32_t *starts, uint32_t n_seqs, uint32_t t) {
    if (!starts) return t;
    uint32_t below = 0;
    for (uint32_t i = threadIdx.x & 31; i < n_seqs; i += 32) below += (uint32_t)(starts[i + 1] <= (int32_t)t);
    return __reduce_add_sync(0xffffffffu, below);
}

// First slot of the window of a query in slot p; slots [sinks, first) are not seen, where sinks = min(sink, first).
__device__ __forceinline__ uint32_t paged_first(const PagedMask &m, uint32_t p) { return m.window && p + 1 > m.window ? p + 1 - m.window : 0; }

// The tiles that queries in slots [p, n) see: those that hold the first `sink` slots, then from the one with the first slot of p's window on.
struct PagedSpan {
    uint32_t len, first, sinks, sink_tiles, skip, tiles;

    __device__ __forceinline__ void set(const PagedMask &mask, uint32_t p, uint32_t n, uint32_t tile) {
        len = n;
        first = n ? paged_first(mask, p) : 0;
        sinks = min(mask.sink, first);
        skip = first / tile;
        sink_tiles = min((sinks + tile - 1) / tile, skip);
        skip -= sink_tiles;
        tiles = (n + tile - 1) / tile - skip;
    }
    __device__ __forceinline__ void newest(const PagedMask &mask, uint32_t n, uint32_t tile) { set(mask, n ? n - 1 : 0, n, tile); }
    __device__ __forceinline__ uint32_t slot(uint32_t t, uint32_t tile) const { return (t < sink_tiles ? t : t + skip) * tile; }
    __device__ __forceinline__ bool sees(uint32_t j) const { return j < len && (j >= first || j < sinks); }
};

// Softmax(scale q K^T) V of one query head by one warp, in f32 and one pass over the slots that it sees, no other is read.  q and out: dim
// numbers.
template <typename T, typename TQ>
__device__ __forceinline__ void paged_attend_row(const PagedView &kv, const PagedMask &mask, uint32_t s, uint32_t kvh, uint32_t p, const TQ *q, float scale, TQ *out) {
    const uint32_t lane = threadIdx.x & 31;
    float qv[8], acc[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        qv[i] = lane + 32 * i < kv.dim ? to_f32(q[lane + 32 * i]) : 0.0f;
        acc[i] = 0.0f;
    }
    const uint32_t first = paged_first(mask, p), sinks = min(mask.sink, first);
    float m = -INFINITY, l = 0.0f;
    bool any = false;
    for (uint32_t x = 0; x < sinks + p + 1 - first; ++x) {
        const uint32_t slot = x < sinks ? x : x - sinks + first;
        uint32_t row;
        const uint32_t page = paged_at(kv, s, slot, row);
        if (page == NO_PAGE) continue;
        any = true;
        const T *kr = reinterpret_cast<const T *>(kv.k + page * kv.k_page + row * kv.k_slot + kvh * kv.k_head);
        const T *vr = reinterpret_cast<const T *>(kv.v + page * kv.v_page + row * kv.v_slot + kvh * kv.v_head);
        float d = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (32 * i < kv.dim) d = fmaf(qv[i], to_f32(kr[lane + 32 * i]), d);
        const float z = warp_sum(d) * scale * PAGED_LOG2E, mn = fmaxf(m, z);
        const float corr = m == mn ? 1.0f : exp2f(m - mn), w = z == -INFINITY ? 0.0f : exp2f(z - mn);
        l = fmaf(l, corr, w);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (32 * i < kv.dim) acc[i] = fmaf(w, to_f32(vr[lane + 32 * i]), acc[i] * corr);
        m = mn;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (32 * i < kv.dim) out[lane + 32 * i] = from_f32<TQ>(any ? acc[i] / l : 0.0f);
}

}  // namespace cera
