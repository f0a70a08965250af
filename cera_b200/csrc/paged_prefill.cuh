// What the prompt kernels over a paged cache share: which rows and keys a CTA works on, and the sum of a row's parts where the keys are split.
#pragma once

#include <algorithm>
#include <cmath>

#include "paged.cuh"

namespace cera {

namespace {

constexpr float PP_FLOOR = -3.0e38f;

struct PpParams {
    PagedView kv;
    PagedMask mask;
    const void *q;
    const int32_t *starts;
    void *out;
    float *part;   // [splits][tokens][heads][dim], for splits > 1
    float2 *ml;    // [splits][tokens][heads]
    float scale;
    uint32_t n, heads, group, box;
};

__device__ __forceinline__ float pp_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pp_low(int32_t n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; }


// What a CTA works on: rows [row0, row0 + ROWS) of a (sequence, KV head), and of the key tiles that some of them sees [x0, x1).
struct PpWork {
    uint32_t s, row0, rows, t0, len;  // t0: the sequence's first token
    int32_t p0;                       // the slot of its first token, negative if it has none
    PagedSpan span;
    uint32_t x0, x1;
    int32_t lo0, lo1, hi0, hi1;  // of either tile of rows: the slots of its first and last row, and what the first's window begins with
    uint32_t first0, first1;

    __device__ __forceinline__ int32_t slot_of(uint32_t row, uint32_t group) const { return p0 + (int32_t)(row / group); }
};

// The unit-th run of ROWS rows of all sequences, by a warp; false: there are not that many.
template <int ROWS>
__device__ __forceinline__ bool pp_find(const PpParams &p, PpWork &w, uint32_t unit) {
    const uint32_t lane = threadIdx.x & 31;
    uint32_t ahead = 0;
    for (uint32_t base = 0; base < p.kv.n_seqs; base += 32) {
        const uint32_t s = base + lane;
        uint32_t rows = 0;
        if (s < p.kv.n_seqs) {
            const int32_t a = min(max(p.starts[s], 0), (int32_t)p.n), b = min(max(p.starts[s + 1], a), (int32_t)p.n);
            rows = (uint32_t)(b - a) * p.group;
        }
        const uint32_t units = (rows + ROWS - 1) / (ROWS);
        uint32_t x = units;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= (uint32_t)o) x += y;
        }
        const uint32_t hit = __ballot_sync(0xffffffffu, ahead + x > unit);
        if (hit) {
            const int src = __ffs(hit) - 1;
            w.s = base + src;
            w.rows = __shfl_sync(0xffffffffu, rows, src);
            const uint32_t first = ahead + __shfl_sync(0xffffffffu, x - units, src), n = __shfl_sync(0xffffffffu, units, src);
            w.row0 = (n - 1 - (unit - first)) * ROWS;  // the last rows see the most: first
            return true;
        }
        ahead += __shfl_sync(0xffffffffu, x, 31);
    }
    return false;
}

// With the run's rows in one tile or two of PART.
template <int ROWS, int PART, int KT>
__device__ __forceinline__ void pp_set(const PpParams &p, PpWork &w) {
    w.t0 = (uint32_t)min(max(p.starts[w.s], 0), (int32_t)p.n);
    w.len = paged_len(p.kv, w.s);
    w.p0 = (int32_t)w.len - (int32_t)(w.rows / p.group);
    const uint32_t last = min(w.row0 + ROWS, w.rows) - 1;
    w.span.set(p.mask, (uint32_t)max(w.slot_of(w.row0, p.group), 0), (uint32_t)max(w.slot_of(last, p.group) + 1, 0), KT);
    auto tile = [&](uint32_t t, int32_t &lo, int32_t &hi, uint32_t &first) {
        const uint32_t a = w.row0 + t * PART;
        const bool some = t * PART < ROWS && a < w.rows;
        lo = some ? w.slot_of(a, p.group) : -1;
        hi = some ? w.slot_of(min(a + PART, w.rows) - 1, p.group) : -1;
        first = paged_first(p.mask, (uint32_t)max(lo, 0));
    };
    tile(0, w.lo0, w.hi0, w.first0);
    tile(1, w.lo1, w.hi1, w.first1);
    w.x0 = (uint32_t)((uint64_t)w.span.tiles * blockIdx.z / gridDim.z);
    w.x1 = (uint32_t)((uint64_t)w.span.tiles * (blockIdx.z + 1) / gridDim.z);
}

// Whether tile t of the CTA's rows sees something of the key tile at slot0.
template <int KT>
__device__ __forceinline__ bool pp_sees(const PpParams &p, const PpWork &w, uint32_t t, uint32_t slot0) {
    return (t ? w.hi1 : w.hi0) >= (int32_t)slot0 && (slot0 + KT > (t ? w.first1 : w.first0) || slot0 < p.mask.sink);
}

// A warp per row of up to 128 K numbers: the parts of its splits added up in their order.  What is loaded does not wait for whether the row is one, nor a part for the others (a lookup first and part by
// part: 9.6 us for 28 tokens of 32 heads in 9 parts, 5.3 so).
template <typename T, typename TQ, int K>
__global__ void __launch_bounds__(128) paged_prefill_join_kernel(const PpParams p, uint32_t splits) {
    pdl_trigger();
    pdl_wait();
    const uint32_t lane = threadIdx.x & 31;
    const size_t r = (size_t)blockIdx.x * 4 + (threadIdx.x >> 5), all = (size_t)p.n * p.heads;
    if (r >= all) return;
    // lane z has the parts z and z + 32
    const float2 none = make_float2(-INFINITY, 0.0f);
    float2 ml[2] = {lane < splits ? p.ml[lane * all + r] : none, lane + 32 < splits ? p.ml[(lane + 32) * all + r] : none};
    const uint32_t t = (uint32_t)(r / p.heads), h = (uint32_t)(r % p.heads), s = paged_seq_of(p.starts, p.kv.n_seqs, t);
    float m = fmaxf(ml[0].x, ml[1].x);
#pragma unroll
    for (int i = 16; i > 0; i >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, i));
    float f[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) f[k] = ml[k].x == -INFINITY ? 0.0f : pp_exp2(ml[k].x - m);  // a part that has met nothing is not there
    float l = 0.0f;
    float4 o[K];
#pragma unroll
    for (int k = 0; k < K; ++k) o[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    constexpr int U = 4;
    for (uint32_t z0 = 0; z0 < splits; z0 += U) {
        float4 x[U][K];
        float g[U], w[U];
        uint32_t some = 0;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t z = z0 + u;
            const float2 v = z < 32 ? ml[0] : ml[1];
            g[u] = __shfl_sync(0xffffffffu, z < 32 ? f[0] : f[1], z & 31);
            w[u] = __shfl_sync(0xffffffffu, v.y, z & 31);
            some |= (uint32_t)(z < splits && __shfl_sync(0xffffffffu, v.x, z & 31) != -INFINITY) << u;
#pragma unroll
            for (int k = 0; k < K; ++k)
                if ((some >> u & 1) && 128 * k + 4 * lane < p.kv.dim) x[u][k] = *reinterpret_cast<const float4 *>(p.part + (z * all + r) * p.kv.dim + 128 * k + 4 * lane);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (!(some >> u & 1)) continue;
            l = fmaf(w[u], g[u], l);
#pragma unroll
            for (int k = 0; k < K; ++k)
                if (128 * k + 4 * lane < p.kv.dim)
                    o[k] = make_float4(fmaf(x[u][k].x, g[u], o[k].x), fmaf(x[u][k].y, g[u], o[k].y), fmaf(x[u][k].z, g[u], o[k].z), fmaf(x[u][k].w, g[u], o[k].w));
        }
    }
    if (s >= p.kv.n_seqs) return;
    TQ *out = reinterpret_cast<TQ *>(p.out) + r * p.kv.dim;
    const uint32_t len = paged_len(p.kv, s), behind = (uint32_t)min(p.starts[s + 1], (int32_t)p.n) - t;
    const bool sees = behind - 1 < len;  // (starts that do not ascend see nothing)
    float check = l > 0.0f || !sees ? 0.0f : NAN;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        o[k] = make_float4(o[k].x / l, o[k].y / l, o[k].z / l, o[k].w / l);
        if (sees && 128 * k + 4 * lane < p.kv.dim) check = fmaf(o[k].x, 0.0f, fmaf(o[k].y, 0.0f, fmaf(o[k].z, 0.0f, fmaf(o[k].w, 0.0f, check))));
    }
    if (__any_sync(0xffffffffu, check != 0.0f)) {  // nothing is stored yet: the queries may be where the result goes
        __syncwarp();
        paged_attend_row<T, TQ>(p.kv, p.mask, s, h / p.group, len - behind, reinterpret_cast<const TQ *>(p.q) + r * p.kv.dim, p.scale, out);
        return;
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
        if (128 * k + 4 * lane >= p.kv.dim) continue;
        const float y[4] = {o[k].x, o[k].y, o[k].z, o[k].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) out[128 * k + 4 * lane + i] = from_f32<TQ>(sees ? y[i] : 0.0f);
    }
}

// CTAs along the rows (an upper bound: the portions' lengths are on the device) and the splits of the keys.
struct PpGrid {
    uint32_t units, splits;
};
// Microseconds that a run of rows takes with 64 slots, and beside all of them (its queries, its result, the launch).
struct PpCost {
    float slots, beside;
};
constexpr size_t PP_PARTS = (size_t)256 << 20;  // bytes of parts, at most

// The splits with which the call should be done first, as far as the host knows the lengths: capacity slots a sequence, the new tokens its last ones.  Where they are few, CTAs
// see alike and come in whole turns of the SMs (152 CTAs of 300 f32 tokens over 2000 slots: 659 us unsplit, 459 so); where they are most of the slots, a CTA sees half of
// them on average and the longest counts.  Parts are written, and read by the join.
inline uint32_t pp_splits(const PagedView &kv, size_t n_heads, size_t n, size_t rows, size_t units, PpCost cost, PagedMask mask) {
    const size_t cap = std::max<size_t>(1, (size_t)kv.max_pages * kv.page_size), seqs = std::max<size_t>(1, std::min<size_t>(kv.n_seqs, n));
    size_t longest = cap;
    if (mask.window) longest = std::min<size_t>(cap, (size_t)mask.window + std::min<size_t>(mask.sink, cap) + rows * kv.hk / n_heads + 64);
    const float tiles = (float)((longest + 63) / 64), turns = (float)(units * kv.hk) / sm_count(), spread = mask.window ? 0.0f : std::min(1.0f, (float)n / seqs / cap);
    const float join = 0.15f + (float)n * n_heads * kv.dim * 8 / 4e6f;  // a part: a turn of the join's loop, and its bytes at 4 TB/s
    const size_t most = std::min<size_t>({(size_t)tiles, 64, std::max<size_t>(1, PP_PARTS / (n * n_heads * ((size_t)kv.dim * 4 + 8)))});
    float best = 0.0f;
    uint32_t splits = 1;
    for (uint32_t z = 1; z <= most; ++z) {
        const float each = std::ceil(tiles / z) * cost.slots, alike = std::ceil(turns * z) * (each + cost.beside),
                    mixed = std::max(each + cost.beside, turns * z * (each / 2 + cost.beside) + each / 2), t = alike + spread * (mixed - alike) + (z > 1 ? 3.0f + z * join : 0.0f);
        if (z == 1 || t < 0.97f * best) {
            best = t;
            splits = z;
        }
    }
    return splits;
}
inline size_t pp_units(const PagedView &kv, size_t n_heads, size_t n, size_t rows) {
    const size_t group = n_heads / kv.hk;
    return std::min<size_t>(n * group / rows + std::min<size_t>(kv.n_seqs, n), n * group);
}

inline size_t pp_workspace(uint32_t splits, const PagedView &kv, size_t n_heads, size_t n) {
    return 16 + (splits > 1 ? splits * n * n_heads * ((size_t)kv.dim * 4 + 8) : 0);
}

inline PpParams pp_params(const PagedView &kv, PagedMask mask, const void *q, size_t n_heads, const int32_t *starts, size_t n, float scale, void *out, void *ws,
                          const PpGrid &g) {
    PpParams p;
    p.kv = kv;
    p.mask = mask;
    p.q = q;
    p.starts = starts;
    p.out = out;
    p.scale = scale;
    p.n = (uint32_t)n;
    p.heads = (uint32_t)n_heads;
    p.group = p.heads / kv.hk;
    p.box = 0;
    p.part = (float *)ws;
    p.ml = (float2 *)((uint8_t *)ws + (size_t)g.splits * n * n_heads * kv.dim * 4);
    return p;
}

// The parts' sum, where there are parts.
template <typename T, typename TQ>
int32_t pp_join(const PpParams &p, const PpGrid &g, cudaStream_t st) {
    if (g.splits == 1) return CERA_CUDA_OK;
    count_launch();
    return check_cuda(launch_k(p.kv.dim <= 128 ? paged_prefill_join_kernel<T, TQ, 1> : paged_prefill_join_kernel<T, TQ, 2>, dim3((uint32_t)(((size_t)p.n * p.heads + 3) / 4)), dim3(128), 0, st, p, g.splits), "paged prefill join launch");
}

}  // namespace

}  // namespace cera
