// Causal attention of ragged prompt portions over a paged f32 cache, in f32 on the CUDA cores.
//
// A row is (token, query head of a KV head).  A CTA of 256 threads owns 64 rows of one (sequence, KV head) and walks tiles of 64 keys with a running maximum and
// sum: a thread forms the scores of 4 rows x 4 keys, two dimensions an FMA, then 4 rows x 4 (8, 16) dimensions of the result, the weights
// passing through shared memory in between.  Sixteen lanes share a row's keys and dimensions.  The keys of the next tile arrive during softmax and values, its
// values during the scores.
//
// What bounds it: loads from shared memory, 8 of 16 bytes for 32 packed FMAs, at 128 bytes a cycle of an SM (300 tokens of 32 heads over 2300 slots: 398 us, 27 TFLOP/s).  Threads of 8
// rows x 4 keys load less, 12 for 64, but half as many warps wait for them one by one: 458 us.
//
// A row that ends without finite values - a weight of zero times an infinite value of a key it does not see - or that has met no weight is computed again by
// paged_attend_row, which reads nothing that the row does not see.  Few rows over a long cache: the keys are split over gridDim.z.
#include "paged_prefill.cuh"
#include "tma.cuh"

namespace cera {

namespace {

constexpr int PF_ROWS = 64, PF_KT = 64, PF_EACH = 4, PF_THREADS = 16 * PF_ROWS / PF_EACH;  // rows of a thread

template <int DP>
struct Pf {
    static constexpr int LD = DP + 4, LP = PF_KT + 4, NV = DP / 64;  // padded rows of Q, K and of the weights: eight of a load meet all banks
    static constexpr size_t SMEM = 4 * (size_t)(2 * PF_ROWS * LD + PF_KT * DP + PF_ROWS * LP);
};

__device__ __forceinline__ void pf_copy(void *dst, const void *src, bool there) {  // 16 bytes, zeros where there is nothing
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(tma::smem_u32(dst)), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void pf_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void pf_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

template <int DP>
__global__ void __launch_bounds__(PF_THREADS) paged_prefill_f32_kernel(const PpParams p) {
    using C = Pf<DP>;
    extern __shared__ __align__(16) float smem[];
    float *qs = smem, *ks = qs + PF_ROWS * C::LD, *vs = ks + PF_KT * C::LD, *ps = vs + PF_KT * DP;
    __shared__ PpWork work;
    __shared__ uint64_t off_k[PF_KT], off_v[PF_KT];
    __shared__ uint32_t there_s[2][2];  // which of a tile's keys there are, of two tiles
    pdl_trigger();
    pdl_wait();
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, h = blockIdx.y, dim = p.kv.dim, g16 = lane & 15, r0 = (warp * 2 + (lane >> 4)) * PF_EACH;
    if (warp == 0) {
        PpWork w;
        if (pp_find<PF_ROWS>(p, w, blockIdx.x)) pp_set<PF_ROWS, PF_ROWS, PF_KT>(p, w);
        else w.rows = 0;
        if (tid == 0) work = w;
    }
    __syncthreads();
    const PpWork w = work;
    if (w.rows == 0) return;

    // keys and values of a tile: rows looked up by 64 threads, copied by all
    auto look = [&](uint32_t x) {
        if (tid < PF_KT) {
            const uint32_t j = w.span.slot(x, PF_KT) + tid;
            uint32_t row = 0;
            const uint32_t page = w.span.sees(j) ? paged_at(p.kv, w.s, j, row) : NO_PAGE;
            const bool there = page != NO_PAGE;
            off_k[tid] = there ? page * (uint64_t)p.kv.k_page + row * (uint64_t)p.kv.k_slot + h * (uint64_t)p.kv.k_head : ~0ull;
            off_v[tid] = there ? page * (uint64_t)p.kv.v_page + row * (uint64_t)p.kv.v_slot + h * (uint64_t)p.kv.v_head : ~0ull;
            const uint32_t mask = __ballot_sync(0xffffffffu, there);
            if (lane == 0) there_s[x & 1][warp] = mask;
        }
    };
    const uint32_t chunks = dim / 4;
    auto copy = [&](const uint64_t *off, const uint8_t *base, float *to, uint32_t ld) {
        for (uint32_t i = tid; i < PF_KT * chunks; i += PF_THREADS) {
            const uint32_t r = i / chunks, c = i - r * chunks;
            const uint64_t o = off[r];
            pf_copy(to + r * ld + c * 4, base + (o == ~0ull ? 0 : o + c * 16), o != ~0ull);
        }
        pf_commit();
    };
    if (w.x0 < w.x1) look(w.x0);
    for (uint32_t i = tid; i < PF_ROWS * chunks; i += PF_THREADS) {
        const uint32_t r = i / chunks, c = i - r * chunks, row = w.row0 + r;
        const bool live = row < w.rows;
        const float *q = reinterpret_cast<const float *>(p.q) + (live ? ((size_t)(w.t0 + row / p.group) * p.heads + h * p.group + row % p.group) * dim + c * 4 : 0);
        pf_copy(qs + r * C::LD + c * 4, q, live);
    }
    pf_commit();
    __syncthreads();
    if (w.x0 < w.x1) copy(off_k, p.kv.k, ks, C::LD);

    int32_t pos[PF_EACH];
#pragma unroll
    for (int r = 0; r < PF_EACH; ++r) pos[r] = w.row0 + r0 + r < w.rows ? w.slot_of(w.row0 + r0 + r, p.group) : -1;
    const int32_t lo = w.lo0, hi = w.hi0, first_hi = hi >= 0 ? (int32_t)paged_first(p.mask, (uint32_t)hi) : 0;
    const float scale = p.scale * PAGED_LOG2E;
    float m[PF_EACH], l[PF_EACH];
    float4 acc[PF_EACH][C::NV];
#pragma unroll
    for (int r = 0; r < PF_EACH; ++r) {
        m[r] = PP_FLOOR;
        l[r] = 0.0f;
#pragma unroll
        for (int i = 0; i < C::NV; ++i) acc[r][i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
    for (uint32_t x = w.x0; x < w.x1; ++x) {
        const uint32_t slot0 = w.span.slot(x, PF_KT);
        copy(off_v, p.kv.v, vs, DP);
        pf_wait<1>();
        __syncthreads();  // the keys are there, and the offsets are read
        const uint32_t there[2] = {there_s[x & 1][0], there_s[x & 1][1]};
        if (x + 1 < w.x1) look(x + 1);
        float2 s2[PF_EACH][4];
#pragma unroll
        for (int r = 0; r < PF_EACH; ++r)
#pragma unroll
            for (int k = 0; k < 4; ++k) s2[r][k] = make_float2(0.0f, 0.0f);
#pragma unroll 2
        for (uint32_t d = 0; d < dim; d += 4) {
            float4 kk[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) kk[k] = *reinterpret_cast<const float4 *>(ks + (g16 + 16 * k) * C::LD + d);
#pragma unroll
            for (int r = 0; r < PF_EACH; ++r) {
                const float4 q = *reinterpret_cast<const float4 *>(qs + (r0 + r) * C::LD + d);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    s2[r][k] = __ffma2_rn(make_float2(q.x, q.y), make_float2(kk[k].x, kk[k].y), s2[r][k]);
                    s2[r][k] = __ffma2_rn(make_float2(q.z, q.w), make_float2(kk[k].z, kk[k].w), s2[r][k]);
                }
            }
        }
        __syncthreads();  // the keys are read, the next offsets there
        if (x + 1 < w.x1) copy(off_k, p.kv.k, ks, C::LD);
        else pf_commit();
        const bool all = (there[0] & there[1]) == 0xffffffffu && (int32_t)(slot0 + PF_KT) <= lo + 1 && ((int32_t)slot0 >= first_hi || slot0 + PF_KT <= p.mask.sink);
#pragma unroll
        for (int r = 0; r < PF_EACH; ++r) {
            float z[4], mx = -INFINITY;
            const int32_t first = all || pos[r] < 0 ? 0 : (int32_t)paged_first(p.mask, (uint32_t)pos[r]);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                z[k] = (s2[r][k].x + s2[r][k].y) * scale;
                if (!all) {
                    const uint32_t i = g16 + 16 * k;
                    const int32_t j = (int32_t)(slot0 + i);
                    if (!(j <= pos[r] && (j >= first || (uint32_t)j < p.mask.sink) && (there[k >> 1] >> (i & 31) & 1))) z[k] = -INFINITY;
                }
                mx = fmaxf(mx, z[k]);
            }
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
            if (mx > m[r]) {
                const float f = pp_exp2(m[r] - mx);
                m[r] = mx;
                l[r] *= f;
#pragma unroll
                for (int i = 0; i < C::NV; ++i) acc[r][i] = make_float4(acc[r][i].x * f, acc[r][i].y * f, acc[r][i].z * f, acc[r][i].w * f);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float e = pp_exp2(z[k] - m[r]);
                l[r] += e;
                ps[(r0 + r) * C::LP + g16 + 16 * k] = e;
            }
        }
        pf_wait<1>();
        __syncthreads();  // the values are there (and the weights, which a warp keeps to itself)
#pragma unroll 2
        for (uint32_t k = 0; k < PF_KT; k += 4) {
            float4 e[PF_EACH];
#pragma unroll
            for (int r = 0; r < PF_EACH; ++r) e[r] = *reinterpret_cast<const float4 *>(ps + (r0 + r) * C::LP + k);
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
#pragma unroll
                for (int i = 0; i < C::NV; ++i) {
                    const float4 v = *reinterpret_cast<const float4 *>(vs + (k + kk) * DP + (g16 + 16 * i) * 4);
#pragma unroll
                    for (int r = 0; r < PF_EACH; ++r) {
                        const float wt = kk == 0 ? e[r].x : kk == 1 ? e[r].y : kk == 2 ? e[r].z : e[r].w;
                        const float2 a = __ffma2_rn(make_float2(wt, wt), make_float2(v.x, v.y), make_float2(acc[r][i].x, acc[r][i].y));
                        const float2 b = __ffma2_rn(make_float2(wt, wt), make_float2(v.z, v.w), make_float2(acc[r][i].z, acc[r][i].w));
                        acc[r][i] = make_float4(a.x, a.y, b.x, b.y);
                    }
                }
        }
        __syncthreads();  // values and weights are read
    }
    pf_wait<0>();
    uint32_t again = 0;
#pragma unroll
    for (int r = 0; r < PF_EACH; ++r) {
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], o);
        const uint32_t row = w.row0 + r0 + r;
        const bool live = row < w.rows;
        const size_t place = live ? (size_t)(w.t0 + row / p.group) * p.heads + h * p.group + row % p.group : 0;
        if (gridDim.z > 1) {
            const size_t at = (size_t)blockIdx.z * p.n * p.heads + place;
            if (live && g16 == 0) p.ml[at] = make_float2(l[r] != l[r] || m[r] != PP_FLOOR ? m[r] : -INFINITY, l[r]);
#pragma unroll
            for (int i = 0; i < C::NV; ++i)
                if (live && (g16 + 16 * i) * 4 < dim) *reinterpret_cast<float4 *>(p.part + at * dim + (g16 + 16 * i) * 4) = acc[r][i];
            continue;
        }
        const float f = 1.0f / l[r];
        float check = l[r] > 0.0f && m[r] != PP_FLOOR ? 0.0f : NAN;
#pragma unroll
        for (int i = 0; i < C::NV; ++i) {
            if (!live || (g16 + 16 * i) * 4 >= dim) continue;
            const float4 o = acc[r][i] = make_float4(acc[r][i].x * f, acc[r][i].y * f, acc[r][i].z * f, acc[r][i].w * f);
            check = fmaf(o.x, 0.0f, fmaf(o.y, 0.0f, fmaf(o.z, 0.0f, fmaf(o.w, 0.0f, check))));
        }
        const uint32_t bad = __ballot_sync(0xffffffffu, pos[r] >= 0 && check != 0.0f);
        if (!(bad >> (lane & 16) & 0xffffu)) {  // what is computed again is stored then: the queries may be where the result goes
#pragma unroll
            for (int i = 0; i < C::NV; ++i)
                if (live && (g16 + 16 * i) * 4 < dim)
                    *reinterpret_cast<float4 *>(reinterpret_cast<float *>(p.out) + place * dim + (g16 + 16 * i) * 4) = pos[r] >= 0 ? acc[r][i] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
        again |= (bad & 0xffffu ? 1u << r : 0) | (bad >> 16 ? 1u << (PF_EACH + r) : 0);
    }
    for (; again; again &= again - 1) {
        const uint32_t row = w.row0 + warp * 2 * PF_EACH + __ffs(again) - 1;
        const size_t place = ((size_t)(w.t0 + row / p.group) * p.heads + h * p.group + row % p.group) * dim;
        __syncwarp();
        paged_attend_row<float, float>(p.kv, p.mask, w.s, h, (uint32_t)w.slot_of(row, p.group), reinterpret_cast<const float *>(p.q) + place, p.scale,
                                       reinterpret_cast<float *>(p.out) + place);
    }
}

uint32_t pf_splits(const PagedView &kv, size_t n_heads, size_t n, PagedMask mask) {
    return pp_splits(kv, n_heads, n, PF_ROWS, pp_units(kv, n_heads, n, PF_ROWS), PpCost{0.065f * kv.dim, 8.0f}, mask);
}

template <int DP>
int32_t pf_launch(const PpParams &p, const PpGrid &g, cudaStream_t st) {
    auto kernel = paged_prefill_f32_kernel<DP>;
    CERA_TRY(paged_smem<paged_prefill_f32_kernel<DP>>(Pf<DP>::SMEM));
    count_launch();
    CERA_CUDA_TRY(launch_k(kernel, dim3(g.units, p.kv.hk, g.splits), dim3(PF_THREADS), Pf<DP>::SMEM, st, p));
    return pp_join<float, float>(p, g, st);
}

}  // namespace

size_t paged_prefill_f32_workspace(const PagedView &kv, size_t n_heads, size_t n) { return pp_workspace(pf_splits(kv, n_heads, n, PagedMask{0, 0}), kv, n_heads, n); }

int32_t launch_paged_prefill_f32(const PagedView &kv, const float *q, size_t n_heads, const int32_t *starts, size_t n_tokens, float scale, PagedMask mask, float *out,
                                 void *ws, cudaStream_t st) {
    uint32_t splits = pf_splits(kv, n_heads, n_tokens, mask);
    if (mask.window) splits = std::min(splits, pf_splits(kv, n_heads, n_tokens, PagedMask{0, 0}));  // which the workspace has room for
    const PpGrid g = {(uint32_t)pp_units(kv, n_heads, n_tokens, PF_ROWS), splits};
    const PpParams p = pp_params(kv, mask, q, n_heads, starts, n_tokens, scale, out, ws, g);
    if (kv.dim <= 64) return pf_launch<64>(p, g, st);
    if (kv.dim <= 128) return pf_launch<128>(p, g, st);
    return pf_launch<256>(p, g, st);
}

}  // namespace cera
