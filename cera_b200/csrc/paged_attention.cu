// Attention over a paged cache, one warp per row.
#include "paged.cuh"

namespace cera {

namespace {

// One warp per (token, query head).  starts == nullptr: token t is the newest of sequence t.
template <typename T, typename TQ>
__global__ void __launch_bounds__(128) paged_rows_kernel(const PagedView kv, const PagedMask mask, const TQ *__restrict__ q, const int32_t *__restrict__ starts, uint32_t n,
                                                         uint32_t heads, float scale, TQ *out, float *lse) {
    pdl_trigger();
    pdl_wait();
    const size_t r = (size_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    const uint32_t t = (uint32_t)(r / heads), h = (uint32_t)(r % heads);
    if (t >= n) return;
    const uint32_t s = paged_seq_of(starts, kv.n_seqs, t);
    if (s >= kv.n_seqs) return;
    const uint32_t len = paged_len(kv, s), behind = starts ? (uint32_t)starts[s + 1] - t : 1;
    if (behind > len) {  // nothing is cached in its place
        for (uint32_t d = threadIdx.x & 31; d < kv.dim; d += 32) out[r * kv.dim + d] = from_f32<TQ>(0.0f);
        if (lse && (threadIdx.x & 31) == 0) lse[r] = INFINITY;
        return;
    }
    paged_attend_row<T, TQ>(kv, mask, s, h / (heads / kv.hk), len - behind, q + r * kv.dim, scale, out + r * kv.dim, lse ? lse + r : nullptr);
}

}  // namespace

template <typename F>
static int32_t by_types(int type, int q_type, F go) {
    if (type == CERA_TYPE_F32) return go(float(), float());
    if (type == CERA_TYPE_F16) return q_type == type ? go(__half(), __half()) : go(__half(), float());
    return q_type == type ? go(__nv_bfloat16(), __nv_bfloat16()) : go(__nv_bfloat16(), float());
}

size_t paged_prefill_workspace(const PagedView &, size_t, size_t) { return 16; }

int32_t launch_paged_prefill(const PagedView &kv, int type, const void *q, int q_type, size_t n_heads, const int32_t *starts, size_t n_tokens, float scale,
                             PagedMask mask, void *out, void *, cudaStream_t st) {
    return by_types(type, q_type, [&](auto cache, auto query) {
        using T = decltype(cache);
        using TQ = decltype(query);
        count_launch();
        return check_cuda(launch_k(paged_rows_kernel<T, TQ>, dim3((uint32_t)((n_tokens * n_heads + 3) / 4)), dim3(128), 0, st, kv, mask, (const TQ *)q, starts,
                                   (uint32_t)n_tokens, (uint32_t)n_heads, scale, (TQ *)out, (float *)nullptr),
                          "paged prefill attention launch");
    });
}

}  // namespace cera
