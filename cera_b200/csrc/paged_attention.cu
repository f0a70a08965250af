// Attention over a paged cache, one warp per row.
#include "paged.cuh"

namespace cera {

namespace {

// One warp per (token, query head).  starts == nullptr: token t is the newest of sequence t.
template <typename T, typename TQ>
__global__ void __launch_bounds__(128) paged_rows_kernel(const PagedView kv, const PagedMask mask, const TQ *__restrict__ q, const int32_t *__restrict__ starts, uint32_t n,
                                                         uint32_t heads, float scale, TQ *out) {
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
        return;
    }
    paged_attend_row<T, TQ>(kv, mask, s, h / (heads / kv.hk), len - behind, q + r * kv.dim, scale, out + r * kv.dim);
}

}  // namespace

size_t paged_prefill_workspace(const PagedView &kv, int type, size_t n_heads, size_t n_tokens) {
    return type == CERA_TYPE_F32 ? 16 : paged_prefill_tc_workspace(kv, n_heads, n_tokens);
}

int32_t launch_paged_prefill(const PagedView &kv, int type, const void *q, int q_type, size_t n_heads, const int32_t *starts, size_t n_tokens, float scale,
                             PagedMask mask, void *out, void *ws, cudaStream_t st) {
    if (type != CERA_TYPE_F32) return launch_paged_prefill_tc(kv, type, q, q_type, n_heads, starts, n_tokens, scale, mask, out, ws, st);
    count_launch();
    return check_cuda(launch_k(paged_rows_kernel<float, float>, dim3((uint32_t)((n_tokens * n_heads + 3) / 4)), dim3(128), 0, st, kv, mask, (const float *)q, starts,
                               (uint32_t)n_tokens, (uint32_t)n_heads, scale, (float *)out),
                      "paged prefill attention launch");
}

}  // namespace cera
