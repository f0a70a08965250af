// C entries of the paged cache: what they refuse, and storing new rows.
#include <algorithm>
#include <cstring>

#include "paged.cuh"

namespace cera {

namespace {

// One CTA per token.  A thread stores 8 numbers, 16 bytes of a 16-bit cache, of the token's key row and then of its value row.  The copy's bytes
// bound a large call.
template <typename T, typename TQ>
__global__ void __launch_bounds__(256) paged_append_kernel(const PagedView kv, const TQ *__restrict__ k, const TQ *__restrict__ v, const int32_t *__restrict__ starts,
                                                           uint32_t n, float *weights, int32_t *positions, size_t track_stride, const int32_t *token_pos) {
    pdl_trigger();
    pdl_wait();
    const uint32_t t = blockIdx.x, s = paged_seq_of(starts, kv.n_seqs, t);
    if (s >= kv.n_seqs) return;
    const uint32_t len = paged_len(kv, s), behind = starts ? (uint32_t)starts[s + 1] - t : 1;  // this token and those behind it in its sequence
    if (behind - 1 >= len) return;  // also where starts do not ascend
    const uint32_t slot = len - behind;
    for (uint32_t h = threadIdx.x; h < kv.hk; h += blockDim.x) {
        const size_t at = ((size_t)s * kv.hk + h) * track_stride + slot;
        if (weights) weights[at] = 0.0f;
        if (positions) positions[at] = token_pos ? token_pos[t] : (int32_t)slot;
    }
    uint32_t row;
    const uint32_t page = paged_at(kv, s, slot, row);
    if (page == NO_PAGE) return;
    const uint32_t per_head = kv.dim / 8, chunks = kv.hk * per_head;
    for (uint32_t i = threadIdx.x; i < 2 * chunks; i += blockDim.x) {
        const bool is_v = i >= chunks;
        const uint32_t c = is_v ? i - chunks : i, h = c / per_head, d = (c - h * per_head) * 8;
        const TQ *src = (is_v ? v : k) + (size_t)t * kv.hk * kv.dim + c * 8;
        uint8_t *to = is_v ? kv.v + page * kv.v_page + row * kv.v_slot + h * kv.v_head : kv.k + page * kv.k_page + row * kv.k_slot + h * kv.k_head;
        alignas(16) TQ in[8];
        alignas(16) T o[8];
#pragma unroll
        for (size_t b = 0; b < sizeof(in) / 16; ++b) reinterpret_cast<uint4 *>(in)[b] = reinterpret_cast<const uint4 *>(src)[b];
#pragma unroll
        for (int b = 0; b < 8; ++b) o[b] = sizeof(T) == sizeof(TQ) ? *reinterpret_cast<T *>(&in[b]) : from_f32<T>(to_f32(in[b]));
#pragma unroll
        for (size_t b = 0; b < sizeof(o) / 16; ++b) reinterpret_cast<uint4 *>(to + d * sizeof(T))[b] = reinterpret_cast<const uint4 *>(o)[b];
    }
}

size_t elem(int type) { return type == CERA_TYPE_F32 ? 4 : 2; }

// The view of a cache, or a refusal.
int32_t view(const char *what, const cera_cuda_paged_kv *kv, PagedView *out) {
    if (!kv) return fail(CERA_CUDA_ERR_BAD_ARG, "%s: null cache", what);
    if (kv->type != CERA_TYPE_F32 && kv->type != CERA_TYPE_F16 && kv->type != CERA_TYPE_BF16)
        return fail(CERA_CUDA_ERR_UNSUPPORTED, "%s: a cache of type %d", what, kv->type);
    if (kv->head_dim == 0 || kv->head_dim % 32 || kv->head_dim > 256)
        return fail(CERA_CUDA_ERR_UNSUPPORTED, "%s: head_dim %u (a multiple of 32 up to 256)", what, kv->head_dim);
    if (kv->n_seqs > 4096) return fail(CERA_CUDA_ERR_UNSUPPORTED, "%s: %u sequences (4096 at most)", what, kv->n_seqs);
    if (kv->n_kv_heads == 0 || kv->n_kv_heads > 4096 || kv->page_size == 0 || kv->n_pages > 0x7fffffffu)
        return fail(CERA_CUDA_ERR_BAD_ARG, "%s: %u KV heads, pages of %u slots, %u pages", what, kv->n_kv_heads, kv->page_size, kv->n_pages);
    if ((uint64_t)kv->max_pages * kv->page_size >= 0x7fffff00u) return fail(CERA_CUDA_ERR_BAD_ARG, "%s: %u pages of %u slots per sequence", what, kv->max_pages, kv->page_size);
    if (kv->n_seqs && ((kv->n_pages && (!kv->k_pages_dev || !kv->v_pages_dev)) || (kv->max_pages && !kv->page_table_dev) || !kv->seq_lens_dev))
        return fail(CERA_CUDA_ERR_BAD_ARG, "%s: null pages, table or lengths", what);
    const size_t e = elem(kv->type), per = 16 / e;
    if ((((uintptr_t)kv->k_pages_dev | (uintptr_t)kv->v_pages_dev) & 15) || kv->k_page_stride % per || kv->k_slot_stride % per || kv->k_head_stride % per ||
        kv->v_page_stride % per || kv->v_slot_stride % per || kv->v_head_stride % per)
        return fail(CERA_CUDA_ERR_BAD_ARG, "%s: pages and strides must be multiples of 16 bytes", what);
    if ((uint64_t)kv->n_seqs * ((uint64_t)kv->max_pages * kv->page_size / 32 + 1) > 0xffffffffu)
        return fail(CERA_CUDA_ERR_BAD_ARG, "%s: %u sequences of %u pages of %u slots", what, kv->n_seqs, kv->max_pages, kv->page_size);
    if (((uintptr_t)kv->page_table_dev | (uintptr_t)kv->seq_lens_dev) & 3) return fail(CERA_CUDA_ERR_BAD_ARG, "%s: table or lengths off a 4-byte boundary", what);
    uint32_t l = 0;
    while ((1ull << l) < kv->page_size) ++l;
    out->page_shift = 31 + l;
    out->page_mul = (uint32_t)(((1ull << out->page_shift) + kv->page_size - 1) / kv->page_size);
    out->page_size = kv->page_size;
    out->k = (uint8_t *)kv->k_pages_dev;
    out->v = (uint8_t *)kv->v_pages_dev;
    out->table = kv->page_table_dev;
    out->lens = kv->seq_lens_dev;
    out->k_page = kv->k_page_stride * e;
    out->k_slot = kv->k_slot_stride * e;
    out->k_head = kv->k_head_stride * e;
    out->v_page = kv->v_page_stride * e;
    out->v_slot = kv->v_slot_stride * e;
    out->v_head = kv->v_head_stride * e;
    out->n_pages = kv->n_pages;
    out->hk = kv->n_kv_heads;
    out->dim = kv->head_dim;
    out->n_seqs = kv->n_seqs;
    out->max_pages = kv->max_pages;
    return CERA_CUDA_OK;
}

// Heads and types of an attention call.
int32_t check_heads(const char *what, const PagedView &v, int32_t type, int32_t q_type, size_t n_heads) {
    if (q_type != type && q_type != CERA_TYPE_F32) return fail(CERA_CUDA_ERR_UNSUPPORTED, "%s: queries of type %d over a cache of type %d", what, q_type, type);
    if (n_heads == 0 || n_heads % v.hk || n_heads > 65535) return fail(CERA_CUDA_ERR_BAD_ARG, "%s: %zu heads over %u KV heads", what, n_heads, v.hk);
    return CERA_CUDA_OK;
}

// A result goes where its queries are, or apart from them.
int32_t check_out(const char *what, const void *q, const void *out, int32_t q_type, const PagedView &v, size_t n, size_t n_heads) {
    const uintptr_t a = (uintptr_t)q, b = (uintptr_t)out;
    if (!q || !out || ((a | b) & 15)) return fail(CERA_CUDA_ERR_BAD_ARG, "%s: queries or result null or off a 16-byte boundary", what);
    if (a != b && (a < b ? b - a : a - b) < n * n_heads * v.dim * elem(q_type)) return fail(CERA_CUDA_ERR_BAD_ARG, "%s: the result covers a part of the queries", what);
    return CERA_CUDA_OK;
}

// Rows (token, head of a KV head) are counted in 31 bits.
int32_t check_tokens(const char *what, const PagedView &v, size_t n_heads, size_t n_tokens) {
    if (n_tokens > 0x7fffffffu / (n_heads / v.hk)) return fail(CERA_CUDA_ERR_BAD_ARG, "%s: %zu tokens", what, n_tokens);
    return CERA_CUDA_OK;
}

int32_t check_workspace(const char *what, const void *ws, size_t have, size_t need) {
    if (have < need || (need && !ws) || ((uintptr_t)ws & 15)) return fail(CERA_CUDA_ERR_BAD_ARG, "%s: a workspace of %zu bytes (%zu, on a 16-byte boundary)", what, have, need);
    return CERA_CUDA_OK;
}

}  // namespace

int32_t paged_maps(const PagedView &kv, int type, uint32_t least, uint32_t *box, CUtensorMap *k, CUtensorMap *v) {
    memset(k, 0, sizeof(*k));
    memset(v, 0, sizeof(*v));
    while (*box >= least && kv.page_size % *box) *box /= 2;
    const size_t far = std::max({kv.k_page, kv.k_slot, kv.k_head, kv.v_page, kv.v_slot, kv.v_head});
    if (*box < least || !kv.n_pages || far >= 1ull << 40) {
        *box = 0;
        return CERA_CUDA_OK;
    }
    const uint32_t e = type == CERA_TYPE_F32 ? 4 : 2, boxes[4] = {128 / e, 1, *box, 1};
    const uint64_t dims[4] = {kv.dim, kv.hk, kv.page_size, kv.n_pages};
    const CUtensorMapDataType t = type == CERA_TYPE_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : type == CERA_TYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    uint64_t ks[3] = {kv.k_head, kv.k_slot, kv.k_page}, vs[3] = {kv.v_head, kv.v_slot, kv.v_page};
    for (int i = 0; i < 3; ++i)
        if (dims[i + 1] == 1) ks[i] = vs[i] = 16;  // nothing is that far
    CERA_TRY(tensor_map_4d(k, t, kv.k, dims, ks, boxes));
    return tensor_map_4d(v, t, kv.v, dims, vs, boxes);
}

size_t paged_prefill_workspace(const PagedView &kv, int type, size_t n_heads, size_t n_tokens) {
    return type == CERA_TYPE_F32 ? paged_prefill_f32_workspace(kv, n_heads, n_tokens) : paged_prefill_tc_workspace(kv, n_heads, n_tokens);
}

int32_t launch_paged_prefill(const PagedView &kv, int type, const void *q, int q_type, size_t n_heads, const int32_t *starts, size_t n_tokens, float scale,
                             PagedMask mask, void *out, void *ws, cudaStream_t st) {
    if (type != CERA_TYPE_F32) return launch_paged_prefill_tc(kv, type, q, q_type, n_heads, starts, n_tokens, scale, mask, out, ws, st);
    return launch_paged_prefill_f32(kv, (const float *)q, n_heads, starts, n_tokens, scale, mask, (float *)out, ws, st);
}

int32_t launch_paged_append(const PagedView &kv, int type, const void *k, const void *v, int src_type, const int32_t *starts, size_t n, float *weights,
                            int32_t *positions, size_t track_stride, const int32_t *token_pos, cudaStream_t st) {
    auto go = [&](auto cache, auto source) {
        using T = decltype(cache);
        using TQ = decltype(source);
        count_launch();
        return check_cuda(launch_k(paged_append_kernel<T, TQ>, dim3((uint32_t)n), dim3(256), 0, st, kv, (const TQ *)k, (const TQ *)v, starts, (uint32_t)n, weights, positions,
                                   track_stride, token_pos),
                          "paged append launch");
    };
    if (type == CERA_TYPE_F32) return go(float(), float());
    if (type == CERA_TYPE_F16) return src_type == type ? go(__half(), __half()) : go(__half(), float());
    return src_type == type ? go(__nv_bfloat16(), __nv_bfloat16()) : go(__nv_bfloat16(), float());
}

}  // namespace cera

using namespace cera;

extern "C" {

int32_t cera_cuda_paged_append(const cera_cuda_paged_kv *kv, const void *k_dev, const void *v_dev, int32_t type, const int32_t *starts_dev, size_t n_tokens,
                               float *weights_dev, int32_t *positions_dev, size_t track_stride, const int32_t *token_positions_dev, void *stream) {
    const char *what = "paged_append";
    PagedView v;
    CERA_TRY(view(what, kv, &v));
    if (type != kv->type && type != CERA_TYPE_F32) return fail(CERA_CUDA_ERR_UNSUPPORTED, "%s: rows of type %d into a cache of type %d", what, type, kv->type);
    if (!starts_dev && n_tokens != v.n_seqs) return fail(CERA_CUDA_ERR_BAD_ARG, "%s: %zu tokens for %u sequences and no starts", what, n_tokens, v.n_seqs);
    if (n_tokens > 0x7fffffffu) return fail(CERA_CUDA_ERR_BAD_ARG, "%s: %zu tokens", what, n_tokens);
    if ((weights_dev || positions_dev) && track_stride < (size_t)v.max_pages * v.page_size)
        return fail(CERA_CUDA_ERR_BAD_ARG, "%s: weights or positions of %zu slots (%zu)", what, track_stride, (size_t)v.max_pages * v.page_size);
    if (n_tokens == 0 || v.n_seqs == 0) return CERA_CUDA_OK;
    if (!k_dev || !v_dev || (((uintptr_t)k_dev | (uintptr_t)v_dev) & 15)) return fail(CERA_CUDA_ERR_BAD_ARG, "%s: rows null or off a 16-byte boundary", what);
    return launch_paged_append(v, kv->type, k_dev, v_dev, type, starts_dev, n_tokens, weights_dev, positions_dev, track_stride, token_positions_dev, (cudaStream_t)stream);
}

size_t cera_cuda_paged_decode_attention_workspace_bytes(const cera_cuda_paged_kv *kv, size_t n_heads, int32_t with_weights) {
    PagedView v;
    if (view("paged_decode_attention", kv, &v) != CERA_CUDA_OK || check_heads("paged_decode_attention", v, kv->type, kv->type, n_heads) != CERA_CUDA_OK) return 0;
    return paged_decode_workspace(v, n_heads, with_weights != 0);
}

int32_t cera_cuda_paged_decode_attention(const cera_cuda_paged_kv *kv, const void *q_dev, int32_t q_type, size_t n_heads, float scale, uint32_t window,
                                         uint32_t n_sink, float *weights_dev, size_t weights_stride, void *out_dev, void *workspace_dev, size_t workspace_bytes,
                                         void *stream) {
    const char *what = "paged_decode_attention";
    PagedView v;
    CERA_TRY(view(what, kv, &v));
    CERA_TRY(check_heads(what, v, kv->type, q_type, n_heads));
    if (weights_dev && weights_stride < (size_t)v.max_pages * v.page_size)
        return fail(CERA_CUDA_ERR_BAD_ARG, "%s: weights of %zu slots (%zu)", what, weights_stride, (size_t)v.max_pages * v.page_size);
    if (v.n_seqs == 0) return CERA_CUDA_OK;
    CERA_TRY(check_out(what, q_dev, out_dev, q_type, v, v.n_seqs, n_heads));
    CERA_TRY(check_workspace(what, workspace_dev, workspace_bytes, paged_decode_workspace(v, n_heads, weights_dev != nullptr)));
    return launch_paged_decode(v, kv->type, q_dev, q_type, n_heads, scale, PagedMask{window, n_sink}, weights_dev, weights_stride, out_dev, workspace_dev,
                               (cudaStream_t)stream);
}

size_t cera_cuda_paged_prefill_attention_workspace_bytes(const cera_cuda_paged_kv *kv, size_t n_heads, size_t n_tokens) {
    PagedView v;
    if (view("paged_prefill_attention", kv, &v) != CERA_CUDA_OK || check_heads("paged_prefill_attention", v, kv->type, kv->type, n_heads) != CERA_CUDA_OK ||
        check_tokens("paged_prefill_attention", v, n_heads, n_tokens) != CERA_CUDA_OK)
        return 0;
    if (n_tokens == 0 || v.n_seqs == 0) return 16;  // nothing to do, which is no refusal
    return paged_prefill_workspace(v, kv->type, n_heads, n_tokens);
}

int32_t cera_cuda_paged_prefill_attention(const cera_cuda_paged_kv *kv, const void *q_dev, int32_t q_type, size_t n_heads, const int32_t *starts_dev,
                                          size_t n_tokens, float scale, uint32_t window, uint32_t n_sink, void *out_dev, void *workspace_dev,
                                          size_t workspace_bytes, void *stream) {
    const char *what = "paged_prefill_attention";
    PagedView v;
    CERA_TRY(view(what, kv, &v));
    CERA_TRY(check_heads(what, v, kv->type, q_type, n_heads));
    CERA_TRY(check_tokens(what, v, n_heads, n_tokens));
    if (n_tokens == 0 || v.n_seqs == 0) return CERA_CUDA_OK;
    if (!starts_dev) return fail(CERA_CUDA_ERR_BAD_ARG, "%s: no starts", what);
    CERA_TRY(check_out(what, q_dev, out_dev, q_type, v, n_tokens, n_heads));
    CERA_TRY(check_workspace(what, workspace_dev, workspace_bytes, paged_prefill_workspace(v, kv->type, n_heads, n_tokens)));
    return launch_paged_prefill(v, kv->type, q_dev, q_type, n_heads, starts_dev, n_tokens, scale, PagedMask{window, n_sink}, out_dev, workspace_dev,
                                (cudaStream_t)stream);
}

int32_t cera_cuda_paged_evict(const cera_cuda_paged_kv *kv, const float *weights_dev, const int32_t *positions_dev, size_t track_stride, size_t budget,
                              uint32_t n_sink, uint32_t n_recent, float *weights_out_dev, int32_t *positions_out_dev, size_t out_stride, int32_t *kept_dev,
                              int32_t *seq_lens_out_dev, void *stream) {
    const char *what = "paged_evict";
    PagedView v;
    CERA_TRY(view(what, kv, &v));
    const size_t cap = (size_t)v.max_pages * v.page_size;
    if (budget == 0 || budget > 0x7fffff00u || (uint64_t)n_sink + n_recent > budget)
        return fail(CERA_CUDA_ERR_BAD_ARG, "%s: a budget of %zu slots for %u first and %u recent ones", what, budget, n_sink, n_recent);
    if (track_stride < cap || out_stride < (budget < cap ? budget : cap))
        return fail(CERA_CUDA_ERR_BAD_ARG, "%s: weights and positions of %zu slots into %zu (%zu, budget %zu)", what, track_stride, out_stride, cap, budget);
    if (v.n_seqs == 0) return CERA_CUDA_OK;
    if ((cap && (!weights_dev || !positions_dev || !weights_out_dev || !positions_out_dev)) || !kept_dev || !seq_lens_out_dev)  // of no slots there is nothing
        return fail(CERA_CUDA_ERR_BAD_ARG, "%s: null argument", what);
    if ((weights_out_dev == weights_dev && out_stride != track_stride) || (positions_out_dev == positions_dev && out_stride != track_stride))
        return fail(CERA_CUDA_ERR_BAD_ARG, "%s: in place with another stride", what);
    return launch_paged_evict(v, kv->type, weights_dev, positions_dev, track_stride, budget, n_sink, n_recent, weights_out_dev, positions_out_dev, out_stride, kept_dev,
                              seq_lens_out_dev, (cudaStream_t)stream);
}

}  // extern "C"
