// A paged key/value cache as kernels see it, and the launches of what reads and writes it.
#pragma once

#include "common.cuh"
#include "tensor_map.h"

namespace cera {

// Strides in bytes.  A quotient by the page size is (n * page_mul) >> page_shift, exact for n below 2^31.
struct PagedView {
    uint8_t *k, *v;
    const int32_t *table, *lens;
    size_t k_page, k_slot, k_head, v_page, v_slot, v_head;
    uint32_t page_mul, page_shift, page_size, n_pages, hk, dim, n_seqs, max_pages;
};

// What a query in slot p sees of the slots: j <= p, and with a window j < sink or j > p - window.
struct PagedMask {
    uint32_t window, sink;
};

// Tensor maps of the pages of keys and values, boxes of *box slots and 128 bytes of one head laid down with the 128-byte swizzle: *box, a power of two, is halved
// until a page holds whole boxes.  0 where that would take it below `least`, or the pages are none or too far apart: no maps, rows are copied one by one.
int32_t paged_maps(const PagedView &kv, int type, uint32_t least, uint32_t *box, CUtensorMap *k, CUtensorMap *v);

// Lets a kernel have that much dynamic shared memory, asked for once per thread and device.
template <auto KERNEL>
inline int32_t paged_smem(size_t bytes) {
    static thread_local int configured = -1;
    int dev = 0;
    CERA_CUDA_TRY(cudaGetDevice(&dev));
    if (configured == dev) return CERA_CUDA_OK;
    CERA_CUDA_TRY(cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
    configured = dev;
    return CERA_CUDA_OK;
}

int32_t launch_paged_append(const PagedView &kv, int type, const void *k, const void *v, int src_type, const int32_t *starts, size_t n, float *weights,
                            int32_t *positions, size_t track_stride, const int32_t *token_pos, cudaStream_t st);
size_t paged_decode_workspace(const PagedView &kv, size_t n_heads, bool weights);
int32_t launch_paged_decode(const PagedView &kv, int type, const void *q, int q_type, size_t n_heads, float scale, PagedMask mask, float *weights,
                            size_t weights_stride, void *out, void *ws, cudaStream_t st);
size_t paged_prefill_workspace(const PagedView &kv, int type, size_t n_heads, size_t n_tokens);
// 16-bit caches on the tensor cores, f32 caches with FMAs.
size_t paged_prefill_tc_workspace(const PagedView &kv, size_t n_heads, size_t n_tokens);
size_t paged_prefill_f32_workspace(const PagedView &kv, size_t n_heads, size_t n_tokens);
int32_t launch_paged_prefill_f32(const PagedView &kv, const float *q, size_t n_heads, const int32_t *starts, size_t n_tokens, float scale, PagedMask mask, float *out,
                                 void *ws, cudaStream_t st);
int32_t launch_paged_prefill_tc(const PagedView &kv, int type, const void *q, int q_type, size_t n_heads, const int32_t *starts, size_t n_tokens, float scale,
                                PagedMask mask, void *out, void *ws, cudaStream_t st);
int32_t launch_paged_prefill(const PagedView &kv, int type, const void *q, int q_type, size_t n_heads, const int32_t *starts, size_t n_tokens, float scale,
                             PagedMask mask, void *out, void *ws, cudaStream_t st);
int32_t launch_paged_evict(const PagedView &kv, int type, const float *weights, const int32_t *positions, size_t track_stride, size_t budget, uint32_t n_sink,
                           uint32_t n_recent, float *weights_out, int32_t *positions_out, size_t out_stride, int32_t *kept, int32_t *lens_out,
                           cudaStream_t st);

}  // namespace cera
