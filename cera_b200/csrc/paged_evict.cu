// Eviction from a paged cache by accumulated attention weight.
//
// paged_pick_kernel, a CTA per (sequence, KV head), finds the budget's largest keys - a protected slot's is above every weight's - by
// four passes over 8 bits each from the top (radix selection: the histogram of the next 8 bits among the slots that agree with the
// threshold so far), ties going to the lower slot; then pairs the gaps below the budget with the kept slots past it, in ascending order.
// paged_move_kernel copies the rows.  A gap's number is below the budget and its source's is not, so no row is both read and written
// and the copies need no order.
//
// The keys are kept in shared memory where they fit and formed again from the weights and positions otherwise.
#include <algorithm>

#include "paged.cuh"

namespace cera {

namespace {

constexpr int PICK_THREADS = 1024, PICK_WARPS = PICK_THREADS / 32;
constexpr uint32_t PICK_WORDS = 56 * 1024;  // of shared memory: the keys, and the slots that move

// Ascending in the weight; a NaN is the smallest, both zeros are alike.  0xffffffff is left for protected slots.
__device__ __forceinline__ uint32_t weight_key(float w) {
    if (!(w == w)) return 0;
    const uint32_t b = __float_as_uint(w + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// Exclusive sums over the CTA of two counts below 2^31 each; `total` receives the sums of all.
__device__ __forceinline__ uint2 cta_scan(uint2 v, uint2 *warps, uint2 &total) {
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint2 x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t a = __shfl_up_sync(0xffffffffu, x.x, o), b = __shfl_up_sync(0xffffffffu, x.y, o);
        if (lane >= (uint32_t)o) {
            x.x += a;
            x.y += b;
        }
    }
    __syncthreads();
    if (lane == 31) warps[warp] = x;
    __syncthreads();
    uint2 w = warps[lane], t = w;  // PICK_WARPS == 32
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t a = __shfl_up_sync(0xffffffffu, t.x, o), b = __shfl_up_sync(0xffffffffu, t.y, o);
        if (lane >= (uint32_t)o) {
            t.x += a;
            t.y += b;
        }
    }
    total = make_uint2(__shfl_sync(0xffffffffu, t.x, 31), __shfl_sync(0xffffffffu, t.y, 31));
    const uint2 before = make_uint2(__shfl_sync(0xffffffffu, t.x - w.x, warp), __shfl_sync(0xffffffffu, t.y - w.y, warp));
    return make_uint2(before.x + x.x - v.x, before.y + x.y - v.y);
}

// A thread owns `per` slots in a row; per is odd, so that the threads of a warp meet different banks.
template <bool SMEM>
__global__ void __launch_bounds__(PICK_THREADS) paged_pick_kernel(const PagedView kv, const float *weights, const int32_t *positions, size_t stride, uint32_t budget,
                                                                  uint32_t n_sink, uint32_t n_recent, float *weights_out, int32_t *positions_out, size_t out_stride,
                                                                  int32_t *kept) {
    extern __shared__ uint32_t keys[];
    __shared__ uint32_t hist[256];
    __shared__ uint2 warps[PICK_WARPS];
    __shared__ int32_t newest_of[PICK_WARPS];
    __shared__ uint32_t s_prefix, s_left;
    pdl_trigger();
    pdl_wait();
    const uint32_t tid = threadIdx.x, lane = tid & 31, s = blockIdx.x / kv.hk;
    const size_t at = blockIdx.x;
    const float *w = weights + at * stride;
    const int32_t *pos = positions + at * stride;
    float *wo = weights_out + at * out_stride;
    int32_t *po = positions_out + at * out_stride, *ko = kept + at * budget;
    const uint32_t len = paged_len(kv, s);
    for (uint32_t j = tid; j < budget; j += PICK_THREADS) ko[j] = j < len ? (int32_t)j : -1;
    if (len <= budget) {
        for (uint32_t j = tid; j < len; j += PICK_THREADS) {
            wo[j] = w[j];
            po[j] = pos[j];
        }
        return;
    }
    int32_t newest = INT32_MIN;
    for (uint32_t j = tid; j < len; j += PICK_THREADS) newest = max(newest, pos[j]);
    newest = __reduce_max_sync(0xffffffffu, newest);
    if (lane == 0) newest_of[tid >> 5] = newest;
    if (tid == 0) {
        s_prefix = 0;
        s_left = budget;
    }
    __syncthreads();
    newest = __reduce_max_sync(0xffffffffu, newest_of[lane]);
    auto form = [&](uint32_t j) {
        const int64_t p = pos[j];
        return p < (int64_t)n_sink || p > (int64_t)newest - (int64_t)n_recent ? 0xffffffffu : weight_key(w[j]);
    };
    if (SMEM) {
        for (uint32_t j = tid; j < len; j += PICK_THREADS) keys[j] = form(j);
        __syncthreads();
    }
    auto key = [&](uint32_t j) { return SMEM ? keys[j] : form(j); };
    // the budget-th largest key: its bits from the top
    for (int shift = 24; shift >= 0; shift -= 8) {
        if (tid < 256) hist[tid] = 0;
        __syncthreads();
        const uint32_t prefix = s_prefix, mask = shift == 24 ? 0 : 0xffffffffu << (shift + 8);
        for (uint32_t j = tid; j < len; j += PICK_THREADS) {
            const uint32_t k = key(j);
            if ((k & mask) == prefix) atomicAdd(&hist[k >> shift & 255], 1);
        }
        __syncthreads();
        if (tid < 32) {
            // lane i holds bins [248 - 8 i, 256 - 8 i): how many are in higher bins
            uint32_t mine = 0;
#pragma unroll
            for (int b = 0; b < 8; ++b) mine += hist[255 - lane * 8 - b];
            uint32_t x = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t a = __shfl_up_sync(0xffffffffu, x, o);
                if (lane >= (uint32_t)o) x += a;
            }
            const uint32_t left = s_left;
            uint32_t above = x - mine;
            if (above < left && left <= x) {  // one lane
                for (int b = 0; b < 8; ++b) {
                    const uint32_t bin = 255 - lane * 8 - b, n = hist[bin];
                    if (above + n >= left) {
                        s_prefix = prefix | bin << shift;
                        s_left = left - above;
                        break;
                    }
                    above += n;
                }
            }
        }
        __syncthreads();
    }
    const uint32_t cut = s_prefix, ties = s_left;  // every key above `cut` is kept, and the first `ties` of those equal to it
    const uint32_t per = (len + PICK_THREADS - 1) / PICK_THREADS | 1, j0 = min(tid * per, len), j1 = min(j0 + per, len);
    uint2 n = make_uint2(0, 0), total;
    for (uint32_t j = j0; j < j1; ++j) n.x += key(j) == cut;
    const uint32_t eq0 = cta_scan(n, warps, total).x;
    auto keeps = [&](uint32_t k, uint32_t &equal) { return k > cut || (k == cut && equal++ < ties); };  // equal: those ahead of the slot
    uint32_t eq = eq0;
    n = make_uint2(0, 0);  // gaps, movers
    for (uint32_t j = j0; j < j1; ++j) {
        const bool keep = keeps(key(j), eq);
        n.x += !keep && j < budget;
        n.y += keep && j >= budget;
    }
    const uint2 first = cta_scan(n, warps, total);
    // every mover's slot by its rank: a list in shared memory past the keys; without keys there, the count ahead of each thread's slots
    uint32_t *list = SMEM ? keys + len : keys;
    if (SMEM) {
        uint32_t i = first.y;
        eq = eq0;
        for (uint32_t j = j0; j < j1; ++j) {
            const uint32_t k = key(j);
            if (keeps(k, eq) && j >= budget) list[i++] = j;
        }
    } else {
        list[tid] = first.y;
        list[PICK_THREADS + tid] = eq0;
    }
    __syncthreads();
    uint32_t i = first.x;
    eq = eq0;
    for (uint32_t j = j0; j < min(j1, budget); ++j) {
        if (keeps(key(j), eq)) continue;
        if (SMEM) {
            ko[j] = (int32_t)list[i];
        } else {
            uint32_t lo = 0, hi = PICK_THREADS;  // the last thread with list[.] <= i owns the slot
            while (hi - lo > 1) {
                const uint32_t mid = (lo + hi) / 2;
                if (list[mid] <= i) lo = mid;
                else hi = mid;
            }
            uint32_t seen = list[lo], e = list[PICK_THREADS + lo], x = lo * per;
            for (;; ++x)
                if (keeps(key(x), e) && x >= budget && seen++ == i) break;
            ko[j] = (int32_t)x;
        }
        ++i;
    }
    __syncthreads();
    for (uint32_t j = tid; j < budget; j += PICK_THREADS) {  // in place too: a source is its own slot, or past the budget
        const uint32_t src = (uint32_t)ko[j];
        wo[j] = w[src];
        po[j] = pos[src];
    }
}

// A warp per slot below the budget; where the slot's content comes from another, it copies the key's and the value's row.
__global__ void __launch_bounds__(256) paged_move_kernel(const PagedView kv, uint32_t row_bytes, uint32_t budget, const int32_t *__restrict__ kept, int32_t *lens_out) {
    pdl_trigger();
    pdl_wait();
    const uint32_t lane = threadIdx.x & 31, s = blockIdx.y / kv.hk, h = blockIdx.y - s * kv.hk;
    if (blockIdx.x == 0 && h == 0 && threadIdx.x == 0) lens_out[s] = (int32_t)min(paged_len(kv, s), budget);
    const int32_t *ko = kept + (size_t)blockIdx.y * budget;
    for (uint32_t j = blockIdx.x * 8 + (threadIdx.x >> 5); j < budget; j += gridDim.x * 8) {
        const int32_t src = ko[j];
        if (src < 0 || (uint32_t)src == j) continue;
        uint32_t r0, r1;
        const uint32_t p0 = paged_at(kv, s, (uint32_t)src, r0), p1 = paged_at(kv, s, j, r1);
        if (p0 == NO_PAGE || p1 == NO_PAGE) continue;
        const uint8_t *ks = kv.k + p0 * kv.k_page + r0 * kv.k_slot + h * kv.k_head, *vs = kv.v + p0 * kv.v_page + r0 * kv.v_slot + h * kv.v_head;
        uint8_t *kd = kv.k + p1 * kv.k_page + r1 * kv.k_slot + h * kv.k_head, *vd = kv.v + p1 * kv.v_page + r1 * kv.v_slot + h * kv.v_head;
        for (uint32_t b = lane * 16; b < 2 * row_bytes; b += 512) {
            const bool is_v = b >= row_bytes;
            const uint32_t o = is_v ? b - row_bytes : b;
            *reinterpret_cast<uint4 *>((is_v ? vd : kd) + o) = *reinterpret_cast<const uint4 *>((is_v ? vs : ks) + o);
        }
    }
}

}  // namespace

int32_t launch_paged_evict(const PagedView &kv, int type, const float *weights, const int32_t *positions, size_t track_stride, size_t budget, uint32_t n_sink,
                           uint32_t n_recent, float *weights_out, int32_t *positions_out, size_t out_stride, int32_t *kept, int32_t *lens_out,
                           cudaStream_t st) {
    const size_t cap = (size_t)kv.max_pages * kv.page_size, movers = cap > budget ? std::min(budget, cap - budget) : 0;
    const bool smem = cap + movers <= PICK_WORDS;
    auto pick = smem ? paged_pick_kernel<true> : paged_pick_kernel<false>;
    const size_t bytes = 4 * (smem ? cap + movers : 2 * (size_t)PICK_THREADS);
    CERA_CUDA_TRY(cudaFuncSetAttribute(pick, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(4 * PICK_WORDS)));
    count_launch(2);
    CERA_CUDA_TRY(launch_k(pick, dim3(kv.n_seqs * kv.hk), dim3(PICK_THREADS), bytes, st, kv, weights, positions, track_stride, (uint32_t)budget, n_sink, n_recent,
                           weights_out, positions_out, out_stride, kept));
    const uint32_t pairs = kv.n_seqs * kv.hk, wide = (uint32_t)std::min<size_t>((budget + 7) / 8, std::max<size_t>(1, 148 * 8 / pairs));
    return check_cuda(launch_k(paged_move_kernel, dim3(wide, pairs), dim3(256), 0, st, kv, kv.dim * (type == CERA_TYPE_F32 ? 4u : 2u), (uint32_t)budget, (const int32_t *)kept, lens_out),
                      "paged evict launch");
}

}  // namespace cera
