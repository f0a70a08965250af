// Eviction from a paged cache by accumulated attention weight.
//
// paged_pick_kernel, a CTA per (sequence, KV head), finds the budget's largest keys - a protected slot's is above every weight's - by
// three passes over 11, 11 and 10 bits from the top (radix selection: the histogram of the next bits among the slots that agree with the
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
constexpr uint32_t PICK_BINS = 2048;
constexpr uint32_t PICK_WORDS = 54 * 1024;  // of shared memory: the keys, and the slots that move

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

// Loads that do not wait for one another: f(j, first[j], second[j]) for j = tid, tid + PICK_THREADS ...
template <typename F>
__device__ __forceinline__ void each_slot(const float *w, const int32_t *pos, uint32_t len, F f) {
    constexpr int U = 8;
    for (uint32_t j = threadIdx.x; j < len; j += U * PICK_THREADS) {
        float a[U];
        int32_t b[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t i = j + u * PICK_THREADS;
            a[u] = w && i < len ? w[i] : 0.0f;
            b[u] = i < len ? pos[i] : 0;
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (j + u * PICK_THREADS < len) f(j + u * PICK_THREADS, a[u], b[u]);
    }
}

constexpr uint32_t MOVE_SLOTS = 16;
// A warp's MOVE_SLOTS slots from j0 on, a lane each with where its slot's content comes from (negative: nowhere): copies the key's and the value's row of those
// that come from another slot, four at a time whose lookups and rows do not wait for one another.
__device__ __forceinline__ void move_slots(const PagedView &kv, uint32_t s, uint32_t h, uint32_t row_bytes, uint32_t j0, int32_t from) {
    constexpr int U = 4;
    const uint32_t lane = threadIdx.x & 31, mine = j0 + lane;
    uint32_t moved = __ballot_sync(0xffffffffu, from >= 0 && (uint32_t)from != mine);
    while (moved) {
        // lanes 0 to 3 look up the sources, 4 to 7 where they go
        uint32_t i = 32, rest = moved;
        for (uint32_t u = 0; u < (lane & 3) && rest; ++u) rest &= rest - 1;
        if (rest) i = __ffs(rest) - 1;
        const int32_t src = __shfl_sync(0xffffffffu, from, i & 31);
        uint32_t row = 0, page = NO_PAGE;
        if (lane < 8 && i < 32) page = paged_at(kv, s, lane < 4 ? (uint32_t)src : j0 + i, row);
        for (int u = 0; u < U && moved; ++u) moved &= moved - 1;
        uint32_t live = __ballot_sync(0xffffffffu, page != NO_PAGE);
        live &= live >> 4 & 15;
        if (!live) continue;
        const uint8_t *from_k[U], *from_v[U];
        uint8_t *to_k[U], *to_v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint64_t p0 = __shfl_sync(0xffffffffu, page, u), r0 = __shfl_sync(0xffffffffu, row, u), p1 = __shfl_sync(0xffffffffu, page, u + 4), r1 = __shfl_sync(0xffffffffu, row, u + 4);
            from_k[u] = kv.k + p0 * kv.k_page + r0 * kv.k_slot + h * kv.k_head;
            from_v[u] = kv.v + p0 * kv.v_page + r0 * kv.v_slot + h * kv.v_head;
            to_k[u] = kv.k + p1 * kv.k_page + r1 * kv.k_slot + h * kv.k_head;
            to_v[u] = kv.v + p1 * kv.v_page + r1 * kv.v_slot + h * kv.v_head;
        }
        for (uint32_t b = lane * 16; b < 2 * row_bytes; b += 512) {
            const bool is_v = b >= row_bytes;
            const uint32_t o = is_v ? b - row_bytes : b;
            uint4 x[U];
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (live >> u & 1) x[u] = *reinterpret_cast<const uint4 *>((is_v ? from_v[u] : from_k[u]) + o);
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (live >> u & 1) *reinterpret_cast<uint4 *>((is_v ? to_v[u] : to_k[u]) + o) = x[u];
        }
    }
}

// With SMEM a thread owns `per` < 64 slots in a row, of which a 64-bit word each says which are kept; per is odd, so that the threads of a warp meet different
// banks.
template <bool SMEM, bool MOVE>
__global__ void __launch_bounds__(PICK_THREADS) paged_pick_kernel(const PagedView kv, const float *weights, const int32_t *positions, size_t stride, uint32_t budget,
                                                                  uint32_t n_sink, uint32_t n_recent, float *weights_out, int32_t *positions_out, size_t out_stride,
                                                                  int32_t *kept, uint32_t row_bytes, int32_t *lens_out) {
    extern __shared__ uint32_t keys[];
    __shared__ uint32_t hist[PICK_BINS];
    __shared__ uint2 warps[PICK_WARPS];
    __shared__ int32_t newest_of[PICK_WARPS];
    __shared__ uint32_t sums[PICK_WARPS], s_prefix, s_left;
    pdl_trigger();
    pdl_wait();
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, s = blockIdx.x / kv.hk;
    const size_t at = blockIdx.x;
    const float *w = weights + at * stride;
    const int32_t *pos = positions + at * stride;
    float *wo = weights_out + at * out_stride;
    int32_t *po = positions_out + at * out_stride, *ko = kept + at * budget;
    const uint32_t len = paged_len(kv, s);
    if (MOVE && blockIdx.x == s * kv.hk && tid == 0) lens_out[s] = (int32_t)min(len, budget);
    for (uint32_t j = tid; j < budget; j += PICK_THREADS) ko[j] = j < len ? (int32_t)j : -1;
    if (len <= budget) {
        for (uint32_t j = tid; j < len; j += PICK_THREADS) {
            wo[j] = w[j];
            po[j] = pos[j];
        }
        return;
    }
    int32_t newest = INT32_MIN;
    each_slot(SMEM ? w : nullptr, pos, len, [&](uint32_t j, float a, int32_t b) {
        newest = max(newest, b);
        if (SMEM) keys[j] = weight_key(a);
    });
    newest = __reduce_max_sync(0xffffffffu, newest);
    if (lane == 0) newest_of[warp] = newest;
    for (uint32_t i = tid; i < PICK_BINS; i += PICK_THREADS) hist[i] = 0;
    if (tid == 0) {
        s_prefix = 0;
        s_left = budget;
    }
    __syncthreads();
    newest = __reduce_max_sync(0xffffffffu, newest_of[lane]);
    auto safe = [&](int64_t p) { return p < (int64_t)n_sink || p > (int64_t)newest - (int64_t)n_recent; };
    auto key = [&](uint32_t j) { return SMEM ? keys[j] : safe(pos[j]) ? 0xffffffffu : weight_key(w[j]); };
    // the budget-th largest key: its bits from the top, eleven, eleven and ten
    for (int shift = 21; shift >= 0; shift -= shift == 10 ? 10 : 11) {
        const uint32_t prefix = s_prefix, mask = shift == 21 ? 0 : 0xffffffffu << (shift == 10 ? 21 : 10), bins = shift == 0 ? 1024 : 2048;
        auto count = [&](uint32_t k) {
            if ((k & mask) == prefix) atomicAdd(&hist[k >> shift & (bins - 1)], 1);
        };
        if (SMEM && shift == 21) {  // the slots' own pass: thread by thread the ones it wrote
            each_slot(nullptr, pos, len, [&](uint32_t j, float, int32_t b) {
                if (safe(b)) keys[j] = 0xffffffffu;
                count(keys[j]);
            });
        } else {
            for (uint32_t j = tid; j < len; j += PICK_THREADS) count(key(j));
        }
        __syncthreads();
        // from the top a warp has bins / 32 of them, a lane one or two
        const uint32_t top = bins - 1 - warp * (bins / 32), n0 = hist[bins == 2048 ? top - 2 * lane : top - lane], n1 = bins == 2048 ? hist[top - 2 * lane - 1] : 0;
        uint32_t x = n0 + n1;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t a = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= (uint32_t)o) x += a;
        }
        if (lane == 31) sums[warp] = x;
        const uint32_t left = s_left;
        __syncthreads();
        for (uint32_t i = tid; i < PICK_BINS; i += PICK_THREADS) hist[i] = 0;
        uint32_t before = 0;
        for (uint32_t i = lane; i < warp; i += 32) before += sums[i];
        before = __reduce_add_sync(0xffffffffu, before) + x - n0 - n1;  // in higher bins
        if (before < left && left <= before + n0 + n1) {  // one thread
            const bool second = left > before + n0;
            s_prefix = prefix | (bins == 2048 ? top - 2 * lane - second : top - lane) << shift;
            s_left = left - before - (second ? n0 : 0);
        }
        __syncthreads();
    }
    const uint32_t cut = s_prefix, ties = s_left;  // every key above `cut` is kept, and the first `ties` of those equal to it
    const uint32_t per = (len + PICK_THREADS - 1) / PICK_THREADS | 1, j0 = min(tid * per, len), j1 = min(j0 + per, len);
    uint2 total;
    if (SMEM) {
        uint64_t keep = 0, equal = 0;
        for (uint32_t j = j0; j < j1; ++j) {
            const uint32_t k = keys[j];
            keep |= (uint64_t)(k > cut) << (j - j0);
            equal |= (uint64_t)(k == cut) << (j - j0);
        }
        const uint32_t eq0 = cta_scan(make_uint2(__popcll(equal), 0), warps, total).x;
        uint32_t more = eq0 < ties ? min(ties - eq0, (uint32_t)__popcll(equal)) : 0;
        if (more == (uint32_t)__popcll(equal)) keep |= equal;
        else
            for (; more; --more, equal &= equal - 1) keep |= equal & -equal;
        const uint64_t mine = j1 - j0 >= 64 ? ~0ull : (1ull << (j1 - j0)) - 1, below = budget <= j0 ? 0 : budget - j0 >= 64 ? ~0ull : (1ull << (budget - j0)) - 1;
        uint64_t gaps = ~keep & mine & below, movers = keep & ~below;
        uint2 i = cta_scan(make_uint2(__popcll(gaps), __popcll(movers)), warps, total);
        uint32_t *list = keys + len;  // every mover's slot by its rank
        for (; movers; movers &= movers - 1) list[i.y++] = j0 + __ffsll(movers) - 1;
        __syncthreads();
        for (; gaps; gaps &= gaps - 1) ko[j0 + __ffsll(gaps) - 1] = (int32_t)list[i.x++];
    } else {
        auto keeps = [&](uint32_t k, uint32_t &equal) { return k > cut || (k == cut && equal++ < ties); };  // equal: those ahead of the slot
        uint2 n = make_uint2(0, 0);
        for (uint32_t j = j0; j < j1; ++j) n.x += key(j) == cut;
        const uint32_t eq0 = cta_scan(n, warps, total).x;
        uint32_t eq = eq0;
        n = make_uint2(0, 0);  // gaps, movers
        for (uint32_t j = j0; j < j1; ++j) {
            const bool keep = keeps(key(j), eq);
            n.x += !keep && j < budget;
            n.y += keep && j >= budget;
        }
        const uint2 first = cta_scan(n, warps, total);
        uint32_t *list = keys;  // the count of movers ahead of each thread's slots, and of keys equal to the cut
        list[tid] = first.y;
        list[PICK_THREADS + tid] = eq0;
        __syncthreads();
        uint32_t i = first.x;
        eq = eq0;
        for (uint32_t j = j0; j < min(j1, budget); ++j) {
            if (keeps(key(j), eq)) continue;
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
            ++i;
        }
    }
    __syncthreads();
    // in place too: a source is its own slot, or past the budget
    constexpr int U = 4;
    for (uint32_t j = tid; j < budget; j += U * PICK_THREADS) {
        float a[U];
        int32_t b[U];
        uint32_t src[U];
#pragma unroll
        for (int u = 0; u < U; ++u) src[u] = j + u * PICK_THREADS < budget ? (uint32_t)ko[j + u * PICK_THREADS] : 0;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            a[u] = w[src[u]];
            b[u] = pos[src[u]];
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (j + u * PICK_THREADS < budget) {
                wo[j + u * PICK_THREADS] = a[u];
                po[j + u * PICK_THREADS] = b[u];
            }
    }
    if (MOVE)
        for (uint32_t j = warp * MOVE_SLOTS; j < budget; j += PICK_WARPS * MOVE_SLOTS)
            move_slots(kv, s, blockIdx.x - s * kv.hk, row_bytes, j, lane < MOVE_SLOTS && j + lane < budget ? ko[j + lane] : -1);
}

// A warp per MOVE_SLOTS slots below the budget.
__global__ void __launch_bounds__(256) paged_move_kernel(const PagedView kv, uint32_t row_bytes, uint32_t budget, const int32_t *__restrict__ kept, int32_t *lens_out) {
    pdl_trigger();
    pdl_wait();
    const uint32_t s = blockIdx.y / kv.hk, h = blockIdx.y - s * kv.hk;
    if (blockIdx.x == 0 && h == 0 && threadIdx.x == 0) lens_out[s] = (int32_t)min(paged_len(kv, s), budget);
    const uint32_t lane = threadIdx.x & 31, j0 = (blockIdx.x * 8 + (threadIdx.x >> 5)) * MOVE_SLOTS;
    move_slots(kv, s, h, row_bytes, j0, lane < MOVE_SLOTS && j0 + lane < budget ? kept[(size_t)blockIdx.y * budget + j0 + lane] : -1);
}

}  // namespace

int32_t launch_paged_evict(const PagedView &kv, int type, const float *weights, const int32_t *positions, size_t track_stride, size_t budget, uint32_t n_sink,
                           uint32_t n_recent, float *weights_out, int32_t *positions_out, size_t out_stride, int32_t *kept, int32_t *lens_out,
                           cudaStream_t st) {
    const size_t cap = (size_t)kv.max_pages * kv.page_size, movers = cap > budget ? std::min(budget, cap - budget) : 0;
    const bool smem = cap + movers <= PICK_WORDS;
    // few slots that can move: the CTA that picks them moves them, unless the lengths that all CTAs of a sequence read are overwritten (8 sequences of 2049 slots and 8
    // heads: FUSED_A us with a second launch, FUSED_B without)
    const bool move = smem && movers <= PICK_THREADS && (lens_out + kv.n_seqs <= kv.lens || kv.lens + kv.n_seqs <= lens_out);
    auto pick = move ? paged_pick_kernel<true, true> : smem ? paged_pick_kernel<true, false> : paged_pick_kernel<false, false>;
    const size_t bytes = 4 * (smem ? cap + movers : 2 * (size_t)PICK_THREADS);
    if (smem) CERA_TRY((move ? paged_smem<paged_pick_kernel<true, true>>(4 * PICK_WORDS) : paged_smem<paged_pick_kernel<true, false>>(4 * PICK_WORDS)));
    const uint32_t row_bytes = kv.dim * (type == CERA_TYPE_F32 ? 4u : 2u), pairs = kv.n_seqs * kv.hk;
    count_launch();
    CERA_CUDA_TRY(launch_k(pick, dim3(pairs), dim3(PICK_THREADS), bytes, st, kv, weights, positions, track_stride, (uint32_t)budget, n_sink, n_recent, weights_out,
                           positions_out, out_stride, kept, row_bytes, lens_out));
    if (move) return CERA_CUDA_OK;
    const uint32_t wide = (uint32_t)((std::min(budget, cap) + 8 * MOVE_SLOTS - 1) / (8 * MOVE_SLOTS));
    count_launch();
    return check_cuda(launch_k(paged_move_kernel, dim3(std::max(1u, wide), pairs), dim3(256), 0, st, kv, row_bytes, (uint32_t)budget, (const int32_t *)kept, lens_out),
                      "paged evict launch");
}

}  // namespace cera
