// Eviction from a paged cache by accumulated attention weight.
//
// paged_pick_kernel, a cluster of CTAs per (sequence, KV head) and each with a slice of the slots, finds the budget's largest keys - a protected slot's is above every
// weight's - by passes over 11, 11 and 10 bits from the top (radix selection: the histogram of the next bits among the slots that agree with the threshold so far), ties
// going to the lower slot; then pairs the gaps below the budget with the kept slots past it, in ascending order.  A slice's keys stay in shared memory.
// paged_move_kernel copies the rows.  A gap's number is below the budget and its source's is not, so no row is both read and written
// and the copies need no order.
#include <algorithm>

#include "paged.cuh"
#include "tc.cuh"

namespace cera {

namespace {

constexpr int PICK_THREADS = 1024, PICK_WARPS = PICK_THREADS / 32;
constexpr uint32_t PICK_BINS = 2048;
constexpr int PICK_CTAS = 8;  // of a cluster, at most
constexpr uint32_t PICK_SLICE = 2048;  // slots that are worth a CTA more
constexpr uint32_t PICK_WORDS = 52 * 1024;  // of shared memory: the keys

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
// A lane each: the slot `to` and the slot its content comes from (negative: nowhere).  Copies the key's and the value's row of those that come from another slot, four at a
// time whose lookups and rows do not wait for one another.
__device__ __forceinline__ void move_slots(const PagedView &kv, uint32_t s, uint32_t h, uint32_t row_bytes, uint32_t to, int32_t from) {
    constexpr int U = 4;
    const uint32_t lane = threadIdx.x & 31;
    uint32_t moved = __ballot_sync(0xffffffffu, from >= 0 && (uint32_t)from != to);
    while (moved) {
        // lanes 0 to 3 look up the sources, 4 to 7 where they go
        uint32_t i = 32, rest = moved;
        for (uint32_t u = 0; u < (lane & 3) && rest; ++u) rest &= rest - 1;
        if (rest) i = __ffs(rest) - 1;
        const uint32_t src = (uint32_t)__shfl_sync(0xffffffffu, from, i & 31), dst = __shfl_sync(0xffffffffu, to, i & 31);
        uint32_t row = 0, page = NO_PAGE;
        if (lane < 8 && i < 32) page = paged_at(kv, s, lane < 4 ? src : dst, row);
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

// ---- a cluster's CTAs share one pair's slots ----
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
// A word of that CTA's shared memory (this one's without clusters).
template <bool CLUSTER>
__device__ __forceinline__ uint32_t of_rank(const uint32_t *p, uint32_t rank) {
    if (!CLUSTER) return *p;
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(tma::smem_of_rank(p, rank)) : "memory");
    return v;
}
// The sum of the first `ranks` CTAs' words; the loads do not wait for one another.
template <bool CLUSTER>
__device__ __forceinline__ uint32_t of_ranks(const uint32_t *p, uint32_t ranks) {
    if (!CLUSTER) return ranks ? *p : 0;
    uint32_t v[PICK_CTAS], sum = 0;
#pragma unroll
    for (int r = 0; r < PICK_CTAS; ++r) v[r] = (uint32_t)r < ranks ? of_rank<true>(p, r) : 0;
#pragma unroll
    for (int r = 0; r < PICK_CTAS; ++r) sum += v[r];
    return sum;
}
template <bool CLUSTER>
__device__ __forceinline__ void pick_barrier() {
    __syncwarp();
    if (CLUSTER) cluster_barrier();
    else __syncthreads();
}
__device__ __forceinline__ uint32_t warp_scan(uint32_t x) {  // inclusive
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t a = __shfl_up_sync(0xffffffffu, x, o);
        if ((threadIdx.x & 31) >= (uint32_t)o) x += a;
    }
    return x;
}
// The lowest `n` bits of 32.
__device__ __forceinline__ uint32_t low_bits(uint32_t n) { return n >= 32 ? 0xffffffffu : (1u << n) - 1; }

// A cluster per pair and a slice of its slots per CTA.  Histograms stay where they are counted: every CTA's first warp adds up their sums of 64 bins each, then the 64
// bins that matter (all bins of four CTAs read by each of them took 3400 clocks a round).  A warp has `wide` <= 64 words of 32 slots of the slice, whose
// kept ones it finds by ballots.  The kept slots past the budget are handed to the gaps by the CTAs that have them, since these are spread evenly.
template <bool CLUSTER, bool MOVE>
__global__ void __launch_bounds__(PICK_THREADS) paged_pick_kernel(const PagedView kv, const float *weights, const int32_t *positions, size_t stride, uint32_t budget,
                                                                  uint32_t n_sink, uint32_t n_recent, float *weights_out, int32_t *positions_out, size_t out_stride,
                                                                  int32_t *kept, uint32_t row_bytes, int32_t *lens_out) {
    extern __shared__ uint32_t keys[];  // and then, by rank, the slots of the slice's gaps, and of the kept ones past the budget
    __shared__ uint32_t hist[2][PICK_BINS], coarse[2][PICK_WARPS];
    __shared__ uint2 warps[PICK_WARPS], mine_s;
    __shared__ int32_t newest_of[PICK_WARPS];
    __shared__ uint32_t newest_s, equals[PICK_WARPS], equal_s, s_prefix, s_left, s_count;
    pdl_trigger();
    pdl_wait();
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rank = CLUSTER ? cluster_rank() : 0, ctas = CLUSTER ? cluster_size() : 1, pair = blockIdx.x / ctas, s = pair / kv.hk;
    const size_t at = pair;
    const float *w = weights + at * stride;
    const int32_t *pos = positions + at * stride;
    float *wo = weights_out + at * out_stride;
    int32_t *po = positions_out + at * out_stride, *ko = kept + at * budget;
    const uint32_t len = paged_len(kv, s), slice = (len + ctas - 1) / ctas, a0 = min(rank * slice, len), n = min(slice, len - a0);
    if (MOVE && pair == s * kv.hk && rank == 0 && tid == 0) lens_out[s] = (int32_t)min(len, budget);
    if (len <= budget) {  // all CTAs of the cluster
        for (uint32_t j = rank * PICK_THREADS + tid; j < budget; j += ctas * PICK_THREADS) {
            ko[j] = j < len ? (int32_t)j : -1;
            if (j < len) {
                wo[j] = w[j];
                po[j] = pos[j];
            }
        }
        return;
    }
    // every slot below the budget as if it stayed; the first batch's positions stay in registers
    constexpr int U = 8;
    int32_t held[U], newest = INT32_MIN;
    for (uint32_t base = 0; base < n; base += U * PICK_THREADS) {
        float a[U];
        int32_t b[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t j = base + u * PICK_THREADS + tid;
            a[u] = j < n ? w[a0 + j] : 0.0f;
            b[u] = j < n ? pos[a0 + j] : INT32_MIN;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t j = base + u * PICK_THREADS + tid;
            newest = max(newest, b[u]);
            if (base == 0) held[u] = b[u];
            if (j < n) keys[j] = weight_key(a[u]);
            if (j < n && a0 + j < budget) {
                ko[a0 + j] = (int32_t)(a0 + j);
                wo[a0 + j] = a[u];
                po[a0 + j] = b[u];
            }
        }
    }
    newest = __reduce_max_sync(0xffffffffu, newest);
    if (lane == 0) newest_of[warp] = newest;
    for (uint32_t i = tid; i < 2 * PICK_BINS; i += PICK_THREADS) hist[0][i] = 0;
    __syncthreads();
    if (warp == 0) {
        newest = __reduce_max_sync(0xffffffffu, newest_of[lane]);
        if (lane == 0) newest_s = (uint32_t)newest;
    }
    pick_barrier<CLUSTER>();
    newest = __reduce_max_sync(0xffffffffu, (int32_t)of_rank<CLUSTER>(&newest_s, lane % ctas));
    // protected: position < n_sink or position > newest - n_recent, in 32 bits that cannot pass their ends
    const bool all_recent = (int64_t)newest - (int64_t)n_recent < INT32_MIN;
    const int32_t recent = all_recent ? INT32_MIN : (int32_t)((int64_t)newest - (int64_t)n_recent);
    const int32_t sinks = (int32_t)min(n_sink, (uint32_t)INT32_MAX);
    // the budget-th largest key: its bits from the top, eleven, eleven and ten
    uint32_t prefix = 0, left = budget, turn = 0;
    bool all = false;  // keys equal to `prefix` in its bits so far are all kept
    for (int shift = 21; shift >= 0 && !all; shift -= shift == 10 ? 10 : 11, turn ^= 1) {
        const uint32_t mask = shift == 21 ? 0 : 0xffffffffu << (shift == 10 ? 21 : 10), bits = shift == 0 ? 1023 : 2047;
        uint32_t *h = hist[turn];
        auto count = [&](uint32_t k) {
            if ((k & mask) == prefix) atomicAdd(&h[k >> shift & bits], 1);
        };
        if (shift == 21) {  // the slots' own pass: thread by thread the ones it wrote
            for (uint32_t base = 0; base < n; base += U * PICK_THREADS) {
                int32_t b[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const uint32_t j = base + u * PICK_THREADS + tid;
                    b[u] = base == 0 ? held[u] : j < n ? pos[a0 + j] : 0;
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const uint32_t j = base + u * PICK_THREADS + tid;
                    if (j >= n) break;
                    uint32_t k = keys[j];
                    if (b[u] < sinks || b[u] > recent || all_recent) keys[j] = k = 0xffffffffu;
                    count(k);
                }
            }
        } else {
            for (uint32_t j = tid; j < n; j += PICK_THREADS) count(keys[j]);
        }
        __syncthreads();
        // from the top a warp has 64 bins, a lane two
        const uint32_t i0 = PICK_BINS - 1 - 2 * tid, sum = __reduce_add_sync(0xffffffffu, h[i0] + h[i0 - 1]);
        if (lane == 0) coarse[turn][warp] = sum;
        pick_barrier<CLUSTER>();
        // the other histogram has been read by all CTAs: this pass's barrier is behind that
        if (shift == 10)
            for (uint32_t i = tid; i < PICK_BINS; i += PICK_THREADS) hist[turn ^ 1][i] = 0;
        if (warp == 0) {
            const uint32_t m = of_ranks<CLUSTER>(&coarse[turn][lane], ctas), x = warp_scan(m);  // x - m: in higher bins
            const uint32_t g = __ffs(__ballot_sync(0xffffffffu, x >= left)) - 1, rest = left - __shfl_sync(0xffffffffu, x - m, g);
            const uint32_t f = PICK_BINS - 1 - 64 * g - 2 * lane, n0 = of_ranks<CLUSTER>(&h[f], ctas), n1 = of_ranks<CLUSTER>(&h[f - 1], ctas);
            const uint32_t before = warp_scan(n0 + n1) - n0 - n1;
            if (before < rest && rest <= before + n0 + n1) {  // one lane
                const bool second = rest > before + n0;
                s_prefix = prefix | (f - second) << shift;
                s_left = rest - before - (second ? n0 : 0);
                s_count = second ? n1 : n0;
            }
        }
        __syncthreads();
        prefix = s_prefix;
        left = s_left;
        all = left == s_count;
    }
    // kept are the keys above `prefix` and the first `left` of those equal to it, or all from it on
    const uint32_t words = (n + 31) / 32, wide = (words + PICK_WARPS - 1) / PICK_WARPS, w0 = min(warp * wide, words), w1 = min(w0 + wide, words), lower = (1u << lane) - 1;
    uint32_t eq = 0;  // equal ones ahead of the warp's
    if (!all) {
        for (uint32_t i = w0; i < w1; ++i) eq += __popc(__ballot_sync(0xffffffffu, i * 32 + lane < n && keys[i * 32 + lane] == prefix));
        if (lane == 0) equals[warp] = eq;
        __syncthreads();
        const uint32_t x = warp_scan(equals[lane]);
        if (tid == 31) equal_s = x;
        pick_barrier<CLUSTER>();
        eq = __shfl_sync(0xffffffffu, x, warp) - eq + of_ranks<CLUSTER>(&equal_s, rank);
    }
    uint32_t keep[2] = {0, 0}, gaps = 0, moves = 0;  // words w0 + lane and w0 + 32 + lane
    auto below = [&](uint32_t i) { return low_bits(budget <= a0 + i * 32 ? 0 : budget - a0 - i * 32); };
    for (uint32_t i = w0; i < w1; ++i) {
        const uint32_t j = i * 32 + lane;
        const bool in = j < n;
        const uint32_t k = in ? keys[j] : 0;
        uint32_t stay = __ballot_sync(0xffffffffu, in && (all ? k >= prefix : k > prefix));
        if (!all) {
            const uint32_t same = __ballot_sync(0xffffffffu, in && k == prefix);
            stay |= __ballot_sync(0xffffffffu, (same >> lane & 1) && eq + __popc(same & lower) < left);
            eq += __popc(same);
        }
        gaps += __popc(~stay & low_bits(n - i * 32) & below(i));
        moves += __popc(stay & ~below(i));
        if (i - w0 == lane) keep[0] = stay;
        if (i - w0 == lane + 32) keep[1] = stay;
    }
    if (lane == 0) warps[warp] = make_uint2(gaps, moves);
    __syncthreads();  // the keys have been read
    uint2 total = warps[lane];
    total.x = warp_scan(total.x);
    total.y = warp_scan(total.y);
    gaps = __shfl_sync(0xffffffffu, total.x, warp) - gaps;
    moves = __shfl_sync(0xffffffffu, total.y, warp) - moves;
    total.x = __shfl_sync(0xffffffffu, total.x, 31);
    total.y = __shfl_sync(0xffffffffu, total.y, 31);
    moves += total.x;
    for (uint32_t i = w0; i < w1; ++i) {
        const uint32_t stay = __shfl_sync(0xffffffffu, i - w0 < 32 ? keep[0] : keep[1], (i - w0) & 31), gap = ~stay & low_bits(n - i * 32) & below(i), move = stay & ~below(i);
        if (gap >> lane & 1) keys[gaps + __popc(gap & lower)] = a0 + i * 32 + lane;
        if (move >> lane & 1) keys[moves + __popc(move & lower)] = a0 + i * 32 + lane;
        gaps += __popc(gap);
        moves += __popc(move);
    }
    if (tid == 0) mine_s = total;
    pick_barrier<CLUSTER>();
    const uint32_t ends = warp_scan(lane < ctas ? of_rank<CLUSTER>(&mine_s.x, lane) : 0);  // of the ranks' gaps
    const uint32_t first = __reduce_add_sync(0xffffffffu, lane + 1 <= rank ? of_rank<CLUSTER>(&mine_s.y, lane) : 0);
    constexpr uint32_t CHUNK = MOVE ? 4 : 32;  // a warp's at a time; with rows to move, few
    for (uint32_t m0 = warp * CHUNK; m0 < total.y; m0 += PICK_WARPS * CHUNK) {
        const bool in = lane < CHUNK && m0 + lane < total.y;
        const uint32_t i = first + m0 + lane;
        uint32_t r = 0, ahead = 0;
        for (uint32_t q = 0; q + 1 < ctas; ++q) {
            const uint32_t end = __shfl_sync(0xffffffffu, ends, q);
            if (i >= end) {
                r = q + 1;
                ahead = end;
            }
        }
        uint32_t gap = 0;
        int32_t from = -1;
        if (in) {
            from = (int32_t)keys[total.x + m0 + lane];
            gap = of_rank<CLUSTER>(keys + (i - ahead), r);
            ko[gap] = from;
            wo[gap] = w[from];
            po[gap] = pos[from];
        }
        if (MOVE) move_slots(kv, s, pair - s * kv.hk, row_bytes, gap, from);
    }
    if (CLUSTER) cluster_barrier();  // shared memory is read by others up to here
}

// The same by one CTA a pair, with keys formed again from the weights and positions: for slots that no cluster's shared memory holds.
__global__ void __launch_bounds__(PICK_THREADS) paged_pick_far_kernel(const PagedView kv, const float *weights, const int32_t *positions, size_t stride, uint32_t budget,
                                                                  uint32_t n_sink, uint32_t n_recent, float *weights_out, int32_t *positions_out, size_t out_stride,
                                                                  int32_t *kept) {
    __shared__ uint32_t list[2 * PICK_THREADS];  // the count of movers ahead of each thread's slots, and of keys equal to the cut
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
    for (uint32_t j = tid; j < budget; j += PICK_THREADS) ko[j] = j < len ? (int32_t)j : -1;
    if (len <= budget) {
        for (uint32_t j = tid; j < len; j += PICK_THREADS) {
            wo[j] = w[j];
            po[j] = pos[j];
        }
        return;
    }
    int32_t newest = INT32_MIN;
    each_slot(nullptr, pos, len, [&](uint32_t, float, int32_t b) { newest = max(newest, b); });
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
    auto key = [&](uint32_t j) { return safe(pos[j]) ? 0xffffffffu : weight_key(w[j]); };
    // the budget-th largest key: its bits from the top, eleven, eleven and ten
    for (int shift = 21; shift >= 0; shift -= shift == 10 ? 10 : 11) {
        const uint32_t prefix = s_prefix, mask = shift == 21 ? 0 : 0xffffffffu << (shift == 10 ? 21 : 10), bins = shift == 0 ? 1024 : 2048;
        auto count = [&](uint32_t k) {
            if ((k & mask) == prefix) atomicAdd(&hist[k >> shift & (bins - 1)], 1);
        };
        each_slot(w, pos, len, [&](uint32_t, float a, int32_t b) { count(safe(b) ? 0xffffffffu : weight_key(a)); });
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
        for (; x + 1 < len; ++x)
            if (keeps(key(x), e) && x >= budget && seen++ == i) break;
        ko[j] = (int32_t)x;
        ++i;
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
}

// A warp per MOVE_SLOTS slots below the budget, a row of CTAs per pair.
__global__ void __launch_bounds__(256) paged_move_kernel(const PagedView kv, uint32_t row_bytes, uint32_t budget, const int32_t *__restrict__ kept, int32_t *lens_out) {
    pdl_trigger();
    pdl_wait();
    const uint32_t s = blockIdx.x / kv.hk, h = blockIdx.x - s * kv.hk, lane = threadIdx.x & 31;
    if (blockIdx.y == 0 && h == 0 && threadIdx.x == 0) lens_out[s] = (int32_t)min(paged_len(kv, s), budget);
    for (uint32_t j0 = (blockIdx.y * 8 + (threadIdx.x >> 5)) * MOVE_SLOTS; j0 < budget; j0 += gridDim.y * 8 * MOVE_SLOTS)
        move_slots(kv, s, h, row_bytes, j0 + lane, lane < MOVE_SLOTS && j0 + lane < budget ? kept[(size_t)blockIdx.x * budget + j0 + lane] : -1);
}

}  // namespace

int32_t launch_paged_evict(const PagedView &kv, int type, const float *weights, const int32_t *positions, size_t track_stride, size_t budget, uint32_t n_sink,
                           uint32_t n_recent, float *weights_out, int32_t *positions_out, size_t out_stride, int32_t *kept, int32_t *lens_out,
                           cudaStream_t st) {
    const size_t cap = (size_t)kv.max_pages * kv.page_size, movers = cap > budget ? std::min(budget, cap - budget) : 0;
    const uint32_t row_bytes = kv.dim * (type == CERA_TYPE_F32 ? 4u : 2u), pairs = kv.n_seqs * kv.hk;
    // CTAs a pair: as many as the SMs have room for and have PICK_SLICE slots each, more where the shared memory of fewer does not hold them.  Eight only on half of the SMs: no GPC
    // has room for many clusters of eight, and 16 of them take two turns (2 sequences of 32000 slots and 8 heads: 45 us with eight, 35 with four, 44 with two; one of 30000: 28
    // with eight, 30 with four, 37 with two, 45 with one).
    auto words = [&](size_t ctas) { return (cap + ctas - 1) / ctas; };
    auto room = [&](uint32_t ctas) { return ctas * pairs <= (uint32_t)sm_count() / (ctas == 8 ? 2 : 1) && cap / ctas >= PICK_SLICE; };
    uint32_t ctas = 1;
    while (ctas < PICK_CTAS && (room(2 * ctas) || words(ctas) > PICK_WORDS)) ctas *= 2;
    const bool smem = words(ctas) <= PICK_WORDS;
    // few slots that can move: the CTAs that pick them move them, unless the lengths that all CTAs of a sequence read are overwritten (8 sequences of 2049 slots and 8
    // heads: 11 us with a second launch, 9.7 without)
    const bool move = smem && movers <= PICK_THREADS && (lens_out + kv.n_seqs <= kv.lens || kv.lens + kv.n_seqs <= lens_out);
    count_launch();
    if (smem) {
        auto go = [&](auto cluster, auto moves) {
            constexpr bool C = decltype(cluster)::value, M = decltype(moves)::value;
            CERA_TRY((paged_smem<paged_pick_kernel<C, M>>(4 * PICK_WORDS)));
            return check_cuda(launch_clusters(paged_pick_kernel<C, M>, ctas, pairs, dim3(PICK_THREADS), 4 * words(ctas), st, kv, weights, positions, track_stride, (uint32_t)budget, n_sink,
                                              n_recent, weights_out, positions_out, out_stride, kept, row_bytes, lens_out),
                              "paged evict launch");
        };
        using Yes = std::true_type;
        using No = std::false_type;
        CERA_TRY(ctas > 1 ? move ? go(Yes(), Yes()) : go(Yes(), No()) : move ? go(No(), Yes()) : go(No(), No()));
    } else {
        CERA_CUDA_TRY(launch_k(paged_pick_far_kernel, dim3(pairs), dim3(PICK_THREADS), 0, st, kv, weights, positions, track_stride, (uint32_t)budget, n_sink, n_recent, weights_out,
                               positions_out, out_stride, kept));
    }
    if (move) return CERA_CUDA_OK;
    const size_t wide = (std::min(budget, cap) + 8 * MOVE_SLOTS - 1) / (8 * MOVE_SLOTS);
    count_launch();
    return check_cuda(launch_k(paged_move_kernel, dim3(pairs, (uint32_t)std::min<size_t>(std::max<size_t>(1, wide), 65535)), dim3(256), 0, st, kv, row_bytes, (uint32_t)budget,
                               (const int32_t *)kept, lens_out),
                      "paged evict launch");
}

}  // namespace cera
