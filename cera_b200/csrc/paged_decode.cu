// Attention of one new token per sequence over a paged cache: o = sum_j p_j v_j, p = softmax(scale q k_j), for every query head.
//
// Every visible key and value is read once for all the query heads of its KV head - eight at a time, more take another pass - so the cache's
// bytes bound a large call.  The visible slots of all (sequence, KV head, eight heads) units are cut into tiles, and the tiles of the whole call are
// dealt out evenly in one line: CTA b has tiles [b T / G, (b + 1) T / G), whatever the sequences' lengths, and at most its first and its
// last unit are shared with others.  What a CTA knows of a shared unit (maximum, sum, weighted values) goes to the workspace, whose size
// therefore does not depend on the lengths; paged_join_kernel adds the parts up in their order, so a call's bits do not depend on timing.
//
// A warp walks its own keys of each tile - 16 of 64 over a 16-bit cache, 8 of 32 over f32 - through a ring of its own in shared memory
// (cp.async, 16 bytes a lane), with a running maximum, sum and weighted values of its own; warps meet at a unit's end only.  The maximum
// is raised when a score has passed it by 2^8 (a vote, no exchange), to which the weights' range is fitted.
//
// 16-bit cache: mma.sync, 16 rows = eight heads twice: the upper half of each query and weight as the type has it, and what that leaves,
// so an f32 query or weight counts with 22 bits (f16) in the same instructions; bf16's 16 bits are too few for an f32 query, whose third
// part takes a second product.  An f16 part is scaled by a power of two per query, weights by 2^7, so that what f16 cannot tell from zero is 2^-32
// of the largest weight.
// f32 cache: FMAs, four lanes a key for the scores, a lane 4 dimensions of every head for the values.
//
// With weights wanted the scaled scores are stored on the way (4 bytes a head and slot, beside the 2 dim that are read for it), and
// paged_weigh_kernel turns them into probabilities once the denominators are known.
#include <algorithm>

#include "mma.cuh"
#include "paged.cuh"

namespace cera {

namespace {

constexpr int PD_WARPS = 4, PD_THREADS = 32 * PD_WARPS, PD_ROWS = 8;
constexpr float PD_FLOOR = -3.0e38f;    // below every score that is a number
constexpr float PD_LIFT = 7.0f;         // weights are 2^7 at the maximum's score, 2^15 at most
constexpr float PD_RAISE = 8.0f;

struct PdParams {
    PagedView kv;
    PagedMask mask;
    const void *q;
    void *out;
    float *part;    // [2 G][8][dim]
    float2 *ml;     // [2 G][8]: maximum, sum; then, with weights, [units][8]
    float *scores;  // [seqs][heads][capacity] or null
    float2 *ml_unit;
    size_t cap;
    float scale;
    uint32_t heads, group, chunks;  // chunks of eight heads in a group
    bool same;                      // keys and values are laid out alike
};

// The tiles of the call in one line; sums live in shared memory.
struct PdLine {
    const uint32_t *sums;  // visible tiles ahead of sequence s, of one unit each; sums[n] is all
    uint32_t n, per_seq;   // units of a sequence
};

template <int KG>
struct PdCursor {
    uint32_t s, unit, tile, tiles, first, sinks, seen;

    __device__ __forceinline__ void sequence(const PdLine &line, const PagedView &kv, const PagedMask &mask) {
        tiles = line.sums[s + 1] - line.sums[s];
        const uint32_t len = paged_len(kv, s);
        first = len ? paged_first(mask, len - 1) : 0;
        sinks = min(mask.sink, first);
        seen = len - first + sinks;
    }
    __device__ __forceinline__ void seek(const PdLine &line, const PagedView &kv, const PagedMask &mask, uint64_t x) {
        uint32_t lo = 0, hi = line.n;  // the last s with sums[s] per_seq <= x, which has tiles
        while (hi - lo > 1) {
            const uint32_t mid = (lo + hi) / 2;
            if ((uint64_t)line.sums[mid] * line.per_seq <= x) lo = mid;
            else hi = mid;
        }
        s = lo;
        sequence(line, kv, mask);
        const uint64_t r = x - (uint64_t)line.sums[s] * line.per_seq;
        unit = tiles ? (uint32_t)(r / tiles) : 0;
        tile = tiles ? (uint32_t)(r - (uint64_t)unit * tiles) : 0;
    }
    __device__ __forceinline__ void step(const PdLine &line, const PagedView &kv, const PagedMask &mask) {
        if (++tile < tiles) return;
        tile = 0;
        if (++unit < line.per_seq) return;
        unit = 0;
        do ++s;
        while (s + 1 < line.n && line.sums[s + 1] == line.sums[s]);
        if (s < line.n) sequence(line, kv, mask);
    }
    __device__ __forceinline__ uint32_t slot(uint32_t x) const { return x < sinks ? x : x - sinks + first; }
};

__device__ __forceinline__ void cp_async16_or_zero(void *dst, const void *src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(tma::smem_u32(dst)), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ float pd_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The tiles ahead of each sequence, by the whole CTA.
template <int KG>
__device__ __forceinline__ PdLine pd_line(const PagedView &kv, const PagedMask &mask, uint32_t per_seq, uint32_t *sums, uint32_t *warps) {
    const uint32_t tid = threadIdx.x, lane = tid & 31, per = (kv.n_seqs + PD_THREADS - 1) / PD_THREADS, s0 = min(tid * per, kv.n_seqs), s1 = min(s0 + per, kv.n_seqs);
    uint32_t mine = 0;
    for (uint32_t s = s0; s < s1; ++s) {
        const uint32_t len = paged_len(kv, s), first = len ? paged_first(mask, len - 1) : 0;
        mine += (len - first + min(mask.sink, first) + PD_WARPS * KG - 1) / (PD_WARPS * KG);
        sums[s + 1] = mine;
    }
    uint32_t x = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t a = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= (uint32_t)o) x += a;
    }
    if (lane == 31) warps[tid >> 5] = x;
    if (tid == 0) sums[0] = 0;
    __syncthreads();
    uint32_t before = x - mine;
    for (uint32_t w = 0; w < tid >> 5; ++w) before += warps[w];
    for (uint32_t s = s0; s < s1; ++s) sums[s + 1] += before;
    __syncthreads();
    return PdLine{sums, kv.n_seqs, per_seq};
}

// ---- what a warp does with its keys of a tile ------------------------------------------------------------------------------

// 16-bit cache.  Lane = (row lane / 4, columns 2 (lane % 4) + {0, 1}) of an mma tile; acc's second half is the lower parts'.
template <typename T, typename TQ, int DP>
struct PdMma {
    static constexpr int KG = 16, ROWB = DP * 2 + 16, CPR = DP / 8, QREGS = 1;
    static constexpr bool SPLIT = sizeof(TQ) == 4, BF = sizeof(T) == 2 && !std::is_same<T, __half>::value, THIRD = SPLIT && BF;
    uint32_t qf[DP / 16][SPLIT ? 4 : 2], q3[THIRD ? DP / 16 : 1][2];
    float acc[DP / 8][4], m, l, factor;

    static __device__ __forceinline__ void split(float x, float y, uint32_t &hi, uint32_t &lo) {
        if (BF) split_bf16(x, y, hi, lo);
        else split_f16(x, y, hi, lo);
    }
    static __device__ __forceinline__ float2 unpack(uint32_t w) {
        return BF ? __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&w)) : __half22float2(*reinterpret_cast<const __half2 *>(&w));
    }
    static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
        if (BF) mma_bf16(c, a, b0, b1);
        else mma_f16(c, a, b0, b1);
    }
    // what hi and lo leave of (x, y)
    static __device__ __forceinline__ uint32_t third(float x, float y, uint32_t hi, uint32_t lo) {
        const float2 h = unpack(hi), w = unpack(lo);
        uint32_t a, b;
        split(x - h.x - w.x, y - h.y - w.y, a, b);
        return a;
    }

    __device__ __forceinline__ void begin(const PdParams &p, uint32_t s, uint32_t head0, uint32_t rows, float *) {
        const uint32_t lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
        const TQ *q = reinterpret_cast<const TQ *>(p.q) + ((size_t)s * p.heads + head0 + r) * p.kv.dim + 2 * c;
        const bool live = r < rows;
        factor = p.scale * PAGED_LOG2E;
        if (!SPLIT) {
#pragma unroll
            for (int k = 0; k < DP / 16; ++k)
#pragma unroll
                for (int i = 0; i < 2; ++i) qf[k][i] = live && k * 16 < p.kv.dim ? *reinterpret_cast<const uint32_t *>(q + k * 16 + 8 * i) : 0;
        } else {
            float x[DP / 16][4];
            float most = 0.0f;
#pragma unroll
            for (int k = 0; k < DP / 16; ++k)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float2 v = live && k * 16 < p.kv.dim ? *reinterpret_cast<const float2 *>(reinterpret_cast<const float *>(q) + k * 16 + 8 * i) : make_float2(0.0f, 0.0f);
                    x[k][2 * i] = v.x;
                    x[k][2 * i + 1] = v.y;
                    most = fmaxf(most, fmaxf(fabsf(v.x), fabsf(v.y)));
                }
            if (!BF) {
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
                // by a power of two to [1, 2); what a float's exponent cannot hold twice over goes in two steps
                const int e = most > 0.0f && most <= 3.4e38f ? min(max((int)(__float_as_uint(most) >> 23 & 255) - 127, -120), 120) : 0;
                const float down = __uint_as_float((uint32_t)(127 - e) << 23);
                factor *= __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll
                for (int k = 0; k < DP / 16; ++k)
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[k][i] *= down;
            }
#pragma unroll
            for (int k = 0; k < DP / 16; ++k)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    split(x[k][2 * i], x[k][2 * i + 1], qf[k][i], qf[k][2 + i]);
                    if (THIRD) q3[k][i] = third(x[k][2 * i], x[k][2 * i + 1], qf[k][i], qf[k][2 + i]);
                }
        }
#pragma unroll
        for (int n = 0; n < DP / 8; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[n][i] = 0.0f;
        m = PD_FLOOR;
        l = 0.0f;
    }

    // ks, vs: 16 rows each; mask: which are seen; scores: the first of these keys' places for head 0 of the unit, or null
    __device__ __forceinline__ void tile(const PdParams &p, const uint8_t *ks, const uint8_t *vs, uint32_t mask, uint32_t rows, float *scores, uint32_t count, float *, float *) {
        const uint32_t lane = threadIdx.x & 31, r = lane >> 2, c2 = 2 * (lane & 3);
        float sc[2][4] = {};
        const uint8_t *ka = ks + ((lane & 7) + (lane >> 4) * 8) * ROWB + (lane >> 3 & 1) * 16;
#pragma unroll
        for (int k = 0; k < DP / 16; ++k) {
            if (k * 16 >= p.kv.dim) break;
            uint32_t b[4];
            ldsm4(b, ka + k * 32);
            const uint32_t a[4] = {qf[k][0], SPLIT ? qf[k][SPLIT ? 2 : 0] : 0u, qf[k][1], SPLIT ? qf[k][SPLIT ? 3 : 1] : 0u};
            mma(sc[0], a, b[0], b[1]);
            mma(sc[1], a, b[2], b[3]);
            if (THIRD) {
                const uint32_t a3[4] = {q3[THIRD ? k : 0][0], 0u, q3[THIRD ? k : 0][1], 0u};
                mma(sc[0], a3, b[0], b[1]);
                mma(sc[1], a3, b[2], b[3]);
            }
        }
        float z[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float hi = sc[i >> 1][i & 1], both = hi + sc[i >> 1][(i & 1) + 2];
            z[i] = (SPLIT && !(fabsf(both) < INFINITY) ? hi : both) * factor;  // of an infinite key the upper part says it all
        }
        if (mask != 0xffffu) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (!(mask >> (c2 + (i & 1) + (i >> 1) * 8) & 1)) z[i] = -INFINITY;
        }
        if (scores && r < rows) {
            float *to = scores + (size_t)r * p.cap + c2;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (c2 + (i & 1) + (i >> 1) * 8 < count) to[(i & 1) + (i >> 1) * 8] = z[i];
        }
        float mx = fmaxf(fmaxf(z[0], z[1]), fmaxf(z[2], z[3]));
        if (__any_sync(0xffffffffu, mx > m + PD_RAISE)) {
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            if (mx > m + PD_RAISE) {
                const float f = pd_exp2(m - mx);
                m = mx;
                l *= f;
#pragma unroll
                for (int n = 0; n < DP / 8; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[n][i] *= f;
            }
        }
        const float base = PD_LIFT - m;
        float w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = pd_exp2(z[i] + base);
        l += (w[0] + w[1]) + (w[2] + w[3]);
        uint32_t a[4], a3[4] = {0, 0, 0, 0};
        split(w[0], w[1], a[0], a[1]);
        split(w[2], w[3], a[2], a[3]);
        if (THIRD) {
            a3[0] = third(w[0], w[1], a[0], a[1]);
            a3[2] = third(w[2], w[3], a[2], a[3]);
        }
        const uint8_t *va = vs + (lane & 15) * ROWB + (lane >> 4) * 16;
#pragma unroll
        for (int n = 0; n < DP / 16; ++n) {
            if (n * 16 >= p.kv.dim) break;
            uint32_t b[4];
            ldsm4_trans(b, va + n * 32);
            mma(acc[2 * n], a, b[0], b[1]);
            mma(acc[2 * n + 1], a, b[2], b[3]);
            if (THIRD) {
                mma(acc[2 * n], a3, b[0], b[1]);
                mma(acc[2 * n + 1], a3, b[2], b[3]);
            }
        }
    }

    // maxima and sums of the warp's rows
    __device__ __forceinline__ void end(float2 *ml) {
        const uint32_t lane = threadIdx.x & 31;
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        if ((lane & 3) == 0) ml[lane >> 2] = make_float2(m, l);
    }
    // the weighted values for the maxima `all` of each row, [8][dim]
    __device__ __forceinline__ void values(const PdParams &p, const float *all, float *to) {
        const uint32_t lane = threadIdx.x & 31, r = lane >> 2;
        const float f = pd_exp2(m - all[r]);
#pragma unroll
        for (int n = 0; n < DP / 8; ++n)
            if (n * 8 < p.kv.dim) {
                float2 o;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float hi = acc[n][i], both = hi + acc[n][i + 2];
                    (i ? o.y : o.x) = (fabsf(both) < INFINITY ? both : hi) * f;
                }
                *reinterpret_cast<float2 *>(to + r * p.kv.dim + n * 8 + 2 * (lane & 3)) = o;
            }
    }
};

// f32 cache.  Scores: lane = (key lane / 4, every fourth 16 bytes of the row), then two heads of that key.  Values: lane = 4 dimensions.
template <int DP>
struct PdFma {
    static constexpr int KG = 8, ROWB = DP * 4 + 64, CPR = DP / 4, NV = (DP + 127) / 128;
    float4 acc[PD_ROWS][NV];
    float m[2], l[2];  // of heads 2 (lane % 4) + {0, 1}; l over this lane's keys

    __device__ __forceinline__ void begin(const PdParams &p, uint32_t s, uint32_t head0, uint32_t rows, float *qs) {
        const uint32_t lane = threadIdx.x & 31;
        const float *q = reinterpret_cast<const float *>(p.q) + ((size_t)s * p.heads + head0) * p.kv.dim;
        __syncwarp();
        for (uint32_t i = lane; i < PD_ROWS * DP; i += 32) {
            const uint32_t r = i / DP, d = i % DP;
            qs[i] = r < rows && d < p.kv.dim ? q[r * p.kv.dim + d] : 0.0f;
        }
        __syncwarp();
#pragma unroll
        for (int r = 0; r < PD_ROWS; ++r)
#pragma unroll
            for (int i = 0; i < NV; ++i) acc[r][i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        m[0] = m[1] = PD_FLOOR;
        l[0] = l[1] = 0.0f;
    }

    __device__ __forceinline__ void tile(const PdParams &p, const uint8_t *ks, const uint8_t *vs, uint32_t mask, uint32_t rows, float *scores, uint32_t count, float *qs, float *ps) {
        const uint32_t lane = threadIdx.x & 31, key = lane >> 2, part = lane & 3;
        float2 d2[PD_ROWS];
#pragma unroll
        for (int r = 0; r < PD_ROWS; ++r) d2[r] = make_float2(0.0f, 0.0f);
#pragma unroll 4
        for (uint32_t c = part; c < p.kv.dim / 4; c += 4) {
            const float4 k = *reinterpret_cast<const float4 *>(ks + key * ROWB + c * 16);
#pragma unroll
            for (int r = 0; r < PD_ROWS; ++r) {
                const float4 q = *reinterpret_cast<const float4 *>(qs + r * DP + c * 4);
                d2[r] = __ffma2_rn(make_float2(k.x, k.y), make_float2(q.x, q.y), d2[r]);
                d2[r] = __ffma2_rn(make_float2(k.z, k.w), make_float2(q.z, q.w), d2[r]);
            }
        }
        float d[PD_ROWS];
#pragma unroll
        for (int r = 0; r < PD_ROWS; ++r) d[r] = d2[r].x + d2[r].y;
        // sums over the four lanes of a key; lane `part` keeps heads 2 part, 2 part + 1
        const bool up2 = part & 2, up1 = part & 1;
        float h4[4], z[2];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float give = up2 ? d[i] : d[4 + i], keep = up2 ? d[4 + i] : d[i];
            h4[i] = keep + __shfl_xor_sync(0xffffffffu, give, 2);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float give = up1 ? h4[i] : h4[2 + i], keep = up1 ? h4[2 + i] : h4[i];
            z[i] = (keep + __shfl_xor_sync(0xffffffffu, give, 1)) * (p.scale * PAGED_LOG2E);
        }
        if (!(mask >> key & 1)) z[0] = z[1] = -INFINITY;
        if (scores && key < count) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
                if (2 * part + i < rows) scores[(size_t)(2 * part + i) * p.cap + key] = z[i];
        }
        if (__any_sync(0xffffffffu, z[0] > m[0] + PD_RAISE || z[1] > m[1] + PD_RAISE)) {
            float f[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float mx = z[i];
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                f[i] = 1.0f;
                if (mx > m[i] + PD_RAISE) {
                    f[i] = pd_exp2(m[i] - mx);
                    m[i] = mx;
                    l[i] *= f[i];
                }
            }
#pragma unroll
            for (int r = 0; r < PD_ROWS; ++r) {
                const float g = __shfl_sync(0xffffffffu, f[r & 1], r >> 1);
#pragma unroll
                for (int i = 0; i < NV; ++i) acc[r][i] = make_float4(acc[r][i].x * g, acc[r][i].y * g, acc[r][i].z * g, acc[r][i].w * g);
            }
        }
        float2 w;
        w.x = pd_exp2(z[0] + (PD_LIFT - m[0]));
        w.y = pd_exp2(z[1] + (PD_LIFT - m[1]));
        l[0] += w.x;
        l[1] += w.y;
        *reinterpret_cast<float2 *>(ps + key * PD_ROWS + 2 * part) = w;
        __syncwarp();
#pragma unroll
        for (int k = 0; k < KG; ++k) {
            const float4 w0 = *reinterpret_cast<const float4 *>(ps + k * PD_ROWS), w1 = *reinterpret_cast<const float4 *>(ps + k * PD_ROWS + 4);
            const float ww[PD_ROWS] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                if ((lane + 32 * i) * 4 >= p.kv.dim) break;
                const float4 v = *reinterpret_cast<const float4 *>(vs + k * ROWB + (lane + 32 * i) * 16);
#pragma unroll
                for (int r = 0; r < PD_ROWS; ++r) {
                    const float2 wr = make_float2(ww[r], ww[r]);
                    const float2 lo = __ffma2_rn(wr, make_float2(v.x, v.y), make_float2(acc[r][i].x, acc[r][i].y));
                    const float2 hi = __ffma2_rn(wr, make_float2(v.z, v.w), make_float2(acc[r][i].z, acc[r][i].w));
                    acc[r][i] = make_float4(lo.x, lo.y, hi.x, hi.y);
                }
            }
        }
        __syncwarp();  // the weights' place is written by the next tile
    }

    __device__ __forceinline__ void end(float2 *ml) {
        const uint32_t lane = threadIdx.x & 31;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 4);
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 8);
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 16);
            if (lane < 4) ml[2 * lane + i] = make_float2(m[i], l[i]);
        }
    }
    __device__ __forceinline__ void values(const PdParams &p, const float *all, float *to) {
        const uint32_t lane = threadIdx.x & 31;
#pragma unroll
        for (int r = 0; r < PD_ROWS; ++r) {
            const float f = pd_exp2(__shfl_sync(0xffffffffu, m[r & 1], r >> 1) - all[r]);
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if ((lane + 32 * i) * 4 < p.kv.dim)
                    *reinterpret_cast<float4 *>(to + r * p.kv.dim + (lane + 32 * i) * 4) = make_float4(acc[r][i].x * f, acc[r][i].y * f, acc[r][i].z * f, acc[r][i].w * f);
        }
    }
};

template <typename T, typename TQ, int DP>
struct PdOf {
    using W = PdMma<T, TQ, DP>;
};
template <int DP>
struct PdOf<float, float, DP> {
    using W = PdFma<DP>;
};

// Shared memory: rings | values of the warps at a unit's end | queries and weights (f32) | the line's sums.
template <typename W, int DP, int ST, bool FMA>
struct PdSmem {
    static constexpr size_t STAGE = 2 * (size_t)W::KG * W::ROWB, RING = ST * STAGE, VALUES = (size_t)PD_WARPS * PD_ROWS * DP * 4,
                            EXTRA = FMA ? PD_WARPS * (size_t)(PD_ROWS * DP + PD_ROWS * W::KG) * 4 : 0, FIXED = PD_WARPS * RING + VALUES + EXTRA;
};

template <typename T, typename TQ, int DP, int ST>
__global__ void __launch_bounds__(PD_THREADS) paged_decode_kernel(const PdParams p) {
    using W = typename PdOf<T, TQ, DP>::W;
    constexpr bool FMA = sizeof(T) == 4;
    using S = PdSmem<W, DP, ST, FMA>;
    constexpr int KG = W::KG, CPR = W::CPR;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float2 ml_s[PD_WARPS][PD_ROWS];
    __shared__ float all_s[PD_ROWS], sum_s[PD_ROWS];
    __shared__ uint32_t mask_s[PD_WARPS][ST], scan_s[PD_WARPS], any_s[PD_WARPS];
    pdl_trigger();
    pdl_wait();
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, G = gridDim.x, b = blockIdx.x;
    uint8_t *ring = smem + warp * S::RING;
    float *values = reinterpret_cast<float *>(smem + PD_WARPS * S::RING);
    float *qs = values + PD_WARPS * PD_ROWS * DP + warp * (PD_ROWS * DP + PD_ROWS * KG), *ps = qs + PD_ROWS * DP;
    const uint32_t per_seq = p.kv.hk * p.chunks;
    const PdLine line = pd_line<KG>(p.kv, p.mask, per_seq, reinterpret_cast<uint32_t *>(smem + S::FIXED), scan_s);
    const uint64_t total = (uint64_t)line.sums[line.n] * per_seq, x0 = b * total / G, x1 = (b + 1) * total / G;
    if (x0 >= x1) return;
    PdCursor<KG> at, ahead;
    at.seek(line, p.kv, p.mask, x0);
    ahead = at;

    // the row that this lane looks up for the tile at the cursor
    auto find = [&](const PdCursor<KG> &c, uint32_t &page, uint32_t &row) {
        const uint32_t x = (c.tile * PD_WARPS + warp) * KG + lane;
        page = NO_PAGE;
        row = 0;
        if (lane < KG && x < c.seen) page = paged_at(p.kv, c.s, c.slot(x), row);
    };
    uint32_t page, row;
    find(ahead, page, row);
    uint64_t next = x0;
    auto load = [&]() {
        if (next < x1) {
            const uint32_t st = (uint32_t)(next - x0) % ST;
            uint8_t *kd = ring + st * S::STAGE, *vd = kd + KG * W::ROWB;
            const uint32_t h = ahead.unit / p.chunks;
            const bool there = page != NO_PAGE;
            const uint64_t ko = there ? page * (uint64_t)p.kv.k_page + row * (uint64_t)p.kv.k_slot + h * (uint64_t)p.kv.k_head : 0;
            const uint64_t vo = there ? page * (uint64_t)p.kv.v_page + row * (uint64_t)p.kv.v_slot + h * (uint64_t)p.kv.v_head : 0;
            const uint32_t mask = __ballot_sync(0xffffffffu, there);
            if (lane == 0) mask_s[warp][st] = mask;
            ++next;
            ahead.step(line, p.kv, p.mask);
            if (next < x1) find(ahead, page, row);  // its answer is not needed before the next call
#pragma unroll
            for (int i = 0; i < KG * CPR / 32; ++i) {
                const uint32_t idx = i * 32 + lane, r = idx / CPR, c = idx % CPR;
                const uint64_t k1 = __shfl_sync(0xffffffffu, ko, r), v1 = p.same ? k1 : __shfl_sync(0xffffffffu, vo, r);
                if (c * 16 < p.kv.dim * sizeof(T)) {
                    const bool seen = mask >> r & 1;
                    cp_async16_or_zero(kd + r * W::ROWB + c * 16, p.kv.k + k1 + (seen ? c * 16 : 0), seen);
                    cp_async16_or_zero(vd + r * W::ROWB + c * 16, p.kv.v + v1 + (seen ? c * 16 : 0), seen);
                }
            }
        }
        cp_async_commit();
    };
#pragma unroll
    for (int i = 0; i < ST; ++i) load();

    W w;
    uint32_t any = 0, first_tile = at.tile;
    uint32_t rows = 0, head0 = 0;
    for (uint64_t x = x0; x < x1; ++x) {
        if (x == x0 || at.tile == 0) {
            const uint32_t h = at.unit / p.chunks, c = at.unit - h * p.chunks;
            head0 = h * p.group + c * PD_ROWS;
            rows = min(p.group - c * PD_ROWS, (uint32_t)PD_ROWS);
            first_tile = at.tile;
            any = 0;
            w.begin(p, at.s, head0, rows, qs);
        }
        const uint32_t st = (uint32_t)(x - x0) % ST, g0 = (at.tile * PD_WARPS + warp) * KG;
        cp_async_wait<ST - 1>();
        __syncwarp();
        const uint32_t mask = mask_s[warp][st];
        const uint8_t *ks = ring + st * S::STAGE;
        any |= mask;
        const uint32_t count = g0 < at.seen ? min(at.seen - g0, (uint32_t)KG) : 0;
        if (mask || (p.scores && count))
            w.tile(p, ks, ks + KG * W::ROWB, mask, rows, p.scores ? p.scores + ((size_t)at.s * p.heads + head0) * p.cap + g0 : nullptr, count, qs, ps);
        __syncwarp();
        load();
        const bool last = at.tile + 1 == at.tiles;
        if (last || x + 1 == x1) {
            // the warps' shares of the unit
            w.end(ml_s[warp]);
            if (lane == 0) any_s[warp] = any;
            __syncthreads();
            if (tid < PD_ROWS) {
                float m = ml_s[0][tid].x, l = 0.0f;
                for (int i = 1; i < PD_WARPS; ++i) m = fmaxf(m, ml_s[i][tid].x);
                for (int i = 0; i < PD_WARPS; ++i) l += ml_s[i][tid].y * pd_exp2(ml_s[i][tid].x - m);
                all_s[tid] = m;
                sum_s[tid] = l;
            }
            const bool seen = any_s[0] | any_s[1] | any_s[2] | any_s[3];
            __syncthreads();
            w.values(p, all_s, values + warp * PD_ROWS * p.kv.dim);
            __syncthreads();
            const bool whole = last && first_tile == 0;
            const uint32_t slot = 2 * b + (x + 1 == x1 && x0 + (at.tile - first_tile) != x);  // the first unit of this CTA, or another, which is its last
            const uint32_t n = PD_ROWS * p.kv.dim, unit = at.s * per_seq + at.unit;
            for (uint32_t i = tid * 4; i < n; i += PD_THREADS * 4) {
                float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int k = 0; k < PD_WARPS; ++k) {
                    const float4 v = *reinterpret_cast<const float4 *>(values + k * n + i);
                    o = make_float4(o.x + v.x, o.y + v.y, o.z + v.z, o.w + v.w);
                }
                const uint32_t r = i / p.kv.dim;
                if (whole) {
                    if (r < rows) {
                        TQ *to = reinterpret_cast<TQ *>(p.out) + ((size_t)at.s * p.heads + head0) * p.kv.dim + i;
                        const float f = sum_s[r];
                        to[0] = from_f32<TQ>(seen ? o.x / f : 0.0f);
                        to[1] = from_f32<TQ>(seen ? o.y / f : 0.0f);
                        to[2] = from_f32<TQ>(seen ? o.z / f : 0.0f);
                        to[3] = from_f32<TQ>(seen ? o.w / f : 0.0f);
                    }
                } else {
                    *reinterpret_cast<float4 *>(p.part + (size_t)slot * n + i) = o;
                }
            }
            if (tid < PD_ROWS) {
                const float2 v = make_float2(seen ? all_s[tid] : -INFINITY, sum_s[tid]);
                if (!whole) p.ml[(size_t)slot * PD_ROWS + tid] = v;
                else if (p.scores) p.ml_unit[(size_t)unit * PD_ROWS + tid] = v;
            }
            __syncthreads();
        }
        at.step(line, p.kv, p.mask);
    }
    cp_async_wait<0>();
}

// A CTA per (unit, row): units without tiles are zeros, whole ones are done, the others' parts are added up.
template <typename TQ, int KG>
__global__ void __launch_bounds__(PD_THREADS) paged_join_kernel(const PdParams p, uint32_t G) {
    __shared__ uint32_t before_s[PD_WARPS], all_s[PD_WARPS], first_s;
    pdl_trigger();
    pdl_wait();
    const uint32_t per_seq = p.kv.hk * p.chunks, unit = blockIdx.x, s = unit / per_seq, u = unit - s * per_seq, r = blockIdx.y, tid = threadIdx.x;
    const uint32_t h = u / p.chunks, c = u - h * p.chunks, rows = min(p.group - c * PD_ROWS, (uint32_t)PD_ROWS);
    if (r >= rows) return;
    uint32_t before = 0, all = 0;
    for (uint32_t i = tid; i < p.kv.n_seqs; i += PD_THREADS) {
        const uint32_t len = paged_len(p.kv, i), first = len ? paged_first(p.mask, len - 1) : 0;
        const uint32_t n = (len - first + min(p.mask.sink, first) + PD_WARPS * KG - 1) / (PD_WARPS * KG);
        all += n;
        if (i < s) before += n;
        if (i == s) first_s = n;
    }
    before = __reduce_add_sync(0xffffffffu, before);
    all = __reduce_add_sync(0xffffffffu, all);
    if ((tid & 31) == 0) {
        before_s[tid >> 5] = before;
        all_s[tid >> 5] = all;
    }
    __syncthreads();
    before = all = 0;
    for (int i = 0; i < PD_WARPS; ++i) {
        before += before_s[i];
        all += all_s[i];
    }
    const uint32_t tiles = first_s;
    TQ *out = reinterpret_cast<TQ *>(p.out) + ((size_t)s * p.heads + h * p.group + c * PD_ROWS + r) * p.kv.dim;
    if (tiles == 0) {
        for (uint32_t d = tid; d < p.kv.dim; d += PD_THREADS) out[d] = from_f32<TQ>(0.0f);
        return;
    }
    const uint64_t total = (uint64_t)all * per_seq, u0 = (uint64_t)before * per_seq + (uint64_t)u * tiles, u1 = u0 + tiles;
    const uint32_t b0 = (uint32_t)(((u0 + 1) * G - 1) / total), b1 = (uint32_t)((u1 * G - 1) / total);  // the CTAs of its first and last tile
    if (b0 == b1) return;
    const uint32_t head = 2 * b0 + (b0 * total / G < u0);  // of the first CTA it may be the last unit
    auto slot = [&](uint32_t b) { return b == b0 ? head : 2 * b; };
    auto empty = [&](uint32_t b) { return b * total / G == (b + 1) * total / G; };
    float m = -INFINITY, l = 0.0f;
    for (uint32_t b = b0; b <= b1; ++b)
        if (!empty(b)) m = fmaxf(m, p.ml[(size_t)slot(b) * PD_ROWS + r].x);
    float o[2] = {0.0f, 0.0f};
    for (uint32_t b = b0; b <= b1; ++b) {
        if (empty(b)) continue;
        const float2 v = p.ml[(size_t)slot(b) * PD_ROWS + r];
        if (v.x == -INFINITY) continue;
        const float f = pd_exp2(v.x - m);
        l += v.y * f;
        const float *part = p.part + ((size_t)slot(b) * PD_ROWS + r) * p.kv.dim;
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (tid + i * PD_THREADS < p.kv.dim) o[i] = fmaf(part[tid + i * PD_THREADS], f, o[i]);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
        if (tid + i * PD_THREADS < p.kv.dim) out[tid + i * PD_THREADS] = from_f32<TQ>(m == -INFINITY ? 0.0f : o[i] / l);
    if (p.scores && tid == 0) p.ml_unit[(size_t)unit * PD_ROWS + r] = make_float2(m, l);
}

// A thread per (sequence, KV head, visible slot): the probabilities of its query heads, in their order, added to the slot's weight.
__global__ void __launch_bounds__(256) paged_weigh_kernel(const PdParams p, float *weights, size_t stride) {
    pdl_trigger();
    pdl_wait();
    const uint32_t s = blockIdx.z, h = blockIdx.y, len = paged_len(p.kv, s);
    if (len == 0) return;
    const uint32_t first = paged_first(p.mask, len - 1), sinks = min(p.mask.sink, first), seen = len - first + sinks;
    const float *scores = p.scores + ((size_t)s * p.heads + h * p.group) * p.cap;
    for (uint32_t x = blockIdx.x * 256 + threadIdx.x; x < seen; x += gridDim.x * 256) {
        float sum = 0.0f;
        for (uint32_t g = 0; g < p.group; ++g) {
            const float2 ml = p.ml_unit[((size_t)(s * p.kv.hk + h) * p.chunks + g / PD_ROWS) * PD_ROWS + g % PD_ROWS];
            const float z = scores[(size_t)g * p.cap + x];
            if (z != -INFINITY) sum += pd_exp2(z - ml.x + PD_LIFT) / ml.y;
        }
        const uint32_t slot = x < sinks ? x : x - sinks + first;
        weights[((size_t)s * p.kv.hk + h) * stride + slot] += sum;
    }
}

uint32_t pd_grid() { return 2 * (uint32_t)sm_count(); }

struct PdLayout {
    size_t part, ml, unit, scores, bytes;
};
PdLayout pd_layout(const PagedView &kv, size_t n_heads, bool weights) {
    const size_t G = pd_grid(), chunks = (n_heads / kv.hk + PD_ROWS - 1) / PD_ROWS;
    PdLayout l;
    l.part = 0;
    l.ml = l.part + 2 * G * PD_ROWS * kv.dim * 4;
    l.unit = l.ml + 2 * G * PD_ROWS * 8;
    l.scores = l.unit + (weights ? kv.n_seqs * kv.hk * chunks * PD_ROWS * 8 : 0);
    l.bytes = l.scores + (weights ? kv.n_seqs * n_heads * kv.max_pages * kv.page_size * 4 : 0) + 16;
    return l;
}

template <typename T, typename TQ, int DP, int ST>
int32_t pd_launch(const PdParams &p, float *weights, size_t weights_stride, cudaStream_t st) {
    using W = typename PdOf<T, TQ, DP>::W;
    const size_t smem = PdSmem<W, DP, ST, sizeof(T) == 4>::FIXED + ((size_t)p.kv.n_seqs + 1) * 4;
    const size_t tiles = (p.cap + PD_WARPS * W::KG - 1) / (PD_WARPS * W::KG) * p.kv.n_seqs * p.kv.hk * p.chunks;
    const uint32_t G = (uint32_t)std::min<size_t>(pd_grid(), std::max<size_t>(tiles, 1));
    auto kernel = paged_decode_kernel<T, TQ, DP, ST>;
    CERA_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    count_launch(weights ? 3 : 2);
    CERA_CUDA_TRY(launch_k(kernel, dim3(G), dim3(PD_THREADS), smem, st, p));
    CERA_CUDA_TRY(launch_k(paged_join_kernel<TQ, W::KG>, dim3(p.kv.n_seqs * p.kv.hk * p.chunks, std::min<uint32_t>(p.group, PD_ROWS)), dim3(PD_THREADS), 0, st, p, G));
    if (!weights) return CERA_CUDA_OK;
    const uint32_t wide = (uint32_t)std::min<size_t>((p.cap + 255) / 256, std::max<size_t>(1, 148 * 8 / std::max(1u, p.kv.n_seqs * p.kv.hk)));
    return check_cuda(launch_k(paged_weigh_kernel, dim3(std::max(1u, wide), p.kv.hk, p.kv.n_seqs), dim3(256), 0, st, p, weights, weights_stride), "paged decode weights launch");
}

}  // namespace

size_t paged_decode_workspace(const PagedView &kv, size_t n_heads, bool weights) { return pd_layout(kv, n_heads, weights).bytes; }

int32_t launch_paged_decode(const PagedView &kv, int type, const void *q, int q_type, size_t n_heads, float scale, PagedMask mask, float *weights,
                            size_t weights_stride, void *out, void *ws, cudaStream_t st) {
    const PdLayout lay = pd_layout(kv, n_heads, weights != nullptr);
    uint8_t *w = (uint8_t *)ws;
    PdParams p;
    p.kv = kv;
    p.mask = mask;
    p.q = q;
    p.out = out;
    p.part = (float *)(w + lay.part);
    p.ml = (float2 *)(w + lay.ml);
    p.ml_unit = (float2 *)(w + lay.unit);
    p.scores = weights ? (float *)(w + lay.scores) : nullptr;
    p.cap = (size_t)kv.max_pages * kv.page_size;
    p.scale = scale;
    p.heads = (uint32_t)n_heads;
    p.group = p.heads / kv.hk;
    p.chunks = (p.group + PD_ROWS - 1) / PD_ROWS;
    p.same = kv.k_page == kv.v_page && kv.k_slot == kv.v_slot && kv.k_head == kv.v_head;
    auto go = [&](auto cache, auto query) {
        using T = decltype(cache);
        using TQ = decltype(query);
        if (kv.dim <= 64) return pd_launch<T, TQ, 64, 3>(p, weights, weights_stride, st);
        if (kv.dim <= 128) return pd_launch<T, TQ, 128, 2>(p, weights, weights_stride, st);
        return pd_launch<T, TQ, 256, 2>(p, weights, weights_stride, st);
    };
    if (type == CERA_TYPE_F32) return go(float(), float());
    if (type == CERA_TYPE_F16) return q_type == type ? go(__half(), __half()) : go(__half(), float());
    return q_type == type ? go(__nv_bfloat16(), __nv_bfloat16()) : go(__nv_bfloat16(), float());
}

}  // namespace cera
