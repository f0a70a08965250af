// Attention of one new token per sequence over a paged cache: o = sum_j p_j v_j, p = softmax(scale q k_j), for every query head.
//
// Every visible key and value is read once for all the query heads of its KV head - eight at a time, more take another pass - so the cache's
// bytes bound a large call.  The visible slots of all (sequence, KV head, eight heads) units are cut into tiles, and the tiles of the whole call are
// dealt out evenly in one line: CTA b has tiles [b T / G, (b + 1) T / G), whatever the sequences' lengths, and at most its first and its
// last unit are shared with others.  What a CTA knows of a shared unit (maximum, sum, weighted values) goes to the workspace, whose size
// therefore does not depend on the lengths; paged_join_kernel adds the parts up in their order, so a call's bits do not depend on timing.
//
// Two warps of a CTA load, keys and values, into a ring of tiles in shared memory: by TMA where a page holds whole groups of eight slots, a box of
// slots an instruction (a copy for every row, by cp.async or in bulk, took most of what the kernel issued), row by row otherwise.  Four warps
// compute, each on its own keys of a tile - 16 of 64 over a 16-bit cache, 8 of 32 over f32 - with a running maximum, sum and weighted values of
// its own; they meet at a unit's end only.  The maximum is raised when a score has passed it by 2^8 (a vote, no exchange), to which the weights'
// range is fitted.  Rows that are not seen are set to zero among the values: what lies there may be a NaN.
//
// 16-bit cache: mma.sync, 16 rows = eight heads twice: the upper half of each query and weight as the type has it, and what that leaves,
// so an f32 query or weight counts with 22 bits (f16) in the same instructions; bf16's 16 bits are too few for an f32 query, whose third
// part takes a second product.  An f16 part is scaled by a power of two per query, weights by 2^7, so that what f16 cannot tell from zero is 2^-32
// of the largest weight.  The tensor cores cut a sum at every step instead of rounding it (one sum a unit: 5.4e-5 off at 40 960 slots, 1.6e-4 at 131 072), so after JOIN tiles a
// warp's sums are added in f32 to those it keeps in shared memory, and begun anew: eight tiles where the result has 32 bits (4.4e-7 off at 40 960 slots; sixteen 1.1e-6), 64 where it has 16 (5.6e-6
// beside its rounding; eight would cost 24 conversations 1.5 us of 39).
// f32 cache: FMAs, four lanes a key for the scores, a lane 4 dimensions of every head for the values.
//
// With weights wanted the scaled scores are stored on the way (4 bytes a head and slot, beside the 2 dim that are read for it), and
// paged_weigh_kernel turns them into probabilities once the denominators are known.
#include <algorithm>

#include "mma.cuh"
#include "paged.cuh"
#include "tc.cuh"

namespace cera {

__device__ unsigned int g_paged_decode_status = 0;

static const bool g_paged_decode_registered = register_kernel_status([] {
    unsigned int v = 0;
    cudaMemcpyFromSymbol(&v, g_paged_decode_status, sizeof(v));
    return STATUS_PAGED_DECODE.of(v);
});

namespace {

constexpr int PD_CTAS = 512;  // at most
constexpr int PD_WARPS = 4, PD_MATH = 32 * PD_WARPS, PD_THREADS = PD_MATH + 64, PD_ROWS = 8;  // a warp for the keys and one for the values
constexpr float PD_FLOOR = -3.402823466e38f;  // no score that is a number is lower
constexpr float PD_LIFT = 7.0f;         // weights are 2^7 at the maximum's score, 2^15 at most
constexpr float PD_RAISE = 8.0f;
constexpr uint32_t PD_BEGIN = 2;

struct PdParams {
    PagedView kv;
    PagedMask mask;
    const void *q;
    void *out;
    float *part;    // [2 G][8][dim]
    float2 *ml;     // [2 G][8]: maximum, sum; then, with weights, [units][8]
    float *scores;  // [seqs][heads][capacity] or null
    float2 *ml_unit;
    size_t cap;                     // of scores, a multiple of 64
    float scale;
    uint32_t heads, group, chunks;  // chunks of eight heads in a group
    uint32_t box;                   // slots a TMA copy brings
};

// a / b; of numbers that fit 32 bits a short division, and they nearly always do.
__device__ __forceinline__ uint32_t pd_div(uint64_t a, uint64_t b) { return (a | b) >> 32 ? (uint32_t)(a / b) : (uint32_t)a / (uint32_t)b; }

// Where CTA b of `parts` begins on a line of `total`.
__device__ __forceinline__ uint64_t pd_start(uint32_t b, uint64_t total, uint64_t parts) {
    const uint64_t a = b * total;
    return (a | parts) >> 32 ? a / parts : (uint32_t)a / (uint32_t)parts;
}

// The tiles of the call in one line, each unit's behind a stretch of PD_BEGIN that stands for what a unit costs beside its tiles (its queries, and
// the warps' meeting at its end): without it a CTA that got many short units took twice as long as the rest (24 sequences of 1 to 9000 slots
// 70 us, with it 39).  Where every tile has a CTA of its own there is none.  sums live in shared memory.
struct PdLine {
    const uint32_t *sums;        // the line ahead of sequence s, of one unit each; sums[n] is all
    uint32_t n, per_seq, begin;  // units of a sequence; a unit's stretch
    __device__ __forceinline__ uint32_t length(uint32_t tiles) const { return tiles ? tiles + begin : 0; }
};

template <int TILE>
struct PdCursor : PagedSpan {
    uint32_t s, unit, tile;

    __device__ __forceinline__ void seek(const PdLine &line, const PagedView &kv, const PagedMask &mask, uint64_t x) {
        uint32_t lo = 0, hi = line.n;  // the last s with sums[s] per_seq <= x, which has tiles
        while (hi - lo > 1) {
            const uint32_t mid = (lo + hi) / 2;
            if ((uint64_t)line.sums[mid] * line.per_seq <= x) lo = mid;
            else hi = mid;
        }
        s = lo;
        newest(mask, paged_len(kv, s), TILE);
        const uint64_t r = x - (uint64_t)line.sums[s] * line.per_seq;
        const uint32_t all = max(line.length(tiles), 1u);
        unit = pd_div(r, all);
        const uint32_t in = (uint32_t)(r - (uint64_t)unit * all);
        tile = in > line.begin ? in - line.begin : 0;
    }
    __device__ __forceinline__ bool behind(const PdCursor &o) const { return s != o.s ? s < o.s : unit != o.unit ? unit < o.unit : tile < o.tile; }
    __device__ __forceinline__ void step(const PdLine &line, const PagedView &kv, const PagedMask &mask) {
        if (++tile < tiles) return;
        tile = 0;
        if (++unit < line.per_seq) return;
        unit = 0;
        do ++s;
        while (s + 1 < line.n && line.sums[s + 1] == line.sums[s]);
        if (s < line.n) newest(mask, paged_len(kv, s), TILE);
    }
};

__device__ __forceinline__ float pd_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The line, by the whole CTA.
template <int TILE>
__device__ __forceinline__ PdLine pd_line(const PagedView &kv, const PagedMask &mask, uint32_t per_seq, uint32_t ctas, uint32_t *sums, uint2 *warps) {
    const uint32_t tid = threadIdx.x, lane = tid & 31, per = (kv.n_seqs + PD_THREADS - 1) / PD_THREADS, s0 = min(tid * per, kv.n_seqs), s1 = min(s0 + per, kv.n_seqs);
    uint32_t tiles = 0, live = 0;
    for (uint32_t s = s0; s < s1; ++s) {
        PagedSpan span;
        span.newest(mask, paged_len(kv, s), TILE);
        sums[s + 1] = span.tiles;
        tiles += span.tiles;
        live += span.tiles != 0;
    }
    uint32_t x = tiles, y = live;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t a = __shfl_up_sync(0xffffffffu, x, o), b = __shfl_up_sync(0xffffffffu, y, o);
        if (lane >= (uint32_t)o) {
            x += a;
            y += b;
        }
    }
    if (lane == 31) warps[tid >> 5] = make_uint2(x, y);
    if (tid == 0) sums[0] = 0;
    __syncthreads();
    uint32_t all = 0;
    x -= tiles;
    y -= live;
    for (uint32_t w = 0; w < PD_THREADS / 32; ++w) {
        all += warps[w].x;
        if (w < tid >> 5) {
            x += warps[w].x;
            y += warps[w].y;
        }
    }
    PdLine line{sums, kv.n_seqs, per_seq, (uint64_t)all * per_seq > ctas ? PD_BEGIN : 0};
    x += y * line.begin;
    for (uint32_t s = s0; s < s1; ++s) {
        x += line.length(sums[s + 1]);
        sums[s + 1] = x;
    }
    __syncthreads();
    return line;
}

// ---- what a warp does with its keys of a tile ------------------------------------------------------------------------------

// 16-bit cache.  Lane = (row lane / 4, columns 2 (lane % 4) + {0, 1}) of an mma tile; acc's second half is the lower parts'.
template <typename T, typename TQ, int DP>
struct PdMma {
    static constexpr int KG = 16, ROWS = PD_ROWS, TILE = PD_WARPS * KG, BLOCK = 64;  // BLOCK: numbers of a 128-byte row
    static constexpr bool SPLIT = sizeof(TQ) == 4, BF = sizeof(T) == 2 && !std::is_same<T, __half>::value, THIRD = SPLIT && BF;
    static constexpr uint32_t JOIN = SPLIT ? 8 : 64;  // a power of two
    uint32_t qf[DP / 16][SPLIT ? 4 : 2], q3[THIRD ? DP / 16 : 1][2];
    uint32_t wf[4], w3[4];
    float acc[DP / 8][4], m, l, factor;
    float *kept;  // this lane's numbers of the warp's sums [8][dim] in shared memory
    bool some;    // there are such sums

    // the value of column pair n that acc has, number i: of an infinite value the weight's upper part says it all
    __device__ __forceinline__ float value(int n, int i) const {
        const float hi = acc[n][i], both = hi + acc[n][i + 2];
        return fabsf(both) < INFINITY ? both : hi;
    }
    __device__ __forceinline__ void keep(const PdParams &p) {
#pragma unroll
        for (int n = 0; n < DP / 8; ++n)
            if (n * 8 < p.kv.dim) {
                float2 *to = reinterpret_cast<float2 *>(kept + n * 8);
                const float2 old = some ? *to : make_float2(0.0f, 0.0f);
                *to = make_float2(old.x + value(n, 0), old.y + value(n, 1));
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[n][i] = 0.0f;
            }
        some = true;
    }

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
    // What takes the upper rows of a product with third parts: nothing but the signs (of bf16's least normal number), since zero times an infinite key or value would be a NaN.
    static __device__ __forceinline__ uint32_t least(uint32_t hi) { return (hi & 0x80008000u) | 0x00800080u; }
    // what hi and lo leave of (x, y)
    static __device__ __forceinline__ uint32_t third(float x, float y, uint32_t hi, uint32_t lo) {
        const float2 h = unpack(hi), w = unpack(lo);
        uint32_t a, b;
        split(x - h.x - w.x, y - h.y - w.y, a, b);
        return a;
    }

    __device__ __forceinline__ void begin(const PdParams &p, uint32_t s, uint32_t head0, uint32_t rows, float *, float *sums) {
        const uint32_t lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
        kept = sums + r * p.kv.dim + 2 * c;
        some = false;
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

    // ks: the tile's keys; mask: which of the warp's are seen; scores: the first of these keys' places for head 0 of the unit, or null
    __device__ __forceinline__ void weigh(const PdParams &p, const uint8_t *ks, uint32_t mask, uint32_t rows, float *scores, const float *, float *) {
        const uint32_t lane = threadIdx.x & 31, r = lane >> 2, c2 = 2 * (lane & 3);
        float sc[2][4] = {}, sd[2][4] = {};  // two sums each: a product waits for the one before the last
        const uint8_t *ka = ks + ((threadIdx.x >> 5) * KG + (lane & 7) + (lane >> 4) * 8) * 128;
        const uint32_t turn = ((lane & 7) ^ (lane >> 3 & 1)) * 16;  // 16-byte chunk c of row i lies at c ^ i % 8
#pragma unroll
        for (int k = 0; k < DP / 16; ++k) {
            if (k * 16 >= p.kv.dim) break;
            uint32_t b[4];
            ldsm4(b, ka + (k >> 2) * TILE * 128 + (turn ^ (k & 3) * 32));
            const uint32_t a[4] = {qf[k][0], SPLIT ? qf[k][SPLIT ? 2 : 0] : 0u, qf[k][1], SPLIT ? qf[k][SPLIT ? 3 : 1] : 0u};
            mma(k & 1 ? sd[0] : sc[0], a, b[0], b[1]);
            mma(k & 1 ? sd[1] : sc[1], a, b[2], b[3]);
            if (THIRD) {
                const uint32_t a3[4] = {least(qf[k][0]), q3[THIRD ? k : 0][0], least(qf[k][1]), q3[THIRD ? k : 0][1]};  // beside the lower parts
                mma(k & 1 ? sd[0] : sc[0], a3, b[0], b[1]);
                mma(k & 1 ? sd[1] : sc[1], a3, b[2], b[3]);
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) sc[i >> 2][i & 3] += sd[i >> 2][i & 3];
        float z[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float hi = sc[i >> 1][i & 1], both = hi + sc[i >> 1][(i & 1) + 2];
            z[i] = (SPLIT && fabsf(both) < INFINITY ? both : hi) * factor;  // of an infinite key the upper part says it all; without a lower part its rows are zeros times the key
        }
        if (mask != 0xffffu) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (!(mask >> (c2 + (i & 1) + (i >> 1) * 8) & 1)) z[i] = -INFINITY;
        }
        if (scores && r < rows) {
            float *to = scores + (size_t)r * p.cap + c2;
#pragma unroll
            for (int i = 0; i < 2; ++i) *reinterpret_cast<float2 *>(to + 8 * i) = make_float2(z[2 * i], z[2 * i + 1]);
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
                if (some)
                    for (uint32_t n = 0; n < p.kv.dim; n += 8) {
                        float2 *to = reinterpret_cast<float2 *>(kept + n);
                        *to = make_float2(to->x * f, to->y * f);
                    }
            }
        }
        const float base = PD_LIFT - m;
        float w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = pd_exp2(z[i] + base);
        l += (w[0] + w[1]) + (w[2] + w[3]);
        split(w[0], w[1], wf[0], wf[1]);
        split(w[2], w[3], wf[2], wf[3]);
        if (THIRD) {
            w3[1] = third(w[0], w[1], wf[0], wf[1]);
            w3[3] = third(w[2], w[3], wf[2], wf[3]);
            w3[0] = w3[2] = least(0);
        }
    }
    __device__ __forceinline__ void add(const PdParams &p, const uint8_t *vs, const float *) {
        const uint32_t lane = threadIdx.x & 31;
        const uint8_t *va = vs + ((threadIdx.x >> 5) * KG + (lane & 15)) * 128;
        const uint32_t turn = ((lane & 7) ^ (lane >> 4)) * 16;
#pragma unroll
        for (int n = 0; n < DP / 16; ++n) {
            if (n * 16 >= p.kv.dim) break;
            uint32_t b[4];
            ldsm4_trans(b, va + (n >> 2) * TILE * 128 + (turn ^ (n & 3) * 32));
            mma(acc[2 * n], wf, b[0], b[1]);
            mma(acc[2 * n + 1], wf, b[2], b[3]);
            if (THIRD) {
                mma(acc[2 * n], w3, b[0], b[1]);
                mma(acc[2 * n + 1], w3, b[2], b[3]);
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
    // the weighted values for the maxima `all` of each row, where the sums are kept
    __device__ __forceinline__ void values(const PdParams &p, const float *all, float *) {
        const float f = pd_exp2(m - all[(threadIdx.x & 31) >> 2]);
#pragma unroll
        for (int n = 0; n < DP / 8; ++n)
            if (n * 8 < p.kv.dim) {
                float2 *to = reinterpret_cast<float2 *>(kept + n * 8);
                const float2 old = some ? *to : make_float2(0.0f, 0.0f);
                *to = make_float2((old.x + value(n, 0)) * f, (old.y + value(n, 1)) * f);
            }
    }
};

// f32 cache.  Scores: lane = (key lane / 4, every fourth 16 bytes of the row), then two heads of that key.  Values: lane = 4 dimensions.
template <int DP, int R>
struct PdFma {
    static constexpr int KG = 8, ROWS = R, NZ = R / 4, TILE = PD_WARPS * KG, BLOCK = 32, NV = (DP + 127) / 128;
    float4 acc[R][NV];
    float m[NZ], l[NZ];  // of heads NZ (lane % 4) + [0, NZ); l over this lane's keys

    static constexpr uint32_t JOIN = 1;
    __device__ __forceinline__ void keep(const PdParams &) {}  // FMAs round
    __device__ __forceinline__ void begin(const PdParams &p, uint32_t s, uint32_t head0, uint32_t rows, float *qs, float *) {
        const uint32_t lane = threadIdx.x & 31;
        const float *q = reinterpret_cast<const float *>(p.q) + ((size_t)s * p.heads + head0) * p.kv.dim;
        __syncwarp();
        for (uint32_t i = lane; i < R * DP; i += 32) {
            const uint32_t r = i / DP, d = i % DP;
            qs[i] = r < rows && d < p.kv.dim ? q[r * p.kv.dim + d] : 0.0f;
        }
        __syncwarp();
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int i = 0; i < NV; ++i) acc[r][i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int i = 0; i < NZ; ++i) {
            m[i] = PD_FLOOR;
            l[i] = 0.0f;
        }
    }

    __device__ __forceinline__ void weigh(const PdParams &p, const uint8_t *ks, uint32_t mask, uint32_t rows, float *scores, const float *qs, float *ps) {
        const uint32_t lane = threadIdx.x & 31, key = lane >> 2, part = lane & 3;
        const uint8_t *ka = ks + ((threadIdx.x >> 5) * KG + key) * 128;
        float2 d2[R];
#pragma unroll
        for (int r = 0; r < R; ++r) d2[r] = make_float2(0.0f, 0.0f);
#pragma unroll 4
        for (uint32_t i = 0; i < p.kv.dim / 16; ++i) {
            const uint32_t c = part + 4 * (i ^ (key & 1));  // chunk c lies at c ^ key % 8: odd keys go the other way round, so that two meet all banks
            const float4 k = *reinterpret_cast<const float4 *>(ka + (c >> 3) * TILE * 128 + ((c & 7) ^ key) * 16);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const float4 q = *reinterpret_cast<const float4 *>(qs + r * DP + c * 4);
                d2[r] = __ffma2_rn(make_float2(k.x, k.y), make_float2(q.x, q.y), d2[r]);
                d2[r] = __ffma2_rn(make_float2(k.z, k.w), make_float2(q.z, q.w), d2[r]);
            }
        }
        float d[R];
#pragma unroll
        for (int r = 0; r < R; ++r) d[r] = d2[r].x + d2[r].y;
        // sums over the four lanes of a key; lane `part` keeps heads NZ part + [0, NZ)
        const bool up2 = part & 2, up1 = part & 1;
        float h2[R / 2], z[NZ];
#pragma unroll
        for (int i = 0; i < R / 2; ++i) {
            const float give = up2 ? d[i] : d[R / 2 + i], keep = up2 ? d[R / 2 + i] : d[i];
            h2[i] = keep + __shfl_xor_sync(0xffffffffu, give, 2);
        }
        bool raise = false;
#pragma unroll
        for (int i = 0; i < NZ; ++i) {
            const float give = up1 ? h2[i] : h2[NZ + i], keep = up1 ? h2[NZ + i] : h2[i];
            z[i] = (keep + __shfl_xor_sync(0xffffffffu, give, 1)) * (p.scale * PAGED_LOG2E);
            if (!(mask >> key & 1)) z[i] = -INFINITY;
            raise |= z[i] > m[i] + PD_RAISE;
        }
        if (scores) {
#pragma unroll
            for (int i = 0; i < NZ; ++i)
                if (NZ * part + i < rows) scores[(size_t)(NZ * part + i) * p.cap + key] = z[i];
        }
        if (__any_sync(0xffffffffu, raise)) {
            float f[NZ];
#pragma unroll
            for (int i = 0; i < NZ; ++i) {
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
            for (int r = 0; r < R; ++r) {
                const float g = __shfl_sync(0xffffffffu, f[r % NZ], r / NZ);
#pragma unroll
                for (int i = 0; i < NV; ++i) acc[r][i] = make_float4(acc[r][i].x * g, acc[r][i].y * g, acc[r][i].z * g, acc[r][i].w * g);
            }
        }
#pragma unroll
        for (int i = 0; i < NZ; ++i) {
            const float w = pd_exp2(z[i] + (PD_LIFT - m[i]));
            l[i] += w;
            ps[key * R + NZ * part + i] = w;
        }
        __syncwarp();
    }
    __device__ __forceinline__ void add(const PdParams &p, const uint8_t *vs, const float *ps) {
        const uint32_t lane = threadIdx.x & 31;
        const uint8_t *va = vs + (threadIdx.x >> 5) * KG * 128;
#pragma unroll
        for (int k = 0; k < KG; ++k) {
            float ww[R];
#pragma unroll
            for (int r = 0; r < R; r += 4) *reinterpret_cast<float4 *>(ww + r) = *reinterpret_cast<const float4 *>(ps + k * R + r);
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                if ((lane + 32 * i) * 4 >= p.kv.dim) break;
                const uint32_t c = lane + 32 * i;
                const float4 v = *reinterpret_cast<const float4 *>(va + (c >> 3) * TILE * 128 + k * 128 + ((c & 7) ^ k) * 16);
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const float2 wr = make_float2(ww[r], ww[r]);
                    const float2 lo = __ffma2_rn(wr, make_float2(v.x, v.y), make_float2(acc[r][i].x, acc[r][i].y));
                    const float2 hi = __ffma2_rn(wr, make_float2(v.z, v.w), make_float2(acc[r][i].z, acc[r][i].w));
                    acc[r][i] = make_float4(lo.x, lo.y, hi.x, hi.y);
                }
            }
        }
    }

    __device__ __forceinline__ void end(float2 *ml) {
        const uint32_t lane = threadIdx.x & 31;
#pragma unroll
        for (int i = 0; i < NZ; ++i) {
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 4);
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 8);
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 16);
            if (lane < 4) ml[NZ * lane + i] = make_float2(m[i], l[i]);
        }
    }
    __device__ __forceinline__ void values(const PdParams &p, const float *all, float *to) {
        const uint32_t lane = threadIdx.x & 31;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const float f = pd_exp2(__shfl_sync(0xffffffffu, m[r % NZ], r / NZ) - all[r]);
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if ((lane + 32 * i) * 4 < p.kv.dim)
                    *reinterpret_cast<float4 *>(to + r * p.kv.dim + (lane + 32 * i) * 4) = make_float4(acc[r][i].x * f, acc[r][i].y * f, acc[r][i].z * f, acc[r][i].w * f);
        }
    }
};

template <typename T, typename TQ, int DP, int R>
struct PdOf {
    using W = PdMma<T, TQ, DP>;
};
template <int DP, int R>
struct PdOf<float, float, DP, R> {
    using W = PdFma<DP, R>;
};

// Shared memory: the ring | values of the warps at a unit's end | queries and weights (f32) | the line's sums.
template <typename W, int DP, int ST, bool FMA>
struct PdSmem {
    static constexpr size_t HALF = (size_t)W::TILE * DP * (FMA ? 4 : 2), STAGE = 2 * HALF, VALUES = (size_t)PD_WARPS * W::ROWS * DP * 4,
                            EXTRA = FMA ? PD_WARPS * (size_t)W::ROWS * (DP + W::KG) * 4 : 0, FIXED = 1024 + ST * STAGE + VALUES + EXTRA;
};

__device__ __forceinline__ void pd_sync() { asm volatile("bar.sync 1, %0;" ::"n"(PD_MATH) : "memory"); }  // the warps that compute

template <typename T, typename TQ, int DP, int ST, int R, bool TMA>
__global__ void __launch_bounds__(PD_THREADS, DP <= 128 ? 2 : 1) paged_decode_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const PdParams p) {
    using W = typename PdOf<T, TQ, DP, R>::W;
    using S = PdSmem<W, DP, ST, sizeof(T) == 4>;
    constexpr int KG = W::KG, TILE = W::TILE;
    extern __shared__ uint8_t raw[];
    __shared__ float2 ml_s[PD_WARPS][PD_ROWS];
    __shared__ float all_s[PD_ROWS], sum_s[PD_ROWS];
    __shared__ uint2 scan_s[PD_THREADS / 32];
    __shared__ uint32_t mask_s[ST][2], any_s[PD_WARPS], abort_s;
    __shared__ uint64_t full_s[2][ST], empty_s[ST];
    uint8_t *smem = raw + (1024 - (tma::smem_u32(raw) & 1023)) % 1024;
    float *values = reinterpret_cast<float *>(smem + ST * S::STAGE);
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, b = blockIdx.x;
    unsigned int *status = &g_paged_decode_status;
    pdl_trigger();
    if (tid == 0) {
        for (int i = 0; i < ST; ++i) {
            tma::mbar_init(&full_s[0][i], TMA ? 1 : 33);
            tma::mbar_init(&full_s[1][i], TMA ? 1 : 33);
            tma::mbar_init(&empty_s[i], PD_WARPS);
        }
        abort_s = 0;
        tma::mbar_init_fence();
    }
    pdl_wait();
    const uint32_t per_seq = p.kv.hk * p.chunks;
    const PdLine line = pd_line<TILE>(p.kv, p.mask, per_seq, gridDim.x, reinterpret_cast<uint32_t *>(smem + S::FIXED - 1024), scan_s);
    const uint64_t total = (uint64_t)line.sums[line.n] * per_seq, parts = min((uint64_t)gridDim.x, total);
    if (b >= parts) return;
    const uint64_t x0 = pd_start(b, total, parts), x1 = pd_start(b + 1, total, parts);
    PdCursor<TILE> at, end;
    at.seek(line, p.kv, p.mask, x0);
    end.seek(line, p.kv, p.mask, x1);  // the place behind everything, for the last CTA
    if (!at.behind(end)) return;

    if (warp >= PD_WARPS) {
        const bool is_v = warp > PD_WARPS;
        uint64_t *full = full_s[is_v];
        uint8_t *half = smem + (is_v ? S::HALF : 0);
        const uint32_t boxes = TILE / p.box, blocks = (p.kv.dim + W::BLOCK - 1) / W::BLOCK;
        const size_t by_page = is_v ? p.kv.v_page : p.kv.k_page, by_slot = is_v ? p.kv.v_slot : p.kv.k_slot, by_head = is_v ? p.kv.v_head : p.kv.k_head;
        const uint8_t *base = is_v ? p.kv.v : p.kv.k;
        // the pages of the tile at the cursor: with TMA lane i looks up box i, otherwise a lane the slots lane and lane + 32 of the tile
        uint32_t page[2], row[2];
        auto find = [&]() {
            const uint32_t slot0 = at.slot(at.tile, TILE);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                page[i] = NO_PAGE;
                row[i] = 0;
                if (TMA) {
                    const uint32_t j = slot0 + lane * p.box;
                    const bool some = j < at.len && (j + p.box > at.first || j < at.sinks);
                    if (i == 0 && lane < boxes && some) page[0] = paged_at(p.kv, at.s, j, row[0]);
                } else if (32 * i < TILE) {
                    const uint32_t j = slot0 + lane + 32 * i;
                    if (at.sees(j)) page[i] = paged_at(p.kv, at.s, j, row[i]);
                }
            }
        };
        find();
        const uint32_t me = elect_one();
        // shared memory must outlive the copies in flight, those of the stages before tile n: whoever reads them may give up while they are
        auto drain = [&](uint32_t n) {
            for (uint32_t y = n > ST ? n - ST : 0; y < n; ++y)
                for (uint32_t i = 0; i < tma::SPIN_LIMIT && !tma::mbar_test(&full[y % ST], y / ST & 1); ++i) __nanosleep(40);
        };
        uint32_t x = 0;
        for (; at.behind(end); ++x) {
            const uint32_t st = x % ST;
            const uint32_t slot0 = at.slot(at.tile, TILE), h = at.unit / p.chunks;
            uint32_t mask[2];
            uint32_t pg[2] = {page[0], page[1]}, rw[2] = {row[0], row[1]};
            const uint32_t live = __ballot_sync(0xffffffffu, pg[0] != NO_PAGE);  // TMA: boxes
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t j = lane + 32 * i;
                const bool there = TMA ? j < TILE && at.sees(slot0 + j) && (live >> j / p.box & 1) : pg[i] != NO_PAGE;
                mask[i] = __ballot_sync(0xffffffffu, there);
            }
            at.step(line, p.kv, p.mask);
            if (at.behind(end)) find();  // its answer is not needed before the next tile
            if (!tma::mbar_wait_warp(&empty_s[st], (x / ST & 1) ^ 1, &abort_s, status, 1u)) return drain(x);
            if (!is_v && lane < 2) mask_s[st][lane] = lane ? mask[1] : mask[0];
            __syncwarp();
            uint8_t *to = half + st * S::STAGE;
            if (TMA) {
                tma::mbar_expect_tx_if(&full[st], __popc(live) * blocks * p.box * 128, me);
                for (uint32_t i = 0; i < boxes; ++i) {
                    const uint32_t pi = __shfl_sync(0xffffffffu, pg[0], i), ri = __shfl_sync(0xffffffffu, rw[0], i);
                    if (pi == NO_PAGE) continue;
                    for (uint32_t k = 0; k < blocks; ++k)
                        tma::tensor_g2s_4d_if(to + k * TILE * 128 + i * p.box * 128, is_v ? &map_v : &map_k, k * W::BLOCK, h, ri, pi, &full[st], me);
                }
            } else {
                const uint32_t per = blocks * 8, used = p.kv.dim * sizeof(T) / 16;
                uint64_t off[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) off[i] = pg[i] != NO_PAGE ? pg[i] * (uint64_t)by_page + rw[i] * (uint64_t)by_slot + h * (uint64_t)by_head : 0;
                for (uint32_t i = lane; i < TILE * per; i += 32) {  // TILE * per is a multiple of 32: the warp stays together
                    const uint32_t r = i / per, c = i - r * per;
                    const uint64_t lo = __shfl_sync(0xffffffffu, off[0], r & 31), hi = __shfl_sync(0xffffffffu, off[1], r & 31);
                    if (c < used && (mask[r >> 5] >> (r & 31) & 1))
                        tma::cp_async16(to + (c >> 3) * TILE * 128 + r * 128 + ((c & 7) ^ (r & 7)) * 16, base + (r < 32 ? lo : hi) + c * 16);
                }
                tma::cp_async_arrive(&full[st]);
                if (lane == 0) tma::mbar_arrive(&full[st]);  // the mask's
            }
        }
        drain(x);
        return;
    }

    float *qs = values + PD_WARPS * R * DP + warp * R * (DP + KG), *ps = qs + R * DP;
    W w;
    uint32_t any = 0, first_tile = at.tile, rows = 0, head0 = 0;
    bool more = true;
    for (uint32_t x = 0; more; ++x) {
        if (x == 0 || at.tile == 0) {
            const uint32_t h = at.unit / p.chunks, c = at.unit - h * p.chunks;
            head0 = h * p.group + c * PD_ROWS;
            rows = min(p.group - c * PD_ROWS, (uint32_t)PD_ROWS);
            first_tile = at.tile;
            any = 0;
            w.begin(p, at.s, head0, rows, qs, values + warp * R * p.kv.dim);
        }
        const uint32_t st = x % ST, slot0 = at.slot(at.tile, TILE) + warp * KG;
        const uint8_t *ks = smem + st * S::STAGE;
        // a warp that gave up goes on without waiting; what it forms is reported as undefined
        tma::mbar_wait_warp(&full_s[0][st], x / ST & 1, &abort_s, status, 2u);
        const uint32_t mask = mask_s[st][warp * KG / 32] >> warp * KG % 32 & ((1u << KG) - 1);
        any |= mask;
        const bool work = mask || (p.scores && slot0 < at.len);
        if (work) w.weigh(p, ks, mask, rows, p.scores ? p.scores + ((size_t)at.s * p.heads + head0) * p.cap + slot0 : nullptr, qs, ps);
        tma::mbar_wait_warp(&full_s[1][st], x / ST & 1, &abort_s, status, 2u);
        if (mask) {
            uint8_t *vs = smem + st * S::STAGE + S::HALF;
            if (mask != (1u << KG) - 1) {  // a weight of zero times what lies there could be a NaN
                const uint32_t r = lane % KG;
                if (!(mask >> r & 1))
                    for (uint32_t c = lane / KG; c < DP * sizeof(T) / 16; c += 32 / KG)
                        *reinterpret_cast<uint4 *>(vs + (c >> 3) * TILE * 128 + (warp * KG + r) * 128 + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
                fence_async_smem();
                __syncwarp();
            }
            w.add(p, vs, ps);
        }
        __syncwarp();
        if (lane == 0) tma::mbar_arrive(&empty_s[st]);
        const PdCursor<TILE> done = at;
        const bool last = at.tile + 1 == at.tiles;
        at.step(line, p.kv, p.mask);
        more = at.behind(end);
        if (x % W::JOIN == W::JOIN - 1) w.keep(p);
        if (last || !more) {
            // the warps' shares of the unit
            w.end(ml_s[warp]);
            if (lane == 0) any_s[warp] = any;
            pd_sync();
            if (tid < R) {
                float m = ml_s[0][tid].x, l = 0.0f;
                for (int i = 1; i < PD_WARPS; ++i) m = fmaxf(m, ml_s[i][tid].x);
                for (int i = 0; i < PD_WARPS; ++i) l += ml_s[i][tid].y * pd_exp2(ml_s[i][tid].x - m);
                all_s[tid] = m;
                sum_s[tid] = l;
            }
            const bool seen = any_s[0] | any_s[1] | any_s[2] | any_s[3];
            pd_sync();
            w.values(p, all_s, values + warp * R * p.kv.dim);
            pd_sync();
            const bool whole = last && first_tile == 0;
            const uint32_t slot = 2 * b + (done.tile - first_tile != x);  // the first unit of this CTA, or another, which is its last
            const uint32_t n = R * p.kv.dim, unit = done.s * per_seq + done.unit;
            for (uint32_t i = tid * 4; i < n; i += PD_MATH * 4) {
                float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int k = 0; k < PD_WARPS; ++k) {
                    const float4 v = *reinterpret_cast<const float4 *>(values + k * n + i);
                    o = make_float4(o.x + v.x, o.y + v.y, o.z + v.z, o.w + v.w);
                }
                const uint32_t r = i / p.kv.dim;
                if (whole) {
                    if (r < rows) {
                        TQ *to = reinterpret_cast<TQ *>(p.out) + ((size_t)done.s * p.heads + head0) * p.kv.dim + i;
                        const float f = sum_s[r];
                        to[0] = from_f32<TQ>(seen ? o.x / f : 0.0f);
                        to[1] = from_f32<TQ>(seen ? o.y / f : 0.0f);
                        to[2] = from_f32<TQ>(seen ? o.z / f : 0.0f);
                        to[3] = from_f32<TQ>(seen ? o.w / f : 0.0f);
                    }
                } else {
                    *reinterpret_cast<float4 *>(p.part + (size_t)slot * PD_ROWS * p.kv.dim + i) = o;
                }
            }
            if (tid < R) {
                const float2 v = make_float2(seen ? all_s[tid] : -INFINITY, sum_s[tid]);
                if (!whole) p.ml[(size_t)slot * PD_ROWS + tid] = v;
                else if (p.scores) p.ml_unit[(size_t)unit * PD_ROWS + tid] = v;
            }
            pd_sync();
        }
    }
}

// A CTA per (unit, row): units without tiles are zeros, whole ones are done, the others' parts are added up.
template <typename TQ, int TILE>
__global__ void __launch_bounds__(PD_MATH) paged_join_kernel(const PdParams p, uint32_t G) {
    __shared__ uint4 sums_s[PD_WARPS];
    __shared__ uint32_t first_s;
    __shared__ float2 share_s[PD_CTAS];
    __shared__ float max_s[PD_WARPS], sum_s[PD_WARPS];
    __shared__ __align__(16) float value_s[PD_WARPS][256];
    pdl_trigger();
    pdl_wait();
    const uint32_t per_seq = p.kv.hk * p.chunks, unit = blockIdx.x, s = unit / per_seq, u = unit - s * per_seq, r = blockIdx.y, tid = threadIdx.x;
    const uint32_t h = u / p.chunks, c = u - h * p.chunks, rows = min(p.group - c * PD_ROWS, (uint32_t)PD_ROWS);
    if (r >= rows) return;
    uint32_t before = 0, all = 0, live_before = 0, live = 0;  // sequences that have tiles count their stretch
    for (uint32_t i = tid; i < p.kv.n_seqs; i += PD_MATH) {
        PagedSpan span;
        span.newest(p.mask, paged_len(p.kv, i), TILE);
        const uint32_t n = span.tiles;
        all += n;
        live += n != 0;
        if (i < s) {
            before += n;
            live_before += n != 0;
        }
        if (i == s) first_s = n;
    }
    before = __reduce_add_sync(0xffffffffu, before);
    all = __reduce_add_sync(0xffffffffu, all);
    live_before = __reduce_add_sync(0xffffffffu, live_before);
    live = __reduce_add_sync(0xffffffffu, live);
    if ((tid & 31) == 0) sums_s[tid >> 5] = make_uint4(before, all, live_before, live);
    __syncthreads();
    before = all = live_before = live = 0;
    for (int i = 0; i < PD_WARPS; ++i) {
        before += sums_s[i].x;
        all += sums_s[i].y;
        live_before += sums_s[i].z;
        live += sums_s[i].w;
    }
    const uint32_t begin = (uint64_t)all * per_seq > G ? PD_BEGIN : 0;
    all += live * begin;
    before += live_before * begin;
    const uint32_t tiles = first_s;
    TQ *out = reinterpret_cast<TQ *>(p.out) + ((size_t)s * p.heads + h * p.group + c * PD_ROWS + r) * p.kv.dim;
    if (tiles == 0) {
        for (uint32_t d = tid; d < p.kv.dim; d += PD_MATH) out[d] = from_f32<TQ>(0.0f);
        return;
    }
    const uint64_t total = (uint64_t)all * per_seq, parts = min((uint64_t)G, total), u0 = (uint64_t)before * per_seq + (uint64_t)u * (tiles + begin);
    // the CTAs of its first and last tile: the last one that begins at or ahead of it
    const uint32_t b0 = pd_div((u0 + begin + 1) * parts - 1, total), b1 = pd_div((u0 + begin + tiles) * parts - 1, total);
    if (b0 == b1) return;
    const uint32_t n = b1 - b0 + 1, lane = tid & 31, warp = tid >> 5;
    const uint32_t head = 2 * b0 + (pd_start(b0, total, parts) < u0);  // of the first CTA it may be the last unit
    auto slot = [&](uint32_t i) { return i ? 2 * (b0 + i) : head; };
    // a warp takes every fourth part, U at a time; the first are on their way before it is known what they count
    constexpr int U = 4;
    float4 x[U][2];
    auto load = [&](uint32_t i0) {
#pragma unroll
        for (int v = 0; v < U; ++v)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const uint32_t i = i0 + v * PD_WARPS, d = lane * 4 + k * 128;
                if (i < n && d < p.kv.dim) x[v][k] = *reinterpret_cast<const float4 *>(p.part + ((size_t)slot(i) * PD_ROWS + r) * p.kv.dim + d);
            }
    };
    load(warp);
    float m = -INFINITY, l = 0.0f;
    for (uint32_t i = tid; i < n; i += PD_MATH) {
        const float2 v = p.ml[(size_t)slot(i) * PD_ROWS + r];
        share_s[i] = v;
        m = fmaxf(m, v.x);
    }
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) max_s[warp] = m;
    __syncthreads();
    m = fmaxf(fmaxf(max_s[0], max_s[1]), fmaxf(max_s[2], max_s[3]));
    float4 o[2] = {};
    for (uint32_t i0 = warp; i0 < n; i0 += U * PD_WARPS) {
        if (i0 != warp) load(i0);
#pragma unroll
        for (int v = 0; v < U; ++v) {
            const uint32_t i = i0 + v * PD_WARPS;
            const float2 s2 = i < n ? share_s[i] : make_float2(-INFINITY, 0.0f);
            if (s2.x == -INFINITY) continue;  // a part that has met nothing is not there; one that has met a NaN is, whatever it weighs
            const float f = pd_exp2(s2.x - m);
            l = fmaf(s2.y, f, l);
#pragma unroll
            for (int k = 0; k < 2; ++k)
                if (lane * 4 + k * 128 < p.kv.dim) o[k] = make_float4(fmaf(x[v][k].x, f, o[k].x), fmaf(x[v][k].y, f, o[k].y), fmaf(x[v][k].z, f, o[k].z), fmaf(x[v][k].w, f, o[k].w));
        }
    }
    if (lane == 0) sum_s[warp] = l;
#pragma unroll
    for (int k = 0; k < 2; ++k)
        if (lane * 4 + k * 128 < p.kv.dim) *reinterpret_cast<float4 *>(&value_s[warp][lane * 4 + k * 128]) = o[k];
    __syncthreads();
    l = sum_s[0] + sum_s[1] + sum_s[2] + sum_s[3];
    for (uint32_t d = tid; d < p.kv.dim; d += PD_MATH)
        out[d] = from_f32<TQ>(m == -INFINITY ? 0.0f : (value_s[0][d] + value_s[1][d] + value_s[2][d] + value_s[3][d]) / l);
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
        const uint32_t slot = x < sinks ? x : x - sinks + first;
        float sum = 0.0f;
        for (uint32_t g = 0; g < p.group; ++g) {
            const float2 ml = p.ml_unit[((size_t)(s * p.kv.hk + h) * p.chunks + g / PD_ROWS) * PD_ROWS + g % PD_ROWS];
            const float z = scores[(size_t)g * p.cap + slot];
            if (z != -INFINITY) sum += pd_exp2(z + (PD_LIFT - ml.x)) / ml.y;  // rounded as the sum's weights are, where scores are far from 0
        }
        weights[((size_t)s * p.kv.hk + h) * stride + slot] += sum;
    }
}

uint32_t pd_grid() { return std::min<uint32_t>(2 * (uint32_t)sm_count(), PD_CTAS); }

size_t pd_cap(const PagedView &kv) { return ((size_t)kv.max_pages * kv.page_size + 63) / 64 * 64; }

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
    l.bytes = l.scores + (weights ? kv.n_seqs * n_heads * pd_cap(kv) * 4 : 0) + 16;
    return l;
}

template <typename T, typename TQ, int DP, int ST, int R>
int32_t pd_launch(PdParams &p, int type, float *weights, size_t weights_stride, cudaStream_t st) {
    using W = typename PdOf<T, TQ, DP, R>::W;
    const size_t smem = PdSmem<W, DP, ST, sizeof(T) == 4>::FIXED + ((size_t)p.kv.n_seqs + 1) * 4;
    const size_t tiles = ((size_t)p.kv.max_pages * p.kv.page_size + W::TILE - 1) / W::TILE * p.kv.n_seqs * p.kv.hk * p.chunks;
    const uint32_t G = (uint32_t)std::min<size_t>(DP <= 128 ? pd_grid() : pd_grid() / 2, std::max<size_t>(tiles, 1));  // what fits the SMs at once
    CUtensorMap mk, mv;
    p.box = W::TILE;
    CERA_TRY(paged_maps(p.kv, type, 8, &p.box, &mk, &mv));
    const bool by_tma = p.box != 0;
    if (!by_tma) p.box = W::TILE;
    auto kernel = by_tma ? paged_decode_kernel<T, TQ, DP, ST, R, true> : paged_decode_kernel<T, TQ, DP, ST, R, false>;
    constexpr size_t most = PdSmem<W, DP, ST, sizeof(T) == 4>::FIXED + 4097 * 4;
    CERA_TRY((by_tma ? paged_smem<paged_decode_kernel<T, TQ, DP, ST, R, true>>(most) : paged_smem<paged_decode_kernel<T, TQ, DP, ST, R, false>>(most)));
    count_launch(weights ? 3 : 2);
    CERA_CUDA_TRY(launch_k(kernel, dim3(G), dim3(PD_THREADS), smem, st, mk, mv, p));
    CERA_CUDA_TRY(launch_k(paged_join_kernel<TQ, W::TILE>, dim3(p.kv.n_seqs * p.kv.hk * p.chunks, std::min<uint32_t>(p.group, PD_ROWS)), dim3(PD_MATH), 0, st, p, G));
    if (!weights) return CERA_CUDA_OK;
    const uint32_t wide = (uint32_t)std::min<size_t>((p.cap + 255) / 256, std::max<size_t>(1, 8 * (size_t)sm_count() / std::max(1u, p.kv.n_seqs * p.kv.hk)));
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
    p.cap = pd_cap(kv);
    p.scale = scale;
    p.heads = (uint32_t)n_heads;
    p.group = p.heads / kv.hk;
    p.chunks = (p.group + PD_ROWS - 1) / PD_ROWS;
    auto go = [&](auto cache, auto query) {
        using T = decltype(cache);
        using TQ = decltype(query);
        auto rows = [&](auto r) {
            constexpr int R = decltype(r)::value;
            if (kv.dim <= 64) return pd_launch<T, TQ, 64, 3, R>(p, type, weights, weights_stride, st);
            if (kv.dim <= 128) return pd_launch<T, TQ, 128, 2, R>(p, type, weights, weights_stride, st);
            return pd_launch<T, TQ, 256, 2, R>(p, type, weights, weights_stride, st);
        };
        // FMAs go by rows: half of eight where the group has no more
        if constexpr (sizeof(T) == 4) {
            if (p.group <= 4) return rows(std::integral_constant<int, 4>());
        }
        return rows(std::integral_constant<int, PD_ROWS>());
    };
    if (type == CERA_TYPE_F32) return go(float(), float());
    if (type == CERA_TYPE_F16) return q_type == type ? go(__half(), __half()) : go(__half(), float());
    return q_type == type ? go(__nv_bfloat16(), __nv_bfloat16()) : go(__nv_bfloat16(), float());
}

}  // namespace cera
