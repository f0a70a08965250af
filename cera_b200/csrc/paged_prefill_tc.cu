// Causal attention of ragged prompt portions over a paged 16-bit cache on tcgen05, with a sliding window and first slots that stay visible.
//
// A row is (token, query head of a KV head), so a tile of 128 rows shares every staged key and value among the group's heads, whatever
// their number.  A CTA owns up to two tiles of one (sequence, KV head) and walks tiles of KT keys: S = Q K^T into TMEM, softmax by a warpgroup a
// tile (thread = row) in f32, P back into TMEM over S, O += P V with V as it lies in the cache (the product's transposed operand).  Two warps
// load keys and values by TMA, a box of a page's slots an instruction (row by row where pages do not hold whole boxes), one warp
// issues the products.  The tensor cores form one tile's products while the other tile's warpgroup is at its softmax.  The products of a tile
// follow one another in the tensor pipe, so S of the next keys may go where P of these is still being read, and when S is complete O
// is too: the warpgroup that finds a maximum raised by more than 2^8 rescales O on the spot.
//
// Weights enter their product as a sum of two parts of the cache's type (f16 22 bits, bf16 16; as one part they put the result, rounded to 16 bits, 1.4 times as far off).
// f32 queries over a 16-bit cache: the query and the weights enter as sums of NP parts of the cache's type (two f16, 22 bits; three
// bf16, 24), a product each; f16 parts are scaled by a power of two per row, weights by 2^7.  The tensor cores cut a sum at every step instead of rounding it, which
// a long row would show (5500 slots in one sum: 4.7e-6 off for f16 and 6.6e-6 for bf16, 1.5e-6 with torch's f32 products): the least parts of the queries come first, and after
// 128 slots O is added to an f32 sum and begun anew (8.7e-7 and 8.9e-7; 1500 queries of 32 heads over them, unsplit, 329 -> 353 us and 587 -> 576).  That sum is in TMEM as far as there is room:
// all of it in local memory takes 536 and 709 us, whose bytes all come from L2.  With 16-bit queries O is emptied likewise, but seldom
// (pp_flush; 131 072 slots of one sign in one sum lose 1.5e-4 with weights of one part).
//
// Few rows over a long cache: the keys are split over gridDim.z CTAs and paged_prefill_join_kernel adds the parts up.
//
// A row that ends without finite values - a weight of zero times an infinite value of a key it does not see, an infinity cut into parts - or
// that has met no weight is computed again by paged_attend_row, which reads nothing that the row does not see.  Every wait is bounded.
#include "mma.cuh"
#include "paged_prefill.cuh"
#include "tc.cuh"

namespace cera {

__device__ unsigned int g_paged_prefill_status = 0;

static const bool g_paged_prefill_registered = register_kernel_status([] {
    unsigned int v = 0;
    cudaMemcpyFromSymbol(&v, g_paged_prefill_status, sizeof(v));
    return STATUS_PAGED_PREFILL.of(v);
});

namespace {

constexpr uint32_t PP_ROWS = 128;
constexpr float PP_LIFT = 7.0f, PP_RAISE = 8.0f;
constexpr uint32_t PP_MATH_REGS = 208, PP_LOAD_REGS = 80;  // of a thread, where there are two tiles of rows: of 168 x 384 at the launch 1024 less
constexpr uint32_t PP_MASKS = 4;  // tiles whose masks are kept: more than the keys' stages and one

// Shapes by the padded head size and the number of parts.
template <int DP, int NP>
struct Pp {
    static constexpr int MT = DP <= 128 ? 2 : 1, WP = NP == 1 ? 2 : NP;  // parts of a weight
    static constexpr int KT = NP == 1 ? 128 : DP == 256 && NP == 3 ? 32 : 64;
    static constexpr uint32_t QPART = PP_ROWS * DP * 2, QBLOCK = PP_ROWS * 128, KBLOCK = KT * 128, HALF = KT * DP * 2;
    static constexpr int ST = (227 * 1024 - 2048 - MT * NP * (int)QPART) / (2 * (int)HALF) >= 3 ? 3 : (227 * 1024 - 2048 - MT * NP * (int)QPART) / (2 * (int)HALF);
    static constexpr uint32_t P_COLS = KT / 2, S_COLS = ((WP * P_COLS > KT ? WP * P_COLS : KT) + 31) / 32 * 32, T_COLS = S_COLS + DP;  // TMEM columns of a tile: S or P, then O
    static constexpr uint32_t SPARE = (512 - MT * T_COLS) / MT / 32 * 32, KEPT = NP == 1 ? 0 : SPARE < DP ? SPARE : DP;  // numbers of a row's sum that TMEM has room for
    static constexpr int MATH = 4 * MT, THREADS = 32 * (MATH + 4);  // warpgroups: softmax of a tile each; products, two loaders and a warp of nothing
    static constexpr size_t SMEM = 1024 + (size_t)MT * NP * QPART + (size_t)ST * 2 * HALF;
    static_assert(ST >= 1 && MT * T_COLS <= 512, "does not fit");
};

// Tiles that O adds up, a power of two.  The tensor cores cut a sum at every step (16 slots of one part): 8192 steps lost 1.5e-4, and a step 2^-23 at most.  With 16-bit queries, whose
// result is rounded itself, 4096 slots (f16: 512 steps, 6e-5 at most of 4.9e-4) or 32 768 (bf16: 4096 steps, 4.9e-4 of 3.9e-3).
template <typename T, int DP, int NP>
constexpr uint32_t pp_flush = (NP > 1 ? 128 : std::is_same<T, __half>::value ? 4096 : 32768) / Pp<DP, NP>::KT;

struct PpBars {
    uint64_t q_full, v_part, k_full[3], k_empty[3], v_full[3], v_empty[3], s_full[2], p_full[2], p_low[2], o_full[2];
};

__device__ __forceinline__ float pp_max3(float a, float b, float c) {
    float y;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
          "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
}
// Waits for every load so far; what follows uses these registers.
__device__ __forceinline__ void tmem_wait_ld32(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]),
                   "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                   "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])::"memory");
}
__device__ __forceinline__ void tmem_wait_ld16(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]),
                   "+r"(r[13]), "+r"(r[14]), "+r"(r[15])::"memory");
}
// D (+)= A[tmem] * B[smem], kind::f16.
__device__ __forceinline__ void tc_mma_f16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate, uint32_t me) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "setp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(tmem_d), "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate), "r"(me)
        : "memory");
}
// A tile of values as the product's second operand, rows of its k (keys) and numbers of its n contiguous: 8-row groups 1024 bytes apart, 64-number
// blocks `block` bytes apart.
__device__ __forceinline__ uint64_t pp_desc_v(uint32_t addr, uint32_t block) {
    return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)(block >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ uint32_t pp_idesc(bool bf, uint32_t N, bool n_major) {
    return (1u << 4) | ((bf ? 1u : 0u) << 7) | ((bf ? 1u : 0u) << 10) | ((n_major ? 1u : 0u) << 16) | ((N >> 3) << 17) | ((PP_ROWS >> 4) << 24);
}
template <typename T>
__device__ __forceinline__ uint32_t pp_pack(float x, float y) {
    if (std::is_same<T, __half>::value) {
        const __half2 h = __floats2half2_rn(x, y);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t *>(&h);
}
template <typename T>
__device__ __forceinline__ float2 pp_unpack(uint32_t w) {
    if (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2 *>(&w));
    return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&w));
}
// (x, y) as a sum of NP pairs of T.
template <typename T, int NP>
__device__ __forceinline__ void pp_parts(float x, float y, uint32_t (&w)[NP]) {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        w[i] = pp_pack<T>(x, y);
        if (i + 1 < NP) {
            const float2 f = pp_unpack<T>(w[i]);
            x -= f.x;
            y -= f.y;
        }
    }
}

// The keys' or the values' loader, a warp.
template <typename T, int DP, int NP, bool TMA>
__device__ __forceinline__ void pp_load(const PpParams &p, const PpWork &w, const CUtensorMap *map, bool is_v, uint8_t *stages, uint64_t *full, uint64_t *empty,
                                        uint64_t *part, uint32_t (*masks)[4], volatile uint32_t *abort_flag, unsigned int *status) {
    using C = Pp<DP, NP>;
    const uint32_t lane = threadIdx.x & 31, h = blockIdx.y, boxes = C::KT / p.box, blocks = (p.kv.dim + 63) / 64, me = elect_one();
    const size_t by_page = is_v ? p.kv.v_page : p.kv.k_page, by_slot = is_v ? p.kv.v_slot : p.kv.k_slot, by_head = is_v ? p.kv.v_head : p.kv.k_head;
    const uint8_t *base = is_v ? p.kv.v : p.kv.k;
    constexpr int N = (C::KT + 31) / 32;
    uint32_t page[N], row[N];
    // with TMA lane i looks up box i, otherwise a lane the slots lane, lane + 32 ... of the tile
    auto find = [&](uint32_t x) {
        const uint32_t slot0 = w.span.slot(x, C::KT);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            page[i] = NO_PAGE;
            row[i] = 0;
            if (TMA) {
                const uint32_t j = slot0 + lane * p.box;
                if (i == 0 && lane < boxes && j < w.span.len && (j + p.box > w.span.first || j < w.span.sinks)) page[0] = paged_at(p.kv, w.s, j, row[0]);
            } else {
                const uint32_t j = slot0 + lane + 32 * i;
                if (w.span.sees(j)) page[i] = paged_at(p.kv, w.s, j, row[i]);
            }
        }
    };
    uint32_t parts = 0;
    // shared memory must outlive the copies in flight, those of the stages before tile n and, if the last was not whole, its own: whoever reads them may give up while they are
    auto drain = [&](uint32_t n, bool all) {
        for (uint32_t y = n > C::ST ? n - C::ST : 0; y < n; ++y)
            for (uint32_t i = 0; i < tma::SPIN_LIMIT && !tma::mbar_test(&full[y % C::ST], y / C::ST & 1); ++i) __nanosleep(40);
        for (uint32_t i = 0; !all && i < tma::SPIN_LIMIT && !tma::mbar_test(part, (parts - 1) & 1); ++i) __nanosleep(40);
    };
    if (w.x0 < w.x1) find(w.x0);
    for (uint32_t x = w.x0; x < w.x1; ++x) {
        const uint32_t i0 = x - w.x0, st = i0 % C::ST, slot0 = w.span.slot(x, C::KT);
        uint32_t pg[N], rw[N], mask[N];
        const uint32_t live = __ballot_sync(0xffffffffu, page[0] != NO_PAGE);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            pg[i] = page[i];
            rw[i] = row[i];
            const uint32_t j = lane + 32 * i;
            mask[i] = __ballot_sync(0xffffffffu, TMA ? w.span.sees(slot0 + j) && (live >> j / p.box & 1) : pg[i] != NO_PAGE);
        }
        if (x + 1 < w.x1) find(x + 1);  // its answer is not needed before the next tile
        if (!tma::mbar_wait_warp(&empty[st], (i0 / C::ST & 1) ^ 1, abort_flag, status, 1u)) return drain(i0, true);
        if (!is_v) {
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (lane == (uint32_t)i) masks[i0 % PP_MASKS][i] = mask[i];
        }
        __syncwarp();
        uint8_t *to = stages + st * C::HALF;
        // rows of values that are not seen are set to zero when the rest is there: a weight of zero times what lies there could be a NaN
        bool whole = !is_v;
        if (is_v) {
            whole = true;
#pragma unroll
            for (int i = 0; i < N; ++i) whole = whole && mask[i] == 0xffffffffu;
        }
        auto clear = [&]() {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                if (mask[i] >> lane & 1) continue;
                for (uint32_t c = 0; c < blocks * 8; ++c) *reinterpret_cast<uint4 *>(to + (c >> 3) * C::KBLOCK + (32 * i + lane) * 128 + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
            }
        };
        if (TMA) {
            uint64_t *bar = whole ? &full[st] : part;
            tma::mbar_expect_tx_if(bar, __popc(live) * blocks * p.box * 128, me);
            for (uint32_t i = 0; i < boxes; ++i) {
                const uint32_t pi = __shfl_sync(0xffffffffu, pg[0], i), ri = __shfl_sync(0xffffffffu, rw[0], i);
                if (pi == NO_PAGE) continue;
                for (uint32_t k = 0; k < blocks; ++k) tma::tensor_g2s_4d_if(to + k * C::KBLOCK + i * p.box * 128, map, k * 64, h, ri, pi, bar, me);
            }
            if (!whole) {
                if (!tma::mbar_wait_warp(part, parts++ & 1, abort_flag, status, 1u)) return drain(i0, false);
                clear();
                fence_async_smem();
                __syncwarp();
                if (lane == 0) tma::mbar_arrive(&full[st]);
            }
        } else {
            const uint32_t per = blocks * 8, used = p.kv.dim / 8;
#pragma unroll
            for (int n = 0; n < N; ++n) {
                const uint64_t off = pg[n] != NO_PAGE ? pg[n] * (uint64_t)by_page + rw[n] * (uint64_t)by_slot + h * (uint64_t)by_head : 0;
                for (uint32_t i = lane; i < 32 * per; i += 32) {
                    const uint32_t r = i / per, c = i - r * per;
                    const uint64_t o = __shfl_sync(0xffffffffu, off, r);
                    if (c < used && (mask[n] >> r & 1)) tma::cp_async16(to + (c >> 3) * C::KBLOCK + (32 * n + r) * 128 + ((c & 7) ^ (r & 7)) * 16, base + o + c * 16);
                }
            }
            // what these copies write is read by the tensor cores: complete, fenced, then announced
            asm volatile("cp.async.wait_all;" ::: "memory");
            if (!whole) clear();
            fence_async_smem();
            __syncwarp();
            if (lane == 0) tma::mbar_arrive(&full[st]);
        }
    }
    drain(w.x1 - w.x0, true);
}

// The products, a warp that stays together (descriptors live in registers that a warp has once: a branch of one lane around them mixes them up): of each tile of rows
// in turn O += P V of these keys, then S of the next.
template <typename T, int DP, int NP>
__device__ __forceinline__ void pp_multiply(const PpParams &p, const PpWork &w, uint8_t *qs, uint8_t *ks, uint8_t *vs, uint32_t tmem, PpBars *b, volatile uint32_t *abort_flag,
                                            unsigned int *status) {
    using C = Pp<DP, NP>;
    constexpr bool BF = !std::is_same<T, __half>::value;
    constexpr uint32_t FLUSH = pp_flush<T, DP, NP>;
    const uint32_t me = elect_one(), id_s = pp_idesc(BF, C::KT, false), id_o = pp_idesc(BF, p.kv.dim, true), n = w.x1 - w.x0, steps = p.kv.dim / 16;
    const uint64_t q0 = smem_desc_sw128(tma::smem_u32(qs)), k0 = smem_desc_sw128(tma::smem_u32(ks)), v0 = pp_desc_v(tma::smem_u32(vs), C::KBLOCK);  // address fields count 16 bytes
    auto arrived = [&](uint64_t *bar, uint32_t parity) { return tma::mbar_wait_warp(bar, parity, abort_flag, status, 2u); };
    uint32_t added[2] = {0, 0};
    auto score = [&](uint32_t t, uint32_t st) {
        const uint32_t d = tmem + t * C::T_COLS;
        const uint64_t kd = k0 + st * (C::HALF / 16);
#pragma unroll 1
        for (int part = 0; part < NP; ++part) {
            const uint64_t qd = q0 + (t * NP + NP - 1 - part) * (C::QPART / 16);  // the least first: sums are cut, not rounded, at every step
#pragma unroll
            for (uint32_t k = 0; k < DP / 16; ++k)
                if (k < steps) tc_mma_f16(d, qd + (k >> 2) * (C::QBLOCK / 16) + 2 * (k & 3), kd + (k >> 2) * (C::KBLOCK / 16) + 2 * (k & 3), id_s, part | k, me);
        }
        tc_commit(&b->s_full[t], me);
    };
    if (n == 0 || !arrived(&b->q_full, 0) || !arrived(&b->k_full[0], 0)) return;
    tc_fence_after();
    uint32_t slot = w.span.slot(w.x0, C::KT);
    bool sees[2] = {pp_sees<C::KT>(p, w, 0, slot), C::MT == 2 && pp_sees<C::KT>(p, w, 1, slot)};
#pragma unroll
    for (uint32_t t = 0; t < C::MT; ++t)
        if (sees[t]) score(t, 0);
    tc_commit(&b->k_empty[0], me);
    uint32_t st = 0, turn = 0;  // the stage of these keys and how often the ring has gone round
    for (uint32_t i = 0; i < n; ++i) {
        const bool more = i + 1 < n;
        const uint32_t next = st + 1 == C::ST ? 0 : st + 1, next_turn = st + 1 == C::ST ? turn ^ 1 : turn;
        bool then[2] = {false, false};
        // what was loaded is waited for ahead of the weights, which are what is waited for in earnest; a stage that no tile of rows sees has to have arrived too
        // before it is filled again
        if (more) {
            slot = w.span.slot(w.x0 + i + 1, C::KT);
            then[0] = pp_sees<C::KT>(p, w, 0, slot);
            then[1] = C::MT == 2 && pp_sees<C::KT>(p, w, 1, slot);
            if (!arrived(&b->k_full[next], next_turn)) return;
        }
        if (!arrived(&b->v_full[st], turn)) return;
#pragma unroll
        for (uint32_t t = 0; t < C::MT; ++t) {
            if (sees[t]) {
                if (!arrived(&b->p_full[t], added[t] & 1)) return;
                tc_fence_after();
                const uint32_t s = tmem + t * C::T_COLS, o = s + C::S_COLS;
                const uint64_t vd = v0 + st * (C::HALF / 16);
#pragma unroll 1
                for (int part = 0; part < C::WP; ++part) {
                    if (NP == 1 && part) {  // the lower parts come while the upper ones are multiplied
                        if (!arrived(&b->p_low[t], added[t] & 1)) return;
                        tc_fence_after();
                    }
#pragma unroll
                    for (uint32_t k = 0; k < C::KT / 16; ++k) tc_mma_f16_ts(o, s + part * C::P_COLS + 8 * k, vd + k * (2048 / 16), id_o, added[t] % FLUSH | part | k, me);
                }
                ++added[t];
            }
            if (t + 1 == C::MT) tc_commit(&b->v_empty[st], me);
            if (then[t]) score(t, next);
        }
        if (more) tc_commit(&b->k_empty[next], me);
        st = next;
        turn = next_turn;
        sees[0] = then[0];
        sees[1] = then[1];
    }
#pragma unroll
    for (uint32_t t = 0; t < C::MT; ++t) tc_commit(&b->o_full[t], me);
}

// A tile's queries into shared memory -> the factor of the lane's row's scores, in units of ln 2.  f32: by warps, a row's pieces of 16 bytes a lane each (a thread a row, whose lines do
// not stay in what shared memory leaves of L1, takes 37 us for a prompt of 512, this 32).  Others: a thread a row (8000 tokens through a window of 4096: by warps 3 % longer).
template <typename T, typename TQ, int DP, int NP>
__device__ __forceinline__ float pp_queries(const PpParams &p, const PpWork &w, uint32_t row, uint8_t *to, uint32_t r) {
    using C = Pp<DP, NP>;
    constexpr int U = 4, L = DP == 256 ? 2 : 1;  // rows at once, loads of a lane
    const uint32_t lane = r & 31, pieces = p.kv.dim * (uint32_t)sizeof(TQ) / 16;
    const bool live = row < w.rows;
    const uint64_t mine = live ? ((uint64_t)(w.t0 + row / p.group) * p.heads + blockIdx.y * p.group + row % p.group) * p.kv.dim : ~0ull;
    // a scale below zero turns the queries; one of zero is multiplied into them, so that what is not finite becomes a NaN and what is not seen stays minus infinity
    const bool turn = p.scale < 0.0f, none = p.scale == 0.0f;
    float factor = none ? 1.0f : fabsf(p.scale) * PAGED_LOG2E;
    if (NP == 1) {
        const uint32_t flip = turn ? 0x80008000u : 0;
        auto zero = [](uint32_t x) {
            const float2 f = pp_unpack<T>(x);
            return pp_pack<T>(f.x * 0.0f, f.y * 0.0f);
        };
        for (uint32_t c0 = 0; c0 < pieces; c0 += 4) {
            uint4 v[4];
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) v[i] = live ? reinterpret_cast<const uint4 *>(reinterpret_cast<const TQ *>(p.q) + mine)[c0 + i] : make_uint4(0, 0, 0, 0);
            if (none) {
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) v[i] = make_uint4(zero(v[i].x), zero(v[i].y), zero(v[i].z), zero(v[i].w));
            }
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                const uint32_t c = c0 + i;
                *reinterpret_cast<uint4 *>(to + (c >> 3) * C::QBLOCK + r * 128 + ((c & 7) ^ (r & 7)) * 16) = make_uint4(v[i].x ^ flip, v[i].y ^ flip, v[i].z ^ flip, v[i].w ^ flip);
            }
        }
        return factor;
    }
    for (uint32_t i0 = 0; i0 < 32; i0 += U) {
        uint4 v[U][L];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint64_t at = __shfl_sync(0xffffffffu, mine, i0 + u);
#pragma unroll
            for (int k = 0; k < L; ++k)
                v[u][k] = at != ~0ull && lane + 32 * k < pieces ? reinterpret_cast<const uint4 *>(reinterpret_cast<const TQ *>(p.q) + at)[lane + 32 * k] : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t rr = r - lane + i0 + u;
            float mul = none ? 0.0f : turn ? -1.0f : 1.0f;
            if (std::is_same<T, __half>::value) {
                uint32_t most = 0;  // of absolute values, whose bits are in their order
#pragma unroll
                for (int k = 0; k < L; ++k) most = max(max(max(most, v[u][k].x & 0x7fffffffu), max(v[u][k].y & 0x7fffffffu, v[u][k].z & 0x7fffffffu)), v[u][k].w & 0x7fffffffu);
                most = __reduce_max_sync(0xffffffffu, most);
                const int e = most && most < 0x7f800000u ? min(max((int)(most >> 23) - 127, -120), 120) : 0;
                mul *= __uint_as_float((uint32_t)(127 - e) << 23);
                if (lane == i0 + u) factor *= __uint_as_float((uint32_t)(127 + e) << 23);
            }
#pragma unroll
            for (int k = 0; k < L; ++k) {
                const uint32_t c = lane + 32 * k;
                if (c >= pieces) break;
                uint32_t lo[NP], hi[NP];
                pp_parts<T, NP>(__uint_as_float(v[u][k].x) * mul, __uint_as_float(v[u][k].y) * mul, lo);
                pp_parts<T, NP>(__uint_as_float(v[u][k].z) * mul, __uint_as_float(v[u][k].w) * mul, hi);
#pragma unroll
                for (int n = 0; n < NP; ++n)
                    *reinterpret_cast<uint2 *>(to + n * C::QPART + (c >> 4) * C::QBLOCK + rr * 128 + ((c >> 1 & 7) ^ (rr & 7)) * 16 + (c & 1) * 8) = make_uint2(lo[n], hi[n]);
            }
        }
    }
    return factor;
}

// Softmax and result of a tile of rows, a warpgroup.
template <typename T, typename TQ, int DP, int NP>
__device__ __forceinline__ void pp_softmax(const PpParams &p, const PpWork &w, uint32_t t, uint8_t *qs, uint32_t tmem, PpBars *b, const uint32_t (*masks)[4],
                                           volatile uint32_t *abort_flag, unsigned int *status) {
    using C = Pp<DP, NP>;
    constexpr uint32_t FLUSH = pp_flush<T, DP, NP>;
    const uint32_t lane = threadIdx.x & 31, quad = threadIdx.x >> 5 & 3, r = quad * 32 + lane, row = w.row0 + t * PP_ROWS + r;
    const uint32_t ts = tmem + t * C::T_COLS + (quad * 32 << 16), to = ts + C::S_COLS;
    const float c = pp_queries<T, TQ, DP, NP>(p, w, row, qs + t * NP * C::QPART, r);
    fence_async_smem();
    __syncwarp();
    if (lane == 0) tma::mbar_arrive(&b->q_full);

    const uint32_t a = w.row0 + t * PP_ROWS;
    const bool live = row < w.rows;
    const int32_t pos = live ? w.slot_of(row, p.group) : -1;
    const int32_t p_lo = t ? w.lo1 : w.lo0, p_hi = t ? w.hi1 : w.hi0;
    const int32_t first = pos >= 0 ? (int32_t)paged_first(p.mask, (uint32_t)pos) : 0, first_hi = p_hi >= 0 ? (int32_t)paged_first(p.mask, (uint32_t)p_hi) : 0;
    const int32_t sinks = (int32_t)min(p.mask.sink, (uint32_t)max(first, 0));
    float m = PP_FLOOR, l = 0.0f;
    uint32_t done = 0;
    bool ok = true;
    // the sums of whole groups of FLUSH tiles, the first KEPT numbers in TMEM and the others in local memory
    const uint32_t ta = tmem + C::MT * C::T_COLS + t * C::KEPT + (quad * 32 << 16);
    constexpr int FAR = DP - (int)C::KEPT;
    alignas(16) float far[FAR ? FAR : 1];
    // f(number, its sum) for every number of the row, 32 at a time
    auto sums = [&](auto f) {
#pragma unroll
        for (int d = 0; d < (int)C::KEPT; d += 32) {
            if ((uint32_t)d >= p.kv.dim) break;
            uint32_t s[32];
            tmem_ld32(ta + d, s);
            tmem_wait_ld32(s);
            f(d, s);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t x[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) x[e] = s[16 * h + e];
                tmem_st16(ta + d + 16 * h, x);
            }
        }
        if (C::KEPT) tmem_wait_st();
#pragma unroll
        for (int d = 0; d < FAR; d += 32) {
            if (C::KEPT + d >= p.kv.dim) break;
            uint32_t s[32];
#pragma unroll
            for (int e = 0; e < 32; ++e) s[e] = __float_as_uint(far[d + e]);
            f(C::KEPT + d, s);
#pragma unroll
            for (int e = 0; e < 32; ++e) far[d + e] = __uint_as_float(s[e]);
        }
    };
    float m_far = PP_FLOOR;  // 16-bit queries: the maximum that `far` stands for
    auto flush = [&] {
        sums([&](uint32_t d, uint32_t (&s)[32]) {
            uint32_t o[32];
            tmem_ld32(to + d, o);
            tmem_wait_ld32(o);
#pragma unroll
            for (int e = 0; e < 32; ++e) s[e] = done == FLUSH ? o[e] : __float_as_uint(__uint_as_float(s[e]) + __uint_as_float(o[e]));
        });
    };
    for (uint32_t i = 0; i < w.x1 - w.x0; ++i) {
        const uint32_t slot0 = w.span.slot(w.x0 + i, C::KT);
        if (!pp_sees<C::KT>(p, w, t, slot0)) continue;
        ok = tma::mbar_wait_warp(&b->s_full[t], done & 1, abort_flag, status, 4u);
        if (!ok) break;
        tc_fence_after();
        if (NP > 1 && done && done % FLUSH == 0) flush();  // O is complete up to the tile before, and begins anew
        // which of the tile's keys this row sees; nothing to look at where every row sees all
        uint32_t see[(C::KT + 31) / 32];
        bool all = (int32_t)(slot0 + C::KT) <= p_lo + 1 && ((int32_t)slot0 >= first_hi || slot0 + C::KT <= p.mask.sink);
#pragma unroll
        for (int k = 0; k < (C::KT + 31) / 32; ++k) {
            see[k] = masks[i % PP_MASKS][k];
            all = all && see[k] == 0xffffffffu;
        }
        if (!all) {
#pragma unroll
            for (int k = 0; k < (C::KT + 31) / 32; ++k) {
                const int32_t at = (int32_t)slot0 + 32 * k;
                see[k] &= pp_low(pos + 1 - at) & (~pp_low(first - at) | pp_low(sinks - at));
            }
        }
        // f32 queries: weights for the maximum that is known; where the tile has a score past it by more than 2^8, O and the
        // sum are rescaled and the weights, whose scores are still in registers, formed again.  16-bit queries: the maximum first, then the weights' upper parts, which take
        // the place of the scores, and the lower parts beside the upper ones' product (all of a weight at once: 752 us for 8000 tokens through a window of 4096, 620 so).
        constexpr int Q = C::KT / 32;
        uint32_t v[Q][32];
#pragma unroll
        for (int j = 0; j < Q; ++j) tmem_ld32(ts + 32 * j, v[j]);
#pragma unroll
        for (int j = 0; j < Q; ++j) tmem_wait_ld32(v[j]);  // one wait, and no barrier to the order of what follows
        float2 base = make_float2(PP_LIFT - m, PP_LIFT - m), sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
        const float2 cc = make_float2(c, c);
        auto form = [&](int j) {
            uint32_t wd[NP][16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                float2 x = __ffma2_rn(make_float2(__uint_as_float(v[j][2 * e]), __uint_as_float(v[j][2 * e + 1])), cc, base);
                x = make_float2(pp_exp2(x.x), pp_exp2(x.y));
                sum[e & 1] = __fadd2_rn(sum[e & 1], x);
                uint32_t u[NP];
                pp_parts<T, NP>(x.x, x.y, u);
#pragma unroll
                for (int n = 0; n < NP; ++n) wd[n][e] = u[n];
                if (NP == 1) {
                    v[j][2 * e] = __float_as_uint(x.x);
                    v[j][2 * e + 1] = __float_as_uint(x.y);
                }
            }
#pragma unroll
            for (int n = 0; n < NP; ++n) tmem_st16(ts + n * C::P_COLS + 16 * j, wd[n]);
        };
        float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        auto stream = [&](auto whole) {
#pragma unroll
            for (int j = 0; j < Q; ++j) {
                if (!decltype(whole)::value) {
#pragma unroll
                    for (int e = 0; e < 32; ++e) v[j][e] = see[j] >> e & 1 ? v[j][e] : 0xff800000u;
                }
#pragma unroll
                for (int e = 0; e < 32; e += 8)
#pragma unroll
                    for (int i = 0; i < 4; ++i) top[i] = pp_max3(top[i], __uint_as_float(v[j][e + 2 * i]), __uint_as_float(v[j][e + 2 * i + 1]));
                if (NP > 1) form(j);
            }
        };
        if (all) stream(std::true_type());
        else stream(std::false_type());
        const float mx = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * c;
        const bool raise = mx > m + PP_RAISE;
        if (__any_sync(0xffffffffu, raise)) {
            const float f = raise ? pp_exp2(m - mx) : 1.0f;
            if (raise) m = mx;
            l *= f;
            if (NP > 1 && done >= FLUSH)
                sums([&](uint32_t, uint32_t (&s)[32]) {
#pragma unroll
                    for (int e = 0; e < 32; ++e) s[e] = __float_as_uint(__uint_as_float(s[e]) * f);
                });
            for (uint32_t d = 0; done && d < p.kv.dim; d += 16) {  // O is complete up to the tile before, and nothing adds to it
                uint32_t o[16];
                tmem_ld16(to + d, o);
                tmem_wait_ld16(o);
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                tmem_st16(to + d, o);
            }
            base = make_float2(PP_LIFT - m, PP_LIFT - m);
            sum[0] = sum[1] = make_float2(0.0f, 0.0f);
            if (NP > 1) {
#pragma unroll
                for (int j = 0; j < Q; ++j) form(j);
            }
        }
        if (NP == 1) {
            if (done && done % FLUSH == 0) {  // O goes to `far` and begins anew
                const float f = pp_exp2(m_far - m);
                m_far = m;
#pragma unroll 1
                for (uint32_t d = 0; d < p.kv.dim; d += 16) {
                    uint32_t o[16];
                    tmem_ld16(to + d, o);
                    tmem_wait_ld16(o);
#pragma unroll
                    for (int e = 0; e < 16; ++e) far[NP == 1 ? d + e : 0] = done == FLUSH ? __uint_as_float(o[e]) : fmaf(far[NP == 1 ? d + e : 0], f, __uint_as_float(o[e]));
                }
            }
#pragma unroll
            for (int j = 0; j < Q; ++j) form(j);
        }
        l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) tma::mbar_arrive(&b->p_full[t]);
        if (NP == 1) {
#pragma unroll
            for (int j = 0; j < Q; ++j) {
                uint32_t wd[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    uint32_t u[2];
                    pp_parts<T, 2>(__uint_as_float(v[j][2 * e]), __uint_as_float(v[j][2 * e + 1]), u);
                    wd[e] = u[1];
                }
                tmem_st16(ts + C::P_COLS + 16 * j, wd);
            }
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) tma::mbar_arrive(&b->p_low[t]);
        }
        ++done;
    }
    if (ok && done) ok = tma::mbar_wait_warp(&b->o_full[t], 0, abort_flag, status, 4u);
    if (!ok) return;
    tc_fence_after();
    if (NP == 1 && done > FLUSH) {
        const float f = pp_exp2(m_far - m);
#pragma unroll 1
        for (uint32_t d = 0; d < p.kv.dim; d += 16) {
            uint32_t o[16];
            tmem_ld16(to + d, o);
            tmem_wait_ld16(o);
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(fmaf(far[NP == 1 ? d + e : 0], f, __uint_as_float(o[e])));
            tmem_st16(to + d, o);
        }
        tmem_wait_st();
    }
    if (NP > 1 && done > FLUSH) {  // O joins the sums
        sums([&](uint32_t d, uint32_t (&s)[32]) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t o[16];
                tmem_ld16(to + d + 16 * h, o);
                tmem_wait_ld16(o);
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(s[16 * h + e]) + __uint_as_float(o[e]));
                tmem_st16(to + d + 16 * h, o);
            }
        });
        tmem_wait_st();
    }
    const size_t place = ((size_t)(w.t0 + row / p.group) * p.heads + blockIdx.y * p.group + row % p.group);
    if (gridDim.z > 1) {
        const size_t at = (size_t)blockIdx.z * p.n * p.heads + place;
        if (live) p.ml[at] = make_float2(l != l || m != PP_FLOOR ? m : -INFINITY, l);
        if (done)
            for (uint32_t d = 0; d < p.kv.dim; d += 32) {
                uint32_t o[32];
                tmem_ld32(to + d, o);
                tmem_wait_ld32(o);
                if (live) {
#pragma unroll
                    for (int e = 0; e < 32; e += 4) *reinterpret_cast<uint4 *>(p.part + at * p.kv.dim + d + e) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                }
            }
        return;
    }
    TQ *out = reinterpret_cast<TQ *>(p.out) + place * p.kv.dim;
    const float f = 1.0f / l;
    float check = l > 0.0f && m != PP_FLOOR ? 0.0f : NAN;
    for (uint32_t d = 0; done && d < p.kv.dim; d += 32) {
        uint32_t o[32];
        tmem_ld32(to + d, o);
        tmem_wait_ld32(o);
#pragma unroll
        for (int e = 0; e < 32; ++e) check = fmaf(__uint_as_float(o[e]) * f, 0.0f, check);
    }
    uint32_t again = __ballot_sync(0xffffffffu, pos >= 0 && check != 0.0f);
    for (uint32_t d = 0; d < p.kv.dim; d += 32) {  // what is computed again is stored then: the queries may be where the result goes
        uint32_t o[32];
        if (done) {
            tmem_ld32(to + d, o);
            tmem_wait_ld32(o);
        }
#pragma unroll
        for (int e = 0; e < 32; e += 16 / sizeof(TQ)) {
            alignas(16) TQ y[16 / sizeof(TQ)];
#pragma unroll
            for (uint32_t k = 0; k < 16 / sizeof(TQ); ++k) {
                const float x = done ? __uint_as_float(o[e + k]) * f : 0.0f;
                y[k] = from_f32<TQ>(pos >= 0 ? x : 0.0f);
            }
            if (live && !(again >> lane & 1)) *reinterpret_cast<uint4 *>(out + d + e) = *reinterpret_cast<const uint4 *>(y);
        }
    }
    for (; again; again &= again - 1) {
        const uint32_t rr = a + quad * 32 + __ffs(again) - 1;
        const size_t pl = ((size_t)(w.t0 + rr / p.group) * p.heads + blockIdx.y * p.group + rr % p.group) * p.kv.dim;
        __syncwarp();
        paged_attend_row<T, TQ>(p.kv, p.mask, w.s, blockIdx.y, (uint32_t)w.slot_of(rr, p.group), reinterpret_cast<const TQ *>(p.q) + pl, p.scale,
                                reinterpret_cast<TQ *>(p.out) + pl);
    }
}

template <typename T, typename TQ, int DP, int NP, bool TMA>
__global__ void __launch_bounds__(Pp<DP, NP>::THREADS, 1) paged_prefill_tc_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                                                                                  const PpParams p) {
    using C = Pp<DP, NP>;
    extern __shared__ uint8_t raw[];
    __shared__ PpBars bars;
    __shared__ uint32_t masks[PP_MASKS][4], tmem_at, abort_s;
    __shared__ PpWork work;
    uint8_t *qs = raw + (1024 - (tma::smem_u32(raw) & 1023)) % 1024, *ks = qs + C::MT * NP * C::QPART, *vs = ks + C::ST * C::HALF;
    const uint32_t warp = threadIdx.x >> 5;
    pdl_trigger();
    pdl_wait();
    if (warp == 0) {
        PpWork w;
        const bool found = pp_find<C::MT * PP_ROWS>(p, w, blockIdx.x);
        if (found) pp_set<C::MT * PP_ROWS, PP_ROWS, C::KT>(p, w);
        else w.rows = 0;
        if (threadIdx.x == 0) {
            work = w;
            abort_s = 0;
            tma::mbar_init(&bars.q_full, C::MATH);
            tma::mbar_init(&bars.v_part, 1);
            for (int i = 0; i < 3; ++i) {
                tma::mbar_init(&bars.k_full[i], 1);
                tma::mbar_init(&bars.v_full[i], 1);
                tma::mbar_init(&bars.k_empty[i], 1);
                tma::mbar_init(&bars.v_empty[i], 1);
            }
            for (int i = 0; i < 2; ++i) {
                tma::mbar_init(&bars.s_full[i], 1);
                tma::mbar_init(&bars.p_full[i], 4);
                tma::mbar_init(&bars.p_low[i], 4);
                tma::mbar_init(&bars.o_full[i], 1);
            }
            tma::mbar_init_fence();
        }
        __syncwarp();
    }
    __syncthreads();
    const PpWork w = work;
    if (w.rows == 0) return;
    if (warp == C::MATH) {
        tmem_alloc(&tmem_at, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_at;
    unsigned int *status = &g_paged_prefill_status;
    if (warp < C::MATH) {
        if (C::MT == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(PP_MATH_REGS));
        pp_softmax<T, TQ, DP, NP>(p, w, warp / 4, qs, tmem, &bars, masks, &abort_s, status);
    } else {
        if (C::MT == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(PP_LOAD_REGS));
        if (warp == C::MATH) {
            pp_multiply<T, DP, NP>(p, w, qs, ks, vs, tmem, &bars, &abort_s, status);
        } else if (warp < C::MATH + 3) {
            const bool is_v = warp == C::MATH + 2;
            pp_load<T, DP, NP, TMA>(p, w, is_v ? &map_v : &map_k, is_v, is_v ? vs : ks, is_v ? bars.v_full : bars.k_full, is_v ? bars.v_empty : bars.k_empty, &bars.v_part, masks, &abort_s,
                                    status);
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == C::MATH) tmem_dealloc(tmem, 512);
}

// np: parts of a query.
uint32_t pp_tc_splits(const PagedView &kv, size_t n_heads, size_t n, int np, PagedMask mask) {
    const size_t rows = (kv.dim <= 128 ? 2 : 1) * PP_ROWS;
    const PpCost cost = {(np == 1 ? 1.3f : np == 2 ? 2.3f : 3.7f) * kv.dim / 128, np == 1 ? 9.0f : 14.0f};
    return pp_splits(kv, n_heads, n, rows, pp_units(kv, n_heads, n, rows), cost, mask);
}
// With any queries and mask.
uint32_t pp_tc_most(const PagedView &kv, size_t n_heads, size_t n) {
    uint32_t most = 1;
    for (int np = 1; np <= 3; ++np) most = std::max(most, pp_tc_splits(kv, n_heads, n, np, PagedMask{0, 0}));
    return most;
}

// A warpgroup that asks for registers which the block was not launched with waits for good: a build that gave the kernel fewer is refused.
template <auto KERNEL>
int32_t pp_registers(uint32_t threads) {
    static thread_local int asked = -1;
    int dev = 0;
    CERA_CUDA_TRY(cudaGetDevice(&dev));
    if (asked == dev) return CERA_CUDA_OK;
    cudaFuncAttributes a;
    CERA_CUDA_TRY(cudaFuncGetAttributes(&a, KERNEL));
    if ((uint32_t)(a.numRegs + 7) / 8 * 8 * threads < (threads - 128) * PP_MATH_REGS + 128 * PP_LOAD_REGS)
        return fail(CERA_CUDA_ERR_UNSUPPORTED, "paged_prefill_attention: built with %d registers a thread", a.numRegs);
    asked = dev;
    return CERA_CUDA_OK;
}

template <typename T, typename TQ, int DP>
int32_t pp_launch(PpParams &p, const PpGrid &g, int type, cudaStream_t st) {
    constexpr int NP = sizeof(TQ) == 2 ? 1 : std::is_same<T, __half>::value ? 2 : 3;
    using C = Pp<DP, NP>;
    CUtensorMap mk, mv;
    p.box = C::KT;
    CERA_TRY(paged_maps(p.kv, type, 8, &p.box, &mk, &mv));
    const bool by_tma = p.box != 0;
    if (!by_tma) p.box = C::KT;
    auto kernel = by_tma ? paged_prefill_tc_kernel<T, TQ, DP, NP, true> : paged_prefill_tc_kernel<T, TQ, DP, NP, false>;
    CERA_TRY((by_tma ? paged_smem<paged_prefill_tc_kernel<T, TQ, DP, NP, true>>(C::SMEM) : paged_smem<paged_prefill_tc_kernel<T, TQ, DP, NP, false>>(C::SMEM)));
    if (C::MT == 2) CERA_TRY((by_tma ? pp_registers<paged_prefill_tc_kernel<T, TQ, DP, NP, true>>(C::THREADS) : pp_registers<paged_prefill_tc_kernel<T, TQ, DP, NP, false>>(C::THREADS)));
    count_launch();
    CERA_CUDA_TRY(launch_k(kernel, dim3(g.units, p.kv.hk, g.splits), dim3(C::THREADS), C::SMEM, st, mk, mv, p));
    return pp_join<T, TQ>(p, g, st);
}

}  // namespace

size_t paged_prefill_tc_workspace(const PagedView &kv, size_t n_heads, size_t n) { return pp_workspace(pp_tc_most(kv, n_heads, n), kv, n_heads, n); }

int32_t launch_paged_prefill_tc(const PagedView &kv, int type, const void *q, int q_type, size_t n_heads, const int32_t *starts, size_t n_tokens, float scale,
                                PagedMask mask, void *out, void *ws, cudaStream_t st) {
    const int np = q_type == type ? 1 : type == CERA_TYPE_F16 ? 2 : 3;
    uint32_t splits = pp_tc_splits(kv, n_heads, n_tokens, np, mask);
    if (mask.window) splits = std::min(splits, pp_tc_splits(kv, n_heads, n_tokens, np, PagedMask{0, 0}));  // which the workspace has room for
    const PpGrid g = {(uint32_t)pp_units(kv, n_heads, n_tokens, (kv.dim <= 128 ? 2 : 1) * PP_ROWS), splits};
    PpParams p = pp_params(kv, mask, q, n_heads, starts, n_tokens, scale, out, ws, g);
    auto go = [&](auto cache, auto query) {
        using T = decltype(cache);
        using TQ = decltype(query);
        if (kv.dim <= 64) return pp_launch<T, TQ, 64>(p, g, type, st);
        if (kv.dim <= 128) return pp_launch<T, TQ, 128>(p, g, type, st);
        return pp_launch<T, TQ, 256>(p, g, type, st);
    };
    if (type == CERA_TYPE_F16) return q_type == type ? go(__half(), __half()) : go(__half(), float());
    return q_type == type ? go(__nv_bfloat16(), __nv_bfloat16()) : go(__nv_bfloat16(), float());
}

}  // namespace cera
