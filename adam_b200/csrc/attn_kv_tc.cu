// Attention of many rows over a paged fp16 cache on the 5th-generation tensor cores (see attn_kv.cu for the operator and the
// precision of its operands).
//
// A CTA has 128 rows (a token's query heads of one key head are neighbours) and walks the positions in chunks of 128:
//   S = (Q_hi + Q_lo) K^T    tcgen05.mma, both operands in shared memory, into 128 columns of tensor memory
//   P = 2^(k S - m + 8)      a row to a thread: S read twice (maximum, weights), P as two fp16 terms over S, column for column
//   O' = (P_hi + P_lo) V     tcgen05.mma, P from tensor memory, V from shared memory as it lies there (its positions are the rows)
//   O = O alpha + O'         in registers: a sum that stays in the tensor core for many chunks would lose bits (attn_kv.cu)
// Two warpgroups take the even and the odd chunks, each with its own S / P, O' and running maximum, so that the tensor core
// works on one's products while the other is at its weights; they merge at the end.  Three warps fetch keys and values
// (16 bytes at a time, so that pages may end anywhere), one thread issues the products.  Bound by the tensor core, which has two
// products where 16-bit operands would have one; the weights need about as many cycles of the other units.
#include "attn_kv.cuh"
#include "gemv_mma.cuh"

#include <type_traits>

namespace ab {

constexpr int TC_ROWS = 128, TC_CB = 128, TC_THREADS = 384, TC_LOADERS = 96;
constexpr uint32_t TC_BLOCK = 128 * 128;             // 128 rows (or positions) of 64 values: 128 bytes each, in the 128-byte swizzle

template <int HD>
struct AttnTc {
    static constexpr uint32_t PLANE = HD / 64 * TC_BLOCK;                       // a tile of 128 rows
    static constexpr uint32_t Q = 0, K = 2 * PLANE, V = K + 2 * PLANE, END = V + 2 * PLANE;      // two planes of Q, two stages of K and V
    static constexpr uint32_t MERGE = 2 * TC_ROWS * (HD + 4) * 4;
    static constexpr uint32_t SMEM = (END > MERGE ? END : MERGE) + 1024;        // + alignment
};

// Value d of row r in a tile
__device__ __forceinline__ uint32_t tc_at(int r, int d) { return (uint32_t)(d >> 6) * TC_BLOCK + r * 128 + ((((d >> 3) & 7) ^ (r & 7)) << 4) + (d & 7) * 2; }

// Matrix descriptors with the 128-byte swizzle (2 at bit 61) and this architecture's version (1 at bit 46); addresses and
// distances in 16-byte units.  Rows along M or N, values along K (Q, K): groups of 8 rows are 1024 bytes apart, the 16 values of an
// instruction 32 bytes of a row.  The other way round (V as the second operand: N along a row, positions are K): groups of 8
// positions 1024 bytes apart, blocks of 64 columns TC_BLOCK, the 16 positions of an instruction 2048 bytes.
__device__ __forceinline__ uint64_t tc_desc(uint32_t addr, uint32_t leading, uint32_t stride) {
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | (uint64_t)(leading >> 4) << 16 | (uint64_t)(stride >> 4) << 32 | 1ull << 46 | 2ull << 61;
}
// kind::f16: D = f32 (1 at bit 4), A = B = f16, second operand with N along its rows (bit 16), N / 8 at bit 17, M / 16 at bit 24
template <int N, bool N_ROWS> constexpr uint32_t ATC_IDESC = (1u << 4) | (N_ROWS ? 1u << 16 : 0u) | ((uint32_t)(N >> 3) << 17) | ((128u >> 4) << 24);

__device__ __forceinline__ void atc_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" :: "r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void atc_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" :: "r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void atc_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" :: "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void atc_arrive(uint64_t* bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" :: "r"(smem_u32(bar)) : "memory"); }
__device__ __forceinline__ bool atc_try(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
    return ok != 0;
}
__device__ __forceinline__ void atc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void atc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void atc_proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// 16 consecutive columns of this thread's lane, valid after atc_ld_wait (through which the values pass, so that nothing is
// computed from them ahead of it); 8 to them
__device__ __forceinline__ void atc_ld16(uint32_t t, float (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]), "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15])
                 : "r"(t) : "memory");
}
__device__ __forceinline__ void atc_ld_wait(float (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+f"(r[0]), "+f"(r[1]), "+f"(r[2]), "+f"(r[3]), "+f"(r[4]), "+f"(r[5]), "+f"(r[6]), "+f"(r[7]), "+f"(r[8]), "+f"(r[9]), "+f"(r[10]), "+f"(r[11]), "+f"(r[12]), "+f"(r[13]), "+f"(r[14]), "+f"(r[15])
                 :: "memory");
}
__device__ __forceinline__ void atc_st8(uint32_t t, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
                 :: "r"(t), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
}
__device__ __forceinline__ void atc_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ float atc_exp2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }

// Columns of tensor memory: S / P of the even chunks, of the odd ones, then O' of each
constexpr uint32_t COL_S = 0, COL_O = 256;

template <int HD, bool TMA, bool CAP>
__global__ void __launch_bounds__(TC_THREADS, 1) k_attn_tc(const __grid_constant__ AttnArgs a, const __grid_constant__ CUtensorMap map, uint32_t run) {
    using F = AttnTc<HD>;
    extern __shared__ uint8_t raw[];
    __shared__ AttnRow s_row[TC_ROWS];
    __shared__ float s_unit[TC_ROWS];
    __shared__ uint32_t s_tmem, s_dead;
    __shared__ Found s_found;
    __shared__ int64_t s_where[2][TMA ? 1 : TC_CB];
    __shared__ End<TC_ROWS, 2> s_end;
    // chunk c, stage c & 1: its keys are there / its scores are (and its keys read); its values / its weights / its output (and its values read)
    __shared__ __align__(8) uint64_t b_k[2], b_s[2], b_v[2], b_p[2], b_o[2];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t kvh = blockIdx.y, split = blockIdx.x % a.splits, t = gridDim.x / a.splits - 1 - blockIdx.x / a.splits;   // late rows see more: first
    AttnTile x;
    if (!find_tile<TC_ROWS, TC_CB>(a, t, kvh, x, s_row, s_found)) return;
    uint32_t sharers, c0, c1;
    if (!share_out(a, x, split, sharers, c0, c1)) return;
    const int n = (int)(c1 - c0);
    uint8_t* const sm = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
    const uint32_t sm_s = smem_u32(sm);
    if (tid == 0) {
        for (int i = 0; i < 2; ++i) { mbar_init(&b_k[i], TMA ? 1 : TC_LOADERS); mbar_init(&b_s[i], 1); mbar_init(&b_v[i], TMA ? 1 : TC_LOADERS); mbar_init(&b_p[i], 128); mbar_init(&b_o[i], 1); }
        s_dead = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 11) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(smem_u32(&s_tmem)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // queries: two fp16 terms of the row times a power of two (with the sign of the scale), four rows of a warp under way at once
    constexpr int W = TC_THREADS / 32, VPL = HD / 32, R4 = 4;
#pragma unroll 1
    for (int r1 = warp; r1 < TC_ROWS; r1 += R4 * W) {
        float v[R4][VPL];
#pragma unroll
        for (int j = 0; j < R4; ++j) {
            const int r = r1 + j * W;
            const bool on = r < TC_ROWS && s_row[r].pos >= 0;
            const float* src = a.act + (on ? s_row[r].q : 0);
#pragma unroll
            for (int i = 0; i < VPL; ++i) v[j][i] = on ? src[lane + 32 * i] : 0.f;
        }
#pragma unroll
        for (int j = 0; j < R4; ++j) {
            const int r = r1 + j * W;
            if (r >= TC_ROWS) break;
            float most = 0.f, up, down;
#pragma unroll
            for (int i = 0; i < VPL; ++i) most = fmaxf(most, fabsf(v[j][i]));
            row_scale(__uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(most))), up, down);
            if (lane == 0) s_unit[r] = down;
            if (a.scale < 0.f) up = -up;
#pragma unroll
            for (int i = 0; i < VPL; ++i) {
                const float y = v[j][i] * up;
                const __half hi = __float2half_rn(y);
                uint8_t* p = sm + F::Q + tc_at(r, lane + 32 * i);
                *reinterpret_cast<__half*>(p) = hi;
                *reinterpret_cast<__half*>(p + F::PLANE) = __float2half_rn(y - __half2float(hi));
            }
        }
    }
    atc_proxy_fence();
    atc_fence_before();
    __syncthreads();
    atc_fence_after();
    const uint32_t tmem = s_tmem;
    bool dead = false;
    auto wait = [&](uint64_t* bar, uint32_t parity) {        // bounded: what comes later then does not wait any more
        if (!dead && !mbar_wait(bar, parity)) { dead = true; s_dead = 1; atomicOr(a.err, DEVERR_WAIT); }
    };

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        if (TMA && warp == 8) {
            // ---- keys and values, a run of positions of one page to a copy; the swizzle is the copy's ----
            const uint32_t runs = TC_CB / run;
            const int32_t outside = (int32_t)(a.pool_rows);      // no row of the pool: a copy from there brings zeros
            auto locate = [&](int c) -> int32_t {
                if (c >= n || (uint32_t)lane >= runs) return outside;
                const int32_t p = chunk_at<TC_CB>(x, c0 + c) + lane * (int32_t)run;
                if (p > x.hi || (p + (int32_t)run <= x.from && (uint32_t)p >= a.n_sink)) return outside;
                const int32_t page = x.pages[(uint32_t)p / a.geo.page];
                return page < 0 ? outside : (int32_t)(kv_index(a.geo, (uint32_t)page, a.layer, 0, kvh, (uint32_t)p % a.geo.page) / HD);
            };
            const int32_t v_row = (int32_t)(a.geo.n_kv * a.geo.page);
            int32_t row = locate(0);
            auto fetch = [&](int c, int32_t y, uint32_t base, uint64_t* free, uint64_t* full) {
                if (c >= 2) wait(free, (uint32_t)((c >> 1) - 1) & 1u);
                if (lane == 0) mbar_expect_tx(full, F::PLANE);
                __syncwarp();
                if ((uint32_t)lane < runs)
#pragma unroll
                    for (int d0 = 0; d0 < HD; d0 += 64)
                        asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                                     :: "r"(sm_s + base + (uint32_t)(c & 1) * F::PLANE + (d0 >> 6) * TC_BLOCK + lane * run * 128), "l"(&map), "r"(d0), "r"(y), "r"(smem_u32(full)) : "memory");
            };
            for (int c = 0; c < n; ++c) {
                const int32_t next = locate(c + 1);
                fetch(c, row, F::K, &b_s[c & 1], &b_k[c & 1]);
                fetch(c, row == outside ? outside : row + v_row, F::V, &b_o[c & 1], &b_v[c & 1]);
                row = next;
            }
            // nothing is under way when the CTA ends, also where a wait ran out
            for (int c = max(n - 2, 0); c < n; ++c) { mbar_wait(&b_k[c & 1], (uint32_t)(c >> 1) & 1u); mbar_wait(&b_v[c & 1], (uint32_t)(c >> 1) & 1u); }
        } else if (!TMA && warp < 11) {
            // ---- keys and values, 16 bytes at a time ----
            const int me = tid - 256;
            const __half* const pool = reinterpret_cast<const __half*>(a.pool);
            const size_t v_off = (size_t)a.geo.n_kv * a.geo.page * HD;
            constexpr int WPR = HD / 8;                      // 16-byte words of a row
            uint64_t* owed = nullptr;                        // whose copies are under way and not yet announced
            auto announce = [&]() { atc_proxy_fence(); atc_arrive(owed); owed = nullptr; };
            auto fetch = [&](int c, uint32_t base, size_t off, uint64_t* free, uint64_t* full) {
                if (c >= 2 && !atc_try(free, (uint32_t)((c >> 1) - 1) & 1u)) {
                    if (owed) { at_wait<0>(); announce(); }
                    wait(free, (uint32_t)((c >> 1) - 1) & 1u);
                }
#pragma unroll 4
                for (int w = me; w < TC_CB * WPR; w += TC_LOADERS) {
                    const int r = w / WPR, ch = w % WPR;
                    const int64_t at = s_where[c & 1][r];
                    at_cp16(sm_s + base + (uint32_t)(c & 1) * F::PLANE + tc_at(r, ch * 8), pool + (at < 0 ? 0 : (size_t)at + off) + ch * 8, at >= 0);
                }
                at_commit();
                if (owed) { at_wait<1>(); announce(); }
                owed = full;
            };
            for (int c = 0; c < n; ++c) {
                const int32_t p0 = chunk_at<TC_CB>(x, c0 + c);
                for (int r = me; r < TC_CB; r += TC_LOADERS) s_where[c & 1][r] = tile_position(a, x, kvh, p0 + r);
                asm volatile("bar.sync 1, %0;" :: "n"(TC_LOADERS) : "memory");
                fetch(c, F::K, 0, &b_s[c & 1], &b_k[c & 1]);
                fetch(c, F::V, v_off, &b_o[c & 1], &b_v[c & 1]);
            }
            at_wait<0>();
            if (owed) announce();
        } else if (warp == 11 && lane == 0) {
            // ---- products: S of chunk c + 1 goes ahead of O' of chunk c ----
            auto scores = [&](int c) {
                const int b = c & 1;
                wait(&b_k[b], (uint32_t)(c >> 1) & 1u);
                atc_fence_after();
                if (dead) return;
#pragma unroll
                for (int pass = 0; pass < 2; ++pass)         // the low terms first: they are added while the sum is small
#pragma unroll
                    for (int k = 0; k < HD / 16; ++k) {
                        const uint32_t off = (uint32_t)(k >> 2) * TC_BLOCK + (k & 3) * 32;
                        atc_mma_ss(tmem + COL_S + b * 128, tc_desc(sm_s + F::Q + (1 - pass) * F::PLANE + off, 16, 1024),
                                   tc_desc(sm_s + F::K + b * F::PLANE + off, 16, 1024), ATC_IDESC<128, false>, pass + k > 0);
                    }
                atc_commit(&b_s[b]);
            };
            auto output = [&](int c) {
                const int b = c & 1;
                wait(&b_v[b], (uint32_t)(c >> 1) & 1u);
                wait(&b_p[b], (uint32_t)(c >> 1) & 1u);
                atc_fence_after();
                if (dead) return;
#pragma unroll
                for (int pass = 0; pass < 2; ++pass)
#pragma unroll
                    for (int k = 0; k < TC_CB / 16; ++k)
                        atc_mma_ts(tmem + COL_O + b * HD, tmem + COL_S + b * 128 + k * 16 + (1 - pass) * 8,
                                   tc_desc(sm_s + F::V + b * F::PLANE + k * 2048, TC_BLOCK, 1024), ATC_IDESC<HD, true>, pass + k > 0);
                atc_commit(&b_o[b]);
            };
            scores(0);
            for (int c = 0; c < n; ++c) {
                if (c + 1 < n) scores(c + 1);
                output(c);
            }
        }
        __syncwarp();
        __syncthreads();
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
        // ---- weights and sums: a row to a thread, every other chunk ----
        const int w = warp >> 2, r = tid & 127;
        const uint32_t col = tmem + ((uint32_t)(warp & 3) << 21), s_col = col + COL_S + w * 128, o_col = col + COL_O + w * HD;
        const int32_t pos = s_row[r].pos;
        // scores to powers of two: times k2, or cap2 tanh of them times k2
        const float unit = s_unit[r] * fabsf(a.scale), k2 = CAP ? unit * __frcp_rn(a.cap) : unit * 1.4426950408889634f, cap2 = a.cap * 1.4426950408889634f;
        float o[HD], m = -INFINITY, l = 0.f, alpha = 0.f;
#pragma unroll
        for (int d = 0; d < HD; ++d) o[d] = 0.f;
        auto collect = [&](int c, float factor) {            // O' of chunk c to the outputs before it, times `factor`
            wait(&b_o[w], (uint32_t)(c >> 1) & 1u);
            atc_fence_after();
            float v[2][16];
            atc_ld16(o_col, v[0]);
#pragma unroll
            for (int d0 = 0; d0 < HD; d0 += 16) {
                float (&u)[16] = v[d0 / 16 & 1];
                atc_ld_wait(u);
                if (d0 + 16 < HD) atc_ld16(o_col + d0 + 16, v[(d0 / 16 + 1) & 1]);
#pragma unroll
                for (int d = 0; d < 16; ++d) o[d0 + d] = fmaf(o[d0 + d], factor, u[d]);
            }
        };
        for (int c = w; c < n; c += 2) {
            const int32_t p0 = chunk_at<TC_CB>(x, c0 + c);
            const bool all = tile_sees(a, x, p0, TC_CB);
            // position p0 + j is seen for j <= j1 and (j > j0 or j < js)
            const int32_t j1 = pos - p0, j0 = a.window ? j1 - (int32_t)a.window : -1, js = (int32_t)min(a.n_sink, 0x40000000u) - p0;
            auto seen = [&](int j) { return j <= j1 && (j > j0 || j < js); };
            wait(&b_s[w], (uint32_t)(c >> 1) & 1u);
            atc_fence_after();
            // Two turns over the scores, 16 columns at a time with the next ones under way: the maximum, the weights.  Loops of two
            // steps, one for chunks that every row sees whole, one for the others: unrolled with every choice inside, the turns took
            // 5500 cycles, most of them fetching instructions.
            constexpr int STEP = 16;
            float v[2][STEP], mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY}, sum[4] = {0.f, 0.f, 0.f, 0.f};
            atc_ld16(s_col, v[0]);
            auto maximum = [&](auto whole) {
#pragma unroll 1
                for (int i = 0; i < TC_CB; i += 2 * STEP)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        atc_ld_wait(v[h]);
                        atc_ld16(s_col + (i + (h + 1) * STEP) % TC_CB, v[1 - h]);
#pragma unroll
                        for (int d = 0; d < STEP; ++d) mx[d & 3] = fmaxf(mx[d & 3], decltype(whole)::value || seen(i + h * STEP + d) ? v[h][d] : -INFINITY);
                    }
            };
            if (all) maximum(std::true_type{});
            else maximum(std::false_type{});
            float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
            top = CAP ? cap2 * at_tanh(top * k2) : top * k2;
            const float mn = fmaxf(m, top), ref = mn == -INFINITY ? 0.f : mn, shift = 8.f - ref;      // times 256: the low terms stay clear of the subnormals
            const float before = alpha;
            alpha = atc_exp2(m - ref);
            m = mn;
            auto turn = [&](auto whole) {
#pragma unroll 1
                for (int i = 0; i < TC_CB; i += 2 * STEP)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float (&u)[STEP] = v[h];
                        atc_ld_wait(u);
                        if (i + h * STEP + STEP < TC_CB) atc_ld16(s_col + i + (h + 1) * STEP, v[1 - h]);
                        uint32_t hi[STEP / 2], lo[STEP / 2];
#pragma unroll
                        for (int d = 0; d < STEP; ++d) {
                            u[d] = atc_exp2(CAP ? fmaf(at_tanh(u[d] * k2), cap2, shift) : fmaf(u[d], k2, shift));
                            if (!decltype(whole)::value && !seen(i + h * STEP + d)) u[d] = 0.f;
                        }
#pragma unroll
                        for (int d = 0; d < STEP / 2; ++d) { sum[d & 3] += u[2 * d] + u[2 * d + 1]; at_split_h(u[2 * d], u[2 * d + 1], hi[d], lo[d]); }
                        atc_st8(s_col + i + h * STEP, hi);
                        atc_st8(s_col + i + h * STEP + 8, lo);
                    }
            };
            if (all) turn(std::true_type{});
            else turn(std::false_type{});
            l = fmaf(l, alpha, (sum[0] + sum[1]) + (sum[2] + sum[3]));
            if (c >= 2) collect(c - 2, before);              // its products ran meanwhile; O' is free for this chunk's
            atc_st_wait();
            atc_fence_before();
            atc_arrive(&b_p[w]);
        }
        if (n > w) collect((n - 1 - w) / 2 * 2 + w, alpha);
        s_end.m[w][r] = m; s_end.l[w][r] = l * (1.f / 256.f);
        atc_fence_before();
        __syncthreads();                                     // all products are done, shared memory is free
        const float f = s_end.factor<true>(w, r) * (1.f / 256.f);
        float* to = reinterpret_cast<float*>(sm) + (w * TC_ROWS + r) * (HD + 4);
#pragma unroll
        for (int d = 0; d < HD; d += 4) *reinterpret_cast<float4*>(to + d) = make_float4(o[d] * f, o[d + 1] * f, o[d + 2] * f, o[d + 3] * f);
    }
    atc_fence_after();
    __syncthreads();
    if (warp == 11) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(tmem), "r"(512u) : "memory");
    if (s_dead) return;
    settle<__half, HD, TC_ROWS, 2, TC_THREADS, true, false>(a, x, s_row, t, kvh, split, sharers, reinterpret_cast<float*>(sm), s_end);
}

template <int HD, bool TMA, bool CAP>
static int launch_tc(const AttnArgs& a, const KvCache& kv, uint32_t tiles) {
    static bool set = false;
    if (!set) {
        if (cudaFuncSetAttribute((const void*)k_attn_tc<HD, TMA, CAP>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)AttnTc<HD>::SMEM) != cudaSuccess)
            return fail(ADAMAH_ERR_BACKEND, "attn_kv: cannot raise the shared-memory limit");
        set = true;
    }
    k_attn_tc<HD, TMA, CAP><<<dim3(tiles * a.splits, a.geo.n_kv), TC_THREADS, AttnTc<HD>::SMEM, g.stream>>>(a, kv.map, kv.run);
    count_launch();
    return check_launch("map_attn_kv");
}
template <int HD, bool TMA>
static int launch_cap(const AttnArgs& a, const KvCache& kv, uint32_t tiles) {
    return a.cap > 0.f ? launch_tc<HD, TMA, true>(a, kv, tiles) : launch_tc<HD, TMA, false>(a, kv, tiles);
}
int launch_attn_tc(const AttnArgs& a, const KvCache& kv, uint32_t tiles) {
    if (kv.run) return a.geo.hd == 64 ? launch_cap<64, true>(a, kv, tiles) : launch_cap<128, true>(a, kv, tiles);
    return a.geo.hd == 64 ? launch_cap<64, false>(a, kv, tiles) : launch_cap<128, false>(a, kv, tiles);
}

}  // namespace ab
