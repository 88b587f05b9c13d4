// Attention of many rows over a paged fp16 cache on the 5th-generation tensor cores (see attn_kv.cu for the operator and the
// precision of its operands).
//
// A CTA has 128 rows (a token's query heads of one key head are neighbours) and walks the positions in chunks of 128:
//   S = (Q_hi + Q_lo) K^T    tcgen05.mma, both operands in shared memory, into 128 columns of tensor memory
//   P = 2^(k S - m + 8)      a row to a thread: S read twice (maximum, weights), P as two fp16 terms over S, column for column
//   O' = (P_hi + P_lo) V     tcgen05.mma, P from tensor memory, V from shared memory as it lies there (its positions are the rows)
//   O = O alpha + O' beta    in registers: a sum that stays in the tensor core for many chunks would lose bits (attn_kv.cu)
// Two warpgroups make the weights of the even and the odd chunks, each relative to its own running maximum; two more have a half
// of the outputs each and add up what comes relative to either.  Three S / P take turns, so that the scores of the next chunks
// are there when a warpgroup is done with its weights (with an S / P of its own, whose scores have to wait for the output of the
// weights before them, a warpgroup stood still for 2900 of 6700 cycles).  One warp fetches keys and another values, by tensor
// copies, or 16 bytes at a time where pages do not come in groups of eight; one thread issues each product.
//
// The roles execute different code at once, and what all of them need for a chunk has to stay in an instruction cache that a few
// SMs refill together: with loops unrolled freely it took 2600 cycles a chunk on some SMs and 4000 on others, with short ones (and
// two values to an instruction) 2900 everywhere.  The products need 2048 of those at the tensor core's rate, shared memory 2000 for
// what it hands to them and takes in, and an output waits for the one before it to be taken.  2048 tokens behind 14000, 32
// heads over 16 of 128: 925 us, two products where fp16 operands would have one, so 1.1 PFLOP/s of them.
#include "attn_kv.cuh"
#include "gemv_mma.cuh"

#include <type_traits>

namespace ab {

constexpr int TC_ROWS = 128, TC_CB = 128, TC_THREADS = 640, TC_LOADERS = 64;
constexpr int TC_OUT = 8, TC_FETCH = 16, TC_ISSUE = 18;       // first warp of the outputs; the two that fetch; the two that issue
constexpr uint32_t TC_BLOCK = 128 * 128;             // 128 rows (or positions) of 64 values: 128 bytes each, in the 128-byte swizzle

template <int HD>
struct AttnTc {
    static constexpr uint32_t PLANE = HD / 64 * TC_BLOCK;                       // a tile of 128 rows
    static constexpr uint32_t Q = 0, K = 2 * PLANE, V = K + 2 * PLANE, END = V + 2 * PLANE;      // two planes of Q, two stages of K and V
    static constexpr uint32_t MERGE = TC_ROWS * (HD + 4) * 4;
    static constexpr uint32_t SMEM = (END > MERGE ? END : MERGE) + 1024;        // + alignment
};

// Value d of row r in a tile
__device__ __forceinline__ uint32_t tc_at(int r, int d) { return (uint32_t)(d >> 6) * TC_BLOCK + r * 128 + ((((d >> 3) & 7) ^ (r & 7)) << 4) + (d & 7) * 2; }

// Matrix descriptors with the 128-byte swizzle (2 at bit 61) and this architecture's version (1 at bit 46); addresses and
// distances in 16-byte units.  Rows along M or N, values along K (Q, K): groups of 8 rows are 1024 bytes apart, the 16 values of an
// instruction 32 bytes of a row.  The other way round (V as the second operand: N along a row, positions are K): groups of 8
// positions 1024 bytes apart, blocks of 64 columns TC_BLOCK, the 16 positions of an instruction 2048 bytes.
// The words of a descriptor: everything but the address is known ahead, and the thread that issues products must not do more
// than an addition for each (built anew for every product, descriptors took it 2000 cycles a chunk).
__device__ __forceinline__ uint32_t tc_desc_lo(uint32_t addr, uint32_t leading) { return (addr & 0x3FFFFu) >> 4 | (leading >> 4) << 16; }
__device__ __forceinline__ uint64_t tc_desc(uint32_t lo) { return (uint64_t)((1024u >> 4) | 1u << 14 | 2u << 29) << 32 | lo; }
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
// 16 or 8 consecutive columns of this thread's lane, valid after atc_ld_wait (through which the values pass, so that nothing is
// computed from them ahead of it); 4 to them
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
__device__ __forceinline__ void atc_ld8(uint32_t t, float (&r)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]) : "r"(t) : "memory");
}
__device__ __forceinline__ void atc_ld_wait(float (&r)[8]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+f"(r[0]), "+f"(r[1]), "+f"(r[2]), "+f"(r[3]), "+f"(r[4]), "+f"(r[5]), "+f"(r[6]), "+f"(r[7]) :: "memory");
}
__device__ __forceinline__ void atc_st4(uint32_t t, const uint32_t (&r)[4]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1,%2,%3,%4};" :: "r"(t), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]) : "memory");
}
__device__ __forceinline__ void atc_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// what three roles execute for every chunk has to come out of a small instruction cache: two values an instruction, three to a maximum
__device__ __forceinline__ float atc_max3(float a, float b, float c) { float r; asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c)); return r; }

// Columns of tensor memory: three S / P of 128, O'
constexpr uint32_t COL_S = 0, COL_O = 384;

template <int HD, bool TMA, bool CAP>
__global__ void __launch_bounds__(TC_THREADS, 1) k_attn_tc(const __grid_constant__ AttnArgs a, const __grid_constant__ CUtensorMap map, uint32_t run) {
    using F = AttnTc<HD>;
    constexpr int LOADERS = TMA ? 1 : TC_LOADERS;        // arrivals of fetched keys or values
    extern __shared__ uint8_t raw[];
    __shared__ AttnRow s_row[TC_ROWS];
    __shared__ float s_unit[TC_ROWS];
    __shared__ uint32_t s_tmem, s_dead;
    __shared__ Found s_found;
    __shared__ int64_t s_where[4][TMA ? 1 : TC_CB];
    __shared__ End<TC_ROWS, 1> s_end;
    __shared__ float s_ref[4][TC_ROWS], s_m[2][TC_ROWS], s_l[2][TC_ROWS];     // what a chunk's weights are relative to; maxima and sums of the two
    // Of chunk c, stage c & 1: its keys are there, are read; its values are there and the output before it is taken, its values are
    // read.  Slot c % 3: its scores are there; its weights are, are read.  c & 3: s_ref is there (its next user is four chunks on, when
    // the output of the next one is asked for).  Its output is there.  Values have come that are not all of them seen.
    __shared__ __align__(8) uint64_t b_k[2], b_kr[2], b_v[2], b_vr[2], b_s[3], b_p[3], b_pr[3], b_ref[4], b_o, b_end;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const AttnShare part = share_of(a);
    const uint32_t kvh = part.kvh;
    AttnTile x;
    if (!find_tile<TC_ROWS, TC_CB>(a, part.tile, kvh, x, s_row, s_found)) return;
    uint32_t sharers, c0, c1;
    if (!share_out(a, x, part, sharers, c0, c1)) return;
    const int n = (int)(c1 - c0);
    uint8_t* const sm = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
    const uint32_t sm_s = smem_u32(sm);
    if (tid == 0) {
        for (int i = 0; i < 2; ++i) { mbar_init(&b_k[i], LOADERS); mbar_init(&b_kr[i], 1); mbar_init(&b_v[i], LOADERS + 256); mbar_init(&b_vr[i], 1); }
        for (int i = 0; i < 3; ++i) { mbar_init(&b_s[i], 1); mbar_init(&b_p[i], 128); mbar_init(&b_pr[i], 1); }
        mbar_init(&b_o, 1); mbar_init(&b_end, 1);
        for (int i = 0; i < 4; ++i) mbar_init(&b_ref[i], 128);
        s_dead = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == TC_ISSUE) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(smem_u32(&s_tmem)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    atc_fence_before();
    __syncthreads();
    atc_fence_after();
    const uint32_t tmem = s_tmem;
    // queries, by all but the warps that fetch (they begin) and issue: two fp16 terms of the row times a power of two (with the
    // sign of the scale), a warp's rows all under way at once
    constexpr int W = TC_FETCH, VPL = HD / 32, R = TC_ROWS / W;
    if (warp < TC_FETCH) {
        float v[R][VPL];
#pragma unroll
        for (int j = 0; j < R; ++j) {
            const AttnRow& row = s_row[warp + j * W];
            const float* src = a.act + row.q + lane * VPL;
#pragma unroll
            for (int i = 0; i < VPL; ++i) v[j][i] = 0.f;
            if (row.pos < 0) continue;
            if (row.q % VPL) {
#pragma unroll
                for (int i = 0; i < VPL; ++i) v[j][i] = src[i];
            } else if constexpr (VPL == 4) {
                const float4 y = *reinterpret_cast<const float4*>(src);
                v[j][0] = y.x; v[j][1] = y.y; v[j][2] = y.z; v[j][3] = y.w;
            } else {
                const float2 y = *reinterpret_cast<const float2*>(src);
                v[j][0] = y.x; v[j][1] = y.y;
            }
        }
#pragma unroll
        for (int j = 0; j < R; ++j) {
            const int r = warp + j * W;
            float most = 0.f, up, down;
#pragma unroll
            for (int i = 0; i < VPL; ++i) most = fmaxf(most, fabsf(v[j][i]));
            row_scale(__uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(most))), up, down);
            if (lane == 0) s_unit[r] = down;
            if (a.scale < 0.f) up = -up;
            uint32_t hi[VPL / 2], lo[VPL / 2];
#pragma unroll
            for (int i = 0; i < VPL; i += 2) at_split_h(v[j][i] * up, v[j][i + 1] * up, hi[i / 2], lo[i / 2]);
            uint8_t* p = sm + F::Q + tc_at(r, lane * VPL);
            if constexpr (VPL == 4) {
                *reinterpret_cast<uint2*>(p) = make_uint2(hi[0], hi[1]);
                *reinterpret_cast<uint2*>(p + F::PLANE) = make_uint2(lo[0], lo[1]);
            } else {
                *reinterpret_cast<uint32_t*>(p) = hi[0];
                *reinterpret_cast<uint32_t*>(p + F::PLANE) = lo[0];
            }
        }
    }
    if (warp >= TC_FETCH) asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    else atc_proxy_fence();
    if (warp < TC_FETCH || warp >= TC_ISSUE) asm volatile("bar.sync 2, %0;" :: "n"(TC_THREADS - TC_LOADERS) : "memory");
    bool dead = false;
    auto wait1 = [&](uint64_t* bar, uint32_t parity) {       // bounded: what comes later then does not wait any more
        if (dead) return;
#pragma unroll 1
        for (int spin = 0; !atc_try(bar, parity); ++spin)
            if (spin == 1 << 20) { dead = true; s_dead = 1; atomicOr(a.err, DEVERR_WAIT); return; }
    };
    auto wait = [&](uint64_t* bar, uint32_t parity) {        // a warp (one lane that asks for the others takes 2900 cycles a chunk to 3160)
        wait1(bar, parity);
        __syncwarp();
    };

    if (warp >= TC_FETCH) {
        if (TMA && warp < TC_ISSUE) {
            // ---- keys (one warp) and values (another: neither waits for the other's stage), a run of positions of one page to a copy;
            // the swizzle is the copy's ----
            const bool keys = warp == TC_FETCH;
            const uint32_t runs = TC_CB / run;
            const int32_t outside = (int32_t)(a.pool_rows);      // no row of the pool: a copy from there brings zeros
            auto locate = [&](int c) -> int32_t {
                if (c >= n || (uint32_t)lane >= runs) return outside;
                const int32_t p = chunk_at<TC_CB>(x, c0 + c) + lane * (int32_t)run;
                if (p > x.hi || (p + (int32_t)run <= x.from && (uint32_t)p >= a.n_sink)) return outside;
                const int32_t page = x.pages[(uint32_t)p / a.geo.page];
                return page < 0 ? outside : (int32_t)(kv_index(a.geo, (uint32_t)page, a.layer, keys ? 0 : 1, kvh, (uint32_t)p % a.geo.page) / HD);
            };
            const uint32_t to = sm_s + (keys ? F::K : F::V) + lane * run * 128;
            uint64_t *const full = keys ? b_k : b_v, *const free = keys ? b_kr : b_vr;
            // A copy brings a run whole where the tile sees any of it.  Values that no row sees become zeros before they are announced: 0
            // times what another sequence has left there could be a NaN, and a row with a NaN is done again by one warp.
            uint32_t ends = 0;                               // chunks with such values
            int32_t y = locate(0);
            for (int c = 0; c < n; ++c) {
                const int32_t next = locate(c + 1);
                const int32_t p0 = chunk_at<TC_CB>(x, c0 + c);
                const bool is_end = !keys && (p0 + TC_CB > x.hi + 1 || (p0 < x.from && (uint32_t)p0 + TC_CB > a.n_sink));
                uint64_t* const bar = is_end ? &b_end : full + (c & 1);
                if (c >= 2) wait(free + (c & 1), (uint32_t)((c >> 1) - 1) & 1u);
                if (lane == 0) mbar_expect_tx(bar, F::PLANE);
                __syncwarp();
                if ((uint32_t)lane < runs)
#pragma unroll
                    for (int d0 = 0; d0 < HD; d0 += 64)
                        asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                                     :: "r"(to + (uint32_t)(c & 1) * F::PLANE + (d0 >> 6) * TC_BLOCK), "l"(&map), "r"(d0), "r"(y), "r"(smem_u32(bar)) : "memory");
                if (is_end) {
                    wait(bar, ends++ & 1u);
#pragma unroll 1
                    for (int i = lane; i < TC_CB * 8; i += 32) {         // 16 bytes, wherever in its row the swizzle has them
                        const int32_t p = p0 + i / 8;
                        if (p <= x.hi && (p >= x.from || (uint32_t)p < a.n_sink)) continue;
#pragma unroll
                        for (int d = 0; d < HD / 64; ++d) *reinterpret_cast<uint4*>(sm + F::V + (c & 1) * F::PLANE + d * TC_BLOCK + i * 16) = make_uint4(0u, 0u, 0u, 0u);
                    }
                    atc_proxy_fence();
                    __syncwarp();
                    if (lane == 0) atc_arrive(full + (c & 1));
                }
                y = next;
            }
            // nothing is under way when the CTA ends, also where a wait ran out
            if (ends) mbar_wait(&b_end, (ends - 1) & 1u);
            for (int c = max(n - 2, 0); c < n; ++c) mbar_wait(full + (c & 1), (uint32_t)(c >> 1) & 1u);
        } else if (!TMA && warp < TC_ISSUE) {
            // ---- keys and values, 16 bytes at a time ----
            const int me = (warp - TC_FETCH) * 32 + lane;
            const __half* const pool = reinterpret_cast<const __half*>(a.pool);
            const size_t v_off = (size_t)a.geo.n_kv * a.geo.page * HD;
            constexpr int WPR = HD / 8;                      // 16-byte words of a row
            uint64_t* owed = nullptr;                        // whose copies are under way and not yet announced
            auto announce = [&]() { atc_proxy_fence(); atc_arrive(owed); owed = nullptr; };
            auto fetch = [&](int c, uint32_t base, size_t off, uint64_t* free, uint64_t* full) {
                if (c >= 2 && !__all_sync(0xffffffffu, atc_try(free, (uint32_t)((c >> 1) - 1) & 1u))) {
                    if (owed) { at_wait<0>(); announce(); }
                    wait(free, (uint32_t)((c >> 1) - 1) & 1u);
                }
#pragma unroll 4
                for (int w = me; w < TC_CB * WPR; w += TC_LOADERS) {
                    const int r = w / WPR, ch = w % WPR;
                    const int64_t at = s_where[c & 3][r];
                    at_cp16(sm_s + base + (uint32_t)(c & 1) * F::PLANE + tc_at(r, ch * 8), pool + (at < 0 ? 0 : (size_t)at + off) + ch * 8, at >= 0);
                }
                at_commit();
                if (owed) { at_wait<1>(); announce(); }
                owed = full;
            };
            auto locate = [&](int c) {                       // (behind the barrier before it everybody is done with chunk c - 4)
                if (c >= n) return;
                const int32_t p0 = chunk_at<TC_CB>(x, c0 + c);
                for (int r = me; r < TC_CB; r += TC_LOADERS) s_where[c & 3][r] = tile_position(a, x, kvh, p0 + r);
            };
            // in the order of their use: keys a chunk ahead of values
            for (int c = 0; c < n + 1; ++c) {
                locate(c);
                asm volatile("bar.sync 1, %0;" :: "n"(TC_LOADERS) : "memory");
                if (c < n) fetch(c, F::K, 0, &b_kr[c & 1], &b_k[c & 1]);
                if (c >= 1) fetch(c - 1, F::V, v_off, &b_vr[(c - 1) & 1], &b_v[(c - 1) & 1]);
            }
            at_wait<0>();
            if (owed) announce();
        } else if (warp == TC_ISSUE && lane == 0) {
            // ---- scores.  A thread that issues is held up until all but a few of its products are done, and a wait beside busy shared
            // memory takes 350 cycles: with one thread for both kinds the tensor core stood still for 1500 of 4200 cycles a chunk ----
            const uint32_t q_hi = tc_desc_lo(sm_s + F::Q, 16), q_lo = tc_desc_lo(sm_s + F::Q + F::PLANE, 16), k_0 = tc_desc_lo(sm_s + F::K, 16);
            for (int c = 0; c < n && !dead; ++c) {
                wait1(&b_k[c & 1], (uint32_t)(c >> 1) & 1u);
                if (c >= 3) wait1(&b_pr[c % 3], (uint32_t)(c / 3 - 1) & 1u);         // the weights that lie there are read
                atc_fence_after();
                if (dead) break;
                const uint32_t d = tmem + COL_S + c % 3 * 128, kd = k_0 + (c & 1) * (F::PLANE >> 4);
#pragma unroll 1
                for (int pass = 0; pass < 2; ++pass)         // the low terms first: they are added while the sum is small
#pragma unroll
                    for (int k = 0; k < HD / 16; ++k) {
                        const uint32_t off = ((k >> 2) * TC_BLOCK + (k & 3) * 32) >> 4;
                        atc_mma_ss(d, tc_desc((pass ? q_hi : q_lo) + off), tc_desc(kd + off), ATC_IDESC<128, false>, pass + k > 0);
                    }
                atc_commit(&b_s[c % 3]);
                atc_commit(&b_kr[c & 1]);
            }
        } else if (warp == TC_ISSUE + 1 && lane == 0) {
            // ---- outputs ----
            const uint32_t v_0 = tc_desc_lo(sm_s + F::V, TC_BLOCK);
            for (int c = 0; c < n; ++c) {
                wait1(&b_v[c & 1], (uint32_t)(c >> 1) & 1u);
                wait1(&b_p[c % 3], (uint32_t)(c / 3) & 1u);
                atc_fence_after();
                if (dead) break;
                const uint32_t d = tmem + COL_O, pd = tmem + COL_S + c % 3 * 128, vd = v_0 + (c & 1) * (F::PLANE >> 4);
#pragma unroll 1
                for (int pass = 0; pass < 2; ++pass)
#pragma unroll
                    for (int k = 0; k < TC_CB / 16; ++k)
                        atc_mma_ts(d, pd + k * 16 + (1 - pass) * 8, tc_desc(vd + k * (2048 >> 4)), ATC_IDESC<HD, true>, pass + k > 0);
                atc_commit(&b_o);
                atc_commit(&b_pr[c % 3]);
                atc_commit(&b_vr[c & 1]);
            }
        }
        __syncwarp();
        __syncthreads();
        asm volatile("setmaxnreg.inc.sync.aligned.u32 96;");
    } else if (warp >= TC_OUT) {
        // ---- outputs: half a row to a thread ----
        asm volatile("setmaxnreg.inc.sync.aligned.u32 104;");
        constexpr int HALF = HD / 2;
        const int r = tid & 127, half = (warp - TC_OUT) >> 2;
        const uint32_t o_col = tmem + ((uint32_t)(warp & 3) << 21) + COL_O + half * HALF;
        float2 o[HALF / 2];
        float top = -INFINITY;
        atc_arrive(&b_v[0]);                                 // no output before the first one
#pragma unroll
        for (int d = 0; d < HALF / 2; ++d) o[d] = make_float2(0.f, 0.f);
        for (int c = 0; c < n; ++c) {
            wait(&b_ref[c & 3], (uint32_t)(c >> 2) & 1u);
            const float ref = s_ref[c & 3][r], now = fmaxf(top, ref), to = now == -INFINITY ? 0.f : now;
            const float alpha = at_exp2(top - to), beta = at_exp2(ref - to);
            top = now;
            wait(&b_o, (uint32_t)c & 1u);
            atc_fence_after();
            float v[2][16];
            atc_ld16(o_col, v[0]);
#pragma unroll
            for (int d0 = 0; d0 < HALF; d0 += 16) {
                float (&u)[16] = v[d0 / 16 & 1];
                atc_ld_wait(u);
                if (d0 + 16 < HALF) atc_ld16(o_col + d0 + 16, v[(d0 / 16 + 1) & 1]);
                else { atc_fence_before(); atc_arrive(&b_v[(c + 1) & 1]); }
#pragma unroll
                for (int d = 0; d < 16; d += 2) {
                    float2& y = o[(d0 + d) / 2];
                    y = at_fma2(y, make_float2(alpha, alpha), at_mul2(make_float2(u[d], u[d + 1]), make_float2(beta, beta)));
                }
            }
        }
        __syncthreads();                                     // all products are done, shared memory is free
        float l = 0.f;
        for (int w = 0; w < 2; ++w) l += s_l[w][r] * End<TC_ROWS, 1>::weight<true>(s_m[w][r], top);
        if (half == 0) { s_end.m[0][r] = top; s_end.l[0][r] = l; }
        float* to = reinterpret_cast<float*>(sm) + r * (HD + 4) + half * HALF;
#pragma unroll
        for (int d = 0; d < HALF; d += 4) *reinterpret_cast<float4*>(to + d) = make_float4(o[d / 2].x, o[d / 2].y, o[d / 2 + 1].x, o[d / 2 + 1].y);      // all times 256, like the sums
        asm volatile("setmaxnreg.dec.sync.aligned.u32 96;");
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 104;");
        // ---- weights and sums: a row to a thread, every other chunk ----
        const int w = warp >> 2, r = tid & 127;
        const uint32_t col = tmem + ((uint32_t)(warp & 3) << 21) + COL_S;
        const int32_t pos = s_row[r].pos;
        // scores to powers of two: times k2, or cap2 tanh of them times k2
        const float unit = s_unit[r] * fabsf(a.scale), k2 = CAP ? unit * __frcp_rn(a.cap) : unit * 1.4426950408889634f, cap2 = a.cap * 1.4426950408889634f;
        float m = -INFINITY, l = 0.f;
        for (int c = w; c < n; c += 2) {
            const int32_t p0 = chunk_at<TC_CB>(x, c0 + c);
            const bool all = tile_sees(a, x, p0, TC_CB);
            // position p0 + j is seen for j <= j1 and (j > j0 or j < js)
            const int32_t j1 = pos - p0, j0 = a.window ? j1 - (int32_t)a.window : -1, js = (int32_t)min(a.n_sink, 0x40000000u) - p0;
            auto seen = [&](int j) { return j <= j1 && (j > j0 || j < js); };
            const uint32_t s_col = col + c % 3 * 128;
            wait(&b_s[c % 3], (uint32_t)(c / 3) & 1u);
            atc_fence_after();
            // Two turns over the scores, 8 columns at a time with the next ones under way: the maximum, the weights.  Loops of two
            // steps, one for chunks that every row sees whole, one for the others: unrolled with every choice inside, the turns took
            // 5500 cycles, most of them fetching instructions.
            constexpr int STEP = 8;
            float v[2][STEP], mx[2] = {-INFINITY, -INFINITY};
            float2 sum[2] = {{0.f, 0.f}, {0.f, 0.f}};
            atc_ld8(s_col, v[0]);
            auto maximum = [&](auto whole) {
#pragma unroll 1
                for (int i = 0; i < TC_CB; i += 2 * STEP)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        atc_ld_wait(v[h]);
                        atc_ld8(s_col + (i + (h + 1) * STEP) % TC_CB, v[1 - h]);
#pragma unroll
                        for (int d = 0; d < STEP; d += 2) {
                            auto score = [&](int e) { return decltype(whole)::value || seen(i + h * STEP + e) ? v[h][e] : -INFINITY; };
                            mx[d >> 1 & 1] = atc_max3(mx[d >> 1 & 1], score(d), score(d + 1));
                        }
                    }
            };
            if (all) maximum(std::true_type{});
            else maximum(std::false_type{});
            float top = fmaxf(mx[0], mx[1]);
            top = CAP ? cap2 * at_tanh(top * k2) : top * k2;
            const float mn = fmaxf(m, top), ref = mn == -INFINITY ? 0.f : mn, shift = 8.f - ref;      // times 256: the low terms stay clear of the subnormals
            const float alpha = at_exp2(m - ref);
            m = mn;
            s_ref[c & 3][r] = mn;
            atc_arrive(&b_ref[c & 3]);
            auto turn = [&](auto whole) {
#pragma unroll 1
                for (int i = 0; i < TC_CB; i += 2 * STEP)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float (&u)[STEP] = v[h];
                        atc_ld_wait(u);
                        if (i + h * STEP + STEP < TC_CB) atc_ld8(s_col + i + (h + 1) * STEP, v[1 - h]);
                        uint32_t hi[STEP / 2], lo[STEP / 2];
#pragma unroll
                        for (int d = 0; d < STEP; d += 2) {
                            float2 y = make_float2(u[d], u[d + 1]);
                            if (CAP) y = at_fma2(make_float2(at_tanh(y.x * k2), at_tanh(y.y * k2)), make_float2(cap2, cap2), make_float2(shift, shift));
                            else y = at_fma2(y, make_float2(k2, k2), make_float2(shift, shift));
                            y.x = at_exp2(y.x); y.y = at_exp2(y.y);
                            if (!decltype(whole)::value) { if (!seen(i + h * STEP + d)) y.x = 0.f; if (!seen(i + h * STEP + d + 1)) y.y = 0.f; }
                            sum[d >> 1 & 1] = at_add2(sum[d >> 1 & 1], y);
                            at_split_h(y.x, y.y, hi[d / 2], lo[d / 2]);
                        }
                        const uint32_t at = (uint32_t)((i + h * STEP) & ~15) + ((i + h * STEP) & 15) / 2;
                        atc_st4(s_col + at, hi);
                        atc_st4(s_col + at + 8, lo);
                    }
            };
            if (all) turn(std::true_type{});
            else turn(std::false_type{});
            const float2 both = at_add2(sum[0], sum[1]);
            l = fmaf(l, alpha, both.x + both.y);
            atc_st_wait();
            atc_fence_before();
            atc_arrive(&b_p[c % 3]);
        }
        s_m[w][r] = m; s_l[w][r] = l;
        atc_fence_before();
        __syncthreads();
        asm volatile("setmaxnreg.dec.sync.aligned.u32 96;");
    }
    atc_fence_after();
    __syncthreads();
    if (warp == TC_ISSUE) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(tmem), "r"(512u) : "memory");
    if (s_dead) {                                        // what it shares stays as no call has left it
        if (tid == 0 && sharers > 1) atomicInc(a.tickets + part.slot, sharers - 1);
        return;
    }
    settle<__half, HD, TC_ROWS, 1, TC_THREADS, true, false>(a, x, s_row, part, sharers, reinterpret_cast<float*>(sm), s_end);
}

template <int HD, bool TMA, bool CAP>
static int launch_tc(const AttnArgs& a, const KvCache& kv) {
    static bool set = false;
    if (!set) {
        if (cudaFuncSetAttribute((const void*)k_attn_tc<HD, TMA, CAP>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)AttnTc<HD>::SMEM) != cudaSuccess)
            return fail(ADAMAH_ERR_BACKEND, "attn_kv: cannot raise the shared-memory limit");
        set = true;
    }
    k_attn_tc<HD, TMA, CAP><<<attn_grid(a), TC_THREADS, AttnTc<HD>::SMEM, g.stream>>>(a, kv.map, kv.run);
    count_launch();
    return check_launch("map_attn_kv");
}
template <int HD, bool TMA>
static int launch_cap(const AttnArgs& a, const KvCache& kv) {
    return a.cap > 0.f ? launch_tc<HD, TMA, true>(a, kv) : launch_tc<HD, TMA, false>(a, kv);
}
int launch_attn_tc(const AttnArgs& a, const KvCache& kv) {
    if (kv.run) return a.geo.hd == 64 ? launch_cap<64, true>(a, kv) : launch_cap<128, true>(a, kv);
    return a.geo.hd == 64 ? launch_cap<64, false>(a, kv) : launch_cap<128, false>(a, kv);
}

}  // namespace ab
