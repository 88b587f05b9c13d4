// Attention of new rows over a paged cache: a token per sequence or a chunk of a prompt, a sliding window and first
// positions that stay visible (map_matmul_t.comp + map_attn_softmax_value.comp over a contiguous cache, a row at a time).
//
//   s_j = scale q.k_j, or cap tanh(scale q.k_j / cap);   o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),   j visible to the row
//
// The rows of an entry times the query heads of a key head are one list, cut into tiles that share what they read of the
// cache: 2 or 4 rows in 32-bit arithmetic (attn_kv_thin.cu), 128 by tcgen05 (attn_kv_tc.cu), the widths between them here.  On
// the tensor cores both products have operands at the precision of 32 bits: the cache's fp16 values are exact operands, and a query row or a row of weights goes in as two fp16 terms (22 bits); a float32 cache takes three tf32
// products (x_hi y_hi + x_hi y_lo + x_lo y_hi).  A chunk's P V goes into fresh accumulators and joins the running output in
// fp32 with the rescaling that the running maximum needs anyway: the tensor core rounds its sums towards zero, and a sum
// over 65000 positions that never left it would be 2e-4 off.
//
// Values of positions that no row of the tile sees are zeros in shared memory, whatever the cache holds there, and scores of
// such positions are not looked at.  Where a value that some rows see and others do not is an infinity or a NaN, the others' results
// are NaN (0 times it); results that are not finite are done again by attend_row, which reads only what the row sees.
#include "attn_kv.cuh"

#include <algorithm>

namespace ab {

// 16-byte words of 16-bit rows, so that eight neighbouring rows of one column lie in different banks
template <int HD>
__device__ __forceinline__ int swz(int r, int ch) { return HD >= 64 ? ch ^ (r & 7) : ch ^ ((r >> 1) & 3); }

// A query row into shared memory by a warp: two fp16 planes (`plane` halves apart) of the row times a power of two, whose inverse
// comes back, or floats.
template <typename T, int HD, int LD>
__device__ __forceinline__ float put_query(const AttnArgs& a, const AttnRow& row, uint8_t* sq, int r, int plane) {
    const int lane = threadIdx.x & 31;
    float v[HD / 32], most = 0.f, up = 1.f, down = 1.f;
#pragma unroll
    for (int j = 0; j < HD / 32; ++j) { v[j] = row.pos >= 0 ? a.act[row.q + lane + 32 * j] : 0.f; most = fmaxf(most, fabsf(v[j])); }
    if (sizeof(T) == 2) row_scale(warp_max(most), up, down);
#pragma unroll
    for (int j = 0; j < HD / 32; ++j) {
        const int d = lane + 32 * j;
        if constexpr (sizeof(T) == 2) {
            const float y = v[j] * up;
            const __half hi = __float2half_rn(y);
            __half* p = reinterpret_cast<__half*>(sq) + r * HD + swz<HD>(r, d >> 3) * 8 + (d & 7);
            p[0] = hi; p[plane] = __float2half_rn(y - __half2float(hi));
        } else reinterpret_cast<float*>(sq)[r * LD + d] = v[j];
    }
    return down;
}
// Scores of 16 rows (r0 ..) and 8 NT positions (p0 ..): s[n][e] is row r0 + g + 8 (e >> 1), position p0 + 8 n + 2 q4 + (e & 1).
template <int HD, int NT>
__device__ __forceinline__ void scores_h(float (&s)[NT][4], uint32_t q_s, int plane, int r0, uint32_t k_s, int p0) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
#pragma unroll 4
    for (int k = 0; k < HD / 16; ++k) {
        uint32_t qh[4], ql[4];
        const int qr = r0 + (lane & 15), qc = 2 * k + (lane >> 4);
        const uint32_t qo = q_s + (uint32_t)(qr * HD + swz<HD>(qr, qc) * 8) * 2u;
        at_ldsm(qo, qh);
        at_ldsm(qo + plane * 2, ql);
#pragma unroll
        for (int n = 0; n < NT / 2; ++n) {
            uint32_t b[4];
            const int kr = p0 + n * 16 + (lane >> 4) * 8 + (lane & 7), kc = 2 * k + ((lane >> 3) & 1);
            at_ldsm(k_s + (uint32_t)(kr * HD + swz<HD>(kr, kc) * 8) * 2u, b);
            at_mma_h(s[2 * n], ql, b[0], b[1]); at_mma_h(s[2 * n + 1], ql, b[2], b[3]);
            at_mma_h(s[2 * n], qh, b[0], b[1]); at_mma_h(s[2 * n + 1], qh, b[2], b[3]);
        }
    }
}
// The same over floats; sums leave the tensor core every 64 dims (96 steps of a head of 256 made 3e-6 of the result)
template <int HD, int LD, int NT>
__device__ __forceinline__ void scores_f(float (&s)[NT][4], const float* q, int r0, const float* k_rows, int p0) {
    const int lane = threadIdx.x & 31, g = lane >> 2, q4 = lane & 3;
    constexpr int PART = HD < 64 ? HD : 64;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
#pragma unroll 1
    for (int k0 = 0; k0 < HD; k0 += PART) {
        float acc[NT][4] = {};
#pragma unroll 4
        for (int k = k0; k < k0 + PART; k += 8) {
            const float* qp = q + (r0 + g) * LD + k + q4;
            uint32_t ah[4], al[4];
            at_split_t(qp[0], ah[0], al[0]); at_split_t(qp[8 * LD], ah[1], al[1]);
            at_split_t(qp[4], ah[2], al[2]); at_split_t(qp[8 * LD + 4], ah[3], al[3]);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const float* kp = k_rows + (p0 + n * 8 + g) * LD + k + q4;
                uint32_t b0h, b0l, b1h, b1l;
                at_split_t(kp[0], b0h, b0l); at_split_t(kp[4], b1h, b1l);
                at_mma_t(acc[n], al, b0h, b1h); at_mma_t(acc[n], ah, b0l, b1l); at_mma_t(acc[n], ah, b0h, b1h);
            }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[n][e] += acc[n][e];
    }
}
// Scores to weights: running maximum and sum of each row over its quad of lanes; alpha: the factor of what was summed before.
template <int NT>
__device__ __forceinline__ void weights(float (&s)[NT][4], const AttnArgs& a, bool all, const int32_t (&pos)[2], const float (&scl)[2], int32_t p0, float (&m)[2],
                                        float (&l)[2], float (&alpha)[2]) {
    const int q4 = threadIdx.x & 3;
    const float rcap = a.cap > 0.f ? __frcp_rn(a.cap) : 0.f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        float mx = -INFINITY;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 2 * h; e < 2 * h + 2; ++e) {
                float y = s[n][e] * scl[h];
                if (a.cap > 0.f) y = a.cap * at_tanh(y * rcap);
                if (!all && !row_sees(a, pos[h], p0 + 8 * n + 2 * q4 + (e & 1))) y = -INFINITY;
                s[n][e] = y;
                mx = max_nan(mx, y);
            }
        mx = max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float mn = max_nan(m[h], mx), ref = mn == -INFINITY ? 0.f : mn;
        alpha[h] = expf(m[h] - ref);
        m[h] = mn;
        float sum = 0.f;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 2 * h; e < 2 * h + 2; ++e) { s[n][e] = expf(s[n][e] - ref); sum += s[n][e]; }
        l[h] = fmaf(l[h], alpha[h], sum);
    }
}
// o = o alpha + weights x values of the positions p0 .. p0 + 8 NT - 1 (fp16: times 256, which keeps the low terms clear of the
// subnormals)
template <int HD, int NT>
__device__ __forceinline__ void values_h(float (&o)[HD / 8][4], const float (&s)[NT][4], const float (&alpha)[2], uint32_t v_s, int p0) {
    const int lane = threadIdx.x & 31;
    uint32_t ph[NT / 2][4], pl[NT / 2][4];
#pragma unroll
    for (int k = 0; k < NT / 2; ++k)
#pragma unroll
        for (int f = 0; f < 4; ++f) {
            const float* p = &s[2 * k + (f >> 1)][2 * (f & 1)];
            at_split_h(p[0] * 256.f, p[1] * 256.f, ph[k][f], pl[k][f]);
        }
    constexpr int DC = HD == 256 && NT > 2 ? 32 : HD >= 64 ? 64 : HD;     // dims per round: what the registers beside `o` allow
#pragma unroll
    for (int d0 = 0; d0 < HD; d0 += DC) {
        float acc[DC / 8][4] = {};
#pragma unroll
        for (int k = 0; k < NT / 2; ++k)
#pragma unroll
            for (int n = 0; n < DC / 16; ++n) {
                uint32_t b[4];
                const int vr = p0 + k * 16 + ((lane >> 3) & 1) * 8 + (lane & 7), vc = d0 / 8 + 2 * n + (lane >> 4);
                at_ldsm_t(v_s + (uint32_t)(vr * HD + swz<HD>(vr, vc) * 8) * 2u, b);
                at_mma_h(acc[2 * n], pl[k], b[0], b[1]); at_mma_h(acc[2 * n + 1], pl[k], b[2], b[3]);
                at_mma_h(acc[2 * n], ph[k], b[0], b[1]); at_mma_h(acc[2 * n + 1], ph[k], b[2], b[3]);
            }
#pragma unroll
        for (int j = 0; j < DC / 8; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[d0 / 8 + j][e] = fmaf(o[d0 / 8 + j][e], alpha[e >> 1], acc[j][e]);
    }
}
// The order of the positions inside a step of 8 is free: slots t and t + 4 are positions 2 t and 2 t + 1, which is how the scores lie
// in the registers.
template <int HD, int LD, int NT>
__device__ __forceinline__ void values_f(float (&o)[HD / 8][4], const float (&s)[NT][4], const float (&alpha)[2], const float* v_rows, int p0) {
    const int lane = threadIdx.x & 31, g = lane >> 2, q4 = lane & 3;
    uint32_t ph[NT][4], pl[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        at_split_t(s[n][0], ph[n][0], pl[n][0]); at_split_t(s[n][2], ph[n][1], pl[n][1]);
        at_split_t(s[n][1], ph[n][2], pl[n][2]); at_split_t(s[n][3], ph[n][3], pl[n][3]);
    }
#pragma unroll
    for (int j = 0; j < HD / 8; ++j) {
        float acc[4] = {};
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const float* vp = v_rows + (p0 + n * 8 + 2 * q4) * LD + j * 8 + g;
            uint32_t b0h, b0l, b1h, b1l;
            at_split_t(vp[0], b0h, b0l); at_split_t(vp[LD], b1h, b1l);
            at_mma_t(acc, pl[n], b0h, b1h); at_mma_t(acc, ph[n], b0l, b1l); at_mma_t(acc, ph[n], b0h, b1h);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) o[j][e] = fmaf(o[j][e], alpha[e >> 1], acc[e]);
    }
}

// The warps' results into shared memory, then the rest of the way.
template <typename T, int HD, int ROWS, int PLANES, int THREADS, bool CLUSTER>
__device__ __forceinline__ void finish(const AttnArgs& a, const AttnTile& x, const AttnRow* rows, const AttnShare& part, uint32_t sharers,
                                       int plane, int r0, const float (&o)[HD / 8][4], const float (&m)[2], float (&l)[2], float* merge, End<ROWS, PLANES>& end) {
    constexpr int LM = HD + 4;
    constexpr float UNIT = sizeof(T) == 2 ? 1.f / 256.f : 1.f;
    const int lane = threadIdx.x & 31, g = lane >> 2, q4 = lane & 3;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
        if (q4 == 0) { end.m[plane][r0 + g + 8 * h] = m[h]; end.l[plane][r0 + g + 8 * h] = l[h]; }
    }
    __syncthreads();                                     // (and nobody reads what `merge` lies on any more)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int r = r0 + g + 8 * h;
        const float f = end.template factor<false>(plane, r) * UNIT;
#pragma unroll
        for (int j = 0; j < HD / 8; ++j)
            *reinterpret_cast<float2*>(merge + (plane * ROWS + r) * LM + 8 * j + 2 * q4) = make_float2(o[j][2 * h] * f, o[j][2 * h + 1] * f);
    }
    settle<T, HD, ROWS, PLANES, THREADS, false, CLUSTER>(a, x, rows, part, sharers, merge, end);
}
// ---- few rows: 16 per tile -------------------------------------------------------------------------------------------
// Every warp has chunks of 16 positions of its own (chunk w, w + W, ..), the next ones under way in STAGES slots of
// shared memory, and its own running maxima, sums and outputs; nothing in the loop waits for another warp.  Bound by what a warp
// has to do in turn for a chunk of 16 positions, most of it for rows that a tile may not have.
template <typename T, int HD>
struct Few {
    static constexpr int ROWS = 16, CB = 16, ROW_BYTES = HD * (int)sizeof(T);
    static constexpr int W = ROW_BYTES == 1024 ? 3 : 4, STAGES = ROW_BYTES == 1024 ? 2 : ROW_BYTES >= 256 ? 3 : 4;
    static constexpr int LD = sizeof(T) == 2 ? HD : HD + 4;                       // elements of a row in shared memory
    static constexpr int SLOT = 2 * CB * LD * (int)sizeof(T);                     // keys and values of a chunk
    static constexpr int Q_BYTES = ROWS * LD * 4;                                 // two fp16 planes, or floats
    static constexpr int RING = W * STAGES * SLOT, MERGE = W * ROWS * (HD + 4) * 4;
    static constexpr int SMEM = Q_BYTES + (RING > MERGE ? RING : MERGE);
    static_assert(SMEM <= 225 * 1024, "shared memory");
};

// CLUSTER: a tile's CTAs are a cluster
template <typename T, int HD, bool CLUSTER>
__global__ void __launch_bounds__(Few<T, HD>::W * 32) k_attn_few(const __grid_constant__ AttnArgs a) {
    using F = Few<T, HD>;
    constexpr int ROWS = F::ROWS, CB = F::CB, W = F::W, LD = F::LD, STAGES = F::STAGES;
    constexpr bool H = sizeof(T) == 2;
    extern __shared__ __align__(128) uint8_t sm[];
    __shared__ AttnRow s_row[ROWS];
    __shared__ float s_unit[ROWS];
    __shared__ Found s_found;
    __shared__ End<ROWS, W> s_end;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2;
    const AttnShare part = share_of(a);
    const uint32_t kvh = part.kvh;
    AttnTile x;
    if (!find_tile<ROWS, CB>(a, part.tile, kvh, x, s_row, s_found)) return;
    uint32_t sharers, c0, c1;
    if (!share_out(a, x, part, sharers, c0, c1) && !CLUSTER) return;         // in a cluster it still takes its rows
    c0 = min(c0, c1);

    uint8_t* const ring = sm + F::Q_BYTES + warp * STAGES * F::SLOT;
    const uint32_t ring_s = at_smem(ring), q_s = at_smem(sm);
    const T* const pool = reinterpret_cast<const T*>(a.pool);
    const size_t v_off = (size_t)a.geo.n_kv * a.geo.page * HD;
    // Chunks of this warp: c0 + warp, + W, ...  Lane l knows where position l % 16 of the next one to be asked for lies.
    uint32_t ask = c0 + warp;
    auto locate = [&]() -> int64_t { return ask < c1 ? tile_position(a, x, kvh, chunk_at<CB>(x, ask) + (lane & 15)) : -1; };
    int64_t where = locate();
    auto request = [&](int slot) {
        constexpr int WPR = HD * (int)sizeof(T) / 16;    // words of a row
        if (ask < c1) {
#pragma unroll 8
            for (int i = 0; i < CB * WPR / 32; ++i) {
                const int w = i * 32 + lane, r = w / WPR, ch = w % WPR;
                const int64_t at = __shfl_sync(0xffffffffu, where, r);
                const T* src = pool + (at < 0 ? 0 : at) + ch * (16 / sizeof(T));
                const uint32_t dst = ring_s + slot * F::SLOT + (H ? (uint32_t)(r * HD + swz<HD>(r, ch) * 8) * 2u : (uint32_t)(r * LD + ch * 4) * 4u);
                at_cp16(dst, src, at >= 0);
                at_cp16(dst + F::SLOT / 2, src + v_off, at >= 0);
            }
        }
        at_commit();
        ask += W;
        where = locate();
    };
#pragma unroll 1
    for (int i = 0; i < STAGES - 1; ++i) request(i);
    for (int r = warp; r < ROWS; r += W) {
        const float unit = put_query<T, HD, LD>(a, s_row[r], sm, r, ROWS * HD);
        if (lane == 0) s_unit[r] = unit;
    }
    __syncthreads();

    const int32_t pos[2] = {s_row[g].pos, s_row[g + 8].pos};
    const float scl[2] = {s_unit[g] * a.scale, s_unit[g + 8] * a.scale};
    float o[HD / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int j = 0; j < HD / 8; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[j][e] = 0.f;
    int slot = 0;
#pragma unroll 1
    for (uint32_t c = c0 + warp; c < c1; c += W) {
        at_wait<STAGES - 2>();
        __syncwarp();
        const uint32_t k_s = ring_s + slot * F::SLOT;
        const float* kf = reinterpret_cast<const float*>(ring + slot * F::SLOT);
        request(slot ? slot - 1 : STAGES - 1);           // the slot that the chunk before this one has left
        const int32_t p0 = chunk_at<CB>(x, c);
        float s[2][4], alpha[2];
        if constexpr (H) scores_h<HD, 2>(s, q_s, ROWS * HD, 0, k_s, 0);
        else scores_f<HD, LD, 2>(s, reinterpret_cast<const float*>(sm), 0, kf, 0);
        weights<2>(s, a, tile_sees(a, x, p0, CB), pos, scl, p0, m, l, alpha);
        if constexpr (H) values_h<HD, 2>(o, s, alpha, k_s + F::SLOT / 2, 0);
        else values_f<HD, LD, 2>(o, s, alpha, kf + CB * LD, 0);
        slot = slot + 1 == STAGES ? 0 : slot + 1;
    }
    at_wait<0>();
    finish<T, HD, ROWS, W, W * 32, CLUSTER>(a, x, s_row, part, sharers, warp, 0, o, m, l, reinterpret_cast<float*>(sm + F::Q_BYTES), s_end);
}

// ---- many rows: 32 or 64 per tile ------------------------------------------------------------------------------------
// RG groups of 16 rows, KH warps to a group, each with its share of every chunk's positions; two chunks of keys and values in
// shared memory for all of them.
template <typename T, int HD, int RG, int KH>
struct Many {
    static constexpr int ROWS = RG * 16, CB = sizeof(T) == 2 ? 64 : 32, LD = sizeof(T) == 2 ? HD : HD + 4;
    static constexpr int PART = CB * LD * (int)sizeof(T);                         // keys, or values, of a chunk
    static constexpr int Q_BYTES = ROWS * LD * 4, MERGE = KH * ROWS * (HD + 4) * 4;
    static constexpr int SMEM = Q_BYTES + 4 * PART > MERGE ? Q_BYTES + 4 * PART : MERGE;
    static_assert(SMEM <= 225 * 1024, "shared memory");
};

template <typename T, int HD, int RG, int KH>
__global__ void __launch_bounds__(RG * KH * 32) k_attn_many(const __grid_constant__ AttnArgs a) {
    using F = Many<T, HD, RG, KH>;
    constexpr int ROWS = F::ROWS, CB = F::CB, LD = F::LD, NT = CB / KH / 8, THREADS = RG * KH * 32;
    constexpr bool H = sizeof(T) == 2;
    extern __shared__ __align__(128) uint8_t sm[];
    __shared__ AttnRow s_row[ROWS];
    __shared__ float s_unit[ROWS];
    __shared__ Found s_found;
    __shared__ int64_t s_where[2][CB];
    __shared__ End<ROWS, KH> s_end;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rg = warp % RG, kh = warp / RG, r0 = rg * 16, g = lane >> 2;
    const AttnShare part = share_of(a);
    const uint32_t kvh = part.kvh;
    AttnTile x;
    if (!find_tile<ROWS, CB>(a, part.tile, kvh, x, s_row, s_found)) return;
    uint32_t sharers, c0, c1;
    if (!share_out(a, x, part, sharers, c0, c1)) return;
    uint8_t* const tiles = sm + F::Q_BYTES;              // chunk c: keys at (c & 1) * 2 PART, values behind them
    const uint32_t tiles_s = at_smem(tiles), q_s = at_smem(sm);
    const T* const pool = reinterpret_cast<const T*>(a.pool);
    const size_t v_off = (size_t)a.geo.n_kv * a.geo.page * HD;
    auto locate = [&](uint32_t c) { if (tid < CB) s_where[c & 1][tid] = c < c1 ? tile_position(a, x, kvh, chunk_at<CB>(x, c) + tid) : -1; };
    auto request = [&](uint32_t c) {                     // c < c1: chunk c, whose positions are located
        constexpr int WPR = HD * (int)sizeof(T) / 16;
        if (c < c1) {
            const uint32_t base = tiles_s + (c & 1) * 2 * F::PART;
#pragma unroll 4
            for (int w = tid; w < CB * WPR; w += THREADS) {
                const int r = w / WPR, ch = w % WPR;
                const int64_t at = s_where[c & 1][r];
                const T* src = pool + (at < 0 ? 0 : at) + ch * (16 / sizeof(T));
                const uint32_t dst = base + (H ? (uint32_t)(r * HD + swz<HD>(r, ch) * 8) * 2u : (uint32_t)(r * LD + ch * 4) * 4u);
                at_cp16(dst, src, at >= 0);
                at_cp16(dst + F::PART, src + v_off, at >= 0);
            }
        }
        at_commit();
    };
    locate(c0); locate(c0 + 1);
    __syncthreads();
    request(c0); request(c0 + 1);
    for (int r = r0 + kh * (16 / KH); r < r0 + (kh + 1) * (16 / KH); ++r) {
        const float unit = put_query<T, HD, LD>(a, s_row[r], sm, r, ROWS * HD);
        if (lane == 0) s_unit[r] = unit;
    }
    __syncthreads();
    const int32_t pos[2] = {s_row[r0 + g].pos, s_row[r0 + g + 8].pos};
    const float scl[2] = {s_unit[r0 + g] * a.scale, s_unit[r0 + g + 8] * a.scale};
    float o[HD / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int j = 0; j < HD / 8; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[j][e] = 0.f;
    // the warp's own rows: positions that none of them sees are left out
    int32_t w_lo = x.hi, w_hi = -1;
    for (int r = r0; r < r0 + 16; ++r) if (s_row[r].pos >= 0) { w_lo = min(w_lo, s_row[r].pos); w_hi = max(w_hi, s_row[r].pos); }
#pragma unroll 1
    for (uint32_t c = c0; c < c1; ++c) {
        at_wait<1>();
        __syncthreads();
        locate(c + 2);
        const int p_in = kh * (CB / KH);
        const int32_t p0 = chunk_at<CB>(x, c) + p_in, p1 = p0 + CB / KH - 1;
        const bool some = p0 <= w_hi && (a.window == 0 || p1 > w_lo - (int32_t)a.window || (uint32_t)p0 < a.n_sink);
        const bool all = p1 <= w_lo && (a.window == 0 || p0 > w_hi - (int32_t)a.window || (uint32_t)p1 < a.n_sink);
        if (some) {
            const uint32_t k_s = tiles_s + (c & 1) * 2 * F::PART;
            const float* kf = reinterpret_cast<const float*>(tiles + (c & 1) * 2 * F::PART);
            float s[NT][4], alpha[2];
            if constexpr (H) scores_h<HD, NT>(s, q_s, ROWS * HD, r0, k_s, p_in);
            else scores_f<HD, LD, NT>(s, reinterpret_cast<const float*>(sm), r0, kf, p_in);
            weights<NT>(s, a, all, pos, scl, p0, m, l, alpha);
            if constexpr (H) values_h<HD, NT>(o, s, alpha, k_s + F::PART, p_in);
            else values_f<HD, LD, NT>(o, s, alpha, kf + CB * LD, p_in);
        }
        __syncthreads();
        request(c + 2);
    }
    at_wait<0>();
    finish<T, HD, ROWS, KH, THREADS, false>(a, x, s_row, part, sharers, kh, r0, o, m, l, reinterpret_cast<float*>(sm), s_end);
}

template <typename T, int HD>
static int launch_few(const AttnArgs& a) {
    static bool set[2] = {false, false};
    using F = Few<T, HD>;
    if (attn_cluster(a)) return launch_attn(k_attn_few<T, HD, true>, set[1], a, F::W * 32, F::SMEM, true);
    return launch_attn(k_attn_few<T, HD, false>, set[0], a, F::W * 32, F::SMEM, false);
}
template <typename T, int HD, int RG, int KH>
static int launch_many(const AttnArgs& a) {
    static bool set = false;
    return launch_attn(k_attn_many<T, HD, RG, KH>, set, a, RG * KH * 32, Many<T, HD, RG, KH>::SMEM, false);
}
template <typename T, int HD>
static int launch_rows(const AttnArgs& a, const KvCache& kv, uint32_t rows) {
    if (rows <= 4) return launch_attn_thin(a, sizeof(T), rows);
    if (rows > 16) {                                     // 32 and 64 for heads of 256 and floats of 128, 128 for fp16 heads of 64 and 128
        if constexpr (HD == 256 || (HD == 128 && sizeof(T) == 4)) return rows == 64 ? launch_many<T, HD, 4, 2>(a) : launch_many<T, HD, 2, 4>(a);
        else if constexpr (HD > 32 && sizeof(T) == 2) return launch_attn_tc(a, kv);
    }
    return launch_few<T, HD>(a);
}
template <typename T>
static int launch_hd(const AttnArgs& a, const KvCache& kv, uint32_t rows) {
    switch (a.geo.hd) {
    case 32: return launch_rows<T, 32>(a, kv, rows);
    case 64: return launch_rows<T, 64>(a, kv, rows);
    case 128: return launch_rows<T, 128>(a, kv, rows);
    default: return launch_rows<T, 256>(a, kv, rows);
    }
}

int kv_batch(const char* name, uint32_t kv_id, uint32_t layer, uint32_t seq_h, uint32_t start_h, uint32_t n_seqs, uint32_t n_rows, uint32_t n_head,
             KvCache** kv_out, KvBatch* b);

}  // namespace ab

using namespace ab;

extern "C" int map_attn_kv_dev(uint32_t map, uint32_t kv_id, uint32_t layer, uint32_t q_h, uint32_t out_h, uint32_t seq_h, uint32_t start_h,
                               uint32_t n_seqs, uint32_t n_rows, uint32_t n_head, uint32_t window, uint32_t n_sink, float scale, float cap) {
    if (!ready()) return ADAMAH_ERR_INVALID;
    Map* m = get_map(map);
    if (!m) return ADAMAH_ERR_NOT_FOUND;
    if (m->dtype != ADAMAH_DTYPE_F32 || m->pack_size != 1) return fail(ADAMAH_ERR_INVALID, "attn_kv: map %u must be float32 with pack_size 1", map);
    KvCache* kv;
    AttnArgs a = {};
    if (int rc = kv_batch("attn_kv", kv_id, layer, seq_h, start_h, n_seqs, n_rows, n_head, &kv, &a.b)) return rc;
    if (!isfinite(scale) || !(cap >= 0.f) || !isfinite(cap)) return fail(ADAMAH_ERR_INVALID, "attn_kv: scale %g, cap %g", scale, cap);
    for (uint32_t h : {q_h, out_h}) if (!handle_ok(h, n_rows * 4)) return ADAMAH_ERR_NOT_FOUND;
    if (!n_rows || !n_seqs) return ADAMAH_OK;
    a.act = (float*)m->buf; a.n_act = m->n_elems; a.l_q = hlocs(q_h); a.l_out = hlocs(out_h);
    a.geo = kv->geo; a.pool = kv->pool; a.layer = layer; a.n_head = n_head; a.group = n_head / kv->d.n_head_kv;
    a.window = window >= 1u << 30 ? 0u : window;         // no sequence is that long
    a.n_sink = n_sink; a.scale = scale; a.cap = cap; a.err = g.dev_err;
    a.part = kv->part; a.tickets = kv->tickets;
    a.pool_rows = (uint32_t)((uint64_t)kv->d.n_pages * kv->geo.page_elems / kv->d.head_dim);
    // Tiles: every entry has its rows * group / ROWS and a part of one more.
    const uint32_t entries = std::min(n_seqs, n_rows), sms = (uint32_t)g.sm_count;
    const uint64_t flat = (uint64_t)n_rows * a.group;
    auto tiles_of = [&](uint64_t rows) { return (flat + (rows - 1) * entries) / rows; };
    if (tiles_of(2) * a.geo.n_kv >= (1u << 30)) return fail(ADAMAH_ERR_INVALID, "attn_kv: %u rows of %u heads", n_rows, n_head);
    // How far the sequences reach only decides the launch; a graph that is replayed later divides what there is then.
    uint32_t reach = kv->pages.longest();
    if (a.window) reach = (uint32_t)std::min<uint64_t>(reach, (uint64_t)a.window + n_sink);
    const uint32_t parts = (reach + 127) / 128, hd = a.geo.hd;
    const bool f16 = kv->elem == 2;
    const uint32_t rows = [&]() -> uint32_t {
        // Rows of a tile.  The measured times are of 32 heads over 16 of 128 dims if not said otherwise, fp16 cache.
        const uint64_t work16 = tiles_of(16) * a.geo.n_kv * parts, work64 = tiles_of(64) * a.geo.n_kv * parts;
        // 2 or 4 in 32-bit arithmetic where an entry has no more (64 decoding sequences of 2047: 125 us against 205 in tiles of 16).
        // Over floats, whose tensor-core products come in threes, also for more: 8 sequences of 16 new tokens behind 1000: 92 us against
        // 139; with heads of 256 until the whole is large: one of 64 behind 8000, 4 heads over 1: 125 us against 121 to 183.  With
        // fp16 heads of 256 while the whole is small: 8 tokens behind 8000, 4 heads over 1: 33 us against 55.
        const bool thin = f16 ? flat <= 4ull * entries || (hd == 256 && work16 <= 2ull * sms) : flat <= 32ull * entries || (hd == 256 && work64 <= 16ull * sms);
        if (thin && a.geo.page % attn_thin_chunk(kv->elem, hd) == 0) return flat <= 2ull * entries ? 2 : 4;
        // 16 where an entry has no more (wider tiles would be empty: 32 entries of 8 tokens behind 1000: 67 us against 85), where the whole is
        // small, so that more CTAs count for more than less reading (16 tokens behind 2000: 20 us against 22; behind 8000 and 64 tokens: 121
        // against 50), and for short rows, where the wider tiles never won.
        if (flat <= 16ull * entries || work16 <= 7ull * sms || hd == 32 || (!f16 && hd == 64)) return 16;
        if (f16 && hd <= 128) return 128;
        // 64 for a large whole (1024 tokens behind 8000, heads of 256, 4 over 1: 333 us against 447; 2048 tokens of a prompt: 156 against 115)
        return work64 > 16ull * sms ? 64 : 32;
    }();
    a.pairs = (uint32_t)tiles_of(rows) * a.geo.n_kv;
    // Splits: what fills the GPU once and again is left whole, and the rest (or all, where it is less) divided among as many CTAs
    // as the GPU holds at once, no more than the workspace has room for: 512 tiles on 148 SMs take 3.5 turns, not 4.
    const uint32_t chunk = rows <= 4 ? attn_thin_chunk(kv->elem, hd) : rows == 16 ? 16 : rows == 128 ? 128 : f16 ? 64 : 32;
    // Positions of a part: 128, but of a short row's 32 or 64 as long as a cluster of 16 has them all (4 heads of 256 over 1: 130 positions
    // 12.4 -> 9.6 us, 300 14.5 -> 9.7; 1000 in 32s 12.5, in 64s 10.5; 4000 in 64s 18.6, in 128s 16.6)
    uint32_t unit = 128;
    while (rows <= 4 && unit > 32 && reach <= unit / 2 * ATTN_CLUSTER) unit /= 2;
    a.least = std::max(1u, unit / chunk);
    const uint32_t slots = std::min(sms * (rows <= 4 ? THIN_CTAS : rows == 16 ? 2 : 1), KV_SPLIT_CTAS), rest = a.pairs % slots;
    a.whole = a.pairs; a.splits = 1;
    if (rest) {
        a.splits = std::min({slots / rest, KV_SPLIT_CTAS * KV_SPLIT_ROWS / rows / rest, (reach + unit - 1) / unit});
        // The last CTA adds up 128 rows of each: no more of them than the square root of twice the parts (8 heads over 1, 8 tokens
        // behind 8000: 71 us with 63 splits, 32 with 11)
        if (rows == 128)
            for (uint32_t most = 1; most < a.splits; ++most)
                if (most * most >= 2 * parts) a.splits = most;
        // Clusters of 2, 4 or 8 where that is about enough, or of 16 as long as they find their place (16 key heads behind 2000: 17 us in
        // 8, 24 in 16).  What a power of two leaves idle counts for long sequences.
        if (rows <= 16 && rest == a.pairs && a.splits <= ATTN_CLUSTER) {
            uint32_t c = 1;
            while (2 * c <= a.splits && (c < 8 || 16 * rest <= sms)) c *= 2;
            if (4 * c >= 3 * a.splits || reach < 1024 * a.splits) a.splits = c;
        }
        if (a.splits > 1) a.whole = a.pairs - rest;
        else a.splits = 1;
    }
    const int rc = kv->elem == 2 ? launch_hd<__half>(a, *kv, rows) : launch_hd<float>(a, *kv, rows);
    end_of_op();
    return rc;
}
