// Attention of new rows over a paged cache: a token per sequence or a chunk of a prompt, a sliding window and first
// positions that stay visible (map_matmul_t.comp + map_attn_softmax_value.comp over a contiguous cache, a row at a time).
//
//   s_j = scale q.k_j, or cap tanh(scale q.k_j / cap);   o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),   j visible to the row
//
// The rows of an entry times the query heads of a key head are one list, cut into tiles that share what they read of the
// cache.  Both products run on the tensor cores with the operands at the precision of 32 bits: the cache's fp16 values are
// exact operands, and a query row or a row of weights goes in as two fp16 terms (22 bits); a float32 cache takes three tf32
// products (x_hi y_hi + x_hi y_lo + x_lo y_hi).  A chunk's P V goes into fresh accumulators and joins the running output in
// fp32 with the rescaling that the running maximum needs anyway: the tensor core rounds its sums towards zero, and a sum
// over 65000 positions that never left it would be 2e-4 off.
//
// Positions that no row of the tile sees are zeros in shared memory, whatever the cache holds there.  Where a value that some
// rows see and others do not is an infinity or a NaN, the others' results are NaN (0 times it); results that are not finite
// are done again by attend_row, which reads only what the row sees.
#include "attn_kv.cuh"

#include <algorithm>

namespace ab {

// ---- few rows: 16 per tile -------------------------------------------------------------------------------------------
// Every warp has chunks of 16 positions of its own (chunk w, w + W, ..), the next ones under way in STAGES slots of
// shared memory, and its own running maxima, sums and outputs; nothing in the loop waits for another warp.  The warps, then the
// CTAs that share the tile, merge at the end.  Bound by HBM: the tensor cores are busy for a few percent.
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

// 16-byte words of 16-bit rows, so that eight neighbouring rows of one column lie in different banks
template <int HD>
__device__ __forceinline__ int swz(int r, int ch) { return HD >= 64 ? ch ^ (r & 7) : ch ^ ((r >> 1) & 3); }

template <typename T, int HD>
__global__ void __launch_bounds__(Few<T, HD>::W * 32) k_attn_few(const __grid_constant__ AttnArgs a) {
    using F = Few<T, HD>;
    constexpr int ROWS = F::ROWS, CB = F::CB, W = F::W, LD = F::LD, STAGES = F::STAGES;
    constexpr bool H = sizeof(T) == 2;
    extern __shared__ __align__(128) uint8_t sm[];
    __shared__ AttnRow s_row[ROWS];
    __shared__ float s_unit[ROWS], s_m[W][ROWS], s_l[W][ROWS];
    __shared__ uint32_t s_scratch[W + 2];
    __shared__ uint32_t s_bad;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, q4 = lane & 3;
    const uint32_t kvh = blockIdx.y, split = blockIdx.x % a.splits, t = blockIdx.x / a.splits;
    AttnTile x;
    if (!find_tile<ROWS, CB>(a, t, kvh, x, s_row, s_scratch)) return;
    // this CTA's chunks
    const uint32_t each = max((x.chunks + a.splits - 1) / a.splits, a.least), sharers = (x.chunks + each - 1) / each;
    if (split >= sharers) return;
    const uint32_t c0 = split * each, c1 = min(x.chunks, c0 + each);
    if (tid == 0) s_bad = 0;

    uint8_t* const sq = sm;                              // the queries
    uint8_t* const ring = sm + F::Q_BYTES + warp * STAGES * F::SLOT;
    const uint32_t ring_s = at_smem(ring);
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
    // queries: fp16 terms of the row times a power of two, or floats; a warp takes every fourth row
    for (int r = warp; r < ROWS; r += W) {
        const AttnRow row = s_row[r];
        float v[HD / 32], most = 0.f;
#pragma unroll
        for (int j = 0; j < HD / 32; ++j) { v[j] = row.pos >= 0 ? a.act[row.q + lane + 32 * j] : 0.f; most = fmaxf(most, fabsf(v[j])); }
        float up = 1.f, down = 1.f;
        if (H) row_scale(warp_max(most), up, down);
        if (lane == 0) s_unit[r] = down;
#pragma unroll
        for (int j = 0; j < HD / 32; ++j) {
            const int d = lane + 32 * j;
            if constexpr (H) {
                const float y = v[j] * up;
                const __half hi = __float2half_rn(y);
                __half* p = reinterpret_cast<__half*>(sq) + r * HD + swz<HD>(r, d >> 3) * 8 + (d & 7);
                p[0] = hi; p[ROWS * HD] = __float2half_rn(y - __half2float(hi));
            } else reinterpret_cast<float*>(sq)[r * LD + d] = v[j];
        }
    }
    __syncthreads();

    const uint32_t sq_s = at_smem(sq);
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
        const uint32_t k_s = ring_s + slot * F::SLOT, v_s = k_s + F::SLOT / 2;
        const float *kf = reinterpret_cast<const float*>(ring + slot * F::SLOT), *vf = kf + CB * LD;
        request(slot ? slot - 1 : STAGES - 1);           // the slot that the chunk before this one has left
        const int32_t p0 = chunk_at<CB>(x, c);
        float s[2][4] = {};                              // scores: positions p0 + 8 n + 2 q4 + (e & 1), rows g + 8 (e >> 1)
        if constexpr (H) {
#pragma unroll 4
            for (int k = 0; k < HD / 16; ++k) {
                uint32_t qh[4], ql[4], b[4];
                const int qr = lane & 15, qc = 2 * k + (lane >> 4), kr = (lane >> 4) * 8 + (lane & 7), kc = 2 * k + ((lane >> 3) & 1);
                const uint32_t qo = (uint32_t)(qr * HD + swz<HD>(qr, qc) * 8) * 2u;
                at_ldsm(sq_s + qo, qh);
                at_ldsm(sq_s + ROWS * HD * 2 + qo, ql);
                at_ldsm(k_s + (uint32_t)(kr * HD + swz<HD>(kr, kc) * 8) * 2u, b);
                at_mma_h(s[0], ql, b[0], b[1]); at_mma_h(s[1], ql, b[2], b[3]);
                at_mma_h(s[0], qh, b[0], b[1]); at_mma_h(s[1], qh, b[2], b[3]);
            }
        } else {
#pragma unroll 4
            for (int k = 0; k < HD; k += 8) {
                const float* qp = reinterpret_cast<const float*>(sq) + g * LD + k + q4;
                uint32_t ah[4], al[4];
                at_split_t(qp[0], ah[0], al[0]); at_split_t(qp[8 * LD], ah[1], al[1]);
                at_split_t(qp[4], ah[2], al[2]); at_split_t(qp[8 * LD + 4], ah[3], al[3]);
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    const float* kp = kf + (n * 8 + g) * LD + k + q4;
                    uint32_t b0h, b0l, b1h, b1l;
                    at_split_t(kp[0], b0h, b0l); at_split_t(kp[4], b1h, b1l);
                    at_mma_t(s[n], al, b0h, b1h); at_mma_t(s[n], ah, b0l, b1l); at_mma_t(s[n], ah, b0h, b1h);
                }
            }
        }
        // weights: running maximum and sum of each row over its quad of lanes
        const bool all = tile_sees(a, x, p0, CB);
        float alpha[2];
        const float rcap = a.cap > 0.f ? __frcp_rn(a.cap) : 0.f;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float mx = -INFINITY;
#pragma unroll
            for (int n = 0; n < 2; ++n)
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
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int e = 2 * h; e < 2 * h + 2; ++e) { s[n][e] = expf(s[n][e] - ref); sum += s[n][e]; }
            l[h] = fmaf(l[h], alpha[h], sum);
        }
        if constexpr (H) {
            uint32_t ph[4], pl[4];                       // times 256: the low terms stay clear of the fp16 subnormals
#pragma unroll
            for (int f = 0; f < 4; ++f) {
                const float* p = &s[f >> 1][2 * (f & 1)];
                at_split_h(p[0] * 256.f, p[1] * 256.f, ph[f], pl[f]);
            }
            constexpr int DC = HD >= 64 ? 64 : HD;
#pragma unroll
            for (int d0 = 0; d0 < HD; d0 += DC) {
                float acc[DC / 8][4] = {};
#pragma unroll
                for (int n = 0; n < DC / 16; ++n) {
                    uint32_t b[4];
                    const int vr = ((lane >> 3) & 1) * 8 + (lane & 7), vc = d0 / 8 + 2 * n + (lane >> 4);
                    at_ldsm_t(v_s + (uint32_t)(vr * HD + swz<HD>(vr, vc) * 8) * 2u, b);
                    at_mma_h(acc[2 * n], pl, b[0], b[1]); at_mma_h(acc[2 * n + 1], pl, b[2], b[3]);
                    at_mma_h(acc[2 * n], ph, b[0], b[1]); at_mma_h(acc[2 * n + 1], ph, b[2], b[3]);
                }
#pragma unroll
                for (int j = 0; j < DC / 8; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[d0 / 8 + j][e] = fmaf(o[d0 / 8 + j][e], alpha[e >> 1], acc[j][e]);
            }
        } else {
            // the order of the positions inside a step of 8 is free: slots t and t + 4 are positions 2 t and 2 t + 1, which is
            // how the scores lie in the registers
            uint32_t ph[2][4], pl[2][4];
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                at_split_t(s[n][0], ph[n][0], pl[n][0]); at_split_t(s[n][2], ph[n][1], pl[n][1]);
                at_split_t(s[n][1], ph[n][2], pl[n][2]); at_split_t(s[n][3], ph[n][3], pl[n][3]);
            }
#pragma unroll
            for (int j = 0; j < HD / 8; ++j) {
                float acc[4] = {};
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    const float* vp = vf + (n * 8 + 2 * q4) * LD + j * 8 + g;
                    uint32_t b0h, b0l, b1h, b1l;
                    at_split_t(vp[0], b0h, b0l); at_split_t(vp[LD], b1h, b1l);
                    at_mma_t(acc, pl[n], b0h, b1h); at_mma_t(acc, ph[n], b0l, b1l); at_mma_t(acc, ph[n], b0h, b1h);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) o[j][e] = fmaf(o[j][e], alpha[e >> 1], acc[e]);
            }
        }
        slot = slot + 1 == STAGES ? 0 : slot + 1;
    }
    at_wait<0>();

    // ---- the warps' results ----
    constexpr float UNIT = H ? 1.f / 256.f : 1.f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
        if (q4 == 0) { s_m[warp][g + 8 * h] = m[h]; s_l[warp][g + 8 * h] = l[h]; }
    }
    __syncthreads();
    float* const merge = reinterpret_cast<float*>(sm + F::Q_BYTES);       // [warp][row][HD + 4]
    float best[2], sum[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        best[h] = -INFINITY; sum[h] = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) best[h] = max_nan(best[h], s_m[w][g + 8 * h]);
        const float ref = best[h] == -INFINITY ? 0.f : best[h];
#pragma unroll
        for (int w = 0; w < W; ++w) sum[h] += s_l[w][g + 8 * h] * expf(s_m[w][g + 8 * h] - ref);
        const float f = expf(m[h] - ref) * UNIT;
#pragma unroll
        for (int j = 0; j < HD / 8; ++j)
            *reinterpret_cast<float2*>(merge + (warp * ROWS + g + 8 * h) * (HD + 4) + 8 * j + 2 * q4) = make_float2(o[j][2 * h] * f, o[j][2 * h + 1] * f);
    }
    __syncthreads();
    if (warp == 0 && q4 == 0)
#pragma unroll
        for (int h = 0; h < 2; ++h) { s_m[0][g + 8 * h] = best[h]; s_l[0][g + 8 * h] = sum[h]; }
    __syncthreads();
    const uint32_t live = min((uint32_t)ROWS, x.n * a.group - x.first);
    auto value = [&](uint32_t r, uint32_t d) {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) v += merge[(w * ROWS + r) * (HD + 4) + d];
        return v;
    };
    if (sharers > 1) {
        // a partial result per CTA; the last one to arrive adds them up in their order
        const size_t tile = (size_t)t * a.geo.n_kv + kvh;
        float* mine = a.part + (tile * a.splits + split) * ROWS * (HD + 2);
        for (uint32_t i = tid; i < live * HD; i += W * 32) mine[ROWS * 2 + i] = value(i / HD, i % HD);
        if (tid < (int)live) { mine[2 * tid] = s_m[0][tid]; mine[2 * tid + 1] = s_l[0][tid]; }
        __threadfence();
        __syncthreads();
        if (tid == 0) s_scratch[0] = atomicInc(a.tickets + tile, sharers - 1);
        __syncthreads();
        if (s_scratch[0] != sharers - 1) return;
        __threadfence();
        const float* all = a.part + tile * a.splits * ROWS * (HD + 2);
        const size_t step = (size_t)ROWS * (HD + 2);
        if (tid < (int)live) {
            float b = -INFINITY, z = 0.f;
            for (uint32_t k = 0; k < sharers; ++k) b = max_nan(b, __ldcg(all + k * step + 2 * tid));
            const float ref = b == -INFINITY ? 0.f : b;
            for (uint32_t k = 0; k < sharers; ++k) z += __ldcg(all + k * step + 2 * tid + 1) * expf(__ldcg(all + k * step + 2 * tid) - ref);
            s_m[0][tid] = ref; s_l[0][tid] = z;
        }
        __syncthreads();
        for (uint32_t i = tid; i < live * HD; i += W * 32) {
            const uint32_t r = i / HD;
            float v = 0.f;
#pragma unroll 8
            for (uint32_t k = 0; k < sharers; ++k) v = fmaf(__ldcg(all + k * step + ROWS * 2 + i), expf(__ldcg(all + k * step + 2 * r) - s_m[0][r]), v);
            merge[r * (HD + 4) + i % HD] = v;
        }
        __syncthreads();
    }
    // ---- out; rows that are not finite once more, by themselves ----
    for (uint32_t i = tid; i < live * HD; i += W * 32) {
        const uint32_t r = i / HD, d = i % HD;
        const float v = (sharers > 1 ? merge[r * (HD + 4) + d] : value(r, d)) / s_l[0][r];
        if (s_row[r].pos < 0) continue;
        if (!(fabsf(v) <= 3.402823466e+38f)) atomicOr(&s_bad, 1u << r);
        merge[r * (HD + 4) + d] = v;
    }
    __syncthreads();
    const uint32_t bad = s_bad;
    for (uint32_t i = tid; i < live * HD; i += W * 32) {
        const uint32_t r = i / HD, d = i % HD;
        if (s_row[r].pos >= 0 && !(bad >> r & 1u)) a.act[s_row[r].o + d] = merge[r * (HD + 4) + d];
    }
    if (bad)
        for (uint32_t r = warp; r < live; r += W)
            if (bad >> r & 1u) attend_row<T, HD>(a, x, s_row[r], kvh);
}

template <typename T, int HD>
static int launch_few(AttnArgs& a, uint32_t tiles) {
    using F = Few<T, HD>;
    static bool set = false;
    if (!set) {
        if (cudaFuncSetAttribute((const void*)k_attn_few<T, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, F::SMEM) != cudaSuccess)
            return fail(ADAMAH_ERR_BACKEND, "attn_kv: cannot raise the shared-memory limit");
        set = true;
    }
    k_attn_few<T, HD><<<dim3(tiles * a.splits, a.geo.n_kv), F::W * 32, F::SMEM, g.stream>>>(a);
    return ADAMAH_OK;
}
template <typename T>
static int launch_hd(AttnArgs& a, uint32_t tiles) {
    switch (a.geo.hd) {
    case 32: return launch_few<T, 32>(a, tiles);
    case 64: return launch_few<T, 64>(a, tiles);
    case 128: return launch_few<T, 128>(a, tiles);
    default: return launch_few<T, 256>(a, tiles);
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
    a.window = window > 0x7FFFFFFFu ? 0u : window; a.n_sink = n_sink; a.scale = scale; a.cap = cap; a.err = g.dev_err;
    a.part = kv->part; a.tickets = kv->tickets;
    // Tiles: every entry has its rows * group / 16 and at most 15 / 16 more.
    const uint64_t flat = (uint64_t)n_rows * a.group, tiles64 = (flat + 15ull * std::min(n_seqs, n_rows)) / 16;
    if (tiles64 * a.geo.n_kv >= (1u << 30)) return fail(ADAMAH_ERR_INVALID, "attn_kv: %u rows of %u heads", n_rows, n_head);
    const uint32_t tiles = (uint32_t)tiles64, ctas = tiles * a.geo.n_kv;
    // Splits: as many CTAs as the GPU holds twice over, no more than the workspace has room for.  How far the sequences reach
    // only decides the launch; a graph that is replayed later divides what there is then.
    uint32_t reach = kv->pages.longest();
    if (a.window) reach = (uint32_t)std::min<uint64_t>(reach, (uint64_t)a.window + n_sink);
    a.least = 8;
    a.splits = std::max(1u, std::min({(uint32_t)g.sm_count * 2 / ctas, KV_SPLIT_CTAS / ctas, (reach + 127) / 128}));
    const int rc0 = kv->elem == 2 ? launch_hd<__half>(a, tiles) : launch_hd<float>(a, tiles);
    if (rc0) return rc0;
    count_launch();
    const int rc = check_launch("map_attn_kv");
    end_of_op();
    return rc;
}
