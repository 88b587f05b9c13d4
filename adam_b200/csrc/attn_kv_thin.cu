// Attention of two or four rows over a paged cache: a token's query heads of one key head, decoding (see attn_kv.cu for the operator).
//
// Nothing is padded to a matrix instruction's rows and nothing is rounded: products and sums are 32-bit, two to an instruction.
// A position's key lies over LP lanes, 16 bytes to a lane, so a warp has 32 / LP positions side by side and CH in a chunk; a
// lane copies its own words to shared memory ahead of their use and is the only one to read them, so nothing in the loop waits
// for another warp.  The partial dot products of a chunk's positions and rows, NB to a lane, are added over the LP lanes by halving:
// at every step a lane gives away half of what it has, so 15 shuffles do for 16 sums, and each score (its tanh, its power) is
// then computed once.  Weights go to the lanes that hold the values through shared memory.  A running maximum changes a few times in a
// sequence; only then the outputs are rescaled.  Bound by HBM: 360 instructions for 16 positions of two rows (heads of 128, fp16), a
// third of what the tiles of 16 rows took with their two fp16 terms.
#include "attn_kv.cuh"

namespace ab {

template <typename T, int HD, int R>
struct Thin {
    static constexpr int ROW_BYTES = HD * (int)sizeof(T), E = 16 / (int)sizeof(T);
    static constexpr int LP = ROW_BYTES / 16 < 32 ? ROW_BYTES / 16 : 32, WORDS = ROW_BYTES / 16 / LP, PP = 32 / LP;
    static constexpr int CH = ROW_BYTES >= 256 ? 4096 / ROW_BYTES : 16, B = CH / PP;       // positions of a chunk, of a lane
    static constexpr int NB = B * R, V = NB > LP ? NB / LP : 1, DUP = LP > NB ? LP / NB : 1;
    static constexpr int W = 4, STAGES = ROW_BYTES >= 256 ? 2 : ROW_BYTES == 128 ? 3 : 4;
    static constexpr int SLOT = 2 * CH * ROW_BYTES;                               // keys and values of a chunk
    static constexpr int RING = W * STAGES * SLOT, MERGE = W * R * (HD + 4) * 4, SMEM = RING > MERGE ? RING : MERGE;
};

// 16 bytes of the cache as pairs of floats
__device__ __forceinline__ void thin_pairs(const uint4& w, float2 (&v)[4], __half*) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
}
__device__ __forceinline__ void thin_pairs(const uint4& w, float2 (&v)[2], float*) {
    v[0] = make_float2(__uint_as_float(w.x), __uint_as_float(w.y)); v[1] = make_float2(__uint_as_float(w.z), __uint_as_float(w.w));
}

// N sums over 2 D lanes: s[0 ..] of lane li are then those from li / DUP * V on
template <int N, int D, int M>
__device__ __forceinline__ void thin_sums(float (&s)[M], int li) {
    if constexpr (D > 0) {
        if constexpr (N > 1) {
            const bool up = li & D;
#pragma unroll
            for (int i = 0; i < N / 2; ++i) {
                const float give = up ? s[i] : s[i + N / 2], keep = up ? s[i + N / 2] : s[i];
                s[i] = keep + __shfl_xor_sync(0xffffffffu, give, D);
            }
            thin_sums<N / 2, D / 2>(s, li);
        } else {
            s[0] += __shfl_xor_sync(0xffffffffu, s[0], D);
            thin_sums<1, D / 2>(s, li);
        }
    }
}

// CLUSTER: a tile's CTAs are a cluster
template <typename T, int HD, int R, bool CLUSTER>
__global__ void __launch_bounds__(128, THIN_CTAS) k_attn_thin(const __grid_constant__ AttnArgs a) {
    using F = Thin<T, HD, R>;
    constexpr int LP = F::LP, WORDS = F::WORDS, PP = F::PP, CH = F::CH, B = F::B, NB = F::NB, V = F::V, DUP = F::DUP, W = F::W, STAGES = F::STAGES, E = F::E;
    extern __shared__ __align__(128) uint8_t sm[];
    __shared__ AttnRow s_row[R];
    __shared__ Found s_found;
    __shared__ End<R, W> s_end;
    __shared__ __align__(16) float s_p[W][CH * R];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, li = lane % LP, grp = lane / LP;
    const AttnShare part = share_of(a);
    const uint32_t kvh = part.kvh;
    AttnTile x;
    if (!find_tile<R, CH>(a, part.tile, kvh, x, s_row, s_found)) return;
    uint32_t sharers, c0, c1;
    if (!share_out(a, x, part, sharers, c0, c1) && !CLUSTER) return;         // in a cluster it still takes its rows
    c0 = min(c0, c1);

    uint8_t* const ring = sm + warp * STAGES * F::SLOT;
    const uint32_t ring_s = at_smem(ring) + lane * 16;
    const T* const pool = reinterpret_cast<const T*>(a.pool) + li * E;
    const size_t v_off = (size_t)a.geo.n_kv * a.geo.page * HD;
    // Chunks of this warp: c0 + warp, + W, ...; a chunk lies in one page, looked up before it is asked for
    uint32_t ask = c0 + warp;
    auto locate = [&]() -> int32_t { return ask < c1 ? x.pages[(uint32_t)chunk_at<CH>(x, ask) / a.geo.page] : -1; };
    int32_t page = locate();
    auto request = [&](int slot) {
        if (ask < c1) {
            const int32_t p0 = chunk_at<CH>(x, ask);
            const T* const from = page < 0 ? pool : pool + kv_index(a.geo, (uint32_t)page, a.layer, 0, kvh, (uint32_t)p0 % a.geo.page);
#pragma unroll
            for (int b = 0; b < B; ++b) {
                const int32_t p = p0 + b * PP + grp;
                const bool on = page >= 0 && p <= x.hi && (p >= x.from || (uint32_t)p < a.n_sink);
#pragma unroll
                for (int w = 0; w < WORDS; ++w) {
                    const T* const src = on ? from + (b * PP + grp) * HD + w * LP * E : pool;
                    const uint32_t dst = ring_s + slot * F::SLOT + (b * WORDS + w) * 512;
                    at_cp16(dst, src, on);
                    at_cp16(dst + F::SLOT / 2, on ? src + v_off : pool, on);
                }
            }
        }
        at_commit();
        ask += W;
        page = locate();
    };
#pragma unroll 1
    for (int i = 0; i < STAGES - 1; ++i) request(i);
    float2 q[R][WORDS * E / 2], o[R][WORDS * E / 2];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int w = 0; w < WORDS; ++w) {
            const bool on = s_row[r].pos >= 0;
            const float* const src = a.act + (on ? s_row[r].q + (w * LP + li) * E : 0);
            const bool fours = s_row[r].q % 4 == 0;
#pragma unroll
            for (int e = 0; e < E; e += 4) {
                float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
                if (on) y = fours ? *reinterpret_cast<const float4*>(src + e) : make_float4(src[e], src[e + 1], src[e + 2], src[e + 3]);
                q[r][(w * E + e) / 2] = make_float2(y.x, y.y); q[r][(w * E + e) / 2 + 1] = make_float2(y.z, y.w);
            }
        }
    float m[R], mine[V], l[V];                           // of the rows, of this lane's scores; this lane's sums
    int32_t pos[V];
    int row[V];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        m[r] = -INFINITY;
#pragma unroll
        for (int e = 0; e < WORDS * E / 2; ++e) o[r][e] = make_float2(0.f, 0.f);
    }
    const int i0 = li / DUP * V;                         // this lane's first score: position i0 / R of its B, row i0 % R
#pragma unroll
    for (int j = 0; j < V; ++j) { row[j] = (i0 + j) % R; pos[j] = s_row[row[j]].pos; mine[j] = -INFINITY; l[j] = 0.f; }
    const float k2 = a.cap > 0.f ? a.scale * __frcp_rn(a.cap) : a.scale * 1.4426950408889634f, cap2 = a.cap * 1.4426950408889634f;
    int slot = 0;
#pragma unroll 1
    for (uint32_t c = c0 + warp; c < c1; c += W) {
        request(slot ? slot - 1 : STAGES - 1);           // the slot that the chunk before this one has left
        at_wait<STAGES - 1>();
        const uint8_t* const at = ring + slot * F::SLOT + lane * 16;
        const int32_t p0 = chunk_at<CH>(x, c);
        float s[NB];
#pragma unroll
        for (int b = 0; b < B; ++b) {
            float2 sum[R];
#pragma unroll
            for (int w = 0; w < WORDS; ++w) {
                float2 k[E / 2];
                thin_pairs(*reinterpret_cast<const uint4*>(at + (b * WORDS + w) * 512), k, (T*)nullptr);
#pragma unroll
                for (int e = 0; e < E / 2; ++e)
#pragma unroll
                    for (int r = 0; r < R; ++r) sum[r] = w + e == 0 ? at_mul2(k[0], q[r][0]) : at_fma2(k[e], q[r][w * E / 2 + e], sum[r]);
            }
#pragma unroll
            for (int r = 0; r < R; ++r) s[b * R + r] = sum[r].x + sum[r].y;
        }
        thin_sums<NB, LP / 2>(s, li);
        bool more = false;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            s[j] = a.cap > 0.f ? cap2 * at_tanh(s[j] * k2) : s[j] * k2;
            if (!row_sees(a, pos[j], p0 + (i0 + j) / R * PP + grp)) s[j] = -INFINITY;
            more |= s[j] > mine[j];
        }
        if (__any_sync(0xffffffffu, more)) {
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float top = m[r];
#pragma unroll
                for (int j = 0; j < V; ++j) if (row[j] == r) top = fmaxf(top, s[j]);
#pragma unroll
                for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                const float alpha = top == -INFINITY ? 1.f : at_exp2(m[r] - top);
                m[r] = top;
#pragma unroll
                for (int e = 0; e < WORDS * E / 2; ++e) o[r][e] = at_mul2(o[r][e], make_float2(alpha, alpha));
#pragma unroll
                for (int j = 0; j < V; ++j) if (row[j] == r) { l[j] *= alpha; mine[j] = top; }
            }
        }
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float p = at_exp2(s[j] - (mine[j] == -INFINITY ? 0.f : mine[j]));
            l[j] += p;
            s_p[warp][grp * NB + i0 + j] = p;
        }
        __syncwarp();
#pragma unroll
        for (int b = 0; b < B; ++b) {
            float p[R];
            if constexpr (R == 2) { const float2 y = *reinterpret_cast<const float2*>(&s_p[warp][grp * NB + b * R]); p[0] = y.x; p[1] = y.y; }
            else { const float4 y = *reinterpret_cast<const float4*>(&s_p[warp][grp * NB + b * R]); p[0] = y.x; p[1] = y.y; p[2] = y.z; p[3] = y.w; }
#pragma unroll
            for (int w = 0; w < WORDS; ++w) {
                float2 v[E / 2];
                thin_pairs(*reinterpret_cast<const uint4*>(at + F::SLOT / 2 + (b * WORDS + w) * 512), v, (T*)nullptr);
#pragma unroll
                for (int e = 0; e < E / 2; ++e)
#pragma unroll
                    for (int r = 0; r < R; ++r) o[r][w * E / 2 + e] = at_fma2(v[e], make_float2(p[r], p[r]), o[r][w * E / 2 + e]);
            }
        }
        __syncwarp();
        slot = slot + 1 == STAGES ? 0 : slot + 1;
    }
    at_wait<0>();
#pragma unroll
    for (int r = 0; r < R; ++r) {
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j) if (row[j] == r && li % DUP == 0) sum += l[j];
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        if (lane == 0) { s_end.m[warp][r] = m[r]; s_end.l[warp][r] = sum; }
#pragma unroll
        for (int e = 0; e < WORDS * E / 2; ++e)
#pragma unroll
            for (int d = LP; d < 32; d <<= 1) {
                o[r][e].x += __shfl_xor_sync(0xffffffffu, o[r][e].x, d);
                o[r][e].y += __shfl_xor_sync(0xffffffffu, o[r][e].y, d);
            }
    }
    __syncthreads();                                     // nobody reads the ring any more
    float* const merge = reinterpret_cast<float*>(sm);
    if (grp == 0)
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const float f = s_end.template factor<true>(warp, r);
#pragma unroll
            for (int w = 0; w < WORDS; ++w)
#pragma unroll
                for (int e = 0; e < E / 2; ++e) {
                    const float2 y = o[r][w * E / 2 + e];
                    *reinterpret_cast<float2*>(merge + (warp * R + r) * (HD + 4) + (w * LP + li) * E + 2 * e) = make_float2(y.x * f, y.y * f);
                }
        }
    settle<T, HD, R, W, W * 32, true, CLUSTER>(a, x, s_row, part, sharers, merge, s_end);
}

template <typename T, int HD, int R, bool CLUSTER>
static int launch_one(const AttnArgs& a) {
    static bool set = false;
    return launch_attn(k_attn_thin<T, HD, R, CLUSTER>, set, a, 128, Thin<T, HD, R>::SMEM, CLUSTER);
}
template <typename T, int HD>
static int launch_rows(const AttnArgs& a, uint32_t rows) {
    if (rows == 2) return attn_cluster(a) ? launch_one<T, HD, 2, true>(a) : launch_one<T, HD, 2, false>(a);
    return attn_cluster(a) ? launch_one<T, HD, 4, true>(a) : launch_one<T, HD, 4, false>(a);
}
template <typename T>
static int launch_hd(const AttnArgs& a, uint32_t rows) {
    switch (a.geo.hd) {
    case 32: return launch_rows<T, 32>(a, rows);
    case 64: return launch_rows<T, 64>(a, rows);
    case 128: return launch_rows<T, 128>(a, rows);
    default: return launch_rows<T, 256>(a, rows);
    }
}
int launch_attn_thin(const AttnArgs& a, uint32_t elem, uint32_t rows) { return elem == 2 ? launch_hd<__half>(a, rows) : launch_hd<float>(a, rows); }
uint32_t attn_thin_chunk(uint32_t elem, uint32_t hd) { return elem * hd >= 256 ? 4096 / (elem * hd) : 16; }

}  // namespace ab
