// Norm and rotation of the new rows' queries and keys, append of keys and values to a paged cache, in one pass over the
// rows (map_qk_norm_rope_x.comp and map_row_copy.comp, which know one position and a contiguous cache).
//
//   y = x / sqrt(mean(x^2) + eps) * w          per head
//   (y_i, y_{i + h}) -> (y_i c_i - y_{i + h} s_i, y_i s_i + y_{i + h} c_i),   c_i, s_i = cos, sin(p base^(-i / h)),   h = head_dim / 2
//
// The angle of a far position has more digits than 32 bits hold (position 30000: 1e-3 off), so the turns p base^(-i / h) / 2 pi are
// formed in 64 bits; what is left of them after the whole turns, at most a half, is a 32-bit number whose sine and cosine
// are as good as any 32-bit ones.
#include "kv_cache.cuh"

namespace ab {

constexpr int AP_T = 256;

struct AppendArgs {
    float* act; uint64_t n_act; const float* wt; uint64_t n_wt;
    const uint32_t *l_q, *l_k, *l_v, *l_qw, *l_kw, *l_dst;
    KvBatch b; KvGeom geo; void* pool;
    uint32_t layer, n_head;
    double log2_base; float eps;
    uint32_t* err;
};

// The entry that holds row r, by all threads of the CTA; -1 = none.  `slot` is shared.
__device__ __forceinline__ int find_entry(const KvBatch& b, uint32_t r, int* slot) {
    if (threadIdx.x == 0) *slot = -1;
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < b.n_seqs; e += blockDim.x)
        if (b.start[e] <= r && r < b.start[e + 1] && b.start[e + 1] - b.start[e] <= b.n_rows) *slot = (int)e;
    __syncthreads();
    const int e = *slot;
    __syncthreads();
    return e;
}

// N neighbouring values of a row, at once where they are aligned
template <int N>
__device__ __forceinline__ void ld_vals(const float* p, bool vec, float (&x)[N]) {
    if constexpr (N == 4) { if (vec) { const float4 v = *reinterpret_cast<const float4*>(p); x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w; return; } }
    if constexpr (N == 2) { if (vec) { const float2 v = *reinterpret_cast<const float2*>(p); x[0] = v.x; x[1] = v.y; return; } }
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = p[i];
}
template <int N>
__device__ __forceinline__ void st_vals(float* p, bool vec, const float (&x)[N]) {
    if constexpr (N == 4) { if (vec) { *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]); return; } }
    if constexpr (N == 2) { if (vec) { *reinterpret_cast<float2*>(p) = make_float2(x[0], x[1]); return; } }
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = x[i];
}
template <int N>
__device__ __forceinline__ void st_vals(__half* p, bool, const float (&x)[N]) {        // always aligned: a cache row
    KvRow<__half, N> row;
    row.from_float(x);
    row.store(p);
}

// A CTA per row at a time; its warps take the row's heads.  Lane l has the dims N l .. of both halves.
template <typename T, int HD>
__global__ void __launch_bounds__(AP_T) k_kv_append(const AppendArgs a) {
    constexpr int HALF = HD / 2, N = HALF >= 32 ? HALF / 32 : 1, W = AP_T / 32, U = N == 4 ? 2 : 4;
    __shared__ __align__(16) float s_cos[HALF], s_sin[HALF];
    __shared__ int s_entry;
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t n_kv = a.geo.n_kv, heads = a.n_head + 2 * n_kv, i0 = lane * N;
    const bool on = i0 < HALF;
    // turns per position of this thread's angle
    const double turn = threadIdx.x < HALF ? exp2(-(double)threadIdx.x / HALF * a.log2_base) * 0.15915494309189533577 : 0.0;
    for (uint32_t r = blockIdx.x; r < a.b.n_rows; r += gridDim.x) {
        const int e = find_entry(a.b, r, &s_entry);
        if (e < 0) continue;
        const uint32_t seq = a.b.seq[e], first = a.b.start[e], n = a.b.start[e + 1] - first;
        if (seq == KV_NO_SEQ) continue;
        int32_t pos = -1, page = -1;
        if (seq < a.b.max_seqs) {
            pos = a.b.lens[seq] - (int32_t)n + (int32_t)(r - first);
            const uint32_t pn = (uint32_t)pos / a.geo.page;
            if (pos >= a.b.own_from[seq] && pn < a.geo.max_pages) page = a.b.table[(size_t)seq * a.geo.max_pages + pn];
        }
        const uint64_t oq = a.l_q[r], ok = a.l_k[r], ov = a.l_v[r], od = a.l_dst[r], oqw = a.l_qw ? a.l_qw[0] : 0, okw = a.l_kw ? a.l_kw[0] : 0;
        const uint64_t q_len = (uint64_t)a.n_head * HD, k_len = (uint64_t)n_kv * HD;
        if (page < 0 || oq + q_len > a.n_act || od + q_len > a.n_act || ok + k_len > a.n_act || ov + k_len > a.n_act ||
            (a.l_qw && oqw + HD > a.n_wt) || (a.l_kw && okw + HD > a.n_wt)) {
            if (threadIdx.x == 0) atomicOr(a.err, DEVERR_OOB_MAP);
            continue;
        }
        // U heads of a warp at a time: all their values are asked for before the first is used
        float x0[U][N], x1[U][N];
        auto ask = [&](uint32_t h0) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const uint32_t h = h0 + u * W;
                const bool is_q = h < a.n_head, is_v = h >= a.n_head + n_kv;
                const uint64_t at = is_q ? oq + (uint64_t)h * HD : (is_v ? ov : ok) + (uint64_t)(h - a.n_head - (is_v ? n_kv : 0)) * HD;
#pragma unroll
                for (int j = 0; j < N; ++j) { x0[u][j] = 0.f; x1[u][j] = 0.f; }
                if (on && h < heads) { ld_vals<N>(a.act + at + i0, at % N == 0, x0[u]); ld_vals<N>(a.act + at + i0 + HALF, at % N == 0, x1[u]); }
            }
        };
        ask(warp);
        if (threadIdx.x < HALF) {
            const double t = (double)pos * turn;
            sincospif(2.0f * (float)(t - rint(t)), &s_sin[threadIdx.x], &s_cos[threadIdx.x]);
        }
        __syncthreads();
        float c[N], s[N];
#pragma unroll
        for (int j = 0; j < N; ++j) { c[j] = on ? s_cos[i0 + j] : 0.f; s[j] = on ? s_sin[i0 + j] : 0.f; }
        T* const cache = reinterpret_cast<T*>(a.pool) + kv_index(a.geo, (uint32_t)page, a.layer, 0, 0, (uint32_t)pos % a.geo.page);
        const size_t head_step = (size_t)a.geo.page * HD, v_step = head_step * n_kv;
        float qw0[N] = {}, qw1[N] = {}, kw0[N] = {}, kw1[N] = {};
        if (on && a.l_qw) { ld_vals<N>(a.wt + oqw + i0, oqw % N == 0, qw0); ld_vals<N>(a.wt + oqw + i0 + HALF, oqw % N == 0, qw1); }
        if (on && a.l_kw) { ld_vals<N>(a.wt + okw + i0, okw % N == 0, kw0); ld_vals<N>(a.wt + okw + i0 + HALF, okw % N == 0, kw1); }
        for (uint32_t h0 = warp; h0 < heads; h0 += U * W) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const uint32_t h = h0 + u * W;
                if (h >= heads) break;
                const bool is_q = h < a.n_head, is_v = h >= a.n_head + n_kv;
                const uint32_t kh = is_v ? h - a.n_head - n_kv : h - a.n_head;
                if (is_v) {
                    T* dst = cache + v_step + kh * head_step + i0;
                    if (on) { st_vals<N>(dst, true, x0[u]); st_vals<N>(dst + HALF, true, x1[u]); }
                    continue;
                }
                if (is_q ? a.l_qw != nullptr : a.l_kw != nullptr) {
                    float ss = 0.f;
#pragma unroll
                    for (int j = 0; j < N; ++j) ss = fmaf(x0[u][j], x0[u][j], fmaf(x1[u][j], x1[u][j], ss));
                    const float rms = sqrtf(warp_sum(ss) * (1.0f / HD) + a.eps), rcp = __frcp_rn(rms);
                    // squares overflow long before values do: x / infinity is 0, where div_by, which multiplies by the divisor too, makes a NaN
                    const float d = rms <= 3.402823466e+38f ? rms : 0.f;
#pragma unroll
                    for (int j = 0; j < N; ++j) {
                        x0[u][j] = div_by(x0[u][j], d, rcp) * (is_q ? qw0[j] : kw0[j]);
                        x1[u][j] = div_by(x1[u][j], d, rcp) * (is_q ? qw1[j] : kw1[j]);
                    }
                }
                float y0[N], y1[N];
#pragma unroll
                for (int j = 0; j < N; ++j) { y0[j] = x0[u][j] * c[j] - x1[u][j] * s[j]; y1[j] = x0[u][j] * s[j] + x1[u][j] * c[j]; }
                if (!on) continue;
                if (is_q) {
                    const uint64_t d = od + (uint64_t)h * HD;
                    st_vals<N>(a.act + d + i0, d % N == 0, y0); st_vals<N>(a.act + d + i0 + HALF, d % N == 0, y1);
                } else {
                    T* dst = cache + kh * head_step + i0;
                    st_vals<N>(dst, true, y0); st_vals<N>(dst + HALF, true, y1);
                }
            }
            if (h0 + U * W < heads) ask(h0 + U * W);
        }
    }
}

template <typename T>
static void launch_append_t(const AppendArgs& a) {
    const dim3 grid(std::min<uint32_t>(a.b.n_rows, (uint32_t)g.sm_count * 8));
    switch (a.geo.hd) {
    case 32: k_kv_append<T, 32><<<grid, AP_T, 0, g.stream>>>(a); break;
    case 64: k_kv_append<T, 64><<<grid, AP_T, 0, g.stream>>>(a); break;
    case 128: k_kv_append<T, 128><<<grid, AP_T, 0, g.stream>>>(a); break;
    default: k_kv_append<T, 256><<<grid, AP_T, 0, g.stream>>>(a);
    }
}

// What both operators ask of a batch.
int kv_batch(const char* name, uint32_t kv_id, uint32_t layer, uint32_t seq_h, uint32_t start_h, uint32_t n_seqs, uint32_t n_rows, uint32_t n_head,
             KvCache** kv_out, KvBatch* b) {
    KvCache* kv = *kv_out = get_kv(kv_id);
    if (!kv) return ADAMAH_ERR_NOT_FOUND;
    if (layer >= kv->d.n_layer) return fail(ADAMAH_ERR_INVALID, "%s: layer %u of %u", name, layer, kv->d.n_layer);
    if (!n_head || n_head % kv->d.n_head_kv || n_head > 65535) return fail(ADAMAH_ERR_INVALID, "%s: %u query heads over %u key heads", name, n_head, kv->d.n_head_kv);
    if (n_seqs > kv->d.max_seqs) return fail(ADAMAH_ERR_INVALID, "%s: %u sequences of a cache for %u", name, n_seqs, kv->d.max_seqs);
    if (n_rows > (1u << 24)) return fail(ADAMAH_ERR_INVALID, "%s: %u rows", name, n_rows);
    if (!handle_ok(seq_h, n_seqs * 4) || !handle_ok(start_h, (n_seqs + 1) * 4)) return ADAMAH_ERR_NOT_FOUND;
    *b = KvBatch{hlocs(seq_h), hlocs(start_h), n_seqs, n_rows, kv->lens, kv->own_from, kv->table, kv->d.max_seqs};
    return ADAMAH_OK;
}

}  // namespace ab

using namespace ab;

extern "C" int map_qk_norm_rope_kv_dev(uint32_t map_act, uint32_t map_wt, uint32_t kv_id, uint32_t layer, uint32_t q_h, uint32_t k_h, uint32_t v_h,
                                       uint32_t qwt_h, uint32_t kwt_h, uint32_t qdst_h, uint32_t seq_h, uint32_t start_h, uint32_t n_seqs,
                                       uint32_t n_rows, uint32_t n_head, float freq_base, float eps) {
    if (!ready()) return ADAMAH_ERR_INVALID;
    Map *m = get_map(map_act), *w = get_map(map_wt);
    if (!m || !w) return ADAMAH_ERR_NOT_FOUND;
    for (const Map* x : {m, w})
        if (x->dtype != ADAMAH_DTYPE_F32 || x->pack_size != 1) return fail(ADAMAH_ERR_INVALID, "qk_norm_rope_kv: maps must be float32 with pack_size 1");
    KvCache* kv;
    AppendArgs a = {};
    if (int rc = kv_batch("qk_norm_rope_kv", kv_id, layer, seq_h, start_h, n_seqs, n_rows, n_head, &kv, &a.b)) return rc;
    if (!(freq_base > 0.f) || !(freq_base < 3.0e38f) || !(eps >= 0.f)) return fail(ADAMAH_ERR_INVALID, "qk_norm_rope_kv: freq_base %g, eps %g", freq_base, eps);
    for (uint32_t h : {q_h, k_h, v_h, qdst_h}) if (!handle_ok(h, n_rows * 4)) return ADAMAH_ERR_NOT_FOUND;
    for (uint32_t h : {qwt_h, kwt_h}) if (h && !handle_ok(h, 4)) return ADAMAH_ERR_NOT_FOUND;
    if (!n_rows || !n_seqs) return ADAMAH_OK;
    a.act = (float*)m->buf; a.n_act = m->n_elems; a.wt = (const float*)w->buf; a.n_wt = w->n_elems;
    a.l_q = hlocs(q_h); a.l_k = hlocs(k_h); a.l_v = hlocs(v_h); a.l_dst = hlocs(qdst_h);
    a.l_qw = qwt_h ? hlocs(qwt_h) : nullptr; a.l_kw = kwt_h ? hlocs(kwt_h) : nullptr;
    a.geo = kv->geo; a.pool = kv->pool; a.layer = layer; a.n_head = n_head; a.eps = eps; a.err = g.dev_err;
    a.log2_base = log2((double)freq_base);
    if (kv->elem == 2) launch_append_t<__half>(a);
    else launch_append_t<float>(a);
    count_launch();
    const int rc = check_launch("map_qk_norm_rope_kv");
    end_of_op();
    return rc;
}
