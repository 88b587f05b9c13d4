// Attention of new rows over a paged cache: a token per sequence or a chunk of a prompt, a sliding window and first
// positions that stay visible (map_matmul_t.comp + map_attn_softmax_value.comp over a contiguous cache, a row at a time).
//
//   s_j = scale q.k_j, or cap tanh(scale q.k_j / cap);   o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),   j visible to the row
#include "kv_cache.cuh"

namespace ab {

struct AttnArgs {
    float* act; uint64_t n_act;
    const uint32_t *l_q, *l_out;
    KvBatch b; KvGeom geo; const void* pool;
    uint32_t layer, n_head, window, n_sink;
    float scale, cap;
    uint32_t* err;
};

__device__ __forceinline__ float capped(float s, const AttnArgs& a) { return a.cap > 0.f ? a.cap * tanhf(s / a.cap) : s; }

// One query head of one row by a warp: running maximum and sum, only positions that the row sees are read.
template <typename T, int HD>
__device__ void attend_row(const AttnArgs& a, uint32_t seq, int32_t pos, uint32_t head, uint64_t oq, uint64_t oo) {
    constexpr int N = HD / 32;
    const uint32_t lane = threadIdx.x & 31, kvh = head / (a.n_head / a.geo.n_kv);
    const int32_t* pages = a.b.table + (size_t)seq * a.geo.max_pages;
    float q[N], o[N] = {}, m = -INFINITY, l = 0.f;
#pragma unroll
    for (int j = 0; j < N; ++j) q[j] = a.act[oq + (uint64_t)head * HD + lane * N + j];
    const int32_t from = a.window && (uint32_t)pos >= a.window ? pos - (int32_t)a.window + 1 : 0;
    for (int32_t t = 0; t <= pos; ++t) {
        if (t < from && (uint32_t)t >= a.n_sink) t = from;
        const int32_t page = pages[(uint32_t)t / a.geo.page];
        if (page < 0) { if (lane == 0) atomicOr(a.err, DEVERR_OOB_MAP); continue; }
        const T* row = reinterpret_cast<const T*>(a.pool) + kv_index(a.geo, (uint32_t)page, a.layer, 0, kvh, (uint32_t)t % a.geo.page);
        KvRow<T, N> k, v;
        k.load(row + lane * N);
        v.load(row + (size_t)a.geo.n_kv * a.geo.page * HD + lane * N);
        float x[N], s = 0.f;
        k.to_float(x);
#pragma unroll
        for (int j = 0; j < N; ++j) s = fmaf(q[j], x[j], s);
        s = capped(warp_sum(s) * a.scale, a);
        const float mn = fmaxf(m, s), alpha = m == mn ? 1.f : expf(m - mn), p = expf(s - mn);
        v.to_float(x);
        l = l * alpha + p;
        m = mn;
#pragma unroll
        for (int j = 0; j < N; ++j) o[j] = fmaf(p, x[j], o[j] * alpha);
    }
#pragma unroll
    for (int j = 0; j < N; ++j) a.act[oo + (uint64_t)head * HD + lane * N + j] = o[j] / l;
}

template <typename T, int HD>
__global__ void __launch_bounds__(256) k_attn_rows(const AttnArgs a) {
    __shared__ int s_entry;
    const uint32_t r = blockIdx.x;
    if (threadIdx.x == 0) s_entry = -1;
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < a.b.n_seqs; e += blockDim.x)
        if (a.b.start[e] <= r && r < a.b.start[e + 1] && a.b.start[e + 1] - a.b.start[e] <= a.b.n_rows) s_entry = (int)e;
    __syncthreads();
    if (s_entry < 0) return;
    const uint32_t e = (uint32_t)s_entry, seq = a.b.seq[e], first = a.b.start[e], n = a.b.start[e + 1] - first;
    if (seq == KV_NO_SEQ) return;
    const int32_t pos = seq < a.b.max_seqs ? a.b.lens[seq] - (int32_t)n + (int32_t)(r - first) : -1;
    const uint64_t oq = a.l_q[r], oo = a.l_out[r], len = (uint64_t)a.n_head * HD;
    if (pos < 0 || oq + len > a.n_act || oo + len > a.n_act) { if (threadIdx.x == 0) atomicOr(a.err, DEVERR_OOB_MAP); return; }
    for (uint32_t h = threadIdx.x >> 5; h < a.n_head; h += 8) attend_row<T, HD>(a, seq, pos, h, oq, oo);
}

template <typename T>
static void launch_rows(const AttnArgs& a) {
    switch (a.geo.hd) {
    case 32: k_attn_rows<T, 32><<<a.b.n_rows, 256, 0, g.stream>>>(a); break;
    case 64: k_attn_rows<T, 64><<<a.b.n_rows, 256, 0, g.stream>>>(a); break;
    case 128: k_attn_rows<T, 128><<<a.b.n_rows, 256, 0, g.stream>>>(a); break;
    default: k_attn_rows<T, 256><<<a.b.n_rows, 256, 0, g.stream>>>(a);
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
    a.geo = kv->geo; a.pool = kv->pool; a.layer = layer; a.n_head = n_head;
    a.window = window > 0x7FFFFFFFu ? 0u : window; a.n_sink = n_sink; a.scale = scale; a.cap = cap; a.err = g.dev_err;
    if (kv->elem == 2) launch_rows<__half>(a);
    else launch_rows<float>(a);
    count_launch();
    const int rc = check_launch("map_attn_kv");
    end_of_op();
    return rc;
}
