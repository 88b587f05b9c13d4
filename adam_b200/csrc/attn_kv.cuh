// Attention over a paged cache: arguments and what the kernels of attn_kv.cu and attn_kv_tc.cu share.
#pragma once
#include "kv_cache.cuh"

namespace ab {

struct AttnArgs {
    float* act; uint64_t n_act;
    const uint32_t *l_q, *l_out;
    KvBatch b; KvGeom geo; const void* pool;
    uint32_t layer, n_head, group, window, n_sink;      // group: query heads of a key head
    float scale, cap;
    uint32_t pairs, whole, splits, least;               // (tile, key head)s; how many of them one CTA has alone; CTAs that may share
                                                        // the positions of each of the others; chunks that one takes at least
    float* part; unsigned int* tickets;
    uint32_t pool_rows;                                 // positions of all planes of the pool
    uint32_t* err;
};

// A row of a tile: an entry's rows times its group's heads, counted token by token, cut into tiles.
struct AttnRow { uint64_t q, o; int32_t pos; };         // offsets of the head's values; pos < 0: no such row

struct AttnTile {
    uint32_t seq, row, n, first;                        // sequence, its first row of the batch and how many, first (row, head) of the tile
    int32_t lo, hi;                                     // least and largest position of the tile's rows
    const int32_t* pages;
    uint32_t sinks, main0, chunks;                      // chunks of first positions, first chunk of the others, all together
    int32_t from;                                       // positions below it are seen by none but as first ones
};

// Tile t of the batch, by the whole CTA; false: there is none, or nothing to do.  Fills rows[0 .. ROWS).  CHUNK: positions per
// chunk.  A chain of three dependent loads (entry, length, row offsets), each of 0.6 us and more, is what a short call waits
// for: an entry's sequence and length are loaded with its rows, before the tile's entry is known.
struct Found { uint32_t seq, row, n, first, len, warp[32]; };
template <int ROWS, int CHUNK>
__device__ __forceinline__ bool find_tile(const AttnArgs& a, uint32_t t, uint32_t kvh, AttnTile& x, AttnRow* rows, Found& f) {
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
    auto entry = [&](uint32_t e, uint32_t& s0, uint32_t& n, uint32_t& seq, uint32_t& len) {
        uint32_t s1 = 0;
        s0 = n = len = 0; seq = KV_NO_SEQ;
        if (e < a.b.n_seqs) { s0 = a.b.start[e]; s1 = a.b.start[e + 1]; seq = a.b.seq[e]; }
        if (seq < a.b.max_seqs) len = (uint32_t)a.b.lens[seq];
        const bool fine = s0 <= s1 && s1 <= a.b.n_rows;
        if (!fine) atomicOr(a.err, DEVERR_OOB_MAP);
        else n = s1 - s0;
        return (n * a.group + ROWS - 1) / ROWS;
    };
    auto scan = [&](uint32_t v) {
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) { const uint32_t y = __shfl_up_sync(0xffffffffu, v, o); if (lane >= (uint32_t)o) v += y; }
        return v;
    };
    uint32_t len;
    if (a.b.n_seqs <= 32) {                              // every warp for itself
        uint32_t s0, n, seq;
        const uint32_t tiles = entry(lane, s0, n, seq, len), incl = scan(tiles), at = incl - tiles;
        const uint32_t hit = __ballot_sync(0xffffffffu, at <= t && t < incl);
        if (!hit) return false;
        const int e = __ffs(hit) - 1;
        x.seq = __shfl_sync(0xffffffffu, seq, e); x.row = __shfl_sync(0xffffffffu, s0, e); x.n = __shfl_sync(0xffffffffu, n, e);
        x.first = (t - __shfl_sync(0xffffffffu, at, e)) * ROWS; len = __shfl_sync(0xffffffffu, len, e);
    } else {
        uint32_t before = 0;
        if (tid == 0) f.seq = KV_NO_SEQ;
        for (uint32_t e0 = 0; e0 < a.b.n_seqs; e0 += blockDim.x) {
            uint32_t s0, n, seq;
            const uint32_t tiles = entry(e0 + tid, s0, n, seq, len), incl = scan(tiles);
            __syncthreads();
            if (lane == 31) f.warp[warp] = incl;
            __syncthreads();
            uint32_t at = before + incl - tiles;
            for (uint32_t w = 0; w < warps; ++w) { if (w < warp) at += f.warp[w]; before += f.warp[w]; }
            if (at <= t && t < at + tiles) { f.seq = seq; f.row = s0; f.n = n; f.first = (t - at) * ROWS; f.len = len; }
            if (before > t) break;
        }
        __syncthreads();
        x.seq = f.seq; x.row = f.row; x.n = f.n; x.first = f.first; len = f.len;
    }
    if (x.seq == KV_NO_SEQ) return false;
    if (x.seq >= a.b.max_seqs) { if (tid == 0) atomicOr(a.err, DEVERR_OOB_MAP); return false; }
    x.pages = a.b.table + (size_t)x.seq * a.geo.max_pages;
    const int32_t pos0 = (int32_t)len - (int32_t)x.n;
    const uint32_t last = min(x.first + ROWS, x.n * a.group) - 1;
    x.lo = max(pos0 + (int32_t)(x.first / a.group), 0); x.hi = pos0 + (int32_t)(last / a.group);
    for (uint32_t r = tid; r < ROWS; r += blockDim.x) {
        AttnRow y{0, 0, -1};
        const uint32_t k = x.first + r, tok = k / a.group, head = kvh * a.group + k % a.group;
        if (k <= last) {
            const uint64_t oq = a.l_q[x.row + tok], oo = a.l_out[x.row + tok], len = (uint64_t)a.n_head * a.geo.hd;
            y.pos = pos0 + (int32_t)tok;
            if (y.pos < 0 || oq + len > a.n_act || oo + len > a.n_act) { y.pos = -1; atomicOr(a.err, DEVERR_OOB_MAP); }
            y.q = oq + (uint64_t)head * a.geo.hd; y.o = oo + (uint64_t)head * a.geo.hd;
        }
        rows[r] = y;
    }
    x.from = a.window && x.lo >= (int32_t)a.window ? x.lo - (int32_t)a.window + 1 : 0;
    x.main0 = (uint32_t)x.from / CHUNK;
    x.sinks = min((min(a.n_sink, (uint32_t)x.from) + CHUNK - 1) / CHUNK, x.main0);
    x.chunks = x.hi < 0 ? 0u : x.sinks + (uint32_t)x.hi / CHUNK + 1 - x.main0;
    __syncthreads();
    return x.chunks > 0;
}
template <int CHUNK>
__device__ __forceinline__ int32_t chunk_at(const AttnTile& x, uint32_t c) { return (int32_t)((c < x.sinks ? c : c - x.sinks + x.main0) * CHUNK); }

__device__ __forceinline__ bool row_sees(const AttnArgs& a, int32_t pos, int32_t p) {
    return p <= pos && (a.window == 0 || p > pos - (int32_t)a.window || (uint32_t)p < a.n_sink);
}
// Does every row of the tile see all of the n positions from p on?
__device__ __forceinline__ bool tile_sees(const AttnArgs& a, const AttnTile& x, int32_t p, int32_t n) {
    return p + n - 1 <= x.lo && (a.window == 0 || p > x.hi - (int32_t)a.window || (uint32_t)(p + n) <= a.n_sink);
}
// Where position p of the tile's sequence lies in the cache (its key; elements), or -1 where no row of the tile sees it.
__device__ __forceinline__ int64_t tile_position(const AttnArgs& a, const AttnTile& x, uint32_t kvh, int32_t p) {
    if (p > x.hi || (p < x.from && (uint32_t)p >= a.n_sink)) return -1;
    const int32_t page = x.pages[(uint32_t)p / a.geo.page];
    return page < 0 ? -1 : (int64_t)kv_index(a.geo, (uint32_t)page, a.layer, 0, kvh, (uint32_t)p % a.geo.page);
}

__device__ __forceinline__ uint32_t at_smem(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
// 16 bytes to shared memory, zeros where there is no source
__device__ __forceinline__ void at_cp16(uint32_t dst, const void* src, bool real) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" :: "r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}
__device__ __forceinline__ void at_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void at_wait() { asm volatile("cp.async.wait_group %0;" :: "n"(N) : "memory"); }
__device__ __forceinline__ void at_ldsm(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void at_ldsm_t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void at_mma_h(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void at_mma_t(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// x as the sum of two 11-bit terms (22 bits of it, and exact where x has no more)
__device__ __forceinline__ void at_split_t(float x, uint32_t& hi, uint32_t& lo) {
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(hi) : "f"(x));
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(lo) : "f"(x - __uint_as_float(hi)));
}
__device__ __forceinline__ void at_split_h(float x, float y, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
    hi = *reinterpret_cast<const uint32_t*>(&h); lo = *reinterpret_cast<const uint32_t*>(&l);
}
// two values an instruction
__device__ __forceinline__ float2 at_fma2(float2 a, float2 b, float2 c) {
    float2 r;
    asm("{\n\t.reg .b64 a, b, c;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\tfma.rn.f32x2 c, a, b, c;\n\tmov.b64 {%0, %1}, c;\n\t}"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return r;
}
__device__ __forceinline__ float2 at_mul2(float2 a, float2 b) {
    float2 r;
    asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmul.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 at_add2(float2 a, float2 b) {
    float2 r;
    asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float at_exp2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
// A power of two that brings the largest of a row's values (its magnitude `most`) into [2^7, 2^8), and its inverse: fp16 terms
// then neither overflow nor lose bits of what counts.
__device__ __forceinline__ void row_scale(float most, float& up, float& down) {
    int ex = 0;
    if (most > 0.f && most < 3.0e38f) ex = max(-120, min(120, 134 - (int)((__float_as_uint(most) >> 23) & 0xFFu)));
    up = __uint_as_float((uint32_t)(127 + ex) << 23); down = __uint_as_float((uint32_t)(127 - ex) << 23);
}
// tanh(x): below 1/4 its power series (the first term left out is 9e-9 of the value), else 1 - 2 / (1 + e^2x).  NaN for NaN: a row
// with such a score must not come out finite.
__device__ __forceinline__ float at_tanh_small(float x) {
    const float y = x * x;
    return fmaf(x * y, fmaf(y, fmaf(y, fmaf(y, 62.f / 2835.f, -17.f / 315.f), 2.f / 15.f), -1.f / 3.f), x);
}
__device__ __forceinline__ float at_tanh(float x) {
    const float d = 1.f + expf(min_nan(2.f * x, 80.f));
    return fabsf(x) < 0.25f ? at_tanh_small(x) : 1.f - div_by(2.f, d, rcp_newton(d));
}

// One row by a warp, positions one after the other, only those that it sees read: for rows in whose tile an infinity or a NaN
// stands that they do not see (a weight of 0 times it is a NaN in the tiles' products).  Sums over 64 positions at a time.
template <typename T, int HD>
__device__ __noinline__ void attend_row(const AttnArgs& a, const AttnTile x, const AttnRow row, uint32_t kvh) {
    constexpr int N = HD / 32;
    const uint32_t lane = threadIdx.x & 31;
    float q[N], o[N] = {}, m = -INFINITY, l = 0.f;
#pragma unroll
    for (int j = 0; j < N; ++j) q[j] = a.act[row.q + lane * N + j];
    for (int32_t t0 = 0; t0 <= row.pos; t0 += 64) {
        float ob[N] = {}, lb = 0.f;
        const float m0 = m;
        for (int32_t t = t0; t < min(t0 + 64, row.pos + 1); ++t) {
            if (!row_sees(a, row.pos, t)) continue;
            const int64_t at = tile_position(a, x, kvh, t);
            if (at < 0) continue;
            const T* k_row = reinterpret_cast<const T*>(a.pool) + at + lane * N;
            KvRow<T, N> k, v;
            k.load(k_row);
            v.load(k_row + (size_t)a.geo.n_kv * a.geo.page * HD);
            float y[N], s = 0.f;
            k.to_float(y);
#pragma unroll
            for (int j = 0; j < N; ++j) s = fmaf(q[j], y[j], s);
            s = warp_sum(s) * a.scale;
            if (a.cap > 0.f) s = a.cap * tanhf(s / a.cap);
            const float mn = max_nan(m, s), alpha = m == mn ? 1.f : expf(m - mn), p = s == -INFINITY ? 0.f : expf(s - mn);
            v.to_float(y);
            lb = fmaf(lb, alpha, p);
            m = mn;
#pragma unroll
            for (int j = 0; j < N; ++j) ob[j] = fmaf(p, y[j], ob[j] * alpha);
        }
        const float alpha = m0 == m ? 1.f : expf(m0 - m);
        l = fmaf(l, alpha, lb);
#pragma unroll
        for (int j = 0; j < N; ++j) o[j] = fmaf(o[j], alpha, ob[j]);
    }
#pragma unroll
    for (int j = 0; j < N; ++j) a.act[row.o + lane * N + j] = o[j] / l;
}

constexpr float FLT_TOP = 3.402823466e+38f;

// What is left at the end of a tile: PLANES sets of sums over different positions of the same ROWS rows, with the maxima that
// they are relative to (BASE2: in units of ln 2).  They meet in shared memory (`merge`, rows of HD + 4 floats, each set's sums
// times factor()), then the CTAs that share the tile: through their shared memory where they are a cluster, each taking some of
// the rows, else in global memory, where the last one to arrive adds up in their order.  Rows that are not finite are done once
// more, by themselves.
template <int ROWS, int PLANES>
struct End {
    float m[PLANES][ROWS], l[PLANES][ROWS];
    uint32_t bad[(ROWS + 31) / 32], ticket;
    __device__ __forceinline__ float best(int r) const {
        float b = m[0][r];
#pragma unroll
        for (int w = 1; w < PLANES; ++w) b = max_nan(b, m[w][r]);
        return b;
    }
    template <bool BASE2> __device__ static __forceinline__ float weight(float from, float to) {   // of what is relative to `from`, relative to `to`
        const float d = from - (to == -INFINITY ? 0.f : to);
        return BASE2 ? exp2f(d) : expf(d);
    }
    template <bool BASE2> __device__ __forceinline__ float factor(int plane, int r) const { return weight<BASE2>(m[plane][r], best(r)); }
};
__device__ __forceinline__ const float* of_rank(const float* p, uint32_t rank) {     // the same place in another CTA's shared memory
    uint64_t q;
    asm("mapa.u64 %0, %1, %2;" : "=l"(q) : "l"(p), "r"(rank));
    return reinterpret_cast<const float*>(q);
}
__device__ __forceinline__ void cluster_meet() { asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// What a CTA does: a tile's rows of a key head, one of `of` parts of their positions.  Tiles from the last one on: late rows see more.
struct AttnShare { uint32_t tile, kvh, split, of, slot; };      // slot: of the shared ones, in the workspace
__device__ __forceinline__ AttnShare share_of(const AttnArgs& a) {
    const uint32_t b = blockIdx.x;
    AttnShare s{0, 0, 0, 1, 0};
    uint32_t pair = b;
    if (b >= a.whole) { s.slot = (b - a.whole) / a.splits; s.split = (b - a.whole) % a.splits; s.of = a.splits; pair = a.whole + s.slot; }
    const uint32_t tiles = a.pairs / a.geo.n_kv;
    s.kvh = pair / tiles; s.tile = tiles - 1 - pair % tiles;
    return s;
}
inline uint32_t attn_grid(const AttnArgs& a) { return a.whole + (a.pairs - a.whole) * a.splits; }
// This CTA's chunks of the tile; false: it has none
__device__ __forceinline__ bool share_out(const AttnArgs& a, const AttnTile& x, const AttnShare& s, uint32_t& sharers, uint32_t& c0, uint32_t& c1) {
    const uint32_t each = max((x.chunks + s.of - 1) / s.of, a.least);
    sharers = s.of > 1 ? (x.chunks + each - 1) / each : 1u;
    c0 = s.split * each; c1 = s.of > 1 ? min(x.chunks, c0 + each) : x.chunks;
    return s.split < sharers;
}

// By all THREADS of the CTA, m, l and merge written.  CLUSTER: the tile's CTAs (a.splits of them) are one.
template <typename T, int HD, int ROWS, int PLANES, int THREADS, bool BASE2, bool CLUSTER>
__device__ __forceinline__ void settle(const AttnArgs& a, const AttnTile& x, const AttnRow* rows, const AttnShare& part, uint32_t sharers,
                                       float* merge, End<ROWS, PLANES>& end) {
    using E = End<ROWS, PLANES>;
    constexpr int LM = HD + 4, VPR = HD / 4, PER = (ROWS * VPR + THREADS - 1) / THREADS;       // values in fours; of a row, of a thread
    const uint32_t tid = threadIdx.x;
    if (tid < (ROWS + 31) / 32) end.bad[tid] = 0;
    __syncthreads();
    for (int r = tid; r < ROWS; r += THREADS) {          // a row's maximum and sum into the first set's place
        const float b = end.best(r);
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < PLANES; ++w) sum += end.l[w][r] * E::template weight<BASE2>(end.m[w][r], b);
        end.m[0][r] = b; end.l[0][r] = sum;
    }
    __syncthreads();
    const uint32_t live = min((uint32_t)ROWS, x.n * a.group - x.first);
    auto value = [&](uint32_t r, uint32_t d) {
        float4 v = *reinterpret_cast<const float4*>(merge + r * LM + d);
#pragma unroll
        for (int w = 1; w < PLANES; ++w) {
            const float4 y = *reinterpret_cast<const float4*>(merge + (w * ROWS + r) * LM + d);
            v.x += y.x; v.y += y.y; v.z += y.z; v.w += y.w;
        }
        return v;
    };
    auto add = [](float4& v, float f, float4 y) { v.x = fmaf(f, y.x, v.x); v.y = fmaf(f, y.y, v.y); v.z = fmaf(f, y.z, v.z); v.w = fmaf(f, y.w, v.w); };
    uint32_t first = 0, every = 1;                       // this CTA's rows
    if (CLUSTER && a.splits > 1) {
        for (uint32_t i = tid; i < live * VPR; i += THREADS) *reinterpret_cast<float4*>(merge + i / VPR * LM + i % VPR * 4) = value(i / VPR, i % VPR * 4);
        cluster_meet();
        first = part.split; every = a.splits;
    } else if (sharers > 1) {
        const size_t step = (size_t)ROWS * (HD + 4);     // per row: the values, the maximum, the sum
        float* mine = a.part + ((size_t)part.slot * a.splits + part.split) * step;
        for (uint32_t i = tid; i < live * VPR; i += THREADS) *reinterpret_cast<float4*>(mine + i / VPR * LM + i % VPR * 4) = value(i / VPR, i % VPR * 4);
        for (uint32_t r = tid; r < live; r += THREADS) *reinterpret_cast<float2*>(mine + r * LM + HD) = make_float2(end.m[0][r], end.l[0][r]);
        __threadfence();
        __syncthreads();
        if (tid == 0) end.ticket = atomicInc(a.tickets + part.slot, sharers - 1);
        __syncthreads();
        if (end.ticket != sharers - 1) return;
        __threadfence();
    }
    const float* all = a.part + (size_t)part.slot * a.splits * ROWS * LM;
    // A few results of a thread stay in registers (also where other CTAs read the sums); more go where the sums lie, by a short loop
    // (seven copies of it, met once by a
    // CTA, took 5 us to fetch).
    constexpr bool KEEP = PER <= 4 || CLUSTER;
    float4 out[KEEP ? PER : 1];
#pragma unroll(KEEP ? PER : 1)
    for (int j = 0; j < PER; ++j) {
        const uint32_t i = tid + j * THREADS, r = first + i / VPR * every, d = i % VPR * 4;
        if (r >= live) break;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        float z = 0.f;
        if ((CLUSTER && a.splits > 1) || sharers > 1) {
            // eight at a time, in their order, relative to the maximum so far
            float b = -INFINITY;
            constexpr uint32_t U = 8;
#pragma unroll 1
            for (uint32_t k0 = 0; k0 < sharers; k0 += U) {
                float2 q[U];
                float4 y[U];
                float top = b;
#pragma unroll
                for (uint32_t k = 0; k < U; ++k) {
                    const uint32_t c = k0 + k;
                    q[k] = make_float2(-INFINITY, 0.f); y[k] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (c >= sharers) continue;
                    if (CLUSTER) {
                        q[k] = make_float2(*of_rank(&end.m[0][r], c), *of_rank(&end.l[0][r], c));
                        y[k] = *reinterpret_cast<const float4*>(of_rank(merge + r * LM + d, c));
                    } else {
                        const float* from = all + ((size_t)c * ROWS + r) * LM;
                        q[k] = __ldcg(reinterpret_cast<const float2*>(from + HD));
                        y[k] = __ldcg(reinterpret_cast<const float4*>(from + d));
                    }
                }
#pragma unroll
                for (uint32_t k = 0; k < U; ++k) top = max_nan(top, q[k].x);
                const float w0 = E::template weight<BASE2>(b, top);
                v.x *= w0; v.y *= w0; v.z *= w0; v.w *= w0; z *= w0;
                b = top;
#pragma unroll
                for (uint32_t k = 0; k < U; ++k) {
                    const float w = E::template weight<BASE2>(q[k].x, b);
                    z = fmaf(q[k].y, w, z);
                    add(v, w, y[k]);
                }
            }
        } else { v = value(r, d); z = end.l[0][r]; }
        const float rcp = __frcp_rn(z);                  // (four divisions took half of this loop's time)
        v = make_float4(div_by(v.x, z, rcp), div_by(v.y, z, rcp), div_by(v.z, z, rcp), div_by(v.w, z, rcp));
        const float most = max_nan(max_nan(fabsf(v.x), fabsf(v.y)), max_nan(fabsf(v.z), fabsf(v.w)));
        if (rows[r].pos >= 0 && !(most <= FLT_TOP)) atomicOr(&end.bad[r >> 5], 1u << (r & 31));
        if constexpr (KEEP) out[j] = v;
        else *reinterpret_cast<float4*>(merge + r * LM + d) = v;
    }
    __syncthreads();
    auto bad = [&](uint32_t r) { return end.bad[r >> 5] >> (r & 31) & 1u; };
#pragma unroll(KEEP ? PER : 1)
    for (int j = 0; j < PER; ++j) {
        const uint32_t i = tid + j * THREADS, r = first + i / VPR * every, d = i % VPR * 4;
        if (r >= live) break;
        if (rows[r].pos < 0 || bad(r)) continue;
        float* to = a.act + rows[r].o + d;
        float4 v;
        if constexpr (KEEP) v = out[j];
        else v = *reinterpret_cast<const float4*>(merge + r * LM + d);
        if (rows[r].o % 4 == 0) *reinterpret_cast<float4*>(to) = v;
        else { to[0] = v.x; to[1] = v.y; to[2] = v.z; to[3] = v.w; }
    }
    for (uint32_t r = first + (tid >> 5) * every; r < live; r += (THREADS >> 5) * every)
        if (bad(r)) attend_row<T, HD>(a, x, rows[r], part.kvh);
    if (CLUSTER && a.splits > 1) cluster_meet();         // nobody leaves while its shared memory is read
}
// Do the CTAs that share a tile come as a cluster?  (Of tiles of 16 rows and less)
constexpr uint32_t ATTN_CLUSTER = 16;                // at most
inline bool attn_cluster(const AttnArgs& a) { return a.whole == 0 && a.splits > 1 && a.splits <= ATTN_CLUSTER && (a.splits & (a.splits - 1)) == 0; }
template <typename K>
inline int launch_attn(K kernel, bool& set, const AttnArgs& a, int threads, int smem, bool cluster) {
    if (!set) {
        if (cudaFuncSetAttribute((const void*)kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess ||
            (cluster && cudaFuncSetAttribute((const void*)kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess))
            return fail(ADAMAH_ERR_BACKEND, "attn_kv: cannot set the kernel's limits");
        set = true;
    }
    const dim3 grid(attn_grid(a));
    if (cluster) launch_k_cluster(kernel, grid, dim3(threads), smem, g.stream, false, a.splits, false, a);
    else kernel<<<grid, threads, smem, g.stream>>>(a);
    count_launch();
    return check_launch("map_attn_kv");
}

// Two or four rows to a tile (attn_kv_thin.cu), pages of whole chunks
constexpr uint32_t THIN_CTAS = 3;                    // on an SM
int launch_attn_thin(const AttnArgs& a, uint32_t elem, uint32_t rows);
uint32_t attn_thin_chunk(uint32_t elem, uint32_t hd);
// The tcgen05 form, 128 rows to a tile, over an fp16 cache with heads of 64 or 128 (attn_kv_tc.cu).
int launch_attn_tc(const AttnArgs& a, const KvCache& kv);

}  // namespace ab
