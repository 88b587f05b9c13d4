// The next tokens out of whole rows of logits: temperature, top-k, nucleus, min-p and the draw, every row by its own rule and
// random number (map_topk.comp, map_topp.comp and map_sample_categorical.comp, which know 64 candidates).
//
//   w_i = exp((l_i - max) / T);   in the order of falling l, lower index first: the first top_k, of those the shortest run
//   whose weights reach top_p of theirs, of those the ones with w >= min_p;   token = first i whose running sum over the
//   kept j <= i is above u times the sum of all kept
//
// Each cut leaves a run of that order, so what is kept is a threshold: a logit, and how many of those that equal it (the
// lowest indices).  Nothing is sorted: a threshold is found by histograms, the first over equal steps of the logit (steps of
// 1/64 of the temperature, where logits spread evenly), then over the bits in which the logits of the crossing bin differ.
//
// Sums of weights decide about whole numbers, so they are exact: weights are 64-bit exponentials rounded to integers, and
// integers add up to the same sum in any order (32-bit sums over 262144 tokens draw another token once in some hundred
// rows; atomics on floating point another one from launch to launch).
//
// A row is a cluster of CTAs, each with its share of the logits in shared memory: one pass over HBM, what follows reads
// shared memory, and the CTAs' histograms and sums meet through it.
#include "common.cuh"

#include <cooperative_groups.h>

namespace ab {

namespace cg = cooperative_groups;

constexpr int SV_T = 1024, SV_W = SV_T / 32;
constexpr uint32_t SV_BINS = 2048;
constexpr uint32_t SV_SUBS = 256;                    // stretches of a CTA's share, a sum for each
constexpr uint32_t SV_RESIDENT = 36864;              // logits that a CTA keeps in shared memory at most
constexpr uint32_t SV_FEW = 2048;                    // candidates that one CTA sorts

struct SampleArgs {
    float* map; uint64_t n_el;
    const uint32_t *l_logits, *l_u, *l_dst; const adam_b200_sample_rule* rules;
    uint32_t V, chunk; int shift;
    uint32_t* err;
};

// A logit as an unsigned number in its order; both zeros are one.
__device__ __forceinline__ uint32_t sv_key(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float sv_value(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key); }
__device__ __forceinline__ uint64_t warp_sum_u64(uint64_t v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ uint64_t warp_scan_u64(uint64_t v) {      // inclusive
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const uint64_t t = __shfl_up_sync(0xffffffffu, v, o); if (lane >= o) v += t; }
    return v;
}

// Weights as integers.  (max - x) / (T ln 2) = y is formed in two 32-bit words; 2^-y = 2^-k 2^(-i/256) (1 - s) with the table's
// entry i, an integer k and s = 1 - 2^-r, |r| <= 1/512, whose series needs three terms.  s is known to 2^-24 of itself, so a
// weight to 1e-10 of itself: what is drawn changes with probability 1e-7 or so, and the 64-bit exponential cost 60 us more
// for 64 rows of 262144.
struct SvWeights {
    const uint64_t* table;                            // 2^62 2^(-i/256)
    float mx, c_hi, c_lo; int shift;
    __device__ __forceinline__ uint64_t operator()(float x) const {
        if (x == mx) return 1ull << shift;
        const float d = mx - x, b = d - mx, d_lo = (mx - (d - b)) + (-x - b);
        float y = d * c_hi, y_lo = fmaf(d, c_hi, -y) + fmaf(d, c_lo, d_lo * c_hi);
        if (d > 3.402823466e+38f) {                    // beyond 32 bits: a logit or the difference of two
            const double e = ((double)mx - (double)x) * ((double)c_hi + (double)c_lo);
            y = (float)e; y_lo = (float)(e - (double)y);
        }
        if (!(y < (float)(shift + 1))) return 0;       // below half a unit, or not a number (an infinite maximum)
        const float t = rintf(y * 256.f), r = fmaf(t, -1.f / 256.f, y) + y_lo;
        const int ti = (int)t;
        const float z = r * 0.69314718055994530942f, s = z * (1.f - z * (0.5f - z * (1.f / 6.f)));
        const uint64_t w = table[ti & 255];
        const int64_t cut = (int64_t)(uint32_t)(w >> 32) * (int)(s * 4294967296.f);
        const int sh = 62 - shift + (ti >> 8);
        return ((w - (uint64_t)cut) + (1ull << (sh - 1))) >> sh;
    }
};

struct SvBins { uint32_t n[SV_BINS], lo[SV_BINS], hi[SV_BINS]; };      // counts; sums in two words (64-bit shared atomics are loops)
struct SvShared {
    union { SvBins own; uint64_t list[SV_FEW]; };     // the CTA's histogram; the first CTA's candidates
    union { SvBins all; uint64_t w[SV_FEW]; };        // its share of the cluster's bins, merged; the candidates' weights
    uint64_t table[256];
    uint64_t seg_v, pass_v; uint32_t ties;            // weights of that share; of what is kept; logits equal to the threshold
    uint32_t kmin, kmax, n_list, first; float max;
    uint64_t sub_v[SV_SUBS], wv[SV_W + 1];
    uint32_t sub_n[SV_SUBS]; float wmax[SV_W];
    uint64_t hit_above, hit_v; uint32_t hit_bin, hit_n, hit_count;
    uint64_t peer_v[16];
};

// n 64-bit keys (a power of two) into falling order, by the whole CTA
__device__ __forceinline__ void sv_sort(uint64_t* key, uint32_t n) {
    for (uint32_t size = 2; size <= n; size <<= 1)
        for (uint32_t half = size >> 1; half > 0; half >>= 1) {
            __syncthreads();
            for (uint32_t t = threadIdx.x; t < n / 2; t += SV_T) {
                const uint32_t i = 2 * t - (t & (half - 1)), j = i + half;
                const uint64_t x = key[i], y = key[j];
                if ((x < y) == ((i & size) == 0)) { key[i] = y; key[j] = x; }
            }
        }
    __syncthreads();
}

template <bool RES>
__global__ void __launch_bounds__(SV_T, 1) k_sample_vocab(const SampleArgs a) {
    extern __shared__ __align__(16) unsigned char sv_sm[];
    SvShared& s = *reinterpret_cast<SvShared*>(sv_sm);
    float* sx = reinterpret_cast<float*>(sv_sm + (sizeof(SvShared) + 15) / 16 * 16);
    cg::cluster_group cl = cg::this_cluster();
    const uint32_t C = cl.num_blocks(), rank = cl.block_rank(), row = blockIdx.x / C;
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint64_t ol = a.l_logits[row], ou = a.l_u[row], od = a.l_dst[row];
    const bool lead = rank == 0 && tid == 0;
    if (ol + a.V > a.n_el || ou >= a.n_el || od >= a.n_el) { if (lead) atomicOr(a.err, DEVERR_OOB_MAP); return; }
    const adam_b200_sample_rule rule = a.rules[row];
    const float u = a.map[ou];
    if (!(u >= 0.f && u < 1.f) || rule.temperature != rule.temperature || rule.top_p != rule.top_p || rule.min_p != rule.min_p) {
        if (lead) { a.map[od] = -1.f; atomicOr(a.err, DEVERR_BAD_RULE); }
        return;
    }
    const uint32_t base = rank * a.chunk, n = base < a.V ? min(a.chunk, a.V - base) : 0u;
    const float* src = a.map + ol + base;
    const bool aligned = ((ol + base) & 3) == 0;
    auto clean = [](float x) { return x == x ? x : -INFINITY; };
    auto get = [&](uint32_t i) { return RES ? sx[i] : clean(src[i]); };
    // f(logit, its place in the CTA's share) for each, in no order
    auto each = [&](auto f) {
        if (RES || aligned) {
            const float4* v4 = reinterpret_cast<const float4*>(RES ? sx : src);
            const uint32_t n4 = n / 4;
#pragma unroll 4
            for (uint32_t i = tid; i < n4; i += SV_T) {
                const float4 v = v4[i];
                f(clean(v.x), 4 * i); f(clean(v.y), 4 * i + 1); f(clean(v.z), 4 * i + 2); f(clean(v.w), 4 * i + 3);
            }
            if (tid < n % 4) f(get(4 * n4 + tid), 4 * n4 + tid);
        } else {
#pragma unroll 8
            for (uint32_t i = tid; i < n; i += SV_T) f(clean(src[i]), i);
        }
    };
    if (tid < 256) s.table[tid] = (uint64_t)__double2ull_rn(exp2(-(double)tid / 256.0) * 4611686018427387904.0);
    if (tid == 0) { s.n_list = 0; s.first = 0xffffffffu; }

    // ---- the largest logit ----
    float mx = -INFINITY;
    if (RES && aligned) {
        const uint32_t n4 = n / 4;
#pragma unroll 4
        for (uint32_t i = tid; i < n4; i += SV_T) {
            float4 v = reinterpret_cast<const float4*>(src)[i];
            v.x = clean(v.x); v.y = clean(v.y); v.z = clean(v.z); v.w = clean(v.w);
            reinterpret_cast<float4*>(sx)[i] = v;
            mx = fmaxf(fmaxf(mx, fmaxf(v.x, v.y)), fmaxf(v.z, v.w));
        }
        if (tid < n % 4) { const float v = clean(src[4 * n4 + tid]); sx[4 * n4 + tid] = v; mx = fmaxf(mx, v); }
    } else if (RES) {
#pragma unroll 8
        for (uint32_t i = tid; i < n; i += SV_T) { const float v = clean(src[i]); sx[i] = v; mx = fmaxf(mx, v); }
    } else
        each([&](float x, uint32_t) { mx = fmaxf(mx, x); });
    mx = warp_max(mx);
    if (lane == 0) s.wmax[warp] = mx;
    __syncthreads();
    if (warp == 0) {
        mx = warp_max(s.wmax[lane]);
        if (lane == 0) s.max = mx;
    }
    cl.sync();
    mx = -INFINITY;
    for (uint32_t c = 0; c < C; ++c) mx = fmaxf(mx, *cl.map_shared_rank(&s.max, c));
    if (mx == -INFINITY || !(rule.temperature > 0.f)) {         // nothing to draw, or the first of the largest: the cluster agrees
        if (mx == -INFINITY) { if (lead) a.map[od] = -1.f; }
        else {
            uint32_t at = 0xffffffffu;
            each([&](float x, uint32_t i) { if (x == mx) at = min(at, i); });
            at = __reduce_min_sync(0xffffffffu, at);
            if (lane == 0 && at != 0xffffffffu) atomicMin(cl.map_shared_rank(&s.first, 0), base + at);
        }
        cl.sync();
        if (lead && mx != -INFINITY) a.map[od] = (float)s.first;
        return;
    }

    const double c = 1.4426950408889634074 / (double)rule.temperature;
    const float c_hi = (float)c;
    const SvWeights weight{s.table, mx, c_hi, c_hi <= 3.402823466e+38f ? (float)(c - (double)c_hi) : 0.f, a.shift};
    const float step = 64.0f / rule.temperature;
    const uint64_t least = (uint64_t)ceil((double)fminf(fmaxf(rule.min_p, 0.f), 1.f) * (double)(1ull << a.shift));    // of min_p
    auto bin_of = [&](float x) -> uint32_t {
        if (x == mx) return 0u;
        const float t = (mx - x) * step;
        return t < (float)(SV_BINS - 1) ? (uint32_t)t : SV_BINS - 1;
    };

    // ---- thresholds: a logit is kept if its key is above key_t, or equals it and it is one of the first n_ties of those ----
    const uint32_t key_none = sv_key(-INFINITY);
    uint32_t key_t = key_none, n_ties = 0;

    // The cluster's histogram: CTA c ends with the bins c * per .. of all, and their totals.
    const uint32_t per = SV_BINS / C;
    auto merge = [&](bool sums) {
        cl.sync();
        uint64_t tv = 0;
        for (uint32_t b = tid; b < per; b += SV_T) {
            uint32_t cn = 0; uint64_t cv = 0;
#pragma unroll 4
            for (uint32_t k = 0; k < C; ++k) {
                const SvBins* h = cl.map_shared_rank(&s.own, k);
                cn += h->n[rank * per + b];
                if (sums) cv += (uint64_t)h->lo[rank * per + b] + ((uint64_t)h->hi[rank * per + b] << 32);
            }
            if (!sums) cv = cn;
            s.all.n[b] = cn; s.all.lo[b] = (uint32_t)cv; s.all.hi[b] = (uint32_t)(cv >> 32);
            tv += cv;
        }
        tv = warp_sum_u64(tv);
        if (lane == 0) s.wv[warp] = tv;
        __syncthreads();
        if (warp == 0) {
            tv = warp_sum_u64(s.wv[lane]);
            if (lane == 0) s.seg_v = tv;
        }
        cl.sync();
        if (tid < C) s.peer_v[tid] = *cl.map_shared_rank(&s.seg_v, tid);
        __syncthreads();
    };
    auto total = [&]() { uint64_t v = 0; for (uint32_t k = 0; k < C; ++k) v += s.peer_v[k]; return v; };
    // The bin in which the running sum reaches `target` (1 .. total), the sum ahead of it, its own and its count: in s.hit_*.
    auto cross = [&](uint64_t target) {
        uint64_t above = 0; uint32_t seg = 0;
        while (seg + 1 < C && above + s.peer_v[seg] < target) above += s.peer_v[seg++];
        const SvBins* h = cl.map_shared_rank(&s.all, seg);
        const uint32_t mine = (per + SV_T - 1) / SV_T, b0 = tid * mine;
        uint64_t v = 0;
        for (uint32_t b = b0; b < min(b0 + mine, per); ++b) v += (uint64_t)h->lo[b] + ((uint64_t)h->hi[b] << 32);
        const uint64_t incl = warp_scan_u64(v);
        if (lane == 31) s.wv[warp] = incl;
        __syncthreads();
        const uint64_t ahead = warp_scan_u64(s.wv[lane]);
        if (warp) above += __shfl_sync(0xffffffffu, ahead, warp - 1);
        above += incl - v;
        if (above < target && target <= above + v)
            for (uint32_t b = b0; b < min(b0 + mine, per); ++b) {
                const uint64_t x = (uint64_t)h->lo[b] + ((uint64_t)h->hi[b] << 32);
                if (target <= above + x) { s.hit_bin = seg * per + b; s.hit_above = above; s.hit_v = x; s.hit_n = h->n[b]; break; }
                above += x;
            }
        __syncthreads();
    };
    auto clear = [&]() {
        for (uint32_t b = tid; b < SV_BINS; b += SV_T) { s.own.n[b] = 0; s.own.lo[b] = 0; s.own.hi[b] = 0; }
        __syncthreads();
    };
    auto count = [&](uint32_t b, float x, bool sums) {
        atomicAdd(&s.own.n[b], 1u);
        if (sums) {
            const uint64_t w = weight(x);
            const uint32_t lo = (uint32_t)w, old = atomicAdd(&s.own.lo[b], lo), hi = (uint32_t)(w >> 32) + (old + lo < old ? 1u : 0u);
            if (hi) atomicAdd(&s.own.hi[b], hi);
        }
    };
    auto share = [&](uint64_t all) {                  // top_p of a sum, rounded up, at least one unit
        const uint64_t p = (uint64_t)((double)fmaxf(rule.top_p, 0.f) * 18446744073709551616.0), t = __umul64hi(p, all) + (p * all != 0 ? 1u : 0u);
        return t ? t : 1ull;
    };
    // Up to SV_FEW candidates in the first CTA's list: sorted, cut by the whole rule and drawn from there.  top_p is a share of
    // `all`, or of the first top_k (all = 0).
    auto few = [&](uint64_t all) {
        const uint32_t m = s.n_list;
        uint32_t size = 2;
        while (size < m) size <<= 1;
        for (uint32_t i = m + tid; i < size; i += SV_T) s.list[i] = 0;
        sv_sort(s.list, size);                        // by key, then the lower index first
        const uint32_t cand = rule.top_k > 0 ? min(m, rule.top_k) : m;
        constexpr int PER = SV_FEW / SV_T;
        uint64_t w[PER], mine = 0;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const uint32_t i = tid * PER + j;
            w[j] = i < cand ? weight(sv_value((uint32_t)(s.list[i] >> 32))) : 0;
            mine += w[j];
        }
        auto scan = [&](uint64_t v, uint64_t& sum) {   // exclusive over the CTA
            const uint64_t incl = warp_scan_u64(v);
            __syncthreads();
            if (lane == 31) s.wv[warp] = incl;
            __syncthreads();
            const uint64_t ahead = warp_scan_u64(s.wv[lane]);
            sum = __shfl_sync(0xffffffffu, ahead, 31);
            const uint64_t before = __shfl_sync(0xffffffffu, ahead, warp ? warp - 1 : 0);
            return incl - v + (warp ? before : 0ull);
        };
        uint64_t sum, at = scan(mine, sum);
        const uint64_t stop = rule.top_p < 1.f ? share(all ? all : sum) : ~0ull;      // kept while the sum ahead is below it
        // the kept ones again, by index
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const uint32_t i = tid * PER + j;
            const bool in = i < cand && (i == 0 || at < stop) && w[j] >= least;
            at += w[j];
            const uint64_t e = i < m ? s.list[i] : 0;
            if (i < SV_FEW) s.w[i] = w[j];
            if (i < size) s.list[i] = in ? (e << 32) | i : 0;         // the low word of an entry falls with the index
        }
        sv_sort(s.list, size);
        mine = 0;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const uint32_t i = tid * PER + j;
            const uint64_t e = i < size ? s.list[i] : 0;
            w[j] = e ? s.w[(uint32_t)e & (SV_FEW - 1)] : 0;
            mine += w[j];
        }
        at = scan(mine, sum);
        const uint64_t target = __umul64hi((uint64_t)((double)u * 18446744073709551616.0), sum);
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            if (at <= target && target < at + w[j]) a.map[od] = (float)(0xffffffffu - (uint32_t)(s.list[tid * PER + j] >> 32));
            at += w[j];
        }
    };
    // Cuts what is kept to the run that reaches a target: so many logits (sums false), or so much weight.  True: the token is drawn.
    auto cut = [&](bool sums) -> bool {
        clear();
        each([&](float x, uint32_t) { if (sv_key(x) > key_t) count(bin_of(x), x, sums); });
        merge(sums);
        const uint64_t above = total();               // of what lies above key_t; the ties at it are n_ties times one weight
        uint64_t target;
        if (sums) {
            const uint64_t wt = n_ties ? weight(sv_value(key_t)) : 0;
            target = share(above + n_ties * wt);
            if (target > above) { n_ties = (uint32_t)((target - above + wt - 1) / wt); return false; }
        } else {
            if (above <= rule.top_k) return false;
            target = rule.top_k;
        }
        cross(target);
        uint32_t in = s.hit_n;
        const uint32_t bin = s.hit_bin;
        uint64_t rest = target - s.hit_above;
        // how many candidates lie in the bins up to it: where the first CTA can sort them, it does the rest
        const uint32_t key_before = key_t, ties_before = n_ties;
        if (ties_before == 0 && key_before == key_none) {
            uint64_t upto = s.hit_above + s.hit_v;
            if (sums) {                               // counts of the bins before it, this CTA's share of them
                uint32_t v = 0;
                for (uint32_t b = tid; b < per; b += SV_T) v += rank * per + b <= bin ? s.all.n[b] : 0u;
                v = __reduce_add_sync(0xffffffffu, v);
                if (tid == 0) s.hit_count = 0;
                __syncthreads();
                if (lane == 0) atomicAdd(&s.hit_count, v);
                cl.sync();
                upto = 0;
                for (uint32_t k = 0; k < C; ++k) upto += *cl.map_shared_rank(&s.hit_count, k);
            }
            if (upto <= SV_FEW) {
                uint32_t* const n_list = cl.map_shared_rank(&s.n_list, 0);
                uint64_t* const list = cl.map_shared_rank(&s.list[0], 0);
                each([&](float x, uint32_t i) {
                    if (x > -INFINITY && bin_of(x) <= bin) list[atomicAdd(n_list, 1u)] = (uint64_t)sv_key(x) << 32 | (0xffffffffu - (base + i));
                });
                cl.sync();
                if (rank == 0) few(sums ? above : 0);
                return true;
            }
        }
        // the keys of the bin
        uint32_t lo = 0xffffffffu, hi = 0u;
        each([&](float x, uint32_t) {
            const uint32_t k = sv_key(x);
            if (k > key_t && bin_of(x) == bin) { lo = min(lo, k); hi = max(hi, k); }
        });
        lo = __reduce_min_sync(0xffffffffu, lo); hi = __reduce_max_sync(0xffffffffu, hi);
        if (tid == 0) { s.kmin = 0xffffffffu; s.kmax = 0u; }
        __syncthreads();
        if (lane == 0) { atomicMin(&s.kmin, lo); atomicMax(&s.kmax, hi); }
        cl.sync();
        lo = 0xffffffffu; hi = 0u;
        for (uint32_t k = 0; k < C; ++k) { lo = min(lo, *cl.map_shared_rank(&s.kmin, k)); hi = max(hi, *cl.map_shared_rank(&s.kmax, k)); }
        for (;;) {
            if (sums ? in == 1 : rest == in) { key_t = lo - 1; n_ties = 0; return false; }       // all of them
            if (lo == hi) {
                if (sums) { const uint64_t w = weight(sv_value(lo)); rest = (rest + w - 1) / w; }
                key_t = lo; n_ties = (uint32_t)rest;
                if (n_ties == in) { key_t = lo - 1; n_ties = 0; }
                return false;
            }
            const int sh = max(0, 32 - __clz(hi - lo) - 11);
            clear();
            each([&](float x, uint32_t) {
                const uint32_t k = sv_key(x);
                if (k >= lo && k <= hi) count((hi - k) >> sh, x, sums);
            });
            merge(sums);
            cross(rest);
            in = s.hit_n; rest -= s.hit_above;
            hi -= s.hit_bin << sh;
            const uint32_t span = (1u << sh) - 1u;
            lo = hi - lo > span ? hi - span : lo;
        }
    };
    if (rule.top_k > 0 && rule.top_k < a.V && cut(false)) return;
    if (rule.top_p < 1.f && cut(true)) return;

    // ---- the draw: sums of stretches in index order, then the stretch that holds the token ----
    const uint32_t sub = max(32u, ((a.chunk + SV_SUBS - 1) / SV_SUBS + 31) & ~31u), n_sub = (n + sub - 1) / sub;
    const bool ranked = n_ties > 0;
    uint32_t ties_before = 0;
    if (ranked) {
        for (uint32_t b = warp; b < n_sub; b += SV_W) {
            uint32_t k = 0;
            for (uint32_t i = b * sub + lane; i < (b + 1) * sub; i += 32) k += i < n && sv_key(get(i)) == key_t;
            k = __reduce_add_sync(0xffffffffu, k);
            if (lane == 0) s.sub_n[b] = k;
        }
        __syncthreads();
        if (tid == 0) {
            uint32_t t = 0;
            for (uint32_t b = 0; b < n_sub; ++b) { const uint32_t k = s.sub_n[b]; s.sub_n[b] = t; t += k; }
            s.ties = t;
        }
        cl.sync();
        for (uint32_t k = 0; k < rank; ++k) ties_before += *cl.map_shared_rank(&s.ties, k);
    }
    // the weight of element i where it is kept; `tie`: its place among the equal ones (called by whole warps)
    auto kept = [&](uint32_t i, uint32_t& tie) -> uint64_t {
        const float x = i < n ? get(i) : -INFINITY;
        const uint32_t k = sv_key(x);
        bool in = k > key_t;
        if (ranked) {
            const uint32_t eq = __ballot_sync(0xffffffffu, k == key_t);
            in |= k == key_t && tie + __popc(eq & ((1u << lane) - 1u)) < n_ties;
            tie += __popc(eq);
        }
        if (!in) return 0;
        const uint64_t w = weight(x);
        return w >= least ? w : 0;
    };
    for (uint32_t b = warp; b < n_sub; b += SV_W) {
        uint64_t v = 0;
        uint32_t tie = ranked ? ties_before + s.sub_n[b] : 0;
#pragma unroll 4
        for (uint32_t i = b * sub; i < (b + 1) * sub; i += 32) v += kept(i + lane, tie);
        v = warp_sum_u64(v);
        if (lane == 0) s.sub_v[b] = v;
    }
    __syncthreads();
    if (warp == 0) {
        uint64_t v = 0;
        for (uint32_t b = lane; b < n_sub; b += 32) v += s.sub_v[b];
        v = warp_sum_u64(v);
        if (lane == 0) s.pass_v = v;
    }
    cl.sync();
    uint64_t before = 0, all = 0;
    for (uint32_t k = 0; k < C; ++k) { const uint64_t v = *cl.map_shared_rank(&s.pass_v, k); before += k < rank ? v : 0; all += v; }
    const uint64_t target = __umul64hi((uint64_t)((double)u * 18446744073709551616.0), all);     // the running sum to be exceeded
    if (before <= target && target < before + s.pass_v && warp == 0) {
        uint64_t v[SV_SUBS / 32], mine = 0;                        // lane l: stretches 8 l ..
#pragma unroll
        for (int j = 0; j < (int)SV_SUBS / 32; ++j) { const uint32_t b = lane * (SV_SUBS / 32) + j; v[j] = b < n_sub ? s.sub_v[b] : 0; mine += v[j]; }
        uint64_t at = before + warp_scan_u64(mine) - mine;
        uint32_t hit = 0xffffffffu;
#pragma unroll
        for (int j = 0; j < (int)SV_SUBS / 32; ++j) { if (hit == 0xffffffffu && at + v[j] > target) hit = lane * (SV_SUBS / 32) + j; if (hit == 0xffffffffu) at += v[j]; }
        const uint32_t who = __ffs(__ballot_sync(0xffffffffu, hit != 0xffffffffu)) - 1u;
        const uint32_t b = __shfl_sync(0xffffffffu, hit, who);
        at = __shfl_sync(0xffffffffu, at, who);
        uint32_t tie = ranked ? ties_before + s.sub_n[b] : 0;
        for (uint32_t i = b * sub; i < (b + 1) * sub; i += 32) {
            const uint64_t w = kept(i + lane, tie), incl = at + warp_scan_u64(w);
            const uint32_t over = __ballot_sync(0xffffffffu, incl > target);
            if (over) {
                if (lane == (uint32_t)__ffs(over) - 1u) a.map[od] = (float)(base + i + lane);
                break;
            }
            at = __shfl_sync(0xffffffffu, incl, 31);
        }
    }
    cl.sync();                                        // nobody leaves while its shared memory is read
}

}  // namespace ab

using namespace ab;

extern "C" int map_sample_dev(uint32_t map, uint32_t logits_h, uint32_t rule_h, uint32_t u_h, uint32_t dst_h, uint32_t n_rows, uint32_t n_vocab) {
    if (!ready()) return ADAMAH_ERR_INVALID;
    Map* m = get_map(map);
    if (!m) return ADAMAH_ERR_NOT_FOUND;
    if (m->dtype != ADAMAH_DTYPE_F32 || m->pack_size != 1) return fail(ADAMAH_ERR_INVALID, "sample: map %u must be float32 with pack_size 1", map);
    if (!n_rows) return ADAMAH_OK;
    if (!n_vocab || n_vocab > (1u << 24) || n_rows > 65536) return fail(ADAMAH_ERR_INVALID, "sample: %u rows of %u logits", n_rows, n_vocab);
    for (uint32_t h : {logits_h, u_h, dst_h}) if (!handle_ok(h, n_rows * 4)) return ADAMAH_ERR_NOT_FOUND;
    if (!handle_ok(rule_h, n_rows * (uint32_t)sizeof(adam_b200_sample_rule))) return ADAMAH_ERR_NOT_FOUND;
    SampleArgs a = {};
    a.map = (float*)m->buf; a.n_el = m->n_elems; a.l_logits = hlocs(logits_h); a.l_u = hlocs(u_h); a.l_dst = hlocs(dst_h);
    a.rules = (const adam_b200_sample_rule*)g.handles[rule_h].dev; a.V = n_vocab; a.err = g.dev_err;
    // CTAs of a row: a CTA gets through 4096 logits while it waits for the others once, and rows enough to fill the GPU need no more
    uint32_t C = 1;
    while (C < 16 && n_vocab / C > 4096 && (uint64_t)n_rows * C * 2 <= (uint32_t)g.sm_count) C *= 2;
    a.chunk = ((n_vocab + C - 1) / C + 31) & ~31u;
    int lg = 0;
    while ((1ull << lg) < n_vocab) ++lg;
    a.shift = 63 - lg < 50 ? 63 - lg : 50;            // n_vocab weights of at most 2^shift stay below 2^64
    const bool res = a.chunk <= SV_RESIDENT;
    void (*k)(const SampleArgs) = res ? k_sample_vocab<true> : k_sample_vocab<false>;
    const size_t smem = (sizeof(SvShared) + 15) / 16 * 16 + (res ? (size_t)a.chunk * 4 : 0);
    static bool set[2] = {false, false};
    if (!set[res]) {
        if (cudaFuncSetAttribute((const void*)k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)((sizeof(SvShared) + 15) / 16 * 16 + (res ? SV_RESIDENT * 4 : 0))) != cudaSuccess ||
            cudaFuncSetAttribute((const void*)k, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)
            return fail(ADAMAH_ERR_BACKEND, "sample: cannot set the kernel's limits");
        set[res] = true;
    }
    launch_k_cluster(k, dim3(n_rows * C), dim3(SV_T), smem, g.stream, false, C, false, a);
    count_launch();
    const int rc = check_launch("map_sample");
    end_of_op();
    return rc;
}
