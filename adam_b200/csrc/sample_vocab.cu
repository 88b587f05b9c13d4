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
// Sums of weights decide about whole numbers, so they are exact: weights are integers of up to 50 bits (SvWeights), which add up
// to the same sum in any order (32-bit sums over 262144 tokens draw another token once in some hundred
// rows; atomics on floating point another one from launch to launch).
//
// A row is a cluster of CTAs, each with its share of the logits in shared memory: one pass over HBM, what follows reads
// shared memory, and the CTAs' histograms and sums meet through it.
#include "common.cuh"

#include <cooperative_groups.h>
#include <type_traits>

namespace ab {

namespace cg = cooperative_groups;

constexpr uint32_t SV_SUBS = 256;                    // stretches of a CTA's share, a sum for each
constexpr uint32_t SV_RESIDENT = 36864;              // logits that a CTA keeps in shared memory at most
constexpr uint32_t SV_TABLE = 1024, SV_GATHER = 8192;
constexpr uint32_t SV_NEAR_BINS = 256;
enum SvMode { SV_COUNT, SV_NEAR, SV_EXACT };
__device__ __forceinline__ float2 sv_fma2(float2 a, float2 b, float2 c) {
    float2 r;
    asm("{\n\t.reg .b64 a, b, c;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\tfma.rn.f32x2 c, a, b, c;\n\tmov.b64 {%0, %1}, c;\n\t}"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return r;
}
__device__ __forceinline__ float2 sv_add2(float2 a, float2 b) {
    float2 r;
    asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
constexpr int SV_T = 1024, SV_W = SV_T / 32;
constexpr uint32_t SV_BINS = 2048, SV_FEW = 2048, SV_SHORT = 512;      // bins; candidates that one CTA sorts, that it sorts twice rather than all others sum up

struct SampleArgs {
    float* map; uint64_t n_el;
    const uint32_t *l_logits, *l_u, *l_dst; const adam_b200_sample_rule* rules;
    uint32_t V, chunk; int shift;
    uint32_t* err;
};

// A logit and its index as a number that falls with the order of the rule; both zeros are one.
__device__ __forceinline__ uint64_t sv_key(float x, uint32_t i) {
    const uint32_t u = __float_as_uint(x + 0.0f);
    return (uint64_t)(u & 0x80000000u ? ~u : u | 0x80000000u) << 32 | (0xffffffffu - i);
}
__device__ __forceinline__ float sv_value(uint64_t key) { const uint32_t k = (uint32_t)(key >> 32); return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }
__device__ __forceinline__ uint32_t sv_index(uint64_t key) { return 0xffffffffu - (uint32_t)key; }
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

// 2^30 2^(-i/1024), by the series of the exponential
struct SvTable {
    uint32_t w[SV_TABLE];
    constexpr SvTable() : w{} {
        for (uint32_t i = 0; i < SV_TABLE; ++i) {
            const double z = -(double)i / SV_TABLE * 0.69314718055994530942;
            double sum = 1.0, term = 1.0;
            for (int n = 1; n < 20; ++n) { term *= z / n; sum += term; }
            w[i] = (uint32_t)(sum * 1073741824.0 + 0.5);
        }
    }
};
__device__ const SvTable sv_table{};

// Weights as integers.  With C = 1024 / (T ln 2), 1024 log2 of a weight is max C - x C.  max C is once split into the nearest integer
// and a rest; of -x C the nearest integer n comes from one fma whose sum has no room for a fraction, the rest from a second
// one, exact but for its own rounding (2^-26), and the low word of C.  2^-(k + i/1024 + r/1024) = 2^-k 2^(-i/1024) (1 - q): the
// table's entry i, an integer k, and |r| <= 1.3, for which three terms of the series leave 1e-14.  A weight is known to 5e-10 of
// itself (the table's and the product's 30 bits), so what is drawn changes with probability 1e-7 or so.  What the last unit cuts
// off is half a unit in the mean: the weights are odd numbers of half units.  (Fewer instructions than with max - x in two words,
// and those on floats two at a time: 64 rows of 262144, all weights once: 63 -> 55 us.)
struct SvWeights {
    const uint32_t* table;
    float mx, low, c_hi, c_lo, rest; int32_t whole; int shift; double c;      // logits up to `low` are no matter of the two fmas
    __device__ __forceinline__ void init(const uint32_t* t, float most, float temperature, int units) {
        table = t; mx = most; shift = units;
        c = 1.4426950408889634074 / (double)temperature;
        const double C = c * SV_TABLE, all = (double)mx * C, limit = 4095.0;
        c_hi = (float)C; c_lo = (float)(C - (double)c_hi);
        const bool fine = fabs(all) < limit * SV_TABLE && c < 1e30;
        whole = fine ? __double2int_rn(all) : 0;
        rest = fine ? (float)(all - (double)whole) : 0.f;
        const double per = 0.69314718055994530942 * (double)temperature;       // a halving of the weight
        low = fine ? (float)fmax((double)mx - ((double)shift - 0.5) * per, -limit * per) : INFINITY;
    }
    __device__ __noinline__ static uint64_t special(float x, float mx, double c, int shift) {       // far below, not a number, or a product that is too large
        if (x == mx) return 1ull << shift | 1u;
        if (!(x < mx) || mx > 3.402823466e+38f) return 0;
        const double y = ((double)mx - (double)x) * c;
        return y < (double)shift ? (uint64_t)(exp2(-y) * (double)(1ull << shift)) | 1u : 0;
    }
    __device__ __forceinline__ uint64_t units(float t, float cut) const {
        constexpr float MAGIC = 12582912.f;
        const int32_t ti = __float_as_int(t) - __float_as_int(MAGIC) + whole;
        const int w = (int)table[ti & (SV_TABLE - 1)];
        return ((uint64_t)(uint32_t)(w + __mulhi(w, __float_as_int(cut) - __float_as_int(MAGIC))) << 33) >> (63 - shift + (ti >> 10)) | 1u;
    }
    __device__ __forceinline__ void pair(float2 x, uint64_t& a, uint64_t& b) const {         // both above `low`
        constexpr float MAGIC = 12582912.f, K = 0.69314718055994530942f / SV_TABLE;     // 1.5 x 2^23: sums with it are integers
        const float2 minus = make_float2(-x.x, -x.y), ch = make_float2(c_hi, c_hi);
        const float2 t = sv_fma2(minus, ch, make_float2(MAGIC, MAGIC)), n = sv_add2(t, make_float2(-MAGIC, -MAGIC));
        const float2 r = sv_add2(sv_fma2(minus, ch, make_float2(-n.x, -n.y)), sv_fma2(minus, make_float2(c_lo, c_lo), make_float2(rest, rest)));
        // q 2^32 = -(z - z^2 / 2 + z^3 / 6) 2^32,  z = K r
        constexpr float TWO32 = 4294967296.f;
        float2 q = sv_fma2(r, make_float2(-K * K * K / 6.f * TWO32, -K * K * K / 6.f * TWO32), make_float2(K * K / 2.f * TWO32, K * K / 2.f * TWO32));
        q = sv_fma2(r, q, make_float2(-K * TWO32, -K * TWO32));
        q = sv_fma2(r, q, make_float2(MAGIC, MAGIC));
        a = units(t.x, q.x);
        b = units(t.y, q.y);
    }
    __device__ __forceinline__ uint64_t operator()(float x) const {
        if (!(x > low)) return special(x, mx, c, shift);
        uint64_t a, b;
        pair(make_float2(x, x), a, b);
        return a;
    }
    __device__ __forceinline__ void four(const float4& x, uint64_t (&w)[4]) const {
        if (x.x > low && x.y > low && x.z > low && x.w > low) {
            pair(make_float2(x.x, x.y), w[0], w[1]);
            pair(make_float2(x.z, x.w), w[2], w[3]);
        } else {
            const float v[4] = {x.x, x.y, x.z, x.w};
#pragma unroll 1
            for (int j = 0; j < 4; ++j) {
                const uint64_t y = (*this)(j < 2 ? (j ? v[1] : v[0]) : (j > 2 ? v[3] : v[2]));
                if (j == 0) w[0] = y; else if (j == 1) w[1] = y; else if (j == 2) w[2] = y; else w[3] = y;
            }
        }
    }
};

struct SvBins { uint32_t n[SV_BINS], lo[SV_BINS], hi[SV_BINS]; };      // counts; sums in two words (64-bit shared atomics are loops)
struct SvShared {
    union { SvBins own; uint64_t list[SV_FEW]; };     // the CTA's histogram; the first CTA's candidates
    union { SvBins all; uint64_t w[SV_FEW]; };        // its share of the cluster's bins, merged; the candidates' weights
    uint32_t table[SV_TABLE];
    uint64_t seg_v, pass_v, all_v, above_v;           // weight of that share; of what is kept, of all, of the bins ahead of the window
    uint64_t kmin, kmax, least;                       // of the crossing bin; the last that is kept
    uint32_t n_list, first, found, n_gather; float max;
    uint64_t sub_v[SV_SUBS], wv[SV_W];
    float wmax[SV_W];
    uint64_t hit_above, hit_v; uint32_t hit_bin, hit_n, hit_upto;         // hit_upto: how many logits up to the end of the bin
    uint64_t peer_v[16]; uint32_t seg_n, peer_n[16];
};

// The first m of the list into falling order by the whole CTA; zeros go last.  Up to 128 by counting the larger ones; beyond
// that a bitonic network whose exchanges inside a warp need no wait (350 candidates, twice: 9 -> 2 us).
__device__ __forceinline__ void sv_sort(uint64_t* key, uint32_t m) {
    const uint32_t tid = threadIdx.x;
    __syncthreads();
    if (m <= 128) {
        const uint64_t mine = tid < m ? key[tid] : 0;
        uint32_t r = 0;
        if (mine)
#pragma unroll 8
            for (uint32_t j = 0; j < m; ++j) r += key[j] > mine;
        __syncthreads();
        if (tid < m) key[tid] = 0;
        __syncthreads();
        if (mine) key[r] = mine;
        __syncthreads();
        return;
    }
    uint32_t n = 256;
    while (n < m) n <<= 1;
    for (uint32_t i = m + tid; i < n; i += SV_T) key[i] = 0;
    for (uint32_t size = 32; size <= n; size <<= 1) {
        for (uint32_t half = size >> 1; half >= 32; half >>= 1) {
            __syncthreads();
            for (uint32_t t = tid; t < n / 2; t += SV_T) {
                const uint32_t i = 2 * t - (t & (half - 1)), j = i + half;
                const uint64_t x = key[i], y = key[j];
                if ((x < y) == ((i & size) == 0)) { key[i] = y; key[j] = x; }
            }
        }
        __syncthreads();
        for (uint32_t i = tid; i < n; i += SV_T) {       // whole warps: n and SV_T are multiples of 32
            uint64_t x = key[i];
            for (uint32_t sz = size == 32 ? 2 : size; sz <= size; sz <<= 1)
                for (uint32_t half = min(sz >> 1, 16u); half > 0; half >>= 1) {
                    const uint64_t y = __shfl_xor_sync(0xffffffffu, x, half);
                    const bool larger = ((i & half) == 0) == ((i & sz) == 0);      // this one of the two keeps the larger
                    x = larger == (x > y) ? x : y;
                }
            key[i] = x;
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
    auto together = [&]() { if (C == 1) __syncthreads(); else cl.sync(); };
    const uint64_t ol = a.l_logits[row], ou = a.l_u[row], od = a.l_dst[row];
    const adam_b200_sample_rule rule = a.rules[row];
    const bool lead = rank == 0 && tid == 0;
    if (ol + a.V > a.n_el || ou >= a.n_el || od >= a.n_el) { if (lead) atomicOr(a.err, DEVERR_OOB_MAP); return; }
    const float u = a.map[ou];
    for (uint32_t i = tid; i < SV_TABLE; i += SV_T) s.table[i] = sv_table.w[i];
    const uint32_t base = rank * a.chunk, n = base < a.V ? min(a.chunk, a.V - base) : 0u;
    const float* src = a.map + ol + base;
    const bool aligned = ((ol + base) & 3) == 0;
    const float* const at = RES ? sx : src;
    // f(logit, its place in the CTA's share) for each, in no order.  A NaN fails every comparison below, like what is not kept.
    // After a cut that leaves few of a streamed row, only those that may still be kept.
    bool gathered = false;
    float* const gx = sx;
    uint32_t* const gi = reinterpret_cast<uint32_t*>(sx + SV_GATHER);
    auto each = [&](auto f) {
        if (!RES && gathered) {
            for (uint32_t i = tid; i < s.n_gather; i += SV_T) f(gx[i], gi[i]);
            return;
        }
        if (RES || aligned) {
            const float4* v4 = reinterpret_cast<const float4*>(at);
            const uint32_t n4 = n / 4;
#pragma unroll 2                                     // (by fours the code that a short row fetches once costs more)
            for (uint32_t i = tid; i < n4; i += SV_T) {
                const float4 v = v4[i];
                f(v.x, 4 * i); f(v.y, 4 * i + 1); f(v.z, 4 * i + 2); f(v.w, 4 * i + 3);
            }
            if (tid < n % 4) f(at[4 * n4 + tid], 4 * n4 + tid);
        } else {
#pragma unroll 8
            for (uint32_t i = tid; i < n; i += SV_T) f(at[i], i);
        }
    };

    // ---- the largest logit ----
    float mx = -INFINITY;
    if (RES && aligned) {
        const uint32_t n4 = n / 4;
#pragma unroll 4
        for (uint32_t i = tid; i < n4; i += SV_T) {
            const float4 v = reinterpret_cast<const float4*>(src)[i];
            reinterpret_cast<float4*>(sx)[i] = v;
            mx = fmaxf(fmaxf(mx, fmaxf(v.x, v.y)), fmaxf(v.z, v.w));
        }
        if (tid < n % 4) { const float v = src[4 * n4 + tid]; sx[4 * n4 + tid] = v; mx = fmaxf(mx, v); }
    } else if (RES) {
#pragma unroll 8
        for (uint32_t i = tid; i < n; i += SV_T) { const float v = src[i]; sx[i] = v; mx = fmaxf(mx, v); }
    } else
        each([&](float x, uint32_t) { mx = fmaxf(mx, x); });
    if (!(u >= 0.f && u < 1.f) || rule.temperature != rule.temperature || rule.top_p != rule.top_p || rule.min_p != rule.min_p) {
        if (lead) { a.map[od] = -1.f; atomicOr(a.err, DEVERR_BAD_RULE); }
        return;
    }
    mx = warp_max(mx);
    if (lane == 0) s.wmax[warp] = mx;
    if (tid == 0) { s.n_list = 0; s.first = 0xffffffffu; s.n_gather = 0; }
    __syncthreads();
    if (warp == 0) {
        mx = warp_max(s.wmax[lane]);
        if (lane == 0) s.max = mx;
    }
    together();
    mx = warp_max(lane < C ? *cl.map_shared_rank(&s.max, lane) : -INFINITY);
    if (mx == -INFINITY || !(rule.temperature > 0.f)) {         // nothing to draw, or the first of the largest: the cluster agrees
        if (mx == -INFINITY) { if (lead) a.map[od] = -1.f; }
        else {
            uint32_t i0 = 0xffffffffu;
            each([&](float x, uint32_t i) { if (x == mx) i0 = min(i0, i); });
            i0 = __reduce_min_sync(0xffffffffu, i0);
            if (lane == 0 && i0 != 0xffffffffu) atomicMin(cl.map_shared_rank(&s.first, 0), base + i0);
        }
        together();
        if (lead && mx != -INFINITY) a.map[od] = (float)s.first;
        return;
    }
    SvWeights weight;
    weight.init(s.table, mx, rule.temperature, a.shift);
    const float step = 64.0f / rule.temperature;
    auto bin_of = [&](float x) -> uint32_t {
        const float t = (mx - x) * step;
        return t < (float)(SV_BINS - 1) ? __float_as_uint(__fadd_rd(t, 8388608.f)) & (SV_BINS - 1) : x == mx ? 0u : SV_BINS - 1;      // (a conversion takes 8 cycles)
    };

    const uint64_t least = (uint64_t)ceil((double)fminf(fmaxf(rule.min_p, 0.f), 1.f) * (double)weight(mx));      // of min_p

    // ---- the threshold: what is kept are the logits above x_t, and those equal to it up to index i_t ----
    float x_t = -INFINITY;
    uint32_t i_t = 0;
    bool whole = true;                                // no cut yet: all but -infinity (and NaN)
    auto kept = [&](float x, uint32_t i) { return x > x_t || (x == x_t && !whole && base + i <= i_t); };

    // Histograms: counts, or sums of weights, exact ones or near ones (exact in the first SV_NEAR_BINS, 4 temperatures below the
    // largest, where single weights matter; counts times the weight in a bin's middle further down).
    auto clear = [&](SvMode mode) {
        for (uint32_t b = tid; b < (mode == SV_EXACT ? SV_BINS : SV_NEAR_BINS); b += SV_T) { s.own.lo[b] = 0; s.own.hi[b] = 0; }
        for (uint32_t b = tid; b < SV_BINS; b += SV_T) s.own.n[b] = 0;
        __syncthreads();
    };
    auto count = [&](uint32_t b, float x, SvMode mode) {
        atomicAdd(&s.own.n[b], 1u);
        if (mode == SV_EXACT || (mode == SV_NEAR && b < SV_NEAR_BINS)) {
            const uint64_t w = weight(x);
            const uint32_t lo = (uint32_t)w, old = atomicAdd(&s.own.lo[b], lo), hi = (uint32_t)(w >> 32) + (old + lo < old ? 1u : 0u);
            if (hi) atomicAdd(&s.own.hi[b], hi);
        }
    };
    // The cluster's histogram: CTA c ends with the bins c * per .. of all, and their totals.
    const uint32_t per = SV_BINS / C;
    auto merge = [&](SvMode mode) {
        together();
        uint64_t tv = 0;
        if (tid == 0) s.seg_n = 0;
        uint32_t tn = 0;
        for (uint32_t b = tid; b < per; b += SV_T) {
            const uint32_t bin = rank * per + b;
            const bool sums = mode == SV_EXACT || (mode == SV_NEAR && bin < SV_NEAR_BINS);
            uint32_t cn = 0; uint64_t cv = 0;
#pragma unroll 4
            for (uint32_t k = 0; k < C; ++k) {
                const SvBins* h = cl.map_shared_rank(&s.own, k);
                cn += h->n[bin];
                if (sums) cv += (uint64_t)h->lo[bin] + ((uint64_t)h->hi[bin] << 32);
            }
            if (mode == SV_COUNT) cv = cn;
            else if (!sums) cv = cn * (uint64_t)(exp2f((bin + 0.5f) * (-1.4426950408889634f / 64.f)) * (float)(1ull << a.shift));
            s.all.n[b] = cn; s.all.lo[b] = (uint32_t)cv; s.all.hi[b] = (uint32_t)(cv >> 32);
            tv += cv; tn += cn;
        }
        tv = warp_sum_u64(tv);
        tn = __reduce_add_sync(0xffffffffu, tn);
        if (lane == 0) s.wv[warp] = tv;
        __syncthreads();
        if (mode != SV_COUNT && lane == 0 && tn) atomicAdd(&s.seg_n, tn);
        if (warp == 0) {
            tv = warp_sum_u64(s.wv[lane]);
            if (lane == 0) s.seg_v = tv;
        }
        together();
        if (tid < C) { s.peer_v[tid] = *cl.map_shared_rank(&s.seg_v, tid); s.peer_n[tid] = *cl.map_shared_rank(&s.seg_n, tid); }
        __syncthreads();
    };
    // A value of every CTA, added up
    auto add_up = [&](const uint64_t* mine) { return warp_sum_u64(lane < C ? *cl.map_shared_rank(mine, lane) : 0ull); };
    auto total = [&]() { uint64_t v = 0; for (uint32_t k = 0; k < C; ++k) v += s.peer_v[k]; return v; };
    // exclusive sums over the CTA, and the sum of all
    auto scan = [&](uint64_t v, uint64_t& sum) {
        const uint64_t incl = warp_scan_u64(v);
        __syncthreads();
        if (lane == 31) s.wv[warp] = incl;
        __syncthreads();
        const uint64_t ahead = warp_scan_u64(s.wv[lane]);
        sum = __shfl_sync(0xffffffffu, ahead, 31);
        const uint64_t before = __shfl_sync(0xffffffffu, ahead, warp ? warp - 1 : 0);
        return incl - v + (warp ? before : 0ull);
    };
    // The bin in which the running sum reaches `target` (1 .. total), the sum ahead of it, its own and its count, and with `counts` how many
    // logits lie up to its end: in s.hit_*.
    auto cross = [&](uint64_t target, bool counts) {
        uint64_t above = 0, sum; uint32_t seg = 0, n_above = 0;
        while (seg + 1 < C && above + s.peer_v[seg] < target) { n_above += s.peer_n[seg]; above += s.peer_v[seg++]; }
        const SvBins* h = cl.map_shared_rank(&s.all, seg);
        const uint32_t mine = (per + SV_T - 1) / SV_T, b0 = tid * mine;
        uint64_t v = 0, n_mine = 0;
        for (uint32_t b = b0; b < min(b0 + mine, per); ++b) { v += (uint64_t)h->lo[b] + ((uint64_t)h->hi[b] << 32); n_mine += h->n[b]; }
        above += scan(v, sum);
        if (counts) n_above += (uint32_t)scan(n_mine, sum);
        if (above < target && target <= above + v)
            for (uint32_t b = b0; b < min(b0 + mine, per); ++b) {
                const uint64_t x = (uint64_t)h->lo[b] + ((uint64_t)h->hi[b] << 32);
                n_above += h->n[b];
                if (target <= above + x) { s.hit_bin = seg * per + b; s.hit_above = above; s.hit_v = x; s.hit_n = h->n[b]; s.hit_upto = n_above; break; }
                above += x;
            }
        __syncthreads();
    };
    auto share = [&](uint64_t all) {                  // top_p of a sum, rounded up, at least one unit
        const uint64_t p = (uint64_t)((double)fmaxf(rule.top_p, 0.f) * 18446744073709551616.0), t = __umul64hi(p, all) + (p * all != 0 ? 1u : 0u);
        return t ? t : 1ull;
    };
    // A logit into the first CTA's list.  Only as many as were counted come, and those fit; but a streamed row is read again for
    // every pass, and no store may depend on its being what it was.
    auto listed = [&]() { return RES ? s.n_list : min(s.n_list, SV_FEW); };
    auto put = [&](float x, uint32_t i) {
        if (const uint32_t at = atomicAdd(cl.map_shared_rank(&s.n_list, 0), 1u); RES || at < SV_FEW) *cl.map_shared_rank(&s.list[at], 0) = sv_key(x, base + i);
    };
    // The logits for which `take` says so, sorted.
    auto collect = [&](auto take) {
        each([&](float x, uint32_t i) { if (take(x, i)) put(x, i); });
        together();
        if (rank == 0) sv_sort(s.list, listed());
    };
    constexpr int PER = SV_FEW / SV_T;                      // candidates of a thread
    // All candidates in the list: cut by the whole rule and drawn from there.  top_p is a share of `all`, or of the first
    // top_k (all = 0).
    auto few = [&](uint64_t all) {
        const uint32_t m = listed(), cand = rule.top_k > 0 ? min(m, rule.top_k) : m;
        uint64_t w[PER], mine = 0, sum;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const uint32_t i = tid * PER + j;
            w[j] = i < cand ? weight(sv_value(s.list[i])) : 0;
            mine += w[j];
        }
        uint64_t ahead = scan(mine, sum);
        const uint64_t stop = rule.top_p < 1.f ? share(all ? all : sum) : ~0ull;      // kept while the sum ahead is below it
        // the kept ones again, by index
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const uint32_t i = tid * PER + j;
            const bool in = i < cand && (i == 0 || ahead < stop) && w[j] >= least;
            ahead += w[j];
            s.w[i] = w[j];
            if (i < m) s.list[i] = in ? s.list[i] << 32 | i : 0;
        }
        sv_sort(s.list, m);
        mine = 0;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const uint32_t i = tid * PER + j;
            const uint64_t e = i < m ? s.list[i] : 0;
            w[j] = e ? s.w[(uint32_t)e] : 0;
            mine += w[j];
        }
        ahead = scan(mine, sum);
        const uint64_t target = __umul64hi((uint64_t)((double)u * 18446744073709551616.0), sum);
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            if (ahead <= target && target < ahead + w[j]) a.map[od] = (float)(0xffffffffu - (uint32_t)(s.list[tid * PER + j] >> 32));
            ahead += w[j];
        }
    };
    // Sums over stretches of the row, in index order, of what is kept and weighs enough: all of it, or (window) what lies ahead
    // of bin b0; the logits of the bins b0 .. b1 then go into the first CTA's list, and all_v and above_v get the weight of all that
    // is kept and of what lies ahead of b0.
    const uint32_t sub = max(128u, ((a.chunk + SV_SUBS - 1) / SV_SUBS + 127) & ~127u), n_sub = (n + sub - 1) / sub;
    auto value = [&](float x, uint32_t i) -> uint64_t {
        if (!kept(x, i)) return 0;
        const uint64_t w = weight(x);
        return w >= least ? w : 0;
    };
    auto sweep = [&](auto window, uint32_t b0, uint32_t b1) {
        uint64_t t_all = 0, t_above = 0, sum;
        // bin_of(x) < b0, <= b1
        const float t0 = (float)b0, t1 = b1 + 1 < SV_BINS ? (float)(b1 + 1) : INFINITY;
        auto one = [&](float x, uint32_t i, uint64_t w) -> uint64_t {
            if (!kept(x, i)) return 0;
            if constexpr (decltype(window)::value) {
                t_all += w;
                const float t = (mx - x) * step;
                if (!(t < t0) && (x != mx || b0 == 0)) {
                    if (t < t1 || t1 == INFINITY || x == mx) put(x, i);
                    return 0;
                }
                t_above += w;
            }
            return least <= 1 || w >= least ? w : 0;
        };
        if (!RES && gathered) {
            for (uint32_t b = tid; b < n_sub; b += SV_T) s.sub_v[b] = 0;
            __syncthreads();
            each([&](float x, uint32_t i) {
                const uint64_t v = one(x, i, weight(x));
                if (v) atomicAdd((unsigned long long*)&s.sub_v[i / sub], (unsigned long long)v);
            });
        } else for (uint32_t b = warp; b < n_sub; b += SV_W) {
            uint64_t v = 0;
            const uint32_t end = min(n, (b + 1) * sub);
            if (RES || aligned) {
#pragma unroll 2
                for (uint32_t i = b * sub + 4 * lane; i + 3 < end; i += 128) {
                    const float4 x = *reinterpret_cast<const float4*>(at + i);
                    uint64_t w[4];
                    weight.four(x, w);
                    v += one(x.x, i, w[0]) + one(x.y, i + 1, w[1]) + one(x.z, i + 2, w[2]) + one(x.w, i + 3, w[3]);
                }
                if (const uint32_t i = (end & ~3u) + lane; i < end) v += one(at[i], i, weight(at[i]));
            } else {
#pragma unroll 4
                for (uint32_t i = b * sub + lane; i < end; i += 32) v += one(at[i], i, weight(at[i]));
            }
            v = warp_sum_u64(v);
            if (lane == 0) s.sub_v[b] = v;
        }
        if constexpr (decltype(window)::value) {
            scan(t_all, sum);
            if (tid == 0) s.all_v = sum;
            scan(t_above, sum);
            if (tid == 0) s.above_v = sum;
        }
        __syncthreads();
    };
    // The last of the sorted list with which the running sum of its weights (or its count) reaches `rest`; false: it does not.
    auto last_of_list = [&](uint64_t rest, bool sums) -> bool {
        uint64_t w[PER], mine = 0, sum;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const uint32_t i = tid * PER + j;
            w[j] = i < s.n_list ? (sums ? weight(sv_value(s.list[i])) : 1ull) : 0;
            mine += w[j];
        }
        uint64_t ahead = scan(mine, sum);
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            if (ahead < rest && rest <= ahead + w[j]) s.least = s.list[tid * PER + j];
            ahead += w[j];
        }
        return rest >= 1 && rest <= sum;
    };
    bool swept = false;
    // The nucleus from counts: they say nearly where its end lies, one pass then has the exact weights and the logits around the
    // end.  1: the token is drawn, 0: it is cut, -1: the end lies elsewhere, or too many logits around it.
    auto nucleus = [&]() -> int {
        clear(SV_NEAR);
        // What all logits below `far` could weigh is less than half the slack of the smallest total: not counted (most of a row that
        // has some logits far above the others).  Neither is the rest of the bin that `far` lies in: what is counted are whole bins, so
        // that the bins b0 .. b1 have as many logits as the counts say when the pass below lists them.
        float far = mx - (logf((float)a.V) + 7.65f) * rule.temperature;
        uint32_t bins = max(bin_of(far), 1u);                   // (no other logit as near to the largest as the first bin's: not below 1)
        if (bins >= SV_BINS - 1) { bins = SV_BINS; far = -INFINITY; }          // differences that are not finite, steps of 0
        each([&](float x, uint32_t i) {
            if (x < far || !kept(x, i)) return;                 // below far: in bin `bins` or a later one
            const uint32_t b = bin_of(x);
            if (b < bins) count(b, x, SV_NEAR);
        });
        merge(SV_NEAR);
        const uint64_t near = total(), target = share(near), slack = near >> 10;
        cross(target > slack ? target - slack : 1, true);
        uint32_t b0 = s.hit_bin;
        const uint32_t ahead = s.hit_upto - s.hit_n;
        cross(min(near, target + slack), true);
        const uint32_t b1 = s.hit_bin;
        const uint32_t end = s.hit_upto;
        bool drawn = whole && end <= SV_SHORT;                  // all candidates fit a list that is sorted twice
        if (drawn) b0 = 0;
        else if (end - ahead > SV_FEW) return -1;
        sweep(std::true_type{}, b0, b1);
        together();
        if (rank == 0) {
            const bool fits = s.n_list <= SV_FEW;
            __syncthreads();                                    // read by all before it is set back
            if (fits) sv_sort(s.list, s.n_list);
            const uint64_t all = add_up(&s.all_v), above = add_up(&s.above_v), goal = share(all);
            const bool found = fits && last_of_list(goal > above ? goal - above : 0, true);
            if (found && drawn) few(all);
            if (tid < C) *cl.map_shared_rank(&s.found, tid) = found;       // to everyone's own: who has drawn leaves
            if (tid == 0 && !found) s.n_list = 0;
        }
        together();
        if (!s.found) return -1;
        if (drawn) return 1;
        const uint64_t k = *cl.map_shared_rank(&s.least, 0);
        const uint32_t m = *cl.map_shared_rank(&s.n_list, 0);
        for (uint32_t j = tid; j < m; j += SV_T) {
            const uint64_t e = *cl.map_shared_rank(&s.list[j], 0);
            const uint32_t i = sv_index(e) - base;
            if (e < k || i >= n) continue;
            const uint64_t w = weight(sv_value(e));
            if (w >= least) atomicAdd((unsigned long long*)&s.sub_v[i / sub], (unsigned long long)w);
        }
        __syncthreads();
        x_t = sv_value(k); i_t = sv_index(k); whole = false; swept = true;
        return 0;
    };
    // Cuts what is kept to the run that reaches a target: so many logits (sums false), or so much weight.  True: the token is drawn.
    auto cut = [&](bool sums) __attribute__((always_inline)) -> bool {         // (a call would put all of these on the stack)
        const SvMode mode = sums ? SV_EXACT : SV_COUNT;
        clear(mode);
        each([&](float x, uint32_t i) { if (kept(x, i)) count(bin_of(x), x, mode); });
        merge(mode);
        const uint64_t all = total();
        if (!sums && all <= rule.top_k) return false;
        const uint64_t target = sums ? share(all) : rule.top_k;
        cross(target, sums);
        const uint32_t bin = s.hit_bin;
        uint64_t rest = target - s.hit_above;
        uint32_t in = s.hit_n;
        if (whole && (sums ? s.hit_upto : s.hit_above + s.hit_v) <= SV_FEW) {          // the first CTA sorts all candidates and does the rest
            collect([&](float x, uint32_t) { return x > -INFINITY && bin_of(x) <= bin; });
            if (rank == 0) few(sums ? all : 0);
            return true;
        }
        // The crossing bin, then the crossing one of 2048 equal pieces of the range of its logits' keys, and so on until the first
        // CTA can sort what is left (logits that are all equal are told apart by their indices).
        uint64_t lo = 0, hi = ~0ull;
        bool ranged = false;
        auto inside = [&](float x, uint32_t i) {
            if (!kept(x, i) || bin_of(x) != bin) return false;
            if (!ranged) return true;
            const uint64_t k = sv_key(x, base + i);
            return k >= lo && k <= hi;
        };
        for (int turn = 0; in > SV_FEW && turn < 6; ++turn) {          // (11 of 64 bits each; a row that is written meanwhile may stay above)
            if (!ranged) {
                uint64_t k0 = ~0ull, k1 = 0;
                each([&](float x, uint32_t i) { if (inside(x, i)) { const uint64_t k = sv_key(x, base + i); k0 = min(k0, k); k1 = max(k1, k); } });
                if (tid == 0) { s.kmin = ~0ull; s.kmax = 0; }
                __syncthreads();
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) { k0 = min(k0, __shfl_xor_sync(0xffffffffu, k0, o)); k1 = max(k1, __shfl_xor_sync(0xffffffffu, k1, o)); }
                if (lane == 0) { atomicMin((unsigned long long*)&s.kmin, (unsigned long long)k0); atomicMax((unsigned long long*)&s.kmax, (unsigned long long)k1); }
                together();
                lo = ~0ull; hi = 0;
                for (uint32_t k = 0; k < C; ++k) { lo = min(lo, *cl.map_shared_rank(&s.kmin, k)); hi = max(hi, *cl.map_shared_rank(&s.kmax, k)); }
                ranged = true;
            }
            const int sh = max(0, 64 - __clzll(hi - lo) - (11));
            clear(mode);
            each([&](float x, uint32_t i) { if (inside(x, i)) count((uint32_t)((hi - sv_key(x, base + i)) >> sh), x, mode); });
            merge(mode);
            cross(rest, false);
            in = s.hit_n; rest -= s.hit_above;
            hi -= (uint64_t)s.hit_bin << sh;
            const uint64_t span = (1ull << sh) - 1u;
            lo = hi - lo > span ? hi - span : lo;
        }
        // (for a streamed row of the bins up to the crossing one all that there is, if it is not too much)
        if (!RES && !gathered) {
            collect([&](float x, uint32_t i) {
                if (x > -INFINITY && bin_of(x) <= bin) {
                    const uint32_t at = atomicAdd(&s.n_gather, 1u);
                    if (at < SV_GATHER) { gx[at] = x; gi[at] = i; }
                }
                return inside(x, i);
            });
            gathered = s.n_gather <= SV_GATHER;          // (behind the wait of all)
        } else collect(inside);
        if (rank == 0) {
            last_of_list(rest, sums);
            __syncthreads();
            if (tid == 0) s.n_list = 0;
        }
        together();
        const uint64_t k = *cl.map_shared_rank(&s.least, 0);
        x_t = sv_value(k); i_t = sv_index(k); whole = false;
        return false;
    };
    if (rule.top_k > 0 && rule.top_k < a.V && cut(false)) return;
    if (rule.top_p < 1.f) {
        // a weight for every logit twice, here and in the draw, costs less than nucleus() where a CTA has few of them
        // (a row of 32003 on eight CTAs 17 against 25 us; 64 rows of 262144 on two each 153 against 111)
        const int done = RES ? -1 : nucleus();
        if (done > 0 || (done < 0 && cut(true))) return;
    }

    // ---- the draw: the stretch that holds the token, then the token ----
    if (!swept) {
        __syncthreads();                              // the table, where nothing was cut
        sweep(std::false_type{}, 0, 0);
    }
    if (warp == 0) {
        uint64_t v = 0;
        for (uint32_t b = lane; b < n_sub; b += 32) v += s.sub_v[b];
        v = warp_sum_u64(v);
        if (lane == 0) s.pass_v = v;
    }
    together();
    const uint64_t share_v = lane < C ? *cl.map_shared_rank(&s.pass_v, lane) : 0, before = warp_sum_u64(lane < rank ? share_v : 0), all = warp_sum_u64(share_v);
    const uint64_t target = __umul64hi((uint64_t)((double)u * 18446744073709551616.0), all);     // the running sum to be exceeded
    if (before <= target && target < before + s.pass_v && warp == 0) {
        uint64_t v[SV_SUBS / 32], mine = 0;                        // lane l: stretches 8 l ..
#pragma unroll
        for (int j = 0; j < (int)SV_SUBS / 32; ++j) { const uint32_t b = lane * (SV_SUBS / 32) + j; v[j] = b < n_sub ? s.sub_v[b] : 0; mine += v[j]; }
        uint64_t ahead = before + warp_scan_u64(mine) - mine;
        uint32_t hit = 0xffffffffu;
#pragma unroll
        for (int j = 0; j < (int)SV_SUBS / 32; ++j) { if (hit == 0xffffffffu && ahead + v[j] > target) hit = lane * (SV_SUBS / 32) + j; if (hit == 0xffffffffu) ahead += v[j]; }
        const uint32_t who = __ffs(__ballot_sync(0xffffffffu, hit != 0xffffffffu)) - 1u;
        const uint32_t b = __shfl_sync(0xffffffffu, hit, who);
        ahead = __shfl_sync(0xffffffffu, ahead, who);
        for (uint32_t i0 = b * sub; i0 < (b + 1) * sub; i0 += 32) {
            const uint32_t i = i0 + lane;
            const uint64_t w = i < n ? value(at[i], i) : 0, incl = ahead + warp_scan_u64(w);
            const uint32_t over = __ballot_sync(0xffffffffu, incl > target);
            if (over) {
                if (lane == (uint32_t)__ffs(over) - 1u) a.map[od] = (float)(base + i);
                break;
            }
            ahead = __shfl_sync(0xffffffffu, incl, 31);
        }
    }
    together();                                       // nobody leaves while its shared memory is read
}

template <bool RES>
static int launch_sample(const SampleArgs& a, uint32_t rows, uint32_t C) {
    constexpr size_t fixed = (sizeof(SvShared) + 15) / 16 * 16;
    static bool set = false;
    if (!set) {
        if (cudaFuncSetAttribute((const void*)k_sample_vocab<RES>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(fixed + (RES ? SV_RESIDENT * 4 : SV_GATHER * 8))) != cudaSuccess ||
            cudaFuncSetAttribute((const void*)k_sample_vocab<RES>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)
            return fail(ADAMAH_ERR_BACKEND, "sample: cannot set the kernel's limits");
        set = true;
    }
    launch_k_cluster(k_sample_vocab<RES>, dim3(rows * C), dim3(SV_T), fixed + (RES ? (size_t)a.chunk * 4 : SV_GATHER * 8), g.stream, false, C, false, a);
    count_launch();
    return check_launch("map_sample");
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
    const int rc = a.chunk <= SV_RESIDENT ? launch_sample<true>(a, n_rows, C) : launch_sample<false>(a, n_rows, C);
    end_of_op();
    return rc;
}
