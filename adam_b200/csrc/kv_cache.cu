// Paged key / value cache for callers that issue the operators themselves: pages are given out, shared between sequences
// (fork), taken back (truncate) and moved together (compact).
//
// The reference keeps one contiguous cache per engine and copies rows into it (map_row_copy.comp); sharing a prompt between
// several continuations has no counterpart there.
//
// Who holds a page is decided on the host, without a wait for the GPU: the caller names sequences and lengths, so counts of
// holders and the lowest free page are host arithmetic.  What changes on the device (table entries, lengths, copied
// positions) goes there as records in the parameters of one kernel per call, in stream order with the operators that read
// the cache: no host-to-device copy and no synchronisation.  A shared page is copied when a sequence that holds it is
// extended into it, and then only the positions that it has there; the last holder keeps the page itself.
//
// Copies are bound by HBM (every byte read and written once; the same prompt's page read by many continuations comes from
// L2).
#include "kv_cache.cuh"

#include <algorithm>
#include <new>

namespace ab {

constexpr int COPY_T = 256, COPY_U = 8;             // threads of a CTA, 16-byte words of a thread
template <int N>
struct KvParams {
    uint4* pool; int32_t *table, *lens, *own_from;
    uint32_t max_pages, n_copy, n_rec;
    uint32_t row16, plane16, planes;                // 16-byte words of a position and of a page's plane; planes of a page
    size_t page16;
    KvRec r[N];                                     // n_copy copies (pages x, y, z positions), then n_rec records
};

template <int N>
__global__ void __launch_bounds__(COPY_T) k_kv_update(const __grid_constant__ KvParams<N> p) {
    // records: shared out over the CTAs of the first column
    if (blockIdx.x == 0)
        for (uint32_t i = blockIdx.y; i < p.n_rec; i += gridDim.y) {
            const KvRec r = p.r[p.n_copy + i];
            const uint32_t seq = r.x & 0x0FFFFFFFu;
            int32_t* row = p.table + (size_t)seq * p.max_pages;
            switch (r.x >> 28) {
            case REC_RUN: for (uint32_t j = threadIdx.x; j < r.w; j += COPY_T) row[r.y + j] = (int32_t)(r.z + j); break;
            case REC_LEN: if (threadIdx.x == 0) { p.lens[seq] = (int32_t)r.y; p.own_from[seq] = (int32_t)r.z; } break;
            case REC_ROW: for (uint32_t j = threadIdx.x; j < r.w; j += COPY_T) row[j] = p.table[(size_t)r.y * p.max_pages + j]; break;
            default: for (uint32_t j = r.y + threadIdx.x; j < r.z; j += COPY_T) row[j] = -1;
            }
        }
    if (blockIdx.y >= p.n_copy) return;
    const KvRec c = p.r[blockIdx.y];
    const uint32_t per = c.z * p.row16, n = per * p.planes;
    const uint4* src = p.pool + (size_t)c.x * p.page16;
    uint4* dst = p.pool + (size_t)c.y * p.page16;
    const uint32_t i0 = blockIdx.x * (COPY_T * COPY_U) + threadIdx.x;
    uint4 v[COPY_U];
    size_t at[COPY_U];
#pragma unroll
    for (int u = 0; u < COPY_U; ++u) {
        const uint32_t i = i0 + u * COPY_T;
        if (i < n) { at[u] = (size_t)(i / per) * p.plane16 + i % per; v[u] = src[at[u]]; }
    }
#pragma unroll
    for (int u = 0; u < COPY_U; ++u)
        if (i0 + u * COPY_T < n) dst[at[u]] = v[u];
}

template <int N>
static int launch_update(const KvCache& kv, const KvCopy* copies, uint32_t n_copy, const KvRec* recs, uint32_t n_rec) {
    KvParams<N> p;
    p.pool = (uint4*)kv.pool; p.table = kv.table; p.lens = kv.lens; p.own_from = kv.own_from;
    p.max_pages = kv.d.max_pages; p.n_copy = n_copy; p.n_rec = n_rec;
    p.row16 = kv.d.head_dim * kv.elem / 16; p.plane16 = p.row16 * kv.d.page_size; p.planes = kv.d.n_layer * 2 * kv.d.n_head_kv;
    p.page16 = (size_t)p.plane16 * p.planes;
    uint32_t rows = 0;
    for (uint32_t i = 0; i < n_copy; ++i) { p.r[i] = KvRec{copies[i].src, copies[i].dst, copies[i].rows, 0}; rows = std::max(rows, copies[i].rows); }
    for (uint32_t i = 0; i < n_rec; ++i) p.r[n_copy + i] = recs[i];
    const uint64_t words = (uint64_t)rows * p.row16 * p.planes;
    const uint32_t gx = std::max<uint32_t>(1, (uint32_t)((words + COPY_T * COPY_U - 1) / (COPY_T * COPY_U)));
    k_kv_update<N><<<dim3(gx, n_copy ? n_copy : std::min<uint32_t>(n_rec, 64)), COPY_T, 0, g.stream>>>(p);
    count_launch();
    return check_launch("kv_update");
}
static int send(const KvCache& kv, const KvUpdate& u) {
    constexpr uint32_t FEW = 60, SOME = 250, MANY = 1000;        // records of a launch: 1, 4 and 16 KB of parameters
    size_t c = 0, r = 0;
    int rc = ADAMAH_OK;
    while (!rc && (c < u.copies.size() || r < u.recs.size())) {
        const size_t left = u.copies.size() - c + u.recs.size() - r, room = left <= FEW ? FEW : left <= SOME ? SOME : MANY;
        const uint32_t nc = (uint32_t)std::min(u.copies.size() - c, room), nr = (uint32_t)std::min(u.recs.size() - r, room - nc);
        rc = (room == FEW ? launch_update<FEW> : room == SOME ? launch_update<SOME> : launch_update<MANY>)(kv, u.copies.data() + c, nc, u.recs.data() + r, nr);
        c += nc; r += nr;
    }
    end_of_op();
    return rc;
}

static KvCache* g_kv[MAX_KV];

KvCache* get_kv(uint32_t id) {
    if (!ready()) return nullptr;
    if (id >= MAX_KV || !g_kv[id]) { fail(ADAMAH_ERR_NOT_FOUND, "kv cache %u does not exist", id); return nullptr; }
    return g_kv[id];
}

static void release(KvCache* kv) {
    cudaFree(kv->pool); cudaFree(kv->table); cudaFree(kv->lens); cudaFree(kv->part); cudaFree(kv->tickets);
    delete kv;
}
void kv_destroy_all() {
    for (KvCache*& kv : g_kv) if (kv) { release(kv); kv = nullptr; }
}

// The pool for the tensor copies of attn_kv_tc.cu, where a page's positions come in groups of eight (the swizzle's period).
static int make_map(KvCache& kv) {
    const adam_b200_kv_desc& d = kv.d;
    const uint64_t rows = (uint64_t)d.n_pages * kv.geo.page_elems / d.head_dim;
    if (!d.kv_dtype || (d.head_dim != 64 && d.head_dim != 128) || d.page_size % 8 || rows >= (1ull << 31) - 256) return ADAMAH_OK;
    kv.run = 8;
    while (kv.run < 128 && d.page_size % (2 * kv.run) == 0) kv.run *= 2;
    void* entry = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &entry, cudaEnableDefault, &found) != cudaSuccess || !entry)
        return fail(ADAMAH_ERR_BACKEND, "kv_create: the driver has no tensor maps");
    const cuuint64_t dims[2] = {d.head_dim, rows}, strides[1] = {(cuuint64_t)d.head_dim * 2};
    const cuuint32_t box[2] = {64, kv.run}, step[2] = {1, 1};
    const CUresult rc = reinterpret_cast<decltype(&cuTensorMapEncodeTiled)>(entry)(&kv.map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, kv.pool, dims, strides, box, step,
        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return rc == CUDA_SUCCESS ? ADAMAH_OK : fail(ADAMAH_ERR_BACKEND, "kv_create: no tensor map (%d)", (int)rc);
}

static int create(const adam_b200_kv_desc& desc, uint32_t id) {
    adam_b200_kv_desc d = desc;
    if (d.page_size == 0) d.page_size = 64;
    if (d.head_dim != 32 && d.head_dim != 64 && d.head_dim != 128 && d.head_dim != 256)
        return fail(ADAMAH_ERR_INVALID, "kv_create: head_dim %u (32, 64, 128 and 256 are supported)", d.head_dim);
    if (d.kv_dtype > 1) return fail(ADAMAH_ERR_INVALID, "kv_create: kv_dtype %u (0 = float32, 1 = float16)", d.kv_dtype);
    if (!d.n_layer || !d.n_head_kv || !d.n_pages || !d.max_seqs || !d.max_pages) return fail(ADAMAH_ERR_INVALID, "kv_create: empty shape");
    if (d.page_size > 1024 || d.n_head_kv > 1024 || d.n_layer > 4096 || d.n_pages > (1u << 28) || d.max_seqs > (1u << 20) ||
        (uint64_t)d.max_pages * d.page_size >= (1ull << 30) || (uint64_t)d.max_seqs * d.max_pages >= (1ull << 31))
        return fail(ADAMAH_ERR_INVALID, "kv_create: shape out of range");
    const uint64_t plane = (uint64_t)d.page_size * d.head_dim, page_elems = plane * d.n_layer * 2 * d.n_head_kv;
    if (page_elems >= (1ull << 31)) return fail(ADAMAH_ERR_INVALID, "kv_create: a page of %llu elements", (unsigned long long)page_elems);
    KvCache* kv = new KvCache();
    struct Guard { KvCache* kv; ~Guard() { if (kv) release(kv); } } guard{kv};
    kv->d = d; kv->elem = d.kv_dtype ? 2 : 4;
    kv->geo = KvGeom{d.n_layer, d.n_head_kv, d.head_dim, d.page_size, d.max_pages, (size_t)page_elems};
    const size_t entries = (size_t)d.max_seqs * d.max_pages, pool = (size_t)d.n_pages * page_elems * kv->elem;
    kv->pages.init(d.page_size, d.n_pages, d.max_seqs, d.max_pages);
    const size_t part = (size_t)KV_SPLIT_CTAS * KV_SPLIT_ROWS * (d.head_dim + 4) * 4;
    if (cudaMalloc(&kv->pool, pool) != cudaSuccess || cudaMalloc((void**)&kv->table, entries * 4) != cudaSuccess ||
        cudaMalloc((void**)&kv->lens, (size_t)d.max_seqs * 8) != cudaSuccess || cudaMalloc((void**)&kv->part, part) != cudaSuccess ||
        cudaMalloc((void**)&kv->tickets, KV_SPLIT_CTAS * 4) != cudaSuccess) {
        cudaGetLastError();
        return fail(ADAMAH_ERR_MEMORY, "kv_create: out of device memory (%zu bytes of pages)", pool);
    }
    kv->own_from = kv->lens + d.max_seqs;
    if (cudaMemsetAsync(kv->pool, 0, pool, g.stream) != cudaSuccess || cudaMemsetAsync(kv->table, 0xFF, entries * 4, g.stream) != cudaSuccess ||
        cudaMemsetAsync(kv->lens, 0, (size_t)d.max_seqs * 8, g.stream) != cudaSuccess || cudaMemsetAsync(kv->tickets, 0, KV_SPLIT_CTAS * 4, g.stream) != cudaSuccess ||
        cudaStreamSynchronize(g.stream) != cudaSuccess)
        return fail(ADAMAH_ERR_BACKEND, "kv_create: %s", cudaGetErrorString(cudaGetLastError()));
    if (int rc = make_map(*kv)) return rc;
    g_kv[id] = kv;
    guard.kv = nullptr;
    return ADAMAH_OK;
}

bool capturing();
// By adam_b200_capture_begin, or by the owner of a stream that the library was lent: the books would change once, the device with
// every replay.  (Nobody else captures the library's own stream, and the default stream cannot be captured.)
static bool recording() {
    if (capturing()) return true;
    if (g.stream == g.own_stream || g.stream == cudaStreamLegacy) return false;
    cudaStreamCaptureStatus state = cudaStreamCaptureStatusNone;
    if (cudaStreamIsCapturing(g.stream, &state) != cudaSuccess) { cudaGetLastError(); return true; }
    return state != cudaStreamCaptureStatusNone;
}
static int page_op(uint32_t id, const char* name, KvCache** kv) {
    *kv = get_kv(id);
    if (!*kv) return ADAMAH_ERR_NOT_FOUND;
    if (recording()) return fail(ADAMAH_ERR_INVALID, "%s: pages cannot change hands while a graph is being captured", name);
    return ADAMAH_OK;
}
// One call on the pages: the books first, then what changes on the device.  The host's vectors may run out of memory; no
// exception leaves an entry point.
template <typename F>
static int change_pages(uint32_t id, const char* name, F f) {
    KvCache* kv;
    if (int rc = page_op(id, name, &kv)) return rc;
    try {
        KvUpdate u;
        if (const int rc = f(kv->pages, u)) return fail(rc, "%s", kv->pages.why);
        return send(*kv, u);
    } catch (const std::exception&) { return fail(ADAMAH_ERR_MEMORY, "%s: out of host memory", name); }
}

}  // namespace ab

using namespace ab;

extern "C" int adam_b200_kv_create(const adam_b200_kv_desc* desc, uint32_t* id_out) {
    if (!ready()) return ADAMAH_ERR_INVALID;
    if (!desc || !id_out) return fail(ADAMAH_ERR_INVALID, "kv_create: null pointer");
    if (recording()) return fail(ADAMAH_ERR_INVALID, "kv_create: a graph is being captured");
    for (uint32_t id = 0; id < MAX_KV; ++id)
        if (!g_kv[id]) {
            int rc;
            try { rc = create(*desc, id); }
            catch (const std::exception&) { rc = fail(ADAMAH_ERR_MEMORY, "kv_create: out of host memory"); }
            if (!rc) *id_out = id;
            return rc;
        }
    return fail(ADAMAH_ERR_INVALID, "kv_create: %u caches exist", MAX_KV);
}
extern "C" int adam_b200_kv_destroy(uint32_t id) {
    KvCache* kv;
    if (int rc = page_op(id, "kv_destroy", &kv)) return rc;
    cudaStreamSynchronize(g.stream);
    release(kv);
    g_kv[id] = nullptr;
    return ADAMAH_OK;
}
extern "C" int adam_b200_kv_extend(uint32_t id, uint32_t n, const uint32_t* seqs, const uint32_t* n_tokens) {
    return change_pages(id, "kv_extend", [&](KvPages& p, KvUpdate& u) { return p.extend(n, seqs, n_tokens, u); });
}
extern "C" int adam_b200_kv_fork(uint32_t id, uint32_t src, uint32_t n, const uint32_t* dsts, uint32_t n_tokens) {
    return change_pages(id, "kv_fork", [&](KvPages& p, KvUpdate& u) { return p.fork(src, n, dsts, n_tokens, u); });
}
extern "C" int adam_b200_kv_truncate(uint32_t id, uint32_t n, const uint32_t* seqs, const uint32_t* lens) {
    return change_pages(id, "kv_truncate", [&](KvPages& p, KvUpdate& u) { return p.truncate(n, seqs, lens, u); });
}
extern "C" int adam_b200_kv_compact(uint32_t id, uint32_t* n_live_out) {
    uint32_t live = 0;
    const int rc = change_pages(id, "kv_compact", [&](KvPages& p, KvUpdate& u) { return p.compact(&live, u); });
    if (!rc && n_live_out) *n_live_out = live;
    return rc;
}
extern "C" int adam_b200_kv_state(uint32_t id, uint32_t* n_free, int32_t* lens, int32_t* table) {
    KvCache* kv = get_kv(id);
    if (!kv) return ADAMAH_ERR_NOT_FOUND;
    const KvPages& p = kv->pages;
    if (n_free) *n_free = p.n_free;
    if (lens) std::copy(p.lens.begin(), p.lens.end(), lens);
    if (table) std::copy(p.table.begin(), p.table.end(), table);
    return ADAMAH_OK;
}
extern "C" int adam_b200_kv_ptr(uint32_t id, uint32_t which, uint64_t* ptr, uint64_t* n_bytes) {
    KvCache* kv = get_kv(id);
    if (!kv) return ADAMAH_ERR_NOT_FOUND;
    if (which > 2 || !ptr || !n_bytes) return fail(ADAMAH_ERR_INVALID, "kv_ptr: bad arguments");
    *ptr = (uint64_t)(uintptr_t)(which == 0 ? kv->pool : which == 1 ? (void*)kv->table : (void*)kv->lens);
    *n_bytes = which == 0 ? (uint64_t)kv->d.n_pages * kv->geo.page_elems * kv->elem : which == 1 ? (uint64_t)kv->pages.table.size() * 4 : (uint64_t)kv->d.max_seqs * 4;
    return ADAMAH_OK;
}
