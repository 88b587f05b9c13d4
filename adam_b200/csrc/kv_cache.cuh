// A paged key / value cache that the operators address by id (adam_b200_kv_*).  Interface of kv_cache.cu.
#pragma once
#include "common.cuh"
#include "kv_pages.h"
#include "token.cuh"

#include <cuda.h>

namespace ab {

constexpr uint32_t MAX_KV = 64;
constexpr uint32_t KV_NO_SEQ = 0xFFFFFFFFu;        // an entry of a batch that stands for no sequence
constexpr uint32_t KV_SPLIT_CTAS = 640;            // attention CTAs with a partial result, at most
constexpr uint32_t KV_SPLIT_ROWS = 64;             // query rows of one

struct KvCache {
    adam_b200_kv_desc d;
    uint32_t elem;                       // bytes of an element
    KvGeom geo;
    void* pool;                          // [n_pages][n_layer][key, value][n_head_kv][page_size][head_dim]
    int32_t* table;                      // [max_seqs][max_pages] page of a sequence's positions, -1 = none
    int32_t* lens;                       // [max_seqs] positions
    int32_t* own_from;                   // [max_seqs] first position that the sequence may write (those before may be others', too)
    float* part;                         // partial results of attention CTAs that share a tile's positions
    unsigned int* tickets;               // arrivals per tile, zero between calls
    CUtensorMap map;                     // the pool as rows of head_dim fp16 values, in boxes of `run` rows of 64 (run = 0: none)
    uint32_t run;                        // positions of a page that a box holds
    KvPages pages;                       // the same on the host, where pages are given out
};

KvCache* get_kv(uint32_t id);            // NULL (+ error text) if absent

// A batch of sequences with their new rows, as the operators get it: entry e is sequence seq[e] with the rows start[e] ..
// start[e + 1] - 1, which are its last positions.
struct KvBatch {
    const uint32_t *seq, *start; uint32_t n_seqs, n_rows;
    const int32_t *lens, *own_from, *table; uint32_t max_seqs;
};

}  // namespace ab
