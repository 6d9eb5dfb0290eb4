// Launch interface of the K/V cache kernels (da_kv_cache.hip): rows into page pools, quantised on the way, and back.
#pragma once
#include "da_common.h"

namespace da {

// One of the two planes (K or V) of a cache and of the packed rows beside it.
struct KvPlane {
    const void* src;             // append: packed rows, 16-bit; head h of token t starts at t * src_token + h * src_head
    void* dst;                   // read: packed rows [tokens, head_k, dim], 16-bit
    void* pool;                  // [pages, page_size, head_k, dim] elements of the cache's format
    float* scale;                // [head_k] factors (null = 1), or (scale, zero) pairs [pages * page_size, head_k, runs, 2]
    int64_t src_token, src_head; // elements
    int64_t page;                // elements between consecutive pages of the pool
    int dim;
    int aligned;                 // append: every 8 elements of src start at a multiple of 16 bytes
    int narrow;                  // append: a work-group's offsets into src fit 24-bit products and 32-bit sums
    uint32_t lanes_magic;        // ceil(2^32 / lanes of a row): chunk -> head as one multiplication
    uint32_t chunks_magic;       // ceil(2^32 / chunks of a token)
};

struct KvCacheParams {
    KvPlane plane[2];
    const int32_t* block_table;  // [batch, max_blocks]
    const int32_t* seq_lens;     // [batch]
    const int32_t* cu_seq;       // [batch + 1], or null: one token per sequence
    int64_t tokens;
    int batch, head_k, page_shift, max_blocks, num_pages;
    int tokens_per_block;
};

// Tokens of a work-group of 256 threads, from p's tokens, heads and widths.
int kv_cache_tokens_per_block(const KvCacheParams& p, bool read, int fmt, int planes);

// pairs: 0 = a factor per KV head, 1 = a (scale, zero) pair per row, 2 = a pair per 64 elements; fmt: 0, kKvFp8, kKvInt8,
// kKvInt4.  planes: 1 (K alone) or 2.
hipError_t launch_kv_append(const KvCacheParams& p, bool is_bf16, int fmt, int pairs, int planes, hipStream_t stream);
hipError_t launch_kv_read(const KvCacheParams& p, bool is_bf16, int fmt, int pairs, int planes, hipStream_t stream);

}  // namespace da
