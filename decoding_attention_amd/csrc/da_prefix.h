// Launch interface of the shared-prefix kernels (da_prefix_kernel.h): one query token per sequence over a prefix that
// all sequences share and each sequence's own tokens behind it.
#pragma once
#include "da_common.h"

namespace da {

constexpr int kPrefixRows = 128;  // query rows of a prefix work-group: 32 for each of its four waves
constexpr int kScanBatch = 1024;  // most sequences whose lengths a work-group adds up in LDS

// The merge: threads that share a row's partials (four columns of it each), and rows of a work-group.  (Four from six partials;
// 4 splits and one own partial of 8192 rows are faster in one.)
constexpr int prefix_merge_shares(int splits, int own_splits) { return splits + own_splits > 5 ? 4 : 1; }
constexpr int prefix_merge_rows(int dim, int shares) { return (dim == 96 ? 8 : 1024 / dim) / shares; }

struct PrefixParams {
    SweepParams own;              // the sequences' own tokens; q, o, slopes, scale and head counts serve the prefix too
    const void* k;                // prefix rows [prefix_len, head_k, dim], or the page pools
    const void* v;
    const int32_t* table;         // page ids of the prefix (null: packed rows); pages as own's pools
    int prefix_len;
    int rows, row_tiles;          // query rows per KV head (batch * ratio), in tiles of kPrefixRows
    int splits, chunk;            // prefix splits and tokens per split (a multiple of the tile)
    int prefix_wgs;               // work-groups in front of own's, a multiple of 8 (see prefix_kernel)
    int spread;                   // row tiles dealt out over all XCDs, not grouped by (KV head, split)
    int own_groups;               // own's work-groups per segment: (head_k or head_k / 4) * own.groups
    int scan;                     // balanced own part over pages: the kernel adds the lengths up itself (flat_cu is written)
    int32_t* flat_out;            // [batch + 1] (scan)
    float* ws_o;                  // [splits, batch * head_q, dim] un-normalised partial outputs
    float* ws_ml;                 // [splits, batch * head_q, 2] running maximum (log2 units) and denominator
};

// wave_per_head: own's form with one KV head to a wave (head_k a multiple of 4).  own_wgs: work-groups behind the prefix's.
hipError_t launch_prefix_d64(const PrefixParams& p, bool is_bf16, bool wave_per_head, int own_wgs, hipStream_t stream);
hipError_t launch_prefix_d96(const PrefixParams& p, bool is_bf16, bool wave_per_head, int own_wgs, hipStream_t stream);
hipError_t launch_prefix_d128(const PrefixParams& p, bool is_bf16, bool wave_per_head, int own_wgs, hipStream_t stream);
hipError_t launch_prefix_d256(const PrefixParams& p, bool is_bf16, bool wave_per_head, int own_wgs, hipStream_t stream);
// the merge of both parts' partials into o
hipError_t launch_prefix_merge(const PrefixParams& p, bool is_bf16, int dim, hipStream_t stream);

}  // namespace da
