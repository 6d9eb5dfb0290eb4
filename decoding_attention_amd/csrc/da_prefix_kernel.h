// Single-query attention behind a shared prefix (wave64, gfx950).
//
//   o[b,h] = softmax_j(scale <q[b,h], K[j]> + slope_h (j - last_b)) V,   j over the prefix, then over sequence b's own tokens
//
// A prefix token serves the query rows of all sequences: for one KV head they are batch * ratio rows, and the prefix is a
// matrix problem (4 flops per row, token and column) where the own tokens are a memory stream (each K/V row serves `ratio`
// rows).  One launch holds both kinds of work-group, so that the stream fills the memory time and the matrix work the rest:
//   * the first prefix_wgs take (KV head, 128 query rows, prefix split);
//   * the others take (sequence, KV heads, split) of the own tokens, with gqa_segment, the grouped kernel's body.
// Both leave un-normalised partials (o, m, l); the merge kernel adds them up: with M = max m_i,
//   o = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i.
//
// A prefix work-group: wave w holds Q rows 32 w .. + 31 in registers as B-operands of v_mfma_f32_32x32x16.  K and V tiles
// go from global memory straight to LDS, two buffers, the next tile in flight behind the one being used.  Per tile
//   S^T[tok x 32 rows] = K . Q^T       (A: K rows from LDS, 16 bytes a lane)
//   P^T = 2^(S^T scale - m)            one row per lane pair (lane, lane + 32): sums and maxima stay in the lane
//   O^T[col x 32 rows] += V^T . P^T    (A: V through transposed LDS reads; P^T is a B-operand as it lies)
// The k order of the second product is the score tile's: lane half h holds tokens 4 h .. + 3 and 8 + 4 h .. + 3 of every
// sixteen.
#pragma once
#include "da_gqa_mfma.h"
#include "da_mla_dev.h"
#include "da_prefix.h"

namespace da {
namespace prefix {

// 16-byte chunk `c` of row `r` of a tile lies in slot swizzle(r, c) of the row: sixteen consecutive rows at one chunk (K),
// and four rows at four consecutive chunks (V), fall into different banks.
template <int D>
__device__ __forceinline__ int swizzle(int r, int c) {
    if constexpr (D == 64) {  // two rows to the 256 bytes of the banks: bits 1 .. 3 of the row, reversed
        return c ^ (((r >> 1) & 1) << 2 | ((r >> 2) & 1) << 1 | ((r >> 3) & 1));
    } else if constexpr (D == 96) {  // twelve chunks: no XOR stays inside the row
        const int s = c + ((r >> 2) & 3);
        return s >= 12 ? s - 12 : s;
    } else {
        return c ^ mla::swz_a(r);
    }
}
// the row whose slot `s` this is holds chunk unswizzle(r, s) there
template <int D>
__device__ __forceinline__ int unswizzle(int r, int s) {
    if constexpr (D == 96) {
        const int c = s - ((r >> 2) & 3);
        return c < 0 ? c + 12 : c;
    } else {
        return swizzle<D>(r, s);
    }
}

template <typename Tag, int D>
__device__ __forceinline__ void prefix_segment(const PrefixParams& p, uint8_t* const smem, const int hk, const int row0,
                                               const int split) {
    using MM = mla::Mma<Tag>;
    using EL = Elem<Tag>;
    using vec8 = typename MM::vec8;
    constexpr int TT = prefix_tile<D>(), TB = TT / 32;
    constexpr int KS = D / 16, CB = D / 32;
    constexpr int PITCH = D * 2, CPR = D / 8;
    constexpr int TILE = TT * PITCH;           // bytes of a K (or V) tile
    constexpr int LOADS = TILE / 4096;         // 1 KiB loads of a wave per tile and buffer
    constexpr float kLazy = 8.0f;              // the running maximum moves only when exceeded by this much (log2 units)
    static_assert(TILE % 4096 == 0, "whole loads");

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 31, h = lane >> 5;
    const SweepParams& w = p.own;

    const int c0 = split * p.chunk, c1 = min(p.prefix_len, c0 + p.chunk);
    // this lane's query row: number `row` among the KV head's; rows past the last one repeat it and are not stored
    const int row = row0 + wave * 32 + n;
    const bool live = row < p.rows;
    const int rr = min(row, p.rows - 1);
    const int b = rr / w.ratio, hq = hk * w.ratio + (rr - b * w.ratio);
    const uint16_t* const qrow = reinterpret_cast<const uint16_t*>(w.q) + ((size_t)b * w.head_q + hq) * D;
    vec8 q[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) q[ks] = __builtin_bit_cast(vec8, *reinterpret_cast<const uint4*>(qrow + ks * 16 + h * 8));
    float slope = 0.0f;
    int last = 0;  // position of the row's query token
    if (w.is_alibi) {
        slope = alibi_slope_log2(w.slopes, hq, w.head_q);
        last = (p.table ? w.seq_lens[b] : p.prefix_len + w.cu_seq_k[b + 1] - w.cu_seq_k[b]) - 1;
    }

    // Tile loads: load i of a wave fills bytes [(wave * LOADS + i) KiB, + 1 KiB) of the tile, 16 bytes a lane; which row
    // and chunk that is follows from the swizzle.  Tokens past the split's end repeat its last one and are masked.
    int trow[LOADS], tcol[LOADS], page[LOADS];
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        const int at = (wave * LOADS + i) * 64 + lane;  // 16-byte slot of the tile
        trow[i] = at / CPR;
        tcol[i] = unswizzle<D>(trow[i], at - trow[i] * CPR) * 8;
    }
    const uint16_t* const kbase = reinterpret_cast<const uint16_t*>(p.k) + (size_t)hk * D;
    const uint16_t* const vbase = reinterpret_cast<const uint16_t*>(p.v) + (size_t)hk * D;
    auto look_up = [&](int tok0) __attribute__((always_inline)) {
        if (p.table == nullptr) return;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) page[i] = p.table[min(tok0 + trow[i], c1 - 1) >> w.page_shift];
    };
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)smem;
    auto load = [&](int tok0, uint32_t buf) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int tok = min(tok0 + trow[i], c1 - 1);
            int64_t ko, vo;
            if (p.table == nullptr) {
                ko = (int64_t)tok * w.k_row + tcol[i];
                vo = ko;
            } else {
                const int64_t in = (int64_t)(tok & ((1 << w.page_shift) - 1)) * w.k_row + tcol[i];
                ko = (int64_t)page[i] * w.k_page + in;
                vo = (int64_t)page[i] * w.v_page + in;
            }
            const uint32_t to = buf + (wave * LOADS + i) * 1024;
            mla::lds_dma16_v(kbase + ko, to);
            mla::lds_dma16_v(vbase + vo, to + TILE);
        }
    };

    f32x16 acc[CB];
#pragma unroll
    for (int cb = 0; cb < CB; ++cb)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[cb][i] = 0.0f;
    float m = kNegBig, l = 0.0f;

    // LDS addresses of this lane: K row n (+ 32 per block) at every k-step, V^T of rows 4 h + (lane >> 2 & 3)
    const uint8_t* const tile0 = smem;
    const int vr = h * 4 + ((lane >> 2) & 3);
    const int vcol = ((lane >> 4) & 1) * 16 + (lane & 3) * 4;  // first of the lane's four columns in a block of 32

    look_up(c0);
    load(c0, lds0);
    look_up(min(c0 + TT, c1 - 1));
    const int ntiles = (c1 - c0 + TT - 1) / TT;
    for (int t = 0; t < ntiles; ++t) {
        const int tok0 = c0 + t * TT;
        // this wave's share of tile t has landed and its reads of tile t - 1 are done; after the barrier, everyone's
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (t + 1 < ntiles) {
            load(tok0 + TT, lds0 + ((t + 1) & 1) * (2 * TILE));
            look_up(min(tok0 + 2 * TT, c1 - 1));
        }
        const uint8_t* const kt = tile0 + (t & 1) * (2 * TILE);
        const uint8_t* const vt = kt + TILE;

        f32x16 s[TB];
#pragma unroll
        for (int tb = 0; tb < TB; ++tb) {
#pragma unroll
            for (int i = 0; i < 16; ++i) s[tb][i] = 0.0f;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const int r = tb * 32 + n;
                const vec8 kf = *reinterpret_cast<const vec8*>(kt + r * PITCH + swizzle<D>(r, ks * 2 + h) * 16);
                s[tb] = MM::mma(kf, q[ks], s[tb]);
            }
        }

        // x = score in log2 units; element i of block tb is token tok0 + 32 tb + 8 (i / 4) + 4 h + i % 4
        const bool tail = tok0 + TT > c1;
        if (w.is_alibi || tail) {
            const float at = (float)(tok0 + 4 * h - last);  // (whole numbers below 2^24: exact)
#pragma unroll
            for (int tb = 0; tb < TB; ++tb)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int j = tb * 32 + (i >> 2) * 8 + (i & 3);
                    float x = s[tb][i] * w.scale_log2 + slope * (at + (float)j);
                    if (tok0 + 4 * h + j >= c1) x = -INFINITY;
                    s[tb][i] = x;
                }
        } else {
#pragma unroll
            for (int tb = 0; tb < TB; ++tb)
#pragma unroll
                for (int i = 0; i < 16; ++i) s[tb][i] *= w.scale_log2;
        }
        float mx = -INFINITY;
#pragma unroll
        for (int tb = 0; tb < TB; ++tb)
#pragma unroll
            for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[tb][i]);
        mx = max_xor32(mx);
        const bool up = mx > m + kLazy;
        if (__any(up)) {
            const float mn = up ? mx : m;
            const float alpha = fast_exp2(m - mn);
            m = mn;
            l *= alpha;
#pragma unroll
            for (int cb = 0; cb < CB; ++cb) acc[cb] *= alpha;
        }
        vec8 pf[TB * 2];
        constexpr uint32_t kOnes = std::is_same<Tag, f16_tag>::value ? 0x3C003C00u : 0x3F803F80u;
#pragma unroll
        for (int tb = 0; tb < TB; ++tb)
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
                uint32_t pw[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float lo = fast_exp2(s[tb][kk * 8 + 2 * j] - m), hi = fast_exp2(s[tb][kk * 8 + 2 * j + 1] - m);
                    pw[j] = EL::pack2(lo, hi);
                    // (the denominator sums the probabilities as the second product sees them)
                    l = EL::dot2(pw[j], kOnes, l);
                }
                pf[tb * 2 + kk] = __builtin_bit_cast(vec8, make_uint4(pw[0], pw[1], pw[2], pw[3]));
            }

        typedef __attribute__((address_space(3))) s16x4_t* lds_s4;
#pragma unroll
        for (int k = 0; k < TB * 2; ++k) {
#pragma unroll
            for (int cb = 0; cb < CB; ++cb) {
                const int r0 = k * 16 + vr, r1 = r0 + 8, c = cb * 4 + (vcol >> 3), in = (vcol & 4) * 2;
                const s16x4_t a = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (lds_s4)(vt + r0 * PITCH + swizzle<D>(r0, c) * 16 + in));
                const s16x4_t d = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (lds_s4)(vt + r1 * PITCH + swizzle<D>(r1, c) * 16 + in));
                const s16x8_t both = __builtin_shufflevector(a, d, 0, 1, 2, 3, 4, 5, 6, 7);
                acc[cb] = MM::mma(__builtin_bit_cast(vec8, both), pf[k], acc[cb]);
            }
        }
    }

    l += __shfl_xor(l, 32);
    if (!live) return;
    const size_t part = (size_t)split * w.batch * w.head_q + (size_t)b * w.head_q + hq;
    float* const out = p.ws_o + part * D + h * 4;
#pragma unroll
    for (int cb = 0; cb < CB; ++cb)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            *reinterpret_cast<f32x4*>(out + cb * 32 + i * 8) =
                f32x4{acc[cb][4 * i], acc[cb][4 * i + 1], acc[cb][4 * i + 2], acc[cb][4 * i + 3]};
    if (h == 0) *reinterpret_cast<float2*>(p.ws_ml + part * 2) = make_float2(m, l);
}

// Work-groups are numbered so that the row tiles of one (KV head, prefix split) run on one XCD (consecutive work-groups go
// to the eight XCDs in turn) and share its K/V through that XCD's L2; likewise the head groups of one own-token segment.
template <typename Tag, int D, bool WH, int PGM>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(D <= 128 ? 2 : 1))) void prefix_kernel(const PrefixParams p) {
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    const int id = (int)blockIdx.x;
    if (id < p.prefix_wgs) {
        const int slot = id >> 3, rest = slot / p.row_tiles;
        const int g = rest * 8 + (id & 7);  // (KV head, split)
        if (g >= p.own.head_k * p.splits) return;
        const int split = g / p.own.head_k;
        prefix_segment<Tag, D>(p, smem, g - split * p.own.head_k, (slot - rest * p.row_tiles) * kPrefixRows, split);
        return;
    }
    const SweepParams& w = p.own;
    const int i = id - p.prefix_wgs;  // (prefix_wgs is a multiple of 8)
    int grp = 0, seg = i;
    if (w.groups > 1) {
        const int slot = i >> 3;
        grp = slot % w.groups;
        seg = (slot / w.groups) * 8 + (i & 7);
    }
    const int ny = p.own_groups / w.groups;
    const int by = (seg % ny) * w.groups + grp;
    const int rest = seg / ny;
    const int split = rest % w.nsplit, b = rest / w.nsplit;
    if (b >= w.batch) return;  // (the last eight of several head groups)
    int start, len;
    seq_range(w, b, start, len);
    const int own0 = p.table ? p.prefix_len : 0;  // paged: the sequence's positions count the prefix
    const int c0 = own0 + split * w.chunk;
    const int c1 = split == w.nsplit - 1 ? len : min(len, c0 + w.chunk);
    gqa_segment<Tag, D, D, 1, (D <= 256), WH, 0, PGM>(p.own, smem, by, b, start, len, c0, c1,
                                                      (size_t)b * w.head_q * w.nsplit + split, w.nsplit, false);
}

template <typename Tag, int D, bool WH, int PGM>
hipError_t launch_form(const PrefixParams& p, int own_wgs, hipStream_t stream) {
    constexpr size_t tiles = 4 * (size_t)prefix_tile<D>() * D * 2, segment = gqa_lds_bytes<D>(1);
    constexpr size_t lds = tiles > segment ? tiles : segment;
    auto kern = prefix_kernel<Tag, D, WH, PGM>;
    if (lds > 48 * 1024) {
        static std::atomic<uint64_t> devices_done{0};
        const hipError_t e = ensure_lds_limit(reinterpret_cast<const void*>(kern), lds, devices_done);
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL(kern, dim3((unsigned)(p.prefix_wgs + own_wgs)), dim3(256), lds, stream, p);
    return hipGetLastError();
}

template <int D>
hipError_t launch_dim(const PrefixParams& p, bool is_bf16, bool wave_per_head, int own_wgs, hipStream_t stream) {
    // pages of fewer than 32 tokens: own's form that looks up the page of every row
    const bool small = p.own.block_table != nullptr && p.own.page_shift < 5;
    if (is_bf16) {
        if (wave_per_head)
            return small ? launch_form<bf16_tag, D, true, 2>(p, own_wgs, stream) : launch_form<bf16_tag, D, true, 0>(p, own_wgs, stream);
        return small ? launch_form<bf16_tag, D, false, 2>(p, own_wgs, stream) : launch_form<bf16_tag, D, false, 0>(p, own_wgs, stream);
    }
    if (wave_per_head)
        return small ? launch_form<f16_tag, D, true, 2>(p, own_wgs, stream) : launch_form<f16_tag, D, true, 0>(p, own_wgs, stream);
    return small ? launch_form<f16_tag, D, false, 2>(p, own_wgs, stream) : launch_form<f16_tag, D, false, 0>(p, own_wgs, stream);
}

}  // namespace prefix
}  // namespace da
