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
// A prefix work-group: wave w holds Q rows 32 w .. + 31 in registers as B-operands of v_mfma_f32_32x32x16.  K and V tiles of
// 32 tokens go from global memory straight to LDS, three buffers each, two tiles in flight behind the one being used.  Per tile
//   S^T[tok x 32 rows] = K . Q^T       (A: K rows from LDS, 16 bytes a lane)
//   P^T = 2^(S^T scale - m)            one row per lane pair (lane, lane + 32): sums and maxima stay in the lane
//   O^T[col x 32 rows] += V^T . P^T    (A: V through transposed LDS reads; P^T is a B-operand as it lies)
// The k order of the second product is the score tile's: lane half h holds tokens 4 h .. + 3 and 8 + 4 h .. + 3 of every
// sixteen.  The loop is skewed: the scores of tile u + 1 run beside the exponentials of tile u, and its value products beside
// the next maximum and the K fragments of tile u + 2.  The running maximum moves only when a score exceeds it by 2^8, so that the
// accumulators are rarely rescaled (weights up to 2^8 lose nothing: sums are float32, and P's 16 bits are relative).
// P is rounded to 16 bits for the second product, as everywhere in this library; the denominator sums the rounded values, so
// that a row's weights still add up to one.
//
// What bounds it: the prefix part alone is power-limited matrix work, 256 sequences behind 16384 tokens, 32/8 heads d 128:
// 71 to 73 us, 960 TFLOP/s with two work-groups per CU; with one per CU it is the latency of a tile's chain (0.6 us for 0.25 us of
// products).  With own tokens (542 MB, alone 95 us) the launch takes 135 us at least and 144 to 168 in the median of runs on several
// GPUs, where one part after the other takes 166.  128 rows a work-group: with 64 the K/V reads from LDS per product double, with
// 256 the splits, and so the partials, do.  Wide rows (d 256) leave one work-group per CU and its chain: 1056 rows behind 32768
// tokens 66 us, 540 TFLOP/s; there the partials of a short call (8192 tokens: 18 MB out and back) are more than twice the K/V.
#pragma once
#include "da_gqa_mfma.h"
#include "da_mla_dev.h"
#include "da_prefix.h"

namespace da {
namespace prefix {

// A tile is 32 tokens.  Rows lie kPitch bytes apart and hold their 16-byte chunks XOR-swizzled with the row index, so that
// sixteen consecutive rows at one chunk (K), and four rows at four consecutive chunks (V), fall into different banks.
// (d = 96: twelve chunks and four empty ones, so that a load instruction fills whole rows here too.)
constexpr int kTok = 32;
template <int D>
constexpr int pitch() {
    return D == 96 ? 256 : D * 2;
}
template <int D>
__device__ __forceinline__ int swizzle(int r) {
    if constexpr (D == 64)  // two rows to the 256 bytes of the banks: bits 1 .. 3 of the row, reversed
        return ((r >> 1) & 1) << 2 | ((r >> 2) & 1) << 1 | ((r >> 3) & 1);
    else
        return mla::swz_a(r);
}

// At most N LDS reads outstanding (the other counters untouched).
template <int N>
__device__ __forceinline__ void wait_lds() {
    __builtin_amdgcn_s_waitcnt(0xC07F | (N < 15 ? N : 15) << 8);
}
__device__ __forceinline__ auto join(s16x4_t lo, s16x4_t hi) { return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7); }

template <int D>
constexpr size_t prefix_lds_bytes() {  // three buffers of K tiles and three of V tiles
    return 6 * (size_t)kTok * pitch<D>();
}

// 16 bytes per lane from a wave-uniform address and a per-lane offset straight into LDS at `to` + lane * 16; the wait for it
// is placed by hand.  (Plain loads: the row tiles of a split share its K/V through the L2.)
__device__ __forceinline__ void dma16(const uint8_t* base, uint32_t lane_off, uint32_t to) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(lane_off), "s"(base), "s"(to) : "memory");
}

// x *= alpha in accumulation registers.  d = 256 keeps its accumulators there, which only matrix instructions and moves reach;
// a plain product in a branch has the compiler move all 128 of them out and back in on both ways round it, every tile.
// wait_products() goes in front of the first (a matrix instruction's result before it is read) and behind the last (what is written
// here before a matrix instruction reads it).
__device__ __forceinline__ void wait_products() { asm volatile("s_nop 15\n\ts_nop 15" ::: "memory"); }
__device__ __forceinline__ void scale_acc(f32x16& x, float alpha) {
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
        float a = x[i], b = x[i + 1], c = x[i + 2], d = x[i + 3], t, u;
        asm volatile(
            "v_accvgpr_read_b32 %4, %0\n\tv_accvgpr_read_b32 %5, %1\n\tv_mul_f32 %4, %4, %6\n\tv_mul_f32 %5, %5, %6\n\t"
            "v_accvgpr_write_b32 %0, %4\n\tv_accvgpr_write_b32 %1, %5\n\t"
            "v_accvgpr_read_b32 %4, %2\n\tv_accvgpr_read_b32 %5, %3\n\tv_mul_f32 %4, %4, %6\n\tv_mul_f32 %5, %5, %6\n\t"
            "v_accvgpr_write_b32 %2, %4\n\tv_accvgpr_write_b32 %3, %5"
            : "+a"(a), "+a"(b), "+a"(c), "+a"(d), "=&v"(t), "=&v"(u)
            : "v"(alpha));
        x[i] = a, x[i + 1] = b, x[i + 2] = c, x[i + 3] = d;
    }
}

// Keeps a matrix product where the source has it (d = 256: with this many registers in use the compiler puts the score products
// behind the value products, and all of a tile's LDS reads in front of both).
template <int D>
__device__ __forceinline__ void pin(f32x16& x) {
    if constexpr (D == 256) asm volatile("" : "+a"(x));
}

template <typename Tag, int D, int PGM>
__device__ __forceinline__ void prefix_segment(const PrefixParams& p, uint8_t* const smem, const int hk, const int row0,
                                               const int split) {
    using MM = mla::Mma<Tag>;
    using EL = Elem<Tag>;
    using vec8 = typename MM::vec8;
    constexpr int KS = D / 16, CB = D / 32;
    constexpr int PITCH = pitch<D>(), SLOTS = PITCH / 16, CPR = D / 8;
    constexpr int TILE = kTok * PITCH;   // bytes of a K (or V) tile
    constexpr int LOADS = TILE / 4096;   // 1 KiB loads of a wave per tile
    constexpr int RPL = 1024 / PITCH;    // rows of such a load
    constexpr float kLazy = 8.0f;        // the running maximum moves only when exceeded by this much (log2 units)
    static_assert(TILE % 4096 == 0 && 1024 % PITCH == 0, "whole loads of whole rows");

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 31, h = lane >> 5;
    const SweepParams& w = p.own;

    const int c0 = split * p.chunk, c1 = min(p.prefix_len, c0 + p.chunk);
    const int last = c1 - 1, nu = (c1 - c0 + kTok - 1) / kTok;
    // Tile number u starts at token at0 + u * ahead.  With ALiBi the last tokens come first: their bias is the highest (of
    // positive slopes), and in the other order a steep head would raise its maximum, and rescale, in every tile (33 sequences
    // behind 8192 tokens, 32/1 heads d 256: 88.8 -> 39.4 us; 256 behind 16384, 32/8 heads d 128: 172 -> 155).  They do as well where
    // the split's last tile is cut, so that a cut tile is always the first one and the loop has none to look after.
    const int tile_last = c0 + (nu - 1) * kTok, cut = c1 - tile_last;  // (cut: tokens of the last tile)
    const bool back = w.is_alibi || cut < kTok;
    const int at0 = back ? tile_last : c0, ahead = back ? -kTok : kTok;

    // Tile loads: a wave fills rows 8 w .. 8 w + 7 of every tile, RPL rows an instruction, 16 bytes a lane, from the address of
    // its first row (one page look-up: its rows lie in one page of 8 tokens and more) and per-lane offsets.  Tokens past the
    // split's end repeat its last one; their scores are masked, and their V rows cleared (an infinite value of the last token
    // would be no number under a weight of zero).
    const int lrow = lane / SLOTS, slot = lane % SLOTS;
    const uint32_t row_bytes = (uint32_t)w.k_row * 2;
    const int first_0 = min(at0 + wave * 8, last);
    uint32_t off[LOADS], off_0[LOADS];  // of any tile, and of the first one
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        const int r = wave * 8 + i * RPL + lrow;
        const int c = slot ^ swizzle<D>(r);
        const uint32_t col = (uint32_t)(c < CPR ? c : c - 8) * 16;  // (an empty chunk: any other one of the row)
        off[i] = (uint32_t)(i * RPL + lrow) * row_bytes + col;
        off_0[i] = (uint32_t)(min(at0 + r, last) - first_0) * row_bytes + col;
    }
    const uint8_t* const kbase = reinterpret_cast<const uint8_t*>(p.k) + (size_t)hk * D * 2;
    const uint8_t* const vbase = reinterpret_cast<const uint8_t*>(p.v) + (size_t)hk * D * 2;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)smem + (uint32_t)(wave * LOADS) * 1024;
    typedef const int32_t __attribute__((address_space(4))) * const_i32;
    const const_i32 table = (const_i32)(uintptr_t)p.table;
    const int page_mask = (1 << w.page_shift) - 1;
    // bytes from the pool's (or the packed rows') start to token j, a wave-uniform one
    auto row_at = [&](int j, int64_t page_stride) __attribute__((always_inline)) {
        if (p.table == nullptr) return (int64_t)j * w.k_row * 2;
        return ((int64_t)table[j >> w.page_shift] * page_stride + (int64_t)(j & page_mask) * w.k_row) * 2;
    };
    auto dma_rows = [&](const uint8_t* at, const uint32_t(&o)[LOADS], uint32_t to) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < LOADS; ++i) dma16(at, o[i], lds0 + to + i * 1024);
    };
    // any tile (those past the last one are not fetched); only the first may be cut
    auto load = [&](const uint8_t* base, int64_t page_stride, int u, uint32_t to, auto first_c) __attribute__((always_inline)) {
        if (u >= nu) return;
        const int tok0 = at0 + u * ahead;
        if (PGM != 2 || page_mask >= 7) {
            if constexpr (decltype(first_c)::value)
                dma_rows(base + row_at(first_0, page_stride), off_0, to);
            else
                dma_rows(base + row_at(tok0 + wave * 8, page_stride), off, to);
        } else {  // smaller pages: those of the wave's eight rows, each lane picking its own
            int32_t page[8];
#pragma unroll
            for (int r = 0; r < 8; ++r) page[r] = table[min(tok0 + wave * 8 + r, last) >> w.page_shift];
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                const int j = min(tok0 + wave * 8 + i * RPL + lrow, last);
                int32_t mine = page[i * RPL];
#pragma unroll
                for (int r = 1; r < RPL; ++r) mine = lrow >= r ? page[i * RPL + r] : mine;
                const int64_t at = (int64_t)mine * page_stride + (int64_t)(j & page_mask) * w.k_row;
                const uint32_t col = off[i] - (uint32_t)(i * RPL + lrow) * row_bytes;
                mla::lds_dma16_v(base + at * 2 + col, lds0 + to + i * 1024);
            }
        }
    };
    auto load_k = [&](int u, int buf) __attribute__((always_inline)) { load(kbase, w.k_page, u, buf * TILE, std::false_type{}); };
    auto load_v = [&](int u, int buf) __attribute__((always_inline)) { load(vbase, w.v_page, u, (3 + buf) * TILE, std::false_type{}); };
    // (packed rows: this wave's addresses in the tiles fetched last)
    const int64_t ahead_bytes = (int64_t)ahead * row_bytes;
    const uint8_t* k_next = kbase + (int64_t)(at0 + 3 * ahead + wave * 8) * row_bytes;
    const uint8_t* v_next = vbase + (int64_t)(at0 + ahead + wave * 8) * row_bytes;
    load(kbase, w.k_page, 0, 0, std::true_type{});
    load_k(1, 1);
    load(vbase, w.v_page, 0, 3 * TILE, std::true_type{});
    load_k(2, 2);
    load_v(1, 1);

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
    int end = 0;  // position of the row's query token
    if (w.is_alibi) {
        slope = alibi_slope_log2(w.slopes, hq, w.head_q);
        end = (p.table ? w.seq_lens[b] : p.prefix_len + w.cu_seq_k[b + 1] - w.cu_seq_k[b]) - 1;
    }

    f32x16 acc[CB];
#pragma unroll
    for (int cb = 0; cb < CB; ++cb)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[cb][i] = 0.0f;
    float m = kNegBig, l = 0.0f;

    // LDS offsets of this lane: K row n at every k-step; V rows 4 h + (lane >> 2 & 3) and eight further down, four columns
    // of every block of 32
    int k_at[KS], v_at[CB][2];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) k_at[ks] = n * PITCH + ((ks * 2 + h) ^ swizzle<D>(n)) * 16;
#pragma unroll
    for (int cb = 0; cb < CB; ++cb)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int r = h * 4 + ((lane >> 2) & 3) + 8 * j, c = ((lane >> 4) & 1) * 16 + (lane & 3) * 4;
            v_at[cb][j] = 3 * TILE + r * PITCH + ((cb * 4 + (c >> 3)) ^ swizzle<D>(r)) * 16 + (c & 4) * 2;
        }

    // The score tile of 32 tokens: element i is token 8 (i / 4) + 4 h + i % 4 of the tile, row n.
    f32x16 s;
    float mul = w.scale_log2;  // what takes s to log2 units
    auto scores = [&](const vec8(&kf)[KS]) __attribute__((always_inline)) {
        f32x16 c;
#pragma unroll
        for (int i = 0; i < 16; ++i) c[i] = 0.0f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) c = MM::mma(kf[ks], q[ks], c);
        return c;
    };
    auto max_of = [](const f32x16& x) __attribute__((always_inline)) {
        float mx = x[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) mx = fmaxf(mx, x[i]);
        return mx;
    };
    // ALiBi and (the first tile) the mask of tokens past the end, the running maximum, and (rarely) the rescaling it asks for;
    // mx: max_of(s)
    auto settle_max = [&](int u, float mx, auto first_c) __attribute__((always_inline)) {
        constexpr bool first = decltype(first_c)::value;
        if (first ? back : (bool)w.is_alibi) {
            if (w.is_alibi) {
                const float at = slope * (float)(at0 + u * ahead + 4 * h - end);
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int j = (i >> 2) * 8 + (i & 3);
                    s[i] = __builtin_fmaf(s[i], w.scale_log2, __builtin_fmaf(slope, (float)j, at));
                }
                mul = 1.0f;
            }
            if constexpr (first) {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (4 * h + (i >> 2) * 8 + (i & 3) >= cut) s[i] = -INFINITY;
            }
            mx = max_of(s);
        }
        mx = max_xor32(mx) * mul;
        if constexpr (first) {  // (nothing to rescale yet)
            m = mx > kNegBig ? mx : kNegBig;
            return;
        }
        const bool up = mx > m + kLazy;
        if (__any(up)) {
            const float mn = up ? mx : m;
            const float alpha = fast_exp2(m - mn);
            m = mn;
            l *= alpha;
            if constexpr (D == 256) wait_products();
#pragma unroll
            for (int cb = 0; cb < CB; ++cb) {
                if constexpr (D == 256)
                    scale_acc(acc[cb], alpha);
                else
                    acc[cb] *= alpha;
            }
            if constexpr (D == 256) wait_products();
        }
    };
    vec8 kf[KS];  // K fragments of the tile whose scores come next
    auto read_k = [&](int ks, int buf) __attribute__((always_inline)) {
        kf[ks] = *reinterpret_cast<const vec8*>(smem + buf * TILE + k_at[ks]);
    };

    // One tile: the score products of the next one beside this one's exponentials, then its value products beside the
    // next one's maximum and the K fragments of the one after.
    auto step = [&](int u, auto buf_c) __attribute__((always_inline)) {
        constexpr int buf = decltype(buf_c)::value, next = (buf + 1) % 3, prev = (buf + 2) % 3;
        // K of tile u + 2 and V of tile u have landed (this wave's share; after the barrier, everyone's), and the reads of
        // K(u + 1) and V(u - 1), whose buffers are filled next, are done
        if (u + 5 < nu) {
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(2 * LOADS) : "memory");
            if (PGM != 2 || page_mask >= 7) {
                if (p.table == nullptr) {
                    k_next += ahead_bytes;
                    v_next += ahead_bytes;
                } else {
                    k_next = kbase + row_at(at0 + (u + 4) * ahead + wave * 8, w.k_page);
                    v_next = vbase + row_at(at0 + (u + 2) * ahead + wave * 8, w.v_page);
                }
                dma_rows(k_next, off, next * TILE);
                dma_rows(v_next, off, (3 + prev) * TILE);
            } else {
                load_k(u + 4, next);
                load_v(u + 2, prev);
            }
        } else {
            if (u + 3 < nu)
                asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(2 * LOADS) : "memory");
            else if (u + 1 < nu)
                asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(LOADS) : "memory");
            else
                asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
            load_k(u + 4, next);
            load_v(u + 2, prev);
        }
        // From here to the maximum the order of issue is the source's: a matrix instruction occupies its unit for 32 cycles, in
        // whose shadow go an exponential or two (16 cycles each) and the LDS reads of what comes later.  A wave issues an
        // instruction every five cycles at best and is often alone on its SIMD, so their number counts: one wait serves
        // several fragments, and a result of the exponential unit is not used by the next instruction, which would need a
        // wait state.  (The K fragments are read in the step before: a step that begins with their reads begins with the latency
        // of all four waves' at once.)
        typedef __attribute__((address_space(3))) s16x4_t* lds_s4;
        uint8_t* const vt = smem + buf * TILE;  // (v_at counts the K buffers: the rest fits the instruction's offset)
        s16x4_t vf[2][CB][2];
        auto read_v = [&](int i) __attribute__((always_inline)) {  // i-th of the 4 CB reads
            const int kk = i / (2 * CB), cb = i / 2 % CB, j = i % 2;
            vf[kk][cb][j] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(vt + kk * 16 * PITCH + v_at[cb][j]));
        };
        float e[16];
        uint32_t pw[8];
        constexpr uint32_t kOnes = std::is_same<Tag, f16_tag>::value ? 0x3C003C00u : 0x3F803F80u;
        auto exponential = [&](int i) __attribute__((always_inline)) { e[i] = fast_exp2(__builtin_fmaf(s[i], mul, -m)); };
        auto pack = [&](int j) __attribute__((always_inline)) { pw[j] = EL::pack2(e[2 * j], e[2 * j + 1]); };
        // The exponentials go out beside the score products, 16 / KS a slot; a pair is packed a slot after its second one.
        auto exps = [](int slot) { return 16 * slot / KS; };
        auto packs = [&](int from, int to) __attribute__((always_inline)) {  // pairs of exponentials [from, to)
#pragma unroll
            for (int j = from / 2; j < to / 2; ++j) pack(j);
        };
        __builtin_amdgcn_sched_barrier(0);
        f32x16 s_next;
#pragma unroll
        for (int i = 0; i < 16; ++i) s_next[i] = 0.0f;
        static_for<0, KS>([&](auto ks_c) __attribute__((always_inline)) {
            constexpr int ks = decltype(ks_c)::value;
            s_next = MM::mma(kf[ks], q[ks], s_next);
            pin<D>(s_next);
#pragma unroll
            for (int i = exps(ks); i < exps(ks + 1); ++i) exponential(i);
#pragma unroll
            for (int i = 4 * CB * ks / KS; i < 4 * CB * (ks + 1) / KS; ++i) read_v(i);
            packs(ks == 0 ? 0 : exps(ks - 1), exps(ks));
            __builtin_amdgcn_sched_barrier(0);
        });
        wait_lds<2 * CB>();  // V of the first sixteen tokens
        __builtin_amdgcn_sched_barrier(0);
        static_for<0, CB>([&](auto cb_c) __attribute__((always_inline)) {
            constexpr int cb = decltype(cb_c)::value;
            const vec8 pf = __builtin_bit_cast(vec8, make_uint4(pw[0], pw[1], pw[2], pw[3]));
            acc[cb] = MM::mma(__builtin_bit_cast(vec8, join(vf[0][cb][0], vf[0][cb][1])), pf, acc[cb]);
            pin<D>(acc[cb]);
            // (the denominator sums the probabilities as the second product sees them)
#pragma unroll
            for (int j = 4 * cb / CB; j < 4 * (cb + 1) / CB; ++j) l = EL::dot2(pw[j], kOnes, l);
            if constexpr (cb == 0) packs(exps(KS - 1), 16);  // (the last slot's: the second value products read them)
#pragma unroll
            for (int ks = cb; ks < KS / 2; ks += CB) read_k(ks, prev);  // (past the last tile: of whatever lies there, not used)
            __builtin_amdgcn_sched_barrier(0);
        });
        wait_lds<KS / 2>();  // V of the other sixteen
        __builtin_amdgcn_sched_barrier(0);
        float mx = -INFINITY;
        static_for<0, CB>([&](auto cb_c) __attribute__((always_inline)) {
            constexpr int cb = decltype(cb_c)::value;
            const vec8 pf = __builtin_bit_cast(vec8, make_uint4(pw[4], pw[5], pw[6], pw[7]));
            acc[cb] = MM::mma(__builtin_bit_cast(vec8, join(vf[1][cb][0], vf[1][cb][1])), pf, acc[cb]);
            pin<D>(acc[cb]);
#pragma unroll
            for (int j = 4 + 4 * cb / CB; j < 4 + 4 * (cb + 1) / CB; ++j) l = EL::dot2(pw[j], kOnes, l);
#pragma unroll
            for (int j = 8 * cb / CB; j < 8 * (cb + 1) / CB; ++j) mx = fmaxf(fmaxf(mx, s_next[2 * j]), s_next[2 * j + 1]);
            asm volatile("" : "+v"(mx));  // (here, not where it is used)
#pragma unroll
            for (int ks = KS / 2 + cb; ks < KS; ks += CB) read_k(ks, prev);
            __builtin_amdgcn_sched_barrier(0);
        });
        s = s_next;
        if (u + 1 < nu) settle_max(u + 1, mx, std::false_type{});
    };

    // the first tile's scores, and the K fragments of the second
    if (nu > 2)
        asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(4 * LOADS) : "memory");
    else
        asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) read_k(ks, 0);
    s = scores(kf);
    if (cut < kTok) {  // this wave's V rows past the end, once they have landed (the barrier of the first step follows)
        if (nu > 2)
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * LOADS) : "memory");
        else
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
        for (int i = 0; i < LOADS; ++i)
            if (wave * 8 + i * RPL + lrow >= cut)
                *reinterpret_cast<uint4*>(smem + 3 * TILE + (wave * LOADS + i) * 1024 + lane * 16) = make_uint4(0u, 0u, 0u, 0u);
    }
    if (nu > 2)
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(3 * LOADS) : "memory");
    else
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    load_k(3, 0);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) read_k(ks, 1);
    settle_max(0, max_of(s), std::true_type{});
    for (int u = 0; u < nu; u += 3) {
        step(u, std::integral_constant<int, 0>{});
        if (u + 1 < nu) step(u + 1, std::integral_constant<int, 1>{});
        if (u + 2 < nu) step(u + 2, std::integral_constant<int, 2>{});
    }

    l += __shfl_xor(l, 32);
    // The partials leave through LDS, whole runs of a row at a time (the lanes hold 16 bytes of 32 rows each), and with stores
    // that do not stay in the L2: the merge runs anywhere, and what the L2 holds is written out at the kernel's end, all of it at
    // once (64 sequences behind 4096 tokens, 32/8 heads d 128: 51.8 -> 49.3 us).
    const int row_id = b * w.head_q + hq;
    const size_t part0 = (size_t)split * w.batch * w.head_q;
    if (live && h == 0) *reinterpret_cast<float2*>(p.ws_ml + (part0 + row_id) * 2) = make_float2(m, l);
    constexpr int GB = D == 64 ? 1 : 2;  // blocks of 32 columns at a time
    constexpr int OPITCH = GB * 128 + 16, LPR = GB * 8, RPI = 64 / LPR;  // lanes per row, rows of a store instruction
    static_assert(4 * 32 * OPITCH <= (int)prefix_lds_bytes<D>(), "fits the tile buffers");
    int id[32 / RPI];  // the rows that this lane stores pieces of
#pragma unroll
    for (int i = 0; i < 32 / RPI; ++i) id[i] = __shfl(row_id, i * RPI + lane / LPR);
    const int rows_here = p.rows - (row0 + wave * 32);
    __syncthreads();  // (the tiles are dead)
    if (rows_here <= 0) return;
    uint8_t* const mine = smem + wave * (32 * OPITCH);
    static_for<0, (CB + GB - 1) / GB>([&](auto g_c) __attribute__((always_inline)) {
        constexpr int cb0 = decltype(g_c)::value * GB, NB = CB - cb0 < GB ? CB - cb0 : GB;
#pragma unroll
        for (int cb = 0; cb < NB; ++cb)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<f32x4*>(mine + n * OPITCH + cb * 128 + i * 32 + h * 16) =
                    f32x4{acc[cb0 + cb][4 * i], acc[cb0 + cb][4 * i + 1], acc[cb0 + cb][4 * i + 2], acc[cb0 + cb][4 * i + 3]};
        const int piece = lane % LPR;
        float* const out = p.ws_o + part0 * D + cb0 * 32 + piece * 4;
#pragma unroll
        for (int i = 0; i < 32 / RPI; ++i) {
            if (i * RPI >= rows_here) break;
            const int r = i * RPI + lane / LPR;
            const f32x4 x = *reinterpret_cast<const f32x4*>(mine + r * OPITCH + piece * 16);
            if (r < rows_here && (NB == GB || piece < NB * 8)) __builtin_nontemporal_store(x, reinterpret_cast<f32x4*>(out + (size_t)id[i] * D));
        }
    });
}

// Own tokens of sequence b (paged sequences count the prefix in their lengths).
__device__ __forceinline__ int own_len(const PrefixParams& p, int b) {
    return p.table ? max(p.own.seq_lens[b] - p.prefix_len, 0) : p.own.cu_seq_k[b + 1] - p.own.cu_seq_k[b];
}

// Positions of the sequences on the balanced grid's line, in units of flat_unit tokens (every sequence rounded up), into LDS:
// at[0 .. batch].  Thread t adds up sequences 4 t .. 4 t + 3.
__device__ __forceinline__ void scan_lengths(const PrefixParams& p, int32_t* at) {
    const SweepParams& w = p.own;
    int n[4], sum = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int b = (int)threadIdx.x * 4 + i;
        n[i] = sum;
        if (b < w.batch) sum += (own_len(p, b) + w.flat_unit - 1) / w.flat_unit;
    }
    int incl = sum;
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int other = __shfl_up(incl, d);
        if (lane >= d) incl += other;
    }
    int32_t* const waves = at + kScanBatch + 1;
    if (lane == 63) waves[threadIdx.x >> 6] = incl;
    __syncthreads();
    int base = incl - sum;
    for (int i = 0; i < (int)(threadIdx.x >> 6); ++i) base += waves[i];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int b = (int)threadIdx.x * 4 + i;
        if (b <= w.batch) at[b] = base + n[i];
    }
    if (threadIdx.x == 255 && w.batch == kScanBatch) at[kScanBatch] = base + sum;
    __syncthreads();
}
constexpr size_t kScanBytes = (kScanBatch + 1 + 4) * sizeof(int32_t);

// Work-groups are numbered so that the row tiles of one (KV head, prefix split) run on one XCD (consecutive work-groups go
// to the eight XCDs in turn) and share its K/V through that XCD's L2; likewise the head groups of one own-token segment.  Where
// that leaves XCDs idle (spread) the tiles go to all of them in turn, and every L2 gets the K/V.
//
// The own tokens are cut in one of two ways, as in the grouped kernel: own.flat_wgs == 0: (sequence, split of own.chunk tokens);
// else the sequences' tokens form one line, and each of flat_wgs shares of it is one work-group's (per KV heads and group).
template <typename Tag, int D, bool WH, int PGM>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(D <= 128 ? 2 : 1))) void prefix_kernel(const PrefixParams p) {
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    const int id = (int)blockIdx.x;
    if (id < p.prefix_wgs) {
        int g, tile;  // (KV head, split), row tile
        if (p.spread) {
            g = id / p.row_tiles;
            tile = id - g * p.row_tiles;
        } else {
            const int slot = id >> 3, rest = slot / p.row_tiles;
            g = rest * 8 + (id & 7);
            tile = slot - rest * p.row_tiles;
        }
        if (g >= p.own.head_k * p.splits) return;
        const int split = g / p.own.head_k;
        prefix_segment<Tag, D, PGM>(p, smem, g - split * p.own.head_k, tile * kPrefixRows, split);
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
    const int own0 = p.table ? p.prefix_len : 0;
    // which tokens: the balanced grid's share, or split number `split` of one sequence
    const int32_t* cu = w.flat_cu;
    int b = 0, r0 = 0, r1 = 0, share = 0, split = 0;
    if (w.flat_wgs > 0) {
        share = seg / ny;
        if (share >= w.flat_wgs) return;
        if (p.scan) {
            int32_t* const at = reinterpret_cast<int32_t*>(smem + gqa_lds_bytes<D>(1));
            scan_lengths(p, at);
            if (share == 0 && by == 0)  // (for the merge)
                for (int j = threadIdx.x; j <= w.batch; j += 256) p.flat_out[j] = at[j];
            cu = at;
        }
        const int total = cu[w.batch];
        const int T = flat_share(total, w.flat_wgs, w.flat_step, w.flat_min);
        r0 = (int)min((long long)share * T, (long long)total);
        r1 = share == w.flat_wgs - 1 ? total : (int)min((long long)r0 + T, (long long)total);
        if (r0 >= r1) return;
        for (int n = w.batch; n > 1;) {  // the last b with cu[b] <= r0: 64 probes at once
            const int stride = (n + 63) >> 6;
            const int idx = b + (int)(threadIdx.x & 63) * stride;
            const int k = max(__popcll(__ballot(idx < b + n && cu[idx] <= r0)), 1) - 1;
            b += k * stride;
            n = min(stride, n - k * stride);
        }
    } else {
        split = (seg / ny) % w.nsplit;
        b = seg / ny / w.nsplit;
        if (b >= w.batch) return;  // (the last eight of several head groups)
    }
    for (;; ++b) {
        int start, len, c0, c1;
        size_t part0;
        if (w.flat_wgs > 0) {
            if (b >= w.batch) break;
            const int s = cu[b], e = cu[b + 1];
            if (s >= r1) break;
            if (e <= s) continue;
            seq_range(w, b, start, len);
            c0 = own0 + (max(r0, s) - s) * w.flat_unit;
            c1 = min(own0 + (min(r1, e) - s) * w.flat_unit, len);
            part0 = (size_t)(share + b) * w.head_q;
        } else {
            seq_range(w, b, start, len);
            c0 = own0 + split * w.chunk;
            c1 = split == w.nsplit - 1 ? len : min(len, c0 + w.chunk);
            part0 = (size_t)b * w.head_q * w.nsplit + split;
        }
        gqa_segment<Tag, D, D, 1, true, WH, 0, PGM, true>(p.own, smem, by, b, start, len, c0, c1, part0,
                                                          w.flat_wgs > 0 ? 1 : w.nsplit, false);
        if (w.flat_wgs == 0) break;
        if (!WH) __syncthreads();  // the merge area of this segment is the V tile area of the next
    }
}

template <typename Tag, int D, bool WH, int PGM>
hipError_t launch_form(const PrefixParams& p, int own_wgs, hipStream_t stream) {
    const size_t segment = gqa_lds_bytes<D>(1) + (p.scan ? kScanBytes : 0);
    const size_t lds = prefix_lds_bytes<D>() > segment ? prefix_lds_bytes<D>() : segment;
    auto kern = prefix_kernel<Tag, D, WH, PGM>;
    if (lds > 48 * 1024) {
        static std::atomic<uint64_t> devices_done{0};
        const hipError_t e = ensure_lds_limit(reinterpret_cast<const void*>(kern), 160 * 1024, devices_done);
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL(kern, dim3((unsigned)(p.prefix_wgs + own_wgs)), dim3(256), lds, stream, p);
    return hipGetLastError();
}

template <typename Tag, int D, bool WH>
hipError_t launch_pages(const PrefixParams& p, int own_wgs, hipStream_t stream) {
    // how the own part finds a tile's rows: whole tiles in pages of 32 tokens and more (and packed rows), a look-up for every row
    // in smaller ones; at d = 256, whose rows leave no registers for that, two runs in 16-token pages.  (Two runs against a look-up
    // per row, 64 sequences of 0 .. 1024 behind 4096, 32/8 heads: d 64 33.8 / 31.1 us, d 96 37.3 / 33.7, d 128 49.3 / 47.2, d 256 79
    // / 126; 128 of 0 .. 256 behind 1024, 32/32 heads: 52 / 46, 82 / 74, 84 / 80, 131 / 247; 16 of 0 .. 512 behind 1024, 32/1 heads:
    // 10.5 / 10.3, 11.6 / 11.3, 12.8 / 13.0, 17 / 21.)
    if (p.own.block_table == nullptr || p.own.page_shift >= 5) return launch_form<Tag, D, WH, 0>(p, own_wgs, stream);
    if constexpr (D == 256)
        if (p.own.page_shift == 4) return launch_form<Tag, D, WH, 1>(p, own_wgs, stream);
    return launch_form<Tag, D, WH, 2>(p, own_wgs, stream);
}

template <int D>
hipError_t launch_dim(const PrefixParams& p, bool is_bf16, bool wave_per_head, int own_wgs, hipStream_t stream) {
    if (is_bf16)
        return wave_per_head ? launch_pages<bf16_tag, D, true>(p, own_wgs, stream) : launch_pages<bf16_tag, D, false>(p, own_wgs, stream);
    return wave_per_head ? launch_pages<f16_tag, D, true>(p, own_wgs, stream) : launch_pages<f16_tag, D, false>(p, own_wgs, stream);
}

}  // namespace prefix
}  // namespace da
