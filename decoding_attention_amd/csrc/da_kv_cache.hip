// K/V rows written into a paged cache, quantised on the way (append), and read back as 16-bit rows (read).
//
// Both kernels move a row in chunks of eight or sixteen elements, one chunk a lane.  A work-group takes a few consecutive tokens of
// one plane (K or V); its first threads look up where each of them lies in the pools -- sequence, position, page -- while
// the chunks' loads are in flight, and hand the rows round through LDS.
//
// Quantisation, per KV head with a given factor s:    n = x / s rounded to the format (ties to even), saturating.
// With a pair per row (or per run of 64 elements):    scale = (max - min) / (2^bits - 1), zero = qmin - min / scale,
//                                                     n = x / scale + zero rounded to an integer (ties to even), clamped.
// The quotients are taken in double precision: a 16-bit input often lies exactly half-way between two steps (the values of
// a row are small multiples of one power of two, and so is max - min), and there the bits of a float32 quotient would
// decide which of the two is stored.  scale and zero are rounded to float32 first, since n has to fit the pair that is
// stored.
//
// What bounds them: a read moves 5 to 6 TB/s, as much as a copy (24 sequences of 0 .. 1300 tokens, 16-bit, 4 heads d 256: 131 MB in
// 22 to 27 us; 114 000 int4 tokens of 8 heads d 128 with a pair per 64: 615 MB in 116 to 133).  An append spends 12 vector
// instructions an element on exact quotients and runs at 4.4 TB/s (26 000 tokens of 8 heads d 128, int8 per 64: 168 MB in 37 to 40 us).
// Small calls are the launch and the three trips of the look-up: 3 to 4 us, for one sequence or 64.
#include "da_kv_cache.h"

namespace da {
namespace {

constexpr int kThreads = 256;
constexpr int kUnroll = 4;        // chunks a thread holds at once
constexpr int kMaxTokens = 128;   // most tokens of a work-group

// i / d by m = ceil(2^32 / d): the excess of m is below 2^-32 d, so the quotient is right while i * d < 2^32 (a work-group holds at
// most 2 kThreads * kUnroll chunks, or the chunks of one token, of which there are 2^15 at most)
__device__ __forceinline__ int magic_div(int i, uint32_t m) { return (int)__umulhi((uint32_t)i, m); }

// Where a token's row lies in the plane's pool.
struct Place {
    int64_t elem;  // its first element; kNowhere in the pools, or kBehind the last sequence (nothing is done for it at all)
    int64_t row;   // its number among the pools' rows
};
constexpr int64_t kNowhere = -1, kBehind = -2;

// Evenly spaced sequences: their entries of cu_seq, and their lengths.
struct Marks {
    int32_t start[kThreads], len[kThreads];
};

// Row of the pools where token t lies, kNowhere if it lies nowhere: a token's sequence ends at seq_lens[b], and the tokens of
// the call are its last ones.  Bounds are checked here, for the row is written: a position before the sequence's first
// token (a padded sequence of no tokens), behind the block table, or a page that the pools do not have.
__device__ __forceinline__ int64_t pool_row(const KvCacheParams& p, int b, int64_t pos) {
    if (pos < 0 || (pos >> p.page_shift) >= p.max_blocks) return kNowhere;
    const int page = p.block_table[(int64_t)b * p.max_blocks + (pos >> p.page_shift)];
    if ((uint32_t)page >= (uint32_t)p.num_pages) return kNowhere;
    return ((int64_t)page << p.page_shift) + (pos & ((1 << p.page_shift) - 1));
}

// Looks the work-group's rows up, one thread a token.  The sequence of a token is found among 256 evenly spaced entries of
// cu_seq, fetched by the threads at once (and the lengths with them) and searched in LDS, and then between two of them: with up
// to 256 sequences one trip to memory, in front of the block table's, where a search in memory takes eight.
__device__ __forceinline__ void find_rows(const KvCacheParams& p, const KvPlane& pl, int64_t tok0, Place* places, Marks& marks) {
    const int64_t t = tok0 + threadIdx.x;
    const bool mine = (int)threadIdx.x < p.tokens_per_block && t < p.tokens;
    int64_t row = kBehind;
    if (p.cu_seq == nullptr) {
        if (mine) row = pool_row(p, (int)t, (int64_t)p.seq_lens[t] - 1);
    } else {
        const int step = (p.batch + kThreads - 1) / kThreads;
        marks.start[threadIdx.x] = p.cu_seq[min((int)threadIdx.x * step, p.batch)];
        marks.len[threadIdx.x] = p.seq_lens[min((int)threadIdx.x * step, p.batch - 1)];
        const int32_t end = p.cu_seq[p.batch];
        __syncthreads();
        if (mine && t >= marks.start[0] && t < end) {
            int lo = 0;  // the last mark at or below t
            for (int half = kThreads / 2; half > 0; half >>= 1)
                if (marks.start[lo + half] <= t) lo += half;
            int64_t len = marks.len[lo], next = lo + 1 < kThreads ? marks.start[lo + 1] : end;
            if (step > 1) {
                lo *= step;
                int n = min(step, p.batch - lo);  // cu_seq[lo] <= t < cu_seq[lo + n]
                while (n > 1) {
                    const int half = n >> 1;
                    if (p.cu_seq[lo + half] <= t) {
                        lo += half;
                        n -= half;
                    } else {
                        n = half;
                    }
                }
                len = p.seq_lens[lo];
                next = p.cu_seq[lo + 1];
            }
            row = pool_row(p, lo, len - (next - t));
        }
    }
    if ((int)threadIdx.x < p.tokens_per_block)
        places[threadIdx.x] = {row < 0 ? row
                                       : (row >> p.page_shift) * pl.page +
                                             (row & ((1 << p.page_shift) - 1)) * (int64_t)(p.head_k * pl.dim),
                               row};
    __syncthreads();
}

template <typename Tag>
__device__ __forceinline__ void widen8(uint4 w, float* x) {
    using EL = Elem<Tag>;
    x[0] = EL::lo(w.x), x[1] = EL::hi(w.x), x[2] = EL::lo(w.y), x[3] = EL::hi(w.y);
    x[4] = EL::lo(w.z), x[5] = EL::hi(w.z), x[6] = EL::lo(w.w), x[7] = EL::hi(w.w);
}

// x / s rounded as one division, x and s finite and s not 0: the reciprocal `inv` (rounded once) gives the quotient to within
// a step, and one correction with the exact remainder settles it.
__device__ __forceinline__ double quotient(double x, double s, double inv) {
    const double q = x * inv;
    return fma(fma(-q, s, x), inv, q);
}

// A double rounded to 24 bits, the last one set whenever anything was lost: a second rounding, to a format of at least two
// bits fewer, then comes out as if it were the only one.  (Below 2^-126 the conversion rounds as well: far below FP8's
// least value.)
__device__ __forceinline__ float round_to_odd(double y) {
    const uint64_t u = (uint64_t)__double_as_longlong(y);
    const uint32_t low = (uint32_t)u, lost = min(low & 0x1FFFFFFFu, 1u) << 29;
    return (float)__longlong_as_double((long long)((u & 0xFFFFFFFF00000000ull) | ((low & 0xE0000000u) | lost)));
}

// max and min of three, none of them a NaN (without the quieting moves that fmaxf brings for operands of unknown origin)
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}
__device__ __forceinline__ float min3(float a, float b, float c) {
    float r;
    asm("v_min3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}

// the nearest integer, clamped to [LO, HI] (a NaN becomes 0): the conversion saturates
template <int LO, int HI>
__device__ __forceinline__ int to_int(double y) {
    int n;
    asm("v_cvt_i32_f64 %0, %1" : "=v"(n) : "v"(rint(y)));
    return min(max(n, LO), HI);
}

template <int FMT>
struct Range;
template <>
struct Range<kKvInt8> {
    static constexpr int lo = -128, hi = 127;
};
template <>
struct Range<kKvInt4> {
    static constexpr int lo = -8, hi = 7;
};

// Index of the pair of a chunk of E elements: a pair per row, or per 64 elements.
template <int PAIRS, int E>
__device__ __forceinline__ int64_t pair_at(const KvCacheParams& p, const KvPlane& pl, int64_t row, int head, int chunk) {
    return PAIRS == 2 ? row * ((p.head_k * pl.dim) >> 6) + chunk / (64 / E) : row * p.head_k + head;
}

// lo and hi over the lanes that hold a row (or a run): a NaN anywhere makes both a NaN
__device__ __forceinline__ float min_nan(float a, float b) { return (b < a || b != b) ? b : a; }
__device__ __forceinline__ float max_nan(float a, float b) { return (b > a || b != b) ? b : a; }

// Elements a lane takes at once.  Append: a row's factors cost a division in double precision per lane, which sixteen elements
// share; a copy takes eight.
constexpr int row_chunk(bool read, int fmt) { return read || fmt == 0 ? 8 : 16; }

// The definition as it stands, for what the ways below leave out: values that are not finite, factors outside any sense, and
// quotients that lie within rounding of half a step.  `span` lanes hold a row or run; `src` are the lane's sixteen values once
// more (a plain loop over them: this is rare, and the registers of an unrolled one would be every wave's).
template <typename Tag, int FMT, int PAIRS>
__device__ __forceinline__ void quantise_any(const uint16_t* src, float factor, int span, uint32_t (&w)[4], float2& pair) {
    using EL = Elem<Tag>;
    constexpr int QLO = Range<FMT>::lo, QHI = Range<FMT>::hi, BITS = FMT == kKvInt8 ? 8 : 4;
    pair = make_float2(factor, 0.0f);
    if constexpr (PAIRS != 0) {
        float lo = EL::lo(src[0]), hi = lo;
#pragma unroll 1
        for (int j = 1; j < 16; ++j) {
            const float x = EL::lo(src[j]);
            lo = min_nan(lo, x);
            hi = max_nan(hi, x);
        }
        for (int d = 1; d < span; d <<= 1) {
            lo = min_nan(lo, __shfl_xor(lo, d));
            hi = max_nan(hi, __shfl_xor(hi, d));
        }
        pair.x = (float)(((double)hi - (double)lo) / (double)(QHI - QLO));
        pair.x = pair.x < 1e-8f ? 1e-8f : pair.x;
        pair.y = (float)((double)QLO - (double)lo / (double)pair.x);
    }
#pragma unroll 1
    for (int j = 0; j < 16; ++j) {
        const double y = (double)EL::lo(src[j]) / (double)pair.x;
        const uint32_t q = (uint32_t)to_int<QLO, QHI>(PAIRS == 0 ? y : y + (double)pair.y) << (32 - BITS);
        // (the words shift right, the new integer comes in at the top: after sixteen the first one has arrived at the bottom)
        if constexpr (BITS == 8) {
            w[0] = w[0] >> 8 | w[1] << 24;
            w[1] = w[1] >> 8 | w[2] << 24;
            w[2] = w[2] >> 8 | w[3] << 24;
            w[3] = w[3] >> 8 | q;
        } else {
            w[0] = w[0] >> 4 | w[1] << 28;
            w[1] = w[1] >> 4 | q;
        }
    }
}

// A NaN when any of the eight values in `w` is not finite.
template <typename Tag>
__device__ __forceinline__ float not_finite(uint4 w, float seen) {
    using EL = Elem<Tag>;
    return EL::dot2(w.x, 0u, EL::dot2(w.y, 0u, EL::dot2(w.z, 0u, EL::dot2(w.w, 0u, seen))));
}

// The same for ordinary values at a fourth of the instructions, sixteen integers packed into four words (int4: two).
// One multiply-add in double precision, x inv + (zero + 1/2 + a constant of 1.5 2^28 or 1.5 2^24), leaves t + 1/2 in the low
// word as a fixed-point number in units of 2^-24 (int8) or 2^-28 (int4), the integer in its upper bits.  It is off from the
// definition's by less than 1 1/8 units: half from the sum in brackets, half from the result, and from inv and the definition's own
// quotient 2^-53 of |x / scale| each, less than 2^-32 together and a sixteenth of a unit (|zero| < 2^20, so |x / scale| < 2^20 + 2^9;
// the definition's sum is below 2^9 and off by 2^-45).  Two units are added, so that the number lies between 7/8 and 3 1/8 units
// above the definition's: a fraction of five units and more lies behind the whole number that the definition rounds to, and one that
// passed the next whole number counts three at most.  The others (of normal values, a lane's sixteen in 200) are settled by the
// quotient itself.
template <typename Tag, int FMT, int PAIRS>
__device__ __forceinline__ void quantise(const uint4 (&raw)[2], const uint16_t* src, float factor, int span, uint32_t (&w)[4],
                                         float2& pair) {
    constexpr int QLO = Range<FMT>::lo, QHI = Range<FMT>::hi, BITS = FMT == kKvInt8 ? 8 : 4, PER = 32 / BITS;
    constexpr double kUnit = FMT == kKvInt8 ? 0x1p-24 : 0x1p-28;
    float x[16];
    widen8<Tag>(raw[0], x);
    widen8<Tag>(raw[1], x + 8);
    bool plain = not_finite<Tag>(raw[0], not_finite<Tag>(raw[1], 0.0f)) == 0.0f;
    pair = make_float2(factor, 0.0f);
    double inv;
    if constexpr (PAIRS != 0) {
        float lo = x[0], hi = x[0];
#pragma unroll
        for (int j = 1; j < 15; j += 2) {
            lo = min3(lo, x[j], x[j + 1]);
            hi = max3(hi, x[j], x[j + 1]);
        }
        lo = min3(lo, lo, x[15]);
        hi = max3(hi, hi, x[15]);
        for (int d = 1; d < span; d <<= 1) {
            const float lo2 = __shfl_xor(lo, d), hi2 = __shfl_xor(hi, d);
            lo = min3(lo, lo, lo2);
            hi = max3(hi, hi, hi2);
        }
        constexpr double kSteps = QHI - QLO;
        pair.x = (float)quotient((double)hi - (double)lo, kSteps, 1.0 / kSteps);
        pair.x = pair.x < 1e-8f ? 1e-8f : pair.x;
        inv = 1.0 / (double)pair.x;
        pair.y = (float)((double)QLO - quotient((double)lo, (double)pair.x, inv));
        // (below this the float32 rounding of zero moves t by less than 1/16: it stays in the range, and needs no clamp)
        plain = plain && fabsf(pair.y) < 1048576.0f;
    } else {
        inv = 1.0 / (double)factor;
        plain = plain && factor > 1e-30f && factor < 1e30f;
    }
    const double s = (double)pair.x, z = (double)pair.y, zc = z + (1.5 * 0x1p52 * kUnit + 0.5 + 2.0 * kUnit);
    const float least = factor * (QLO - 0.25f), most = factor * (QHI + 0.25f);
    uint32_t near = ~0u;
#pragma unroll
    for (int j = 15; j >= 0; --j) {
        // (factors per head: what lies beyond the range is cut to just outside the outermost integers)
        const float c = PAIRS == 0 ? __builtin_amdgcn_fmed3f(x[j], least, most) : x[j];
        const double u = fma((double)c, inv, zc);
        const uint32_t v = (uint32_t)__double_as_longlong(u);
        near = min(near, v << BITS);  // (the fraction)
        w[j / PER] = __builtin_amdgcn_alignbit(j % PER == PER - 1 ? 0u : w[j / PER], v, 32 - BITS);
    }
    const bool sure = near >= (5u << BITS);
    if (__any(!(plain && sure))) {
        if (__any(!plain)) {
            quantise_any<Tag, FMT, PAIRS>(src, factor, span, w, pair);
        } else {
            uint32_t again[8] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w, raw[1].x, raw[1].y, raw[1].z, raw[1].w};
#pragma unroll
            for (int j = 0; j < 8; ++j) asm volatile("" : "+v"(again[j]));  // (widened once more: x is not kept for this)
#pragma unroll
            for (int j = 15; j >= 0; --j) {
                const double y = quotient((double)(j & 1 ? Elem<Tag>::hi(again[j >> 1]) : Elem<Tag>::lo(again[j >> 1])), s, inv);
                const uint32_t n = (uint32_t)to_int<QLO, QHI>(PAIRS == 0 ? y : y + z) << (32 - BITS);
                w[j / PER] = __builtin_amdgcn_alignbit(j % PER == PER - 1 ? 0u : w[j / PER], n, 32 - BITS);
            }
        }
    }
}

__device__ __forceinline__ uint32_t pack_fp8(float a, float b, float c, float d) {
    const int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}

// Sixteen values in FP8, four words.  x / s in float32, off by less than 2^-22 (a factor that is a power of two: exact), is
// converted from just below and just above; where the two agree they are the definition's.  The others (of normal values, a
// lane's sixteen in 2000) are settled by the quotient in double precision.
template <typename Tag>
__device__ __forceinline__ void quantise_fp8(const uint4 (&raw)[2], const uint16_t* src, float factor, uint32_t (&b)[4]) {
    float x[16];
    widen8<Tag>(raw[0], x);
    widen8<Tag>(raw[1], x + 8);
    const bool plain = not_finite<Tag>(raw[0], not_finite<Tag>(raw[1], 0.0f)) == 0.0f && factor > 1e-30f && factor < 1e30f;
    const float inv = 1.0f / factor, delta = (__float_as_uint(factor) & 0x7FFFFFu) == 0 ? 0.0f : 0x1p-22f;
    uint32_t differ = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        float y[4], lo[4], hi[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            y[i] = __builtin_amdgcn_fmed3f(x[4 * j + i] * inv, -448.0f, 448.0f);
            lo[i] = y[i] * (1.0f - delta);
            hi[i] = y[i] * (1.0f + delta);
        }
        b[j] = pack_fp8(lo[0], lo[1], lo[2], lo[3]);
        differ |= b[j] ^ pack_fp8(hi[0], hi[1], hi[2], hi[3]);
    }
    if (__any(!plain || differ != 0)) {
        const double s = (double)factor;
        if (__any(!plain)) {  // (the definition as it stands)
#pragma unroll 1
            for (int j = 0; j < 16; ++j) {
                double y = (double)Elem<Tag>::lo(src[j]) / s;
                y = y > 448.0 ? 448.0 : (y < -448.0 ? -448.0 : y);
                const float g = y == y ? round_to_odd(y) : __uint_as_float(0x7FC00000u);
                const uint32_t byte = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(g, g, 0, false) << 24;
                b[0] = b[0] >> 8 | b[1] << 24;
                b[1] = b[1] >> 8 | b[2] << 24;
                b[2] = b[2] >> 8 | b[3] << 24;
                b[3] = b[3] >> 8 | byte;
            }
        } else {
            const double wide = 1.0 / s;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float f[4];
#pragma unroll
                for (int i = 0; i < 4; ++i)  // (beyond the greatest value the rounded quotient is cut to it)
                    f[i] = __builtin_amdgcn_fmed3f(round_to_odd(quotient((double)x[4 * j + i], s, wide)), -448.0f, 448.0f);
                b[j] = pack_fp8(f[0], f[1], f[2], f[3]);
            }
        }
    }
}

template <typename Tag, int FMT, int PAIRS>
__global__ __launch_bounds__(kThreads) void kv_append_kernel(const KvCacheParams p) {
    constexpr int E = row_chunk(false, FMT), V = E / 8, U = kUnroll / V;  // V: 16-byte loads of a chunk
    __shared__ Place places[kMaxTokens];
    __shared__ Marks marks;
    const KvPlane& pl = p.plane[blockIdx.y];
    const int64_t tok0 = (int64_t)blockIdx.x * p.tokens_per_block;
    const int lanes = pl.dim / E, chunks = p.head_k * lanes;
    // (rows behind the last sequence need not be there: they are not read)
    const int64_t tokens = p.cu_seq ? min(p.tokens, (int64_t)p.cu_seq[p.batch]) : p.tokens;
    const int n = (int)min((int64_t)p.tokens_per_block, tokens - tok0) * chunks;
    if (n <= 0) return;
    uint8_t* const pool = reinterpret_cast<uint8_t*>(pl.pool);
    const uint16_t* const src0 = reinterpret_cast<const uint16_t*>(pl.src) + tok0 * pl.src_token;
    bool looked = false;
    for (int base = 0; base < n; base += kThreads * U) {
        uint4 w[U][V];
        const uint16_t* src[U];
        int tok[U], head[U], chunk[U];  // (chunk: of the token)
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = min(base + u * kThreads + (int)threadIdx.x, n - 1);
            tok[u] = magic_div(i, pl.chunks_magic);
            chunk[u] = i - __mul24(tok[u], chunks);
            head[u] = magic_div(chunk[u], pl.lanes_magic);
            const int in_head = (chunk[u] - __mul24(head[u], lanes)) * E;
            // (64-bit products are four quarter-rate instructions: only where a stride asks for them)
            if (pl.narrow)
                src[u] = src0 + (uint32_t)(__mul24(tok[u], (int)pl.src_token) + __mul24(head[u], (int)pl.src_head) + in_head);
            else
                src[u] = src0 + (tok[u] * pl.src_token + head[u] * pl.src_head + in_head);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                if (pl.aligned) {
                    w[u][v] = stream_load16(src[u] + v * 8);
                } else {
                    uint32_t e[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) e[j] = src[u][v * 8 + j];
                    w[u][v] = make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
                }
            }
        }
        if (!looked) {
            find_rows(p, pl, tok0, places, marks);
            looked = true;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (base + u * kThreads + (int)threadIdx.x >= n) break;
            const int64_t row = places[tok[u]].elem;  // (negative: nothing to write)
            const int64_t elem = row + chunk[u] * E;
            if constexpr (FMT == 0) {
                if (row >= 0) *reinterpret_cast<uint4*>(pool + elem * 2) = w[u][0];
                continue;
            }
            const float factor = PAIRS == 0 && pl.scale ? pl.scale[head[u]] : 1.0f;
            if constexpr (FMT == kKvFp8) {
                const uint4 raw[2] = {w[u][0], w[u][V - 1]};
                uint32_t b[4];
                quantise_fp8<Tag>(raw, src[u], factor, b);
                if (row >= 0) *reinterpret_cast<uint4*>(pool + elem) = make_uint4(b[0], b[1], b[2], b[3]);
            } else if constexpr (FMT == kKvInt8 || FMT == kKvInt4) {
                // (a row's lanes are neighbours and start at a multiple of their number, a power of two)
                const int span = PAIRS == 2 ? 64 / E : (PAIRS == 1 ? lanes : 1);
                uint32_t q[4];
                float2 pair;
                const uint4 raw[2] = {w[u][0], w[u][V - 1]};
                quantise<Tag, FMT, PAIRS>(raw, src[u], factor, span, q, pair);
                if (row >= 0) {
                    if (PAIRS != 0 && (chunk[u] & (span - 1)) == 0)  // (the first lane of a row or run)
                        reinterpret_cast<float2*>(pl.scale)[pair_at<PAIRS, E>(p, pl, places[tok[u]].row, head[u], chunk[u])] = pair;
                    if constexpr (FMT == kKvInt8)
                        *reinterpret_cast<uint4*>(pool + elem) = make_uint4(q[0], q[1], q[2], q[3]);
                    else
                        *reinterpret_cast<uint2*>(pool + (elem >> 1)) = make_uint2(q[0], q[1]);
                }
            }
        }
    }
}

template <typename Tag, int FMT, int PAIRS>
__global__ __launch_bounds__(kThreads) void kv_read_kernel(const KvCacheParams p) {
    using EL = Elem<Tag>;
    __shared__ Place places[kMaxTokens];
    __shared__ Marks marks;
    const KvPlane& pl = p.plane[blockIdx.y];
    const int64_t tok0 = (int64_t)blockIdx.x * p.tokens_per_block;
    const int lanes = pl.dim >> 3, chunks = p.head_k * lanes;
    const int n = (int)min((int64_t)p.tokens_per_block, p.tokens - tok0) * chunks;
    const uint8_t* const pool = reinterpret_cast<const uint8_t*>(pl.pool);
    uint4* const dst = reinterpret_cast<uint4*>(pl.dst) + tok0 * chunks;
    find_rows(p, pl, tok0, places, marks);
    for (int base = 0; base < n; base += kThreads * kUnroll) {
        uint4 w[kUnroll];
        float2 pair[kUnroll];
        bool behind[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const int i = min(base + u * kThreads + (int)threadIdx.x, n - 1);
            const int tok = magic_div(i, pl.chunks_magic);
            const int c = i - __mul24(tok, chunks);
            const int64_t row = places[tok].elem;
            behind[u] = row == kBehind;
            w[u] = make_uint4(0u, 0u, 0u, 0u);
            pair[u] = make_float2(0.0f, 0.0f);  // (a token that lies nowhere reads as zeros)
            if (row < 0) continue;
            const int64_t elem = row + c * 8;
            if constexpr (FMT == 0) {
                w[u] = stream_load16(pool + elem * 2);
            } else if constexpr (FMT == kKvInt4) {
                w[u].x = *reinterpret_cast<const uint32_t*>(pool + (elem >> 1));
            } else {
                const uint2 v = *reinterpret_cast<const uint2*>(pool + elem);
                w[u].x = v.x;
                w[u].y = v.y;
            }
            if constexpr (PAIRS != 0) {
                pair[u] = reinterpret_cast<const float2*>(
                    pl.scale)[pair_at<PAIRS, 8>(p, pl, places[tok].row, magic_div(c, pl.lanes_magic), c)];
            } else if constexpr (FMT != 0) {
                pair[u].x = pl.scale ? pl.scale[magic_div(c, pl.lanes_magic)] : 1.0f;
            }
        }
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            if (base + u * kThreads + (int)threadIdx.x >= n) break;
            if (behind[u]) continue;
            uint4 r = w[u];
            if constexpr (FMT != 0) {
                float x[8];
                if constexpr (FMT == kKvFp8) {
                    const uint4 h = fp8x8_to_16<f16_tag>(make_uint2(w[u].x, w[u].y));
                    widen8<f16_tag>(h, x);
                } else if constexpr (FMT == kKvInt8) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        x[j] = (float)(int8_t)(w[u].x >> (8 * j));
                        x[4 + j] = (float)(int8_t)(w[u].y >> (8 * j));
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) x[j] = (float)((int32_t)(w[u].x << (28 - 4 * j)) >> 28);
                }
                // scale (n - zero), two roundings in float32, then the one to 16 bits
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = pair[u].x * (PAIRS != 0 ? x[j] - pair[u].y : x[j]);
                r = make_uint4(EL::pack2(x[0], x[1]), EL::pack2(x[2], x[3]), EL::pack2(x[4], x[5]), EL::pack2(x[6], x[7]));
            }
            dst[base + u * kThreads + (int)threadIdx.x] = r;
        }
    }
}

// Tokens per work-group: a thread holds up to kUnroll chunks, fewer while that leaves CUs without a work-group.  Large calls take
// two turns, for the rows' look-up is three trips to memory one after the other: int8 with a pair per 64, 26 000 tokens of 8
// heads d 128, 47.2 -> 39.2 us with half the work-groups; a read gains less, int4 per 64, 114 000 tokens, 138 -> 132 us, and at
// 26 000 it loses, 29.5 -> 30.0.
}  // namespace

int kv_cache_tokens_per_block(const KvCacheParams& p, bool read, int fmt, int planes) {
    const int elems = row_chunk(read, fmt);
    const int chunks = p.head_k * (p.plane[0].dim >> 3);  // (of eight elements: kUnroll of them to a thread)
    int tpb = kThreads * kUnroll / chunks;
    const auto groups = [&](int t) { return (p.tokens + t - 1) / t * planes; };
    if (tpb > 0 && 2 * tpb <= kMaxTokens && groups(2 * tpb) >= (read ? 8192 : 1024)) return 2 * tpb;
    while (tpb > 1 && tpb * chunks > kThreads * elems / 8 && groups(tpb) < 512) tpb >>= 1;
    return tpb < 1 ? 1 : (tpb > kMaxTokens ? kMaxTokens : tpb);
}

namespace {

template <bool READ, typename Tag, int FMT, int PAIRS>
hipError_t launch_form(const KvCacheParams& p, int planes, hipStream_t stream) {
    const dim3 grid((unsigned)((p.tokens + p.tokens_per_block - 1) / p.tokens_per_block), (unsigned)planes);
    if constexpr (READ)
        hipLaunchKernelGGL((kv_read_kernel<Tag, FMT, PAIRS>), grid, dim3(kThreads), 0, stream, p);
    else
        hipLaunchKernelGGL((kv_append_kernel<Tag, FMT, PAIRS>), grid, dim3(kThreads), 0, stream, p);
    return hipGetLastError();
}

template <bool READ, typename Tag>
hipError_t launch_tag(KvCacheParams p, int fmt, int pairs, int planes, hipStream_t stream) {
    const int elems = row_chunk(READ, fmt);
    p.tokens_per_block = kv_cache_tokens_per_block(p, READ, fmt, planes);
    for (int i = 0; i < planes; ++i) {
        const uint64_t lanes = (uint64_t)p.plane[i].dim / elems, chunks = lanes * (uint64_t)p.head_k;
        p.plane[i].lanes_magic = (uint32_t)(((1ull << 32) + lanes - 1) / lanes);
        p.plane[i].chunks_magic = (uint32_t)(((1ull << 32) + chunks - 1) / chunks);
        const int64_t st = p.plane[i].src_token, sh = p.plane[i].src_head;
        p.plane[i].narrow = st < (1 << 23) && sh < (1 << 23) && kMaxTokens * st + p.head_k * sh < (1ll << 30) ? 1 : 0;
    }
    switch (fmt * 4 + pairs) {
        case 0: return launch_form<READ, Tag, 0, 0>(p, planes, stream);
        case kKvFp8 * 4: return launch_form<READ, Tag, kKvFp8, 0>(p, planes, stream);
        case kKvInt8 * 4: return launch_form<READ, Tag, kKvInt8, 0>(p, planes, stream);
        case kKvInt8 * 4 + 1: return launch_form<READ, Tag, kKvInt8, 1>(p, planes, stream);
        case kKvInt8 * 4 + 2: return launch_form<READ, Tag, kKvInt8, 2>(p, planes, stream);
        case kKvInt4 * 4: return launch_form<READ, Tag, kKvInt4, 0>(p, planes, stream);
        case kKvInt4 * 4 + 1: return launch_form<READ, Tag, kKvInt4, 1>(p, planes, stream);
        case kKvInt4 * 4 + 2: return launch_form<READ, Tag, kKvInt4, 2>(p, planes, stream);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace

hipError_t launch_kv_append(const KvCacheParams& p, bool is_bf16, int fmt, int pairs, int planes, hipStream_t stream) {
    // (a 16-bit row is copied whatever its type)
    return is_bf16 && fmt != 0 ? launch_tag<false, bf16_tag>(p, fmt, pairs, planes, stream)
                               : launch_tag<false, f16_tag>(p, fmt, pairs, planes, stream);
}

hipError_t launch_kv_read(const KvCacheParams& p, bool is_bf16, int fmt, int pairs, int planes, hipStream_t stream) {
    return is_bf16 && fmt != 0 ? launch_tag<true, bf16_tag>(p, fmt, pairs, planes, stream)
                               : launch_tag<true, f16_tag>(p, fmt, pairs, planes, stream);
}

}  // namespace da
