// K/V rows written into a paged cache, quantised on the way (append), and read back as 16-bit rows (read).
//
// Both kernels move a row in chunks of eight elements, one chunk a lane.  A work-group takes a few consecutive tokens of
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
#include "da_kv_cache.h"

namespace da {
namespace {

constexpr int kThreads = 256;
constexpr int kUnroll = 4;        // chunks a thread holds at once
constexpr int kMaxTokens = 128;   // most tokens of a work-group

// i / d for 0 <= i < 2^16 * 2^11, d <= 2^16, by m = ceil(2^32 / d): the excess of m is below 2^-32 d, so the quotient is
// right while i * d < 2^32 (here i < 2048 + d and the two never reach it together: a work-group holds at most
// kThreads * kUnroll chunks, or the chunks of one token)
__device__ __forceinline__ int magic_div(int i, uint32_t m) { return (int)__umulhi((uint32_t)i, m); }

// Row of the pools where token t lies, -1 if it lies nowhere: a token's sequence ends at seq_lens[b], and the tokens of
// the call are its last ones.  Bounds are checked here, for the row is written: a position before the sequence's first
// token (a padded sequence of no tokens), behind the block table, or a page that the pools do not have.
__device__ __forceinline__ int64_t pool_row(const KvCacheParams& p, int b, int64_t pos) {
    if (pos < 0 || (pos >> p.page_shift) >= p.max_blocks) return -1;
    const int page = p.block_table[(int64_t)b * p.max_blocks + (pos >> p.page_shift)];
    if ((uint32_t)page >= (uint32_t)p.num_pages) return -1;
    return ((int64_t)page << p.page_shift) + (pos & ((1 << p.page_shift) - 1));
}

// (-1: the token lies nowhere in the pools; kBehind: it lies behind the last sequence, nothing is done for it at all)
constexpr int64_t kBehind = -2;

__device__ __forceinline__ int64_t token_row(const KvCacheParams& p, int64_t t) {
    if (t >= p.tokens) return kBehind;
    if (p.cu_seq == nullptr) return pool_row(p, (int)t, (int64_t)p.seq_lens[t] - 1);
    if (t >= p.cu_seq[p.batch] || t < p.cu_seq[0]) return kBehind;
    int lo = 0, n = p.batch;  // cu_seq[lo] <= t < cu_seq[lo + n]
    while (n > 1) {
        const int half = n >> 1;
        if (p.cu_seq[lo + half] <= t) {
            lo += half;
            n -= half;
        } else {
            n = half;
        }
    }
    return pool_row(p, lo, (int64_t)p.seq_lens[lo] - (p.cu_seq[lo + 1] - t));
}

// Looks the work-group's rows up, one thread a token.
__device__ __forceinline__ void find_rows(const KvCacheParams& p, int64_t tok0, int64_t* rows) {
    if ((int)threadIdx.x < p.tokens_per_block) rows[threadIdx.x] = token_row(p, tok0 + threadIdx.x);
    __syncthreads();
}

template <typename Tag>
__device__ __forceinline__ void widen8(uint4 w, float (&x)[8]) {
    using EL = Elem<Tag>;
    x[0] = EL::lo(w.x), x[1] = EL::hi(w.x), x[2] = EL::lo(w.y), x[3] = EL::hi(w.y);
    x[4] = EL::lo(w.z), x[5] = EL::hi(w.z), x[6] = EL::lo(w.w), x[7] = EL::hi(w.w);
}

// A double rounded to a float whose last bit is set whenever the float is not exact: a second rounding, to a format of at
// least two bits fewer, then comes out as if it were the only one.
__device__ __forceinline__ float round_to_odd(double y) {
    const float f = (float)y;
    if ((double)f == y || y != y) return f;
    uint32_t u = __float_as_uint(f);
    if (fabs((double)f) > fabs(y)) --u;
    return __uint_as_float(u | 1u);
}

// the nearest integer, clamped to [LO, HI] (a NaN becomes 0)
template <int LO, int HI>
__device__ __forceinline__ int to_int(double y) {
    y = y < (double)LO ? (double)LO : (y > (double)HI ? (double)HI : y);
    return (int)rint(y);
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

// Eight quantised integers to the pool: 8 bytes (int8) or 4 bytes (int4) of the chunk.
template <int FMT>
__device__ __forceinline__ void store_ints(uint8_t* pool, int64_t elem, const int (&n)[8]) {
    if constexpr (FMT == kKvInt8) {
        uint2 w;
        w.x = (uint32_t)(n[0] & 255) | (uint32_t)(n[1] & 255) << 8 | (uint32_t)(n[2] & 255) << 16 | (uint32_t)n[3] << 24;
        w.y = (uint32_t)(n[4] & 255) | (uint32_t)(n[5] & 255) << 8 | (uint32_t)(n[6] & 255) << 16 | (uint32_t)n[7] << 24;
        *reinterpret_cast<uint2*>(pool + elem) = w;
    } else {
        uint32_t w = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) w |= (uint32_t)(n[j] & 15) << (4 * j);
        *reinterpret_cast<uint32_t*>(pool + (elem >> 1)) = w;
    }
}

// lo and hi over the lanes that hold a row (or a run): a NaN anywhere makes both a NaN
__device__ __forceinline__ float min_nan(float a, float b) { return (b < a || b != b) ? b : a; }
__device__ __forceinline__ float max_nan(float a, float b) { return (b > a || b != b) ? b : a; }

template <typename Tag, int FMT, int PAIRS>
__global__ __launch_bounds__(kThreads) void kv_append_kernel(const KvCacheParams p) {
    __shared__ int64_t rows[kMaxTokens];
    const KvPlane& pl = p.plane[blockIdx.y];
    const int64_t tok0 = (int64_t)blockIdx.x * p.tokens_per_block;
    const int lanes = pl.dim >> 3, chunks = p.head_k * lanes;
    const int n = (int)min((int64_t)p.tokens_per_block, p.tokens - tok0) * chunks;
    uint8_t* const pool = reinterpret_cast<uint8_t*>(pl.pool);
    bool looked = false;
    for (int base = 0; base < n; base += kThreads * kUnroll) {
        uint4 w[kUnroll];
        int tok[kUnroll], head[kUnroll], ch[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const int i = min(base + u * kThreads + (int)threadIdx.x, n - 1);
            tok[u] = magic_div(i, pl.chunks_magic);
            const int c = i - tok[u] * chunks;
            head[u] = magic_div(c, pl.lanes_magic);
            ch[u] = c - head[u] * lanes;
            const uint16_t* const src = reinterpret_cast<const uint16_t*>(pl.src) + (tok0 + tok[u]) * pl.src_token +
                                        head[u] * pl.src_head + ch[u] * 8;
            if (pl.aligned) {
                w[u] = stream_load16(src);
            } else {
                uint32_t e[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) e[j] = src[j];
                w[u] = make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
            }
        }
        if (!looked) {
            find_rows(p, tok0, rows);
            looked = true;
        }
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            if (base + u * kThreads + (int)threadIdx.x >= n) break;
            const int64_t row = rows[tok[u]];
            const int64_t page = row >> p.page_shift;
            const int64_t elem = page * pl.page + ((row & ((1 << p.page_shift) - 1)) * p.head_k + head[u]) * pl.dim + ch[u] * 8;
            if constexpr (FMT == 0) {
                if (row >= 0) *reinterpret_cast<uint4*>(pool + elem * 2) = w[u];
                continue;
            }
            float x[8];
            widen8<Tag>(w[u], x);
            if constexpr (FMT == kKvFp8) {
                const double s = pl.scale ? (double)pl.scale[head[u]] : 1.0;
                float f[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    double y = (double)x[j] / s;
                    y = y > 448.0 ? 448.0 : (y < -448.0 ? -448.0 : y);
                    f[j] = round_to_odd(y);
                }
                uint2 b;
                b.x = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(f[0], f[1], 0, false);
                b.x = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(f[2], f[3], (int)b.x, true);
                b.y = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(f[4], f[5], 0, false);
                b.y = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(f[6], f[7], (int)b.y, true);
                if (row >= 0) *reinterpret_cast<uint2*>(pool + elem) = b;
            } else if constexpr (FMT == kKvInt8 || FMT == kKvInt4) {
                constexpr int QLO = Range<FMT>::lo, QHI = Range<FMT>::hi;
                double s = 1.0, z = 0.0;
                if constexpr (PAIRS == 0) {
                    if (pl.scale) s = (double)pl.scale[head[u]];
                } else {
                    float lo = x[0], hi = x[0];
#pragma unroll
                    for (int j = 1; j < 8; ++j) {
                        lo = min_nan(lo, x[j]);
                        hi = max_nan(hi, x[j]);
                    }
                    // (a row's lanes are neighbours and start at a multiple of their number, a power of two)
                    const int span = PAIRS == 2 ? 8 : lanes;
                    for (int d = 1; d < span; d <<= 1) {
                        lo = min_nan(lo, __shfl_xor(lo, d));
                        hi = max_nan(hi, __shfl_xor(hi, d));
                    }
                    float sf = (float)(((double)hi - (double)lo) / (double)(QHI - QLO));
                    sf = sf < 1e-8f ? 1e-8f : sf;
                    const float zf = (float)((double)QLO - (double)lo / (double)sf);
                    s = (double)sf;
                    z = (double)zf;
                    if (row >= 0 && (ch[u] & (span - 1)) == 0) {
                        const int runs = PAIRS == 2 ? lanes >> 3 : 1;
                        const int64_t at = (row * p.head_k + head[u]) * runs + (PAIRS == 2 ? ch[u] >> 3 : 0);
                        reinterpret_cast<float2*>(pl.scale)[at] = make_float2(sf, zf);
                    }
                }
                int q[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) q[j] = to_int<QLO, QHI>((double)x[j] / s + z);
                if (row >= 0) store_ints<FMT>(pool, elem, q);
            }
        }
    }
}

template <typename Tag, int FMT, int PAIRS>
__global__ __launch_bounds__(kThreads) void kv_read_kernel(const KvCacheParams p) {
    using EL = Elem<Tag>;
    __shared__ int64_t rows[kMaxTokens];
    const KvPlane& pl = p.plane[blockIdx.y];
    const int64_t tok0 = (int64_t)blockIdx.x * p.tokens_per_block;
    const int lanes = pl.dim >> 3, chunks = p.head_k * lanes;
    const int n = (int)min((int64_t)p.tokens_per_block, p.tokens - tok0) * chunks;
    const uint8_t* const pool = reinterpret_cast<const uint8_t*>(pl.pool);
    find_rows(p, tok0, rows);
    for (int base = 0; base < n; base += kThreads * kUnroll) {
        uint4 w[kUnroll];
        float2 pair[kUnroll];
        int64_t out[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const int i = min(base + u * kThreads + (int)threadIdx.x, n - 1);
            const int tok = magic_div(i, pl.chunks_magic);
            const int c = i - tok * chunks;
            const int head = magic_div(c, pl.lanes_magic);
            const int ch = c - head * lanes;
            const int64_t row = rows[tok];
            out[u] = row == kBehind ? -1 : ((tok0 + tok) * chunks + c) * 8;
            w[u] = make_uint4(0u, 0u, 0u, 0u);
            pair[u] = make_float2(0.0f, 0.0f);  // (a token that lies nowhere reads as zeros)
            if (row < 0) continue;
            const int64_t elem = (row >> p.page_shift) * pl.page +
                                 ((row & ((1 << p.page_shift) - 1)) * p.head_k + head) * pl.dim + ch * 8;
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
                const int64_t at = PAIRS == 2 ? (row * p.head_k + head) * (lanes >> 3) + (ch >> 3) : row * p.head_k + head;
                pair[u] = reinterpret_cast<const float2*>(pl.scale)[at];
            } else if constexpr (FMT != 0) {
                pair[u].x = pl.scale ? pl.scale[head] : 1.0f;
            }
        }
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            if (base + u * kThreads + (int)threadIdx.x >= n) break;
            if (out[u] < 0) continue;
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
            *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(pl.dst) + out[u]) = r;
        }
    }
}

// Tokens per work-group: a thread holds up to kUnroll chunks, fewer while that leaves CUs without a work-group.
int tokens_per_block(const KvCacheParams& p, int planes) {
    const int chunks = p.head_k * (p.plane[0].dim >> 3);
    int tpb = kThreads * kUnroll / chunks;
    while (tpb > 1 && (p.tokens + tpb - 1) / tpb * planes < 512) tpb >>= 1;
    return tpb < 1 ? 1 : (tpb > kMaxTokens ? kMaxTokens : tpb);
}

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
    p.tokens_per_block = tokens_per_block(p, planes);
    for (int i = 0; i < planes; ++i) {
        const uint64_t lanes = (uint64_t)p.plane[i].dim >> 3, chunks = lanes * (uint64_t)p.head_k;
        p.plane[i].lanes_magic = (uint32_t)(((1ull << 32) + lanes - 1) / lanes);
        p.plane[i].chunks_magic = (uint32_t)(((1ull << 32) + chunks - 1) / chunks);
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
