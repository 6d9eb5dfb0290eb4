// Merge of the shared-prefix kernel's partials: a row's prefix splits and its own ones are dealt out over G threads (partial
// j to thread j mod G), each adds up its share with a running maximum, and the G sums meet in LDS in thread order, so the result
// does not depend on timing.  One thread per (row, four columns, share).
//
// Bound by the trips to memory that a thread makes one after the other, 3 to 4 us for the smallest call (the length, the partials'
// places, the partials); large ones read at 3 TB/s what the sweep has just written past the L2 (8192 rows of d 128, five partials
// each, 21 MB: 7 us; 1056 rows of d 256 and 17 partials, 18 MB: 5.8).  With G = 1 and 20 partials of 2048 rows (17 MB, d 128) the
// merge took 9.3 us, half of its sweep's time.
#include "da_prefix.h"

namespace da {
namespace {

template <typename Tag, int D, int G>
__global__ __launch_bounds__(256) void prefix_merge_kernel(const PrefixParams p) {
    using EL = Elem<Tag>;
    constexpr int C4 = D / 4, R = prefix_merge_rows(D, G);
    static_assert(R >= 1 && R * G * C4 <= 256, "shape");
    __shared__ f32x4 nums[G][R][C4];
    __shared__ float2 mls[G][R];
    const SweepParams& w = p.own;
    const int rows = w.batch * w.head_q;
    const int c4 = threadIdx.x % C4, rg = threadIdx.x / C4, r = rg % R, g = rg / R;
    const int row = (int)blockIdx.x * R + r;
    const bool live = rg < R * G && row < rows;
    int np = 0, ns = 0;
    float mm = kNegBig, den = 0.0f;
    f32x4 num = {0.0f, 0.0f, 0.0f, 0.0f};
    if (live) {
        // Four partials at a time.  The first four are asked for before the sequence's length is known, as far as they are the
        // prefix's: their trip to memory runs beside the length's.
        float2 e[4];
        f32x4 x[4];
        auto fetch = [&](const float* ml, const float* o, size_t part, int u) __attribute__((always_inline)) {
            e[u] = reinterpret_cast<const float2*>(ml)[part];
            x[u] = reinterpret_cast<const f32x4*>(o)[part * C4 + c4];
        };
#pragma unroll
        for (int u = 0; u < 4; ++u) fetch(p.ws_ml, p.ws_o, (size_t)min(g + u * G, p.splits - 1) * rows + row, u);
        const int b = row / w.head_q;
        int own = p.table ? w.seq_lens[b] - p.prefix_len : w.cu_seq_k[b + 1] - w.cu_seq_k[b];
        np = own < 0 ? 0 : p.splits;  // (a row of the batch without a sequence)
        // own partial j of the row lies in workspace row own0 + j * stride
        size_t own0 = (size_t)row * w.nsplit, stride = 1;
        if (own > 0 && w.flat_wgs > 0) {
            const int lo = w.flat_cu[b], hi = w.flat_cu[b + 1];
            const int T = flat_share(w.flat_cu[w.batch], w.flat_wgs, w.flat_step, w.flat_min);
            const int first = min(lo / T, w.flat_wgs - 1);
            ns = min((hi - 1) / T, w.flat_wgs - 1) - first + 1;
            own0 = (size_t)(first + b) * w.head_q + (size_t)(row - b * w.head_q);
            stride = (size_t)w.head_q;
        } else if (own > 0) {
            ns = min(w.nsplit, (own + w.chunk - 1) / w.chunk);
        }
        const int count = np + ns;
        for (int j0 = g; j0 < count; j0 += 4 * G) {
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int j = min(j0 + u * G, count - 1);
                if (j >= np)
                    fetch(w.ws_ml, w.ws_o, own0 + (size_t)(j - np) * stride, u);
                else if (j0 != g)
                    fetch(p.ws_ml, p.ws_o, (size_t)j * rows + row, u);
            }
            float mn = mm;
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (j0 + u * G < count) mn = fmaxf(mn, e[u].x);
            const float keep = fast_exp2(mm - mn);
            mm = mn;
            den *= keep;
            num *= keep;
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                if (j0 + u * G >= count) break;
                const float wt = fast_exp2(e[u].x - mn);
                den += e[u].y * wt;
                num += x[u] * wt;
            }
        }
    }
    if constexpr (G > 1) {
        if (live) {
            nums[g][r][c4] = num;
            if (c4 == 0) mls[g][r] = make_float2(mm, den);
        }
        __syncthreads();
        if (!live || g != 0) return;
        float top = mm;
#pragma unroll
        for (int i = 1; i < G; ++i) top = fmaxf(top, mls[i][r].x);
        const float keep = fast_exp2(mm - top);
        den *= keep;
        num *= keep;
#pragma unroll
        for (int i = 1; i < G; ++i) {
            const float wt = fast_exp2(mls[i][r].x - top);
            den += mls[i][r].y * wt;
            num += nums[i][r][c4] * wt;
        }
    } else if (!live) {
        return;
    }
    const float inv = np + ns > 0 ? 1.0f / den : 0.0f;
    uint2 o;
    o.x = EL::pack2(num[0] * inv, num[1] * inv);
    o.y = EL::pack2(num[2] * inv, num[3] * inv);
    *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(w.o) + (size_t)row * D + c4 * 4) = o;
}

template <typename Tag, int D, int G>
hipError_t launch_one(const PrefixParams& p, hipStream_t stream) {
    constexpr int R = prefix_merge_rows(D, G);
    const unsigned rows = (unsigned)(p.own.batch * p.own.head_q);
    hipLaunchKernelGGL((prefix_merge_kernel<Tag, D, G>), dim3((rows + R - 1) / R), dim3(256), 0, stream, p);
    return hipGetLastError();
}

template <int D>
hipError_t launch_dim(const PrefixParams& p, bool is_bf16, hipStream_t stream) {
    const bool shares = prefix_merge_shares(p.splits, p.own.nsplit) > 1;
    if (is_bf16) return shares ? launch_one<bf16_tag, D, 4>(p, stream) : launch_one<bf16_tag, D, 1>(p, stream);
    return shares ? launch_one<f16_tag, D, 4>(p, stream) : launch_one<f16_tag, D, 1>(p, stream);
}

}  // namespace

hipError_t launch_prefix_merge(const PrefixParams& p, bool is_bf16, int dim, hipStream_t stream) {
    switch (dim) {
        case 64: return launch_dim<64>(p, is_bf16, stream);
        case 96: return launch_dim<96>(p, is_bf16, stream);
        case 128: return launch_dim<128>(p, is_bf16, stream);
        default: return launch_dim<256>(p, is_bf16, stream);
    }
}

}  // namespace da
