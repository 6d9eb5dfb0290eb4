// Merge of the shared-prefix kernel's partials: prefix splits first, then the sequence's own, one thread per (row, four
// columns), in that order (deterministic).
#include "da_prefix.h"

namespace da {
namespace {

template <typename Tag, int D>
__global__ __launch_bounds__(256) void prefix_merge_kernel(const PrefixParams p) {
    using EL = Elem<Tag>;
    constexpr int C4 = D / 4;
    const SweepParams& w = p.own;
    const int rows = w.batch * w.head_q;
    const long long gid = (long long)blockIdx.x * 256 + threadIdx.x;
    const int row = (int)(gid / C4), c4 = (int)(gid % C4);
    if (row >= rows) return;
    const int b = row / w.head_q;
    int own, np = p.splits;
    if (p.table) {
        const int len = w.seq_lens[b];
        own = len - p.prefix_len;
        if (own < 0) np = own = 0;  // (a row of the batch without a sequence)
    } else {
        own = w.cu_seq_k[b + 1] - w.cu_seq_k[b];
    }
    const int ns = own > 0 ? min(w.nsplit, (own + w.chunk - 1) / w.chunk) : 0;
    float mm = kNegBig, den = 0.0f;
    f32x4 num = {0.0f, 0.0f, 0.0f, 0.0f};
    auto add = [&](const float* ml, const float* o, size_t first, size_t stride, int count) {
        for (int s0 = 0; s0 < count; s0 += 4) {
            float2 e[4];
            f32x4 x[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const size_t part = first + (size_t)min(s0 + u, count - 1) * stride;
                e[u] = reinterpret_cast<const float2*>(ml)[part];
                x[u] = reinterpret_cast<const f32x4*>(o)[part * C4 + c4];
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                if (s0 + u >= count) break;
                const float mn = fmaxf(mm, e[u].x);
                const float keep = fast_exp2(mm - mn), wt = fast_exp2(e[u].x - mn);
                mm = mn;
                den = den * keep + e[u].y * wt;
                num = num * keep + x[u] * wt;
            }
        }
    };
    add(p.ws_ml, p.ws_o, row, rows, np);
    add(w.ws_ml, w.ws_o, (size_t)row * w.nsplit, 1, ns);
    const float inv = np + ns > 0 ? 1.0f / den : 0.0f;
    uint2 r;
    r.x = EL::pack2(num[0] * inv, num[1] * inv);
    r.y = EL::pack2(num[2] * inv, num[3] * inv);
    *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(w.o) + (size_t)row * D + c4 * 4) = r;
}

template <int D>
hipError_t launch_dim(const PrefixParams& p, bool is_bf16, hipStream_t stream) {
    const long long threads = (long long)p.own.batch * p.own.head_q * (D / 4);
    const dim3 grid((unsigned)((threads + 255) / 256));
    if (is_bf16)
        hipLaunchKernelGGL((prefix_merge_kernel<bf16_tag, D>), grid, dim3(256), 0, stream, p);
    else
        hipLaunchKernelGGL((prefix_merge_kernel<f16_tag, D>), grid, dim3(256), 0, stream, p);
    return hipGetLastError();
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
