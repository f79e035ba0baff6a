// Attention of a step's drafted nodes over a paged key/value cache.
//
// For a row (node i of sequence s) and query head h with KV head h / G:
//   o = sum_t p_t v_t / sum_t p_t,  p_t = exp(scale q.k_t - m)
// over the sequence's cached positions and the drafted ones that the row's
// mask names, in one pass with a running maximum m and running sums in f32.
// A warp owns one (row, head), a lane 4 (2) of its 128 (64) dims.
#include <cuda_runtime.h>

#include "common.cuh"
#include "internal.h"
#include "paged.cuh"
#include "sm100.cuh"

namespace afb {
namespace tattn {

__device__ __forceinline__ int out_column(int d, int pair_order) {
    const int e = d & 7;
    return pair_order ? (d & ~7) + (e < 4 ? 2 * e : 2 * (e - 4) + 1) : d;
}

template <int HD>
__global__ void tree_attention_kernel(PagedShape s, PagedStep t, TreeAttnArgs a, unsigned *status) {
    constexpr int W = HD / 32;
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31, head = blockIdx.y * (blockDim.x >> 5) + (threadIdx.x >> 5);
    const int row = blockIdx.x;
    if (head >= a.q_heads) return;
    if (row < t.cu_nodes[0] || row >= t.cu_nodes[s.seqs]) return;
    int lo = 0, hi = s.seqs;  // the last sequence that starts at or before the row
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (t.cu_nodes[mid] <= row) lo = mid;
        else hi = mid;
    }
    const SeqSpan sp = seq_span(s, t, lo);
    if (!sp.ok || row < sp.first || row >= sp.last) {
        if (lane == 0) atomicExch(status, static_cast<unsigned>(DEV_BOUNDS));
        return;
    }
    const int n = sp.last - sp.first, node = row - sp.first, kvh = head / (a.q_heads / s.kv_heads);
    float q[W], o[W], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int e = 0; e < W; ++e) {
        q[e] = bf16_bits_to_f32(a.q[row * a.ld_q + head * HD + lane * W + e]) * a.scale;
        o[e] = 0.0f;
    }
    for (int pos = 0; pos < sp.ctx + n; ++pos) {
        if (pos >= sp.ctx) {
            const int j = pos - sp.ctx;
            const bool see = a.mask ? (a.mask[static_cast<int64_t>(row) * s.mask_words + (j >> 5)] >> (j & 31)) & 1u
                                    : j <= node;
            if (!see) continue;
        }
        const int page = t.page_table[static_cast<int64_t>(lo) * s.ld_table + (pos >> s.page_shift)];
        const bool ok = page >= 0 && page < s.pages;
        if (!ok && lane == 0) atomicExch(status, static_cast<unsigned>(DEV_BOUNDS));
        const int64_t at = page * s.page_stride + kvh * s.head_stride +
                           (pos & ((1 << s.page_shift) - 1)) * s.token_stride + lane * W;
        float sc = 0.0f;
        for (int e = 0; e < W; ++e) sc += q[e] * (ok ? bf16_bits_to_f32(a.k_cache[at + e]) : 0.0f);
        for (int x = 16; x; x >>= 1) sc += __shfl_xor_sync(0xffffffffu, sc, x);
        const float mn = fmaxf(m, sc);
        const float corr = m == -INFINITY ? 0.0f : expf(m - mn), p = expf(sc - mn);
        m = mn;
        l = l * corr + p;
        for (int e = 0; e < W; ++e) o[e] = o[e] * corr + p * (ok ? bf16_bits_to_f32(a.v_cache[at + e]) : 0.0f);
    }
#pragma unroll
    for (int e = 0; e < W; ++e)
        a.out[row * a.ld_out + head * HD + out_column(lane * W + e, a.out_pair_order)] =
            f32_to_bf16_bits(l == 0.0f ? 0.0f : o[e] / l);
}

}  // namespace tattn

cudaError_t launch_tree_attention(const PagedShape &s, const PagedStep &t, const TreeAttnArgs &a, void *workspace,
                                  int num_sms, cudaStream_t stream, bool pdl) {
    const dim3 grid(s.rows, (a.q_heads + 3) / 4);
    unsigned *status = static_cast<unsigned *>(workspace);
    cudaError_t e = s.head_dim == 128
                        ? launch_ex(tattn::tree_attention_kernel<128>, grid, dim3(128), 0, stream, false, pdl, s, t, a,
                                    status)
                        : launch_ex(tattn::tree_attention_kernel<64>, grid, dim3(128), 0, stream, false, pdl, s, t, a,
                                    status);
    count_launch();
    return e;
}

}  // namespace afb
