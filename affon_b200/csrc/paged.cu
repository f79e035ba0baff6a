// Kernels around a paged key/value cache: the plan of a step (rotation
// positions, cache slots and ancestor masks of the drafted trees), the
// rotation and append of the step's rows, and the greedy acceptance of a
// verified tree with the move of its rows.  All of them check the lengths,
// tables and indices that they read from device memory and report DEV_BOUNDS
// instead of following a bad one.  They move little data, so the small calls
// are bound by launch and memory latency and the large ones by HBM.
#include <cuda_runtime.h>

#include "common.cuh"
#include "internal.h"
#include "paged.cuh"
#include "sm100.cuh"

namespace afb {
namespace paged {

// ------------------------------------------------------------------- plan
// One CTA per sequence, a thread per node; one more CTA marks the padding
// rows.  Ancestors by pointer doubling: after round r a node's mask holds its
// nearest 2^r ancestors-or-self and `up` the next one, so 8 rounds cover 256
// nodes whatever the tree's depth; the depth is the mask's population minus 1.
constexpr int PLAN_THREADS = kMaxTreeNodes;

__global__ void __launch_bounds__(PLAN_THREADS) plan_kernel(PagedShape s, PagedStep t, int *positions, int *slots,
                                                           uint32_t *mask, unsigned *status) {
    __shared__ uint32_t sets[2][8][kMaxTreeNodes];
    __shared__ int ups[2][kMaxTreeNodes];
    pdl_launch_dependents();
    pdl_wait();
    const int tid = threadIdx.x, seq = blockIdx.x;
    if (seq == s.seqs) {  // rows outside every sequence
        const int64_t first = t.cu_nodes[0], last = t.cu_nodes[s.seqs];
        for (int64_t r = tid; r < s.rows; r += PLAN_THREADS) {
            if (r >= first && r < last) continue;
            positions[r] = 0;
            slots[r] = -1;
            for (int w = 0; w < s.mask_words; ++w) mask[r * s.mask_words + w] = 0u;
        }
        return;
    }
    const SeqSpan sp = seq_span(s, t, seq);
    if (!sp.ok) {  // no slot for any row that this sequence claims
        if (tid == 0) atomicExch(status, static_cast<unsigned>(DEV_BOUNDS));
        const int64_t first = max(sp.first, 0), last = min(sp.last, s.rows);
        for (int64_t r = first + tid; r < last; r += PLAN_THREADS) {
            positions[r] = 0;
            slots[r] = -1;
            for (int w = 0; w < s.mask_words; ++w) mask[r * s.mask_words + w] = 0u;
        }
        return;
    }
    const int n = sp.last - sp.first, words = (n + 31) >> 5;
    const int64_t row = static_cast<int64_t>(sp.first) + tid;
    int up = -1;
    if (tid < n) {
        up = t.parents ? t.parents[row] : tid - 1;
        if (up >= tid) {
            atomicExch(status, static_cast<unsigned>(DEV_BOUNDS));
            up = -1;
        }
        if (up < 0) up = -1;
        const int64_t place = static_cast<int64_t>(sp.ctx) + tid;
        const int page = t.page_table[static_cast<int64_t>(seq) * s.ld_table + (place >> s.page_shift)];
        const bool ok = page >= 0 && page < s.pages;
        if (!ok) atomicExch(status, static_cast<unsigned>(DEV_BOUNDS));
        slots[row] = ok ? static_cast<int>((static_cast<int64_t>(page) << s.page_shift) +
                                           (place & ((1 << s.page_shift) - 1)))
                        : -1;
        for (int w = 0; w < words; ++w) sets[0][w][tid] = w == (tid >> 5) ? 1u << (tid & 31) : 0u;
        ups[0][tid] = up;
    }
    int cur = 0;
    for (int reach = 1; __syncthreads_or(up >= 0 && tid < n) && reach <= kMaxTreeNodes; reach *= 2) {
        if (tid < n) {
            for (int w = 0; w < words; ++w)
                sets[cur ^ 1][w][tid] = sets[cur][w][tid] | (up >= 0 ? sets[cur][w][up] : 0u);
            up = up >= 0 ? ups[cur][up] : -1;
            ups[cur ^ 1][tid] = up;
        }
        cur ^= 1;
    }
    if (tid < n) {
        int size = 0;
        for (int w = 0; w < s.mask_words; ++w) {
            const uint32_t m = w < words ? sets[cur][w][tid] : 0u;
            size += __popc(m);
            mask[row * s.mask_words + w] = m;
        }
        positions[row] = sp.ctx + size - 1;
    }
}

// ----------------------------------------------------------------- append
// A thread rotates or copies 16 dims of one head of one row: two runs of 8
// (d and d + head_dim/2) or one of 16 (interleaved pairs, values).
template <bool F32>
__device__ __forceinline__ void load8(const void *base, int64_t at, float (&x)[8]) {
    if (F32) {
        const float4 *p = reinterpret_cast<const float4 *>(static_cast<const float *>(base) + at);
        const float4 a = p[0], b = p[1];
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
        const uint4 a = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(base) + at);
        const uint32_t u[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = __uint_as_float(u[i] << 16);
            x[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
        }
    }
}
__device__ __forceinline__ void store8(uint16_t *dst, const float (&x)[8]) {
    *reinterpret_cast<uint4 *>(dst) = make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]),
                                                 pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
}

template <bool F32>
__global__ void append_kernel(PagedShape s, AppendArgs a, unsigned *status) {
    pdl_launch_dependents();
    pdl_wait();
    const int chunks = s.head_dim >> 4, heads = a.q_heads + 2 * s.kv_heads;
    const int item = blockIdx.y * blockDim.x + threadIdx.x;
    const int64_t row = blockIdx.x;
    if (item >= heads * chunks) return;
    const int head = item / chunks, chunk = item % chunks, half = s.head_dim >> 1;
    const int slot = a.slots[row];
    if (slot == -1) return;
    const int pos = a.rope ? a.positions[row] : 0;
    if (slot < 0 || (slot >> s.page_shift) >= s.pages || (a.rope && (pos < 0 || pos >= a.table_rows))) {
        if (item == 0) atomicExch(status, static_cast<unsigned>(DEV_BOUNDS));
        return;
    }
    const int64_t place = (slot >> s.page_shift) * s.page_stride +
                          static_cast<int64_t>(slot & ((1 << s.page_shift) - 1)) * s.token_stride;
    const bool is_q = head < a.q_heads, is_v = head >= a.q_heads + s.kv_heads;
    const int kv = is_q ? 0 : is_v ? head - a.q_heads - s.kv_heads : head - a.q_heads;
    const int col = is_q ? a.q_off + head * s.head_dim : (is_v ? a.v_off : a.k_off) + kv * s.head_dim;
    uint16_t *dst = is_q ? a.q_out + row * a.ld_q + static_cast<int64_t>(head) * s.head_dim
                         : (is_v ? a.v_cache : a.k_cache) + place + kv * s.head_stride;
    const bool apart = a.rope == AFFON_B200_ROPE_HALF && !is_v;
    const int d0 = apart ? chunk * 8 : chunk * 16, d1 = apart ? d0 + half : d0 + 8;
    float x[8], y[8];
    load8<F32>(a.qkv, row * a.ld_qkv + col + d0, x);
    load8<F32>(a.qkv, row * a.ld_qkv + col + d1, y);
    if (a.rope && !is_v) {
        float c[8], sn[8];
        load8<true>(a.cos_t, static_cast<int64_t>(pos) * half + chunk * 8, c);
        load8<true>(a.sin_t, static_cast<int64_t>(pos) * half + chunk * 8, sn);
        if (apart) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float p = x[i], q = y[i];
                x[i] = p * c[i] - q * sn[i];
                y[i] = q * c[i] + p * sn[i];
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float p = x[2 * i], q = x[2 * i + 1];
                x[2 * i] = p * c[i] - q * sn[i];
                x[2 * i + 1] = q * c[i] + p * sn[i];
                p = y[2 * i], q = y[2 * i + 1];
                y[2 * i] = p * c[4 + i] - q * sn[4 + i];
                y[2 * i + 1] = q * c[4 + i] + p * sn[4 + i];
            }
        }
    }
    store8(dst + d0, x);
    store8(dst + d1, y);
}

// ----------------------------------------------------------------- accept
// Every CTA of a sequence walks its tree (a warp's ballots find the lowest
// fitting child; children have higher indices, so the walk ends) and moves
// its share of the rows: a thread owns 8 dims of one (layer, key or value,
// head) and takes the path in order.  path[i] >= i and both ascend, so a
// place is written only after every row that is read from it has been.  The
// last CTA of a sequence to finish writes the length, which may be the buffer
// that the others read theirs from.
constexpr int ACCEPT_THREADS = 256;
constexpr int MOVE_BATCH = 8;

__global__ void __launch_bounds__(ACCEPT_THREADS) accept_kernel(PagedShape s, PagedStep t, AcceptArgs a,
                                                                unsigned *counters, unsigned *status) {
    __shared__ int parent[kMaxTreeNodes], token[kMaxTreeNodes], next[kMaxTreeNodes], path[kMaxTreeNodes];
    __shared__ int64_t from[kMaxTreeNodes], to[kMaxTreeNodes];
    __shared__ int count_s, moves_s, last_s;
    pdl_launch_dependents();
    pdl_wait();
    const int tid = threadIdx.x, seq = blockIdx.x;
    const SeqSpan sp = seq_span(s, t, seq);
    if (!sp.ok) {
        if (tid == 0) atomicExch(status, static_cast<unsigned>(DEV_BOUNDS));
        return;
    }
    const int n = sp.last - sp.first;
    if (tid < n) {
        const int64_t row = static_cast<int64_t>(sp.first) + tid;
        const int up = t.parents ? t.parents[row] : tid - 1;
        parent[tid] = up < tid ? up : -1;
        token[tid] = a.tokens[row];
        next[tid] = a.predicted[row];
    }
    if (tid == 0) moves_s = 0;
    __syncthreads();
    if (tid < 32) {
        int count = 0;
        for (int cur = n > 0 ? 0 : -1; cur >= 0;) {
            if (tid == 0) path[count] = cur;
            ++count;
            const int want = next[cur];
            int found = -1;
            for (int base = cur + 1 - ((cur + 1) & 31); base < n && found < 0; base += 32) {
                const int i = base + tid;
                const unsigned hit = __ballot_sync(0xffffffffu, i > cur && i < n && parent[i] == cur && token[i] == want);
                if (hit) found = base + __ffs(hit) - 1;
            }
            cur = found;
        }
        if (tid == 0) count_s = count;
    }
    __syncthreads();
    const int count = count_s;
    // The rows that move, as element offsets of (page, position).
    if (tid < count && path[tid] != tid) {
        int64_t off[2];
        bool ok = true;
        for (int e = 0; e < 2; ++e) {
            const int64_t place = static_cast<int64_t>(sp.ctx) + (e ? tid : path[tid]);
            const int page = t.page_table[static_cast<int64_t>(seq) * s.ld_table + (place >> s.page_shift)];
            ok = ok && page >= 0 && page < s.pages;
            off[e] = page * s.page_stride + (place & ((1 << s.page_shift) - 1)) * s.token_stride;
        }
        if (!ok) atomicExch(status, static_cast<unsigned>(DEV_BOUNDS));
        from[tid] = ok ? off[0] : -1;
        to[tid] = off[1];
        atomicMax(&moves_s, tid + 1);
    } else if (tid < count) {
        from[tid] = -1;
    }
    __syncthreads();
    const int moves = moves_s;
    if (moves > 0) {
        const int runs = s.head_dim >> 3;
        const int64_t items = static_cast<int64_t>(a.layers) * 2 * s.kv_heads * runs;
        for (int64_t it = static_cast<int64_t>(blockIdx.y) * ACCEPT_THREADS + tid; it < items;
             it += static_cast<int64_t>(gridDim.y) * ACCEPT_THREADS) {
            const int run = static_cast<int>(it % runs);
            const int64_t h = it / runs;
            const int head = static_cast<int>(h % s.kv_heads);
            const int64_t lk = h / s.kv_heads;
            uint16_t *base = ((lk & 1) ? a.v_cache : a.k_cache) + (lk >> 1) * a.layer_stride + head * s.head_stride +
                             run * 8;
            for (int i = 1; i < moves; i += MOVE_BATCH) {
                uint4 x[MOVE_BATCH];
#pragma unroll
                for (int e = 0; e < MOVE_BATCH; ++e)
                    if (i + e < moves && from[i + e] >= 0) x[e] = *reinterpret_cast<const uint4 *>(base + from[i + e]);
#pragma unroll
                for (int e = 0; e < MOVE_BATCH; ++e)
                    if (i + e < moves && from[i + e] >= 0) *reinterpret_cast<uint4 *>(base + to[i + e]) = x[e];
            }
        }
    }
    if (blockIdx.y == 0) {
        if (tid < s.max_nodes) a.path[seq * a.ld_path + tid] = tid < count ? path[tid] : -1;
        if (tid == 0) {
            a.counts[seq] = count;
            a.next_tokens[seq] = count ? next[path[count - 1]] : -1;
        }
    }
    if (tid == 0) {
        last_s = gridDim.y == 1 || atomicAdd(&counters[seq], 1u) == gridDim.y - 1;
        if (last_s) {
            if (gridDim.y > 1) counters[seq] = 0u;
            a.lens_out[seq] = sp.ctx + count;
        }
    }
}

}  // namespace paged

static unsigned *status_word(void *workspace) { return static_cast<unsigned *>(workspace); }

cudaError_t launch_paged_plan(const PagedShape &s, const PagedStep &t, int *positions, int *slots, uint32_t *mask,
                              void *workspace, cudaStream_t stream, bool pdl) {
    cudaError_t e = launch_ex(paged::plan_kernel, dim3(s.seqs + 1), dim3(paged::PLAN_THREADS), 0, stream, false, pdl, s,
                              t, positions, slots, mask, status_word(workspace));
    count_launch();
    return e;
}

cudaError_t launch_paged_append(const PagedShape &s, const AppendArgs &a, void *workspace, cudaStream_t stream,
                                bool pdl) {
    const int items = (a.q_heads + 2 * s.kv_heads) * (s.head_dim >> 4);
    const dim3 grid(s.rows, (items + 127) / 128);
    cudaError_t e = a.x_f32 ? launch_ex(paged::append_kernel<true>, grid, dim3(128), 0, stream, false, pdl, s, a,
                                        status_word(workspace))
                            : launch_ex(paged::append_kernel<false>, grid, dim3(128), 0, stream, false, pdl, s, a,
                                        status_word(workspace));
    count_launch();
    return e;
}

cudaError_t launch_tree_accept(const PagedShape &s, const PagedStep &t, const AcceptArgs &a, void *workspace,
                               cudaStream_t stream, bool pdl) {
    const int64_t items = static_cast<int64_t>(a.layers) * 2 * s.kv_heads * (s.head_dim >> 3);
    int64_t ctas = (items + paged::ACCEPT_THREADS - 1) / paged::ACCEPT_THREADS;
    ctas = ctas < 1 ? 1 : ctas > 64 ? 64 : ctas;
    unsigned *counters = reinterpret_cast<unsigned *>(static_cast<char *>(workspace) + kCounterOffset);
    cudaError_t e = launch_ex(paged::accept_kernel, dim3(s.seqs, static_cast<unsigned>(ctas)),
                              dim3(paged::ACCEPT_THREADS), 0, stream, false, pdl, s, t, a, counters,
                              status_word(workspace));
    count_launch();
    return e;
}

}  // namespace afb
