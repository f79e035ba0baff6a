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
// A thread takes 16 dims of up to HEADS heads of one row, in two runs of 8 (d
// and d + head_dim/2, or 16 in a row for interleaved pairs and values): the
// row's 16 table values are loaded once for all of them, and all loads are
// issued before the first is used.  Bound by HBM where there are many rows:
// 13,921 rows of 8 + 8 + 32 heads of 128 (349 MB) take 59.5 us (5.9 TB/s,
// 0.90 of the copy rate; one head a thread, which reads the tables again for
// every head, took 69), from f32 (520 MB) 86 us, with interleaved pairs 60.5
// and 90.
constexpr int APPEND_HEADS = 4, APPEND_THREADS = 128;

template <bool F32>
struct Run8 {
    uint4 a, b;  // b: f32 only
    __device__ __forceinline__ void load(const void *base, int64_t at) {
        if (F32) {
            const uint4 *p = reinterpret_cast<const uint4 *>(static_cast<const float *>(base) + at);
            a = __ldg(p), b = __ldg(p + 1);
        } else {
            a = __ldg(reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(base) + at));
        }
    }
    __device__ __forceinline__ void get(float (&x)[8]) const {
        const uint32_t u[4] = {a.x, a.y, a.z, a.w}, w[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (F32) {
                x[i] = __uint_as_float(u[i]);
                x[4 + i] = __uint_as_float(w[i]);
            } else {
                x[2 * i] = __uint_as_float(u[i] << 16);
                x[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
            }
        }
    }
};
__device__ __forceinline__ void store8(uint16_t *dst, const float (&x)[8]) {
    *reinterpret_cast<uint4 *>(dst) = make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]),
                                                 pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
}

template <bool F32>
__global__ void __launch_bounds__(APPEND_THREADS) append_kernel(PagedShape s, AppendArgs a, unsigned per_row,
                                                                unsigned *status) {
    pdl_launch_dependents();
    pdl_wait();
    const int chunks = s.head_dim >> 4, heads = a.q_heads + 2 * s.kv_heads, half = s.head_dim >> 1;
    const int64_t item = static_cast<int64_t>(blockIdx.x) * APPEND_THREADS + threadIdx.x;
    // per_row items a row; a block's items start in one row and reach into at most APPEND_THREADS more
    const int64_t row0 = gridDim.x < 1u << 24 ? blockIdx.x * APPEND_THREADS / per_row
                                              : static_cast<int64_t>(blockIdx.x) * APPEND_THREADS / per_row;
    const unsigned within = static_cast<unsigned>(item - row0 * per_row);
    const int64_t row = row0 + within / per_row;
    if (row >= s.rows) return;
    const int rest = within % per_row, chunk = rest % chunks, head0 = rest / chunks * APPEND_HEADS;
    const int slot = a.slots[row];
    if (slot == -1) return;
    const int pos = a.rope ? a.positions[row] : 0;
    if (slot < 0 || (slot >> s.page_shift) >= s.pages || (a.rope && (pos < 0 || pos >= a.table_rows))) {
        if (rest == 0) atomicExch(status, static_cast<unsigned>(DEV_BOUNDS));
        return;
    }
    const bool half_pairs = a.rope == AFFON_B200_ROPE_HALF;
    Run8<F32> x0[APPEND_HEADS], x1[APPEND_HEADS];
#pragma unroll
    for (int i = 0; i < APPEND_HEADS; ++i) {
        const int head = head0 + i;
        if (head >= heads) break;
        const bool is_v = head >= a.q_heads + s.kv_heads;
        const int col = head < a.q_heads ? a.q_off + head * s.head_dim
                        : is_v           ? a.v_off + (head - a.q_heads - s.kv_heads) * s.head_dim
                                         : a.k_off + (head - a.q_heads) * s.head_dim;
        const bool apart = half_pairs && !is_v;
        const int d0 = apart ? chunk * 8 : chunk * 16;
        x0[i].load(a.qkv, row * a.ld_qkv + col + d0);
        x1[i].load(a.qkv, row * a.ld_qkv + col + (apart ? d0 + half : d0 + 8));
    }
    float c[8], sn[8];
    if (a.rope && head0 < a.q_heads + s.kv_heads) {
        Run8<true> t0, t1;
        t0.load(a.cos_t, static_cast<int64_t>(pos) * half + chunk * 8);
        t1.load(a.sin_t, static_cast<int64_t>(pos) * half + chunk * 8);
        t0.get(c), t1.get(sn);
    }
    const int64_t place = (slot >> s.page_shift) * s.page_stride +
                          static_cast<int64_t>(slot & ((1 << s.page_shift) - 1)) * s.token_stride;
#pragma unroll
    for (int i = 0; i < APPEND_HEADS; ++i) {
        const int head = head0 + i;
        if (head >= heads) break;
        const bool is_q = head < a.q_heads, is_v = head >= a.q_heads + s.kv_heads;
        const int kv = is_q ? 0 : is_v ? head - a.q_heads - s.kv_heads : head - a.q_heads;
        uint16_t *dst = is_q ? a.q_out + row * a.ld_q + static_cast<int64_t>(head) * s.head_dim
                             : (is_v ? a.v_cache : a.k_cache) + place + kv * s.head_stride;
        const bool apart = half_pairs && !is_v;
        const int d0 = apart ? chunk * 8 : chunk * 16, d1 = apart ? d0 + half : d0 + 8;
        float x[8], y[8];
        x0[i].get(x), x1[i].get(y);
        if (a.rope && !is_v) {
            if (apart) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float p = x[e], q = y[e];
                    x[e] = p * c[e] - q * sn[e];
                    y[e] = q * c[e] + p * sn[e];
                }
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float p = x[2 * e], q = x[2 * e + 1];
                    x[2 * e] = p * c[e] - q * sn[e];
                    x[2 * e + 1] = q * c[e] + p * sn[e];
                    p = y[2 * e], q = y[2 * e + 1];
                    y[2 * e] = p * c[4 + e] - q * sn[4 + e];
                    y[2 * e + 1] = q * c[4 + e] + p * sn[4 + e];
                }
            }
        }
        store8(dst + d0, x);
        store8(dst + d1, y);
    }
}

// ----------------------------------------------------------------- accept
// Every CTA of a sequence walks its tree (a warp's ballots find the lowest
// fitting child; children have higher indices, so the walk ends) and moves
// its share of the rows: a thread owns 8 dims of one (layer, key or value,
// head) and takes the path in order.  path[i] >= i and both ascend, so a
// place is written only after every row that is read from it has been.  The
// last CTA of a sequence to finish writes the length, which may be the buffer
// that the others read theirs from.  The pages of all nodes' positions are
// read with the tree, so that a path over positions without a page (nothing
// was appended there) is found before any of it is accepted.
constexpr int ACCEPT_THREADS = 256;
constexpr int MOVE_BATCH = 8;

__global__ void __launch_bounds__(ACCEPT_THREADS) accept_kernel(PagedShape s, PagedStep t, AcceptArgs a,
                                                                unsigned *counters, unsigned *status) {
    __shared__ int parent[kMaxTreeNodes], token[kMaxTreeNodes], next[kMaxTreeNodes], path[kMaxTreeNodes];
    __shared__ int64_t place_of[kMaxTreeNodes];  // element offset of (page, position) of a node, -1: no page
    __shared__ int count_s, first_s, last_s;
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
        const int64_t place = static_cast<int64_t>(sp.ctx) + tid;
        const int page = t.page_table[static_cast<int64_t>(seq) * s.ld_table + (place >> s.page_shift)];
        parent[tid] = up < tid ? up : -1;
        token[tid] = a.tokens[row];
        next[tid] = a.predicted[row];
        place_of[tid] = page >= 0 && page < s.pages
                            ? page * s.page_stride + (place & ((1 << s.page_shift) - 1)) * s.token_stride
                            : -1;
    }
    if (tid == 0) first_s = kMaxTreeNodes;  // the first node that moves: all behind it do
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
    // Every CTA of the sequence comes to the same answer.
    if (__syncthreads_or(tid < count && (place_of[tid] < 0 || place_of[path[tid]] < 0))) {
        if (tid == 0) atomicExch(status, static_cast<unsigned>(DEV_BOUNDS));
        return;
    }
    if (tid < count && path[tid] != tid) atomicMin(&first_s, tid);
    __syncthreads();
    if (first_s < count) {
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
            for (int i = first_s; i < count; i += MOVE_BATCH) {
                uint4 x[MOVE_BATCH];
#pragma unroll
                for (int e = 0; e < MOVE_BATCH; ++e)
                    if (i + e < count) x[e] = *reinterpret_cast<const uint4 *>(base + place_of[path[i + e]]);
#pragma unroll
                for (int e = 0; e < MOVE_BATCH; ++e)
                    if (i + e < count) *reinterpret_cast<uint4 *>(base + place_of[i + e]) = x[e];
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
    const unsigned per_row = (a.q_heads + 2 * s.kv_heads + paged::APPEND_HEADS - 1) / paged::APPEND_HEADS *
                             (s.head_dim >> 4);
    const int64_t blocks = (static_cast<int64_t>(s.rows) * per_row + paged::APPEND_THREADS - 1) / paged::APPEND_THREADS;
    if (blocks > 0x7FFFFFFF) return cudaErrorInvalidConfiguration;
    const dim3 grid(static_cast<unsigned>(blocks)), block(paged::APPEND_THREADS);
    cudaError_t e = a.x_f32 ? launch_ex(paged::append_kernel<true>, grid, block, 0, stream, false, pdl, s, a, per_row,
                                        status_word(workspace))
                            : launch_ex(paged::append_kernel<false>, grid, block, 0, stream, false, pdl, s, a, per_row,
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
