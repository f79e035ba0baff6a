// Attention of a step's drafted nodes over a paged key/value cache.
//
// For a row (node i of sequence s) and query head h with KV head h / G:
//   o = sum_t p_t v_t / sum_t p_t,  p_t = exp(scale q.k_t - m)
// over the sequence's cached positions and the drafted ones that the row's
// mask names, in one pass over keys and values with a running maximum m and
// sums in f32.
//
// Work.  A unit is one KV head of one sequence and up to 256 of its n*G query
// rows, so every key and value is read once for all of them; its cache is cut
// into tiles of 128 positions.  The tiles of all units, in order, are divided
// evenly over a persistent grid of one CTA per SM: ragged lengths balance
// without the host knowing them (they live in device memory, so a captured
// graph follows them).  A tile counts one whatever its unit's rows, though one
// of 129 to 256 rows takes 2.2 times as long as the others, so steps that mix
// such units with smaller ones balance less well; and each CTA reads the
// lengths of all sequences first, 32 at a time.
// A CTA's range covers the end of one unit, whole units
// and the start of another; whole units are finished in place, pieces go to
// the workspace and the CTAs that share a unit merge it together at the end,
// each a share of its rows, in piece order (results do not depend on timing).
// A second piece costs a CTA about 2.5 us and a merge 4, as much as several
// tiles, so where there are no more units than CTAs the scheduler weighs equal
// shares against one piece for each CTA, and against whole units without any
// merge (5 trees of 4 to 16 tiles, 8 KV heads: 28 -> 20 us with pieces, 34
// whole; 16 sequences of 6 to 11 tiles: 28 -> 22 whole).
//
// Roles.  A scheduler warp reads the lengths and queues the CTA's pieces; a
// query warp copies their rows ahead of time; a producer warp brings K and V
// tiles page by page through a shared-memory ring (TMA, 128-byte swizzle); an
// MMA warp issues S = Q K^T (both from shared memory) and O += P V (P from
// tensor memory, V read along its dims); two warpgroups, a thread per row,
// turn S into P.  The two are two streams with their own S, O, maximum and
// sum: units of more than 128 rows give each its own 128 rows and both take
// every tile; smaller units give both the same rows and they take alternate
// tiles.  While one stream is in its softmax the tensor cores work for the
// other.  Units of at most 64 (32) rows fill the 128 rows of the MMA with 2
// (4) copies, and each copy's warps take half (a quarter) of a tile's
// positions: the softmax of few rows then runs on all warps.  The streams'
// and copies' results are joined when the piece ends.
//
// A row's maximum is only raised when a score passes it by more than 2^8, and
// then by a whole power of two: the sums, the tile's probabilities so far and
// O are rescaled without another rounding, and rarely.  What is subtracted is a
// whole number of log2 units, and the factor is that of the difference of the
// old and the new one as f32 holds them, so weights from before and after a
// raise have one base however far the scores are from zero (up to 2^30, where
// f32 steps by 128 and a probability may leave its range).  A run of 32 scores
// is read once, and little code does for all of it: short contexts wait for
// instructions as much as for data (a pass for the maximum before the one for
// the exponentials, with loads ahead, took 12.8 us instead of 11.7 for one
// token, 20.2 instead of 18.0 for 5 small trees, 114 instead of 113 for wide
// ones).  Hidden scores are cleared in tensor memory before the softmax of the
// few tiles that have any, which keeps the masks out of the common path.
//
// Rounding: P is rounded to bf16 for the tensor cores (as V is bf16, it is the
// smaller part of the result's own rounding); the sum l adds the rounded
// values, so a row's weights still sum to one.  Scores, maxima, sums and O are
// f32.
//
// Bounds.  Units of up to 128 rows are bound by HBM once a CTA has enough
// tiles: 64 rows on 4 x 128K positions (2.06 GB) take 314 us, 6.5 TB/s, 0.99 of
// the measured copy rate (375 us in a loop of seconds, where the power cap
// holds the SMs at 1.1 GHz).  Units of 129 to 256 rows are bound by the turns of
// their two streams, 2.9 us a tile: 2.0 for a row's softmax (1.1 is what the
// exponentials of both streams' warps take, 8 cycles each) and 0.9 from its P
// to its next scores, since P lies over S and both products come between; the
// products alone take 1.2 and the tile's bytes 1.4.  (8 x 8K positions under
// 60 drafts, 256 rows: 110 us.  Two warps a row, turns between the streams,
// items of half a tile and all scores in registers measured 114, 123, 126 and
// 119.)  Short contexts are bound by latency: 4 us to the first scores, 2.5 to
// store a piece, 4 to merge a unit (16 x 1000 positions, one node each: 19.2
// us; one sequence of 333: 11.2).
#include <cuda_runtime.h>

#include "common.cuh"
#include "internal.h"
#include "paged.cuh"
#include "sm100.cuh"

namespace afb {
namespace tattn {

constexpr int TILE = 128;           // positions per tile
constexpr int ROWS = 256;           // query rows of a unit, at most
constexpr int SOFTMAX_WARPS = 8;    // two warpgroups
constexpr int PRODUCER = 8, MMA = 9, SCHEDULER = 10, QUERIES = 11;
constexpr int THREADS = 32 * 12;
constexpr int SOFTMAX_THREADS = 32 * SOFTMAX_WARPS;
constexpr int HALF_BYTES = TILE * 128;  // 64 dims of a tile
constexpr int PIECES = 4;           // pieces queued ahead
// What the scheduler weighs, in measured 0.1 us: a tile of units of up to 128
// (256) rows, the end of a piece, the merge of a unit.
constexpr int TILE_COST = 13, TILE2_COST = 29, PIECE_COST = 25, MERGE_COST = 40;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float RAISE = 8.0f;       // log2: how far scores may pass the running maximum before it is raised

// Named barriers: all softmax threads; a warpgroup's.
constexpr int BAR_ALL = 1, BAR_GROUP = 2;

template <int HD>
struct Cfg {
    static constexpr int HALVES = HD / 64;
    static constexpr int TILE_BYTES = HALVES * HALF_BYTES;
    static constexpr int STAGES = 163840 / TILE_BYTES;  // 160 KB of ring
    static constexpr int SMEM = 1024 + 2 * TILE_BYTES + STAGES * TILE_BYTES + 1024;
    static constexpr int RECORD = ROWS * (HD + 2);      // f32 of one partial: O, then m, then l
};

struct Params {
    PagedShape s;
    PagedStep t;
    TreeAttnArgs a;
    int group;           // query heads per KV head
    float *partial;      // [grid][2] records
    unsigned *arrived, *done, *status;
    CombineWait merge;   // limit of a merge's wait for the other CTAs of a unit
};

// The tiles of one sequence: kv_heads * row tiles * position tiles.
struct SeqTiles {
    SeqSpan sp;
    int n, units, nt;
    __device__ __forceinline__ int64_t tiles(int kv_heads) const { return static_cast<int64_t>(kv_heads) * units * nt; }
};
__device__ __forceinline__ SeqTiles seq_tiles(const Params &p, int seq) {
    SeqTiles r;
    r.sp = seq_span(p.s, p.t, seq);
    r.n = r.sp.ok ? r.sp.last - r.sp.first : 0;
    r.units = (r.n * p.group + ROWS - 1) / ROWS;
    r.nt = r.n ? (r.sp.ctx + r.n + TILE - 1) / TILE : 0;
    return r;
}

// The division of all tiles over the grid: the first `extra` CTAs take
// per + 1, the others per.
struct Shares {
    int grid, per, extra;
    __device__ __forceinline__ int begin(int cta) const { return cta * per + min(cta, extra); }
    __device__ __forceinline__ int owner(int tile) const {
        const int big = extra * (per + 1);
        return tile < big ? tile / (per + 1) : extra + (tile - big) / per;
    }
};

// A piece of a unit: tiles [t0, t1) of nt.  rows 0 ends the queue.
struct Piece {
    int seq, first, n, ctx, kv, row0, rows, t0, t1, nt;
    int owner0, owners;  // the CTAs that share the unit
    __device__ __forceinline__ bool both() const { return rows > TILE; }  // two row tiles, every position tile for both
    // log2 of the copies of the rows in the 128 rows of the MMA.
    __device__ __forceinline__ int copies() const { return rows <= 32 ? 2 : rows <= 64 ? 1 : 0; }
};

// Which of the two query buffers a piece uses and how often each was used.
struct QuerySlots {
    unsigned uses0 = 0u, uses1 = 0u;
    int next = 0;
    __device__ __forceinline__ int take(bool both) {
        const int s = both ? 0 : next;
        next = both ? 0 : next ^ 1;
        uses0 += s == 0;
        uses1 += both || s == 1;
        return s;
    }
    __device__ __forceinline__ uint32_t parity(int slot) const {  // of its current use
        return ((slot ? uses1 : uses0) - 1) & 1;
    }
};

// 32 visibility bits of a row, for drafted nodes j0 .. j0+31 (cached
// positions are j < 0: always visible).
struct RowMask {
    const uint32_t *words;  // null: nodes up to `node`
    int n, node;
    __device__ __forceinline__ uint32_t word(int w) const {  // nodes 32w .. 32w+31
        if (w < 0) return 0xFFFFFFFFu;
        const int left = n - 32 * w;
        if (left <= 0) return 0u;
        const uint32_t keep = left >= 32 ? 0xFFFFFFFFu : (1u << left) - 1;
        if (words) return words[w] & keep;
        const int k = node + 1 - 32 * w;
        return k <= 0 ? 0u : k >= 32 ? 0xFFFFFFFFu : (1u << k) - 1;
    }
    __device__ __forceinline__ uint32_t bits(int j0) const {
        return __funnelshift_r(word(j0 >> 5), word((j0 >> 5) + 1), j0 & 31);
    }
};

// The bounded wait, its slow part once for the whole kernel: instructions are
// fetched from cold (all waits inlined took 1% more, short contexts or long).
// Once another wait of the CTA has given up, none is begun: the softmax warps
// still walk every tile of the pieces that were queued.
__device__ __noinline__ bool wait_slow(uint64_t *bar, uint32_t parity, volatile int *abort, unsigned *status) {
    if (mbar_try_wait(bar, parity)) return true;
    return !*abort && mbar_wait(bar, parity, abort, status);
}
__device__ __forceinline__ bool wait(uint64_t *bar, uint32_t parity, volatile int *abort, unsigned *status) {
    return mbar_try_wait(bar, parity) || wait_slow(bar, parity, abort, status);
}
// A whole warp's wait, with one answer: false when it gave up, or when another
// wait of the CTA had.
__device__ __forceinline__ bool warp_wait(uint64_t *bar, uint32_t parity, volatile int *abort, unsigned *status) {
    return __all_sync(0xffffffffu, wait(bar, parity, abort, status));
}

// A value that is the same in all lanes, known as such to the compiler.
__device__ __forceinline__ int uniform(int x) { return __shfl_sync(0xffffffffu, x, 0); }

// Copies 16 bytes to shared memory without registers.
__device__ __forceinline__ void copy16_async(void *dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}

// 8 results of a row, dims in order or in the 4-bit qmv's pair order.
__device__ __forceinline__ void store8_bf16(uint16_t *dst, const float (&o)[8], int pair_order) {
    *reinterpret_cast<uint4 *>(dst) =
        pair_order ? make_uint4(pack_bf16x2(o[0], o[4]), pack_bf16x2(o[1], o[5]), pack_bf16x2(o[2], o[6]),
                                pack_bf16x2(o[3], o[7]))
                   : make_uint4(pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3]), pack_bf16x2(o[4], o[5]),
                                pack_bf16x2(o[6], o[7]));
}
// Output of row rr of a unit.
template <int HD>
__device__ __forceinline__ uint16_t *out_row(const Params &p, const Piece &d, int rr) {
    const int x = d.row0 + rr, node = x / p.group, g = x - node * p.group;
    return p.a.out + (static_cast<int64_t>(d.first) + node) * p.a.ld_out +
           (static_cast<int64_t>(d.kv) * p.group + g) * HD;
}
template <int N>
__device__ __forceinline__ void tmem_ld_row(uint32_t taddr, uint32_t (&r)[N]) {
    if constexpr (N == 32) tmem_ld_32x32b_x32(taddr, r);
    else tmem_ld_32x32b_x16(taddr, r);
}

// Rows row0 .. row0+rows-1 of a unit into a query buffer (K-major, 128-byte
// swizzle), 1 << copies times.  Rows that the unit lacks stay as they are: the
// rows of the MMA do not mix.
template <int HD>
__device__ __forceinline__ void load_queries(const Params &p, const Piece &d, int row0, int rows, int copies, char *dst,
                                             int thread, int threads) {
    constexpr int CHUNKS = HD / 8;  // a thread keeps its 16 bytes of every step-th row
    const int c = thread % CHUNKS, step = threads / CHUNKS, dn = step / p.group, dg = step - dn * p.group;
    const int first = d.row0 + row0 + thread / CHUNKS;
    int node = first / p.group, g = first - node * p.group;
    const uint16_t *src = p.a.q + static_cast<int64_t>(d.first) * p.a.ld_q + static_cast<int64_t>(d.kv) * p.group * HD +
                          c * 8;
#pragma unroll 2
    for (int r = thread / CHUNKS; r < rows; r += step) {
        const uint16_t *from = src + node * p.a.ld_q + g * HD;
        char *to = dst + (c >> 3) * HALF_BYTES + r * 128 + (((c & 7) ^ (r & 7)) << 4);
        copy16_async(to, from);
        if (copies) copy16_async(to + TILE * 64, from);  // a copy's rows start at a multiple of 8
        if (copies > 1) copy16_async(to + TILE * 32, from), copy16_async(to + TILE * 96, from);
        g += dg, node += dn;
        if (g >= p.group) g -= p.group, ++node;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    fence_proxy_async_smem();
}

// Infinities and NaN among the drafted values, which were kept from the
// tensor cores, for a row that sees them: added to what the row's thread has
// just stored (dims dim0 .. dim1-1; rec: f32 partial, out: bf16 result).
__device__ __noinline__ void add_odd_values(const Params &p, const Piece &d, const RowMask &mask, const uint32_t *odd,
                                            int dim0, int dim1, float *rec, uint16_t *out) {
    for (int k = 0; k < kMaxTreeNodes / 32; ++k) {
        for (uint32_t set = odd[k] ? odd[k] & mask.word(k) : 0u; set; set &= set - 1) {
            const int pos = d.ctx + 32 * k + __ffs(set) - 1;
            const int page = p.t.page_table[d.seq * p.s.ld_table + (pos >> p.s.page_shift)];
            if (page < 0 || page >= p.s.pages) continue;
            const uint16_t *src = p.a.v_cache + page * p.s.page_stride + d.kv * p.s.head_stride +
                                  (pos & ((1 << p.s.page_shift) - 1)) * p.s.token_stride;
            for (int dim = dim0; dim < dim1; ++dim) {
                if ((src[dim] & 0x7F80u) != 0x7F80u) continue;
                const float v = bf16_bits_to_f32(src[dim]);
                if (rec) {
                    rec[dim] += v;
                } else {
                    const int e = dim & 7;
                    uint16_t *o = out + (p.a.out_pair_order ? (dim & ~7) + (e < 4 ? 2 * e : 2 * (e - 4) + 1) : dim);
                    *o = f32_to_bf16_bits(bf16_bits_to_f32(*o) + v);
                }
            }
        }
    }
}

// A probability of zero does not hide what is not finite.  Of a tile's drafted
// positions (rows `from` to valid-1) the infinities and NaN, which only some
// query rows see, become zeros and are noted; those rows get them back when
// the piece ends.  Rows behind the last position that the last 16-position
// step still takes (never loaded, or whatever a page held) become zeros.
template <int HD>
__device__ __forceinline__ void clean_values(char *v, int from, int valid, int node0, uint32_t *odd) {
    constexpr int CHUNKS = HD / 8;
    const int lane = threadIdx.x & 31;
    auto at = [&](int i) {
        return reinterpret_cast<uint4 *>(v + (i % CHUNKS >> 3) * HALF_BYTES + (i / CHUNKS) * 128 + (i & 7) * 16);
    };
    for (int i = valid * CHUNKS + lane; i < ((valid + 15) & ~15) * CHUNKS; i += 32) *at(i) = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll 1
    for (int i0 = from * CHUNKS + lane; i0 < valid * CHUNKS; i0 += 128) {
        uint4 u[4];
        uint32_t bad[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) u[e] = i0 + 32 * e < valid * CHUNKS ? *at(i0 + 32 * e) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
        for (int e = 0; e < 4; ++e) {  // an exponent of all ones carries into the sign's place
            auto carry = [](uint32_t x) { return (x & 0x7F807F80u) + 0x00800080u; };
            bad[e] = (carry(u[e].x) | carry(u[e].y) | carry(u[e].z) | carry(u[e].w)) & 0x80008000u;
        }
        if (!(bad[0] | bad[1] | bad[2] | bad[3])) continue;
#pragma unroll 1
        for (int e = 0; e < 4; ++e) {
            const int i = i0 + 32 * e;
            if (i >= valid * CHUNKS) break;
            uint32_t *x = reinterpret_cast<uint32_t *>(at(i));
            bool found = false;
            for (int k = 0; k < 4; ++k) {
                uint32_t y = x[k];
                if ((y & 0x7F80u) == 0x7F80u) y &= 0xFFFF0000u, found = true;
                if ((y & 0x7F800000u) == 0x7F800000u) y &= 0x0000FFFFu, found = true;
                x[k] = y;
            }
            const int j = node0 + i / CHUNKS;
            if (found) atomicOr(&odd[j >> 5], 1u << (j & 31));
        }
    }
    fence_proxy_async_smem();
    __syncwarp();
}

template <int HD>
__global__ void __launch_bounds__(THREADS, 1) tree_attention_kernel(const __grid_constant__ CUtensorMap kmap,
                                                                 const __grid_constant__ CUtensorMap vmap,
                                                                 const __grid_constant__ Params p) {
    using C = Cfg<HD>;
    extern __shared__ char smem_raw[];
    char *qbuf = reinterpret_cast<char *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    char *ring = qbuf + 2 * C::TILE_BYTES;
    uint64_t *full = reinterpret_cast<uint64_t *>(ring + C::STAGES * C::TILE_BYTES);
    uint64_t *empty = full + C::STAGES;
    uint64_t *s_full = empty + C::STAGES;  // [2] scores of a stream are in tensor memory
    uint64_t *p_full = s_full + 2;         // [2] probabilities of a stream are
    uint64_t *q_full = p_full + 2;         // [2] query buffers
    uint64_t *q_empty = q_full + 2;
    uint64_t *d_full = q_empty + 2;        // [PIECES] the queue
    uint64_t *d_empty = d_full + PIECES;
    uint64_t *unit_done = d_empty + PIECES;  // every MMA of the piece has ended
    uint64_t *o_free = unit_done + 1;        // its O has been read
    Piece *queue = reinterpret_cast<Piece *>(o_free + 1);
    Piece *shared_units = queue + PIECES;    // [2] pieces of shared units: the end of one, the start of another
    uint32_t *odd = reinterpret_cast<uint32_t *>(shared_units + 2);  // drafted nodes whose values are not all finite
    uint32_t *tmem_addr = odd + kMaxTreeNodes / 32;
    volatile int *abort = reinterpret_cast<volatile int *>(tmem_addr + 1);
    volatile uint32_t *closed = tmem_addr + 2;  // how many pieces were queued, known at the end

    const int tid = threadIdx.x, lane = tid & 31;
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);  // warp-uniform for the compiler, too
    if (tid == 0) {
        for (int i = 0; i < C::STAGES; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], SOFTMAX_WARPS / 2);
            mbar_init(&q_full[i], 1);
            mbar_init(&q_empty[i], SOFTMAX_WARPS);
        }
        for (int i = 0; i < PIECES; ++i) {
            mbar_init(&d_full[i], 1);
            mbar_init(&d_empty[i], SOFTMAX_WARPS + 3);
        }
        mbar_init(unit_done, 2);
        mbar_init(o_free, SOFTMAX_WARPS);
        *abort = 0;
        *closed = 0xFFFFFFFFu;
        fence_mbar_init();
    }
    if (warp == MMA) {
        tmem_alloc(tmem_addr, 512);
        tmem_relinquish();
    }
    if (warp == PRODUCER && lane == 0) {
        tma_prefetch_desc(&kmap);
        tma_prefetch_desc(&vmap);
    }
    pdl_launch_dependents();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_wait();  // lengths, queries and the cache come from the preceding kernels
    const uint32_t tmem = static_cast<uint32_t>(uniform(static_cast<int>(*tmem_addr)));

    // The next piece of the queue (all threads of a warp); rows 0 at its end
    // or after an abort.  The softmax warps meet at barriers, so all of them
    // take every piece that was queued, abort or not: they leave only once the
    // scheduler, whose own waits are bounded, has closed the queue.
    uint32_t taken = 0;
    auto next_piece = [&](Piece &d) {
        const uint32_t i = taken++;
        bool ok;
        if (warp < SOFTMAX_WARPS) {
            while (!(ok = mbar_try_wait(&d_full[i % PIECES], (i / PIECES) & 1)) && i < *closed) {}
            ok = __all_sync(0xffffffffu, ok);
        } else {
            ok = warp_wait(&d_full[i % PIECES], (i / PIECES) & 1, abort, p.status);
        }
        d = queue[i % PIECES];
        d.rows = uniform(ok ? d.rows : 0);
        __syncwarp();
        if (lane == 0) mbar_arrive(&d_empty[i % PIECES]);
        return d.rows > 0;
    };

    if (warp == SCHEDULER) {  // ------------------------------------------------- the CTA's pieces
        unsigned total = 0, mine = 0, high = 0;  // high: the total / 1024, should it not fit
        SeqTiles q{};
        for (int base = 0; base < p.s.seqs; base += 32) {
            mine = 0;
            unsigned part = 0;
            if (base + lane < p.s.seqs) {
                q = seq_tiles(p, base + lane);
                const int64_t tiles = q.tiles(p.s.kv_heads);
                mine = static_cast<unsigned>(tiles);
                part = static_cast<unsigned>(min(tiles >> 10, int64_t(1) << 26));
                if (!q.sp.ok && blockIdx.x == 0) atomicExch(p.status, static_cast<unsigned>(DEV_BOUNDS));
            }
            total += __reduce_add_sync(0xffffffffu, mine);
            high = min(high + __reduce_add_sync(0xffffffffu, part), 1u << 30);
        }
        if (high >= 1u << 20) {  // 2^30 tiles: more cache than there can be
            if (blockIdx.x == 0 && lane == 0) atomicExch(p.status, static_cast<unsigned>(DEV_BOUNDS));
            total = 0;
        }
        Shares sh;
        sh.grid = min(static_cast<int>(total), static_cast<int>(gridDim.x));
        sh.per = sh.grid ? static_cast<int>(total) / sh.grid : 0;
        sh.extra = static_cast<int>(total) - sh.per * sh.grid;
        // With few units a piece each for every CTA may be better than equal
        // numbers of tiles.  Weighed for up to 32 sequences, a lane each.
        int pieces = 0;  // of the lane's sequence's units, 0: equal shares
        if (p.s.seqs <= 32 && total) {
            const int units = q.nt ? p.s.kv_heads * q.units : 0;
            const int longest = __reduce_max_sync(0xffffffffu, q.nt);
            if (__reduce_add_sync(0xffffffffu, units) <= gridDim.x) {
                const int cost = __any_sync(0xffffffffu, q.n * p.group > TILE) ? TILE2_COST : TILE_COST;
                const int even = sh.per + (sh.extra > 0);
                int best = even * cost + PIECE_COST + MERGE_COST;
#pragma unroll 1
                for (int c = even; c < longest && c * cost + MERGE_COST < best; ++c) {
                    const int n = q.nt ? (q.nt + c - 1) / c : 0;
                    if (__reduce_add_sync(0xffffffffu, units * n) <= gridDim.x) {
                        best = c * cost + MERGE_COST;
                        pieces = n;
                    }
                }
                if (longest * cost < best) pieces = q.nt ? 1 : 0;
            }
        }
        const bool single = __any_sync(0xffffffffu, pieces > 0);
        int pos = 0, end = 0, seq = 0, at = 0, owners = 0;
        if (single) {
            mine = pieces * p.s.kv_heads * q.units;
            int upto = static_cast<int>(mine);
#pragma unroll 1
            for (int o = 1; o < p.s.seqs; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += v;
            }
            const unsigned past = __ballot_sync(0xffffffffu, upto > static_cast<int>(blockIdx.x));
            if (past) {
                seq = __ffs(past) - 1;
                at = blockIdx.x - __shfl_sync(0xffffffffu, upto - static_cast<int>(mine), seq);
                owners = __shfl_sync(0xffffffffu, pieces, seq);
                end = 1;
            }
            q.sp.first = __shfl_sync(0xffffffffu, q.sp.first, seq);
            q.sp.ctx = __shfl_sync(0xffffffffu, q.sp.ctx, seq);
            q.n = __shfl_sync(0xffffffffu, q.n, seq);
            q.units = __shfl_sync(0xffffffffu, q.units, seq);
            q.nt = __shfl_sync(0xffffffffu, q.nt, seq);
        } else if (static_cast<int>(blockIdx.x) < sh.grid) {
            pos = sh.begin(blockIdx.x);
            end = sh.begin(blockIdx.x + 1);
            int before = 0;
            for (int base = 0; base < p.s.seqs; base += 32) {  // the sequence that holds tile `pos`
                if (p.s.seqs > 32)
                    mine = base + lane < p.s.seqs
                               ? static_cast<unsigned>(seq_tiles(p, base + lane).tiles(p.s.kv_heads))
                               : 0u;
                int upto = static_cast<int>(mine);
#pragma unroll 1
                for (int o = 1; o < 32; o <<= 1) {
                    const int v = __shfl_up_sync(0xffffffffu, upto, o);
                    if (lane >= o) upto += v;
                }
                const unsigned past = __ballot_sync(0xffffffffu, before + upto > pos);
                if (past) {
                    const int l = __ffs(past) - 1;
                    seq = base + l;
                    at = pos - before - __shfl_sync(0xffffffffu, upto - static_cast<int>(mine), l);
                    break;
                }
                before += __shfl_sync(0xffffffffu, upto, 31);
            }
        }
        uint32_t queued = 0;
        auto over = [](int a, int b) {  // a / b; few divisions have a divisor
            return b == 1 ? a : static_cast<int>(static_cast<unsigned>(a) / static_cast<unsigned>(b));
        };
        int tiles = 0;
        if (pos < end && !single) q = seq_tiles(p, seq), tiles = static_cast<int>(q.tiles(p.s.kv_heads));
        for (uint32_t i = 0;; ++i) {
            Piece d{};
            if (pos < end && !single) {
                while (at >= tiles) {
                    at = 0;
                    if (++seq >= p.s.seqs) break;  // lengths that changed under the kernel
                    q = seq_tiles(p, seq);
                    tiles = static_cast<int>(q.tiles(p.s.kv_heads));
                }
                if (seq >= p.s.seqs) pos = end;
            }
            if (pos < end) {
                const int unit = over(at, single ? owners : q.nt);
                d.seq = seq;
                d.first = q.sp.first;
                d.n = q.n;
                d.ctx = q.sp.ctx;
                d.nt = q.nt;
                if (single) {
                    const int j = at - unit * owners;
                    d.t0 = over(q.nt * j, owners);
                    d.t1 = over(q.nt * (j + 1), owners);
                    d.owner0 = blockIdx.x - j;
                    d.owners = owners;
                } else {
                    d.t0 = at - unit * q.nt;
                    d.t1 = min(q.nt, d.t0 + end - pos);
                    d.owner0 = sh.owner(pos - d.t0);
                    d.owners = sh.owner(pos - d.t0 + q.nt - 1) - d.owner0 + 1;
                }
                d.kv = over(unit, q.units);
                d.row0 = (unit - d.kv * q.units) * ROWS;
                d.rows = min(ROWS, q.n * p.group - d.row0);
                at += d.t1 - d.t0;
                pos = single ? end : pos + d.t1 - d.t0;
            }
            if (!warp_wait(&d_empty[i % PIECES], ((i / PIECES) & 1) ^ 1, abort, p.status)) break;
            if (lane == 0) {
                queue[i % PIECES] = d;
                mbar_arrive(&d_full[i % PIECES]);
            }
            __syncwarp();
            queued = i + 1;
            if (d.rows == 0) break;
        }
        if (lane == 0) *closed = queued;
    } else if (warp == QUERIES) {  // ---------------------------------------------- query rows
        QuerySlots slots;
        Piece d;
        while (next_piece(d)) {
            const bool both = d.both();
            const int s = slots.take(both);
            // Waits for every use in turn: a parity tells only neighbouring uses apart.
            if (!warp_wait(&q_empty[s], slots.parity(s) ^ 1, abort, p.status)) break;
            if (both && !warp_wait(&q_empty[1], slots.parity(1) ^ 1, abort, p.status)) break;
            if (!both) {  // two row tiles are loaded by the softmax warps, who are free then
                load_queries<HD>(p, d, 0, d.rows, d.copies(), qbuf + s * C::TILE_BYTES, lane, 32);
                __syncwarp();
                if (lane == 0) mbar_arrive(&q_full[s]);
            }
        }
    } else if (warp == PRODUCER) {  // --------------------------------------------- K and V tiles
        const int shift = p.s.page_shift, box_shift = min(shift, 7), rows_per_box = 1 << box_shift;
        const uint64_t once = l2_evict_first(), again = l2_evict_normal();
        const uint32_t ring_addr = smem_u32(ring);
        int next = 0;  // the ring's next stage, over all pieces
        uint32_t next_phase = 0, sent = 0, phases = 0;
        Piece d;
        while (next_piece(d)) {
            const int *table = p.t.page_table + d.seq * p.s.ld_table;
            // Several row tiles read the same cache: keep it in L2 for them.
            const uint64_t policy = d.n * p.group > ROWS ? again : once;
            const int t0 = uniform(d.t0), t1 = uniform(d.t1), len = uniform(d.ctx + d.n), kv = uniform(d.kv);
            // The sequence's page table, 64 entries at a time, a lane two of
            // them; the second half is fetched while the first is used.
            const int last_page = (len - 1) >> shift;
            int page0 = (t0 * TILE) >> shift;
            auto fetch = [&](int i) {
                int page = table[min(i + lane, last_page)];
                if (page < 0 || page >= p.s.pages) {  // a coordinate outside the map reads zeros
                    if (i + lane <= last_page) atomicExch(p.status, static_cast<unsigned>(DEV_BOUNDS));
                    page = static_cast<int>(p.s.pages);
                }
                return page;
            };
            int ids = fetch(page0), more = fetch(page0 + 32);
            auto load = [&](const CUtensorMap *map, int t) {
                const int pos = t * TILE, boxes = (min(TILE, len - pos) + rows_per_box - 1) >> box_shift;
                const int stage = next;
                if (!warp_wait(&empty[stage], next_phase ^ 1, abort, p.status) || __any_sync(0xffffffffu, *abort))
                    return;  // never re-arm a stage after an abort
                if (lane == 0) mbar_arrive_expect_tx(&full[stage], boxes * C::HALVES * rows_per_box * 128);
                __syncwarp();
                const uint32_t dst = ring_addr + stage * C::TILE_BYTES;
                const int first = (pos >> shift) - page0, row = pos & ((1 << shift) - 1);
#pragma unroll 4
                for (int b = 0; b < boxes; ++b) {
                    const int i = first + b;
                    const int page = __shfl_sync(0xffffffffu, i < 32 ? ids : more, i & 31);
                    tma_load_4d_elect<C::HALVES>(dst + b * rows_per_box * 128, HALF_BYTES, map, &full[stage], row, kv, page,
                                                 policy);
                }
                sent |= 1u << stage;
                phases = (phases & ~(1u << stage)) | next_phase << stage;
                if (++next == C::STAGES) next = 0, next_phase ^= 1;
            };
            // The order in which the MMA warp consumes them: with two row
            // tiles K0 V0 K1 V1 .., else K0 K1 V0 K2 V1 .. (a tile's values
            // follow the next tile's keys).
            const int lag = uniform(d.both() ? 0 : 1);
#pragma unroll 1
            for (int t = t0; t < t1 + lag && !*abort; ++t) {
                if (((t - lag) * TILE >> shift) - page0 >= 32 && t > t0) {  // the first half is used up
                    page0 += 32;
                    ids = more;
                    more = fetch(page0 + 32);
                }
                if (t < t1) load(&kmap, t);
                if (t - lag >= t0) load(&vmap, t - lag);
            }
        }
        // Copies in flight land before the CTA leaves.
        for (int i = 0; i < C::STAGES; ++i)
            if (sent >> i & 1) mbar_wait_drain(&full[i], phases >> i & 1);
    } else if (warp == MMA) {  // ---------------------------------------------------- tensor cores
        // A negative scale negates the queries, so the running maximum can
        // work on the scores as they come.
        const uint32_t idesc_s = umma_idesc_bf16(128, TILE) | (p.a.scale < 0.0f ? kUmmaNegateA : 0u);
        const uint32_t idesc_o = umma_idesc_bf16(128, HD) | kUmmaTransposeB;
        const uint32_t q_lo = umma_lo(smem_u32(qbuf), 16), k_lo = umma_lo(smem_u32(ring), 16);
        const uint32_t v_lo = umma_lo(smem_u32(ring), HALF_BYTES);
        constexpr uint32_t TILE_LO = C::TILE_BYTES >> 4;
        int next = 0;  // the ring's next stage: tiles are used in the order in which they are loaded
        uint32_t next_phase = 0, p_phase = 0, pieces = 0;
        bool live = true;
        QuerySlots slots;
        Piece d;
        while (live && next_piece(d)) {
            const int nt = uniform(d.t1 - d.t0), both = uniform(d.both());
            const int tile0 = uniform(d.t0), ctx = uniform(d.ctx), len = uniform(d.ctx + d.n);
            const int slot = uniform(slots.take(both));
            live = warp_wait(&q_full[slot], slots.parity(slot), abort, p.status);
            if (live && both) live = warp_wait(&q_full[1], slots.parity(1), abort, p.status);
            if (!live) break;
            auto take = [&]() {  // waits for the next stage to land
                const int stage = next;
                live = live && warp_wait(&full[stage], next_phase, abort, p.status);
                if (++next == C::STAGES) next = 0, next_phase ^= 1;
                return stage;
            };
            auto p_ready = [&](int st) {
                live = live && warp_wait(&p_full[st], (p_phase >> st) & 1, abort, p.status);
                p_phase ^= 1u << st;
                tc_fence_after();
            };
            auto scores = [&](int st, int q, int k) {
                umma_run_ss<HD / 16>(tmem + st * TILE, q_lo + q * TILE_LO, k_lo + k * TILE_LO, idesc_s, &s_full[st]);
            };
            // O += P V over the 16-position steps that hold any position of the sequence.
            auto values = [&](int st, int v, int steps, bool accumulate) {
                const uint32_t o = tmem + 2 * TILE + st * HD, pr = tmem + st * TILE, lo = v_lo + v * TILE_LO;
                if (steps == 8) {
                    umma_run_ts4(o, pr, lo, idesc_o, accumulate);
                    umma_run_ts4(o, pr + 32, lo + 512, idesc_o, 1u);
                } else {
#pragma unroll 1
                    for (int ks = 0; ks < steps; ++ks)
                        umma_step_ts(o, pr + 8 * ks, lo + 128 * ks, idesc_o, accumulate || ks > 0);
                }
            };
            // A tile's values have landed; returns their steps.
            auto enter = [&](int t, int stage) {
                const int pos = (tile0 + t) * TILE, valid = min(TILE, len - pos);
                if (live && pos + TILE > ctx)
                    clean_values<HD>(ring + stage * C::TILE_BYTES, max(0, ctx - pos), valid, pos - ctx, odd);
                return (valid + 15) >> 4;
            };
#pragma unroll 1
            for (int t = 0; t < (both ? 1 : 2) && t < nt; ++t) {
                const int k = take();
                if (!live) break;
                scores(t, both ? 0 : slot, k);
                if (both) scores(1, 1, k);
                umma_commit_elect(&empty[k]);
            }
            if (pieces && live) live = warp_wait(o_free, (pieces - 1) & 1, abort, p.status);
            if (!live) break;
            if (lane < kMaxTreeNodes / 32) odd[lane] = 0u;  // the last piece's have been read
            __syncwarp();
#pragma unroll 1
            for (int t = 0; t < nt && live; ++t) {
                const int v = take();
                const int steps = enter(t, v);
                if (both) {
                    const bool more = t + 1 < nt;
                    p_ready(0);
                    if (!live) break;
                    values(0, v, steps, t > 0);
                    const int k = more ? take() : 0;
                    if (!live) break;
                    if (more) scores(0, 0, k);
                    p_ready(1);
                    if (!live) break;
                    values(1, v, steps, t > 0);
                    umma_commit_elect(&empty[v]);
                    if (more) {
                        scores(1, 1, k);
                        umma_commit_elect(&empty[k]);
                    }
                } else {
                    const int st = t & 1;
                    p_ready(st);
                    if (!live) break;
                    values(st, v, steps, t >= 2);
                    umma_commit_elect(&empty[v]);
                    if (t + 2 < nt) {
                        const int k = take();
                        if (!live) break;
                        scores(st, slot, k);
                        umma_commit_elect(&empty[k]);
                    }
                }
            }
            if (!live) break;
            __syncwarp();
            if (lane == 0) mbar_arrive(unit_done);  // `odd` is written
            umma_commit_elect(unit_done);
            ++pieces;
        }
        // On the way out of an abort, MMAs in flight end before tensor memory is freed.
        if (!live) {
            umma_commit_elect(&s_full[0]);
            for (int i = 0; i < 2; ++i) mbar_wait_drain(&s_full[0], i, 1000000ull);
        }
    } else {  // ------------------------------------------------------------------------ softmax
        const int st = warp >> 2, r = tid & 127;
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t ts = tmem + lanes + st * TILE, to = tmem + lanes + 2 * TILE;
        const float sc = fabsf(p.a.scale) * LOG2E;
        uint32_t s_phase = 0, u_phase = 0;
        bool shares_end = false, shares_start = false;  // units that other CTAs have a part of
        QuerySlots slots;
        Piece d;
        while (next_piece(d)) {
            const bool both = d.both();
            const int slot = slots.take(both), copies = d.copies();
            const int copy = r >> (7 - copies);             // which copy of the rows this thread holds
            const int rr = both ? st * TILE + r : r & ((TILE >> copies) - 1);  // its row of the unit
            const bool mine = rr < d.rows;
            const bool warp_on = __any_sync(0xffffffffu, mine);
            const int x = d.row0 + rr, node = mine ? x / p.group : 0;
            const int64_t row = static_cast<int64_t>(d.first) + node;
            const RowMask mask{p.a.mask ? p.a.mask + row * p.s.mask_words : nullptr, d.n, node};
            if (both) {
                wait(&q_empty[st], slots.parity(st) ^ 1, abort, p.status);
                load_queries<HD>(p, d, st * TILE, min(TILE, d.rows - st * TILE), 0, qbuf + st * C::TILE_BYTES, r, 128);
                named_bar_sync(BAR_GROUP + st, 128);
                if (r == 0) mbar_arrive(&q_full[st]);
            }
            float off = -INFINITY, l = 0.0f;  // the maximum that is weighed against, in log2 units, and the sum
            const int nt = d.t1 - d.t0, stride = both ? 1 : 2;
            const int k0 = copy << (2 - copies), k1 = (copy + 1) << (2 - copies);  // this copy's runs of 32 positions
#pragma unroll 1
            for (int t = both ? 0 : st; t < nt; t += stride) {
                wait(&s_full[st], s_phase, abort, p.status);
                s_phase ^= 1;
                tc_fence_after();
                uint32_t v[32];  // a run of 32 positions
                if (warp_on) {
                    const int pos = (d.t0 + t) * TILE;
                    if (pos + 32 * k1 > d.ctx) {  // drafted positions, or the end: hidden scores become -inf
#pragma unroll 1
                        for (int k = 2 * k0; k < 2 * k1; ++k) {
                            uint32_t x[16];
                            tmem_ld_32x32b_x16(ts + 16 * k, x);
                            const uint32_t see = mask.bits(pos + 16 * k - d.ctx);
                            tmem_wait_ld(x);
#pragma unroll
                            for (int e = 0; e < 16; ++e)
                                if (!((see >> e) & 1u)) x[e] = 0xFF800000u;
                            tmem_st_32x32b_x16(ts + 16 * k, x);
                        }
                        tmem_wait_st();
                    }
                    float sum[2] = {0.0f, 0.0f};  // of the tile: a long sum of sums loses less
                    // Raises the maximum if a score of this run asks for it.
                    auto look = [&](const uint32_t (&x)[32], int run) {
                        float a[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) a[e] = __uint_as_float(x[e]);
#pragma unroll
                        for (int e = 4; e < 32; ++e) a[e & 3] = fmaxf(a[e & 3], __uint_as_float(x[e]));
                        const float top = fmaxf(fmaxf(a[0], a[1]), fmaxf(a[2], a[3]));
                        const float over = fmaf(top, sc, -off);  // infinite at first, NaN while nothing is visible
                        const bool raise = mine && over > RAISE;
                        if (!__any_sync(0xffffffffu, raise)) return;
                        float corr = 1.0f;  // a power of two: nothing is rounded again
                        if (raise) {
                            if (off == -INFINITY) {
                                off = ceilf(top * sc);
                            } else {
                                const float up = off + ceilf(over), by = up - off;
                                off = up;
                                corr = by > 126.0f ? 0.0f : __int_as_float((127 - static_cast<int>(by)) << 23);
                            }
                        }
                        l *= corr, sum[0] *= corr, sum[1] *= corr;
                        tmem_wait_st();
#pragma unroll 1
                        for (int k = k0; k < run; ++k) {  // this tile's probabilities so far
                            uint32_t u[16];
                            tmem_ld_32x32b_x16(ts + 16 * k, u);
                            tmem_wait_ld(u);
#pragma unroll
                            for (int e = 0; e < 16; ++e)
                                u[e] = pack_bf16x2(__uint_as_float(u[e] << 16) * corr,
                                                   __uint_as_float(u[e] & 0xFFFF0000u) * corr);
                            tmem_st_32x32b_x16(ts + 16 * k, u);
                        }
                        if (t >= stride) {  // O holds something: the scores came after the last product
#pragma unroll 1
                            for (int c = 0; c < HD; c += 16) {
                                uint32_t o[16];
                                tmem_ld_32x32b_x16(to + st * HD + c, o);
                                tmem_wait_ld(o);
#pragma unroll
                                for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * corr);
                                tmem_st_32x32b_x16(to + st * HD + c, o);
                            }
                        }
                    };
                    auto weigh = [&](const uint32_t (&x)[32], int run) {
                        const float base = off == -INFINITY ? 0.0f : off;
                        uint32_t u[16];
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const float a = exp2_approx(fmaf(__uint_as_float(x[2 * e]), sc, -base));
                            const float b = exp2_approx(fmaf(__uint_as_float(x[2 * e + 1]), sc, -base));
                            u[e] = pack_bf16x2(a, b);
                            add_bf16x2(sum[0], sum[1], u[e]);
                        }
                        tmem_st_32x32b_x16(ts + 16 * run, u);  // over scores that have been read
                    };
#pragma unroll 1
                    for (int k = k0; k < k1; ++k) {
                        tmem_ld_32x32b_x32(ts + 32 * k, v);
                        tmem_wait_ld();
                        tie_regs(v);
                        look(v, k);
                        weigh(v, k);
                    }
                    if (copies) {  // the other copies' positions
                        const uint32_t zero[16] = {};
#pragma unroll 1
                        for (int k = 0; k < 4; ++k)
                            if (k < k0 || k >= k1) tmem_st_32x32b_x16(ts + 16 * k, zero);
                    }
                    l += sum[0] + sum[1];
                    tmem_wait_st();
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[st]);
            }
            // The rows that this thread stores: every STEP-th, from its own first.
            constexpr int W = HD / 4, CH = W / 8, STEP = 128 / CH;
            const int x1 = d.row0 + (both ? st * TILE : 0) + r / CH;
            const int node1 = x1 / p.group, g1 = x1 - node1 * p.group;
            const int dn = STEP / p.group, dg = STEP - dn * p.group;
            wait(unit_done, u_phase, abort, p.status);
            u_phase ^= 1;
            tc_fence_after();

            // The piece's result.  A row whose sum is NaN keeps a finite
            // maximum, so that no join takes it for one that saw nothing.
            const float m2 = l != l ? 0.0f : off;
            float top = m2, lsum = l, w0 = m2 == -INFINITY ? 0.0f : 1.0f, w1 = 0.0f;
            char *scratch = qbuf + slot * C::TILE_BYTES;  // the queries are done with
            if (!both) {  // join the streams' and copies' maxima and sums
                float2 *ex = reinterpret_cast<float2 *>(scratch);
                ex[st * TILE + r] = make_float2(m2, l);
                named_bar_sync(BAR_ALL, SOFTMAX_THREADS);
                const int states = 2 << copies, step = TILE >> copies;  // state i: stream i & 1, copy i >> 1
                float2 e[8];
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    e[i] = i < states ? ex[(i & 1) * TILE + (i >> 1) * step + rr] : make_float2(-INFINITY, 0.0f);
                top = -INFINITY;
                lsum = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; ++i) top = fmaxf(top, e[i].x);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float wt = e[i].x == -INFINITY ? 0.0f : exp2_approx(e[i].x - top);
                    lsum += e[i].y * wt;
                    if (i >> 1 == copy) (i & 1 ? w1 : w0) = wt;
                }
                named_bar_sync(BAR_ALL, SOFTMAX_THREADS);
            }
            const bool whole = d.t0 == 0 && d.t1 == d.nt;
            if (whole) {
                const float inv = lsum == 0.0f ? 0.0f : 1.0f / lsum;
                w0 *= inv, w1 *= inv;
            }
            // O in rounds of HD/4 dims: a thread leaves its row's in shared
            // memory, then the warpgroup adds the copies up and stores whole
            // sectors.  Each warpgroup takes all dims of its own rows, or
            // half the dims of both streams' rows.
            const int dim0 = both ? 0 : st * (HD / 2), dim1 = both ? HD : dim0 + HD / 2;
            const int rows = both ? min(TILE, d.rows - st * TILE) : d.rows;
            const bool pair = !both && nt > 1;  // the second stream's O holds something
            char *stage = both ? qbuf + st * C::TILE_BYTES : scratch + st * (C::TILE_BYTES / 2);
            auto cell = [&](int row, int c) {  // 16 bytes, spread over the banks
                return reinterpret_cast<float4 *>(stage + row * (W * 4) + ((c ^ (row >> (HD == 64) & (W / 4 - 1))) << 4));
            };
            float *rec = p.partial + (2 * static_cast<int64_t>(blockIdx.x) + (d.t0 == 0 ? 1 : 0)) * C::RECORD;
            const int lead = both ? st * TILE : 0;
#pragma unroll 1
            for (int c = dim0; c < dim1; c += W) {
                if (warp_on) {
                    uint32_t a[W], b[W];
                    tmem_ld_row<W>(to + (both ? st * HD : 0) + c, a);
                    if (pair) tmem_ld_row<W>(to + HD + c, b);
                    tmem_wait_ld();
                    tie_regs(a);
                    tie_regs(b);
#pragma unroll
                    for (int e = 0; e < W; e += 4) {
                        float o[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            o[i] = __uint_as_float(a[e + i]) * w0;
                            if (pair) o[i] = fmaf(__uint_as_float(b[e + i]), w1, o[i]);
                        }
                        if (mine) *cell(r, e / 4) = make_float4(o[0], o[1], o[2], o[3]);
                    }
                }
                named_bar_sync(BAR_GROUP + st, 128);
#pragma unroll 1
                for (int row = r / CH, node = node1, g = g1; row < rows; row += STEP) {
                    const int k = r % CH;  // 8 dims of a row
                    float o[8] = {};
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        if (q >> copies) break;
                        const float4 y0 = *cell(row + q * (TILE >> copies), 2 * k);
                        const float4 y1 = *cell(row + q * (TILE >> copies), 2 * k + 1);
                        o[0] += y0.x, o[1] += y0.y, o[2] += y0.z, o[3] += y0.w;
                        o[4] += y1.x, o[5] += y1.y, o[6] += y1.z, o[7] += y1.w;
                    }
                    if (whole) {
                        uint16_t *dst = p.a.out + (static_cast<int64_t>(d.first) + node) * p.a.ld_out +
                                        (static_cast<int64_t>(d.kv) * p.group + g) * HD;
                        store8_bf16(dst + c + 8 * k, o, p.a.out_pair_order);
                        g += dg, node += dn;
                        if (g >= p.group) g -= p.group, ++node;
                    } else {
                        float4 *dst = reinterpret_cast<float4 *>(rec + (lead + row) * HD + c + 8 * k);
                        dst[0] = make_float4(o[0], o[1], o[2], o[3]);
                        dst[1] = make_float4(o[4], o[5], o[6], o[7]);
                    }
                }
                named_bar_sync(BAR_GROUP + st, 128);
            }
            if (__any_sync(0xffffffffu, odd[lane & 7] != 0u) && mine && copy == 0) {
                // Copies, so that what the call takes by address stays in registers elsewhere.
                const Piece piece = d;
                const RowMask seen = mask;
                add_odd_values(p, piece, seen, odd, dim0, dim1, whole ? nullptr : rec + rr * HD, out_row<HD>(p, d, rr));
            }
            if (!whole && mine && copy == 0 && dim0 == 0) {
                rec[ROWS * HD + rr] = top;
                rec[ROWS * HD + ROWS + rr] = lsum;
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(o_free);
                mbar_arrive(&q_empty[slot]);
                if (both) mbar_arrive(&q_empty[1]);
            }
            if (!whole) {
                (d.t0 == 0 ? shares_start : shares_end) = true;
                if (tid == 0) shared_units[d.t0 == 0] = d;
                named_bar_sync(BAR_ALL, SOFTMAX_THREADS);
                if (tid == 0) {  // the barrier's order and this fence publish all threads' stores
                    asm volatile("fence.acq_rel.gpu;" ::: "memory");
                    atomicAdd(&p.arrived[d.owner0], 1u);
                }
            }
        }
        // Merge the shared units: this CTA's share of their rows.  A thread
        // takes 8 dims of a row and a part of the unit's pieces.
#pragma unroll 1
        for (int which = 0; which < 2; ++which) {
            if (!(which ? shares_start : shares_end)) continue;
            const Piece u = shared_units[which];
            const int owner0 = u.owner0, k = u.owners;
            const int me = blockIdx.x - owner0;
            const int r0 = u.rows * me / k, rows = u.rows * (me + 1) / k - r0;
            bool ok = true;
            if (rows > 0) {
                if (lane == 0) {
                    const uint64_t since = globaltimer();
                    const unsigned want = static_cast<unsigned>(k) + p.merge.extra_arrivals;
                    while (ok && *reinterpret_cast<volatile unsigned *>(&p.arrived[owner0]) != want)
                        if (*abort || globaltimer() - since > p.merge.limit_ns) {
                            atomicExch(p.status, static_cast<unsigned>(DEV_TIMEOUT));
                            ok = false;
                        }
                    asm volatile("fence.acq_rel.gpu;" ::: "memory");
                }
                ok = __all_sync(0xffffffffu, ok);
            }
            // Every warp of the unit's CTAs counts itself once it has seen all
            // arrivals; the last clears the counters for the next launch.
            unsigned seen = 0;
            if (lane == 0) seen = atomicAdd(&p.done[owner0], 1u);
            constexpr int CHUNKS = HD / 8;
            int parts = 1;  // as many threads for a row's 8 dims as there are, each with at least two pieces
            while (2 * parts * rows * CHUNKS <= SOFTMAX_THREADS && 4 * parts <= k) parts *= 2;
            const int c = tid % CHUNKS, part = tid / CHUNKS % parts, step = SOFTMAX_THREADS / CHUNKS / parts;
            float *ex = reinterpret_cast<float *>(ring);  // no copies are in flight any more
#pragma unroll 1
            for (int base = 0; base < rows; base += step) {
                const int row = base + tid / CHUNKS / parts, rr = r0 + row;
                const bool on = ok && row < rows;
                float top = -INFINITY, lsum = 0.0f, o[8] = {};
                if (on) {
                    const int j1 = k * (part + 1) / parts;
#pragma unroll 1
                    for (int j0 = k * part / parts; j0 < j1; j0 += 4) {
                        float mj[4], lj[4];
                        float4 q[4][2];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {  // every load of four pieces first
                            const int j = min(j0 + i, j1 - 1);
                            const float *rec = p.partial + (2 * static_cast<int64_t>(owner0 + j) + (j == 0)) * C::RECORD;
                            mj[i] = j0 + i < j1 ? __ldcg(rec + ROWS * HD + rr) : -INFINITY;
                            lj[i] = __ldcg(rec + ROWS * HD + ROWS + rr);
                            const float4 *src = reinterpret_cast<const float4 *>(rec + rr * HD) + 2 * c;
                            q[i][0] = __ldcg(src);
                            q[i][1] = __ldcg(src + 1);
                        }
                        const float t = fmaxf(fmaxf(fmaxf(mj[0], mj[1]), fmaxf(mj[2], mj[3])), top);
                        const float keep = top == -INFINITY ? 0.0f : exp2_approx(top - t);
                        top = t;
                        lsum *= keep;
#pragma unroll
                        for (int e = 0; e < 8; ++e) o[e] *= keep;
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (mj[i] != -INFINITY) {
                                const float wt = exp2_approx(mj[i] - t);
                                lsum = fmaf(lj[i], wt, lsum);
                                o[0] = fmaf(q[i][0].x, wt, o[0]), o[1] = fmaf(q[i][0].y, wt, o[1]);
                                o[2] = fmaf(q[i][0].z, wt, o[2]), o[3] = fmaf(q[i][0].w, wt, o[3]);
                                o[4] = fmaf(q[i][1].x, wt, o[4]), o[5] = fmaf(q[i][1].y, wt, o[5]);
                                o[6] = fmaf(q[i][1].z, wt, o[6]), o[7] = fmaf(q[i][1].w, wt, o[7]);
                            }
                    }
                }
                if (parts > 1) {  // join the parts, in order, in the row's first
                    float *my = ex + tid;  // value e of a thread at ex[e * threads + thread]
                    named_bar_sync(BAR_ALL, SOFTMAX_THREADS);
#pragma unroll
                    for (int e = 0; e < 8; ++e) my[e * SOFTMAX_THREADS] = o[e];
                    my[8 * SOFTMAX_THREADS] = top, my[9 * SOFTMAX_THREADS] = lsum;
                    named_bar_sync(BAR_ALL, SOFTMAX_THREADS);
                    if (part == 0) {
#pragma unroll 1
                        for (int i = 1; i < parts; ++i) top = fmaxf(top, my[8 * SOFTMAX_THREADS + i * CHUNKS]);
                        lsum = 0.0f;
#pragma unroll
                        for (int e = 0; e < 8; ++e) o[e] = 0.0f;
#pragma unroll 1
                        for (int i = 0; i < parts; ++i) {
                            const float mi = my[8 * SOFTMAX_THREADS + i * CHUNKS];
                            if (mi == -INFINITY) continue;
                            const float wt = exp2_approx(mi - top);
                            lsum = fmaf(my[9 * SOFTMAX_THREADS + i * CHUNKS], wt, lsum);
#pragma unroll
                            for (int e = 0; e < 8; ++e) o[e] = fmaf(my[e * SOFTMAX_THREADS + i * CHUNKS], wt, o[e]);
                        }
                    }
                }
                if (on && part == 0) {
                    const float inv = lsum == 0.0f ? 0.0f : 1.0f / lsum;
#pragma unroll
                    for (int e = 0; e < 8; ++e) o[e] *= inv;
                    store8_bf16(out_row<HD>(p, u, rr) + 8 * c, o, p.a.out_pair_order);
                }
            }
            if (lane == 0 && seen == static_cast<unsigned>(k * SOFTMAX_WARPS - 1)) {
                atomicExch(&p.arrived[owner0], 0u);
                atomicExch(&p.done[owner0], 0u);
            }
            named_bar_sync(BAR_ALL, SOFTMAX_THREADS);  // the next unit uses `ex` again
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == MMA) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

}  // namespace tattn

size_t tree_attention_workspace_bytes(int head_dim, int num_sms) {
    return kPartialOffset + size_t(num_sms) * 2 * tattn::ROWS * (head_dim + 2) * 4;
}

template <int HD>
static cudaError_t launch(const tattn::Params &p, int grid, cudaStream_t stream, bool pdl) {
    using C = tattn::Cfg<HD>;
    const uint64_t dims[4] = {uint64_t(HD), uint64_t(1) << p.s.page_shift, uint64_t(p.s.kv_heads), uint64_t(p.s.pages)};
    const uint64_t strides[3] = {uint64_t(p.s.token_stride) * 2, uint64_t(p.s.head_stride) * 2,
                                 uint64_t(p.s.page_stride) * 2};
    const uint32_t rows = p.s.page_shift < 7 ? 1u << p.s.page_shift : 128u;
    const uint32_t box[4] = {64u, rows, 1u, 1u};
    CUtensorMap km, vm;
    if (!encode_tensor_map_4d(&km, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, p.a.k_cache, dims, strides, box,
                              CU_TENSOR_MAP_SWIZZLE_128B) ||
        !encode_tensor_map_4d(&vm, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, p.a.v_cache, dims, strides, box,
                              CU_TENSOR_MAP_SWIZZLE_128B))
        return cudaErrorInvalidValue;
    cudaError_t e = ensure_smem_attr(reinterpret_cast<const void *>(tattn::tree_attention_kernel<HD>), C::SMEM);
    if (e != cudaSuccess) return e;
    // CTAs of a unit wait for one another at its merge: all must be resident
    // (one per SM; a dependent launch's CTAs are, once each has started).
    e = launch_ex(tattn::tree_attention_kernel<HD>, dim3(grid), dim3(tattn::THREADS), C::SMEM, stream, !pdl, pdl, km, vm,
                  p);
    count_launch();
    return e;
}

cudaError_t launch_tree_attention(const PagedShape &s, const PagedStep &t, const TreeAttnArgs &a, void *workspace,
                                  int num_sms, cudaStream_t stream, bool pdl) {
    tattn::Params p{};
    p.s = s;
    p.t = t;
    p.a = a;
    p.group = a.q_heads / s.kv_heads;
    char *ws = static_cast<char *>(workspace);
    p.status = reinterpret_cast<unsigned *>(ws);
    p.arrived = reinterpret_cast<unsigned *>(ws + kCounterOffset);
    p.done = p.arrived + kMaxTiles / 2;
    p.partial = reinterpret_cast<float *>(ws + kPartialOffset);
    p.merge = qmv_combine_wait();
    // No more CTAs than tiles there can be.
    const int64_t positions = s.ld_table << s.page_shift;
    const int64_t tiles = (positions + tattn::TILE - 1) / tattn::TILE * s.kv_heads *
                          ((int64_t(s.max_nodes) * p.group + tattn::ROWS - 1) / tattn::ROWS);
    const int grid = tiles > num_sms / s.seqs ? num_sms : int(tiles * s.seqs);
    return s.head_dim == 128 ? launch<128>(p, grid, stream, pdl) : launch<64>(p, grid, stream, pdl);
}

}  // namespace afb
