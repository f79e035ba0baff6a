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
// graph follows them).  A CTA's range covers the end of one unit, whole units
// and the start of another; whole units are finished in place, pieces go to
// the workspace and the CTAs that share a unit merge it together at the end,
// each a share of its rows, in piece order (results do not depend on timing).
//
// Pipeline.  A producer warp brings K and V tiles page by page through a
// shared-memory ring (TMA, 128-byte swizzle); an MMA warp issues S = Q K^T
// (both from shared memory) and O += P V (P from tensor memory, V read along
// its dims); two warpgroups, a thread per row, turn S into P.  The two are two
// streams with their own S, O, maximum and sum: units of more than 128 rows
// give each its own 128 rows and both take every tile; smaller units give both
// the same rows and they take alternate tiles, merged when the unit ends.
// While one stream is in its softmax the tensor cores work for the other.
// A row's maximum is only raised (and O rescaled) when it grows by more than
// 2^8, so O is rarely touched.
//
// Rounding: P is rounded to bf16 for the tensor cores (as V is bf16, it is the
// smaller part of the result's own rounding); the sum l adds the rounded
// values, so a row's weights still sum to one.  Scores, maxima, sums and O are
// f32.
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
constexpr int PRODUCER = 8, MMA = 9;
constexpr int THREADS = 32 * 12;    // the last two warps only complete a warpgroup
// Registers per thread: 168 at launch, moved from the third warpgroup to the
// two softmax ones, whose threads hold a row of 128 scores.
constexpr int LAUNCH_REGS = 168, SOFTMAX_REGS = 208, OTHER_REGS = 88;
static_assert(2 * SOFTMAX_REGS + OTHER_REGS <= 3 * LAUNCH_REGS, "register split exceeds the launch allocation");
constexpr int HALF_BYTES = TILE * 128;  // 64 dims of a tile
constexpr float LOG2E = 1.4426950408889634f;
constexpr float RAISE = 8.0f;       // log2: how far scores may pass the running maximum before it is raised

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
};

// Where a CTA's share of the tiles begins.
struct Share {
    int64_t begin, end, total, at;  // at: `begin`'s offset within its sequence
    int seq, grid;
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

// Computed by one warp.
__device__ __forceinline__ void find_share(const Params &p, Share *out) {
    const int lane = threadIdx.x & 31;
    int64_t total = 0;
    for (int base = 0; base < p.s.seqs; base += 32) {
        int64_t mine = 0;
        if (base + lane < p.s.seqs) {
            const SeqTiles q = seq_tiles(p, base + lane);
            mine = q.tiles(p.s.kv_heads);
            if (!q.sp.ok && blockIdx.x == 0) atomicExch(p.status, static_cast<unsigned>(DEV_BOUNDS));
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
        total += mine;
    }
    Share r{};
    r.total = total;
    r.grid = static_cast<int>(total < gridDim.x ? total : gridDim.x);
    if (static_cast<int>(blockIdx.x) < r.grid) {
        r.begin = blockIdx.x * total / r.grid;
        r.end = (blockIdx.x + 1) * total / r.grid;
        int64_t before = 0;
        for (int base = 0; base < p.s.seqs; base += 32) {
            const int64_t mine = base + lane < p.s.seqs ? seq_tiles(p, base + lane).tiles(p.s.kv_heads) : 0;
            int64_t upto = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int64_t v = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += v;
            }
            const unsigned past = __ballot_sync(0xffffffffu, before + upto > r.begin);
            if (past) {
                const int l = __ffs(past) - 1;
                r.seq = base + l;
                r.at = r.begin - before - __shfl_sync(0xffffffffu, upto - mine, l);
                break;
            }
            before += __shfl_sync(0xffffffffu, upto, 31);
        }
    }
    if (lane == 0) *out = r;
}
// The CTA whose share holds tile x.
__device__ __forceinline__ int owner(const Share &sh, int64_t x) {
    return static_cast<int>(((x + 1) * sh.grid - 1) / sh.total);
}

// A piece of a unit: tiles [t0, t1) of nt.
struct Piece {
    int seq, first, n, ctx, kv, row0, rows, t0, t1, nt;
    int64_t start;  // the unit's first tile in the order of all tiles
    __device__ __forceinline__ bool both() const { return rows > TILE; }  // two row tiles, every position tile for both
    __device__ __forceinline__ int items() const { return both() ? 2 * (t1 - t0) : t1 - t0; }
};
struct Walk {
    int64_t pos, end, at;
    int seq;
    SeqTiles q;
    __device__ __forceinline__ Walk(const Params &p, const Share &sh) : pos(sh.begin), end(sh.end), at(sh.at), seq(sh.seq) {
        if (pos < end) q = seq_tiles(p, seq);
    }
    __device__ __forceinline__ bool next(const Params &p, Piece &d) {
        if (pos >= end) return false;
        while (at >= q.tiles(p.s.kv_heads)) {
            at = 0;
            q = seq_tiles(p, ++seq);
        }
        const int64_t unit = at / q.nt;
        d.seq = seq;
        d.first = q.sp.first;
        d.n = q.n;
        d.ctx = q.sp.ctx;
        d.nt = q.nt;
        d.t0 = static_cast<int>(at - unit * q.nt);
        const int64_t left = end - pos;
        d.t1 = left < q.nt - d.t0 ? d.t0 + static_cast<int>(left) : q.nt;
        d.kv = static_cast<int>(unit / q.units);
        d.row0 = static_cast<int>(unit % q.units) * ROWS;
        d.rows = min(ROWS, q.n * p.group - d.row0);
        d.start = pos - d.t0;
        pos += d.t1 - d.t0;
        at += d.t1 - d.t0;
        return true;
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

// A whole warp's wait, with one answer: false once any wait of the CTA gave up.
__device__ __forceinline__ bool warp_wait(uint64_t *bar, uint32_t parity, volatile int *abort, unsigned *status) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort, status) && !*abort);
}

template <int N>
__device__ __forceinline__ void store_out(uint16_t *dst, const float (&x)[N], int pair_order) {
#pragma unroll
    for (int i = 0; i < N; i += 8) {
        uint4 u;
        if (pair_order)
            u = make_uint4(pack_bf16x2(x[i], x[i + 4]), pack_bf16x2(x[i + 1], x[i + 5]), pack_bf16x2(x[i + 2], x[i + 6]),
                           pack_bf16x2(x[i + 3], x[i + 7]));
        else
            u = make_uint4(pack_bf16x2(x[i], x[i + 1]), pack_bf16x2(x[i + 2], x[i + 3]), pack_bf16x2(x[i + 4], x[i + 5]),
                           pack_bf16x2(x[i + 6], x[i + 7]));
        *reinterpret_cast<uint4 *>(dst + i) = u;
    }
}
__device__ __forceinline__ float finish(float o, float l) { return l == 0.0f ? 0.0f : o / l; }

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
    uint64_t *q_full = p_full + 2;
    uint64_t *unit_done = q_full + 1;      // every MMA of the piece has ended
    Share *share = reinterpret_cast<Share *>(unit_done + 1);
    Piece *shared_units = reinterpret_cast<Piece *>(share + 1);  // [2] pieces of shared units: the end of one, the start of another
    uint32_t *odd = reinterpret_cast<uint32_t *>(shared_units + 2);  // [8] drafted nodes whose values are not all finite
    uint32_t *tmem_addr = odd + 8;
    volatile int *abort = reinterpret_cast<volatile int *>(tmem_addr + 1);
    int *go = const_cast<int *>(abort) + 1;

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) {
        for (int i = 0; i < C::STAGES; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 128);
        }
        mbar_init(q_full, 32 * SOFTMAX_WARPS);
        mbar_init(unit_done, 2);
        *abort = 0;
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
    pdl_wait();  // lengths, queries and the cache come from the preceding kernels
    if (warp == 0) find_share(p, share);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const Share sh = *share;
    const uint32_t tmem = *tmem_addr;

    if (warp == PRODUCER) {  // ------------------------------------------------- K and V tiles
        regs_release<OTHER_REGS>();
        const int rows_per_box = min(1 << p.s.page_shift, TILE);
        const uint64_t once = l2_evict_first(), again = l2_evict_normal();
        uint32_t seq_no = 0;  // ring position, over all pieces
        bool live = true;
        Walk walk(p, sh);
        Piece d;
        while (live && walk.next(p, d)) {
            const int *table = p.t.page_table + d.seq * p.s.ld_table;
            // Several row tiles read the same cache: keep it in L2 for them.
            const uint64_t policy = d.n * p.group > ROWS ? again : once;
            const int nt = d.t1 - d.t0;
            for (int i = 0; i < 2 * nt && live; ++i, ++seq_no) {
                // The order in which the MMA warp consumes them.
                bool is_v;
                int t;
                if (d.both()) {
                    is_v = i & 1;
                    t = i >> 1;
                } else {  // K0 K1 V0 K2 V1 .. K(nt-1) V(nt-2) V(nt-1)
                    is_v = i == 2 * nt - 1 || (i >= 2 && !(i & 1));
                    t = i == 2 * nt - 1 ? nt - 1 : is_v ? i / 2 - 1 : (i + 1) / 2;
                }
                const int pos = (d.t0 + t) * TILE;
                const int valid = min(TILE, d.ctx + d.n - pos);
                const int boxes = (valid + rows_per_box - 1) / rows_per_box * C::HALVES;
                const int box = lane / C::HALVES, half = lane % C::HALVES;
                int page = 0;
                if (lane < boxes) {
                    page = table[(pos + box * rows_per_box) >> p.s.page_shift];
                    if (page < 0 || page >= p.s.pages) {  // a coordinate outside the map reads zeros
                        atomicExch(p.status, static_cast<unsigned>(DEV_BOUNDS));
                        page = static_cast<int>(p.s.pages);
                    }
                }
                const int stage = seq_no % C::STAGES;
                live = warp_wait(&empty[stage], ((seq_no / C::STAGES) & 1) ^ 1, abort, p.status);
                if (!live) break;  // never re-arm after an abort
                if (lane == 0) mbar_arrive_expect_tx(&full[stage], boxes * rows_per_box * 128);
                __syncwarp();
                if (lane < boxes)
                    tma_load_4d_hint(ring + stage * C::TILE_BYTES + half * HALF_BYTES + box * rows_per_box * 128,
                                     is_v ? &vmap : &kmap, &full[stage], half * 64, pos & ((1 << p.s.page_shift) - 1),
                                     d.kv, page, policy);
                __syncwarp();
            }
        }
        // Copies in flight land before the CTA leaves.
        for (uint32_t back = 1; back <= C::STAGES && back <= seq_no; ++back) {
            const uint32_t i = seq_no - back;
            mbar_wait_drain(&full[i % C::STAGES], (i / C::STAGES) & 1);
        }
    } else if (warp == MMA) {  // ------------------------------------------------ tensor cores
        regs_release<OTHER_REGS>();
        const uint32_t idesc_s = umma_idesc_bf16(128, TILE), idesc_o = umma_idesc_bf16(128, HD) | kUmmaTransposeB;
        const uint32_t q_addr = smem_u32(qbuf), ring_addr = smem_u32(ring);
        uint32_t base = 0, q_phase = 0, p_phase[2] = {0, 0};
        bool live = true;
        Walk walk(p, sh);
        Piece d;
        while (live && walk.next(p, d)) {
            const int nt = d.t1 - d.t0, items = d.items();
            const bool both = d.both();
            live = warp_wait(q_full, q_phase, abort, p.status);
            q_phase ^= 1;
            if (!live) break;
            tc_fence_after();
            if (lane < 8) odd[lane] = 0u;
            __syncwarp();
            auto scores = [&](int w) {
                const int t = both ? w >> 1 : w, st = w & 1;
                const uint32_t no = base + (both ? 2 * t : t == 0 ? 0 : 2 * t - 1);
                const int stage = no % C::STAGES;
                if (!both || st == 0) live = warp_wait(&full[stage], (no / C::STAGES) & 1, abort, p.status);
                if (!live) return;
                if (lane == 0) {
                    const uint32_t a = q_addr + (both ? st : 0) * C::TILE_BYTES, b = ring_addr + stage * C::TILE_BYTES;
#pragma unroll
                    for (int ks = 0; ks < HD / 16; ++ks) {
                        const uint32_t off = (ks >> 2) * HALF_BYTES + (ks & 3) * 32;
                        umma_bf16_ss(tmem + st * TILE, umma_desc_sw128(a + off), umma_desc_sw128(b + off), idesc_s,
                                     ks > 0);
                    }
                    umma_commit(&s_full[st]);
                    if (!both || st == 1) umma_commit(&empty[stage]);
                }
                __syncwarp();
            };
            auto values = [&](int w) {
                const int t = both ? w >> 1 : w, st = w & 1;
                const uint32_t no = base + (both ? 2 * t + 1 : t == nt - 1 ? 2 * nt - 1 : 2 * t + 2);
                const int stage = no % C::STAGES;
                if (!both || st == 0) {
                    live = warp_wait(&full[stage], (no / C::STAGES) & 1, abort, p.status);
                    if (!live) return;
                    const int pos = (d.t0 + t) * TILE, valid = min(TILE, d.ctx + d.n - pos);
                    if (valid < TILE || pos + TILE > d.ctx) {
                        // A probability of zero does not hide what is not
                        // finite: rows behind the last position (never
                        // loaded, or whatever a page held) become zeros, and
                        // so do the infinities and NaN of drafted values,
                        // which only some rows see; those rows get them back
                        // at the end.
                        char *v = ring + stage * C::TILE_BYTES;
                        const int from = max(0, d.ctx - pos);
                        for (int i = from * 8 + lane; i < TILE * 8; i += 32) {
#pragma unroll
                            for (int h = 0; h < C::HALVES; ++h) {
                                uint4 *c = reinterpret_cast<uint4 *>(v + h * HALF_BYTES + i * 16);
                                if ((i >> 3) >= valid) {
                                    *c = make_uint4(0u, 0u, 0u, 0u);
                                    continue;
                                }
                                const uint4 u = *c;
                                uint32_t x[4] = {u.x, u.y, u.z, u.w};
                                bool bad = false;
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    if ((x[e] & 0x7F80u) == 0x7F80u) x[e] &= 0xFFFF0000u, bad = true;
                                    if ((x[e] & 0x7F800000u) == 0x7F800000u) x[e] &= 0x0000FFFFu, bad = true;
                                }
                                if (bad) {
                                    *c = make_uint4(x[0], x[1], x[2], x[3]);
                                    const int j = pos + (i >> 3) - d.ctx;
                                    atomicOr(&odd[j >> 5], 1u << (j & 31));
                                }
                            }
                        }
                        fence_proxy_async_smem();
                        __syncwarp();
                    }
                }
                live = warp_wait(&p_full[st], p_phase[st], abort, p.status);
                p_phase[st] ^= 1;
                if (!live) return;
                tc_fence_after();
                if (lane == 0) {
                    const uint32_t b = ring_addr + stage * C::TILE_BYTES;
#pragma unroll
                    for (int ks = 0; ks < TILE / 16; ++ks)
                        umma_bf16_ts(tmem + 2 * TILE + st * HD, tmem + st * TILE + ks * 8,
                                     umma_desc_mn_sw128(b + ks * 2048, HALF_BYTES), idesc_o, w >= 2 || ks > 0);
                    if (!both || st == 1) umma_commit(&empty[stage]);
                }
                __syncwarp();
            };
            scores(0);
            if (live && items > 1) scores(1);
            for (int w = 0; w < items && live; ++w) {
                values(w);
                if (live && w + 2 < items) scores(w + 2);
            }
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(unit_done);  // `odd` is written
                umma_commit(unit_done);
            }
            base += 2 * nt;
        }
        // On the way out of an abort, MMAs in flight end before tensor memory is freed.
        if (!live) {
            if (lane == 0) umma_commit(&s_full[0]);
            for (int i = 0; i < 2; ++i) mbar_wait_drain(&s_full[0], i, 1000000ull);
        }
    } else if (warp < SOFTMAX_WARPS) {  // ----------------------------------------- softmax
        regs_claim<SOFTMAX_REGS>();
        const int st = warp >> 2, r = tid & 127;
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t ts = tmem + lanes + st * TILE, to = tmem + lanes + 2 * TILE;
        const float sc = (p.a.scale == 0.0f ? 1.0f : fabsf(p.a.scale)) * LOG2E;
        uint32_t s_phase = 0, u_phase = 0;
        bool head = false, tail = false;
        Walk walk(p, sh);
        Piece d;
        while (walk.next(p, d)) {
            const bool both = d.both();
            // Queries, in the operand layout; zeros in rows that the unit lacks.
            // A negative scale flips their signs and a zero one clears them,
            // so the running maximum can work on the scores as they come.
            const uint32_t flip = p.a.scale < 0.0f ? 0x80008000u : 0u;
            const int chunks = (both ? ROWS : TILE) * (HD / 8);
            for (int i = tid; i < chunks; i += 32 * SOFTMAX_WARPS) {
                const int rr = i / (HD / 8), c = i % (HD / 8);
                uint4 u = make_uint4(0u, 0u, 0u, 0u);
                if (rr < d.rows && p.a.scale != 0.0f) {
                    const int x = d.row0 + rr, node = x / p.group, g = x - node * p.group;
                    u = *reinterpret_cast<const uint4 *>(p.a.q + (static_cast<int64_t>(d.first) + node) * p.a.ld_q +
                                                         (static_cast<int64_t>(d.kv) * p.group + g) * HD + c * 8);
                    u.x ^= flip, u.y ^= flip, u.z ^= flip, u.w ^= flip;
                }
                *reinterpret_cast<uint4 *>(qbuf + (rr >> 7) * C::TILE_BYTES + (c >> 3) * HALF_BYTES + (rr & 127) * 128 +
                                           (((c & 7) ^ (rr & 7)) << 4)) = u;
            }
            fence_proxy_async_smem();
            tc_fence_before();  // the last piece's reads of tensor memory, too
            mbar_arrive(q_full);

            const int rr = both ? st * TILE + r : r;  // this thread's row of the unit
            const bool mine = rr < d.rows;
            const bool warp_on = __any_sync(0xffffffffu, mine);
            const int x = d.row0 + rr, node = mine ? x / p.group : 0;
            const int64_t row = static_cast<int64_t>(d.first) + node;
            const RowMask mask{p.a.mask ? p.a.mask + row * p.s.mask_words : nullptr, d.n, node};
            float m = -INFINITY, l = 0.0f;
            const int items = d.items();
            for (int w = st; w < items; w += 2) {
                mbar_wait(&s_full[st], s_phase, abort, p.status);
                s_phase ^= 1;
                tc_fence_after();
                if (warp_on) {
                    uint32_t v[4][32];
#pragma unroll
                    for (int k = 0; k < 4; ++k) tmem_ld_32x32b_x32(ts + 32 * k, v[k]);
                    tmem_wait_ld();
#pragma unroll
                    for (int k = 0; k < 4; ++k) tie_regs(v[k]);
                    const int pos = (d.t0 + (both ? w >> 1 : w)) * TILE;
                    if (pos + TILE > d.ctx) {
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const uint32_t see = mask.bits(pos + 32 * k - d.ctx);
#pragma unroll
                            for (int e = 0; e < 32; ++e)
                                if (!((see >> e) & 1u)) v[k][e] = 0xFF800000u;  // -inf
                        }
                    }
                    float mx[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        mx[k] = __uint_as_float(v[k][0]);
#pragma unroll
                        for (int e = 1; e < 32; ++e) mx[k] = fmaxf(mx[k], __uint_as_float(v[k][e]));
                    }
                    const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
                    const bool raise = top > m && (m == -INFINITY || (top - m) * sc > RAISE);
                    if (__any_sync(0xffffffffu, raise)) {
                        const float corr = !raise ? 1.0f : m == -INFINITY ? 0.0f : exp2_approx((m - top) * sc);
                        if (raise) m = top;
                        l *= corr;
                        if (w >= 2) {  // this stream's O holds something
#pragma unroll
                            for (int c = 0; c < HD; c += 16) {
                                uint32_t o[16];
                                tmem_ld_32x32b_x16(to + st * HD + c, o);
                                tmem_wait_ld(o);
#pragma unroll
                                for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * corr);
                                tmem_st_32x32b_x16(to + st * HD + c, o);
                            }
                        }
                    }
                    const float off = m == -INFINITY ? 0.0f : m * sc;
                    float sum[2] = {0.0f, 0.0f};
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        uint32_t u[16];
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const float a = exp2_approx(fmaf(__uint_as_float(v[k][2 * e]), sc, -off));
                            const float b = exp2_approx(fmaf(__uint_as_float(v[k][2 * e + 1]), sc, -off));
                            u[e] = pack_bf16x2(a, b);
                            sum[0] += __uint_as_float(u[e] << 16);
                            sum[1] += __uint_as_float(u[e] & 0xFFFF0000u);
                        }
                        tmem_st_32x32b_x16(ts + 16 * k, u);
                    }
                    l += sum[0] + sum[1];
                    tmem_wait_st();
                }
                tc_fence_before();
                mbar_arrive(&p_full[st]);
            }
            mbar_wait(unit_done, u_phase, abort, p.status);
            u_phase ^= 1;
            tc_fence_after();

            // The piece's result: one stream's rows, or both streams' halves
            // of the tiles joined (each warpgroup half of the dims).
            // Log2 units; a row whose sum is NaN keeps a finite maximum, so
            // that no join takes it for one that saw nothing.
            const float m2 = l != l ? 0.0f : m == -INFINITY ? -INFINITY : m * sc;
            float top = m2, lsum = l, w_own = m2 == -INFINITY ? 0.0f : 1.0f, w_other = 0.0f;
            if (!both) {
                float *ex = reinterpret_cast<float *>(qbuf);  // the queries are done with
                ex[st * TILE + r] = m2;
                ex[2 * TILE + st * TILE + r] = l;
                named_bar_sync(1, 32 * SOFTMAX_WARPS);
                const float mo = ex[(st ^ 1) * TILE + r], lo = ex[2 * TILE + (st ^ 1) * TILE + r];
                named_bar_sync(1, 32 * SOFTMAX_WARPS);
                top = fmaxf(m2, mo);
                w_own = m2 == -INFINITY ? 0.0f : exp2_approx(m2 - top);
                w_other = mo == -INFINITY ? 0.0f : exp2_approx(mo - top);
                lsum = st == 0 ? l * w_own + lo * w_other : lo * w_other + l * w_own;
            }
            const bool whole = d.t0 == 0 && d.t1 == d.nt;
            float *rec = p.partial + (2 * static_cast<int64_t>(blockIdx.x) + (d.t0 == 0 ? 1 : 0)) * C::RECORD;
            const int dim0 = both ? 0 : st * (HD / 2), dim1 = both ? HD : dim0 + HD / 2;
            const float w0 = both ? w_own : st == 0 ? w_own : w_other, w1 = both ? 0.0f : st == 0 ? w_other : w_own;
            if (warp_on) {
                for (int c = dim0; c < dim1; c += 32) {
                    uint32_t a[32], b[32];
                    float o[32];
                    tmem_ld_32x32b_x32(to + (both ? st * HD : 0) + c, a);
                    if (!both) tmem_ld_32x32b_x32(to + HD + c, b);
                    tmem_wait_ld();
                    tie_regs(a);
                    if (!both) tie_regs(b);
#pragma unroll
                    for (int e = 0; e < 32; ++e) {
                        // a stream that saw nothing may hold anything
                        o[e] = w0 == 0.0f ? 0.0f : __uint_as_float(a[e]) * w0;
                        if (!both && w1 != 0.0f) o[e] = fmaf(__uint_as_float(b[e]), w1, o[e]);
                    }
                    // Infinities and NaN among the drafted values, for the rows that see them.
                    for (int k = 0; k < 8; ++k) {
                        uint32_t set = odd[k];
                        if (set) set &= mask.word(k);
                        for (; set && mine; set &= set - 1) {
                            const int pos = d.ctx + 32 * k + __ffs(set) - 1;
                            const int page = p.t.page_table[d.seq * p.s.ld_table + (pos >> p.s.page_shift)];
                            if (page < 0 || page >= p.s.pages) continue;
                            const uint16_t *src = p.a.v_cache + page * p.s.page_stride + d.kv * p.s.head_stride +
                                                  (pos & ((1 << p.s.page_shift) - 1)) * p.s.token_stride + c;
#pragma unroll
                            for (int e = 0; e < 32; ++e) {
                                const uint16_t h = src[e];
                                if ((h & 0x7F80u) == 0x7F80u) o[e] += bf16_bits_to_f32(h);
                            }
                        }
                    }
                    if (mine && whole) {
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = finish(o[e], lsum);
                        store_out(p.a.out + row * p.a.ld_out +
                                      (static_cast<int64_t>(d.kv) * p.group + (x - node * p.group)) * HD + c,
                                  o, p.a.out_pair_order);
                    } else if (mine) {
#pragma unroll
                        for (int e = 0; e < 32; e += 4)
                            *reinterpret_cast<float4 *>(rec + rr * HD + c + e) =
                                make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                    }
                }
                if (mine && !whole && dim0 == 0) {
                    rec[ROWS * HD + rr] = top;
                    rec[ROWS * HD + ROWS + rr] = lsum;
                }
            }
            if (!whole) {
                (d.t0 > 0 ? head : tail) = true;
                if (tid == 0) shared_units[d.t0 > 0 ? 0 : 1] = d;
                asm volatile("fence.acq_rel.gpu;" ::: "memory");
                named_bar_sync(1, 32 * SOFTMAX_WARPS);
                if (tid == 0) atomicAdd(&p.arrived[owner(sh, d.start)], 1u);
            }
        }
        // Merge the shared units: this CTA's share of their rows.
        for (int which = 0; which < 2; ++which) {
            if (!(which ? tail : head)) continue;
            const Piece u = shared_units[which];
            const int c0 = owner(sh, u.start), c1 = owner(sh, u.start + u.nt - 1), k = c1 - c0 + 1;
            const int me = blockIdx.x - c0;
            const int r0 = u.rows * me / k, r1 = u.rows * (me + 1) / k;
            if (r1 > r0) {
                if (tid == 0) {
                    const uint64_t since = globaltimer();
                    int ok = 1;
                    while (ok && *reinterpret_cast<volatile unsigned *>(&p.arrived[c0]) != static_cast<unsigned>(k)) {
                        if (*abort || globaltimer() - since > kArrivalWaitNs) {
                            atomicExch(p.status, static_cast<unsigned>(DEV_TIMEOUT));
                            ok = 0;
                        }
                    }
                    *go = ok;
                }
                named_bar_sync(1, 32 * SOFTMAX_WARPS);
                if (*go) {
                    asm volatile("fence.acq_rel.gpu;" ::: "memory");
                    constexpr int W = HD / 32;
                    for (int rr = r0 + warp; rr < r1; rr += SOFTMAX_WARPS) {
                        // weights: lanes over pieces
                        float top = -INFINITY;
                        for (int j = lane; j < k; j += 32)
                            top = fmaxf(top, __ldcg(p.partial + (2 * static_cast<int64_t>(c0 + j) + (j == 0)) * C::RECORD +
                                                    ROWS * HD + rr));
#pragma unroll
                        for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                        float lsum = 0.0f, o[W];
#pragma unroll
                        for (int e = 0; e < W; ++e) o[e] = 0.0f;
                        for (int j0 = 0; j0 < k; j0 += 32) {
                            float wt = 0.0f;
                            if (j0 + lane < k) {
                                const float *rec = p.partial + (2 * static_cast<int64_t>(c0 + j0 + lane) + (j0 + lane == 0)) * C::RECORD;
                                const float mj = __ldcg(rec + ROWS * HD + rr);
                                wt = mj == -INFINITY ? 0.0f : exp2_approx(mj - top);
                                lsum = fmaf(__ldcg(rec + ROWS * HD + ROWS + rr), wt, lsum);
                            }
                            const int cnt = min(32, k - j0);
#pragma unroll 8
                            for (int j = 0; j < cnt; ++j) {
                                const float wj = __shfl_sync(0xffffffffu, wt, j);
                                const float *rec = p.partial + (2 * static_cast<int64_t>(c0 + j0 + j) + (j0 + j == 0)) * C::RECORD +
                                                   rr * HD + lane * W;
                                float q[W];
                                if (W == 4) *reinterpret_cast<float4 *>(q) = __ldcg(reinterpret_cast<const float4 *>(rec));
                                else *reinterpret_cast<float2 *>(q) = __ldcg(reinterpret_cast<const float2 *>(rec));
#pragma unroll
                                for (int e = 0; e < W; ++e) o[e] = fmaf(q[e], wj, o[e]);
                            }
                        }
#pragma unroll
                        for (int s = 16; s; s >>= 1) lsum += __shfl_xor_sync(0xffffffffu, lsum, s);
                        const int x = u.row0 + rr, node = x / p.group, g = x - node * p.group;
                        uint16_t *dst = p.a.out + (static_cast<int64_t>(u.first) + node) * p.a.ld_out +
                                        (static_cast<int64_t>(u.kv) * p.group + g) * HD;
#pragma unroll
                        for (int e = 0; e < W; ++e) {
                            const int dim = lane * W + e, in8 = dim & 7;
                            const int col = p.a.out_pair_order ? (dim & ~7) + (in8 < 4 ? 2 * in8 : 2 * (in8 - 4) + 1) : dim;
                            dst[col] = f32_to_bf16_bits(finish(o[e], lsum));
                        }
                    }
                }
                named_bar_sync(1, 32 * SOFTMAX_WARPS);
            }
            // The last of the unit's CTAs clears its counters for the next launch.
            if (tid == 0 && atomicAdd(&p.done[c0], 1u) == static_cast<unsigned>(k - 1)) {
                atomicExch(&p.arrived[c0], 0u);
                atomicExch(&p.done[c0], 0u);
            }
        }
    } else {
        regs_release<OTHER_REGS>();
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
    // No more CTAs than tiles there can be.
    const int64_t positions = s.ld_table << s.page_shift;
    const int64_t tiles = (positions + tattn::TILE - 1) / tattn::TILE * s.kv_heads *
                          ((int64_t(s.max_nodes) * p.group + tattn::ROWS - 1) / tattn::ROWS);
    const int grid = tiles > num_sms / s.seqs ? num_sms : int(tiles * s.seqs);
    return s.head_dim == 128 ? launch<128>(p, grid, stream, pdl) : launch<64>(p, grid, stream, pdl);
}

}  // namespace afb
