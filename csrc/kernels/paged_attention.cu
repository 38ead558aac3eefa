// Attention of a ragged batch of new tokens over a paged KV cache.
//
//     out[t, h] = sum_p w_p v_p / sum_p w_p,   w_p = exp(scale * q[t, h] . k_p - m)
//
// over the keys p that row t sees; m is a reference near the row's largest
// score, and a row that sees no key gives zeros.
//
// One persistent CTA an SM goes through its part of the plan
// (attention_plan.h) in one pass over the keys. Two streams of 128 rows run
// against each other so that the tensor core works on one while the other's
// softmax is computed: stream s has the scores S_s (128 x 128, fp32) and the
// output O_s (128 x dim, fp32) in tensor memory, and the weights P_s, 16-bit,
// in place of S_s. A tile of more than 128 rows gives each stream half of its
// rows, over the same keys. A smaller one (single tokens) gives both streams
// the same rows and every second block of keys, and they are joined at the
// end, so the loads never wait for one stream's softmax.
//
//   warps 0-3, 4-7  the softmax of stream 0, 1: a thread has a row
//   warp 8          walks the plan, loads K and V blocks by TMA (a page, or
//                   the part of one that lies in the block, a box)
//   warp 9          issues the matrix instructions
//   warps 10, 11    load the queries
//
// Weights are rounded to the cache's type for the second product; sums,
// maxima, scores and outputs are 32-bit. m only moves when a score passes it
// by 2^8 (kRescale), so O_s is hardly ever rescaled; the weights then reach
// 2^8, which both types hold with the same relative precision.
//
// Keys that no row of a tile sees (behind a sequence, before a window, on a
// page that is none) are read as zeros: their boxes are put outside the pool,
// where the TMA fills zeros. So nothing that lies there reaches a result, and
// a masked score is replaced, never added to.
#include <atomic>
#include <cstring>

#include "cuda/gpu.h"
#include "kernels/attention_plan.h"
#include "kernels/kv.cuh"
#include "kernels/umma.cuh"

namespace mpcomm {
namespace kern {
namespace {

constexpr int kThreads = 384;
constexpr int kStreamRows = 128;
constexpr int kRunSlots = 4;
constexpr int kMaskSlots = 16;  // blocks whose masks are kept: more than are ever in flight
constexpr float kRescale = 8.f;

__device__ uint32_t g_attention_status;

// What the plan's warp tells the others of a run.
struct RunInfo {
    int blocks;  // 0: no more runs
    int pair;    // each stream its own rows; else both streams the same
    int rows;    // of the tile
    int r0;      // the tile's first row in its sequence
    int q0;      // the sequence's first row of the query tensor
    int h;       // key head
    int key0;    // first key of the run's first block
    int first;   // position of the sequence's first new token
    int end;     // keys of the sequence
    int part;    // -1: the run is the whole tile; else its slot in the workspace
};

template <int DP>
struct Layout {
    static constexpr int kTile = kStreamRows * DP * 2;  // 128 rows of DP 16-bit elements
    static constexpr int kStages = DP == 128 ? 5 : 10;
    static constexpr int kQ = 0;
    static constexpr int kKv = 2 * kTile;
    static constexpr int kControl = kKv + kStages * kTile;
};

template <int STAGES>
struct Control {
    uint64_t kv_full[STAGES], kv_empty[STAGES];
    uint64_t q_full[2], q_empty[2];
    uint64_t s_full[2], p_full[2], o_full[2];
    uint64_t join_full, join_empty, drain;
    uint64_t run_full[kRunSlots], run_empty[kRunSlots];
    uint32_t mask[kMaskSlots];  // good boxes of a block
    RunInfo run[kRunSlots];
    float join[kStreamRows][2];  // m and sum of stream 1's rows, for stream 0
    uint32_t tmem;
    uint32_t dead;  // a wait ran out: nothing is waited for any more
};

struct Part {  // a tile whose blocks several CTAs share, from its first CTA on
    int pieces;
    int q0, r0, rows, h;
};

// Bytes of a workspace: the parts, then two slots a CTA of kTileRows rows each.
__host__ __device__ constexpr size_t parts_bytes(int ctas) { return (sizeof(Part) * ctas + 255) / 256 * 256; }
__host__ __device__ constexpr size_t slot_bytes(int dp) { return static_cast<size_t>(kTileRows) * (dp + 2) * 4; }

struct KernelArgs {
    PagedAttentionArgs a;
    PlanShape shape;
    float scale_log2;  // |scale| * log2(e)
    uint32_t negate;   // sign bits to flip in the queries: scale is negative
    int ctas;
    int box;  // tokens of a full box
    uint64_t budget;
};

template <int DP, typename T>
struct Kernel {
    using L = Layout<DP>;
    using C = Control<L::kStages>;
    static constexpr int kHalves = DP / 64;
    static constexpr int kHalfBytes = kStreamRows * 128;
    // columns of tensor memory: scores and weights, output of a stream
    static __device__ __forceinline__ uint32_t s_at(int s) { return s * 128; }
    static __device__ __forceinline__ uint32_t o_at(int s) { return 256 + s * DP; }
    static constexpr bool kBf16Type = std::is_same_v<T, __nv_bfloat16>;

    const KernelArgs &g;
    char *smem;
    C *c;
    int lane;

    __device__ uint32_t *status() const { return g.a.status ? g.a.status : &g_attention_status; }

    // Waits for a phase; gives up after the budget, and at once when any wait of the CTA has given up.
    __device__ __noinline__ void wait_slow(uint64_t *bar, uint32_t parity) const {
        volatile uint32_t *dead = &c->dead;
        const uint64_t t0 = globaltimer_ns();
        for (;;) {
            if (mbar_try_wait(bar, parity) || *dead) return;
            if (globaltimer_ns() - t0 > g.budget) {
                *dead = 1;
                atomicOr(status(), kStatusLoadTimeout);
                return;
            }
        }
    }
    __device__ __forceinline__ void wait(uint64_t *bar, uint32_t parity) const {
        if (!mbar_try_wait(bar, parity)) wait_slow(bar, parity);
    }

    // Whether some wait has given up, the same for a whole warp.
    __device__ __forceinline__ bool gave_up() const {
        return __any_sync(~0u, *const_cast<volatile uint32_t *>(&c->dead) != 0);
    }

    // The next run, read by a whole warp; the slot is given back at once.
    __device__ __forceinline__ RunInfo take_run(int &n) const {
        const int slot = n % kRunSlots;
        wait(&c->run_full[slot], (n / kRunSlots) & 1);
        RunInfo r = c->run[slot];
        if (gave_up()) r.blocks = 0;
        if (lane == 0) mbar_arrive(&c->run_empty[slot]);
        ++n;
        return r;
    }

    // ---- warp 8: the plan, and K and V ----
    __device__ void load_loop(const CUtensorMap *boxes, const CUtensorMap *lines) const {
        const KvBatch &k = g.a.batch;
        const PlanShape &s = g.shape;
        int64_t units = 0;
        for (int b0 = 0; b0 < k.seqs; b0 += 32) {
            const int b = b0 + lane;
            if (b < k.seqs) units += s.kv_heads * plan_head_units(s, plan_seq(s, k.starts.at(b), k.starts.at(b + 1), k.lens.at(b)));
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) units += __shfl_xor_sync(~0u, units, o);
        const int64_t share = plan_share(units, g.ctas);
        int64_t at = blockIdx.x * share;
        int64_t left = units - at < share ? units - at : share;
        Part *part = static_cast<Part *>(g.a.workspace) + blockIdx.x;
        Part mine{0, 0, 0, 0, 0};
        int n_run = 0;
        int64_t n_kv = 0;
        int n_block = 0;
        if (left > 0) {
            // the sequence that holds unit `at`
            int b = 0;
            int64_t head = 0;
            for (int b0 = 0; b0 < k.seqs; b0 += 32) {
                int64_t own = 0, sum;
                if (b0 + lane < k.seqs)
                    own = plan_head_units(s, plan_seq(s, k.starts.at(b0 + lane), k.starts.at(b0 + lane + 1), k.lens.at(b0 + lane)));
                sum = own * s.kv_heads;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int64_t up = __shfl_up_sync(~0u, sum, o);
                    if (lane >= o) sum += up;
                }
                const uint32_t past = __ballot_sync(~0u, sum > at);
                if (past) {
                    const int i = __ffs(past) - 1;
                    b = b0 + i;
                    head = __shfl_sync(~0u, own, i);
                    at -= __shfl_sync(~0u, sum, i) - head * s.kv_heads;
                    break;
                }
                at -= __shfl_sync(~0u, sum, 31);
            }
            PlanSeq q = plan_seq(s, k.starts.at(b), k.starts.at(b + 1), k.lens.at(b));
            PlanCursor cur;
            cur.seek(s, q, head, at);
            while (left > 0) {
                PlanRun run;
                if (!cur.next(s, q, left, &run)) {
                    ++b;
                    q = plan_seq(s, k.starts.at(b), k.starts.at(b + 1), k.lens.at(b));
                    cur = PlanCursor();
                    continue;
                }
                left -= run.to - run.from;
                const bool whole = run.from == 0 && run.to == run.tile.blocks;
                if (run.from == 0 && !whole) {
                    const int64_t rest = run.tile.blocks - run.to;
                    mine = Part{static_cast<int>(1 + (rest + share - 1) / share), q.q0, run.m * kTileRows, run.tile.rows, run.h};
                }
                const int slot = n_run % kRunSlots;
                wait(&c->run_empty[slot], ((n_run / kRunSlots) & 1) ^ 1);
                if (lane == 0) {
                    RunInfo &r = c->run[slot];
                    r.blocks = run.to - run.from;
                    r.pair = run.tile.rows > kStreamRows;
                    r.rows = run.tile.rows;
                    r.r0 = run.m * kTileRows;
                    r.q0 = q.q0;
                    r.h = run.h;
                    r.key0 = (run.tile.block0 + run.from) * kBlockKeys;
                    r.first = q.first;
                    r.end = q.end;
                    r.part = whole ? -1 : run.from == 0 ? 1 : 0;
                    mbar_arrive(&c->run_full[slot]);
                }
                ++n_run;
                load_run(boxes, lines, b, run, n_kv, n_block);
            }
        }
        const int slot = n_run % kRunSlots;
        wait(&c->run_empty[slot], ((n_run / kRunSlots) & 1) ^ 1);
        if (lane == 0) {
            c->run[slot].blocks = 0;
            mbar_arrive(&c->run_full[slot]);
            if (g.a.workspace) *part = mine;
        }
        // After a wait that ran out, loads may be in flight that nobody has
        // waited for: shared memory stays ours until they have landed.
        if (gave_up() && lane == 0) {
            for (int64_t i = n_kv > L::kStages ? n_kv - L::kStages : 0; i < n_kv; ++i)
                mbar_wait_bounded(&c->kv_full[i % L::kStages], (i / L::kStages) & 1, g.budget);
        }
    }

    __device__ __forceinline__ int page_at(int b, int key, int lo, int hi, bool *bad) const {
        if (key >= hi || key + g.box <= lo) return static_cast<int>(g.a.batch.pages);  // nobody sees it: zeros
        const int64_t page = page_of(g.a.batch, b, key);
        *bad = page < 0;
        return page < 0 ? static_cast<int>(g.a.batch.pages) : static_cast<int>(page);
    }

    __device__ void load_run(const CUtensorMap *boxes, const CUtensorMap *lines, int b, const PlanRun &run, int64_t &n_kv,
                             int &n_block) const {
        const int nbox = kBlockKeys / g.box;
        const int half = lane / nbox, box = lane - half * nbox;  // up to 16 boxes in each half
        const bool active = half < kHalves;
        const int lo = run.tile.lo, hi = run.tile.hi, none = static_cast<int>(g.a.batch.pages);
        int key = (run.tile.block0 + run.from) * kBlockKeys + box * g.box;
        bool bad = false;
        int page = active ? page_at(b, key, lo, hi, &bad) : none;
        for (int i = run.from; i < run.to; ++i) {
            const int now = page, now_key = key;
            const uint32_t bads = __ballot_sync(~0u, active && half == 0 && bad);
            if (bads && lane == 0) atomicOr(status(), kStatusBadIndex);
            key += kBlockKeys;
            bad = false;
            if (i + 1 < run.to && active) page = page_at(b, key, lo, hi, &bad);  // in flight while the block is loaded
            const int slot = now_key % g.a.batch.page_tokens;
            for (int plane = 0; plane < 2; ++plane, ++n_kv) {
                const int stage = static_cast<int>(n_kv % L::kStages);
                wait(&c->kv_empty[stage], ((n_kv / L::kStages) & 1) ^ 1);
                if (gave_up()) return;
                char *tile = smem + L::kKv + stage * L::kTile + half * kHalfBytes + box * g.box * 128;
                uint64_t *bar = &c->kv_full[stage];
                if (lane == 0) {
                    if (plane == 0) c->mask[n_block % kMaskSlots] = ~bads;
                    mbar_arrive_expect_tx(bar, L::kTile);
                }
                __syncwarp();
                if (g.a.batch.pages == 0) {
                    // no pool to read: the tile is zeroed in place of its loads
                    for (int e = lane; e < L::kTile / 16; e += 32)
                        reinterpret_cast<uint4 *>(smem + L::kKv + stage * L::kTile)[e] = make_uint4(0, 0, 0, 0);
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0)
                        asm volatile("mbarrier.complete_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)),
                                     "r"(static_cast<uint32_t>(L::kTile))
                                     : "memory");
                    continue;
                }
                // A box of values that is seen in part goes row by row: the rows that nobody sees as zeros.
                const bool cut = plane == 1 && active && now != none && (now_key < lo || now_key + g.box > hi);
                if (active && !cut) tma_load_5d(tile, boxes, bar, half * 64, slot, run.h, plane, now);
                uint32_t cuts = __ballot_sync(~0u, cut);
                while (cuts) {
                    const int l = __ffs(cuts) - 1;
                    cuts &= cuts - 1;
                    const int ck = __shfl_sync(~0u, now_key, l), cp = __shfl_sync(~0u, now, l), cs = __shfl_sync(~0u, slot, l);
                    const int ch = l / nbox, cb = l - ch * nbox;
                    char *to = smem + L::kKv + stage * L::kTile + ch * kHalfBytes + cb * g.box * 128;
                    for (int r = lane; r < g.box; r += 32)
                        tma_load_5d(to + r * 128, lines, bar, ch * 64, cs + r, run.h, 1, ck + r >= lo && ck + r < hi ? cp : none);
                }
            }
            ++n_block;
        }
    }

    // ---- warp 9: matrix instructions ----
    __device__ void mma_loop(uint32_t tmem) const {
        const int ksteps = (g.a.dim + 15) / 16;
        const uint32_t qk = mma_desc(kBf16Type, false, kBlockKeys);
        const uint32_t pv = mma_desc(kBf16Type, true, ksteps * 16);
        const uint32_t base = smem_u32(smem);
        int n_run = 0, n_q[2] = {0, 0}, n_p[2] = {0, 0};
        int64_t kv0 = 0;
        for (;;) {
            const RunInfo r = take_run(n_run);
            if (!r.blocks) break;
            const int n[2] = {r.pair ? r.blocks : (r.blocks + 1) / 2, r.pair ? r.blocks : r.blocks / 2};
            for (int t = 0; t <= r.pair; ++t) wait(&c->q_full[t], n_q[t]++ & 1);
            auto scores = [&](int s, int i) {
                const int block = r.pair ? i : 2 * i + s;
                const int64_t idx = kv0 + 2 * block;
                const int stage = static_cast<int>(idx % L::kStages);
                wait(&c->kv_full[stage], (idx / L::kStages) & 1);
                tmem_fence_after();
                if (lane == 0) {
                    const uint32_t qa = base + L::kQ + (r.pair ? s : 0) * L::kTile, ka = base + L::kKv + stage * L::kTile;
                    for (int e = 0; e < ksteps; ++e) {
                        const uint32_t off = (e >> 2) * kHalfBytes + (e & 3) * 32;
                        mma_ss(tmem + s_at(s), smem_tile_desc(qa + off, 16, 1024), smem_tile_desc(ka + off, 16, 1024), qk, e > 0);
                    }
                    if (!r.pair || s == 1) mma_commit(&c->kv_empty[stage]);
                    if (r.pair ? i + 1 == n[s] : block + 1 == r.blocks) mma_commit(&c->q_empty[r.pair ? s : 0]);
                    mma_commit(&c->s_full[s]);
                }
                __syncwarp();
            };
            auto values = [&](int s, int i) {
                const int block = r.pair ? i : 2 * i + s;
                const int64_t idx = kv0 + 2 * block + 1;
                const int stage = static_cast<int>(idx % L::kStages);
                wait(&c->kv_full[stage], (idx / L::kStages) & 1);
                wait(&c->p_full[s], n_p[s]++ & 1);
                tmem_fence_after();
                if (lane == 0) {
                    const uint32_t va = base + L::kKv + stage * L::kTile;
                    for (int e = 0; e < kBlockKeys / 16; ++e)
                        mma_ts(tmem + o_at(s), tmem + s_at(s) + e * 8, smem_tile_desc(va + e * 2048, kHalfBytes, 1024), pv,
                               i > 0 || e > 0);
                    if (!r.pair || s == 1) mma_commit(&c->kv_empty[stage]);
                    if (i + 1 == n[s]) mma_commit(&c->o_full[s]);
                }
                __syncwarp();
            };
            scores(0, 0);
            if (n[1]) scores(1, 0);
            for (int i = 0; i < n[0]; ++i) {
                for (int s = 0; s < 2; ++s) {
                    if (i >= n[s]) continue;
                    values(s, i);
                    if (i + 1 < n[s]) scores(s, i + 1);
                }
            }
            kv0 += 2 * r.blocks;
        }
        if (gave_up()) {
            // instructions may be in flight whose end nobody has seen: tensor memory stays ours until then
            if (lane == 0) {
                mma_commit(&c->drain);
                mbar_wait_bounded(&c->drain, 0, g.budget);
            }
            __syncwarp();
        }
    }

    // ---- warps 10, 11: queries ----
    __device__ void query_loop(int t) const {
        constexpr int kChunks = DP / 8;
        const PagedAttentionArgs &a = g.a;
        const T *q = static_cast<const T *>(a.q);
        int n_run = 0, n_q[2] = {0, 0};
        for (;;) {
            const RunInfo r = take_run(n_run);
            if (!r.blocks) break;
            for (int half = 0; half <= r.pair; ++half) {
                wait(&c->q_empty[half], (n_q[half]++ & 1) ^ 1);
                const int left = r.rows - half * kStreamRows;
                const int todo = (left < kStreamRows ? left : kStreamRows) * kChunks;
                char *tile = smem + L::kQ + half * L::kTile;
#pragma unroll 4
                for (int e = t; e < todo; e += 64) {
                    const int row = e / kChunks, chunk = e % kChunks;
                    const int at = r.r0 + half * kStreamRows + row;
                    const int token = at / g.shape.group, head = r.h * g.shape.group + at - token * g.shape.group;
                    uint4 v = make_uint4(0, 0, 0, 0);
                    if (chunk * 8 < a.dim)
                        v = *reinterpret_cast<const uint4 *>(q + (r.q0 + token) * a.q_st + head * a.q_sh + chunk * 8);
                    v.x ^= g.negate, v.y ^= g.negate, v.z ^= g.negate, v.w ^= g.negate;
                    *reinterpret_cast<uint4 *>(tile + (chunk / 8) * kHalfBytes + row * 128 + ((chunk ^ row) & 7) * 16) = v;
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&c->q_full[half]);
            }
        }
        if (a.fill_tail) {
            // rows of no sequence
            const int n = a.batch.seqs;
            const int head = n ? plan_clamp(a.batch.starts.at(0), 0, a.rows) : static_cast<int>(a.rows);
            const int tail = n ? plan_clamp(a.batch.starts.at(n), head, a.rows) : static_cast<int>(a.rows);
            const int64_t rows = head + a.rows - tail, per = a.q_heads * static_cast<int64_t>(a.dim);
            for (int64_t i = blockIdx.x * 64 + t; i < rows * per; i += gridDim.x * 64) {
                const int64_t k = i / per, e = i - k * per, row = k < head ? k : tail + (k - head);
                static_cast<T *>(a.out)[row * a.o_st + e / a.dim * a.o_sh + e % a.dim] = from_f32<T>(0.f);
                if (a.lse && e % a.dim == 0) a.lse[row * a.q_heads + e / a.dim] = -INFINITY;
            }
        }
    }

    // ---- warps 0-7: softmax ----
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
        uint32_t r;
        if constexpr (kBf16Type) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
        else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
        return r;
    }

    __device__ void softmax_loop(uint32_t tmem, int s) const {
        const PagedAttentionArgs &a = g.a;
        const int warp = (threadIdx.x >> 5) & 3, row = warp * 32 + lane;
        const uint32_t lanes = static_cast<uint32_t>(warp * 32) << 16;
        const uint32_t ts = tmem + s_at(s) + lanes, to = tmem + o_at(s) + lanes;
        const float scale = g.scale_log2;
        int n_run = 0, n_s = 0, n_o = 0, n_block = 0, n_join = 0;
        for (;;) {
            const RunInfo r = take_run(n_run);
            if (!r.blocks) break;
            const int steps = r.pair ? r.blocks : (r.blocks + 1 - s) / 2;
            const int mine = r.pair ? s * kStreamRows + row : row;  // row of the tile
            const bool live = mine < r.rows;
            const bool work = __any_sync(~0u, live);
            const int token = (r.r0 + mine) / g.shape.group;
            int lo = 0, hi = 1 << 30;  // keys that the row sees
            if (live) {
                const int at = r.first + token;
                hi = a.causal && at + 1 < r.end ? at + 1 : r.end;
                if (a.window > 0) lo = at + 1 - g.shape.window;
            }
            float m = -INFINITY, ref = 0.f, sum = 0.f;  // m = ref * scale
            for (int i = 0; i < steps; ++i) {
                const int block = r.pair ? i : 2 * i + s;
                const int key0 = r.key0 + block * kBlockKeys;
                wait(&c->s_full[s], n_s++ & 1);
                tmem_fence_after();
                if (work) {
                    uint32_t x[4][32];
#pragma unroll
                    for (int j = 0; j < 4; ++j) tmem_ld32(ts + j * 32, x[j]);
                    tmem_wait_ld();
                    const uint32_t boxes = c->mask[(n_block + block) % kMaskSlots];
                    if (__any_sync(~0u, live && (hi < key0 + kBlockKeys || lo > key0)) || boxes != ~0u) {
                        const int up = hi - key0, down = lo - key0, shift = __ffs(g.box) - 1;
#pragma unroll
                        for (int j = 0; j < 128; ++j)
                            if (j >= up || j < down || !(boxes >> (j >> shift) & 1)) x[j / 32][j % 32] = 0xff800000u;
                    }
                    float top = __uint_as_float(x[0][0]);
#pragma unroll
                    for (int j = 1; j < 128; ++j) top = fmaxf(top, __uint_as_float(x[j / 32][j % 32]));
                    // m, a reference in units of log2
                    const float next = top * scale;
                    const bool move = next > m + kRescale || (m == -INFINITY && next > m);
                    const float was = m;
                    if (move) m = next, ref = top;
                    float less = m == -INFINITY ? 0.f : -m, times = scale;
                    // x * scale - m is off by what m was rounded by, the same for the whole row, so it cancels;
                    // where it could pass 1 (the lowest value of a type as a score) the reference comes off first.
                    if (__any_sync(~0u, live && fabsf(m) > 0x1p24f && m != -INFINITY)) {
                        const float off = m == -INFINITY ? 0.f : ref;
#pragma unroll
                        for (int j = 0; j < 128; ++j)
                            x[j / 32][j % 32] = __float_as_uint((__uint_as_float(x[j / 32][j % 32]) - off) * scale);
                        less = 0.f;
                        times = 1.f;
                    }
                    float add = 0.f;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        uint32_t p[16];
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const float u = exp2_approx(fmaf(__uint_as_float(x[j][2 * e]), times, less));
                            const float v = exp2_approx(fmaf(__uint_as_float(x[j][2 * e + 1]), times, less));
                            add += u + v;
                            p[e] = pack(u, v);
                        }
                        tmem_st16(ts + j * 16, p);
                    }
                    if (i > 0 && __any_sync(~0u, move && live)) {
                        const float keep = move ? exp2_approx(was - m) : 1.f;
                        sum *= keep;
                        for (int j = 0; j < a.dim; j += 16) {
                            uint32_t o[16];
                            tmem_ld16(to + j, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
                            tmem_st16(to + j, o);
                        }
                    }
                    sum += add;
                    tmem_wait_st();
                }
                tmem_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&c->p_full[s]);
            }
            n_block += r.blocks;
            if (steps) {
                wait(&c->o_full[s], n_o++ & 1);
                tmem_fence_after();
            }
            if (!r.pair) {
                if (s == 1) {
                    c->join[row][0] = m;
                    c->join[row][1] = sum;
                    tmem_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&c->join_full);
                } else {
                    wait(&c->join_full, n_join & 1);
                }
            }
            if (work && (r.pair || s == 0)) {
                tmem_fence_after();
                float k0 = 1.f, k1 = 0.f;
                const bool both = !r.pair && r.blocks > 1;
                if (both) {
                    const float m1 = c->join[row][0], all = fmaxf(m, m1), ref = all == -INFINITY ? 0.f : all;
                    k0 = exp2_approx(m - ref);
                    k1 = exp2_approx(m1 - ref);
                    sum = sum * k0 + c->join[row][1] * k1;
                    m = all;
                }
                const int64_t q_row = r.q0 + token;
                const int head = r.h * g.shape.group + (r.r0 + mine - token * g.shape.group);
                char *slot = static_cast<char *>(a.workspace) + parts_bytes(g.ctas) + (2 * blockIdx.x + r.part) * slot_bytes(DP);
                T *out = static_cast<T *>(a.out) + q_row * a.o_st + head * a.o_sh;
                if (r.part < 0) {
                    const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;
                    k0 *= inv;
                    k1 *= inv;
                }
                for (int j = 0; j < a.dim; j += 16) {
                    uint32_t o[16];
                    tmem_ld16(to + j, o);
                    tmem_wait_ld();
                    float f[16];
#pragma unroll
                    for (int e = 0; e < 16; ++e) f[e] = __uint_as_float(o[e]) * k0;
                    if (both) {
                        tmem_ld16(tmem + o_at(1) + lanes + j, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 16; ++e) f[e] = fmaf(__uint_as_float(o[e]), k1, f[e]);
                    }
                    if (sum == 0.f) {
#pragma unroll
                        for (int e = 0; e < 16; ++e) f[e] = 0.f;
                    }
                    if (!live) continue;
                    if (r.part < 0) {
#pragma unroll
                        for (int e = 0; e < 16; e += 8)
                            if (j + e < a.dim)
                                *reinterpret_cast<uint4 *>(out + j + e) =
                                    make_uint4(pack(f[e], f[e + 1]), pack(f[e + 2], f[e + 3]), pack(f[e + 4], f[e + 5]),
                                               pack(f[e + 6], f[e + 7]));
                    } else {
                        float *o32 = reinterpret_cast<float *>(slot) + mine * DP + j;
#pragma unroll
                        for (int e = 0; e < 16; e += 4) *reinterpret_cast<float4 *>(o32 + e) = make_float4(f[e], f[e + 1], f[e + 2], f[e + 3]);
                    }
                }
                if (live && r.part >= 0)
                    reinterpret_cast<float2 *>(slot + static_cast<size_t>(kTileRows) * DP * 4)[mine] = make_float2(m, sum);
                if (live && r.part < 0 && a.lse)
                    a.lse[q_row * a.q_heads + head] = sum == 0.f ? -INFINITY : m * 0.6931471805599453f + logf(sum);
                tmem_fence_before();
            }
            if (!r.pair) {
                // stream 1's output has been read before its next weights can overwrite it
                if (s == 0) {
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&c->join_empty);
                } else {
                    wait(&c->join_empty, n_join & 1);
                }
                ++n_join;
            }
        }
    }
};

template <int DP, typename T>
__global__ void __launch_bounds__(kThreads, 1)
    paged_attention_kernel(const __grid_constant__ KernelArgs g, const __grid_constant__ CUtensorMap boxes,
                           const __grid_constant__ CUtensorMap lines) {
    using K = Kernel<DP, T>;
    extern __shared__ __align__(1024) char raw[];
    typename K::C *c = reinterpret_cast<typename K::C *>(raw + K::L::kControl);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    K k{g, raw, c, lane};
    if (warp == 9) {
        tmem_alloc(&c->tmem, 512);
    } else if (warp == 8 && lane == 0) {
        c->dead = 0;
        for (int i = 0; i < K::L::kStages; ++i) {
            mbar_init(&c->kv_full[i], 1);
            mbar_init(&c->kv_empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&c->q_full[i], 2);
            mbar_init(&c->q_empty[i], 1);
            mbar_init(&c->s_full[i], 1);
            mbar_init(&c->p_full[i], 4);
            mbar_init(&c->o_full[i], 1);
        }
        mbar_init(&c->join_full, 4);
        mbar_init(&c->join_empty, 4);
        mbar_init(&c->drain, 1);
        for (int i = 0; i < kRunSlots; ++i) {
            mbar_init(&c->run_full[i], 1);
            mbar_init(&c->run_empty[i], 11);  // warps 0-7 and 9-11
        }
        fence_proxy_async_smem();
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        if (g.a.batch.pages) {
            tma_prefetch_map(&boxes);
            tma_prefetch_map(&lines);
        }
    }
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    const uint32_t tmem = c->tmem;
    pdl_launch();
    if (warp < 8) k.softmax_loop(tmem, warp >> 2);
    else if (warp == 8) k.load_loop(&boxes, &lines);
    else if (warp == 9) k.mma_loop(tmem);
    else k.query_loop(threadIdx.x - 320);
    tmem_fence_before();
    __syncthreads();
    if (warp == 9) tmem_free(tmem, 512);
}

// Joins the tiles that several CTAs share: block (c, y) the one that begins in
// CTA c and does not end there, the y-th part of its rows.
constexpr int kJoinThreads = 128;
template <int DP, typename T>
__global__ void __launch_bounds__(kJoinThreads) join_parts_kernel(const __grid_constant__ KernelArgs g) {
    pdl_wait();
    const PagedAttentionArgs &a = g.a;
    const Part p = static_cast<const Part *>(a.workspace)[blockIdx.x];
    if (p.pieces < 2) return;
    constexpr int kLanes = DP / 4;
    const int e = threadIdx.x % kLanes * 4;
    const char *slots = static_cast<const char *>(a.workspace) + parts_bytes(g.ctas);
    for (int r = blockIdx.y * (kJoinThreads / kLanes) + threadIdx.x / kLanes; r < p.rows; r += gridDim.y * (kJoinThreads / kLanes)) {
        float m = -INFINITY, sum = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int i = 0; i < p.pieces; ++i) {
            const char *slot = slots + (2 * static_cast<size_t>(blockIdx.x + i) + (i == 0)) * slot_bytes(DP);
            const float2 ms = reinterpret_cast<const float2 *>(slot + static_cast<size_t>(kTileRows) * DP * 4)[r];
            const float4 v = *reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(slot) + r * DP + e);
            const float all = fmaxf(m, ms.x), ref = all == -INFINITY ? 0.f : all;
            const float k0 = exp2_approx(m - ref), k1 = exp2_approx(ms.x - ref);
            m = all;
            sum = sum * k0 + ms.y * k1;
            o.x = o.x * k0 + v.x * k1;
            o.y = o.y * k0 + v.y * k1;
            o.z = o.z * k0 + v.z * k1;
            o.w = o.w * k0 + v.w * k1;
        }
        const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;
        const int token = (p.r0 + r) / g.shape.group, head = p.h * g.shape.group + p.r0 + r - token * g.shape.group;
        const int64_t row = p.q0 + token;
        if (e < a.dim) {
            T *out = static_cast<T *>(a.out) + row * a.o_st + head * a.o_sh + e;
            const uint2 v = make_uint2(Kernel<DP, T>::pack(o.x * inv, o.y * inv), Kernel<DP, T>::pack(o.z * inv, o.w * inv));
            *reinterpret_cast<uint2 *>(out) = v;
        }
        if (a.lse && e == 0) a.lse[row * a.q_heads + head] = sum == 0.f ? -INFINITY : m * 0.6931471805599453f + logf(sum);
    }
}

// CTAs that a call is given: no more than its units can be, and one an SM.
int plan_ctas(const PagedAttentionArgs &a, int sms) {
    const int64_t group = a.q_heads / a.kv_heads;
    const int64_t tokens = a.batch.table_width * a.batch.page_tokens;
    const int64_t blocks = tokens > kBlockKeys ? (tokens + kBlockKeys - 1) / kBlockKeys : 1;
    const int64_t seqs = a.batch.seqs < a.rows ? a.batch.seqs : a.rows;
    const int64_t tiles = (seqs + a.rows * group / kTileRows) * a.kv_heads;
    const int64_t units = blocks > sms || tiles > sms ? sms : tiles * blocks;
    return static_cast<int>(units < 1 ? 1 : units < sms ? units : sms);
}

using EncodeFn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                              const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// The pool as (element, slot, key head, plane, page), in boxes of `tokens` slots of 64 elements.
int encode_pool(const PagedAttentionArgs &a, int dtype, int tokens, CUtensorMap *map) {
    static const auto encode = reinterpret_cast<EncodeFn>(gpu::driver_symbol("cuTensorMapEncodeTiled"));
    if (!encode) return cudaErrorNotSupported;
    const cuuint64_t dims[5] = {static_cast<cuuint64_t>(a.dim), static_cast<cuuint64_t>(a.batch.page_tokens),
                                static_cast<cuuint64_t>(a.kv_heads), 2, static_cast<cuuint64_t>(a.batch.pages)};
    const cuuint64_t strides[4] = {static_cast<cuuint64_t>(a.pool_token) * 2, static_cast<cuuint64_t>(a.pool_head) * 2,
                                   static_cast<cuuint64_t>(a.pool_plane) * 2, static_cast<cuuint64_t>(a.pool_page) * 2};
    const cuuint32_t box[5] = {64, static_cast<cuuint32_t>(tokens), 1, 1, 1}, one[5] = {1, 1, 1, 1, 1};
    const CUresult e = encode(map, dtype == kBf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 5,
                              const_cast<void *>(a.pool), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return e == CUDA_SUCCESS ? 0 : static_cast<int>(cudaErrorInvalidValue);
}

template <int DP, typename T>
int launch(const KernelArgs &g, int dtype, int device, bool join, cudaStream_t st) {
    using K = Kernel<DP, T>;
    constexpr int smem = K::L::kControl + static_cast<int>(sizeof(typename K::C));
    static_assert(smem <= 227 * 1024, "shared memory of one CTA");
    CUtensorMap boxes, lines;
    std::memset(&boxes, 0, sizeof boxes);
    std::memset(&lines, 0, sizeof lines);
    if (g.a.batch.pages) {
        int e = encode_pool(g.a, dtype, g.box, &boxes);
        if (!e) e = encode_pool(g.a, dtype, 1, &lines);
        if (e) return e;
    }
    static std::atomic<uint64_t> configured{0};  // devices
    cudaError_t e = cudaSuccess;
    if (device > 63 || !(configured.load(std::memory_order_acquire) >> device & 1)) {
        e = cudaFuncSetAttribute(paged_attention_kernel<DP, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return static_cast<int>(e);
        if (device <= 63) configured.fetch_or(1ull << device, std::memory_order_release);
    }
    paged_attention_kernel<DP, T><<<g.ctas, kThreads, smem, st>>>(g, boxes, lines);
    note_launch();
    e = cudaGetLastError();
    if (e != cudaSuccess || !join) return static_cast<int>(e);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(g.ctas, 8);
    cfg.blockDim = dim3(kJoinThreads);
    cfg.stream = st;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, join_parts_kernel<DP, T>, g);
    note_launch();
    return static_cast<int>(e);
}

}  // namespace

size_t paged_attention_workspace(int64_t rows, int q_heads, int kv_heads, int dim, int seqs, int device) {
    (void)rows, (void)q_heads, (void)kv_heads, (void)seqs;
    const int sms = sm_count(device);
    return parts_bytes(sms) + 2 * static_cast<size_t>(sms) * slot_bytes(dim <= 64 ? 64 : 128);
}

int paged_attention(const PagedAttentionArgs &a, int dtype, int device, void *stream) {
    if (a.rows <= 0 || a.q_heads <= 0) return 0;
    if (a.dim <= 0 || a.dim % 8 || a.dim > 128 || a.kv_heads <= 0 || a.q_heads % a.kv_heads || a.rows > 0x7fffffff ||
        a.batch.page_tokens <= 0 || a.batch.page_tokens % 8 || a.batch.pages > 0x7fffffff || (dtype != kBf16 && dtype != kFp16))
        return cudaErrorInvalidValue;
    DeviceScope on(device);
    if (on.error()) return on.error();
    KernelArgs g;
    g.a = a;
    const int64_t tokens = a.batch.pages > 0 ? a.batch.table_width * a.batch.page_tokens : 0;
    g.shape.group = a.q_heads / a.kv_heads;
    g.shape.kv_heads = a.kv_heads;
    g.shape.causal = a.causal;
    g.shape.window = plan_clamp(a.window, 0, kMostTokens);
    g.shape.rows = static_cast<int>(a.rows);
    g.shape.tokens = plan_clamp(tokens, 0, kMostTokens);
    // a scale of zero would make NaN of a masked score; this one gives every seen score the same weight
    g.scale_log2 = fmaxf(fabsf(a.scale) * 1.4426950408889634f, 1e-30f);
    g.negate = a.scale < 0.f ? 0x80008000u : 0u;
    g.box = a.batch.page_tokens & -a.batch.page_tokens;
    if (g.box > kBlockKeys) g.box = kBlockKeys;
    g.budget = wait_budget_ns();
    g.ctas = plan_ctas(a, sm_count(device));
    if (!a.workspace || a.workspace_bytes < parts_bytes(g.ctas) + 2 * g.ctas * slot_bytes(a.dim <= 64 ? 64 : 128))
        return cudaErrorInvalidValue;
    const bool join = g.ctas > 1 && tokens > kBlockKeys;  // a tile of one block is never shared
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (a.dim <= 64)
        return dtype == kBf16 ? launch<64, __nv_bfloat16>(g, dtype, device, join, st) : launch<64, __half>(g, dtype, device, join, st);
    return dtype == kBf16 ? launch<128, __nv_bfloat16>(g, dtype, device, join, st) : launch<128, __half>(g, dtype, device, join, st);
}

}  // namespace kern
}  // namespace mpcomm
