// Attention of a ragged batch of new tokens over a paged KV cache.
//
//     out[t, h] = sum_p w_p v_p / sum_p w_p,   w_p = exp(scale * q[t, h] . k_p - m)
//
// over the keys p that row t sees; m is a reference near the row's largest
// score, and a row that sees no key gives zeros.
//
// One persistent CTA an SM goes through its part of the plan
// (attention_plan.h) in one pass over the keys. Two streams of 128 rows run
// against each other: stream s has two buffers of scores (128 x 64, fp32) and
// the output O_s (128 x dim, fp32) in tensor memory, and the weights, 16-bit, in
// place of their scores. While a stream's softmax works in one buffer the tensor
// core fills the other and multiplies the other stream's weights. Each stream
// has its own warp that issues its matrix instructions: the queue of the tensor
// core is short, and one warp for both would wait in it with one stream's while
// the other's weights are ready. A tile of more than 128 rows gives each stream
// half of its rows, over the same keys. A smaller one (single tokens) gives both streams
// the same rows and every second block of keys, and they are joined at the
// end, so the loads never wait for one stream's softmax.
//
//   warps 0-3, 4-7  the softmax of stream 0, 1: a thread has a row
//   warp 8          walks the plan, loads K blocks by TMA (a page, or the
//                   part of one that lies in the block, a box)
//   warps 9, 10     issue the matrix instructions of stream 0, 1
//   warp 11         loads the queries and V blocks
//
// Weights are rounded to the cache's type for the second product, whose two
// operands have one type (outputs in bf16 are off by 0.0023 of their norm, by
// 0.0017 through their own rounding alone); sums, maxima, scores and outputs
// are 32-bit. m only moves when a score passes the one it was taken from by
// 2^8 (kRescale), so O_s is hardly ever rescaled. In bf16 m is that score and
// weights reach 2^8. In fp16 weights below 2^-14 have a step of 2^-24, so m is taken 2^7 lower
// (kDepth): weights reach 2^15 of the 65,504 that the type holds, and each is
// off by at most 2^-25 where the largest is at least 2^7, 2^-32 of it. (With m
// at the score, 8,191 keys 25.2 powers of two below one other lost half of
// their share.) Outputs below 2^-14 have fp16's step of 2^-24 in any case.
//
// Keys that no row of a tile sees (behind a sequence, before a window, on a
// page that is none) are read as zeros: their boxes are put outside the pool,
// where the TMA fills zeros. So nothing that lies there reaches a result, and
// a masked score is replaced, never added to.
//
// What bounds it: single tokens, reading K and V (32 sequences of 4,096, 537
// MB: 97 us, 5.5 TB/s; the products are done for 128 rows, most of them
// unused, and keep the tensor pipe busy for a third of that). Chunks, the chain
// of a half block's scores, exponentials and products, of which two overlap:
// 1,024 tokens over 8,192 take 133 us (971 TFLOP/s), 4,096 over 16,384 take
// 798 alone, after a pause (1.21 PFLOP/s), and 932 back to back (1.03; a
// library product reaches 1.66 in a burst, 1.38 when it runs for seconds).
#include <atomic>
#include <cstring>
#include <mutex>

#include "cuda/gpu.h"
#include "kernels/attention_plan.h"
#include "kernels/kv.cuh"
#include "kernels/umma.cuh"

namespace mpcomm {
namespace kern {
namespace {

constexpr int kThreads = 384;
constexpr int kHalfKeys = kBlockKeys / 2;  // keys of a buffer of scores
// Registers a thread: at launch, then of the softmax's warps, which hold a row
// of scores, and of the others. What is taken is no more than what is given.
constexpr int kRegsLaunch = 168, kRegsSoftmax = 200, kRegsOther = 104;
static_assert(256 * kRegsSoftmax + 128 * kRegsOther <= kThreads * kRegsLaunch, "registers of a CTA");
constexpr int kRunSlots = 4;
// Tiles of a sequence that one lane counts while the others count theirs; longer ones are counted by the warp, one
// after the other. 64 prompts of 512 (8 tiles each) take 317 us, by the warp 332; 512 of 200 170, by the warp 278; one
// of 64 tiles 798 to 802 by a lane, 798 by the warp.
constexpr int kFewTiles = 16;
constexpr int kMaskSlots = 16;  // blocks whose masks are kept: more than are ever in flight
constexpr float kRescale = 8.f;
constexpr float kFp16Depth = 7.f;

__device__ uint32_t g_attention_status;

// What the plan's warp tells the others of a run.
struct RunInfo {
    int blocks;    // 0: no more runs
    int tokens;    // of the tile
    int t0;        // the tile's first token among its sequence's new ones
    int q0;        // the sequence's first row of the query tensor
    int part;      // of the query heads
    int key0;      // first key of the run's first block
    int lo, hi;    // keys that some row of the tile sees
    int first;     // position of the sequence's first new token
    int end;       // keys of the sequence
    int seq;
    int slot;      // -1: the run is the whole tile; else its slot in the workspace
};

template <int DP>
struct Layout {
    static constexpr int kTile = kStreamRows * DP * 2;  // 128 rows of DP 16-bit elements
    // Tiles of K and of V. A wait tells a tile's phase from the next one only, so whoever waits for a tile's n-th use
    // must have seen the one before: K and V are rings of their own, each filled by one warp, and both streams go
    // through every tile, a stream that has no use for one passes it.
    static constexpr int kKeys = DP == 128 ? 2 : 4, kValues = DP == 128 ? 3 : 6;
    static constexpr int kStages = kKeys + kValues;
    static constexpr int kQ = 0;
    static constexpr int kKv = 2 * kTile;
    static constexpr int kControl = kKv + kStages * kTile;
};

template <int STAGES>
struct Control {
    uint64_t kv_full[STAGES], kv_empty[STAGES];
    uint64_t q_full[2], q_empty[2];
    uint64_t s_full[2][2], p_full[2][2], o_step[2], o_full[2];  // o_step: after each half block, o_full: after a run's last
    uint64_t turn[2][4];  // of a warp's exponentials
    uint64_t join_full, join_empty, drain[2];
    uint64_t run_full[kRunSlots], run_empty[kRunSlots];
    uint32_t mask[kMaskSlots];  // good boxes of a block
    RunInfo run[kRunSlots];
    float join[kStreamRows][2];  // m and sum of stream 1's rows, for stream 0
    uint32_t tmem;
    uint32_t dead;  // a wait ran out: nothing is waited for any more
};

struct Shared {  // a tile whose blocks several CTAs share, from its first CTA on
    int pieces;
    int q0, t0, tokens, part;
};

// Bytes of a workspace: what is shared, then two slots a CTA of two streams' rows each.
__host__ __device__ constexpr size_t shared_bytes(int ctas) { return (sizeof(Shared) * ctas + 255) / 256 * 256; }
__host__ __device__ constexpr size_t slot_bytes(int dp) { return static_cast<size_t>(2 * kStreamRows) * (dp + 2) * 4; }

// How the pool lies in memory for the TMA. (page, plane, key head) is one
// index in units of the greatest stride that divides all three, so that a box
// of whole rows has dimensions to spare for its order in shared memory: with
// heads of 64 or 128 elements one box is (64 elements, 8 slots, halves,
// groups of 8 slots) and lands as groups of 8 rows, half by half. Other heads
// end inside 64 elements, where the TMA has to fill up with zeros: their
// boxes are (64 elements, slots), each half by itself.
struct PoolView {
    int page, plane, head;  // strides of the index
    int none;               // an index behind the pool: reads as zeros
    int whole;              // a box has both halves
    int group_bytes, half_bytes;  // in shared memory: distance of 8-row groups, of halves
};

struct KernelArgs {
    PagedAttentionArgs a;
    PlanShape shape;
    PoolView pool;
    FastDiv page_tokens, each;  // each: parts of a key head
    int group;         // query heads of a key head
    float scale_log2;  // |scale| * log2(e)
    int ctas;
    int box;  // tokens of a full box
    int box_shift;  // a block has 2^box_shift boxes
    uint32_t *gave_up;  // host memory: where a kernel without a status word says that a wait ran out
    uint64_t budget;  // of a wait, ns
    uint32_t tries;   // the same, in tries of a microsecond
};

template <int DP, typename T>
struct Kernel {
    using L = Layout<DP>;
    using C = Control<L::kStages>;
    static constexpr int kHalves = DP / 64;
    static constexpr int kHalfBytes = kStreamRows * 128;
    // columns of tensor memory: scores and weights, output of a stream
    static __device__ __forceinline__ uint32_t s_at(int s, int half) { return s * 128 + half * 64; }
    static __device__ __forceinline__ uint32_t o_at(int s) { return 256 + s * DP; }
    static constexpr bool kBf16Type = std::is_same_v<T, __nv_bfloat16>;
    // powers of two that a row's reference lies below the score it was taken from
    static constexpr float kDepth = kBf16Type ? 0.f : kFp16Depth;
    static_assert(kBf16Type || kRescale + kFp16Depth < 16.f, "weights in fp16");

    const KernelArgs &g;
    char *smem;
    C *c;
    int lane;

    __device__ uint32_t *status() const { return g.a.status ? g.a.status : &g_attention_status; }

    __device__ __noinline__ void ran_out() const {
        if (g.a.status) atomicOr(g.a.status, kStatusLoadTimeout);
        else *static_cast<volatile uint32_t *>(g.gave_up) = 1;
    }

    // Waits for a phase; gives up after the budget (a try waits for about a microsecond), and at once when any wait
    // of the CTA has given up.
    __device__ __forceinline__ void wait(uint64_t *bar, uint32_t parity) const {
        uint32_t left = g.tries;
        while (__builtin_expect(!mbar_try_wait_1us(bar, parity), 0)) {
            volatile uint32_t *dead = &c->dead;
            if (*dead) break;
            if (--left == 0) {
                *dead = 1;
                ran_out();
            }
        }
    }

    // A value that all lanes have, in a form that the compiler knows to be the same for all: control flow that
    // hangs on it stays uniform, and matrix instructions take their operands without a detour per lane.
    static __device__ __forceinline__ int same(int v) { return __reduce_or_sync(~0u, v); }

    // Whether some wait has given up, the same for a whole warp.
    __device__ __forceinline__ bool gave_up() const {
        return __any_sync(~0u, *const_cast<volatile uint32_t *>(&c->dead) != 0);
    }

    // The next run, read by a whole warp; the slot is given back at once.
    __device__ __forceinline__ RunInfo take_run(int &n) const {
        const int slot = n % kRunSlots;
        wait(&c->run_full[slot], (n / kRunSlots) & 1);
        RunInfo r = c->run[slot];
        int *fields = reinterpret_cast<int *>(&r);
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(RunInfo) / sizeof(int)); ++i) fields[i] = same(fields[i]);
        if (gave_up()) r.blocks = 0;
        if (lane == 0) mbar_arrive(&c->run_empty[slot]);
        ++n;
        return r;
    }

    // ---- warp 8: the plan, and K ----
    __device__ void plan_loop(const CUtensorMap *boxes, const CUtensorMap *lines) const {
        const KvBatch &k = g.a.batch;
        const PlanShape &s = g.shape;
        auto sequence = [&](int b) { return plan_seq(s, k.starts.at(b), k.starts.at(b + 1), k.lens.at(b)); };
        // Units of a part of each lane's sequence. A sequence of many tiles is counted by the whole warp.
        auto count = [&](int b) {
            PlanSeq q;
            if (b < k.seqs) q = sequence(b);
            if (q.cut && blockIdx.x == 0) atomicOr(status(), kStatusBadIndex);
            int64_t own = q.tiles <= kFewTiles ? plan_part_units(s, q) : 0;
            for (uint32_t many = __ballot_sync(~0u, q.tiles > kFewTiles); many; many &= many - 1) {
                const int l = __ffs(many) - 1;
                PlanSeq o;
                o.new_tokens = __shfl_sync(~0u, q.new_tokens, l);
                o.first = __shfl_sync(~0u, q.first, l);
                o.end = __shfl_sync(~0u, q.end, l);
                o.tiles = __shfl_sync(~0u, q.tiles, l);
                int64_t n = plan_part_units(s, o, lane, 32);
#pragma unroll
                for (int i = 16; i; i >>= 1) n += __shfl_xor_sync(~0u, n, i);
                if (lane == l) own = n;
            }
            return own;
        };
        auto scan = [&](int64_t n) {
#pragma unroll
            for (int i = 1; i < 32; i <<= 1) {
                const int64_t up = __shfl_up_sync(~0u, n, i);
                if (lane >= i) n += up;
            }
            return n;
        };
        // The ring's memory, which nothing is loaded into yet, keeps the counts of a batch of more than a warp.
        int64_t *kept = reinterpret_cast<int64_t *>(smem + L::kKv);
        constexpr int kKept = L::kStages * L::kTile / 8;
        int64_t own = 0, units = 0;
        for (int b0 = 0; b0 < k.seqs; b0 += 32) {
            own = count(b0 + lane);
            units += own;
            if (k.seqs > 32 && b0 + lane < kKept) kept[b0 + lane] = own;
        }
        int64_t sum = scan(units);
        units = __shfl_sync(~0u, sum, 31) * s.parts;
        const int64_t share = plan_share(units, g.ctas);
        int64_t at = blockIdx.x * share;
        int64_t left = units - at < share ? units - at : share;
        Shared mine{0, 0, 0, 0, 0};
        int n_run = 0;
        int64_t n_block = 0;
        if (left > 0) {
            // the sequence that holds unit `at`
            int b = 0;
            for (int b0 = 0;; b0 += 32) {
                if (k.seqs > 32) {
                    own = b0 + lane < kKept ? (b0 + lane < k.seqs ? kept[b0 + lane] : 0) : count(b0 + lane);
                    sum = scan(own);
                }
                const uint32_t past = __ballot_sync(~0u, sum * s.parts > at);
                if (past) {
                    const int i = __ffs(past) - 1;
                    b = b0 + i;
                    own = __shfl_sync(~0u, own, i);
                    at -= (__shfl_sync(~0u, sum, i) - own) * s.parts;
                    break;
                }
                at -= __shfl_sync(~0u, sum, 31) * s.parts;
            }
            fence_proxy_async_smem();
            PlanSeq q = sequence(b);
            PlanCursor cur;
            cur.part = static_cast<int>(plan_div(at, own));
            at -= cur.part * own;
            for (;; cur.m += 32) {  // its tile
                const int blocks = cur.m + lane < q.tiles ? plan_tile(s, q, cur.m + lane).blocks : 0;
                sum = scan(blocks);
                const uint32_t past = __ballot_sync(~0u, sum > at);
                if (past || cur.m + 32 >= q.tiles) {
                    const int i = past ? __ffs(past) - 1 : 0;
                    cur.block = static_cast<int>(at - __shfl_sync(~0u, sum - blocks, i));
                    cur.m += i;
                    break;
                }
                at -= __shfl_sync(~0u, sum, 31);
            }
            while (left > 0) {
                PlanRun run;
                if (!cur.next(s, q, left, &run)) {
                    if (++b >= k.seqs) break;
                    q = sequence(b);
                    cur = PlanCursor();
                    continue;
                }
                left -= run.to - run.from;
                const bool whole = run.from == 0 && run.to == run.tile.blocks;
                RunInfo r;
                r.blocks = run.to - run.from;
                r.tokens = run.tile.tokens;
                r.t0 = run.m * 2 * s.tokens_stream;
                r.q0 = q.q0;
                r.part = run.part;
                r.key0 = (run.tile.block0 + run.from) * kBlockKeys;
                r.lo = run.tile.lo;
                r.hi = run.tile.hi;
                r.first = q.first;
                r.end = q.end;
                r.seq = b;
                r.slot = whole ? -1 : run.from == 0 ? 1 : 0;
                if (r.slot == 1) {
                    const int64_t rest = run.tile.blocks - run.to;
                    mine = Shared{static_cast<int>(1 + plan_div(rest + share - 1, share)), r.q0, r.t0, r.tokens, r.part};
                }
                const int slot = n_run % kRunSlots;
                wait(&c->run_empty[slot], ((n_run / kRunSlots) & 1) ^ 1);
                if (lane == 0) {
                    c->run[slot] = r;
                    mbar_arrive(&c->run_full[slot]);
                }
                ++n_run;
                if (!load_blocks<0>(boxes, lines, r, n_block)) break;
            }
        }
        const int slot = n_run % kRunSlots;
        wait(&c->run_empty[slot], ((n_run / kRunSlots) & 1) ^ 1);
        if (lane == 0) {
            c->run[slot].blocks = 0;
            mbar_arrive(&c->run_full[slot]);
            static_cast<Shared *>(g.a.workspace)[blockIdx.x] = mine;
        }
        drain_loads<0>(n_block);
    }

    // ---- warp 11: queries, and V ----
    __device__ void value_loop(const CUtensorMap *boxes, const CUtensorMap *lines, const CUtensorMap *queries) const {
        const int each = g.shape.parts / g.a.kv_heads, tokens = g.shape.tokens_stream;
        int n_run = 0, n_q[2] = {0, 0};
        int64_t n_block = 0;
        for (;;) {
            const RunInfo r = take_run(n_run);
            if (!r.blocks) break;
            const int head = g.each.div(r.part);
            for (int s = 0; s <= (r.tokens > tokens); ++s) {
                wait(&c->q_empty[s], (n_q[s] & 1) ^ 1);
                if (gave_up()) break;
                ++n_q[s];
                if (elect_one()) {
                    mbar_arrive_expect_tx(&c->q_full[s], tokens * g.shape.heads * 128 * kHalves);
                    for (int h = 0; h < kHalves; ++h)
                        tma_load_4d(smem + L::kQ + s * L::kTile + h * kHalfBytes, queries, &c->q_full[s], h * 64,
                                    (r.part - head * each) * g.shape.heads, head, r.q0 + r.t0 + s * tokens);
                }
                __syncwarp();
            }
            if (!load_blocks<1>(boxes, lines, r, n_block)) break;
        }
        drain_loads<1>(n_block);
        if (gave_up() && lane == 0)
            for (int s = 0; s < 2; ++s)
                if (n_q[s]) mbar_wait_bounded(&c->q_full[s], (n_q[s] - 1) & 1, g.budget / 8);
        if (g.a.fill_tail || g.a.lse) fill_tail();
    }

    // The rows of no sequence: zeros in an output that is to have them, -inf in log-sum-exps. A warp a row, in wide
    // stores (element by element, 4,096 rows of 32 x 128 behind 32 single tokens took 890 us, this 18).
    __device__ void fill_tail() const {
        const PagedAttentionArgs &a = g.a;
        const int n = a.batch.seqs;
        const int head = n ? plan_clamp(a.batch.starts.at(0), 0, a.rows) : static_cast<int>(a.rows);
        const int tail = n ? plan_clamp(a.batch.starts.at(n), head, a.rows) : static_cast<int>(a.rows);
        const int64_t rows = head + a.rows - tail;
        const int chunks = a.dim / 8, over = 32 / chunks, step = 32 - over * chunks;  // 16 bytes of a head a lane
        for (int64_t k = blockIdx.x; k < rows; k += gridDim.x) {
            const int64_t row = k < head ? k : tail + (k - head);
            int h = lane / chunks, c8 = lane - h * chunks;
            if (a.fill_tail)
                while (h < a.q_heads) {
                    *reinterpret_cast<uint4 *>(static_cast<T *>(a.out) + row * a.o_st + h * a.o_sh + c8 * 8) = make_uint4(0, 0, 0, 0);
                    h += over;
                    if ((c8 += step) >= chunks) c8 -= chunks, ++h;
                }
            if (a.lse)
                for (int i = lane; i < a.q_heads; i += 32) a.lse[row * a.q_heads + i] = -INFINITY;
        }
    }

    static constexpr int ring(int plane) { return plane ? L::kValues : L::kKeys; }
    static constexpr int ring_at(int plane) { return plane ? L::kKeys : 0; }

    // After a wait that ran out, loads may be in flight that nobody has waited
    // for: shared memory stays ours until they have landed. `next`: the
    // warp's next load.
    template <int PLANE>
    __device__ void drain_loads(int64_t next) const {
        constexpr int R = ring(PLANE);
        if (!gave_up() || lane) return;
        for (int64_t i = next - 1; i >= 0 && i >= next - R; --i)
            mbar_wait_bounded(&c->kv_full[ring_at(PLANE) + i % R], (i / R) & 1, g.budget / 8);
    }

    // The index of the page of key `key` on, g.pool.none where nobody sees the box or there is no page.
    __device__ __forceinline__ int place(const RunInfo &r, int head, int plane, int key, bool *bad) const {
        if (key >= r.hi || key + g.box <= r.lo) return g.pool.none;
        // key is below plan's end, so its column is in the table
        const int64_t page = g.a.batch.table.at(r.seq * g.a.batch.table_stride + g.page_tokens.div(key));
        *bad = page < 0 || page >= g.a.batch.pages;
        return *bad ? g.pool.none : static_cast<int>(page) * g.pool.page + plane * g.pool.plane + head * g.pool.head;
    }

    // Loads K or V of a run's blocks into its ring. False: a wait gave up.
    template <int PLANE>
    __device__ bool load_blocks(const CUtensorMap *boxes, const CUtensorMap *lines, const RunInfo &r, int64_t &n_block) const {
        const int nbox = 1 << g.box_shift, nhalf = g.pool.whole ? 1 : kHalves;
        const int half = lane >> g.box_shift, box = lane & (nbox - 1);  // up to 16 boxes in each half
        const bool active = half < nhalf;
        const int head = g.each.div(r.part), none = g.pool.none;
        const uint32_t at = box * (g.box / 8) * g.pool.group_bytes + half * g.pool.half_bytes;
        int key = r.key0 + box * g.box;
        bool bad = false;
        int index = active ? place(r, head, PLANE, key, &bad) : none;
        for (int i = 0; i < r.blocks; ++i, ++n_block) {
            const int now = index, now_key = key;
            const uint32_t bads = __ballot_sync(~0u, active && half == 0 && bad);
            if (PLANE == 0 && bads && lane == 0) atomicOr(status(), kStatusBadIndex);
            key += kBlockKeys;
            bad = false;
            if (i + 1 < r.blocks && active) index = place(r, head, PLANE, key, &bad);  // in flight while this block is loaded
            const int slot = now_key - g.page_tokens.div(now_key) * g.a.batch.page_tokens;
            const int stage = ring_at(PLANE) + static_cast<int>(n_block % ring(PLANE));
            wait(&c->kv_empty[stage], ((n_block / ring(PLANE)) & 1) ^ 1);
            if (gave_up()) return false;
            char *tile = smem + L::kKv + stage * L::kTile;
            uint64_t *bar = &c->kv_full[stage];
            if (lane == 0) {
                if (PLANE == 0) c->mask[n_block % kMaskSlots] = ~bads;
                mbar_arrive_expect_tx(bar, L::kTile);
            }
            __syncwarp();
            if (g.a.batch.pages == 0) {
                // no pool to read: the tile is zeroed in place of its loads
                for (int e = lane; e < L::kTile / 16; e += 32) reinterpret_cast<uint4 *>(tile)[e] = make_uint4(0, 0, 0, 0);
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0)
                    asm volatile("mbarrier.complete_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)),
                                 "r"(static_cast<uint32_t>(L::kTile))
                                 : "memory");
                continue;
            }
            // A box of values that is seen in part goes row by row: the rows that nobody sees as zeros.
            const bool cut = PLANE == 1 && active && now != none && (now_key < r.lo || now_key + g.box > r.hi);
            if (active && !cut) {
                if (g.pool.whole) tma_load_5d(tile + at, boxes, bar, 0, 0, 0, slot / 8, now);
                else tma_load_5d(tile + at, boxes, bar, half * 64, slot, 0, 0, now);
            }
            if (PLANE == 1) {
                uint32_t cuts = __ballot_sync(~0u, cut);
                while (cuts) {
                    const int l = __ffs(cuts) - 1;
                    cuts &= cuts - 1;
                    const int ck = __shfl_sync(~0u, now_key, l), ci = __shfl_sync(~0u, now, l), cs = __shfl_sync(~0u, slot, l);
                    const uint32_t to = __shfl_sync(~0u, at, l);
                    const int from = g.pool.whole ? 0 : l >> g.box_shift, rows = g.box * (g.pool.whole ? kHalves : 1);
                    for (int e = lane; e < rows; e += 32) {
                        const int h = e >> (7 - g.box_shift), row = e & (g.box - 1);
                        tma_load_5d(tile + to + h * g.pool.half_bytes + row / 8 * g.pool.group_bytes + row % 8 * 128, lines, bar,
                                    (from + h) * 64, cs + row, 0, 0, ck + row >= r.lo && ck + row < r.hi ? ci : none);
                    }
                }
            }
        }
        return true;
    }

    // ---- warps 9, 10: matrix instructions of a stream ----
    __device__ void mma_loop(uint32_t tmem, int s) const {
        const int ksteps = (g.a.dim + 15) / 16;
        const uint32_t qk = mma_desc(kBf16Type, false, kHalfKeys) | (g.a.scale < 0.f ? kMmaNegateA : 0u);
        const uint32_t pv = mma_desc(kBf16Type, true, ksteps * 16);
        const uint32_t base = smem_u32(smem);
        const uint32_t group = g.pool.group_bytes, halves = g.pool.half_bytes;
        const uint32_t to = tmem + o_at(s);
        int n_run = 0, n_q[2] = {0, 0}, n_p = 0;
        int k_stage = 0, k_phase = 0, v_stage = L::kKeys, v_phase = 0;  // of the next tile
        auto next_k = [&] {
            if (++k_stage == L::kKeys) k_stage = 0, k_phase ^= 1;
        };
        auto next_v = [&] {
            if (++v_stage == L::kStages) v_stage = L::kKeys, v_phase ^= 1;
        };
        auto pass_k = [&] {
            wait(&c->kv_full[k_stage], k_phase);
            if (lane == 0) mbar_arrive(&c->kv_empty[k_stage]);
            next_k();
        };
        auto pass_v = [&] {
            wait(&c->kv_full[v_stage], v_phase);
            if (lane == 0) mbar_arrive(&c->kv_empty[v_stage]);
            next_v();
        };
        for (;;) {
            const RunInfo r = take_run(n_run);
            if (!r.blocks) break;
            const bool pair = r.tokens > g.shape.tokens_stream;
            const int q_tile = pair ? s : 0;
            const int n = 2 * (pair ? r.blocks : (r.blocks + 1 - s) / 2);  // half blocks
            // With the same rows in both streams, blocks 2 t and 2 t + 1 are taken together, one by each stream.
            const bool before = !pair && s == 1;
            // Scores of the next block before this one's values are free: always for two streams of rows, and for one
            // where K has four tiles (heads of up to 64; single tokens of 64 sequences of 8,192 take 258 us, later 281;
            // of 256 of 500, 114 and 119). With two tiles the streams hold both, and little is left to load ahead: 256
            // of 500 would take 132 us for 134, but 64 of 8,192 would take 357 for 352.
            const bool early = pair || L::kKeys >= 4;
            wait(&c->q_full[0], n_q[0]++ & 1);
            if (pair && s == 1) wait(&c->q_full[1], n_q[1]++ & 1);
            tmem_fence_after();
            // Scores of the i-th half block of the stream's keys.
            auto scores = [&](int i) {
                if (!(i & 1)) {
                    if (before) pass_k();
                    wait(&c->kv_full[k_stage], k_phase);
                }
                if (elect_one()) {
                    const uint64_t qd = smem_tile_desc(base + L::kQ + q_tile * L::kTile, 16, 1024);
                    const uint64_t kd = smem_tile_desc(base + L::kKv + k_stage * L::kTile + (i & 1) * 8 * group, 16, group);
                    const uint32_t at = tmem + s_at(s, i & 1);
#pragma unroll
                    for (int e = 0; e < DP / 16; ++e)
                        if (e < ksteps)
                            mma_ss(at, qd + ((e >> 2) * kHalfBytes + (e & 3) * 32) / 16, kd + ((e >> 2) * halves + (e & 3) * 32) / 16,
                                   qk, e > 0);
                    mma_commit(&c->s_full[s][i & 1]);
                    if (i & 1) {
                        mma_commit(&c->kv_empty[k_stage]);
                        if (i + 1 == n) mma_commit(&c->q_empty[q_tile]);
                    }
                }
                __syncwarp();
                if (i & 1) {
                    next_k();
                    if (!pair && s == 0 && i < r.blocks) pass_k();  // block i, the other stream's
                }
            };
            if (s == 1 && (pair || !n) && lane == 0) mbar_arrive(&c->q_empty[0]);  // no use for the first tile: passed
            if (n) {
                scores(0);
                scores(1);
            }
            for (int i = 0; i < n; ++i) {
                // output += weights times values
                if (!(i & 1)) {
                    if (before) pass_v();
                    wait(&c->kv_full[v_stage], v_phase);
                }
                wait(&c->p_full[s][i & 1], n_p++ >> 1 & 1);
                tmem_fence_after();
                if (elect_one()) {
                    const uint64_t vd = smem_tile_desc(base + L::kKv + v_stage * L::kTile + (i & 1) * 8 * group, halves, group);
                    const uint32_t from = tmem + s_at(s, i & 1);
#pragma unroll
                    for (int e = 0; e < kHalfKeys / 16; ++e) mma_ts(to, from + e * 8, vd + e * (group / 8), pv, i > 0 || e > 0);
                    mma_commit(&c->o_step[s]);
                    if (i & 1) {
                        mma_commit(&c->kv_empty[v_stage]);
                        if (i + 1 == n) mma_commit(&c->o_full[s]);
                    }
                }
                __syncwarp();
                if (i & 1) {
                    next_v();
                    if (!pair && s == 0 && i < r.blocks) pass_v();
                }
                if (early) {
                    if (i + 2 < n) scores(i + 2);
                } else if ((i & 1) && i + 1 < n) {
                    scores(i + 1);
                    scores(i + 2);
                }
            }
            if (before && r.blocks % 2) {  // the last block, which only stream 0 has
                pass_k();
                pass_v();
            }
        }
        // What the last instructions arrive on is this CTA's memory, and they use tensor memory: both stay until they
        // are done.
        if (elect_one()) {
            mma_commit(&c->drain[s]);
            if (!mbar_wait_bounded(&c->drain[s], 0, g.budget)) ran_out();
        }
        __syncwarp();
    }

    // ---- warps 0-7: softmax ----
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
        uint32_t r;
        if constexpr (kBf16Type) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
        else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
        return r;
    }

    // Replaces, in tensor memory, a half block's scores of columns outside [lo, hi) and on boxes that are not there;
    // its first column is key `at` of its block. Few blocks need it, so it is little code away from the loop's:
    // fetching instructions that run once a tile is what costs here. A way through them on registers, with a copy of
    // the loop's step, took 3 us a tile more (windows of 512 tokens, 8 x 777 new tokens, cold: 99 us, with this 85, now 82).
    __device__ __forceinline__ void mask_scores(uint32_t ts, int lo, int hi, int at, uint32_t boxes) const {
        const int shift = 7 - g.box_shift;
#pragma unroll 1
        for (int j = 0; j < kHalfKeys; j += 32) {
            const int up = hi - j, down = lo - j;
            uint32_t seen = up >= 32 ? ~0u : up <= 0 ? 0u : (1u << up) - 1;
            if (down > 0) seen = down >= 32 ? 0u : seen & (~0u << down);
            if (boxes != ~0u)
                for (int e = 0; e < 32; ++e) seen &= ~((~boxes >> ((at + j + e) >> shift) & 1u) << e);
            uint32_t x[32];
            tmem_ld32(ts + j, x);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e)
                if (!(seen >> e & 1u)) x[e] = 0xff800000u;
            tmem_st32(ts + j, x);
        }
        tmem_wait_st();
    }

    // The largest of a row's 64 scores, by four chains; NaN if one is.
    static __device__ __forceinline__ float largest(const uint32_t (&x)[2][32]) {
        float t[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t *y = x[j / 2] + j % 2 * 16;
            t[j] = max_nan(__uint_as_float(y[0]), __uint_as_float(y[1]));
#pragma unroll
            for (int e = 2; e < 16; e += 2) t[j] = max_nan(t[j], __uint_as_float(y[e]), __uint_as_float(y[e + 1]));
        }
        return max_nan(max_nan(t[0], t[1]), t[2], t[3]);
    }

    // Scores to weights: x[j] = 2^(x[j] * times + less), and the weights in 16 bits to tensor memory. All
    // exponentials go to the special function unit (512 cycles for a warp's half block). Two to six of 16 by
    // polynomials on the FMA pipes instead were slower: a step waits for latencies, not for that unit.
    static __device__ __forceinline__ void weigh(uint32_t (&x)[32], float times, float less, uint32_t to) {
        const Pair times2 = make_pair(times, times), less2 = make_pair(less, less);
        uint32_t p[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            float u, v;
            split(fma2(make_pair(x[2 * e], x[2 * e + 1]), times2, less2), u, v);
            u = exp2_approx(u);
            v = exp2_approx(v);
            p[e] = pack(u, v);
            x[2 * e] = __float_as_uint(u);
            x[2 * e + 1] = __float_as_uint(v);
        }
        tmem_st16(to, p);
    }

    __device__ __forceinline__ void hand_over(uint64_t *bar) const {
        tmem_wait_st();
        tmem_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar);
    }

    __device__ void softmax_loop(uint32_t tmem, int s) const {
        const PagedAttentionArgs &a = g.a;
        const PlanShape &shape = g.shape;
        const int warp = (threadIdx.x >> 5) & 3, row = warp * 32 + lane;
        const int row_token = row / shape.heads, row_head = row - row_token * shape.heads;
        const int each = shape.parts / a.kv_heads;
        const uint32_t lanes = static_cast<uint32_t>(warp * 32) << 16;
        const uint32_t to = tmem + o_at(s) + lanes;
        const float scale = g.scale_log2;
        int n_run = 0, n_s = 0, n_o = 0, n_block = 0, n_join = 0, n_turn = 0;
        for (;;) {
            const RunInfo r = take_run(n_run);
            if (!r.blocks) break;
            const bool pair = r.tokens > shape.tokens_stream;
            const int steps = pair ? r.blocks : (r.blocks + 1 - s) / 2;
            const int token = pair ? s * shape.tokens_stream + row_token : row_token;  // of the tile
            const int kv_head = g.each.div(r.part);
            const int head_group = (r.part - kv_head * each) * shape.heads + row_head;
            const bool live = row_token < shape.tokens_stream && token < r.tokens && head_group < g.group;
            const bool work = __any_sync(~0u, live);
            int lo = 0, hi = 1 << 30;  // keys that the row sees
            if (live) {
                const int at = r.first + r.t0 + token;
                hi = a.causal && at + 1 < r.end ? at + 1 : r.end;
                if (a.window > 0) lo = at + 1 - shape.window;
            }
            // keys that every row of the warp sees: blocks inside need no mask
            const int all_lo = __reduce_max_sync(~0u, lo), all_hi = __reduce_min_sync(~0u, hi);
            // m, the reference, is ref * scale - kDepth, rounded; a weight is 2^(x * times + less).
            float m = -INFINITY, ref = 0.f, times = scale, less = 0.f, sum = 0.f;
            // A half block from its scores to its weights.
            auto step = [&](int i, uint32_t ts, uint32_t (&x)[2][32]) {
                const float top = largest(x), next = top * scale;
                const bool move = !(next <= m + (kRescale + kDepth));  // NaN moves it too
                if (__builtin_expect(__any_sync(~0u, move && live), 0)) {
                    const float was = m;
                    if (move) {
                        const bool far = fabsf(next) > 0x1p26f;
                        m = far ? next : next - kDepth;
                        ref = top;
                        // What m was rounded by is the same for the whole row and cancels. Where it could be many
                        // powers of two (the lowest value of a type as a score) the scores are taken times a power of
                        // two instead, which rounds nothing: equal scores have equal weights, and others none.
                        times = far ? __uint_as_float(__float_as_uint(scale) & 0x7f800000u) : scale;
                        // the weights of a row with a NaN or an infinite score are NaN; nothing seen yet: zero
                        less = m == -INFINITY ? 0.f : m == INFINITY ? NAN : far ? -ref * times : -m;
                    }
                    if (__any_sync(~0u, move && live && was != -INFINITY)) {  // a row without weights so far has no output
                        const float keep = move ? exp2_approx(was - m) : 1.f;
                        sum *= keep;
                        // The output so far is complete when the last half block's weights have been used (the one
                        // before has: its buffer holds these scores). n_s counts this half block already.
                        wait(&c->o_step[s], n_s & 1);
                        tmem_fence_after();
#pragma unroll 1
                        for (int j = 0; j < a.dim; j += 32) {
                            uint32_t o[32];
                            tmem_ld32(to + j, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
                            tmem_st32(to + j, o);
                        }
                    }
                }
                if (pair) wait(&c->turn[s][warp], (n_turn++ & 1) ^ (s == 0));
                weigh(x[0], times, less, ts);
                weigh(x[1], times, less, ts + 16);
                if (pair && lane == 0) mbar_arrive(&c->turn[s ^ 1][warp]);
                hand_over(&c->p_full[s][i & 1]);
                // the sum is taken while the tensor core has the weights
                Pair add[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t *y = x[j / 2] + j % 2 * 16;
                    add[j] = make_pair(y[0], y[1]);
#pragma unroll
                    for (int e = 2; e < 16; e += 2) add[j] = add2(add[j], make_pair(y[e], y[e + 1]));
                }
                float s0, s1;
                split(add2(add2(add[0], add[1]), add2(add[2], add[3])), s0, s1);
                sum += s0 + s1;
            };
            for (int i = 0; i < 2 * steps; ++i) {
                const int half = i & 1, block = pair ? i / 2 : i / 2 * 2 + s;
                const int key0 = r.key0 + block * kBlockKeys + half * kHalfKeys;
                const uint32_t ts = tmem + s_at(s, half) + lanes;
                wait(&c->s_full[s][half], n_s++ >> 1 & 1);
                tmem_fence_after();
                if (!work) {
                    if (pair) wait(&c->turn[s][warp], (n_turn++ & 1) ^ (s == 0));
                    tmem_fence_before();
                    __syncwarp();
                    if (lane == 0) {
                        if (pair) mbar_arrive(&c->turn[s ^ 1][warp]);
                        mbar_arrive(&c->p_full[s][half]);
                    }
                    continue;
                }
                const uint32_t boxes = c->mask[(n_block + block) % kMaskSlots];
                if (__builtin_expect(all_hi < key0 + kHalfKeys || all_lo > key0 || boxes != ~0u, 0))
                    mask_scores(ts, lo - key0, hi - key0, half * kHalfKeys, boxes);
                uint32_t x[2][32];
                tmem_ld32(ts, x[0]);
                tmem_ld32(ts + 32, x[1]);
                tmem_wait_ld();
                step(i, ts, x);
            }
            n_block += r.blocks;
            if (steps) {
                wait(&c->o_full[s], n_o++ & 1);
                tmem_fence_after();
            }
            if (!pair) {
                if (s == 1) {
                    if (m == -INFINITY) sum = 0.f;
                    c->join[row][0] = m;
                    c->join[row][1] = sum;
                    tmem_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&c->join_full);
                } else {
                    wait(&c->join_full, n_join & 1);
                }
            }
            if (m == -INFINITY) sum = 0.f;  // no score: the weights are what 2^x gives at the least
            if (work && (pair || s == 0)) {
                tmem_fence_after();
                float k0 = 1.f, k1 = 0.f;
                const bool both = !pair && r.blocks > 1;
                if (both) {
                    const float m1 = c->join[row][0], all = fmaxf(m, m1), base = all == -INFINITY ? 0.f : all;
                    k0 = exp2_approx(m - base);
                    k1 = exp2_approx(m1 - base);
                    sum = sum * k0 + c->join[row][1] * k1;
                    m = all;
                }
                const int64_t q_row = r.q0 + r.t0 + token;
                const int head = kv_head * g.group + head_group;
                const int slot_row = (pair ? s * kStreamRows : 0) + row;
                char *slot = static_cast<char *>(a.workspace) + shared_bytes(g.ctas) + (2 * blockIdx.x + r.slot) * slot_bytes(DP);
                T *out = static_cast<T *>(a.out) + q_row * a.o_st + head * a.o_sh;
                // rows of whole sectors: half the stores
                const bool sectors = ((reinterpret_cast<uintptr_t>(a.out) & 31) | (a.o_st | a.o_sh | a.dim) % 16) == 0;
                if (r.slot < 0) {
                    const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;
                    k0 *= inv;
                    k1 *= inv;
                }
#pragma unroll 1
                for (int j = 0; j < a.dim; j += 32) {
                    uint32_t o[32], o1[32];
                    tmem_ld32(to + j, o);
                    if (both) tmem_ld32(tmem + o_at(1) + lanes + j, o1);
                    tmem_wait_ld();
                    if (!live) continue;
                    float f[32];
#pragma unroll
                    for (int e = 0; e < 32; ++e) {
                        f[e] = __uint_as_float(o[e]) * k0;
                        if (both) f[e] = fmaf(__uint_as_float(o1[e]), k1, f[e]);
                        if (sum == 0.f) f[e] = 0.f;
                    }
                    if (r.slot >= 0) {
                        float *o32 = reinterpret_cast<float *>(slot) + slot_row * DP + j;
#pragma unroll
                        for (int e = 0; e < 32; e += 8) {
                            uint32_t p[8];
#pragma unroll
                            for (int k = 0; k < 8; ++k) p[k] = __float_as_uint(f[e + k]);
                            st_sector(o32 + e, p);
                        }
                    } else if (sectors) {
#pragma unroll
                        for (int e = 0; e < 32; e += 16) {
                            uint32_t p[8];
#pragma unroll
                            for (int k = 0; k < 8; ++k) p[k] = pack(f[e + 2 * k], f[e + 2 * k + 1]);
                            if (j + e < a.dim) st_sector(out + j + e, p);
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; e += 8)
                            if (j + e < a.dim)
                                *reinterpret_cast<uint4 *>(out + j + e) =
                                    make_uint4(pack(f[e], f[e + 1]), pack(f[e + 2], f[e + 3]), pack(f[e + 4], f[e + 5]),
                                               pack(f[e + 6], f[e + 7]));
                    }
                }
                if (live && r.slot >= 0)
                    reinterpret_cast<float2 *>(slot + static_cast<size_t>(2 * kStreamRows) * DP * 4)[slot_row] = make_float2(m, sum);
                if (live && r.slot < 0 && a.lse)
                    a.lse[q_row * a.q_heads + head] = sum == 0.f ? -INFINITY : m * 0.6931471805599453f + logf(sum);
                tmem_fence_before();
            }
            if (!pair) {
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
                           const __grid_constant__ CUtensorMap lines, const __grid_constant__ CUtensorMap queries) {
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
            mbar_init(&c->kv_empty[i], 2);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&c->q_full[i], 1);
            mbar_init(&c->q_empty[i], 2 - i);  // the first tile of queries goes through both streams
            for (int j = 0; j < 4; ++j) mbar_init(&c->turn[i][j], 1);
            for (int j = 0; j < 2; ++j) {
                mbar_init(&c->s_full[i][j], 1);
                mbar_init(&c->p_full[i][j], 4);
            }
            mbar_init(&c->o_step[i], 1);
            mbar_init(&c->o_full[i], 1);
        }
        mbar_init(&c->join_full, 4);
        mbar_init(&c->join_empty, 4);
        mbar_init(&c->drain[0], 1);
        mbar_init(&c->drain[1], 1);
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
        tma_prefetch_map(&queries);
    }
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    const uint32_t tmem = K::same(c->tmem);
    pdl_launch();
    if (warp < 8) {
        take_registers<kRegsSoftmax>();
        k.softmax_loop(tmem, warp >> 2);
    } else {
        give_registers<kRegsOther>();
        if (warp == 8) k.plan_loop(&boxes, &lines);
        else if (warp < 11) k.mma_loop(tmem, warp - 9);
        else k.value_loop(&boxes, &lines, &queries);
    }
    tmem_fence_before();
    __syncthreads();
    if (warp == 9) tmem_free(tmem, 512);
}

// Joins the tiles that several CTAs share: block (c, y) the one that begins in
// CTA c and does not end there, the y-th part of its rows. A launch of its own
// that is on its way while the first one ends: joined in the first one, by the
// warp that finds all parts marked, decode of one sequence took 23 us and not
// 19, of 32 ragged ones 271 and not 255, since every part then waits until its
// stores are seen by all.
constexpr int kJoinThreads = 128;
template <int DP, typename T>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const __grid_constant__ KernelArgs g) {
    pdl_wait();
    const PagedAttentionArgs &a = g.a;
    const Shared p = static_cast<const Shared *>(a.workspace)[blockIdx.x];
    const int pieces = min(p.pieces, static_cast<int>(gridDim.x - blockIdx.x));
    if (pieces < 2) return;
    constexpr int kLanes = DP / 4;
    const int e = threadIdx.x % kLanes * 4, each = g.shape.parts / a.kv_heads, step = gridDim.y * (kJoinThreads / kLanes);
    const char *slots = static_cast<const char *>(a.workspace) + shared_bytes(g.ctas);
    for (int n = blockIdx.y * (kJoinThreads / kLanes) + threadIdx.x / kLanes; n < p.tokens * g.shape.heads; n += step) {
        const int token = n / g.shape.heads, row_head = n - token * g.shape.heads;
        const int stream = token >= g.shape.tokens_stream;
        const int r = stream * kStreamRows + (token - stream * g.shape.tokens_stream) * g.shape.heads + row_head;
        const int head_group = p.part % each * g.shape.heads + row_head;
        if (head_group >= g.group) continue;
        float m = -INFINITY, sum = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int i = 0; i < pieces; ++i) {
            const char *slot = slots + (2 * static_cast<size_t>(blockIdx.x + i) + (i == 0)) * slot_bytes(DP);
            const float2 ms = reinterpret_cast<const float2 *>(slot + static_cast<size_t>(2 * kStreamRows) * DP * 4)[r];
            const float4 v = *reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(slot) + r * DP + e);
            const float all = fmaxf(m, ms.x), base = all == -INFINITY ? 0.f : all;
            const float k0 = exp2_approx(m - base), k1 = exp2_approx(ms.x - base);
            m = all;
            sum = sum * k0 + ms.y * k1;
            o.x = o.x * k0 + v.x * k1;
            o.y = o.y * k0 + v.y * k1;
            o.z = o.z * k0 + v.z * k1;
            o.w = o.w * k0 + v.w * k1;
        }
        const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;
        const int64_t row = p.q0 + p.t0 + token;
        const int head = p.part / each * g.group + head_group;
        if (e < a.dim)
            *reinterpret_cast<uint2 *>(static_cast<T *>(a.out) + row * a.o_st + head * a.o_sh + e) =
                make_uint2(Kernel<DP, T>::pack(o.x * inv, o.y * inv), Kernel<DP, T>::pack(o.z * inv, o.w * inv));
        if (a.lse && e == 0) a.lse[row * a.q_heads + head] = sum == 0.f ? -INFINITY : m * 0.6931471805599453f + logf(sum);
    }
}

// A word of pinned host memory that kernels write whose wait ran out, and that
// the next call reads: such a kernel ends with outputs that mean nothing, and
// no call waits for the GPU to see it. Null where there is no GPU.
uint32_t *gave_up_word() {
    static std::mutex mu;
    static std::atomic<uint32_t *> word{nullptr};
    if (uint32_t *w = word.load(std::memory_order_acquire)) return w;
    std::lock_guard<std::mutex> lock(mu);
    if (!word.load(std::memory_order_relaxed)) {
        cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;  // the first call may be a captured one
        void *p = nullptr;
        if (cudaThreadExchangeStreamCaptureMode(&mode) != cudaSuccess) return nullptr;
        const cudaError_t e = cudaHostAlloc(&p, 64, cudaHostAllocPortable | cudaHostAllocMapped);
        cudaThreadExchangeStreamCaptureMode(&mode);
        if (e != cudaSuccess) return nullptr;
        std::memset(p, 0, 64);
        word.store(static_cast<uint32_t *>(p), std::memory_order_release);
    }
    return word.load(std::memory_order_relaxed);
}

// CTAs that a call is given: no more than its units can be, and one an SM.
int plan_ctas(const PagedAttentionArgs &a, const PlanShape &s, int sms) {
    const int64_t blocks = s.tokens > kBlockKeys ? (s.tokens + kBlockKeys - 1) / kBlockKeys : 1;
    const int64_t seqs = a.batch.seqs < a.rows ? a.batch.seqs : a.rows;
    const int64_t tiles = (seqs + a.rows / (2 * s.tokens_stream)) * s.parts;
    const int64_t units = blocks > sms || tiles > sms ? sms : tiles * blocks;
    return static_cast<int>(units < 1 ? 1 : units < sms ? units : sms);
}

using EncodeFn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                              const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

int encode(int dtype, void *base, int rank, const cuuint64_t *dims, const cuuint64_t *strides, const cuuint32_t *box,
           CUtensorMap *map) {
    static const auto fn = reinterpret_cast<EncodeFn>(gpu::driver_symbol("cuTensorMapEncodeTiled"));
    if (!fn) return cudaErrorNotSupported;
    const cuuint32_t one[5] = {1, 1, 1, 1, 1};
    const CUresult e = fn(map, dtype == kBf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, rank, base,
                          dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return e == CUDA_SUCCESS ? 0 : static_cast<int>(cudaErrorInvalidValue);
}

// The pool's index and its maps: boxes of g->box slots, and lines of one.
int view_pool(KernelArgs *g, int dtype, CUtensorMap *boxes, CUtensorMap *lines) {
    const PagedAttentionArgs &a = g->a;
    const int64_t page = a.batch.pages > 1 ? a.pool_page : 0, head = a.kv_heads > 1 ? a.pool_head : 0;
    int64_t unit = a.pool_plane;
    for (int64_t other : {page, head})
        while (other) {
            const int64_t rest = unit % other;
            unit = other;
            other = rest;
        }
    if (unit <= 0 || unit % 8) return cudaErrorInvalidValue;
    const int64_t last = ((a.batch.pages - 1) * page + a.pool_plane + (a.kv_heads - 1) * head) / unit;
    if (last >= 0x7fffffff) return cudaErrorInvalidValue;
    g->pool.page = static_cast<int>(page / unit);
    g->pool.plane = static_cast<int>(a.pool_plane / unit);
    g->pool.head = static_cast<int>(head / unit);
    g->pool.none = static_cast<int>(last + 1);
    void *base = const_cast<void *>(a.pool);
    const cuuint64_t token = static_cast<cuuint64_t>(a.pool_token) * 2, index = static_cast<cuuint64_t>(unit) * 2;
    const cuuint64_t dim = a.dim, slots = a.batch.page_tokens, all = static_cast<cuuint64_t>(last) + 1;
    const cuuint32_t box = g->box;
    const cuuint64_t dims[5] = {dim, slots, 1, 1, all}, strides[4] = {token, token * slots, token * slots, index};
    const cuuint32_t line[5] = {64, 1, 1, 1, 1}, rows[5] = {64, box, 1, 1, 1};
    int e = encode(dtype, base, 5, dims, strides, line, lines);
    if (e) return e;
    if (!g->pool.whole) return encode(dtype, base, 5, dims, strides, rows, boxes);
    const cuuint64_t dims_whole[5] = {64, 8, dim / 64, slots / 8, all}, strides_whole[4] = {token, 128, token * 8, index};
    const cuuint32_t box_whole[5] = {64, 8, static_cast<cuuint32_t>(dim / 64), box / 8, 1};
    return encode(dtype, base, 5, dims_whole, strides_whole, box_whole, boxes);
}

// The queries as (element, query head of a key head, key head, token), a stream's rows a box.
int view_queries(const KernelArgs &g, int dtype, CUtensorMap *queries) {
    const PagedAttentionArgs &a = g.a;
    const cuuint64_t dims[4] = {static_cast<cuuint64_t>(a.dim), static_cast<cuuint64_t>(g.group),
                                static_cast<cuuint64_t>(a.kv_heads), static_cast<cuuint64_t>(a.rows)};
    const cuuint64_t strides[3] = {static_cast<cuuint64_t>(a.q_sh) * 2, static_cast<cuuint64_t>(a.q_sh) * g.group * 2,
                                   static_cast<cuuint64_t>(a.q_st) * 2};
    const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(g.shape.heads), 1, static_cast<cuuint32_t>(g.shape.tokens_stream)};
    return encode(dtype, const_cast<void *>(a.q), 4, dims, strides, box, queries);
}

template <int DP, typename T>
int launch(KernelArgs &g, int dtype, int device, bool join, cudaStream_t st) {
    using K = Kernel<DP, T>;
    constexpr int smem = K::L::kControl + static_cast<int>(sizeof(typename K::C));
    static_assert(smem <= 227 * 1024, "shared memory of one CTA");
    CUtensorMap boxes, lines, queries;
    std::memset(&boxes, 0, sizeof boxes);
    std::memset(&lines, 0, sizeof lines);
    int bad = g.a.batch.pages ? view_pool(&g, dtype, &boxes, &lines) : 0;
    if (!bad) bad = view_queries(g, dtype, &queries);
    if (bad) return bad;
    static std::atomic<uint64_t> configured{0};  // devices
    cudaError_t e = cudaSuccess;
    if (device > 63 || !(configured.load(std::memory_order_acquire) >> device & 1)) {
        e = cudaFuncSetAttribute(paged_attention_kernel<DP, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        cudaFuncAttributes attr;
        if (e == cudaSuccess) e = cudaFuncGetAttributes(&attr, paged_attention_kernel<DP, T>);
        if (e != cudaSuccess) return static_cast<int>(e);
        if (attr.numRegs != kRegsLaunch) return cudaErrorLaunchOutOfResources;  // the split above would not add up
        if (device <= 63) configured.fetch_or(1ull << device, std::memory_order_release);
    }
    paged_attention_kernel<DP, T><<<g.ctas, kThreads, smem, st>>>(g, boxes, lines, queries);
    note_launch();
    e = cudaGetLastError();
    if (e != cudaSuccess || !join) return static_cast<int>(e);
    cudaLaunchConfig_t cfg = {};
    // Blocks for the rows of a tile, two passes of four rows each at most: 256 rows take 32 (against 8: a chunk of 1,024
    // over 8,192 tokens 152 -> 143 us); where each sequence has one new token a tile has few rows, and idle blocks
    // would cost 2 us.
    const int64_t rows = (g.a.rows - g.a.batch.seqs + 1) * g.shape.heads;
    cfg.gridDim = dim3(g.ctas, static_cast<unsigned>(plan_clamp((rows + 7) / 8, 4, 32)));
    cfg.blockDim = dim3(kJoinThreads);
    cfg.stream = st;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, join_kernel<DP, T>, g);
    note_launch();
    return static_cast<int>(e);
}

}  // namespace

size_t paged_attention_workspace(int dim, int device) {
    const int sms = sm_count(device);
    return shared_bytes(sms) + 2 * static_cast<size_t>(sms) * slot_bytes(dim <= 64 ? 64 : 128);
}

bool paged_attention_give_up() {
    uint32_t *word = gave_up_word();
    if (word) __atomic_store_n(word, 1u, __ATOMIC_RELEASE);
    return word != nullptr;
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
    g.gave_up = gave_up_word();
    if (!g.gave_up) return cudaErrorMemoryAllocation;
    if (*static_cast<volatile uint32_t *>(g.gave_up) && __atomic_exchange_n(g.gave_up, 0u, __ATOMIC_ACQ_REL)) return kWaitRanOut;
    const int64_t tokens = a.batch.pages > 0 ? a.batch.table_width * a.batch.page_tokens : 0;
    g.group = a.q_heads / a.kv_heads;
    plan_parts(&g.shape, a.kv_heads, g.group);
    g.shape.causal = a.causal;
    g.shape.window = plan_clamp(a.window, 0, kMostTokens);
    g.shape.rows = static_cast<int>(a.rows);
    g.shape.tokens = plan_clamp(tokens, 0, kMostTokens);
    // a scale of zero would make NaN of a masked score; this one gives every seen score the same weight
    g.scale_log2 = fmaxf(fabsf(a.scale) * 1.4426950408889634f, 1e-30f);
    g.box = a.batch.page_tokens & -a.batch.page_tokens;
    if (g.box > kBlockKeys) g.box = kBlockKeys;
    g.box_shift = 0;
    while (g.box << g.box_shift < kBlockKeys) ++g.box_shift;
    g.page_tokens = FastDiv(static_cast<uint32_t>(a.batch.page_tokens));
    g.each = FastDiv(static_cast<uint32_t>(g.shape.parts / a.kv_heads));
    g.pool = PoolView();
    g.pool.whole = a.dim % 64 == 0;
    const int halves = a.dim <= 64 ? 1 : 2, tile_half = kStreamRows * 128;
    g.pool.group_bytes = g.pool.whole ? 1024 * halves : 1024;
    g.pool.half_bytes = g.pool.whole ? 1024 : tile_half;
    g.budget = wait_budget_ns();
    g.tries = static_cast<uint32_t>(plan_clamp(static_cast<int64_t>(g.budget / 1000), 1, 0x7fffffff));
    g.ctas = plan_ctas(a, g.shape, sm_count(device));
    if (!a.workspace || a.workspace_bytes < shared_bytes(g.ctas) + 2 * g.ctas * slot_bytes(a.dim <= 64 ? 64 : 128))
        return cudaErrorInvalidValue;
    const bool join = g.ctas > 1 && tokens > kBlockKeys;  // a tile of one block is never shared
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (a.dim <= 64)
        return dtype == kBf16 ? launch<64, __nv_bfloat16>(g, dtype, device, join, st) : launch<64, __half>(g, dtype, device, join, st);
    return dtype == kBf16 ? launch<128, __nv_bfloat16>(g, dtype, device, join, st) : launch<128, __half>(g, dtype, device, join, st);
}

}  // namespace kern
}  // namespace mpcomm
