// How paged attention splits a ragged batch, for the kernels and for tests on
// the host. The query heads of a key head are taken up to kStreamRows at a
// time (a part); a stream has the rows of one part of as many whole tokens as
// fit into kStreamRows, token by token, and a tile is two streams' tokens. A
// tile reads the blocks of kBlockKeys keys that some row of it sees. The unit
// of work is one block of one tile. All units stand in one line (sequence,
// part, tile, block); every CTA takes a contiguous share of equally many
// units, so neighbours read the same keys. A unit is a block whatever its tile
// is: shares are even in blocks for any lengths, and in time where all tiles
// have one stream's rows or all have two's. In a batch of both, the CTAs with
// the tiles of two streams end last (about 2 us a block; two chunks of 512
// tokens take 90 us, 32 single tokens 82, both together 165).
#ifndef MPCOMM_B200_CSRC_KERNELS_ATTENTION_PLAN_H_
#define MPCOMM_B200_CSRC_KERNELS_ATTENTION_PLAN_H_

#include "kernels/kv.h"

namespace mpcomm {
namespace kern {

constexpr int kStreamRows = 128;
constexpr int kBlockKeys = 128;
constexpr int kMostTokens = 1 << 30;  // of a sequence: positions are 32-bit in the kernel

struct PlanShape {
    int heads = 1;   // query heads of a part
    int tokens_stream = kStreamRows;
    int parts = 1;   // of all key heads
    int causal = 1;
    int window = 0;
    int rows = 0;    // of the query tensor
    int tokens = 0;  // that a row of the page table has room for
};

struct PlanSeq {
    int q0 = 0, new_tokens = 0;  // its rows of the query tensor
    int first = 0;               // position of the first new token (may be negative)
    int end = 0;                 // keys there are
    int tiles = 0;
    bool cut = false;            // new tokens see keys that the page table has no room for
};

struct PlanTile {
    int tokens = 0;           // of the tile
    int lo = 0, hi = 0;       // keys that some row sees: [lo, hi)
    int block0 = 0, blocks = 1;  // a tile that sees nothing still has a block, all of it masked
};

// The parts of `kv_heads` key heads with `group` query heads each: as even as they can be.
MPCOMM_HD inline void plan_parts(PlanShape *s, int kv_heads, int group) {
    const int each = (group + kStreamRows - 1) / kStreamRows;
    s->heads = (group + each - 1) / each;
    s->tokens_stream = kStreamRows / s->heads;
    s->parts = kv_heads * each;
}

MPCOMM_HD inline int plan_clamp(int64_t v, int64_t lo, int64_t hi) {
    return static_cast<int>(v < lo ? lo : v > hi ? hi : v);
}

// Quotients of values that hardly ever need 64 bits, whose division is a long
// routine on the GPU. a >= 0, b > 0.
MPCOMM_HD inline int64_t plan_div(int64_t a, int64_t b) {
    if (((a | b) >> 32) == 0) return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
    return a / b;
}

MPCOMM_HD inline PlanSeq plan_seq(const PlanShape &s, int64_t start, int64_t stop, int64_t len) {
    PlanSeq q;
    q.q0 = plan_clamp(start, 0, s.rows);
    q.new_tokens = plan_clamp(stop, q.q0, s.rows) - q.q0;
    const int n = plan_clamp(len, 0, kMostTokens);
    q.first = n - q.new_tokens;
    q.end = n < s.tokens ? n : s.tokens;
    q.cut = q.new_tokens > 0 && len > s.tokens;  // the last one sees itself, whatever the mask
    const int both = 2 * s.tokens_stream;
    q.tiles = q.new_tokens / both + (q.new_tokens % both > 0);
    return q;
}

MPCOMM_HD inline PlanTile plan_tile(const PlanShape &s, const PlanSeq &q, int m) {
    PlanTile t;
    const int t0 = m * 2 * s.tokens_stream;
    t.tokens = q.new_tokens - t0 < 2 * s.tokens_stream ? q.new_tokens - t0 : 2 * s.tokens_stream;
    t.hi = q.end;
    if (s.causal) {
        const int after = q.first + t0 + t.tokens;
        if (after < t.hi) t.hi = after;
        if (t.hi < 0) t.hi = 0;
    }
    if (s.window > 0) {
        const int lo = q.first + t0 + 1 - s.window;
        if (lo > 0) t.lo = lo;
    }
    if (t.lo >= t.hi) t.lo = t.hi = 0;
    t.block0 = t.lo / kBlockKeys;
    const int n = (t.hi + kBlockKeys - 1) / kBlockKeys - t.block0;
    t.blocks = n > 0 ? n : 1;
    return t;
}

// Units of one part of a sequence: its tiles from `m` on, every `step`-th.
MPCOMM_HD inline int64_t plan_part_units(const PlanShape &s, const PlanSeq &q, int m = 0, int step = 1) {
    int64_t n = 0;
    for (; m < q.tiles; m += step) n += plan_tile(s, q, m).blocks;
    return n;
}

// Units of each CTA; CTA c has [c * share, (c + 1) * share).
MPCOMM_HD inline int64_t plan_share(int64_t units, int ctas) { return units > ctas ? plan_div(units + ctas - 1, ctas) : 1; }

// A run of blocks of one tile: what one CTA does of it.
struct PlanRun {
    int part = 0, m = 0;
    int from = 0, to = 0;  // blocks of the tile, [from, to) of tile.blocks
    PlanTile tile;
};

// Goes through the units of one sequence from (part, tile m, block) on.
// `left` is what the CTA still has to do.
struct PlanCursor {
    int part = 0, m = 0, block = 0;
    MPCOMM_HD bool next(const PlanShape &s, const PlanSeq &q, int64_t left, PlanRun *run) {
        if (q.tiles == 0 || part >= s.parts || left <= 0) return false;
        run->part = part;
        run->m = m;
        run->tile = plan_tile(s, q, m);
        run->from = block;
        const int rest = run->tile.blocks - block;
        run->to = block + static_cast<int>(left < rest ? left : rest);
        block = run->to;
        if (block == run->tile.blocks) {
            block = 0;
            if (++m == q.tiles) {
                m = 0;
                ++part;
            }
        }
        return true;
    }
};

}  // namespace kern
}  // namespace mpcomm

#endif  // MPCOMM_B200_CSRC_KERNELS_ATTENTION_PLAN_H_
