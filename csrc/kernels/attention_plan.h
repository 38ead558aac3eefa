// How paged attention splits a ragged batch, for the kernels and for tests on
// the host. A sequence's rows for one key head are its new tokens' query
// heads, token by token: row r is token r / group, head r % group. They are
// cut into tiles of up to kTileRows rows; a tile reads the blocks of
// kBlockKeys keys that some row of it sees. The unit of work is one block of
// one tile. All units stand in one line (sequence, key head, tile, block);
// every CTA takes an equal, contiguous part of it, so the work is even
// whatever the lengths are, and neighbours read the same keys.
#ifndef MPCOMM_B200_CSRC_KERNELS_ATTENTION_PLAN_H_
#define MPCOMM_B200_CSRC_KERNELS_ATTENTION_PLAN_H_

#include "kernels/kv.h"

namespace mpcomm {
namespace kern {

constexpr int kTileRows = 256;
constexpr int kBlockKeys = 128;
constexpr int kMostTokens = 1 << 30;  // of a sequence: positions are 32-bit in the kernel

struct PlanShape {
    int group = 1;  // query heads of a key head
    int kv_heads = 1;
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
};

struct PlanTile {
    int rows = 0;             // of the tile
    int lo = 0, hi = 0;       // keys that some row sees: [lo, hi)
    int block0 = 0, blocks = 1;  // a tile that sees nothing still has a block, all of it masked
};

MPCOMM_HD inline int plan_clamp(int64_t v, int64_t lo, int64_t hi) {
    return static_cast<int>(v < lo ? lo : v > hi ? hi : v);
}

MPCOMM_HD inline PlanSeq plan_seq(const PlanShape &s, int64_t start, int64_t stop, int64_t len) {
    PlanSeq q;
    q.q0 = plan_clamp(start, 0, s.rows);
    q.new_tokens = plan_clamp(stop, q.q0, s.rows) - q.q0;
    const int n = plan_clamp(len, 0, kMostTokens);
    q.first = n - q.new_tokens;
    q.end = n < s.tokens ? n : s.tokens;
    q.tiles = static_cast<int>((static_cast<int64_t>(q.new_tokens) * s.group + kTileRows - 1) / kTileRows);
    return q;
}

MPCOMM_HD inline PlanTile plan_tile(const PlanShape &s, const PlanSeq &q, int m) {
    PlanTile t;
    const int64_t all = static_cast<int64_t>(q.new_tokens) * s.group;
    const int64_t r0 = static_cast<int64_t>(m) * kTileRows;
    t.rows = static_cast<int>(all - r0 < kTileRows ? all - r0 : kTileRows);
    t.hi = q.end;
    if (s.causal) {
        const int last = q.first + static_cast<int>((r0 + t.rows - 1) / s.group);
        if (last + 1 < t.hi) t.hi = last + 1;
        if (t.hi < 0) t.hi = 0;
    }
    if (s.window > 0) {
        const int lo = q.first + static_cast<int>(r0 / s.group) + 1 - s.window;
        if (lo > 0) t.lo = lo;
    }
    if (t.lo >= t.hi) t.lo = t.hi = 0;
    t.block0 = t.lo / kBlockKeys;
    const int n = (t.hi + kBlockKeys - 1) / kBlockKeys - t.block0;
    t.blocks = n > 0 ? n : 1;
    return t;
}

// Units of one key head of a sequence.
MPCOMM_HD inline int64_t plan_head_units(const PlanShape &s, const PlanSeq &q) {
    int64_t n = 0;
    for (int m = 0; m < q.tiles; ++m) n += plan_tile(s, q, m).blocks;
    return n;
}

// Units of each CTA; CTA c has [c * share, (c + 1) * share).
MPCOMM_HD inline int64_t plan_share(int64_t units, int ctas) { return units > ctas ? (units + ctas - 1) / ctas : 1; }

// A run of blocks of one tile: what one CTA does of it.
struct PlanRun {
    int h = 0, m = 0;
    int from = 0, to = 0;  // blocks of the tile, [from, to) of tile.blocks
    PlanTile tile;
};

// Goes through the units of one sequence from `offset` on. `left` is what
// the CTA still has to do.
struct PlanCursor {
    int h = 0, m = 0, block = 0;
    MPCOMM_HD void seek(const PlanShape &s, const PlanSeq &q, int64_t head_units, int64_t offset) {
        h = static_cast<int>(offset / head_units);
        int64_t rest = offset - h * head_units;
        for (m = 0;; ++m) {
            const int n = plan_tile(s, q, m).blocks;
            if (rest < n) break;
            rest -= n;
        }
        block = static_cast<int>(rest);
    }
    MPCOMM_HD bool next(const PlanShape &s, const PlanSeq &q, int64_t left, PlanRun *run) {
        if (q.tiles == 0 || h >= s.kv_heads || left <= 0) return false;
        run->h = h;
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
                ++h;
            }
        }
        return true;
    }
};

}  // namespace kern
}  // namespace mpcomm

#endif  // MPCOMM_B200_CSRC_KERNELS_ATTENTION_PLAN_H_
