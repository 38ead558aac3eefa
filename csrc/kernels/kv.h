// Host-side entry points of the paged KV cache operators (kv_rows.cu,
// paged_attention.cu). Like launch.h: streams are void* (a cudaStream_t), a
// launcher returns 0 or a cudaError_t value and never synchronises. All
// strides count elements. Launchers run on `device`, whatever the calling
// thread's current device is.
#ifndef MPCOMM_B200_CSRC_KERNELS_KV_H_
#define MPCOMM_B200_CSRC_KERNELS_KV_H_

#include <cstddef>
#include <cstdint>

#ifdef __CUDACC__
#define MPCOMM_HD __host__ __device__
#else
#define MPCOMM_HD
#endif

namespace mpcomm {
namespace kern {

enum KvType { kBf16 = 0, kFp16 = 1, kFp32 = 2 };

// An array of int32 or int64 in device memory.
struct IndexPtr {
    const void *ptr = nullptr;
    int is64 = 0;
    MPCOMM_HD int64_t at(int64_t i) const {
        return is64 ? static_cast<const int64_t *>(ptr)[i] : static_cast<const int32_t *>(ptr)[i];
    }
};

// Division of 31-bit values by a constant: a multiplication.
struct FastDiv {
    uint32_t times = 0, shift = 0;
    FastDiv() = default;
    explicit FastDiv(uint32_t d) {
        // 2^(31 + ceil(log2 d)) / d, rounded up, is at most 2^32 - 1 and exact for 31-bit dividends
        while ((1ull << shift) < d) ++shift;
        times = static_cast<uint32_t>(((1ull << (31 + shift)) + d - 1) / d);
    }
    MPCOMM_HD int div(int n) const {
        return static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(n)) * times) >> (31 + shift));
    }
};

// A ragged batch over a paged cache. Rows starts[b] .. starts[b + 1] are the
// newest tokens of sequence b, lens[b] counts all its tokens. Token p lies
// in slot p % page_tokens of page table[b * table_stride + p / page_tokens].
struct KvBatch {
    IndexPtr table, lens, starts;
    int64_t table_stride = 0, table_width = 0;
    int64_t pages = 0;
    int seqs = 0;
    int page_tokens = 1;
};

// The sequence that holds `row`, or -1 (padding). starts is ascending; rows
// of a table that is not are put somewhere, and checked there as any other.
MPCOMM_HD inline int sequence_of(const KvBatch &k, int64_t row) {
    int lo = 0, hi = k.seqs;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (k.starts.at(mid + 1) > row) hi = mid;
        else lo = mid + 1;
    }
    return lo < k.seqs && k.starts.at(lo) <= row ? lo : -1;
}

// The page of token p of sequence b, or -1 where the table or the pool has none.
MPCOMM_HD inline int64_t page_of(const KvBatch &k, int b, int64_t p) {
    if (p < 0) return -1;
    const int64_t column = p / k.page_tokens;
    if (column >= k.table_width) return -1;
    const int64_t page = k.table.at(b * k.table_stride + column);
    return page >= 0 && page < k.pages ? page : -1;
}

// Heads that lie side by side in a row: source and destination of each.
// Offsets are b * sb + t * st + head * sh + element * sd with row =
// b * tokens + t; with plane >= 0 the destination is a slot of the cache:
// page * db + slot * dt + head * dh + element * dd (dst: the plane's base).
struct KvRowGroup {
    const void *src = nullptr;
    void *dst = nullptr;
    int64_t sb = 0, st = 0, sh = 0, sd = 1;
    int64_t db = 0, dt = 0, dh = 0, dd = 1;
    int heads = 0;
    int rotate = 0;
    int plane = -1;
};

constexpr int kMostHeads = 1 << 30;  // of a row: a block's (row, head) pairs are counted in 32 bits

struct KvRowsArgs {
    KvRowGroup group[3];
    int groups = 0;
    int heads = 0;  // of all groups
    int dim = 0;
    int pairs = 0;  // rotated pairs of a head
    int interleaved = 0;
    int64_t rows = 0, tokens = 1;  // below 2^31
    const void *inv_freq = nullptr;  // radians a position, one for each pair
    int freq_f64 = 0;
    float magnitude = 1.f, sign = 1.f;
    IndexPtr positions;  // null: the rows' places in their sequences
    int64_t pos_sb = 0, pos_st = 0;
    KvBatch batch;  // seqs == 0: rows of no batch
    int in_batch = 0;
    uint32_t *status = nullptr;
};
// Rotates (and copies) the heads of `rows` rows. Rows behind the batch's
// last sequence are not written; a row whose page is not in the table or the
// pool writes nothing to the cache and sets kStatusBadIndex.
int kv_rows(const KvRowsArgs &a, int dtype, int device, void *stream);

struct PagedAttentionArgs {
    const void *q = nullptr;
    void *out = nullptr;
    float *lse = nullptr;  // [rows, q_heads] contiguous, may be null
    const void *pool = nullptr;  // [pages, 2, kv_heads, page_tokens, dim]
    int64_t q_st = 0, q_sh = 0, o_st = 0, o_sh = 0;
    int64_t pool_page = 0, pool_plane = 0, pool_head = 0, pool_token = 0;
    int64_t rows = 0;
    int q_heads = 0, kv_heads = 0, dim = 0;
    float scale = 1.f;
    int causal = 1;
    int64_t window = 0;  // keys that a causal row sees, itself among them; 0: all
    int fill_tail = 0;   // write zeros to rows of no sequence (their lse is -inf in any case)
    KvBatch batch;
    void *workspace = nullptr;
    size_t workspace_bytes = 0;
    uint32_t *status = nullptr;
};
// Bytes of workspace that a call needs (its contents do not matter), 16-byte aligned.
size_t paged_attention_workspace(int dim, int device);
// A wait in the kernel that runs out (wait_budget_ns(); never in a run that
// works) sets kStatusLoadTimeout in `status` and ends the call with outputs
// that mean nothing. Without `status` the next call on any device returns
// kWaitRanOut, once, and does nothing.
constexpr int kWaitRanOut = -1;
int paged_attention(const PagedAttentionArgs &a, int dtype, int device, void *stream);
// Says on the host what a kernel says whose wait ran out (for tests). False without a GPU.
bool paged_attention_give_up();

}  // namespace kern
}  // namespace mpcomm

#endif  // MPCOMM_B200_CSRC_KERNELS_KV_H_
