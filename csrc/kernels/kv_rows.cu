// Rotary positions, and appending keys and values to a paged cache with the
// rotation applied on the way: one kernel over rows of heads.
//
// A row is one token. Pair i of a head's first 2 * pairs elements is turned
// by t = position * inv_freq[i]:
//     a' = m (a cos t - b sin t),   b' = m (b cos t + a sin t)
// with (a, b) = (x[i], x[i + pairs]), or (x[2i], x[2i + 1]) when interleaved;
// the elements behind them are copied. The gradient is the same rotation by
// -t. The angle is reduced in 64 bits (a position of 2^20 at one radian each
// would be off by 2^-4 radians in 32), in turns, so that the reduction is one
// rint(); sine, cosine and the products are 32-bit, rounded once to the type.
//
// Bound by memory: each element is read and written once. 8,192 x 32 heads x
// 128 in bf16, 134 MB, take 29 us (4.6 TB/s, of 6.55 that a copy of gigabytes
// reaches); 4,096 tokens of 8 heads' keys and values into 64 KiB pages with 32
// heads' queries beside them, 101 MB, 24 us. Few tokens take what a launch
// does.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "kernels/kv.cuh"

namespace mpcomm {
namespace kern {
namespace {

constexpr int kRowThreads = 256;
constexpr int kMaxRowsPerCta = 32;
constexpr int kSeqsKept = 1024;  // whose ends a block keeps in shared memory

// N elements: 16 bytes of them, loaded and stored at once, or one.
template <typename T, int N>
struct alignas(N == 1 ? sizeof(T) : 16) Chunk {
    T e[N];
};

template <typename T, int N>
__device__ __forceinline__ Chunk<T, N> load_chunk(const T *p) {
    return *reinterpret_cast<const Chunk<T, N> *>(p);
}
template <typename T, int N>
__device__ __forceinline__ void store_chunk(T *p, const Chunk<T, N> &c) {
    *reinterpret_cast<Chunk<T, N> *>(p) = c;
}

// Two 16-bit elements of a word as 32-bit values, and back with one rounding each.
template <typename T>
__device__ __forceinline__ float2 unpack(uint32_t w) {
    if constexpr (std::is_same_v<T, __nv_bfloat16>)
        return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    else
        return __half22float2(*reinterpret_cast<const __half2 *>(&w));
}
template <typename T>
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
    uint32_t r;
    if constexpr (std::is_same_v<T, __nv_bfloat16>) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// Turns the pairs (x[j], y[j]).
template <typename T, int N>
__device__ __forceinline__ void turn_two(Chunk<T, N> &x, Chunk<T, N> &y, const float *c, const float *s) {
    if constexpr (N > 1 && sizeof(T) == 2) {
        uint32_t *xw = reinterpret_cast<uint32_t *>(&x), *yw = reinterpret_cast<uint32_t *>(&y);
#pragma unroll
        for (int j = 0; j < N / 2; ++j) {
            const float2 p = unpack<T>(xw[j]), o = unpack<T>(yw[j]);
            xw[j] = pack<T>(p.x * c[2 * j] - o.x * s[2 * j], p.y * c[2 * j + 1] - o.y * s[2 * j + 1]);
            yw[j] = pack<T>(o.x * c[2 * j] + p.x * s[2 * j], o.y * c[2 * j + 1] + p.y * s[2 * j + 1]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const float p = to_f32(x.e[j]), o = to_f32(y.e[j]);
            x.e[j] = from_f32<T>(p * c[j] - o * s[j]);
            y.e[j] = from_f32<T>(o * c[j] + p * s[j]);
        }
    }
}

// Turns the pairs (x[2 j], x[2 j + 1]).
template <typename T, int N>
__device__ __forceinline__ void turn_one(Chunk<T, N> &x, const float *c, const float *s) {
    if constexpr (sizeof(T) == 2) {
        uint32_t *xw = reinterpret_cast<uint32_t *>(&x);
#pragma unroll
        for (int j = 0; j < N / 2; ++j) {
            const float2 p = unpack<T>(xw[j]);
            xw[j] = pack<T>(p.x * c[j] - p.y * s[j], p.y * c[j] + p.x * s[j]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < N / 2; ++j) {
            const float p = x.e[2 * j], o = x.e[2 * j + 1];
            x.e[2 * j] = p * c[j] - o * s[j];
            x.e[2 * j + 1] = o * c[j] + p * s[j];
        }
    }
}

struct RowInfo {
    int64_t page;  // -1: the row has no slot (padding, no page); paged groups skip it
    int32_t slot;
    int32_t live;  // 0: padding behind the last sequence, nothing is written
    double pos;
};

__device__ uint32_t g_rows_status;

// Where row `row`, of sequence `seq` (-1: padding), goes. Everything read from
// the batch's tables is checked against the rows, pages and columns there are.
__device__ __forceinline__ RowInfo place_row(const KvBatch &k, int seq, int64_t row, uint32_t *status) {
    RowInfo r{-1, 0, 0, 0.0};
    if (seq < 0) return r;
    const int64_t p = k.lens.at(seq) - (k.starts.at(seq + 1) - row);
    r.live = 1;
    r.pos = static_cast<double>(p);
    r.page = page_of(k, seq, p);
    r.slot = r.page >= 0 ? static_cast<int32_t>(p % k.page_tokens) : 0;
    if (r.page < 0) atomicOr(status, kStatusBadIndex);
    return r;
}

// How a launch divides its work, and the divisions that its threads do.
struct RowsShape {
    int units, lanes, rows;  // of a block
    FastDiv by_units, by_heads, by_pairs, by_tokens;
};

// Threads: unit of a head (N pairs or elements; blocks of y go on with them),
// then a lane of the block's (row, head) pairs. A thread holds its first
// pair's elements before the rows' places, sines and cosines are known, and
// always those of the next pair while it turns and stores one, so that the
// trips to memory overlap (two pairs ahead, in registers, at the price of
// occupancy: 3 % slower). A block's sines and cosines are computed once for all
// heads. N > 1 needs unit element strides, 16-byte aligned bases and
// strides and pairs, dim multiples of N (of N / 2 for interleaved pairs).
template <typename T, int N, bool INTERLEAVED, bool PAGED>
__global__ void __launch_bounds__(kRowThreads, 4) kv_rows_kernel(const __grid_constant__ KvRowsArgs a, const __grid_constant__ RowsShape g) {
    constexpr int H = INTERLEAVED && N > 1 ? N / 2 : N;  // pairs of a rotating unit
    constexpr bool kTwo = !INTERLEAVED || N == 1;        // whose pairs lie in two places
    extern __shared__ __align__(16) float trig[];        // [rows][2][pairs]: cosines, sines
    __shared__ RowInfo info[PAGED ? kMaxRowsPerCta : 1];
    __shared__ int ends[PAGED ? kSeqsKept : 1];
    const int row0 = blockIdx.x * g.rows, tid = threadIdx.x;
    const int rows = min(g.rows, static_cast<int>(a.rows) - row0);
    const int lane = g.by_units.div(tid), u = tid - lane * g.units + blockIdx.y * g.units;
    const int turning = a.pairs / H;
    const bool turn = u < turning;
    const int all = lane < g.lanes && u < turning + (a.dim - 2 * a.pairs) / N ? rows * a.heads : 0;  // (row, head) pairs
    // elements of the unit, and of the other half of its pairs
    const int at = turn ? (INTERLEAVED ? 2 * H * u : N * u) : 2 * a.pairs + (u - turning) * N;
    const int other = at + (INTERLEAVED ? 1 : a.pairs);

    auto group_of = [&](int h) { return PAGED ? (h >= a.group[0].heads) + (h >= a.group[0].heads + a.group[1].heads) : 0; };
    auto first_of = [&](int group) { return (group > 0 ? a.group[0].heads : 0) + (group > 1 ? a.group[1].heads : 0); };
    Chunk<T, N> v, w;
    auto load = [&](int i) {
        const int r = g.by_heads.div(i), h = i - r * a.heads, k = group_of(h);
        const KvRowGroup &q = a.group[k];
        const int b = PAGED ? 0 : g.by_tokens.div(row0 + r);
        const int64_t t = row0 + r - (PAGED ? 0 : b * static_cast<int>(a.tokens));
        const T *src = static_cast<const T *>(q.src) + b * q.sb + t * q.st + (h - first_of(k)) * q.sh;
        v = load_chunk<T, N>(src + (N == 1 ? at * q.sd : at));
        if (kTwo && turn) w = load_chunk<T, N>(src + (N == 1 ? other * q.sd : other));
    };
    if (lane < all) load(lane);

    if (PAGED) {
        uint32_t *status = a.status ? a.status : &g_rows_status;
        const KvBatch &k = a.batch;
        if (k.seqs <= kSeqsKept) {
            for (int i = tid; i < k.seqs; i += blockDim.x) {
                const int64_t end = k.starts.at(i + 1);
                ends[i] = static_cast<int>(end < 0 ? 0 : end > a.rows ? a.rows : end);
            }
            __syncthreads();
        }
        if (tid < rows) {
            int seq;
            if (k.seqs <= kSeqsKept) {
                int lo = 0, hi = k.seqs;
                while (lo < hi) {
                    const int mid = (lo + hi) >> 1;
                    if (ends[mid] > row0 + tid) hi = mid;
                    else lo = mid + 1;
                }
                seq = lo < k.seqs && k.starts.at(lo) <= row0 + tid ? lo : -1;
            } else {
                seq = sequence_of(k, row0 + tid);
            }
            info[tid] = place_row(k, seq, row0 + tid, status);
        }
        __syncthreads();
    }
    for (int i = tid; i < rows * a.pairs; i += blockDim.x) {
        const int r = g.by_pairs.div(i), p = i - r * a.pairs;
        double pos;
        if (!PAGED || a.positions.ptr) {
            const int b = g.by_tokens.div(row0 + r);
            pos = static_cast<double>(a.positions.at(b * a.pos_sb + (row0 + r - b * static_cast<int>(a.tokens)) * a.pos_st));
        } else {
            pos = info[r].pos;
        }
        const double f = a.freq_f64 ? static_cast<const double *>(a.inv_freq)[p]
                                    : static_cast<double>(static_cast<const float *>(a.inv_freq)[p]);
        double turns = pos * (f * 0.15915494309189533577);  // 1 / (2 pi)
        turns -= rint(turns);
        float sine, cosine;
        sincospif(static_cast<float>(2.0 * turns), &sine, &cosine);
        trig[2 * r * a.pairs + p] = cosine * a.magnitude;
        trig[(2 * r + 1) * a.pairs + p] = sine * a.magnitude * a.sign;
    }
    __syncthreads();

    for (int i = lane; i < all;) {
        const int r = g.by_heads.div(i), h = i - r * a.heads, k = group_of(h);
        const KvRowGroup &q = a.group[k];
        Chunk<T, N> x = v, y = w;
        i += g.lanes;
        if (i < all) load(i);
        if (PAGED && !info[r].live) continue;
        T *dst = static_cast<T *>(q.dst) + (h - first_of(k)) * q.dh;
        if (PAGED && q.plane >= 0) {
            if (info[r].page < 0) continue;
            dst += info[r].page * q.db + info[r].slot * q.dt;
        } else {
            const int b = PAGED ? 0 : g.by_tokens.div(row0 + r);
            dst += b * q.db + static_cast<int64_t>(row0 + r - (PAGED ? 0 : b * static_cast<int>(a.tokens))) * q.dt;
        }
        if (turn && (!PAGED || q.rotate)) {
            float c[H], s[H];
            const float *cs = trig + 2 * r * a.pairs + u * H, *sn = cs + a.pairs;
#pragma unroll
            for (int j = 0; j < H; j += H % 4 ? 1 : 4) {
                if constexpr (H % 4 == 0) {
                    *reinterpret_cast<float4 *>(c + j) = *reinterpret_cast<const float4 *>(cs + j);
                    *reinterpret_cast<float4 *>(s + j) = *reinterpret_cast<const float4 *>(sn + j);
                } else {
                    c[j] = cs[j];
                    s[j] = sn[j];
                }
            }
            if constexpr (kTwo) turn_two<T, N>(x, y, c, s);
            else turn_one<T, N>(x, c, s);
        }
        store_chunk<T, N>(dst + (N == 1 ? at * q.dd : at), x);
        if (kTwo && turn) store_chunk<T, N>(dst + (N == 1 ? other * q.dd : other), y);
    }
}

bool aligned16(const KvRowsArgs &a, int size) {
    const int n = 16 / size;
    if (a.dim % n || (2 * a.pairs) % n || (!a.interleaved && a.pairs % n)) return false;
    for (int g = 0; g < a.groups; ++g) {
        const KvRowGroup &q = a.group[g];
        if (q.sd != 1 || q.dd != 1) return false;
        const int64_t all = q.sb | q.st | q.sh | q.db | q.dt | q.dh;
        if (all % n) return false;
        if ((reinterpret_cast<uintptr_t>(q.src) | reinterpret_cast<uintptr_t>(q.dst)) & 15u) return false;
    }
    return true;
}

template <typename T, int N, bool I>
int launch_rows(const KvRowsArgs &a, int sms, cudaStream_t st) {
    const int h = I && N > 1 ? N / 2 : N;
    int64_t units = a.pairs / h + (a.dim - 2 * a.pairs) / N, parts = 1;
    if (units > kRowThreads) {  // of a very long head with odd strides: a row of blocks for each part
        parts = (units + kRowThreads - 1) / kRowThreads;
        units = (units + parts - 1) / parts;
    }
    // Rows of a block: one wave of four blocks an SM, so that the places and angles of all rows are found at once,
    // up to what shared memory is taken for sines and cosines (32 KiB); single rows where there are no more.
    const int64_t wave = 4 * static_cast<int64_t>(sms);
    int64_t rows = (a.rows + wave - 1) / wave;
    const int64_t fit = 4096 / (a.pairs > 0 ? a.pairs : 1);
    if (fit < 1 || parts > 65535) return cudaErrorInvalidValue;
    if (rows > fit) rows = fit;
    if (rows > kMaxRowsPerCta) rows = kMaxRowsPerCta;
    if (rows > kMostHeads / a.heads) rows = kMostHeads / a.heads;
    int64_t lanes = kRowThreads / units;
    if (lanes > rows * a.heads) lanes = rows * a.heads;
    const int64_t ctas = (a.rows + rows - 1) / rows;
    const int threads = static_cast<int>((units * lanes + 31) / 32 * 32);
    RowsShape g;
    g.units = static_cast<int>(units);
    g.lanes = static_cast<int>(lanes);
    g.rows = static_cast<int>(rows);
    g.by_units = FastDiv(g.units);
    g.by_heads = FastDiv(a.heads);
    g.by_pairs = FastDiv(a.pairs > 0 ? a.pairs : 1);
    g.by_tokens = FastDiv(static_cast<uint32_t>(a.tokens));
    const dim3 grid(static_cast<unsigned>(ctas), static_cast<unsigned>(parts));
    const size_t smem = static_cast<size_t>(rows) * a.pairs * 8;
    if (a.in_batch) kv_rows_kernel<T, N, I, true><<<grid, threads, smem, st>>>(a, g);
    else kv_rows_kernel<T, N, I, false><<<grid, threads, smem, st>>>(a, g);
    note_launch();
    return static_cast<int>(cudaGetLastError());
}

// A batch whose rows lie evenly through it, in sources, destinations and positions, is one of a single sequence.
void join_batch(KvRowsArgs *a) {
    if (a->tokens == a->rows) return;
    bool even = a->pos_sb == a->tokens * a->pos_st;
    for (int i = 0; i < a->groups; ++i) {
        const KvRowGroup &q = a->group[i];
        even = even && q.sb == a->tokens * q.st && (q.plane >= 0 || q.db == a->tokens * q.dt);
    }
    if (even) a->tokens = a->rows;
}

template <typename T>
int launch_typed(const KvRowsArgs &a, int sms, cudaStream_t st) {
    constexpr int N = 16 / sizeof(T);
    if (aligned16(a, sizeof(T)))
        return a.interleaved ? launch_rows<T, N, true>(a, sms, st) : launch_rows<T, N, false>(a, sms, st);
    return a.interleaved ? launch_rows<T, 1, true>(a, sms, st) : launch_rows<T, 1, false>(a, sms, st);
}

}  // namespace

int kv_rows(const KvRowsArgs &args, int dtype, int device, void *stream) {
    KvRowsArgs a = args;
    if (a.rows <= 0 || a.heads <= 0 || a.dim <= 0) return 0;
    if (a.rows > 0x7fffffff || a.heads > kMostHeads || a.tokens <= 0 || a.tokens > a.rows || a.groups < 1 || a.groups > 3 || (!a.in_batch && a.groups > 1))
        return cudaErrorInvalidValue;
    join_batch(&a);
    DeviceScope on(device);
    if (on.error()) return on.error();
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (dtype) {
        case kBf16: return launch_typed<__nv_bfloat16>(a, sm_count(device), st);
        case kFp16: return launch_typed<__half>(a, sm_count(device), st);
        case kFp32: return launch_typed<float>(a, sm_count(device), st);
    }
    return cudaErrorInvalidValue;
}

}  // namespace kern
}  // namespace mpcomm
