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
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "kernels/kv.cuh"

namespace mpcomm {
namespace kern {
namespace {

constexpr int kRowThreads = 256;
constexpr int kMaxRowsPerCta = 32;

template <typename T, int N>
struct alignas(N == 1 ? sizeof(T) : 16) Chunk {
    T e[N];
};

// Loads / stores N elements; N > 1 is one aligned 16-byte access, N == 1 an element.
template <typename T, int N>
__device__ __forceinline__ Chunk<T, N> load_chunk(const T *p) {
    return *reinterpret_cast<const Chunk<T, N> *>(p);
}
template <typename T, int N>
__device__ __forceinline__ void store_chunk(T *p, const Chunk<T, N> &c) {
    *reinterpret_cast<Chunk<T, N> *>(p) = c;
}

struct RowInfo {
    int64_t page;  // -1: the row has no slot (padding, no page); paged groups skip it
    int32_t slot;
    int32_t live;  // 0: padding behind the last sequence, nothing is written
    double pos;
};

// Where row `row` goes. Everything read from the batch's tables is checked
// against the rows, pages and columns there are.
__device__ __forceinline__ RowInfo place_row(const KvRowsArgs &a, int64_t row, uint32_t *status) {
    RowInfo r{-1, 0, 1, 0.0};
    if (a.in_batch) {
        const KvBatch &k = a.batch;
        const int b = sequence_of(k, row);
        if (b < 0) {
            r.live = 0;
            return r;
        }
        const int64_t p = k.lens.at(b) - (k.starts.at(b + 1) - row);
        r.pos = static_cast<double>(p);
        r.page = page_of(k, b, p);
        r.slot = r.page >= 0 ? static_cast<int32_t>(p % k.page_tokens) : 0;
        if (r.page < 0) atomicOr(status, kStatusBadIndex);
    }
    if (a.positions.ptr) {
        const int64_t b = row / a.tokens, t = row - b * a.tokens;
        r.pos = static_cast<double>(a.positions.at(b * a.pos_sb + t * a.pos_st));
    }
    return r;
}

__device__ uint32_t g_rows_status;

// Block: x = unit of a head (N pairs, or N copied elements), y = head lane,
// z = row. N > 1 needs unit element strides, 16-byte aligned bases and
// strides and pairs, dim multiples of N (of N / 2 for interleaved pairs).
template <typename T, int N, bool INTERLEAVED>
__global__ void __launch_bounds__(kRowThreads) kv_rows_kernel(const __grid_constant__ KvRowsArgs a) {
    extern __shared__ float trig[];  // [rows][2][pairs]: cosines, sines
    __shared__ RowInfo info[kMaxRowsPerCta];
    const int rows_cta = blockDim.z;
    const int64_t row0 = static_cast<int64_t>(blockIdx.x) * rows_cta;
    const int threads = blockDim.x * blockDim.y * blockDim.z;
    const int tid = threadIdx.x + blockDim.x * (threadIdx.y + blockDim.y * threadIdx.z);
    uint32_t *status = a.status ? a.status : &g_rows_status;
    if (tid < rows_cta && row0 + tid < a.rows) info[tid] = place_row(a, row0 + tid, status);
    __syncthreads();
    for (int i = tid; i < rows_cta * a.pairs; i += threads) {
        const int r = i / a.pairs, p = i - r * a.pairs;
        if (row0 + r >= a.rows) break;
        const double f = a.freq_f64 ? static_cast<const double *>(a.inv_freq)[p]
                                    : static_cast<double>(static_cast<const float *>(a.inv_freq)[p]);
        double turns = info[r].pos * (f * 0.15915494309189533577);  // 1 / (2 pi)
        turns -= rint(turns);
        float s, c;
        sincospif(static_cast<float>(2.0 * turns), &s, &c);
        trig[(2 * r) * a.pairs + p] = c * a.magnitude;
        trig[(2 * r + 1) * a.pairs + p] = s * a.magnitude * a.sign;
    }
    __syncthreads();

    const int r = threadIdx.z;
    const int64_t row = row0 + r;
    if (row >= a.rows || !info[r].live) return;
    constexpr int H = INTERLEAVED && N > 1 ? N / 2 : N;  // pairs of a rotating unit
    const int turning = a.pairs / H;
    const int copied = (a.dim - 2 * a.pairs) / N;
    const float *cs = trig + 2 * r * a.pairs, *sn = cs + a.pairs;
    const int64_t b = row / a.tokens, t = row - b * a.tokens;
    for (int u = threadIdx.x; u < turning + copied; u += blockDim.x) {
        const bool turn = u < turning;
        float c[H], s[H];
        if (turn) {
#pragma unroll
            for (int j = 0; j < H; ++j) {
                c[j] = cs[u * H + j];
                s[j] = sn[u * H + j];
            }
        }
        const int copy_at = 2 * a.pairs + (u - turning) * N;
        for (int h = threadIdx.y + blockIdx.y * blockDim.y; h < a.heads; h += blockDim.y * gridDim.y) {
            int g = 0, hg = h;
            while (hg >= a.group[g].heads) hg -= a.group[g++].heads;
            const KvRowGroup &q = a.group[g];
            const T *src = static_cast<const T *>(q.src) + b * q.sb + t * q.st + hg * q.sh;
            T *dst = static_cast<T *>(q.dst);
            if (q.plane >= 0) {
                if (info[r].page < 0) continue;
                dst += info[r].page * q.db + info[r].slot * q.dt + hg * q.dh;
            } else {
                dst += b * q.db + t * q.dt + hg * q.dh;
            }
            if (turn && INTERLEAVED) {
                if (N == 1) {
                    const float x = to_f32(src[2 * u * q.sd]), y = to_f32(src[(2 * u + 1) * q.sd]);
                    const bool rot = q.rotate;
                    dst[2 * u * q.dd] = from_f32<T>(rot ? x * c[0] - y * s[0] : x);
                    dst[(2 * u + 1) * q.dd] = from_f32<T>(rot ? y * c[0] + x * s[0] : y);
                } else {
                    Chunk<T, N> v = load_chunk<T, N>(src + u * N);
                    if (q.rotate) {
#pragma unroll
                        for (int j = 0; j < H; ++j) {
                            const int e = N > 1 ? 2 * j : 0;
                            const float x = to_f32(v.e[e]), y = to_f32(v.e[e + (N > 1)]);
                            v.e[e] = from_f32<T>(x * c[j] - y * s[j]);
                            v.e[e + (N > 1)] = from_f32<T>(y * c[j] + x * s[j]);
                        }
                    }
                    store_chunk<T, N>(dst + u * N, v);
                }
            } else if (turn) {
                Chunk<T, N> v = load_chunk<T, N>(src + u * N * q.sd);
                Chunk<T, N> w = load_chunk<T, N>(src + (a.pairs + u * N) * q.sd);
                if (q.rotate) {
#pragma unroll
                    for (int j = 0; j < N; ++j) {
                        const float x = to_f32(v.e[j]), y = to_f32(w.e[j]);
                        v.e[j] = from_f32<T>(x * c[j] - y * s[j]);
                        w.e[j] = from_f32<T>(y * c[j] + x * s[j]);
                    }
                }
                store_chunk<T, N>(dst + u * N * q.dd, v);
                store_chunk<T, N>(dst + (a.pairs + u * N) * q.dd, w);
            } else {
                store_chunk<T, N>(dst + copy_at * q.dd, load_chunk<T, N>(src + copy_at * q.sd));
            }
        }
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
int launch_rows(const KvRowsArgs &a, cudaStream_t st) {
    const int h = I && N > 1 ? N / 2 : N;
    const int units = a.pairs / h + (a.dim - 2 * a.pairs) / N;
    dim3 block;
    block.x = units < kRowThreads ? units : kRowThreads;
    int lanes = kRowThreads / block.x;
    if (lanes > a.heads) lanes = a.heads;
    block.y = lanes;
    int rows = kRowThreads / (block.x * block.y);
    const int fit = 32768 / (a.pairs > 0 ? 8 * a.pairs : 8);  // trig table of at most 32 KiB
    if (rows > fit) rows = fit;
    if (rows > kMaxRowsPerCta) rows = kMaxRowsPerCta;
    if (rows < 1) rows = 1;
    block.z = rows;
    const int64_t ctas = (a.rows + rows - 1) / rows;
    if (ctas > 0x7fffffff) return cudaErrorInvalidValue;
    const dim3 grid(static_cast<unsigned>(ctas), 1, 1);
    kv_rows_kernel<T, N, I><<<grid, block, static_cast<size_t>(rows) * a.pairs * 8, st>>>(a);
    note_launch();
    return static_cast<int>(cudaGetLastError());
}

template <typename T>
int launch_typed(const KvRowsArgs &a, cudaStream_t st) {
    constexpr int N = 16 / sizeof(T);
    if (aligned16(a, sizeof(T)))
        return a.interleaved ? launch_rows<T, N, true>(a, st) : launch_rows<T, N, false>(a, st);
    return a.interleaved ? launch_rows<T, 1, true>(a, st) : launch_rows<T, 1, false>(a, st);
}

}  // namespace

int kv_rows(const KvRowsArgs &a, int dtype, int device, void *stream) {
    if (a.rows <= 0 || a.heads <= 0 || a.dim <= 0) return 0;
    DeviceScope on(device);
    if (on.error()) return on.error();
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (dtype) {
        case kBf16: return launch_typed<__nv_bfloat16>(a, st);
        case kFp16: return launch_typed<__half>(a, st);
        case kFp32: return launch_typed<float>(a, st);
    }
    return cudaErrorInvalidValue;
}

}  // namespace kern
}  // namespace mpcomm
