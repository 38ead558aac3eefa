// Attention of a ragged batch of new tokens over a paged KV cache.
//
//     out[t, h] = sum_p w_p v_p / sum_p w_p,   w_p = exp(scale * q[t, h] . k_p - m)
//
// over the keys p of the row's sequence that the row sees, m their largest
// score. One warp takes one row and one query head and goes through the keys
// once, with the running maximum and sum; a key's dot product is spread over
// the lanes. A row that sees no key gives zeros, and -inf as log-sum-exp.
#include "kernels/kv.cuh"

namespace mpcomm {
namespace kern {
namespace {

constexpr int kWarps = 8;
constexpr int kMaxDim = 128;

__device__ uint32_t g_attention_status;

template <typename T>
__global__ void __launch_bounds__(kWarps * 32) rows_attention_kernel(const __grid_constant__ PagedAttentionArgs a) {
    const int lane = threadIdx.x & 31;
    const int64_t item = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
    if (item >= a.rows * a.q_heads) return;
    const int64_t row = item / a.q_heads;
    const int h = static_cast<int>(item - row * a.q_heads);
    const KvBatch &k = a.batch;
    constexpr int E = kMaxDim / 32;
    T *out = static_cast<T *>(a.out) + row * a.o_st + h * a.o_sh;
    const int b = sequence_of(k, row);
    if (b < 0) {
        if (!a.fill_tail) return;
        for (int e = lane; e < a.dim; e += 32) out[e] = from_f32<T>(0.f);
        if (a.lse && lane == 0) a.lse[row * a.q_heads + h] = -INFINITY;
        return;
    }
    const int64_t len = k.lens.at(b), at = len - (k.starts.at(b + 1) - row);
    int64_t begin = 0, end = len;
    if (a.causal) end = at + 1 < len ? at + 1 : len;
    if (a.window > 0 && at + 1 - a.window > 0) begin = at + 1 - a.window;
    const int64_t most = k.table_width * k.page_tokens;
    if (end > most) end = most;
    const T *q = static_cast<const T *>(a.q) + row * a.q_st + h * a.q_sh;
    const T *kbase = static_cast<const T *>(a.pool) + (h / (a.q_heads / a.kv_heads)) * a.pool_head;
    float qe[E], acc[E];
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const int e = i * 32 + lane;
        qe[i] = e < a.dim ? to_f32(q[e]) * a.scale : 0.f;
        acc[i] = 0.f;
    }
    float m = -INFINITY, sum = 0.f;
    for (int64_t p = begin; p < end; ++p) {
        const int64_t page = page_of(k, b, p);
        if (page < 0) {
            if (lane == 0) atomicOr(a.status ? a.status : &g_attention_status, kStatusBadIndex);
            continue;
        }
        const T *kp = kbase + page * a.pool_page + (p % k.page_tokens) * a.pool_token;
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i)
            if (i * 32 + lane < a.dim) s += qe[i] * to_f32(kp[i * 32 + lane]);
#pragma unroll
        for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
        const float next = fmaxf(m, s), base = next == -INFINITY ? 0.f : next;
        const float keep = __expf(m - base), w = __expf(s - base);
        sum = sum * keep + w;
        m = next;
#pragma unroll
        for (int i = 0; i < E; ++i)
            if (i * 32 + lane < a.dim) acc[i] = acc[i] * keep + w * to_f32(kp[a.pool_plane + i * 32 + lane]);
    }
    const float inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);
#pragma unroll
    for (int i = 0; i < E; ++i)
        if (i * 32 + lane < a.dim) out[i * 32 + lane] = from_f32<T>(acc[i] * inv);
    if (a.lse && lane == 0) a.lse[row * a.q_heads + h] = sum == 0.f ? -INFINITY : m + logf(sum);
}

}  // namespace

size_t paged_attention_workspace(int64_t, int, int, int, int, int) { return 0; }

int paged_attention(const PagedAttentionArgs &a, int dtype, int device, void *stream) {
    if (a.rows <= 0 || a.q_heads <= 0) return 0;
    if (a.dim <= 0 || a.dim > kMaxDim || a.kv_heads <= 0 || a.q_heads % a.kv_heads) return cudaErrorInvalidValue;
    DeviceScope on(device);
    if (on.error()) return on.error();
    const int64_t ctas = (a.rows * a.q_heads + kWarps - 1) / kWarps;
    if (ctas > 0x7fffffff) return cudaErrorInvalidValue;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == kBf16)
        rows_attention_kernel<__nv_bfloat16><<<static_cast<unsigned>(ctas), kWarps * 32, 0, st>>>(a);
    else if (dtype == kFp16)
        rows_attention_kernel<__half><<<static_cast<unsigned>(ctas), kWarps * 32, 0, st>>>(a);
    else
        return cudaErrorInvalidValue;
    note_launch();
    return static_cast<int>(cudaGetLastError());
}

}  // namespace kern
}  // namespace mpcomm
