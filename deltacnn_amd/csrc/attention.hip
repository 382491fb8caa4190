// Attention of new tokens over a paged cache of earlier frames.
//
// One pass over the visible slots with a running maximum m and sum l of the softmax:
//   m' = max(m, s),  l' = l e^(m - m') + sum e^(s - m'),  o' = o e^(m - m') + sum e^(s - m') v.
// The attention that a slot receives needs the finished log-sum of every row, so it is a second
// launch: weight[s] = decay weight[s] + sum over rows of e^(s - lse).
#include "cache.hpp"

namespace dc {
namespace {

struct AttnPlan {
    PagePool pool;
    int32_t tokens, q_heads, kv_heads, dim, group, streams, causal_block;
    float scale, decay;
    int64_t qt, qh, ot, oh;
};

// Number of visible slots of token i of a stream's `count` (0 <= result <= len).
__device__ __forceinline__ int visible(int len, int count, int i, int block) {
    if (block == 0) return len;
    const int64_t end = int64_t(len) - count + (int64_t(i / block) + 1) * block;
    return int(min(max(end, int64_t(0)), int64_t(len)));
}

__device__ __forceinline__ int stream_len(const AttnPlan &p, const int32_t *lens, int b) {
    return int(min(int64_t(max(lens[b], 0)), int64_t(p.pool.max_pages) * p.pool.page_size));
}

// One wavefront per token and query head; a lane scores one slot and sums four elements of the output.
template <typename T>
__global__ void __launch_bounds__(64)
paged_attention_kernel(AttnPlan p, const T *__restrict__ q, T *__restrict__ out, float *__restrict__ lse,
                       const T *__restrict__ keys, const T *__restrict__ values, const int32_t *__restrict__ lens,
                       const int32_t *__restrict__ starts) {
    __shared__ float prob[WAVE];
    __shared__ int64_t row_of[WAVE];
    const int t = blockIdx.x, head = blockIdx.y, h = head / p.group, lane = lane_id();
    const int b = stream_of(starts, p.streams, p.tokens, t);
    if (b < 0) return;
    int first, count;
    stream_tokens(starts, b, p.streams, p.tokens, first, count);
    const int n = visible(stream_len(p, lens, b), count, t - first, p.causal_block);
    const int32_t *table = p.pool.table + int64_t(b) * p.pool.max_pages;
    const T *qr = q + t * p.qt + head * p.qh;
    float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    bool bad = false;
    for (int s0 = 0; s0 < n; s0 += WAVE) {
        const int s = s0 + lane;
        int64_t row = -1;
        float score = -INFINITY;
        if (s < n) {
            row = slot_row(p.pool, table, s, p.kv_heads, h);
            bad = bad || row < 0;
            if (row >= 0) {
                float sum = 0.f;
                for (int d = 0; d < p.dim; ++d) sum = fmaf(float(qr[d]), float(keys[row * p.dim + d]), sum);
                score = sum * p.scale;
            }
        }
        float top = score;
#pragma unroll
        for (int d = 32; d >= 1; d >>= 1) top = fmaxf(top, __shfl_xor(top, d, WAVE));
        const float m2 = fmaxf(m, top), ref = m2 == -INFINITY ? 0.f : m2;
        const float pr = row < 0 ? 0.f : expf(score - ref), fade = expf(m - ref);
        m = m2;
        l = l * fade + pr;
        prob[lane] = pr;
        row_of[lane] = row;
        __syncthreads();
#pragma unroll
        for (int c = 0; c < 4; ++c) o[c] *= fade;
        for (int j = 0; j < min(WAVE, n - s0); ++j) {
            if (row_of[j] < 0) continue;
#pragma unroll
            for (int c = 0; c < 4; ++c)
                if (c * WAVE + lane < p.dim) o[c] = fmaf(prob[j], float(values[row_of[j] * p.dim + c * WAVE + lane]), o[c]);
        }
        __syncthreads();
    }
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) l += __shfl_xor(l, d, WAVE);
    bad = ballot(bad) != 0;
    const float inv = bad ? NAN : l > 0.f || l != l ? 1.f / l : 0.f;
#pragma unroll
    for (int c = 0; c < 4; ++c)
        if (c * WAVE + lane < p.dim) out[t * p.ot + head * p.oh + c * WAVE + lane] = T(o[c] * inv);
    if (lane == 0 && lse != nullptr) lse[int64_t(t) * p.q_heads + head] = bad ? NAN : l == 0.f ? -INFINITY : m + logf(l);
}

// One thread per slot and kv head: the sum of its probabilities over the rows that share the head.
template <typename T>
__global__ void __launch_bounds__(64)
attention_weights_kernel(AttnPlan p, const T *__restrict__ q, const float *__restrict__ lse, const T *__restrict__ keys,
                         float *__restrict__ weights, const int32_t *__restrict__ lens, const int32_t *__restrict__ starts) {
    const int b = blockIdx.z, h = blockIdx.y, len = stream_len(p, lens, b);
    const int s = blockIdx.x * WAVE + threadIdx.x;
    if (s >= len) return;
    int first, count;
    stream_tokens(starts, b, p.streams, p.tokens, first, count);
    const int64_t row = slot_row(p.pool, p.pool.table + int64_t(b) * p.pool.max_pages, s, p.kv_heads, h);
    if (row < 0) return;
    float received = 0.f;
    for (int i = 0; i < count; ++i) {
        if (s >= visible(len, count, i, p.causal_block)) continue;
        for (int g = 0; g < p.group; ++g) {
            const T *qr = q + (first + i) * p.qt + (h * p.group + g) * p.qh;
            float sum = 0.f;
            for (int d = 0; d < p.dim; ++d) sum = fmaf(float(qr[d]), float(keys[row * p.dim + d]), sum);
            const float z = lse[int64_t(first + i) * p.q_heads + h * p.group + g];
            if (z != -INFINITY) received += expf(sum * p.scale - z);
        }
    }
    weights[row] = p.decay == 0.f ? received : fmaf(p.decay, weights[row], received);
}

template <typename T>
hipError_t attention_t(const dc_attention_args &a, AttnPlan p, hipStream_t s) {
    float *lse = a.lse != nullptr || a.weights == nullptr ? a.lse : (float *)a.workspace;
    note_kernel("paged_attention_kernel");
    paged_attention_kernel<T><<<dim3(p.tokens, p.q_heads), 64, 0, s>>>(p, (const T *)a.q, (T *)a.out, lse, (const T *)a.keys,
                                                                      (const T *)a.values, a.lens, a.starts);
    if (a.weights != nullptr) {
        note_kernel("attention_weights_kernel");
        const int most = int(ceil_div64(int64_t(a.max_pages) * a.page_size, WAVE));
        attention_weights_kernel<T><<<dim3(most, p.kv_heads, p.streams), 64, 0, s>>>(p, (const T *)a.q, lse, (const T *)a.keys,
                                                                                    a.weights, a.lens, a.starts);
    }
    return hipGetLastError();
}

}  // namespace

int64_t paged_attention_workspace(const dc_attention_args &a, int) {
    return a.weights != nullptr && a.lse == nullptr ? int64_t(a.tokens) * a.q_heads * 4 : 0;
}

hipError_t launch_paged_attention(const dc_attention_args &a, int dtype, hipStream_t s) {
    AttnPlan p = {};
    p.pool = {a.page_table, a.num_pages, a.page_size, a.max_pages, FastDiv(uint32_t(a.page_size))};
    p.tokens = a.tokens, p.q_heads = a.q_heads, p.kv_heads = a.kv_heads, p.dim = a.dim, p.group = a.q_heads / a.kv_heads;
    p.streams = a.streams, p.causal_block = a.causal_block, p.scale = a.scale, p.decay = a.decay;
    p.qt = a.q_token_stride, p.qh = a.q_head_stride, p.ot = a.out_token_stride, p.oh = a.out_head_stride;
    if (dtype == DC_F32) return attention_t<float>(a, p, s);
    if (dtype == DC_BF16) return attention_t<bf16_t>(a, p, s);
    return attention_t<half_t>(a, p, s);
}

}  // namespace dc
