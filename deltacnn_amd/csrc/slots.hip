// Which slots of a paged cache give way to new tokens: per stream and kv head the e tokens that have
// received the least attention, in ascending order of their slots, then the slots behind those in use.
//
// The e-th smallest key is found by radix selection on a monotone 32-bit image of the weight (11, 11
// and 10 bits, one LDS histogram each), so every slot is looked at a fixed number of times whatever
// the weights are; counts, not values, decide, so the result does not depend on the order of atomics.
// Protection is folded into the key: with u unprotected tokens and e <= u the protected ones get the
// highest key of all, else the unprotected ones get the lowest (they all go) and the choice is among
// the protected.  Every wavefront owns one contiguous run of slots: its counts below and at the
// threshold, summed over the wavefronts in front, are its write positions, ascending without a sort.
//
// What bounds it: 8 bytes a slot once, and, at these sizes, the chain of dependent passes.
#include "cache.hpp"

namespace dc {
namespace {

constexpr int SLOT_THREADS = 1024;
constexpr int SLOT_WAVES = SLOT_THREADS / WAVE;
constexpr int SLOT_BINS = 2048;

// Monotone image of a weight: -0 = +0, NaN above everything; 0 and ~0 stay free.
__device__ __forceinline__ uint32_t weight_key(float w) {
    if (w != w) return 0xfffffffeu;
    const uint32_t u = __float_as_uint(w + 0.f);
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

struct SlotsPlan {
    PagePool pool;
    int32_t streams, tokens, kv_heads, budget;
};

__global__ void __launch_bounds__(SLOT_THREADS)
cache_slots_kernel(SlotsPlan p, const float *__restrict__ weights, const int32_t *__restrict__ stamps,
                   const int32_t *__restrict__ keep_from, const int32_t *__restrict__ lens, const int32_t *__restrict__ starts,
                   int32_t *__restrict__ slots, int32_t *__restrict__ new_lens) {
    __shared__ uint32_t hist[SLOT_BINS];
    __shared__ uint32_t wave_sum[SLOT_WAVES];
    __shared__ uint32_t wave_sum2[SLOT_WAVES];
    __shared__ uint32_t found[2];
    const int b = blockIdx.x, h = blockIdx.y;
    const int lane = lane_id(), wv = wave_id();
    int first, c;
    stream_tokens(starts, b, p.streams, p.tokens, first, c);
    const int n = min(max(lens[b], 0), int(min(int64_t(p.pool.max_pages) * p.pool.page_size, int64_t(INT32_MAX))));
    const int most = max(p.budget, n);
    const int e = int(max(int64_t(0), min(min(int64_t(n) + c - p.budget, int64_t(n)), int64_t(c))));
    if (h == 0 && threadIdx.x == 0) new_lens[b] = int(min(int64_t(n) + c - e, int64_t(most)));
    int32_t *out = slots + int64_t(h) * p.tokens + first;
    for (int i = e + threadIdx.x; i < c; i += SLOT_THREADS) {
        const int64_t s = int64_t(n) + i - e;
        out[i] = s < most ? int32_t(s) : -1;
    }
    if (e == 0) return;

    const int32_t *table = p.pool.table + int64_t(b) * p.pool.max_pages;
    const int32_t keep = stamps != nullptr ? keep_from[b] : 0;
    // this wavefront's run of slots, in whole rows of 64
    const int run = ((n + SLOT_WAVES - 1) / SLOT_WAVES + WAVE - 1) / WAVE * WAVE;
    const int lo = min(wv * run, n), hi = min(lo + run, n);

    auto is_protected = [&](int s) {
        const int64_t row = slot_row(p.pool, table, s, p.kv_heads, h);
        return row >= 0 && stamps != nullptr && stamps[row] >= keep;
    };
    uint32_t open = 0;
    for (int s = lo + lane; s < hi; s += WAVE) open += is_protected(s) ? 0 : 1;
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) open += __shfl_xor(open, d, WAVE);
    if (lane == 0) wave_sum[wv] = open;
    __syncthreads();
    open = 0;
    for (int i = 0; i < SLOT_WAVES; ++i) open += wave_sum[i];
    const bool among_protected = uint32_t(e) > open;

    auto key_of = [&](int s) -> uint32_t {
        const int64_t row = slot_row(p.pool, table, s, p.kv_heads, h);
        if (row < 0) return 0u;
        const bool prot = stamps != nullptr && stamps[row] >= keep;
        if (prot != among_protected) return prot ? 0xffffffffu : 0u;
        return weight_key(weights[row]);
    };

    // radix selection of the e-th smallest key: `want` counts the rank left inside the bin
    uint32_t prefix = 0, want = uint32_t(e);
    int shift = 21;
    for (int pass = 0; pass < 3; ++pass) {
        const int bits = pass < 2 ? 11 : 10;
        for (int i = threadIdx.x; i < SLOT_BINS; i += SLOT_THREADS) hist[i] = 0;
        __syncthreads();
        for (int s = lo + lane; s < hi; s += WAVE) {
            const uint32_t key = key_of(s);
            if (pass == 0 || (key >> (shift + bits)) == prefix) atomicAdd(&hist[(key >> shift) & ((1u << bits) - 1)], 1u);
        }
        __syncthreads();
        // the bin that holds rank `want`: two bins a thread, a scan over the workgroup
        const uint32_t h0 = hist[2 * threadIdx.x], h1 = hist[2 * threadIdx.x + 1];
        uint32_t sum = h0 + h1;
#pragma unroll
        for (int d = 1; d < WAVE; d <<= 1) {
            const uint32_t o = __shfl_up(sum, d, WAVE);
            if (lane >= d) sum += o;
        }
        if (lane == WAVE - 1) wave_sum[wv] = sum;
        __syncthreads();
        uint32_t before = sum - h0 - h1;
        for (int i = 0; i < wv; ++i) before += wave_sum[i];
        if (before < want && want <= before + h0) found[0] = 2 * threadIdx.x, found[1] = before;
        if (before + h0 < want && want <= before + h0 + h1) found[0] = 2 * threadIdx.x + 1, found[1] = before + h0;
        __syncthreads();
        prefix = (prefix << bits) | found[0];
        want -= found[1];
        shift -= pass == 0 ? 11 : 10;
        __syncthreads();
    }
    // prefix is the threshold; `want` of the keys equal to it go, the lowest slots first
    uint32_t less = 0, same = 0;
    for (int s = lo + lane; s < hi; s += WAVE) {
        const uint32_t key = key_of(s);
        less += key < prefix ? 1 : 0;
        same += key == prefix ? 1 : 0;
    }
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) less += __shfl_xor(less, d, WAVE), same += __shfl_xor(same, d, WAVE);
    if (lane == 0) wave_sum[wv] = less, wave_sum2[wv] = same;
    __syncthreads();
    uint32_t at = 0, eq = 0;
    for (int i = 0; i < wv; ++i) at += wave_sum[i], eq += wave_sum2[i];
    at += min(eq, want);
    for (int s0 = lo; s0 < hi; s0 += WAVE) {
        const int s = s0 + lane;
        const uint32_t key = s < hi ? key_of(s) : 0xffffffffu;
        const bool is_eq = s < hi && key == prefix;
        int neq;
        const uint32_t my_eq = eq + wave_rank(is_eq, neq);
        const bool goes = s < hi && (key < prefix || (is_eq && my_eq < want));
        int ngo;
        const uint32_t pos = at + wave_rank(goes, ngo);
        if (goes && pos < uint32_t(e)) out[pos] = s;
        eq += neq;
        at += ngo;
    }
}

}  // namespace

hipError_t launch_cache_slots(const dc_slots_args &a, hipStream_t s) {
    SlotsPlan p = {};
    p.pool = {a.page_table, a.num_pages, a.page_size, a.max_pages, FastDiv(uint32_t(a.page_size))};
    p.streams = a.streams;
    p.tokens = a.tokens;
    p.kv_heads = a.kv_heads;
    p.budget = a.budget;
    note_kernel("cache_slots_kernel");
    cache_slots_kernel<<<dim3(a.streams, a.kv_heads), SLOT_THREADS, 0, s>>>(p, a.weights, a.stamps, a.keep_from, a.lens, a.starts,
                                                                         a.slots, a.new_lens);
    return hipGetLastError();
}

}  // namespace dc
