// Rotary positions with several axes, and the write of the turned keys and the values into the
// paged cache, in one launch.
//
// Pair p of a head belongs to axis a(p) and turns by angle = position[t][a] * frequency[p].  The
// frame index of a camera that has run for hours is beyond 10^5, where an angle in fp32 is off by
// 10^-2 rad; so the angle is formed in turns (angle / 2 pi) in 64 bits, its whole turns are dropped
// there, and only the fraction, at most half a turn, goes to fp32 (error 2^-25 of a turn at most).
//
// What bounds it: one read of q, k and v, one write of each -- memory, and at one token the launch.
// The angles do not depend on the head: a workgroup makes those of ROT_TOKENS tokens once, in LDS
// beside the cache rows of their slots, and its threads then walk over (token, head, vector) items
// of 16 bytes (half layout: of both vectors of VE pairs).
#include "cache.hpp"

namespace dc {
namespace {

constexpr int ROT_THREADS = 256;

// Stores that leave no line behind in the L2: nothing here is read again before the attention, by whichever
// XCD (a clip of 32640 tokens x 16 + 2 x 4 heads of 128: 97 us with plain stores, 62 us, 6.5 TB/s, with these).
template <typename T, int N>
__device__ __forceinline__ void pass_on(T *p, const Vec<T, N> &x) {
    if constexpr (sizeof(Vec<T, N>) == 16) __builtin_nontemporal_store(__builtin_bit_cast(u32x4_t, x), reinterpret_cast<u32x4_t *>(p));
    else vstore<T, N>(p, x);
}

struct RotaryPlan {
    int32_t tokens, q_heads, kv_heads, dim, pairs, axes;
    int32_t pair_end[4];  // running pair counts of the axes
    int32_t block_tokens; // tokens of a workgroup
    int32_t uq, ur, uv;   // items of a turned head, those of its rotated part, items of a value head
    int32_t per_token;
    FastDiv by_pairs, by_block, by_token, by_uq, by_uv;
    int64_t qt, qh, ot, oh, kt, kh, vt, vh;
    bool inverse, cache;
    int32_t streams;
    PagePool pool;
};

template <typename T, int VE, bool INTER>
__global__ void __launch_bounds__(ROT_THREADS)
rotary_kernel(RotaryPlan r, const T *__restrict__ q, T *out, const int32_t *__restrict__ positions,
              const double *__restrict__ frequencies, const T *__restrict__ k, const T *__restrict__ v, T *keys, T *values,
              float *weights, int32_t *stamps, const int32_t *__restrict__ token_stamps, const int32_t *__restrict__ slots,
              const int32_t *__restrict__ starts, int32_t *lens, const int32_t *__restrict__ new_lens) {
    extern __shared__ char lds[];
    int64_t *rows = reinterpret_cast<int64_t *>(lds);  // [kv_heads][block_tokens]
    float2 *turn = reinterpret_cast<float2 *>(rows + (r.cache ? r.kv_heads * r.block_tokens : 0));  // [block_tokens][pairs]
    const int t0 = blockIdx.x * r.block_tokens;
    const int nt = min(r.block_tokens, r.tokens - t0);

    for (int i = threadIdx.x; i < nt * r.pairs; i += ROT_THREADS) {
        const int t = int(r.by_pairs.quot(i)), p = i - t * r.pairs;
        int axis = 0;
#pragma unroll
        for (int a = 0; a < 3; ++a) axis += p >= r.pair_end[a] ? 1 : 0;
        const double turns = double(positions[int64_t(t0 + t) * r.axes + axis]) * (frequencies[p] * 0.15915494309189533576888);
        float sn, cs;
        sincospif(2.f * float(turns - rint(turns)), &sn, &cs);
        turn[i] = make_float2(cs, r.inverse ? -sn : sn);
    }
    if (r.cache) {
        for (int i = threadIdx.x; i < r.kv_heads * r.block_tokens; i += ROT_THREADS) {
            const int h = int(r.by_block.quot(i)), t = i - h * r.block_tokens;
            if (t >= nt) continue;
            const int b = stream_of(starts, r.streams, r.tokens, t0 + t);
            int64_t row = -1;
            if (b >= 0)
                row = slot_row(r.pool, r.pool.table + int64_t(b) * r.pool.max_pages, slots[int64_t(h) * r.tokens + t0 + t], r.kv_heads, h);
            rows[i] = row;
            if (row >= 0 && weights != nullptr) weights[row] = 0.f;
            if (row >= 0 && stamps != nullptr)
                stamps[row] = token_stamps != nullptr ? token_stamps[t0 + t] : positions[int64_t(t0 + t) * r.axes];
        }
        if (lens != nullptr && blockIdx.x == 0)
            for (int b = threadIdx.x; b < r.streams; b += ROT_THREADS) lens[b] = new_lens[b];
    }
    __syncthreads();

    const int q_items = r.q_heads * r.uq, k_items = r.cache ? r.kv_heads * r.uq : 0;
    for (int i = threadIdx.x; i < nt * r.per_token; i += ROT_THREADS) {
        const int t = int(r.by_token.quot(i));
        int u = i - t * r.per_token;
        const T *src;
        T *dst;
        if (u >= q_items + k_items) {  // a value vector: copied
            u -= q_items + k_items;
            const int h = int(r.by_uv.quot(u)), c = (u - h * r.uv) * VE;
            const int64_t row = rows[h * r.block_tokens + t];
            if (row >= 0) pass_on<T, VE>(values + row * r.dim + c, vload<T, VE>(v + (t0 + t) * r.vt + h * r.vh + c));
            continue;
        }
        if (u >= q_items) {
            u -= q_items;
            const int h = int(r.by_uq.quot(u));
            u -= h * r.uq;
            const int64_t row = rows[h * r.block_tokens + t];
            if (row < 0) continue;
            src = k + (t0 + t) * r.kt + h * r.kh;
            dst = keys + row * r.dim;
        } else {
            const int h = int(r.by_uq.quot(u));
            u -= h * r.uq;
            src = q + (t0 + t) * r.qt + h * r.qh;
            dst = out + (t0 + t) * r.ot + h * r.oh;
        }
        if (u >= r.ur) {  // behind the rotated part
            const int c = 2 * r.pairs + (u - r.ur) * VE;
            pass_on<T, VE>(dst + c, vload<T, VE>(src + c));
            continue;
        }
        if constexpr (VE == 1) {
            const float2 w = turn[t * r.pairs + u];
            const int ia = INTER ? 2 * u : u, ib = INTER ? 2 * u + 1 : u + r.pairs;
            const float a = float(src[ia]), b = float(src[ib]);
            dst[ia] = T(fmaf(-b, w.y, a * w.x));
            dst[ib] = T(fmaf(b, w.x, a * w.y));
        } else if constexpr (INTER) {
            Vec<T, VE> x = vload<T, VE>(src + u * VE);
#pragma unroll
            for (int j = 0; j < VE / 2; ++j) {
                const float2 w = turn[t * r.pairs + u * (VE / 2) + j];
                const float a = float(x.v[2 * j]), b = float(x.v[2 * j + 1]);
                x.v[2 * j] = T(fmaf(-b, w.y, a * w.x));
                x.v[2 * j + 1] = T(fmaf(b, w.x, a * w.y));
            }
            pass_on<T, VE>(dst + u * VE, x);
        } else {
            Vec<T, VE> x = vload<T, VE>(src + u * VE), y = vload<T, VE>(src + r.pairs + u * VE);
#pragma unroll
            for (int j = 0; j < VE; ++j) {
                const float2 w = turn[t * r.pairs + u * VE + j];
                const float a = float(x.v[j]), b = float(y.v[j]);
                x.v[j] = T(fmaf(-b, w.y, a * w.x));
                y.v[j] = T(fmaf(b, w.x, a * w.y));
            }
            pass_on<T, VE>(dst + u * VE, x);
            pass_on<T, VE>(dst + r.pairs + u * VE, y);
        }
    }
}

template <typename T, int VE, bool INTER>
hipError_t rotary_go(const dc_rotary_args &a, RotaryPlan &r, hipStream_t s) {
    r.ur = INTER && VE > 1 ? 2 * r.pairs / VE : r.pairs / VE;
    r.uq = r.ur + (r.dim - 2 * r.pairs) / VE;
    r.uv = r.dim / VE;
    r.per_token = r.q_heads * r.uq + (r.cache ? r.kv_heads * (r.uq + r.uv) : 0);
    // enough workgroups to spread over the chip, enough items for a workgroup's threads
    int bt = 1;
    while (bt < 16 && bt * r.per_token < 4 * ROT_THREADS && ceil_div(r.tokens, 2 * bt) >= 512) bt *= 2;
    r.block_tokens = bt;
    r.by_pairs = FastDiv(r.pairs);
    r.by_block = FastDiv(bt);
    r.by_token = FastDiv(r.per_token);
    r.by_uq = FastDiv(r.uq);
    r.by_uv = FastDiv(r.uv);
    const size_t lds = size_t(bt) * (size_t(r.pairs) * 8 + (r.cache ? size_t(r.kv_heads) * 8 : 0));
    note_kernel("rotary_kernel");
    rotary_kernel<T, VE, INTER><<<ceil_div(r.tokens, bt), ROT_THREADS, lds, s>>>(
        r, (const T *)a.q, (T *)a.out, a.positions, a.frequencies, (const T *)a.k, (const T *)a.v, (T *)a.keys, (T *)a.values,
        a.weights, a.stamps, a.token_stamps, a.slots, a.starts, a.lens, a.new_lens);
    return hipGetLastError();
}

template <typename T>
hipError_t rotary_t(const dc_rotary_args &a, hipStream_t s) {
    constexpr int N = Vec16<T>::N;
    RotaryPlan r = {};
    r.tokens = a.tokens;
    r.q_heads = a.q_heads;
    r.kv_heads = a.kv_heads;
    r.dim = a.dim;
    r.axes = a.axes;
    int total = 0;
    for (int i = 0; i < 4; ++i) {
        total += i < a.axes ? a.sections[i] / 2 : 0;
        r.pair_end[i] = i + 1 < a.axes ? total : INT32_MAX;
    }
    r.pairs = total;
    r.cache = a.keys != nullptr;
    r.inverse = a.inverse != 0;
    r.qt = a.q_token_stride, r.qh = a.q_head_stride, r.ot = a.out_token_stride, r.oh = a.out_head_stride;
    r.kt = a.k_token_stride, r.kh = a.k_head_stride, r.vt = a.v_token_stride, r.vh = a.v_head_stride;
    uintptr_t bits = uintptr_t(a.q) | uintptr_t(a.out);
    uint64_t odd = uint64_t(r.qt | r.qh | r.ot | r.oh) | uint64_t(r.dim) | uint64_t(a.interleaved ? 2 * r.pairs : r.pairs);
    if (r.cache) {
        r.streams = a.streams;
        r.pool = {a.page_table, a.num_pages, a.page_size, a.max_pages, FastDiv(uint32_t(a.page_size))};
        bits |= uintptr_t(a.k) | uintptr_t(a.v) | uintptr_t(a.keys) | uintptr_t(a.values);
        odd |= uint64_t(r.kt | r.kh | r.vt | r.vh);
    }
    const bool vec = bits % 16 == 0 && odd % N == 0;  // every row and every half in whole 16-byte vectors
    if (vec) return a.interleaved ? rotary_go<T, N, true>(a, r, s) : rotary_go<T, N, false>(a, r, s);
    return a.interleaved ? rotary_go<T, 1, true>(a, r, s) : rotary_go<T, 1, false>(a, r, s);
}

}  // namespace

hipError_t launch_rotary(const dc_rotary_args &a, int dtype, hipStream_t s) {
    if (dtype == DC_F32) return rotary_t<float>(a, s);
    if (dtype == DC_BF16) return rotary_t<bf16_t>(a, s);
    return rotary_t<half_t>(a, s);
}

}  // namespace dc
