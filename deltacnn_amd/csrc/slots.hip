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
// What bounds it: 8 bytes a slot once, and, at these sizes, the chain of dependent passes.  Up to
// 32 slots a thread one workgroup per stream and head reads them once and keeps the keys in registers
// (cache_slots_kernel).  Longer caches are cut into pieces, a workgroup each, and the selection becomes
// four launches that meet in histograms in the workspace (cache_slots_piece_kernel): one workgroup
// alone draws too little from memory (130560 slots x 4 heads: 389 us that way, 8 + 13 + 10 + 12 us in pieces).
// 12544 slots x 8 heads x 32 streams, 256 workgroups at once: 21 us; 3136 slots x 4 heads: 11 us.
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
    int32_t pieces, run;  // pieces of a cache, slots of a wavefront's run in one
    uint32_t *space;      // [stream][head][PIECE_WORDS words of each piece, level by level]
};

// What a stream and head has to do.
struct Job {
    int n, e, c, most;
    int32_t *out;
    const int32_t *table;
    int32_t keep;
};

__device__ __forceinline__ Job make_job(const SlotsPlan &p, const int32_t *lens, const int32_t *starts, const int32_t *stamps,
                                        const int32_t *keep_from, int32_t *slots, int b, int h) {
    Job j;
    int first;
    stream_tokens(starts, b, p.streams, p.tokens, first, j.c);
    j.n = int(min(int64_t(max(lens[b], 0)), int64_t(p.pool.max_pages) * p.pool.page_size));
    j.most = max(p.budget, j.n);
    j.e = int(max(int64_t(0), min(min(int64_t(j.n) + j.c - p.budget, int64_t(j.n)), int64_t(j.c))));
    j.out = slots + int64_t(h) * p.tokens + first;
    j.table = p.pool.table + int64_t(b) * p.pool.max_pages;
    j.keep = stamps != nullptr ? keep_from[b] : 0;
    return j;
}

// The tokens that find room behind the slots in use, and the new length.
__device__ __forceinline__ void place_rest(const Job &j, int b, int h, int32_t *new_lens) {
    if (h == 0 && threadIdx.x == 0) new_lens[b] = int(min(int64_t(j.n) + j.c - j.e, int64_t(j.most)));
    for (int i = j.e + threadIdx.x; i < j.c; i += SLOT_THREADS) {
        const int64_t s = int64_t(j.n) + i - j.e;
        j.out[i] = s < j.most ? int32_t(s) : -1;
    }
}

// Weight keys of 8 slots 64 apart and which of them are protected: all requests of a kind go out together.
struct Eight {
    uint32_t key[8];
    uint32_t prot;
};
__device__ __forceinline__ Eight load_eight(const SlotsPlan &p, const Job &j, const float *weights, const int32_t *stamps, int h, int s0, int end) {
    Eight r;
    int64_t row[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) row[k] = s0 + k * WAVE < end ? slot_row(p.pool, j.table, s0 + k * WAVE, p.kv_heads, h) : -1;
    float w[8];
    int32_t st[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        w[k] = row[k] >= 0 ? weights[row[k]] : 0.f;
        st[k] = stamps != nullptr && row[k] >= 0 ? stamps[row[k]] : INT32_MIN;
    }
    r.prot = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        r.key[k] = row[k] >= 0 ? weight_key(w[k]) : 0u;
        r.prot |= (stamps != nullptr && row[k] >= 0 && st[k] >= j.keep ? 1u : 0u) << k;
    }
    return r;
}
__device__ __forceinline__ uint32_t final_key(uint32_t key, bool prot, bool among_protected) {
    return prot == among_protected ? key : prot ? 0xffffffffu : 0u;
}

// A histogram and the places of its scan for every level, so that a level need not wait for the one before.
// The first one, whose keys share few leading bits, has four copies: four lanes in a row that meet in a bin
// do not wait for each other, and the copies start in different banks.
constexpr int COPY = SLOT_BINS + 16, COPIES = 4;
struct SlotsLds {
    uint32_t hist[COPIES * COPY + 2 * SLOT_BINS];
    uint32_t scan[3][SLOT_WAVES], found[3][2];
    uint32_t wave_sum[SLOT_WAVES], wave_sum2[SLOT_WAVES];
};

// Sum of x[i] over the wavefronts in front of this one (all of them read at once).
__device__ __forceinline__ uint32_t sum_front(const uint32_t *x) {
    const int wv = wave_id();
    uint32_t sum = 0;
#pragma unroll
    for (int i = 0; i < SLOT_WAVES; ++i) sum += i < wv ? x[i] : 0;
    return sum;
}

__device__ __forceinline__ uint32_t block_sum(SlotsLds &l, uint32_t x) {
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) x += __shfl_xor(x, d, WAVE);
    if (lane_id() == 0) l.wave_sum[wave_id()] = x;
    __syncthreads();
    x = 0;
    for (int i = 0; i < SLOT_WAVES; ++i) x += l.wave_sum[i];
    __syncthreads();
    return x;
}

// Bin of rank `want` (1 ..) among the counts h0, h1 of this thread's bins 2 t, 2 t + 1: returns the bin
// and lowers `want` by what lies in front of it.
__device__ __forceinline__ uint32_t find_bin(SlotsLds &l, int level, uint32_t h0, uint32_t h1, uint32_t &want) {
    uint32_t sum = h0 + h1;
    const int lane = lane_id();
#pragma unroll
    for (int d = 1; d < WAVE; d <<= 1) {
        const uint32_t o = __shfl_up(sum, d, WAVE);
        if (lane >= d) sum += o;
    }
    if (lane == WAVE - 1) l.scan[level][wave_id()] = sum;
    __syncthreads();
    const uint32_t before = sum - h0 - h1 + sum_front(l.scan[level]);
    if (before < want && want <= before + h0) l.found[level][0] = 2 * threadIdx.x, l.found[level][1] = before;
    if (before + h0 < want && want <= before + h0 + h1) l.found[level][0] = 2 * threadIdx.x + 1, l.found[level][1] = before + h0;
    __syncthreads();
    want -= l.found[level][1];
    return l.found[level][0];
}

constexpr int level_shift(int level) { return level == 0 ? 21 : level == 1 ? 10 : 0; }
constexpr int level_bits(int level) { return level == 2 ? 10 : 11; }

__device__ __forceinline__ void count_key(uint32_t *hist, int level, uint32_t prefix, uint32_t key) {
    const int shift = level_shift(level), bits = level_bits(level);
    if (level == 0 || (key >> (shift + bits)) == prefix) atomicAdd(&hist[(key >> shift) & ((1u << bits) - 1)], 1u);
}

// This wavefront's 64 slots from s0: those that go are written at `at`, ascending; `eq` counts the slots
// at the threshold so far, of which `want` go.
__device__ __forceinline__ void give(const Job &j, uint32_t threshold, uint32_t want, int s, bool in, uint32_t key, uint32_t &at, uint32_t &eq) {
    const bool is_eq = in && key == threshold;
    int neq, ngo;
    const uint32_t my_eq = eq + wave_rank(is_eq, neq);
    const bool goes = in && (key < threshold || (is_eq && my_eq < want));
    const uint32_t pos = at + wave_rank(goes, ngo);
    if (goes && pos < uint32_t(j.e)) j.out[pos] = s;
    eq += neq;
    at += ngo;
}

// One workgroup per stream and head, 8 EIGHTS slots a thread in registers.
template <int EIGHTS>
__global__ void __launch_bounds__(SLOT_THREADS)
cache_slots_kernel(SlotsPlan p, const float *__restrict__ weights, const int32_t *__restrict__ stamps,
                   const int32_t *__restrict__ keep_from, const int32_t *__restrict__ lens, const int32_t *__restrict__ starts,
                   int32_t *__restrict__ slots, int32_t *__restrict__ new_lens) {
    __shared__ SlotsLds l;
    const int b = blockIdx.x, h = blockIdx.y, lane = lane_id(), wv = wave_id();
    const Job j = make_job(p, lens, starts, stamps, keep_from, slots, b, h);
    place_rest(j, b, h, new_lens);
    if (j.e == 0) return;
    // runs in whole rows of 64, spread over the wavefronts
    const int run = ((j.n + SLOT_WAVES - 1) / SLOT_WAVES + WAVE - 1) / WAVE * WAVE;
    const int lo = min(wv * run, j.n), hi = min(lo + run, j.n);
    for (int i = threadIdx.x; i < COPIES * COPY + 2 * SLOT_BINS; i += SLOT_THREADS) l.hist[i] = 0;
    Eight v[EIGHTS];
    uint32_t open = 0;
#pragma unroll
    for (int i = 0; i < EIGHTS; ++i) {
        v[i] = load_eight(p, j, weights, stamps, h, lo + i * 8 * WAVE + lane, hi);
#pragma unroll
        for (int k = 0; k < 8; ++k) open += lo + (i * 8 + k) * WAVE + lane < hi && !(v[i].prot >> k & 1) ? 1 : 0;
    }
    const bool among_protected = uint32_t(j.e) > block_sum(l, open);
#pragma unroll
    for (int i = 0; i < EIGHTS; ++i)
#pragma unroll
        for (int k = 0; k < 8; ++k) v[i].key[k] = final_key(v[i].key[k], v[i].prot >> k & 1, among_protected);

    uint32_t prefix = 0, want = uint32_t(j.e);
#pragma unroll
    for (int level = 0; level < 3; ++level) {
        uint32_t *hist = level == 0 ? l.hist + (lane & 3) * COPY : l.hist + COPIES * COPY + (level - 1) * SLOT_BINS;
#pragma unroll
        for (int i = 0; i < EIGHTS; ++i)
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (lo + (i * 8 + k) * WAVE + lane < hi) count_key(hist, level, prefix, v[i].key[k]);
        __syncthreads();
        uint32_t h0 = 0, h1 = 0;
        const int t2 = 2 * threadIdx.x;
        if (level == 0) {
#pragma unroll
            for (int c = 0; c < COPIES; ++c) h0 += l.hist[c * COPY + t2], h1 += l.hist[c * COPY + t2 + 1];
        } else {
            h0 = hist[t2], h1 = hist[t2 + 1];
        }
        prefix = prefix << level_bits(level) | find_bin(l, level, h0, h1, want);
    }
    uint32_t less = 0, same = 0;
#pragma unroll
    for (int i = 0; i < EIGHTS; ++i)
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const bool in = lo + (i * 8 + k) * WAVE + lane < hi;
            less += __popcll(ballot(in && v[i].key[k] < prefix));
            same += __popcll(ballot(in && v[i].key[k] == prefix));
        }
    if (lane == 0) l.wave_sum[wv] = less, l.wave_sum2[wv] = same;
    __syncthreads();
    uint32_t eq = sum_front(l.wave_sum2);
    uint32_t at = sum_front(l.wave_sum) + min(eq, want);
#pragma unroll
    for (int i = 0; i < EIGHTS; ++i)
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int s = lo + (i * 8 + k) * WAVE + lane;
            if (lo + (i * 8 + k) * WAVE < hi) give(j, prefix, want, s, s < hi, v[i].key[k], at, eq);
        }
}

// Words of a piece in the workspace: its number of unprotected slots and what is known so far, the first
// level's histograms of the unprotected and of the protected, those of the second and the third level.
constexpr int PIECE_OPEN = 0, PIECE_AMONG = 1, PIECE_PREFIX = 2, PIECE_WANT = 3, PIECE_FRONT = 4;
constexpr int PIECE_L0 = 16, PIECE_L1 = PIECE_L0 + 2 * SLOT_BINS, PIECE_L2 = PIECE_L1 + SLOT_BINS;
constexpr int PIECE_WORDS = PIECE_L2 + SLOT_BINS;

// Launch PHASE of four over (piece, head, stream): the histograms of levels 0, 1 and 2, then the slots.
// Each sums the histogram of the launch before over all pieces and finds the bin for itself.
template <int PHASE>
__global__ void __launch_bounds__(SLOT_THREADS)
cache_slots_piece_kernel(SlotsPlan p, const float *__restrict__ weights, const int32_t *__restrict__ stamps,
                         const int32_t *__restrict__ keep_from, const int32_t *__restrict__ lens, const int32_t *__restrict__ starts,
                         int32_t *__restrict__ slots, int32_t *__restrict__ new_lens) {
    __shared__ SlotsLds l;
    const int piece = blockIdx.x, h = blockIdx.y, b = blockIdx.z, lane = lane_id(), wv = wave_id();
    const Job j = make_job(p, lens, starts, stamps, keep_from, slots, b, h);
    if (PHASE == 0 && piece == 0) place_rest(j, b, h, new_lens);
    if (j.e == 0) return;
    uint32_t *space = p.space + (int64_t(b) * p.kv_heads + h) * p.pieces * PIECE_WORDS, *mine = space + int64_t(piece) * PIECE_WORDS;
    const int t2 = 2 * threadIdx.x;
    const int lo = int(min((int64_t(piece) * SLOT_WAVES + wv) * p.run, int64_t(j.n))), hi = int(min(int64_t(lo) + p.run, int64_t(j.n)));

    // Everything that is read is asked for at once: the first eight slots of a thread (all of them in caches up
    // to 2^19 slots) and the counts of the launch before.
    const Eight front_keys = load_eight(p, j, weights, stamps, h, lo + lane, hi);
    auto eight = [&](int s0) { return s0 == lo ? front_keys : load_eight(p, j, weights, stamps, h, s0 + lane, hi); };

    // What is known so far: whether the choice is among the protected, the threshold's leading bits, its rank
    // among the keys that share them, and how many slots in front of this piece go for certain or (at last)
    // lie at the threshold.  Each launch adds the level of the one before and leaves its piece the sum.
    bool among_protected = false;
    uint32_t prefix = 0, want = uint32_t(j.e), front = 0, eq = 0;
    if constexpr (PHASE > 0) {
        constexpr int KINDS = PHASE == 1 ? 2 : 1, FIRST = PHASE == 1 ? PIECE_L0 : PHASE == 2 ? PIECE_L1 : PIECE_L2;
        uint2 all[KINDS], before[KINDS];
        uint32_t open = 0, open_front = 0;
#pragma unroll
        for (int q = 0; q < KINDS; ++q) all[q] = before[q] = make_uint2(0, 0);
        if (PHASE > 1) among_protected = mine[PIECE_AMONG] != 0, prefix = mine[PIECE_PREFIX], want = mine[PIECE_WANT], front = mine[PIECE_FRONT];
#pragma unroll 8
        for (int i = 0; i < p.pieces; ++i) {
            const uint32_t *from = space + int64_t(i) * PIECE_WORDS;
            if (PHASE == 1 && threadIdx.x == 0) {
                open += from[PIECE_OPEN];
                open_front += i < piece ? from[PIECE_OPEN] : 0;
            }
#pragma unroll
            for (int q = 0; q < KINDS; ++q) {
                const uint2 x = *reinterpret_cast<const uint2 *>(from + FIRST + q * SLOT_BINS + t2);
                all[q].x += x.x, all[q].y += x.y;
                before[q].x += i < piece ? x.x : 0, before[q].y += i < piece ? x.y : 0;
            }
        }
        uint32_t below = 0;
        if (PHASE == 1) {
            open = block_sum(l, open);
            among_protected = uint32_t(j.e) > open;
            if (among_protected) want -= open, below = open_front;
        }
        const uint2 x = among_protected ? all[KINDS - 1] : all[0], y = among_protected ? before[KINDS - 1] : before[0];
        const uint32_t bin = find_bin(l, PHASE - 1, x.x, x.y, want);
        below += (uint32_t(t2) < bin ? y.x : 0) + (uint32_t(t2 + 1) < bin ? y.y : 0);
        front += block_sum(l, below);
        if (PHASE == 3) eq = block_sum(l, (uint32_t(t2) == bin ? y.x : 0) + (uint32_t(t2 + 1) == bin ? y.y : 0));
        prefix = prefix << level_bits(PHASE - 1) | bin;
        if (PHASE < 3 && threadIdx.x == 0)
            mine[PIECE_AMONG] = among_protected, mine[PIECE_PREFIX] = prefix, mine[PIECE_WANT] = want, mine[PIECE_FRONT] = front;
    }
    if constexpr (PHASE < 3) {
        constexpr int HISTS = PHASE == 0 ? 2 : 1;
        for (int i = threadIdx.x; i < HISTS * SLOT_BINS; i += SLOT_THREADS) l.hist[i] = 0;
        __syncthreads();
        uint32_t open = 0;
        for (int s0 = lo; s0 < hi; s0 += 8 * WAVE) {
            const Eight v = eight(s0);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                if (s0 + k * WAVE + lane >= hi) continue;
                const bool prot = v.prot >> k & 1;
                open += prot ? 0 : 1;
                if (PHASE == 0) atomicAdd(&l.hist[(prot ? SLOT_BINS : 0) + (v.key[k] >> level_shift(0))], 1u);
                else if (prot == among_protected) count_key(l.hist, PHASE, prefix, v.key[k]);
            }
        }
        if (PHASE == 0) {
            open = block_sum(l, open);
            if (threadIdx.x == 0) mine[PIECE_OPEN] = open;
        }
        __syncthreads();
        uint32_t *to = mine + (PHASE == 0 ? PIECE_L0 : PHASE == 1 ? PIECE_L1 : PIECE_L2);
        for (int i = threadIdx.x; i < HISTS * SLOT_BINS; i += SLOT_THREADS) to[i] = l.hist[i];
    } else {
        uint32_t less = 0, same = 0;
        for (int s0 = lo; s0 < hi; s0 += 8 * WAVE) {
            const Eight v = eight(s0);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const bool in = s0 + k * WAVE + lane < hi;
                const uint32_t key = final_key(v.key[k], v.prot >> k & 1, among_protected);
                less += __popcll(ballot(in && key < prefix));
                same += __popcll(ballot(in && key == prefix));
            }
        }
        if (lane == 0) l.wave_sum[wv] = less, l.wave_sum2[wv] = same;
        __syncthreads();
        eq += sum_front(l.wave_sum2);
        uint32_t at = front + sum_front(l.wave_sum) + min(eq, want);
        for (int s0 = lo; s0 < hi; s0 += 8 * WAVE) {
            const Eight v = eight(s0);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int s = s0 + k * WAVE + lane;
                give(j, prefix, want, s, s < hi, final_key(v.key[k], v.prot >> k & 1, among_protected), at, eq);
            }
        }
    }
}

// Slots that one workgroup keeps in registers at most.
constexpr int64_t ONE_GROUP = 32 * SLOT_THREADS;

void plan_pieces(const dc_slots_args &a, int &pieces, int &run) {
    const int64_t cap = int64_t(a.max_pages) * a.page_size;
    run = 8 * WAVE;
    while (ceil_div64(cap, int64_t(run) * SLOT_WAVES) > 64) run *= 2;
    pieces = int(ceil_div64(cap, int64_t(run) * SLOT_WAVES));
}

}  // namespace

int64_t cache_slots_workspace(const dc_slots_args &a) {
    if (int64_t(a.max_pages) * a.page_size <= ONE_GROUP) return 0;
    int pieces, run;
    plan_pieces(a, pieces, run);
    return int64_t(a.streams) * a.kv_heads * pieces * PIECE_WORDS * 4;
}

hipError_t launch_cache_slots(const dc_slots_args &a, hipStream_t s) {
    SlotsPlan p = {};
    p.pool = {a.page_table, a.num_pages, a.page_size, a.max_pages, FastDiv(uint32_t(a.page_size))};
    p.streams = a.streams;
    p.tokens = a.tokens;
    p.kv_heads = a.kv_heads;
    p.budget = a.budget;
    const int64_t cap = int64_t(a.max_pages) * a.page_size;
    if (cap <= ONE_GROUP) {
        const dim3 grid(a.streams, a.kv_heads);
        note_kernel("cache_slots_kernel");
#define DC_SLOTS_GO(E) cache_slots_kernel<E><<<grid, SLOT_THREADS, 0, s>>>(p, a.weights, a.stamps, a.keep_from, a.lens, a.starts, a.slots, a.new_lens)
        if (cap <= 8 * SLOT_THREADS) DC_SLOTS_GO(1);
        else if (cap <= 16 * SLOT_THREADS) DC_SLOTS_GO(2);
        else DC_SLOTS_GO(4);
#undef DC_SLOTS_GO
        return hipGetLastError();
    }
    plan_pieces(a, p.pieces, p.run);
    p.space = (uint32_t *)a.workspace;
    const dim3 grid(p.pieces, a.kv_heads, a.streams);
    note_kernel("cache_slots_piece_kernel");
    cache_slots_piece_kernel<0><<<grid, SLOT_THREADS, 0, s>>>(p, a.weights, a.stamps, a.keep_from, a.lens, a.starts, a.slots, a.new_lens);
    cache_slots_piece_kernel<1><<<grid, SLOT_THREADS, 0, s>>>(p, a.weights, a.stamps, a.keep_from, a.lens, a.starts, a.slots, a.new_lens);
    cache_slots_piece_kernel<2><<<grid, SLOT_THREADS, 0, s>>>(p, a.weights, a.stamps, a.keep_from, a.lens, a.starts, a.slots, a.new_lens);
    cache_slots_piece_kernel<3><<<grid, SLOT_THREADS, 0, s>>>(p, a.weights, a.stamps, a.keep_from, a.lens, a.starts, a.slots, a.new_lens);
    return hipGetLastError();
}

}  // namespace dc
