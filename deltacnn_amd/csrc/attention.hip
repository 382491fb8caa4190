// Attention of new tokens over a paged cache of earlier frames.
//
// One pass over the visible slots with a running maximum m and sum l of the softmax:
//   m' = max(m, s),  l' = l e^(m - m') + sum e^(s - m'),  o' = o e^(m - m') + sum e^(s - m') v.
// The attention that a slot receives needs the finished log-sum of every row, so it is a second
// launch: weight[s] = decay weight[s] + sum over rows of e^(s - lse).
//
// What bounds it, and what it reaches (MI355X; a large copy moves 5.2 TB/s, a large matrix product makes 1200 TFLOP/s in
// bf16 and 150 in fp32; single kernels: medians under the profiler, where those bound by the matrix cores run slower):
//   a token of 32 streams over 18360 .. 32640 slots, 2 kv heads of 128, bf16: reading the cache; 145 + 7 us, 5.8 TB/s
//   12240 tokens in 24 frames, 16 query and 4 kv heads of 128, bf16: the matrix cores; a call 612 us, 1.04 PFLOP/s
//   510 tokens over 32640 slots, the same heads: the matrix cores; 160 us, joining 12 us, weights 119 us, a call 247 us
//   64 tokens of 4 streams over 4096 slots, 8 heads of 64, fp32: the matrix cores; 29 + 5 us, weights 21 us
//   49 tokens over 3136 slots, 20 query and 4 kv heads of 64: its launches and the way through one tile; 9 + 5 us
#include "cache.hpp"

namespace dc {
namespace {

struct AttnPlan {
    PagePool pool;
    int32_t tokens, q_heads, kv_heads, dim, group, streams, causal_block;
    float scale, decay;
    uint32_t flip;  // sign bits of the elements in 32 bits, or 0
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
// A value that is the same in all lanes, as a scalar.
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

typedef float float16_t __attribute__((ext_vector_type(16)));
typedef float float2v_t __attribute__((ext_vector_type(2)));
typedef half_t half2v_t __attribute__((ext_vector_type(2)));
typedef bf16_t bf16x2_t __attribute__((ext_vector_type(2)));
typedef short short4_t __attribute__((ext_vector_type(4)));
#define DC_LDS(T) __attribute__((address_space(3))) T

// 32 x 32 outputs, 16 reduction elements.  Operand A: lane (half, m) holds A[m][8 half + i]; operand B the
// same of its columns; result: lane (half, n) holds rows 8 (r / 4) + 4 half + r % 4 of column n, r = 0 .. 15.
__device__ __forceinline__ float16_t mfma32(half8_t a, half8_t b, float16_t c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ float16_t mfma32(bf16x8_t a, bf16x8_t b, float16_t c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }

__device__ __forceinline__ uint32_t pack2(float a, float b, half_t) { return __builtin_bit_cast(uint32_t, __builtin_convertvector((float2v_t{a, b}), half2v_t)); }
__device__ __forceinline__ uint32_t pack2(float a, float b, bf16_t) { return __builtin_bit_cast(uint32_t, __builtin_convertvector((float2v_t{a, b}), bf16x2_t)); }

// A 16-byte operand chunk of each type and what it does in a product: one instruction over 2 x 8 elements
// for the 16-bit types, four over 2 x 1 in fp32 (element i of both halves' chunks: the order of a
// sum's terms is free as long as both operands keep it).
template <typename E>
struct Chunk {
    static constexpr int N = 8;
    typedef typename Elem16<E>::v8 v;
    typedef typename Elem16<E>::v4 v4;
    static __device__ __forceinline__ float16_t mma(v a, v b, float16_t c) { return mfma32(a, b, c); }
};
template <>
struct Chunk<float> {
    static constexpr int N = 4;
    typedef float4_t v, v4;
    static __device__ __forceinline__ float16_t mma(v a, v b, float16_t c) {
#pragma unroll
        for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b[i], c, 0, 0, 0);
        return c;
    }
};

// The sign bit of each infinite or NaN element of a 32-bit word: zero elements of the complemented exponents
// (an element behind a zero one would have to be 1 to be taken for zero too, and exponents have no bit there).
template <typename E>
__device__ __forceinline__ uint32_t odd_bits(uint32_t w) {
    constexpr uint32_t EXPONENT = sizeof(E) == 4 ? 0x7f800000u : __is_same(E, half_t) ? 0x7c007c00u : 0x7f807f80u;
    constexpr uint32_t ONES = sizeof(E) == 4 ? 1u : 0x00010001u, SIGNS = sizeof(E) == 4 ? 0x80000000u : 0x80008000u;
    const uint32_t x = (w & EXPONENT) ^ EXPONENT;
    return (x - ONES) & ~x & SIGNS;
}
template <typename E>
__device__ __forceinline__ uint32_t without_odd(uint32_t w) {
    const uint32_t b = odd_bits<E>(w);
    return w & ~(sizeof(E) == 4 ? 0u - (b >> 31) : (b >> 15) * 0xffffu);
}

// The larger of the two halves' values, in both.
__device__ __forceinline__ float max_halves(float x) {
    const uint32_t u = __float_as_uint(x);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_halves(float x) {
    const uint32_t u = __float_as_uint(x);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

__device__ const uint4 zero_chunk = {0, 0, 0, 0};

// Exponentials are formed as 2^(score - m) with m up to LIFT below a row's largest score.  The second product's
// operand in fp16 has no value between 0 and 2^-24, so many small probabilities beside a large one would
// leave the sum of values and stay in the normaliser (2^19 slots 17.4 below one: off by 0.015); formed from 2^7 down, what
// is lost begins at 2^-32 of a row's largest.
template <typename E>
constexpr float LIFT = __is_same(E, half_t) ? 7.f : 0.f;

// Log-sum of a row from its m and the sum l of its exponentials; LIFT cancels first, which leaves a single term exact.
template <typename E>
__device__ __forceinline__ float log_sum(float m, float l) {
    if (l == 0.f) return -INFINITY;
    const float top = m == -INFINITY ? 0.f : m + LIFT<E>;
    return (top + __builtin_amdgcn_logf(l * (1.f / float(1 << int(LIFT<E>))))) * 0.693147180559945309f;
}

// Where a workgroup's rows and slots are.  A ROW is one (token, head of the group) pair of a stream and
// kv head: row r is token r / group, query head h * group + r % group, so the heads that share keys
// share their tiles too.
struct AttnGrid {
    int32_t block_rows;     // rows of a workgroup
    int32_t stream_blocks;  // row blocks of a stream (no starts)
    int32_t flat;           // row blocks of all streams (an upper bound with starts)
    int32_t splits;         // pieces of the slot axis
    int32_t split_keys;     // slots of a piece
    int32_t unit;           // consecutive row blocks that run on one XCD
    int32_t pairs;          // heads x pieces
    FastDiv by_group, by_unit, by_pairs, by_blocks, by_kv;
    float *part;            // [splits][T * q_heads][dim] sums over a piece, [splits][T * q_heads][2] their maximum and normaliser behind
};

template <bool B>
struct Flag {
    static constexpr bool value = B;
};

struct Work {
    int b, h, split, rb, first, count;
};

// Row block f of all streams -> stream and block, a wavefront at a time over the streams.
__device__ __forceinline__ bool find_block(const int32_t *starts, const AttnPlan &p, const AttnGrid &g, int f, Work &w) {
    if (starts == nullptr) {
        w.b = int(g.by_blocks.quot(f));
        w.rb = f - w.b * g.stream_blocks;
        w.count = p.tokens / p.streams;
        w.first = w.b * w.count;
    } else {
        int base = 0;
        bool hit = false;
        for (int b0 = 0; b0 < p.streams && !hit; b0 += WAVE) {
            const int b = b0 + lane_id();
            int first = 0, count = 0;
            if (b < p.streams) stream_tokens(starts, b, p.streams, p.tokens, first, count);
            const int nb = int((int64_t(count) * p.group + g.block_rows - 1) / g.block_rows);
            int sum = nb;
#pragma unroll
            for (int d = 1; d < WAVE; d <<= 1) {
                const int o = __shfl_up(sum, d, WAVE);
                if (lane_id() >= d) sum += o;
            }
            const bool mine = f >= base + sum - nb && f < base + sum;
            const uint64_t who = ballot(mine);
            if (who != 0) {
                const int l = __ffsll((unsigned long long)who) - 1;
                w.b = b0 + l;
                w.rb = f - (base + __shfl(sum - nb, l, WAVE));
                w.first = __shfl(first, l, WAVE);
                w.count = __shfl(count, l, WAVE);
                hit = true;
            }
            base += __shfl(sum, WAVE - 1, WAVE);
        }
        if (!hit) return false;
    }
    return true;
}

// Workgroups go to the 8 XCDs in turn, each with an L2 of its own: units of consecutive row blocks, which
// read the same keys and values, stay on one.  With a causal mask a stream's row blocks are counted from
// its end and every head's come before the next unit's, so that the longest start first (a 12240-token
// clip: the longest of 1532 workgroups takes half of the time that all of them need); every other
// round of units goes backwards over the XCDs, which evens out their sums.
__device__ __forceinline__ bool find_work(const int32_t *starts, const AttnPlan &p, const AttnGrid &g, Work &w) {
    const int x = blockIdx.x & 7, j = blockIdx.x >> 3;
    const int round = int(g.by_unit.quot(j));
    const int u = (round & 1 ? 7 - x : x) + 8 * round;
    const int group = int(g.by_pairs.quot(u)), pair = u - group * g.pairs;
    const int f = group * g.unit + (j - round * g.unit);
    if (f >= g.flat) return false;
    w.split = int(g.by_kv.quot(pair));
    w.h = pair - w.split * p.kv_heads;
    if (!find_block(starts, p, g, f, w)) return false;
    if (p.causal_block != 0) {  // the longest rows first
        const int blocks = int((int64_t(w.count) * p.group + g.block_rows - 1) / g.block_rows);
        w.rb = blocks - 1 - w.rb;
    }
    w.b = __builtin_amdgcn_readfirstlane(w.b), w.rb = __builtin_amdgcn_readfirstlane(w.rb), w.h = __builtin_amdgcn_readfirstlane(w.h);
    w.split = __builtin_amdgcn_readfirstlane(w.split);
    w.first = __builtin_amdgcn_readfirstlane(w.first), w.count = __builtin_amdgcn_readfirstlane(w.count);
    return true;
}

// 16 bytes a lane from memory straight into LDS: lane l's go to `to` + 16 l.  Written as assembly because
// the compiler, which knows such a request of its own making for a write to LDS, waits for all of them in
// front of every transposing read (it cannot tell the two stages apart): that wait cost a third of the
// kernel's time.  There is no output register; arrived() below is the wait, in front of every barrier or read
// that needs the data.
__device__ __forceinline__ uint32_t lds_place(const char *to) { return uint32_t(__builtin_amdgcn_readfirstlane(uint32_t(uintptr_t((DC_LDS(const char) *)to)))); }
template <typename V>
__device__ __forceinline__ V lds_read(uint32_t at) {
    return *(DC_LDS(const V) *)(uintptr_t)at;
}
__device__ __forceinline__ void fetch_bounded(u32x4_t resource, uint32_t offset, uint32_t to) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(offset), "s"(resource), "s"(to) : "memory");
}
__device__ __forceinline__ void fetch(const void *from, uint32_t to) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(from), "s"(to) : "memory");
}
__device__ __forceinline__ void arrived() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
// The loads that the compiler knows of: waited for in front of a loop they do not make it wait in there, where
// it would be for the newest requests above.
__device__ __forceinline__ void loaded() { __builtin_amdgcn_s_waitcnt(0x0f70); }  // vmcnt(0)
// .. all but the newest N requests
template <int N>
__device__ __forceinline__ void arrived_but() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// Where 16-byte chunk c of row r of a tile lies: at place c ^ swizzle(r) of the row.  The LDS serves 256 bytes a
// cycle from 64 banks: of keys 16 rows' chunks side by side, of values 32 lanes of the transposing read,
// 64 bytes of each of four consecutive rows.  Both hit every bank once this way.  fp32 values are read as
// words along a row.
template <typename E, int DP>
__device__ __forceinline__ int key_swizzle(int row) {
    return DP * int(sizeof(E)) >= 256 ? row & 15 : row >> 1 & 7;
}
template <typename E, int DP>
__device__ __forceinline__ int value_swizzle(int row) {
    return sizeof(E) == 4 ? 0 : DP >= 128 ? (row & 3) << 2 : (row & 2) << 1;
}

// How many pages a tile of slots may touch: in ONE its rows follow each other, in TWO there is one seam, and
// the pages' numbers are the same for all lanes; only for MANY does every row look for its page.
enum Pages { ONE, TWO, MANY };

// BN slots of one head on their way into LDS.  The lanes choose what they fetch, the places they fill are
// fixed.  What lies behind `end` or in no page of the pool, and the elements from dim to DP, arrive as
// zeros: from the bound of the buffer resource (ONE), else from a chunk of zeros.
template <typename E, int DP, int BN, int LOADERS, Pages PAGES>
struct TileLoader {
    static constexpr int N = Chunk<E>::N, CPR = DP / N, RPI = WAVE / CPR, REQ = BN / RPI / LOADERS;
    static_assert(REQ >= 1, "one request a wavefront at least");
    const int32_t *table;
    const E *keys, *values;  // ONE, TWO: from this head's first row of a page
    int dim, h, page_size, num_pages;
    bool bad = false;
    // ONE, TWO: bytes of a lane from the tile's first element; the tile to be found next: its page (ONE, `fresh`:
    // not looked at yet) and the one behind it, the bytes in front in the pool, its place inside
    // Bytes of every request in registers, or (long rows, whose sums need them) formed when it goes out: a token of 8
    // streams over 4096 slots, 8 heads of 256, bf16 148 -> 42 us, fp32 1125 -> 424 us.
    static constexpr bool KEPT = REQ <= 8;
    uint32_t koffset[KEPT ? REQ : 1], voffset[KEPT ? REQ : 1], page_bytes, row_bytes;
    int index, inside, page, behind;
    uint64_t page_at;
    bool fresh, lost;
    static constexpr uint32_t NOWHERE = 0x40000000u;  // behind any tile: elements from dim on

    __device__ __forceinline__ void init(const AttnPlan &p, const int32_t *table_, const E *k, const E *v, int h_, int loader, int k0) {
        table = table_, dim = p.dim, h = h_, page_size = p.pool.page_size, num_pages = p.pool.num_pages;
        const int64_t head = PAGES != MANY ? int64_t(h) * page_size * dim : 0;
        keys = k + head, values = v + head;
        if constexpr (PAGES != MANY) {
            row_bytes = uint32_t(dim) * sizeof(E);
            page_bytes = uint32_t(p.kv_heads) * page_size * row_bytes;
            index = uniform(p.pool.by_page.quot(uint32_t(k0)));
            inside = uniform(k0 - index * page_size);
            page = behind = 0, page_at = 0, fresh = true, lost = false;
            if constexpr (KEPT) {
#pragma unroll
                for (int j = 0; j < REQ; ++j) koffset[j] = form<false>(lane_id(), loader, j), voffset[j] = form<true>(lane_id(), loader, j);
            }
        }
    }
    template <bool VALUES>
    __device__ __forceinline__ uint32_t form(int lane, int loader, int j) const {
        const int row = loader * REQ * RPI + lane / CPR + j * RPI, c = lane % CPR ^ (VALUES ? value_swizzle<E, DP>(row) : key_swizzle<E, DP>(row));
        return c * N < dim ? uint32_t(row) * row_bytes + uint32_t(c) * 16 : NOWHERE;
    }
    template <bool VALUES>
    __device__ __forceinline__ uint32_t offset(int lane, int loader, int j) const {
        if constexpr (KEPT) return VALUES ? voffset[j] : koffset[j];
        else return form<VALUES>(lane, loader, j);
    }
    // The pages of the next tile, which starts at slot k, a step ahead of its request.  (Nothing writes the table
    // meanwhile: scalar loads, which the counted waits do not see.)
    __device__ __forceinline__ void look(int k, int end) {
        if constexpr (PAGES != MANY) {
            const auto *at = (const __attribute__((address_space(4))) int32_t *)(table + index);
            if (PAGES == TWO || fresh) page = at[0];
            if (PAGES == TWO && k + min(BN, page_size - inside) < min(k + BN, end)) behind = at[1];
        }
    }
    __device__ __forceinline__ void advance(int by) {
        if constexpr (PAGES != MANY) {
            inside += by;
            while (inside >= page_size) inside -= page_size, ++index, fresh = true;
        }
    }
    // Where a tile's rows are: ONE its bytes from the head's first page and how many are in use; TWO the same for the
    // rows up to the seam and behind it, and the rows in use of both; MANY a row of each request (or -1).
    struct Place {
        uint64_t at, at_behind;
        uint32_t bytes;
        int seam, rows, rows_behind;
        int64_t row[PAGES == MANY ? REQ : 1];
    };
    // Slots [k0, end); behind `end` nothing
    __device__ __forceinline__ Place find(const AttnPlan &p, int loader, int k0, int end) {
        Place x;
        if constexpr (PAGES == ONE) {
            if (fresh && k0 < end) {
                lost = uint32_t(page) >= uint32_t(num_pages);
                bad = bad || lost;
                page_at = lost ? 0 : uint64_t(uint32_t(page)) * page_bytes;
                fresh = false;
            }
            x.at = page_at + uint32_t(inside) * row_bytes;
            x.bytes = lost ? 0u : uint32_t(max(min(BN, end - k0), 0)) * row_bytes;
        } else if constexpr (PAGES == TWO) {
            const int rows = max(min(BN, end - k0), 0);
            x.seam = page_size - inside;
            const bool lost0 = rows > 0 && uint32_t(page) >= uint32_t(num_pages), lost1 = rows > x.seam && uint32_t(behind) >= uint32_t(num_pages);
            bad = bad || lost0 || lost1;
            x.at = lost0 ? 0 : uint64_t(uint32_t(page)) * page_bytes + uint32_t(inside) * row_bytes;
            x.at_behind = lost1 ? 0 : uint64_t(uint32_t(behind)) * page_bytes - uint64_t(x.seam) * row_bytes;  // row `seam` is its first
            x.rows = lost0 ? 0 : min(rows, x.seam);
            x.rows_behind = lost1 ? 0 : rows;
        } else {
            const int row0 = loader * REQ * RPI + lane_id() / CPR;
#pragma unroll
            for (int j = 0; j < REQ; ++j) {
                const int s = k0 + row0 + j * RPI;
                x.row[j] = -1;
                if (s < end) {
                    x.row[j] = slot_row(p.pool, table, s, p.kv_heads, h);
                    bad = bad || x.row[j] < 0;
                }
            }
        }
        return x;
    }
    // .. into LDS from place `to` (of this wavefront's first row)
    template <bool VALUES>
    __device__ __forceinline__ void request(const Place &x, int loader, uint32_t to) {
        const E *from = VALUES ? values : keys;
        int lane = lane_id();
        if constexpr (!KEPT) asm volatile("" : "+v"(lane));  // .. formed anew each time
        const int row0 = loader * REQ * RPI + lane / CPR;
        if constexpr (PAGES == ONE) {
            const uint64_t a = uint64_t(uintptr_t(from)) + x.at;
            u32x4_t r;
            r[0] = uniform(uint32_t(a)), r[1] = uniform(uint32_t(a >> 32)), r[2] = uniform(x.bytes), r[3] = 0x00027000u;  // addresses have 48 bits
#pragma unroll
            for (int j = 0; j < REQ; ++j) fetch_bounded(r, offset<VALUES>(lane, loader, j), to + j * 1024);
        } else if constexpr (PAGES == TWO) {
            const uint64_t zero = uint64_t(uintptr_t(&zero_chunk)), a = uint64_t(uintptr_t(from)) + x.at, b = uint64_t(uintptr_t(from)) + x.at_behind;
#pragma unroll
            for (int j = 0; j < REQ; ++j) {
                const int row = row0 + j * RPI;
                const uint32_t bytes = offset<VALUES>(lane, loader, j);
                const bool over = row >= x.seam, in = row < (over ? x.rows_behind : x.rows) && bytes != NOWHERE;
                const uint64_t at = (over ? b : a) + bytes;
                fetch(reinterpret_cast<const void *>(uintptr_t(in ? at : zero)), to + j * 1024);
            }
        } else {
            const E *zero = reinterpret_cast<const E *>(&zero_chunk);
            const int c = lane % CPR;
#pragma unroll
            for (int j = 0; j < REQ; ++j) {
                const int row = row0 + j * RPI, e = (c ^ (VALUES ? value_swizzle<E, DP>(row) : key_swizzle<E, DP>(row))) * N;
                fetch(x.row[j] >= 0 && e < dim ? from + x.row[j] * dim + e : zero, to + j * 1024);
            }
        }
    }
};

// The running state of 32 rows over the slots seen so far.  Scores are computed transposed, S^T = K Q^T,
// so that a lane holds one row's scores for half of the slots: the maximum and the sum of a row are
// sums over a lane's own registers, and the probabilities leave the first product in exactly the
// places in which the second one, O^T += V^T P^T, wants them, if V's slots are taken in the order in
// which a lane holds them (the order of a sum's terms is free).  V^T comes from LDS through the
// transposing read.
template <typename E, int DP, int BN>
struct RowState {
    typedef typename Chunk<E>::v chunk;
    static constexpr int ROW = DP * int(sizeof(E)), BLK = BN / 32, STEPS = DP / (2 * Chunk<E>::N), DB = DP / 32;
    float16_t o[DB];
    float m, l;
    chunk q[STEPS];
    int koff, voff;  // this lane's places in a tile of keys / values

    __device__ __forceinline__ void init() {
        m = -INFINITY, l = 0.f;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[d][r] = 0.f;
        const int lane = lane_id(), half = lane >> 5, col = lane & 31, l16 = lane & 15;
        koff = col * ROW + ((half ^ key_swizzle<E, DP>(col)) << 4);
        if constexpr (sizeof(E) == 2)
            voff = (4 * half + (l16 >> 2)) * ROW + (((2 * ((lane >> 4) & 1) + ((l16 & 3) >> 1)) ^ value_swizzle<E, DP>(l16 >> 2)) << 4) + (l16 & 1) * 8;
        else
            voff = 4 * half * ROW + col * 4;
    }

    // Operand t of the keys: chunk 2 t + half of row 32 b + col, at a place that differs from that of t = 0 in
    // the bits of t alone (rows, tiles and stages are whole multiples of their range)
    __device__ __forceinline__ chunk kfrag(uint32_t kt, int b, int t) const { return lds_read<chunk>(((kt + koff) ^ (t << 5)) + b * 32 * ROW); }
    // 16-bit: V^T fragment of 32 elements x 16 slots: slot 16 t + 8 e + 4 half + i of the tile in element 4 e + i
    __device__ __forceinline__ chunk vfrag(uint32_t vt, int t, int d) const {
        union {
            short4_t h[2];
            chunk v;
        } f;
        const uint32_t at = (vt + voff) ^ (d << 6);
#pragma unroll
        for (int e = 0; e < 2; ++e)
            f.h[e] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((DC_LDS(short4_t) *)(uintptr_t)(at + (16 * t + 8 * e) * ROW));
        return f.v;
    }
    // fp32: element 32 d + col of slot 32 b + 8 (r / 4) + 4 half + r % 4
    __device__ __forceinline__ float vword(uint32_t vt, int b, int r, int d) const {
        return lds_read<float>(vt + voff + (32 * b + 8 * (r / 4) + r % 4) * ROW + 128 * d);
    }

    // .. of WORDS such slots from number `first` (16 b + r) on
    template <int WORDS>
    __device__ __forceinline__ void words(float (&w)[WORDS][DB], uint32_t vt, int first) const {
#pragma unroll
        for (int i = 0; i < WORDS; ++i)
#pragma unroll
            for (int d = 0; d < DB; ++d) w[i][d] = vword(vt, (first + i) / 16, (first + i) % 16, d);
    }

    // Slots that some rows see and others do not may hold infinities or NaN, and 0 * inf would carry them
    // over: such elements leave the product and join the rows that see them one by one.
    static __device__ __forceinline__ uint32_t chunk_odd(chunk v) {
        const u32x4_t w = __builtin_bit_cast(u32x4_t, v);
        return odd_bits<E>(w[0]) | odd_bits<E>(w[1]) | odd_bits<E>(w[2]) | odd_bits<E>(w[3]);
    }
    static __device__ __forceinline__ chunk chunk_even(chunk v) {
        u32x4_t w = __builtin_bit_cast(u32x4_t, v);
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = without_odd<E>(w[i]);
        return __builtin_bit_cast(chunk, w);
    }
    __device__ __forceinline__ bool any_odd(uint32_t vt) const {
        uint32_t odd = 0;
        if constexpr (sizeof(E) == 2) {
#pragma unroll
            for (int t = 0; t < BN / 16; ++t)
#pragma unroll
                for (int d = 0; d < DB; ++d) odd |= chunk_odd(vfrag(vt, t, d));
        } else {
#pragma unroll
            for (int b = 0; b < BLK; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r)
#pragma unroll
                    for (int d = 0; d < DB; ++d) odd |= odd_bits<E>(__float_as_uint(vword(vt, b, r, d)));
        }
        return ballot(odd != 0) != 0;
    }
    __device__ __forceinline__ void add_odd(uint32_t vt, int k0, int limit) {
        constexpr int N = Chunk<E>::N;
        typedef typename Chunk<E>::v4 v4;
        const int half = lane_id() >> 5;
#pragma unroll 1
        for (int k = 0; k < BN; ++k) {
            const uint32_t seen = k0 + k < limit ? ~0u : 0u;
            const int swz = value_swizzle<E, DP>(k) << 4;
            const uint32_t row = vt + k * ROW;
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int e = 32 * d + 8 * j + 4 * half;  // four elements side by side in one chunk
                    union {
                        v4 v;
                        uint32_t w[sizeof(v4) / 4];
                    } x;
                    x.v = lds_read<v4>(row + (((e / N) << 4) ^ swz) + (e % N) * int(sizeof(E)));
#pragma unroll
                    for (int i = 0; i < int(sizeof(v4) / 4); ++i) x.w[i] = (x.w[i] ^ without_odd<E>(x.w[i])) & seen;
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[d][4 * j + i] += float(E(x.v[i]));
                }
        }
    }

    // The products with the values of a block, requested and rounded a step before.
    template <bool MASK>
    __device__ __forceinline__ void add_values(chunk (&vf)[2][DB], const chunk (&pr)[2], uint32_t vt, int k0, int limit) {
        if constexpr (MASK) {
            uint32_t odd = 0;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int d = 0; d < DB; ++d) odd |= chunk_odd(vf[t][d]);
            if (__builtin_expect(ballot(odd != 0) != 0, 0)) {
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int d = 0; d < DB; ++d) vf[t][d] = chunk_even(vf[t][d]);
                add_odd(vt, k0, limit);
            }
        }
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int d = 0; d < DB; ++d) o[d] = Chunk<E>::mma(vf[t][d], pr[t], o[d]);
    }

    // One turn of the pipeline: the scores s of block i become probabilities while the matrix cores work on
    // the scores of block i + 1 and the values of block i - 1.  The wavefront issues products and vector
    // instructions side by side this way: one after the other, as the two wavefronts of a SIMD fall into
    // step on the matrix cores, the kernel took their sum.
    //   kt: keys of i + 1;  vt_old, k_old: values and first slot of i - 1;  vt: values of i, which starts at k0
    template <bool MASK>
    __device__ __forceinline__ void turn(float16_t &s, float16_t &next, chunk (&vf)[2][DB], chunk (&pr)[2], uint32_t kt, uint32_t vt_old,
                                         uint32_t vt, float scale, int k_old, int k0, int limit) {
        const int half = lane_id() >> 5;
        chunk kf[STEPS];
#pragma unroll
        for (int t = 0; t < STEPS; ++t) kf[t] = kfrag(kt, 0, t);
        add_values<MASK>(vf, pr, vt_old, k_old, limit);
        if constexpr (MASK) {
#pragma unroll
            for (int r = 0; r < 16; ++r)
                if (k0 + 8 * (r / 4) + 4 * half + r % 4 >= limit) s[r] = -INFINITY;
        }
        float top = s[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) top = fmaxf(top, s[r]);
        top = max_halves(top) * scale;
        follow(top);
        const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int d = 0; d < DB; ++d) vf[t][d] = vfrag(vt, t, d);
#pragma unroll
        for (int r = 0; r < 16; ++r) next[r] = 0.f;
#pragma unroll
        for (int t = 0; t < STEPS; ++t) next = Chunk<E>::mma(kf[t], q[t], next);
        float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], scale, -ref));
            part[r & 3] += s[r];
        }
        l += (part[0] + part[1]) + (part[2] + part[3]);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            u32x4_t u;
#pragma unroll
            for (int i = 0; i < 4; ++i) u[i] = pack2(s[8 * t + 2 * i], s[8 * t + 2 * i + 1], E());
            pr[t] = __builtin_bit_cast(chunk, u);
        }
    }

    // The reference of the exponentials follows the maximum only when that outgrows it by 2^8 (fp16: by 2^15, from
    // 2^7 on): any reference gives the same quotient, and a step without a new one leaves the sums alone.
    __device__ __forceinline__ void follow(float top) {
        bool more;
        // `top` is off by half a step, |top| 2^-24, which counts as soon as that is not small: fp16 overflows at 2^16
        if constexpr (LIFT<E> > 0.f) more = fmaf(fabsf(top), 0x1p-22f, top) - m > LIFT<E> + 8.f;
        else more = top > m + 8.f;
        if (ballot(more) != 0) {
            float next = top - LIFT<E>;
            if constexpr (LIFT<E> > 0.f) {  // half a step is more than 2^-1, or, from 2^28 on, may be more than 2^4
                const float size = fabsf(top);
                if (size >= 0x1p24f) next = size < 0x1p28f ? top : fmaf(size, 0x1p-23f, top);
            }
            const float m2 = fmaxf(m, next), fade = m2 == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - m2);
            m = m2;
            l *= fade;
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[d][r] *= fade;
        }
    }

    // One tile: slots [k0, k0 + BN); this lane's row sees slots below `limit` (MASK: some row does not see some of the tile's)
    template <bool MASK>
    __device__ __forceinline__ void step(uint32_t kt, uint32_t vt, float scale, int k0, int limit) {
        // LDS answers after some hundred cycles, three products' time: a block's operands are requested in one
        // go, those of the next block before the products of this one, and the first values before the
        // exponentials (left to itself the compiler asks for two operands at a time and waits for each)
        // (fp32: a chunk's products take longer than that, so four on their way are enough, and their registers go to
        // the sums: 1568 rows of 64 heads of 128 / 256 over 4096 slots 2.25 -> 1.97 / 19.3 -> 8.7 ms)
        float16_t s[BLK];
        if constexpr (sizeof(E) == 4) {
            static_assert(BLK == 1 && STEPS >= 4, "one block");
            chunk kf[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) kf[t] = kfrag(kt, 0, t);
#pragma unroll
            for (int r = 0; r < 16; ++r) s[0][r] = 0.f;
#pragma unroll
            for (int t = 0; t < STEPS; ++t) {
                __builtin_amdgcn_sched_barrier(0);
                s[0] = Chunk<E>::mma(kf[t & 3], q[t], s[0]);
                if (t + 4 < STEPS) kf[t & 3] = kfrag(kt, 0, t + 4);
            }
        } else {
            chunk kf[2][STEPS];
#pragma unroll
            for (int t = 0; t < STEPS; ++t) kf[0][t] = kfrag(kt, 0, t);
#pragma unroll
            for (int b = 0; b < BLK; ++b) {
                if (b + 1 < BLK) {
#pragma unroll
                    for (int t = 0; t < STEPS; ++t) kf[(b + 1) & 1][t] = kfrag(kt, b + 1, t);
                }
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int r = 0; r < 16; ++r) s[b][r] = 0.f;
#pragma unroll
                for (int t = 0; t < STEPS; ++t) s[b] = Chunk<E>::mma(kf[b & 1][t], q[t], s[b]);
            }
        }
        chunk vf[2][sizeof(E) == 2 ? DB : 1];
        constexpr int WORDS = sizeof(E) == 4 ? 16 / DB : 1;  // fp32: slots of a request
        float vw[2][WORDS][DB];
        if constexpr (sizeof(E) == 2) {
#pragma unroll
            for (int d = 0; d < DB; ++d) vf[0][d] = vfrag(vt, 0, d);
        } else {
            words<WORDS>(vw[0], vt, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
        const int half = lane_id() >> 5;
        if constexpr (MASK) {
#pragma unroll
            for (int b = 0; b < BLK; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (k0 + 32 * b + 8 * (r / 4) + 4 * half + r % 4 >= limit) s[b][r] = -INFINITY;
        }
        float top = s[0][0];
#pragma unroll
        for (int b = 0; b < BLK; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) top = fmaxf(top, s[b][r]);
        top = max_halves(top) * scale;
        follow(top);
        const float ref = m == -INFINITY ? 0.f : m;
        float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int b = 0; b < BLK; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                s[b][r] = __builtin_amdgcn_exp2f(fmaf(s[b][r], scale, -ref));
                part[r & 3] += s[b][r];
            }
        l += (part[0] + part[1]) + (part[2] + part[3]);
        bool odd = false;
        if constexpr (MASK) odd = any_odd(vt);
        if constexpr (sizeof(E) == 2) {
            // the sum above is of the probabilities in fp32; the product's operand is rounded to the 16-bit type (half a
            // step of it relative to each, as much as the values that it multiplies carry; fp16: or 2^-32 of the
            // row's largest, see LIFT)
            chunk pr[BLK][2];
#pragma unroll
            for (int b = 0; b < BLK; ++b)
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    union {
                        uint32_t u[4];
                        chunk v;
                    } f;
#pragma unroll
                    for (int i = 0; i < 4; ++i) f.u[i] = pack2(s[b][8 * t + 2 * i], s[b][8 * t + 2 * i + 1], E());
                    pr[b][t] = f.v;
                }
            if (MASK && __builtin_expect(odd, 0)) {
#pragma unroll
                for (int b = 0; b < BLK; ++b)
#pragma unroll
                    for (int t = 0; t < 2; ++t)
#pragma unroll
                        for (int d = 0; d < DB; ++d) o[d] = Chunk<E>::mma(chunk_even(vfrag(vt, 2 * b + t, d)), pr[b][t], o[d]);
                add_odd(vt, k0, limit);
                return;
            }
#pragma unroll
            for (int t = 0; t < BN / 16; ++t) {
                if (t + 1 < BN / 16) {
#pragma unroll
                    for (int d = 0; d < DB; ++d) vf[(t + 1) & 1][d] = vfrag(vt, t + 1, d);
                }
#pragma unroll
                for (int d = 0; d < DB; ++d) o[d] = Chunk<E>::mma(vf[t & 1][d], pr[t / 2][t % 2], o[d]);
                __builtin_amdgcn_sched_barrier(0);
            }
        } else {
            if (MASK && __builtin_expect(odd, 0)) {
#pragma unroll
                for (int b = 0; b < BLK; ++b)
#pragma unroll
                    for (int r = 0; r < 16; ++r)
#pragma unroll
                        for (int d = 0; d < DB; ++d) {
                            const float v = __uint_as_float(without_odd<E>(__float_as_uint(vword(vt, b, r, d))));
                            o[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(v, s[b][r], o[d], 0, 0, 0);
                        }
                add_odd(vt, k0, limit);
                return;
            }
#pragma unroll
            for (int g = 0; g < 16 * BLK / WORDS; ++g) {
                if (g + 1 < 16 * BLK / WORDS) words<WORDS>(vw[(g + 1) & 1], vt, (g + 1) * WORDS);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < WORDS; ++i)
#pragma unroll
                    for (int d = 0; d < DB; ++d)
                        o[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(vw[g & 1][i][d], s[(g * WORDS + i) / 16][(g * WORDS + i) % 16], o[d], 0, 0, 0);
            }
        }
    }
};

struct AttnCall {
    AttnPlan p;
    AttnGrid g;
    const void *q, *keys, *values;
    void *out;
    float *lse;
    const int32_t *lens, *starts;
};

// The kernel's arguments, loaded anew: what is needed behind a loop alone does not take scalar registers in it.
__device__ __forceinline__ const AttnCall &call_again() {
    uint64_t at = uint64_t(__builtin_amdgcn_kernarg_segment_ptr());
    asm volatile("" : "+s"(at));
    return *(const AttnCall *)(const __attribute__((address_space(4))) AttnCall *)at;
}

// How a workgroup goes about its slots.
//   PIPE (16-bit types, many rows): 4 wavefronts own different rows and share blocks of 32 slots, rings of 3
//   blocks of keys and 4 of values; see RowState::turn().
//   KEYS (few rows, or little work): the wavefronts own the same rows and blocks of 32 slots each in turn, two stages of
//   their own, without a barrier between them, and join their sums at the end.
//   NARROW: 2 wavefronts, for streams of at most 64 rows whose tiles leave no room for KEYS' four.
//   else (fp32, whose products take sixteen times as long as anything beside them): 4 wavefronts own
//   different rows and share two stages of 32 slots.
template <typename E, int DP, bool KEYS, bool NARROW = false>
struct Shape {
    static constexpr int ROW = DP * int(sizeof(E)), BN = 32, TILE = BN * ROW;
    static constexpr bool PIPE = !KEYS && sizeof(E) == 2;
    static constexpr int NW = !KEYS ? NARROW ? 2 : 4 : ROW <= 256 ? 4 : ROW <= 512 ? 2 : 1;
    static constexpr int TILES = PIPE ? 7 * TILE : 4 * TILE * (KEYS ? NW : 1), JOIN = KEYS ? NW * 32 * (DP + 6) * 4 : 0;
    static constexpr int LDS = TILES > JOIN ? TILES : JOIN;
    // workgroups a compute unit is to hold (fp32 rows of 512 bytes: two, though some registers spill, 510 us instead of
    // 568 us for 392 rows of 64 heads over 4096 slots, but one of the narrow ones, 82 instead of 130 us for 49 rows)
    static constexpr int GROUPS = LDS <= 79 << 10 && ROW <= (sizeof(E) == 4 && !NARROW ? 512 : 256) ? 2 : 1;
};

// Attention on the matrix cores.  A wavefront owns 32 rows.
template <typename E, int DP, bool KEYS, bool NARROW, Pages PAGES>
__global__ void __launch_bounds__((WAVE * Shape<E, DP, KEYS, NARROW>::NW), (Shape<E, DP, KEYS, NARROW>::GROUPS))
attention_mfma_kernel(AttnCall call) {
    const AttnPlan &p = call.p;
    const AttnGrid &g = call.g;
    const E *q = static_cast<const E *>(call.q), *keys = static_cast<const E *>(call.keys), *values = static_cast<const E *>(call.values);
    const int32_t *lens = call.lens, *starts = call.starts;
    typedef Shape<E, DP, KEYS, NARROW> S;
    typedef typename Chunk<E>::v chunk;
    constexpr int BN = S::BN, TILE = S::TILE, NW = S::NW, N = Chunk<E>::N;
    extern __shared__ __attribute__((aligned(1024))) char lds[];  // whole rows of any tile: see kfrag()
    Work w;
    if (!find_work(starts, p, g, w)) return;
    const int lane = lane_id(), wv = wave_id(), half = lane >> 5, col = lane & 31;
    const int len = uniform(stream_len(p, lens, w.b));
    const int rows = w.count * p.group;
    const int r0 = w.rb * g.block_rows, row = r0 + (KEYS ? 0 : wv * 32) + col;
    const int tok = int(g.by_group.quot(uint32_t(min(row, rows - 1))));
    const int head = w.h * p.group + min(row, rows - 1) - tok * p.group;
    const bool real = row < rows;
    const int last_tok = int(g.by_group.quot(uint32_t(min(r0 + g.block_rows, rows) - 1)));
    const int end_all = uniform(visible(len, w.count, last_tok, p.causal_block));  // slots that any row of the workgroup sees
    const int kb = w.split * g.split_keys, ke = min(end_all, kb + g.split_keys);
    if (kb >= end_all && w.split > 0) return;  // nothing: the joining launch knows
    const int limit = real ? min(visible(len, w.count, tok, p.causal_block), ke) : 0;
    // slots below `all` are seen by every row of the workgroup, those from wave_end by none of this wavefront's
    const int all = uniform(min(visible(len, w.count, int(g.by_group.quot(uint32_t(r0))), p.causal_block), ke));
    const int wave_r0 = r0 + (KEYS ? 0 : wv * 32), wave_last = min(wave_r0 + 32, rows) - 1;
    const int wave_end = uniform(wave_r0 < rows ? min(visible(len, w.count, int(g.by_group.quot(uint32_t(wave_last))), p.causal_block), ke) : 0);

    RowState<E, DP, BN> st;
    st.init();
    const E *qr = q + int64_t(w.first + tok) * p.qt + head * p.qh;
#pragma unroll
    for (int t = 0; t < RowState<E, DP, BN>::STEPS; ++t) {
        uint4 u = make_uint4(0, 0, 0, 0);
        const int e = (2 * t + half) * N;
        if (real && e < p.dim) u = *reinterpret_cast<const uint4 *>(qr + e);
        u.x ^= p.flip, u.y ^= p.flip, u.z ^= p.flip, u.w ^= p.flip;
        st.q[t] = __builtin_bit_cast(chunk, u);
    }
    const int32_t *table = p.pool.table + int64_t(w.b) * p.pool.max_pages;
    typedef TileLoader<E, DP, BN, KEYS ? 1 : NW, PAGES> Loader;
    Loader load;
    const int loader = KEYS ? 0 : wv, first = kb + (KEYS ? wv * BN : 0), stride = KEYS ? NW * BN : BN;
    load.init(p, table, keys, values, w.h, loader, first);
    const uint32_t place = lds_place(lds) + (KEYS ? wv * 4 * TILE : 0), mine = place + loader * Loader::REQ * 1024;  // [stage][K, V]
    if constexpr (S::PIPE) {
        // Group i of requests, {keys of i + 3, values of i + 2}, goes out in turn i, behind the barrier at which
        // everybody has left turn i - 1 (and with it the keys of i and the values of i - 2, whose places it
        // takes); what turn i reads came with group i - 2, so one group stays in flight.  Blocks behind the
        // last are requested as nothing, which keeps the count.
        constexpr int FLIGHT = 2 * Loader::REQ;
        const uint32_t vplace = place + 3 * TILE, vmine = mine + 3 * TILE;
        typename Loader::Place held;
        auto next_place = [&](int k0) {
            const auto x = load.find(p, loader, k0, ke);
            load.advance(BN);
            if (k0 + BN < ke) load.look(k0 + BN, ke);  // a turn ahead
            return x;
        };
        if (kb < ke) load.look(kb, ke);
        held = next_place(kb);
        load.template request<false>(held, loader, mine);
        for (int i = 1; i < 3; ++i) {
            const auto x = next_place(kb + i * BN);
            load.template request<false>(x, loader, mine + i * TILE);
            load.template request<true>(held, loader, vmine + (i - 1) * TILE);
            held = x;
        }
        auto meet = [&]() {  // all but the newest group are there, everybody's
            arrived_but<FLIGHT>();
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
        };
        meet();
        float16_t sa, sb;
        chunk vf[2][DP / 32], pr[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            pr[t] = __builtin_bit_cast(chunk, make_uint4(0, 0, 0, 0));
#pragma unroll
            for (int d = 0; d < DP / 32; ++d) vf[t][d] = pr[t];
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) sa[r] = 0.f;
#pragma unroll
        for (int t = 0; t < RowState<E, DP, BN>::STEPS; ++t) sa = Chunk<E>::mma(st.kfrag(place, 0, t), st.q[t], sa);
        uint32_t kslot = 0, vslot = 0;  // of block i
        int k0 = kb;
        auto turn = [&](auto mask, float16_t &s, float16_t &next) {
            meet();
            const uint32_t knext = kslot == 2 * TILE ? 0 : kslot + TILE;
            const auto x = next_place(k0 + 3 * BN);
            load.template request<false>(x, loader, mine + kslot);
            load.template request<true>(held, loader, vmine + ((vslot + 2 * TILE) & 3 * TILE));
            held = x;
            st.template turn<decltype(mask)::value>(s, next, vf, pr, place + knext, vplace + ((vslot + 3 * TILE) & 3 * TILE), vplace + vslot,
                                                    p.scale, k0 - BN, k0, limit);
            kslot = knext;
            vslot = (vslot + TILE) & 3 * TILE;
            k0 += BN;
        };
        // blocks that every row of the workgroup sees, two by two so that scores need not be copied, then the rest
        while (k0 + 2 * BN <= all) {
            turn(Flag<false>(), sa, sb);
            turn(Flag<false>(), sb, sa);
        }
        while (k0 < ke) {
            turn(Flag<true>(), sa, sb);
            sa = sb;
        }
        st.template add_values<true>(vf, pr, vplace + ((vslot + 3 * TILE) & 3 * TILE), k0 - BN, limit);
        arrived();  // nothing may reach this LDS after the workgroup has left it
    } else {
        loaded();
        if (first < ke) {
            load.look(first, ke);
            const auto x = load.find(p, loader, first, ke);
            load.template request<false>(x, loader, mine);
            load.template request<true>(x, loader, mine + TILE);
            load.advance(stride);
            if (first + stride < ke) load.look(first + stride, ke);
        }
        uint32_t stage = 0;
        int k0 = first;
        // the next tile's requests and the page of the one behind it, once this tile is there
        auto turn = [&]() {
            arrived();                             // this tile, of this wavefront's requests
            if constexpr (!KEYS) __syncthreads();  // .. of everybody's, and the other stage is free
            if (k0 + stride < ke) {
                const uint32_t to = mine + (stage ^ 2 * TILE);
                const auto x = load.find(p, loader, k0 + stride, ke);
                load.template request<false>(x, loader, to);
                load.template request<true>(x, loader, to + TILE);
                load.advance(stride);
                if (k0 + 2 * stride < ke) load.look(k0 + 2 * stride, ke);
            }
        };
        // tiles that every row of the workgroup sees as a whole, then the rest
        for (; k0 + BN <= all; k0 += stride, stage ^= 2 * TILE) {
            turn();
            st.template step<false>(place + stage, place + stage + TILE, p.scale, k0, limit);
        }
        for (; k0 < ke; k0 += stride, stage ^= 2 * TILE) {
            turn();
            if (k0 < wave_end) st.template step<true>(place + stage, place + stage + TILE, p.scale, k0, limit);
        }
    }

    float l = sum_halves(st.l);
    const AttnCall &again = call_again();
    const AttnPlan &tp = again.p;
    const AttnGrid &tg = again.g;
    E *out = static_cast<E *>(again.out);
    float *lse = again.lse;
    const bool bad = __syncthreads_or(load.bad) != 0;
    const int64_t grow = int64_t(w.first + tok) * tp.q_heads + head;  // this row among all
    const int64_t all_rows = int64_t(tp.tokens) * tp.q_heads;
    if constexpr (KEYS) {
        // the four wavefronts' sums meet in LDS: [wavefront][row][DP + 4] and their (m, l)
        constexpr int PITCH = DP + 4;
        float *ml = reinterpret_cast<float *>(lds), *os = ml + NW * 32 * 2;
        if (half == 0) ml[(wv * 32 + col) * 2] = st.m, ml[(wv * 32 + col) * 2 + 1] = l;
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                *reinterpret_cast<float4_t *>(os + (wv * 32 + col) * PITCH + 32 * d + 8 * j + 4 * half) =
                    float4_t{st.o[d][4 * j], st.o[d][4 * j + 1], st.o[d][4 * j + 2], st.o[d][4 * j + 3]};
        __syncthreads();
        const int here = min(32, rows - r0);
        const int vecs = tp.dim / 4;
        for (int i = threadIdx.x; i < here * vecs; i += NW * WAVE) {
            const int rr = i / vecs, c = (i - rr * vecs) * 4;
            float mm = -INFINITY;
#pragma unroll
            for (int k = 0; k < NW; ++k) mm = fmaxf(mm, ml[(k * 32 + rr) * 2]);
            const float ref = mm == -INFINITY ? 0.f : mm;
            float ll = 0.f;
            float4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < NW; ++k) {
                const float f = __builtin_amdgcn_exp2f(ml[(k * 32 + rr) * 2] - ref);
                ll = fmaf(f, ml[(k * 32 + rr) * 2 + 1], ll);
                const float4_t v = *reinterpret_cast<const float4_t *>(os + (k * 32 + rr) * PITCH + c);
#pragma unroll
                for (int j = 0; j < 4; ++j) o[j] = fmaf(f, v[j], o[j]);
            }
            const int tk = int(tg.by_group.quot(uint32_t(r0 + rr))), hd = w.h * tp.group + r0 + rr - tk * tp.group;
            const int64_t gr = int64_t(w.first + tk) * tp.q_heads + hd;
            if (bad) ll = NAN;
            if (tg.splits > 1) {
                *reinterpret_cast<float4_t *>(tg.part + (w.split * all_rows + gr) * tp.dim + c) = o;
                if (c == 0) {
                    float *x = tg.part + tg.splits * all_rows * tp.dim + (w.split * all_rows + gr) * 2;
                    x[0] = mm, x[1] = ll;
                }
            } else {
                const float inv = ll == 0.f ? 0.f : 1.f / ll;
                Vec<E, 4> v;
#pragma unroll
                for (int j = 0; j < 4; ++j) v.v[j] = E(o[j] * inv);
                E *dst = out + int64_t(w.first + tk) * tp.ot + hd * tp.oh + c;
#pragma unroll
                for (int j = 0; j < 4; ++j) dst[j] = v.v[j];
                if (c == 0 && lse != nullptr) lse[gr] = log_sum<E>(mm, ll);
            }
        }
    } else {
        if (!real) return;
        if (bad) l = NAN;
        if (tg.splits > 1) {
            float *dst = tg.part + (w.split * all_rows + grow) * tp.dim;
#pragma unroll
            for (int d = 0; d < DP / 32; ++d)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (32 * d + 8 * j + 4 * half < tp.dim)
                        *reinterpret_cast<float4_t *>(dst + 32 * d + 8 * j + 4 * half) =
                            float4_t{st.o[d][4 * j], st.o[d][4 * j + 1], st.o[d][4 * j + 2], st.o[d][4 * j + 3]};
            if (half == 0) {
                float *x = tg.part + tg.splits * all_rows * tp.dim + (w.split * all_rows + grow) * 2;
                x[0] = st.m, x[1] = l;
            }
            return;
        }
        const float inv = l == 0.f ? 0.f : 1.f / l;
        E *dst = out + int64_t(w.first + tok) * tp.ot + head * tp.oh;
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (32 * d + 8 * j + 4 * half >= tp.dim) continue;
#pragma unroll
                for (int i = 0; i < 4; ++i) dst[32 * d + 8 * j + 4 * half + i] = E(st.o[d][4 * j + i] * inv);
            }
        if (half == 0 && lse != nullptr) lse[grow] = log_sum<E>(st.m, l);
    }
}

// The attention that slots receive, once every row's log-sum is known.  A wavefront keeps the keys of
// 32 slots in registers as the first operand and walks over all rows of its stream and head, tiles
// of 64 at a time through LDS; a lane's scores are those of one row, so its sums over the rows stay
// in place until the end, where the lanes of a half are added up in a fixed order.
//
// Bound by its products and its vector work one after the other: an exponential, a multiplication and two sums for
// every score take about as long as the score's product, and the full wait and the barrier in front of every tile of rows
// keep the two wavefronts of a SIMD in step.  2040 rows x 32640 slots x 4 heads of 128, bf16: 112 .. 127 us under the
// profiler, 0.6 PFLOP/s.  A workgroup walks over all rows by itself, so few slots fill the card poorly: 8160 rows of one kv
// head over 2040 slots 145 us.  (64 slots a wavefront, half of the reads from LDS: alike in the first case, 455 instead of
// 437 us for 8 streams over 16320 slots, and 1300 instead of 650 us for 8192 tokens in frames of 512, where the workgroups
// of the first slots have most rows.)
template <typename E, int DP>
__global__ void __launch_bounds__(256, DP * sizeof(E) <= 256 ? 2 : 1)
attention_weights_kernel(AttnPlan p, FastDiv by_group, const E *__restrict__ q, const float *__restrict__ lse,
                         const E *__restrict__ keys, float *__restrict__ weights, const int32_t *__restrict__ lens,
                         const int32_t *__restrict__ starts) {
    typedef typename Chunk<E>::v chunk;
    constexpr int N = Chunk<E>::N, ROW = DP * int(sizeof(E)), STEPS = DP / (2 * N), BM = DP * sizeof(E) <= 512 ? 64 : 32, TILE = BM * ROW;
    constexpr int CPR = DP / N, RPI = WAVE / CPR, REQ = BM / RPI / 4;
    extern __shared__ __attribute__((aligned(1024))) char lds[];  // whole rows of any tile: see kfrag()
    const int b = blockIdx.z, h = blockIdx.y, len = uniform(stream_len(p, lens, b));
    const int lane = lane_id(), wv = wave_id(), half = lane >> 5, col = lane & 31;
    const int s_block = blockIdx.x * (4 * 32), s0 = s_block + wv * 32;
    if (s_block >= len) return;
    int first, count;
    stream_tokens(starts, b, p.streams, p.tokens, first, count);
    const int32_t *table = p.pool.table + int64_t(b) * p.pool.max_pages;
    chunk k[STEPS];
    {
        const int64_t row = s0 + col < len ? slot_row(p.pool, table, s0 + col, p.kv_heads, h) : -1;
#pragma unroll
        for (int t = 0; t < STEPS; ++t) {
            const int e = (2 * t + half) * N;
            uint4 u = make_uint4(0, 0, 0, 0);
            if (row >= 0 && e < p.dim) u = *reinterpret_cast<const uint4 *>(keys + row * p.dim + e);
            k[t] = __builtin_bit_cast(chunk, u);
        }
    }
    // the first token that sees this workgroup's first slot
    int begin = 0;
    if (p.causal_block != 0) {
        const int past = s_block - (len - count);
        begin = past > 0 ? past / p.causal_block * p.causal_block : 0;
    }
    const int rows = count * p.group, r_first = min(begin * p.group, rows) / BM * BM;
    const E *zero = reinterpret_cast<const E *>(&zero_chunk);
    const int ahead_tok = int(by_group.quot(BM)), ahead_head = BM - ahead_tok * p.group;  // a tile of rows further on
    // A lane's way through the rows, BM at a time, without a division: its token and head of the group, and what it
    // reads there.
    struct Walk {
        int tok, g;
    };
    auto start = [&](int r) {
        Walk w;
        w.tok = int(by_group.quot(uint32_t(r)));
        w.g = r - w.tok * p.group;
        return w;
    };
    auto step = [&](Walk &w, auto *&at, int64_t by_tok, int64_t by_head) {  // strides of a token and of a head
        w.tok += ahead_tok, w.g += ahead_head;
        const bool carry = w.g >= p.group;
        w.tok += carry ? 1 : 0, w.g -= carry ? p.group : 0;
        at += ahead_tok * by_tok + ahead_head * by_head + (carry ? by_tok - p.group * by_head : 0);
    };
    Walk qw[REQ];
    const E *qp[REQ];
#pragma unroll
    for (int j = 0; j < REQ; ++j) {
        const int rr = (wv * REQ + j) * RPI + lane / CPR;
        qw[j] = start(r_first + rr);
        qp[j] = q + int64_t(first + qw[j].tok) * p.qt + (h * p.group + qw[j].g) * p.qh + ((lane % CPR) ^ key_swizzle<E, DP>(rr)) * N;
    }
    auto request = [&](uint32_t to) {  // the next tile of rows
#pragma unroll
        for (int j = 0; j < REQ; ++j) {
            const int rr = (wv * REQ + j) * RPI + lane / CPR, e = ((lane % CPR) ^ key_swizzle<E, DP>(rr)) * N;
            fetch(qw[j].tok < count && e < p.dim ? qp[j] : zero, to + (wv * REQ + j) * 1024);
            step(qw[j], qp[j], p.qt, p.qh);
        }
    };
    const float scale = p.flip != 0 ? -p.scale : p.scale;
    float16_t acc;
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[r] = 0.f;
    // this lane's row of a tile: its log-sum (-inf: no row, or one that sees nothing) and what it sees
    struct Row {
        float lse;
        int limit;
    };
    Walk lw[BM / 32];
    const float *lp[BM / 32];
#pragma unroll
    for (int i = 0; i < BM / 32; ++i) {
        lw[i] = start(r_first + 32 * i + col);
        lp[i] = lse + int64_t(first + lw[i].tok) * p.q_heads + h * p.group + lw[i].g;
    }
    auto next_row = [&](int i) {
        Row x = {-INFINITY, 0};
        if (lw[i].tok < count) x.lse = *lp[i], x.limit = visible(len, count, lw[i].tok, p.causal_block);
        step(lw[i], lp[i], p.q_heads, 1);
        return x;
    };
    const uint32_t place = lds_place(lds);
    chunk qf[STEPS];
    auto rows_of = [&](uint32_t qt) {
#pragma unroll
        for (int t = 0; t < STEPS; ++t) qf[t] = lds_read<chunk>((qt + col * ROW + ((half ^ key_swizzle<E, DP>(col)) << 4)) ^ (t << 5));
        __builtin_amdgcn_sched_barrier(0);  // all requested before anything else
    };
    auto scores = [&](float16_t &s) {
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll
        for (int t = 0; t < STEPS; ++t) s = Chunk<E>::mma(k[t], qf[t], s);
    };
    auto add = [&](const float16_t &s, Row x, bool whole) {
        const float less = x.lse == -INFINITY ? -INFINITY : x.lse * -1.44269504088896341f;
        if (whole) {
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[r] += __builtin_amdgcn_exp2f(fmaf(s[r], scale, less));
        } else {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const float e = __builtin_amdgcn_exp2f(fmaf(s[r], scale, less));
                acc[r] += s0 + 8 * (r / 4) + 4 * half + r % 4 < x.limit ? e : 0.f;
            }
        }
    };
    if (r_first < rows) {
        request(place);
        Row x[BM / 32];
#pragma unroll
        for (int i = 0; i < BM / 32; ++i) x[i] = next_row(i);
        uint32_t stage = 0;
        loaded();
        for (int r0 = r_first; r0 < rows; r0 += BM, stage ^= 1) {
            arrived();
            __syncthreads();
            rows_of(place + stage * TILE);
            // the next tile and its rows' log-sums are on their way while this one is worked on
            Row y[BM / 32];
            if (r0 + BM < rows) request(place + (stage ^ 1) * TILE);
#pragma unroll
            for (int i = 0; i < BM / 32; ++i) y[i] = next_row(i);
            // (no row behind the last: its scores are zeros, or NaN of an infinite key that gives a real row a weight of 0)
            const bool whole = r0 + BM <= rows && s0 + 32 <= visible(len, count, int(by_group.quot(uint32_t(r0))), p.causal_block);
#pragma unroll
            for (int i = 0; i < BM / 32; ++i) {
                float16_t s;
                scores(s);
                if (i + 1 < BM / 32) rows_of(place + stage * TILE + 32 * (i + 1) * ROW);  // in time for the exponentials
                add(s, x[i], whole);
                x[i] = y[i];
            }
        }
    }
    // sums over the 32 lanes of a half; lane `col` keeps sum number `col`
    float mine = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        float x = acc[r];
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) x += __shfl_xor(x, d, WAVE);
        if (col == r) mine = x;
    }
    const int s = s0 + 8 * (col / 4) + 4 * half + col % 4;
    if (col >= 16 || s >= len) return;
    const int64_t row = slot_row(p.pool, table, s, p.kv_heads, h);
    if (row >= 0) weights[row] = p.decay == 0.f ? mine : fmaf(p.decay, weights[row], mine);
}

// Joins the pieces of the slot axis: one wavefront per row, a lane per piece for the maxima, then 16 lanes for each
// of four pieces.  Bound by its launch and three dependent trips to memory: 4 .. 6 us up to 2000 rows.
template <typename T>
__global__ void __launch_bounds__(256)
attention_join_kernel(AttnPlan p, AttnGrid g, T *__restrict__ out, float *__restrict__ lse, const int32_t *__restrict__ lens,
                      const int32_t *__restrict__ starts) {
    const int64_t all_rows = int64_t(p.tokens) * p.q_heads, row = int64_t(blockIdx.x) * 4 + wave_id();
    if (row >= all_rows) return;
    const int t = int(row / p.q_heads), head = int(row - int64_t(t) * p.q_heads), lane = lane_id();
    const int b = stream_of(starts, p.streams, p.tokens, t);
    if (b < 0) return;
    int first, count;
    stream_tokens(starts, b, p.streams, p.tokens, first, count);
    const int n = visible(stream_len(p, lens, b), count, t - first, p.causal_block);
    const int pieces = min(g.splits, max(1, (n + g.split_keys - 1) / g.split_keys));
    const float *ml = g.part + g.splits * all_rows * p.dim;
    // a lane per piece: their maxima and sums in one request
    float top = -INFINITY, m_here = -INFINITY, l_here = 0.f;
    for (int s = lane; s < pieces; s += WAVE) top = fmaxf(top, ml[(s * all_rows + row) * 2]);
    if (lane < pieces) {
        const float2 x = *reinterpret_cast<const float2 *>(ml + (lane * all_rows + row) * 2);
        m_here = x.x, l_here = x.y;
    }
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) top = fmaxf(top, __shfl_xor(top, d, WAVE));
    const float ref = top == -INFINITY ? 0.f : top;
    const int vecs = p.dim / 4, c = lane % 16 * 4;  // 16 lanes hold 64 elements of a piece's row, 4 pieces at a time
    float l = 0.f;
    float4_t o[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) o[k] = float4_t{0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < pieces; s0 += WAVE) {
        if (s0 > 0) {
            const int s = s0 + lane;
            m_here = -INFINITY, l_here = 0.f;
            if (s < pieces) m_here = ml[(s * all_rows + row) * 2], l_here = ml[(s * all_rows + row) * 2 + 1];
        }
        const float f_here = s0 + lane < pieces ? __builtin_amdgcn_exp2f(m_here - ref) : 0.f;
        l = fmaf(f_here, l_here, l);
        const int n4 = min(WAVE, pieces - s0);
        for (int s = lane / 16; s < (n4 + 3) / 4 * 4; s += 4) {
            const float f = __shfl(f_here, s, WAVE);
            if (s >= n4) continue;
            const float *src = g.part + ((s0 + s) * all_rows + row) * p.dim;
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (k * 16 + lane % 16 < vecs) {
                    const float4_t v = *reinterpret_cast<const float4_t *>(src + k * 64 + c);
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[k][i] = fmaf(f, v[i], o[k][i]);
                }
        }
    }
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) l += __shfl_xor(l, d, WAVE);
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            o[k][i] += __shfl_xor(o[k][i], 16, WAVE);
            o[k][i] += __shfl_xor(o[k][i], 32, WAVE);
        }
        if (lane < 16 && k * 16 + lane < vecs) {
            T *dst = out + t * p.ot + head * p.oh + k * 64 + c;
#pragma unroll
            for (int i = 0; i < 4; ++i) dst[i] = T(o[k][i] * inv);
        }
    }
    if (lane == 0 && lse != nullptr) lse[row] = log_sum<T>(top, l);
}

// Rows of a workgroup.  32 (KEYS) where a stream has no more, and, as long as four wavefronts' blocks have room in LDS
// (rows of a tile up to 256 bytes), also up to 64 and where all the work is at most 28 blocks of 32 x 32 for each
// wavefront of the card: fewer pieces, which end in shorter sums.  8 heads of 128 in bf16: 4 / 32 streams of 49
// tokens over 4096 slots 23 / 106 us, with the narrow workgroups 25 / 115 us; one stream of 196 tokens over 4096 slots
// (7 blocks) 21 us, with 128 rows 29 us; of 98 over 32640 (32 blocks) 44 us both; of 196 (56) 73 and 54 us.  64 in
// fp32: 38 / 192 and 45 / 282 us; 30 and 36 us; 88 and 84 us; 165 and 144 us.  Rows of 512 bytes, two wavefronts a
// workgroup in either form: 88 / 590 and 56 / 342 us for the first two.
template <typename E>
int block_rows(const AttnPlan &p) {
    const int row_bytes = (p.dim <= 64 ? 64 : p.dim <= 128 ? 128 : 256) * int(sizeof(E));
    const int64_t rows = int64_t(p.tokens) * p.group, streams = p.streams;
    const int64_t work = ceil_div64(rows, 32 * streams) * streams * p.kv_heads * ceil_div64(int64_t(p.pool.max_pages) * p.pool.page_size, 32);
    if (rows <= 32 * streams || (row_bytes <= 256 && (rows <= 64 * streams || work <= 28 * 1024))) return 32;
    return rows <= 64 * streams ? 64 : 128;
}

// How the rows and the slots are divided.
AttnGrid plan_grid(const AttnPlan &p, bool ragged, int bm) {
    AttnGrid g = {};
    g.block_rows = bm;
    const int64_t rows = int64_t(p.tokens) * p.group;
    // (with starts there may be fewer rows than streams: a token each of 20 of 32 streams over 32640 slots, one head of 128
    // in bf16, 63 us in pieces, 284 us without)
    g.stream_blocks = max(1, int(ceil_div64(rows / p.streams, bm)));
    g.flat = ragged ? int(rows / bm) + p.streams : g.stream_blocks * p.streams;
    const int64_t cap = int64_t(p.pool.max_pages) * p.pool.page_size;
    const int64_t base = int64_t(g.flat) * p.kv_heads;
    // Pieces of the slot axis (by the table's capacity: the lengths are the device's) until every compute unit has two workgroups, or one with few rows, whose LDS it
    // takes (a token of 32 streams over 32640 slots: 146 us, with two 159 us and twice as much to join), and
    // not more than are resident at once; none below 128 slots, in whole turns of a workgroup's blocks.
    const bool few = bm == 32;
    const int64_t want = few ? 256 : 512, least = 128, turn = few ? 128 : 32, per_xcd = want / 8;
    int64_t splits = 1;
    g.unit = 1;
    if (base < want) {
        // .. a unit of row blocks with the same slots on one XCD as a whole, as long as that leaves three quarters
        // of the workgroups (392 rows over 32640 slots, one head of 128 in bf16: 13 row blocks in 16 pieces 24 us,
        // in 19 pieces spread over all XCDs 38 us, or 8 to an XCD, some of which then get a second round, 37 us)
        const int64_t most = want / base;
        for (int k = 1; k <= g.stream_blocks; ++k) {
            const int64_t unit = ceil_div64(g.stream_blocks, k), fit = 8 * (per_xcd / unit) / (ceil_div64(g.flat, unit) * p.kv_heads);
            if (4 * fit < 3 * most && unit > 1) continue;
            g.unit = int(unit);
            splits = max(int64_t(1), fit);
            break;
        }
    } else {
        while (g.unit < 16 && g.unit * 2 <= g.flat && base >= 8 * 2 * g.unit * 2) g.unit *= 2;
    }
    const int64_t keys = max(least, ceil_div64(ceil_div64(cap, splits), turn) * turn);
    splits = ceil_div64(cap, keys);
    g.splits = int(splits);
    g.split_keys = int(keys);
    g.pairs = p.kv_heads * g.splits;
    g.by_group = FastDiv(uint32_t(p.group));
    g.by_unit = FastDiv(uint32_t(g.unit));
    g.by_pairs = FastDiv(uint32_t(g.pairs));
    g.by_blocks = FastDiv(uint32_t(max(1, g.stream_blocks)));
    g.by_kv = FastDiv(uint32_t(p.kv_heads));
    return g;
}

int64_t part_bytes(const AttnPlan &p, const AttnGrid &g) {
    return g.splits > 1 ? int64_t(g.splits) * p.tokens * p.q_heads * (p.dim + 2) * 4 : 0;
}

// Raises a kernel's limit of dynamic LDS, once per device.
hipError_t raise_lds(const void *kernel, int bytes, uint64_t &raised) {
    int dev = 0;
    hipError_t err = hipGetDevice(&dev);
    if (err != hipSuccess || (dev < 64 && (raised >> dev & 1))) return err;
    err = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (err == hipSuccess && dev < 64) raised |= 1ull << dev;
    return err;
}

template <typename E, int DP, bool KEYS, bool NARROW, Pages PAGES>
hipError_t attention_go(const dc_attention_args &a, const AttnPlan &p, const AttnGrid &g, float *lse, hipStream_t s) {
    typedef Shape<E, DP, KEYS, NARROW> S;
    auto kernel = attention_mfma_kernel<E, DP, KEYS, NARROW, PAGES>;
    static thread_local uint64_t raised = 0;
    const hipError_t err = raise_lds((const void *)kernel, S::LDS, raised);
    if (err != hipSuccess) return err;
    const int64_t blocks = ceil_div64(ceil_div64(g.flat, g.unit) * g.pairs, 8) * 8 * g.unit;
    if (blocks > (1 << 30)) return hipErrorInvalidConfiguration;
    note_kernel("attention_mfma_kernel");
    const AttnCall call = {p, g, a.q, a.keys, a.values, a.out, lse, a.lens, a.starts};
    kernel<<<dim3(uint32_t(blocks)), S::NW * WAVE, S::LDS, s>>>(call);
    return hipGetLastError();
}

template <typename E, int DP>
hipError_t weights_go(const dc_attention_args &a, const AttnPlan &p, const AttnGrid &g, const float *lse, hipStream_t s) {
    auto kernel = attention_weights_kernel<E, DP>;
    constexpr int BM = DP * sizeof(E) <= 512 ? 64 : 32, LDS = 2 * BM * DP * int(sizeof(E));
    static thread_local uint64_t raised = 0;
    const hipError_t err = raise_lds((const void *)kernel, LDS, raised);
    if (err != hipSuccess) return err;
    const int64_t blocks = ceil_div64(int64_t(a.max_pages) * a.page_size, 128);
    note_kernel("attention_weights_kernel");
    kernel<<<dim3(uint32_t(blocks), p.kv_heads, p.streams), 256, LDS, s>>>(p, g.by_group, (const E *)a.q, lse, (const E *)a.keys, a.weights,
                                                                           a.lens, a.starts);
    return hipGetLastError();
}

template <typename E, int DP, Pages PAGES>
hipError_t attention_pages(const dc_attention_args &a, const AttnPlan &p, const AttnGrid &g, float *lse, hipStream_t s) {
    if (g.block_rows == 32) return attention_go<E, DP, true, false, PAGES>(a, p, g, lse, s);
    if constexpr (DP * sizeof(E) > 256)
        if (g.block_rows == 64) return attention_go<E, DP, false, true, PAGES>(a, p, g, lse, s);
    return attention_go<E, DP, false, false, PAGES>(a, p, g, lse, s);
}

template <typename E, int DP>
hipError_t attention_dp(const dc_attention_args &a, const AttnPlan &p, const AttnGrid &g, float *lse, hipStream_t s) {
    // Tiles start at multiples of 32: in pages of a multiple of 32 slots they touch one page, in larger ones two at
    // most, and two in pages of 16.  A token of 32 streams over 32640 slots, 128 elements, 16 bit: 156 us in ONE
    // (64 slots a page), 164 / 167 us in TWO and 337 / 318 us in MANY (49 / 16 slots), where a lane's look at the
    // table waits for the tiles on their way; 16320 tokens in 32 frames: 645, 775 / 754 and 913 / 884 us.
    // A page of 4 GiB has no 32-bit size.
    const int ps = p.pool.page_size;
    const Pages pages = int64_t(p.kv_heads) * ps * p.dim * int(sizeof(E)) >= (int64_t(1) << 32) ? MANY
                        : ps % 32 == 0                                                    ? ONE
                        : ps > 32 || ps == 16                                             ? TWO
                                                                                         : MANY;
    hipError_t e = pages == ONE   ? attention_pages<E, DP, ONE>(a, p, g, lse, s)
                   : pages == TWO ? attention_pages<E, DP, TWO>(a, p, g, lse, s)
                                  : attention_pages<E, DP, MANY>(a, p, g, lse, s);
    if (e == hipSuccess && g.splits > 1) {
        note_kernel("attention_join_kernel");
        attention_join_kernel<E><<<ceil_div(p.tokens * p.q_heads, 4), 256, 0, s>>>(p, g, (E *)a.out, lse, a.lens, a.starts);
        e = hipGetLastError();
    }
    if (e != hipSuccess || a.weights == nullptr) return e;
    return weights_go<E, DP>(a, p, g, lse, s);
}

AttnPlan make_plan(const dc_attention_args &a) {
    AttnPlan p = {};
    p.pool = {a.page_table, a.num_pages, a.page_size, a.max_pages, FastDiv(uint32_t(a.page_size))};
    p.tokens = a.tokens, p.q_heads = a.q_heads, p.kv_heads = a.kv_heads, p.dim = a.dim, p.group = a.q_heads / a.kv_heads;
    p.streams = a.streams, p.causal_block = a.causal_block, p.decay = a.decay;
    p.scale = a.scale;
    p.qt = a.q_token_stride, p.qh = a.q_head_stride, p.ot = a.out_token_stride, p.oh = a.out_head_stride;
    return p;
}

// Layout of the workspace: partial sums, then the log-sums.
struct Room {
    int64_t part, lse;
};
template <typename E>
Room room(const dc_attention_args &a) {
    const AttnPlan p = make_plan(a);
    Room r = {0, 0};
    r.part = part_bytes(p, plan_grid(p, a.starts != nullptr, block_rows<E>(p)));
    if (a.weights != nullptr && a.lse == nullptr) r.lse = int64_t(a.tokens) * a.q_heads * 4;
    return r;
}

template <typename E>
hipError_t attention_t(const dc_attention_args &a, AttnPlan p, hipStream_t s) {
    const Room r = room<E>(a);
    float *lse = a.lse != nullptr || a.weights == nullptr ? a.lse : (float *)((char *)a.workspace + r.part);
    AttnGrid g = plan_grid(p, a.starts != nullptr, block_rows<E>(p));
    g.part = (float *)a.workspace;
    // exponentials are powers of two; with a negative scale q changes its signs instead, so that the largest
    // product has the largest score
    p.flip = p.scale < 0.f ? sizeof(E) == 2 ? 0x80008000u : 0x80000000u : 0u;
    // (a scale of zero: as good as zero, but -inf times it stays -inf)
    p.scale = fmaxf(fabsf(p.scale) * 1.44269504088896341f, 1.2e-38f);
    return p.dim <= 64 ? attention_dp<E, 64>(a, p, g, lse, s) : p.dim <= 128 ? attention_dp<E, 128>(a, p, g, lse, s)
                                                                                 : attention_dp<E, 256>(a, p, g, lse, s);
}

}  // namespace

int64_t paged_attention_workspace(const dc_attention_args &a, int dtype) {
    const Room r = dtype == DC_F32 ? room<float>(a) : room<half_t>(a);
    return r.part + r.lse;
}

hipError_t launch_paged_attention(const dc_attention_args &a, int dtype, hipStream_t s) {
    const AttnPlan p = make_plan(a);
    if (dtype == DC_F32) return attention_t<float>(a, p, s);
    if (dtype == DC_BF16) return attention_t<bf16_t>(a, p, s);
    return attention_t<half_t>(a, p, s);
}

}  // namespace dc
