// The paged cache of the frame-attention operators: slot -> page -> row, and where the new tokens
// of a stream lie.
#pragma once

#include "common.hpp"

namespace dc {

// Division of 0 <= n < 2^31 by a constant d in 1 .. 2^31 - 1: with l = ceil(log2 d) and
// m = ceil(2^(31 + l) / d) < 2^32 the quotient is (n * m) >> (31 + l), exact because
// m * d - 2^(31 + l) < d <= 2^l.
struct FastDiv {
    uint32_t d, m;
    int32_t shift;
    FastDiv() = default;
    explicit FastDiv(uint32_t div) : d(div) {
        int l = 0;
        while ((1ull << l) < div) ++l;
        shift = 31 + l;
        m = uint32_t(((1ull << shift) + div - 1) / div);
    }
    __host__ __device__ __forceinline__ uint32_t quot(uint32_t n) const { return uint32_t((uint64_t(n) * m) >> shift); }
    __host__ __device__ __forceinline__ uint32_t mod(uint32_t n) const { return n - quot(n) * d; }
};

struct PagePool {
    const int32_t *table;  // [streams][max_pages]
    int32_t num_pages, page_size, max_pages;
    FastDiv by_page;
};

// Row (head h of the pool [page][kv_heads][page_size]) of slot s of the stream whose page table is
// `table`, or -1 if it lies in no page of the pool.
__device__ __forceinline__ int64_t slot_row(const PagePool &p, const int32_t *table, int s, int kv_heads, int h) {
    const uint32_t i = p.by_page.quot(uint32_t(s));
    if (s < 0 || int(i) >= p.max_pages) return -1;
    const int32_t page = table[i];
    if (uint32_t(page) >= uint32_t(p.num_pages)) return -1;
    return (int64_t(page) * kv_heads + h) * p.page_size + (s - int(i) * p.page_size);
}

// First token and number of tokens of stream b, inside [0, tokens] whatever `starts` holds.
__device__ __forceinline__ void stream_tokens(const int32_t *starts, int b, int streams, int tokens, int &first, int &count) {
    if (starts == nullptr) {
        count = tokens / streams;
        first = b * count;
        return;
    }
    first = min(max(starts[b], 0), tokens);
    count = min(max(starts[b + 1], first), tokens) - first;
}

// Stream of token t, or -1 behind the last one: the last b with starts[b] <= t (streams without
// tokens share their start with the next one).
__device__ __forceinline__ int stream_of(const int32_t *starts, int streams, int tokens, int t) {
    if (starts == nullptr) return t / (tokens / streams);
    if (t < starts[0] || t >= starts[streams]) return -1;
    int lo = 0, hi = streams;  // starts[lo] <= t < starts[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (starts[mid] <= t) lo = mid;
        else hi = mid;
    }
    return lo;
}

}  // namespace dc
