// zq_paged.cuh -- a batch of requests over a paged key/value cache, as the
// append and attention kernels see it.
//
// Rows are the new tokens of all requests, one request after the other: request
// b owns rows [starts[b], starts[b + 1]).  lengths[b] counts its own cached
// tokens, the new ones included, so its i-th row of n stands at position
// lengths[b] - n + i.  What device memory says is clamped to what the call's
// sizes allow, so that no table, length or start can lead outside them.
#pragma once

#include "zq_common.cuh"
#include "zq_kernels.h"

namespace zq {

struct Request {
    int first;   // first row
    int rows;    // new tokens
    int length;  // own cached tokens, new ones included
};

__device__ __forceinline__ Request load_request(const PagedBatch& p, int b) {
    Request r;
    if (p.starts) {
        const int a = load_l2(p.starts + b), e = load_l2(p.starts + b + 1);
        r.first = min(max(a, 0), p.rows);
        r.rows = min(max(e, r.first), p.rows) - r.first;
    } else {
        r.first = b;
        r.rows = 1;
    }
    // a tile's end behind the last token stays an int
    const long long most = min((long long)p.max_pages * p.page, 0x7FFFFFFFLL - 4096);
    const int n = load_l2(p.lengths + b);
    r.length = (int)(n < 0 ? 0 : n < most ? (long long)n : most);
    return r;
}

// The last index of starts[0 .. requests] that is at most t, or -1: a search by a
// whole warp, 32 places a round (one round up to 32 requests, two up to 1024).
__device__ __forceinline__ int last_start(const PagedBatch& p, int t) {
    const int lane = threadIdx.x & 31;
    // invariant: the last index with starts[i] <= t is in [lo, lo + n), or there is none
    int lo = 0, n = p.requests + 1;
    while (n > 1) {
        const int step = (n + 31) / 32;
        const int i = lo + lane * step;
        const bool below = lane * step < n && load_l2(p.starts + i) <= t;
        const unsigned m = __ballot_sync(0xffffffffu, below);
        if (m == 0) return -1;
        const int last = 31 - __clz(m);
        n = min(step, n - last * step);
        lo += last * step;
    }
    return lo;
}
__device__ __forceinline__ int owner(const PagedBatch& p, int b, int t) {
    if (b < 0 || b >= p.requests) return -1;
    return load_l2(p.starts + b) <= t && t < load_l2(p.starts + b + 1) ? b : -1;
}
// The request that owns row t, or -1, found by a whole warp.
__device__ __forceinline__ int request_of_row(const PagedBatch& p, int t) {
    if (!p.starts) return t < p.requests ? t : -1;
    return owner(p, last_start(p, t), t);
}
// The same of a row a lane, all in [first, last]: the whole warp finds the requests of
// the two, a lane its own between them.
__device__ __forceinline__ int request_of_lane(const PagedBatch& p, int first, int last, int t) {
    if (!p.starts) return t < p.requests ? t : -1;
    int lo = max(last_start(p, first), 0), hi = max(last_start(p, last), lo);
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (load_l2(p.starts + mid) <= t)
            lo = mid;
        else
            hi = mid - 1;
    }
    return owner(p, lo, t);
}

// The cache page that holds a request's own token `at`, or -1.
__device__ __forceinline__ int page_of(const PagedBatch& p, int b, int index) {
    const int id = load_l2(p.pages + (long long)b * p.ld_pages + index);
    return id >= 0 && id < p.cache_pages ? id : -1;
}

}  // namespace zq
