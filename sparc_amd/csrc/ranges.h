// Memory that a launch writes must belong to one tensor alone: two workgroups that update the same element race.
#pragma once
#include <algorithm>
#include <new>

#include "common.h"

struct MemoryRange {
    uintptr_t from, to;
    bool written;
};

// Host.  range(i), i in [0, n): SPARC_ERR_OVERLAP where one that is written shares a byte with another, whatever the order
// (empty ranges share none).  The 32 ranges of an Adam step of eight tensors take 0.7 us on the host, 128 ranges 3.5.
template <typename F>
int check_ranges(const int64_t n, F&& range) {
    constexpr int64_t FEW = 256;
    MemoryRange few[FEW], *r = few;
    if (n > FEW && !(r = new (std::nothrow) MemoryRange[n])) return SPARC_ERR_SIZE;
    int64_t count = 0;
    for (int64_t i = 0; i < n; ++i) {
        const MemoryRange next = range(i);
        if (next.to > next.from) r[count++] = next;
    }
    std::sort(r, r + count, [](const MemoryRange& a, const MemoryRange& b) { return a.from < b.from; });
    uintptr_t any = 0, written = 0;   // where the ranges so far, and those written, end
    int rc = SPARC_OK;
    for (int64_t i = 0; i < count && rc == SPARC_OK; ++i) {
        if (r[i].from < (r[i].written ? any : written)) rc = SPARC_ERR_OVERLAP;
        any = std::max(any, r[i].to);
        if (r[i].written) written = std::max(written, r[i].to);
    }
    if (r != few) delete[] r;
    return rc;
}

// Of Adam records: parameters and moments are written, gradients read (and may be shared).
inline int check_adam_ranges(const int64_t n_tensors, const sparc_adam_tensor_t* t) {
    return check_ranges(4 * n_tensors, [t](const int64_t i) {
        const sparc_adam_tensor_t& a = t[i >> 2];
        const void* p[4] = {a.p, a.m, a.v, a.g};
        const uintptr_t from = reinterpret_cast<uintptr_t>(p[i & 3]);
        return MemoryRange{from, from + 4 * static_cast<uintptr_t>(a.n), (i & 3) < 3};
    });
}
