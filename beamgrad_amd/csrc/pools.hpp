// SPDX-License-Identifier: MIT
//
// Page tables and pools as the calls that change them take them: checks of the
// C entries' arguments, and the table that a kernel reads and writes.
#pragma once

#include <hip/hip_runtime.h>

#include <stdint.h>

#include "beamgrad_state.h"
#include "paged.hpp"

namespace dbs_hip {

struct Table {
    const int32_t* pages;
    const int32_t* lengths;
    const int32_t* refs;
    int32_t* pages_out;
    int32_t* lengths_out;
    int32_t* refs_out;
    PageSpan span;
    int32_t S;
};

__device__ __forceinline__ int page_at(const Table& t, int s, int column) {
    const int32_t entry = t.pages[static_cast<int64_t>(s) * t.span.P + column];
    return t.span.is_page(entry) ? entry : -1;
}

// Tables of up to 2^30 entries: what all sequences want together is summed, and
// becomes places in a list, in 31 bits.
inline bool valid_span(int sequences, int table_pages, int n_pages, int page_tokens) {
    return sequences > 0 && table_pages > 0 && n_pages > 0 && page_tokens > 0 &&
           static_cast<int64_t>(sequences) * table_pages <= int64_t{1} << 30 &&
           (static_cast<int64_t>(table_pages) + 1) * page_tokens <= INT32_MAX - 65536;
}

inline bool valid_pools(const BeamgradPools* p) {
    if (!p || p->n < 0 || p->reserved != 0) return false;
    if (p->n > 0 && (!p->base || !p->row_bytes || !p->page_stride || !p->token_stride)) return false;
    for (int i = 0; i < p->n; ++i)
        if (!p->base[i] || p->row_bytes[i] <= 0 || p->page_stride[i] < 0 || p->token_stride[i] < 0) return false;
    return true;
}

inline bool valid_table(const BeamgradTable* t) { return t && t->pages && t->lengths && t->refs; }

// The new table is written while the old one is read: none of its parts may lie in
// it, or in each other.
inline bool tables_apart(const BeamgradTable& from, const BeamgradTable& to, int S, int P, int n_pages) {
    const int32_t* const parts[6] = {to.pages, to.lengths, to.refs, from.pages, from.lengths, from.refs};
    const int64_t size[3] = {static_cast<int64_t>(S) * P, S, n_pages};
    for (int i = 0; i < 3; ++i)
        for (int j = i + 1; j < 6; ++j) {
            const uintptr_t a = reinterpret_cast<uintptr_t>(parts[i]), b = reinterpret_cast<uintptr_t>(parts[j]);
            if (a < b + size[j % 3] * sizeof(int32_t) && b < a + size[i] * sizeof(int32_t)) return false;
        }
    return true;
}

inline Table table_of(const BeamgradTable& from, const BeamgradTable& to, int S, int P, int n_pages, int page_tokens) {
    return {from.pages, from.lengths, from.refs, to.pages, to.lengths, to.refs,
            {Divider::of(static_cast<uint32_t>(page_tokens)), n_pages, P}, S};
}

}  // namespace dbs_hip
