// SPDX-License-Identifier: MIT
//
// A paged cache as the kernels of a model's state read it: where a token lies,
// what a page-table entry may be, how long a sequence is.
#pragma once

#include <hip/hip_runtime.h>

#include <stdint.h>

namespace dbs_hip {

// Quotients by a number of [1, 2^31) of numerators of [0, 2^31), without a
// division: q = (n * m) >> (31 + l), l = ceil(log2 d), m = floor(2^(31+l) / d)
// + 1. m * d exceeds 2^(31+l) by at most d <= 2^l, so n * m / 2^(31+l) exceeds
// n / d by at most n * 2^l / (d * 2^(31+l)) < 1 / d: the floor is n / d's.
// d > 2^(l-1), so m < 2^32: but for d = 1 the high word of n * m, shifted by l - 1,
// is all that is needed.
struct Divider {
    uint32_t d;
    uint32_t m;
    uint32_t shift;  // l - 1; of d = 1: 0, unused

    static Divider of(uint32_t d) {
        uint32_t l = 0;
        while ((uint64_t{1} << l) < d) ++l;
        return {d, static_cast<uint32_t>((uint64_t{1} << (31 + l)) / d + 1), l > 0 ? l - 1 : 0};
    }
    __host__ __device__ uint32_t quotient(uint32_t n) const {
        const uint32_t high = static_cast<uint32_t>((static_cast<uint64_t>(n) * m) >> 32);
        return d == 1 ? n : high >> shift;
    }
};

// The pages of a pool that a table's entries name.
struct PageSpan {
    Divider page;    // tokens of a page
    int32_t n_pages; // of the pool
    int32_t P;       // entries of a sequence

    __host__ __device__ bool is_page(int32_t entry) const { return static_cast<uint32_t>(entry) < static_cast<uint32_t>(n_pages); }
    // a sequence's length as the table can hold it
    __host__ __device__ int32_t length(int32_t n) const {
        const int64_t most = static_cast<int64_t>(P) * page.d;
        return n < 0 ? 0 : static_cast<int32_t>(n < most ? n : most);
    }
    __host__ __device__ int32_t held(int32_t tokens) const { // pages that hold so many tokens
        return static_cast<int32_t>(page.quotient(static_cast<uint32_t>(tokens) + page.d - 1));
    }
};

}  // namespace dbs_hip
