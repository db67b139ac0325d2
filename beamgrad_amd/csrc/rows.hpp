// SPDX-License-Identifier: MIT
//
// Rows of bytes copied by kernels: 16 bytes a lane, whatever their alignment
// (the hardware takes a 16-byte access at any address), the rest of a row byte
// by byte.
#pragma once

#include <hip/hip_runtime.h>

#include <stdint.h>

namespace dbs_hip {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_any __attribute__((aligned(1)));

template <class W>
struct Unaligned {
    typedef W type __attribute__((aligned(1)));
};

// Up to 16 bytes at `from`: all of them, or a row's last `left`.
__device__ __forceinline__ u32x4 load16(const char* from, int64_t left) {
    if (left >= 16) return *reinterpret_cast<const u32x4_any*>(from);
    u32x4 x = {0, 0, 0, 0};
    const int n = static_cast<int>(left);
    if (n & 8) {
        const uint64_t w = *reinterpret_cast<const Unaligned<uint64_t>::type*>(from);
        x[0] = static_cast<uint32_t>(w), x[1] = static_cast<uint32_t>(w >> 32);
    }
    uint32_t w = 0;
    if (n & 4) w = *reinterpret_cast<const Unaligned<uint32_t>::type*>(from + (n & 8));
    uint32_t t = 0;
    if (n & 2) t = *reinterpret_cast<const Unaligned<uint16_t>::type*>(from + (n & 12));
    if (n & 1) t |= static_cast<uint32_t>(static_cast<uint8_t>(from[n & 14])) << (8 * (n & 2));
    // the words lie one after the other
    uint32_t* const out = reinterpret_cast<uint32_t*>(&x);
    if (n & 8) {
        out[2] = n & 4 ? w : t;
        out[3] = n & 4 ? t : 0;
    } else {
        out[0] = n & 4 ? w : t;
        out[1] = n & 4 ? t : 0;
    }
    return x;
}

__device__ __forceinline__ void store16(char* to, u32x4 x, int64_t left) {
    if (left >= 16) {
        *reinterpret_cast<u32x4_any*>(to) = x;
        return;
    }
    const int n = static_cast<int>(left);
    if (n & 8) *reinterpret_cast<Unaligned<uint64_t>::type*>(to) = x[0] | static_cast<uint64_t>(x[1]) << 32;
    const uint32_t a = n & 8 ? x[2] : x[0], b = n & 8 ? x[3] : x[1];
    if (n & 4) *reinterpret_cast<Unaligned<uint32_t>::type*>(to + (n & 8)) = a;
    const uint32_t t = n & 4 ? b : a;
    if (n & 2) *reinterpret_cast<Unaligned<uint16_t>::type*>(to + (n & 12)) = static_cast<uint16_t>(t);
    if (n & 1) to[n & 14] = static_cast<char>(n & 2 ? t >> 16 : t);
}

// parents[i], int32 or int64, as a number of [0, n) or -1.
__device__ __forceinline__ int parent_of(const void* parents, bool i64, int64_t i, int n) {
    const int64_t p = i64 ? static_cast<const int64_t*>(parents)[i] : static_cast<const int32_t*>(parents)[i];
    return p >= 0 && p < n ? static_cast<int>(p) : -1;
}

}  // namespace dbs_hip
