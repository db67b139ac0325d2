// SPDX-License-Identifier: MIT
//
// Attention over a paged cache: internal interface between the C entry
// (attend.hip) and the kernels (attend_kernels.hpp, one source per data type).
#pragma once

#include <hip/hip_runtime.h>

#include <stdint.h>

#include "dbs_cuda.h"
#include "paged.hpp"

namespace dbs_hip {

constexpr int kAttendThreads = 256;  // four wavefronts
constexpr int kAttendMaxDim = 256;
constexpr int kAttendMaxTree = 512;  // drafted tokens with parents
constexpr int kAttendSequences = 256; // of a launch: a thread of each workgroup reads one's length

// Tiles of query rows of a workgroup: its four wavefronts lie along the rows, the
// keys, or two and two.
enum AttendShape : int { kRows16 = 0, kRows32 = 1, kRows64 = 2, kRows128 = 3, kAttendShapes = 4 };
constexpr int attend_rows(int shape) { return 16 << shape; }
// Wide float32 heads: 16 rows a wavefront, so tiles of 64 rows at most.
constexpr bool attend_thin(int data_type, int dim) { return data_type == DBS_CUDA_DTYPE_F32 && dim >= 128; }
constexpr AttendShape attend_most(int data_type, int dim) { return attend_thin(data_type, dim) ? kRows64 : kRows128; }

struct AttendParams {
    const void* q;
    const void* k;
    const void* v;
    int64_t qs, qn, qh;  // strides in bytes
    int64_t kp, kt, kh;
    int64_t vp, vt, vh;
    uint32_t kp16, kt16, vp16, vt16;  // of a page and a token, in 16 bytes
    PageSpan span;
    const int32_t* pages;
    const int32_t* lengths;
    const int32_t* counts;
    const int32_t* parents;
    const int32_t* shared;  // null unless beams > 1
    int32_t S, N, H, Hkv, D, K;
    Divider G, beam_rows;  // N * G rows of a beam
    int32_t shared_tiles;  // row tiles of a group's shared pages, 0 without
    int32_t own_tiles;     // row tiles of a sequence, at most
    int32_t head_items;    // items of a cache head
    int32_t unit_shift;    // a unit is the kernel's tile of keys times 2^unit_shift
    float scale;           // of the scores, times log2(e)
    float slack;           // a maximum is raised where a score passes it by so much: 2^8, of float16 2^7
    void* out;
    float* lse;
    // workspace
    int4* info;      // per item of a sequence: its first and last workgroup, whether pages are shared
    float* partial;  // per slot: [rows][width] sums, [rows] maxima, [rows] totals
    int32_t grid;    // workgroups
};

// Of a kernel: workgroups of a CU, floats of a partial result, keys of a tile.
struct AttendSizes {
    int resident, slot, keys;
};
template <int DTYPE>
AttendSizes attend_sizes(int dim, int shape);
template <int DTYPE>
hipError_t launch_attend(const AttendParams& p, int dim, int shape, hipStream_t stream);

}  // namespace dbs_hip
