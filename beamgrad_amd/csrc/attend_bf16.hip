// SPDX-License-Identifier: MIT
//
// Attention over a paged cache of bfloat16 keys and values.
#include "attend_kernels.hpp"

namespace dbs_hip {

template AttendSizes attend_sizes<2>(int, int);
template hipError_t launch_attend<2>(const AttendParams&, int, int, hipStream_t);

}  // namespace dbs_hip
