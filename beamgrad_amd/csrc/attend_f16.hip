// SPDX-License-Identifier: MIT
//
// Attention over a paged cache of float16 keys and values.
#include "attend_kernels.hpp"

namespace dbs_hip {

template AttendSizes attend_sizes<1>(int, int);
template hipError_t launch_attend<1>(const AttendParams&, int, int, hipStream_t);

}  // namespace dbs_hip
