// The kernels of attention (kv_attend.h) that leave the rows' statistics and scores behind, and take a page table for each head: kv_mass.hip and kv_sparse.hip
// call them.
#include <hip/hip_runtime.h>

#include "kv_attend.h"

namespace altius {
namespace attend {

int launch_attend_kept(DeviceCtx &ctx, const AttendArgs &g, bool bf16) { return launch_attend<KEPT>(ctx, g, bf16); }

}  // namespace attend
}  // namespace altius
