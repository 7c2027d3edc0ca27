// Instances of the shared-prefix attention kernels: half-precision queries, keys and values of the same type.
#include "sid_shared_kernel.hpp"

namespace sid_shared {
int launch_f16(const Params& p, int qt, unsigned grid, hipStream_t st) { return launch_type<_Float16, SID_KV_NONE>(p, qt, grid, st); }
}  // namespace sid_shared
