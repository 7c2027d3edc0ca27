// Instances of the shared-prefix attention kernels: bf16 queries, keys and values of the same type.
#include "sid_shared_kernel.hpp"

namespace sid_shared {
int launch_bf16(const Params& p, int qt, unsigned grid, hipStream_t st) { return launch_type<__bf16, SID_KV_NONE>(p, qt, grid, st); }
}  // namespace sid_shared
