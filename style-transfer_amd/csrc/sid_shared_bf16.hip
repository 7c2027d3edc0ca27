// bf16 instances of the shared-prefix attention kernels.
#include "sid_shared_kernel.hpp"

namespace sid_shared {
int launch_bf16(const Params& p, int qt, unsigned grid, hipStream_t st) { return launch_type<__bf16>(p, qt, grid, st); }
}  // namespace sid_shared
