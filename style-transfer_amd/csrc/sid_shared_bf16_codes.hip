// Instances of the shared-prefix attention kernels: bf16 queries, keys and values held in 8 bits.
#include "sid_shared_kernel.hpp"

namespace sid_shared {
int launch_bf16_codes(const Params& p, int fmt, int qt, unsigned grid, hipStream_t st) {
    return fmt == SID_KV_INT8 ? launch_type<__bf16, SID_KV_INT8>(p, qt, grid, st) : launch_type<__bf16, SID_KV_E4M3>(p, qt, grid, st);
}
}  // namespace sid_shared
