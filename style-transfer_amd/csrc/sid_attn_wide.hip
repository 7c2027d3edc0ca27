// Instantiation unit: the flash kernels of the widest head-dim class (145-160) in every arithmetic mode.
#include "sid_attn_kernel.hpp"

namespace sid_attn {
template int launch_flash_nw<10, 6, false, false, false>(const FlashParams&, const Geometry&, hipStream_t);
template int launch_flash_nw<10, 6, false, false, true>(const FlashParams&, const Geometry&, hipStream_t);
template int launch_flash_nw<10, 6, true, false, false>(const FlashParams&, const Geometry&, hipStream_t);
}  // namespace sid_attn
