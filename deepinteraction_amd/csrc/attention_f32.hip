// The attention kernels of attention_fwd.h and attention_bwd.h for one element type.
#include "attention_launch.h"

namespace di {
namespace at {
template int launch_fwd<DI_F32>(const Args &, const Plan &, hipStream_t);
template int launch_bwd<DI_F32>(const Args &, const Plan &, const Plan &, hipStream_t);
}  // namespace at
}  // namespace di
