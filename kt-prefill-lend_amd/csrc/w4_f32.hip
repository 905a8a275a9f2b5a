// The 4-bit products' kernels (w4_kernel.h) for one activation type.
#include "w4_kernel.h"

namespace ktmi {

int launch_w4_f32(const W4Args& a, hipStream_t stream, ktmi_w4_kernel* tell) { return launch_t<float>(a, stream, tell); }

}  // namespace ktmi
