// Root-mean-square norm: the kernels for f16 rows.
#include "rmsnorm.cuh"

namespace tcb {

void rms_launch_f16(const RmsArgs &a, int ytype, RmsMode mode, cudaStream_t st) { rms_launch_type<f16>(a, ytype, mode, st); }

}  // namespace tcb
