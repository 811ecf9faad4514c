// Root-mean-square norm: the kernels for f32 rows.
#include "rmsnorm.cuh"

namespace tcb {

void rms_launch_f32(const RmsArgs &a, int ytype, RmsMode mode, cudaStream_t st) { rms_launch_type<float>(a, ytype, mode, st); }

}  // namespace tcb
