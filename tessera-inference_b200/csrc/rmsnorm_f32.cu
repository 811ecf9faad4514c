// Root-mean-square norm: the kernels for f32 rows.
#include "rmsnorm.cuh"

namespace tcb {

void rms_launch_f32(const RmsArgs &a, int ytype, bool vec, cudaStream_t st) { rms_launch_type<float>(a, ytype, vec, st); }

}  // namespace tcb
