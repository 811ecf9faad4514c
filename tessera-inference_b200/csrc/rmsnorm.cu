// Root-mean-square norm: the checks, and the kernels for bf16 rows.
#include "rmsnorm.cuh"

namespace tcb {

void launch_rmsnorm(RmsArgs a, int dtype, int ytype, cudaStream_t st) {
    need(dtype == TCB_BF16 || dtype == TCB_F16 || dtype == TCB_F32, "dtype is not TCB_BF16, TCB_F16 or TCB_F32");
    const bool codes = ytype == TCB_I8 || ytype == TCB_E4M3;
    need(codes || ytype == dtype, "ytype is neither dtype, TCB_I8 nor TCB_E4M3");
    need(a.M >= 0 && a.D >= 1 && a.D <= RMS_MAX_TEAM * RMS_MAX_UNITS * RMS_UNIT, "M is negative or D is not in 1..16384");
    need(a.eps >= 0.f && a.eps <= 3.4e38f, "eps is negative or not finite");
    need(codes ? a.group == 0 || a.group == 32 || a.group == 64 || a.group == 128 : a.group == 0,
         codes ? "group is not 0, 32, 64 or 128" : "group without 8-bit output");
    need(a.ldx >= a.D && a.ldy >= a.D && (!a.res || a.ldr >= a.D) && (!a.sum || a.lds >= a.D),
         "a row pitch is smaller than D");
    need(!a.sum || a.res, "sum without res");
    need(codes == (a.scales != nullptr), codes ? "scales is NULL" : "scales without 8-bit output");
    if (a.M == 0) return;
    need(a.x && a.y, "x or y is NULL");
    const int size = type_bytes(dtype);
    need(on(a.x, size) && on(a.res, size) && on(a.sum, size) && on(a.y, type_bytes(ytype)) && on(a.g, 4) && on(a.scales, 4),
         "a pointer is not aligned to its elements");
    // in place: a row's elements are read by the threads that write them
    const auto apart = [&](const void *p, int64_t ldp, const void *q, int64_t ldq) { return p != q || !p || ldp == ldq || a.M == 1; };
    need(apart(a.sum, a.lds, a.x, a.ldx) && apart(a.sum, a.lds, a.res, a.ldr) && apart(a.y, a.ldy, a.x, a.ldx) &&
             apart(a.y, a.ldy, a.sum, a.lds), "in place with another pitch");
    need(!codes || (a.y != a.x && a.y != a.res && a.y != a.sum), "8-bit output over its input");
    need(a.y != a.res || !a.res || a.sum == a.res, "y is res");  // but for y over sum over res
    a.inv_d = (float)(1.0 / a.D);
    a.shift = a.group == 128 ? 7 : a.group == 64 ? 6 : 5;
    // Where the rows start, in elements behind a boundary of 8: the same for every tensor, or one element at a time. Groups of
    // columns on rows of several warps need boundaries.
    const auto start = [](const void *p, int bytes) { return reinterpret_cast<uintptr_t>(p) / bytes % 8; };
    const auto like_x = [&](const void *p, int64_t ld, int bytes) {
        return !p || (start(p, bytes) == start(a.x, size) && (ld - a.ldx) % 8 == 0);
    };
    const bool same = like_x(a.res, a.ldr, size) && like_x(a.sum, a.lds, size) && like_x(a.y, a.ldy, codes ? 1 : size);
    const bool bounds = start(a.x, size) == 0 && a.ldx % 8 == 0;
    RmsMode mode = SINGLE;
    if (same && bounds && a.D % 8 == 0 && reinterpret_cast<uintptr_t>(a.g) % 16 == 0) mode = ALIGNED;
    else if (same && (bounds || !a.group || a.D + 7 <= 32 * RMS_MAX_UNITS * RMS_UNIT)) mode = EDGED;
    if (dtype == TCB_BF16) rms_launch_bf16(a, ytype, mode, st);
    else if (dtype == TCB_F16) rms_launch_f16(a, ytype, mode, st);
    else rms_launch_f32(a, ytype, mode, st);
    check_token_launch("k_rmsnorm");
}

void rms_launch_bf16(const RmsArgs &a, int ytype, RmsMode mode, cudaStream_t st) { rms_launch_type<bf16>(a, ytype, mode, st); }

}  // namespace tcb
