// Rotary positions on the heads of token rows.
#include <algorithm>

#include "token_ops.cuh"

namespace tcb {
namespace {

// cos and sin (times mscale) of pos * freq. The angle is reduced to a fraction
// of a turn in f64, so a far position keeps its phase; the fraction is then
// within half a turn, where f32 holds it to 2^-26 turns.
template <class P>
__device__ __forceinline__ float2 turn_of(P pos, double freq, float mscale, float sign) {
    const double turns = (double)pos * freq * 0.15915494309189533577;  // 1 / (2 pi)
    float s, c;
    sincospif(2.f * (float)(turns - rint(turns)), &s, &c);
    return make_float2(c * mscale, s * mscale * sign);
}

// One thread per (row, pair or copied column), over the heads.
template <class T, class P, bool INTER>
__global__ void __launch_bounds__(256) k_rope(RopeArgs a) {
    const int half = a.rot / 2, units = half + a.hd - a.rot;
    const int64_t n = a.M * units;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / units;
        const int u = (int)(i - r * units);
        const T *x = static_cast<const T *>(a.x) + r * a.ldx;
        T *o = static_cast<T *>(a.out) + r * a.ldo;
        if (u < half) {
            const float2 t = turn_of(static_cast<const P *>(a.pos)[r * a.pos_stride], a.freq[u], a.mscale, a.sign);
            const int p = INTER ? 2 * u : u, q = INTER ? p + 1 : u + half;
            for (int h = 0; h < a.heads; ++h) {
                const float v = to_f32(x[h * a.hsx + p]), w = to_f32(x[h * a.hsx + q]);
                o[h * a.hso + p] = from_f32<T>(v * t.x - w * t.y);
                o[h * a.hso + q] = from_f32<T>(v * t.y + w * t.x);
            }
        } else {
            const int c = u - half + a.rot;
            for (int h = 0; h < a.heads; ++h) o[h * a.hso + c] = x[h * a.hsx + c];
        }
    }
}

template <class T, class P>
void launch(const RopeArgs &a, bool inter, cudaStream_t st) {
    const int64_t n = a.M * (a.hd - a.rot / 2);
    const unsigned grid = (unsigned)std::min<int64_t>((n + 255) / 256, 1 << 20);
    if (inter) k_rope<T, P, true><<<grid, 256, 0, st>>>(a);
    else k_rope<T, P, false><<<grid, 256, 0, st>>>(a);
}

template <class T>
void launch_p(const RopeArgs &a, int pos_type, bool inter, cudaStream_t st) {
    if (pos_type == TCB_F32) launch<T, float>(a, inter, st);
    else if (pos_type == TCB_I32) launch<T, int32_t>(a, inter, st);
    else launch<T, int64_t>(a, inter, st);
}

}  // namespace

void launch_rope(const RopeArgs &a, int dtype, int pos_type, bool inter, cudaStream_t st) {
    need(dtype == TCB_BF16 || dtype == TCB_F16 || dtype == TCB_F32, "dtype is not TCB_BF16, TCB_F16 or TCB_F32");
    need(pos_type == TCB_F32 || pos_type == TCB_I32 || pos_type == TCB_I64,
         "pos_type is not TCB_F32, TCB_I32 or TCB_I64");
    need(a.M >= 0 && a.heads >= 1 && a.heads <= 65535, "M is negative or heads is not in 1..65535");
    need(a.hd >= 2 && a.hd <= 1024, "hd is not in 2..1024");
    need(a.rot >= 2 && a.rot <= a.hd && a.rot % 2 == 0, "rot is not even or not in 2..hd");
    need(a.hsx >= a.hd && a.hso >= a.hd, "a head stride is smaller than hd");
    need(a.pos_stride >= 0, "pos_stride is negative");
    // heads inside a row or rows inside a head's plane: either way no two elements of out meet
    const int64_t row = (a.heads - 1) * a.hso + a.hd, plane = a.M > 0 ? (a.M - 1) * a.ldo + a.hd : 0;
    need(a.ldx >= 0 && a.ldo >= 0, "a row pitch is negative");
    need(a.M <= 1 || a.ldo >= row || (a.ldo >= a.hd && a.hso >= plane), "rows overlap in out");
    if (a.M == 0) return;
    need(a.x && a.pos && a.freq && a.out, "x, pos, freq or out is NULL");
    need(a.out != a.x || ((a.ldo == a.ldx || a.M == 1) && (a.hso == a.hsx || a.heads == 1)),
         "out is x with other strides");
    if (dtype == TCB_BF16) launch_p<bf16>(a, pos_type, inter, st);
    else if (dtype == TCB_F16) launch_p<f16>(a, pos_type, inter, st);
    else launch_p<float>(a, pos_type, inter, st);
    check_token_launch("k_rope");
}

}  // namespace tcb
