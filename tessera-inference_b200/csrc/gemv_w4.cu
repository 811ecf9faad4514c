// Linear of a few token rows with 4-bit weights and group scales.
#include <algorithm>

#include "token_ops.cuh"

namespace tcb {
namespace {

// One warp per (output column, token row), lanes over the columns of a record.
template <class X, class O>
__global__ void __launch_bounds__(128) k_gemv_w4(W4Args a) {
    const int n = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (n >= a.N) return;
    const int kb = (a.K + W4_COLS - 1) / W4_COLS, rec = w4_record_bytes(a.group), r = n % W4_ROWS;
    const int xg = a.xgroup ? a.xgroup : a.K, nxg = (a.K + xg - 1) / xg;
    const uint8_t *w = static_cast<const uint8_t *>(a.w) + (int64_t)(n / W4_ROWS) * kb * rec;
    for (int m = blockIdx.y; m < a.M; m += gridDim.y) {
        const X *x = static_cast<const X *>(a.x) + m * a.ldx;
        float acc = 0.f;
        for (int b = 0; b < kb; ++b, w += rec) {
            const bf16 *s = reinterpret_cast<const bf16 *>(w + W4_CODE_BYTES) + r;
            for (int j = lane; j < W4_COLS; j += 32) {
                const int k = b * W4_COLS + j;
                if (k >= a.K) break;
                const int i = j / 32, t = j / 8 % 4, c = j % 8, nib = c / 2 + 4 * (c % 2);
                const int code = w[512 * (r / 8) + 64 * (r % 8) + 16 * t + 4 * i + nib / 2] >> (4 * (nib % 2)) & 15;
                float v = to_f32(x[k]) * (float)(code - 8) * to_f32(s[j / a.group * W4_ROWS]);
                if constexpr (sizeof(X) == 1) v *= a.xscales[(int64_t)m * nxg + k / xg];
                acc += v;
            }
        }
        w -= (int64_t)kb * rec;
        for (int o = 16; o; o >>= 1) acc += __shfl_xor_sync(~0u, acc, o);
        if (lane == 0) {
            if (a.bias) acc += a.bias[n];
            if (a.relu) acc = acc < 0.f ? 0.f : acc;
            if (a.res) acc += to_f32(static_cast<const O *>(a.res)[m * a.ldr + n]);
            static_cast<O *>(a.out)[m * a.ldo + n] = from_f32<O>(acc);
        }
    }
}

template <class X, class O>
void launch(const W4Args &a, cudaStream_t st) {
    k_gemv_w4<X, O><<<dim3((a.N + 3) / 4, std::min(a.M, 65535)), 128, 0, st>>>(a);
}

template <class X>
void launch_o(const W4Args &a, int otype, cudaStream_t st) {
    if (otype == TCB_BF16) launch<X, bf16>(a, st);
    else if (otype == TCB_F16) launch<X, f16>(a, st);
    else launch<X, float>(a, st);
}

}  // namespace

void launch_gemv_w4(const W4Args &a, int xtype, int otype, cudaStream_t st) {
    const bool codes = xtype == TCB_I8 || xtype == TCB_E4M3;
    need(codes || xtype == TCB_BF16 || xtype == TCB_F16, "xtype is not TCB_BF16, TCB_F16, TCB_I8 or TCB_E4M3");
    need(otype == TCB_BF16 || otype == TCB_F16 || otype == TCB_F32, "otype is not TCB_BF16, TCB_F16 or TCB_F32");
    need(a.M >= 0 && w4_bytes(a.N, a.K, a.group) > 0, "M is negative, N < 1, K is not in 1..2^20 or group is not 32, 64 or 128");
    need(codes ? a.xgroup == 0 || a.xgroup == 32 || a.xgroup == 64 || a.xgroup == 128 : a.xgroup == 0,
         codes ? "xgroup is not 0, 32, 64 or 128" : "xgroup without 8-bit x");
    need(codes == (a.xscales != nullptr), codes ? "xscales is NULL" : "xscales without 8-bit x");
    need(a.ldx >= a.K && a.ldo >= a.N && (!a.res || a.ldr >= a.N), "a row pitch is smaller than the row");
    if (a.M == 0) return;
    need(a.x && a.w && a.out, "x, w or out is NULL");
    need(reinterpret_cast<uintptr_t>(a.w) % 16 == 0, "w is not 16-byte aligned");
    need(a.res != a.out || !a.res || a.ldr == a.ldo || a.M == 1, "res is out with another pitch");
    if (xtype == TCB_BF16) launch_o<bf16>(a, otype, st);
    else if (xtype == TCB_F16) launch_o<f16>(a, otype, st);
    else if (xtype == TCB_I8) launch_o<int8_t>(a, otype, st);
    else launch_o<e4m3>(a, otype, st);
    check_token_launch("k_gemv_w4");
}

}  // namespace tcb
