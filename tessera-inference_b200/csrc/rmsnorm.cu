// Root-mean-square norm of token rows, with the residual's addition in front
// and, on request, 8-bit codes with scales behind.
#include <algorithm>

#include "token_ops.cuh"

namespace tcb {
namespace {

constexpr int RMS_THREADS = 256;

template <class Op>
__device__ float block_reduce(float v, float *red, Op op) {
    for (int o = 16; o; o >>= 1) v = op(v, __shfl_xor_sync(~0u, v, o));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = red[0];
    for (int i = 1; i < RMS_THREADS / 32; ++i) v = op(v, red[i]);
    return v;
}

// One CTA per row.
template <class T, class Y>
__global__ void __launch_bounds__(RMS_THREADS) k_rmsnorm(RmsArgs a) {
    extern __shared__ float h[];
    __shared__ float red[RMS_THREADS / 32];
    const auto add = [](float p, float q) { return p + q; };
    const auto top = [](float p, float q) { return max_nan(p, q); };
    const int G = a.group ? a.group : a.D, ng = (a.D + G - 1) / G;
    for (int64_t r = blockIdx.x; r < a.M; r += gridDim.x) {
        const T *x = static_cast<const T *>(a.x) + r * a.ldx;
        const T *res = static_cast<const T *>(a.res) + r * a.ldr;
        T *sum = static_cast<T *>(a.sum) + r * a.lds;
        float ss = 0.f, big = 0.f;
        for (int c = threadIdx.x; c < a.D; c += RMS_THREADS) {
            float v = to_f32(x[c]);
            if (a.res) v = to_f32(from_f32<T>(v + to_f32(res[c])));
            if (a.sum) sum[c] = from_f32<T>(v);
            h[c] = v;
            ss += v * v;
            big = fmaxf(big, fabsf(v));
        }
        ss = block_reduce(ss, red, add);
        float pre = 1.f;
        if (isinf(ss)) {  // finite rows whose squares pass 3.4e38: scaled by a power of two first
            big = block_reduce(big, red, top);
            if (!isinf(big)) {
                pre = 0x1p-100f;
                ss = 0.f;
                for (int c = threadIdx.x; c < a.D; c += RMS_THREADS) ss += (h[c] * pre) * (h[c] * pre);
                ss = block_reduce(ss, red, add);
            }
        }
        const float rstd = 1.f / sqrtf(ss / (float)a.D + a.eps * pre * pre);
        Y *y = static_cast<Y *>(a.y) + r * a.ldy;
        for (int k = 0; k < ng; ++k) {
            const int c0 = k * G, c1 = min(a.D, c0 + G);
            if constexpr (sizeof(Y) > 1) {
                for (int c = c0 + threadIdx.x; c < c1; c += RMS_THREADS)
                    y[c] = from_f32<Y>(h[c] * pre * rstd * (a.g ? a.g[c] : 1.f));
            } else {
                float m = 0.f;
                for (int c = c0 + threadIdx.x; c < c1; c += RMS_THREADS)
                    m = max_nan(m, fabsf(h[c] * pre * rstd * (a.g ? a.g[c] : 1.f)));
                m = block_reduce(m, red, top);
                const float s = max_nan(m, 1e-12f) / code_top<Y>();
                for (int c = c0 + threadIdx.x; c < c1; c += RMS_THREADS)
                    y[c] = to_code<Y>(h[c] * pre * rstd * (a.g ? a.g[c] : 1.f) / s);
                if (threadIdx.x == 0) a.scales[r * ng + k] = s;
            }
        }
        __syncthreads();
    }
}

template <class T, class Y>
void launch(const RmsArgs &a, cudaStream_t st) {
    const size_t smem = a.D * sizeof(float);
    if (smem > 48 * 1024)
        cudaFuncSetAttribute(k_rmsnorm<T, Y>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    k_rmsnorm<T, Y><<<(unsigned)std::min<int64_t>(a.M, 1 << 20), RMS_THREADS, smem, st>>>(a);
}

template <class T>
void launch_y(const RmsArgs &a, int ytype, cudaStream_t st) {
    if (ytype == TCB_I8) launch<T, int8_t>(a, st);
    else if (ytype == TCB_E4M3) launch<T, e4m3>(a, st);
    else launch<T, T>(a, st);
}

}  // namespace

void launch_rmsnorm(const RmsArgs &a, int dtype, int ytype, cudaStream_t st) {
    need(dtype == TCB_BF16 || dtype == TCB_F16 || dtype == TCB_F32, "dtype is not TCB_BF16, TCB_F16 or TCB_F32");
    const bool codes = ytype == TCB_I8 || ytype == TCB_E4M3;
    need(codes || ytype == dtype, "ytype is neither dtype, TCB_I8 nor TCB_E4M3");
    need(a.M >= 0 && a.D >= 1 && a.D <= 16384, "M is negative or D is not in 1..16384");
    need(a.eps >= 0.f && a.eps <= 3.4e38f, "eps is negative or not finite");
    need(codes ? a.group == 0 || a.group == 32 || a.group == 64 || a.group == 128 : a.group == 0,
         codes ? "group is not 0, 32, 64 or 128" : "group without 8-bit output");
    need(a.ldx >= a.D && a.ldy >= a.D && (!a.res || a.ldr >= a.D) && (!a.sum || a.lds >= a.D),
         "a row pitch is smaller than D");
    need(!a.sum || a.res, "sum without res");
    need(codes == (a.scales != nullptr), codes ? "scales is NULL" : "scales without 8-bit output");
    if (a.M == 0) return;
    need(a.x && a.y, "x or y is NULL");
    if (dtype == TCB_BF16) launch_y<bf16>(a, ytype, st);
    else if (dtype == TCB_F16) launch_y<f16>(a, ytype, st);
    else launch_y<float>(a, ytype, st);
    check_token_launch("k_rmsnorm");
}

}  // namespace tcb
