// Linear of a few token rows with 4-bit weights and group scales.
//
// Bound: the bytes of the weights, read once per tile of up to 32 token rows.
// The products run on mma.sync m16n8k16: 16 weight rows are its M side, 8 token
// rows its N side. With one to 32 columns on that side the tensor pipe has
// nothing to win, the weights' codes arrive in the order of the instruction's
// A operand, and a code is turned into a 16-bit float with one logic and one
// subtract instruction per pair. A code times an activation is exact in f32,
// where the sums are kept; a group's sum is multiplied by its scale in f32.
#include <algorithm>

#include "token_ops.cuh"

namespace tcb {
namespace {

constexpr int W4_WARPS = 8, W4_THREADS = W4_WARPS * 32;
constexpr int W4_AHEAD = 4;      // records a warp loads ahead, in registers
constexpr int RED_PITCH = 20;    // floats between token rows of a warp's partial sums: no bank conflicts
constexpr int X_PAD = 32;        // 16-bit elements behind a staged token row, for the same reason
constexpr int X_BYTES = 64 * 1024;  // shared memory for staged token rows

template <class X>
using mma_type = std::conditional_t<std::is_same_v<X, f16>, f16, bf16>;

__device__ __forceinline__ uint4 ldg_stream(const void *p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p));
    return v;
}

template <class T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same_v<T, bf16>)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Codes q + 8 in nibbles p and p + 4 of w as two floats q. A code in the low bits of the significand of 128 (bf16) or
// 1024 (fp16) adds exactly its value; 136 or 1032 is subtracted, exactly.
template <class T>
__device__ __forceinline__ uint32_t codes2(uint32_t w, int p) {
    uint32_t v = w >> (4 * p);
    if constexpr (std::is_same_v<T, bf16>) {
        asm("lop3.b32 %0, %0, 0x000f000f, 0x43004300, 0xea;" : "+r"(v));  // (v & mask) | 128
        const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162 *>(&v), __nv_bfloat162{bf16(136.f), bf16(136.f)});
        return *reinterpret_cast<const uint32_t *>(&r);
    } else {
        asm("lop3.b32 %0, %0, 0x000f000f, 0x64006400, 0xea;" : "+r"(v));  // (v & mask) | 1024
        const __half2 r = __hsub2(*reinterpret_cast<const __half2 *>(&v), __half2{f16(1032.f), f16(1032.f)});
        return *reinterpret_cast<const uint32_t *>(&r);
    }
}

// 8 elements of x as the matrix instruction's type; 8-bit values are exact in bf16.
template <class X>
__device__ __forceinline__ uint4 as_mma8(const X *p) {
    if constexpr (sizeof(X) == 2) return *reinterpret_cast<const uint4 *>(p);
    const uint2 q = *reinterpret_cast<const uint2 *>(p);
    X v[8];
    memcpy(v, &q, 8);
    return make_uint4(pack_bf16x2(to_f32(v[0]), to_f32(v[1])), pack_bf16x2(to_f32(v[2]), to_f32(v[3])),
                      pack_bf16x2(to_f32(v[4]), to_f32(v[5])), pack_bf16x2(to_f32(v[6]), to_f32(v[7])));
}
template <class X>
__device__ __forceinline__ mma_type<X> as_mma1(X v) {
    if constexpr (sizeof(X) == 2) return v;
    else return __float2bfloat16_rn(to_f32(v));
}

// How a launch cuts the work: warps of a block are `wr` tiles of 16 weight rows times 8 / wr slices of the records;
// `rc` records are staged at a time (a multiple of the slices).
struct W4Cut {
    int wr = 1, rc = 0;
    bool vec = false;  // x rows can be read in 8-element steps
};

// X: type of x. SUB: columns whose products share both scales. NT: tiles of 8 token rows. XG: x's scales change along a row.
template <class X, int SUB, int NT, bool XG>
__global__ void __launch_bounds__(W4_THREADS) k_gemv_w4(W4Args a, W4Cut cut, int otype) {
    using T = mma_type<X>;
    extern __shared__ __align__(16) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int wks = W4_WARPS / cut.wr, wr = warp / wks, wk = warp % wks;
    const int kb = (a.K + W4_COLS - 1) / W4_COLS, rec = w4_record_bytes(a.group), tiles = (a.N + W4_ROWS - 1) / W4_ROWS;
    const int tile = blockIdx.x * cut.wr + wr;
    const int m0 = blockIdx.y * 8 * NT, rows = min(8 * NT, a.M - m0);
    const int pitch = cut.rc * W4_COLS + X_PAD;
    T *xs = reinterpret_cast<T *>(smem);
    const int xg = a.xgroup ? a.xgroup : a.K, nxg = (a.K + xg - 1) / xg, xgs = XG ? cut.rc * W4_COLS / xg : 0;
    float *xsc = reinterpret_cast<float *>(smem + (size_t)rows * pitch * 2);
    const X *x = static_cast<const X *>(a.x) + (int64_t)m0 * a.ldx;
    const uint8_t *w = static_cast<const uint8_t *>(a.w) + (int64_t)tile * kb * rec;
    const int mine = tile < tiles ? (kb - wk + wks - 1) / wks : 0;  // records of this warp: wk, wk + wks, ...

    uint4 q[W4_AHEAD][2];
    uint32_t sw[W4_AHEAD];
    const int words = W4_COLS / a.group * W4_ROWS / 2;  // scales of a record, two to a word: one word per lane
    const auto fetch = [&](int i, int end, int slot) {
        if (i < end) {
            const uint8_t *p = w + (int64_t)(wk + i * wks) * rec;
            q[slot][0] = ldg_stream(p + lane * 16);
            q[slot][1] = ldg_stream(p + 512 + lane * 16);
            sw[slot] = lane < words ? __ldg(reinterpret_cast<const uint32_t *>(p + W4_CODE_BYTES) + lane) : 0;
        }
    };

    int brow[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) brow[n] = min(8 * n + g, rows - 1) * pitch + 8 * t;

    float acc[NT][4] = {};
    const int per = cut.rc / wks;  // records of a warp per stage
    for (int c0 = 0, i0 = 0; c0 < kb; c0 += cut.rc, i0 += per) {
        // the stage's first records are on their way while its token rows are written
        const int end = min(mine, i0 + per);
#pragma unroll
        for (int s = 0; s < W4_AHEAD; ++s) fetch(i0 + s, end, s);
        if (c0) __syncthreads();
        const int k0 = c0 * W4_COLS, kn = min(cut.rc, kb - c0) * W4_COLS;
        if (cut.vec) {
            for (int e = threadIdx.x; e < rows * (kn / 8); e += W4_THREADS) {
                const int m = e / (kn / 8), k = (e - m * (kn / 8)) * 8;
                const X *p = x + m * a.ldx + k0 + k;
                uint4 v = make_uint4(0, 0, 0, 0);
                if (k0 + k + 8 <= a.K) v = as_mma8(p);
                else {
                    T u[8];
                    for (int j = 0; j < 8; ++j) u[j] = k0 + k + j < a.K ? as_mma1(p[j]) : T(0.f);
                    memcpy(&v, u, 16);
                }
                *reinterpret_cast<uint4 *>(xs + m * pitch + k) = v;
            }
        } else {
            for (int m = 0; m < rows; ++m)
                for (int k = threadIdx.x; k < kn; k += W4_THREADS)
                    xs[m * pitch + k] = k0 + k < a.K ? as_mma1(x[m * a.ldx + k0 + k]) : T(0.f);
        }
        if constexpr (XG)
            for (int e = threadIdx.x; e < rows * xgs; e += W4_THREADS) {
                const int m = e / xgs, k = k0 / xg + e - m * xgs;
                xsc[e] = k < nxg ? a.xscales[(int64_t)(m0 + m) * nxg + k] : 0.f;
            }
        __syncthreads();
        for (int i = i0; i < end; i += W4_AHEAD) {
#pragma unroll
            for (int s = 0; s < W4_AHEAD; ++s) {
                if (i + s >= end) break;
                const uint4 lo = q[s][0], hi = q[s][1];
                const uint32_t scales = sw[s];
                fetch(i + s + W4_AHEAD, end, s);
                const uint32_t wl[4] = {lo.x, lo.y, lo.z, lo.w}, wh[4] = {hi.x, hi.y, hi.z, hi.w};
                const int kl = (wk + (i + s) * wks - c0) * W4_COLS;
                float sum[NT][4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (j * 32 % SUB == 0) {
#pragma unroll
                        for (int n = 0; n < NT; ++n)
#pragma unroll
                            for (int c = 0; c < 4; ++c) sum[n][c] = 0.f;
                    }
                    uint32_t A[2][4];
#pragma unroll
                    for (int p = 0; p < 4; ++p) {
                        A[p / 2][p % 2 * 2] = codes2<T>(wl[j], p);
                        A[p / 2][p % 2 * 2 + 1] = codes2<T>(wh[j], p);
                    }
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        const uint4 b = *reinterpret_cast<const uint4 *>(xs + brow[n] + kl + 32 * j);
                        mma16816<T>(sum[n], A[0], b.x, b.y);
                        mma16816<T>(sum[n], A[1], b.z, b.w);
                    }
                    if ((j + 1) * 32 % SUB == 0) {
                        const int word = j * 32 / a.group * (W4_ROWS / 2) + g / 2;
                        const uint32_t u = __shfl_sync(~0u, scales, word), v = __shfl_sync(~0u, scales, word + 4);
                        const float su = g % 2 ? bf16hi(u) : bf16lo(u), sv = g % 2 ? bf16hi(v) : bf16lo(v);
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            float x0 = 1.f, x1 = 1.f;
                            if constexpr (XG) {
                                const int k = (kl + 32 * j) / xg;
                                x0 = xsc[min(8 * n + 2 * t, rows - 1) * xgs + k];
                                x1 = xsc[min(8 * n + 2 * t + 1, rows - 1) * xgs + k];
                            }
                            acc[n][0] = fmaf(sum[n][0], XG ? su * x0 : su, acc[n][0]);
                            acc[n][1] = fmaf(sum[n][1], XG ? su * x1 : su, acc[n][1]);
                            acc[n][2] = fmaf(sum[n][2], XG ? sv * x0 : sv, acc[n][2]);
                            acc[n][3] = fmaf(sum[n][3], XG ? sv * x1 : sv, acc[n][3]);
                        }
                    }
                }
            }
        }
    }

    // the slices' sums meet in shared memory, in slice order
    __syncthreads();
    float *red = reinterpret_cast<float *>(smem);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 4; ++c)
            red[(warp * 8 * NT + 8 * n + 2 * t + c % 2) * RED_PITCH + g + c / 2 * 8] = acc[n][c];
    __syncthreads();
    const int width = cut.wr * W4_ROWS;
    for (int e = threadIdx.x; e < rows * width; e += W4_THREADS) {
        const int m = e / width, r = e - m * width, n = blockIdx.x * width + r;
        if (n >= a.N) continue;
        const float *p = red + ((r / W4_ROWS) * wks * 8 * NT + m) * RED_PITCH + r % W4_ROWS;
        float v = 0.f;
        for (int k = 0; k < wks; ++k) v += p[k * 8 * NT * RED_PITCH];
        if constexpr (sizeof(X) == 1 && !XG) v *= a.xscales[m0 + m];
        if (a.bias) v += a.bias[n];
        if (a.relu) v = v < 0.f ? 0.f : v;
        const int64_t at = (int64_t)(m0 + m) * a.ldo + n, ar = (int64_t)(m0 + m) * a.ldr + n;
        if (otype == TCB_BF16) {
            if (a.res) v += to_f32(static_cast<const bf16 *>(a.res)[ar]);
            static_cast<bf16 *>(a.out)[at] = from_f32<bf16>(v);
        } else if (otype == TCB_F16) {
            if (a.res) v += to_f32(static_cast<const f16 *>(a.res)[ar]);
            static_cast<f16 *>(a.out)[at] = from_f32<f16>(v);
        } else {
            if (a.res) v += static_cast<const float *>(a.res)[ar];
            static_cast<float *>(a.out)[at] = v;
        }
    }
}

template <class X, int SUB, int NT, bool XG>
void launch(const W4Args &a, int otype, cudaStream_t st) {
    const int kb = (a.K + W4_COLS - 1) / W4_COLS, tiles = (a.N + W4_ROWS - 1) / W4_ROWS;
    const int mt = (int)((a.M + 8ll * NT - 1) / (8 * NT)), rows = std::min(a.M, 8 * NT);
    W4Cut cut;
    cut.vec = reinterpret_cast<uintptr_t>(a.x) % (8 * sizeof(X)) == 0 && a.ldx % 8 == 0;
    while (cut.wr < W4_WARPS && (int64_t)tiles * mt >= 296 * 2 * cut.wr) cut.wr *= 2;
    const int wks = W4_WARPS / cut.wr;
    const int row_bytes = W4_COLS * 2 + (XG ? W4_COLS / a.xgroup * 4 : 0);  // of a staged record
    cut.rc = std::max(wks, std::min((kb + wks - 1) / wks * wks, X_BYTES / (rows * row_bytes) / wks * wks));
    const size_t smem = std::max<size_t>((size_t)rows * (cut.rc * row_bytes + X_PAD * 2),
                                         (size_t)W4_WARPS * 8 * NT * RED_PITCH * 4);
    if (smem > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(k_gemv_w4<X, SUB, NT, XG>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        need(e == cudaSuccess, cudaGetErrorString(e));
    }
    // token tiles beyond the grid's 65,535 rows: several launches
    for (int64_t m = 0; m < a.M; m += 65535 * 8 * NT) {
        W4Args p = a;
        const size_t xb = sizeof(X), ob = otype == TCB_F32 ? 4 : 2;
        p.M = (int)std::min<int64_t>(a.M - m, 65535 * 8 * NT);
        p.x = static_cast<const uint8_t *>(a.x) + m * a.ldx * xb;
        p.out = static_cast<uint8_t *>(a.out) + m * a.ldo * ob;
        if (a.res) p.res = static_cast<const uint8_t *>(a.res) + m * a.ldr * ob;
        if (a.xscales) p.xscales = a.xscales + m * (a.xgroup ? (a.K + a.xgroup - 1) / a.xgroup : 1);
        const dim3 grid((tiles + cut.wr - 1) / cut.wr, (p.M + 8 * NT - 1) / (8 * NT));
        k_gemv_w4<X, SUB, NT, XG><<<grid, W4_THREADS, smem, st>>>(p, cut, otype);
    }
}

// Token rows are cut into equal tiles of at most 32.
template <class X, int SUB, bool XG>
void launch_n(const W4Args &a, int otype, cudaStream_t st) {
    const int64_t mt = (a.M + 31ll) / 32, nt = ((a.M + mt - 1) / mt + 7) / 8;
    if (nt == 1) launch<X, SUB, 1, XG>(a, otype, st);
    else if (nt == 2) launch<X, SUB, 2, XG>(a, otype, st);
    else if (nt == 3) launch<X, SUB, 3, XG>(a, otype, st);
    else launch<X, SUB, 4, XG>(a, otype, st);
}

template <class X, bool XG>
void launch_s(const W4Args &a, int otype, cudaStream_t st) {
    const int sub = XG ? std::min(a.group, a.xgroup) : a.group;
    if (sub == 32) launch_n<X, 32, XG>(a, otype, st);
    else if (sub == 64) launch_n<X, 64, XG>(a, otype, st);
    else launch_n<X, 128, XG>(a, otype, st);
}

template <class X>
void launch_x(const W4Args &a, int otype, cudaStream_t st) {
    if constexpr (sizeof(X) == 1) {
        if (a.xgroup) return launch_s<X, true>(a, otype, st);
    }
    launch_s<X, false>(a, otype, st);
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
    if (xtype == TCB_BF16) launch_x<bf16>(a, otype, st);
    else if (xtype == TCB_F16) launch_x<f16>(a, otype, st);
    else if (xtype == TCB_I8) launch_x<int8_t>(a, otype, st);
    else launch_x<e4m3>(a, otype, st);
    check_token_launch("k_gemv_w4");
}

}  // namespace tcb
