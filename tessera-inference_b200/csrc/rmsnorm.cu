// Root-mean-square norm of token rows, with the residual's addition in front
// and, on request, 8-bit codes with scales behind.
//
// Bound: HBM. Each element of x (and res) is read once and each of sum and y
// written once; a row stays in registers between the sum of its squares and
// its output, so there is no second read. A row belongs to a team of 32, 128
// or 512 threads, the smallest whose registers hold it at 32 columns a thread.
//
// Codes: with p = h g, v / s = p Q / max|p| whatever the row's norm is, so a
// code is taken from p and Q / max|p|, both carried with their rounding error.
// It then differs from the definition's only where v / s is within a rounding
// of the middle between two codes.
#include <algorithm>

#include "token_ops.cuh"

namespace tcb {
namespace {

constexpr int UNIT = 8;       // columns per load (16 bytes of a 16-bit type)
constexpr int MAX_UNITS = 4;  // units per thread
constexpr int TEAMS[3] = {32, 128, 512};

// 8 consecutive elements at a 16-byte boundary.
template <class T>
__device__ __forceinline__ void load8(const T *p, float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
        const float4 a = reinterpret_cast<const float4 *>(p)[0], b = reinterpret_cast<const float4 *>(p)[1];
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
        v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
        const uint4 q = *reinterpret_cast<const uint4 *>(p);
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (std::is_same_v<T, bf16>) {
                v[2 * j] = bf16lo(w[j]);
                v[2 * j + 1] = bf16hi(w[j]);
            } else {
                const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[j]));
                v[2 * j] = f.x;
                v[2 * j + 1] = f.y;
            }
        }
    }
}

template <class T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (std::is_same_v<T, bf16>) return pack_bf16x2(a, b);
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}

template <class T>
__device__ __forceinline__ void store8(T *p, const float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
        reinterpret_cast<float4 *>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4 *>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else if constexpr (sizeof(T) == 2) {
        *reinterpret_cast<uint4 *>(p) =
            make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
    } else {
        uint32_t w[2] = {0, 0};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const T c = to_code<T>(v[j]);
            w[j / 4] |= (uint32_t)*reinterpret_cast<const uint8_t *>(&c) << (8 * (j % 4));
        }
        *reinterpret_cast<uint2 *>(p) = make_uint2(w[0], w[1]);
    }
}

// Sum over the team; every thread gets it. Teams of one warp use no memory.
template <int TEAM>
__device__ __forceinline__ float team_sum(float v, float *red) {
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
    if constexpr (TEAM > 32) {
        __syncthreads();
        if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
        __syncthreads();
        v = red[threadIdx.x % (TEAM / 32)];
        for (int o = TEAM / 64; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
    }
    return v;
}

// Largest magnitude over the team, as bits: magnitudes order like their bits, and a NaN is above all.
template <int TEAM>
__device__ __forceinline__ uint32_t team_max(uint32_t v, uint32_t *red) {
    v = __reduce_max_sync(~0u, v);
    if constexpr (TEAM > 32) {
        __syncthreads();
        if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
        __syncthreads();
        v = __reduce_max_sync(~0u, red[threadIdx.x % (TEAM / 32)]);
    }
    return v;
}

__device__ __forceinline__ uint32_t mag(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// What a group's codes are made with: p -> p hi + p lo, and its scale.
struct Step {
    float hi, lo, s;
};
template <class Y>
__device__ __forceinline__ Step step_of(uint32_t top_bits, float rstd) {
    const float am = __uint_as_float(top_bits), vm = am * rstd, Q = code_top<Y>();
    Step t;
    t.s = max_nan(vm, 1e-12f) / Q;
    if (vm >= 1e-12f) {
        t.hi = Q / am;
        t.lo = fmaf(-t.hi, am, Q) / am;  // the remainder of the division
    } else {  // all but zero, or NaN
        t.hi = rstd / t.s;
        t.lo = vm != vm ? vm : 0.f;
    }
    return t;
}

// VEC: unit i of thread t is columns 8 (i TEAM + t) .. + 7, one 16-byte access
// per 16-bit tensor. Otherwise (a pitch, pointer or width that is no multiple of
// 8 elements) value (i, j) is column (8 i + j) TEAM + t, so that the accesses of
// a warp are consecutive.
template <class T, class Y, int TEAM, int NU, bool VEC>
__global__ void __launch_bounds__(TEAM == 512 ? 512 : 256) k_rmsnorm(RmsArgs a) {
    constexpr int ROWS = TEAM == 32 ? 8 : 1;  // rows per block and pass
    __shared__ uint32_t red[TEAM / 32];
    __shared__ uint32_t gtop[TEAM > 32 && !VEC && sizeof(Y) == 1 ? TEAM * NU * UNIT / 32 : 1];
    const int t = threadIdx.x % TEAM, D = a.D;
    const auto col = [&](int i, int j) { return VEC ? (i * TEAM + t) * UNIT + j : (i * UNIT + j) * TEAM + t; };
    for (int64_t r = (int64_t)blockIdx.x * ROWS + threadIdx.x / TEAM; r < a.M; r += (int64_t)gridDim.x * ROWS) {
        const T *x = static_cast<const T *>(a.x) + r * a.ldx;
        const T *res = static_cast<const T *>(a.res) + r * a.ldr;
        T *sum = static_cast<T *>(a.sum) + r * a.lds;
        float h[NU][UNIT], ss = 0.f;
        if constexpr (VEC) {
            float q[NU][UNIT];
#pragma unroll
            for (int i = 0; i < NU; ++i)
                if (col(i, 0) < D) load8(x + col(i, 0), h[i]);
            if (a.res) {
#pragma unroll
                for (int i = 0; i < NU; ++i)
                    if (col(i, 0) < D) load8(res + col(i, 0), q[i]);
#pragma unroll
                for (int i = 0; i < NU; ++i)
                    if (col(i, 0) < D) {
#pragma unroll
                        for (int j = 0; j < UNIT; ++j) h[i][j] = to_f32(from_f32<T>(h[i][j] + q[i][j]));
                        if (a.sum) store8(sum + col(i, 0), h[i]);
                    }
            }
        } else {
            T u[NU][UNIT];
#pragma unroll
            for (int i = 0; i < NU; ++i)
#pragma unroll
                for (int j = 0; j < UNIT; ++j)
                    if (col(i, j) < D) u[i][j] = x[col(i, j)];
            if (a.res) {
                T q[NU][UNIT];
#pragma unroll
                for (int i = 0; i < NU; ++i)
#pragma unroll
                    for (int j = 0; j < UNIT; ++j)
                        if (col(i, j) < D) q[i][j] = res[col(i, j)];
#pragma unroll
                for (int i = 0; i < NU; ++i)
#pragma unroll
                    for (int j = 0; j < UNIT; ++j)
                        if (col(i, j) < D) {
                            u[i][j] = from_f32<T>(to_f32(u[i][j]) + to_f32(q[i][j]));
                            if (a.sum) sum[col(i, j)] = u[i][j];
                        }
            }
#pragma unroll
            for (int i = 0; i < NU; ++i)
#pragma unroll
                for (int j = 0; j < UNIT; ++j)
                    if (col(i, j) < D) h[i][j] = to_f32(u[i][j]);
        }
#pragma unroll
        for (int i = 0; i < NU; ++i)
#pragma unroll
            for (int j = 0; j < UNIT; ++j) {
                if (!(col(i, VEC ? 0 : j) < D)) h[i][j] = 0.f;
                ss = fmaf(h[i][j], h[i][j], ss);
            }
        ss = team_sum<TEAM>(ss, reinterpret_cast<float *>(red));
        float eps = a.eps;
        // Finite rows whose squares leave f32's range: scaled by a power of two first. (The rows of a team of one warp
        // are apart, so the branch is uniform over whoever reduces.)
        if (isinf(ss) || (ss < 0x1p-90f && eps < 0x1p-80f)) {
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < NU; ++i)
#pragma unroll
                for (int j = 0; j < UNIT; ++j) m = max(m, mag(h[i][j]));
            m = team_max<TEAM>(m, red);
            if (m < 0x7f800000u) {
                const float pre = isinf(ss) ? 0x1p-100f : 0x1p100f;
                eps = eps * pre * pre;
                ss = 0.f;
#pragma unroll
                for (int i = 0; i < NU; ++i)
#pragma unroll
                    for (int j = 0; j < UNIT; ++j) {
                        h[i][j] *= pre;
                        ss = fmaf(h[i][j], h[i][j], ss);
                    }
                ss = team_sum<TEAM>(ss, reinterpret_cast<float *>(red));
            }
        }
        const float rstd = 1.f / sqrtf(ss / (float)D + eps);
        Y *y = static_cast<Y *>(a.y) + r * a.ldy;
        // the weights of a unit's columns; 1 where there are none
        const auto weights = [&](int i, float (&g)[UNIT]) {
#pragma unroll
            for (int j = 0; j < UNIT; ++j) g[j] = 1.f;
            if (!a.g) return;
            if constexpr (VEC) {
                if (col(i, 0) < D) load8(a.g + col(i, 0), g);
            } else {
#pragma unroll
                for (int j = 0; j < UNIT; ++j)
                    if (col(i, j) < D) g[j] = a.g[col(i, j)];
            }
        };
        if constexpr (sizeof(Y) > 1) {
#pragma unroll
            for (int i = 0; i < NU; ++i) {
                float g[UNIT];
                weights(i, g);
#pragma unroll
                for (int j = 0; j < UNIT; ++j) g[j] *= h[i][j] * rstd;
                if constexpr (VEC) {
                    if (col(i, 0) < D) store8(y + col(i, 0), g);
                } else {
#pragma unroll
                    for (int j = 0; j < UNIT; ++j)
                        if (col(i, j) < D) y[col(i, j)] = from_f32<Y>(g[j]);
                }
            }
        } else {
            // p = h g, with the error of the product
            float e[NU][UNIT];
#pragma unroll
            for (int i = 0; i < NU; ++i) {
                float g[UNIT];
                weights(i, g);
#pragma unroll
                for (int j = 0; j < UNIT; ++j) {
                    const float p = h[i][j] * g[j];
                    e[i][j] = fmaf(h[i][j], g[j], -p);
                    h[i][j] = p;
                }
            }
            const auto code = [&](int i, int j, const Step &s) {
                return fmaf(h[i][j], s.hi, fmaf(e[i][j], s.hi, h[i][j] * s.lo));
            };
            const int ng = a.group ? (D + a.group - 1) / a.group : 1;
            float *scales = a.scales + r * ng;
            const auto put = [&](int i, const Step (&s)[VEC ? 1 : UNIT]) {
                float q[UNIT];
#pragma unroll
                for (int j = 0; j < UNIT; ++j) q[j] = code(i, j, s[VEC ? 0 : j]);
                if constexpr (VEC) {
                    if (col(i, 0) < D) store8(y + col(i, 0), q);
                } else {
#pragma unroll
                    for (int j = 0; j < UNIT; ++j)
                        if (col(i, j) < D) y[col(i, j)] = to_code<Y>(q[j]);
                }
            };
            uint32_t m[NU];
            if (a.group == 0) {
                m[0] = 0;
#pragma unroll
                for (int i = 0; i < NU; ++i)
#pragma unroll
                    for (int j = 0; j < UNIT; ++j) m[0] = max(m[0], mag(h[i][j]));
                Step s[VEC ? 1 : UNIT];
                s[0] = step_of<Y>(team_max<TEAM>(m[0], red), rstd);
                for (int j = 1; j < (VEC ? 1 : UNIT); ++j) s[j] = s[0];
                if (t == 0) scales[0] = s[0].s;
#pragma unroll
                for (int i = 0; i < NU; ++i) put(i, s);
            } else if constexpr (VEC) {
                // a group is 4, 8 or 16 consecutive lanes
                const int lanes = a.group / UNIT;
#pragma unroll
                for (int i = 0; i < NU; ++i) {
                    m[i] = 0;
#pragma unroll
                    for (int j = 0; j < UNIT; ++j) m[i] = max(m[i], mag(h[i][j]));
                    for (int o = 1; o < lanes; o <<= 1) m[i] = max(m[i], __shfl_xor_sync(~0u, m[i], o));
                    const Step s[1] = {step_of<Y>(m[i], rstd)};
                    if (t % lanes == 0 && col(i, 0) < D) scales[col(i, 0) / a.group] = s[0].s;
                    put(i, s);
                }
            } else if constexpr (TEAM == 32) {
                // a group is 1, 2 or 4 consecutive values j of all lanes
                const int values = a.group / 32;
#pragma unroll
                for (int i = 0; i < NU; ++i) {
                    Step s[UNIT];
                    uint32_t w[UNIT];
#pragma unroll
                    for (int j = 0; j < UNIT; ++j) w[j] = __reduce_max_sync(~0u, mag(h[i][j]));
#pragma unroll
                    for (int j = 0; j < UNIT; ++j) {
                        uint32_t top = max(w[j], values > 1 ? w[j ^ 1] : 0u);
                        if (values > 2) top = max(top, max(w[j ^ 2], w[j ^ 3]));
                        s[j] = step_of<Y>(top, rstd);
                        if (t == 0 && j % values == 0 && col(i, j) < D) scales[col(i, j) / a.group] = s[j].s;
                    }
                    put(i, s);
                }
            } else {
                // a group is one to four neighbouring warps at one value j: joined in shared memory
                __syncthreads();
                for (int k = t; k < ng; k += TEAM) gtop[k] = 0;
                __syncthreads();
#pragma unroll
                for (int i = 0; i < NU; ++i)
#pragma unroll
                    for (int j = 0; j < UNIT; ++j) {
                        const uint32_t w = __reduce_max_sync(~0u, mag(h[i][j]));
                        if (t % 32 == 0 && col(i, j) < D) atomicMax(&gtop[col(i, j) / a.group], w);
                    }
                __syncthreads();
#pragma unroll
                for (int i = 0; i < NU; ++i) {
                    Step s[UNIT];
#pragma unroll
                    for (int j = 0; j < UNIT; ++j) {
                        const int c = min(col(i, j), D - 1);
                        s[j] = step_of<Y>(gtop[c / a.group], rstd);
                        if (col(i, j) < D && c % a.group == 0) scales[c / a.group] = s[j].s;
                    }
                    put(i, s);
                }
            }
        }
    }
}

template <class T, class Y, int TEAM, int NU, bool VEC>
void launch(const RmsArgs &a, cudaStream_t st) {
    constexpr int rows = TEAM == 32 ? 8 : 1, threads = TEAM == 32 ? 256 : TEAM;
    k_rmsnorm<T, Y, TEAM, NU, VEC><<<(unsigned)std::min<int64_t>((a.M + rows - 1) / rows, 1 << 30), threads, 0, st>>>(a);
}

// The team, and the units per thread: loads past the row are skipped, so a few
// sizes serve all widths; teams of one warp, which the narrow rows of long
// streams use, have them all.
template <class T, class Y>
void launch_y(const RmsArgs &a, bool vec, cudaStream_t st) {
    const int units = (a.D + UNIT - 1) / UNIT;
    if (!vec) {
        if (units <= TEAMS[0]) launch<T, Y, TEAMS[0], 1, false>(a, st);
        else if (units <= TEAMS[0] * MAX_UNITS) launch<T, Y, TEAMS[0], MAX_UNITS, false>(a, st);
        else if (units <= TEAMS[1] * MAX_UNITS) launch<T, Y, TEAMS[1], MAX_UNITS, false>(a, st);
        else launch<T, Y, TEAMS[2], MAX_UNITS, false>(a, st);
    } else if (units <= TEAMS[0]) launch<T, Y, TEAMS[0], 1, true>(a, st);
    else if (units <= TEAMS[0] * 2) launch<T, Y, TEAMS[0], 2, true>(a, st);
    else if (units <= TEAMS[0] * 3) launch<T, Y, TEAMS[0], 3, true>(a, st);
    else if (units <= TEAMS[0] * 4) launch<T, Y, TEAMS[0], 4, true>(a, st);
    else if (units <= TEAMS[1] * 2) launch<T, Y, TEAMS[1], 2, true>(a, st);
    else if (units <= TEAMS[1] * 4) launch<T, Y, TEAMS[1], 4, true>(a, st);
    else if (units <= TEAMS[2] * 2) launch<T, Y, TEAMS[2], 2, true>(a, st);
    else launch<T, Y, TEAMS[2], 4, true>(a, st);
}

template <class T>
void launch_t(const RmsArgs &a, int ytype, bool vec, cudaStream_t st) {
    if (ytype == TCB_I8) launch_y<T, int8_t>(a, vec, st);
    else if (ytype == TCB_E4M3) launch_y<T, e4m3>(a, vec, st);
    else launch_y<T, T>(a, vec, st);
}

}  // namespace

void launch_rmsnorm(const RmsArgs &a, int dtype, int ytype, cudaStream_t st) {
    need(dtype == TCB_BF16 || dtype == TCB_F16 || dtype == TCB_F32, "dtype is not TCB_BF16, TCB_F16 or TCB_F32");
    const bool codes = ytype == TCB_I8 || ytype == TCB_E4M3;
    need(codes || ytype == dtype, "ytype is neither dtype, TCB_I8 nor TCB_E4M3");
    need(a.M >= 0 && a.D >= 1 && a.D <= TEAMS[2] * MAX_UNITS * UNIT, "M is negative or D is not in 1..16384");
    need(a.eps >= 0.f && a.eps <= 3.4e38f, "eps is negative or not finite");
    need(codes ? a.group == 0 || a.group == 32 || a.group == 64 || a.group == 128 : a.group == 0,
         codes ? "group is not 0, 32, 64 or 128" : "group without 8-bit output");
    need(a.ldx >= a.D && a.ldy >= a.D && (!a.res || a.ldr >= a.D) && (!a.sum || a.lds >= a.D),
         "a row pitch is smaller than D");
    need(!a.sum || a.res, "sum without res");
    need(codes == (a.scales != nullptr), codes ? "scales is NULL" : "scales without 8-bit output");
    if (a.M == 0) return;
    need(a.x && a.y, "x or y is NULL");
    // every tensor that the call uses in steps of 8 columns and 16 bytes (8 for codes)
    const auto at = [](const void *p, int64_t ld, int bytes) {
        return !p || (reinterpret_cast<uintptr_t>(p) % bytes == 0 && ld % UNIT == 0);
    };
    const bool vec = a.D % UNIT == 0 && at(a.x, a.ldx, 16) && at(a.res, a.ldr, 16) && at(a.sum, a.lds, 16) &&
                     at(a.y, a.ldy, codes ? 8 : 16) && at(a.g, 0, 16);
    if (dtype == TCB_BF16) launch_t<bf16>(a, ytype, vec, st);
    else if (dtype == TCB_F16) launch_t<f16>(a, ytype, vec, st);
    else launch_t<float>(a, ytype, vec, st);
    check_token_launch("k_rmsnorm");
}

}  // namespace tcb
