// Root-mean-square norm of token rows, with the residual's addition in front
// and, on request, 8-bit codes with scales behind. Included by one source file
// per element type.
//
// Bound: HBM. Each element of x (and res) is read once and each of sum and y
// written once; a row stays in registers between the sum of its squares and
// its output, so there is no second read. A row belongs to a team of threads,
// the smallest whose registers hold it: narrow rows share a warp, wide ones take
// several warps.
//
// Codes: with p = h g, v / s = p Q / max|p| whatever the row's norm is. A code is
// p times Q / max|p|, the latter carried to twice f32's precision, so it differs
// from the definition's only where v / s is within a rounding or two of the middle
// between two codes.
#pragma once

#include <algorithm>

#include "token_ops.cuh"

namespace tcb {

constexpr int RMS_UNIT = 8;       // columns per load (16 bytes of a 16-bit type)
constexpr int RMS_MAX_UNITS = 4;  // units per thread
constexpr int RMS_MAX_TEAM = 512;

// 8 columns of a row: packed as they are stored for 16-bit types.
template <class T>
struct Unit {
    uint32_t w[sizeof(T) * 2];

    __device__ __forceinline__ void zero() {
#pragma unroll
        for (uint32_t &v : w) v = 0;
    }
    __device__ __forceinline__ void load(const T *p) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
            const uint4 q = reinterpret_cast<const uint4 *>(p)[i];
            w[4 * i] = q.x, w[4 * i + 1] = q.y, w[4 * i + 2] = q.z, w[4 * i + 3] = q.w;
        }
    }
    __device__ __forceinline__ void store(T *p) const {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i)
            reinterpret_cast<uint4 *>(p)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
    }
    __device__ __forceinline__ void get(float (&v)[8]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (std::is_same_v<T, bf16>) {
                v[2 * i] = bf16lo(w[i]);
                v[2 * i + 1] = bf16hi(w[i]);
            } else if constexpr (std::is_same_v<T, f16>) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
                v[2 * i] = f.x;
                v[2 * i + 1] = f.y;
            } else {
                v[2 * i] = __uint_as_float(w[2 * i]);
                v[2 * i + 1] = __uint_as_float(w[2 * i + 1]);
            }
        }
    }
    __device__ __forceinline__ void set(const float (&v)[8]) {  // rounded to T
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (std::is_same_v<T, bf16>) w[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
            else if constexpr (std::is_same_v<T, f16>) {
                const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
                w[i] = *reinterpret_cast<const uint32_t *>(&h);
            } else {
                w[2 * i] = __float_as_uint(v[2 * i]);
                w[2 * i + 1] = __float_as_uint(v[2 * i + 1]);
            }
        }
    }
    // one element at a time, for rows that no vector fits
    __device__ __forceinline__ void put(int j, T v) {
        if constexpr (sizeof(T) == 4) w[j] = __float_as_uint(v);
        else {
            const uint32_t b = *reinterpret_cast<const uint16_t *>(&v);
            w[j / 2] = j % 2 ? (w[j / 2] & 0xffffu) | b << 16 : (w[j / 2] & 0xffff0000u) | b;
        }
    }
    __device__ __forceinline__ T at(int j) const {
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[j]);
        else {
            const uint16_t b = (uint16_t)(j % 2 ? w[j / 2] >> 16 : w[j / 2]);
            T v;
            memcpy(&v, &b, 2);
            return v;
        }
    }
};

__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// Sum over the team; every thread gets it. `red` is not written again before the next barrier.
template <int TEAM>
__device__ __forceinline__ float team_sum(float v, float *red) {
#pragma unroll
    for (int o = (TEAM < 32 ? TEAM : 32) / 2; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
    if constexpr (TEAM > 32) {
        if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
        __syncthreads();
        v = red[threadIdx.x % (TEAM / 32)];
#pragma unroll
        for (int o = TEAM / 64; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
    }
    return v;
}

// Largest magnitude over `lanes` neighbouring lanes, as bits: magnitudes order like their bits, a NaN above all.
__device__ __forceinline__ uint32_t lanes_max(uint32_t v, int lanes) {
    if (lanes >= 32) return __reduce_max_sync(~0u, v);
    for (int o = 1; o < lanes; o <<= 1) v = max(v, __shfl_xor_sync(~0u, v, o));
    return v;
}
template <int TEAM>
__device__ __forceinline__ uint32_t team_max(uint32_t v, uint32_t *red) {
    v = lanes_max(v, TEAM);
    if constexpr (TEAM > 32) {
        if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
        __syncthreads();
        v = __reduce_max_sync(~0u, red[threadIdx.x % (TEAM / 32)]);
    }
    return v;
}

// What a group's codes are made with: p -> p hi + p lo, and its scale.
struct Step {
    float hi, lo, s;
};
template <class Y>
__device__ __forceinline__ Step step_of(uint32_t top_bits, float rstd) {
    constexpr float Q = code_top<Y>(), R = 1.f / Q;
    const float am = __uint_as_float(top_bits), vm = am * rstd, m = max_nan(vm, 1e-12f);
    Step t;
    t.s = m * R;
    t.s = fmaf(fmaf(-t.s, Q, m), R, t.s);  // m / Q to f32's rounding
    if (vm >= 1e-12f && am < 0x1p100f) {
        float r;
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(am));
        t.hi = Q * r;
        t.lo = fmaf(-t.hi, am, Q) * r;  // what hi lacks of the quotient
    } else {  // all but zero, far out of range, or NaN
        t.hi = rstd / t.s;
        t.lo = vm != vm ? vm : 0.f;
    }
    return t;
}

// 8 codes from p.
template <class Y>
__device__ __forceinline__ uint2 codes8(const float (&p)[8], const Step (&s)[8]) {
    uint32_t w[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        float q[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) q[j] = fmaf(p[4 * h + j], s[4 * h + j].hi, p[4 * h + j] * s[4 * h + j].lo);
        if constexpr (std::is_same_v<Y, int8_t>) {
            // adding 1.5 x 2^23 rounds to a whole number, to even, and leaves it in the low bits
            uint32_t b[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) b[j] = q[j] != q[j] ? 0u : __float_as_uint(q[j] + 12582912.f);
            w[h] = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
        } else {
            const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(q[0], q[1]), __NV_SATFINITE, __NV_E4M3);
            const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(q[2], q[3]), __NV_SATFINITE, __NV_E4M3);
            w[h] = lo | hi << 16;
        }
    }
    return make_uint2(w[0], w[1]);
}

// VEC: unit i of thread t is columns 8 (i TEAM + t) .. + 7, one 16-byte access
// per 16-bit tensor. Otherwise (a pitch, pointer or width that is no multiple of
// 8 elements) value (i, j) is column (8 i + j) TEAM + t, so that the accesses of
// a warp are consecutive.
template <class T, class Y, int TEAM, int NU, bool VEC>
__global__ void __launch_bounds__(TEAM == 512 ? 512 : TEAM == 128 ? 128 : 256) k_rmsnorm(const RmsArgs a) {
    constexpr int ROWS = TEAM <= 32 ? 256 / TEAM : 1;  // rows per block and pass
    constexpr bool CODES = sizeof(Y) == 1;
    __shared__ uint32_t red[3][TEAM > 32 ? TEAM / 32 : 1];
    __shared__ uint32_t gtop[TEAM > 32 && !VEC && CODES ? TEAM * NU * RMS_UNIT / 32 : 1];
    const int t = threadIdx.x % TEAM, D = a.D;
    const auto col = [&](int i, int j) { return VEC ? (i * TEAM + t) * RMS_UNIT + j : (i * RMS_UNIT + j) * TEAM + t; };
    for (int64_t r0 = (int64_t)blockIdx.x * ROWS; r0 < a.M; r0 += (int64_t)gridDim.x * ROWS) {
        if (TEAM > 32 && r0 >= gridDim.x) __syncthreads();  // the shared words of the pass before are free
        const int64_t r = r0 + (TEAM <= 32 ? threadIdx.x / TEAM : 0);
        const int Dr = TEAM <= 32 && r >= a.M ? 0 : D;  // a team behind the last row goes through the motions
        const T *x = static_cast<const T *>(a.x) + r * a.ldx;
        const T *res = static_cast<const T *>(a.res) + r * a.ldr;
        T *sum = static_cast<T *>(a.sum) + r * a.lds;
        Unit<T> h[NU];
#pragma unroll
        for (int i = 0; i < NU; ++i) h[i].zero();
        if constexpr (VEC) {
#pragma unroll
            for (int i = 0; i < NU; ++i)
                if (col(i, 0) < Dr) h[i].load(x + col(i, 0));
            if (a.res) {
                Unit<T> q[NU];
#pragma unroll
                for (int i = 0; i < NU; ++i)
                    if (col(i, 0) < Dr) q[i].load(res + col(i, 0));
#pragma unroll
                for (int i = 0; i < NU; ++i)
                    if (col(i, 0) < Dr) {
                        float u[8], v[8];
                        h[i].get(u);
                        q[i].get(v);
#pragma unroll
                        for (int j = 0; j < 8; ++j) u[j] += v[j];
                        h[i].set(u);
                        if (a.sum) h[i].store(sum + col(i, 0));
                    }
            }
        } else {
#pragma unroll
            for (int i = 0; i < NU; ++i)
#pragma unroll
                for (int j = 0; j < RMS_UNIT; ++j)
                    if (col(i, j) < Dr) h[i].put(j, x[col(i, j)]);
            if (a.res) {
#pragma unroll
                for (int i = 0; i < NU; ++i) {
                    Unit<T> q;
                    q.zero();
#pragma unroll
                    for (int j = 0; j < RMS_UNIT; ++j)
                        if (col(i, j) < Dr) q.put(j, res[col(i, j)]);
                    float u[8], v[8];
                    h[i].get(u);
                    q.get(v);
#pragma unroll
                    for (int j = 0; j < 8; ++j) u[j] += v[j];
                    h[i].set(u);
                    if (a.sum) {
#pragma unroll
                        for (int j = 0; j < RMS_UNIT; ++j)
                            if (col(i, j) < Dr) sum[col(i, j)] = h[i].at(j);
                    }
                }
            }
        }
        const auto squares = [&](float pre) {
            float ss = 0.f;
#pragma unroll
            for (int i = 0; i < NU; ++i) {
                float v[8];
                h[i].get(v);
#pragma unroll
                for (int j = 0; j < 8; ++j) ss = fmaf(v[j] * pre, v[j] * pre, ss);
            }
            return ss;
        };
        float ss = team_sum<TEAM>(squares(1.f), reinterpret_cast<float *>(red[0]));
        // Finite rows whose squares leave f32's range are scaled by a power of two first. Teams that share a warp go
        // together; one that needs nothing multiplies by 1.
        float pre = 1.f, eps = a.eps;
        const bool far = isinf(ss) || (ss < 0x1p-90f && eps < 0x1p-80f);
        if (TEAM < 32 ? __any_sync(~0u, far) : far) {
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < NU; ++i) {
                float v[8];
                h[i].get(v);
#pragma unroll
                for (int j = 0; j < 8; ++j) m = max(m, magnitude(v[j]));
            }
            if (TEAM > 32) __syncthreads();
            m = team_max<TEAM>(m, red[1]);
            if (far && m < 0x7f800000u) pre = isinf(ss) ? 0x1p-100f : 0x1p100f;
            eps = eps * pre * pre;
            if (TEAM > 32) __syncthreads();
            ss = team_sum<TEAM>(squares(pre), reinterpret_cast<float *>(red[0]));
            if (TEAM > 32) __syncthreads();
        }
        const float rstd = 1.f / sqrtf(ss / (float)D + eps);
        Y *y = static_cast<Y *>(a.y) + r * a.ldy;
        // the weights of a unit's columns; 1 where there are none
        const auto weights = [&](int i, float (&g)[8]) {
#pragma unroll
            for (int j = 0; j < 8; ++j) g[j] = 1.f;
            if (!a.g) return;
            if constexpr (VEC) {
                if (col(i, 0) < D) {
                    const float4 u = __ldg(reinterpret_cast<const float4 *>(a.g + col(i, 0)));
                    const float4 v = __ldg(reinterpret_cast<const float4 *>(a.g + col(i, 0)) + 1);
                    g[0] = u.x, g[1] = u.y, g[2] = u.z, g[3] = u.w, g[4] = v.x, g[5] = v.y, g[6] = v.z, g[7] = v.w;
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (col(i, j) < D) g[j] = __ldg(a.g + col(i, j));
            }
        };
        if constexpr (!CODES) {
            const float k = pre * rstd;
#pragma unroll
            for (int i = 0; i < NU; ++i) {
                float g[8], v[8];
                weights(i, g);
                h[i].get(v);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = (pre == 1.f ? v[j] * k : v[j] * pre * rstd) * g[j];
                Unit<T> o;
                o.set(v);
                if constexpr (VEC) {
                    if (col(i, 0) < Dr) o.store(y + col(i, 0));
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (col(i, j) < Dr) y[col(i, j)] = o.at(j);
                }
            }
        } else {
            float p[NU][8];
#pragma unroll
            for (int i = 0; i < NU; ++i) {
                float g[8];
                weights(i, g);
                h[i].get(p[i]);
#pragma unroll
                for (int j = 0; j < 8; ++j) p[i][j] = p[i][j] * pre * g[j];
            }
            const int ng = a.group ? (D + a.group - 1) / a.group : 1;
            float *scales = a.scales + r * ng;
            const auto put = [&](int i, const Step (&s)[8]) {
                const uint2 q = codes8<Y>(p[i], s);
                if constexpr (VEC) {
                    if (col(i, 0) < Dr) *reinterpret_cast<uint2 *>(y + col(i, 0)) = q;
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (col(i, j) < Dr) reinterpret_cast<uint8_t *>(y)[col(i, j)] = (uint8_t)((j < 4 ? q.x : q.y) >> 8 * (j % 4));
                }
            };
            const auto fill = [](Step (&s)[8], const Step &v) {
#pragma unroll
                for (int j = 0; j < 8; ++j) s[j] = v;
            };
            Step s[8];
            if (a.group == 0) {
                uint32_t m = 0;
#pragma unroll
                for (int i = 0; i < NU; ++i)
#pragma unroll
                    for (int j = 0; j < 8; ++j) m = max(m, magnitude(p[i][j]));
                fill(s, step_of<Y>(team_max<TEAM>(m, red[2]), rstd));
                if (t == 0 && Dr) scales[0] = s[0].s;
#pragma unroll
                for (int i = 0; i < NU; ++i) put(i, s);
            } else if constexpr (VEC) {
                // a group is 4, 8 or 16 neighbouring lanes, or the team
                const int lanes = min(a.group / RMS_UNIT, TEAM);
#pragma unroll
                for (int i = 0; i < NU; ++i) {
                    uint32_t m = 0;
#pragma unroll
                    for (int j = 0; j < 8; ++j) m = max(m, magnitude(p[i][j]));
                    fill(s, step_of<Y>(lanes_max(m, lanes), rstd));
                    if (t % lanes == 0 && col(i, 0) < Dr) scales[col(i, 0) / a.group] = s[0].s;
                    put(i, s);
                }
            } else if constexpr (TEAM <= 32) {
                // a group is one or more neighbouring values j of all the team
                const int values = a.group / TEAM;
#pragma unroll
                for (int i = 0; i < NU; ++i) {
                    uint32_t m[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) m[j] = magnitude(p[i][j]);
#pragma unroll
                    for (int o = 1; o < 8; o <<= 1)
                        if (o < values) {
#pragma unroll
                            for (int j = 0; j < 8; ++j)
                                if (!(j & o)) m[j] = m[j | o] = max(m[j], m[j | o]);
                        }
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        if (j % min(values, 8) == 0) {
                            s[j] = step_of<Y>(lanes_max(m[j], TEAM), rstd);
                            if (t == 0 && col(i, j) < Dr) scales[col(i, j) / a.group] = s[j].s;
                        } else s[j] = s[j - 1];
                    }
                    put(i, s);
                }
            } else {
                // a group is one to four neighbouring warps at one value j: joined in shared memory
                for (int k = t; k < ng; k += TEAM) gtop[k] = 0;
                __syncthreads();
#pragma unroll
                for (int i = 0; i < NU; ++i)
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const uint32_t w = __reduce_max_sync(~0u, magnitude(p[i][j]));
                        if (t % 32 == 0 && col(i, j) < D) atomicMax(&gtop[col(i, j) / a.group], w);
                    }
                __syncthreads();
#pragma unroll
                for (int i = 0; i < NU; ++i) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
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
void rms_launch(const RmsArgs &a, cudaStream_t st) {
    constexpr int threads = TEAM <= 32 ? 256 : TEAM, rows = TEAM <= 32 ? 256 / TEAM : 1;
    k_rmsnorm<T, Y, TEAM, NU, VEC><<<(unsigned)std::min<int64_t>((a.M + rows - 1) / rows, 1 << 30), threads, 0, st>>>(a);
}

// The smallest team that holds the row. Loads past the row are skipped, so a few sizes serve all widths.
template <class T, class Y, bool VEC>
void rms_launch_team(const RmsArgs &a, cudaStream_t st) {
    const int units = (a.D + RMS_UNIT - 1) / RMS_UNIT;
    if (units <= 2) rms_launch<T, Y, 2, 1, VEC>(a, st);
    else if (units <= 8) rms_launch<T, Y, 8, 1, VEC>(a, st);
    else if (units <= 32) rms_launch<T, Y, 32, 1, VEC>(a, st);
    else if (units <= 64) rms_launch<T, Y, 32, 2, VEC>(a, st);
    else if (units <= 96) rms_launch<T, Y, 32, 3, VEC>(a, st);
    else if (units <= 128) rms_launch<T, Y, 32, 4, VEC>(a, st);
    else if (units <= 256) rms_launch<T, Y, 128, 2, VEC>(a, st);
    else if (units <= 384) rms_launch<T, Y, 128, 3, VEC>(a, st);
    else if (units <= 512) rms_launch<T, Y, 128, 4, VEC>(a, st);
    else if (units <= 1024) rms_launch<T, Y, 512, 2, VEC>(a, st);
    else rms_launch<T, Y, 512, 4, VEC>(a, st);
}

template <class T>
void rms_launch_type(const RmsArgs &a, int ytype, bool vec, cudaStream_t st) {
    if (ytype == TCB_I8) vec ? rms_launch_team<T, int8_t, true>(a, st) : rms_launch_team<T, int8_t, false>(a, st);
    else if (ytype == TCB_E4M3) vec ? rms_launch_team<T, e4m3, true>(a, st) : rms_launch_team<T, e4m3, false>(a, st);
    else vec ? rms_launch_team<T, T, true>(a, st) : rms_launch_team<T, T, false>(a, st);
}

void rms_launch_bf16(const RmsArgs &a, int ytype, bool vec, cudaStream_t st);
void rms_launch_f16(const RmsArgs &a, int ytype, bool vec, cudaStream_t st);
void rms_launch_f32(const RmsArgs &a, int ytype, bool vec, cudaStream_t st);

}  // namespace tcb
