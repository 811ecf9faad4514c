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

// 4 codes from q.
template <class Y>
__device__ __forceinline__ uint32_t codes4(float q0, float q1, float q2, float q3) {
    if constexpr (std::is_same_v<Y, int8_t>) {
        // adding 1.5 x 2^23 rounds to a whole number, to even, and leaves it in the low bits; a NaN gives 0
        const uint32_t b0 = q0 != q0 ? 0u : __float_as_uint(q0 + 12582912.f), b1 = q1 != q1 ? 0u : __float_as_uint(q1 + 12582912.f);
        const uint32_t b2 = q2 != q2 ? 0u : __float_as_uint(q2 + 12582912.f), b3 = q3 != q3 ? 0u : __float_as_uint(q3 + 12582912.f);
        return __byte_perm(__byte_perm(b0, b1, 0x0040), __byte_perm(b2, b3, 0x0040), 0x5410);
    } else {
        const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(q0, q1), __NV_SATFINITE, __NV_E4M3);
        const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(q2, q3), __NV_SATFINITE, __NV_E4M3);
        return __byte_perm(lo, hi, 0x5410);
    }
}
__device__ __forceinline__ float coded(float p, const Step &s) { return fmaf(p, s.hi, p * s.lo); }
template <class Y>
__device__ __forceinline__ uint2 codes8(const float (&p)[8], const Step &s) {
    return make_uint2(codes4<Y>(coded(p[0], s), coded(p[1], s), coded(p[2], s), coded(p[3], s)),
                      codes4<Y>(coded(p[4], s), coded(p[5], s), coded(p[6], s), coded(p[7], s)));
}

// How a row's columns lie on a team's threads. Unit i of thread t is 8 columns from 8 (i TEAM + t) - o on, one 16-byte access
// per 16-bit tensor:
//   ALIGNED  every row of every tensor starts at a 16-byte boundary and is whole units (o = 0);
//   EDGED    the tensors' rows start equally far (o elements) behind such boundaries; the first and the last unit of a row
//            are partly outside it and go element by element;
//   SINGLE   nothing fits: value (i, j) is column (8 i + j) TEAM + t, one element per access, consecutive over a warp.
enum RmsMode { ALIGNED, EDGED, SINGLE };

template <class T, class Y, int TEAM, int NU, RmsMode MODE>
__global__ void __launch_bounds__(TEAM == 512 ? 512 : TEAM == 128 ? 128 : 256) k_rmsnorm(const RmsArgs a) {
    constexpr int ROWS = TEAM <= 32 ? 256 / TEAM : 1;  // rows per block and pass
    constexpr bool CODES = sizeof(Y) == 1;
    __shared__ uint32_t red[3][TEAM > 32 ? TEAM / 32 : 1];
    __shared__ uint32_t gtop[TEAM > 32 && MODE == SINGLE && CODES ? TEAM * NU * RMS_UNIT / 32 : 1];
    const int t = threadIdx.x % TEAM, D = a.D;
    for (int64_t r0 = (int64_t)blockIdx.x * ROWS; r0 < a.M; r0 += (int64_t)gridDim.x * ROWS) {
        if (TEAM > 32 && r0 >= gridDim.x) __syncthreads();  // the shared words of the pass before are free
        const int64_t r = r0 + (TEAM <= 32 ? threadIdx.x / TEAM : 0);
        const int Dr = TEAM <= 32 && r >= a.M ? 0 : D;  // a team behind the last row goes through the motions
        const int o = MODE == EDGED ? (int)((reinterpret_cast<uintptr_t>(a.x) / sizeof(T) + r * a.ldx) % 8) : 0;
        const auto col = [&](int i, int j) {
            return MODE == SINGLE ? (i * RMS_UNIT + j) * TEAM + t : (i * TEAM + t) * RMS_UNIT + j - o;
        };
        const auto whole = [&](int i) { return MODE == ALIGNED ? col(i, 0) < Dr : col(i, 0) >= 0 && col(i, 8) <= Dr; };
        const auto in = [&](int i, int j) { return (MODE != EDGED || col(i, j) >= 0) && col(i, j) < Dr; };
        // unit i of a row that starts at p, zero outside the row; and back
        const auto get = [&](const T *p, int i) {
            Unit<T> u;
            u.zero();
            if (MODE != SINGLE && whole(i)) u.load(p + col(i, 0));
            else if (MODE != ALIGNED && (MODE == SINGLE || (col(i, 8) > 0 && col(i, 0) < Dr))) {
#pragma unroll
                for (int j = 0; j < RMS_UNIT; ++j)
                    if (in(i, j)) u.put(j, p[col(i, j)]);
            }
            return u;
        };
        const auto put = [&](T *p, int i, const Unit<T> &u) {
            if (MODE != SINGLE && whole(i)) u.store(p + col(i, 0));
            else if (MODE != ALIGNED) {
#pragma unroll
                for (int j = 0; j < RMS_UNIT; ++j)
                    if (in(i, j)) p[col(i, j)] = u.at(j);
            }
        };
        Unit<T> h[NU];
        {
            const T *x = static_cast<const T *>(a.x) + r * a.ldx;
#pragma unroll
            for (int i = 0; i < NU; ++i) h[i] = get(x, i);
        }
        if (a.res) {
            const T *res = static_cast<const T *>(a.res) + r * a.ldr;
            T *sum = static_cast<T *>(a.sum) + r * a.lds;
            Unit<T> q[NU];
#pragma unroll
            for (int i = 0; i < NU; ++i) q[i] = get(res, i);
#pragma unroll
            for (int i = 0; i < NU; ++i) {
                float u[8], v[8];
                h[i].get(u);
                q[i].get(v);
#pragma unroll
                for (int j = 0; j < 8; ++j) u[j] += v[j];
                h[i].set(u);
                if (a.sum) put(sum, i, h[i]);
            }
        }
        const auto squares = [&] {
            float ss = 0.f;
#pragma unroll
            for (int i = 0; i < NU; ++i) {
                float v[8];
                h[i].get(v);
#pragma unroll
                for (int j = 0; j < 8; ++j) ss = fmaf(v[j], v[j], ss);
            }
            return ss;
        };
        float ss = team_sum<TEAM>(squares(), reinterpret_cast<float *>(red[0])), eps = a.eps;
        // Finite rows whose squares leave f32's range are scaled by a power of two first, which in bf16 and f32 rounds nothing
        // that counts beside the row's largest value; fp16 rows never leave it. Teams that share a warp go together.
        const bool far = !std::is_same_v<T, f16> && (isinf(ss) || (ss < 0x1p-90f && eps < 0x1p-80f));
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
            if (far && m < 0x7f800000u) {
                const float pre = isinf(ss) ? 0x1p-100f : 0x1p100f;
                eps = eps * pre * pre;
#pragma unroll
                for (int i = 0; i < NU; ++i) {
                    float v[8];
                    h[i].get(v);
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[j] *= pre;
                    h[i].set(v);
                }
            }
            if (TEAM > 32) __syncthreads();
            ss = team_sum<TEAM>(squares(), reinterpret_cast<float *>(red[0]));
            if (TEAM > 32) __syncthreads();
        }
        const float rstd = 1.f / sqrtf(ss / (float)D + eps);
        // v = h g, the weights being 1 where there are none
        const auto weighted = [&](int i, float (&v)[8]) {
            h[i].get(v);
            if (!a.g) return;
            if constexpr (MODE == ALIGNED) {
                if (col(i, 0) < D) {
                    const float4 u = __ldg(reinterpret_cast<const float4 *>(a.g + col(i, 0)));
                    const float4 w = __ldg(reinterpret_cast<const float4 *>(a.g + col(i, 0)) + 1);
                    v[0] *= u.x, v[1] *= u.y, v[2] *= u.z, v[3] *= u.w, v[4] *= w.x, v[5] *= w.y, v[6] *= w.z, v[7] *= w.w;
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (in(i, j)) v[j] *= __ldg(a.g + col(i, j));
            }
        };
        Y *y = static_cast<Y *>(a.y) + r * a.ldy;
        if constexpr (!CODES) {
#pragma unroll
            for (int i = 0; i < NU; ++i) {
                float v[8];
                weighted(i, v);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] *= rstd;
                Unit<T> u;
                u.set(v);
                put(y, i, u);
            }
        } else {
            float p[NU][8];
#pragma unroll
            for (int i = 0; i < NU; ++i) weighted(i, p[i]);
            const int ng = a.group ? (D + a.group - 1) / a.group : 1;
            float *scales = a.scales + r * ng;
            const auto top_of = [&](int i) {
                float m = 0.f;
#pragma unroll
                for (int j = 0; j < 8; ++j) m = max_nan(m, fabsf(p[i][j]));
                return magnitude(m);
            };
            const auto write = [&](int i, uint2 q) {
                if (MODE != SINGLE && whole(i)) *reinterpret_cast<uint2 *>(y + col(i, 0)) = q;
                else if (MODE != ALIGNED) {
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (in(i, j)) reinterpret_cast<uint8_t *>(y)[col(i, j)] = (uint8_t)((j < 4 ? q.x : q.y) >> 8 * (j % 4));
                }
            };
            if (a.group == 0) {
                uint32_t m = 0;
#pragma unroll
                for (int i = 0; i < NU; ++i) m = max(m, top_of(i));
                const Step s = step_of<Y>(team_max<TEAM>(m, red[2]), rstd);
                if (t == 0 && Dr) scales[0] = s.s;
#pragma unroll
                for (int i = 0; i < NU; ++i) write(i, codes8<Y>(p[i], s));
            } else if constexpr (MODE == ALIGNED || (MODE == EDGED && TEAM > 32)) {
                // a group is 4, 8 or 16 neighbouring lanes, or the team (o = 0 here)
                const int lanes = min(a.group / RMS_UNIT, TEAM);
#pragma unroll
                for (int i = 0; i < NU; ++i) {
                    const Step s = step_of<Y>(lanes_max(top_of(i), lanes), rstd);
                    if (t % lanes == 0 && col(i, 0) < Dr) scales[col(i, 0) / a.group] = s.s;
                    write(i, codes8<Y>(p[i], s));
                }
            } else if constexpr (MODE == EDGED) {
                // The same, o columns late: values j >= o of a unit belong to the 8 columns that o = 0 would give this lane,
                // values j < o to the lane in front.
                const int lanes = min(a.group / RMS_UNIT, TEAM);
                uint32_t own[NU], front[NU];
#pragma unroll
                for (int i = 0; i < NU; ++i) {
                    own[i] = front[i] = 0;
#pragma unroll
                    for (int j = 0; j < 8; ++j) (j < o ? front[i] : own[i]) = max(j < o ? front[i] : own[i], magnitude(p[i][j]));
                }
                Step before = {0.f, 0.f, 0.f};  // of the last lane's group, one unit back
#pragma unroll
                for (int i = 0; i < NU; ++i) {
                    uint32_t next = __shfl_down_sync(~0u, front[i], 1, TEAM);
                    if (i + 1 < NU) {
                        const uint32_t wrap = __shfl_sync(~0u, front[(i + 1) % NU], 0, TEAM);
                        if (t == TEAM - 1) next = wrap;
                    } else if (t == TEAM - 1) next = 0;
                    const Step s = step_of<Y>(lanes_max(max(own[i], next), lanes), rstd);
                    const int at = col(i, 0) + o;
                    if (t % lanes == 0 && at < Dr) scales[at / a.group] = s.s;
                    Step f;
                    f.hi = __shfl_up_sync(~0u, s.hi, 1, TEAM);
                    f.lo = __shfl_up_sync(~0u, s.lo, 1, TEAM);
                    if (t == 0) f = before;
                    before.hi = __shfl_sync(~0u, s.hi, TEAM - 1, TEAM);
                    before.lo = __shfl_sync(~0u, s.lo, TEAM - 1, TEAM);
                    float q[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) q[j] = fmaf(p[i][j], j < o ? f.hi : s.hi, p[i][j] * (j < o ? f.lo : s.lo));
                    write(i, make_uint2(codes4<Y>(q[0], q[1], q[2], q[3]), codes4<Y>(q[4], q[5], q[6], q[7])));
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
                    for (int k = 1; k < 8; k <<= 1)
                        if (k < values) {
#pragma unroll
                            for (int j = 0; j < 8; ++j)
                                if (!(j & k)) m[j] = m[j | k] = max(m[j], m[j | k]);
                        }
                    Step s;
                    float q[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        if (j % min(values, 8) == 0) {
                            s = step_of<Y>(lanes_max(m[j], TEAM), rstd);
                            if (t == 0 && col(i, j) < Dr) scales[col(i, j) / a.group] = s.s;
                        }
                        q[j] = coded(p[i][j], s);
                    }
                    write(i, make_uint2(codes4<Y>(q[0], q[1], q[2], q[3]), codes4<Y>(q[4], q[5], q[6], q[7])));
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
                    float q[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const int c = min(col(i, j), D - 1);
                        const Step s = step_of<Y>(gtop[c / a.group], rstd);
                        if (col(i, j) < D && c % a.group == 0) scales[c / a.group] = s.s;
                        q[j] = coded(p[i][j], s);
                    }
                    write(i, make_uint2(codes4<Y>(q[0], q[1], q[2], q[3]), codes4<Y>(q[4], q[5], q[6], q[7])));
                }
            }
        }
    }
}

template <class T, class Y, int TEAM, int NU, RmsMode MODE>
void rms_launch(const RmsArgs &a, cudaStream_t st) {
    constexpr int threads = TEAM <= 32 ? 256 : TEAM, rows = TEAM <= 32 ? 256 / TEAM : 1;
    k_rmsnorm<T, Y, TEAM, NU, MODE><<<(unsigned)std::min<int64_t>((a.M + rows - 1) / rows, 1 << 30), threads, 0, st>>>(a);
}

// The smallest team that holds the row (and up to 7 columns in front of it). Loads outside the row are skipped, so a few
// sizes serve all widths.
template <class T, class Y, RmsMode MODE>
void rms_launch_team(const RmsArgs &a, cudaStream_t st) {
    const int units = (a.D + RMS_UNIT - 1 + (MODE == EDGED ? 7 : 0)) / RMS_UNIT;
    if (units <= 2) return rms_launch<T, Y, 2, 1, MODE>(a, st);
    if (units <= 8) return rms_launch<T, Y, 8, 1, MODE>(a, st);
    if (units <= 32) return rms_launch<T, Y, 32, 1, MODE>(a, st);
    if constexpr (MODE != SINGLE) {
        if (units <= 64) return rms_launch<T, Y, 32, 2, MODE>(a, st);
        if (units <= 96) return rms_launch<T, Y, 32, 3, MODE>(a, st);
    }
    if (units <= 128) return rms_launch<T, Y, 32, 4, MODE>(a, st);
    if constexpr (MODE != SINGLE) {
        if (units <= 256) return rms_launch<T, Y, 128, 2, MODE>(a, st);
        if (units <= 384) return rms_launch<T, Y, 128, 3, MODE>(a, st);
    }
    if (units <= 512) return rms_launch<T, Y, 128, 4, MODE>(a, st);
    if constexpr (MODE != SINGLE) {
        if (units <= 1024) return rms_launch<T, Y, 512, 2, MODE>(a, st);
    }
    if (units <= 2048) return rms_launch<T, Y, 512, 4, MODE>(a, st);
    // EDGED, 16,378 columns or more
    rms_launch<T, Y, 512, 4, SINGLE>(a, st);
}

template <class T>
void rms_launch_type(const RmsArgs &a, int ytype, RmsMode mode, cudaStream_t st) {
    const auto by_mode = [&](auto y) {
        using Y = decltype(y);
        if (mode == ALIGNED) rms_launch_team<T, Y, ALIGNED>(a, st);
        else if (mode == EDGED) rms_launch_team<T, Y, EDGED>(a, st);
        else rms_launch_team<T, Y, SINGLE>(a, st);
    };
    if (ytype == TCB_I8) by_mode(int8_t());
    else if (ytype == TCB_E4M3) by_mode(e4m3());
    else by_mode(T());
}

void rms_launch_bf16(const RmsArgs &a, int ytype, RmsMode mode, cudaStream_t st);
void rms_launch_f16(const RmsArgs &a, int ytype, RmsMode mode, cudaStream_t st);
void rms_launch_f32(const RmsArgs &a, int ytype, RmsMode mode, cudaStream_t st);

}  // namespace tcb
