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
// Codes: with p = h g, v / s = p Q / max|p| whatever the row's norm is, so a code
// comes from four roundings and differs from the definition's only where v / s is
// that near the middle between two codes (28 to 44 of 84 million e4m3 codes on eight
// inputs; f32 arithmetic in the definition's order: 33 to 66, more on each).
//
// Measured, bf16 rows: 524,288 x 640 with the residual to e4m3 with scales of 128
// columns in 342 us (6.9 TB/s), to bf16 in 390 us (6.9 TB/s); 32,768 x 2,560 to e4m3
// in 51 us (4.9 TB/s); 8,192 x 16,384 with the residual to int8 in 146 us (6.4 TB/s);
// fp16 rows of 1,337 at a pitch of 1,341 to int8, 10,007 of them, in 34 us (2.8 TB/s,
// bound by instructions: weights and edges come one by one).
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
    __device__ __forceinline__ void add(const Unit &b) {  // rounded to T once
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) * 2; ++i) {
            if constexpr (std::is_same_v<T, bf16>) {
                const __nv_bfloat162 v = __hadd2(*reinterpret_cast<const __nv_bfloat162 *>(&w[i]), *reinterpret_cast<const __nv_bfloat162 *>(&b.w[i]));
                w[i] = *reinterpret_cast<const uint32_t *>(&v);
            } else if constexpr (std::is_same_v<T, f16>) {
                const __half2 v = __hadd2(*reinterpret_cast<const __half2 *>(&w[i]), *reinterpret_cast<const __half2 *>(&b.w[i]));
                w[i] = *reinterpret_cast<const uint32_t *>(&v);
            } else w[i] = __float_as_uint(__uint_as_float(w[i]) + __uint_as_float(b.w[i]));
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

// Largest magnitude over `lanes` (2 to 32) neighbouring lanes, NaN if any is; of magnitudes, which order like their bits.
__device__ __forceinline__ float lanes_max(float v, int lanes) {
    uint32_t b = __float_as_uint(v);
    if (lanes >= 32) return __uint_as_float(__reduce_max_sync(~0u, b));
    b = max(b, __shfl_xor_sync(~0u, b, 1));
    if (lanes > 2) b = max(b, __shfl_xor_sync(~0u, b, 2));
    if (lanes > 4) b = max(b, __shfl_xor_sync(~0u, b, 4));
    if (lanes > 8) b = max(b, __shfl_xor_sync(~0u, b, 8));
    return __uint_as_float(b);
}
template <int TEAM>
__device__ __forceinline__ float team_max(float v, float *red) {
    v = lanes_max(v, TEAM);
    if constexpr (TEAM > 32) {
        if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
        __syncthreads();
        v = lanes_max(red[threadIdx.x % (TEAM / 32)], 32);
    }
    return v;
}

__device__ __forceinline__ float rcp_approx(float v) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}

// What a group's codes are made with: p -> p k, and its scale. k = Q / max|p|, with the error of the approximate reciprocal
// taken out by one Newton step.
struct Step {
    float k, s;
};
template <class Y>
__device__ __forceinline__ Step step_of(float top, float rstd) {
    constexpr float Q = code_top<Y>(), R = 1.f / Q;
    const float v = top * rstd, m = max_nan(v, 1e-12f);
    Step t;
    t.s = m * R;
    t.s = fmaf(fmaf(-t.s, Q, m), R, t.s);  // m / Q to f32's rounding
    const float r = rcp_approx(top);
    t.k = Q * r;
    t.k = fmaf(fmaf(-t.k, top, Q), r, t.k);
    if (!(v >= 1e-12f) || top > 0x1p100f) t.k = rstd / t.s;  // all but zero, NaN, or far out of range
    return t;
}

// 4 codes of p.
template <class Y>
__device__ __forceinline__ uint32_t codes4(float p0, float p1, float p2, float p3, const Step &s) {
    const float q0 = p0 * s.k, q1 = p1 * s.k, q2 = p2 * s.k, q3 = p3 * s.k;
    if constexpr (std::is_same_v<Y, int8_t>) {
        // adding 1.5 x 2^23 rounds to a whole number, to even, and leaves it in the low bits; a group with a NaN gives 0
        const uint32_t b0 = __float_as_uint(q0 + 12582912.f), b1 = __float_as_uint(q1 + 12582912.f);
        const uint32_t b2 = __float_as_uint(q2 + 12582912.f), b3 = __float_as_uint(q3 + 12582912.f);
        const uint32_t w = __byte_perm(__byte_perm(b0, b1, 0x0040), __byte_perm(b2, b3, 0x0040), 0x5410);
        return s.s != s.s ? 0u : w;
    } else {
        const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(q0, q1), __NV_SATFINITE, __NV_E4M3);
        const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(q2, q3), __NV_SATFINITE, __NV_E4M3);
        return __byte_perm(lo, hi, 0x5410);
    }
}
template <class Y>
__device__ __forceinline__ uint2 codes8(const float (&p)[8], const Step &s) {
    return make_uint2(codes4<Y>(p[0], p[1], p[2], p[3], s), codes4<Y>(p[4], p[5], p[6], p[7], s));
}

// How a row's columns lie on a team's threads. Unit i of thread t is 8 columns from 8 (i TEAM + t) - o on, one 16-byte access
// per 16-bit tensor:
//   ALIGNED  every row of every tensor starts at a 16-byte boundary and is whole units (o = 0);
//   EDGED    the tensors' rows start equally far (o elements) behind such boundaries; the first and the last unit of a row
//            are partly outside it and go element by element;
//   SINGLE   nothing fits: value (i, j) is column (8 i + j) TEAM + t, one element per access, consecutive over a warp.
//
// ALIGNED_ROW is ALIGNED for codes with one scale per row: a kernel of its own, since the two kinds of scales together take
// registers that rows of 2,560 columns and more miss (16,384: 151 us instead of 142).
enum RmsMode { ALIGNED, EDGED, SINGLE, ALIGNED_ROW };

// Threads of a block, and the registers of a thread, which bound the blocks on an SM: about what the packed row, and for
// EDGED rows the row in f32, needs. Fewer spill, more leave HBM waiting (bf16 to e4m3, 524,288 x 640: 48 registers 396 us, 64
// 422, 40 456; 32,768 x 2,560 with 64 threads a row: 80 registers 50 us, 96 54, 112 56). Set on bf16 rows: f32 rows of six units
// a thread, whose 9 blocks of two warps are five warps in a quarter of an SM, get 96 registers and spill.
template <class T, int TEAM, int NU, RmsMode MODE>
struct RmsShape {
    static constexpr int THREADS = TEAM <= 32 ? 128 : TEAM;
    static constexpr int PACKED = NU <= 2 ? 40 : NU == 3 ? (TEAM == 32 ? 48 : 56) : NU == 4 ? 64 : NU == 5 ? 80 : 96;
    static constexpr int REGS = MODE == EDGED ? (24 + 16 * NU) * (sizeof(T) == 4 ? 5 : 4) / 4
                                : sizeof(T) == 4 && NU > 1 ? PACKED + 16 : PACKED;
    static constexpr int BLOCKS = 65536 / (THREADS * REGS);
};

template <class T, class Y, int TEAM, int NU, RmsMode MODE>
__global__ void __launch_bounds__(RmsShape<T, TEAM, NU, MODE>::THREADS, RmsShape<T, TEAM, NU, MODE>::BLOCKS) k_rmsnorm(const RmsArgs a) {
    constexpr int THREADS = RmsShape<T, TEAM, NU, MODE>::THREADS, ROWS = THREADS / TEAM;  // rows per block and pass
    constexpr bool CODES = sizeof(Y) == 1, BOUND = MODE == ALIGNED || MODE == ALIGNED_ROW;
    // units that the choice of the team leaves whole in aligned rows (a team of 512 with 4 units starts at 8,200 columns)
    constexpr int FULL = !BOUND || TEAM < 32 ? 0 : TEAM == 512 ? NU / 2 : NU - 1;
    __shared__ float red[3][TEAM > 32 ? TEAM / 32 : 1];
    __shared__ uint32_t gtop[TEAM > 32 && MODE == SINGLE && CODES ? TEAM * NU * RMS_UNIT / 32 : 1];
    const int t = threadIdx.x % TEAM;
    for (int64_t r0 = (int64_t)blockIdx.x * ROWS; r0 < a.M; r0 += (int64_t)gridDim.x * ROWS) {
        if (TEAM > 32 && r0 >= gridDim.x) __syncthreads();  // the shared words of the pass before are free
        const int64_t r = r0 + threadIdx.x / TEAM;
        if (TEAM == 32 && r >= a.M) break;
        const int D = TEAM < 32 && r >= a.M ? 0 : a.D;  // a team behind the last row that shares a warp goes through the motions
        const int o = MODE == EDGED ? (int)((reinterpret_cast<uintptr_t>(a.x) / sizeof(T) + r * a.ldx) % 8) : 0;
        const auto col = [&](int i, int j) {
            return MODE == SINGLE ? (i * RMS_UNIT + j) * TEAM + t : (i * TEAM + t) * RMS_UNIT + j - o;
        };
        const auto whole = [&](int i) {
            return BOUND ? i < FULL || col(i, 0) < D : MODE == EDGED && col(i, 0) >= 0 && col(i, 8) <= D;
        };
        const auto in = [&](int i, int j) { return (MODE != EDGED || col(i, j) >= 0) && col(i, j) < D; };
        // unit i of a row that starts at p, zero outside the row; and back
        const auto get = [&](const T *p, int i) {
            Unit<T> u;
            if (!(BOUND && i < FULL)) u.zero();
            if (whole(i)) u.load(p + col(i, 0));
            else if (MODE == SINGLE || (MODE == EDGED && col(i, 8) > 0 && col(i, 0) < D)) {
#pragma unroll
                for (int j = 0; j < RMS_UNIT; ++j)
                    if (in(i, j)) u.put(j, p[col(i, j)]);
            }
            return u;
        };
        const auto put = [&](T *p, int i, const Unit<T> &u) {
            if (whole(i)) u.store(p + col(i, 0));
            else if (MODE == SINGLE || (MODE == EDGED && col(i, 8) > 0 && col(i, 0) < D)) {
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
            Unit<T> q[NU];
#pragma unroll
            for (int i = 0; i < NU; ++i) q[i] = get(res, i);
            T *sum = static_cast<T *>(a.sum) + r * a.lds;
#pragma unroll
            for (int i = 0; i < NU; ++i) {
                h[i].add(q[i]);
                if (a.sum) put(sum, i, h[i]);
            }
        }
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < NU; ++i) {
            float v[8];
            h[i].get(v);
#pragma unroll
            for (int j = 0; j < 8; ++j) ss = fmaf(v[j], v[j], ss);
        }
        // p = h g, the weights being 1 where there are none. Made when it is needed, so that a row waits packed for its sum;
        // EDGED rows, whose weights come one by one, make it once.
        const auto weigh = [&](int i, float (&p)[8]) {
            h[i].get(p);
            if (!a.g) return;
            if (BOUND) {
                if (whole(i)) {
                    const float4 u = __ldg(reinterpret_cast<const float4 *>(a.g + col(i, 0)));
                    const float4 w = __ldg(reinterpret_cast<const float4 *>(a.g + col(i, 0)) + 1);
                    p[0] *= u.x, p[1] *= u.y, p[2] *= u.z, p[3] *= u.w, p[4] *= w.x, p[5] *= w.y, p[6] *= w.z, p[7] *= w.w;
                }
            } else if (whole(i)) {
#pragma unroll
                for (int j = 0; j < 8; ++j) p[j] *= __ldg(a.g + col(i, 0) + j);
            } else if (MODE == SINGLE || (col(i, 8) > 0 && col(i, 0) < D)) {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (in(i, j)) p[j] *= __ldg(a.g + col(i, j));
            }
        };
        constexpr bool KEEP = MODE == EDGED;
        float kept[KEEP ? NU : 1][8];
        if constexpr (KEEP) {
#pragma unroll
            for (int i = 0; i < NU; ++i) weigh(i, kept[i]);
        }
        const auto weighted = [&](int i, float (&p)[8]) {
            if constexpr (KEEP) {
#pragma unroll
                for (int j = 0; j < 8; ++j) p[j] = kept[i][j];
            } else weigh(i, p);
        };
        ss = team_sum<TEAM>(ss, red[0]);
        float eps = a.eps;
        // Finite rows whose squares leave f32's range (or do with eps) are scaled by a power of two first; fp16 rows never leave it. Large rows
        // come down until their largest value is 2^55 to 2^56, 16,384 squares of which f32 holds, and no further: what goes
        // below f32's and bf16's normal values there would do so in the output. Teams that share a warp go together.
        const bool over = isinf(fmaf(ss, a.inv_d, eps));
        const bool far = !std::is_same_v<T, f16> && (over || (ss < 0x1p-90f && eps < 0x1p-80f));
        if (TEAM < 32 ? __any_sync(~0u, far) : far) {
            float m = 0.f;
#pragma unroll
            for (int i = 0; i < NU; ++i) {
                float v[8];
                h[i].get(v);
#pragma unroll
                for (int j = 0; j < 8; ++j) m = max_nan(m, fabsf(v[j]));
            }
            if (TEAM > 32) __syncthreads();
            m = team_max<TEAM>(m, red[1]);
            const float down = __uint_as_float(min(309u - (__float_as_uint(m) >> 23), 119u) << 23);  // 2^(55 - m's exponent), at most 2^-8
            const float pre = !far || !(m <= 3.4028235e38f) ? 1.f : over ? down : 0x1p100f;
            eps = eps * pre * pre;
            ss = 0.f;
#pragma unroll
            for (int i = 0; i < NU; ++i) {
                float v[8];
                h[i].get(v);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    v[j] *= pre;
                    ss = fmaf(v[j], v[j], ss);
                }
                h[i].set(v);
                if constexpr (KEEP) weigh(i, kept[i]);
            }
            if (TEAM > 32) __syncthreads();
            ss = team_sum<TEAM>(ss, red[0]);
            if (TEAM > 32) __syncthreads();
        }
        const float rstd = rsqrtf(fmaf(ss, a.inv_d, eps));
        Y *y = static_cast<Y *>(a.y) + r * a.ldy;
        if constexpr (!CODES) {
#pragma unroll
            for (int i = 0; i < NU; ++i) {
                float p[8];
                weighted(i, p);
#pragma unroll
                for (int j = 0; j < 8; ++j) p[j] *= rstd;
                Unit<T> u;
                u.set(p);
                put(y, i, u);
            }
        } else {
            const int ng = a.group ? (a.D + a.group - 1) >> a.shift : 1;
            float *scales = a.scales + r * ng;
            const auto top_of = [](const float (&p)[8]) {
                float m = 0.f;
#pragma unroll
                for (int j = 0; j < 8; ++j) m = max_nan(m, fabsf(p[j]));
                return m;
            };
            const auto write = [&](int i, uint2 q) {
                if (whole(i)) *reinterpret_cast<uint2 *>(y + col(i, 0)) = q;
                else if (MODE == SINGLE || (MODE == EDGED && col(i, 8) > 0 && col(i, 0) < D)) {
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (in(i, j)) reinterpret_cast<uint8_t *>(y)[col(i, j)] = (uint8_t)((j < 4 ? q.x : q.y) >> 8 * (j % 4));
                }
            };
            if (MODE == ALIGNED_ROW || (MODE != ALIGNED && a.group == 0)) {
                float m = 0.f, p[NU][8];
#pragma unroll
                for (int i = 0; i < NU; ++i) {
                    weighted(i, p[i]);
                    m = max_nan(m, top_of(p[i]));
                }
                const Step s = step_of<Y>(team_max<TEAM>(m, red[2]), rstd);
                if (t == 0 && D) scales[0] = s.s;
#pragma unroll
                for (int i = 0; i < NU; ++i) write(i, codes8<Y>(p[i], s));
            } else if constexpr (BOUND || (MODE == EDGED && TEAM > 32)) {
                // a group is 4, 8 or 16 neighbouring lanes, or the team (o = 0 here)
                const int lanes = min(a.group / RMS_UNIT, TEAM);
#pragma unroll
                for (int i = 0; i < NU; ++i) {
                    float p[8];
                    weighted(i, p);
                    const Step s = step_of<Y>(lanes_max(top_of(p), lanes), rstd);
                    if ((t & (lanes - 1)) == 0 && col(i, 0) < D) scales[col(i, 0) >> a.shift] = s.s;
                    write(i, codes8<Y>(p, s));
                }
            } else if constexpr (MODE == EDGED) {
                // The same, o columns late: values j >= o of a unit belong to the 8 columns that o = 0 would give this lane,
                // values j < o to the lane in front.
                const int lanes = min(a.group / RMS_UNIT, TEAM);
                float p[NU][8], own[NU], front[NU];
#pragma unroll
                for (int i = 0; i < NU; ++i) weighted(i, p[i]);
#pragma unroll
                for (int i = 0; i < NU; ++i) {
                    own[i] = front[i] = 0.f;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        own[i] = max_nan(own[i], j < o ? 0.f : fabsf(p[i][j]));
                        front[i] = max_nan(front[i], j < o ? fabsf(p[i][j]) : 0.f);
                    }
                }
                Step before = {0.f, 0.f};  // of the last lane's group, one unit back
#pragma unroll
                for (int i = 0; i < NU; ++i) {
                    float next = __shfl_down_sync(~0u, front[i], 1, TEAM);
                    if (i + 1 < NU) {
                        const float wrap = __shfl_sync(~0u, front[(i + 1) % NU], 0, TEAM);
                        if (t == TEAM - 1) next = wrap;
                    } else if (t == TEAM - 1) next = 0.f;
                    const Step s = step_of<Y>(lanes_max(max_nan(own[i], next), lanes), rstd);
                    const int at = col(i, 0) + o;
                    if ((t & (lanes - 1)) == 0 && at < D) scales[at >> a.shift] = s.s;
                    Step f = {__shfl_up_sync(~0u, s.k, 1, TEAM), __shfl_up_sync(~0u, s.s, 1, TEAM)};
                    if (t == 0) f = before;
                    before = {__shfl_sync(~0u, s.k, TEAM - 1, TEAM), __shfl_sync(~0u, s.s, TEAM - 1, TEAM)};
                    const uint2 u = codes8<Y>(p[i], s), v = codes8<Y>(p[i], f);
                    // the first o codes by f
                    const uint64_t mask = o ? ~0ull >> (64 - 8 * o) : 0ull;
                    const uint64_t w = ((uint64_t)v.y << 32 | v.x) & mask | ((uint64_t)u.y << 32 | u.x) & ~mask;
                    write(i, make_uint2((uint32_t)w, (uint32_t)(w >> 32)));
                }
            } else if constexpr (TEAM <= 32) {
                // a group is one or more neighbouring values j of all the team
                const int values = a.group / TEAM;
#pragma unroll
                for (int i = 0; i < NU; ++i) {
                    float p[8], m[8];
                    weighted(i, p);
#pragma unroll
                    for (int j = 0; j < 8; ++j) m[j] = fabsf(p[j]);
#pragma unroll
                    for (int k = 1; k < 8; k <<= 1)
                        if (k < values) {
#pragma unroll
                            for (int j = 0; j < 8; ++j)
                                if (!(j & k)) m[j] = m[j | k] = max_nan(m[j], m[j | k]);
                        }
                    Step s;
                    uint32_t w[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        if ((j & (min(values, 8) - 1)) == 0) {
                            s = step_of<Y>(lanes_max(m[j], TEAM), rstd);
                            if (t == 0 && col(i, j) < D) scales[col(i, j) >> a.shift] = s.s;
                        }
                        w[j] = codes4<Y>(p[j], 0.f, 0.f, 0.f, s) & 0xff;
                    }
                    write(i, make_uint2(w[0] | w[1] << 8 | w[2] << 16 | w[3] << 24, w[4] | w[5] << 8 | w[6] << 16 | w[7] << 24));
                }
            } else {
                // a group is one to four neighbouring warps at one value j: joined in shared memory
                for (int k = t; k < ng; k += TEAM) gtop[k] = 0;
                __syncthreads();
#pragma unroll
                for (int i = 0; i < NU; ++i) {
                    float p[8];
                    weighted(i, p);
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const uint32_t w = __reduce_max_sync(~0u, magnitude(p[j]));
                        if (t % 32 == 0 && col(i, j) < D) atomicMax(&gtop[col(i, j) >> a.shift], w);
                    }
                }
                __syncthreads();
#pragma unroll
                for (int i = 0; i < NU; ++i) {
                    float p[8];
                    weighted(i, p);
                    uint32_t w[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const int c = min(col(i, j), D - 1);
                        const Step s = step_of<Y>(__uint_as_float(gtop[c >> a.shift]), rstd);
                        if (col(i, j) < D && (c & (a.group - 1)) == 0) scales[c >> a.shift] = s.s;
                        w[j] = codes4<Y>(p[j], 0.f, 0.f, 0.f, s) & 0xff;
                    }
                    write(i, make_uint2(w[0] | w[1] << 8 | w[2] << 16 | w[3] << 24, w[4] | w[5] << 8 | w[6] << 16 | w[7] << 24));
                }
            }
        }
    }
}

template <class T, class Y, int TEAM, int NU, RmsMode MODE>
void rms_launch(const RmsArgs &a, cudaStream_t st) {
    constexpr int threads = RmsShape<T, TEAM, NU, MODE>::THREADS, rows = threads / TEAM;
    k_rmsnorm<T, Y, TEAM, NU, MODE><<<(unsigned)std::min<int64_t>((a.M + rows - 1) / rows, 1 << 30), threads, 0, st>>>(a);
}

// The team whose registers hold the row (and up to 7 columns in front of it) with the least to spare, as far as a few sizes
// serve all widths; loads outside the row are skipped. Two rows of 80 units a warp take 343 us on 524,288 x 640 (bf16 to
// e4m3), a row a warp, with a sixth of it idle, 363; on a single row 2.9 and 2.2. The number of rows has no say, so that a
// row's bits are the same in any batch.
template <class T, class Y, RmsMode MODE>
void rms_launch_team(const RmsArgs &a, cudaStream_t st) {
    const int units = (a.D + RMS_UNIT - 1 + (MODE == EDGED ? 7 : 0)) / RMS_UNIT;
    if (units <= 2) return rms_launch<T, Y, 2, 1, MODE>(a, st);
    if (units <= 8) return rms_launch<T, Y, 8, 1, MODE>(a, st);
    if (units <= 32) return rms_launch<T, Y, 32, 1, MODE>(a, st);
    if constexpr (MODE != SINGLE) {
        if (units <= 64) return rms_launch<T, Y, 32, 2, MODE>(a, st);
        if ((MODE == ALIGNED || MODE == ALIGNED_ROW) && units <= 80) return rms_launch<T, Y, 16, 5, MODE>(a, st);
        if (units <= 96) return rms_launch<T, Y, 32, 3, MODE>(a, st);
    }
    if (units <= 128) return rms_launch<T, Y, 32, 4, MODE>(a, st);
    if constexpr (MODE != SINGLE) {
        if (units <= 192) return rms_launch<T, Y, 64, 3, MODE>(a, st);
        if (units <= 256) return rms_launch<T, Y, 64, 4, MODE>(a, st);
        if (units <= 320) return rms_launch<T, Y, 64, 5, MODE>(a, st);
        if (units <= 384) return rms_launch<T, Y, 64, 6, MODE>(a, st);
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
        if (mode == ALIGNED) {
            if constexpr (sizeof(Y) == 1) {
                if (a.group == 0) return rms_launch_team<T, Y, ALIGNED_ROW>(a, st);
            }
            rms_launch_team<T, Y, ALIGNED>(a, st);
        }
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
