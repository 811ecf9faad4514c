// Rotary positions on the heads of token rows.
//
// Bound: HBM; every element is read and written once. A thread owns one unit of
// a row, the same columns in every head, so that the cosines and sines of its
// pairs are computed once per row and used by all heads.
//
// Measured: 524,288 rows of 8 heads x 160 in bf16, halves paired, 435 us (6.2 TB/s);
// 131,072 rows of 10 x 128 with 64 turned columns, interleaved, 106 us (6.4 TB/s);
// 141,877 rows of 5 x 224 in f32 193 us (6.6 TB/s). Rows that no vector fits (50,000
// of 10 x 75, 50 turned) go element by element: 55 us (2.7 TB/s).
#include <algorithm>

#include "token_ops.cuh"

namespace tcb {
namespace {

constexpr int ROPE_THREADS = 256;

// Blocks per SM, which bound the registers, and the heads whose loads a thread issues together. Many threads with few loads
// each hide HBM better than the reverse: on 524,288 rows of 8 heads x 160 in bf16, 6 blocks and one head (two vectors) take
// 440 us, 4 and two heads 501, 2 and four heads 538. Narrower vectors take more heads.
template <class T, bool INTER, int V>
struct RopeShape {
    static constexpr bool ONE = INTER && V > 1;  // a unit is one vector
    static constexpr int BYTES = V * sizeof(T);
    static constexpr bool WIDE = sizeof(T) == 4 && BYTES == 16;
    static constexpr int BLOCKS = WIDE ? 5 : 6;
    static constexpr int AHEAD = BYTES == 16 ? (ONE ? 2 : 1) * (WIDE ? 2 : 1) : BYTES == 8 && !ONE ? 2 : 4;
};

// cos and sin (times mscale) of pos * freq. The angle is reduced to a fraction
// of a turn in f64, so a far position keeps its phase; the fraction is then
// within half a turn, where f32 holds it to 2^-26 turns.
__device__ __forceinline__ float2 turn_of(double pos, double freq, float mscale, float sign) {
    const double turns = pos * freq * 0.15915494309189533577;  // 1 / (2 pi)
    float s, c;
    sincospif(2.f * (float)(turns - rint(turns)), &s, &c);
    return make_float2(c * mscale, s * mscale * sign);
}

// V elements at once, up to 16 bytes.
template <class T, int V>
struct Vec {
    T v[V];
};
template <int BYTES>
struct Word {
    using type = std::conditional_t<BYTES == 16, uint4, std::conditional_t<BYTES == 8, uint2, std::conditional_t<BYTES == 4, uint32_t, uint16_t>>>;
};
template <class T, int V>
__device__ __forceinline__ Vec<T, V> load(const T *p) {
    using W = typename Word<V * sizeof(T)>::type;
    const W q = *reinterpret_cast<const W *>(p);
    Vec<T, V> r;
    memcpy(&r, &q, sizeof(W));
    return r;
}
template <class T, int V>
__device__ __forceinline__ void store(T *p, const Vec<T, V> &r) {
    using W = typename Word<V * sizeof(T)>::type;
    W q;
    memcpy(&q, &r, sizeof(W));
    *reinterpret_cast<W *>(p) = q;
}

// Units of a row: first those that turn, then those that are copied (none when
// out is x). A unit is the same one or two vectors of V columns in every head. Half layout: the
// first and the second elements of V pairs, rot/2 apart. Interleaved: one vector
// of V/2 pairs (V = 1: the two elements of a pair). blockIdx.y is a slice of the
// heads.
template <class T, class P, bool INTER, int V>
__global__ void __launch_bounds__(ROPE_THREADS, RopeShape<T, INTER, V>::BLOCKS) k_rope(const RopeArgs a, int units, int rows, int slice) {
    constexpr bool ONE = RopeShape<T, INTER, V>::ONE;
    constexpr int PAIRS = ONE ? V / 2 : V;  // of a unit
    constexpr int AHEAD = RopeShape<T, INTER, V>::AHEAD;
    const int half = a.rot / 2, turning = half / PAIRS;
    const int h0 = blockIdx.y * slice, h1 = min(a.heads, h0 + slice);
    const int rl = units < ROPE_THREADS ? threadIdx.x / units : 0;
    if (rl >= rows) return;
    for (int64_t r = (int64_t)blockIdx.x * rows + rl; r < a.M; r += (int64_t)gridDim.x * rows) {
        for (int u = threadIdx.x - rl * units; u < units; u += ROPE_THREADS) {
            const bool turns = u < turning;
            const int p = !turns ? a.rot + (u - turning) * V : INTER ? 2 * PAIRS * u : V * u;
            const int second = INTER ? 1 : half;  // from a pair's first element to its second
            float2 t[PAIRS];
            const auto angles = [&] {
                const double pos = (double)static_cast<const P *>(a.pos)[r * a.pos_stride];
#pragma unroll
                for (int j = 0; j < PAIRS; ++j) t[j] = turn_of(pos, a.freq[u * PAIRS + j], a.mscale, a.sign);
            };
            // Before the loads for the widest unit, whose registers they would take (524,288 x 8 x 160 in bf16: 440 us, 517 with
            // them behind); while the first heads' loads are on their way for the others (131,072 x 3 x 151: 127 us, was 139).
            constexpr bool BEHIND = ONE || V * sizeof(T) < 16;
            if (!BEHIND && turns) angles();
            const T *x = static_cast<const T *>(a.x) + r * a.ldx + h0 * a.hsx + p;
            T *o = static_cast<T *>(a.out) + r * a.ldo + h0 * a.hso + p;
            for (int h = h0; h < h1; h += AHEAD, x += AHEAD * a.hsx, o += AHEAD * a.hso) {
                Vec<T, V> b[AHEAD], c[AHEAD];
#pragma unroll
                for (int k = 0; k < AHEAD; ++k)
                    if (h + k < h1) {
                        b[k] = load<T, V>(x + k * a.hsx);
                        if (!ONE && turns) c[k] = load<T, V>(x + k * a.hsx + second);
                    }
                if (BEHIND && h == h0 && turns) angles();
#pragma unroll
                for (int k = 0; k < AHEAD; ++k)
                    if (h + k < h1) {
                        if (turns) {
#pragma unroll
                            for (int j = 0; j < PAIRS; ++j) {
                                T &v = ONE ? b[k].v[2 * j % V] : b[k].v[j];
                                T &w = ONE ? b[k].v[(2 * j + 1) % V] : c[k].v[j];
                                const float f = to_f32(v), g = to_f32(w);
                                v = from_f32<T>(f * t[j].x - g * t[j].y);
                                w = from_f32<T>(f * t[j].y + g * t[j].x);
                            }
                            if (!ONE) store<T, V>(o + k * a.hso + second, c[k]);
                        }
                        store<T, V>(o + k * a.hso, b[k]);
                    }
            }
        }
    }
}

template <class T, class P, bool INTER, int V>
void launch(const RopeArgs &a, cudaStream_t st) {
    const int units = a.rot / (INTER && V > 1 ? V : 2 * V) + (a.out == a.x ? 0 : (a.hd - a.rot) / V);
    const int rows = std::max(1, ROPE_THREADS / units);
    const int64_t blocks = (a.M + rows - 1) / rows;
    // With few rows the heads are spread over the grid too, at the price of the angles' being computed again.
    const int64_t spread = std::min<int64_t>(a.heads, std::max<int64_t>(1, 148 / blocks));
    const int slice = (int)((a.heads + spread - 1) / spread);
    const dim3 grid((unsigned)std::min<int64_t>(blocks, 1 << 30), (a.heads + slice - 1) / slice);
    k_rope<T, P, INTER, V><<<grid, ROPE_THREADS, 0, st>>>(a, units, rows, slice);
}

// The widest vectors, of V columns or fewer, that the pairs, the copied columns and every row and head are whole multiples of.
template <class T, class P, int V>
void launch_v(const RopeArgs &a, bool inter, cudaStream_t st) {
    const auto at = [](const void *p, int64_t ld, int64_t hs) { return on(p, V * sizeof(T)) && ld % V == 0 && hs % V == 0; };
    if constexpr (V > 1) {
        if (a.rot % (inter ? V : 2 * V) || (a.hd - a.rot) % V || !at(a.x, a.ldx, a.hsx) || !at(a.out, a.ldo, a.hso))
            return launch_v<T, P, V / 2>(a, inter, st);
    }
    if (inter) launch<T, P, true, V>(a, st);
    else launch<T, P, false, V>(a, st);
}

template <class T>
void launch_p(const RopeArgs &a, int pos_type, bool inter, cudaStream_t st) {
    if (pos_type == TCB_F32) launch_v<T, float, 16 / sizeof(T)>(a, inter, st);
    else if (pos_type == TCB_I32) launch_v<T, int32_t, 16 / sizeof(T)>(a, inter, st);
    else launch_v<T, int64_t, 16 / sizeof(T)>(a, inter, st);
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
    const __int128 row = (__int128)(a.heads - 1) * a.hso + a.hd, plane = a.M > 0 ? (__int128)(a.M - 1) * a.ldo + a.hd : 0;
    need(a.ldx >= 0 && a.ldo >= 0, "a row pitch is negative");
    need(a.M <= 1 || a.ldo >= row || (a.ldo >= a.hd && a.hso >= plane), "rows overlap in out");
    if (a.M == 0) return;
    need(a.x && a.pos && a.freq && a.out, "x, pos, freq or out is NULL");
    need(on(a.x, type_bytes(dtype)) && on(a.out, type_bytes(dtype)) && on(a.pos, type_bytes(pos_type)) && on(a.freq, 8),
         "a pointer is not aligned to its elements");
    need(a.out != a.x || ((a.ldo == a.ldx || a.M == 1) && (a.hso == a.hsx || a.heads == 1)),
         "out is x with other strides");
    if (dtype == TCB_BF16) launch_p<bf16>(a, pos_type, inter, st);
    else if (dtype == TCB_F16) launch_p<f16>(a, pos_type, inter, st);
    else launch_p<float>(a, pos_type, inter, st);
    check_token_launch("k_rope");
}

}  // namespace tcb
