// Rotary positions on the heads of token rows.
//
// Bound: HBM; every element is read and written once. A thread owns one unit of
// a row, the same columns in every head, so that the cosines and sines of its
// pairs are computed once per row and used by all heads.
//
// Measured: 524,288 rows of 8 heads x 160 in bf16, halves paired, 435 us (6.2 TB/s);
// 131,072 rows of 10 x 128 with 64 turned columns, interleaved, 106 us (6.4 TB/s);
// 141,877 rows of 5 x 224 in f32 193 us (6.6 TB/s); heads that no vector fits,
// 131,072 rows of 8 x 151 in bf16 with 90 turned, 125 us (5.1 TB/s).
#include <algorithm>
#include <atomic>

#include "token_ops.cuh"

namespace tcb {
namespace {

constexpr int ROPE_THREADS = 256;
constexpr int ROPE_SMEM = 96 * 1024, ROPE_SM_SMEM = 227 * 1024;  // of a block that holds rows, and of an SM

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

// cos and sin (times mscale) of pos * freq, for heads of type T. The angle is reduced to a fraction of a turn in f64, so a far
// position keeps its phase; the fraction is then within half a turn, where f32 holds it to 2^-26 turns. For f32 heads, which
// would show that, what it leaves turns the cosine and the sine once more (f32 results: 3.4e-8 of the pair's size off in the
// root mean square without, 2.5e-8 with, 2.3e-8 with both rounded once from f64).
template <class T>
__device__ __forceinline__ float2 turn_of(double pos, double freq, float mscale, float sign) {
    double turns = pos * freq * 0.15915494309189533577;  // 1 / (2 pi)
    turns -= rint(turns);
    const float near = (float)turns;
    float s, c;
    sincospif(2.f * near, &s, &c);
    if constexpr (sizeof(T) == 4) {
        const float left = (float)((turns - near) * 6.283185307179586477), c0 = c;
        c = fmaf(-s, left, c);
        s = fmaf(c0, left, s);
    }
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
                for (int j = 0; j < PAIRS; ++j) t[j] = turn_of<T>(pos, a.freq[u * PAIRS + j], a.mscale, a.sign);
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

// Rows that take vectors of 4 bytes or less, in packed heads: a warp brings a whole row to shared memory in 16-byte copies,
// the next one while it works, turns the pairs there element by element, and writes the row back in 16-byte stores. x and out
// rows start equally far behind 16-byte boundaries; a row's first and last bytes go alone where the 16 are not all its own.
template <class T, class P, bool INTER>
__global__ void __launch_bounds__(ROPE_THREADS) k_rope_rows(const RopeArgs a, const int bytes) {
    extern __shared__ __align__(16) uint8_t tiles[];
    const int lane = threadIdx.x & 31, half = a.rot / 2, pieces = bytes / 16 + 2, pitch = pieces * 16;
    uint8_t *mine = tiles + (threadIdx.x >> 5) * 2 * pitch;
    const int64_t stride = (int64_t)gridDim.x * (blockDim.x >> 5);
    const uint8_t *const first = static_cast<const uint8_t *>(a.x);
    const uint8_t *const end = first + (a.M - 1) * a.ldx * (int64_t)sizeof(T) + bytes;  // of x's last row
    const auto fetch = [&](int64_t r, int slot) {
        if (r < a.M) {
            const uint8_t *row = first + r * a.ldx * (int64_t)sizeof(T);
            const int off = (int)(reinterpret_cast<uintptr_t>(row) % 16);
            uint8_t *to = mine + slot * pitch;
            for (int q = lane; q < pieces; q += 32) {
                const uint8_t *p = row - off + q * 16;
                if (p >= first && p + 16 <= end) {  // may hold bytes between rows too
                    if (q * 16 - off < bytes) cp_async16(smem_u32(to + q * 16), p);
                } else {
                    for (int j = 0; j < 16; j += (int)sizeof(T))
                        if (p + j >= row && p + j < row + bytes)
                            *reinterpret_cast<T *>(to + q * 16 + j) = *reinterpret_cast<const T *>(p + j);
                }
            }
        }
        cp_async_commit();
    };
    // with fewer pairs than lanes, the heads are dealt out to several lanes of a pair
    const int slices = half < 32 ? 32 / half : 1, slice = half < 32 ? lane / half : 0, own = half < 32 ? lane % half : lane;
    int64_t r = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    int slot = 0;
    fetch(r, 0);
    for (; r < a.M; r += stride, slot ^= 1) {
        fetch(r + stride, slot ^ 1);
        cp_async_wait<1>();
        __syncwarp();
        uint8_t *tile = mine + slot * pitch;
        const int off = (int)((reinterpret_cast<uintptr_t>(a.x) + r * a.ldx * sizeof(T)) % 16);
        if (slice < slices) {
            const double pos = (double)static_cast<const P *>(a.pos)[r * a.pos_stride];
            for (int i = own; i < half; i += 32) {
                const float2 t = turn_of<T>(pos, a.freq[i], a.mscale, a.sign);
                T *p = reinterpret_cast<T *>(tile + off) + (INTER ? 2 * i : i), *q = p + (INTER ? 1 : half);
#pragma unroll 4
                for (int h = slice; h < a.heads; h += slices) {
                    const float v = to_f32(p[h * a.hd]), w = to_f32(q[h * a.hd]);
                    p[h * a.hd] = from_f32<T>(v * t.x - w * t.y);
                    q[h * a.hd] = from_f32<T>(v * t.y + w * t.x);
                }
            }
        }
        __syncwarp();
        uint8_t *row = static_cast<uint8_t *>(a.out) + r * a.ldo * (int64_t)sizeof(T);
        for (int q = lane; q < pieces; q += 32) {
            const int b = q * 16 - off;
            if (b >= 0 && b + 16 <= bytes) *reinterpret_cast<uint4 *>(row + b) = *reinterpret_cast<const uint4 *>(tile + q * 16);
            else {
                for (int j = 0; j < 16; j += (int)sizeof(T))
                    if (b + j >= 0 && b + j < bytes) *reinterpret_cast<T *>(row + b + j) = *reinterpret_cast<const T *>(tile + q * 16 + j);
            }
        }
        __syncwarp();  // the slot is free
    }
}

// Launches k_rope_rows where it fits. Long streams only, since it spreads no heads, and rows that give a warp enough to do:
// 131,072 rows of 8 x 151 (bf16, 90 turned) take 125 us, 219 without it, of 3 x 151 86 and 127; 500,000 rows of 2 x 15 would
// take 198, 54 without it.
template <class T, class P>
bool launch_rows(const RopeArgs &a, bool inter, cudaStream_t st) {
    const int64_t bytes = (int64_t)a.heads * a.hd * sizeof(T), pitch = (bytes / 16 + 2) * 16;
    if (a.M < 2048 || bytes < 512 || (a.heads > 1 && (a.hsx != a.hd || a.hso != a.hd)) || a.ldx * (int64_t)sizeof(T) < bytes) return false;
    if ((reinterpret_cast<uintptr_t>(a.x) - reinterpret_cast<uintptr_t>(a.out)) % 16 || (a.ldx - a.ldo) * (int64_t)sizeof(T) % 16) return false;
    int warps = ROPE_THREADS / 32;
    while (warps > 1 && warps * 2 * pitch > ROPE_SMEM) warps /= 2;
    if (warps * 2 * pitch > ROPE_SMEM) return false;
    const auto kernel = inter ? k_rope_rows<T, P, true> : k_rope_rows<T, P, false>;
    static std::atomic<int> known[64][2];
    int dev = 0;
    cudaGetDevice(&dev);
    int sms = known[dev & 63][inter].load(std::memory_order_relaxed);
    if (!sms) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, ROPE_SMEM);
        need(e == cudaSuccess, cudaGetErrorString(e));
        cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
        known[dev & 63][inter].store(sms, std::memory_order_relaxed);
    }
    const int smem = (int)(warps * 2 * pitch);
    const int64_t blocks = std::min<int64_t>((a.M + warps - 1) / warps, (int64_t)sms * std::min(64 / warps, ROPE_SM_SMEM / (smem + 1024)));
    kernel<<<(unsigned)blocks, warps * 32, smem, st>>>(a, (int)bytes);
    return true;
}

// The widest vectors, of V columns or fewer, that the pairs, the copied columns and every row and head are whole multiples of.
template <class T, class P, int V>
void launch_v(const RopeArgs &a, bool inter, cudaStream_t st) {
    const auto at = [](const void *p, int64_t ld, int64_t hs) { return on(p, V * sizeof(T)) && ld % V == 0 && hs % V == 0; };
    if constexpr (V > 1) {
        if (a.rot % (inter ? V : 2 * V) || (a.hd - a.rot) % V || !at(a.x, a.ldx, a.hsx) || !at(a.out, a.ldo, a.hso))
            return launch_v<T, P, V / 2>(a, inter, st);
    }
    if constexpr (V * sizeof(T) <= 4) {
        if (launch_rows<T, P>(a, inter, st)) return;
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
