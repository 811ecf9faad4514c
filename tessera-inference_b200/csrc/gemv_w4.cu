// Linear of a few token rows with 4-bit weights and group scales.
//
// Bound: the bytes of the weights, read once per tile of up to 32 token rows.
// The products run on mma.sync m16n8k16: 16 weight rows are its M side, 8 token
// rows its N side. With one to 32 columns on that side the tensor pipe has
// nothing to win, the weights' codes arrive in the order of the instruction's
// A operand, and a pair of codes becomes two 16-bit floats with a shift, a logic
// and a subtract instruction. A code times an activation is exact in f32, where
// the sums are kept; a group's sum is multiplied by its scale in f32.
//
// One block of 16 warps per SM stays for the whole call. It keeps its token rows
// in shared memory and streams weight records, each warp through a ring of its
// own, filled by asynchronous copies that run on across the ends of tiles. Where
// the token rows of all K columns are large beside a block's share of the
// weights, a cluster of 2, 4 or 8 blocks splits K, and each block stages only its
// slice; the sums of the slices are joined over distributed shared memory.
#include <algorithm>
#include <atomic>

#include <cooperative_groups.h>

#include "token_ops.cuh"

namespace tcb {
namespace {

constexpr int W4_WARPS = 16, W4_THREADS = W4_WARPS * 32;
constexpr int W4_RING = 4;   // records in flight per warp
constexpr int X_PAD = 32;    // 16-bit elements behind a staged token row: rows start 16 banks apart
constexpr int X_SMALL = 32 * 1024, X_PART = 4;  // token rows of up to 32 KB, or a quarter of the weights' share, stay whole
constexpr int SMEM_MAX = 227 * 1024;

template <class X>
using mma_type = std::conditional_t<std::is_same_v<X, f16>, f16, bf16>;

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

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void *src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t p) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(p) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t lds32(uint32_t p) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(p) : "memory");
    return v;
}

// How a launch cuts the work. `split` blocks of a cluster share K; within a block the warps are 16 / wk row tiles times wk
// slices of the records. Cluster c of `clusters` takes row tiles ((c + i clusters) (16 / wk)) + 0 .. in step i < steps.
struct W4Cut {
    int split = 1, wk = 1, clusters = 1, steps = 1;
    int rows = 1;                                    // token rows of a full tile
    int x_at = 0, xsc_at = 0, red_at = 0, part_at = 0;  // byte offsets in shared memory
    bool vec = false;                                // x rows can be read in 8-element steps
};

__device__ __forceinline__ void put_out(const W4Args &a, int otype, int64_t m, int n, float v) {
    if (a.bias) v += a.bias[n];
    if (a.relu) v = v < 0.f ? 0.f : v;
    const int64_t at = m * a.ldo + n, ar = m * a.ldr + n;
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

// X: type of x. SUB: columns whose products share both scales. NT: tiles of 8 token rows. XG: x's scales change along a row.
template <class X, int SUB, int NT, bool XG>
__global__ void __launch_bounds__(W4_THREADS, 1) k_gemv_w4(const W4Args a, const W4Cut cut, const int otype) {
    using T = mma_type<X>;
    extern __shared__ __align__(16) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int wt = W4_WARPS / cut.wk, my_t = warp / cut.wk, my_k = warp % cut.wk;
    const int kb = (a.K + W4_COLS - 1) / W4_COLS, rec = w4_record_bytes(a.group), tiles = (a.N + W4_ROWS - 1) / W4_ROWS;
    const int cluster = blockIdx.x / cut.split, rank = blockIdx.x % cut.split;
    const int b0 = (int)((int64_t)kb * rank / cut.split), b1 = (int)((int64_t)kb * (rank + 1) / cut.split);
    const int m0 = blockIdx.y * cut.rows, rows = min(cut.rows, a.M - m0);
    const int count = (b1 - b0 - my_k + cut.wk - 1) / cut.wk;  // records of this warp in a tile, at least 1

    // the ring: a warp's lanes copy what they read themselves, so no lane waits for another
    const uint32_t ring = smem_u32(smem) + warp * W4_RING * rec;
    const int words = W4_COLS / a.group * W4_ROWS / 2;  // scales of a record, two to a word: one word per lane
    int f_step = 0, f_rec = 0, f_slot = 0;
    const auto fetch = [&] {
        const int tile = (cluster + f_step * cut.clusters) * wt + my_t;
        if (f_step < cut.steps && tile < tiles) {
            const uint8_t *p = static_cast<const uint8_t *>(a.w) + ((int64_t)tile * kb + b0 + my_k + f_rec * cut.wk) * rec;
            const uint32_t d = ring + f_slot * rec;
            cp_async16(d + lane * 16, p + lane * 16);
            cp_async16(d + 512 + lane * 16, p + 512 + lane * 16);
            if (lane < words) cp_async4(d + W4_CODE_BYTES + lane * 4, p + W4_CODE_BYTES + lane * 4);
        }
        cp_async_commit();
        if (++f_rec == count) f_rec = 0, ++f_step;
        f_slot = f_slot + 1 == W4_RING ? 0 : f_slot + 1;
    };
#pragma unroll
    for (int s = 0; s < W4_RING - 1; ++s) fetch();

    // this slice of the token rows, zero behind the last column
    const int pitch = (kb + cut.split - 1) / cut.split * W4_COLS + X_PAD, k0 = b0 * W4_COLS, kn = (b1 - b0) * W4_COLS;
    T *xs = reinterpret_cast<T *>(smem + cut.x_at);
    const X *x = static_cast<const X *>(a.x) + (int64_t)m0 * a.ldx;
    if (cut.vec) {
        const int per = kn / 8;
        for (int e = threadIdx.x; e < rows * per; e += W4_THREADS) {
            const int m = e / per, k = (e - m * per) * 8;
            const X *p = x + m * a.ldx + k0 + k;
            uint4 v;
            if (k0 + k + 8 <= a.K) v = as_mma8(p);
            else {
                T u[8];
                for (int j = 0; j < 8; ++j) u[j] = k0 + k + j < a.K ? as_mma1(p[j]) : T(0.f);
                memcpy(&v, u, 16);
            }
            *reinterpret_cast<uint4 *>(xs + m * pitch + k) = v;
        }
    } else {
        for (int m = 0; m < rows; ++m) {
            const X *p = x + m * a.ldx + k0;
#pragma unroll 4
            for (int k = threadIdx.x; k < kn; k += W4_THREADS) xs[m * pitch + k] = k0 + k < a.K ? as_mma1(p[k]) : T(0.f);
        }
    }
    const int xg = a.xgroup ? a.xgroup : W4_COLS, xgs = kn / xg, nxg = (a.K + xg - 1) / xg;
    float *xsc = reinterpret_cast<float *>(smem + cut.xsc_at);
    if constexpr (XG)
        for (int e = threadIdx.x; e < rows * xgs; e += W4_THREADS) {
            const int m = e / xgs, k = k0 / xg + e - m * xgs;
            xsc[e] = k < nxg ? a.xscales[(int64_t)(m0 + m) * nxg + k] : 0.f;
        }
    __syncthreads();

    uint32_t brow[NT];  // lanes behind the last token row read it again; their sums are not written
#pragma unroll
    for (int n = 0; n < NT; ++n) brow[n] = smem_u32(xs) + (min(8 * n + g, rows - 1) * pitch + 8 * t) * 2;

    float *red = reinterpret_cast<float *>(smem + cut.red_at), *part = reinterpret_cast<float *>(smem + cut.part_at);
    int slot = 0;
    for (int step = 0; step < cut.steps; ++step) {
        const int tile = (cluster + step * cut.clusters) * wt + my_t;
        if (tile >= tiles) break;  // the same for all warps of a tile
        float acc[NT][4] = {};
#pragma unroll 1
        for (int r = 0; r < count; ++r) {
            cp_async_wait<W4_RING - 2>();
            const uint32_t d = ring + slot * rec;
            const uint4 lo = lds128(d + lane * 16), hi = lds128(d + 512 + lane * 16);
            const uint32_t scales = lane < words ? lds32(d + W4_CODE_BYTES + lane * 4) : 0;
            fetch();  // into the slot read in the round before
            slot = slot + 1 == W4_RING ? 0 : slot + 1;
            const uint32_t wl[4] = {lo.x, lo.y, lo.z, lo.w}, wh[4] = {hi.x, hi.y, hi.z, hi.w};
            const int kl = (my_k + r * cut.wk) * W4_COLS;
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
                    const uint4 b = lds128(brow[n] + (kl + 32 * j) * 2);
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
        if constexpr (sizeof(X) == 1 && !XG) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int c = 0; c < 4; ++c) acc[n][c] *= __ldg(a.xscales + m0 + min(8 * n + 2 * t + c % 2, rows - 1));
        }
        // value c of tile n is weight row g + 8 (c / 2), token row 8 n + 2 t + c % 2
        if (cut.wk == 1) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const int m = 8 * n + 2 * t + c % 2, i = g + c / 2 * 8;
                    if (m >= rows) continue;
                    if (cut.split > 1) part[((step * wt + my_t) * rows + m) * W4_ROWS + i] = acc[n][c];
                    else if (tile * W4_ROWS + i < a.N) put_out(a, otype, m0 + m, tile * W4_ROWS + i, acc[n][c]);
                }
            continue;
        }
        // the slices' sums meet in shared memory, in slice order; two buffers in turn, so one barrier does
        float *buf = red + ((step % 2) * wt + my_t) * cut.wk * rows * W4_ROWS;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int m = 8 * n + 2 * t + c % 2;
                if (m < rows) buf[(my_k * rows + m) * W4_ROWS + g + c / 2 * 8] = acc[n][c];
            }
        asm volatile("bar.sync %0, %1;" ::"r"(my_t + 1), "r"(cut.wk * 32) : "memory");
        for (int e = my_k * 32 + lane; e < rows * W4_ROWS; e += cut.wk * 32) {
            float v = 0.f;
            for (int k = 0; k < cut.wk; ++k) v += buf[k * rows * W4_ROWS + e];
            const int m = e / W4_ROWS, n = tile * W4_ROWS + e % W4_ROWS;
            if (cut.split > 1) part[(step * wt + my_t) * rows * W4_ROWS + e] = v;
            else if (n < a.N) put_out(a, otype, m0 + m, n, v);
        }
    }
    if (cut.split == 1) return;

    namespace cg = cooperative_groups;
    const cg::cluster_group cl = cg::this_cluster();
    cl.sync();
    const int all = cut.steps * wt * rows * W4_ROWS;
    for (int e = rank * W4_THREADS + threadIdx.x; e < all; e += cut.split * W4_THREADS) {
        const int local = e / (rows * W4_ROWS), i = e - local * rows * W4_ROWS;
        const int tile = (cluster + local / wt * cut.clusters) * wt + local % wt;
        const int m = i / W4_ROWS, n = tile * W4_ROWS + i % W4_ROWS;
        if (n >= a.N) continue;
        float v = 0.f;
        for (int k = 0; k < cut.split; ++k) v += *cl.map_shared_rank(part + e, k);
        put_out(a, otype, m0 + m, n, v);
    }
    cl.sync();  // no block's sums go while another reads them
}

// Blocks that the device holds at once when every `split` of them form a cluster. Looked up once per device, as the kernel
// gets its shared memory.
template <class X, int SUB, int NT, bool XG>
int resident(int split) {
    const auto kernel = k_gemv_w4<X, SUB, NT, XG>;
    static std::atomic<int> known[64][4];
    int dev = 0, n = 0;
    cudaGetDevice(&dev);
    std::atomic<int> &slot = known[dev & 63][split == 1 ? 0 : split == 2 ? 1 : split == 4 ? 2 : 3];
    if ((n = slot.load(std::memory_order_relaxed))) return n;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_MAX);
    need(e == cudaSuccess, cudaGetErrorString(e));
    if (split == 1) cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    else {
        cudaLaunchConfig_t c = {};
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim.x = split;
        at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
        c.gridDim = dim3(split);
        c.blockDim = dim3(W4_THREADS);
        c.dynamicSmemBytes = SMEM_MAX;
        c.attrs = at;
        c.numAttrs = 1;
        cudaOccupancyMaxActiveClusters(&n, kernel, &c);
        n *= split;
    }
    slot.store(std::max(n, split), std::memory_order_relaxed);
    return std::max(n, split);
}

template <class X, int SUB, int NT, bool XG>
void launch(const W4Args &a, int mt, int otype, cudaStream_t st) {
    const auto kernel = k_gemv_w4<X, SUB, NT, XG>;
    const int kb = (a.K + W4_COLS - 1) / W4_COLS, tiles = (a.N + W4_ROWS - 1) / W4_ROWS, rec = w4_record_bytes(a.group);
    W4Cut cut;
    cut.rows = (int)((a.M + (int64_t)mt - 1) / mt);
    cut.vec = reinterpret_cast<uintptr_t>(a.x) % (8 * sizeof(X)) == 0 && a.ldx % 8 == 0;
    const int ring = W4_WARPS * W4_RING * rec;
    const auto x_bytes = [&](int split) {
        return cut.rows * ((kb + split - 1) / split * W4_COLS * 2 + X_PAD * 2);
    };
    const auto xsc_bytes = [&](int split) { return XG ? cut.rows * ((kb + split - 1) / split) * (W4_COLS / a.xgroup) * 4 : 0; };
    // K is split until a block's token rows are small beside its weights, or small at all
    const int64_t share = (int64_t)tiles * kb * rec / resident<X, SUB, NT, XG>(1);
    const int tile_bytes = cut.rows * W4_ROWS * 4;
    const auto fixed_bytes = [&](int split) { return ring + x_bytes(split) + xsc_bytes(split); };
    while (cut.split < 8 && cut.split * 2 <= kb &&
           (x_bytes(cut.split) > std::max<int64_t>(X_SMALL, share / X_PART) ||
            fixed_bytes(cut.split) + W4_WARPS * tile_bytes > SMEM_MAX))
        cut.split *= 2;
    const int fixed = fixed_bytes(cut.split);
    // Slices of the records within a block: the fewest record times, where a tile's end costs one or two of them.
    const int most = std::max(1, resident<X, SUB, NT, XG>(cut.split) / cut.split / mt);
    int64_t best = INT64_MAX;
    W4Cut found = cut;
    for (int wk = 1; wk <= W4_WARPS && wk <= kb / cut.split; wk *= 2) {
        const int wt = W4_WARPS / wk, red = wk > 1 ? 2 * W4_WARPS * tile_bytes : 0;
        const int all = (tiles + wt - 1) / wt, room = SMEM_MAX - fixed - red;
        if (room < (cut.split > 1 ? wt * tile_bytes : 0)) continue;
        int steps = (all + most - 1) / most;
        if (cut.split > 1) steps = std::min(steps, room / (wt * tile_bytes));
        const int clusters = (all + steps - 1) / steps, waves = (clusters + most - 1) / most;
        const int64_t cost = (int64_t)waves * steps * (((kb + cut.split - 1) / cut.split + wk - 1) / wk + (wk > 1 ? 2 : 1));
        if (cost >= best) continue;
        best = cost;
        found.wk = wk;
        found.clusters = clusters;
        found.steps = steps;
        found.split = cut.split;
        found.x_at = ring;
        found.xsc_at = ring + x_bytes(cut.split);
        found.red_at = fixed;
        found.part_at = fixed + red;
    }
    need(best < INT64_MAX, "the token rows do not fit the shared memory");
    cut = found;
    const int bytes = cut.part_at + (cut.split > 1 ? cut.steps * (W4_WARPS / cut.wk) * tile_bytes : 0);

    cudaLaunchConfig_t c = {};
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = cut.split;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    c.gridDim = dim3(cut.clusters * cut.split, mt);
    c.blockDim = dim3(W4_THREADS);
    c.dynamicSmemBytes = bytes;
    c.stream = st;
    c.attrs = at;
    c.numAttrs = cut.split > 1 ? 1 : 0;
    const cudaError_t e = cudaLaunchKernelEx(&c, kernel, a, cut, otype);
    need(e == cudaSuccess, cudaGetErrorString(e));
}

// Token rows are cut into equal tiles of at most 32, and of no more than a cluster's shared memory holds.
template <class X, int SUB, bool XG>
void launch_n(const W4Args &a, int otype, cudaStream_t st) {
    const int kb = (a.K + W4_COLS - 1) / W4_COLS, split = kb >= 8 ? 8 : kb >= 4 ? 4 : kb >= 2 ? 2 : 1;
    const int row = (kb + split - 1) / split * (W4_COLS * 2 + (XG ? W4_COLS / a.xgroup * 4 : 0)) + X_PAD * 2;
    const int room = SMEM_MAX - W4_WARPS * W4_RING * w4_record_bytes(a.group);
    const int fit = std::min(32, room / (row + W4_WARPS * W4_ROWS * 4));  // with one step of sums
    const int64_t mt = (a.M + fit - 1ll) / fit;
    const int64_t rows = (a.M + mt - 1) / mt;
    if (rows <= 8) launch<X, SUB, 1, XG>(a, (int)mt, otype, st);
    else if (rows <= 16) launch<X, SUB, 2, XG>(a, (int)mt, otype, st);
    else if (rows <= 24) launch<X, SUB, 3, XG>(a, (int)mt, otype, st);
    else launch<X, SUB, 4, XG>(a, (int)mt, otype, st);
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
    need(a.M >= 0 && a.M <= 1 << 18, "M is not in 0..2^18");
    need(w4_bytes(a.N, a.K, a.group) > 0, "N < 1, K is not in 1..65536 or group is not 32, 64 or 128");
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
