// Linear of a few token rows with 4-bit weights and group scales.
//
// Bound: the bytes of the weights, read once per tile of up to 32 token rows. The
// products run on mma.sync m16n8k16: 16 weight rows are its M side, 8 token rows
// its N side, and the weights' codes arrive in the order of its A operand. What has
// to be cheap is turning codes into 16-bit floats:
//
//   u = q + 8 in the low bits of a 16-bit float (fp16 or bf16, as the token rows) is the subnormal u e, in bits 4-7 it is
//   16 u e, e the type's smallest step. One logic instruction per pair of codes brings it there (and one shift per eight), one
//   fused multiply-add makes it q 2^-10: both exact, so a code of 0 is a 0 whatever x it meets.
//
// Products are exact, sums are f32; a group's sum is multiplied by its scale in f32. With the 2^-10 no group's sum leaves
// f32's range, whatever bf16 values it has, and no product falls below its smallest step; the outputs are multiplied by 2^10.
// Infinities and NaN among the activations take their course. Outputs of 8-bit x that are not finite are computed again from
// the definition: a sum may leave f32's range before the scale that brings it back, and an infinite scale meets each x there,
// not their sum.
//
// bf16 and fp16 token rows are staged as they are, 8-bit ones as fp16, which holds them exactly.
//
// One block of 16 warps per SM stays for the whole call. It keeps its token rows
// in shared memory and streams weight records, each warp through a ring of its
// own, filled by asynchronous copies that start before the token rows are there and
// run on across the ends of tiles. A cluster of 2, 4 or 8 blocks may split K, where
// the token rows of all K columns are too many for a block or the weight rows too
// few for the SMs; the sums of the slices are joined over distributed shared memory.
//
// Measured (bf16 rows): 1 x 16,384 x 8,192 in 18.6 us, 3.7 TB/s of weights, with
// scales of 32 in 22.7. Of that 2 us are the launch and 4 the code's first run and
// the token rows, while only the rings fill; the codes' way to 16 bits keeps 63% of
// the issue slots busy. 8 x 8,192 x 8,192 in 13.0 us (14.3 with scales of 64), 32 x
// 8,192 x 8,192 in 29.6, 1 x 2,560 x 1,280 in 4.4 to 5.0 us.
#include <algorithm>
#include <atomic>

#include <cooperative_groups.h>

#include "token_ops.cuh"

namespace tcb {
namespace {

constexpr int W4_WARPS = 16, W4_THREADS = W4_WARPS * 32;
constexpr int RING = 4;    // records in flight per warp; eight are faster by 2% at most on 46 sizes and take the room of token rows
constexpr int X_PAD = 32;  // 16-bit elements behind a staged token row: rows start 16 banks apart
constexpr int SMEM_MAX = 227 * 1024;

// d = A B + c on bf16 (BF) or fp16
template <bool BF>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, float4 c) {
    if constexpr (BF)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c.x), "f"(c.y), "f"(c.z), "f"(c.w));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c.x), "f"(c.y), "f"(c.z), "f"(c.w));
}

// Two codes u = q + 8, in the low bits of a word's halves (HIGH: in their bits 4-7), as q 2^-10.
constexpr float W4_CODE = 0x1p-10f;
template <bool BF, bool HIGH>
__device__ __forceinline__ uint32_t codes2(uint32_t u) {
    constexpr float UP = (BF ? 0x1p123f : 0x1p14f) / (HIGH ? 16.f : 1.f);  // 2^-10 over the type's smallest step
    uint32_t w;
    if constexpr (BF) {
        const __nv_bfloat162 v = __hfma2(*reinterpret_cast<const __nv_bfloat162 *>(&u), __float2bfloat162_rn(UP), __float2bfloat162_rn(-8.f * W4_CODE));
        memcpy(&w, &v, 4);
    } else {
        const __half2 v = __hfma2(*reinterpret_cast<const __half2 *>(&u), __float2half2_rn(UP), __float2half2_rn(-8.f * W4_CODE));
        memcpy(&w, &v, 4);
    }
    return w;
}

// An 8-bit element of x, or two, as fp16.
__device__ __forceinline__ uint16_t half_of(uint8_t v, int xtype) {
    if (xtype == TCB_I8) return __half_as_ushort(__short2half_rn((int8_t)v));
    return __nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)v, __NV_E4M3).x;
}
__device__ __forceinline__ uint32_t half2_of(uint32_t v, int xtype) {
    __half2 h;
    if (xtype == TCB_I8) h = __floats2half2_rn((float)(int8_t)v, (float)(int8_t)(v >> 8));
    else h = __half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(v & 0xffffu), __NV_E4M3));
    return *reinterpret_cast<const uint32_t *>(&h);
}

__device__ __forceinline__ uint4 lds128(uint32_t p) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(p) : "memory");
    return v;
}
__device__ __forceinline__ float2 lds_f32x2(uint32_t p) {
    float2 v;
    asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(p) : "memory");
    return v;
}
__device__ __forceinline__ float lds_bf16(uint32_t p) {
    uint16_t v;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(p) : "memory");
    return bf16lo(v);
}

// 8 elements of x from element i on, a multiple of 8, as they are stored: 16-bit ones fill four words, 8-bit ones two.
// Elements from `end` on are zero.
__device__ __forceinline__ uint4 x8(const void *x, int64_t i, int64_t end, bool wide) {
    if (i + 8 <= end) {
        if (wide) return *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(x) + i);
        const uint2 q = *reinterpret_cast<const uint2 *>(static_cast<const uint8_t *>(x) + i);
        return make_uint4(q.x, q.y, 0, 0);
    }
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (i + j < end) {
            if (wide) w[j / 2] |= (uint32_t)static_cast<const uint16_t *>(x)[i + j] << 16 * (j % 2);
            else w[j / 4] |= (uint32_t)static_cast<const uint8_t *>(x)[i + j] << 8 * (j % 4);
        }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// A pass is 256 columns of a token row; a warp takes every 16th of a block's.
struct Pass {
    int m, p, passes, dm, dp;
    __device__ __forceinline__ Pass(int passes, int first)
        : m(first / passes), p(first % passes), passes(passes), dm(W4_WARPS / passes), dp(W4_WARPS % passes) {}
    __device__ __forceinline__ void next() {
        m += dm;
        p += dp;
        if (p >= passes) p -= passes, ++m;
    }
};

// A warp's passes of `rows` rows of x into shared memory, N passes' loads at once. `left`: columns of x
// from its first one here on; the rest up to kn are zero. 8-bit elements become fp16.
template <int N, class E>
__device__ __forceinline__ void x_scatter(const E *x, int xtype, int64_t ldx, int left, int kn, int rows, uint16_t *xs, int pitch) {
    const int lane = threadIdx.x & 31;
    Pass load((kn + 255) / 256, threadIdx.x >> 5), put = load;
#pragma unroll 1
    while (load.m < rows) {
        uint32_t u[N][8];
#pragma unroll
        for (int i = 0; i < N; ++i, load.next()) {
            const int c = load.p * 256 + lane, end = load.m < rows ? left : 0;
            const E *p = x + load.m * ldx + c;
#pragma unroll
            for (int j = 0; j < 8; ++j) u[i][j] = c + 32 * j < end ? (uint32_t)p[32 * j] : 0u;
        }
#pragma unroll
        for (int i = 0; i < N; ++i, put.next()) {
            const int c = put.p * 256 + lane, end = put.m < rows ? kn : 0;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (c + 32 * j < end) xs[put.m * pitch + c + 32 * j] = sizeof(E) == 1 ? half_of((uint8_t)u[i][j], xtype) : (uint16_t)u[i][j];
        }
    }
}

// How a launch cuts the work. `split` blocks of a cluster share K; within a block the warps are 16 / wk row tiles times wk
// slices of the records. Tile j of cluster c of `clusters` in step i is row tile c + (16 / wk i + j) clusters, so that all SMs
// get work; after every `steps` steps, `batches` times, a cluster joins its slices' sums.
struct W4Cut {
    int split = 1, wk = 1, clusters = 1, steps = 1, batches = 1;
    int rows = 1;                                                    // token rows of a full tile
    int x_at = 0, xs_at = 0, red_at = 0, part_at = 0;                // byte offsets in shared memory
    bool vec = false;                                                // x rows can be read in 8-element steps
};

// Whether a NaN is among a row's codes or scales; all lanes of a warp ask together.
__device__ __forceinline__ bool nan_row(const W4Args &a, int xtype, int m) {
    const int lane = threadIdx.x & 31, nxg = a.xgroup ? (a.K + a.xgroup - 1) / a.xgroup : 1;
    bool found = false;
    for (int g = lane; g < nxg; g += 32) found |= isnan(a.xscales[(int64_t)m * nxg + g]);
    found = __any_sync(~0u, found);
    const uint8_t *x = static_cast<const uint8_t *>(a.x) + m * a.ldx;
    for (int k0 = 0; xtype == TCB_E4M3 && !found && k0 < a.K; k0 += 128) {
#pragma unroll
        for (int j = 0; j < 4; ++j) found |= (x[min(k0 + 32 * j + lane, a.K - 1)] & 0x7f) == 0x7f;
        found = __any_sync(~0u, found);
    }
    return found;
}

// Outputs (m, n) of 8-bit x from the definition, for the lanes that ask: all lanes of the warp come here and sum one output after
// the other, in f64, where every product is exact. Rows with a NaN, a padded batch's for instance, need no sum.
__device__ __noinline__ float w4_plain(const W4Args &a, int xtype, bool ask, int m, int n, float v) {
    const int lane = threadIdx.x & 31, kb = (a.K + W4_COLS - 1) / W4_COLS, rec = w4_record_bytes(a.group);
    const int xg = a.xgroup ? a.xgroup : a.K, nxg = (a.K + xg - 1) / xg;
    int last = -1;
    bool nan = false;
    for (uint32_t asked = __ballot_sync(~0u, ask); asked; asked &= asked - 1) {
        const int who = __ffs(asked) - 1, row = __shfl_sync(~0u, m, who), r = __shfl_sync(~0u, n, who);
        if (row != last) last = row, nan = nan_row(a, xtype, row);
        if (nan) {
            if (lane == who) v = __int_as_float(0x7fffffff);
            continue;
        }
        const uint8_t *w = static_cast<const uint8_t *>(a.w) + (int64_t)(r / W4_ROWS) * kb * rec;
        const int half = r % W4_ROWS / 8, low = r % 8;
        double sum = 0.;
#pragma unroll 1
        for (int first = 0; first < a.K; first += 256) {
            const int k0 = first + lane * 8;  // 8 columns: one word of codes, one scale of each kind
            if (k0 < a.K) {
                const int j = k0 % W4_COLS, i = j / 32, t = j / 8 % 4;
                const uint8_t *p = w + (int64_t)(k0 / W4_COLS) * rec;
                const uint32_t codes = *reinterpret_cast<const uint32_t *>(p + 512 * half + 64 * low + 16 * t + 4 * i);
                const double s = to_f32(reinterpret_cast<const bf16 *>(p + W4_CODE_BYTES)[j / a.group * W4_ROWS + r % W4_ROWS]);
                const double xs = a.xscales[(int64_t)row * nxg + k0 / xg];
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    const int64_t at = row * a.ldx + min(k0 + c, a.K - 1);
                    const float x = xtype == TCB_I8 ? to_f32(static_cast<const int8_t *>(a.x)[at]) : to_f32(static_cast<const e4m3 *>(a.x)[at]);
                    if (k0 + c < a.K) sum += x * xs * ((int)(codes >> 4 * (c / 2 + 4 * (c % 2)) & 15) - 8) * s;
                }
            }
            if (__any_sync(~0u, sum != sum) || (__any_sync(~0u, sum > 1e300) && __any_sync(~0u, sum < -1e300))) break;  // NaN for good
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
        if (lane == who) v = (float)sum;
    }
    return v;
}

// What output (m, n) is made of beside its sum.
struct Beside {
    float scale, bias, res;
};
__device__ __forceinline__ Beside beside(const W4Args &a, int otype, bool row_scales, int m, int n) {
    Beside b = {1.f, 0.f, 0.f};
    if (row_scales) b.scale = a.xscales[m];
    if (a.bias) b.bias = a.bias[n];
    if (a.res) {
        const int64_t at = m * a.ldr + n;
        b.res = otype == TCB_BF16  ? to_f32(static_cast<const bf16 *>(a.res)[at])
                : otype == TCB_F16 ? to_f32(static_cast<const f16 *>(a.res)[at])
                                   : static_cast<const float *>(a.res)[at];
    }
    return b;
}
// Writes the outputs of a warp's lanes that have one; all lanes come here.
template <bool CODES>
__device__ __forceinline__ void put_out(const W4Args &a, int xtype, int otype, bool out, int m, int n, float v, const Beside &b) {
    v *= 1.f / W4_CODE;
    if (CODES && a.xscales) {
        v *= b.scale;
        const bool ask = out && !(fabsf(v) <= 3.4028235e38f);
        if (__any_sync(~0u, ask)) v = w4_plain(a, xtype, ask, m, n, v);
    }
    if (!out) return;
    v += b.bias;
    if (a.relu) v = v < 0.f ? 0.f : v;
    if (a.res) v += b.res;
    const int64_t at = m * a.ldo + n;
    if (otype == TCB_BF16) static_cast<bf16 *>(a.out)[at] = from_f32<bf16>(v);
    else if (otype == TCB_F16) static_cast<f16 *>(a.out)[at] = from_f32<f16>(v);
    else static_cast<float *>(a.out)[at] = v;
}

// SUB: columns whose products share both scales. NT: tiles of 8 token rows. X: bf16 x, fp16 x (or 8-bit with one scale per row),
// or 8-bit x with scales along its rows.
enum W4X { X_BF16, X_F16, X_SCALED };
template <int SUB, int NT, W4X X>
__global__ void __launch_bounds__(W4_THREADS, 1)
    k_gemv_w4(const __grid_constant__ W4Args a, const __grid_constant__ W4Cut cut, const int xtype, const int otype) {
    extern __shared__ __align__(16) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int wt = W4_WARPS / cut.wk, my_t = warp / cut.wk, my_k = warp % cut.wk;
    const int kb = (a.K + W4_COLS - 1) / W4_COLS, rec = w4_record_bytes(a.group), tiles = (a.N + W4_ROWS - 1) / W4_ROWS;
    const int cluster = blockIdx.x / cut.split, rank = blockIdx.x % cut.split;
    const int b0 = (int)((int64_t)kb * rank / cut.split), b1 = (int)((int64_t)kb * (rank + 1) / cut.split);
    const int m0 = blockIdx.y * cut.rows, rows = min(cut.rows, a.M - m0);
    // records of this warp in a tile, at least one, in a row
    const int r0 = (b1 - b0) * my_k / cut.wk, count = (b1 - b0) * (my_k + 1) / cut.wk - r0;

    // the ring: a warp's lanes copy what they read themselves, but for the scales (lanes below `tail`, 16 bytes each)
    const uint32_t ring = smem_u32(smem) + warp * RING * rec, ring_end = ring + RING * rec;
    const int tail = (rec - W4_CODE_BYTES) / 16;
    const int first = cluster + my_t * cut.clusters, hop = cut.clusters * wt;  // tiles of this warp: first, first + hop, ...
    const uint8_t *f_src = static_cast<const uint8_t *>(a.w) + ((int64_t)first * kb + b0 + r0) * rec + lane * 16;
    int f_left = first < tiles ? (tiles - first + hop - 1) / hop * count : 0, f_rec = count;
    const int64_t f_hop = ((int64_t)hop * kb - count) * rec;
    const auto fetch = [&](uint32_t dst) {
        if (--f_left >= 0) {
            cp_async16(dst, f_src);
            cp_async16(dst + 512, f_src + 512);
            if (lane < tail) cp_async16(dst + W4_CODE_BYTES, f_src + W4_CODE_BYTES);
            f_src += rec;
            if (--f_rec == 0) f_rec = count, f_src += f_hop;
        }
        cp_async_commit();
    };
    fetch(ring + lane * 16);
    fetch(ring + rec + lane * 16);

    // This slice of the token rows: 32 times 8 columns of a row per warp and pass, zero behind the last column. Loads go out
    // four passes ahead of their use, the first ones before most of the ring's.
    const int pitch = (kb + cut.split - 1) / cut.split * W4_COLS + X_PAD, k0 = b0 * W4_COLS, kn = (b1 - b0) * W4_COLS;
    const int passes = (kn + 255) / 256;
    const bool wide = xtype == TCB_BF16 || xtype == TCB_F16;
    Pass go(passes, warp), load(passes, warp);  // the pass at work, and the next one to load
    const auto x_load = [&] {
        const int k = k0 + load.p * 256 + lane * 8;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (cut.vec && load.m < rows && k < min(a.K, k0 + kn)) {
            const int64_t row = (int64_t)(m0 + load.m) * a.ldx;
            v = x8(a.x, row + k, row + a.K, wide);
        }
        load.next();
        return v;
    };
    uint4 ahead[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) ahead[i] = x_load();

#pragma unroll 1
    for (int s = 2; s < RING - 1; ++s) fetch(ring + s * rec + lane * 16);

    uint16_t *xs = reinterpret_cast<uint16_t *>(smem + cut.x_at);
    if (!cut.vec) {
        // rows that no vector fits: one element per access, consecutive over the warp
        if (wide) x_scatter<4>(static_cast<const uint16_t *>(a.x) + (int64_t)m0 * a.ldx + k0, xtype, a.ldx, a.K - k0, kn, rows, xs, pitch);
        else x_scatter<4>(static_cast<const uint8_t *>(a.x) + (int64_t)m0 * a.ldx + k0, xtype, a.ldx, a.K - k0, kn, rows, xs, pitch);
    } else {
#pragma unroll 1
        for (; go.m < rows; go.next()) {
            uint4 v = ahead[0];
            ahead[0] = ahead[1], ahead[1] = ahead[2], ahead[2] = ahead[3];
            ahead[3] = x_load();
            const int k = go.p * 256 + lane * 8;
            if (!wide) v = make_uint4(half2_of(v.x, xtype), half2_of(v.x >> 16, xtype), half2_of(v.y, xtype), half2_of(v.y >> 16, xtype));
            if (k < kn) *reinterpret_cast<uint4 *>(xs + go.m * pitch + k) = v;
        }
    }
    // x's scales, per SUB columns and pair of token rows
    float *xsc = reinterpret_cast<float *>(smem + cut.xs_at);
    constexpr bool XG = X == X_SCALED;
    constexpr int GROUP = 8 * NT;
    if constexpr (XG) {
        const int subs = kn / SUB, nxg = (a.K + a.xgroup - 1) / a.xgroup;
        for (int e = threadIdx.x; e < rows * subs; e += W4_THREADS) {
            const int m = e / subs, j = e - m * subs, k = k0 + j * SUB;
            xsc[j * GROUP + m] = k < a.K ? __ldg(a.xscales + (int64_t)(m0 + m) * nxg + k / a.xgroup) : 0.f;
        }
    }
    __syncthreads();

    uint32_t brow[NT];  // lanes behind the last token row read it again; their sums are not written
#pragma unroll
    for (int n = 0; n < NT; ++n) brow[n] = smem_u32(xs) + (min(8 * n + g, rows - 1) * pitch + 8 * t) * 2;
    const uint32_t my_xsc = smem_u32(xsc) + 8 * t;
    float *red = reinterpret_cast<float *>(smem + cut.red_at), *part = reinterpret_cast<float *>(smem + cut.part_at);
    const int tile_floats = rows * W4_ROWS;
    namespace cg = cooperative_groups;
    const cg::cluster_group cl = cg::this_cluster();

    uint32_t slot = ring, before = ring + (RING - 1) * rec;
    int tile = first;
#pragma unroll 1
    for (int batch = 0; batch < cut.batches; ++batch) {
#pragma unroll 1
        for (int step = 0; step < cut.steps && tile < tiles; ++step, tile += hop) {  // alike for all warps of a tile
            float acc[NT][4] = {};
            uint32_t xo = r0 * W4_COLS * 2, so = my_xsc + r0 * (W4_COLS / SUB) * GROUP * 4;
            // two records' chains of products side by side, where the registers allow (one token on 16,384 x 8,192 with scales of
            // 32: one record at a time takes 8% more; 32 tokens on 8,192 x 8,192: two take 3% more)
#pragma unroll (NT == 1 ? 2 : 1)
            for (int r = 0; r < count; ++r) {
                cp_async_wait<RING - 2>();
                __syncwarp();
                const uint4 lo = lds128(slot + lane * 16), hi = lds128(slot + 512 + lane * 16);
                float su[W4_COLS / SUB], sv[W4_COLS / SUB];  // scales of rows g and g + 8
#pragma unroll
                for (int j = 0; j < W4_COLS / SUB; ++j) {
                    const uint32_t p = slot + W4_CODE_BYTES + (j * SUB / a.group * W4_ROWS + g) * 2;
                    su[j] = lds_bf16(p);
                    sv[j] = lds_bf16(p + 16);
                }
                fetch(before + lane * 16);  // the slot read in the round before
                before = slot;
                slot = slot + rec == ring_end ? ring : slot + rec;
                const uint32_t wl[4] = {lo.x, lo.y, lo.z, lo.w}, wh[4] = {hi.x, hi.y, hi.z, hi.w};
                float v[NT][4];  // sums of SUB columns
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int sub = j * 32 / SUB;
                    const uint32_t vl = wl[j] >> 8, vh = wh[j] >> 8;
                    constexpr bool BF = X == X_BF16;
                    const uint32_t A[4] = {codes2<BF, false>(wl[j] & 0x000f000fu), codes2<BF, false>(wh[j] & 0x000f000fu),
                                           codes2<BF, true>(wl[j] & 0x00f000f0u), codes2<BF, true>(wh[j] & 0x00f000f0u)};
                    const uint32_t B[4] = {codes2<BF, false>(vl & 0x000f000fu), codes2<BF, false>(vh & 0x000f000fu),
                                           codes2<BF, true>(vl & 0x00f000f0u), codes2<BF, true>(vh & 0x00f000f0u)};
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        const uint4 b = lds128(brow[n] + xo + 64 * j);
                        mma16816<BF>(v[n], A, b.x, b.y, j * 32 % SUB == 0 ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(v[n][0], v[n][1], v[n][2], v[n][3]));
                        mma16816<BF>(v[n], B, b.z, b.w, make_float4(v[n][0], v[n][1], v[n][2], v[n][3]));
                    }
                    if ((j + 1) * 32 % SUB == 0) {
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            if constexpr (XG) {
                                const float2 xf = lds_f32x2(so + (sub * GROUP + 8 * n) * 4);
                                v[n][0] *= xf.x, v[n][1] *= xf.y, v[n][2] *= xf.x, v[n][3] *= xf.y;
                            }
                            acc[n][0] = fmaf(v[n][0], su[sub], acc[n][0]);
                            acc[n][1] = fmaf(v[n][1], su[sub], acc[n][1]);
                            acc[n][2] = fmaf(v[n][2], sv[sub], acc[n][2]);
                            acc[n][3] = fmaf(v[n][3], sv[sub], acc[n][3]);
                        }
                    }
                }
                xo += W4_COLS * 2;
                so += W4_COLS / SUB * GROUP * 4;
            }
            // Slices' sums meet in shared memory, in slice order. Two buffers in turn, so one barrier does; a warp that has
            // its tile alone needs one buffer, or none when the cluster joins slices anyway.
            float *joined = part + (step * wt + my_t) * tile_floats;
            float *buf = cut.wk > 1 ? red + (((step & 1) * wt + my_t) * cut.wk + my_k) * tile_floats
                         : cut.split > 1 ? joined : red + my_t * tile_floats;
            __syncwarp();
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int c = 0; c < 4; ++c) {  // weight row g + 8 (c / 2), token row 8 n + 2 t + c % 2
                    const int m = 8 * n + 2 * t + c % 2;
                    if (m < rows) buf[m * W4_ROWS + g + c / 2 * 8] = acc[n][c];
                }
            if (cut.wk > 1) asm volatile("bar.sync %0, %1;" ::"r"(my_t + 1), "r"(cut.wk * 32) : "memory");
            else __syncwarp();
            if (cut.wk == 1 && cut.split > 1) continue;
            buf -= my_k * tile_floats;
#pragma unroll 1
            for (int e0 = my_k * 32; e0 < tile_floats; e0 += cut.wk * 32) {  // a warp's lanes stay together
                const int e = e0 + lane, m = m0 + e / W4_ROWS, n = tile * W4_ROWS + e % W4_ROWS;
                const bool mine = e < tile_floats, out = mine && cut.split == 1 && n < a.N;
                Beside b = {};
                if (out) b = beside(a, otype, !XG && a.xscales, m, n);
                float v = 0.f;
                if (mine)
                    for (int k = 0; k < cut.wk; ++k) v += buf[k * tile_floats + e];
                if (cut.split > 1) {
                    if (mine) joined[e] = v;
                } else put_out<X != X_BF16>(a, xtype, otype, out, m, n, v, b);
            }
        }
        if (cut.split == 1) break;
        cl.sync();
        const int all = cut.steps * wt * tile_floats;
#pragma unroll 1
        for (int e0 = rank * W4_THREADS + warp * 32; e0 < all; e0 += 2 * cut.split * W4_THREADS) {  // a warp's lanes stay together
            const int e = e0 + lane;
            int m[2], n[2];
            float u[2][8];
            Beside b[2] = {};
#pragma unroll
            for (int i = 0; i < 2; ++i) {  // two outputs' loads, remote and global, before the first sum
                const int f = e + i * cut.split * W4_THREADS, local = f / tile_floats, r = f - local * tile_floats;
                const int at = cluster + (batch * cut.steps * wt + local) * cut.clusters;
                m[i] = m0 + r / W4_ROWS;
                n[i] = at * W4_ROWS + r % W4_ROWS;
                if (f >= all || at >= tiles || n[i] >= a.N) n[i] = -1;
                if (n[i] >= 0) b[i] = beside(a, otype, !XG && a.xscales, m[i], n[i]);
#pragma unroll
                for (int k = 0; k < 8; ++k) u[i][k] = n[i] >= 0 && k < cut.split ? *cl.map_shared_rank(part + f, k) : 0.f;
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float v = 0.f;
#pragma unroll
                for (int k = 0; k < 8; ++k) v += u[i][k];
                put_out<X != X_BF16>(a, xtype, otype, n[i] >= 0, m[i], n[i], v, b[i]);
            }
        }
        cl.sync();  // no block's sums go while another reads them
    }
}

// Blocks that the device holds at once when every `split` of them form a cluster. Looked up once per device, as the kernel
// gets its shared memory.
template <int SUB, int NT, W4X X>
int resident(int split) {
    const auto kernel = k_gemv_w4<SUB, NT, X>;
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

// Shared memory of the ring, and of `rows` token rows and their scales in one of `split` slices.
struct Fixed {
    int ring, x, scales;
    int all() const { return ring + x + scales; }
};
Fixed fixed_bytes(int group, int rows, int kb, int split, int sub, bool xg) {
    const int recs = (kb + split - 1) / split;
    return {W4_WARPS * RING * w4_record_bytes(group), rows * (recs * W4_COLS * 2 + X_PAD * 2),
            xg ? (rows + 7) / 8 * 8 * recs * (W4_COLS / sub) * 4 : 0};
}

// The cheapest cut by a model in clock cycles: a record takes an SM 46 cycles at HBM's rate or 52 per 8 token rows (the codes'
// way to 16 bits, the products, the fragments from shared memory), and a warp 500 and 200 per 8 token rows at least; a tile's
// end 1,100, and 270 per slice that meets there, staging 2,000 and 17 bytes in two, a join 4,200. Fitted to every cut of 46
// sizes of 1 to 64 token rows: what it takes is 0.6% slower than the best in the mean, 5% at most (1.2% and 5% on 38
// sizes of one to four rows that it was not fitted to). Sizes only: the cut sets the order of the sums, and pointers' alignment
// shall not.
// Returns its cost, or INT64_MAX where nothing fits.
int64_t best_cut(const W4Args &a, int mt, int sub, bool xg, int split, int blocks, W4Cut &out, int &bytes) {
    const int kb = (a.K + W4_COLS - 1) / W4_COLS, tiles = (a.N + W4_ROWS - 1) / W4_ROWS, nt = (out.rows + 7) / 8;
    const Fixed f = fixed_bytes(a.group, out.rows, kb, split, sub, xg);
    const int tile_bytes = out.rows * W4_ROWS * 4, most = std::max(1, blocks / split / mt);
    int64_t best = INT64_MAX;
    for (int wk = 1; wk <= W4_WARPS && wk <= kb / split; wk *= 2) {
        const int wt = W4_WARPS / wk, red = wk > 1 ? 2 * W4_WARPS * tile_bytes : split > 1 ? 0 : W4_WARPS * tile_bytes;
        const int room = SMEM_MAX - f.all() - red, clusters = std::min(tiles, most), each = (tiles + clusters - 1) / clusters;
        int steps = (each + wt - 1) / wt, batches = 1;
        if (room < (split > 1 ? wt * tile_bytes : 0)) continue;
        if (split > 1) {
            batches = (int)(((int64_t)steps * wt * tile_bytes + room - 1) / room);  // 2^31 bytes of sums and more at the largest N
            while ((steps + batches - 1) / batches * wt * tile_bytes > room) ++batches;
            steps = (steps + batches - 1) / batches;
        }
        const int64_t count = ((kb + split - 1) / split + wk - 1) / wk;
        int64_t cost = std::max((int64_t)each * ((kb + split - 1) / split) * std::max(46, 52 * nt), batches * steps * count * (500 + 200 * nt));
        cost += 2000 + f.x * 2 / 17 + (int64_t)batches * steps * (1100 + (wk > 1 ? 270 * wk : 0));
        if (split > 1) cost += batches * 4200;
        if (cost >= best) continue;
        best = cost;
        out.split = split, out.wk = wk, out.clusters = clusters, out.steps = steps, out.batches = batches;
        out.x_at = f.ring;
        out.xs_at = out.x_at + f.x;
        out.red_at = f.all();
        out.part_at = f.all() + red;
        bytes = out.part_at + (split > 1 ? steps * wt * tile_bytes : 0);
    }
    return best;
}

template <int SUB, int NT, W4X X>
void launch(const W4Args &a, const W4Cut &cut, int bytes, int mt, int xtype, int otype, cudaStream_t st) {
    resident<SUB, NT, X>(1);
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
    const cudaError_t e = cudaLaunchKernelEx(&c, k_gemv_w4<SUB, NT, X>, a, cut, xtype, otype);
    need(e == cudaSuccess, cudaGetErrorString(e));
}

template <int SUB, int NT, W4X X>
void launch_cut(const W4Args &a, int mt, int xtype, int otype, cudaStream_t st) {
    const int kb = (a.K + W4_COLS - 1) / W4_COLS;
    W4Cut base, cut;
    base.rows = (int)((a.M + (int64_t)mt - 1) / mt);
    base.vec = reinterpret_cast<uintptr_t>(a.x) % (xtype == TCB_I8 || xtype == TCB_E4M3 ? 8 : 16) == 0 && a.ldx % 8 == 0;
    int64_t best = INT64_MAX;
    int bytes = 0;
    for (int split = 1; split <= 8 && split <= kb; split *= 2) {
        W4Cut c = base;
        int b = 0;
        const int64_t cost = best_cut(a, mt, SUB, X == X_SCALED, split, resident<SUB, NT, X>(split), c, b);
        if (cost < best) best = cost, cut = c, bytes = b;
    }
    need(best < INT64_MAX, "the token rows do not fit the shared memory");
    launch<SUB, NT, X>(a, cut, bytes, mt, xtype, otype, st);
}

// Token rows are cut into equal tiles of at most 32, and of no more than a cluster's shared memory holds.
template <int SUB, W4X X>
void launch_n(const W4Args &a, int xtype, int otype, cudaStream_t st) {
    const int kb = (a.K + W4_COLS - 1) / W4_COLS, split = kb >= 8 ? 8 : kb >= 4 ? 4 : kb >= 2 ? 2 : 1;
    int fit = 32;
    while (fit > 1 && fixed_bytes(a.group, fit, kb, split, SUB, X == X_SCALED).all() + W4_WARPS * fit * W4_ROWS * 4 > SMEM_MAX) --fit;
    const int64_t mt = (a.M + fit - 1ll) / fit, rows = (a.M + mt - 1) / mt;
    if (rows <= 8) launch_cut<SUB, 1, X>(a, (int)mt, xtype, otype, st);
    else if (rows <= 16) launch_cut<SUB, 2, X>(a, (int)mt, xtype, otype, st);
    else if (rows <= 24) launch_cut<SUB, 3, X>(a, (int)mt, xtype, otype, st);
    else launch_cut<SUB, 4, X>(a, (int)mt, xtype, otype, st);
}

template <W4X X>
void launch_s(const W4Args &a, int xtype, int otype, cudaStream_t st) {
    const int sub = a.xgroup ? std::min(a.group, a.xgroup) : a.group;
    if (sub == 32) launch_n<32, X>(a, xtype, otype, st);
    else if (sub == 64) launch_n<64, X>(a, xtype, otype, st);
    else launch_n<128, X>(a, xtype, otype, st);
}

}  // namespace

void launch_gemv_w4(const W4Args &a, int xtype, int otype, cudaStream_t st) {
    const bool codes = xtype == TCB_I8 || xtype == TCB_E4M3;
    need(codes || xtype == TCB_BF16 || xtype == TCB_F16, "xtype is not TCB_BF16, TCB_F16, TCB_I8 or TCB_E4M3");
    need(otype == TCB_BF16 || otype == TCB_F16 || otype == TCB_F32, "otype is not TCB_BF16, TCB_F16 or TCB_F32");
    need(a.M >= 0 && a.M <= 1 << 18, "M is not in 0..2^18");
    need(w4_bytes(a.N, a.K, a.group) > 0, "N is not in 1..2^24, K not in 1..65536 or group not 32, 64 or 128");
    need(codes ? a.xgroup == 0 || a.xgroup == 32 || a.xgroup == 64 || a.xgroup == 128 : a.xgroup == 0,
         codes ? "xgroup is not 0, 32, 64 or 128" : "xgroup without 8-bit x");
    need(codes == (a.xscales != nullptr), codes ? "xscales is NULL" : "xscales without 8-bit x");
    need(a.ldx >= a.K && a.ldo >= a.N && (!a.res || a.ldr >= a.N), "a row pitch is smaller than the row");
    if (a.M == 0) return;
    need(a.x && a.w && a.out, "x, w or out is NULL");
    need(reinterpret_cast<uintptr_t>(a.w) % 16 == 0, "w is not 16-byte aligned");
    need(on(a.x, type_bytes(xtype)) && on(a.xscales, 4) && on(a.bias, 4) && on(a.res, type_bytes(otype)) && on(a.out, type_bytes(otype)),
         "a pointer is not aligned to its elements");
    need(a.out != a.x, "out is x");
    need(a.res != a.out || !a.res || a.ldr == a.ldo || a.M == 1, "res is out with another pitch");
    if (xtype == TCB_BF16) launch_s<X_BF16>(a, xtype, otype, st);
    else if (!a.xgroup) launch_s<X_F16>(a, xtype, otype, st);
    else launch_s<X_SCALED>(a, xtype, otype, st);
    check_token_launch("k_gemv_w4");
}

}  // namespace tcb
