// Launchers of the token-stream operators (rmsnorm.cu, rope.cu, gemv_w4.cu)
// and their host helpers. All check their arguments before any CUDA call,
// throw std::runtime_error on bad ones, and enqueue on `st`.
#pragma once

#include <cstdint>

#include <cuda_runtime.h>

namespace tcb {

struct RmsArgs {
    const void *x = nullptr, *res = nullptr;
    void *sum = nullptr, *y = nullptr;
    int64_t ldx = 0, ldr = 0, lds = 0, ldy = 0, M = 0;
    const float *g = nullptr;
    float *scales = nullptr;
    float eps = 0.f;
    int D = 0, group = 0;  // group 0 = the whole row
    // set by the launcher
    float inv_d = 0.f;  // 1 / D
    int shift = 0;      // log2 group
};
void launch_rmsnorm(RmsArgs a, int dtype, int ytype, cudaStream_t st);

struct RopeArgs {
    const void *x = nullptr, *pos = nullptr;
    void *out = nullptr;
    const double *freq = nullptr;
    int64_t ldx = 0, hsx = 0, ldo = 0, hso = 0, pos_stride = 0, M = 0;
    float mscale = 1.f, sign = 1.f;  // sign -1 turns back
    int rot = 0, heads = 0, hd = 0;
};
void launch_rope(const RopeArgs &a, int dtype, int pos_type, bool interleaved, cudaStream_t st);

// Packed 4-bit weights: records of 16 rows x 128 columns.
constexpr int W4_ROWS = 16, W4_COLS = 128, W4_CODE_BYTES = W4_ROWS * W4_COLS / 2;
__host__ __device__ constexpr int w4_record_bytes(int group) { return W4_CODE_BYTES + W4_COLS / group * W4_ROWS * 2; }

struct W4Args {
    const void *x = nullptr, *w = nullptr, *res = nullptr;
    void *out = nullptr;
    const float *xscales = nullptr, *bias = nullptr;
    int64_t ldx = 0, ldr = 0, ldo = 0;
    int xgroup = 0, group = 0, relu = 0, M = 0, N = 0, K = 0;
};
void launch_gemv_w4(const W4Args &a, int xtype, int otype, cudaStream_t st);

// Host only (token_ops_host.cpp).
int64_t w4_bytes(int N, int K, int group);
void w4_pack(const float *w, int N, int K, int group, void *packed);
void w4_pack_codes(const int8_t *codes, const float *scales, int N, int K, int group, void *packed);
void rope_freqs(int rot, double base, int scaling, double factor, double span, double fast, double slow, double *freq,
                float *mscale);

}  // namespace tcb
