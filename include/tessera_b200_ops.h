/* tessera_b200_ops.h - per-kernel entry points of libtessera_b200.so, for
 * parity tests of each stage of the forward pass against the CPU oracle.
 *
 * Every pointer is device memory of the current CUDA device; every call
 * enqueues on `stream` (a cudaStream_t, NULL = legacy default stream) and
 * returns 0, or -1 with a "tcb_op_...: message" line on stderr. bf16 arrays
 * are passed as raw 16-bit storage (void *).
 */
#ifndef TESSERA_B200_OPS_H
#define TESSERA_B200_OPS_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* out[M,N] = bf16([relu](A[M,K] W[N,K]^T + bias) + residual).
 * Replaces the reference's Linear (src/tessera_cpu.cpp:215-243 make_linear,
 * src/tessera_cuda.cu:438-445 gemm). Residual: res (pitch ldr), or the DOY
 * sinusoid of pe_doy[row * pe_stride] looked up in pe_table (367 x 640 bf16,
 * src/tessera_cpu.cpp:503-509) with pe_div (320 f32) for non-table days.
 * bn = tile width (0 = automatic); variant 0 = default kernel, 1 = single-CTA
 * (M = 128 tiles), 2 = CTA pair (tcgen05 cta_group::2, M = 256 tiles). */
int tcb_op_gemm(const void *A, int lda, const void *W, const float *bias, int relu, const void *res, int ldr,
                const float *pe_doy, int pe_stride, const void *pe_table, const float *pe_div, void *out, int ldo,
                int M, int N, int K, int bn, int variant, int *status, void *stream);

/* out[M,640] = bf16(LayerNorm(y) * ln_g + ln_b), y = bf16(A[M,K] W[640,K]^T + bias + res),
 * LayerNorm eps 1e-5 over the 640 columns: the reference's out-proj + LN1 and
 * FFN2 + LN2 (src/tessera_cpu.cpp:424-428, 245-263) fused into one GEMM whose
 * epilogue exchanges row statistics across a 4-CTA cluster. */
int tcb_op_gemm_ln(const void *A, int lda, const void *W, const float *bias, const void *res, int ldr,
                   const float *ln_g, const float *ln_b, void *out, int ldo, int M, int K, int *status, void *stream);

/* Allocation-free form of tcb_op_gemm_ln, with no counterpart in the
 * reference. For callers that may not allocate device memory, such as a plugin
 * whose host framework owns the whole device-memory budget, or a hot path
 * where cudaMalloc could fail or would synchronise the device: the caller
 * passes inputs and the output only (out has pitch 640), and the intermediate
 * rows and status word live in a fixed 10 MiB static device array that every
 * GPU loading this library holds until exit. M is at most 8192 (larger M
 * returns -1 with a message). The first call on a device looks up the array's
 * address, so make it before any stream capture. Calls share the array: two
 * calls that overlap on the GPU race. Returns after the work completes. */
int tcb_op_gemm_ln_noalloc(const void *A, int lda, const void *W, const float *bias, const void *res, int ldr,
                           const float *ln_g, const float *ln_b, void *out, int M, int K, void *stream);

/* Valid-observation counts (src/tessera_encode.cpp:245-257) of pixels [p0, p0+np). */
int tcb_op_count(const uint8_t *masks, const int16_t *asc, const int16_t *desc, int64_t T2, int64_t Ta, int64_t Td,
                 int64_t N, int64_t p0, int64_t np, int32_t *n2, int32_t *n1, void *stream);

/* Gather + pad + z-score of one modality (src/tessera_encode.cpp:281-329).
 * bins[i] = rows of pixel i, off[i] = its first record (np + 1 entries);
 * rec receives (sum bins, C+1) f32 records. */
int tcb_op_gather(int modality, const uint16_t *bands, const uint8_t *masks, const uint16_t *doys,
                  const int16_t *asc, const int16_t *asc_doy, const int16_t *desc, const int16_t *desc_doy,
                  int64_t T2, int64_t Ta, int64_t Td, int64_t N, int64_t p0, int64_t np, const int32_t *bins,
                  const int64_t *off, float *rec, void *stream);

/* emb1: y = bf16(relu(bf16(rec[:, :C]) W1^T + b1)); w1t = W1^T as f32 (C x 640)
 * (src/tessera_cpu.cpp:387-404). */
int tcb_op_emb1(int C, const float *rec, int64_t M, const float *w1t, const float *b1, void *y, void *stream);

/* Self-attention per pixel segment (src/tessera_cpu.cpp:333-352,410-418).
 * off (npix+1 entries, device memory) or, when NULL, uniform segments of
 * uniform_T tokens. Each pixel's kernel follows its own length, as in the
 * tile path (tcb_attention_plan): with offsets the call reads them back,
 * lists the pixels by class, runs one launch per class and synchronizes the
 * stream before returning. Tmax must be at least every segment's length
 * (-1 otherwise) and at most 256. */
int tcb_op_attention(const void *qkv, const int64_t *off, int64_t uniform_T, int64_t npix, int Tmax, void *att,
                     void *stream);

/* LayerNorm over rows of 640 (src/tessera_cpu.cpp:245-263); g/b may be NULL. */
int tcb_op_layernorm640(const void *x, int64_t M, const float *g, const float *b, void *y, void *stream);

/* Attention pooling (src/tessera_cpu.cpp:434-455) into fused[:, col0:col0+640]. */
int tcb_op_pool(const void *x, const int64_t *off, int64_t uniform_T, int64_t npix, const float *q, float qb,
                void *fused, int col0, void *stream);

/* Head LayerNorm(2560) + ReLU in place (src/tessera_cpu.cpp:568-571). */
int tcb_op_ln_relu2560(void *r, int64_t P, const float *g, const float *b, void *stream);

/* Final LayerNorm(128, no affine) -> bf16 -> f32 out, or int8 codes + scales
 * (src/tessera_cpu.cpp:573-575, src/tessera_encode.cpp:344-361). */
int tcb_op_out128(const void *r2, int64_t P, const uint8_t *empty, float *out, int8_t *codes, float *scales,
                  void *stream);

/* ---- token-stream operators of students served in few bits ----------------
 * The front of a pre-norm block: RMS norm with the residual's addition and an
 * 8-bit output, rotary positions (by day of year or by index) and the Linear
 * of a few tokens with 4-bit weights. No reference counterpart: the Large
 * student has LayerNorm, an additive day-of-year sinusoid and bf16 weights.
 * They compose with tcb_op_attention, tcb_op_pool and tcb_op_gemm on the same
 * token rows. None allocates, synchronises or keeps state between calls, so
 * each can be captured into a CUDA graph and calls on different streams are
 * independent. Zero rows (M = 0) are a no-op returning 0. Pointers need the
 * alignment of their elements only; rows that start at 16-byte boundaries, or
 * equally far behind them in every tensor, are the faster ones. */

/* Element types of the operators below. */
enum {
    TCB_BF16 = 0,
    TCB_F16 = 1,
    TCB_F32 = 2,
    TCB_I8 = 3,   /* int8 codes in -127..127, with f32 scales */
    TCB_E4M3 = 4, /* 8-bit floats (4-bit exponent, largest 448), with f32 scales */
    TCB_I32 = 5,  /* positions only */
    TCB_I64 = 6   /* positions only */
};

/* Root-mean-square norm of M rows of D columns (1 <= D <= 16384):
 *   h = x, or x + res rounded to `dtype` when res is given;
 *   v = h / sqrt(mean(h^2) + eps) * g       (g: D f32 values, NULL = ones).
 * x, res, sum and y have row pitches of ldx, ldr, lds and ldy elements (>= D).
 * dtype is TCB_BF16, TCB_F16 or TCB_F32. h is written to sum when sum is not
 * NULL (needs res). ytype is dtype (y = v rounded once; scales NULL, group 0),
 * or TCB_I8 / TCB_E4M3: per row and group of columns (group 0 = the whole row,
 * else 32, 64 or 128; the last group may be short)
 *   s = max(max|v|, 1e-12) / Q,  y = round(v / s),  Q = 127 / 448,
 * with scales[row * ceil(D / group) + column / group] = s, the rule of
 * tcb_op_out128. Statistics are f32 and do not overflow for finite h. A NaN
 * makes its whole row NaN; an infinity makes its own v NaN and the row's other
 * v zero. A group with a NaN gets the scale NaN, int8 codes 0, e4m3 codes NaN.
 * A row's result does not depend on M or on the other rows. Its last bits depend
 * on how far its address in each tensor is behind a boundary of 8 elements, since
 * that sets the order of the sum; a pitch that is a multiple of 8 gives all rows
 * one order. h g is formed before the division, in f32: |h g| below 2^128.
 * sum may be x or res itself, and y of dtype may be x or sum (same pitch);
 * other overlaps are not allowed. */
int tcb_op_rmsnorm(const void *x, int64_t ldx, const void *res, int64_t ldr, void *sum, int64_t lds, const float *g,
                   float eps, int dtype, void *y, int64_t ldy, int ytype, float *scales, int group, int64_t M, int D,
                   void *stream);

/* Rotary positions: turns the first `rot` columns (even, 2..hd) of each of
 * `heads` heads of hd columns (hd <= 1024) of M token rows by the row's position,
 *   (a, b) -> mscale * (a cos t - b sin t, a sin t + b cos t),  t = pos * freq[i],
 * where pair i is columns (2i, 2i + 1) with interleaved != 0 and columns
 * (i, i + rot/2) otherwise. Columns rot..hd-1 are copied. inverse != 0 turns by
 * -t, which is also the gradient of the turn. Element (row, head, column) of x
 * is x[row * ldx + head * hsx + column], of out likewise with ldo and hso, so
 * q and k of a packed qkv row (or grouped k heads behind the q heads) are one
 * call. hsx, hso >= hd; rows and heads must not overlap in out. dtype is TCB_BF16,
 * TCB_F16 or TCB_F32, for both. out may be x with the same strides; other
 * overlaps are not allowed. Row r's position is pos[r * pos_stride]
 * (pos_stride >= 0; 0 = one position for all), of type TCB_F32 (the day of year
 * of a token record), TCB_I32 or TCB_I64. freq: rot/2 f64 radians per position
 * (tcb_rope_freqs). Angles are reduced in f64, so positions far beyond 2^24
 * keep their phase. */
int tcb_op_rope(const void *x, int64_t ldx, int64_t hsx, int dtype, const void *pos, int64_t pos_stride, int pos_type,
                const double *freq, float mscale, int rot, int interleaved, int inverse, void *out, int64_t ldo,
                int64_t hso, int64_t M, int heads, int hd, void *stream);

/* Ways of stretching rotary positions over a longer span than a model was
 * trained on. */
enum {
    TCB_ROPE_PLAIN = 0,  /* freq[i] = base^(-2i/rot) */
    TCB_ROPE_LINEAR = 1, /* positions divided by factor */
    TCB_ROPE_BASE = 2,   /* base multiplied by factor^(rot/(rot-2)): the slowest pair slows by factor, the fastest stays */
    TCB_ROPE_WAVES = 3   /* by wavelength: pairs that turn more than `fast` times over the trained span stay, those
                            that turn less than `slow` times are divided by factor, a linear ramp between;
                            mscale = 0.1 ln(factor) + 1 */
};

/* Fills freq[0 .. rot/2) (host memory; copy it to the device for tcb_op_rope)
 * and *mscale (1 except for TCB_ROPE_WAVES). Host only, no CUDA call. span,
 * fast and slow are read for TCB_ROPE_WAVES only (usual: 32 and 1). Returns
 * 0, or -1 on bad arguments. */
int tcb_rope_freqs(int rot, double base, int scaling, double factor, double span, double fast, double slow, double *freq,
                   float *mscale);

/* out[M,N] = [relu](x[M,K] W[N,K]^T + bias) + res for a few rows, with W in 4
 * bits: W[n,k] = q[n,k] * s[n, k / group], q in -8..7, s bf16, in the layout of
 * tcb_w4_pack (device memory, 16-byte aligned; group 32, 64 or 128). xtype is
 * TCB_BF16, TCB_F16, or TCB_I8 / TCB_E4M3 with xscales[m, k / xgroup] (f32,
 * contiguous rows of ceil(K / xgroup); xgroup 0 = one per row, else 32, 64 or
 * 128): the output of tcb_op_rmsnorm. bias: N f32 or NULL. res (pitch ldr) has
 * the output's type and may be out itself. otype is TCB_BF16, TCB_F16 or
 * TCB_F32. Products are exact and summed in f32 in an order that depends on
 * xtype, M, N, K, group, xgroup and the GPU's SMs only; the output is rounded
 * once. A code of 0 adds 0, whatever finite value it meets. The
 * weights are read once per 32 rows or so: tcb_op_gemm on bf16 weights is the
 * faster call from some 64 rows on at 8,192 x 8,192 weights, from 128 at 2,560 x
 * 1,280 and 1,920 x 640, from 192 at 2,560 x 2,560. M <= 2^18, N <= 2^24, K <= 65536. */
int tcb_op_gemv_w4(const void *x, int64_t ldx, int xtype, const float *xscales, int xgroup, const void *w, int group,
                   const float *bias, int relu, const void *res, int64_t ldr, void *out, int64_t ldo, int otype, int M,
                   int N, int K, void *stream);

/* 4-bit weights (host only, no CUDA call). tcb_w4_bytes: size of the packed
 * form of an N x K matrix, or -1 on bad arguments. tcb_w4_pack quantises f32
 * weights (row-major, finite): s = bf16(max|w| / 7) per row and group,
 * q = round(w / s). tcb_w4_pack_codes packs another quantiser's codes (N x K
 * int8 in -8..7) and scales (N x ceil(K / group) f32, rounded to bf16, finite).
 *
 * Layout: the matrix padded with zeros to multiples of 16 rows and 128 columns,
 * as records of 16 rows x 128 columns, row tile by row tile, each tile's
 * records in column order. A record is 1024 bytes of codes (q + 8) and its
 * 128/group x 16 bf16 scales, group by group. The codes of row r of the record
 * start at byte 512 * (r / 8) + 64 * (r % 8): four lanes of 16 bytes, lane t
 * with four little-endian 32-bit words, word i holding columns 32 i + 8 t + c,
 * c = 0..7, in nibble c / 2 + 4 * (c % 2). Both return 0, or -1. */
int64_t tcb_w4_bytes(int N, int K, int group);
int tcb_w4_pack(const float *w, int N, int K, int group, void *packed);
int tcb_w4_pack_codes(const int8_t *codes, const float *scales, int N, int K, int group, void *packed);

/* Attention kernel classes of a chunk's pixels (host only, no CUDA call; no
 * reference counterpart: the reference has one attention path). off[0..npix]
 * are the segment offsets. list receives the pixels with a non-empty series,
 * class by class in pixel order: class 0 the mma.sync kernel for T <= 48,
 * class 1 the tcgen05 kernel for 48 < T <= 128, class 2 the mma.sync kernel
 * for T > 128 (TC_ATTN_TC=0 / 2 move every T <= 128 to class 0 / 1).
 * n[3] receives the pixels per class and tmax[3] the longest series per
 * class. The class of a pixel depends on its own length only. Returns 0, or
 * -1 on bad arguments (null pointers, negative npix, decreasing offsets). */
int tcb_attention_plan(const int64_t *off, int64_t npix, int32_t *list, int64_t *n, int32_t *tmax);

/* Failure-detection probe (no reference counterpart: the reference has no
 * device-side waits). One kernel waits limit_us on an mbarrier that nothing
 * signals, through the same bounded wait every pipeline kernel uses, then
 * writes its error code (6) to *status and returns; the context stays usable. */
int tcb_op_wait_probe(int64_t limit_us, int *status, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* TESSERA_B200_OPS_H */
