// Host helpers of the token-stream operators: rotary frequencies and the
// packing of 4-bit weights. No CUDA call.
#include <algorithm>
#include <cmath>
#include <cstring>
#include <stdexcept>
#include <vector>

#include "token_ops.cuh"

namespace tcb {

void rope_freqs(int rot, double base, int scaling, double factor, double span, double fast, double slow, double *freq,
                float *mscale) {
    need(freq && mscale, "freq or mscale is NULL");
    need(rot >= 2 && rot % 2 == 0 && rot <= 1024, "rot is not even or not in 2..1024");
    need(std::isfinite(base) && base > 1, "base is not above 1");
    need(scaling >= TCB_ROPE_PLAIN && scaling <= TCB_ROPE_WAVES, "unknown scaling");
    if (scaling != TCB_ROPE_PLAIN) need(std::isfinite(factor) && factor >= 1, "factor is below 1");
    if (scaling == TCB_ROPE_BASE) {
        need(rot > 2, "a single pair has no base to stretch");
        base *= std::pow(factor, rot / (rot - 2.0));
        need(std::isfinite(base), "the stretched base is not finite");
    }
    if (scaling == TCB_ROPE_WAVES) {
        need(std::isfinite(span) && span > 0, "span is not positive");
        need(std::isfinite(fast) && std::isfinite(slow) && slow >= 0 && fast > slow, "fast is not above slow");
    }
    for (int i = 0; i < rot / 2; ++i) {
        double f = std::pow(base, -2.0 * i / rot);
        if (scaling == TCB_ROPE_LINEAR) f /= factor;
        if (scaling == TCB_ROPE_WAVES) {
            const double turns = span * f / (2 * M_PI);
            const double keep = std::min(1.0, std::max(0.0, (turns - slow) / (fast - slow)));
            f = f * keep + f / factor * (1 - keep);
        }
        freq[i] = f;
    }
    *mscale = scaling == TCB_ROPE_WAVES ? (float)(0.1 * std::log(factor) + 1) : 1.f;
}

int64_t w4_bytes(int N, int K, int group) {
    if (N < 1 || N > 1 << 24 || K < 1 || K > 65536 || (group != 32 && group != 64 && group != 128)) return -1;
    const int64_t tiles = ((int64_t)N + W4_ROWS - 1) / W4_ROWS, recs = (K + W4_COLS - 1) / W4_COLS;
    return tiles * recs * w4_record_bytes(group);
}

void w4_pack_codes(const int8_t *codes, const float *scales, int N, int K, int group, void *packed) {
    const int64_t bytes = w4_bytes(N, K, group);
    need(bytes > 0, "N is not in 1..2^24, K not in 1..65536 or group not 32, 64 or 128");
    need(codes && scales && packed, "codes, scales or packed is NULL");
    const int recs = (K + W4_COLS - 1) / W4_COLS, rec = w4_record_bytes(group), ng = (K + group - 1) / group;
    for (int64_t i = 0; i < (int64_t)N * K; ++i)
        if (codes[i] < -8 || codes[i] > 7) throw std::runtime_error("a code is not in -8..7");
    for (int64_t i = 0; i < (int64_t)N * ng; ++i)
        if (!std::isfinite(__bfloat162float(__float2bfloat16_rn(scales[i])))) throw std::runtime_error("a scale is not finite");
    uint8_t *out = static_cast<uint8_t *>(packed);
    std::memset(out, 0, (size_t)bytes);
    for (int64_t b = 0; b < bytes; b += rec) std::memset(out + b, 0x88, W4_CODE_BYTES);  // q = 0
    for (int n = 0; n < N; ++n) {
        const int r = n % W4_ROWS;
        uint8_t *tile = out + (int64_t)(n / W4_ROWS) * recs * rec;
        for (int k = 0; k < K; ++k) {
            const int j = k % W4_COLS, i = j / 32, t = j / 8 % 4, c = j % 8, nib = c / 2 + 4 * (c % 2);
            uint8_t &byte = tile[(int64_t)(k / W4_COLS) * rec + 512 * (r / 8) + 64 * (r % 8) + 16 * t + 4 * i + nib / 2];
            const int shift = 4 * (nib % 2), q = codes[(int64_t)n * K + k] + 8;
            byte = (uint8_t)((byte & ~(15 << shift)) | q << shift);
        }
        for (int g = 0; g < ng; ++g) {
            const int per = W4_COLS / group;
            const bf16 s = __float2bfloat16_rn(scales[(int64_t)n * ng + g]);
            std::memcpy(tile + (int64_t)(g / per) * rec + W4_CODE_BYTES + (g % per * W4_ROWS + r) * 2, &s, 2);
        }
    }
}

void w4_pack(const float *w, int N, int K, int group, void *packed) {
    need(w4_bytes(N, K, group) > 0, "N is not in 1..2^24, K not in 1..65536 or group not 32, 64 or 128");
    need(w && packed, "w or packed is NULL");
    const int ng = (K + group - 1) / group;
    std::vector<int8_t> codes((size_t)N * K);
    std::vector<float> scales((size_t)N * ng);
    for (int n = 0; n < N; ++n)
        for (int g = 0; g < ng; ++g) {
            const int64_t at = (int64_t)n * K + (int64_t)g * group;
            const int len = std::min(group, K - g * group);
            float top = 0.f;
            for (int k = 0; k < len; ++k) {
                if (!std::isfinite(w[at + k])) throw std::runtime_error("a weight is not finite");
                top = std::max(top, std::fabs(w[at + k]));
            }
            // codes are chosen for the scale as it is stored; one that is no finite bf16 has no codes
            const float s = __bfloat162float(__float2bfloat16_rn(top / 7.f));
            if (!std::isfinite(s)) throw std::runtime_error("a scale is not finite");
            scales[(size_t)n * ng + g] = s;
            for (int k = 0; k < len; ++k) {
                const float q = s > 0.f ? std::nearbyint(w[at + k] / s) : 0.f;
                codes[(size_t)(at + k)] = (int8_t)std::min(7.f, std::max(-7.f, q));
            }
        }
    w4_pack_codes(codes.data(), scales.data(), N, K, group, packed);
}

}  // namespace tcb
