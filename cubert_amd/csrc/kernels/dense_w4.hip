// Dense layers of few tokens on weights of 4 bits:
//
//     out[t, f] = act(sum_g scale[f, g] * (sum of code[f, k] x[t, k] over the columns k of group g) + bias[f])
//
// with codes of -8..7 and one fp16 scale for 32, 64 or 128 columns of a weight row.  A group's products are summed before
// its scale is applied, so that no weight is ever rounded.
//
// cubert_w4_pack lays the weights out once in the order the kernel takes them: 16 features and 128 columns are 1 KB, 16
// bytes to a lane of a wavefront.  Lane l has feature l % 16 and, in its word s, the 8 columns 32 s + 8 (l / 16) + e: the
// even e in the low four nibbles and the odd ones in the high four, as code + 8, so that
// ((word >> 4 j) & 0x000f000f) | 0x64006400 is a pair of the fp16 numbers 1032 + code.  Features are filled up to 16 and
// columns to 128 with code 0 and scale 0.  Behind the codes stand the scales, per 16 features and group the 16 of them.

#include "activations.h"
#include "cubert_kernels.h"
#include "device_common.h"

namespace cubert {
namespace {

constexpr int kTile = 16;      // features of a packed block
constexpr int kColumns = 128;  // columns of a packed block
constexpr int kBlockBytes = kTile * kColumns / 2;

bool good_group(int group) { return group == 32 || group == 64 || group == 128; }

__host__ __device__ inline size_t packed_blocks(int width) { return (width + kColumns - 1) / kColumns; }
__host__ __device__ inline size_t packed_tiles(int features) { return (features + kTile - 1) / kTile; }

// ---- preparing weights (once per model) -----------------------------------

// One lane per group of a row: the largest weight becomes code 7 or -7.
template <typename T>
__global__ void w4_quantize_kernel(const T *__restrict__ w, size_t groups, int group, uint8_t *__restrict__ codes,
                                   half_t *__restrict__ scales, int *__restrict__ overflow) {
    const size_t at = (size_t) blockIdx.x * blockDim.x + threadIdx.x;
    if (at >= groups) return;
    w += at * group;
    float top = 0.f;
    bool finite = true;
    for (int i = 0; i < group; ++i) {
        const float x = fabsf(to_f32(w[i]));
        finite = finite && x < INFINITY;
        top = fmaxf(top, x);
    }
    const half_t scale = (half_t) (top / 7.f);
    const bool usable = finite && (float) scale < INFINITY;
    if (!usable && overflow != nullptr) *overflow = 1;
    scales[at] = usable ? scale : (half_t) NAN;
    const float by = (float) scale;
    for (int i = 0; i < group; i += 2) {
        int c[2];
        for (int j = 0; j < 2; ++j)
            c[j] = usable && by > 0.f ? (int) fminf(fmaxf(rintf(to_f32(w[i + j]) / by), -8.f), 7.f) : 0;
        codes[(at * group + i) / 2] = (uint8_t) ((c[0] & 15) | (c[1] & 15) << 4);
    }
}

__global__ void w4_pack_kernel(const uint8_t *__restrict__ codes, const half_t *__restrict__ scales, int features, int width,
                               int group, uint32_t *__restrict__ packed) {
    const size_t blocks = packed_blocks(width), tiles = packed_tiles(features);
    const size_t words = blocks * tiles * (kBlockBytes / 4);
    const size_t at = (size_t) blockIdx.x * blockDim.x + threadIdx.x;
    if (at < words) {
        const int s = at & 3, lane = (int) (at >> 2) & 63;
        const size_t block = at / (kBlockBytes / 4) % blocks, tile = at / (kBlockBytes / 4) / blocks;
        const size_t f = tile * kTile + lane % 16;
        uint32_t word = 0x88888888u;
        for (int e = 0; e < 8; ++e) {
            const size_t k = block * kColumns + 32 * s + 8 * (lane / 16) + e;
            if (f < (size_t) features && k < (size_t) width) {
                const uint32_t c = codes[(f * width + k) / 2] >> (4 * (k & 1)) & 15u;  // two's complement
                const int nibble = e / 2 + 4 * (e & 1);
                word ^= c << (4 * nibble);  // c ^ 8 = c + 8 in four bits
            }
        }
        packed[at] = word;
    }
    const size_t groups = blocks * (kColumns / group), real = width / group;
    if (at < tiles * groups * kTile) {
        const size_t f = at / (groups * kTile) * kTile + at % kTile, g = at / kTile % groups;
        half_t *to = reinterpret_cast<half_t *>(packed + words);
        to[at] = f < (size_t) features && g < real ? scales[f * real + g] : (half_t) 0.f;
    }
}

// ---- the product ----------------------------------------------------------

// One wavefront per feature and token: a lane takes every 64th run of 8 columns.
template <typename X, typename T>
__global__ __launch_bounds__(kBlock) void dense_w4_kernel(int tokens, int features, int width, const X *__restrict__ x, int ldx,
                                                          const float *__restrict__ x_scales, const uint32_t *__restrict__ packed,
                                                          int group, const T *__restrict__ bias, int activation,
                                                          T *__restrict__ out, int ldo) {
    const size_t at = (size_t) blockIdx.x * (kBlock / kWave) + wave_in_block();
    if (at >= (size_t) tokens * features) return;
    const int lane = threadIdx.x & (kWave - 1);
    const int t = (int) (at / features), f = (int) (at % features);
    const size_t blocks = packed_blocks(width), tiles = packed_tiles(features), groups = blocks * (kColumns / group);
    const half_t *scales = reinterpret_cast<const half_t *>(packed + blocks * tiles * (kBlockBytes / 4));
    x += (size_t) t * ldx;
    float sum = 0.f;
    for (int k = 8 * lane; k < width; k += 8 * kWave) {
        const size_t block = (f / kTile) * blocks + k / kColumns;
        const int s = k % kColumns / 32, g = k % 32 / 8;
        const uint32_t word = packed[block * (kBlockBytes / 4) + (size_t) (16 * g + f % kTile) * 4 + s];
        float part = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) part = fmaf((float) ((int) (word >> (4 * (e / 2 + 4 * (e & 1))) & 15u) - 8), (float) x[k + e], part);
        sum = fmaf((float) scales[((f / kTile) * groups + k / group) * kTile + f % kTile], part, sum);
    }
    sum = wave_sum(sum);
    if (lane == 0) {
        if (x_scales != nullptr) sum *= x_scales[t];
        if (bias != nullptr) sum += to_f32(bias[f]);
        if (activation != 0) sum = GeluOp<float>()(sum);
        out[(size_t) t * ldo + f] = from_f32<T>(sum);
    }
}

template <typename X, typename T>
int dense_w4(void *stream, int tokens, int features, int in, const X *x, int ldx, const float *x_scales, const void *packed, int group,
             const T *bias, int activation, T *out, int ldo) {
    if (tokens < 0 || features < 1 || in < 1 || ldx < in || ldo < features || (activation != 0 && activation != 1))
        return CUBERT_BAD_ARGUMENT;
    if (tokens == 0) return 0;
    if (x == nullptr || packed == nullptr || out == nullptr || (sizeof(X) == 1 && x_scales == nullptr)) return CUBERT_BAD_ARGUMENT;
    if (!good_group(group) || in % group != 0 || !is_aligned(x, 16) || (size_t) ldx * sizeof(X) % 16 != 0 || !is_aligned(packed, 16))
        return CUBERT_UNSUPPORTED;
    const size_t waves = (size_t) tokens * features;
    if (waves >= (size_t) 1 << 26) return CUBERT_UNSUPPORTED;  // a launch holds less than 2^32 threads
    return launch(dense_w4_kernel<X, T>, dim3((unsigned) ((waves + 3) / 4)), dim3(kBlock), (hipStream_t) stream, tokens, features, in,
                  x, ldx, x_scales, (const uint32_t *) packed, group, bias, activation, out, ldo);
}

template <typename T>
int w4_quantize(const T *w, int features, int in, int group, uint8_t *codes, cubert_half *scales, int *overflow, void *stream) {
    if (features < 1 || in < 1 || w == nullptr || codes == nullptr || scales == nullptr) return CUBERT_BAD_ARGUMENT;
    if (!good_group(group) || in % group != 0) return CUBERT_UNSUPPORTED;
    const size_t groups = (size_t) features * (in / group);
    if (groups >= (size_t) 1 << 31) return CUBERT_UNSUPPORTED;
    return launch(w4_quantize_kernel<T>, dim3((unsigned) ((groups + kBlock - 1) / kBlock)), dim3(kBlock), (hipStream_t) stream, w,
                  groups, group, codes, (half_t *) scales, overflow);
}

}  // namespace
}  // namespace cubert

using cubert::half_t;

extern "C" {

int cubert_w4_quantize_f32(const float *w, int features, int in, int group, uint8_t *codes, cubert_half *scales, int *overflow,
                           void *stream) {
    return cubert::w4_quantize<float>(w, features, in, group, codes, scales, overflow, stream);
}

int cubert_w4_quantize_f16(const cubert_half *w, int features, int in, int group, uint8_t *codes, cubert_half *scales, int *overflow,
                           void *stream) {
    return cubert::w4_quantize<half_t>((const half_t *) w, features, in, group, codes, scales, overflow, stream);
}

size_t cubert_w4_packed_bytes(int features, int in, int group) {
    if (features < 1 || in < 1 || !cubert::good_group(group) || in % group != 0) return 0;
    const size_t blocks = cubert::packed_blocks(in) * cubert::packed_tiles(features);
    return blocks * cubert::kBlockBytes + blocks * (cubert::kColumns / group) * cubert::kTile * sizeof(half_t);
}

int cubert_w4_pack(const uint8_t *codes, const cubert_half *scales, int features, int in, int group, void *packed, void *stream) {
    if (features < 1 || in < 1 || codes == nullptr || scales == nullptr || packed == nullptr) return CUBERT_BAD_ARGUMENT;
    if (!cubert::good_group(group) || in % group != 0 || !cubert::is_aligned(packed, 16)) return CUBERT_UNSUPPORTED;
    const size_t words = cubert::packed_blocks(in) * cubert::packed_tiles(features) * (cubert::kBlockBytes / 4);
    if (words >= (size_t) 1 << 31) return CUBERT_UNSUPPORTED;
    return cubert::launch(cubert::w4_pack_kernel, dim3((unsigned) ((words + cubert::kBlock - 1) / cubert::kBlock)), dim3(cubert::kBlock),
                          (hipStream_t) stream, codes, (const half_t *) scales, features, in, group, (uint32_t *) packed);
}

int cubert_dense_w4_f32(void *stream, int tokens, int features, int in, const float *x, int ldx, const void *packed, int group,
                        const float *bias, int activation, float *out, int ldo) {
    return cubert::dense_w4<float, float>(stream, tokens, features, in, x, ldx, nullptr, packed, group, bias, activation, out, ldo);
}

int cubert_dense_w4_f16(void *stream, int tokens, int features, int in, const cubert_half *x, int ldx, const void *packed, int group,
                        const cubert_half *bias, int activation, cubert_half *out, int ldo) {
    return cubert::dense_w4<half_t, half_t>(stream, tokens, features, in, (const half_t *) x, ldx, nullptr, packed, group,
                                            (const half_t *) bias, activation, (half_t *) out, ldo);
}

int cubert_dense_w4_i8_f32(void *stream, int tokens, int features, int in, const int8_t *x, int ldx, const float *x_scales,
                           const void *packed, int group, const float *bias, int activation, float *out, int ldo) {
    return cubert::dense_w4<int8_t, float>(stream, tokens, features, in, x, ldx, x_scales, packed, group, bias, activation, out, ldo);
}

int cubert_dense_w4_i8_f16(void *stream, int tokens, int features, int in, const int8_t *x, int ldx, const float *x_scales,
                           const void *packed, int group, const cubert_half *bias, int activation, cubert_half *out, int ldo) {
    return cubert::dense_w4<int8_t, half_t>(stream, tokens, features, in, x, ldx, x_scales, packed, group, (const half_t *) bias,
                                            activation, (half_t *) out, ldo);
}

}  // extern "C"
