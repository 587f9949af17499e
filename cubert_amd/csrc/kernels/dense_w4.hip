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
// columns to 128 with code 0 and scale 0.  Behind the codes stand the scales, of each block feature by feature, groups in order.

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
    const size_t each = kColumns / group, real = width / group;
    if (at < tiles * blocks * kTile * each) {
        const size_t block = at / (kTile * each), f = block / blocks * kTile + at / each % kTile, g = block % blocks * each + at % each;
        half_t *to = reinterpret_cast<half_t *>(packed + words);
        to[at] = f < (size_t) features && g < real ? scales[f * real + g] : (half_t) 0.f;
    }
}

// ---- the product ----------------------------------------------------------

typedef _Float16 v8f16 __attribute__((ext_vector_type(8)));
typedef _Float16 v2f16 __attribute__((ext_vector_type(2)));
typedef __bf16 v8bf16 __attribute__((ext_vector_type(8)));
typedef float v4f32 __attribute__((ext_vector_type(4)));
typedef int v4i32 __attribute__((ext_vector_type(4)));
typedef unsigned v4u32 __attribute__((ext_vector_type(4)));
typedef unsigned v2u32 __attribute__((ext_vector_type(2)));

// What 8 columns are as operands of v_mfma_*_16x16x32, of a token (from memory) and of a feature (from a word of codes), and
// how a group's products become a number: sums[i] * kUnit * scale.
template <typename X>
struct Operand;

template <>
struct Operand<half_t> {
    typedef v4f32 Raw;
    typedef v4f32 Sums;
    static constexpr float kUnit = 1.f;
    v8f16 w;
    __device__ __forceinline__ void weights(uint32_t word) {
        uint32_t pair[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t biased = (word >> (4 * j) & 0x000f000fu) | 0x64006400u;  // 1024 + 8 + code
            pair[j] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(v2f16, biased) - v2f16{(half_t) 1032.f, (half_t) 1032.f});
        }
        w = __builtin_bit_cast(v8f16, v4u32{pair[0], pair[1], pair[2], pair[3]});
    }
    __device__ __forceinline__ static Sums add(const Raw &x, const Operand &o, Sums sums) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8f16, x), o.w, sums, 0, 0, 0);
    }
};

// A code in the high half of a byte is 16 times the code; the columns of a word stand in the order 0 4 1 5 2 6 3 7.
template <>
struct Operand<int8_t> {
    typedef v2u32 Raw;
    typedef v4i32 Sums;
    static constexpr float kUnit = 1.f / 16.f;
    long w;
    __device__ __forceinline__ void weights(uint32_t word) {
        word ^= 0x88888888u;
        w = __builtin_bit_cast(long, v2u32{word << 4 & 0xf0f0f0f0u, word & 0xf0f0f0f0u});
    }
    __device__ __forceinline__ static Sums add(const Raw &x, const Operand &o, Sums sums) {
        const v2u32 turned = {__builtin_amdgcn_perm(x[1], x[0], 0x05010400u), __builtin_amdgcn_perm(x[1], x[0], 0x07030602u)};
        return __builtin_amdgcn_mfma_i32_16x16x32_i8(__builtin_bit_cast(long, turned), o.w, sums, 0, 0, 0);
    }
};

// An fp32 value is the sum of three bf16 numbers, its leading, middle and last 8 bits, and codes are bf16 numbers: every
// product is exact, anywhere in fp32's range.
template <>
struct Operand<float> {
    struct Raw {
        v4f32 part[2];
    };
    typedef v4f32 Sums;
    static constexpr float kUnit = 1.f;
    v8bf16 w;
    __device__ __forceinline__ void weights(uint32_t word) {
        const uint32_t low = word & 0x0f0f0f0fu, high = word >> 4 & 0x0f0f0f0fu;  // columns 0 4 1 5 and 2 6 3 7
        float f[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int nibble = e / 2 + 4 * (e & 1);
            f[e] = (float) ((nibble & 1 ? high : low) >> (8 * (nibble / 2)) & 0xffu) - 8.f;
        }
        w = top_halves(f);
    }
    __device__ __forceinline__ static v8bf16 top_halves(const float (&f)[8]) {
        v4u32 r;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            r[i] = __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, f[2 * i + 1]), __builtin_bit_cast(uint32_t, f[2 * i]), 0x07060302u);
        return __builtin_bit_cast(v8bf16, r);
    }
    __device__ __forceinline__ static float top(float x) {
        return __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, x) & 0xffff0000u);
    }
    struct Terms {
        v8bf16 t[3];
    };
    __device__ __forceinline__ static Terms terms(const Raw &x) {
        float a[8], b[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            a[e] = x.part[e / 4][e % 4];
            const float lead = top(a[e]);
            b[e] = a[e] == lead ? 0.f : a[e] - lead;  // (an infinity is its own first term; a NaN stays one in the second)
        }
        Terms r;
        r.t[0] = top_halves(a);
        r.t[1] = top_halves(b);
#pragma unroll
        for (int e = 0; e < 8; ++e) b[e] -= top(b[e]);
        r.t[2] = top_halves(b);
        return r;
    }
    __device__ __forceinline__ static Sums add(const Terms &x, const Operand &o, Sums sums) {
        sums = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x.t[2], o.w, sums, 0, 0, 0);
        sums = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x.t[1], o.w, sums, 0, 0, 0);
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(x.t[0], o.w, sums, 0, 0, 0);
    }
};

__device__ __forceinline__ v4f32 prepared(const v4f32 &x) { return x; }
__device__ __forceinline__ v2u32 prepared(const v2u32 &x) { return x; }
__device__ __forceinline__ Operand<float>::Terms prepared(const Operand<float>::Raw &x) { return Operand<float>::terms(x); }

// The scales of a lane's feature in a block, 128 / group of them, as the low halves of one number.
__device__ __forceinline__ unsigned long long load_scales(const half_t *scales, size_t row, int each) {
    if (each == 4) return *reinterpret_cast<const unsigned long long *>(scales + row * 4);
    if (each == 2) return *reinterpret_cast<const unsigned *>(scales + row * 2);
    return *reinterpret_cast<const unsigned short *>(scales + row);
}

// A workgroup has 16 FT features and 16 TT tokens; its W wavefronts take every W-th block of 128 columns, so that all of a weight
// row that fits is on its way at once, and their sums meet in LDS, in wavefront order.  The matrix product has tokens as rows
// and features as columns: a lane keeps one feature per 16, whose scale it multiplies each group's sums with.
template <typename X, typename T, int TT, int FT, int W>
__global__ __launch_bounds__(W * kWave) void dense_w4_kernel(int tokens, int features, int width, const X *__restrict__ x, size_t ldx,
                                                             const float *__restrict__ x_scales, const v4u32 *__restrict__ packed,
                                                             int group, const T *__restrict__ bias, int activation,
                                                             T *__restrict__ out, size_t ldo) {
    typedef Operand<X> Op;
    __shared__ float traded[W][TT * 16][17];
    const int wave = wave_in_block(), lane = threadIdx.x & (kWave - 1), col = lane & 15, quarter = lane >> 4;
    const int tile0 = blockIdx.x * FT, token0 = blockIdx.y * (16 * TT);
    const int blocks = (int) packed_blocks(width), tiles = (int) packed_tiles(features), each = kColumns / group;
    const half_t *scales = reinterpret_cast<const half_t *>(packed + (size_t) blocks * tiles * kWave);
    const X *rows[TT];
#pragma unroll
    for (int t = 0; t < TT; ++t) {
        const int token = token0 + 16 * t + col;
        rows[t] = x + (size_t) (token < tokens ? token : tokens - 1) * ldx + 8 * quarter;  // (rows past the last are not stored)
    }
    size_t first[FT];  // block of a feature tile; tiles past the last repeat it and are not stored
#pragma unroll
    for (int f = 0; f < FT; ++f) first[f] = (size_t) (tile0 + f < tiles ? tile0 + f : tiles - 1) * blocks;

    v4f32 acc[TT][FT] = {};
    v4u32 codes[FT];
    unsigned long long by[FT];
    auto bring = [&](int block) {
#pragma unroll
        for (int f = 0; f < FT; ++f) {
            codes[f] = packed[(first[f] + block) * kWave + lane];
            by[f] = load_scales(scales, (first[f] + block) * kTile + col, each);
        }
    };
    if (wave < blocks) bring(wave);
    for (int block = wave; block < blocks; block += W) {
        v4u32 now[FT];
        unsigned long long scale[FT];
#pragma unroll
        for (int f = 0; f < FT; ++f) now[f] = codes[f], scale[f] = by[f];
        typename Op::Raw piece[TT][4];
        const int steps = (width - block * kColumns) / 32;  // of this block, 4 but in the last one
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int t = 0; t < TT; ++t)  // (steps past the end read the last one again)
                piece[t][s] = *reinterpret_cast<const typename Op::Raw *>(rows[t] + block * kColumns + 32 * (s < steps ? s : steps - 1));
        if (block + W < blocks) bring(block + W);
        typename Op::Sums sums[TT][FT] = {};
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            if (s < steps) {
                Op o[FT];
#pragma unroll
                for (int f = 0; f < FT; ++f) o[f].weights(now[f][s]);
#pragma unroll
                for (int t = 0; t < TT; ++t) {
                    const auto ready = prepared(piece[t][s]);
#pragma unroll
                    for (int f = 0; f < FT; ++f) sums[t][f] = Op::add(ready, o[f], sums[t][f]);
                }
                if ((s + 1) * 32 % group == 0) {
#pragma unroll
                    for (int f = 0; f < FT; ++f) {
                        const float by_now = (float) __builtin_bit_cast(half_t, (unsigned short) (scale[f] >> (s * 32 / group * 16))) * Op::kUnit;
#pragma unroll
                        for (int t = 0; t < TT; ++t) {
#pragma unroll
                            for (int i = 0; i < 4; ++i) acc[t][f][i] = fmaf((float) sums[t][f][i], by_now, acc[t][f][i]);
                            sums[t][f] = typename Op::Sums{};
                        }
                    }
                }
            }
        }
    }
#pragma unroll
    for (int f = 0; f < FT; ++f) {
        if (f > 0) __syncthreads();
#pragma unroll
        for (int t = 0; t < TT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) traded[wave][16 * t + 4 * quarter + i][col] = acc[t][f][i];
        __syncthreads();
        for (int i = threadIdx.x; i < TT * 256; i += W * kWave) {
            const int token = token0 + i / 16, feature = (tile0 + f) * kTile + i % 16;
            if (token >= tokens || feature >= features) continue;
            float sum = 0.f;
#pragma unroll
            for (int w = 0; w < W; ++w) sum += traded[w][i / 16][i % 16];
            if (sizeof(X) == 1) sum *= x_scales[token];
            if (bias != nullptr) sum += to_f32(bias[feature]);
            if (activation != 0) sum = GeluOp<float>()(sum);
            out[token * ldo + feature] = from_f32<T>(sum);
        }
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
    const int tiles = (int) packed_tiles(features), blocks = (int) packed_blocks(in);
    const int token_tiles = tokens <= 16 ? 1 : tokens <= 32 ? 2 : 4;
    const int strips = (tokens + 16 * token_tiles - 1) / (16 * token_tiles);
    if (strips > 65535) return CUBERT_UNSUPPORTED;
    const bool wide = tiles >= 2048, deep = blocks >= 16;
    const hipStream_t s = (hipStream_t) stream;
#define RUN(TT, FT, W)                                                                                                        \
    return launch(dense_w4_kernel<X, T, TT, FT, W>, dim3((tiles + FT - 1) / FT, strips), dim3(W * kWave), s, tokens, features, in, x, \
                  ldx, x_scales, (const v4u32 *) packed, group, bias, activation, out, ldo);
    // (with 64 tokens, fewer features or wavefronts keep the sums and the rows of x in registers)
    constexpr int kWide4 = sizeof(X) == 4 ? 1 : sizeof(X) == 2 ? 2 : 4, kDeep4 = sizeof(X) == 4 ? 8 : 16;
    if (wide) {
        if (token_tiles == 1) RUN(1, 4, 8)
        if (token_tiles == 2) RUN(2, 4, 8)
        RUN(4, kWide4, 8)
    }
    if (deep) {
        if (token_tiles == 1) RUN(1, 1, 16)
        if (token_tiles == 2) RUN(2, 1, 16)
        RUN(4, 1, kDeep4)
    }
    if (token_tiles == 1) RUN(1, 1, 8)
    if (token_tiles == 2) RUN(2, 1, 8)
    RUN(4, 1, 8)
#undef RUN
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
