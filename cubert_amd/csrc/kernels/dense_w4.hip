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
// (word & 0x000f000f) | 0x64006400 is a pair of the fp16 numbers 1032 + code.  Features are filled up to 16 and
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

__host__ __device__ inline size_t packed_blocks(int width) { return ((size_t) width + kColumns - 1) / kColumns; }
__host__ __device__ inline size_t packed_tiles(int features) { return ((size_t) features + kTile - 1) / kTile; }

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

// (x & mask) | bits in one instruction, which the compiler makes two of where both are constants.
__device__ __forceinline__ uint32_t and_or(uint32_t x, uint32_t mask, uint32_t bits) {
    uint32_t r;
    asm("v_and_or_b32 %0, %1, %2, %3" : "=v"(r) : "v"(x), "s"(mask), "v"(bits));
    return r;
}

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
        for (int j = 0; j < 4; j += 2) {
            const uint32_t part = j == 0 ? word : word >> 8;
            const uint32_t low = and_or(part, 0x000f000fu, 0x64006400u), high = and_or(part, 0x00f000f0u, 0x64006400u);
            // 1024 + (8 + code), and 1024 + 16 (8 + code): both exact
            pair[j] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(v2f16, low) - v2f16{(half_t) 1032.f, (half_t) 1032.f});
            pair[j + 1] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(__builtin_bit_cast(v2f16, high), v2f16{(half_t) 0.0625f, (half_t) 0.0625f},
                                                                                 v2f16{(half_t) -72.f, (half_t) -72.f}));
        }
        w = __builtin_bit_cast(v8f16, v4u32{pair[0], pair[1], pair[2], pair[3]});
    }
    __device__ __forceinline__ static Raw ready(const Raw &x) { return x; }
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
    __device__ __forceinline__ static long ready(const Raw &x) {
        return __builtin_bit_cast(long, v2u32{__builtin_amdgcn_perm(x[1], x[0], 0x05010400u), __builtin_amdgcn_perm(x[1], x[0], 0x07030602u)});
    }
    __device__ __forceinline__ static Sums add(long x, const Operand &o, Sums sums) {
        return __builtin_amdgcn_mfma_i32_16x16x32_i8(x, o.w, sums, 0, 0, 0);
    }
};

// An fp32 value is the sum of three bf16 numbers, its leading, middle and last 8 bits, and codes are bf16 numbers: every
// product is exact, anywhere in fp32's range.  (fp32 matrix instructions, a sixteenth as fast: 16 tokens, 4096 x 16384, 29 us
// against 19.)
template <>
struct Operand<float> {
    struct Raw {
        v4f32 part[2];
    };
    struct Ready {
        v8bf16 term[3];
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
        w = leading(f);
    }
    __device__ __forceinline__ static v8bf16 leading(const float (&f)[8]) {
        v4u32 r;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            r[i] = __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, f[2 * i + 1]), __builtin_bit_cast(uint32_t, f[2 * i]), 0x07060302u);
        return __builtin_bit_cast(v8bf16, r);
    }
    __device__ __forceinline__ static float lead(float x) {
        return __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, x) & 0xffff0000u);
    }
    __device__ __forceinline__ static Ready ready(const Raw &x) {
        float a[8];
        Ready r;
#pragma unroll
        for (int e = 0; e < 8; ++e) a[e] = x.part[e / 4][e % 4];
        r.term[0] = leading(a);
#pragma unroll
        for (int e = 0; e < 8; ++e) {  // (an infinity is its own first term; a NaN stays one in the second)
            const float top = lead(a[e]);
            a[e] = a[e] == top ? 0.f : a[e] - top;
        }
        r.term[1] = leading(a);
#pragma unroll
        for (int e = 0; e < 8; ++e) a[e] -= lead(a[e]);
        r.term[2] = leading(a);
        return r;
    }
    __device__ __forceinline__ static Sums add(const Ready &x, const Operand &o, Sums sums) {
#pragma unroll
        for (int n = 2; n >= 0; --n) sums = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x.term[n], o.w, sums, 0, 0, 0);
        return sums;
    }
};

// The scales of a lane's feature in a block: 128 / group = EACH halves.
template <int EACH>
struct Scales {
    Vec<half_t, EACH> v;

    __device__ __forceinline__ void load(const half_t *scales, size_t row) { v = load_vec<half_t, EACH>(scales + row * EACH); }
};

template <typename X, typename T>
struct DenseArgs {
    int tokens, features, steps;  // steps of 32 columns
    int blocks, tiles, strips;    // of 128 columns, 16 features, 16 tokens
    const X *x;
    size_t ldx;
    const float *x_scales;
    const v4u32 *packed;
    const half_t *scales;
    const T *bias;
    int activation;
    T *out;
    size_t ldo;
};

// The products of 16 tokens with 16 FT features over one block, whose operands are there.  The matrix product has tokens as rows and
// features as columns: a lane keeps one feature per 16, whose scale it multiplies each group's sums with.
template <typename X, int FT, int EACH>
__device__ __forceinline__ void multiply_block(v4f32 (&acc)[FT], const typename Operand<X>::Raw (&piece)[4], const v4u32 (&codes)[FT],
                                               const Scales<EACH> (&by)[FT]) {
    typedef Operand<X> Op;
    typename Op::Sums sums[FT];
#pragma unroll
    for (int s = 0; s < 4; ++s) {
        const auto x = Op::ready(piece[s]);
#pragma unroll
        for (int f = 0; f < FT; ++f) {
            Op o;
            o.weights(codes[f][s]);
            sums[f] = Op::add(x, o, s % (4 / EACH) == 0 ? typename Op::Sums{} : sums[f]);
        }
        if ((s + 1) % (4 / EACH) == 0) {  // the end of a group
#pragma unroll
            for (int f = 0; f < FT; ++f) {
                const float scale = (float) by[f].v.v[s * EACH / 4] * Op::kUnit;
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[f][i] = fmaf((float) sums[f][i], scale, acc[f][i]);
            }
        }
    }
}

// A workgroup has 16 FT features and 16 tokens; its W wavefronts take every W-th block of 128 columns, and their sums meet in LDS, in
// wavefront order.  The operands come straight into registers, where the matrix instructions take them: weights are used once per 16
// tokens, and so many wavefronts fit a unit that the others cover one's wait.  (Operands of the next block in registers of their own:
// 16 x 8192 x 32768 33 and 31 us, 64 x 4096 x 4096 10 and 11.)
// Few tokens on large layers are bound by reading the weights: 16 rows of 8 bits, 8192 x 32768, 140 MB in 29 us, 4.8 TB/s; 1 token in
// fp16 29.6 us.  Small layers by latency: 1 x 1024 x 4096 3.2 us.  More tokens by the loads of x, which every 64 features repeat in 16
// rows of 64 bytes: 64 x 4096 x 16384 in fp16 27 us, where the weights take 6.7; codes unpacked once for 32 or 64 tokens left that
// as it was (26 and 27 us).
template <typename X, typename T, int EACH, int FT, int W>
__global__ __launch_bounds__(W * kWave) void dense_w4_kernel(DenseArgs<X, T> a) {
    typedef typename Operand<X>::Raw Raw;
    __shared__ float traded[FT][W][kTile][17];
    const int wave = wave_in_block(), lane = threadIdx.x & (kWave - 1);
    // Workgroups are handed to the eight dies in turn: those of one feature tile, 16 tokens each, follow each other on one die,
    // whose cache then has the weights.
    const int on_die = blockIdx.x / 8, tile0 = (on_die / a.strips * 8 + blockIdx.x % 8) * FT, token0 = on_die % a.strips * kTile;
    if (tile0 >= a.tiles) return;
    const int token = token0 + (lane & 15);  // rows past the last repeat it and are not stored
    const X *row = a.x + (size_t) (token < a.tokens ? token : a.tokens - 1) * a.ldx + 8 * (lane >> 4);
    size_t first[FT];  // block of a feature tile; tiles past the last repeat it and are not stored
#pragma unroll
    for (int f = 0; f < FT; ++f) first[f] = (size_t) (tile0 + f < a.tiles ? tile0 + f : a.tiles - 1) * a.blocks;
    v4f32 acc[FT] = {};
    v4u32 codes[FT];
    Scales<EACH> by[FT];
    Raw piece[4];
    auto bring = [&](int block) {
#pragma unroll
        for (int f = 0; f < FT; ++f) {
            codes[f] = a.packed[(first[f] + block) * kWave + lane];
            by[f].load(a.scales, (first[f] + block) * kTile + (lane & 15));
        }
        const X *at = row + (size_t) block * kColumns;
        if (a.steps - 4 * block >= 4) {
#pragma unroll
            for (int s = 0; s < 4; ++s) piece[s] = *reinterpret_cast<const Raw *>(at + 32 * s);
        } else {  // past the end of the rows there is nothing: zeros, as the codes there are
#pragma unroll
            for (int s = 0; s < 4; ++s) piece[s] = 4 * block + s < a.steps ? *reinterpret_cast<const Raw *>(at + 32 * s) : Raw{};
        }
    };
    if (wave < a.blocks) bring(wave);
    for (int block = wave; block < a.blocks; block += W) {
        multiply_block<X, FT, EACH>(acc, piece, codes, by);
        if (block + W < a.blocks) bring(block + W);
    }
#pragma unroll
    for (int f = 0; f < FT; ++f)
#pragma unroll
        for (int i = 0; i < 4; ++i) traded[f][wave][4 * (lane >> 4) + i][lane & 15] = acc[f][i];
    __syncthreads();
    constexpr int kQuarter = W / 4;  // four threads to a result
#pragma unroll
    for (int i = threadIdx.x; i < FT * 1024; i += W * kWave) {
        const int m = i / (FT * 64), n = i / 4 % (FT * 16), part = i % 4;
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < kQuarter; ++w) sum += traded[n / 16][part * kQuarter + w][m][n % 16];
        sum += dpp_move<kDppQuadXor1>(sum);
        sum += dpp_move<kDppQuadXor2>(sum);
        const int to = token0 + m, feature = tile0 * kTile + n;
        if (part == 0 && to < a.tokens && feature < a.features) {
            if (sizeof(X) == 1) sum *= a.x_scales[to];
            if (a.bias != nullptr) sum += to_f32(a.bias[feature]);
            if (a.activation != 0) sum = GeluOp<float>()(sum);
            a.out[to * a.ldo + feature] = from_f32<T>(sum);
        }
    }
}

// How many features a workgroup has: more make less of reading and taking apart x again, fewer fill the card.  Microseconds with 16 /
// 32 / 64 features: 16 fp16 tokens, 8192 x 32768 (2048 units of 16 features and 16 tokens) 65 / 40 / 34; 33 tokens, 4096 x 4096 (768)
// 12 / 12 / 8.6; 1 token, 4096 x 16384 (1024) 10.8 / 9.5 / 10.1, 4096 x 1024 (64) 4.4 / 5.1 / 7.3.  Up to 8 tokens, 16 features and sixteen
// wavefronts / 32 and eight: 7 tokens, 4096 x 4100 (257) 7.6 / 6.3, 4096 x 5120 (320) 8.2 / 6.3, in 8 bits 7.6 / 6.0, in fp32 15 / 12, 4096 x
// 8192 (512) 9.0 / 7.8; 1 token, 4096 x 4100 5.3 / 5.5, 1024 x 8192 3.7 / 3.8.
template <typename X, typename T, int EACH>
int run_dense_w4(const DenseArgs<X, T> &a, hipStream_t s) {
    const long long units = (long long) a.tiles * a.strips;
    auto groups = [&](int ft) { return ((long long) a.tiles + 8 * ft - 1) / (8 * ft) * 8 * a.strips; };
    auto grid = [&](int ft) { return dim3((unsigned) groups(ft)); };
    if (units > 1024 && groups(4) * 8 * kWave >= 1ll << 32) return CUBERT_UNSUPPORTED;  // (what a launch holds)
    if (units > 1024 || (units > 512 && a.tokens > 8)) return launch(dense_w4_kernel<X, T, EACH, 4, 8>, grid(4), dim3(8 * kWave), s, a);
    if (units > 256) return launch(dense_w4_kernel<X, T, EACH, 2, 8>, grid(2), dim3(8 * kWave), s, a);
    // (sixteen wavefronts / eight: 1 token, 4096 x 1024 4.0 / 4.4 us, 8192 x 4096 7.0 / 8.5; 8 tokens, 8192 x 4096 8.8 / 9.2; 16 tokens, 4096 x
    // 4096 7.2 / 6.8)
    if ((units <= 128 || (units <= 256 && a.tokens <= 8)) && a.blocks > 8) return launch(dense_w4_kernel<X, T, EACH, 1, 16>, grid(1), dim3(16 * kWave), s, a);
    return launch(dense_w4_kernel<X, T, EACH, 1, 8>, grid(1), dim3(8 * kWave), s, a);
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
    DenseArgs<X, T> a;
    a.tokens = tokens, a.features = features, a.steps = in / 32;
    a.blocks = (int) packed_blocks(in), a.tiles = (int) packed_tiles(features), a.strips = (int) (((long long) tokens + kTile - 1) / kTile);
    a.x = x, a.ldx = ldx, a.x_scales = x_scales;
    a.packed = (const v4u32 *) packed, a.scales = reinterpret_cast<const half_t *>(a.packed + (size_t) a.blocks * a.tiles * kWave);
    a.bias = bias, a.activation = activation, a.out = out, a.ldo = ldo;
    const hipStream_t s = (hipStream_t) stream;
    return group == 128 ? run_dense_w4<X, T, 1>(a, s) : group == 64 ? run_dense_w4<X, T, 2>(a, s) : run_dense_w4<X, T, 4>(a, s);
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
    if (blocks * (cubert::kBlockBytes / 4) >= (size_t) 1 << 31) return 0;
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
