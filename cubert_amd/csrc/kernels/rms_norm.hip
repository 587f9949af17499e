// Residual + root-mean-square norm, the step between the layers of a pre-norm model:
//
//     s = x + r,    y = gamma * s / sqrt(mean(s^2) + eps)
//
// with s handed on as the next residual and y either in the storage type or as whole numbers of 8 bits with one scale
// per row, the operand form of cubert_dense_w4_i8_*:
//
//     t = gamma * s,  m = max |t|,  code = rint(t * (127 / m)),  scale = m / (127 sqrt(mean(s^2) + eps)).
//
// The norm's factor is the same for a whole row, so it divides out of the codes: they follow from fp32 operations on
// single elements and a maximum, and no order of a sum can move one across a border.  A thread keeps its part of a row between
// the statistics and the results, so that the sum may be written over either input: in registers, but for rows of more than 4096 elements
// that are no whole 16-byte pieces, which have 34 of them in scratch memory.

#include "cubert_kernels.h"
#include "device_common.h"

namespace cubert {
namespace {

constexpr int kMaxHidden = 32768;

// Bound by memory where there are many rows: fp16, 32768 x 1024 with a residual, 268 MB in 49 us, 5.5 TB/s (a large copy reaches 5.1);
// fp32 in 8 bits, 4099 x 1000, 53 MB in 10.2 us, 5.2 TB/s.  A few rows are one read, two exchanges and one write behind each other:
// 1 x 768 1.8 us, 8 x 4096 in 8 bits 4.2 us.
//
// The largest, or a NaN where there is one (fmaxf takes the number).
struct LargestOp {
    __device__ __forceinline__ float operator()(float a, float b) const { return __builtin_elementwise_maximum(a, b); }
};

// WAVES wavefronts per row, ROWS rows to a workgroup; a lane has CHUNKS runs of VEC elements, WAVES * 64 runs apart.
template <typename T, int VEC, int CHUNKS, int WAVES, int ROWS, bool CODES>
__global__ __launch_bounds__(WAVES * ROWS * kWave) void rms_norm_kernel(const T *x, const T *residual, const T *__restrict__ gamma, float eps,
                                                                        T *sum_out, T *__restrict__ out, int8_t *__restrict__ codes,
                                                                        float *__restrict__ scales, int rows, int hidden) {
    static_assert(WAVES == 1 || ROWS == 1, "a row of several wavefronts has the workgroup to itself");
    __shared__ float traded[2][WAVES];
    const int wave = wave_in_block(), row = blockIdx.x * ROWS + (WAVES == 1 ? wave : 0);
    if (row >= rows) return;  // (with several wavefronts to a row, never)
    const int run = WAVES == 1 ? threadIdx.x & (kWave - 1) : threadIdx.x;
    const size_t at = (size_t) row * hidden;
    Vec<T, VEC> a[CHUNKS], r[CHUNKS], g[CHUNKS];
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
        const int col = (c * WAVES * kWave + run) * VEC;
        if (col < hidden) a[c] = load_vec<T, VEC>(x + at + col);
    }
    if (residual != nullptr) {
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            const int col = (c * WAVES * kWave + run) * VEC;
            if (col < hidden) r[c] = load_vec<T, VEC>(residual + at + col);
        }
    }
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
        const int col = (c * WAVES * kWave + run) * VEC;
        if (col < hidden) g[c] = load_vec<T, VEC>(gamma + col);
    }
    float s[CHUNKS][VEC];
    float squares = 0.f, top = 0.f;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
        if ((c * WAVES * kWave + run) * VEC < hidden) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                s[c][i] = to_f32(a[c].v[i]);
                if (residual != nullptr) s[c][i] += to_f32(r[c].v[i]);
                squares = fmaf(s[c][i], s[c][i], squares);
                if (CODES) top = LargestOp()(top, fabsf(to_f32(g[c].v[i]) * s[c][i]));
            }
        }
    }
    squares = wave_sum(squares);
    if (CODES) top = group_reduce<kWave>(top, LargestOp());
    if constexpr (WAVES > 1) {
        if ((threadIdx.x & (kWave - 1)) == 0) {
            traded[0][wave] = squares;
            traded[1][wave] = top;
        }
        __syncthreads();
        squares = 0.f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            squares += traded[0][w];
            if (CODES) top = LargestOp()(top, traded[1][w]);
        }
    }
    const float power = squares / (float) hidden + eps, rstd = power == 0.f ? 0.f : 1.f / sqrtf(power);
    // Neither a NaN nor an infinity leaves a finite factor: such a row's scale is NaN and its codes are 0.  gamma may bring them as well.
    const bool finite = squares < INFINITY && top < INFINITY;
    // 127 / m leaves fp32's range for m below 2^-121: rows that small are raised by a power of two first, which is exact.
    const float raise = top < 0x1p-60f ? 0x1p80f : 1.f;
    const float inverse = top > 0.f && finite ? 127.f / (top * raise) : 0.f;
    if (CODES && run == 0) scales[row] = finite ? top * rstd / 127.f : NAN;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
        const int col = (c * WAVES * kWave + run) * VEC;
        if (col < hidden) {
            Vec<T, VEC> total, y;
            Vec<int8_t, VEC> code;
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const float gain = to_f32(g[c].v[i]);
                total.v[i] = from_f32<T>(s[c][i]);
                if (CODES) code.v[i] = finite ? (int8_t) rintf(((gain * s[c][i]) * raise) * inverse) : (int8_t) 0;
                else y.v[i] = from_f32<T>(gain * (s[c][i] * rstd));
            }
            if (sum_out != nullptr) store_vec<T, VEC>(sum_out + at + col, total);
            if (CODES) store_vec<int8_t, VEC>(codes + at + col, code);
            else store_vec<T, VEC>(out + at + col, y);
        }
    }
}

template <typename T, bool CODES>
int rms_norm(const T *x, const T *residual, const T *gamma, float eps, T *sum_out, T *out, int8_t *codes, float *scales, int rows,
             int hidden, void *stream) {
    if (rows < 0 || hidden < 1 || !(eps >= 0.f) || !(eps < INFINITY)) return CUBERT_BAD_ARGUMENT;
    if (hidden > kMaxHidden) return CUBERT_UNSUPPORTED;
    if (rows == 0) return 0;
    if (x == nullptr || gamma == nullptr || (CODES ? codes == nullptr || scales == nullptr : out == nullptr)) return CUBERT_BAD_ARGUMENT;
    const hipStream_t s = (hipStream_t) stream;
    constexpr int kVec = 16 / (int) sizeof(T);
    const bool whole = hidden % kVec == 0 && is_aligned(x, 16) && is_aligned(gamma, 16) && (residual == nullptr || is_aligned(residual, 16)) &&
                       (sum_out == nullptr || is_aligned(sum_out, 16)) && (CODES ? is_aligned(codes, kVec) : is_aligned(out, 16));
#define RUN(VEC, CHUNKS, WAVES, ROWS)                                                                                         \
    if (hidden <= VEC * CHUNKS * WAVES * kWave) {                                                                             \
        if ((rows + (ROWS - 1ll)) / ROWS * (WAVES * ROWS * kWave) >= 1ll << 32) return CUBERT_UNSUPPORTED;                    \
        return launch(rms_norm_kernel<T, VEC, CHUNKS, WAVES, ROWS, CODES>, dim3((rows + (ROWS - 1ll)) / ROWS),         \
                      dim3(WAVES * ROWS * kWave), s, x, residual, gamma, eps, sum_out, out, codes, scales, rows, hidden);     \
    }
    // A wavefront per row where a row is one run of its lanes or the rows fill the card, otherwise four (or sixteen) per row.  Microseconds
    // with one / four: fp16, 16384 x 256 9.3 / 17.4, 128 x 256 2.6 / 2.7, 4096 x 1024 8.3 / 8.5, 1024 x 1024 4.5 / 3.5, 64 x 1024
    // 3.2 / 2.7, 4096 x 2000 15.3 / 16.0, 300 x 2000 4.7 / 3.2; fp32 in 8 bits, 512 x 256 2.7 / 2.9, 1024 x 1024 5.2 / 5.0.
    if (whole && (rows >= 2048 || hidden <= kVec * kWave)) {
        RUN(kVec, 1, 1, 4) RUN(kVec, 2, 1, 4) RUN(kVec, 4, 1, 4)
    }
    if (whole) {
        RUN(kVec, 1, 4, 1) RUN(kVec, 2, 4, 1) RUN(kVec, 1, 16, 1) RUN(kVec, 4, 16, 1)
        if constexpr (sizeof(T) == 4) RUN(kVec, 8, 16, 1)
    }
    // Rows of no whole 16-byte pieces, an element at a time; microseconds against rows of pieces as long: fp16, 4096 x 1001 13 and 8, 32768
    // x 1025 200 and 53, 4096 x 4100 132 and 28; fp32, 4096 x 1001 16 and 14, 32768 x 1025 161 and 94, 1024 x 32767 195
    // and 106.
    RUN(1, 4, 4, 1) RUN(1, 4, 16, 1) RUN(1, 32, 16, 1)
#undef RUN
    return CUBERT_UNSUPPORTED;
}

}  // namespace
}  // namespace cubert

using cubert::half_t;

extern "C" {

int cubert_res_rms_norm_f32(const float *in, const float *residual, const float *gamma, float eps, float *sum_out, float *out,
                            int rows, int hidden, void *stream) {
    return cubert::rms_norm<float, false>(in, residual, gamma, eps, sum_out, out, nullptr, nullptr, rows, hidden, stream);
}

int cubert_res_rms_norm_f16(const cubert_half *in, const cubert_half *residual, const cubert_half *gamma, float eps,
                            cubert_half *sum_out, cubert_half *out, int rows, int hidden, void *stream) {
    return cubert::rms_norm<half_t, false>((const half_t *) in, (const half_t *) residual, (const half_t *) gamma, eps,
                                           (half_t *) sum_out, (half_t *) out, nullptr, nullptr, rows, hidden, stream);
}

int cubert_res_rms_norm_i8_f32(const float *in, const float *residual, const float *gamma, float eps, float *sum_out, int8_t *out,
                               float *scales, int rows, int hidden, void *stream) {
    return cubert::rms_norm<float, true>(in, residual, gamma, eps, sum_out, nullptr, out, scales, rows, hidden, stream);
}

int cubert_res_rms_norm_i8_f16(const cubert_half *in, const cubert_half *residual, const cubert_half *gamma, float eps,
                               cubert_half *sum_out, int8_t *out, float *scales, int rows, int hidden, void *stream) {
    return cubert::rms_norm<half_t, true>((const half_t *) in, (const half_t *) residual, (const half_t *) gamma, eps,
                                          (half_t *) sum_out, nullptr, out, scales, rows, hidden, stream);
}

}  // extern "C"
