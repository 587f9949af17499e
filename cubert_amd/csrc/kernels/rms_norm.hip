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
// single elements and a maximum, and no order of a sum can move one across a border.  A row lives in registers between
// the statistics and the results, so that the sum may be written over either input.

#include "cubert_kernels.h"
#include "device_common.h"

namespace cubert {
namespace {

constexpr int kMaxHidden = 32768;
constexpr int kMaxRows = 1 << 21;  // a launch holds less than 2^32 threads

// One workgroup of WAVES wavefronts per row, PER elements to a lane, WAVES * 64 apart.
template <typename T, int WAVES, int PER, bool CODES>
__global__ __launch_bounds__(WAVES * kWave) void rms_norm_kernel(const T *x, const T *residual, const T *__restrict__ gamma, float eps,
                                                                T *sum_out, T *__restrict__ out, int8_t *__restrict__ codes,
                                                                float *__restrict__ scales, int hidden) {
    __shared__ float traded[2][WAVES];
    const size_t row = blockIdx.x;
    const int thread = threadIdx.x, wave = wave_in_block();
    x += row * hidden;
    if (residual != nullptr) residual += row * hidden;
    float s[PER];
    float squares = 0.f, top = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int col = i * WAVES * kWave + thread;
        s[i] = 0.f;
        if (col < hidden) {
            s[i] = to_f32(x[col]);
            if (residual != nullptr) s[i] += to_f32(residual[col]);
            squares = fmaf(s[i], s[i], squares);
            if (CODES) top = fmaxf(top, fabsf(to_f32(gamma[col]) * s[i]));
        }
    }
    squares = wave_sum(squares);
    if (CODES) top = wave_max(top);
    if ((thread & (kWave - 1)) == 0) {
        traded[0][wave] = squares;
        traded[1][wave] = top;
    }
    __syncthreads();
    squares = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        squares += traded[0][w];
        top = fmaxf(top, traded[1][w]);
    }
    const float rstd = 1.f / sqrtf(squares / (float) hidden + eps);
    // A NaN is lost in a maximum and an infinity leaves no finite factor: such a row's scale is NaN and its codes are 0.
    const bool finite = squares < INFINITY;
    // 127 / m leaves fp32's range for m below 2^-121: rows that small are raised by a power of two first, which is exact.
    const float raise = top < 0x1p-60f ? 0x1p80f : 1.f;
    const float inverse = top > 0.f && finite ? 127.f / (top * raise) : 0.f;
    if (CODES && thread == 0) scales[row] = finite ? top * rstd / 127.f : NAN;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int col = i * WAVES * kWave + thread;
        if (col < hidden) {
            const float g = to_f32(gamma[col]);
            if (sum_out != nullptr) sum_out[row * hidden + col] = from_f32<T>(s[i]);
            if (CODES) codes[row * hidden + col] = finite ? (int8_t) rintf(((g * s[i]) * raise) * inverse) : (int8_t) 0;
            else out[row * hidden + col] = from_f32<T>(g * (s[i] * rstd));
        }
    }
}

template <typename T, bool CODES>
int rms_norm(const T *x, const T *residual, const T *gamma, float eps, T *sum_out, T *out, int8_t *codes, float *scales, int rows,
             int hidden, void *stream) {
    if (rows < 0 || hidden < 1 || !(eps >= 0.f) || !(eps < INFINITY)) return CUBERT_BAD_ARGUMENT;
    if (hidden > kMaxHidden || rows > kMaxRows) return CUBERT_UNSUPPORTED;
    if (rows == 0) return 0;
    if (x == nullptr || gamma == nullptr || (CODES ? codes == nullptr || scales == nullptr : out == nullptr)) return CUBERT_BAD_ARGUMENT;
    const hipStream_t s = (hipStream_t) stream;
#define RUN(WAVES, PER)                                                                                                     \
    if (hidden <= WAVES * kWave * PER)                                                                                      \
        return launch(rms_norm_kernel<T, WAVES, PER, CODES>, dim3(rows), dim3(WAVES * kWave), s, x, residual, gamma, eps, sum_out, \
                      out, codes, scales, hidden);
    RUN(4, 4) RUN(4, 16) RUN(16, 8) RUN(16, 32)
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
