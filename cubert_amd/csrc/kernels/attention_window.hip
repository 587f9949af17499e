// Attention with a sliding window and first tokens that stay visible, over whole sequences or over a cache:
//
//     query i of sequence b stands at p = first[b] + i and sees key j if
//         j < length[b],  mask[b, j] != 0,  j <= p + right  and  (j >= p - left  or  j < sinks);
//     ctx = sum_j e^(alpha q.k_j - m) v_j / sum_j e^(alpha q.k_j - m) over what it sees, m the largest score.
//
// A query that sees nothing, or that stands outside its sequence (p < 0 or p >= length[b]), gets zeros.  Heads share keys
// and values in groups of heads / kv_heads.

#include "cubert_kernels.h"
#include "device_common.h"

namespace cubert {
namespace {

constexpr int kFar = 1 << 30;  // a bound, position or length that no sequence reaches

struct WindowArgs {
    const void *q, *k, *v;
    void *ctx;
    const int *first, *lengths;
    const int8_t *mask;
    float *partials;
    float scale;  // alpha * log2(e)
    int ldq, ldkv, ld_ctx;
    int batch, heads, kv_heads, q_rows, kv_rows;
    int left, right, sinks;
};

__device__ __forceinline__ int clamp_to(int x, int low, int high) { return x < low ? low : x > high ? high : x; }

// One wavefront per query and head, 64 keys at a time: a lane scores one key, then sums D / 64 columns over the keys.
template <typename T, int D>
__global__ __launch_bounds__(kBlock) void attention_window_kernel(WindowArgs a) {
    __shared__ float probs[kBlock / kWave][kWave];
    const int wave = wave_in_block(), lane = threadIdx.x & (kWave - 1);
    const size_t at = (size_t) blockIdx.x * (kBlock / kWave) + wave;
    if (at >= (size_t) a.batch * a.heads * a.q_rows) return;
    const int i = (int) (at % a.q_rows), head = (int) (at / a.q_rows % a.heads), b = (int) (at / a.q_rows / a.heads);
    const int length = a.lengths != nullptr ? clamp_to(a.lengths[b], 0, a.kv_rows) : a.kv_rows;
    const int p = (a.first != nullptr ? clamp_to(a.first[b], -kFar, kFar) : 0) + i;
    const T *q = (const T *) a.q + ((size_t) b * a.q_rows + i) * a.ldq + head * D;
    const int kv_head = head / (a.heads / a.kv_heads);
    const T *k = (const T *) a.k + (size_t) b * a.kv_rows * a.ldkv + kv_head * D;
    const T *v = (const T *) a.v + (size_t) b * a.kv_rows * a.ldkv + kv_head * D;
    const int8_t *mask = a.mask != nullptr ? a.mask + (size_t) b * a.kv_rows : nullptr;
    constexpr int kCols = (D + kWave - 1) / kWave;
    float acc[kCols] = {};
    float top = -INFINITY, sum = 0.f;
    const bool there = p >= 0 && p < length;
    const int end = there ? (p < length - a.right ? p + a.right + 1 : length) : 0;  // (p + right does not overflow here)
    const int begin = p > a.left ? p - a.left : 0;
    for (int base = 0; base < end; base += kWave) {
        if (base >= a.sinks && base + kWave <= begin) base = begin / kWave * kWave;  // nothing between the sinks and the window
        const int j = base + lane;
        const bool seen = j < end && (j >= begin || j < a.sinks) && (mask == nullptr || mask[j] != 0);
        float score = -INFINITY;
        if (seen) {
            score = 0.f;
            for (int d = 0; d < D; ++d) score = fmaf(to_f32(q[d]), to_f32(k[(size_t) j * a.ldkv + d]), score);
            score *= a.scale;
        }
        const float high = fmaxf(top, wave_max(score));
        if (high == -INFINITY) continue;  // (the same in every lane)
        const float shrink = exp2f(top - high), prob = seen ? exp2f(score - high) : 0.f;
        sum = sum * shrink + wave_sum(prob);
        top = high;
        probs[wave][lane] = prob;
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int c = 0; c < kCols; ++c) {
            const int d = c * kWave + lane;
            acc[c] *= shrink;
            for (int n = 0; n < kWave && base + n < end; ++n) {
                const float pn = probs[wave][n];
                if (pn != 0.f && d < D) acc[c] = fmaf(pn, to_f32(v[(size_t) (base + n) * a.ldkv + d]), acc[c]);
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
    T *ctx = (T *) a.ctx + ((size_t) b * a.q_rows + i) * a.ld_ctx + head * D;
#pragma unroll
    for (int c = 0; c < kCols; ++c) {
        const int d = c * kWave + lane;
        if (d < D) ctx[d] = from_f32<T>(sum > 0.f ? acc[c] / sum : 0.f);
    }
}

template <typename T>
int attention_window(const T *q, int ldq, const T *k, const T *v, int ldkv, const int *first, const int *lengths, const int8_t *mask,
                     T *ctx, int ld_ctx, float alpha, int batch, int heads, int kv_heads, int q_rows, int kv_rows, int head_size,
                     int left, int right, int sinks, float *partials, size_t partial_floats, void *stream) {
    if (batch < 0 || heads < 1 || kv_heads < 1 ||
        heads % kv_heads != 0 || q_rows < 0 || kv_rows < 0 || head_size < 1 || sinks < 0 || kv_rows > kFar || q_rows > kFar)
        return CUBERT_BAD_ARGUMENT;
    const long long width = (long long) heads * head_size, kv_width = (long long) kv_heads * head_size;
    if (ldq < width || ldkv < kv_width || ld_ctx < width) return CUBERT_BAD_ARGUMENT;
    if (batch == 0 || q_rows == 0) return 0;
    if (q == nullptr || ctx == nullptr || (kv_rows > 0 && (k == nullptr || v == nullptr))) return CUBERT_BAD_ARGUMENT;
    const int piece = 16 / (int) sizeof(T);
    if (!is_aligned(q, 16) || !is_aligned(k, 16) || !is_aligned(v, 16) || !is_aligned(ctx, 16) || ldq % piece != 0 ||
        ldkv % piece != 0 || ld_ctx % piece != 0)
        return CUBERT_UNSUPPORTED;
    if (head_size != 32 && head_size != 64 && head_size != 128) return CUBERT_UNSUPPORTED;
    const unsigned long long rows = (unsigned long long) batch * q_rows * heads;
    if (rows >= 1u << 26) return CUBERT_UNSUPPORTED;  // a launch holds less than 2^32 threads
    WindowArgs a;
    a.q = q, a.k = k, a.v = v, a.ctx = ctx, a.first = first, a.lengths = lengths, a.mask = mask;
    a.partials = partials;
    a.scale = alpha * 1.44269504089f;
    a.ldq = ldq, a.ldkv = ldkv, a.ld_ctx = ld_ctx;
    a.batch = batch, a.heads = heads, a.kv_heads = kv_heads, a.q_rows = q_rows, a.kv_rows = kv_rows;
    a.left = left < 0 || left > kFar ? kFar : left, a.right = right < 0 || right > kFar ? kFar : right;
    a.sinks = sinks;
    (void) partial_floats;
    const dim3 grid((unsigned) ((rows + 3) / 4));
    if (head_size == 32) return launch(attention_window_kernel<T, 32>, grid, dim3(kBlock), (hipStream_t) stream, a);
    if (head_size == 64) return launch(attention_window_kernel<T, 64>, grid, dim3(kBlock), (hipStream_t) stream, a);
    return launch(attention_window_kernel<T, 128>, grid, dim3(kBlock), (hipStream_t) stream, a);
}

}  // namespace
}  // namespace cubert

using cubert::half_t;

extern "C" {

size_t cubert_attention_window_partials(int half_precision, int batch, int heads, int kv_heads, int q_rows, int kv_rows,
                                        int head_size, int left, int right, int sinks) {
    (void) half_precision, (void) batch, (void) heads, (void) kv_heads, (void) q_rows, (void) kv_rows, (void) head_size;
    (void) left, (void) right, (void) sinks;
    return 0;
}

int cubert_attention_window_f32(const float *q, int ldq, const float *k, const float *v, int ldkv, const int *first,
                                const int *lengths, const int8_t *mask, float *ctx, int ld_ctx, float alpha, int batch, int heads,
                                int kv_heads, int q_rows, int kv_rows, int head_size, int left, int right, int sinks,
                                float *partials, size_t partial_floats, void *stream) {
    return cubert::attention_window<float>(q, ldq, k, v, ldkv, first, lengths, mask, ctx, ld_ctx, alpha, batch, heads, kv_heads,
                                           q_rows, kv_rows, head_size, left, right, sinks, partials, partial_floats, stream);
}

int cubert_attention_window_f16(const cubert_half *q, int ldq, const cubert_half *k, const cubert_half *v, int ldkv, const int *first,
                                const int *lengths, const int8_t *mask, cubert_half *ctx, int ld_ctx, float alpha, int batch,
                                int heads, int kv_heads, int q_rows, int kv_rows, int head_size, int left, int right, int sinks,
                                float *partials, size_t partial_floats, void *stream) {
    return cubert::attention_window<half_t>((const half_t *) q, ldq, (const half_t *) k, (const half_t *) v, ldkv, first, lengths, mask,
                                            (half_t *) ctx, ld_ctx, alpha, batch, heads, kv_heads, q_rows, kv_rows, head_size, left,
                                            right, sinks, partials, partial_floats, stream);
}

}  // extern "C"
