// Attention of new tokens over a key/value cache in pages:
//
//     query i of sequence b stands at p = first[b] + i and sees key j if
//         j <= p,  j < length[b],  table[b, j / page] is a page  and  (j >= p - left  or  j < sinks);
//     ctx = sum_j e^(alpha q.k_j - m) v_j / sum_j e^(alpha q.k_j - m) over what it sees, m the largest score.
//
// A query that sees nothing, or that stands outside its sequence (p < 0 or p >= length[b]), gets zeros.  Heads share keys
// and values in groups of heads / kv_heads.

#include "cubert_kernels.h"
#include "device_common.h"
#include "paged.h"

namespace cubert {
namespace {

constexpr int kFar = (1 << 30) - 1;  // a bound or position that no sequence reaches
constexpr float kNone = -3e38f;      // the maximum of no scores: finite, so that differences to it are numbers

struct PagedArgs {
    const void *q, *k, *v;
    void *ctx;
    const int *table, *lengths, *first;
    float *partials;
    float scale;  // |alpha| * log2(e)
    long long page_stride, head_stride, row_stride;
    int ldq, ld_ctx, width, ld_table;
    int batch, heads, kv_heads, q_rows, pages, shift;
    int left, sinks;
    bool negate;  // alpha is negative: q changes its sign, so that the largest score is that of the largest product
};

__device__ __forceinline__ int clamp_to(int x, int low, int high) { return x < low ? low : x > high ? high : x; }

// A workgroup per query and head, a thread per key for the scores and D / 4 threads to a key for the sums.
template <typename T, int D>
__global__ __launch_bounds__(kBlock) void attention_paged_kernel(PagedArgs a) {
    constexpr int kQuads = D / 4, kAtOnce = kBlock / kQuads;
    __shared__ float q[D], probs[kBlock], shared[kBlock / kWave], parts[kAtOnce][D];
    __shared__ long long rows[kBlock];
    const int head = blockIdx.x % a.heads, row = blockIdx.x / a.heads, b = row / a.q_rows, thread = threadIdx.x;
    const int length = clamp_to(a.lengths[b], 0, a.width << a.shift);
    const int p = (a.first != nullptr ? clamp_to(a.first[b], -kFar, kFar) : length - a.q_rows) + row - b * a.q_rows;
    const bool there = p >= 0 && p < length;
    const int begin = p > a.left ? p - a.left : 0, far = a.sinks < begin ? a.sinks : begin, count = there ? far + p + 1 - begin : 0;
    const T *k = (const T *) a.k + head / (a.heads / a.kv_heads) * a.head_stride, *v = (const T *) a.v + head / (a.heads / a.kv_heads) * a.head_stride;
    if (thread < D) {
        const float x = to_f32(((const T *) a.q)[(size_t) row * a.ldq + head * D + thread]);
        q[thread] = a.negate ? -x : x;
    }
    float top = kNone, sum = 0.f, x[4] = {};
    const int group = thread / kQuads, d = thread % kQuads * 4;
    for (int base = 0; base < count; base += kBlock) {
        const int n = base + thread;
        float score = -INFINITY;
        long long at = -1;
        __syncthreads();
        if (n < count) {
            const int j = n < far ? n : begin + n - far, page = a.table[(size_t) b * a.ld_table + (j >> a.shift)];
            if (page >= 0 && page < a.pages) {
                at = page * a.page_stride + (j & ((1 << a.shift) - 1)) * a.row_stride;
                score = 0.f;
                for (int e = 0; e < D; e += 4) {
                    const Vec<T, 4> piece = load_vec<T, 4>(k + at + e);
#pragma unroll
                    for (int i = 0; i < 4; ++i) score = fmaf(q[e + i], to_f32(piece.v[i]), score);
                }
            }
        }
        rows[thread] = at;
        float high = wave_max(score);
        if ((thread & (kWave - 1)) == 0) shared[thread / kWave] = high;
        __syncthreads();
        high = top;
#pragma unroll
        for (int w = 0; w < kBlock / kWave; ++w) high = fmaxf(high, shared[w]);
        const float shrink = __builtin_amdgcn_exp2f((top - high) * a.scale);
        top = high;
        probs[thread] = __builtin_amdgcn_exp2f((score - top) * a.scale);
        __syncthreads();
        const float part = wave_sum(probs[thread]);
        if ((thread & (kWave - 1)) == 0) shared[thread / kWave] = part;
        __syncthreads();
        sum *= shrink;
#pragma unroll
        for (int w = 0; w < kBlock / kWave; ++w) sum += shared[w];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] *= shrink;
        for (int m = group; m < kBlock; m += kAtOnce) {
            if (rows[m] < 0) continue;
            const Vec<T, 4> piece = load_vec<T, 4>(v + rows[m] + d);
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = fmaf(probs[m], to_f32(piece.v[i]), x[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) parts[group][d + i] = x[i];
    __syncthreads();
    if (thread < D) {
        float total = 0.f;
        for (int g = 0; g < kAtOnce; ++g) total += parts[g][thread];
        ((T *) a.ctx)[(size_t) row * a.ld_ctx + head * D + thread] = from_f32<T>(sum != 0.f ? total / sum : 0.f);
    }
}

template <typename T>
int attention_paged(const T *q, int ldq, const T *k_pages, const T *v_pages, long long page_stride, long long head_stride, long long row_stride,
                    const int *table, int width, int ld_table, const int *lengths, const int *first, T *ctx, int ld_ctx, float alpha, int batch,
                    int heads, int kv_heads, int q_rows, int pages, int page, int head_size, int left, int sinks, float *partials,
                    size_t partial_floats, void *stream) {
    if (batch < 0 || heads < 1 || kv_heads < 1 || heads % kv_heads != 0 || !(alpha > -INFINITY && alpha < INFINITY) || q_rows < 0 || q_rows > kFar ||
        pages < 1 || page < 1 || head_size < 1 || sinks < 0 || width < 1 || ld_table < width)
        return CUBERT_BAD_ARGUMENT;
    const long long q_width = (long long) heads * head_size;
    if (ldq < q_width || ld_ctx < q_width) return CUBERT_BAD_ARGUMENT;
    if (!pages_apart(page_stride, head_stride, row_stride, pages, kv_heads, page, head_size)) return CUBERT_BAD_ARGUMENT;
    if (batch == 0 || q_rows == 0) return 0;
    if (q == nullptr || ctx == nullptr || k_pages == nullptr || v_pages == nullptr || table == nullptr || lengths == nullptr) return CUBERT_BAD_ARGUMENT;
    const int piece = 16 / (int) sizeof(T);
    if (!is_aligned(q, 16) || !is_aligned(k_pages, 16) || !is_aligned(v_pages, 16) || !is_aligned(ctx, 16) || ldq % piece != 0 || ld_ctx % piece != 0 ||
        page_stride % piece != 0 || head_stride % piece != 0 || row_stride % piece != 0)
        return CUBERT_UNSUPPORTED;
    if (head_size != 32 && head_size != 64 && head_size != 128) return CUBERT_UNSUPPORTED;
    if (page < 16 || (page & (page - 1)) != 0) return CUBERT_UNSUPPORTED;
    if ((long long) width * page > kFar || (long long) pages * page >= 1ll << 31) return CUBERT_UNSUPPORTED;
    if (row_stride > (1ll << 31) / page / 4) return CUBERT_UNSUPPORTED;  // (rows of a page are addressed with 32 bits)
    PagedArgs a;
    a.q = q, a.k = k_pages, a.v = v_pages, a.ctx = ctx, a.table = table, a.lengths = lengths, a.first = first, a.partials = partials;
    a.negate = alpha < 0.f;
    // (a factor of 0 would make numbers of the infinities that stand for keys left out, an infinite one no number of a difference of 0)
    a.scale = fminf(fmaxf(fabsf(alpha) * 1.44269504089f, 1e-30f), 3e38f);
    a.page_stride = page_stride, a.head_stride = head_stride, a.row_stride = row_stride;
    a.ldq = ldq, a.ld_ctx = ld_ctx, a.width = width, a.ld_table = ld_table;
    a.batch = batch, a.heads = heads, a.kv_heads = kv_heads, a.q_rows = q_rows, a.pages = pages, a.shift = __builtin_ctz((unsigned) page);
    a.left = left < 0 || left > kFar ? kFar : left, a.sinks = sinks < kFar ? sinks : kFar;
    (void) partial_floats;
    const unsigned long long blocks = (unsigned long long) batch * q_rows * heads;
    if ((unsigned long long) batch * q_rows >= 1u << 24 || blocks >= 1u << 24) return CUBERT_UNSUPPORTED;
    const dim3 grid((unsigned) blocks), block(kBlock);
    if (head_size == 32) return launch(attention_paged_kernel<T, 32>, grid, block, (hipStream_t) stream, a);
    if (head_size == 64) return launch(attention_paged_kernel<T, 64>, grid, block, (hipStream_t) stream, a);
    return launch(attention_paged_kernel<T, 128>, grid, block, (hipStream_t) stream, a);
}

}  // namespace
}  // namespace cubert

using cubert::half_t;

extern "C" {

size_t cubert_attention_paged_partials(int half_precision, int batch, int heads, int kv_heads, int q_rows, int width, int page, int head_size, int left,
                                       int sinks) {
    (void) half_precision, (void) batch, (void) heads, (void) kv_heads, (void) q_rows, (void) width, (void) page, (void) head_size, (void) left, (void) sinks;
    return 0;
}

int cubert_attention_paged_f32(const float *q, int ldq, const float *k_pages, const float *v_pages, long long page_stride, long long head_stride,
                               long long row_stride, const int *table, int width, int ld_table, const int *lengths, const int *first, float *ctx,
                               int ld_ctx, float alpha, int batch, int heads, int kv_heads, int q_rows, int pages, int page, int head_size, int left,
                               int sinks, float *partials, size_t partial_floats, void *stream) {
    return cubert::attention_paged<float>(q, ldq, k_pages, v_pages, page_stride, head_stride, row_stride, table, width, ld_table, lengths, first, ctx, ld_ctx,
                                          alpha, batch, heads, kv_heads, q_rows, pages, page, head_size, left, sinks, partials, partial_floats, stream);
}

int cubert_attention_paged_f16(const cubert_half *q, int ldq, const cubert_half *k_pages, const cubert_half *v_pages, long long page_stride,
                               long long head_stride, long long row_stride, const int *table, int width, int ld_table, const int *lengths,
                               const int *first, cubert_half *ctx, int ld_ctx, float alpha, int batch, int heads, int kv_heads, int q_rows, int pages,
                               int page, int head_size, int left, int sinks, float *partials, size_t partial_floats, void *stream) {
    return cubert::attention_paged<half_t>((const half_t *) q, ldq, (const half_t *) k_pages, (const half_t *) v_pages, page_stride, head_stride, row_stride,
                                           table, width, ld_table, lengths, first, (half_t *) ctx, ld_ctx, alpha, batch, heads, kv_heads, q_rows, pages,
                                           page, head_size, left, sinks, partials, partial_floats, stream);
}

}  // extern "C"
