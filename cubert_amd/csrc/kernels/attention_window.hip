// Attention with a sliding window and first tokens that stay visible, over whole sequences or over a cache:
//
//     query i of sequence b stands at p = first[b] + i and sees key j if
//         j < length[b],  mask[b, j] != 0,  j <= p + right  and  (j >= p - left  or  j < sinks);
//     ctx = sum_j e^(alpha q.k_j - m) v_j / sum_j e^(alpha q.k_j - m) over what it sees, m the largest score.
//
// A query that sees nothing, or that stands outside its sequence (p < 0 or p >= length[b]), gets zeros.  Heads share keys
// and values in groups of heads / kv_heads.

#include <atomic>

#include "cubert_kernels.h"
#include "device_common.h"

namespace cubert {
namespace {

constexpr int kMaxPieces = 128;  // of an axis that is cut
constexpr int kFewPieces = 8;    // that one thread takes
constexpr int kFar = (1 << 30) - 1;  // a bound, position or length that no sequence reaches

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
    bool negate;  // alpha is negative: q changes its sign, so that the largest score is that of the largest product
};

typedef _Float16 v8f16 __attribute__((ext_vector_type(8)));
typedef _Float16 v2f16 __attribute__((ext_vector_type(2)));
typedef float v4f32 __attribute__((ext_vector_type(4)));
typedef float v2f32 __attribute__((ext_vector_type(2)));
typedef int v4i32 __attribute__((ext_vector_type(4)));
typedef float v16f32 __attribute__((ext_vector_type(16)));

// Probabilities are 2^(scale (s - top)) of scores s and a maximum `top` of them, both as the products leave them: the difference is
// taken first.  (One fused 2^(scale s - top), with a scaled maximum, is an instruction less, but that maximum's rounding grows with the
// scores: beyond 2^26 the largest probability itself was 0 or infinite.)
constexpr float kNone = -3e38f;  // the maximum of no scores: finite, so that differences to it are numbers
constexpr float kSlack = 8.f;    // how far a maximum may rise, in powers of two, before sums are scaled anew (fp32)
// Probabilities in 16 bits are 2^kRaise times as large, so that fp16's subnormals begin far below the maximum: a
// probability loses 2^-25 of that at most, 2^-35 or 2^-37 of the largest, and a long axis of small ones is not lost next to one
// large.  At the top end what a maximum may rise before sums are scaled anew keeps them within fp16.
template <int N>
struct Range;
template <>
struct Range<1> {  // few rows: the maximum is looked at
    static constexpr float kRaise = 12.f, kSlack = 3.f;
};
template <>
struct Range<2> {  // many: what the probabilities of a tile add up to in half a row, 32 of them
    static constexpr float kRaise = 10.f, kMost = 60000.f;
};

// 32 rows (queries and heads of one key head) meet 32 keys in one matrix product with the keys as its rows: lane l has row
// l % 32 and, in accumulator i, key 8 (i / 4) + 4 (l / 32) + i % 4.  The probabilities are then the second operand of the
// product with V transposed, whose reduction may take its keys in any order that both operands keep, so they never
// leave their lane, and neither does what belongs to a row: maximum, sum and the D / 2 results that a lane holds.
template <typename T, int D>
struct Rows {
    static constexpr int kSteps = D * (int) sizeof(T) / 32;  // 16-byte pieces of an operand row in a half wavefront
    static constexpr int kRowBytes = D * (int) sizeof(T);
    static constexpr int kPieces = kRowBytes / 16;

    v4f32 q[kSteps];  // pieces 2 s + l / 32 of the row
    v16f32 ctx[D / 32];
    float top, sum;
    bool fresh = true;  // no key yet (the same in every lane)

    __device__ __forceinline__ void load(const T *row, int half_wave, bool negate) {
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            q[s] = *reinterpret_cast<const v4f32 *>(reinterpret_cast<const char *>(row) + (2 * s + half_wave) * 16);
            if (negate) {
                if constexpr (sizeof(T) == 2) q[s] = __builtin_bit_cast(v4f32, -__builtin_bit_cast(v8f16, q[s]));
                else q[s] = -q[s];
            }
        }
#pragma unroll
        for (int d = 0; d < D / 32; ++d) ctx[d] = v16f32{};
        top = kNone, sum = 0.f;
    }
};

// Which of its 16-byte pieces a row of K or V keeps its piece `at` in, so that the lanes that read together find their
// pieces on different banks (64 of 4 bytes): of K 16 lanes read one piece of as many rows; of V in 16 bits a half wavefront reads
// 64 bytes of four rows, in 32 bits either half 128 bytes of rows that are four apart.
template <int ROW_BYTES>
__device__ __forceinline__ int k_piece(int key, int at) {
    constexpr int kShift = ROW_BYTES >= 256 ? 0 : ROW_BYTES == 128 ? 1 : 2, kMask = ROW_BYTES >= 256 ? 15 : ROW_BYTES / 16 - 1;
    return at ^ ((key >> kShift) & kMask);
}
template <typename T, int ROW_BYTES>
__device__ __forceinline__ int v_piece(int key, int at) {
    if constexpr (sizeof(T) == 2) return ROW_BYTES == 256 ? at ^ ((key & 3) << 2) : ROW_BYTES == 128 ? at ^ ((key & 2) << 1) : at;
    return ROW_BYTES >= 256 ? at ^ ((key & 4) << 1) : at;
}

// e as a sum of two fp16 numbers, exact to 22 bits: pairs of `high` and `low`
__device__ __forceinline__ void two_terms(float e0, float e1, v2f16 &high, v2f16 &low) {
    high = __builtin_convertvector((v2f32{e0, e1}), v2f16);
    float minus = -1.f;
    asm("" : "+v"(minus));  // (as a constant it makes a conversion and a subtraction of one instruction)
    low = __builtin_convertvector((v2f32{fmaf((float) high[0], minus, e0), fmaf((float) high[1], minus, e1)}), v2f16);
}

// 32 N keys of K and V in LDS, keys of bits 0 in `visible` left out where not all of them are seen.  The product with V takes
// probabilities in 16 bits as sums of two numbers, so that a result is rounded once, at the end.  (As single numbers their error is as
// large as that rounding, 2^-12 of them on average, and one query would differ with the number of rows it comes with.)
template <typename T, int D, int N>
__device__ __forceinline__ void attend(Rows<T, D> &r, const unsigned char *k, const unsigned char *v, float scale, bool all,
                                       unsigned long long visible, int lane) {
    typedef Rows<T, D> R;
    const int col = lane & 31, half_wave = lane >> 5;
    v16f32 s[N];
    auto products = [&]() {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            s[n] = v16f32{};
            const int key = 32 * n + col;
#pragma unroll
            for (int t = 0; t < R::kSteps; ++t) {
                const v4f32 piece = *reinterpret_cast<const v4f32 *>(k + key * R::kRowBytes + k_piece<R::kRowBytes>(key, 2 * t + half_wave) * 16);
                if constexpr (sizeof(T) == 2) {
                    s[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8f16, piece), __builtin_bit_cast(v8f16, r.q[t]), s[n], 0, 0, 0);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[n] = __builtin_amdgcn_mfma_f32_32x32x2f32(piece[e], r.q[t][e], s[n], 0, 0, 0);
                }
            }
        }
        products_done();
        if (!all) {
#pragma unroll
            for (int n = 0; n < N; ++n) {
                const unsigned word = (unsigned) (visible >> (32 * n)) >> (4 * half_wave);
#pragma unroll
                for (int i = 0; i < 16; ++i) s[n][i] = word >> (8 * (i / 4) + i % 4) & 1u ? s[n][i] : -INFINITY;
            }
        }
    };
    // Sums are scaled anew only when some maximum has risen by a factor that a probability in 16 bits and the sums bear.
    auto rescale = [&](float top) {
        const float high = fmaxf(r.top, fmaxf(top, __shfl_xor(top, 32, kWave)));
        const float shrink = __builtin_amdgcn_exp2f((r.top - high) * scale);
        r.top = high;
        r.sum *= shrink;
#pragma unroll
        for (int d = 0; d < D / 32; ++d) r.ctx[d] *= shrink;
    };
    auto largest = [&]() {
        float top = s[0][0];
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i) top = fmaxf(top, s[n][i]);
        return top;
    };
    products();
    if constexpr (sizeof(T) == 2) {
        auto weigh = [&]() {
            float sum = 0.f;
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    s[n][i] = __builtin_amdgcn_exp2f(fmaf(s[n][i] - r.top, scale, Range<N>::kRaise));
                    sum += s[n][i];
                }
            return sum;
        };
        if constexpr (N == 1) {  // (for kernels that wait for memory)
            const float top = largest();
            if (__any((top - r.top) * scale > Range<N>::kSlack)) rescale(top);
            r.sum += weigh();
        } else {
            // Probabilities against the maximum so far, in the scores' place; their sum, which is wanted anyway, says whether it was
            // too small by far, and only then the scores are made again and their maximum is looked for.
            if (r.fresh) rescale(largest());
            r.fresh = false;
            float sum = weigh();
            if (__any(!(sum <= Range<N>::kMost))) {
                products();
                rescale(largest());
                sum = weigh();
            }
            r.sum += sum;
        }
        const int patch = lane & 15, side = (lane >> 4) & 1;
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
                v8f16 p, low;
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    v2f16 a, b;
                    two_terms(s[n][8 * ks + i], s[n][8 * ks + i + 1], a, b);
                    p[i] = a[0], p[i + 1] = a[1], low[i] = b[0], low[i + 1] = b[1];
                }
#pragma unroll
                for (int d = 0; d < D / 32; ++d) {
                    v4f16 part[2];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int key = 32 * n + 16 * ks + 8 * h + 4 * half_wave + patch / 4, at = 4 * d + 2 * side + (patch & 3) / 2;
                        part[h] = read_transposed(v + key * R::kRowBytes + v_piece<T, R::kRowBytes>(key, at) * 16 + (patch & 1) * 8);
                    }
                    const v8f16 a = __builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7);
                    r.ctx[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, low, r.ctx[d], 0, 0, 0);
                    r.ctx[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, p, r.ctx[d], 0, 0, 0);
                }
            }
    } else {
        const float top = largest();
        if (__any((top - r.top) * scale > kSlack)) rescale(top);
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[n][i] = __builtin_amdgcn_exp2f((s[n][i] - r.top) * scale);
                r.sum += s[n][i];
                const int key = 32 * n + 8 * (i / 4) + 4 * half_wave + i % 4;
#pragma unroll
                for (int d = 0; d < D / 32; ++d) {
                    const float a = *reinterpret_cast<const float *>(v + key * R::kRowBytes + v_piece<T, R::kRowBytes>(key, 8 * d + col / 4) * 16 +
                                                                     (col & 3) * 4);
                    r.ctx[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, s[n][i], r.ctx[d], 0, 0, 0);
                }
            }
    }
}

// At most 16 rows in fp32, whose matrix instructions take as long as four times the rows need: tiles of 16 x 16.  Lane l has row l % 16
// and, of every 16 keys or columns, the four from 4 (l / 16) on.  (8 x 1 over 4096 keys of 128, 4 rows: 56 us with tiles of 32, 40 with
// these; 32 x 1 over up to 4096 of 64, 1 row: 98 and 90, where the bytes take 78.)
template <int D>
struct FewRows {
    v4f32 q[D / 16], ctx[D / 16];
    float top, sum;

    __device__ __forceinline__ void load(const float *row, int quarter, bool negate) {
#pragma unroll
        for (int s = 0; s < D / 16; ++s) {
            q[s] = *reinterpret_cast<const v4f32 *>(row + 16 * s + 4 * quarter);
            if (negate) q[s] = -q[s];
            ctx[s] = v4f32{};
        }
        top = kNone, sum = 0.f;
    }
};

// 32 keys, those with bits 0 in `visible` left out unless all of them are seen
template <int D>
__device__ __forceinline__ void attend_few(FewRows<D> &r, const unsigned char *k, const unsigned char *v, float scale, bool all,
                                           unsigned visible, int lane) {
    constexpr int kRowBytes = D * 4;
    const int col = lane & 15, quarter = lane >> 4;
    v4f32 s[2] = {};
#pragma unroll
    for (int t = 0; t < D / 16; ++t) {
        v4f32 piece[2];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            const int key = 16 * n + col;
            piece[n] = *reinterpret_cast<const v4f32 *>(k + key * kRowBytes + k_piece<kRowBytes>(key, 4 * t + quarter) * 16);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int n = 0; n < 2; ++n) s[n] = __builtin_amdgcn_mfma_f32_16x16x4f32(piece[n][e], r.q[t][e], s[n], 0, 0, 0);
    }
    products_done();
    if (!all) {
        const unsigned word = visible >> (4 * quarter);
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[n][i] = word >> (16 * n + i) & 1u ? s[n][i] : -INFINITY;
    }
    float top = s[0][0];
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, s[n][i]);
    if (__any((top - r.top) * scale > kSlack)) {
        const float high = fmaxf(r.top, quarters_max(top)), shrink = __builtin_amdgcn_exp2f((r.top - high) * scale);
        r.top = high;
        r.sum *= shrink;
#pragma unroll
        for (int d = 0; d < D / 16; ++d) r.ctx[d] *= shrink;
    }
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            s[n][i] = __builtin_amdgcn_exp2f((s[n][i] - r.top) * scale);
            r.sum += s[n][i];
            const int key = 16 * n + 4 * quarter + i;
#pragma unroll
            for (int d = 0; d < D / 16; ++d) {
                const float a = *reinterpret_cast<const float *>(v + key * kRowBytes + v_piece<float, kRowBytes>(key, 4 * d + col / 4) * 16 + (col & 3) * 4);
                r.ctx[d] = __builtin_amdgcn_mfma_f32_16x16x4f32(a, s[n][i], r.ctx[d], 0, 0, 0);
            }
        }
}

__device__ __forceinline__ unsigned long long bits_below(int n) { return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1; }

// The keys that queries at the positions low..high of a sequence see between them, and those that each of them sees.
struct Reach {
    int first_begin, last_begin, first_end, last_end;  // of the window's bounds; sinks come on top
    bool any;

    __device__ __forceinline__ Reach(const WindowArgs &a, int low, int high, int length) {
        low = low < 0 ? 0 : low, high = high < length ? high : length - 1;
        any = low <= high;
        first_begin = low > a.left ? low - a.left : 0, last_begin = high > a.left ? high - a.left : 0;
        first_end = low < length - a.right ? low + a.right + 1 : length;  // (position + right may leave 32 bits)
        last_end = high < length - a.right ? high + a.right + 1 : length;
    }
    // of the keys base .. base + 63: what some query may see, leaving the mask aside
    __device__ __forceinline__ unsigned long long of(int base, int sinks) const {
        return bits_below(last_end - base) & (~bits_below(first_begin - base) | bits_below(sinks - base));
    }
    __device__ __forceinline__ void cut(int end) {  // nothing is seen from `end` on
        first_end = first_end < end ? first_end : end, last_end = last_end < end ? last_end : end;
    }
    __device__ __forceinline__ bool all(int base, int keys, int sinks) const {
        return base + keys <= first_end && (base >= last_begin || base + keys <= sinks);
    }
};

// Tiles of KEYS keys that a reach takes: those of the sinks, then those of the window.
template <int KEYS>
struct Tiles {
    int of_sinks, first, count;

    __device__ __forceinline__ Tiles(const Reach &reach, int sinks) {
        first = reach.first_begin / KEYS;
        const int end = (reach.last_end + KEYS - 1) / KEYS, far = sinks > reach.last_end ? reach.last_end : sinks;
        of_sinks = (far + KEYS - 1) / KEYS;
        of_sinks = of_sinks < first ? of_sinks : first;
        count = reach.any ? of_sinks + (end > first ? end - first : 0) : 0;
    }
    __device__ __forceinline__ int base(int tile) const { return (tile < of_sinks ? tile : tile - of_sinks + first) * KEYS; }
};

// 16 bytes per lane from `base` + `offset` to LDS at `to` + 16 * lane, without passing through registers.  As an instruction of its
// own, not the builtin: behind that the compiler lets every transposing read of LDS wait for all that is on its way, also to other
// buffers.  The waits are the callers' (landed, and the ones that count).  The compiler does not look into the statement, so it has the
// five states that a load needs behind a vector instruction that wrote its scalar base (one, behind m0), and leaves m0 as it was.
__device__ __forceinline__ void copy_to_lds(const char *base, unsigned offset, unsigned to) {
    unsigned m0;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 2\n\tglobal_load_lds_dwordx4 %2, %3\n\ts_mov_b32 m0, %0"
                 : "=&s"(m0)
                 : "s"(to), "v"(offset), "s"(base)
                 : "memory");
}

__device__ __forceinline__ unsigned lds_address(const unsigned char *p) {
    return (unsigned) (uintptr_t) (const __attribute__((address_space(3))) unsigned char *) p;
}

// Whole 16-byte pieces of KEYS rows, brought to LDS by WAVES wavefronts: where a lane's pieces are in a tile, and the requests for a
// tile from row `base` on; rows past the last are read from it.
template <typename T, int D, int KEYS, int WAVES, bool IS_V>
struct Bring {
    static constexpr int kRowBytes = D * (int) sizeof(T), kPieces = kRowBytes / 16, kRequests = KEYS * kPieces / (kWave * WAVES);
    static_assert(KEYS * kPieces % (kWave * WAVES) == 0, "whole requests");
    unsigned offset[kRequests];

    __device__ __forceinline__ static unsigned offset_of(int i, int wave, int lane, int last, unsigned pitch) {
        const int at = (i * WAVES + wave) * kWave + lane, key = at / kPieces, place = at % kPieces;
        const int piece = IS_V ? v_piece<T, kRowBytes>(key, place) : k_piece<kRowBytes>(key, place);  // (its own inverse)
        return (unsigned) (key < last ? key : last) * pitch + piece * 16;
    }
    __device__ __forceinline__ Bring(int wave, int lane, unsigned pitch) {
#pragma unroll
        for (int i = 0; i < kRequests; ++i) offset[i] = offset_of(i, wave, lane, KEYS, pitch);
    }
    __device__ __forceinline__ void operator()(const T *from, int base, int rows, unsigned pitch, unsigned to, int wave, int lane) const {
        const char *tile = reinterpret_cast<const char *>(from) + (size_t) base * pitch;
        if (base + KEYS <= rows) {
#pragma unroll
            for (int i = 0; i < kRequests; ++i) copy_to_lds(tile, offset[i], to + (i * WAVES + wave) * 1024);
        } else {
#pragma unroll
            for (int i = 0; i < kRequests; ++i)
                copy_to_lds(tile, offset_of(i, wave, lane, rows - 1 - base, pitch), to + (i * WAVES + wave) * 1024);
        }
    }
};

// A key that nobody sees has probability 0, but 0 times what its row of V may hold need not be 0.  A wavefront clears these rows, one at a
// time where they are few (holes in a mask).
template <typename T, int D, int KEYS>
__device__ __forceinline__ void clear_rows(unsigned char *v, unsigned long long seen, int lane) {
    constexpr int kPieces = D * (int) sizeof(T) / 16;
    unsigned long long unseen = ~seen & (KEYS == 64 ? ~0ull : (1ull << (KEYS % 64)) - 1);
    if (__builtin_popcountll(unseen) <= 12) {
        for (; unseen != 0; unseen &= unseen - 1)
            if (lane < kPieces) *reinterpret_cast<v4f32 *>(v + (__builtin_ctzll(unseen) * kPieces + lane) * 16) = v4f32{};
    } else {
#pragma unroll
        for (int i = 0; i < KEYS * kPieces / kWave; ++i) {
            const int at = i * kWave + lane;
            if (!(seen >> (at / kPieces) & 1ull)) *reinterpret_cast<v4f32 *>(v + at * 16) = v4f32{};
        }
    }
    asm volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();
}

// A bound of the keys below `end` that the mask keeps (padding is given as a mask, and is not to be computed): behind the last one, or,
// where that is far, up to 16 behind it.
__device__ __forceinline__ int kept_end(const int8_t *mask, int end, int lane) {
    int byte[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int j = end - 1 - (64 * i + lane);
        byte[i] = mask[j > 0 ? j : 0];
        byte[i] = j >= 0 ? byte[i] : 0;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const unsigned long long kept = __ballot(byte[i] != 0);
        if (kept != 0) return end - 64 * i - __builtin_ctzll(kept);
    }
    if (end <= 512) return 0;
    end -= 512;
    end += -(int) (uintptr_t) (mask + end) & 15;  // to whole 16-byte pieces, with some bytes seen already
    for (; end >= 16; end -= 4096) {
        v4i32 piece[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int j = end - 16 * (64 * i + lane + 1);
            piece[i] = j >= 0 ? *reinterpret_cast<const v4i32 *>(mask + j) : v4i32{};
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const unsigned long long kept = __ballot((piece[i][0] | piece[i][1] | piece[i][2] | piece[i][3]) != 0);
            if (kept != 0) return end - 16 * (64 * i + __builtin_ctzll(kept));
        }
        if (end <= 4096) return end & 15;  // (bytes before the first whole piece)
    }
    return end;
}

struct Problem {
    int b, kv_head, length, first;

    __device__ __forceinline__ Problem(const WindowArgs &a, int b_, int kv_head_) : b(b_), kv_head(kv_head_) {
        length = a.lengths != nullptr ? clamp_to(a.lengths[b], 0, a.kv_rows) : a.kv_rows;
        first = a.first != nullptr ? clamp_to(a.first[b], -kFar, kFar) : 0;
    }
};

template <typename T>
__device__ __forceinline__ void store4(T *to, float a, float b, float c, float d) {
    store_vec<T, 4>(to, Vec<T, 4>{from_f32<T>(a), from_f32<T>(b), from_f32<T>(c), from_f32<T>(d)});
}

__device__ __forceinline__ void landed() {  // what this wavefront requested is in LDS
    wait_loads<0>();
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");
}

// Which rows a workgroup takes, `rows` of them.  Workgroups are handed to the eight dies in turn and to the units of a die as they come free, so
// the ones with work come first: handed out with the others between them, which end at once, one unit got 8 of 1280 and another 2
// (4 sequences of 1024 to 4096 tokens, 99 us for 56 us of work).  A die has consecutive ones, which read the same keys.
struct Place {
    int b, kv_head, tile;

    // `count` things, those of a die consecutive: the number of the die's first one
    __device__ __forceinline__ static int before(int count, int die) { return die * (count / 8) + (die < count % 8 ? die : count % 8); }

    __device__ __forceinline__ Place(const WindowArgs &a, int share, int rows, int row_tiles, int block, int lane) {
        const int die = block % 8, on_die = block / 8, total = a.batch * a.kv_heads * row_tiles;
        if ((a.lengths == nullptr && a.first == nullptr) || a.batch > kWave) {
            const int i = before(total, die) + on_die, problem = i / row_tiles;
            tile = i - problem * row_tiles, b = problem / a.kv_heads, kv_head = problem - b * a.kv_heads;
            return;
        }
        // a lane per sequence: the tiles with a query inside of it
        int from = 0, count = 0;
        if (lane < a.batch) {
            const int length = a.lengths != nullptr ? clamp_to(a.lengths[lane], 0, a.kv_rows) : a.kv_rows;
            const int first = a.first != nullptr ? clamp_to(a.first[lane], -kFar, kFar) : 0;
            const int low = first < 0 ? -first : 0, high = length - first < a.q_rows ? length - first : a.q_rows;
            if (low < high) from = low * share / rows, count = (high * share + rows - 1) / rows - from;
        }
        int active = 0;
        for (int n = 0; n < a.batch; ++n) active += __builtin_amdgcn_readlane(count, n);
        active *= a.kv_heads;
        const int mine = before(active, die + 1) - before(active, die);
        const bool works = on_die < mine;
        int i = works ? before(active, die) + on_die : before(total, die) - before(active, die) + on_die - mine;
        int n = 0;  // tiles of a sequence and key head
        for (b = 0; b < a.batch; ++b) {
            n = __builtin_amdgcn_readlane(count, b);
            n = works ? n : row_tiles - n;
            if (i < n * a.kv_heads) break;
            i -= n * a.kv_heads;
        }
        const int begin = __builtin_amdgcn_readlane(from, b);
        kv_head = i / n;
        tile = i - kv_head * n;
        tile += works ? begin : tile < begin ? 0 : __builtin_amdgcn_readlane(count, b);
        // (the same in every lane, which the compiler has to be told)
        b = __builtin_amdgcn_readfirstlane(b), kv_head = __builtin_amdgcn_readfirstlane(kv_head), tile = __builtin_amdgcn_readfirstlane(tile);
    }
};

// What a workgroup of four wavefronts works on, KEYS keys at a time: its rows, and which tiles of keys they reach.  A wavefront has
// 32 rows and, where only ROWS / 32 of them have rows of their own, one of the parts of a tile.
template <typename T, int D, int KEYS, int ROWS>
struct Strip {
    static constexpr int kRowGroups = ROWS / 32, kParts = 4 / kRowGroups;
    const WindowArgs &a;
    int share, rows, row0, row, query, head, begin, end;  // this wavefront's first row; a lane's, its query and head, the bounds of its window
    int pieces, piece;  // of the axis, and which one this is
    Place place;
    Problem at;
    bool there;
    Reach reach, mine;  // of the workgroup's rows, and of this wavefront's
    const int8_t *mask;
    Tiles<KEYS> tiles;
    int low, high;  // the piece's tiles
    const T *k, *v;

    __device__ __forceinline__ static int last_of(int row, int count, int rows) { return (row + count < rows ? row + count : rows) - 1; }
    __device__ __forceinline__ Strip(const WindowArgs &args, int row_tiles, int pieces_, int wave, int lane)
        : a(args), share(a.heads / a.kv_heads), rows(a.q_rows * share), row0(0), pieces(pieces_), piece(pieces == 1 ? 0 : blockIdx.x * pieces / gridDim.x),
          place(a, share, ROWS, row_tiles, blockIdx.x - piece * (gridDim.x / pieces), lane),
          at(a, place.b, place.kv_head), reach(a, at.first + place.tile * ROWS / share, at.first + last_of(place.tile * ROWS, ROWS, rows) / share, at.length),
          mine(a, at.first + (place.tile * ROWS + 32 * (wave % kRowGroups)) / share,
               at.first + last_of(place.tile * ROWS + 32 * (wave % kRowGroups), 32, rows) / share, at.length),
          mask(a.mask != nullptr ? a.mask + (size_t) at.b * a.kv_rows : nullptr), tiles(cut_to_mask(lane), a.sinks) {
        row0 = place.tile * ROWS + 32 * (wave % kRowGroups), row = row0 + (lane & 31);
        mine.any = mine.any && row0 < rows;
        const int my_row = row < rows ? row : rows - 1;
        query = share == 1 ? my_row : my_row / share, head = at.kv_head * share + my_row - query * share;
        const int p = at.first + query;
        there = row < rows && p >= 0 && p < at.length;
        begin = p > a.left ? p - a.left : 0, end = p < at.length - a.right ? p + a.right + 1 : at.length;
        k = (const T *) a.k + (size_t) at.b * a.kv_rows * a.ldkv + at.kv_head * D;
        v = (const T *) a.v + (size_t) at.b * a.kv_rows * a.ldkv + at.kv_head * D;
        low = 0, high = tiles.count;
        if (pieces > 1) {
            const int each = tiles.count / pieces, more = tiles.count - each * pieces;
            low = piece * each + (piece < more ? piece : more), high = low + each + (piece < more ? 1 : 0);
        }
    }
    __device__ __forceinline__ const Reach &cut_to_mask(int lane) {
        if (mask != nullptr && reach.any) {
            const int kept = kept_end(mask, reach.last_end, lane);
            reach.cut(kept), mine.cut(kept);
        }
        return reach;
    }
    __device__ __forceinline__ const T *q() const { return (const T *) a.q + ((size_t) at.b * a.q_rows + query) * a.ldq + (size_t) head * D; }
    __device__ __forceinline__ int mask_byte(int key) const { return mask != nullptr && key < a.kv_rows ? mask[key] : 1; }
    // of the keys base .. base + 63 that the mask keeps, those that this lane's row sees
    __device__ __forceinline__ unsigned long long visible(int base, unsigned long long kept) const {
        return bits_below(end - base) & (~bits_below(begin - base) | bits_below(a.sinks - base)) & kept;
    }
    // take(tile, busy) for every tile of the workgroup's piece, in order.  This wavefront's are those of the sinks (which reach into the
    // window's where there is no gap between them) and a run among those of the window.  (Tiles passed over by loops of their own:
    // a branch around the work has the compiler copy every accumulator.)
    template <typename Take>
    __device__ __forceinline__ void walk(Take take) const {
        const int my_sinks = a.sinks < mine.last_end ? a.sinks : mine.last_end, sinks_end = mine.any && my_sinks > 0 ? (my_sinks + KEYS - 1) / KEYS : 0;
        int from = mine.any ? tiles.of_sinks + mine.first_begin / KEYS - tiles.first : tiles.count;
        int until = mine.any ? tiles.of_sinks + (mine.last_end + KEYS - 1) / KEYS - tiles.first : tiles.count;
        from = from < high ? from : high, until = until < high ? until : high;
        const int sinks_until = sinks_end < high ? sinks_end : high;
        int tile = low;
        for (int part = 0; part < 2; ++part) {
            for (; tile < (part == 0 ? low : from); ++tile) take(tile, false);
            for (; tile < (part == 0 ? sinks_until : until); ++tile) take(tile, true);
        }
        for (; tile < high; ++tile) take(tile, false);
    }
    // The rows' results: sums relative to their maxima, of all parts of the tiles, which meet in LDS (`traded`, kTraded bytes) in order.
    static constexpr int kPitch = D + 4, kTraded = (kParts - 1) * ROWS * kPitch * 4;
    __device__ __forceinline__ void store(v16f32 (&sums)[D / 32], float top, float sum, unsigned char *traded, int wave, int lane) const {
        const int half_wave = lane >> 5;
        products_done();
        sum += __shfl_xor(sum, 32, kWave);
        if constexpr (kParts > 1) {
            static_assert(kParts == 2, "one other part");
            float *with = reinterpret_cast<float *>(traded) + (32 * (wave % kRowGroups) + (lane & 31)) * kPitch;
            __syncthreads();  // nobody reads tiles any more
            if (wave >= kRowGroups) {
#pragma unroll
                for (int d = 0; d < D / 32; ++d)
#pragma unroll
                    for (int i = 0; i < 16; i += 4)
                        *reinterpret_cast<v4f32 *>(with + 32 * d + 2 * i + 4 * half_wave) = v4f32{sums[d][i], sums[d][i + 1], sums[d][i + 2], sums[d][i + 3]};
                if (half_wave == 0) with[D] = top, with[D + 1] = sum;
            }
            __syncthreads();
            if (wave >= kRowGroups) return;
            const float other = with[D], high = fmaxf(top, other);
            const float mine_by = __builtin_amdgcn_exp2f((top - high) * a.scale), other_by = __builtin_amdgcn_exp2f((other - high) * a.scale);
            sum = sum * mine_by + with[D + 1] * other_by, top = high;
#pragma unroll
            for (int d = 0; d < D / 32; ++d)
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                    const v4f32 x = *reinterpret_cast<const v4f32 *>(with + 32 * d + 2 * i + 4 * half_wave);
#pragma unroll
                    for (int e = 0; e < 4; ++e) sums[d][i + e] = sums[d][i + e] * mine_by + x[e] * other_by;
                }
        }
        if (row >= rows) return;
        if (pieces > 1) {
            const size_t tile32 = (size_t) (at.b * a.kv_heads + at.kv_head) * ((rows + ROWS - 1) / ROWS * kRowGroups) + row0 / 32;
            float *out = a.partials + ((tile32 * pieces + piece) * 32 + (lane & 31)) * kPitch;
#pragma unroll
            for (int d = 0; d < D / 32; ++d)
#pragma unroll
                for (int i = 0; i < 16; i += 4)
                    *reinterpret_cast<v4f32 *>(out + 32 * d + 2 * i + 4 * half_wave) =
                            there ? v4f32{sums[d][i], sums[d][i + 1], sums[d][i + 2], sums[d][i + 3]} : v4f32{};
            if (half_wave == 0) out[D] = there ? top : kNone, out[D + 1] = there ? sum : 0.f;
            return;
        }
        const float by = there && sum != 0.f ? 1.f / sum : 0.f;  // (a sum that is no number stays none)
        T *ctx = (T *) a.ctx + ((size_t) at.b * a.q_rows + query) * a.ld_ctx + (size_t) head * D + 4 * half_wave;
#pragma unroll
        for (int d = 0; d < D / 32; ++d)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                if (by != 0.f) store4(ctx + 32 * d + 2 * i, sums[d][i] * by, sums[d][i + 1] * by, sums[d][i + 2] * by, sums[d][i + 3] * by);
                else store4(ctx + 32 * d + 2 * i, 0.f, 0.f, 0.f, 0.f);
            }
    }
};

// fp16, many rows, bound by exponentials and what else the probabilities take, matrix instructions and reads of LDS, that three wavefronts to
// a SIMD overlap in part: 4 x up to 4096 tokens of 16 heads of 64, window 512, 39 Gflop in 97 us (400 Tflop/s); 2 x 4096 causal tokens of
// 16 heads of 128, 137 Gflop in 265 us (520).  (The probabilities in one fp16 term each: 88 and 214 us, with a second rounding as
// large as that of the results.)  Four wavefronts share every tile of K and V, the next one on its way while they work on this
// one.  (Two on their way: 80 and 77 us, but 214 and 280 for heads of 128, with one term.)  A wavefront has 64
// keys of a tile with its 32 rows: ROWS = 128, the same ones for all, 64, either half of 128.
template <int D, int ROWS>
__global__ __launch_bounds__(kBlock, D == 128 ? 2 : 1) void attention_window_shared_kernel(WindowArgs a, int row_tiles) {
    typedef half_t T;
    constexpr int kKeys = 64 * 128 / ROWS, kTileBytes = kKeys * D * (int) sizeof(T), kPartBytes = 64 * D * (int) sizeof(T);
    typedef Strip<T, D, kKeys, ROWS> Work;
    extern __shared__ __align__(16) unsigned char smem[];  // two buffers of K and V
    static_assert(4 * kTileBytes >= Work::kTraded, "room for what is traded");
    const int wave = wave_in_block(), lane = threadIdx.x & (kWave - 1), part = wave / Work::kRowGroups;
    const Work strip(a, row_tiles, 1, wave, lane);  // (an axis in one piece)
    const unsigned pitch = (unsigned) a.ldkv * sizeof(T), lds = lds_address(smem);
    const Bring<T, D, kKeys, 4, false> bring_k(wave, lane, pitch);
    const Bring<T, D, kKeys, 4, true> bring_v(wave, lane, pitch);
    auto bring = [&](int tile, int buffer) {
        const unsigned to = lds + buffer * 2 * kTileBytes;
        bring_k(strip.k, strip.tiles.base(tile), a.kv_rows, pitch, to, wave, lane);
        bring_v(strip.v, strip.tiles.base(tile), a.kv_rows, pitch, to + kTileBytes, wave, lane);
    };
    int kept = 1;
    if (strip.low < strip.high) {
        bring(strip.low, strip.low & 1);
        kept = strip.mask_byte(strip.tiles.base(strip.low) + 64 * part + lane);
    }
    Rows<T, D> r;
    r.load(strip.q(), lane >> 5, a.negate);
    // One tile of the workgroup's: everybody waits for it, brings a share of the next one and, `busy`, works on it.
    strip.walk([&](int tile, bool busy) {
        landed();
        const unsigned long long kept_bits = strip.mask != nullptr ? __ballot(kept != 0) : ~0ull;
        __syncthreads();  // everybody's; and nobody reads the other buffer any more
        if (tile + 1 < strip.high) {
            bring(tile + 1, (tile + 1) & 1);
            kept = strip.mask_byte(strip.tiles.base(tile + 1) + 64 * part + lane);
        }
        if (!busy) return;
        unsigned char *kt = smem + (tile & 1) * 2 * kTileBytes + part * kPartBytes, *vt = kt + kTileBytes;
        const int base = strip.tiles.base(tile) + 64 * part;
        const bool all = kept_bits == ~0ull && strip.mine.all(base, 64, a.sinks);
        unsigned long long visible = ~0ull;
        if (!all) {
            visible = strip.visible(base, kept_bits);
            // (each wavefront that reads these rows clears them, with the same zeros)
            const unsigned long long seen = strip.reach.of(base, a.sinks) & kept_bits;
            if (seen != ~0ull) clear_rows<T, D, 64>(vt, seen, lane);
        }
        attend<T, D, 2>(r, kt, vt, a.scale, all, visible, lane);
    });
    strip.store(r.ctx, r.top, r.sum, smem, wave, lane);
}

// ---- fp32, many rows ------------------------------------------------------
// An fp32 number is the sum of three bf16 numbers, each the nearest to what those before it leave: the second is at most 2^-8 of the
// leading power of two, the third at most 2^-17, and nothing is left.  Of the nine products of two such sums the three smallest are
// left out, 2 * 2^-25 of the product together and of either sign; the six others run on the bf16 matrix cores, whose rate is sixteen times that
// of fp32's, with fp32 sums.  (Terms cut off instead of rounded take as many instructions, but leave out up to 2^-21, always of the product's
// sign.)  V's first term is cut off, because the nearest to the largest fp32 numbers is infinite; its second is then at most 2^-7 and its third
// 2^-16, and what is left out of its products with probabilities 2 * 2^-24.  K and V are taken apart on their way into LDS, once for the
// four wavefronts that read them; the probabilities in their lanes.

typedef __bf16 v8bf16 __attribute__((ext_vector_type(8)));
typedef unsigned v2u32 __attribute__((ext_vector_type(2)));
typedef unsigned v4u32 __attribute__((ext_vector_type(4)));

typedef __bf16 v2bf16 __attribute__((ext_vector_type(2)));

// The next terms of two numbers, and in their place what those leave; CUT: the leading bits as they are.  (Of an infinity a NaN is left, and
// an infinite term times a term of 0 is one as well: scores that are none are made again from the numbers themselves, below.  Of an infinite V
// both are as good: what sees it is not finite.)
template <bool CUT>
__device__ __forceinline__ unsigned next_terms(float &a, float &b) {
    unsigned pair;
    if constexpr (CUT) pair = __builtin_amdgcn_perm(__builtin_bit_cast(unsigned, b), __builtin_bit_cast(unsigned, a), 0x07060302u);
    else pair = __builtin_bit_cast(unsigned, __builtin_convertvector((v2f32{a, b}), v2bf16));
    a -= __builtin_bit_cast(float, pair << 16), b -= __builtin_bit_cast(float, pair & 0xffff0000u);
    return pair;
}

struct Terms {  // of 8 numbers
    v8bf16 t[3];

    __device__ __forceinline__ Terms() {}
    __device__ __forceinline__ explicit Terms(const float (&x)[8]) {
        v4u32 r[3];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float a = x[2 * i], b = x[2 * i + 1];
#pragma unroll
            for (int n = 0; n < 3; ++n) r[n][i] = next_terms<false>(a, b);
        }
#pragma unroll
        for (int n = 0; n < 3; ++n) t[n] = __builtin_bit_cast(v8bf16, r[n]);
    }
};

// sums + one of the six products of a and b, of which the smallest come first
__device__ __forceinline__ v16f32 multiply_term(int m, const v8bf16 (&a)[3], const v8bf16 (&b)[3], v16f32 sums) {
    constexpr int kA[6] = {2, 1, 0, 1, 0, 0}, kB[6] = {0, 1, 2, 0, 1, 0};
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[kA[m]], b[kB[m]], sums, 0, 0, 0);
}

// The largest, or a NaN where there is one (fmaxf takes the number).
__device__ __forceinline__ float largest_or_nan(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// Bound by the matrix instructions and, next to them, by taking K and V apart and reading the terms: 16 x 512 tokens of 16 heads of 64, 17
// Gflop in 110 to 119 us, 150 Tflop/s, what a large fp32 matrix product reaches on fp32's own matrix instructions.
// As above; a wavefront has 32 keys of a tile with its 32 rows: ROWS = 128, the same ones for all, 64, either half of 64.
template <int D, int ROWS>
__global__ __launch_bounds__(kBlock, D == 128 ? 1 : 2) void attention_window_terms_kernel(WindowArgs a, int row_tiles, int pieces) {
    constexpr int kKeys = 32 * 128 / ROWS, kRowBytes = 2 * D, kPlane = kKeys * kRowBytes, kQuads = D / 4, kMine = kKeys * kQuads / kBlock;
    typedef Strip<float, D, kKeys, ROWS> Work;
    extern __shared__ __align__(16) unsigned char smem[];
    static_assert(6 * kPlane >= Work::kTraded, "room for what is traded");
    unsigned char *planes = smem;  // of K, then of V
    const int wave = wave_in_block(), lane = threadIdx.x & (kWave - 1), col = lane & 31, half_wave = lane >> 5;
    const int part = wave / Work::kRowGroups;
    const Work strip(a, row_tiles, pieces, wave, lane);
    // a thread's pieces of a tile: 16 bytes of `kMine` rows of K and of V
    v4f32 next[2][kMine];
    const unsigned pitch = (unsigned) a.ldkv * 4u;
    auto offset_of = [&](int i, int last) {
        const int at = i * kBlock + threadIdx.x, key = at / kQuads;
        return (unsigned) (key < last ? key : last) * pitch + at % kQuads * 16;
    };
    unsigned offset[kMine];
#pragma unroll
    for (int i = 0; i < kMine; ++i) offset[i] = offset_of(i, kKeys);
    auto bring = [&](int tile) {
        const int base = strip.tiles.base(tile);
        const char *k = (const char *) strip.k + (size_t) base * pitch, *v = (const char *) strip.v + (size_t) base * pitch;
        const bool whole = base + kKeys <= a.kv_rows;  // (rows past the last are read from it)
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
            const unsigned from = whole ? offset[i] : offset_of(i, a.kv_rows - 1 - base);
            next[0][i] = *reinterpret_cast<const v4f32 *>(k + from);
            next[1][i] = *reinterpret_cast<const v4f32 *>(v + from);
        }
    };
    int kept = 1;
    if (strip.low < strip.high) {
        bring(strip.low);
        kept = strip.mask_byte(strip.tiles.base(strip.low) + lane);
    }
    Terms q[D / 16];
    {
        const float *from = strip.q() + 8 * half_wave;
#pragma unroll
        for (int t = 0; t < D / 16; ++t) {
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = a.negate ? -from[16 * t + e] : from[16 * t + e];
            q[t] = Terms(x);
        }
    }
    v16f32 ctx[D / 32] = {};
    float top = kNone, sum = 0.f;
    const int patch = lane & 15, side = (lane >> 4) & 1;

    strip.walk([&](int tile, bool busy) {
        const unsigned long long kept_bits = strip.mask != nullptr ? __ballot(kept != 0) : ~0ull;
        const int base = strip.tiles.base(tile) + 32 * part;
        const unsigned long long seen = strip.reach.of(strip.tiles.base(tile), a.sinks) & kept_bits;
        __syncthreads();  // nobody reads the tile before any more
#pragma unroll
        for (int w = 0; w < 2; ++w)
#pragma unroll
            for (int i = 0; i < kMine; ++i) {
                const int at = i * kBlock + threadIdx.x, key = at / kQuads, quad = at % kQuads;
                // (a key that nobody sees has probability 0, but 0 times what its row of V may hold need not be 0)
                const bool use = w == 0 || (seen >> key & 1ull);
                float x[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = use ? next[w][i][e] : 0.f;
                const int piece = w == 0 ? k_piece<kRowBytes>(key, quad / 2) : v_piece<half_t, kRowBytes>(key, quad / 2);
                unsigned char *to = planes + w * 3 * kPlane + key * kRowBytes + piece * 16 + (quad & 1) * 8;
                *reinterpret_cast<v2u32 *>(to) = w == 0 ? v2u32{next_terms<false>(x[0], x[1]), next_terms<false>(x[2], x[3])}
                                                        : v2u32{next_terms<true>(x[0], x[1]), next_terms<true>(x[2], x[3])};
#pragma unroll
                for (int n = 1; n < 3; ++n)
                    *reinterpret_cast<v2u32 *>(to + n * kPlane) = v2u32{next_terms<false>(x[0], x[1]), next_terms<false>(x[2], x[3])};
            }
        if (tile + 1 < strip.high) {
            bring(tile + 1);
            kept = strip.mask_byte(strip.tiles.base(tile + 1) + lane);
        }
        __syncthreads();
        if (!busy) return;
        const unsigned kept_part = (unsigned) (kept_bits >> (32 * part));
        const bool all = kept_part == ~0u && strip.mine.all(base, 32, a.sinks);
        // (two sums in turn: a product waits for the one before it in its sum)
        v16f32 s = {}, odd = {};
#pragma unroll
        for (int t = 0; t < D / 16; t += 2) {
            v8bf16 k[2][3];
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int n = 0; n < 3; ++n)
                    k[u][n] = *reinterpret_cast<const v8bf16 *>(planes + n * kPlane + (32 * part + col) * kRowBytes +
                                                                k_piece<kRowBytes>(col, 2 * (t + u) + half_wave) * 16);
#pragma unroll
            for (int m = 0; m < 6; ++m) {
                s = multiply_term(m, k[0], q[t].t, s);
                odd = multiply_term(m, k[1], q[t + 1].t, odd);
            }
        }
        products_done();
        s += odd;
        unsigned word = ~0u;
        if (!all) {
            word = (unsigned) strip.visible(base, kept_part) >> (4 * half_wave);
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = word >> (8 * (i / 4) + i % 4) & 1u ? s[i] : -INFINITY;
        }
        float high = s[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) high = largest_or_nan(high, s[i]);
        if (__any(!((high - top) * a.scale <= kSlack))) {
            if (__any(high != high)) {
                // Something infinite, or no number: these scores from Q and K themselves.  An infinite K against a q of the other sign is a
                // score of -infinity and no more.
                const float *qr = strip.q();
#pragma unroll 1
                for (int i = 0; i < 16; ++i) {
                    float score = s[0];
#pragma unroll
                    for (int j = 1; j < 16; ++j) score = i == j ? s[j] : score;
                    const int at = 8 * (i / 4) + i % 4;
                    if (score != score && (word >> at & 1u)) {
                        const float *kr = strip.k + (size_t) (base + 4 * half_wave + at) * a.ldkv;
                        score = 0.f;
#pragma unroll 1
                        for (int d = 0; d < D; ++d) score = fmaf(a.negate ? -qr[d] : qr[d], kr[d], score);
                    }
#pragma unroll
                    for (int j = 0; j < 16; ++j) s[j] = i == j ? score : s[j];
                }
                high = s[0];
#pragma unroll
                for (int i = 1; i < 16; ++i) high = fmaxf(high, s[i]);
            }
            high = fmaxf(top, fmaxf(high, __shfl_xor(high, 32, kWave)));
            const float shrink = __builtin_amdgcn_exp2f((top - high) * a.scale);
            top = high;
            sum *= shrink;
#pragma unroll
            for (int d = 0; d < D / 32; ++d) ctx[d] *= shrink;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            s[i] = __builtin_amdgcn_exp2f((s[i] - top) * a.scale);
            sum += s[i];
        }
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = s[8 * ks + e];
            const Terms p(x);
            constexpr int kTogether = D == 32 ? 1 : 2;  // columns of 32 whose sums take turns
#pragma unroll
            for (int d = 0; d < D / 32; d += kTogether) {
                v8bf16 v[kTogether][3];
#pragma unroll
                for (int u = 0; u < kTogether; ++u)
#pragma unroll
                    for (int n = 0; n < 3; ++n) {
                        v4f16 from[2];
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const int key = 16 * ks + 8 * h + 4 * half_wave + patch / 4, at = 4 * (d + u) + 2 * side + (patch & 3) / 2;
                            from[h] = read_transposed(planes + (3 + n) * kPlane + (32 * part + key) * kRowBytes +
                                                      v_piece<half_t, kRowBytes>(key, at) * 16 + (patch & 1) * 8);
                        }
                        v[u][n] = __builtin_bit_cast(v8bf16, __builtin_shufflevector(from[0], from[1], 0, 1, 2, 3, 4, 5, 6, 7));
                    }
#pragma unroll
                for (int m = 0; m < 6; ++m)
#pragma unroll
                    for (int u = 0; u < kTogether; ++u) ctx[d + u] = multiply_term(m, v[u], p.t, ctx[d + u]);
            }
        }
    });
    strip.store(ctx, top, sum, smem, wave, lane);
}

template <typename T, int D>
struct Spread {
    static constexpr int kTileBytes = 32 * D * (int) sizeof(T);                // of K, and of V
    // (two where two workgroups with them fit a compute unit: 32 tokens over 4096 keys of 128, fp16, 62 us with one workgroup of two
    // buffers to a wavefront, 54 with two of one)
    static constexpr int kBuffers = kTileBytes * 2 * 2 * 4 <= 64 * 1024 ? 2 : 1;
    static constexpr int kWaveBytes = kBuffers * 2 * kTileBytes;
    static constexpr int kPitch = D + 4;                                       // floats between rows of a wavefront's results
    static constexpr int kMergeBytes = 4 * 32 * kPitch * 4;
    static constexpr int kLds = 4 * kWaveBytes > kMergeBytes ? 4 * kWaveBytes : kMergeBytes;
};

// Few rows, bound by reading K and V: 32 tokens over up to 4096 keys of 4 heads of 128 in fp16, 219 MB in 50 us (4.4 TB/s); 1 token over
// 131072 keys of 2 heads, 134 MB in 26 us (5.2 TB/s), and 4.3 us for the join.  32 rows per workgroup, whose four wavefronts take every
// fourth tile of 32 keys of this workgroup's piece of the axis; their sums meet in LDS, in wavefront order, and go out as results or, where
// the axis is cut, as sums for the kernel below.
template <typename T, int D, bool FEW>
struct SpreadRows {
    typedef Rows<T, D> type;
};
template <typename T, int D>
struct SpreadRows<T, D, true> {
    typedef FewRows<D> type;
};

// FEW: at most 16 rows in fp32.
template <typename T, int D, bool FEW>
__global__ __launch_bounds__(kBlock, sizeof(T) * D == 512 && !FEW ? 1 : 2) void attention_window_spread_kernel(WindowArgs a, int row_tiles, int pieces) {
    typedef Spread<T, D> S;
    constexpr int kRows = FEW ? 16 : 32;
    extern __shared__ __align__(16) unsigned char smem[];
    const int wave = wave_in_block(), lane = threadIdx.x & (kWave - 1);
    const int piece = blockIdx.x % pieces, tile_at = blockIdx.x / pieces;
    const int problem = tile_at / row_tiles, row0 = (tile_at - problem * row_tiles) * 32;
    const Problem at(a, problem / a.kv_heads, problem % a.kv_heads);
    const int share = a.heads / a.kv_heads, rows = a.q_rows * share;
    const int row = row0 + (lane & (kRows - 1)), my_row = row < rows ? row : rows - 1;
    const int query = my_row / share, head = at.kv_head * share + my_row - query * share;
    const int p = at.first + query;
    const int begin = p > a.left ? p - a.left : 0, end = p < at.length - a.right ? p + a.right + 1 : at.length;

    const T *k = (const T *) a.k + (size_t) at.b * a.kv_rows * a.ldkv + at.kv_head * D;
    const T *v = (const T *) a.v + (size_t) at.b * a.kv_rows * a.ldkv + at.kv_head * D;
    const int8_t *mask = a.mask != nullptr ? a.mask + (size_t) at.b * a.kv_rows : nullptr;
    const int last_row = (row0 + 32 < rows ? row0 + 32 : rows) - 1;
    Reach reach(a, at.first + row0 / share, at.first + last_row / share, at.length);
    if (mask != nullptr && reach.any) reach.cut(kept_end(mask, reach.last_end, lane));
    const Tiles<32> tiles(reach, a.sinks);

    typename SpreadRows<T, D, FEW>::type r;
    r.load((const T *) a.q + ((size_t) at.b * a.q_rows + query) * a.ldq + (size_t) head * D, lane / kRows, a.negate);
    unsigned char *buffers = smem + wave * S::kWaveBytes;
    // pieces of the axis: whole tiles, the first ones one more where they do not divide
    const int each = tiles.count / pieces, more = tiles.count - each * pieces;
    const int until = piece * each + (piece < more ? piece : more) + each + (piece < more ? 1 : 0);
    int tile = piece * each + (piece < more ? piece : more) + wave;
    const unsigned pitch = (unsigned) a.ldkv * sizeof(T), lds = lds_address(buffers);
    const Bring<T, D, 32, 1, false> bring_k(0, lane, pitch);
    const Bring<T, D, 32, 1, true> bring_v(0, lane, pitch);
    auto bring = [&](int t, int buffer) {
        const unsigned to = lds + buffer * 2 * S::kTileBytes;
        bring_k(k, tiles.base(t), a.kv_rows, pitch, to, 0, lane);
        bring_v(v, tiles.base(t), a.kv_rows, pitch, to + S::kTileBytes, 0, lane);
    };
    auto mask_byte = [&](int t) -> int {
        const int j = tiles.base(t) + lane;
        return mask != nullptr && lane < 32 && j < a.kv_rows ? mask[j] : 1;
    };
    int kept = 1, buffer = 0;
    if (tile < until) {
        bring(tile, 0);
        kept = mask_byte(tile);
    }
    for (; tile < until; tile += 4) {
        constexpr int kRequests = 2 * S::kTileBytes / 1024;
        unsigned long long kept_bits;
        if (S::kBuffers == 2 && tile + 4 < until) {
            const int now = kept;
            bring(tile + 4, buffer ^ 1);
            kept = mask_byte(tile + 4);
            wait_loads<kRequests>();  // (one more where a mask was read: its request is the youngest)
            __builtin_amdgcn_sched_barrier(0);
            asm volatile("" ::: "memory");
            kept_bits = __ballot(now != 0);
        } else {
            landed();
            kept_bits = __ballot(kept != 0);
        }
        unsigned char *kt = buffers + buffer * 2 * S::kTileBytes, *vt = kt + S::kTileBytes;
        const int base = tiles.base(tile);
        const unsigned long long seen = reach.of(base, a.sinks) & kept_bits, whole = bits_below(32);
        if ((seen & whole) != whole) clear_rows<T, D, 32>(vt, seen, lane);
        if ((seen & whole) != 0) {
            const bool all = reach.all(base, 32, a.sinks) && (kept_bits & whole) == whole;
            const unsigned long long visible =
                    all ? ~0ull : bits_below(end - base) & (~bits_below(begin - base) | bits_below(a.sinks - base)) & kept_bits;
            if constexpr (FEW) attend_few<D>(r, kt, vt, a.scale, all, (unsigned) visible, lane);
            else attend<T, D, 1>(r, kt, vt, a.scale, all, visible, lane);
        }
        if (S::kBuffers == 2) {
            buffer ^= 1;
            __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): this tile has been read, its buffer is free
            __builtin_amdgcn_sched_barrier(0);
        } else {
            __builtin_amdgcn_s_waitcnt(0xc07f);
            __builtin_amdgcn_sched_barrier(0);
            if (tile + 4 < until) {
                bring(tile + 4, 0);
                kept = mask_byte(tile + 4);
            }
        }
    }
    // the four wavefronts' sums, 32 rows of D + 4 floats each: results, maximum, sum
    products_done();
    __syncthreads();
    float *merge = reinterpret_cast<float *>(smem);
    float sum = r.sum + __shfl_xor(r.sum, 32, kWave);
    float *to = merge + (wave * 32 + (lane & (kRows - 1))) * S::kPitch;
    if constexpr (FEW) {
        sum += __shfl_xor(sum, 16, kWave);
#pragma unroll
        for (int d = 0; d < D / 16; ++d) *reinterpret_cast<v4f32 *>(to + 16 * d + 4 * (lane >> 4)) = r.ctx[d];
    } else {
#pragma unroll
        for (int d = 0; d < D / 32; ++d)
#pragma unroll
            for (int i = 0; i < 16; i += 4)
                *reinterpret_cast<v4f32 *>(to + 32 * d + 2 * i + 4 * (lane >> 5)) = v4f32{r.ctx[d][i], r.ctx[d][i + 1], r.ctx[d][i + 2], r.ctx[d][i + 3]};
    }
    if (lane < kRows) to[D] = r.top, to[D + 1] = sum;
    __syncthreads();
    constexpr int kQuads = D / 4;  // a thread has four columns of a row
    for (int i = threadIdx.x; i < (last_row - row0 + 1) * kQuads; i += kBlock) {
        const int m = i / kQuads, d = (i - m * kQuads) * 4;
        float top = kNone;
#pragma unroll
        for (int w = 0; w < 4; ++w) top = fmaxf(top, merge[(w * 32 + m) * S::kPitch + D]);
        v4f32 x = v4f32{};
        float total = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float *from = merge + (w * 32 + m) * S::kPitch;
            const float f = __builtin_amdgcn_exp2f((from[D] - top) * a.scale);
            total += from[D + 1] * f;
            x += *reinterpret_cast<const v4f32 *>(from + d) * f;
        }
        const int out_row = row0 + m, out_query = out_row / share, out_head = at.kv_head * share + out_row - out_query * share;
        const int out_p = at.first + out_query;
        const bool out_there = out_p >= 0 && out_p < at.length;
        if (pieces > 1) {
            float *out = a.partials + ((size_t) blockIdx.x * 32 + m) * S::kPitch;
            *reinterpret_cast<v4f32 *>(out + d) = out_there ? x : v4f32{};
            if (d == 0) out[D] = out_there ? top : kNone, out[D + 1] = out_there ? total : 0.f;
        } else {
            const float by = out_there && total != 0.f ? 1.f / total : 0.f;
            T *ctx = (T *) a.ctx + ((size_t) at.b * a.q_rows + out_query) * a.ld_ctx + (size_t) out_head * D + d;
            if (by != 0.f) store4(ctx, x[0] * by, x[1] * by, x[2] * by, x[3] * by);
            else store4(ctx, 0.f, 0.f, 0.f, 0.f);
        }
    }
}

// The pieces' sums of a row joined, where they are at most kFewPieces: D / 4 lanes to a row.
template <typename T, int D>
__global__ __launch_bounds__(kBlock) void attention_window_join_few_kernel(WindowArgs a, int row_tiles, int pieces, int total_rows) {
    constexpr int kPitch = Spread<T, D>::kPitch, kQuads = D / 4;
    const int i = blockIdx.x * (kBlock / kQuads) + threadIdx.x / kQuads, d = threadIdx.x % kQuads * 4;
    if (i >= total_rows) return;
    const int share = a.heads / a.kv_heads, rows = a.q_rows * share;
    const int problem = i / rows, row = i - problem * rows, b = problem / a.kv_heads, kv_head = problem - b * a.kv_heads;
    const float *from = a.partials + ((size_t) (problem * row_tiles + row / 32) * pieces * 32 + row % 32) * kPitch;
    const size_t step = (size_t) 32 * kPitch;
    // all that there is to read at once (past the last piece the first one again)
    v4f32 part[kFewPieces];
    float tops[kFewPieces], sums[kFewPieces];
#pragma unroll
    for (int n = 0; n < kFewPieces; ++n) {
        const float *at = from + (n < pieces ? n : 0) * step;
        part[n] = *reinterpret_cast<const v4f32 *>(at + d);
        tops[n] = at[D], sums[n] = at[D + 1];
    }
    float top = tops[0];
#pragma unroll
    for (int n = 1; n < kFewPieces; ++n) top = fmaxf(top, tops[n]);
    v4f32 x = v4f32{};
    float sum = 0.f;
#pragma unroll
    for (int n = 0; n < kFewPieces; ++n) {
        if (n < pieces) {
            const float f = __builtin_amdgcn_exp2f((tops[n] - top) * a.scale);
            sum += sums[n] * f;
            x += part[n] * f;
        }
    }
    const int query = row / share, head = kv_head * share + row - query * share;
    T *ctx = (T *) a.ctx + ((size_t) b * a.q_rows + query) * a.ld_ctx + (size_t) head * D + d;
    const float by = sum != 0.f ? 1.f / sum : 0.f;
    if (by != 0.f) store4(ctx, x[0] * by, x[1] * by, x[2] * by, x[3] * by);
    else store4(ctx, 0.f, 0.f, 0.f, 0.f);
}

// The same for many pieces: a workgroup per row, D / 4 threads to a piece's results, the pieces' weights in LDS.
template <typename T, int D>
__global__ __launch_bounds__(kBlock) void attention_window_join_kernel(WindowArgs a, int row_tiles, int pieces) {
    constexpr int kPitch = Spread<T, D>::kPitch, kQuads = D / 4, kAtOnce = kBlock / kQuads;
    __shared__ float weights[kMaxPieces], tops[kBlock / kWave], sums[kBlock / kWave];
    __shared__ v4f32 parts[kAtOnce][kQuads];
    const int share = a.heads / a.kv_heads, rows = a.q_rows * share, thread = threadIdx.x;
    const int problem = blockIdx.x / rows, row = blockIdx.x - problem * rows, b = problem / a.kv_heads, kv_head = problem - b * a.kv_heads;
    const float *from = a.partials + ((size_t) (problem * row_tiles + row / 32) * pieces * 32 + row % 32) * kPitch;
    const size_t step = (size_t) 32 * kPitch;
    const int at = thread / kQuads, d = thread % kQuads * 4;
    static_assert(kMaxPieces <= kBlock, "a thread per piece");
    const bool mine = thread < pieces;
    const float my_top = mine ? from[thread * step + D] : kNone, my_sum = mine ? from[thread * step + D + 1] : 0.f;
    const float wave_top = wave_max(my_top);
    if ((thread & (kWave - 1)) == 0) tops[thread / kWave] = wave_top;
    __syncthreads();
    float top = tops[0];
#pragma unroll
    for (int w = 1; w < kBlock / kWave; ++w) top = fmaxf(top, tops[w]);
    const float weight = __builtin_amdgcn_exp2f((my_top - top) * a.scale);
    if (mine) weights[thread] = weight;
    const float wave_total = wave_sum(weight * my_sum);
    if ((thread & (kWave - 1)) == 0) sums[thread / kWave] = wave_total;
    __syncthreads();
    v4f32 x = v4f32{};
#pragma unroll 4
    for (int n = at; n < pieces; n += kAtOnce) x += *reinterpret_cast<const v4f32 *>(from + n * step + d) * weights[n];
    parts[at][thread % kQuads] = x;
    __syncthreads();
    if (at != 0) return;
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kBlock / kWave; ++w) sum += sums[w];
#pragma unroll
    for (int n = 1; n < kAtOnce; ++n) x += parts[n][thread];
    const int query = row / share, head = kv_head * share + row - query * share;
    T *ctx = (T *) a.ctx + ((size_t) b * a.q_rows + query) * a.ld_ctx + (size_t) head * D + d;
    const float by = sum != 0.f ? 1.f / sum : 0.f;
    if (by != 0.f) store4(ctx, x[0] * by, x[1] * by, x[2] * by, x[3] * by);
    else store4(ctx, 0.f, 0.f, 0.f, 0.f);
}

// How a call is run: rows of a workgroup (32: the spread kernel), and into how many pieces the axis is cut.
struct WindowPlan {
    int rows, row_tiles, pieces;
    size_t floats;
};

// The rule, measured on heads of 64 with 128 / 64 / 32 rows, microseconds.  fp16: 4 x 4096 tokens of 16 heads, window 512 (2048 workgroups of
// 128) 109 / 135 / 179; 32 x 128 of 12 (384) 13 / 19 / 19; 2 x 4096 of 4 (256) 84 / 57 / 80; 2 x 512 of 12 over 8192 (192 of 64) 161 / 93 / 104;
// 3 x 517 of 12 (180) 32 / 28 / 28; 1 x 600 (60) 18 / 13 / 16; 1 x 64 over 1000 (12) 25 / 17 / 10.  Heads of 128, whose tiles for 64 rows
// leave room for one workgroup to a unit: 2048 causal tokens of 16 (256 of 128) 68 / 75 / 73; 1024 of 32 to 8 over 16384 (256) 467 / 597 / 512;
// 2 x 800 of 16 to 4 over 6000 (200) 176 / 209 / 138; 512 of 32 to 8 over 16384 (128) 464 / 321 / 280; 1000 of 16 (128) 38 / 27 / 28.
// fp32: 2 x 2000 of 16 (512) 189 / 211 / 303; 3 x 517 (180) 47 / 43 / 59; 2 x 400 of 12 (168 of 64) 29 / 22 / 31; 1 x 64 over 1000 (12) 57 / 27 / 13.
WindowPlan plan_window(bool half_precision, int batch, int heads, int kv_heads, int q_rows, int kv_rows, int head_size, int left, int right, int sinks) {
    WindowPlan plan;
    const long long rows = (long long) q_rows * (heads / kv_heads), problems = (long long) batch * kv_heads;
    const long long of_128 = (rows + 127) / 128 * problems, of_64 = (rows + 63) / 64 * problems;
    if (half_precision && head_size == 128) plan.rows = rows <= 32 || of_128 < 256 ? 32 : 128;
    else plan.rows = rows <= 32 ? 32 : of_128 >= 320 ? 128 : of_64 >= (half_precision ? 96 : 16) ? 64 : 32;
    plan.row_tiles = (int) ((rows + plan.rows - 1) / plan.rows);
    plan.pieces = 1, plan.floats = 0;
    // the most tiles of 32 keys that a workgroup's rows reach
    long long reach = kv_rows;
    if (left >= 0 && right >= 0) reach = (long long) left + right + plan.rows + 1 + sinks < reach ? (long long) left + right + plan.rows + 1 + sinks : reach;
    const long long tiles = (reach + 31) / 32, blocks = problems * plan.row_tiles;
    long long pieces = 1, most = 1;
    if (plan.rows == 32) {
        // About 384 workgroups, three for two units, with a tile to every wavefront at least.  Microseconds with 256 / 384 / 512 / 768:
        // fp16, 48 tokens over up to 1000 keys 20 / 20 / 24 / 23, 2 x 100 over 6000 28 / 23 / 27 / 26, 32 over 4096 52 / 54 / 52 / 53.  (Pieces
        // of 8 tiles at least and of 4: fp32, 7 x 1 over 413 keys of 128 20 and 14 us, 12 x 1 over 396 15 and 12; fp16, 1 x 1 over 4096 both 12.)
        pieces = blocks > 0 ? (384 + blocks - 1) / blocks : 1, most = (tiles + 3) / 4;
    } else if (plan.rows == 64 && !half_precision) {
        // 512 workgroups, which two units share, with 512 keys at least.  Microseconds uncut (or with 32 rows, where 64 are too few) / so: 4 x 64
        // of 32 heads to 8 of 128 over 8192 312 / 272; 2048 causal tokens of 12 heads of 64 91 / 75; 2 x 100 of 14 to 2 over 6000 53 / 46;
        // 430 over 7327 of 8 to 2 of 32 79 / 71.  With 256 keys at least 3 x 517 45 / 48, 2 x 1000 of 7 to 1, window 300, 35 / 44.  Not in
        // fp16, which has less to do for the sums that it would write and read again: 2048 causal tokens 26 / 34, 600 of 12 11 / 15.
        pieces = (512 + blocks - 1) / blocks, most = tiles / 16;
    }
    pieces = pieces < most ? pieces : most;
    plan.pieces = (int) (pieces < 1 ? 1 : pieces > kMaxPieces ? kMaxPieces : pieces);
    if (plan.pieces > 1) plan.floats = (size_t) blocks * plan.pieces * plan.rows * (head_size + 4);
    return plan;
}

template <typename T, int D, int ROWS>
int run_window_rows(const WindowArgs &a, int row_tiles, int pieces, hipStream_t stream) {
    static std::atomic<unsigned long long> done{0};
    const dim3 grid(a.batch * a.kv_heads * row_tiles * pieces);
    if constexpr (sizeof(T) == 4) {
        constexpr int kLds = 6 * (32 * 128 / ROWS) * 2 * D;
        if (kLds > 48 * 1024 && !allow_large_lds(attention_window_terms_kernel<D, ROWS>, done)) return CUBERT_UNSUPPORTED;
        return launch_lds(attention_window_terms_kernel<D, ROWS>, grid, dim3(kBlock), kLds, stream, a, row_tiles, pieces);
    } else {
        constexpr int kLds = 4 * (64 * 128 / ROWS) * 2 * D;
        if (kLds > 48 * 1024 && !allow_large_lds(attention_window_shared_kernel<D, ROWS>, done)) return CUBERT_UNSUPPORTED;
        return launch_lds(attention_window_shared_kernel<D, ROWS>, grid, dim3(kBlock), kLds, stream, a, row_tiles);
    }
}

template <typename T, int D, bool FEW>
int run_spread(const WindowArgs &a, WindowPlan plan, hipStream_t stream) {
    static std::atomic<unsigned long long> done{0};
    if (Spread<T, D>::kLds > 48 * 1024 && !allow_large_lds(attention_window_spread_kernel<T, D, FEW>, done)) return CUBERT_UNSUPPORTED;
    return launch_lds(attention_window_spread_kernel<T, D, FEW>, dim3(a.batch * a.kv_heads * plan.row_tiles * plan.pieces), dim3(kBlock),
                      Spread<T, D>::kLds, stream, a, plan.row_tiles, plan.pieces);
}

template <typename T, int D>
int run_window(const WindowArgs &a, WindowPlan plan, hipStream_t stream) {
    const int problems = a.batch * a.kv_heads, rows = a.q_rows * (a.heads / a.kv_heads), row_tiles = plan.row_tiles * (plan.rows / 32);
    int rc;
    constexpr int kHalfRows = sizeof(T) == 2 && D == 128 ? 128 : 64;  // (heads of 128 in fp16 have no rows in between)
    if (plan.rows == 128) rc = run_window_rows<T, D, 128>(a, plan.row_tiles, plan.pieces, stream);
    else if (plan.rows == 64) rc = run_window_rows<T, D, kHalfRows>(a, plan.row_tiles, plan.pieces, stream);
    else if (sizeof(T) == 4 && rows <= 16) rc = run_spread<T, D, sizeof(T) == 4>(a, plan, stream);
    else rc = run_spread<T, D, false>(a, plan, stream);
    if (rc != 0 || plan.pieces == 1) return rc;
    const int total = problems * rows, per_block = kBlock / (D / 4);
    // (the whole call with D / 4 threads to a row / a workgroup: 8 x 1 of 16 heads over up to 2048 keys, 6 pieces, 14.0 / 14.6 us, 12 x 1 of 12
    // over up to 1000, 3 pieces, 14.5 / 15.1; the join alone, 18612 rows of 2 pieces, 5 / 22)
    if (plan.pieces <= kFewPieces)
        return launch(attention_window_join_few_kernel<T, D>, dim3((total + per_block - 1) / per_block), dim3(kBlock), stream, a, row_tiles,
                      plan.pieces, total);
    return launch(attention_window_join_kernel<T, D>, dim3(total), dim3(kBlock), stream, a, row_tiles, plan.pieces);
}

template <typename T>
int attention_window(const T *q, int ldq, const T *k, const T *v, int ldkv, const int *first, const int *lengths, const int8_t *mask,
                     T *ctx, int ld_ctx, float alpha, int batch, int heads, int kv_heads, int q_rows, int kv_rows, int head_size,
                     int left, int right, int sinks, float *partials, size_t partial_floats, void *stream) {
    if (batch < 0 || heads < 1 || kv_heads < 1 || heads % kv_heads != 0 || !(alpha > -INFINITY && alpha < INFINITY) || q_rows < 0 ||
        kv_rows < 0 || head_size < 1 || sinks < 0 || kv_rows > kFar || q_rows > kFar)
        return CUBERT_BAD_ARGUMENT;
    const long long width = (long long) heads * head_size, kv_width = (long long) kv_heads * head_size;
    if (ldq < width || ldkv < kv_width || ld_ctx < width) return CUBERT_BAD_ARGUMENT;
    if (batch == 0 || q_rows == 0) return 0;
    if (q == nullptr || ctx == nullptr || (kv_rows > 0 && (k == nullptr || v == nullptr))) return CUBERT_BAD_ARGUMENT;
    const int piece = 16 / (int) sizeof(T);
    if (!is_aligned(q, 16) || !is_aligned(k, 16) || !is_aligned(v, 16) || !is_aligned(ctx, 16) || ldq % piece != 0 ||
        ldkv % piece != 0 || ld_ctx % piece != 0)
        return CUBERT_UNSUPPORTED;
    if (ldkv > 1 << 22) return CUBERT_UNSUPPORTED;  // (pieces of a tile are addressed with 32 bits)
    if (head_size != 32 && head_size != 64 && head_size != 128) return CUBERT_UNSUPPORTED;
    // a launch holds less than 2^32 threads, and rows of a key head are counted in 32 bits
    const unsigned long long problems = (unsigned long long) batch * kv_heads, rows = (unsigned long long) q_rows * (heads / kv_heads);
    if (problems >= 1u << 24 || rows >= 1u << 30) return CUBERT_UNSUPPORTED;
    WindowArgs a;
    a.q = q, a.k = k, a.v = v, a.ctx = ctx, a.first = first, a.lengths = lengths, a.mask = mask;
    a.partials = partials;
    a.negate = alpha < 0.f;
    // (a factor of 0 would make numbers of the infinities that stand for keys left out, an infinite one no number of a difference of 0)
    a.scale = fminf(fmaxf(fabsf(alpha) * 1.44269504089f, 1e-30f), 3e38f);
    a.ldq = ldq, a.ldkv = ldkv, a.ld_ctx = ld_ctx;
    a.batch = batch, a.heads = heads, a.kv_heads = kv_heads, a.q_rows = q_rows, a.kv_rows = kv_rows;
    a.left = left < 0 || left > kFar ? kFar : left, a.right = right < 0 || right > kFar ? kFar : right;
    a.sinks = sinks;
    WindowPlan plan = plan_window(sizeof(T) == 2, batch, heads, kv_heads, q_rows, kv_rows, head_size, left, right, sinks);
    if (problems * plan.row_tiles * plan.pieces >= 1u << 24) return CUBERT_UNSUPPORTED;
    if (plan.pieces > 1 && (partials == nullptr || partial_floats < plan.floats || !is_aligned(partials, 16))) plan.pieces = 1;
    if (head_size == 32) return run_window<T, 32>(a, plan, (hipStream_t) stream);
    if (head_size == 64) return run_window<T, 64>(a, plan, (hipStream_t) stream);
    return run_window<T, 128>(a, plan, (hipStream_t) stream);
}

}  // namespace
}  // namespace cubert

using cubert::half_t;

extern "C" {

size_t cubert_attention_window_partials(int half_precision, int batch, int heads, int kv_heads, int q_rows, int kv_rows,
                                        int head_size, int left, int right, int sinks) {
    if (batch < 1 || heads < 1 || kv_heads < 1 || heads % kv_heads != 0 || q_rows < 1 || kv_rows < 1 || head_size < 1) return 0;
    if ((long long) batch * kv_heads >= 1 << 24) return 0;  // refused
    return cubert::plan_window(half_precision != 0, batch, heads, kv_heads, q_rows, kv_rows, head_size, left, right, sinks).floats;
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
