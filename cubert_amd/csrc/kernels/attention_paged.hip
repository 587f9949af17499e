// Attention of new tokens over a key/value cache in pages:
//
//     query i of sequence b stands at p = first[b] + i and sees key j if
//         j <= p,  j < length[b],  table[b, j / page] is a page  and  (j >= p - left  or  j < sinks);
//     ctx = sum_j e^(alpha q.k_j - m) v_j / sum_j e^(alpha q.k_j - m) over what it sees, m the largest score.
//
// A query that sees nothing, or that stands outside its sequence (p < 0 or p >= length[b]), gets zeros.  Heads share keys
// and values in groups of heads / kv_heads.

#include <atomic>
#include <type_traits>

#include "cubert_kernels.h"
#include "device_common.h"
#include "paged.h"

namespace cubert {
namespace {

constexpr int kFar = (1 << 30) - 1;  // a bound or position that no sequence reaches
constexpr float kNone = -3.402823466e38f;  // the maximum of no scores: no finite score is less

constexpr int kShared = 64;  // bytes of LDS in which wavefronts tell each other which piece theirs is

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

template <typename T, typename V>
__device__ __forceinline__ void store4(T *to, V x) {
    store_vec<T, 4>(to, Vec<T, 4>{from_f32<T>(x[0]), from_f32<T>(x[1]), from_f32<T>(x[2]), from_f32<T>(x[3])});
}

typedef _Float16 v8f16 __attribute__((ext_vector_type(8)));
typedef _Float16 v2f16 __attribute__((ext_vector_type(2)));
typedef float v4f32 __attribute__((ext_vector_type(4)));
typedef float v2f32 __attribute__((ext_vector_type(2)));
typedef int v2i32 __attribute__((ext_vector_type(2)));

// 16 rows (queries and heads of one key head) meet 16 keys in products of 16 x 16 with the keys as their rows: lane l has row l % 16 and
// the keys 4 (l / 16) + i, i = 0..3, so that what belongs to a row, its maximum, its sum and its results, stays in four lanes.  Keys come from
// memory as the products take them, lane l has of key l % 16 every fourth 16-byte piece, and do not pass through LDS.
//
// fp16: V passes through LDS, out of which it comes transposed, and the probabilities are the other factor as they are, as sums of two fp16
// numbers, so that a result is rounded once, at the end.  (With fp32's own products instead, which take V as it lies in memory, four times
// the cycles: 1 x 1 over 64 keys of 12 heads 5.9 us for 4.5.)
// fp32: a product with V takes a single number of one key from a lane.  Of the i-th key of its four a lane brings D / 16 columns of V, one after
// the other, as they lie in memory, and nothing is transposed.
//
// What is on its way together, a unit, is 32 keys for a wavefront (16 where rows have 512 bytes): while it works on one, K of the next is requested as
// soon as this one's has been multiplied, and V as soon as this one's lies in LDS.  Rows of 256 bytes: twelve wavefronts to a compute unit have 192
// KB on their way.  (64 keys where rows have 128 bytes, and fewer wavefronts: 256 x 1 over up to 512 keys of 12 heads of 64 43.9 us for 42.1, 4 x 1
// over up to 300 6.8 for 6.0.)
template <typename T, int D>
struct Shape {
    static constexpr bool kHalf = sizeof(T) == 2;
    static constexpr int kRowBytes = D * (int) sizeof(T);
    static constexpr int kKeyLoads = kRowBytes / 64;                                // 16-byte pieces of a key that a lane has
    static constexpr int kSub = kRowBytes == 512 ? 1 : 2;                           // 16 keys each: what is on its way together
    static constexpr int kKeys = 16 * kSub;
    // V: requests for 16 keys, their size, and how many keys one has
    static constexpr int kValueBytes = kHalf || kRowBytes >= 256 ? 16 : kRowBytes / 16;
    static constexpr int kValueLoads = 16 * kRowBytes / (kWave * kValueBytes);
    static constexpr int kColumns = kValueBytes / (int) sizeof(T);                  // neighbouring columns that a lane has
    static constexpr int kValueLds = kHalf ? kKeys * kRowBytes : 0;                 // of a wavefront
    static constexpr int kPitch = D + 4;                                            // floats between rows of sums
    // How far a maximum may rise, in powers of two, before sums are scaled anew, and how much larger probabilities are, so that fp16's subnormals
    // begin far below the maximum (2^-37 of it; 2^15 is still fp16).  fp32: probabilities are 1 at most, as V may be as large as fp32 goes.
    static constexpr float kSlack = kHalf ? 3.f : 0.f, kRaise = kHalf ? 12.f : 0.f;
};

// (the same in every lane, which the compiler has to be told)
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// Registers of a request, and the numbers in them.
template <int WORDS>
using Words = int __attribute__((ext_vector_type(WORDS)));
template <typename T, int N>
using Numbers = T __attribute__((ext_vector_type(N)));

template <bool ONCE, typename W>
__device__ __forceinline__ W read(const W *p) {
    if constexpr (ONCE) return __builtin_nontemporal_load(p);
    return *p;
}

// Which of its 16-byte pieces a row of V keeps its piece `at` in: 32 lanes read 32 bytes of eight rows together, which lie on different banks.
template <int ROW_BYTES>
__device__ __forceinline__ int v_piece(int key, int at) {
    return at ^ (key / (256 / ROW_BYTES) % (ROW_BYTES / 32) * 2);
}

// Probabilities as sums of two fp16 numbers: pairs of `high` and `low`, off by 2^-21 of those from kSmall on, and by 2^-24 below it.  Neither is
// negative, and the second one is not 0 where the probability is more than 2^-37 of the largest, so that an infinite value of V stays infinite in
// either product.
__device__ __forceinline__ void two_terms(float e0, float e1, v2f16 &high, v2f16 &low) {
    constexpr float kLeast = 0x1p-24f;  // fp16's smallest
    high = __builtin_bit_cast(v2f16, __builtin_amdgcn_cvt_pkrtz(e0, e1));
    float minus = -1.f;
    asm("" : "+v"(minus));  // (as a constant it makes a conversion and a subtraction of one instruction)
    // (the middle one of the rest, the probability and the smallest: the rest, or as much of the smallest as there is)
    low = __builtin_convertvector((v2f32{__builtin_amdgcn_fmed3f(fmaf((float) high[0], minus, e0), e0, kLeast),
                                         __builtin_amdgcn_fmed3f(fmaf((float) high[1], minus, e1), e1, kLeast)}), v2f16);
}

// What the two terms of a probability below kSmall (2^-15 to 2^-18 of the largest) leave out, kLeftOverBy times: 2^-24 at most in either direction, which
// is exact in fp32, as two fp16 numbers.  With them probabilities down to 2^-54 of the largest are exact to 2^-21 of themselves, each.  (A first
// token often has nearly all of the weight and a value near 0, and a result is what the small ones leave.)  Only units that have such
// probabilities take these products; microseconds without any / with them in every unit / of the two terms alone: 64 x 1 over up to 4096 keys of 4 heads
// of 128 53.8 / 56.8 / 53.4, 1 x 1 over 131072 of 2 heads 30.1 / 35.4 / 30.0, over 64 of 12 heads of 64 4.3 / 4.7 / 4.2.
constexpr float kSmall = 0x1p-3f, kLeftOverBy = 0x1p38f;

__device__ __forceinline__ void left_over(float e0, float e1, v2f16 &high, v2f16 &low) {
    v2f16 x, y;
    two_terms(e0, e1, x, y);
    const float r0 = e0 < kSmall ? (e0 - (float) x[0] - (float) y[0]) * kLeftOverBy : 0.f;
    const float r1 = e1 < kSmall ? (e1 - (float) x[1] - (float) y[1]) * kLeftOverBy : 0.f;
    high = __builtin_bit_cast(v2f16, __builtin_amdgcn_cvt_pkrtz(r0, r1));
    low = __builtin_convertvector((v2f32{r0 - (float) high[0], r1 - (float) high[1]}), v2f16);
}

// Infinities as the largest numbers: they reach a result with the two terms, and what those leave out may be negative, or nothing.
__device__ __forceinline__ v8f16 finite(v8f16 x) {
    constexpr _Float16 kMost = 65504;
    return __builtin_elementwise_maximum(__builtin_elementwise_minimum(x, (v8f16) kMost), (v8f16) -kMost);
}

// A problem is a tile of rows of a sequence and a key head; sequences and tiles are numbered together, tile * batch + sequence.  A workgroup has one
// (pieces = 0) or a piece of one: about `pieces` of all units, kLeast units at least, so pieces + problems of them at most.
constexpr int kLeast = 4;

struct PagedPlan {
    int rows, row_tiles, pieces;  // rows of a tile
    int slot_rows;                       // of which that many are there
    bool once;                           // K and V are read once, and are too large to be there still when they are read again
    long long problems;
    long long bytes;  // of K and V, of all sequences, if they are as long as their tables and the window let them be
    size_t floats;
};

// The keys that the queries of a tile of rows of a sequence see between them, in units of KEYS keys: those of the sinks, then those of the window.
template <int KEYS>
struct Reach {
    int length, first, low, high;  // positions of the queries inside of the sequence
    int of_sinks, begin, units;    // units of the sinks, the window's first, and all of them: one at least, so that somebody writes the zeros
    bool any;

    __device__ __forceinline__ Reach(const PagedArgs &a, const PagedPlan &plan, int length_, int first_, int tile) {
        length = clamp_to(length_, 0, a.width << a.shift);
        first = a.first != nullptr ? clamp_to(first_, -kFar, kFar) : length - a.q_rows;
        low = first, high = first + a.q_rows - 1;
        if (plan.row_tiles > 1) {
            const int share = a.heads / a.kv_heads, rows = a.q_rows * share, row0 = tile * plan.rows;
            low = first + row0 / share, high = first + ((row0 + plan.rows < rows ? row0 + plan.rows : rows) - 1) / share;
        }
        low = low < 0 ? 0 : low, high = high < length ? high : length - 1;
        any = low <= high;
        const int first_begin = low > a.left ? low - a.left : 0, end = high + 1, far = a.sinks < end ? a.sinks : end;
        begin = first_begin / KEYS;
        of_sinks = (far + KEYS - 1) / KEYS;
        of_sinks = of_sinks < begin ? of_sinks : begin;
        units = any ? of_sinks + (end + KEYS - 1) / KEYS - begin : 1;
        if (!any) begin = of_sinks = 0;
    }
    __device__ __forceinline__ int key_of(int unit) const { return (unit < of_sinks ? unit : unit - of_sinks + begin) * KEYS; }
};

// The sum of x over this lane and those before it.
__device__ __forceinline__ int sum_through(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr:1, 2, 4, 8
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast:15 into rows 1 and 3
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row_bcast:31 into rows 2 and 3
    return x;
}

// Length, first position and units of the sequence and tile `entry` (0 units behind the last).
template <int KEYS>
struct Entry {
    int length = 0, first = 0, units = 0;

    __device__ __forceinline__ Entry() {}
    __device__ __forceinline__ Entry(const PagedArgs &a, const PagedPlan &plan, int entry) {
        if (entry >= a.batch * plan.row_tiles) return;
        const int tile = plan.row_tiles > 1 ? entry / a.batch : 0, b = entry - tile * a.batch;
        length = a.lengths[b];
        if (a.first != nullptr) first = a.first[b];
        units = Reach<KEYS>(a, plan, length, first, tile).units;
    }
};

template <typename T, int D, int TILES>
struct Rows {
    typedef Shape<T, D> S;
    v4f32 q[TILES][S::kKeyLoads], ctx[TILES][D / 16];
    float top[TILES], sum[TILES];
};

// Bound by reading K and V, and by what comes before and behind it: a chain of reads from the lengths over the table to the first keys takes 2.5
// us, the join 4.  fp16, 64 x 1 over up to 4096 keys of 4 heads of 128, 272 MB in 53 us (5.1 TB/s); 256 x 1 over up to 512 of 12 heads of 64, 223
// MB in 42 us (5.3 TB/s); 1 x 1 over 131072 of 2 heads of 128, 134 MB in 31 us; fp32, 32 x 1 over up to 4096 of 12 heads of 64, 443 MB in 78 us (5.7
// TB/s).  One tile of rows: 168 registers at most, with which three workgroups and more fit a unit (two: the first of these calls 57 us).
// The four wavefronts have a run of the piece's units each; their sums meet in LDS, in wavefront order.
template <typename T, int D, int TILES, bool ONCE>
__global__ __launch_bounds__(kBlock, TILES == 1 ? 3 : 2) void attention_paged_kernel(PagedArgs a, PagedPlan plan) {
    typedef Shape<T, D> S;
    typedef Reach<S::kKeys> Reached;
    constexpr int kWaves = kBlock / kWave, kRows = 16 * TILES, kSub = S::kSub, kKeys = S::kKeys;
    extern __shared__ __align__(16) unsigned char smem[];
    const int wave = wave_in_block(), lane = threadIdx.x & (kWave - 1), col = lane & 15, quarter = lane >> 4;
    const int share = a.heads / a.kv_heads, rows = a.q_rows * share;

    // which problem, and which piece of it
    int entry, kv_head, piece = 0, pieces = 1, length, first = 0;
    if (plan.pieces == 0) {
        entry = blockIdx.x / a.kv_heads, kv_head = blockIdx.x - entry * a.kv_heads;
        const int b = plan.row_tiles > 1 ? entry % a.batch : entry;
        length = a.lengths[b];
        if (a.first != nullptr) first = a.first[b];
    } else {
        typedef Entry<kKeys> Found;
        const int all = a.batch * plan.row_tiles, block = (int) blockIdx.x;
        int before = 0, most = 0;
        bool found = false;
        auto units_of_piece = [&](int units) {  // (units of all sequences and tiles for a key head; of all of them below 2^30: see plan_paged)
            const int least = (units * a.kv_heads + plan.pieces - 1) / plan.pieces;
            most = least > kLeast ? least : kLeast;
        };
        auto own_pieces = [&](const Found &of) { return (of.units + most - 1) / most; };
        auto look = [&](int from, const Found &of) {
            const int own = own_pieces(of), through = sum_through(own * a.kv_heads);
            const unsigned long long here = __ballot(before + through > block);
            if (here != 0) {
                const int at = __builtin_ctzll(here);
                found = true, entry = from + at, pieces = __builtin_amdgcn_readlane(own, at);
                length = __builtin_amdgcn_readlane(of.length, at), first = __builtin_amdgcn_readlane(of.first, at);
                piece = block - (before + __builtin_amdgcn_readlane(through, at) - pieces * a.kv_heads);
                kv_head = piece / pieces, piece -= kv_head * pieces;
            }
            before += __builtin_amdgcn_readlane(through, kWave - 1);
        };
        if (all <= kWave) {
            // every wavefront looks through the sequences by itself, and none waits
            const Found own(a, plan, lane);
            units_of_piece(__builtin_amdgcn_readlane(sum_through(own.units), kWave - 1));
            look(0, own);
            if (!found) return;
        } else {
            // a quarter of them to a wavefront, the first 128 of it in registers (all of them to every one: 512 x 1 over up to 300, tables for 32768,
            // 1 of 64 25 us for 15)
            constexpr int kKept = 2;
            int *shared = reinterpret_cast<int *>(smem);
            const int chunks = (all + kBlock - 1) / kBlock, from = wave * chunks * kWave;
            Found kept[kKept];
            int units = 0, own = 0;
#pragma unroll
            for (int n = 0; n < kKept; ++n)
                if (n < chunks) kept[n] = Found(a, plan, from + n * kWave + lane);
            for (int n = kKept; n < chunks; ++n) units += Found(a, plan, from + n * kWave + lane).units;
#pragma unroll
            for (int n = 0; n < kKept; ++n) units += kept[n].units;
            units = __builtin_amdgcn_readlane(sum_through(units), kWave - 1);
            if (lane == 0) shared[wave] = units;
            __syncthreads();
            units_of_piece(shared[0] + shared[1] + shared[2] + shared[3]);
#pragma unroll
            for (int n = 0; n < kKept; ++n) own += own_pieces(kept[n]);
            for (int n = kKept; n < chunks; ++n) own += own_pieces(Found(a, plan, from + n * kWave + lane));
            own = __builtin_amdgcn_readlane(sum_through(own), kWave - 1) * a.kv_heads;
            if (lane == 0) shared[kWaves + wave] = own;
            __syncthreads();
            int through = 0;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                before += w < wave ? shared[kWaves + w] : 0;
                through += shared[kWaves + w];
            }
            if (block >= uniform(through)) return;
            before = uniform(before);
            if (before <= block && block < before + own) {
#pragma unroll
                for (int n = 0; n < kKept; ++n)
                    if (!found && n < chunks) look(from + n * kWave, kept[n]);
                for (int n = kKept; !found && n < chunks; ++n) look(from + n * kWave, Found(a, plan, from + n * kWave + lane));
                if (lane == 0) {
                    int *to = shared + 2 * kWaves;
                    to[0] = entry, to[1] = kv_head, to[2] = piece, to[3] = pieces, to[4] = length, to[5] = first;
                }
            }
            __syncthreads();
            const int *of = shared + 2 * kWaves;
            entry = uniform(of[0]), kv_head = uniform(of[1]), piece = uniform(of[2]), pieces = uniform(of[3]), length = uniform(of[4]), first = uniform(of[5]);
        }
    }
    const int tile = plan.row_tiles > 1 ? entry / a.batch : 0, sequence = entry - tile * a.batch, row0 = tile * kRows;
    const Reached reach(a, plan, length, first, tile);
    const int each = reach.units / pieces, rest = reach.units - each * pieces;
    const int unit = each * piece + (piece < rest ? piece : rest), count = each + (piece < rest ? 1 : 0);  // units of this piece

    const int page_mask = (1 << a.shift) - 1;
    const long long page_bytes = a.page_stride * (long long) sizeof(T);
    const unsigned row_bytes = (unsigned) a.row_stride * (unsigned) sizeof(T);
    const unsigned k_offset = (unsigned) col * row_bytes + (unsigned) quarter * 16;
    constexpr int kPieces = S::kRowBytes / 16;  // of a row; fp16: the l / kPieces-th key of a request
    const int v_key = S::kHalf ? lane / kPieces : quarter * 4;
    const unsigned v_offset = (unsigned) v_key * row_bytes + (unsigned) (S::kHalf ? lane % kPieces * 16 : col * S::kValueBytes);
    // of the j-th request for 16 keys: which of them it begins with, and which 256 bytes of a row it has
    auto value_key = [](int j) { return S::kHalf ? j * (kWave / kPieces) : j * 4 / S::kValueLoads; };
    auto value_part = [](int j) { return S::kHalf ? 0 : j % (S::kValueLoads / 4 > 0 ? S::kValueLoads / 4 : 1); };
    unsigned char *const v_lds = smem + kShared + wave * S::kValueLds;
    const char *k_base = (const char *) a.k + kv_head * a.head_stride * (long long) sizeof(T);
    const char *v_base = (const char *) a.v + kv_head * a.head_stride * (long long) sizeof(T);
    const int *table = a.table + (size_t) sequence * a.ld_table;
    const int seen_begin = reach.low > a.left ? reach.low - a.left : 0, all_begin = reach.high > a.left ? reach.high - a.left : 0;
    const int seen_end = reach.any ? reach.high + 1 : 0, all_end = reach.any ? reach.low + 1 : 0;

    // a wavefront's run among them; lane l has the page of the l-th 16 keys from unit x0 on
    int x = unit + count * wave / kWaves;
    const int until = unit + count * (wave + 1) / kWaves;
    int x0 = x, pages = -1;
    auto look_up = [&](int from_unit) {
        x0 = from_unit;
        const int key = reach.key_of(x0 + lane / kSub) + lane % kSub * 16;
        pages = -1;
        if (key < seen_end) {
            const int page = table[key >> a.shift];
            if (page >= 0 && page < a.pages) pages = page;
        }
    };
    if (x < until) look_up(x);

    Rows<T, D, TILES> r;
    int begin[TILES], end[TILES];  // of what a lane's row sees, the sinks aside
#pragma unroll
    for (int m = 0; m < TILES; ++m) {
        const int row = row0 + 16 * m + col, my_row = row < rows ? row : rows - 1, query = share == 1 ? my_row : my_row / share;
        const char *q = (const char *) a.q + ((size_t) (sequence * a.q_rows + query) * a.ldq +
                                              (size_t) (kv_head * share + my_row - query * share) * D) * sizeof(T);
#pragma unroll
        for (int t = 0; t < S::kKeyLoads; ++t) {
            r.q[m][t] = *reinterpret_cast<const v4f32 *>(q + 64 * t + 16 * quarter);
            if (a.negate) {
                if constexpr (S::kHalf) r.q[m][t] = __builtin_bit_cast(v4f32, -__builtin_bit_cast(v8f16, r.q[m][t]));
                else r.q[m][t] = -r.q[m][t];
            }
        }
#pragma unroll
        for (int d = 0; d < D / 16; ++d) r.ctx[m][d] = v4f32{};
        r.top[m] = kNone, r.sum[m] = 0.f;
        const int p = reach.first + query;
        begin[m] = p > a.left ? p - a.left : 0, end[m] = p >= 0 && p < reach.length ? p + 1 : 0;
    }

    Words<4> k[kSub][S::kKeyLoads];
    Words<S::kValueBytes / 4> v[kSub][S::kValueLoads];
    unsigned there_next = 0;  // which 16 keys of a unit have a page
    auto offset_of = [&](int unit_at, int n) -> long long {
        const int page = __builtin_amdgcn_readlane(pages, (unit_at - x0) * kSub + n);
        return (page < 0 ? 0 : page) * page_bytes + (long long) ((reach.key_of(unit_at) + 16 * n) & page_mask) * row_bytes;
    };
    auto bring_keys = [&](int unit_at) {
        if (unit_at - x0 == kWave / kSub) look_up(unit_at);
        there_next = 0;
#pragma unroll
        for (int n = 0; n < kSub; ++n) {
            if (__builtin_amdgcn_readlane(pages, (unit_at - x0) * kSub + n) >= 0) there_next |= 1u << n;
            const char *at = k_base + offset_of(unit_at, n);
#pragma unroll
            for (int t = 0; t < S::kKeyLoads; ++t) k[n][t] = read<ONCE>(reinterpret_cast<const Words<4> *>(at + k_offset + 64 * t));
        }
    };
    auto bring_values = [&](int unit_at) {
#pragma unroll
        for (int n = 0; n < kSub; ++n) {
            const char *at = v_base + offset_of(unit_at, n);
#pragma unroll
            for (int j = 0; j < S::kValueLoads; ++j)
                v[n][j] = read<ONCE>(reinterpret_cast<const Words<S::kValueBytes / 4> *>(at + value_key(j) * row_bytes + v_offset + 256 * value_part(j)));
        }
    };
    auto transposed_values = [&](int n, int d) {  // columns 16 d.. of keys 16 n.. of the unit in LDS
        v4f16 part[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int key = 16 * (n + h) + 4 * quarter + col / 4, at = 2 * d + col % 4 / 2;
            part[h] = read_transposed(v_lds + key * S::kRowBytes + v_piece<S::kRowBytes>(key, at) * 16 + col % 2 * 8);
        }
        return __builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7);
    };
    auto take = [&](int unit_at, auto more) {
        const unsigned there = there_next;
        const int key0 = reach.key_of(unit_at);
        v4f32 s[TILES][kSub];
#pragma unroll
        for (int n = 0; n < kSub; ++n)
#pragma unroll
            for (int m = 0; m < TILES; ++m) s[m][n] = v4f32{};
#pragma unroll
        for (int t = 0; t < S::kKeyLoads; ++t)
#pragma unroll
            for (int n = 0; n < kSub; ++n)
#pragma unroll
                for (int m = 0; m < TILES; ++m) {
                    if constexpr (S::kHalf) {
                        s[m][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8f16, k[n][t]), __builtin_bit_cast(v8f16, r.q[m][t]), s[m][n], 0, 0, 0);
                    } else {
                        const v4f32 piece = __builtin_bit_cast(v4f32, k[n][t]);
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[m][n] = __builtin_amdgcn_mfma_f32_16x16x4f32(piece[e], r.q[m][t][e], s[m][n], 0, 0, 0);
                    }
                }
        products_done();
        if constexpr (decltype(more)::value) bring_keys(unit_at + 1);
        __builtin_amdgcn_sched_barrier(0);
        const bool all = there == (1u << kSub) - 1 && key0 + kKeys <= all_end && (key0 >= all_begin || key0 + kKeys <= a.sinks);
        if (!all) {
#pragma unroll
            for (int n = 0; n < kSub; ++n) {
                const bool is = there >> n & 1u;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int key = key0 + 16 * n + 4 * quarter + i;
#pragma unroll
                    for (int m = 0; m < TILES; ++m) s[m][n][i] = is && key < end[m] && (key >= begin[m] || key < a.sinks) ? s[m][n][i] : -INFINITY;
                }
                // (a key that nobody sees has probability 0, but 0 times what its row of V may hold need not be 0)
#pragma unroll
                for (int j = 0; j < S::kValueLoads; ++j) {
                    const int key = key0 + 16 * n + value_key(j) + v_key;
                    const bool use = is && key < seen_end && (key >= seen_begin || key < a.sinks);
#pragma unroll
                    for (int w = 0; w < S::kValueBytes / 4; ++w) v[n][j][w] = use ? v[n][j][w] : 0;
                }
            }
        }
        if constexpr (S::kHalf) {
#pragma unroll
            for (int n = 0; n < kSub; ++n)
#pragma unroll
                for (int j = 0; j < S::kValueLoads; ++j) {
                    const int key = 16 * n + value_key(j) + v_key;
                    *reinterpret_cast<Words<4> *>(v_lds + key * S::kRowBytes + v_piece<S::kRowBytes>(key, lane % kPieces) * 16) = v[n][j];
                }
            asm volatile("" ::: "memory");
            __builtin_amdgcn_wave_barrier();
            if constexpr (decltype(more)::value) bring_values(unit_at + 1);
            __builtin_amdgcn_sched_barrier(0);
        }
        unsigned least = ~0u;  // of the probabilities that are not 0, as bits and less 1
#pragma unroll
        for (int m = 0; m < TILES; ++m) {
            float top = s[m][0][0];
#pragma unroll
            for (int n = 0; n < kSub; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) top = fmaxf(top, s[m][n][i]);
            // sums are scaled anew only when some maximum has risen by more than they bear
            if (__any((top - r.top[m]) * a.scale > S::kSlack)) {
                const float high = fmaxf(r.top[m], quarters_max(top)), shrink = __builtin_amdgcn_exp2f((r.top[m] - high) * a.scale);
                r.top[m] = high;
                r.sum[m] *= shrink;
#pragma unroll
                for (int d = 0; d < D / 16; ++d) r.ctx[m][d] *= shrink;
            }
#pragma unroll
            for (int n = 0; n < kSub; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    s[m][n][i] = __builtin_amdgcn_exp2f(fmaf(s[m][n][i] - r.top[m], a.scale, S::kRaise));
                    r.sum[m] += s[m][n][i];
                    if constexpr (S::kHalf) {
                        const unsigned bits = __builtin_bit_cast(unsigned, s[m][n][i]) - 1;
                        least = bits < least ? bits : least;
                    }
                }
        }
        [[maybe_unused]] const bool some_small = S::kHalf && __any(least < __builtin_bit_cast(unsigned, kSmall) - 1);
        if constexpr (S::kHalf) {
            // (Sums are scaled by a power of two in place, which keeps them as they are, 2^99 at most: sums of their own would be 32 registers more.
            // So would all of V, which is read anew for each product, and copies of sums and probabilities, which the pins prevent.)
            if (some_small) {
#pragma unroll
                for (int m = 0; m < TILES; ++m)
#pragma unroll
                    for (int d = 0; d < D / 16; ++d) {
                        pin_registers(r.ctx[m][d]);
                        r.ctx[m][d] *= kLeftOverBy;
                    }
#pragma unroll
                for (int n = 0; n < kSub; n += 2) {
                    v8f16 p[TILES], low[TILES];
#pragma unroll
                    for (int m = 0; m < TILES; ++m)
#pragma unroll
                        for (int i = 0; i < 8; i += 2) {
                            v2f16 x, y;
                            left_over(s[m][n + i / 4][i % 4], s[m][n + i / 4][i % 4 + 1], x, y);
                            p[m][i] = x[0], p[m][i + 1] = x[1], low[m][i] = y[0], low[m][i + 1] = y[1];
                        }
#pragma unroll
                    for (int d = 0; d < D / 16; ++d) {
                        asm volatile("" ::: "memory");
                        const v8f16 x = finite(transposed_values(n, d));
#pragma unroll
                        for (int m = 0; m < TILES; ++m) {
                            r.ctx[m][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, low[m], r.ctx[m][d], 0, 0, 0);
                            r.ctx[m][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, p[m], r.ctx[m][d], 0, 0, 0);
                        }
                    }
                }
                products_done();
#pragma unroll
                for (int m = 0; m < TILES; ++m)
#pragma unroll
                    for (int d = 0; d < D / 16; ++d) {
                        r.ctx[m][d] *= 1 / kLeftOverBy;
                        pin_registers(r.ctx[m][d]);
                    }
                asm volatile("" ::: "memory");
            }
#pragma unroll
            for (int m = 0; m < TILES; ++m)
#pragma unroll
                for (int n = 0; n < kSub; ++n) pin_registers(s[m][n]);
#pragma unroll
            for (int n = 0; n < kSub; n += 2) {
                v8f16 p[TILES], low[TILES];  // of the keys that the transposed V has in the same places
#pragma unroll
                for (int m = 0; m < TILES; ++m)
#pragma unroll
                    for (int i = 0; i < 8; i += 2) {
                        v2f16 x, y;
                        two_terms(s[m][n + i / 4][i % 4], s[m][n + i / 4][i % 4 + 1], x, y);
                        p[m][i] = x[0], p[m][i + 1] = x[1], low[m][i] = y[0], low[m][i + 1] = y[1];
                    }
#pragma unroll
                for (int d = 0; d < D / 16; ++d) {
                    const v8f16 x = transposed_values(n, d);
#pragma unroll
                    for (int m = 0; m < TILES; ++m) {
                        r.ctx[m][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, low[m], r.ctx[m][d], 0, 0, 0);
                        r.ctx[m][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, p[m], r.ctx[m][d], 0, 0, 0);
                    }
                }
            }
            asm volatile("" ::: "memory");
            __builtin_amdgcn_wave_barrier();
        } else {
#pragma unroll
            for (int n = 0; n < kSub; ++n)
#pragma unroll
                for (int j = 0; j < S::kValueLoads; ++j) {
                    Words<S::kValueBytes / 4> words = v[n][j];
                    pin_registers(words);  // (taken apart here, not where they arrive)
                    const Numbers<T, S::kColumns> piece = __builtin_bit_cast(Numbers<T, S::kColumns>, words);
#pragma unroll
                    for (int e = 0; e < S::kColumns; ++e)
#pragma unroll
                        for (int m = 0; m < TILES; ++m) {
                            v4f32 &to = r.ctx[m][value_part(j) * S::kColumns + e];
                            to = __builtin_amdgcn_mfma_f32_16x16x4f32((float) piece[e], s[m][n][value_key(j)], to, 0, 0, 0);
                        }
                }
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (decltype(more)::value) bring_values(unit_at + 1);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    if (x < until) {
        bring_keys(x);
        bring_values(x);
        for (; x + 1 < until; ++x) take(x, std::true_type());
        take(x, std::false_type());
    }
    products_done();

    // the four wavefronts' sums: rows of D results, the maximum and the sum
    const int present = rows - row0 < kRows ? rows - row0 : kRows;
    float *merge = reinterpret_cast<float *>(smem + kShared);
    __syncthreads();  // nobody reads V any more
#pragma unroll
    for (int m = 0; m < TILES; ++m) {
        float sum = r.sum[m] + __shfl_xor(r.sum[m], 16, kWave);
        sum += __shfl_xor(sum, 32, kWave);
        const int row = 16 * m + col;
        if (row < present) {
            float *to = merge + (wave * present + row) * S::kPitch;
            if constexpr (S::kHalf) {
#pragma unroll
                for (int d = 0; d < D / 16; ++d) *reinterpret_cast<v4f32 *>(to + 16 * d + 4 * quarter) = r.ctx[m][d];
            } else {
#pragma unroll
                for (int d = 0; d < D / 16; d += 2)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        *reinterpret_cast<v2f32 *>(to + d / S::kColumns * 64 + (4 * quarter + i) * S::kColumns + d % S::kColumns) =
                                v2f32{r.ctx[m][d][i], r.ctx[m][d + 1][i]};
            }
            if (quarter == 0) to[D] = r.top[m], to[D + 1] = sum;
        }
    }
    __syncthreads();
    constexpr int kQuads = D / 4;  // a thread has four columns of a row
    for (int i = threadIdx.x; i < present * kQuads; i += kBlock) {
        const int row = i / kQuads, d = (i - row * kQuads) * 4;
        float top = kNone;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) top = fmaxf(top, merge[(w * present + row) * S::kPitch + D]);
        v4f32 x4 = v4f32{};
        float total = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float *of = merge + (w * present + row) * S::kPitch;
            const float f = __builtin_amdgcn_exp2f((of[D] - top) * a.scale);
            total += of[D + 1] * f;
            x4 += *reinterpret_cast<const v4f32 *>(of + d) * f;
        }
        const int out_row = row0 + row, query = share == 1 ? out_row : out_row / share, p = reach.first + query;
        const bool there = p >= 0 && p < reach.length;
        if (pieces == 1) {
            T *ctx = (T *) a.ctx + (size_t) (sequence * a.q_rows + query) * a.ld_ctx + (size_t) (kv_head * share + out_row - query * share) * D + d;
            const float by = there && total != 0.f ? 1.f / total : 0.f;  // (a sum that is no number stays none)
            store4(ctx, by != 0.f ? x4 * by : v4f32{});
        } else {
            float *to = a.partials + ((size_t) blockIdx.x * plan.slot_rows + row) * S::kPitch;
            *reinterpret_cast<v4f32 *>(to + d) = there ? x4 : v4f32{};
            if (d == 0) to[D] = there ? top : kNone, to[D + 1] = there ? total : 0.f;
        }
    }
    // where a problem's pieces stand, for those who join them
    if (plan.pieces != 0 && piece == 0 && threadIdx.x == 0)
        reinterpret_cast<v2i32 *>(a.partials + (size_t) (plan.pieces + plan.problems) * plan.slot_rows * S::kPitch)[(size_t) entry * a.kv_heads + kv_head] =
                v2i32{(int) blockIdx.x, pieces};
}

// The pieces' sums of a row joined, COLUMNS at a time, by WAVES wavefronts: COLUMNS / 4 lanes to a piece, their maxima and sums a lane each.
template <typename T, int D, int COLUMNS, int WAVES>
__global__ __launch_bounds__(WAVES * kWave < kBlock ? kBlock : WAVES * kWave) void attention_paged_join_kernel(PagedArgs a, PagedPlan plan) {
    typedef Shape<T, D> S;
    constexpr int kQuads = COLUMNS / 4, kAtOnce = kWave / kQuads, kPer = WAVES < 4 ? 4 / WAVES : 1, kAhead = kAtOnce >= 8 ? 4 : 8;
    __shared__ float shared[WAVES > 1 ? WAVES * S::kPitch : 1];
    const int wave = wave_in_block(), lane = threadIdx.x & (kWave - 1), share = a.heads / a.kv_heads, rows = a.q_rows * share;
    const int i = blockIdx.x * kPer + wave / WAVES, part = wave % WAVES;
    const int problem = i / plan.slot_rows, row = i - problem * plan.slot_rows;
    if (problem >= plan.problems) return;
    const v2i32 note = reinterpret_cast<const v2i32 *>(a.partials + (size_t) (plan.pieces + plan.problems) * plan.slot_rows * S::kPitch)[problem];
    const int pieces = uniform(note[1]);
    if (pieces == 1) return;  // its one workgroup has written it
    const int entry = problem / a.kv_heads, kv_head = problem - entry * a.kv_heads;
    const int tile = plan.row_tiles > 1 ? entry / a.batch : 0, sequence = entry - tile * a.batch, out_row = tile * plan.rows + row;
    if (out_row >= rows) return;
    const size_t step = (size_t) plan.slot_rows * S::kPitch;
    const float *first = a.partials + uniform(note[0]) * step + row * S::kPitch;
    const int until = pieces * (part + 1) / WAVES, at = lane / kQuads, d = blockIdx.y * COLUMNS + lane % kQuads * 4;
    float top = kNone, sum = 0.f;
    v4f32 x = v4f32{};
    for (int n0 = pieces * part / WAVES; n0 < until; n0 += kWave) {
        // all that there is to read at once, where that is little (past the last piece the first one again)
        const int here = until - n0 < kWave ? until - n0 : kWave;
        const float *of = first + (n0 + (lane < here ? lane : 0)) * step;
        const v2f32 mine = *reinterpret_cast<const v2f32 *>(of + D);
        v4f32 y[kAhead];
        auto bring = [&](int n) {
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const int m = n + u * kAtOnce + at;
                y[u] = *reinterpret_cast<const v4f32 *>(first + (n0 + (m < here ? m : 0)) * step + d);
            }
        };
        bring(0);
        const float high = fmaxf(top, wave_max(mine[0])), shrink = __builtin_amdgcn_exp2f((top - high) * a.scale);
        const float weight = lane < here ? __builtin_amdgcn_exp2f((mine[0] - high) * a.scale) : 0.f;
        top = high;
        sum = sum * shrink + wave_sum(weight * mine[1]);
        x *= shrink;
        for (int n = 0;;) {
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const int m = n + u * kAtOnce + at;
                const float f = __shfl(weight, m < here ? m : 0, kWave);
                if (m < here) x += y[u] * f;
            }
            n += kAtOnce * kAhead;
            if (n >= here) break;
            bring(n);
        }
    }
#pragma unroll
    for (int m = kQuads; m < kWave; m *= 2)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] += __shfl_xor(x[e], m, kWave);
    if constexpr (WAVES > 1) {
        float *mine = shared + part * S::kPitch;
        if (at == 0) *reinterpret_cast<v4f32 *>(mine + d) = x;
        if (lane == 0) mine[D] = top, mine[D + 1] = sum;
        __syncthreads();
        if (part != 0) return;
        float high = kNone;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) high = fmaxf(high, shared[w * S::kPitch + D]);
        x = v4f32{}, sum = 0.f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            const float f = __builtin_amdgcn_exp2f((shared[w * S::kPitch + D] - high) * a.scale);
            sum += shared[w * S::kPitch + D + 1] * f;
            x += *reinterpret_cast<const v4f32 *>(shared + w * S::kPitch + d) * f;
        }
    }
    if (at != 0) return;
    const int query = out_row / share;
    T *ctx = (T *) a.ctx + (size_t) (sequence * a.q_rows + query) * a.ld_ctx + (size_t) (kv_head * share + out_row - query * share) * D + d;
    const float by = sum != 0.f ? 1.f / sum : 0.f;
    store4(ctx, by != 0.f ? x * by : v4f32{});
}

// How a call is cut.  Microseconds of calls in a captured graph, over inputs in turn, fp16 where nothing is said:
//
// Rows of a tile, where there are more than 16, 16 / 32, by what K and V of a sequence and of all may come to: 8 x 1 over up to 4000, 32 heads to 1 of 64 (1
// MB, 8) 11.2 / 11.9; 32 x 2 over up to 1000, 48 heads to 4 of 64 (0.25, 33) 10.3 / 12.9; 8 x 32 over up to 2000, 16 of 64 (0.5, 65) 15.2 / 18.3; 16 x
// 4 over up to 4000, 64 to 4 of 64 (1, 65) 24.6 / 21.2; 8 x 4 over up to 4000, 32 to 4 of 128 (2, 65) 20.6 / 18.1; 1 x 8 over up to 16800, 96 to 12 of 128
// (17, 206) 47 / 34; fp32, 8 x 1 over up to 8000, 32 to 1 of 128 (8, 65) 19.1 / 21.8; 4 x 4 over up to 16000, 32 to 4 of 64 (8, 131) 30.1 / 25.5.
//
// A workgroup to a problem / pieces and a join.  Few problems are cut where they have more than 256 KB, many where they have more than 2 KB for each of
// their number: 1 x 1 over 2000 keys, 16 heads of 64 (16 problems of 0.5 MB) 14.3 / 10.4; 8 x 1 over up to 1000, 4 of 128 (32 of 0.5) 13.7 / 11.3;
// 128 x 1 over up to 1500, 2 of 64 (256 of 0.4) 13.9 / 18.4; 256 x 1 over up to 512, 12 of 64 (256 x 12 of 0.1) 42 / 52; 128 x 1 over up to 2048, 12 of 64
// (1536 of 0.5, tables for 4) 85 / 81; 1 x 1 over 131072, 2 of 128 (2 of 67) 1781 / 31.  More than 1280 sequences and tiles never are, as every
// workgroup looks through all of them, which short sequences in wide tables have nothing to set against: 1 of 64, tables for 32768 keys, over up to 300 / 1500
// / 6000 each, 512 x 1 9.0 / 15.5, 27 / 31, 95 / 80; 1024 x 1 12.6 / 25.9, 48 / 52, 179 / 152; 1280 x 1 14.2 / 32.4, 58 / 63, 217 / 189; 1536 x 1 16.7 / 39.1,
// 66 / 73, 254 / 226; 2048 x 1 22 / 53, 85 / 97, 319 / 299; 4096 x 1 37 / 108, 153 / 193, 585 / 600; 2 of 128, tables for 8192, over up to 300 / 2000 / 8000,
// 768 x 1 30 / 47, 166 / 161, 648 / 581; 1024 x 1 39 / 43, 208 / 208, 805 / 811.
//
// Pieces of all.  With few problems as many as fit the card together, a workgroup or two to a unit of it, which leaves the join the least to do; 256 /
// 512 / 1024 / 2048: 4 x 1 over up to 30000, 4 of 128 (16 problems) 31.0 / 30.7 / 32.9 / 33.8; 1 x 8 over up to 16800, 96 heads to 12 of 128 (24) 34 / 44
// / 50 / 76; 48 x 1 over up to 4000, 2 of 128 (96) 31.3 / 26.3 / 29.3 / 29.9.  (Less one / half a one for each problem, as a problem ends with half a piece
// where lengths differ: fp32, 4 x 8 over up to 8000, 32 heads to 4 of 64 (64 problems: four tiles of 16) 35.4 / 29.4, 48 x 1 31.3 / 27.3; 1 x 8 over up to
// 16800, of one length, 34 / 55, so not where one round of workgroups is all.)  Many problems of unlike lengths want more, which are handed out as
// units come free, up to 2048, but what the pieces write and the join reads should be little next to K and V: 1/64 of them, or three pieces to a
// problem; and a last round of workgroups that has few of them costs as much as a full one, so they are whole rounds of 256.
// 2048 / this: 64 x 1 over up to 4096, 4 of 128 (256) 53.1 / 53.2; 32 x 1, window 4096, 4 of 128 (128) 46.0 / 46.9; 32 x 1 over
// up to 4096, 16 to 4 of 128 (128) 35.9 / 32.6, 64 to 4 (16 rows) 43.1 / 34.8, 32 x 5 over up to 4000, 16 to 4 (20 rows) 52 / 36.5; 16 x 8 over up to
// 4000, 64 to 8 (256, 32 rows) 75 / 63; 512 x 1 over up to 6000, 1 of 64 78.3 / 79.0.
//
// Units of a piece at least (a wavefront has one then), 4 / 8: 8 x 1 over up to 1000, 4 of 128 (32 problems of 32) 11.1 / 12.2; fp32, 9 x 5 over up to 1000,
// 12 of 64 (108 of 32) 15.0 / 16.7, 8 x 1 (96) 13.9 / 13.5; 24 x 4 over up to 1000, 32 to 8 of 128 (192 of 32) 20.3 / 19.0; 16 x 1 over up to 500,
// tables for 8192, 12 of 64 14.3 / 16.8.
PagedPlan plan_paged(bool half_precision, int batch, int heads, int kv_heads, int q_rows, long long limit, int head_size, int left, int sinks) {
    PagedPlan plan;
    if (left >= kFar) left = -1;
    const long long rows = (long long) q_rows * (heads / kv_heads);
    const int row_bytes = head_size * (half_precision ? 2 : 4), keys = row_bytes == 512 ? 16 : 32;
    const long long most = left >= 0 && (long long) left + q_rows + sinks < limit ? (long long) left + q_rows + sinks : limit;  // keys of a sequence
    const long long bytes = most * 2 * row_bytes, of = (long long) batch * kv_heads, all_bytes = of < (1ll << 62) / bytes ? of * bytes : 1ll << 62;
    plan.rows = rows > 16 && bytes >= 768 << 10 && all_bytes >= (half_precision ? 24 << 20 : 96 << 20) ? 32 : 16;
    plan.row_tiles = (int) ((rows + plan.rows - 1) / plan.rows);
    plan.slot_rows = (int) (rows < plan.rows ? rows : plan.rows);
    plan.problems = (long long) batch * kv_heads * plan.row_tiles, plan.bytes = all_bytes;
    plan.pieces = 0, plan.floats = 0, plan.once = false;
    long long reach = limit;  // the most keys that a tile of rows sees, and how many units of them
    if (left >= 0 && (long long) left + plan.rows + sinks < reach) reach = (long long) left + plan.rows + sinks;
    const long long units = (reach + keys - 1) / keys + (left >= 0 ? 2 : 0), all = plan.problems * units;
    const long long uncut = plan.problems / 8 < 16 ? 16 : plan.problems / 8 < 256 ? plan.problems / 8 : 256;  // (16 KB each)
    if (units * keys * row_bytes <= uncut * 8192 || (long long) batch * plan.row_tiles > 1280 || all >= 1 << 30) return plan;  // (units are counted in 32 bits)
    if (plan.problems <= 32) {
        plan.pieces = 256 - (int) plan.problems;
    } else if (plan.problems <= 100) {
        plan.pieces = 512 - (int) plan.problems / 2;
    } else {
        const long long worth = all_bytes / 64 / (plan.slot_rows * (head_size + 4) * 8), few = 3 * plan.problems;
        const long long rounds = ((worth > few ? worth : few) + 255) / 256;
        plan.pieces = rounds < 8 ? (int) (256 * rounds - plan.problems / 2) : 2048;
    }
    if ((all + kLeast - 1) / kLeast < plan.pieces) plan.pieces = (int) ((all + kLeast - 1) / kLeast);
    plan.floats = (size_t) (plan.pieces + plan.problems) * plan.slot_rows * (head_size + 4) + 2 * (size_t) plan.problems;
    return plan;
}

// Whether K and V are read past the caches: once, by one tile of rows, and where neither the pools nor what the tables have room for stays in the 256 MB
// behind the L2 caches until the next call, from 101 MB on.  Microseconds without / with, four sets of inputs in turn / sixteen, of which little is there
// still, in pools of 1 GB: 64 x 1 over up to 4096, 4 of 128 (322 MB read, tables for 537) 67.2 / 60.9, 65.4 / 58.5; 48 x 1 over up to 4000, 2 of 128 (116,
// 201) 29.7 / 27.6, 29.4 / 27.4; 64 x 1 over up to 1000, 4 of 128 (80, 134) 20.2 / 23.6, 22.7 / 23.4; below 101 MB of tables 128 x 1 over up to 1500, 2 of 64
// (58, 98) 15.5 / 18.6, 18.7 / 18.3; 16 x 1 over up to 500, 12 of 64 (15, 25) 7.8 / 8.2, 7.6 / 8.0; fp32, 9 x 5 over up to 1000, 12 of 64 (33, 57) 15.7 /
// 16.5, 16.7 / 16.3.  Tables that are far wider than sequences are long take the same side as long sequences: 64 x 1 over up to 500 in tables for 8192, 4 of 128
// (40) 16.0 / 16.7, 18.3 / 17.8.  Two tiles of 32 rows, 1 x 8 over up to 16800, 96 heads to 12 of 128, 34 / 41.
bool read_once(const PagedPlan &plan, long long pages, int page, int kv_heads, int row_bytes) {
    constexpr long long kLarge = 96ll << 20;
    return plan.row_tiles == 1 && plan.bytes >= kLarge && 2 * pages * page * kv_heads * row_bytes >= kLarge;
}

template <typename T, int D, int TILES, bool ONCE>
int run_paged(const PagedArgs &a, const PagedPlan &plan, hipStream_t stream) {
    static std::atomic<unsigned long long> done{0};
    typedef Shape<T, D> S;
    const unsigned merge = (unsigned) (4 * plan.slot_rows * S::kPitch * 4), lds = kShared + (merge > 4 * S::kValueLds ? merge : 4 * S::kValueLds);
    if (lds > 48 * 1024 && !allow_large_lds(attention_paged_kernel<T, D, TILES, ONCE>, done)) return CUBERT_UNSUPPORTED;
    const int rc = launch_lds(attention_paged_kernel<T, D, TILES, ONCE>, dim3((unsigned) (plan.pieces + plan.problems)), dim3(kBlock), lds, stream, a, plan);
    if (rc != 0 || plan.pieces == 0) return rc;
    const unsigned joins = (unsigned) (plan.problems * plan.slot_rows);
    // Wavefronts to a row, by its pieces on average, 1 / 4 / 16 (which have 32 columns of it): fp32, 9 x 5 over up to 1000, 12 of 64 (8 pieces)
    // 15.2 / 15.6 / 20.6 us the whole call; fp16, 64 x 1 over up to 4096 (8) 54.1 / 54.9 / 79.2; 1 x 1 over 60000, 1 of 128 (234) 27.1 / 17.0 / 15.1.
    const int of_problem = plan.pieces / (int) plan.problems;
    if (of_problem <= 16) return launch(attention_paged_join_kernel<T, D, D, 1>, dim3((joins + 3) / 4), dim3(kBlock), stream, a, plan);
    if (of_problem <= 64) return launch(attention_paged_join_kernel<T, D, D, 4>, dim3(joins), dim3(kBlock), stream, a, plan);
    return launch(attention_paged_join_kernel<T, D, 32, 16>, dim3(joins, D / 32), dim3(16 * kWave), stream, a, plan);
}

template <typename T, int D>
int run_paged_size(const PagedArgs &a, const PagedPlan &plan, hipStream_t stream) {
    if (plan.once) return plan.rows == 16 ? run_paged<T, D, 1, true>(a, plan, stream) : run_paged<T, D, 2, true>(a, plan, stream);
    return plan.rows == 16 ? run_paged<T, D, 1, false>(a, plan, stream) : run_paged<T, D, 2, false>(a, plan, stream);
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
    // (a launch holds less than 2^32 threads, and rows are counted in 32 bits)
    if ((long long) batch * q_rows >= 1ll << 31 || (long long) batch * kv_heads >= 1 << 24 || (long long) q_rows * (heads / kv_heads) >= 1 << 30)
        return CUBERT_UNSUPPORTED;
    PagedPlan plan = plan_paged(sizeof(T) == 2, batch, heads, kv_heads, q_rows, (long long) width * page, head_size, left, sinks);
    if (plan.problems * plan.rows >= 1 << 24) return CUBERT_UNSUPPORTED;
    plan.once = read_once(plan, pages, page, kv_heads, head_size * (int) sizeof(T));
    if (plan.pieces != 0 && (partials == nullptr || partial_floats < plan.floats || !is_aligned(partials, 16))) plan.pieces = 0;
    if (head_size == 32) return run_paged_size<T, 32>(a, plan, (hipStream_t) stream);
    if (head_size == 64) return run_paged_size<T, 64>(a, plan, (hipStream_t) stream);
    return run_paged_size<T, 128>(a, plan, (hipStream_t) stream);
}

}  // namespace
}  // namespace cubert

using cubert::half_t;

extern "C" {

size_t cubert_attention_paged_partials(int half_precision, int batch, int heads, int kv_heads, int q_rows, int width, int page, int head_size, int left,
                                       int sinks) {
    if (batch < 1 || heads < 1 || kv_heads < 1 || heads % kv_heads != 0 || q_rows < 1 || width < 1 || page < 1 || head_size < 1 || sinks < 0) return 0;
    if ((long long) batch * kv_heads >= 1 << 24 || (long long) q_rows * (heads / kv_heads) >= 1 << 30 || (long long) width * page > cubert::kFar) return 0;  // refused
    const cubert::PagedPlan plan = cubert::plan_paged(half_precision != 0, batch, heads, kv_heads, q_rows, (long long) width * page, head_size, left, sinks);
    return plan.problems * plan.rows >= 1 << 24 ? 0 : plan.floats;
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
