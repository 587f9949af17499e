// A key/value cache in pages: which page of a sequence is which, where new tokens go, and keys and values on their way there.
//
//     page i of sequence b is table[b, i]; its token at position p has slot table[b, p / page] * page + p % page
//
// Pages of nobody stand on a stack of some places, free[0 .. *free_count), and are taken from its top.

#include "cubert_kernels.h"
#include "device_common.h"
#include "paged.h"

namespace cubert {
namespace {

__device__ __forceinline__ int pages_of(int tokens, int shift) { return tokens == 0 ? 0 : ((tokens - 1) >> shift) + 1; }

constexpr int kSpan = 1024;  // slots of a workgroup

struct ExtendArgs {
    int *table;
    const int *lengths, *counts, *free, *free_count;
    int *slots, *lengths_out, *free_out;
    int width, ld_table, places, pages, shift, batch, rows;  // places of the stack, pages that there are
    int spans;  // of kSpan slots, of a workgroup
};

// What a sequence has and asks for: `need` pages more for `count` tokens; none, and no tokens, where its table has no room for them.
struct Growth {
    int length, count, need;
    bool fits;

    __device__ __forceinline__ Growth(const ExtendArgs &a, int b) {
        const int room = a.width << a.shift;
        length = clamp_to(a.lengths[b], 0, room);
        count = a.counts != nullptr ? clamp_to(a.counts[b], 0, a.rows) : a.rows;
        fits = count <= room - length;
        need = fits ? pages_of(length + count, a.shift) - pages_of(length, a.shift) : 0;
    }
};

// The sum over a workgroup's threads.
__device__ __forceinline__ int block_sum(int x, int *shared) {
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) x += __shfl_xor(x, d, kWave);
    if ((threadIdx.x & (kWave - 1)) == 0) shared[threadIdx.x / kWave] = x;
    __syncthreads();
    int sum = 0;
#pragma unroll
    for (int w = 0; w < kBlock / kWave; ++w) sum += shared[w];
    __syncthreads();
    return sum;
}

// A sequence is served if it needs no page, or if all that is asked for up to it is there.  A workgroup has kSpan slots, or several times as many, one
// after the other; it adds up what the sequences before them ask for (a few bytes per sequence, which the cache has), so that none waits for another.
__global__ __launch_bounds__(kBlock) void paged_extend_kernel(ExtendArgs a) {
    __shared__ int shared[kBlock / kWave], starts[kSpan], lengths[kSpan], counts[kSpan];
    const int rows = a.rows > 0 ? a.rows : 1, total = a.batch * rows, thread = threadIdx.x, lane = thread & (kWave - 1);
    const int there = clamp_to(*a.free_count, 0, a.places);
    if (total == 0) {
        if (thread == 0) *a.free_out = there;
        return;
    }
    const int spans = (total - 1) / kSpan + 1, begin = blockIdx.x * a.spans, end = begin + a.spans < spans ? begin + a.spans : spans;
    int before = 0, first = 0;  // what the sequences before `first` ask for
    for (int span = begin; span < end; ++span) {
        const int from = span * kSpan, until = total - from < kSpan ? total : from + kSpan;
        const int next = from / rows, last = (until - 1) / rows;  // the sequences that these slots belong to
        int passed = 0;
        for (int b = first + thread; b < next; b += kBlock) passed += Growth(a, b).need;
        before += block_sum(passed, shared);
        first = next;
        // sequences in runs of kSpan / kBlock to a thread
        constexpr int kRun = kSpan / kBlock;
        int need[kRun], sum = 0;
#pragma unroll
        for (int n = 0; n < kRun; ++n) {
            const int at = thread * kRun + n;
            need[n] = 0;
            if (first + at <= last) {
                const Growth g(a, first + at);
                need[n] = g.need, lengths[at] = g.length, counts[at] = g.fits ? g.count : 0;
            }
            sum += need[n];
        }
        int through = sum;
#pragma unroll
        for (int d = 1; d < kWave; d *= 2) {
            const int other = __shfl_up(through, d, kWave);
            through += lane >= d ? other : 0;
        }
        if (lane == kWave - 1) shared[thread / kWave] = through;
        __syncthreads();
        int start = before + through - sum;
#pragma unroll
        for (int w = 0; w < kBlock / kWave; ++w)
            if (w < thread / kWave) start += shared[w];
#pragma unroll
        for (int n = 0; n < kRun; ++n) {
            const int at = thread * kRun + n, b = first + at;
            if (b <= last) {
                starts[at] = start;
                const bool granted = need[n] == 0 || start + need[n] <= there;
                if (!granted) counts[at] = 0;
                // what stays on the stack is what the first one left that did not get its pages, or else the last one (several workgroups may
                // have its slots, and all write this)
                if (start <= there && (start + need[n] > there || b == a.batch - 1)) *a.free_out = there - start - (granted ? need[n] : 0);
            }
            start += need[n];
        }
        __syncthreads();
        for (int i = from + thread; i < until; i += kBlock) {
            const int b = i / rows, t = i - b * rows, at = b - first, length = lengths[at], count = counts[at];
            if (t == 0) a.lengths_out[b] = length + count;
            if (a.rows == 0) continue;
            int slot = -1;
            if (t < count) {
                const int p = length + t, index = p >> a.shift, held = pages_of(length, a.shift);
                int *entry = a.table + (size_t) b * a.ld_table + index;
                int page;
                if (index < held) {
                    page = *entry;
                } else {
                    page = a.free[there - 1 - (starts[at] + index - held)];
                    if ((p & ((1 << a.shift) - 1)) == 0) *entry = page;
                }
                if (page >= 0 && page < a.pages) slot = (page << a.shift) + (p & ((1 << a.shift) - 1));
            }
            a.slots[i] = slot;
        }
        __syncthreads();  // (the next span's sequences take their places)
    }
}

// ---- and back ---------------------------------------------------------------

struct CutArgs {
    const int *table, *lengths, *keep;
    int *free;
    const int *free_count;
    int *lengths_out, *free_out, *returned;
    int width, ld_table, places, pages, shift, batch;
};

struct Shrink {
    int keep, begin, end;  // the entries of the table's row that go

    __device__ __forceinline__ Shrink(const CutArgs &a, int b) {
        const int length = clamp_to(a.lengths[b], 0, a.width << a.shift);
        keep = a.keep != nullptr ? clamp_to(a.keep[b], 0, length) : 0;
        begin = pages_of(keep, a.shift), end = pages_of(length, a.shift);
    }
};

constexpr int kAhead = 8;  // entries of a lane that are on their way together

// How many pages a sequence gives back (to a wavefront): entries that are no pages (a window has passed them, and they were taken out) do not
// count.
__device__ __forceinline__ int pages_back(const CutArgs &a, int b, const Shrink &s, int lane) {
    const int *row = a.table + (size_t) b * a.ld_table;
    int count = 0;
    for (int i = s.begin + lane; i < s.end; i += kWave * kAhead) {
        int page[kAhead];
#pragma unroll
        for (int n = 0; n < kAhead; ++n) page[n] = i + n * kWave < s.end ? row[i + n * kWave] : -1;
#pragma unroll
        for (int n = 0; n < kAhead; ++n) count += page[n] >= 0 && page[n] < a.pages ? 1 : 0;
    }
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) count += __shfl_xor(count, d, kWave);
    return count;
}

// They go onto the stack from `height` on, as far as it has room.
__device__ __forceinline__ void put_back(const CutArgs &a, int b, const Shrink &s, long long height, int lane) {
    const int *row = a.table + (size_t) b * a.ld_table;
    const int free_places = height < a.places ? a.places - (int) height : 0;
    int *to = a.free + height;
    int at = 0;
    for (int base = s.begin; base < s.end && at < free_places; base += kWave * kAhead) {
        int page[kAhead];
#pragma unroll
        for (int n = 0; n < kAhead; ++n) {
            const int i = base + n * kWave + lane;
            page[n] = i < s.end ? row[i] : -1;
        }
#pragma unroll
        for (int n = 0; n < kAhead; ++n) {
            const bool is = page[n] >= 0 && page[n] < a.pages;
            const unsigned long long all = __ballot(is);
            const int place = at + __builtin_popcountll(all & ((1ull << lane) - 1));
            if (is && place < free_places) to[place] = page[n];
            at += __builtin_popcountll(all);
        }
    }
}

__global__ __launch_bounds__(kBlock) void paged_cut_count_kernel(CutArgs a) {
    const int b = blockIdx.x * (kBlock / kWave) + wave_in_block(), lane = threadIdx.x & (kWave - 1);
    if (b >= a.batch) return;
    const Shrink s(a, b);
    const int count = pages_back(a, b, s, lane);
    if (lane == 0) a.returned[b] = count, a.lengths_out[b] = s.keep;
}

// A wavefront per sequence puts its pages onto the stack, behind those of the sequences before it.
__global__ __launch_bounds__(kBlock) void paged_cut_kernel(CutArgs a) {
    const int b = blockIdx.x * (kBlock / kWave) + wave_in_block(), lane = threadIdx.x & (kWave - 1);
    const int there = clamp_to(*a.free_count, 0, a.places);
    if (b >= a.batch) return;
    const Shrink s(a, b);
    long long before = 0;
    for (int i = lane; i < b; i += kWave) before += a.returned[i];
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) before += __shfl_xor(before, d, kWave);
    const long long height = there + before;
    if (b == a.batch - 1 && lane == 0) {
        const long long all = height + a.returned[b];
        *a.free_out = (int) (all < a.places ? all : a.places);
    }
    put_back(a, b, s, height, lane);
}

// Few sequences with short tables: both in one workgroup of 16 wavefronts, which take the sequences in turn.
constexpr int kFewSequences = 64, kFewWaves = 16;
constexpr long long kFewEntries = 1 << 15;

__global__ __launch_bounds__(kFewWaves * kWave) void paged_cut_few_kernel(CutArgs a) {
    __shared__ int back[kFewSequences];
    const int wave = wave_in_block(), lane = threadIdx.x & (kWave - 1);
    const int there = clamp_to(*a.free_count, 0, a.places);
    for (int b = wave; b < a.batch; b += kFewWaves) {
        const Shrink s(a, b);
        const int count = pages_back(a, b, s, lane);
        if (lane == 0) back[b] = count, a.lengths_out[b] = s.keep;
    }
    __syncthreads();
    const int mine = lane < a.batch ? back[lane] : 0;
    int through = mine;
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) {
        const int other = __shfl_up(through, d, kWave);
        through += lane >= d ? other : 0;
    }
    if (wave == 0 && lane == kWave - 1) {
        const long long all = (long long) there + through;
        *a.free_out = (int) (all < a.places ? all : a.places);
    }
    for (int b = wave; b < a.batch; b += kFewWaves)
        put_back(a, b, Shrink(a, b), there + __builtin_amdgcn_readlane(through - mine, b), lane);
}

// One launch / two, microseconds on the GPU: 8 sequences of up to 4096 tokens in pages of 16 4.2 / 5.5, 64 of up to 8192 10.5 / 6.5; as a call, in
// which a second launch and its memory are 4 of the host's, 7.9 / 12.2 and 10.5 / 12.
bool few_to_cut(int batch, int width) { return batch <= kFewSequences && (long long) batch * width <= kFewEntries; }

// ---- rows into pages ----------------------------------------------------------

struct WriteArgs {
    const char *k, *v;
    char *k_pages, *v_pages;
    const int *slots;
    long long page_bytes, head_bytes, row_bytes, from_bytes;
    unsigned tokens, slots_there;
    int shift, pieces_of_head, pieces;  // of 16 bytes, of a head and of all of a token's
};

typedef float v4f32 __attribute__((ext_vector_type(4)));

// A 16-byte piece of a key and of a value to a thread.  Bound by memory: 16 prompts of up to 2048 tokens of 8 heads of 128, 134 MB, in 26.5 us (5.1
// TB/s).  ONCE: past the caches, which large ones leave nothing in, from 64 MB on; microseconds without / with: 16384 tokens of 8 heads of 128 (134 MB) 29.6
// / 25.1, 32768 53.8 / 46.1, 65536 of 2 of 64 (67 MB) 15.1 / 14.5; 131072 of 1 of 32 (33 MB) 8.4 / 9.4.
template <bool ONCE>
__global__ __launch_bounds__(kBlock) void paged_write_kernel(WriteArgs a) {
    const unsigned long long i = (unsigned long long) blockIdx.x * kBlock + threadIdx.x;
    const unsigned token = (unsigned) (i / (unsigned) a.pieces);
    if (token >= a.tokens) return;
    const int piece = (int) (i - (unsigned long long) token * a.pieces), head = piece / a.pieces_of_head;
    const unsigned slot = (unsigned) a.slots[token];
    if (slot >= a.slots_there) return;  // (a negative one is a large one)
    const long long from = token * a.from_bytes + (long long) piece * 16;
    const long long to = (long long) (slot >> a.shift) * a.page_bytes + (long long) (slot & ((1u << a.shift) - 1)) * a.row_bytes +
                         head * a.head_bytes + (piece - head * a.pieces_of_head) * 16;
    const v4f32 *k = (const v4f32 *) (a.k + from), *v = (const v4f32 *) (a.v + from);
    v4f32 *k_to = (v4f32 *) (a.k_pages + to), *v_to = (v4f32 *) (a.v_pages + to);
    if constexpr (ONCE) {
        const v4f32 x = __builtin_nontemporal_load(k), y = __builtin_nontemporal_load(v);
        __builtin_nontemporal_store(x, k_to);
        __builtin_nontemporal_store(y, v_to);
    } else {
        const v4f32 x = *k, y = *v;
        *k_to = x, *v_to = y;
    }
}

// What a sequence asks for or returns is added up by all behind it: by a wavefront for each, when they are cut, by 2048 workgroups at most (eight to a
// unit of the card) when they grow.
constexpr int kMostSequences = 1 << 18, kExtendGroups = 2048;

// What extend and cut have in common: sizes of tables and pages that 32 bits count.
int check_tables(const void *table, int width, int ld_table, const void *lengths, const void *free, const void *free_count, int places, int pages, int page,
                 int batch, const void *lengths_out, const void *free_out) {
    if (width < 1 || ld_table < width || places < 1 || pages < 1 || page < 1 || batch < 0) return CUBERT_BAD_ARGUMENT;
    if (free == nullptr || free_count == nullptr || free_out == nullptr || free_out == free_count) return CUBERT_BAD_ARGUMENT;
    if (batch > 0 && (table == nullptr || lengths == nullptr || lengths_out == nullptr || lengths_out == lengths)) return CUBERT_BAD_ARGUMENT;
    if ((page & (page - 1)) != 0 || batch > kMostSequences) return CUBERT_UNSUPPORTED;
    const long long most = (1ll << 31) - 1;
    if ((long long) width * page > most || (long long) pages * page > most) return CUBERT_UNSUPPORTED;
    return 0;
}

// `count` ints that a call reads or writes.
struct Ints {
    const int *at;
    long long count;

    bool meets(const Ints &other) const {
        if (at == nullptr || other.at == nullptr || count == 0 || other.count == 0) return false;
        const uintptr_t a = (uintptr_t) at, b = (uintptr_t) other.at;
        return a < b + 4 * (unsigned long long) other.count && b < a + 4 * (unsigned long long) count;
    }
};

// Whether what a call writes shares memory with what it reads (workgroups read it that have not begun when others write) or with its other results.
template <int OUT, int IN>
bool results_apart(const Ints (&out)[OUT], const Ints (&in)[IN]) {
    for (int i = 0; i < OUT; ++i) {
        for (int j = 0; j < i; ++j)
            if (out[i].meets(out[j])) return false;
        for (int j = 0; j < IN; ++j)
            if (out[i].meets(in[j])) return false;
    }
    return true;
}

int paged_write(const void *k, const void *v, int ld, const int *slots, int tokens, void *k_pages, void *v_pages, long long page_stride,
                long long head_stride, long long row_stride, int pages, int page, int kv_heads, int head_size, int element, void *stream) {
    if (tokens < 0 || pages < 1 || page < 1 || kv_heads < 1 || head_size < 1 || ld < (long long) kv_heads * head_size) return CUBERT_BAD_ARGUMENT;
    if (!cubert::pages_apart(page_stride, head_stride, row_stride, pages, kv_heads, page, head_size)) return CUBERT_BAD_ARGUMENT;
    if (tokens == 0) return 0;
    if (k == nullptr || v == nullptr || slots == nullptr || k_pages == nullptr || v_pages == nullptr) return CUBERT_BAD_ARGUMENT;
    if ((page & (page - 1)) != 0 || (long long) pages * page >= 1ll << 31) return CUBERT_UNSUPPORTED;
    const int piece = 16 / element;
    if (!is_aligned(k, 16) || !is_aligned(v, 16) || !is_aligned(k_pages, 16) || !is_aligned(v_pages, 16) || ld % piece != 0 || head_size % piece != 0 ||
        page_stride % piece != 0 || head_stride % piece != 0 || row_stride % piece != 0)
        return CUBERT_UNSUPPORTED;
    WriteArgs a;
    a.k = (const char *) k, a.v = (const char *) v, a.k_pages = (char *) k_pages, a.v_pages = (char *) v_pages, a.slots = slots;
    a.page_bytes = page_stride * element, a.head_bytes = head_stride * element, a.row_bytes = row_stride * element;
    a.from_bytes = (long long) ld * element;
    a.tokens = (unsigned) tokens, a.slots_there = (unsigned) pages * (unsigned) page;
    a.shift = __builtin_ctz((unsigned) page);
    a.pieces_of_head = head_size / piece, a.pieces = kv_heads * a.pieces_of_head;
    const unsigned long long blocks = ((unsigned long long) tokens * a.pieces + kBlock - 1) / kBlock;
    if (blocks >= 1u << 24) return CUBERT_UNSUPPORTED;  // (a launch holds less than 2^32 threads)
    if (k_pages == v_pages) return CUBERT_BAD_ARGUMENT;  // (keys and values would be written over each other)
    const bool once = (unsigned long long) tokens * a.pieces * 32 >= 64ull << 20;
    return launch(once ? paged_write_kernel<true> : paged_write_kernel<false>, dim3((unsigned) blocks), dim3(kBlock), (hipStream_t) stream, a);
}

}  // namespace
}  // namespace cubert

extern "C" {

int cubert_paged_extend(int *table, int width, int ld_table, const int *lengths, const int *counts, const int *free, const int *free_count, int places,
                        int pages, int page, int batch, int rows, int *slots, int *lengths_out, int *free_out, void *stream) {
    using namespace cubert;
    if (rows < 0) return CUBERT_BAD_ARGUMENT;
    const int rc = check_tables(table, width, ld_table, lengths, free, free_count, places, pages, page, batch, lengths_out, free_out);
    if (rc != 0) return rc;
    if (batch > 0 && rows > 0 && slots == nullptr) return CUBERT_BAD_ARGUMENT;
    const long long total = (long long) batch * (rows > 0 ? rows : 1);
    if (total > (1ll << 31) - 1 - kSpan) return CUBERT_UNSUPPORTED;
    if (!results_apart({{slots, (long long) batch * rows}, {lengths_out, batch}, {free_out, 1}}, {{lengths, batch}, {counts, batch}, {free, places}, {free_count, 1}}))
        return CUBERT_BAD_ARGUMENT;
    ExtendArgs a;
    a.table = table, a.lengths = lengths, a.counts = counts, a.free = free, a.free_count = free_count;
    a.slots = slots, a.lengths_out = lengths_out, a.free_out = free_out;
    a.width = width, a.ld_table = ld_table, a.places = places, a.pages = pages, a.shift = __builtin_ctz((unsigned) page), a.batch = batch, a.rows = rows;
    const int spans = total > 0 ? (int) ((total + kSpan - 1) / kSpan) : 1;
    a.spans = (spans + kExtendGroups - 1) / kExtendGroups;
    const unsigned blocks = (unsigned) ((spans + a.spans - 1) / a.spans);
    return launch(paged_extend_kernel, dim3(blocks), dim3(kBlock), (hipStream_t) stream, a);
}

size_t cubert_paged_cut_work(int batch, int width) {
    return batch < 1 || width < 1 || cubert::few_to_cut(batch, width) ? 0 : (size_t) batch;
}

int cubert_paged_cut(const int *table, int width, int ld_table, const int *lengths, const int *keep, int *free, const int *free_count, int places,
                     int pages, int page, int batch, int *lengths_out, int *free_out, int *work, void *stream) {
    using namespace cubert;
    const int rc = check_tables(table, width, ld_table, lengths, free, free_count, places, pages, page, batch, lengths_out, free_out);
    if (rc != 0) return rc;
    const bool few = few_to_cut(batch, width);
    if (!few && work == nullptr) return CUBERT_BAD_ARGUMENT;
    // (what is written over keep[b] is keep[b] within its range, which another look at it does not change)
    if (!results_apart({{lengths_out, batch}, {free_out, 1}, {few ? nullptr : work, batch}},
                       {{lengths, batch}, {keep != lengths_out ? keep : nullptr, batch}, {free, places}, {free_count, 1}}))
        return CUBERT_BAD_ARGUMENT;
    CutArgs a;
    a.table = table, a.lengths = lengths, a.keep = keep, a.free = free, a.free_count = free_count;
    a.lengths_out = lengths_out, a.free_out = free_out, a.returned = work;
    a.width = width, a.ld_table = ld_table, a.places = places, a.pages = pages, a.shift = __builtin_ctz((unsigned) page), a.batch = batch;
    if (few) return launch(paged_cut_few_kernel, dim3(1), dim3(kFewWaves * kWave), (hipStream_t) stream, a);
    constexpr int kEach = kBlock / kWave;
    const unsigned blocks = (unsigned) ((batch + kEach - 1) / kEach);
    const int failed = launch(paged_cut_count_kernel, dim3(blocks), dim3(kBlock), (hipStream_t) stream, a);
    if (failed != 0) return failed;
    return launch(paged_cut_kernel, dim3(blocks), dim3(kBlock), (hipStream_t) stream, a);
}

int cubert_paged_write_f32(const float *k, const float *v, int ld, const int *slots, int tokens, float *k_pages, float *v_pages, long long page_stride,
                           long long head_stride, long long row_stride, int pages, int page, int kv_heads, int head_size, void *stream) {
    return cubert::paged_write(k, v, ld, slots, tokens, k_pages, v_pages, page_stride, head_stride, row_stride, pages, page, kv_heads, head_size, 4, stream);
}

int cubert_paged_write_f16(const cubert_half *k, const cubert_half *v, int ld, const int *slots, int tokens, cubert_half *k_pages, cubert_half *v_pages,
                           long long page_stride, long long head_stride, long long row_stride, int pages, int page, int kv_heads, int head_size,
                           void *stream) {
    return cubert::paged_write(k, v, ld, slots, tokens, k_pages, v_pages, page_stride, head_stride, row_stride, pages, page, kv_heads, head_size, 2, stream);
}

}  // extern "C"
