// The paged 8-bit cache: page tables and slot maps of a step's ragged batch, and new keys and values into their pages.
#include <algorithm>

#include "device_math.h"
#include "kernels.h"

namespace sthip {

namespace {

// ---- page tables ----------------------------------------------------------------------------------------------------------------
// Row r of the batch begins at the sum of fresh[] before it, and its new pages at the sum of the pages before it: two prefix sums over
// the requests, and then a division for every row.  Both sums are taken with an addition that stops at 2^31 - 1 (still associative), so
// that no counts can wrap, and rows and free_count are below that: a sum that stopped is never within them.
constexpr unsigned kTablesStop = 0x7fffffffu;
__device__ __forceinline__ unsigned stopping_add(unsigned a, unsigned b) { return min(a + b, kTablesStop); }

struct TablesArgs {
    const int *cached, *fresh, *free_pages, *taken_before;
    int *page_table, *row_offsets, *lengths, *positions, *slots, *counts;
    int requests, page_shift, free_count, rows;
    long long table_width;
};

constexpr int kTablesThreads = 1024;
constexpr int kTablesRequests = 256;  // whose own entries a workgroup writes
constexpr int kTablesRows = 1024;     // of the batch, a workgroup

// Every workgroup takes the sums over all requests up to its own (a few thousand at the most in earnest: each 1024 of them are one
// load and one scan), which saves a second launch; then each row of its own finds its request in LDS.
__global__ __launch_bounds__(kTablesThreads) void page_tables_kernel(TablesArgs p)
{
    __shared__ unsigned wave_rows[16], wave_pages[16];
    __shared__ unsigned row_ends[kTablesThreads], page_starts[kTablesThreads];
    __shared__ int had_pages[kTablesThreads], positions_at[kTablesThreads];  // (of the first row; -1 in had_pages: refused)
    __shared__ int taken, refused;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int own_first = blockIdx.x * kTablesRequests, own_end = min(p.requests, own_first + kTablesRequests);
    const unsigned row_first = static_cast<unsigned>(blockIdx.x) * kTablesRows;
    const unsigned row_last = min(static_cast<unsigned>(p.rows), row_first + kTablesRows);
    const int before = p.taken_before ? max(0, *p.taken_before) : 0;
    const unsigned left = static_cast<unsigned>(max(0, p.free_count - before));
    if (tid == 0) taken = refused = 0;
    if (blockIdx.x == 0 && tid == 0) p.row_offsets[0] = 0;
    unsigned rows_before = 0, pages_before = 0;
    for (int first = 0; first < p.requests; first += kTablesThreads) {
        // Workgroup 0 counts all of them; the others stop behind their own.
        if (blockIdx.x != 0 && first >= own_end && rows_before >= row_last) break;
        const int r = first + tid;
        const bool is = r < p.requests;
        const int cached = is ? p.cached[r] : 0, fresh = is ? p.fresh[r] : 0;
        const long long after = static_cast<long long>(cached) + fresh;
        const long long page_mask = (1ll << p.page_shift) - 1;
        const long long had = (cached + page_mask) >> p.page_shift, used = (after + page_mask) >> p.page_shift;
        const bool possible = cached >= 0 && fresh >= 0 && used <= p.table_width && after <= 0x7fffffff;
        const unsigned my_rows = fresh > 0 ? fresh : 0, need = possible ? static_cast<unsigned>(used - had) : 0;
        unsigned rows_to = my_rows, pages_to = need;
#pragma unroll
        for (int step = 1; step < 64; step <<= 1) {
            const unsigned a = __shfl_up(rows_to, step), b = __shfl_up(pages_to, step);
            if (lane >= step) {
                rows_to = stopping_add(rows_to, a);
                pages_to = stopping_add(pages_to, b);
            }
        }
        if (lane == 63) {
            wave_rows[wave] = rows_to;
            wave_pages[wave] = pages_to;
        }
        __syncthreads();
        unsigned chunk_rows = 0, chunk_pages = 0, rows_in = rows_before, pages_in = pages_before;
#pragma unroll
        for (int w = 0; w < kTablesThreads / 64; ++w) {
            if (w == wave) {
                rows_in = stopping_add(rows_in, chunk_rows);
                pages_in = stopping_add(pages_in, chunk_pages);
            }
            chunk_rows = stopping_add(chunk_rows, wave_rows[w]);
            chunk_pages = stopping_add(chunk_pages, wave_pages[w]);
        }
        rows_to = stopping_add(rows_to, rows_in);
        pages_to = stopping_add(pages_to, pages_in);
        const bool served = possible && rows_to <= static_cast<unsigned>(p.rows) && (need == 0 || pages_to <= left);
        row_ends[tid] = rows_to;
        page_starts[tid] = served ? pages_to - need : 0;
        had_pages[tid] = served ? static_cast<int>(had) : -1;
        positions_at[tid] = cached;
        if (is && r >= own_first && r < own_end) {
            p.lengths[r] = served ? static_cast<int>(after) : 0;
            p.row_offsets[r + 1] = static_cast<int>(min(rows_to, static_cast<unsigned>(p.rows)));
        }
        if (blockIdx.x == 0) {
            if (served && need) atomicMax(&taken, static_cast<int>(pages_to));  // those served are dealt in order
            const unsigned long long no = __ballot(is && !served);
            if (lane == 0 && no) atomicAdd(&refused, __popcll(no));
        }
        __syncthreads();
        // The rows of these requests that are this workgroup's.
        const unsigned ends = stopping_add(rows_before, chunk_rows);
        for (unsigned row = max(row_first, rows_before) + tid; row < min(row_last, ends); row += kTablesThreads) {
            int low = 0, high = kTablesThreads - 1;  // the first whose rows end behind this one
            while (low < high) {
                const int middle = (low + high) >> 1;
                if (row_ends[middle] > row) high = middle;
                else low = middle + 1;
            }
            const unsigned starts = low ? row_ends[low - 1] : rows_before;
            int position = -1, slot = -1;
            if (had_pages[low] >= 0) {
                position = positions_at[low] + static_cast<int>(row - starts);
                const int column = position >> p.page_shift, place = position & static_cast<int>(page_mask);
                int *const entry = p.page_table + (first + low) * p.table_width + column;
                int page;
                if (column >= had_pages[low]) {
                    page = p.free_pages[static_cast<long long>(before) + page_starts[low] + (column - had_pages[low])];
                    if (place == 0) *entry = page;  // the first row of a new page stands at its place 0
                } else {
                    page = *entry;
                }
                const long long wide = (static_cast<long long>(page) << p.page_shift) + place;
                if (page >= 0 && wide <= 0x7fffffff) slot = static_cast<int>(wide);
            }
            p.positions[row] = position;
            p.slots[row] = slot;
        }
        rows_before = ends;
        pages_before = stopping_add(pages_before, chunk_pages);
        __syncthreads();
    }
    // (All requests have been looked at, or this workgroup's rows are all taken.)
    for (unsigned row = max(row_first, rows_before) + tid; row < row_last; row += kTablesThreads) p.positions[row] = p.slots[row] = -1;
    if (blockIdx.x == 0) {
        __syncthreads();  // (no requests: the first barrier behind `taken` and `refused`)
        if (tid == 0) {
            p.counts[0] = before + taken;
            p.counts[1] = static_cast<int>(min(rows_before, static_cast<unsigned>(p.rows)));
            p.counts[2] = refused;
        }
    }
}

// ---- new keys and values --------------------------------------------------------------------------------------------------------
// The smallest power of two s >= 2^-118 with largest <= 448 s: 448 is 1.75 * 2^8, so that the exponent follows from the value's own
// and from whether its significand is above 1.75.
__device__ __forceinline__ float needed_scale(float largest)
{
    const unsigned bits = __float_as_uint(largest);
    const int exponent = static_cast<int>(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    return __uint_as_float(static_cast<unsigned>(max(exponent, -118) + 127) << 23);
}

// Codes of four values over a power of two, none of them above 448 times it; infinities go in as NaN.
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ unsigned e4m3_four(float a, float b, float c, float d, float scale)
{
    s16x2 codes = {0, 0};
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(codes, a, b, scale, false);
    return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(codes, c, d, scale, true));
}
__device__ __forceinline__ unsigned e4m3_four(unsigned low, unsigned high, float scale)  // of bf16 pairs
{
    s16x2 codes = {0, 0};
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(codes, __builtin_bit_cast(bf16x2, low), scale, false);
    return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(codes, __builtin_bit_cast(bf16x2, high), scale, true));
}
__device__ __forceinline__ unsigned rescaled_four(unsigned codes, float ratio)
{
    const auto low = __builtin_amdgcn_cvt_pk_f32_fp8(codes, false), high = __builtin_amdgcn_cvt_pk_f32_fp8(codes, true);
    return e4m3_four(low[0] * ratio, low[1] * ratio, high[0] * ratio, high[1] * ratio, 1.0f);
}

struct AppendArgs {
    const void *k, *v;
    const int *slots;
    uint8_t *cache_k, *cache_v;
    float *k_scales, *v_scales;
    long long ld;
    int rows, pages, page_shift, kv_heads;
    unsigned sharers;
};

constexpr int kAppendMostPage = 256;  // tokens of the largest page
constexpr int kAppendMostRows = 64;   // that a workgroup looks at for the beginnings of pages

// Eight neighbouring values of a row, as they are.
template <typename T>
struct Eight {
    u32x4 raw[sizeof(T) / 2];
    // The sizes' bits, as an unsigned number as large as they are; of bf16 two at a time.
    __device__ __forceinline__ void widen(unsigned &largest) const
    {
#pragma unroll
        for (unsigned i = 0; i < sizeof(T) * 2; ++i) {
            const unsigned bits = raw[i >> 2][i & 3];
            if constexpr (sizeof(T) == 4) {
                largest = max(largest, bits & 0x7fffffffu);
            } else {
                typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
                largest = __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(u16x2, largest), __builtin_bit_cast(u16x2, bits & 0x7fff7fffu)));
            }
        }
    }
    // What e4m3 cannot hold, infinities and NaN, as another value (its bits).
    __device__ __forceinline__ void replace(unsigned with)
    {
        constexpr unsigned all = sizeof(T) == 4 ? 0x7f800000u : 0x7f80u;
#pragma unroll
        for (unsigned i = 0; i < sizeof(T) * 2; ++i) {
            unsigned bits = raw[i >> 2][i & 3];
            if constexpr (sizeof(T) == 4) {
                if ((bits & all) == all) bits = with;
            } else {
                if ((bits & all) == all) bits = (bits & 0xffff0000u) | with;
                if ((bits >> 16 & all) == all) bits = (bits & 0xffffu) | with << 16;
            }
            raw[i >> 2][i & 3] = bits;
        }
    }
    __device__ __forceinline__ unsigned codes(int half, float scale) const
    {
        if constexpr (sizeof(T) == 4) {
            const u32x4 x = raw[half];
            return e4m3_four(__uint_as_float(x[0]), __uint_as_float(x[1]), __uint_as_float(x[2]), __uint_as_float(x[3]), scale);
        } else {
            return e4m3_four(raw[0][2 * half], raw[0][2 * half + 1], scale);
        }
    }
};
template <bool VECTOR, typename T>
__device__ __forceinline__ Eight<T> load_eight(const T *at)
{
    Eight<T> x;
    if constexpr (VECTOR) {
#pragma unroll
        for (unsigned i = 0; i < sizeof(T) / 2; ++i) x.raw[i] = reinterpret_cast<const u32x4 *>(at)[i];
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x.raw[i >> 2][i & 3] = __float_as_uint(at[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) x.raw[0][i] = at[2 * i] | static_cast<unsigned>(at[2 * i + 1]) << 16;
    }
    return x;
}

// A workgroup takes pages that begin (in the order of the rows) within its 64 rows, for one head, and their keys or their values.  Where
// every row begins a page, as in a decode step, several workgroups share the rows' pages.  For every place of a
// page the last row that is for it is noted first; everything behind that goes by place, so that no two threads write the same.
// A thread has eight values of four neighbouring places (of places a quarter of the page apart, for keys), so that both layouts are
// read and written in runs: keys 8 bytes of a place at a time, 128 a row of lanes; values, which lie transposed, 4 bytes of a value at a
// time, 64 in a page of 64.  Blocks of up to 8192 values (a page of 64 places and heads of 128 values) stay in registers between the
// maximum and the rounding, larger ones are read again where threads have more than one such share.  VECTOR: rows on 16-byte boundaries.
// What bounds it is instructions and their latencies as much as memory: sizes are compared as integers, two of bf16 at a time, and values are
// scaled and rounded by the instruction that makes two codes of them.  (8192 rows of bf16, 8 heads of 128 values, in pages of 64: 17.1 us,
// 2.9 TB/s; 22.4 when each value was widened, compared and scaled by itself, 18.2 when a workgroup had both keys and values.)
template <typename T, int HD, bool VECTOR, int THREADS>
__global__ __launch_bounds__(THREADS) void kv_append_kernel(AppendArgs p)
{
    constexpr int RUNS = HD / 8;  // of eight values
    constexpr int WAVES = THREADS / 64;
    static_assert(kAppendMostPage <= THREADS, "a place for each thread");
    __shared__ int owners[kAppendMostPage];
    __shared__ unsigned wave_largest[WAVES];
    __shared__ unsigned long long changes[WAVES], beginnings;
    __shared__ int run_end, pages[kAppendMostRows];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int page_size = 1 << p.page_shift, quarter = page_size >> 2;
    const bool keys = (blockIdx.x & 1) == 0;
    const unsigned head = blockIdx.x / 2 % p.kv_heads, of_head = blockIdx.x / 2 / p.kv_heads;
    const unsigned sharer = of_head & (p.sharers - 1);
    const int block_first = static_cast<int>(of_head / p.sharers) * kAppendMostRows;
    const T *const source = static_cast<const T *>(keys ? p.k : p.v) + static_cast<size_t>(head) * HD;

    auto page_of = [&](int row) {  // -1: skipped
        const int slot = p.slots[row];
        const int page = slot < 0 ? -1 : slot >> p.page_shift;
        return page < p.pages ? page : -1;
    };
    // The THREADS rows from the block's first on, one a thread; where the page is another one than the row's before.
    const int own_row = block_first + tid;
    const int own_page = own_row < p.rows ? page_of(own_row) : -2, own_place = own_row < p.rows ? p.slots[own_row] & (page_size - 1) : 0;
    const bool change = own_row == 0 || (own_row <= p.rows ? page_of(own_row - 1) : -2) != own_page;
    const unsigned long long changed = __ballot(change), begun_here = __ballot(change && own_page >= 0);
    if (lane == 0) {
        changes[wave] = changed;
        if (wave == 0) beginnings = begun_here;
    }
    if (tid < kAppendMostRows) pages[tid] = own_page;
    __syncthreads();
    // Of the pages that begin here, this workgroup's: every sharers-th (a power of two).
    const unsigned long long all_begun = beginnings;
    const unsigned rank = __builtin_amdgcn_mbcnt_hi(static_cast<unsigned>(all_begun >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<unsigned>(all_begun), 0));
    for (unsigned long long pending = __ballot((all_begun >> lane & 1) != 0 && (rank & (p.sharers - 1)) == sharer); pending != 0; pending &= pending - 1) {
        const int which = __builtin_ctzll(pending), page = __builtin_amdgcn_readfirstlane(pages[which]);
        int end = THREADS;  // of the page's rows, among those
        for (int w = WAVES - 1; w >= 0; --w) {
            const unsigned long long later = w == 0 ? changes[0] & (~1ull << which) : changes[w];
            if (later != 0) end = 64 * w + __builtin_ctzll(later);
        }
        const size_t block = static_cast<size_t>(page) * p.kv_heads + head;
        float *const scale_at = (keys ? p.k_scales : p.v_scales) + block;
        const float held = *scale_at;
        if (tid < page_size) owners[tid] = -1;
        if (tid == 0) run_end = p.rows;
        __syncthreads();
        if (tid >= which && tid < end) atomicMax(&owners[own_place], own_row);
        if (end == THREADS) {  // repeated rows alone make a page's so many
            for (int at = block_first + THREADS; at < p.rows; at += THREADS) {
                const int row = at + tid;
                const bool mine = row < p.rows && page_of(row) == page;
                if (!mine && row < p.rows) atomicMin(&run_end, row);
                __syncthreads();
                if (mine && row < run_end) atomicMax(&owners[p.slots[row] & (page_size - 1)], row);
                if (run_end < at + THREADS) break;
            }
        }
        __syncthreads();

        const int items = quarter * RUNS;
        // Item i: its four places, and its eight values.
        auto item_run = [&](int i) { return keys ? i % RUNS : i / quarter; };
        auto item_place = [&](int i, int j) { return keys ? i / RUNS + j * quarter : i % quarter * 4 + j; };
        Eight<T> x[4];
        int rows[4];
        auto load = [&](int i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                rows[j] = owners[item_place(i, j)];
                if (rows[j] >= 0) x[j] = load_eight<VECTOR>(source + static_cast<size_t>(rows[j]) * p.ld + item_run(i) * 8);
            }
        };
        // The largest size, by its bits; where a value is none, which its bits show, once more without those.
        auto measure = [&](bool finite) {
            unsigned sizes = 0;
            for (int i = tid; i < items; i += THREADS) {
                load(i);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (finite) x[j].replace(0);
                    if (rows[j] >= 0) x[j].widen(sizes);
                }
            }
            if constexpr (sizeof(T) == 2) sizes = max(sizes << 16, sizes & 0xffff0000u);
            sizes = wave_scan(sizes, [](unsigned a, unsigned b) { return max(a, b); });
            if (lane == 63) wave_largest[wave] = sizes;
            __syncthreads();
        };
        measure(false);
        auto largest_of_all = [&] {
            unsigned most = 0;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) most = max(most, wave_largest[w]);
            return __builtin_amdgcn_readfirstlane(most);
        };
        unsigned largest = largest_of_all();
        const bool special = largest >= 0x7f800000u;
        if (special) {
            __syncthreads();
            measure(true);
            largest = largest_of_all();
        }

        const bool begun = owners[0] >= 0;
        const float before = begun ? 0.0f : held;
        const float scale = fmaxf(before, needed_scale(__uint_as_float(largest)));
        const bool grown = !begun && scale > before;
        const float ratio = before / scale;
        uint8_t *const codes = (keys ? p.cache_k : p.cache_v) + (block << p.page_shift) * HD;
        for (int i = tid; i < items; i += THREADS) {
            if (items > THREADS || special) load(i);
            if (special) {
#pragma unroll
                for (int j = 0; j < 4; ++j) x[j].replace(sizeof(T) == 4 ? 0x7fc00000u : 0x7fc0u);
            }
            const int d = item_run(i) * 8;
            if (keys) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    uint2 *const to = reinterpret_cast<uint2 *>(codes + item_place(i, j) * HD + d);
                    if (rows[j] >= 0) {
                        *to = uint2{x[j].codes(0, scale), x[j].codes(1, scale)};
                    } else if (grown) {
                        const uint2 old = *to;
                        *to = uint2{rescaled_four(old.x, ratio), rescaled_four(old.y, ratio)};
                    }
                }
                continue;
            }
            const bool any = (rows[0] & rows[1] & rows[2] & rows[3]) >= 0, all = (rows[0] | rows[1] | rows[2] | rows[3]) >= 0;
            if (!any && !grown) continue;
            const unsigned mine = (rows[0] < 0 ? 0 : 0xffu) | (rows[1] < 0 ? 0 : 0xff00u) | (rows[2] < 0 ? 0 : 0xff0000u) | (rows[3] < 0 ? 0 : 0xff000000u);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                unsigned codes_of[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) codes_of[j] = rows[j] >= 0 ? x[j].codes(h, scale) : 0;
                // Bytes e of the four places: a word of value 4h + e.
                const unsigned low_ab = __builtin_amdgcn_perm(codes_of[1], codes_of[0], 0x05010400u), high_ab = __builtin_amdgcn_perm(codes_of[1], codes_of[0], 0x07030602u);
                const unsigned low_cd = __builtin_amdgcn_perm(codes_of[3], codes_of[2], 0x05010400u), high_cd = __builtin_amdgcn_perm(codes_of[3], codes_of[2], 0x07030602u);
                const unsigned words[4] = {__builtin_amdgcn_perm(low_cd, low_ab, 0x05040100u), __builtin_amdgcn_perm(low_cd, low_ab, 0x07060302u),
                                           __builtin_amdgcn_perm(high_cd, high_ab, 0x05040100u), __builtin_amdgcn_perm(high_cd, high_ab, 0x07060302u)};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    unsigned *const to = reinterpret_cast<unsigned *>(codes + (static_cast<size_t>(d + 4 * h + e) << p.page_shift) + item_place(i, 0));
                    unsigned word = words[e];
                    if (!all) {
                        const unsigned old = *to;
                        word = (word & mine) | ((grown ? rescaled_four(old, ratio) : old) & ~mine);
                    }
                    *to = word;
                }
            }
        }
        __syncthreads();  // everyone has read the scale, and the next page takes `owners`
        if (tid == 0) *scale_at = scale;
    }
}

template <typename T, int HD>
hipError_t launch_append(const st_hip_kv_cache &cache, size_t rows, const int32_t *slots, const T *k, const T *v, size_t ld, hipStream_t stream)
{
    AppendArgs args{k, v, slots, cache.k, cache.v, cache.k_scales, cache.v_scales, static_cast<long long>(ld), static_cast<int>(rows),
                    static_cast<int>(cache.pages), __builtin_ctzll(cache.page_size), static_cast<int>(cache.kv_heads), 1};
    // A thread has 32 values at once; where a page has more than 256 threads do, it takes 512.  (us for 49 times 8 rows in pages of 256, 4 heads of
    // 128 values: 28.4, 15.8 with 512 and 13.7 with 1024; 88 times 3 rows, 10 heads of 64 values: 25.0, 21.3 and 64.)
    const bool large = cache.page_size * HD > 256 * 32;
    const size_t blocks = (rows + kAppendMostRows - 1) / kAppendMostRows * cache.kv_heads * 2;
    // Up to 2048 workgroups of four wavefronts, which the chip holds at once, share the rows' pages (us for 77 single rows of 5 heads at 1024, 2048 and
    // 4096: 7.7, 5.6, 5.6; for 8192 rows of 16 prompts, whose 64 rows begin a page or two: 17.1, 17.1, 19.5).
    args.sharers = 1;
    while (args.sharers < kAppendMostRows && args.sharers < rows && blocks * args.sharers * 2 <= (large ? 1024u : 2048u)) args.sharers *= 2;
    const size_t grid = blocks * args.sharers;
    if (grid > 0x7fffffffu) return hipErrorInvalidValue;
    const bool aligned = ld * sizeof(T) % 16 == 0 && reinterpret_cast<uintptr_t>(k) % 16 == 0 && reinterpret_cast<uintptr_t>(v) % 16 == 0;
    const dim3 blocks_of(static_cast<unsigned>(grid));
    if (large && aligned) kv_append_kernel<T, HD, true, 512><<<blocks_of, 512, 0, stream>>>(args);
    else if (large) kv_append_kernel<T, HD, false, 512><<<blocks_of, 512, 0, stream>>>(args);
    else if (aligned) kv_append_kernel<T, HD, true, 256><<<blocks_of, 256, 0, stream>>>(args);
    else kv_append_kernel<T, HD, false, 256><<<blocks_of, 256, 0, stream>>>(args);
    return hipGetLastError();
}

template <typename T>
hipError_t launch_append_any(const st_hip_kv_cache &cache, size_t rows, const int32_t *slots, const T *k, const T *v, size_t ld, hipStream_t stream)
{
    if (cache.head_dim == 64) return launch_append<T, 64>(cache, rows, slots, k, v, ld, stream);
    if (cache.head_dim == 128) return launch_append<T, 128>(cache, rows, slots, k, v, ld, stream);
    return launch_append<T, 256>(cache, rows, slots, k, v, ld, stream);
}

}  // namespace

hipError_t launch_page_tables(size_t requests, size_t page_size, const int32_t *cached, const int32_t *fresh, size_t free_count,
                              const int32_t *free_pages, const int32_t *taken_before, size_t table_width, int32_t *page_table, size_t rows,
                              int32_t *row_offsets, int32_t *lengths, int32_t *positions, int32_t *slots, int32_t *counts, hipStream_t stream)
{
    const TablesArgs args{cached, fresh, free_pages, taken_before, page_table, row_offsets, lengths, positions, slots, counts,
                          static_cast<int>(requests), __builtin_ctzll(page_size), static_cast<int>(free_count), static_cast<int>(rows),
                          static_cast<long long>(table_width)};
    const size_t by_requests = (requests + kTablesRequests - 1) / kTablesRequests, by_rows = (rows + kTablesRows - 1) / kTablesRows;
    const size_t blocks = std::max<size_t>(1, std::max(by_requests, by_rows));
    page_tables_kernel<<<static_cast<unsigned>(blocks), kTablesThreads, 0, stream>>>(args);
    return hipGetLastError();
}

hipError_t launch_kv_cache_append_f32(const st_hip_kv_cache &cache, size_t rows, const int32_t *slots, const float *k, const float *v, size_t ld, hipStream_t stream)
{
    return launch_append_any(cache, rows, slots, k, v, ld, stream);
}

hipError_t launch_kv_cache_append_bf16(const st_hip_kv_cache &cache, size_t rows, const int32_t *slots, const uint16_t *k, const uint16_t *v, size_t ld, hipStream_t stream)
{
    return launch_append_any(cache, rows, slots, k, v, ld, stream);
}

}  // namespace sthip
