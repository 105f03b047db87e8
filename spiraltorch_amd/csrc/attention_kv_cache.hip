// Attention over a paged cache of e4m3 keys and values with a power of two for every page and head: single tokens, chunks of prompts, and
// an encoder's states, of many requests at once.
//
// The kernel computes the transposed problem, S^T = K Q^T and O^T += V^T P^T, on v_mfma_f32_16x16x32_bf16: a lane owns one column, a
// (token, head) pair, so that the running maximum and sum are its own scalars.  An e4m3 value times a power of two is a bf16 value: codes are
// widened and scaled in registers by one instruction for two of them (v_cvt_scalef32_pk_bf16_fp8), without loss.
// Both operands come from memory in the layout that the matrix cores take, with 16-byte loads and without LDS.  Within a tile of 64
// keys, lane group g (of 16 lanes) owns keys 16g .. 16g+15: row m of the score tile s is key (m/4)*16 + 4s + m%4, which hands lane
// group g of the accumulators keys 16g + 4s + (0..3).  The four tiles together are then a run of 16 keys, in the order in which the
// second product takes them: V^T, which the cache holds as (head_dim, tokens), gives a lane the same 16 keys of one value with one load.
// Every 16-key group lies within a page whatever its size, so that a tile may span up to four pages.
#include <algorithm>
#include <cmath>
#include <limits>
#include <type_traits>

#include "device_math.h"
#include "kernels.h"

namespace sthip {

namespace {

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));

struct KvAttentionArgs {
    const uint8_t *k, *v;
    const float *k_scales, *v_scales;
    const int *row_offsets, *lengths, *page_table;
    const uint16_t *q;
    uint16_t *out;
    float *parts;       // where keys are cut over workgroups: for each part, up to `room` for a key head, 16 columns of head_dim sums, and then 16
                        // maxima and sums
    float *wide_parts;  // the same for each workgroup of wide tiles
    unsigned *arrived;  // and for every tile of columns, as many narrow ones as there is room for parts and the wide ones, how many of its workgroups
                        // are done: 0 before a launch and after it
    long long ld_q, ld_out, table_width;
    int requests, rows, kv_heads, group, pages, page_shift;
    int few;         // requests of so many columns or fewer go to the kernel whose wavefronts share them, others to the one of wide tiles
    unsigned units;  // workgroups of the former
    unsigned wide;   // and of the latter
    unsigned room;        // see kKvRoom
    unsigned wide_items;  // the most that there can be of (wide tile of columns, key head) pairs: a counter for each
    float heads_by_target;
    bool halves_own;  // whether a share of wide tiles counts half of a request's own rows
    float scale_log2;  // |scale| * log2(e), not quite 0
    bool causal, negative;
};

constexpr int kKvTile = 64;     // keys
constexpr int kKvColumns = 16;  // (token, head) pairs of a tile
constexpr int kKvMostParts = 128, kKvMostWideParts = 16;
constexpr int kKvLeastShare = 4;  // tiles that a workgroup takes at the least: one for each of its wavefronts

__device__ __forceinline__ int clamped(int x, int low, int high) { return min(max(x, low), high); }

struct KvRequest {
    int first_row, rows, length, id;
};

__device__ __forceinline__ KvRequest load_request(const KvAttentionArgs &p, int r)
{
    KvRequest q;
    q.id = r;
    q.first_row = clamped(p.row_offsets[r], 0, p.rows);
    q.rows = max(0, clamped(p.row_offsets[r + 1], 0, p.rows) - q.first_row);
    q.length = static_cast<int>(min(static_cast<long long>(max(0, p.lengths[r])), p.table_width << p.page_shift));
    return q;
}

__device__ __forceinline__ unsigned key_tiles(int keys) { return (static_cast<unsigned>(keys) + kKvTile - 1) / kKvTile; }
__device__ __forceinline__ unsigned few_tiles(const KvAttentionArgs &p, const KvRequest &q)
{
    const int columns = q.rows * p.group;
    return columns <= p.few ? (static_cast<unsigned>(columns) + kKvColumns - 1) / kKvColumns : 0;
}
// A context in parts of `share` tiles, or more where they would be too many to put together; whole, if it is not much longer, or short and
// not longer than two: putting parts together takes 3 us, and its last part would leave a workgroup with little to do.  (16 contexts of 300 to
// 1000 keys with 64 columns each took 26 us when cut at every share, and 19 so; 12 heads' 16 contexts of 1500 keys, 24 tiles at a share
// of 12, 14.4 and 12.0; decoding 64 contexts of up to 8192 41.2 and 40.2, and 43.5 with contexts of up to two shares whole.)
__device__ __forceinline__ unsigned share_of_tiles(unsigned tiles, unsigned share, unsigned most)
{
    const unsigned mine = max(share, ((tiles + most - 1) / most + 3u) & ~3u);
    return tiles <= max(mine + mine / 2, min(2 * mine, 24u)) ? max(tiles, 1u) : mine;
}
__device__ __forceinline__ unsigned share_of(const KvRequest &q, unsigned share, unsigned most = kKvMostParts) { return share_of_tiles(key_tiles(q.length), share, most); }
__device__ __forceinline__ unsigned parts_of(const KvRequest &q, unsigned share, unsigned most = kKvMostParts)
{
    const unsigned mine = share_of(q, share, most);
    return max(1u, (key_tiles(q.length) + mine - 1) / mine);
}

// Calls `with` for this lane's requests, `step` of them from low + lane * step on and below end, whose loads are two or eight at a time: a plan
// of many requests is a chain of them.
template <int AHEAD, class With>
__device__ __forceinline__ void for_requests_by(const KvAttentionArgs &p, int first, int end, With &&with)
{
    for (int r = first; r < end; r += AHEAD) {
        KvRequest q[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) q[i] = load_request(p, min(r + i, end - 1));
#pragma unroll
        for (int i = 0; i < AHEAD; ++i)
            if (r + i < end) with(q[i]);
    }
}
template <class With>
__device__ __forceinline__ void for_requests(const KvAttentionArgs &p, int low, int end, int step, With &&with)
{
    const int first = low + (threadIdx.x & 63) * step;
    if (step <= 2) for_requests_by<2>(p, first, min(end, first + step), with);
    else for_requests_by<8>(p, first, min(end, first + step), with);
}

// Sums stop at 2^32 - 1 (and stay associative): those of any row offsets can be compared with what there is room for.
__device__ __forceinline__ unsigned stopping_sum(unsigned x, unsigned y) { return __builtin_elementwise_add_sat(x, y); }
// Sum over the lanes up to and with this one.
__device__ __forceinline__ unsigned wave_scan_sum(unsigned v)
{
    return wave_scan(v, stopping_sum);
}

// Work is numbered by prefix sums over the requests, which a wavefront of every workgroup takes: `count(request)` items each, and the
// request of item number `item` is found by 64 sums at a time (one round of loads for up to 64 requests, two for 4096 ...).  `own`: this lane's
// request where there are no more than 64.
constexpr unsigned kKvWhole = 0x7fffffffu;  // as a share: no context is cut
struct KvFound {
    KvRequest of;
    unsigned offset;  // of the item within its request's
    unsigned before;  // sum of `other` over the requests before it
};
// False behind the last item; and for all items where they, or `other`, are more than there is room for, which row offsets out of order can make
// them: a launch does all the work of one kind or none of it, and its counters are within their buffer and 0 after it.  `known`, if it is: the sum
// of `count` over this lane's requests of the first level, where `before` will not be looked at.
template <class Count, class Other>
__device__ __forceinline__ bool find_request(const KvAttentionArgs &p, const KvRequest &own, unsigned item, unsigned most, unsigned most_other, Count &&count, Other &&other, KvFound *found,
                                             bool is_known, unsigned known)
{
    int low = 0, left = p.requests;
    unsigned items_before = 0;
    found->before = 0;
    for (;;) {
        const int step = (left + 63) / 64;
        unsigned items = 0, others = 0;
        KvRequest q = own;
        if (p.requests <= 64) {
            items = count(q);
            others = other(q);
        } else if (is_known && left == p.requests) {
            items = known;
        } else {
            for_requests(p, low, low + left, step, [&](const KvRequest &of) {
                q = of;
                items = stopping_sum(items, count(of));
                others = stopping_sum(others, other(of));
            });
        }
        const unsigned to = wave_scan_sum(items), to_other = wave_scan_sum(others);
        const unsigned long long behind = __ballot(items_before + to > item);
        if (behind == 0) return false;
        if (left == p.requests && (__builtin_amdgcn_readlane(to, 63) > most || __builtin_amdgcn_readlane(to_other, 63) > most_other)) return false;
        const int which = __builtin_ctzll(behind);
        items_before += __builtin_amdgcn_readlane(to - items, which);
        found->before += __builtin_amdgcn_readlane(to_other - others, which);
        low += which * step;
        left = min(step, left - which * step);
        if (step > 1) continue;
        found->offset = item - items_before;
        found->of.first_row = __builtin_amdgcn_readlane(q.first_row, which);
        found->of.rows = __builtin_amdgcn_readlane(q.rows, which);
        found->of.length = __builtin_amdgcn_readlane(q.length, which);
        found->of.id = __builtin_amdgcn_readlane(q.id, which);
        return true;
    }
}

// This lane's request where there are no more than 64 (none: no rows).
__device__ __forceinline__ KvRequest own_request(const KvAttentionArgs &p)
{
    const int lane = threadIdx.x & 63;
    KvRequest q{0, 0, 0, 0};
    if (p.requests <= 64 && lane < p.requests) q = load_request(p, lane);
    return q;
}

// What one wavefront found for all of a workgroup's.
__device__ __forceinline__ KvFound uniform(const KvFound &f)
{
    auto one = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
    return KvFound{{one(f.of.first_row), one(f.of.rows), one(f.of.length), one(f.of.id)}, static_cast<unsigned>(one(f.offset)), static_cast<unsigned>(one(f.before))};
}

// The same with the longest first, so that the longest work begins first: sorted, or by eight classes half an octave wide and the rest.
// (Sorting took 2.8 us for 64 requests, for 16 it takes 0.6 us.  What is done in a few microseconds goes without, and work that takes
// long has requests in the order of their lengths.)
template <bool SORT>
__device__ __forceinline__ KvRequest longest_first(const KvAttentionArgs &p, const KvRequest &own)
{
    if (p.requests > 64) return own;
    const int lane = threadIdx.x & 63;
    int rank = 0;
    if (SORT && p.requests <= 16) {
        for (int i = 0; i < p.requests; ++i) {
            const int other = __builtin_amdgcn_readlane(own.length, i);
            rank += other > own.length || (other == own.length && i < lane);
        }
        if (lane >= p.requests) rank = lane;
    } else {
        const unsigned width = own.rows == 0 ? 0 : __float_as_uint(static_cast<float>(own.length)) >> 22;  // exponent and a bit more
        const unsigned widest = __builtin_amdgcn_readlane(wave_scan(width, [](unsigned x, unsigned y) { return max(x, y); }), 63);
        const int of_class = static_cast<int>(min(widest - width, 8u));
        if (__all(of_class == 0 || own.rows == 0)) return own;
        int before = 0;
#pragma unroll
        for (int i = 0; i <= 8; ++i) {
            const unsigned long long in = __ballot(of_class == i);
            const int among = __builtin_amdgcn_mbcnt_hi(static_cast<unsigned>(in >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<unsigned>(in), 0));
            if (of_class == i) rank = before + among;
            before += __popcll(in);
        }
    }
    auto moved = [&](int x) { return __builtin_amdgcn_ds_permute(4 * rank, x); };
    return KvRequest{moved(own.first_row), moved(own.rows), moved(own.length), moved(own.id)};
}

// Workgroups that all contexts are cut over, beside one for each tile of columns: as many as the chip holds at once of the kernel's registers
// for 128 and 256 values.  (64 contexts of 16 to 8192 keys and eight heads took 45, 41, 41 and 46 us with 256, 384, 512 and 768 of them at
// dimension 128, 24, 22 and 22 with 256, 512 and 1024 at 64; at 256, two heads, 30, 34 and 43.)
template <int HD>
constexpr int kKvTarget = HD == 256 ? 256 : 512;

// The 64-key tiles that a workgroup takes of a context at the most: all the tiles that there are, `work(request)` for one, over the
// workgroups that there should be.  Contexts of very different lengths fill the chip evenly so, whatever the host knows of them (it
// knows the table's width alone).  `work` is 0 where `tiles(request)`, the tiles of columns, are.  The one look at more than 64 requests also says
// whether even the longest is not cut (kKvWhole), and how many items there are at the most, where cuts add up to `more`: 1024 requests with a
// token each, none cut, 267 us, 318 when all were counted once more; a prompt of 500 rows beside 511 that wait 80 and 92.
struct KvShare {
    unsigned share, tiles, most_items;  // tiles: this lane's, of columns
};
template <class Tiles, class Work>
__device__ __forceinline__ KvShare find_share(const KvAttentionArgs &p, const KvRequest &own, unsigned most_parts, unsigned more, Tiles &&tiles, Work &&work)
{
    float all = 0.0f;  // (rounded, but alike in every workgroup, and what it may fall short of the sum by is added below)
    unsigned longest = 0, mine = 0;
    if (p.requests <= 64) {
        all = work(own);
    } else {
        for_requests(p, 0, p.requests, (p.requests + 63) / 64, [&](const KvRequest &q) {
            const unsigned columns = tiles(q);
            mine = stopping_sum(mine, columns);
            all += work(q);
            if (columns != 0) longest = max(longest, key_tiles(q.length));
        });
    }
    const float even = wave_sum(all) * p.heads_by_target * 1.001f + 1.0f;
    const unsigned whole = (static_cast<unsigned>(fminf(even, 1073741824.0f)) + 3u) & ~3u;  // (the same for each of four wavefronts)
    const unsigned share = __builtin_amdgcn_readfirstlane(max(static_cast<unsigned>(kKvLeastShare), whole));
    if (p.requests <= 64) return KvShare{share, 0, ~0u};
    longest = __builtin_amdgcn_readlane(wave_scan(longest, [](unsigned x, unsigned y) { return max(x, y); }), 63);
    const unsigned most_items = stopping_sum(__builtin_amdgcn_readlane(wave_scan_sum(mine), 63), more);
    return KvShare{share_of_tiles(longest, share, most_parts) >= longest ? kKvWhole : share, mine, most_items};
}

// Eight e4m3 values times a power of two, as bf16: both are exact.
__device__ __forceinline__ bf16x8 widened(unsigned low, unsigned high, float scale)
{
    u32x4 r;
    r[0] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(low, scale, false));
    r[1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(low, scale, true));
    r[2] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(high, scale, false));
    r[3] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(high, scale, true));
    return __builtin_bit_cast(bf16x8, r);
}

// 1 in the bytes of `codes` that hold NaN, else 0.
__device__ __forceinline__ unsigned nan_bytes(unsigned codes) { return (((codes & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7; }

// NaN becomes 0; not 0 where there was one.
__device__ __forceinline__ unsigned drop_nan(u32x4 &codes)
{
    asm volatile("");  // (a branch where this is called in one)
    unsigned any = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const unsigned is = nan_bytes(codes[i]);
        any |= is;
        codes[i] &= ~((is << 8) - is);
    }
    return any;
}

__device__ __forceinline__ float across_groups_max(float v)  // over the four lane groups, same column
{
    const auto halves = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(halves[0]), __uint_as_float(halves[1]));
    const auto rows = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(rows[0]), __uint_as_float(rows[1]));
}
__device__ __forceinline__ float across_groups_sum(float v)
{
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}

// A wavefront's columns: NC tiles of sixteen, tile c at `first + 16c`, of the request's rows*group; behind the last one they repeat it.
// Sums of weighted values are divided by the weights' only at the end, and weights may be 2^8 (see weigh): for 2^31 keys on pages of scale 2^70 or
// less they stay below 2^31 * 2^8 * 448 * 2^70, 2^118.  From the first page above that on, weights are 2^-64 of what they were, so that the largest
// values that there are, averaged over as many keys as there can be, keep as far from f32's border.
constexpr float kKvLargeScale = 0x1p70f, kKvLowered = 64.0f;

template <int HD, int NC>
struct KvColumnsState {
    f32x4 out[NC][HD / 16];
    f32x4 sum[NC];      // of the weights, as they go into `out`: a product with ones, four times the same
    float run_max[NC];  // in log2, of scaled scores, and `lowered` more
    float lowered;      // weights are smaller by that power of two: 0, or kKvLowered once values have been met that are as large as kKvLargeScale
    int limit[NC];                   // keys that the column sees
    int keys, fewest;                // the most and the fewest that any of them does
};

template <int HD, int NC>
__device__ __forceinline__ void begin_columns(const KvAttentionArgs &p, const KvRequest &of, int first, KvColumnsState<HD, NC> &s)
{
    const int n = threadIdx.x & 15, columns = of.rows * p.group;
    auto sees = [&](int column) { return p.causal ? max(0, of.length - of.rows + column / p.group + 1) : of.length; };
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        s.run_max[c] = -INFINITY;
        s.lowered = 0.0f;
        s.sum[c] = f32x4{0.f, 0.f, 0.f, 0.f};
        s.limit[c] = sees(min(columns - 1, first + 16 * c + n));
#pragma unroll
        for (int t = 0; t < HD / 16; ++t) s.out[c][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    s.fewest = sees(first);
    s.keys = sees(min(columns, first + 16 * NC) - 1);
}

// Q^T of a wavefront's columns: value 64j + 16g + 8h + (0..7) of the column, for step (j, h) of the first product; keys are loaded alike.  A
// negative scale goes into its signs, so that the largest score is that of the largest product.
template <int HD, int NC>
__device__ __forceinline__ void load_queries(const KvAttentionArgs &p, const KvRequest &of, int kv_head, int first, bf16x8 (&query)[NC][HD / 32])
{
    const int n = threadIdx.x & 15, g = (threadIdx.x & 63) >> 4, columns = of.rows * p.group;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const int column = min(columns - 1, first + 16 * c + n);
        const uint16_t *const q = p.q + (static_cast<size_t>(of.first_row) + column / p.group) * p.ld_q +
                                  static_cast<size_t>(kv_head * p.group + column % p.group) * HD;
#pragma unroll
        for (int j = 0; j < HD / 32; ++j) {
            u32x4 raw = *reinterpret_cast<const u32x4 *>(q + 64 * (j / 2) + 16 * g + 8 * (j % 2));
            if (p.negative) raw ^= 0x80008000u;
            query[c][j] = __builtin_bit_cast(bf16x8, raw);
        }
    }
}

// -infinity for the scores of keys that a column does not see; `fits`: whether this lane's 16 keys are on a page of the cache.
template <int HD, int NC>
__device__ __forceinline__ void hide_unseen(const KvColumnsState<HD, NC> &s, unsigned key0, bool fits, f32x4 (&scores)[NC][4])
{
    asm volatile("");  // (a branch, not selects in every tile)
    const int group = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const int seen = fits ? s.limit[c] - static_cast<int>(key0) - 16 * group : 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            if (i >= seen) scores[c][i >> 2][i & 3] = -INFINITY;
            if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);  // (comparisons one by one take no scalar registers)
        }
    }
}

// Before a tile's values count, if one of them is on a page of a scale above kKvLargeScale.
template <int HD, int NC>
__device__ __forceinline__ void lower_for(float value_scale, KvColumnsState<HD, NC> &s)
{
    if (__builtin_expect(!__any(value_scale > kKvLargeScale), 1) || s.lowered != 0.0f) return;
    s.lowered = kKvLowered;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        s.run_max[c] += kKvLowered;
        s.sum[c] *= 0x1p-64f;
#pragma unroll
        for (int t = 0; t < HD / 16; ++t) s.out[c][t] *= 0x1p-64f;
    }
}

// A tile's scores (products of queries and keys; -infinity where a column does not see the key) to the weights of its values, and the
// columns' maxima, sums and outputs with them.
template <int HD, int NC, int PIECES>
__device__ __forceinline__ void weigh(const KvAttentionArgs &p, f32x4 (&scores)[NC][4], KvColumnsState<HD, NC> &s, bf16x8 (&weights)[PIECES][NC][2])
{
    float most[NC];
    bool grows = false;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        most[c] = -INFINITY;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            most[c] = fmaxf(fmaxf(most[c], scores[c][i][0]), scores[c][i][1]);
            most[c] = fmaxf(fmaxf(most[c], scores[c][i][2]), scores[c][i][3]);
        }
        most[c] = fmaf(across_groups_max(most[c]), p.scale_log2, s.lowered);
        grows |= most[c] > s.run_max[c] + 8.0f;
    }
    // The maximum may lag behind by a factor of 2^8: weights are that much larger then, and nothing has to be scaled for most tiles.
    if (__builtin_expect(__any(grows), 0)) {
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const float up = fmaxf(s.run_max[c], most[c]), shrink = up == s.run_max[c] ? 1.0f : __builtin_amdgcn_exp2f(s.run_max[c] - up);
            s.run_max[c] = up;
            s.sum[c] *= shrink;
#pragma unroll
            for (int t = 0; t < HD / 16; ++t) s.out[c][t] *= shrink;
        }
    }
    // Weights go into the second product, which is that of bf16, as two pieces of it (the second is what the first's rounding leaves: 2^-16 of a
    // weight is lost) or as one, and are summed as they go in: what their rounding adds to the values' sum, it adds to the weights' as well.  With
    // two the result's error is that of its own rounding to bf16, 0.00166 of its size (root mean square), with one 0.0017 to 0.0019.  The second
    // piece costs half of a tile's products again and 40 other instructions.  Narrow tiles wait for memory most of the time and have it
    // (decode_64x8192 41.0 us with one piece and 42.0 with two, decode_1x4097 10.8 and 11.0, cross_16x1500 12.1 and 12.9, 16 contexts of 2000 keys
    // with 16 rows of 64 values 21.2 and 23.2); wide ones are bound by the issue of just these (prefill_8x500 148 and 189, the same at 64 values 117
    // and 166) and have one.
    const u32x4 ones = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const float base = s.run_max[c] == -INFINITY ? 0.0f : s.run_max[c];  // (a column that has seen nothing: its weights are 2^-inf)
        u32x4 packed[PIECES][2];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = __builtin_amdgcn_exp2f(fmaf(scores[c][i][e], p.scale_log2, -base));
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const unsigned pair = pack_bf16x2_rne(w[2 * half], w[2 * half + 1]);
                packed[0][i >> 1][2 * (i & 1) + half] = pair;
                if constexpr (PIECES == 2)
                    packed[1][i >> 1][2 * (i & 1) + half] = pack_bf16x2_rne(w[2 * half] - __uint_as_float(pair << 16), w[2 * half + 1] - __uint_as_float(pair & 0xffff0000u));
            }
        }
#pragma unroll
        for (int piece = 0; piece < PIECES; ++piece)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                weights[piece][c][h] = __builtin_bit_cast(bf16x8, packed[piece][h]);
                s.sum[c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, ones), weights[piece][c][h], s.sum[c], 0, 0, 0);
            }
    }
}

// Values that a column does not see may be anything, above all those behind the last key or on a page outside the cache, and 0 * NaN is not
// 0.  In a tile that not every column sees whole, NaN among the values goes into the product as 0, and this makes up for it, in tiles
// `tile`, tile + step, ... below `end`: every sum that met one is NaN.  The same product, of 1 where a value is NaN and 1 where it is seen, says
// which.
template <int HD, int NC>
__device__ __forceinline__ void mark_nan(const KvAttentionArgs &p, const KvRequest &of, int kv_head, unsigned tile, unsigned end, unsigned step, KvColumnsState<HD, NC> &s)
{
    const int n = threadIdx.x & 15, g = (threadIdx.x & 63) >> 4, page_mask = (1 << p.page_shift) - 1;
    for (; tile < end; tile += step) {
        const unsigned key = tile * kKvTile + 16 * g;
        int page = key < static_cast<unsigned>(of.length) ? p.page_table[of.id * p.table_width + (key >> p.page_shift)] : -1;
        const bool fits = page >= 0 && page < p.pages;
        if (!fits) page = 0;
        const uint8_t *const v = p.v + (((static_cast<size_t>(page) * p.kv_heads + kv_head) * HD + n) << p.page_shift) + (key & page_mask);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int seen = fits ? s.limit[c] - static_cast<int>(key) : 0;
            u32x4 sees[2];
#pragma unroll
            for (int i = 0; i < 8; ++i) sees[i >> 2][i & 3] = (2 * i < seen ? 0x3f80u : 0u) | (2 * i + 1 < seen ? 0x3f800000u : 0u);
#pragma unroll
            for (int t = 0; t < HD / 16; ++t) {
                u32x4 is = *reinterpret_cast<const u32x4 *>(v + (static_cast<size_t>(16 * t) << p.page_shift));
#pragma unroll
                for (int i = 0; i < 4; ++i) is[i] = nan_bytes(is[i]) * 0x38u;  // 1.0
                f32x4 met = {0.f, 0.f, 0.f, 0.f};
                met = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widened(is[0], is[1], 1.0f), __builtin_bit_cast(bf16x8, sees[0]), met, 0, 0, 0);
                met = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widened(is[2], is[3], 1.0f), __builtin_bit_cast(bf16x8, sees[1]), met, 0, 0, 0);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (met[i] > 0.0f) s.out[c][t][i] = NAN;
            }
        }
    }
}

// Tiles `tile`, tile + step, ... below `end` of the request's keys for a wavefront's columns.
template <int HD, int NC>
__device__ __forceinline__ void attend(const KvAttentionArgs &p, const KvRequest &of, int kv_head, int first, unsigned tile_first,
                                       unsigned end, unsigned step, KvColumnsState<HD, NC> &s)
{
    constexpr int KL = HD / 64;  // 16-byte loads of a key's row, per lane
    constexpr int VT = HD / 16;  // tiles of O^T
    if (tile_first >= end) return;
    const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4, columns = of.rows * p.group;

    bf16x8 query[NC][2 * KL];
    load_queries<HD, NC>(p, of, kv_head, first, query);

    const int *const table = p.page_table + of.id * p.table_width;
    const int page_mask = (1 << p.page_shift) - 1;
    // The pages of the 16 keys that this lane loads (a row of the first product: group n/4), and of those whose scores it holds.
    const int key_group = 16 * (n >> 2), value_group = 16 * g;
    auto page_at = [&](unsigned key) { return key < static_cast<unsigned>(of.length) ? table[key >> p.page_shift] : -1; };
    auto fits = [&](int page) { return page >= 0 && page < p.pages; };
    auto block_of = [&](int page) { return static_cast<size_t>(fits(page) ? page : 0) * p.kv_heads + kv_head; };
    u32x4 key_codes[4][KL], value_codes[VT];
    float key_scale, value_scale;
    bool value_fits;
    auto load_keys = [&](unsigned key0, int key_page) {
        const size_t block = block_of(key_page);
        const uint8_t *const k = p.k + ((block << p.page_shift) + ((key0 + key_group) & page_mask) + (n & 3)) * HD + 16 * g;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < KL; ++j) key_codes[i][j] = *reinterpret_cast<const u32x4 *>(k + 4 * i * HD + 64 * j);
        key_scale = p.k_scales[block];
    };
    auto values_at = [&](unsigned key0, int value_page) { return p.v + ((block_of(value_page) * HD + n) << p.page_shift) + ((key0 + value_group) & page_mask); };
    auto load_values = [&](unsigned key0, int value_page) {
        const uint8_t *const v = values_at(key0, value_page);
#pragma unroll
        for (int t = 0; t < VT; ++t) value_codes[t] = *reinterpret_cast<const u32x4 *>(v + (static_cast<size_t>(16 * t) << p.page_shift));
        value_fits = fits(value_page);
        value_scale = value_fits ? p.v_scales[block_of(value_page)] : 1.0f;  // (a scale that nobody set can turn the zeros below into NaN)
    };
    // Pages are looked up two tiles ahead; keys are loaded when the scores before are done with their registers, values likewise.
    unsigned tile = tile_first;
    int key_page = page_at(tile * kKvTile + key_group), value_page = page_at(tile * kKvTile + value_group);
    load_keys(tile * kKvTile, key_page);
    load_values(tile * kKvTile, value_page);
    key_page = page_at((tile + step) * kKvTile + key_group);
    value_page = page_at((tile + step) * kKvTile + value_group);
    unsigned masked_first = end;
    for (; tile < end; tile += step) {
        const unsigned key0 = tile * kKvTile, next = key0 + step * kKvTile;
        const bool more = tile + step < end;
        // Whether every column sees all of the tile's keys, and none of them is on a page outside the cache.
        const bool whole = __all(value_fits) && key0 + kKvTile <= static_cast<unsigned>(s.fewest);
        f32x4 scores[NC][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int c = 0; c < NC; ++c) scores[c][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < 2 * KL; ++j) {
                const bf16x8 key = widened(key_codes[i][j / 2][j % 2 * 2], key_codes[i][j / 2][j % 2 * 2 + 1], key_scale);
#pragma unroll
                for (int c = 0; c < NC; ++c) scores[c][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(key, query[c][j], scores[c][i], 0, 0, 0);
            }
        }
        __builtin_amdgcn_sched_barrier(0);  // (what is widened too early takes registers)
        if (more) load_keys(next, key_page);

        if (!whole) hide_unseen<HD, NC>(s, key0, value_fits, scores);
        lower_for<HD, NC>(value_scale, s);
        bf16x8 weights[2][NC][2];
        weigh<HD, NC, 2>(p, scores, s, weights);
        if (!whole) {
            unsigned is = 0;  // (see mark_nan)
#pragma unroll
            for (int t = 0; t < VT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) is |= nan_bytes(value_codes[t][i]);
            if (__any(is != 0)) {
#pragma unroll
                for (int t = 0; t < VT; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) value_codes[t][i] &= ~(nan_bytes(value_codes[t][i]) * 0xffu);
                masked_first = min(masked_first, tile);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int t = 0; t < VT; ++t) {
            const bf16x8 low = widened(value_codes[t][0], value_codes[t][1], value_scale), high = widened(value_codes[t][2], value_codes[t][3], value_scale);
#pragma unroll
            for (int piece = 0; piece < 2; ++piece) {
#pragma unroll
                for (int c = 0; c < NC; ++c) s.out[c][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(low, weights[piece][c][0], s.out[c][t], 0, 0, 0);
#pragma unroll
                for (int c = 0; c < NC; ++c) s.out[c][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(high, weights[piece][c][1], s.out[c][t], 0, 0, 0);
            }
        }
        if (more) {
            load_values(next, value_page);
            key_page = page_at(next + step * kKvTile + key_group);
            value_page = page_at(next + step * kKvTile + value_group);
        }
    }
    mark_nan<HD, NC>(p, of, kv_head, masked_first, end, step, s);
}

__device__ __forceinline__ uint16_t *out_at(const KvAttentionArgs &p, const KvRequest &of, int kv_head, int column, int head_dim)
{
    return p.out + (static_cast<size_t>(of.first_row) + column / p.group) * p.ld_out + static_cast<size_t>(kv_head * p.group + column % p.group) * head_dim;
}
__device__ __forceinline__ u32x2 rounded_four(const f32x4 &x, float factor)
{
    u32x2 packed;
    packed[0] = pack_bf16x2_rne(x[0] * factor, x[1] * factor);
    packed[1] = pack_bf16x2_rne(x[2] * factor, x[3] * factor);
    return packed;
}
// Parts pass between XCDs, whose L2 caches do not see each other's writes: eight bytes at a time by relaxed atomics of device scope, which
// write through and read past them.  (A fence of that scope instead writes back and drops all that an L2 holds: with one in every workgroup
// a decode step of 64 contexts took 250 us for 53.)
__device__ __forceinline__ void store_shared(float *at, const float2 &x)
{
    __hip_atomic_store(reinterpret_cast<unsigned long long *>(at), __builtin_bit_cast(unsigned long long, x), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 load_shared(const float *at)
{
    return __builtin_bit_cast(float2, __hip_atomic_load(reinterpret_cast<const unsigned long long *>(at), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
}

// A sum of 0 is a column without keys.  (Scores of NaN make it NaN.)
__device__ __forceinline__ float inverse_of(float sum) { return sum == 0.0f ? 0.0f : 1.0f / sum; }

template <int HD>
constexpr int kKvFewFloats = 4 * kKvColumns * (HD + 4);

// Few columns: a workgroup takes sixteen of them and a share of their keys, which its four wavefronts deal out among themselves.  (32 columns,
// which halves the conversions of codes: 4 % slower over fifty batches of 2 to 60 rows a request, for half as many workgroups.)  Where
// a context is cut over workgroups, the last of them to finish puts their parts together, in the parts' order: the result does not
// depend on who that was.
template <int HD>
__device__ __forceinline__ void few_columns(const KvAttentionArgs &p, unsigned unit, float *lds_out)
{
    constexpr int VT = HD / 16;
    constexpr int OS = HD + 4;  // row stride of the wavefronts' sums in LDS
    __shared__ float lds_max[4][kKvColumns], lds_sum[4][kKvColumns];
    __shared__ bool is_last;
    __shared__ KvFound found;
    __shared__ unsigned found_share;

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, g = lane >> 4;
    const int kv_head = unit % p.kv_heads;  // neighbouring workgroups, on different XCDs, share nothing
    if (wave == 0) {
        const KvRequest own = longest_first<false>(p, own_request(p));
        auto tiles = [&](const KvRequest &q) { return few_tiles(p, q); };
        KvShare even{kKvWhole, 0, ~0u};
        if (p.parts)
            even = find_share(p, own, kKvMostParts, kKvTarget<HD>, tiles, [&](const KvRequest &q) { return static_cast<float>(tiles(q)) * static_cast<float>(key_tiles(q.length)); });
        const unsigned share = even.share;
        KvFound at;
        const bool is = unit / p.kv_heads < even.most_items && find_request(p, own, unit / p.kv_heads, p.units / p.kv_heads, p.room, [&](const KvRequest &q) { return tiles(q) * parts_of(q, share); },
                                     [&](const KvRequest &q) { return parts_of(q, share) > 1 ? tiles(q) * parts_of(q, share) : 0; }, &at,
                                     p.parts && share == kKvWhole, even.tiles);
        if (lane == 0) {
            found = at;
            found_share = is ? share : 0;
        }
    }
    __syncthreads();
    const unsigned share = __builtin_amdgcn_readfirstlane(found_share);
    if (share == 0) return;
    const KvFound at = uniform(found);
    const unsigned parts = parts_of(at.of, share), part = at.offset % parts, own_share = share_of(at.of, share);
    const unsigned column_tile = at.offset / parts;
    const int first = static_cast<int>(column_tile) * kKvColumns, columns = min(kKvColumns, at.of.rows * p.group - first);

    KvColumnsState<HD, 1> s;
    begin_columns<HD, 1>(p, at.of, first, s);
    const unsigned tiles = key_tiles(s.keys), tile_first = part * own_share, tile_end = min(tiles, tile_first + min(own_share, 0x40000000u));
    attend<HD, 1>(p, at.of, kv_head, first, tile_first + wave, tile_end, 4, s);

    // The four wavefronts' sums, each on its own maximum, put together.
    if (g == 0) {
        lds_max[wave][n] = s.run_max[0];
        lds_sum[wave][n] = s.sum[0][0];
    }
#pragma unroll
    for (int t = 0; t < VT; ++t) *reinterpret_cast<f32x4 *>(&lds_out[(wave * kKvColumns + n) * OS + 16 * t + 4 * g]) = s.out[0][t];
    __syncthreads();
    float *const statistics = p.parts + static_cast<size_t>(p.room) * p.kv_heads * kKvColumns * HD;
    const size_t parts_before = at.before + static_cast<size_t>(column_tile) * parts;  // those of contexts that are cut
    auto place = [&](unsigned of_part, int c) { return ((parts_before + of_part) * p.kv_heads + kv_head) * kKvColumns + c; };
    for (int i = tid; i < columns * (HD / 4); i += 256) {
        const int c = i / (HD / 4), d = i % (HD / 4) * 4;
        float most = -INFINITY;
#pragma unroll
        for (int w = 0; w < 4; ++w) most = fmaxf(most, lds_max[w][c]);
        const float base = most == -INFINITY ? 0.0f : most;
        float sum = 0.0f;
        f32x4 total = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float factor = __builtin_amdgcn_exp2f(lds_max[w][c] - base);
            sum += lds_sum[w][c] * factor;
            total += *reinterpret_cast<const f32x4 *>(&lds_out[(w * kKvColumns + c) * OS + d]) * factor;
        }
        if (parts > 1) {
            const size_t at_part = place(part, c);
            store_shared(p.parts + at_part * HD + d, float2{total[0], total[1]});
            store_shared(p.parts + at_part * HD + d + 2, float2{total[2], total[3]});
            if (d == 0) store_shared(statistics + 2 * at_part, float2{most, sum});
        } else {
            *reinterpret_cast<u32x2 *>(out_at(p, at.of, kv_head, first + c, HD) + d) = rounded_four(total, inverse_of(sum));
        }
    }
    if (parts == 1) return;

    // Every thread's stores are done before the workgroup says so, and who has heard it from all the others loads after that.
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (tid == 0) {
        unsigned *const arrived = p.arrived + parts_before * p.kv_heads + kv_head;
        is_last = atomicAdd(arrived, 1u) == parts - 1;
        if (is_last) atomicExch(arrived, 0u);
    }
    __syncthreads();
    if (!is_last) return;

    // Sixteen bytes a thread; where there are fewer columns than rows of threads, several rows share a column's parts.  A thread asks for its
    // first parts before their factors are known: what this takes is one memory latency after the other, and what it asks for.  (One context of
    // 1000 keys and eight heads of 128 values: 8.8 us with 8 parts ahead, 9.5 with 16.)
    constexpr int LANES = HD / 4, ROWS = 256 / LANES, AHEAD = 8;
    const int across = min(ROWS, columns > 8 ? 16 : columns > 4 ? 8 : columns > 2 ? 4 : columns);
    const int d = tid % LANES * 4, thread_row = tid / LANES, slices = ROWS / across, mine = thread_row / across;
    float2 low[AHEAD], high[AHEAD];
    auto ask = [&](int c, unsigned from) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const unsigned of_part = from + i * slices;
            low[i] = high[i] = float2{0.0f, 0.0f};
            if (c < columns && of_part < parts) {
                const float *const at_part = p.parts + place(of_part, c) * HD + d;
                low[i] = load_shared(at_part);
                high[i] = load_shared(at_part + 2);
            }
        }
    };
    ask(thread_row % across, mine);

    float *const factors = lds_out;  // (parts, 16)
    static_assert(kKvMostParts * kKvColumns + 256 * 4 <= kKvFewFloats<64>, "factors and the threads' sums");
    constexpr int MINE = kKvMostParts / 16;
    const int slice = tid >> 4;
    float2 held[MINE];
    float most = -INFINITY;
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
        const unsigned of_part = slice + 16 * i;
        held[i] = float2{-INFINITY, 0.0f};
        if (of_part < parts && n < columns) held[i] = load_shared(statistics + 2 * place(of_part, n));
    }
#pragma unroll
    for (int i = 0; i < MINE; ++i) most = fmaxf(most, held[i].x);
    most = across_groups_max(most);
    if (g == 0) lds_max[wave][n] = most;
    __syncthreads();
    most = fmaxf(fmaxf(lds_max[0][n], lds_max[1][n]), fmaxf(lds_max[2][n], lds_max[3][n]));
    const float base = most == -INFINITY ? 0.0f : most;
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
        const float factor = __builtin_amdgcn_exp2f(held[i].x - base);
        sum += held[i].y * factor;
        if (slice + 16 * i < parts) factors[(slice + 16 * i) * kKvColumns + n] = factor;
    }
    sum = across_groups_sum(sum);
    if (g == 0) lds_sum[wave][n] = sum;
    __syncthreads();
    f32x4 *const sums = reinterpret_cast<f32x4 *>(lds_out + kKvMostParts * kKvColumns);
    for (int c0 = 0; c0 < columns; c0 += across) {
        const int c = c0 + thread_row % across;
        f32x4 total = {0.f, 0.f, 0.f, 0.f};
        for (unsigned from = mine; from < parts; from += AHEAD * slices) {
            if (c0 != 0 || from != mine) ask(c, from);
            if (c < columns) {
#pragma unroll
                for (int i = 0; i < AHEAD; ++i)
                    if (from + i * slices < parts) total += f32x4{low[i].x, low[i].y, high[i].x, high[i].y} * factors[(from + i * slices) * kKvColumns + c];
            }
        }
        sums[tid] = total;
        __syncthreads();
        if (c < columns && mine == 0) {
            for (int i = 1; i < slices; ++i) total += sums[tid + i * across * LANES];
            const float whole = (lds_sum[0][c] + lds_sum[1][c]) + (lds_sum[2][c] + lds_sum[3][c]);
            *reinterpret_cast<u32x2 *>(out_at(p, at.of, kv_head, first + c, HD) + d) = rounded_four(total, inverse_of(whole));
        }
        __syncthreads();
    }
}

// Many columns: each wavefront has 16 NC of its own, and the workgroup brings the keys and values that all of them read through LDS, as the
// cache holds them, in a ring of four stages: two tiles are worked on between barriers while loads that write LDS themselves fill the other
// two stages.  The wavefronts' registers hold columns, and a tile is read from memory once for four of them.  A stage holds 64 keys' rows and
// the values' HD rows of 64 bytes; their 16-byte pieces are stored at places that keep the sixteen rows that a fragment reads on banks of
// their own.
// What bounds this is the issue of vector instructions.  A tile of 64 keys and 32 columns of 128 values has 68 products, which take 8 cycles of it
// each, and 338 others, 128 of them conversions of codes, at 5 cycles (exponentials 8.5): 2350 cycles, and the matrix cores' own 1088 hide among
// them.  8 prompts of 500 rows over 1000 to 4000 keys, 32 heads on 8 of 128 values: 150 us, 0.83 PFLOP/s.  (Ways there: 158 us when each 16
// keys' page was looked up for itself, 149 with a barrier for each tile.  Three wavefronts a SIMD: 180, for spilled registers; 48 columns a
// wavefront: 143 to 157; priority to wavefronts within products: 143 to 147.)
typedef __attribute__((address_space(3))) void *kv_lds_ptr;
typedef __attribute__((address_space(1))) const void *kv_global_ptr;
typedef __attribute__((address_space(4))) int kv_constant_int;
// One for each 16 keys of a tile.
template <typename T>
struct Four {
    T a, b, c, d;
};
// (Values, not places: a choice among places would put them into memory.)
template <typename T>
__device__ __forceinline__ T pick(T a, T b, T c, T d, int group)
{
    const T low = group & 1 ? b : a, high = group & 1 ? d : c;
    return group & 2 ? high : low;
}
template <typename T>
__device__ __forceinline__ T pick(const Four<T> of, int group) { return pick(of.a, of.b, of.c, of.d, group); }
constexpr int kKvStages = 4;
template <int HD>
constexpr int kKvStageBytes = 2 * kKvTile * HD + 4 * 256;

// Which piece of a key's row stands at a place is the exclusive or of the place and this: by the bits in which the sixteen rows of a
// fragment differ (0 and 1, 4 and 5) beyond those that choose among the rows in the 256 bytes of all banks.
template <int HD>
__device__ __forceinline__ int key_swizzle(int row)
{
    if constexpr (HD == 64) return row >> 4 & 3;
    else if constexpr (HD == 128) return (row >> 1 & 1) | (row >> 4 & 3) << 1;
    else return (row & 3) | (row >> 4 & 3) << 2;
}

// A tile of columns and the tiles of keys tile_first .. end-1 of their context: all of it, or part `part` of `parts`.
struct KvWideWork {
    KvRequest of;
    unsigned column_tile, tile_first, end, part, parts, arrived;
};

template <int HD, int NC, bool JOINS>
__device__ __forceinline__ void attend_wide(const KvAttentionArgs &p, const KvWideWork &work, int kv_head, unsigned item, unsigned char *lds)
{
    constexpr int WIDTH = 4 * 16 * NC, VT = HD / 16, KL = HD / 64, LOADS = kKvTile * HD / 4096;  // of 16 bytes, a thread, for keys and for values
    constexpr int AHEAD = 2;  // pieces that are read before their use
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, g = lane >> 4;
    const KvRequest &of = work.of;
    const unsigned tile_first = JOINS ? work.tile_first : 0, end = work.end;
    const int columns = of.rows * p.group, first = static_cast<int>(work.column_tile) * WIDTH + wave * 16 * NC;
    KvColumnsState<HD, NC> s;
    begin_columns<HD, NC>(p, of, first, s);
    const unsigned own_end = first < columns ? min(end, key_tiles(s.keys)) : 0;  // (behind the last column a wavefront helps with the loads)
    bf16x8 query[NC][2 * KL];
    load_queries<HD, NC>(p, of, kv_head, first, query);

    // What a tile's four groups of keys are on, the same for all threads: read by the scalar unit, whose loads the counting of vector loads
    // below does not meet.
    struct Pages {
        Four<int> block;  // page * kv_heads + head, of page 0 for none
        int fits;         // bit i: there is one
    };
    const kv_constant_int *const table = (const kv_constant_int *)(p.page_table + of.id * p.table_width);
    const int page_mask = (1 << p.page_shift) - 1;
    auto look_up = [&](unsigned tile) {
        Pages pages;
        pages.fits = 0;
        auto one = [&](int i) {
            const unsigned key = tile * kKvTile + 16 * i, there = min(key, static_cast<unsigned>(of.length - 1));
            const int page = table[there >> p.page_shift];
            const bool fits = key == there && page >= 0 && page < p.pages;
            pages.fits |= fits << i;
            return (fits ? page : 0) * p.kv_heads + kv_head;
        };
        if (p.page_shift >= 6) {
            const int block = one(0);
            pages.fits *= 15;
            pages.block = Four<int>{block, block, block, block};
        } else {
            pages.block = Four<int>{one(0), one(1), one(2), one(3)};
        }
        return pages;
    };
    // Where a thread's pieces stand: 16-byte loads of keys begin at a place of the wavefront's 16-key group, those of values at one of the
    // thread's own group, but for pages that hold whole tiles at one of all threads' page.
    unsigned key_offset[LOADS];
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        const int place = i * 256 + tid, row = place / (HD / 16);
        key_offset[i] = (row & 15) * HD + (place % (HD / 16) ^ key_swizzle<HD>(row)) * 16;
    }
    const int load_group = (lane & 3) ^ (lane >> 4);
    const unsigned value_offset = (static_cast<unsigned>(tid >> 2) << p.page_shift) + (p.page_shift >= 6 ? 16 * load_group : 0);
    const float *const scales = lane & 4 ? p.v_scales : p.k_scales;
    auto request = [&](unsigned tile, unsigned char *stage_at, const Pages &pages) {
        const unsigned key0 = tile * kKvTile;
        unsigned char *const to = stage_at + wave * 1024;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const unsigned group = (i * 256u + wave * 64u) / HD;  // (a wavefront's rows are of one)
            const uint8_t *const from = p.k + ((static_cast<size_t>(static_cast<unsigned>(pick(pages.block, group))) << p.page_shift) + ((key0 + 16 * group) & page_mask)) * HD;
            __builtin_amdgcn_global_load_lds((kv_global_ptr)(from + key_offset[i]), (kv_lds_ptr)(to + i * 4096), 16, 0, 0);
        }
        const uint8_t *values;
        if (p.page_shift >= 6) values = p.v + ((static_cast<size_t>(static_cast<unsigned>(pages.block.a)) * HD) << p.page_shift) + (key0 & page_mask);
        else values = p.v + ((static_cast<size_t>(static_cast<unsigned>(pick(pages.block, load_group))) * HD) << p.page_shift) + ((key0 + 16 * load_group) & page_mask);
#pragma unroll
        for (int i = 0; i < LOADS; ++i)
            __builtin_amdgcn_global_load_lds((kv_global_ptr)(values + (static_cast<size_t>(i * 64) << p.page_shift) + value_offset), (kv_lds_ptr)(to + kKvTile * HD + i * 4096), 16, 0, 0);
        // (each wavefront its own: the keys' four scales, then the values', again and again)
        __builtin_amdgcn_global_load_lds((kv_global_ptr)(scales + static_cast<unsigned>(pick(pages.block, lane))), (kv_lds_ptr)(stage_at + 2 * kKvTile * HD + wave * 256), 4, 0, 0);
    };
    const int key_at = ((n >> 2) * 16 + (n & 3)) * HD, key_turn = key_swizzle<HD>((n >> 2) * 16 + (n & 3));
    const int value_at = kKvTile * HD + n * 64 + ((g ^ (n >> 2)) * 16), scale_at = 2 * kKvTile * HD + wave * 256;
    unsigned nan_first = own_end;  // see mark_nan
    // One tile from its stage, while the tile two behind it comes into another.  (That the two do not meet has to be said, or every read of
    // the one waits for all of the other.)
    auto take_tile = [&](const unsigned char *__restrict held, unsigned char *__restrict coming, unsigned tile, int fits, const Pages &after) __attribute__((always_inline)) {
        if (tile + 2 < end) request(tile + 2, coming, after);
        if (tile >= own_end) return;
        const unsigned key0 = tile * kKvTile;
        const float scale_of_keys = *reinterpret_cast<const float *>(held + scale_at + 4 * (n >> 2));
        const float held_scale = *reinterpret_cast<const float *>(held + scale_at + 16 + 4 * g);
        const float scale_of_values = fits >> g & 1 ? held_scale : 1.0f;
        f32x4 scores[NC][4];
        auto key_piece = [&](int i) { return *reinterpret_cast<const u32x4 *>(held + key_at + 4 * (i / KL) * HD + ((4 * (i % KL) + g) ^ key_turn) * 16); };
        auto value_piece = [&](int t) { return *reinterpret_cast<const u32x4 *>(held + value_at + t * 1024); };
        u32x4 ahead[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) ahead[i] = key_piece(i);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int c = 0; c < NC; ++c) scores[c][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < KL; ++j) {
                const int at = i * KL + j;
                const u32x4 codes = ahead[at % AHEAD];
                if (at + AHEAD < 4 * KL) ahead[at % AHEAD] = key_piece(at + AHEAD);
                else ahead[at % AHEAD] = value_piece(at + AHEAD - 4 * KL);
                const bf16x8 low = widened(codes[0], codes[1], scale_of_keys), high = widened(codes[2], codes[3], scale_of_keys);
#pragma unroll
                for (int c = 0; c < NC; ++c) scores[c][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(low, query[c][2 * j], scores[c][i], 0, 0, 0);
#pragma unroll
                for (int c = 0; c < NC; ++c) scores[c][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(high, query[c][2 * j + 1], scores[c][i], 0, 0, 0);
            }
        }
        const bool whole = fits == 15 && key0 + kKvTile <= static_cast<unsigned>(s.fewest);
        if (__builtin_expect(!whole, 0)) hide_unseen<HD, NC>(s, key0, fits >> g & 1, scores);
        lower_for<HD, NC>(scale_of_values, s);
        bf16x8 weights[1][NC][2];
        weigh<HD, NC, 1>(p, scores, s, weights);
        unsigned nan = 0;
#pragma unroll
        for (int t = 0; t < VT; ++t) {
            u32x4 codes = ahead[t % AHEAD];
            if (t + AHEAD < VT) ahead[t % AHEAD] = value_piece(t + AHEAD);
            if (__builtin_expect(!whole, 0)) nan |= drop_nan(codes);
            const bf16x8 low = widened(codes[0], codes[1], scale_of_values), high = widened(codes[2], codes[3], scale_of_values);
#pragma unroll
            for (int c = 0; c < NC; ++c) s.out[c][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(low, weights[0][c][0], s.out[c][t], 0, 0, 0);
#pragma unroll
            for (int c = 0; c < NC; ++c) s.out[c][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(high, weights[0][c][1], s.out[c][t], 0, 0, 0);
        }
        if (__any(nan != 0)) nan_first = min(nan_first, tile);
    };
    if (tile_first < end) {
        // Two tiles at a time: the pair has landed in every wavefront's share of it, and everyone is done with the pair before, whose stages
        // the next one's loads take.
        int fits = 0, other_fits = 0;
        auto begin = [&](unsigned tile, unsigned char *stage_at) {
            const Pages pages = look_up(tile);
            if (tile < end) request(tile, stage_at, pages);
            return pages.fits;
        };
        unsigned char *now = lds, *then = lds + 2 * kKvStageBytes<HD>;
        fits = begin(tile_first, now);
        other_fits = begin(tile_first + 1, now + kKvStageBytes<HD>);
        Pages next = look_up(tile_first + 2), after = look_up(tile_first + 3);
        for (unsigned tile = tile_first; tile < end; tile += 2) {
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            take_tile(now, then, tile, fits, next);
            take_tile(now + kKvStageBytes<HD>, then + kKvStageBytes<HD>, tile + 1, other_fits, after);
            fits = next.fits, other_fits = after.fits;
            next = look_up(tile + 4), after = look_up(tile + 5);
            unsigned char *const done = now;
            now = then, then = done;
        }
    }
    mark_nan<HD, NC>(p, of, kv_head, nan_first, own_end, 1, s);

    // Parts lie as the lanes hold them, 8 bytes of each beside the next one's, and are put together by the last workgroup likewise.
    if constexpr (JOINS) {
        const unsigned part = work.part, parts = work.parts;
        __shared__ bool is_last;
        const size_t all = static_cast<size_t>(p.wide) * WIDTH;
        auto sums_at = [&](size_t unit, int c, int t, int half) {
            return p.wide_parts + ((((unit * 4 + wave) * NC + c) * VT + t) * 2 + half) * 128 + 2 * lane;
        };
        auto statistics_at = [&](size_t unit, int c) { return p.wide_parts + all * HD + 2 * (unit * WIDTH + wave * 16 * NC + 16 * c + n); };
#pragma unroll
        for (int c = 0; c < NC; ++c) {
#pragma unroll
            for (int t = 0; t < VT; ++t) {
                store_shared(sums_at(item, c, t, 0), float2{s.out[c][t][0], s.out[c][t][1]});
                store_shared(sums_at(item, c, t, 1), float2{s.out[c][t][2], s.out[c][t][3]});
            }
            if (g == 0) store_shared(statistics_at(item, c), float2{s.run_max[c], s.sum[c][0]});
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (tid == 0) {
            unsigned *const arrived = p.arrived + (static_cast<size_t>(p.room) + work.arrived) * p.kv_heads + kv_head;
            is_last = atomicAdd(arrived, 1u) == parts - 1;
            if (is_last) atomicExch(arrived, 0u);
        }
        __syncthreads();
        if (!is_last) return;
        // Lane group g asks for the statistics of parts g, g + 4, ...; what each part counts for goes to all four through LDS, each
        // wavefront's to a place of its own.  The sums of two parts are asked for at once (registers
        // end there; one, for heads of 256): this takes one memory latency after the other.
        auto unit_of = [&](unsigned of_part) { return static_cast<size_t>(item) + (static_cast<size_t>(of_part) - part) * p.kv_heads; };
        static_assert(kKvMostWideParts == 16 && 4 * NC * 16 * kKvMostWideParts * sizeof(float) <= kKvStages * kKvStageBytes<HD>, "factors");
        float *const factors = reinterpret_cast<float *>(lds) + wave * NC * 16 * kKvMostWideParts;  // (NC, parts, 16 columns)
        float2 held[NC][4];
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                held[c][i] = float2{-INFINITY, 0.0f};
                if (g + 4 * i < parts) held[c][i] = load_shared(statistics_at(unit_of(g + 4 * i), c));
            }
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const float most = across_groups_max(fmaxf(fmaxf(held[c][0].x, held[c][1].x), fmaxf(held[c][2].x, held[c][3].x)));
            const float base = most == -INFINITY ? 0.0f : most;
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float factor = __builtin_amdgcn_exp2f(held[c][i].x - base);
                sum += held[c][i].y * factor;
                factors[(c * kKvMostWideParts + g + 4 * i) * 16 + n] = factor;
            }
            s.sum[c][0] = across_groups_sum(sum);
#pragma unroll
            for (int t = 0; t < VT; ++t) s.out[c][t] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
        auto ask = [&](unsigned of_part, float2 (&sums)[NC][VT][2]) __attribute__((always_inline)) {
            const float *const at = sums_at(unit_of(of_part), 0, 0, 0);
#pragma unroll
            for (int i = 0; i < 2 * NC * VT; ++i) sums[i / (2 * VT)][i / 2 % VT][i % 2] = load_shared(at + i * 128);
        };
        auto add = [&](unsigned of_part, const float2 (&sums)[NC][VT][2]) __attribute__((always_inline)) {
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const float factor = factors[(c * kKvMostWideParts + of_part) * 16 + n];
#pragma unroll
                for (int t = 0; t < VT; ++t) s.out[c][t] += f32x4{sums[c][t][0].x, sums[c][t][0].y, sums[c][t][1].x, sums[c][t][1].y} * factor;
            }
        };
        float2 one[NC][VT][2];
        unsigned of_part = 0;
        if constexpr (HD < 256) {
            float2 two[NC][VT][2];
#pragma unroll 1
            for (; of_part + 1 < parts; of_part += 2) {
                ask(of_part, one);
                ask(of_part + 1, two);
                add(of_part, one);
                add(of_part + 1, two);
            }
        }
#pragma unroll 1
        for (; of_part < parts; ++of_part) {
            ask(of_part, one);
            add(of_part, one);
        }
    }
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const int column = first + 16 * c + n;
        const float inverse = inverse_of(s.sum[c][0]);
        if (column >= columns) continue;
        uint16_t *const out = out_at(p, of, kv_head, column, HD) + 4 * g;
#pragma unroll
        for (int t = 0; t < VT; ++t) *reinterpret_cast<u32x2 *>(out + 16 * t) = rounded_four(s.out[c][t], inverse);
    }
}

template <int HD, int NC, bool CUT>
__device__ __forceinline__ void many_columns(const KvAttentionArgs &p, unsigned item, unsigned char *lds)
{
    constexpr int WIDTH = 4 * 16 * NC;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kv_head = item % p.kv_heads;
    __shared__ KvFound found;
    __shared__ unsigned found_share;
    auto tiles_of = [&](const KvRequest &q) {
        const int columns = q.rows * p.group;
        return columns > p.few ? (static_cast<unsigned>(columns) + WIDTH - 1) / WIDTH : 0;
    };
    if (wave == 0) {
        const KvRequest own = longest_first<true>(p, own_request(p));
        KvShare even{kKvWhole, 0, ~0u};
        if (CUT)  // (of the rows that see their own keys one by one, each sees half of them on average)
            even = find_share(p, own, kKvMostWideParts, 2 * kKvTarget<HD>, tiles_of, [&](const KvRequest &q) {
                return static_cast<float>(tiles_of(q)) * (static_cast<float>(key_tiles(q.length)) - (p.halves_own ? 0.5f / kKvTile * min(q.rows, q.length) : 0.0f));
            });
        const unsigned share = even.share;
        KvFound at;
        const bool is = item / p.kv_heads < even.most_items && find_request(p, own, item / p.kv_heads, p.wide / p.kv_heads, p.wide_items / p.kv_heads, [&](const KvRequest &q) { return tiles_of(q) * (CUT ? parts_of(q, share, kKvMostWideParts) : 1); },
                                     tiles_of, &at, CUT && share == kKvWhole, even.tiles);
        if (lane == 0) {
            found = at;
            found_share = is ? share : 0;
        }
    }
    __syncthreads();
    const unsigned share = __builtin_amdgcn_readfirstlane(found_share);
    if (share == 0) return;
    const KvFound at = uniform(found);
    const KvRequest of = at.of;
    // (the last columns see the most keys: they come first)
    const unsigned most_parts = CUT ? parts_of(of, share, kKvMostWideParts) : 1;
    KvWideWork work{of, tiles_of(of) - 1 - at.offset / most_parts, 0, 0, at.offset % most_parts, 1, 0};
    const int last_column = min(of.rows * p.group, static_cast<int>(work.column_tile + 1) * WIDTH) - 1;
    work.end = key_tiles(p.causal ? max(0, of.length - of.rows + last_column / p.group + 1) : of.length);
    work.arrived = at.before + work.column_tile;
    if constexpr (CUT) {
        const unsigned own_share = share_of(of, share, kKvMostWideParts);
        work.parts = max(1u, (work.end + own_share - 1) / own_share);
        if (work.part >= work.parts) return;  // (these columns see fewer keys than others of the request)
        work.tile_first = work.part * own_share;
        work.end = min(work.end, work.tile_first + own_share);
        // (A loop of its own for whole contexts: 145 us instead of 150 for 8 prompts none of which is cut.)
        if (work.parts > 1) return attend_wide<HD, NC, true>(p, work, kv_head, item, lds);
    }
    attend_wide<HD, NC, false>(p, work, kv_head, item, lds);
}

template <int HD>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(HD == 64 ? 4 : HD == 128 ? 2 : 1, HD == 64 ? 4 : HD == 128 ? 2 : 1))) void kv_attention_few_kernel(KvAttentionArgs p)
{
    __shared__ __attribute__((aligned(16))) float lds[kKvFewFloats<HD>];
    few_columns<HD>(p, blockIdx.x, lds);
}

// Batches that may hold requests of either kind.
template <int HD>
constexpr int kKvWideTiles = HD == 64 ? 4 : 2;
template <int HD, bool CUT>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(HD == 256 ? 1 : 2))) void kv_attention_mixed_kernel(KvAttentionArgs p)
{
    constexpr size_t few = kKvFewFloats<HD> * sizeof(float), wide = kKvStages * kKvStageBytes<HD>;
    __shared__ __attribute__((aligned(16))) unsigned char lds[few > wide ? few : wide];
    if (blockIdx.x < p.wide) many_columns<HD, kKvWideTiles<HD>, CUT>(p, blockIdx.x, lds);
    else few_columns<HD>(p, blockIdx.x - p.wide, reinterpret_cast<float *>(lds));
}

// Requests of more columns than half a wide tile go to wide tiles: keys and values are widened once for four or two times as many columns
// there.  Below that the wide tile's other wavefronts would have nothing to do.  (At 128 columns of head dimension 64, 4 contexts of 5000
// keys: 60 us in wide tiles, 25 without.  At 64 columns, 16 contexts of 2000: 39 and 33 of dimension 128, 95 and 73 of 256.)
template <int HD>
constexpr int kKvFew = kKvWideTiles<HD> * 32;
// And the room for parts, for each key head: contexts that are cut are longer than one and a half shares, so that they are cut into fewer parts than 5/3
// of their length in shares, and all contexts together are as many shares as there should be workgroups.
template <int HD>
constexpr int kKvRoom = kKvTarget<HD> * 5 / 3;

template <int HD>
hipError_t launch_kv_attention(KvAttentionArgs args, hipStream_t stream)
{
    constexpr long long WIDTH = 4 * 16 * kKvWideTiles<HD>;
    const long long columns = static_cast<long long>(args.rows) * args.group;
    long long tiles = columns / kKvColumns + args.requests, wide_tiles = 0;  // of sixteen columns: each request has one that is not full
    args.few = 0x7fffffff;
    // Each request counts as one row, so that single tokens, however many requests they are of, have the kernel of narrow tiles alone (64 of up to
    // 4096 keys 24.4 us there and 27.4 in the other, 256 of 64 values 61.4 and 82.6).  A prompt among as many that wait goes there as well: one of 300
    // rows behind 2000 keys beside 511 that wait takes 54 us there and 53 in wide tiles, one of 100 49 and 44, one of 500 80 and 70, at 64 values 38 and
    // 49.  A caller to whom that matters leaves out who waits, or gives more rows.
    if (static_cast<long long>(args.rows - args.requests) * args.group > kKvFew<HD>) {
        args.few = kKvFew<HD>;
        // Requests that are wide have more than `few` columns: so many at the most.
        wide_tiles = columns / WIDTH + std::min<long long>(args.requests, columns / (args.few + 1));
        tiles = std::min<long long>(tiles, static_cast<long long>(args.requests) * ((args.few + kKvColumns - 1) / kKvColumns));
    }
    const long long items = tiles * args.kv_heads, wide_items = wide_tiles * args.kv_heads;
    args.room = static_cast<unsigned>(kKvRoom<HD> / args.kv_heads) + 1;
    args.wide_items = static_cast<unsigned>(wide_items);
    args.heads_by_target = static_cast<float>(args.kv_heads) / kKvTarget<HD>;
    const bool fills = wide_items > kKvTarget<HD>;
    args.halves_own = args.causal && !fills;
    // Contexts of narrow tiles are cut wherever one may be longer than the least share, however many requests there are: a long one among many
    // is what is waited for, and shares of a batch without such are longer than its contexts.  (420 and 1024 requests of 16 to 500 keys and one of 131072,
    // a token each, 32 heads on 8 of 128 values: 1163 and 1223 us uncut, 121 and 276.  1024 of 16 to 2000 keys, none of which is cut: 279 and 267.  A
    // prompt of 100 rows behind 2000 keys beside 511 requests that wait, cut into three: 33 and 49, of 500, not cut, 82 and 80.)
    // Those of wide tiles are cut where there may be too few of these for the chip, or few enough that a context much longer than the others is
    // what is waited for.  (47 prompts of 24 rows over 16 to 6834 keys, 80 heads on 5: 166 us uncut, 105; 55 of 108 rows over up to 3537,
    // 16 on 1: 82 and 55.  Even batches pay for it: 8 of 500 rows 147 and 148 at dimension 128, 106 and 117 at 64.)
    // Cuts add at most a target of workgroups, and another where half of a prompt's own keys were left out of the sum that they share.
    // (More key heads than that target are more shares than there should be workgroups: no context is as long as one.)
    const bool cut = (args.table_width << args.page_shift) > kKvLeastShare * kKvTile && args.kv_heads <= kKvTarget<HD>, wide_cut = cut && wide_items != 0 && wide_items <= 4 * kKvTarget<HD>;
    long long units = items + (cut ? kKvTarget<HD> : 0), wide_units = wide_items + (wide_cut ? fills ? kKvTarget<HD> : 2 * kKvTarget<HD> : 0);
    if (cut) {
        const size_t room = static_cast<size_t>(args.room) * args.kv_heads, floats = room * kKvColumns * (HD + 2);
        void *scratch = nullptr;
        hipError_t rc = stream_workspace(stream, (floats + (wide_cut ? static_cast<size_t>(wide_units) * WIDTH * (HD + 2) : 0)) * sizeof(float), &scratch);
        if (rc == hipSuccess) rc = stream_counters(stream, room + (wide_cut ? static_cast<size_t>(wide_items) : 0), &args.arrived);
        if (rc == hipSuccess) {
            args.parts = static_cast<float *>(scratch);
            if (wide_cut) args.wide_parts = static_cast<float *>(scratch) + floats;
        } else if (scratch_unavailable(rc)) {
            units = items;
            wide_units = wide_items;
        } else {
            return rc;
        }
    }
    args.units = static_cast<unsigned>(units);
    args.wide = static_cast<unsigned>(wide_units);
    if (args.wide_parts) kv_attention_mixed_kernel<HD, true><<<args.wide + args.units, 256, 0, stream>>>(args);
    else if (args.wide) kv_attention_mixed_kernel<HD, false><<<args.wide + args.units, 256, 0, stream>>>(args);
    else kv_attention_few_kernel<HD><<<args.units, 256, 0, stream>>>(args);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_attention_kv_cache_bf16(const st_hip_kv_cache &cache, size_t requests, size_t rows, size_t heads, float scale, bool causal,
                                          const int32_t *row_offsets, const int32_t *lengths, const int32_t *page_table, size_t table_width,
                                          const uint16_t *q, size_t ld_q, uint16_t *out, size_t ld_out, hipStream_t stream)
{
    KvAttentionArgs args{};
    args.k = cache.k;
    args.v = cache.v;
    args.k_scales = cache.k_scales;
    args.v_scales = cache.v_scales;
    args.row_offsets = row_offsets;
    args.lengths = lengths;
    args.page_table = page_table;
    args.q = q;
    args.out = out;
    args.ld_q = static_cast<long long>(ld_q);
    args.ld_out = static_cast<long long>(ld_out);
    args.table_width = static_cast<long long>(table_width);
    args.requests = static_cast<int>(requests);
    args.rows = static_cast<int>(rows);
    args.kv_heads = static_cast<int>(cache.kv_heads);
    args.group = static_cast<int>(heads / cache.kv_heads);
    args.pages = static_cast<int>(cache.pages);
    args.page_shift = __builtin_ctzll(cache.page_size);
    // (Not quite 0, so that masked scores of -infinity keep their weight of 0 where the scale is: so small that it makes nothing of any other.)
    args.scale_log2 = std::fabs(scale) * 1.4426950408889634f;
    if (!(args.scale_log2 > 0.0f)) args.scale_log2 = std::numeric_limits<float>::denorm_min();
    args.negative = scale < 0.0f;
    args.causal = causal;
    if (cache.head_dim == 64) return launch_kv_attention<64>(args, stream);
    if (cache.head_dim == 128) return launch_kv_attention<128>(args, stream);
    return launch_kv_attention<256>(args, stream);
}

}  // namespace sthip
