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
    float *parts;       // where keys are cut over workgroups: for each of `units` of them 16 columns of head_dim sums, and then 16 maxima and sums
    unsigned *arrived;  // and for every tile of columns how many of its workgroups are done: 0 before a launch and after it
    long long ld_q, ld_out, table_width;
    int requests, rows, heads, kv_heads, group, pages, page_shift;
    int few;         // requests of so many columns or fewer go to the kernel whose wavefronts share them, others to the one of wide tiles
    unsigned units;  // workgroups of the former
    unsigned wide;   // and of the latter
    float heads_by_target;
    float scale_log2;  // |scale| * log2(e), not quite 0
    bool causal, negative;
};

constexpr int kKvTile = 64;     // keys
constexpr int kKvColumns = 16;  // (token, head) pairs of a tile
constexpr int kKvMostParts = 128;
constexpr int kKvLeastShare = 4;  // tiles that a workgroup takes at the least: one for each of its wavefronts

__device__ __forceinline__ int clamped(int x, int low, int high) { return min(max(x, low), high); }

struct KvRequest {
    int first_row, rows, length;
};

__device__ __forceinline__ KvRequest load_request(const KvAttentionArgs &p, int r)
{
    KvRequest q;
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
// A context in parts of `share` tiles, or more where they would be too many to put together.
__device__ __forceinline__ unsigned share_of(const KvRequest &q, unsigned share) { return max(share, (key_tiles(q.length) + kKvMostParts - 1) / kKvMostParts); }
__device__ __forceinline__ unsigned parts_of(const KvRequest &q, unsigned share)
{
    const unsigned mine = share_of(q, share);
    return max(1u, (key_tiles(q.length) + mine - 1) / mine);
}

// Sum over the lanes up to and with this one.
__device__ __forceinline__ unsigned wave_scan(unsigned v)
{
    auto shifted = [](unsigned x, auto control, auto rows) {
        return static_cast<unsigned>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), decltype(control)::value, decltype(rows)::value, 0xf, false));
    };
    using All = std::integral_constant<int, 0xf>;
    v += shifted(v, std::integral_constant<int, 0x111>{}, All{});  // within rows of sixteen: from 1, 2, 4 and 8 lanes before
    v += shifted(v, std::integral_constant<int, 0x112>{}, All{});
    v += shifted(v, std::integral_constant<int, 0x114>{}, All{});
    v += shifted(v, std::integral_constant<int, 0x118>{}, All{});
    v += shifted(v, std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xa>{});  // the last of a row to the next one, in rows 1 and 3
    v += shifted(v, std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xc>{});  // lane 31 to rows 2 and 3
    return v;
}

// Work is numbered by prefix sums over the requests, which every wavefront takes for itself: `count(request)` items each, and the
// request of item number `item` is found by 64 sums at a time (one round of loads for up to 64 requests, two for 4096 ...).  `own`: this lane's
// request where there are no more than 64.
struct KvFound {
    KvRequest of;
    int request;
    unsigned offset;  // of the item within its request's
    unsigned before;  // sum of `other` over the requests before it
};
// False behind the last item; and for all items where they are more than `most`, which row offsets out of order can make them: a launch
// does all of its work or none.
template <class Count, class Other>
__device__ __forceinline__ bool find_request(const KvAttentionArgs &p, const KvRequest &own, unsigned item, unsigned most, Count &&count, Other &&other, KvFound *found)
{
    const int lane = threadIdx.x & 63;
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
        } else {
            const int first = low + lane * step, end = min(low + left, first + step);
            for (int r = first; r < end; ++r) {
                q = load_request(p, r);
                items += count(q);
                others += other(q);
            }
        }
        const unsigned to = wave_scan(items), to_other = wave_scan(others);
        const unsigned long long behind = __ballot(items_before + to > item);
        if (behind == 0 || (left == p.requests && __builtin_amdgcn_readlane(to, 63) > most)) return false;
        const int which = __builtin_ctzll(behind);
        items_before += __builtin_amdgcn_readlane(to - items, which);
        found->before += __builtin_amdgcn_readlane(to_other - others, which);
        low += which * step;
        left = min(step, left - which * step);
        if (step > 1) continue;
        found->request = low;
        found->offset = item - items_before;
        found->of.first_row = __builtin_amdgcn_readlane(q.first_row, which);
        found->of.rows = __builtin_amdgcn_readlane(q.rows, which);
        found->of.length = __builtin_amdgcn_readlane(q.length, which);
        return true;
    }
}

// This lane's request where there are no more than 64 (none: no rows).
__device__ __forceinline__ KvRequest own_request(const KvAttentionArgs &p)
{
    const int lane = threadIdx.x & 63;
    KvRequest q{0, 0, 0};
    if (p.requests <= 64 && lane < p.requests) q = load_request(p, lane);
    return q;
}

// The 64-key tiles that a workgroup takes of a context at the most: all the tiles that there are, over `target` workgroups.  Contexts of
// very different lengths fill the chip evenly so, whatever the host knows of them (it knows the table's width alone).
__device__ __forceinline__ unsigned find_share(const KvAttentionArgs &p, const KvRequest &own)
{
    if (p.parts == nullptr) return 0x7fffffffu;
    float tiles = 0.0f;  // (rounded, but alike in every workgroup, and what it may fall short of the sum by is added below)
    auto add = [&](const KvRequest &q) { tiles += static_cast<float>(few_tiles(p, q)) * static_cast<float>(key_tiles(q.length)); };
    if (p.requests <= 64) {
        add(own);
    } else {
        const int step = (p.requests + 63) / 64, first = (threadIdx.x & 63) * step, end = min(p.requests, first + step);
        for (int r = first; r < end; ++r) add(load_request(p, r));
    }
    const float share = wave_sum(tiles) * p.heads_by_target * 1.001f + 1.0f;
    return __builtin_amdgcn_readfirstlane(max(static_cast<unsigned>(kKvLeastShare), static_cast<unsigned>(fminf(share, 1073741824.0f))));
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
template <int HD, int NC>
struct KvColumnsState {
    f32x4 out[NC][HD / 16];
    float run_max[NC], run_sum[NC];  // in log2, of scaled scores; this lane's share of the sum
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
        s.run_sum[c] = 0.0f;
        s.limit[c] = sees(min(columns - 1, first + 16 * c + n));
#pragma unroll
        for (int t = 0; t < HD / 16; ++t) s.out[c][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    s.fewest = sees(first);
    s.keys = sees(min(columns, first + 16 * NC) - 1);
}

// Tiles `tile`, tile + step, ... below `end` of the request's keys for a wavefront's columns.
template <int HD, int NC>
__device__ __forceinline__ void attend(const KvAttentionArgs &p, const KvRequest &of, int request, int kv_head, int first, unsigned tile_first,
                                       unsigned end, unsigned step, KvColumnsState<HD, NC> &s)
{
    constexpr int KL = HD / 64;  // 16-byte loads of a key's row, per lane
    constexpr int VT = HD / 16;  // tiles of O^T
    if (tile_first >= end) return;
    const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4, columns = of.rows * p.group;

    // Q^T: value 64j + 16g + 8h + (0..7) of the column, for step (j, h) of the first product; keys are loaded alike.  A negative scale
    // goes into its signs, so that the largest score is that of the largest product.
    bf16x8 query[NC][2 * KL];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const int column = min(columns - 1, first + 16 * c + n);
        const uint16_t *const q = p.q + (static_cast<size_t>(of.first_row) + column / p.group) * p.ld_q +
                                  static_cast<size_t>(kv_head * p.group + column % p.group) * HD;
#pragma unroll
        for (int j = 0; j < 2 * KL; ++j) {
            u32x4 raw = *reinterpret_cast<const u32x4 *>(q + 64 * (j / 2) + 16 * g + 8 * (j % 2));
            if (p.negative) raw ^= 0x80008000u;
            query[c][j] = __builtin_bit_cast(bf16x8, raw);
        }
    }

    const int *const table = p.page_table + request * p.table_width;
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

        int seen[NC];  // of this lane's 16 keys
#pragma unroll
        for (int c = 0; c < NC; ++c) seen[c] = value_fits ? s.limit[c] - static_cast<int>(key0) - value_group : 0;
        if (!whole) {
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (i >= seen[c]) scores[c][i >> 2][i & 3] = -INFINITY;
        }
        float most[NC];
        bool grows = false;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            most[c] = -INFINITY;
#pragma unroll
            for (int i = 0; i < 4; ++i) most[c] = fmaxf(most[c], fmaxf(fmaxf(scores[c][i][0], scores[c][i][1]), fmaxf(scores[c][i][2], scores[c][i][3])));
            most[c] = across_groups_max(most[c]) * p.scale_log2;
            grows |= most[c] > s.run_max[c] + 8.0f;
        }
        // The maximum may lag behind by a factor of 2^8: weights are that much larger then, and nothing has to be scaled for most tiles.
        if (__any(grows)) {
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const float up = fmaxf(s.run_max[c], most[c]), shrink = up == s.run_max[c] ? 1.0f : __builtin_amdgcn_exp2f(s.run_max[c] - up);
                s.run_max[c] = up;
                s.run_sum[c] *= shrink;
#pragma unroll
                for (int t = 0; t < VT; ++t) s.out[c][t] *= shrink;
            }
        }
        bf16x8 weights[NC][2];
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const float base = s.run_max[c] == -INFINITY ? 0.0f : s.run_max[c];  // (a column that has seen nothing: its weights are 2^-inf)
            u32x4 packed[2];
            float sums[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = __builtin_amdgcn_exp2f(fmaf(scores[c][i][e], p.scale_log2, -base));
                sums[i] = (w[0] + w[1]) + (w[2] + w[3]);
                packed[i >> 1][2 * (i & 1)] = pack_bf16x2_rne(w[0], w[1]);
                packed[i >> 1][2 * (i & 1) + 1] = pack_bf16x2_rne(w[2], w[3]);
            }
            s.run_sum[c] += (sums[0] + sums[1]) + (sums[2] + sums[3]);
            weights[c][0] = __builtin_bit_cast(bf16x8, packed[0]);
            weights[c][1] = __builtin_bit_cast(bf16x8, packed[1]);
        }
        if (!whole) {
            // Values that a column does not see may be anything, above all those behind the last key or on a page outside the cache, and
            // 0 * NaN is not 0: NaN goes in as 0, and where it is seen is looked for below.
            unsigned is = 0;
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
            for (int c = 0; c < NC; ++c) s.out[c][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(low, weights[c][0], s.out[c][t], 0, 0, 0);
#pragma unroll
            for (int c = 0; c < NC; ++c) s.out[c][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(high, weights[c][1], s.out[c][t], 0, 0, 0);
        }
        if (more) {
            load_values(next, value_page);
            key_page = page_at(next + step * kKvTile + key_group);
            value_page = page_at(next + step * kKvTile + value_group);
        }
    }

    // From the first tile on where NaN was left out: every sum that met one is one.  The same product, of 1 where a value is NaN and 1
    // where it is seen, says which.
    for (tile = masked_first; tile < end; tile += step) {
        const unsigned key0 = tile * kKvTile;
        const int page = page_at(key0 + value_group);
        const uint8_t *const v = values_at(key0, page);
        value_fits = fits(page);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int seen = value_fits ? s.limit[c] - static_cast<int>(key0) - value_group : 0;
            u32x4 sees[2];
#pragma unroll
            for (int i = 0; i < 8; ++i) sees[i >> 2][i & 3] = (2 * i < seen ? 0x3f80u : 0u) | (2 * i + 1 < seen ? 0x3f800000u : 0u);
#pragma unroll
            for (int t = 0; t < VT; ++t) {
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

// Few columns: a workgroup takes sixteen of them and a share of their keys, which its four wavefronts deal out among themselves.  Where
// a context is cut over workgroups, the last of them to finish puts their parts together, in the parts' order: the result does not
// depend on who that was.
template <int HD>
__device__ __forceinline__ void few_columns(const KvAttentionArgs &p, unsigned unit)
{
    constexpr int VT = HD / 16;
    constexpr int OS = HD + 4;  // row stride of the wavefronts' sums in LDS
    __shared__ __attribute__((aligned(16))) float lds_out[4 * kKvColumns * OS];
    __shared__ float lds_max[4][kKvColumns], lds_sum[4][kKvColumns];
    __shared__ bool is_last;

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, g = lane >> 4;
    const int kv_head = unit % p.kv_heads;  // neighbouring workgroups, on different XCDs, share nothing
    const KvRequest own = own_request(p);
    const unsigned share = find_share(p, own);
    KvFound at;
    if (!find_request(p, own, unit / p.kv_heads, p.units / p.kv_heads, [&](const KvRequest &q) { return few_tiles(p, q) * parts_of(q, share); },
                      [&](const KvRequest &q) { return few_tiles(p, q); }, &at))
        return;
    const unsigned parts = parts_of(at.of, share), part = at.offset % parts, own_share = share_of(at.of, share);
    const unsigned column_tile = at.offset / parts;
    const int first = static_cast<int>(column_tile) * kKvColumns, columns = min(kKvColumns, at.of.rows * p.group - first);

    KvColumnsState<HD, 1> s;
    begin_columns<HD, 1>(p, at.of, first, s);
    const unsigned tiles = key_tiles(s.keys), tile_first = part * own_share, tile_end = min(tiles, tile_first + min(own_share, 0x40000000u));
    attend<HD, 1>(p, at.of, at.request, kv_head, first, tile_first + wave, tile_end, 4, s);

    // The four wavefronts' sums, each on its own maximum, put together.
    const float wave_sum_of = across_groups_sum(s.run_sum[0]);
    if (g == 0) {
        lds_max[wave][n] = s.run_max[0];
        lds_sum[wave][n] = wave_sum_of;
    }
#pragma unroll
    for (int t = 0; t < VT; ++t) *reinterpret_cast<f32x4 *>(&lds_out[(wave * kKvColumns + n) * OS + 16 * t + 4 * g]) = s.out[0][t];
    __syncthreads();
    float *const statistics = p.parts + static_cast<size_t>(p.units) * kKvColumns * HD;
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
            const size_t place = static_cast<size_t>(unit) * kKvColumns + c;
            store_shared(p.parts + place * HD + d, float2{total[0], total[1]});
            store_shared(p.parts + place * HD + d + 2, float2{total[2], total[3]});
            if (d == 0) store_shared(statistics + 2 * place, float2{most, sum});
        } else {
            *reinterpret_cast<u32x2 *>(out_at(p, at.of, kv_head, first + c, HD) + d) = rounded_four(total, inverse_of(sum));
        }
    }
    if (parts == 1) return;

    // Every thread's stores are done before the workgroup says so, and who has heard it from all the others loads after that.
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (tid == 0) {
        unsigned *const arrived = p.arrived + static_cast<size_t>(at.before + column_tile) * p.kv_heads + kv_head;
        is_last = atomicAdd(arrived, 1u) == parts - 1;
        if (is_last) atomicExch(arrived, 0u);
    }
    __syncthreads();
    if (!is_last) return;

    auto place = [&](unsigned of_part, int c) { return (static_cast<size_t>(unit) + (static_cast<size_t>(of_part) - part) * p.kv_heads) * kKvColumns + c; };
    float *const factors = lds_out;  // (parts, 16)
    static_assert(kKvMostParts * kKvColumns + 256 * 4 <= 4 * kKvColumns * (64 + 4), "factors and the threads' sums");
    constexpr int MINE = kKvMostParts / 16;
    const int slice = tid >> 4;
    float2 held[MINE];
    float most = -INFINITY;
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
        const unsigned of_part = slice + 16 * i;
        held[i] = float2{-INFINITY, 0.0f};
        if (of_part < parts && n < columns) held[i] = load_shared(statistics + 2 * place(of_part, n));
        most = fmaxf(most, held[i].x);
    }
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
    // Sixteen bytes a thread; where there are fewer columns than rows of threads, several rows share a column's parts.
    constexpr int LANES = HD / 4, ROWS = 256 / LANES;
    const int across = min(ROWS, columns > 8 ? 16 : columns > 4 ? 8 : columns > 2 ? 4 : columns);
    const int d = tid % LANES * 4, thread_row = tid / LANES, slices = ROWS / across, mine = thread_row / across;
    f32x4 *const sums = reinterpret_cast<f32x4 *>(lds_out + kKvMostParts * kKvColumns);
    for (int c0 = 0; c0 < columns; c0 += across) {
        const int c = c0 + thread_row % across;
        f32x4 total = {0.f, 0.f, 0.f, 0.f};
        if (c < columns) {
#pragma unroll 4
            for (unsigned of_part = mine; of_part < parts; of_part += slices) {
                const float *const from = p.parts + place(of_part, c) * HD + d;
                const float2 low = load_shared(from), high = load_shared(from + 2);
                total += f32x4{low.x, low.y, high.x, high.y} * factors[of_part * kKvColumns + c];
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

// Many columns: each wavefront has 16 NC of its own, and all keys that they see.
template <int HD, int NC>
__device__ __forceinline__ void many_columns(const KvAttentionArgs &p, unsigned tile)
{
    constexpr int WIDTH = 4 * 16 * NC;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 15, g = lane >> 4;
    const int kv_head = tile % p.kv_heads;
    KvFound at;
    auto tiles = [&](const KvRequest &q) {
        const int columns = q.rows * p.group;
        return columns > p.few ? (static_cast<unsigned>(columns) + WIDTH - 1) / WIDTH : 0;
    };
    if (!find_request(p, own_request(p), tile / p.kv_heads, p.wide / p.kv_heads, tiles, [](const KvRequest &) { return 0u; }, &at)) return;
    // (the last columns see the most keys: they come first)
    const int columns = at.of.rows * p.group, first = static_cast<int>(tiles(at.of) - 1 - at.offset) * WIDTH + wave * 16 * NC;
    if (first >= columns) return;
    KvColumnsState<HD, NC> s;
    begin_columns<HD, NC>(p, at.of, first, s);
    attend<HD, NC>(p, at.of, at.request, kv_head, first, 0, key_tiles(s.keys), 1, s);
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const int column = first + 16 * c + n;
        const float inverse = inverse_of(across_groups_sum(s.run_sum[c]));
        if (column >= columns) continue;
        uint16_t *const out = out_at(p, at.of, kv_head, column, HD) + 4 * g;
#pragma unroll
        for (int t = 0; t < HD / 16; ++t) *reinterpret_cast<u32x2 *>(out + 16 * t) = rounded_four(s.out[c][t], inverse);
    }
}

template <int HD>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(HD == 64 ? 4 : HD == 128 ? 3 : 2))) void kv_attention_few_kernel(KvAttentionArgs p)
{
    few_columns<HD>(p, blockIdx.x);
}

// Batches that may hold requests of either kind.
template <int HD>
constexpr int kKvWideTiles = HD == 64 ? 4 : 2;
template <int HD>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(HD == 256 ? 1 : 2))) void kv_attention_mixed_kernel(KvAttentionArgs p)
{
    if (blockIdx.x < p.wide) many_columns<HD, kKvWideTiles<HD>>(p, blockIdx.x);
    else few_columns<HD>(p, blockIdx.x - p.wide);
}

// Requests of more columns go to wide tiles: keys and values are widened once for four or two times as many columns there, but a
// context cannot be shared by several workgroups.
constexpr int kKvFew = 32;
// Workgroups that all contexts are cut over, beside one for each tile of columns.
constexpr int kKvTarget = 512;

template <int HD>
hipError_t launch_kv_attention(KvAttentionArgs args, hipStream_t stream)
{
    constexpr int WIDTH = 4 * 16 * kKvWideTiles<HD>;
    const long long columns = static_cast<long long>(args.rows) * args.group;
    long long tiles = columns / kKvColumns + args.requests;  // of sixteen columns: each request has one that is not full
    args.few = 0x7fffffff;
    if (static_cast<long long>(args.rows - args.requests) * args.group > kKvFew) {
        args.few = kKvFew;
        // Requests that are wide have more than `few` columns: so many at the most.
        args.wide = static_cast<unsigned>((columns / WIDTH + std::min<long long>(args.requests, columns / (args.few + 1))) * args.kv_heads);
        tiles = std::min<long long>(tiles, static_cast<long long>(args.requests) * ((args.few + kKvColumns - 1) / kKvColumns));
    }
    const long long items = tiles * args.kv_heads;
    args.heads_by_target = static_cast<float>(args.kv_heads) / kKvTarget;
    long long units = items;
    if (items <= 4096 && (args.table_width << args.page_shift) > kKvLeastShare * kKvTile) {
        units = items + kKvTarget;
        void *scratch = nullptr;
        hipError_t rc = stream_workspace(stream, static_cast<size_t>(units) * kKvColumns * (HD + 2) * sizeof(float), &scratch);
        if (rc == hipSuccess) rc = stream_counters(stream, static_cast<size_t>(items), &args.arrived);
        if (rc == hipSuccess) {
            args.parts = static_cast<float *>(scratch);
        } else if (scratch_unavailable(rc)) {
            units = items;
        } else {
            return rc;
        }
    }
    args.units = static_cast<unsigned>(units);
    if (args.wide) kv_attention_mixed_kernel<HD><<<args.wide + args.units, 256, 0, stream>>>(args);
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
    args.heads = static_cast<int>(heads);
    args.kv_heads = static_cast<int>(cache.kv_heads);
    args.group = static_cast<int>(heads / cache.kv_heads);
    args.pages = static_cast<int>(cache.pages);
    args.page_shift = __builtin_ctzll(cache.page_size);
    // (Not quite 0, so that masked scores of -infinity keep their weight of 0 where the scale is.)
    args.scale_log2 = std::max(std::fabs(scale) * 1.4426950408889634f, 1e-30f);
    args.negative = scale < 0.0f;
    args.causal = causal;
    if (cache.head_dim == 64) return launch_kv_attention<64>(args, stream);
    if (cache.head_dim == 128) return launch_kv_attention<128>(args, stream);
    return launch_kv_attention<256>(args, stream);
}

}  // namespace sthip
