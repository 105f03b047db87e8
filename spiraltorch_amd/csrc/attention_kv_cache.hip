// Attention over a paged cache of e4m3 keys and values with a power of two for every page and head: single tokens, chunks of prompts, and
// an encoder's states, of many requests at once.
//
// The kernel computes the transposed problem, S^T = K Q^T and O^T += V^T P^T, on v_mfma_f32_16x16x32_bf16: a lane owns one column, a
// (token, head) pair, so that the running maximum and sum are its own scalars.  e4m3 values are bf16 values too, so that codes are widened in
// registers without loss (v_cvt_scalef32_pk_bf16_fp8) and the scales stay outside of the products: a page's key scale multiplies its
// scores, its value scale the weights.
// Both operands come from memory in the layout that the matrix cores take, with 16-byte loads and without LDS.  Within a tile of 64
// keys, lane group g (of 16 lanes) owns keys 16g .. 16g+15: row m of the score tile s is key (m/4)*16 + 4s + m%4, which hands lane
// group g of the accumulators keys 16g + 4s + (0..3).  The four tiles together are then a run of 16 keys, in the order in which the
// second product takes them: V^T, which the cache holds as (head_dim, tokens), gives a lane the same 16 keys of one value with one load.
// Every 16-key group lies within a page whatever its size, so that a tile may span up to four pages.
#include <algorithm>

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
    float *parts;  // where the keys are cut over workgroups: (part, row, head): head_dim sums; behind all of them (part, row, head): maximum, sum
    long long ld_q, ld_out, table_width;
    int requests, rows, heads, kv_heads, group, pages, page_shift;
    int tiles, parts_most, part_tiles;  // workgroups along the rows; along the keys, and the least 64-key tiles that one of them takes
    float scale_log2;                   // scale * log2(e)
    bool causal;
};

constexpr int kKvTile = 64;     // keys
constexpr int kKvColumns = 16;  // (token, head) pairs

// The rows' tiles of request r begin at tile row_offsets[r]*group/columns + r: rows fewer than a tile leave room for one
// per request, so that the tile's request follows from its number and the offsets alone.
struct KvItem {
    int request, tile, first_row, rows, length;
};

__device__ __forceinline__ int clamped(int x, int low, int high) { return min(max(x, low), high); }

__device__ __forceinline__ KvItem find_item(const KvAttentionArgs &p, int columns, int tile)
{
    const int lane = threadIdx.x & 63;
    auto first_tile = [&](int r) { return static_cast<int>(static_cast<long long>(clamped(p.row_offsets[r], 0, p.rows)) * p.group / columns) + r; };
    int low = 0, count = p.requests;  // the request is among these
    while (count > 1) {
        const int step = (count + 63) / 64, at = low + lane * step;
        const bool begun = lane * step < count && (lane == 0 || first_tile(at) <= tile);
        const int which = max(0, static_cast<int>(__popcll(__ballot(begun))) - 1);
        const int next = __builtin_amdgcn_readfirstlane(which * step);
        low += next;
        count = min(step, count - next);
    }
    KvItem item;
    item.request = low;
    item.first_row = clamped(p.row_offsets[low], 0, p.rows);
    item.rows = max(0, clamped(p.row_offsets[low + 1], 0, p.rows) - item.first_row);
    item.tile = tile - first_tile(low);
    const long long most = p.table_width << p.page_shift;
    item.length = static_cast<int>(min(static_cast<long long>(max(0, p.lengths[low])), most));
    return item;
}

// The share of a context's `tiles` that part number `part` takes.
__device__ __forceinline__ void part_range(const KvAttentionArgs &p, int tiles, int part, int *first, int *end)
{
    const int share = max(p.part_tiles, (tiles + p.parts_most - 1) / p.parts_most);
    *first = min(static_cast<long long>(tiles), static_cast<long long>(part) * share);
    *end = min(tiles, *first + share);
}

__device__ __forceinline__ bf16x8 widened(unsigned low, unsigned high)
{
    u32x4 r;
    r[0] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(low, 1.0f, false));
    r[1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(low, 1.0f, true));
    r[2] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(high, 1.0f, false));
    r[3] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(high, 1.0f, true));
    return __builtin_bit_cast(bf16x8, r);
}

// 0x7f in the bytes of `codes` that hold NaN, as bytes of 1.0 (0x38), else 0.
__device__ __forceinline__ unsigned nan_bytes(unsigned codes)
{
    const unsigned is = (((codes & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7;  // 1 in a byte
    return is * 0x38u;
}

__device__ __forceinline__ float across_groups_max(float v)  // over the four lane groups, same column
{
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float across_groups_sum(float v)
{
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}

// Four wavefronts share a tile of columns and deal out the keys, 64 at a time.
template <int HD>
__global__ __launch_bounds__(256) void kv_attention_kernel(KvAttentionArgs p)
{
    constexpr int KL = HD / 64;  // 16-byte loads of a key's row, per lane
    constexpr int VT = HD / 16;  // tiles of O^T
    constexpr int OS = HD + 4;   // row stride of the parts in LDS
    __shared__ __attribute__((aligned(16))) float lds_out[4][kKvColumns][OS];
    __shared__ float lds_max[4][kKvColumns], lds_sum[4][kKvColumns];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 15, g = lane >> 4;
    unsigned block = blockIdx.x;
    const int part = block % p.parts_most;
    block /= p.parts_most;
    const int kv_head = block % p.kv_heads;
    const KvItem item = find_item(p, kKvColumns, block / p.kv_heads);
    const int columns = item.rows * p.group;  // of the request: at most rows*heads, below 2^31
    if (item.tile < 0 || static_cast<long long>(item.tile) * kKvColumns >= columns) return;

    const int last = min(columns, item.tile * kKvColumns + kKvColumns) - 1;
    const int column = min(last, item.tile * kKvColumns + n);  // (the last tile's spare columns do what the last one does)
    const int token = column / p.group, head = kv_head * p.group + column % p.group;
    const size_t row = static_cast<size_t>(item.first_row) + token;
    // Keys that the column sees, and the most that any of them here does: those of the last one.
    const int limit = p.causal ? max(0, item.length - item.rows + token + 1) : item.length;
    const int keys = p.causal ? max(0, item.length - item.rows + last / p.group + 1) : item.length;
    int first_tile, end_tile;
    part_range(p, (keys + kKvTile - 1) / kKvTile, part, &first_tile, &end_tile);

    float run_max = -INFINITY, run_sum = 0.0f;
    f32x4 out[VT];
#pragma unroll
    for (int t = 0; t < VT; ++t) out[t] = f32x4{0.f, 0.f, 0.f, 0.f};

    if (first_tile + wave < end_tile) {
        // Q^T: value 64j + 16g + 8h + (0..7) of the column, for step (j, h) of the first product; keys are loaded alike.
        bf16x8 query[2 * KL];
        const uint16_t *const q = p.q + row * p.ld_q + static_cast<size_t>(head) * HD;
#pragma unroll
        for (int j = 0; j < KL; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h)
                query[2 * j + h] = *reinterpret_cast<const bf16x8 *>(q + 64 * j + 16 * g + 8 * h);

        const int *const table = p.page_table + item.request * p.table_width;
        const int page_mask = (1 << p.page_shift) - 1;
        for (int tile = first_tile + wave; tile < end_tile; tile += 4) {
            const int key0 = tile * kKvTile;
            // The pages of the 16 keys that this lane loads (a row of the first product: group n/4), and of those whose scores it holds.
            auto page_at = [&](int key, bool *fits) {
                const int page = key < item.length ? table[key >> p.page_shift] : -1;
                *fits = page >= 0 && page < p.pages;
                return static_cast<size_t>(*fits ? page : 0) * p.kv_heads + kv_head;
            };
            bool key_fits, value_fits;
            const int key_group = key0 + 16 * (n >> 2), value_group = key0 + 16 * g;
            const size_t key_block = page_at(key_group, &key_fits), value_block = page_at(value_group, &value_fits);
            const uint8_t *const k = p.k + ((key_block << p.page_shift) + (key_group & page_mask) + (n & 3)) * HD + 16 * g;
            const uint8_t *const v = p.v + ((value_block * HD + n) << p.page_shift) + (value_group & page_mask);
            u32x4 key_codes[4][KL], value_codes[VT];
#pragma unroll
            for (int s = 0; s < 4; ++s)
#pragma unroll
                for (int j = 0; j < KL; ++j) key_codes[s][j] = *reinterpret_cast<const u32x4 *>(k + 4 * s * HD + 64 * j);
#pragma unroll
            for (int t = 0; t < VT; ++t) value_codes[t] = *reinterpret_cast<const u32x4 *>(v + (static_cast<size_t>(16 * t) << p.page_shift));
            const float key_scale = p.k_scales[value_block] * p.scale_log2, value_scale = p.v_scales[value_block];

            f32x4 scores[4];
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                scores[s] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = 0; j < KL; ++j) {
                    scores[s] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widened(key_codes[s][j][0], key_codes[s][j][1]), query[2 * j], scores[s], 0, 0, 0);
                    scores[s] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widened(key_codes[s][j][2], key_codes[s][j][3]), query[2 * j + 1], scores[s], 0, 0, 0);
                }
            }
            const int seen = value_fits ? limit - value_group : 0;  // of this lane's 16 keys
            const bool whole = __all(seen >= 16);
#pragma unroll
            for (int s = 0; s < 4; ++s)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float x = scores[s][i] * key_scale;
                    scores[s][i] = whole || 4 * s + i < seen ? x : -INFINITY;
                }
            float most = -INFINITY;
#pragma unroll
            for (int s = 0; s < 4; ++s) most = fmaxf(most, fmaxf(fmaxf(scores[s][0], scores[s][1]), fmaxf(scores[s][2], scores[s][3])));
            most = fmaxf(run_max, across_groups_max(most));
            const float base = most == -INFINITY ? 0.0f : most;  // (a column that has seen nothing: its weights are 2^-inf)
            const float shrink = __builtin_amdgcn_exp2f(run_max - base);
            run_max = most;
            run_sum *= shrink;
#pragma unroll
            for (int t = 0; t < VT; ++t) out[t] *= shrink;
            u32x4 weights[2];
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                float w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    w[i] = __builtin_amdgcn_exp2f(scores[s][i] - base);
                    run_sum += w[i];
                    w[i] *= value_scale;
                    if (!whole && 4 * s + i >= seen) w[i] = 0.0f;  // (whatever the scale of a page without keys)
                }
                weights[s >> 1][2 * (s & 1)] = pack_bf16x2_rne(w[0], w[1]);
                weights[s >> 1][2 * (s & 1) + 1] = pack_bf16x2_rne(w[2], w[3]);
            }
            if (!whole) {
                // Values that no column sees, behind the last key or on a page outside the cache, may be anything: 0.  Values that only
                // some columns see go in as they are, and a NaN among them is put where it is seen by hand: 0 * NaN is not 0.
                const int valid = value_fits ? clamped(item.length - value_group, 0, 16) : 0;
                bool nan = false;
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const int bytes = clamped(valid - 4 * c, 0, 4);
                    const unsigned mask = bytes == 4 ? ~0u : (1u << 8 * bytes) - 1u;
#pragma unroll
                    for (int t = 0; t < VT; ++t) {
                        value_codes[t][c] &= mask;
                        nan |= nan_bytes(value_codes[t][c]) != 0;
                    }
                }
                if (__any(nan)) {
                    u32x4 sees[2];
#pragma unroll
                    for (int c = 0; c < 8; ++c)
                        sees[c >> 2][c & 3] = (2 * c < seen ? 0x3f80u : 0u) | (2 * c + 1 < seen ? 0x3f800000u : 0u);
#pragma unroll
                    for (int t = 0; t < VT; ++t) {
                        f32x4 met = {0.f, 0.f, 0.f, 0.f};
                        unsigned is[4];
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            is[c] = nan_bytes(value_codes[t][c]);
                            value_codes[t][c] &= ~((is[c] >> 3 & 0x01010101u) * 0xffu);
                        }
                        met = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widened(is[0], is[1]), __builtin_bit_cast(bf16x8, sees[0]), met, 0, 0, 0);
                        met = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widened(is[2], is[3]), __builtin_bit_cast(bf16x8, sees[1]), met, 0, 0, 0);
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (met[i] > 0.0f) out[t][i] = NAN;
                    }
                }
            }
#pragma unroll
            for (int t = 0; t < VT; ++t) {
                out[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widened(value_codes[t][0], value_codes[t][1]), __builtin_bit_cast(bf16x8, weights[0]), out[t], 0, 0, 0);
                out[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widened(value_codes[t][2], value_codes[t][3]), __builtin_bit_cast(bf16x8, weights[1]), out[t], 0, 0, 0);
            }
        }
        run_sum = across_groups_sum(run_sum);
    }

    // The four wavefronts' sums, each on its own maximum, put together.
    if (g == 0) {
        lds_max[wave][n] = run_max;
        lds_sum[wave][n] = run_sum;
    }
#pragma unroll
    for (int t = 0; t < VT; ++t) *reinterpret_cast<f32x4 *>(&lds_out[wave][n][16 * t + 4 * g]) = out[t];
    __syncthreads();
    for (int i = threadIdx.x; i < kKvColumns * (HD / 4); i += 256) {
        const int c = i / (HD / 4), d = i % (HD / 4) * 4, at = item.tile * kKvColumns + c;
        if (at >= columns) break;
        const int c_token = at / p.group, c_head = kv_head * p.group + at % p.group;
        const size_t c_row = static_cast<size_t>(item.first_row) + c_token;
        float most = -INFINITY;
#pragma unroll
        for (int w = 0; w < 4; ++w) most = fmaxf(most, lds_max[w][c]);
        const float base = most == -INFINITY ? 0.0f : most;
        float sum = 0.0f;
        f32x4 total = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float share = __builtin_amdgcn_exp2f(lds_max[w][c] - base);
            sum += lds_sum[w][c] * share;
            total += *reinterpret_cast<const f32x4 *>(&lds_out[w][c][d]) * share;
        }
        if (p.parts_most > 1) {
            const size_t place = (static_cast<size_t>(part) * p.rows + c_row) * p.heads + c_head;
            float *const statistics = p.parts + static_cast<size_t>(p.parts_most) * p.rows * p.heads * HD;
            if (d == 0) *reinterpret_cast<float2 *>(statistics + 2 * place) = float2{most, sum};
            if (first_tile < end_tile) *reinterpret_cast<f32x4 *>(p.parts + place * HD + d) = total;
            continue;
        }
        // A sum of 0 is a column without keys.  (Scores of NaN make it NaN.)
        const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
        u32x2 packed;
        packed[0] = pack_bf16x2_rne(total[0] * inverse, total[1] * inverse);
        packed[1] = pack_bf16x2_rne(total[2] * inverse, total[3] * inverse);
        *reinterpret_cast<u32x2 *>(p.out + c_row * p.ld_out + static_cast<size_t>(c_head) * HD + d) = packed;
    }
}

// The parts of a context that was cut over workgroups: a wavefront takes a row of a head.
template <int HD>
__global__ __launch_bounds__(256) void kv_attention_join_kernel(KvAttentionArgs p)
{
    constexpr int LANES = HD / 4;
    static_assert(256 % LANES == 0, "whole columns");
    const int d = threadIdx.x % LANES * 4;
    const size_t place = static_cast<size_t>(blockIdx.x) * (256 / LANES) + threadIdx.x / LANES, all = static_cast<size_t>(p.rows) * p.heads;
    if (place >= all) return;
    const size_t row = place / p.heads;
    const int head = static_cast<int>(place % p.heads);
    if (row >= static_cast<size_t>(clamped(p.row_offsets[p.requests], 0, p.rows))) return;  // rows behind the last request's
    const float2 *const statistics = reinterpret_cast<const float2 *>(p.parts + p.parts_most * all * HD);
    float most = -INFINITY;
    for (int part = 0; part < p.parts_most; ++part) most = fmaxf(most, statistics[part * all + place].x);
    const float base = most == -INFINITY ? 0.0f : most;
    float sum = 0.0f;
    f32x4 total = {0.f, 0.f, 0.f, 0.f};
    for (int part = 0; part < p.parts_most; ++part) {
        const float2 own = statistics[part * all + place];
        if (own.y == 0.0f) continue;  // no keys of this column (and perhaps no sums)
        const float share = __builtin_amdgcn_exp2f(own.x - base);
        sum += own.y * share;
        total += *reinterpret_cast<const f32x4 *>(p.parts + (part * all + place) * HD + d) * share;
    }
    const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
    u32x2 packed;
    packed[0] = pack_bf16x2_rne(total[0] * inverse, total[1] * inverse);
    packed[1] = pack_bf16x2_rne(total[2] * inverse, total[3] * inverse);
    *reinterpret_cast<u32x2 *>(p.out + row * p.ld_out + static_cast<size_t>(head) * HD + d) = packed;
}

template <int HD>
hipError_t launch_kv_attention(KvAttentionArgs args, hipStream_t stream)
{
    args.tiles = static_cast<int>(static_cast<long long>(args.rows) * args.group / kKvColumns + args.requests);
    const size_t items = static_cast<size_t>(args.tiles) * args.kv_heads;
    const long long most_tiles = (std::min<long long>(args.table_width << args.page_shift, 0x7fffffff) + kKvTile - 1) / kKvTile;
    args.part_tiles = 16;
    args.parts_most = 1;
    if (items < 2048) args.parts_most = static_cast<int>(std::min<long long>(64, std::max<long long>(1, (most_tiles + args.part_tiles - 1) / args.part_tiles)));
    if (args.parts_most > 1) {
        const size_t columns = static_cast<size_t>(args.rows) * args.heads, bytes = args.parts_most * columns * (HD + 2) * sizeof(float);
        void *scratch = nullptr;
        const hipError_t rc = stream_workspace(stream, bytes, &scratch);
        if (rc == hipSuccess) args.parts = static_cast<float *>(scratch);
        else if (scratch_unavailable(rc)) args.parts_most = 1;
        else return rc;
    }
    const size_t blocks = items * args.parts_most;
    if (blocks > 0x7fffffffu) return hipErrorInvalidValue;
    kv_attention_kernel<HD><<<static_cast<unsigned>(blocks), 256, 0, stream>>>(args);
    hipError_t rc = hipGetLastError();
    if (rc != hipSuccess || args.parts_most == 1) return rc;
    constexpr size_t at_once = 256 / (HD / 4);
    const size_t columns = static_cast<size_t>(args.rows) * args.heads;
    kv_attention_join_kernel<HD><<<static_cast<unsigned>((columns + at_once - 1) / at_once), 256, 0, stream>>>(args);
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
    args.scale_log2 = scale * 1.4426950408889634f;
    args.causal = causal;
    if (cache.head_dim == 64) return launch_kv_attention<64>(args, stream);
    if (cache.head_dim == 128) return launch_kv_attention<128>(args, stream);
    return launch_kv_attention<256>(args, stream);
}

}  // namespace sthip
