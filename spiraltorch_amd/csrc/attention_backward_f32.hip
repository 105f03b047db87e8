// The backward pass of f32 scaled-dot-product attention with its additive biases: the gradients of
// softmax(scale·q·kᵀ + z_bias + attn_bias)·v with respect to all five, the probabilities worked out again.
//
//   p = exp(s − lse),  dv = pᵀ·g,  ds = p·(g·vᵀ − δ) with δ = Σ g·o,  dq = scale·ds·k,  dk = scale·dsᵀ·q,  dattn = ds,  dz = Σ_query ds
//
// Products run on v_mfma_f32_32x32x2_f32, whose 157 TFLOP/s bound the pass, and on nothing narrower: the operands are f32, and gradients of bf16
// products would not be this function's.  Six products of 2·S²·D against the five that it cannot do without: the scores twice, once for lse,
// which the forward pass does not keep.  One launch works out lse and δ; one dk, dv and the biases' gradients, and leaves ds; one takes dq from
// ds.  Where nobody asks for ds (attn_bias's gradient) and it is above kPairsKept, the first launch works out dq as well, with eight products.
// That instruction takes a value a lane from either operand, so that one copy of a tile in LDS serves rows and columns alike, and accumulators
// go into the next product register by register.
//
// A workgroup owns 32 rows (queries for dq, keys for dk and dv), which its wavefronts all hold as B operands; they deal the tiles of 32
// rows of the other two matrices out among themselves (wavefront w takes tiles w, w + WAVES, ...), each through LDS of its own, and add
// up through LDS at the end, in the order of the wavefronts.  So 16 contexts of 1024 are 512 workgroups, and nothing waits for another
// wavefront before the end.  Few contexts of many tiles have several workgroups a tile, whose sums a further launch adds.  No atomics: the same call
// gives the same bits.
//
// 16 contexts of 1024 x 64 with both biases and all five gradients take 136 µs in three launches (38, 90, 26 µs by themselves), 79 TFLOP/s of
// needed products where a large library product reaches 154; 96 causal ones of 333 x 80 take 109 µs.  What is left: with the rows that stay, the
// sums and a tile's scores in registers there are two wavefronts a SIMD (one above 64 values a head), and the softmax's instructions and a
// tile's wait stand beside the products only where the other wavefront has some.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "device_math.h"
#include "kernels.h"

namespace sthip {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kRows = 32;

typedef unsigned int u32x4_t __attribute__((ext_vector_type(4)));

struct BackwardArgs {
    const float *q, *k, *v, *z_bias, *attn_bias, *out, *grad_out;
    float *grad_q, *grad_k, *grad_v, *grad_z_bias, *grad_attn_bias;
    float *lse, *delta;  // (contexts, padded): lse·log2 e; rows behind the last +infinity and 0
    float *pairs;        // ds, (contexts, S, pair_row): grad_attn_bias, or scratch, or null where dq works it out again
    int contexts, S, D, padded, tiles, swizzle, pair_row;
    // Workgroups to a tile, each of which takes every parts-th of the others' rounds; then sums of theirs, (parts, ...), not scaled yet: of rows, of keys,
    // and the rows' maxima and totals.
    int parts;
    float *part_q, *part_k, *part_v, *part_z, *part_max, *part_total;
    float scale, keep;  // ds counts `keep` times: once, or, where there is one key, not at all (the roundings of p and dp would leave something of it)
    bool wide_bias, wide_pairs;  // four neighbouring values of a row are one aligned load
};

// Workgroup -> (context, tile), XCDs with whole contexts where they divide evenly; under a causal mask the longest tiles first.
__host__ __device__ inline int2 decode(int contexts, int tiles, int swizzle, bool by_tile, bool last_first, unsigned block)
{
    const unsigned of_xcd = swizzle ? contexts >> 3 : contexts, first = swizzle ? (block & 7) * of_xcd : 0, i = swizzle ? block >> 3 : block;
    const unsigned n = static_cast<unsigned>(tiles), tile = by_tile ? i / of_xcd : i % n;
    return int2{static_cast<int>(first + (by_tile ? i % of_xcd : i / n)), static_cast<int>(last_first ? n - 1 - tile : tile)};
}

// A tile of 32 rows of DC values (a multiple of 16; zeros from D on) in LDS.  A row is an odd number of 16-byte chunks, the last of them empty: sixteen
// rows' same chunk lies in sixteen places of the banks, and where a value lies is a lane's place and a constant.
template <int DC>
struct Tile {
    static constexpr int kChunks = DC / 4 + 1, kRow = kChunks * 16, kBytes = (kRows * kChunks + 63) / 64 * 1024, kAcross = (DC + 31) / 32;
};

// Rows of a context, zeros behind the last.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_of(const float *first, int rows, int dim)
{
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<float *>(first), 0, static_cast<int>(static_cast<unsigned>(rows) * dim * 4u), 0x00020000);
}
template <bool VEC>
__device__ __forceinline__ f32x4 fetch4(const __amdgpu_buffer_rsrc_t &rows, int dim, int row, int column)
{
    const unsigned at = (static_cast<unsigned>(row) * dim + column) * 4u;
    if (VEC) {
        const u32x4_t raw = __builtin_amdgcn_raw_buffer_load_b128(rows, at, 0, 0);
        return column < dim ? __builtin_bit_cast(f32x4, raw) : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    f32x4 x;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float raw = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rows, at + e * 4, 0, 0));
        x[e] = column + e < dim ? raw : 0.0f;
    }
    return x;
}

typedef __attribute__((address_space(3))) void *lds_void_ptr;
typedef __attribute__((address_space(3))) void *lds_void_ptr;
// Rows first .. first + 31 of a context's `rows` on their way straight into LDS, 16 bytes (VEC) or 4 a lane and step: what lies at a place is fetched by
// the lane that stands for it, from beyond the descriptor (zeros) where it stands for no value.  The matrix instructions wait for what a wavefront
// computes between them, so that wide loads find where a step's values come from in a table in LDS, which a wavefront writes with its FIRST tile (every
// one writes the same, so that none waits for another).
template <int DC, bool VEC, bool FIRST>
__device__ __forceinline__ void load_tile(const float *matrix, int rows, int dim, int first, unsigned char *to, unsigned char *places, int lane)
{
    constexpr int SIZE = VEC ? 16 : 4, STEPS = Tile<DC>::kBytes / (64 * SIZE);
    constexpr unsigned OF_ROW = Tile<DC>::kRow / SIZE, DOWN = 64 / OF_ROW, ACROSS = 64 % OF_ROW * (SIZE / 4);
    const __amdgpu_buffer_rsrc_t from = rows_of(matrix + static_cast<size_t>(first) * dim, min(rows - first, kRows), dim);
    asm volatile("" : "+v"(lane));  // (kept for all steps, the places would be registers the products need)
    unsigned row = lane / OF_ROW, column = lane % OF_ROW * (SIZE / 4);
    unsigned *const table = reinterpret_cast<unsigned *>(places) + lane;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        unsigned at;
        if (VEC && !FIRST) {
            at = table[s * 64];
        } else {
            at = column < static_cast<unsigned>(dim) && row < kRows ? (row * static_cast<unsigned>(dim) + column) * 4u : 0x80000000u;
            if (VEC) table[s * 64] = at;
            row += DOWN;
            column += ACROSS;
            if (column >= OF_ROW * (SIZE / 4)) {
                row += 1;
                column -= OF_ROW * (SIZE / 4);
            }
        }
        if (VEC) __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (lds_void_ptr)(to + s * 64 * SIZE), 16, at, 0, 0, 0);
        else __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (lds_void_ptr)(to + s * 64 * SIZE), 4, at, 0, 0, 0);
    }
    if (VEC && FIRST) {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
}
template <int DC, bool VEC>
constexpr size_t kPlaces = VEC ? Tile<DC>::kBytes / 4 : 0;  // bytes of the table

__device__ __forceinline__ void wait_for_loads()
{
    __builtin_amdgcn_s_waitcnt(0x0f70);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// Up to 32 rows of biases, or of ds, zeros behind the last: loads beyond them give 0, and stores are dropped.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t bias_rows(const float *first, int rows, int row)
{
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<float *>(first), 0, static_cast<int>(static_cast<unsigned>(min(rows, kRows)) * row * 4u), 0x00020000);
}
// (Which of both is known where it is compiled: loads on two sides of a branch are waited for where the sides meet.)
template <bool WIDE>
__device__ __forceinline__ f32x4 bias4(const __amdgpu_buffer_rsrc_t &from, unsigned at)
{
    if (WIDE) return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(from, at * 4u, 0, 0));
    f32x4 x;
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(from, (at + e) * 4u, 0, 0));
    return x;
}

__device__ __forceinline__ f32x16 mfma(float a, float b, f32x16 sum) { return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, sum, 0, 0, 0); }
__device__ constexpr int row_of(int r) { return (r >> 2) * 8 + (r & 3); }

// What a product reads from LDS is on its way some instructions early: a read takes longer than the matrix instruction that it feeds, and there
// are one or two wavefronts to a SIMD.
// tile · staysᵀ: accumulator registers are the tile's rows, lanes the rows that stay.
template <int DC>
__device__ __forceinline__ f32x16 product(const unsigned char *tile, const f32x4 (&stays)[DC / 8], int li, int lh)
{
    constexpr int AHEAD = 2;
    f32x16 sum = {};
    f32x4 ring[AHEAD];
    const unsigned char *const mine = tile + li * Tile<DC>::kRow + lh * 16;
    auto load = [&](int g) { ring[g % AHEAD] = *reinterpret_cast<const f32x4 *>(mine + g * 32); };
#pragma unroll
    for (int g = 0; g < AHEAD; ++g) load(g);
#pragma unroll
    for (int g = 0; g < DC / 8; ++g) {
        const f32x4 a = ring[g % AHEAD];
        if (g + AHEAD < DC / 8) load(g + AHEAD);
#pragma unroll
        for (int e = 0; e < 4; ++e) sum = mfma(a[e], stays[g][e], sum);
        __builtin_amdgcn_sched_barrier(0);
    }
    return sum;
}
// sums += tileᵀ · weights: registers are the tile's columns, lanes the rows that stay.
template <int DC>
__device__ __forceinline__ void add_product(const unsigned char *tile, const f32x16 &weights, f32x16 (&sums)[Tile<DC>::kAcross], int li, int lh)
{
    constexpr int AHEAD = 8, DT = Tile<DC>::kAcross, STEPS = 16 * DT;
    const unsigned char *const mine = tile + 4 * lh * Tile<DC>::kRow + li * 4;
    float ring[AHEAD];
    auto load = [&](int n) { ring[n % AHEAD] = *reinterpret_cast<const float *>(mine + row_of(n / DT) * Tile<DC>::kRow + n % DT * 128); };
#pragma unroll
    for (int n = 0; n < AHEAD; ++n) load(n);
#pragma unroll
    for (int n = 0; n < STEPS; ++n) {
        sums[n % DT] = mfma(ring[n % AHEAD], weights[n / DT], sums[n % DT]);
        if (n + AHEAD < STEPS) load(n + AHEAD);
        __builtin_amdgcn_sched_barrier(0);
    }
}

// What the wavefront reads from LDS has been read, before loads into the same place.
__device__ __forceinline__ void wait_for_reads()
{
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_s_waitcnt(0xc07f);
    __builtin_amdgcn_wave_barrier();
}

// The wavefronts' sums (a lane has its row, registers the columns), times `by`, into rows first .. first + 31 of a matrix.
template <int DC, int WAVES, bool VEC>
__device__ __forceinline__ void write_rows(const f32x16 (&sums)[Tile<DC>::kAcross], float by, float *to, int first, int rows, int dim, unsigned char *lds)
{
    constexpr int STRIDE = Tile<DC>::kAcross * 32 + 4;
    float *const parts = reinterpret_cast<float *>(lds);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, li = lane & 31, lh = lane >> 5;
    __syncthreads();
#pragma unroll
    for (int dt = 0; dt < Tile<DC>::kAcross; ++dt)
#pragma unroll
        for (int a = 0; a < 4; ++a)
            *reinterpret_cast<f32x4 *>(parts + (wave * kRows + li) * STRIDE + dt * 32 + a * 8 + lh * 4) =
                f32x4{sums[dt][a * 4], sums[dt][a * 4 + 1], sums[dt][a * 4 + 2], sums[dt][a * 4 + 3]};
    __syncthreads();
    constexpr int UNIT = VEC ? 4 : 1, OF_ROW = DC / UNIT;
#pragma unroll 4
    for (int i = tid; i < kRows * OF_ROW; i += WAVES * 64) {
        const int row = i / OF_ROW, column = i % OF_ROW * UNIT;
        if (first + row >= rows || column >= dim) continue;
        const float *const from = parts + row * STRIDE + column;
        float *const at = to + static_cast<size_t>(first + row) * dim + column;
        if constexpr (VEC) {
            f32x4 sum = *reinterpret_cast<const f32x4 *>(from);
#pragma unroll
            for (int w = 1; w < WAVES; ++w) sum += *reinterpret_cast<const f32x4 *>(from + w * kRows * STRIDE);
            *reinterpret_cast<f32x4 *>(at) = sum * by;
        } else {
            float sum = *from;
#pragma unroll
            for (int w = 1; w < WAVES; ++w) sum += from[w * kRows * STRIDE];
            *at = sum * by;
        }
    }
}

// ---- lse, δ, dq: queries stay -----------------------------------------------------------------------------------------------------------
template <int DC, int WAVES, bool VEC, bool CAUSAL, bool DQ>
__global__ __launch_bounds__(WAVES * 64) __attribute__((amdgpu_waves_per_eu(DC <= 64 ? 2 : 1, 4))) void attention_f32_grad_q_kernel(BackwardArgs p)
{
    extern __shared__ __attribute__((aligned(16))) unsigned char backward_lds[];
    __shared__ float maxima[WAVES][kRows], totals[WAVES][kRows];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), li = lane & 31, lh = lane >> 5;
    const int2 item = decode(p.contexts, p.tiles * p.parts, p.swizzle, CAUSAL, CAUSAL, blockIdx.x);
    const int context = item.x, part = item.y % p.parts, q0 = item.y / p.parts * kRows, my_q = q0 + li, S = p.S, D = p.D;
    const int begin = (part * WAVES + wave) * kRows, step = p.parts * WAVES * kRows;  // the wavefront's first tile, and to its next one
    const size_t first = static_cast<size_t>(context) * S;
    unsigned char *const k_tile = backward_lds + wave * 2 * Tile<DC>::kBytes, *const v_tile = k_tile + Tile<DC>::kBytes;
    unsigned char *const places = backward_lds + WAVES * 2 * Tile<DC>::kBytes;
    const int key_end = CAUSAL ? min(S, q0 + kRows) : S, last_key = CAUSAL ? min(my_q, S - 1) : S - 1;
    if (begin < key_end) load_tile<DC, VEC, true>(p.k + first * D, S, D, begin, k_tile, places, lane);
    f32x4 q[DC / 8], g[DC / 8];
    float delta = 0.0f;
    {
        const __amdgpu_buffer_rsrc_t q_rows = rows_of(p.q + first * D, S, D), g_rows = rows_of(p.grad_out + first * D, S, D),
                                     o_rows = rows_of(p.out + first * D, S, D);
#pragma unroll
        for (int c = 0; c < DC / 8; ++c) {
            q[c] = fetch4<VEC>(q_rows, D, my_q, c * 8 + lh * 4);
            g[c] = fetch4<VEC>(g_rows, D, my_q, c * 8 + lh * 4);
            const f32x4 o = fetch4<VEC>(o_rows, D, my_q, c * 8 + lh * 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) delta = fmaf(g[c][e], o[e], delta);
        }
    }
    delta += __shfl_xor(delta, 32);
    const __amdgpu_buffer_rsrc_t biases = bias_rows(p.attn_bias + (first + q0) * S, S - q0, S), z_biases = bias_rows(p.z_bias + first, 1, S);
    // A tile's biases, four keys at a time; what is behind a row's last key is masked with it.
    struct Biases {
        f32x4 of_pair[4], of_key[4];
    };
    auto load_biases = [&](auto wide, int key0, Biases &to) {
        constexpr bool WIDE = decltype(wide)::value;
#pragma unroll
        for (int a = 0; a < 4; ++a) {
            const unsigned key = key0 + a * 8 + lh * 4;
            if (p.attn_bias) to.of_pair[a] = bias4<WIDE>(biases, static_cast<unsigned>(li) * S + key);
            if (p.z_bias) to.of_key[a] = bias4<WIDE>(z_biases, key);
        }
    };
    auto sum_of = [&](const Biases &from, f32x4 (&to)[4]) {
#pragma unroll
        for (int a = 0; a < 4; ++a) {
            to[a] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            if (p.attn_bias) to[a] += from.of_pair[a];
            if (p.z_bias) to[a] += from.of_key[a];
            asm volatile("" : "+v"(to[a]));
        }
    };
    // the scores of a tile, in units of log2 e
    auto scores = [&](const unsigned char *tile, const f32x4 (&with)[4], int key0) {
        f32x16 s = product<DC>(tile, q, li, lh);
#pragma unroll
        for (int a = 0; a < 4; ++a) {
            const int key = key0 + a * 8 + lh * 4;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float x = fmaf(s[a * 4 + e], p.scale, with[a][e]) * kLog2e;
                s[a * 4 + e] = key + e > last_key ? -INFINITY : x;
            }
        }
        return s;
    };
    float most = -INFINITY, total = 0.0f;
    // (the wavefront's two tiles take turns; biases come with their tile, as what is waited for behind the next tile's loads is waited for with them)
    auto sweep = [&](auto wide) {
        Biases next;
        load_biases(wide, begin, next);
        for (int key0 = begin, turn = 0; key0 < key_end; key0 += step, turn ^= 1) {
            f32x4 with[4];
            wait_for_loads();
            wait_for_reads();
            sum_of(next, with);
            load_biases(wide, key0 + step, next);
            if (key0 + step < key_end) load_tile<DC, VEC, false>(p.k + first * D, S, D, key0 + step, turn ? k_tile : v_tile, places, lane);
            const f32x16 s = scores(turn ? v_tile : k_tile, with, key0);
            float top = most;
#pragma unroll
            for (int r = 0; r < 16; ++r) top = fmaxf(top, s[r]);
            const float safe = top == -INFINITY ? 0.0f : top;
            total *= __builtin_amdgcn_exp2f(most - safe);
            most = top;
#pragma unroll
            for (int r = 0; r < 16; ++r) total += __builtin_amdgcn_exp2f(s[r] - safe);
        }
    };
    if (p.wide_bias) sweep(std::true_type{});
    else sweep(std::false_type{});
    auto load_keys = [&](int key0) {
        if (key0 < key_end) load_tile<DC, VEC, false>(p.k + first * D, S, D, key0, k_tile, places, lane);
    };
    auto load_values = [&](int key0) {
        if (key0 < key_end) load_tile<DC, VEC, false>(p.v + first * D, S, D, key0, v_tile, places, lane);
    };
    if constexpr (DQ) {
        wait_for_reads();
        load_values(begin);
        load_keys(begin);
    }
    {
        const float other = __shfl_xor(most, 32), other_total = __shfl_xor(total, 32), top = fmaxf(most, other), safe = top == -INFINITY ? 0.0f : top;
        total = total * __builtin_amdgcn_exp2f(most - safe) + other_total * __builtin_amdgcn_exp2f(other - safe);
        most = top;
    }
    if (lh == 0) {
        maxima[wave][li] = most;
        totals[wave][li] = total;
    }
    __syncthreads();
    float top = maxima[0][li];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) top = fmaxf(top, maxima[w][li]);
    const float safe = top == -INFINITY ? 0.0f : top;
    float sum = 0.0f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) sum += totals[w][li] * __builtin_amdgcn_exp2f(maxima[w][li] - safe);
    // (a row without keys: every p is 0)
    const float lse = my_q < S && sum != 0.0f ? safe + __log2f(sum) : INFINITY;
    if (wave == 0 && lh == 0) {
        const size_t at = static_cast<size_t>(context) * p.padded + my_q, of_part = static_cast<size_t>(part) * p.contexts * p.padded;
        if (p.parts > 1) {
            p.part_max[of_part + at] = top;
            p.part_total[of_part + at] = sum;
        } else {
            p.lse[at] = lse;
        }
        if (part == 0) p.delta[at] = my_q < S ? delta : 0.0f;
    }
    if constexpr (DQ) {
        f32x16 dq[Tile<DC>::kAcross];
#pragma unroll
        for (int dt = 0; dt < Tile<DC>::kAcross; ++dt) dq[dt] = f32x16{};
        auto second = [&](auto wide) {
            for (int key0 = begin; key0 < key_end; key0 += step) {
                Biases biases_of;
                f32x4 with[4];
                wait_for_loads();
                load_biases(wide, key0, biases_of);
                const f32x16 dp = product<DC>(v_tile, g, li, lh);
                sum_of(biases_of, with);
                wait_for_reads();
                load_values(key0 + step);  // each tile's successor as soon as it has been read
                f32x16 s = scores(k_tile, with, key0);
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(s[r] - lse) * (dp[r] - delta);
                add_product<DC>(k_tile, s, dq, li, lh);
                wait_for_reads();
                load_keys(key0 + step);
            }
        };
        if (p.wide_bias) second(std::true_type{});
        else second(std::false_type{});
        write_rows<DC, WAVES, VEC>(dq, p.scale * p.keep, p.grad_q + first * D, q0, S, D, backward_lds);
    }
}

// dq = scale·ds·k where the pass for dk and dv has left ds.
template <int DC, int WAVES, bool VEC, bool CAUSAL>
__global__ __launch_bounds__(WAVES * 64) __attribute__((amdgpu_waves_per_eu(DC <= 128 ? 2 : 1, 4))) void attention_f32_grad_q_of_pairs_kernel(BackwardArgs p)
{
    extern __shared__ __attribute__((aligned(16))) unsigned char backward_lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), li = lane & 31, lh = lane >> 5;
    const int2 item = decode(p.contexts, p.tiles * p.parts, p.swizzle, CAUSAL, CAUSAL, blockIdx.x);
    const int context = item.x, part = item.y % p.parts, q0 = item.y / p.parts * kRows, my_q = q0 + li, S = p.S, D = p.D;
    const int begin = (part * WAVES + wave) * kRows, step = p.parts * WAVES * kRows;  // the wavefront's first tile, and to its next one
    const size_t first = static_cast<size_t>(context) * S;
    const int key_end = CAUSAL ? min(S, q0 + kRows) : S, last_key = CAUSAL ? min(my_q, S - 1) : S - 1;
    unsigned char *const tiles = backward_lds + wave * 2 * Tile<DC>::kBytes;  // they take turns
    unsigned char *const places = backward_lds + WAVES * 2 * Tile<DC>::kBytes;
    const __amdgpu_buffer_rsrc_t pairs = bias_rows(p.pairs + (first + q0) * p.pair_row, S - q0, p.pair_row);
    f32x4 ds[4];
    f32x16 dq[Tile<DC>::kAcross];
#pragma unroll
    for (int dt = 0; dt < Tile<DC>::kAcross; ++dt) dq[dt] = f32x16{};
    auto sweep = [&](auto wide) {
        auto load = [&](auto starts, int key0, int turn) {
            if (key0 >= key_end) return;
            load_tile<DC, VEC, decltype(starts)::value>(p.k + first * D, S, D, key0, tiles + turn * Tile<DC>::kBytes, places, lane);
#pragma unroll
            for (int a = 0; a < 4; ++a) ds[a] = bias4<decltype(wide)::value>(pairs, static_cast<unsigned>(li) * p.pair_row + key0 + a * 8 + lh * 4);
        };
        load(std::true_type{}, begin, 0);
        for (int key0 = begin, turn = 0; key0 < key_end; key0 += step, turn ^= 1) {
            f32x16 weights;
            wait_for_loads();
            wait_for_reads();
#pragma unroll
            for (int r = 0; r < 16; ++r) weights[r] = key0 + row_of(r) + 4 * lh > last_key ? 0.0f : ds[r >> 2][r & 3];
            load(std::false_type{}, key0 + step, turn ^ 1);
            add_product<DC>(tiles + turn * Tile<DC>::kBytes, weights, dq, li, lh);
        }
    };
    if (p.wide_pairs) sweep(std::true_type{});
    else sweep(std::false_type{});
    if (p.parts > 1) write_rows<DC, WAVES, VEC>(dq, 1.0f, p.part_q + (static_cast<size_t>(part) * p.contexts * S + first) * D, q0, S, D, backward_lds);
    else write_rows<DC, WAVES, VEC>(dq, p.scale * p.keep, p.grad_q + first * D, q0, S, D, backward_lds);
}

// ---- dk, dv, the biases' gradients: keys stay -----------------------------------------------------------------------------------------------
// Heads above 128 values have room for one of dk and dv in their registers, and take two launches.
template <int DC, int WAVES, bool VEC, bool CAUSAL, bool DK, bool DV>
__global__ __launch_bounds__(WAVES * 64) __attribute__((amdgpu_waves_per_eu(DC <= 64 ? 2 : 1, 4))) void attention_f32_grad_kv_kernel(BackwardArgs p)
{
    extern __shared__ __attribute__((aligned(16))) unsigned char backward_lds[];
    __shared__ float totals[WAVES][kRows];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), li = lane & 31, lh = lane >> 5;
    const int2 item = decode(p.contexts, p.tiles * p.parts, p.swizzle, CAUSAL, false, blockIdx.x);
    const int context = item.x, part = item.y % p.parts, k0 = item.y / p.parts * kRows, my_key = k0 + li, S = p.S, D = p.D;
    const int step = p.parts * WAVES * kRows;
    const size_t first = static_cast<size_t>(context) * S;
    unsigned char *const q_tile = backward_lds + wave * 2 * Tile<DC>::kBytes, *const g_tile = q_tile + Tile<DC>::kBytes;
    unsigned char *const places = backward_lds + WAVES * 2 * Tile<DC>::kBytes;
    auto load_queries = [&](auto starts, int row0) {
        if (row0 < S) load_tile<DC, VEC, decltype(starts)::value>(p.q + first * D, S, D, row0, q_tile, places, lane);
    };
    auto load_grads = [&](int row0) {
        if (row0 < S) load_tile<DC, VEC, false>(p.grad_out + first * D, S, D, row0, g_tile, places, lane);
    };
    const int start = (CAUSAL ? k0 : 0) + (part * WAVES + wave) * kRows;
    load_queries(std::true_type{}, start);
    load_grads(start);
    f32x4 k[DC / 8], v[DK ? DC / 8 : 1];
    {
        const __amdgpu_buffer_rsrc_t k_rows = rows_of(p.k + first * D, S, D), v_rows = rows_of(p.v + first * D, S, D);
#pragma unroll
        for (int c = 0; c < DC / 8; ++c) {
            k[c] = fetch4<VEC>(k_rows, D, my_key, c * 8 + lh * 4);
            if (DK) v[DK ? c : 0] = fetch4<VEC>(v_rows, D, my_key, c * 8 + lh * 4);
        }
    }
    const float z = p.z_bias && my_key < S ? p.z_bias[first + my_key] : 0.0f;
    f32x16 dk[DK ? Tile<DC>::kAcross : 1], dv[DV ? Tile<DC>::kAcross : 1];
    if (DK)
#pragma unroll
        for (int dt = 0; dt < Tile<DC>::kAcross; ++dt) dk[DK ? dt : 0] = f32x16{};
    if (DV)
#pragma unroll
        for (int dt = 0; dt < Tile<DC>::kAcross; ++dt) dv[DV ? dt : 0] = f32x16{};
    float dz = 0.0f;
    if (CAUSAL && DK && p.grad_attn_bias && my_key < S)  // queries before the tile do not see it
        for (int q = (part * WAVES + wave) * 2 + lh; q < k0; q += p.parts * WAVES * 2) p.grad_attn_bias[(first + q) * S + my_key] = 0.0f;
    for (int row0 = start; row0 < S; row0 += step) {
        // the biases of the lane's key; beyond the descriptor for a key behind the last
        const unsigned at = my_key < S ? (4u * lh * S + my_key) * 4u : 0x80000000u;
        float bias[16];
        f32x4 lse[4], delta[4];
        const size_t of_rows = static_cast<size_t>(context) * p.padded + row0 + 4 * lh;
        wait_for_loads();
        if (p.attn_bias) {
            const __amdgpu_buffer_rsrc_t biases = bias_rows(p.attn_bias + (first + row0) * S, S - row0, S);
#pragma unroll
            for (int r = 0; r < 16; ++r) bias[r] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(biases, at + row_of(r) * S * 4u, 0, 0));
        }
#pragma unroll
        for (int a = 0; a < 4; ++a) {
            lse[a] = *reinterpret_cast<const f32x4 *>(p.lse + of_rows + a * 8);
            if (DK) delta[a] = *reinterpret_cast<const f32x4 *>(p.delta + of_rows + a * 8);
        }
        f32x16 s = product<DC>(q_tile, k, li, lh);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const float with = p.attn_bias ? bias[r] + z : z;
            const float x = __builtin_amdgcn_exp2f(fmaf(s[r], p.scale, with) * kLog2e - lse[r >> 2][r & 3]);
            s[r] = CAUSAL && my_key > row0 + row_of(r) + 4 * lh ? 0.0f : x;
        }
        f32x16 dp;
        if constexpr (DK) dp = product<DC>(g_tile, v, li, lh);
        if constexpr (DV) add_product<DC>(g_tile, s, dv, li, lh);
        // (what was loaded into registers is used before the next loads: these stand behind a branch, where waiting for others is waiting for them)
        if constexpr (DK) {
#pragma unroll
            for (int a = 0; a < 4; ++a) asm volatile("" : "+v"(delta[a]));
        }
        wait_for_reads();
        load_grads(row0 + step);  // each tile's successor as soon as it has been read
        if constexpr (DK) {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                s[r] *= dp[r] - delta[r >> 2][r & 3];
                dz += s[r];
            }
            add_product<DC>(q_tile, s, dk, li, lh);
            if (p.pairs) {
                const __amdgpu_buffer_rsrc_t pairs = bias_rows(p.pairs + (first + row0) * p.pair_row, S - row0, p.pair_row);
                const unsigned to = my_key < S ? (4u * lh * p.pair_row + my_key) * 4u : 0x80000000u;
#pragma unroll
                for (int r = 0; r < 16; ++r) __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(s[r] * p.keep), pairs, to + row_of(r) * p.pair_row * 4u, 0, 0);
            }
        }
        wait_for_reads();
        load_queries(std::false_type{}, row0 + step);
    }
    if constexpr (DK) {
        if (p.grad_z_bias) {
            dz += __shfl_xor(dz, 32);
            if (lh == 0) totals[wave][li] = dz;
            __syncthreads();
            if (tid < kRows && my_key < S) {
                float sum = totals[0][li];
#pragma unroll
                for (int w = 1; w < WAVES; ++w) sum += totals[w][li];
                if (p.parts > 1) p.part_z[static_cast<size_t>(part) * p.contexts * S + first + my_key] = sum;
                else p.grad_z_bias[first + my_key] = sum * p.keep;
            }
        }
        if (p.parts > 1) write_rows<DC, WAVES, VEC>(dk, 1.0f, p.part_k + (static_cast<size_t>(part) * p.contexts * S + first) * D, k0, S, D, backward_lds);
        else write_rows<DC, WAVES, VEC>(dk, p.scale * p.keep, p.grad_k + first * D, k0, S, D, backward_lds);
    }
    if constexpr (DV) {
        float *const to = p.parts > 1 ? p.part_v + static_cast<size_t>(part) * p.contexts * S * D : p.grad_v;
        write_rows<DC, WAVES, VEC>(dv, 1.0f, to + first * D, k0, S, D, backward_lds);
    }
}

// The parts of rows' log-sum-exps together.
__global__ __launch_bounds__(256) void attention_f32_join_lse_kernel(BackwardArgs p)
{
    const size_t rows = static_cast<size_t>(p.contexts) * p.padded, at = static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x;
    if (at >= rows) return;
    float top = p.part_max[at];
    for (int part = 1; part < p.parts; ++part) top = fmaxf(top, p.part_max[part * rows + at]);
    const float safe = top == -INFINITY ? 0.0f : top;
    float sum = 0.0f;
    for (int part = 0; part < p.parts; ++part) sum += p.part_total[part * rows + at] * __builtin_amdgcn_exp2f(p.part_max[part * rows + at] - safe);
    p.lse[at] = static_cast<int>(at % p.padded) < p.S && sum != 0.0f ? safe + __log2f(sum) : INFINITY;
}
// The parts of the gradients together, in their order.
__global__ __launch_bounds__(256) void attention_f32_join_kernel(BackwardArgs p)
{
    const size_t rows = static_cast<size_t>(p.contexts) * p.S, values = blockIdx.y == 3 ? rows : rows * p.D;
    const float *const from = blockIdx.y == 0 ? p.part_q : blockIdx.y == 1 ? p.part_k : blockIdx.y == 2 ? p.part_v : p.part_z;
    float *const to = blockIdx.y == 0 ? p.grad_q : blockIdx.y == 1 ? p.grad_k : blockIdx.y == 2 ? p.grad_v : p.grad_z_bias;
    const float by = blockIdx.y < 2 ? p.scale : 1.0f;  // (more than one part has more than one key)
    if (!to) return;
    for (size_t at = static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x; at < values; at += static_cast<size_t>(gridDim.x) * 256) {
        float sum = from[at];
        for (int part = 1; part < p.parts; ++part) sum += from[part * values + at];
        to[at] = sum * by;
    }
}

// Values of ds that are kept from dk's pass for dq's where nobody asked for them: 256 MiB, as much as the last-level cache holds.  Kept and worked out
// again: 16 contexts of 1024 x 64 145 and 170 µs, 4 of 2048 x 80 217 and 270, 96 causal ones of 333 x 80 134 and 139.
constexpr size_t kPairsKept = 64u << 20;

// Workgroups to a tile: as many as the chip has room for at once where one a tile would be half of that or less, of two rounds or more each.  3 causal
// contexts of 659 x 256 with biases take 195 µs so and 490 with one a tile, 8 of 512 x 128 64 and 78; 16 of 512 x 128, one a tile, 82.
int parts_of(size_t workgroups, size_t tiles, size_t head_dim)
{
    const size_t room = head_dim <= 64 ? 512 : 256, rounds = tiles / (head_dim <= 128 ? 4 : 2);
    return static_cast<int>(std::max<size_t>(1, std::min({room / workgroups, rounds / 2, static_cast<size_t>(16)})));
}

template <class Kernel>
hipError_t launch(Kernel kernel, const BackwardArgs &args, int waves, size_t lds, bool by_tile, bool last_first, hipStream_t stream)
{
    const size_t blocks = static_cast<size_t>(args.contexts) * args.tiles * args.parts;
    for (const size_t block : {static_cast<size_t>(0), blocks - 1}) {  // the grid is what the kernels' decode assumes
        const int2 item = decode(args.contexts, args.tiles * args.parts, args.swizzle, by_tile, last_first, static_cast<unsigned>(block));
        if (blocks > kMaxDim || item.x < 0 || item.x >= args.contexts || item.y < 0 || item.y >= args.tiles * args.parts) return hipErrorInvalidConfiguration;
    }
    const hipError_t rc = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds));
    if (rc != hipSuccess) return rc;
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(waves * 64), lds, stream, args);
    return hipGetLastError();
}

template <int DC, int WAVES, bool VEC, bool CAUSAL>
hipError_t launch_waves(const BackwardArgs &args, hipStream_t stream)
{
    constexpr size_t lds = std::max<size_t>(WAVES * 2 * Tile<DC>::kBytes + kPlaces<DC, VEC>, WAVES * kRows * (Tile<DC>::kAcross * 32 + 4) * sizeof(float));
    hipError_t rc = args.pairs ? launch(attention_f32_grad_q_kernel<DC, WAVES, VEC, CAUSAL, false>, args, WAVES, lds, CAUSAL, CAUSAL, stream)
                               : launch(attention_f32_grad_q_kernel<DC, WAVES, VEC, CAUSAL, true>, args, WAVES, lds, CAUSAL, CAUSAL, stream);
    if (rc != hipSuccess) return rc;
    if (args.parts > 1) {
        hipLaunchKernelGGL(attention_f32_join_lse_kernel, dim3(static_cast<unsigned>((static_cast<size_t>(args.contexts) * args.padded + 255) / 256)), dim3(256), 0,
                           stream, args);
        rc = hipGetLastError();
        if (rc != hipSuccess) return rc;
    }
    if constexpr (DC <= 128) {
        rc = launch(attention_f32_grad_kv_kernel<DC, WAVES, VEC, CAUSAL, true, true>, args, WAVES, lds, CAUSAL, false, stream);
    } else {
        rc = launch(attention_f32_grad_kv_kernel<DC, WAVES, VEC, CAUSAL, true, false>, args, WAVES, lds, CAUSAL, false, stream);
        if (rc != hipSuccess) return rc;
        rc = launch(attention_f32_grad_kv_kernel<DC, WAVES, VEC, CAUSAL, false, true>, args, WAVES, lds, CAUSAL, false, stream);
    }
    if (rc != hipSuccess || !args.pairs) return rc;
    rc = launch(attention_f32_grad_q_of_pairs_kernel<DC, WAVES, VEC, CAUSAL>, args, WAVES, lds, CAUSAL, CAUSAL, stream);
    if (rc != hipSuccess || args.parts == 1) return rc;
    const size_t values = static_cast<size_t>(args.contexts) * args.S * std::max(args.D, 1);
    hipLaunchKernelGGL(attention_f32_join_kernel, dim3(static_cast<unsigned>(std::min<size_t>((values + 255) / 256, 2048)), 4), dim3(256), 0, stream, args);
    return hipGetLastError();
}

template <int DC, bool VEC, bool CAUSAL>
hipError_t launch_variant(const BackwardArgs &args, hipStream_t stream)
{
    if constexpr (DC > 128) {
        return launch_waves<DC, 2, VEC, CAUSAL>(args, stream);  // 64 KiB of tiles a wavefront
    } else if constexpr (DC > 64) {
        // One wavefront a SIMD: two workgroups of two a compute unit cover each other's waits where there are enough of them, and a causal mask's
        // uneven ones even out (longest first).  Two and four wavefronts: 96 causal contexts of 333 x 80 (1056 workgroups) 134 and 151 µs, 48
        // (528) 93 and 92; 64 of 1024 x 128 without a mask (2048) 1375 and 1432, 96 of 333 x 96 (1056) 269 and 246.
        const bool many = static_cast<size_t>(args.contexts) * args.tiles >= (CAUSAL ? 768 : 2048);
        return many ? launch_waves<DC, 2, VEC, CAUSAL>(args, stream) : launch_waves<DC, 4, VEC, CAUSAL>(args, stream);
    } else {
        return launch_waves<DC, 4, VEC, CAUSAL>(args, stream);
    }
}

template <int DC>
hipError_t launch_width(const BackwardArgs &args, bool vec, bool causal, hipStream_t stream)
{
    if (vec) return causal ? launch_variant<DC, true, true>(args, stream) : launch_variant<DC, true, false>(args, stream);
    return causal ? launch_variant<DC, false, true>(args, stream) : launch_variant<DC, false, false>(args, stream);
}

}  // namespace

hipError_t launch_attention_backward_f32(size_t contexts, size_t sequence, size_t head_dim, float scale, bool causal, const float *q, const float *k,
                                         const float *v, const float *z_bias, const float *attn_bias, const float *out, const float *grad_out,
                                         float *grad_q, float *grad_k, float *grad_v, float *grad_z_bias, float *grad_attn_bias, hipStream_t stream)
{
    BackwardArgs args{};
    args.q = q;
    args.k = k;
    args.v = v;
    args.z_bias = z_bias;
    args.attn_bias = attn_bias;
    args.out = out;
    args.grad_out = grad_out;
    args.grad_q = grad_q;
    args.grad_k = grad_k;
    args.grad_v = grad_v;
    args.grad_z_bias = grad_z_bias;
    args.grad_attn_bias = grad_attn_bias;
    args.contexts = static_cast<int>(contexts);
    args.S = static_cast<int>(sequence);
    args.D = static_cast<int>(head_dim);
    args.tiles = static_cast<int>((sequence + kRows - 1) / kRows);
    args.padded = args.tiles * kRows;
    args.swizzle = contexts % 8 == 0;
    args.scale = scale;
    args.keep = sequence == 1 ? 0.0f : 1.0f;
    auto aligned = [](const void *at) { return reinterpret_cast<uintptr_t>(at) % 16 == 0; };
    args.wide_bias = sequence % 4 == 0 && aligned(attn_bias) && aligned(z_bias);
    const size_t rows = contexts * args.padded, pair_row = grad_attn_bias ? sequence : (sequence + 3) / 4 * 4;
    const size_t kept = !grad_attn_bias && contexts * sequence * pair_row <= kPairsKept ? contexts * sequence * pair_row : 0;
    const size_t values = (contexts * sequence * head_dim + 63) / 64 * 64, keys = (contexts * sequence + 63) / 64 * 64;
    args.parts = grad_attn_bias || kept ? parts_of(contexts * args.tiles, args.tiles, head_dim) : 1;
    const size_t of_parts = args.parts > 1 ? args.parts * (3 * values + keys + 2 * rows) : 0;
    void *scratch = nullptr;
    const hipError_t rc = stream_workspace(stream, (kept + 2 * rows + of_parts) * sizeof(float), &scratch);
    if (rc != hipSuccess) return rc;
    args.pairs = grad_attn_bias ? grad_attn_bias : kept ? static_cast<float *>(scratch) : nullptr;
    args.pair_row = static_cast<int>(pair_row);
    args.wide_pairs = pair_row % 4 == 0 && aligned(args.pairs);
    args.lse = static_cast<float *>(scratch) + kept;
    args.delta = args.lse + rows;
    args.part_q = args.delta + rows;
    args.part_k = args.part_q + args.parts * values;
    args.part_v = args.part_k + args.parts * values;
    args.part_z = args.part_v + args.parts * values;
    args.part_max = args.part_z + args.parts * keys;
    args.part_total = args.part_max + args.parts * rows;
    const bool vec = head_dim % 4 == 0 && aligned(q) && aligned(k) && aligned(v) && aligned(out) && aligned(grad_out) &&
                     aligned(grad_q) && aligned(grad_k) && aligned(grad_v);
    if (head_dim <= 32) return launch_width<32>(args, vec, causal, stream);
    if (head_dim <= 64) return launch_width<64>(args, vec, causal, stream);
    if (head_dim <= 80) return launch_width<80>(args, vec, causal, stream);
    if (head_dim <= 96) return launch_width<96>(args, vec, causal, stream);
    if (head_dim <= 128) return launch_width<128>(args, vec, causal, stream);
    return launch_width<256>(args, vec, causal, stream);
}

}  // namespace sthip
