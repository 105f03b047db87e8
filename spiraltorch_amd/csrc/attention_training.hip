// Attention that is trained (bf16 operands, gfx950): the forward pass with every row's log-sum-exp kept, and the backward pass, which
// works the probabilities out again from it.
//
//   s = scale·q·k + bias(key − query),  p = exp(s − lse),  o = p·v
//   dv = pᵀ·do,  dp = do·vᵀ,  δ = Σ p·dp (= do·o),  ds = p·(dp − δ),  dq = scale·ds·k,  dk = scale·dsᵀ·q,  dbias = Σ ds
//
// Every product runs on v_mfma_f32_32x32x16_bf16 with f32 sums; the softmax, p, dp − δ and ds are f32, and p and ds are rounded once to
// bf16 where they enter a product.  A wavefront owns 32 rows of the two matrices that stay (queries and their gradients, or keys and
// values) in its registers as B operands, and 64-row stages of the two that move come by through LDS: as A operands for the scores, and
// read transposed for the products behind them.  The scores then lie as a B operand lies (a lane owns one of the rows that stay), so
// that p and ds never leave the registers.
//
// The backward pass is two kernels, and nothing is added by atomics: one for dq (queries stay), which also gives δ and the bias's
// gradient, and one for dk and dv (keys stay), which walks all heads of queries that share them.  Seven products instead of five (nine
// where δ is worked out exactly), for results that do not depend on the order of workgroups, and no f32 copy of dq in memory.
//
// What bounds it: on a long sequence the matrix cores and what is issued between their instructions (8192 causal tokens, 32 heads on 8 of 128:
// forward 515 µs, 1.07 PFLOP/s of unmasked products, dq 690, 1.2, dk and dv 1075, 1.02; a large library product reaches 1.31), on shorter ones
// how full the chip is and how long a tile's loads, first products and results take (16 sequences of 1024 on 8 heads of 64: 32, 40 and 52 µs,
// of which 16 each are the bytes).
#include <algorithm>
#include <cmath>
#include <limits>
#include <type_traits>

#include "device_math.h"
#include "kernels.h"

namespace sthip {

namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int kStay = 128;  // rows of a workgroup: 32 of each of its four wavefronts
constexpr int kStage = 64;  // rows that come by at once

typedef unsigned int u32x4_t __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2_t __attribute__((ext_vector_type(2)));
typedef s16x4 __attribute__((address_space(3))) *lds_s16x4_ptr;

// The buckets of one side: bucket j begins at distance first[j]; what is behind the last one's begins nowhere.
struct Buckets {
    int count, side, far;  // of both sides; of one; from `far` on the last one
    int bidirectional;
    int first[ST_HIP_POSITION_BIAS_MOST_BUCKETS];
};

struct TrainingArgs {
    const uint16_t *q, *k, *v, *grad_out;
    const uint16_t *out_read;
    uint16_t *out, *grad_q, *grad_k, *grad_v;
    float *lse, *delta;
    const int *lengths;
    const float *table;
    float *partial;  // of the table's gradient: by distance, for every workgroup of the dq kernel
    int batch, heads, kv_heads, group, S;
    unsigned ld_q, ld_kv, ld_out, ld_grad_out, ld_grad_q, ld_grad_kv;
    int tiles, swizzle;
    int parts;          // workgroups to a tile of keys
    float *part_sums;   // of dk and dv, f32: (parts, 2, rows, kv_heads * head_dim)
    float scale;
    Buckets buckets;
};

struct Item {
    int context, tile;
};
// Workgroup -> (context, tile), `group` neighbouring contexts sharing keys: each XCD (workgroup id mod 8) keeps whole groups where they divide
// evenly, so that what comes by stays in its L2, every eighth one, so that a batch's long sequences are spread over them; under a causal
// mask the longest tiles of all its contexts run first.
__host__ __device__ inline Item decode(int groups, int group, int tiles, int swizzle, bool by_tile, bool last_first, unsigned block)
{
    const unsigned contexts = static_cast<unsigned>(groups) * group, of_xcd = swizzle ? contexts >> 3 : contexts, i = swizzle ? block >> 3 : block;
    const unsigned n = static_cast<unsigned>(tiles), tile = by_tile ? i / of_xcd : i % n, j = by_tile ? i % of_xcd : i / n;
    const unsigned context = swizzle ? (j / group * 8 + (block & 7)) * group + j % group : j;
    return Item{static_cast<int>(context), static_cast<int>(last_first ? n - 1 - tile : tile)};
}

// A 64-row stage in LDS: rows of D values as they are in memory, their 16-byte chunks swapped about so that neither kind of read meets
// itself on a bank.  Sixteen neighbouring rows' same chunk (a fragment) need sixteen places in the 256 bytes of the banks; four rows'
// 64 neighbouring bytes (half a wavefront of a transposing read) four groups of four.  Rows of 128 bytes come two to the banks' width:
// the three bits of row / 2, reversed, give both; rows of 256 bytes: the low two bits of the row above the next two.
template <int D>
struct Stage {
    static constexpr int kRow = D * 2, kBytes = kStage * kRow, kLoads = kBytes / 16 / 256;
    static __device__ __forceinline__ unsigned place(unsigned row, unsigned chunk)
    {
        const unsigned pair = row >> 1;
        const unsigned turn = D == 64 ? ((pair & 1) << 2) | (pair & 2) | ((pair >> 2) & 1) : ((row & 3) << 2) | ((row >> 2) & 3);
        return row * kRow + (chunk ^ turn) * 16;
    }
};

template <int D>
struct Reader {
    unsigned rows[D / 16], columns[D / 32][2];
    __device__ __forceinline__ explicit Reader(int lane)
    {
        const int li = lane & 31, lh = lane >> 5, i16 = lane & 15, c16 = (lane >> 4) & 1;
#pragma unroll
        for (int c = 0; c < D / 16; ++c) rows[c] = Stage<D>::place(li, 2 * c + lh);
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
            for (int hi = 0; hi < 2; ++hi)
                columns[dt][hi] = Stage<D>::place(8 * hi + 4 * lh + (i16 >> 2), dt * 4 + c16 * 2 + ((i16 & 3) >> 1)) + (i16 & 1) * 8;
    }
    // 16 values of rows 32t .. 32t + 31, as an A operand: a lane has eight of one row.
    __device__ __forceinline__ bf16x8 row_fragment(const unsigned char *m, int t, int c) const
    {
        return *reinterpret_cast<const bf16x8 *>(m + t * 32 * Stage<D>::kRow + rows[c]);
    }
    // Columns 32dt .. 32dt + 31 of 16 rows from 16j, as an A operand of the transposed matrix: a lane has eight rows of one column, those that
    // an accumulator's registers 8(j % 2) .. + 7 stand for.
    __device__ __forceinline__ bf16x8 column_fragment(const unsigned char *m, int j, int dt) const
    {
        const unsigned char *at = m + j * 16 * Stage<D>::kRow;
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)(at + columns[dt][0]));
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)(at + columns[dt][1]));
        return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
};

// Rows of a head, those from `length` on read as zeros.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_of(const uint16_t *first, unsigned ld, int length, int dim)
{
    const unsigned bytes = length > 0 ? (static_cast<unsigned>(length - 1) * ld + dim) * 2u : 0u;
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t *>(first), 0, static_cast<int>(bytes), 0x00020000);
}
__device__ __forceinline__ u32x4_t fetch8(const __amdgpu_buffer_rsrc_t &rows, unsigned ld, int row, int column)
{
    return __builtin_amdgcn_raw_buffer_load_b128(rows, (static_cast<unsigned>(row) * ld + column) * 2u, 0, 0);
}

// A matrix's stages on their way from memory straight into LDS, 16 bytes a lane: no registers, and no instructions to store them.  A wavefront's
// instruction fills 1 KiB; what lies at a place is fetched by the lane that stands for it.
typedef __attribute__((address_space(3))) void *lds_void_ptr;
template <int D>
struct Mover {
    static constexpr int kRows = 1024 / Stage<D>::kRow;  // of an instruction; those of the four wavefronts together hold every turn once or twice
    unsigned from, ld;                                   // of this lane in the first instruction, bytes; row stride, bytes
    int wave;
    __device__ __forceinline__ Mover(unsigned ld_values, int lane, int wave) : ld(ld_values * 2u), wave(wave)
    {
        constexpr int LANES = Stage<D>::kRow / 16;
        const unsigned row = wave * kRows + lane / LANES, held = Stage<D>::place(row, lane % LANES) - row * Stage<D>::kRow;  // (a turn undoes itself)
        from = row * ld + held;
    }
    __device__ __forceinline__ void load(const __amdgpu_buffer_rsrc_t &rows, int first, unsigned char *to) const
    {
#pragma unroll
        for (int i = 0; i < Stage<D>::kLoads; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rows, (lds_void_ptr)(to + (i * 4 + wave) * 1024), 16, from + (first + i * 4 * kRows) * ld, 0, 0, 0);
    }
};

// Every load has arrived.  Before a loop that works on what was loaded ahead of it: where the compiler sees such a load pending at the loop's head,
// it waits within the loop, and there for the next stage's loads as well.
__device__ __forceinline__ void wait_for_loads() { __builtin_amdgcn_s_waitcnt(0x0f70); }

__device__ __forceinline__ f32x16 mfma(bf16x8 a, bf16x8 b, f32x16 sum) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, sum, 0, 0, 0); }

// Accumulator registers 8j .. 8j + 7 as a B operand.
__device__ __forceinline__ bf16x8 packed(const f32x16 &x, int j)
{
    u32x4_t words;
#pragma unroll
    for (int e = 0; e < 4; ++e) words[e] = pack_bf16x2_rne(x[8 * j + 2 * e], x[8 * j + 2 * e + 1]);
    return __builtin_bit_cast(bf16x8, words);
}

// The accumulator register's row within its 32, for lanes 0 to 31; lanes 32 to 63 hold the fourth row behind it.
__device__ constexpr int row_of(int r) { return (r >> 2) * 8 + (r & 3); }

// Biases and sums by distance hold those of -far - 64 .. far + 64: a 32x32 block whose distances are not all beyond `far` on one side lies within.
constexpr int kMargin = 64;
__host__ __device__ inline int distances_of(int far) { return 2 * far + 2 * kMargin + 1; }

// Whether some distance of a 32x32 block, d0 - 31 .. d0 + 31, is not beyond `far`.
__device__ __forceinline__ bool near(int d0, int far) { return d0 - 31 < far && d0 + 31 > -far; }
// Where a block's distances begin among those held: those of a block beyond `far` are all the same, as they are 32 behind it.
__device__ __forceinline__ int window(int d0, int far) { return min(max(d0, -far - 32), far + 32) + far + kMargin; }

// What a key `distance` behind its query (negative: before it) is given: bias[distance + far + 64], in units of log2 e.
__device__ __forceinline__ void fill_bias(const TrainingArgs &p, int head, float *bias, int tid)
{
    const Buckets &b = p.buckets;
    for (int i = tid; i < distances_of(b.far); i += 256) {
        const int distance = min(max(i - b.far - kMargin, -b.far), b.far), m = b.bidirectional ? abs(distance) : max(-distance, 0);
        int bucket = b.bidirectional && distance > 0 ? b.side - 1 : -1;
        for (int j = 0; j < b.side; j += 16)  // sixteen at a load (a pass over a single token 39 µs; one after the other 48)
#pragma unroll
            for (int e = 0; e < 16; ++e) bucket += m >= b.first[j + e];
        bias[i] = p.table[static_cast<size_t>(bucket) * p.heads + head] * kLog2e;
    }
}

// The sequence that is taken as the `place`-th: of a padded batch of up to 64 without a causal mask, in the order of their lengths, the longest
// first, as those that begin last are what the launch waits for: a pass over 8 sequences of 90 to 1500 tokens on 12 heads of 64 takes 152 µs so
// against 178 in the order given, 16 of 200 to 512 120 against 127.  Under a causal mask the longest tiles run first anyhow (32 of 64 to 1024 on
// 8 heads: 135 sorted, 131 not).
template <bool CAUSAL>
__device__ __forceinline__ int sequence_at(const TrainingArgs &p, int place, int lane)
{
    if (CAUSAL || !p.lengths || p.batch > 64) return place;
    const int mine = lane < p.batch ? min(max(p.lengths[lane], 0), p.S) : -1;
    int before = 0;
    for (int j = 0; j < p.batch; ++j) {
        const int other = __builtin_amdgcn_readlane(mine, j);
        before += other > mine || (other == mine && j < lane);
    }
    return __ffsll(__ballot(before == place)) - 1;
}

__device__ __forceinline__ int length_of(const TrainingArgs &p, int batch) { return p.lengths ? min(max(p.lengths[batch], 0), p.S) : p.S; }

// One head's 32 rows as they left the matrix cores: a lane has its row's values 4 at a time.
template <int D>
__device__ __forceinline__ void store_row(uint16_t *row, const f32x16 (&sums)[D / 32], float by, int lh)
{
#pragma unroll
    for (int t = 0; t < D / 32; ++t)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const u32x2_t words = {pack_bf16x2_rne(sums[t][g * 4] * by, sums[t][g * 4 + 1] * by),
                                   pack_bf16x2_rne(sums[t][g * 4 + 2] * by, sums[t][g * 4 + 3] * by)};
            *reinterpret_cast<u32x2_t *>(row + t * 32 + g * 8 + lh * 4) = words;
        }
}
template <int D>
__device__ __forceinline__ void store_zeros(uint16_t *row, int lh)
{
#pragma unroll
    for (int i = 0; i < D / 8; ++i) *reinterpret_cast<u32x2_t *>(row + i * 8 + lh * 4) = u32x2_t{0u, 0u};
}

// ---- forward ------------------------------------------------------------------------------------------------------------------------
// Queries stay; stages of keys and values, two of them in LDS, come by, the next one straight into LDS while one is worked on.  The running maximum is
// moved only when a weight would pass 2^8 (p·v stays far below f32's range), so that most stages rescale nothing.  Two wavefronts a SIMD: one's
// exponentials run under the other's products.
template <int D, bool CAUSAL, bool BIAS>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 4))) void attention_training_kernel(TrainingArgs p)
{
    constexpr int KC = D / 16, DT = D / 32, BYTES = Stage<D>::kBytes;
    extern __shared__ __attribute__((aligned(16))) unsigned char training_lds[];  // [K, V][2]; bias
    float *const bias = reinterpret_cast<float *>(training_lds + 4 * BYTES);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), li = lane & 31, lh = lane >> 5;

    const Item item = decode(p.batch * p.kv_heads, p.group, p.tiles, p.swizzle, CAUSAL, CAUSAL, blockIdx.x);
    const int b = sequence_at<CAUSAL>(p, item.context / p.heads, lane), h = item.context % p.heads, q0 = item.tile * kStay, wq0 = q0 + wave * 32, my_q = wq0 + li;
    const size_t context = static_cast<size_t>(b) * p.heads + h;
    const int length = length_of(p, b);
    uint16_t *const out_row = p.out + (static_cast<size_t>(b) * p.S + my_q) * p.ld_out + static_cast<size_t>(h) * D;
    float *const lse = p.lse + context * p.S;
    if (q0 >= length) {
        if (my_q < p.S) {
            store_zeros<D>(out_row, lh);
            if (lh == 0) lse[my_q] = -INFINITY;
        }
        return;
    }
    const size_t first_q = static_cast<size_t>(b) * p.S * p.ld_q + static_cast<size_t>(h) * D;
    const size_t first_k = static_cast<size_t>(b) * p.S * p.ld_kv + static_cast<size_t>(h / p.group) * D;
    const __amdgpu_buffer_rsrc_t q_rows = rows_of(p.q + first_q, p.ld_q, length, D), k_rows = rows_of(p.k + first_k, p.ld_kv, length, D),
                                 v_rows = rows_of(p.v + first_k, p.ld_kv, length, D);
    const Reader<D> reader(lane);
    const Mover<D> mover(p.ld_kv, lane, wave);
    auto load = [&](int t) {
        unsigned char *const to = training_lds + (t & 1) * 2 * BYTES;
        mover.load(k_rows, t * kStage, to);
        mover.load(v_rows, t * kStage, to + BYTES);
    };
    load(0);
    if (BIAS) fill_bias(p, h, bias, tid);
    // Without biases the running maximum is kept in units of the product q·k; a negative scale goes into q's signs for that.
    bf16x8 qf[KC];
#pragma unroll
    for (int c = 0; c < KC; ++c) {
        u32x4_t raw = fetch8(q_rows, p.ld_q, my_q, c * 16 + lh * 8);
        if (!BIAS && p.scale < 0.0f) raw ^= 0x80008000u;
        qf[c] = __builtin_bit_cast(bf16x8, raw);
    }
    // (a scale of 0 is taken as a tiny one, so that masked scores stay -inf)
    const float by = BIAS ? p.scale * kLog2e : fmaxf(fabsf(p.scale) * kLog2e, 1e-30f);
    const float unit = BIAS ? 1.0f : by, lag = 8.0f / unit;
    f32x16 oacc[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t) oacc[t] = f32x16{};
    float run_max = -INFINITY, run_sum = 0.0f;

    auto compute = [&](auto mask_tag, const unsigned char *ks, const unsigned char *vs, int key0) {
        f32x16 s[2] = {f32x16{}, f32x16{}};
#pragma unroll
        for (int c = 0; c < KC; ++c)
#pragma unroll
            for (int t = 0; t < 2; ++t) s[t] = mfma(reader.row_fragment(ks, t, c), qf[c], s[t]);
        if (BIAS) {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const float *const of = bias + window(key0 + t * 32 - wq0, p.buckets.far) - li + 4 * lh;
#pragma unroll
                for (int r = 0; r < 16; ++r) s[t][r] = fmaf(s[t][r], by, of[row_of(r)]);
            }
        }
        float most = -INFINITY;
        if (decltype(mask_tag)::value) {
            const int last = (CAUSAL ? min(my_q, length - 1) : length - 1) - key0 - 4 * lh;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (t * 32 + row_of(r) > last) s[t][r] = -INFINITY;
        }
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) most = fmaxf(most, s[t][r]);
        most = fmaxf(most, __shfl_xor(most, 32));
        if (__any(most > run_max + lag)) {  // weights may reach 2^8 before everything is scaled anew
            const float new_max = fmaxf(run_max, most);
            const float alpha = __builtin_amdgcn_exp2f((run_max - (new_max == -INFINITY ? 0.0f : new_max)) * unit);
            run_sum *= alpha;
#pragma unroll
            for (int t = 0; t < DT; ++t)
#pragma unroll
                for (int r = 0; r < 16; ++r) oacc[t][r] *= alpha;
            run_max = new_max;
        }
        const float shift = -(run_max == -INFINITY ? 0.0f : run_max) * unit;
        float sum = 0.0f;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                s[t][r] = __builtin_amdgcn_exp2f(fmaf(s[t][r], unit, shift));
                sum += s[t][r];
            }
        run_sum += sum;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const bf16x8 pf = packed(s[j >> 1], j & 1);
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) oacc[dt] = mfma(reader.column_fragment(vs, j, dt), pf, oacc[dt]);
        }
    };

    const int key_end = CAUSAL ? min(length, q0 + kStay) : length, stages = (key_end + kStage - 1) / kStage;
    const int seen = CAUSAL ? min(length, wq0 + 32) : length, plain = (CAUSAL ? min(length, q0) : length) / kStage;
    wait_for_loads();
    __syncthreads();
    auto step = [&](auto mask_tag, int t) {
        if (t + 1 < stages) load(t + 1);
        const unsigned char *const ks = training_lds + (t & 1) * 2 * BYTES;
        if (!decltype(mask_tag)::value || t * kStage < seen) compute(mask_tag, ks, ks + BYTES, t * kStage);
        wait_for_loads();
        __syncthreads();
    };
    // Stages without masked keys in a loop of their own: where a body branches, the accumulators are copied behind its last product, and the
    // compiler makes masks of all scores in either case.
    int t = 0;
    for (; t < plain; ++t) step(std::false_type{}, t);
    for (; t < stages; ++t) step(std::true_type{}, t);
    const float total = run_sum + __shfl_xor(run_sum, 32);
    if (my_q >= p.S) return;
    const bool live = my_q < length && total > 0.0f;
    if (lh == 0) lse[my_q] = live || total != total ? (run_max * unit + __log2f(total)) * kLn2 : -INFINITY;
    if (my_q < length) store_row<D>(out_row, oacc, total > 0.0f ? 1.0f / total : total, lh);
    else store_zeros<D>(out_row, lh);
}

// ---- backward: dq, δ, the bias's gradient -------------------------------------------------------------------------------------------
// As forward, with q and do in registers: three products.  The bias's gradient is summed by distance, in f32, in bins of each wavefront in LDS, and
// written once a workgroup: 16 sequences of 200 to 512 on 12 heads of 64 with 32 buckets take 60 µs, where both products run twice for δ.
// Adds a 32×32 block's ds (a lane has query q0 + li, its registers keys key0 + row_of(r) + 4·lh), whose distances lie around d0 = key0 − q0, to
// the bins (of a wavefront, sums of ds by distance): every register's values go to the lanes that stand for their distances modulo 32, by a
// permutation of the lanes, the non-negative and the negative ones apart; then 64 distances are added at once, each by one lane.
__device__ __forceinline__ void add_by_distance(const f32x16 &ds, int d0, int far, float *bins, int lane)
{
    const int li = lane & 31, lh = lane >> 5;
    float upper = 0.0f, lower = 0.0f;  // distances li and li − 32 behind d0
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const int m = row_of(r) + 4 * lh;
        const int from = ((m - li) & 31) | (lh << 5);
        const float x = __int_as_float(__builtin_amdgcn_ds_bpermute(from * 4, __float_as_int(ds[r])));
        upper += m >= li ? x : 0.0f;
        lower += m >= li ? 0.0f : x;
    }
    upper += __shfl_xor(upper, 32);
    lower += __shfl_xor(lower, 32);
    float *const at = bins + d0 + (lh ? li - 32 : li) + far + kMargin;
    *at += lh ? lower : upper;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // the next block's lanes stand for other distances
    __builtin_amdgcn_wave_barrier();
}

// A sum over a whole row, with what each addition lost: the sums of ds by distance cancel to a small part of what is added, of a long sequence's last
// bucket above all.
struct LongSum {
    float sum = 0.0f, lost = 0.0f;
    __device__ __forceinline__ void add(float x)
    {
        const float y = x - lost, to = sum + y;
        lost = (to - sum) - y;
        sum = to;
    }
};

template <int D, bool CAUSAL, bool BIAS>
__device__ __forceinline__ void grad_q(const TrainingArgs &p, unsigned char *training_lds)  // [K, V][2]; bias; bins of four wavefronts
{
    constexpr int KC = D / 16, DT = D / 32, BYTES = Stage<D>::kBytes;
    float *const bias = reinterpret_cast<float *>(training_lds + 4 * BYTES);
    const int far = p.buckets.far, width = distances_of(far);
    float *const all_bins = bias + width;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), li = lane & 31, lh = lane >> 5;
    float *const bins = all_bins + wave * width;

    const Item item = decode(p.batch * p.kv_heads, p.group, p.tiles, p.swizzle, CAUSAL, CAUSAL, blockIdx.x);
    const int b = sequence_at<CAUSAL>(p, item.context / p.heads, lane), h = item.context % p.heads, q0 = item.tile * kStay, wq0 = q0 + wave * 32, my_q = wq0 + li;
    const size_t context = static_cast<size_t>(b) * p.heads + h;
    const int length = length_of(p, b);
    const bool to_table = BIAS && p.partial != nullptr;
    float *const partial = to_table ? p.partial + (context * p.tiles + item.tile) * width : nullptr;
    uint16_t *const grad_row = p.grad_q + (static_cast<size_t>(b) * p.S + my_q) * p.ld_grad_q + static_cast<size_t>(h) * D;
    float *const delta_row = p.delta + context * p.S + my_q;
    if (q0 >= length) {
        if (my_q < p.S) store_zeros<D>(grad_row, lh);
        if (to_table)
            for (int i = tid; i < width; i += 256) partial[i] = 0.0f;
        return;
    }
    const size_t first_q = static_cast<size_t>(b) * p.S * p.ld_q + static_cast<size_t>(h) * D;
    const size_t first_k = static_cast<size_t>(b) * p.S * p.ld_kv + static_cast<size_t>(h / p.group) * D;
    const __amdgpu_buffer_rsrc_t q_rows = rows_of(p.q + first_q, p.ld_q, length, D), k_rows = rows_of(p.k + first_k, p.ld_kv, length, D),
                                 v_rows = rows_of(p.v + first_k, p.ld_kv, length, D);
    const __amdgpu_buffer_rsrc_t g_rows =
        rows_of(p.grad_out + static_cast<size_t>(b) * p.S * p.ld_grad_out + static_cast<size_t>(h) * D, p.ld_grad_out, length, D);
    const __amdgpu_buffer_rsrc_t o_rows = rows_of(p.out_read + static_cast<size_t>(b) * p.S * p.ld_out + static_cast<size_t>(h) * D, p.ld_out, length, D);
    const Reader<D> reader(lane);
    const Mover<D> mover(p.ld_kv, lane, wave);
    auto load_stage = [&](int t) {
        unsigned char *const to = training_lds + (t & 1) * 2 * BYTES;
        mover.load(k_rows, t * kStage, to);
        mover.load(v_rows, t * kStage, to + BYTES);
    };
    load_stage(0);
    if (BIAS) {
        fill_bias(p, h, bias, tid);
        if (to_table)
            for (int i = tid; i < 4 * width; i += 256) all_bins[i] = 0.0f;
    }
    bf16x8 qf[KC], gf[KC];
    float delta = 0.0f;
#pragma unroll
    for (int c = 0; c < KC; ++c) {
        qf[c] = __builtin_bit_cast(bf16x8, fetch8(q_rows, p.ld_q, my_q, c * 16 + lh * 8));
        gf[c] = __builtin_bit_cast(bf16x8, fetch8(g_rows, p.ld_grad_out, my_q, c * 16 + lh * 8));
        const bf16x8 of = __builtin_bit_cast(bf16x8, fetch8(o_rows, p.ld_out, my_q, c * 16 + lh * 8));
#pragma unroll
        for (int e = 0; e < 8; ++e) delta = fmaf(static_cast<float>(gf[c][e]), static_cast<float>(of[e]), delta);
    }
    delta += __shfl_xor(delta, 32);
    float lse = my_q < length ? p.lse[context * p.S + my_q] : INFINITY;
    // A row without keys: every p is 0.  So is ds where there is one key, exactly: the roundings of p and dp would leave something.
    if (lse == -INFINITY || length == 1) lse = INFINITY;
    const float by = p.scale * kLog2e, shift = -lse * kLog2e;

    // A stage is two blocks of 32 keys.  Its products are dealt out in steps of one chunk, with what is read from LDS `AHEAD` steps early and
    // the other block's softmax spread over the steps: there are one or two wavefronts to a SIMD, and nothing else hides the reads' way
    // or the exponentials.
    constexpr int AHEAD = BIAS && D == 128 ? 4 : 1, STEPS = D / 16, EACH = 16 / STEPS;
    struct Block {
        f32x16 s, dp;
        float bias[BIAS ? 16 : 1];
    };
    // scores and dp of both blocks; `behind(t, step)` goes on with the first block while the second one's products run
    auto products = [&](const unsigned char *ks, const unsigned char *vs, int key0, Block (&blocks)[2], auto &&ahead, auto &&behind) {
        bf16x8 ring_k[AHEAD], ring_v[AHEAD];
        auto load = [&](int i) {
            ring_k[i % AHEAD] = reader.row_fragment(ks, i / KC, i % KC);
            ring_v[i % AHEAD] = reader.row_fragment(vs, i / KC, i % KC);
        };
        auto load_bias = [&](int t) {
            if (!BIAS) return;
            const float *const of = bias + window(key0 + t * 32 - wq0, far) - li + 4 * lh;
#pragma unroll
            for (int r = 0; r < 16; ++r) blocks[t].bias[BIAS ? r : 0] = of[row_of(r)];
        };
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) load(i);
#pragma unroll
        for (int i = 0; i < 2 * KC; ++i) {
            Block &x = blocks[i / KC];
            if (i % KC == 0) {
                x.s = f32x16{};
                x.dp = f32x16{};
                load_bias(i / KC);
            }
            x.s = mfma(ring_k[i % AHEAD], qf[i % KC], x.s);
            x.dp = mfma(ring_v[i % AHEAD], gf[i % KC], x.dp);
            if (i + AHEAD < 2 * KC) load(i + AHEAD);
            else ahead(i + AHEAD - 2 * KC);
            if (i >= KC) behind(0, i - KC);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    // p of EACH registers of a block
    auto weights = [&](auto mask_tag, Block &x, int key0, int step) {
        const int last = (CAUSAL ? min(my_q, length - 1) : length - 1) - key0 - 4 * lh;
#pragma unroll
        for (int r = step * EACH; r < (step + 1) * EACH; ++r) {
            const float score = BIAS ? fmaf(x.s[r], by, x.bias[BIAS ? r : 0]) + shift : fmaf(x.s[r], by, shift);
            const float weight = __builtin_amdgcn_exp2f(score);
            x.s[r] = decltype(mask_tag)::value && row_of(r) > last ? 0.0f : weight;
        }
    };
    const int key_end = CAUSAL ? min(length, q0 + kStay) : length, stages = (key_end + kStage - 1) / kStage;
    const int seen = CAUSAL ? min(length, wq0 + 32) : length, plain = (CAUSAL ? min(length, q0) : length) / kStage;
    auto walk = [&](auto &&body) {
        wait_for_loads();
        __syncthreads();
        auto step = [&](auto mask_tag, int t) {
            if (t + 1 < stages) load_stage(t + 1);
            const unsigned char *const ks = training_lds + (t & 1) * 2 * BYTES;
            if (!decltype(mask_tag)::value || t * kStage < seen) body(mask_tag, ks, ks + BYTES, t * kStage);
            wait_for_loads();
            __syncthreads();
        };
        int t = 0;  // (as in the forward pass)
        for (; t < plain; ++t) step(std::false_type{}, t);
        for (; t < stages; ++t) step(std::true_type{}, t);
    };
    // do·o carries the roundings of o, which are to those of ds (rounded to bf16 as well) as one to the root of the keys.  The table's gradient
    // though is f32 and adds ds over whole diagonals, and a sequence may have few keys: there δ is Σ p·dp, at the price of both products again
    // (of one stage, where the sequence is short), and over Σ p, which lse's rounding makes a little less or more than 1: so a row's ds add up to 0, and
    // nothing of that is summed over whole columns.
    if (to_table || length <= kStage) {
        LongSum delta_sum, total_sum;
        walk([&](auto mask_tag, const unsigned char *ks, const unsigned char *vs, int key0) {
            Block blocks[2];
            float of_delta = 0.0f, of_total = 0.0f;
            auto add = [&](int t, int step) {
                weights(mask_tag, blocks[t], key0 + t * 32, step);
#pragma unroll
                for (int r = step * EACH; r < (step + 1) * EACH; ++r) {
                    of_delta = fmaf(blocks[t].s[r], blocks[t].dp[r], of_delta);
                    of_total += blocks[t].s[r];
                }
            };
            products(ks, vs, key0, blocks, [](int) {}, add);
#pragma unroll
            for (int step = 0; step < STEPS; ++step) add(1, step);
            delta_sum.add(of_delta);
            total_sum.add(of_total);
        });
        delta = delta_sum.sum + __shfl_xor(delta_sum.sum, 32);
        const float total = total_sum.sum + __shfl_xor(total_sum.sum, 32);
        if (total > 0.0f) delta /= total;
        if (stages > 1) load_stage(0);
    }
    if (lh == 0 && my_q < length) *delta_row = delta;

    f32x16 dq[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t) dq[t] = f32x16{};
    LongSum before, behind;  // ds of blocks beyond `far`
    walk([&](auto mask_tag, const unsigned char *ks, const unsigned char *vs, int key0) {
        Block blocks[2];
        bf16x8 ring[AHEAD], df[2][2];
        auto load = [&](int m) { ring[m % AHEAD] = reader.column_fragment(ks, m / DT, m % DT); };
        auto grads = [&](int t, int step) {
            Block &x = blocks[t];
            weights(mask_tag, x, key0 + t * 32, step);
#pragma unroll
            for (int r = step * EACH; r < (step + 1) * EACH; ++r) x.s[r] *= x.dp[r] - delta;
            if ((step + 1) * EACH % 8 == 0) df[t][(step + 1) * EACH / 8 - 1] = packed(x.s, (step + 1) * EACH / 8 - 1);
        };
        products(ks, vs, key0, blocks, load, grads);
#pragma unroll
        for (int m = 0; m < 4 * DT; ++m) {
            dq[m % DT] = mfma(ring[m % AHEAD], df[m / (2 * DT)][m / DT % 2], dq[m % DT]);
            if (m + AHEAD < 4 * DT) load(m + AHEAD);
            if (m < 2 * DT) grads(1, m);
            __builtin_amdgcn_sched_barrier(0);
        }
        if (to_table) {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const int d0 = key0 + t * 32 - wq0;
                if (near(d0, far)) {
                    add_by_distance(blocks[t].s, d0, far, bins, lane);
                } else {
                    float sum = 0.0f;
#pragma unroll
                    for (int r = 0; r < 16; ++r) sum += blocks[t].s[r];
                    if (d0 > 0) behind.add(sum);
                    else before.add(sum);
                }
            }
        }
    });
    if (my_q < length) store_row<D>(grad_row, dq, p.scale, lh);
    else if (my_q < p.S) store_zeros<D>(grad_row, lh);
    if (to_table) {
        const float all_before = wave_sum(before.sum), all_behind = wave_sum(behind.sum);
        if (lane == 0) {
            bins[0] += all_before;
            bins[width - 1] += all_behind;
        }
        __syncthreads();
        for (int i = tid; i < width; i += 256) partial[i] = (all_bins[i] + all_bins[width + i]) + (all_bins[2 * width + i] + all_bins[3 * width + i]);
    }
}

template <int D, bool CAUSAL, bool BIAS>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(BIAS && D == 128 ? 1 : 2, 4))) void attention_grad_q_kernel(TrainingArgs p)
{
    extern __shared__ __attribute__((aligned(16))) unsigned char training_lds[];
    grad_q<D, CAUSAL, BIAS>(p, training_lds);
}

// The table's gradient: a workgroup adds the workgroups' sums for the distances of one bucket and head, in an order of its own: 5 µs, a launch and two
// rounds of loads (with four wavefronts instead of sixteen 10).
constexpr int kTableThreads = 1024;
__global__ __launch_bounds__(kTableThreads) void position_bias_grad_kernel(const float *partial, float *grad_table, int batch, int heads, int tiles, Buckets buckets)
{
    __shared__ float sums[kTableThreads / 64];
    const int bucket = blockIdx.x / heads, h = blockIdx.x % heads, far = buckets.far, width = distances_of(far);
    const bool behind = buckets.bidirectional && bucket >= buckets.side;
    const int j = behind ? bucket - buckets.side : bucket;
    // the distances' sizes: from `low` to below `high`
    int low = buckets.first[j], high = j + 1 < buckets.side ? buckets.first[j + 1] : far + kMargin + 1;
    if (behind) low = max(low, 1);  // 0 is on the other side
    int first = behind ? low : -(high - 1), last = behind ? high - 1 : -low;  // distances
    if (!buckets.bidirectional && j == 0) last = far + kMargin;  // all keys ahead
    // Threads side by side take neighbouring distances, up to sixteen, and the others further workgroups' sums.
    const int run = max(last - first + 1, 0), parts = batch * tiles;
    int wide = 1;
    while (wide < 16 && wide < run) wide *= 2;
    float sum = 0.0f;
    const int distance = threadIdx.x % wide;
    for (int part = threadIdx.x / wide; part < parts; part += kTableThreads / wide) {
        const size_t context = static_cast<size_t>(part / tiles) * heads + h;
        const float *const from = partial + (context * tiles + part % tiles) * width + first + far + kMargin;
#pragma unroll 8
        for (int d = distance; d < run; d += wide) sum += from[d];
    }
    sum = wave_sum(sum);
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        sum = 0.0f;
#pragma unroll
        for (int w = 0; w < kTableThreads / 64; ++w) sum += sums[w];
        grad_table[static_cast<size_t>(bucket) * heads + h] = sum;
    }
}

// ---- backward: dk, dv ---------------------------------------------------------------------------------------------------------------
// Keys and values stay, q and do come by: four products, and 4·D/32 accumulators, which at heads of 128 leave one wavefront a SIMD: a stage's reads
// from LDS run four steps ahead of their products then, but what neither covers shows (of 1075 µs at 8192 tokens the matrix instructions
// alone are 645, and the reads from LDS, 64 KB of a wavefront's for 64 of them, take as long).
template <int D, bool CAUSAL, bool BIAS>
__device__ __forceinline__ void grad_kv(const TrainingArgs &p, unsigned char *training_lds)  // [Q, dO][2]; [lse, δ][2]; bias
{
    constexpr int KC = D / 16, DT = D / 32, BYTES = Stage<D>::kBytes;
    float *const statistics = reinterpret_cast<float *>(training_lds + 4 * BYTES), *const bias = statistics + 4 * kStage;
    const int far = p.buckets.far;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), li = lane & 31, lh = lane >> 5;

    const Item item = decode(p.batch * p.kv_heads, 1, p.tiles * p.parts, p.swizzle, CAUSAL, false, blockIdx.x);
    const int tile = item.tile / p.parts, part = item.tile % p.parts;
    const int b = sequence_at<CAUSAL>(p, item.context / p.kv_heads, lane), kv_head = item.context % p.kv_heads, k0 = tile * kStay, wk0 = k0 + wave * 32, my_key = wk0 + li;
    const int length = length_of(p, b);
    const size_t grad_at = (static_cast<size_t>(b) * p.S + my_key) * p.ld_grad_kv + static_cast<size_t>(kv_head) * D;
    if (k0 >= length) {
        if (p.parts == 1 && my_key < p.S) {
            store_zeros<D>(p.grad_k + grad_at, lh);
            store_zeros<D>(p.grad_v + grad_at, lh);
        }
        return;
    }
    const size_t first_k = static_cast<size_t>(b) * p.S * p.ld_kv + static_cast<size_t>(kv_head) * D;
    const __amdgpu_buffer_rsrc_t k_rows = rows_of(p.k + first_k, p.ld_kv, length, D), v_rows = rows_of(p.v + first_k, p.ld_kv, length, D);
    bf16x8 kf[KC], vf[KC];
#pragma unroll
    for (int c = 0; c < KC; ++c) {
        kf[c] = __builtin_bit_cast(bf16x8, fetch8(k_rows, p.ld_kv, my_key, c * 16 + lh * 8));
        vf[c] = __builtin_bit_cast(bf16x8, fetch8(v_rows, p.ld_kv, my_key, c * 16 + lh * 8));
    }
    const Reader<D> reader(lane);
    const float by = p.scale * kLog2e;
    f32x16 dk[DT], dv[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t) {
        dk[t] = f32x16{};
        dv[t] = f32x16{};
    }
    // The stages of all heads that share the keys, one after the other; a part takes its share of them.
    const int first_stage = CAUSAL ? k0 / kStage : 0, of_head = (length + kStage - 1) / kStage - first_stage;
    const long long all = static_cast<long long>(of_head) * p.group;
    const int begin = static_cast<int>(all * part / p.parts), end = static_cast<int>(all * (part + 1) / p.parts);
    const Mover<D> mover_q(p.ld_q, lane, wave), mover_g(p.ld_grad_out, lane, wave);
    // A stage's lse and δ, a row a thread: what is made of them waits for the store, as it would wait here for the whole stage's loads.
    float statistic = 0.0f;
    int statistic_row = 0;
    auto load = [&](int head, int stage, int buffer) {
        const int first = stage * kStage;
        const __amdgpu_buffer_rsrc_t q_rows =
            rows_of(p.q + static_cast<size_t>(b) * p.S * p.ld_q + static_cast<size_t>(head) * D, p.ld_q, length, D);
        const __amdgpu_buffer_rsrc_t g_rows =
            rows_of(p.grad_out + static_cast<size_t>(b) * p.S * p.ld_grad_out + static_cast<size_t>(head) * D, p.ld_grad_out, length, D);
        const size_t of_context = (static_cast<size_t>(b) * p.heads + head) * p.S;
        unsigned char *const to = training_lds + buffer * 2 * BYTES;
        statistic_row = first + (tid & 63);
        statistic = (tid < 64 ? p.lse : p.delta)[of_context + min(statistic_row, length - 1)];
        mover_q.load(q_rows, first, to);
        mover_g.load(g_rows, first, to + BYTES);
    };
    auto store = [&](int buffer) {
        const bool within = statistic_row < length;
        const float shift = within && statistic != -INFINITY ? -statistic * kLog2e : -INFINITY;  // rows without keys: every p is 0
        if (tid < 128) statistics[buffer * 2 * kStage + tid] = tid < 64 ? shift : within ? statistic : 0.0f;
    };
    // (In steps, as in the dq kernel.)
    constexpr int AHEAD = D == 64 ? 2 : 4, STEPS = D / 16, EACH = 16 / STEPS;
    auto compute = [&](auto mask_tag, int buffer, int row0) {
        const unsigned char *const qs = training_lds + buffer * 2 * BYTES, *const gs = qs + BYTES;
        const float *const of_rows = statistics + buffer * 2 * kStage + 4 * lh;
        f32x16 s[2], dp[2];
        f32x4 shift[4], delta[4];  // of the rows of the block whose softmax is next
        float of_bias[BIAS ? 16 : 1];
        bf16x8 ring_q[AHEAD], ring_g[AHEAD], pf[2][2], df[2][2];
        auto load_rows = [&](int i) {
            ring_q[i % AHEAD] = reader.row_fragment(qs, i / KC, i % KC);
            ring_g[i % AHEAD] = reader.row_fragment(gs, i / KC, i % KC);
        };
        auto load_columns = [&](int m) {
            ring_q[m % AHEAD] = reader.column_fragment(qs, m / DT, m % DT);
            ring_g[m % AHEAD] = reader.column_fragment(gs, m / DT, m % DT);
        };
        auto load_statistics = [&](int t) {
#pragma unroll
            for (int a = 0; a < 4; ++a) {
                shift[a] = *reinterpret_cast<const f32x4 *>(of_rows + t * 32 + a * 8);
                delta[a] = *reinterpret_cast<const f32x4 *>(of_rows + kStage + t * 32 + a * 8);
            }
            if (!BIAS) return;
            const float *const of = bias + window(wk0 - row0 - t * 32, far) + li - 4 * lh - row_of(15);
#pragma unroll
            for (int r = 0; r < 16; ++r) of_bias[BIAS ? r : 0] = of[row_of(15) - row_of(r)];
        };
        auto grads = [&](int t, int step) {
            const int at = my_key - row0 - t * 32 - 4 * lh;  // the key's distance from the block's first row
#pragma unroll
            for (int r = step * EACH; r < (step + 1) * EACH; ++r) {
                const float of_row = shift[r >> 2][r & 3];
                float x = __builtin_amdgcn_exp2f(BIAS ? fmaf(s[t][r], by, of_bias[BIAS ? r : 0]) + of_row : fmaf(s[t][r], by, of_row));
                if (decltype(mask_tag)::value && at > row_of(r)) x = 0.0f;
                s[t][r] = x;
                dp[t][r] = x * (dp[t][r] - delta[r >> 2][r & 3]);
            }
            if ((step + 1) * EACH % 8 == 0) {
                const int j = (step + 1) * EACH / 8 - 1;
                pf[t][j] = packed(s[t], j);
                df[t][j] = packed(dp[t], j);
            }
        };
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) load_rows(i);
#pragma unroll
        for (int i = 0; i < 2 * KC; ++i) {
            const int t = i / KC, c = i % KC;
            if (c == 0) {
                s[t] = f32x16{};
                dp[t] = f32x16{};
            }
            if (i == KC - AHEAD) load_statistics(0);
            s[t] = mfma(ring_q[i % AHEAD], kf[c], s[t]);
            dp[t] = mfma(ring_g[i % AHEAD], vf[c], dp[t]);
            if (i + AHEAD < 2 * KC) load_rows(i + AHEAD);
            else load_columns(i + AHEAD - 2 * KC);
            if (i >= KC) grads(0, i - KC);
            __builtin_amdgcn_sched_barrier(0);
        }
        load_statistics(1);
#pragma unroll
        for (int m = 0; m < 4 * DT; ++m) {
            const int t = m / (2 * DT), j = m / DT % 2, dt = m % DT;
            dv[dt] = mfma(ring_g[m % AHEAD], pf[t][j], dv[dt]);
            dk[dt] = mfma(ring_q[m % AHEAD], df[t][j], dk[dt]);
            if (m + AHEAD < 4 * DT) load_columns(m + AHEAD);
            if (m < 2 * DT) grads(1, m);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    const int last_stage = first_stage + of_head;
    int head = 0, stage = first_stage;
    if (begin < end) {
        head = begin / of_head;
        stage = first_stage + begin % of_head;
        head += kv_head * p.group;
        load(head, stage, 0);
        if (BIAS) fill_bias(p, head, bias, tid);
        store(0);
    }
    wait_for_loads();
    __syncthreads();
    int buffer = 0;
    for (int left = end - begin; left > 0;) {
        auto step = [&](auto mask_tag) {
            const int row0 = stage * kStage;
            const bool more = --left > 0, next_head = ++stage == last_stage;
            if (next_head) {
                ++head;
                stage = first_stage;
            }
            if (more) load(head, stage, buffer ^ 1);
            if (!decltype(mask_tag)::value || row0 + kStage > wk0) compute(mask_tag, buffer, row0);
            if (BIAS && more && next_head) {  // another head's biases, when this one's have been read
                __syncthreads();
                fill_bias(p, head, bias, tid);
            }
            buffer ^= 1;
            if (more) store(buffer);
            wait_for_loads();
            __syncthreads();
            return more && !next_head;
        };
        // the stages that hold a key's own place or queries before it, then the others of the head, as in the forward pass
        bool same = true;
        while (CAUSAL && same && stage * kStage < k0 + kStay) same = step(std::true_type{});
        while (same) same = step(std::false_type{});
    }
    if (length == 1) {  // (ds, as in the dq kernel)
#pragma unroll
        for (int t = 0; t < DT; ++t) dk[t] *= 0.0f;
    }
    if (p.parts > 1) {
        if (my_key >= length) return;
        const size_t rows = static_cast<size_t>(p.batch) * p.S, width = static_cast<size_t>(p.kv_heads) * D;
        float *const to = p.part_sums + ((static_cast<size_t>(part) * 2 * rows + static_cast<size_t>(b) * p.S + my_key) * width + static_cast<size_t>(kv_head) * D);
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int d = t * 32 + g * 8 + lh * 4;
                *reinterpret_cast<f32x4 *>(to + d) = f32x4{dk[t][g * 4], dk[t][g * 4 + 1], dk[t][g * 4 + 2], dk[t][g * 4 + 3]};
                *reinterpret_cast<f32x4 *>(to + rows * width + d) = f32x4{dv[t][g * 4], dv[t][g * 4 + 1], dv[t][g * 4 + 2], dv[t][g * 4 + 3]};
            }
        return;
    }
    if (my_key < length) {
        store_row<D>(p.grad_k + grad_at, dk, p.scale, lh);
        store_row<D>(p.grad_v + grad_at, dv, 1.0f, lh);
    } else if (my_key < p.S) {
        store_zeros<D>(p.grad_k + grad_at, lh);
        store_zeros<D>(p.grad_v + grad_at, lh);
    }
}

template <int D, bool CAUSAL, bool BIAS>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(D == 64 ? 2 : 1, 4))) void attention_grad_kv_kernel(TrainingArgs p)
{
    extern __shared__ __attribute__((aligned(16))) unsigned char training_lds[];
    grad_kv<D, CAUSAL, BIAS>(p, training_lds);
}

// Sequences of one tile on heads of their own: both in one launch, as the workgroup that gave a tile's δ is the one that needs it.  A pass over
// 3 sequences of 37 tokens on 4 heads takes 13.7 µs so against 15.2 in two launches, 32 of 100 on 8 heads 24.6 against 26.2; where the card is
// full, 64 of 128 on 12 heads, both take 62 (heads of 128 values: 127 against 126).
template <int D, bool CAUSAL, bool BIAS>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(D == 64 ? 2 : 1, 4))) void attention_grad_tile_kernel(TrainingArgs p)
{
    extern __shared__ __attribute__((aligned(16))) unsigned char training_lds[];
    grad_q<D, CAUSAL, BIAS>(p, training_lds);
    __syncthreads();
    grad_kv<D, CAUSAL, BIAS>(p, training_lds);
}

// The parts of dk and dv together, four values a thread.
__global__ __launch_bounds__(256) void attention_grad_kv_parts_kernel(TrainingArgs p, int width)
{
    const size_t rows = static_cast<size_t>(p.batch) * p.S, units = rows * (width / 4);
    const bool of_v = blockIdx.y == 1;
    uint16_t *const to = of_v ? p.grad_v : p.grad_k;
    const float by = of_v ? 1.0f : p.scale;
    for (size_t i = static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x; i < units; i += static_cast<size_t>(gridDim.x) * 256) {
        const size_t row = i / (width / 4), column = i % (width / 4) * 4;
        f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
        if (static_cast<int>(row % p.S) < length_of(p, static_cast<int>(row / p.S))) {
            const float *from = p.part_sums + (of_v ? rows * width : 0) + row * width + column;
            for (int part = 0; part < p.parts; ++part, from += 2 * rows * width) sum += *reinterpret_cast<const f32x4 *>(from);
        }
        const u32x2_t words = {pack_bf16x2_rne(sum[0] * by, sum[1] * by), pack_bf16x2_rne(sum[2] * by, sum[3] * by)};
        *reinterpret_cast<u32x2_t *>(to + row * p.ld_grad_kv + column) = words;
    }
}

// ---- launches -----------------------------------------------------------------------------------------------------------------------
// The check before a launch: the grid is what the decode assumes, and its first and last workgroups lie inside.
bool grid_consistent(int groups, int group, int tiles, int parts, int swizzle, bool by_tile, bool last_first, size_t blocks, int S)
{
    const size_t contexts = static_cast<size_t>(groups) * group, of_context = static_cast<size_t>(tiles) * parts;
    if (contexts == 0 || tiles <= 0 || blocks > kMaxDim || blocks != contexts * of_context) return false;
    if (static_cast<long long>(tiles) * kStay < S || static_cast<long long>(tiles - 1) * kStay >= S || (swizzle && groups % 8 != 0)) return false;
    for (const size_t block : {static_cast<size_t>(0), blocks - 1}) {
        const Item item = decode(groups, group, tiles * parts, swizzle, by_tile, last_first, static_cast<unsigned>(block));
        if (item.context < 0 || static_cast<size_t>(item.context) >= contexts || item.tile < 0 || item.tile >= tiles * parts) return false;
    }
    return true;
}

// `group`: of the contexts that share keys, 1 where they are one.
template <class Kernel>
hipError_t launch(Kernel kernel, TrainingArgs &args, int group, int parts, bool by_tile, bool last_first, size_t lds_bytes, hipStream_t stream)
{
    const int groups = args.batch * args.kv_heads;
    args.tiles = (args.S + kStay - 1) / kStay;
    args.swizzle = groups % 8 == 0;
    const size_t blocks = static_cast<size_t>(groups) * group * args.tiles * parts;
    if (!grid_consistent(groups, group, args.tiles, parts, args.swizzle, by_tile, last_first, blocks, args.S)) return hipErrorInvalidConfiguration;
    const hipError_t rc = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds_bytes));
    if (rc != hipSuccess) return rc;
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), lds_bytes, stream, args);
    return hipGetLastError();
}

// Workgroups to a tile of keys: two rounds of the chip where one workgroup a tile would not be one, none with less than eight stages.  A pass over 2
// causal sequences of 2048 on 16 heads on 4 of 128 with 32 buckets takes 293 µs so, 443 with a workgroup to a tile, one of 2048 on 8 on 2 of 64
// 88 and 214, 4 of 512 without a mask on 16 on 4 of 128 76 and 115.
int parts_of_keys(size_t groups, size_t group, size_t sequence, size_t head_dim)
{
    const size_t tiles = groups * ((sequence + kStay - 1) / kStay), round = head_dim == 64 ? 512 : 256;
    if (tiles >= round) return 1;
    const size_t stages = (sequence + kStage - 1) / kStage * group;
    return static_cast<int>(std::max<size_t>(1, std::min({2 * round / tiles, stages / 8, static_cast<size_t>(16)})));
}

// Runs `body(d, causal, biased)` with the three as compile-time constants.
template <class Body>
hipError_t with_variant(size_t head_dim, bool causal, bool biased, Body &&body)
{
    auto by_bias = [&](auto d, auto c) { return biased ? body(d, c, std::true_type{}) : body(d, c, std::false_type{}); };
    auto by_mask = [&](auto d) { return causal ? by_bias(d, std::true_type{}) : by_bias(d, std::false_type{}); };
    return head_dim == 64 ? by_mask(std::integral_constant<int, 64>{}) : by_mask(std::integral_constant<int, 128>{});
}

TrainingArgs arguments(const st_hip_attention_training &shape, const uint16_t *q, size_t ld_q, const uint16_t *k, const uint16_t *v, size_t ld_kv,
                       size_t ld_out, float *lse)
{
    TrainingArgs args{};
    args.q = q;
    args.k = k;
    args.v = v;
    args.lse = lse;
    args.lengths = shape.lengths;
    args.batch = static_cast<int>(shape.batch);
    args.heads = static_cast<int>(shape.heads);
    args.kv_heads = static_cast<int>(shape.kv_heads);
    args.group = static_cast<int>(shape.heads / shape.kv_heads);
    args.S = static_cast<int>(shape.sequence);
    args.ld_q = static_cast<unsigned>(ld_q);
    args.ld_kv = static_cast<unsigned>(ld_kv);
    args.ld_out = static_cast<unsigned>(ld_out);
    args.scale = shape.scale;
    if (const st_hip_position_bias *bias = shape.position_bias) {
        Buckets &to = args.buckets;
        args.table = bias->table;
        to.count = static_cast<int>(bias->buckets);
        to.bidirectional = bias->bidirectional != 0;
        to.side = to.bidirectional ? to.count / 2 : to.count;
        to.far = static_cast<int>(bias->max_distance);
        const int exact = to.side / 2, steps = to.side - exact;
        // the smallest distance that reaches bucket j, in 64 bits; whole where it is within 1e-9, as where far / exact is a power of two
        int m = 0;
        for (int j = 0; j < to.side; ++j) {
            auto reached = [&](int distance) {
                if (distance < exact) return distance >= j;
                const double further = steps * std::log(static_cast<double>(distance) / exact) / std::log(static_cast<double>(to.far) / exact);
                return exact + std::floor(further + 1e-9) >= j;
            };
            while (m < to.far && !reached(m)) ++m;
            to.first[j] = m;
        }
        std::fill(to.first + to.side, to.first + ST_HIP_POSITION_BIAS_MOST_BUCKETS, std::numeric_limits<int>::max());
    }
    return args;
}

}  // namespace

hipError_t launch_attention_training_bf16(const st_hip_attention_training &shape, const uint16_t *q, size_t ld_q, const uint16_t *k, const uint16_t *v,
                                          size_t ld_kv, uint16_t *out, size_t ld_out, float *lse, hipStream_t stream)
{
    TrainingArgs args = arguments(shape, q, ld_q, k, v, ld_kv, ld_out, lse);
    args.out = out;
    const bool biased = shape.position_bias != nullptr;
    return with_variant(shape.head_dim, shape.causal != 0, biased, [&](auto d, auto causal, auto bias) {
        constexpr int D = decltype(d)::value;
        constexpr bool CAUSAL = decltype(causal)::value, BIAS = decltype(bias)::value;
        const size_t lds = 4 * Stage<D>::kBytes + (BIAS ? distances_of(args.buckets.far) * sizeof(float) : 0);
        return launch(attention_training_kernel<D, CAUSAL, BIAS>, args, args.group, 1, CAUSAL, CAUSAL, lds, stream);
    });
}

hipError_t launch_attention_backward_bf16(const st_hip_attention_training &shape, const uint16_t *q, size_t ld_q, const uint16_t *k, const uint16_t *v,
                                          size_t ld_kv, const uint16_t *out, size_t ld_out, const float *lse, const uint16_t *grad_out, size_t ld_grad_out,
                                          uint16_t *grad_q, size_t ld_grad_q, uint16_t *grad_k, uint16_t *grad_v, size_t ld_grad_kv, float *grad_table,
                                          hipStream_t stream)
{
    TrainingArgs args = arguments(shape, q, ld_q, k, v, ld_kv, ld_out, const_cast<float *>(lse));
    args.out_read = out;
    args.grad_out = grad_out;
    args.grad_q = grad_q;
    args.grad_k = grad_k;
    args.grad_v = grad_v;
    args.ld_grad_out = static_cast<unsigned>(ld_grad_out);
    args.ld_grad_q = static_cast<unsigned>(ld_grad_q);
    args.ld_grad_kv = static_cast<unsigned>(ld_grad_kv);
    const bool biased = shape.position_bias != nullptr;
    auto add_up = [&](const float *partial, size_t tiles) {
        hipLaunchKernelGGL(position_bias_grad_kernel, dim3(static_cast<unsigned>(args.buckets.count * args.heads)), dim3(kTableThreads), 0, stream, partial, grad_table,
                           args.batch, args.heads, static_cast<int>(tiles), args.buckets);
        return hipGetLastError();
    };
    const size_t contexts = shape.batch * shape.heads, tiles = (shape.sequence + kStay - 1) / kStay;
    if (contexts * tiles == 0) return add_up(nullptr, 0);
    const size_t deltas = (contexts * shape.sequence + 63) / 64 * 64;
    const size_t sums = grad_table ? contexts * tiles * distances_of(args.buckets.far) : 0;
    const size_t kv_width = shape.kv_heads * shape.head_dim, sums_padded = (sums + 63) / 64 * 64;
    args.parts = parts_of_keys(shape.batch * shape.kv_heads, args.group, shape.sequence, shape.head_dim);
    const size_t part_sums = args.parts > 1 ? args.parts * 2 * shape.batch * shape.sequence * kv_width : 0;
    void *scratch = nullptr;
    hipError_t rc = stream_workspace(stream, (deltas + sums_padded + part_sums) * sizeof(float), &scratch);
    if (rc != hipSuccess) return rc;
    args.delta = static_cast<float *>(scratch);
    args.partial = grad_table ? args.delta + deltas : nullptr;
    args.part_sums = args.delta + deltas + sums_padded;
    rc = with_variant(shape.head_dim, shape.causal != 0, biased, [&](auto d, auto causal, auto bias) {
        constexpr int D = decltype(d)::value;
        constexpr bool CAUSAL = decltype(causal)::value, BIAS = decltype(bias)::value;
        const size_t distances = BIAS ? distances_of(args.buckets.far) : 0;
        const size_t lds_q = 4 * Stage<D>::kBytes + (grad_table ? 5 : 1) * distances * sizeof(float);
        const size_t lds_kv = 4 * Stage<D>::kBytes + (4 * kStage + distances) * sizeof(float);
        if (tiles == 1 && args.group == 1 && args.parts == 1)
            return launch(attention_grad_tile_kernel<D, CAUSAL, BIAS>, args, 1, 1, CAUSAL, false, std::max(lds_q, lds_kv), stream);
        const hipError_t first = launch(attention_grad_q_kernel<D, CAUSAL, BIAS>, args, args.group, 1, CAUSAL, CAUSAL, lds_q, stream);
        if (first != hipSuccess) return first;
        return launch(attention_grad_kv_kernel<D, CAUSAL, BIAS>, args, 1, args.parts, CAUSAL, false, lds_kv, stream);
    });
    if (rc == hipSuccess && args.parts > 1) {
        const size_t units = shape.batch * shape.sequence * kv_width / 4;
        hipLaunchKernelGGL(attention_grad_kv_parts_kernel, dim3(static_cast<unsigned>(std::min<size_t>((units + 255) / 256, 4096)), 2), dim3(256), 0, stream, args,
                           static_cast<int>(kv_width));
        rc = hipGetLastError();
    }
    if (rc != hipSuccess || !grad_table) return rc;
    return add_up(args.partial, tiles);
}

}  // namespace sthip
