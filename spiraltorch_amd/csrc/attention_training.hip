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
// gradient, and one for dk and dv (keys stay), which walks all heads of queries that share them.  Seven products instead of five, for
// results that do not depend on the order of workgroups, and no f32 copy of dq in memory.
#include <algorithm>
#include <cmath>
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

// The buckets of one side: bucket j begins at distance first[j].
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
    float scale;
    Buckets buckets;
};

struct Item {
    int context, tile;
};
// Workgroup -> (context, tile): each XCD (workgroup id mod 8) keeps whole contexts where they divide evenly, so that what comes by stays
// in its L2; under a causal mask the longest tiles of all its contexts run first.
__host__ __device__ inline Item decode(int contexts, int tiles, int swizzle, bool by_tile, bool last_first, unsigned block)
{
    const unsigned of_xcd = swizzle ? contexts >> 3 : contexts, first = swizzle ? (block & 7) * of_xcd : 0, i = swizzle ? block >> 3 : block;
    const unsigned n = static_cast<unsigned>(tiles), tile = by_tile ? i / of_xcd : i % n;
    return Item{static_cast<int>(first + (by_tile ? i % of_xcd : i / n)), static_cast<int>(last_first ? n - 1 - tile : tile)};
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

// Two matrices' stages on their way: from memory into registers, and into LDS when the stage before has been read.
template <int D>
struct Moving {
    u32x4_t a[Stage<D>::kLoads], b[Stage<D>::kLoads];
    __device__ __forceinline__ void load(const __amdgpu_buffer_rsrc_t &rows_a, unsigned ld_a, const __amdgpu_buffer_rsrc_t &rows_b, unsigned ld_b, int first,
                                         int tid)
    {
#pragma unroll
        for (int r = 0; r < Stage<D>::kLoads; ++r) {
            const int f = tid + 256 * r, row = f / (D / 8), column = f % (D / 8) * 8;
            a[r] = fetch8(rows_a, ld_a, first + row, column);
            b[r] = fetch8(rows_b, ld_b, first + row, column);
        }
    }
    __device__ __forceinline__ void store(unsigned char *to_a, unsigned char *to_b, int tid) const
    {
#pragma unroll
        for (int r = 0; r < Stage<D>::kLoads; ++r) {
            const int f = tid + 256 * r;
            const unsigned at = Stage<D>::place(f / (D / 8), f % (D / 8));
            *reinterpret_cast<u32x4_t *>(to_a + at) = a[r];
            *reinterpret_cast<u32x4_t *>(to_b + at) = b[r];
        }
    }
};

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

// What a key `distance` behind its query (negative: before it) is given, for distances of −far .. far: bias[distance + far], in units of
// log2 e.  Beyond them it is that of the ends.
__device__ __forceinline__ void fill_bias(const TrainingArgs &p, int head, float *bias, int tid)
{
    const Buckets &b = p.buckets;
    for (int i = tid; i <= 2 * b.far; i += 256) {
        const int distance = i - b.far, m = b.bidirectional ? abs(distance) : max(-distance, 0);
        int bucket = b.bidirectional && distance > 0 ? b.side : 0;
        for (int j = 1; j < b.side; ++j) bucket += m >= b.first[j];
        bias[i] = p.table[static_cast<size_t>(bucket) * p.heads + head] * kLog2e;
    }
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
template <int D, bool CAUSAL, bool BIAS>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 4))) void attention_training_kernel(TrainingArgs p)
{
    constexpr int KC = D / 16, DT = D / 32, BYTES = Stage<D>::kBytes;
    extern __shared__ __attribute__((aligned(16))) unsigned char training_lds[];  // [K, V][2]; bias
    float *const bias = reinterpret_cast<float *>(training_lds + 4 * BYTES);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), li = lane & 31, lh = lane >> 5;

    const Item item = decode(p.batch * p.heads, p.tiles, p.swizzle, CAUSAL, CAUSAL, blockIdx.x);
    const int b = item.context / p.heads, h = item.context % p.heads, q0 = item.tile * kStay, wq0 = q0 + wave * 32, my_q = wq0 + li;
    const int length = length_of(p, b);
    uint16_t *const out_row = p.out + (static_cast<size_t>(b) * p.S + my_q) * p.ld_out + static_cast<size_t>(h) * D;
    float *const lse = p.lse + static_cast<size_t>(item.context) * p.S;
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
    Moving<D> moving;
    moving.load(k_rows, p.ld_kv, v_rows, p.ld_kv, 0, tid);
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

    auto compute = [&](auto may_mask_tag, const unsigned char *ks, const unsigned char *vs, int key0) {
        constexpr bool MAY_MASK = decltype(may_mask_tag)::value;
        f32x16 s[2] = {f32x16{}, f32x16{}};
#pragma unroll
        for (int c = 0; c < KC; ++c)
#pragma unroll
            for (int t = 0; t < 2; ++t) s[t] = mfma(reader.row_fragment(ks, t, c), qf[c], s[t]);
        if (BIAS) {
            const int at = key0 - my_q + 4 * lh, far = p.buckets.far;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int r = 0; r < 16; ++r) s[t][r] = fmaf(s[t][r], by, bias[min(max(at + t * 32 + row_of(r), -far), far) + far]);
        }
        float most = -INFINITY;
        if (MAY_MASK) {
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
    const int seen = CAUSAL ? min(length, wq0 + 32) : length, plain = (CAUSAL ? min(length, wq0 + 1) : length) / kStage;
    moving.store(training_lds, training_lds + BYTES, tid);
    __syncthreads();
    int t = 0;
    for (; t < stages; ++t) {
        const bool more = t + 1 < stages;
        if (more) moving.load(k_rows, p.ld_kv, v_rows, p.ld_kv, (t + 1) * kStage, tid);
        const unsigned char *const ks = training_lds + (t & 1) * 2 * BYTES;
        if (t < plain) compute(std::false_type{}, ks, ks + BYTES, t * kStage);
        else if (t * kStage < seen) compute(std::true_type{}, ks, ks + BYTES, t * kStage);
        if (more) moving.store(training_lds + ((t + 1) & 1) * 2 * BYTES, training_lds + ((t + 1) & 1) * 2 * BYTES + BYTES, tid);
        __syncthreads();
    }
    const float total = run_sum + __shfl_xor(run_sum, 32);
    if (my_q >= p.S) return;
    const bool live = my_q < length && total > 0.0f;
    if (lh == 0) lse[my_q] = live || total != total ? (run_max * unit + __log2f(total)) * kLn2 : -INFINITY;
    if (my_q < length) store_row<D>(out_row, oacc, total > 0.0f ? 1.0f / total : total, lh);
    else store_zeros<D>(out_row, lh);
}

// ---- backward: dq, δ, the bias's gradient -------------------------------------------------------------------------------------------
// By distance: `bins` (of a wavefront) holds sums of ds for distances of −far − 64 .. far + 64.
constexpr int kBinsMargin = 64;
__host__ __device__ inline int bins_width(int far) { return 2 * far + 2 * kBinsMargin + 1; }

// Adds a 32×32 block's ds (a lane has query q0 + li, its registers keys key0 + row_of(r) + 4·lh), whose distances lie around d0 = key0 − q0, to
// the bins: every register's values go to the lanes that stand for their distances modulo 32, by a permutation of the lanes, the
// non-negative and the negative ones apart; then 64 distances are added at once, each by one lane.
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
    float *const at = bins + d0 + (lh ? li - 32 : li) + far + kBinsMargin;
    *at += lh ? lower : upper;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // the next block's lanes stand for other distances
    __builtin_amdgcn_wave_barrier();
}

template <int D, bool CAUSAL, bool BIAS>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(D == 64 ? 2 : 1, 4))) void attention_grad_q_kernel(TrainingArgs p)
{
    constexpr int KC = D / 16, DT = D / 32, BYTES = Stage<D>::kBytes;
    extern __shared__ __attribute__((aligned(16))) unsigned char training_lds[];  // [K, V][2]; bias; bins of four wavefronts
    float *const bias = reinterpret_cast<float *>(training_lds + 4 * BYTES);
    const int far = p.buckets.far, width = bins_width(far);
    float *const all_bins = bias + 2 * far + 1;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), li = lane & 31, lh = lane >> 5;
    float *const bins = all_bins + wave * width;

    const Item item = decode(p.batch * p.heads, p.tiles, p.swizzle, CAUSAL, CAUSAL, blockIdx.x);
    const int b = item.context / p.heads, h = item.context % p.heads, q0 = item.tile * kStay, wq0 = q0 + wave * 32, my_q = wq0 + li;
    const int length = length_of(p, b);
    const bool to_table = BIAS && p.partial != nullptr;
    float *const partial = to_table ? p.partial + (static_cast<size_t>(item.context) * p.tiles + item.tile) * width : nullptr;
    uint16_t *const grad_row = p.grad_q + (static_cast<size_t>(b) * p.S + my_q) * p.ld_grad_q + static_cast<size_t>(h) * D;
    float *const delta_row = p.delta + static_cast<size_t>(item.context) * p.S + my_q;
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
    Moving<D> moving;
    moving.load(k_rows, p.ld_kv, v_rows, p.ld_kv, 0, tid);
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
    float lse = my_q < length ? p.lse[static_cast<size_t>(item.context) * p.S + my_q] : INFINITY;
    if (lse == -INFINITY) lse = INFINITY;  // a row without keys: every p is 0
    const float by = p.scale * kLog2e, shift = -lse * kLog2e;

    // p of a 32-key block from its products
    auto weights = [&](auto may_mask_tag, f32x16 &s, int key0) {
        constexpr bool MAY_MASK = decltype(may_mask_tag)::value;
        const int at = key0 - my_q + 4 * lh, last = (CAUSAL ? min(my_q, length - 1) : length - 1) - key0 - 4 * lh;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            float x = fmaf(s[r], by, shift);
            if (BIAS) x += bias[min(max(at + row_of(r), -far), far) + far];
            x = __builtin_amdgcn_exp2f(x);
            if (MAY_MASK && row_of(r) > last) x = 0.0f;
            s[r] = x;
        }
    };
    auto products = [&](const unsigned char *ks, const unsigned char *vs, int t, f32x16 &s, f32x16 &dp) {
        s = f32x16{};
        dp = f32x16{};
#pragma unroll
        for (int c = 0; c < KC; ++c) {
            s = mfma(reader.row_fragment(ks, t, c), qf[c], s);
            dp = mfma(reader.row_fragment(vs, t, c), gf[c], dp);
        }
    };
    const int key_end = CAUSAL ? min(length, q0 + kStay) : length, stages = (key_end + kStage - 1) / kStage;
    const int seen = CAUSAL ? min(length, wq0 + 32) : length, plain = (CAUSAL ? min(length, wq0 + 1) : length) / kStage;
    auto walk = [&](auto &&body) {
        moving.store(training_lds, training_lds + BYTES, tid);
        __syncthreads();
        for (int t = 0; t < stages; ++t) {
            const bool more = t + 1 < stages;
            if (more) moving.load(k_rows, p.ld_kv, v_rows, p.ld_kv, (t + 1) * kStage, tid);
            const unsigned char *const ks = training_lds + (t & 1) * 2 * BYTES;
            if (t < plain) body(std::false_type{}, ks, ks + BYTES, t * kStage);
            else if (t * kStage < seen) body(std::true_type{}, ks, ks + BYTES, t * kStage);
            if (more) moving.store(training_lds + ((t + 1) & 1) * 2 * BYTES, training_lds + ((t + 1) & 1) * 2 * BYTES + BYTES, tid);
            __syncthreads();
        }
    };
    // do·o carries the roundings of o, a step of bf16 in all: little where ds is rounded to bf16 anyway, but the table's gradient is f32 and
    // adds ds over whole diagonals.  There δ is Σ p·dp, at the price of both products again.
    if (to_table) {
        delta = 0.0f;
        walk([&](auto may_mask_tag, const unsigned char *ks, const unsigned char *vs, int key0) {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                f32x16 s, dp;
                products(ks, vs, t, s, dp);
                weights(may_mask_tag, s, key0 + t * 32);
#pragma unroll
                for (int r = 0; r < 16; ++r) delta = fmaf(s[r], dp[r], delta);
            }
        });
        delta += __shfl_xor(delta, 32);
        moving.load(k_rows, p.ld_kv, v_rows, p.ld_kv, 0, tid);
    }
    if (lh == 0 && my_q < length) *delta_row = delta;

    f32x16 dq[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t) dq[t] = f32x16{};
    float before = 0.0f, behind = 0.0f;  // ds of blocks beyond `far`
    walk([&](auto may_mask_tag, const unsigned char *ks, const unsigned char *vs, int key0) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            f32x16 s, dp;
            products(ks, vs, t, s, dp);
            weights(may_mask_tag, s, key0 + t * 32);
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] *= dp[r] - delta;
            if (to_table) {
                const int d0 = key0 + t * 32 - wq0;
                if (d0 - 31 < far && d0 + 31 > -far) {
                    add_by_distance(s, d0, far, bins, lane);
                } else {
                    float sum = 0.0f;
#pragma unroll
                    for (int r = 0; r < 16; ++r) sum += s[r];
                    if (d0 > 0) behind += sum;
                    else before += sum;
                }
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const bf16x8 df = packed(s, j);
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) dq[dt] = mfma(reader.column_fragment(ks, 2 * t + j, dt), df, dq[dt]);
            }
        }
    });
    if (my_q < length) store_row<D>(grad_row, dq, p.scale, lh);
    else if (my_q < p.S) store_zeros<D>(grad_row, lh);
    if (to_table) {
        before = wave_sum(before);
        behind = wave_sum(behind);
        if (lane == 0) {
            bins[0] += before;
            bins[width - 1] += behind;
        }
        __syncthreads();
        for (int i = tid; i < width; i += 256) partial[i] = (all_bins[i] + all_bins[width + i]) + (all_bins[2 * width + i] + all_bins[3 * width + i]);
    }
}

// The table's gradient: a workgroup adds the workgroups' sums for the distances of one bucket and head, in an order of its own.
__global__ __launch_bounds__(256) void position_bias_grad_kernel(const float *partial, float *grad_table, int batch, int heads, int tiles, Buckets buckets)
{
    __shared__ float sums[4];
    const int bucket = blockIdx.x / heads, h = blockIdx.x % heads, far = buckets.far, width = bins_width(far);
    const bool behind = buckets.bidirectional && bucket >= buckets.side;
    const int j = behind ? bucket - buckets.side : bucket;
    // the distances' sizes: from `low` to below `high`
    int low = buckets.first[j], high = j + 1 < buckets.side ? buckets.first[j + 1] : far + kBinsMargin + 1;
    if (behind) low = max(low, 1);  // 0 is on the other side
    int first = behind ? low : -(high - 1), last = behind ? high - 1 : -low;  // distances
    if (!buckets.bidirectional && j == 0) last = far + kBinsMargin;  // all keys ahead
    const long long run = max(last - first + 1, 0), all = run * batch * tiles;
    float sum = 0.0f;
    for (long long i = threadIdx.x; i < all; i += 256) {
        const long long part = i / run, context = part / tiles * heads + h;
        sum += partial[(context * tiles + part % tiles) * width + first + i % run + far + kBinsMargin];
    }
    sum = wave_sum(sum);
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0) grad_table[static_cast<size_t>(bucket) * heads + h] = (sums[0] + sums[1]) + (sums[2] + sums[3]);
}

// ---- backward: dk, dv ---------------------------------------------------------------------------------------------------------------
template <int D, bool CAUSAL, bool BIAS>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(D == 64 ? 2 : 1, 4))) void attention_grad_kv_kernel(TrainingArgs p)
{
    constexpr int KC = D / 16, DT = D / 32, BYTES = Stage<D>::kBytes;
    extern __shared__ __attribute__((aligned(16))) unsigned char training_lds[];  // [Q, dO][2]; [lse, δ][2]; bias
    float *const statistics = reinterpret_cast<float *>(training_lds + 4 * BYTES), *const bias = statistics + 4 * kStage;
    const int far = p.buckets.far;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), li = lane & 31, lh = lane >> 5;

    const Item item = decode(p.batch * p.kv_heads, p.tiles, p.swizzle, CAUSAL, false, blockIdx.x);
    const int b = item.context / p.kv_heads, kv_head = item.context % p.kv_heads, k0 = item.tile * kStay, wk0 = k0 + wave * 32, my_key = wk0 + li;
    const int length = length_of(p, b);
    const size_t grad_at = (static_cast<size_t>(b) * p.S + my_key) * p.ld_grad_kv + static_cast<size_t>(kv_head) * D;
    if (k0 >= length) {
        if (my_key < p.S) {
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
    const int first_stage = CAUSAL ? k0 / kStage : 0, stages = (length + kStage - 1) / kStage;
    Moving<D> moving;
    float statistic = 0.0f;
    for (int head = kv_head * p.group; head < (kv_head + 1) * p.group; ++head) {
        const __amdgpu_buffer_rsrc_t q_rows =
            rows_of(p.q + static_cast<size_t>(b) * p.S * p.ld_q + static_cast<size_t>(head) * D, p.ld_q, length, D);
        const __amdgpu_buffer_rsrc_t g_rows =
            rows_of(p.grad_out + static_cast<size_t>(b) * p.S * p.ld_grad_out + static_cast<size_t>(head) * D, p.ld_grad_out, length, D);
        const size_t of_context = (static_cast<size_t>(b) * p.heads + head) * p.S;
        auto load = [&](int stage) {
            moving.load(q_rows, p.ld_q, g_rows, p.ld_grad_out, stage * kStage, tid);
            const int row = stage * kStage + (tid & 63);
            if (tid < 64) {
                const float lse = row < length ? p.lse[of_context + row] : INFINITY;
                statistic = lse == -INFINITY ? -INFINITY : -lse * kLog2e;  // rows without keys: every p is 0
            } else if (tid < 128) {
                statistic = row < length ? p.delta[of_context + row] : 0.0f;
            }
        };
        auto store = [&](int buffer) {
            moving.store(training_lds + buffer * 2 * BYTES, training_lds + buffer * 2 * BYTES + BYTES, tid);
            if (tid < 128) statistics[buffer * 2 * kStage + tid] = statistic;
        };
        auto compute = [&](auto may_mask_tag, int buffer, int row0) {
            constexpr bool MAY_MASK = decltype(may_mask_tag)::value;
            const unsigned char *const qs = training_lds + buffer * 2 * BYTES, *const gs = qs + BYTES;
            const float *const of_rows = statistics + buffer * 2 * kStage + 4 * lh;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                f32x16 s = f32x16{}, dp = f32x16{};
#pragma unroll
                for (int c = 0; c < KC; ++c) {
                    s = mfma(reader.row_fragment(qs, t, c), kf[c], s);
                    dp = mfma(reader.row_fragment(gs, t, c), vf[c], dp);
                }
                const int at = my_key - row0 - t * 32 - 4 * lh;  // the key's distance from row 0
#pragma unroll
                for (int a = 0; a < 4; ++a) {
                    const f32x4 shift = *reinterpret_cast<const f32x4 *>(of_rows + t * 32 + a * 8);
                    const f32x4 delta = *reinterpret_cast<const f32x4 *>(of_rows + kStage + t * 32 + a * 8);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int r = a * 4 + e;
                        float x = fmaf(s[r], by, shift[e]);
                        if (BIAS) x += bias[min(max(at - row_of(r), -far), far) + far];
                        x = __builtin_amdgcn_exp2f(x);
                        if (MAY_MASK && CAUSAL && at > row_of(r)) x = 0.0f;
                        s[r] = x;
                        dp[r] = x * (dp[r] - delta[e]);
                    }
                }
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const bf16x8 pf = packed(s, j), df = packed(dp, j);
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt) {
                        dv[dt] = mfma(reader.column_fragment(gs, 2 * t + j, dt), pf, dv[dt]);
                        dk[dt] = mfma(reader.column_fragment(qs, 2 * t + j, dt), df, dk[dt]);
                    }
                }
            }
        };
        load(first_stage);
        if (BIAS) fill_bias(p, head, bias, tid);
        store(first_stage & 1);
        __syncthreads();
        for (int t = first_stage; t < stages; ++t) {
            const bool more = t + 1 < stages;
            if (more) load(t + 1);
            const int row0 = t * kStage;
            if (!CAUSAL || row0 >= wk0 + 31) compute(std::false_type{}, t & 1, row0);
            else if (row0 + kStage > wk0) compute(std::true_type{}, t & 1, row0);
            if (more) store((t + 1) & 1);
            __syncthreads();
        }
    }
    if (my_key < length) {
        store_row<D>(p.grad_k + grad_at, dk, p.scale, lh);
        store_row<D>(p.grad_v + grad_at, dv, 1.0f, lh);
    } else if (my_key < p.S) {
        store_zeros<D>(p.grad_k + grad_at, lh);
        store_zeros<D>(p.grad_v + grad_at, lh);
    }
}

// ---- launches -----------------------------------------------------------------------------------------------------------------------
// The check before a launch: the grid is what the decode assumes, and its first and last workgroups lie inside.
bool grid_consistent(int contexts, int tiles, int swizzle, bool by_tile, bool last_first, size_t blocks, int S)
{
    if (contexts <= 0 || tiles <= 0 || blocks > kMaxDim || blocks != static_cast<size_t>(contexts) * tiles) return false;
    if (static_cast<long long>(tiles) * kStay < S || static_cast<long long>(tiles - 1) * kStay >= S || (swizzle && contexts % 8 != 0)) return false;
    for (const size_t block : {static_cast<size_t>(0), blocks - 1}) {
        const Item item = decode(contexts, tiles, swizzle, by_tile, last_first, static_cast<unsigned>(block));
        if (item.context < 0 || item.context >= contexts || item.tile < 0 || item.tile >= tiles) return false;
    }
    return true;
}

template <class Kernel>
hipError_t launch(Kernel kernel, TrainingArgs &args, int contexts, bool by_tile, bool last_first, size_t lds_bytes, hipStream_t stream)
{
    args.tiles = (args.S + kStay - 1) / kStay;
    args.swizzle = contexts % 8 == 0;
    const size_t blocks = static_cast<size_t>(contexts) * args.tiles;
    if (!grid_consistent(contexts, args.tiles, args.swizzle, by_tile, last_first, blocks, args.S)) return hipErrorInvalidConfiguration;
    const hipError_t rc = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds_bytes));
    if (rc != hipSuccess) return rc;
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), lds_bytes, stream, args);
    return hipGetLastError();
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
        const size_t lds = 4 * Stage<D>::kBytes + (BIAS ? (2 * args.buckets.far + 1) * sizeof(float) : 0);
        return launch(attention_training_kernel<D, CAUSAL, BIAS>, args, args.batch * args.heads, CAUSAL, CAUSAL, lds, stream);
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
        hipLaunchKernelGGL(position_bias_grad_kernel, dim3(static_cast<unsigned>(args.buckets.count * args.heads)), dim3(256), 0, stream, partial, grad_table,
                           args.batch, args.heads, static_cast<int>(tiles), args.buckets);
        return hipGetLastError();
    };
    const size_t contexts = shape.batch * shape.heads, tiles = (shape.sequence + kStay - 1) / kStay;
    if (contexts * tiles == 0) return add_up(nullptr, 0);
    const size_t deltas = (contexts * shape.sequence + 63) / 64 * 64;
    const size_t sums = grad_table ? contexts * tiles * bins_width(args.buckets.far) : 0;
    void *scratch = nullptr;
    hipError_t rc = stream_workspace(stream, (deltas + sums) * sizeof(float), &scratch);
    if (rc != hipSuccess) return rc;
    args.delta = static_cast<float *>(scratch);
    args.partial = grad_table ? args.delta + deltas : nullptr;
    rc = with_variant(shape.head_dim, shape.causal != 0, biased, [&](auto d, auto causal, auto bias) {
        constexpr int D = decltype(d)::value;
        constexpr bool CAUSAL = decltype(causal)::value, BIAS = decltype(bias)::value;
        const size_t distances = BIAS ? 2 * args.buckets.far + 1 : 0;
        const size_t lds_q = 4 * Stage<D>::kBytes + (distances + (grad_table ? 4 * bins_width(args.buckets.far) : 0)) * sizeof(float);
        const hipError_t first = launch(attention_grad_q_kernel<D, CAUSAL, BIAS>, args, args.batch * args.heads, CAUSAL, CAUSAL, lds_q, stream);
        if (first != hipSuccess) return first;
        const size_t lds_kv = 4 * Stage<D>::kBytes + (4 * kStage + distances) * sizeof(float);
        return launch(attention_grad_kv_kernel<D, CAUSAL, BIAS>, args, args.batch * args.kv_heads, CAUSAL, false, lds_kv, stream);
    });
    if (rc != hipSuccess || !grad_table) return rc;
    return add_up(args.partial, tiles);
}

}  // namespace sthip
