// Rotary positions: the leading values of every head turn in pairs by an angle that grows with the row's position.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "device_math.h"
#include "kernels.h"

namespace sthip {

namespace {

struct RotaryArgs {
    const void *in;
    void *out;
    const int *positions;
    long long ld_in, ld_out;
    int rows, sequence, heads, head_dim, half, rows_per_block, heads_per_block, head_blocks;  // half: pairs of a head
    bool interleaved, transposed, copies;                                        // copies: what does not turn has to be copied
    double log2_base_step;  // turns of pair i in a position, before scaling: 2^(-i * step) / 2 pi
    double by_factor, original_length, low_turns, by_turns;  // 1 / factor, 1 / (high - low)
    float magnitude;
};

constexpr int kRotaryThreads = 256;

// How often pair i turns in one position, in 64 bits: a far position multiplies it by a million, and what is left of the product
// behind its whole turns is the angle.
__device__ __forceinline__ double turns_per_position(const RotaryArgs &p, int pair)
{
    const double plain = exp2(-pair * p.log2_base_step) * 0.15915494309189535;  // 1 / 2 pi
    if (p.original_length <= 0.0) return plain * p.by_factor;
    const double kept = fmin(fmax((p.original_length * plain - p.low_turns) * p.by_turns, 0.0), 1.0);
    return plain * (kept + (1.0 - kept) * p.by_factor);
}

// cos and sin of so many turns, times the magnitude: the nearest quarter of a turn is taken off in 64 bits, and the rest is an eighth
// at the most, whose rounding to 32 bits is off by 2^-27 of a turn.
__device__ __forceinline__ float2 turned(double turns, float magnitude, bool back)
{
    const double quarter = rint(turns * 4.0);
    const float rest = static_cast<float>(turns * 4.0 - quarter) * 0.5f;  // in half turns
    float s, c;
    sincospif(rest, &s, &c);
    const int which = static_cast<int>(static_cast<long long>(quarter) & 3);
    float cosine = which & 1 ? s : c, sine = which & 1 ? c : s;
    if (which == 1 || which == 2) cosine = -cosine;
    if (which == 2 || which == 3) sine = -sine;
    return float2{cosine * magnitude, (back ? -sine : sine) * magnitude};
}


// cos and sin of the block's rows and all pairs, into LDS: (rows, pairs).
__device__ __forceinline__ void fill_table(const RotaryArgs &p, int row_first, int block_rows, float2 *table)
{
    for (int i = threadIdx.x; i < block_rows * p.half; i += kRotaryThreads) {
        const int row = row_first + i / p.half;
        const int position = p.positions ? p.positions[row] : row % p.sequence;
        table[i] = turned(position * turns_per_position(p, i % p.half), p.magnitude, p.transposed);
    }
}

// COUNT neighbouring values, up to 16 bytes, loaded and stored at once: words of two bf16 or one f32, or a single bf16.
template <typename T, int COUNT>
struct alignas(COUNT * sizeof(T)) Run {
    static constexpr int WORDS = COUNT * sizeof(T) / 4;
    std::conditional_t<WORDS == 0, uint16_t, uint32_t> word[WORDS == 0 ? 1 : WORDS];
    __device__ __forceinline__ float at(int i) const
    {
        if constexpr (sizeof(T) == 4) return __uint_as_float(word[i]);
        else if constexpr (WORDS == 0) return __uint_as_float(static_cast<uint32_t>(word[0]) << 16);
        else return __uint_as_float(i & 1 ? word[i >> 1] & 0xffff0000u : word[i >> 1] << 16);
    }
    static __device__ __forceinline__ Run of(const float (&values)[COUNT])
    {
        Run run;
        if constexpr (WORDS == 0) {
            run.word[0] = f32_to_bf16_rne(values[0]);
        } else {
#pragma unroll
            for (int i = 0; i < WORDS; ++i) {
                if constexpr (sizeof(T) == 4) run.word[i] = __float_as_uint(values[i]);
                else run.word[i] = pack_bf16x2_rne(values[2 * i], values[2 * i + 1]);
            }
        }
        return run;
    }
};

// COUNT pairs at a time: two runs half a rotary_dim apart, or beside each other.  A thread has BATCH of them at once, and loads the first
// ones before the angles are worked out.
template <typename T, int COUNT, bool INTERLEAVED, int BATCH>
__global__ __launch_bounds__(kRotaryThreads) void rotary_runs_kernel(RotaryArgs p)
{
    extern __shared__ __attribute__((aligned(16))) float2 rotary_lds[];
    const int tid = threadIdx.x, half = p.half;
    const int row_first = blockIdx.x / p.head_blocks * p.rows_per_block, block_rows = min(p.rows - row_first, p.rows_per_block);
    const int head_first = blockIdx.x % p.head_blocks * p.heads_per_block, block_heads = min(p.heads - head_first, p.heads_per_block);
    const int turning = half / COUNT, units = turning + (p.copies ? (p.head_dim - 2 * half) / COUNT : 0);
    const int total = block_rows * block_heads * units;  // (a block's share is small)
    const int second = INTERLEAVED ? COUNT : half;
    using Values = Run<T, COUNT>;
    Values x[BATCH][2];
    struct Place {
        int unit, row;
        long long head, at;  // offsets within a row, and of the first run within the head
    };
    auto place_of = [&](int i) {
        Place w;
        const int of = i / units;
        w.unit = i - of * units;
        w.row = of / block_heads;
        w.head = static_cast<long long>(head_first + of - w.row * block_heads) * p.head_dim;
        w.at = w.unit >= turning ? half + w.unit * COUNT : INTERLEAVED ? 2 * w.unit * COUNT : w.unit * COUNT;
        return w;
    };
    auto load = [&](int first) {
#pragma unroll
        for (int b = 0; b < BATCH; ++b) {
            const int i = first + b * kRotaryThreads;
            if (i < total) {
                const Place w = place_of(i);
                const T *const in = static_cast<const T *>(p.in) + (row_first + w.row) * p.ld_in + w.head + w.at;
                x[b][0] = *reinterpret_cast<const Values *>(in);
                if (w.unit < turning) x[b][1] = *reinterpret_cast<const Values *>(in + second);
            }
        }
    };
    load(tid);
    fill_table(p, row_first, block_rows, rotary_lds);
    __syncthreads();
    for (int first = tid; first < total; first += BATCH * kRotaryThreads) {
        if (first != tid) load(first);
#pragma unroll
        for (int b = 0; b < BATCH; ++b) {
            const int i = first + b * kRotaryThreads;
            if (i < total) {
                const Place w = place_of(i);
                T *const out = static_cast<T *>(p.out) + (row_first + w.row) * p.ld_out + w.head + w.at;
                Values low = x[b][0];
                if (w.unit < turning) {
                    const float2 *const by = rotary_lds + w.row * half + w.unit * COUNT;
                    float values[2][COUNT];  // in the order in which the runs hold them
#pragma unroll
                    for (int e = 0; e < COUNT; ++e) {
                        const float2 cs = by[e];
                        const int ra = INTERLEAVED ? 2 * e / COUNT : 0, ia = INTERLEAVED ? 2 * e % COUNT : e;
                        const int rb = INTERLEAVED ? (2 * e + 1) / COUNT : 1, ib = INTERLEAVED ? (2 * e + 1) % COUNT : e;
                        const float a = x[b][ra].at(ia), c = x[b][rb].at(ib);
                        values[ra][ia] = a * cs.x - c * cs.y;
                        values[rb][ib] = a * cs.y + c * cs.x;
                    }
                    low = Values::of(values[0]);
                    *reinterpret_cast<Values *>(out + second) = Values::of(values[1]);
                }
                *reinterpret_cast<Values *>(out) = low;
            }
        }
    }
}

template <typename T, int COUNT>
void launch_runs(dim3 grid, size_t table, size_t batch, const RotaryArgs &args, hipStream_t stream)
{
    if (batch == 4 && args.interleaved) rotary_runs_kernel<T, COUNT, true, 4><<<grid, kRotaryThreads, table, stream>>>(args);
    else if (batch == 4) rotary_runs_kernel<T, COUNT, false, 4><<<grid, kRotaryThreads, table, stream>>>(args);
    else if (args.interleaved) rotary_runs_kernel<T, COUNT, true, 1><<<grid, kRotaryThreads, table, stream>>>(args);
    else rotary_runs_kernel<T, COUNT, false, 1><<<grid, kRotaryThreads, table, stream>>>(args);
}

template <typename T>
hipError_t launch_rotary(size_t rows, size_t sequence, size_t heads, size_t head_dim, const st_hip_rotary &r, bool transposed,
                         const int32_t *positions, const T *in, size_t ld_in, T *out, size_t ld_out, hipStream_t stream)
{
    RotaryArgs args{};
    args.in = in;
    args.out = out;
    args.positions = positions;
    args.ld_in = static_cast<long long>(ld_in);
    args.ld_out = static_cast<long long>(ld_out);
    args.rows = static_cast<int>(rows);
    args.sequence = static_cast<int>(sequence);
    args.heads = static_cast<int>(heads);
    args.head_dim = static_cast<int>(head_dim);
    args.half = static_cast<int>(r.rotary_dim / 2);
    args.interleaved = r.interleaved != 0;
    args.transposed = transposed;
    args.copies = in != out;
    args.log2_base_step = std::log2(static_cast<double>(r.base)) / (r.rotary_dim ? args.half : 1);
    args.by_factor = 1.0 / r.factor;
    args.original_length = r.original_length;
    args.low_turns = r.low_turns;
    args.by_turns = 1.0 / (static_cast<double>(r.high_turns) - r.low_turns);
    args.magnitude = r.magnitude;
    // Runs as long as every one of them begins on a boundary of its length, up to 16 bytes.  (6815 rows of 33 bf16 heads of 80 values, 40 of
    // which turn, 8 bytes at a time: 20 us, 70 by single values.)
    const size_t together = args.half | head_dim | ld_in | ld_out | reinterpret_cast<uintptr_t>(in) / sizeof(T) | reinterpret_cast<uintptr_t>(out) / sizeof(T) | 16 / sizeof(T);
    const size_t count = together & -together;
    const size_t turning = args.half / count, copied = args.copies ? (head_dim - r.rotary_dim) / count : 0;
    const size_t units = std::max<size_t>(1, turning + copied);  // of a head
    // A block of 256 threads takes as many whole rows as give each thread a batch, or a part of a row's heads.
    const size_t batch = rows * heads * units >= size_t(1) << 19 ? 4 : 1, wanted = batch * kRotaryThreads;
    args.heads_per_block = static_cast<int>(std::max<size_t>(1, std::min(heads, wanted / units)));
    args.head_blocks = static_cast<int>((heads + args.heads_per_block - 1) / args.heads_per_block);
    args.rows_per_block = static_cast<int>(std::max<size_t>(1, std::min({rows, wanted / (units * args.heads_per_block), size_t(2048) / std::max(1, args.half)})));
    const size_t blocks = (rows + args.rows_per_block - 1) / args.rows_per_block * args.head_blocks;
    if (blocks > 0x7fffffffu) return hipErrorInvalidValue;
    const size_t table = static_cast<size_t>(args.rows_per_block) * args.half * sizeof(float2);
    const dim3 grid(static_cast<unsigned>(blocks));
    if constexpr (sizeof(T) == 2) {
        if (count == 8) launch_runs<T, 8>(grid, table, batch, args, stream);
    }
    if (count == 4) launch_runs<T, 4>(grid, table, batch, args, stream);
    if (count == 2) launch_runs<T, 2>(grid, table, batch, args, stream);
    if (count == 1) launch_runs<T, 1>(grid, table, batch, args, stream);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_rotary_f32(size_t rows, size_t sequence, size_t heads, size_t head_dim, const st_hip_rotary &rotary, bool transposed,
                             const int32_t *positions, const float *in, size_t ld_in, float *out, size_t ld_out, hipStream_t stream)
{
    return launch_rotary(rows, sequence, heads, head_dim, rotary, transposed, positions, in, ld_in, out, ld_out, stream);
}

hipError_t launch_rotary_bf16(size_t rows, size_t sequence, size_t heads, size_t head_dim, const st_hip_rotary &rotary, bool transposed,
                              const int32_t *positions, const uint16_t *in, size_t ld_in, uint16_t *out, size_t ld_out, hipStream_t stream)
{
    return launch_rotary(rows, sequence, heads, head_dim, rotary, transposed, positions, in, ld_in, out, ld_out, stream);
}

}  // namespace sthip
