// Rotary positions: the leading values of every head turn in pairs by an angle that grows with the row's position.
#include <algorithm>
#include <cmath>

#include "device_math.h"
#include "kernels.h"

namespace sthip {

namespace {

struct RotaryArgs {
    const void *in;
    void *out;
    const int *positions;
    long long ld_in, ld_out;
    int rows, sequence, heads, head_dim, half, rows_per_block, heads_per_block;  // half: pairs of a head
    bool interleaved, transposed, copies;                                        // copies: what does not turn has to be copied
    double log2_base_step;  // turns of pair i in a position, before scaling: 2^(-i * step) / 2 pi
    double factor, original_length, low_turns, high_turns;
    float magnitude;
};

constexpr int kRotaryThreads = 256;

// How often pair i turns in one position, in 64 bits: a far position multiplies it by a million, and what is left of the product
// behind its whole turns is the angle.
__device__ __forceinline__ double turns_per_position(const RotaryArgs &p, int pair)
{
    const double plain = exp2(-pair * p.log2_base_step) * 0.15915494309189535;  // 1 / 2 pi
    if (p.original_length <= 0.0) return plain / p.factor;
    const double kept = fmin(fmax((p.original_length * plain - p.low_turns) / (p.high_turns - p.low_turns), 0.0), 1.0);
    return plain * (kept + (1.0 - kept) / p.factor);
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

__device__ __forceinline__ float load_one(const float *at) { return *at; }
__device__ __forceinline__ float load_one(const uint16_t *at) { return __uint_as_float(static_cast<unsigned>(*at) << 16); }
__device__ __forceinline__ void store_one(float *at, float x) { *at = x; }
__device__ __forceinline__ void store_one(uint16_t *at, float x) { *at = f32_to_bf16_rne(x); }

// One pair a thread, of any stride and alignment.
template <typename T>
__global__ __launch_bounds__(kRotaryThreads) void rotary_pairs_kernel(RotaryArgs p)
{
    extern __shared__ __attribute__((aligned(16))) float2 rotary_lds[];  // (rows, pairs)
    const int tid = threadIdx.x, half = p.half;
    const int row_first = blockIdx.x * p.rows_per_block, block_rows = min(p.rows - row_first, p.rows_per_block);
    const int head_first = blockIdx.y * p.heads_per_block, block_heads = min(p.heads - head_first, p.heads_per_block);
    for (int i = tid; i < block_rows * half; i += kRotaryThreads) {
        const int row = row_first + i / half;
        const int position = p.positions ? p.positions[row] : row % p.sequence;
        rotary_lds[i] = turned(position * turns_per_position(p, i % half), p.magnitude, p.transposed);
    }
    __syncthreads();
    const int rest = p.copies ? p.head_dim - 2 * half : 0, units = half + rest;
    const long long total = static_cast<long long>(block_rows) * block_heads * units;
    for (long long i = tid; i < total; i += kRotaryThreads) {
        const int unit = static_cast<int>(i % units);
        const long long of = i / units;
        const int head = head_first + static_cast<int>(of % block_heads), row = static_cast<int>(of / block_heads);
        const T *const in = static_cast<const T *>(p.in) + (row_first + row) * p.ld_in + static_cast<long long>(head) * p.head_dim;
        T *const out = static_cast<T *>(p.out) + (row_first + row) * p.ld_out + static_cast<long long>(head) * p.head_dim;
        if (unit >= half) {
            out[half + unit] = in[half + unit];
            continue;
        }
        const int first = p.interleaved ? 2 * unit : unit, second = p.interleaved ? first + 1 : unit + half;
        const float2 by = rotary_lds[row * half + unit];
        const float a = load_one(in + first), b = load_one(in + second);
        store_one(out + first, a * by.x - b * by.y);
        store_one(out + second, a * by.y + b * by.x);
    }
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
    args.factor = r.factor;
    args.original_length = r.original_length;
    args.low_turns = r.low_turns;
    args.high_turns = r.high_turns;
    args.magnitude = r.magnitude;
    args.rows_per_block = 4;
    args.heads_per_block = static_cast<int>(std::min<size_t>(heads, 16));
    const size_t by_rows = (rows + args.rows_per_block - 1) / args.rows_per_block, by_heads = (heads + args.heads_per_block - 1) / args.heads_per_block;
    const dim3 grid(static_cast<unsigned>(by_rows), static_cast<unsigned>(by_heads));
    rotary_pairs_kernel<T><<<grid, kRotaryThreads, static_cast<size_t>(args.rows_per_block) * args.half * sizeof(float2), stream>>>(args);
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
