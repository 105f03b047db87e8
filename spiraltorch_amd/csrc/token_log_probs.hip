// Log-probabilities of given tokens, entropies and the likeliest alternatives from rows of logits, and the logits' gradient.
//
//   lse = log Σ e^x,  log p = x − lse,  H = −Σ p log p = log L − T / L  with  L = Σ e^(x−m),  T = Σ e^(x−m)·(x − m),  m = max x
//   dx = g·([x is the token's] − p) − h·p·(log p + H)   for gradients g of the token's log p and h of H
//
// Memory bounds both: the forward pass reads the logits once, with the running maximum, L and T in every thread (f32), and collects the
// likeliest alternatives on the way; the backward pass reads them once and writes once.  A value stands for itself in an integer key
// (order of the value, then the lower index), so that which alternatives are taken, and in which order, does not depend on who finds them.
#include <algorithm>
#include <cfloat>
#include <type_traits>

#include "device_math.h"
#include "kernels.h"

namespace sthip {

namespace {

constexpr int kUnroll = 4;  // 16-byte loads that a thread has on their way
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kFar = -1e30f;  // a difference beyond every exponential that is not 0, and whose products are finite

typedef unsigned int u32x4_t __attribute__((ext_vector_type(4)));
typedef unsigned long long key_t;

struct LogProbsArgs {
    const void *logits;
    const int *tokens;
    float *log_probs, *entropies, *normalizers, *top_log_probs;
    int *top_ids;
    long long ld;
    int rows, vocab, top, parts, part_size;  // a part: so many values of a row
    float *part_sums;                        // (rows, parts, 3): m, L, T
    key_t *part_keys;                        // (rows, parts, top)
};

template <typename T>
__device__ __forceinline__ float value_of(T x)
{
    if constexpr (sizeof(T) == 4) return x;
    else return __uint_as_float(static_cast<unsigned>(x) << 16);
}
// Value i of a 16-byte run.
template <typename T>
__device__ __forceinline__ float value_at(const u32x4_t &run, int i)
{
    if constexpr (sizeof(T) == 4) return __uint_as_float(run[i]);
    else return __uint_as_float(i & 1 ? run[i >> 1] & 0xffff0000u : run[i >> 1] << 16);
}

__device__ __forceinline__ key_t key_of(float x, int index)
{
    const unsigned bits = __float_as_uint(x + 0.0f);  // -0 is 0
    const unsigned ordered = bits & 0x80000000u ? ~bits : bits | 0x80000000u;
    return static_cast<key_t>(ordered) << 32 | ~static_cast<unsigned>(index);
}
__device__ __forceinline__ float value_of_key(key_t key)
{
    const unsigned ordered = static_cast<unsigned>(key >> 32);
    return __uint_as_float(ordered & 0x80000000u ? ordered & 0x7fffffffu : ~ordered);
}
__device__ __forceinline__ int index_of_key(key_t key) { return static_cast<int>(~static_cast<unsigned>(key)); }

// m, L and T of some values.  No value at all: L = 0.
struct Sums {
    float m, l, t;
    static __device__ __forceinline__ Sums none() { return Sums{-FLT_MAX, 0.0f, 0.0f}; }
    __device__ __forceinline__ void raise(float to)
    {
        if (!(to > m)) return;
        const float by = fmaxf(m - to, kFar), a = __builtin_amdgcn_exp2f(by * kLog2e);
        t = a * fmaf(by, l, t);
        l *= a;
        m = to;
    }
    __device__ __forceinline__ void add(float x)  // m is not below x
    {
        const float d = x - m, e = __builtin_amdgcn_exp2f(d * kLog2e);
        l += e;
        t = fmaf(e, fmaxf(d, kFar), t);  // (a value of -infinity adds nothing)
    }
    __device__ __forceinline__ void join(const Sums &other)
    {
        const float most = fmaxf(m, other.m);
        Sums o = other;
        raise(most);
        o.raise(most);
        l += o.l;
        t += o.t;
    }
    __device__ __forceinline__ void join_wave()
    {
#pragma unroll
        for (int by = 32; by > 0; by >>= 1) {
            Sums other;
            other.m = __shfl_xor(m, by);
            other.l = __shfl_xor(l, by);
            other.t = __shfl_xor(t, by);
            join(other);
        }
    }
};

// The best `top` of the first `count` keys, sorted, into `best`, by a group of threads: a key's place is the number of larger ones.
__device__ __forceinline__ void rank_keys(const key_t *keys, int count, int top, key_t *best, int thread, int threads)
{
    for (int i = thread; i < count; i += threads) {
        const key_t mine = keys[i];
        int place = 0;
        for (int j = 0; j < count; ++j) place += keys[j] > mine;
        if (place < top) best[place] = mine;
    }
}

template <typename T>
__device__ __forceinline__ void write_row(const LogProbsArgs &p, int row, const Sums &s)
{
    const float lse = s.l == 0.0f ? -INFINITY : s.m + __log2f(s.l) * 0.6931471805599453f;
    if (p.normalizers) p.normalizers[row] = lse;
    if (p.entropies) p.entropies[row] = s.l == 0.0f ? 0.0f : __log2f(s.l) * 0.6931471805599453f - s.t / s.l;
    if (p.log_probs) {
        const int token = p.tokens[row];
        const bool counts = token >= 0 && token < p.vocab;
        const float x = counts ? value_of(static_cast<const T *>(p.logits)[row * p.ld + token]) : 0.0f;
        p.log_probs[row] = !counts ? 0.0f : lse == -INFINITY ? -INFINITY : x - lse;
    }
}
__device__ __forceinline__ void write_top(const LogProbsArgs &p, int row, int i, key_t key, const Sums &s)
{
    const float lse = s.l == 0.0f ? -INFINITY : s.m + __log2f(s.l) * 0.6931471805599453f;
    const size_t at = static_cast<size_t>(row) * p.top + i;
    p.top_ids[at] = key ? index_of_key(key) : -1;
    p.top_log_probs[at] = !key ? NAN : lse == -INFINITY ? -INFINITY : value_of_key(key) - lse;
}

// How many keys a group of `waves` wavefronts may find in a round, `top` lanes of each with all their values at the most.
constexpr int kLaneValues(int size) { return kUnroll * 16 / size + 1; }
__host__ __device__ constexpr int keys_of_round(int waves, int size, int top) { return waves * top * kLaneValues(size); }

// WAVES wavefronts to a part of a row: all four of a workgroup, or one.
template <typename T, int WAVES, bool TOP>
__global__ __launch_bounds__(256) void token_log_probs_kernel(LogProbsArgs p)
{
    constexpr int N = 16 / sizeof(T), THREADS = WAVES * 64, GROUPS = 4 / WAVES;
    extern __shared__ __attribute__((aligned(16))) key_t log_probs_lds[];  // of every group: best [top], then keys [top + two rounds]
    __shared__ Sums wave_sums[4];
    __shared__ int counts[4];
    __shared__ key_t bounds[4];
    const int tid = threadIdx.x % THREADS, group = __builtin_amdgcn_readfirstlane(threadIdx.x / THREADS), lane = tid & 63;
    const long long item = static_cast<long long>(blockIdx.x) * GROUPS + group;
    const bool works = item < static_cast<long long>(p.rows) * p.parts;  // (all of a group, and of a workgroup of one)
    auto sync = [] {
        if (WAVES > 1) {
            __syncthreads();
        } else {
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
    };
    if (!works) return;
    const int row = static_cast<int>(item / p.parts), part = static_cast<int>(item % p.parts);
    const int from = part * p.part_size, to = min(p.vocab, from + p.part_size);
    const T *const x = static_cast<const T *>(p.logits) + row * p.ld;
    const int round = keys_of_round(WAVES, sizeof(T), p.top), held = 2 * p.top + 2 * round;
    key_t *const best = log_probs_lds + group * held, *const keys = best + p.top;
    int *const count = counts + group;
    key_t *const bound = bounds + group;
    if (TOP) {
        if (tid == 0) {
            *count = 0;
            *bound = 0;
        }
        sync();
    }
    // 16-byte runs from the first boundary within the part; what stands before and behind them is one value a thread
    const int ahead = min(to - from, static_cast<int>((16 - reinterpret_cast<uintptr_t>(x + from) % 16) % 16 / sizeof(T)));
    const int runs = (to - from - ahead) / N, first = from + ahead, edges = to - from - runs * N;
    const u32x4_t *const run_at = reinterpret_cast<const u32x4_t *>(x + first);
    Sums sums = Sums::none();
    for (int at = 0; at == 0 || at < runs; at += THREADS * kUnroll) {
        u32x4_t loaded[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const int i = at + u * THREADS + tid;
            constexpr unsigned nothing = sizeof(T) == 4 ? 0xff800000u : 0xff80ff80u;  // -infinity
            loaded[u] = i < runs ? run_at[i] : u32x4_t{nothing, nothing, nothing, nothing};
        }
        float edge = -INFINITY;
        const int edge_at = tid < ahead ? from + tid : first + runs * N + tid - ahead;
        if (at == 0 && tid < edges) edge = value_of(x[edge_at]);
        float most = edge;
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
#pragma unroll
            for (int i = 0; i < N; ++i) most = fmaxf(most, value_at<T>(loaded[u], i));
        sums.raise(most);
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
#pragma unroll
            for (int i = 0; i < N; ++i) sums.add(value_at<T>(loaded[u], i));
        if (at == 0 && tid < edges) sums.add(edge);
        if (TOP) {
            const key_t least = *bound;
            // every value this lane has in the round, with its index
            auto each = [&](auto &&of) {
                if (at == 0 && tid < edges) of(edge, edge_at);
#pragma unroll
                for (int u = 0; u < kUnroll; ++u) {
                    const int run = at + u * THREADS + tid;
                    if (run < runs) {
#pragma unroll
                        for (int i = 0; i < N; ++i) of(value_at<T>(loaded[u], i), first + run * N + i);
                    }
                }
            };
            bool may = least == 0 || most >= value_of_key(least);
            key_t mine = 0;
            if (__any(may)) {
                if (may) each([&](float v, int index) {
                    if (v == v) mine = max(mine, key_of(v, index));  // (NaN is no alternative)
                });
                may = mine > least;
                key_t lower = least + 1;
                if (__popcll(__ballot(may)) > p.top) {  // the best of more than `top` lanes: what is below the top-th of them is not among the best
                    int place = 0;
                    for (int j = 0; j < 64; ++j) {
                        const key_t other = static_cast<key_t>(__builtin_amdgcn_readlane(static_cast<int>(mine >> 32), j)) << 32 |
                                            static_cast<unsigned>(__builtin_amdgcn_readlane(static_cast<int>(mine), j));
                        place += other > mine;
                    }
                    const int which = __ffsll(__ballot(place == p.top - 1 && mine != 0)) - 1;
                    lower = static_cast<key_t>(__builtin_amdgcn_readlane(static_cast<int>(mine >> 32), which)) << 32 |
                            static_cast<unsigned>(__builtin_amdgcn_readlane(static_cast<int>(mine), which));
                    may = mine >= lower;
                }
                if (may) each([&](float v, int index) {
                    if (v != v) return;
                    const key_t key = key_of(v, index);
                    if (key >= lower) keys[atomicAdd(count, 1)] = key;
                });
            }
            sync();
            const int found = *count;
            const bool last = at + THREADS * kUnroll >= runs;
            // the first round gives a bound to begin with; later ones only where another might not fit
            if (last || at == 0 || found > p.top + round) {
                rank_keys(keys, found, p.top, best, tid, THREADS);
                sync();
                const int kept = min(found, p.top);
                for (int i = tid; i < kept; i += THREADS) keys[i] = best[i];
                if (tid == 0) {
                    *count = kept;
                    if (found >= p.top) *bound = best[p.top - 1];
                }
            }
            sync();
        }
    }
    sums.join_wave();
    if (WAVES > 1) {
        if (lane == 0) wave_sums[threadIdx.x >> 6] = sums;
        __syncthreads();
        sums = wave_sums[0];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) sums.join(wave_sums[w]);
    }
    const int kept = TOP ? *count : 0;
    if (p.parts == 1) {
        if (tid == 0) write_row<T>(p, row, sums);
        if (TOP && tid < p.top) write_top(p, row, tid, tid < kept ? best[tid] : 0, sums);
    } else {
        float *const to_sums = p.part_sums + item * 3;
        if (tid == 0) {
            to_sums[0] = sums.m;
            to_sums[1] = sums.l;
            to_sums[2] = sums.t;
        }
        if (TOP && tid < p.top) p.part_keys[item * p.top + tid] = tid < kept ? best[tid] : 0;
    }
}

// A workgroup puts a row's parts together.
constexpr int kMostParts = 64;
template <typename T>
__global__ __launch_bounds__(256) void token_log_probs_join_kernel(LogProbsArgs p)
{
    __shared__ key_t keys[kMostParts * ST_HIP_LOG_PROBS_MOST_TOP], best[ST_HIP_LOG_PROBS_MOST_TOP];
    __shared__ Sums all;
    __shared__ int count;
    const int row = blockIdx.x, tid = threadIdx.x;
    if (tid == 0) count = 0;
    if (tid < p.top) best[tid] = 0;
    __syncthreads();
    for (int i = tid; i < p.parts * p.top; i += 256) {
        const key_t key = p.part_keys[static_cast<long long>(row) * p.parts * p.top + i];
        if (key) keys[atomicAdd(&count, 1)] = key;
    }
    if (tid < 64) {
        Sums sums = Sums::none();
        if (tid < p.parts) {
            const float *const from = p.part_sums + (static_cast<long long>(row) * p.parts + tid) * 3;
            sums.m = from[0];
            sums.l = from[1];
            sums.t = from[2];
        }
        sums.join_wave();
        if (tid == 0) {
            all = sums;
            write_row<T>(p, row, sums);
        }
    }
    __syncthreads();
    rank_keys(keys, count, p.top, best, tid, 256);
    __syncthreads();
    if (tid < p.top) write_top(p, row, tid, best[tid], all);
}

// ---- backward -----------------------------------------------------------------------------------------------------------------------
struct LogProbsGradArgs {
    const void *logits;
    void *grad;
    const int *tokens;
    const float *normalizers, *entropies, *grad_log_probs, *grad_entropies;
    long long ld, ld_grad;
    int rows, vocab, parts, part_size;
};

template <typename T>
__device__ __forceinline__ T stored(float x)
{
    if constexpr (sizeof(T) == 4) return x;
    else return f32_to_bf16_rne(x);
}

template <typename T, int WAVES, bool ALIGNED>
__global__ __launch_bounds__(256) void token_log_probs_grad_kernel(LogProbsGradArgs p)
{
    constexpr int N = 16 / sizeof(T), THREADS = WAVES * 64, GROUPS = 4 / WAVES;
    const int tid = threadIdx.x % THREADS, group = __builtin_amdgcn_readfirstlane(threadIdx.x / THREADS);
    const long long item = static_cast<long long>(blockIdx.x) * GROUPS + group;
    if (item >= static_cast<long long>(p.rows) * p.parts) return;
    const int row = static_cast<int>(item / p.parts), part = static_cast<int>(item % p.parts);
    const int from = part * p.part_size, to = min(p.vocab, from + p.part_size);
    const T *const x = static_cast<const T *>(p.logits) + row * p.ld;
    T *const y = static_cast<T *>(p.grad) + row * p.ld_grad;
    const float lse = p.normalizers[row];
    int token = p.tokens ? p.tokens[row] : -1;
    if (token < 0 || token >= p.vocab || !p.grad_log_probs) token = -1;
    const float g = token >= 0 ? p.grad_log_probs[row] : 0.0f;
    const float h = p.grad_entropies ? p.grad_entropies[row] : 0.0f, entropy = p.grad_entropies ? p.entropies[row] : 0.0f;
    const bool empty = lse == -INFINITY;  // nothing has a probability
    auto gradient = [&](float v, int index) {
        const float log_p = fmaxf(v - lse, kFar), prob = __builtin_amdgcn_exp2f((v - lse) * kLog2e);
        float d = -prob * fmaf(h, log_p + entropy, g);
        if (index == token) d += g;
        return empty ? 0.0f : d;
    };
    if (!ALIGNED) {
        for (int i = from + tid; i < to; i += THREADS) y[i] = stored<T>(gradient(value_of(x[i]), i));
        return;
    }
    const int ahead = min(to - from, static_cast<int>((16 - reinterpret_cast<uintptr_t>(x + from) % 16) % 16 / sizeof(T)));
    const int runs = (to - from - ahead) / N, first = from + ahead, edges = to - from - runs * N;
    if (tid < edges) {
        const int i = tid < ahead ? from + tid : first + runs * N + tid - ahead;
        y[i] = stored<T>(gradient(value_of(x[i]), i));
    }
    const u32x4_t *const run_at = reinterpret_cast<const u32x4_t *>(x + first);
    u32x4_t *const run_to = reinterpret_cast<u32x4_t *>(y + first);
    for (int at = tid; at < runs; at += THREADS * kUnroll) {
        u32x4_t loaded[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
            if (at + u * THREADS < runs) loaded[u] = run_at[at + u * THREADS];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const int run = at + u * THREADS;
            if (run >= runs) break;
            float d[N];
#pragma unroll
            for (int i = 0; i < N; ++i) d[i] = gradient(value_at<T>(loaded[u], i), first + run * N + i);
            u32x4_t words;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                if constexpr (sizeof(T) == 4) words[w] = __float_as_uint(d[w]);
                else words[w] = pack_bf16x2_rne(d[2 * w], d[2 * w + 1]);
            }
            run_to[run] = words;
        }
    }
}

// A wavefront takes a row of up to so many bytes, a workgroup longer ones.
constexpr size_t kWaveRow = 4096;
// Rows are cut into parts where there are fewer than workgroups to fill the chip with, of 16 KiB or more.
int parts_of(size_t rows, size_t vocab, size_t size, size_t most)
{
    const size_t wanted = (512 + rows - 1) / rows, possible = vocab * size / (16u << 10);
    return static_cast<int>(std::max<size_t>(1, std::min({wanted, possible, most})));
}

template <typename T>
hipError_t launch_forward(LogProbsArgs args, hipStream_t stream)
{
    const size_t rows = args.rows, vocab = args.vocab;
    const bool wave = vocab * sizeof(T) <= kWaveRow;
    args.parts = wave ? 1 : parts_of(rows, vocab, sizeof(T), kMostParts);
    // (whole 16-byte runs, so that no two parts share one)
    args.part_size = static_cast<int>((vocab + args.parts - 1) / args.parts + 15) / 16 * 16;
    args.parts = static_cast<int>((vocab + args.part_size - 1) / args.part_size);
    const size_t items = rows * args.parts, groups = wave ? 4 : 1;
    const size_t blocks = (items + groups - 1) / groups;
    if (blocks > kMaxDim) return hipErrorInvalidConfiguration;
    if (args.parts > 1) {
        void *scratch = nullptr;
        const size_t keys = items * args.top * sizeof(key_t);
        const hipError_t rc = stream_workspace(stream, keys + items * 3 * sizeof(float), &scratch);
        if (rc != hipSuccess) return rc;
        args.part_keys = static_cast<key_t *>(scratch);
        args.part_sums = reinterpret_cast<float *>(static_cast<unsigned char *>(scratch) + keys);
    }
    const size_t lds = args.top ? groups * (2 * args.top + 2 * keys_of_round(wave ? 1 : 4, sizeof(T), args.top)) * sizeof(key_t) : 0;
    auto run = [&](auto kernel) {
        const hipError_t rc = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds));
        if (rc != hipSuccess) return rc;
        hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), lds, stream, args);
        return hipGetLastError();
    };
    hipError_t rc;
    if (wave) rc = args.top ? run(token_log_probs_kernel<T, 1, true>) : run(token_log_probs_kernel<T, 1, false>);
    else rc = args.top ? run(token_log_probs_kernel<T, 4, true>) : run(token_log_probs_kernel<T, 4, false>);
    if (rc != hipSuccess || args.parts == 1) return rc;
    hipLaunchKernelGGL(token_log_probs_join_kernel<T>, dim3(static_cast<unsigned>(rows)), dim3(256), 0, stream, args);
    return hipGetLastError();
}

template <typename T>
hipError_t launch_backward(LogProbsGradArgs args, hipStream_t stream)
{
    const size_t rows = args.rows, vocab = args.vocab;
    const bool wave = vocab * sizeof(T) <= kWaveRow;
    args.parts = wave ? 1 : parts_of(rows, vocab, sizeof(T), 4096);
    args.part_size = static_cast<int>((vocab + args.parts - 1) / args.parts + 15) / 16 * 16;
    args.parts = static_cast<int>((vocab + args.part_size - 1) / args.part_size);
    const size_t items = rows * args.parts, blocks = wave ? (items + 3) / 4 : items;
    if (blocks > kMaxDim) return hipErrorInvalidConfiguration;
    // runs of 16 bytes where every row of both begins at the same place within one
    const uintptr_t a = reinterpret_cast<uintptr_t>(args.logits), b = reinterpret_cast<uintptr_t>(args.grad);
    const bool aligned = a % 16 == b % 16 && a % sizeof(T) == 0 && (rows == 1 || (args.ld - args.ld_grad) * static_cast<long long>(sizeof(T)) % 16 == 0);
    auto run = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, stream, args);
        return hipGetLastError();
    };
    if (wave) return aligned ? run(token_log_probs_grad_kernel<T, 1, true>) : run(token_log_probs_grad_kernel<T, 1, false>);
    return aligned ? run(token_log_probs_grad_kernel<T, 4, true>) : run(token_log_probs_grad_kernel<T, 4, false>);
}

LogProbsArgs forward_arguments(size_t rows, size_t vocab, const void *logits, size_t ld, const int32_t *tokens, float *log_probs, float *entropies,
                               float *normalizers, size_t top, int32_t *top_ids, float *top_log_probs)
{
    LogProbsArgs args{};
    args.logits = logits;
    args.tokens = tokens;
    args.log_probs = log_probs;
    args.entropies = entropies;
    args.normalizers = normalizers;
    args.top_ids = top_ids;
    args.top_log_probs = top_log_probs;
    args.ld = static_cast<long long>(ld);
    args.rows = static_cast<int>(rows);
    args.vocab = static_cast<int>(vocab);
    args.top = static_cast<int>(top);
    return args;
}

}  // namespace

hipError_t launch_token_log_probs(bool bf16, size_t rows, size_t vocab, const void *logits, size_t ld, const int32_t *tokens, float *log_probs,
                                  float *entropies, float *normalizers, size_t top, int32_t *top_ids, float *top_log_probs, hipStream_t stream)
{
    const LogProbsArgs args = forward_arguments(rows, vocab, logits, ld, tokens, log_probs, entropies, normalizers, top, top_ids, top_log_probs);
    return bf16 ? launch_forward<uint16_t>(args, stream) : launch_forward<float>(args, stream);
}

hipError_t launch_token_log_probs_backward(bool bf16, size_t rows, size_t vocab, const void *logits, size_t ld, const int32_t *tokens,
                                           const float *normalizers, const float *entropies, const float *grad_log_probs, const float *grad_entropies,
                                           void *grad_logits, size_t ld_grad, hipStream_t stream)
{
    LogProbsGradArgs args{};
    args.logits = logits;
    args.grad = grad_logits;
    args.tokens = tokens;
    args.normalizers = normalizers;
    args.entropies = entropies;
    args.grad_log_probs = grad_log_probs;
    args.grad_entropies = grad_entropies;
    args.ld = static_cast<long long>(ld);
    args.ld_grad = static_cast<long long>(ld_grad);
    args.rows = static_cast<int>(rows);
    args.vocab = static_cast<int>(vocab);
    return bf16 ? launch_backward<uint16_t>(args, stream) : launch_backward<float>(args, stream);
}

}  // namespace sthip
