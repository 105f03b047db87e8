// Log-probabilities of given tokens, entropies and the likeliest alternatives from rows of logits, and the logits' gradient.
//
//   lse = log Σ e^x,  log p = x − lse,  H = −Σ p log p = log L − T / L  with  L = Σ e^(x−m),  T = Σ e^(x−m)·(x − m),  m = max x
//   dx = g·([x is the token's] − p) − h·p·(log p + H)   for gradients g of the token's log p and h of H
//
// Memory bounds both where there are many rows (8192 of 50001 in bf16: forward 819 MB in 199 µs, 4.1 TB/s, backward 1.64 GB in 325 µs, 5.0 TB/s;
// a copy reaches 4.9), latency where there are few (one row of 131072 with the first 20: 11.7 µs, of which 8.7 the parts and 3 putting them
// together; a workgroup that finds itself the last of its row and does that at once takes longer, 44 µs, for the fences between the
// chip's caches).  The forward pass reads the logits once, with the running maximum, L and T in every thread (f32), and collects the
// likeliest alternatives on the way; the backward pass reads them once and writes once.  A value stands for itself in an integer key
// (order of the value, then the lower index), so that which alternatives are taken, and in which order, does not depend on who finds them.
#include <algorithm>
#include <cfloat>
#include <type_traits>

#include "device_math.h"
#include "kernels.h"

namespace sthip {

namespace {

constexpr int kUnroll = 4;  // 16-byte loads that a thread of the backward pass has on their way (2 and 8 take the same where memory is what it waits for)
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
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

// m, L and T of some values; T in units of log2 e, as it is summed.  No value at all: L = 0.
struct Sums {
    float m, l, t;
    static __device__ __forceinline__ Sums none() { return Sums{-FLT_MAX, 0.0f, 0.0f}; }
    // m·log2 e is far from overflow: exponentials are taken of x·log2 e less this product as it was rounded, one multiply-add each.
    static __device__ __forceinline__ bool usual(float m) { return fabsf(m) < 1e38f; }
    static __device__ __forceinline__ float scaled(float m)
    {
#pragma clang fp contract(off)
        return m * kLog2e;
    }
    __device__ __forceinline__ void raise(float to)
    {
        if (!(to > m)) return;
        const float from = scaled(m), at = scaled(to);
        float by = (m - to) * kLog2e;
        if (usual(m) && usual(to)) {
#pragma clang fp contract(off)
            by = from - at;
        }
        by = fmaxf(by, kFar);
        const float a = __builtin_amdgcn_exp2f(by);
        t = a * fmaf(by, l, t);
        l *= a;
        m = to;
    }
    // m is not below the value.  `ordinary`: usual(m) throughout the wavefront.
    __device__ __forceinline__ void add(float x, bool ordinary)
    {
        const float d = ordinary || usual(m) ? fmaf(x, kLog2e, -scaled(m)) : (x - m) * kLog2e, e = __builtin_amdgcn_exp2f(d);
        l += e;
        t = fmaf(e, fmaxf(d, kFar), t);  // (a value of -infinity adds nothing)
    }
    __device__ __forceinline__ bool ordinary() const { return __all(usual(m)); }
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
        raise(wave_max(m));
        l = wave_sum(l);
        t = wave_sum(t);
    }
    static __device__ __forceinline__ float wave_max(float v)
    {
        const auto halves = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = fmaxf(__uint_as_float(halves[0]), __uint_as_float(halves[1]));
        const auto rows = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = fmaxf(__uint_as_float(rows[0]), __uint_as_float(rows[1]));
        auto rotated = [](float x, auto control) {
            return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), decltype(control)::value, 0xf, 0xf, true));
        };
        v = fmaxf(v, rotated(v, std::integral_constant<int, 0x128>{}));  // row_ror:8, 4, 2, 1
        v = fmaxf(v, rotated(v, std::integral_constant<int, 0x124>{}));
        v = fmaxf(v, rotated(v, std::integral_constant<int, 0x122>{}));
        return fmaxf(v, rotated(v, std::integral_constant<int, 0x121>{}));
    }
    // log Σ e^(x−m): less what scaled(m) was rounded by, which T / L has as well
    __device__ __forceinline__ float shift() const { return usual(m) ? fmaf(m, kLog2e, -scaled(m)) : 0.0f; }
    __device__ __forceinline__ float log_l() const { return (__log2f(l) - shift()) * kLn2; }
    __device__ __forceinline__ float lse() const { return l == 0.0f ? -INFINITY : m + log_l(); }
    // With the normalizer's rounding, where that is small: then log p + H, of which the gradient is made, is exact where both are nearly 0 (a likely
    // token's row: 21 rows of 3 values, two thirds of the gradient's error).
    __device__ __forceinline__ float entropy() const
    {
        if (l == 0.0f) return 0.0f;
        const float of_l = log_l(), rounding = (lse() - m) - of_l;
        return of_l - (t / l - shift()) * kLn2 + (fabsf(rounding) < 0x1p-20f ? rounding : 0.0f);
    }
};

// How many of the first `count` keys are larger.
__device__ __forceinline__ int larger_keys(const key_t *keys, int count, key_t than)
{
    int larger = 0, j = 0;
    for (; j + 8 <= count; j += 8) {  // eight reads on their way: one after the other would wait for each
        key_t other[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) other[u] = keys[j + u];
#pragma unroll
        for (int u = 0; u < 8; ++u) larger += other[u] > than;
    }
    for (; j < count; ++j) larger += keys[j] > than;
    return larger;
}
// The best `top` of the first `count` keys, sorted, into `best`, by a group of threads: a key's place is the number of larger ones.
__device__ __forceinline__ void rank_keys(const key_t *keys, int count, int top, key_t *best, int thread, int threads)
{
    for (int i = thread; i < count; i += threads) {
        const key_t mine = keys[i];
        const int place = larger_keys(keys, count, mine);
        if (place < top) best[place] = mine;
    }
}

template <typename T>
__device__ __forceinline__ void write_row(const LogProbsArgs &p, int row, const Sums &s)
{
    const float lse = s.lse();
    if (p.normalizers) p.normalizers[row] = lse;
    if (p.entropies) p.entropies[row] = s.entropy();
    if (p.log_probs) {
        const int token = p.tokens[row];
        const bool counts = token >= 0 && token < p.vocab;
        const float x = counts ? value_of(static_cast<const T *>(p.logits)[row * p.ld + token]) : 0.0f;
        p.log_probs[row] = !counts ? 0.0f : lse == -INFINITY ? -INFINITY : x - lse;
    }
}
__device__ __forceinline__ void write_top(const LogProbsArgs &p, int row, int i, key_t key, const Sums &s)
{
    const float lse = s.lse();
    const size_t at = static_cast<size_t>(row) * p.top + i;
    p.top_ids[at] = key ? index_of_key(key) : -1;
    p.top_log_probs[at] = !key ? NAN : lse == -INFINITY ? -INFINITY : value_of_key(key) - lse;
}

// What a wavefront's list has room for: the best so far and a round of `runs` 16-byte runs a lane, in which no more than `top` lanes with all their
// values (one of them from the part's edges) have anything to add.
__host__ __device__ constexpr int room_of(int runs, int size, int top) { return top + top * (runs * 16 / size + 1); }

// A number that at least `top` of the lanes' values reach, and few more: the top-th largest of them but for its last six bits, which tell equal
// ones apart here.
__device__ __forceinline__ unsigned wave_bound(unsigned ordered, int top)
{
    const unsigned mine = (ordered & ~63u) | (63u - (threadIdx.x & 63));
    int place = 0;
#pragma unroll
    for (int j = 0; j < 64; ++j) place += static_cast<unsigned>(__builtin_amdgcn_readlane(static_cast<int>(mine), j)) > mine;
    const int which = __ffsll(__ballot(place == top - 1)) - 1;
    return static_cast<unsigned>(__builtin_amdgcn_readlane(static_cast<int>(mine), which)) & ~63u;
}

// The next number below a finite one; -infinity for that and, as it comes from a bound without its last bits, for NaN.
__device__ __forceinline__ float below(float x)
{
    if (!(x > -INFINITY)) return -INFINITY;
    const float y = x + 0.0f;  // -0 is 0
    return y == 0.0f ? -1e-45f : __uint_as_float(__float_as_uint(y) + (y > 0.0f ? ~0u : 1u));
}

__device__ __forceinline__ void wave_fence()
{
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// WAVES wavefronts to a part of a row: all four of a workgroup, or one.  A round: RUNS 16-byte runs a lane, those of the next one on their way
// meanwhile.  Every wavefront keeps a list of its own of what may be among the best, and they are put together at the end.
template <typename T, int WAVES, int RUNS, bool TOP>
__global__ __launch_bounds__(256) void token_log_probs_kernel(LogProbsArgs p)
{
    constexpr int N = 16 / sizeof(T), THREADS = WAVES * 64, GROUPS = 4 / WAVES;
    extern __shared__ __attribute__((aligned(16))) key_t log_probs_lds[];  // of every wavefront: best [top], then keys
    __shared__ Sums wave_sums[4];
    __shared__ int counts[4];
    __shared__ float reached[4];  // by `top` values of a wavefront's list
    const int tid = threadIdx.x % THREADS, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = tid & 63;
    const long long item = static_cast<long long>(blockIdx.x) * GROUPS + wave / WAVES;
    if (item >= static_cast<long long>(p.rows) * p.parts) return;  // (all of a workgroup of one part)
    const int row = static_cast<int>(item / p.parts), part = static_cast<int>(item % p.parts);
    const int from = part * p.part_size, to = min(p.vocab, from + p.part_size);
    const T *const x = static_cast<const T *>(p.logits) + row * p.ld;
    const int top = p.top, room = TOP ? room_of(RUNS, sizeof(T), top) : 0;
    key_t *const best = log_probs_lds + wave * (top + room), *const keys = best + top;
    // 16-byte runs from the first boundary within the part; what stands before and behind them is one value a thread, in the first and in the
    // last round: of equal values, those of later rounds have the higher index
    const int ahead = min(to - from, static_cast<int>((16 - reinterpret_cast<uintptr_t>(x + from) % 16) % 16 / sizeof(T)));
    const int runs = (to - from - ahead) / N, first = from + ahead, behind = first + runs * N;
    const u32x4_t *const run_at = reinterpret_cast<const u32x4_t *>(x + first);
    constexpr unsigned nothing = sizeof(T) == 4 ? 0xff800000u : 0xff80ff80u;  // -infinity
    u32x4_t next[RUNS];
    auto load = [&](int at) {
#pragma unroll
        for (int u = 0; u < RUNS; ++u) {
            const int i = at + u * THREADS + tid;
            next[u] = u32x4_t{nothing, nothing, nothing, nothing};
            if (i < runs) next[u] = run_at[i];
        }
    };
    load(0);
    if (TOP && WAVES > 1) {
        if (lane == 0) reached[wave] = -INFINITY;
        __syncthreads();
    }
    const bool has_head = tid < ahead, has_tail = tid >= 8 && behind + tid - 8 < to;  // (fewer than eight of each, a lane for each)
    const float edge = has_head ? value_of(x[from + tid]) : has_tail ? value_of(x[behind + tid - 8]) : -INFINITY;
    const int edge_at = has_head ? from + tid : behind + tid - 8;
    Sums sums = Sums::none();
    int count = 0;             // of the wavefront's list
    float above = -INFINITY;   // what is not above it is not among the best
    for (int at = 0; at == 0 || at < runs; at += THREADS * RUNS) {
        u32x4_t loaded[RUNS];
#pragma unroll
        for (int u = 0; u < RUNS; ++u) loaded[u] = next[u];
        const bool begins = at == 0, ends = at + THREADS * RUNS >= runs;
        if (!ends) load(at + THREADS * RUNS);
        const bool has_edge = (begins && has_head) || (ends && has_tail);
        float most = has_edge ? fmaxf(edge, -INFINITY) : -INFINITY;  // (never NaN)
#pragma unroll
        for (int u = 0; u < RUNS; ++u)
#pragma unroll
            for (int i = 0; i < N; ++i) most = fmaxf(most, value_at<T>(loaded[u], i));
        sums.raise(most);
        auto add_all = [&](bool ordinary) {
#pragma unroll
            for (int u = 0; u < RUNS; ++u)
#pragma unroll
                for (int i = 0; i < N; ++i) sums.add(value_at<T>(loaded[u], i), ordinary);
        };
        if (sums.ordinary()) add_all(true);
        else add_all(false);
        if (has_edge) sums.add(edge, false);
        if (TOP) {
            // every value this lane has in the round, with its index
            auto each = [&](auto &&of) {
                if (has_edge) of(edge, edge_at);
#pragma unroll
                for (int u = 0; u < RUNS; ++u) {
                    const int run = at + u * THREADS + tid;
                    if (run < runs) {
#pragma unroll
                        for (int i = 0; i < N; ++i) of(value_at<T>(loaded[u], i), first + run * N + i);
                    }
                }
            };
            auto compact = [&] {
                rank_keys(keys, count, top, best, lane, 64);
                wave_fence();
                count = min(count, top);
                if (lane < count) keys[lane] = best[lane];
                if (count == top) {
                    above = value_of_key(best[top - 1]);  // equal ones to come have a higher index
                    if (WAVES > 1 && lane == 0) __hip_atomic_store(&reached[wave], above, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
                }
                wave_fence();
            };
            if (begins) {
                above = below(value_of_key(static_cast<key_t>(wave_bound(static_cast<unsigned>(key_of(most, 0) >> 32), top)) << 32));
            } else if (WAVES > 1) {  // what `top` values of another wavefront reach; equal ones here may have a lower index than those
#pragma unroll
                for (int w = 0; w < WAVES; ++w)
                    above = fmaxf(above, below(__hip_atomic_load(&reached[w], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP)));
            }
            // (-infinity: everything but NaN may be among the best, -infinity too)
            if (__any(most > above) || above == -INFINITY) {
                // How many values the lane adds, as many as there is room for; where many reach the bound and are equal, below the top-th of
                // the lanes' best keys is nothing to add.
                key_t lower = 0;
                bool by_key = above == -INFINITY;
                auto found = [&] {
                    unsigned n = 0;
                    if (by_key) {
                        each([&](float v, int index) { n += v >= above && key_of(v, index) >= lower; });
                    } else {  // (lanes without a run have -infinity in its place)
                        n += has_edge && edge > above;
#pragma unroll
                        for (int u = 0; u < RUNS; ++u)
#pragma unroll
                            for (int i = 0; i < N; ++i) n += value_at<T>(loaded[u], i) > above;
                    }
                    return n;
                };
                unsigned mine = 0, up_to = 0;
                int all = 0;
                auto rank = [&] {
                    mine = found();
                    up_to = wave_scan(mine, [](unsigned a, unsigned b) { return a + b; });
                    all = __builtin_amdgcn_readlane(static_cast<int>(up_to), 63);
                };
                rank();
                if (count + all > room && count > top) {
                    compact();
                    by_key = above == -INFINITY;
                    rank();
                }
                if (count + all > room) {
                    key_t highest = 0;
                    each([&](float v, int index) {
                        if (by_key ? v >= above : v > above) highest = max(highest, key_of(v, index));
                    });
                    int place = 0;
                    for (int j = 0; j < 64; ++j) {
                        const key_t other =
                            static_cast<key_t>(static_cast<unsigned>(__builtin_amdgcn_readlane(static_cast<int>(highest >> 32), j))) << 32 |
                            static_cast<unsigned>(__builtin_amdgcn_readlane(static_cast<int>(highest), j));
                        place += other > highest;
                    }
                    // (more than `top` lanes have some, or they would have room)
                    const int which = __ffsll(__ballot(place == top - 1)) - 1;
                    lower = static_cast<key_t>(static_cast<unsigned>(__builtin_amdgcn_readlane(static_cast<int>(highest >> 32), which))) << 32 |
                            static_cast<unsigned>(__builtin_amdgcn_readlane(static_cast<int>(highest), which));
                    by_key = true;
                    rank();
                }
                int place = count + static_cast<int>(up_to - mine);
                if (mine) {
                    if (by_key) each([&](float v, int index) {
                        if (v >= above && key_of(v, index) >= lower) keys[place++] = key_of(v, index);
                    });
                    else each([&](float v, int index) {
                        if (v > above) keys[place++] = key_of(v, index);
                    });
                }
                count += all;
                wave_fence();
                // a first bound of its own, and a better one when the list has grown
                if (count > 2 * top + 32 || (begins && !ends)) compact();
            }
        }
    }
    sums.join_wave();
    if (WAVES == 1) {
        if (TOP) {
            rank_keys(keys, count, top, best, lane, 64);
            wave_fence();
        }
    } else {
        if (lane == 0) {
            wave_sums[wave] = sums;
            counts[wave] = count;
        }
        __syncthreads();
        sums = wave_sums[0];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) sums.join(wave_sums[w]);
        if (TOP) {
            key_t *const list = log_probs_lds + top;
            for (int i = lane; i < counts[wave]; i += 64) {  // a wavefront's keys among everyone's
                const key_t mine = keys[i];
                int place = 0;
                for (int w = 0; w < WAVES; ++w) place += larger_keys(list + w * (top + room), counts[w], mine);
                if (place < top) log_probs_lds[place] = mine;  // the first wavefront's `best`
            }
            count = 0;
            for (int w = 0; w < WAVES; ++w) count += counts[w];
            __syncthreads();
        }
    }
    const key_t *const sorted = WAVES == 1 ? best : log_probs_lds;
    if (p.parts == 1) {
        if (tid == 0) write_row<T>(p, row, sums);
        if (TOP && tid < top) write_top(p, row, tid, tid < count ? sorted[tid] : 0, sums);
    } else {
        float *const to_sums = p.part_sums + item * 3;
        if (tid == 0) {
            to_sums[0] = sums.m;
            to_sums[1] = sums.l;
            to_sums[2] = sums.t;
        }
        if (TOP && tid < top) p.part_keys[item * top + tid] = tid < count ? sorted[tid] : 0;
    }
}

// A workgroup puts a row's parts together.
constexpr int kMostParts = 64;
template <typename T>
__global__ __launch_bounds__(256) void token_log_probs_join_kernel(LogProbsArgs p)
{
    constexpr int KEYS = kMostParts * ST_HIP_LOG_PROBS_MOST_TOP / 256;  // of a thread
    __shared__ key_t keys[KEYS * 256], best[ST_HIP_LOG_PROBS_MOST_TOP];
    __shared__ Sums all;
    __shared__ int count;
    __shared__ unsigned least;
    const int row = blockIdx.x, tid = threadIdx.x, found = p.parts * p.top;
    const key_t *const part_keys = p.part_keys + static_cast<long long>(row) * found;
    // everything that is read, on its way at once
    key_t mine[KEYS];
#pragma unroll
    for (int i = 0; i < KEYS; ++i) mine[i] = i * 256 + tid < found ? part_keys[i * 256 + tid] : 0;
    // A number that at least `top` keys reach: the top-th largest of the parts' first ones, or, of few parts, the least of their r-th ones with
    // parts * r not below top.
    const int rank = p.parts >= p.top ? 0 : (p.top + p.parts - 1) / p.parts - 1;
    const unsigned of_part = tid < p.parts && p.top ? static_cast<unsigned>(part_keys[tid * p.top + rank] >> 32) : 0;
    Sums sums = Sums::none();
    if (tid < p.parts) {
        const float *const from = p.part_sums + (static_cast<long long>(row) * p.parts + tid) * 3;
        sums = Sums{from[0], from[1], from[2]};
    }
    if (tid < p.top) best[tid] = 0;
    if (tid < 64) {
        sums.join_wave();
        unsigned bound = 0;
        if (p.top && rank == 0) {
            bound = wave_bound(of_part, p.top);
        } else if (p.top) {
            bound = tid < p.parts ? of_part : ~0u;
#pragma unroll
            for (int by = 32; by > 0; by >>= 1) bound = min(bound, static_cast<unsigned>(__shfl_xor(static_cast<int>(bound), by)));
        }
        if (tid == 0) {
            all = sums;
            least = bound;
            count = 0;
        }
    }
    __syncthreads();
    const unsigned from = least;
#pragma unroll
    for (int i = 0; i < KEYS; ++i)
        if (mine[i] && static_cast<unsigned>(mine[i] >> 32) >= from) keys[atomicAdd(&count, 1)] = mine[i];
    if (tid == 0) write_row<T>(p, row, sums);
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
        // (g − g·p rounded once: a likely token's is a small part of g)
        const float of_token = fmaf(-prob, g, index == token ? g : 0.0f), d = fmaf(-prob, h * (log_p + entropy), of_token);
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

// A wavefront takes a row of up to so many bytes, a workgroup longer ones: 16384 rows of 256 f32 take a wavefront each 6.4 µs forward and 7.7 backward, a
// workgroup each 20 and 16; of 1000 12.5 and 21.1, against 20.8 and 21.7; from 8 KB on both take the same.
constexpr size_t kWaveRow = 4096;
// Rows are cut into parts of 8 KiB (two runs a thread) or more, enough for so many workgroups.
int parts_of(size_t rows, size_t vocab, size_t size, size_t workgroups, size_t most)
{
    const size_t wanted = (workgroups + rows - 1) / rows, possible = vocab * size / (8u << 10);
    return static_cast<int>(std::max<size_t>(1, std::min({wanted, possible, most})));
}

template <typename T>
hipError_t launch_forward(LogProbsArgs args, hipStream_t stream)
{
    const size_t rows = args.rows, vocab = args.vocab;
    const bool wave = vocab * sizeof(T) <= kWaveRow;
    // Lists of the likeliest keep a workgroup busy: four of them to a compute unit (64 rows of 100001 in f32 with the first 5: 16.0 µs; two 17.4, one
    // 22.5, whole rows 45.8), also where every compute unit would have a row (300 rows: 35, whole 49).  Without lists two, and then whole rows
    // (128 rows: 13.5 µs, four 14.4; 300 rows of 32000: 9.4 whole, 10.9 in parts; of 100001 21 and 24).
    args.parts = wave ? 1 : parts_of(rows, vocab, sizeof(T), args.top ? 1024 : rows < 256 ? 512 : 1, kMostParts);
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
    auto run = [&](auto waves, auto runs, auto top) {
        auto kernel = token_log_probs_kernel<T, decltype(waves)::value, decltype(runs)::value, decltype(top)::value>;
        const size_t keys = args.top ? args.top + room_of(decltype(runs)::value, sizeof(T), args.top) : 0;
        const size_t lds = 4 * keys * sizeof(key_t);
        const hipError_t rc = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds));
        if (rc != hipSuccess) return rc;
        hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), lds, stream, args);
        return hipGetLastError();
    };
    // no more runs to a round than a lane has
    auto with_runs = [&](auto waves, auto top) {
        const size_t of_lane = args.part_size * sizeof(T) / (16 * 64 * decltype(waves)::value);
        if (of_lane <= 1) return run(waves, std::integral_constant<int, 1>{}, top);
        if (of_lane <= 2) return run(waves, std::integral_constant<int, 2>{}, top);
        return run(waves, std::integral_constant<int, 4>{}, top);
    };
    auto with_top = [&](auto waves) { return args.top ? with_runs(waves, std::true_type{}) : with_runs(waves, std::false_type{}); };
    const hipError_t rc = wave ? with_top(std::integral_constant<int, 1>{}) : with_top(std::integral_constant<int, 4>{});
    if (rc != hipSuccess || args.parts == 1) return rc;
    hipLaunchKernelGGL(token_log_probs_join_kernel<T>, dim3(static_cast<unsigned>(rows)), dim3(256), 0, stream, args);
    return hipGetLastError();
}

template <typename T>
hipError_t launch_backward(LogProbsGradArgs args, hipStream_t stream)
{
    const size_t rows = args.rows, vocab = args.vocab;
    const bool wave = vocab * sizeof(T) <= kWaveRow;
    // (300 rows of 32000 12.6 µs, with two workgroups to a compute unit 13.4, with one, and whole, 14.2; a row of 131072 4.1 and whole 20)
    args.parts = wave ? 1 : parts_of(rows, vocab, sizeof(T), 1024, 1024);
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
