// One position of each row of logits, chosen by a given number (see cumo_hip_sample_kernel_launch in include/cumo_hip.h).
//
// Every limit (top_k, top_p, min_p) keeps a run from the start of the order "falling x, equal ones by index", and the answer is
// itself the end of such a run, so rows are not sorted: what is asked of the order is always "the element at which the running
// sum first exceeds t", with the sum a count or a sum of weights. A row's elements are counted into bins by their distance from
// its maximum, the running sum over the bins says in which bin that element is, and the elements of that bin alone (or of all
// bins up to it, where they are few, as for a small top_k) are put into a list and ordered.
// Weights are whole numbers, exp((x - max) / temperature) in units of 2^-S with S such that the sum of a row fits 62 bits:
// sums do not depend on their order, and neither does the answer, although bins are added to by atomics. In rows of up to 2^18, S is that
// of a row whose weights are all the largest; a sum is off by n 2^-(S+1) of that, 2^-27 at most. Longer rows each have an S to what their
// weights can come to, by the chunks' maxima (256 times the sum at most): a sum is off by n 2^-51 of itself at most.
//
// Three launches (and a small one for the units of long rows). The largest and the smallest number of each row's parts, and the largest of every chunk of 64 vectors; the bins of
// each row's parts, a block to a part with its bins in shared memory; then a block to a row, which adds the parts' bins up, takes
// their running sums and reads the chunks that reach the list's bins once more. The rows come from memory once and from the
// last-level cache the other times. What bounds it is the order of steps within a row, and for many rows the weights' arithmetic as
// well: forty instructions an element, which keep the vector units busy for half of the second launch (shared memory 15 % of it, its
// conflicts 7 %); its blocks, all at work at once, clear, read, count and write their bins in step. SFloat, temperature 0.8, top_k 50,
// top_p 0.95: one row of 131072 in 24 us (4.1, 5.7 and 15.8 in the three), 256 rows of 50001 in 39 us with one setting for all, and
// in 63 us (13, 27.5 and 24; 0.8 TB/s of logits) with settings of their own, most of which need weights in every bin. Without the
// chunks' maxima the last launch read whole rows: 20.4 and 27.8 us of it, where the first one took 4.0 and 11.2.
#include "common.h"
#include "ew_ops.h"

#include <cstring>
#include <type_traits>

namespace cumo_hip {
namespace {

constexpr int kSaBlock = 1024;
constexpr int kSaBins = 2048;     // the last one: what has no weight
constexpr int kSaList = 1024;
constexpr uint32_t kSaFew = 256;  // elements that are ordered together rather than a bin at a time
constexpr double kSaBinsPerNat = 48.0;   // the last bin then begins at exp(-42.6), less than half of the smallest unit
constexpr uint64_t kSaSmallK = 512;

// an unsigned integer that orders as the numbers do; both zeros have one
template <class T> struct SaKey;
template <> struct SaKey<float> {
    typedef uint32_t U;
    __device__ __forceinline__ static U of(float x) {
        const uint32_t b = __float_as_uint(x + 0.0f);
        return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
    }
    __device__ __forceinline__ static float value(U k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }
};
template <> struct SaKey<double> {
    typedef uint64_t U;
    __device__ __forceinline__ static U of(double x) {
        const uint64_t b = (uint64_t)__double_as_longlong(x + 0.0);
        return b ^ ((uint64_t)((int64_t)b >> 63) | 0x8000000000000000ull);
    }
    __device__ __forceinline__ static double value(U k) {
        return __longlong_as_double((long long)(k & 0x8000000000000000ull ? k ^ 0x8000000000000000ull : ~k));
    }
};

// a value that every lane of the block holds, as one of the wave's: branches on it are the wave's too, and it takes no lane's registers
template <class V>
__device__ __forceinline__ V sa_same(V v) {
    if constexpr (sizeof(V) <= 4) {
        union { V v; int w; } u;
        u.w = 0;
        u.v = v;
        u.w = __builtin_amdgcn_readfirstlane(u.w);
        return u.v;
    } else {
        union { V v; int w[2]; } u;
        u.v = v;
        u.w[0] = __builtin_amdgcn_readfirstlane(u.w[0]);
        u.w[1] = __builtin_amdgcn_readfirstlane(u.w[1]);
        return u.v;
    }
}

// A row's number in two steps: its words, without a branch, so that several numbers are on their way together (from `any`, some
// memory, where there is one number for all rows), then what they say.
struct SaNumber {
    uint32_t low, high;
    __device__ __forceinline__ SaNumber(const cumo_hip_row_number_t& a, uint64_t row, const void* any) {
        const uint32_t* at = reinterpret_cast<const uint32_t*>(a.each ? a.each : static_cast<const char*>(any));
        const uint64_t k = a.each ? (a.type == 1 ? 2 * row : row) : 0;
        low = at[k];
        high = at[a.each && a.type == 1 ? k + 1 : k];
    }
    __device__ __forceinline__ double value(const cumo_hip_row_number_t& a) const {
        if (!a.each) return a.value;
        const uint32_t l = sa_same(low);
        if (a.type == 0) return (double)__uint_as_float(l);
        if (a.type == 1) return __hiloint2double((int)sa_same(high), (int)l);
        return (double)(int32_t)l;
    }
};

// Weights of a row, 2^S for its maximum, and the bins. The sum with 1.5 * 2^52 leaves the rounded product in the lower bits.
// Differences are of h x, h being 1, or 1/2 in rows whose largest and smallest number are further apart than their type reaches: an
// infinite difference would put a number that has weight (at temperatures of the type's largest numbers) among those that have none.
template <class T>
struct SaWeight {
    T max, bins_per;   // bins per unit of h x
    double h, per_h, far;      // 1 / h, h max
    double rate, unit;  // rate: log2(e) / (h temperature); unit: 2^S, S <= 50
    __device__ __forceinline__ double share(T x) const {
        if (x == max) return 1.0;
        const double e = __builtin_fma((double)x, h, -far) * rate;
        // (2^-70 and less is less than half of a unit; so is NaN, from -inf * 0. The table's to 2^-39; DFloat by it: [256,50001] 71 us, 76.)
        if constexpr (sizeof(T) == 4) return e > -70.0 ? exp2_by_table(e, float_tables()) : 0.0;
        else return e > -70.0 ? exp2(e) : 0.0;
    }
    __device__ __forceinline__ uint64_t units(double share) const {
        return (uint64_t)__double_as_longlong(__builtin_fma(share, unit, 6755399441055744.0)) & 0x7ffffffffffffull;
    }
    // falls with x, never out of order: a difference, a product and a cut, each rounded
    __device__ __forceinline__ uint32_t bin(T x) const {
        const T d = x == max ? (T)0 : __builtin_elementwise_fma(x, -(T)h, (T)far) * bins_per;
        return d < (T)(kSaBins - 1) ? (uint32_t)d : (uint32_t)(kSaBins - 1);   // (NaN, from inf * 0: the last)
    }
};

struct SaPart {
    double max, least;   // of what is finite the smallest
    uint64_t nan;
};

struct SaParams : cumo_hip_sample_t {
    int unit_bits;
    double* units;           // [rows]: 2^S of each row instead, where rows are long; else NULL
    uint32_t looks, fills;   // parts of a row in the first two launches (64 and 16 at most)
    uint32_t chunks;         // of a row: what a wave reads at once
    SaPart* parts;           // [rows][looks]
    char* chunk_max;         // [rows][chunks]
    uint64_t* masses;        // [rows][fills][bins]
    uint64_t* likely;        // [rows][fills]: the weights that min_p leaves of a part, where other limits come before it
    uint32_t* counts;        // the same, where a row may have a top_k
};

// f of the elements [from, to) of a row, by whole waves: lanes without one bring -inf. U: vectors of a lane that are on their way at
// once (a second set behind them is no gain: 256 rows at once are bound by the last-level cache's rate).
template <class T, int BLOCK, int U, class F>
__device__ __forceinline__ void sa_each(const T* row, uint32_t from, uint32_t to, F f) {
    constexpr int V = 16 / (int)sizeof(T);
    typedef uint32_t u4 __attribute__((ext_vector_type(4)));
    union Vec { u4 q; T t[V]; __device__ Vec() {} };
    const T* part = row + from;
    const uint32_t n = to - from, whole = n / V;
#pragma unroll 1
    for (uint32_t first = 0; first < whole; first += BLOCK * U) {
        Vec x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t at = first + (uint32_t)u * BLOCK + threadIdx.x;
            x[u].q = reinterpret_cast<const u4*>(part)[at < whole ? at : 0];
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t at = first + (uint32_t)u * BLOCK + threadIdx.x;
#pragma unroll
            for (int j = 0; j < V; ++j) f(at < whole ? x[u].t[j] : (T)-INFINITY, from + at * V + j);
        }
    }
    f(threadIdx.x < n % V ? part[whole * V + threadIdx.x] : (T)-INFINITY, from + whole * V + threadIdx.x);
}

// a part's first and last element, whole chunks of it but for the row's end
template <class T> constexpr uint32_t kSaChunk = 64 * 16 / sizeof(T);
__device__ __forceinline__ void sa_part(uint32_t n, uint32_t parts, uint32_t part, uint32_t& from, uint32_t& to) {
    const uint32_t per = ((n + parts - 1) / parts + 255) & ~255u;
    from = part * per < n ? part * per : n;
    to = n - from < per ? n : from + per;
}

// (a NaN is lost here; rows that hold one are told apart)
__device__ __forceinline__ float sa_max(float a, float b) { return __builtin_fmaxf(a, b); }
__device__ __forceinline__ double sa_max(double a, double b) { return __builtin_fmax(a, b); }
__device__ __forceinline__ float sa_min(float a, float b) { return __builtin_fminf(a, b); }
__device__ __forceinline__ double sa_min(double a, double b) { return __builtin_fmin(a, b); }

// the largest of a wave's values, in lane 63: shifts within 16 lanes, then the last lanes of those handed on
template <class T, int CTRL, int ROWS>
__device__ __forceinline__ T sa_larger_from(T v) {
    union { T t; int w[sizeof(T) / 4]; } u, o;
    u.t = v;
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) / 4); ++i) o.w[i] = __builtin_amdgcn_update_dpp(u.w[i], u.w[i], CTRL, ROWS, 0xf, false);
    return sa_max(o.t, v);
}
template <class T>
__device__ __forceinline__ T sa_largest(T v) {
    v = sa_larger_from<T, 0x111, 0xf>(v);
    v = sa_larger_from<T, 0x112, 0xf>(v);
    v = sa_larger_from<T, 0x114, 0xf>(v);
    v = sa_larger_from<T, 0x118, 0xf>(v);
    v = sa_larger_from<T, 0x142, 0xa>(v);
    return sa_larger_from<T, 0x143, 0xc>(v);
}

// of all lanes, the same in each
template <class T>
__device__ __forceinline__ T sa_largest_of_all(T v) {
    union { T t; int w[sizeof(T) / 4]; } u;
    u.t = sa_largest(v);
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) / 4); ++i) u.w[i] = __builtin_amdgcn_readlane(u.w[i], 63);
    return u.t;
}

constexpr int kSaLook = 256;
template <class T>
__global__ __launch_bounds__(kSaLook) void sample_look_kernel(SaParams p) {
    constexpr int V = 16 / (int)sizeof(T), U = 4;
    typedef uint32_t u4 __attribute__((ext_vector_type(4)));
    union Vec { u4 q; T t[V]; __device__ Vec() {} };
    __shared__ T wave_max[kSaLook / 64], wave_least[kSaLook / 64];
    __shared__ uint32_t wave_nan[kSaLook / 64];
    uint32_t from, to;
    sa_part((uint32_t)p.n, p.looks, blockIdx.y, from, to);
    T m = -INFINITY, least = INFINITY;
    bool nan = false;
    auto look = [&](T v) {
        nan |= v != v;
        m = sa_max(m, v);
        least = sa_min(least, v > (T)-INFINITY ? v : (T)INFINITY);
    };
    const T* part = reinterpret_cast<const T*>(p.x + (int64_t)blockIdx.x * p.x_step) + from;
    T* chunk_max = reinterpret_cast<T*>(p.chunk_max) + (uint64_t)blockIdx.x * p.chunks + from / kSaChunk<T>;
    const uint32_t whole = (to - from) / V, tail = (to - from) % V;
#pragma unroll 1
    for (uint32_t begin = 0; begin < whole; begin += kSaLook * U) {
        Vec x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t at = begin + (uint32_t)u * kSaLook + threadIdx.x;
            x[u].q = reinterpret_cast<const u4*>(part)[at < whole ? at : 0];
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t at = begin + (uint32_t)u * kSaLook + threadIdx.x;
            T most = -INFINITY;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const T v = at < whole ? x[u].t[j] : (T)-INFINITY;
                look(v);
                most = sa_max(most, v);
            }
            most = sa_largest(most);
            if ((threadIdx.x & 63) == 63 && at - 63 < whole) chunk_max[at / 64] = most;
        }
    }
    if (threadIdx.x < tail) look(part[whole * V + threadIdx.x]);
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) {
        m = sa_max(m, __shfl_xor(m, d));
        least = sa_min(least, __shfl_xor(least, d));
    }
    const bool wave_has_nan = __ballot(nan) != 0;
    const uint32_t wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) {
        wave_max[wave] = m;
        wave_least[wave] = least;
        wave_nan[wave] = wave_has_nan;
    }
    __syncthreads();
    if (threadIdx.x != 0) return;
    nan = wave_has_nan;
    for (int w = 1; w < kSaLook / 64; ++w) {
        m = sa_max(m, wave_max[w]);
        least = sa_min(least, wave_least[w]);
        nan |= wave_nan[w] != 0;
    }
    p.parts[(uint64_t)blockIdx.x * p.looks + blockIdx.y] = {(double)m, (double)least, nan ? 1u : 0u};
}

// a row's settings, the same for every lane
template <class T>
struct SaSettings {
    SaWeight<T> weight;
    bool none, greedy;         // nothing to choose; the first of the largest
    bool all, cut_p, cut_m, small;   // no top_k; top_p, min_p cut; a top_k small enough for a list
    uint64_t top_k;
    double u, top_p, likely, bin_size;
    __device__ __forceinline__ SaSettings(const SaParams& p, uint64_t row) {
        const uint32_t lane = threadIdx.x & 63;
        const SaPart part = p.parts[row * p.looks + (lane < p.looks ? lane : 0)];   // (one of them more than once changes nothing)
        const SaNumber u_at(p.u, row, p.parts), temperature_at(p.temperature, row, p.parts), k_at(p.top_k, row, p.parts), top_p_at(p.top_p, row, p.parts),
            min_p_at(p.min_p, row, p.parts);
        if constexpr (sizeof(T) == 4) float_tables_prepare();
        T m = (T)part.max, least = (T)part.least;
        m = sa_largest_of_all(m);
        least = -sa_largest_of_all(-least);
        none = __ballot(part.nan != 0) != 0 || m == (T)-INFINITY;
        const double temperature = temperature_at.value(p.temperature), k = k_at.value(p.top_k), min_p = min_p_at.value(p.min_p);
        u = u_at.value(p.u);
        top_p = top_p_at.value(p.top_p);
        all = !(k > 0.0 && k < (double)p.n);
        greedy = !(temperature > 0.0) || (!all && k < 2.0) || top_p <= 0.0;
        top_k = all ? p.n : (uint64_t)k;
        cut_p = top_p < 1.0;
        cut_m = min_p > 0.0;
        likely = min_p < 1.0 ? min_p : 1.0;
        small = !all && top_k <= kSaSmallK;
        weight.max = m;
        const bool within = (double)m - (double)least <= (sizeof(T) == 4 ? (double)__FLT_MAX__ : __DBL_MAX__);
        const double h = sa_same(within ? 1.0 : 0.5), per_h = sa_same(within ? 1.0 : 2.0);
        weight.h = h;
        weight.per_h = per_h;
        weight.far = sa_same((double)m * h);
        weight.rate = sa_same(1.44269504088896338700e+00 / temperature * per_h);
        weight.unit = p.units ? sa_same(p.units[row]) : __longlong_as_double((long long)(1023 + p.unit_bits) << 52);
        // bins of 1/48 of a factor e, or finer ones where the row's numbers span less than the bins then reach
        const double per = kSaBinsPerNat / temperature * per_h, span = (double)m * h - (double)least * h, most = sizeof(T) == 4 ? 1e37 : 1e300;
        weight.bins_per = sa_same((T)__builtin_fmin(span * per < (double)(kSaBins - 2) ? (double)(kSaBins - 2) / span : per, most));   // (span 0: one number)
        bin_size = sa_same(1.0 / (double)weight.bins_per);
    }
};

// 2^S of long rows: a chunk's weights are 256 (DFloat 128) times its largest number's at most
template <class T>
__global__ __launch_bounds__(kSaBlock) void sample_unit_kernel(SaParams p, double* units) {
    __shared__ double slots[kSaBlock / 64];
    const SaSettings<T> s(p, blockIdx.x);
    if (s.none || s.greedy) return;   // (nobody asks)
    constexpr int V = 16 / (int)sizeof(T);
    const T* chunk_max = reinterpret_cast<const T*>(p.chunk_max) + (uint64_t)blockIdx.x * p.chunks;
    double most = 0.0;
    for (uint32_t c = threadIdx.x; c < p.chunks; c += kSaBlock) most += s.weight.share(chunk_max[c]) * kSaChunk<T>;
    if (threadIdx.x < p.n % V) most += s.weight.share(reinterpret_cast<const T*>(p.x + (int64_t)blockIdx.x * p.x_step)[p.n / V * V + threadIdx.x]);
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) most += __shfl_xor(most, d);
    if ((threadIdx.x & 63) == 0) slots[threadIdx.x >> 6] = most;
    __syncthreads();
    if (threadIdx.x != 0) return;
    for (int w = 1; w < kSaBlock / 64; ++w) most += slots[w];
    // less than 2^61 of units, and half a unit for each of fewer than 2^31 weights
    const int bits = 61 - __builtin_amdgcn_frexp_exp(most);
    units[blockIdx.x] = ldexp(1.0, bits < 50 ? bits : 50);
}

template <class T>   // (two blocks a compute unit: DFloat's exponential would take 66 registers, [256,50001] 81 us instead of 76)
__global__ __launch_bounds__(kSaBlock, 8) void sample_fill_kernel(SaParams p) {
    __shared__ uint64_t masses[kSaBins], likely;
    __shared__ uint32_t counts[kSaBins];
    const SaSettings<T> s(p, blockIdx.x);
    if (s.none || s.greedy) return;
    if (threadIdx.x == 0) likely = 0;
    for (uint32_t b = threadIdx.x; b < kSaBins; b += kSaBlock) {
        masses[b] = 0;
        counts[b] = 0;
    }
    __syncthreads();
    uint32_t from, to;
    sa_part((uint32_t)p.n, p.fills, blockIdx.y, from, to);
    const T* x = reinterpret_cast<const T*>(p.x + (int64_t)blockIdx.x * p.x_step);
    if (from < to) {
        if (s.small) {
            sa_each<T, kSaBlock, 4>(x, from, to, [&](T v, uint32_t) {
                if (v > (T)-INFINITY) atomicAdd(&counts[s.weight.bin(v)], 1u);
            });
        } else {
            // (where min_p alone cuts, what it leaves out need not be summed)
            const double least = s.cut_m && s.all && !s.cut_p ? s.likely : 0.0;
            uint64_t mine = 0;
            sa_each<T, kSaBlock, 4>(x, from, to, [&](T v, uint32_t) {
                const double share = s.weight.share(v);
                const uint64_t units = share >= least ? s.weight.units(share) : 0;
                mine += share >= s.likely ? units : 0;
                asm("" : "+v"(mine));   // (one after the other: sixteen numbers' weights side by side are twice the registers, and half the blocks)
                const uint32_t b = s.weight.bin(v);
                if (units) atomicAdd((unsigned long long*)&masses[b], (unsigned long long)units);
                if (!s.all && v > (T)-INFINITY) atomicAdd(&counts[b], 1u);
            });
            if (s.cut_m) {
#pragma unroll
                for (int d = 32; d > 0; d >>= 1) mine += (uint64_t)__shfl_xor((unsigned long long)mine, d);
                if ((threadIdx.x & 63) == 0) atomicAdd((unsigned long long*)&likely, (unsigned long long)mine);
            }
        }
    }
    __syncthreads();
    if (threadIdx.x == 0) p.likely[(uint64_t)blockIdx.x * p.fills + blockIdx.y] = likely;
    const uint64_t at = ((uint64_t)blockIdx.x * p.fills + blockIdx.y) * kSaBins;
    for (uint32_t b = threadIdx.x; b < kSaBins; b += kSaBlock) {
        if (!s.small) p.masses[at + b] = masses[b];
        if (!s.all) p.counts[at + b] = counts[b];
    }
}

template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t sa_from(uint64_t v) {   // 0 for lanes that none hands on to
    const uint32_t low = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROWS, 0xf, false);
    const uint32_t high = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), CTRL, ROWS, 0xf, false);
    return ((uint64_t)high << 32) | low;
}

// inclusive sums over the block's lanes, in the lanes' order; slots: one for each wave
__device__ __forceinline__ uint64_t sa_scan(uint64_t v, uint64_t* slots) {
    const uint32_t lane = threadIdx.x & 63, wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    // within 16 lanes by shifts, then the last lanes of those handed on
    v += sa_from<0x111, 0xf>(v);
    v += sa_from<0x112, 0xf>(v);
    v += sa_from<0x114, 0xf>(v);
    v += sa_from<0x118, 0xf>(v);
    v += sa_from<0x142, 0xa>(v);
    v += sa_from<0x143, 0xc>(v);
    __syncthreads();
    if (lane == 63) slots[wave] = v;
    __syncthreads();
    uint64_t before = 0;
#pragma unroll 5
    for (uint32_t w = 0; w + 1 < kSaBlock / 64; ++w) before += w < wave ? slots[w] : 0;
    return v + sa_same(before);
}

template <class T>
__global__ __launch_bounds__(kSaBlock) void sample_kernel(SaParams p) {
    typedef SaKey<T> Key;
    typedef typename Key::U U;
    constexpr int kWaves = kSaBlock / 64, KV = 16 / (int)sizeof(U);
    typedef U UV __attribute__((ext_vector_type(KV)));
    typedef uint32_t IV __attribute__((ext_vector_type(KV)));
    __shared__ uint64_t masses[kSaBins];   // running sums of the bins
    __shared__ uint32_t counts[kSaBins];
    __shared__ __attribute__((aligned(16))) U list_key[kSaList];
    __shared__ U sorted_key[kSaList];
    __shared__ __attribute__((aligned(16))) uint32_t list_index[kSaList];
    __shared__ uint32_t sorted_index[kSaList];
    __shared__ uint64_t list_sum[kSaList], slots[kWaves], found[3], digit_count[256], digit_mass[256];
    __shared__ uint32_t list_size;
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const uint32_t n = (uint32_t)p.n;
    const uint64_t row = blockIdx.x;
    const T* x = reinterpret_cast<const T*>(p.x + (int64_t)row * p.x_step);
    const SaSettings<T> s(p, row);
    const SaWeight<T>& weight = s.weight;
    if (s.none) {
        if (tid == 0) p.out[row] = -1;
        return;
    }
    const T* chunk_max = reinterpret_cast<const T*>(p.chunk_max) + row * p.chunks;
    constexpr int V = 16 / (int)sizeof(T);
    const uint32_t whole = n / V;   // vectors; 64 of them are a chunk
    if (s.greedy) {
        // the first of the largest: the first chunk that has it, or one of the elements behind the chunks
        if (tid == 0) list_size = p.chunks;
        __syncthreads();
        uint32_t chunk = p.chunks;
        for (uint32_t c = tid; c < p.chunks && chunk == p.chunks; c += kSaBlock) chunk = chunk_max[c] == weight.max ? c : chunk;
        if (chunk < p.chunks) atomicMin(&list_size, chunk);
        __syncthreads();
        if (wave != 0) return;
        chunk = sa_same(list_size);
        const uint32_t at = chunk < p.chunks ? (chunk * 64 + lane) * V : whole * V + lane;
        const uint32_t here = chunk < p.chunks ? (chunk * 64 + lane < whole ? V : 0) : (lane < n % V ? 1 : 0);
        uint32_t found_at = 0xffffffffu;
        for (int j = V - 1; j >= 0; --j) found_at = (uint32_t)j < here && x[at + j] == weight.max ? at + j : found_at;
        const uint64_t hits = __ballot(found_at != 0xffffffffu);
        if (hits && lane == (uint32_t)__builtin_ctzll(hits)) p.out[row] = (int32_t)found_at;
        return;
    }
    const double u = s.u;
    const uint64_t part_likely = lane < p.fills ? p.likely[row * p.fills + lane] : 0;
    bool small = s.small;
    {
        const uint32_t b = 2 * tid;   // (two bins a lane)
        uint64_t one = 0, two = 0;
        uint32_t c_one = 0, c_two = 0;
        const uint64_t at = row * p.fills * kSaBins + b;
        if (!small) {
#pragma unroll 8
            for (uint32_t part = 0; part < p.fills; ++part) {
                const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(p.masses + at + (uint64_t)part * kSaBins);
                one += v.x;
                two += v.y;
            }
        }
        if (!s.all) {
#pragma unroll 8
            for (uint32_t part = 0; part < p.fills; ++part) {
                const uint2 v = *reinterpret_cast<const uint2*>(p.counts + at + (uint64_t)part * kSaBins);
                c_one += v.x;
                c_two += v.y;
            }
        }
        if (!small) {
            const uint64_t run = sa_scan(one + two, slots);
            masses[b] = run - two;
            masses[b + 1] = run;
        }
        if (!s.all) {
            const uint32_t run = (uint32_t)sa_scan(c_one + c_two, slots);
            counts[b] = run - c_two;
            counts[b + 1] = run;
        }
        __syncthreads();
    }

    // f of the elements that are `least` or more, and of others: of the chunks whose largest number is. Chunks four at a time; each
    // wave has every sixteenth, and all of its lanes call f (those without an element with -inf).
    auto gather = [&](auto held_at_once, T least, auto f) {
        constexpr int G = decltype(held_at_once)::value;
        typedef uint32_t u4 __attribute__((ext_vector_type(4)));
        union Vec { u4 q; T t[V]; __device__ Vec() {} };
#pragma unroll 1
        for (uint32_t first = wave; first < p.chunks; first += 64 * kWaves) {
            const uint32_t mine = first + lane * kWaves;
            uint64_t want = __ballot(mine < p.chunks && chunk_max[mine < p.chunks ? mine : 0] >= least);
#pragma unroll 1
            while (want) {
                Vec held[G];
                uint32_t at[G];
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    at[g] = want ? (first + (uint32_t)__builtin_ctzll(want) * kWaves) * 64 + lane : whole;
                    want &= want - 1;
                    held[g].q = reinterpret_cast<const u4*>(x)[at[g] < whole ? at[g] : 0];
                }
#pragma unroll
                for (int g = 0; g < G; ++g) {
#pragma unroll
                    for (int j = 0; j < V; ++j) f(at[g] < whole ? held[g].t[j] : (T)-INFINITY, at[g] * V + j);
                }
            }
        }
        f(tid < n % V ? x[whole * V + tid] : (T)-INFINITY, whole * V + tid);
    };
    // What may be in bins [from, to], half a bin more on either side. (The bins' rounding moves a number by less than a thousandth
    // of a bin, and the bounds' keeps the order.)
    auto most_of = [&](uint32_t from) {
        const double above = from == 0 ? -INFINITY : ((double)from - 0.5) * s.bin_size;
        return (T)((weight.far - above) * weight.per_h);
    };
    auto least_of = [&](uint32_t to) {
        const double lowest = (weight.far - ((double)to + 1.5) * s.bin_size) * weight.per_h;
        return to < kSaBins - 1 && lowest == lowest ? (T)lowest : (T)-INFINITY;
    };

    // the list: of the elements in bins [lo, hi], in order, with their running sum of weights; false where they are too many
    uint32_t lo = 1, hi = 0;
    auto make_list = [&](uint32_t from, uint32_t to) {
        __syncthreads();
        if (tid == 0) list_size = 0;
        list_key[tid] = 0;   // (below every number's key)
        list_sum[tid] = 0;
        __syncthreads();
        const T most = most_of(from), least = least_of(to);   // (two comparisons for each number that is not)
        auto enter = [&](T v, uint32_t i) {
            if (__ballot(v >= least && v <= most)) {
                const uint32_t b = weight.bin(v);
                const bool hit = b >= from && b <= to && v > (T)-INFINITY;
                const uint64_t hits = __ballot(hit);
                uint32_t at = 0;
                if (lane == 0) at = atomicAdd(&list_size, (uint32_t)__popcll(hits));
                at = (uint32_t)__builtin_amdgcn_readfirstlane((int)at) + (uint32_t)__popcll(hits & ((1ull << lane) - 1));
                if (hit && at < kSaList) {
                    list_key[at] = Key::of(v);
                    list_index[at] = i;
                }
            }
        };
        gather(std::integral_constant<int, 4>(), least, enter);
        __syncthreads();
        const uint32_t size = sa_same(list_size);
        lo = 1;
        hi = 0;
        if (size > kSaList) return false;
        // An element's place is the number of those before it, counted in as many parts as the block has lanes for.
        const uint32_t lanes = size <= kSaBlock / 4 ? kSaBlock / 4 : size <= kSaBlock / 2 ? kSaBlock / 2 : kSaBlock, groups = kSaBlock / lanes;
        const uint32_t group = tid / lanes, mine = tid & (lanes - 1), per = ((size + groups - 1) / groups + KV - 1) & ~(uint32_t)(KV - 1);
        if ((mine & ~63u) < size) {
            const U key = list_key[mine];
            const uint32_t index = list_index[mine], end = size < (group + 1) * per ? size : (group + 1) * per;
            uint32_t place = 0;
#pragma unroll 2
            for (uint32_t i = group * per; i < end; i += KV) {   // (behind the list's end are keys of 0, which no number has)
                const UV other = *reinterpret_cast<const UV*>(&list_key[i]);
                const IV other_index = *reinterpret_cast<const IV*>(&list_index[i]);
#pragma unroll
                for (int j = 0; j < KV; ++j) place += (other[j] > key) | ((other[j] == key) & (other_index[j] < index)) ? 1 : 0;
            }
            atomicAdd(reinterpret_cast<uint32_t*>(&list_sum[mine]), place);
        }
        __syncthreads();
        if (tid < size) {
            const uint32_t place = (uint32_t)list_sum[tid];
            sorted_key[place] = list_key[tid];
            sorted_index[place] = list_index[tid];
        }
        __syncthreads();
        const uint64_t sum = sa_scan(tid < size ? weight.units(weight.share(Key::value(sorted_key[tid]))) : 0, slots);
        if (tid < size) list_sum[tid] = sum;
        __syncthreads();
        lo = from;
        hi = to;
        return true;
    };
    // the position in the list at which its running sum passes t (which it does)
    auto in_list = [&](uint64_t t) {
        if (tid < list_size && list_sum[tid] > t && (tid == 0 || list_sum[tid - 1] <= t)) found[0] = tid;
        __syncthreads();
        const uint32_t at = sa_same((uint32_t)found[0]);
        __syncthreads();
        return at;
    };
    // the bin in which the running sum passes t; the last one where it does not
    auto bin_of = [&](bool by_weight, uint64_t t) {
        if (tid == 0) found[0] = kSaBins - 1;
        __syncthreads();
#pragma unroll
        for (uint32_t k = 0; k < 2; ++k) {
            const uint32_t b = 2 * tid + k;
            const uint64_t run = by_weight ? masses[b] : counts[b], before = b == 0 ? 0 : (by_weight ? masses[b - 1] : counts[b - 1]);
            if (run > t && before <= t) found[0] = b;
        }
        __syncthreads();
        const uint32_t b = sa_same((uint32_t)found[0]);
        __syncthreads();
        return b;
    };
    // the weights of the elements that share `least` of the largest or more
    auto sum_of = [&](double least) {
        uint64_t mine = 0;
        sa_each<T, kSaBlock, 4>(x, 0, n, [&](T v, uint32_t) {
            const double share = weight.share(v);
            mine += share >= least ? weight.units(share) : 0;
            asm("" : "+v"(mine));   // (one after the other)
        });
        const uint64_t run = sa_scan(mine, slots);
        __syncthreads();
        if (tid == kSaBlock - 1) found[0] = run;
        __syncthreads();
        const uint64_t all = sa_same(found[0]);
        __syncthreads();
        return all;
    };
    // For a bin that holds more than a list does: its smallest and its largest key, then the key in question by eight more bits of what
    // lies between the two, and again. Elements of one key have one weight, so which of them it is follows from a division. (One row
    // of 131072 in steps of 1/4, top_p 0.95: 144 us, all of a key's bits by 256s over the whole row 858; 256 rows of 50001 129, 490.)
    U key = 0;
    uint64_t number = 0;   // how many of that key stand before it
    // the least and the largest key of bin b, or (b: none) of those in [lowest, highest]; weights: those of the bins before b
    auto narrow = [&](uint32_t b, U& lowest, U& highest, uint64_t& weights) {
        const bool weigh = b < kSaBins && s.small;
        const T least = b < kSaBins ? least_of(b) : Key::value(lowest);
        U low = ~(U)0, high = 0;
        uint64_t sum_before = 0;
        gather(std::integral_constant<int, 2>(), least, [&](T v, uint32_t) {
            if (!(v >= least && v > (T)-INFINITY)) return;
            const U k = Key::of(v);
            const uint32_t of = b < kSaBins ? weight.bin(v) : kSaBins;
            const bool in = b < kSaBins ? of == b : k >= lowest && k <= highest;
            low = in && k < low ? k : low;
            high = in && k > high ? k : high;
            if (weigh && of < b) sum_before += weight.units(weight.share(v));
            asm("" : "+v"(sum_before));   // (one after the other)
        });
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) {
            const U l = __shfl_xor(low, d), h = __shfl_xor(high, d);
            low = l < low ? l : low;
            high = h > high ? h : high;
        }
        __syncthreads();
        if (lane == 0) {
            digit_count[wave] = low;
            digit_mass[wave] = high;
        }
        weights = weigh ? sa_scan(sum_before, slots) : 0;
        if (tid == kSaBlock - 1) found[0] = weights;
        __syncthreads();
        low = (U)digit_count[lane & (kWaves - 1)];
        high = (U)digit_mass[lane & (kWaves - 1)];
#pragma unroll
        for (int d = kWaves / 2; d > 0; d >>= 1) {
            const U l = __shfl_xor(low, d), h = __shfl_xor(high, d);
            low = l < low ? l : low;
            high = h > high ? h : high;
        }
        low = sa_same(low);
        high = sa_same(high);
        if (low <= high) {
            lowest = low;
            highest = high;
        }
        weights = sa_same(found[0]);
        __syncthreads();
    };
    // b: the bin; none after a top_k that went this way with no weights of bins: its key and all above it
    auto by_digits = [&](bool by_weight, uint64_t t, uint32_t b) {
        U lowest = key, highest = Key::of(weight.max);
        uint64_t before = 0, before_weight = 0;
        if (b < kSaBins) {
            narrow(b, lowest, highest, before_weight);
            if (!s.small) before_weight = b ? sa_same(masses[b - 1]) : 0;
            before = by_weight ? before_weight : b ? sa_same(counts[b - 1]) : 0;
        }
#pragma unroll 1
        while (lowest < highest) {   // (fewer bits each time)
            const int bits = 64 - __builtin_clzll((uint64_t)(highest - lowest)), shift = bits > 8 ? bits - 8 : 0;
            if (tid < 256) digit_count[tid] = digit_mass[tid] = 0;
            if (tid == 0) {
                found[0] = 0;
                found[1] = before;
                found[2] = before_weight;
            }
            __syncthreads();
            const T least = Key::value(lowest);
            gather(std::integral_constant<int, 2>(), least, [&](T v, uint32_t) {
                const U k = Key::of(v);
                if (!(v >= least && k <= highest)) return;
                const uint32_t digit = (uint32_t)((k - lowest) >> shift);
                if (!by_weight) atomicAdd((unsigned long long*)&digit_count[digit], 1ull);
                atomicAdd((unsigned long long*)&digit_mass[digit], (unsigned long long)weight.units(weight.share(v)));
            });
            __syncthreads();
            const uint64_t mass = tid < 256 ? digit_mass[255 - tid] : 0, count = tid < 256 ? digit_count[255 - tid] : 0;
            const uint64_t run_mass = sa_scan(mass, slots), run = by_weight ? run_mass : sa_scan(count, slots), one = by_weight ? mass : count;
            if (before + run > t && before + run - one <= t && one) {
                found[0] = 255 - tid;
                found[1] = before + run - one;
                found[2] = before_weight + run_mass - mass;
            }
            __syncthreads();
            lowest += (U)sa_same(found[0]) << shift;
            const U span = ((U)1 << shift) - 1;   // (at infinity's key there need not be room for it)
            highest = highest - lowest < span ? highest : lowest + span;
            before = sa_same(found[1]);
            before_weight = sa_same(found[2]);
            __syncthreads();
            uint64_t none;
            if (shift) narrow(kSaBins, lowest, highest, none);
        }
        const uint64_t one = sa_same(weight.units(weight.share(Key::value(lowest))));
        key = lowest;
        number = by_weight && one ? (t - before) / one : t - before;
        return before_weight + (number + 1) * one;
    };

    // top_k, top_p, then the answer itself: each the element at which a running sum first passes t. For a small top_k the elements
    // of the bins that hold it are all that is needed: those alone have weights here. Where they do not fit the list, everything
    // goes by digits.
    bool digits = false, listed = false;
    uint32_t index = 0;
    uint64_t sum = small ? 0 : sa_same(masses[kSaBins - 1]);
#pragma unroll 1
    for (int stage = s.all ? 1 : 0; stage < 3; ++stage) {
        const bool by_weight = stage > 0;
        uint64_t t = s.top_k - 1;
        if (stage == 0) {   // (of what is not -inf)
            const uint32_t there = sa_same(counts[kSaBins - 1]);
            t = t < there ? t : there - 1;
        } else if (stage == 1) {
            if (!s.cut_p) continue;
            const double want = sa_same(ceil(s.top_p * (double)sum));
            t = want > 1.0 ? (uint64_t)want - 1 : 0;
            t = t < sum ? t : sum - 1;
        } else if (stage == 2) {
            if (s.cut_m && (!s.all || s.cut_p)) {
                uint64_t likely;
                if (small) {
                    const bool mine = tid < list_size && weight.share(Key::value(sorted_key[tid])) >= s.likely;
                    const uint64_t those = __ballot(mine);   // (the first ones of the list)
                    if (lane == 0) slots[wave] = (uint64_t)__popcll(those);
                    __syncthreads();
                    uint64_t number_of = lane < kWaves ? slots[lane] : 0;
#pragma unroll
                    for (int d = 8; d > 0; d >>= 1) number_of += (uint64_t)__shfl_xor((unsigned long long)number_of, d);
                    likely = sa_same(list_sum[sa_same((uint32_t)number_of) - 1]);
                    __syncthreads();
                } else if (s.small) {   // (no part has taken weights)
                    likely = sum_of(s.likely);
                } else {
                    likely = part_likely;
#pragma unroll
                    for (int d = 32; d > 0; d >>= 1) likely += (uint64_t)__shfl_xor((unsigned long long)likely, d);
                    likely = sa_same(likely);
                }
                sum = likely < sum ? likely : sum;
            }
            const double want = sa_same(floor((u > 0.0 ? u : 0.0) * (double)sum));
            t = want < (double)sum && (uint64_t)want < sum ? (uint64_t)want : sum - 1;
        }
        uint32_t b = kSaBins;
        if (!digits && !(small && by_weight)) {
            b = bin_of(by_weight, t);
            if (stage == 0 && b == kSaBins - 1 && !small) continue;   // (a count that reaches what has no weight: everything that has is in front of it)
            if (b < lo || b > hi) {
                bool few;
                if (s.all) {
                    // few for sure: each element of the bins up to it weighs what the last one's end does, or more
                    const double edge = weight.unit * exp2(-((double)(b + 1) * s.bin_size) * weight.rate);
                    few = sa_same((uint32_t)((double)masses[b] < edge * (0.999 * kSaFew))) != 0;
                } else {
                    few = sa_same(counts[b]) <= (small ? (uint32_t)kSaList : kSaFew);
                }
                digits = small && !few;
                if (!digits) digits = !make_list(few ? 0 : b, b);
                small = small && !digits;
            }
        }
        listed = !digits;
        if (digits) {
            sum = by_digits(by_weight, t, b);
            // (a bin that is too full says nothing of the next one; without the bins' weights all goes by digits)
            digits = s.small;
        } else {
            const uint64_t base = lo == 0 ? 0 : sa_same(masses[lo - 1]);
            const uint32_t place = by_weight ? in_list(t - base) : (uint32_t)t - (lo == 0 ? 0 : sa_same(counts[lo - 1]));
            index = sa_same(sorted_index[place]);
            sum = base + sa_same(list_sum[place]);
        }
    }
    if (listed) {
        if (tid == 0) p.out[row] = (int32_t)index;
        return;
    }
    // the element of that key with `number` before it, in order of the index: a part of the row to each wave, then the part that has it
    uint32_t from = 0, to = n;
    uint64_t left = number;
#pragma unroll 1
    while (to - from > 64) {
        const uint32_t per = ((to - from + kWaves - 1) / kWaves + 63) & ~63u;
        const uint32_t begin = from + wave * per < to ? from + wave * per : to, end = to - begin < per ? to : begin + per;
        uint64_t here = 0;
#pragma unroll 1
        for (uint32_t i = begin; i < end; i += 8 * 64) {
            T held[8];
#pragma unroll
            for (uint32_t g = 0; g < 8; ++g) held[g] = x[i + g * 64 + lane < end ? i + g * 64 + lane : begin];
#pragma unroll
            for (uint32_t g = 0; g < 8; ++g) here += (uint64_t)__popcll(__ballot(i + g * 64 + lane < end && Key::of(held[g]) == key));
        }
        if (lane == 0) slots[wave] = here;
        __syncthreads();
        uint32_t w = 0;
        for (; w + 1 < kWaves && left >= slots[w]; ++w) left -= slots[w];
        __syncthreads();
        w = sa_same(w);
        left = sa_same(left);
        from = from + w * per < to ? from + w * per : to;
        to = to - from < per ? to : from + per;
    }
    const bool hit = from + lane < to && Key::of(x[from + lane]) == key;
    const uint64_t hits = __ballot(hit);
    if (wave == 0 && hit && (uint64_t)__popcll(hits & ((1ull << lane) - 1)) == left) p.out[row] = (int32_t)(from + lane);
}

// rows of one round of launches: their bins take 12 to 24 KiB a part
constexpr uint64_t kSaRows = 4096;
// rows that are longer have units of their own, for another launch
constexpr uint64_t kSaLong = 1u << 18;

template <class T>
int sa_launch(const cumo_hip_sample_t& d, hipStream_t stream) {
    SaParams p;
    std::memset(&p, 0, sizeof(p));
    static_cast<cumo_hip_sample_t&>(p) = d;
    int bits = 0;
    while ((1ull << bits) < d.n) ++bits;
    p.unit_bits = 62 - bits < 50 ? 62 - bits : 50;
    const uint64_t rows = d.rows < kSaRows ? d.rows : kSaRows;
    // enough blocks for every compute unit, and enough elements for every block
    auto parts = [&](uint64_t blocks, uint64_t elements, uint64_t most) {
        uint64_t k = blocks / rows, fit = d.n / elements;
        k = k < fit ? k : fit;
        k = k < most ? k : most;
        return (uint32_t)(k ? k : 1);
    };
    p.looks = parts(2048, 2048, 64);
    p.fills = parts(512, 4096, 16);
    p.chunks = (uint32_t)((d.n / (16 / sizeof(T)) + 63) / 64);
    const bool may_count = d.top_k.each || (d.top_k.value > 0.0 && d.top_k.value < (double)d.n);
    const uint64_t part_bytes = (rows * p.looks * sizeof(SaPart) + 15) & ~15ull, bins = rows * p.fills * kSaBins, own_units = d.n > kSaLong ? rows : 0;
    char* memory = cumo_cuda_runtime_malloc(part_bytes + (bins + rows * p.fills + own_units) * 8 + rows * p.chunks * sizeof(T) + (may_count ? bins * 4 : 0));
    if (!memory) return CUMO_HIP_ERROR_OUT_OF_MEMORY;
    p.parts = reinterpret_cast<SaPart*>(memory);
    p.masses = reinterpret_cast<uint64_t*>(memory + part_bytes);
    p.likely = p.masses + bins;
    double* const units = reinterpret_cast<double*>(p.likely + rows * p.fills);
    p.counts = may_count ? reinterpret_cast<uint32_t*>(units + own_units) : nullptr;
    p.chunk_max = reinterpret_cast<char*>(units + own_units) + (may_count ? bins * 4 : 0);
    cumo_hip_row_number_t* const settings[5] = {&p.u, &p.temperature, &p.top_k, &p.top_p, &p.min_p};
    for (uint64_t done = 0; done < d.rows; done += rows) {
        const unsigned now = (unsigned)(d.rows - done < rows ? d.rows - done : rows);
        hipLaunchKernelGGL((sample_look_kernel<T>), dim3(now, p.looks), dim3(kSaLook), 0, stream, p);
        if (own_units) {
            p.units = nullptr;
            hipLaunchKernelGGL((sample_unit_kernel<T>), dim3(now), dim3(kSaBlock), 0, stream, p, units);
            p.units = units;
        }
        hipLaunchKernelGGL((sample_fill_kernel<T>), dim3(now, p.fills), dim3(kSaBlock), 0, stream, p);
        hipLaunchKernelGGL((sample_kernel<T>), dim3(now), dim3(kSaBlock), 0, stream, p);
        p.x += (int64_t)now * p.x_step;
        p.out += now;
        for (cumo_hip_row_number_t* a : settings)
            if (a->each) a->each += (uint64_t)now * (a->type == 1 ? 8 : 4);
    }
    cumo_cuda_runtime_check_kernel_launch();
    scratch_free(memory);
    return CUMO_HIP_OK;
}

}  // namespace
}  // namespace cumo_hip

using namespace cumo_hip;

extern "C" int cumo_hip_sample_kernel_launch(int type, const cumo_hip_sample_t* d) {
    if (d->rows == 0) return CUMO_HIP_OK;
    return type == 0 ? sa_launch<float>(*d, current_stream()) : sa_launch<double>(*d, current_stream());
}
