// One position of each row of logits, chosen by a given number (see cumo_hip_sample_kernel_launch in include/cumo_hip.h).
//
// Every limit (top_k, top_p, min_p) keeps a run from the start of the order "falling x, equal ones by index", and the answer is
// itself the end of such a run, so nothing is sorted: what is asked of the order is always "the element at which the running
// sum first exceeds t", with the sum a count or a sum of weights. That element is found by its key, an unsigned integer that
// orders as the numbers do, digit by digit from the top: sums over the elements by digit, the digit where the running sum
// passes t, then the next digit of the elements that share it. Elements of the same key have the same weight, so which of them
// it is follows from a division.
// Weights are whole numbers, exp((x - max) / temperature) in units of 2^-S with S such that the sum of a row fits 62 bits:
// sums do not depend on their order, and neither does the answer, although the sums are taken by atomics.
#include "common.h"
#include "ew_ops.h"

#include <cstring>

namespace cumo_hip {
namespace {

constexpr int kSaBlock = 1024;
constexpr int kSaDigit = 8;
constexpr int kSaBins = 1 << kSaDigit;

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

__device__ __forceinline__ double sa_number(const cumo_hip_row_number_t& a, uint64_t row) {
    if (!a.each) return a.value;
    if (a.type == 0) return (double)reinterpret_cast<const float*>(a.each)[row];
    if (a.type == 1) return reinterpret_cast<const double*>(a.each)[row];
    return (double)reinterpret_cast<const int32_t*>(a.each)[row];
}

// weights of a row: 2^S for its maximum. The sum with 1.5 * 2^52 leaves the rounded product in the lower bits.
struct SaWeight {
    double max, rate, unit;  // rate: log2(e) / temperature; unit: 2^S, S <= 50
    __device__ __forceinline__ double share(double x) const {
        if (x == max) return 1.0;
        const double e = (x - max) * rate;
        return e > -70.0 ? exp2_by_table(e, float_tables()) : 0.0;  // (2^-70 and less is less than half of a unit; so is NaN, from -inf * 0)
    }
    __device__ __forceinline__ uint64_t of(double x) const { return units(share(x)); }
    __device__ __forceinline__ uint64_t units(double share) const {
        return (uint64_t)__double_as_longlong(__builtin_fma(share, unit, 6755399441055744.0)) & 0x7ffffffffffffull;
    }
};

// the element at which a running sum passes what was asked
template <class T>
struct SaPlace {
    typename SaKey<T>::U key;
    uint64_t before_weight;   // of the elements in front of the first of its key
    uint64_t number;          // how many of its key stand in front of it
};

struct SaParams : cumo_hip_sample_t {
    int unit_bits;
};

template <class T>
__global__ __launch_bounds__(kSaBlock) void sample_kernel(SaParams p) {
    typedef SaKey<T> Key;
    typedef typename Key::U U;
    __shared__ uint64_t counts[kSaBins], weights[kSaBins];
    __shared__ T wave_max[kSaBlock / 64];
    __shared__ uint32_t wave_nan[kSaBlock / 64], wave_count[kSaBlock / 64];
    __shared__ uint64_t shared_place[3], shared_sum;
    float_tables_prepare();
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    for (uint64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T* x = reinterpret_cast<const T*>(p.x + (int64_t)row * p.x_step);
        T m = -INFINITY;
        bool nan = false;
        for (uint64_t i = tid; i < p.n; i += kSaBlock) {
            const T v = x[i];
            nan |= v != v;
            m = v > m ? v : m;
        }
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) {
            const T o = __shfl_xor(m, d);
            m = o > m ? o : m;
        }
        const bool wave_has_nan = __ballot(nan) != 0;
        __syncthreads();
        if (lane == 0) {
            wave_max[wave] = m;
            wave_nan[wave] = wave_has_nan;
        }
        __syncthreads();
        nan = false;
        for (int w = 0; w < kSaBlock / 64; ++w) {
            m = wave_max[w] > m ? wave_max[w] : m;
            nan |= wave_nan[w] != 0;
        }
        if (nan || m == (T)-INFINITY) {   // (the same for the whole block)
            if (tid == 0) p.out[row] = -1;
            continue;
        }
        const double temperature = sa_number(p.temperature, row);
        const bool greedy = !(temperature > 0.0);
        SaWeight weight;
        weight.max = (double)m;
        weight.rate = 1.44269504088896338700e+00 / (greedy ? 1.0 : temperature);
        weight.unit = __longlong_as_double((long long)(1023 + p.unit_bits) << 52);

        // the element at which the running count (weight) first exceeds t, which the whole sum does
        auto find = [&](bool by_weight, uint64_t t) {
            SaPlace<T> at;
            U prefix = 0;
            uint64_t before = 0, before_weight = 0, number = 0;
            for (int shift = (int)sizeof(U) * 8 - kSaDigit; shift >= 0; shift -= kSaDigit) {
                if (tid < kSaBins) counts[tid] = weights[tid] = 0;
                __syncthreads();
                for (uint64_t i = tid; i < p.n; i += kSaBlock) {
                    const U k = Key::of(x[i]);
                    // (a shift by the whole width would not be one: the first digit compares nothing)
                    if (shift + kSaDigit < (int)sizeof(U) * 8 && (k >> (shift + kSaDigit)) != prefix) continue;
                    const uint32_t digit = (uint32_t)(k >> shift) & (kSaBins - 1);
                    atomicAdd((unsigned long long*)&counts[digit], 1ull);
                    atomicAdd((unsigned long long*)&weights[digit], (unsigned long long)weight.of((double)x[i]));
                }
                __syncthreads();
                if (tid == 0) {
                    uint64_t run = before, run_weight = before_weight;
                    int digit = kSaBins - 1;
                    for (; digit > 0; --digit) {
                        const uint64_t next = run + (by_weight ? weights[digit] : counts[digit]);
                        if (next > t) break;
                        run = next;
                        run_weight += weights[digit];
                    }
                    shared_place[0] = (uint64_t)digit;
                    shared_place[1] = run;
                    shared_place[2] = run_weight;
                }
                __syncthreads();
                prefix = (U)((prefix << kSaDigit) | (U)shared_place[0]);
                before = shared_place[1];
                before_weight = shared_place[2];
                if (shift == 0) {
                    const uint64_t one = by_weight ? weights[shared_place[0]] / counts[shared_place[0]] : 1;
                    number = (t - before) / (one ? one : 1);
                }
                __syncthreads();
            }
            at.key = prefix;
            at.before_weight = before_weight;
            at.number = number;
            return at;
        };
        auto sum_of = [&](double least) {   // of the weights whose share is `least` or more
            uint64_t mine = 0;
            for (uint64_t i = tid; i < p.n; i += kSaBlock) {
                const double s = weight.share((double)x[i]);
                mine += s >= least ? weight.units(s) : 0;
            }
            if (tid == 0) shared_sum = 0;
            __syncthreads();
            atomicAdd((unsigned long long*)&shared_sum, (unsigned long long)mine);
            __syncthreads();
            const uint64_t all = shared_sum;
            __syncthreads();
            return all;
        };

        const double k_given = sa_number(p.top_k, row), p_given = sa_number(p.top_p, row), m_given = sa_number(p.min_p, row);
        const uint64_t top_k = greedy ? 1 : (k_given > 0.0 && k_given < (double)p.n ? (uint64_t)k_given : p.n);
        uint64_t sum;
        if (top_k < p.n) {
            const SaPlace<T> at = find(false, top_k - 1);
            sum = at.before_weight + (at.number + 1) * weight.of((double)Key::value(at.key));
        } else {
            sum = sum_of(0.0);
        }
        if (p_given < 1.0) {
            double want = ceil((p_given > 0.0 ? p_given : 0.0) * (double)sum);
            want = want < 1.0 ? 1.0 : want;
            const uint64_t t = (uint64_t)want - 1;
            const SaPlace<T> at = find(true, t < sum ? t : sum - 1);
            sum = at.before_weight + (at.number + 1) * weight.of((double)Key::value(at.key));
        }
        if (m_given > 0.0) {
            const uint64_t likely = sum_of(m_given < 1.0 ? m_given : 1.0);
            sum = likely < sum ? likely : sum;
        }
        const double u = sa_number(p.u, row);
        const double want = floor((u > 0.0 ? u : 0.0) * (double)sum);
        const SaPlace<T> at = find(true, want < (double)sum ? (uint64_t)want < sum ? (uint64_t)want : sum - 1 : sum - 1);

        // the element of that key with `number` before it, in order of the index
        uint64_t left = at.number;
        for (uint64_t first = 0; first < p.n; first += kSaBlock) {
            const uint64_t i = first + tid;
            const bool hit = i < p.n && Key::of(x[i]) == at.key;
            const uint64_t hits = __ballot(hit);
            if (lane == 0) wave_count[wave] = (uint32_t)__popcll(hits);
            __syncthreads();
            uint32_t ahead = (uint32_t)__popcll(hits & ((1ull << lane) - 1)), all = 0;
            for (uint32_t w = 0; w < kSaBlock / 64; ++w) {
                ahead += w < wave ? wave_count[w] : 0;
                all += wave_count[w];
            }
            if (hit && ahead == left) p.out[row] = (int32_t)i;
            __syncthreads();
            if (left < all) break;
            left -= all;
        }
    }
}

}  // namespace
}  // namespace cumo_hip

using namespace cumo_hip;

extern "C" int cumo_hip_sample_kernel_launch(int type, const cumo_hip_sample_t* d) {
    if (d->rows == 0) return CUMO_HIP_OK;
    SaParams p;
    std::memset(&p, 0, sizeof(p));
    static_cast<cumo_hip_sample_t&>(p) = *d;
    int bits = 0;
    while ((1ull << bits) < d->n) ++bits;
    p.unit_bits = 62 - bits < 50 ? 62 - bits : 50;
    const dim3 grid((unsigned)(d->rows < 65536 ? d->rows : 65536)), block(kSaBlock);
    if (type == 0) hipLaunchKernelGGL((sample_kernel<float>), grid, block, 0, current_stream(), p);
    else hipLaunchKernelGGL((sample_kernel<double>), grid, block, 0, current_stream(), p);
    cumo_cuda_runtime_check_kernel_launch();
    return CUMO_HIP_OK;
}
