// Root-mean-square normalisation of rows, with the addition of a residual before it, an 8-bit form of the result and the
// gradients:
//   s = x + residual        r = 1 / sqrt(sum(s^2) / n + eps)        y = s r w
//   c = r^2 sum(g w s) / n  gx = r (g w - s c) + gsum               gw = sum over rows of g s r
// (gx: with u = s r the derivative of u_i by s_j is r (delta_ij - u_i u_j / n).)
//
// Memory bounds all of them: a row is read once into the registers of the lanes that share it, its sums meet across those
// lanes, and what is computed from them is written once. The sums, and everything between them and the one rounding of a
// result, are in double: a square of a float is exact there, and the vector units do a hundred such operations in the time
// that an element's bytes take. SFloat [8192,4096], with a residual, a sum and a weight: 87 us (6.2 TB/s, what an addition of two
// large arrays reaches); in 8 bits [8192,4095] 80 us (5.4; the vector units are busy for more than half of it), and 30 us back
// (5.5); gradients with gsum 94 + 5 us (5.7 and the weight's parts); DFloat [131072,257] gradients 200 + 5 (5.4), [8192,2047] in 8 bits 76
// and 31 back. One row of 4096: 3.5 us, the launch's.
#include "common.h"

namespace cumo_hip {
namespace {

__device__ __forceinline__ double rn_add(double a, double b) { return a + b; }
__device__ __forceinline__ double rn_max_nan(double a, double b) { return (a != a) ? a : ((b != b) ? b : (a > b ? a : b)); }

// Combines K values a lane over the TPR lanes that share a row, in a fixed order; every lane gets the results.
template <int TPR, int BLOCK, int K, class F>
__device__ __forceinline__ void rn_allreduce(double (&v)[K], F f) {
    constexpr int SPAN = TPR < 64 ? TPR : 64;
#pragma unroll
    for (int m = SPAN >> 1; m > 0; m >>= 1) {
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] = f(v[k], __shfl_xor(v[k], m));
    }
    if constexpr (TPR > 64) {
        __shared__ double slot[BLOCK / 64][K];
        __syncthreads();  // the slots may still be read from the previous use
        if ((threadIdx.x & 63) == 0) {
#pragma unroll
            for (int k = 0; k < K; ++k) slot[threadIdx.x >> 6][k] = v[k];
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] = slot[0][k];
#pragma unroll
        for (int w = 1; w < BLOCK / 64; ++w) {
#pragma unroll
            for (int k = 0; k < K; ++k) v[k] = f(v[k], slot[w][k]);
        }
    }
}

// How rows are written: through the second-level cache where their pieces are whole (store_form.h); else past it, or, `meet`, plainly
// where rows follow one another, so that a row's end and the next one's start meet in that cache: for y beside s. us past it / plainly,
// with a residual: SFloat [8192,4095] 94 / 88, [8192,4092] 96 / 85, [32768,1001] 96 / 100, [131072,257] 134 / 100, DFloat [131072,257]
// 223 / 209, [8192,2047] 97 / 86. Otherwise it does not pay: 8 bits [8192,4092] 77 / 84, dequantize [8192,4095] 30 / 35, y alone [8192,4095]
// 49 / 53, gradients DFloat [131072,257] 200 / 218.
struct RnStore {
    bool pieces, meet;
    __device__ __forceinline__ RnStore(const char* p, int64_t step, bool through, bool may_meet) : pieces(through && store_pieces(p, step)), meet(through && may_meet) {}
    template <bool NT, class Q>
    __device__ __forceinline__ void put(Q* at, Q v) const {
        if (NT && !pieces && meet) *at = v;
        else store_vector<NT>(at, v, pieces);
    }
};

// A row in the registers of TPR lanes: whole 128-bit vectors, lane l holding vectors l, l + TPR, ..., and, one to a lane, the
// elements behind the last whole one. What is not there is 0.
template <class T, int TPR, int NV>
struct RnRow {
    static constexpr int V = 16 / (int)sizeof(T);
    typedef uint32_t u4 __attribute__((ext_vector_type(4)));
    union Vec { u4 q; T t[V]; __device__ Vec() {} };
    Vec x[NV];
    T last;

    // `whole` and `rest`: vectors, and elements behind them, of this lane's row, 0 where there is no such row. A lane without a
    // vector reads the row's first one (`any`: there is one), so that no branch stands between the loads.
    // It waits for them before it goes on (what is not there is made 0): a row's arrays come one after the other, a stretch of memory each
    // time. That suits kernels bound by memory alone, SFloat [8192,4096] with a residual 88 us, on their way together 90, DFloat [131072,257]
    // gradients 201, 213; 8 bits, with more to compute, 84 and 80.
    template <bool NT>
    __device__ __forceinline__ void load(const char* row, uint32_t lane, uint32_t whole, uint32_t rest, bool any) {
        if (any) {
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const uint32_t at = (uint32_t)k * TPR + lane;
                const u4* from = reinterpret_cast<const u4*>(row + (at < whole ? at * 16u : 0u));
                x[k].q = NT ? __builtin_nontemporal_load(from) : *from;
            }
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const bool there = (uint32_t)k * TPR + lane < whole;
#pragma unroll
                for (int j = 0; j < V; ++j) x[k].t[j] = there ? x[k].t[j] : (T)0;
            }
        } else {
#pragma unroll
            for (int k = 0; k < NV; ++k) {
#pragma unroll
                for (int j = 0; j < V; ++j) x[k].t[j] = (T)0;
            }
        }
        last = lane < rest ? reinterpret_cast<const T*>(row)[whole * V + lane] : (T)0;
    }
    // the same in two steps: what is not there is something else until it is cut off
    template <bool NT>
    __device__ __forceinline__ void send_for(const char* row, uint32_t lane, uint32_t whole, uint32_t rest, bool any) {
        if (any) {
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const uint32_t at = (uint32_t)k * TPR + lane;
                const u4* from = reinterpret_cast<const u4*>(row + (at < whole ? at * 16u : 0u));
                x[k].q = NT ? __builtin_nontemporal_load(from) : *from;
            }
        } else {
            fill((T)0);
        }
        last = lane < rest ? reinterpret_cast<const T*>(row)[whole * V + lane] : (T)0;
    }
    __device__ __forceinline__ void trim(uint32_t lane, uint32_t whole) {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const bool there = (uint32_t)k * TPR + lane < whole;
#pragma unroll
            for (int j = 0; j < V; ++j) x[k].t[j] = there ? x[k].t[j] : (T)0;
        }
    }
    __device__ __forceinline__ void fill(T v) {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
#pragma unroll
            for (int j = 0; j < V; ++j) x[k].t[j] = v;
        }
        last = v;
    }
    template <bool NT>
    __device__ __forceinline__ void store(char* row, uint32_t lane, uint32_t whole, uint32_t rest, RnStore to) const {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const uint32_t at = (uint32_t)k * TPR + lane;
            if (at < whole) to.put<NT>(reinterpret_cast<u4*>(row + at * 16u), x[k].q);
            if constexpr (NV > 4) __builtin_amdgcn_sched_barrier(0);
        }
        if (lane < rest) reinterpret_cast<T*>(row)[whole * V + lane] = last;
    }
    // 8-bit integers, V of them side by side a lane: on any boundary
    template <class F>
    __device__ __forceinline__ void store_bytes(char* row, uint32_t lane, uint32_t whole, uint32_t rest, F f) const {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const uint32_t at = (uint32_t)k * TPR + lane;
            int8_t b[V];
#pragma unroll
            for (int j = 0; j < V; ++j) b[j] = f(k, j);
            if (at < whole) __builtin_memcpy(row + at * (uint32_t)V, b, V);
            if constexpr (NV > 4) __builtin_amdgcn_sched_barrier(0);
        }
        if (lane < rest) row[whole * V + lane] = f(NV, 0);
    }
    // The numbers as if they came anew: what has been worked out from them, their conversions to double above all, is not kept in
    // registers beside them until it is wanted again (232 registers a lane in the gradients' kernel, 1024 lanes spilled).
    __device__ __forceinline__ void forget() {
        each([](T& v, int, int) { asm("" : "+v"(v)); });
    }
    __device__ __forceinline__ T at(int k, int j) const { return k < NV ? x[k < NV ? k : 0].t[j] : last; }
    template <class F>
    __device__ __forceinline__ void each(F f) {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
#pragma unroll
            for (int j = 0; j < V; ++j) f(x[k].t[j], k, j);
            if constexpr (NV > 4) __builtin_amdgcn_sched_barrier(0);  // (else what all vectors need is worked out side by side, and spilled)
        }
        f(last, NV, 0);
    }
};

struct RnParams : cumo_hip_rmsnorm_t {
    bool y_through, sum_through;  // whether rows may be written through (StoreRows)
};

// A row in 8 bits: y = p a, of which p is an element's, exact for SFloat, and a the row's (DFloat: 1, as s w can overflow where y
// does not). The nearest integer of p b is what the sum with 1.5 * 2^52 leaves in its lower 32 bits; b: a / scale, or 0 where the
// row's bytes are all 0 (a scale of 0, of infinity, of NaN), and so is then `kept`. A scale below the normal numbers can be half its
// row's largest / 127, rounded: then the bytes end at 127. SFloat [8192,4096] 47 us; 58 with y itself,
// its quotient and its limits in double for each element.
template <class T>
__device__ __forceinline__ double rn_product(T s, double r, T w) { return sizeof(T) == 4 ? (double)s * (double)w : (double)s * r * (double)w; }
template <class T>
__device__ __forceinline__ double rn_common(double r) { return sizeof(T) == 4 ? r : 1.0; }
__device__ __forceinline__ int8_t rn_byte(double p, double b, int kept) {
    const int z = (int)__double_as_longlong(__builtin_fma(p, b, 6755399441055744.0)) & kept;
    return (int8_t)(z < -127 ? -127 : z > 127 ? 127 : z);
}
// 1 / scale, where there is something to divide; `lift` a power of two for p and scale, with which it is no infinity
template <class T>
__device__ __forceinline__ double rn_lift(T scale) { return sizeof(T) == 8 && (double)scale < 0x1p-1000 ? 0x1p200 : 1.0; }
template <class T>
__device__ __forceinline__ double rn_inverse(T scale, double lift) {
    return scale > (T)0 && scale < (T)INFINITY ? 1.0 / ((double)scale * lift) : 0.0;
}

template <class T, int TPR, int NV, int BLOCK, bool Q8, bool NT>
__global__ __launch_bounds__(BLOCK) void rmsnorm_kernel(RnParams p) {
    typedef RnRow<T, TPR, NV> Row;
    constexpr int RPB = BLOCK / TPR;  // rows a block
    const uint32_t lane = threadIdx.x % TPR;
    const uint32_t vectors = (uint32_t)p.n / Row::V, behind = (uint32_t)p.n % Row::V;
    // the weight stays in registers from row to row where there are enough; lanes with sixteen vectors read it again for each
    constexpr bool HELD = NV <= 4;
    Row w;
    auto read_weight = [&] {
        if (p.weight) w.template load<false>(p.weight, lane, vectors, behind, vectors != 0);
        else w.fill((T)1);
    };
    if constexpr (HELD) read_weight();
    const RnStore to_y(p.y, p.y_step, p.y_through, p.sum != nullptr), to_sum(p.sum, p.sum_step, p.sum_through, !Q8);
    for (uint64_t first = (uint64_t)blockIdx.x * RPB; first < p.rows; first += (uint64_t)gridDim.x * RPB) {
        const uint64_t mine = first + threadIdx.x / TPR;
        const bool there = mine < p.rows;
        const int64_t row = there ? (int64_t)mine : 0;
        const uint32_t whole = there ? vectors : 0, rest = there ? behind : 0;
        Row s;
        if constexpr (Q8) s.template send_for<NT>(p.x + row * p.x_step, lane, whole, rest, vectors != 0);
        else s.template load<NT>(p.x + row * p.x_step, lane, whole, rest, vectors != 0);
        if (p.residual) {
            Row add;
            if constexpr (Q8) add.template send_for<NT>(p.residual + row * p.residual_step, lane, whole, rest, vectors != 0);
            else add.template load<NT>(p.residual + row * p.residual_step, lane, whole, rest, vectors != 0);
            s.each([&](T& v, int k, int j) { v += add.at(k, j); });
            s.template store<NT>(p.sum + row * p.sum_step, lane, whole, rest, to_sum);
        }
        if constexpr (Q8) s.trim(lane, whole);
        double q[1] = {0.0};
        s.each([&](T& v, int, int) { q[0] = __builtin_fma((double)v, (double)v, q[0]); });
        rn_allreduce<TPR, BLOCK>(q, rn_add);
        const double r = 1.0 / sqrt(q[0] / (double)p.n + p.eps);
        if constexpr (!HELD) read_weight();
        s.forget();
        w.forget();
        if constexpr (Q8) {
            double most[1] = {0.0};
            bool nan = false;
            s.each([&](T& v, int k, int j) {
                const double product = rn_product(v, r, w.at(k, j));
                nan |= product != product;
                most[0] = __builtin_fmax(most[0], __builtin_fabs(product));
            });
            most[0] = nan ? __builtin_nan("") : most[0];
            rn_allreduce<TPR, BLOCK>(most, rn_max_nan);
            if constexpr (NV > 4) {
                s.forget();
                w.forget();
            }
            const T scale = (T)(most[0] * rn_common<T>(r) / 127.0);
            if (there && lane == 0) reinterpret_cast<T*>(p.scale)[row] = scale;
            const double lift = rn_lift(scale), inverse = rn_inverse(scale, lift), b = rn_common<T>(r) * inverse, raised = r * lift;
            const int kept = inverse > 0.0 ? -1 : 0;
            s.store_bytes(p.y + row * p.y_step, lane, whole, rest, [&](int k, int j) { return rn_byte(rn_product(s.at(k, j), raised, w.at(k, j)), b, kept); });
        } else {
            s.each([&](T& v, int k, int j) { v = (T)((double)v * r * (double)w.at(k, j)); });
            s.template store<NT>(p.y + row * p.y_step, lane, whole, rest, to_y);
        }
    }
}

// Rows that no block's registers hold: read again from the caches for each of their sums. With a residual SFloat [512,40000] 97 us
// (3.4 TB/s), [256,131072] 224 (2.4), where [2048,16384] in registers takes 85 (6.3).
constexpr int kRnWide = 1024;
template <class T, bool Q8>
__global__ __launch_bounds__(kRnWide) void rmsnorm_long_kernel(cumo_hip_rmsnorm_t p) {
    for (uint64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T* x = reinterpret_cast<const T*>(p.x + (int64_t)row * p.x_step);
        const T* res = p.residual ? reinterpret_cast<const T*>(p.residual + (int64_t)row * p.residual_step) : nullptr;
        const T* w = reinterpret_cast<const T*>(p.weight);
        T* sum = p.sum ? reinterpret_cast<T*>(p.sum + (int64_t)row * p.sum_step) : nullptr;
        double q[1] = {0.0};
        for (uint64_t i = threadIdx.x; i < p.n; i += kRnWide) {
            const T s = res ? x[i] + res[i] : x[i];
            if (sum) sum[i] = s;
            q[0] = __builtin_fma((double)s, (double)s, q[0]);
        }
        rn_allreduce<kRnWide, kRnWide>(q, rn_add);
        const double r = 1.0 / sqrt(q[0] / (double)p.n + p.eps);
        const T* from = sum ? sum : x;
        auto product = [&](uint64_t i, double by) { return rn_product(from[i], by, w ? w[i] : (T)1); };
        if constexpr (Q8) {
            double most[1] = {0.0};
            for (uint64_t i = threadIdx.x; i < p.n; i += kRnWide) most[0] = rn_max_nan(most[0], fabs(product(i, r)));
            rn_allreduce<kRnWide, kRnWide>(most, rn_max_nan);
            const T scale = (T)(most[0] * rn_common<T>(r) / 127.0);
            if (threadIdx.x == 0) reinterpret_cast<T*>(p.scale)[row] = scale;
            const double lift = rn_lift(scale), inverse = rn_inverse(scale, lift), b = rn_common<T>(r) * inverse, raised = r * lift;
            const int kept = inverse > 0.0 ? -1 : 0;
            int8_t* y = reinterpret_cast<int8_t*>(p.y + (int64_t)row * p.y_step);
            for (uint64_t i = threadIdx.x; i < p.n; i += kRnWide) y[i] = rn_byte(product(i, raised), b, kept);
        } else {
            T* y = reinterpret_cast<T*>(p.y + (int64_t)row * p.y_step);
            for (uint64_t i = threadIdx.x; i < p.n; i += kRnWide) y[i] = (T)((double)from[i] * r * (w ? (double)w[i] : 1.0));
        }
    }
}

// V numbers to a lane and turn: 4 (DFloat 2) bytes in, 16 bytes out
constexpr int kDqBlock = 256;
template <class T, int TPR, bool NT>
__global__ __launch_bounds__(kDqBlock) void dequantize_kernel(cumo_hip_dequantize_t p, bool through) {
    typedef RnRow<T, TPR, 1> Row;
    constexpr int RPB = kDqBlock / TPR;
    const uint32_t lane = threadIdx.x % TPR;
    const uint64_t vectors = p.n / Row::V;
    const RnStore to(p.y, p.y_step, through, false);
    for (uint64_t row = (uint64_t)blockIdx.x * RPB + threadIdx.x / TPR; row < p.rows; row += (uint64_t)gridDim.x * RPB) {
        const int8_t* q = reinterpret_cast<const int8_t*>(p.q + (int64_t)row * p.q_step);
        char* y = p.y + (int64_t)row * p.y_step;
        const T scale = reinterpret_cast<const T*>(p.scale)[row];
        constexpr int U = 4;
        for (uint64_t k = lane; k < vectors; k += (uint64_t)TPR * U) {
            int8_t b[U][Row::V];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const uint64_t at = k + (uint64_t)u * TPR;
                __builtin_memcpy(b[u], q + (at < vectors ? at : k) * Row::V, Row::V);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const uint64_t at = k + (uint64_t)u * TPR;
                typename Row::Vec v;
#pragma unroll
                for (int j = 0; j < Row::V; ++j) v.t[j] = (T)b[u][j] * scale;
                if (at < vectors) to.template put<NT>(reinterpret_cast<typename Row::u4*>(y + at * 16), v.q);
            }
        }
        if (lane < p.n % Row::V) reinterpret_cast<T*>(y)[vectors * Row::V + lane] = (T)q[vectors * Row::V + lane] * scale;
    }
}

// ---- gradients ------------------------------------------------------------------------
// A block takes every gridDim-th group of rows, so that what its rows add to the weight's gradient stays in registers until its
// end; the blocks' parts, one row of doubles each, are added up by a second launch (or are the gradient, where one block has
// taken all rows). Which rows a block takes, and the order of both sums, go by the sizes alone.
struct RnGradParams : cumo_hip_rmsnorm_grad_t {
    double* parts;  // [gridDim.x][n]; NULL: the weight's gradient is written at once, or not wanted
    bool through;
};

template <class T, int NV, int BLOCK> constexpr bool kRnAhead = NV == 4 && (sizeof(T) == 4 || BLOCK > 256);

template <class T, int TPR, int NV, int BLOCK, bool NT>
__global__ __launch_bounds__(BLOCK) void rmsnorm_grad_kernel(RnGradParams p) {
    typedef RnRow<T, TPR, NV> Row;
    constexpr int RPB = BLOCK / TPR, V = Row::V;
    const uint32_t lane = threadIdx.x % TPR;
    const uint32_t vectors = (uint32_t)p.n / V, behind = (uint32_t)p.n % V;
    constexpr bool HELD = NV <= 4;  // (as in the forward kernel; here the weight's gradient takes registers too)
    Row w;
    auto read_weight = [&] {
        if (p.weight) w.template load<false>(p.weight, lane, vectors, behind, vectors != 0);
        else w.fill((T)1);
    };
    if constexpr (HELD) read_weight();
    double sum[NV + 1][V];
#pragma unroll
    for (int k = 0; k <= NV; ++k) {
#pragma unroll
        for (int j = 0; j < V; ++j) sum[k][j] = 0.0;
    }
    const RnStore to(p.gx, p.gx_step, p.through, false);
    // Where few blocks share a compute unit they read their next rows while they work on some: SFloat [4096,8192] 104 us without, 93
    // with (gsum: 128, 109), [32768,4096] 301, 273 (394, 370), [131072,257] 105, 98 (130, 124); DFloat of 256 lanes, three blocks, not:
    // [8192,2048] 69, 70, [131072,257] 170, 171.
    constexpr bool AHEAD = kRnAhead<T, NV, BLOCK>;
    Row next_s, next_g;
    auto read = [&](Row& s, Row& g, uint64_t first) {
        const uint64_t mine = first + threadIdx.x / TPR;
        const bool there = mine < p.rows;
        const int64_t row = there ? (int64_t)mine : 0;
        s.template send_for<NT>(p.s + row * p.s_step, lane, there ? vectors : 0, there ? behind : 0, vectors != 0);
        g.template send_for<NT>(p.g + row * p.g_step, lane, there ? vectors : 0, there ? behind : 0, vectors != 0);
    };
    if constexpr (AHEAD) read(next_s, next_g, (uint64_t)blockIdx.x * RPB);
    for (uint64_t first = (uint64_t)blockIdx.x * RPB; first < p.rows; first += (uint64_t)gridDim.x * RPB) {
        const uint64_t mine = first + threadIdx.x / TPR;
        const bool there = mine < p.rows;
        const int64_t row = there ? (int64_t)mine : 0;
        const uint32_t whole = there ? vectors : 0, rest = there ? behind : 0;
        Row s, g, gs;
        if constexpr (AHEAD) {
            s = next_s;
            g = next_g;
            read(next_s, next_g, first + (uint64_t)gridDim.x * RPB);
            s.trim(lane, whole);
            g.trim(lane, whole);
        } else {
            s.template load<NT>(p.s + row * p.s_step, lane, whole, rest, vectors != 0);
            g.template load<NT>(p.g + row * p.g_step, lane, whole, rest, vectors != 0);
        }
        auto read_gsum = [&] {
            if (p.gsum) gs.template load<NT>(p.gsum + row * p.gsum_step, lane, whole, rest, vectors != 0);
            else gs.fill((T)0);
        };
        if constexpr (HELD) read_gsum();
        else read_weight();
        w.forget();
        double q[2] = {0.0, 0.0};
        s.each([&](T& v, int k, int j) {
            q[0] = __builtin_fma((double)v, (double)v, q[0]);
            q[1] = __builtin_fma((double)g.at(k, j) * (double)w.at(k, j), (double)v, q[1]);
        });
        rn_allreduce<TPR, BLOCK>(q, rn_add);
        // (a row that is not there has no s: its r may be infinite, and 0 * infinity is no 0)
        const double r = there ? 1.0 / sqrt(q[0] / (double)p.n + p.eps) : 0.0;
        const double c = r * r * q[1] / (double)p.n;
        if constexpr (!HELD) read_gsum();
        s.forget();
        g.forget();
        w.forget();
        s.each([&](T& v, int k, int j) {
            const double gv = (double)g.at(k, j), sv = (double)v;
            sum[k][j] = __builtin_fma(gv * sv, r, sum[k][j]);
            v = (T)__builtin_fma(r, gv * (double)w.at(k, j) - sv * c, (double)gs.at(k, j));
        });
        s.template store<NT>(p.gx + row * p.gx_step, lane, whole, rest, to);
    }
    if (!p.gweight) return;
    // the rows that the block holds side by side
    __shared__ double other[RPB > 1 ? BLOCK : 1];
    const uint32_t slot = threadIdx.x / TPR;
    double* part = p.parts ? p.parts + (uint64_t)blockIdx.x * p.n : nullptr;
#pragma unroll
    for (int k = 0; k <= NV; ++k) {
#pragma unroll
        for (int j = 0; j < (k < NV ? V : 1); ++j) {
            double all = sum[k][j];
            if constexpr (RPB > 1) {
                __syncthreads();
                other[threadIdx.x] = all;
                __syncthreads();
                if (slot == 0) {
#pragma unroll
                    for (int i = 1; i < RPB; ++i) all += other[i * TPR + lane];
                }
            }
            const uint32_t at = k < NV ? ((uint32_t)k * TPR + lane) * V + j : vectors * V + lane;
            const bool mine = slot == 0 && (k < NV ? (uint32_t)k * TPR + lane < vectors : lane < behind);
            if (mine) {
                if (part) part[at] = all;
                else reinterpret_cast<T*>(p.gweight)[at] = (T)all;
            }
        }
    }
}

// Rows that no block's registers hold (more than 16387 SFloat, 8193 DFloat); r of each row is left for the weight's gradient. SFloat
// [1024,32768] with gsum and weight 239 + 54 + 7 us, DFloat [2048,16384] 263 + 129 + 5, [2048,8192] in registers 101 + 5.
template <class T>
__global__ __launch_bounds__(kRnWide) void rmsnorm_grad_long_kernel(cumo_hip_rmsnorm_grad_t p, double* rs) {
    for (uint64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T* g = reinterpret_cast<const T*>(p.g + (int64_t)row * p.g_step);
        const T* s = reinterpret_cast<const T*>(p.s + (int64_t)row * p.s_step);
        const T* gs = p.gsum ? reinterpret_cast<const T*>(p.gsum + (int64_t)row * p.gsum_step) : nullptr;
        const T* w = reinterpret_cast<const T*>(p.weight);
        T* gx = reinterpret_cast<T*>(p.gx + (int64_t)row * p.gx_step);
        double q[2] = {0.0, 0.0};
        for (uint64_t i = threadIdx.x; i < p.n; i += kRnWide) {
            const double si = (double)s[i], gw = (double)g[i] * (w ? (double)w[i] : 1.0);
            q[0] = __builtin_fma(si, si, q[0]);
            q[1] = __builtin_fma(gw, si, q[1]);
        }
        rn_allreduce<kRnWide, kRnWide>(q, rn_add);
        const double r = 1.0 / sqrt(q[0] / (double)p.n + p.eps);
        const double c = r * r * q[1] / (double)p.n;
        if (rs && threadIdx.x == 0) rs[row] = r;
        for (uint64_t i = threadIdx.x; i < p.n; i += kRnWide) {
            const double gw = (double)g[i] * (w ? (double)w[i] : 1.0);
            gx[i] = (T)__builtin_fma(r, gw - (double)s[i] * c, gs ? (double)gs[i] : 0.0);
        }
    }
}

// the weight's part of every blockIdx.y-th run of rows, by columns
template <class T>
__global__ __launch_bounds__(256) void rmsnorm_grad_columns_kernel(RnGradParams p, const double* rs, uint64_t per) {
    const uint64_t from = blockIdx.y * per, to = from + per < p.rows ? from + per : p.rows;
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < p.n; i += (uint64_t)gridDim.x * 256) {
        double sum = 0.0;
        for (uint64_t row = from; row < to; ++row) {
            const double g = (double)reinterpret_cast<const T*>(p.g + (int64_t)row * p.g_step)[i], s = (double)reinterpret_cast<const T*>(p.s + (int64_t)row * p.s_step)[i];
            sum = __builtin_fma(g * s, rs[row], sum);
        }
        p.parts[blockIdx.y * p.n + i] = sum;
    }
}

// [parts][n] down its columns: 16 columns a block, every lane of the 64 to a column taking every 64th part (64 columns a block
// and sixteen lanes to a column took 7.5 us for 768 parts of 4096, and as long for 257)
template <class T>
__global__ __launch_bounds__(1024) void rmsnorm_grad_parts_kernel(const double* parts, uint32_t n_parts, uint64_t n, T* out) {
    __shared__ double slot[16][16];
    const uint32_t column = threadIdx.x & 15, group = threadIdx.x >> 4;
    for (uint64_t first = (uint64_t)blockIdx.x * 16; first < n; first += (uint64_t)gridDim.x * 16) {
        const uint64_t i = first + column;
        double sum = 0.0;
        if (i < n) {
#pragma unroll 4
            for (uint32_t k = group; k < n_parts; k += 64) sum += parts[k * n + i];
        }
        // the wave's four groups, then the waves
        sum += __shfl_xor(sum, 16);
        sum += __shfl_xor(sum, 32);
        if ((group & 3) == 0) slot[group >> 2][column] = sum;
        __syncthreads();
        if (threadIdx.x < 16 && i < n) {
            sum = slot[0][column];
#pragma unroll
            for (int w = 1; w < 16; ++w) sum += slot[w][column];
            out[i] = (T)sum;
        }
        __syncthreads();
    }
}

unsigned rn_grid(uint64_t blocks, uint64_t most) { return (unsigned)(blocks < most ? blocks : most); }
dim3 rn_columns(uint64_t n) { return dim3(rn_grid((n + 15) / 16, 1u << 20)); }   // of the parts (a launch holds fewer than 2^32 lanes)

template <class T>
bool rn_through(const void* p, uint64_t rows, uint64_t n, int64_t step, bool nt) {
    StoreRows at(p, n * sizeof(T));
    at.dimension(rows, step);
    return at.through(nt);
}

// Lanes to a row: as many as hold it in four vectors each (the loads that a lane has on their way), two for 257 to 512 vectors, whose
// sum then takes one block's lanes; behind 4096 vectors sixteen. us, norm / gradients (not reading ahead), of 2^25 SFloat elements in rows of n, lanes x
// vectors as here and otherwise: n = 128, 8x4 44 / 72, 32x1 45 / 103; 1024, 64x4 47 / 68, 256x1 45 / 121; 2048, 256x2 39 / 81, 128x4
// 48 / 74; 4096, 256x4 43 / 80, 512x2 41 / 112; 8192, 512x4 49 / 104, 1024x2 47 / -, 256x8 - / 115; 32768, 512x16 61, 1024x8 105.
template <class T, int TPR, int NV, int BLOCK, bool Q8>
void rn_launch_one(RnParams p, bool nt, hipStream_t stream) {
    constexpr int RPB = BLOCK / TPR;
    const dim3 grid(rn_grid((p.rows + RPB - 1) / RPB, 256u * 64u)), block(BLOCK);
    if (nt) hipLaunchKernelGGL((rmsnorm_kernel<T, TPR, NV, BLOCK, Q8, true>), grid, block, 0, stream, p);
    else hipLaunchKernelGGL((rmsnorm_kernel<T, TPR, NV, BLOCK, Q8, false>), grid, block, 0, stream, p);
}

template <class T, bool Q8>
void rn_launch(const cumo_hip_rmsnorm_t& d, hipStream_t stream) {
    RnParams p;
    static_cast<cumo_hip_rmsnorm_t&>(p) = d;
    const bool nt = stream_past_caches(p.rows * p.n * (sizeof(T) * (p.residual ? 3 : 1) + (Q8 ? 1 : sizeof(T))));
    p.y_through = !Q8 && rn_through<T>(p.y, p.rows, p.n, p.y_step, nt);
    p.sum_through = p.sum && rn_through<T>(p.sum, p.rows, p.n, p.sum_step, nt);
    const uint64_t nv = p.n / (16 / sizeof(T));   // (whole vectors: the elements behind them have registers of their own)
    if (nv <= 8) rn_launch_one<T, 8, 1, 256, Q8>(p, nt, stream);
    else if (nv <= 16) rn_launch_one<T, 8, 2, 256, Q8>(p, nt, stream);
    else if (nv <= 32) rn_launch_one<T, 8, 4, 256, Q8>(p, nt, stream);
    else if (nv <= 64) rn_launch_one<T, 16, 4, 256, Q8>(p, nt, stream);
    else if (nv <= 128) rn_launch_one<T, 32, 4, 256, Q8>(p, nt, stream);
    else if (nv <= 256) rn_launch_one<T, 64, 4, 256, Q8>(p, nt, stream);
    else if (nv <= 512) rn_launch_one<T, 256, 2, 256, Q8>(p, nt, stream);
    else if (nv <= 1024) rn_launch_one<T, 256, 4, 256, Q8>(p, nt, stream);
    else if (nv <= 2048) rn_launch_one<T, 512, 4, 512, Q8>(p, nt, stream);
    else if (nv <= 4096) rn_launch_one<T, 1024, 4, 1024, Q8>(p, nt, stream);
    else if (nv <= 8192) rn_launch_one<T, 512, 16, 512, Q8>(p, nt, stream);
    else hipLaunchKernelGGL((rmsnorm_long_kernel<T, Q8>), dim3(rn_grid(p.rows, 1u << 20)), dim3(kRnWide), 0, stream, d);
    cumo_cuda_runtime_check_kernel_launch();
}

template <class T, int TPR>
void dq_launch_one(const cumo_hip_dequantize_t& d, hipStream_t stream) {
    constexpr int RPB = kDqBlock / TPR;
    const bool nt = stream_past_caches(d.rows * d.n * (1 + sizeof(T)));
    const bool through = rn_through<T>(d.y, d.rows, d.n, d.y_step, nt);
    const dim3 grid(rn_grid((d.rows + RPB - 1) / RPB, 256u * 64u)), block(kDqBlock);
    if (nt) hipLaunchKernelGGL((dequantize_kernel<T, TPR, true>), grid, block, 0, stream, d, through);
    else hipLaunchKernelGGL((dequantize_kernel<T, TPR, false>), grid, block, 0, stream, d, through);
    cumo_cuda_runtime_check_kernel_launch();
}

template <class T>
void dq_launch(const cumo_hip_dequantize_t& d, hipStream_t stream) {
    const uint64_t nv = d.n / (16 / sizeof(T));
    if (nv <= 32) dq_launch_one<T, 8>(d, stream);
    else if (nv <= 256) dq_launch_one<T, 64>(d, stream);
    else dq_launch_one<T, 256>(d, stream);
}

// Blocks that take the rows of a gradient, as many as the compute units hold at once: of 256 lanes three, two where they read ahead,
// of 512 one. More of them leave more parts and take turns. us at 256, 512, 768, 1024, 2048 blocks: DFloat [131072,257] 479, 304, 242, 323, 275;
// SFloat [131072,64] 50, 36, 34, 35, 46; reading ahead, [32768,4096] at 512 and 768 273, 325, [131072,257] 98, 109; [1024,8192], 512 lanes, at
// 256, 512, 768 42, 50, 54.
template <class T, int NV, int BLOCK> constexpr uint64_t kRnGradBlocks = BLOCK > 256 ? 256 : kRnAhead<T, NV, BLOCK> ? 512 : 768;

template <class T, int TPR, int NV, int BLOCK>
bool rn_grad_one(RnGradParams p, hipStream_t stream) {
    constexpr int RPB = BLOCK / TPR;
    const unsigned blocks = rn_grid((p.rows + RPB - 1) / RPB, p.gweight ? kRnGradBlocks<T, NV, BLOCK> : 256u * 64u);
    const bool nt = stream_past_caches(p.rows * p.n * sizeof(T) * (p.gsum ? 4 : 3));
    p.through = rn_through<T>(p.gx, p.rows, p.n, p.gx_step, nt);
    char* parts = nullptr;
    if (p.gweight && blocks > 1 && !(parts = cumo_cuda_runtime_malloc(blocks * p.n * sizeof(double)))) return false;
    p.parts = reinterpret_cast<double*>(parts);
    const dim3 grid(blocks), block(BLOCK);
    if (nt) hipLaunchKernelGGL((rmsnorm_grad_kernel<T, TPR, NV, BLOCK, true>), grid, block, 0, stream, p);
    else hipLaunchKernelGGL((rmsnorm_grad_kernel<T, TPR, NV, BLOCK, false>), grid, block, 0, stream, p);
    if (parts) {
        hipLaunchKernelGGL((rmsnorm_grad_parts_kernel<T>), rn_columns(p.n), dim3(1024), 0, stream, p.parts, (uint32_t)blocks, p.n,
                           reinterpret_cast<T*>(p.gweight));
        scratch_free(parts);
    }
    return true;
}

template <class T>
bool rn_grad_long(RnGradParams p, hipStream_t stream) {
    uint64_t runs = p.rows < 64 ? p.rows : 64;
    const uint64_t per = (p.rows + runs - 1) / runs;
    runs = (p.rows + per - 1) / per;
    char* memory = nullptr;
    if (p.gweight && !(memory = cumo_cuda_runtime_malloc((p.rows + runs * p.n) * sizeof(double)))) return false;
    double* rs = reinterpret_cast<double*>(memory);
    hipLaunchKernelGGL((rmsnorm_grad_long_kernel<T>), dim3(rn_grid(p.rows, 1u << 20)), dim3(kRnWide), 0, stream, p, rs);
    if (memory) {
        p.parts = rs + p.rows;
        hipLaunchKernelGGL((rmsnorm_grad_columns_kernel<T>), dim3(rn_grid((p.n + 255) / 256, 1u << 20), (unsigned)runs), dim3(256), 0, stream, p, rs, per);
        hipLaunchKernelGGL((rmsnorm_grad_parts_kernel<T>), rn_columns(p.n), dim3(1024), 0, stream, p.parts, (uint32_t)runs, p.n,
                           reinterpret_cast<T*>(p.gweight));
        scratch_free(memory);
    }
    return true;
}

template <class T>
int rn_grad(const cumo_hip_rmsnorm_grad_t& d, hipStream_t stream) {
    RnGradParams p;
    static_cast<cumo_hip_rmsnorm_grad_t&>(p) = d;
    p.parts = nullptr;
    p.through = false;
    const uint64_t nv = p.n / (16 / sizeof(T));   // (whole vectors: the elements behind them have registers of their own)
    bool ok = true;
    if (p.rows == 0) {
        if (p.gweight)
            hipLaunchKernelGGL((rmsnorm_grad_parts_kernel<T>), rn_columns(p.n), dim3(1024), 0, stream, nullptr, 0u, p.n, reinterpret_cast<T*>(p.gweight));
    }
    else if (nv <= 8) ok = rn_grad_one<T, 8, 1, 256>(p, stream);
    else if (nv <= 16) ok = rn_grad_one<T, 8, 2, 256>(p, stream);
    else if (nv <= 32) ok = rn_grad_one<T, 8, 4, 256>(p, stream);
    else if (nv <= 64) ok = rn_grad_one<T, 16, 4, 256>(p, stream);
    else if (nv <= 128) ok = rn_grad_one<T, 32, 4, 256>(p, stream);
    else if (nv <= 256) ok = rn_grad_one<T, 64, 4, 256>(p, stream);
    else if (nv <= 512) ok = rn_grad_one<T, 256, 2, 256>(p, stream);
    else if (nv <= 1024) ok = rn_grad_one<T, 256, 4, 256>(p, stream);
    else if (nv <= 2048) ok = rn_grad_one<T, 512, 4, 512>(p, stream);
    else if (nv <= 4096) ok = rn_grad_one<T, 512, 8, 512>(p, stream);
    else ok = rn_grad_long<T>(p, stream);
    cumo_cuda_runtime_check_kernel_launch();
    return ok ? CUMO_HIP_OK : CUMO_HIP_ERROR_OUT_OF_MEMORY;
}

}  // namespace
}  // namespace cumo_hip

using namespace cumo_hip;

extern "C" void cumo_hip_rmsnorm_kernel_launch(int type, int quantised, const cumo_hip_rmsnorm_t* d) {
    hipStream_t stream = current_stream();
    if (type == 0) quantised ? rn_launch<float, true>(*d, stream) : rn_launch<float, false>(*d, stream);
    else quantised ? rn_launch<double, true>(*d, stream) : rn_launch<double, false>(*d, stream);
}

extern "C" void cumo_hip_dequantize_kernel_launch(int type, const cumo_hip_dequantize_t* d) {
    if (type == 0) dq_launch<float>(*d, current_stream());
    else dq_launch<double>(*d, current_stream());
}

extern "C" int cumo_hip_rmsnorm_grad_kernel_launch(int type, const cumo_hip_rmsnorm_grad_t* d) {
    return type == 0 ? rn_grad<float>(*d, current_stream()) : rn_grad<double>(*d, current_stream());
}
