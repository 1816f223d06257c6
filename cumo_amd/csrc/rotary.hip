// Rotary positions: pairs (u, v) of a head's elements turned by t = position * frequency,
//   (u cos t - v sin t, v cos t + u sin t) * amplitude
// (the inverse turn, which is the gradient, by -t), whatever is behind the pairs copied.
//
// Memory bounds it: an element is read and written once. The angle of a far position wants more than 32 bits (131072 * 1 radian rounded to a
// float is off by 2^-8), so it is a double, and what is worked out from it too: the remainder of a quarter turn by two fused steps, sine
// and cosine by their series on an eighth of a turn either way. A lane keeps them for the heads that it takes. SFloat 4 x 4096 x 32 heads of 96,
// neighbours: 74 us, 5.4 TB/s; 64 x 1 x 32 of 128: 3.5, the launch's.
#include "common.h"

namespace cumo_hip {
namespace {

// sin x and cos x for |x| < 2^50, NaN otherwise. k quarter turns: x - k * 1.57... is exact (both are multiples of 2^-52, and nearer
// than a turn), pi / 2 goes on with 6.1e-17. k comes from a rounded product: far from 0 the quarter next to the nearest is taken at times (|r| up to
// 1.004 pi / 4 at 2^44, 1.21 near 2^50), so from there on what is left is turned back once more. The first term left out is r^19 / 19! and
// r^18 / 18!, below 3e-18, for SFloat r^13 / 13! and r^14 / 14!, below 8e-12.
template <bool LONG>
__device__ __forceinline__ void rt_sincos(double x, double* s, double* c) {
    double k = __builtin_rint(x * 0.63661977236758134308);
    double r = __builtin_fma(-k, 1.57079632679489661923, x);
    r = __builtin_fma(-k, 6.123233995736766036e-17, r);
    if (__builtin_fabs(x) >= 0x1p44) {
        const double more = __builtin_rint(r * 0.63661977236758134308);
        k += more;
        r = __builtin_fma(-more, 1.57079632679489661923, r);
        r = __builtin_fma(-more, 6.123233995736766036e-17, r);
    }
    const double z = r * r;
    double ps, pc;
    if constexpr (LONG) {
        ps = 1.0 / 355687428096000.0;                                  // 17!
        ps = __builtin_fma(ps, z, -1.0 / 1307674368000.0);             // 15!
        ps = __builtin_fma(ps, z, 1.0 / 6227020800.0);                 // 13!
        ps = __builtin_fma(ps, z, -1.0 / 39916800.0);                  // 11!
        pc = 1.0 / 20922789888000.0;                                   // 16!
        pc = __builtin_fma(pc, z, -1.0 / 87178291200.0);               // 14!
        pc = __builtin_fma(pc, z, 1.0 / 479001600.0);                  // 12!
    } else {
        ps = -1.0 / 39916800.0;
        pc = 1.0 / 479001600.0;
    }
    ps = __builtin_fma(ps, z, 1.0 / 362880.0);
    ps = __builtin_fma(ps, z, -1.0 / 5040.0);
    ps = __builtin_fma(ps, z, 1.0 / 120.0);
    ps = __builtin_fma(ps, z, -1.0 / 6.0);
    pc = __builtin_fma(pc, z, -1.0 / 3628800.0);
    pc = __builtin_fma(pc, z, 1.0 / 40320.0);
    pc = __builtin_fma(pc, z, -1.0 / 720.0);
    pc = __builtin_fma(pc, z, 1.0 / 24.0);
    pc = __builtin_fma(pc, z, -0.5);
    const double sn = __builtin_fma(ps * z, r, r), cs = __builtin_fma(pc, z, 1.0);
    const int turn = __builtin_fabs(x) < 0x1p50 ? (int)((int64_t)k & 3) : 0;
    double a = turn & 1 ? cs : sn, b = turn & 1 ? sn : cs;
    a = turn & 2 ? -a : a;
    b = (turn + 1) & 2 ? -b : b;
    const double bad = __builtin_fabs(x) < 0x1p50 ? 0.0 : __builtin_nan("");
    *s = a + bad;
    *c = b + bad;
}

struct RtParams : cumo_hip_rotary_t {
    uint32_t per;     // heads that a lane takes
    uint32_t chunks;  // such groups of heads
    uint32_t turns;   // pieces of W pairs
    uint32_t copies;  // pieces of C elements behind the pairs
};

// N numbers on any boundary of their type
template <class T, int N>
struct __attribute__((aligned(sizeof(T) * N))) RtVec {
    T t[N];
    template <bool NT>
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (NT && sizeof(t) == 16) *reinterpret_cast<store_u4*>(t) = __builtin_nontemporal_load(reinterpret_cast<const store_u4*>(p));
        else __builtin_memcpy(t, p, sizeof(t));
    }
    template <bool NT>
    __device__ __forceinline__ void store(T* p) const {
        if constexpr (NT && sizeof(t) == 16) __builtin_nontemporal_store(*reinterpret_cast<const store_u4*>(t), reinterpret_cast<store_u4*>(p));
        else __builtin_memcpy(p, t, sizeof(t));
    }
};

// A lane takes W pairs, two vectors of W (neighbours: one of 2 W), or C elements behind the pairs, of `per` heads in a row: U of them are read
// before the first is written. Lanes beside each other take pieces beside each other.
template <class T, int W, int C, bool NEIGHBOURS, int U, bool NT>
__global__ __launch_bounds__(256) void rotary_kernel(RtParams p) {
    const uint32_t pieces = p.turns + p.copies;
    const uint64_t total = p.batch * p.time * p.chunks * pieces;
    for (uint64_t item = (uint64_t)blockIdx.x * 256 + threadIdx.x; item < total; item += (uint64_t)gridDim.x * 256) {
        const uint32_t piece = (uint32_t)(item % pieces);
        const uint64_t rest = item / pieces;
        const uint32_t first = (uint32_t)(rest % p.chunks) * p.per;
        const uint64_t token = rest / p.chunks;
        const uint64_t b = token / p.time, t = token - b * p.time;
        const char* x = p.x + (int64_t)b * p.x_step[0] + (int64_t)t * p.x_step[1] + (int64_t)first * p.x_step[2];
        char* y = p.y + (int64_t)b * p.y_step[0] + (int64_t)t * p.y_step[1] + (int64_t)first * p.y_step[2];
        const uint32_t n = p.heads - first < p.per ? (uint32_t)(p.heads - first) : p.per;
        auto from = [&](uint32_t h) { return reinterpret_cast<const T*>(x + (int64_t)(h < n ? h : n - 1) * p.x_step[2]); };
        auto to = [&](uint32_t h) { return reinterpret_cast<T*>(y + (int64_t)h * p.y_step[2]); };
        if (piece < p.turns) {
            const double at = (double)p.positions[token];
            double sn[W], cs[W];
#pragma unroll
            for (int j = 0; j < W; ++j) {
                rt_sincos<sizeof(T) == 8>(at * p.frequencies[(uint64_t)piece * W + j], &sn[j], &cs[j]);
                sn[j] *= p.inverse ? -p.amplitude : p.amplitude;
                cs[j] *= p.amplitude;
            }
            auto turn = [&](T& u, T& v, int j) {
                const double l = (double)u, r = (double)v;
                u = (T)__builtin_fma(l, cs[j], -(r * sn[j]));
                v = (T)__builtin_fma(r, cs[j], l * sn[j]);
            };
            for (uint32_t h = 0; h < n; h += U) {
                if constexpr (NEIGHBOURS) {
                    const uint64_t one = (uint64_t)piece * W * 2;
                    RtVec<T, 2 * W> a[U];
#pragma unroll
                    for (int u = 0; u < U; ++u) a[u].template load<NT>(from(h + u) + one);
#pragma unroll
                    for (int u = 0; u < U; ++u) {
#pragma unroll
                        for (int j = 0; j < W; ++j) turn(a[u].t[2 * j], a[u].t[2 * j + 1], j);
                        if (h + u < n) a[u].template store<NT>(to(h + u) + one);
                    }
                } else {
                    const uint64_t one = (uint64_t)piece * W, two = one + p.pairs;
                    RtVec<T, W> a[U], d[U];
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        a[u].template load<NT>(from(h + u) + one);
                        d[u].template load<NT>(from(h + u) + two);
                    }
#pragma unroll
                    for (int u = 0; u < U; ++u) {
#pragma unroll
                        for (int j = 0; j < W; ++j) turn(a[u].t[j], d[u].t[j], j);
                        if (h + u < n) {
                            a[u].template store<NT>(to(h + u) + one);
                            d[u].template store<NT>(to(h + u) + two);
                        }
                    }
                }
            }
        } else {
            const uint64_t one = p.pairs * 2 + (uint64_t)(piece - p.turns) * C;
            for (uint32_t h = 0; h < n; h += U) {
                RtVec<T, C> a[U];
#pragma unroll
                for (int u = 0; u < U; ++u) a[u].template load<NT>(from(h + u) + one);
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (h + u < n) a[u].template store<NT>(to(h + u) + one);
            }
        }
    }
}

template <class T, int W, int C, bool NEIGHBOURS>
void rt_launch_one(RtParams p, hipStream_t stream) {
    p.turns = (uint32_t)(p.pairs / W);
    p.copies = (uint32_t)((p.dim - 2 * p.pairs) / C);
    const uint64_t items = p.batch * p.time * (p.turns + p.copies);
    // a lane takes so many heads that the machine is full, eight at most
    const uint64_t per = items * p.heads >> 18;
    p.per = (uint32_t)(per < 1 ? 1 : per > 8 ? 8 : per);
    p.chunks = (uint32_t)((p.heads + p.per - 1) / p.per);
    const uint64_t blocks = (items * p.chunks + 255) / 256;
    const dim3 grid((unsigned)(blocks < 65536 ? blocks : 65536)), block(256);
    // (heads read four at a time where a lane has as many: for one, 64 x 1 x 32 of 128, the others' reading took 5.7 us)
    if (p.per < 4) hipLaunchKernelGGL((rotary_kernel<T, W, C, NEIGHBOURS, 1, false>), grid, block, 0, stream, p);
    else if (stream_past_caches(p.batch * p.time * p.heads * p.dim * sizeof(T) * 2)) hipLaunchKernelGGL((rotary_kernel<T, W, C, NEIGHBOURS, 4, true>), grid, block, 0, stream, p);
    else hipLaunchKernelGGL((rotary_kernel<T, W, C, NEIGHBOURS, 4, false>), grid, block, 0, stream, p);
    cumo_cuda_runtime_check_kernel_launch();
}

// whole vectors where the pairs, and what is behind them, are some number of those; else one by one
template <class T>
void rt_launch(const cumo_hip_rotary_t& d, hipStream_t stream) {
    constexpr int V = 16 / (int)sizeof(T);
    RtParams p;
    static_cast<cumo_hip_rotary_t&>(p) = d;
    const bool copies = (d.dim - 2 * d.pairs) % V == 0;
    if (d.interleaved) {
        if (d.pairs % (V / 2) == 0) copies ? rt_launch_one<T, V / 2, V, true>(p, stream) : rt_launch_one<T, V / 2, 1, true>(p, stream);
        else rt_launch_one<T, 1, 1, true>(p, stream);
    } else {
        if (d.pairs % V == 0) copies ? rt_launch_one<T, V, V, false>(p, stream) : rt_launch_one<T, V, 1, false>(p, stream);
        else rt_launch_one<T, 1, 1, false>(p, stream);
    }
}

}  // namespace
}  // namespace cumo_hip

using namespace cumo_hip;

extern "C" void cumo_hip_rotary_kernel_launch(int type, const cumo_hip_rotary_t* d) {
    if (type == 0) rt_launch<float>(*d, current_stream());
    else rt_launch<double>(*d, current_stream());
}
