// The gated linear recurrence h[t] = a[t] h[t-1] + b[t] along one axis, and its gradients:
//   l[t] = g[t] + a[t+1] l[t+1] from the end;  gb = l;  ga[t] = l[t] h[t-1];  gh0 = a[0] l[0]
// Backwards what is carried from step to step is m[t] = a[t] l[t], so that a step needs its own elements alone:
//   l[t] = g[t] + m[t+1],  m[t] = a[t] l[t]
// and both directions are one kernel: the launch turns time around by its strides.
//
// A stretch of steps takes a state s to A s + B, with A the product of its gates and B the state that it reaches from zero,
// and stretches join: (A1, B1) then (A2, B2) is (A1 A2, A2 B1 + B2). Lanes and waves hold stretches side by side in registers,
// hand on A and B, and then take their own steps from the state that reaches them, each step the one fused multiply-add of the
// definition: a lane's states are those of one step after the other from where its stretch begins, only what reaches it has
// gone through joins. Products of gates leave the type's range long before the states do: A is a double for SFloat and a double with an
// exponent of its own for DFloat (ReGates).
//
// Two layouts. Down columns (time across memory): a lane a column, 64 columns a wave, a wave's rows in registers, the waves of
// a block one behind the other in time. Along rows (time along memory): a lane a stretch of 64 bytes.
// Where there are enough columns or rows to fill the machine each is walked from its first step to its last by one block. Where
// there are not, time is cut into tiles, a block each, all in one launch: a tile leaves its A and B in memory for the ones after
// it, folds those of the tiles before it from the nearest one whose state is there already, and leaves its own state.
// Memory bounds all but the shortest: SFloat [8,4096,2048] 158 us (5.1 TB/s, a large copy's rate), gradients of [8,2048,2048] 140
// us (4.8), DFloat [4096,4095] along rows 82 us (4.9), its gradients 141 (4.8; SFloat 87, 3.8); in tiles [1,65536,1000] 184 us with
// 6.5 for clearing the words (4.3: in each tile loads, joins and stores follow one another, and 10% more bytes go through the words).
// One step of 64 x 4096: 5.5 us.
#include "common.h"
#include "wait_ctl.h"

#include <cstring>

namespace cumo_hip {
namespace {

// In the order in which the steps are taken, element 0 first. h: the state before each step (the first step's is h0).
struct ReArgs {
    const char *a, *b, *h, *h0;
    char *out, *gb, *last;                       // h, or ga; gradients: gb, gh0
    int64_t a_step[3], b_step[3], h_step[3], out_step[3], gb_step[3];   // outer, time, inner
    uint64_t columns, inner, time;
    uint64_t before;   // columns of the launches in front of this one
};

// the smaller magnitude
__device__ __forceinline__ float re_less(float least, float a) { return __builtin_fminf(least, __builtin_fabsf(a)); }
__device__ __forceinline__ double re_less(double least, double a) { return __builtin_fmin(least, __builtin_fabs(a)); }

// A: the product of a stretch's gates, always a finite number: infinite and NaN gates show in B, which they reach from zero as well.
template <class T> struct ReGates;

// SFloat: in double. Beyond 2^+-300 nothing is left of a finite state, or it is infinite, and neither changes with the gates that come
// after, but for one of 0, which forgets either. So a product out there stays as it is but for its sign, or becomes 0.
template <> struct ReGates<float> {
    static constexpr int W = 2;   // words
    double product;
    // (0 too)
    __device__ __forceinline__ static bool out(double v, int reach) { return (((uint32_t)__double2hiint(v) >> 20) & 0x7ffu) - (uint32_t)(1023 - reach) > 2u * reach; }
    __device__ __forceinline__ static ReGates none() { return {1.0}; }
    template <bool BACK, int N>   // (BACK: in the order of falling j)
    __device__ __forceinline__ static ReGates of(const float (&a)[N]) {
        double own = 1.0;
        float least = 1.0f;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            own *= (double)a[BACK ? N - 1 - j : j];
            least = re_less(least, a[j]);
        }
        if (out(own, 600) && !(own == 0.0 && least == 0.0f)) {   // (rare; it may have been out of double's range in between)
            double m = 1.0;
            int e = 0;
#pragma unroll
            for (int j = 0; j < N; ++j) {
                m *= (double)__builtin_amdgcn_frexp_mantf(a[j]);
                e += __builtin_amdgcn_frexp_expf(a[j]);
            }
            own = __builtin_fabs(m) <= 1.0 ? ldexp(m, e < -600 ? -600 : e > 600 ? 600 : e) : 0x1p600;
        }
        return {own};
    }
    // of two stretches, one after the other
    __device__ __forceinline__ ReGates then(ReGates after) const {
        const bool far = out(product, 300), far_after = out(after.product, 300);
        const double x = far_after && !far ? __builtin_copysign(1.0, product) : product;
        const double y = far && after.product != 0.0 ? __builtin_copysign(1.0, after.product) : after.product;
        return {x * y};
    }
    __device__ __forceinline__ float join(float reached, float state) const { return (float)__builtin_fma(product, (double)state, (double)reached); }
    __device__ __forceinline__ ReGates whole() const { return *this; }
    __device__ __forceinline__ ReGates of_lane_below(int d) const { return {__shfl_up(product, d)}; }
    __device__ __forceinline__ void to(uint32_t* w) const {
        const uint64_t bits = (uint64_t)__double_as_longlong(product);
        w[0] = (uint32_t)bits;
        w[1] = (uint32_t)(bits >> 32);
    }
    __device__ __forceinline__ static ReGates from(const uint32_t* w) { return {__longlong_as_double((long long)(((uint64_t)w[1] << 32) | w[0]))}; }
};

// DFloat: m 2^e, as a state may be small where a product is large, or large where it is small, and stay finite. m is 0, or
// at least 1/2 and less than 1 where it is whole(), half as much for each stretch that has come behind it since.
template <> struct ReGates<double> {
    static constexpr int W = 3;
    static constexpr int kFar = 1 << 28;   // (of no account beyond 2^12: numbers reach from 2^-1074 to 2^1024)
    double m;
    int e;
    __device__ __forceinline__ static ReGates none() { return {1.0, 0}; }
    __device__ __forceinline__ ReGates whole() const { return {__builtin_amdgcn_frexp_mant(m), e + __builtin_amdgcn_frexp_exp(m)}; }
    template <bool BACK, int N>
    __device__ __forceinline__ static ReGates of(const double (&a)[N]) {
        double own = 1.0, least = 1.0;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            own *= a[BACK ? N - 1 - j : j];
            least = re_less(least, a[j]);
        }
        ReGates all = {own, 0};
        const double size = __builtin_fabs(own);
        if (!(size < 0x1p1000) || (size < 0x1p-1000 && !(own == 0.0 && least == 0.0))) {   // (rare)
            all = none();
#pragma unroll
            for (int j = 0; j < N; ++j) {
                all.m *= __builtin_amdgcn_frexp_mant(a[BACK ? N - 1 - j : j]);
                all.e += __builtin_amdgcn_frexp_exp(a[j]);
            }
            if (!(__builtin_fabs(all.m) <= 1.0)) all = {1.0, kFar};
        }
        return all.whole();
    }
    __device__ __forceinline__ ReGates then(ReGates after) const {
        const int both = e + after.e;
        return {m * after.m, both < -kFar ? -kFar : both > kFar ? kFar : both};
    }
    __device__ __forceinline__ double join(double reached, double state) const {
        const int near = e < -900 ? -900 : e > 900 ? 900 : e;   // (m has up to 65 halves: the product below is a normal number)
        double there = state;
        if (e != near && m != 0.0) there = ldexp(state, e - near);   // (rare)
        return __builtin_fma(ldexp(m, near), there, reached);
    }
    __device__ __forceinline__ ReGates of_lane_below(int d) const { return {__shfl_up(m, d), __shfl_up(e, d)}; }
    __device__ __forceinline__ void to(uint32_t* w) const {
        const uint64_t bits = (uint64_t)__double_as_longlong(m);
        w[0] = (uint32_t)bits;
        w[1] = (uint32_t)(bits >> 32);
        w[2] = (uint32_t)e;
    }
    __device__ __forceinline__ static ReGates from(const uint32_t* w) {
        return {__longlong_as_double((long long)(((uint64_t)w[1] << 32) | w[0])), (int)w[2]};
    }
};

// Products of N stretches in shared memory, for joins alone. A DFloat one is held as a plain double where it is one, and looked up where
// that is NaN: [4,4096,2048] walked 190 us, 204 with all of them as m and e (tiles, which multiply them too: [1,65536,1000] 381 and 368).
template <class T, int N> struct ReShelf {
    double plain[N];
    __device__ __forceinline__ void put(int at, ReGates<T> g) { plain[at] = g.product; }
    __device__ __forceinline__ T join(int at, T reached, T state) const { return ReGates<T>{plain[at]}.join(reached, state); }
};
template <int N> struct ReShelf<double, N> {
    double plain[N];
    ReGates<double> other[N];
    __device__ __forceinline__ void put(int at, ReGates<double> g) {
        const bool is = (g.e >= -900 && g.e <= 900) || g.m == 0.0;
        plain[at] = is ? ldexp(g.m, g.e) : __builtin_nan("");
        if (!is) other[at] = g;
    }
    __device__ __forceinline__ double join(int at, double reached, double state) const {
        const double a = plain[at];
        return a == a ? __builtin_fma(a, state, reached) : other[at].join(reached, state);
    }
};

// one step, in place: (a, b) forwards makes b the state; backwards (a, g, h before) makes g the l and h the gate's gradient.
// Both leave what is carried on in `state`.
template <class T, bool GRAD>
__device__ __forceinline__ void re_step(T a, T& b, T& h, T& state) {
    if constexpr (GRAD) {
        b = b + state;
        h = b * h;
        state = a * b;
    } else {
        b = state = __builtin_elementwise_fma(a, state, b);
    }
}
template <class T, bool GRAD>
__device__ __forceinline__ T re_carry(T a, T b, T state) {
    if constexpr (GRAD) return a * (b + state);
    else return __builtin_elementwise_fma(a, state, b);
}

// rows that a wave holds of a column: two tiles of them, of two arrays or three, in the 128 registers of a block of sixteen waves
template <class T, bool GRAD> constexpr int kReRows = (sizeof(T) == 4 ? 16 : 8) / (GRAD ? 2 : 1);

// A wave's columns of one array: the lowest of its lanes' addresses, the same for all, and how far up each lane's lies. A row's
// address is then a number of the wave's and the row's (scalar), and the lane's 32 bits.
struct ReLanes {
    const char* low;
    uint32_t up;
    __device__ __forceinline__ ReLanes(const char* start, int64_t o, int64_t i, const int64_t (&step)[3]) {
        const uint64_t at = (uint64_t)(uintptr_t)(start + o * step[0] + i * step[2]);
        uint64_t least = at;
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) {
            const uint64_t other = (uint64_t)__shfl_xor((unsigned long long)least, d);
            least = other < least ? other : least;
        }
        up = (uint32_t)(at - least);
        low = reinterpret_cast<const char*>(((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(least >> 32)) << 32) |
                                            (uint32_t)__builtin_amdgcn_readfirstlane((int)least));
    }
    template <class T>
    __device__ __forceinline__ T get(int64_t offset) const { return *reinterpret_cast<const T*>(low + offset + up); }
    template <class T>
    __device__ __forceinline__ T get_once(int64_t offset) const { return __builtin_nontemporal_load(reinterpret_cast<const T*>(low + offset + up)); }
    template <class T>
    __device__ __forceinline__ void put(int64_t offset, T v) const { *reinterpret_cast<T*>(const_cast<char*>(low) + offset + up) = v; }
    template <class T>
    __device__ __forceinline__ void put_away(int64_t offset, T v) const { __builtin_nontemporal_store(v, reinterpret_cast<T*>(const_cast<char*>(low) + offset + up)); }
    template <class T>   // written through the second-level cache
    __device__ __forceinline__ void put_through(int64_t offset, T v) const {
        __hip_atomic_store(reinterpret_cast<T*>(const_cast<char*>(low) + offset + up), v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
};

// Forms of a pass over arrays larger than the caches, us. SFloat [8,4096,2048] forwards (with a sum of the result behind it) and
// [1,65536,1000] in tiles; gradients of [8,2048,2048]:
//   loads plain / nt, stores nt              161 (201) / 156 (197),  184 (224) / 190 (231),  139 / 133
//   loads nt, stores plain / written through 145 (182) / 140 (178),  190 (220) / 195 (224),  - / 143
enum ReStore { RE_PLAIN, RE_AWAY, RE_THROUGH };

// what a wave holds of a, b and h: R rows of 64 columns
template <class T, bool GRAD>
struct ReTile {
    static constexpr int R = kReRows<T, GRAD>;
    T a[R], b[R], h[GRAD ? R : 1];
    // rows [t, t + R) that there are; the others leave a state as it is
    template <bool NT>
    __device__ __forceinline__ void load(const ReArgs& p, const ReLanes& la, const ReLanes& lb, const ReLanes& lh, uint64_t t, T first) {
        auto get = [](const ReLanes& x, int64_t offset) { return NT ? x.template get_once<T>(offset) : x.template get<T>(offset); };
        const int64_t at = (int64_t)t;
        if (t + R <= p.time && (!GRAD || t + R < p.time)) {
#pragma unroll
            for (int j = 0; j < R; ++j) {
                a[j] = get(la, (at + j) * p.a_step[1]);
                b[j] = get(lb, (at + j) * p.b_step[1]);
                if (GRAD) h[j] = get(lh, (at + j) * p.h_step[1]);
            }
        } else {
#pragma unroll
            for (int j = 0; j < R; ++j) {
                a[j] = (T)1;
                b[j] = (T)0;
                if (GRAD) h[j] = (T)0;
                if (t + j < p.time) {
                    a[j] = get(la, (at + j) * p.a_step[1]);
                    b[j] = get(lb, (at + j) * p.b_step[1]);
                    if (GRAD) h[j] = t + j + 1 < p.time ? get(lh, (at + j) * p.h_step[1]) : first;
                }
            }
        }
    }
    __device__ __forceinline__ void sum_up(ReGates<T>& product, T& reached) const {
        reached = (T)0;
#pragma unroll
        for (int j = 0; j < R; ++j) reached = re_carry<T, GRAD>(a[j], b[j], reached);
        product = ReGates<T>::template of<false>(a);
    }
    template <ReStore FORM>
    __device__ __forceinline__ void take(const ReArgs& p, const ReLanes& lout, const ReLanes& lgb, uint64_t t, uint64_t to, bool there, T& state) {
        auto put = [](const ReLanes& x, int64_t offset, T v) {
            if constexpr (FORM == RE_AWAY) x.put_away(offset, v);
            else if constexpr (FORM == RE_THROUGH) x.put_through(offset, v);
            else x.put(offset, v);
        };
        const int64_t at = (int64_t)t;
#pragma unroll
        for (int j = 0; j < R; ++j) re_step<T, GRAD>(a[j], b[j], h[GRAD ? j : 0], state);   // (rows that are not there change nothing)
        if (!there) return;
#pragma unroll
        for (int j = 0; j < R; ++j) {
            if (t + j < to) {
                put(lout, (at + j) * p.out_step[1], GRAD ? h[GRAD ? j : 0] : b[j]);
                if constexpr (GRAD) put(lgb, (at + j) * p.gb_step[1], b[j]);
            }
        }
    }
};

// NW waves one behind the other in time over 64 columns. ONCE: one pass over arrays larger than the last-level cache.
template <class T, bool GRAD, int NW, bool ONCE>
__global__ __launch_bounds__(NW * 64) void recurrence_columns_kernel(ReArgs p) {
    typedef ReTile<T, GRAD> Tile;
    constexpr int R = Tile::R;
    constexpr uint64_t kTile = (uint64_t)NW * R;
    __shared__ ReShelf<T, NW * 64> products[2];
    __shared__ T reached[2][NW][64];
    const uint32_t lane = threadIdx.x & 63, wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const uint64_t mine = p.before + (uint64_t)blockIdx.x * 64 + lane;
    const bool there = mine < p.columns;
    const uint64_t c = there ? mine : p.columns - 1;   // (a lane without a column reads the last one's)
    const int64_t o = (int64_t)(c / p.inner), i = (int64_t)(c - (uint64_t)o * p.inner);
    const ReLanes la(p.a, o, i, p.a_step), lb(p.b, o, i, p.b_step), lh(GRAD ? p.h : p.a, o, i, GRAD ? p.h_step : p.a_step);
    const ReLanes lout(p.out, o, i, p.out_step), lgb(GRAD ? p.gb : p.out, o, i, GRAD ? p.gb_step : p.out_step);
    const T first = p.h0 ? reinterpret_cast<const T*>(p.h0)[c] : (T)0;
    T state = GRAD ? (T)0 : first;
    int turn = 0;
    auto walk = [&](Tile& tile, uint64_t t) {   // t: of the wave's first row
        T own = state;
        if constexpr (NW > 1) {
            ReGates<T> product;
            T b;
            tile.sum_up(product, b);
            products[turn].put((int)threadIdx.x, product);
            reached[turn][wave][lane] = b;
            __syncthreads();   // (the other half of the slots is what a wave may still be reading)
#pragma unroll
            for (uint32_t w = 0; w < NW; ++w) {
                own = w == wave ? state : own;
                state = products[turn].join((int)(w * 64 + lane), reached[turn][w][lane], state);
            }
            turn ^= 1;
        }
        tile.template take<!ONCE ? RE_PLAIN : GRAD ? RE_AWAY : RE_THROUGH>(p, lout, lgb, t, p.time, there, own);
        if constexpr (NW == 1) state = own;
        if (GRAD && p.last && there && t < p.time && t + R >= p.time) reinterpret_cast<T*>(p.last)[c] = own;   // (carried past the last step)
    };
    // two tiles in turn: one is on its way while the other's steps are taken. Every wave of the block goes round equally often.
    Tile one, two;
    uint64_t t = (uint64_t)wave * R, at = 0;
    one.template load<ONCE>(p, la, lb, lh, t, first);
    for (;;) {
        two.template load<ONCE>(p, la, lb, lh, t + kTile, first);
        walk(one, t);
        t += kTile;
        if ((at += kTile) >= p.time) break;
        one.template load<ONCE>(p, la, lb, lh, t + kTile, first);
        walk(two, t);
        t += kTile;
        if ((at += kTile) >= p.time) break;
    }
}

// ---- tiles of one launch that hand states on -------------------------------------------
// Every block takes the next tile from a ticket, so that a tile only waits for tiles whose blocks are at work. What it hands on
// travels in 64-bit words {1, 32 bits of the value}, written and read at agent scope: a word is there when its upper half is, and
// no fence is needed. A small kernel clears the words, and the ticket, in front of the launch. A wait gives up after kReLooks looks
// (not reached while every earlier tile has a block at work); it then raises the host's word (wait_ctl.h), and the next point
// where the host waits for the device reports the launch as failed.
// A state is folded one tile after the other whichever tile's state it starts from, so results do not depend on the blocks' timing.
constexpr uint32_t kReLooks = 1u << 22;

struct ReChain {
    uint64_t* words;
    uint32_t* ticket;
    WaitCtl* wait;
    uint32_t tiles;   // of a strip of columns, or of a row
};

template <class T> constexpr int kReWords = (int)(2 * sizeof(T) / 4) + ReGates<T>::W;   // of a tile and column: its state, its A, its B

template <int W>
__device__ __forceinline__ void re_publish(uint64_t* slot, uint32_t stride, const uint32_t (&v)[W]) {
#pragma unroll
    for (int i = 0; i < W; ++i) __hip_atomic_store(slot + (uint64_t)i * stride, (1ull << 32) | v[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <int W>
__device__ __forceinline__ bool re_peek(const uint64_t* slot, uint32_t stride, uint32_t (&v)[W]) {
    uint64_t x[W];
#pragma unroll
    for (int i = 0; i < W; ++i) x[i] = __hip_atomic_load(slot + (uint64_t)i * stride, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    bool all = true;
#pragma unroll
    for (int i = 0; i < W; ++i) {
        all = all && (x[i] >> 32) != 0;
        v[i] = (uint32_t)x[i];
    }
    return all;
}

// the words of one tile and column (or row), `stride` words from one to the next
template <class T>
struct ReSlot {
    static constexpr int W = (int)(sizeof(T) / 4), G = ReGates<T>::W;
    union Number { T t; uint32_t w[W]; };
    uint64_t* at;
    uint32_t stride;
    __device__ __forceinline__ void put_state(T v) const {
        Number s;
        s.t = v;
        re_publish<W>(at, stride, s.w);
    }
    __device__ __forceinline__ void put_sum(ReGates<T> product, T reached) const {
        uint32_t w[G + W];
        Number s;
        s.t = reached;
        product.whole().to(w);
#pragma unroll
        for (int i = 0; i < W; ++i) w[G + i] = s.w[i];
        re_publish<G + W>(at + (uint64_t)W * stride, stride, w);
    }
    __device__ __forceinline__ bool state(T& v) const {
        Number s;
        const bool is = re_peek<W>(at, stride, s.w);
        v = s.t;
        return is;
    }
    __device__ __forceinline__ bool sum(ReGates<T>& product, T& reached) const {
        uint32_t w[G + W];
        const bool is = re_peek<G + W>(at + (uint64_t)W * stride, stride, w);
        Number s;
#pragma unroll
        for (int i = 0; i < W; ++i) s.w[i] = w[G + i];
        product = ReGates<T>::from(w);
        reached = s.t;
        return is;
    }
};

__global__ __launch_bounds__(256) void recurrence_clear_kernel(ulonglong2* pairs, uint64_t n) {
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (uint64_t)gridDim.x * 256) pairs[i] = make_ulonglong2(0, 0);
}

// Down columns: a block of sixteen waves to a tile, and as many tiles before it looked at, a wave each.
constexpr int kReChainWaves = 16;
template <class T, bool GRAD>
__global__ __launch_bounds__(kReChainWaves * 64, sizeof(T) == 4 ? 8 : 4) void recurrence_columns_chain_kernel(ReArgs p, ReChain chain) {
    typedef ReTile<T, GRAD> Tile;
    constexpr int NW = kReChainWaves, R = Tile::R;
    __shared__ ReGates<T> products[NW][64], before_product[NW][64];
    __shared__ T reached[NW][64], before_reached[NW][64];   // (of a tile whose state is there: that)
    __shared__ uint32_t is_state[NW], ticket;
    const uint32_t lane = threadIdx.x & 63, wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    if (threadIdx.x == 0) ticket = __hip_atomic_fetch_add(chain.ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    const uint32_t strips = (uint32_t)((p.columns + 63) / 64);
    const uint32_t k = (uint32_t)__builtin_amdgcn_readfirstlane((int)(ticket / strips)), strip = (uint32_t)__builtin_amdgcn_readfirstlane((int)(ticket - k * strips));
    const uint64_t mine = (uint64_t)strip * 64 + lane;
    const bool there = mine < p.columns;
    const uint64_t c = there ? mine : p.columns - 1;
    const int64_t o = (int64_t)(c / p.inner), i = (int64_t)(c - (uint64_t)o * p.inner);
    const T first = p.h0 ? reinterpret_cast<const T*>(p.h0)[c] : (T)0;
    const uint64_t t = ((uint64_t)k * NW + wave) * R;
    Tile tile;
    {
        const ReLanes la(p.a, o, i, p.a_step), lb(p.b, o, i, p.b_step), lh(GRAD ? p.h : p.a, o, i, GRAD ? p.h_step : p.a_step);
        tile.template load<false>(p, la, lb, lh, t, first);
    }
    ReGates<T> product;
    T b;
    tile.sum_up(product, b);
    products[wave][lane] = product;
    reached[wave][lane] = b;
    __syncthreads();
    auto slot = [&](uint32_t tile_number) {
        return ReSlot<T>{chain.words + ((uint64_t)strip * chain.tiles + tile_number) * (kReWords<T> * 64) + lane, 64};
    };
    if (wave == 0) {
#pragma unroll
        for (int w = 1; w < NW; ++w) {
            b = products[w][lane].join(reached[w][lane], b);
            product = product.then(products[w][lane]);
        }
        if (k > 0) slot(k).put_sum(product, b);
    }
    // the tile `wave` + 1 before this one: its state, or what it makes of one
    auto look = [&](bool want_state) {
        ReGates<T> found_product = ReGates<T>::none();
        T found = GRAD ? (T)0 : first;   // (before the first tile)
        bool state = true;
        if (k >= wave + 1) {
            const ReSlot<T> from = slot(k - wave - 1);
            const uint32_t limit = wait_limit(chain.wait, kReLooks);
            for (uint32_t looks = 0;; ++looks) {
                if (__all(from.state(found))) break;
                state = false;
                if (!want_state && __all(from.sum(found_product, found))) break;
                state = true;
                if (looks >= limit) {
                    if (lane == 0) wait_gave_up(chain.wait, WAIT_SCAN);
                    break;
                }
                __builtin_amdgcn_s_sleep(1);
            }
        }
        before_product[wave][lane] = found_product;
        before_reached[wave][lane] = found;
        if (lane == 0) is_state[wave] = state;
    };
    look(false);
    __syncthreads();
    int near = 0;
    while (near < NW && !is_state[near]) ++near;
    __syncthreads();   // (every wave has found the same)
    if (near == NW) {
        if (wave == NW - 1) look(true);
        near = NW - 1;
        __syncthreads();
    }
    near = __builtin_amdgcn_readfirstlane(near);
    T state = before_reached[near][lane];
    for (int w = near - 1; w >= 0; --w) state = before_product[w][lane].join(before_reached[w][lane], state);
    if (wave == 0 && k + 1 < chain.tiles) slot(k).put_state(product.join(b, state));
    for (uint32_t w = 0; w < wave; ++w) state = products[w][lane].join(reached[w][lane], state);
    const ReLanes lout(p.out, o, i, p.out_step), lgb(GRAD ? p.gb : p.out, o, i, GRAD ? p.gb_step : p.out_step);
    tile.template take<RE_AWAY>(p, lout, lgb, t, p.time, there, state);
    if (GRAD && p.last && there && t < p.time && t + R >= p.time) reinterpret_cast<T*>(p.last)[c] = state;   // (carried past the last step)
}

// Columns that lie further apart than a lane's 32 bits reach: a lane each, one step after the other.
template <class T, bool GRAD>
__global__ __launch_bounds__(64) void recurrence_apart_kernel(ReArgs p) {
    const uint64_t c = p.before + (uint64_t)blockIdx.x * 64 + threadIdx.x;
    if (c >= p.columns) return;
    const int64_t o = (int64_t)(c / p.inner), i = (int64_t)(c - (uint64_t)o * p.inner);
    auto at = [&](const char* x, const int64_t (&step)[3], uint64_t t) { return reinterpret_cast<T*>(const_cast<char*>(x) + o * step[0] + (int64_t)t * step[1] + i * step[2]); };
    const T first = p.h0 ? reinterpret_cast<const T*>(p.h0)[c] : (T)0;
    T state = GRAD ? (T)0 : first;
    for (uint64_t t = 0; t < p.time; ++t) {
        T b = *at(p.b, p.b_step, t), h = (T)0;
        if constexpr (GRAD) h = t + 1 < p.time ? *at(p.h, p.h_step, t) : first;
        re_step<T, GRAD>(*at(p.a, p.a_step, t), b, h, state);
        *at(p.out, p.out_step, t) = GRAD ? h : b;
        if constexpr (GRAD) *at(p.gb, p.gb_step, t) = b;
    }
    if (GRAD && p.last) reinterpret_cast<T*>(p.last)[c] = state;
}

// ---- along rows -----------------------------------------------------------------------
// E consecutive elements a lane, 64 bytes. `back`: time runs against memory, and so do a lane's elements and the lanes.
template <class T, bool GRAD>
struct ReStretch {
    static constexpr int E = 64 / (int)sizeof(T), V = 16 / (int)sizeof(T);
    typedef uint32_t u4 __attribute__((ext_vector_type(4)));
    union Held { u4 q[E / V]; T t[E]; __device__ Held() {} };
    Held a, b, h;   // in the order of memory

    // where element 0 of the stretch that begins with step t lies in memory, in elements from a row's lowest one
    __device__ __forceinline__ static int64_t lowest(const ReArgs& p, uint64_t t) { return GRAD ? (int64_t)(p.time - t) - E : (int64_t)t; }
    // the step of element j of it
    __device__ __forceinline__ static uint64_t step_of(uint64_t t, int j) { return GRAD ? t + (E - 1 - j) : t + j; }

    __device__ __forceinline__ static void whole(Held& x, const T* from) {
        const u4* q = reinterpret_cast<const u4*>(from);
#pragma unroll
        for (int i = 0; i < E / V; ++i) x.q[i] = q[i];
    }
    // rows point at a row's lowest element; steps from `to` on leave a state as it is
    __device__ __forceinline__ void load(const ReArgs& p, const T* pa, const T* pb, const T* ph, uint64_t t, uint64_t to, T first) {
        const int64_t at = lowest(p, t);
        if (t + E <= to) {
            whole(a, pa + at);
            whole(b, pb + at);
            if (GRAD) {
                if (at > 0) {
                    whole(h, ph + at - 1);
                } else {
#pragma unroll
                    for (int j = 0; j < E; ++j) h.t[j] = j > 0 ? ph[j - 1] : first;
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < E; ++j) {
                const bool there = step_of(t, j) < to;
                a.t[j] = there ? pa[at + j] : (T)1;
                b.t[j] = there ? pb[at + j] : (T)0;
                if (GRAD) h.t[j] = !there ? (T)0 : (at + j > 0 ? ph[at + j - 1] : first);
            }
        }
    }
    __device__ __forceinline__ void sum_up(ReGates<T>& product, T& reached) const {
        reached = (T)0;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const int j = GRAD ? E - 1 - i : i;
            reached = re_carry<T, GRAD>(a.t[j], b.t[j], reached);
        }
        product = ReGates<T>::template of<GRAD>(a.t);
    }
    __device__ __forceinline__ T take(T state) {   // the state that is carried past it
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const int j = GRAD ? E - 1 - i : i;
            re_step<T, GRAD>(a.t[j], b.t[j], h.t[j], state);
        }
        return state;
    }
    __device__ __forceinline__ static void put(const Held& x, const ReArgs& p, T* row, uint64_t t, uint64_t to) {
        const int64_t at = lowest(p, t);
        if (t + E <= to) {
            u4* q = reinterpret_cast<u4*>(row + at);
#pragma unroll
            for (int i = 0; i < E / V; ++i) q[i] = x.q[i];
        } else {
#pragma unroll
            for (int j = 0; j < E; ++j)
                if (step_of(t, j) < to) row[at + j] = x.t[j];
        }
    }
};

// joins of L lanes' stretches in the lanes' order: what stands before a lane's (product, reached)
template <class T, int L>
__device__ __forceinline__ void re_scan_lanes(ReGates<T>& product, T& reached) {
    const int lane = (int)(threadIdx.x & 63) & (L - 1);
#pragma unroll
    for (int d = 1; d < L; d <<= 1) {
        const ReGates<T> before = product.of_lane_below(d);
        const T b = __shfl_up(reached, d);
        if (lane >= d) {
            reached = product.join(reached, b);
            product = before.then(product);
        }
    }
    product = product.whole();
}

template <class T>
struct ReRow {
    const T *a, *b, *h;
    T *out, *gb;
    __device__ __forceinline__ ReRow(const ReArgs& p, uint64_t c, bool grad) {
        const int64_t o = (int64_t)(c / p.inner), i = (int64_t)c - o * (int64_t)p.inner;
        a = reinterpret_cast<const T*>(p.a + o * p.a_step[0] + i * p.a_step[2]);
        b = reinterpret_cast<const T*>(p.b + o * p.b_step[0] + i * p.b_step[2]);
        out = reinterpret_cast<T*>(p.out + o * p.out_step[0] + i * p.out_step[2]);
        if (grad) {
            h = reinterpret_cast<const T*>(p.h + o * p.h_step[0] + i * p.h_step[2]);
            gb = reinterpret_cast<T*>(p.gb + o * p.gb_step[0] + i * p.gb_step[2]);
        }
    }
};

constexpr int kReBlock = 256;

// rows that L lanes hold: 256 / L of them a block
template <class T, bool GRAD, int L>
__global__ __launch_bounds__(kReBlock) void recurrence_short_rows_kernel(ReArgs p) {
    typedef ReStretch<T, GRAD> Stretch;
    const uint32_t lane = threadIdx.x % L;
    for (uint64_t first_row = (uint64_t)blockIdx.x * (kReBlock / L); first_row < p.columns; first_row += (uint64_t)gridDim.x * (kReBlock / L)) {
        const uint64_t mine = first_row + threadIdx.x / L;
        const bool there = mine < p.columns;
        const uint64_t c = there ? mine : p.columns - 1;
        const ReRow<T> row(p, c, GRAD);
        const T first = p.h0 ? reinterpret_cast<const T*>(p.h0)[c] : (T)0;
        const uint64_t t = (uint64_t)lane * Stretch::E, to = there ? p.time : 0;
        Stretch s;
        s.load(p, row.a, row.b, row.h, t, to, first);
        T state = GRAD ? (T)0 : first;
        ReGates<T> product;
        T reached;
        if constexpr (L > 1) {
            s.sum_up(product, reached);
            re_scan_lanes<T, L>(product, reached);
        }
        if constexpr (L > 1) {
            const T end = product.join(reached, state);   // after this lane's stretch
            const T before = __shfl_up(end, 1);
            state = lane > 0 ? before : state;
        }
        state = s.take(state);
        if (GRAD && p.last && there && t < p.time && t + Stretch::E >= p.time) reinterpret_cast<T*>(p.last)[c] = state;
        Stretch::put(GRAD ? s.h : s.b, p, row.out, t, to);
        if constexpr (GRAD) Stretch::put(s.b, p, row.gb, t, to);
    }
}

// a block to a row: tiles of its lanes' stretches, the state carried along
template <class T, bool GRAD>
__global__ __launch_bounds__(kReBlock) void recurrence_rows_kernel(ReArgs p) {
    typedef ReStretch<T, GRAD> Stretch;
    constexpr uint64_t kTile = (uint64_t)kReBlock * Stretch::E;
    constexpr int NW = kReBlock / 64;
    __shared__ ReGates<T> products[2][NW];
    __shared__ T reached[2][NW];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (uint64_t c = blockIdx.x; c < p.columns; c += gridDim.x) {
        const ReRow<T> row(p, c, GRAD);
        const T first = p.h0 ? reinterpret_cast<const T*>(p.h0)[c] : (T)0;
        T state = GRAD ? (T)0 : first;
        int turn = 0;
        for (uint64_t at = 0; at < p.time; at += kTile) {
            const uint64_t t = at + (uint64_t)threadIdx.x * Stretch::E;
            Stretch s;
            s.load(p, row.a, row.b, row.h, t, p.time, first);
            ReGates<T> product;
            T b;
            s.sum_up(product, b);
            re_scan_lanes<T, 64>(product, b);
            if (lane == 63) {
                products[turn][wave] = product;
                reached[turn][wave] = b;
            }
            __syncthreads();   // (the other half of the slots is what a wave may still be reading)
            T own = state;
#pragma unroll
            for (uint32_t w = 0; w < NW; ++w) {
                own = w == wave ? state : own;
                state = products[turn][w].join(reached[turn][w], state);
            }
            turn ^= 1;
            const T reach = product.join(b, own);   // after this lane's stretch
            const T before = __shfl_up(reach, 1);
            own = s.take(lane > 0 ? before : own);
            if (GRAD && p.last && t < p.time && t + Stretch::E >= p.time) reinterpret_cast<T*>(p.last)[c] = own;
            Stretch::put(GRAD ? s.h : s.b, p, row.out, t, p.time);
            if constexpr (GRAD) Stretch::put(s.b, p, row.gb, t, p.time);
        }
        __syncthreads();   // (the next row begins with the first half again)
    }
}

// a lane's value for the whole wave; `lane` is the same for all
template <class V>
__device__ __forceinline__ V re_lane(V v, int lane) {
    union { V v; int w[sizeof(V) / 4]; } u;
    u.v = v;
#pragma unroll
    for (int i = 0; i < (int)(sizeof(V) / 4); ++i) u.w[i] = __builtin_amdgcn_readlane(u.w[i], lane);
    return u.v;
}

// Few long rows: a block of sixteen waves to a tile, the 64 tiles before it looked at by a wave, a lane each.
template <class T, bool GRAD>
__global__ __launch_bounds__(kReChainWaves * 64) void recurrence_rows_chain_kernel(ReArgs p, ReChain chain) {
    typedef ReStretch<T, GRAD> Stretch;
    constexpr int NW = kReChainWaves;
    __shared__ ReGates<T> products[NW];
    __shared__ T reached[NW], start;
    __shared__ uint32_t ticket;
    const uint32_t lane = threadIdx.x & 63, wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    if (threadIdx.x == 0) ticket = __hip_atomic_fetch_add(chain.ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    const uint32_t k = ticket / (uint32_t)p.columns;
    const uint64_t c = ticket - k * (uint32_t)p.columns;
    const ReRow<T> row(p, c, GRAD);
    const T first = p.h0 ? reinterpret_cast<const T*>(p.h0)[c] : (T)0;
    const uint64_t t = ((uint64_t)k * (NW * 64) + threadIdx.x) * Stretch::E;
    Stretch s;
    s.load(p, row.a, row.b, row.h, t, p.time, first);
    ReGates<T> product;
    T b;
    s.sum_up(product, b);
    re_scan_lanes<T, 64>(product, b);
    if (lane == 63) {
        products[wave] = product;
        reached[wave] = b;
    }
    __syncthreads();
    auto slot = [&](uint32_t tile_number) { return ReSlot<T>{chain.words + (c * chain.tiles + tile_number) * kReWords<T>, 1}; };
    if (wave == 0) {
        ReGates<T> all = products[0];
        T end = reached[0];
#pragma unroll
        for (int w = 1; w < NW; ++w) {
            end = products[w].join(reached[w], end);
            all = all.then(products[w]);
        }
        if (lane == 0 && k > 0 && k + 1 < chain.tiles) slot(k).put_sum(all, end);
        T state = GRAD ? (T)0 : first;
        if (k > 0) {
            // lane l: the tile l + 1 before this one. Lanes up to the nearest that has a state need a sum.
            const bool asks = lane < k;
            const ReSlot<T> from = slot(asks ? k - 1 - lane : 0);
            const uint32_t limit = wait_limit(chain.wait, kReLooks);
            bool have_state = false, have_sum = false;
            T found_state = (T)0, found = (T)0;
            ReGates<T> found_product = ReGates<T>::none();
            int near;
            for (uint32_t looks = 0;; ++looks) {
                if (asks && !have_state) have_state = from.state(found_state);
                if (asks && !have_state && !have_sum) have_sum = from.sum(found_product, found);
                const uint64_t states = __ballot(have_state), sums = __ballot(have_sum || have_state);
                near = states ? __builtin_ctzll(states) : 64;
                const uint64_t wanted = near == 64 ? ~0ull : (1ull << near) - 1;
                if (near < 64 && (sums & wanted) == wanted) break;
                if (looks >= limit) {
                    if (lane == 0) wait_gave_up(chain.wait, WAIT_SCAN);
                    near = near < 64 ? near : 0;
                    break;
                }
                __builtin_amdgcn_s_sleep(1);
            }
            // (a tile whose state came first and sum was never asked for: only the nearest such is used, as a state)
            near = __builtin_amdgcn_readfirstlane(near);
            state = re_lane(found_state, near);
            for (int l = near - 1; l >= 0; --l) state = re_lane(found_product, l).join(re_lane(found, l), state);
        }
        if (lane == 0) {
            start = state;
            if (k + 1 < chain.tiles) slot(k).put_state(all.join(end, state));
        }
    }
    __syncthreads();
    T state = start;
    for (uint32_t w = 0; w < wave; ++w) state = products[w].join(reached[w], state);
    const T reach = product.join(b, state);
    const T before = __shfl_up(reach, 1);
    state = s.take(lane > 0 ? before : state);
    if (GRAD && p.last && t < p.time && t + Stretch::E >= p.time) reinterpret_cast<T*>(p.last)[c] = state;
    Stretch::put(GRAD ? s.h : s.b, p, row.out, t, p.time);
    if constexpr (GRAD) Stretch::put(s.b, p, row.gb, t, p.time);
}

// ---- launches -------------------------------------------------------------------------
// Waves that a walk down columns is given, sixteen to a compute unit: SFloat [8,4096,2048], 256 strips, with 1, 2, 4, 8 and 16 waves
// each 303, 195, 157, 165 and 158 us.
constexpr uint64_t kReWaves = 4096;
// Time is cut where there are fewer rows or strips of columns than these, and more than so many tiles of them. us walked / in tiles,
// SFloat, down columns: [1,2048,1000] 36 / 15, [15,1024,1000] 58 / 45, of [n,4096,2048] 128 strips 106 / 85, 160 110 / 104, 192 117 / 122, 224 127 /
// 142 (gradients 181 / 144, 190 / 174, 208 / 214, 229 / 260), DFloat 96 strips 180 / 145, 128 185 / 194 (319 / 272, 331 / 357); SFloat
// [1,512,1000] (2 tiles) 10.8 / 12.3, [1,700,1000] (3) 14.2 / 12.5. Along rows: [64,40000] 28 / 15, [160,40000] 30 / 25, [200,40000] 31 / 33,
// [200,131072] 104 / 78, [300,131072] 123 / 110, [400,40000] 45 / 52, [1000,20000] 53 / 70, [1,2^24] 10980 / 96.
constexpr uint64_t kReFewRows = 256, kReFewTiles = 2;
template <class T> constexpr uint64_t kReFewStrips = sizeof(T) == 4 ? 192 : 128;
constexpr uint64_t kReMostTiles = 1u << 21;   // (of all lines together: a launch holds fewer than 2^32 lanes)

// strips of 64 columns, in as many launches as it takes: a launch holds fewer than 2^32 lanes
template <class F>
void re_strips(ReArgs p, unsigned lanes, F launch) {
    const uint64_t most = (1ull << 31) / lanes;
    for (p.before = 0; p.before < p.columns; p.before += most * 64) {
        const uint64_t strips = (p.columns - p.before + 63) / 64;
        launch(p, dim3((unsigned)(strips < most ? strips : most)), dim3(lanes));
    }
}

template <class T, bool GRAD, int NW>
void re_launch_columns(const ReArgs& p, hipStream_t stream) {
    const bool once = stream_past_caches(p.columns * p.time * sizeof(T) * (GRAD ? 5 : 3));
    re_strips(p, NW * 64, [&](const ReArgs& part, dim3 grid, dim3 block) {
        if (once) hipLaunchKernelGGL((recurrence_columns_kernel<T, GRAD, NW, true>), grid, block, 0, stream, part);
        else hipLaunchKernelGGL((recurrence_columns_kernel<T, GRAD, NW, false>), grid, block, 0, stream, part);
    });
}

// `lines`: strips of columns (`lanes` 64), or rows (1); `tile`: steps of a block
template <class T, bool GRAD, bool ROWS>
int re_chain(const ReArgs& p, uint64_t lines, uint64_t tile, hipStream_t stream) {
    ReChain chain;
    chain.wait = wait_ctl();
    if (!chain.wait) {
        report_error(CUMO_HIP_ERROR_RUNTIME, 0, "recurrence: no memory for what the kernels' waits report to");
        return CUMO_HIP_ERROR_RUNTIME;
    }
    chain.tiles = (uint32_t)((p.time + tile - 1) / tile);
    const uint64_t words = (lines * chain.tiles * kReWords<T> * (ROWS ? 1 : 64) + 2) & ~1ull;   // (an even number, the ticket behind the tiles')
    char* memory = cumo_cuda_runtime_malloc(words * sizeof(uint64_t));
    if (!memory) return CUMO_HIP_ERROR_OUT_OF_MEMORY;
    chain.words = reinterpret_cast<uint64_t*>(memory);
    chain.ticket = reinterpret_cast<uint32_t*>(chain.words + words - 1);
    const uint64_t blocks = (words / 2 + 255) / 256;
    hipLaunchKernelGGL(recurrence_clear_kernel, dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(256), 0, stream, reinterpret_cast<ulonglong2*>(memory), words / 2);
    const dim3 grid((unsigned)(lines * chain.tiles)), block(kReChainWaves * 64);
    if constexpr (ROWS) hipLaunchKernelGGL((recurrence_rows_chain_kernel<T, GRAD>), grid, block, 0, stream, p, chain);
    else hipLaunchKernelGGL((recurrence_columns_chain_kernel<T, GRAD>), grid, block, 0, stream, p, chain);
    cumo_cuda_runtime_check_kernel_launch();
    scratch_free(memory);
    return CUMO_HIP_OK;
}

template <class T, bool GRAD>
int re_launch(ReArgs p, hipStream_t stream) {
    const int64_t es = (int64_t)sizeof(T);
    const int64_t along = GRAD ? -es : es;
    // time along memory: every array's steps are its neighbours
    const bool rows = p.a_step[1] == along && p.b_step[1] == along && p.out_step[1] == along &&
                      (!GRAD || (p.h_step[1] == along && p.gb_step[1] == along));
    constexpr uint64_t E = 64 / sizeof(T);
    if (rows && p.time > 1) {
        if (GRAD) {   // (the kernels' rows point at the lowest element)
            const int64_t back = (int64_t)(p.time - 1) * es;
            p.a -= back;
            p.b -= back;
            p.out -= back;
            p.gb -= back;
            p.h -= back - es;
        }
        if (p.time <= 64 * E) {
            const uint64_t lanes = (p.time + E - 1) / E;
            auto go = [&](auto kernel, uint64_t l) {
                const uint64_t blocks = (p.columns - 1) / (kReBlock / l) + 1;
                hipLaunchKernelGGL(kernel, dim3((unsigned)(blocks < (1u << 20) ? blocks : (1u << 20))), dim3(kReBlock), 0, stream, p);
            };
            if (lanes <= 1) go(recurrence_short_rows_kernel<T, GRAD, 1>, 1);
            else if (lanes <= 2) go(recurrence_short_rows_kernel<T, GRAD, 2>, 2);
            else if (lanes <= 4) go(recurrence_short_rows_kernel<T, GRAD, 4>, 4);
            else if (lanes <= 8) go(recurrence_short_rows_kernel<T, GRAD, 8>, 8);
            else if (lanes <= 16) go(recurrence_short_rows_kernel<T, GRAD, 16>, 16);
            else if (lanes <= 32) go(recurrence_short_rows_kernel<T, GRAD, 32>, 32);
            else go(recurrence_short_rows_kernel<T, GRAD, 64>, 64);
            cumo_cuda_runtime_check_kernel_launch();
            return CUMO_HIP_OK;
        }
        constexpr uint64_t kTile = kReChainWaves * 64 * E;
        if (p.columns < kReFewRows && p.time > kTile && p.columns * (p.time / kTile + 1) < kReMostTiles) return re_chain<T, GRAD, true>(p, p.columns, kTile, stream);
        hipLaunchKernelGGL((recurrence_rows_kernel<T, GRAD>), dim3((unsigned)(p.columns < (1u << 20) ? p.columns : (1u << 20))), dim3(kReBlock), 0, stream, p);
        cumo_cuda_runtime_check_kernel_launch();
        return CUMO_HIP_OK;
    }
    const uint64_t strips = (p.columns + 63) / 64;
    auto near = [&](const int64_t (&step)[3]) {   // 64 columns within 2^32 bytes of each other
        const uint64_t across = (uint64_t)(step[0] < 0 ? -step[0] : step[0]), beside = (uint64_t)(step[2] < 0 ? -step[2] : step[2]);
        const uint64_t rows_across = p.columns / p.inner > 1 ? 63 / p.inner + 1 : 0, columns_beside = p.inner < 64 ? p.inner : 64;
        return across < (1ull << 40) && beside < (1ull << 40) && rows_across * across + columns_beside * beside < (1ull << 32);
    };
    if (!near(p.a_step) || !near(p.b_step) || !near(p.out_step) || (GRAD && (!near(p.h_step) || !near(p.gb_step)))) {
        re_strips(p, 64, [&](const ReArgs& part, dim3 grid, dim3 block) { hipLaunchKernelGGL((recurrence_apart_kernel<T, GRAD>), grid, block, 0, stream, part); });
        cumo_cuda_runtime_check_kernel_launch();
        return CUMO_HIP_OK;
    }
    int waves = 1;
    while (waves < 16 && strips * waves < kReWaves && (uint64_t)waves * kReRows<T, GRAD> < p.time) waves *= 2;
    constexpr uint64_t kTile = kReChainWaves * kReRows<T, GRAD>;
    if (strips < kReFewStrips<T> && p.time > kReFewTiles * kTile && strips * (p.time / kTile + 1) < kReMostTiles) return re_chain<T, GRAD, false>(p, strips, kTile, stream);
    if (waves >= 16) re_launch_columns<T, GRAD, 16>(p, stream);
    else if (waves >= 8) re_launch_columns<T, GRAD, 8>(p, stream);
    else if (waves >= 4) re_launch_columns<T, GRAD, 4>(p, stream);
    else if (waves >= 2) re_launch_columns<T, GRAD, 2>(p, stream);
    else re_launch_columns<T, GRAD, 1>(p, stream);
    cumo_cuda_runtime_check_kernel_launch();
    return CUMO_HIP_OK;
}

}  // namespace
}  // namespace cumo_hip

using namespace cumo_hip;

extern "C" int cumo_hip_recurrence_kernel_launch(int type, const cumo_hip_recurrence_t* d) {
    ReArgs p;
    std::memset(&p, 0, sizeof(p));
    p.a = d->a;
    p.b = d->b;
    p.h0 = d->h0;
    p.out = d->h;
    std::memcpy(p.a_step, d->a_step, sizeof(p.a_step));
    std::memcpy(p.b_step, d->b_step, sizeof(p.b_step));
    std::memcpy(p.out_step, d->h_step, sizeof(p.out_step));
    p.columns = d->outer * d->inner;
    p.inner = d->inner;
    p.time = d->time;
    if (p.columns == 0 || p.time == 0) return CUMO_HIP_OK;
    return type == 0 ? re_launch<float, false>(p, current_stream()) : re_launch<double, false>(p, current_stream());
}

extern "C" int cumo_hip_recurrence_grad_kernel_launch(int type, const cumo_hip_recurrence_grad_t* d) {
    ReArgs p;
    std::memset(&p, 0, sizeof(p));
    p.columns = d->outer * d->inner;
    p.inner = d->inner;
    p.time = d->time;
    if (p.columns == 0 || p.time == 0) return CUMO_HIP_OK;
    // from the last step to the first; the state before step t is h[t - 1]
    const int64_t last = (int64_t)d->time - 1;
    p.a = d->a + last * d->a_step[1];
    p.b = d->g + last * d->g_step[1];
    p.h = d->h + (last - 1) * d->h_step[1];
    p.h0 = d->h0;
    p.out = d->ga + last * d->ga_step[1];
    p.gb = d->gb + last * d->gb_step[1];
    p.last = d->gh0;
    for (int k = 0; k < 3; ++k) {
        const int64_t sign = k == 1 ? -1 : 1;
        p.a_step[k] = sign * d->a_step[k];
        p.b_step[k] = sign * d->g_step[k];
        p.h_step[k] = sign * d->h_step[k];
        p.out_step[k] = sign * d->ga_step[k];
        p.gb_step[k] = sign * d->gb_step[k];
    }
    return type == 0 ? re_launch<float, true>(p, current_stream()) : re_launch<double, true>(p, current_stream());
}
