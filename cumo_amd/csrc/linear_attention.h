// Linear attention with a decay for each head, S[t] = a S[t-1] + k[t] (x) v[t], o[t] = scale (S[t] by q[t]), and its gradients.
//
// A walk is this: from q, k (of `dim` elements) and v, o (of `wide`), forwards or backwards in time. With G[t] what the loss has for S[t],
// G[t] = a G[t+1] + scale q[t] (x) g[t], the gradients are three walks more:
//   gq[t] = scale (S[t] by g[t]):  g in the place of q, v of k, k of v, the state transposed
//   gk[t] = G[t] by v[t]:          backwards, v in the place of q, scale g of k, q of v, the state transposed
//   gv[t] = G[t] by k[t]:          backwards, k in the place of q, scale q of k, g of v
// Backwards the state decays behind a step instead of before it (`late`): what is handed on is a G.
//
// One step is bound by the state's bytes, many by the products: SFloat 8 x 2048 x 16 heads of 128 222 us, the matrix units busy for 60 % of them,
// other vector instructions 11 %, LDS 6 %, waits for rows and at a turn's two meetings 14 %. What is beside the products adds up with them, as a SIMD does
// not work on 32 or 64-bit products and on vector instructions at once (one wave: a product of 16 x 16 x 4 floats in 39 cycles, with two vector instructions beside each 56, with four 65). Others: SFloat 1 x 65536 x 8 of 64 191 us
// (62 for what segments leave, 12 for their starts), 64 x 1 x 16 of 128 25; DFloat 4 x 2048 x 16 of 128 355, 6 x 777 x 12 of 72 by 100 140. Gradients:
// SFloat 4 x 2048 x 16 of 128 380, DFloat 3 x 500 x 8 of 64 53.
#pragma once
#include "common.h"

namespace cumo_hip {
namespace {

struct LaWalk {
    const char *q, *k, *v, *state;
    char *o, *last;                            // last: NULL, not wanted
    int64_t q_step[3], k_step[3], v_step[3], o_step[3];  // bytes: sequence, step, head
    uint32_t q_share, k_share, v_share;        // heads of the walk to one of the array
    uint32_t dim, wide;
    uint32_t state_row, state_col;             // elements from S's row to row (of dim), column to column
    double o_scale, k_scale;
    bool backwards;                            // and late
};
struct LaCommon {
    uint64_t batch, time, heads;
    const char* decay;
    const int32_t* lengths;
};

template <class T> __device__ __forceinline__ T la_fma(T a, T b, T c);
template <> __device__ __forceinline__ float la_fma(float a, float b, float c) { return __builtin_fmaf(a, b, c); }
template <> __device__ __forceinline__ double la_fma(double a, double b, double c) { return __builtin_fma(a, b, c); }

__device__ __forceinline__ uint64_t la_length(const LaCommon& c, uint64_t b) {
    if (!c.lengths) return c.time;
    const int64_t n = c.lengths[b];
    return n < 0 ? 0 : (uint64_t)n < c.time ? (uint64_t)n : c.time;
}

// the block's waves meet, for what LDS holds alone: loads from memory stay on their way
__device__ __forceinline__ void la_meet() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// One step, or one after the other where a walk is not one for stretches. LPR lanes hold VE columns each of a row of S, the block's other
// lanes other rows, each a run of them; S goes through memory from step to step (`memory`: last, or scratch), which every lane reads as it
// wrote it. A step is bound by the state's bytes: a lane has U vectors of it on their way at a time, past the caches where they are many: SFloat
// 64 x 16 heads of 128 25 us (5.4 TB/s), eight at a time 28, through the caches 40.
constexpr int kLaStepBlock = 256;
template <class T, int VE> struct __attribute__((aligned(sizeof(T) * VE))) LaColumns { T t[VE]; };
template <class T, int VE, int LPR, bool LATE, bool NT>
__global__ __launch_bounds__(kLaStepBlock) void la_step_kernel(LaWalk w, LaCommon c, char* memory, uint32_t slices) {
    constexpr int RG = kLaStepBlock / LPR, U = 16;
    typedef LaColumns<T, VE> Columns;
    __shared__ T part[kLaStepBlock * VE];
    __shared__ T qs[256], ks[256];
    const uint64_t which = blockIdx.x / slices, b = which / c.heads, h = which - b * c.heads;
    const uint32_t lane = threadIdx.x % LPR, group = threadIdx.x / LPR;
    const uint32_t e = ((uint32_t)(blockIdx.x % slices) * LPR + lane) * VE;
    const bool there = e < w.wide;
    const uint32_t rows = (w.dim + RG - 1) / RG, d0 = group * rows, d1 = d0 + rows < w.dim ? d0 + rows : w.dim;
    const uint64_t length = la_length(c, b), size = (uint64_t)w.dim * w.wide;
    const T a = reinterpret_cast<const T*>(c.decay)[h];
    const T* from = w.state ? reinterpret_cast<const T*>(w.state) + which * size : nullptr;
    T* to = memory ? reinterpret_cast<T*>(memory) + which * size : nullptr;
    const bool near = w.state_col == 1;
    auto read = [&](uint32_t d) {
        Columns x;
        const T* p = from + (uint64_t)d * w.state_row + (uint64_t)e * w.state_col;
        if (near) {
            if constexpr (NT && VE * sizeof(T) == 16) *reinterpret_cast<store_u4*>(&x) = __builtin_nontemporal_load(reinterpret_cast<const store_u4*>(p));
            else __builtin_memcpy(&x, p, sizeof(x));
        } else {
#pragma unroll
            for (int j = 0; j < VE; ++j) x.t[j] = p[(uint64_t)j * w.state_col];
        }
        return x;
    };
    auto write = [&](uint32_t d, const Columns& x) {
        T* p = to + (uint64_t)d * w.state_row + (uint64_t)e * w.state_col;
        if (near) {
            if constexpr (NT && VE * sizeof(T) == 16) __builtin_nontemporal_store(*reinterpret_cast<const store_u4*>(&x), reinterpret_cast<store_u4*>(p));
            else __builtin_memcpy(p, &x, sizeof(x));
        } else {
#pragma unroll
            for (int j = 0; j < VE; ++j) p[(uint64_t)j * w.state_col] = x.t[j];
        }
    };
    const char* q = w.q + (int64_t)b * w.q_step[0] + (int64_t)(h / w.q_share) * w.q_step[2];
    const char* k = w.k + (int64_t)b * w.k_step[0] + (int64_t)(h / w.k_share) * w.k_step[2];
    const char* v = w.v + (int64_t)b * w.v_step[0] + (int64_t)(h / w.v_share) * w.v_step[2];
    char* o = w.o + (int64_t)b * w.o_step[0] + (int64_t)h * w.o_step[2];
    for (uint64_t n = 0; n < length; ++n) {
        const uint64_t t = LATE ? length - 1 - n : n;
        la_meet();
        if (threadIdx.x < w.dim) {
            qs[threadIdx.x] = reinterpret_cast<const T*>(q + (int64_t)t * w.q_step[1])[threadIdx.x];
            ks[threadIdx.x] = reinterpret_cast<const T*>(k + (int64_t)t * w.k_step[1])[threadIdx.x] * (T)w.k_scale;
        }
        const T* vt = reinterpret_cast<const T*>(v + (int64_t)t * w.v_step[1]);
        T sum[VE], vv[VE];
#pragma unroll
        for (int j = 0; j < VE; ++j) {
            sum[j] = (T)0;
            vv[j] = there ? vt[e + j] : (T)0;
        }
        Columns s[U];
        const bool known = there && from;
        for (uint32_t d = d0; d < d1 || d == d0; d += U) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (known && d + u < d1) {
                    s[u] = read(d + u);
                } else {
#pragma unroll
                    for (int j = 0; j < VE; ++j) s[u].t[j] = (T)0;
                }
            }
            if (d == d0) la_meet();
            if (!there) continue;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (d + u >= d1) continue;
                const T kd = ks[d + u], qd = qs[d + u];
#pragma unroll
                for (int j = 0; j < VE; ++j) {
                    T x = LATE ? la_fma(kd, vv[j], s[u].t[j]) : la_fma(kd, vv[j], a * s[u].t[j]);
                    sum[j] = la_fma(qd, x, sum[j]);
                    s[u].t[j] = LATE ? a * x : x;
                }
                if (to) write(d + u, s[u]);
            }
        }
        from = to;
#pragma unroll
        for (int j = 0; j < VE; ++j) part[threadIdx.x * VE + j] = sum[j];
        la_meet();
        if (group == 0 && there) {
            Columns all;
#pragma unroll
            for (int j = 0; j < VE; ++j) {
                all.t[j] = (T)0;
#pragma unroll
                for (int g = 0; g < RG; ++g) all.t[j] += part[(g * LPR + lane) * VE + j];
                all.t[j] *= (T)w.o_scale;
            }
            __builtin_memcpy(o + (int64_t)t * w.o_step[1] + (uint64_t)e * sizeof(T), &all, sizeof(all));
        }
    }
    if (length == 0 && to && there) {
        Columns none;
#pragma unroll
        for (int j = 0; j < VE; ++j) none.t[j] = (T)0;
        for (uint32_t d = d0; d < d1; ++d) write(d, from ? read(d) : none);
    }
    if (there && group == 0) {
        for (uint64_t t = length; t < c.time; ++t)
            for (int j = 0; j < VE; ++j) reinterpret_cast<T*>(o + (int64_t)t * w.o_step[1])[e + j] = (T)0;
    }
}

template <class T, int VE, int LPR>
void la_step_one(const LaWalk& w, const LaCommon& c, char* memory, hipStream_t stream) {
    const uint32_t slices = (w.wide + LPR * VE - 1) / (LPR * VE);
    const dim3 grid((unsigned)(c.batch * c.heads * slices)), block(kLaStepBlock);
    const bool nt = stream_past_caches(c.batch * c.heads * w.dim * w.wide * sizeof(T) * 2) && c.time == 1;
    if (w.backwards) hipLaunchKernelGGL((la_step_kernel<T, VE, LPR, true, false>), grid, block, 0, stream, w, c, memory, slices);
    else if (nt) hipLaunchKernelGGL((la_step_kernel<T, VE, LPR, false, true>), grid, block, 0, stream, w, c, memory, slices);
    else hipLaunchKernelGGL((la_step_kernel<T, VE, LPR, false, false>), grid, block, 0, stream, w, c, memory, slices);
}

template <class T>
void la_step(const LaWalk& w, const LaCommon& c, char* memory, hipStream_t stream) {
    constexpr int V = 16 / (int)sizeof(T);
    // (few heads: eight lanes to a row, so that more blocks share a head)
    if (w.wide % V == 0) {
        if (w.wide <= 8 * V || c.batch * c.heads * ((w.wide + 32 * V - 1) / (32 * V)) < (uint64_t)device_compute_units()) la_step_one<T, V, 8>(w, c, memory, stream);
        else if (w.wide <= 16 * V) la_step_one<T, V, 16>(w, c, memory, stream);
        else if (w.wide <= 32 * V) la_step_one<T, V, 32>(w, c, memory, stream);
        else la_step_one<T, V, 64>(w, c, memory, stream);
    } else {
        if (w.wide <= 16) la_step_one<T, 1, 16>(w, c, memory, stream);
        else la_step_one<T, 1, 64>(w, c, memory, stream);
    }
}

// ---- stretches of sixteen steps ------------------------------------------------------------------------------------
// For a stretch of n steps behind a state S, with i and j counted in it,
//   o[i] = a^(i+1) q[i] S + sum over j <= i of a^(i-j) (q[i] . k[j]) v[j],   S' = a^n S + sum over j of a^(n-1-j) k[j] (x) v[j]
// (late: a^i, a^(n-j)), four products by matrix instructions of 16 x 16 x 4. A wave holds 16 columns of S in registers from stretch to
// stretch, as the instruction leaves them: lane (m, g) of 16 x 4 has rows 4 g to 4 g + 3 of its column m. So held, S is the first operand of the
// next product as it is (S^T by q^T, o transposed), and so is what k by q^T leaves (the masked products, transposed: the second operand of v^T by
// them); v by columns serves as the second operand of k^T by v and the first of v^T. Nothing is moved between lanes but the products k q^T, of
// which each of the NW waves works out a share, over its part of dim: they meet in LDS. Rows of q, k and v go through LDS too, a stretch ahead, and
// are on their way there for a stretch before: read from memory by every wave as its lanes want them, they kept the first-level cache at
// work for four fifths of the time (SFloat 8 x 2048 x 16 heads of 128: 266 us, and 222 so). Not kept: dim shared out over two waves of a SIMD 272, rows
// three stretches ahead in registers 274, vector instructions spread between the products by hand 231.
//
// Double precision counts rows otherwise (lane (m, g) has rows g, g + 4, ...): operands are read by la_label, so that what
// stands above holds for it too.
template <class T> using LaQuad = T __attribute__((ext_vector_type(4)));
__device__ __forceinline__ LaQuad<float> la_mma(float a, float b, LaQuad<float> c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }
__device__ __forceinline__ LaQuad<double> la_mma(double a, double b, LaQuad<double> c) { return __builtin_amdgcn_mfma_f64_16x16x4f64(a, b, c, 0, 0, 0); }
// four elements of a row in LDS, which starts on a boundary of 16 bytes (four doubles by themselves would be taken to start on one of 32)
template <class T>
__device__ __forceinline__ LaQuad<T> la_quad(const T* p) {
    LaQuad<T> x;
    __builtin_memcpy(&x, __builtin_assume_aligned(p, 16), sizeof(x));
    return x;
}
template <class T> __device__ __forceinline__ uint32_t la_label(uint32_t m) { return sizeof(T) == 4 ? m : 4 * (m & 3) + (m >> 2); }

constexpr uint32_t kLaStretch = 16;

// A power as the sum of two doubles where T is double: squares of squares would be off by n / 2 roundings, on one side for all of a sequence's stretches
// (DFloat 6 x 777: states off by 4e-15 in norm).
template <class T>
struct LaPower {
    double hi, lo;
    __device__ __forceinline__ LaPower by(const LaPower& o) const {
        const double h = hi * o.hi;
        if (sizeof(T) == 4) return LaPower{h, 0.0};
        double l = __builtin_fma(hi, o.lo, __builtin_fma(lo, o.hi, __builtin_fma(hi, o.hi, -h)));
        l = h - h == 0.0 ? l : 0.0;
        const double s = h + l;
        return LaPower{s, l - (s - h)};
    }
};
// a^n by squares, n >= 0
template <class T>
__device__ __forceinline__ LaPower<T> la_power(double a, uint64_t n) {
    LaPower<T> p = {1.0, 0.0}, x = {a, 0.0};
    for (; n; n >>= 1) {
        if (n & 1) p = p.by(x);
        x = x.by(x);
    }
    return p;
}
// of n up to 16 for many n
template <class T>
struct LaPowers {
    LaPower<T> a[5];
    __device__ __forceinline__ explicit LaPowers(double x) {
        a[0] = LaPower<T>{x, 0.0};
#pragma unroll
        for (int k = 1; k < 5; ++k) a[k] = a[k - 1].by(a[k - 1]);
    }
    __device__ __forceinline__ LaPower<T> whole(uint32_t n) const {
        LaPower<T> p = n & 1 ? a[0] : LaPower<T>{1.0, 0.0};
#pragma unroll
        for (int k = 1; k < 5; ++k) p = n >> k & 1 ? p.by(a[k]) : p;
        return p;
    }
    __device__ __forceinline__ double operator()(uint32_t n) const {   // (to a rounding or four)
        double p = n & 1 ? a[0].hi : 1.0;
#pragma unroll
        for (int k = 1; k < 5; ++k) p *= n >> k & 1 ? a[k].hi : 1.0;
        return p;
    }
};

struct LaPlan {
    uint32_t walks, segments, slices;
    uint64_t steps;         // of a segment, a multiple of kLaStretch
    char* starts[3];        // [segments - 1][batch * heads][dim * wide]: the state that each segment but the last leaves to the next, by walk
};
struct LaWalks {
    LaWalk walk[3];
};

// rows of an array as a turn takes them, in its direction: from `low`, unsigned offsets
template <uint32_t TURN>
struct LaRows {
    const char* low;
    int64_t advance;
    uint32_t step;
    bool down;
    __device__ __forceinline__ LaRows(const char* p, const int64_t* steps, uint64_t b, uint64_t h, uint64_t first, bool backwards) {
        const int64_t one = backwards ? -steps[1] : steps[1];
        down = one < 0;
        step = (uint32_t)(down ? -one : one);
        advance = one * (int64_t)TURN;
        low = p + (int64_t)b * steps[0] + (int64_t)h * steps[2] + (int64_t)first * steps[1] + (down ? one * (int64_t)(TURN - 1) : 0);
    }
    __device__ __forceinline__ uint32_t row(uint32_t k) const { return (down ? TURN - 1 - k : k) * step; }
};

// LANES lanes to a row of N elements (a multiple of 16) in LDS, of which `cols` are there; 16 bytes of them a lane and turn, or one
template <class T, int N, int LANES, bool QUADS>
struct LaStage {
    static constexpr uint32_t W = QUADS ? 16 / sizeof(T) : 1;             // elements at a time
    static constexpr int COUNT = (N / (int)W + LANES - 1) / LANES;
    static constexpr uint32_t ROW = N + 16 / sizeof(T);                   // (lanes that read one column of neighbouring rows meet in no bank)
    struct Piece { T t[W]; };
    Piece held[COUNT];
    __device__ __forceinline__ void fetch(const char* low, uint32_t row_offset, uint32_t lane, uint32_t cols) {
#pragma unroll
        for (int i = 0; i < COUNT; ++i) {
            const uint32_t c = (lane + (uint32_t)i * LANES) * W;
            __builtin_memcpy(&held[i], low + (row_offset + (c < cols ? c : 0) * (uint32_t)sizeof(T)), sizeof(Piece));
        }
    }
    // zeros for a row that is not there, and behind its end; `whole`: there is neither
    __device__ __forceinline__ void place(T* rows, uint32_t row, uint32_t lane, uint32_t cols, bool there, bool whole) const {
        if (whole) {
#pragma unroll
            for (int i = 0; i < COUNT; ++i) {
                const uint32_t c = (lane + (uint32_t)i * LANES) * W;
                if (N % ((int)W * LANES) == 0 || c < N) __builtin_memcpy(__builtin_assume_aligned(rows + row * ROW + c, QUADS ? 16 : sizeof(T)), &held[i], sizeof(Piece));
            }
            return;
        }
#pragma unroll
        for (int i = 0; i < COUNT; ++i) {
            const uint32_t c = (lane + (uint32_t)i * LANES) * W;
            Piece x = held[i];
#pragma unroll
            for (uint32_t j = 0; j < W; ++j) x.t[j] = there && c < cols ? x.t[j] : (T)0;
            if (N % ((int)W * LANES) == 0 || c < N) __builtin_memcpy(__builtin_assume_aligned(rows + row * ROW + c, QUADS ? 16 : sizeof(T)), &x, sizeof(Piece));
        }
    }
};

// A turn takes two stretches, one behind the other; one, where their rows would fill LDS or the registers that bring them, and in double precision
// where dim's tiles are shared out by fours (DFloat 4 x 2048 x 16 heads of 128 401 and 353 us, gradients 3 x 500 x 8 of 64 63 and 56). Its rows are in
// LDS, in two buffers where they fit twice.
template <class T, int DT> constexpr int kLaSubs = sizeof(T) == 8 && DT % 4 == 0 ? 1 : sizeof(T) * DT <= 64 ? 2 : 1;
template <class T, int DT> constexpr uint32_t kLaTurn = kLaStretch * kLaSubs<T, DT>;
// products k q^T on their way from wave to wave: those of the next turn may meet those of this one where a turn has one barrier
template <class T, int DT, int NW> constexpr uint64_t kLaSlots = (kLaSubs<T, DT> == 1 ? 2 : 1) * NW * 256 * sizeof(T);
template <class T, int DT, int NW> constexpr uint64_t kLaBuffer = kLaTurn<T, DT> * (2 * (DT * 16 * sizeof(T) + 16) + NW * 16 * sizeof(T) + 16);
template <class T, int DT, int NW> constexpr bool kLaTwice = 2 * kLaBuffer<T, DT, NW> + kLaSlots<T, DT, NW> <= 160 * 1024;
template <class T, int DT, int NW, int BUFFERS, bool ONLY>
constexpr uint64_t kLaShared = BUFFERS * (kLaBuffer<T, DT, NW> - (ONLY ? kLaTurn<T, DT> * (DT * 16 * sizeof(T) + 16) : 0)) + (ONLY ? 0 : kLaSlots<T, DT, NW>);
// Waves to a SIMD that the registers are shared out for: two, so 256 of one kind, where a lane holds less (else the compiler spreads them over both
// kinds, and moves them: also where it knows that LDS, hence told at the launch, holds one block alone).
template <class T, int DT, int NW> constexpr int kLaWaves = sizeof(T) == 4 ? (DT <= 8 ? 2 : 1) : DT <= 4 && NW == 4 ? 2 : 1;
// Tiles of dim that a walk of DT surely has; one behind them is left out where dim does not reach it, which takes a branch in front of each pair of
// products. It pays where the tile is a sixth of them and most dims of the class do without it, DFloat of 65 to 96, us with / without: of 65 to 80 a
// twentieth and more (6 x 777 x 12 of 66 by 100 164 / 174, of 72 146 / 155, of 80 148 / 158; 4 x 2048 x 16 of 68 by 64 155 / 165; gradients 4 x 512 x 8 of 76
// 92 / 99), of 81 to 96 up to 2 % lost (84 163 / 160, 96 158 / 158). Not so the next classes, with tiles left out from the tenth and the
// fourteenth on: 144 270 / 278, but 160 284 / 281, 176 291 / 282, 192 297 / 278; 196 616 / 619, 240 645 / 632, 256 645 / 625. SFloat of 72 gains 5 % where 96 loses 4.
template <class T, int DT> constexpr int kLaLeast = sizeof(T) == 8 && DT == 6 ? 5 : DT;
extern __shared__ __attribute__((aligned(32))) char la_shared[];

// DT: tiles of 16 that hold dim. NW: tiles of 16 columns to a block, a wave each. QUADS: rows of dim and of wide are whole fours. ONLY: what a
// segment leaves by itself.
template <class T, int DT, int NW, int BUFFERS, bool QUADS, bool ONLY>
__global__ __launch_bounds__(64 * NW, (kLaWaves<T, DT, NW>)) void la_stretch_kernel(LaWalks walks, LaCommon c, LaPlan plan) {
    typedef LaQuad<T> Quad;
    constexpr uint32_t E = sizeof(T);
    constexpr int SUBS = kLaSubs<T, DT>;
    constexpr uint32_t TURN = kLaTurn<T, DT>;
    constexpr int LANES = 4 * NW / SUBS < 4 ? 4 : 4 * NW / SUBS;   // to a row, of a part of the turn's rows at a time
    constexpr int ROWS = 64 * NW / LANES, LOADS = (int)TURN / ROWS;   // rows that the block brings at a time, and how often
    constexpr int PARTS = NW / SUBS < 1 ? 1 : NW / SUBS, EACH = NW < SUBS ? SUBS / NW : 1;   // waves to a product k q^T; products to a wave
    constexpr int PM = DT / PARTS;
    static_assert(DT % PARTS == 0 && DT % 2 == 0, "tiles of dim are shared out whole, and taken in pairs");
    typedef LaStage<T, DT * 16, LANES, QUADS> Keys;
    typedef LaStage<T, NW * 16, LANES, QUADS> Values;
    constexpr uint32_t KEYS = TURN * Keys::ROW, VALUES = TURN * Values::ROW;
    T* const k_rows = reinterpret_cast<T*>(la_shared);
    T* const v_rows = k_rows + BUFFERS * KEYS;
    T* const q_rows = v_rows + BUFFERS * VALUES;
    Quad* const slot = reinterpret_cast<Quad*>(q_rows + BUFFERS * KEYS);
    static_assert(sizeof(T) * (BUFFERS * (2 * KEYS + VALUES)) + kLaSlots<T, DT, NW> == kLaShared<T, DT, NW, BUFFERS, false> && kLaShared<T, DT, NW, BUFFERS, false> <= 160 * 1024, "LDS");
    static_assert(Keys::ROW * sizeof(T) % 16 == 0 && sizeof(T) * KEYS % 32 == 0 && sizeof(T) * VALUES % 32 == 0, "rows and slots stand where they are read");
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), m = lane & 15, g = lane >> 4, label = la_label<T>(m);
    const uint64_t bh_all = c.batch * c.heads;
    uint64_t at = blockIdx.x;
    const uint64_t bh = at % bh_all;
    at /= bh_all;
    const uint32_t slice = (uint32_t)(at % plan.slices);
    at /= plan.slices;
    const uint32_t segment = (uint32_t)(at % plan.segments), which = (uint32_t)(at / plan.segments);
    const LaWalk& w = walks.walk[which];
    const uint64_t b = bh / c.heads, h = bh - b * c.heads;
    const uint32_t D = w.dim, W = w.wide;
    const uint64_t length = la_length(c, b), begin = segment * plan.steps;
    const uint64_t end = begin + plan.steps < length ? begin + plan.steps : length;
    const uint32_t total = end > begin ? (uint32_t)(end - begin) : 0;
    const uint32_t b0 = slice * NW * 16, e0 = b0 + wave * 16;     // the block's columns, and the wave's
    const uint32_t cols = W - b0 < NW * 16 ? W - b0 : NW * 16;
    const bool column = e0 + label < W;
    const int tiles = (int)((D + 15) / 16);
    auto there = [&](int t) { return t < kLaLeast<T, DT> || t < tiles; };
    const LaPowers<T> power((double)reinterpret_cast<const T*>(c.decay)[h]);
    const bool late = w.backwards;

    // the state
    Quad S[DT];
    {
        const char* from = segment == 0 || ONLY ? w.state : plan.starts[which] + (uint64_t)(segment - 1) * bh_all * D * W * E;
        const uint32_t row = segment == 0 ? w.state_row : W, col = segment == 0 ? w.state_col : 1;
        const T* s = reinterpret_cast<const T*>(from) + bh * D * W;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) S[dt] = Quad{(T)0, (T)0, (T)0, (T)0};
        if (!ONLY && from && column) {
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const uint32_t d = dt * 16 + 4 * g + r;
                    const T x = s[(d < D ? d : D - 1) * row + (e0 + label) * col];
                    S[dt][r] = d < D ? x : (T)0;
                }
            }
        }
    }

    const uint64_t first = w.backwards ? (length ? length - 1 - begin : 0) : begin;
    LaRows<TURN> q(w.q, w.q_step, b, h / w.q_share, first, w.backwards), k(w.k, w.k_step, b, h / w.k_share, first, w.backwards), v(w.v, w.v_step, b, h / w.v_share, first, w.backwards);
    v.low += b0 * E;
    char* o = w.o + (int64_t)b * w.o_step[0] + (int64_t)h * w.o_step[2] + (int64_t)first * w.o_step[1];
    const int64_t o_one = w.backwards ? -w.o_step[1] : w.o_step[1];

    // Every lane brings parts of rows; rows behind the last are read as that one. One turn's rows are on their way while another's are worked
    // on; behind the last, those again.
    const uint32_t my_row = threadIdx.x / LANES, my_lane = threadIdx.x % LANES;
    Keys q_held[LOADS], k_held[LOADS];
    Values v_held[LOADS];
    uint32_t sent = 0;   // steps sent for, up to the last turn
    auto of_turn = [&](uint32_t done) { return total - done < TURN ? total - done : TURN; };
    auto fetch = [&] {
        const uint32_t n = of_turn(sent);
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const uint32_t row = my_row + i * ROWS < n ? my_row + i * ROWS : n - 1;
            if constexpr (!ONLY) q_held[i].fetch(q.low, q.row(row), my_lane, D);
            k_held[i].fetch(k.low, k.row(row), my_lane, D);
            v_held[i].fetch(v.low, v.row(row), my_lane, cols);
        }
        const bool more = sent + TURN < total;
        sent += more ? TURN : 0;
        q.low += more ? q.advance : 0;
        k.low += more ? k.advance : 0;
        v.low += more ? v.advance : 0;
    };
    auto place = [&](uint32_t buffer, uint32_t n) {
        const bool whole_keys = n == TURN && D == DT * 16, whole_values = n == TURN && cols == NW * 16;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const uint32_t row = my_row + i * ROWS;
            if constexpr (!ONLY) q_held[i].place(q_rows + buffer * KEYS, row, my_lane, D, row < n, whole_keys);
            k_held[i].place(k_rows + buffer * KEYS, row, my_lane, D, row < n, whole_keys);
            v_held[i].place(v_rows + buffer * VALUES, row, my_lane, cols, row < n, whole_values);
        }
    };

    // decays: of the products of step i = m with steps j = 4 g + r, of what S gives to step i, of what step j of a stretch leaves
    T decay_p[4], decay_k[SUBS][4], decay_q, decay_s[SUBS];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const uint32_t j = 4 * g + r;
        decay_p[r] = j <= m ? (T)(power(m - j) * w.k_scale) : (T)0;
    }
    decay_q = (T)power(m + (late ? 0 : 1));
    T o_scale = (T)w.o_scale;
    asm("" : "+v"(o_scale));   // (held: read from the arguments in every turn, it would wait for all that LDS has been asked for)
    // S is multiplied by a^16 in every stretch. Rounded to its type, that would be off by as much each time, on one side: SFloat 1.4e-6 of a state that
    // forgets over 2000 steps. So each factor is rounded from what makes the product of all so far the power that it stands for (5.7e-7: what the
    // additions round). `behind`: by how much of itself that product is too small.
    double behind = 0.0;
    const LaPower<T> a16 = power.whole(kLaStretch);
    const double inverse16 = a16.hi > 0x1p-100 && a16.hi < 0x1p100 ? 1.0 / a16.hi : 0.0;   // (0: as they are)
    auto rounded = [&](const LaPower<T>& exact) { return (T)(inverse16 != 0.0 ? exact.hi + __builtin_fma(exact.hi, behind, exact.lo) : exact.hi); };
    auto next_decay = [&] {
        const T s = rounded(a16);
        behind = __builtin_fma((a16.hi - (double)s) + a16.lo, inverse16, behind);
        return s;
    };
    auto ends = [&](uint32_t of_all) {   // a turn of so many steps, fewer than it can have: the last
#pragma unroll 1
        for (int sub = 0; sub < SUBS; ++sub) {
            const uint32_t n = of_all <= sub * kLaStretch ? 0 : of_all - sub * kLaStretch < kLaStretch ? of_all - sub * kLaStretch : kLaStretch;
            T k4[4], s1 = n ? rounded(power.whole(n)) : (T)1;
            behind = 0.0;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const uint32_t j = 4 * g + r;
                k4[r] = j < n ? (T)(power(n - 1 - j + (late ? 1 : 0)) * w.k_scale) : (T)0;
            }
#pragma unroll
            for (int to = 0; to < SUBS; ++to) {
                decay_s[to] = sub == to ? s1 : decay_s[to];
#pragma unroll
                for (int r = 0; r < 4; ++r) decay_k[to][r] = sub == to ? k4[r] : decay_k[to][r];
            }
        }
    };

    // A turn, in the order in which the wave goes through it. What LDS has of the tiles is asked for well ahead of the products that take it (left to
    // itself the compiler asks in front of each pair of them), and the waves meet where products are left to be worked on:
    //   k q^T of the turn, shared out; with S of the first stretch q S, and meanwhile columns of k asked for, S decayed, the next turn's rows put into LDS
    //   meet: the shares of k q^T are there;  k^T v of the stretch, between them what k q^T gives, and rows of q asked for;  q S of the second stretch
    //   meet: the next turn's rows are there;  k^T v, meanwhile the first rows of that turn asked for
    if (total) {
        ends(TURN);
        fetch();
        place(0, of_turn(0));
        if constexpr (BUFFERS == 2) fetch();
        la_meet();
        uint32_t buffer = 0, done = 0;
        const T *qr = q_rows, *kr = k_rows, *vr = v_rows;
        Quad V, F[DT];   // (F: rows of q, and each, once used, columns of k, and then those of q again)
        Quad PQ[ONLY ? 1 : EACH][ONLY ? 1 : PM], PK[ONLY ? 1 : EACH][ONLY ? 1 : PM];
        auto read_v = [&](int sub) {
#pragma unroll
            for (int r = 0; r < 4; ++r) V[r] = vr[(sub * 16 + 4 * g + r) * Values::ROW + wave * 16 + label];
        };
        auto read_k = [&](int sub, int dt) {
#pragma unroll
            for (int r = 0; r < 4; ++r) F[dt][r] = kr[(sub * 16 + 4 * g + r) * Keys::ROW + dt * 16 + label];
        };
        auto read_q = [&](int sub, int dt) { F[dt] = la_quad(qr + (sub * 16 + m) * Keys::ROW + dt * 16 + 4 * g); };
        auto read_first = [&](int sub, int dt) {
            if constexpr (ONLY) read_k(sub, dt);
            else read_q(sub, dt);
        };
        auto read_p = [&] {
            if constexpr (!ONLY) {
                const int part = wave % PARTS;
#pragma unroll
                for (int e = 0; e < EACH; ++e) {
                    const int sub = EACH > 1 ? e : (int)(wave / PARTS);
#pragma unroll
                    for (int i = 0; i < PM; ++i) {
                        PQ[e][i] = la_quad(qr + (sub * 16 + m) * Keys::ROW + (part * PM + i) * 16 + 4 * g);
                        PK[e][i] = la_quad(kr + (sub * 16 + label) * Keys::ROW + (part * PM + i) * 16 + 4 * g);
                    }
                }
            }
        };
        read_p();
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) read_first(0, dt);
        read_v(0);
        uint32_t slots = 0;
        do {
            const uint32_t n = of_turn(done);
            done += n;
            if (n < TURN) {
                ends(n);
            } else {
#pragma unroll
                for (int sub = 0; sub < SUBS; ++sub) decay_s[sub] = next_decay();
            }
            Quad P[EACH], all[SUBS];
            if constexpr (!ONLY) {
#pragma unroll
                for (int e = 0; e < EACH; ++e) {
                    Quad one = {(T)0, (T)0, (T)0, (T)0}, two = one;
#pragma unroll
                    for (int i = 0; i < PM; ++i) {
#pragma unroll
                        for (int r = 0; r < 4; ++r) (i & 1 ? two : one) = la_mma(PK[e][i][r], PQ[e][i][r], i & 1 ? two : one);
                    }
                    P[e] = one + two;
                }
            }
#pragma unroll
            for (int sub = 0; sub < SUBS; ++sub) {
                const bool last = sub + 1 == SUBS;
                const uint32_t here = n <= sub * kLaStretch ? 0 : n - sub * kLaStretch < kLaStretch ? n - sub * kLaStretch : kLaStretch;
                Quad O = {(T)0, (T)0, (T)0, (T)0}, O2 = O;
                if constexpr (!ONLY) {
#pragma unroll
                    for (int dt = 0; dt < DT; dt += 2) {
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            if (there(dt)) O = la_mma(S[dt][r], F[dt][r], O);
                            if (there(dt + 1)) O2 = la_mma(S[dt + 1][r], F[dt + 1][r], O2);
                        }
                        S[dt] *= decay_s[sub];
                        S[dt + 1] *= decay_s[sub];
                        read_k(sub, dt);
                        read_k(sub, dt + 1);
                        if (sub == 0 && dt == 0 && NW > 1) slot[slots + wave * 64 + lane] = P[0];
                        __builtin_amdgcn_sched_barrier(0);
                        if (sub == 0 && dt == 0) {
                            if constexpr (BUFFERS == 2) place(buffer ^ 1, done < total ? of_turn(done) : 0);   // (behind the last turn, for nobody)
                            fetch();
                            __builtin_amdgcn_sched_barrier(0);
                        }
                    }
                } else {
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt) S[dt] *= decay_s[sub];
                    if (sub == 0) {
                        if constexpr (BUFFERS == 2) place(buffer ^ 1, done < total ? of_turn(done) : 0);
                        fetch();
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
                Quad VW, U = V;
#pragma unroll
                for (int r = 0; r < 4; ++r) VW[r] = V[r] * decay_k[sub][r];
                if (last || (sub == 0 && NW > 1 && !ONLY)) la_meet();
                if constexpr (!ONLY) {
                    if (sub == 0) {
#pragma unroll
                        for (int to = 0; to < SUBS; ++to) {
                            if constexpr (NW > 1) {
                                all[to] = slot[slots + to * PARTS * 64 + lane];
#pragma unroll
                                for (int i = 1; i < PARTS; ++i) all[to] += slot[slots + (to * PARTS + i) * 64 + lane];
                            } else {
                                all[to] = P[to];
                            }
#pragma unroll
                            for (int r = 0; r < 4; ++r) all[to][r] = 4 * g + r <= m ? all[to][r] * decay_p[r] : (T)0;
                        }
                        if (SUBS == 1) slots ^= NW * 64;
                    }
                }
                if (last) {   // from here on what is read is the next turn's (behind the last, whatever is there)
                    if constexpr (BUFFERS == 2) buffer ^= 1;
                    qr = q_rows + buffer * KEYS, kr = k_rows + buffer * KEYS, vr = v_rows + buffer * VALUES;
                }
#pragma unroll
                for (int dt = 0; dt < DT; dt += 2) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        if (there(dt)) S[dt] = la_mma(F[dt][r], VW[r], S[dt]);
                        if (there(dt + 1)) S[dt + 1] = la_mma(F[dt + 1][r], VW[r], S[dt + 1]);
                    }
                    if constexpr (BUFFERS == 2) {
                        read_first(last ? 0 : sub + 1, dt);
                        read_first(last ? 0 : sub + 1, dt + 1);
                        if (dt == 0) read_v(last ? 0 : sub + 1);
                        if (dt == (DT > 2 ? 2 : 0) && last) read_p();
                    }
                    __builtin_amdgcn_sched_barrier(0);
                    if constexpr (!ONLY) {
                        if (dt == 0) {
                            O = (O + O2) * decay_q;
                            // A v that is no number would meet the zeros of the steps before its own: then one step at a time.
                            T odd = (T)0;
#pragma unroll
                            for (int r = 0; r < 4; ++r) odd = la_fma(U[r], (T)0, odd);
                            if (__builtin_expect(__ballot(odd != odd) == 0, 1)) {
#pragma unroll
                                for (int r = 0; r < 4; ++r) O = la_mma(U[r], all[sub][r], O);
                            } else {
#pragma unroll 1
                                for (int j = 0; j < 16; ++j) {
                                    const bool mine = (int)g == j / 4;
                                    const Quad zero = {(T)0, (T)0, (T)0, (T)0}, p = all[sub];
                                    const T vj = j % 4 == 0 ? U[0] : j % 4 == 1 ? U[1] : j % 4 == 2 ? U[2] : U[3], pj = j % 4 == 0 ? p[0] : j % 4 == 1 ? p[1] : j % 4 == 2 ? p[2] : p[3];
                                    const Quad x = la_mma(mine ? vj : (T)0, mine ? pj : (T)0, zero);
#pragma unroll
                                    for (int r = 0; r < 4; ++r) O[r] = (int)m >= j ? O[r] + x[r] : O[r];
                                }
                            }
                        }
                    }
                }
                if constexpr (BUFFERS == 1) {
                    if (last) {
                        // (one buffer: every wave has read what it needs, its rows are on their way)
                        place(0, done < total ? of_turn(done) : 0);
                        la_meet();
                        read_p();
                    }
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt) read_first(last ? 0 : sub + 1, dt);
                    read_v(last ? 0 : sub + 1);
                }
                if (!ONLY && m < here) {
                    O *= o_scale;
                    char* to = o + (int64_t)m * o_one + (uint64_t)(e0 + 4 * g) * E;
                    if constexpr (QUADS) {
                        if (e0 + 4 * g < W) __builtin_memcpy(to, &O, sizeof(O));
                    } else {
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (e0 + 4 * g + r < W) {
                                const T one = O[r];
                                __builtin_memcpy(to + r * E, &one, E);
                            }
                    }
                }
                if constexpr (!ONLY) o += o_one * (int64_t)kLaStretch;
            }
        } while (done < total);
    }

    // what is left behind, and what is not there
    {
        char* to = ONLY ? plan.starts[which] + (uint64_t)segment * bh_all * D * W * E : segment + 1 == plan.segments ? w.last : nullptr;
        const uint32_t row = ONLY ? W : w.state_row, col = ONLY ? 1 : w.state_col;
        if (to && column) {
            T* s = reinterpret_cast<T*>(to) + bh * D * W;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const uint32_t d = dt * 16 + 4 * g + r;
                    if (d < D) s[d * row + (e0 + label) * col] = S[dt][r];
                }
            }
        }
        const uint64_t behind = begin + plan.steps < c.time && segment + 1 < plan.segments ? begin + plan.steps : c.time;
        if (!ONLY && column) {
            char* z = w.o + (int64_t)b * w.o_step[0] + (int64_t)h * w.o_step[2] + (uint64_t)(e0 + label) * E;
            const T none = (T)0;
            for (uint64_t t = (begin > length ? begin : length) + g; t < behind; t += 4) __builtin_memcpy(z + (int64_t)t * w.o_step[1], &none, E);
        }
    }
}

// starts[s] from what segment s leaves by itself to what is left behind it: decay^steps times the start of s, and that. Segments are read eight
// at a time, as none waits for another (one at a time SFloat 1 x 65536 x 8 heads of 64, 63 of them, took 24 us).
template <class T>
__global__ __launch_bounds__(256) void la_starts_kernel(LaWalks walks, LaCommon c, LaPlan plan) {
    constexpr uint32_t U = 8;
    const LaWalk& w = walks.walk[blockIdx.y];
    const uint32_t size = w.dim * w.wide;
    const uint64_t all = c.batch * c.heads * size;
    for (uint64_t at = (uint64_t)blockIdx.x * 256 + threadIdx.x; at < all; at += (uint64_t)gridDim.x * 256) {
        const uint64_t bh = at / size, b = bh / c.heads;
        const uint32_t in = (uint32_t)(at - bh * size), d = in / w.wide, e = in - d * w.wide;
        const uint64_t length = la_length(c, b);
        const double a = (double)reinterpret_cast<const T*>(c.decay)[bh - b * c.heads];
        double s = w.state ? (double)reinterpret_cast<const T*>(w.state)[bh * size + d * w.state_row + e * w.state_col] : 0.0;
        T* p = reinterpret_cast<T*>(plan.starts[blockIdx.y]) + at;
        const double whole = la_power<T>(a, plan.steps).hi;
        const uint32_t n_starts = plan.segments - 1;
        for (uint32_t k = 0; k < n_starts; k += U) {
            T own[U];
#pragma unroll
            for (uint32_t u = 0; u < U; ++u) own[u] = p[(uint64_t)(k + u < n_starts ? k + u : k) * all];
#pragma unroll
            for (uint32_t u = 0; u < U; ++u) {
                if (k + u >= n_starts) continue;
                const uint64_t begin = (k + u) * plan.steps;
                const uint64_t n = begin >= length ? 0 : length - begin < plan.steps ? length - begin : plan.steps;
                s = __builtin_fma(n == plan.steps ? whole : n == 0 ? 1.0 : la_power<T>(a, n).hi, s, (double)own[u]);
                p[(uint64_t)(k + u) * all] = (T)s;
            }
        }
    }
}

template <class T, int DT, int NW, int BUFFERS, bool QUADS, bool ONLY>
void la_stretch_launch(unsigned blocks, const LaWalks& walks, const LaCommon& c, const LaPlan& p, hipStream_t stream) {
    hipLaunchKernelGGL((la_stretch_kernel<T, DT, NW, BUFFERS, QUADS, ONLY>), dim3(blocks), dim3(64 * NW), (kLaShared<T, DT, NW, BUFFERS, ONLY>), stream, walks, c, p);
}
template <class T, int DT, int NW, int BUFFERS>
void la_stretch_quads(unsigned blocks, bool only, const LaWalks& walks, const LaCommon& c, const LaPlan& p, hipStream_t stream) {
    const bool quads = walks.walk[0].dim % 4 == 0 && walks.walk[0].wide % 4 == 0;
    if (only) quads ? la_stretch_launch<T, DT, NW, BUFFERS, true, true>(blocks, walks, c, p, stream) : la_stretch_launch<T, DT, NW, BUFFERS, false, true>(blocks, walks, c, p, stream);
    else quads ? la_stretch_launch<T, DT, NW, BUFFERS, true, false>(blocks, walks, c, p, stream) : la_stretch_launch<T, DT, NW, BUFFERS, false, false>(blocks, walks, c, p, stream);
}
// Two buffers where a compute unit still holds two blocks, or gets no more than one. SFloat, heads of 128, one buffer / two: 8 x 2048 x 16 (256 blocks)
// 235 / 225 us, 32 x 2048 x 16 (1024) 823 / 898; gradients 4 x 2048 x 16 (384) 382 / 444.
template <class T, int DT, int NW>
void la_stretch_buffers(bool only, const LaWalks& walks, const LaCommon& c, const LaPlan& p, hipStream_t stream) {
    const unsigned blocks = (unsigned)((uint64_t)p.walks * p.segments * p.slices * c.batch * c.heads);
    if constexpr (2 * kLaShared<T, DT, NW, 2, false> <= 160 * 1024) {
        la_stretch_quads<T, DT, NW, 2>(blocks, only, walks, c, p, stream);
    } else {
        if constexpr (kLaTwice<T, DT, NW>)
            if (blocks <= (unsigned)device_compute_units()) return la_stretch_quads<T, DT, NW, 2>(blocks, only, walks, c, p, stream);
        la_stretch_quads<T, DT, NW, 1>(blocks, only, walks, c, p, stream);
    }
}
// Tiles of columns to a block: as many as wide has, four at most; and four where rows of dim would be too many registers for fewer lanes.
template <class T>
uint32_t la_columns(uint32_t dim, uint32_t wide) {
    const uint32_t bytes = (dim + 31) / 32 * 32 * (uint32_t)sizeof(T);
    return wide <= 16 && bytes <= 256 ? 1 : wide <= 32 && bytes <= 384 ? 2 : 4;
}
template <class T, int DT>
void la_stretch_columns(uint32_t columns, bool only, const LaWalks& walks, const LaCommon& c, const LaPlan& p, hipStream_t stream) {
    if constexpr (DT * 16 * sizeof(T) <= 256)
        if (columns == 1) return la_stretch_buffers<T, DT, 1>(only, walks, c, p, stream);
    if constexpr (DT * 16 * sizeof(T) <= 384)
        if (columns == 2) return la_stretch_buffers<T, DT, 2>(only, walks, c, p, stream);
    la_stretch_buffers<T, DT, 4>(only, walks, c, p, stream);
}
template <class T>
void la_stretch(uint32_t dim, uint32_t columns, bool only, const LaWalks& walks, const LaCommon& c, const LaPlan& p, hipStream_t stream) {
    if (dim <= 32) la_stretch_columns<T, 2>(columns, only, walks, c, p, stream);
    else if (dim <= 64) la_stretch_columns<T, 4>(columns, only, walks, c, p, stream);
    else if (dim <= 96) la_stretch_columns<T, 6>(columns, only, walks, c, p, stream);
    else if (dim <= 128) la_stretch_columns<T, 8>(columns, only, walks, c, p, stream);
    else if (dim <= 192) la_stretch_columns<T, 12>(columns, only, walks, c, p, stream);
    else la_stretch_columns<T, 16>(columns, only, walks, c, p, stream);
}

// whether a stretch's rows are within 32 bits of each other
bool la_near(const int64_t* step) { return (step[1] < 0 ? -step[1] : step[1]) <= (int64_t)1 << 26; }

// walks of one dim and one wide each, side by side
template <class T>
int la_walk(const LaWalk* w, uint32_t n, const LaCommon& c, hipStream_t stream) {
    bool near = true;
    for (uint32_t k = 0; k < n; ++k) near = near && la_near(w[k].q_step) && la_near(w[k].k_step) && la_near(w[k].v_step);
    const uint64_t heads = c.batch * c.heads, size = (uint64_t)w[0].dim * w[0].wide;
    if (c.time <= 1 || !near || !w[0].dim) {
        for (uint32_t k = 0; k < n; ++k) {
            char* memory = w[k].last;
            char* scratch = nullptr;
            if (!memory && c.time > 1 && w[k].dim) {
                scratch = cumo_cuda_runtime_malloc(heads * size * sizeof(T));
                if (!scratch) return CUMO_HIP_ERROR_OUT_OF_MEMORY;
                memory = scratch;
            }
            la_step<T>(w[k], c, memory, stream);
            if (scratch) scratch_free(scratch);
        }
        cumo_cuda_runtime_check_kernel_launch();
        return CUMO_HIP_OK;
    }
    LaWalks walks;
    for (uint32_t k = 0; k < n; ++k) walks.walk[k] = w[k];
    LaPlan p;
    p.walks = n;
    const uint32_t waves = la_columns<T>(w[0].dim, w[0].wide);
    p.slices = (w[0].wide + 16 * waves - 1) / (16 * waves);
    p.segments = 1;
    p.steps = (c.time + kLaStretch - 1) / kLaStretch * kLaStretch;
    // A sequence is cut where that leaves a block or two, as the registers allow, to each compute unit, and no segment short of 64 steps: all but
    // the last are then walked twice, the first time for half of the products.
    const uint64_t blocks = (uint64_t)n * p.slices * heads, units = (uint64_t)device_compute_units();
    if (blocks * 2 <= units) {
        uint64_t cuts = units * (w[0].dim <= (sizeof(T) == 4 ? 128 : 64) ? 2 : 1) / blocks;
        const uint64_t most = (c.time + 63) / 64;
        if (cuts > most) cuts = most;
        if (cuts > 1) {
            p.steps = ((c.time + cuts - 1) / cuts + kLaStretch - 1) / kLaStretch * kLaStretch;
            p.segments = (uint32_t)((c.time + p.steps - 1) / p.steps);
        }
    }
    char* scratch = nullptr;
    for (int k = 0; k < 3; ++k) p.starts[k] = nullptr;
    if (p.segments > 1) {
        const uint64_t bytes = (p.segments - 1) * heads * size * sizeof(T);
        if (!(scratch = cumo_cuda_runtime_malloc(n * bytes))) return CUMO_HIP_ERROR_OUT_OF_MEMORY;
        for (uint32_t k = 0; k < n; ++k) p.starts[k] = scratch + k * bytes;
        LaPlan alone = p;
        alone.segments = p.segments - 1;
        la_stretch<T>(w[0].dim, waves, true, walks, c, alone, stream);
        const uint64_t fold = (heads * size + 255) / 256;
        hipLaunchKernelGGL((la_starts_kernel<T>), dim3((unsigned)(fold < 65536 ? fold : 65536), n), dim3(256), 0, stream, walks, c, p);
    }
    la_stretch<T>(w[0].dim, waves, false, walks, c, p, stream);
    cumo_cuda_runtime_check_kernel_launch();
    if (scratch) scratch_free(scratch);
    return CUMO_HIP_OK;
}

// [batch, time, shared, group, n] contiguous into [batch, time, shared, n] with steps: the heads that share an array's head, in their order
template <class T>
__global__ __launch_bounds__(256) void la_share_kernel(const T* x, char* y, uint64_t batch, uint64_t time, uint64_t shared, uint32_t group, uint32_t n, int64_t y0, int64_t y1,
                                                       int64_t y2) {
    const uint64_t total = batch * time * shared * n;
    for (uint64_t at = (uint64_t)blockIdx.x * 256 + threadIdx.x; at < total; at += (uint64_t)gridDim.x * 256) {
        const uint64_t row = at / n, i = at - row * n, bt = row / shared, h = row - bt * shared, b = bt / time, t = bt - b * time;
        const T* from = x + row * group * n + i;
        T sum = from[0];
        for (uint32_t g = 1; g < group; ++g) sum += from[(uint64_t)g * n];
        reinterpret_cast<T*>(y + (int64_t)b * y0 + (int64_t)t * y1 + (int64_t)h * y2)[i] = sum;
    }
}

void la_steps(int64_t* to, const ssize_t* from) {
    for (int k = 0; k < 3; ++k) to[k] = from[k];
}

template <class T>
int la_forward(const cumo_hip_linear_attention_t& d, hipStream_t stream) {
    if (!d.batch || !d.heads || !d.wide) return CUMO_HIP_OK;
    LaCommon c = {d.batch, d.time, d.heads, d.decay, d.lengths};
    LaWalk w;
    const uint32_t share = (uint32_t)(d.heads / d.shared);
    w.q = d.q, w.k = d.k, w.v = d.v, w.state = d.state, w.o = d.o, w.last = d.last;
    la_steps(w.q_step, d.q_step), la_steps(w.k_step, d.k_step), la_steps(w.v_step, d.v_step), la_steps(w.o_step, d.o_step);
    w.q_share = 1, w.k_share = w.v_share = share;
    w.dim = (uint32_t)d.dim, w.wide = (uint32_t)d.wide;
    w.state_row = w.wide, w.state_col = 1;
    w.o_scale = d.scale, w.k_scale = 1.0;
    w.backwards = false;
    return la_walk<T>(&w, 1, c, stream);
}

template <class T>
int la_backward(const cumo_hip_linear_attention_grad_t& d, hipStream_t stream) {
    if (!d.batch || !d.heads) return CUMO_HIP_OK;
    LaCommon c = {d.batch, d.time, d.heads, d.decay, d.lengths};
    const uint32_t share = (uint32_t)(d.heads / d.shared), dim = (uint32_t)d.dim, wide = (uint32_t)d.wide;
    const uint64_t rows = d.batch * d.time * d.heads;
    // gradients of heads that are shared, before their sum
    char* parts = nullptr;
    if (share > 1 && rows * (dim + wide) && !(parts = cumo_cuda_runtime_malloc(rows * (dim + wide) * sizeof(T)))) return CUMO_HIP_ERROR_OUT_OF_MEMORY;
    char* const part_k = parts;
    char* const part_v = parts ? parts + rows * dim * sizeof(T) : nullptr;
    const int64_t e = sizeof(T), heads = (int64_t)d.heads, time = (int64_t)d.time;
    LaWalk walk[3];
    LaWalk &wq = walk[0], &wk = walk[1], &wv = walk[2];
    wq.q = d.g, wq.k = d.v, wq.v = d.k, wq.state = d.state, wq.o = d.gq, wq.last = nullptr;
    la_steps(wq.q_step, d.g_step), la_steps(wq.k_step, d.v_step), la_steps(wq.v_step, d.k_step), la_steps(wq.o_step, d.gq_step);
    wq.q_share = 1, wq.k_share = wq.v_share = share;
    wq.dim = wide, wq.wide = dim, wq.state_row = 1, wq.state_col = wide;
    wq.o_scale = d.scale, wq.k_scale = 1.0, wq.backwards = false;

    wk.q = d.v, wk.k = d.g, wk.v = d.q, wk.state = d.glast, wk.o = d.gk, wk.last = nullptr;
    la_steps(wk.q_step, d.v_step), la_steps(wk.k_step, d.g_step), la_steps(wk.v_step, d.q_step), la_steps(wk.o_step, d.gk_step);
    if (parts) wk.o = part_k, wk.o_step[0] = time * heads * dim * e, wk.o_step[1] = heads * dim * e, wk.o_step[2] = dim * e;
    wk.q_share = share, wk.k_share = wk.v_share = 1;
    wk.dim = wide, wk.wide = dim, wk.state_row = 1, wk.state_col = wide;
    wk.o_scale = 1.0, wk.k_scale = d.scale, wk.backwards = true;

    wv.q = d.k, wv.k = d.q, wv.v = d.g, wv.state = d.glast, wv.o = d.gv, wv.last = d.gstate;
    la_steps(wv.q_step, d.k_step), la_steps(wv.k_step, d.q_step), la_steps(wv.v_step, d.g_step), la_steps(wv.o_step, d.gv_step);
    if (parts) wv.o = part_v, wv.o_step[0] = time * heads * wide * e, wv.o_step[1] = heads * wide * e, wv.o_step[2] = wide * e;
    wv.q_share = share, wv.k_share = wv.v_share = 1;
    wv.dim = dim, wv.wide = wide, wv.state_row = wide, wv.state_col = 1;
    wv.o_scale = 1.0, wv.k_scale = d.scale, wv.backwards = true;

    int rc = CUMO_HIP_OK;
    if (dim == wide) {
        if (dim) rc = la_walk<T>(walk, 3, c, stream);
    } else {
        if (dim) rc = la_walk<T>(walk, 2, c, stream);
        if (!rc && wide) rc = la_walk<T>(walk + 2, 1, c, stream);
    }
    if (!rc && parts) {
        for (int k = 0; k < 2; ++k) {
            const uint32_t n = k ? wide : dim;
            const uint64_t blocks = (d.batch * d.time * d.shared * n + 255) / 256;
            const ssize_t* step = k ? d.gv_step : d.gk_step;
            if (blocks)
                hipLaunchKernelGGL((la_share_kernel<T>), dim3((unsigned)(blocks < 65536 ? blocks : 65536)), dim3(256), 0, stream, reinterpret_cast<const T*>(k ? part_v : part_k),
                                   k ? d.gv : d.gk, d.batch, d.time, d.shared, share, n, step[0], step[1], step[2]);
        }
        cumo_cuda_runtime_check_kernel_launch();
    }
    if (parts) scratch_free(parts);
    return rc;
}

}  // namespace
}  // namespace cumo_hip
