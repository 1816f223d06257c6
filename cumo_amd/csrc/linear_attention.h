// Linear attention with a decay for each head, S[t] = a S[t-1] + k[t] (x) v[t], o[t] = scale (S[t] by q[t]), and its gradients.
//
// A walk is this: from q, k (of `dim` elements) and v, o (of `wide`), forwards or backwards in time. With G[t] what the loss has for S[t],
// G[t] = a G[t+1] + scale q[t] (x) g[t], the gradients are three walks more:
//   gq[t] = scale (S[t] by g[t]):  g in the place of q, v of k, k of v, the state transposed
//   gk[t] = G[t] by v[t]:          backwards, v in the place of q, scale g of k, q of v, the state transposed
//   gv[t] = G[t] by k[t]:          backwards, k in the place of q, scale q of k, g of v
// Backwards the state decays behind a step instead of before it (`late`): what is handed on is a G.
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

// One step, or one after the other where a walk is not one for stretches. LPR lanes hold VE columns each of a row of S, the block's other
// lanes other rows, each a run of them; S goes through memory from step to step (`memory`: last, or scratch), which every lane reads as it
// wrote it. A step is bound by the state's bytes: a lane has U vectors of it on their way at a time.
constexpr int kLaStepBlock = 256;
template <class T, int VE> struct LaColumns { T t[VE]; };
template <class T, int VE, int LPR, bool LATE>
__global__ __launch_bounds__(kLaStepBlock) void la_step_kernel(LaWalk w, LaCommon c, char* memory, uint32_t slices) {
    constexpr int RG = kLaStepBlock / LPR, U = 8;
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
            __builtin_memcpy(&x, p, sizeof(x));
        } else {
#pragma unroll
            for (int j = 0; j < VE; ++j) x.t[j] = p[(uint64_t)j * w.state_col];
        }
        return x;
    };
    auto write = [&](uint32_t d, const Columns& x) {
        T* p = to + (uint64_t)d * w.state_row + (uint64_t)e * w.state_col;
        if (near) {
            __builtin_memcpy(p, &x, sizeof(x));
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
        __syncthreads();
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
            if (d == d0) __syncthreads();
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
        __syncthreads();
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
    if (w.backwards) hipLaunchKernelGGL((la_step_kernel<T, VE, LPR, true>), grid, block, 0, stream, w, c, memory, slices);
    else hipLaunchKernelGGL((la_step_kernel<T, VE, LPR, false>), grid, block, 0, stream, w, c, memory, slices);
}

template <class T>
void la_step(const LaWalk& w, const LaCommon& c, char* memory, hipStream_t stream) {
    constexpr int V = 16 / (int)sizeof(T);
    if (w.wide % V == 0) {
        if (w.wide <= 16 * V) la_step_one<T, V, 16>(w, c, memory, stream);
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
// which each of the NW waves works out a share, over its part of dim: they meet in LDS, one barrier a stretch. Operands are read straight
// from memory as the lanes want them, each as soon as its predecessor has been used, so that they are on their way for most of a stretch.
//
// Double precision counts rows otherwise (lane (m, g) has rows g, g + 4, ...): operands are read by la_label, so that what
// stands above holds for it too.
template <class T> using LaQuad = T __attribute__((ext_vector_type(4)));
__device__ __forceinline__ LaQuad<float> la_mma(float a, float b, LaQuad<float> c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }
__device__ __forceinline__ LaQuad<double> la_mma(double a, double b, LaQuad<double> c) { return __builtin_amdgcn_mfma_f64_16x16x4f64(a, b, c, 0, 0, 0); }
template <class T> __device__ __forceinline__ uint32_t la_label(uint32_t m) { return sizeof(T) == 4 ? m : 4 * (m & 3) + (m >> 2); }

// a^n by squares, n >= 0; in double
__device__ __forceinline__ double la_power(double a, uint64_t n) {
    double p = 1.0;
    for (; n; n >>= 1) {
        if (n & 1) p *= a;
        a *= a;
    }
    return p;
}

constexpr uint32_t kLaStretch = 16;
struct LaPlan {
    uint32_t walks, segments, slices;
    uint64_t steps;         // of a segment, a multiple of kLaStretch
    char* starts[3];        // [segments - 1][batch * heads][dim * wide]: the state that each segment but the last leaves to the next, by walk
};
struct LaWalks {
    LaWalk walk[3];
};

// rows of an array as a stretch takes them, in its direction: from `low`, unsigned offsets
struct LaRows {
    const char* low;
    int64_t advance;
    uint32_t step;
    bool down;
    __device__ __forceinline__ LaRows(const char* p, const int64_t* steps, uint64_t b, uint64_t h, uint64_t first, bool backwards) {
        const int64_t one = backwards ? -steps[1] : steps[1];
        down = one < 0;
        step = (uint32_t)(down ? -one : one);
        advance = one * (int64_t)kLaStretch;
        low = p + (int64_t)b * steps[0] + (int64_t)h * steps[2] + (int64_t)first * steps[1] + (down ? one * (int64_t)(kLaStretch - 1) : 0);
    }
    __device__ __forceinline__ uint32_t row(uint32_t k) const { return (down ? kLaStretch - 1 - k : k) * step; }
};
template <class T>
__device__ __forceinline__ T la_at(const char* low, uint32_t offset) {
    T v;
    __builtin_memcpy(&v, low + offset, sizeof(T));
    return v;
}

// DT: tiles of 16 that hold dim, of which the first FULL are whole. QUADS: rows of dim and of wide are whole fours. ONLY: what a segment
// leaves by itself. Tiles of q and of k's columns are held a ring of RING at a time, each read again as soon as it has been used.
template <class T, int DT> constexpr int kLaRing = DT <= (sizeof(T) == 4 ? 8 : 4) ? DT : DT % 4 == 0 ? 4 : 3;
template <class T, int DT> constexpr int kLaWavesPerSimd = sizeof(T) * DT <= 64 ? 2 : 1;

template <class T, int DT, int FULL, int NW, bool QUADS, bool ONLY>
__global__ __launch_bounds__(64 * NW, (kLaWavesPerSimd<T, DT>)) void la_stretch_kernel(LaWalks walks, LaCommon c, LaPlan plan) {
    typedef LaQuad<T> Quad;
    constexpr uint32_t E = sizeof(T);
    constexpr int PM = (DT + NW - 1) / NW, RING = kLaRing<T, DT>;
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, m = lane & 15, g = lane >> 4, label = la_label<T>(m);
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
    const uint64_t total = end > begin ? end - begin : 0;
    const uint32_t e0 = (slice * NW + wave) * 16;             // the wave's columns
    const uint32_t e_in = e0 + label < W ? e0 + label : W - 1;  // (columns behind the last are computed as that one, and not written)
    const bool column = e0 + label < W;
    const double a = (double)reinterpret_cast<const T*>(c.decay)[h];
    const bool late = w.backwards;

    // the state
    Quad S[DT];
    {
        const char* from = segment == 0 || ONLY ? w.state : plan.starts[which] + (uint64_t)(segment - 1) * bh_all * D * W * E;
        const uint32_t row = segment == 0 ? w.state_row : W, col = segment == 0 ? w.state_col : 1;
        const T* s = reinterpret_cast<const T*>(from) + bh * D * W;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) S[dt] = Quad{(T)0, (T)0, (T)0, (T)0};
        if (!ONLY && from) {
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const uint32_t d = dt * 16 + 4 * g + r;
                    S[dt][r] = s[(d < D ? d : D - 1) * row + e_in * col];   // (rows behind the last meet zeros of q, and are not written)
                }
            }
        }
    }

    const uint64_t first = w.backwards ? (length ? length - 1 - begin : 0) : begin;
    LaRows q(w.q, w.q_step, b, h / w.q_share, first, w.backwards), k(w.k, w.k_step, b, h / w.k_share, first, w.backwards), v(w.v, w.v_step, b, h / w.v_share, first, w.backwards);
    char* o = w.o + (int64_t)b * w.o_step[0] + (int64_t)h * w.o_step[2] + (int64_t)first * w.o_step[1];
    const int64_t o_one = w.backwards ? -w.o_step[1] : w.o_step[1];

    // where the lanes read, for stretches of n steps (rows behind the last are read as that one)
    uint32_t q_at, k_at, v_at[4], kc_at[4];
    auto places = [&](uint32_t n) {
        auto in = [&](uint32_t row) { return row < n ? row : n - 1; };
        q_at = q.row(in(m));
        k_at = k.row(in(label));
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            kc_at[r] = k.row(in(4 * g + r));
            v_at[r] = v.row(in(4 * g + r)) + e_in * E;
        }
    };
    // four neighbours of a row from d on; behind the end of dim anything that is there
    auto quad = [&](const char* low, uint32_t row, uint32_t d) {
        Quad x;
        if constexpr (QUADS) {
            __builtin_memcpy(&x, low + (row + (d < D ? d : D - 4) * E), sizeof(x));
        } else {
#pragma unroll
            for (int r = 0; r < 4; ++r) x[r] = la_at<T>(low, row + (d + r < D ? d + r : D - 1) * E);
        }
        return x;
    };
    auto cut = [&](Quad x, uint32_t d) {
#pragma unroll
        for (int r = 0; r < 4; ++r) x[r] = d + r < D ? x[r] : (T)0;
        return x;
    };

    Quad Q[RING], KC[RING], V, PQ[PM], PK[PM];
    auto read_q = [&](int dt) {
        if (QUADS && dt < FULL) __builtin_memcpy(&Q[dt % RING], q.low + (q_at + (dt * 16 + 4 * g) * E), sizeof(Quad));
        else Q[dt % RING] = quad(q.low, q_at, dt * 16 + 4 * g);
    };
    auto read_p = [&] {
#pragma unroll
        for (int i = 0; i < PM; ++i) {
            const uint32_t d = (wave + NW * i) * 16 + 4 * g;
            PQ[i] = quad(q.low, q_at, d);
            PK[i] = quad(k.low, k_at, d);
        }
    };
    auto read_v = [&] {
#pragma unroll
        for (int r = 0; r < 4; ++r) V[r] = la_at<T>(v.low, v_at[r]);
    };
    auto read_k = [&](int dt) {
        const uint32_t d = dt * 16 + label, col = (dt < FULL || d < D ? d : D - 1) * E;
#pragma unroll
        for (int r = 0; r < 4; ++r) KC[dt % RING][r] = la_at<T>(k.low, kc_at[r] + col);
    };

    // decays: of the products of step i = m with steps j = 4 g + r, of what S gives to step i, of what step j leaves
    T decay_p[4], decay_k[4], decay_q, decay_s;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const uint32_t j = 4 * g + r;
        decay_p[r] = j <= m ? (T)(la_power(a, m - j) * w.k_scale) : (T)0;
    }
    decay_q = (T)la_power(a, m + (late ? 0 : 1));
    auto ends = [&](uint32_t n) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const uint32_t j = 4 * g + r;
            decay_k[r] = j < n ? (T)(la_power(a, n - 1 - j + (late ? 1 : 0)) * w.k_scale) : (T)0;
        }
        decay_s = (T)la_power(a, n);
    };

    __shared__ Quad slot[NW > 1 && !ONLY ? 2 : 1][NW][64];
    uint64_t left = total;
    if (left) {
    {
        const uint32_t n = left < kLaStretch ? (uint32_t)left : kLaStretch;
        places(n);
        ends(n);
        // (in the order of the loop below: what a turn waits for is counted from the last load)
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (!ONLY) {
            read_p();
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int dt = 0; dt < RING; ++dt) {
                read_q(dt);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        read_v();
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int dt = 0; dt < RING; ++dt) {
            read_k(dt);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    uint32_t turn = 0;
    do {
        const uint32_t n = left < kLaStretch ? (uint32_t)left : kLaStretch;
        left -= n;
        const uint32_t next = left < kLaStretch ? (uint32_t)left : kLaStretch;
        // What is read ahead is of the next stretch; behind the last, of that one again. (Tiles that the rings do not hold yet are of this one.)
        const char *q_low = q.low, *k_low = k.low;
        const uint32_t q_was = q_at;
        uint32_t kc_was[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) kc_was[r] = kc_at[r];
        if (next) {
            q.low += q.advance;
            k.low += k.advance;
            v.low += v.advance;
            if (next < kLaStretch) places(next);
        }
        auto tile_q = [&](int dt) {   // into the ring behind tile dt
            if (dt + RING < DT) {
                const char* low = q.low;
                const uint32_t here = q_at;
                q.low = q_low, q_at = q_was;
                read_q(dt + RING);
                q.low = low, q_at = here;
            } else {
                read_q(dt + RING - DT);
            }
        };
        auto tile_k = [&](int dt) {
            if (dt + RING < DT) {
                const char* low = k.low;
                uint32_t here[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) here[r] = kc_at[r], kc_at[r] = kc_was[r];
                k.low = k_low;
                read_k(dt + RING);
                k.low = low;
#pragma unroll
                for (int r = 0; r < 4; ++r) kc_at[r] = here[r];
            } else {
                read_k(dt + RING - DT);
            }
        };
        if constexpr (!ONLY) {
            Quad P = {(T)0, (T)0, (T)0, (T)0};
#pragma unroll
            for (int i = 0; i < PM; ++i) {
                const Quad x = cut(PQ[i], (wave + NW * i) * 16 + 4 * g);
#pragma unroll
                for (int r = 0; r < 4; ++r) P = la_mma(PK[i][r], x[r], P);
            }
            read_p();
            if constexpr (NW > 1) slot[turn & 1][wave][lane] = P;
            Quad O = {(T)0, (T)0, (T)0, (T)0};
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                const Quad x = dt < FULL ? Q[dt % RING] : cut(Q[dt % RING], dt * 16 + 4 * g);
#pragma unroll
                for (int r = 0; r < 4; ++r) O = la_mma(S[dt][r], x[r], O);
                tile_q(dt);
            }
            O *= decay_q;
            if constexpr (NW > 1) {
                __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
                __builtin_amdgcn_s_barrier();
                __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
                P = slot[turn & 1][0][lane];
#pragma unroll
                for (int i = 1; i < NW; ++i) P += slot[turn & 1][i][lane];
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) P[r] = 4 * g + r <= m ? P[r] * decay_p[r] : (T)0;
            // A v that is no number would meet the zeros of the steps before its own: then one step at a time.
            T odd = (T)0;
#pragma unroll
            for (int r = 0; r < 4; ++r) odd = la_fma(V[r], (T)0, odd);
            if (__builtin_expect(__ballot(odd != odd) == 0, 1)) {
#pragma unroll
                for (int r = 0; r < 4; ++r) O = la_mma(V[r], P[r], O);
            } else {
#pragma unroll 1
                for (int j = 0; j < 16; ++j) {
                    const bool mine = (int)g == j / 4;
                    const Quad zero = {(T)0, (T)0, (T)0, (T)0};
                    const T vj = j % 4 == 0 ? V[0] : j % 4 == 1 ? V[1] : j % 4 == 2 ? V[2] : V[3], pj = j % 4 == 0 ? P[0] : j % 4 == 1 ? P[1] : j % 4 == 2 ? P[2] : P[3];
                    const Quad x = la_mma(mine ? vj : (T)0, mine ? pj : (T)0, zero);
#pragma unroll
                    for (int r = 0; r < 4; ++r) O[r] = (int)m >= j ? O[r] + x[r] : O[r];
                }
            }
            if (m < n) {
                O *= (T)w.o_scale;
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
            o += o_one * (int64_t)kLaStretch;
        }
        Quad VW;
#pragma unroll
        for (int r = 0; r < 4; ++r) VW[r] = 4 * g + r < n ? V[r] * decay_k[r] : (T)0;
        read_v();
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
            S[dt] *= decay_s;
#pragma unroll
            for (int r = 0; r < 4; ++r) S[dt] = la_mma(KC[dt % RING][r], VW[r], S[dt]);
            tile_k(dt);
        }
        if (next < kLaStretch && next) ends(next);
        ++turn;
    } while (left);
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
        if (!ONLY && g == 0 && column) {
            char* z = w.o + (int64_t)b * w.o_step[0] + (int64_t)h * w.o_step[2] + (uint64_t)(e0 + label) * E;
            const T none = (T)0;
            for (uint64_t t = begin > length ? begin : length; t < behind; ++t) __builtin_memcpy(z + (int64_t)t * w.o_step[1], &none, E);
        }
    }
}

// starts[s] from what segment s leaves by itself to what is left behind it: decay^steps times the start of s, and that
template <class T>
__global__ __launch_bounds__(256) void la_starts_kernel(LaWalks walks, LaCommon c, LaPlan plan) {
    const LaWalk& w = walks.walk[blockIdx.y];
    const uint64_t size = (uint64_t)w.dim * w.wide, all = c.batch * c.heads * size;
    for (uint64_t at = (uint64_t)blockIdx.x * 256 + threadIdx.x; at < all; at += (uint64_t)gridDim.x * 256) {
        const uint64_t bh = at / size, in = at - bh * size, b = bh / c.heads, h = bh - b * c.heads, d = in / w.wide, e = in - d * w.wide;
        const uint64_t length = la_length(c, b);
        const double a = (double)reinterpret_cast<const T*>(c.decay)[h];
        T s = w.state ? reinterpret_cast<const T*>(w.state)[bh * size + d * w.state_row + e * w.state_col] : (T)0;
        T* p = reinterpret_cast<T*>(plan.starts[blockIdx.y]) + at;
        const T whole = (T)la_power(a, plan.steps);
        for (uint32_t k = 0; k + 1 < plan.segments; ++k) {
            const uint64_t begin = k * plan.steps;
            const uint64_t n = begin >= length ? 0 : length - begin < plan.steps ? length - begin : plan.steps;
            s = la_fma(n == plan.steps ? whole : (T)la_power(a, n), s, p[k * all]);
            p[k * all] = s;
        }
    }
}

template <class T, int DT, int FULL, int NW, bool QUADS, bool ONLY>
void la_stretch_launch(const LaWalks& walks, const LaCommon& c, const LaPlan& p, hipStream_t stream) {
    const uint64_t blocks = (uint64_t)p.walks * p.segments * p.slices * c.batch * c.heads;
    hipLaunchKernelGGL((la_stretch_kernel<T, DT, FULL, NW, QUADS, ONLY>), dim3((unsigned)blocks), dim3(64 * NW), 0, stream, walks, c, p);
}
template <class T, int DT, int FULL, int NW>
void la_stretch_quads(bool only, const LaWalks& walks, const LaCommon& c, const LaPlan& p, hipStream_t stream) {
    if (only) la_stretch_launch<T, DT, FULL, NW, true, true>(walks, c, p, stream);
    else if (walks.walk[0].dim % 4 == 0 && walks.walk[0].wide % 4 == 0) la_stretch_launch<T, DT, FULL, NW, true, false>(walks, c, p, stream);
    else la_stretch_launch<T, DT, FULL, NW, false, false>(walks, c, p, stream);
}
template <class T, int DT, int FULL>
void la_stretch_waves(uint32_t waves, bool only, const LaWalks& walks, const LaCommon& c, const LaPlan& p, hipStream_t stream) {
    if (waves == 1) la_stretch_quads<T, DT, FULL, 1>(only, walks, c, p, stream);
    else if (waves == 2) la_stretch_quads<T, DT, FULL, 2>(only, walks, c, p, stream);
    else la_stretch_quads<T, DT, FULL, 4>(only, walks, c, p, stream);
}
template <class T>
void la_stretch(uint32_t dim, uint32_t waves, bool only, const LaWalks& walks, const LaCommon& c, const LaPlan& p, hipStream_t stream) {
    if (dim <= 32) la_stretch_waves<T, 2, 0>(waves, only, walks, c, p, stream);
    else if (dim <= 64) la_stretch_waves<T, 4, 2>(waves, only, walks, c, p, stream);
    else if (dim <= 96) la_stretch_waves<T, 6, 4>(waves, only, walks, c, p, stream);
    else if (dim <= 128) la_stretch_waves<T, 8, 6>(waves, only, walks, c, p, stream);
    else if (dim <= 192) la_stretch_waves<T, 12, 8>(waves, only, walks, c, p, stream);
    else la_stretch_waves<T, 16, 12>(waves, only, walks, c, p, stream);
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
    const uint32_t waves = w[0].wide <= 16 ? 1 : w[0].wide <= 32 ? 2 : 4;
    p.slices = (w[0].wide + 16 * waves - 1) / (16 * waves);
    p.segments = 1;
    p.steps = (c.time + kLaStretch - 1) / kLaStretch * kLaStretch;
    const uint64_t blocks = (uint64_t)n * p.slices * heads;
    const uint64_t wanted = 1024 / waves;   // a wave to every SIMD
    if (blocks * 2 <= wanted) {
        uint64_t cuts = wanted * 2 / blocks;
        const uint64_t most = (c.time + 255) / 256;
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
    LaCommon c = {d.batch, d.time, d.heads, d.decay, d.lengths};
    const uint32_t share = (uint32_t)(d.heads / d.shared), dim = (uint32_t)d.dim, wide = (uint32_t)d.wide;
    const uint64_t rows = d.batch * d.time * d.heads;
    // gradients of heads that are shared, before their sum
    char* parts = nullptr;
    if (share > 1 && !(parts = cumo_cuda_runtime_malloc(rows * (dim + wide) * sizeof(T)))) return CUMO_HIP_ERROR_OUT_OF_MEMORY;
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
