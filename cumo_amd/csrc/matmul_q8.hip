// The product of 8-bit rows by 8-bit rows, y[i][j] = (sum of x[i][k] w[j][k]) xscale[i] wscale[j] + bias[j], by matrix instructions of
// 16 x 16 x 64 bytes whose sums are 32-bit integers: exact, in whatever order, so that how inner is cut changes no bit.
//
// w is the first operand and x the second: a lane has four neighbouring numbers of a row of y. What follows the sum is in double, the products by the two
// scales and the bias one after the other, and then rounded to y's type.
//
// Few rows are bound by w's bytes on their way through the last-level cache: SFloat 16 x 4096 by 4096 7.5 us, 2.3 TB/s, three of them the launch's.
// Many: 8191 x 4096 by 8192 266 us, 2.07 POP/s; the library's product of bytes, without scales, takes 241 (of 8192 cubed 437, 2.5 POP/s, and this one 481). The
// matrix units are busy for half of the waves' cycles, LDS for a third, no bank met twice: what a step waits for is its rows on their way, 64 KiB of them. With rows placed in the step in which they
// are sent for, and LDS read just before its products, 280 us; four waves of 128 x 128 each, which spill, 345.
#include "common.h"

namespace cumo_hip {
namespace {

typedef int32_t mq_i4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ mq_i4 mq_mma(mq_i4 a, mq_i4 b, mq_i4 c) { return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0); }

// the block's waves meet, for what LDS holds alone
__device__ __forceinline__ void mq_meet() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// sixteen bytes on any boundary
__device__ __forceinline__ mq_i4 mq_read(const char* p) {
    mq_i4 v;
    __builtin_memcpy(&v, p, 16);
    return v;
}
// the first n of them, zeros behind (n may be 0 or less: nothing is read)
__device__ __forceinline__ mq_i4 mq_read_part(const char* p, int64_t n) {
    if (n >= 16) return mq_read(p);
    union { mq_i4 v; int8_t b[16]; } u;
    u.v = mq_i4{0, 0, 0, 0};
#pragma unroll
    for (int k = 0; k < 15; ++k) u.b[k] = k < n ? (int8_t)p[k] : (int8_t)0;
    return u.v;
}

// sixteen bytes of a row of which some, on the way to p, are behind its end: those before it (sixteen at least), moved down, and zeros
__device__ __forceinline__ mq_i4 mq_read_end(const char* p, int64_t behind) {
    if (behind <= 0) return mq_read(p);
    unsigned __int128 u;
    __builtin_memcpy(&u, p - behind, 16);
    u = behind < 16 ? u >> (8 * (uint32_t)behind) : 0;
    mq_i4 v;
    __builtin_memcpy(&v, &u, 16);
    return v;
}

struct MqParams : cumo_hip_matmul_q8_t {
    int32_t* parts;    // [splits][rows][cols], where inner is cut
    uint32_t splits;
    uint64_t per;      // bytes of a row that a split takes
    uint32_t tiles_m, tiles_n;
};

template <class T> struct __attribute__((aligned(16))) MqFour { T t[4]; };
// what stands beside four numbers of a row of y: scales of w, and the bias
template <class T>
struct MqBeside {
    double scale[4], bias[4];
    __device__ __forceinline__ void read(const cumo_hip_matmul_q8_t& p, uint64_t j) {
        const T* ws = reinterpret_cast<const T*>(p.wscale);
        const T* bs = reinterpret_cast<const T*>(p.bias);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const uint64_t at = j + r < p.cols ? j + r : p.cols - 1;
            scale[r] = (double)ws[at];
            bias[r] = bs ? (double)bs[at] : 0.0;
        }
    }
};
// Four numbers of a row of y from column j on, from their sums; `row`: where the row starts. NT: past the caches. (What is beside them is read before the
// first is written: y may be any memory for all that the compiler knows, and each would wait for the one before.)
template <class T, bool NT>
__device__ __forceinline__ void mq_put(char* row, uint64_t j, uint64_t cols, bool biased, double xs, const MqBeside<T>& beside, mq_i4 sum) {
    MqFour<T> out;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const double v = (double)sum[r] * xs;
        out.t[r] = (T)(biased ? __builtin_fma(v, beside.scale[r], beside.bias[r]) : v * beside.scale[r]);
    }
    T* y = reinterpret_cast<T*>(row) + j;
    if (j + 4 <= cols) {
        if constexpr (NT) {
            const store_u4* from = reinterpret_cast<const store_u4*>(&out);
#pragma unroll
            for (int k = 0; k < (int)(sizeof(out) / 16); ++k) __builtin_nontemporal_store(from[k], reinterpret_cast<store_u4*>(y) + k);
        } else {
            __builtin_memcpy(y, &out, sizeof(out));
        }
    } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (j + r < cols) y[r] = out.t[r];
    }
}

// ---- few rows: a block takes sixteen rows of w, its waves every WAVES-th piece of inner, TM sixteens of x's rows --------------------------------------
template <class T, int TM, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void matmul_q8_rows_kernel(cumo_hip_matmul_q8_t p) {
    constexpr int U = TM <= 2 ? 4 : TM <= 4 ? 2 : 1;  // pieces of 64 on their way at a time
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, m = lane & 15, g = lane >> 4;
    const uint64_t j0 = (uint64_t)blockIdx.x * 16;
    const uint64_t wrow = j0 + m < p.cols ? j0 + m : p.cols - 1;
    const char* w = p.w + (int64_t)wrow * p.w_step + g * 16;
    const char* x[TM];
#pragma unroll
    for (int t = 0; t < TM; ++t) {
        const uint64_t row = (uint64_t)t * 16 + m;
        x[t] = p.x + (int64_t)(row < p.rows ? row : p.rows - 1) * p.x_step + g * 16;
    }
    mq_i4 sum[TM];
#pragma unroll
    for (int t = 0; t < TM; ++t) sum[t] = mq_i4{0, 0, 0, 0};
    const uint64_t whole = p.inner / 64;
    uint64_t piece = wave;
    for (; piece + (U - 1) * WAVES < whole; piece += U * WAVES) {
        mq_i4 a[U], b[U][TM];
#pragma unroll
        for (int u = 0; u < U; ++u) a[u] = mq_read(w + (piece + u * WAVES) * 64);
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int t = 0; t < TM; ++t) b[u][t] = mq_read(x[t] + (piece + u * WAVES) * 64);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int t = 0; t < TM; ++t) sum[t] = mq_mma(a[u], b[u][t], sum[t]);
        }
    }
    for (; piece * 64 < p.inner; piece += WAVES) {
        const int64_t n = (int64_t)(p.inner - piece * 64) - g * 16;
        const mq_i4 a = mq_read_part(w + piece * 64, n);
#pragma unroll
        for (int t = 0; t < TM; ++t) sum[t] = mq_mma(a, mq_read_part(x[t] + piece * 64, n), sum[t]);
    }
    __shared__ mq_i4 slot[WAVES][TM][64];
#pragma unroll
    for (int t = 0; t < TM; ++t) slot[wave][t][lane] = sum[t];
    __syncthreads();
    for (uint32_t t = wave; t < TM; t += WAVES) {
        mq_i4 all = slot[0][t][lane];
#pragma unroll
        for (int k = 1; k < WAVES; ++k) all += slot[k][t][lane];
        const uint64_t i = (uint64_t)t * 16 + m, j = j0 + 4 * g;
        if (i < p.rows && j < p.cols) {
            MqBeside<T> beside;
            beside.read(p, j);
            mq_put<T, false>(p.y + (int64_t)i * p.y_step, j, p.cols, p.bias != nullptr, (double)reinterpret_cast<const T*>(p.xscale)[i], beside, all);
        }
    }
}

// ---- tiles: BM rows of x by BN of w, 128 bytes of inner at a time through LDS -----------------------------------------------------------
// A row's eight pieces of sixteen bytes lie in its 128 bytes of LDS in the order piece ^ (row % 8), so that lanes that read one piece of
// neighbouring rows, and those that write a row, meet in no bank.
constexpr uint32_t kMqDepth = 128;

template <class T, int BM, int BN, int WM, int WN, bool NT>
__global__ __launch_bounds__(64 * WM * WN) void matmul_q8_tiles_kernel(MqParams p) {
    constexpr int THREADS = 64 * WM * WN, TM = BM / WM / 16, TN = BN / WN / 16, PIECES = (BM + BN) * 8 / THREADS;
    __shared__ __attribute__((aligned(16))) char tile[2][(BM + BN) * kMqDepth];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, m = lane & 15, g = lane >> 4;
    const uint32_t tiles = p.tiles_m * p.tiles_n, part = blockIdx.x / tiles;
    uint32_t at = blockIdx.x % tiles;
    // blocks go to the eight dies in turn: each die takes a run of tiles, in strips of eight tiles of x
    if (tiles % 8 == 0) at = (at % 8) * (tiles / 8) + at / 8;
    const uint32_t strip = at / (8 * p.tiles_n), in = at % (8 * p.tiles_n);
    const uint32_t high = p.tiles_m - strip * 8 < 8 ? p.tiles_m - strip * 8 : 8;
    const uint64_t i0 = (uint64_t)(strip * 8 + in % high) * BM, j0 = (uint64_t)(in / high) * BN;
    const uint64_t from = part * p.per, to = from + p.per < p.inner ? from + p.per : p.inner;

    const char* src[PIECES];
    constexpr uint32_t STEP = THREADS / 8;   // rows from piece to piece of a lane
    static_assert(STEP % 8 == 0, "a lane's pieces lie alike in their rows");
    const uint32_t dst = threadIdx.x / 8 * kMqDepth + ((threadIdx.x % 8 ^ (threadIdx.x / 8 & 7)) * 16);
#pragma unroll
    for (int k = 0; k < PIECES; ++k) {
        const uint32_t id = threadIdx.x + k * THREADS, row = id / 8, piece = id % 8;
        if (row < BM) {
            const uint64_t i = i0 + row < p.rows ? i0 + row : p.rows - 1;
            src[k] = p.x + (int64_t)i * p.x_step + piece * 16;
        } else {
            const uint64_t j = j0 + row - BM < p.cols ? j0 + row - BM : p.cols - 1;
            src[k] = p.w + (int64_t)j * p.w_step + piece * 16;
        }
    }
    mq_i4 held[PIECES];
    auto fetch = [&](uint64_t k0) {
        if (k0 + kMqDepth <= to) {
#pragma unroll
            for (int k = 0; k < PIECES; ++k) held[k] = mq_read(src[k] + k0);
        } else if (to >= 16) {
            const int64_t behind = (int64_t)(k0 + (threadIdx.x % 8) * 16 + 16 - to);
#pragma unroll
            for (int k = 0; k < PIECES; ++k) held[k] = mq_read_end(src[k] + k0, behind);
        } else {
            const int64_t n = (int64_t)(to - k0) - (threadIdx.x % 8) * 16;
#pragma unroll
            for (int k = 0; k < PIECES; ++k) held[k] = mq_read_part(src[k] + k0, n);
        }
    };
    auto place = [&](uint32_t buffer) {
#pragma unroll
        for (int k = 0; k < PIECES; ++k) *reinterpret_cast<mq_i4*>(&tile[buffer][dst + k * STEP * kMqDepth]) = held[k];
    };

    mq_i4 sum[TN][TM];
#pragma unroll
    for (int n = 0; n < TN; ++n) {
#pragma unroll
        for (int t = 0; t < TM; ++t) sum[n][t] = mq_i4{0, 0, 0, 0};
    }
    const uint32_t x_row = (wave % WM) * (TM * 16) + m, w_row = BM + (wave / WM) * (TN * 16) + m;
    // What LDS has is asked for ahead of the products that take it: the second half of a step's x in the first's registers as those are done with, and
    // the next step's first half behind the middle of the second, where the waves meet.
    mq_i4 a[2][TN], b[TM];
    auto read_w = [&](const char* rows, int half) {
#pragma unroll
        for (int n = 0; n < TN; ++n) a[half][n] = *reinterpret_cast<const mq_i4*>(rows + (w_row + n * 16) * kMqDepth + ((half * 4 + g) ^ (m & 7)) * 16);
    };
    auto read_x = [&](const char* rows, int half, int t) { b[t] = *reinterpret_cast<const mq_i4*>(rows + (x_row + t * 16) * kMqDepth + ((half * 4 + g) ^ (m & 7)) * 16); };
    auto multiply = [&](int half, int t) {
#pragma unroll
        for (int n = 0; n < TN; ++n) sum[n][t] = mq_mma(a[half][n], b[t], sum[n][t]);
    };
    if (from < to) {
        fetch(from);
        place(0);
        if (from + kMqDepth < to) fetch(from + kMqDepth);
    }
    __syncthreads();
    uint32_t buffer = 0;
    if (from < to) {
        read_w(tile[0], 0);
#pragma unroll
        for (int t = 0; t < TM; ++t) read_x(tile[0], 0, t);
    }
    for (uint64_t k0 = from; k0 < to; k0 += kMqDepth) {
        const bool more = k0 + kMqDepth < to;
        if (more) place(buffer ^ 1);
        if (k0 + 2 * kMqDepth < to) fetch(k0 + 2 * kMqDepth);
        const char* rows = tile[buffer];
        read_w(rows, 1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int t = 0; t < TM; ++t) {
            multiply(0, t);
            read_x(rows, 1, t);
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int t = 0; t < TM / 2; ++t) multiply(1, t);
        mq_meet();
        buffer ^= 1;
        rows = tile[buffer];
        if (more) {
            read_w(rows, 0);
#pragma unroll
            for (int t = 0; t < TM / 2; ++t) read_x(rows, 0, t);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int t = TM / 2; t < TM; ++t) {
            multiply(1, t);
            if (more) read_x(rows, 0, t);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    const uint64_t i_first = i0 + (wave % WM) * (TM * 16) + m, j_first = j0 + (wave / WM) * (TN * 16) + 4 * g;
    if (p.splits == 1) {
        double xs[TM];
#pragma unroll
        for (int t = 0; t < TM; ++t) xs[t] = (double)reinterpret_cast<const T*>(p.xscale)[i_first + t * 16 < p.rows ? i_first + t * 16 : p.rows - 1];
#pragma unroll
        for (int n = 0; n < TN; ++n) {
            const uint64_t j = j_first + n * 16;
            MqBeside<T> beside;
            beside.read(p, j);
#pragma unroll
            for (int t = 0; t < TM; ++t) {
                const uint64_t i = i_first + t * 16;
                if (i < p.rows && j < p.cols) mq_put<T, NT>(p.y + (int64_t)i * p.y_step, j, p.cols, p.bias != nullptr, xs[t], beside, sum[n][t]);
            }
        }
        return;
    }
#pragma unroll
    for (int t = 0; t < TM; ++t) {
        const uint64_t i = i_first + t * 16;
        if (i >= p.rows) continue;
#pragma unroll
        for (int n = 0; n < TN; ++n) {
            const uint64_t j = j_first + n * 16;
            int32_t* q = p.parts + ((uint64_t)part * p.rows + i) * p.cols + j;
            if (j + 4 <= p.cols) {
                __builtin_memcpy(q, &sum[n][t], 16);
            } else {
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (j + r < p.cols) q[r] = sum[n][t][r];
            }
        }
    }
}

template <class T>
__global__ __launch_bounds__(256) void matmul_q8_parts_kernel(MqParams p) {
    const uint64_t fours = (p.cols + 3) / 4, total = p.rows * fours;
    for (uint64_t at = (uint64_t)blockIdx.x * 256 + threadIdx.x; at < total; at += (uint64_t)gridDim.x * 256) {
        const uint64_t i = at / fours, j = (at - i * fours) * 4;
        mq_i4 sum = {0, 0, 0, 0};
        const int32_t* q = p.parts + i * p.cols + j;
        const uint64_t one = p.rows * p.cols;
        if (j + 4 <= p.cols) {
#pragma unroll 8
            for (uint32_t k = 0; k < p.splits; ++k) sum += mq_read(reinterpret_cast<const char*>(q + k * one));
        } else {
            for (uint32_t k = 0; k < p.splits; ++k) {
#pragma unroll
                for (int r = 0; r < 4; ++r) sum[r] += j + r < p.cols ? q[k * one + r] : 0;
            }
        }
        MqBeside<T> beside;
        beside.read(p, j);
        mq_put<T, false>(p.y + (int64_t)i * p.y_step, j, p.cols, p.bias != nullptr, (double)reinterpret_cast<const T*>(p.xscale)[i], beside, sum);
    }
}

template <class T, int BM, int BN, int WM, int WN>
int mq_tiles(const cumo_hip_matmul_q8_t& d, hipStream_t stream) {
    MqParams p;
    static_cast<cumo_hip_matmul_q8_t&>(p) = d;
    p.tiles_m = (uint32_t)((d.rows + BM - 1) / BM);
    p.tiles_n = (uint32_t)((d.cols + BN - 1) / BN);
    const uint64_t tiles = (uint64_t)p.tiles_m * p.tiles_n;
    // Inner is cut where tiles are few, into parts of 512 bytes or more, as many as leave a block to each of 256 compute units. 64, 128 and 256 rows by 4096
    // by 4096, 256 blocks 12.2, 14.8 and 17.2 us; 512 13.3, 14.7 and 18.7; 1024 13.3, 17.3 and 20.0.
    const uint64_t most = d.inner / 512, wanted = (uint64_t)device_compute_units() / tiles;
    p.splits = (uint32_t)(wanted < most ? wanted : most);
    if (p.splits < 1) p.splits = 1;
    p.per = ((d.inner + p.splits - 1) / p.splits + kMqDepth - 1) / kMqDepth * kMqDepth;
    if (p.per == 0) p.per = kMqDepth;
    char* scratch = nullptr;
    if (p.splits > 1 && !(scratch = cumo_cuda_runtime_malloc((uint64_t)p.splits * d.rows * d.cols * 4))) return CUMO_HIP_ERROR_OUT_OF_MEMORY;
    p.parts = reinterpret_cast<int32_t*>(scratch);
    const dim3 grid((unsigned)(tiles * p.splits)), block(64 * WM * WN);
    if (stream_past_caches(d.rows * d.cols * sizeof(T))) hipLaunchKernelGGL((matmul_q8_tiles_kernel<T, BM, BN, WM, WN, true>), grid, block, 0, stream, p);
    else hipLaunchKernelGGL((matmul_q8_tiles_kernel<T, BM, BN, WM, WN, false>), grid, block, 0, stream, p);
    if (scratch) {
        const uint64_t blocks = (d.rows * ((d.cols + 3) / 4) + 255) / 256;
        hipLaunchKernelGGL((matmul_q8_parts_kernel<T>), dim3((unsigned)(blocks < 65536 ? blocks : 65536)), dim3(256), 0, stream, p);
    }
    cumo_cuda_runtime_check_kernel_launch();
    if (scratch) scratch_free(scratch);
    return CUMO_HIP_OK;
}

template <class T, int TM>
int mq_rows(const cumo_hip_matmul_q8_t& d, hipStream_t stream) {
    constexpr int WAVES = 8;
    hipLaunchKernelGGL((matmul_q8_rows_kernel<T, TM, WAVES>), dim3((unsigned)((d.cols + 15) / 16)), dim3(64 * WAVES), 0, stream, d);
    cumo_cuda_runtime_check_kernel_launch();
    return CUMO_HIP_OK;
}

template <class T>
int mq_launch(const cumo_hip_matmul_q8_t& d, hipStream_t stream) {
    if (d.rows == 0 || d.cols == 0) return CUMO_HIP_OK;
    // (tiles are counted in 32 bits, and a launch holds fewer than 2^32 lanes)
    if (d.rows >= (uint64_t)1 << 31 || d.cols >= (uint64_t)1 << 31 || ((d.rows + 255) / 256) * ((d.cols + 255) / 256) >= (uint64_t)1 << 22) {
        report_error(CUMO_HIP_ERROR_ARGUMENT, 0, "matmul_q8: too many rows by columns");
        return CUMO_HIP_ERROR_ARGUMENT;
    }
    // Few rows: straight from memory, unless inner is so long, or columns so few, that parts of it are better shared out. us so / in tiles, cut:
    // 1 x 4096 by 256 5.4 / 8.0; 16 x 4096 by 2048 6.0 / 7.8; 16 x 16384 by 1024 16.2 / 10.5; 64 x 1024 by 512 5.6 / 7.8; 64 x 4096 by 1024 11.1 / 8.3.
    // (A block of 512 lanes to sixteen columns: as many columns as a launch's 2^32 lanes are enough for.)
    const bool reach = (d.inner <= 8192 || d.cols >= 4096) && d.cols <= (uint64_t)1 << 26;
    if (d.rows <= 16 && reach) return mq_rows<T, 1>(d, stream);
    if (d.rows <= 32 && reach) return mq_rows<T, 2>(d, stream);
    if (d.rows <= 64 && d.inner <= 1024 && reach) return mq_rows<T, 4>(d, stream);
    // A larger tile reads less for each product; smaller ones leave fewer units without a block, and have others beside them on theirs. The large one from
    // three blocks to four units on, the middle one from 25 to 32 on, where small ones would come to more than three a unit. On 256 units, us by the number
    // of the larger tiles, for inner of 512, 4096, 4095 and 16384:
    //   large / middle   160  28 / 26, 67 / 74, 90 / 103, 219 / 251     192  29 / 26, 69 / 77, 91 / 106, 223 / 277     256  27 / 25, 70 / 92, 89 / 124, 242 / 341
    //   middle / small   192  12.4 / 9.6, 35 / 27, 46 / 44, 112 / 92    200  12.4 / 10.6, 35 / 33, 46 / 56, 112 / 110    256  12.5 / 11.0, 35 / 35, 45 / 56, 114 / 126
    //                    384  18 / 16, 47 / 50, 68 / 81, 160 / 194      512  17 / 19, 50 / 65, 68 / 106, 184 / 253
    const uint64_t units = (uint64_t)device_compute_units(), large = ((d.rows + 255) / 256) * ((d.cols + 255) / 256);
    if (large * 4 >= units * 3) return mq_tiles<T, 256, 256, 2, 4>(d, stream);
    const uint64_t middle = ((d.rows + 127) / 128) * ((d.cols + 127) / 128);
    if (middle * 32 >= units * 25) return mq_tiles<T, 128, 128, 2, 2>(d, stream);
    return mq_tiles<T, 64, 64, 2, 2>(d, stream);
}

}  // namespace
}  // namespace cumo_hip

using namespace cumo_hip;

extern "C" int cumo_hip_matmul_q8_kernel_launch(int type, const cumo_hip_matmul_q8_t* d) {
    return type == 0 ? mq_launch<float>(*d, current_stream()) : mq_launch<double>(*d, current_stream());
}
