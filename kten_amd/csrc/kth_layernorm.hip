// Layer normalisation over the trailing dims of a tensor, seen as [rows, cols]: forward, and backward with the reduction
// of the weights' gradients. The reference has batch normalisation only; the operands, the optional ones and the float
// conventions follow BatchNormOperation (kten-api/.../tensor/operations/nn/BatchNormOperation.kt:5-41).
//
//   forward    m = sum x / n,  v = sum (x - m)^2 / n,  r = 1 / sqrt(v + eps),  y = (x - m) r gamma + beta
//   backward   xh = (x - m) r,  w = go gamma:   gin = r (w - mean(w) - xh mean(w xh)),
//              grad_gamma = sum over rows of go xh,  grad_beta = sum over rows of go
//
// Every sum is made in f64 from d = x - k with k the row's first element (0 if that is not finite): the sums of d and
// d^2 then give the mean and the variance in one pass, at a cancellation of at most n 2^-53 of the spread around k; the
// backward pass takes the sums of w and w d along and works the statistics out again, so that it needs nothing saved.
// Sums are folded in a fixed order: the same input gives the same bits.
#include "kth_internal.h"

#include <algorithm>

using namespace kth;

namespace {

constexpr int kBlock = 256;

typedef float v4f_any __attribute__((ext_vector_type(4), aligned(4)));     // 16 bytes at any dword address

__device__ __forceinline__ uint32_t divide(uint32_t n, FastDiv f) { return (__umulhi(n, f.mul) + n) >> f.shift; }

struct Shape2 {
    uint32_t rows, cols;
    double   inv_cols;
};

// What the apply kernels need of a row.
struct RowForward { double mean, rstd; };
struct RowBackward { double mean, rstd, w_mean, dot; };        // gin = rstd (w - w_mean - (x - mean) dot)

__device__ __forceinline__ double row_variance(double s1, double s2, double inv_n) {
    const double m = s1 * inv_n;
    const double v = s2 * inv_n - m * m;
    return v < 0.0 ? 0.0 : v;              // (a NaN stays one)
}

// 1 / sqrt(v + eps); a row without variance and without epsilon is all mean, and its result beta (JVMBatchNorm.kt:66-68)
__device__ __forceinline__ double row_rstd(double v, double eps) {
    const double s = v + eps;
    return s == 0.0 ? 0.0 : 1.0 / sqrt(s);
}

// (the product with rstd in f64: without epsilon it may be beyond fp32's range where a row's values are subnormal)
__device__ __forceinline__ float ln_forward(float x, double mean, double rstd, float gamma, float beta) {
    return static_cast<float>((static_cast<double>(x) - mean) * rstd) * gamma + beta;
}

// The value k that a row's sums are made around, from the row's first: around an infinity the sums would lose the mean. (Where
// lanes behind the last column have that infinity for their values, the row's sum has it already.)
__device__ __forceinline__ float around(float first) { return fabsf(first) < INFINITY ? first : 0.0f; }

// Sums of NS doubles over a workgroup of kBlock threads; every thread of wave 0 returns them.
template <int NS>
__device__ __forceinline__ void block_fold(double (&s)[NS], double* lds) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1)
#pragma unroll
        for (int i = 0; i < NS; i++) s[i] += __shfl_xor(s[i], off);
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    if (lane == 0)
#pragma unroll
        for (int i = 0; i < NS; i++) lds[wave * NS + i] = s[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NS; i++) {
        s[i] = lds[i];
        for (int w = 1; w < kBlock / 64; w++) s[i] += lds[w * NS + i];
    }
}

// ---------------------------------------------------------------- rows that stay in registers

// G lanes hold a row, U float4s each (column (u G + lane) 4 + e), so that a pass reads its operands once: a row is summed,
// its statistics are worked out by every lane, and the results are written from the registers. G = 4, 16 and 64 put
// several rows into a wave or one, larger G a row into two waves or more. Forward, a row that waves share has a workgroup to
// itself. Backward, a workgroup takes several rows at a time, because each leaves partial sums of the weights' gradients:
// with 512 threads instead of 256 [8192,768] takes 21.4 us instead of 22.8, [2000,700] 12.3 instead of 14.6, [4096,512] 13.9
// instead of 17.4; but two rows of 4096 columns, 256 lanes each, wait for each other ([16384,4096] 158 us instead of 153).
template <int G, int T>
struct RowGroup {
    static constexpr int threads = G > T ? G : T;              // of a workgroup
    static constexpr int groups = threads / G;                 // rows of a workgroup at a time
};
template <int G> using ForwardGroup = RowGroup<G, (G > 64 ? G : kBlock)>;
template <int G, int U> using BackwardGroup = RowGroup<G, (G == 256 && U == 4 ? 256 : 512)>;

// Lane sums of a double without LDS: both halves of the other lane's value by a register move (DPP inside 16 lanes, the
// row swaps of permlane across them), then an f64 addition. Every step adds the same two values in every lane that takes
// part, in either order, so all lanes end with the same bits.
template <int CTRL>
__device__ __forceinline__ double add_moved(double v) {
    const int lo = __builtin_amdgcn_update_dpp(0, __double2loint(v), CTRL, 0xf, 0xf, false);
    const int hi = __builtin_amdgcn_update_dpp(0, __double2hiint(v), CTRL, 0xf, 0xf, false);
    return v + __hiloint2double(hi, lo);
}
__device__ __forceinline__ double add_row16(double v) {        // rows of 16 lanes: 0 + 1, 2 + 3
    const auto lo = __builtin_amdgcn_permlane16_swap(__double2loint(v), __double2loint(v), false, false);
    const auto hi = __builtin_amdgcn_permlane16_swap(__double2hiint(v), __double2hiint(v), false, false);
    return __hiloint2double(hi[0], lo[0]) + __hiloint2double(hi[1], lo[1]);
}
__device__ __forceinline__ double add_half(double v) {         // the halves of the wave
    const auto lo = __builtin_amdgcn_permlane32_swap(__double2loint(v), __double2loint(v), false, false);
    const auto hi = __builtin_amdgcn_permlane32_swap(__double2hiint(v), __double2hiint(v), false, false);
    return __hiloint2double(hi[0], lo[0]) + __hiloint2double(hi[1], lo[1]);
}
// Over W neighbouring lanes (W = 2, 4, 8, 16: of values that repeat every W lanes of a row of 16 if W < 16; 4: of each quad).
template <int W>
__device__ __forceinline__ double lanes_sum(double v) {
    if constexpr (W == 4) { v = add_moved<0x4e>(v); v = add_moved<0xb1>(v); return v; }      // quad_perm [2,3,0,1], [1,0,3,2]
    if constexpr (W >= 16) v = add_moved<0x128>(v);                                          // row_ror 8, 4, 2, 1
    if constexpr (W >= 8) v = add_moved<0x124>(v);
    if constexpr (W >= 8) v = add_moved<0x122>(v);
    if constexpr (W >= 2) v = add_moved<0x121>(v);
    if constexpr (W >= 32) v = add_row16(v);
    if constexpr (W >= 64) v = add_half(v);
    return v;
}

// Sums of NS doubles over the G lanes of a row; every lane gets them, added in the same order. `lds` holds two sets of
// NS doubles a wave: sets alternate from row to row, so one barrier a row is enough.
template <int G, int THREADS, int NS>
__device__ __forceinline__ void row_fold(double (&s)[NS], double* lds, uint32_t& set) {
#pragma unroll
    for (int i = 0; i < NS; i++) s[i] = lanes_sum<(G > 64 ? 64 : G)>(s[i]);
    if constexpr (G > 64) {
        constexpr int waves = G / 64;
        double* mine = lds + (set * (THREADS / G) + threadIdx.x / G) * NS * waves;
        set ^= 1;
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int i = 0; i < NS; i++) mine[i * waves + (threadIdx.x % G >> 6)] = s[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NS; i++) s[i] = lanes_sum<waves>(mine[i * waves + threadIdx.x % waves]);
    }
}

// 1 / sqrt(v + eps) in f64: the hardware's estimate (24 bits) and one Newton step.
__device__ __forceinline__ double row_rstd_fast(double v, double eps) {
    const double s = v + eps;
    if (s == 0.0 || s == INFINITY) return 0.0;         // (an infinite epsilon: the step would make NaN of it)
    const double y = __builtin_amdgcn_rsq(s);
    return fma(0.5 * y, fma(-s * y, y, 1.0), y);
}

// Few columns' f64 values at a time, where a lane holds many columns: the compiler would work on all of them at once.
#define KTH_FEW_AT_A_TIME(e) do { if ((e) % 2 == 1) __builtin_amdgcn_sched_barrier(0); } while (0)

// Four values from column c on; `fill` behind the last column.
template <bool ONCE>
__device__ __forceinline__ void load4(const float* p, uint32_t c, uint32_t cols, float fill, float (&v)[4]) {
    if (c + 4 <= cols) {
        const v4f_any* q = reinterpret_cast<const v4f_any*>(p + c);
        const v4f_any t = ONCE ? __builtin_nontemporal_load(q) : *q;
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = t[e];
    } else {
#pragma unroll
        for (uint32_t e = 0; e < 4; e++) v[e] = c + e < cols ? p[c + e] : fill;
    }
}
__device__ __forceinline__ void store4(float* p, uint32_t c, uint32_t cols, const float (&v)[4]) {
    if (c + 4 <= cols) {
        *reinterpret_cast<v4f_any*>(p + c) = v4f_any{v[0], v[1], v[2], v[3]};
    } else {
#pragma unroll
        for (uint32_t e = 0; e < 4; e++) if (c + e < cols) p[c + e] = v[e];
    }
}

// Bound by memory: [16384,4096] 94.7 us, 5.7 TB/s; [8191,1021] 13.8 us, 4.9 TB/s, a round of workgroups and its start and end.
template <int G, int U>
__global__ __launch_bounds__(ForwardGroup<G>::threads) void ln_forward_rows_kernel(const float* x, const float* __restrict__ gamma, const float* __restrict__ beta,
                                                                               float* out, float* __restrict__ out_mean, float* __restrict__ out_std,
                                                                               Shape2 sh, double eps) {
    __shared__ double lds[G > 64 ? 2 * 2 * G / 64 : 1];
    const uint32_t lane = threadIdx.x % G;
    uint32_t set = 0;
    float ga[U][4], be[U][4];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const uint32_t c = (u * G + lane) * 4;
#pragma unroll
        for (int e = 0; e < 4; e++) { ga[u][e] = 1.0f; be[u][e] = 0.0f; }
        if (gamma) load4<false>(gamma, c, sh.cols, 1.0f, ga[u]);
        if (beta) load4<false>(beta, c, sh.cols, 0.0f, be[u]);
    }
    for (uint32_t row = blockIdx.x * ForwardGroup<G>::groups + threadIdx.x / G; row < sh.rows; row += gridDim.x * ForwardGroup<G>::groups) {
        const uint64_t at = static_cast<uint64_t>(row) * sh.cols;
        const float first = x[at];
        float v[U][4];
#pragma unroll
        for (int u = 0; u < U; u++) load4<false>(x + at, (u * G + lane) * 4, sh.cols, first, v[u]);
        const double k = static_cast<double>(around(first));
        double s[2] = {};
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const double d = static_cast<double>(v[u][e]) - k;
                s[0] += d; s[1] = fma(d, d, s[1]);
            }
        row_fold<G, ForwardGroup<G>::threads, 2>(s, lds, set);
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int e = 0; e < 4; e++) forget(v[u][e]);
        const double mean = k + s[0] * sh.inv_cols;
        const double rstd = row_rstd_fast(row_variance(s[0], s[1], sh.inv_cols), eps);
#pragma unroll
        for (int u = 0; u < U; u++) {
            float r[4];
#pragma unroll
            for (int e = 0; e < 4; e++) r[e] = ln_forward(v[u][e], mean, rstd, ga[u][e], be[u][e]);
            store4(out + at, (u * G + lane) * 4, sh.cols, r);
        }
        if (lane == 0) {
            if (out_mean) out_mean[row] = static_cast<float>(mean);
            if (out_std) out_std[row] = static_cast<float>(rstd);
        }
    }
}

// The input gradient of each row, and down the workgroup's rows the weights' gradients, in f64 registers; a workgroup
// leaves one row [2, cols] of partial sums as floats, each rounded once (2^-24 of itself), which ln_fold_kernel adds in f64;
// one that is alone (no `partial`) writes the weights' gradients themselves. Bound by memory where there are rows enough:
// [16384,4096] 147.6 us with the fold, 5.5 TB/s; [8192,768] 20.6 us, of which the fold's launch takes 4.
template <int G, int U>
__global__ __launch_bounds__((BackwardGroup<G, U>::threads)) void ln_backward_rows_kernel(const float* __restrict__ x, const float* go, const float* __restrict__ gamma, float* grad_in,
                                                                                float* __restrict__ partial, float* __restrict__ grad_gamma, float* __restrict__ grad_beta,
                                                                                Shape2 sh, double eps) {
    constexpr int threads = BackwardGroup<G, U>::threads, groups = BackwardGroup<G, U>::groups;
    __shared__ double lds[groups > 1 ? threads * 4 : 2 * 4 * threads / 64];    // (rows' sums, then the columns' sums)
    const uint32_t lane = threadIdx.x % G;
    uint32_t set = 0;
    float ga[U][4];
    double sg[U][4], sb[U][4];
#pragma unroll
    for (int u = 0; u < U; u++) {
#pragma unroll
        for (int e = 0; e < 4; e++) { ga[u][e] = 1.0f; sg[u][e] = 0.0; sb[u][e] = 0.0; }
        if (gamma) load4<false>(gamma, (u * G + lane) * 4, sh.cols, 1.0f, ga[u]);
    }
    // (rows that several waves share meet at barriers: a workgroup's last rows may be none, which read the last one again)
    constexpr bool meet = G > 64 && groups > 1;
    for (uint32_t row0 = blockIdx.x * groups + (meet ? 0 : threadIdx.x / G); row0 < sh.rows; row0 += gridDim.x * groups) {
        const uint32_t row = meet ? min(row0 + threadIdx.x / G, sh.rows - 1) : row0;
        const bool none = meet && row0 + threadIdx.x / G >= sh.rows;
        const uint64_t at = static_cast<uint64_t>(row) * sh.cols;
        const float first = x[at];
        float v[U][4], g[U][4];
#pragma unroll
        for (int u = 0; u < U; u++) {
            load4<false>(x + at, (u * G + lane) * 4, sh.cols, first, v[u]);
            load4<true>(go + at, (u * G + lane) * 4, sh.cols, 0.0f, g[u]);
        }
        const double k = static_cast<double>(first);
        double s[4] = {};
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const double d = static_cast<double>(v[u][e]) - k;
                const double w = static_cast<double>(g[u][e]) * static_cast<double>(ga[u][e]);
                s[0] += d; s[1] = fma(d, d, s[1]); s[2] += w; s[3] = fma(w, d, s[3]);
                KTH_FEW_AT_A_TIME(e);
            }
        row_fold<G, threads, 4>(s, lds, set);
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int e = 0; e < 4; e++) { forget(v[u][e]); forget(g[u][e]); forget(ga[u][e]); }
        const double inv = sh.inv_cols, delta = s[0] * inv, mean = k + delta;
        const double rstd = row_rstd_fast(row_variance(s[0], s[1], inv), eps);
        const double w_mean = s[2] * inv, dot = (s[3] - delta * s[2]) * rstd * rstd * inv;
        if (none) break;
#pragma unroll
        for (int u = 0; u < U; u++) {
            float r[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const double d = static_cast<double>(v[u][e]) - mean, gd = static_cast<double>(g[u][e]);
                const double w = gd * static_cast<double>(ga[u][e]);
                r[e] = static_cast<float>((w - w_mean - d * dot) * rstd);
                sg[u][e] = fma(gd, d * rstd, sg[u][e]);
                sb[u][e] += gd;
                KTH_FEW_AT_A_TIME(e);
            }
            if (grad_in) store4(grad_in + at, (u * G + lane) * 4, sh.cols, r);
        }
    }
    if (!partial && !grad_gamma && !grad_beta) return;
    float* mine = partial + static_cast<uint64_t>(blockIdx.x) * 2 * sh.cols;
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
        for (int which = 0; which < 2; which++) {
            double (&t)[4] = which == 0 ? sg[u] : sb[u];
            float* to = partial ? mine + which * sh.cols : which == 0 ? grad_gamma : grad_beta;
            if constexpr (groups > 1) {                        // the workgroup's rows side by side, its threads on the columns
                __syncthreads();
#pragma unroll
                for (int e = 0; e < 4; e++) lds[e * threads + threadIdx.x] = t[e];
                __syncthreads();
                for (uint32_t e = threadIdx.x / G; e < 4; e += groups) {
                    const uint32_t c = (u * G + lane) * 4 + e;
                    if (!to || c >= sh.cols) continue;
                    double sum = lds[e * threads + lane];
                    for (int r = 1; r < groups; r++) sum += lds[e * threads + r * G + lane];
                    to[c] = static_cast<float>(sum);
                }
            } else {
                float f[4];
#pragma unroll
                for (int e = 0; e < 4; e++) f[e] = static_cast<float>(t[e]);
                if (to) store4(to, (u * G + lane) * 4, sh.cols, f);
            }
        }
}

// ---------------------------------------------------------------- longer rows, in LDS and registers

// A workgroup of 1024 threads holds a row: R float4s a lane in registers, the columns after them in LDS, where a lane reads
// back only what it wrote (the barrier of the row's sums is the only one). The weights are read again for every row, from
// the cache. [1000,30000] 64 us, 3.7 TB/s: a compute unit has one row at a time, and reads nothing while it writes.
constexpr uint32_t kLongThreads = 1024, kLdsRowFloats = 36864;
template <int R>
__global__ __launch_bounds__(kLongThreads) void ln_forward_long_kernel(const float* x, const float* __restrict__ gamma, const float* __restrict__ beta, float* out,
                                                                       float* __restrict__ out_mean, float* __restrict__ out_std, Shape2 sh, double eps) {
    extern __shared__ float4 held[];
    __shared__ double lds[2 * 2 * kLongThreads / 64];
    constexpr uint32_t after = R * kLongThreads * 4;         // the first column that lies in LDS
    constexpr uint32_t kInFlight = 4;
    const uint32_t many = (sh.cols - after + 3) / 4;         // float4s in LDS
    uint32_t set = 0;
    for (uint32_t row = blockIdx.x; row < sh.rows; row += gridDim.x) {
        const uint64_t at = static_cast<uint64_t>(row) * sh.cols;
        const float first = x[at];
        const double k = static_cast<double>(around(first));
        double s[2] = {};
        v4f_any v[R > 0 ? R : 1];                            // (columns that every such row has)
#pragma unroll
        for (int u = 0; u < R; u++) v[u] = *reinterpret_cast<const v4f_any*>(x + at + (u * kLongThreads + threadIdx.x) * 4);
        for (uint32_t i0 = threadIdx.x; i0 < many; i0 += kInFlight * kLongThreads) {
            float t[kInFlight][4];
#pragma unroll
            for (uint32_t j = 0; j < kInFlight; j++) {
                const uint32_t i = i0 + j * kLongThreads;
                if (i < many) load4<false>(x + at, after + i * 4, sh.cols, first, t[j]);
            }
#pragma unroll
            for (uint32_t j = 0; j < kInFlight; j++) {
                const uint32_t i = i0 + j * kLongThreads;
                if (i < many) {
                    held[i] = float4{t[j][0], t[j][1], t[j][2], t[j][3]};
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const double d = static_cast<double>(t[j][e]) - k;
                        s[0] += d; s[1] = fma(d, d, s[1]);
                    }
                }
            }
        }
#pragma unroll
        for (int u = 0; u < R; u++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const double d = static_cast<double>(v[u][e]) - k;
                s[0] += d; s[1] = fma(d, d, s[1]);
                KTH_FEW_AT_A_TIME(e);
            }
        row_fold<kLongThreads, kLongThreads, 2>(s, lds, set);
#pragma unroll
        for (int u = 0; u < R; u++)
#pragma unroll
            for (int e = 0; e < 4; e++) { float keep = v[u][e]; forget(keep); v[u][e] = keep; }
        const double mean = k + s[0] * sh.inv_cols;
        const double rstd = row_rstd_fast(row_variance(s[0], s[1], sh.inv_cols), eps);
        auto apply = [&](const float (&t)[4], uint32_t c) {
            float ga[4] = {1.0f, 1.0f, 1.0f, 1.0f}, be[4] = {}, y[4];
            if (gamma) load4<false>(gamma, c, sh.cols, 1.0f, ga);
            if (beta) load4<false>(beta, c, sh.cols, 0.0f, be);
#pragma unroll
            for (int e = 0; e < 4; e++) y[e] = ln_forward(t[e], mean, rstd, ga[e], be[e]);
            store4(out + at, c, sh.cols, y);
        };
#pragma unroll
        for (int u = 0; u < R; u++) {
            const uint32_t c = (u * kLongThreads + threadIdx.x) * 4;
            v4f_any ga{1.0f, 1.0f, 1.0f, 1.0f}, be{}, y;
            if (gamma) ga = *reinterpret_cast<const v4f_any*>(gamma + c);
            if (beta) be = *reinterpret_cast<const v4f_any*>(beta + c);
#pragma unroll
            for (int e = 0; e < 4; e++) y[e] = ln_forward(v[u][e], mean, rstd, ga[e], be[e]);
            *reinterpret_cast<v4f_any*>(out + at + c) = y;
            if (u % 2 == 1) __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll 2
        for (uint32_t i = threadIdx.x; i < many; i += kLongThreads) {
            const float4 h = held[i];
            const float t[4] = {h.x, h.y, h.z, h.w};
            apply(t, after + i * 4);
        }
        if (threadIdx.x == 0) {
            if (out_mean) out_mean[row] = static_cast<float>(mean);
            if (out_std) out_std[row] = static_cast<float>(rstd);
        }
    }
}

// ---------------------------------------------------------------- the same in segments

struct SegPlan {
    Shape2   sh;
    uint32_t segments, seg_len;      // segments per row, columns per segment (a multiple of 4)
    uint32_t blocks;                 // rows x segments: below 2^19, for the rows are longer than 8192
    FastDiv  seg_div;
};

// Workgroup b sums segment b % segments of row b / segments: forward d, d^2; backward also w, w d.
template <bool BACKWARD>
__global__ __launch_bounds__(kBlock) void ln_sums_kernel(const float* __restrict__ x, const float* __restrict__ go,
                                                         const float* __restrict__ gamma, double* __restrict__ partial, SegPlan pl) {
    constexpr int NS = BACKWARD ? 4 : 2;
    __shared__ double lds[NS * kBlock / 64];
    const uint32_t b = blockIdx.x;
    const uint32_t row = divide(b, pl.seg_div);
    const uint32_t seg = b - row * pl.segments;
    const float* xr = x + static_cast<uint64_t>(row) * pl.sh.cols;
    const float* gr = BACKWARD ? go + static_cast<uint64_t>(row) * pl.sh.cols : nullptr;
    const uint32_t first = seg * pl.seg_len;
    const uint32_t last = min(first + pl.seg_len, pl.sh.cols);
    const double k = static_cast<double>(around(xr[0]));
    double s[NS] = {};
    auto add = [&](float xv, float gv, float ga) {
        const double d = static_cast<double>(xv) - k;
        s[0] += d; s[1] += d * d;
        if (BACKWARD) {
            const double w = static_cast<double>(gv) * static_cast<double>(ga);
            s[NS - 2] += w; s[NS - 1] += w * d;
        }
    };
    for (uint32_t c = first + threadIdx.x * 4; c < last; c += kBlock * 4) {
        if (c + 4 <= last) {
            const v4f_any vx = *reinterpret_cast<const v4f_any*>(xr + c);
            v4f_any vg{}, va{1.0f, 1.0f, 1.0f, 1.0f};
            if (BACKWARD) {
                vg = *reinterpret_cast<const v4f_any*>(gr + c);
                if (gamma) va = *reinterpret_cast<const v4f_any*>(gamma + c);
            }
#pragma unroll
            for (int e = 0; e < 4; e++) add(vx[e], vg[e], va[e]);
        } else {
            for (uint32_t e = c; e < last; e++) add(xr[e], BACKWARD ? gr[e] : 0.0f, BACKWARD && gamma ? gamma[e] : 1.0f);
        }
    }
    block_fold<NS>(s, lds);
    if (threadIdx.x == 0)
#pragma unroll
        for (int i = 0; i < NS; i++) partial[static_cast<uint64_t>(b) * NS + i] = s[i];
}

// The statistics of the backward pass where a workgroup sums a whole row: in segments / whole, us for the pass: [1,10000] 9.0 /
// 7.2, [100,10000] 21.8 / 19.0, [500,9000] 29.4 / 25.9, [2000,10000] 91 / 86, [1000,65536] 277 / 269; but [64,65536] 27 / 29 and
// [8,1000000] 66 / 239, a few long rows, which leave most of the chip idle.
__global__ __launch_bounds__(kLongThreads) void ln_row_sums_kernel(const float* __restrict__ x, const float* __restrict__ go, const float* __restrict__ gamma,
                                                                   RowBackward* __restrict__ rows, Shape2 sh, double eps) {
    __shared__ double lds[2 * 4 * kLongThreads / 64];
    const uint64_t at = static_cast<uint64_t>(blockIdx.x) * sh.cols;
    const float first = x[at];
    const double k = static_cast<double>(first);
    double s[4] = {};
    for (uint32_t c = threadIdx.x * 4; c < sh.cols; c += kLongThreads * 4) {
        float v[4], g[4], ga[4] = {1.0f, 1.0f, 1.0f, 1.0f};
        load4<false>(x + at, c, sh.cols, first, v);                    // (behind the last column terms of zero)
        load4<false>(go + at, c, sh.cols, 0.0f, g);
        if (gamma) load4<false>(gamma, c, sh.cols, 1.0f, ga);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const double d = static_cast<double>(v[e]) - k;
            const double w = static_cast<double>(g[e]) * static_cast<double>(ga[e]);
            s[0] += d; s[1] = fma(d, d, s[1]); s[2] += w; s[3] = fma(w, d, s[3]);
        }
    }
    uint32_t set = 0;
    row_fold<kLongThreads, kLongThreads, 4>(s, lds, set);
    if (threadIdx.x != 0) return;
    const double inv = sh.inv_cols, delta = s[0] * inv;
    const double rstd = row_rstd_fast(row_variance(s[0], s[1], inv), eps);
    rows[blockIdx.x] = RowBackward{k + delta, rstd, s[2] * inv, (s[3] - delta * s[2]) * rstd * rstd * inv};
}

// One wave per row folds its segments (lane l takes l, l + 64, ...; then the lanes by xor-shuffles).
template <bool BACKWARD>
__global__ __launch_bounds__(kBlock) void ln_rows_kernel(const float* __restrict__ x, const double* __restrict__ partial, SegPlan pl, double eps,
                                                         RowForward* __restrict__ fwd, RowBackward* __restrict__ bwd,
                                                         float* __restrict__ out_mean, float* __restrict__ out_std) {
    constexpr int NS = BACKWARD ? 4 : 2;
    const uint32_t row = blockIdx.x * (kBlock / 64) + (threadIdx.x >> 6);
    if (row >= pl.sh.rows) return;
    double s[NS] = {};
    for (uint32_t t = threadIdx.x & 63; t < pl.segments; t += 64)
#pragma unroll
        for (int i = 0; i < NS; i++) s[i] += partial[(static_cast<uint64_t>(row) * pl.segments + t) * NS + i];
#pragma unroll
    for (int off = 32; off > 0; off >>= 1)
#pragma unroll
        for (int i = 0; i < NS; i++) s[i] += __shfl_xor(s[i], off);
    if ((threadIdx.x & 63) != 0) return;
    const double inv = pl.sh.inv_cols;
    const double delta = s[0] * inv;
    const double mean = static_cast<double>(around(x[static_cast<uint64_t>(row) * pl.sh.cols])) + delta;
    const double rstd = row_rstd(row_variance(s[0], s[1], inv), eps);
    if (BACKWARD) {
        bwd[row] = RowBackward{mean, rstd, s[NS - 2] * inv, (s[NS - 1] - delta * s[NS - 2]) * rstd * rstd * inv};
    } else {
        fwd[row] = RowForward{mean, rstd};
        if (out_mean) out_mean[row] = static_cast<float>(mean);
        if (out_std) out_std[row] = static_cast<float>(rstd);
    }
}

__global__ __launch_bounds__(kBlock) void ln_apply_kernel(const float* x, const float* __restrict__ gamma, const float* __restrict__ beta, float* out,
                                                          const RowForward* __restrict__ fwd, SegPlan pl) {
    const uint32_t row = divide(blockIdx.x, pl.seg_div);
    const uint32_t seg = blockIdx.x - row * pl.segments;
    const uint64_t at = static_cast<uint64_t>(row) * pl.sh.cols;
    const uint32_t first = seg * pl.seg_len;
    const uint32_t last = min(first + pl.seg_len, pl.sh.cols);
    const double mean = fwd[row].mean;
    const double rstd = fwd[row].rstd;
    for (uint32_t c = first + threadIdx.x * 4; c < last; c += kBlock * 4) {
        if (c + 4 <= last) {
            const v4f_any vx = *reinterpret_cast<const v4f_any*>(x + at + c);
            v4f_any va{1.0f, 1.0f, 1.0f, 1.0f}, vb{}, r;
            if (gamma) va = *reinterpret_cast<const v4f_any*>(gamma + c);
            if (beta) vb = *reinterpret_cast<const v4f_any*>(beta + c);
#pragma unroll
            for (int e = 0; e < 4; e++) r[e] = ln_forward(vx[e], mean, rstd, va[e], vb[e]);
            *reinterpret_cast<v4f_any*>(out + at + c) = r;
        } else {
            for (uint32_t e = c; e < last; e++) out[at + e] = ln_forward(x[at + e], mean, rstd, gamma ? gamma[e] : 1.0f, beta ? beta[e] : 0.0f);
        }
    }
}

// ---------------------------------------------------------------- backward by columns

struct ColPlan {
    Shape2   sh;
    uint32_t col_blocks, ranges, rows_per_range;
    FastDiv  col_div;
};

// ([2000,10000] 41 us, 5.8 TB/s.) A thread owns four columns of one range of rows: it writes the input gradient of each row and sums the weights'
// gradients down the range. The partials are floats: each is a f64 sum rounded once (2^-24 of itself), folded in f64.
__global__ __launch_bounds__(kBlock) void ln_cols_kernel(const float* __restrict__ x, const float* go, const float* __restrict__ gamma, float* grad_in,
                                                         const RowBackward* __restrict__ rows, float* __restrict__ partial, float* __restrict__ grad_gamma,
                                                         float* __restrict__ grad_beta, ColPlan pl) {
    const uint32_t range = divide(blockIdx.x, pl.col_div);
    const uint32_t c = ((blockIdx.x - range * pl.col_blocks) * kBlock + threadIdx.x) * 4;
    if (c >= pl.sh.cols) return;
    const uint32_t width = min(4u, pl.sh.cols - c);
    const uint32_t last = min((range + 1) * pl.rows_per_range, pl.sh.rows);
    float ga[4];
#pragma unroll
    for (uint32_t e = 0; e < 4; e++) ga[e] = gamma && e < width ? gamma[c + e] : 1.0f;
    double sg[4] = {}, sb[4] = {};
    for (uint32_t row = range * pl.rows_per_range; row < last; row++) {
        const uint64_t at = static_cast<uint64_t>(row) * pl.sh.cols + c;
        const RowBackward p = rows[row];
        float vx[4] = {}, vg[4] = {}, r[4];
        if (width == 4) {
            const v4f_any tx = *reinterpret_cast<const v4f_any*>(x + at), tg = *reinterpret_cast<const v4f_any*>(go + at);
#pragma unroll
            for (int e = 0; e < 4; e++) { vx[e] = tx[e]; vg[e] = tg[e]; }
        } else {
#pragma unroll
            for (uint32_t e = 0; e < 4; e++) if (e < width) { vx[e] = x[at + e]; vg[e] = go[at + e]; }
        }
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const double d = static_cast<double>(vx[e]) - p.mean, g = static_cast<double>(vg[e]);
            r[e] = static_cast<float>((g * static_cast<double>(ga[e]) - p.w_mean - d * p.dot) * p.rstd);
            sg[e] += g * (d * p.rstd);
            sb[e] += g;
        }
        if (grad_in) {
            if (width == 4) *reinterpret_cast<v4f_any*>(grad_in + at) = v4f_any{r[0], r[1], r[2], r[3]};
            else
#pragma unroll
                for (uint32_t e = 0; e < 4; e++) if (e < width) grad_in[at + e] = r[e];
        }
    }
    float* to_gamma = partial ? partial + static_cast<uint64_t>(range) * 2 * pl.sh.cols : grad_gamma;
    float* to_beta = partial ? to_gamma + pl.sh.cols : grad_beta;
    for (uint32_t e = 0; e < width; e++) {
        if (to_gamma) to_gamma[c + e] = static_cast<float>(sg[e]);
        if (to_beta) to_beta[c + e] = static_cast<float>(sb[e]);
    }
}

// grad_gamma and grad_beta from `ranges` partial rows of [2, cols]: a column has kFoldLanes lanes, each with every
// kFoldLanes-th range, eight of them asked for before the first is added; then a tree over the lanes. Which of the two
// sums: blockIdx.y. 64 lanes (16 columns a workgroup), or 4 where there are at most 16 ranges (1024 ranges of 768 columns
// take 7 us with 64 lanes a column, 36 with 8).
constexpr uint32_t kMaxFoldGrid = 1u << 18;
constexpr uint32_t kFoldBlock = 1024;
template <uint32_t kFoldLanes>
__global__ __launch_bounds__(kFoldBlock) void ln_fold_kernel(const float* __restrict__ partial, uint32_t cols, uint32_t ranges,
                                                             float* __restrict__ grad_gamma, float* __restrict__ grad_beta) {
    constexpr uint32_t kFoldCols = kFoldBlock / kFoldLanes;
    __shared__ double lds[kFoldBlock];
    float* out = blockIdx.y == 0 ? grad_gamma : grad_beta;
    if (!out) return;
    const uint32_t lane = threadIdx.x / kFoldCols;
    for (uint32_t c0 = blockIdx.x * kFoldCols; c0 < cols; c0 += gridDim.x * kFoldCols) {
        const uint32_t c = c0 + threadIdx.x % kFoldCols;
        double s = 0.0;
        constexpr uint32_t kAhead = 8;
        for (uint32_t r0 = lane; c < cols && r0 < ranges; r0 += kFoldLanes * kAhead) {
            float v[kAhead];
#pragma unroll
            for (uint32_t k = 0; k < kAhead; k++) {
                const uint32_t r = r0 + k * kFoldLanes;
                v[k] = r < ranges ? partial[(static_cast<uint64_t>(r) * 2 + blockIdx.y) * cols + c] : 0.0f;
            }
#pragma unroll
            for (uint32_t k = 0; k < kAhead; k++) s += static_cast<double>(v[k]);
        }
        lds[threadIdx.x] = s;
        __syncthreads();
#pragma unroll
        for (uint32_t step = kFoldLanes / 2; step > 0; step >>= 1) {
            if (lane < step) lds[threadIdx.x] += lds[threadIdx.x + step * kFoldCols];
            __syncthreads();
        }
        if (lane == 0 && c < cols) out[c] = static_cast<float>(lds[threadIdx.x]);
        __syncthreads();
    }
}

// ---------------------------------------------------------------- host side

int shape_of(const char* what, const int32_t* shape, int dims, int axis, Shape2* sh, uint64_t* n) {
    if (dims < 1 || dims > KTH_MAX_DIMS) return fail(KTH_E_ARGUMENT, "%s: %d dims", what, dims);
    if (!shape) return fail(KTH_E_ARGUMENT, "%s: null shape", what);
    if (axis < 0 || axis >= dims) return fail(KTH_E_ARGUMENT, "%s: axis %d of %d dims", what, axis, dims);
    uint64_t rows = 1, cols = 1;
    for (int d = 0; d < dims; d++) {
        if (shape[d] < 1) return fail(KTH_E_ARGUMENT, "%s: dim %d is %d", what, d, shape[d]);
        (d < axis ? rows : cols) *= static_cast<uint64_t>(shape[d]);
        if (rows * cols > kMaxElements) return fail(KTH_E_ARGUMENT, "%s: more than 2^31-1 elements", what);
    }
    sh->rows = static_cast<uint32_t>(rows);
    sh->cols = static_cast<uint32_t>(cols);
    sh->inv_cols = 1.0 / static_cast<double>(cols);
    *n = rows * cols;
    return KTH_OK;
}

uint32_t device_units() { return static_cast<uint32_t>(state().compute_units > 0 ? state().compute_units : 256); }

SegPlan plan_segments(const Shape2& sh) {
    SegPlan pl{};
    pl.sh = sh;
    // enough workgroups for the chip, segments of at least 4096 columns
    uint32_t segments = (device_units() * 8 + sh.rows - 1) / sh.rows;
    segments = std::min(segments, (sh.cols + 4095) / 4096);
    if (segments < 1) segments = 1;
    pl.seg_len = ((sh.cols + segments - 1) / segments + 3) / 4 * 4;
    pl.segments = (sh.cols + pl.seg_len - 1) / pl.seg_len;
    pl.seg_div = make_div(pl.segments);
    pl.blocks = sh.rows * pl.segments;
    return pl;
}

// The widest rows that stay in registers. (With 8 float4s a lane the forward kernel spills.)
constexpr uint32_t kForwardRowCols = 16384, kBackwardRowCols = 8192;

// Rows that ln_forward_long_kernel takes: those that LDS holds, and longer ones where there are rows enough (segments / a
// workgroup a row, us: [1,20000] 8.9 / 5.7, [64,36000] 11.9 / 11.1, [1000,30000] 81 / 64; [32,65536] 10.9 / 15.8, [100,65536] 18.5 / 18.0,
// [1000,65536] 188 / 123).
constexpr int kLongRegisters = 7;
// Rows that ln_row_sums_kernel takes: up to so many columns, or longer ones where every compute unit has two.
constexpr uint32_t kWholeRowCols = 32768;
constexpr uint32_t kLongRowCols = kLdsRowFloats + kLongRegisters * kLongThreads * 4, kLongRows = 96;

uint32_t grid_for(const Shape2& sh, uint32_t groups, uint32_t per_unit) {
    return std::min((sh.rows - 1) / groups + 1, device_units() * per_unit);       // (fewer than 2^32 threads in all)
}

// A kernel for the rows' width and its grid. Rows of 65 to 2048 columns: a workgroup for each few rows (kOneShot; with
// workgroups that stride over the rows [65536,1024] takes 98 us instead of 95, [262144,128] 52 instead of 48); shorter and
// longer ones: so many workgroups a compute unit that stride over the rows and keep the weights ([1000000,33] 82 us instead
// of 114; [16384,4096] 96 us with 2, 100 with 5, 105 with a workgroup each).
constexpr uint32_t kOneShot = 1u << 12;
struct ForwardRows {
    void (*kernel)(const float*, const float*, const float*, float*, float*, float*, Shape2, double);
    uint32_t threads, grid;
};
template <int G, int U>
ForwardRows forward_rows_of(const Shape2& sh, uint32_t per_unit) {
    return ForwardRows{ln_forward_rows_kernel<G, U>, ForwardGroup<G>::threads, grid_for(sh, ForwardGroup<G>::groups, per_unit)};
}
ForwardRows forward_rows_kernel(const Shape2& sh) {
    const uint32_t c = sh.cols;
    return c <= 16 ? forward_rows_of<4, 1>(sh, 8) : c <= 64 ? forward_rows_of<16, 1>(sh, 8) : c <= 128 ? forward_rows_of<16, 2>(sh, kOneShot)
         : c <= 256 ? forward_rows_of<64, 1>(sh, kOneShot) : c <= 512 ? forward_rows_of<64, 2>(sh, kOneShot)
         : c <= 768 ? forward_rows_of<64, 3>(sh, kOneShot) : c <= 1024 ? forward_rows_of<64, 4>(sh, kOneShot)
         : c <= 2048 ? forward_rows_of<128, 4>(sh, kOneShot) : c <= 4096 ? forward_rows_of<256, 4>(sh, 2)
         : c <= 8192 ? forward_rows_of<512, 4>(sh, 2) : forward_rows_of<1024, 4>(sh, 1);
}

struct BackwardRows {
    void (*kernel)(const float*, const float*, const float*, float*, float*, float*, float*, Shape2, double);
    uint32_t threads, grid;
};
// Two rows a group or fewer are left to one workgroup, which needs no second launch: [64,64] 4.1 us against 5.9, [16,256] 4.3
// against 6.4; with four rows a group ([100,100] 7.9 against 7.6, [30,512] 8.2 against 7.0) it is as slow or slower.
template <int G, int U>
BackwardRows backward_rows_of(const Shape2& sh, uint32_t per_unit) {
    constexpr uint32_t groups = BackwardGroup<G, U>::groups;
    const bool alone = groups > 1 && sh.rows <= 2 * groups;
    return BackwardRows{ln_backward_rows_kernel<G, U>, BackwardGroup<G, U>::threads, alone ? 1 : grid_for(sh, groups, per_unit)};
}
BackwardRows backward_rows_kernel(const Shape2& sh) {
    const uint32_t c = sh.cols;
    // Four float4s a lane are the fastest where there are rows enough for the chip ([65536,1024] 150 us against 217 with
    // one, [1000,1024] 11.0 against 13.6); fewer rows are spread over four waves each ([500,1024] 9.3 us against 10.0,
    // [100,1024] 7.4 against 9.7).
    if (c > 512 && c <= 1024 && sh.rows <= 2 * device_units()) return backward_rows_of<256, 1>(sh, 2);
    return c <= 16 ? backward_rows_of<4, 1>(sh, 3) : c <= 64 ? backward_rows_of<16, 1>(sh, 3) : c <= 128 ? backward_rows_of<16, 2>(sh, 2)
         : c <= 256 ? backward_rows_of<64, 1>(sh, 3) : c <= 512 ? backward_rows_of<64, 2>(sh, 2) : c <= 768 ? backward_rows_of<64, 3>(sh, 1)
         : c <= 1024 ? backward_rows_of<64, 4>(sh, 1) : c <= 2048 ? backward_rows_of<128, 4>(sh, 1) : c <= 4096 ? backward_rows_of<256, 4>(sh, 2)
         : backward_rows_of<1024, 2>(sh, 1);
}

void launch_fold(const float* partial, uint32_t cols, uint32_t ranges, float* grad_gamma, float* grad_beta) {
    LaunchScope scope("ln_fold_kernel", "", static_cast<uint64_t>(ranges) * 2 * cols * sizeof(float));
    const uint32_t lanes = ranges <= 16 ? 4 : ranges <= 128 ? 16 : 64, per_block = kFoldBlock / lanes;
    const dim3 grid(std::min((cols - 1) / per_block + 1, kMaxFoldGrid), 2);
    auto* kernel = lanes == 4 ? ln_fold_kernel<4> : lanes == 16 ? ln_fold_kernel<16> : ln_fold_kernel<64>;
    hipLaunchKernelGGL(kernel, grid, dim3(kFoldBlock), 0, state().stream, partial, cols, ranges, grad_gamma, grad_beta);
}

uint64_t align256(uint64_t v) { return (v + 255) & ~255ull; }

}  // namespace

// A workgroup may use 64 KiB of dynamic LDS unless the kernel is granted more.
bool kth::layer_norm_init() {
    bool ok = true;
    for (const void* f : {reinterpret_cast<const void*>(&ln_forward_long_kernel<0>), reinterpret_cast<const void*>(&ln_forward_long_kernel<kLongRegisters>)})
        ok = ok && hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, kLdsRowFloats * 4) == hipSuccess;
    if (!ok) (void)hipGetLastError();
    return ok;
}

extern "C" {

int kth_layer_norm_forward(uint64_t in, const int32_t* shape, int dims, int axis, float epsilon, uint64_t gamma, uint64_t beta,
                           uint64_t out, uint64_t current_mean, uint64_t current_std) {
    std::lock_guard<std::mutex> guard(lock());
    KTH_REQUIRE_INIT();
    Shape2 sh; uint64_t n;
    if (int rc = shape_of("kth_layer_norm_forward", shape, dims, axis, &sh, &n)) return rc;
    if (!(epsilon >= 0.0f)) return fail(KTH_E_ARGUMENT, "kth_layer_norm_forward: epsilon %g is negative or NaN", epsilon);
    if (in == 0 || out == 0) return fail(KTH_E_ARGUMENT, "kth_layer_norm_forward: in and out must be given");
    Operand ops[6] = {{"in", in, n, false}, {"gamma", gamma, sh.cols, false}, {"beta", beta, sh.cols, false},
                      {"out", out, n, true}, {"current_mean", current_mean, sh.rows, true}, {"current_std", current_std, sh.rows, true}};
    if (int rc = resolve_operands("kth_layer_norm_forward", ops, 6, {{3, 0}})) return rc;
    float* const px = ops[0].ptr; float* const pga = ops[1].ptr; float* const pbe = ops[2].ptr;
    float* const pout = ops[3].ptr; float* const pmean = ops[4].ptr; float* const pstd = ops[5].ptr;

    if (sh.cols <= kForwardRowCols) {
        overwrite_results(ops, 6);
        LaunchScope scope("ln_forward_rows_kernel", "", n * 8);
        const ForwardRows k = forward_rows_kernel(sh);
        hipLaunchKernelGGL(k.kernel, dim3(k.grid), dim3(k.threads), 0, state().stream, px, pga, pbe, pout, pmean, pstd, sh, static_cast<double>(epsilon));
        KTH_LAUNCH_CHECK("layer_norm_forward");
        return KTH_OK;
    }
    if (sh.cols <= (sh.rows >= kLongRows ? kLongRowCols : kLdsRowFloats) && state().long_rows) {
        overwrite_results(ops, 6);
        LaunchScope scope("ln_forward_long_kernel", "", n * 8);
        const bool lds_alone = sh.cols <= kLdsRowFloats;
        const uint32_t held = lds_alone ? sh.cols : sh.cols - kLongRegisters * kLongThreads * 4;
        const uint32_t lds = (held + 3) / 4 * 16;
        const dim3 grid(std::min(sh.rows, device_units() * (lds <= 72 * 1024 ? 2u : 1u)));
        auto* kernel = lds_alone ? ln_forward_long_kernel<0> : ln_forward_long_kernel<kLongRegisters>;
        hipLaunchKernelGGL(kernel, grid, dim3(kLongThreads), lds, state().stream, px, pga, pbe, pout, pmean, pstd, sh, static_cast<double>(epsilon));
        KTH_LAUNCH_CHECK("layer_norm_forward");
        return KTH_OK;
    }
    const SegPlan pl = plan_segments(sh);
    const uint64_t rows_bytes = align256(static_cast<uint64_t>(sh.rows) * sizeof(RowForward));
    const uint64_t blocks = static_cast<uint64_t>(sh.rows) * pl.segments;
    const uint64_t ws_bytes = rows_bytes + blocks * 2 * sizeof(double);
    uint64_t cap;
    char* ws = reinterpret_cast<char*>(workspace_acquire(ws_bytes, &cap));
    if (!ws) return fail(KTH_E_MEMORY, "kth_layer_norm_forward: no workspace of %llu bytes", static_cast<unsigned long long>(ws_bytes));
    overwrite_results(ops, 6);
    RowForward* rows = reinterpret_cast<RowForward*>(ws);
    double* partial = reinterpret_cast<double*>(ws + rows_bytes);
    hipStream_t stream = state().stream;
    {
        LaunchScope scope("ln_sums_kernel", "forward", n * 4);
        hipLaunchKernelGGL((ln_sums_kernel<false>), dim3(pl.blocks), dim3(kBlock), 0, stream, px, nullptr, nullptr, partial, pl);
    }
    {
        LaunchScope scope("ln_rows_kernel", "forward", blocks * 16);
        hipLaunchKernelGGL((ln_rows_kernel<false>), dim3((sh.rows - 1) / 4 + 1), dim3(kBlock), 0, stream, px, partial, pl, static_cast<double>(epsilon),
                           rows, nullptr, pmean, pstd);
    }
    {
        LaunchScope scope("ln_apply_kernel", "", n * 8);
        hipLaunchKernelGGL(ln_apply_kernel, dim3(pl.blocks), dim3(kBlock), 0, stream, px, pga,
                           pbe, pout, rows, pl);
    }
    workspace_release(reinterpret_cast<float*>(ws), cap);
    KTH_LAUNCH_CHECK("layer_norm_forward");
    return KTH_OK;
}

int kth_layer_norm_backward(uint64_t in, const int32_t* shape, int dims, int axis, float epsilon, uint64_t gamma, uint64_t grad_out,
                            uint64_t grad_in, uint64_t grad_gamma, uint64_t grad_beta) {
    std::lock_guard<std::mutex> guard(lock());
    KTH_REQUIRE_INIT();
    Shape2 sh; uint64_t n;
    if (int rc = shape_of("kth_layer_norm_backward", shape, dims, axis, &sh, &n)) return rc;
    if (!(epsilon >= 0.0f)) return fail(KTH_E_ARGUMENT, "kth_layer_norm_backward: epsilon %g is negative or NaN", epsilon);
    if (in == 0 || grad_out == 0) return fail(KTH_E_ARGUMENT, "kth_layer_norm_backward: in and grad_out must be given");
    if (grad_in == 0 && grad_gamma == 0 && grad_beta == 0) return KTH_OK;
    Operand ops[6] = {{"in", in, n, false}, {"gamma", gamma, sh.cols, false}, {"grad_out", grad_out, n, false},
                      {"grad_in", grad_in, n, true}, {"grad_gamma", grad_gamma, sh.cols, true}, {"grad_beta", grad_beta, sh.cols, true}};
    if (int rc = resolve_operands("kth_layer_norm_backward", ops, 6, {{3, 2}})) return rc;
    float* const px = ops[0].ptr; float* const pga = ops[1].ptr; float* const pgo = ops[2].ptr;
    float* const pgi = ops[3].ptr; float* const pgg = ops[4].ptr; float* const pgb = ops[5].ptr;

    if (sh.cols <= kBackwardRowCols) {
        const BackwardRows k = backward_rows_kernel(sh);
        const uint64_t part_bytes = (pgg || pgb) && k.grid > 1 ? static_cast<uint64_t>(k.grid) * 2 * sh.cols * sizeof(float) : 0;
        uint64_t part_cap = 0;
        float* part = part_bytes ? workspace_acquire(part_bytes, &part_cap) : nullptr;
        if (part_bytes && !part) return fail(KTH_E_MEMORY, "kth_layer_norm_backward: no workspace of %llu bytes", static_cast<unsigned long long>(part_bytes));
        overwrite_results(ops, 6);
        {
            LaunchScope scope("ln_backward_rows_kernel", "", n * (pgi ? 12 : 8) + part_bytes);
            hipLaunchKernelGGL(k.kernel, dim3(k.grid), dim3(k.threads), 0, state().stream, px, pgo, pga, pgi, part, part ? nullptr : pgg, part ? nullptr : pgb, sh, static_cast<double>(epsilon));
        }
        if (part) {
            launch_fold(part, sh.cols, k.grid, pgg, pgb);
            workspace_release(part, part_cap);
        }
        KTH_LAUNCH_CHECK("layer_norm_backward");
        return KTH_OK;
    }
    const SegPlan pl = plan_segments(sh);
    ColPlan cp{};
    cp.sh = sh;
    cp.col_blocks = (sh.cols + kBlock * 4 - 1) / (kBlock * 4);
    cp.ranges = std::min(sh.rows, std::max(1u, (device_units() * 4 + cp.col_blocks - 1) / cp.col_blocks));
    cp.rows_per_range = (sh.rows + cp.ranges - 1) / cp.ranges;
    cp.ranges = (sh.rows + cp.rows_per_range - 1) / cp.rows_per_range;
    cp.col_div = make_div(cp.col_blocks);
    const bool weights = (pgg || pgb) && cp.ranges > 1;
    const uint64_t blocks = static_cast<uint64_t>(sh.rows) * pl.segments;
    const uint64_t rows_bytes = align256(static_cast<uint64_t>(sh.rows) * sizeof(RowBackward));
    const bool whole_rows = sh.cols <= kWholeRowCols || sh.rows >= 2 * device_units();
    const uint64_t sums_bytes = whole_rows ? 0 : align256(blocks * 4 * sizeof(double));
    const uint64_t cols_bytes = weights ? static_cast<uint64_t>(cp.ranges) * 2 * sh.cols * sizeof(float) : 0;
    const uint64_t ws_bytes = rows_bytes + sums_bytes + cols_bytes;
    uint64_t cap;
    char* ws = reinterpret_cast<char*>(workspace_acquire(ws_bytes, &cap));
    if (!ws) return fail(KTH_E_MEMORY, "kth_layer_norm_backward: no workspace of %llu bytes", static_cast<unsigned long long>(ws_bytes));
    overwrite_results(ops, 6);
    RowBackward* rows = reinterpret_cast<RowBackward*>(ws);
    double* sums = reinterpret_cast<double*>(ws + rows_bytes);
    float* partial = weights ? reinterpret_cast<float*>(ws + rows_bytes + sums_bytes) : nullptr;
    hipStream_t stream = state().stream;
    if (whole_rows) {
        LaunchScope scope("ln_row_sums_kernel", "", n * 8);
        hipLaunchKernelGGL(ln_row_sums_kernel, dim3(sh.rows), dim3(kLongThreads), 0, stream, px, pgo, pga, rows, sh, static_cast<double>(epsilon));
    } else {
        {
            LaunchScope scope("ln_sums_kernel", "backward", n * 8);
            hipLaunchKernelGGL((ln_sums_kernel<true>), dim3(pl.blocks), dim3(kBlock), 0, stream, px, pgo, pga, sums, pl);
        }
        {
            LaunchScope scope("ln_rows_kernel", "backward", blocks * 32);
            hipLaunchKernelGGL((ln_rows_kernel<true>), dim3((sh.rows - 1) / 4 + 1), dim3(kBlock), 0, stream, px, sums, pl, static_cast<double>(epsilon),
                               nullptr, rows, nullptr, nullptr);
        }
    }
    {
        LaunchScope scope("ln_cols_kernel", "", n * (pgi ? 12 : 8) + cols_bytes);
        hipLaunchKernelGGL(ln_cols_kernel, dim3(cp.col_blocks * cp.ranges), dim3(kBlock), 0, stream, px, pgo, pga, pgi,
                           rows, partial, weights ? nullptr : pgg, weights ? nullptr : pgb, cp);
    }
    if (weights) launch_fold(partial, sh.cols, cp.ranges, pgg, pgb);
    workspace_release(reinterpret_cast<float*>(ws), cap);
    KTH_LAUNCH_CHECK("layer_norm_backward");
    return KTH_OK;
}

}  // extern "C"
