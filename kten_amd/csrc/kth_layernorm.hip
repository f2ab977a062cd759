// Layer normalisation over the trailing dims of a tensor, seen as [rows, cols]: forward, and backward with the reduction
// of the weights' gradients. The reference has batch normalisation only; the operands, the optional ones and the float
// conventions follow BatchNormOperation (kten-api/.../tensor/operations/nn/BatchNormOperation.kt:5-41).
//
//   forward    m = sum x / n,  v = sum (x - m)^2 / n,  r = 1 / sqrt(v + eps),  y = (x - m) r gamma + beta
//   backward   xh = (x - m) r,  w = go gamma:   gin = r (w - mean(w) - xh mean(w xh)),
//              grad_gamma = sum over rows of go xh,  grad_beta = sum over rows of go
//
// Every sum is made in f64 from d = x - k with k the row's first element (as the batch norm kernels do): the sums of d and
// d^2 then give the mean and the variance in one pass, at a cancellation of at most n 2^-53 of the spread around k; the
// backward pass takes the sums of w and w d along and works the statistics out again, so that it needs nothing saved.
// Sums are folded in a fixed order: the same input gives the same bits.
#include "kth_internal.h"

#include <algorithm>

using namespace kth;

namespace {

constexpr int kBlock = 256;
constexpr uint32_t kMaxGrid = 1u << 20;      // (a launch may have fewer than 2^32 threads)

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

__device__ __forceinline__ float ln_forward(float x, double mean, float rstd, float gamma, float beta) {
    return static_cast<float>(static_cast<double>(x) - mean) * rstd * gamma + beta;
}

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

// ---------------------------------------------------------------- rows in segments (any size)

struct SegPlan {
    Shape2   sh;
    uint32_t segments, seg_len;      // segments per row, columns per segment (a multiple of 4)
    uint32_t blocks;                 // rows x segments; a grid of at most kMaxGrid workgroups strides over them
    FastDiv  seg_div;
};

// Workgroup b sums segment b % segments of row b / segments: forward d, d^2; backward also w, w d.
template <bool BACKWARD>
__global__ __launch_bounds__(kBlock) void ln_sums_kernel(const float* __restrict__ x, const float* __restrict__ go,
                                                         const float* __restrict__ gamma, double* __restrict__ partial, SegPlan pl) {
    constexpr int NS = BACKWARD ? 4 : 2;
    __shared__ double lds[NS * kBlock / 64];
    for (uint32_t b = blockIdx.x; b < pl.blocks; b += gridDim.x) {
    const uint32_t row = divide(b, pl.seg_div);
    const uint32_t seg = b - row * pl.segments;
    const float* xr = x + static_cast<uint64_t>(row) * pl.sh.cols;
    const float* gr = BACKWARD ? go + static_cast<uint64_t>(row) * pl.sh.cols : nullptr;
    const uint32_t first = seg * pl.seg_len;
    const uint32_t last = min(first + pl.seg_len, pl.sh.cols);
    const double k = static_cast<double>(xr[0]);
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
    __syncthreads();
    }
}

// One wave per row folds its segments (lane l takes l, l + 64, ...; then the lanes by xor-shuffles).
template <bool BACKWARD>
__global__ __launch_bounds__(kBlock) void ln_rows_kernel(const float* __restrict__ x, const double* __restrict__ partial, SegPlan pl, double eps,
                                                         RowForward* __restrict__ fwd, RowBackward* __restrict__ bwd,
                                                         float* __restrict__ out_mean, float* __restrict__ out_std) {
    constexpr int NS = BACKWARD ? 4 : 2;
    for (uint32_t row = blockIdx.x * (kBlock / 64) + (threadIdx.x >> 6); row < pl.sh.rows; row += gridDim.x * (kBlock / 64)) {
    double s[NS] = {};
    for (uint32_t t = threadIdx.x & 63; t < pl.segments; t += 64)
#pragma unroll
        for (int i = 0; i < NS; i++) s[i] += partial[(static_cast<uint64_t>(row) * pl.segments + t) * NS + i];
#pragma unroll
    for (int off = 32; off > 0; off >>= 1)
#pragma unroll
        for (int i = 0; i < NS; i++) s[i] += __shfl_xor(s[i], off);
    if ((threadIdx.x & 63) != 0) continue;
    const double inv = pl.sh.inv_cols;
    const double delta = s[0] * inv;
    const double mean = static_cast<double>(x[static_cast<uint64_t>(row) * pl.sh.cols]) + delta;
    const double rstd = row_rstd(row_variance(s[0], s[1], inv), eps);
    if (BACKWARD) {
        bwd[row] = RowBackward{mean, rstd, s[NS - 2] * inv, (s[NS - 1] - delta * s[NS - 2]) * rstd * rstd * inv};
    } else {
        fwd[row] = RowForward{mean, rstd};
        if (out_mean) out_mean[row] = static_cast<float>(mean);
        if (out_std) out_std[row] = static_cast<float>(rstd);
    }
    }
}

__global__ __launch_bounds__(kBlock) void ln_apply_kernel(const float* x, const float* __restrict__ gamma, const float* __restrict__ beta, float* out,
                                                          const RowForward* __restrict__ fwd, SegPlan pl) {
    for (uint32_t b = blockIdx.x; b < pl.blocks; b += gridDim.x) {
    const uint32_t row = divide(b, pl.seg_div);
    const uint32_t seg = b - row * pl.segments;
    const uint64_t at = static_cast<uint64_t>(row) * pl.sh.cols;
    const uint32_t first = seg * pl.seg_len;
    const uint32_t last = min(first + pl.seg_len, pl.sh.cols);
    const double mean = fwd[row].mean;
    const float rstd = static_cast<float>(fwd[row].rstd);
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
}

// ---------------------------------------------------------------- backward by columns

struct ColPlan {
    Shape2   sh;
    uint32_t col_blocks, ranges, rows_per_range;
    FastDiv  col_div;
};

// A thread owns four columns of one range of rows: it writes the input gradient of each row and sums the weights'
// gradients down the range. The partials are floats: each is a f64 sum rounded once (2^-24 of itself), folded in f64.
__global__ __launch_bounds__(kBlock) void ln_cols_kernel(const float* __restrict__ x, const float* go, const float* __restrict__ gamma, float* grad_in,
                                                         const RowBackward* __restrict__ rows, float* __restrict__ partial, ColPlan pl) {
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
    if (partial) {
        float* pg = partial + static_cast<uint64_t>(range) * 2 * pl.sh.cols;
        for (uint32_t e = 0; e < width; e++) { pg[c + e] = static_cast<float>(sg[e]); pg[pl.sh.cols + c + e] = static_cast<float>(sb[e]); }
    }
}

// grad_gamma and grad_beta from `ranges` partial rows of [2, cols]: a workgroup takes 32 columns, eight lanes a column,
// each with every eighth range; then a tree over the eight. Which of the two sums: blockIdx.y.
constexpr uint32_t kFoldCols = 32, kFoldLanes = kBlock / kFoldCols;
__global__ __launch_bounds__(kBlock) void ln_fold_kernel(const float* __restrict__ partial, uint32_t cols, uint32_t ranges,
                                                         float* __restrict__ grad_gamma, float* __restrict__ grad_beta) {
    __shared__ double lds[kBlock];
    float* out = blockIdx.y == 0 ? grad_gamma : grad_beta;
    if (!out) return;
    const uint32_t lane = threadIdx.x / kFoldCols;
    for (uint32_t c0 = blockIdx.x * kFoldCols; c0 < cols; c0 += gridDim.x * kFoldCols) {
        const uint32_t c = c0 + threadIdx.x % kFoldCols;
        double s = 0.0;
        if (c < cols)
            for (uint32_t r = lane; r < ranges; r += kFoldLanes) s += static_cast<double>(partial[(static_cast<uint64_t>(r) * 2 + blockIdx.y) * cols + c]);
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

uint64_t align256(uint64_t v) { return (v + 255) & ~255ull; }

}  // namespace

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

    const SegPlan pl = plan_segments(sh);
    const uint64_t rows_bytes = align256(static_cast<uint64_t>(sh.rows) * sizeof(RowForward));
    const uint64_t blocks = static_cast<uint64_t>(sh.rows) * pl.segments;
    const uint64_t ws_bytes = rows_bytes + blocks * 2 * sizeof(double);
    uint64_t cap;
    char* ws = reinterpret_cast<char*>(workspace_acquire(ws_bytes, &cap));
    if (!ws) return fail(KTH_E_MEMORY, "kth_layer_norm_forward: no workspace of %llu bytes", static_cast<unsigned long long>(ws_bytes));
    RowForward* rows = reinterpret_cast<RowForward*>(ws);
    double* partial = reinterpret_cast<double*>(ws + rows_bytes);
    hipStream_t stream = state().stream;
    {
        LaunchScope scope("ln_sums_kernel", "forward", n * 4);
        hipLaunchKernelGGL((ln_sums_kernel<false>), dim3(std::min(pl.blocks, kMaxGrid)), dim3(kBlock), 0, stream, px, nullptr, nullptr, partial, pl);
    }
    {
        LaunchScope scope("ln_rows_kernel", "forward", blocks * 16);
        hipLaunchKernelGGL((ln_rows_kernel<false>), dim3(std::min((sh.rows - 1) / 4 + 1, kMaxGrid)), dim3(kBlock), 0, stream, px, partial, pl, static_cast<double>(epsilon),
                           rows, nullptr, pmean, pstd);
    }
    {
        LaunchScope scope("ln_apply_kernel", "", n * 8);
        hipLaunchKernelGGL(ln_apply_kernel, dim3(std::min(pl.blocks, kMaxGrid)), dim3(kBlock), 0, stream, px, pga,
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

    const SegPlan pl = plan_segments(sh);
    ColPlan cp{};
    cp.sh = sh;
    cp.col_blocks = (sh.cols + kBlock * 4 - 1) / (kBlock * 4);
    cp.ranges = std::min(sh.rows, std::max(1u, (device_units() * 4 + cp.col_blocks - 1) / cp.col_blocks));
    cp.rows_per_range = (sh.rows + cp.ranges - 1) / cp.ranges;
    cp.ranges = (sh.rows + cp.rows_per_range - 1) / cp.rows_per_range;
    cp.col_div = make_div(cp.col_blocks);
    const bool weights = pgg || pgb;
    const uint64_t blocks = static_cast<uint64_t>(sh.rows) * pl.segments;
    const uint64_t rows_bytes = align256(static_cast<uint64_t>(sh.rows) * sizeof(RowBackward));
    const uint64_t sums_bytes = align256(blocks * 4 * sizeof(double));
    const uint64_t cols_bytes = weights ? static_cast<uint64_t>(cp.ranges) * 2 * sh.cols * sizeof(float) : 0;
    const uint64_t ws_bytes = rows_bytes + sums_bytes + cols_bytes;
    uint64_t cap;
    char* ws = reinterpret_cast<char*>(workspace_acquire(ws_bytes, &cap));
    if (!ws) return fail(KTH_E_MEMORY, "kth_layer_norm_backward: no workspace of %llu bytes", static_cast<unsigned long long>(ws_bytes));
    RowBackward* rows = reinterpret_cast<RowBackward*>(ws);
    double* sums = reinterpret_cast<double*>(ws + rows_bytes);
    float* partial = weights ? reinterpret_cast<float*>(ws + rows_bytes + sums_bytes) : nullptr;
    hipStream_t stream = state().stream;
    {
        LaunchScope scope("ln_sums_kernel", "backward", n * 8);
        hipLaunchKernelGGL((ln_sums_kernel<true>), dim3(std::min(pl.blocks, kMaxGrid)), dim3(kBlock), 0, stream, px, pgo, pga, sums, pl);
    }
    {
        LaunchScope scope("ln_rows_kernel", "backward", blocks * 32);
        hipLaunchKernelGGL((ln_rows_kernel<true>), dim3(std::min((sh.rows - 1) / 4 + 1, kMaxGrid)), dim3(kBlock), 0, stream, px, sums, pl, static_cast<double>(epsilon),
                           nullptr, rows, nullptr, nullptr);
    }
    {
        LaunchScope scope("ln_cols_kernel", "", n * (pgi ? 12 : 8) + cols_bytes);
        hipLaunchKernelGGL(ln_cols_kernel, dim3(cp.col_blocks * cp.ranges), dim3(kBlock), 0, stream, px, pgo, pga, pgi,
                           rows, partial, cp);
    }
    if (weights) {
        LaunchScope scope("ln_fold_kernel", "", cols_bytes);
        hipLaunchKernelGGL(ln_fold_kernel, dim3(std::min((sh.cols - 1) / kFoldCols + 1, kMaxGrid), 2), dim3(kBlock), 0, stream, partial, sh.cols, cp.ranges,
                           pgg, pgb);
    }
    workspace_release(reinterpret_cast<float*>(ws), cap);
    KTH_LAUNCH_CHECK("layer_norm_backward");
    return KTH_OK;
}

}  // extern "C"
