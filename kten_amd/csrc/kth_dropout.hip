// Dropout from a counter-based generator: out = [residual +] in * 1 / (1 - p) where the element's random number is at least
// p * 2^32, [residual +] 0 elsewhere. The mask is a function of (seed, offset, position) and is never stored: the backward
// pass is the same call on the gradient.
//
// The generator is the ten-round 4x32 one of Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as 1, 2, 3"
// (2011): four 32-bit words from a 128-bit counter and a 64-bit key. Key: seed. Counter: offset + i / 4 in its low 64 bits,
// for element i, which takes word i % 4; so a lane's float4 is one evaluation.
#include "kth_internal.h"

using namespace kth;

namespace {

constexpr int kBlock = 256;
constexpr int kUnroll = 2;

typedef float v4f __attribute__((ext_vector_type(4)));

struct Words { uint32_t w[4]; };

__device__ __forceinline__ Words random_words(uint64_t counter, uint64_t seed) {
    uint32_t c0 = static_cast<uint32_t>(counter), c1 = static_cast<uint32_t>(counter >> 32), c2 = 0, c3 = 0;
    uint32_t k0 = static_cast<uint32_t>(seed), k1 = static_cast<uint32_t>(seed >> 32);
#pragma unroll
    for (int round = 0; round < 10; round++) {
        const uint64_t p0 = static_cast<uint64_t>(c0) * 0xD2511F53u, p1 = static_cast<uint64_t>(c2) * 0xCD9E8D57u;
        c0 = static_cast<uint32_t>(p1 >> 32) ^ c1 ^ k0;
        c1 = static_cast<uint32_t>(p1);
        c2 = static_cast<uint32_t>(p0 >> 32) ^ c3 ^ k1;
        c3 = static_cast<uint32_t>(p0);
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return Words{{c0, c1, c2, c3}};
}

struct DropoutPlan {
    uint64_t seed, offset;
    uint32_t n;
    uint32_t threshold;     // kept where the number is at least this
    uint32_t none;          // p == 1: no number reaches 2^32
    float    scale;
};

__device__ __forceinline__ float drop(float x, uint32_t number, const DropoutPlan& pl) {
    return number >= pl.threshold && !pl.none ? x * pl.scale : 0.0f;
}

// A thread takes kUnroll float4s, kBlock apart. Results may be written over either operand. Bound by memory: 2^26 values with a
// residual take 135.5 us (5.9 TB/s; a plain sum of two tensors 129.5), the generator's 20 multiplications a float4 hide behind it.
template <bool RESIDUAL>
__global__ __launch_bounds__(kBlock) void dropout_kernel(const float* in, const float* residual, float* out, DropoutPlan pl) {
    const uint32_t base = blockIdx.x * (kBlock * kUnroll) + threadIdx.x;
    const uint32_t n4 = pl.n >> 2;
    v4f x[kUnroll], y[kUnroll];
#pragma unroll
    for (int k = 0; k < kUnroll; k++) {
        const uint32_t i = base + k * kBlock;
        if (i < n4) {
            x[k] = __builtin_nontemporal_load(reinterpret_cast<const v4f*>(in) + i);
            if (RESIDUAL) y[k] = __builtin_nontemporal_load(reinterpret_cast<const v4f*>(residual) + i);
        }
    }
#pragma unroll
    for (int k = 0; k < kUnroll; k++) {
        const uint32_t i = base + k * kBlock;
        if (i < n4) {
            const Words r = random_words(pl.offset + i, pl.seed);
            v4f z;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                z[e] = drop(x[k][e], r.w[e], pl);
                if (RESIDUAL) z[e] = y[k][e] + z[e];
            }
            reinterpret_cast<v4f*>(out)[i] = z;
        }
    }
    const uint32_t rest = pl.n & 3u;                   // the last n % 4 elements
    if (blockIdx.x == 0 && threadIdx.x < rest) {
        const uint32_t i = (n4 << 2) + threadIdx.x;
        const Words r = random_words(pl.offset + n4, pl.seed);
        const float z = drop(in[i], threadIdx.x == 0 ? r.w[0] : threadIdx.x == 1 ? r.w[1] : r.w[2], pl);
        out[i] = RESIDUAL ? residual[i] + z : z;
    }
}

}  // namespace

extern "C" {

int kth_dropout(uint64_t in, uint64_t n, double p, uint64_t seed, uint64_t offset, uint64_t residual, uint64_t out) {
    std::lock_guard<std::mutex> guard(lock());
    KTH_REQUIRE_INIT();
    if (!(p >= 0.0 && p <= 1.0)) return fail(KTH_E_ARGUMENT, "kth_dropout: probability %g outside [0, 1]", p);
    if (in == 0 || out == 0) return fail(KTH_E_HANDLE, "kth_dropout: in and out must be given");
    Operand ops[3] = {{"in", in, n, false}, {"residual", residual, n, false}, {"out", out, n, true}};
    if (int rc = resolve_operands("kth_dropout", ops, 3, {{2, 0}, {2, 1}}, KTH_E_ARGUMENT)) return rc;
    if (n == 0) return KTH_OK;
    overwrite_results(ops, 3);
    const float* sr = ops[1].ptr;
    DropoutPlan pl{};
    pl.seed = seed; pl.offset = offset;
    pl.n = static_cast<uint32_t>(n);
    pl.none = p == 1.0 ? 1u : 0u;
    // (the largest double below 1 times 2^32 is below 2^32)
    pl.threshold = pl.none ? 0u : static_cast<uint32_t>(p * 4294967296.0);
    pl.scale = pl.none ? 0.0f : static_cast<float>(1.0 / (1.0 - p));
    const uint32_t blocks = ((pl.n >> 2) + kBlock * kUnroll - 1) / (kBlock * kUnroll);
    const dim3 grid(blocks == 0 ? 1 : blocks);
    LaunchScope scope("dropout_kernel", sr ? "residual" : "", n * (sr ? 12 : 8));
    if (sr) hipLaunchKernelGGL((dropout_kernel<true>), grid, dim3(kBlock), 0, state().stream, ops[0].ptr, sr, ops[2].ptr, pl);
    else    hipLaunchKernelGGL((dropout_kernel<false>), grid, dim3(kBlock), 0, state().stream, ops[0].ptr, nullptr, ops[2].ptr, pl);
    KTH_LAUNCH_CHECK("dropout");
    return KTH_OK;
}

}  // extern "C"
