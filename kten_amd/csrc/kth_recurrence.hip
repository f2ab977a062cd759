// The gated linear recurrence along one axis of a tensor seen as [outer, steps, inner], a channel per (outer, inner):
//
//   h_t = a_t h_{t-1} + u_t,   h_{-1} = initial (0 if not given)
//     KTH_GATE_GIVEN:    a = gate, u = in
//     KTH_GATE_SIGMOID:  a = 1 / (1 + exp(-gate)), u = (1 - a) in
//   d_t = grad_out_t + a_{t+1} d_{t+1},   d_{steps-1} = grad_out + grad_final
//     KTH_GATE_GIVEN:    grad_gate = d_t h_{t-1},  grad_in = d_t
//     KTH_GATE_SIGMOID:  grad_gate = d_t (h_{t-1} - in_t) a_t (1 - a_t),  grad_in = d_t (1 - a_t)
//     grad_initial = a_0 d_0
//
// States and their gradients are held in f64: a decay near 1 sums thousands of steps.
#include "kth_internal.h"

#include <algorithm>

using namespace kth;

namespace {

constexpr int kBlock = 256;
constexpr int kAhead = 8;            // steps whose loads are in flight at a time

__device__ __forceinline__ uint32_t divide(uint32_t n, FastDiv f) { return (__umulhi(n, f.mul) + n) >> f.shift; }

struct ScanShape {
    uint32_t outer, steps, inner;
    uint32_t channels;               // outer * inner
    FastDiv  inner_div;
};

// a and b = 1 - a of a gate, each to a relative error of a few 2^-24 (1 - a as a difference would lose it near a = 1,
// and with it the decay over many steps).
template <bool SIGMOID>
struct Gate {
    double a;
    float  b;
    __device__ __forceinline__ explicit Gate(float g) {
        if (SIGMOID) {
            const float e = expf(-fabsf(g));
            const float r = 1.0f / (1.0f + e), s = e * r;
            a = g >= 0.0f ? 1.0 - static_cast<double>(s) : static_cast<double>(s);
            b = g >= 0.0f ? s : r;
            if (g != g) { a = static_cast<double>(g); b = g; }
        } else {
            a = static_cast<double>(g);
            b = 1.0f;
        }
    }
    __device__ __forceinline__ double input(float x) const {
        return SIGMOID ? static_cast<double>(b) * static_cast<double>(x) : static_cast<double>(x);
    }
};

// A thread per channel walks its steps.
template <bool SIGMOID>
__global__ __launch_bounds__(kBlock) void recurrence_forward_kernel(const float* __restrict__ gate, const float* __restrict__ in, const float* initial,
                                                                    float* __restrict__ out, float* final_state, ScanShape sh) {
    const uint32_t ch = blockIdx.x * kBlock + threadIdx.x;
    if (ch >= sh.channels) return;
    const uint32_t o = divide(ch, sh.inner_div);
    uint64_t at = static_cast<uint64_t>(o) * sh.steps * sh.inner + (ch - o * sh.inner);
    double h = initial ? static_cast<double>(initial[ch]) : 0.0;
    for (uint32_t t0 = 0; t0 < sh.steps; t0 += kAhead) {
        float g[kAhead], x[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; k++)
            if (t0 + k < sh.steps) { g[k] = gate[at + static_cast<uint64_t>(k) * sh.inner]; x[k] = in[at + static_cast<uint64_t>(k) * sh.inner]; }
#pragma unroll
        for (int k = 0; k < kAhead; k++)
            if (t0 + k < sh.steps) {
                const Gate<SIGMOID> c(g[k]);
                h = fma(c.a, h, c.input(x[k]));
                out[at + static_cast<uint64_t>(k) * sh.inner] = static_cast<float>(h);
            }
        at += static_cast<uint64_t>(kAhead) * sh.inner;
    }
    if (final_state) final_state[ch] = static_cast<float>(h);
}

template <bool SIGMOID>
__global__ __launch_bounds__(kBlock) void recurrence_backward_kernel(const float* __restrict__ gate, const float* __restrict__ in, const float* __restrict__ initial,
                                                                     const float* __restrict__ out, const float* __restrict__ grad_out,
                                                                     const float* __restrict__ grad_final, float* __restrict__ grad_gate,
                                                                     float* __restrict__ grad_in, float* __restrict__ grad_initial, ScanShape sh) {
    const uint32_t ch = blockIdx.x * kBlock + threadIdx.x;
    if (ch >= sh.channels) return;
    const uint32_t o = divide(ch, sh.inner_div);
    const uint64_t first = static_cast<uint64_t>(o) * sh.steps * sh.inner + (ch - o * sh.inner);
    const float h0 = initial ? initial[ch] : 0.0f;
    double carry = grad_final ? static_cast<double>(grad_final[ch]) : 0.0;      // a_{t+1} d_{t+1}
    for (uint32_t left = sh.steps; left > 0; left--) {
        const uint32_t t = left - 1;
        const uint64_t at = first + static_cast<uint64_t>(t) * sh.inner;
        const Gate<SIGMOID> c(gate[at]);
        const double d = static_cast<double>(grad_out[at]) + carry;
        if (grad_gate) {                                 // (without it out and in need not be given)
            const float before = t > 0 ? out[at - sh.inner] : h0;
            grad_gate[at] = static_cast<float>(SIGMOID ? d * (static_cast<double>(before) - static_cast<double>(in[at])) * (c.a * static_cast<double>(c.b))
                                                       : d * static_cast<double>(before));
        }
        if (grad_in) grad_in[at] = static_cast<float>(SIGMOID ? d * static_cast<double>(c.b) : d);
        carry = c.a * d;
    }
    if (grad_initial) grad_initial[ch] = static_cast<float>(carry);
}

// ---------------------------------------------------------------- host side

int shape_of(const char* what, const int32_t* shape, int dims, int axis, int mode, ScanShape* sh, uint64_t* n) {
    if (mode != KTH_GATE_GIVEN && mode != KTH_GATE_SIGMOID) return fail(KTH_E_ARGUMENT, "%s: gate mode %d", what, mode);
    if (dims < 1 || dims > KTH_MAX_DIMS) return fail(KTH_E_ARGUMENT, "%s: %d dims", what, dims);
    if (!shape) return fail(KTH_E_ARGUMENT, "%s: null shape", what);
    if (axis < 0 || axis >= dims) return fail(KTH_E_ARGUMENT, "%s: axis %d of %d dims", what, axis, dims);
    uint64_t total = 1, outer = 1, inner = 1;
    for (int d = 0; d < dims; d++) {
        if (shape[d] < 1) return fail(KTH_E_ARGUMENT, "%s: dim %d is %d", what, d, shape[d]);
        total *= static_cast<uint64_t>(shape[d]);
        if (total > kMaxElements) return fail(KTH_E_ARGUMENT, "%s: more than 2^31-1 elements", what);
        if (d < axis) outer *= static_cast<uint64_t>(shape[d]);
        if (d > axis) inner *= static_cast<uint64_t>(shape[d]);
    }
    sh->outer = static_cast<uint32_t>(outer);
    sh->steps = static_cast<uint32_t>(shape[axis]);
    sh->inner = static_cast<uint32_t>(inner);
    sh->channels = static_cast<uint32_t>(outer * inner);
    sh->inner_div = make_div(sh->inner);
    *n = total;
    return KTH_OK;
}

}  // namespace

extern "C" {

int kth_gated_recurrence_forward(uint64_t gate, uint64_t in, const int32_t* shape, int dims, int axis, int mode, uint64_t initial,
                                 uint64_t out, uint64_t final_state) {
    static const char* what = "kth_gated_recurrence_forward";
    std::lock_guard<std::mutex> guard(lock());
    KTH_REQUIRE_INIT();
    ScanShape sh{}; uint64_t n;
    if (int rc = shape_of(what, shape, dims, axis, mode, &sh, &n)) return rc;
    if (gate == 0 || in == 0 || out == 0) return fail(KTH_E_ARGUMENT, "%s: gate, in and out must be given", what);
    Operand ops[5] = {{"gate", gate, n, false}, {"in", in, n, false}, {"initial", initial, sh.channels, false},
                      {"out", out, n, true}, {"final_state", final_state, sh.channels, true}};
    if (int rc = resolve_operands(what, ops, 5, {{4, 2}})) return rc;          // the state may be updated in place
    LaunchScope scope("recurrence_forward_kernel", mode == KTH_GATE_SIGMOID ? "sigmoid" : "given", (3 * n + 2 * sh.channels) * 4);
    const dim3 grid((sh.channels - 1) / kBlock + 1);
    if (mode == KTH_GATE_SIGMOID)
        hipLaunchKernelGGL((recurrence_forward_kernel<true>), grid, dim3(kBlock), 0, state().stream, ops[0].ptr, ops[1].ptr, ops[2].ptr, ops[3].ptr, ops[4].ptr, sh);
    else
        hipLaunchKernelGGL((recurrence_forward_kernel<false>), grid, dim3(kBlock), 0, state().stream, ops[0].ptr, ops[1].ptr, ops[2].ptr, ops[3].ptr, ops[4].ptr, sh);
    KTH_LAUNCH_CHECK("gated_recurrence_forward");
    return KTH_OK;
}

int kth_gated_recurrence_backward(uint64_t gate, uint64_t in, const int32_t* shape, int dims, int axis, int mode, uint64_t initial, uint64_t out,
                                  uint64_t grad_out, uint64_t grad_final, uint64_t grad_gate, uint64_t grad_in, uint64_t grad_initial) {
    static const char* what = "kth_gated_recurrence_backward";
    std::lock_guard<std::mutex> guard(lock());
    KTH_REQUIRE_INIT();
    ScanShape sh{}; uint64_t n;
    if (int rc = shape_of(what, shape, dims, axis, mode, &sh, &n)) return rc;
    const bool sigmoid = mode == KTH_GATE_SIGMOID;
    if (gate == 0 || grad_out == 0) return fail(KTH_E_ARGUMENT, "%s: gate and grad_out must be given", what);
    if (grad_gate == 0 && grad_in == 0 && grad_initial == 0) return KTH_OK;
    if (grad_gate != 0 && (out == 0 || (sigmoid && in == 0)))
        return fail(KTH_E_ARGUMENT, "%s: the gate's gradient needs out%s", what, sigmoid ? " and in" : "");
    Operand ops[9] = {{"gate", gate, n, false}, {"in", sigmoid && grad_gate ? in : 0, n, false},
                      {"initial", grad_gate ? initial : 0, sh.channels, false}, {"out", grad_gate ? out : 0, n, false},
                      {"grad_out", grad_out, n, false}, {"grad_final", grad_final, sh.channels, false},
                      {"grad_gate", grad_gate, n, true}, {"grad_in", grad_in, n, true},
                      {"grad_initial", grad_initial, sh.channels, true}};
    if (int rc = resolve_operands(what, ops, 9, {})) return rc;
    LaunchScope scope("recurrence_backward_kernel", sigmoid ? "sigmoid" : "given", (sigmoid ? 6 : 5) * n * 4);
    const dim3 grid((sh.channels - 1) / kBlock + 1);
    if (sigmoid)
        hipLaunchKernelGGL((recurrence_backward_kernel<true>), grid, dim3(kBlock), 0, state().stream, ops[0].ptr, ops[1].ptr, ops[2].ptr, ops[3].ptr, ops[4].ptr,
                           ops[5].ptr, ops[6].ptr, ops[7].ptr, ops[8].ptr, sh);
    else
        hipLaunchKernelGGL((recurrence_backward_kernel<false>), grid, dim3(kBlock), 0, state().stream, ops[0].ptr, ops[1].ptr, ops[2].ptr, ops[3].ptr, ops[4].ptr,
                           ops[5].ptr, ops[6].ptr, ops[7].ptr, ops[8].ptr, sh);
    KTH_LAUNCH_CHECK("gated_recurrence_backward");
    return KTH_OK;
}

}  // extern "C"
