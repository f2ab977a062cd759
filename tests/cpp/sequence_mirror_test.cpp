// The layers over sequences through the C++ host mirror (include/kten_hip.hpp) on values worked out by hand, all of them
// exact in fp32, and their refusals. Exit status 0 means every check held.
#include <cstdio>
#include <initializer_list>
#include <stdexcept>

#include "kten_hip.hpp"

using namespace kten::hip;

static int g_checks = 0, g_failed = 0;

static void expect(bool ok, const char* what) {
    g_checks++;
    if (!ok) { g_failed++; std::printf("FAILED: %s\n", what); std::fflush(stdout); }
}

static void expect_values(const Raw& t, const Shape& shape, std::initializer_list<float> values, const char* what) {
    expect(t && t->shape == shape && t->toVector() == std::vector<float>(values), what);
}

template <class E, class F>
static void expect_throw(F&& f, const char* what) {
    bool thrown = false;
    try { f(); } catch (const E&) { thrown = true; }
    expect(thrown, what);
}

static Raw tensor(HipTensorOperations& ops, const Shape& shape, std::initializer_list<float> values) {
    std::vector<float> v(values);
    return ops.createRaw(shape, [&](int i) { return v[static_cast<size_t>(i)]; });
}

static void layer_norm(HipTensorOperations& ops) {
    // rows (1, 3) and (2, 6): means 2 and 4, variances 1 and 4, normalised (-1, 1) both
    Raw x = tensor(ops, {2, 1, 2}, {1, 3, 2, 6}), gamma = tensor(ops, {2}, {2, 4}), beta = tensor(ops, {2}, {10, 20});
    auto norm = ops.layerNorm(-1, 0.0f);
    auto out = norm.calculateOutput(x, gamma, beta);
    expect_values(out.output, {2, 1, 2}, {8, 24, 8, 24}, "layerNorm with gamma and beta");
    expect_values(out.currentMean, {2, 1}, {2, 4}, "layerNorm: row means");
    expect_values(out.currentStd, {2, 1}, {1, 0.5f}, "layerNorm: 1 / sqrt(var)");
    expect_values(ops.layerNorm(0, 0.0f).calculateOutput(tensor(ops, {2}, {1, 3}), nullptr, nullptr).output, {2}, {-1, 1}, "one row, no weights");
    auto g = norm.calculateGrads(x, nullptr, ops.createRawFill({2, 1, 2}, 1.0f), true, true, true);
    expect_values(g.gradIn, {2, 1, 2}, {0, 0, 0, 0}, "layerNorm: a constant gradient gives no input gradient");
    expect_values(g.gradGamma, {2}, {-2, 2}, "layerNorm gradGamma");
    expect_values(g.gradBeta, {2}, {2, 2}, "layerNorm gradBeta");
    auto only = norm.calculateGrads(x, gamma, out.output, false, false, true);
    expect(!only.gradIn && !only.gradGamma, "a gradient that is not required is not produced");
    expect_values(only.gradBeta, {2}, {16, 48}, "layerNorm gradBeta alone");
    expect(!norm.calculateGrads(x, gamma, out.output, false, false, false).gradBeta, "nothing required, nothing done");
    expect_throw<std::invalid_argument>([&] { norm.calculateOutput(x, x, nullptr); }, "gamma of the wrong size");
    expect_throw<std::invalid_argument>([&] { norm.calculateGrads(x, gamma, gamma, true, true, true); }, "a gradient of the wrong size");
    expect_throw<std::invalid_argument>([&] { ops.layerNorm(3, 0.0f).calculateOutput(x, nullptr, nullptr); }, "an axis outside the shape");
    expect_throw<std::invalid_argument>([&] { ops.layerNorm(-1, -1.0f).calculateOutput(x, nullptr, nullptr); }, "a negative epsilon");
}

static void dropout(HipTensorOperations& ops) {
    const int n = 1000;
    Raw x = ops.createRaw({n}, [](int i) { return static_cast<float>(i + 1); }), ones = ops.createRawFill({n}, 1.0f);
    expect(ops.dropout(0.0, 7).calculateOutput(x)->toVector() == x->toVector(), "dropout with p = 0 keeps all");
    expect(ops.dropout(1.0, 7).calculateOutput(x, ones)->toVector() == ones->toVector(), "dropout with p = 1 leaves the residual");
    auto half = ops.dropout(0.5, 7);
    const std::vector<float> y = half.calculateOutput(x)->toVector(), g = half.calculateGrad(ones)->toVector(),
                             r = half.calculateOutput(x, ones)->toVector();
    int kept = 0;
    bool same = true;
    for (int i = 0; i < n; i++) {
        kept += g[i] != 0.0f;
        same = same && (g[i] == 0.0f || g[i] == 2.0f) && y[i] == g[i] * static_cast<float>(i + 1) && r[i] == y[i] + 1.0f;
    }
    expect(same, "the gradient and the residual form keep the values that the output keeps");
    expect(kept > 400 && kept < 600, "about half of the values are kept (six standard deviations of 16)");
    // values 4 k .. 4 k + 3 belong to counter offset + k
    const std::vector<float> later = ops.dropout(0.5, 7, 100).calculateOutput(ones)->toVector();
    expect(std::vector<float>(later.begin(), later.begin() + 600) == std::vector<float>(g.begin() + 400, g.end()), "offset 100 goes on at value 400");
    expect_throw<std::invalid_argument>([&] { ops.dropout(1.5, 7); }, "a probability above 1");
    expect_throw<std::invalid_argument>([&] { half.calculateOutput(x, tensor(ops, {1}, {1})); }, "a residual of the wrong size");
}

static void recurrence(HipTensorOperations& ops) {
    // two channels, three steps: h = 0.5 h + 1 from 4, and h = 2 h + 1 from 1
    Raw gate = tensor(ops, {3, 2}, {0.5f, 2, 0.5f, 2, 0.5f, 2}), in = ops.createRawFill({3, 2}, 1.0f), h0 = tensor(ops, {2}, {4, 1});
    auto given = ops.gatedRecurrence(0, false);
    auto out = given.calculateOutput(gate, in, h0);
    expect_values(out.output, {3, 2}, {3, 3, 2.5f, 7, 2.25f, 15}, "recurrence: the states");
    expect_values(out.finalState, {2}, {2.25f, 15}, "recurrence: the last state");
    expect_values(given.calculateOutput(gate, in, nullptr).finalState, {2}, {1.75f, 7}, "recurrence from zeros");
    Raw state = h0->copy(false), token_gate = tensor(ops, {1, 2}, {0.5f, 2}), token = ops.createRawFill({1, 2}, 1.0f);
    expect_values(given.step(token_gate, token, state), {1, 2}, {3, 3}, "one step");
    expect_values(given.step(token_gate, token, state), {1, 2}, {2.5f, 7}, "the next step goes on from the state");
    expect_values(state, {2}, {2.5f, 7}, "the state is updated in place");
    expect_values(h0, {2}, {4, 1}, "the store it was copied from is not");
    // a gradient of the last state alone: 1, then times the gate per step
    Raw last = tensor(ops, {2}, {1, 1}), none = ops.createRawFill({3, 2}, 0.0f);
    auto g = given.calculateGrads(gate, in, h0, out.output, none, last, true, true, true);
    expect_values(g.gradIn, {3, 2}, {0.25f, 4, 0.5f, 2, 1, 1}, "recurrence gradIn");
    expect_values(g.gradGate, {3, 2}, {1, 4, 1.5f, 6, 2.5f, 7}, "recurrence gradGate");
    expect_values(g.gradInitial, {2}, {0.125f, 8}, "recurrence gradInitial");
    auto part = given.calculateGrads(gate, in, nullptr, nullptr, none, last, false, true, false);
    expect(!part.gradGate && !part.gradInitial, "a gradient that is not required is not produced");
    expect_values(part.gradIn, {3, 2}, {0.25f, 4, 0.5f, 2, 1, 1}, "gradIn needs no output");
    // sigmoid(0) = 0.5: the mean of the state and the input
    Raw zeros = ops.createRawFill({1, 2}, 0.0f);
    expect_values(ops.gatedRecurrence(0).calculateOutput(zeros, tensor(ops, {1, 2}, {2, 5}), h0).output, {1, 2}, {3, 3}, "sigmoid gate");
    expect_throw<std::invalid_argument>([&] { given.calculateOutput(gate, token, h0); }, "gate and input of different shapes");
    expect_throw<std::invalid_argument>([&] { given.calculateOutput(gate, in, in); }, "an initial state of the wrong size");
    expect_throw<std::invalid_argument>([&] { given.calculateGrads(gate, in, h0, out.output, h0, nullptr, true, true, true); }, "a gradient of the wrong size");
    ops.release(h0);
    expect_throw<std::runtime_error>([&] { given.calculateOutput(gate, in, h0); }, "a released state");
}

int main() {
    HipTensorOperations ops(0);
    {
        auto gc = ops.garbageCollector();
        layer_norm(ops);
        dropout(ops);
        recurrence(ops);
    }
    std::printf("%d checks, %d failed\n", g_checks, g_failed);
    return g_failed == 0 ? 0 : 1;
}
