// The gated recurrence through the C++ host mirror (include/kten_hip.hpp) without the tensors that its backward pass does not
// read, on values worked out by hand, all of them exact in fp32. Exit status 0 means every check held.
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

template <class F>
static void expect_refused(F&& f, const char* what) {
    bool thrown = false;
    try { f(); } catch (const std::invalid_argument&) { thrown = true; }
    expect(thrown, what);
}

static Raw tensor(HipTensorOperations& ops, const Shape& shape, std::initializer_list<float> values) {
    std::vector<float> v(values);
    return ops.createRaw(shape, [&](int i) { return v[static_cast<size_t>(i)]; });
}

int main() {
    HipTensorOperations ops;
    {
        // one channel of three steps: h = 0.5 * 8 + 1, 2 * 5 + 1, 0.25 * 11 + 1 = 5, 11, 3.75
        Raw gate = tensor(ops, {3, 1}, {0.5f, 2, 0.25f}), x = tensor(ops, {3, 1}, {1, 1, 1}), first = tensor(ops, {1}, {8}), go = tensor(ops, {3, 1}, {1, 1, 4});
        auto given = ops.gatedRecurrence(0, false);
        Raw out = given.calculateOutput(gate, x, first).output;
        expect_values(out, {3, 1}, {5, 11, 3.75f}, "states");
        // d = 4, 1 + 0.25 * 4 = 2, 1 + 2 * 2 = 5; gate: d times the state before; first state: 0.5 * 5
        auto grads = given.calculateGrads(gate, nullptr, first, out, go, nullptr, true, true, true);
        expect_values(grads.gradGate, {3, 1}, {40, 10, 44}, "gradient of a given gate without the input");
        expect_values(grads.gradIn, {3, 1}, {5, 2, 4}, "gradient of the input without the input");
        expect_values(grads.gradInitial, {1}, {2.5f}, "gradient of the first state without the input");
        grads = given.calculateGrads(gate, nullptr, nullptr, nullptr, go, nullptr, false, true, true);
        expect(!grads.gradGate, "no gradient that was not asked for");
        expect_values(grads.gradIn, {3, 1}, {5, 2, 4}, "gradient of the input alone");
        expect_values(grads.gradInitial, {1}, {2.5f}, "gradient of the first state alone");
        expect_refused([&] { given.calculateGrads(gate, nullptr, first, nullptr, go, nullptr, true, false, false); }, "the gate's gradient needs the output");
        expect_refused([&] { given.calculateOutput(gate, nullptr, first); }, "the states need the input");
        expect_refused([&] { given.step(gate, nullptr, first); }, "a step needs the input");
        auto sigmoid = ops.gatedRecurrence(0, true);
        expect_refused([&] { sigmoid.calculateGrads(gate, nullptr, first, out, go, nullptr, true, false, false); }, "a sigmoid gate's gradient needs the input");
        // logits of 0: a = b = 0.5; d = 4, 1 + 2 = 3, 1 + 1.5 = 2.5
        Raw zero = tensor(ops, {3, 1}, {0, 0, 0});
        grads = sigmoid.calculateGrads(zero, nullptr, nullptr, nullptr, go, nullptr, false, true, true);
        expect_values(grads.gradIn, {3, 1}, {1.25f, 1.5f, 2}, "sigmoid: gradient of the input alone");
        expect_values(grads.gradInitial, {1}, {1.25f}, "sigmoid: gradient of the first state alone");
    }
    std::printf("%d checks, %d failed\n", g_checks, g_failed);
    return g_failed == 0 ? 0 : 1;
}
