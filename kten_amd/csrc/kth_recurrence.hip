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
#include <climits>

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

// exp(-|g|) to 2 u (u = 2^-24), results below the normal range included: 2^(f + n) with f the fraction of |g| log2(e), by the
// hardware's exponential. The product with log2(e) is made in two: by the float next to it, and by what that leaves of it.
__device__ __forceinline__ float exp_minus_abs(float g) {
    float x = -fabsf(g);
    x = x < -110.0f ? -110.0f : x;                           // (gives 0: below half the smallest float; NaN stays NaN)
    const float n = rintf(x * 1.44269504f);
    const float f = fmaf(x, 1.92596299e-8f, fmaf(x, 1.44269504f, -n));
    return ldexpf(__builtin_amdgcn_exp2f(f), static_cast<int>(n));
}

// 1 / d for d in [1, 2]: the hardware's reciprocal and a Newton step.
__device__ __forceinline__ float reciprocal(float d) {
    const float r = __builtin_amdgcn_rcpf(d);
    return fmaf(fmaf(-d, r, 1.0f), r, r);
}

// A gate as the scans keep it in one register. GIVEN: the gate. SIGMOID: s, the smaller of a and b = 1 - a, with the sign of
// the logit, which says which of the two it is: a = 1 - s or 0 + s, b = 0 + s or 1 - s. Both come out to a few u of
// themselves (b as a difference from a rounded a would be lost near a = 1, and with it the decay over many steps).
template <bool SIGMOID>
__device__ __forceinline__ float pack_gate(float g) {
    if (!SIGMOID) return g;
    const float e = exp_minus_abs(g);
    return copysignf(e * reciprocal(1.0f + e), g);
}
template <bool SIGMOID>
__device__ __forceinline__ double gate_a(float v) {
    if (!SIGMOID) return static_cast<double>(v);
    const int one = ~(__float_as_int(v) >> 31) & 0x3ff00000;             // the high word of 1.0 or 0.0
    return __hiloint2double(one, 0) - static_cast<double>(v);
}
__device__ __forceinline__ float sigmoid_b(float v) {
    return __int_as_float((__float_as_int(v) >> 31) & 0x3f800000) + v;   // 1 or 0
}

// A thread per channel walks its steps: for one step a launch and little else ([64,1,1024] 2.7 us), for many channels bound by
// memory ([100000,20,24] forward 127 us, 4.5 TB/s).
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
                const float v = pack_gate<SIGMOID>(g[k]);
                h = fma(gate_a<SIGMOID>(v), h, static_cast<double>(SIGMOID ? sigmoid_b(v) * x[k] : x[k]));
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
    for (uint32_t left = sh.steps; left > 0; left -= min(left, static_cast<uint32_t>(kAhead))) {
        // steps left - 1, left - 2, ...; what only the gate's gradient needs (without it out and in need not be given) too
        float v[kAhead], g[kAhead], before[kAhead], x[kAhead];
        const uint64_t top = first + static_cast<uint64_t>(left - 1) * sh.inner;
#pragma unroll
        for (int k = 0; k < kAhead; k++) {
            const uint64_t at = top - static_cast<uint64_t>(k) * sh.inner;
            if (static_cast<uint32_t>(k) < left) {
                v[k] = gate[at]; g[k] = grad_out[at];
                if (grad_gate) {
                    before[k] = static_cast<uint32_t>(k) + 1 < left ? out[at - sh.inner] : h0;
                    if (SIGMOID) x[k] = in[at];
                }
            }
        }
#pragma unroll
        for (int k = 0; k < kAhead; k++) {
            const uint64_t at = top - static_cast<uint64_t>(k) * sh.inner;
            if (static_cast<uint32_t>(k) < left) {
                const float p = pack_gate<SIGMOID>(v[k]);
                const double a = gate_a<SIGMOID>(p), b = SIGMOID ? static_cast<double>(sigmoid_b(p)) : 1.0;
                const double d = static_cast<double>(g[k]) + carry;
                if (grad_gate)
                    grad_gate[at] = static_cast<float>(SIGMOID ? d * (static_cast<double>(before[k]) - static_cast<double>(x[k])) * (a * b)
                                                               : d * static_cast<double>(before[k]));
                if (grad_in) grad_in[at] = static_cast<float>(d * b);
                carry = a * d;
            }
        }
    }
    if (grad_initial) grad_initial[ch] = static_cast<float>(carry);
}

// ---------------------------------------------------------------- long sequences: tiles of steps

// The scan is cut into tiles that pass a state on. A workgroup takes one tile: 64 adjacent channels of one outer index
// (a lane per channel) and tw x L successive steps, L to a wave, which the wave keeps in registers, so that every operand
// is read once. A step is the map K -> a K + u of the state, so a run of steps is one pair (A, H): waves exchange theirs
// through LDS, tiles through memory.
//
// Tiles are drawn from a counter, earliest steps of all channels first. A tile only waits for tiles of earlier steps, which
// are drawn before it and thus run already or have ended: every wait ends. Tile p reads the pairs of the tiles since the
// last multiple of kSuper before it, and the state that the tile before that multiple published: at most kSuper - 1 pairs
// and one state, always composed in the same order, so the bits do not depend on who came first.
//
// A published value is one 64-bit word that carries its own sign of life, a double whose last kTagBits bits hold the
// launch's number: no fence, no flag, no clearing between launches (the words are cleared when the number starts again).
// What the doubles lose is 2^-41 of themselves a tile.
//
// [8,2048,1024] sigmoid forward 48 us (4.2 TB/s), [1,65536,512] given forward 89 (4.5), backward 143 (4.7), [5,1999,1001] sigmoid
// backward 69 (3.5; odd rows share cache lines with their neighbours). What bounds it is a tile's life, loads, the wait for
// the state, stores, with two tiles in a compute unit's registers: the vector ALU is 40 % busy, and without the hand-over (its results
// would be wrong) the same four take 46, 79, 122 and 68. Longer runs of steps spill, shorter ones have more tiles to hand over.
constexpr int kTagBits = 12;
constexpr uint32_t kTags = (1u << kTagBits) - 1;     // tag 0: never published
constexpr uint32_t kSuper = 16;

__device__ __forceinline__ void publish(uint64_t* word, double v, uint32_t tag) {
    const uint64_t bits = static_cast<uint64_t>(__double_as_longlong(v)) + (1ull << (kTagBits - 1));
    __hip_atomic_store(word, (bits & ~static_cast<uint64_t>(kTags)) | tag, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// Waits for a word of an earlier tile. Should it not come within `most` looks (the default takes seconds; a tile takes
// microseconds) the wave goes on with NaN and leaves a mark for the host, which reports it at its next wait for the stream. Who
// finds the mark while waiting, a look at the host's memory every thousand, gives up too: no wait is endless, nor is one given
// up after another in a chain of tiles.
struct Wait {
    uint32_t tag, most;
    int*     lost;                   // the host's word for a wait that was given up
};
__device__ __forceinline__ double await(const uint64_t* word, const Wait& wait) {
    uint64_t bits = wait.most != 0 ? __hip_atomic_load(word, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0;
    for (uint32_t looks = 1; (bits & kTags) != wait.tag; looks++) {
        if (looks >= wait.most || (looks % 1024 == 0 && __hip_atomic_load(wait.lost, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM) != 0)) {
            __hip_atomic_store(wait.lost, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
            return __builtin_nan("");
        }
        __builtin_amdgcn_s_sleep(1);
        bits = __hip_atomic_load(word, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    return __longlong_as_double(static_cast<long long>(bits & ~static_cast<uint64_t>(kTags)));
}

// The map K -> A K + H of a run of steps, A the product of its gates. A product of gates none of which is zero does not become
// zero: below the normal range it is kLeast, of which an infinite state stays infinite. Where gates are given, and
// may be above one, it stays kLeast whatever follows, and of a finite state it leaves nothing.
struct Pair { double A, H; };
constexpr double kLeast = 2.2250738585072014e-308;       // 2^-1022

// The state after the run.
template <bool SIGMOID>
__device__ __forceinline__ double advance(const Pair& p, double state) {
    if (SIGMOID) return state == 0.0 ? p.H : fma(p.A, state, p.H);
    const bool lost = fabs(p.A) <= kLeast;
    return fma(lost && fabs(state) < INFINITY ? 0.0 : p.A, state, p.H);
}
template <bool SIGMOID>
__device__ __forceinline__ Pair after(const Pair& later, const Pair& earlier) {
    double A = later.A * earlier.A;
    const bool lost = SIGMOID ? fabs(A) < kLeast : fabs(A) < kLeast || fabs(later.A) <= kLeast || fabs(earlier.A) <= kLeast;
    if (lost && later.A != 0.0 && earlier.A != 0.0 && (SIGMOID || fabs(A) < INFINITY)) A = copysign(kLeast, A);
    return Pair{A, advance<SIGMOID>(later, earlier.H)};
}
// The state after `count` runs, their pairs `apart` from one another; and such runs as one. With given gates the chain is first
// made without the looks that `advance` and `after` take on the way at what is lost, infinite or NaN: an infinity on the way shows
// in the end, and the least magnitude of the products tells the rest (together 2 % of [1,65536,512]).
template <bool SIGMOID>
__device__ __forceinline__ double through(const Pair* pairs, uint32_t apart, uint32_t count, double state) {
    if (!SIGMOID) {
        double s = state;
        for (uint32_t i = 0; i < count; i++) {
            const Pair p = pairs[i * apart];
            s = fma(fabs(p.A) <= kLeast ? 0.0 : p.A, s, p.H);
        }
        if (!__any(!(fabs(s) < INFINITY))) return s;
    }
    for (uint32_t i = 0; i < count; i++) state = advance<SIGMOID>(pairs[i * apart], state);
    return state;
}
template <bool SIGMOID>
__device__ __forceinline__ Pair together(const Pair* pairs, uint32_t apart, uint32_t count) {
    Pair total = pairs[0];
    if (!SIGMOID) {
        double least = fabs(total.A);
        for (uint32_t i = 1; i < count; i++) {
            const Pair p = pairs[i * apart];
            total = Pair{p.A * total.A, fma(p.A, total.H, p.H)};
            least = fmin(least, fmin(fabs(p.A), fabs(total.A)));
        }
        if (!__any(!(least > kLeast && fabs(total.H) < INFINITY))) return total;
        total = pairs[0];
    }
    for (uint32_t i = 1; i < count; i++) total = after<SIGMOID>(pairs[i * apart], total);
    return total;
}
// A run after which the state is known to be `end`, whatever came before; `state` is what did (an infinite one stays infinite or
// becomes NaN).
__device__ __forceinline__ Pair known(double state, double end) { return Pair{copysign(1.0, state) * copysign(kLeast, end), end}; }

// The product of a run's gates, one by one. Whether a gate was zero is told by `abs` or `bits`, an instruction a step without
// a branch (a look at the gates where A is that small makes the compiler keep twice the registers: 48 to 78 us for
// [8,2048,1024]): -0 is a closed gate where gates are packed logits, the smallest of all integers.
//
// Runs are composed where they are tame: every product of sigmoids is, and one of given gates that is finite and (looked at every
// fourth step) never more than 2^kRise above where it has been. Others, whose products may leave a double's range where the
// states do not, or come back into it where the states are lost, are walked step by step once the state before them is known.
// That costs a tile its independence: where every run rises by 2^18, [8,2048,1024] forward takes 52 us instead of 46, [1,65536,512]
// 960 instead of 90, [1,66000,2] 864 instead of 14 (a thread a channel: 4419). Decays never rise, and gates of a normal
// distribution or close to one hardly ever so far: they take the time of decays. A bound of 2^48 would still keep the products
// of two tiles in range, but gates that halve and double a state by turns would then bring back what is lost on the way.
constexpr int kRise = 16;
template <bool SIGMOID>
struct Product {
    double A = 1.0;
    float  abs = INFINITY;
    int    bits = INT_MAX, low = 1023, rise = 0;         // exponents as a double's bits have them
    __device__ __forceinline__ void look() {
        const int now = __double2hiint(A) >> 20 & 0x7ff;
        low = min(low, now);
        rise = max(rise, now - low);
    }
    __device__ __forceinline__ void take(double a, float v, int k) {       // v: the gate as it is packed; k: the step's number in the run
        A *= a;
        if (SIGMOID) bits = min(bits, __float_as_int(v)); else abs = fminf(abs, fabsf(v));
        if (!SIGMOID && k % 4 == 3) look();
    }
    __device__ __forceinline__ double gates() const {
        return fabs(A) < kLeast && (SIGMOID ? bits != INT_MIN : abs != 0.0f) ? copysign(kLeast, A) : A;
    }
    __device__ __forceinline__ bool tame() {
        if (SIGMOID) return true;
        look();
        return rise <= kRise;                            // (an infinity or NaN is far above)
    }
};

struct TilePlan {
    uint32_t steps, inner;
    uint32_t col_blocks, groups;     // workgroups across one outer index; across all channels (outer x col_blocks)
    uint32_t tiles;                  // along the steps
    uint32_t tw;                     // waves of a workgroup, along the steps
    uint32_t padded;                 // groups x 64: channels with their padding
    Wait     wait;                   // with this launch's tag
    uint32_t* tickets;               // this launch's counter
    uint64_t* pairs;                 // [tiles][padded][2]
    uint64_t* states;                // [tiles / kSuper][padded]
    FastDiv  group_div, col_div;
};

// Keeps the instructions of few steps at a time in flight: the f64 values of all of them would not fit a lane's registers.
#define KTH_STEPS_APART(k) do { if ((k) % 4 == 3) __builtin_amdgcn_sched_barrier(0); } while (0)

// Where a workgroup and its waves stand.
struct TilePlace {
    uint32_t tile, group, lane, twi;
    uint32_t channel;                // in its outer index
    uint32_t slot;                   // among the padded channels
    uint64_t base;                   // of the outer index's first step
    uint32_t first_state;            // channel's place among all channels (outer x inner)
    bool     valid;
};

__device__ __forceinline__ TilePlace place_tile(const TilePlan& pl, uint32_t* lds_ticket, uint32_t* wild) {
    TilePlace w;
    if (threadIdx.x == 0) *wild = 0;
    if (threadIdx.x == 0) *lds_ticket = pl.tiles > 1 ? atomicAdd(pl.tickets, 1u) : blockIdx.x;
    __syncthreads();
    const uint32_t ticket = __builtin_amdgcn_readfirstlane(*lds_ticket);
    w.twi = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    w.lane = threadIdx.x & 63;
    w.tile = divide(ticket, pl.group_div);
    w.group = ticket - w.tile * pl.groups;
    const uint32_t o = divide(w.group, pl.col_div);
    const uint32_t c = (w.group - o * pl.col_blocks) * 64 + w.lane;
    w.valid = c < pl.inner;
    w.channel = w.valid ? c : pl.inner - 1;          // (a padding lane reads the last channel and writes nothing)
    w.slot = w.group * 64 + w.lane;
    w.base = static_cast<uint64_t>(o) * pl.steps * pl.inner;
    w.first_state = o * pl.inner + w.channel;
    return w;
}

// The state before this tile, from the pairs of its waves' steps and whether they are `tame`; `initial` is the state before
// the first tile. lds: pairs of the waves, [tw][64], then of the tiles before, as many again; wild: 0 before the last
// barrier. in_turn: a run of this tile is to be walked, so all are, one wave after another.
template <bool SIGMOID>
__device__ __forceinline__ double state_before_tile(const TilePlan& pl, const TilePlace& w, const Pair& mine, bool tame, double initial, Pair* lds, uint32_t* wild,
                                                    bool& in_turn) {
    Pair* before = lds + pl.tw * 64;
    lds[w.twi * 64 + w.lane] = mine;
    if (!SIGMOID && !tame) *wild = 1;
    __syncthreads();
    in_turn = !SIGMOID && __builtin_amdgcn_readfirstlane(*wild) != 0;
    double state = initial;
    const uint32_t super = w.tile / kSuper, first = super * kSuper, many = w.tile - first;
    if (pl.tiles > 1) {
        if (w.twi == pl.tw - 1 && w.tile + 1 < pl.tiles && many + 1 < kSuper && !in_turn) {
            Pair total = together<SIGMOID>(lds + w.lane, 64, pl.tw);
            if (w.tile == 0) total = Pair{0.0, advance<SIGMOID>(total, initial)};     // nobody else reads `initial`
            uint64_t* word = pl.pairs + (static_cast<uint64_t>(w.tile) * pl.padded + w.slot) * 2;
            publish(word, total.A, pl.wait.tag);
            publish(word + 1, total.H, pl.wait.tag);
        }
        if (w.tile > 0) {
            // the waves along the steps share out the tiles before
            const uint32_t per = (many + pl.tw - 1) / pl.tw;
            const uint32_t from = min(w.twi * per, many), to = min(from + per, many);
            Pair p{1.0, 0.0};
            for (uint32_t i = from; i < to; i++) {
                const uint64_t* word = pl.pairs + (static_cast<uint64_t>(first + i) * pl.padded + w.slot) * 2;
                const double a = await(word, pl.wait), h = await(word + 1, pl.wait);
                p = after<SIGMOID>(Pair{a, h}, p);
            }
            before[w.twi * 64 + w.lane] = p;
            state = super == 0 ? 0.0 : await(pl.states + static_cast<uint64_t>(super - 1) * pl.padded + w.slot, pl.wait);
            __syncthreads();
            state = through<SIGMOID>(before + w.lane, 64, pl.tw, state);
        }
    }
    return state;
}
// The state before this wave's first step from that before the tile, where the waves' pairs are composed.
template <bool SIGMOID>
__device__ __forceinline__ double state_before_wave(const TilePlan& pl, const TilePlace& w, double state, const Pair* lds) {
    if (w.twi == pl.tw - 1 && w.tile % kSuper + 1 == kSuper && w.tile + 1 < pl.tiles) {
        const double end = through<SIGMOID>(lds + w.lane, 64, pl.tw, state);
        publish(pl.states + static_cast<uint64_t>(w.tile / kSuper) * pl.padded + w.slot, end, pl.wait.tag);
    }
    return through<SIGMOID>(lds + w.lane, 64, w.twi, state);
}
// What the last wave of a tile whose waves took turns hands on.
__device__ __forceinline__ void hand_on_end(const TilePlan& pl, const TilePlace& w, double before_tile, double end) {
    if (w.twi != pl.tw - 1 || w.tile + 1 >= pl.tiles) return;
    if (w.tile % kSuper + 1 == kSuper) {
        publish(pl.states + static_cast<uint64_t>(w.tile / kSuper) * pl.padded + w.slot, end, pl.wait.tag);
    } else {
        uint64_t* word = pl.pairs + (static_cast<uint64_t>(w.tile) * pl.padded + w.slot) * 2;
        const Pair total = known(before_tile, end);
        publish(word, total.A, pl.wait.tag);
        publish(word + 1, total.H, pl.wait.tag);
    }
}

constexpr uint32_t kTileThreads = 512;

// LINES: rows are multiples of 128 bytes, so no two workgroups read the same cache line and it need not be kept
// ([8,2048,1024] 53 to 50 us; with odd rows the lines' second readers would wait: [5,1999,1001] backward 70 to 75 us).
template <bool LINES>
__device__ __forceinline__ float read_once(const float* p) { return LINES ? __builtin_nontemporal_load(p) : *p; }

template <bool SIGMOID, bool LINES, int L>
__global__ __launch_bounds__(kTileThreads, 4) void recurrence_forward_tiles_kernel(const float* __restrict__ gate, const float* __restrict__ in, const float* initial,
                                                                                   float* __restrict__ out, float* final_state, TilePlan pl) {
    extern __shared__ Pair lds[];
    __shared__ uint32_t lds_ticket, wild;
    const TilePlace w = place_tile(pl, &lds_ticket, &wild);
    if (w.tile >= pl.tiles) return;
    const uint32_t t0 = (w.tile * pl.tw + w.twi) * L;
    const uint64_t row0 = w.base + static_cast<uint64_t>(t0) * pl.inner;
    float v[L], u[L];
#pragma unroll
    for (int k = 0; k < L; k++) {
        const uint64_t row = w.base + static_cast<uint64_t>(min(t0 + k, pl.steps - 1)) * pl.inner;
        v[k] = read_once<LINES>(gate + row + w.channel);
        u[k] = read_once<LINES>(in + row + w.channel);
    }
#pragma unroll
    for (int k = 0; k < L; k++)                              // a step behind the last one leaves the state as it is
        if (t0 + k >= pl.steps) { v[k] = SIGMOID ? INFINITY : 1.0f; u[k] = 0.0f; }
    double start = w.tile == 0 && initial ? static_cast<double>(initial[w.first_state]) : 0.0;
    // final_state may be the same store: every wave's load has arrived before the barrier behind which another may write it
    asm volatile("" : "+v"(start));
    double H = 0.0;
    Product<SIGMOID> product;
#pragma unroll
    for (int k = 0; k < L; k++) {
        if (SIGMOID) {
            v[k] = pack_gate<SIGMOID>(v[k]);
            u[k] = sigmoid_b(v[k]) * u[k];
        }
        const double a = gate_a<SIGMOID>(v[k]);
        H = fma(a, H, static_cast<double>(u[k]));
        product.take(a, v[k], k);
        KTH_STEPS_APART(k);
    }
#pragma unroll
    for (int k = 0; k < L; k++) { forget(v[k]); forget(u[k]); }
    const Pair mine{product.gates(), H};
    bool in_turn;
    double h = state_before_tile<SIGMOID>(pl, w, mine, product.tame(), start, lds, &wild, in_turn);
    if (in_turn) {
        Pair* slot = lds + w.lane;                           // wave i's of this channel: slot[i * 64]; H: the state behind it
        double end = h;
        const double before_tile = h;
        for (uint32_t i = 0; i < pl.tw; i++) {
            if (i == w.twi) {
                if (i > 0) h = slot[(i - 1) * 64].H;
                end = h;
#pragma unroll
                for (int k = 0; k < L; k++) { forget(v[k]); forget(u[k]); }
#pragma unroll
                for (int k = 0; k < L; k++) {
                    end = fma(gate_a<SIGMOID>(v[k]), end, static_cast<double>(u[k]));
                    KTH_STEPS_APART(k);
                }
                slot[i * 64].H = end;
            }
            __syncthreads();
        }
        hand_on_end(pl, w, before_tile, end);
    } else {
        h = state_before_wave<SIGMOID>(pl, w, h, lds);
    }
#pragma unroll
    for (int k = 0; k < L; k++) {
        if (t0 + k < pl.steps) {
            h = fma(gate_a<SIGMOID>(v[k]), h, static_cast<double>(u[k]));
            if (w.valid) (out + row0 + static_cast<uint64_t>(k) * pl.inner)[w.channel] = static_cast<float>(h);
        }
        KTH_STEPS_APART(k);
    }
    if (final_state && w.valid && t0 < pl.steps && t0 + L >= pl.steps) final_state[w.first_state] = static_cast<float>(h);
}

// The gradient of the state runs from the last step to the first: K_t = a_t (grad_out_t + K_{t+1}), K behind the last step
// being grad_final, d_t = grad_out_t + K_{t+1}; K_0 is grad_initial. Tiles, waves and steps are counted from the end.
template <bool SIGMOID, bool LINES, int L>
__global__ __launch_bounds__(kTileThreads, 4) void recurrence_backward_tiles_kernel(const float* __restrict__ gate, const float* __restrict__ in,
                                                                                    const float* __restrict__ initial, const float* __restrict__ out,
                                                                                    const float* __restrict__ grad_out, const float* __restrict__ grad_final,
                                                                                    float* __restrict__ grad_gate, float* __restrict__ grad_in,
                                                                                    float* __restrict__ grad_initial, TilePlan pl) {
    extern __shared__ Pair lds[];
    __shared__ uint32_t lds_ticket, wild;
    const TilePlace w = place_tile(pl, &lds_ticket, &wild);
    if (w.tile >= pl.tiles) return;
    const uint32_t q0 = (w.tile * pl.tw + w.twi) * L;        // step t = steps - 1 - (q0 + k)
    const uint64_t last_row = w.base + static_cast<uint64_t>(pl.steps - 1) * pl.inner;
    float v[L], g[L];
#pragma unroll
    for (int k = 0; k < L; k++) {
        const uint64_t row = last_row - static_cast<uint64_t>(min(q0 + k, pl.steps - 1)) * pl.inner;
        v[k] = read_once<LINES>(gate + row + w.channel);
        g[k] = read_once<LINES>(grad_out + row + w.channel);
    }
#pragma unroll
    for (int k = 0; k < L; k++)
        if (q0 + k >= pl.steps) { v[k] = SIGMOID ? INFINITY : 1.0f; g[k] = 0.0f; }
    const double start = w.tile == 0 && grad_final ? static_cast<double>(grad_final[w.first_state]) : 0.0;
    double H = 0.0;
    Product<SIGMOID> product;
#pragma unroll
    for (int k = 0; k < L; k++) {
        if (SIGMOID) v[k] = pack_gate<SIGMOID>(v[k]);
        const double a = gate_a<SIGMOID>(v[k]);
        H = a * (static_cast<double>(g[k]) + H);
        product.take(a, v[k], k);
        KTH_STEPS_APART(k);
    }
#pragma unroll
    for (int k = 0; k < L; k++) { forget(v[k]); forget(g[k]); }
    // what only the gate's gradient needs arrives while the state does (without it out and in need not be given)
    float before[L], x[L];
    if (grad_gate) {
#pragma unroll
        for (int k = 0; k < L; k++) {
            const uint32_t q = min(q0 + k, pl.steps - 1);
            const uint64_t row = last_row - static_cast<uint64_t>(q) * pl.inner;
            before[k] = (out + (q + 1 < pl.steps ? row - pl.inner : row))[w.channel];
            if (SIGMOID) x[k] = read_once<LINES>(in + row + w.channel);
        }
        if (q0 < pl.steps && q0 + L >= pl.steps) {
            const float h0 = initial ? initial[w.first_state] : 0.0f;
#pragma unroll
            for (int k = 0; k < L; k++) if (q0 + k + 1 == pl.steps) before[k] = h0;
        }
    }
    const Pair mine{product.gates(), H};
    bool in_turn;
    double K = state_before_tile<SIGMOID>(pl, w, mine, product.tame(), start, lds, &wild, in_turn);
    if (in_turn) {
        Pair* slot = lds + w.lane;                           // wave i's of this channel: slot[i * 64]; H: the state behind it
        double end = K;
        const double before_tile = K;
        for (uint32_t i = 0; i < pl.tw; i++) {
            if (i == w.twi) {
                if (i > 0) K = slot[(i - 1) * 64].H;
                end = K;
#pragma unroll
                for (int k = 0; k < L; k++) { forget(v[k]); forget(g[k]); }
#pragma unroll
                for (int k = 0; k < L; k++) {
                    end = gate_a<SIGMOID>(v[k]) * (static_cast<double>(g[k]) + end);
                    KTH_STEPS_APART(k);
                }
                slot[i * 64].H = end;
            }
            __syncthreads();
        }
        hand_on_end(pl, w, before_tile, end);
    } else {
        K = state_before_wave<SIGMOID>(pl, w, K, lds);
    }
#pragma unroll
    for (int k = 0; k < L; k++) {
        if (q0 + k < pl.steps) {
            const uint64_t row = last_row - static_cast<uint64_t>(q0 + k) * pl.inner;
            const double a = gate_a<SIGMOID>(v[k]), b = SIGMOID ? static_cast<double>(sigmoid_b(v[k])) : 1.0;
            const double d = static_cast<double>(g[k]) + K;
            if (grad_gate) {
                const double r = SIGMOID ? d * (static_cast<double>(before[k]) - static_cast<double>(x[k])) * (a * b) : d * static_cast<double>(before[k]);
                if (w.valid) (grad_gate + row)[w.channel] = static_cast<float>(r);
            }
            if (grad_in && w.valid) (grad_in + row)[w.channel] = static_cast<float>(d * b);
            K = a * d;
        }
        KTH_STEPS_APART(k);
    }
    if (grad_initial && w.valid && q0 < pl.steps && q0 + L >= pl.steps) grad_initial[w.first_state] = static_cast<float>(K);
}

// ---------------------------------------------------------------- few channels side by side

// With few channels side by side (inner) a wave's lanes would each walk memory of their own. Here a workgroup
// takes a stretch of up to 4096 floats as memory has them, through LDS, and a thread kSub steps of one channel: thread
// (row, j, channel), j counting the kSub-step pieces of a row. Rows that fit are taken several at a time; longer ones are
// cut into tiles that hand a state on as above. A piece's place in LDS is padded by one float, so that the threads of a
// wave, a piece apart, do not meet in a bank. [100000,64,1] 38 us forward (2.0 TB/s) and 87 backward (1.8 TB/s), bound by the
// LDS and the barriers of the scan over the pieces.
constexpr uint32_t kNarrowThreads = 256, kSub = 16, kNarrowInner = 32;     // (inner is below kNarrowInner)
constexpr uint32_t kNarrowFloats = kNarrowThreads * (kSub + 1);

struct NarrowPlan {
    uint32_t outer, steps, inner;
    uint32_t rows;                   // outer indices of a workgroup (1 if tiles > 1)
    uint32_t pieces;                 // of kSub steps, of a row in a workgroup
    uint32_t tile_steps, tiles;
    uint32_t channels;               // outer x inner
    Wait     wait;                   // with this launch's tag
    uint32_t* tickets;               // this launch's counter
    uint64_t* pairs;                 // [tiles][channels][2]
    uint64_t* states;                // [tiles / kSuper][channels]
    FastDiv  inner_div, row_div, outer_div, piece_div;     // row_div divides by the floats of a row of this workgroup
};

struct NarrowPlace {
    uint32_t tile, o0, rows;         // first outer index and how many
    uint32_t q0, count;              // first step (counted in the scan's direction) and how many
    uint32_t r, j, c;                // this thread's
    bool     works;
    uint32_t channel;                // of all, this thread's
};

__device__ __forceinline__ bool place_narrow(const NarrowPlan& pl, uint32_t* lds_ticket, uint32_t* wild, NarrowPlace& w) {
    uint32_t ticket = blockIdx.x;
    if (threadIdx.x == 0) *wild = 0;
    if (pl.tiles > 1) {
        if (threadIdx.x == 0) *lds_ticket = atomicAdd(pl.tickets, 1u);
        __syncthreads();
        ticket = __builtin_amdgcn_readfirstlane(*lds_ticket);
        if (ticket >= pl.tiles * pl.outer) return false;
        w.tile = divide(ticket, pl.outer_div);
        w.o0 = ticket - w.tile * pl.outer;
        w.rows = 1;
    } else {
        w.tile = 0;
        w.o0 = ticket * pl.rows;
        w.rows = min(pl.rows, pl.outer - w.o0);
    }
    w.q0 = w.tile * pl.tile_steps;
    w.count = min(pl.tile_steps, pl.steps - w.q0);
    const uint32_t piece = divide(threadIdx.x, pl.inner_div);          // row and j together
    w.c = threadIdx.x - piece * pl.inner;
    w.r = divide(piece, pl.piece_div);
    w.j = piece - w.r * pl.pieces;
    w.works = w.r < w.rows;
    w.channel = (w.o0 + w.r) * pl.inner + w.c;
    return true;
}

// Where the float e of the workgroup's stretch lies in memory and in LDS. REVERSE: steps are counted from the last one.
template <bool REVERSE>
__device__ __forceinline__ uint64_t narrow_index(const NarrowPlan& pl, const NarrowPlace& w, uint32_t e, uint32_t& place) {
    const uint32_t r = w.rows > 1 ? divide(e, pl.row_div) : 0;
    const uint32_t in_row = e - r * (w.count * pl.inner);
    const uint32_t t = divide(in_row, pl.inner_div);
    const uint32_t c = in_row - t * pl.inner;
    const uint32_t s = REVERSE ? w.count - 1 - t : t;                  // in the scan's order
    place = (r * pl.pieces + s / kSub) * (kSub * pl.inner + 1) + (s % kSub) * pl.inner + c;
    const uint32_t first = REVERSE ? pl.steps - w.q0 - w.count : w.q0;
    return (static_cast<uint64_t>(w.o0 + r) * pl.steps + first + t) * pl.inner + c;
}

// The state before this thread's piece from the piece's pair and whether its steps are `tame`. `initial` is its channel's, read by
// the first piece of the first tile. pair: kNarrowThreads pairs of LDS; handed: kSuper x inner more, and inner states; wild: 0
// before the last barrier. in_turn: a piece of this tile is to be walked, so all are, one after another, and what is
// returned is the state before the tile.
template <bool SIGMOID>
__device__ __forceinline__ double narrow_state_before(const NarrowPlan& pl, const NarrowPlace& w, const Pair& run, bool tame, double initial,
                                                      Pair* pair, Pair* handed, double* carried, uint32_t* wild, bool& in_turn) {
    Pair mine = w.works ? run : Pair{1.0, 0.0};
    if (w.works && w.tile == 0 && w.j == 0) mine = Pair{0.0, advance<SIGMOID>(run, initial)};   // nobody else reads `initial`
    for (uint32_t d = 1; d < pl.pieces; d <<= 1) {                     // pieces up to and with this one
        pair[threadIdx.x] = mine;
        __syncthreads();
        if (w.works && w.j >= d) mine = after<SIGMOID>(mine, pair[threadIdx.x - d * pl.inner]);
        __syncthreads();
    }
    pair[threadIdx.x] = mine;
    if (!SIGMOID && w.works && (!tame || !(fabs(mine.A) < INFINITY))) *wild = 1;
    __syncthreads();
    in_turn = !SIGMOID && __builtin_amdgcn_readfirstlane(*wild) != 0;
    double state = 0.0;
    const uint32_t super = w.tile / kSuper, first = super * kSuper, many = w.tile - first;
    if (pl.tiles > 1) {
        const Pair* total = pair + (pl.pieces - 1) * pl.inner;        // (a tile that is cut short is the last: nobody reads its total)
        if (threadIdx.x < pl.inner && w.tile + 1 < pl.tiles && many + 1 < kSuper && !in_turn) {
            uint64_t* word = pl.pairs + (static_cast<uint64_t>(w.tile) * pl.channels + w.o0 * pl.inner + threadIdx.x) * 2;
            publish(word, total[threadIdx.x].A, pl.wait.tag);
            publish(word + 1, total[threadIdx.x].H, pl.wait.tag);
        }
        if (w.tile > 0) {
            for (uint32_t i = threadIdx.x; i < many * pl.inner; i += kNarrowThreads) {
                const uint32_t t = divide(i, pl.inner_div);
                const uint64_t* word = pl.pairs + (static_cast<uint64_t>(first + t) * pl.channels + w.o0 * pl.inner + (i - t * pl.inner)) * 2;
                const double a = await(word, pl.wait), h = await(word + 1, pl.wait);
                handed[i] = Pair{a, h};
            }
            __syncthreads();
            if (threadIdx.x < pl.inner) {
                const uint32_t channel = w.o0 * pl.inner + threadIdx.x;
                double s = super == 0 ? 0.0 : await(pl.states + static_cast<uint64_t>(super - 1) * pl.channels + channel, pl.wait);
                s = through<SIGMOID>(handed + threadIdx.x, pl.inner, many, s);
                carried[threadIdx.x] = s;
                if (many + 1 == kSuper && w.tile + 1 < pl.tiles && !in_turn)
                    publish(pl.states + static_cast<uint64_t>(super) * pl.channels + channel, advance<SIGMOID>(total[threadIdx.x], s), pl.wait.tag);
            }
            __syncthreads();
            state = carried[w.c];
        }
    }
    if (in_turn) return w.tile == 0 ? initial : state;
    if (w.tile == 0 && w.j == 0) return initial;
    if (w.j == 0) return state;
    return advance<SIGMOID>(pair[threadIdx.x - pl.inner], state);
}
// What a tile whose pieces took turns hands on; `before_tile` is that of thread i's channel i.
__device__ __forceinline__ void narrow_hand_on_end(const NarrowPlan& pl, const NarrowPlace& w, double before_tile, const Pair* pair) {
    if (threadIdx.x >= pl.inner || w.tile + 1 >= pl.tiles) return;
    const uint32_t channel = w.o0 * pl.inner + threadIdx.x;
    const double end = pair[(pl.pieces - 1) * pl.inner + threadIdx.x].H;
    if (w.tile % kSuper + 1 == kSuper) {
        publish(pl.states + static_cast<uint64_t>(w.tile / kSuper) * pl.channels + channel, end, pl.wait.tag);
    } else {
        uint64_t* word = pl.pairs + (static_cast<uint64_t>(w.tile) * pl.channels + channel) * 2;
        const Pair total = known(before_tile, end);
        publish(word, total.A, pl.wait.tag);
        publish(word + 1, total.H, pl.wait.tag);
    }
}

// LDS of both kernels: two stretches of floats, the pairs, what earlier tiles handed on.
struct NarrowShared {
    float  a[kNarrowFloats], b[kNarrowFloats];
    Pair   pair[kNarrowThreads];
    Pair   handed[kSuper * kNarrowInner];
    double carried[kNarrowInner];
    uint32_t ticket, wild;
};

template <bool SIGMOID>
__global__ __launch_bounds__(kNarrowThreads) void recurrence_forward_narrow_kernel(const float* __restrict__ gate, const float* __restrict__ in, const float* initial,
                                                                                   float* __restrict__ out, float* final_state, NarrowPlan pl) {
    __shared__ NarrowShared sh;
    NarrowPlace w;
    if (!place_narrow(pl, &sh.ticket, &sh.wild, w)) return;
    const uint32_t floats = w.rows * w.count * pl.inner;
#pragma unroll 8
    for (uint32_t e = threadIdx.x; e < floats; e += kNarrowThreads) {
        uint32_t place;
        const uint64_t at = narrow_index<false>(pl, w, e, place);
        sh.a[place] = gate[at];
        sh.b[place] = in[at];
    }
    const double start = w.works && w.tile == 0 && w.j == 0 && initial ? static_cast<double>(initial[w.channel]) : 0.0;
    __syncthreads();
    const uint32_t base = (w.r * pl.pieces + w.j) * (kSub * pl.inner + 1) + w.c;
    const uint32_t count = w.works && w.j * kSub < w.count ? min(kSub, w.count - w.j * kSub) : 0;
    double H = 0.0;
    Product<SIGMOID> product;
    for (uint32_t k = 0; k < count; k++) {
        const uint32_t i = base + k * pl.inner;
        const float v = pack_gate<SIGMOID>(sh.a[i]);
        const float u = SIGMOID ? sigmoid_b(v) * sh.b[i] : sh.b[i];
        if (SIGMOID) { sh.a[i] = v; sh.b[i] = u; }
        const double a = gate_a<SIGMOID>(v);
        H = fma(a, H, static_cast<double>(u));
        product.take(a, v, k);
    }
    const Pair mine{product.gates(), H};
    bool in_turn;
    double h = narrow_state_before<SIGMOID>(pl, w, mine, product.tame(), start, sh.pair, sh.handed, sh.carried, &sh.wild, in_turn);
    if (in_turn) {
        const double before_tile = h;
        float v[kSub], u[kSub];
#pragma unroll
        for (uint32_t k = 0; k < kSub; k++) if (k < count) { v[k] = sh.a[base + k * pl.inner]; u[k] = sh.b[base + k * pl.inner]; }
        for (uint32_t j = 0; j < pl.pieces; j++) {
            if (w.works && w.j == j) {
                if (j > 0) h = sh.pair[threadIdx.x - pl.inner].H;
                double end = h;
#pragma unroll
                for (uint32_t k = 0; k < kSub; k++) if (k < count) end = fma(gate_a<SIGMOID>(v[k]), end, static_cast<double>(u[k]));
                sh.pair[threadIdx.x].H = end;
            }
            __syncthreads();
        }
        narrow_hand_on_end(pl, w, before_tile, sh.pair);
    }
    for (uint32_t k = 0; k < count; k++) {
        const uint32_t i = base + k * pl.inner;
        h = fma(gate_a<SIGMOID>(sh.a[i]), h, static_cast<double>(sh.b[i]));
        sh.b[i] = static_cast<float>(h);
    }
    if (final_state && count > 0 && w.q0 + w.j * kSub + count == pl.steps) final_state[w.channel] = static_cast<float>(h);
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < floats; e += kNarrowThreads) {
        uint32_t place;
        const uint64_t at = narrow_index<false>(pl, w, e, place);
        out[at] = sh.b[place];
    }
}

template <bool SIGMOID>
__global__ __launch_bounds__(kNarrowThreads) void recurrence_backward_narrow_kernel(const float* __restrict__ gate, const float* __restrict__ in,
                                                                                    const float* __restrict__ initial, const float* __restrict__ out,
                                                                                    const float* __restrict__ grad_out, const float* __restrict__ grad_final,
                                                                                    float* __restrict__ grad_gate, float* __restrict__ grad_in,
                                                                                    float* __restrict__ grad_initial, NarrowPlan pl) {
    __shared__ NarrowShared sh;
    NarrowPlace w;
    if (!place_narrow(pl, &sh.ticket, &sh.wild, w)) return;
    const uint32_t floats = w.rows * w.count * pl.inner;
#pragma unroll 8
    for (uint32_t e = threadIdx.x; e < floats; e += kNarrowThreads) {
        uint32_t place;
        const uint64_t at = narrow_index<true>(pl, w, e, place);
        sh.a[place] = gate[at];
        sh.b[place] = grad_out[at];
    }
    const double start = w.works && w.tile == 0 && w.j == 0 && grad_final ? static_cast<double>(grad_final[w.channel]) : 0.0;
    __syncthreads();
    const uint32_t base = (w.r * pl.pieces + w.j) * (kSub * pl.inner + 1) + w.c;
    const uint32_t count = w.works && w.j * kSub < w.count ? min(kSub, w.count - w.j * kSub) : 0;
    double H = 0.0;
    Product<SIGMOID> product;
    float v[kSub], g[kSub];
#pragma unroll
    for (uint32_t k = 0; k < kSub; k++) {
        if (k < count) {
            const uint32_t i = base + k * pl.inner;
            v[k] = pack_gate<SIGMOID>(sh.a[i]);
            g[k] = sh.b[i];
            const double a = gate_a<SIGMOID>(v[k]);
            H = a * (static_cast<double>(g[k]) + H);
            product.take(a, v[k], k);
        }
    }
    const Pair mine{product.gates(), H};
    bool in_turn;
    double K = narrow_state_before<SIGMOID>(pl, w, mine, product.tame(), start, sh.pair, sh.handed, sh.carried, &sh.wild, in_turn);
    if (in_turn) {
        const double before_tile = K;
        for (uint32_t j = 0; j < pl.pieces; j++) {
            if (w.works && w.j == j) {
                if (j > 0) K = sh.pair[threadIdx.x - pl.inner].H;
                double end = K;
#pragma unroll
                for (uint32_t k = 0; k < kSub; k++) if (k < count) end = gate_a<SIGMOID>(v[k]) * (static_cast<double>(g[k]) + end);
                sh.pair[threadIdx.x].H = end;
            }
            __syncthreads();
        }
        narrow_hand_on_end(pl, w, before_tile, sh.pair);
    }
    __syncthreads();                                                   // gate and grad_out are in registers: their LDS is free
    if (grad_gate) {                                                   // (without it out and in need not be given)
#pragma unroll 8
        for (uint32_t e = threadIdx.x; e < floats; e += kNarrowThreads) {
            uint32_t place;
            const uint64_t at = narrow_index<true>(pl, w, e, place);
            // the state before the step; before the first step of a row it is `initial`
            const uint32_t r = w.rows > 1 ? divide(e, pl.row_div) : 0;
            const uint32_t t = e - r * (w.count * pl.inner);
            const bool first = t < pl.inner && w.q0 + w.count == pl.steps;
            sh.a[place] = !first ? out[at - pl.inner] : initial ? initial[(w.o0 + r) * pl.inner + t] : 0.0f;
            if (SIGMOID) sh.b[place] = in[at];
        }
    }
    __syncthreads();
#pragma unroll
    for (uint32_t k = 0; k < kSub; k++) {
        if (k < count) {
            const uint32_t i = base + k * pl.inner;
            const double a = gate_a<SIGMOID>(v[k]), b = SIGMOID ? static_cast<double>(sigmoid_b(v[k])) : 1.0;
            const double d = static_cast<double>(g[k]) + K;
            if (grad_gate) {
                const double before = static_cast<double>(sh.a[i]);
                sh.a[i] = static_cast<float>(SIGMOID ? d * (before - static_cast<double>(sh.b[i])) * (a * b) : d * before);
            }
            sh.b[i] = static_cast<float>(d * b);
            K = a * d;
        }
    }
    if (grad_initial && count > 0 && w.q0 + w.j * kSub + count == pl.steps) grad_initial[w.channel] = static_cast<float>(K);
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < floats; e += kNarrowThreads) {
        uint32_t place;
        const uint64_t at = narrow_index<true>(pl, w, e, place);
        if (grad_gate) grad_gate[at] = sh.a[place];
        if (grad_in) grad_in[at] = sh.b[place];
    }
}

// ---------------------------------------------------------------- host side

// Which kernel takes a call. Times in us, sigmoid gates, walk / tiles / narrow:
//   few steps: [64,8,1024] 3.9 / 5.9 forward and 5.9 / 6.3 backward, [64,16,1024] 4.7 / 6.6 and 11.4 / 9.2,
//     [64,32,1024] 8.5 / 9.0 and 19.8 / 12.1; [1000,8,3] 4.1 / 5.6 / 7.0 and 6.0 / 5.5 / 12.5;
//   8 to 31 side by side, many channels: [16384,200,8] 78 / 301 / 165 and 233 / 615 / 286, [8192,200,16] 68 / 162 / 159 and
//     238 / 321 / 283, [8456,40,31] 32 / 50 / 75 and 99 / 72 / 127, [100000,20,24] forward 126 / - / 311;
//     few channels: [512,2000,8] 371 / 103 / 69 and 1554 / 181 / 107, [256,2000,16] 368 / 62 / 67 and 1782 / 103 / 105,
//     [132,200,31] 32 / 9 / 16 and 121 / 15 / 24, [1000,100,20] 18 / 14 / 21 and 61 / 21 / 34. Between, the border of 2^17 channels
//     is not where the times cross, which depends on how many lie side by side: below it [2048,200,8] takes 33 / 44 / 26 and
//     127 / 84 / 46, [8192,200,8] 48 / 154 / 90 and 172 / 310 / 154, [4096,200,16] 47 / 87 / 86 and 193 / 167 / 152,
//     [2114,200,31] 49 / 56 / 104 and 197 / 102 / 162;
//   hardly any side by side: [100000,64,1] 85 / 421 / 38 and 354 / 735 / 87, [1,66000,2] 4419 / - / 14; few of them: [100,100,5]
//     18 / 6 / 10 and 44 / 7.5 / 15.
enum class Path { walk, tiles, narrow };
Path path_of(const ScanShape& sh, bool forward) {
    const uint32_t few = forward && sh.inner >= 8 ? 32 : 8;
    if (sh.steps <= few) return Path::walk;
    if (sh.inner >= kNarrowInner) return Path::tiles;
    if (sh.inner >= 8) return sh.channels >= (1u << 17) ? Path::walk : Path::tiles;
    if (sh.inner >= 4 && static_cast<uint64_t>(sh.channels) * sh.steps < (1u << 20)) return Path::tiles;
    return Path::narrow;
}

// The words that tiles publish through live in memory of the library's own, kept between calls: calls follow one another on
// one stream, and each has a tag and a counter of its own. (Nothing that may take memory comes between this and the launch.)
int take_words(const char* what, uint64_t words, Wait* wait, uint32_t** counter, uint64_t** first) {
    constexpr uint64_t kHead = (kTags + 1) / 2;              // every tag's counter
    State& s = state();
    words += kHead;
    if (words > s.scan_words || s.scan_tag == kTags) {
        if (words > s.scan_words && !scan_reserve(words))
            return fail(KTH_E_MEMORY, "%s: no workspace of %llu bytes", what, static_cast<unsigned long long>(words * 8));
        for (uint64_t at = 0; at < s.scan_words; at += 1ull << 29)
            launch_fill(reinterpret_cast<float*>(s.scan + at), 2 * std::min<uint64_t>(s.scan_words - at, 1ull << 29), 0.0f);
        s.scan_tag = 0;
    }
    s.scan_tag += 1;
    *wait = Wait{s.scan_tag, s.scan_polls, s.host_index_flag_device + State::kScanLost};
    *counter = reinterpret_cast<uint32_t*>(s.scan) + s.scan_tag;
    *first = s.scan + kHead;
    return KTH_OK;
}

int plan_tiles(const char* what, const ScanShape& sh, int L, TilePlan* out) {
    TilePlan pl{};
    pl.steps = sh.steps; pl.inner = sh.inner;
    pl.tw = std::min<uint32_t>(kTileThreads / 64, (sh.steps + L - 1) / L);
    pl.col_blocks = (sh.inner + 63) / 64;
    pl.groups = sh.outer * pl.col_blocks;
    pl.tiles = (sh.steps + pl.tw * L - 1) / (pl.tw * L);
    pl.padded = pl.groups * 64;
    pl.group_div = make_div(pl.groups);
    pl.col_div = make_div(pl.col_blocks);
    if (pl.tiles > 1) {
        const uint64_t pairs = static_cast<uint64_t>(pl.tiles) * pl.padded * 2;
        if (int rc = take_words(what, pairs + static_cast<uint64_t>(pl.tiles / kSuper) * pl.padded, &pl.wait, &pl.tickets, &pl.pairs)) return rc;
        pl.states = pl.pairs + pairs;
    }
    *out = pl;
    return KTH_OK;
}

int plan_narrow(const char* what, const ScanShape& sh, NarrowPlan* out, uint32_t* grid) {
    NarrowPlan pl{};
    pl.outer = sh.outer; pl.steps = sh.steps; pl.inner = sh.inner; pl.channels = sh.channels;
    const uint32_t most = kNarrowThreads / sh.inner;         // pieces of a workgroup
    const uint32_t pieces = (sh.steps - 1) / kSub + 1;
    pl.pieces = std::min(pieces, most);
    pl.rows = std::min(sh.outer, most / pl.pieces);
    pl.tile_steps = pieces <= most ? sh.steps : most * kSub;
    pl.tiles = (sh.steps - 1) / pl.tile_steps + 1;
    if (pl.tiles > 1) pl.rows = 1;
    pl.inner_div = make_div(sh.inner);
    pl.row_div = make_div(sh.steps * sh.inner);              // (used where whole rows are taken)
    pl.outer_div = make_div(sh.outer);
    pl.piece_div = make_div(pl.pieces);
    *grid = pl.tiles > 1 ? pl.tiles * sh.outer : (sh.outer - 1) / pl.rows + 1;
    if (pl.tiles > 1) {
        const uint64_t pairs = static_cast<uint64_t>(pl.tiles) * pl.channels * 2;
        if (int rc = take_words(what, pairs + static_cast<uint64_t>(pl.tiles / kSuper) * pl.channels, &pl.wait, &pl.tickets, &pl.pairs))
            return rc;
        pl.states = pl.pairs + pairs;
    }
    *out = pl;
    return KTH_OK;
}

uint32_t tile_lds(const TilePlan& pl) { return 2 * pl.tw * 64 * static_cast<uint32_t>(sizeof(Pair)); }

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

int kth_recurrence_wait_limit(uint32_t looks) {
    std::lock_guard<std::mutex> guard(lock());
    KTH_REQUIRE_INIT();
    state().scan_polls = looks;
    return KTH_OK;
}

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
    const bool sigmoid = mode == KTH_GATE_SIGMOID;
    const Path path = path_of(sh, true);
    if (path == Path::narrow) {
        NarrowPlan pl; uint32_t grid;
        if (int rc = plan_narrow(what, sh, &pl, &grid)) return rc;
        overwrite_results(ops, 5);
        LaunchScope scope("recurrence_forward_narrow_kernel", sigmoid ? "sigmoid" : "given", (3 * n + 2 * sh.channels) * 4);
        auto* kernel = sigmoid ? recurrence_forward_narrow_kernel<true> : recurrence_forward_narrow_kernel<false>;
        hipLaunchKernelGGL(kernel, dim3(grid), dim3(kNarrowThreads), 0, state().stream, ops[0].ptr, ops[1].ptr, ops[2].ptr, ops[3].ptr, ops[4].ptr, pl);
        KTH_LAUNCH_CHECK("gated_recurrence_forward");
        return KTH_OK;
    }
    if (path == Path::tiles) {
        constexpr int L = 32;
        TilePlan pl;
        if (int rc = plan_tiles(what, sh, L, &pl)) return rc;
        overwrite_results(ops, 5);
        LaunchScope scope("recurrence_forward_tiles_kernel", sigmoid ? "sigmoid" : "given", (3 * n + 2 * sh.channels) * 4);
        const dim3 grid(pl.tiles * pl.groups), block(pl.tw * 64);
        const bool lines = sh.inner % 32 == 0;
        auto* kernel = sigmoid ? (lines ? recurrence_forward_tiles_kernel<true, true, L> : recurrence_forward_tiles_kernel<true, false, L>)
                               : (lines ? recurrence_forward_tiles_kernel<false, true, L> : recurrence_forward_tiles_kernel<false, false, L>);
        hipLaunchKernelGGL(kernel, grid, block, tile_lds(pl), state().stream, ops[0].ptr, ops[1].ptr, ops[2].ptr, ops[3].ptr, ops[4].ptr, pl);
        KTH_LAUNCH_CHECK("gated_recurrence_forward");
        return KTH_OK;
    }
    overwrite_results(ops, 5);
    LaunchScope scope("recurrence_forward_kernel", sigmoid ? "sigmoid" : "given", (3 * n + 2 * sh.channels) * 4);
    const dim3 grid((sh.channels - 1) / kBlock + 1);
    if (sigmoid)
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
    const Path path = path_of(sh, false);
    if (path == Path::narrow) {
        NarrowPlan pl; uint32_t grid;
        if (int rc = plan_narrow(what, sh, &pl, &grid)) return rc;
        overwrite_results(ops, 9);
        LaunchScope scope("recurrence_backward_narrow_kernel", sigmoid ? "sigmoid" : "given", (sigmoid ? 6 : 5) * n * 4);
        auto* kernel = sigmoid ? recurrence_backward_narrow_kernel<true> : recurrence_backward_narrow_kernel<false>;
        hipLaunchKernelGGL(kernel, dim3(grid), dim3(kNarrowThreads), 0, state().stream, ops[0].ptr, ops[1].ptr, ops[2].ptr, ops[3].ptr, ops[4].ptr,
                           ops[5].ptr, ops[6].ptr, ops[7].ptr, ops[8].ptr, pl);
        KTH_LAUNCH_CHECK("gated_recurrence_backward");
        return KTH_OK;
    }
    if (path == Path::tiles) {
        constexpr int L = 16;
        TilePlan pl;
        if (int rc = plan_tiles(what, sh, L, &pl)) return rc;
        overwrite_results(ops, 9);
        LaunchScope scope("recurrence_backward_tiles_kernel", sigmoid ? "sigmoid" : "given", (sigmoid ? 6 : 5) * n * 4);
        const dim3 grid(pl.tiles * pl.groups), block(pl.tw * 64);
        const bool lines = sh.inner % 32 == 0;
        auto* kernel = sigmoid ? (lines ? recurrence_backward_tiles_kernel<true, true, L> : recurrence_backward_tiles_kernel<true, false, L>)
                               : (lines ? recurrence_backward_tiles_kernel<false, true, L> : recurrence_backward_tiles_kernel<false, false, L>);
        hipLaunchKernelGGL(kernel, grid, block, tile_lds(pl), state().stream, ops[0].ptr, ops[1].ptr, ops[2].ptr, ops[3].ptr, ops[4].ptr,
                           ops[5].ptr, ops[6].ptr, ops[7].ptr, ops[8].ptr, pl);
        KTH_LAUNCH_CHECK("gated_recurrence_backward");
        return KTH_OK;
    }
    overwrite_results(ops, 9);
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
