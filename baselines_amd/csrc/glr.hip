// Gated linear recurrence over a time-major sequence, forward and backward:
//   a = sigmoid(f + bias)   p = reset ? 0 : h[t-1]   h[t] = a p + (1 - a) x[t]
//   g[t] = dy[t] + (reset[t+1] ? 0 : a[t+1] g[t+1])   dx = (1 - a) g   df = g (p - x) a (1 - a)
// The backward pass recomputes the states from float32 states kept every PPO2HIP_GLR_SPAN steps: they cost
// 4 / SPAN bytes per element where reading y back costs its whole width, and y is rounded to its type while p - x cancels.
#include <cstdlib>
#include <initializer_list>
#include <type_traits>

#include "kernels.hpp"

// Products and sums round one by one unless fmaf says otherwise: the same step written in two places gives the same bits, so
// that a span walked the slow way changes no other column, and the states that the backward pass recomputes are those that forward
// walked (a chain in 16 bits puts its outputs together from products instead, a few roundings of float32 from them).
#pragma clang fp contract(off)

namespace ppo2hip {

constexpr int kSpan = PPO2HIP_GLR_SPAN;                     // steps a wave holds in registers at a time
constexpr int kHeld = 16;                                   // spans that a workgroup can hold at once, one per wave

// ---------------------------------------------------------------------------------------------------------------------
// gates
// ---------------------------------------------------------------------------------------------------------------------

// How a step's gate is held between the passes over a span: the smaller side s = min(a, 1 - a) <= 1/2, negated where that is 1 - a
// (a >= 1/2, by the sign bit, -0 included), so that both sides keep their relative accuracy.  1 - a from a rounded a would lose the
// memory's length as soon as a is near one, and a from a rounded 1 - a what is left of a large state behind a gate near zero.
// For float32 sequences what the exponent's product and the reciprocal round is made good; 16 bits keep it (|z| 2^-24 and two ulp).
template <bool EXACT>
struct Gate {
    static __device__ inline float of(float z) {
        if (!EXACT) {
            const float e = __builtin_amdgcn_exp2f(fabsf(z) * -1.44269502f), s = e * __builtin_amdgcn_rcpf(1.f + e);
            return z >= 0.f ? -s : s;                       // a NaN is one on both sides
        }
        float m = fabsf(z);
        m = m > 128.f ? 128.f : m;                          // e^-128 is 0 in float32; a NaN stays one
        const float t = m * -1.44269502f;
        const float rest = fmaf(m, -1.92596299e-8f, fmaf(m, -1.44269502f, -t));
        float e = __builtin_amdgcn_exp2f(t);
        e = fmaf(e * 0.693147182f, rest, e);
        const float d = 1.f + e;
        float r = __builtin_amdgcn_rcpf(d);
        r = fmaf(fmaf(-d, r, 1.f), r, r);
        return copysignf(e * r, -z);
    }
    static __device__ inline float of(float z, float &slope) {                                       // a (1 - a), the gate's derivative
        const float v = of(z);
        slope = fabsf(v) * (1.f - fabsf(v));
        return v;
    }
    static __device__ inline bool keeps(float v) { return (int)__float_as_uint(v) < 0; }
    static __device__ inline float take(float v) { return keeps(v) ? -v : 1.f - v; }                 // 1 - a
    static __device__ inline float pass(float v, float h) { return fmaf(v, h, keeps(v) ? h : 0.f); } // a h
    // where h may not be finite: an infinite state passes every gate, however little of it is open, as it passes a run of gates
    static __device__ inline float pass_any(float v, float h) { return fabsf(h) < INFINITY ? pass(v, h) : v + h; }
    static __device__ inline float open() { return -0.f; }  // a = 1
    static __device__ inline float shut() { return 0.f; }   // a = 0
};

// ---------------------------------------------------------------------------------------------------------------------
// runs of steps
// ---------------------------------------------------------------------------------------------------------------------

// What a run of steps does to the state that enters it: h -> A h + B, words of which are handed from wave to wave.  Going back in
// time the same numbers carry the gradient that leaves a run at its front.
template <bool EXACT>
struct Run;

// float32: A, D and B with D = 1 - A kept beside A because a product of gates next to one has lost D's figures; A < 0 marks a
// run with a reset in it, which lets nothing through, infinities and NaN included.
template <>
struct Run<true> {
    static constexpr int kWords = 3;
    float w[3];
    static __device__ inline Run none() { return {{1.f, 0.f, 0.f}}; }
    static __device__ inline Run of(float A, float D, bool reset) { return {{reset ? -1.f : A, D, 0.f}}; }
    __device__ inline void add(float B) { w[2] = B; }
    __device__ inline float through(float h) const {
        if (w[0] < 0.f) return w[2];
        const float kept = w[1] <= 0.5f ? fmaf(-w[1], h, h) : w[0] * h;
        return (fabsf(h) < INFINITY ? kept : h) + w[2];    // an infinite state stays one however small A became
    }
    // this run and then that one
    __device__ inline Run join(const Run &r) const {
        return {{r.w[0] < 0.f || w[0] < 0.f ? -1.f : w[0] * r.w[0], fmaf(1.f - w[1], r.w[1], w[1]), r.through(w[2])}};
    }
};

// 16 bits: A, rounded once from whichever of A and D has more figures, and B.  A is zero where a reset is, and else never: its
// least value moves no finite state by as much as 5e-7 and keeps an infinite one.
template <>
struct Run<false> {
    static constexpr int kWords = 2;
    float w[2];
    static __device__ inline float live(float A) { return fmaxf(A, 0x1p-149f); }
    static __device__ inline Run none() { return {{1.f, 0.f}}; }
    static __device__ inline Run of(float A, float D, bool reset) { return {{reset ? 0.f : live(A > 0.75f ? 1.f - D : A), 0.f}}; }
    __device__ inline void add(float B) { w[1] = B; }
    __device__ inline float through(float h) const { return w[0] == 0.f ? w[1] : fmaf(w[0], h, w[1]); }
    __device__ inline Run join(const Run &r) const { return {{r.w[0] == 0.f || w[0] == 0.f ? 0.f : live(w[0] * r.w[0]), r.through(w[1])}}; }
};

// ---------------------------------------------------------------------------------------------------------------------
// addresses
// ---------------------------------------------------------------------------------------------------------------------

template <class T>
struct Seq {
    T *p;
    int64_t t, e;
};

// V neighbouring channels of one step, at any address an element may have.  Inputs of 16 bits stay bits until they are used: as
// vectors of their type the compiler keeps them in more registers than they have.
template <class T, int V>
struct Lane {
    typedef T Out __attribute__((ext_vector_type(V)));
    typedef Out AnyOut __attribute__((aligned(sizeof(T))));
    static __device__ inline void store(void *p, const float (&v)[V]) {
        Out r;
#pragma unroll
        for (int k = 0; k < V; k++) {
            float w = v[k];
            // float32 first: a product fused with its rounding to float16 rounds once, and not the same in two places
            if (std::is_same<T, _Float16>::value) asm("" : "+v"(w));
            r[k] = (T)w;                                  // to nearest: the type that the layer hands on; states stay float32
        }
        *(AnyOut *)p = r;
    }
};
template <int Bytes>
struct Bits;
template <>
struct Bits<2> {
    typedef unsigned short Word;
    typedef Word Any __attribute__((aligned(2)));
};
template <>
struct Bits<4> {
    typedef unsigned Word;
    typedef Word Any __attribute__((aligned(2)));
};
template <class T>
__device__ inline float widen(unsigned bits);
template <>
__device__ inline float widen<float>(unsigned bits) { return __uint_as_float(bits); }
template <>
__device__ inline float widen<__bf16>(unsigned bits) { return __uint_as_float(bits << 16); }
template <>
__device__ inline float widen<_Float16>(unsigned bits) { return (float)__builtin_bit_cast(_Float16, (unsigned short)bits); }

// Which columns a wave works on.  Addresses are a wave-uniform 64-bit part (step, the wave's first env) and a 32-bit part
// per lane: kept as 64 bits per lane and step they cost 2 registers each and the kernels spill.
struct Place {
    unsigned c;         // the lane's first column e * H + j
    int e0, de, j;      // first env of the wave, lane's env less that, channel
    bool mine;          // false: a lane behind the last column, which repeats it and writes nothing
};
// env_tiles 0: columns in a row over all envs.  Else that many tiles per env, where envs lie too far apart for 32 bits.
template <int V>
__device__ inline Place place_of(unsigned tile, unsigned C, unsigned H, unsigned env_tiles) {
    const unsigned lane = threadIdx.x & 63;
    Place p;
    if (env_tiles == 0) {
        const uint64_t c = ((uint64_t)tile * 64 + lane) * V;
        p.mine = c < C;
        p.c = p.mine ? (unsigned)c : C - V;
        const unsigned e = p.c / H;
        p.e0 = __builtin_amdgcn_readfirstlane(e);
        p.de = (int)e - p.e0;
        p.j = (int)(p.c - e * H);
    } else {
        const unsigned e = tile / env_tiles, j = ((tile - e * env_tiles) * 64 + lane) * V;
        p.mine = j < H;
        p.j = (int)(p.mine ? j : H - V);
        p.e0 = (int)e;
        p.de = 0;
        p.c = e * H + (unsigned)p.j;
    }
    return p;
}
// Tile of a workgroup.  Workgroups go to the 8 XCDs in turn, and rows whose length is no multiple of a cache line leave
// neighbouring tiles with a line in common: eight tiles in a row are given to one XCD, whose L2 then fetches and merges it once.
// [200, 300, 777] bfloat16: 103 / 204 us forward / backward without, 90 / 181 with.
__device__ inline unsigned seat_of(unsigned b) { return (b | 63u) < gridDim.x ? (b & ~63u) | (b & 7) << 3 | (b >> 3 & 7) : b; }
template <class T>
__device__ inline unsigned lane_offset(const Seq<T> &s, const Place &at) {
    return (unsigned)(at.de * (int)s.e + at.j) * (unsigned)sizeof(T);
}
// A lane's offset, said anew where it is used: extended to 64 bits in another block it is no longer seen to be 32, and every
// access adds 64-bit addresses in vector registers instead of taking a scalar base and this.
__device__ inline unsigned here(unsigned off) {
    asm volatile("" : "+v"(off));
    return off;
}
// A step's distance in bytes, said anew for every span: as loop invariants the 16 multiples of every array's distance are kept
// in scalar registers, which do not hold them.
template <class T>
__device__ inline int64_t distance(const Seq<T> &s) {
    int64_t d = s.t * (int64_t)sizeof(T);
    asm volatile("" : "+s"(d));
    return d;
}
template <class T>
__device__ inline char *step_base(const Seq<T> &s, const Place &at, int64_t t0) {
    return (char *)(s.p + t0 * s.t + at.e0 * s.e);
}

// Flags of the span's steps t0 .. t0+n-1 as bits.  Where all lanes look at one env, 16 of them fetch one flag each.
__device__ inline unsigned span_resets(const Seq<const uint8_t> &r, int64_t t0, int n, const Place &at) {
    if (!r.p || n <= 0) return 0u;
    const uint8_t *p = r.p + t0 * r.t + at.e0 * r.e;
    if (__all(at.de == 0)) {
        const int lane = threadIdx.x & 63;
        const bool on = lane < n && p[(int64_t)lane * r.t] != 0;
        return (unsigned)__ballot(on);
    }
    const unsigned off = (unsigned)(at.de * (int)r.e);
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < kSpan; i++)
        if (i < n && p[(int64_t)i * r.t + off] != 0) m |= 1u << i;
    return m;
}

template <class T, int V>
struct Raw {
    typedef Bits<sizeof(T) * V> Kind;
    typename Kind::Word v[kSpan];
    __device__ inline float get(int i, int k) const {
        if (sizeof(T) == 4 || V == 1) return widen<T>(v[i]);
        return widen<T>(k == 0 ? v[i] & 0xffffu : (unsigned)v[i] >> 16);
    }
    static __device__ inline typename Kind::Word one(const char *p) { return *(const typename Kind::Any *)p; }
    __device__ inline void load(const Seq<const T> &s, const Place &at, unsigned off, int64_t t0, int n) {
        const char *p = step_base(s, at, t0);
        const int64_t step = distance(s);
        if (n >= kSpan) {
            off = here(off);
#pragma unroll
            for (int i = 0; i < kSpan; i++, p += step) v[i] = one(p + off);
        } else {
#pragma unroll
            for (int i = 0; i < kSpan; i++, p += step) {
                v[i] = 0;
                if (i < n) v[i] = one(p + off);
            }
        }
    }
};

// ---------------------------------------------------------------------------------------------------------------------
// spans
// ---------------------------------------------------------------------------------------------------------------------

template <int V>
using Span = float[kSpan][V];

// The value, of which the compiler knows nothing: what the seldom walked slow paths derive from a span is otherwise worked out,
// and kept in registers, ahead of the branch to them.
__device__ inline float anew(float v) {
    asm volatile("" : "+v"(v));
    return v;
}
__device__ inline unsigned anew(unsigned v) {
    asm volatile("" : "+v"(v));
    return v;
}

// A gate with a reset at its step is shut for the state: a finite one is multiplied by zero, a NaN stays one.
template <bool EXACT>
__device__ inline float with_reset(float g, unsigned rm, int i) { return rm >> i & 1 ? Gate<EXACT>::shut() : g; }

// A span's gates, shut at resets, and what each step adds to the state, u = (1 - a) x of the gate itself.  Steps behind the last
// one keep the state as it is.
template <class T, int V>
__device__ inline void span_open(const Raw<T, V> &f, const Raw<T, V> &x, const float (&b)[V], int n, unsigned rm, Span<V> &g, Span<V> &u) {
    typedef Gate<sizeof(T) == 4> G;
#pragma unroll
    for (int i = 0; i < kSpan; i++)
#pragma unroll
        for (int k = 0; k < V; k++) {
            g[i][k] = G::of(f.get(i, k) + b[k]);
            u[i][k] = G::take(g[i][k]) * x.get(i, k);
        }
    if (n < kSpan)
#pragma unroll
        for (int i = 0; i < kSpan; i++)
#pragma unroll
            for (int k = 0; k < V; k++)
                if (i >= n) g[i][k] = G::open(), u[i][k] = 0.f;
    if (__any(rm != 0))
#pragma unroll
        for (int i = 0; i < kSpan; i++)
#pragma unroll
            for (int k = 0; k < V; k++) g[i][k] = with_reset<sizeof(T) == 4>(g[i][k], rm, i);
}

template <int V>
__device__ inline bool any_not_finite(const float (&h)[V]) {
    bool bad = false;
#pragma unroll
    for (int k = 0; k < V; k++) bad |= !(fabsf(h[k]) < INFINITY);
    return __any(bad);
}

// Walks a span from state h, handing every step's state to `out(i, h)`: the quick way where `whole` says that out may be called for
// all steps, the general way (out only for steps below n) elsewhere.  The quick form of a step turns an infinite state to NaN, and
// NaN goes through shut gates: a span that met either ends in NaN and is walked again.
template <bool EXACT, int V, class Out>
__device__ inline void span_walk(const Span<V> &g, const Span<V> &u, unsigned rm, bool whole, int n, float (&h)[V], Out out) {
    typedef Gate<EXACT> G;
    if (whole) {
        float h0[V];
#pragma unroll
        for (int k = 0; k < V; k++) h0[k] = h[k];
#pragma unroll
        for (int i = 0; i < kSpan; i++) {
#pragma unroll
            for (int k = 0; k < V; k++) h[k] = G::pass(g[i][k], h[k]) + u[i][k];
            out(i, h);
        }
        if (!any_not_finite(h)) return;
#pragma unroll
        for (int k = 0; k < V; k++) h[k] = h0[k];
    }
#pragma unroll
    for (int i = 0; i < kSpan; i++) {
#pragma unroll
        for (int k = 0; k < V; k++) h[k] = anew(rm) >> i & 1 ? u[i][k] : G::pass_any(anew(g[i][k]), h[k]) + u[i][k];
        if (i < n) out(i, h);
    }
}

// What a span lets through.  D = 1 - A grows by 1 - a of what is left of it, so that it keeps its figures while it is small.  For 16
// bits D counts only where A ends above 3/4, which no gate of 1/2 and less leaves it: there 1 - a is the gate as it is held, negated.
template <bool EXACT, int V>
__device__ inline void span_passes(const Span<V> &g, unsigned rm, Run<EXACT> (&r)[V]) {
    typedef Gate<EXACT> G;
    float A[V], D[V];
#pragma unroll
    for (int k = 0; k < V; k++) A[k] = 1.f, D[k] = 0.f;
#pragma unroll
    for (int i = 0; i < kSpan; i++)
#pragma unroll
        for (int k = 0; k < V; k++) {
            const float om = EXACT ? G::take(g[i][k]) : -g[i][k];
            A[k] = G::pass(g[i][k], A[k]);
            D[k] = D[k] + fmaf(-D[k], om, om);
        }
#pragma unroll
    for (int k = 0; k < V; k++) r[k] = Run<EXACT>::of(A[k], D[k], rm != 0);
}

// A span's run in the direction of time.
template <bool EXACT, int V>
__device__ inline void span_run(const Span<V> &g, const Span<V> &u, unsigned rm, Run<EXACT> (&r)[V]) {
    float h[V];
#pragma unroll
    for (int k = 0; k < V; k++) h[k] = 0.f;
    span_passes<EXACT, V>(g, rm, r);
    span_walk<EXACT, V>(g, u, rm, true, kSpan, h, [](int, const float (&)[V]) {});
#pragma unroll
    for (int k = 0; k < V; k++) r[k].add(h[k]);
}

// The same for a chain in 16 bits, which leaves in g and u what the steps up to each let through of the state in front of the span and
// the state that they build up from zero, so that the outputs are one product and sum each once that state is known.  What a step
// lets through is off by 2^-25 for each step before it, which 16 bits do not show; the state behind the span goes by D.
// [65536, 1, 1000] bfloat16: 131 us with a walk in either place, 127 so; where a workgroup holds the sequence the walk is quicker
// ([128, 512, 256]: 24.5, 27).
template <class T, int V, bool WHOLE>
__device__ inline void scan_steps(const Raw<T, V> &f, const Raw<T, V> &x, const float (&b)[V], int n, unsigned rm, Span<V> &g, Span<V> &u, float (&D)[V]) {
    typedef Gate<false> G;
    float A[V], h[V];
#pragma unroll
    for (int k = 0; k < V; k++) A[k] = 1.f, D[k] = h[k] = 0.f;
#pragma unroll
    for (int i = 0; i < kSpan; i++)
#pragma unroll
        for (int k = 0; k < V; k++) {
            float v = G::of(f.get(i, k) + b[k]), add = G::take(v) * x.get(i, k);
            if (!WHOLE) {
                if (i >= n) v = G::open(), add = 0.f;
                v = with_reset<false>(v, rm, i);
            }
            A[k] = G::pass(v, A[k]);
            D[k] = D[k] + fmaf(-D[k], -v, -v);              // as in span_passes
            h[k] = G::pass(v, h[k]) + add;
            g[i][k] = A[k];
            u[i][k] = h[k];
        }
}
template <class T, int V, class Args>
__device__ inline void span_scan(const Args &a, const Place &at, const Raw<T, V> &f, const Raw<T, V> &x, const float (&b)[V], int64_t t0, int n, unsigned rm,
                                 Span<V> &g, Span<V> &u, Run<false> (&r)[V]) {
    typedef Gate<false> G;
    float D[V];
    if (n >= kSpan && !__any(rm != 0)) scan_steps<T, V, true>(f, x, b, n, rm, g, u, D);
    else scan_steps<T, V, false>(f, x, b, n, rm, g, u, D);
    if (any_not_finite(u[kSpan - 1])) {
        // the inputs once more from memory: kept for this, they would cost 32 registers
        asm volatile("" : "+s"(t0));
        const char *fp = step_base(a.f, at, t0), *xp = step_base(a.x, at, t0);
        const int64_t fstep = distance(a.f), xstep = distance(a.x);
        const unsigned fo = lane_offset(a.f, at), xo = lane_offset(a.x, at);
        Raw<T, V> in;
        float h[V];
#pragma unroll
        for (int k = 0; k < V; k++) h[k] = 0.f;
#pragma unroll
        for (int i = 0; i < kSpan; i++, fp += fstep, xp += xstep) {
            if (i < n) {
                in.v[0] = in.one(fp + here(fo)), in.v[1] = in.one(xp + here(xo));
#pragma unroll
                for (int k = 0; k < V; k++) {
                    const float v = G::of(in.get(0, k) + b[k]), add = G::take(v) * in.get(1, k);
                    h[k] = anew(rm) >> i & 1 ? add : G::pass_any(v, h[k]) + add;
                }
            }
#pragma unroll
            for (int k = 0; k < V; k++) {
                u[i][k] = h[k];
                if (anew(rm) << (31 - i)) g[i][k] = 0.f;    // a reset at step i or before also hides a gate that is no number
            }
        }
    }
#pragma unroll
    for (int k = 0; k < V; k++) {
        r[k] = Run<false>::of(g[kSpan - 1][k], D[k], rm != 0);
        r[k].add(u[kSpan - 1][k]);
    }
}

// A span's run against time, for the gradient: dy enters a step before the gate does, a reset stands behind it.
template <class T>
__device__ inline void span_run_back(const Span<1> &g, const Raw<T, 1> &dy, unsigned rm, Run<sizeof(T) == 4> (&r)[1]) {
    typedef Gate<sizeof(T) == 4> G;
    span_passes<sizeof(T) == 4, 1>(g, rm, r);
    float c[1] = {0.f};
    if (!__any(rm != 0)) {
#pragma unroll
        for (int i = kSpan - 1; i >= 0; i--) c[0] = G::pass(g[i][0], c[0] + dy.get(i, 0));
    } else {
#pragma unroll
        for (int i = kSpan - 1; i >= 0; i--) c[0] = G::pass(with_reset<sizeof(T) == 4>(g[i][0], rm, i), c[0] + dy.get(i, 0));
    }
    r[0].add(c[0]);
    if (!any_not_finite(c)) return;
    c[0] = 0.f;
#pragma unroll
    for (int i = kSpan - 1; i >= 0; i--) c[0] = anew(rm) >> i & 1 ? 0.f : G::pass_any(anew(g[i][0]), c[0] + dy.get(i, 0));
    r[0].add(c[0]);
}

// A tile's runs, as waves of a workgroup hand them on.
template <bool EXACT, int V>
struct RunSpace {
    float w[Run<EXACT>::kWords][64 * V];
    __device__ inline void put(const Run<EXACT> (&r)[V]) {
#pragma unroll
        for (int q = 0; q < Run<EXACT>::kWords; q++)
#pragma unroll
            for (int k = 0; k < V; k++) w[q][(threadIdx.x & 63) * V + k] = r[k].w[q];
    }
    __device__ inline Run<EXACT> get(int k) const {
        Run<EXACT> r;
#pragma unroll
        for (int q = 0; q < Run<EXACT>::kWords; q++) r.w[q] = w[q][(threadIdx.x & 63) * V + k];
        return r;
    }
};

// ---------------------------------------------------------------------------------------------------------------------
// a chain of workgroups
// ---------------------------------------------------------------------------------------------------------------------

// Long sequences in one pass over the data: a workgroup holds kChainWaves spans of a tile in registers, a batch, and the batches of
// a tile hand each other what they do to the state.  kChainWaves batches in a row form a group and as many groups a block.  A batch
// publishes its run, the last one of a group the group's run, and the last one of a block the state behind it; a batch waits for the
// runs of its group's earlier batches, one per wave, then for the runs of its block's earlier groups and the state in front of the
// block.  What is joined with what does not depend on who came first, so that results are the same bits every time.
// A word is published by one agent-scope store and is its own flag: a launch before fills all words with kEmpty, a NaN that no
// arithmetic makes.  Every wait is bounded; a wave that gives up raises the library's fault word and carries on with NaN.
//
// Four tiles in a row share a counter, behind which their batches are given out in order, all four tiles' first ones before the second
// ones: what a batch waits for, earlier batches of its own tile, has been drawn by workgroups that are running and that wait for still
// earlier ones only, whatever else runs on the card and wherever workgroups start.  One counter for all tiles is drawn from once in
// 10 ns: [2048, 16, 512] float32 48 us forward, a counter per four tiles 41, per tile 41 and [16384, 4, 1024] bfloat16 102, 104, 110
// (tiles that drift apart in time share no cache lines).  Lists of seats per XCD took 14 us off [65536, 1, 1000] bfloat16, but a
// workgroup then waits for seats that no running one has drawn, which two such launches at once can turn into a deadlock.
constexpr int kChainWaves = 8, kBatch = kChainWaves * kSpan;
constexpr unsigned kEmpty = 0xffffffffu;
constexpr int kTurnWords = 64, kTurns = 64, kTurnTiles = 4, kTurnBytes = kTurns * kTurnWords * sizeof(unsigned);

struct Chain {
    unsigned *turn;         // counters, kTurnWords apart; behind them
    float *runs;            // [batches][words of a run][C]
    float *groups;          // [groups][words of a run][C]
    float *states;          // [blocks][C]: in front of blocks 1, 2, ...
    unsigned tiles;
    int batches, max_spins;
    unsigned *fault;
};

__device__ inline void publish(float *p, float v) {
    const unsigned bits = __float_as_uint(v);
    __hip_atomic_store((unsigned *)p, bits == kEmpty ? 0x7fc00000u : bits, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// from a base that the wave shares
__device__ inline unsigned peek(const float *base, unsigned c) {
    return __hip_atomic_load((const unsigned *)((const char *)base + c), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

__global__ __launch_bounds__(256) void glr_chain_clear_kernel(Chain ch, int64_t words) {
    const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
    if (i < 4 * kTurns) ch.turn[i / 4 * kTurnWords] = 0;
    unsigned *p = (unsigned *)ch.runs + i;
    if (i + 4 <= words) *(uint4 *)p = make_uint4(kEmpty, kEmpty, kEmpty, kEmpty);
    else
        for (int k = 0; i + k < words; k++) p[k] = kEmpty;
}

template <bool EXACT, int V>
struct ChainSpace {
    RunSpace<EXACT, V> runs[kChainWaves], before[kChainWaves - 1], far[kChainWaves - 1];      // of spans, batches, groups
    float state[64 * V];
    unsigned turn;
};

// Waits until the lane's words at base [N][C], V of each, have been published.
template <int N, int V>
__device__ inline void await(const Chain &ch, const float *base, unsigned C, const Place &at, float (&v)[N][V]) {
    const unsigned byte = at.c * 4u;                      // C < 2^30
    unsigned bits[N][V];
    for (int tries = 0;; tries++) {
        bool ok = true;
#pragma unroll
        for (int q = 0; q < N; q++)
#pragma unroll
            for (int k = 0; k < V; k++) bits[q][k] = peek(base + q * (int64_t)C + k, byte);
#pragma unroll
        for (int q = 0; q < N; q++)
#pragma unroll
            for (int k = 0; k < V; k++) ok &= bits[q][k] != kEmpty;
        if (__all(ok) && ch.max_spins >= 0) break;
        if (tries >= ch.max_spins) {
            if ((threadIdx.x & 63) == 0) atomicOr(ch.fault, kFaultGridSync);
#pragma unroll
            for (int q = 0; q < N; q++)
#pragma unroll
                for (int k = 0; k < V; k++) bits[q][k] = kEmpty;    // NaN as a whole: some words may have come
            break;
        }
        __builtin_amdgcn_s_sleep(1);
    }
#pragma unroll
    for (int q = 0; q < N; q++)
#pragma unroll
        for (int k = 0; k < V; k++) v[q][k] = __uint_as_float(bits[q][k]);
}
template <bool EXACT, int V>
__device__ inline void await_run(const Chain &ch, const float *runs, int64_t i, unsigned C, const Place &at, RunSpace<EXACT, V> &out) {
    constexpr int kWords = Run<EXACT>::kWords;
    float v[kWords][V];
    await<kWords, V>(ch, runs + i * kWords * C, C, at, v);
    Run<EXACT> r[V];
#pragma unroll
    for (int k = 0; k < V; k++)
#pragma unroll
        for (int q = 0; q < kWords; q++) r[k].w[q] = v[q][k];
    out.put(r);
}
template <bool EXACT, int V>
__device__ inline void publish_run(float *runs, int64_t i, unsigned C, const Place &at, const Run<EXACT> (&r)[V]) {
    constexpr int kWords = Run<EXACT>::kWords;
    if (!at.mine) return;
#pragma unroll
    for (int k = 0; k < V; k++)
#pragma unroll
        for (int q = 0; q < kWords; q++) publish(runs + (i * kWords + q) * C + at.c + k, r[k].w[q]);
}

// State (gradient, when BACK) in front of wave w's span, from the span's own run and the value h in front of the whole sequence.
// All waves of the workgroup call it; publishes what later batches wait for.
template <bool EXACT, bool BACK, int V>
__device__ inline void chain_through(const Chain &ch, ChainSpace<EXACT, V> &m, unsigned C, const Place &at, int order, int w, const Run<EXACT> (&own)[V],
                                     float (&h)[V]) {
    constexpr int kLast = kChainWaves - 1;
    const int group = order / kChainWaves, rank = order % kChainWaves, block = group / kChainWaves, grank = group % kChainWaves;
    const bool more = order + 1 < ch.batches;
    Run<EXACT> all[V];
#pragma unroll
    for (int k = 0; k < V; k++) all[k] = Run<EXACT>::none();
    m.runs[w].put(own);
    __syncthreads();
    if (w < rank) {
        await_run<EXACT, V>(ch, ch.runs, (int64_t)group * kChainWaves + w, C, at, m.before[w]);
    } else if (w == kLast && more) {
        for (int i = 0; i < kChainWaves; i++)
#pragma unroll
            for (int k = 0; k < V; k++) all[k] = all[k].join(m.runs[BACK ? kLast - i : i].get(k));
        if (rank < kLast) publish_run<EXACT, V>(ch.runs, order, C, at, all);
    }
    __syncthreads();
    if (w < grank) {
        await_run<EXACT, V>(ch, ch.groups, (int64_t)block * kChainWaves + w, C, at, m.far[w]);
    } else if (w == kLast) {
        if (rank == kLast && grank < kLast && more) {
            Run<EXACT> whole[V];
#pragma unroll
            for (int k = 0; k < V; k++) whole[k] = Run<EXACT>::none();
            for (int i = 0; i < kLast; i++)
#pragma unroll
                for (int k = 0; k < V; k++) whole[k] = whole[k].join(m.before[i].get(k));
#pragma unroll
            for (int k = 0; k < V; k++) whole[k] = whole[k].join(all[k]);
            publish_run<EXACT, V>(ch.groups, group, C, at, whole);
        }
        float v[1][V];
#pragma unroll
        for (int k = 0; k < V; k++) v[0][k] = h[k];
        if (block > 0) await<1, V>(ch, ch.states + (int64_t)block * C, C, at, v);
#pragma unroll
        for (int k = 0; k < V; k++) m.state[(threadIdx.x & 63) * V + k] = v[0][k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < V; k++) h[k] = m.state[(threadIdx.x & 63) * V + k];
    for (int i = 0; i < grank; i++)
#pragma unroll
        for (int k = 0; k < V; k++) h[k] = m.far[i].get(k).through(h[k]);
    for (int i = 0; i < rank; i++)
#pragma unroll
        for (int k = 0; k < V; k++) h[k] = m.before[i].get(k).through(h[k]);
    const int steps = BACK ? kLast - w : w;
    for (int i = 0; i < steps; i++)
#pragma unroll
        for (int k = 0; k < V; k++) h[k] = m.runs[BACK ? kLast - i : i].get(k).through(h[k]);
    if (steps == kLast && rank == kLast && grank == kLast && more && at.mine)
#pragma unroll
        for (int k = 0; k < V; k++) publish(ch.states + (block + 1) * (int64_t)C + at.c + k, own[k].through(h[k]));
}

// The batch that this workgroup draws: its tile's columns and wave w's span in it.
struct Drawn {
    Place at;
    int order, batch, n;
    int64_t t0;
};
template <bool BACK, int V, class Args>
__device__ inline Drawn draw(const Args &a, const Chain &ch, unsigned &turn, int w) {
    // counter c serves the tiles of groups c, c + kTurns, ...; as many workgroups draw from it as it has seats
    const unsigned groups = (ch.tiles + kTurnTiles - 1) / kTurnTiles, c = seat_of(blockIdx.x) % ch.tiles / kTurnTiles % kTurns;
    const unsigned last = c + (groups - 1 - c) / kTurns * kTurns, share = (last - c) / kTurns * kTurnTiles + min(ch.tiles - last * kTurnTiles, (unsigned)kTurnTiles);
    if (threadIdx.x == 0) turn = atomicAdd(ch.turn + c * kTurnWords, 1u);
    __syncthreads();
    const unsigned n = __builtin_amdgcn_readfirstlane(turn), i = n % share;
    Drawn d;
    d.order = (int)(n / share);
    d.batch = BACK ? ch.batches - 1 - d.order : d.order;
    d.at = place_of<V>((c + i / kTurnTiles * kTurns) * kTurnTiles + i % kTurnTiles, a.C, a.H, a.env_tiles);
    d.t0 = ((int64_t)d.batch * kChainWaves + w) * kSpan;
    d.n = (int)(a.T_ - d.t0 < kSpan ? a.T_ - d.t0 : kSpan);
    return d;
}

// ---------------------------------------------------------------------------------------------------------------------
// forward
// ---------------------------------------------------------------------------------------------------------------------

template <class T>
struct ForwardArgs {
    Seq<const T> f, x;
    Seq<const uint8_t> resets;
    Seq<T> y;
    const float *bias, *h0;
    float *h_last, *saved;
    int T_;
    unsigned C, H, env_tiles;
};

template <class T, int V, bool SCAN>
__device__ inline void forward_span(const ForwardArgs<T> &a, const Place &at, unsigned yo, int64_t t0, int n, unsigned rm, const Span<V> &g,
                                    const Span<V> &u, const Run<sizeof(T) == 4> (&r)[V], float (&h)[V]) {
    if (!at.mine) return;
    if (a.saved)
#pragma unroll
        for (int k = 0; k < V; k++) a.saved[t0 / kSpan * a.C + at.c + k] = h[k];
    char *p = nullptr;
    const int64_t step = distance(a.y);
    auto put = [&](int i, const float (&v)[V]) {
        p = i == 0 ? step_base(a.y, at, t0) : p + step;
        Lane<T, V>::store(p + here(yo), v);
    };
    if constexpr (!SCAN) {
        span_walk<sizeof(T) == 4, V>(g, u, rm, n >= kSpan, n, h, put);
    } else {
        float v[V];
        if (n >= kSpan && !any_not_finite(h)) {
#pragma unroll
            for (int i = 0; i < kSpan; i++) {
#pragma unroll
                for (int k = 0; k < V; k++) v[k] = fmaf(g[i][k], h[k], u[i][k]);
                put(i, v);
            }
        } else {
#pragma unroll
            for (int i = 0; i < kSpan; i++)
                if (i < n) {
#pragma unroll
                    for (int k = 0; k < V; k++) {
                        v[k] = fabsf(h[k]) < INFINITY ? fmaf(g[i][k], h[k], u[i][k]) : h[k] + u[i][k];
                        if (anew(rm) << (31 - i)) v[k] = u[i][k];           // a reset at step i or before
                    }
                    put(i, v);
                }
        }
#pragma unroll
        for (int k = 0; k < V; k++) h[k] = r[k].through(h[k]);
    }
    if (a.h_last && t0 + kSpan >= a.T_)
#pragma unroll
        for (int k = 0; k < V; k++) a.h_last[at.c + k] = h[k];
}

// Short sequences in one launch: a workgroup holds the whole of its columns, one span per wave, and the waves exchange their
// spans' runs through LDS.  Bound by memory: [128, 512, 256] bfloat16, 101 MB in 25 us, float32 and training 206 MB in 48 us (4.3 TB/s).
template <class T, int V>
__global__ __launch_bounds__(64 * kHeld) void glr_forward_held_kernel(ForwardArgs<T> a) {
    __shared__ RunSpace<sizeof(T) == 4, V> runs[kHeld];
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Place at = place_of<V>(seat_of(blockIdx.x), a.C, a.H, a.env_tiles);
    const int64_t t0 = (int64_t)w * kSpan;
    const int n = (int)(a.T_ - t0 < kSpan ? a.T_ - t0 : kSpan);
    Raw<T, V> fr, xr;
    fr.load(a.f, at, lane_offset(a.f, at), t0, n);
    xr.load(a.x, at, lane_offset(a.x, at), t0, n);
    const unsigned rm = span_resets(a.resets, t0, n, at);
    float b[V], h[V];
#pragma unroll
    for (int k = 0; k < V; k++) b[k] = a.bias ? a.bias[at.j + k] : 0.f;
    Span<V> g, u;
    Run<sizeof(T) == 4> r[V];
    span_open<T, V>(fr, xr, b, n, rm, g, u);
    span_run<sizeof(T) == 4, V>(g, u, rm, r);
    runs[w].put(r);
#pragma unroll
    for (int k = 0; k < V; k++) h[k] = a.h0 ? a.h0[at.c + k] : 0.f;
    __syncthreads();
    for (int i = 0; i < w; i++)
#pragma unroll
        for (int k = 0; k < V; k++) h[k] = runs[i].get(k).through(h[k]);
    forward_span<T, V, false>(a, at, lane_offset(a.y, at), t0, n, rm, g, u, r, h);
}

// Bound by what of the loads and the hand-over the 16 waves of a CU do not hide from each other, and 31 operations per element (55 us
// of all SIMDs for 66 M elements).  bfloat16 [65536, 1, 1000], 393 MB: 125 us (3.1 TB/s; a copy in the same tiles 102: rows of 2000
// bytes, whose lines neighbouring tiles fetch twice), [65536, 1, 1024] 107, [16384, 4, 1024] 100.  Two channels per lane: with one 139,
// 115, 107.  Waves of a workgroup: with 4 and 16 in place of 8 154 and 152, 131 and 139, 111 and 129.
template <class T, int V>
__global__ __launch_bounds__(64 * kChainWaves, V == 2 ? 4 : 5) void glr_forward_chain_kernel(ForwardArgs<T> a, Chain ch) {
    __shared__ ChainSpace<sizeof(T) == 4, V> mem;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Drawn d = draw<false, V>(a, ch, mem.turn, w);
    Raw<T, V> fr, xr;
    fr.load(a.f, d.at, lane_offset(a.f, d.at), d.t0, d.n);
    xr.load(a.x, d.at, lane_offset(a.x, d.at), d.t0, d.n);
    const unsigned rm = span_resets(a.resets, d.t0, d.n, d.at);
    float b[V], h[V];
#pragma unroll
    for (int k = 0; k < V; k++) b[k] = a.bias ? a.bias[d.at.j + k] : 0.f;
    Span<V> g, u;
    Run<sizeof(T) == 4> r[V];
    if constexpr (sizeof(T) == 4) {
        span_open<T, V>(fr, xr, b, d.n, rm, g, u);
        span_run<true, V>(g, u, rm, r);
    } else {
        span_scan<T, V>(a, d.at, fr, xr, b, d.t0, d.n, rm, g, u, r);
    }
#pragma unroll
    for (int k = 0; k < V; k++) h[k] = a.h0 ? a.h0[d.at.c + k] : 0.f;
    chain_through<sizeof(T) == 4, false, V>(ch, mem, a.C, d.at, d.order, w, r, h);
    if (d.n > 0) forward_span<T, V, sizeof(T) == 2>(a, d.at, lane_offset(a.y, d.at), d.t0, d.n, rm, g, u, r, h);
}

// ---------------------------------------------------------------------------------------------------------------------
// backward
// ---------------------------------------------------------------------------------------------------------------------

template <class T>
struct BackwardArgs {
    Seq<const T> f, x, dy;
    Seq<const uint8_t> resets;
    Seq<T> df, dx;
    const float *bias, *saved, *dh_last;
    float *dbias_rows, *dh0;        // dbias_rows [workgroups along time][C] or null
    int T_;
    unsigned C, H, env_tiles;
};

// Gates and q = (p - x) a (1 - a), what df is per unit of g, from the states recomputed off the kept one.
template <class T>
__device__ inline void back_open(const BackwardArgs<T> &a, const Place &at, const Raw<T, 1> &f, const Raw<T, 1> &x, float b, float kept, int64_t t0, int n,
                                 unsigned rm, Span<1> &g, Span<1> &q) {
    typedef Gate<sizeof(T) == 4> G;
    constexpr bool kExact = sizeof(T) == 4;
    float h[1] = {kept}, slope;
    if (!__any(rm != 0)) {
#pragma unroll
        for (int i = 0; i < kSpan; i++) {
            const float xv = x.get(i, 0), v = G::of(f.get(i, 0) + b, slope);
            g[i][0] = v;
            q[i][0] = (h[0] - xv) * slope;
            h[0] = G::pass(v, h[0]) + G::take(v) * xv;
        }
    } else {
#pragma unroll
        for (int i = 0; i < kSpan; i++) {
            const float xv = x.get(i, 0), v = G::of(f.get(i, 0) + b, slope);
            g[i][0] = v;
            q[i][0] = ((rm >> i & 1 ? 0.f : h[0]) - xv) * slope;
            h[0] = G::pass(with_reset<kExact>(v, rm, i), h[0]) + G::take(v) * xv;
        }
    }
    if (any_not_finite(h)) {
        // the inputs once more from memory: kept for this, they would cost 32 registers
        const char *fp = step_base(a.f, at, t0), *xp = step_base(a.x, at, t0);
        const int64_t fstep = distance(a.f), xstep = distance(a.x);
        const unsigned fo = lane_offset(a.f, at), xo = lane_offset(a.x, at);
        h[0] = kept;
#pragma unroll
        for (int i = 0; i < kSpan; i++, fp += fstep, xp += xstep) {
            if (i < n) {
                const float xv = widen<T>(Raw<T, 1>::one(xp + here(xo))), v = G::of(widen<T>(Raw<T, 1>::one(fp + here(fo))) + b, slope);
                if (anew(rm) >> i & 1) h[0] = 0.f;
                g[i][0] = v;
                q[i][0] = (h[0] - xv) * slope;
                h[0] = G::pass_any(v, h[0]) + G::take(v) * xv;
            }
        }
    }
    if (n < kSpan)
#pragma unroll
        for (int i = 0; i < kSpan; i++)
            if (i >= n) g[i][0] = G::open(), q[i][0] = 0.f;
}

// Walks a span back from gradient `in`, writes df and dx and adds up df.
template <class T>
__device__ inline void back_span(const BackwardArgs<T> &a, const Place &at, unsigned dfo, unsigned dxo, int64_t t0, int n, unsigned rm,
                                 const Span<1> &g, const Span<1> &q, const Raw<T, 1> &dy, float &in, double &total) {
    typedef Gate<sizeof(T) == 4> G;
    if (!at.mine) return;
    char *fp = nullptr, *xp = nullptr;
    const int64_t fstep = distance(a.df), xstep = distance(a.dx);
    auto put = [&](int i, float of, float ox) {
        fp = i == kSpan - 1 ? step_base(a.df, at, t0 + kSpan - 1) : fp - fstep;
        xp = i == kSpan - 1 ? step_base(a.dx, at, t0 + kSpan - 1) : xp - xstep;
        const float f1[1] = {of}, x1[1] = {ox};
        if (i < n) {
            Lane<T, 1>::store(fp + here(dfo), f1);
            Lane<T, 1>::store(xp + here(dxo), x1);
        }
    };
    constexpr bool kExact = sizeof(T) == 4;
    float sum = 0.f, c[1] = {in};
    bool done = false;
    if (n >= kSpan) {
        n = kSpan;
        if (!__any(rm != 0)) {
#pragma unroll
            for (int i = kSpan - 1; i >= 0; i--) {
                const float gs = dy.get(i, 0) + c[0], of = gs * q[i][0];
                sum += of;
                put(i, of, G::take(g[i][0]) * gs);
                c[0] = G::pass(g[i][0], gs);
            }
        } else {
#pragma unroll
            for (int i = kSpan - 1; i >= 0; i--) {
                const float gs = dy.get(i, 0) + c[0], of = gs * q[i][0];
                sum += of;
                put(i, of, G::take(g[i][0]) * gs);
                c[0] = G::pass(with_reset<kExact>(g[i][0], rm, i), gs);
            }
        }
        done = !any_not_finite(c);
    }
    if (!done) {
        sum = 0.f;
        c[0] = in;
#pragma unroll
        for (int i = kSpan - 1; i >= 0; i--) {
            const float v = anew(g[i][0]), gs = dy.get(i, 0) + c[0], of = gs * q[i][0];
            if (i < n) sum += of;
            put(i, of, G::take(v) * gs);
            c[0] = anew(rm) >> i & 1 ? 0.f : G::pass_any(v, gs);
        }
    }
    in = c[0];
    total += (double)sum;
    if (a.dh0 && t0 == 0) a.dh0[at.c] = in;
}

// a workgroup's sums of df per column, the waves' in wave order
template <int W>
__device__ inline void dbias_row(float *row, const Place &at, int nw, double total, double (&sums)[W][64]) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    sums[w][lane] = total;
    __syncthreads();
    if (w == 0 && at.mine) {
        double s = 0.0;
        for (int i = 0; i < nw; i++) s += sums[i][lane];
        row[at.c] = (float)s;
    }
}

// A wave walks spans end-1 .. first of its columns back from gradient `in` and adds up df.
template <class T>
__device__ inline void backward_walk(const BackwardArgs<T> &a, const Place &at, int64_t first, int64_t end, float (&in)[1], double (&total)[1]) {
    const unsigned fo = lane_offset(a.f, at), xo = lane_offset(a.x, at), go = lane_offset(a.dy, at), dfo = lane_offset(a.df, at), dxo = lane_offset(a.dx, at);
    const float b = a.bias ? a.bias[at.j] : 0.f;
    Raw<T, 1> fr, xr, gr;
    float kept;
    auto fetch = [&](int64_t s) {
        const int64_t t0 = s * kSpan;
        const int n = (int)(a.T_ - t0 < kSpan ? a.T_ - t0 : kSpan);
        fr.load(a.f, at, fo, t0, n);
        xr.load(a.x, at, xo, t0, n);
        kept = a.saved[s * a.C + at.c];
    };
    if (first < end) fetch(end - 1);
    for (int64_t s = end - 1; s >= first; s--) {
        const int64_t t0 = s * kSpan;
        const int n = (int)(a.T_ - t0 < kSpan ? a.T_ - t0 : kSpan);
        gr.load(a.dy, at, go, t0, n);
        const unsigned rm = span_resets(a.resets, t0, n, at);
        Span<1> g, q;
        back_open<T>(a, at, fr, xr, b, kept, t0, n, rm, g, q);
        if (s > first) fetch(s - 1);
        back_span<T>(a, at, dfo, dxo, t0, n, rm, g, q, gr, in[0], total[0]);
    }
}

// Many 16-bit columns: a wave per tile.  [2048, 512, 256] bfloat16, 2.7 GB in 665 us (4.1 TB/s).
template <class T>
__global__ __launch_bounds__(64, 2) void glr_backward_kernel(BackwardArgs<T> a) {
    const Place at = place_of<1>(seat_of(blockIdx.x), a.C, a.H, a.env_tiles);
    float in[1] = {a.dh_last ? a.dh_last[at.c] : 0.f};
    double total[1] = {0.0};
    backward_walk<T>(a, at, 0, (a.T_ + kSpan - 1) / kSpan, in, total);
    if (a.dbias_rows && at.mine) a.dbias_rows[at.c] = (float)total[0];
}

// [128, 512, 256] float32, 340 MB in 69 us (4.9 TB/s).
template <class T>
__global__ __launch_bounds__(64 * kHeld) void glr_backward_held_kernel(BackwardArgs<T> a) {
    __shared__ RunSpace<sizeof(T) == 4, 1> runs[kHeld];
    __shared__ double sums[kHeld][64];
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), nw = blockDim.x >> 6;
    const Place at = place_of<1>(seat_of(blockIdx.x), a.C, a.H, a.env_tiles);
    const int64_t t0 = (int64_t)w * kSpan;
    const int n = (int)(a.T_ - t0 < kSpan ? a.T_ - t0 : kSpan);
    Raw<T, 1> fr, xr, gr;
    fr.load(a.f, at, lane_offset(a.f, at), t0, n);
    xr.load(a.x, at, lane_offset(a.x, at), t0, n);
    gr.load(a.dy, at, lane_offset(a.dy, at), t0, n);
    const unsigned rm = span_resets(a.resets, t0, n, at);
    const float b = a.bias ? a.bias[at.j] : 0.f, kept = a.saved[(int64_t)w * a.C + at.c];
    float in[1] = {a.dh_last ? a.dh_last[at.c] : 0.f};
    double total[1] = {0.0};
    Span<1> g, q;
    Run<sizeof(T) == 4> r[1];
    back_open<T>(a, at, fr, xr, b, kept, t0, n, rm, g, q);
    span_run_back<T>(g, gr, rm, r);
    runs[w].put(r);
    __syncthreads();
    for (int i = nw - 1; i > w; i--) in[0] = runs[i].get(0).through(in[0]);
    back_span<T>(a, at, lane_offset(a.df, at), lane_offset(a.dx, at), t0, n, rm, g, q, gr, in[0], total[0]);
    if (a.dbias_rows) dbias_row<kHeld>(a.dbias_rows, at, nw, total[0], sums);
}

// 54 operations per element (95 us of all SIMDs for 67 M elements) beside five streams, two workgroups per CU: [16384, 4, 1024]
// bfloat16, 688 MB in 185 us (3.7 TB/s).  At 6 waves per SIMD its span no longer fits the registers (40 us slower).
template <class T>
__global__ __launch_bounds__(64 * kChainWaves, 4) void glr_backward_chain_kernel(BackwardArgs<T> a, Chain ch) {
    __shared__ ChainSpace<sizeof(T) == 4, 1> mem;
    __shared__ double sums[kChainWaves][64];
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Drawn d = draw<true, 1>(a, ch, mem.turn, w);
    Raw<T, 1> fr, xr, gr;
    fr.load(a.f, d.at, lane_offset(a.f, d.at), d.t0, d.n);
    xr.load(a.x, d.at, lane_offset(a.x, d.at), d.t0, d.n);
    gr.load(a.dy, d.at, lane_offset(a.dy, d.at), d.t0, d.n);
    const unsigned rm = span_resets(a.resets, d.t0, d.n, d.at);
    const float b = a.bias ? a.bias[d.at.j] : 0.f, kept = d.n > 0 ? a.saved[d.t0 / kSpan * a.C + d.at.c] : 0.f;
    float in[1] = {a.dh_last ? a.dh_last[d.at.c] : 0.f};
    double total[1] = {0.0};
    Span<1> g, q;
    Run<sizeof(T) == 4> r[1];
    back_open<T>(a, d.at, fr, xr, b, kept, d.t0, d.n, rm, g, q);
    span_run_back<T>(g, gr, rm, r);
    chain_through<sizeof(T) == 4, true, 1>(ch, mem, a.C, d.at, d.order, w, r, in);
    if (d.n > 0) back_span<T>(a, d.at, lane_offset(a.df, d.at), lane_offset(a.dx, d.at), d.t0, d.n, rm, g, q, gr, in[0], total[0]);
    if (a.dbias_rows) dbias_row<kChainWaves>(a.dbias_rows + (int64_t)d.batch * a.C, d.at, kChainWaves, total[0], sums);
}

// One step: every thread V channels, nothing to share.  [2048, 256] float32, 10.5 MB in 4 us, of which a launch of nothing takes 3.5.
template <class T, int V>
__global__ __launch_bounds__(256) void glr_step_kernel(Seq<const T> f, Seq<const T> x, const float *__restrict__ bias, Seq<const uint8_t> resets,
                                                       const float *h0, unsigned C, unsigned H, Seq<T> y, float *h_last, float *__restrict__ saved) {
    typedef Gate<sizeof(T) == 4> G;
    const uint64_t at = ((uint64_t)blockIdx.x * 256 + threadIdx.x) * V;
    if (at >= C) return;
    const unsigned c = (unsigned)at, e = c / H, j = c - e * H;
    typedef Raw<T, V> In;
    In in;
    in.v[0] = In::one((const char *)(f.p + (int64_t)e * f.e + j)), in.v[1] = In::one((const char *)(x.p + (int64_t)e * x.e + j));
    const bool fresh = resets.p && resets.p[(int64_t)e * resets.e];
    float h[V];
#pragma unroll
    for (int k = 0; k < V; k++) {
        h[k] = h0 ? h0[c + k] : 0.f;
        if (saved) saved[c + k] = h[k];
        if (fresh) h[k] = 0.f;
        const float g = G::of(in.get(0, k) + (bias ? bias[j + k] : 0.f));
        h[k] = G::pass_any(g, h[k]) + G::take(g) * in.get(1, k);
    }
    Lane<T, V>::store(y.p + (int64_t)e * y.e + j, h);
    if (h_last)
#pragma unroll
        for (int k = 0; k < V; k++) h_last[c + k] = h[k];
}

// Column sums of in [rows, H]: a workgroup sums kSumRows rows of 32 columns, 32 rows side by side, into a row of out.  One launch for
// up to 2048 rows: [512, 256] 4.7 us.
constexpr int kSumRows = 2048;
__global__ __launch_bounds__(1024) void glr_column_sum_kernel(const float *__restrict__ in, int64_t rows, int H, float *__restrict__ out) {
    __shared__ double red[32][33];
    const unsigned across = (unsigned)(H + 31) / 32, part = blockIdx.x / across;
    const int col = threadIdx.x & 31, grp = threadIdx.x >> 5, j = (int)(blockIdx.x - part * across) * 32 + col;
    const int64_t r0 = (int64_t)part * kSumRows, r1 = r0 + kSumRows < rows ? r0 + kSumRows : rows;
    double s = 0.0;
    if (j < H)
#pragma unroll 8
        for (int64_t r = r0 + grp; r < r1; r += 32) s += (double)in[r * H + j];
    red[grp][col] = s;
    __syncthreads();
    if (threadIdx.x < 32 && j < H) {
        s = 0.0;
#pragma unroll
        for (int g = 0; g < 32; g++) s += red[g][col];
        out[(int64_t)part * H + j] = (float)s;
    }
}

__global__ void glr_copy_state_kernel(const float *src, float *dst, int64_t n) {
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i < n) dst[i] = src ? src[i] : 0.f;
}

}  // namespace ppo2hip

using namespace ppo2hip;

constexpr int64_t kWalkTiles = 1280;      // tiles of a 16-bit sequence from which a wave walks back over all of its columns' steps

template <class T>
static Seq<T> seq_of(const ppo2hip_seq *s) {
    return s ? Seq<T>{(T *)s->data, s->t, s->e} : Seq<T>{nullptr, 0, 0};
}

static int glr_check(const char *what, int dtype, int T, int E, int H) {
    PPO2HIP_REQUIRE(dtype == PPO2HIP_F32 || dtype == PPO2HIP_BF16 || dtype == PPO2HIP_F16, "%s: unknown dtype %d", what, dtype);
    PPO2HIP_REQUIRE(T >= 0 && E >= 0 && H >= 0, "%s: negative size T=%d E=%d H=%d", what, T, E, H);
    PPO2HIP_REQUIRE((int64_t)E * H <= 0x7fffffffll, "%s: E*H=%lld beyond 2^31 - 1 columns", what, (long long)E * H);
    PPO2HIP_REQUIRE(H < 1 << 26, "%s: H=%d beyond 2^26 - 1 channels", what, H);           // lanes' offsets and launches stay within 32 bits
    return PPO2HIP_OK;
}

static int glr_check_seq(const char *what, const char *name, const ppo2hip_seq *s) {
    PPO2HIP_REQUIRE(s && s->data, "%s: %s is null", what, name);
    PPO2HIP_REQUIRE(s->t >= 0 && s->e >= 0, "%s: %s has a negative stride", what, name);
    return PPO2HIP_OK;
}

static int copy_state(const float *src, float *dst, int64_t n, hipStream_t s) {
    if (!dst || dst == src || n == 0) return PPO2HIP_OK;
    hipLaunchKernelGGL(glr_copy_state_kernel, dim3((unsigned)ceil_div(n, 256)), dim3(256), 0, s, src, dst, n);
    return check_launch("glr_copy_state_kernel");
}

extern "C" int64_t ppo2hip_glr_saved_floats(int T, int E, int H) {
    if (T < 0 || E < 0 || H < 0) return 0;
    return ceil_div(T, kSpan) * (int64_t)E * H;
}

// How a call is cut: tiles of 64 V columns (V channels per lane), and the time axis held by one workgroup per tile (up to 256 steps),
// passed along a chain of workgroups, or, back over many 16-bit columns, walked by one wave per tile, which has no exchange and keeps
// 3 waves per SIMD loading.  Measured, us:
//   held and chain, forward / backward: [128, 1024 x 64] float32 20 / 36 and 23 / 39, [128, 768 x 64] bfloat16 12 / 23 and 16 / 26,
//   [256, 1279 x 64] 32 / 61 and 31 / 59
//   bfloat16 backward, held and walked: [128, E, H] of 768 x 64 columns 23 and 31, 1279 x 64: 32 and 37, 1536 x 64: 37 and 40,
//   2048 x 64: 45 and 48, 8192 x 64: 201 and 193; [256, E, H] 1279 x 64: 61 and 62, 1536 x 64: 72 and 67, 4096 x 64: 200 and 191
//   chain and walked: [2048, E, H] 768 x 64: 275 and 370, 1279 x 64: 449 and 446, 1536 x 64: 542 and 488, 4096 x 64: 1415 and 1380
struct Cut {
    enum { kHold, kWalk, kChain } how;
    int V, env_tiles, batches, words;        // words of a run
    int64_t tiles;
};
static Cut cut_of(int dtype, int T, int E, int H, bool back) {
    Cut k;
    const int64_t C = (int64_t)E * H;
    const int wide = dtype != PPO2HIP_F32 && H % 2 == 0 ? 2 : 1;
    const bool walk = back && dtype != PPO2HIP_F32 && ceil_div(C, 64) >= kWalkTiles;
    k.how = walk ? Cut::kWalk : T <= kHeld * kSpan ? Cut::kHold : Cut::kChain;
    // two channels per lane halve a 16-bit sequence's loads and double what is in flight; going back there are no registers for them
    k.V = back ? 1 : wide;
    k.tiles = ceil_div(C, 64 * k.V);
    k.env_tiles = 0;
    k.words = dtype == PPO2HIP_F32 ? Run<true>::kWords : Run<false>::kWords;
    k.batches = k.how == Cut::kChain ? (int)ceil_div(T, kBatch) : 1;
    return k;
}
// Lanes of a tile in a row reach over up to 64 V / H envs behind the first: their offsets must fit 31 bits in every array,
// else each env gets tiles of its own (lanes behind H idle there).
static void place_envs(Cut &k, int E, int H, std::initializer_list<const ppo2hip_seq *> seqs) {
    int64_t reach = (64 * k.V - 1) / H + 1;
    if (reach > E - 1) reach = E - 1;
    bool far = false;
    for (const ppo2hip_seq *s : seqs) far |= s && reach > 0 && s->e > ((1ll << 29) - 1 - H) / reach;
    if (!far) return;
    k.env_tiles = (int)ceil_div(H, 64 * k.V);
    k.tiles = (int64_t)E * k.env_tiles;
}

static unsigned threads_of(const Cut &k, int T) {
    return 64 * (unsigned)(k.how == Cut::kHold ? ceil_div(T, kSpan) : k.how == Cut::kChain ? kChainWaves : 1);
}
static int cut_check(const char *what, const Cut &k, int T, int64_t C) {
    PPO2HIP_REQUIRE(k.tiles * k.batches <= (int64_t)(0xffffffffu / threads_of(k, T)), "%s: T=%d, %lld columns: beyond one launch", what, T, (long long)C);
    PPO2HIP_REQUIRE(k.how != Cut::kChain || C < 1ll << 30, "%s: T=%d, %lld columns: beyond 2^30 - 1 for so many steps", what, T, (long long)C);
    return PPO2HIP_OK;
}

// words of a chain behind its counters
static int64_t chain_words(const Cut &k, int64_t C) {
    const int64_t groups = ceil_div(k.batches, kChainWaves), blocks = ceil_div(groups, kChainWaves);
    return (k.words * (k.batches + groups) + blocks) * C;
}
static size_t chain_bytes(const Cut &k, int64_t C) { return k.how == Cut::kChain ? kTurnBytes + align_up((size_t)chain_words(k, C) * sizeof(float), 256) : 0; }
static int chain_begin(const Cut &k, int64_t C, void *workspace, Chain &ch, hipStream_t s) {
    ch.turn = (unsigned *)workspace;
    ch.runs = (float *)((char *)workspace + kTurnBytes);
    ch.groups = ch.runs + (int64_t)k.words * k.batches * C;
    ch.states = ch.groups + k.words * (int64_t)ceil_div(k.batches, kChainWaves) * C;
    ch.tiles = (unsigned)k.tiles;
    ch.batches = k.batches;
    // polls before a waiting wave gives up, about a second; PPO2HIP_GRID_SYNC_SPINS overrides it (negative: the first poll already counts as given up)
    static const int spins = getenv("PPO2HIP_GRID_SYNC_SPINS") ? atoi(getenv("PPO2HIP_GRID_SYNC_SPINS")) : (1 << 20);
    ch.max_spins = spins;
    ch.fault = fault_word();
    if (!ch.fault) return PPO2HIP_EINVAL;
    const int64_t words = chain_words(k, C);
    hipLaunchKernelGGL(glr_chain_clear_kernel, dim3((unsigned)ceil_div(words, 1024)), dim3(256), 0, s, ch, words);
    return check_launch("glr_chain_clear_kernel");
}

extern "C" size_t ppo2hip_glr_forward_workspace_bytes(int dtype, int T, int E, int H) {
    if (T <= 1 || E <= 0 || H <= 0) return 0;
    return chain_bytes(cut_of(dtype, T, E, H, false), (int64_t)E * H);
}

extern "C" size_t ppo2hip_glr_backward_workspace_bytes(int dtype, int T, int E, int H, int want_dbias) {
    if (T <= 0 || E <= 0 || H <= 0) return 0;
    const Cut k = cut_of(dtype, T, E, H, true);
    const int64_t C = (int64_t)E * H, rows = (int64_t)k.batches * E;
    size_t n = chain_bytes(k, C);
    if (want_dbias) n += align_up((size_t)rows * H * sizeof(float), 256) + align_up((size_t)ceil_div(rows, kSumRows) * H * sizeof(float), 256);
    return n;
}

template <class T, int V>
static int forward_of(const Cut &k, const ppo2hip_seq *f, const ppo2hip_seq *x, const float *bias, const ppo2hip_seq *resets, const float *h0,
                      const ppo2hip_seq *y, float *h_last, float *saved, void *workspace, int T_, int E, int H, hipStream_t s) {
    const int64_t C = (int64_t)E * H;
    if (T_ == 1) {
        hipLaunchKernelGGL((glr_step_kernel<T, V>), dim3((unsigned)ceil_div(C, 256 * V)), dim3(256), 0, s, seq_of<const T>(f), seq_of<const T>(x),
                           bias, seq_of<const uint8_t>(resets), h0, (unsigned)C, (unsigned)H, seq_of<T>(y), h_last, saved);
        return check_launch("glr_step_kernel");
    }
    const ForwardArgs<T> a = {seq_of<const T>(f), seq_of<const T>(x), seq_of<const uint8_t>(resets), seq_of<T>(y), bias, h0, h_last, saved,
                              T_, (unsigned)C, (unsigned)H, (unsigned)k.env_tiles};
    if (k.how == Cut::kHold) {
        hipLaunchKernelGGL((glr_forward_held_kernel<T, V>), dim3((unsigned)k.tiles), dim3(threads_of(k, T_)), 0, s, a);
        return check_launch("glr_forward_held_kernel");
    }
    Chain ch;
    int rc = chain_begin(k, C, workspace, ch, s);
    if (rc) return rc;
    hipLaunchKernelGGL((glr_forward_chain_kernel<T, V>), dim3((unsigned)(k.tiles * k.batches)), dim3(64 * kChainWaves), 0, s, a, ch);
    return check_launch("glr_forward_chain_kernel");
}

extern "C" int ppo2hip_glr_forward(int dtype, int T, int E, int H, const ppo2hip_seq *f, const ppo2hip_seq *x, const float *bias,
                                   const ppo2hip_seq *resets, const float *h0, const ppo2hip_seq *y, float *h_last, float *saved,
                                   void *workspace, size_t workspace_bytes, void *stream) {
    int rc = glr_check("glr_forward", dtype, T, E, H);
    if (rc) return rc;
    const int64_t C = (int64_t)E * H;
    hipStream_t s = (hipStream_t)stream;
    if (C == 0) return PPO2HIP_OK;
    if (T == 0) return copy_state(h0, h_last, C, s);
    if ((rc = glr_check_seq("glr_forward", "f", f)) || (rc = glr_check_seq("glr_forward", "x", x)) || (rc = glr_check_seq("glr_forward", "y", y)))
        return rc;
    if (resets && (rc = glr_check_seq("glr_forward", "resets", resets))) return rc;
    PPO2HIP_REQUIRE(T == 1 || !h_last || h_last != h0, "glr_forward: h_last may be h0 for a single step only");
    if (workspace_bytes < ppo2hip_glr_forward_workspace_bytes(dtype, T, E, H)) {
        set_error("glr_forward: workspace of %zu bytes is too small", workspace_bytes);
        return PPO2HIP_ENOSPACE;
    }
    Cut k = cut_of(dtype, T, E, H, false);
    place_envs(k, E, H, {f, x, resets, y});
    if ((rc = cut_check("glr_forward", k, T, C))) return rc;
    PPO2HIP_REQUIRE(T == 1 || chain_bytes(k, C) == 0 || workspace, "glr_forward: workspace is null");
    PPO2HIP_REQUIRE((uintptr_t)workspace % 16 == 0, "glr_forward: workspace must be aligned to 16 bytes");
#define PPO2HIP_GLR_FORWARD(type, V) forward_of<type, V>(k, f, x, bias, resets, h0, y, h_last, saved, workspace, T, E, H, s)
    if (dtype == PPO2HIP_F32) return PPO2HIP_GLR_FORWARD(float, 1);
    if (dtype == PPO2HIP_BF16) return k.V == 2 ? PPO2HIP_GLR_FORWARD(__bf16, 2) : PPO2HIP_GLR_FORWARD(__bf16, 1);
    return k.V == 2 ? PPO2HIP_GLR_FORWARD(_Float16, 2) : PPO2HIP_GLR_FORWARD(_Float16, 1);
#undef PPO2HIP_GLR_FORWARD
}

extern "C" int ppo2hip_glr_step(int dtype, int E, int H, const void *f, int64_t f_e, const void *x, int64_t x_e, const float *bias,
                                const uint8_t *resets, int64_t resets_e, float *state, void *y, int64_t y_e, void *stream) {
    PPO2HIP_REQUIRE(state || (int64_t)E * H == 0, "glr_step: state is null");
    const ppo2hip_seq fs = {(void *)f, 0, f_e}, xs = {(void *)x, 0, x_e}, ys = {y, 0, y_e}, rs = {(void *)resets, 0, resets_e};
    return ppo2hip_glr_forward(dtype, 1, E, H, &fs, &xs, bias, resets ? &rs : nullptr, state, &ys, state, nullptr, nullptr, 0, stream);
}

template <class T>
static int backward_of(const Cut &k, const ppo2hip_seq *f, const ppo2hip_seq *x, const float *bias, const ppo2hip_seq *resets, const float *saved,
                       const ppo2hip_seq *dy, const float *dh_last, const ppo2hip_seq *df, const ppo2hip_seq *dx, float *dbias, float *dh0,
                       void *workspace, int T_, int E, int H, hipStream_t s) {
    const int64_t C = (int64_t)E * H, rows = (int64_t)k.batches * E;
    float *sums = (float *)((char *)workspace + chain_bytes(k, C));
    const BackwardArgs<T> a = {seq_of<const T>(f), seq_of<const T>(x), seq_of<const T>(dy), seq_of<const uint8_t>(resets), seq_of<T>(df), seq_of<T>(dx),
                               bias, saved, dh_last, dbias ? sums : nullptr, dh0, T_, (unsigned)C, (unsigned)H, (unsigned)k.env_tiles};
    int rc;
    if (k.how == Cut::kHold) {
        hipLaunchKernelGGL((glr_backward_held_kernel<T>), dim3((unsigned)k.tiles), dim3(threads_of(k, T_)), 0, s, a);
        rc = check_launch("glr_backward_held_kernel");
    } else if (k.how == Cut::kChain) {
        Chain ch;
        if ((rc = chain_begin(k, C, workspace, ch, s))) return rc;
        hipLaunchKernelGGL((glr_backward_chain_kernel<T>), dim3((unsigned)(k.tiles * k.batches)), dim3(64 * kChainWaves), 0, s, a, ch);
        rc = check_launch("glr_backward_chain_kernel");
    } else {
        if constexpr (sizeof(T) == 2) hipLaunchKernelGGL((glr_backward_kernel<T>), dim3((unsigned)k.tiles), dim3(64), 0, s, a);
        rc = check_launch("glr_backward_kernel");
    }
    if (rc || !dbias) return rc;
    // rows [batch][env] of H channels each, kSumRows of them to a workgroup, until one row is left
    float *in = sums, *out = (float *)((char *)sums + align_up((size_t)rows * H * sizeof(float), 256));
    for (int64_t n = rows;;) {
        const int64_t left = ceil_div(n, kSumRows);
        hipLaunchKernelGGL(glr_column_sum_kernel, dim3((unsigned)(ceil_div(H, 32) * left)), dim3(1024), 0, s, in, n, H, left == 1 ? dbias : out);
        if ((rc = check_launch("glr_column_sum_kernel")) || left == 1) return rc;
        float *t = in;
        in = out, out = t, n = left;
    }
}

extern "C" int ppo2hip_glr_backward(int dtype, int T, int E, int H, const ppo2hip_seq *f, const ppo2hip_seq *x, const float *bias,
                                    const ppo2hip_seq *resets, const float *saved, const ppo2hip_seq *dy, const float *dh_last,
                                    const ppo2hip_seq *df, const ppo2hip_seq *dx, float *dbias, float *dh0, void *workspace,
                                    size_t workspace_bytes, void *stream) {
    int rc = glr_check("glr_backward", dtype, T, E, H);
    if (rc) return rc;
    const int64_t C = (int64_t)E * H;
    hipStream_t s = (hipStream_t)stream;
    if (C == 0 || T == 0) {
        if (dbias && H && (rc = copy_state(nullptr, dbias, H, s))) return rc;
        return C ? copy_state(dh_last, dh0, C, s) : PPO2HIP_OK;
    }
    const char *what = "glr_backward";
    if ((rc = glr_check_seq(what, "f", f)) || (rc = glr_check_seq(what, "x", x)) || (rc = glr_check_seq(what, "dy", dy)) ||
        (rc = glr_check_seq(what, "df", df)) || (rc = glr_check_seq(what, "dx", dx)))
        return rc;
    if (resets && (rc = glr_check_seq(what, "resets", resets))) return rc;
    PPO2HIP_REQUIRE(saved, "glr_backward: saved is null");
    PPO2HIP_REQUIRE(!dh0 || dh0 != dh_last, "glr_backward: dh0 may not be dh_last");
    if (workspace_bytes < ppo2hip_glr_backward_workspace_bytes(dtype, T, E, H, dbias != nullptr)) {
        set_error("glr_backward: workspace of %zu bytes is too small", workspace_bytes);
        return PPO2HIP_ENOSPACE;
    }
    Cut k = cut_of(dtype, T, E, H, true);
    place_envs(k, E, H, {f, x, resets, dy, df, dx});
    if ((rc = cut_check("glr_backward", k, T, C))) return rc;
    PPO2HIP_REQUIRE((!dbias && chain_bytes(k, C) == 0) || workspace, "glr_backward: workspace is null");
    PPO2HIP_REQUIRE((uintptr_t)workspace % 16 == 0, "glr_backward: workspace must be aligned to 16 bytes");
#define PPO2HIP_GLR_BACKWARD(type) backward_of<type>(k, f, x, bias, resets, saved, dy, dh_last, df, dx, dbias, dh0, workspace, T, E, H, s)
    if (dtype == PPO2HIP_F32) return PPO2HIP_GLR_BACKWARD(float);
    if (dtype == PPO2HIP_BF16) return PPO2HIP_GLR_BACKWARD(__bf16);
    return PPO2HIP_GLR_BACKWARD(_Float16);
#undef PPO2HIP_GLR_BACKWARD
}
