// Gated linear recurrence over a time-major sequence, forward and backward:
//   a = sigmoid(f + bias)   p = reset ? 0 : h[t-1]   h[t] = a p + (1 - a) x[t]
//   g[t] = dy[t] + (reset[t+1] ? 0 : a[t+1] g[t+1])   dx = (1 - a) g   df = g (p - x) a (1 - a)
// The backward pass recomputes the states from float32 states kept every PPO2HIP_GLR_SPAN steps: they cost
// 4 / SPAN bytes per element where reading y back costs its whole width, and y is rounded to its type while p - x cancels.
#include <initializer_list>
#include <type_traits>

#include "kernels.hpp"

// Products and sums round one by one unless fmaf says otherwise: the same step written in two places gives the same bits, so
// that a state recomputed in the backward pass is the forward's, and a span walked the slow way changes no other column.
#pragma clang fp contract(off)

namespace ppo2hip {

constexpr int kSpan = PPO2HIP_GLR_SPAN;                     // steps a wave holds in registers at a time
constexpr int kWaves = 4;                                   // waves of a workgroup that walk
constexpr int kHeld = 16;                                   // spans that a workgroup can hold at once, one per wave

// ---------------------------------------------------------------------------------------------------------------------
// gates
// ---------------------------------------------------------------------------------------------------------------------

// How a step's gate is held between the passes over a span, by the sequence's type.
//   16 bits: om = 1 - a itself.  a v is v - om v: off by 2^-25 of v at most, which shows in 16 bits only where a single step shrinks
//   the state by 2^13 and more.  The rounding of the exponent and of the reciprocal stay.
//   float32: the smaller side s = min(a, 1 - a) <= 1/2, negated where that is 1 - a (a >= 1/2, by the sign bit, -0 included): both
//   sides keep their relative accuracy, and what the exponent's product and the reciprocal round is made good.
// Either way 1 - a is never taken from a rounded a: it would lose the memory's length as soon as a is near one.
// slope: a (1 - a), the gate's derivative.
template <bool EXACT>
struct Gate;

template <>
struct Gate<true> {
    static __device__ inline float of(float z) {
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
    static __device__ inline float of(float z, float &slope) {
        const float v = of(z);
        slope = fabsf(v) * (1.f - fabsf(v));
        return v;
    }
    static __device__ inline bool keeps(float v) { return (int)__float_as_uint(v) < 0; }
    static __device__ inline float take(float v) { return keeps(v) ? -v : 1.f - v; }                 // 1 - a
    static __device__ inline float pass(float v, float h) { return fmaf(v, h, keeps(v) ? h : 0.f); } // a h
    static __device__ inline float pass_any(float v, float h) {                                     // where h may not be finite
        return fabsf(h) < INFINITY ? pass(v, h) : (keeps(v) ? 1.f + v : v) * h;
    }
    static __device__ inline float open() { return -0.f; }  // a = 1
    static __device__ inline float shut() { return 0.f; }   // a = 0
};

template <>
struct Gate<false> {
    static __device__ inline float of(float z) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z * 1.44269502f)); }
    static __device__ inline float of(float z, float &slope) {
        const float e = __builtin_amdgcn_exp2f(fabsf(z) * -1.44269502f), r = __builtin_amdgcn_rcpf(1.f + e), s = e * r;
        slope = s * r;                                      // from the smaller side: 1 - om has no figures left where a is small
        return z >= 0.f ? s : r;                            // a NaN is one on both sides
    }
    static __device__ inline float take(float v) { return v; }
    static __device__ inline float pass(float v, float h) { return fmaf(-v, h, h); }
    static __device__ inline float pass_any(float v, float h) { return fabsf(h) < INFINITY ? pass(v, h) : (1.f - v) * h; }
    static __device__ inline float open() { return 0.f; }
    static __device__ inline float shut() { return 1.f; }
};

// ---------------------------------------------------------------------------------------------------------------------
// runs of steps
// ---------------------------------------------------------------------------------------------------------------------

// What a run of steps does to the state that enters it: h -> A h + B, with D = 1 - A kept beside A because a product of gates
// next to one has lost D's figures; A < 0 marks a run with a reset in it, which lets nothing through, infinities and NaN included.
// Going back in time the same three numbers carry the gradient that leaves a run at its front.
struct Run {
    float A, D, B;
};
__device__ inline float run_through(const Run &r, float h) {
    if (r.A < 0.f) return r.B;
    const float kept = r.D <= 0.5f ? fmaf(-r.D, h, h) : r.A * h;
    return (fabsf(h) < INFINITY ? kept : h) + r.B;         // an infinite state stays one however small A became
}
__device__ inline Run run_join(const Run &first, const Run &then) {
    return {then.A < 0.f || first.A < 0.f ? -1.f : first.A * then.A, fmaf(1.f - first.D, then.D, first.D), run_through(then, first.B)};
}

// ---------------------------------------------------------------------------------------------------------------------
// addresses
// ---------------------------------------------------------------------------------------------------------------------

template <class T>
struct Seq {
    T *p;
    int64_t t, e;
};

// V neighbouring channels of one step, at any address an element may have
template <class T, int V>
struct Lane {
    typedef T Vec __attribute__((ext_vector_type(V)));
    typedef Vec Any __attribute__((aligned(sizeof(T))));
    static __device__ inline Vec load(const void *p) { return *(const Any *)p; }
    static __device__ inline void store(void *p, const float (&v)[V]) {
        Vec r;
#pragma unroll
        for (int k = 0; k < V; k++) r[k] = (T)v[k];       // to nearest: the type that the layer hands on; states stay float32
        *(Any *)p = r;
    }
};

// Which columns a wave works on.  Addresses are a wave-uniform 64-bit part (step, the wave's first env) and a 32-bit part
// per lane: kept as 64 bits per lane and step they cost 2 registers each and the kernels spill.
struct Place {
    unsigned c;         // the lane's first column e * H + j
    int e0, de, j;      // first env of the wave, lane's env less that, channel
    bool mine;          // false: a lane behind the last column, which repeats it and writes nothing
};
// env_tiles 0: columns in a row over all envs.  Else that many tiles per env, where envs lie too far apart for 32 bits.
template <int V>
__device__ inline Place place_of(unsigned C, unsigned H, unsigned env_tiles) {
    const unsigned lane = threadIdx.x & 63;
    Place p;
    if (env_tiles == 0) {
        const uint64_t c = ((uint64_t)blockIdx.x * 64 + lane) * V;
        p.mine = c < C;
        p.c = p.mine ? (unsigned)c : C - V;
        const unsigned e = p.c / H;
        p.e0 = __builtin_amdgcn_readfirstlane(e);
        p.de = (int)e - p.e0;
        p.j = (int)(p.c - e * H);
    } else {
        const unsigned e = blockIdx.x / env_tiles, j = ((blockIdx.x - e * env_tiles) * 64 + lane) * V;
        p.mine = j < H;
        p.j = (int)(p.mine ? j : H - V);
        p.e0 = (int)e;
        p.de = 0;
        p.c = e * H + (unsigned)p.j;
    }
    return p;
}
template <class T>
__device__ inline unsigned lane_offset(const Seq<T> &s, const Place &at) {
    return (unsigned)(at.de * (int)s.e + at.j) * (unsigned)sizeof(T);
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
    typename Lane<T, V>::Vec v[kSpan];
    __device__ inline void load(const Seq<const T> &s, const Place &at, unsigned off, int64_t t0, int n) {
        const char *p = step_base(s, at, t0);
        const int64_t step = distance(s);
        if (n >= kSpan) {
#pragma unroll
            for (int i = 0; i < kSpan; i++, p += step) v[i] = Lane<T, V>::load(p + off);
        } else {
#pragma unroll
            for (int i = 0; i < kSpan; i++, p += step) {
                v[i] = (typename Lane<T, V>::Vec)(T)0.f;
                if (i < n) v[i] = Lane<T, V>::load(p + off);
            }
        }
    }
};

// ---------------------------------------------------------------------------------------------------------------------
// spans
// ---------------------------------------------------------------------------------------------------------------------

template <int V>
using Span = float[kSpan][V];

// A span's gates and what each step adds to the state, u = (1 - a) x.  Steps behind the last one keep the state as it is;
// a step with a reset has its gate shut once u is formed, which multiplies a finite state by zero.
template <class T, int V, bool BACK = false>
__device__ inline void span_open(const Raw<T, V> &f, const Raw<T, V> &x, const float (&b)[V], int n, unsigned rm, Span<V> &g, Span<V> &u) {
    typedef Gate<sizeof(T) == 4> G;
#pragma unroll
    for (int i = 0; i < kSpan; i++)
#pragma unroll
        for (int k = 0; k < V; k++) {
            g[i][k] = G::of((float)f.v[i][k] + b[k]);
            u[i][k] = BACK ? (float)x.v[i][k] : G::take(g[i][k]) * (float)x.v[i][k];
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
            for (int k = 0; k < V; k++) g[i][k] = rm >> i & 1 ? G::shut() : g[i][k];
}

// Walks a span from state h, handing every step's state to `out(i, h)`.  The quick form of a step has no value for an infinite
// state and turns it to NaN; NaN goes through shut gates, so a span that met either ends in NaN and is walked again the slow way.
template <bool EXACT, int V, class Out>
__device__ inline void span_walk(const Span<V> &g, const Span<V> &u, unsigned rm, float (&h)[V], Out out) {
    typedef Gate<EXACT> G;
    float h0[V];
    bool bad = false;
#pragma unroll
    for (int k = 0; k < V; k++) h0[k] = h[k];
#pragma unroll
    for (int i = 0; i < kSpan; i++) {
#pragma unroll
        for (int k = 0; k < V; k++) h[k] = G::pass(g[i][k], h[k]) + u[i][k];
        out(i, h);
    }
#pragma unroll
    for (int k = 0; k < V; k++) bad |= !(fabsf(h[k]) < INFINITY);
    if (__any(bad)) {
#pragma unroll
        for (int k = 0; k < V; k++) h[k] = h0[k];
#pragma unroll
        for (int i = 0; i < kSpan; i++) {
#pragma unroll
            for (int k = 0; k < V; k++) h[k] = rm >> i & 1 ? u[i][k] : G::pass_any(g[i][k], h[k]) + u[i][k];
            out(i, h);
        }
    }
}

// A and D of a span.  D grows by 1 - a of what is left of it, so that it keeps its figures while it is small.
template <bool EXACT, int V>
__device__ inline void span_passes(const Span<V> &g, unsigned rm, Run (&r)[V]) {
    typedef Gate<EXACT> G;
#pragma unroll
    for (int k = 0; k < V; k++) r[k].A = 1.f, r[k].D = 0.f;
#pragma unroll
    for (int i = 0; i < kSpan; i++)
#pragma unroll
        for (int k = 0; k < V; k++) {
            const float om = G::take(g[i][k]);
            r[k].A = G::pass(g[i][k], r[k].A);
            r[k].D = r[k].D + fmaf(-r[k].D, om, om);
        }
#pragma unroll
    for (int k = 0; k < V; k++)
        if (rm) r[k].A = -1.f;
}

// The same against time, for the gradient: dy enters a step before the gate does, a reset stands behind it.
template <bool EXACT, int V>
__device__ inline void span_back(const Span<V> &g, const Span<V> &dy, unsigned rm, Run (&r)[V]) {
    typedef Gate<EXACT> G;
    bool bad = false;
#pragma unroll
    for (int k = 0; k < V; k++) r[k].B = 0.f;
#pragma unroll
    for (int i = kSpan - 1; i >= 0; i--)
#pragma unroll
        for (int k = 0; k < V; k++) r[k].B = G::pass(g[i][k], r[k].B + dy[i][k]);
#pragma unroll
    for (int k = 0; k < V; k++) bad |= !(fabsf(r[k].B) < INFINITY);
    if (__any(bad)) {
#pragma unroll
        for (int k = 0; k < V; k++) r[k].B = 0.f;
#pragma unroll
        for (int i = kSpan - 1; i >= 0; i--)
#pragma unroll
            for (int k = 0; k < V; k++) r[k].B = rm >> i & 1 ? 0.f : G::pass_any(g[i][k], r[k].B + dy[i][k]);
    }
}

// ---------------------------------------------------------------------------------------------------------------------
// how a sequence is cut
// ---------------------------------------------------------------------------------------------------------------------

// Shares: every wave walks `spans` spans of its tile of columns; kWaves shares in a row make a segment, a workgroup's.  With one
// share per tile (segs = 1, shares = 1) a wave walks the whole sequence.  Else a first launch finds what every share does to the
// state that enters it, and the second starts every share from what the shares before it make of h0.
struct Shares {
    int spans, shares, segs;
    float *seg_runs;        // [segs][3][C]
    float *share_runs;      // [segs * kWaves][3][C]
};

// State that enters share `w` of segment `seg` (BACK: gradient, from the other end).  Every wave joins a part of the segments
// before it, the parts meet in LDS; then the segment's own shares.
template <int V, bool BACK>
__device__ inline void shares_through(const Shares &cut, unsigned C, unsigned c, int seg, int w, float (&part)[kWaves][3][64 * V], float (&h)[V]) {
    const int lane = threadIdx.x & 63;
    const int n = BACK ? cut.segs - 1 - seg : seg, per = (n + kWaves - 1) / kWaves;
    if (n > 0) {
        const int lo = w * per, hi = lo + per < n ? lo + per : n;
        Run r[V];
#pragma unroll
        for (int k = 0; k < V; k++) r[k] = {1.f, 0.f, 0.f};
#pragma unroll 8
        for (int i = lo; i < hi; i++) {
            const float *q = cut.seg_runs + (int64_t)(BACK ? cut.segs - 1 - i : i) * 3 * C + c;
#pragma unroll
            for (int k = 0; k < V; k++) r[k] = run_join(r[k], Run{q[k], q[(int64_t)C + k], q[2 * (int64_t)C + k]});
        }
#pragma unroll
        for (int k = 0; k < V; k++) part[w][0][lane * V + k] = r[k].A, part[w][1][lane * V + k] = r[k].D, part[w][2][lane * V + k] = r[k].B;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kWaves; i++)
#pragma unroll
            for (int k = 0; k < V; k++) h[k] = run_through(Run{part[i][0][lane * V + k], part[i][1][lane * V + k], part[i][2][lane * V + k]}, h[k]);
    }
    for (int i = BACK ? kWaves - 1 : 0; i != w; i += BACK ? -1 : 1) {
        const float *q = cut.share_runs + ((int64_t)seg * kWaves + i) * 3 * C + c;
#pragma unroll
        for (int k = 0; k < V; k++) h[k] = run_through(Run{q[k], q[(int64_t)C + k], q[2 * (int64_t)C + k]}, h[k]);
    }
}

// First launch of a sequence that is cut: the runs of every share and segment.  x stands for dy when BACK.
template <class T, int V, bool BACK>
__global__ __launch_bounds__(64 * kWaves) void glr_runs_kernel(Seq<const T> f, Seq<const T> x, const float *__restrict__ bias,
                                                               Seq<const uint8_t> resets, int T_, unsigned C, unsigned H, unsigned env_tiles,
                                                               Shares cut) {
    __shared__ float part[kWaves][3][64 * V];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), seg = blockIdx.y;
    const Place at = place_of<V>(C, H, env_tiles);
    const unsigned fo = lane_offset(f, at), xo = lane_offset(x, at);
    float b[V];
    Run r[V];
#pragma unroll
    for (int k = 0; k < V; k++) b[k] = bias ? bias[at.j + k] : 0.f, r[k] = {1.f, 0.f, 0.f};
    const int64_t first = ((int64_t)seg * kWaves + w) * cut.spans, last = (T_ + kSpan - 1) / kSpan;
    const int64_t end = first + cut.spans < last ? first + cut.spans : last;
    Raw<T, V> fr, xr;
    auto fetch = [&](int64_t s) {
        const int64_t t0 = s * kSpan;
        const int n = (int)(T_ - t0 < kSpan ? T_ - t0 : kSpan);
        fr.load(f, at, fo, t0, n);
        xr.load(x, at, xo, t0, n);
    };
    if (first < end) fetch(BACK ? end - 1 : first);
    for (int64_t i = first; i < end; i++) {
        const int64_t s = BACK ? end - 1 - (i - first) : i, t0 = s * kSpan;
        const int n = (int)(T_ - t0 < kSpan ? T_ - t0 : kSpan);
        const unsigned rm = span_resets(resets, t0, n, at);
        Span<V> g, u;                                       // BACK: u is dy
        Run one[V];
        span_open<T, V, BACK>(fr, xr, b, n, rm, g, u);
        if (i + 1 < end) fetch(BACK ? s - 1 : s + 1);
        span_passes<sizeof(T) == 4, V>(g, rm, one);
        if (BACK) {
            span_back<sizeof(T) == 4, V>(g, u, rm, one);
        } else {
            float h[V];
#pragma unroll
            for (int k = 0; k < V; k++) h[k] = 0.f;
            span_walk<sizeof(T) == 4, V>(g, u, rm, h, [](int, const float (&)[V]) {});
#pragma unroll
            for (int k = 0; k < V; k++) one[k].B = h[k];
        }
#pragma unroll
        for (int k = 0; k < V; k++) r[k] = run_join(r[k], one[k]);
    }
    float *own = cut.share_runs + ((int64_t)seg * kWaves + w) * 3 * C + at.c;
#pragma unroll
    for (int k = 0; k < V; k++) {
        if (at.mine) own[k] = r[k].A, own[(int64_t)C + k] = r[k].D, own[2 * (int64_t)C + k] = r[k].B;
        part[w][0][lane * V + k] = r[k].A;
        part[w][1][lane * V + k] = r[k].D;
        part[w][2][lane * V + k] = r[k].B;
    }
    __syncthreads();
    if (w == 0 && at.mine) {
        float *o = cut.seg_runs + (int64_t)seg * 3 * C + at.c;
#pragma unroll
        for (int k = 0; k < V; k++) {
            Run all = {1.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < kWaves; i++) {
                const int q = BACK ? kWaves - 1 - i : i;
                all = run_join(all, Run{part[q][0][lane * V + k], part[q][1][lane * V + k], part[q][2][lane * V + k]});
            }
            o[k] = all.A, o[(int64_t)C + k] = all.D, o[2 * (int64_t)C + k] = all.B;
        }
    }
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

template <class T, int V>
__device__ inline void forward_span(const ForwardArgs<T> &a, const Place &at, unsigned yo, int64_t t0, int n, unsigned rm, const Span<V> &g,
                                    const Span<V> &u, float (&h)[V]) {
    if (a.saved && at.mine)
#pragma unroll
        for (int k = 0; k < V; k++) a.saved[t0 / kSpan * a.C + at.c + k] = h[k];
    char *base = step_base(a.y, at, t0);
    const int64_t step = distance(a.y);
    span_walk<sizeof(T) == 4, V>(g, u, rm, h, [&](int i, const float (&v)[V]) {
        if (i < n && at.mine) Lane<T, V>::store(base + i * step + yo, v);
    });
    if (a.h_last && t0 + kSpan >= a.T_ && at.mine)
#pragma unroll
        for (int k = 0; k < V; k++) a.h_last[at.c + k] = h[k];
}

// Every wave walks its share; the next span's inputs are on their way while a span is walked.
template <class T, int V>
__global__ __launch_bounds__(64 * kWaves) void glr_forward_kernel(ForwardArgs<T> a, Shares cut) {
    __shared__ float part[kWaves][3][64 * V];
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), seg = cut.shares == 1 ? 0 : (int)(gridDim.y - 1 - blockIdx.y);
    const Place at = place_of<V>(a.C, a.H, a.env_tiles);
    const unsigned fo = lane_offset(a.f, at), xo = lane_offset(a.x, at), yo = lane_offset(a.y, at);
    float b[V], h[V];
#pragma unroll
    for (int k = 0; k < V; k++) b[k] = a.bias ? a.bias[at.j + k] : 0.f, h[k] = a.h0 ? a.h0[at.c + k] : 0.f;
    int64_t span = 0, end = cut.spans;
    if (cut.shares > 1) {
        shares_through<V, false>(cut, a.C, at.c, seg, w, part, h);
        span = ((int64_t)seg * kWaves + w) * cut.spans;
        end = span + cut.spans;
    }
    const int64_t last = (a.T_ + kSpan - 1) / kSpan;
    if (end > last) end = last;
    Raw<T, V> fr, xr;
    auto fetch = [&](int64_t s) {
        const int64_t t0 = s * kSpan;
        const int n = (int)(a.T_ - t0 < kSpan ? a.T_ - t0 : kSpan);
        fr.load(a.f, at, fo, t0, n);
        xr.load(a.x, at, xo, t0, n);
    };
    if (span < end) fetch(span);
    for (; span < end; span++) {
        const int64_t t0 = span * kSpan;
        const int n = (int)(a.T_ - t0 < kSpan ? a.T_ - t0 : kSpan);
        const unsigned rm = span_resets(a.resets, t0, n, at);
        Span<V> g, u;
        span_open<T, V>(fr, xr, b, n, rm, g, u);
        if (span + 1 < end) fetch(span + 1);
        forward_span<T, V>(a, at, yo, t0, n, rm, g, u, h);
    }
}

// Short sequences of few columns in one launch: a workgroup holds the whole of its columns, one span per wave, and the waves
// exchange their spans' runs through LDS.
template <class T, int V>
__global__ __launch_bounds__(64 * kHeld) void glr_forward_held_kernel(ForwardArgs<T> a) {
    __shared__ float runs[kHeld][3][64 * V];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Place at = place_of<V>(a.C, a.H, a.env_tiles);
    const int64_t t0 = (int64_t)w * kSpan;
    const int n = (int)(a.T_ - t0 < kSpan ? a.T_ - t0 : kSpan);
    Raw<T, V> fr, xr;
    fr.load(a.f, at, lane_offset(a.f, at), t0, n);
    xr.load(a.x, at, lane_offset(a.x, at), t0, n);
    const unsigned rm = span_resets(a.resets, t0, n, at);
    float b[V], h[V];
#pragma unroll
    for (int k = 0; k < V; k++) b[k] = a.bias ? a.bias[at.j + k] : 0.f, h[k] = 0.f;
    Span<V> g, u;
    Run r[V];
    span_open<T, V>(fr, xr, b, n, rm, g, u);
    span_passes<sizeof(T) == 4, V>(g, rm, r);
    span_walk<sizeof(T) == 4, V>(g, u, rm, h, [](int, const float (&)[V]) {});
#pragma unroll
    for (int k = 0; k < V; k++) {
        runs[w][0][lane * V + k] = r[k].A, runs[w][1][lane * V + k] = r[k].D, runs[w][2][lane * V + k] = h[k];
        h[k] = a.h0 ? a.h0[at.c + k] : 0.f;
    }
    __syncthreads();
    for (int i = 0; i < w; i++)
#pragma unroll
        for (int k = 0; k < V; k++) h[k] = run_through(Run{runs[i][0][lane * V + k], runs[i][1][lane * V + k], runs[i][2][lane * V + k]}, h[k]);
    forward_span<T, V>(a, at, lane_offset(a.y, at), t0, n, rm, g, u, h);
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
    float *dbias_rows, *dh0;        // dbias_rows [segs][C] or null
    int T_;
    unsigned C, H, env_tiles;
};

// Gates (resets not in them) and q = (p - x) a (1 - a), what df is per unit of g, from the states recomputed off the kept one.
template <class T, int V>
__device__ inline void back_open(const Raw<T, V> &f, const Raw<T, V> &x, const float (&b)[V], const float (&kept)[V], int n, unsigned rm,
                                 Span<V> &g, Span<V> &q) {
    typedef Gate<sizeof(T) == 4> G;
    float h[V];
    bool bad = false;
#pragma unroll
    for (int k = 0; k < V; k++) h[k] = kept[k];
#pragma unroll
    for (int i = 0; i < kSpan; i++)
#pragma unroll
        for (int k = 0; k < V; k++) {
            float slope;
            const float xv = (float)x.v[i][k];
            g[i][k] = G::of((float)f.v[i][k] + b[k], slope);
            if (rm >> i & 1) h[k] = 0.f;
            q[i][k] = (h[k] - xv) * slope;
            bad |= !(fabsf(h[k]) < INFINITY);
            h[k] = G::pass(g[i][k], h[k]) + G::take(g[i][k]) * xv;
        }
    if (__any(bad)) {
#pragma unroll
        for (int k = 0; k < V; k++) h[k] = kept[k];
#pragma unroll
        for (int i = 0; i < kSpan; i++)
#pragma unroll
            for (int k = 0; k < V; k++) {
                float slope;
                const float xv = (float)x.v[i][k];
                g[i][k] = G::of((float)f.v[i][k] + b[k], slope);
                if (rm >> i & 1) h[k] = 0.f;
                q[i][k] = (h[k] - xv) * slope;
                h[k] = G::pass_any(g[i][k], h[k]) + G::take(g[i][k]) * xv;
            }
    }
    if (n < kSpan)
#pragma unroll
        for (int i = 0; i < kSpan; i++)
#pragma unroll
            for (int k = 0; k < V; k++)
                if (i >= n) g[i][k] = G::open(), q[i][k] = 0.f;
}

// Walks a span back from gradient `in`, writes df and dx and adds up df.
template <class T, int V>
__device__ inline void back_span(const BackwardArgs<T> &a, const Place &at, unsigned dfo, unsigned dxo, int64_t t0, int n, unsigned rm,
                                 const Span<V> &g, const Span<V> &q, const Raw<T, V> &dy, float (&in)[V], double (&total)[V]) {
    typedef Gate<sizeof(T) == 4> G;
    char *fp = step_base(a.df, at, t0), *xp = step_base(a.dx, at, t0);
    const int64_t fstep = distance(a.df), xstep = distance(a.dx);
    float sum[V], in0[V];
    bool bad = false;
    auto walk = [&](auto slow) {
#pragma unroll
        for (int k = 0; k < V; k++) sum[k] = 0.f;
#pragma unroll
        for (int i = kSpan - 1; i >= 0; i--) {
            float of[V], ox[V];
#pragma unroll
            for (int k = 0; k < V; k++) {
                const float gs = (float)dy.v[i][k] + in[k];
                ox[k] = G::take(g[i][k]) * gs;
                of[k] = gs * q[i][k];
                sum[k] += of[k];
                in[k] = decltype(slow)::value ? G::pass_any(g[i][k], gs) : G::pass(g[i][k], gs);
                bad |= !(fabsf(in[k]) < INFINITY);
                if (rm >> i & 1) in[k] = 0.f;
            }
            if (i < n && at.mine) {
                Lane<T, V>::store(fp + i * fstep + dfo, of);
                Lane<T, V>::store(xp + i * xstep + dxo, ox);
            }
        }
    };
#pragma unroll
    for (int k = 0; k < V; k++) in0[k] = in[k];
    walk(std::false_type{});
    if (__any(bad)) {
#pragma unroll
        for (int k = 0; k < V; k++) in[k] = in0[k];
        walk(std::true_type{});
    }
#pragma unroll
    for (int k = 0; k < V; k++) total[k] += (double)sum[k];
    if (a.dh0 && t0 == 0 && at.mine)
#pragma unroll
        for (int k = 0; k < V; k++) a.dh0[at.c + k] = in[k];
}

// per segment and column: the waves' sums in wave order
template <int W, int V>
__device__ inline void dbias_row(float *row, unsigned c, bool mine, int nw, const double (&total)[V], double (&sums)[W][64 * V]) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
    for (int k = 0; k < V; k++) sums[w][lane * V + k] = total[k];
    __syncthreads();
    if (w == 0 && mine)
#pragma unroll
        for (int k = 0; k < V; k++) {
            double s = 0.0;
            for (int i = 0; i < nw; i++) s += sums[i][lane * V + k];
            row[c + k] = (float)s;
        }
}

template <class T, int V>
__global__ __launch_bounds__(64 * kWaves, 2) void glr_backward_kernel(BackwardArgs<T> a, Shares cut) {
    __shared__ float part[kWaves][3][64 * V];
    __shared__ double sums[kWaves][64 * V];
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), seg = blockIdx.y;
    const Place at = place_of<V>(a.C, a.H, a.env_tiles);
    const unsigned fo = lane_offset(a.f, at), xo = lane_offset(a.x, at), go = lane_offset(a.dy, at), dfo = lane_offset(a.df, at), dxo = lane_offset(a.dx, at);
    float b[V], in[V];
    double total[V];
#pragma unroll
    for (int k = 0; k < V; k++) b[k] = a.bias ? a.bias[at.j + k] : 0.f, in[k] = a.dh_last ? a.dh_last[at.c + k] : 0.f, total[k] = 0.0;
    int64_t first = 0, end = cut.spans;
    if (cut.shares > 1) {
        shares_through<V, true>(cut, a.C, at.c, seg, w, part, in);
        first = ((int64_t)seg * kWaves + w) * cut.spans;
        end = first + cut.spans;
    }
    const int64_t last = (a.T_ + kSpan - 1) / kSpan;
    if (end > last) end = last;
    Raw<T, V> fr, xr, gr;
    float kept[V];
    auto fetch = [&](int64_t s) {
        const int64_t t0 = s * kSpan;
        const int n = (int)(a.T_ - t0 < kSpan ? a.T_ - t0 : kSpan);
        fr.load(a.f, at, fo, t0, n);
        xr.load(a.x, at, xo, t0, n);
#pragma unroll
        for (int k = 0; k < V; k++) kept[k] = a.saved[s * a.C + at.c + k];
    };
    if (first < end) fetch(end - 1);
    for (int64_t s = end - 1; s >= first; s--) {
        const int64_t t0 = s * kSpan;
        const int n = (int)(a.T_ - t0 < kSpan ? a.T_ - t0 : kSpan);
        gr.load(a.dy, at, go, t0, n);
        const unsigned rm = span_resets(a.resets, t0, n, at);
        Span<V> g, q;
        back_open<T, V>(fr, xr, b, kept, n, rm, g, q);
        if (s > first) fetch(s - 1);
        back_span<T, V>(a, at, dfo, dxo, t0, n, rm, g, q, gr, in, total);
    }
    if (a.dbias_rows) dbias_row<kWaves, V>(a.dbias_rows + (int64_t)seg * a.C, at.c, at.mine, cut.shares > 1 ? kWaves : 1, total, sums);
}

template <class T, int V>
__global__ __launch_bounds__(64 * kHeld) void glr_backward_held_kernel(BackwardArgs<T> a) {
    __shared__ float runs[kHeld][3][64 * V];
    __shared__ double sums[kHeld][64 * V];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), nw = blockDim.x >> 6;
    const Place at = place_of<V>(a.C, a.H, a.env_tiles);
    const int64_t t0 = (int64_t)w * kSpan;
    const int n = (int)(a.T_ - t0 < kSpan ? a.T_ - t0 : kSpan);
    Raw<T, V> fr, xr, gr;
    fr.load(a.f, at, lane_offset(a.f, at), t0, n);
    xr.load(a.x, at, lane_offset(a.x, at), t0, n);
    gr.load(a.dy, at, lane_offset(a.dy, at), t0, n);
    const unsigned rm = span_resets(a.resets, t0, n, at);
    float b[V], kept[V], in[V];
    double total[V];
#pragma unroll
    for (int k = 0; k < V; k++) {
        b[k] = a.bias ? a.bias[at.j + k] : 0.f;
        kept[k] = a.saved[(int64_t)w * a.C + at.c + k];
        in[k] = a.dh_last ? a.dh_last[at.c + k] : 0.f;
        total[k] = 0.0;
    }
    Span<V> g, q;
    Run r[V];
    back_open<T, V>(fr, xr, b, kept, n, rm, g, q);
    span_passes<sizeof(T) == 4, V>(g, rm, r);
    {
        Span<V> shut, dy;
#pragma unroll
        for (int i = 0; i < kSpan; i++)
#pragma unroll
            for (int k = 0; k < V; k++) shut[i][k] = rm >> i & 1 ? Gate<sizeof(T) == 4>::shut() : g[i][k], dy[i][k] = (float)gr.v[i][k];
        span_back<sizeof(T) == 4, V>(shut, dy, rm, r);
    }
#pragma unroll
    for (int k = 0; k < V; k++) runs[w][0][lane * V + k] = r[k].A, runs[w][1][lane * V + k] = r[k].D, runs[w][2][lane * V + k] = r[k].B;
    __syncthreads();
    for (int i = nw - 1; i > w; i--)
#pragma unroll
        for (int k = 0; k < V; k++) in[k] = run_through(Run{runs[i][0][lane * V + k], runs[i][1][lane * V + k], runs[i][2][lane * V + k]}, in[k]);
    back_span<T, V>(a, at, lane_offset(a.df, at), lane_offset(a.dx, at), t0, n, rm, g, q, gr, in, total);
    if (a.dbias_rows) dbias_row<kHeld, V>(a.dbias_rows, at.c, at.mine, nw, total, sums);
}

// One step: every thread V channels, nothing to share.
template <class T, int V>
__global__ __launch_bounds__(256) void glr_step_kernel(Seq<const T> f, Seq<const T> x, const float *__restrict__ bias, Seq<const uint8_t> resets,
                                                       const float *h0, unsigned C, unsigned H, Seq<T> y, float *h_last, float *__restrict__ saved) {
    typedef Gate<sizeof(T) == 4> G;
    const uint64_t at = ((uint64_t)blockIdx.x * 256 + threadIdx.x) * V;
    if (at >= C) return;
    const unsigned c = (unsigned)at, e = c / H, j = c - e * H;
    const auto fr = Lane<T, V>::load(f.p + (int64_t)e * f.e + j), xr = Lane<T, V>::load(x.p + (int64_t)e * x.e + j);
    const bool fresh = resets.p && resets.p[(int64_t)e * resets.e];
    float h[V];
#pragma unroll
    for (int k = 0; k < V; k++) {
        h[k] = h0 ? h0[c + k] : 0.f;
        if (saved) saved[c + k] = h[k];
        if (fresh) h[k] = 0.f;
        const float g = G::of((float)fr[k] + (bias ? bias[j + k] : 0.f));
        h[k] = G::pass_any(g, h[k]) + G::take(g) * (float)xr[k];
    }
    Lane<T, V>::store(y.p + (int64_t)e * y.e + j, h);
    if (h_last)
#pragma unroll
        for (int k = 0; k < V; k++) h_last[c + k] = h[k];
}

// Column sums of in [rows, H]: workgroup (i, r) sums rows r * kSumRows .. of 32 columns, 32 rows side by side, into out[r, H]
constexpr int kSumRows = 2048;
__global__ __launch_bounds__(1024) void glr_column_sum_kernel(const float *__restrict__ in, int64_t rows, int H, float *__restrict__ out) {
    __shared__ double red[32][33];
    const int col = threadIdx.x & 31, grp = threadIdx.x >> 5, j = blockIdx.x * 32 + col;
    const int64_t r0 = (int64_t)blockIdx.y * kSumRows, r1 = r0 + kSumRows < rows ? r0 + kSumRows : rows;
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
        out[(int64_t)blockIdx.y * H + j] = (float)s;
    }
}

__global__ void glr_copy_state_kernel(const float *src, float *dst, int64_t n) {
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i < n) dst[i] = src ? src[i] : 0.f;
}

}  // namespace ppo2hip

using namespace ppo2hip;

constexpr int64_t kWaveTarget = 4096;     // waves that walk shares
constexpr int64_t kAlone = 640;           // tiles from which a wave walks a whole sequence

template <class T>
static Seq<T> seq_of(const ppo2hip_seq *s) {
    return s ? Seq<T>{(T *)s->data, s->t, s->e} : Seq<T>{nullptr, 0, 0};
}

static int glr_check(const char *what, int dtype, int T, int E, int H) {
    PPO2HIP_REQUIRE(dtype == PPO2HIP_F32 || dtype == PPO2HIP_BF16 || dtype == PPO2HIP_F16, "%s: unknown dtype %d", what, dtype);
    PPO2HIP_REQUIRE(T >= 0 && E >= 0 && H >= 0, "%s: negative size T=%d E=%d H=%d", what, T, E, H);
    PPO2HIP_REQUIRE((int64_t)E * H <= 0x7fffffffll, "%s: E*H=%lld beyond 2^31 - 1 columns", what, (long long)E * H);
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

// How a call is cut: tiles of 64 V columns (V channels per lane), and the time axis held by one workgroup per tile, walked by
// one wave per tile, or cut into shares.
struct Cut {
    int V, run_V, env_tiles, run_env_tiles;     // run_*: of the launch that finds the shares' runs
    int64_t tiles, run_tiles;
    bool held;
    Shares sh;
};
static Cut cut_of(int dtype, int T, int E, int H, bool back) {
    Cut k;
    const int64_t C = (int64_t)E * H, spans = ceil_div(T, kSpan);
    const int wide = dtype != PPO2HIP_F32 && H % 2 == 0 ? 2 : 1;
    k.env_tiles = k.run_env_tiles = 0;
    k.run_V = wide;
    k.run_tiles = ceil_div(C, 64 * wide);
    k.held = spans <= kHeld && k.run_tiles < kAlone;
    // two channels per lane halve a 16-bit sequence's loads; the backward walk and the held spans have no registers for them
    k.V = back || k.held ? 1 : wide;
    k.tiles = ceil_div(C, 64 * k.V);
    k.sh = Shares{(int)spans, 1, 1, nullptr, nullptr};
    if (k.held || k.run_tiles >= kAlone) return k;
    int64_t want = ceil_div(kWaveTarget, k.run_tiles);
    if (want > spans) want = spans;
    k.sh.spans = (int)ceil_div(spans, want);
    k.sh.segs = (int)ceil_div(spans, (int64_t)k.sh.spans * kWaves);
    k.sh.shares = k.sh.segs * kWaves;
    return k;
}
// Lanes of a tile in a row reach over up to 64 V / H envs behind the first: their offsets must fit 31 bits in every array,
// else each env gets tiles of its own (lanes behind H idle there).
static void place_envs(Cut &k, int E, int H, std::initializer_list<const ppo2hip_seq *> seqs) {
    int64_t reach = (64 * 2 - 1) / H + 1;
    if (reach > E - 1) reach = E - 1;
    bool far = false;
    for (const ppo2hip_seq *s : seqs) far |= s && reach > 0 && s->e > ((1ll << 29) - 1 - H) / reach;
    if (!far) return;
    k.env_tiles = (int)ceil_div(H, 64 * k.V);
    k.run_env_tiles = (int)ceil_div(H, 64 * k.run_V);
    k.tiles = (int64_t)E * k.env_tiles;
    k.run_tiles = (int64_t)E * k.run_env_tiles;
}

static size_t runs_bytes(const Cut &k, int64_t C) { return k.sh.shares > 1 ? align_up((size_t)(k.sh.segs + k.sh.shares) * 3 * C * sizeof(float), 256) : 0; }
static void place_runs(Cut &k, int64_t C, void *workspace) {
    k.sh.seg_runs = (float *)workspace;
    k.sh.share_runs = (float *)workspace + (int64_t)k.sh.segs * 3 * C;
}

extern "C" size_t ppo2hip_glr_forward_workspace_bytes(int dtype, int T, int E, int H) {
    if (T <= 1 || E <= 0 || H <= 0) return 0;
    return runs_bytes(cut_of(dtype, T, E, H, false), (int64_t)E * H);
}

extern "C" size_t ppo2hip_glr_backward_workspace_bytes(int dtype, int T, int E, int H, int want_dbias) {
    if (T <= 0 || E <= 0 || H <= 0) return 0;
    const Cut k = cut_of(dtype, T, E, H, true);
    const int64_t C = (int64_t)E * H, rows = (int64_t)k.sh.segs * E;
    size_t n = runs_bytes(k, C);
    if (want_dbias) n += align_up((size_t)rows * H * sizeof(float), 256) + align_up((size_t)ceil_div(rows, kSumRows) * H * sizeof(float), 256);
    return n;
}

template <class T, bool BACK>
static int launch_runs(const Cut &k, const Seq<const T> &f, const Seq<const T> &x, const float *bias, const Seq<const uint8_t> &resets, int T_,
                       unsigned C, unsigned H, hipStream_t s) {
    const dim3 grid((unsigned)k.run_tiles, k.sh.segs), block(64 * kWaves);
    if (sizeof(T) == 2 && k.run_V == 2)
        hipLaunchKernelGGL((glr_runs_kernel<T, sizeof(T) == 2 ? 2 : 1, BACK>), grid, block, 0, s, f, x, bias, resets, T_, C, H, k.run_env_tiles, k.sh);
    else
        hipLaunchKernelGGL((glr_runs_kernel<T, 1, BACK>), grid, block, 0, s, f, x, bias, resets, T_, C, H, k.run_env_tiles, k.sh);
    return check_launch("glr_runs_kernel");
}

template <class T, int V>
static int forward_of(const Cut &k, const ppo2hip_seq *f, const ppo2hip_seq *x, const float *bias, const ppo2hip_seq *resets, const float *h0,
                      const ppo2hip_seq *y, float *h_last, float *saved, int T_, int E, int H, hipStream_t s) {
    const int64_t C = (int64_t)E * H;
    if (T_ == 1) {
        hipLaunchKernelGGL((glr_step_kernel<T, V>), dim3((unsigned)ceil_div(C, 256 * V)), dim3(256), 0, s, seq_of<const T>(f), seq_of<const T>(x),
                           bias, seq_of<const uint8_t>(resets), h0, (unsigned)C, (unsigned)H, seq_of<T>(y), h_last, saved);
        return check_launch("glr_step_kernel");
    }
    const ForwardArgs<T> a = {seq_of<const T>(f), seq_of<const T>(x), seq_of<const uint8_t>(resets), seq_of<T>(y), bias, h0, h_last, saved,
                              T_, (unsigned)C, (unsigned)H, (unsigned)k.env_tiles};
    if (k.held) {
        hipLaunchKernelGGL((glr_forward_held_kernel<T, 1>), dim3((unsigned)k.tiles), dim3(64 * (unsigned)ceil_div(T_, kSpan)), 0, s, a);
        return check_launch("glr_forward_held_kernel");
    }
    if (k.sh.shares > 1) {
        int rc = launch_runs<T, false>(k, a.f, a.x, bias, a.resets, T_, a.C, a.H, s);
        if (rc) return rc;
    }
    hipLaunchKernelGGL((glr_forward_kernel<T, V>), dim3((unsigned)k.tiles, k.sh.segs), dim3(64 * (k.sh.shares > 1 ? kWaves : 1)), 0, s, a, k.sh);
    return check_launch("glr_forward_kernel");
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
    PPO2HIP_REQUIRE(T == 1 || k.sh.shares == 1 || workspace, "glr_forward: workspace is null");
    place_runs(k, C, workspace);
#define PPO2HIP_GLR_FORWARD(type, V) forward_of<type, V>(k, f, x, bias, resets, h0, y, h_last, saved, T, E, H, s)
    if (dtype == PPO2HIP_F32) return PPO2HIP_GLR_FORWARD(float, 1);
    if (dtype == PPO2HIP_BF16) return k.V == 2 ? PPO2HIP_GLR_FORWARD(__bf16, 2) : PPO2HIP_GLR_FORWARD(__bf16, 1);
    return k.V == 2 ? PPO2HIP_GLR_FORWARD(_Float16, 2) : PPO2HIP_GLR_FORWARD(_Float16, 1);
#undef PPO2HIP_GLR_FORWARD
}

template <class T, int V>
static int backward_of(const Cut &k, const ppo2hip_seq *f, const ppo2hip_seq *x, const float *bias, const ppo2hip_seq *resets, const float *saved,
                       const ppo2hip_seq *dy, const float *dh_last, const ppo2hip_seq *df, const ppo2hip_seq *dx, float *dbias, float *dh0,
                       void *workspace, int T_, int E, int H, hipStream_t s) {
    const int64_t C = (int64_t)E * H, rows = (int64_t)k.sh.segs * E;
    float *sums = (float *)((char *)workspace + runs_bytes(k, C));
    const BackwardArgs<T> a = {seq_of<const T>(f), seq_of<const T>(x), seq_of<const T>(dy), seq_of<const uint8_t>(resets), seq_of<T>(df), seq_of<T>(dx),
                               bias, saved, dh_last, dbias ? sums : nullptr, dh0, T_, (unsigned)C, (unsigned)H, (unsigned)k.env_tiles};
    int rc;
    if (k.held) {
        hipLaunchKernelGGL((glr_backward_held_kernel<T, V>), dim3((unsigned)k.tiles), dim3(64 * (unsigned)ceil_div(T_, kSpan)), 0, s, a);
        rc = check_launch("glr_backward_held_kernel");
    } else {
        if (k.sh.shares > 1 && (rc = launch_runs<T, true>(k, a.f, a.dy, bias, a.resets, T_, a.C, a.H, s))) return rc;
        hipLaunchKernelGGL((glr_backward_kernel<T, V>), dim3((unsigned)k.tiles, k.sh.segs), dim3(64 * (k.sh.shares > 1 ? kWaves : 1)), 0, s, a, k.sh);
        rc = check_launch("glr_backward_kernel");
    }
    if (rc || !dbias) return rc;
    // rows [segment][env] of H channels each, kSumRows of them to a workgroup, until one row is left
    float *in = sums, *out = (float *)((char *)sums + align_up((size_t)rows * H * sizeof(float), 256));
    for (int64_t n = rows;;) {
        const int64_t left = ceil_div(n, kSumRows);
        hipLaunchKernelGGL(glr_column_sum_kernel, dim3((unsigned)ceil_div(H, 32), (unsigned)left), dim3(1024), 0, s, in, n, H, left == 1 ? dbias : out);
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
    PPO2HIP_REQUIRE((!dbias && k.sh.shares == 1) || workspace, "glr_backward: workspace is null");
    place_runs(k, C, workspace);
#define PPO2HIP_GLR_BACKWARD(type) backward_of<type, 1>(k, f, x, bias, resets, saved, dy, dh_last, df, dx, dbias, dh0, workspace, T, E, H, s)
    if (dtype == PPO2HIP_F32) return PPO2HIP_GLR_BACKWARD(float);
    if (dtype == PPO2HIP_BF16) return PPO2HIP_GLR_BACKWARD(__bf16);
    return PPO2HIP_GLR_BACKWARD(_Float16);
#undef PPO2HIP_GLR_BACKWARD
}
