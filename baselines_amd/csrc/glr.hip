// Gated linear recurrence over a time-major sequence, forward and backward:
//   a = sigmoid(f + bias)   p = reset ? 0 : h[t-1]   h[t] = a p + (1 - a) x[t]
//   g[t] = dy[t] + (reset[t+1] ? 0 : a[t+1] g[t+1])   dx = (1 - a) g   df = g (p - x) a (1 - a)
// The backward pass recomputes the states from float32 states kept every PPO2HIP_GLR_SPAN steps: they cost
// 4 / SPAN bytes per element where reading y back costs its whole width, and y is rounded to its type while p - x cancels.
#include <initializer_list>

#include "kernels.hpp"

// Products and sums round one by one unless fmaf says otherwise: the same step written in two places gives the same bits, so
// that a state recomputed in the backward pass is the forward's, and a span walked the slow way changes no other column.
#pragma clang fp contract(off)

namespace ppo2hip {

constexpr int kSpan = PPO2HIP_GLR_SPAN;

// A gate a is held as its smaller side s = min(a, 1 - a) <= 1/2, negated where that is 1 - a (a >= 1/2, the sign bit of -0
// included).  Both sides keep their relative accuracy this way: 1 - a taken from a rounded a loses the memory's length as soon
// as a is near one.  `nz` is -(f + bias).  EXACT is for float32 sequences: the rounding of nz's product with log2(e) and the
// reciprocal's are made good; in 16 bits what is written is 2^12 times coarser than that.
template <bool EXACT>
__device__ inline float gate_of(float nz) {
    float m = fabsf(nz), e;
    if (EXACT) {
        m = m > 128.f ? 128.f : m;                          // e^-128 is 0 in float32; a NaN stays one
        const float t = m * -1.44269502f;
        const float rest = fmaf(m, -1.92596299e-8f, fmaf(m, -1.44269502f, -t));
        e = __builtin_amdgcn_exp2f(t);
        e = fmaf(e * 0.693147182f, rest, e);
    } else {
        e = __builtin_amdgcn_exp2f(m * -1.44269502f);
    }
    const float d = 1.f + e;
    float r = __builtin_amdgcn_rcpf(d);
    if (EXACT) r = fmaf(fmaf(-d, r, 1.f), r, r);
    return copysignf(e * r, nz);
}
__device__ inline bool gate_keeps(float g) { return (int)__float_as_uint(g) < 0; }
// 1 - a
__device__ inline float gate_take(float g) { return gate_keeps(g) ? -g : 1.f - g; }
// a v, as v - (1 - a) v where a >= 1/2
__device__ inline float gate_pass(float g, float v) { return fmaf(g, v, gate_keeps(g) ? v : 0.f); }
// the same where v may not be finite, for which v - (1 - a) v has no value
__device__ inline float gate_pass_any(float g, float v) {
    return fabsf(v) < INFINITY ? gate_pass(g, v) : (gate_keeps(g) ? 1.f + g : g) * v;
}

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

template <class T>
struct SeqIn {
    const T *p;
    int64_t t, e;
};
template <class T>
struct SeqOut {
    T *p;
    int64_t t, e;
};

// V neighbouring channels of one step, at any address an element may have
template <class T, int V>
struct Lane {
    typedef T Vec __attribute__((ext_vector_type(V)));
    typedef Vec Any __attribute__((aligned(sizeof(T))));
    static __device__ inline Vec load(const T *p) { return *(const Any *)p; }
    static __device__ inline void store(T *p, const float (&v)[V]) {
        Vec r;
#pragma unroll
        for (int k = 0; k < V; k++) r[k] = (T)v[k];       // to nearest: the type that the layer hands on; states stay float32
        *(Any *)p = r;
    }
};

constexpr int kWaves = 8;                                   // spans a workgroup works on at a time
constexpr int kBatch = kWaves * kSpan;                      // steps of such a batch

// Which columns a wave works on.  Addresses are a wave-uniform 64-bit part (step, the wave's first env) and a 32-bit part
// per lane: kept as 64 bits per lane and step they cost 2 registers each and the kernels spill.
struct Place {
    int64_t c, e0;      // the lane's first column e * H + j, first env of the wave
    int de, j;          // lane's env less e0, channel
    bool mine;          // false: a lane behind the last column, which repeats it and writes nothing
};
// env_tiles 0: columns in a row over all envs.  Else that many tiles per env, where envs lie too far apart for 32 bits.
template <int V>
__device__ inline Place place_of(int64_t C, int H, int env_tiles) {
    const int lane = threadIdx.x & 63;
    Place p;
    if (env_tiles == 0) {
        const int64_t c = ((int64_t)blockIdx.x * 64 + lane) * V;
        p.mine = c < C;
        p.c = p.mine ? c : C - V;
        const int e = (int)(p.c / H);
        p.e0 = __builtin_amdgcn_readfirstlane(e);
        p.de = e - (int)p.e0;
        p.j = (int)(p.c - (int64_t)e * H);
    } else {
        const int e = blockIdx.x / env_tiles, j = ((blockIdx.x - e * env_tiles) * 64 + lane) * V;
        p.mine = j < H;
        p.j = p.mine ? j : H - V;
        p.e0 = e;
        p.de = 0;
        p.c = (int64_t)e * H + p.j;
    }
    return p;
}
template <class S>
__device__ inline unsigned lane_offset(const S &s, const Place &p) { return (unsigned)(p.de * (int)s.e + p.j) * (unsigned)sizeof(*s.p); }

// Flags of the span's steps t0 .. t0+n-1 as bits.  Where all lanes look at one env, 16 of them fetch one flag each.
__device__ inline unsigned span_resets(const SeqIn<uint8_t> &r, int64_t t0, int n, const Place &at) {
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

// A step's distance in bytes, said anew for every span: as loop invariants the 16 multiples of every array's distance are kept
// in scalar registers, which do not hold them.
template <class S>
__device__ inline int64_t distance(const S &s) {
    int64_t d = s.t * (int64_t)sizeof(*s.p);
    asm volatile("" : "+s"(d));
    return d;
}

template <class T, int V>
__device__ inline void span_load(const SeqIn<T> &s, const Place &at, unsigned off, int64_t t0, int n, typename Lane<T, V>::Vec (&out)[kSpan]) {
    const char *p = (const char *)(s.p + t0 * s.t + at.e0 * s.e);
    const int64_t step = distance(s);
    if (n >= kSpan) {
#pragma unroll
        for (int i = 0; i < kSpan; i++) out[i] = Lane<T, V>::load((const T *)(p + i * step + off));
    } else {
#pragma unroll
        for (int i = 0; i < kSpan; i++) {
            out[i] = (typename Lane<T, V>::Vec)(T)0.f;
            if (i < n) out[i] = Lane<T, V>::load((const T *)(p + i * step + off));
        }
    }
}
template <class T, int V>
__device__ inline void step_store(char *p, int64_t step, unsigned off, int i, const float (&v)[V]) { Lane<T, V>::store((T *)(p + i * step + off), v); }

// Keeps the compiler from carrying the comparisons that one pass over a span made into the next: as lane masks they fill the
// scalar registers and are spilled lane by lane, and repeating one is a single instruction.
template <int V>
__device__ inline void afresh(float (&g)[kSpan][V], unsigned &rm) {
    asm volatile("" : "+v"(rm));
#pragma unroll
    for (int i = 0; i < kSpan; i++)
#pragma unroll
        for (int k = 0; k < V; k++) asm volatile("" : "+v"(g[i][k]));
}

// gates of a span; steps behind the last one keep the state as it is
template <class T, int V>
__device__ inline void span_gates(const typename Lane<T, V>::Vec (&f)[kSpan], const float (&b)[V], int n, float (&g)[kSpan][V]) {
#pragma unroll
    for (int i = 0; i < kSpan; i++)
#pragma unroll
        for (int k = 0; k < V; k++) g[i][k] = gate_of<sizeof(T) == 4>(-(float)f[i][k] - b[k]);
    if (n < kSpan)
#pragma unroll
        for (int i = 0; i < kSpan; i++)
#pragma unroll
            for (int k = 0; k < V; k++) g[i][k] = i >= n ? -0.f : g[i][k];
}

// A span's run in the direction of time.  u: what each step adds, (1 - a) x.  The quick form of a step has no value for an
// infinite state; a span that ends in none is walked again the slow way.
template <int V>
__device__ inline void span_run(float (&g)[kSpan][V], const float (&u)[kSpan][V], unsigned rm, Run (&r)[V]) {
#pragma unroll
    for (int k = 0; k < V; k++) r[k] = {1.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < kSpan; i++)
#pragma unroll
        for (int k = 0; k < V; k++) {
            const float v = g[i][k];
            r[k].A = gate_pass(v, r[k].A);
            r[k].D = gate_pass(v, r[k].D) + gate_take(v);
            r[k].B = gate_pass(v, rm >> i & 1 ? 0.f : r[k].B) + u[i][k];
        }
    bool bad = false;
#pragma unroll
    for (int k = 0; k < V; k++) bad |= !(fabsf(r[k].B) < INFINITY);
    if (__any(bad)) {
        afresh<V>(g, rm);
#pragma unroll
        for (int k = 0; k < V; k++) r[k].B = 0.f;
#pragma unroll
        for (int i = 0; i < kSpan; i++)
#pragma unroll
            for (int k = 0; k < V; k++) r[k].B = gate_pass_any(g[i][k], rm >> i & 1 ? 0.f : r[k].B) + u[i][k];
    }
    if (rm)
#pragma unroll
        for (int k = 0; k < V; k++) r[k].A = -1.f;
}
// and against it: dy enters a step before the gate does, the reset stands behind it
template <class T, int V>
__device__ inline void span_run_back(float (&g)[kSpan][V], const typename Lane<T, V>::Vec (&dy)[kSpan], unsigned rm, Run (&r)[V]) {
#pragma unroll
    for (int k = 0; k < V; k++) r[k] = {1.f, 0.f, 0.f};
#pragma unroll
    for (int i = kSpan - 1; i >= 0; i--)
#pragma unroll
        for (int k = 0; k < V; k++) {
            const float v = g[i][k];
            r[k].A = gate_pass(v, r[k].A);
            r[k].D = gate_pass(v, r[k].D) + gate_take(v);
            r[k].B = gate_pass(v, r[k].B + (float)dy[i][k]);
            if (rm >> i & 1) r[k].B = 0.f;
        }
    bool bad = false;
#pragma unroll
    for (int k = 0; k < V; k++) bad |= !(fabsf(r[k].B) < INFINITY);
    if (__any(bad)) {
        afresh<V>(g, rm);
#pragma unroll
        for (int k = 0; k < V; k++) r[k].B = 0.f;
#pragma unroll
        for (int i = kSpan - 1; i >= 0; i--)
#pragma unroll
            for (int k = 0; k < V; k++) {
                r[k].B = gate_pass_any(g[i][k], r[k].B + (float)dy[i][k]);
                if (rm >> i & 1) r[k].B = 0.f;
            }
    }
    if (rm)
#pragma unroll
        for (int k = 0; k < V; k++) r[k].A = -1.f;
}

// State (or gradient) that enters segment `seg`: the runs of the segments before it (behind it), in order.  Every wave joins a
// share of them, the shares meet in LDS.  parts [segments][3][C].
template <int V, bool BACK>
__device__ inline void segments_through(const float *__restrict__ parts, int64_t C, int64_t c, int seg, int nseg, int w, int lane,
                                        float (&share)[kWaves][3][64 * V], float (&h)[V]) {
    const int n = BACK ? nseg - 1 - seg : seg, per = (n + kWaves - 1) / kWaves;
    const int lo = w * per, hi = lo + per < n ? lo + per : n;
    Run r[V];
#pragma unroll
    for (int k = 0; k < V; k++) r[k] = {1.f, 0.f, 0.f};
#pragma unroll 4
    for (int i = lo; i < hi; i++) {
        const float *q = parts + (int64_t)(BACK ? nseg - 1 - i : i) * 3 * C + c;
#pragma unroll
        for (int k = 0; k < V; k++) r[k] = run_join(r[k], Run{q[k], q[C + k], q[2 * C + k]});
    }
#pragma unroll
    for (int k = 0; k < V; k++) share[w][0][lane * V + k] = r[k].A, share[w][1][lane * V + k] = r[k].D, share[w][2][lane * V + k] = r[k].B;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kWaves; i++)
#pragma unroll
        for (int k = 0; k < V; k++) h[k] = run_through(Run{share[i][0][lane * V + k], share[i][1][lane * V + k], share[i][2][lane * V + k]}, h[k]);
    __syncthreads();
}

// First launch of a sequence that is cut into segments of `batches` batches: every segment's run, [segment][A, D, B][C].  Each
// wave walks an equal share of the segment's spans, the shares are joined in LDS.  x stands for dy when BACK.
template <class T, int V, bool BACK>
__global__ __launch_bounds__(64 * kWaves) void glr_segment_kernel(SeqIn<T> f, SeqIn<T> x, const float *__restrict__ bias, SeqIn<uint8_t> resets,
                                                                  int T_, int64_t C, int H, int env_tiles, int batches, float *__restrict__ parts) {
    __shared__ float share[kWaves][3][64 * V];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), seg = blockIdx.y + (BACK ? 1 : 0);
    const Place at = place_of<V>(C, H, env_tiles);
    const int64_t c = at.c;
    const int j = at.j;
    const unsigned fo = lane_offset(f, at), xo = lane_offset(x, at);
    float b[V];
    Run r[V];
#pragma unroll
    for (int k = 0; k < V; k++) b[k] = bias ? bias[j + k] : 0.f, r[k] = {1.f, 0.f, 0.f};
    for (int i = 0; i < batches; i++) {
        const int64_t span = ((int64_t)seg * kWaves + w) * batches + (BACK ? batches - 1 - i : i), t0 = span * kSpan;
        if (t0 >= T_) continue;
        const int n = (int)(T_ - t0 < kSpan ? T_ - t0 : kSpan);
        typename Lane<T, V>::Vec fr[kSpan], xr[kSpan];
        span_load<T, V>(f, at, fo, t0, n, fr);
        span_load<T, V>(x, at, xo, t0, n, xr);
        unsigned rm = span_resets(resets, t0, n, at);
        float g[kSpan][V];
        span_gates<T, V>(fr, b, n, g);
        Run one[V];
        if (BACK) {
            span_run_back<T, V>(g, xr, rm, one);
        } else {
            float u[kSpan][V];
#pragma unroll
            for (int q = 0; q < kSpan; q++)
#pragma unroll
                for (int k = 0; k < V; k++) u[q][k] = gate_take(g[q][k]) * (float)xr[q][k];
            span_run<V>(g, u, rm, one);
        }
#pragma unroll
        for (int k = 0; k < V; k++) r[k] = run_join(r[k], one[k]);
    }
#pragma unroll
    for (int k = 0; k < V; k++) {
        share[w][0][lane * V + k] = r[k].A;
        share[w][1][lane * V + k] = r[k].D;
        share[w][2][lane * V + k] = r[k].B;
    }
    __syncthreads();
    if (w == 0 && at.mine) {
#pragma unroll
        for (int k = 0; k < V; k++) {
            Run all = {1.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < kWaves; i++) {
                const int q = BACK ? kWaves - 1 - i : i;
                all = run_join(all, Run{share[q][0][lane * V + k], share[q][1][lane * V + k], share[q][2][lane * V + k]});
            }
            float *o = parts + (int64_t)seg * 3 * C + c + k;
            o[0] = all.A, o[C] = all.D, o[2 * C] = all.B;
        }
    }
}

template <class T, int V>
__global__ __launch_bounds__(64 * kWaves) void glr_forward_kernel(SeqIn<T> f, SeqIn<T> x, const float *__restrict__ bias, SeqIn<uint8_t> resets,
                                                                  const float *h0, int T_, int64_t C, int H, int env_tiles, int batches,
                                                                  const float *__restrict__ parts, SeqOut<T> y, float *h_last,
                                                                  float *__restrict__ saved) {
    __shared__ float runs[2][kWaves][3][64 * V];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), seg = blockIdx.y;
    const Place at = place_of<V>(C, H, env_tiles);
    const int64_t c = at.c;
    const int j = at.j;
    const bool mine = at.mine;
    const unsigned fo = lane_offset(f, at), xo = lane_offset(x, at), yo = lane_offset(y, at);
    float b[V], h[V];
#pragma unroll
    for (int k = 0; k < V; k++) b[k] = bias ? bias[j + k] : 0.f, h[k] = h0 ? h0[c + k] : 0.f;
    if (seg > 0) segments_through<V, false>(parts, C, c, seg, gridDim.y, w, lane, runs[0], h);
    for (int i = 0; i < batches; i++) {
        const int64_t first = ((int64_t)seg * batches + i) * kWaves, t0 = (first + w) * kSpan;
        if (first * kSpan >= T_) break;
        const int n = (int)(T_ - t0 < kSpan ? T_ - t0 : kSpan);
        typename Lane<T, V>::Vec fr[kSpan], xr[kSpan];
        span_load<T, V>(f, at, fo, t0, n, fr);
        span_load<T, V>(x, at, xo, t0, n, xr);
        unsigned rm = span_resets(resets, t0, n, at);
        float g[kSpan][V], u[kSpan][V];
        span_gates<T, V>(fr, b, n, g);
#pragma unroll
        for (int q = 0; q < kSpan; q++)
#pragma unroll
            for (int k = 0; k < V; k++) u[q][k] = gate_take(g[q][k]) * (float)xr[q][k];
        auto &mem = runs[i & 1];
        Run r[V];
        span_run<V>(g, u, rm, r);
#pragma unroll
        for (int k = 0; k < V; k++) mem[w][0][lane * V + k] = r[k].A, mem[w][1][lane * V + k] = r[k].D, mem[w][2][lane * V + k] = r[k].B;
        afresh<V>(g, rm);
        __syncthreads();
        float in[V];
#pragma unroll
        for (int q = 0; q < kWaves; q++)
#pragma unroll
            for (int k = 0; k < V; k++) {
                if (q == w) in[k] = h[k];
                h[k] = run_through(Run{mem[q][0][lane * V + k], mem[q][1][lane * V + k], mem[q][2][lane * V + k]}, h[k]);
            }
        if (n <= 0) continue;
        if (saved && mine)
#pragma unroll
            for (int k = 0; k < V; k++) saved[(first + w) * C + c + k] = in[k];
        char *yp = (char *)(y.p + t0 * y.t + at.e0 * y.e);
        const int64_t ystep = distance(y);
        float out[V];
        bool bad = false;
#pragma unroll
        for (int k = 0; k < V; k++) out[k] = in[k];
#pragma unroll
        for (int q = 0; q < kSpan; q++) {
#pragma unroll
            for (int k = 0; k < V; k++) {
                out[k] = gate_pass(g[q][k], rm >> q & 1 ? 0.f : out[k]) + u[q][k];
                bad |= !(fabsf(out[k]) < INFINITY);
            }
            if (q < n && mine) step_store<T, V>(yp, ystep, yo, q, out);
        }
        if (__any(bad)) {
            afresh<V>(g, rm);
#pragma unroll
            for (int k = 0; k < V; k++) out[k] = in[k];
#pragma unroll
            for (int q = 0; q < kSpan; q++) {
#pragma unroll
                for (int k = 0; k < V; k++) out[k] = gate_pass_any(g[q][k], rm >> q & 1 ? 0.f : out[k]) + u[q][k];
                if (q < n && mine) step_store<T, V>(yp, ystep, yo, q, out);
            }
        }
        if (h_last && t0 + kSpan >= T_ && mine)
#pragma unroll
            for (int k = 0; k < V; k++) h_last[c + k] = out[k];
    }
}

template <class T, int V>
__global__ __launch_bounds__(64 * kWaves) void glr_backward_kernel(SeqIn<T> f, SeqIn<T> x, const float *__restrict__ bias, SeqIn<uint8_t> resets,
                                                                   const float *__restrict__ saved, SeqIn<T> dy, const float *__restrict__ dh_last,
                                                                   int T_, int64_t C, int H, int env_tiles, int batches, const float *__restrict__ parts,
                                                                   SeqOut<T> df, SeqOut<T> dx, float *__restrict__ dbias_part, float *__restrict__ dh0) {
    __shared__ float runs[2][kWaves][3][64 * V];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), seg = blockIdx.y;
    const Place at = place_of<V>(C, H, env_tiles);
    const int64_t c = at.c;
    const int j = at.j;
    const bool mine = at.mine;
    const unsigned fo = lane_offset(f, at), xo = lane_offset(x, at), go = lane_offset(dy, at), dfo = lane_offset(df, at), dxo = lane_offset(dx, at);
    float b[V], back[V];
    double total[V];
#pragma unroll
    for (int k = 0; k < V; k++) b[k] = bias ? bias[j + k] : 0.f, back[k] = dh_last ? dh_last[c + k] : 0.f, total[k] = 0.0;
    if (seg + 1 < (int)gridDim.y) segments_through<V, true>(parts, C, c, seg, gridDim.y, w, lane, runs[0], back);
    for (int i = batches - 1; i >= 0; i--) {
        const int64_t first = ((int64_t)seg * batches + i) * kWaves, t0 = (first + w) * kSpan;
        if (first * kSpan >= T_) continue;
        const int n = (int)(T_ - t0 < kSpan ? T_ - t0 : kSpan);
        typename Lane<T, V>::Vec fr[kSpan], xr[kSpan], gr[kSpan];
        span_load<T, V>(f, at, fo, t0, n, fr);
        span_load<T, V>(x, at, xo, t0, n, xr);
        span_load<T, V>(dy, at, go, t0, n, gr);
        float h[V];
#pragma unroll
        for (int k = 0; k < V; k++) h[k] = n > 0 ? saved[(first + w) * C + c + k] : 0.f;
        unsigned rm = span_resets(resets, t0, n, at);
        float g[kSpan][V], away[kSpan][V];                  // away: state in front of the step minus x
        span_gates<T, V>(fr, b, n, g);
        auto &mem = runs[i & 1];
        Run r[V];
        span_run_back<T, V>(g, gr, rm, r);
#pragma unroll
        for (int k = 0; k < V; k++) mem[w][0][lane * V + k] = r[k].A, mem[w][1][lane * V + k] = r[k].D, mem[w][2][lane * V + k] = r[k].B;
        afresh<V>(g, rm);
        bool bad = false;
#pragma unroll
        for (int q = 0; q < kSpan; q++)
#pragma unroll
            for (int k = 0; k < V; k++) {
                if (rm >> q & 1) h[k] = 0.f;
                away[q][k] = h[k] - (float)xr[q][k];
                bad |= !(fabsf(away[q][k]) < INFINITY);
                h[k] = gate_pass(g[q][k], h[k]) + gate_take(g[q][k]) * (float)xr[q][k];
            }
        if (__any(bad)) {
#pragma unroll
            for (int k = 0; k < V; k++) h[k] = n > 0 ? saved[(first + w) * C + c + k] : 0.f;
#pragma unroll
            for (int q = 0; q < kSpan; q++)
#pragma unroll
                for (int k = 0; k < V; k++) {
                    if (rm >> q & 1) h[k] = 0.f;
                    away[q][k] = h[k] - (float)xr[q][k];
                    h[k] = gate_pass_any(g[q][k], h[k]) + gate_take(g[q][k]) * (float)xr[q][k];
                }
        }
        afresh<V>(g, rm);
        __syncthreads();
        float in[V];
#pragma unroll
        for (int q = kWaves - 1; q >= 0; q--)
#pragma unroll
            for (int k = 0; k < V; k++) {
                if (q == w) in[k] = back[k];
                back[k] = run_through(Run{mem[q][0][lane * V + k], mem[q][1][lane * V + k], mem[q][2][lane * V + k]}, back[k]);
            }
        if (n <= 0) continue;
        char *fp = (char *)(df.p + t0 * df.t + at.e0 * df.e), *xp = (char *)(dx.p + t0 * dx.t + at.e0 * dx.e);
        const int64_t fstep = distance(df), xstep = distance(dx);
        float sum[V], c_in[V];
        bad = false;
#pragma unroll
        for (int k = 0; k < V; k++) sum[k] = 0.f, c_in[k] = in[k];
        auto walk = [&](auto pass) {
#pragma unroll
            for (int q = kSpan - 1; q >= 0; q--) {
                float of[V], ox[V];
#pragma unroll
                for (int k = 0; k < V; k++) {
                    const float v = g[q][k], gs = (float)gr[q][k] + in[k], take = gate_take(v);
                    ox[k] = take * gs;
                    of[k] = gs * away[q][k] * (fabsf(v) * (1.f - fabsf(v)));
                    in[k] = pass(v, gs);
                    bad |= !(fabsf(in[k]) < INFINITY);
                    if (rm >> q & 1) in[k] = 0.f;
                    if (q < n) sum[k] += of[k];
                }
                if (q < n && mine) {
                    step_store<T, V>(fp, fstep, dfo, q, of);
                    step_store<T, V>(xp, xstep, dxo, q, ox);
                }
            }
        };
        walk([](float v, float x) { return gate_pass(v, x); });
        if (__any(bad)) {
            afresh<V>(g, rm);
#pragma unroll
            for (int k = 0; k < V; k++) sum[k] = 0.f, in[k] = c_in[k];
            walk([](float v, float x) { return gate_pass_any(v, x); });
        }
#pragma unroll
        for (int k = 0; k < V; k++) total[k] += (double)sum[k];
        if (dh0 && t0 == 0 && mine)
#pragma unroll
            for (int k = 0; k < V; k++) dh0[c + k] = in[k];
    }
    if (dbias_part) {                                       // per segment and column: the waves' sums in wave order
        __shared__ double sums[kWaves][64 * V];
#pragma unroll
        for (int k = 0; k < V; k++) sums[w][lane * V + k] = total[k];
        __syncthreads();
        if (w == 0 && mine) {
#pragma unroll
            for (int k = 0; k < V; k++) {
                double s = 0.0;
#pragma unroll
                for (int q = 0; q < kWaves; q++) s += sums[q][lane * V + k];
                dbias_part[(int64_t)seg * C + c + k] = (float)s;
            }
        }
    }
}

// One step: every thread V channels, nothing to share.
template <class T, int V>
__global__ __launch_bounds__(256) void glr_step_kernel(SeqIn<T> f, SeqIn<T> x, const float *__restrict__ bias, SeqIn<uint8_t> resets,
                                                       const float *h0, int64_t C, int H, SeqOut<T> y, float *h_last, float *__restrict__ saved) {
    const int64_t c = ((int64_t)blockIdx.x * 256 + threadIdx.x) * V;
    if (c >= C) return;
    const int64_t e = c / H, j = c - e * H;
    const auto fr = Lane<T, V>::load(f.p + e * f.e + j), xr = Lane<T, V>::load(x.p + e * x.e + j);
    const bool fresh = resets.p && resets.p[e * resets.e];
    float h[V];
#pragma unroll
    for (int k = 0; k < V; k++) {
        h[k] = h0 ? h0[c + k] : 0.f;
        if (saved) saved[c + k] = h[k];
        if (fresh) h[k] = 0.f;
        const float g = gate_of<sizeof(T) == 4>(-(float)fr[k] - (bias ? bias[j + k] : 0.f));
        h[k] = gate_pass_any(g, h[k]) + gate_take(g) * (float)xr[k];
    }
    Lane<T, V>::store(y.p + e * y.e + j, h);
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

template <class T>
static SeqIn<T> seq_in(const ppo2hip_seq *s) {
    return s ? SeqIn<T>{(const T *)s->data, s->t, s->e} : SeqIn<T>{nullptr, 0, 0};
}
template <class T>
static SeqOut<T> seq_out(const ppo2hip_seq *s) {
    return SeqOut<T>{(T *)s->data, s->t, s->e};
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

// How a call is cut: V channels per lane, `segs` segments of `batches` batches of kBatch steps.
struct Cut {
    int V, batches, segs, env_tiles;
    int64_t tiles;
};
static Cut cut_of(int dtype, int T, int E, int H) {
    Cut k;
    const int64_t C = (int64_t)E * H;
    k.V = dtype != PPO2HIP_F32 && H % 2 == 0 ? 2 : 1;
    k.tiles = ceil_div(C, 64 * k.V);
    k.env_tiles = 0;
    const int64_t all = ceil_div(T, kBatch);
    int64_t segs = k.tiles >= 512 ? 1 : ceil_div(1024, k.tiles);
    if (segs > all) segs = all;
    k.batches = (int)ceil_div(all, segs);
    k.segs = (int)ceil_div(all, k.batches);
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

static size_t parts_bytes(const Cut &k, int64_t C) { return k.segs > 1 ? align_up((size_t)k.segs * 3 * C * sizeof(float), 256) : 0; }

extern "C" size_t ppo2hip_glr_forward_workspace_bytes(int dtype, int T, int E, int H) {
    if (T <= 1 || E <= 0 || H <= 0) return 0;
    return parts_bytes(cut_of(dtype, T, E, H), (int64_t)E * H);
}

extern "C" size_t ppo2hip_glr_backward_workspace_bytes(int dtype, int T, int E, int H, int want_dbias) {
    if (T <= 0 || E <= 0 || H <= 0) return 0;
    const Cut k = cut_of(dtype, T, E, H);
    const int64_t C = (int64_t)E * H, rows = (int64_t)k.segs * E;
    size_t n = parts_bytes(k, C);
    if (want_dbias) n += align_up((size_t)rows * H * sizeof(float), 256) + align_up((size_t)ceil_div(rows, kSumRows) * H * sizeof(float), 256);
    return n;
}

template <class T, int V>
static int forward_of(const Cut &k, int T_, int E, int H, const ppo2hip_seq *f, const ppo2hip_seq *x, const float *bias, const ppo2hip_seq *resets,
                      const float *h0, const ppo2hip_seq *y, float *h_last, float *saved, float *parts, hipStream_t s) {
    const int64_t C = (int64_t)E * H;
    if (T_ == 1) {
        hipLaunchKernelGGL((glr_step_kernel<T, V>), dim3((unsigned)ceil_div(C, 256 * V)), dim3(256), 0, s, seq_in<T>(f), seq_in<T>(x), bias,
                           seq_in<uint8_t>(resets), h0, C, H, seq_out<T>(y), h_last, saved);
        return check_launch("glr_step_kernel");
    }
    if (k.segs > 1) {
        hipLaunchKernelGGL((glr_segment_kernel<T, V, false>), dim3((unsigned)k.tiles, k.segs - 1), dim3(64 * kWaves), 0, s, seq_in<T>(f),
                           seq_in<T>(x), bias, seq_in<uint8_t>(resets), T_, C, H, k.env_tiles, k.batches, parts);
        int rc = check_launch("glr_segment_kernel");
        if (rc) return rc;
    }
    hipLaunchKernelGGL((glr_forward_kernel<T, V>), dim3((unsigned)k.tiles, k.segs), dim3(64 * kWaves), 0, s, seq_in<T>(f), seq_in<T>(x), bias,
                       seq_in<uint8_t>(resets), h0, T_, C, H, k.env_tiles, k.batches, parts, seq_out<T>(y), h_last, saved);
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
    Cut k = cut_of(dtype, T, E, H);
    place_envs(k, E, H, {f, x, resets, y});
    float *parts = (float *)workspace;
    PPO2HIP_REQUIRE(T == 1 || k.segs == 1 || parts, "glr_forward: workspace is null");
#define PPO2HIP_GLR_FORWARD(type, V) forward_of<type, V>(k, T, E, H, f, x, bias, resets, h0, y, h_last, saved, parts, s)
    if (dtype == PPO2HIP_F32) return PPO2HIP_GLR_FORWARD(float, 1);
    if (dtype == PPO2HIP_BF16) return k.V == 2 ? PPO2HIP_GLR_FORWARD(__bf16, 2) : PPO2HIP_GLR_FORWARD(__bf16, 1);
    return k.V == 2 ? PPO2HIP_GLR_FORWARD(_Float16, 2) : PPO2HIP_GLR_FORWARD(_Float16, 1);
#undef PPO2HIP_GLR_FORWARD
}

template <class T, int V>
static int backward_of(const Cut &k, int T_, int E, int H, const ppo2hip_seq *f, const ppo2hip_seq *x, const float *bias, const ppo2hip_seq *resets,
                       const float *saved, const ppo2hip_seq *dy, const float *dh_last, const ppo2hip_seq *df, const ppo2hip_seq *dx,
                       float *dbias, float *dh0, void *workspace, hipStream_t s) {
    const int64_t C = (int64_t)E * H, rows = (int64_t)k.segs * E;
    float *parts = (float *)workspace;
    float *sums = (float *)((char *)workspace + parts_bytes(k, C));
    int rc;
    if (k.segs > 1) {
        hipLaunchKernelGGL((glr_segment_kernel<T, V, true>), dim3((unsigned)k.tiles, k.segs - 1), dim3(64 * kWaves), 0, s, seq_in<T>(f),
                           seq_in<T>(dy), bias, seq_in<uint8_t>(resets), T_, C, H, k.env_tiles, k.batches, parts);
        if ((rc = check_launch("glr_segment_kernel"))) return rc;
    }
    hipLaunchKernelGGL((glr_backward_kernel<T, V>), dim3((unsigned)k.tiles, k.segs), dim3(64 * kWaves), 0, s, seq_in<T>(f), seq_in<T>(x), bias,
                       seq_in<uint8_t>(resets), saved, seq_in<T>(dy), dh_last, T_, C, H, k.env_tiles, k.batches, parts, seq_out<T>(df), seq_out<T>(dx),
                       dbias ? sums : nullptr, dh0);
    if ((rc = check_launch("glr_backward_kernel")) || !dbias) return rc;
    // rows [segment][env] of H channels each, 2048 rows to a workgroup, until one row is left
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
    Cut k = cut_of(dtype, T, E, H);
    place_envs(k, E, H, {f, x, resets, dy, df, dx});
    PPO2HIP_REQUIRE((!dbias && k.segs == 1) || workspace, "glr_backward: workspace is null");
#define PPO2HIP_GLR_BACKWARD(type, V) \
    backward_of<type, V>(k, T, E, H, f, x, bias, resets, saved, dy, dh_last, df, dx, dbias, dh0, workspace, s)
    if (dtype == PPO2HIP_F32) return PPO2HIP_GLR_BACKWARD(float, 1);
    if (dtype == PPO2HIP_BF16) return k.V == 2 ? PPO2HIP_GLR_BACKWARD(__bf16, 2) : PPO2HIP_GLR_BACKWARD(__bf16, 1);
    return k.V == 2 ? PPO2HIP_GLR_BACKWARD(_Float16, 2) : PPO2HIP_GLR_BACKWARD(_Float16, 1);
#undef PPO2HIP_GLR_BACKWARD
}
