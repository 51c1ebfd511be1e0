// Gated linear recurrence over a time-major sequence, forward and backward:
//   a = sigmoid(f + bias)   p = reset ? 0 : h[t-1]   h[t] = a p + (1 - a) x[t]
//   g[t] = dy[t] + (reset[t+1] ? 0 : a[t+1] g[t+1])   dx = (1 - a) g   df = g (p - x) a (1 - a)
// The backward pass recomputes the states from float32 states kept every PPO2HIP_GLR_SPAN steps: they cost
// 4 / SPAN bytes per element where reading y back costs its whole width, and y is rounded to its type while p - x cancels.
#include "kernels.hpp"

namespace ppo2hip {

constexpr int kSpan = PPO2HIP_GLR_SPAN;

// The gate as its smaller side s = min(a, 1 - a) <= 1/2, with `keep` telling whether it is 1 - a (z >= 0).  The larger
// side is 1 - s.  Formed this way both sides keep their relative accuracy: 1 - a taken from a rounded a loses the
// memory's length as soon as a is near one.
struct Gate {
    float s;
    bool keep;
};

__device__ inline Gate gate_of(float z) {
    float m = fabsf(z);
    m = m > 128.f ? 128.f : m;                   // e^-128 is 0 in float32; a NaN stays one
    const float t = m * -1.44269502f;            // e^-m as 2^t times the rest of t's rounding and of log2(e)'s
    const float rest = fmaf(m, -1.44269502f, -t) + m * -1.92596299e-8f;
    float e = __builtin_amdgcn_exp2f(t);
    e = fmaf(e * 0.693147182f, rest, e);
    const float d = 1.f + e;
    float r = __builtin_amdgcn_rcpf(d);
    r = fmaf(fmaf(-d, r, 1.f), r, r);
    return {e * r, z >= 0.f};
}

// a h + (1 - a) x as the larger side's operand plus s times the distance to the other one: one rounding of the size of
// the result's change.  Where the distance is not finite the products are formed one by one.
__device__ inline float gate_mix(Gate g, float h, float x) {
    const float base = g.keep ? h : x, other = g.keep ? x : h;
    const float d = other - base;
    return fabsf(d) < INFINITY ? fmaf(g.s, d, base) : fmaf(1.f - g.s, base, g.s * other);
}

// a v
__device__ inline float gate_keep(Gate g, float v) {
    return g.keep ? (fabsf(v) < INFINITY ? fmaf(-g.s, v, v) : (1.f - g.s) * v) : g.s * v;
}

// (1 - a) v
__device__ inline float gate_take(Gate g, float v) {
    return gate_keep({g.s, !g.keep}, v);
}

template <class T>
__device__ inline float to_f32(T v);
template <>
__device__ inline float to_f32<float>(float v) { return v; }
template <>
__device__ inline float to_f32<__bf16>(__bf16 v) { return (float)v; }
template <>
__device__ inline float to_f32<_Float16>(_Float16 v) { return (float)v; }

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

template <class T>
__global__ __launch_bounds__(64) void glr_forward_kernel(SeqIn<T> f, SeqIn<T> x, const float *__restrict__ bias, SeqIn<uint8_t> resets,
                                                         const float *h0, int T_, int64_t C, int H, SeqOut<T> y, float *h_last,
                                                         float *__restrict__ saved) {
    const int64_t c = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (c >= C) return;
    const int64_t e = c / H, j = c - e * H;
    float h = h0 ? h0[c] : 0.f;
    const float b = bias ? bias[j] : 0.f;
    for (int t = 0; t < T_; t++) {
        if (saved && t % kSpan == 0) saved[(int64_t)(t / kSpan) * C + c] = h;
        const Gate g = gate_of(to_f32(f.p[t * f.t + e * f.e + j]) + b);
        if (resets.p && resets.p[t * resets.t + e * resets.e]) h = 0.f;
        h = gate_mix(g, h, to_f32(x.p[t * x.t + e * x.e + j]));
        y.p[t * y.t + e * y.e + j] = (T)h;          // rounded to nearest: what the layer hands on; the state itself stays float32
    }
    if (h_last) h_last[c] = h;
}

template <class T>
__global__ __launch_bounds__(64) void glr_backward_kernel(SeqIn<T> f, SeqIn<T> x, const float *__restrict__ bias, SeqIn<uint8_t> resets,
                                                          const float *__restrict__ saved, SeqIn<T> dy, const float *__restrict__ dh_last,
                                                          int T_, int64_t C, int H, SeqOut<T> df, SeqOut<T> dx, float *__restrict__ dbias_part,
                                                          float *__restrict__ dh0) {
    const int64_t c = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (c >= C) return;
    const int64_t e = c / H, j = c - e * H;
    const float b = bias ? bias[j] : 0.f;
    float carry = dh_last ? dh_last[c] : 0.f, total = 0.f;
    for (int k = (T_ + kSpan - 1) / kSpan - 1; k >= 0; k--) {
        const int t0 = k * kSpan, n = T_ - t0 < kSpan ? T_ - t0 : kSpan;
        Gate g[kSpan];
        float xs[kSpan], before[kSpan], part = 0.f;
        float h = saved[(int64_t)k * C + c];
#pragma unroll
        for (int i = 0; i < kSpan; i++) {
            if (i < n) {
                const int64_t t = t0 + i;
                g[i] = gate_of(to_f32(f.p[t * f.t + e * f.e + j]) + b);
                xs[i] = to_f32(x.p[t * x.t + e * x.e + j]);
                if (resets.p && resets.p[t * resets.t + e * resets.e]) h = 0.f;
                before[i] = h;
                h = gate_mix(g[i], h, xs[i]);
            }
        }
#pragma unroll
        for (int i = kSpan - 1; i >= 0; i--) {
            if (i < n) {
                const int64_t t = t0 + i;
                const float gt = to_f32(dy.p[t * dy.t + e * dy.e + j]) + carry;
                const float d = gt * (before[i] - xs[i]) * (g[i].s * (1.f - g[i].s));
                dx.p[t * dx.t + e * dx.e + j] = (T)gate_take(g[i], gt);
                df.p[t * df.t + e * df.e + j] = (T)d;
                part += d;
                carry = resets.p && resets.p[t * resets.t + e * resets.e] ? 0.f : gate_keep(g[i], gt);
            }
        }
        total += part;
    }
    if (dbias_part) dbias_part[c] = total;
    if (dh0) dh0[c] = carry;
}

// dbias[j] = sum over the `rows` rows of part [rows, H], in row order per thread row and a fixed order over them
__global__ __launch_bounds__(256) void glr_dbias_kernel(const float *__restrict__ part, int64_t rows, int H, float *__restrict__ dbias) {
    __shared__ double red[4][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int j = blockIdx.x * 64 + lane;
    double s = 0.0;
    if (j < H)
        for (int64_t r = w; r < rows; r += 4) s += (double)part[r * H + j];
    red[w][lane] = s;
    __syncthreads();
    if (w == 0 && j < H) dbias[j] = (float)(red[0][lane] + red[1][lane] + red[2][lane] + red[3][lane]);
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

extern "C" size_t ppo2hip_glr_forward_workspace_bytes(int dtype, int T, int E, int H) {
    (void)dtype, (void)T, (void)E, (void)H;
    return 0;
}

extern "C" size_t ppo2hip_glr_backward_workspace_bytes(int dtype, int T, int E, int H, int want_dbias) {
    (void)dtype;
    if (T <= 0 || E <= 0 || H <= 0) return 0;
    return want_dbias ? align_up((size_t)E * H * sizeof(float), 256) : 0;
}

template <class T>
static int forward_of(int T_, int E, int H, const ppo2hip_seq *f, const ppo2hip_seq *x, const float *bias, const ppo2hip_seq *resets,
                      const float *h0, const ppo2hip_seq *y, float *h_last, float *saved, hipStream_t s) {
    const int64_t C = (int64_t)E * H;
    hipLaunchKernelGGL(glr_forward_kernel<T>, dim3((unsigned)ceil_div(C, 64)), dim3(64), 0, s, seq_in<T>(f), seq_in<T>(x), bias,
                       seq_in<uint8_t>(resets), h0, T_, C, H, seq_out<T>(y), h_last, saved);
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
    (void)workspace;
    if (dtype == PPO2HIP_F32) return forward_of<float>(T, E, H, f, x, bias, resets, h0, y, h_last, saved, s);
    if (dtype == PPO2HIP_BF16) return forward_of<__bf16>(T, E, H, f, x, bias, resets, h0, y, h_last, saved, s);
    return forward_of<_Float16>(T, E, H, f, x, bias, resets, h0, y, h_last, saved, s);
}

template <class T>
static int backward_of(int T_, int E, int H, const ppo2hip_seq *f, const ppo2hip_seq *x, const float *bias, const ppo2hip_seq *resets,
                       const float *saved, const ppo2hip_seq *dy, const float *dh_last, const ppo2hip_seq *df, const ppo2hip_seq *dx,
                       float *dbias, float *dh0, float *part, hipStream_t s) {
    const int64_t C = (int64_t)E * H;
    hipLaunchKernelGGL(glr_backward_kernel<T>, dim3((unsigned)ceil_div(C, 64)), dim3(64), 0, s, seq_in<T>(f), seq_in<T>(x), bias,
                       seq_in<uint8_t>(resets), saved, seq_in<T>(dy), dh_last, T_, C, H, seq_out<T>(df), seq_out<T>(dx), part, dh0);
    int rc = check_launch("glr_backward_kernel");
    if (rc || !dbias) return rc;
    hipLaunchKernelGGL(glr_dbias_kernel, dim3((unsigned)ceil_div(H, 64)), dim3(256), 0, s, part, (int64_t)E, H, dbias);
    return check_launch("glr_dbias_kernel");
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
    PPO2HIP_REQUIRE(!dbias || workspace, "glr_backward: workspace is null");
    float *part = dbias ? (float *)workspace : nullptr;
    if (dtype == PPO2HIP_F32) return backward_of<float>(T, E, H, f, x, bias, resets, saved, dy, dh_last, df, dx, dbias, dh0, part, s);
    if (dtype == PPO2HIP_BF16) return backward_of<__bf16>(T, E, H, f, x, bias, resets, saved, dy, dh_last, df, dx, dbias, dh0, part, s);
    return backward_of<_Float16>(T, E, H, f, x, bias, resets, saved, dy, dh_last, df, dx, dbias, dh0, part, s);
}
