// AdamW over a list of tensors, moments held in float32 or in 8 bits per block of 256 elements, in one launch; clipped by the
// global norm in two, in three for long lists, in one for those of few elements:
//   m = b1 m + (1 - b1) g    v = b2 v + (1 - b2) g^2    p -= lr (m / (1 - b1^t) / (sqrt(v / (1 - b2^t)) + eps) + wd p)
//   8 bits: m = sm sign(c) (c / 127)^2,  v = sv (c / 255)^4, sm and sv the block's largest |m| and v.
// The powers space the codes by a constant share of the square (fourth) root, so that a code's relative step is 2 / c
// (4 / c): 1.6 % at the block's largest element, and v reaches down to 2^-32 of it, where even steps would round all
// that is below 1/510 to zero and divide by epsilon alone.  A v that is not zero never gets code 0 for the same reason.
#include <cmath>

#include "kernels.hpp"

namespace ppo2hip {

constexpr int kBlock = PPO2HIP_ADAMW_BLOCK;      // elements of one scale
constexpr int kChunk = 2048;                     // elements a workgroup takes at a time: 8 per thread, 8 blocks of 8-bit moments
constexpr int kThreads = 256;
constexpr int kMaxGrads = 448;                   // gradient pointers of one launch: they ride in its 4 KB of arguments
constexpr int kNormGroups = 4096;                // most workgroups of the norm launch, each with a partial sum
// Up to kOwnChunks chunks every workgroup of the step adds up the norm's partial sums, kOwnSums at most, by itself; beyond, one more
// launch does.  By itself / by the launch, us per replay, 32-bit and 8-bit moments: 64 chunks 7.6 / 8.9 and 10.0 / 11.3, 512: 10.0 /
// 11.0 and 11.5 / 12.6, 2048: 24.7 / 25.9 and 25.7 / 25.7, 4096: 46.5 / 47.0 and 43.1 / 41.1, 8192: 92 / 87 and 74 / 65.  256, 512, 1024 sums:
// 1235 chunks 17.8, 17.0, 16.5 and 17.4, 16.9, 17.1, 2048 chunks 28.1, 24.7, 24.4 and 28.2, 25.7, 25.2.
constexpr int kOwnSums = 512;
constexpr int kOwnChunks = 2048;
constexpr int kSmallThreads = 1024, kSmallChunks = 32;   // chunks up to which every workgroup of the step sums all squares itself

struct TensorRow {                               // one tensor in the device image of a plan
    void *p;
    int64_t n;                                   // elements
    int64_t off;                                 // first element in the moments
    int32_t p_type, g_type;
    float decay;
    int32_t pad;
};
struct ChunkRow {
    int32_t tensor, index;                       // chunk `index` of kChunk elements of that tensor
};

struct AdamwArgs {
    const TensorRow *tensors;
    const ChunkRow *chunks;
    int32_t first_tensor, nchunks;               // of this launch
    void *m, *v;
    float *m_scale, *v_scale;
    const double *partial;
    int32_t npartial;                            // 0: the factor is found already
    float lr, c1, c2, b1, b2, omb1, omb2, eps, wd, gscale, max_norm;
    float *norm_out;
    const float *factor;
    const void *g[kMaxGrads];
};
static_assert(sizeof(AdamwArgs) <= 4096, "arguments beyond what a launch carries");

struct NormArgs {
    const TensorRow *tensors;
    const ChunkRow *chunks;
    int32_t first_tensor, nchunks;
    double *partial;
    float gscale;
    const void *g[kMaxGrads];
};

// four elements from any element-aligned address: one wide load where all four exist
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef f32x4 f32x4_any __attribute__((aligned(4)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef bf16x4 bf16x4_any __attribute__((aligned(2)));

__device__ inline f32x4 load4(const void *base, int type, int64_t i, int64_t n) {
    f32x4 r = {0.f, 0.f, 0.f, 0.f};
    if (type == PPO2HIP_F32) {
        const float *p = (const float *)base + i;
        if (i + 4 <= n) return *(const f32x4_any *)p;
#pragma unroll
        for (int k = 0; k < 3; k++)
            if (i + k < n) r[k] = p[k];
    } else {
        const __bf16 *p = (const __bf16 *)base + i;
        if (i + 4 <= n) return __builtin_convertvector(*(const bf16x4_any *)p, f32x4);
#pragma unroll
        for (int k = 0; k < 3; k++)
            if (i + k < n) r[k] = (float)p[k];
    }
    return r;
}
// a bfloat16 parameter is rounded to nearest: an update below half its step is lost, as in any bfloat16 weight without a
// wider copy
__device__ inline void store4(void *base, int type, int64_t i, int64_t n, f32x4 v) {
    if (type == PPO2HIP_F32) {
        float *p = (float *)base + i;
        if (i + 4 <= n) *(f32x4_any *)p = v;
        else
#pragma unroll
            for (int k = 0; k < 3; k++)
                if (i + k < n) p[k] = v[k];
    } else {
        __bf16 *p = (__bf16 *)base + i;
        if (i + 4 <= n) *(bf16x4_any *)p = __builtin_convertvector(v, bf16x4);
        else
#pragma unroll
            for (int k = 0; k < 3; k++)
                if (i + k < n) p[k] = (__bf16)v[k];
    }
}

// The values codes stand for.  The integer powers are exact (a fourth power past 2^24 rounds once), so that what is raised
// carries no rounding that the power would multiply.
__device__ inline float moment_of(int8_t c, float scale) {
    const float x = (float)c;
    return scale * (x * fabsf(x) * (1.f / 16129.f));
}
__device__ inline float square_of(uint8_t c, float scale) {
    const float x = (float)((unsigned)c * c);
    return scale * (x * x * (1.f / 4228250625.f));
}

constexpr int kParts = kChunk / (4 * kThreads);      // four-element parts of a chunk that a thread has

// The squares of chunk c, THREADS threads with `thread` among them sharing it.  In 64 bits: squares of float32 leave its range.
template <int THREADS, class Args>
__device__ inline double chunk_squares(const Args &a, int c, int thread) {
    constexpr int kParts = kChunk / (4 * THREADS);
    const ChunkRow ch = a.chunks[c];
    const TensorRow &t = a.tensors[ch.tensor];
    const void *g = a.g[ch.tensor - a.first_tensor];
    const int64_t n = g ? t.n : 0;
    f32x4 x[kParts];
#pragma unroll
    for (int u = 0; u < kParts; u++) x[u] = load4(g, t.g_type, (int64_t)ch.index * kChunk + u * (4 * THREADS) + thread * 4, n);
    double s = 0.0;
#pragma unroll
    for (int u = 0; u < kParts; u++)
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const double d = (double)(x[u][k] * a.gscale);
            s += d * d;
        }
    return s;
}

// Partial sums of the squares, a fixed number of workgroups that walk the chunks: 504 MB in 111 to 127 us (4.0 to 4.5 TB/s; 90 at best).
__global__ __launch_bounds__(kThreads) void adamw_norm_kernel(NormArgs a) {
    __shared__ double red[17];
    double s = 0.0;
    for (int c = blockIdx.x; c < a.nchunks; c += gridDim.x) s += chunk_squares<kThreads>(a, c, threadIdx.x);
    s = block_sum(s, red);
    if (threadIdx.x == 0) a.partial[blockIdx.x] = s;
}

__device__ inline float norm_of(const double *partial, int n, double *red) {
    double s = 0.0;
    for (int i = threadIdx.x; i < n; i += blockDim.x) s += partial[i];
    return (float)sqrt(block_sum(s, red));
}
// not fmaxf: a norm that is not a number stays one
__device__ inline float factor_of(float norm, float gscale, float max_norm) {
    return gscale * (norm > max_norm ? max_norm / norm : (norm <= max_norm ? 1.f : norm));
}
// {norm, factor} for lists of many chunks: one workgroup adds up what every workgroup of the step would have to
__global__ __launch_bounds__(1024) void adamw_factor_kernel(const double *partial, int npartial, float gscale, float max_norm, float *factor, float *norm_out) {
    __shared__ double red[17];
    const float norm = norm_of(partial, npartial, red);
    if (threadIdx.x == 0) {
        factor[0] = norm;
        factor[1] = factor_of(norm, gscale, max_norm);
        if (norm_out) norm_out[0] = norm, norm_out[1] = factor[1];
    }
}

__device__ inline unsigned wave_umax(unsigned v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const unsigned w = (unsigned)__shfl_xor((int)v, o, 64);
        v = v > w ? v : w;
    }
    return v;
}

// The codes of a wave's block of 256, four elements to a lane, and their scale: the largest bit pattern, so that an infinity or
// a NaN wins over every finite value; its block then decodes to NaN instead of to something that looks sound.  Roots of the
// ratio to the scale, by the hardware's root (off by 2^-23 of its value, of a code's place by 3e-5 of a step at most).
template <int ROOT>
__device__ inline unsigned encode(const f32x4 &v, float &scale) {
    constexpr float kTop = ROOT == 2 ? 127.f : 255.f;
    unsigned top = 0;
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const unsigned x = __float_as_uint(v[k]) & 0x7fffffffu;
        top = top > x ? top : x;
    }
    top = wave_umax(top);
    const bool sound = top < 0x7f800000u;
    scale = sound ? __uint_as_float(top) : __builtin_nanf("");
    // a scale whose reciprocal would leave float32 is lifted together with its block
    const float lift = scale < 0x1p-100f ? 0x1p120f : 1.f, inv = scale > 0.f ? 1.f / (scale * lift) : 0.f;
    unsigned codes = 0;
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const float ratio = sound ? fabsf(v[k]) * lift * inv : 0.f;
        float root = __builtin_amdgcn_sqrtf(ratio);
        if (ROOT == 4) root = __builtin_amdgcn_sqrtf(root);
        int c = (int)rintf(root * kTop);
        c = c < (int)kTop ? c : (int)kTop;
        if (ROOT == 4) {
            if (sound && v[k] > 0.f && c == 0) c = 1;
        } else {
            c = v[k] < 0.f ? -c : c;
        }
        codes |= (unsigned)(c & 255) << (8 * k);
    }
    return codes;
}

// m / (sqrt(v) + eps).  The hardware's root and reciprocal are each off by an ulp, a step's 4 x 2^-24 against a parameter that rounds
// by 2^-24 of itself.  They may flush a denormal, whose root is at most 1.1e-19: an epsilon under 2^24 of that takes the exact ones.
__device__ inline float over_root(float m, float v, float eps) {
    if (eps >= 1e-11f) return m * __builtin_amdgcn_rcpf(__builtin_amdgcn_sqrtf(v) + eps);
    return m / (sqrtf(v) + eps);
}

// THREADS kThreads: a workgroup per chunk.  kSmallThreads, for lists of at most kSmallChunks chunks that are clipped: the same,
// after its waves have summed the squares of the whole list, so that the norm needs no launch of its own.  In one launch / in two, us
// per replay, 32-bit moments: 24 chunks 6.5 / 7.1, 32 chunks 7.9 / 7.2, 64 chunks 11.5 / 7.2; 8-bit, 32 chunks: 8.7 / 9.3.  An eager
// call, which waits for the host, takes 3 us less in one.
// Bound by memory: 126 M parameters in 100 tensors, float32 moments 3.5 GB in 638 us (5.5 TB/s), 8 bits 2.0 GB in 355 (5.7); 43 M
// bfloat16 ones 1.0 GB in 182 (5.3).
template <int BITS, int THREADS>
__global__ __launch_bounds__(THREADS) void adamw_kernel(AdamwArgs a) {
    constexpr int kParts = (kChunk + 4 * THREADS - 1) / (4 * THREADS);
    __shared__ double red[17];
    const ChunkRow ch = a.chunks[blockIdx.x];
    const TensorRow t = a.tensors[ch.tensor];
    const void *gp = a.g[ch.tensor - a.first_tensor];
    const int64_t i0 = (int64_t)ch.index * kChunk + threadIdx.x * 4;
    const bool works = gp && (int)threadIdx.x * 4 < kChunk;
    // this thread's elements are on their way while the norm is added up
    f32x4 g[kParts], p[kParts], m[kParts], v[kParts];
    unsigned mc[kParts], vc[kParts];
    float sm[kParts], sv[kParts];
#pragma unroll
    for (int u = 0; u < kParts; u++) {
        const int64_t i = i0 + u * (4 * THREADS), n = works ? t.n : 0;
        g[u] = load4(gp, t.g_type, i, n);
        p[u] = load4(t.p, t.p_type, i, n);
        if (BITS == 32) {
            m[u] = load4((const float *)a.m + t.off, PPO2HIP_F32, i, n);
            v[u] = load4((const float *)a.v + t.off, PPO2HIP_F32, i, n);
        } else {
            mc[u] = vc[u] = 0;
            sm[u] = sv[u] = 0.f;
            if (i - (threadIdx.x & 63) * 4 < n) {            // whole blocks: the codes reach to a block's end
                mc[u] = ((const unsigned *)a.m)[(t.off + i) / 4];
                vc[u] = ((const unsigned *)a.v)[(t.off + i) / 4];
                sm[u] = a.m_scale[(t.off + i) / kBlock];
                sv[u] = a.v_scale[(t.off + i) / kBlock];
            }
        }
    }
    float scale = a.gscale;
    if (a.max_norm > 0.f && a.npartial == 0) {
        scale = a.factor[1];
    } else {
        if (a.max_norm > 0.f) {
            float norm;
            if (THREADS == kSmallThreads) {
                double sum = 0.0;
                for (int c = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); c < a.nchunks; c += THREADS / 64) sum += chunk_squares<64>(a, c, threadIdx.x & 63);
                norm = (float)sqrt(block_sum(sum, red));
            } else {
                norm = norm_of(a.partial, a.npartial, red);
            }
            scale = factor_of(norm, a.gscale, a.max_norm);
            if (a.norm_out && blockIdx.x == 0 && threadIdx.x == 0) a.norm_out[0] = norm;
        }
        if (a.norm_out && blockIdx.x == 0 && threadIdx.x == 0) a.norm_out[1] = scale;
    }
    if (!works) return;
    const float wd = a.wd * t.decay;
#pragma unroll
    for (int u = 0; u < kParts; u++) {
        const int64_t i = i0 + u * (4 * THREADS);
#pragma unroll
        for (int k = 0; k < 4; k++) {
            if (BITS == 8) {
                m[u][k] = moment_of((int8_t)(mc[u] >> (8 * k)), sm[u]);
                v[u][k] = square_of((uint8_t)(vc[u] >> (8 * k)), sv[u]);
            }
            const float gs = g[u][k] * scale;
            m[u][k] = a.b1 * m[u][k] + a.omb1 * gs;
            v[u][k] = a.b2 * v[u][k] + a.omb2 * (gs * gs);
            p[u][k] = p[u][k] - a.lr * (over_root(m[u][k] * a.c1, v[u][k] * a.c2, a.eps) + wd * p[u][k]);
            if (BITS == 8 && i + k >= t.n) m[u][k] = 0.f, v[u][k] = 0.f;
        }
        if (i < t.n) store4(t.p, t.p_type, i, t.n, p[u]);
        if (BITS == 32) {
            if (i < t.n) {
                store4((float *)a.m + t.off, PPO2HIP_F32, i, t.n, m[u]);
                store4((float *)a.v + t.off, PPO2HIP_F32, i, t.n, v[u]);
            }
        } else if (i - (threadIdx.x & 63) * 4 < t.n) {
            mc[u] = encode<2>(m[u], sm[u]);
            vc[u] = encode<4>(v[u], sv[u]);
            ((unsigned *)a.m)[(t.off + i) / 4] = mc[u];
            ((unsigned *)a.v)[(t.off + i) / 4] = vc[u];
            if ((threadIdx.x & 63) == 0) {
                a.m_scale[(t.off + i) / kBlock] = sm[u];
                a.v_scale[(t.off + i) / kBlock] = sv[u];
            }
        }
    }
}

// moments as the values they stand for, packed in list order (no padding between tensors): 126 M, 760 MB in 151 us (5.0 TB/s)
template <class T>
__global__ __launch_bounds__(kThreads) void adamw_state_kernel(const TensorRow *tensors, const ChunkRow *chunks, const int64_t *packed, int nchunks,
                                                               const unsigned *mc_, const unsigned *vc_, const float *m_scale, const float *v_scale,
                                                               T *m_out, T *v_out) {
    const int type = sizeof(T) == 4 ? PPO2HIP_F32 : PPO2HIP_BF16;
    const ChunkRow ch = chunks[blockIdx.x];
    const TensorRow t = tensors[ch.tensor];
    const int64_t at = packed[ch.tensor], i0 = (int64_t)ch.index * kChunk + threadIdx.x * 4;
    unsigned mc[kParts], vc[kParts];
    float sm[kParts], sv[kParts];
#pragma unroll
    for (int u = 0; u < kParts; u++) {
        const int64_t i = i0 + u * (4 * kThreads);
        if (i < t.n) {
            mc[u] = mc_[(t.off + i) / 4], vc[u] = vc_[(t.off + i) / 4];
            sm[u] = m_scale[(t.off + i) / kBlock], sv[u] = v_scale[(t.off + i) / kBlock];
        }
    }
#pragma unroll
    for (int u = 0; u < kParts; u++) {
        const int64_t i = i0 + u * (4 * kThreads);
        if (i < t.n) {
            f32x4 m, v;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                m[k] = moment_of((int8_t)(mc[u] >> (8 * k)), sm[u]);
                v[k] = square_of((uint8_t)(vc[u] >> (8 * k)), sv[u]);
            }
            store4(m_out + at, type, i, t.n, m);
            store4(v_out + at, type, i, t.n, v);
        }
    }
}

}  // namespace ppo2hip

using namespace ppo2hip;

static int64_t chunks_of(int64_t n) { return ceil_div(n, kChunk); }

static int adamw_check(const char *what, const ppo2hip_adamw_tensor *t, int nt, int bits) {
    PPO2HIP_REQUIRE(nt >= 0 && (t || nt == 0), "%s: bad tensor list", what);
    PPO2HIP_REQUIRE(bits == 32 || bits == 8, "%s: moments in %d bits (32 and 8 exist)", what, bits);
    int64_t chunks = 0;
    for (int k = 0; k < nt; k++) {
        PPO2HIP_REQUIRE(t[k].n >= 0 && (t[k].param || t[k].n == 0), "%s: tensor %d is null or has a negative size", what, k);
        PPO2HIP_REQUIRE((t[k].param_dtype == PPO2HIP_F32 || t[k].param_dtype == PPO2HIP_BF16) &&
                            (t[k].grad_dtype == PPO2HIP_F32 || t[k].grad_dtype == PPO2HIP_BF16),
                        "%s: tensor %d: parameters and gradients are float32 or bfloat16", what, k);
        PPO2HIP_REQUIRE(t[k].n <= (1ll << 42), "%s: tensor %d is too large", what, k);
        chunks += chunks_of(t[k].n);
    }
    PPO2HIP_REQUIRE(chunks < (1ll << 32) / kThreads, "%s: %lld elements in one list (a launch holds 2^32 threads)", what, (long long)(chunks * kChunk));
    return PPO2HIP_OK;
}

struct PlanShape {
    size_t chunk_off, packed_off, bytes;
};
static PlanShape plan_shape(const ppo2hip_adamw_tensor *t, int nt) {
    int64_t chunks = 0;
    for (int k = 0; k < nt; k++) chunks += chunks_of(t[k].n);
    PlanShape s;
    s.packed_off = align_up(nt * sizeof(TensorRow), 16);
    s.chunk_off = align_up(s.packed_off + nt * sizeof(int64_t), 16);
    s.bytes = align_up(s.chunk_off + chunks * sizeof(ChunkRow), 16) + 16;
    return s;
}

extern "C" int64_t ppo2hip_adamw_state_elements(const ppo2hip_adamw_tensor *tensors, int ntensors, int state_bits) {
    int rc = adamw_check("adamw_state_elements", tensors, ntensors, state_bits);
    if (rc) return rc;
    int64_t n = 0;
    for (int k = 0; k < ntensors; k++) n += state_bits == 32 ? tensors[k].n : ceil_div(tensors[k].n, kBlock) * kBlock;
    return n;
}

extern "C" size_t ppo2hip_adamw_plan_bytes(const ppo2hip_adamw_tensor *tensors, int ntensors) {
    if (adamw_check("adamw_plan_bytes", tensors, ntensors, 32)) return 0;
    return plan_shape(tensors, ntensors).bytes;
}

extern "C" int ppo2hip_adamw_plan_fill(const ppo2hip_adamw_tensor *tensors, int ntensors, int state_bits, void *image, size_t image_bytes) {
    int rc = adamw_check("adamw_plan_fill", tensors, ntensors, state_bits);
    if (rc) return rc;
    const PlanShape s = plan_shape(tensors, ntensors);
    PPO2HIP_REQUIRE(image, "adamw_plan_fill: image is null");
    if (image_bytes < s.bytes) {
        set_error("adamw_plan_fill: image of %zu bytes, %zu needed", image_bytes, s.bytes);
        return PPO2HIP_ENOSPACE;
    }
    TensorRow *rows = (TensorRow *)image;
    int64_t *packed = (int64_t *)((char *)image + s.packed_off);
    ChunkRow *chunks = (ChunkRow *)((char *)image + s.chunk_off);
    int64_t off = 0, at = 0;
    for (int k = 0; k < ntensors; k++) {
        const ppo2hip_adamw_tensor &t = tensors[k];
        rows[k] = TensorRow{t.param, t.n, off, t.param_dtype, t.grad_dtype, t.decay, 0};
        packed[k] = at;
        for (int64_t c = 0; c < chunks_of(t.n); c++) *chunks++ = ChunkRow{k, (int32_t)c};
        off += state_bits == 32 ? t.n : ceil_div(t.n, kBlock) * kBlock;
        at += t.n;
    }
    return PPO2HIP_OK;
}

extern "C" size_t ppo2hip_adamw_workspace_bytes(const ppo2hip_adamw_tensor *tensors, int ntensors) {
    (void)tensors;
    const int64_t launches = ceil_div(ntensors > 0 ? ntensors : 1, kMaxGrads);
    return 16 + (size_t)launches * kNormGroups * sizeof(double);
}

extern "C" int ppo2hip_adamw_step(const ppo2hip_adamw_tensor *tensors, int ntensors, int state_bits, const void *plan, const void *const *grads,
                                  void *m, float *m_scale, void *v, float *v_scale, double lr, int64_t t, double beta1, double beta2,
                                  double epsilon, double weight_decay, double grad_scale, double max_grad_norm, float *norm_out,
                                  void *workspace, size_t workspace_bytes, void *stream) {
    int rc = adamw_check("adamw_step", tensors, ntensors, state_bits);
    if (rc) return rc;
    PPO2HIP_REQUIRE(t >= 1, "adamw_step: step count t=%lld must be at least 1", (long long)t);
    PPO2HIP_REQUIRE(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0, "adamw_step: beta1=%g, beta2=%g outside [0, 1)", beta1, beta2);
    PPO2HIP_REQUIRE(epsilon >= 0.0, "adamw_step: epsilon=%g is negative", epsilon);
    PPO2HIP_REQUIRE(max_grad_norm <= 0.0 || (float)max_grad_norm > 0.f, "adamw_step: max_grad_norm=%g is not a norm in float32", max_grad_norm);
    PPO2HIP_REQUIRE((uintptr_t)workspace % 16 == 0 && (uintptr_t)plan % 16 == 0, "adamw_step: plan and workspace must be aligned to 16 bytes");
    const PlanShape shape = plan_shape(tensors, ntensors);
    int64_t total = 0;
    for (int k = 0; k < ntensors; k++) total += tensors[k].n;
    if (total == 0) return PPO2HIP_OK;
    PPO2HIP_REQUIRE(plan && grads && m && v, "adamw_step: null pointer");
    PPO2HIP_REQUIRE(state_bits == 32 || (m_scale && v_scale), "adamw_step: 8-bit moments need their scales");
    const bool clip = max_grad_norm > 0.0;
    if (clip && (!workspace || workspace_bytes < ppo2hip_adamw_workspace_bytes(tensors, ntensors))) {
        set_error("adamw_step: workspace of %zu bytes, %zu needed to clip", workspace ? workspace_bytes : (size_t)0,
                  ppo2hip_adamw_workspace_bytes(tensors, ntensors));
        return PPO2HIP_ENOSPACE;
    }
    hipStream_t s = (hipStream_t)stream;
    const TensorRow *rows = (const TensorRow *)plan;
    const ChunkRow *chunks = (const ChunkRow *)((const char *)plan + shape.chunk_off);
    float *factor = (float *)workspace;
    double *partial = (double *)((char *)workspace + 16);
    int npartial = 0;
    int64_t all_chunks = 0;
    for (int k = 0; k < ntensors; k++) all_chunks += chunks_of(tensors[k].n);
    const bool small = clip && all_chunks <= kSmallChunks && ntensors <= kMaxGrads;
    if (small) npartial = 1;                                 // not 0
    if (clip && !small) {
        int64_t chunk = 0;
        for (int k0 = 0; k0 < ntensors; k0 += kMaxGrads) {
            NormArgs a;
            a.tensors = rows;
            a.chunks = chunks + chunk;
            a.first_tensor = k0;
            a.partial = partial + npartial;
            a.gscale = (float)grad_scale;
            int64_t here = 0;
            for (int k = k0; k < ntensors && k < k0 + kMaxGrads; k++) {
                a.g[k - k0] = grads[k];
                here += chunks_of(tensors[k].n);
            }
            a.nchunks = (int32_t)here;
            chunk += here;
            if (here == 0) continue;
            const int most = all_chunks <= kOwnChunks ? kOwnSums : kNormGroups;
            const int groups = (int)(here < most ? here : most);
            hipLaunchKernelGGL(adamw_norm_kernel, dim3(groups), dim3(kThreads), 0, s, a);
            if ((rc = check_launch("adamw_norm_kernel"))) return rc;
            npartial += groups;
        }
    }
    if (clip && all_chunks > kOwnChunks) {
        hipLaunchKernelGGL(adamw_factor_kernel, dim3(1), dim3(1024), 0, s, partial, npartial, (float)grad_scale, (float)max_grad_norm, factor, norm_out);
        if ((rc = check_launch("adamw_factor_kernel"))) return rc;
        npartial = 0;
    }
    AdamwArgs a;
    a.factor = factor;
    a.tensors = rows;
    a.m = m;
    a.v = v;
    a.m_scale = m_scale;
    a.v_scale = v_scale;
    a.partial = partial;
    a.npartial = npartial;
    a.lr = (float)lr;
    a.c1 = (float)(1.0 / (1.0 - pow(beta1, (double)t)));
    a.c2 = (float)(1.0 / (1.0 - pow(beta2, (double)t)));
    a.b1 = (float)beta1;
    a.b2 = (float)beta2;
    a.omb1 = (float)(1.0 - beta1);               // formed in 64 bits: 1.f - 0.999f is off by 4.7e-5 of its value
    a.omb2 = (float)(1.0 - beta2);
    a.eps = (float)epsilon;
    a.wd = (float)weight_decay;
    a.gscale = (float)grad_scale;
    a.max_norm = clip ? (float)max_grad_norm : 0.f;
    a.norm_out = norm_out;
    int64_t chunk = 0;
    for (int k0 = 0; k0 < ntensors; k0 += kMaxGrads) {
        a.first_tensor = k0;
        a.chunks = chunks + chunk;
        int64_t here = 0;
        for (int k = k0; k < ntensors && k < k0 + kMaxGrads; k++) {
            a.g[k - k0] = grads[k];
            here += chunks_of(tensors[k].n);
        }
        a.nchunks = (int32_t)here;
        chunk += here;
        if (here == 0) continue;
        if (small && state_bits == 32)
            hipLaunchKernelGGL((adamw_kernel<32, kSmallThreads>), dim3((unsigned)here), dim3(kSmallThreads), 0, s, a);
        else if (small)
            hipLaunchKernelGGL((adamw_kernel<8, kSmallThreads>), dim3((unsigned)here), dim3(kSmallThreads), 0, s, a);
        else if (state_bits == 32)
            hipLaunchKernelGGL((adamw_kernel<32, kThreads>), dim3((unsigned)here), dim3(kThreads), 0, s, a);
        else
            hipLaunchKernelGGL((adamw_kernel<8, kThreads>), dim3((unsigned)here), dim3(kThreads), 0, s, a);
        if ((rc = check_launch("adamw_kernel"))) return rc;
        a.norm_out = nullptr;
    }
    return PPO2HIP_OK;
}

extern "C" int ppo2hip_adamw_state(const ppo2hip_adamw_tensor *tensors, int ntensors, const void *plan, const void *m, const float *m_scale,
                                   const void *v, const float *v_scale, int out_dtype, void *m_out, void *v_out, void *stream) {
    int rc = adamw_check("adamw_state", tensors, ntensors, 8);
    if (rc) return rc;
    PPO2HIP_REQUIRE(out_dtype == PPO2HIP_F32 || out_dtype == PPO2HIP_BF16, "adamw_state: outputs are float32 or bfloat16");
    int64_t nchunks = 0;
    for (int k = 0; k < ntensors; k++) nchunks += chunks_of(tensors[k].n);
    if (nchunks == 0) return PPO2HIP_OK;
    PPO2HIP_REQUIRE(plan && m && m_scale && v && v_scale && m_out && v_out, "adamw_state: null pointer");
    const PlanShape shape = plan_shape(tensors, ntensors);
    const TensorRow *rows = (const TensorRow *)plan;
    const int64_t *packed = (const int64_t *)((const char *)plan + shape.packed_off);
    const ChunkRow *chunks = (const ChunkRow *)((const char *)plan + shape.chunk_off);
    const unsigned groups = (unsigned)nchunks;
    hipStream_t s = (hipStream_t)stream;
    if (out_dtype == PPO2HIP_F32)
        hipLaunchKernelGGL(adamw_state_kernel<float>, dim3(groups), dim3(kThreads), 0, s, rows, chunks, packed, (int)nchunks, (const unsigned *)m,
                           (const unsigned *)v, m_scale, v_scale, (float *)m_out, (float *)v_out);
    else
        hipLaunchKernelGGL(adamw_state_kernel<__bf16>, dim3(groups), dim3(kThreads), 0, s, rows, chunks, packed, (int)nchunks, (const unsigned *)m,
                           (const unsigned *)v, m_scale, v_scale, (__bf16 *)m_out, (__bf16 *)v_out);
    return check_launch("adamw_state_kernel");
}
