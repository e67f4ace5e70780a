// GroupNorm + activation (+ residual added before the activation) over NHWC tensors, forward and backward.
//
//   mean, var over one image's H*W pixels x the k = C/groups channels of a group;  rstd = (var + eps)^-1/2
//   pre = (x - mean) * rstd * gamma + beta (+ residual),  y = act(pre)
//   g = dy * act'(pre);  S1 = sum_pixels g,  S2 = sum_pixels g * xhat  per (image, channel)
//   dbeta = sum_images S1,  dgamma = sum_images S2
//   P1 = sum_group gamma * S1 / M,  P2 = sum_group gamma * S2 / M  (M = H*W*k)
//   dx = rstd * (gamma * g - P1 - xhat * P2),  dresidual = g
//
// Everything is bound by HBM: forward reads x (and the residual) and writes y, backward reads dy, x (and the residual) and
// writes dx (and the residual's gradient).
//
// Arithmetic.  The statistics are plain sums of x and x^2 in 64 bits: fp64 vector arithmetic runs at the fp32 rate here, a
// sum costs four instructions per element against a budget of about thirteen at the HBM rate, and E[x^2] - mean^2 then
// keeps full precision however large the mean is.  The passes over the elements run in fp32 with the mean split into its
// fp32 value and the rest: d = x - mean_hi (exact for x near the mean), pre = d * A + B with A = rstd * gamma and
// B = beta - mean_lo * A.  The activations with a kink have a gradient that jumps there, and bf16 inputs take few distinct
// values, so one pre-activation on the wrong side of a kink by a rounding would put thousands of elements on the wrong
// side: within the fp32 error of a kink the backward pass evaluates pre again in 64 bits (rare, one comparison otherwise).
#include "ur_common.h"

namespace {

constexpr int NT = 256;

typedef __attribute__((ext_vector_type(4))) float fvec4_t;

// V consecutive channels of one pixel: 16 bytes (8 bf16, 4 fp32) or one element
template <typename T, int V> struct Chunk;
template <> struct Chunk<bf16_t, 8> {
    bf16x8_t d;
    __device__ __forceinline__ void load(const bf16_t* p) { d = __builtin_nontemporal_load(reinterpret_cast<const bf16x8_t*>(p)); }
    __device__ __forceinline__ void store(bf16_t* p) const { __builtin_nontemporal_store(d, reinterpret_cast<bf16x8_t*>(p)); }
    __device__ __forceinline__ float get(int i) const { return (float)d[i]; }
    __device__ __forceinline__ void set(int i, float v) { d[i] = (bf16_t)v; }
};
template <> struct Chunk<float, 4> {
    fvec4_t d;
    __device__ __forceinline__ void load(const float* p) { d = __builtin_nontemporal_load(reinterpret_cast<const fvec4_t*>(p)); }
    __device__ __forceinline__ void store(float* p) const { __builtin_nontemporal_store(d, reinterpret_cast<fvec4_t*>(p)); }
    __device__ __forceinline__ float get(int i) const { return d[i]; }
    __device__ __forceinline__ void set(int i, float v) { d[i] = v; }
};
template <typename T> struct Chunk<T, 1> {
    T d;
    __device__ __forceinline__ void load(const T* p) { d = *p; }
    __device__ __forceinline__ void store(T* p) const { *p = d; }
    __device__ __forceinline__ float get(int) const { return ur_to_float(d); }
    __device__ __forceinline__ void set(int, float v) { d = ur_from_float<T>(v); }
};

// ------------------------------------------------------------------ activations
template <int ACT> __device__ __forceinline__ float gn_act(float p, float slope) {
    if constexpr (ACT == UR_ACT_RELU) return p <= 0.f ? 0.f : p;                       // (NaN stays NaN)
    if constexpr (ACT == UR_ACT_RELU6) return p <= 0.f ? 0.f : (p >= 6.f ? 6.f : p);
    if constexpr (ACT == UR_ACT_LEAKYRELU) return p > 0.f ? p : p * slope;
    if constexpr (ACT == UR_ACT_GELU) return 0.5f * p * (1.f + erff(p * 0.70710678118654752f));
    if constexpr (ACT == UR_ACT_HSWISH) return p <= -3.f ? 0.f : (p >= 3.f ? p : p * (p + 3.f) * (1.f / 6.f));
    if constexpr (ACT == UR_ACT_SILU) return p / (1.f + __expf(-p));
    return p;
}
template <int ACT, typename F> __device__ __forceinline__ float gn_act_grad(F p, float slope) {
    if constexpr (ACT == UR_ACT_RELU) return p <= (F)0 ? 0.f : 1.f;
    if constexpr (ACT == UR_ACT_RELU6) return (p > (F)0 && p < (F)6) ? 1.f : 0.f;
    if constexpr (ACT == UR_ACT_LEAKYRELU) return p > (F)0 ? 1.f : slope;
    if constexpr (ACT == UR_ACT_HSWISH) return p <= (F)-3 ? 0.f : (p < (F)3 ? (2.f * (float)p + 3.f) * (1.f / 6.f) : 1.f);
    const float q = (float)p;
    if constexpr (ACT == UR_ACT_GELU)
        return 0.5f * (1.f + erff(q * 0.70710678118654752f)) + q * 0.3989422804014327f * __expf(-0.5f * q * q);
    if constexpr (ACT == UR_ACT_SILU) {
        const float s = 1.f / (1.f + __expf(-q));
        return s * (1.f + q * (1.f - s));
    }
    return 1.f;
}
// whether p is so close to a kink of the activation's derivative that its fp32 value may be on the wrong side.  Near a kink
// at t: d * A = t - B - r up to the result, and d, A, B, the products and the sums each carry at most 2^-24 relative to
// max(|d * A|, |B|, |r|, |t|): six such errors are 3.6e-7.
template <int ACT> __device__ __forceinline__ bool gn_near_kink(float p, float size) {
    const float tol = 3.6e-7f * size;
    if constexpr (ACT == UR_ACT_RELU || ACT == UR_ACT_LEAKYRELU) return fabsf(p) <= tol;
    if constexpr (ACT == UR_ACT_RELU6) return fabsf(p) <= tol || fabsf(p - 6.f) <= tol + 2.2e-6f;
    if constexpr (ACT == UR_ACT_HSWISH) return fabsf(fabsf(p) - 3.f) <= tol + 1.1e-6f;
    return false;
}

struct GnShape {
    long long hw;
    int c, groups, k;             // channels, groups, channels per group
    int cqb;                      // channel vectors a workgroup covers (a slab)
    int chunks;                   // workgroups over one image's pixels
};

// A workgroup owns pixels [r0, r1) of image blockIdx.y and the channel vectors of slab blockIdx.z; thread (slot, cg) walks
// pixels r0 + slot, r0 + slot + slots, ... of one channel vector.
struct Place {
    int slot, slots, cg, col;
    bool active;
    long long r0, r1;
    template <int V> __device__ __forceinline__ void set(const GnShape& s) {
        slots = NT / s.cqb;
        slot = threadIdx.x / s.cqb;
        cg = threadIdx.x - slot * s.cqb;
        col = (blockIdx.z * s.cqb + cg) * V;
        active = slot < slots && col < s.c;
        r0 = s.hw * blockIdx.x / s.chunks;
        r1 = s.hw * (blockIdx.x + 1) / s.chunks;
    }
};

// ------------------------------------------------------------------ forward: sums of one image's groups
// SPAN: channels of a vector that share a group (a power of two that divides both V and k): V / SPAN pairs of sums per thread
template <typename T, int V, int SPAN>
__global__ __launch_bounds__(NT) void gn_stats_kernel(const T* __restrict__ x, int ld, GnShape s, double* __restrict__ partial) {
    constexpr int NA = V / SPAN;
    __shared__ double red[NA * 2][NT];
    Place at;
    at.set<V>(s);
    double a[NA], q[NA];
#pragma unroll
    for (int i = 0; i < NA; ++i) a[i] = q[i] = 0.0;
    if (at.active) {
        const T* p = x + (size_t)blockIdx.y * s.hw * ld + at.col;
#pragma unroll 4
        for (long long r = at.r0 + at.slot; r < at.r1; r += at.slots) {
            Chunk<T, V> v;
            v.load(p + (size_t)r * ld);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const double f = (double)v.get(i);
                a[i / SPAN] += f;
                q[i / SPAN] = fma(f, f, q[i / SPAN]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < NA; ++i) { red[2 * i][threadIdx.x] = a[i]; red[2 * i + 1][threadIdx.x] = q[i]; }
    __syncthreads();
    for (int n = at.slots; n > 1;) {                     // slots folded in halves, always in the same order
        const int half = (n + 1) >> 1;
        if (at.slot + half < n) {
#pragma unroll
            for (int i = 0; i < 2 * NA; ++i) red[i][threadIdx.x] += red[i][threadIdx.x + half * s.cqb];
        }
        __syncthreads();
        n = half;
    }
    // channels to groups; groups without a channel in this slab get zeros, so that the slabs' rows can simply be added
    double* out = partial + (((size_t)blockIdx.y * s.chunks + blockIdx.x) * gridDim.z + blockIdx.z) * s.groups * 2;
    const int c_lo = blockIdx.z * s.cqb * V, c_hi = min(s.c, c_lo + s.cqb * V);
    for (int g = threadIdx.x; g < s.groups; g += NT) {
        double sa = 0.0, sq = 0.0;
        for (int c = max(c_lo, g * s.k); c < min(c_hi, (g + 1) * s.k); c += SPAN) {
            const int t = (c - c_lo) / V, i = ((c - c_lo) % V) / SPAN;
            sa += red[2 * i][t];
            sq += red[2 * i + 1][t];
        }
        out[2 * g] = sa;
        out[2 * g + 1] = sq;
    }
}

// one wave per (image, group): the partial rows added in a fixed order, {mean, rstd}
__global__ __launch_bounds__(64) void gn_finalize_kernel(const double* __restrict__ partial, int rows, int groups, double count,
                                                         float eps, double* __restrict__ stats) {
    const int g = blockIdx.x, n = blockIdx.y, lane = threadIdx.x;
    const double* p = partial + (size_t)n * rows * groups * 2;
    double a = 0.0, q = 0.0;
    for (int r = lane; r < rows; r += 64) { a += p[((size_t)r * groups + g) * 2]; q += p[((size_t)r * groups + g) * 2 + 1]; }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) { a += __shfl_xor(a, o, 64); q += __shfl_xor(q, o, 64); }
    if (lane == 0) {
        const double mean = a / count;
        double var = q / count - mean * mean;
        if (var < 0.0) var = 0.0;
        stats[((size_t)n * groups + g) * 2] = mean;
        stats[((size_t)n * groups + g) * 2 + 1] = 1.0 / sqrt(var + (double)eps);
    }
}

// the constants of V channels of one image: pre = (x - mean_hi) * a + b
template <int V> struct Affine {
    float m[V], a[V], b[V];
    __device__ __forceinline__ void load(const double* __restrict__ stats, const float* __restrict__ gamma,
                                         const float* __restrict__ beta, int n, int col, const GnShape& s) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const double* st = stats + ((size_t)n * s.groups + (col + i) / s.k) * 2;
            const double ga = gamma ? (double)gamma[col + i] : 1.0, be = beta ? (double)beta[col + i] : 0.0;
            m[i] = (float)st[0];
            a[i] = (float)(st[1] * ga);
            b[i] = (float)(be - (st[0] - (double)m[i]) * (st[1] * ga));
        }
    }
};

template <typename T, int V, int ACT, bool RES>
__global__ __launch_bounds__(NT) void gn_fwd_kernel(const T* __restrict__ x, int ld, const T* __restrict__ res, int res_ld,
                                                    const double* __restrict__ stats, const float* __restrict__ gamma,
                                                    const float* __restrict__ beta, float slope, T* __restrict__ y, int y_ld,
                                                    GnShape s) {
    Place at;
    at.set<V>(s);
    if (!at.active) return;
    const int n = blockIdx.y;
    Affine<V> k;
    k.load(stats, gamma, beta, n, at.col, s);
    const T* xp = x + (size_t)n * s.hw * ld + at.col;
    const T* rp = RES ? res + (size_t)n * s.hw * res_ld + at.col : nullptr;
    T* yp = y + (size_t)n * s.hw * y_ld + at.col;
#pragma unroll 4
    for (long long r = at.r0 + at.slot; r < at.r1; r += at.slots) {
        Chunk<T, V> v, w, o;
        v.load(xp + (size_t)r * ld);
        if constexpr (RES) w.load(rp + (size_t)r * res_ld);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            float p = fmaf(v.get(i) - k.m[i], k.a[i], k.b[i]);
            if constexpr (RES) p += w.get(i);
            o.set(i, gn_act<ACT>(p, slope));
        }
        o.store(yp + (size_t)r * y_ld);
    }
}

// ------------------------------------------------------------------ backward
// act'(pre) of element i of a vector, with the kinks decided in 64 bits
template <int V, int ACT, bool RES>
__device__ __forceinline__ float gn_slope_at(const Affine<V>& k, int i, float xv, float d, float rv, float slope,
                                             const double* __restrict__ stats, const float* __restrict__ gamma,
                                             const float* __restrict__ beta, int n, int col, const GnShape& s) {
    if constexpr (ACT == UR_ACT_NONE) return 1.f;
    float p = fmaf(d, k.a[i], k.b[i]);
    float size = fabsf(k.b[i]);
    if constexpr (RES) { p += rv; size += fabsf(rv); }
    if (gn_near_kink<ACT>(p, size)) {
        const double* st = stats + ((size_t)n * s.groups + (col + i) / s.k) * 2;
        const double ga = gamma ? (double)gamma[col + i] : 1.0, be = beta ? (double)beta[col + i] : 0.0;
        double e = ((double)xv - st[0]) * st[1] * ga + be;
        if constexpr (RES) e += (double)rv;
        return gn_act_grad<ACT, double>(e, slope);
    }
    return gn_act_grad<ACT, float>(p, slope);
}

// per (image, chunk, channel): {sum g, sum g * (x - mean_hi)}
template <typename T, int V, int ACT, bool RES>
__global__ __launch_bounds__(NT) void gn_bwd_reduce_kernel(const T* __restrict__ dy, int dy_ld, const T* __restrict__ x, int ld,
                                                           const T* __restrict__ res, int res_ld, const double* __restrict__ stats,
                                                           const float* __restrict__ gamma, const float* __restrict__ beta,
                                                           float slope, GnShape s, float* __restrict__ partial) {
    __shared__ float red[V * 2][NT];
    Place at;
    at.set<V>(s);
    const int n = blockIdx.y;
    float s1[V], s2[V];
#pragma unroll
    for (int i = 0; i < V; ++i) s1[i] = s2[i] = 0.f;
    if (at.active) {
        Affine<V> k;
        k.load(stats, gamma, beta, n, at.col, s);
        const T* gp = dy + (size_t)n * s.hw * dy_ld + at.col;
        const T* xp = x + (size_t)n * s.hw * ld + at.col;
        const T* rp = RES ? res + (size_t)n * s.hw * res_ld + at.col : nullptr;
#pragma unroll 4
        for (long long r = at.r0 + at.slot; r < at.r1; r += at.slots) {
            Chunk<T, V> u, v, w;
            u.load(gp + (size_t)r * dy_ld);
            v.load(xp + (size_t)r * ld);
            if constexpr (RES) w.load(rp + (size_t)r * res_ld);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float xv = v.get(i), d = xv - k.m[i];
                const float g = u.get(i) * gn_slope_at<V, ACT, RES>(k, i, xv, d, RES ? w.get(i) : 0.f, slope, stats, gamma, beta, n, at.col, s);
                s1[i] += g;
                s2[i] = fmaf(g, d, s2[i]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < V; ++i) { red[2 * i][threadIdx.x] = s1[i]; red[2 * i + 1][threadIdx.x] = s2[i]; }
    __syncthreads();
    for (int m = at.slots; m > 1;) {
        const int half = (m + 1) >> 1;
        if (at.slot + half < m) {
#pragma unroll
            for (int i = 0; i < 2 * V; ++i) red[i][threadIdx.x] += red[i][threadIdx.x + half * s.cqb];
        }
        __syncthreads();
        m = half;
    }
    if (at.slot == 0 && at.active) {
        float* out = partial + (((size_t)n * s.chunks + blockIdx.x) * s.c + at.col) * 2;
#pragma unroll
        for (int i = 0; i < V; ++i) { out[2 * i] = red[2 * i][threadIdx.x]; out[2 * i + 1] = red[2 * i + 1][threadIdx.x]; }
    }
}

// the chunks of one image added per channel in 64 bits: sums[image][channel] = {S1, S2}
__global__ __launch_bounds__(NT) void gn_bwd_sums_kernel(const float* __restrict__ partial, const double* __restrict__ stats,
                                                         GnShape s, double* __restrict__ sums) {
    __shared__ double red[8][32][2];
    const int n = blockIdx.y, ch = threadIdx.x & 31, slot = threadIdx.x >> 5, c = blockIdx.x * 32 + ch;
    double a = 0.0, b = 0.0;
    if (c < s.c) {
        const float2* p = reinterpret_cast<const float2*>(partial) + (size_t)n * s.chunks * s.c + c;
        for (int r = slot; r < s.chunks; r += 8) { const float2 v = p[(size_t)r * s.c]; a += v.x; b += v.y; }
    }
    red[slot][ch][0] = a;
    red[slot][ch][1] = b;
    __syncthreads();
    if (slot || c >= s.c) return;
    for (int j = 1; j < 8; ++j) { a += red[j][ch][0]; b += red[j][ch][1]; }
    const double* st = stats + ((size_t)n * s.groups + c / s.k) * 2;
    sums[((size_t)n * s.c + c) * 2] = a;
    sums[((size_t)n * s.c + c) * 2 + 1] = (b - (st[0] - (double)(float)st[0]) * a) * st[1];        // xhat = (x - mean) * rstd
}

// dx = g * a + d * k2 + k1 with the group's k1, k2 (coef[image][group]); workgroups beyond the images: dgamma, dbeta
__global__ __launch_bounds__(NT) void gn_bwd_coef_kernel(const double* __restrict__ sums, const double* __restrict__ stats,
                                                         const float* __restrict__ gamma, int images, GnShape s,
                                                         float* __restrict__ coef, float* __restrict__ dgamma,
                                                         float* __restrict__ dbeta) {
    if ((int)blockIdx.x < images) {
        const int n = blockIdx.x;
        const double m = (double)s.hw * s.k;
        for (int g = threadIdx.x; g < s.groups; g += NT) {
            double p1 = 0.0, p2 = 0.0;
            for (int c = g * s.k; c < (g + 1) * s.k; ++c) {
                const double ga = gamma ? (double)gamma[c] : 1.0;
                p1 += ga * sums[((size_t)n * s.c + c) * 2];
                p2 += ga * sums[((size_t)n * s.c + c) * 2 + 1];
            }
            p1 /= m;
            p2 /= m;
            const double* st = stats + ((size_t)n * s.groups + g) * 2;
            const double lo = st[0] - (double)(float)st[0];
            coef[((size_t)n * s.groups + g) * 2] = (float)(st[1] * (lo * st[1] * p2 - p1));
            coef[((size_t)n * s.groups + g) * 2 + 1] = (float)(-st[1] * st[1] * p2);
        }
        return;
    }
    const int c = (blockIdx.x - images) * NT + threadIdx.x;
    if (c >= s.c) return;
    double a = 0.0, b = 0.0;
    for (int n = 0; n < images; ++n) { a += sums[((size_t)n * s.c + c) * 2]; b += sums[((size_t)n * s.c + c) * 2 + 1]; }
    if (dbeta) dbeta[c] = (float)a;
    if (dgamma) dgamma[c] = (float)b;
}

template <typename T, int V, int ACT, bool RES>
__global__ __launch_bounds__(NT) void gn_bwd_apply_kernel(const T* __restrict__ dy, int dy_ld, const T* __restrict__ x, int ld,
                                                          const T* __restrict__ res, int res_ld, const double* __restrict__ stats,
                                                          const float* __restrict__ gamma, const float* __restrict__ beta,
                                                          const float* __restrict__ coef, float slope, T* __restrict__ dx,
                                                          T* __restrict__ dres, GnShape s) {
    Place at;
    at.set<V>(s);
    if (!at.active) return;
    const int n = blockIdx.y;
    Affine<V> k;
    k.load(stats, gamma, beta, n, at.col, s);
    float k1[V], k2[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const float* q = coef + ((size_t)n * s.groups + (at.col + i) / s.k) * 2;
        k1[i] = q[0];
        k2[i] = q[1];
    }
    const T* gp = dy + (size_t)n * s.hw * dy_ld + at.col;
    const T* xp = x + (size_t)n * s.hw * ld + at.col;
    const T* rp = RES ? res + (size_t)n * s.hw * res_ld + at.col : nullptr;
    T* op = dx + (size_t)n * s.hw * s.c + at.col;
    T* qp = dres ? dres + (size_t)n * s.hw * s.c + at.col : nullptr;
#pragma unroll 4
    for (long long r = at.r0 + at.slot; r < at.r1; r += at.slots) {
        Chunk<T, V> u, v, w, o, t;
        u.load(gp + (size_t)r * dy_ld);
        v.load(xp + (size_t)r * ld);
        if constexpr (RES) w.load(rp + (size_t)r * res_ld);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float xv = v.get(i), d = xv - k.m[i];
            const float g = u.get(i) * gn_slope_at<V, ACT, RES>(k, i, xv, d, RES ? w.get(i) : 0.f, slope, stats, gamma, beta, n, at.col, s);
            o.set(i, fmaf(g, k.a[i], fmaf(d, k2[i], k1[i])));
            if constexpr (RES) t.set(i, g);
        }
        o.store(op + (size_t)r * s.c);
        if constexpr (RES) { if (qp) t.store(qp + (size_t)r * s.c); }
    }
}

// ------------------------------------------------------------------ host
struct Plan {
    GnShape s;
    int v, zs;                    // vector width, channel slabs
};

Plan make_plan(int dtype, int n, long long hw, int c, int groups, bool vec) {
    Plan p;
    p.v = vec ? (dtype == UR_BF16 ? 8 : 4) : 1;
    const int cq = (c + p.v - 1) / p.v;
    p.s.hw = hw;
    p.s.c = c;
    p.s.groups = groups;
    p.s.k = c / groups;
    p.s.cqb = cq < NT ? cq : NT;
    p.zs = (cq + p.s.cqb - 1) / p.s.cqb;
    const int slots = NT / p.s.cqb;
    // about four workgroups per CU, each with at least four pixels per slot
    long long chunks = 1024 / ((long long)n * p.zs), most = (hw + 4LL * slots - 1) / (4LL * slots);
    if (chunks > most) chunks = most;
    p.s.chunks = chunks < 1 ? 1 : (int)chunks;
    return p;
}

bool aligned(const void* p, int dtype, long long ld) { return p == nullptr || ((((uintptr_t)p) & 15) == 0 && ld % (dtype == UR_BF16 ? 8 : 4) == 0); }

template <typename T, int V>
void launch_stats(const void* x, int ld, const Plan& p, int n, double* partial, hipStream_t st) {
    const dim3 grid(p.s.chunks, n, p.zs);
    if constexpr (V == 8) {
        if (p.s.k % 8 == 0) { hipLaunchKernelGGL((gn_stats_kernel<T, V, 8>), grid, dim3(NT), 0, st, (const T*)x, ld, p.s, partial); return; }
    }
    if constexpr (V >= 4) {
        if (p.s.k % 4 == 0) { hipLaunchKernelGGL((gn_stats_kernel<T, V, 4>), grid, dim3(NT), 0, st, (const T*)x, ld, p.s, partial); return; }
        if (p.s.k % 2 == 0) { hipLaunchKernelGGL((gn_stats_kernel<T, V, 2>), grid, dim3(NT), 0, st, (const T*)x, ld, p.s, partial); return; }
    }
    hipLaunchKernelGGL((gn_stats_kernel<T, V, 1>), grid, dim3(NT), 0, st, (const T*)x, ld, p.s, partial);
}

#define GN_ACT(act, ...)                                                              \
    switch (act) {                                                                    \
    case UR_ACT_NONE: { constexpr int ACT = UR_ACT_NONE; __VA_ARGS__; } break;         \
    case UR_ACT_RELU: { constexpr int ACT = UR_ACT_RELU; __VA_ARGS__; } break;         \
    case UR_ACT_RELU6: { constexpr int ACT = UR_ACT_RELU6; __VA_ARGS__; } break;       \
    case UR_ACT_LEAKYRELU: { constexpr int ACT = UR_ACT_LEAKYRELU; __VA_ARGS__; } break; \
    case UR_ACT_GELU: { constexpr int ACT = UR_ACT_GELU; __VA_ARGS__; } break;         \
    case UR_ACT_HSWISH: { constexpr int ACT = UR_ACT_HSWISH; __VA_ARGS__; } break;     \
    default: { constexpr int ACT = UR_ACT_SILU; __VA_ARGS__; } break;                  \
    }
#define GN_TYPE(dtype, v, ...)                                                                                   \
    do {                                                                                                         \
        if ((dtype) == UR_BF16 && (v) == 8) { typedef bf16_t T; constexpr int V = 8; __VA_ARGS__; }               \
        else if ((dtype) == UR_BF16) { typedef bf16_t T; constexpr int V = 1; __VA_ARGS__; }                      \
        else if ((v) == 4) { typedef float T; constexpr int V = 4; __VA_ARGS__; }                                 \
        else { typedef float T; constexpr int V = 1; __VA_ARGS__; }                                               \
    } while (0)

int check(const char* what, int dtype, int n, long long hw, int c, int groups, int act) {
    UR_REQUIRE(dtype == UR_F32 || dtype == UR_BF16, "%s: bad dtype %d", what, dtype);
    UR_REQUIRE(n > 0 && hw > 0 && c > 0 && groups > 0, "%s: non-positive sizes (n %d, pixels %lld, channels %d, groups %d)", what, n, hw, c, groups);
    UR_REQUIRE(c % groups == 0, "%s: %d channels are not divisible by %d groups", what, c, groups);
    UR_REQUIRE(n <= 65535 && hw <= (1LL << 40) && c <= (1 << 20), "%s: sizes beyond the limits (65535 images, 2^40 pixels, 2^20 channels)", what);
    UR_REQUIRE(act >= UR_ACT_NONE && act <= UR_ACT_SILU, "%s: bad activation %d", what, act);
    return UR_OK;
}

// the larger of what the vector and the element-wise plan need: the caller need not know which one a call takes
size_t fwd_bytes(int dtype, int n, long long hw, int c, int groups) {
    size_t most = 0;
    for (int vec = 0; vec < 2; ++vec) {
        if (vec && c % (dtype == UR_BF16 ? 8 : 4)) continue;
        const Plan p = make_plan(dtype, n, hw, c, groups, vec);
        const size_t b = (size_t)n * p.s.chunks * p.zs * groups * 2 * sizeof(double);
        if (b > most) most = b;
    }
    return most;
}
size_t bwd_bytes(int dtype, int n, long long hw, int c, int groups) {
    size_t most = 0;
    for (int vec = 0; vec < 2; ++vec) {
        if (vec && c % (dtype == UR_BF16 ? 8 : 4)) continue;
        const Plan p = make_plan(dtype, n, hw, c, groups, vec);
        const size_t b = (size_t)n * p.s.chunks * c * 2 * sizeof(float);
        if (b > most) most = b;
    }
    most = (most + 15) / 16 * 16;
    return most + (size_t)n * c * 2 * sizeof(double) + (size_t)n * groups * 2 * sizeof(float);
}

}  // namespace

extern "C" {

size_t ur_gn_fwd_workspace(int dtype, int n, long long hw, int c, int groups) {
    return check("gn_fwd_workspace", dtype, n, hw, c, groups, 0) ? 0 : fwd_bytes(dtype, n, hw, c, groups);
}
size_t ur_gn_bwd_workspace(int dtype, int n, long long hw, int c, int groups) {
    return check("gn_bwd_workspace", dtype, n, hw, c, groups, 0) ? 0 : bwd_bytes(dtype, n, hw, c, groups);
}

int ur_gn_act_fwd(const void* x, int x_ld, const void* residual, int res_ld, const float* gamma, const float* beta, void* y, int y_ld,
                  double* stats, int dtype, int n, long long hw, int c, int groups, float eps, int act, float slope, void* workspace,
                  size_t ws_bytes, ur_stream_t s) {
    if (int e = check("gn_act_fwd", dtype, n, hw, c, groups, act)) return e;
    if (x_ld == 0) x_ld = c;
    if (y_ld == 0) y_ld = c;
    if (res_ld == 0) res_ld = c;
    UR_REQUIRE(x && y && stats && workspace, "gn_act_fwd: null pointer");
    UR_REQUIRE(x_ld >= c && y_ld >= c && res_ld >= c, "gn_act_fwd: a pixel pitch is smaller than the channel count");
    UR_REQUIRE(ws_bytes >= fwd_bytes(dtype, n, hw, c, groups), "gn_act_fwd: workspace too small");
    hipStream_t st = (hipStream_t)s;
    const bool vec = c % (dtype == UR_BF16 ? 8 : 4) == 0 && aligned(x, dtype, x_ld) && aligned(residual, dtype, res_ld) && aligned(y, dtype, y_ld);
    const Plan p = make_plan(dtype, n, hw, c, groups, vec);
    double* partial = (double*)workspace;
    const dim3 grid(p.s.chunks, n, p.zs);
    GN_TYPE(dtype, p.v, (launch_stats<T, V>(x, x_ld, p, n, partial, st)));
    hipLaunchKernelGGL(gn_finalize_kernel, dim3(groups, n), dim3(64), 0, st, partial, p.s.chunks * p.zs, groups, (double)hw * p.s.k, eps, stats);
    GN_TYPE(dtype, p.v, GN_ACT(act, {
        if (residual) hipLaunchKernelGGL((gn_fwd_kernel<T, V, ACT, true>), grid, dim3(NT), 0, st, (const T*)x, x_ld, (const T*)residual, res_ld, stats, gamma, beta, slope, (T*)y, y_ld, p.s);
        else hipLaunchKernelGGL((gn_fwd_kernel<T, V, ACT, false>), grid, dim3(NT), 0, st, (const T*)x, x_ld, (const T*)nullptr, 0, stats, gamma, beta, slope, (T*)y, y_ld, p.s);
    }));
    return ur_check_launch("gn_act_fwd");
}

int ur_gn_act_bwd(const void* dy, int dy_ld, const void* x, int x_ld, const void* residual, int res_ld, const float* gamma,
                  const float* beta, const double* stats, void* dx, void* dres, float* dgamma, float* dbeta, int dtype, int n,
                  long long hw, int c, int groups, int act, float slope, void* workspace, size_t ws_bytes, ur_stream_t s) {
    if (int e = check("gn_act_bwd", dtype, n, hw, c, groups, act)) return e;
    if (x_ld == 0) x_ld = c;
    if (dy_ld == 0) dy_ld = c;
    if (res_ld == 0) res_ld = c;
    UR_REQUIRE(dy && x && stats && workspace, "gn_act_bwd: null pointer");
    UR_REQUIRE(x_ld >= c && dy_ld >= c && res_ld >= c, "gn_act_bwd: a pixel pitch is smaller than the channel count");
    UR_REQUIRE(!dres || residual, "gn_act_bwd: a residual gradient without a residual");
    UR_REQUIRE(!dres || dx, "gn_act_bwd: a residual gradient without dx");
    UR_REQUIRE(ws_bytes >= bwd_bytes(dtype, n, hw, c, groups), "gn_act_bwd: workspace too small");
    hipStream_t st = (hipStream_t)s;
    const bool vec = c % (dtype == UR_BF16 ? 8 : 4) == 0 && aligned(x, dtype, x_ld) && aligned(dy, dtype, dy_ld)
                     && aligned(residual, dtype, res_ld) && aligned(dx, dtype, c) && aligned(dres, dtype, c);
    const Plan p = make_plan(dtype, n, hw, c, groups, vec);
    float* partial = (float*)workspace;
    double* sums = (double*)((char*)workspace + ((size_t)n * p.s.chunks * c * 2 * sizeof(float) + 15) / 16 * 16);
    float* coef = (float*)(sums + (size_t)n * c * 2);
    const dim3 grid(p.s.chunks, n, p.zs);
    GN_TYPE(dtype, p.v, GN_ACT(act, {
        if (residual) hipLaunchKernelGGL((gn_bwd_reduce_kernel<T, V, ACT, true>), grid, dim3(NT), 0, st, (const T*)dy, dy_ld, (const T*)x, x_ld, (const T*)residual, res_ld, stats, gamma, beta, slope, p.s, partial);
        else hipLaunchKernelGGL((gn_bwd_reduce_kernel<T, V, ACT, false>), grid, dim3(NT), 0, st, (const T*)dy, dy_ld, (const T*)x, x_ld, (const T*)nullptr, 0, stats, gamma, beta, slope, p.s, partial);
    }));
    hipLaunchKernelGGL(gn_bwd_sums_kernel, dim3(ur_cdiv(c, 32), n), dim3(NT), 0, st, partial, stats, p.s, sums);
    hipLaunchKernelGGL(gn_bwd_coef_kernel, dim3(n + ur_cdiv(c, NT)), dim3(NT), 0, st, sums, stats, gamma, n, p.s, coef, dgamma, dbeta);
    if (dx) {
        GN_TYPE(dtype, p.v, GN_ACT(act, {
            if (residual) hipLaunchKernelGGL((gn_bwd_apply_kernel<T, V, ACT, true>), grid, dim3(NT), 0, st, (const T*)dy, dy_ld, (const T*)x, x_ld, (const T*)residual, res_ld, stats, gamma, beta, coef, slope, (T*)dx, (T*)dres, p.s);
            else hipLaunchKernelGGL((gn_bwd_apply_kernel<T, V, ACT, false>), grid, dim3(NT), 0, st, (const T*)dy, dy_ld, (const T*)x, x_ld, (const T*)nullptr, 0, stats, gamma, beta, coef, slope, (T*)dx, (T*)nullptr, p.s);
        }));
    }
    return ur_check_launch("gn_act_bwd");
}

}  // extern "C"
