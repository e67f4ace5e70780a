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
// writes dx (and the residual's gradient).  The sums need all of x (dy and x) before the first result, so what does not fit
// the registers of one workgroup is read twice: three passes over a tensor forward and five backward instead of two and three.
// Keeping an image in the registers of many workgroups that exchange their sums was slower (262 and 613 us for the shape
// below).  All passes read past the caches.  A microbenchmark of two such passes gains 4 to 20 % from 32 to 384 MB where the
// first one leaves its data in them; these kernels have not been measured that way.
// Measured, 6x64x512x1024 bf16 (403 MB a tensor): statistics 64 us (6.3 TB/s), forward 135 (6.0), sums of the backward pass 120
// (6.7), gradient 195 (6.2); 64x64x32x32 fp32 in cells: forward 10.7 us, backward 19 + 4.
//
// Arithmetic.  The statistics are plain sums of x and x^2 in 64 bits: fp64 vector arithmetic runs at the fp32 rate here, a
// sum costs four instructions per element against a budget of about thirteen at the HBM rate, and E[x^2] - mean^2 then
// loses 2^-53 (mean / deviation)^2 of the variance: less than an fp32 rounding up to a mean of 2e4 deviations, percents at 1e7,
// where fp32 inputs have no digit left behind the deviation.  The sums of the backward pass are fp32 within a workgroup (a
// thread adds its own pixels one by one: 64 of 6x64x512x1024, some thousands where one workgroup has a large image to itself,
// as with thousands of images) and 64-bit across workgroups.  The passes over the elements run in fp32 with the mean split into its
// fp32 value and the rest: d = x - mean_hi (exact for x near the mean), pre = d * A + B with A = rstd * gamma and
// B = beta - mean_lo * A.  The activations with a kink have a gradient that jumps there, and bf16 inputs take few distinct
// values, so one pre-activation on the wrong side of a kink by a rounding would put thousands of elements on the wrong
// side: within the fp32 error of a kink the backward pass evaluates pre again in 64 bits (rare, one comparison otherwise).
#include "ur_common.h"

#include <type_traits>

namespace {

constexpr int NT = 256;

typedef __attribute__((ext_vector_type(4))) float fvec4_t;
typedef __attribute__((ext_vector_type(4))) unsigned uvec4_t;

// V consecutive channels of one pixel: 16 bytes (8 bf16, 4 fp32) or one element.  bf16 vectors are kept as four words: the
// compiler spreads a bf16 vector that lives across branches over eight registers.  forget(): the compiler no longer knows
// what it computed from the vector, so that it does not keep unpacked copies of data that waits in registers.
template <typename T, int V> struct Chunk;
template <> struct Chunk<bf16_t, 8> {
    uvec4_t d;
    __device__ __forceinline__ void load(const bf16_t* p) { d = __builtin_nontemporal_load(reinterpret_cast<const uvec4_t*>(p)); }
    __device__ __forceinline__ void store(bf16_t* p) const { __builtin_nontemporal_store(d, reinterpret_cast<uvec4_t*>(p)); }
    __device__ __forceinline__ float get(int i) const { return __uint_as_float(i & 1 ? d[i >> 1] & 0xffff0000u : d[i >> 1] << 16); }
    __device__ __forceinline__ void put(const float (&v)[8]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bf16x2_t w = {(bf16_t)v[2 * i], (bf16_t)v[2 * i + 1]};
            d[i] = __builtin_bit_cast(unsigned, w);
        }
    }
    __device__ __forceinline__ void forget() { asm volatile("" : "+v"(d)); }
};
template <> struct Chunk<float, 4> {
    fvec4_t d;
    __device__ __forceinline__ void load(const float* p) { d = __builtin_nontemporal_load(reinterpret_cast<const fvec4_t*>(p)); }
    __device__ __forceinline__ void store(float* p) const { __builtin_nontemporal_store(d, reinterpret_cast<fvec4_t*>(p)); }
    __device__ __forceinline__ float get(int i) const { return d[i]; }
    __device__ __forceinline__ void put(const float (&v)[4]) { d = fvec4_t{v[0], v[1], v[2], v[3]}; }
    __device__ __forceinline__ void forget() { asm volatile("" : "+v"(d)); }
};
template <typename T> struct Chunk<T, 1> {
    T d;
    __device__ __forceinline__ void load(const T* p) { d = *p; }
    __device__ __forceinline__ void store(T* p) const { *p = d; }
    __device__ __forceinline__ float get(int) const { return ur_to_float(d); }
    __device__ __forceinline__ void put(const float (&v)[1]) { d = ur_from_float<T>(v[0]); }
    __device__ __forceinline__ void forget() {}
};

// ------------------------------------------------------------------ activations
// Phi(p) = (1 + erf(p / sqrt 2)) / 2 and e = exp(-p^2 / 2): Abramowitz and Stegun 7.1.26, without the branches of erff (they cost
// registers in unrolled loops) and with the exponential that the derivative needs as well.  The formula is off by at most
// 0.75e-7; evaluated here in fp32, with the hardware's reciprocal and exponential, Phi and the slope were off by at most 2.9e-7
// (a million arguments in [-8, 8])
__device__ __forceinline__ float gn_phi(float p, float& e) {
    const float z = fabsf(p) * 0.70710678118654752f, t = __builtin_amdgcn_rcpf(fmaf(0.3275911f, z, 1.f));
    float s = fmaf(t, 1.061405429f, -1.453152027f);
    s = fmaf(t, s, 1.421413741f);
    s = fmaf(t, s, -0.284496736f);
    s = fmaf(t, s, 0.254829592f);
    e = __expf(-0.5f * p * p);
    const float tail = 0.5f * t * s * e;
    return p < 0.f ? tail : 1.f - tail;
}
template <int ACT> __device__ __forceinline__ float gn_act(float p, float slope) {
    if constexpr (ACT == UR_ACT_RELU) return p <= 0.f ? 0.f : p;                       // (NaN stays NaN)
    if constexpr (ACT == UR_ACT_RELU6) return p <= 0.f ? 0.f : (p >= 6.f ? 6.f : p);
    if constexpr (ACT == UR_ACT_LEAKYRELU) return p > 0.f ? p : p * slope;
    if constexpr (ACT == UR_ACT_GELU) { float e; return p * gn_phi(p, e); }
    if constexpr (ACT == UR_ACT_HSWISH) return p <= -3.f ? 0.f : (p >= 3.f ? p : p * (p + 3.f) * (1.f / 6.f));
    if constexpr (ACT == UR_ACT_SILU) return p * __builtin_amdgcn_rcpf(1.f + __expf(-p));
    return p;
}
// dy * act'(p).  Where the slope is 0 dy is left out, not multiplied: infinite or NaN there, it counts for nothing
template <int ACT, typename F> __device__ __forceinline__ float gn_act_grad(float dy, F p, float slope) {
    if constexpr (ACT == UR_ACT_RELU) return p <= (F)0 ? 0.f : dy;
    if constexpr (ACT == UR_ACT_RELU6) return (p > (F)0 && p < (F)6) ? dy : 0.f;
    if constexpr (ACT == UR_ACT_LEAKYRELU) return p > (F)0 ? dy : dy * slope;
    if constexpr (ACT == UR_ACT_HSWISH) return p <= (F)-3 ? 0.f : (p < (F)3 ? dy * ((2.f * (float)p + 3.f) * (1.f / 6.f)) : dy);
    const float q = (float)p;
    if constexpr (ACT == UR_ACT_GELU) { float e; const float c = gn_phi(q, e); return dy * fmaf(q * 0.3989422804014327f, e, c); }
    if constexpr (ACT == UR_ACT_SILU) {
        const float s = __builtin_amdgcn_rcpf(1.f + __expf(-q));
        return dy * (s * (1.f + q * (1.f - s)));
    }
    return dy;
}
// whether p is so close to a kink of the activation's derivative that its fp32 value may be on the wrong side.  Near a kink
// at t: d * A = t - B - r up to the result, and d, A, B, the products and the sums each carry at most 2^-24 relative to
// max(|d * A|, |B|, |r|, |t|): six such errors are 3.6e-7.  At zero strictly: where B = r = 0 nothing is added to d * A, whose
// sign is certain (short of underflow).  That is every element with a zero weight and bias (the usual start of a block's last norm) whose residual is
// 0, as half of them are behind a ReLU: settled one by one they made the backward pass of 6x64x512x1024 bf16 3393 us instead
// of 586.
template <int ACT> __device__ __forceinline__ bool gn_near_kink(float p, float size) {
    const float tol = 3.6e-7f * size;
    if constexpr (ACT == UR_ACT_RELU || ACT == UR_ACT_LEAKYRELU) return fabsf(p) < tol;
    if constexpr (ACT == UR_ACT_RELU6) return fabsf(p) < tol || fabsf(p - 6.f) <= tol + 2.2e-6f;
    if constexpr (ACT == UR_ACT_HSWISH) return fabsf(fabsf(p) - 3.f) <= tol + 1.1e-6f;
    return false;
}

// a / b for 0 <= a < 2^20: (a + 1/2) / b is at least 1 / (2 b) from an integer, its relative error at most 2^-21
__device__ __forceinline__ int small_div(int a, int b) { return (int)(((float)a + 0.5f) * __builtin_amdgcn_rcpf((float)b)); }

struct GnShape {
    long long hw;
    int c, groups, k;             // channels, groups, channels per group
    int cqb;                      // channel vectors a workgroup covers (a slab)
    int chunks;                   // workgroups over one image's pixels
};

// A workgroup owns pixels of image blockIdx.y and the channel vectors of slab blockIdx.z; thread (slot, cg) one channel
// vector.  The workgroups of an image sweep it together: trip t of workgroup b covers the U * slots pixels from
// (t * chunks + b) * U * slots on, so that the chip reads one moving window per image.
struct Place {
    int slot, slots, cg, col;
    bool active;
    template <int V> __device__ __forceinline__ void set(const GnShape& s) {
        slots = small_div(NT, s.cqb);
        slot = small_div(threadIdx.x, s.cqb);
        cg = threadIdx.x - slot * s.cqb;
        col = (blockIdx.z * s.cqb + cg) * V;
        active = slot < slots && col < s.c;
    }
    // load(h, r) and full(h, r): U pixels r, r + slots, ... into and out of buffer h; once(): what full and one need besides,
    // while the first loads are on their way; one(r): a single pixel (the end of the image).  BUFFERS 2: a trip is loaded
    // while the one before it is worked on.
    template <int U, int BUFFERS, typename Load, typename Once, typename Full, typename One>
    __device__ __forceinline__ void walk(const GnShape& s, const Load& load, const Once& once, const Full& full, const One& one) const {
        constexpr std::integral_constant<int, 0> first;
        constexpr std::integral_constant<int, BUFFERS - 1> second;
        const long long step = (long long)s.chunks * U * slots;
        long long r = (long long)blockIdx.x * U * slots + slot;
        const auto whole = [&](long long at) { return at + (U - 1) * slots < s.hw; };
        bool go = whole(r);
        if (go) load(first, r);
        __builtin_amdgcn_sched_barrier(0);
        once();
        const auto trip = [&](auto now, auto next) {
            go = whole(r + step);
            if (BUFFERS == 2 && go) load(next, r + step);
            __builtin_amdgcn_sched_barrier(0);
            full(now, r);
            r += step;
            if (BUFFERS == 1 && go) load(next, r);
        };
        while (go) {
            trip(first, second);
            if (BUFFERS == 2 && go) trip(second, first);
        }
        for (; r < s.hw; r += slots) one(r);
    }
};

// Rows of sums in the LDS are padded by eight entries: threads that read one slot of several rows then meet different banks.
constexpr int PAD = 8;

// adds the rows of red[values][slots * cqb] over the slots, always in the same order; result at slot 0.  Every sum of one row
// and channel vector is made by up to 16 threads, a strided part of the slots each, and one of them adds their results: two
// waits whatever the number of slots, and reads that do not depend on each other.
template <typename F, int N>
__device__ __forceinline__ void fold_slots(F (*red)[N], int values, int slots, int cqb) {
    constexpr int THREADS = N - PAD;
    __syncthreads();
    const int outs = values * cqb, parts = min(slots, max(1, min(16, small_div(THREADS, outs))));
    for (int left = slots, way = parts;; left = way, way = 1) {            // (slots to parts, parts to one)
        for (int o = threadIdx.x; o < outs * way; o += THREADS) {
            const int part = small_div(o, outs), q = o - part * outs, i = small_div(q, cqb), cg = q - i * cqb;
            F s = red[i][part * cqb + cg];                                   // slots part, part + way, ...: no other thread's
#pragma unroll 4
            for (int r = part + way; r < left; r += way) s += red[i][r * cqb + cg];
            red[i][part * cqb + cg] = s;
        }
        __syncthreads();
        if (way == 1) break;
    }
}

__device__ __forceinline__ void mean_rstd(double a, double q, double count, float eps, double& mean, double& rstd) {
    mean = a / count;
    double var = q / count - mean * mean;
    if (var < 0.0) var = 0.0;                              // (a NaN stays one)
    rstd = 1.0 / sqrt(var + (double)eps);
}

// the group of a channel and of those after it, with one division
struct GroupOf {
    int g, left, k;
    __device__ __forceinline__ GroupOf(int c, int k_) : g(small_div(c, k_)), left((g + 1) * k_ - c), k(k_) {}
    __device__ __forceinline__ void next() { if (--left == 0) { ++g; left = k; } }
};

// the constants of V channels of one image: pre = (x - mean_hi) * a + b.  They are fetched first, so that they arrive while
// the loads of the data are on their way
// (a module without parameters reads zeros and adds one: a branch around each load would wait for it, sixteen times in turn)
__device__ const float gn_zeros[8] = {};
template <int V> struct AffineIn {
    float ga[V], be[V], one;
    double mean[V], rstd[V];
    __device__ __forceinline__ void params(const float* __restrict__ gamma, const float* __restrict__ beta, int col) {
        const float *g = gamma ? gamma + col : gn_zeros, *b = beta ? beta + col : gn_zeros;
        one = gamma ? 0.f : 1.f;
#pragma unroll
        for (int i = 0; i < V; ++i) { ga[i] = g[i]; be[i] = b[i]; }
    }
    __device__ __forceinline__ double weight(int i) const { return (double)(ga[i] + one); }
    // stats: {mean, rstd} of the groups from g0 on
    __device__ __forceinline__ void groups(const double* stats, int g0, int col, int k) {
        GroupOf at(col, k);
#pragma unroll
        for (int i = 0; i < V; ++i, at.next()) { mean[i] = stats[(at.g - g0) * 2]; rstd[i] = stats[(at.g - g0) * 2 + 1]; }
    }
};
template <int V> struct Affine {
    float m[V], a[V], b[V];
    __device__ __forceinline__ void set(const AffineIn<V>& in) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const double s = in.rstd[i] * in.weight(i);
            m[i] = (float)in.mean[i];
            a[i] = (float)s;
            b[i] = (float)((double)in.be[i] - (in.mean[i] - (double)m[i]) * s);
        }
    }
};

template <typename T, int V, int ACT, bool RES>
__device__ __forceinline__ Chunk<T, V> fwd_vector(const Affine<V>& k, const Chunk<T, V>& v, const Chunk<T, V>& w, float slope) {
    float z[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        float p = fmaf(v.get(i) - k.m[i], k.a[i], k.b[i]);
        if constexpr (RES) p += w.get(i);
        z[i] = gn_act<ACT>(p, slope);
    }
    Chunk<T, V> o;
    o.put(z);
    return o;
}

// g = dy * act'(pre) of a vector, d = x - mean_hi; returns whether an element lies near a kink.  Then the caller corrects
// the vector with settle().
template <typename T, int V, int ACT, bool RES>
__device__ __forceinline__ bool bwd_vector(const Affine<V>& k, const Chunk<T, V>& u, const Chunk<T, V>& v, const Chunk<T, V>& w, float slope,
                                           float (&g)[V], float (&d)[V]) {
    bool near = false;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        d[i] = v.get(i) - k.m[i];
        float p = fmaf(d[i], k.a[i], k.b[i]), size = fabsf(k.b[i]);
        if constexpr (RES) { p += w.get(i); size += fabsf(w.get(i)); }
        near |= gn_near_kink<ACT>(p, size);
        g[i] = gn_act_grad<ACT, float>(u.get(i), p, slope);
    }
    return near;
}
template <typename T, int V, int ACT, bool RES>
__device__ __forceinline__ void settle(const T* dy, const T* x, const T* res, float slope, const double* stats, int g0,
                                       const float* __restrict__ gamma, const float* __restrict__ beta, int col, int per, float (&g)[V]) {
#pragma unroll 1
    for (int i = 0; i < V; ++i) {                          // (read again, one by one: few registers)
        const double* st = stats + ((col + i) / per - g0) * 2;
        double e = ((double)ur_to_float(x[i]) - st[0]) * st[1] * (gamma ? (double)gamma[col + i] : 1.0) + (beta ? (double)beta[col + i] : 0.0);
        if constexpr (RES) e += (double)ur_to_float(res[i]);
        const float exact = gn_act_grad<ACT, double>(ur_to_float(dy[i]), e, slope);
#pragma unroll
        for (int j = 0; j < V; ++j) g[j] = j == i ? exact : g[j];
    }
}

// a vector near a kink, from memory again, outside of the unrolled loops (their code would be several times as long)
template <typename T, int V, int ACT, bool RES>
__device__ __forceinline__ void again(const Affine<V>& k, long long r, const T* dy, int dy_ld, const T* x, int ld, const T* res, int res_ld, float slope,
                                      const double* stats, int g0, const float* __restrict__ gamma, const float* __restrict__ beta, int col, int per,
                                      float (&g)[V], float (&d)[V]) {
    Chunk<T, V> u, v, w;
    u.load(dy + (size_t)r * dy_ld);
    v.load(x + (size_t)r * ld);
    if constexpr (RES) w.load(res + (size_t)r * res_ld);
    if (bwd_vector<T, V, ACT, RES>(k, u, v, w, slope, g, d))
        settle<T, V, ACT, RES>(dy + (size_t)r * dy_ld, x + (size_t)r * ld, RES ? res + (size_t)r * res_ld : nullptr, slope, stats, g0, gamma, beta, col, per, g);
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

// ================================================================== one workgroup per cell
// Small and middle sizes: a cell is one image x a slab of channels that holds whole groups, and one workgroup keeps it in
// registers: one launch, one read, no sums through memory.
constexpr int CT = 512;                                    // threads per cell

struct Cell {
    int hw, c, groups, k, slab, slabs;                     // slab: channels per cell (the last one of an image may have fewer)
};

struct CellPlace {
    int n, c0, sc, cqs, slot, slots, cg, col;
    bool active;                                           // (the others have a channel vector, too, and load without a branch: a
                                                           // branch around a load waits for it and for all before it)
    template <int V> __device__ __forceinline__ void set(const Cell& s) {
        n = blockIdx.x / s.slabs;
        c0 = (blockIdx.x - n * s.slabs) * s.slab;
        sc = min(s.slab, s.c - c0);
        cqs = sc / V;
        slots = small_div(CT, cqs);
        slot = small_div(threadIdx.x, cqs);
        cg = threadIdx.x - slot * cqs;
        col = c0 + cg * V;
        active = slot < slots;
    }
};

template <typename T, int V, int K, bool RES>
__global__ __launch_bounds__(CT) void gn_fwd_cell_kernel(const T* __restrict__ x, int ld, const T* __restrict__ res, int res_ld,
                                                         const float* __restrict__ gamma, const float* __restrict__ beta, float eps, int act,
                                                         float slope, T* __restrict__ y, int y_ld, double* __restrict__ stats, Cell s) {
    extern __shared__ double cell_lds[];
    CellPlace at;
    at.set<V>(s);
    const size_t row0 = (size_t)at.n * s.hw;
    AffineIn<V> in;
    in.params(gamma, beta, at.col);
    __builtin_amdgcn_sched_barrier(0);
    Chunk<T, V> v[K], w[RES ? K : 1];
    const T* xp = x + row0 * ld + at.col;
    const T* rp = RES ? res + row0 * res_ld + at.col : nullptr;
#pragma unroll
    for (int j = 0; j < K; ++j) v[j].load(xp + (size_t)min(at.slot + j * at.slots, s.hw - 1) * ld);
    if constexpr (RES) {
#pragma unroll
        for (int j = 0; j < K; ++j) w[j].load(rp + (size_t)min(at.slot + j * at.slots, s.hw - 1) * res_ld);
    }
    double a[V], q[V];
#pragma unroll
    for (int i = 0; i < V; ++i) a[i] = q[i] = 0.0;
#pragma unroll
    for (int j = 0; j < K; ++j) {
        if (at.active && at.slot + j * at.slots < s.hw) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const double f = (double)v[j].get(i);
                a[i] += f;
                q[i] = fma(f, f, q[i]);
            }
        }
    }
    // channels of the vector that share a group are added first: span of them (1, 2, 4 or 8)
    int span = 1, shift = 0;
#pragma unroll
    for (int w = 1; w < V; w *= 2) {
        if (s.k % (2 * w) == 0) {
#pragma unroll
            for (int i = 0; i < V; i += 2 * w) { a[i] += a[i + w]; q[i] += q[i + w]; }
            span = 2 * w;
            ++shift;
        }
    }
    // sums and squares folded together, or one after the other where eight of each per thread would not fit the LDS at once
    double(*red)[CT + PAD] = reinterpret_cast<double(*)[CT + PAD]>(cell_lds);
    const int na = V / span, rows = na > 4 ? na : 2 * na;
    double* mine = cell_lds + rows * (CT + PAD);
    const int gs = at.sc / s.k, g0 = at.c0 / s.k, g = threadIdx.x;         // a slab begins with a group and has at most CT
    const auto group_sum = [&](int first) {
        double t = 0.0;
        if (g < gs) {
#pragma unroll 4
            for (int ch = g * s.k; ch < (g + 1) * s.k; ch += span) t += red[first + (ch % V >> shift)][ch / V];
        }
        return t;
    };
    double sa, sq;
#pragma unroll
    for (int i = 0; i < V; ++i)
        if (i % span == 0) {
            red[i / span][threadIdx.x] = a[i];
            if (rows > na) red[na + i / span][threadIdx.x] = q[i];
        }
    fold_slots(red, rows, at.slots, at.cqs);
    sa = group_sum(0);
    if (rows > na) sq = group_sum(na);
    else {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i % span == 0) red[i / span][threadIdx.x] = q[i];
        fold_slots(red, rows, at.slots, at.cqs);
        sq = group_sum(0);
    }
    if (g < gs) {
        double mean, rstd;
        mean_rstd(sa, sq, (double)s.hw * s.k, eps, mean, rstd);
        mine[2 * g] = mean;
        mine[2 * g + 1] = rstd;
        double* st = stats + ((size_t)at.n * s.groups + g0 + g) * 2;
        st[0] = mean;
        st[1] = rstd;
    }
    __syncthreads();
    if (!at.active) return;
    Affine<V> k;
    in.groups(mine, g0, at.col, s.k);
    k.set(in);
    T* yp = y + row0 * y_ld + at.col;
    GN_ACT(act, {
_Pragma("unroll")
        for (int j = 0; j < K; ++j) {
            const int r = at.slot + j * at.slots;
            if (r < s.hw) {
                v[j].forget();
                fwd_vector<T, V, ACT, RES>(k, v[j], w[RES ? j : 0], slope).store(yp + (size_t)r * y_ld);
            }
        }
    });
}

// sums: {S1, S2} of every image and channel; one image: dgamma and dbeta themselves
template <typename T, int V, int K, bool RES>
__global__ __launch_bounds__(CT) void gn_bwd_cell_kernel(const T* __restrict__ dy, int dy_ld, const T* __restrict__ x, int ld,
                                                         const T* __restrict__ res, int res_ld, const double* __restrict__ stats,
                                                         const float* __restrict__ gamma, const float* __restrict__ beta, int act, float slope,
                                                         T* __restrict__ dx, T* __restrict__ dres, double* __restrict__ sums,
                                                         float* __restrict__ dgamma, float* __restrict__ dbeta, Cell s) {
    extern __shared__ double cell_lds[];
    float(*red)[CT + PAD] = reinterpret_cast<float(*)[CT + PAD]>(cell_lds);   // [2 V][CT + PAD] floats, [sc][2] doubles, [gs][2] floats
    CellPlace at;
    at.set<V>(s);
    const size_t row0 = (size_t)at.n * s.hw;
    const int g0 = at.c0 / s.k, gs = at.sc / s.k;
    double* ch_sums = reinterpret_cast<double*>(red + 2 * V);
    float* coef = reinterpret_cast<float*>(ch_sums + 2 * at.sc);
    const double* st0 = stats + ((size_t)at.n * s.groups + g0) * 2;
    Chunk<T, V> u[K], v[K], w[RES ? K : 1];
    const T* gp = dy + row0 * dy_ld + at.col;
    const T* xp = x + row0 * ld + at.col;
    const T* rp = RES ? res + row0 * res_ld + at.col : nullptr;
    AffineIn<V> in;
    in.params(gamma, beta, at.col);
    in.groups(st0, g0, at.col, s.k);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < K; ++j) {
        const int r = min(at.slot + j * at.slots, s.hw - 1);
        u[j].load(gp + (size_t)r * dy_ld);
        v[j].load(xp + (size_t)r * ld);
        if constexpr (RES) w[j].load(rp + (size_t)r * res_ld);
    }
    Affine<V> k;
    k.set(in);
    float s1[V], s2[V], g[V], d[V];
#pragma unroll
    for (int i = 0; i < V; ++i) s1[i] = s2[i] = 0.f;
    if (at.active) {
        GN_ACT(act, {
            unsigned near = 0;
_Pragma("unroll")
            for (int j = 0; j < K; ++j) {
                const int r = at.slot + j * at.slots;
                if (r < s.hw) {
                    const bool skip = bwd_vector<T, V, ACT, RES>(k, u[j], v[j], w[RES ? j : 0], slope, g, d);
                    near |= (unsigned)skip << j;
_Pragma("unroll")
                    for (int i = 0; i < V; ++i) { g[i] = skip ? 0.f : g[i]; s1[i] += g[i]; s2[i] = fmaf(g[i], d[i], s2[i]); }
                }
            }
            for (; near; near &= near - 1) {               // rare
                again<T, V, ACT, RES>(k, at.slot + __builtin_ctz(near) * at.slots, gp, dy_ld, xp, ld, rp, res_ld, slope, st0, g0, gamma, beta, at.col, s.k, g, d);
_Pragma("unroll")
                for (int i = 0; i < V; ++i) { s1[i] += g[i]; s2[i] = fmaf(g[i], d[i], s2[i]); }
            }
        });
    }
#pragma unroll
    for (int i = 0; i < V; ++i) { red[2 * i][threadIdx.x] = s1[i]; red[2 * i + 1][threadIdx.x] = s2[i]; }
    fold_slots(red, 2 * V, at.slots, at.cqs);
    if (at.slot == 0) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const double* st = st0 + ((at.col + i) / s.k - g0) * 2;
            const double a = red[2 * i][threadIdx.x], b = red[2 * i + 1][threadIdx.x];
            const double q = (b - (st[0] - (double)(float)st[0]) * a) * st[1];         // xhat = (x - mean) * rstd
            const int c = at.col + i;
            const double ga = in.weight(i);
            ch_sums[2 * (c - at.c0)] = ga * a;
            ch_sums[2 * (c - at.c0) + 1] = ga * q;
            if (sums) {
                sums[((size_t)at.n * s.c + c) * 2] = a;
                sums[((size_t)at.n * s.c + c) * 2 + 1] = q;
            } else {
                if (dbeta) dbeta[c] = (float)a;
                if (dgamma) dgamma[c] = (float)q;
            }
        }
    }
    if (!dx) return;
    __syncthreads();
    const double m = (double)s.hw * s.k;
    for (int h = threadIdx.x; h < gs; h += CT) {
        double p1 = 0.0, p2 = 0.0;
#pragma unroll 4
        for (int c = h * s.k; c < (h + 1) * s.k; ++c) { p1 += ch_sums[2 * c]; p2 += ch_sums[2 * c + 1]; }
        const double mean = st0[2 * h], rstd = st0[2 * h + 1], lo = mean - (double)(float)mean;
        coef[2 * h] = (float)(rstd * (lo * rstd * p2 - p1) / m);
        coef[2 * h + 1] = (float)(-rstd * rstd * p2 / m);
    }
    __syncthreads();
    if (!at.active) return;
    float k1[V], k2[V];
    GroupOf of(at.col, s.k);
#pragma unroll
    for (int i = 0; i < V; ++i, of.next()) { k1[i] = coef[2 * (of.g - g0)]; k2[i] = coef[2 * (of.g - g0) + 1]; }
    T* op = dx + row0 * s.c + at.col;
    T* qp = RES && dres ? dres + row0 * s.c + at.col : nullptr;
    const auto write = [&](int r) {
        Chunk<T, V> o, t;
#pragma unroll
        for (int i = 0; i < V; ++i) d[i] = fmaf(g[i], k.a[i], fmaf(d[i], k2[i], k1[i]));
        o.put(d);
        o.store(op + (size_t)r * s.c);
        if constexpr (RES) { if (qp) { t.put(g); t.store(qp + (size_t)r * s.c); } }
    };
    GN_ACT(act, {
        unsigned near = 0;
_Pragma("unroll")
        for (int j = 0; j < K; ++j) {
            const int r = at.slot + j * at.slots;
            if (r < s.hw) {
                u[j].forget();
                v[j].forget();
                near |= (unsigned)bwd_vector<T, V, ACT, RES>(k, u[j], v[j], w[RES ? j : 0], slope, g, d) << j;
                write(r);
            }
        }
        for (; near; near &= near - 1) {                   // rare: written again
            const int r = at.slot + __builtin_ctz(near) * at.slots;
            again<T, V, ACT, RES>(k, r, gp, dy_ld, xp, ld, rp, res_ld, slope, st0, g0, gamma, beta, at.col, s.k, g, d);
            write(r);
        }
    });
}

// dgamma, dbeta: {S1, S2} added over the images, 32 channels x 8 image slots per workgroup
__device__ __forceinline__ void sum_images(const double* __restrict__ sums, int images, int c_all, int block, float* __restrict__ dgamma,
                                           float* __restrict__ dbeta) {
    __shared__ double red[8][32][2];
    const int ch = threadIdx.x & 31, slot = threadIdx.x >> 5, c = block * 32 + ch;
    double a = 0.0, b = 0.0;
    if (c < c_all && slot < 8) {
#pragma unroll 4
        for (int n = slot; n < images; n += 8) { const double* p = sums + ((size_t)n * c_all + c) * 2; a += p[0]; b += p[1]; }
    }
    if (slot < 8) { red[slot][ch][0] = a; red[slot][ch][1] = b; }
    __syncthreads();
    if (slot == 0 && c < c_all) {
        for (int j = 1; j < 8; ++j) { a += red[j][ch][0]; b += red[j][ch][1]; }
        if (dbeta) dbeta[c] = (float)a;
        if (dgamma) dgamma[c] = (float)b;
    }
    __syncthreads();
}
__global__ __launch_bounds__(NT) void gn_params_kernel(const double* __restrict__ sums, int images, int c_all, float* __restrict__ dgamma,
                                                       float* __restrict__ dbeta) {
    sum_images(sums, images, c_all, blockIdx.x, dgamma, dbeta);
}

// ================================================================== streaming passes
// Large sizes: two passes over memory with the sums of all workgroups between them.
// pixels a thread loads at a time; in the statistics.  The last backward pass loads a trip ahead (6x64x512x1024 bf16 204 -> 198
// us, 6x512x64x128 with residual 57 -> 54); the forward pass gains nothing by it (139 and 138), and the sums of the first
// backward pass leave too few registers (125 -> 135).
constexpr int UNR = 4, SUNR = 8;

// SPAN: channels of a vector that share a group (a power of two that divides both V and k): V / SPAN pairs of sums per thread
template <typename T, int V, int SPAN>
__global__ __launch_bounds__(NT) void gn_stats_kernel(const T* __restrict__ x, int ld, GnShape s, double* __restrict__ partial) {
    constexpr int NA = V / SPAN;
    __shared__ double red[NA * 2][NT + PAD];
    Place at;
    at.set<V>(s);
    double a[NA], q[NA];
#pragma unroll
    for (int i = 0; i < NA; ++i) a[i] = q[i] = 0.0;
    if (at.active) {
        const T* p = x + (size_t)blockIdx.y * s.hw * ld + at.col;
        const auto add = [&](const Chunk<T, V>& v) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const double f = (double)v.get(i);
                a[i / SPAN] += f;
                q[i / SPAN] = fma(f, f, q[i / SPAN]);
            }
        };
        Chunk<T, V> v[SUNR];
        at.walk<SUNR, 1>(s, [&](auto, long long r) {
#pragma unroll
            for (int j = 0; j < SUNR; ++j) v[j].load(p + (size_t)(r + j * at.slots) * ld);
        }, [] {}, [&](auto, long long) {
#pragma unroll
            for (int j = 0; j < SUNR; ++j) add(v[j]);
        }, [&](long long r) { Chunk<T, V> e; e.load(p + (size_t)r * ld); add(e); });
    }
#pragma unroll
    for (int i = 0; i < NA; ++i) { red[2 * i][threadIdx.x] = a[i]; red[2 * i + 1][threadIdx.x] = q[i]; }
    fold_slots(red, 2 * NA, at.slots, s.cqb);
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
    for (int r = lane; r < rows; r += 8 * 64) {              // eight loads at a time, the last ones of them possibly idle
        double v[8][2];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const double* t = p + ((size_t)min(r + 64 * j, rows - 1) * groups + g) * 2;
            v[j][0] = t[0];
            v[j][1] = t[1];
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) { const bool in = r + 64 * j < rows; a += in ? v[j][0] : 0.0; q += in ? v[j][1] : 0.0; }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) { a += __shfl_xor(a, o, 64); q += __shfl_xor(q, o, 64); }
    if (lane == 0) {
        double mean, rstd;
        mean_rstd(a, q, count, eps, mean, rstd);
        stats[((size_t)n * groups + g) * 2] = mean;
        stats[((size_t)n * groups + g) * 2 + 1] = rstd;
    }
}

template <typename T, int V, int ACT, bool RES>
__global__ __launch_bounds__(NT) void gn_fwd_kernel(const T* __restrict__ x, int ld, const T* __restrict__ res, int res_ld,
                                                    const double* __restrict__ stats, const float* __restrict__ gamma,
                                                    const float* __restrict__ beta, float slope, T* __restrict__ y, int y_ld,
                                                    GnShape s) {
    Place at;
    at.set<V>(s);
    if (!at.active) return;
    const int n = blockIdx.y;
    AffineIn<V> in;
    in.params(gamma, beta, at.col);
    in.groups(stats + (size_t)n * s.groups * 2, 0, at.col, s.k);
    __builtin_amdgcn_sched_barrier(0);
    Affine<V> k;
    const T* xp = x + (size_t)n * s.hw * ld + at.col;
    const T* rp = RES ? res + (size_t)n * s.hw * res_ld + at.col : nullptr;
    T* yp = y + (size_t)n * s.hw * y_ld + at.col;
    Chunk<T, V> v[UNR], w[UNR];
    at.walk<UNR, 1>(s, [&](auto, long long r) {
#pragma unroll
        for (int j = 0; j < UNR; ++j) {
            v[j].load(xp + (size_t)(r + j * at.slots) * ld);
            if constexpr (RES) w[j].load(rp + (size_t)(r + j * at.slots) * res_ld);
        }
    }, [&] { k.set(in); }, [&](auto, long long r) {
#pragma unroll
        for (int j = 0; j < UNR; ++j) fwd_vector<T, V, ACT, RES>(k, v[j], w[j], slope).store(yp + (size_t)(r + j * at.slots) * y_ld);
    }, [&](long long r) {
        Chunk<T, V> v, w;
        v.load(xp + (size_t)r * ld);
        if constexpr (RES) w.load(rp + (size_t)r * res_ld);
        fwd_vector<T, V, ACT, RES>(k, v, w, slope).store(yp + (size_t)r * y_ld);
    });
}

// per (image, chunk, channel): {sum g, sum g * (x - mean_hi)}
template <typename T, int V, int ACT, bool RES>
__global__ __launch_bounds__(NT) void gn_bwd_reduce_kernel(const T* __restrict__ dy, int dy_ld, const T* __restrict__ x, int ld,
                                                           const T* __restrict__ res, int res_ld, const double* __restrict__ stats,
                                                           const float* __restrict__ gamma, const float* __restrict__ beta,
                                                           float slope, GnShape s, float* __restrict__ partial) {
    __shared__ float red[V * 2][NT + PAD];
    Place at;
    at.set<V>(s);
    const int n = blockIdx.y;
    const double* st0 = stats + (size_t)n * s.groups * 2;
    float s1[V], s2[V];
#pragma unroll
    for (int i = 0; i < V; ++i) s1[i] = s2[i] = 0.f;
    if (at.active) {
        AffineIn<V> in;
        in.params(gamma, beta, at.col);
        in.groups(st0, 0, at.col, s.k);
        __builtin_amdgcn_sched_barrier(0);
        Affine<V> k;
        const T* gp = dy + (size_t)n * s.hw * dy_ld + at.col;
        const T* xp = x + (size_t)n * s.hw * ld + at.col;
        const T* rp = RES ? res + (size_t)n * s.hw * res_ld + at.col : nullptr;
        const auto add = [&](const float (&g)[V], const float (&d)[V]) {
#pragma unroll
            for (int i = 0; i < V; ++i) { s1[i] += g[i]; s2[i] = fmaf(g[i], d[i], s2[i]); }
        };
        const auto one = [&](long long r) {
            float g[V], d[V];
            again<T, V, ACT, RES>(k, r, gp, dy_ld, xp, ld, rp, res_ld, slope, st0, 0, gamma, beta, at.col, s.k, g, d);
            add(g, d);
        };
        Chunk<T, V> u[UNR], v[UNR], w[UNR];
        at.walk<UNR, 1>(s, [&](auto, long long r) {
#pragma unroll
            for (int j = 0; j < UNR; ++j) {
                u[j].load(gp + (size_t)(r + j * at.slots) * dy_ld);
                v[j].load(xp + (size_t)(r + j * at.slots) * ld);
                if constexpr (RES) w[j].load(rp + (size_t)(r + j * at.slots) * res_ld);
            }
        }, [&] { k.set(in); }, [&](auto, long long r) {
            unsigned near = 0;
#pragma unroll
            for (int j = 0; j < UNR; ++j) {
                float g[V], d[V];
                u[j].forget();
                v[j].forget();
                const bool skip = bwd_vector<T, V, ACT, RES>(k, u[j], v[j], w[j], slope, g, d);
                near |= (unsigned)skip << j;
#pragma unroll
                for (int i = 0; i < V; ++i) g[i] = skip ? 0.f : g[i];
                add(g, d);
#pragma unroll
                for (int i = 0; i < V; ++i) asm volatile("" : "+v"(s1[i]), "+v"(s2[i]));
                __builtin_amdgcn_sched_barrier(0);         // vector by vector: interleaved they would cost registers and so waves
            }
            for (; near; near &= near - 1) one(r + __builtin_ctz(near) * at.slots);        // rare
        }, one);
    }
#pragma unroll
    for (int i = 0; i < V; ++i) { red[2 * i][threadIdx.x] = s1[i]; red[2 * i + 1][threadIdx.x] = s2[i]; }
    fold_slots(red, 2 * V, at.slots, s.cqb);
    if (at.slot == 0 && at.active) {
        float* out = partial + (((size_t)n * s.chunks + blockIdx.x) * s.c + at.col) * 2;
#pragma unroll
        for (int i = 0; i < V; ++i) { out[2 * i] = red[2 * i][threadIdx.x]; out[2 * i + 1] = red[2 * i + 1][threadIdx.x]; }
    }
}

// The sums of one image's channels and the constants of its groups: a workgroup owns `bundle` groups of image blockIdx.y, one
// or as many as lie in 32 channels; its waves share the chunks, and the first one does the rest.
// sums[image][channel] = {S1, S2};  dx = g * a + d * k2 + k1 with coef[image][group] = {k1, k2}
constexpr int COEF_WAVES = 16;
__global__ __launch_bounds__(64 * COEF_WAVES) void gn_bwd_coef_kernel(const float* __restrict__ partial, const double* __restrict__ stats,
                                                         const float* __restrict__ gamma, GnShape s, int bundle,
                                                         double* __restrict__ sums, float* __restrict__ coef) {
    __shared__ double red[COEF_WAVES][64][2];
    const int n = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int g_lo = blockIdx.x * bundle, g_hi = min(s.groups, g_lo + bundle), c_lo = g_lo * s.k, c_hi = g_hi * s.k;
    double p1 = 0.0, p2 = 0.0;
    for (int c0 = c_lo; c0 < c_hi; c0 += 64) {
        const int c = c0 + lane;
        double a = 0.0, b = 0.0, ga = 1.0, mean = 0.0, rstd = 0.0;
        if (wave == 0 && c < c_hi) {
            const double* st = stats + ((size_t)n * s.groups + c / s.k) * 2;
            mean = st[0];
            rstd = st[1];
            if (gamma) ga = gamma[c];
        }
        if (c < c_hi) {
            const float2* p = reinterpret_cast<const float2*>(partial) + (size_t)n * s.chunks * s.c + c;
            for (int r = wave; r < s.chunks; r += 8 * COEF_WAVES) {
                float2 v[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = p[(size_t)min(r + j * COEF_WAVES, s.chunks - 1) * s.c];
#pragma unroll
                for (int j = 0; j < 8; ++j) { const bool in = r + j * COEF_WAVES < s.chunks; a += in ? v[j].x : 0.f; b += in ? v[j].y : 0.f; }
            }
        }
        red[wave][lane][0] = a;
        red[wave][lane][1] = b;
        __syncthreads();
        if (wave == 0 && c < c_hi) {
#pragma unroll
            for (int j = 1; j < COEF_WAVES; ++j) { a += red[j][lane][0]; b += red[j][lane][1]; }
            b = (b - (mean - (double)(float)mean) * a) * rstd;               // xhat = (x - mean) * rstd
            double* out = sums + ((size_t)n * s.c + c) * 2;
            out[0] = a;
            out[1] = b;
            p1 += ga * a;
            p2 += ga * b;
        }
        __syncthreads();
    }
    if (wave) return;
    int groups = 1;
    if (bundle == 1) {
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) { p1 += __shfl_xor(p1, o, 64); p2 += __shfl_xor(p2, o, 64); }
    } else {                                                 // lane: channel -> lane: group
        red[0][lane][0] = p1;
        red[0][lane][1] = p2;
        __builtin_amdgcn_wave_barrier();
        groups = g_hi - g_lo;
        p1 = p2 = 0.0;
        if (lane < groups)
            for (int c = lane * s.k; c < (lane + 1) * s.k; ++c) { p1 += red[0][c][0]; p2 += red[0][c][1]; }
    }
    if (lane < groups) {
        const double m = (double)s.hw * s.k;
        const double* st = stats + ((size_t)n * s.groups + g_lo + lane) * 2;
        const double lo = st[0] - (double)(float)st[0];
        float* out = coef + ((size_t)n * s.groups + g_lo + lane) * 2;
        out[0] = (float)(st[1] * (lo * st[1] * p2 - p1) / m);
        out[1] = (float)(-st[1] * st[1] * p2 / m);
    }
}

// image row gridDim.y - 1 of the grid adds the images' sums to dgamma and dbeta instead
template <typename T, int V, int ACT, bool RES>
__global__ __launch_bounds__(NT) void gn_bwd_apply_kernel(const T* __restrict__ dy, int dy_ld, const T* __restrict__ x, int ld,
                                                          const T* __restrict__ res, int res_ld, const double* __restrict__ stats,
                                                          const float* __restrict__ gamma, const float* __restrict__ beta,
                                                          const float* __restrict__ coef, float slope, T* __restrict__ dx,
                                                          T* __restrict__ dres, const double* __restrict__ sums, float* __restrict__ dgamma,
                                                          float* __restrict__ dbeta, GnShape s) {
    const int n = blockIdx.y;
    if (n == (int)gridDim.y - 1) {
        if (blockIdx.z == 0)
            for (int b = blockIdx.x; b * 32 < s.c; b += gridDim.x) sum_images(sums, n, s.c, b, dgamma, dbeta);
        return;
    }
    Place at;
    at.set<V>(s);
    if (!at.active) return;
    const double* st0 = stats + (size_t)n * s.groups * 2;
    AffineIn<V> in;
    in.params(gamma, beta, at.col);
    in.groups(st0, 0, at.col, s.k);
    float k1[V], k2[V];
    GroupOf of(at.col, s.k);
#pragma unroll
    for (int i = 0; i < V; ++i, of.next()) {
        const float* q = coef + ((size_t)n * s.groups + of.g) * 2;
        k1[i] = q[0];
        k2[i] = q[1];
    }
    __builtin_amdgcn_sched_barrier(0);
    Affine<V> k;
    const T* gp = dy + (size_t)n * s.hw * dy_ld + at.col;
    const T* xp = x + (size_t)n * s.hw * ld + at.col;
    const T* rp = RES ? res + (size_t)n * s.hw * res_ld + at.col : nullptr;
    T* op = dx + (size_t)n * s.hw * s.c + at.col;
    T* qp = RES && dres ? dres + (size_t)n * s.hw * s.c + at.col : nullptr;
    const auto write = [&](float (&g)[V], float (&d)[V], long long row) {
        Chunk<T, V> o, t;
#pragma unroll
        for (int i = 0; i < V; ++i) d[i] = fmaf(g[i], k.a[i], fmaf(d[i], k2[i], k1[i]));
        o.put(d);
        o.store(op + (size_t)row * s.c);
        if constexpr (RES) { if (qp) { t.put(g); t.store(qp + (size_t)row * s.c); } }
    };
    const auto one = [&](long long r) {
        float g[V], d[V];
        again<T, V, ACT, RES>(k, r, gp, dy_ld, xp, ld, rp, res_ld, slope, st0, 0, gamma, beta, at.col, s.k, g, d);
        write(g, d, r);
    };
    Chunk<T, V> u[2][UNR], v[2][UNR], w[2][UNR];
    at.walk<UNR, 2>(s, [&](auto h, long long r) {
#pragma unroll
        for (int j = 0; j < UNR; ++j) {
            u[h][j].load(gp + (size_t)(r + j * at.slots) * dy_ld);
            v[h][j].load(xp + (size_t)(r + j * at.slots) * ld);
            if constexpr (RES) w[h][j].load(rp + (size_t)(r + j * at.slots) * res_ld);
        }
    }, [&] { k.set(in); }, [&](auto h, long long r) {
        unsigned near = 0;
#pragma unroll
        for (int j = 0; j < UNR; ++j) {
            float g[V], d[V];
            near |= (unsigned)bwd_vector<T, V, ACT, RES>(k, u[h][j], v[h][j], w[h][j], slope, g, d) << j;
            write(g, d, r + j * at.slots);
            __builtin_amdgcn_sched_barrier(0);             // vector by vector, as above
        }
        for (; near; near &= near - 1) one(r + __builtin_ctz(near) * at.slots);            // rare: written again
    }, one);
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
    // Up to six workgroups per CU, as many as share both the trips of an image and the CUs evenly: 6x64x512x1024 bf16,
    // forward + backward, takes 584 us with 1,896 workgroups (7.4 per CU), 551 with 1,536.  A small image goes down to one
    // trip per workgroup (3x80x77x131: 52 us, 63 with at least three; 6x512x64x128 with residual: 124 with two trips of six
    // workgroups per CU, 131 with four of three).
    const long long trips = (hw + (long long)UNR * slots - 1) / ((long long)UNR * slots), per = (long long)n * p.zs;
    double best = 0.0;
    for (int w = 6; w >= 1; --w) {
        long long chunks = 256LL * w / per;
        if (chunks > trips) chunks = trips;
        if (chunks < 1) chunks = 1;
        const long long each = (trips + chunks - 1) / chunks;
        chunks = (trips + each - 1) / each;
        const double even = (double)(trips * per) / (double)(each * ((per * chunks + 255) / 256 * 256));
        if (even > best * 1.02) { best = even; p.s.chunks = (int)chunks; }
    }
    return p;
}

// The cell kernels' split, or slabs = 0 where a cell of whole groups does not fit `most` vectors per thread.  Slabs are as
// narrow as 128 bytes (one memory line) if there would be fewer than 256 cells otherwise, or 64 where only that fits.
Cell make_cell(int dtype, int n, long long hw, int c, int groups, bool vec, int most) {
    Cell s = {(int)hw, c, groups, c / groups, 0, 0};
    if (!vec || hw > 64 * CT) return s;
    const int v = dtype == UR_BF16 ? 8 : 4, esz = dtype == UR_BF16 ? 2 : 4;
    int base = s.k;
    while (base % v) base += s.k;                          // whole groups and whole vectors; divides c
    if (base / v > CT / 4) return s;                       // (with a wide slab's sums the backward pass would need more than 64 KB of LDS)
    const int units = c / base;
    const auto fits = [&](int m) {
        const int cqs = m * base / v;
        return (cqs <= 64 || m == 1) && (hw + CT / cqs - 1) / (CT / cqs) <= most;
    };
    int m = units;
    while (m > 1 && (!fits(m) || (long long)n * ((units + m - 1) / m) < 256)) {
        if (fits(m) && (m - 1) * base * esz < 128) break;
        --m;
    }
    if (!fits(m) || (m * base * esz < 64 && m < units)) return s;
    if ((long long)n * ((units + m - 1) / m) > 0x7fffffLL) return s;   // a launch has fewer than 2^32 threads
    s.slab = m * base;
    s.slabs = (units + m - 1) / m;
    return s;
}
int cell_vectors(const Cell& s, int v) { const int slots = CT / (s.slab / v); return (s.hw + slots - 1) / slots; }

constexpr int FWD_MOST = 16, BWD_MOST = 8;              // vectors (pairs of vectors) per thread of a cell

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

#define GN_TYPE(dtype, v, ...)                                                                                   \
    do {                                                                                                         \
        if ((dtype) == UR_BF16 && (v) == 8) { typedef bf16_t T; constexpr int V = 8; __VA_ARGS__; }               \
        else if ((dtype) == UR_BF16) { typedef bf16_t T; constexpr int V = 1; __VA_ARGS__; }                      \
        else if ((v) == 4) { typedef float T; constexpr int V = 4; __VA_ARGS__; }                                 \
        else { typedef float T; constexpr int V = 1; __VA_ARGS__; }                                               \
    } while (0)
#define GN_VEC_TYPE(dtype, ...)                                                                                   \
    do {                                                                                                          \
        if ((dtype) == UR_BF16) { typedef bf16_t T; constexpr int V = 8; __VA_ARGS__; }                            \
        else { typedef float T; constexpr int V = 4; __VA_ARGS__; }                                                \
    } while (0)
// vectors per thread of a cell, rounded up to a built size
#define GN_K2(k, ...)                                                                     \
    do {                                                                                  \
        if ((k) <= 2) { constexpr int K = 2; __VA_ARGS__; }                                \
        else { constexpr int K = 8; __VA_ARGS__; }                                         \
    } while (0)
#define GN_K3(k, ...)                                                                     \
    do {                                                                                  \
        if ((k) <= 2) { constexpr int K = 2; __VA_ARGS__; }                                \
        else if ((k) <= 8) { constexpr int K = 8; __VA_ARGS__; }                           \
        else { constexpr int K = 16; __VA_ARGS__; }                                        \
    } while (0)

int check(const char* what, int dtype, int n, long long hw, int c, int groups, int act) {
    UR_REQUIRE(dtype == UR_F32 || dtype == UR_BF16, "%s: bad dtype %d", what, dtype);
    UR_REQUIRE(n > 0 && hw > 0 && c > 0 && groups > 0, "%s: non-positive sizes (n %d, pixels %lld, channels %d, groups %d)", what, n, hw, c, groups);
    UR_REQUIRE(c % groups == 0, "%s: %d channels are not divisible by %d groups", what, c, groups);
    UR_REQUIRE(n < 65535 && hw <= (1LL << 40) && c <= 16384, "%s: sizes beyond the limits (65534 images, 2^40 pixels, 16384 channels)", what);
    UR_REQUIRE(act >= UR_ACT_NONE && act <= UR_ACT_SILU, "%s: bad activation %d", what, act);
    return UR_OK;
}

// the largest of what the variants need: the caller need not know which one a call takes
size_t fwd_bytes(int dtype, int n, long long hw, int c, int groups) {
    size_t most = 16;
    for (int vec = 0; vec < 2; ++vec) {
        if (vec && c % (dtype == UR_BF16 ? 8 : 4)) continue;
        const Plan p = make_plan(dtype, n, hw, c, groups, vec);
        const size_t b = (size_t)n * p.s.chunks * p.zs * groups * 2 * sizeof(double);
        if (b > most) most = b;
    }
    return most;
}
size_t bwd_sums_bytes(int n, int c) { return (size_t)n * c * 2 * sizeof(double); }
size_t bwd_bytes(int dtype, int n, long long hw, int c, int groups) {
    size_t most = 0;
    for (int vec = 0; vec < 2; ++vec) {
        if (vec && c % (dtype == UR_BF16 ? 8 : 4)) continue;
        const Plan p = make_plan(dtype, n, hw, c, groups, vec);
        const size_t b = (size_t)n * p.s.chunks * c * 2 * sizeof(float);
        if (b > most) most = b;
    }
    return bwd_sums_bytes(n, c) + most + (size_t)n * groups * 2 * sizeof(float);
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
    const Cell cell = make_cell(dtype, n, hw, c, groups, vec, FWD_MOST);
    if (cell.slabs) {
        GN_VEC_TYPE(dtype, {
            const int span = cell.k % V == 0 ? V : cell.k % 4 == 0 ? 4 : cell.k % 2 == 0 ? 2 : 1;
            const int na = V / span;
            const size_t lds = sizeof(double) * ((na > 4 ? na : 2 * na) * (CT + PAD) + 2 * (cell.slab / cell.k));
            const dim3 grid(n * cell.slabs);
            GN_K3(cell_vectors(cell, V), {
                if (residual) hipLaunchKernelGGL((gn_fwd_cell_kernel<T, V, K, true>), grid, dim3(CT), lds, st, (const T*)x, x_ld, (const T*)residual, res_ld, gamma, beta, eps, act, slope, (T*)y, y_ld, stats, cell);
                else hipLaunchKernelGGL((gn_fwd_cell_kernel<T, V, K, false>), grid, dim3(CT), lds, st, (const T*)x, x_ld, (const T*)nullptr, 0, gamma, beta, eps, act, slope, (T*)y, y_ld, stats, cell);
            });
        });
        return ur_check_launch("gn_act_fwd");
    }
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
    double* sums = (double*)workspace;
    const Cell cell = make_cell(dtype, n, hw, c, groups, vec, BWD_MOST);
    if (cell.slabs) {
        GN_VEC_TYPE(dtype, {
            const size_t lds = sizeof(float) * 2 * V * (CT + PAD) + sizeof(double) * 2 * cell.slab + sizeof(float) * 2 * (cell.slab / cell.k);
            const dim3 grid(n * cell.slabs);
            double* to = n > 1 ? sums : nullptr;
            GN_K2(cell_vectors(cell, V), {
                if (residual) hipLaunchKernelGGL((gn_bwd_cell_kernel<T, V, K, true>), grid, dim3(CT), lds, st, (const T*)dy, dy_ld, (const T*)x, x_ld, (const T*)residual, res_ld, stats, gamma, beta, act, slope, (T*)dx, (T*)dres, to, dgamma, dbeta, cell);
                else hipLaunchKernelGGL((gn_bwd_cell_kernel<T, V, K, false>), grid, dim3(CT), lds, st, (const T*)dy, dy_ld, (const T*)x, x_ld, (const T*)nullptr, 0, stats, gamma, beta, act, slope, (T*)dx, (T*)nullptr, to, dgamma, dbeta, cell);
            });
        });
        if (n > 1 && (dgamma || dbeta)) hipLaunchKernelGGL(gn_params_kernel, dim3(ur_cdiv(c, 32)), dim3(NT), 0, st, sums, n, c, dgamma, dbeta);
        return ur_check_launch("gn_act_bwd");
    }
    const Plan p = make_plan(dtype, n, hw, c, groups, vec);
    float* partial = (float*)(sums + (size_t)n * c * 2);
    float* coef = partial + (size_t)n * p.s.chunks * c * 2;
    const dim3 grid(p.s.chunks, n, p.zs);
    GN_TYPE(dtype, p.v, GN_ACT(act, {
        if (residual) hipLaunchKernelGGL((gn_bwd_reduce_kernel<T, V, ACT, true>), grid, dim3(NT), 0, st, (const T*)dy, dy_ld, (const T*)x, x_ld, (const T*)residual, res_ld, stats, gamma, beta, slope, p.s, partial);
        else hipLaunchKernelGGL((gn_bwd_reduce_kernel<T, V, ACT, false>), grid, dim3(NT), 0, st, (const T*)dy, dy_ld, (const T*)x, x_ld, (const T*)nullptr, 0, stats, gamma, beta, slope, p.s, partial);
    }));
    const int bundle = p.s.k >= 32 ? 1 : 32 / p.s.k;
    hipLaunchKernelGGL(gn_bwd_coef_kernel, dim3(ur_cdiv(groups, bundle), n), dim3(64 * COEF_WAVES), 0, st, partial, stats, gamma, p.s, bundle, sums, coef);
    if (dx) {
        const dim3 grid2(p.s.chunks, n + 1, p.zs);
        GN_TYPE(dtype, p.v, GN_ACT(act, {
            if (residual) hipLaunchKernelGGL((gn_bwd_apply_kernel<T, V, ACT, true>), grid2, dim3(NT), 0, st, (const T*)dy, dy_ld, (const T*)x, x_ld, (const T*)residual, res_ld, stats, gamma, beta, coef, slope, (T*)dx, (T*)dres, sums, dgamma, dbeta, p.s);
            else hipLaunchKernelGGL((gn_bwd_apply_kernel<T, V, ACT, false>), grid2, dim3(NT), 0, st, (const T*)dy, dy_ld, (const T*)x, x_ld, (const T*)nullptr, 0, stats, gamma, beta, coef, slope, (T*)dx, (T*)nullptr, sums, dgamma, dbeta, p.s);
        }));
    } else if (dgamma || dbeta) {
        hipLaunchKernelGGL(gn_params_kernel, dim3(ur_cdiv(c, 32)), dim3(NT), 0, st, sums, n, c, dgamma, dbeta);
    }
    return ur_check_launch("gn_act_bwd");
}

}  // extern "C"
