// AdamW over many tensors at once, with the moments in 32 or in 8 bits, and gradient clipping by the global norm.
//
//   factor = grad_scale * min(1, max_norm / (norm + 1e-6)),  norm = grad_scale * sqrt(sum over all tensors of grad^2)
//   g = factor * grad;  m += (g - m) (1 - b1);  v = b2 v + (1 - b2) g^2
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// Bound by HBM: 28 bytes per element with 32-bit moments, 16 + 1/16 with 8-bit ones, 4 more where the norm is taken (the
// gradients are read twice, the second time partly from the last-level cache).  Measured on the 134 tensors of the
// segmentation network (32 M elements): norm 23 us (5.6 TB/s), step with 32-bit moments 137 us (6.6 TB/s), with 8-bit ones
// 87 us (6.0 TB/s); a whole step of 198 M elements in 8 bits 540 us (5.9 TB/s; its kernel 534 to 590 under the profiler), where
// some 75 instructions per element are left of a budget of about 100 at the HBM rate: the square root is the correctly rounded
// one (codes depend on it), the quotient of the update is not, and what only NaN, infinity or codes below the normal ones need
// is behind one branch per wave.  The scales are reciprocals and products where the definition divides: a code next to a border
// between two can differ from the definition's.
//
// Work list.  The host hands over the tensors by value (as kernel arguments); param_table_kernel writes them as a table in
// the caller's workspace, advances the step counts and derives the bias corrections.  No staging buffer and no copy from
// the host: a captured graph replays the whole step.  The other kernels walk chunks of 2048 elements of all
// tensors in one launch and find a chunk's tensor in the sorted list of first chunks, 64 entries per look.
//
// 8-bit moments.  m and r = sqrt(v) are stored as e4m3 codes (3 mantissa bits, exponents over 2^17) with one fp32 scale per
// 256 elements that maps the block's largest value to the largest code, 448.  m is rounded to the nearest code: it moves by
// a tenth of itself per step, more than half a code step (3 to 6 %).  Below the normal codes, whose steps are larger than
// that, a falling m is rounded towards zero: to the nearest, the m of a weight without a gradient would stop at four steps
// and the weight drift for good.  That takes b1 <= 17/18: nearest rounding moves a falling m off every code only if b1 *
// 9/8 is below 17/16, so larger b1 are refused.  r moves by at most 0.05 % per step when the gradients get smaller, so
// nearest rounding would pin it for good; it is rounded up with the probability of its fraction instead, so that a rounding
// keeps its expectation (v = r^2 gains the variance: 4 to 5 % at b2 = 0.999).  A root above zero never gets the code 0: the
// next update would divide m by eps (hundreds of lr where the gradients of a block span six decades).  The 20 random bits
// per element come from a hash of the element's place in the state and the step count: the same step gives the same bits,
// and nothing is kept between calls.  The step itself uses m and v before they are rounded.
#include "ur_common.h"

namespace {

constexpr int NT = 256;
constexpr int BLOCK = 256;                   // elements per scale
constexpr int U = 2;                         // 16-byte accesses per thread, chunk and array
constexpr int CHUNK = U * NT * 4;            // elements per unit of work
constexpr int MAX_ROWS = 1024;               // tensors per table: the kernels keep its list of first chunks in the LDS
constexpr int BATCH = 136;                   // rows per table launch: kernel arguments stay under 4 KB
constexpr int MAX_PARTS = 1024;             // partial sums of the norm
constexpr long long MAX_CHUNKS = 1LL << 30;  // a chunk's number plus the grid's size stays an int
constexpr float TOP = 448.f;
constexpr double BETA1_MOST_8 = 17.0 / 18.0; // largest b1 for 8-bit moments

typedef __attribute__((ext_vector_type(4))) float fvec4_t;
typedef __attribute__((ext_vector_type(2))) float fvec2_t;

struct Row {
    float* p;
    float* g;
    long long n;
    long long block;                         // first block of 256 elements in the state buffers
    float step_size, bc2_rsqrt;              // lr / (1 - b1^t), (1 - b2^t)^-1/2
    unsigned step;
    unsigned pad;
};

struct ListBatch {
    int count, at;
    void* p[BATCH];
    void* g[BATCH];                          // null: nothing to do for this tensor
    long long n[BATCH];
    int first[BATCH];
};

// table: Row[ntensors], then int first[ntensors] (first chunk of every tensor)

__global__ __launch_bounds__(192) void param_table_kernel(ListBatch b, Row* __restrict__ rows, int ntensors,
                                                          const long long* __restrict__ blocks, int* __restrict__ steps, double lr,
                                                          double beta1, double beta2) {
    const int i = threadIdx.x, t = b.at + i;
    if (i >= b.count) return;
    Row w;
    w.p = (float*)b.p[i];
    w.g = (float*)b.g[i];
    w.n = b.g[i] ? b.n[i] : 0;
    w.block = blocks ? blocks[t] : 0;
    w.step_size = 0.f;
    w.bc2_rsqrt = 1.f;
    w.step = 0;
    w.pad = 0;
    if (steps && w.n) {
        const int step = steps[t] + 1;
        steps[t] = step;
        w.step = (unsigned)step;
        w.step_size = (float)(lr / (1.0 - pow(beta1, (double)step)));
        w.bc2_rsqrt = (float)(1.0 / sqrt(1.0 - pow(beta2, (double)step)));
    }
    rows[t] = w;
    reinterpret_cast<int*>(rows + ntensors)[t] = b.first[i];
}

// The list of first chunks in the LDS, and the tensor that a chunk belongs to: the last entry of the sorted list that is not
// above it (a whole wave looks, 64 entries at a time).
struct Finder {
    const int* first;
    int ntensors;
    __device__ __forceinline__ Finder(const Row* rows, int n) : ntensors(n) {
        __shared__ int list[MAX_ROWS];
        const int* src = reinterpret_cast<const int*>(rows + n);
        for (int i = threadIdx.x; i < n; i += NT) list[i] = src[i];
        __syncthreads();
        first = list;
    }
    __device__ __forceinline__ int operator()(int chunk) const {
        const int lane = threadIdx.x & 63;
        int lo = 0, len = ntensors;
        while (len > 1) {
            const int step = (len + 63) >> 6, at = lane * step;
            const bool below = at < len && first[lo + at] <= chunk;
            const int hits = __popcll(__ballot(below));                      // entries are sorted: a prefix of the lanes
            lo += (hits - 1) * step;
            len = min(step, len - (hits - 1) * step);
        }
        return __builtin_amdgcn_readfirstlane(lo);
    }
};

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}
// sum over a workgroup of NT threads, in every thread
__device__ __forceinline__ double group_sum(double v) {
    __shared__ double red[NT / 64];
    v = wave_sum(v);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return (red[0] + red[1]) + (red[2] + red[3]);
}

__device__ __forceinline__ bool aligned16(const void* a, const void* b) { return (((uintptr_t)a | (uintptr_t)b) & 15) == 0; }

// Addresses out of a table are global ones, which the compiler cannot know: without these types it takes the flat accesses,
// whose two wait counters hold up everything else (with that and the loads in one go: 32.5 M elements in 8 bits 87 -> 85 us,
// in 32 bits 138 -> 136).
typedef __attribute__((address_space(1))) float gfloat_t;
typedef __attribute__((address_space(1))) fvec4_t gvec4_t;
__device__ __forceinline__ fvec4_t ld4(const float* p) { return __builtin_nontemporal_load((const gvec4_t*)p); }
__device__ __forceinline__ void st4(float* p, fvec4_t v) { __builtin_nontemporal_store(v, (gvec4_t*)p); }

// squares summed in 64 bits (two fp64 instructions per element against the four bytes it is read by)
__global__ __launch_bounds__(NT) void grad_sqnorm_kernel(const Row* __restrict__ rows, int ntensors, int nchunks, double* __restrict__ parts) {
    const Finder find(rows, ntensors);
    double s = 0.0;
    for (int c = blockIdx.x; c < nchunks; c += gridDim.x) {
        const int t = find(c);
        const long long base = (long long)(c - find.first[t]) * CHUNK, n = rows[t].n;
        const gfloat_t* g = (const gfloat_t*)rows[t].g;
        if (aligned16(rows[t].g, rows[t].g) && base + CHUNK <= n) {
            fvec4_t v[U];
#pragma unroll
            for (int u = 0; u < U; ++u) v[u] = *(const gvec4_t*)(g + base + u * (NT * 4) + threadIdx.x * 4);
#pragma unroll
            for (int u = 0; u < U; ++u) {
#pragma unroll
                for (int i = 0; i < 4; ++i) s = fma((double)v[u][i], (double)v[u][i], s);
            }
        } else {
            for (long long i = base + threadIdx.x; i < n && i < base + CHUNK; i += NT) s = fma((double)g[i], (double)g[i], s);
        }
    }
    s = group_sum(s);
    if (threadIdx.x == 0) parts[blockIdx.x] = s;
}

// the factor every gradient is multiplied by; workgroup 0 writes the norm
__device__ __forceinline__ float clip_factor(const double* __restrict__ parts, int nparts, float max_norm, float grad_scale,
                                             float* __restrict__ out_norm) {
    double s = 0.0;
    for (int at = threadIdx.x; at < nparts; at += 4 * NT) {                  // four loads at a time, in a fixed order
        double v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = parts[min(at + j * NT, nparts - 1)];
#pragma unroll
        for (int j = 0; j < 4; ++j) s += at + j * NT < nparts ? v[j] : 0.0;
    }
    const float norm = (float)(sqrt(group_sum(s)) * (double)fabsf(grad_scale));
    if (out_norm && blockIdx.x == 0 && threadIdx.x == 0) *out_norm = norm;
    float f = max_norm / (norm + 1e-6f);
    if (f > 1.f) f = 1.f;                                                    // (a NaN norm stays one)
    return f * grad_scale;
}

__global__ __launch_bounds__(NT) void grad_scale_kernel(const Row* __restrict__ rows, int ntensors, int nchunks,
                                                        const double* __restrict__ parts, int nparts, float max_norm,
                                                        float* __restrict__ out_norm) {
    const float f = clip_factor(parts, nparts, max_norm, 1.f, out_norm);
    if (f == 1.f) return;                                                    // within the limit: nothing to write
    const Finder find(rows, ntensors);
    for (int c = blockIdx.x; c < nchunks; c += gridDim.x) {
        const int t = find(c);
        const long long base = (long long)(c - find.first[t]) * CHUNK, n = rows[t].n;
        float* g = rows[t].g;
        if (aligned16(g, g) && base + CHUNK <= n) {
            fvec4_t v[U];
            float* p = g + base + threadIdx.x * 4;
#pragma unroll
            for (int u = 0; u < U; ++u) v[u] = ld4(p + u * (NT * 4));
#pragma unroll
            for (int u = 0; u < U; ++u) st4(p + u * (NT * 4), v[u] * f);
        } else {
            for (long long i = base + threadIdx.x; i < n && i < base + CHUNK; i += NT) ((gfloat_t*)g)[i] *= f;
        }
    }
}

// ------------------------------------------------------------------ 8-bit codes
// 20 pseudo-random bits for element `place` of the state at step `step`: a multiplicative hash of place * HASH_PLACE + step *
// HASH_STEP
constexpr unsigned HASH_PLACE = 0x9E3779B9u, HASH_STEP = 0xA3D8F1B5u;
__device__ __forceinline__ unsigned dither(unsigned h) {
    h = (h ^ (h >> 16)) * 0x45D9F3B5u;
    h = (h ^ (h >> 15)) * 0x2C92774Du;
    return (h ^ (h >> 16)) & 0xFFFFFu;
}
__device__ __forceinline__ bool is_finite(float v) { return (__float_as_uint(v) & 0x7f800000u) != 0x7f800000u; }

__device__ __forceinline__ fvec4_t decode4(unsigned q) {
    const fvec2_t a = __builtin_amdgcn_cvt_pk_f32_fp8((int)q, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)q, true);
    fvec4_t v = {a[0], a[1], b[0], b[1]};
    return v;
}
// nearest codes of values within [-448, 448]
__device__ __forceinline__ unsigned encode4(fvec4_t y) {
    int q = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], q, true);
}
// y in [0, 448]: the code below plus one with the probability of the fraction.  Normal codes drop 20 mantissa bits, so
// adding the dither there carries into the code; below 2^-6 the codes are multiples of 2^-9.
constexpr float LOWEST_NORMAL = 0.015625f;
__device__ __forceinline__ unsigned encode_up(float y, unsigned d) { return ((__float_as_uint(y) + d) >> 20) - ((127 - 7) << 3); }
__device__ __forceinline__ unsigned encode_up_low(float y, unsigned d) { return ((unsigned)(y * 536870912.f) + d) >> 20; }     // y * 2^9 * 2^20
constexpr unsigned CODE_NAN = 0x7f;

// maximum of non-negative values over a wave, in every lane
template <int CTRL, int ROWS> __device__ __forceinline__ float max_with(float v) {
    return fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, ROWS, 0xf, false)));
}
__device__ __forceinline__ float wave_max(float v) {
    v = max_with<0x111, 0xf>(v);             // row_shr 1, 2, 4, 8: the last lane of a row of 16 has the row's maximum
    v = max_with<0x112, 0xf>(v);
    v = max_with<0x114, 0xf>(v);
    v = max_with<0x118, 0xf>(v);
    v = max_with<0x142, 0xa>(v);             // row_bcast 15 into rows 1 and 3, row_bcast 31 into rows 2 and 3
    v = max_with<0x143, 0xc>(v);
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}

struct Hyper {
    float b1c, b2, b2c, eps, keep;           // 1 - b1, b2, 1 - b2, eps, 1 - lr * wd
};

// Every operation rounded by itself: the codes of an 8-bit state are then a function of the inputs alone, and not of which
// products the compiler contracts (a value next to a border between two codes would go another way).
__device__ __forceinline__ void adamw_one(float& p, float g, float& m, float& v, float& root, const Hyper& h, float step_size, float bc2_rsqrt) {
#pragma clang fp contract(off)
    m = m + (g - m) * h.b1c;
    v = v * h.b2 + (h.b2c * g) * g;
    root = sqrtf(v);
    p = p * h.keep - step_size * (m * __builtin_amdgcn_rcpf(root * bc2_rsqrt + h.eps));
}

// Four elements of the state: 32 bits as they are, 8 bits as codes (the root of the second moment) with one scale per block
// of 256, which one wave holds at four elements per lane.
template <int BITS> struct State;
template <> struct State<32> {
    fvec4_t m, v;
    __device__ __forceinline__ void load(const void* m_, const void* v_, const float*, const float*, long long at, long long) {
        m = ld4((const float*)m_ + at);
        v = ld4((const float*)v_ + at);
    }
    __device__ __forceinline__ void decode() {}
    __device__ __forceinline__ void store(void* m_, void* v_, float*, float*, long long at, long long, const fvec4_t&, unsigned) {
        st4((float*)m_ + at, m);
        st4((float*)v_ + at, v);
    }
};
template <> struct State<8> {
    fvec4_t m, v;
    unsigned qm, qv;
    float sm, sv;
    __device__ __forceinline__ void load(const void* m_, const void* v_, const float* ms, const float* vs, long long at, long long blk) {
        qm = __builtin_nontemporal_load((const unsigned*)m_ + (at >> 2));
        qv = __builtin_nontemporal_load((const unsigned*)v_ + (at >> 2));
        sm = ms[blk];
        sv = vs[blk];
    }
    __device__ __forceinline__ void decode() {
        m = decode4(qm) * sm;
        v = decode4(qv) * sv;
        v = v * v;
    }
    __device__ __forceinline__ void store(void* m_, void* v_, float* ms, float* vs, long long at, long long blk, const fvec4_t& root, unsigned step) {
        float am = 0.f, ar = 0.f, z = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            am = fmaxf(am, fabsf(m[i]));
            ar = fmaxf(ar, root[i]);
            z = fmaf(m[i], 0.f, fmaf(root[i], 0.f, z));                       // NaN if any of them is infinite or NaN
        }
        const bool all_finite = !__any(z != 0.f);
        if (!all_finite) {                                                    // scales from the finite values
            am = ar = 0.f;
            for (int i = 0; i < 4; ++i) {
                if (is_finite(m[i])) am = fmaxf(am, fabsf(m[i]));
                if (is_finite(root[i])) ar = fmaxf(ar, root[i]);
            }
        }
        am = fmaxf(wave_max(am), 0x1p-100f);                                  // keeps 448 / am finite
        ar = fmaxf(wave_max(ar), 0x1p-100f);
        const float im = 1.f / am * TOP, ir = 1.f / ar * TOP;
        fvec4_t y, r;
        unsigned d[4], q = 0;
        bool low = false;
        const unsigned h0 = (unsigned)at * HASH_PLACE + step * HASH_STEP;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            y[i] = m[i] * im;                                                 // at most a rounding above 448, which is its nearest code
            r[i] = fminf(root[i] * ir, TOP);
            low |= fminf(r[i], fabsf(y[i])) < LOWEST_NORMAL;
            d[i] = dither(h0 + i * HASH_PLACE);
            q |= encode_up(r[i], d[i]) << (8 * i);
        }
        if (__any(low)) {
            q = 0;
            const fvec4_t before = decode4(qm) * sm;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (fabsf(y[i]) < LOWEST_NORMAL && fabsf(m[i]) < fabsf(before[i])) y[i] = truncf(y[i] * 512.f) * (1.f / 512.f);
                const unsigned code = r[i] < LOWEST_NORMAL ? encode_up_low(r[i], d[i]) : encode_up(r[i], d[i]);
                q |= (root[i] > 0.f ? max(code, 1u) : code) << (8 * i);
            }
        }
        unsigned qm_new = encode4(y);
        if (!all_finite) {                                                    // an infinite or NaN value becomes the NaN code and stays alone
            for (int i = 0; i < 4; ++i) {
                if (!is_finite(m[i])) qm_new |= CODE_NAN << (8 * i);
                if (!is_finite(root[i])) q |= CODE_NAN << (8 * i);
            }
        }
        __builtin_nontemporal_store(qm_new, (unsigned*)m_ + (at >> 2));
        __builtin_nontemporal_store(q, (unsigned*)v_ + (at >> 2));
        if ((threadIdx.x & 63) == 0) { ms[blk] = am * (1.f / TOP); vs[blk] = ar * (1.f / TOP); }
    }
};

template <int BITS>
__global__ __launch_bounds__(NT) void adamw_kernel(const Row* __restrict__ rows, int ntensors, int nchunks, void* __restrict__ m_,
                                                   void* __restrict__ v_, float* __restrict__ ms, float* __restrict__ vs, Hyper h,
                                                   const double* __restrict__ parts, int nparts, float max_norm, float grad_scale,
                                                   float* __restrict__ out_norm) {
    float factor = grad_scale;
    if (nparts) factor = clip_factor(parts, nparts, max_norm, grad_scale, out_norm);
    const Finder find(rows, ntensors);
    for (int c = blockIdx.x; c < nchunks; c += gridDim.x) {
        const int t = find(c);
        const Row row = rows[t];
        const long long base = (long long)(c - find.first[t]) * CHUNK, n = row.n;
        const long long at0 = row.block * BLOCK;                              // the state is padded to whole blocks
        if (aligned16(row.p, row.g) && base + CHUNK <= n) {
            const long long e0 = base + threadIdx.x * 4;
            const long long b0 = row.block + (base + (threadIdx.x & ~63) * 4) / BLOCK;
            fvec4_t p[U], g[U];
            State<BITS> st[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const long long e = e0 + u * (NT * 4);
                p[u] = ld4(row.p + e);
                g[u] = ld4(row.g + e);
                st[u].load(m_, v_, ms, vs, at0 + e, b0 + u * (NT * 4 / BLOCK));
            }
            __builtin_amdgcn_sched_barrier(0);                                // all loads of the chunk before the first wait
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const long long e = e0 + u * (NT * 4);
                fvec4_t root;
                st[u].decode();
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float pi = p[u][i], mi = st[u].m[i], vi = st[u].v[i], ri;
                    adamw_one(pi, g[u][i] * factor, mi, vi, ri, h, row.step_size, row.bc2_rsqrt);
                    p[u][i] = pi; st[u].m[i] = mi; st[u].v[i] = vi; root[i] = ri;
                }
                st4(row.p + e, p[u]);
                st[u].store(m_, v_, ms, vs, at0 + e, b0 + u * (NT * 4 / BLOCK), root, row.step);
            }
        } else {
            // the end of a tensor, or one that is not aligned to 16 bytes: element-wise parameters and gradients
            for (int u = 0; u < U; ++u) {
                const long long wave0 = base + u * (NT * 4) + (threadIdx.x & ~63) * 4, e = base + u * (NT * 4) + threadIdx.x * 4;
                if (wave0 >= n) break;                                        // (a whole wave: its block does not exist)
                fvec4_t p = {0.f, 0.f, 0.f, 0.f}, g = p, root;
#pragma unroll
                for (int i = 0; i < 4; ++i) if (e + i < n) { p[i] = ((const gfloat_t*)row.p)[e + i]; g[i] = ((const gfloat_t*)row.g)[e + i]; }
                State<BITS> st;
                st.load(m_, v_, ms, vs, at0 + e, row.block + wave0 / BLOCK);
                st.decode();
#pragma unroll
                for (int i = 0; i < 4; ++i) {                                 // (behind the end zero also under a NaN factor)
                    float pi = p[i], mi = st.m[i], vi = st.v[i], ri;
                    adamw_one(pi, e + i < n ? g[i] * factor : 0.f, mi, vi, ri, h, row.step_size, row.bc2_rsqrt);
                    p[i] = pi; st.m[i] = mi; st.v[i] = vi; root[i] = ri;
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) if (e + i < n) ((gfloat_t*)row.p)[e + i] = p[i];
                st.store(m_, v_, ms, vs, at0 + e, row.block + wave0 / BLOCK, root, row.step);
            }
        }
    }
}

int norm_parts(long long chunks) { return (int)(chunks < MAX_PARTS ? chunks : MAX_PARTS); }

}  // namespace

extern "C" {

size_t ur_param_table_bytes(int ntensors) { return ntensors <= 0 ? 0 : (size_t)ntensors * (sizeof(Row) + sizeof(int)); }
int ur_param_table_max_rows(void) { return MAX_ROWS; }
int ur_grad_sqnorm_max_parts(void) { return MAX_PARTS; }

int ur_param_table(const long long* params, const long long* grads, const long long* sizes, const long long* blocks, int ntensors,
                   void* table, size_t table_bytes, int* steps, double lr, double beta1, double beta2, long long* nchunks,
                   ur_stream_t s) {
    UR_REQUIRE(grads && sizes && ntensors > 0 && table && nchunks, "param_table: bad arguments");
    UR_REQUIRE(ntensors <= MAX_ROWS, "param_table: more than %d tensors in one table", MAX_ROWS);
    UR_REQUIRE(table_bytes >= ur_param_table_bytes(ntensors), "param_table: table too small");
    long long chunks = 0;
    for (int i = 0; i < ntensors; ++i) {
        UR_REQUIRE(sizes[i] >= 0 && sizes[i] <= (1LL << 40), "param_table: a tensor of %lld elements", sizes[i]);
        if (grads[i]) chunks += (sizes[i] + CHUNK - 1) / CHUNK;
    }
    UR_REQUIRE(chunks > 0 && chunks <= MAX_CHUNKS, "param_table: no gradient with elements, or too many elements");
    int first = 0;
    for (int at = 0; at < ntensors; at += BATCH) {
        ListBatch b = {};
        b.count = ntensors - at < BATCH ? ntensors - at : BATCH;
        b.at = at;
        for (int i = 0; i < b.count; ++i) {
            b.p[i] = params ? (void*)params[at + i] : nullptr;
            b.g[i] = sizes[at + i] ? (void*)grads[at + i] : nullptr;
            b.n[i] = sizes[at + i];
            b.first[i] = first;
            if (b.g[i]) first += (int)((b.n[i] + CHUNK - 1) / CHUNK);
        }
        hipLaunchKernelGGL(param_table_kernel, dim3(1), dim3(192), 0, (hipStream_t)s, b, (Row*)table, ntensors, blocks, steps, lr, beta1, beta2);
    }
    *nchunks = chunks;
    return ur_check_launch("param_table");
}

int ur_grad_sqnorm(const void* table, int ntensors, long long nchunks, double* parts, int* nparts, ur_stream_t s) {
    UR_REQUIRE(table && ntensors > 0 && ntensors <= MAX_ROWS && nchunks > 0 && nchunks <= MAX_CHUNKS && parts && nparts, "grad_sqnorm: bad arguments");
    *nparts = norm_parts(nchunks);
    hipLaunchKernelGGL(grad_sqnorm_kernel, dim3(*nparts), dim3(NT), 0, (hipStream_t)s, (const Row*)table, ntensors, (int)nchunks, parts);
    return ur_check_launch("grad_sqnorm");
}

int ur_grad_clip(const void* table, int ntensors, long long nchunks, const double* parts, int nparts, float max_norm, float* out_norm,
                 ur_stream_t s) {
    UR_REQUIRE(table && ntensors > 0 && ntensors <= MAX_ROWS && nchunks > 0 && nchunks <= MAX_CHUNKS && parts && nparts > 0, "grad_clip: bad arguments");
    hipLaunchKernelGGL(grad_scale_kernel, dim3(norm_parts(nchunks)), dim3(NT), 0, (hipStream_t)s, (const Row*)table, ntensors, (int)nchunks,
                       parts, nparts, max_norm, out_norm);
    return ur_check_launch("grad_clip");
}

int ur_adamw_multi(const void* table, int ntensors, long long nchunks, int state_bits, void* exp_avg, void* exp_avg_sq, float* exp_avg_scale,
                   float* exp_avg_sq_scale, double lr, double beta1, double beta2, double eps, double weight_decay, const double* parts,
                   int nparts, float max_norm, float grad_scale, float* out_norm, ur_stream_t s) {
    UR_REQUIRE(table && ntensors > 0 && ntensors <= MAX_ROWS && nchunks > 0 && nchunks <= MAX_CHUNKS && exp_avg && exp_avg_sq, "adamw_multi: bad arguments");
    UR_REQUIRE(state_bits == 32 || state_bits == 8, "adamw_multi: state_bits is 32 or 8 (got %d)", state_bits);
    UR_REQUIRE(state_bits == 32 || (exp_avg_scale && exp_avg_sq_scale), "adamw_multi: 8-bit states without scales");
    UR_REQUIRE(state_bits == 32 || beta1 <= BETA1_MOST_8, "adamw_multi: 8-bit moments need beta1 <= 17/18 (got %g)", beta1);
    UR_REQUIRE((((uintptr_t)exp_avg | (uintptr_t)exp_avg_sq) & 15) == 0, "adamw_multi: the state buffers are not 16-byte aligned");
    UR_REQUIRE(nparts == 0 || (nparts > 0 && parts), "adamw_multi: bad partial sums");
    const Hyper h = {(float)(1.0 - beta1), (float)beta2, (float)(1.0 - beta2), (float)eps, (float)(1.0 - lr * weight_decay)};
    // A workgroup per chunk streams best (32 M elements in 32 bits 135 us, 147 at 2048 workgroups; 198 M in 8 bits 583 and 656
    // before the accesses became global ones); with clipping every workgroup adds up the partial sums first, which 8192 of them
    // repay (8 bits 87 us, one per chunk 94).
    const long long most = nparts ? 8192 : 65536;
    const int grid = (int)(nchunks < most ? nchunks : most);
    if (state_bits == 32)
        hipLaunchKernelGGL(adamw_kernel<32>, dim3(grid), dim3(NT), 0, (hipStream_t)s, (const Row*)table, ntensors, (int)nchunks, exp_avg,
                           exp_avg_sq, exp_avg_scale, exp_avg_sq_scale, h, parts, nparts, max_norm, grad_scale, out_norm);
    else
        hipLaunchKernelGGL(adamw_kernel<8>, dim3(grid), dim3(NT), 0, (hipStream_t)s, (const Row*)table, ntensors, (int)nchunks, exp_avg,
                           exp_avg_sq, exp_avg_scale, exp_avg_sq_scale, h, parts, nparts, max_norm, grad_scale, out_norm);
    return ur_check_launch("adamw_multi");
}

}  // extern "C"
