// AdamW over many tensors at once, states in 32 or in 8 bits (clip_adamw in train.hip is the form for ONE flat fp32 buffer).
//   g = coef * grad,  coef = grad_scale * min(1, max_norm / (|grad| * grad_scale + 1e-6)),  |grad| over all tensors
//   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
// 8-bit states: every 256 consecutive elements of a tensor share two fp32 scales S = (largest of the block) / 448, and hold
// m = Sm * e4m3 and r = sqrt(v) = Sr * e4m3.  The ROOT is held because e4m3 spans a ratio of 2^17.8 between its smallest and
// largest code, and v spans the square of what its root spans.  A root that is not zero is stored at least as the smallest
// code (2^-9): it never becomes zero beside a first moment that is not, which would divide by eps alone.  The largest of a
// block keeps fp32 precision through its scale, so a block whose elements grow evenly keeps its codes and none stands
// still under the slow decay of v.  The step itself uses m and v before they are rounded.
// Bound by memory: 120 M parameters in 32 bits 82 us for the norm (5.8 TB/s) and 547 for the step (6.1 TB/s), 30 M with 8-bit states
// 14 and 86 us (5.0 TB/s; 230 vector instructions per 256 elements keep the vector units busy 56 % of it), 479 M 1386 us together.  Small models are two launches
// of 4.5 and 6.2 us: the table, the data, for the step also the partial sums, one trip to memory each.  Without clipping one thread's
// launch (the step count and two powers in 64 bits, 2.5 to 5 us) stands in the norm's place.  With 8-bit states the instructions are the
// same for 16-bit parameters and gradients as for fp32 ones: 120 M of them 334 us instead of 358, at 10 bytes per element instead of 16.
// A block that holds an infinity or a NaN gets a scale that is not finite: all its elements are NaN from the next step on.
#include <float.h>

#include "common.h"

namespace {

// the products and sums below are rounded one by one (no fused multiply-add): codes are rounded results, and whoever
// repeats the formulas operation by operation in fp32 gets the same ones
#pragma clang fp contract(off)

typedef f32x4 f32x4_u __attribute__((aligned(4)));
typedef u32x2 u32x2_u __attribute__((aligned(2)));
typedef unsigned u32_u __attribute__((aligned(1)));

constexpr int BLOCK = 256;                // elements that share a scale: one wave, four per lane
constexpr int SCALARS = 4;                // floats at the workspace's head, the partial sums of squares follow

// A launch's table of tensors travels in its arguments (4 KB at most): nothing is copied to the device, nothing has to live
// on, and a captured launch holds its own table.
struct tensor32 {
    void* p; const void* g; float* m; float* v;
    long long n;
    float wd;
    int kinds;                            // bit 0: p in 16 bits, bit 1: g in 16 bits
};
struct tensor8 {
    void* p; const void* g; unsigned char* m; unsigned char* v;
    long long n;
    float wd;
    int kinds;
    float* ms; float* vs;
};
struct gradient {
    const void* g;
    long long n;                          // elements; their complement where they have 16 bits
};
template <typename T, int N> struct batch {
    T t[N];
    int first[N + 1];                     // first chunk of each tensor, then their number
    int count;
};
typedef batch<tensor32, 76> batch32;
typedef batch<tensor8, 58> batch8;
constexpr int GRADIENTS = 190;
typedef batch<gradient, GRADIENTS> batchg;

template <bool WHOLE> __device__ __forceinline__ f32x4 ld4e(const float* p, int k) {
    if (WHOLE || k >= 4) return __builtin_nontemporal_load((const f32x4_u*)p);
    f32x4 o;
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = j < k ? p[j] : 0.f;
    return o;
}
template <bool WHOLE> __device__ __forceinline__ f32x4 ld4e(const bf16_t* p, int k) {
    if (WHOLE || k >= 4) {
        const u32x2 v = __builtin_nontemporal_load((const u32x2_u*)p);
        return f32x4{bf_lo(v[0]), bf_hi(v[0]), bf_lo(v[1]), bf_hi(v[1])};
    }
    f32x4 o;
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = j < k ? bf2f(p[j]) : 0.f;
    return o;
}
template <bool WHOLE> __device__ __forceinline__ void st4e(float* p, int k, f32x4 o) {
    if (WHOLE || k >= 4) {
        __builtin_nontemporal_store(o, (f32x4_u*)p);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j < k) p[j] = o[j];
    }
}
template <bool WHOLE> __device__ __forceinline__ void st4e(bf16_t* p, int k, f32x4 o) {
    if (WHOLE || k >= 4) {
        const u32x2 v = {to_2h16(o[0], o[1]), to_2h16(o[2], o[3])};
        __builtin_nontemporal_store(v, (u32x2_u*)p);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j < k) p[j] = to_h16(o[j]);
    }
}
template <bool WHOLE> __device__ __forceinline__ unsigned ld_codes(const unsigned char* p, int k) {
    if (WHOLE || k >= 4) return __builtin_nontemporal_load((const u32_u*)p);
    unsigned v = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (j < k) v |= (unsigned)p[j] << (8 * j);
    return v;
}
template <bool WHOLE> __device__ __forceinline__ void st_codes(unsigned char* p, int k, unsigned v) {
    if (WHOLE || k >= 4) {
        __builtin_nontemporal_store(v, (u32_u*)p);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j < k) p[j] = (unsigned char)(v >> (8 * j));
    }
}
__device__ __forceinline__ f32x4 from_e4m3(unsigned v, float scale) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)v, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)v, true);
    return f32x4{lo[0] * scale, lo[1] * scale, hi[0] * scale, hi[1] * scale};
}
__device__ __forceinline__ unsigned to_e4m3(f32x4 v) {
    const int r = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], r, true);
}
// largest magnitude over a wave, by the bits: NaN is above infinity, infinity above every number
__device__ __forceinline__ float wave_amax(f32x4 v) {
    unsigned a = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) a = max(a, __builtin_bit_cast(unsigned, (float)v[j]) & 0x7fffffffu);
    return __builtin_bit_cast(float, wave_umax_dpp(a));
}
// Scales of a wave's blocks, and what their elements are multiplied by before they become codes.  One division for up to eight of
// them: lanes k and 8 + k (of every 16) come with the k-th block's largest magnitude t, lane k leaves with 448 / t, lane 8 + k
// with t / 448.  Below 1e-30 the factor would leave the range of fp32: such blocks are scaled as if t were 1e-30.
__device__ __forceinline__ float block_scales(float t) {
    const bool scale = threadIdx.x & 8;
    if (t > 0.f && t < 1e-30f) t = 1e-30f;
    const float q = (scale ? t : 448.0f) / (scale ? 448.0f : t);
    return t == 0.f ? 0.f : q;
}
__device__ __forceinline__ float of_lane(float v, int k) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), k));
}

// The tensor of a workgroup's first chunk: all borders are compared at once (one trip to the table, which no cache holds yet; a
// walk makes one per 16 borders, one after the other).
template <typename T, int N> __device__ __forceinline__ int tensor_of(const batch<T, N>& b, int chunk) {
    const int lane = threadIdx.x & 63;
    int below = 0;
#pragma unroll
    for (int i = 0; i < (N + 63) / 64; ++i) {
        const int k = i * 64 + lane;
        const int border = b.first[min(k + 1, N)];
        below += __popcll(__builtin_amdgcn_ballot_w64(k < b.count && border <= chunk));
    }
    return below;
}

// step count and the two bias corrections of this step, by one thread
__device__ void next_step(int32_t* step_dev, float* scalars, double lr, double b1, double b2) {
    const int t = *step_dev + 1;
    *step_dev = t;
    scalars[0] = (float)(lr / (1.0 - pow(b1, (double)t)));
    scalars[1] = (float)sqrt(1.0 - pow(b2, (double)t));
}
__global__ void adamw_prepare_kernel(int32_t* step_dev, float* scalars, float* norm, double lr, double b1, double b2) {
    if (threadIdx.x) return;
    next_step(step_dev, scalars, lr, b1, b2);
    if (norm) *norm = 0.f;                // there is no gradient
}

// sum of squares of the gradients: one partial sum per workgroup, joined by every workgroup of the update in one order
constexpr int NORM_CHUNK = 8192;
__global__ __launch_bounds__(256) void adamw_norm_kernel(batchg b, float* parts, int32_t* step_dev, float* scalars, double lr,
                                                         double b1, double b2) {
    if (step_dev && blockIdx.x == 0 && threadIdx.x == 0) next_step(step_dev, scalars, lr, b1, b2);
    f32x4 acc[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
    int chunk = b.first[b.count] - 1 - (int)blockIdx.x;
    for (int t = tensor_of(b, chunk); chunk >= 0; chunk -= gridDim.x) {
        while (chunk < b.first[t]) --t;
        const bool half = b.t[t].n < 0;
        const long long n = half ? ~b.t[t].n : b.t[t].n, start = (long long)(chunk - b.first[t]) * NORM_CHUNK;
        const float* g32 = (const float*)b.t[t].g + start + threadIdx.x * 4;
        const bf16_t* g16 = (const bf16_t*)b.t[t].g + start + threadIdx.x * 4;
        f32x4 g[NORM_CHUNK / 1024];
        if (start + NORM_CHUNK <= n) {
            if (half) {
#pragma unroll
                for (int u = 0; u < NORM_CHUNK / 1024; ++u) {
                    const u32x2 v = *(const u32x2_u*)(g16 + u * 1024);
                    g[u] = f32x4{bf_lo(v[0]), bf_hi(v[0]), bf_lo(v[1]), bf_hi(v[1])};
                }
            } else {
#pragma unroll
                for (int u = 0; u < NORM_CHUNK / 1024; ++u) g[u] = *(const f32x4_u*)(g32 + u * 1024);
            }
        } else {
#pragma unroll
            for (int u = 0; u < NORM_CHUNK / 1024; ++u) {
                const int k = (int)std::max<long long>(0, std::min<long long>(4, n - start - threadIdx.x * 4 - u * 1024));
                g[u] = half ? ld4e<false>(g16 + u * 1024, k) : ld4e<false>(g32 + u * 1024, k);
            }
        }
#pragma unroll
        for (int u = 0; u < NORM_CHUNK / 1024; ++u) acc[u & 1] += g[u] * g[u];
    }
    acc[0] += acc[1];
    const float s = wave_sum_dpp((acc[0][0] + acc[0][1]) + (acc[0][2] + acc[0][3]));
    __shared__ float part[4];
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) parts[blockIdx.x] = (part[0] + part[1]) + (part[2] + part[3]);
}

struct update_arg {
    const float* scalars;
    const float* parts;                   // NULL: no norm was asked for
    int n_parts;
    float* norm;
    float max_norm, grad_scale, lr, b1, b2, omb1, omb2, eps;
};

// what every gradient is multiplied by; the first workgroup also writes the norm
__device__ float gradient_factor(const update_arg& a, float* part) {
    if (!a.parts) return a.grad_scale;
    float s = 0.f;
    for (int i = threadIdx.x; i < a.n_parts; i += 256) s += a.parts[i];
    s = wave_sum_dpp(s);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
    __syncthreads();
    const float norm = sqrtf((part[0] + part[1]) + (part[2] + part[3])) * a.grad_scale;
    if (a.norm && blockIdx.x == 0 && threadIdx.x == 0) *a.norm = norm;
    if (!(a.max_norm > 0.f)) return a.grad_scale;
    const float r = a.max_norm / (norm + 1e-6f);
    return (r > 1.f ? 1.f : r) * a.grad_scale;                      // a NaN stays one
}

struct factors {
    float coef, step, inv_second;
    bool known;
};

// One turn of a workgroup: U * 1024 elements of one tensor, a block of 256 per wave and U.  All loads are issued before anything
// is computed, on the first turn also before the partial sums of the norm are joined.
template <int BITS, int U, bool WHOLE, typename TP, typename TG, typename T>
__device__ __forceinline__ void turn(const T& q, long long start, const update_arg& a, factors& f, float* part) {
    const long long at = start + threadIdx.x * 4;
    const float keep = 1.0f - a.lr * q.wd;
    int k[U];
    f32x4 p[U], g[U], m[U], v[U];
    unsigned mc[U], vc[U];
    float ms[U], vs[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const long long i = at + u * 1024;
        k[u] = WHOLE ? 4 : (int)std::max<long long>(0, std::min<long long>(4, q.n - i));
        p[u] = ld4e<WHOLE>((const TP*)q.p + i, k[u]);
        g[u] = ld4e<WHOLE>((const TG*)q.g + i, k[u]);
        if constexpr (BITS == 8) {
            mc[u] = ld_codes<WHOLE>(q.m + i, k[u]);
            vc[u] = ld_codes<WHOLE>(q.v + i, k[u]);
            const bool in = WHOLE || i - (threadIdx.x & 63) * 4 < q.n;
            ms[u] = in ? q.ms[i / BLOCK] : 0.f;
            vs[u] = in ? q.vs[i / BLOCK] : 0.f;
        } else {
            m[u] = ld4e<WHOLE>(q.m + i, k[u]);
            v[u] = ld4e<WHOLE>(q.v + i, k[u]);
        }
    }
    if (!f.known) {
        f.known = true;
        f.step = a.scalars[0];
        f.inv_second = 1.0f / a.scalars[1];
        f.coef = gradient_factor(a, part);
    }
    f32x4 r[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const long long i = at + u * 1024;
        if constexpr (BITS == 8) {
            m[u] = from_e4m3(mc[u], ms[u]);
            v[u] = from_e4m3(vc[u], vs[u]);
            v[u] = v[u] * v[u];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float gr = g[u][j] * f.coef;
            m[u][j] = m[u][j] * a.b1 + gr * a.omb1;
            v[u][j] = v[u][j] * a.b2 + gr * gr * a.omb2;
            r[u][j] = sqrtf(v[u][j]);
            // the quotient by the hardware's reciprocal (off by one unit in the last place): a few 2^-24 of a step that
            // is itself a small part of p; two full divisions cost a third of this kernel's instructions
            p[u][j] = p[u][j] * keep - f.step * (m[u][j] * __builtin_amdgcn_rcpf(r[u][j] * f.inv_second + a.eps));
        }
        st4e<WHOLE>((TP*)q.p + i, k[u], p[u]);
        if constexpr (BITS == 32) {
            st4e<WHOLE>(q.m + i, k[u], m[u]);
            st4e<WHOLE>(q.v + i, k[u], v[u]);
        }
    }
    if constexpr (BITS == 8) {
        const int slot = threadIdx.x & 7;
        float top = 0.f;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if constexpr (!WHOLE) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (j >= k[u]) m[u][j] = r[u][j] = 0.f;         // behind the end: no part of the block
            }
            const float tm = wave_amax(m[u]), tr = wave_amax(r[u]);
            if (slot == 2 * u) top = tm;
            if (slot == 2 * u + 1) top = tr;
        }
        const float scales = block_scales(top);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const float fr = of_lane(scales, 2 * u + 1);
            f32x4 z;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                z[j] = r[u][j] * fr;
                if (r[u][j] > 0.f && z[j] < 0x1p-9f) z[j] = 0x1p-9f;
            }
            st_codes<WHOLE>(q.m + at + u * 1024, k[u], to_e4m3(m[u] * of_lane(scales, 2 * u)));
            st_codes<WHOLE>(q.v + at + u * 1024, k[u], to_e4m3(z));
        }
        // lanes 8 .. 8 + 2 U - 1 hold the scales
        const int lane = threadIdx.x & 63, own = lane - 8, u = own >> 1;
        const long long first = start + (threadIdx.x - lane) * 4 + u * 1024;          // first element of this lane's block
        if (own >= 0 && own < 2 * U && (WHOLE || first < q.n)) (own & 1 ? q.vs : q.ms)[first / BLOCK] = scales;
    }
}

// The norm kernel walks the tensors from the last element to the first, the update from the first: what the norm kernel read
// last is still in the memory-side cache when the update begins with it.
template <int BITS, int U, typename B>
__global__ __launch_bounds__(256) void adamw_update_kernel(B b, update_arg a) {
    __shared__ float part[4];
    factors f;
    f.known = false;
    int chunk = blockIdx.x;
    for (int t = tensor_of(b, chunk); chunk < b.first[b.count]; chunk += gridDim.x) {
        while (chunk >= b.first[t + 1]) ++t;
        const auto& q = b.t[t];
        const long long start = (long long)(chunk - b.first[t]) * (U * 1024);
#define TURN(TP, TG)                                                                                      \
    do {                                                                                                  \
        if (start + U * 1024 <= q.n) turn<BITS, U, true, TP, TG>(q, start, a, f, part);                   \
        else turn<BITS, U, false, TP, TG>(q, start, a, f, part);                                          \
    } while (0)
        switch (q.kinds) {
            case 0: TURN(float, float); break;
            case 1: TURN(bf16_t, float); break;
            case 2: TURN(float, bf16_t); break;
            default: TURN(bf16_t, bf16_t); break;
        }
#undef TURN
    }
}

inline bool at_bytes(const void* p, int size) { return ((uintptr_t)p & (size - 1)) == 0; }
inline int max_blocks() { return 4 * cu_count(); }
// Workgroups per CU of the update: four, but where the data are much, as few as keep the memory busy: fewer streams suit it better.
// 32-bit states, four and one: 5 M elements 26.6 and 27.1 us, 10 M 53.3 and 52.1, 30 M 157 and 146, two and one: 120 M 633 and 601.
// 8-bit states, whose codes cost instructions: 60 M four 183, two with half the elements each 181; 470 M two 1442, two with half
// 1339, one 1675.
inline bool much8(long long elements) { return elements > (1ll << 26); }
inline int update_blocks(int bits, long long elements) {
    return (bits == 32 ? elements > (1ll << 23) ? 1 : 4 : much8(elements) ? 2 : 4) * cu_count();
}

void set_tensor(tensor32& t, const stdiff_adamw_tensor& s) {
    t.p = s.param; t.g = s.grad; t.m = (float*)s.exp_avg; t.v = (float*)s.exp_avg_sq; t.n = s.n; t.wd = s.weight_decay;
    t.kinds = (s.param_dtype == STDIFF_BF16 ? 1 : 0) | (s.grad_dtype == STDIFF_BF16 ? 2 : 0);
}
void set_tensor(tensor8& t, const stdiff_adamw_tensor& s) {
    t.p = s.param; t.g = s.grad; t.m = (unsigned char*)s.exp_avg; t.v = (unsigned char*)s.exp_avg_sq; t.n = s.n; t.wd = s.weight_decay;
    t.ms = s.exp_avg_scale; t.vs = s.exp_avg_sq_scale;
    t.kinds = (s.param_dtype == STDIFF_BF16 ? 1 : 0) | (s.grad_dtype == STDIFF_BF16 ? 2 : 0);
}
void set_tensor(gradient& t, const stdiff_adamw_tensor& s) {
    t.g = s.grad;
    t.n = s.grad_dtype == STDIFF_BF16 ? ~s.n : s.n;
}

// Fills a table with the tensors from *at on, without the empty ones, and moves *at behind the last one that found room.
template <typename T, int N> int fill(const stdiff_adamw_multi_args* a, int* at, int chunk, batch<T, N>* b) {
    b->count = 0;
    b->first[0] = 0;
    for (; *at < a->n_tensors && b->count < N; ++*at) {
        const stdiff_adamw_tensor& s = a->tensors[*at];
        if (s.n == 0) continue;
        set_tensor(b->t[b->count], s);
        b->first[b->count + 1] = b->first[b->count] + (int)((s.n + chunk - 1) / chunk);
        ++b->count;
    }
    return b->first[b->count];
}

template <int BITS, int U, typename B> int update(const stdiff_adamw_multi_args* a, const update_arg& u, long long total, hipStream_t st) {
    B b;
    for (int at = 0; at < a->n_tensors;) {
        const int chunks = fill(a, &at, U * 1024, &b);
        if (!chunks) continue;
        hipLaunchKernelGGL((adamw_update_kernel<BITS, U, B>), dim3(std::min(chunks, update_blocks(BITS, total))), dim3(256), 0, st, b, u);
        STDIFF_LAUNCH_STATUS();
    }
    return STDIFF_OK;
}

int check_multi(const stdiff_adamw_multi_args* a) {
    STDIFF_CHECK_ARG(a && a->n_tensors >= 0 && (a->tensors || a->n_tensors == 0) && (a->state_bits == 8 || a->state_bits == 32));
    STDIFF_CHECK_ARG(a->step_dev && a->workspace && a->beta1 >= 0.0 && a->beta1 < 1.0 && a->beta2 >= 0.0 && a->beta2 < 1.0 &&
                     a->eps >= 0.0 && a->lr >= 0.0 && a->max_norm == a->max_norm);
    long long chunks = 0;
    for (int i = 0; i < a->n_tensors; ++i) {
        const stdiff_adamw_tensor& s = a->tensors[i];
        STDIFF_CHECK_ARG(s.n >= 0 && (s.param_dtype == STDIFF_F32 || s.param_dtype == STDIFF_BF16) &&
                         (s.grad_dtype == STDIFF_F32 || s.grad_dtype == STDIFF_BF16) && s.weight_decay >= 0.f);
        if (s.n == 0) continue;
        STDIFF_CHECK_ARG(s.param && s.grad && s.exp_avg && s.exp_avg_sq);
        STDIFF_CHECK_ARG(a->state_bits == 32 || (s.exp_avg_scale && s.exp_avg_sq_scale));
        if (!at_bytes(s.param, (int)dtype_size(s.param_dtype)) || !at_bytes(s.grad, (int)dtype_size(s.grad_dtype)) ||
            (a->state_bits == 32 && (!at_bytes(s.exp_avg, 4) || !at_bytes(s.exp_avg_sq, 4))) ||
            (a->state_bits == 8 && (!at_bytes(s.exp_avg_scale, 4) || !at_bytes(s.exp_avg_sq_scale, 4))))
            return STDIFF_ERR_ALIGN;
        chunks += s.n / 1024 + 1;
        if (s.n > (1ll << 40) || chunks > (1ll << 30)) return STDIFF_ERR_SHAPE;      // chunks are counted in 32 bits
    }
    if (!at_bytes(a->step_dev, 4) || !at_bytes(a->workspace, 4) || !at_bytes(a->norm, 4)) return STDIFF_ERR_ALIGN;
    if (a->workspace_bytes < stdiff_adamw_multi_workspace(a->n_tensors)) return STDIFF_ERR_WORKSPACE;
    return STDIFF_OK;
}

}  // namespace

extern "C" long long stdiff_adamw_multi_workspace(int n_tensors) {
    if (n_tensors < 0) return STDIFF_ERR_ARG;
    return (SCALARS + (long long)cdiv(n_tensors, GRADIENTS) * max_blocks()) * 4;
}

extern "C" int stdiff_adamw_multi(const stdiff_adamw_multi_args* a, void* stream) {
    int rc = check_multi(a);
    if (rc != STDIFF_OK) return rc;
    hipStream_t st = (hipStream_t)stream;
    update_arg u = {};
    u.scalars = a->workspace;
    u.norm = a->norm;
    u.max_norm = a->max_norm > 0.0 ? std::max((float)a->max_norm, FLT_MIN) : 0.f;     // what is positive stays it
    u.grad_scale = (float)a->grad_scale; u.lr = (float)a->lr;
    u.b1 = (float)a->beta1; u.b2 = (float)a->beta2; u.eps = (float)a->eps;
    u.omb1 = (float)(1.0 - a->beta1);                               // rounded once: 1 - 0.9f is not 0.1f
    u.omb2 = (float)(1.0 - a->beta2);
    bool counted = false;
    if (a->max_norm > 0.0 || a->norm) {
        float* parts = a->workspace + SCALARS;
        batchg b;
        for (int at = 0; at < a->n_tensors;) {
            const int chunks = fill(a, &at, NORM_CHUNK, &b);
            if (!chunks) continue;
            const int grid = std::min(chunks, max_blocks());
            hipLaunchKernelGGL(adamw_norm_kernel, dim3(grid), dim3(256), 0, st, b, parts + u.n_parts, counted ? nullptr : a->step_dev,
                               a->workspace, a->lr, a->beta1, a->beta2);
            STDIFF_LAUNCH_STATUS();
            u.n_parts += grid;
            counted = true;
        }
        u.parts = parts;
    }
    if (!counted) {
        hipLaunchKernelGGL(adamw_prepare_kernel, dim3(1), dim3(64), 0, st, a->step_dev, a->workspace, a->norm, a->lr, a->beta1, a->beta2);
        STDIFF_LAUNCH_STATUS();
    }
    long long total = 0;
    for (int i = 0; i < a->n_tensors; ++i) total += a->tensors[i].n;
    // turns of 1024 elements instead of 4096 spread little work over all CUs (32 tensors of 1000: 8.7 against 11.5 us, of 20000: 9.4
    // and 10.7; 8 of 200000: 13.1 and 12.5, with 8-bit states 12.3 and 13.0)
    const bool few = total < 4096ll * 2 * cu_count();
    if (a->state_bits == 8 && much8(total)) return update<8, 2, batch8>(a, u, total, st);
    if (a->state_bits == 8) return few ? update<8, 1, batch8>(a, u, total, st) : update<8, 4, batch8>(a, u, total, st);
    return few ? update<32, 1, batch32>(a, u, total, st) : update<32, 4, batch32>(a, u, total, st);
}
