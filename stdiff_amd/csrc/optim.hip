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
// A block that holds an infinity or a NaN gets a scale that is not finite: all its elements are NaN from the next step on.
#include "common.h"

namespace {

// the products and sums below are rounded one by one (no fused multiply-add): codes are rounded results, and whoever
// repeats the formulas operation by operation in fp32 gets the same ones
#pragma clang fp contract(off)

typedef f32x4 f32x4_u __attribute__((aligned(4)));
typedef u32x2 u32x2_u __attribute__((aligned(2)));
typedef unsigned u32_u __attribute__((aligned(1)));

constexpr int TENSORS = 48;               // per launch: the table travels in the kernel's arguments (4 KB at most)
constexpr int BLOCK = 256;                // elements that share a scale: one wave, four per lane
constexpr int CHUNK = 4096;               // elements of one turn of a workgroup: four blocks per wave
constexpr int SCALARS = 4;                // floats at the workspace's head, the partial sums of squares follow

struct tensor_arg {
    void* p;
    const void* g;
    void* m;
    void* v;
    float* ms;
    float* vs;
    long long n;
    float wd;
    int kinds;                            // bit 0: p in 16 bits, bit 1: g in 16 bits
};
struct batch_arg {
    tensor_arg t[TENSORS];
    int first[TENSORS + 1];               // first chunk of each tensor, then their number
    int count;
};

__device__ __forceinline__ void ld4e(const float* p, int k, float* o) {
    if (k >= 4) {
        const f32x4 v = *(const f32x4_u*)p;
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = v[j];
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = j < k ? p[j] : 0.f;
    }
}
__device__ __forceinline__ void ld4e(const bf16_t* p, int k, float* o) {
    if (k >= 4) {
        const u32x2 v = *(const u32x2_u*)p;
        o[0] = bf_lo(v[0]); o[1] = bf_hi(v[0]); o[2] = bf_lo(v[1]); o[3] = bf_hi(v[1]);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = j < k ? bf2f(p[j]) : 0.f;
    }
}
__device__ __forceinline__ void st4e(float* p, int k, const float* o) {
    if (k >= 4) {
        *(f32x4_u*)p = f32x4{o[0], o[1], o[2], o[3]};
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j < k) p[j] = o[j];
    }
}
__device__ __forceinline__ void st4e(bf16_t* p, int k, const float* o) {
    if (k >= 4) {
        *(u32x2_u*)p = u32x2{pack2bf(o[0], o[1]), pack2bf(o[2], o[3])};
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j < k) p[j] = f2bf(o[j]);
    }
}
__device__ __forceinline__ unsigned ld_codes(const unsigned char* p, int k) {
    if (k >= 4) return *(const u32_u*)p;
    unsigned v = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (j < k) v |= (unsigned)p[j] << (8 * j);
    return v;
}
__device__ __forceinline__ void st_codes(unsigned char* p, int k, unsigned v) {
    if (k >= 4) {
        *(u32_u*)p = v;
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j < k) p[j] = (unsigned char)(v >> (8 * j));
    }
}
__device__ __forceinline__ void from_e4m3(unsigned v, float scale, float* o) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)v, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)v, true);
    o[0] = lo[0] * scale; o[1] = lo[1] * scale; o[2] = hi[0] * scale; o[3] = hi[1] * scale;
}
__device__ __forceinline__ unsigned to_e4m3(const float* v) {
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], r, true);
}
// largest magnitude over a wave, by the bits: NaN is above infinity, infinity above every number
__device__ __forceinline__ float wave_amax(const float* v) {
    unsigned a = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) a = max(a, __builtin_bit_cast(unsigned, v[j]) & 0x7fffffffu);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) a = max(a, (unsigned)__shfl_xor((int)a, o, 64));
    return __builtin_bit_cast(float, a);
}
// scale of a block, and what its elements are multiplied by before they become codes.  Below 1e-30 the factor
// 448 / largest would leave the range of fp32: such blocks are scaled as if their largest were 1e-30.
__device__ __forceinline__ float block_scale(float top, float* factor) {
    if (top > 0.f && top < 1e-30f) top = 1e-30f;
    *factor = top == 0.f ? 0.f : 448.0f / top;
    return top / 448.0f;
}

__device__ __forceinline__ int tensor_of(const batch_arg& b, int chunk, int t) {
    while (chunk >= b.first[t + 1]) ++t;
    return t;
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
__global__ __launch_bounds__(256) void adamw_norm_kernel(batch_arg b, float* parts, int32_t* step_dev, float* scalars, double lr,
                                                         double b1, double b2) {
    if (step_dev && blockIdx.x == 0 && threadIdx.x == 0) next_step(step_dev, scalars, lr, b1, b2);
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    int t = 0;
    for (int chunk = blockIdx.x; chunk < b.first[b.count]; chunk += gridDim.x) {
        t = tensor_of(b, chunk, t);
        const long long n = b.t[t].n, at = (long long)(chunk - b.first[t]) * CHUNK + threadIdx.x * 4;
        const bool half = b.t[t].kinds & 2;
#pragma unroll
        for (int u = 0; u < CHUNK / 1024; ++u) {
            const long long i = at + u * 1024;
            if (i >= n) break;
            const int k = (int)std::min<long long>(4, n - i);
            float g[4];
            if (half) ld4e((const bf16_t*)b.t[t].g + i, k, g);
            else ld4e((const float*)b.t[t].g + i, k, g);
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[j] += g[j] * g[j];
        }
    }
    const float s = wave_sum((acc[0] + acc[1]) + (acc[2] + acc[3]));
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

template <int BITS>
__global__ __launch_bounds__(256) void adamw_update_kernel(batch_arg b, update_arg a) {
    float coef = a.grad_scale;
    if (a.parts) {
        __shared__ float part[4];
        float s = 0.f;
        for (int i = threadIdx.x; i < a.n_parts; i += 256) s += a.parts[i];
        s = wave_sum(s);
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
        __syncthreads();
        const float norm = sqrtf((part[0] + part[1]) + (part[2] + part[3])) * a.grad_scale;
        if (a.norm && blockIdx.x == 0 && threadIdx.x == 0) *a.norm = norm;
        if (a.max_norm > 0.f) {
            const float r = a.max_norm / (norm + 1e-6f);
            coef = (r > 1.f ? 1.f : r) * a.grad_scale;              // a NaN stays one
        }
    }
    const float step = a.scalars[0], second = a.scalars[1];
    int t = 0;
    for (int chunk = blockIdx.x; chunk < b.first[b.count]; chunk += gridDim.x) {
        t = tensor_of(b, chunk, t);
        const tensor_arg& q = b.t[t];
        const long long n = q.n, at = (long long)(chunk - b.first[t]) * CHUNK + threadIdx.x * 4;
        const float keep = 1.0f - a.lr * q.wd;
#pragma unroll
        for (int u = 0; u < CHUNK / 1024; ++u) {
            const long long i = at + u * 1024;
            if (i - (threadIdx.x & 63) * 4 >= n) break;             // the whole wave is behind the end
            const int k = (int)std::max<long long>(0, std::min<long long>(4, n - i));
            float p[4], g[4], m[4], v[4], r[4];
            if (q.kinds & 1) ld4e((const bf16_t*)q.p + i, k, p);
            else ld4e((const float*)q.p + i, k, p);
            if (q.kinds & 2) ld4e((const bf16_t*)q.g + i, k, g);
            else ld4e((const float*)q.g + i, k, g);
            if constexpr (BITS == 8) {
                from_e4m3(ld_codes((const unsigned char*)q.m + i, k), q.ms[i / BLOCK], m);
                from_e4m3(ld_codes((const unsigned char*)q.v + i, k), q.vs[i / BLOCK], v);
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = v[j] * v[j];
            } else {
                ld4e((const float*)q.m + i, k, m);
                ld4e((const float*)q.v + i, k, v);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float gr = g[j] * coef;
                m[j] = m[j] * a.b1 + gr * a.omb1;
                v[j] = v[j] * a.b2 + gr * gr * a.omb2;
                r[j] = sqrtf(v[j]);
                p[j] = p[j] * keep - step * (m[j] / (r[j] / second + a.eps));
            }
            if (q.kinds & 1) st4e((bf16_t*)q.p + i, k, p);
            else st4e((float*)q.p + i, k, p);
            if constexpr (BITS == 8) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (j >= k) m[j] = r[j] = 0.f;                  // behind the end: no part of the block
                float fm, fr;
                const float sm = block_scale(wave_amax(m), &fm), sr = block_scale(wave_amax(r), &fr);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    m[j] *= fm;
                    const float z = r[j] * fr;
                    r[j] = r[j] > 0.f && z < 0x1p-9f ? 0x1p-9f : z;
                }
                st_codes((unsigned char*)q.m + i, k, to_e4m3(m));
                st_codes((unsigned char*)q.v + i, k, to_e4m3(r));
                if ((threadIdx.x & 63) == 0) {
                    q.ms[i / BLOCK] = sm;
                    q.vs[i / BLOCK] = sr;
                }
            } else {
                st4e((float*)q.m + i, k, m);
                st4e((float*)q.v + i, k, v);
            }
        }
    }
}

inline bool at_bytes(const void* p, int size) { return ((uintptr_t)p & (size - 1)) == 0; }
inline int max_blocks() { return 2 * cu_count(); }

// the table of tensors [from, from + TENSORS), without the empty ones
int fill_batch(const stdiff_adamw_multi_args* a, int from, batch_arg* b) {
    b->count = 0;
    b->first[0] = 0;
    long long chunks = 0;
    for (int i = from; i < a->n_tensors && i < from + TENSORS; ++i) {
        const stdiff_adamw_tensor& s = a->tensors[i];
        if (s.n == 0) continue;
        tensor_arg& t = b->t[b->count++];
        t.p = s.param; t.g = s.grad; t.m = s.exp_avg; t.v = s.exp_avg_sq; t.ms = s.exp_avg_scale; t.vs = s.exp_avg_sq_scale;
        t.n = s.n; t.wd = s.weight_decay;
        t.kinds = (s.param_dtype == STDIFF_BF16 ? 1 : 0) | (s.grad_dtype == STDIFF_BF16 ? 2 : 0);
        chunks += (s.n + CHUNK - 1) / CHUNK;
        if (chunks > (1ll << 30)) return STDIFF_ERR_SHAPE;
        b->first[b->count] = (int)chunks;
    }
    return STDIFF_OK;
}

int check_multi(const stdiff_adamw_multi_args* a) {
    STDIFF_CHECK_ARG(a && a->n_tensors >= 0 && (a->tensors || a->n_tensors == 0) && (a->state_bits == 8 || a->state_bits == 32));
    STDIFF_CHECK_ARG(a->step_dev && a->workspace && a->beta1 >= 0.0 && a->beta1 < 1.0 && a->beta2 >= 0.0 && a->beta2 < 1.0 &&
                     a->eps >= 0.0 && a->lr >= 0.0 && a->max_norm == a->max_norm);
    for (int i = 0; i < a->n_tensors; ++i) {
        const stdiff_adamw_tensor& s = a->tensors[i];
        STDIFF_CHECK_ARG(s.n >= 0 && (s.param_dtype == STDIFF_F32 || s.param_dtype == STDIFF_BF16) &&
                         (s.grad_dtype == STDIFF_F32 || s.grad_dtype == STDIFF_BF16));
        if (s.n == 0) continue;
        STDIFF_CHECK_ARG(s.param && s.grad && s.exp_avg && s.exp_avg_sq);
        STDIFF_CHECK_ARG(a->state_bits == 32 || (s.exp_avg_scale && s.exp_avg_sq_scale));
        if (!at_bytes(s.param, (int)dtype_size(s.param_dtype)) || !at_bytes(s.grad, (int)dtype_size(s.grad_dtype)) ||
            (a->state_bits == 32 && (!at_bytes(s.exp_avg, 4) || !at_bytes(s.exp_avg_sq, 4))) ||
            (a->state_bits == 8 && (!at_bytes(s.exp_avg_scale, 4) || !at_bytes(s.exp_avg_sq_scale, 4))))
            return STDIFF_ERR_ALIGN;
    }
    if (!at_bytes(a->step_dev, 4) || !at_bytes(a->workspace, 4) || !at_bytes(a->norm, 4)) return STDIFF_ERR_ALIGN;
    if (a->workspace_bytes < stdiff_adamw_multi_workspace(a->n_tensors)) return STDIFF_ERR_WORKSPACE;
    return STDIFF_OK;
}

}  // namespace

extern "C" long long stdiff_adamw_multi_workspace(int n_tensors) {
    if (n_tensors < 0) return STDIFF_ERR_ARG;
    return (SCALARS + (long long)cdiv(n_tensors, TENSORS) * max_blocks()) * 4;
}

extern "C" int stdiff_adamw_multi(const stdiff_adamw_multi_args* a, void* stream) {
    int rc = check_multi(a);
    if (rc != STDIFF_OK) return rc;
    hipStream_t st = (hipStream_t)stream;
    batch_arg b;
    for (int from = 0; from < a->n_tensors; from += TENSORS)       // before the first launch: nothing is half done
        if ((rc = fill_batch(a, from, &b)) != STDIFF_OK) return rc;
    update_arg u = {};
    u.scalars = a->workspace;
    u.norm = a->norm;
    u.max_norm = (float)a->max_norm; u.grad_scale = (float)a->grad_scale; u.lr = (float)a->lr;
    u.b1 = (float)a->beta1; u.b2 = (float)a->beta2; u.eps = (float)a->eps;
    u.omb1 = (float)(1.0 - a->beta1);                               // rounded once: 1 - 0.9f is not 0.1f
    u.omb2 = (float)(1.0 - a->beta2);
    bool counted = false;
    if (a->max_norm > 0.0 || a->norm) {
        float* parts = a->workspace + SCALARS;
        for (int from = 0; from < a->n_tensors; from += TENSORS) {
            fill_batch(a, from, &b);
            if (b.first[b.count] == 0) continue;
            const int grid = std::min(b.first[b.count], max_blocks());
            hipLaunchKernelGGL(adamw_norm_kernel, dim3(grid), dim3(256), 0, st, b, parts + u.n_parts, counted ? nullptr : a->step_dev,
                               a->workspace, a->lr, a->beta1, a->beta2);
            STDIFF_LAUNCH_STATUS();
            u.n_parts += grid;
            counted = true;
        }
        u.parts = parts;
    }
    if (!counted) {
        hipLaunchKernelGGL(adamw_prepare_kernel, dim3(1), dim3(64), 0, st, a->step_dev, a->workspace, a->norm, a->lr,
                           a->beta1, a->beta2);
        STDIFF_LAUNCH_STATUS();
    }
    for (int from = 0; from < a->n_tensors; from += TENSORS) {
        fill_batch(a, from, &b);
        if (b.first[b.count] == 0) continue;
        const int grid = std::min(b.first[b.count], max_blocks());
        if (a->state_bits == 8)
            hipLaunchKernelGGL(adamw_update_kernel<8>, dim3(grid), dim3(256), 0, st, b, u);
        else
            hipLaunchKernelGGL(adamw_update_kernel<32>, dim3(grid), dim3(256), 0, st, b, u);
        STDIFF_LAUNCH_STATUS();
    }
    return STDIFF_OK;
}
