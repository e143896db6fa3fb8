// Matrix product in 8-bit integers with one scale per row of either operand, and the row quantisation that makes them.
//   q[r, k] = rint(x[r, k] * (127 / max_k |x[r, k]|)),   scale[r] = max_k |x[r, k]| / 127        (a zero row: zeros, scale 0)
//   C[m, n] = sum_k A[m, k] W[n, k] * a_scale[m] * w_scale[n] + bias[n]
// The sum over k is exact: int32 holds K * 127 * 127 up to K = 133143 (and K * 128 * 128 up to 131071, the limit here).  The
// scales are applied to the finished sum in fp32, the weight's first: sum * a_scale would overflow for activations above
// 1e31 whose product with a weight is still a number.
#include "common.h"

namespace {

typedef __attribute__((ext_vector_type(4))) int i32x4;
typedef f32x4 f32x4_u __attribute__((aligned(4)));
typedef u32x4 u32x4_u __attribute__((aligned(2)));
typedef u32x2 u32x2_u __attribute__((aligned(2)));

// ---------------------------------------------------------------- row quantisation
__device__ __forceinline__ unsigned abs_bits(float v) { return __builtin_bit_cast(unsigned, v) & 0x7fffffffu; }

__device__ __forceinline__ void ld8(const float* p, int k, float* o) {
    if (k >= 8) {
        const f32x4 a = *(const f32x4_u*)p, b = *(const f32x4_u*)(p + 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) { o[j] = a[j]; o[4 + j] = b[j]; }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = j < k ? p[j] : 0.f;
    }
}
__device__ __forceinline__ void ld8(const bf16_t* p, int k, float* o) {
    if (k >= 8) {
        const u32x4 v = *(const u32x4_u*)p;
#pragma unroll
        for (int j = 0; j < 4; ++j) { o[2 * j] = bf_lo(v[j]); o[2 * j + 1] = bf_hi(v[j]); }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = j < k ? bf2f(p[j]) : 0.f;
    }
}

// one workgroup of T threads per row, eight elements per thread and turn; the row is read a second time from the cache.
// The largest magnitude is found by the bits, so a NaN is above infinity and makes the scale a NaN: with a scale that is
// not finite the whole row of the product is NaN.  Columns K .. round_up(K, 16) - 1 of q become zeros.
template <typename TX>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const TX* x, long long ldx, signed char* q, long long ldq, float* scale,
                                                            int R, int K) {
    __shared__ unsigned part[2][4];
    int odd = 0;
    for (long long row = blockIdx.x; row < R; row += gridDim.x, odd ^= 1) {
        unsigned top = 0;
        for (int c = threadIdx.x * 8; c < K; c += 2048) {
            float v[8];
            ld8(x + row * ldx + c, K - c, v);
#pragma unroll
            for (int j = 0; j < 8; ++j) top = max(top, abs_bits(v[j]));
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) top = max(top, (unsigned)__shfl_xor((int)top, o, 64));
        if ((threadIdx.x & 63) == 0) part[odd][threadIdx.x >> 6] = top;
        __syncthreads();
        const float t = __builtin_bit_cast(float, max(max(part[odd][0], part[odd][1]), max(part[odd][2], part[odd][3])));
        // below 1e-30 the factor 127 / t would leave the range of fp32: such rows are scaled as if their largest were 1e-30
        const float m = t > 0.f && t < 1e-30f ? 1e-30f : t, f = m == 0.f ? 0.f : 127.0f / m;
        if (threadIdx.x == 0) scale[row] = m / 127.0f;
        for (int c = threadIdx.x * 8; c < (K + 15) / 16 * 16; c += 2048) {
            float v[8];
            ld8(x + row * ldx + c, K - c, v);
            unsigned o[2] = {0, 0};
#pragma unroll
            for (int j = 0; j < 8; ++j) o[j >> 2] |= ((unsigned)(int)rintf(v[j] * f) & 0xffu) << (8 * (j & 3));
            *(u32x2*)(q + row * ldq + c) = u32x2{o[0], o[1]};
        }
    }
}

// ---------------------------------------------------------------- product
struct Params8 {
    int M, N, K;
    const signed char* A; long long lda;
    const signed char* W; long long ldw;
    const float* a_scale; const float* w_scale; const float* bias;
    void* C; long long ldc;
};

// the bytes of a 16-byte piece that begin at k0 and lie before K (the rest as zeros): W's padding may hold anything
__device__ __forceinline__ i32x4 before_end(i32x4 v, int k0, int K) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int n = K - (k0 + 4 * j);
        v[j] = n >= 4 ? v[j] : n <= 0 ? 0 : v[j] & (int)((1u << (8 * n)) - 1u);
    }
    return v;
}

template <typename TC>
__global__ __launch_bounds__(256) void gemm_i8_kernel(Params8 p) {
    constexpr int BM = 128, BN = 128, BK = 64, LD = BK + 16;
    __shared__ __attribute__((aligned(16))) signed char As[BM * LD], Ws[BN * LD];
    const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
    const int wr = wid >> 1, wc = wid & 1, fr = lane & 15, fq = lane >> 4;
    const int m0 = blockIdx.y * BM, n0 = blockIdx.x * BN;
    i32x4 acc[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = i32x4{0, 0, 0, 0};
    for (int k0 = 0; k0 < p.K; k0 += BK) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int piece = tid + 256 * i, row = piece >> 2, k = k0 + (piece & 3) * 16;
            i32x4 a = {0, 0, 0, 0}, w = {0, 0, 0, 0};
            if (k < p.K) {
                if (m0 + row < p.M) a = before_end(*(const i32x4*)(p.A + (m0 + row) * p.lda + k), k, p.K);
                if (n0 + row < p.N) w = *(const i32x4*)(p.W + (n0 + row) * p.ldw + k);
            }
            *(i32x4*)(As + row * LD + (piece & 3) * 16) = a;
            *(i32x4*)(Ws + row * LD + (piece & 3) * 16) = w;
        }
        __syncthreads();
        i32x4 a[4], w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            a[i] = *(const i32x4*)(As + (wr * 64 + i * 16 + fr) * LD + fq * 16);
            w[i] = *(const i32x4*)(Ws + (wc * 64 + i * 16 + fr) * LD + fq * 16);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[j], a[i], acc[i][j], 0, 0, 0);
    }
    // W stands where the instruction takes its first operand: a lane holds four consecutive n of one m
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int m = m0 + wr * 64 + i * 16 + fr;
        if (m >= p.M) continue;
        const float as = p.a_scale[m];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int n = n0 + wc * 64 + j * 16 + fq * 4;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (n + e < p.N) {
                    float v = (float)acc[i][j][e] * p.w_scale[n + e] * as;
                    if (p.bias) v += p.bias[n + e];
                    Elem<TC>::st((TC*)p.C + m * p.ldc + n + e, v);
                }
        }
    }
}

}  // namespace

extern "C" int stdiff_quantize_rows(const void* x, long long ldx, int x_dtype, void* q, long long ldq, float* scale, int R, int K,
                                    void* stream) {
    STDIFF_CHECK_ARG(R >= 0 && K > 0 && (R == 0 || (x && q && scale)) && ldx >= 0 && (x_dtype == STDIFF_F32 || x_dtype == STDIFF_BF16));
    if (R == 0) return STDIFF_OK;
    if (K > (1 << 30)) return STDIFF_ERR_SHAPE;
    STDIFF_CHECK_ARG(ldq >= (K + 15) / 16 * 16);
    if (ldq % 16 || ((uintptr_t)q & 15) || ((uintptr_t)x & (dtype_size(x_dtype) - 1)) || ((uintptr_t)scale & 3)) return STDIFF_ERR_ALIGN;
    const dim3 grid((unsigned)std::min<long long>(R, 16ll * cu_count()));
    if (x_dtype == STDIFF_BF16)
        hipLaunchKernelGGL(quantize_rows_kernel<bf16_t>, grid, dim3(256), 0, (hipStream_t)stream, (const bf16_t*)x, ldx,
                           (signed char*)q, ldq, scale, R, K);
    else
        hipLaunchKernelGGL(quantize_rows_kernel<float>, grid, dim3(256), 0, (hipStream_t)stream, (const float*)x, ldx,
                           (signed char*)q, ldq, scale, R, K);
    STDIFF_LAUNCH_STATUS();
    return STDIFF_OK;
}

extern "C" int stdiff_gemm_i8(const stdiff_gemm_i8_args* a, void* stream) {
    STDIFF_CHECK_ARG(a && a->M >= 0 && a->N >= 0 && a->K > 0 && (a->c_dtype == STDIFF_F32 || a->c_dtype == STDIFF_BF16));
    if (a->M == 0 || a->N == 0) return STDIFF_OK;
    STDIFF_CHECK_ARG(a->A && a->W && a->a_scale && a->w_scale && a->C && a->ldc >= a->N);
    if (a->K > 131071) return STDIFF_ERR_SHAPE;
    const long long kp = (a->K + 15) / 16 * 16;
    STDIFF_CHECK_ARG(a->lda >= kp && a->ldw >= kp);
    if (a->lda > (1 << 23) || a->ldw > (1 << 23)) return STDIFF_ERR_SHAPE;
    if (a->lda % 16 || a->ldw % 16 || ((uintptr_t)a->A & 15) || ((uintptr_t)a->W & 15) || ((uintptr_t)a->C & (dtype_size(a->c_dtype) - 1)) ||
        ((uintptr_t)a->a_scale & 3) || ((uintptr_t)a->w_scale & 3) || ((uintptr_t)a->bias & 3))
        return STDIFF_ERR_ALIGN;
    Params8 p = {a->M, a->N, a->K, (const signed char*)a->A, a->lda, (const signed char*)a->W, a->ldw, a->a_scale, a->w_scale,
                 a->bias, a->C, a->ldc};
    const long long ty = ((long long)a->M + 127) / 128;
    if (ty > 65535) return STDIFF_ERR_SHAPE;
    const dim3 grid(cdiv(a->N, 128), (unsigned)ty);
    if (a->c_dtype == STDIFF_BF16)
        hipLaunchKernelGGL(gemm_i8_kernel<bf16_t>, grid, dim3(256), 0, (hipStream_t)stream, p);
    else
        hipLaunchKernelGGL(gemm_i8_kernel<float>, grid, dim3(256), 0, (hipStream_t)stream, p);
    STDIFF_LAUNCH_STATUS();
    return STDIFF_OK;
}
