// Matrix product in 8-bit integers with one scale per row of either operand, and the row quantisation that makes them.
//   q[r, k] = rint(x[r, k] * (127 / max_k |x[r, k]|)),   scale[r] = max_k |x[r, k]| / 127        (a zero row: zeros, scale 0)
//   C[m, n] = sum_k A[m, k] W[n, k] * a_scale[m] * w_scale[n] + bias[n]
// The sum over k is exact: int32 holds K * 127 * 127 up to K = 133143 (and K * 128 * 128 up to 131071, the limit here).  The
// scales are applied to the finished sum in fp32, the weight's first: sum * a_scale would overflow for activations above
// 1e31 whose product with a weight is still a number.
// Measured: quantisation of 65536 x 2048 bf16 71 us (5.6 TB/s), of 4 rows 2.1 us; product
// of 4 x 4096 x 1024 3.7 us (a launch, one trip to memory and one barrier), of 65536 x 8192 x 2048 865 to 950 us (2.3 to 2.5 POP/s, by
// what clock the card holds that day; 8192 x 8192 x 8192 up to 2.97): the matrix units are busy 69 % of the cycles, and the clock
// falls to 1.9 GHz and below.
#include "common.h"

namespace {

typedef __attribute__((ext_vector_type(4))) int i32x4;
typedef f32x4 f32x4_u __attribute__((aligned(4)));
typedef u32x4 u32x4_u __attribute__((aligned(2)));
typedef u32x2 u32x2_u __attribute__((aligned(2)));

// ---------------------------------------------------------------- row quantisation
__device__ __forceinline__ unsigned abs_bits(float v) { return __builtin_bit_cast(unsigned, v) & 0x7fffffffu; }

// NT: past the caches
template <bool NT = false> __device__ __forceinline__ void ld8(const float* p, int k, float* o) {
    if (k >= 8) {
        const f32x4 a = NT ? __builtin_nontemporal_load((const f32x4_u*)p) : *(const f32x4_u*)p;
        const f32x4 b = NT ? __builtin_nontemporal_load((const f32x4_u*)(p + 4)) : *(const f32x4_u*)(p + 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) { o[j] = a[j]; o[4 + j] = b[j]; }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = j < k ? p[j] : 0.f;
    }
}
template <bool NT = false> __device__ __forceinline__ void ld8(const bf16_t* p, int k, float* o) {
    if (k >= 8) {
        const u32x4 v = NT ? __builtin_nontemporal_load((const u32x4_u*)p) : *(const u32x4_u*)p;
#pragma unroll
        for (int j = 0; j < 4; ++j) { o[2 * j] = bf_lo(v[j]); o[2 * j + 1] = bf_hi(v[j]); }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = j < k ? bf2f(p[j]) : 0.f;
    }
}

// The largest magnitude is found by the bits, so a NaN is above infinity and makes the scale a NaN: with a scale that is not
// finite the whole row of the product is NaN.  Columns K .. round_up(K, 16) - 1 of q become zeros.
__device__ __forceinline__ float row_factor(unsigned top_bits, float* scale) {
    const float t = __builtin_bit_cast(float, top_bits);
    // below 3.8e-37 the factor 127 / t would leave the range of fp32: such rows are scaled as if their largest were 4e-37
    const float m = t > 0.f && t < 4e-37f ? 4e-37f : t;
    *scale = m / 127.0f;
    return m == 0.f ? 0.f : 127.0f / m;
}
__device__ __forceinline__ u32x2 to_i8(const float* v, float f) {
    unsigned o[2] = {0, 0};
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j >> 2] |= ((unsigned)(int)rintf(v[j] * f) & 0xffu) << (8 * (j & 3));
    return u32x2{o[0], o[1]};
}
template <int T> __device__ __forceinline__ unsigned row_max(unsigned top, unsigned* part) {
    top = lanes_umax_dpp<T < 64 ? T : 64>(top);
    if constexpr (T > 64) {
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < T / 64; ++i) top = max(top, part[i]);
    }
    return top;
}

// a row stays in the registers of T lanes, eight elements per lane and vector
template <typename TX, int NV, int T, bool NT>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const TX* x, long long ldx, signed char* q, long long ldq, float* scale,
                                                            int R, int K) {
    __shared__ unsigned part[2][4];
    const int t = threadIdx.x % T, kp = (K + 15) / 16 * 16;
    int odd = 0;
    for (long long row = (long long)blockIdx.x * (256 / T) + threadIdx.x / T; row < R; row += (long long)gridDim.x * (256 / T), odd ^= 1) {
        float v[NV][8], s;
        unsigned top = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i) ld8<NT>(x + row * ldx + (i * T + t) * 8, K - (i * T + t) * 8, v[i]);
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) top = max(top, abs_bits(v[i][j]));
        const float f = row_factor(row_max<T>(top, part[odd]), &s);
        if (t == 0) scale[row] = s;
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if ((i * T + t) * 8 < kp) *(u32x2*)(q + row * ldq + (i * T + t) * 8) = to_i8(v[i], f);
    }
}

// rows too long for the registers are read a second time, from the cache
template <typename TX>
__global__ __launch_bounds__(256) void quantize_rows_long_kernel(const TX* x, long long ldx, signed char* q, long long ldq, float* scale,
                                                                 int R, int K) {
    __shared__ unsigned part[2][4];
    int odd = 0;
    for (long long row = blockIdx.x; row < R; row += gridDim.x, odd ^= 1) {
        unsigned top = 0;
        float v[8], s;
        for (int c = threadIdx.x * 8; c < K; c += 2048) {
            ld8(x + row * ldx + c, K - c, v);
#pragma unroll
            for (int j = 0; j < 8; ++j) top = max(top, abs_bits(v[j]));
        }
        const float f = row_factor(row_max<256>(top, part[odd]), &s);
        if (threadIdx.x == 0) scale[row] = s;
        for (int c = threadIdx.x * 8; c < (K + 15) / 16 * 16; c += 2048) {
            ld8(x + row * ldx + c, K - c, v);
            *(u32x2*)(q + row * ldq + c) = to_i8(v, f);
        }
    }
}

template <typename TX>
int launch_quantize(const void* x, long long ldx, void* q, long long ldq, float* scale, int R, int K, hipStream_t st) {
    // 16-bit rows that are larger than the memory-side cache (256 MB) go past the caches (65536 x 4096 bf16: 126 us, through them 148;
    // 200000 x 300, which it holds: 72 and 50; fp32 rows are read in two pieces per lane, 65536 x 1024: 64 and 59)
    const bool streams = sizeof(TX) == 2 && (long long)R * K * 3 > (256ll << 20);
#define QR_AT(NV, T, NT)                                                                                                       \
    hipLaunchKernelGGL((quantize_rows_kernel<TX, NV, T, NT>), dim3((unsigned)std::min<long long>((R + 256 / T - 1ll) / (256 / T), 8ll * cu_count())), \
                       dim3(256), 0, st, (const TX*)x, ldx, (signed char*)q, ldq, scale, R, K)
#define QR(NV, T)                                                              \
    do {                                                                       \
        if (streams) QR_AT(NV, T, sizeof(TX) == 2);                            \
        else QR_AT(NV, T, false);                                              \
    } while (0)
    // 8, 32 or 64 lanes per row up to 1024 columns (400000 x 128 bf16: 8 lanes 25 us, a wave 74; 200000 x 300: 32 lanes 36, a wave
    // 50), then the workgroup (65536 x 1024 bf16: a wave 31.7 us, the workgroup the same, but 4
    // rows 2.4 and 2.9; 65536 x 2048: 80 and 76, 4 rows 3.0 and 2.4)
    if (K <= 128) QR(2, 8);
    else if (K <= 512) QR(2, 32);
    else if (K <= 1024) QR(2, 64);
    else if (K <= 2048) QR(1, 256);
    else if (K <= 4096) QR(2, 256);
    else if (K <= 8192) QR(4, 256);
    else
        hipLaunchKernelGGL(quantize_rows_long_kernel<TX>, dim3((unsigned)std::min<long long>(R, 8ll * cu_count())), dim3(256), 0, st,
                           (const TX*)x, ldx, (signed char*)q, ldq, scale, R, K);
#undef QR
#undef QR_AT
    STDIFF_LAUNCH_STATUS();
    return STDIFF_OK;
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

#define VMCNT(n) asm volatile("s_waitcnt vmcnt(" #n ")" ::: "memory")
#define LGKMCNT0() asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory")
#define BARRIER()                      \
    do {                               \
        __builtin_amdgcn_s_barrier();  \
        asm volatile("" ::: "memory"); \
    } while (0)

constexpr int SLAB = 128;                  // bytes of K that are staged at once: one row of a tile image, eight 16-byte pieces
constexpr unsigned OUTSIDE = 0x80000000u;  // an offset behind every descriptor's range: the load gives zeros

// Rows [first, first + count) of an operand as a buffer whose range ends with the last valid row's last piece: rows behind
// the matrix read as zeros.  The base moves with the tile, so offsets stay below 2^31 whatever the matrix's size.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_of(const signed char* base, long long ld, int first, int count, int rows, int K) {
    const int n = min(count, rows - first);
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<signed char*>(base + first * ld), 0,
                                             n > 0 ? (int)((n - 1) * ld) + (K + 15) / 16 * 16 : 0, 0x00020000);
}
__device__ __forceinline__ void load_lds(__amdgpu_buffer_rsrc_t r, unsigned char* dst, unsigned offset) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)dst, 16, offset, 0, 0, 0);
}
// columns n .. n + 3 of a vector of N
__device__ __forceinline__ f32x4 four(const float* v, int n, int N) {
    if (n + 4 <= N) return *(const f32x4_u*)(v + n);
    f32x4 o;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = n + e < N ? v[n + e] : 0.f;
    return o;
}
__device__ __forceinline__ f32x4 scaled(i32x4 sum, float as, f32x4 ws, f32x4 b) {
    f32x4 o;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = (float)sum[e] * ws[e] * as + b[e];
    return o;
}
__device__ __forceinline__ void put1(float* p, float v) { *p = v; }
__device__ __forceinline__ void put1(bf16_t* p, float v) { *p = to_h16(v); }
__device__ __forceinline__ void put4(float* p, f32x4 v) { *(f32x4*)p = v; }
__device__ __forceinline__ void put4(bf16_t* p, f32x4 v) { *(u32x2*)p = u32x2{to_2h16(v[0], v[1]), to_2h16(v[2], v[3])}; }
// 16 bytes of a row of C, which may begin at any element and end inside the piece
template <typename TC> __device__ __forceinline__ void store16(TC* row, int n, int N, u32x4 v) {
    constexpr int E = 16 / sizeof(TC);
    if (n + E <= N) {
        if constexpr (sizeof(TC) == 4) {
            *(f32x4_u*)(row + n) = __builtin_bit_cast(f32x4, v);
        } else {
            *(u32x4_u*)(row + n) = v;
        }
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (n + e < N) {
                if constexpr (sizeof(TC) == 4) ((unsigned*)row)[n + e] = v[e];
                else ((bf16_t*)row)[n + e] = (bf16_t)(v[e >> 1] >> (16 * (e & 1)));
            }
    }
}
// Tile of workgroup i.  Workgroups i and i + 8 share an XCD's L2: each XCD gets a contiguous range of tiles, in groups of four rows
// of tiles (16384 x 6144 x 2048: two 170, four 168, eight 176 us; 8192 x 8192 x 8192: 390, 380 and 380; 131072 x 4096 x 1024: 530, 530 and 523).
__device__ __forceinline__ void tile_at(int i, int tiles_m, int tiles_n, int* tm, int* tn) {
    constexpr int HIGH = 4;
    const int n = tiles_m * tiles_n, q = n >> 3, r = n & 7, x = i & 7;
    const int at = (x < r ? x * (q + 1) : r * (q + 1) + (x - r) * q) + (i >> 3);
    const int group = at / (HIGH * tiles_n), in = at - group * HIGH * tiles_n, high = min(tiles_m - group * HIGH, HIGH);
    *tm = group * HIGH + in % high;
    *tn = in / high;
}

// ---- small outputs: bound by one trip to memory, so all loads of a wave are issued at once.  A workgroup owns 16 columns of 16 * MT rows, its eight waves a share of K each, straight from memory into the
// instruction's operands (a lane holds 16 consecutive bytes of one row); the eight sums meet in LDS.
template <int MT, typename TC>
__global__ __launch_bounds__(512) void gemm_i8_rows_kernel(Params8 p) {
    __shared__ i32x4 sums[8][MT][64];
    const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), fr = lane & 15, fq = lane >> 4;
    const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 16 * MT;
    i32x4 acc[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[i] = i32x4{0, 0, 0, 0};
    const signed char* w = p.W + (long long)min(n0 + fr, p.N - 1) * p.ldw;
    const signed char* a[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) a[i] = p.A + (long long)min(m0 + i * 16 + fr, p.M - 1) * p.lda;    // rows behind the end repeat the last
    constexpr int U = MT < 4 ? 4 : 2;      // turns whose loads are in flight together
    for (int k0 = wid * 64; k0 < p.K; k0 += U * 512) {
        i32x4 wv[U], av[U][MT];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = k0 + u * 512 + fq * 16;
            const bool in = k < p.K;
            wv[u] = in ? *(const i32x4*)(w + k) : i32x4{0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < MT; ++i) av[u][i] = in ? *(const i32x4*)(a[i] + k) : i32x4{0, 0, 0, 0};
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < MT; ++i)
                acc[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wv[u], before_end(av[u][i], k0 + u * 512 + fq * 16, p.K), acc[i], 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) sums[wid][i][lane] = acc[i];
    __syncthreads();
    if (wid >= MT) return;
    i32x4 s = sums[0][wid][lane];
#pragma unroll
    for (int j = 1; j < 8; ++j) s += sums[j][wid][lane];
    const int m = m0 + wid * 16 + fr, n = n0 + fq * 4;
    if (m >= p.M || n >= p.N) return;
    const f32x4 v = scaled(s, p.a_scale[m], four(p.w_scale, n, p.N), p.bias ? four(p.bias, n, p.N) : f32x4{0.f, 0.f, 0.f, 0.f});
    TC* row = (TC*)p.C + m * p.ldc;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (n + e < p.N) put1(row + n + e, v[e]);
}

// ---- BM x BN tiles, one per workgroup of NW waves: both operands by LDS-DMA into a ring of four slabs, three ahead, one barrier
// per slab.  An image row is 128 bytes; its piece c lies in slot c ^ (row & 7) (the swizzle is on the source's side, the
// DMA writes in lane order), so the 16 rows of a fragment read fall on different banks.
template <int BM, int BN, int NW, typename TC>
__global__ __launch_bounds__(NW * 64) void gemm_i8_tile_kernel(Params8 p, int tiles_m, int tiles_n) {
    constexpr int STAGES = 4, STAGE = (BM + BN) * SLAB, WAVES_N = NW / 2, MT = BM / 2 / 16, NT = BN / WAVES_N / 16;
    constexpr int DA = BM / 8 / NW, DB = BN / 8 / NW;                   // DMA instructions per wave: eight rows each
    constexpr int ROW = BN * (int)sizeof(TC) + 16;                      // row of the C image
    static_assert(DA + DB == 4, "the counted waits below");
    static_assert(STAGES * STAGE >= BM * ROW, "the C image takes the ring's place");
    __shared__ __attribute__((aligned(16))) unsigned char smem[STAGES * STAGE];
    const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wid / WAVES_N, wn = wid % WAVES_N, fr = lane & 15, fq = lane >> 4;
    int tm, tn;
    tile_at(blockIdx.x, tiles_m, tiles_n, &tm, &tn);
    const int m0 = tm * BM, n0 = tn * BN, nk = (p.K + SLAB - 1) / SLAB;
    const __amdgpu_buffer_rsrc_t ra = rows_of(p.A, p.lda, m0, BM, p.M, p.K), rw = rows_of(p.W, p.ldw, n0, BN, p.N, p.K);
    const int piece = ((lane & 7) ^ (lane >> 3)) * 16;
    auto stage = [&](int slab) {
        unsigned char* dst = smem + (slab & (STAGES - 1)) * STAGE;
        const int k = slab * SLAB + piece;
#pragma unroll
        for (int j = 0; j < DA; ++j) {
            const int r = (DA * wid + j) * 8;
            load_lds(ra, dst + r * SLAB, k < p.K ? (unsigned)((r + (lane >> 3)) * (int)p.lda + k) : OUTSIDE);
        }
#pragma unroll
        for (int j = 0; j < DB; ++j) {
            const int r = (DB * wid + j) * 8;
            load_lds(rw, dst + (BM + r) * SLAB, k < p.K ? (unsigned)((r + (lane >> 3)) * (int)p.ldw + k) : OUTSIDE);
        }
    };
    i32x4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = i32x4{0, 0, 0, 0};
#pragma unroll
    for (int d = 0; d < STAGES - 1; ++d)
        if (d < nk) stage(d);
#pragma unroll 1
    for (int t = 0; t < nk; ++t) {
        const int rem = min(STAGES - 2, nk - 1 - t);                    // slabs behind this one that may still be in flight
        if (rem == 2) VMCNT(8);                                         // four instructions each
        else if (rem == 1) VMCNT(4);
        else VMCNT(0);
        BARRIER();                                                      // slab t is here; every wave is done with slab t - 1
        if (t + STAGES - 1 < nk) stage(t + STAGES - 1);
        const unsigned char* img = smem + (t & (STAGES - 1)) * STAGE;
        i32x4 a[2][MT], w[2][NT];
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            const int slot = ((ks * 4 + fq) ^ (fr & 7)) * 16;
#pragma unroll
            for (int i = 0; i < MT; ++i) a[ks][i] = *(const i32x4*)(img + (wm * (BM / 2) + i * 16 + fr) * SLAB + slot);
#pragma unroll
            for (int j = 0; j < NT; ++j) w[ks][j] = *(const i32x4*)(img + (BM + wn * (BN / WAVES_N) + j * 16 + fr) * SLAB + slot);
        }
        if (t == nk - 1 && (p.K & 15)) {
#pragma unroll
            for (int ks = 0; ks < 2; ++ks)
#pragma unroll
                for (int i = 0; i < MT; ++i) a[ks][i] = before_end(a[ks][i], t * SLAB + ks * 64 + fq * 16, p.K);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[ks][j], a[ks][i], acc[i][j], 0, 0, 0);
    }
    BARRIER();                                                          // the last slab has been read
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        const int n = wn * (BN / WAVES_N) + j * 16 + fq * 4;
        const f32x4 ws = four(p.w_scale, n0 + n, p.N), b = p.bias ? four(p.bias, n0 + n, p.N) : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            const int m = wm * (BM / 2) + i * 16 + fr;
            put4((TC*)(smem + m * ROW) + n, scaled(acc[i][j], p.a_scale[min(m0 + m, p.M - 1)], ws, b));
        }
    }
    __syncthreads();
    constexpr int PIECES = BN * (int)sizeof(TC) / 16;
#pragma unroll 4
    for (int i = tid; i < BM * PIECES; i += NW * 64) {
        const int m = i / PIECES, c = i % PIECES;
        if (m0 + m < p.M) store16((TC*)p.C + (m0 + m) * p.ldc, n0 + c * (16 / (int)sizeof(TC)), p.N, *(const u32x4*)(smem + m * ROW + c * 16));
    }
}

// ---- 256 x 256 tiles, eight waves, persistent: the scheme of gemm256q_kernel (gemm.hip).  A slab is four half tiles of 128 rows
// (A0 A1 W0 W1, 16 KiB each), two buffers of them; a phase multiplies one half of A with both halves of W (32
// instructions per wave) while the halves that were read last are refilled two slabs ahead; the waits are counted, and
// waves 4-7 run one barrier behind waves 0-3, so that on every SIMD one wave multiplies while the other reads.  The
// first loads of the next tile are issued before C leaves through the buffers that they do not use.
// All of LDS is one array: with another for the scales the compiler lets every read wait for all DMA under way.
// Measured per tile: 1.36 us for a slab (the instructions alone 1.1 at the clock that they leave), 5 us for C, half of it conversions and
// scales.  The stores of C are under way during the next tile's first slab: the counted waits know how many they are.
// PAST: C goes past the caches.  TAIL: K is no multiple of 16.  (A form of its own: 229 to 233 registers without the masks, 248 to 251 with them, of 256.)
template <typename TC, bool TAIL, bool PAST>
__global__ __launch_bounds__(512, 1) void gemm_i8_256_kernel(Params8 p, int tiles_m, int tiles_n, int whole, int units) {
    constexpr int HALF = 128 * SLAB;
    constexpr int SCALES = 9 * HALF;
    __shared__ __attribute__((aligned(16))) unsigned char smem[SCALES + 6 * 1024];
    float* scales = (float*)(smem + SCALES);                            // a_scale, w_scale and bias of the tile, 256 of each; the next tile's
    const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wr = wid >> 2, wc = wid & 3, fr = lane & 15, fq = lane >> 4, nk = (p.K + SLAB - 1) / SLAB;
    const int piece = ((lane & 7) ^ (lane >> 3)) * 16;
    const unsigned va = (unsigned)((16 * wid + (lane >> 3)) * (int)p.lda + piece), vw = (unsigned)((16 * wid + (lane >> 3)) * (int)p.ldw + piece);
    __amdgpu_buffer_rsrc_t ra, rw;
    bool full = true;                      // a whole tile; else (the tail of the grid) rows m0 .. m0 + 127 only
    int m0, n0;
    float s0, s1;                          // this thread's share of the next tile's scales, on their way
    auto set_tile = [&](int unit) {
        int tm, tn, tile = unit, low = 0;
        full = unit < whole;
        if (!full) { tile = whole + ((unit - whole) >> 1); low = (unit - whole) & 1; }
        tile_at(tile, tiles_m, tiles_n, &tm, &tn);
        m0 = tm * 256 + low * 128;
        n0 = tn * 256;
        ra = rows_of(p.A, p.lda, m0, full ? 256 : 128, p.M, p.K);
        rw = rows_of(p.W, p.ldw, n0, 256, p.N, p.K);
        const int m = min(m0 + (tid & 255), p.M - 1), n = min(n0 + (tid & 255), p.N - 1);
        s0 = tid < 256 ? p.a_scale[m] : p.w_scale[n];
        s1 = p.bias ? p.bias[n] : 0.f;
    };
    auto dma = [&](int buf, int slot, int t) {                          // half tile `slot` of slab t into buffer buf
        unsigned char* dst = smem + (buf * 4 + slot) * HALF + 2 * wid * 1024;
        const bool in = t * SLAB + piece < p.K;
        unsigned at = slot < 2 ? va : vw;
        asm volatile("" : "+v"(at));       // the offsets are added up here, not kept (and spilled) across the K loop
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (slot < 2) load_lds(ra, dst + i * 1024, in ? at + (unsigned)(((slot & 1) * 128 + i * 8) * (int)p.lda + t * SLAB) : OUTSIDE);
            else load_lds(rw, dst + i * 1024, in ? at + (unsigned)(((slot & 1) * 128 + i * 8) * (int)p.ldw + t * SLAB) : OUTSIDE);
        }
    };
    auto prologue = [&]() {                                             // slab 0, and all of slab 1 but A1
        dma(0, 0, 0); dma(0, 2, 0); dma(0, 3, 0); dma(0, 1, 0);
        if (nk > 1) { dma(1, 0, 1); dma(1, 2, 1); dma(1, 3, 1); }
    };
    int oa[2], ow[2];
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
        const int slot = ((ks * 4 + fq) ^ (fr & 7)) * 16;
        oa[ks] = (wr * 64 + fr) * SLAB + slot;
        ow[ks] = (wc * 32 + fr) * SLAB + slot;
    }
    i32x4 af[4][2], wf[2][2][2], acc[2][2][4][2];
    auto load_a = [&](int buf, int mh, int t) {
        const unsigned char* b = smem + (buf * 4 + mh) * HALF;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) af[i][ks] = *(const i32x4*)(b + oa[ks] + i * 16 * SLAB);
        if (TAIL && t == nk - 1) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int ks = 0; ks < 2; ++ks) af[i][ks] = before_end(af[i][ks], t * SLAB + ks * 64 + fq * 16, p.K);
        }
    };
    auto load_w = [&](int buf, int nh) {
        const unsigned char* b = smem + (buf * 4 + 2 + nh) * HALF;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) wf[nh][j][ks] = *(const i32x4*)(b + ow[ks] + j * 16 * SLAB);
    };
#define MMA(MH, NH)                                                                                          \
    do {                                                                                                     \
        __builtin_amdgcn_s_setprio(1);                                                                       \
        _Pragma("unroll") for (int ks = 0; ks < 2; ++ks)                                                     \
        _Pragma("unroll") for (int i = 0; i < 4; ++i)                                                        \
        _Pragma("unroll") for (int j = 0; j < 2; ++j)                                                        \
            acc[MH][NH][i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[NH][j][ks], af[i][ks], acc[MH][NH][i][j], 0, 0, 0); \
        __builtin_amdgcn_s_setprio(0);                                                                       \
    } while (0)

    constexpr int STORES = sizeof(TC) == 2 ? 16 : 32;                   // of C, per wave and whole tile
    int unit = blockIdx.x, side = 0;
    bool behind = false;                                                // so many are under way when a tile begins
    set_tile(unit);
    prologue();
    scales[tid] = s0;
    if (tid >= 256) scales[256 + tid] = s1;
    while (true) {
#pragma unroll
        for (int mh = 0; mh < 2; ++mh)
#pragma unroll
            for (int nh = 0; nh < 2; ++nh)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j) acc[mh][nh][i][j] = i32x4{0, 0, 0, 0};
        if (nk == 1) VMCNT(0);                                          // slab 0 is here
        else if (!behind) VMCNT(6);
        else if (STORES == 16) VMCNT(22);
        else VMCNT(38);
        LGKMCNT0();
        BARRIER();                                                      // every wave's share too; the C image has been read
        if (wr == 1) BARRIER();
        for (int t = 0; t < nk; ++t) {
            const int b = t & 1, nb = b ^ 1;
            const bool n1 = t + 1 < nk, n2 = t + 2 < nk;
            load_w(b, 0);
            load_w(b, 1);
            __builtin_amdgcn_sched_barrier(0);
            load_a(b, 0, t);
            if (n1) {
                dma(nb, 1, t + 1);
                if (t || !behind) VMCNT(8);                             // A1(t) is here
            } else {
                VMCNT(0);
            }
            LGKMCNT0();                                                 // what was read may be overwritten behind the barrier
            BARRIER();
            MMA(0, 0);
            MMA(0, 1);
            BARRIER();
            if (full) load_a(b, 1, t);
            if (n2) {
                dma(b, 0, t + 2); dma(b, 2, t + 2); dma(b, 3, t + 2);
                if (t || !behind) VMCNT(8);                             // A0 W0 W1 (t + 1) are here
                else if (STORES == 16) VMCNT(24);
                else VMCNT(40);
            } else if (n1) {
                VMCNT(2);
            }
            LGKMCNT0();
            BARRIER();
            if (full) {
                MMA(1, 0);
                MMA(1, 1);
            }
            BARRIER();
        }
        if (wr == 0) BARRIER();                                         // all waves are past their last read of the buffers
        const int em = m0, en = n0, next = unit + (int)gridDim.x;
        const bool was_full = full;
        behind = was_full && em + 256 <= p.M && en + 256 <= p.N;
        const float* now = scales + side * 768;
        if (next < units) {
            set_tile(next);
            prologue();
        }
        // C by eighths of 32 rows (16 of each wave group) through images in the half tiles 5 (A1 of slab 1) and 8, which the
        // loads under way do not use: 16-bit eighths alternate, so one barrier each is enough, fp32 ones take both
        constexpr int ROW = 256 * (int)sizeof(TC);
        const auto image = [&](int e, int group) { return smem + ((sizeof(TC) == 2 ? e & 1 : group) ? 8 : 5) * HALF + (sizeof(TC) == 2 ? group * 16 * ROW : 0); };
        f32x4 ws[2][2], bs[2][2];
#pragma unroll
        for (int nh = 0; nh < 2; ++nh)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int n = nh * 128 + wc * 32 + j * 16 + fq * 4;
                ws[nh][j] = *(const f32x4*)&now[256 + n];
                bs[nh][j] = *(const f32x4*)&now[512 + n];
            }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (e == 4 && !was_full) break;
            if (e && sizeof(TC) == 4) BARRIER();                        // the previous eighth's image has been read
            unsigned char* put = image(e, wr) + fr * ROW;
            const float as = now[(e >> 2) * 128 + wr * 64 + (e & 3) * 16 + fr];
#pragma unroll
            for (int nh = 0; nh < 2; ++nh)
#pragma unroll
                for (int jn = 0; jn < 2; ++jn) {
                    const int c = nh * 32 + wc * 8 + jn * 4 + fq;       // group of four columns
                    const f32x4 v = scaled(acc[e >> 2][nh][e & 3][jn], as, ws[nh][jn], bs[nh][jn]);
                    if constexpr (sizeof(TC) == 2) put4((TC*)(put + ((c ^ (fr << 1)) << 3)), v);
                    else put4((TC*)(put + ((c ^ fr) << 4)), v);
                }
            LGKMCNT0();
            BARRIER();
            constexpr int PIECES = ROW / 16, EACH = 32 * PIECES / 512;
            u32x4 v[EACH];
#pragma unroll
            for (int i = 0; i < EACH; ++i) {
                const int r = (tid + 512 * i) / PIECES, c = (tid + 512 * i) % PIECES;
                const unsigned char* get = image(e, r >> 4) + (r & 15) * ROW;
                if constexpr (sizeof(TC) == 2) v[i] = *(const u32x4*)(get + (((2 * c) ^ ((r & 15) << 1)) << 3));
                else v[i] = *(const u32x4*)(get + ((c ^ (r & 15)) << 4));
            }
#pragma unroll
            for (int i = 0; i < EACH; ++i) {
                const int r = (tid + 512 * i) / PIECES, c = (tid + 512 * i) % PIECES;
                const int m = em + (e >> 2) * 128 + (r >> 4) * 64 + (e & 3) * 16 + (r & 15), n = en + c * (16 / (int)sizeof(TC));
                TC* row = (TC*)p.C + m * p.ldc;
                if (behind) {
                    if (PAST) __builtin_nontemporal_store(v[i], (u32x4_u*)(row + n));
                    else *(u32x4_u*)(row + n) = v[i];
                } else if (m < p.M) {
                    store16(row, n, p.N, v[i]);
                }
            }
            if (e == 3) {                                               // the next tile's scales are here
                float* then = scales + (side ^ 1) * 768;
                then[tid] = s0;
                if (tid >= 256) then[256 + tid] = s1;
            }
            LGKMCNT0();
        }
        if (next >= units) break;
        unit = next;
        side ^= 1;
    }
#undef MMA
}

template <typename TC> int launch_gemm_i8(const Params8& p, hipStream_t st) {
    const long long t256 = ((p.M + 255ll) / 256) * ((p.N + 255ll) / 256), t128 = ((p.M + 127ll) / 128) * ((p.N + 127ll) / 128);
    const long long t64 = ((p.M + 63ll) / 64) * ((p.N + 63ll) / 64);
    if (t256 > (1 << 28)) return STDIFF_ERR_SHAPE;
    const int cus = cu_count();
    // Small outputs: bytes of K that the busiest CU reads, a workgroup of 16 x 16 MT against a tile of 64 x 64 (the latter through
    // LDS, 1.5 times as fast a byte).  M x N x K, rows kernel and 64 tiles: 4 x 4096 x 1024 3.2 and 5.0 us, 64 x 1024 x 4096 6.1
    // and 11.9, 64 x 8192 x 4096 22.4 and 12.6.
    // Otherwise the smallest tiles that are done at once, with two of 64 or one of 128 per CU.  Tiles of 64 and 128: 512 x 4096 x 1024
    // 6.9 and 8.6 us, 1024 x 4096 x 1024 12.2 and 9.5; of 128 and 256: 2048 x 2048 x 2048 16.5 and 20.2, 2000 x 1500 x 4096 23.9
    // and 33.4, but where the CUs have a second one of 128, 1500 x 3000 x 1000 17.3 and 14.5, 2048 x 2560 x 2048 24.9 and 19.4.
    const auto busiest = [&](int mt) { return ((p.N + 15ll) / 16 * ((p.M + 16ll * mt - 1) / (16 * mt)) + cus - 1) / cus * (16 + 16 * mt) * 3 / 2; };
    const long long r1 = busiest(1), r2 = busiest(2), r4 = busiest(4), least = std::min(r1, std::min(r2, r4));
    const int kind = p.M <= 65536 && p.N <= 1 << 26 && least <= (t64 + cus - 1) / cus * 128 ? 1 : t128 > cus ? 4 : t64 > 2 * cus ? 3 : 2;
    if (kind == 1) {
        const int mt = least == r1 ? 1 : least == r2 ? 2 : 4;
        const dim3 grid(cdiv(p.N, 16), cdiv(p.M, 16 * mt));
        if (mt == 1) hipLaunchKernelGGL((gemm_i8_rows_kernel<1, TC>), grid, dim3(512), 0, st, p);
        else if (mt == 2) hipLaunchKernelGGL((gemm_i8_rows_kernel<2, TC>), grid, dim3(512), 0, st, p);
        else hipLaunchKernelGGL((gemm_i8_rows_kernel<4, TC>), grid, dim3(512), 0, st, p);
    } else if (kind == 2) {
        hipLaunchKernelGGL((gemm_i8_tile_kernel<64, 64, 4, TC>), dim3((unsigned)t64), dim3(256), 0, st, p, cdiv(p.M, 64), cdiv(p.N, 64));
    } else if (kind == 3) {
        hipLaunchKernelGGL((gemm_i8_tile_kernel<128, 128, 8, TC>), dim3((unsigned)t128), dim3(512), 0, st, p, cdiv(p.M, 128), cdiv(p.N, 128));
    } else {
        // a last round of at most half the CUs' tiles is cut into half tiles (4096 x 5120 x 2048: 49.6 us, whole ones 50.6; 8192 x
        // 4352 x 1024: 47.2 and 49.8)
        const int tail = (int)(t256 % cus);
        const int whole = tail && tail <= cus / 2 ? (int)t256 - tail : (int)t256, units = whole + 2 * ((int)t256 - whole);
        // Past the caches, but where rows begin inside cache lines and the caches hold most of C: its lines are whole before they leave
        // (us past the caches and through them: 26628 x 3464 x 128 -> fp32, 369 MB, 98 and 95, -> bf16 61 and 50; 25055 x 5127 x 449 ->
        // fp32, 514 MB, 171 and 185).  Whole lines: 131072 x 4096 x 128 -> bf16 216 and 249, 65536 x 1024 x 256 -> bf16 34 and 45, 8192 x
        // 8192 x 512 -> fp32 68 and 82, 65536 x 8192 x 2048 -> bf16 923 and 952, 2048 x 2560 x 2048 -> bf16 the same, but 8192 x 4096 x
        // 1024 -> bf16 41 and 38.  With a kernel behind that reads C (quantize_rows): 547 and 549, 79 and 83, 141 and 133, 1200 and 1263,
        // 28 and 28, 59 and 53: what the stores gain there is lost in part to reads that no cache serves, for C of 60 to 270 MB up to a tenth.
        const bool past = (((uintptr_t)p.C | (uintptr_t)(p.ldc * sizeof(TC))) & 127) == 0 || (long long)p.M * p.N * (long long)sizeof(TC) > (400ll << 20);
#define TILES(TAIL, PAST)                                                                                                      \
    hipLaunchKernelGGL((gemm_i8_256_kernel<TC, TAIL, PAST>), dim3(std::min(units, cus)), dim3(512), 0, st, p, cdiv(p.M, 256),  \
                       cdiv(p.N, 256), whole, units)
        if (p.K % 16) {
            if (past) TILES(true, true);
            else TILES(true, false);
        } else {
            if (past) TILES(false, true);
            else TILES(false, false);
        }
#undef TILES
    }
    STDIFF_LAUNCH_STATUS();
    return STDIFF_OK;
}

}  // namespace

extern "C" int stdiff_quantize_rows(const void* x, long long ldx, int x_dtype, void* q, long long ldq, float* scale, int R, int K,
                                    void* stream) {
    STDIFF_CHECK_ARG(R >= 0 && K > 0 && (R == 0 || (x && q && scale)) && ldx >= 0 && (x_dtype == STDIFF_F32 || x_dtype == STDIFF_BF16));
    if (R == 0) return STDIFF_OK;
    if (K > (1 << 30)) return STDIFF_ERR_SHAPE;
    STDIFF_CHECK_ARG(ldq >= (K + 15) / 16 * 16);
    if (ldq % 16 || ((uintptr_t)q & 15) || ((uintptr_t)x & (dtype_size(x_dtype) - 1)) || ((uintptr_t)scale & 3)) return STDIFF_ERR_ALIGN;
    return x_dtype == STDIFF_BF16 ? launch_quantize<bf16_t>(x, ldx, q, ldq, scale, R, K, (hipStream_t)stream)
                                  : launch_quantize<float>(x, ldx, q, ldq, scale, R, K, (hipStream_t)stream);
}

extern "C" int stdiff_gemm_i8(const stdiff_gemm_i8_args* a, void* stream) {
    STDIFF_CHECK_ARG(a && a->M >= 0 && a->N >= 0 && a->K > 0 && (a->c_dtype == STDIFF_F32 || a->c_dtype == STDIFF_BF16));
    if (a->M == 0 || a->N == 0) return STDIFF_OK;
    STDIFF_CHECK_ARG(a->A && a->W && a->a_scale && a->w_scale && a->C && a->ldc >= a->N);
    if (a->K > 131071 || a->M > (1 << 30) || a->N > (1 << 30)) return STDIFF_ERR_SHAPE;      // a tile behind the last row or column: still 32 bits
    const long long kp = (a->K + 15) / 16 * 16;
    STDIFF_CHECK_ARG(a->lda >= kp && a->ldw >= kp);
    if (a->lda > (1 << 23) || a->ldw > (1 << 23)) return STDIFF_ERR_SHAPE;
    if (a->lda % 16 || a->ldw % 16 || ((uintptr_t)a->A & 15) || ((uintptr_t)a->W & 15) || ((uintptr_t)a->C & (dtype_size(a->c_dtype) - 1)) ||
        ((uintptr_t)a->a_scale & 3) || ((uintptr_t)a->w_scale & 3) || ((uintptr_t)a->bias & 3))
        return STDIFF_ERR_ALIGN;
    Params8 p = {a->M, a->N, a->K, (const signed char*)a->A, a->lda, (const signed char*)a->W, a->ldw, a->a_scale, a->w_scale,
                 a->bias, a->C, a->ldc};
    return a->c_dtype == STDIFF_BF16 ? launch_gemm_i8<bf16_t>(p, (hipStream_t)stream) : launch_gemm_i8<float>(p, (hipStream_t)stream);
}
