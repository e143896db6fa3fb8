// LayerNorm over rows with a weight and a bias per column, forward and backward (the adaLN form, whose shift and scale
// differ from row to row, is ln_modulate in pointwise.hip / train.hip).
//   forward :  mu = mean x, var = mean (x - mu)^2, rstd = 1 / sqrt(var + eps), y = (x - mu) * rstd * w + b
//   backward:  xhat = (x - mu) * rstd, g = dy * w, dx = rstd * (g - mean g - xhat * mean(g * xhat)),
//              dw = sum over rows of dy * xhat, db = sum over rows of dy
// A row is read once and stays in registers, 16 elements per lane in vectors of 16 bytes of x: 8, 32 or 64 lanes share a row of
// up to 128, 512 or 1024 elements (a wave holds 8, 2 or 1 of them), longer rows have a workgroup of ceil(H / 1024) waves,
// up to 16384; beyond that (and below 8) the row is read again from the cache.  Small shares keep many rows in flight: with
// one row per wave whatever its length, rows of 64 and 300 16-bit elements ran at 1.1 and 3.9 TB/s.
// The kernels for rows beyond 16384 and below 8 are simple ones: 4096 x 20000 fp32 forward 215 us (3.1 TB/s), backward 402 (2.4), bf16 123 and
// 245; rows below 8 leave nearly all lanes idle, 1000000 x 7 fp32 1.4 ms forward and 15 ms backward (64 threads walk down all rows).
// The vector that the row's end cuts is moved left until it fits: its lane holds some of its neighbour's columns again, leaves
// them out of the sums and stores them a second time with the same bits.  (Element by element, the 7 elements at the end
// of rows of 999 cost 0.8 of the time of all others.)
// Bound by memory where there are many rows, by launch and one trip to memory where there are few: forward of one row of
// 1024 1.8 us, of 131072 x 1024 fp32 -> bf16 131 us (6.2 TB/s), backward of 32768 x 2048 fp32 135 + 6 us for the partial sums (5.7
// TB/s), of 512 x 1024 bf16 3.8 us in one launch.
// The variance is formed from the centred values (a second walk over the registers), so a row whose mean is far larger
// than its spread keeps its digits.  Statistics and sums are fp32; a thread's own sum of the rows beyond 16384, and of the columns of
// those and of rows below 8, is held in 64 bits, since its terms may be millions (one row of 2^26 columns around 3.3 with a spread
// of 0.01: the mean off by 2e-4 in fp32; the time does not change).
#include "common.h"

namespace {

typedef f32x4 f32x4_u __attribute__((aligned(4)));       // rows may begin at any element: gfx950 loads and stores of
typedef u32x4 u32x4_u __attribute__((aligned(2)));       // 16 bytes need no alignment in global memory
typedef u32x2 u32x2_u __attribute__((aligned(2)));

// NT: past the caches (for what is used once and is larger than they are)
template <int V, bool NT = false> __device__ __forceinline__ void ldv(const float* p, float* o) {
#pragma unroll
    for (int i = 0; i < V; i += 4) {
        const f32x4 v = NT ? __builtin_nontemporal_load((const f32x4_u*)(p + i)) : *(const f32x4_u*)(p + i);
#pragma unroll
        for (int j = 0; j < 4; ++j) o[i + j] = v[j];
    }
}
template <int V, bool NT = false> __device__ __forceinline__ void ldv(const bf16_t* p, float* o) {
    if constexpr (V == 8) {
        const u32x4 v = NT ? __builtin_nontemporal_load((const u32x4_u*)p) : *(const u32x4_u*)p;
#pragma unroll
        for (int j = 0; j < 4; ++j) { o[2 * j] = bf_lo(v[j]); o[2 * j + 1] = bf_hi(v[j]); }
    } else {
        const u32x2 v = NT ? __builtin_nontemporal_load((const u32x2_u*)p) : *(const u32x2_u*)p;
#pragma unroll
        for (int j = 0; j < 2; ++j) { o[2 * j] = bf_lo(v[j]); o[2 * j + 1] = bf_hi(v[j]); }
    }
}
template <int V, bool NT = false> __device__ __forceinline__ void stv(float* p, const float* o) {
#pragma unroll
    for (int i = 0; i < V; i += 4) {
        const f32x4 v = {o[i], o[i + 1], o[i + 2], o[i + 3]};
        if (NT) __builtin_nontemporal_store(v, (f32x4_u*)(p + i));
        else *(f32x4_u*)(p + i) = v;
    }
}
template <int V, bool NT = false> __device__ __forceinline__ void stv(bf16_t* p, const float* o) {
    if constexpr (V == 8) {
        const u32x4 v = {to_2h16(o[0], o[1]), to_2h16(o[2], o[3]), to_2h16(o[4], o[5]), to_2h16(o[6], o[7])};
        if (NT) __builtin_nontemporal_store(v, (u32x4_u*)p);
        else *(u32x4_u*)p = v;
    } else {
        const u32x2 v = {to_2h16(o[0], o[1]), to_2h16(o[2], o[3])};
        if (NT) __builtin_nontemporal_store(v, (u32x2_u*)p);
        else *(u32x2_u*)p = v;
    }
}
__device__ __forceinline__ void st1(float* p, float v) { *p = v; }
__device__ __forceinline__ void st1(bf16_t* p, float v) { *p = to_h16(v); }
// V elements at column c of a row of H; what lies behind the row's end reads as `fill` and is not written
template <int V, typename T> __device__ __forceinline__ void ld_edge(const T* row, int c, int H, float fill, float* o) {
    if (c + V <= H) return ldv<V>(row + c, o);
#pragma unroll
    for (int j = 0; j < V; ++j) o[j] = c + j < H ? Elem<T>::ld(row + c + j) : fill;
}
template <int V, typename T> __device__ __forceinline__ void st_edge(T* row, int c, int H, const float* o) {
    if (c + V <= H) return stv<V>(row + c, o);
#pragma unroll
    for (int j = 0; j < V; ++j)
        if (c + j < H) st1(row + c + j, o[j]);
}

// the columns of a lane's vector that begins at c in a row of H >= V
template <int V> struct span {
    int at, skip;                          // the vector is read and written at `at`; its first `skip` elements are not its own
    __device__ __forceinline__ span() {}
    __device__ __forceinline__ span(int c, int H) : at(min(c, H - V)), skip(c - at) {}
    __device__ __forceinline__ float own(float v, int j) const { return j >= skip ? v : 0.f; }
    __device__ __forceinline__ bool in() const { return skip < V; }
};

// T lanes share a row; BLOCK and BIG_BLOCK: the whole workgroup does.  The backward needs 118 to 124 registers for 16-bit rows, so
// BLOCK has up to 1024 threads there; for fp32 rows it needs 138, and BLOCK has up to 512 threads (held to the 128 registers of
// 1024 threads 30000 x 2050 takes 146 us instead of 130), BIG_BLOCK, which keeps 11 of them in memory, up to 1024.
enum { BLOCK = 0, BIG_BLOCK = 1 };
constexpr int E = 16;                     // elements per lane
template <int T> __device__ __forceinline__ int row_lanes() { return T > BIG_BLOCK ? T : (int)blockDim.x; }
template <int T> __device__ __forceinline__ int row_lane() { return T > BIG_BLOCK ? threadIdx.x % (T > BIG_BLOCK ? T : 1) : threadIdx.x; }
template <int T> __device__ __forceinline__ int row_in_block() { return T > BIG_BLOCK ? threadIdx.x / (T > BIG_BLOCK ? T : 1) : 0; }
template <int T> constexpr int rows_per_block(int threads) { return T > BIG_BLOCK ? threads / (T > BIG_BLOCK ? T : 1) : 1; }
template <int T, int V> constexpr int most_threads() { return T > BIG_BLOCK ? 256 : T == BLOCK && V == 4 ? 512 : 1024; }

// sum over the lanes of a row, the same bits in all of them; `part` (a workgroup's row): a float per wave, not used again before another
// barrier
template <int T> __device__ __forceinline__ float row_sum(float v, float* part) {
    if constexpr (T <= BIG_BLOCK || T == 64) v = wave_sum_dpp(v);
    else v = lanes_sum_dpp<T>(v);
    if constexpr (T <= BIG_BLOCK) {
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0.f;
        for (int i = 0; i < (int)blockDim.x / 64; ++i) v += part[i];
    }
    return v;
}

template <typename TX, typename TY, typename TW, int V, int T, bool NT>
__global__ __launch_bounds__((most_threads<T, V>())) void layer_norm_kernel(const TX* x, long long ldx, const TW* w, const TW* b, float eps,
                                                                    TY* y, long long ldy, float* mean, float* rstd, int R, int H) {
    __shared__ float part[2][2][16];
    constexpr int NV = E / V;
    constexpr int rows = rows_per_block<T>(256);
    const int lanes = row_lanes<T>(), t = row_lane<T>();
    float wv[NV][V], bv[NV][V];
    span<V> col[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        col[i] = span<V>((i * lanes + t) * V, H);
#pragma unroll
        for (int j = 0; j < V; ++j) { wv[i][j] = 1.f; bv[i][j] = 0.f; }
        if (w) ldv<V>(w + col[i].at, wv[i]);
        if (b) ldv<V>(b + col[i].at, bv[i]);
    }
    const float inv = 1.0f / (float)H;
    int odd = 0;
    for (long long row = (long long)blockIdx.x * rows + row_in_block<T>(); row < R;
         row += (long long)gridDim.x * rows, odd ^= 1) {
        float v[NV][V], s = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) ldv<V, NT>(x + row * ldx + col[i].at, v[i]);
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) s += col[i].own(v[i][j], j);
        const float mu = row_sum<T>(s, part[odd][0]) * inv;
        float q = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                v[i][j] -= mu;
                q += col[i].own(v[i][j] * v[i][j], j);
            }
        const float rs = 1.0f / sqrtf(row_sum<T>(q, part[odd][1]) * inv + eps);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float o[V];
#pragma unroll
            for (int j = 0; j < V; ++j) o[j] = v[i][j] * rs * wv[i][j] + bv[i][j];
            if (col[i].in()) stv<V, NT>(y + row * ldy + col[i].at, o);
        }
        if (t == 0) {
            if (mean) mean[row] = mu;
            if (rstd) rstd[row] = rs;
        }
    }
}

// rows too long for the registers: one block per row, the row is read three times (the second and third from the L2)
template <typename TX, typename TY, typename TW>
__global__ __launch_bounds__(256) void layer_norm_long_kernel(const TX* x, long long ldx, const TW* w, const TW* b, float eps,
                                                              TY* y, long long ldy, float* mean, float* rstd, int R, int H) {
    __shared__ float part[2][2][16];
    const float inv = 1.0f / (float)H;
    int odd = 0;
    for (long long row = blockIdx.x; row < R; row += gridDim.x, odd ^= 1) {
        const TX* xr = x + row * ldx;
        TY* yr = y + row * ldy;
        double s = 0.0, q = 0.0;
        for (int c = threadIdx.x * 4; c < H; c += 1024) {
            float v[4];
            ld_edge<4>(xr, c, H, 0.f, v);
            s += (v[0] + v[1]) + (v[2] + v[3]);
        }
        const float mu = row_sum<BLOCK>((float)s, part[odd][0]) * inv;
        for (int c = threadIdx.x * 4; c < H; c += 1024) {
            float v[4];
            ld_edge<4>(xr, c, H, mu, v);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = (v[j] - mu) * (v[j] - mu);
            q += (v[0] + v[1]) + (v[2] + v[3]);
        }
        const float rs = 1.0f / sqrtf(row_sum<BLOCK>((float)q, part[odd][1]) * inv + eps);
        for (int c = threadIdx.x * 4; c < H; c += 1024) {
            float v[4], wv[4] = {1.f, 1.f, 1.f, 1.f}, bv[4] = {0.f, 0.f, 0.f, 0.f};
            ld_edge<4>(xr, c, H, 0.f, v);
            if (w) ld_edge<4>(w, c, H, 0.f, wv);
            if (b) ld_edge<4>(b, c, H, 0.f, bv);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = (v[j] - mu) * rs * wv[j] + bv[j];
            st_edge<4>(yr, c, H, v);
        }
        if (threadIdx.x == 0) {
            if (mean) mean[row] = mu;
            if (rstd) rstd[row] = rs;
        }
    }
}

// dx of the rows first, first + step, ..; SUMS: also this thread's share of sum dy * xhat and sum dy of its columns
template <typename TX, typename TD, typename TW, int V, int T, bool SUMS, bool NT>
__device__ __forceinline__ void norm_bwd_rows(const TD* dy, long long lddy, const TX* x, long long ldx, const float* mean,
                                              const float* rstd, const TW* w, TX* dx, long long lddx, int R, int H, int t,
                                              long long first, long long step, float (&aw)[E / V][V], float (&ab)[E / V][V]) {
    __shared__ float part[2][2][16];
    constexpr int NV = E / V;
    // A workgroup's row chooses a lane's own elements once and stores them one by one where the row's end cuts the vector (16000 x
    // 4096 bf16: 79 us, with a choice for each of the three sums 92; where a wave has the row the memory is the bound
    // either way and whole stores are better: 65536 x 1024 bf16 74 us, 77 with single ones).
    constexpr bool ONCE = T <= BIG_BLOCK;
    constexpr bool WHOLE = SUMS && T == BLOCK && V == 8;      // ceil(H / 1024) waves: no row ends in the first of two vectors
    const int lanes = row_lanes<T>();
    float wv[NV][V];
    span<V> col[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        col[i] = span<V>((i * lanes + t) * V, H);
#pragma unroll
        for (int j = 0; j < V; ++j) { wv[i][j] = 1.f; aw[i][j] = ab[i][j] = 0.f; }
        if (w) ldv<V>(w + col[i].at, wv[i]);
    }
    const float inv = 1.0f / (float)H;
    int odd = 0;
    for (long long row = first; row < R; row += step, odd ^= 1) {
        float d[NV][V], h[NV][V], sg = 0.f, sgx = 0.f;
        const float mu = mean[row], rs = rstd[row];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            ldv<V, NT>(dy + row * lddy + col[i].at, d[i]);
            ldv<V, NT>(x + row * ldx + col[i].at, h[i]);
        }
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                h[i][j] = (h[i][j] - mu) * rs;
                const float own = WHOLE && i == 0 ? d[i][j] : col[i].own(d[i][j], j);
                if constexpr (SUMS) {
                    aw[i][j] += own * h[i][j];
                    ab[i][j] += own;
                }
                d[i][j] = (ONCE ? own : d[i][j]) * wv[i][j];
                const float g = ONCE ? d[i][j] : col[i].own(d[i][j], j);
                sg += g;
                sgx += g * h[i][j];
            }
        const float mg = row_sum<T>(sg, part[odd][0]) * inv, mgx = row_sum<T>(sgx, part[odd][1]) * inv;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float o[V];
#pragma unroll
            for (int j = 0; j < V; ++j) o[j] = rs * (d[i][j] - mg - h[i][j] * mgx);
            TX* to = dx + row * lddx + col[i].at;
            if (ONCE ? !col[i].skip : col[i].in()) {
                stv<V, NT>(to, o);
            } else if (ONCE && col[i].in()) {
#pragma unroll
                for (int j = 1; j < V; ++j)
                    if (j >= col[i].skip) st1(to + j, o[j]);
            }
        }
    }
}

// Many rows.  Every workgroup walks its rows with the column sums in registers and leaves one pair of partial sums:
// ws [gridDim.x][2][ldp] of (dy * xhat, dy); ws NULL: dx only.
template <typename TX, typename TD, typename TW, int V, int T, bool NT>
__global__ __launch_bounds__((most_threads<T, V>())) void layer_norm_bwd_kernel(const TD* dy, long long lddy, const TX* x, long long ldx,
                                                                        const float* mean, const float* rstd, const TW* w, TX* dx,
                                                                        long long lddx, float* ws, int ldp, int R, int H) {
    constexpr int NV = E / V, ROWS = rows_per_block<T>(256), WIDTH = T * E;        // WIDTH: columns of a row's lanes
    __shared__ __attribute__((aligned(16))) float comb[T > BIG_BLOCK ? ROWS * WIDTH : 4];
    const int t = row_lane<T>(), r = row_in_block<T>();
    float aw[NV][V], ab[NV][V];
    norm_bwd_rows<TX, TD, TW, V, T, true, NT>(dy, lddy, x, ldx, mean, rstd, w, dx, lddx, R, H, t, (long long)blockIdx.x * ROWS + r,
                                              (long long)gridDim.x * ROWS, aw, ab);
    if (!ws) return;
    float* out = ws + (size_t)blockIdx.x * 2 * ldp;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const float(&a)[NV][V] = k ? ab : aw;
        if constexpr (T > BIG_BLOCK) {               // the workgroup's rows, added in their order
            if (k) __syncthreads();
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int j = 0; j < V; j += 4)
                    *(f32x4*)(comb + r * WIDTH + (i * T + t) * V + j) = f32x4{a[i][j], a[i][j + 1], a[i][j + 2], a[i][j + 3]};
            __syncthreads();
            const int whole = H / V * V, shift = (V - H % V) % V;        // the last vector's own elements are its last ones
            for (int c = threadIdx.x; c < H; c += 256) {
                const float* e = comb + c + (c >= whole ? shift : 0);
                float s = e[0];
#pragma unroll
                for (int i = 1; i < ROWS; ++i) s += e[i * WIDTH];
                out[k * ldp + c] = s;
            }
        } else {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const span<V> col((i * (int)blockDim.x + t) * V, H);
                if (!col.skip) {
                    stv<V>(out + k * ldp + col.at, a[i]);
                    continue;
                }
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (j >= col.skip) out[k * ldp + col.at + j] = a[i][j];
            }
        }
    }
}

// Few rows, one launch: the column sums need only the statistics, which are there already, so they do not wait for dx.  The
// first `cols` workgroups own 32 columns each and walk down ALL rows (x and dy are read twice, the second time from the
// cache); the others own rows and give dx.
template <typename TX, typename TD, typename TW, int V, int T>
__global__ __launch_bounds__(512) void layer_norm_bwd_few_kernel(const TD* dy, long long lddy, const TX* x, long long ldx,
                                                                 const float* mean, const float* rstd, const TW* w, TX* dx,
                                                                 long long lddx, float* dweight, float* dbias, int accumulate,
                                                                 int cols, int R, int H) {
    if ((int)blockIdx.x >= cols) {
        constexpr int ROWS = rows_per_block<T>(512);
        float aw[E / V][V], ab[E / V][V];
        norm_bwd_rows<TX, TD, TW, V, T, false, false>(dy, lddy, x, ldx, mean, rstd, w, dx, lddx, R, H,
                                                      row_lane<T>(), (long long)(blockIdx.x - cols) * ROWS + row_in_block<T>(),
                                                      (long long)(gridDim.x - cols) * ROWS, aw, ab);
        return;
    }
    // workgroups b and b + 8 share an XCD's L2: they own neighbouring columns, which share lines (1200 x 4096
    // bf16 12.9 -> 10.7 us, 2077 x 1001 11.4 -> 10.9)
    const int b = blockIdx.x, group = b < (cols & ~15) ? (b & ~15) | (b & 7) << 1 | (b >> 3 & 1) : b;
    constexpr int LANES = 32 / V, SLOTS = 512 / LANES;
    __shared__ float sums[2][SLOTS][32 + 1];
    const int lane = threadIdx.x % LANES, slot = threadIdx.x / LANES;
    const span<V> at(group * 32 + lane * V, H);
    float aw[V], ab[V];
#pragma unroll
    for (int j = 0; j < V; ++j) aw[j] = ab[j] = 0.f;
#pragma unroll 4
    for (int row = slot; row < R; row += SLOTS) {
        float d[V], h[V];
        ldv<V>(dy + row * lddy + at.at, d);
        ldv<V>(x + row * ldx + at.at, h);
        const float mu = mean[row], rs = rstd[row];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            aw[j] += d[j] * ((h[j] - mu) * rs);
            ab[j] += d[j];
        }
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
        sums[0][slot][lane * V + j] = aw[j];
        sums[1][slot][lane * V + j] = ab[j];
    }
    __syncthreads();
    // 64 sums (two of 32 columns) of SLOTS terms each: eight threads per sum, then their eight in order
    const int col = threadIdx.x & 31, which = (threadIdx.x >> 5) & 1, share = threadIdx.x >> 6;
    const int from = min(col + (group * 32 + col >= H / V * V ? (V - H % V) % V : 0), 31);
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < SLOTS / 8; ++i) s += sums[which][share * (SLOTS / 8) + i][from];
    __syncthreads();
    sums[which][share][col] = s;
    __syncthreads();
    float* dst = which ? dbias : dweight;
    if (share || !dst || group * 32 + col >= H) return;
#pragma unroll
    for (int i = 1; i < 8; ++i) s += sums[which][i][col];
    dst += group * 32 + col;
    *dst = accumulate ? *dst + s : s;
}

// long rows: dx row by row (two walks over the row), and the column sums by a kernel of their own
template <typename TX, typename TD, typename TW>
__global__ __launch_bounds__(256) void layer_norm_bwd_long_kernel(const TD* dy, long long lddy, const TX* x, long long ldx,
                                                                  const float* mean, const float* rstd, const TW* w, TX* dx,
                                                                  long long lddx, int R, int H) {
    __shared__ float part[2][2][16];
    const float inv = 1.0f / (float)H;
    int odd = 0;
    for (long long row = blockIdx.x; row < R; row += gridDim.x, odd ^= 1) {
        const float mu = mean[row], rs = rstd[row];
        double sg = 0.0, sgx = 0.0;
        for (int c = threadIdx.x * 4; c < H; c += 1024) {
            float d[4], v[4], wv[4] = {1.f, 1.f, 1.f, 1.f};
            ld_edge<4>(dy + row * lddy, c, H, 0.f, d);
            ld_edge<4>(x + row * ldx, c, H, 0.f, v);
            if (w) ld_edge<4>(w, c, H, 0.f, wv);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                d[j] *= wv[j];
                v[j] = d[j] * ((v[j] - mu) * rs);
            }
            sg += (d[0] + d[1]) + (d[2] + d[3]);
            sgx += (v[0] + v[1]) + (v[2] + v[3]);
        }
        const float mg = row_sum<BLOCK>((float)sg, part[odd][0]) * inv, mgx = row_sum<BLOCK>((float)sgx, part[odd][1]) * inv;
        for (int c = threadIdx.x * 4; c < H; c += 1024) {
            float d[4], v[4], wv[4] = {1.f, 1.f, 1.f, 1.f};
            ld_edge<4>(dy + row * lddy, c, H, 0.f, d);
            ld_edge<4>(x + row * ldx, c, H, 0.f, v);
            if (w) ld_edge<4>(w, c, H, 0.f, wv);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = rs * (d[j] * wv[j] - mg - (v[j] - mu) * rs * mgx);
            st_edge<4>(dx + row * lddx, c, H, v);
        }
    }
}

template <typename TX, typename TD>
__global__ __launch_bounds__(256) void layer_norm_bwd_columns_kernel(const TD* dy, long long lddy, const TX* x, long long ldx,
                                                                     const float* mean, const float* rstd, float* ws, int ldp,
                                                                     int R, int H) {
    const int c = (blockIdx.x * 256 + threadIdx.x) * 4;
    double sw[4] = {0.0, 0.0, 0.0, 0.0}, sb[4] = {0.0, 0.0, 0.0, 0.0};
    if (c >= H) return;
    for (long long row = blockIdx.y; row < R; row += gridDim.y) {
        float d[4], v[4];
        ld_edge<4>(dy + row * lddy, c, H, 0.f, d);
        ld_edge<4>(x + row * ldx, c, H, 0.f, v);
        const float mu = mean[row], rs = rstd[row];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            sw[j] += d[j] * ((v[j] - mu) * rs);
            sb[j] += d[j];
        }
    }
    float aw[4], ab[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) { aw[j] = (float)sw[j]; ab[j] = (float)sb[j]; }
    float* out = ws + (size_t)blockIdx.y * 2 * ldp;
    st_edge<4>(out, c, H, aw);
    st_edge<4>(out + ldp, c, H, ab);
}

// dweight / dbias (+)= the partial sums, in the order of the blocks that left them: 8 lanes of four columns, 32 slots
__global__ __launch_bounds__(256) void layer_norm_bwd_join_kernel(const float* ws, int ldp, int parts, float* dweight,
                                                                  float* dbias, int accumulate, int H) {
    __shared__ f32x4 sum[32][8];
    const int lane = threadIdx.x & 7, slot = threadIdx.x >> 3, c = (blockIdx.x * 8 + lane) * 4;
    const float* src = ws + (size_t)blockIdx.y * ldp + c;
    float* dst = blockIdx.y ? dbias : dweight;
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
    if (c < ldp) {
#pragma unroll 8
        for (int p = slot; p < parts; p += 32) s += *(const f32x4*)(src + (size_t)p * 2 * ldp);
    }
    sum[slot][lane] = s;
    __syncthreads();
    for (int h = 16; h > 0; h >>= 1) {
        if (slot < h) sum[slot][lane] += sum[slot + h][lane];
        __syncthreads();
    }
    if (slot || !dst) return;
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (c + j < H) dst[c + j] = accumulate ? dst[c + j] + sum[0][lane][j] : sum[0][lane][j];
}

__global__ __launch_bounds__(256) void fill_zero_kernel(float* a, float* b, int n) {
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    if (a) a[i] = 0.f;
    if (b) b[i] = 0.f;
}

constexpr int LONGEST = 1 << 30;          // columns are counted in 32 bits, a workgroup's stride behind the end included
constexpr int IN_REGISTERS = 16384;       // longest row that the register kernels take; the shortest is a vector
inline bool in_registers(int H) { return H >= 8 && H <= IN_REGISTERS; }

inline int norm_blocks(long long R, int rows_per_block, int per_cu) {
    return (int)std::min<long long>((R + rows_per_block - 1) / rows_per_block, (long long)per_cu * cu_count());
}
// A call that moves more than the memory-side cache holds (256 MB) goes past the caches (us past them, through them): 131072 x 1024
// fp32 -> bf16 133 and 152, 65536 x 2048 bf16 94 and 103, backward of 32768 x 2048 fp32 142 and 155, of 65536 x 1024 bf16 76 and 83, of
// 32768 x 4096 bf16 144 and 147.  16-bit rows of 32 lanes gain nothing: 262144 x 300 bf16 75 and 75, its backward 101 and 98.  Below
// that the next kernel finds the result in a cache.
inline bool past_caches(long long bytes) { return bytes > (256ll << 20); }
inline int lanes_of(int H) { return H <= 128 ? 8 : H <= 512 ? 32 : H <= 1024 ? 64 : BLOCK; }
inline int threads_of(int H) { return H <= 1024 ? 256 : cdiv(H, 1024) * 64; }
inline int rows_of_block(int H) { return H <= 1024 ? 256 / lanes_of(H) : 1; }
// Few rows: the column sums walk down the rows in the launch that gives dx, without the second launch, the workspace and the
// partial sums.  A workgroup reads 32 columns of all rows, 320 KB at most.  GPU us by one and by two launches, with operands that the
// last call did not have: 512 x 1024 bf16 3.0 and 7.2, 1000 x 1024 5.1 and 8.1, 1500 x 1024 8.0 and 9.5, 1024 x 1024 fp32 7.9 and
// 9.3, 1200 x 4096 bf16 11.0 and 15.2, fp32 15.6 and 16.8; rows that begin anywhere, 1000 x 1001 bf16 7.1 and 8.6, 1500 x 1001 9.3
// and 10.1.  The limit suits operands that are still in the L2 (the same ones again, 2500 x 1024 bf16: 7.8 and 10.2); for others
// two launches are better from about 250 KB on: 2000 x 1024 bf16 11.3 and 11.0, 2500 x 1024 13.6 and 10.7, 2077 x 1001 12.0 and
// 10.2.  Behind the limit, 4096 x 1024 bf16: 21 and 11.
inline bool one_launch(int R, int H, int x_size, int dy_size) {
    return (long long)R * 32 * (x_size + dy_size) <= 320 << 10 && H >= 8 && H <= 8192;
}
// Workgroups of the backward, each of which leaves partial sums as large as two fp32 rows: at least six rows for each where that
// leaves one per CU (4096 x 2048 bf16: two 40, six 26 us; 16 x 16384 fp32: one 14, six 44).  fp32 rows: eight waves per CU
// (32768 x 2048: 142 us, sixteen 157).  Rows of 16 bits have half the bytes in flight: sixteen waves where a wave has a row
// (65536 x 1024 bf16: 74 us, eight 78), else four workgroups of two or three waves (30000 x 2050: 78, three 90), two of four to
// eight (32768 x 4096: 144, four 152; 16000 x 8192: 138, one 158).
inline int bwd_parts(int R, int H, int size) {
    if (!in_registers(H)) return (int)std::min<long long>(R, 64);
    const int waves = threads_of(H) / 64, places = waves > 4 ? (waves + 3) / 4 * 4 : waves;     // the same number on all four SIMDs
    const int per_cu = size == 4 ? std::max(1, 8 / places) : H <= 1024 || waves <= 3 ? 4 : waves <= 8 ? 2 : 1;
    const int least = std::max(1, std::min(6, R / cu_count()));
    return norm_blocks(R, std::max(rows_of_block(H) * 2, least), per_cu);
}
inline int ld_parts(int H) { return (H + 3) / 4 * 4; }

#define NORM_LANES(CALL)                                  \
    switch (lanes_of(H)) {                                \
        case 8: CALL(8); break;                           \
        case 32: CALL(32); break;                         \
        case 64: CALL(64); break;                         \
        default:                                          \
            if constexpr (V == 4) {                       \
                if (H > 8192) { CALL(BIG_BLOCK); break; } \
            }                                             \
            CALL(BLOCK);                                  \
    }

template <typename TX, typename TY, typename TW>
int launch_ln(const void* x, long long ldx, const void* w, const void* b, float eps, void* y, long long ldy, float* mean,
              float* rstd, int R, int H, hipStream_t st) {
    constexpr int V = sizeof(TX) == 2 ? 8 : 4;
    const bool streams = past_caches((long long)R * H * (sizeof(TX) + sizeof(TY)));
    // all the threads that a CU holds; past the caches fewer streams suit the memory better: sixteen waves (262144 x 300 bf16 76 -> 69
    // us, 131072 x 1024 bf16 102 -> 99), for fp32 rows eight or two workgroups (131072 x 1024 -> bf16 140 -> 131, 65536 x 2048 197 -> 180,
    // 16384 x 8192 -> bf16 142 -> 127, one workgroup 166)
    const int threads = threads_of(std::min(H, IN_REGISTERS));
    const int per_cu = !streams ? 2048 / threads : V == 8 ? 1024 / threads : std::max(2, 512 / threads);
    const dim3 grid(norm_blocks(R, rows_of_block(H), per_cu)), block(threads_of(H));
#define LN_AT(T, NT)                                                                                                           \
    hipLaunchKernelGGL((layer_norm_kernel<TX, TY, TW, V, T, NT>), grid, block, 0, st, (const TX*)x, ldx, (const TW*)w, (const TW*)b, eps, \
                       (TY*)y, ldy, mean, rstd, R, H)
#define LN(T)                                                                  \
    do {                                                                       \
        if (streams) LN_AT(T, true);                                           \
        else LN_AT(T, false);                                                  \
    } while (0)
    if (!in_registers(H))
        hipLaunchKernelGGL((layer_norm_long_kernel<TX, TY, TW>), dim3(norm_blocks(R, 1, 8)), dim3(256), 0, st, (const TX*)x, ldx,
                           (const TW*)w, (const TW*)b, eps, (TY*)y, ldy, mean, rstd, R, H);
    else
        NORM_LANES(LN)
#undef LN
#undef LN_AT
    STDIFF_LAUNCH_STATUS();
    return STDIFF_OK;
}

template <typename TX, typename TD, typename TW>
int launch_ln_grad(const void* dy, long long lddy, const void* x, long long ldx, const float* mean, const float* rstd,
                   const void* w, void* dx, long long lddx, float* dweight, float* dbias, int accumulate, float* ws, int R, int H,
                   hipStream_t st) {
    constexpr int V = sizeof(TX) == 2 ? 8 : 4;
    const int ldp = ld_parts(H), parts = bwd_parts(R, H, sizeof(TX));
    if (one_launch(R, H, sizeof(TX), sizeof(TD)) && (dweight || dbias)) {
        const int cols = cdiv(H, 32), rows = norm_blocks(R, H <= 1024 ? 8 : 1, 4);
        const auto meets = [&](const void* p, long long ld, size_t size) {
            const uintptr_t a = (uintptr_t)p, b = (uintptr_t)dx;
            return a < b + ((R - 1) * lddx + H) * sizeof(TX) && b < a + ((R - 1) * ld + H) * size;
        };
        // dx in the place of x or dy: the columns first, in a launch of their own
        const bool in_place = meets(x, ldx, sizeof(TX)) || meets(dy, lddy, sizeof(TD));
#define FEW(GRID, COLS, T)                                                                                                        \
    hipLaunchKernelGGL((layer_norm_bwd_few_kernel<TX, TD, TW, V, T>), dim3(GRID), dim3(512), 0, st, (const TD*)dy, lddy, (const TX*)x, \
                       ldx, mean, rstd, (const TW*)w, (TX*)dx, lddx, dweight, dbias, accumulate, COLS, R, H)
#define FEW_AT(GRID, COLS)                        \
    do {                                          \
        if (H <= 1024) FEW(GRID, COLS, 64);       \
        else FEW(GRID, COLS, BLOCK);              \
    } while (0)
        if (in_place) {
            FEW_AT(cols, cols);
            FEW_AT(rows, 0);
        } else {
            FEW_AT(cols + rows, cols);
        }
#undef FEW
#undef FEW_AT
        STDIFF_LAUNCH_STATUS();
        return STDIFF_OK;
    }
    const bool streams = past_caches((long long)R * H * (2 * sizeof(TX) + sizeof(TD)));
    const dim3 grid(parts), block(threads_of(H));
#define LN_AT(T, NT)                                                                                                          \
    hipLaunchKernelGGL((layer_norm_bwd_kernel<TX, TD, TW, V, T, NT>), grid, block, 0, st, (const TD*)dy, lddy, (const TX*)x, ldx, mean, \
                       rstd, (const TW*)w, (TX*)dx, lddx, ws, ldp, R, H)
#define LN(T)                                                                  \
    do {                                                                       \
        if (streams) LN_AT(T, true);                                           \
        else LN_AT(T, false);                                                  \
    } while (0)
    if (!in_registers(H)) {
        if (ws)
            hipLaunchKernelGGL((layer_norm_bwd_columns_kernel<TX, TD>), dim3(cdiv(H, 1024), parts), dim3(256), 0, st, (const TD*)dy,
                               lddy, (const TX*)x, ldx, mean, rstd, ws, ldp, R, H);
        hipLaunchKernelGGL((layer_norm_bwd_long_kernel<TX, TD, TW>), dim3(norm_blocks(R, 1, 8)), dim3(256), 0, st, (const TD*)dy,
                           lddy, (const TX*)x, ldx, mean, rstd, (const TW*)w, (TX*)dx, lddx, R, H);
    } else {
        NORM_LANES(LN)
    }
#undef LN
#undef LN_AT
    STDIFF_LAUNCH_STATUS();
    if (ws) {
        hipLaunchKernelGGL(layer_norm_bwd_join_kernel, dim3(cdiv(H, 32), 2), dim3(256), 0, st, ws, ldp, parts, dweight, dbias, accumulate, H);
        STDIFF_LAUNCH_STATUS();
    }
    return STDIFF_OK;
}

inline bool dtype_ok(int dt) { return dt == STDIFF_F32 || dt == STDIFF_BF16; }
inline bool at_element(const void* p, int dt) { return ((uintptr_t)p & (dt == STDIFF_BF16 ? 1 : 3)) == 0; }

}  // namespace

extern "C" int stdiff_layer_norm(const void* x, long long ldx, int x_dtype, const void* weight, const void* bias, int w_dtype,
                                 float eps, void* y, long long ldy, int y_dtype, float* mean, float* rstd, int R, int H,
                                 void* stream) {
    STDIFF_CHECK_ARG(R >= 0 && H > 0 && (R == 0 || (x && y)) && ldx >= 0 && ldy >= H && eps >= 0.f);
    STDIFF_CHECK_ARG(dtype_ok(x_dtype) && dtype_ok(y_dtype) && dtype_ok(w_dtype));
    if (R == 0) return STDIFF_OK;
    if (H > LONGEST) return STDIFF_ERR_SHAPE;
    if (!at_element(x, x_dtype) || !at_element(y, y_dtype) || !at_element(weight, w_dtype) || !at_element(bias, w_dtype) ||
        !at_element(mean, STDIFF_F32) || !at_element(rstd, STDIFF_F32))
        return STDIFF_ERR_ALIGN;
#define LN(TX, TY, TW) launch_ln<TX, TY, TW>(x, ldx, weight, bias, eps, y, ldy, mean, rstd, R, H, (hipStream_t)stream)
    switch ((x_dtype == STDIFF_BF16) * 4 + (y_dtype == STDIFF_BF16) * 2 + (w_dtype == STDIFF_BF16)) {
        case 0: return LN(float, float, float);
        case 1: return LN(float, float, bf16_t);
        case 2: return LN(float, bf16_t, float);
        case 3: return LN(float, bf16_t, bf16_t);
        case 4: return LN(bf16_t, float, float);
        case 5: return LN(bf16_t, float, bf16_t);
        case 6: return LN(bf16_t, bf16_t, float);
        default: return LN(bf16_t, bf16_t, bf16_t);
    }
#undef LN
}

extern "C" long long stdiff_layer_norm_bwd_workspace(int R, int H, int x_dtype, int dy_dtype) {
    if (R < 0 || H <= 0 || !dtype_ok(x_dtype) || !dtype_ok(dy_dtype)) return STDIFF_ERR_ARG;
    if (H > LONGEST) return STDIFF_ERR_SHAPE;
    const int size = (int)dtype_size(x_dtype);
    return one_launch(R, H, size, (int)dtype_size(dy_dtype)) ? 0 : (long long)bwd_parts(R, H, size) * 2 * ld_parts(H) * 4;
}

extern "C" int stdiff_layer_norm_bwd(const void* dy, long long lddy, int dy_dtype, const void* x, long long ldx, int x_dtype,
                                     const float* mean, const float* rstd, const void* weight, int w_dtype, void* dx,
                                     long long lddx, float* dweight, float* dbias, int accumulate, float* workspace,
                                     long long workspace_bytes, int R, int H, void* stream) {
    STDIFF_CHECK_ARG(R >= 0 && H > 0 && (R == 0 || (dy && x && mean && rstd && dx)) && lddy >= 0 && ldx >= 0 && lddx >= H);
    STDIFF_CHECK_ARG(dtype_ok(dy_dtype) && dtype_ok(x_dtype) && dtype_ok(w_dtype));
    if (H > LONGEST) return STDIFF_ERR_SHAPE;
    if (!at_element(dy, dy_dtype) || !at_element(x, x_dtype) || !at_element(dx, x_dtype) || !at_element(weight, w_dtype) ||
        !at_element(mean, STDIFF_F32) || !at_element(rstd, STDIFF_F32) || !at_element(dweight, STDIFF_F32) ||
        !at_element(dbias, STDIFF_F32) || ((uintptr_t)workspace & 15))
        return STDIFF_ERR_ALIGN;
    const bool params = dweight || dbias;
    hipStream_t st = (hipStream_t)stream;
    if (R == 0) {
        if (params && !accumulate) {
            hipLaunchKernelGGL(fill_zero_kernel, dim3(cdiv(H, 256)), dim3(256), 0, st, dweight, dbias, H);
            STDIFF_LAUNCH_STATUS();
        }
        return STDIFF_OK;
    }
    const long long need = params ? stdiff_layer_norm_bwd_workspace(R, H, x_dtype, dy_dtype) : 0;
    if (need && (!workspace || workspace_bytes < need)) return STDIFF_ERR_WORKSPACE;
    float* ws = need ? workspace : nullptr;
#define LN(TX, TD, TW)                                                                                                            \
    return launch_ln_grad<TX, TD, TW>(dy, lddy, x, ldx, mean, rstd, weight, dx, lddx, dweight, dbias, accumulate, ws, R, H, st)
    switch ((x_dtype == STDIFF_BF16) * 4 + (dy_dtype == STDIFF_BF16) * 2 + (w_dtype == STDIFF_BF16)) {
        case 0: LN(float, float, float);
        case 1: LN(float, float, bf16_t);
        case 2: LN(float, bf16_t, float);
        case 3: LN(float, bf16_t, bf16_t);
        case 4: LN(bf16_t, float, float);
        case 5: LN(bf16_t, float, bf16_t);
        case 6: LN(bf16_t, bf16_t, float);
        default: LN(bf16_t, bf16_t, bf16_t);
    }
#undef LN
}
