// Layer norm over the last dimension, forward and backward:
//   y  = xhat * w + b,   xhat = (x - mean) * rstd,   rstd = 1 / sqrt(mean((x - mean)^2) + eps)
//   dx = rstd * (h - mean(h) - xhat * mean(h * xhat)),   h = dy * w
//   dw = sum over rows of dy * xhat,   db = sum over rows of dy
// Bound by memory: the forward reads x and writes y, the backward reads x and dy and writes dx.
//
// A row lies in the registers of TPR threads (16 to 64 lanes of a wave, or a whole workgroup), so
// that it is read once: the mean first, then the squared differences from it (a sum of squares
// minus a squared mean would lose the variance of rows far from zero). All sums are fp32 or wider.
// The backward's threads keep their columns' dw and db over all rows that their workgroup takes
// and write one fp32 partial row per workgroup; a second kernel adds the partial rows in order
// (in double), so gradients do not change from run to run. fp32 inputs keep a compensation term
// beside each of these sums; 16-bit ones do not (add_to).
//
// Measured, forward and backward with the second kernel, averages (a large copy runs at 4.96 TB/s): 16,384 x 4,096 bf16
// 54 and 98 + 8 us (5.0 and 4.1 TB/s); 2 M x 256 fp32 805 and 1236 + 9 us (5.1 and 5.0 TB/s); 14,541 x 128 fp32 5.9 and
// 8.2 + 4.4 us, launches and latency.
#include <algorithm>

#include "num_types.h"

namespace mpgnn {
namespace {

struct NormArgs {
    const void* x;
    const void* dy;
    void* out;         // y, or dx
    const void* w;
    const void* b;
    float* mean;       // [rows] written by the forward (or null), read by the backward
    float* rstd;
    float* part;       // backward: [blocks][2][width] partials of dw and db (or null)
    int64_t rows, x_pitch, dy_pitch;
    int32_t width;
    int32_t w_f32;     // w and b are fp32 beside 16-bit x
    float eps;
};

template <typename T>
__device__ __forceinline__ float param_at(const void* p, int w_f32, int64_t c) {
    return w_f32 ? ((const float*)p)[c] : (float)((const T*)p)[c];
}

// Parameters c .. c + V - 1 (`none` where there is no vector or it ends): in whole vectors, whatever their alignment.
template <typename T, int V>
__device__ __forceinline__ void params_at(float (&o)[V], const void* p, int w_f32, int c, int F, float none) {
#pragma unroll
    for (int j = 0; j < V; ++j) o[j] = none;
    if (!p) return;
    if (c + V <= F) {
        if (w_f32) {
            __builtin_memcpy(o, (const float*)p + c, sizeof(o));
        } else {
            T e[V];
            __builtin_memcpy(e, (const T*)p + c, sizeof(e));
#pragma unroll
            for (int j = 0; j < V; ++j) o[j] = (float)e[j];
        }
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (c + j < F) o[j] = param_at<T>(p, w_f32, c + j);
    }
}

// The sum of N values over the TPR threads of a row: a butterfly inside a wave, then LDS. `lds`
// holds two buffers used in turn, so one barrier a sum is enough.
template <int TPR, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float* lds, int& turn) {
    constexpr int LANES = TPR < 64 ? TPR : 64;
#pragma unroll
    for (int d = LANES / 2; d > 0; d >>= 1)
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += __shfl_xor(v[i], d, 64);
    if constexpr (TPR > 64) {
        constexpr int W = TPR / 64;
        float* buf = lds + turn * (W * 2);
        turn ^= 1;
        if (threadIdx.x % 64 == 0) {
#pragma unroll
            for (int i = 0; i < N; ++i) buf[(threadIdx.x / 64) * 2 + i] = v[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float s = buf[i];
#pragma unroll
            for (int w = 1; w < W; ++w) s += buf[w * 2 + i];
            v[i] = s;
        }
    }
}

// The mean of a row and its summed squared differences from the mean, from those of each thread's n values:
// two equal parts join to the mean of their means and the sum of their squares plus what the means differ by.
// One exchange where a mean first and differences from it after take two.
template <int TPR>
__device__ __forceinline__ void join_stats(float& mean, float& m2, float n, float* lds, int& turn) {
    constexpr int LANES = TPR < 64 ? TPR : 64;
#pragma unroll
    for (int d = 1; d < LANES; d <<= 1) {
        const float om = __shfl_xor(mean, d, 64), os = __shfl_xor(m2, d, 64);
        const float dm = om - mean;
        mean = 0.5f * (mean + om);
        m2 = __builtin_fmaf(dm * dm, 0.5f * n, m2 + os);
        n *= 2.0f;
    }
    if constexpr (TPR > 64) {
        constexpr int W = TPR / 64;
        float* buf = lds + turn * (W * 2);
        turn ^= 1;
        if (threadIdx.x % 64 == 0) {
            buf[threadIdx.x / 64 * 2] = mean;
            buf[threadIdx.x / 64 * 2 + 1] = m2;
        }
        __syncthreads();
        float ms[W], qs[W];
#pragma unroll
        for (int w = 0; w < W; ++w) {
            ms[w] = buf[w * 2];
            qs[w] = buf[w * 2 + 1];
        }
#pragma unroll
        for (int d = 1; d < W; d <<= 1) {
#pragma unroll
            for (int w = 0; w < W; w += 2 * d) {
                const float dm = ms[w + d] - ms[w];
                ms[w] = 0.5f * (ms[w] + ms[w + d]);
                qs[w] = __builtin_fmaf(dm * dm, 0.5f * n, qs[w] + qs[w + d]);
            }
            n *= 2.0f;
        }
        mean = ms[0];
        m2 = qs[0];
    }
}

template <int TPR>
struct RowShape {
    static constexpr int threads = TPR > 256 ? TPR : 256;
    static constexpr int rows = threads / TPR;          // rows a workgroup has at a time
    static constexpr int lds = TPR > 64 ? TPR / 64 * 4 : 1;
};

// A thread's part of a row on its way from memory: the next row is asked for before the current
// one's sums, whose barriers it does not wait for. WHOLE: rows of whole 16-byte vectors at multiples of 16
// bytes. Else vectors start where they may (the hardware's loads need no more than an element's alignment),
// and the one that the end of the row cuts goes element by element.
template <typename T, int V, int TPR, int NV, bool WHOLE>
struct Row {
    typedef typename VecOf<T, V>::type Vec;
    Vec v[NV];

    __device__ __forceinline__ void load(const T* p, int64_t pitch, int64_t r, int64_t rows, int t, int F) {
        const bool live = r < rows;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * TPR + t) * V;
            const T* at = p + r * pitch + c;
            v[i] = Vec(0);
            if (!live) continue;
            if constexpr (WHOLE) {
                if (c < F) v[i] = *reinterpret_cast<const Vec*>(at);
            } else if (c + V <= F) {
                __builtin_memcpy(&v[i], at, sizeof(Vec));
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (c + j < F) v[i][j] = at[j];
            }
        }
    }
    __device__ __forceinline__ void widen(float (&f)[NV][V]) const {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) f[i][j] = (float)v[i][j];
    }
    static __device__ __forceinline__ void store(T* p, const float (&f)[NV][V], int t, int F) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * TPR + t) * V;
            if (c >= F) continue;
            Vec o;
#pragma unroll
            for (int j = 0; j < V; ++j) o[j] = (T)f[i][j];
            if constexpr (WHOLE) {
                *reinterpret_cast<Vec*>(p + c) = o;
            } else if (c + V <= F) {
                __builtin_memcpy(p + c, &o, sizeof(Vec));
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (c + j < F) p[c + j] = o[j];
            }
        }
    }
    // is element j of a thread's vector i inside the row?
    static __device__ __forceinline__ bool in(int i, int j, int t, int F) {
        return (i * TPR + t) * V + (WHOLE ? 0 : j) < F;
    }
};

template <typename T, int V, int TPR, int NV, bool WHOLE>
__global__ __launch_bounds__(RowShape<TPR>::threads) void layer_norm_fwd_kernel(NormArgs a) {
    using S = RowShape<TPR>;
    using R = Row<T, V, TPR, NV, WHOLE>;
    __shared__ float lds[S::lds];
    const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR;
    const int F = a.width;
    const int64_t step = (int64_t)gridDim.x * S::rows;
    R next;  // on its way before the parameters: a call of few rows is one latency after another
    next.load((const T*)a.x, a.x_pitch, (int64_t)blockIdx.x * S::rows + sub, a.rows, t, F);
    float w[NV][V], b[NV][V];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        params_at<T>(w[i], a.w, a.w_f32, (i * TPR + t) * V, F, 1.0f);
        params_at<T>(b[i], a.b, a.w_f32, (i * TPR + t) * V, F, 0.0f);
    }
    const float width = (float)F;
    const bool full = F == TPR * NV * V;
    int turn = 0;
    // every thread of the workgroup takes part in each turn's sums; rows past the end are not touched
    for (int64_t r0 = (int64_t)blockIdx.x * S::rows; r0 < a.rows; r0 += step) {
        const int64_t r = r0 + sub;
        const bool live = r < a.rows;
        float v[NV][V], s[1] = {0.0f};
        next.widen(v);
        next.load((const T*)a.x, a.x_pitch, r + step, a.rows, t, F);
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) s[0] += v[i][j];
        float mean, q[1] = {0.0f};
        if (full) {  // every thread has as many values
            const float own = s[0] * (1.0f / (NV * V));
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int j = 0; j < V; ++j) q[0] = __builtin_fmaf(v[i][j] - own, v[i][j] - own, q[0]);
            mean = own;
            join_stats<TPR>(mean, q[0], (float)(NV * V), lds, turn);
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int j = 0; j < V; ++j) v[i][j] -= mean;
        } else {
            row_sum<TPR, 1>(s, lds, turn);
            mean = s[0] / width;
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    v[i][j] -= mean;
                    if (R::in(i, j, t, F)) q[0] = __builtin_fmaf(v[i][j], v[i][j], q[0]);
                }
            row_sum<TPR, 1>(q, lds, turn);
        }
        const float rstd = 1.0f / sqrtf(q[0] / width + a.eps);
        if (!live) continue;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) v[i][j] = __builtin_fmaf(v[i][j] * rstd, w[i][j], b[i][j]);
        R::store((T*)a.out + r * F, v, t, F);
        if (a.mean && t == 0) {
            a.mean[r] = mean;
            a.rstd[r] = rstd;
        }
    }
}

// a + v with the rounding error carried in c (Kahan's sum; an infinite sum has none, and stays what it
// is). Plain for 16-bit inputs: their parameters' gradients round far coarser, and where these are fp32 a thread's
// rows are few beside the threads whose sums are then added in double: the largest error of dw in 2^-24 of its value
// is 1.15 from bf16 inputs and 1.03 from fp32 ones, with compensation, at 16,384 x 4,096, and 0.91 and 0.94 at 2 M x 64.
template <bool COMP>
__device__ __forceinline__ void add_to(float& a, float& c, float v) {
    if constexpr (COMP) {
        const float u = v - c;
        const float s = a + u;
        c = __builtin_fabsf(s) <= 3.402823466e38f ? (s - a) - u : 0.0f;
        a = s;
    } else {
        a += v;
    }
}

template <typename T, int V, int TPR, int NV, bool WHOLE>
__global__ __launch_bounds__(RowShape<TPR>::threads) void layer_norm_bwd_kernel(NormArgs a) {
    using S = RowShape<TPR>;
    using R = Row<T, V, TPR, NV, WHOLE>;
    constexpr bool COMP = sizeof(T) == 4;
    constexpr int COLS = TPR * NV * V;
    __shared__ float lds[S::lds];
    __shared__ float s_part[S::rows > 1 ? S::rows * COLS : 1];
    const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR;
    const int F = a.width;
    // the weight stays in registers, but for the largest teams, whose 128 a thread have no room
    constexpr bool KEEP = TPR < 1024;
    float w[KEEP ? NV : 1][V], dw[NV][V], db[NV][V], dwc[COMP ? NV : 1][V], dbc[COMP ? NV : 1][V];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        if constexpr (KEEP) params_at<T>(w[i], a.w, a.w_f32, (i * TPR + t) * V, F, 1.0f);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            dw[i][j] = db[i][j] = 0.0f;
            dwc[COMP ? i : 0][j] = dbc[COMP ? i : 0][j] = 0.0f;
        }
    }
    const float width = (float)F;
    int turn = 0;
    const int64_t step = (int64_t)gridDim.x * S::rows;
    R next_x, next_dy;
    float next_mean = 0.0f, next_rstd = 0.0f;
    auto fetch = [&](int64_t r) {
        next_x.load((const T*)a.x, a.x_pitch, r, a.rows, t, F);
        next_dy.load((const T*)a.dy, a.dy_pitch, r, a.rows, t, F);
        if (r < a.rows) {
            next_mean = a.mean[r];
            next_rstd = a.rstd[r];
        }
    };
    fetch((int64_t)blockIdx.x * S::rows + sub);
    for (int64_t r0 = (int64_t)blockIdx.x * S::rows; r0 < a.rows; r0 += step) {
        const int64_t r = r0 + sub;
        const bool live = r < a.rows;
        const float mean = next_mean, rstd = next_rstd;
        float xh[NV][V], g[NV][V], s[2] = {0.0f, 0.0f};
        next_x.widen(xh);
        next_dy.widen(g);
        fetch(r + step);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float wi[V];
            if constexpr (!KEEP) params_at<T>(wi, a.w, a.w_f32, (i * TPR + t) * V, F, 1.0f);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                if (!(live && R::in(i, j, t, F))) continue;
                xh[i][j] = (xh[i][j] - mean) * rstd;
                add_to<COMP>(dw[i][j], dwc[COMP ? i : 0][j], g[i][j] * xh[i][j]);
                add_to<COMP>(db[i][j], dbc[COMP ? i : 0][j], g[i][j]);
                g[i][j] *= KEEP ? w[KEEP ? i : 0][j] : wi[j];
                s[0] += g[i][j];
                s[1] = __builtin_fmaf(g[i][j], xh[i][j], s[1]);
            }
        }
        if (!a.out) continue;
        row_sum<TPR, 2>(s, lds, turn);
        if (!live) continue;
        const float m1 = s[0] / width, m2 = s[1] / width;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) g[i][j] = rstd * (g[i][j] - m1 - xh[i][j] * m2);
        R::store((T*)a.out + r * F, g, t, F);
    }
    if (!a.part) return;
    // one partial row per workgroup: its row slots added in order through LDS
    float* pw = a.part + (int64_t)blockIdx.x * 2 * F;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        float(&d)[NV][V] = k ? db : dw;
        if constexpr (S::rows > 1) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int j = 0; j < V; ++j) s_part[sub * COLS + (i * TPR + t) * V + j] = d[i][j];
            __syncthreads();
            for (int c = threadIdx.x; c < F; c += S::threads) {
                float v = s_part[c];
                for (int q = 1; q < S::rows; ++q) v += s_part[q * COLS + c];
                pw[(int64_t)k * F + c] = v;
            }
        } else {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = (i * TPR + t) * V;
                if (c + V <= F) {
                    __builtin_memcpy(pw + (int64_t)k * F + c, d[i], sizeof(d[i]));
                } else {
#pragma unroll
                    for (int j = 0; j < V; ++j)
                        if (c + j < F) pw[(int64_t)k * F + c + j] = d[i][j];
                }
            }
        }
    }
}

// Rows too wide for registers: a workgroup per row, which is read again (from L2) for each sum.
constexpr int kWide = 1024;

template <typename T>
__global__ __launch_bounds__(kWide) void layer_norm_fwd_wide_kernel(NormArgs a) {
    __shared__ float lds[kWide / 64 * 4];
    const int F = a.width;
    int turn = 0;
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T* x = (const T*)a.x + r * a.x_pitch;
        T* y = (T*)a.out + r * F;
        float s[1] = {0.0f}, q[1] = {0.0f};
        for (int c = threadIdx.x; c < F; c += kWide) s[0] += (float)x[c];
        row_sum<kWide, 1>(s, lds, turn);
        const float mean = s[0] / (float)F;
        for (int c = threadIdx.x; c < F; c += kWide) {
            const float d = (float)x[c] - mean;
            q[0] = __builtin_fmaf(d, d, q[0]);
        }
        row_sum<kWide, 1>(q, lds, turn);
        const float rstd = 1.0f / sqrtf(q[0] / (float)F + a.eps);
        for (int c = threadIdx.x; c < F; c += kWide) {
            const float w = a.w ? param_at<T>(a.w, a.w_f32, c) : 1.0f, b = a.b ? param_at<T>(a.b, a.w_f32, c) : 0.0f;
            y[c] = (T)__builtin_fmaf(((float)x[c] - mean) * rstd, w, b);
        }
        if (a.mean && threadIdx.x == 0) {
            a.mean[r] = mean;
            a.rstd[r] = rstd;
        }
    }
}

template <typename T>
__global__ __launch_bounds__(kWide) void layer_norm_bwd_wide_kernel(NormArgs a) {
    __shared__ float lds[kWide / 64 * 4];
    const int F = a.width;
    int turn = 0;
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T* x = (const T*)a.x + r * a.x_pitch;
        const T* dy = (const T*)a.dy + r * a.dy_pitch;
        T* dx = (T*)a.out + r * F;
        const float mean = a.mean[r], rstd = a.rstd[r];
        float s[2] = {0.0f, 0.0f};
        for (int c = threadIdx.x; c < F; c += kWide) {
            const float h = (float)dy[c] * (a.w ? param_at<T>(a.w, a.w_f32, c) : 1.0f);
            s[0] += h;
            s[1] = __builtin_fmaf(h, ((float)x[c] - mean) * rstd, s[1]);
        }
        row_sum<kWide, 2>(s, lds, turn);
        const float m1 = s[0] / (float)F, m2 = s[1] / (float)F;
        for (int c = threadIdx.x; c < F; c += kWide) {
            const float h = (float)dy[c] * (a.w ? param_at<T>(a.w, a.w_f32, c) : 1.0f);
            dx[c] = (T)(rstd * (h - m1 - ((float)x[c] - mean) * rstd * m2));
        }
    }
}

// dw and db partials of wide rows: a thread per column, a row slice per blockIdx.y
template <typename T>
__global__ __launch_bounds__(256) void layer_norm_cols_kernel(NormArgs a, int64_t slice) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= a.width) return;
    const int64_t lo = (int64_t)blockIdx.y * slice, hi = min(lo + slice, a.rows);
    float dw = 0.0f, db = 0.0f, dwc = 0.0f, dbc = 0.0f;
    for (int64_t r = lo; r < hi; ++r) {
        const float g = (float)((const T*)a.dy)[r * a.dy_pitch + c];
        const float xh = ((float)((const T*)a.x)[r * a.x_pitch + c] - a.mean[r]) * a.rstd[r];
        add_to<true>(dw, dwc, g * xh);
        add_to<true>(db, dbc, g);
    }
    float* p = a.part + (int64_t)blockIdx.y * 2 * a.width;
    p[c] = dw;
    p[(int64_t)a.width + c] = db;
}

// out[c] = sum over p of part[p][c], c over dw's columns then db's: 16 columns x 64 row slices a
// workgroup, the slices joined in order
template <typename T>
__global__ __launch_bounds__(1024) void layer_norm_reduce_kernel(const float* part, int n_part, int32_t width, T* dw,
                                                                  T* db, float* dw32, float* db32) {
    __shared__ double s[64][17];
    const int64_t cols = 2 * (int64_t)width;
    const int64_t c = (int64_t)blockIdx.x * 16 + threadIdx.x % 16;
    const int slice = threadIdx.x / 16;
    double v = 0.0;
    if (c < cols) {
#pragma unroll 8
        for (int p = slice; p < n_part; p += 64) v += (double)part[(int64_t)p * cols + c];
    }
    s[slice][threadIdx.x % 16] = v;
    __syncthreads();
    if (slice || c >= cols) return;
    for (int k = 1; k < 64; ++k) v += s[k][threadIdx.x % 16];
    const int64_t col = c < width ? c : c - width;
    T* o = c < width ? dw : db;
    float* o32 = c < width ? dw32 : db32;
    if (o) o[col] = (T)(float)v;
    if (o32) o32[col] = (float)v;
}

// Workgroups, and with them partial rows, of a backward: eight per CU as long as the partial rows, written
// and read once in fp32, are at most a tenth of the traffic of x, dy and dx.
int64_t norm_partials(int64_t rows, int eb) { return std::max<int64_t>(256, std::min<int64_t>(2048, rows * eb / 54)); }

template <typename T, int TPR, int NV, bool WHOLE>
void launch_rows(const NormArgs& a, bool bwd, int max_blocks, hipStream_t strm) {
    using S = RowShape<TPR>;
    constexpr int V = 16 / sizeof(T);
    const int blocks = (int)std::min<int64_t>(max_blocks, (a.rows + S::rows - 1) / S::rows);
    if (bwd)
        hipLaunchKernelGGL((layer_norm_bwd_kernel<T, V, TPR, NV, WHOLE>), dim3(blocks), dim3(S::threads), 0, strm, a);
    else
        hipLaunchKernelGGL((layer_norm_fwd_kernel<T, V, TPR, NV, WHOLE>), dim3(blocks), dim3(S::threads), 0, strm, a);
}

// The narrowest team of threads that holds a row of `vecs` vectors, at most 2,048.
template <typename T, bool WHOLE>
void launch_by_width(const NormArgs& a, int vecs, bool bwd, int max_blocks, hipStream_t strm) {
    if (vecs <= 16) launch_rows<T, 16, 1, WHOLE>(a, bwd, max_blocks, strm);
    else if (vecs <= 32) launch_rows<T, 32, 1, WHOLE>(a, bwd, max_blocks, strm);
    else if (vecs <= 64) launch_rows<T, 64, 1, WHOLE>(a, bwd, max_blocks, strm);
    else if (vecs <= 128) launch_rows<T, 64, 2, WHOLE>(a, bwd, max_blocks, strm);
    else if (vecs <= 256) launch_rows<T, 256, 1, WHOLE>(a, bwd, max_blocks, strm);
    else if (vecs <= 512) launch_rows<T, 256, 2, WHOLE>(a, bwd, max_blocks, strm);
    else if (vecs <= 1024) launch_rows<T, 256, 4, WHOLE>(a, bwd, max_blocks, strm);
    else launch_rows<T, 1024, 2, WHOLE>(a, bwd, max_blocks, strm);
}

template <typename T>
int row_vecs(const NormArgs& a) { return (a.width + 16 / (int)sizeof(T) - 1) / (16 / (int)sizeof(T)); }

bool vec_ok(const NormArgs& a, int eb) {
    const int v = 16 / eb;
    return a.width % v == 0 && a.x_pitch % v == 0 && a.dy_pitch % v == 0 && aligned16(a.x) && aligned16(a.dy) &&
           aligned16(a.out);
}

template <typename T>
int32_t norm_fwd(const NormArgs& a, hipStream_t strm) {
    constexpr int max_blocks = 256 * 8;
    const int vecs = row_vecs<T>(a);
    if (vecs <= 2048) {
        if (vec_ok(a, sizeof(T))) launch_by_width<T, true>(a, vecs, false, max_blocks, strm);
        else launch_by_width<T, false>(a, vecs, false, max_blocks, strm);
    } else {
        hipLaunchKernelGGL(layer_norm_fwd_wide_kernel<T>, dim3((unsigned)std::min<int64_t>(a.rows, 1024)), dim3(kWide),
                           0, strm, a);
    }
    return launch_status("mpgnn_layer_norm_fwd: the launch failed");
}

template <typename T>
int32_t norm_bwd(const NormArgs& a, void* dw, void* db, hipStream_t strm) {
    int parts = 0;
    const int max_parts = (int)norm_partials(a.rows, sizeof(T));
    const int vecs = row_vecs<T>(a);
    const int rows_per = vecs <= 16 ? 16 : vecs <= 32 ? 8 : vecs <= 128 ? 4 : 1;
    if (a.rows == 0) {  // no partial rows: the parameters' gradients are zero
    } else if (vecs <= 2048) {
        parts = (int)std::min<int64_t>(max_parts, (a.rows + rows_per - 1) / rows_per);
        if (vec_ok(a, sizeof(T))) launch_by_width<T, true>(a, vecs, true, max_parts, strm);
        else launch_by_width<T, false>(a, vecs, true, max_parts, strm);
    } else {
        if (a.out)
            hipLaunchKernelGGL(layer_norm_bwd_wide_kernel<T>, dim3((unsigned)std::min<int64_t>(a.rows, 1024)),
                               dim3(kWide), 0, strm, a);
        if (a.part) {
            const int64_t slice = (a.rows + max_parts - 1) / max_parts;
            parts = (int)((a.rows + slice - 1) / slice);
            hipLaunchKernelGGL(layer_norm_cols_kernel<T>, dim3((a.width + 255) / 256, parts), dim3(256), 0, strm, a,
                               slice);
        }
    }
    if (a.part) {
        T* w = a.w_f32 ? nullptr : (T*)dw;
        T* b = a.w_f32 ? nullptr : (T*)db;
        float* w32 = a.w_f32 ? (float*)dw : nullptr;
        float* b32 = a.w_f32 ? (float*)db : nullptr;
        hipLaunchKernelGGL(layer_norm_reduce_kernel<T>, dim3((unsigned)((2 * (int64_t)a.width + 15) / 16)), dim3(1024), 0,
                           strm, a.part, parts, a.width, w, b, w32, b32);
    }
    return launch_status("mpgnn_layer_norm_bwd: a launch failed");
}

int32_t check_norm(int64_t rows, int64_t width, int64_t pitch, int32_t dtype, int32_t wdtype) {
    if (rows < 0 || width <= 0 || (rows > 1 && pitch < width))
        return arg_error("layer norm: rows < 0, width < 1 or a row pitch below the width");
    if (!dtype_bytes(dtype)) return arg_error("layer norm: unknown dtype");
    if (wdtype != dtype && wdtype != MPGNN_F32)
        return arg_error("layer norm: weight and bias must have the input's type or fp32");
    if (width > (1 << 24)) return unsupported("layer norm: more than 2^24 columns");
    return MPGNN_OK;
}

}  // namespace
}  // namespace mpgnn

extern "C" int32_t mpgnn_layer_norm_fwd(const void* x, int64_t rows, int64_t width, int64_t x_pitch, int32_t dtype,
                                        const void* weight, const void* bias, int32_t wdtype, double eps, void* y,
                                        float* mean, float* rstd, void* stream) {
    using namespace mpgnn;
    int32_t st = check_norm(rows, width, x_pitch, dtype, wdtype);
    if (st != MPGNN_OK) return st;
    if (rows == 0) return MPGNN_OK;
    if (!x || !y || (mean == nullptr) != (rstd == nullptr))
        return arg_error("mpgnn_layer_norm_fwd: x or y is null, or one of mean and rstd alone");
    NormArgs a{};
    a.x = x; a.out = y; a.w = weight; a.b = bias; a.mean = mean; a.rstd = rstd;
    a.rows = rows; a.x_pitch = x_pitch; a.width = (int32_t)width; a.w_f32 = wdtype == MPGNN_F32; a.eps = (float)eps;
    hipStream_t strm = static_cast<hipStream_t>(stream);
    if (dtype == MPGNN_F32) return norm_fwd<float>(a, strm);
    return dtype == MPGNN_BF16 ? norm_fwd<__bf16>(a, strm) : norm_fwd<_Float16>(a, strm);
}

extern "C" int32_t mpgnn_layer_norm_bwd_workspace_bytes(int64_t rows, int64_t width, int64_t* bytes) {
    using namespace mpgnn;
    if (rows < 0 || width <= 0 || !bytes)
        return arg_error("mpgnn_layer_norm_bwd_workspace_bytes: bad shape or bytes is null");
    *bytes = std::min<int64_t>(rows, norm_partials(rows, 4)) * 2 * width * (int64_t)sizeof(float);
    return MPGNN_OK;
}

extern "C" int32_t mpgnn_layer_norm_bwd(const void* dy, int64_t dy_pitch, const void* x, int64_t x_pitch, int64_t rows,
                                        int64_t width, int32_t dtype, const void* weight, int32_t wdtype,
                                        const float* mean, const float* rstd, void* dx, void* dweight, void* dbias,
                                        void* workspace, void* stream) {
    using namespace mpgnn;
    int32_t st = check_norm(rows, width, x_pitch, dtype, wdtype);
    if (st != MPGNN_OK) return st;
    if (rows > 1 && dy_pitch < width) return arg_error("mpgnn_layer_norm_bwd: dy's row pitch is below the width");
    if ((dweight || dbias) && !workspace) return arg_error("mpgnn_layer_norm_bwd: no workspace");
    if (rows > 0 && (!x || !dy || !mean || !rstd)) return arg_error("mpgnn_layer_norm_bwd: a null input");
    if (!dx && !dweight && !dbias) return MPGNN_OK;
    NormArgs a{};
    a.x = x; a.dy = dy; a.out = dx; a.w = weight;
    a.mean = const_cast<float*>(mean); a.rstd = const_cast<float*>(rstd);
    a.part = dweight || dbias ? static_cast<float*>(workspace) : nullptr;
    a.rows = rows; a.x_pitch = x_pitch; a.dy_pitch = dy_pitch; a.width = (int32_t)width; a.w_f32 = wdtype == MPGNN_F32;
    hipStream_t strm = static_cast<hipStream_t>(stream);
    if (dtype == MPGNN_F32) return norm_bwd<float>(a, dweight, dbias, strm);
    return dtype == MPGNN_BF16 ? norm_bwd<__bf16>(a, dweight, dbias, strm) : norm_bwd<_Float16>(a, dweight, dbias, strm);
}
