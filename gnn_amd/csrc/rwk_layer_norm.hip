// Layer norm over the last dimension of a (rows, width) matrix and its backward pass:
//
//   h = (x - mean) * rstd,  y = h * w + b,      mean, var of the row, rstd = 1 / sqrt(var + eps)
//   dx = rstd * (t - mean(t) - h * mean(t * h)),  t = dy * w;      dw = sum_rows dy * h,  db = sum_rows dy
//
// Both passes are bound by memory: the forward reads and writes each element once, the backward reads x and dy and
// writes dx.  A row stays in the registers of the lanes that share it between its statistics and its output (the
// variance is the mean of squared distances from the mean, not a difference of two large sums).  The sum of a row is
// rounded on its way, so that its mean is off by a few roundings of x, which the distances of a row of nearly equal
// values do not forgive; the sum of these distances says by how much, and comes with the sum of their squares.  All
// arithmetic is fp32, one rounding to the element type at the store.
#include "rwk_vec.h"

// Every product and sum is rounded by itself, as the formula is written: the gradient of rows of two elements is what
// is left of equal terms, and a fused step on one side only would be most of it.
#pragma clang fp contract(off)

namespace {

constexpr int kBlock = 256;
constexpr int kWaves = kBlock / RWK_WAVE;

// Sums over the TPR threads that share a row (a part of a wavefront, a wavefront or the workgroup), to all of them.
// `red` holds kWaves entries and is used by workgroup-wide rows only; the callers alternate between two of them, which
// saves the barrier after the reads.
template <int TPR>
__device__ inline float row_sum(float v, float *red) {
    if (TPR <= RWK_WAVE) return rwk_group_sum(v, TPR);
    v = rwk_wave_sum(v);
    if ((threadIdx.x & (RWK_WAVE - 1)) == 0) red[threadIdx.x / RWK_WAVE] = v;
    __syncthreads();
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) s += red[w];
    return s;
}

template <int TPR>
__device__ inline void row_sums(float &a, float &c, float2 *red) {
    if (TPR <= RWK_WAVE) {
        a = rwk_group_sum(a, TPR);
        c = rwk_group_sum(c, TPR);
        return;
    }
    a = rwk_wave_sum(a);
    c = rwk_wave_sum(c);
    if ((threadIdx.x & (RWK_WAVE - 1)) == 0) red[threadIdx.x / RWK_WAVE] = make_float2(a, c);
    __syncthreads();
    a = c = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        a += red[w].x;
        c += red[w].y;
    }
}

// The V * IT elements of a row that thread t of TPR holds: vectors t, t + TPR, ...  Beyond the row: zeros.
template <typename T, int V, int IT>
struct Row {
    typename RwkPack<T, V>::type v[IT];
    __device__ float at(int i) const { return (float)v[i / V][i % V]; }
};

template <int TPR, typename T, int V, int IT>
__device__ inline void load_row(const T *__restrict__ row, int width, int t, Row<T, V, IT> &out) {
#pragma unroll
    for (int i = 0; i < IT; ++i) {
        const int c = (t + i * TPR) * V;
        if (c + V <= width) {
            out.v[i] = rwk_load<T, V>(row + c);
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) out.v[i][j] = c + j < width ? row[c + j] : (T)0.f;
        }
    }
}

template <typename T, int TPR, int V, int IT>
__device__ inline void store_row(T *__restrict__ row, int width, int t, const float (&in)[IT * V]) {
#pragma unroll
    for (int i = 0; i < IT; ++i) {
        const int c = (t + i * TPR) * V;
        if (c + V <= width) {
            typename RwkPack<T, V>::type v;
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] = (T)in[i * V + j];
            rwk_store<T, V>(row + c, v);
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (c + j < width) row[c + j] = (T)in[i * V + j];
        }
    }
}

// What is left of a row's mean and its variance from the sums of the distances from the mean and of their squares.  Equal
// values: distances of a small whole number of x's roundings, whose sums are exact, so both come out exact too.  Up to
// two elements the mean itself is rounded once only, and the distances are all there is.
struct Spread { float shift, var; };
__device__ inline Spread spread(float sum, float squares, int width) {
    const float shift = width > 2 ? sum / (float)width : 0.f, rest = squares - sum * shift;
    return {shift, (rest < 0.f ? 0.f : rest) / (float)width};
}

template <typename T, typename W, int TPR, int V, int IT>
__global__ void __launch_bounds__(kBlock)
norm_forward_kernel(const T *__restrict__ x, long long x_stride, const W *__restrict__ weight,
                    const W *__restrict__ bias, long long rows, int width, float eps, T *__restrict__ y,
                    float *__restrict__ mean_out, float *__restrict__ rstd_out) {
    __shared__ float red[kWaves];
    __shared__ float2 red2[kWaves];
    constexpr int kRows = kBlock / TPR;
    const int t = threadIdx.x % TPR;
    const long long step = (long long)gridDim.x * kRows;
    Row<W, V, IT> w, b;
    load_row<TPR>(weight, width, t, w);
    if (bias != nullptr) load_row<TPR>(bias, width, t, b);
    // the next row is on its way while this one is summed
    long long r = (long long)blockIdx.x * kRows + threadIdx.x / TPR;
    Row<T, V, IT> next;
    load_row<TPR>(x + (r < rows ? r : rows - 1) * x_stride, width, t, next);
    for (; r - threadIdx.x / TPR < rows; r += step) {       // the whole workgroup takes part in the sums
        const bool there = r < rows;
        float v[IT * V], s = 0.f;
#pragma unroll
        for (int i = 0; i < IT * V; ++i) {
            v[i] = next.at(i);
            s += v[i];
        }
        if (r + step - threadIdx.x / TPR < rows)
            load_row<TPR>(x + (r + step < rows ? r + step : rows - 1) * x_stride, width, t, next);
        const float mean = row_sum<TPR>(s, red) / (float)width;
        float q = 0.f;
        s = 0.f;
#pragma unroll
        for (int i = 0; i < IT * V; ++i) {
            v[i] = (t + i / V * TPR) * V + i % V < width ? v[i] - mean : 0.f;
            s += v[i];
            q += v[i] * v[i];
        }
        row_sums<TPR>(s, q, red2);
        const Spread by = spread(s, q, width);
        const float rstd = 1.f / sqrtf(by.var + eps);
#pragma unroll
        for (int i = 0; i < IT * V; ++i) {
            v[i] = (v[i] - by.shift) * rstd * w.at(i);
            if (bias != nullptr) v[i] += b.at(i);
        }
        if (!there) continue;
        store_row<T, TPR, V, IT>(y + r * width, width, t, v);
        if (t == 0 && mean_out != nullptr) {
            mean_out[r] = mean + by.shift;
            rstd_out[r] = rstd;
        }
    }
}

// dx of the workgroup's rows and its sums of dy * h and dy over them: one row [dw | db] of `partials` per workgroup.
template <typename T, typename W, int TPR, int V, int IT>
__global__ void __launch_bounds__(kBlock)
norm_backward_kernel(const T *__restrict__ x, long long x_stride, const T *__restrict__ dy, long long dy_stride,
                     const W *__restrict__ weight, const float *__restrict__ mean_in,
                     const float *__restrict__ rstd_in, long long rows, int width, T *__restrict__ dx,
                     float *__restrict__ partials) {
    constexpr int kRows = kBlock / TPR;
    __shared__ float2 red[2][kWaves];
    const int t = threadIdx.x % TPR;
    const long long step = (long long)gridDim.x * kRows;
    const float inv = 1.f / (float)width;
    Row<W, V, IT> w;
    load_row<TPR>(weight, width, t, w);
    float dw[IT * V], db[IT * V];
#pragma unroll
    for (int i = 0; i < IT * V; ++i) dw[i] = db[i] = 0.f;
    // the next row is on its way while this one is summed
    Row<T, V, IT> x_next, g_next;
    float mean_next, rstd_next;
    const auto fetch = [&](long long r) {
        const long long rc = r < rows ? r : rows - 1;
        load_row<TPR>(x + rc * x_stride, width, t, x_next);
        load_row<TPR>(dy + rc * dy_stride, width, t, g_next);
        mean_next = mean_in[rc];
        rstd_next = rstd_in[rc];
    };
    long long r = (long long)blockIdx.x * kRows + threadIdx.x / TPR;
    fetch(r);
    for (int turn = 0; r - threadIdx.x / TPR < rows; r += step, turn ^= 1) {
        const Row<T, V, IT> xr = x_next, gr = g_next;
        const float mean = mean_next, rstd = rstd_next;
        const bool there = r < rows;
        if (r + step - threadIdx.x / TPR < rows) fetch(r + step);
        float h[IT * V], g[IT * V], a = 0.f, c = 0.f;
#pragma unroll
        for (int i = 0; i < IT * V; ++i) {
            h[i] = (xr.at(i) - mean) * rstd;              // beyond the row: dy = 0 and w = 0 take it out
            g[i] = gr.at(i);
            if (there) {
                dw[i] += g[i] * h[i];
                db[i] += g[i];
            }
            g[i] *= w.at(i);
            a += g[i];
            c += g[i] * h[i];
        }
        row_sums<TPR>(a, c, red[turn]);
        a *= inv;
        c *= inv;
#pragma unroll
        for (int i = 0; i < IT * V; ++i) h[i] = rstd * (g[i] - a - h[i] * c);
        if (there) store_row<T, TPR, V, IT>(dx + r * width, width, t, h);
    }
    float *out = partials + (long long)blockIdx.x * 2 * width;
    if (TPR == kBlock) {
        store_row<float, TPR, V, IT>(out, width, t, dw);
        store_row<float, TPR, V, IT>(out + width, width, t, db);
    } else {
        // the workgroup's kRows row slots in slot order
        __shared__ float sums[kBlock * V];
#pragma unroll
        for (int k = 0; k < 2 * IT; ++k) {
            __syncthreads();
#pragma unroll
            for (int j = 0; j < V; ++j)
                sums[threadIdx.x * V + j] = k < IT ? dw[(k % IT) * V + j] : db[(k % IT) * V + j];
            __syncthreads();
            for (int e = threadIdx.x; e < TPR * V; e += kBlock) {
                float s = 0.f;
                for (int q = 0; q < kRows; ++q) s += sums[q * TPR * V + e];
                const int col = (k % IT) * TPR * V + e;
                if (col < width) out[(k < IT ? 0 : width) + col] = s;
            }
        }
    }
}

// Rows too wide for registers: the same sums in three passes over the row, which the second and third find in the
// cache of the compute unit's die.
template <typename T, typename W>
__global__ void __launch_bounds__(kBlock)
norm_forward_wide_kernel(const T *__restrict__ x, long long x_stride, const W *__restrict__ weight,
                         const W *__restrict__ bias, int width, float eps, T *__restrict__ y,
                         float *__restrict__ mean_out, float *__restrict__ rstd_out) {
    __shared__ float red[kWaves];
    __shared__ float2 red2[kWaves];
    const long long r = blockIdx.x;
    const T *row = x + r * x_stride;
    float s = 0.f;
    for (int c = threadIdx.x; c < width; c += kBlock) s += (float)row[c];
    const float mean = row_sum<kBlock>(s, red) / (float)width;
    float q = 0.f;
    s = 0.f;
    for (int c = threadIdx.x; c < width; c += kBlock) {
        const float d = (float)row[c] - mean;
        s += d;
        q += d * d;
    }
    row_sums<kBlock>(s, q, red2);
    const Spread by = spread(s, q, width);
    const float rstd = 1.f / sqrtf(by.var + eps);
    for (int c = threadIdx.x; c < width; c += kBlock)
        y[r * width + c] = (T)(((float)row[c] - mean - by.shift) * rstd * (float)weight[c] + (bias != nullptr ? (float)bias[c] : 0.f));
    if (threadIdx.x == 0 && mean_out != nullptr) {
        mean_out[r] = mean + by.shift;
        rstd_out[r] = rstd;
    }
}

template <typename T, typename W>
__global__ void __launch_bounds__(kBlock)
norm_backward_wide_kernel(const T *__restrict__ x, long long x_stride, const T *__restrict__ dy, long long dy_stride,
                          const W *__restrict__ weight, const float *__restrict__ mean_in,
                          const float *__restrict__ rstd_in, int width, T *__restrict__ dx) {
    __shared__ float red[2][kWaves];
    const long long r = blockIdx.x;
    const T *row = x + r * x_stride, *grad = dy + r * dy_stride;
    const float mean = mean_in[r], rstd = rstd_in[r];
    float a = 0.f, c = 0.f;
    for (int i = threadIdx.x; i < width; i += kBlock) {
        const float t = (float)grad[i] * (float)weight[i];
        a += t;
        c += t * (((float)row[i] - mean) * rstd);
    }
    a = row_sum<kBlock>(a, red[0]) / (float)width;
    c = row_sum<kBlock>(c, red[1]) / (float)width;
    for (int i = threadIdx.x; i < width; i += kBlock)
        dx[r * width + i] = (T)(rstd * ((float)grad[i] * (float)weight[i] - a - ((float)row[i] - mean) * rstd * c));
}

// [dw | db] partials of wide rows: workgroup (column block, row split)
template <typename T>
__global__ void __launch_bounds__(kBlock)
norm_weight_wide_kernel(const T *__restrict__ x, long long x_stride, const T *__restrict__ dy, long long dy_stride,
                        const float *__restrict__ mean_in, const float *__restrict__ rstd_in, long long rows,
                        int width, float *__restrict__ partials) {
    const int c = blockIdx.x * kBlock + threadIdx.x;
    if (c >= width) return;
    float dw = 0.f, db = 0.f;
    for (long long r = blockIdx.y; r < rows; r += gridDim.y) {
        const float g = (float)dy[r * dy_stride + c];
        dw += g * (((float)x[r * x_stride + c] - mean_in[r]) * rstd_in[r]);
        db += g;
    }
    float *out = partials + (long long)blockIdx.y * 2 * width;
    out[c] = dw;
    out[width + c] = db;
}

// dw, db = column sums of the partial rows [dw | db], in row order within 32 fixed groups, then in group order
constexpr int kSumCols = 32, kSumGroups = 32;
template <typename W>
__global__ void __launch_bounds__(kSumCols * kSumGroups)
norm_weight_sum_kernel(const float *__restrict__ partials, int n_partials, int width, W *__restrict__ dw,
                       W *__restrict__ db) {
    __shared__ float part[kSumGroups][kSumCols];
    const int lane = threadIdx.x % kSumCols, group = threadIdx.x / kSumCols;
    const long long c = (long long)blockIdx.x * kSumCols + lane;
    float s = 0.f;
    if (c < 2ll * width)
#pragma unroll 16
        for (int p = group; p < n_partials; p += kSumGroups) s += partials[(long long)p * 2 * width + c];
    part[group][lane] = s;
    __syncthreads();
    if (group != 0 || c >= 2ll * width) return;
    for (int g = 1; g < kSumGroups; ++g) s += part[g][lane];
    if (c < width) {
        dw[c] = (W)s;
    } else if (db != nullptr) {
        db[c - width] = (W)s;
    }
}

// ---------------------------------------------------------------------------------------------------------------
// Launch shapes.  Threads per row: as few as hold the row in one vector each up to a wavefront, so that narrow rows
// (node features of a few channels) still fill every lane; wider rows give each lane of a wavefront, then of a
// workgroup, more vectors.  A wavefront alone needs no barrier: up to 256 vectors it is at least as fast as a workgroup
// (65536 x 1024 bf16 forward 44 us = 6.1 TB/s; 40000 x 2048 fp16 58), at 512 its registers leave too few rows in flight
// (32768 x 4096 bf16: 148 us, by workgroups 98 = 5.5 TB/s).  The backward pass keeps two column sums per element besides
// the row and turns to the workgroup at 128.  A large copy runs at 5.1 TB/s on the same card.
// Workgroups are few enough to stay resident and walk over the rows.  In the backward pass each also leaves a row of
// partial sums: 512 of them are faster than 1024 for workgroup-wide rows (32768 x 4096 bf16: 150 + 5 us against
// 169 + 8), but not for rows at odd addresses, whose loads take longer (16384 x 2001: 82 against 63) and narrow ones.
// ---------------------------------------------------------------------------------------------------------------
constexpr int kWideSplit = 64;

constexpr int kRegisterWidth = 8192;    // wider rows do not fit a workgroup's registers

int row_threads(int64_t vectors) {         // of the backward pass
    return vectors <= 4 ? 4 : vectors <= 8 ? 8 : vectors <= 16 ? 16 : vectors <= 32 ? 32 : vectors <= 128 ? 64 : 256;
}

int64_t backward_blocks(int64_t rows, int64_t width, int vec) {
    if (width > kRegisterWidth) return rows < kWideSplit ? rows : kWideSplit;
    const int threads = row_threads(rwk_ceil_div(width, vec));
    const int64_t blocks = rwk_ceil_div(rows, kBlock / threads), most = threads == kBlock && width % vec == 0 ? 512 : 1024;
    return blocks < most ? blocks : most;
}

struct NormArgs : rwk_layer_norm {
    hipStream_t stream;
};

template <typename T, typename W, int TPR, int IT>
int launch_forward(const NormArgs &a) {
    constexpr int V = RwkVecOf<T>::n;
    long long grid = rwk_ceil_div(a.rows, kBlock / TPR);
    constexpr long long kMost = TPR < RWK_WAVE ? 4096 : 2048;
    if (grid > kMost) grid = kMost;
    hipLaunchKernelGGL((norm_forward_kernel<T, W, TPR, V, IT>), dim3((unsigned)grid), dim3(kBlock), 0, a.stream,
                       (const T *)a.x, (long long)a.x_stride, (const W *)a.weight, (const W *)a.bias, (long long)a.rows, (int)a.width, a.eps,
                       (T *)a.y, a.mean, a.rstd);
    RWK_LAUNCH_CHECK();
    return RWK_OK;
}

template <typename T, typename W>
int forward(const NormArgs &a) {
    constexpr int V = RwkVecOf<T>::n;
    const int64_t vectors = rwk_ceil_div(a.width, V);
    if (vectors <= 4) return launch_forward<T, W, 4, 1>(a);
    if (vectors <= 8) return launch_forward<T, W, 8, 1>(a);
    if (vectors <= 16) return launch_forward<T, W, 16, 1>(a);
    if (vectors <= 32) return launch_forward<T, W, 32, 1>(a);
    if (vectors <= 64) return launch_forward<T, W, 64, 1>(a);
    if (vectors <= 128) return launch_forward<T, W, 64, 2>(a);
    if (vectors <= 256) return launch_forward<T, W, 64, 4>(a);
    if (vectors <= 512) return launch_forward<T, W, 256, 2>(a);
    if (vectors <= 1024) return launch_forward<T, W, 256, 4>(a);
    if (vectors <= 2048 && V == 4) return launch_forward<T, W, 256, 8>(a);
    if (a.rows > 0x7FFFFFFFll) return RWK_E_SIZE;
    hipLaunchKernelGGL((norm_forward_wide_kernel<T, W>), dim3((unsigned)a.rows), dim3(kBlock), 0, a.stream,
                       (const T *)a.x, (long long)a.x_stride, (const W *)a.weight, (const W *)a.bias, (int)a.width, a.eps, (T *)a.y,
                       a.mean, a.rstd);
    RWK_LAUNCH_CHECK();
    return RWK_OK;
}

template <typename T, typename W, int TPR, int IT>
int launch_backward(const NormArgs &a, int64_t blocks) {
    constexpr int V = RwkVecOf<T>::n;
    hipLaunchKernelGGL((norm_backward_kernel<T, W, TPR, V, IT>), dim3((unsigned)blocks), dim3(kBlock), 0, a.stream,
                       (const T *)a.x, (long long)a.x_stride, (const T *)a.dy, (long long)a.dy_stride, (const W *)a.weight, a.mean, a.rstd,
                       (long long)a.rows, (int)a.width, (T *)a.dx, a.partials);
    RWK_LAUNCH_CHECK();
    return RWK_OK;
}

template <typename T, typename W>
int backward(const NormArgs &a) {
    constexpr int V = RwkVecOf<T>::n;
    const int64_t vectors = rwk_ceil_div(a.width, V);
    const int64_t blocks = backward_blocks(a.rows, a.width, V);
    int code = RWK_OK;
    if (a.width > kRegisterWidth) {
        if (a.rows > 0x7FFFFFFFll) return RWK_E_SIZE;
        hipLaunchKernelGGL((norm_backward_wide_kernel<T, W>), dim3((unsigned)a.rows), dim3(kBlock), 0, a.stream,
                           (const T *)a.x, (long long)a.x_stride, (const T *)a.dy, (long long)a.dy_stride, (const W *)a.weight, a.mean,
                           a.rstd, (int)a.width, (T *)a.dx);
        RWK_LAUNCH_CHECK();
        hipLaunchKernelGGL((norm_weight_wide_kernel<T>), dim3((unsigned)rwk_ceil_div(a.width, kBlock), (unsigned)blocks),
                           dim3(kBlock), 0, a.stream, (const T *)a.x, (long long)a.x_stride, (const T *)a.dy, (long long)a.dy_stride, a.mean,
                           a.rstd, (long long)a.rows, (int)a.width, a.partials);
        RWK_LAUNCH_CHECK();
    } else if (vectors <= 4) {
        code = launch_backward<T, W, 4, 1>(a, blocks);
    } else if (vectors <= 8) {
        code = launch_backward<T, W, 8, 1>(a, blocks);
    } else if (vectors <= 16) {
        code = launch_backward<T, W, 16, 1>(a, blocks);
    } else if (vectors <= 32) {
        code = launch_backward<T, W, 32, 1>(a, blocks);
    } else if (vectors <= 64) {
        code = launch_backward<T, W, 64, 1>(a, blocks);
    } else if (vectors <= 128) {
        code = launch_backward<T, W, 64, 2>(a, blocks);
    } else if (vectors <= 256) {
        code = launch_backward<T, W, 256, 1>(a, blocks);
    } else if (vectors <= 512) {
        code = launch_backward<T, W, 256, 2>(a, blocks);
    } else if (vectors <= 1024) {
        code = launch_backward<T, W, 256, 4>(a, blocks);
    } else {
        code = launch_backward<T, W, 256, V == 4 ? 8 : 4>(a, blocks);     // fp32 rows of 4097 to 8192
    }
    if (code != RWK_OK) return code;
    hipLaunchKernelGGL((norm_weight_sum_kernel<W>), dim3((unsigned)rwk_ceil_div(2ll * a.width, kSumCols)),
                       dim3(kSumCols * kSumGroups), 0, a.stream, a.partials, (int)blocks, (int)a.width, (W *)a.dw,
                       (W *)a.db);
    RWK_LAUNCH_CHECK();
    return RWK_OK;
}

int check(const rwk_layer_norm &a, bool backward) {
    RWK_REQUIRE_PTR(a.x);
    RWK_REQUIRE_PTR(a.weight);
    if (a.type < RWK_F32 || a.type > RWK_BF16 || (a.weight_type != a.type && a.weight_type != RWK_F32))
        return RWK_E_UNSUPPORTED;
    if (a.rows <= 0 || a.width <= 0 || a.width > 0x3FFFFFFF || a.x_stride < a.width) return RWK_E_SIZE;
    if (!backward) {
        RWK_REQUIRE_PTR(a.y);
        return (a.mean == nullptr) != (a.rstd == nullptr) ? RWK_E_NULL : RWK_OK;
    }
    RWK_REQUIRE_PTR(a.dy);
    RWK_REQUIRE_PTR(a.dx);
    RWK_REQUIRE_PTR(a.mean);
    RWK_REQUIRE_PTR(a.rstd);
    RWK_REQUIRE_PTR(a.partials);
    RWK_REQUIRE_PTR(a.dw);
    return a.dy_stride < a.width ? RWK_E_SIZE : RWK_OK;
}

}  // namespace

extern "C" {

int64_t rwk_layer_norm_backward_blocks(int64_t rows, int64_t width, int32_t type) {
    if (rows <= 0 || width <= 0 || width > 0x3FFFFFFF) return 0;
    return backward_blocks(rows, width, type == RWK_F32 ? 4 : 8);
}

int rwk_layer_norm_forward(const rwk_layer_norm *args, rwk_stream_t stream) {
    RWK_REQUIRE_PTR(args);
    const int code = check(*args, false);
    if (code != RWK_OK) return code;
    const NormArgs a{*args, (hipStream_t)stream};
    const bool wide = a.weight_type == RWK_F32;
    if (a.type == RWK_F32) return forward<float, float>(a);
    if (a.type == RWK_F16) return wide ? forward<rwk_f16, float>(a) : forward<rwk_f16, rwk_f16>(a);
    return wide ? forward<rwk_bf16, float>(a) : forward<rwk_bf16, rwk_bf16>(a);
}

int rwk_layer_norm_backward(const rwk_layer_norm *args, rwk_stream_t stream) {
    RWK_REQUIRE_PTR(args);
    const int code = check(*args, true);
    if (code != RWK_OK) return code;
    const NormArgs a{*args, (hipStream_t)stream};
    const bool wide = a.weight_type == RWK_F32;
    if (a.type == RWK_F32) return backward<float, float>(a);
    if (a.type == RWK_F16) return wide ? backward<rwk_f16, float>(a) : backward<rwk_f16, rwk_f16>(a);
    return wide ? backward<rwk_bf16, float>(a) : backward<rwk_bf16, rwk_bf16>(a);
}

}  // extern "C"
