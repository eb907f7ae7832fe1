// Entry points of the attention inside packed segments, the reduction of the bias gradient and the kernels that lay
// out the bucket codes of the pairs.  The attention kernels themselves: rwk_attention_body.h.
#include "rwk_attention.h"
#include "rwk_vec.h"

namespace {

constexpr int kBlock = 256;

// d_table[h][b] = sum over the blocks of rows, one workgroup per entry, in a fixed order
template <typename T>
__global__ void __launch_bounds__(kBlock)
bias_sum_kernel(const float *__restrict__ partials, long long n_items, T *__restrict__ d_table) {
    __shared__ float part[kBlock / RWK_WAVE];
    const float *row = partials + (long long)blockIdx.x * n_items;
    float s = 0.f;
    for (long long i = threadIdx.x; i < n_items; i += kBlock) s += row[i];
    s = rwk_wave_sum(s);
    if ((threadIdx.x & (RWK_WAVE - 1)) == 0) part[threadIdx.x / RWK_WAVE] = s;
    __syncthreads();
    if (threadIdx.x == 0) d_table[blockIdx.x] = (T)(part[0] + part[1] + part[2] + part[3]);
}

int bias_sum(const rwk_attention &a, hipStream_t stream) {
    const dim3 grid((unsigned)(a.heads * a.n_buckets));
    if (a.type == RWK_F32)
        hipLaunchKernelGGL(bias_sum_kernel<float>, grid, dim3(kBlock), 0, stream, a.d_table_partials,
                           (long long)a.n_items, (float *)a.d_table);
    else if (a.type == RWK_F16)
        hipLaunchKernelGGL(bias_sum_kernel<rwk_f16>, grid, dim3(kBlock), 0, stream, a.d_table_partials,
                           (long long)a.n_items, (rwk_f16 *)a.d_table);
    else
        hipLaunchKernelGGL(bias_sum_kernel<rwk_bf16>, grid, dim3(kBlock), 0, stream, a.d_table_partials,
                           (long long)a.n_items, (rwk_bf16 *)a.d_table);
    RWK_LAUNCH_CHECK();
    return RWK_OK;
}

int check(const rwk_attention *a, bool backward) {
    RWK_REQUIRE_PTR(a);
    if (a->type < RWK_F32 || a->type > RWK_BF16) return RWK_E_UNSUPPORTED;
    if (a->heads < 1 || a->kv_heads < 1 || a->heads % a->kv_heads != 0 || a->dim < 1 || a->rows < 0 ||
        a->rows >= 0x7FFFFFFFll || a->n_segments < 0 || a->n_items < 0 || a->n_buckets < 0)
        return RWK_E_SIZE;
    if (a->dim > 128 || a->n_buckets > 32 || (a->block_rows != 32 && a->block_rows != 128)) return RWK_E_UNSUPPORTED;
    if (!(a->scale > 0.f) || a->n_items > 0x7FFFFFFFll / a->heads) return RWK_E_SIZE;
    if (a->n_buckets > 0) {
        RWK_REQUIRE_PTR(a->table);
        if (backward) {
            RWK_REQUIRE_PTR(a->d_table);
            if (a->n_items > 0) RWK_REQUIRE_PTR(a->d_table_partials);
        }
    }
    if (a->n_items == 0) return RWK_OK;
    RWK_REQUIRE_PTR(a->q);
    RWK_REQUIRE_PTR(a->k);
    RWK_REQUIRE_PTR(a->v);
    RWK_REQUIRE_PTR(a->out);
    RWK_REQUIRE_PTR(a->seg_ptr);
    RWK_REQUIRE_PTR(a->q_items);
    if (a->n_buckets > 0) {
        RWK_REQUIRE_PTR(a->codes);
        RWK_REQUIRE_PTR(a->code_start);
    }
    if (backward) {
        RWK_REQUIRE_PTR(a->d_out);
        RWK_REQUIRE_PTR(a->dq);
        RWK_REQUIRE_PTR(a->dk);
        RWK_REQUIRE_PTR(a->dv);
        RWK_REQUIRE_PTR(a->stats);
        RWK_REQUIRE_PTR(a->delta);
        RWK_REQUIRE_PTR(a->k_items);
    }
    return RWK_OK;
}

int launch(RwkAttnPass pass, const rwk_attention &a, const int32_t *items, hipStream_t stream) {
    RwkAttnArgs p;
    p.a = a;
    p.items = items;
    p.group = (int)(a.heads / a.kv_heads);
    if (a.type == RWK_F32) return rwk_attention_launch_f32(pass, p, stream);
    if (a.type == RWK_F16) return rwk_attention_launch_f16(pass, p, stream);
    return rwk_attention_launch_bf16(pass, p, stream);
}

// segment of a row: the last g with seg_ptr[g] <= row (segments without rows are passed over)
__device__ inline int segment_of(const int *__restrict__ seg_ptr, int n_segments, int row) {
    int lo = 0, hi = n_segments;                 // seg_ptr[lo] <= row < seg_ptr[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (seg_ptr[mid] <= row) lo = mid; else hi = mid;
    }
    return lo;
}

struct CodeRow {
    int g, i, n, padded;
    uint8_t *out;
};
__device__ inline CodeRow code_row(const int *seg_ptr, int n_segments, const int64_t *code_start, uint8_t *codes,
                                   int row) {
    CodeRow r;
    r.g = segment_of(seg_ptr, n_segments, row);
    r.i = row - seg_ptr[r.g];
    r.n = seg_ptr[r.g + 1] - seg_ptr[r.g];
    r.padded = (r.n + 31) / 32 * 32;
    r.out = codes + code_start[r.g] + (long long)r.i * r.padded;
    return r;
}

__global__ void __launch_bounds__(kBlock)
pair_dense_kernel(const uint8_t *__restrict__ dense, const int64_t *__restrict__ pair_start,
                  const int *__restrict__ seg_ptr, const int64_t *__restrict__ code_start, int n_segments,
                  uint8_t *__restrict__ codes) {
    const CodeRow r = code_row(seg_ptr, n_segments, code_start, codes, (int)blockIdx.x);
    const uint8_t *in = dense + pair_start[r.g] + (long long)r.i * r.n;
    for (int j = threadIdx.x; j < r.padded; j += kBlock) r.out[j] = j < r.n ? in[j] : 255;
}

__global__ void __launch_bounds__(kBlock)
pair_relative_kernel(const uint8_t *__restrict__ by_offset, int reach, const int *__restrict__ seg_ptr,
                     const int64_t *__restrict__ code_start, int n_segments, uint8_t *__restrict__ codes) {
    const CodeRow r = code_row(seg_ptr, n_segments, code_start, codes, (int)blockIdx.x);
    for (int j = threadIdx.x; j < r.padded; j += kBlock) {
        int d = j - r.i;
        d = d < -reach ? -reach : d > reach ? reach : d;
        r.out[j] = j < r.n ? by_offset[d + reach] : 255;
    }
}

__global__ void __launch_bounds__(kBlock)
pair_hops_kernel(const int *__restrict__ row_start, const int *__restrict__ col, const int *__restrict__ dist,
                 int far_code, const int *__restrict__ seg_ptr, const int64_t *__restrict__ code_start,
                 int n_segments, uint8_t *__restrict__ codes) {
    const int row = (int)blockIdx.x;
    const CodeRow r = code_row(seg_ptr, n_segments, code_start, codes, row);
    for (int j = threadIdx.x; j < r.padded; j += kBlock)
        r.out[j] = j == r.i ? 0 : j < r.n ? (uint8_t)far_code : 255;
    __syncthreads();                              // the listed pairs overwrite what other threads wrote
    for (int e = row_start[row] + threadIdx.x; e < row_start[row + 1]; e += kBlock) {
        const int j = col[e] - (row - r.i);
        if ((unsigned)j < (unsigned)r.n) r.out[j] = (uint8_t)dist[e];
    }
}

int check_codes(const int32_t *seg_ptr, const int64_t *code_start, int64_t n_segments, int64_t rows,
                const uint8_t *codes) {
    if (n_segments < 0 || n_segments >= 0x7FFFFFFFll || rows < 0 || rows >= 0x7FFFFFFFll) return RWK_E_SIZE;
    if (rows > 0 && n_segments < 1) return RWK_E_SIZE;
    if (rows == 0) return RWK_OK;
    RWK_REQUIRE_PTR(seg_ptr);
    RWK_REQUIRE_PTR(code_start);
    RWK_REQUIRE_PTR(codes);
    return RWK_OK;
}

}  // namespace

extern "C" {

int rwk_attention_forward(const rwk_attention *a, rwk_stream_t stream) {
    const int code = check(a, false);
    if (code != RWK_OK || a->n_items == 0) return code;
    return launch(kRwkAttnForward, *a, a->q_items, (hipStream_t)stream);
}

int rwk_attention_backward(const rwk_attention *a, rwk_stream_t stream) {
    int code = check(a, true);
    if (code != RWK_OK) return code;
    if (a->n_items > 0) {
        code = launch(kRwkAttnDq, *a, a->q_items, (hipStream_t)stream);       // leaves delta for the second launch
        if (code == RWK_OK) code = launch(kRwkAttnDkv, *a, a->k_items, (hipStream_t)stream);
        if (code != RWK_OK) return code;
    }
    return a->n_buckets > 0 ? bias_sum(*a, (hipStream_t)stream) : RWK_OK;
}

int rwk_pair_buckets_dense(const uint8_t *dense, const int64_t *pair_start, const int32_t *seg_ptr,
                           const int64_t *code_start, int64_t n_segments, int64_t rows, uint8_t *codes,
                           rwk_stream_t stream) {
    const int code = check_codes(seg_ptr, code_start, n_segments, rows, codes);
    if (code != RWK_OK || rows == 0) return code;
    RWK_REQUIRE_PTR(dense);
    RWK_REQUIRE_PTR(pair_start);
    hipLaunchKernelGGL(pair_dense_kernel, dim3((unsigned)rows), dim3(kBlock), 0, (hipStream_t)stream, dense,
                       pair_start, seg_ptr, code_start, (int)n_segments, codes);
    RWK_LAUNCH_CHECK();
    return RWK_OK;
}

int rwk_pair_buckets_relative(const uint8_t *by_offset, int64_t reach, const int32_t *seg_ptr,
                              const int64_t *code_start, int64_t n_segments, int64_t rows, uint8_t *codes,
                              rwk_stream_t stream) {
    const int code = check_codes(seg_ptr, code_start, n_segments, rows, codes);
    if (reach < 0 || reach > 0x3FFFFFFF) return RWK_E_SIZE;
    if (code != RWK_OK || rows == 0) return code;
    RWK_REQUIRE_PTR(by_offset);
    hipLaunchKernelGGL(pair_relative_kernel, dim3((unsigned)rows), dim3(kBlock), 0, (hipStream_t)stream, by_offset,
                       (int)reach, seg_ptr, code_start, (int)n_segments, codes);
    RWK_LAUNCH_CHECK();
    return RWK_OK;
}

int rwk_pair_buckets_hops(const int32_t *row_start, const int32_t *col, const int32_t *dist, int32_t far_code,
                          const int32_t *seg_ptr, const int64_t *code_start, int64_t n_segments, int64_t rows,
                          uint8_t *codes, rwk_stream_t stream) {
    const int code = check_codes(seg_ptr, code_start, n_segments, rows, codes);
    if (far_code < 0 || far_code > 255) return RWK_E_SIZE;
    if (code != RWK_OK || rows == 0) return code;
    RWK_REQUIRE_PTR(row_start);
    hipLaunchKernelGGL(pair_hops_kernel, dim3((unsigned)rows), dim3(kBlock), 0, (hipStream_t)stream, row_start, col,
                       dist, far_code, seg_ptr, code_start, (int)n_segments, codes);
    RWK_LAUNCH_CHECK();
    return RWK_OK;
}

}  // extern "C"
