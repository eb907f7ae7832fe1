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

// dK and dV from their parts, which lie 2 n elements apart, dV n behind dK: elements of the rows inside segments
template <typename T>
__global__ void __launch_bounds__(kBlock)
dkv_sum_kernel(const float *__restrict__ partials, int parts, long long n, const int *__restrict__ rows, long long width,
               T *__restrict__ dk, T *__restrict__ dv) {
    const long long end = *rows * width, i = ((long long)blockIdx.x * kBlock + threadIdx.x) * 4;
    if (i >= end) return;
    const float *from = partials + blockIdx.y * n + i;
    T *to = (blockIdx.y == 0 ? dk : dv) + i;
    if (i + 4 <= end) {
        auto sum = rwk_load<float, 4>(from);
        for (int part = 1; part < parts; ++part) sum += rwk_load<float, 4>(from + 2 * part * n);
        typename RwkPack<T, 4>::type v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (T)sum[e];
        rwk_store<T, 4>(to, v);
    } else {
        for (int e = 0; i + e < end; ++e) {
            float sum = from[e];
            for (int part = 1; part < parts; ++part) sum += from[2 * part * n + e];
            to[e] = (T)sum;
        }
    }
}

template <typename T>
int dkv_sum(const rwk_attention &a, hipStream_t stream) {
    const long long width = a.kv_heads * a.dim, n = a.rows * width;
    const dim3 grid((unsigned)rwk_ceil_div(n, 4 * kBlock), 2);
    hipLaunchKernelGGL(dkv_sum_kernel<T>, grid, dim3(kBlock), 0, stream, a.dkv_partials, (int)a.key_parts, n,
                       a.seg_ptr + a.n_segments, width, (T *)a.dk, (T *)a.dv);
    RWK_LAUNCH_CHECK();
    return RWK_OK;
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
    // scales whose reciprocal times log2(e) is a normal number, too
    if (!(a->scale >= 1e-30f && a->scale <= 1e30f) || a->n_items > 0x7FFFFFFFll / a->heads) return RWK_E_SIZE;
    if (a->key_parts < 0 || (a->key_parts > 1 && (a->heads / a->kv_heads % a->key_parts != 0 ||
                                                  a->rows > (1ll << 33) / a->kv_heads)))
        return RWK_E_SIZE;
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
        if (backward) RWK_REQUIRE_PTR(a->codes_by_key);
        if ((uintptr_t)a->codes % 16 != 0 || (uintptr_t)a->codes_by_key % 16 != 0) return RWK_E_ALIGN;
    }
    if (backward) {
        RWK_REQUIRE_PTR(a->d_out);
        RWK_REQUIRE_PTR(a->dq);
        RWK_REQUIRE_PTR(a->dk);
        RWK_REQUIRE_PTR(a->dv);
        RWK_REQUIRE_PTR(a->stats);
        RWK_REQUIRE_PTR(a->delta);
        RWK_REQUIRE_PTR(a->k_items);
        if (a->key_parts > 1) RWK_REQUIRE_PTR(a->dkv_partials);
    }
    return RWK_OK;
}

int launch(RwkAttnPass pass, const rwk_attention &a, const int32_t *items, hipStream_t stream) {
    RwkAttnArgs p;
    p.a = a;
    p.items = items;
    p.group = (int)(a.heads / a.kv_heads);
    p.parts = a.key_parts > 1 ? a.key_parts : 1;
    p.part_heads = p.group / p.parts;
    if (a.type == RWK_F32) return rwk_attention_launch_f32(pass, p, stream);
    if (a.type == RWK_F16) return rwk_attention_launch_f16(pass, p, stream);
    return rwk_attention_launch_bf16(pass, p, stream);
}

// The workgroups of the kernels below each take one block of rows of a segment.
struct CodeBlock {
    int g, first, n, rows, padded;
    long long start;
};
__device__ inline CodeBlock code_block(const int *items, const int *seg_ptr, const int64_t *code_start, int block_rows) {
    CodeBlock b;
    b.g = items[2 * blockIdx.x];
    b.first = items[2 * blockIdx.x + 1];
    b.n = seg_ptr[b.g + 1] - seg_ptr[b.g];
    b.rows = min(block_rows, b.n - b.first);
    b.padded = (b.n + 31) / 32 * 32;
    b.start = code_start[b.g];
    return b;
}

// four codes of a row of n at j, 255 from n on
__device__ inline uint32_t four_codes(const uint8_t *row, int j, int n) {
    uint32_t v = 0xFFFFFFFFu;
    if (j + 4 <= n) {
        __builtin_memcpy(&v, row + j, 4);
    } else {
        for (int e = 0; e < 4; ++e)
            if (j + e < n) v = (v & ~(255u << (8 * e))) | ((uint32_t)row[j + e] << (8 * e));
    }
    return v;
}

// Rows of n bytes at any address to rows of a multiple of 32, four bytes a lane, a wavefront per row; and, by 64 x 64
// tiles through LDS, to the same with a row per key.  kDenseSplit workgroups share a block of rows.
constexpr int kDenseSplit = 8;
__global__ void __launch_bounds__(kBlock)
pair_dense_kernel(const uint8_t *__restrict__ dense, const int64_t *__restrict__ pair_start,
                  const int *__restrict__ seg_ptr, const int64_t *__restrict__ code_start,
                  const int *__restrict__ items, int block_rows, uint8_t *__restrict__ codes,
                  uint8_t *__restrict__ codes_by_key) {
    __shared__ __attribute__((aligned(4))) uint8_t tile[64][68];
    const CodeBlock b = code_block(items, seg_ptr, code_start, block_rows);
    const uint8_t *in = dense + pair_start[b.g];
    const int lane = threadIdx.x & 63, share = blockIdx.y;
    for (int r = (threadIdx.x >> 6) + share * (kBlock / 64); r < b.rows; r += kDenseSplit * (kBlock / 64))
        for (int j = 4 * lane; j < b.padded; j += 256)
            *(uint32_t *)(codes + b.start + (long long)(b.first + r) * b.padded + j) =
                four_codes(in + (long long)(b.first + r) * b.n, j, b.n);
    const int i = threadIdx.x >> 4, four = 4 * (threadIdx.x & 15);       // row of sixteen, first of four columns
    for (int k0 = b.first; k0 < b.first + b.rows; k0 += 64)
        for (int q0 = 64 * share; q0 < b.padded; q0 += 64 * kDenseSplit) {
            __syncthreads();
            for (int r = i; r < 64; r += 16)
                *(uint32_t *)&tile[r][four] = q0 + r < b.n ? four_codes(in + (long long)(q0 + r) * b.n, k0 + four, b.n)
                                                           : 0xFFFFFFFFu;
            __syncthreads();
            for (int k = i; k < 64; k += 16)
                if (k0 + k < b.first + b.rows && q0 + four < b.padded) {
                    uint32_t v = 0;
                    for (int e = 0; e < 4; ++e) v |= (uint32_t)tile[four + e][k] << (8 * e);
                    *(uint32_t *)(codes_by_key + b.start + (long long)(k0 + k) * b.padded + q0 + four) = v;
                }
        }
}

__global__ void __launch_bounds__(kBlock)
pair_relative_kernel(const uint8_t *__restrict__ by_offset, int reach, const int *__restrict__ seg_ptr,
                     const int64_t *__restrict__ code_start, const int *__restrict__ items, int block_rows,
                     uint8_t *__restrict__ codes, uint8_t *__restrict__ codes_by_key) {
    const CodeBlock b = code_block(items, seg_ptr, code_start, block_rows);
    const auto code = [&](int d) { return (uint32_t)by_offset[min(max(d, -reach), reach) + reach]; };
    for (int r = threadIdx.x >> 6; r < b.rows; r += kBlock / 64) {
        const int i = b.first + r;
        const long long at = b.start + (long long)i * b.padded;
        for (int j = 4 * (threadIdx.x & 63); j < b.padded; j += 256) {
            uint32_t forward = 0, back = 0;
            for (int e = 0; e < 4; ++e) {
                forward |= (j + e < b.n ? code(j + e - i) : 255u) << (8 * e);
                back |= (j + e < b.n ? code(i - j - e) : 255u) << (8 * e);
            }
            *(uint32_t *)(codes + at + j) = forward;
            *(uint32_t *)(codes_by_key + at + j) = back;
        }
    }
}

__global__ void __launch_bounds__(kBlock)
pair_hops_kernel(const int *__restrict__ row_start, const int *__restrict__ col, const int *__restrict__ dist,
                 int far_code, const int *__restrict__ seg_ptr, const int64_t *__restrict__ code_start,
                 const int *__restrict__ items, int block_rows, uint8_t *__restrict__ codes) {
    const CodeBlock b = code_block(items, seg_ptr, code_start, block_rows);
    const int lo = seg_ptr[b.g];
    for (int r = 0; r < b.rows; ++r) {
        const int i = b.first + r;
        uint8_t *out = codes + b.start + (long long)i * b.padded;
        for (int j = threadIdx.x; j < b.padded; j += kBlock) out[j] = j == i ? 0 : j < b.n ? (uint8_t)far_code : 255;
    }
    __syncthreads();                              // the listed pairs overwrite what other threads wrote
    for (int r = threadIdx.x >> 6; r < b.rows; r += kBlock / 64) {
        const int i = b.first + r;
        uint8_t *out = codes + b.start + (long long)i * b.padded;
        for (int e = row_start[lo + i] + (int)(threadIdx.x & 63); e < row_start[lo + i + 1]; e += 64) {
            const int j = col[e] - lo;
            if ((unsigned)j < (unsigned)b.n) out[j] = (uint8_t)dist[e];
        }
    }
}

int check_codes(const int32_t *seg_ptr, const int64_t *code_start, const int32_t *items, int64_t n_items,
                int32_t block_rows, const uint8_t *codes) {
    if (n_items < 0 || n_items > 0x7FFFFFFFll) return RWK_E_SIZE;
    if (block_rows != 32 && block_rows != 128) return RWK_E_UNSUPPORTED;
    if (n_items == 0) return RWK_OK;
    RWK_REQUIRE_PTR(seg_ptr);
    RWK_REQUIRE_PTR(code_start);
    RWK_REQUIRE_PTR(items);
    RWK_REQUIRE_PTR(codes);
    return (uintptr_t)codes % 16 == 0 ? RWK_OK : RWK_E_ALIGN;
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
        if (code == RWK_OK && a->key_parts > 1)
            code = a->type == RWK_F32   ? dkv_sum<float>(*a, (hipStream_t)stream)
                   : a->type == RWK_F16 ? dkv_sum<rwk_f16>(*a, (hipStream_t)stream)
                                        : dkv_sum<rwk_bf16>(*a, (hipStream_t)stream);
        if (code != RWK_OK) return code;
    }
    return a->n_buckets > 0 ? bias_sum(*a, (hipStream_t)stream) : RWK_OK;
}

int rwk_pair_buckets_dense(const uint8_t *dense, const int64_t *pair_start, const int32_t *seg_ptr,
                           const int64_t *code_start, const int32_t *items, int64_t n_items, int32_t block_rows,
                           uint8_t *codes, uint8_t *codes_by_key, rwk_stream_t stream) {
    int code = check_codes(seg_ptr, code_start, items, n_items, block_rows, codes);
    if (code == RWK_OK) code = check_codes(seg_ptr, code_start, items, n_items, block_rows, codes_by_key);
    if (code != RWK_OK || n_items == 0) return code;
    RWK_REQUIRE_PTR(dense);
    RWK_REQUIRE_PTR(pair_start);
    hipLaunchKernelGGL(pair_dense_kernel, dim3((unsigned)n_items, kDenseSplit), dim3(kBlock), 0, (hipStream_t)stream, dense,
                       pair_start, seg_ptr, code_start, items, block_rows, codes, codes_by_key);
    RWK_LAUNCH_CHECK();
    return RWK_OK;
}

int rwk_pair_buckets_relative(const uint8_t *by_offset, int64_t reach, const int32_t *seg_ptr,
                              const int64_t *code_start, const int32_t *items, int64_t n_items, int32_t block_rows,
                              uint8_t *codes, uint8_t *codes_by_key, rwk_stream_t stream) {
    if (reach < 0 || reach > 0x3FFFFFFF) return RWK_E_SIZE;
    int code = check_codes(seg_ptr, code_start, items, n_items, block_rows, codes);
    if (code == RWK_OK) code = check_codes(seg_ptr, code_start, items, n_items, block_rows, codes_by_key);
    if (code != RWK_OK || n_items == 0) return code;
    RWK_REQUIRE_PTR(by_offset);
    hipLaunchKernelGGL(pair_relative_kernel, dim3((unsigned)n_items), dim3(kBlock), 0, (hipStream_t)stream, by_offset,
                       (int)reach, seg_ptr, code_start, items, block_rows, codes, codes_by_key);
    RWK_LAUNCH_CHECK();
    return RWK_OK;
}

int rwk_pair_buckets_hops(const int32_t *row_start, const int32_t *col, const int32_t *dist, int32_t far_code,
                          const int32_t *seg_ptr, const int64_t *code_start, const int32_t *items, int64_t n_items,
                          int32_t block_rows, uint8_t *codes, rwk_stream_t stream) {
    if (far_code < 0 || far_code > 255) return RWK_E_SIZE;
    const int code = check_codes(seg_ptr, code_start, items, n_items, block_rows, codes);
    if (code != RWK_OK || n_items == 0) return code;
    RWK_REQUIRE_PTR(row_start);
    hipLaunchKernelGGL(pair_hops_kernel, dim3((unsigned)n_items), dim3(kBlock), 0, (hipStream_t)stream, row_start, col,
                       dist, far_code, seg_ptr, code_start, items, block_rows, codes);
    RWK_LAUNCH_CHECK();
    return RWK_OK;
}

}  // extern "C"
