// Attention inside packed segments: kernels, for one element type per including source.
//
// Rows i, j of one segment, query head h with key / value head h / group:
//   s_ij = scale * q_i . k_j (+ table[h][code_ij]),   j <= i if causal, code_ij < n_buckets if there is a table
//   p_ij = exp(s_ij - m_i) / l_i,  o_i = sum_j p_ij v_j     (a row without pairs: p = 0, o = 0)
// Backward, with delta_i = do_i . o_i:
//   dv_j = sum_i p_ij do_i,  ds_ij = p_ij (do_i . v_j - delta_i),  dq_i = scale sum_j ds_ij k_j,
//   dk_j = scale sum_i ds_ij q_i,  d_table[h][b] = sum over pairs with code b of ds_ij
//
// One pass over the keys with the running maximum and sum of the softmax; scores never leave the registers.  All
// products are 32x32 matrix instructions (16-bit types: 16 products deep, fp32: 2 deep, eight in a row), all sums,
// maxima and exponentials fp32.  A wavefront owns 32 rows and computes scores TRANSPOSED to what it owns as columns:
// lane l holds row (or key) l % 32 of its own and 16 of the other index, which is the operand layout of the next
// product up to a permutation of the summed index, so probabilities go from one product to the next without leaving
// their lane.  They are rounded to the element type there (the matrix instructions take nothing wider); the sums l_i,
// delta and d_table use the unrounded fp32 values.
//
// Summed index of the second product: slot e of lane half h (h = lane / 32) of step s is row 16 s + 4 h + e for
// e < 4 and 16 s + 8 + 4 h + (e - 4) otherwise, the registers 8 s + e of a 32x32 result.
//
// Tiles of the other operand lie in LDS row by row, the 16-byte chunks of a row permuted by the row's number
// (chunk ^ row) so that both kinds of reads - eight consecutive elements of a row per lane, and columns of four rows -
// spread over the banks.
#pragma once

#include "rwk_attention.h"
#include "rwk_vec.h"

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));

template <typename T> struct Frag { typename RwkPack<T, 8>::type v; };
template <> struct Frag<float> { float v[8]; };

__device__ inline f32x16 mma(const Frag<rwk_bf16> &a, const Frag<rwk_bf16> &b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.v, b.v, c, 0, 0, 0);
}
__device__ inline f32x16 mma(const Frag<rwk_f16> &a, const Frag<rwk_f16> &b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a.v, b.v, c, 0, 0, 0);
}
__device__ inline f32x16 mma(const Frag<float> &a, const Frag<float> &b, f32x16 c) {
#pragma unroll
    for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.v[e], b.v[e], c, 0, 0, 0);
    return c;
}

// Scores are worked on as arrays and replaced as a whole by selects: elements of a result's vector assigned under a
// lane's condition were compiled wrongly (the other elements took the first one's value).
__device__ inline void unpack(const f32x16 &x, float (&s)[16]) {
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = x[i];
}

// elements 8 s .. 8 s + 7 as the operand of a further product
template <typename T>
__device__ inline Frag<T> pack(const float (&x)[16], int s) {
    Frag<T> f;
#pragma unroll
    for (int e = 0; e < 8; ++e) f.v[e] = (T)x[8 * s + e];
    return f;
}

// row (of the transposed index) that register i of lane half h holds in a 32x32 result
__device__ inline int reg_row(int i, int h) { return 8 * (i >> 2) + 4 * h + (i & 3); }

// D elements padded to KS * 16 for the first product's sum and to DT * 32 rows of the second's result
template <typename T, int KS>
struct Shape {
    static constexpr int DT = (KS + 1) / 2;
    static constexpr int W = 32 * DT;                             // elements of a row in LDS
    static constexpr int E = 16 / (int)sizeof(T);                 // elements of a chunk
    static constexpr int C = W / E;                               // chunks of a row: 4, 8, 16 or 32
    __device__ static int swizzle(int row) { return C == 4 ? (row >> 1) & 3 : row & (C - 1); }
    // place of chunk c of a row
    __device__ static int at(int row, int c) { return row * W + ((c ^ swizzle(row)) * E); }
};

// eight consecutive elements of a row in memory, zeros from element `dim` on
template <typename T>
__device__ inline Frag<T> load_global(const T *row, int first, int dim) {
    Frag<T> f;
    if (first + 8 <= dim) {
        if constexpr (sizeof(T) == 2) {
            f.v = rwk_load<T, 8>(row + first);
        } else {
            const auto lo = rwk_load<T, 4>(row + first), hi = rwk_load<T, 4>(row + first + 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                f.v[e] = lo[e];
                f.v[4 + e] = hi[e];
            }
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) f.v[e] = first + e < dim ? row[first + e] : (T)0.f;
    }
    return f;
}

// ROWS rows from `first` of a (rows, dim) matrix into LDS; rows from `rows` on and elements from `dim` on are zeros
template <typename T, int KS, int ROWS, int NT>
__device__ inline void load_tile(const T *base, long long stride, int first, int rows, int dim, T *lds) {
    using S = Shape<T, KS>;
#pragma unroll
    for (int i = 0; i < (ROWS * S::C + NT - 1) / NT; ++i) {
        const int k = (int)threadIdx.x + i * NT;
        if (ROWS * S::C % NT != 0 && k >= ROWS * S::C) break;
        const int row = k / S::C, c = k % S::C;
        typename RwkPack<T, S::E>::type v;
#pragma unroll
        for (int e = 0; e < S::E; ++e) v[e] = (T)0.f;
        if (first + row < rows) {
            const T *p = base + (long long)(first + row) * stride + c * S::E;
            if ((c + 1) * S::E <= dim) {
                v = rwk_load<T, S::E>(p);
            } else {
#pragma unroll
                for (int e = 0; e < S::E; ++e)
                    if (c * S::E + e < dim) v[e] = p[e];
            }
        }
        *reinterpret_cast<typename RwkPack<T, S::E>::type *>(lds + S::at(row, c)) = v;
    }
}

// operand whose 32 rows are rows of the tile and whose summed index is the element: step ks
template <typename T, int KS>
__device__ inline Frag<T> row_operand(const T *tile, int row, int ks, int h) {
    using S = Shape<T, KS>;
    Frag<T> f;
    if constexpr (sizeof(T) == 2) {
        f.v = *reinterpret_cast<const typename RwkPack<T, 8>::type *>(tile + S::at(row, 2 * ks + h));
    } else {
        typedef float f32x4 __attribute__((ext_vector_type(4)));
        const f32x4 lo = *reinterpret_cast<const f32x4 *>(tile + S::at(row, 4 * ks + 2 * h));
        const f32x4 hi = *reinterpret_cast<const f32x4 *>(tile + S::at(row, 4 * ks + 2 * h + 1));
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            f.v[e] = lo[e];
            f.v[4 + e] = hi[e];
        }
    }
    return f;
}

// operand whose 32 rows are the elements 32 dt .. of the tile's rows and whose summed index are the tile's rows
// first .. first + 15 in the order of a result's registers.  16-bit types: the transposing LDS read hands lane i of
// 16 the elements of column i in four rows, lane i addressing row i / 4, columns 4 (i % 4).
template <typename T, int KS>
__device__ inline Frag<T> column_operand(const T *tile, int first, int dt, int lane) {
    using S = Shape<T, KS>;
    const int h = lane >> 5;
    Frag<T> f;
    if constexpr (sizeof(T) == 2) {
        typedef short s16x4 __attribute__((ext_vector_type(4)));
        const int col = 32 * dt + (lane & 16) + 4 * (lane & 3);
        s16x4 part[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int row = first + 8 * u + 4 * h + ((lane & 15) >> 2);
            const T *p = tile + S::at(row, col >> 3) + (col & 7);
            part[u] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) s16x4 *)(__attribute__((address_space(3))) void *)p);
        }
        f.v = __builtin_bit_cast(typename RwkPack<T, 8>::type,
                                 __builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
        const int col = 32 * dt + (lane & 31);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int row = first + 8 * (e >> 2) + 4 * h + (e & 3);
            f.v[e] = tile[S::at(row, col >> 2) + (col & 3)];
        }
    }
    return f;
}

// a transposed result, DT tiles of 32 elements: lane l % 32 is the row, its registers four elements each
template <typename T, int DT>
__device__ inline void store_rows(T *row, int dim, int h, const f32x16 (&acc)[DT], float scale) {
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int d = 32 * dt + 8 * g + 4 * h;
            if (d + 4 <= dim) {
                typename RwkPack<T, 4>::type v;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = (T)(acc[dt][4 * g + e] * scale);
                rwk_store<T, 4>(row + d, v);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (d + e < dim) row[d + e] = (T)(acc[dt][4 * g + e] * scale);
            }
        }
}

constexpr float kLog2e = 1.4426950408889634f;

// One workgroup's place in the launch: consecutive workgroups go to different dies, so the key / value head varies
// fastest - a die that meets one head's keys and values again finds them in its own cache - then the query heads that
// share it, then the blocks of rows, which the caller lists with the most work first.
struct Place {
    int item, seg, first, head, kv_head, n;
    long long base;
};
__device__ inline Place place_of(const RwkAttnArgs &p, long long b) {
    Place s;
    s.kv_head = (int)(b % p.a.kv_heads);
    b /= p.a.kv_heads;
    s.head = s.kv_head * p.group;
    s.item = (int)b;
    return s;
}
__device__ inline void find_rows(const RwkAttnArgs &p, Place &s) {
    s.seg = p.items[2 * s.item];
    s.first = p.items[2 * s.item + 1];
    s.base = p.a.seg_ptr[s.seg];
    s.n = (int)(p.a.seg_ptr[s.seg + 1] - s.base);
}
// of a launch over query heads
__device__ inline Place query_place(const RwkAttnArgs &p, long long b) {
    Place s = place_of(p, b);
    s.head += s.item % p.group;
    s.item /= p.group;
    find_rows(p, s);
    return s;
}
// of a launch over key / value heads
__device__ inline Place key_place(const RwkAttnArgs &p, long long b) {
    Place s = place_of(p, b);
    find_rows(p, s);
    return s;
}

// the bias of one head in LDS, -infinity for codes that do not attend
template <typename T, int NT>
__device__ inline void load_table(const RwkAttnArgs &p, int head, float *table) {
    for (int b = threadIdx.x; b <= p.a.n_buckets; b += NT)
        table[b] = b < p.a.n_buckets ? (float)((const T *)p.a.table)[(long long)head * p.a.n_buckets + b] : -INFINITY;
}

template <typename T, int KS, int NW, bool BIAS>
__global__ void __launch_bounds__(64 * NW)
attention_forward_kernel(const RwkAttnArgs p) {
    using S = Shape<T, KS>;
    constexpr int NT = 64 * NW, DT = S::DT, BN = sizeof(T) == 2 ? 64 : 32, TN = BN / 32;
    extern __shared__ __attribute__((aligned(16))) char attn_lds[];
    T *k_tile = (T *)attn_lds, *v_tile = k_tile + BN * S::W;
    float *table = (float *)(v_tile + BN * S::W);
    const Place at = query_place(p, blockIdx.x);
    const int lane = threadIdx.x & 63, h = lane >> 5, dim = (int)p.a.dim, n = at.n;
    const int q0 = at.first + 32 * (int)(threadIdx.x >> 6), q = q0 + (lane & 31), qc = q < n ? q : n - 1;
    const bool causal = p.a.causal != 0;
    const int nb = (int)p.a.n_buckets;
    if (BIAS) load_table<T, NT>(p, at.head, table);

    Frag<T> qf[KS];
    const T *q_row = (const T *)p.a.q + (at.base + qc) * p.a.q_row + at.head * p.a.q_head;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[ks] = load_global<T>(q_row, 16 * ks + 8 * h, dim);
    const T *k_base = (const T *)p.a.k + at.base * p.a.k_row + at.kv_head * p.a.k_head;
    const T *v_base = (const T *)p.a.v + at.base * p.a.v_row + at.kv_head * p.a.v_head;
    const uint8_t *code_row = nullptr;
    if (BIAS) code_row = p.a.codes + p.a.code_start[at.seg] + (long long)qc * ((n + 31) / 32 * 32);

    // without a bias the maximum is taken over q . k and the scale meets it in the exponent; with one the scores are
    // the sum, and the difference is formed before the change of base, so that a bias of the type's lowest value
    // stays finite
    const float scale = p.a.scale, c = BIAS ? kLog2e : scale * kLog2e;
    f32x16 acc[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) acc[dt] = f32x16{};
    float top = -INFINITY, sum = 0.f;
    const int end = causal && at.first + 32 * NW < n ? at.first + 32 * NW : n;
    for (int k0 = 0; k0 < end; k0 += BN) {
        __syncthreads();
        load_tile<T, KS, BN, NT>(k_base, p.a.k_row, k0, n, dim, k_tile);
        load_tile<T, KS, BN, NT>(v_base, p.a.v_row, k0, n, dim, v_tile);
        __syncthreads();
        if (q0 >= n || (causal && k0 > q0 + 31)) continue;
        float s[TN][16];
#pragma unroll
        for (int t = 0; t < TN; ++t) {
            f32x16 x = f32x16{};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) x = mma(row_operand<T, KS>(k_tile, 32 * t + (lane & 31), ks, h), qf[ks], x);
            unpack(x, s[t]);
        }
        if (BIAS) {
#pragma unroll
            for (int t = 0; t < TN; ++t)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    // columns from n on are padded with codes that do not attend
                    const uint32_t codes = k0 + 32 * t < n
                        ? *(const uint32_t *)(code_row + k0 + 32 * t + 8 * g + 4 * h) : 0xFFFFFFFFu;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int b = min((int)((codes >> (8 * e)) & 255u), nb);
                        const float x = fmaf(s[t][4 * g + e], scale, table[b]);
                        s[t][4 * g + e] = b < nb ? x : -INFINITY;
                    }
                }
        }
        if (k0 + BN > n || (causal && k0 + BN - 1 > q0)) {
            const int last = causal ? min(q, n - 1) : n - 1;
#pragma unroll
            for (int t = 0; t < TN; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i) s[t][i] = k0 + 32 * t + reg_row(i, h) <= last ? s[t][i] : -INFINITY;
        }
        float here = s[0][0];
#pragma unroll
        for (int t = 0; t < TN; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) here = fmaxf(here, s[t][i]);
        here = fmaxf(here, __shfl_xor(here, 32, 64));
        const float now = fmaxf(top, here), ref = now == -INFINITY ? 0.f : now;
        const float shrink = exp2f((top - ref) * c);
        top = now;
        float part = 0.f;
#pragma unroll
        for (int t = 0; t < TN; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[t][i] = exp2f(BIAS ? (s[t][i] - ref) * c : fmaf(s[t][i], c, -ref * c));
                part += s[t][i];
            }
        sum = fmaf(sum, shrink, part);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[dt][i] *= shrink;
#pragma unroll
        for (int t = 0; t < TN; ++t)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const Frag<T> pf = pack<T>(s[t], u);
#pragma unroll
                for (int dt = 0; dt < DT; ++dt)
                    acc[dt] = mma(column_operand<T, KS>(v_tile, 32 * t + 16 * u, dt, lane), pf, acc[dt]);
            }
    }
    if (q >= n) return;
    sum += __shfl_xor(sum, 32, 64);
    const float inv = sum == 0.f ? 0.f : 1.f / sum;      // a row without pairs: zeros
    store_rows<T, DT>((T *)p.a.out + ((at.base + q) * p.a.heads + at.head) * dim, dim, h, acc, inv);
    if (p.a.stats != nullptr && h == 0) {
        float *st = p.a.stats + 2 * (at.head * p.a.rows + at.base + q);
        st[0] = top == -INFINITY ? 0.f : top;
        st[1] = inv;
    }
}

template <typename T, int KS, int NW, bool BIAS>
__global__ void __launch_bounds__(64 * NW)
attention_dq_kernel(const RwkAttnArgs p) {
    using S = Shape<T, KS>;
    constexpr int NT = 64 * NW, DT = S::DT, BN = sizeof(T) == 2 ? 64 : 32, TN = BN / 32;
    extern __shared__ __attribute__((aligned(16))) char attn_lds[];
    T *k_tile = (T *)attn_lds, *v_tile = k_tile + BN * S::W;
    float *table = (float *)(v_tile + BN * S::W), *hist = table + 64;
    const Place at = query_place(p, blockIdx.x);
    const int lane = threadIdx.x & 63, h = lane >> 5, dim = (int)p.a.dim, n = at.n;
    const int q0 = at.first + 32 * (int)(threadIdx.x >> 6), q = q0 + (lane & 31), qc = q < n ? q : n - 1;
    const bool causal = p.a.causal != 0;
    const int nb = (int)p.a.n_buckets;
    if (BIAS) {
        load_table<T, NT>(p, at.head, table);
        for (int b = 0; b <= nb; ++b) hist[b * NT + threadIdx.x] = 0.f;    // a thread's own sums
    }

    Frag<T> qf[KS], of[KS];
    const long long o_at = ((at.base + qc) * p.a.heads + at.head) * dim;
    const T *q_row = (const T *)p.a.q + (at.base + qc) * p.a.q_row + at.head * p.a.q_head;
    const T *do_row = (const T *)p.a.d_out + (at.base + qc) * p.a.do_row + at.head * p.a.do_head;
    float delta = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        qf[ks] = load_global<T>(q_row, 16 * ks + 8 * h, dim);
        of[ks] = load_global<T>(do_row, 16 * ks + 8 * h, dim);
        const Frag<T> o = load_global<T>((const T *)p.a.out + o_at, 16 * ks + 8 * h, dim);
#pragma unroll
        for (int e = 0; e < 8; ++e) delta = fmaf((float)of[ks].v[e], (float)o.v[e], delta);
    }
    delta += __shfl_xor(delta, 32, 64);
    const long long row_at = at.head * p.a.rows + at.base + qc;
    if (q < n && h == 0) p.a.delta[row_at] = delta;
    const float ref = p.a.stats[2 * row_at], inv = p.a.stats[2 * row_at + 1];
    const T *k_base = (const T *)p.a.k + at.base * p.a.k_row + at.kv_head * p.a.k_head;
    const T *v_base = (const T *)p.a.v + at.base * p.a.v_row + at.kv_head * p.a.v_head;
    const uint8_t *code_row = nullptr;
    if (BIAS) code_row = p.a.codes + p.a.code_start[at.seg] + (long long)qc * ((n + 31) / 32 * 32);
    const float scale = p.a.scale, c = BIAS ? kLog2e : scale * kLog2e;

    f32x16 acc[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) acc[dt] = f32x16{};
    const int end = causal && at.first + 32 * NW < n ? at.first + 32 * NW : n;
    for (int k0 = 0; k0 < end; k0 += BN) {
        __syncthreads();
        load_tile<T, KS, BN, NT>(k_base, p.a.k_row, k0, n, dim, k_tile);
        load_tile<T, KS, BN, NT>(v_base, p.a.v_row, k0, n, dim, v_tile);
        __syncthreads();
        if (q0 >= n) continue;
#pragma unroll
        for (int t = 0; t < TN; ++t) {
            const int kt = k0 + 32 * t;
            if (kt >= n || (causal && kt > q0 + 31)) break;
            f32x16 sx = f32x16{}, dx = f32x16{};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                sx = mma(row_operand<T, KS>(k_tile, 32 * t + (lane & 31), ks, h), qf[ks], sx);
                dx = mma(row_operand<T, KS>(v_tile, 32 * t + (lane & 31), ks, h), of[ks], dx);
            }
            float s[16], d[16];
            unpack(sx, s);
            unpack(dx, d);
            uint32_t codes[4];
            if (BIAS) {
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    codes[g] = *(const uint32_t *)(code_row + kt + 8 * g + 4 * h);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int b = min((int)((codes[g] >> (8 * e)) & 255u), nb);
                        const float x = fmaf(s[4 * g + e], scale, table[b]);
                        s[4 * g + e] = b < nb ? x : -INFINITY;
                    }
                }
            }
            const bool masked = kt + 32 > n || (causal && kt + 31 > q0);
            if (masked) {
                const int last = causal ? min(q, n - 1) : n - 1;
#pragma unroll
                for (int i = 0; i < 16; ++i) s[i] = kt + reg_row(i, h) <= last ? s[i] : -INFINITY;
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const bool off = (BIAS || masked) && s[i] == -INFINITY;
                const float pr = exp2f(BIAS ? (s[i] - ref) * c : fmaf(s[i], c, -ref * c)) * inv;
                s[i] = off ? 0.f : pr * (d[i] - delta);      // a masked pair's value may be anything
            }
            if (BIAS) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int b = min((int)((codes[i >> 2] >> (8 * (i & 3))) & 255u), nb);
                    hist[b * NT + threadIdx.x] += q < n ? s[i] : 0.f;
                }
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const Frag<T> sf = pack<T>(s, u);
#pragma unroll
                for (int dt = 0; dt < DT; ++dt)
                    acc[dt] = mma(column_operand<T, KS>(k_tile, 32 * t + 16 * u, dt, lane), sf, acc[dt]);
            }
        }
    }
    if (q < n) store_rows<T, DT>((T *)p.a.dq + o_at, dim, h, acc, scale);
    if (BIAS) {
        __syncthreads();
        // a wavefront per bucket sums the threads' slots in a fixed order
        for (int b = threadIdx.x >> 6; b < nb; b += NW) {
            float v = 0.f;
#pragma unroll
            for (int w = 0; w < NW; ++w) v += hist[b * NT + 64 * w + lane];
            v = rwk_wave_sum(v);
            if (lane == 0) p.a.d_table_partials[((long long)at.head * nb + b) * p.a.n_items + at.item] = v;
        }
    }
}

template <typename T, int KS, int NW, bool BIAS>
__global__ void __launch_bounds__(64 * NW)
attention_dkv_kernel(const RwkAttnArgs p) {
    using S = Shape<T, KS>;
    constexpr int NT = 64 * NW, DT = S::DT, BQ = 32;
    extern __shared__ __attribute__((aligned(16))) char attn_lds[];
    T *q_tile = (T *)attn_lds, *o_tile = q_tile + BQ * S::W;
    float *st = (float *)(o_tile + BQ * S::W), *table = st + 3 * BQ;       // st: maximum, 1 / sum, delta per row
    const Place at = key_place(p, blockIdx.x);
    const int lane = threadIdx.x & 63, h = lane >> 5, dim = (int)p.a.dim, n = at.n;
    const int k0 = at.first + 32 * (int)(threadIdx.x >> 6), k = k0 + (lane & 31), kc = k < n ? k : n - 1;
    const bool causal = p.a.causal != 0;
    const int nb = (int)p.a.n_buckets;

    Frag<T> kf[KS], vf[KS];
    const T *k_row = (const T *)p.a.k + (at.base + kc) * p.a.k_row + at.kv_head * p.a.k_head;
    const T *v_row = (const T *)p.a.v + (at.base + kc) * p.a.v_row + at.kv_head * p.a.v_head;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        kf[ks] = load_global<T>(k_row, 16 * ks + 8 * h, dim);
        vf[ks] = load_global<T>(v_row, 16 * ks + 8 * h, dim);
    }
    const long long code_stride = (n + 31) / 32 * 32;
    const uint8_t *code_col = nullptr;
    if (BIAS) code_col = p.a.codes + p.a.code_start[at.seg] + kc;
    const float scale = p.a.scale, c = BIAS ? kLog2e : scale * kLog2e;

    f32x16 dk[DT], dv[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) dk[dt] = dv[dt] = f32x16{};
    for (int g = 0; g < p.group; ++g) {
        const int head = at.head + g;
        const T *q_base = (const T *)p.a.q + at.base * p.a.q_row + head * p.a.q_head;
        const T *o_base = (const T *)p.a.d_out + at.base * p.a.do_row + head * p.a.do_head;
        const long long row_at = head * p.a.rows + at.base;
        if (BIAS) {
            __syncthreads();
            load_table<T, NT>(p, head, table);
        }
        for (int q0 = causal ? at.first : 0; q0 < n; q0 += BQ) {
            __syncthreads();
            load_tile<T, KS, BQ, NT>(q_base, p.a.q_row, q0, n, dim, q_tile);
            load_tile<T, KS, BQ, NT>(o_base, p.a.do_row, q0, n, dim, o_tile);
            if (threadIdx.x < BQ) {
                const int q = q0 + (int)threadIdx.x;
                st[threadIdx.x] = q < n ? p.a.stats[2 * (row_at + q)] : 0.f;
                st[BQ + threadIdx.x] = q < n ? p.a.stats[2 * (row_at + q) + 1] : 0.f;     // rows beyond: p = 0
                st[2 * BQ + threadIdx.x] = q < n ? p.a.delta[row_at + q] : 0.f;
            }
            __syncthreads();
            if (k0 >= n || (causal && q0 + BQ - 1 < k0)) continue;
            f32x16 sx = f32x16{}, dx = f32x16{};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                sx = mma(row_operand<T, KS>(q_tile, lane & 31, ks, h), kf[ks], sx);
                dx = mma(row_operand<T, KS>(o_tile, lane & 31, ks, h), vf[ks], dx);
            }
            float s[16], d[16];
            unpack(sx, s);
            unpack(dx, d);
            const bool masked = causal && q0 < k0 + 31;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int r = reg_row(i, h);
                const float ref = st[r], inv = st[BQ + r], delta = st[2 * BQ + r];
                bool off = false;
                if (BIAS) {
                    const int b = q0 + r < n ? min((int)code_col[(q0 + r) * code_stride], nb) : nb;
                    off = b >= nb;
                    s[i] = fmaf(s[i], scale, table[b]);
                }
                if (masked) off = off || q0 + r < k;
                float pr = exp2f(BIAS ? (s[i] - ref) * c : fmaf(s[i], c, -ref * c)) * inv;
                if (BIAS) off = off || s[i] == -INFINITY;
                pr = off ? 0.f : pr;
                d[i] = off ? 0.f : pr * (d[i] - delta);
                s[i] = pr;
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const Frag<T> pf = pack<T>(s, u), sf = pack<T>(d, u);
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) {
                    dv[dt] = mma(column_operand<T, KS>(o_tile, 16 * u, dt, lane), pf, dv[dt]);
                    dk[dt] = mma(column_operand<T, KS>(q_tile, 16 * u, dt, lane), sf, dk[dt]);
                }
            }
        }
    }
    if (k >= n) return;
    const long long to = ((at.base + k) * p.a.kv_heads + at.kv_head) * dim;
    store_rows<T, DT>((T *)p.a.dk + to, dim, h, dk, scale);
    store_rows<T, DT>((T *)p.a.dv + to, dim, h, dv, 1.f);
}

template <typename K>
int launch_kernel(K kernel, long long grid, int threads, size_t lds, const RwkAttnArgs &args, hipStream_t stream) {
    if (lds > 64 * 1024) {
        const hipError_t e = hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return (int)e;
    }
    hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3((unsigned)threads), lds, stream, args);
    RWK_LAUNCH_CHECK();
    return RWK_OK;
}

template <typename T, int KS, int NW, bool BIAS>
int launch_shape(RwkAttnPass pass, const RwkAttnArgs &p, hipStream_t stream) {
    using S = Shape<T, KS>;
    constexpr int NT = 64 * NW;
    const size_t row = S::W * sizeof(T), keys = sizeof(T) == 2 ? 64 : 32;
    if (pass == kRwkAttnForward)
        return launch_kernel(attention_forward_kernel<T, KS, NW, BIAS>, p.a.n_items * p.a.heads, NT,
                             2 * keys * row + 64 * sizeof(float), p, stream);
    if (pass == kRwkAttnDq)
        return launch_kernel(attention_dq_kernel<T, KS, NW, BIAS>, p.a.n_items * p.a.heads, NT,
                             2 * keys * row + (64 + (BIAS ? (p.a.n_buckets + 1) * NT : 0)) * sizeof(float), p, stream);
    return launch_kernel(attention_dkv_kernel<T, KS, NW, BIAS>, p.a.n_items * p.a.kv_heads, NT,
                         2 * 32 * row + (3 * 32 + 64) * sizeof(float), p, stream);
}

template <typename T, int KS>
int launch_width(RwkAttnPass pass, const RwkAttnArgs &p, hipStream_t stream) {
    const bool bias = p.a.n_buckets > 0;
    if (p.a.block_rows == 128)
        return bias ? launch_shape<T, KS, 4, true>(pass, p, stream) : launch_shape<T, KS, 4, false>(pass, p, stream);
    return bias ? launch_shape<T, KS, 1, true>(pass, p, stream) : launch_shape<T, KS, 1, false>(pass, p, stream);
}

template <typename T>
int launch_type(RwkAttnPass pass, const RwkAttnArgs &p, hipStream_t stream) {
    if (p.a.dim <= 16) return launch_width<T, 1>(pass, p, stream);
    if (p.a.dim <= 32) return launch_width<T, 2>(pass, p, stream);
    if (p.a.dim <= 64) return launch_width<T, 4>(pass, p, stream);
    return launch_width<T, 8>(pass, p, stream);
}

}  // namespace
