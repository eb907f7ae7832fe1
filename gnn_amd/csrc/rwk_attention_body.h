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
// products are 32x32 matrix instructions (16-bit types: 16 products deep, fp32: 2 deep, eight in a row; fp32 heads of
// up to 16 elements have 16x16 second products), all sums, maxima and exponentials fp32.  A wavefront owns 32 rows and
// computes scores TRANSPOSED to what it owns as columns: lane l holds row (or key) l % 32 of its own and 16 of the other
// index, which is the operand layout of the next product up to a permutation of the summed index, so probabilities go
// from one product to the next without leaving their lane.  They are rounded to the element type there (the matrix
// instructions take nothing wider; the forward pass and narrow heads' dQ keep what that leaves over where it counts most,
// see FINE); the sums l_i, delta and d_table use the unrounded fp32 values.  16-bit outputs leave what their own rounding left over
// (out_low) for delta, whose error all of a row's ds share.
//
// The forward pass needs 2 products of a pair's rows, dQ 3 and dK/dV 4, and between them per pair an exponential (the
// time of four other instructions) and four to eight more.  At 128 elements of 16 bits the matrix unit bounds all three,
// at 64 none of the units is busy all the time - a wavefront's
// scores, exponentials and second products follow each other - with the vector unit the busiest; fp32 matrix instructions stop the vector unit, so there the two times add up.  4 prompts
// of up to 8192 rows, 32 heads of 128 in bf16 over 8 of keys, causal: 907 us forward (0.82 of a large product's rate),
// 1250 dQ (0.89), 1994 + 60 dK/dV (0.73); 48 of up to 1500, 16 heads of 64 in fp16 over 4: 148, 248, 280 us; 1024 graphs
// of 100 to 500 nodes, 4 heads of 16 in fp32, a bias of 8 buckets: 495, 757, 789 us.
//
// Summed index of the second product: slot e of lane half h (h = lane / 32) of step s is row 16 s + 4 h + e for
// e < 4 and 16 s + 8 + 4 h + (e - 4) otherwise, the registers 8 s + e of a 32x32 result.
//
// Tiles of the other operand lie in LDS row by row, the 16-byte chunks of a row permuted by the row's number
// (swizzle()) so that both kinds of reads - eight consecutive elements of a row per lane, and columns of four rows -
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

// what pack's rounding left over
template <typename T>
__device__ inline Frag<T> left_over(const float (&x)[16], const Frag<T> &packed, int s) {
    Frag<T> f;
#pragma unroll
    for (int e = 0; e < 8; ++e) f.v[e] = (T)(x[8 * s + e] - (float)packed.v[e]);
    return f;
}

// row (of the transposed index) that register i of lane half h holds in a 32x32 result
__device__ inline int reg_row(int i, int h) { return 8 * (i >> 2) + 4 * h + (i & 3); }

// D elements padded to KS * 16 for the first product's sum and to DT * 32 rows of the second's result.  The second
// product of KS = 1 reads past a row's 16 elements into the next: rows of the result that nobody stores.
template <typename T, int KS>
struct Shape {
    static constexpr int DT = (KS + 1) / 2;
    static constexpr int W = 16 * KS;                             // elements of a row in LDS
    static constexpr int E = 16 / (int)sizeof(T);                 // elements of a chunk
    static constexpr int C = W / E;                               // chunks of a row: a power of two, 2 .. 32
    // 64 banks of 4 bytes serve 16 lanes of 16 bytes, or 32 of 8, at once.  Row reads: 16 rows at one chunk have to
    // lie in 16 different places of 256 bytes.  Column reads: 16-bit types four rows of four chunks, fp32 the rows r
    // and r + 4 of eight chunks each.
    __device__ static int swizzle(int row) {
        if (C == 2) return (row >> 3) & 1;
        if (C == 4) return (row >> 2) & 3;
        if (C == 8) return ((row & 2) << 1) | ((row >> 2) & 3);
        if (sizeof(T) == 2) return ((row & 3) << 2) | ((row >> 2) & 3);
        return ((row & 4) << 1) | ((row & 8) >> 1) | (row & 3);
    }
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

typedef int i32x4 __attribute__((ext_vector_type(4)));

__device__ inline uint32_t lds_address(const void *p) {
    return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void *)p;
}

__device__ inline void load_to_lds(i32x4 rsrc, uint32_t offset, uint32_t to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                 :
                 : "s"(to), "v"(offset), "s"(rsrc)
                 : "memory");          // m0 is set right before every use by the compiler too
}

// ROWS rows at a time of a (rows, dim) matrix of a segment into LDS; rows from `rows` on and elements from `dim` on are
// zeros.  issue() starts the tile that begins at row `first`, commit() finishes it; in between, the workgroup computes
// on the other buffer.
//   ASYNC: the loads write LDS by themselves, 16 bytes a lane, and the buffer's bounds give the zeros; finish() waits.
//     Written as asm: for the builtin the compiler waits for all of them before any read of LDS.
//   otherwise (elements that are not whole 16-byte chunks, or unaligned rows): through registers, element by element
//     where a chunk is not whole.
template <typename T, int KS, int ROWS, int NT, bool ASYNC>
struct TileLoader {
    using S = Shape<T, KS>;
    static constexpr int N = (ROWS * S::C + NT - 1) / NT;
    typedef typename RwkPack<T, S::E>::type Chunk;
    const T *base;
    long long stride;
    int rows, dim;
    uint32_t offset[ASYNC ? N : 1];
    Chunk held[ASYNC ? 1 : N];

    __device__ TileLoader(const T *base_, long long stride_, int rows_, int dim_)
        : base(base_), stride(stride_), rows(rows_), dim(dim_) {
        if constexpr (ASYNC) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int k = (int)threadIdx.x + i * NT, row = k / S::C, c = (k % S::C) ^ S::swizzle(row);
                // a chunk behind the row's elements: an offset that no buffer reaches
                offset[i] = c * S::E < dim ? (uint32_t)(row * (int)stride * (int)sizeof(T) + c * 16) : 0xFFFFFF00u;
            }
        }
    }

    __device__ void issue(int first, T *lds) {
        if constexpr (ASYNC) {
            const uint64_t at = (uint64_t)(base + (long long)first * stride);
            const int left = min(rows - first, ROWS);
            i32x4 rsrc;
            rsrc[0] = __builtin_amdgcn_readfirstlane((int)at);
            rsrc[1] = __builtin_amdgcn_readfirstlane((int)((at >> 32) & 0xFFFFu));
            rsrc[2] = __builtin_amdgcn_readfirstlane(
                left > 0 ? ((left - 1) * (int)stride + dim) * (int)sizeof(T) : 0);
            rsrc[3] = 0x00027000;
            const uint32_t to = __builtin_amdgcn_readfirstlane(lds_address(lds) + (threadIdx.x & ~63u) * 16);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                if (ROWS * S::C % NT != 0 && (int)(threadIdx.x & ~63u) + i * NT >= ROWS * S::C) break;
                load_to_lds(rsrc, offset[i], to + i * NT * 16);
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int k = (int)threadIdx.x + i * NT, row = k / S::C, c = k % S::C;
                Chunk v;
#pragma unroll
                for (int e = 0; e < S::E; ++e) v[e] = (T)0.f;
                if (first + row < rows && row < ROWS) {
                    const T *p = base + (long long)(first + row) * stride + c * S::E;
                    if ((c + 1) * S::E <= dim) {
                        v = rwk_load<T, S::E>(p);
                    } else {
#pragma unroll
                        for (int e = 0; e < S::E; ++e) v[e] = c * S::E + e < dim ? p[e] : (T)0.f;
                    }
                }
                held[i] = v;
            }
        }
    }

    __device__ void commit(T *lds) {
        if constexpr (!ASYNC) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int k = (int)threadIdx.x + i * NT, row = k / S::C, c = k % S::C;
                if (ROWS * S::C % NT != 0 && k >= ROWS * S::C) break;
                *reinterpret_cast<Chunk *>(lds + S::at(row, c)) = held[i];
            }
        }
    }
};

// Bucket codes of ROWS rows (the workgroup's own rows, the last of the segment for those behind it) and COLS columns
// at a time, straight into LDS.  Columns from the segment's end on hold anything.
template <int ROWS, int COLS, int NT>
struct CodeLoader {
    static constexpr int C = COLS / 16, N = (ROWS * C + NT - 1) / NT;
    const uint8_t *base;
    int pitch, records;
    uint32_t offset[N];
    __device__ static int at(int row, int chunk) {
        return row * COLS + (chunk ^ (C == 4 ? (row >> 2) & 3 : (row >> 3) & 1)) * 16;
    }
    __device__ CodeLoader(const uint8_t *codes, int first, int n) {
        pitch = (n + 31) / 32 * 32;
        base = codes + (long long)first * pitch;
        const int last = min(ROWS, n - first) - 1;
        records = (last + 1) * pitch;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int k = (int)threadIdx.x + i * NT, row = k / C, c = (at(row, k % C) - row * COLS) / 16;
            offset[i] = (uint32_t)(min(row, last) * pitch + c * 16);
        }
    }
    __device__ void issue(int column, uint8_t *lds) const {
        const uint64_t from = (uint64_t)(base + column);
        i32x4 rsrc;
        rsrc[0] = __builtin_amdgcn_readfirstlane((int)from);
        rsrc[1] = __builtin_amdgcn_readfirstlane((int)((from >> 32) & 0xFFFFu));
        rsrc[2] = __builtin_amdgcn_readfirstlane(records - column);
        rsrc[3] = 0x00027000;
        const uint32_t to = __builtin_amdgcn_readfirstlane(lds_address(lds) + (threadIdx.x & ~63u) * 16);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (ROWS * C % NT != 0 && (int)(threadIdx.x & ~63u) + i * NT >= ROWS * C) break;
            load_to_lds(rsrc, offset[i], to + i * NT * 16);
        }
    }
    // codes of the columns first .. first + 3 (a multiple of four)
    __device__ static uint32_t read(const uint8_t *lds, int row, int first) {
        return *(const uint32_t *)(lds + at(row, first >> 4) + (first & 15));
    }
};

// everything this workgroup's loads and writes put into LDS is there, and nobody reads the buffer before it any more
template <bool DIRECT>
__device__ inline void tile_ready() {
    if (DIRECT) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
}

// Rows and statistics read before the loop are there: without this the compiler waits for them at their first use
// inside it, and with them for the tiles in flight, again in every round.
__device__ inline void loads_done() { __builtin_amdgcn_s_waitcnt(0x0F70); }          // vmcnt(0)

// Order of as many LDS reads and products that the compiler has put into one block: a few reads first, then one behind
// every product.  By itself it reads every operand of the forward pass's scores right before its product and waits.
template <typename T, int N>
__device__ inline void interleave() {
    if constexpr (sizeof(T) == 2) {
        constexpr int AHEAD = N < 6 ? N : 6;
        __builtin_amdgcn_sched_group_barrier(0x100, AHEAD, 0);
#pragma unroll
        for (int i = 0; i < N - AHEAD; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, AHEAD, 0);
    }
}

__device__ inline float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }     // one instruction

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

// a transposed result, DT tiles of 32 elements: lane l % 32 is the row, its registers four elements each.  LOW: what
// the rounding to T left over, as T.
template <bool LOW, typename T, int DT>
__device__ inline void store_rows(T *row, int dim, int h, const f32x16 (&acc)[DT], float scale) {
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int d = 32 * dt + 8 * g + 4 * h;
            typename RwkPack<T, 4>::type v;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float x = acc[dt][4 * g + e] * scale;
                v[e] = LOW ? (T)(x - (float)(T)x) : (T)x;
            }
            if (d + 4 <= dim) {
                rwk_store<T, 4>(row + d, v);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (d + e < dim) row[d + e] = v[e];
            }
        }
}

// Result of the second product: DT tiles of 32 elements by the wavefront's 32 rows.
template <typename T, int KS>
struct Result {
    f32x16 a[Shape<T, KS>::DT];
    __device__ void clear() {
#pragma unroll
        for (auto &x : a) x = f32x16{};
    }
    __device__ void scale(float by) {             // of the lane's row
#pragma unroll
        for (auto &x : a)
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] *= by;
    }
    // `f`: eight weights of the lane's row, for the tile's rows first .. first + 15 as column_operand has them
    template <typename F>
    __device__ void add(const T *tile, int first, const F &f, int lane) {
#pragma unroll
        for (int dt = 0; dt < Shape<T, KS>::DT; ++dt) a[dt] = mma(column_operand<T, KS>(tile, first, dt, lane), f, a[dt]);
    }
    // the same with what the rounding of the weights left over
    __device__ void add(const T *tile, int first, const Frag<T> &f, const Frag<T> &rest, int lane) {
#pragma unroll
        for (int dt = 0; dt < Shape<T, KS>::DT; ++dt) {
            const Frag<T> x = column_operand<T, KS>(tile, first, dt, lane);
            a[dt] = mma(x, f, mma(x, rest, a[dt]));
        }
    }
    __device__ void finish() {}
};

// fp32, up to 16 elements: a tile of 32 would be half empty, and the products are what bounds such kernels.  Two tiles
// of 16 elements by 16 rows instead, the summed index four at a time: a lane gives away the weights of the row that its
// neighbouring sixteen lanes hold and takes theirs for another key (2 of 3 products' time; 1024 protein-sized graphs,
// 4 heads of 16: 2.62 to 2.20 ms).
struct SwappedRows { float low, high; };
__device__ inline SwappedRows swap_rows(float x, float y) {          // lanes 16-31, 48-63 of x with 0-15, 32-47 of y
    const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, y), false, false);
    return {__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1])};
}
template <>
struct Result<float, 1> {
    typedef float f32x4 __attribute__((ext_vector_type(4)));
    using S = Shape<float, 1>;
    f32x4 low, high;                              // rows 0 - 15 and 16 - 31: lane l row l % 16, elements 4 (l / 16) ..
    f32x16 a[1];
    __device__ void clear() { low = high = f32x4{}; }
    __device__ void scale(float by) {
        const SwappedRows r = swap_rows(by, by);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            low[e] *= r.low;
            high[e] *= r.high;
        }
    }
    __device__ void add(const float *tile, int first, const Frag<float> &f, int lane) {
        const int odd = (lane >> 4) & 1, col = lane & 15;
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            const int row = first + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3) + odd;
            const float x = tile[S::at(row, col >> 2) + (col & 3)];
            const SwappedRows r = swap_rows(f.v[e], f.v[e + 1]);
            low = __builtin_amdgcn_mfma_f32_16x16x4f32(x, r.low, low, 0, 0, 0);
            high = __builtin_amdgcn_mfma_f32_16x16x4f32(x, r.high, high, 0, 0, 0);
        }
    }
    __device__ void finish() {                    // as a 32 x 32 result, elements 16 .. 31 zeros
        a[0] = f32x16{};
        float x[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const SwappedRows r = swap_rows(low[e], high[e]);
            const auto t = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, r.low),
                                                            __builtin_bit_cast(uint32_t, r.high), false, false);
            x[e] = __builtin_bit_cast(float, (uint32_t)t[0]);
            x[4 + e] = __builtin_bit_cast(float, (uint32_t)t[1]);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) a[0][i] = x[i];
    }
};

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
// of a launch over key / value heads and the parts of their query heads
__device__ inline Place key_place(const RwkAttnArgs &p, long long b, int *part) {
    Place s = place_of(p, b);
    *part = s.item % p.parts;
    s.item /= p.parts;
    s.head += *part * p.part_heads;
    find_rows(p, s);
    return s;
}

// code e of four, at most n_buckets
__device__ inline int code_of(uint32_t codes, int e, int nb) { return min((int)((codes >> (8 * e)) & 255u), nb); }

// The bias gradient's sums of a dQ workgroup: every thread its own per bucket, NT floats apart, without atomics.  (The
// LDS float atomic works through its lanes one by one: 180 cycles for a wavefront's 64 separate places, measured.)
// SPLIT: four sets of them, one per place among four neighbouring pairs, each with a slot for the pairs that have no
// bucket, so that four values are read, added and written without a look at each other's codes (fp32, 8 buckets, 1024
// protein-sized graphs: dQ in seven eighths of the time).  Otherwise all four
// sums are read before the first is written, and an equal code before takes the place of what was read.
template <int NT, bool SPLIT>
struct BucketSums {
    float *at;
    int nb;
    __device__ static int slots(int nb) { return SPLIT ? 4 * (nb + 1) : nb; }
    __device__ BucketSums(float *sums, int nb_) : at(sums + threadIdx.x), nb(nb_) {
        for (int b = 0; b < slots(nb); ++b) at[b * NT] = 0.f;
    }
    __device__ void add(uint32_t codes, const float *x) {       // a masked pair's 0 to any
        int c[4];
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            c[e] = SPLIT ? e * (nb + 1) + code_of(codes, e, nb) : code_of(codes, e, nb - 1);
            v[e] = at[c[e] * NT];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (!SPLIT) {
#pragma unroll
                for (int f = 0; f < e; ++f) v[e] = c[f] == c[e] ? v[f] : v[e];
            }
            v[e] += x[e];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) at[c[e] * NT] = v[e];
    }
    __device__ void add_all(uint32_t codes, const float (&x)[16]) {       // of one code
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) sum += x[i];
        at[code_of(codes, 0, SPLIT ? nb : nb - 1) * NT] += sum;
    }
    __device__ void times_zero() {
        for (int b = 0; b < slots(nb); ++b) at[b * NT] *= 0.f;
    }
    // the lane's part of a bucket's sum over the workgroup, in a fixed order
    __device__ float part(int b) const {
        const float *from = at - threadIdx.x + (threadIdx.x & 63);
        float v = 0.f;
#pragma unroll
        for (int e = 0; e < (SPLIT ? 4 : 1); ++e)
#pragma unroll
            for (int w = 0; w < NT; w += 64) v += from[(e * (nb + 1) + b) * NT + w];
        return v;
    }
};

// product of a probability and a value: 0 where the probability is 0 (a masked pair), whatever the value
// (v_mul_legacy_f32)
extern "C" __device__ float rwk_mul_legacy(float, float) __asm("llvm.amdgcn.fmul.legacy");
__device__ inline float weigh(float p, float x) { return rwk_mul_legacy(p, x); }

// The bias of one head times log2(e), bucket b in lane b of every wavefront, -infinity from n_buckets on (a pair that
// does not attend): a look-up fetches another lane's register.  Finite entries stay finite, the type's lowest value too:
// a row that has nothing else weighs its pairs alike.
template <typename T>
__device__ inline float load_table(const RwkAttnArgs &p, int head) {
    const int b = (int)(threadIdx.x & 63);
    const float x = b < p.a.n_buckets ? (float)((const T *)p.a.table)[(long long)head * p.a.n_buckets + b] : -INFINITY;
    const float most = 3.402823466e38f;
    return fabsf(x) <= most ? fminf(fmaxf(x * kLog2e, -most), most) : x;
}
__device__ inline float look_up(float table, int bucket) {
    return __builtin_bit_cast(float, __builtin_amdgcn_ds_bpermute(4 * bucket, __builtin_bit_cast(int, table)));
}

// Adds the bias to a lane's 16 products, `codes` their four words.  Far from each other pairs mostly share a bucket - rows
// beyond the longest distance that has one of its own, nodes that no walk joins: where every lane of the wavefront has
// one code for all its 16 pairs, one look-up does and the codes stay packed (64 walks of up to 1024 rows, 8 heads of 64
// in bf16, 32 buckets by distance: 418 to 380 us).  Returns whether it was so.
__device__ inline bool add_bias(float (&s)[16], const uint32_t (&codes)[4], float scale, float table, int nb) {
    const uint32_t all = (codes[0] & 255u) * 0x01010101u;
    const uint32_t differ = ((codes[0] ^ all) | (codes[1] ^ all)) | ((codes[2] ^ all) | (codes[3] ^ all));
    if (__builtin_amdgcn_ballot_w64(differ != 0) == 0) {
        const int b = code_of(all, 0, nb);
        const float bias = look_up(table, b);
        const bool on = b < nb;
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = on ? fmaf(s[i], scale, bias) : -INFINITY;
        return true;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int b = code_of(codes[i >> 2], i & 3, nb);
        const float x = fmaf(s[i], scale, look_up(table, b));
        s[i] = b < nb ? x : -INFINITY;
    }
    return false;
}

// How the backward pass has a row's probabilities again: exp2((score + start) c) * factor.  16-bit types without a bias
// begin their products at a start that holds the logarithm of the factor too, and save the product.  With a bias that
// would be lost beside a large reference - a row all of whose pairs carry a mask's -1e9 - and for fp32 the rounding of
// the larger exponent would be the largest error of all: there the exponentials are the forward pass's, bit for bit.
// start -infinity for a row without pairs and for rows that do not exist.  `up`: the weights times 2^up.
template <typename T, bool BIAS>
struct RowWeight {
    static constexpr bool FOLDED = sizeof(T) == 2 && !BIAS;
    float start, factor;
    __device__ RowWeight(float ref, float inv, float c, int up = 0) {
        start = FOLDED ? (__log2f(inv) + (float)up) / c - ref : inv == 0.f ? -INFINITY : -ref;
        factor = ldexpf(inv, up);
    }
    // what the product begins at, and the weight from what it ends at or, with a bias, from the score
    __device__ float begin() const { return FOLDED ? start : 0.f; }
    __device__ static float weight(float x, float start, float factor, float c) {
        if (FOLDED) return exp2_fast(x * c);
        return exp2_fast(BIAS ? x + start : (x + start) * c) * factor;
    }
    __device__ float of(float score, float c) const { return weight(score + begin(), start, factor, c); }
};

// fp16 in the backward pass: its normal numbers end at 2^-14, and weights of many keys and gradients of scores - a weight
// times a gradient - lie below that long before the results do (d_out of 1e-4, 4096 keys: a fifth of all ds would round to
// 0).  dK/dV takes the weights times 2^kWeightUp, normal down to 2^-26 and far from the largest number, as no weight
// exceeds 1 by more than its exponent's rounding.  The ds have no such bound: a wavefront multiplies them by a power of two
// of its own for each of its rows (dQ) or keys (dK), which begins large and shrinks when a ds would pass 2^15, to where
// that one is below 2^13; the sums shrink with it and are divided by it at the end.  Eight maxima of three and a branch per
// 32 x 32 pairs: 48 prompts of up to 1500 rows, 64 elements, forward and backward 559 to 591 us.
template <typename T> constexpr bool kNarrowRange = sizeof(T) == 2 && (T)1e-30f == (T)0.f;
template <typename T> constexpr int kWeightUp = kNarrowRange<T> ? 12 : 0;
template <typename T>
struct GradientScale {
    static constexpr float TOP = 0x1p15f;
    float by = kNarrowRange<T> ? 0x1p60f : 1.f, limit = TOP / 0x1p60f;
    // makes room for these ds in `acc`, the sums of the ones before, and multiplies them
    template <typename R>
    __device__ void apply(float (&x)[16], R &acc) {
        if constexpr (kNarrowRange<T>) {
            float most = 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i) most = fmaxf(most, fabsf(x[i]));
            if (__builtin_amdgcn_ballot_w64(most > limit) != 0) {
                most = fmaxf(most, __shfl_xor(most, 32, 64));          // both halves of a row or key
                const float now = most > limit ? fminf(by, ldexpf(1.f, 13 - __builtin_amdgcn_frexp_expf(most))) : by;
                acc.scale(now / by);
                by = now;
                limit = TOP / now;
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] *= by;
        }
    }
    // the sums as they are
    template <typename R>
    __device__ void undo(R &acc, int up) const {
        if constexpr (kNarrowRange<T>) acc.scale(ldexpf(1.f / by, -up));
    }
};

// ---------------------------------------------------------------------------------------------------------------
// A pair that does not attend counts for nothing whatever its rows hold, but a matrix instruction adds 0 times what it
// finds: not a number where that is not finite.  So rows whose result is not finite are computed again - if pairs that do
// not attend can be the reason: there are such pairs (a causal mask: in the tiles on the diagonal only) and one of their
// rows does hold something that is not finite.  An overflow in d_out, say, is none for dQ, whose products take keys.  The
// second time what is not finite is taken out of the operands and counted where it is weighed: elements whose sum would
// have had any come out as NaN, the others as they should.  The operands come from memory, 32 elements of a result in a
// pass with all of its scores over again, which needs few registers, so that the code costs the kernels' loops none; a
// pass ends early once nothing is left that could be finite.
// ---------------------------------------------------------------------------------------------------------------
// whether the lane's row is not finite
template <int KS, int DT>
__device__ inline bool not_finite(const f32x16 (&acc)[DT]) {
    constexpr int N = KS == 1 ? 8 : 16;           // KS = 1: the upper half is no element's
    float t = 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int i = 0; i < N; ++i) t = fmaf(acc[dt][i], 0.f, t);
    t += __shfl_xor(t, 32, 64);
    return t != t;                                // 0 times infinity, or NaN
}
__device__ inline bool any_lane(bool x) { return __builtin_amdgcn_ballot_w64(x) != 0; }

// whether rows lo .. hi - 1 of a head, `base` its first, hold anything that is not finite: the wavefront together
template <typename T>
__device__ inline bool holds_not_finite(const T *base, long long stride, int lo, int hi, int dim) {
    float t = 0.f;
#pragma unroll 1
    for (int r = lo + (int)(threadIdx.x & 63); r < hi; r += 64)
#pragma unroll 1
        for (int d = 0; d < dim; d += 8) {
            const Frag<T> x = load_global<T>(base + r * stride, d, dim);
#pragma unroll
            for (int e = 0; e < 8; ++e) t = fmaf((float)x.v[e], 0.f, t);
        }
    return any_lane(t != t);
}

// products of the lane's row with 32 rows of a head, from `first` (the last of n for those behind it): a transposed result
template <typename T>
__device__ inline f32x16 row_products(const T *base, long long stride, int first, int n, const T *row, int dim) {
    const int lane = threadIdx.x & 63, h = lane >> 5;
    const T *other = base + min(first + (lane & 31), n - 1) * stride;
    f32x16 x = f32x16{};
#pragma unroll 1
    for (int d = 8 * h; d < dim + 8 * h; d += 16)              // both halves in the same rounds
        x = mma(load_global<T>(other, d, dim), load_global<T>(row, d, dim), x);
    return x;
}

// 32 elements, from `d`, of a sum over rows of a head: what is finite, and how often anything else was weighed
template <typename T>
struct FiniteSum {
    f32x16 sum = f32x16{}, spoilt = f32x16{};
    // eight weights of the lane's row, for the rows first .. first + 15 of n as column_operand has them
    __device__ void add(const T *base, long long stride, int first, int n, int d, int dim, const float (&weight)[16], int s) {
        const int lane = threadIdx.x & 63, h = lane >> 5, col = d + (lane & 31);
        Frag<T> x, other, on;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int row = first + 8 * (e >> 2) + 4 * h + (e & 3);
            const float v = (float)base[min(row, n - 1) * stride + min(col, dim - 1)];      // no branches
            const bool there = row < n && col < dim, finite = fabsf(v) <= 3.402823466e38f;
            x.v[e] = (T)(there && finite ? v : 0.f);
            other.v[e] = (T)(there && !finite ? 1.f : 0.f);
            on.v[e] = (T)(weight[8 * s + e] == 0.f ? 0.f : 1.f);
        }
        const Frag<T> f = pack<T>(weight, s);
        sum = mma(x, f, sum);
        if constexpr (sizeof(T) == 2) sum = mma(x, left_over<T>(weight, f, s), sum);
        spoilt = mma(other, on, spoilt);
    }
    // whether no element of any of the wavefront's rows that count can be finite any more
    __device__ bool lost(int d, int dim, bool mine) const {
        const int h = (int)(threadIdx.x >> 5) & 1;
        bool all = true;
#pragma unroll
        for (int i = 0; i < 16; ++i) all = all && (d + reg_row(i, h) >= dim || sum[i] != sum[i] || spoilt[i] > 0.f);
        return !any_lane(mine && !all);
    }
    // LOW: what the rounding to R left over
    template <bool LOW, typename R>
    __device__ void store(R *row, int d, int dim, float undo, float scale) const {
        const int h = (int)(threadIdx.x >> 5) & 1;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float x = spoilt[i] > 0.f ? __builtin_nanf("") : sum[i] * undo * scale;
            if (d + reg_row(i, h) < dim) row[d + reg_row(i, h)] = LOW ? (R)(x - (float)(R)x) : (R)x;
        }
    }
};

// exponent (less the reference's part) of pair (q, k) from its product, -infinity if it does not attend
template <bool BIAS>
__device__ inline float pair_score(const RwkAttnArgs &p, const Place &at, float table, int q, int k, float product) {
    bool on = q < at.n && k < at.n && !(p.a.causal != 0 && k > q);
    float x = product;
    if (BIAS) {
        const int nb = (int)p.a.n_buckets;
        const int b = min((int)p.a.codes[p.a.code_start[at.seg] + (long long)min(q, at.n - 1) * ((at.n + 31) / 32 * 32) +
                                         min(k, at.n - 1)], nb);
        x = fmaf(product, p.a.scale * kLog2e, look_up(table, b));
        on = on && b < nb;
    }
    return on ? x : -INFINITY;
}

// row `row` of a head; 0 for the first of the segment
template <typename T>
__device__ inline const T *row_of(const void *base, const Place &at, int row, long long stride, long long head, long long head_stride) {
    return (const T *)base + (at.base + row) * stride + head * head_stride;
}

// Whether pairs of the wavefront's rows from q0 that do not attend may be why a result is not finite: `base` holds what
// is weighed, the keys or the values.
template <typename T, bool BIAS>
__device__ inline bool masked_may_spoil(const RwkAttnArgs &p, const Place &at, const T *base, long long stride, int q0, int end) {
    if (!BIAS && p.a.causal == 0) return false;
    // causal: tiles of at most 64 keys, the last of which begins no later than the wavefront's last row
    return holds_not_finite(base, stride, BIAS ? 0 : q0, min(at.n, BIAS ? end + 32 : q0 + 64 + 32), (int)p.a.dim);
}

template <typename T, bool BIAS>
__device__ inline void again_forward(const RwkAttnArgs &p, const Place &at, float table, int q, int end, float base,
                                     float factor, float c, bool mine) {
    const int h = (int)(threadIdx.x >> 5) & 1, dim = (int)p.a.dim, qc = min(q, at.n - 1);
    const T *q_row = row_of<T>(p.a.q, at, qc, p.a.q_row, at.head, p.a.q_head);
    const T *keys = row_of<T>(p.a.k, at, 0, p.a.k_row, at.kv_head, p.a.k_head);
    const T *values = row_of<T>(p.a.v, at, 0, p.a.v_row, at.kv_head, p.a.v_head);
    const long long to = ((at.base + qc) * p.a.heads + at.head) * dim;
#pragma unroll 1
    for (int d = 0; d < dim; d += 32) {
        FiniteSum<T> o;
#pragma unroll 1
        for (int k0 = 0; k0 < end; k0 += 32) {
            float s[16];
            unpack(row_products(keys, p.a.k_row, k0, at.n, q_row, dim), s);
#pragma unroll
            for (int i = 0; i < 16; ++i)
                s[i] = exp2_fast((pair_score<BIAS>(p, at, table, q, k0 + reg_row(i, h), s[i]) - base) * c);
#pragma unroll
            for (int u = 0; u < 2; ++u) o.add(values, p.a.v_row, k0 + 16 * u, at.n, d, dim, s, u);
            if (o.lost(d, dim, mine)) break;
        }
        if (mine) o.template store<false>((T *)p.a.out + to, d, dim, 1.f, factor);
        if (mine && p.a.out_low != nullptr) o.template store<true>((T *)p.a.out_low + to, d, dim, 1.f, factor);
    }
}

template <typename T, bool BIAS>
__device__ inline void again_dq(const RwkAttnArgs &p, const Place &at, float table, int q, int end,
                                const RowWeight<T, BIAS> &weight, float delta, float c, float by, float scale, bool mine) {
    const int h = (int)(threadIdx.x >> 5) & 1, dim = (int)p.a.dim, qc = min(q, at.n - 1);
    const T *q_row = row_of<T>(p.a.q, at, qc, p.a.q_row, at.head, p.a.q_head);
    const T *o_row = row_of<T>(p.a.d_out, at, qc, p.a.do_row, at.head, p.a.do_head);
    const T *keys = row_of<T>(p.a.k, at, 0, p.a.k_row, at.kv_head, p.a.k_head);
    const T *values = row_of<T>(p.a.v, at, 0, p.a.v_row, at.kv_head, p.a.v_head);
#pragma unroll 1
    for (int d = 0; d < dim; d += 32) {
        FiniteSum<T> g;
#pragma unroll 1
        for (int k0 = 0; k0 < end; k0 += 32) {
            float s[16], dp[16];
            unpack(row_products(keys, p.a.k_row, k0, at.n, q_row, dim), s);
            unpack(row_products(values, p.a.v_row, k0, at.n, o_row, dim), dp);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float x = pair_score<BIAS>(p, at, table, q, k0 + reg_row(i, h), s[i]);
                s[i] = weigh(weight.of(x, c), dp[i] - delta) * by;
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) g.add(keys, p.a.k_row, k0 + 16 * u, at.n, d, dim, s, u);
            if (g.lost(d, dim, mine)) break;
        }
        if (mine) g.template store<false>((T *)p.a.dq + ((at.base + qc) * p.a.heads + at.head) * dim, d, dim, 1.f / by, scale);
    }
}

// Where dK and dV of a part of the query heads go: straight out, or as fp32 sums for dkv_sum_kernel.
struct KeyGradients {
    long long at;                                 // of the workgroup's first key
    float *dk, *dv;                               // a part's sums, or null
    __device__ KeyGradients(const RwkAttnArgs &p, const Place &s, int part) {
        const long long n = p.a.rows * p.a.kv_heads * p.a.dim;
        at = (s.base * p.a.kv_heads + s.kv_head) * p.a.dim;
        dk = dv = nullptr;
        if (p.parts > 1) {
            dk = p.a.dkv_partials + 2 * part * n + at;
            dv = dk + n;
        }
    }
};

// as masked_may_spoil, for the wavefront's keys from k0: queries and d_out
template <typename T, bool BIAS>
__device__ inline bool masked_may_spoil_keys(const RwkAttnArgs &p, const Place &at, int k0, int begin) {
    if (!BIAS && p.a.causal == 0) return false;
    const int lo = BIAS ? begin : k0, hi = BIAS ? at.n : min(at.n, k0 + 64);
    bool any = false;
#pragma unroll 1
    for (int head = at.head; head < at.head + p.part_heads && !any; ++head)
        any = holds_not_finite(row_of<T>(p.a.q, at, 0, p.a.q_row, head, p.a.q_head), p.a.q_row, lo, hi, (int)p.a.dim) ||
              holds_not_finite(row_of<T>(p.a.d_out, at, 0, p.a.do_row, head, p.a.do_head), p.a.do_row, lo, hi, (int)p.a.dim);
    return any;
}

template <typename T, bool BIAS>
__device__ inline void again_dkv(const RwkAttnArgs &p, const Place &at, int part, int k, int begin, float c, float by,
                                 float dk_scale, bool mine) {
    const int h = (int)(threadIdx.x >> 5) & 1, dim = (int)p.a.dim, kc = min(k, at.n - 1);
    const T *k_row = row_of<T>(p.a.k, at, kc, p.a.k_row, at.kv_head, p.a.k_head);
    const T *v_row = row_of<T>(p.a.v, at, kc, p.a.v_row, at.kv_head, p.a.v_head);
    const KeyGradients out(p, at, part);
    const long long to = kc * p.a.kv_heads * dim;
#pragma unroll 1
    for (int pass = 0; pass < 2; ++pass) {                     // dK, then dV
        const float times = ldexpf(pass == 0 ? by : 1.f, kWeightUp<T>), scale = pass == 0 ? dk_scale : 1.f;
        float *sums = pass == 0 ? out.dk : out.dv;
        T *result = (pass == 0 ? (T *)p.a.dk : (T *)p.a.dv) + out.at;
#pragma unroll 1
        for (int d = 0; d < dim; d += 32) {
            FiniteSum<T> g;
            bool lost = false;
#pragma unroll 1
            for (int head = at.head; head < at.head + p.part_heads && !lost; ++head) {
                const float table = BIAS ? load_table<T>(p, head) : 0.f;
                const T *queries = row_of<T>(p.a.q, at, 0, p.a.q_row, head, p.a.q_head);
                const T *grads = row_of<T>(p.a.d_out, at, 0, p.a.do_row, head, p.a.do_head);
#pragma unroll 1
                for (int q0 = begin; q0 < at.n && !lost; q0 += 32) {
                    float s[16], dp[16];
                    unpack(row_products(queries, p.a.q_row, q0, at.n, k_row, dim), s);
                    f32x16 x = f32x16{};
                    if (pass == 0) x = row_products(grads, p.a.do_row, q0, at.n, v_row, dim);
                    unpack(x, dp);
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int q = q0 + reg_row(i, h);
                        const long long st = head * p.a.rows + at.base + min(q, at.n - 1);
                        const RowWeight<T, BIAS> weight(p.a.stats[2 * st], p.a.stats[2 * st + 1], c);
                        const float w = weight.of(pair_score<BIAS>(p, at, table, q, k, s[i]), c);
                        s[i] = (pass == 0 ? weigh(w, dp[i] - p.a.delta[st]) : w) * times;
                    }
                    const T *from = pass == 0 ? queries : grads;
                    const long long stride = pass == 0 ? p.a.q_row : p.a.do_row;
#pragma unroll
                    for (int u = 0; u < 2; ++u) g.add(from, stride, q0 + 16 * u, at.n, d, dim, s, u);
                    lost = g.lost(d, dim, mine);
                }
            }
            if (mine && p.parts > 1) g.template store<false>(sums + to, d, dim, 1.f / times, scale);
            else if (mine) g.template store<false>(result + to, d, dim, 1.f / times, scale);
        }
    }
}

// Bytes of LDS for the tiles: two buffers of two, and the elements that the second product of KS = 1 reads past the
// last row.
template <typename T, int KS, int ROWS> constexpr int tile_bytes() { return ROWS * 16 * KS * (int)sizeof(T); }
template <typename T, int KS, int ROWS> constexpr int tiles_bytes() {
    return 4 * tile_bytes<T, KS, ROWS>() + (KS == 1 ? 32 * (int)sizeof(T) : 0);
}
// bytes of LDS behind the tiles for a bias: two buffers of codes of 32 NW rows and as many columns as the other
// operand's tile has rows
template <int NW, int COLS> constexpr int code_bytes() { return 2 * 32 * NW * COLS; }
template <typename T, int NW> constexpr int tile_rows() { return sizeof(T) == 2 && NW > 1 ? 64 : 32; }

// Scores below the reference by this much or less (in powers of two) leave it as it is: the sums and the output are
// rescaled only when a row's maximum has grown by that factor in its exponential, and stay far inside fp32's range.
// fp16: the weights are 2^6 times the exponentials and so at most 2^13 - 2^15 where a large bias leaves the reference no
// digits for the 6 - and keys that a row hardly looks at count down to 2^-31 of its largest weight, by thousands of them.
template <typename T> constexpr float kSlack = kNarrowRange<T> ? 7.f : 8.f;
template <typename T> constexpr int kExpUp = kNarrowRange<T> ? 6 : 0;

// FINE (16-bit types): a weight meets the values as two numbers of the type, the second what the rounding to the first
// left over.  The weights' rounding counts most where few of them are added up and, through delta, which comes from the
// output, in the query gradients of narrow heads.  Half as many products more, and the registers of a wavefront per
// SIMD: 48 prompts of up to 1500 rows, 64 elements, 193 us against 149; so wide heads have it for short segments only.
template <typename T, int KS, int NW, bool BIAS, bool FINE, bool ASYNC>
__global__ void __launch_bounds__(64 * NW, (sizeof(T) == 2 && ASYNC && !(FINE && KS == 8)) || KS == 1 ? 2 : 1)
attention_forward_kernel(const RwkAttnArgs p) {
    using S = Shape<T, KS>;
    constexpr int NT = 64 * NW, DT = S::DT, BN = tile_rows<T, NW>(), TN = BN / 32;
    extern __shared__ __attribute__((aligned(16))) char attn_lds[];
    T *tiles = (T *)attn_lds;                                       // buffer b: keys at 2 b, values at 2 b + 1
    uint8_t *codes = (uint8_t *)attn_lds + tiles_bytes<T, KS, BN>();
    typedef CodeLoader<32 * NW, BN, NT> Codes;
    const Place at = query_place(p, blockIdx.x);
    const int lane = threadIdx.x & 63, h = lane >> 5, dim = (int)p.a.dim, n = at.n;
    const int q0 = at.first + 32 * (int)(threadIdx.x >> 6), q = q0 + (lane & 31), qc = q < n ? q : n - 1;
    const bool causal = p.a.causal != 0;
    const int nb = (int)p.a.n_buckets;
    const float table = BIAS ? load_table<T>(p, at.head) : 0.f;

    TileLoader<T, KS, BN, NT, ASYNC> keys((const T *)p.a.k + at.base * p.a.k_row + at.kv_head * p.a.k_head, p.a.k_row, n, dim);
    TileLoader<T, KS, BN, NT, ASYNC> values((const T *)p.a.v + at.base * p.a.v_row + at.kv_head * p.a.v_head, p.a.v_row, n, dim);
    keys.issue(0, tiles);
    values.issue(0, tiles + BN * S::W);
    Frag<T> qf[KS];
    const T *q_row = (const T *)p.a.q + (at.base + qc) * p.a.q_row + at.head * p.a.q_head;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[ks] = load_global<T>(q_row, 16 * ks + 8 * h, dim);
    const Codes code_tiles(BIAS ? p.a.codes + p.a.code_start[at.seg] : nullptr, at.first, n);
    if (BIAS) code_tiles.issue(0, codes);

    // without a bias the maximum is taken over q . k and the scale meets it in the exponent; with one the scores are
    // the sum, in units of log2(e) (load_table)
    const float scale = p.a.scale * kLog2e, c = BIAS ? 1.f : scale, slack = kSlack<T> / c;
    Result<T, KS> acc;
    acc.clear();
    float ref = -INFINITY, sum = 0.f;           // ref: what the exponentials are taken relative to
    const int end = causal && at.first + 32 * NW < n ? at.first + 32 * NW : n;
    keys.commit(tiles);
    values.commit(tiles + BN * S::W);
    loads_done();
    for (int k0 = 0, turn = 0; k0 < end; k0 += BN, turn ^= 1) {
        const T *k_tile = tiles + 2 * turn * BN * S::W, *v_tile = k_tile + BN * S::W;
        T *next = tiles + 2 * (turn ^ 1) * BN * S::W;
        tile_ready<ASYNC || BIAS>();
        if (k0 + BN < end) {
            keys.issue(k0 + BN, next);
            values.issue(k0 + BN, next + BN * S::W);
            if (BIAS) code_tiles.issue(k0 + BN, codes + (turn ^ 1) * 32 * NW * BN);
        }
        if (q0 < n && !(causal && k0 > q0 + 31)) {
            float s[TN][16];
#pragma unroll
            for (int t = 0; t < TN; ++t) {
                f32x16 x = f32x16{};
#pragma unroll
                for (int ks = 0; ks < KS; ++ks)
                    x = mma(row_operand<T, KS>(k_tile, 32 * t + (lane & 31), ks, h), qf[ks], x);
                unpack(x, s[t]);
            }
            interleave<T, TN * KS>();
            if (BIAS) {
#pragma unroll
                for (int t = 0; t < TN; ++t) {
                    uint32_t four[4];
#pragma unroll
                    for (int g = 0; g < 4; ++g)
                        four[g] = Codes::read(codes + turn * 32 * NW * BN, q - at.first, 32 * t + 8 * g + 4 * h);
                    add_bias(s[t], four, scale, table, nb);
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
            const bool grown = here > ref + slack || (ref == -INFINITY && here > -INFINITY);
            if (__builtin_amdgcn_ballot_w64(grown) != 0) {
                const float now = grown ? here : ref;
                const float shrink = ref == now ? 1.f : exp2_fast((ref - now) * c);
                ref = now;
                sum *= shrink;
                acc.scale(shrink);
            }
            const float base = (ref == -INFINITY ? 0.f : ref) - (BIAS ? kExpUp<T> : 0), base_c = base * c - kExpUp<T>;
            float part = 0.f;
#pragma unroll
            for (int t = 0; t < TN; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    // fp32: the difference first, which is exact near the maximum
                    s[t][i] = exp2_fast(BIAS             ? s[t][i] - base
                                        : sizeof(T) == 4 ? (s[t][i] - base) * c
                                                         : fmaf(s[t][i], c, -base_c));
                    part += s[t][i];
                }
            sum += part;
#pragma unroll
            for (int t = 0; t < TN; ++t)
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const Frag<T> f = pack<T>(s[t], u);
                    if constexpr (sizeof(T) == 2 && FINE)
                        acc.add(v_tile, 32 * t + 16 * u, f, left_over<T>(s[t], f, u), lane);
                    else
                        acc.add(v_tile, 32 * t + 16 * u, f, lane);
                }
        }
        keys.commit(next);
        values.commit(next + BN * S::W);
    }
    acc.finish();
    sum += __shfl_xor(sum, 32, 64);
    const float inv = sum == 0.f ? 0.f : 1.f / sum;      // a row without pairs: zeros
    // what pairs' weights follow from: exp2((score - base) c) * factor
    const float base = (ref == -INFINITY ? 0.f : ref) - (BIAS ? kExpUp<T> : 0), factor = BIAS ? inv : ldexpf(inv, kExpUp<T>);
    const long long o_at = ((at.base + qc) * p.a.heads + at.head) * dim;
    bool again = q < n && not_finite<KS>(acc.a);
    if (any_lane(again) && !masked_may_spoil<T, BIAS>(p, at, values.base, p.a.v_row, q0, end)) again = false;
    if (q < n && !again) {
        store_rows<false, T, DT>((T *)p.a.out + o_at, dim, h, acc.a, inv);
        if (p.a.out_low != nullptr) store_rows<true, T, DT>((T *)p.a.out_low + o_at, dim, h, acc.a, inv);
    }
    if (any_lane(again)) again_forward<T, BIAS>(p, at, table, q, end, base, factor, c, again);
    if (q < n && p.a.stats != nullptr && h == 0) {
        float *st = p.a.stats + 2 * (at.head * p.a.rows + at.base + q);
        st[0] = base;
        st[1] = factor;
    }
}

template <typename T, int KS, int NW, bool BIAS, bool SPLIT, bool ASYNC>
__global__ void __launch_bounds__(64 * NW, (sizeof(T) == 2 && ASYNC && (!BIAS || KS < 8)) || KS == 1 ? 2 : 1)
attention_dq_kernel(const RwkAttnArgs p) {
    using S = Shape<T, KS>;
    constexpr int NT = 64 * NW, DT = S::DT, BN = tile_rows<T, NW>(), TN = BN / 32;
    extern __shared__ __attribute__((aligned(16))) char attn_lds[];
    T *tiles = (T *)attn_lds;
    uint8_t *codes = (uint8_t *)attn_lds + tiles_bytes<T, KS, BN>();
    typedef CodeLoader<32 * NW, BN, NT> Codes;
    const Place at = query_place(p, blockIdx.x);
    const int lane = threadIdx.x & 63, h = lane >> 5, dim = (int)p.a.dim, n = at.n;
    const int q0 = at.first + 32 * (int)(threadIdx.x >> 6), q = q0 + (lane & 31), qc = q < n ? q : n - 1;
    const bool causal = p.a.causal != 0;
    const int nb = (int)p.a.n_buckets;
    const float table = BIAS ? load_table<T>(p, at.head) : 0.f;
    BucketSums<NT, SPLIT> buckets((float *)(codes + 2 * 32 * NW * BN), BIAS ? nb : 0);

    TileLoader<T, KS, BN, NT, ASYNC> keys((const T *)p.a.k + at.base * p.a.k_row + at.kv_head * p.a.k_head, p.a.k_row, n, dim);
    TileLoader<T, KS, BN, NT, ASYNC> values((const T *)p.a.v + at.base * p.a.v_row + at.kv_head * p.a.v_head, p.a.v_row, n, dim);
    keys.issue(0, tiles);
    values.issue(0, tiles + BN * S::W);
    Frag<T> qf[KS], of[KS];
    const long long o_at = ((at.base + qc) * p.a.heads + at.head) * dim;
    const T *q_row = (const T *)p.a.q + (at.base + qc) * p.a.q_row + at.head * p.a.q_head;
    const T *do_row = (const T *)p.a.d_out + (at.base + qc) * p.a.do_row + at.head * p.a.do_head;
    // fp32: delta by the instructions that give d_out . v, as the diagonal of a product, so that a row that one pair
    // takes nearly whole has the difference of two equal sums
    float delta = 0.f;
    f32x16 deltas = f32x16{};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        qf[ks] = load_global<T>(q_row, 16 * ks + 8 * h, dim);
        of[ks] = load_global<T>(do_row, 16 * ks + 8 * h, dim);
        const Frag<T> o = load_global<T>((const T *)p.a.out + o_at, 16 * ks + 8 * h, dim);
        if constexpr (sizeof(T) == 4) {
            deltas = mma(o, of[ks], deltas);
            continue;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) delta = fmaf((float)of[ks].v[e], (float)o.v[e], delta);
        if (sizeof(T) == 2 && p.a.out_low != nullptr) {
            const Frag<T> low = load_global<T>((const T *)p.a.out_low + o_at, 16 * ks + 8 * h, dim);
#pragma unroll
            for (int e = 0; e < 8; ++e) delta = fmaf((float)of[ks].v[e], (float)low.v[e], delta);
        }
    }
    if (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 16; ++i) delta = reg_row(i, h) == (lane & 31) ? deltas[i] : delta;
    }
    delta += __shfl_xor(delta, 32, 64);
    const long long row_at = at.head * p.a.rows + at.base + qc;
    if (q < n && h == 0) p.a.delta[row_at] = delta;
    const Codes code_tiles(BIAS ? p.a.codes + p.a.code_start[at.seg] : nullptr, at.first, n);
    if (BIAS) code_tiles.issue(0, codes);
    const float scale = p.a.scale * kLog2e, c = BIAS ? 1.f : scale;
    const RowWeight<T, BIAS> weight(p.a.stats[2 * row_at], p.a.stats[2 * row_at + 1], c);

    Result<T, KS> acc;
    acc.clear();
    GradientScale<T> scaled;
    const int end = causal && at.first + 32 * NW < n ? at.first + 32 * NW : n;
    keys.commit(tiles);
    values.commit(tiles + BN * S::W);
    loads_done();
    for (int k0 = 0, turn = 0; k0 < end; k0 += BN, turn ^= 1) {
        const T *k_tile = tiles + 2 * turn * BN * S::W, *v_tile = k_tile + BN * S::W;
        T *next = tiles + 2 * (turn ^ 1) * BN * S::W;
        tile_ready<ASYNC || BIAS>();
        if (k0 + BN < end) {
            keys.issue(k0 + BN, next);
            values.issue(k0 + BN, next + BN * S::W);
            if (BIAS) code_tiles.issue(k0 + BN, codes + (turn ^ 1) * 32 * NW * BN);
        }
#pragma unroll
        for (int t = 0; t < TN; ++t) {
            const int kt = k0 + 32 * t;
            if (q0 >= n || kt >= n || (causal && kt > q0 + 31)) break;
            // the products begin at the row's reference and, 16-bit types, at minus its delta
            f32x16 sx, dx;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                sx[i] = weight.begin();
                dx[i] = sizeof(T) == 2 ? -delta : 0.f;
            }
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                sx = mma(row_operand<T, KS>(k_tile, 32 * t + (lane & 31), ks, h), qf[ks], sx);
                dx = mma(row_operand<T, KS>(v_tile, 32 * t + (lane & 31), ks, h), of[ks], dx);
            }
            float s[16], d[16];
            unpack(sx, s);
            unpack(dx, d);
#pragma unroll
            for (int i = 0; i < 16; ++i) d[i] -= sizeof(T) == 2 ? 0.f : delta;
            uint32_t four[4];
            bool alike = false;
            if (BIAS) {
#pragma unroll
                for (int g = 0; g < 4; ++g)
                    four[g] = Codes::read(codes + turn * 32 * NW * BN, q - at.first, 32 * t + 8 * g + 4 * h);
                alike = add_bias(s, four, scale, table, nb);
            }
            if (kt + 32 > n || (causal && kt + 31 > q0)) {
                const int last = causal ? min(q, n - 1) : n - 1;
#pragma unroll
                for (int i = 0; i < 16; ++i) s[i] = kt + reg_row(i, h) <= last ? s[i] : -INFINITY;
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = weigh(weight.weight(s[i], weight.start, weight.factor, c), d[i]);
            if (BIAS && q < n) {
                if (alike) {
                    buckets.add_all(four[0], s);
                } else {
#pragma unroll
                    for (int g = 0; g < 4; ++g) buckets.add(four[g], s + 4 * g);
                }
            }
            scaled.apply(s, acc);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const Frag<T> f = pack<T>(s, u);
                // narrow heads: keys that a row weighs lie in its query's direction, and what they have in common drops
                // out of the gradient (ds adds up to 0) but not out of its roundings
                if constexpr (sizeof(T) == 2 && KS <= 2) acc.add(k_tile, 32 * t + 16 * u, f, left_over<T>(s, f, u), lane);
                else acc.add(k_tile, 32 * t + 16 * u, f, lane);
            }
        }
        keys.commit(next);
        values.commit(next + BN * S::W);
    }
    acc.finish();
    bool again = q < n && not_finite<KS>(acc.a);
    if (any_lane(again) && !masked_may_spoil<T, BIAS>(p, at, keys.base, p.a.k_row, q0, end)) again = false;
    scaled.undo(acc, 0);
    // A row's only pair has weight 1 whatever its score: no gradient, where d_out . v and delta, summed in different
    // orders, differ by a rounding.  (Times 0: what is not a number stays.)
    const float some = n == 1 || (causal && q == 0) ? 0.f : 1.f;
    if (q < n && !again) store_rows<false, T, DT>((T *)p.a.dq + o_at, dim, h, acc.a, p.a.scale * some);
    if (any_lane(again)) again_dq<T, BIAS>(p, at, table, q, end, weight, delta, c, scaled.by, p.a.scale * some, again);
    if (BIAS) {
        if (some == 0.f) buckets.times_zero();
        __syncthreads();
        for (int b = threadIdx.x >> 6; b < nb; b += NW) {                  // a wavefront per bucket
            const float v = rwk_wave_sum(buckets.part(b));
            if (lane == 0) p.a.d_table_partials[((long long)at.head * nb + b) * p.a.n_items + at.item] = v;
        }
    }
}

// dK and dV of 32 keys per wavefront.  Two wavefronts per SIMD hide each other's exponentials and LDS reads, which
// leaves 256 registers each: at 128 elements of 16 bits the sums take 128 and the keys 32 of them, and the values stay
// in LDS.  fp32 of up to 16 elements needs half of that, and four hide more (1024 protein-sized graphs: 789 us; by
// three 5 % more).
template <typename T, int KS> constexpr bool values_in_lds() { return sizeof(T) == 2 && KS == 8; }
template <typename T, int KS, int NW> constexpr int dkv_rows() {
    return values_in_lds<T, KS>() ? 32 : tile_rows<T, NW>();
}
template <typename T, int KS, int NW, bool BIAS> constexpr int dkv_lds() {
    return tiles_bytes<T, KS, dkv_rows<T, KS, NW>()>() + (BIAS || sizeof(T) == 4 ? 6 : 4) * dkv_rows<T, KS, NW>() * (int)sizeof(float) +
           (BIAS ? code_bytes<NW, dkv_rows<T, KS, NW>()>() : 0) +
           (values_in_lds<T, KS>() ? tile_bytes<T, KS, 32 * NW>() : 0);
}

template <typename T, int KS, int NW, bool BIAS, bool ASYNC>
__global__ void __launch_bounds__(64 * NW, KS == 8 && (sizeof(T) == 4 || BIAS || !ASYNC) ? 1 : sizeof(T) == 4 && KS == 1 ? 4 : 2)
attention_dkv_kernel(const RwkAttnArgs p) {
    using S = Shape<T, KS>;
    constexpr int NT = 64 * NW, DT = S::DT, BQ = dkv_rows<T, KS, NW>(), TQ = BQ / 32;
    constexpr bool VL = values_in_lds<T, KS>();
    extern __shared__ __attribute__((aligned(16))) char attn_lds[];
    T *tiles = (T *)attn_lds;                                       // buffer b: q at 2 b, d_out at 2 b + 1
    typedef RowWeight<T, BIAS> Weight;
    constexpr int NS = Weight::FOLDED ? 2 : 3;                      // per buffer and row: start, - delta, factor
    float *stats = (float *)(attn_lds + tiles_bytes<T, KS, BQ>());
    uint8_t *codes = (uint8_t *)(stats + 2 * NS * BQ);
    typedef CodeLoader<32 * NW, BQ, NT> Codes;
    T *v_tile = (T *)(codes + (BIAS ? 2 * 32 * NW * BQ : 0));
    int part;
    const Place at = key_place(p, blockIdx.x, &part);
    const int lane = threadIdx.x & 63, h = lane >> 5, dim = (int)p.a.dim, n = at.n;
    const int wave = (int)(threadIdx.x >> 6), k0 = at.first + 32 * wave, k = k0 + (lane & 31), kc = min(k, n - 1);
    const bool causal = p.a.causal != 0;
    const int nb = (int)p.a.n_buckets;

    Frag<T> kf[KS], vf[VL ? 1 : KS];
    const T *k_row = (const T *)p.a.k + (at.base + kc) * p.a.k_row + at.kv_head * p.a.k_head;
    const T *v_base = (const T *)p.a.v + at.base * p.a.v_row + at.kv_head * p.a.v_head;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        kf[ks] = load_global<T>(k_row, 16 * ks + 8 * h, dim);
        if constexpr (!VL) vf[ks] = load_global<T>(v_base + kc * p.a.v_row, 16 * ks + 8 * h, dim);
    }
    if constexpr (VL) {
        TileLoader<T, KS, 32 * NW, NT, ASYNC> values(v_base, p.a.v_row, n, dim);
        values.issue(at.first, v_tile);
        values.commit(v_tile);                    // there with the first tile of queries
    }
    const T *v_own = v_tile + 32 * wave * S::W;   // the swizzle repeats: offsets as in the other tiles
    const Codes code_tiles(BIAS ? p.a.codes_by_key + p.a.code_start[at.seg] : nullptr, at.first, n);
    const float scale = p.a.scale * kLog2e, c = BIAS ? 1.f : scale;

    Result<T, KS> dk, dv;
    dk.clear();
    dv.clear();
    GradientScale<T> scaled;
    const int begin = causal ? at.first : 0;
    for (int g = 0; g < p.part_heads; ++g) {
        const int head = at.head + g;
        const long long row_at = head * p.a.rows + at.base;
        TileLoader<T, KS, BQ, NT, ASYNC> queries((const T *)p.a.q + at.base * p.a.q_row + head * p.a.q_head, p.a.q_row, n, dim);
        TileLoader<T, KS, BQ, NT, ASYNC> grads((const T *)p.a.d_out + at.base * p.a.do_row + head * p.a.do_head, p.a.do_row, n, dim);
        const float table = BIAS ? load_table<T>(p, head) : 0.f;
        __syncthreads();                          // the head before is done with the buffers
        float held[NS];
        const auto start = [&](int q0, int turn) {
            queries.issue(q0, tiles + 2 * turn * BQ * S::W);
            grads.issue(q0, tiles + (2 * turn + 1) * BQ * S::W);
            if (BIAS) code_tiles.issue(q0, codes + turn * 32 * NW * BQ);
            const int q = q0 + (int)threadIdx.x;
            if (threadIdx.x < BQ) {
                const bool there = q < n;
                const Weight w(there ? p.a.stats[2 * (row_at + q)] : 0.f,
                               there ? p.a.stats[2 * (row_at + q) + 1] : 0.f, c, kWeightUp<T>);
                held[0] = w.start;
                held[1] = there ? -p.a.delta[row_at + q] : 0.f;
                if (!Weight::FOLDED) held[NS - 1] = w.factor;
            }
        };
        const auto finish = [&](int turn) {
            queries.commit(tiles + 2 * turn * BQ * S::W);
            grads.commit(tiles + (2 * turn + 1) * BQ * S::W);
            if (threadIdx.x < BQ) {
#pragma unroll
                for (int j = 0; j < NS; ++j) stats[(NS * turn + j) * BQ + threadIdx.x] = held[j];
            }
        };
        start(begin, 0);
        finish(0);
        loads_done();
        for (int q0 = begin, turn = 0; q0 < n; q0 += BQ, turn ^= 1) {
            tile_ready<ASYNC || BIAS>();
            if (q0 + BQ < n) start(q0 + BQ, turn ^ 1);
            const T *q_tile = tiles + 2 * turn * BQ * S::W, *o_tile = q_tile + BQ * S::W;
            const float *st = stats + NS * turn * BQ;
#pragma unroll
            for (int t = 0; t < TQ; ++t) {
                const int qt = q0 + 32 * t;
                if (k0 >= n || qt >= n) break;
                if (causal && qt + 31 < k0) continue;
                typedef float f32x4 __attribute__((ext_vector_type(4)));
                f32x16 sx, dx;
#pragma unroll
                for (int g4 = 0; g4 < 4; ++g4) {
                    const int r = 32 * t + 8 * g4 + 4 * h;
                    const f32x4 begins = *(const f32x4 *)(st + r), d = *(const f32x4 *)(st + BQ + r);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        sx[4 * g4 + e] = Weight::FOLDED ? begins[e] : 0.f;
                        dx[4 * g4 + e] = sizeof(T) == 2 ? d[e] : 0.f;
                    }
                }
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    sx = mma(row_operand<T, KS>(q_tile, 32 * t + (lane & 31), ks, h), kf[ks], sx);
                    const Frag<T> o = row_operand<T, KS>(o_tile, 32 * t + (lane & 31), ks, h);
                    if constexpr (VL) dx = mma(o, row_operand<T, KS>(v_own, lane & 31, ks, h), dx);
                    else dx = mma(o, vf[ks], dx);
                }
                float s[16], d[16];
                unpack(sx, s);
                unpack(dx, d);
                if (BIAS) {
                    uint32_t four[4];
#pragma unroll
                    for (int g4 = 0; g4 < 4; ++g4)
                        four[g4] = Codes::read(codes + turn * 32 * NW * BQ, k - at.first, 32 * t + 8 * g4 + 4 * h);
                    add_bias(s, four, scale, table, nb);
                }
                if (causal && qt < k0 + 31) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[i] = qt + reg_row(i, h) >= k ? s[i] : -INFINITY;
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int r = 32 * t + reg_row(i, h);
                    if (sizeof(T) == 4) d[i] += st[BQ + r];
                    s[i] = Weight::FOLDED ? Weight::weight(s[i], 0.f, 1.f, c) : Weight::weight(s[i], st[r], st[2 * BQ + r], c);
                    d[i] = weigh(s[i], d[i]);
                }
                scaled.apply(d, dk);
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    dv.add(o_tile, 32 * t + 16 * u, pack<T>(s, u), lane);
                    dk.add(q_tile, 32 * t + 16 * u, pack<T>(d, u), lane);
                }
            }
            if (q0 + BQ < n) finish(turn ^ 1);
        }
    }
    const KeyGradients out(p, at, part);
    const long long to = kc * p.a.kv_heads * dim;
    dk.finish();
    dv.finish();
    const bool bad_k = not_finite<KS>(dk.a), bad_v = not_finite<KS>(dv.a);
    bool again = k < n && (bad_k || bad_v);
    if (any_lane(again) && !masked_may_spoil_keys<T, BIAS>(p, at, k0, begin)) again = false;
    const float by = n == 1 ? 0.f * p.a.scale : p.a.scale;        // as in dQ: a segment of one row has one pair
    constexpr float dv_by = 1.f / (1 << kWeightUp<T>);
    scaled.undo(dk, kWeightUp<T>);
    if (k < n && !again && p.parts > 1) {
        store_rows<false, float, DT>(out.dk + to, dim, h, dk.a, by);
        store_rows<false, float, DT>(out.dv + to, dim, h, dv.a, dv_by);
    } else if (k < n && !again) {
        store_rows<false, T, DT>((T *)p.a.dk + out.at + to, dim, h, dk.a, by);
        store_rows<false, T, DT>((T *)p.a.dv + out.at + to, dim, h, dv.a, dv_by);
    }
    if (any_lane(again)) again_dkv<T, BIAS>(p, at, part, k, begin, c, scaled.by, by, again);
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

template <typename T, int KS, bool WIDE, bool BIAS, bool ASYNC>
int launch_shape(RwkAttnPass pass, const RwkAttnArgs &p, hipStream_t stream) {
    constexpr int NW = WIDE ? 4 : 1, NT = 64 * NW, ROWS = tile_rows<T, NW>();
    constexpr int LDS = tiles_bytes<T, KS, ROWS>() + (BIAS ? code_bytes<NW, ROWS>() : 0);
    if (pass == kRwkAttnForward) {
        constexpr bool NARROW = sizeof(T) == 2 && KS <= 2;
        if (sizeof(T) == 2 && p.a.few_keys)
            return launch_kernel(attention_forward_kernel<T, KS, NW, BIAS, sizeof(T) == 2, ASYNC>, p.a.n_items * p.a.heads,
                                 NT, LDS, p, stream);
        return launch_kernel(attention_forward_kernel<T, KS, NW, BIAS, NARROW, ASYNC>, p.a.n_items * p.a.heads, NT, LDS,
                             p, stream);
    }
    if (pass == kRwkAttnDq) {
        const int nb = (int)p.a.n_buckets, split = LDS + 4 * (nb + 1) * NT * (int)sizeof(float);
        // four sets of bucket sums where three workgroups still share a compute unit's 160 KB
        if (BIAS && split <= 160 * 1024 / 3)
            return launch_kernel(attention_dq_kernel<T, KS, NW, BIAS, BIAS, ASYNC>, p.a.n_items * p.a.heads, NT, split, p, stream);
        return launch_kernel(attention_dq_kernel<T, KS, NW, BIAS, false, ASYNC>, p.a.n_items * p.a.heads, NT,
                             LDS + nb * NT * (int)sizeof(float), p, stream);
    }
    return launch_kernel(attention_dkv_kernel<T, KS, NW, BIAS, ASYNC>, p.a.n_items * p.a.kv_heads * p.parts, NT,
                         dkv_lds<T, KS, NW, BIAS>(), p, stream);
}

// Rows whose elements are whole 16-byte chunks at 16-byte addresses, not too far apart for 32-bit offsets inside a
// tile, are loaded straight into LDS.
template <typename T>
bool chunked(const RwkAttnArgs &p, bool backward) {
    const long long e = 16 / (long long)sizeof(T), far = 0x7FFFFFFFll / (128 * (long long)sizeof(T)) - 1;
    const auto fits = [&](const void *at, long long row, long long head) {
        return (uintptr_t)at % 16 == 0 && row % e == 0 && head % e == 0 && row >= 0 && row < far;
    };
    return p.a.dim % e == 0 && fits(p.a.q, p.a.q_row, p.a.q_head) && fits(p.a.k, p.a.k_row, p.a.k_head) &&
           fits(p.a.v, p.a.v_row, p.a.v_head) && (!backward || fits(p.a.d_out, p.a.do_row, p.a.do_head));
}

template <typename T, int KS>
int launch_width(RwkAttnPass pass, const RwkAttnArgs &p, hipStream_t stream) {
    const bool bias = p.a.n_buckets > 0, wide = p.a.block_rows == 128, async = chunked<T>(p, pass != kRwkAttnForward);
#define RWK_ATTN_CASE(W, B, A) if (wide == W && bias == B && async == A) return launch_shape<T, KS, W, B, A>(pass, p, stream)
    RWK_ATTN_CASE(true, true, true);
    RWK_ATTN_CASE(true, true, false);
    RWK_ATTN_CASE(true, false, true);
    RWK_ATTN_CASE(true, false, false);
    RWK_ATTN_CASE(false, true, true);
    RWK_ATTN_CASE(false, true, false);
    RWK_ATTN_CASE(false, false, true);
    RWK_ATTN_CASE(false, false, false);
#undef RWK_ATTN_CASE
    return RWK_E_UNSUPPORTED;
}

template <typename T>
int launch_type(RwkAttnPass pass, const RwkAttnArgs &p, hipStream_t stream) {
    if (p.a.dim <= 16) return launch_width<T, 1>(pass, p, stream);
    if (p.a.dim <= 32) return launch_width<T, 2>(pass, p, stream);
    if (p.a.dim <= 64) return launch_width<T, 4>(pass, p, stream);
    return launch_width<T, 8>(pass, p, stream);
}

}  // namespace
