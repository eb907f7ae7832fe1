// AdamW (decoupled weight decay) over many tensors in one launch, with the moment estimates in 32 or in 8 bits:
//
//   m = beta1 m + (1 - beta1) g,   v = beta2 v + (1 - beta2) g^2
//   p = p (1 - lr wd) - lr / (1 - beta1^t) * m / (sqrt(v) / sqrt(1 - beta2^t) + eps)
//
// Bound by memory: per element p, m, v in and out and g in (28 bytes for fp32 with 32-bit states, 16 with 8-bit
// states, 10 for 16-bit weights with 8-bit states).  The tensors are cut into chunks, one workgroup
// each; a table on the device describes them, the gradients' addresses - the only ones that change from step to step -
// travel in the launch's arguments, so a step copies nothing to the device.
// Every chunk counts its own steps (a tensor without a gradient is skipped and does not age), so a captured launch
// replays correctly.
//
// 8-bit states: blocks of 256 consecutive elements of a tensor share an fp32 scale s = max |x| * (1 / 448), an element is
// the float8 (e4m3) value next to x / s.  v moves by a thousandth per step while neighbouring float8 values are an
// eighth apart: rounding to nearest would freeze it.  So x / s is rounded up or down at random in proportion to the
// distances (16 bits of Philox4x32 per value, counter = {element / 4, tensor, step, 0}), which leaves every moment's
// expectation where fp32 would have it.  A positive v never becomes zero (the step would divide by eps alone).  The
// update itself uses m and v before they are rounded.  One wavefront holds one block, four elements a lane.
#include "rwk_vec.h"

// every product and sum below is rounded by itself unless fmaf is written: the states are the same numbers however
// the compiler orders its work
#pragma clang fp contract(off)

namespace {

constexpr int kBlock = 256;
constexpr int kStateBlock = 256;                       // elements that share a scale: one wavefront, four per lane
// Blocks per wavefront, loaded together: four where there are chunks enough for every compute unit that way (50 M fp32
// elements with 32-bit states 264 us, 5.3 TB/s), one for few elements, whose time is latency (1.3 M with 8-bit states:
// 11.5 us by four, 8.9 by one).
constexpr int chunk_elements(int per_wave) { return kBlock / RWK_WAVE * per_wave * kStateBlock; }
constexpr int64_t kFewElements = 4 << 20;
constexpr int kTensors = RWK_ADAMW_TENSORS;            // gradient addresses of one launch

struct AdamwGrads {
    const void *grad[kTensors];
};

struct AdamwHyper {
    double beta1, beta2, weight_decay;
    float eps;
    uint32_t seed_lo, seed_hi;
};

__device__ inline double power(double b, long long t) {
    double r = 1.0;
    while (t > 0) {
        if (t & 1) r *= b;
        b *= b;
        t >>= 1;
    }
    return r;
}

// largest bit pattern of a wavefront's non-negative floats: NaN above infinity above all finite values
__device__ inline float wave_max(float v) {
    uint32_t u = __builtin_bit_cast(uint32_t, v);
#define RWK_MAX_STEP(CTRL)                                                            \
    {                                                                                 \
        const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)u, CTRL, 0xF, 0xF, false); \
        u = u > o ? u : o;                                                            \
    }
    RWK_MAX_STEP(0xB1)
    RWK_MAX_STEP(0x4E)
    RWK_MAX_STEP(0x141)
    RWK_MAX_STEP(0x140)
#undef RWK_MAX_STEP
    uint32_t o = (uint32_t)__shfl_xor((int)u, 16, 64);
    u = u > o ? u : o;
    o = (uint32_t)__shfl_xor((int)u, 32, 64);
    u = u > o ? u : o;
    return __builtin_bit_cast(float, u);
}

constexpr float kF8Max = 448.f;

// scale and its inverse of a block whose largest magnitude is `top`; a block of zeros (or of magnitudes whose scale
// is not a normal number) has scale 0, and all its values are 0
__device__ inline float block_scale(float top, float *inverse) {
    float s = top * (1.f / kF8Max);
    if (s < 1.17549435e-38f) s = 0.f;
    *inverse = s == 0.f ? 0.f : 1.f / s;
    return s;
}

// float8 code of |x| * inverse rounded by the 16 random bits `r`.  The code is the float's upper bits less the
// difference of the exponent biases, so that adding r below them and dropping the rest rounds at random; below the
// smallest normal value (2^-6) the codes are multiples of 2^-9.
__device__ inline uint32_t f8_code(float x, float inverse, uint32_t r) {
    const float y = fminf(fabsf(x) * inverse, kF8Max);
    const uint32_t add = r << 4;
    const uint32_t normal = ((__builtin_bit_cast(uint32_t, y) + add) >> 20) - (120u << 3);
    const uint32_t small = ((uint32_t)(y * 536870912.f) + add) >> 20;            // y * 2^9 in units of 2^-20
    return (y >= 0.015625f ? normal : small) & 0x7Fu;
}

__device__ inline void f8_decode(uint32_t codes, float scale, float (&out)[4]) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    const f2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, true);
    out[0] = lo[0] * scale;
    out[1] = lo[1] * scale;
    out[2] = hi[0] * scale;
    out[3] = hi[1] * scale;
}

// m / (sqrt(v) inv_root + eps) with the one-instruction root and reciprocal, good to an ulp each, on an update that is
// a small part of the parameter; a root below 2^-63 that the instruction takes for zero counts for nothing beside eps.
// Where eps says nothing, by the exact operations.
constexpr float kPlainEps = 1e-12f;
template <bool PLAIN>
__device__ inline float ratio(float m, float v, float inv_root, float eps) {
    if (!PLAIN && eps < kPlainEps) return m / fmaf(sqrtf(v), inv_root, eps);
    return m * __builtin_amdgcn_rcpf(fmaf(__builtin_amdgcn_sqrtf(v), inv_root, eps));
}

// FULL: all of the chunk's elements exist (and eps is not tiny: ratio())
template <typename T, bool STATE8, int kPerWave, bool FULL>
__device__ inline void update(RwkGlobal<T> param, RwkGlobal<T> grad, const rwk_adamw_chunk &t, long long step, const double *__restrict__ lr_ptr, const AdamwHyper &hyper) {
    const long long n = t.n, start = t.start;
    // 32-bit states; 8-bit states by the bytes, and their scales
    const RwkGlobal<float> avg = rwk_global<float>(t.exp_avg), avg_sq = rwk_global<float>(t.exp_avg_sq);
    const RwkGlobal<uint8_t> avg8 = rwk_global<uint8_t>(t.exp_avg), avg_sq8 = rwk_global<uint8_t>(t.exp_avg_sq);
    const RwkGlobal<float> scale = rwk_global<float>(t.exp_avg_scale), scale_sq = rwk_global<float>(t.exp_avg_sq_scale);
    const int lane = threadIdx.x & (RWK_WAVE - 1), wave = threadIdx.x / RWK_WAVE;

    float p[kPerWave][4], g[kPerWave][4], m[kPerWave][4], v[kPerWave][4];
    const long long first = start + (long long)wave * kPerWave * kStateBlock + 4 * lane;
#pragma unroll
    for (int k = 0; k < kPerWave; ++k) {
        const long long i = first + (long long)k * kStateBlock;
#pragma unroll
        for (int j = 0; j < 4; ++j) p[k][j] = g[k][j] = m[k][j] = v[k][j] = 0.f;
        if (FULL || i + 4 <= n) {
            const auto pv = rwk_load<T, 4>(param + i);
            const auto gv = rwk_load<T, 4>(grad + i);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                p[k][j] = (float)pv[j];
                g[k][j] = (float)gv[j];
            }
            if (!STATE8) {
                const auto mv = rwk_load<float, 4>(avg + i);
                const auto vv = rwk_load<float, 4>(avg_sq + i);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    m[k][j] = mv[j];
                    v[k][j] = vv[j];
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (i + j < n) {
                    p[k][j] = (float)param[i + j];
                    g[k][j] = (float)grad[i + j];
                    if (!STATE8) {
                        m[k][j] = avg[i + j];
                        v[k][j] = avg_sq[i + j];
                    }
                }
        }
        // the 8-bit states are padded to whole blocks: every lane of a block that begins inside the tensor reads them
        if (STATE8 && (FULL || i - 4 * lane < n)) {
            const long long b = (i - 4 * lane) / kStateBlock;
            f8_decode(*(RwkGlobal<uint32_t>)(avg8 + i), scale[b], m[k]);
            f8_decode(*(RwkGlobal<uint32_t>)(avg_sq8 + i), scale_sq[b], v[k]);
        }
    }

    const double lr = lr_ptr[0];
    const float beta1 = (float)hyper.beta1, beta2 = (float)hyper.beta2;
    const float rest1 = (float)(1.0 - hyper.beta1), rest2 = (float)(1.0 - hyper.beta2);
    const float decay = (float)(1.0 - lr * hyper.weight_decay);
    const float size = (float)(lr / (1.0 - power(hyper.beta1, step)));
    const float inv_root = (float)(1.0 / sqrt(1.0 - power(hyper.beta2, step)));

#pragma unroll
    for (int k = 0; k < kPerWave; ++k) {
        const long long i = first + (long long)k * kStateBlock;
        float top_m = 0.f, top_v = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            m[k][j] = m[k][j] * beta1 + g[k][j] * rest1;
            v[k][j] = v[k][j] * beta2 + g[k][j] * rest2 * g[k][j];
            p[k][j] = fmaf(-size, ratio<FULL>(m[k][j], v[k][j], inv_root, hyper.eps), p[k][j] * decay);
            if (STATE8) {
                const float am = fabsf(m[k][j]), av = fabsf(v[k][j]);
                // as integers: NaN is the largest
                top_m = __builtin_bit_cast(uint32_t, am) > __builtin_bit_cast(uint32_t, top_m) ? am : top_m;
                top_v = __builtin_bit_cast(uint32_t, av) > __builtin_bit_cast(uint32_t, top_v) ? av : top_v;
            }
        }
        if (FULL || i + 4 <= n) {
            typename RwkPack<T, 4>::type pv;
#pragma unroll
            for (int j = 0; j < 4; ++j) pv[j] = (T)p[k][j];
            rwk_store<T, 4>(param + i, pv);
            if (!STATE8) {
                typename RwkPack<float, 4>::type mv, vv;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    mv[j] = m[k][j];
                    vv[j] = v[k][j];
                }
                rwk_store<float, 4>(avg + i, mv);
                rwk_store<float, 4>(avg_sq + i, vv);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (i + j < n) {
                    param[i + j] = (T)p[k][j];
                    if (!STATE8) {
                        avg[i + j] = m[k][j];
                        avg_sq[i + j] = v[k][j];
                    }
                }
        }
        if (STATE8) {
            const long long begin = i - 4 * lane;
            if (!FULL && begin >= n) continue;                       // the same for the whole wavefront
            float inv_m, inv_v;
            const float scale_m = block_scale(wave_max(top_m), &inv_m), scale_v = block_scale(wave_max(top_v), &inv_v);
            const RwkPhilox4 r = rwk_philox4x32<7>((uint32_t)(i >> 2), t.stream,
                                                   (uint32_t)step, 0u, hyper.seed_lo, hyper.seed_hi);
            const uint32_t bits[4] = {r.x, r.y, r.z, r.w};
            uint32_t cm = 0, cv = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                uint32_t a = f8_code(m[k][j], inv_m, bits[j] & 0xFFFFu);
                uint32_t b = f8_code(v[k][j], inv_v, bits[j] >> 16);
                a |= (__builtin_bit_cast(uint32_t, m[k][j]) >> 31) << 7;
                if (b == 0 && v[k][j] > 0.f) b = 1;
                cm |= a << (8 * j);
                cv |= b << (8 * j);
            }
            *(RwkGlobal<uint32_t>)(avg8 + i) = cm;
            *(RwkGlobal<uint32_t>)(avg_sq8 + i) = cv;
            if (lane == 0) {
                scale[begin / kStateBlock] = scale_m;
                scale_sq[begin / kStateBlock] = scale_v;
            }
        }
    }
}

template <typename T, bool STATE8, int kPerWave>
__global__ void __launch_bounds__(kBlock)
adamw_kernel(const rwk_adamw_chunk *__restrict__ chunks, int tensor_base, AdamwGrads grads,
             const double *__restrict__ lr_ptr, AdamwHyper hyper, long long *__restrict__ chunk_steps) {
    const rwk_adamw_chunk chunk = chunks[blockIdx.x];
    const long long step = chunk_steps[blockIdx.x] + 1;
    const void *grad = grads.grad[chunk.tensor - tensor_base];
    if (grad == nullptr) return;
    const RwkGlobal<T> p = rwk_global<T>(chunk.param), g = rwk_global<T>((void *)grad);
    if (chunk.start + chunk_elements(kPerWave) <= chunk.n && hyper.eps >= kPlainEps)
        update<T, STATE8, kPerWave, true>(p, g, chunk, step, lr_ptr, hyper);
    else
        update<T, STATE8, kPerWave, false>(p, g, chunk, step, lr_ptr, hyper);
    __syncthreads();                              // every wavefront has read the count
    if (threadIdx.x == 0) chunk_steps[blockIdx.x] = step;
}

struct AdamwLaunch {
    const rwk_adamw_chunk *chunks;
    unsigned n_chunks;
    int tensor_base;
    AdamwGrads grads;
    const double *lr;
    AdamwHyper hyper;
    long long *steps;
    hipStream_t stream;
};

template <typename T, bool STATE8, int PER>
int launch(const AdamwLaunch &a) {
    hipLaunchKernelGGL((adamw_kernel<T, STATE8, PER>), dim3(a.n_chunks), dim3(kBlock), 0, a.stream, a.chunks,
                       a.tensor_base, a.grads, a.lr, a.hyper, a.steps);
    RWK_LAUNCH_CHECK();
    return RWK_OK;
}

template <typename T>
int launch_type(const AdamwLaunch &a, int state_bits, int64_t chunk_size) {
    if (chunk_size == chunk_elements(1)) return state_bits == 8 ? launch<T, true, 1>(a) : launch<T, false, 1>(a);
    return state_bits == 8 ? launch<T, true, 4>(a) : launch<T, false, 4>(a);
}

}  // namespace

extern "C" {

int64_t rwk_adamw_chunk_size(int64_t n) { return n < kFewElements ? chunk_elements(1) : chunk_elements(4); }

int rwk_adamw_step(const rwk_adamw_chunk *chunks, int64_t n_chunks, int64_t chunk_size, int64_t tensor_base,
                   const void *const *grads, int64_t n_grads, int32_t type, int32_t state_bits, const double *lr,
                   double beta1, double beta2, double eps, double weight_decay, uint64_t seed, int64_t *chunk_steps,
                   rwk_stream_t stream) {
    RWK_REQUIRE_PTR(chunks);
    RWK_REQUIRE_PTR(grads);
    RWK_REQUIRE_PTR(lr);
    RWK_REQUIRE_PTR(chunk_steps);
    if (n_chunks <= 0 || n_chunks > 0x7FFFFFFFll || tensor_base < 0 || tensor_base > 0x7FFFFFFFll || n_grads <= 0)
        return RWK_E_SIZE;
    if (n_grads > kTensors || type < RWK_F32 || type > RWK_BF16 || (state_bits != 8 && state_bits != 32) ||
        (chunk_size != chunk_elements(1) && chunk_size != chunk_elements(4)))
        return RWK_E_UNSUPPORTED;
    AdamwLaunch a;
    a.chunks = chunks;
    a.n_chunks = (unsigned)n_chunks;
    a.tensor_base = (int)tensor_base;
    for (int i = 0; i < kTensors; ++i) a.grads.grad[i] = i < n_grads ? grads[i] : nullptr;
    a.lr = lr;
    a.hyper = AdamwHyper{beta1, beta2, weight_decay, (float)eps, (uint32_t)seed, (uint32_t)(seed >> 32)};
    a.steps = (long long *)chunk_steps;
    a.stream = (hipStream_t)stream;
    if (type == RWK_F32) return launch_type<float>(a, state_bits, chunk_size);
    if (type == RWK_F16) return launch_type<rwk_f16>(a, state_bits, chunk_size);
    return launch_type<rwk_bf16>(a, state_bits, chunk_size);
}

}  // extern "C"
