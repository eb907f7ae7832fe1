// AdamW (decoupled weight decay) over many tensors in one launch, with the moment estimates in 32 or in 8 bits:
//
//   m = beta1 m + (1 - beta1) g,   v = beta2 v + (1 - beta2) g^2
//   p = p (1 - lr wd) - lr / (1 - beta1^t) * m / (sqrt(v) / sqrt(1 - beta2^t) + eps)
//
// Bound by memory: per element p, m, v in and out and g in (28 bytes for fp32 with 32-bit states, 16 with 8-bit
// states, 10 for 16-bit weights with 8-bit states).  The tensors are cut into chunks of kChunk elements, one
// workgroup each; a table on the device says which tensor a chunk belongs to, the gradients' addresses - the only
// ones that change from step to step - travel in the launch's arguments, so a step copies nothing to the device.
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
constexpr int kPerWave = 4;                            // blocks per wavefront, loaded together
constexpr int kChunk = kBlock / RWK_WAVE * kPerWave * kStateBlock;
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

template <typename T, bool STATE8>
__global__ void __launch_bounds__(kBlock)
adamw_kernel(const rwk_adamw_tensor *__restrict__ tensors, const rwk_adamw_chunk *__restrict__ chunks, int tensor_base,
             AdamwGrads grads, const double *__restrict__ lr_ptr, AdamwHyper hyper,
             long long *__restrict__ chunk_steps) {
    const rwk_adamw_chunk chunk = chunks[blockIdx.x];
    const T *grad = (const T *)grads.grad[chunk.tensor - tensor_base];
    if (grad == nullptr) return;
    const rwk_adamw_tensor t = tensors[chunk.tensor];
    T *param = (T *)t.param;
    const long long step = chunk_steps[blockIdx.x] + 1;
    const int lane = threadIdx.x & (RWK_WAVE - 1), wave = threadIdx.x / RWK_WAVE;

    float p[kPerWave][4], g[kPerWave][4], m[kPerWave][4], v[kPerWave][4];
    const long long first = chunk.start + (long long)wave * kPerWave * kStateBlock + 4 * lane;
#pragma unroll
    for (int k = 0; k < kPerWave; ++k) {
        const long long i = first + (long long)k * kStateBlock;
#pragma unroll
        for (int j = 0; j < 4; ++j) p[k][j] = g[k][j] = m[k][j] = v[k][j] = 0.f;
        if (i + 4 <= t.n) {
            const auto pv = rwk_load<T, 4>(param + i);
            const auto gv = rwk_load<T, 4>(grad + i);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                p[k][j] = (float)pv[j];
                g[k][j] = (float)gv[j];
            }
            if (!STATE8) {
                const auto mv = rwk_load<float, 4>((const float *)t.exp_avg + i);
                const auto vv = rwk_load<float, 4>((const float *)t.exp_avg_sq + i);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    m[k][j] = mv[j];
                    v[k][j] = vv[j];
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (i + j < t.n) {
                    p[k][j] = (float)param[i + j];
                    g[k][j] = (float)grad[i + j];
                    if (!STATE8) {
                        m[k][j] = ((const float *)t.exp_avg)[i + j];
                        v[k][j] = ((const float *)t.exp_avg_sq)[i + j];
                    }
                }
        }
        // the 8-bit states are padded to whole blocks: every lane of a block that begins inside the tensor reads them
        if (STATE8 && i - 4 * lane < t.n) {
            const long long b = (i - 4 * lane) / kStateBlock;
            f8_decode(*(const uint32_t *)((const uint8_t *)t.exp_avg + i), t.exp_avg_scale[b], m[k]);
            f8_decode(*(const uint32_t *)((const uint8_t *)t.exp_avg_sq + i), t.exp_avg_sq_scale[b], v[k]);
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
            p[k][j] = fmaf(-size, m[k][j] / fmaf(sqrtf(v[k][j]), inv_root, hyper.eps), p[k][j] * decay);
            if (STATE8) {
                const float am = fabsf(m[k][j]), av = fabsf(v[k][j]);
                // as integers: NaN is the largest
                top_m = __builtin_bit_cast(uint32_t, am) > __builtin_bit_cast(uint32_t, top_m) ? am : top_m;
                top_v = __builtin_bit_cast(uint32_t, av) > __builtin_bit_cast(uint32_t, top_v) ? av : top_v;
            }
        }
        if (i + 4 <= t.n) {
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
                rwk_store<float, 4>((float *)t.exp_avg + i, mv);
                rwk_store<float, 4>((float *)t.exp_avg_sq + i, vv);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (i + j < t.n) {
                    param[i + j] = (T)p[k][j];
                    if (!STATE8) {
                        ((float *)t.exp_avg)[i + j] = m[k][j];
                        ((float *)t.exp_avg_sq)[i + j] = v[k][j];
                    }
                }
        }
        if (STATE8) {
            const long long begin = i - 4 * lane;
            if (begin >= t.n) continue;                       // the same for the whole wavefront
            float inv_m, inv_v;
            const float scale_m = block_scale(wave_max(top_m), &inv_m), scale_v = block_scale(wave_max(top_v), &inv_v);
            const RwkPhilox4 r = rwk_philox4x32<7>((uint32_t)(i >> 2), (uint32_t)chunk.tensor + (uint32_t)t.id_offset,
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
            *(uint32_t *)((uint8_t *)t.exp_avg + i) = cm;
            *(uint32_t *)((uint8_t *)t.exp_avg_sq + i) = cv;
            if (lane == 0) {
                t.exp_avg_scale[begin / kStateBlock] = scale_m;
                t.exp_avg_sq_scale[begin / kStateBlock] = scale_v;
            }
        }
    }
    if (threadIdx.x == 0) chunk_steps[blockIdx.x] = step;
}

template <typename T>
int launch(int state_bits, const rwk_adamw_tensor *tensors, const rwk_adamw_chunk *chunks, int64_t n_chunks,
           int tensor_base, const AdamwGrads &grads, const double *lr, const AdamwHyper &hyper, int64_t *steps,
           hipStream_t stream) {
    if (state_bits == 8) {
        hipLaunchKernelGGL((adamw_kernel<T, true>), dim3((unsigned)n_chunks), dim3(kBlock), 0, stream, tensors, chunks,
                           tensor_base, grads, lr, hyper, (long long *)steps);
    } else {
        hipLaunchKernelGGL((adamw_kernel<T, false>), dim3((unsigned)n_chunks), dim3(kBlock), 0, stream, tensors,
                           chunks, tensor_base, grads, lr, hyper, (long long *)steps);
    }
    RWK_LAUNCH_CHECK();
    return RWK_OK;
}

}  // namespace

extern "C" {

int64_t rwk_adamw_chunk_size(void) { return kChunk; }

int rwk_adamw_step(const rwk_adamw_tensor *tensors, const rwk_adamw_chunk *chunks, int64_t n_chunks,
                   int64_t tensor_base, const void *const *grads, int64_t n_grads, int32_t type, int32_t state_bits,
                   const double *lr, double beta1, double beta2, double eps, double weight_decay, uint64_t seed,
                   int64_t *chunk_steps, rwk_stream_t stream_) {
    RWK_REQUIRE_PTR(tensors);
    RWK_REQUIRE_PTR(chunks);
    RWK_REQUIRE_PTR(grads);
    RWK_REQUIRE_PTR(lr);
    RWK_REQUIRE_PTR(chunk_steps);
    if (n_chunks <= 0 || n_chunks > 0x7FFFFFFFll || tensor_base < 0 || tensor_base > 0x7FFFFFFFll || n_grads <= 0)
        return RWK_E_SIZE;
    if (n_grads > kTensors || type < RWK_F32 || type > RWK_BF16 || (state_bits != 8 && state_bits != 32))
        return RWK_E_UNSUPPORTED;
    AdamwGrads g;
    for (int i = 0; i < kTensors; ++i) g.grad[i] = i < n_grads ? grads[i] : nullptr;
    const AdamwHyper h{beta1, beta2, weight_decay, (float)eps, (uint32_t)seed, (uint32_t)(seed >> 32)};
    hipStream_t stream = (hipStream_t)stream_;
    if (type == RWK_F32)
        return launch<float>(state_bits, tensors, chunks, n_chunks, (int)tensor_base, g, lr, h, chunk_steps, stream);
    if (type == RWK_F16)
        return launch<rwk_f16>(state_bits, tensors, chunks, n_chunks, (int)tensor_base, g, lr, h, chunk_steps, stream);
    return launch<rwk_bf16>(state_bits, tensors, chunks, n_chunks, (int)tensor_base, g, lr, h, chunk_steps, stream);
}

}  // extern "C"
