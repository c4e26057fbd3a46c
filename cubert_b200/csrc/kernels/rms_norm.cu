// K6: residual addition and root-mean-square norm, with the output in the storage type or in 8 bits.
//
//   t = x (+ residual);  y = t / sqrt(mean(t^2) + eps) * gamma
//
// t leaves in the storage type (the next residual); y leaves in the storage type, or as e4m3 codes with one
// float32 scale = max|y| / 448 per row or per 128 columns. Arithmetic is float32: y is computed from the
// unrounded t, so t and y are each rounded once, on their way out.
#include "common.cuh"

namespace cubk {

constexpr float kE4m3Max = 448.f;
// A group whose largest |y| is below this is stored as zeros with scale 0: 448 / max|y| must stay finite.
constexpr float kTinyGroup = 7.888609e-31f;   // 2^-100

// The larger of two values; NaN if either is (a row that holds a NaN must not come out as zeros).
__device__ __forceinline__ float max_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}

// Two float32 values to e4m3, round to nearest even, beyond +-448 to +-448; `lo` in the low byte.
__device__ __forceinline__ uint16_t e4m3_pair(float lo, float hi) {
    uint16_t d;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(d) : "f"(hi), "f"(lo));
    return d;
}

// Scale of a group and what its values are multiplied by, from its largest magnitude.
__device__ __forceinline__ float2 e4m3_scale(float top) {
    return top < kTinyGroup ? make_float2(0.f, 0.f) : make_float2(top * (1.f / kE4m3Max), kE4m3Max / top);
}

constexpr int kRmsGenericBlock = 256;

// Any row length and alignment: a block per row, three passes over it (sum of squares, largest magnitude of
// each group, output); x and residual are read again from L2 in each.
template <typename T, bool E4M3>
__global__ void __launch_bounds__(kRmsGenericBlock)
rms_norm_generic_kernel(const T *x, const T *residual, const T *gamma, int64_t rows, int channels, float eps, int group,
                        T *sum, T *out, uint8_t *codes, float *scales) {
    __shared__ float red[kRmsGenericBlock / 32];
    const int groups = (channels + group - 1) / group;
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const T *xr = x + row * channels;
        const T *rr = residual != nullptr ? residual + row * channels : nullptr;
        auto term = [&](int c) { return to_float<T>(xr[c]) + (rr != nullptr ? to_float<T>(rr[c]) : 0.f); };
        float ss = 0.f;
        for (int c = threadIdx.x; c < channels; c += kRmsGenericBlock) {
            const float t = term(c);
            ss = fmaf(t, t, ss);
        }
        ss = block_sum<kRmsGenericBlock / 32>(ss, red);
        const float rstd = 1.f / sqrtf(ss / (float) channels + eps);
        for (int g = 0; g < groups; ++g) {
            const int c0 = g * group, c1 = min(channels, c0 + group);
            float2 sc = make_float2(1.f, 1.f);
            if (E4M3) {
                float top = 0.f;
                for (int c = c0 + threadIdx.x; c < c1; c += kRmsGenericBlock) {
                    top = max_nan(top, fabsf(term(c) * rstd * to_float<T>(gamma[c])));
                }
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) {
                    top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
                }
                __syncthreads();
                if ((threadIdx.x & 31) == 0) {
                    red[threadIdx.x >> 5] = top;
                }
                __syncthreads();
#pragma unroll
                for (int w = 0; w < kRmsGenericBlock / 32; ++w) {
                    top = max_nan(top, red[w]);
                }
                sc = e4m3_scale(top);
                if (threadIdx.x == 0) {
                    scales[row * groups + g] = sc.x;
                }
            }
            for (int c = c0 + threadIdx.x; c < c1; c += kRmsGenericBlock) {
                const float t = term(c);
                const float y = t * rstd * to_float<T>(gamma[c]);
                if (sum != nullptr) {
                    sum[row * channels + c] = from_float<T>(t);
                }
                if (E4M3) {
                    codes[row * channels + c] = (uint8_t) e4m3_pair(y * sc.y, 0.f);
                } else {
                    out[row * channels + c] = from_float<T>(y);
                }
            }
        }
    }
}

template <typename T, bool E4M3>
int residual_rms_norm(const T *x, const T *residual, const T *gamma, int64_t rows, int channels, float eps, int group, T *sum,
                      T *out, uint8_t *codes, float *scales, cudaStream_t stream) {
    if (x == nullptr || gamma == nullptr || rows < 0 || channels <= 0 || !(eps >= 0.f) || (E4M3 ? codes == nullptr || scales == nullptr : out == nullptr) ||
        (E4M3 && group != 0 && group != 128)) {
        return CUBK_ERR_INVALID_ARG;
    }
    if (rows == 0) {
        return CUBK_OK;
    }
    const unsigned blocks = (unsigned) (rows < 148 * 8 ? rows : 148 * 8);
    rms_norm_generic_kernel<T, E4M3><<<blocks, kRmsGenericBlock, 0, stream>>>(x, residual, gamma, rows, channels, eps,
                                                                             E4M3 && group != 0 ? group : channels, sum, out, codes, scales);
    return check_launch();
}

}  // namespace cubk

extern "C" {

int cubk_residual_rms_norm_f32(const float *x, const float *residual, const float *gamma, int64_t rows, int channels, float eps,
                               float *sum, float *out, void *stream) {
    return cubk::residual_rms_norm<float, false>(x, residual, gamma, rows, channels, eps, 0, sum, out, nullptr, nullptr,
                                                 (cudaStream_t) stream);
}

int cubk_residual_rms_norm_f16(const void *x, const void *residual, const void *gamma, int64_t rows, int channels, float eps,
                               void *sum, void *out, void *stream) {
    return cubk::residual_rms_norm<__half, false>((const __half *) x, (const __half *) residual, (const __half *) gamma, rows, channels,
                                                  eps, 0, (__half *) sum, (__half *) out, nullptr, nullptr, (cudaStream_t) stream);
}

int cubk_residual_rms_norm_e4m3_f32(const float *x, const float *residual, const float *gamma, int64_t rows, int channels, float eps,
                                    int group, float *sum, void *codes, float *scales, void *stream) {
    return cubk::residual_rms_norm<float, true>(x, residual, gamma, rows, channels, eps, group, sum, nullptr, (uint8_t *) codes, scales,
                                                (cudaStream_t) stream);
}

int cubk_residual_rms_norm_e4m3_f16(const void *x, const void *residual, const void *gamma, int64_t rows, int channels, float eps,
                                    int group, void *sum, void *codes, float *scales, void *stream) {
    return cubk::residual_rms_norm<__half, true>((const __half *) x, (const __half *) residual, (const __half *) gamma, rows, channels,
                                                 eps, group, (__half *) sum, nullptr, (uint8_t *) codes, scales, (cudaStream_t) stream);
}

}  // extern "C"
