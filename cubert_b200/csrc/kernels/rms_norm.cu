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

enum NormOut { NORM_SAME, NORM_E4M3_ROW, NORM_E4M3_128 };

// Largest magnitude over WIDTH adjacent lanes, NaN if any is.
template <int WIDTH>
__device__ __forceinline__ float group_max_nan(float v) {
#pragma unroll
    for (int o = WIDTH / 2; o > 0; o >>= 1) {
        v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
    }
    return v;
}

// Rows of any length and alignment up to 128 * GROUPS * WARPS elements: in registers too, an element at a time, and so bound by issue
// (8000 x 1001 binary16: 17 us, 73 % of the issue slots). A warp takes groups of
// 128 columns, four elements a lane, so that a group's largest magnitude stays within it. One warp a row (four rows a block) or a block.
template <typename T, int WARPS, int GROUPS, NormOut OUT>
__global__ void __launch_bounds__(WARPS == 1 ? 128 : 32 * WARPS)
rms_norm_elements_kernel(const T *x, const T *residual, const T *gamma, int64_t rows, int channels, float eps, T *sum, T *out, uint8_t *codes,
                         float *scales) {
    constexpr int ROWS = WARPS == 1 ? 4 : 1;   // of a block
    __shared__ float red[2][WARPS];
    const int warp = WARPS == 1 ? 0 : threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int groups = (channels + 127) / 128;
    for (int64_t row = (int64_t) blockIdx.x * ROWS + (WARPS == 1 ? threadIdx.x >> 5 : 0); row < rows; row += (int64_t) gridDim.x * ROWS) {
        const int64_t base = row * channels;
        float t[GROUPS][4], gm[GROUPS][4];
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < GROUPS; ++i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int c = (warp + WARPS * i) * 128 + 32 * j + lane;
                const bool in = c < channels;
                t[i][j] = in ? to_float<T>(x[base + c]) : 0.f;
                gm[i][j] = in ? to_float<T>(gamma[c]) : 0.f;
                if (residual != nullptr) {
                    t[i][j] += in ? to_float<T>(residual[base + c]) : 0.f;
                }
                ss = fmaf(t[i][j], t[i][j], ss);
            }
        }
        ss = group_sum<32>(ss);
        if (WARPS > 1) {
            __syncthreads();   // the row before is done with `red`
            if (lane == 0) {
                red[0][warp] = ss;
            }
            __syncthreads();
            ss = 0.f;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                ss += red[0][w];
            }
        }
        const float rstd = 1.f / sqrtf(ss / (float) channels + eps);
        float top[GROUPS], all = 0.f;
#pragma unroll
        for (int i = 0; i < GROUPS; ++i) {
            top[i] = 0.f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int c = (warp + WARPS * i) * 128 + 32 * j + lane;
                if (c < channels) {
                    if (sum != nullptr) {
                        sum[base + c] = from_float<T>(t[i][j]);
                    }
                    t[i][j] = t[i][j] * rstd * gm[i][j];
                    top[i] = max_nan(top[i], fabsf(t[i][j]));
                    if (OUT == NORM_SAME) {
                        out[base + c] = from_float<T>(t[i][j]);
                    }
                }
            }
            all = max_nan(all, top[i]);
        }
        if (OUT == NORM_SAME) {
            continue;
        }
        float2 sc = make_float2(0.f, 0.f);
        if (OUT == NORM_E4M3_ROW) {
            all = group_max_nan<32>(all);
            if (WARPS > 1) {
                if (lane == 0) {
                    red[1][warp] = all;
                }
                __syncthreads();
#pragma unroll
                for (int w = 0; w < WARPS; ++w) {
                    all = max_nan(all, red[1][w]);
                }
            }
            sc = e4m3_scale(all);
            if (lane == 0 && warp == 0) {
                scales[row] = sc.x;
            }
        }
#pragma unroll
        for (int i = 0; i < GROUPS; ++i) {
            const int g = warp + WARPS * i;
            if (OUT == NORM_E4M3_128) {
                sc = e4m3_scale(group_max_nan<32>(top[i]));
                if (lane == 0 && g < groups) {
                    scales[row * groups + g] = sc.x;
                }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int c = g * 128 + 32 * j + lane;
                if (c < channels) {
                    codes[base + c] = (uint8_t) e4m3_pair(t[i][j] * sc.y, 0.f);
                }
            }
        }
    }
}

constexpr int kRmsGenericBlock = 256;

// Any row length and alignment: a block per row, three passes over it (sum of squares, largest magnitude of
// each group, output); x and residual are read again from L2 in each. 2000 x 20000 binary16: 100 us, with residual and scales per 128
// columns, whose groups are two barriers each, 452.
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

// Rows of whole 16-byte vectors: a row stays in the registers of TPR threads (a warp, or a block), VPT vectors each, so x and
// residual are read once and every output is written once: the kernel is bound by those bytes. Blocks are persistent: a thread's
// columns do not change, and neither do its gamma registers. The next row is fetched before this one is reduced: 32768 x 1024
// binary16 rows with residual and e4m3 output take 43.7 us without that and 39.5 (5.9 TB/s) with it, 4096 x 8192 ones 53.7 and 44.5.
template <typename T, int TPR, int VPT, NormOut OUT>
__global__ void __launch_bounds__(TPR == 32 ? 128 : TPR)
rms_norm_kernel(const T *x, const T *residual, const T *gamma, int64_t rows, int channels, int nvec, float eps, T *sum, T *out, uint8_t *codes,
                float *scales) {
    constexpr int BLOCK = TPR == 32 ? 128 : TPR, EPV = Vec<T>::EPV, PAIRS = Vec2<T>::PAIRS, WARPS = TPR / 32;
    __shared__ float red[2][WARPS];
    const int l = TPR == 32 ? threadIdx.x & 31 : threadIdx.x;
    uint4 graw[VPT];
#pragma unroll
    for (int u = 0; u < VPT; ++u) {
        graw[u] = l + u * TPR < nvec ? ld_param(gamma + (size_t) (l + u * TPR) * EPV) : make_uint4(0, 0, 0, 0);
    }
    const float inv_channels = 1.f / (float) channels;
    const int64_t stride = (int64_t) gridDim.x * (BLOCK / TPR);
    uint4 xr[VPT], rr[VPT];
    auto fetch = [&](int64_t row) {
        const int64_t base = row * channels;
#pragma unroll
        for (int u = 0; u < VPT; ++u) {
            xr[u] = l + u * TPR < nvec ? ld_stream(x + base + (size_t) (l + u * TPR) * EPV) : make_uint4(0, 0, 0, 0);
        }
        if (residual != nullptr) {
#pragma unroll
            for (int u = 0; u < VPT; ++u) {
                rr[u] = l + u * TPR < nvec ? ld_stream(residual + base + (size_t) (l + u * TPR) * EPV) : make_uint4(0, 0, 0, 0);
            }
        }
    };
    int64_t row = (int64_t) blockIdx.x * (BLOCK / TPR) + threadIdx.x / TPR;
    if (row < rows) {
        fetch(row);
    }
    for (; row < rows; row += stride) {
        const int64_t base = row * channels;
        float2 t[VPT][PAIRS];
        float2 ss2 = make_float2(0.f, 0.f);
#pragma unroll
        for (int u = 0; u < VPT; ++u) {
            Vec2<T>::unpack(xr[u], t[u]);
            if (residual != nullptr) {
                accumulate_vec<T, false>(rr[u], t[u]);
            }
#pragma unroll
            for (int e = 0; e < PAIRS; ++e) {
                ss2 = fma2(t[u][e], t[u][e], ss2);
            }
        }
        if (row + stride < rows) {   // the next row is on its way while this one is reduced and written
            fetch(row + stride);
        }
        float ss = group_sum<32>(ss2.x + ss2.y);
        if (WARPS > 1) {
            __syncthreads();   // the row before is done with `red`
            if ((threadIdx.x & 31) == 0) {
                red[0][threadIdx.x >> 5] = ss;
            }
            __syncthreads();
            ss = 0.f;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                ss += red[0][w];
            }
        }
        if (sum != nullptr) {
#pragma unroll
            for (int u = 0; u < VPT; ++u) {
                if (l + u * TPR < nvec) {
                    st_vec(sum + base + (size_t) (l + u * TPR) * EPV, Vec2<T>::pack(t[u]));
                }
            }
        }
        const float2 rstd2 = splat2(1.f / sqrtf(ss * inv_channels + eps));
        float top[VPT];
#pragma unroll
        for (int u = 0; u < VPT; ++u) {
            float2 gm[PAIRS];
            Vec2<T>::unpack(graw[u], gm);
            top[u] = 0.f;
#pragma unroll
            for (int e = 0; e < PAIRS; ++e) {
                t[u][e] = mul2(mul2(t[u][e], rstd2), gm[e]);
                if (OUT != NORM_SAME && l + u * TPR < nvec) {
                    top[u] = max_nan(top[u], max_nan(fabsf(t[u][e].x), fabsf(t[u][e].y)));
                }
            }
        }
        float2 sc = make_float2(0.f, 0.f);
        if (OUT == NORM_E4M3_ROW) {
            float all = top[0];
#pragma unroll
            for (int u = 1; u < VPT; ++u) {
                all = max_nan(all, top[u]);
            }
            all = group_max_nan<32>(all);
            if (WARPS > 1) {
                if ((threadIdx.x & 31) == 0) {
                    red[1][threadIdx.x >> 5] = all;
                }
                __syncthreads();
#pragma unroll
                for (int w = 0; w < WARPS; ++w) {
                    all = max_nan(all, red[1][w]);
                }
            }
            sc = e4m3_scale(all);
            if (l == 0) {
                scales[row] = sc.x;
            }
        }
#pragma unroll
        for (int u = 0; u < VPT; ++u) {
            const int idx = l + u * TPR;
            if (OUT == NORM_SAME) {
                if (idx < nvec) {
                    st_vec(out + base + (size_t) idx * EPV, Vec2<T>::pack(t[u]));
                }
                continue;
            }
            if (OUT == NORM_E4M3_128) {   // 128 columns: 16 or 32 adjacent lanes
                constexpr int LANES = 128 / EPV;
                sc = e4m3_scale(group_max_nan<LANES>(top[u]));
                if (idx < nvec && idx % LANES == 0) {
                    scales[row * ((channels + 127) / 128) + idx / LANES] = sc.x;
                }
            }
            if (idx < nvec) {
                const float2 by = splat2(sc.y);
                uint32_t w[PAIRS / 2];
#pragma unroll
                for (int e = 0; e < PAIRS; e += 2) {
                    const float2 a = mul2(t[u][e], by), z = mul2(t[u][e + 1], by);
                    w[e / 2] = (uint32_t) e4m3_pair(a.x, a.y) | (uint32_t) e4m3_pair(z.x, z.y) << 16;
                }
                if (PAIRS == 4) {
                    *reinterpret_cast<uint2 *>(codes + base + (size_t) idx * EPV) = make_uint2(w[0], w[PAIRS / 2 - 1]);
                } else {
                    *reinterpret_cast<uint32_t *>(codes + base + (size_t) idx * EPV) = w[0];
                }
            }
        }
    }
}

template <typename T, int TPR, int VPT, NormOut OUT>
int rms_norm_launch(const T *x, const T *residual, const T *gamma, int64_t rows, int channels, float eps, T *sum, T *out, uint8_t *codes,
                    float *scales, cudaStream_t stream) {
    constexpr int BLOCK = TPR == 32 ? 128 : TPR, ROWS = BLOCK / TPR;
    static OccupancyCache cache;
    const int64_t resident = resident_blocks(rms_norm_kernel<T, TPR, VPT, OUT>, BLOCK, 0, &cache), want = (rows + ROWS - 1) / ROWS;
    rms_norm_kernel<T, TPR, VPT, OUT><<<(unsigned) (want < resident ? want : resident), BLOCK, 0, stream>>>(
        x, residual, gamma, rows, channels, channels / Vec<T>::EPV, eps, sum, out, codes, scales);
    return check_launch();
}

// By the vectors of a row: a warp per row up to four vectors a lane, a block of 128 to 512 threads beyond (251 float32 vectors: 12.4 us
// for 5001 rows with a warp each, 7.9 with a block of 128). False: longer rows, for the general kernel.
template <typename T, NormOut OUT>
bool rms_norm_vectors(const T *x, const T *residual, const T *gamma, int64_t rows, int channels, float eps, T *sum, T *out, uint8_t *codes,
                      float *scales, cudaStream_t stream, int *rc) {
    const int nvec = channels / Vec<T>::EPV;
#define NORM(TPR, VPT) (*rc = rms_norm_launch<T, TPR, VPT, OUT>(x, residual, gamma, rows, channels, eps, sum, out, codes, scales, stream))
    if (nvec <= 32) {
        NORM(32, 1);
    } else if (nvec <= 64) {
        NORM(32, 2);
    } else if (nvec <= 128) {
        NORM(32, 4);
    } else if (nvec <= 256) {
        NORM(128, 2);
    } else if (nvec <= 512) {
        NORM(128, 4);
    } else if (nvec <= 1024) {
        NORM(256, 4);
    } else if (nvec <= 2048) {
        NORM(512, 4);
    } else {
        return false;
    }
#undef NORM
    return true;
}

template <typename T, bool E4M3>
int residual_rms_norm(const T *x, const T *residual, const T *gamma, int64_t rows, int channels, float eps, int group, T *sum,
                      T *out, uint8_t *codes, float *scales, cudaStream_t stream) {
    if (x == nullptr || gamma == nullptr || rows < 0 || channels <= 0 || !(eps >= 0.f) || (E4M3 ? codes == nullptr || scales == nullptr : out == nullptr) ||
        (E4M3 && group != 0 && group != 128)) {
        return CUBK_ERR_INVALID_ARG;
    }
    if (channels > (1 << 30)) {   // column arithmetic is 32-bit
        return CUBK_ERR_UNSUPPORTED;
    }
    if (rows == 0) {
        return CUBK_OK;
    }
    constexpr int EPV = Vec<T>::EPV;
    if (channels % EPV == 0 && aligned16(x) && aligned16(residual) && aligned16(gamma) && aligned16(sum) && aligned16(out) && aligned8(codes)) {
        int rc = CUBK_OK;
        bool taken;
        if constexpr (E4M3) {
            taken = group == 0 ? rms_norm_vectors<T, NORM_E4M3_ROW>(x, residual, gamma, rows, channels, eps, sum, out, codes, scales, stream, &rc)
                               : rms_norm_vectors<T, NORM_E4M3_128>(x, residual, gamma, rows, channels, eps, sum, out, codes, scales, stream, &rc);
        } else {
            taken = rms_norm_vectors<T, NORM_SAME>(x, residual, gamma, rows, channels, eps, sum, out, codes, scales, stream, &rc);
        }
        if (taken) {
            return rc;
        }
    }
    if (channels <= 128 * 4 * 16) {   // 8000 x 1001 binary16: 17 us, with the three passes below 23
#define ELEMENTS(WARPS, GROUPS, OUT)                                                                                                        \
    do {                                                                                                                                    \
        const int64_t want = WARPS == 1 ? (rows + 3) / 4 : rows, most = 148 * (WARPS == 16 ? 4 : 16);                                       \
        rms_norm_elements_kernel<T, WARPS, GROUPS, OUT><<<(unsigned) (want < most ? want : most), WARPS == 1 ? 128 : 32 * WARPS, 0, stream>>>( \
            x, residual, gamma, rows, channels, eps, sum, out, codes, scales);                                                              \
    } while (0)
#define ELEMENTS_BY_LENGTH(OUT)                                                                                     \
    do {                                                                                                            \
        if (channels <= 128) {                                                                                      \
            ELEMENTS(1, 1, OUT);                                                                                    \
        } else if (channels <= 512) {                                                                               \
            ELEMENTS(1, 4, OUT);                                                                                    \
        } else if (channels <= 2048) {                                                                              \
            ELEMENTS(4, 4, OUT);                                                                                    \
        } else {                                                                                                    \
            ELEMENTS(16, 4, OUT);                                                                                   \
        }                                                                                                           \
    } while (0)
        if constexpr (E4M3) {
            if (group == 0) {
                ELEMENTS_BY_LENGTH(NORM_E4M3_ROW);
            } else {
                ELEMENTS_BY_LENGTH(NORM_E4M3_128);
            }
        } else {
            ELEMENTS_BY_LENGTH(NORM_SAME);
        }
#undef ELEMENTS_BY_LENGTH
#undef ELEMENTS
        return check_launch();
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
