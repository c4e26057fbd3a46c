// K7: products of a few rows with 4-bit weights and group scales.
//
//   out[m, n] = bias[n] + sum_k x[m, k] * code[n, k] * scale[k / group, n],   code in -8..7
//
// The codes are laid out once for warp-level matrix instructions: tiles of 16 weight rows x 128 columns (1 KB).
// Lane (g, t) = (lane / 4, lane % 4) of a warp reads 16 bytes each of rows g and g + 8 of a tile, 512 contiguous
// bytes per instruction; its word j holds columns 32 j + 8 t .. + 7 with the even ones in the low half, so that
// word & 0x000f000f, word >> 4 & ..., >> 8, >> 12 are the four operand pairs of two mma.m16n8k16 steps. The
// reduction index of an mma may be permuted as long as both operands agree: the lane's x operands are the same
// eight consecutive columns, one or two 16-byte loads. A code becomes an exact number of the operand type by
// 0x6400 | c = 1024 + c (binary16) or 0x4300 | c = 128 + c (bfloat16) and one packed subtraction, so the scales are
// applied to float32 sums of whole groups and nothing is rounded but those sums.
//   binary16 x: operands as they are.  e4m3 x: exact in binary16; their scales meet the float32 sums.
//   float32 x: split exactly into three bfloat16 parts (8 bits of mantissa each), three products.
#include <cuda_fp8.h>

#include "common.cuh"

namespace cubk {

constexpr int kW4Tile = 16;           // weight rows of a tile
constexpr int kW4Block = 128;         // columns of a tile
constexpr int kW4TileBytes = kW4Tile * kW4Block / 2;
constexpr int kW4Warps = 8;

enum XKind { X_F16, X_F32, X_E4M3 };

template <bool BF16>
__device__ __forceinline__ void w4_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if (BF16) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    } else {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
}

// The eight codes of a word as four pairs of the operand type (exact).
template <bool BF16>
__device__ __forceinline__ void w4_expand(uint32_t w, uint32_t (&p)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t c = (w >> (4 * i)) & 0x000f000fu;
        if (BF16) {
            asm("sub.bf16x2 %0, %1, %2;" : "=r"(p[i]) : "r"(c | 0x43004300u), "r"(0x43084308u));   // 128 + c - 136
        } else {
            asm("sub.f16x2 %0, %1, %2;" : "=r"(p[i]) : "r"(c | 0x64006400u), "r"(0x64086408u));    // 1024 + c - 1032
        }
    }
}

// The x operands of one lane: eight consecutive columns from k0 of a row, as SPLITS sets of four pairs.
template <XKind X>
struct XLoad;

template <>
struct XLoad<X_F16> {
    typedef __half Elem;
    static constexpr int SPLITS = 1;
    static constexpr bool BF16 = false;
    static __device__ __forceinline__ void load(const __half *row, int k0, int k, bool vec, uint32_t (&b)[1][4]) {
        if (vec && k0 + 8 <= k) {
            const uint4 v = ld_param(row + k0);
            b[0][0] = v.x, b[0][1] = v.y, b[0][2] = v.z, b[0][3] = v.w;
            return;
        }
        const unsigned short *r = reinterpret_cast<const unsigned short *>(row);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t lo = k0 + 2 * i < k ? r[k0 + 2 * i] : 0, hi = k0 + 2 * i + 1 < k ? r[k0 + 2 * i + 1] : 0;
            b[0][i] = lo | hi << 16;
        }
    }
};

template <>
struct XLoad<X_E4M3> {
    typedef uint8_t Elem;
    static constexpr int SPLITS = 1;
    static constexpr bool BF16 = false;
    static __device__ __forceinline__ void load(const uint8_t *row, int k0, int k, bool vec, uint32_t (&b)[1][4]) {
        uint32_t w[2] = {0, 0};
        if (vec && k0 + 8 <= k) {
            const uint2 v = __ldg(reinterpret_cast<const uint2 *>(row + k0));
            w[0] = v.x, w[1] = v.y;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (k0 + i < k) {
                    w[i / 4] |= (uint32_t) row[k0 + i] << (8 * (i % 4));
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint16_t pair = (uint16_t) (w[i / 2] >> (16 * (i % 2)));
            asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(b[0][i]) : "h"(pair));
        }
    }
};

template <>
struct XLoad<X_F32> {
    typedef float Elem;
    static constexpr int SPLITS = 3;
    static constexpr bool BF16 = true;
    static __device__ __forceinline__ void load(const float *row, int k0, int k, bool vec, uint32_t (&b)[3][4]) {
        float v[8];
        if (vec && k0 + 8 <= k) {
            const float4 lo = __ldg(reinterpret_cast<const float4 *>(row + k0)), hi = __ldg(reinterpret_cast<const float4 *>(row + k0) + 1);
            v[0] = lo.x, v[1] = lo.y, v[2] = lo.z, v[3] = lo.w, v[4] = hi.x, v[5] = hi.y, v[6] = hi.z, v[7] = hi.w;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                v[i] = k0 + i < k ? row[k0 + i] : 0.f;
            }
        }
        // the top 16 bits of a float32 are a bfloat16; what is left of 24 bits of mantissa after two of them fits a third
#pragma unroll
        for (int s = 0; s < 3; ++s) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t lo = __float_as_uint(v[2 * i]), hi = __float_as_uint(v[2 * i + 1]);
                b[s][i] = __byte_perm(lo, hi, 0x7632);
                v[2 * i] = rest(v[2 * i]);
                v[2 * i + 1] = rest(v[2 * i + 1]);
            }
        }
    }
    static __device__ __forceinline__ float rest(float v) {
        const uint32_t top = __float_as_uint(v) & 0xffff0000u;
        return (top & 0x7f800000u) == 0x7f800000u ? 0.f : v - __uint_as_float(top);   // an infinity leaves nothing
    }
};

// Block: one tile of 16 weight rows x 8 * TT rows of x; the warps take the column blocks in turn and join in shared memory.
template <typename T, XKind X, int TT>
__global__ void __launch_bounds__(32 * kW4Warps)
w4_matvec_kernel(const typename XLoad<X>::Elem *x, const float *x_scales, int x_groups, int rows, int k, const uint8_t *packed,
                 const T *scales, int group, int n, const T *bias, T *out, bool vec) {
    constexpr int SPLITS = XLoad<X>::SPLITS;
    constexpr bool BF16 = XLoad<X>::BF16;
    __shared__ float s_acc[kW4Warps][TT][32][5];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
    const int kblocks = (k + kW4Block - 1) / kW4Block;
    const int row0 = blockIdx.y * (8 * TT);
    const int n0 = blockIdx.x * kW4Tile;
    const uint8_t *tile = packed + (size_t) blockIdx.x * kblocks * kW4TileBytes + lane * 16;
    const int na = n0 + g < n ? n0 + g : n - 1, nb = n0 + g + 8 < n ? n0 + g + 8 : n - 1;   // rows past n are discarded at the end
    const int steps = group / 32;   // 32-column steps of a group

    float acc[TT][4];
#pragma unroll
    for (int m = 0; m < TT; ++m) {
        acc[m][0] = acc[m][1] = acc[m][2] = acc[m][3] = 0.f;
    }
    for (int kb = warp; kb < kblocks; kb += kW4Warps) {
        const uint4 ra = ld_stream(tile + (size_t) kb * kW4TileBytes), rb = ld_stream(tile + (size_t) kb * kW4TileBytes + 512);
        const uint32_t wa[4] = {ra.x, ra.y, ra.z, ra.w}, wb[4] = {rb.x, rb.y, rb.z, rb.w};
        float sum[TT][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int k0 = kb * kW4Block + 32 * j;
            if (k0 >= k) {
                break;
            }
            if (j % steps == 0) {
#pragma unroll
                for (int m = 0; m < TT; ++m) {
                    sum[m][0] = sum[m][1] = sum[m][2] = sum[m][3] = 0.f;
                }
            }
            uint32_t pa[4], pb[4];
            w4_expand<BF16>(wa[j], pa);
            w4_expand<BF16>(wb[j], pb);
            const uint32_t a0[4] = {pa[0], pb[0], pa[1], pb[1]}, a1[4] = {pa[2], pb[2], pa[3], pb[3]};
#pragma unroll
            for (int m = 0; m < TT; ++m) {
                const int row = row0 + 8 * m + g;
                uint32_t b[SPLITS][4];
#pragma unroll
                for (int s = 0; s < SPLITS; ++s) {
                    b[s][0] = b[s][1] = b[s][2] = b[s][3] = 0;
                }
                if (row < rows) {
                    XLoad<X>::load(x + (size_t) row * k, k0 + 8 * t, k, vec, b);
                }
#pragma unroll
                for (int s = SPLITS - 1; s >= 0; --s) {
                    w4_mma<BF16>(sum[m], a0, b[s][0], b[s][1]);
                    w4_mma<BF16>(sum[m], a1, b[s][2], b[s][3]);
                }
            }
            if ((j + 1) % steps == 0 || k0 + 32 >= k) {
                const T *sc = scales + (size_t) (k0 / group) * n;
                const float sa = to_float<T>(sc[na]), sb = to_float<T>(sc[nb]);
#pragma unroll
                for (int m = 0; m < TT; ++m) {
                    float x0 = 1.f, x1 = 1.f;
                    if (X == X_E4M3 && x_groups > 1) {
                        const int r = row0 + 8 * m + 2 * t;
                        x0 = r < rows ? x_scales[(size_t) r * x_groups + kb] : 0.f;
                        x1 = r + 1 < rows ? x_scales[(size_t) (r + 1) * x_groups + kb] : 0.f;
                    }
                    acc[m][0] = fmaf(sum[m][0] * x0, sa, acc[m][0]);
                    acc[m][1] = fmaf(sum[m][1] * x1, sa, acc[m][1]);
                    acc[m][2] = fmaf(sum[m][2] * x0, sb, acc[m][2]);
                    acc[m][3] = fmaf(sum[m][3] * x1, sb, acc[m][3]);
                }
            }
        }
    }
#pragma unroll
    for (int m = 0; m < TT; ++m) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            s_acc[warp][m][lane][i] = acc[m][i];
        }
    }
    __syncthreads();
    // output element e of the block: weight row e % 16 (contiguous in out), x row e / 16
    for (int e = threadIdx.x; e < 16 * 8 * TT; e += 32 * kW4Warps) {
        const int c = e % 16, r = e / 16;
        const int from = (c % 8) * 4 + (r % 8) / 2, i = 2 * (c / 8) + r % 2;
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < kW4Warps; ++w) {
            v += s_acc[w][r / 8][from][i];
        }
        if (n0 + c < n && row0 + r < rows) {
            if (X == X_E4M3 && x_groups == 1) {
                v *= x_scales[row0 + r];
            }
            if (bias != nullptr) {
                v += to_float<T>(bias[n0 + c]);
            }
            out[(size_t) (row0 + r) * n + n0 + c] = from_float<T>(v);
        }
    }
}

template <typename T, XKind X>
int w4_matvec(const typename XLoad<X>::Elem *x, const float *x_scales, int x_group, int rows, int k, const void *packed,
              const T *scales, int group, int n, const T *bias, T *out, cudaStream_t stream) {
    if (x == nullptr || packed == nullptr || scales == nullptr || out == nullptr || rows < 0 || k <= 0 || n <= 0 || k > (1 << 30) ||
        (group != 32 && group != 64 && group != 128) || (X == X_E4M3 && (x_scales == nullptr || (x_group != 0 && x_group != 128)))) {
        return CUBK_ERR_INVALID_ARG;
    }
    if (!aligned16(packed) || (rows + 63) / 64 > 65535) {
        return CUBK_ERR_UNSUPPORTED;
    }
    if (rows == 0) {
        return CUBK_OK;
    }
    constexpr int kLane = 8 * (int) sizeof(*x);   // bytes of a lane's eight columns
    const bool vec = k % (X == X_E4M3 ? 8 : 16 / (int) sizeof(*x)) == 0 && reinterpret_cast<uintptr_t>(x) % (kLane < 16 ? kLane : 16) == 0;
    const int x_groups = x_group == 0 ? 1 : (k + 127) / 128;
    const int xg = X == X_E4M3 ? x_groups : 1;
    const unsigned tiles = (unsigned) ((n + kW4Tile - 1) / kW4Tile);
#define W4_LAUNCH(TT)                                                                                                  \
    w4_matvec_kernel<T, X, TT><<<dim3(tiles, (unsigned) ((rows + 8 * TT - 1) / (8 * TT))), 32 * kW4Warps, 0, stream>>>( \
        x, x_scales, xg, rows, k, (const uint8_t *) packed, scales, group, n, bias, out, vec)
    if (rows <= 8) {
        W4_LAUNCH(1);
    } else if (rows <= 16) {
        W4_LAUNCH(2);
    } else {
        W4_LAUNCH(4);
    }
#undef W4_LAUNCH
    return check_launch();
}

// ---------------------------------------------------------------- laying the weights out
// One thread per word (eight consecutive columns of a row). Rows and columns past the matrix get code 0.
__device__ __forceinline__ size_t w4_word_index(int row, int word_col, int kblocks) {
    const int kb = word_col >> 4, i = word_col & 15;              // the word's columns: 128 kb + 8 i
    return ((size_t) (row >> 4) * kblocks + kb) * (kW4TileBytes / 4) + (row & 15) * 16 + 4 * (i & 3) + (i >> 2);
}

__device__ __forceinline__ uint32_t w4_word(const int (&c)[8]) {
    uint32_t w = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        w |= (uint32_t) (c[e] + 8) << (16 * (e & 1) + 4 * (e >> 1));
    }
    return w;
}

// Codes by rounding to nearest even under the group's scale = max|w| / 7, rounded to the storage type first.
template <typename T>
__global__ void __launch_bounds__(256)
w4_quantize_kernel(const T *weights, int n, int k, int group, int kblocks, int64_t words, uint32_t *packed, T *scales) {
    const int64_t i = (int64_t) blockIdx.x * 256 + threadIdx.x;   // `words` is a multiple of 256: no lane is alone in its group
    if (i >= words) {
        return;
    }
    const int per_row = kblocks * 16;
    const int row = (int) (i / per_row), wc = (int) (i - (int64_t) row * per_row);
    const int k0 = wc * 8;
    float v[8];
    float top = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        v[e] = row < n && k0 + e < k ? to_float<T>(weights[(size_t) row * k + k0 + e]) : 0.f;
        top = fmaxf(top, fabsf(v[e]));
    }
    for (int o = 1; o < group / 8; o <<= 1) {
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    }
    const T stored = from_float<T>(top / 7.f);
    const float scale = to_float<T>(stored);
    int c[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float q = scale > 0.f ? rintf(v[e] / scale) : 0.f;
        c[e] = (int) fminf(fmaxf(q, -8.f), 7.f);
    }
    packed[w4_word_index(row, wc, kblocks)] = w4_word(c);
    if (row < n && k0 < k && (k0 % group) == 0) {
        scales[(size_t) (k0 / group) * n + row] = stored;
    }
}

__global__ void __launch_bounds__(256)
w4_pack_kernel(const int8_t *codes, int n, int k, int kblocks, int64_t words, uint32_t *packed) {
    const int64_t i = (int64_t) blockIdx.x * 256 + threadIdx.x;
    if (i >= words) {
        return;
    }
    const int per_row = kblocks * 16;
    const int row = (int) (i / per_row), wc = (int) (i - (int64_t) row * per_row);
    int c[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        c[e] = row < n && wc * 8 + e < k ? min(max((int) codes[(size_t) row * k + wc * 8 + e], -8), 7) : 0;
    }
    packed[w4_word_index(row, wc, kblocks)] = w4_word(c);
}

struct W4Grid {
    int kblocks;
    int64_t words;
    unsigned blocks;
    bool ok;
};

inline W4Grid w4_grid(int n, int k) {
    W4Grid w;
    w.kblocks = (k + kW4Block - 1) / kW4Block;
    w.words = (int64_t) ((n + kW4Tile - 1) / kW4Tile) * kW4Tile * w.kblocks * 16;   // a multiple of 256
    w.ok = w.words / 256 <= 0x7fffffffLL;
    w.blocks = (unsigned) (w.words / 256);
    return w;
}

template <typename T>
int w4_quantize(const T *weights, int n, int k, int group, void *packed, T *scales, cudaStream_t stream) {
    if (weights == nullptr || packed == nullptr || scales == nullptr || n <= 0 || k <= 0 || k > (1 << 30) ||
        (group != 32 && group != 64 && group != 128)) {
        return CUBK_ERR_INVALID_ARG;
    }
    const W4Grid w = w4_grid(n, k);
    if (!aligned16(packed) || !w.ok) {
        return CUBK_ERR_UNSUPPORTED;
    }
    w4_quantize_kernel<T><<<w.blocks, 256, 0, stream>>>(weights, n, k, group, w.kblocks, w.words, (uint32_t *) packed, scales);
    return check_launch();
}

}  // namespace cubk

extern "C" {

size_t cubk_w4_packed_bytes(int n, int k) {
    if (n <= 0 || k <= 0) {
        return 0;
    }
    return (((size_t) n + cubk::kW4Tile - 1) / cubk::kW4Tile) * (((size_t) k + cubk::kW4Block - 1) / cubk::kW4Block) * cubk::kW4TileBytes;
}

int cubk_w4_quantize_f32(const float *weights, int n, int k, int group, void *packed, float *scales, void *stream) {
    return cubk::w4_quantize<float>(weights, n, k, group, packed, scales, (cudaStream_t) stream);
}

int cubk_w4_quantize_f16(const void *weights, int n, int k, int group, void *packed, void *scales, void *stream) {
    return cubk::w4_quantize<__half>((const __half *) weights, n, k, group, packed, (__half *) scales, (cudaStream_t) stream);
}

int cubk_w4_pack(const int8_t *codes, int n, int k, void *packed, void *stream) {
    if (codes == nullptr || packed == nullptr || n <= 0 || k <= 0 || k > (1 << 30)) {
        return CUBK_ERR_INVALID_ARG;
    }
    const cubk::W4Grid w = cubk::w4_grid(n, k);
    if (!cubk::aligned16(packed) || !w.ok) {
        return CUBK_ERR_UNSUPPORTED;
    }
    cubk::w4_pack_kernel<<<w.blocks, 256, 0, (cudaStream_t) stream>>>(codes, n, k, w.kblocks, w.words, (uint32_t *) packed);
    return cubk::check_launch();
}

int cubk_w4_matvec_f32(const float *x, int rows, int k, const void *packed, const float *scales, int group, int n, const float *bias,
                       float *out, void *stream) {
    return cubk::w4_matvec<float, cubk::X_F32>(x, nullptr, 0, rows, k, packed, scales, group, n, bias, out, (cudaStream_t) stream);
}

int cubk_w4_matvec_f16(const void *x, int rows, int k, const void *packed, const void *scales, int group, int n, const void *bias,
                       void *out, void *stream) {
    return cubk::w4_matvec<__half, cubk::X_F16>((const __half *) x, nullptr, 0, rows, k, packed, (const __half *) scales, group, n,
                                                (const __half *) bias, (__half *) out, (cudaStream_t) stream);
}

int cubk_w4_matvec_e4m3_f32(const void *codes, const float *code_scales, int code_group, int rows, int k, const void *packed,
                            const float *scales, int group, int n, const float *bias, float *out, void *stream) {
    return cubk::w4_matvec<float, cubk::X_E4M3>((const uint8_t *) codes, code_scales, code_group, rows, k, packed, scales, group, n, bias,
                                                out, (cudaStream_t) stream);
}

int cubk_w4_matvec_e4m3_f16(const void *codes, const float *code_scales, int code_group, int rows, int k, const void *packed,
                            const void *scales, int group, int n, const void *bias, void *out, void *stream) {
    return cubk::w4_matvec<__half, cubk::X_E4M3>((const uint8_t *) codes, code_scales, code_group, rows, k, packed,
                                                 (const __half *) scales, group, n, (const __half *) bias, (__half *) out,
                                                 (cudaStream_t) stream);
}

}  // extern "C"
