// K8, whole sequences: attention with a sliding window and first tokens that stay visible (sinks).
//
// Query i sees key j when the key is kept, j <= i + after, and j >= i - before or j < sinks. Softmax statistics and all sums
// are float32. A key that a query does not see contributes nothing at all, whatever bits its rows hold; a query that sees no
// key gets zeros.
#include <cuda.h>

#include <atomic>
#include <type_traits>

#include "window_row.cuh"
#include "window_turns.h"

namespace cubk {

struct WindowShape {
    int batch, seq, heads, kv_heads, dim;
    int before, after, sinks;
    float scale;
    int64_t q_stride, kv_stride, context_stride;
};

// Row (b, i) of head h of a whole sequence.
template <typename T, int COLS>
__device__ __forceinline__ void window_prompt_row(const T *q, const T *k, const T *v, const int8_t *mask, T *context, const WindowShape &s,
                                                  float *s_q, int b, int i, int h) {
    const int64_t first = (int64_t) b * s.seq;
    const int kh = h / (s.heads / s.kv_heads);
    const int8_t *kept = mask != nullptr ? mask + first : nullptr;
    const T *kb = k + first * s.kv_stride + (int64_t) kh * s.dim, *vb = v + first * s.kv_stride + (int64_t) kh * s.dim;
    const int lo = i > s.before ? i - s.before : 0;
    const int hi = s.after < s.seq - 1 - i ? i + s.after + 1 : s.seq;
    window_row<T, COLS>(q + (first + i) * s.q_stride + (int64_t) h * s.dim, s_q, s.dim, s.scale, min(min(s.sinks, lo), hi), lo, hi,
                  [&](int j) { return kb + j * s.kv_stride; }, [&](int j) { return vb + j * s.kv_stride; },
                  [&](int j) { return kept == nullptr || kept[j] != 0; }, context + (first + i) * s.context_stride + (int64_t) h * s.dim);
}

template <typename T, int COLS>
__global__ void __launch_bounds__(32 * kWindowRowWarps)
window_rows_kernel(const T *q, const T *k, const T *v, const int8_t *mask, T *context, WindowShape s) {
    __shared__ float s_q[kWindowRowWarps][kWindowMaxDim];
    const int warp = threadIdx.x >> 5;
    const int64_t total = (int64_t) s.batch * s.seq * s.heads;
    for (int64_t r = (int64_t) blockIdx.x * kWindowRowWarps + warp; r < total; r += (int64_t) gridDim.x * kWindowRowWarps) {
        const int64_t bh = r / s.seq;
        window_prompt_row<T, COLS>(q, k, v, mask, context, s, s_q[warp], (int) (bh / s.heads), (int) (r - bh * s.seq), (int) (bh % s.heads));
    }
}

// ---- whole sequences on the float32 pipes (float32 storage; binary16 rows that TMA cannot read)
// 64 query rows of a head a block, 64 keys a step out of one list: the kept ones of the sinks below the window, then of the window (so
// that masked keys, wherever they are, cost neither loads nor multiply-adds). A thread owns 8 rows
// x 4 keys of the scores and 8 rows x DP / 16 columns of the context; Q and K are transposed on their way into shared memory, so that
// each step of a reduction is two or three 16-byte reads for 32 or 64 multiply-adds, issued in pairs of rows. The 16 threads of a row
// are half a warp: maxima and sums need shuffles only. Bound by the multiply-adds, and for short windows by the latency of a block's
// two or three steps: 3 x 777 tokens, 12 heads of 64, window 131, half of the keys masked: 37 us, 468 blocks in 1.05 waves.
constexpr int kPlainRows = 64, kPlainKeys = 64, kPlainThreads = 128;

template <int DP>
struct WindowPlain {
    static constexpr int QK = kPlainRows + 4;       // floats between columns of the transposed tiles: 16-byte rows over all banks
    static constexpr int FLOATS = 2 * DP * QK + kPlainKeys * DP;   // the weights take the keys' place
    static constexpr int BYTES = FLOATS * 4;
};

// Bits lo .. hi - 1 of a word that stands for positions base .. base + 31.
__device__ __forceinline__ uint32_t range_bits(int lo, int hi, int base) {
    const int a = min(max(lo - base, 0), 32), b = min(max(hi - base, 0), 32);
    const uint32_t below_b = b == 32 ? 0xffffffffu : (1u << b) - 1u, below_a = a == 32 ? 0xffffffffu : (1u << a) - 1u;
    return below_b & ~below_a;
}

// Columns c .. c + 3 of a row as float32, zeros past the dimension.
template <typename T>
__device__ __forceinline__ float4 four_columns(const T *row, int c, int dim, bool vec) {
    if (sizeof(T) == 4 && vec) {
        return c < dim ? __ldg(reinterpret_cast<const float4 *>(row + c)) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    return make_float4(c < dim ? to_float<T>(row[c]) : 0.f, c + 1 < dim ? to_float<T>(row[c + 1]) : 0.f,
                       c + 2 < dim ? to_float<T>(row[c + 2]) : 0.f, c + 3 < dim ? to_float<T>(row[c + 3]) : 0.f);
}

constexpr int kNotFinite = 1, kSumZero = 2;   // what a row came out with

// The rows of a block that need another look, out of the way of the others' code. A row that is not finite is computed again over its
// visible keys alone. A row with a sum of 0 sees no key, and is zeros, or nothing but scores of minus infinity, and is NaN (0 / 0):
// which, the mask says, 4096 candidates at a time as bits in the list's place, a word a lane.
template <typename T, int DP>
__device__ __noinline__ void window_plain_again(const T *q, const T *k, const T *v, const int8_t *mask, T *context, const WindowShape *s, float *s_q,
                                                int *s_list, int *s_bad, int b, int h, int row0) {
    constexpr int WARPS = kPlainThreads / 32, WORDS = 128;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int last_row = min(row0 + kPlainRows, s->seq) - 1;
    const int lo = row0 > s->before ? row0 - s->before : 0;
    const int hi = s->after < s->seq - 1 - last_row ? last_row + s->after + 1 : s->seq;
    const int sinks_end = min(s->sinks, lo), listed = sinks_end + hi - lo;
    const int8_t *kept = mask != nullptr ? mask + (int64_t) b * s->seq : nullptr;
    if (__syncthreads_or(threadIdx.x < kPlainRows && s_bad[threadIdx.x] == kSumZero)) {
        for (int base = 0; base < listed; base += 32 * WORDS) {
            const int words = min(WORDS, (listed - base + 31) / 32);
#pragma unroll 4
            for (int w = warp; w < words; w += WARPS) {
                const int u = base + 32 * w + lane, j = u < sinks_end ? u : lo + u - sinks_end;
                const unsigned on = __ballot_sync(0xffffffffu, u < listed && (kept == nullptr || kept[j] != 0));
                if (lane == 0) {
                    s_list[w] = (int) on;
                }
            }
            __syncthreads();
            if (threadIdx.x < kPlainRows && s_bad[threadIdx.x] == kSumZero) {
                const int i = row0 + (int) threadIdx.x;
                const int i_lo = i > s->before ? i - s->before : 0, i_hi = s->after < s->seq - 1 - i ? i + s->after + 1 : s->seq;
                const int sinks = min(s->sinks, i_hi), from = i_lo - lo + sinks_end, to = i_hi - lo + sinks_end;   // candidates that the row may see
                unsigned seen = 0;
                for (int w = 0; w < words; ++w) {
                    const int bit = base + 32 * w;
                    seen |= (unsigned) s_list[w] & (range_bits(0, sinks, bit) | range_bits(from, to, bit));
                }
                if (seen != 0) {
                    s_bad[threadIdx.x] = kNotFinite;
                }
            }
            __syncthreads();
        }
    }
    for (int r = warp; r < kPlainRows; r += WARPS) {
        if (s_bad[r] == kNotFinite) {
            window_prompt_row<T, DP / 32>(q, k, v, mask, context, *s, s_q + warp * kWindowMaxDim, b, row0 + r, h);
        }
    }
}

template <typename T, int DP>
__global__ void __launch_bounds__(kPlainThreads, DP == 64 ? 3 : 2)
window_plain_kernel(const T *q, const T *k, const T *v, const int8_t *mask, T *context, const __grid_constant__ WindowShape s, int row_blocks, bool vec) {
    typedef WindowPlain<DP> C;
    constexpr int VC = DP / 64;   // 4-column groups of a thread's context
    extern __shared__ __align__(16) float plain_smem[];
    float *s_q = plain_smem, *s_k = s_q + DP * C::QK, *s_v = s_k + DP * C::QK, *s_p = s_k;   // [column][row], .., [key][column], [key][row]
    __shared__ __align__(16) int s_list[kPlainKeys + kPlainThreads];   // kept keys not yet used
    __shared__ int s_found[kPlainThreads / 32], s_bad[kPlainRows];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int rg = threadIdx.x >> 4, cg = threadIdx.x & 15;   // rows 8 rg .., keys 4 cg .., columns 4 cg + 64 x ..
    const int rb = row_blocks - 1 - (int) (blockIdx.x % row_blocks);
    const int64_t bh = blockIdx.x / row_blocks;
    const int b = (int) (bh / s.heads), h = (int) (bh - (int64_t) b * s.heads), kh = h / (s.heads / s.kv_heads);
    const int row0 = rb * kPlainRows, last_row = min(row0 + kPlainRows, s.seq) - 1;
    const int64_t first = (int64_t) b * s.seq;
    const T *qb = q + first * s.q_stride + (int64_t) h * s.dim, *kb = k + first * s.kv_stride + (int64_t) kh * s.dim;
    const T *vb = v + first * s.kv_stride + (int64_t) kh * s.dim;
    const int8_t *kept = mask != nullptr ? mask + first : nullptr;
    const int lo = row0 > s.before ? row0 - s.before : 0;
    const int hi = s.after < s.seq - 1 - last_row ? last_row + s.after + 1 : s.seq;
    const int sinks_end = min(s.sinks, lo), listed = sinks_end + hi - lo;

#pragma unroll
    for (int part = 0; part < VC; ++part) {   // eight loads of a thread in flight
        constexpr int LOADS = kPlainRows * 16 / kPlainThreads;
        float4 x[LOADS];
#pragma unroll
        for (int u = 0; u < LOADS; ++u) {
            const int i = threadIdx.x + u * kPlainThreads, r = i % kPlainRows, c = 64 * part + 4 * (i / kPlainRows);
            x[u] = row0 + r < s.seq ? four_columns<T>(qb + (int64_t) (row0 + r) * s.q_stride, c, s.dim, vec) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
#pragma unroll
        for (int u = 0; u < LOADS; ++u) {
            const int i = threadIdx.x + u * kPlainThreads, r = i % kPlainRows, c = 64 * part + 4 * (i / kPlainRows);
            s_q[c * C::QK + r] = x[u].x, s_q[(c + 1) * C::QK + r] = x[u].y, s_q[(c + 2) * C::QK + r] = x[u].z, s_q[(c + 3) * C::QK + r] = x[u].w;
        }
    }
    const float c2 = s.scale * kLog2e;
    float top[8], total[8];
    float2 o[4][4 * VC];   // pairs of rows x columns
#pragma unroll
    for (int r = 0; r < 8; ++r) {
        top[r] = -INFINITY;
        total[r] = 0.f;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
#pragma unroll
        for (int c = 0; c < 4 * VC; ++c) {
            o[r][c] = make_float2(0.f, 0.f);
        }
    }
    int cursor = 0, have = 0;   // candidates looked at, keys in the list
    bool met = false;           // any key at all
    for (;;) {
        while (have < kPlainKeys && cursor < listed) {
            const int u = cursor + threadIdx.x, j = u < sinks_end ? u : lo + u - sinks_end;
            const bool on = u < listed && (kept == nullptr || kept[j] != 0);
            const unsigned found = __ballot_sync(0xffffffffu, on);
            if (lane == 0) {
                s_found[warp] = __popc(found);
            }
            __syncthreads();
            int at = have;
#pragma unroll
            for (int w = 0; w < kPlainThreads / 32; ++w) {
                at += w < warp ? s_found[w] : 0;
                have += s_found[w];
            }
            if (on) {
                s_list[at + __popc(found & ((1u << lane) - 1u))] = j;
            }
            cursor += kPlainThreads;
            __syncthreads();
        }
        const int keys = min(have, kPlainKeys);
        if (keys == 0) {
            break;
        }
        met = true;
        __syncthreads();   // the list, also where it needed nothing
        // eight loads of a thread in flight at a time
#pragma unroll
        for (int half = 0; half < 2 * VC; ++half) {
            constexpr int LOADS = kPlainKeys * 16 / kPlainThreads;   // of 64 columns
            const bool is_v = half >= VC;
            float4 x[LOADS];
#pragma unroll
            for (int u = 0; u < LOADS; ++u) {
                const int i = threadIdx.x + u * kPlainThreads;
                const int r = is_v ? i / 16 : i % kPlainKeys, c = 64 * (half % VC) + 4 * (is_v ? i % 16 : i / kPlainKeys);
                x[u] = r < keys ? four_columns<T>((is_v ? vb : kb) + (int64_t) s_list[r] * s.kv_stride, c, s.dim, vec)
                                : make_float4(0.f, 0.f, 0.f, 0.f);
            }
#pragma unroll
            for (int u = 0; u < LOADS; ++u) {
                const int i = threadIdx.x + u * kPlainThreads;
                const int r = is_v ? i / 16 : i % kPlainKeys, c = 64 * (half % VC) + 4 * (is_v ? i % 16 : i / kPlainKeys);
                if (is_v) {
                    *reinterpret_cast<float4 *>(&s_v[r * DP + c]) = x[u];
                } else {
                    s_k[c * C::QK + r] = x[u].x, s_k[(c + 1) * C::QK + r] = x[u].y, s_k[(c + 2) * C::QK + r] = x[u].z, s_k[(c + 3) * C::QK + r] = x[u].w;
                }
            }
        }
        __syncthreads();
        float2 sc[4][4];   // pairs of rows x keys
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            sc[r][0] = sc[r][1] = sc[r][2] = sc[r][3] = make_float2(0.f, 0.f);
        }
#pragma unroll 4
        for (int c = 0; c < s.dim; ++c) {
            const float4 q0 = *reinterpret_cast<const float4 *>(&s_q[c * C::QK + 8 * rg]), q1 = *reinterpret_cast<const float4 *>(&s_q[c * C::QK + 8 * rg + 4]);
            const float4 kk = *reinterpret_cast<const float4 *>(&s_k[c * C::QK + 4 * cg]);
            const float2 rows[4] = {make_float2(q0.x, q0.y), make_float2(q0.z, q0.w), make_float2(q1.x, q1.y), make_float2(q1.z, q1.w)};
            const float2 ks[4] = {splat2(kk.x), splat2(kk.y), splat2(kk.z), splat2(kk.w)};
#pragma unroll
            for (int r = 0; r < 4; ++r) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    sc[r][e] = fma2(rows[r], ks[e], sc[r][e]);
                }
            }
        }
        // a key of the list counts for row i when it is at most i + after, and at least i - before or below the sinks
        const int4 js = *reinterpret_cast<const int4 *>(&s_list[4 * cg]);
        const int j4[4] = {4 * cg < keys ? js.x : -1, 4 * cg + 1 < keys ? js.y : -1, 4 * cg + 2 < keys ? js.z : -1, 4 * cg + 3 < keys ? js.w : -1};
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            const int i = row0 + 8 * rg + r;
            const int i_lo = i > s.before ? i - s.before : 0, i_hi = s.after < s.seq ? i + s.after : s.seq;
            float p[4], here = top[r];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float x = (r & 1) ? sc[r / 2][e].y : sc[r / 2][e].x;
                const bool see = j4[e] >= 0 && j4[e] <= i_hi && (j4[e] >= i_lo || j4[e] < s.sinks);
                p[e] = see ? x * c2 : -INFINITY;
                here = fmaxf(here, p[e]);
            }
            here = group_max<16>(here);
            const float base = here == -INFINITY ? 0.f : here, shrink = top[r] == here ? 1.f : fast_exp2(top[r] - here);
            top[r] = here;
            float sum = 0.f;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                p[e] = fast_exp2(p[e] - base);
                sum += p[e];
                if (r & 1) {
                    sc[r / 2][e].y = p[e];
                } else {
                    sc[r / 2][e].x = p[e];
                }
            }
            total[r] = fmaf(total[r], shrink, sum);   // of this thread's keys
#pragma unroll
            for (int c = 0; c < 4 * VC; ++c) {
                if (r & 1) {
                    o[r / 2][c].y *= shrink;
                } else {
                    o[r / 2][c].x *= shrink;
                }
            }
        }
        __syncthreads();   // the keys have been read
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float *to = &s_p[(4 * cg + e) * C::QK + 8 * rg];
            *reinterpret_cast<float4 *>(to) = make_float4(sc[0][e].x, sc[0][e].y, sc[1][e].x, sc[1][e].y);
            *reinterpret_cast<float4 *>(to + 4) = make_float4(sc[2][e].x, sc[2][e].y, sc[3][e].x, sc[3][e].y);
        }
        __syncwarp();   // a row's weights stay within its warp
#pragma unroll 4
        for (int j = 0; j < keys; ++j) {
            const float4 p0 = *reinterpret_cast<const float4 *>(&s_p[j * C::QK + 8 * rg]), p1 = *reinterpret_cast<const float4 *>(&s_p[j * C::QK + 8 * rg + 4]);
            const float2 rows[4] = {make_float2(p0.x, p0.y), make_float2(p0.z, p0.w), make_float2(p1.x, p1.y), make_float2(p1.z, p1.w)};
#pragma unroll
            for (int x = 0; x < VC; ++x) {
                const float4 vv = *reinterpret_cast<const float4 *>(&s_v[j * DP + 64 * x + 4 * cg]);
                const float2 vs[4] = {splat2(vv.x), splat2(vv.y), splat2(vv.z), splat2(vv.w)};
#pragma unroll
                for (int r = 0; r < 4; ++r) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        o[r][4 * x + e] = fma2(rows[r], vs[e], o[r][4 * x + e]);
                    }
                }
            }
        }
        // what the list holds beyond this step moves to its front
        const int left = have - keys;
        __syncthreads();   // the list, keys, values and weights of this step have been read
        const int moved = (int) threadIdx.x < left ? s_list[kPlainKeys + threadIdx.x] : 0;
        __syncthreads();
        if ((int) threadIdx.x < left) {
            s_list[threadIdx.x] = moved;
        }
        have = left;
    }
    const float most = sizeof(T) == 4 ? 3.402823466e38f : 65504.f;
    bool rest = false;
#pragma unroll
    for (int r = 0; r < 8; ++r) {
        const float all = group_sum<16>(total[r]);
        const float inv = all == 0.f ? 0.f : 1.f / all;
        const int i = row0 + 8 * rg + r;
        bool finite = true;   // or NaN as it is, from a visible score
        T *out = context + (first + i) * s.context_stride + (int64_t) h * s.dim;
#pragma unroll
        for (int c = 0; c < 4 * VC; ++c) {
            const int col = 64 * (c / 4) + 4 * cg + c % 4;
            const float x = ((r & 1) ? o[r / 2][c].y : o[r / 2][c].x) * inv;
            if (col < s.dim) {
                finite = finite && (fabsf(x) <= most || all != all);
                if (i < s.seq) {
                    out[col] = from_float<T>(x);
                }
            }
        }
        const unsigned bad = __ballot_sync(0xffffffffu, !finite);
        if (cg == 0) {
            s_bad[8 * rg + r] = i >= s.seq ? 0 : (bad >> (lane & 16) & 0xffffu) != 0 ? kNotFinite : all == 0.f ? kSumZero : 0;
            rest = rest || s_bad[8 * rg + r] != 0;
        }
    }
    if (__syncthreads_or(rest && met)) {   // Q is no longer read: its place serves the rows that are computed again
        window_plain_again<T, DP>(q, k, v, mask, context, &s, s_q, s_list, s_bad, b, h, row0);
    }
}

template <typename T, int DP>
int window_plain_launch(const T *q, const T *k, const T *v, const int8_t *mask, T *context, const WindowShape &s, cudaStream_t stream) {
    static std::atomic<uint64_t> prepared{0};
    int dev = 0;
    cudaError_t err = cudaGetDevice(&dev);
    if (err == cudaSuccess && (dev >= 64 || ((prepared.load(std::memory_order_acquire) >> dev) & 1ull) == 0)) {
        err = cudaFuncSetAttribute(window_plain_kernel<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, WindowPlain<DP>::BYTES);
        if (err == cudaSuccess && dev < 64) {
            prepared.fetch_or(1ull << dev, std::memory_order_release);
        }
    }
    if (err != cudaSuccess) {
        set_last_error(err);
        return CUBK_ERR_LAUNCH;
    }
    const int row_blocks = (s.seq + kPlainRows - 1) / kPlainRows;
    const int64_t blocks = (int64_t) row_blocks * s.batch * s.heads;
    if (blocks > 0x7fffffffLL) {
        return CUBK_ERR_UNSUPPORTED;
    }
    const bool vec = sizeof(T) == 4 && s.dim % 4 == 0 && s.q_stride % 4 == 0 && s.kv_stride % 4 == 0 && aligned16(q) && aligned16(k) && aligned16(v);
    window_plain_kernel<T, DP><<<(unsigned) blocks, kPlainThreads, WindowPlain<DP>::BYTES, stream>>>(q, k, v, mask, context, s, row_blocks, vec);
    return check_launch();
}

// Head dimensions up to 128; CUBK_ERR_UNSUPPORTED beyond.
template <typename T>
int window_plain(const T *q, const T *k, const T *v, const int8_t *mask, T *context, const WindowShape &s, cudaStream_t stream) {
    return s.dim > 128 ? CUBK_ERR_UNSUPPORTED
           : s.dim > 64 ? window_plain_launch<T, 128>(q, k, v, mask, context, s, stream)
                        : window_plain_launch<T, 64>(q, k, v, mask, context, s, stream);
}

// ---------------------------------------------------------------- whole sequences on tcgen05 (binary16)
// A work item is NQ tiles of 128 query rows: two heads that share their keys, or consecutive rows of one head. The grid has a block
// per item; a block that runs takes over items of blocks that have not started yet (cluster launch control), loading and multiplying
// ahead into the next while the last one's rows are written, so that only the first block on an SM waits for its first loads. Per
// step of up to KEYS keys and per tile: S = Q.K^T (tcgen05.mma, float32 accumulators in tensor memory), softmax by 128 threads that
// own a row each (tensor-memory lane = query row, so no shuffles), P back into tensor memory as binary16, O += P.V with P as the
// tensor-memory operand. Warps: 4 NQ for the softmax, NQ that issue the MMAs of a tile, one that takes items, chooses their steps and
// loads Q, K and V with TMA (128-byte swizzle; V is read as it lies, as an MN-major operand).
//   * The scores' place is free as soon as a row is in registers, so the next step's scores are computed while this step's
//     exponentials are; the weights have a place of their own, so their product runs under the next step's softmax. KEYS is what
//     fits beside the contexts: 128 for heads of up to 64 (two blocks of one tile share an SM), 80 for 128 (one of two tiles).
//   * Steps of an item: first the sinks below the window, then the window, then one without keys that ends it. A step whose keys are
//     all masked is left out; one that every row of a tile sees whole skips the masking.
//   * The running maximum of a row is raised only when a step's maximum exceeds it by 2^8, so that O is read back and scaled in few steps;
//     weights are 2^7 times as large as they need be (at most 2^15, inside binary16), so that small ones last; the sums are float32.
//   * Weights of unseen keys are exactly 0, but 0 times an infinity or NaN in an unseen V row is NaN. V rows of masked keys, and of
//     those outside the item's keys, are cleared in shared memory while the weights are awaited. That leaves keys that some rows of a
//     tile see and others do not: a row that comes out not finite from finite scores is computed again by one warp over its visible
//     keys alone (a visible score of infinity or NaN makes the row NaN as it is). That takes long, and others wait for the warp
//     with bounded waits, so it happens behind the block's last item, and a block with such rows takes over no more items.
// Bound by the softmax: per 128 x 128 tile the exponentials take 1024 cycles of an SM's special-function unit and the products 512 of
// its tensor cores (heads of 64; 1024 for heads of 128), a step 1500. Measured: 8192 tokens, 32 / 8 heads of 128, window 2048: 265 to
// 290 us by the clock under the power cap (840 to 910 TFLOP/s); 4 x 4096 tokens, 16 heads of 64, no window 400 us, window 513 and ragged
// lengths 81 us (3 steps an item that ran; half of it goes into the ends of items). Rows computed
// again are far slower: one causal sequence of 40000 tokens, 2 heads of 64, all of it from token 100 on: 180 ms (0.64 ms without). Tried
// and slower: two threads a row, part of the exponentials by polynomial, scores of 96 keys twice, masks gathered by a warp of their own.
// Every wait is bounded; a block that gives up writes NaN into the rows of the items it has not finished, counts in g_window_give_ups,
// frees its tensor memory and returns.
__device__ unsigned int g_window_give_ups = 0;     // blocks, on this device

constexpr int kTileRows = 128;
constexpr int kHalfTileBytes = kTileRows * 128;    // 128 rows x 64 binary16
constexpr int kStepSlots = 8;                      // descriptors of steps in flight; more than the stages + 2
// Items of a warp with rows to compute again. The queries of item X are loaded once every warp has read the last scores of item X - 2, and
// so has noted the rows of item X - 4; the next item is asked for after that. With the first such rows in item T, none follows T + 4.
constexpr int kAgainItems = 8;

struct WindowStep {
    int item, j0;
    int columns;             // KEYS, 16 where no more keys are left, 0 at the end of an item, -1 at the end of all
    uint32_t kept[4];
    uint32_t flags;          // bit t: tile t takes part; bit 4 + t: some row of tile t does not see some key
};

template <int DP, int NQ>
struct WindowTc {
    static constexpr int KEYS = DP == 64 ? 128 : 80;         // of a step
    static constexpr int CHUNKS = KEYS / 16;                 // the softmax goes by 16 columns
    static constexpr int HALVES = DP / 64;
    static constexpr int TILE_BYTES = HALVES * kHalfTileBytes;
    static constexpr int HALF_KV = KEYS * 128, KV_BYTES = HALVES * HALF_KV;
    static constexpr int STAGES = 2, QUERIES = 2;            // tiles of K and V, and of Q, on their way or in use
    static constexpr int SOFTMAX_WARPS = 4 * NQ;
    // Softmax warps in whole groups of four, and one more group for the others (one or two of it idle), which hands most of its
    // registers to them: a row's scores stay in registers, 128 of them. Launched with 65536 / (THREADS x blocks per SM) each:
    // 128 x 256 >= 192 x 128 + 56 x 128, 168 x 384 >= 224 x 256 + 56 x 128.
    static constexpr int THREADS = 32 * (SOFTMAX_WARPS + 4);
    // The context's rows leave through the place of the item's queries by TMA, or as 16-byte stores from registers. TMA holds the queries
    // of the item after the next back until they have left: 8192 tokens, 32 heads of 128: 265 us against 277, but 4 x 4096 tokens, 16
    // heads of 64, window 513, whose items are short: 88 against 84 as the kernel was then.
    static constexpr bool ROWS_BY_TMA = NQ == 2;
    static constexpr int LAUNCH_REGS = NQ == 1 ? 128 : 168, SOFTMAX_REGS = NQ == 1 ? 192 : 224, OTHER_REGS = 56;
    static_assert(LAUNCH_REGS * THREADS >= SOFTMAX_REGS * 32 * SOFTMAX_WARPS + OTHER_REGS * 128, "a group that asks for more would wait forever");
    static constexpr int WEIGHTS = NQ * KEYS, CONTEXT = WEIGHTS + NQ * KEYS / 2;   // columns of tensor memory behind the scores
    static constexpr int TMEM_COLS = NQ == 1 ? 256 : 512;
    static constexpr int SMEM_BYTES = 1024 + QUERIES * NQ * TILE_BYTES + 2 * STAGES * KV_BYTES;   // 1024: alignment of the swizzled tiles
    static_assert(CONTEXT + NQ * DP <= TMEM_COLS, "scores, weights and contexts of all tiles");
    static_assert(STAGES + 2 < kStepSlots, "a descriptor outlives its step");
};

__device__ __forceinline__ uint64_t swizzled_desc(uint32_t saddr, uint32_t lbo_bytes) {
    // 128-byte swizzle, groups of 8 rows 1024 bytes apart, descriptor version 1
    return (uint64_t) ((saddr & 0x3ffffu) >> 4) | ((uint64_t) (lbo_bytes >> 4) << 16) | ((uint64_t) (1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
                 "l"(a), "l"(b), "r"(idesc), "r"((uint32_t) accumulate)
                 : "memory");
}

__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
                 "r"(a), "l"(b), "r"(idesc), "r"((uint32_t) accumulate)
                 : "memory");
}

__device__ __forceinline__ void mma_commit(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar)) : "memory");
}

__device__ __forceinline__ void mbar_arrive(uint64_t *bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}

// True on one lane of the warp, the same every time.
__device__ __forceinline__ bool elect_one() {
    uint32_t mine;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(mine));
    return mine != 0;
}

// A wait of a whole warp: false on every lane when any gave up.
__device__ __forceinline__ bool wait_together(uint64_t *bar, uint32_t parity) {
    return __all_sync(0xffffffffu, mbar_wait_bounded(bar, parity)) != 0;
}

__device__ __forceinline__ void tmem_load16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
          "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}

__device__ __forceinline__ void tmem_store8(uint32_t taddr, const uint32_t *r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]),
                 "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}

__device__ __forceinline__ void tmem_store16(uint32_t taddr, const uint32_t *r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
        "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

__device__ __forceinline__ void tmem_wait_loads() {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

__device__ __forceinline__ void tmem_wait_stores() {
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

__device__ __forceinline__ void tmem_fence_before() {
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}

__device__ __forceinline__ void tmem_fence_after() {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}

// The map's box of rows x 64 columns of one head into a swizzled tile; rows and columns outside the tensor arrive as zeros.
__device__ __forceinline__ void tma_tile(void *dst, const CUtensorMap *map, int column, int row, int head, int batch, uint64_t *bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(
                     smem_addr(dst)),
                 "l"(map), "r"(column), "r"(row), "r"(head), "r"(batch), "r"(smem_addr(bar))
                 : "memory");
}

// The largest of three, NaN if any is: one instruction.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// Asks for a block that has not started yet; 16 bytes of answer arrive on the barrier. Not to be asked again after a refusal.
__device__ __forceinline__ void take_block(void *answer, uint64_t *bar) {
    asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(smem_addr(answer)),
                 "r"(smem_addr(bar))
                 : "memory");
}

// The block that was taken over, or -1.
__device__ __forceinline__ int taken_block(const void *answer) {
    uint32_t got, x;
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b128 a;\n\t"
        "ld.shared.b128 a, [%2];\n\t"
        "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, a;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t"
        "mov.u32 %1, 0;\n\t"
        "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, a;\n\t}"
        : "=r"(got), "=r"(x)
        : "r"(smem_addr(answer))
        : "memory");
    return got != 0 ? (int) x : -1;
}

// A warp's 32 rows x 64 columns from a swizzled tile to the context; rows and columns outside the tensor are not written.
__device__ __forceinline__ void tma_rows(const CUtensorMap *map, const void *src, int column, int row, int head, int batch) {
    asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4, %5}], [%1];" ::"l"(map), "r"(smem_addr(src)), "r"(column),
                 "r"(row), "r"(head), "r"(batch)
                 : "memory");
}

// Zeros into the rows of a swizzled tile of V whose bits are not set (whole rows, so that the swizzle does not matter), for the MMAs
// that the warp issues next. Two warps may clear the same tile, one while the other's MMAs read it: they write what is there.
template <int KEYS, int HALVES>
__device__ __forceinline__ void clear_rows(unsigned char *tile, const uint32_t (&kept)[4], int columns) {
    const int lane = threadIdx.x & 31;
    const bool gap = lane < 4 && (range_bits(0, columns, 32 * lane) & ~kept[lane & 3]) != 0;
    if (__any_sync(0xffffffffu, gap)) {
        for (int j = lane >> 3; j < columns; j += 4) {   // eight lanes a row
            if ((kept[j >> 5] >> (j & 31) & 1u) == 0) {
#pragma unroll
                for (int x = 0; x < HALVES; ++x) {
                    *reinterpret_cast<uint4 *>(tile + x * KEYS * 128 + j * 128 + (lane & 7) * 16) = make_uint4(0, 0, 0, 0);
                }
            }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
    }
}

// One row again over its visible keys alone (rows whose tile held an infinity or NaN).
template <int DP>
__device__ __noinline__ void window_row_again(const __half *q, const __half *k, const __half *v, const int8_t *mask, __half *context,
                                              const WindowShape *s, float *s_q, int b, int i, int h) {
    window_prompt_row<__half, DP / 32>(q, k, v, mask, context, *s, s_q, b, i, h);
}

// The rows and heads of a work item.
template <int NQ>
struct WindowItem {
    int b, kh, row0, last_row, tile_row[NQ], tile_head[NQ];

    __device__ __forceinline__ WindowItem(int item, const WindowShape &s, int row_blocks, int pair_heads) {
        const int rb = row_blocks - 1 - item % row_blocks;   // last rows first: with a one-sided window they have the most keys
        const int bh = item / row_blocks, head_groups = pair_heads ? s.heads / 2 : s.heads;
        b = bh / head_groups;
        const int h0 = (bh - b * head_groups) * (pair_heads ? 2 : 1);
        const int tiles = pair_heads ? 1 : NQ;
        row0 = rb * tiles * kTileRows;
        last_row = min(row0 + tiles * kTileRows, s.seq) - 1;
        kh = h0 / (s.heads / s.kv_heads);
#pragma unroll
        for (int t = 0; t < NQ; ++t) {
            tile_row[t] = pair_heads ? row0 : row0 + t * kTileRows;
            tile_head[t] = pair_heads ? h0 + t : h0;
        }
    }
};

template <int DP, int NQ>
__global__ void __launch_bounds__(WindowTc<DP, NQ>::THREADS, NQ == 1 ? 2 : 1)
window_tc_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                 const __grid_constant__ CUtensorMap o_map, bool row_vectors, const __half *q, const __half *k, const __half *v,
                 const int8_t *mask, __half *context, const __grid_constant__ WindowShape s, int row_blocks, int pair_heads) {
    typedef WindowTc<DP, NQ> C;
    extern __shared__ unsigned char tc_raw[];
    __shared__ uint64_t s_qfull[C::QUERIES], s_qempty[C::QUERIES], s_kfull[C::STAGES], s_kempty[C::STAGES], s_vfull[C::STAGES], s_vempty[C::STAGES];
    __shared__ uint64_t s_sfull[NQ], s_sfree[NQ], s_pfull[NQ], s_ofull[NQ];   // scores written, scores read, weights written, O added to
    __shared__ __align__(16) uint4 s_taken[2];
    __shared__ uint64_t s_takes;
    __shared__ WindowTurns s_turns;
    __shared__ uint32_t s_tmem;
    __shared__ WindowStep s_steps[kStepSlots];
    __shared__ float s_row[C::SOFTMAX_WARPS][kWindowMaxDim];
    __shared__ int4 s_again[C::SOFTMAX_WARPS][kAgainItems];   // rows to compute again: sequence, first row, head, which of 32
    __shared__ int s_agains[C::SOFTMAX_WARPS];
    __shared__ volatile int s_stop;                           // no more items
    __shared__ uint32_t s_bits[32][4];   // kept keys of 32 candidate steps
    unsigned char *tiles = tc_raw + ((1024u - (smem_addr(tc_raw) & 1023u)) & 1023u);
    unsigned char *s_qt = tiles, *s_kt = tiles + C::QUERIES * NQ * C::TILE_BYTES, *s_vt = s_kt + C::STAGES * C::KV_BYTES;
    const int warp = __shfl_sync(0xffffffffu, (int) threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

    if (threadIdx.x == 64) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&q_map) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&k_map) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&v_map) : "memory");
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&s_tmem)), "r"((uint32_t) C::TMEM_COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (threadIdx.x == 32) {
        s_turns.reset();
        s_stop = 0;
        for (int w = 0; w < C::SOFTMAX_WARPS; ++w) {
            s_agains[w] = 0;
        }
        mbar_init(&s_takes, 1);
        for (int i = 0; i < C::QUERIES; ++i) {
            mbar_init(&s_qfull[i], 1);
            mbar_init(&s_qempty[i], NQ + (C::ROWS_BY_TMA ? C::SOFTMAX_WARPS : 0));   // its products are done, and it has served the rows
        }
        for (int i = 0; i < C::STAGES; ++i) {
            mbar_init(&s_kfull[i], 1);
            mbar_init(&s_kempty[i], NQ);
            mbar_init(&s_vfull[i], 1);
            mbar_init(&s_vempty[i], NQ);
        }
        for (int t = 0; t < NQ; ++t) {
            mbar_init(&s_sfull[t], 2);   // the MMAs' completion and the issuing warp, which has seen the step's descriptor
            mbar_init(&s_sfree[t], 4);
            mbar_init(&s_pfull[t], 4);
            mbar_init(&s_ofull[t], 1);
        }
        mbar_init_fence();
    }
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, s_tmem, 0);

    // Every barrier below completes one phase per step (or item), whatever the step is, so `step` and `turn`, which count through
    // all items, give their parities.
    if (warp >= C::SOFTMAX_WARPS) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::OTHER_REGS));
        if (warp == C::SOFTMAX_WARPS + NQ) {
            // ---- items, steps and loads
            bool ok = true;
            int step = 0, turn = 0;
            bool asked = true;
            for (int item = blockIdx.x; item >= 0 && ok; ++turn) {
                const WindowItem<NQ> w(item, s, row_blocks, pair_heads);
                if (lane == 0) {
                    s_turns.add(turn, item);
                }
                const int lo = w.row0 > s.before ? (w.row0 - s.before) & ~15 : 0;   // whole vectors of the mask
                const int hi = s.after < s.seq - 1 - w.last_row ? w.last_row + s.after + 1 : s.seq;
                const int sinks_end = min(s.sinks, lo), sink_steps = (sinks_end + C::KEYS - 1) / C::KEYS;
                const int steps = sink_steps + (hi - lo + C::KEYS - 1) / C::KEYS;
                const int8_t *kept = mask != nullptr ? mask + (int64_t) w.b * s.seq : nullptr;
                const int qb = turn % C::QUERIES;
                if (turn >= C::QUERIES) {
                    ok = wait_together(&s_qempty[qb], (turn / C::QUERIES - 1) & 1);
                }
                if (ok && lane == 0) {
                    mbar_arrive_expect(&s_qfull[qb], NQ * C::TILE_BYTES);
                    for (int t = 0; t < NQ; ++t) {
                        for (int x = 0; x < C::HALVES; ++x) {
                            tma_tile(s_qt + (qb * NQ + t) * C::TILE_BYTES + x * kHalfTileBytes, &q_map, 64 * x, w.tile_row[t], w.tile_head[t], w.b,
                                     &s_qfull[qb]);
                        }
                    }
                }
                // 32 candidates at a time, one per lane; then those that hold a kept key, and the item's end, one after another.
                for (int base = 0; base <= steps && ok; base += 32) {
                    // Sixteen keys a lane and load where the mask's rows allow it, else four or one: 4 x 4096 tokens, window 513, ragged
                    // lengths: 81.2 us by sixteens, 86.0 by fours.
                    if (kept != nullptr) {
                        const int candidates = min(32, steps - base);
                        const bool words = s.seq % 4 == 0 && (reinterpret_cast<uintptr_t>(mask) & 3) == 0;   // of four keys: none reaches past its row
                        const bool vectors = C::KEYS % 16 == 0 && s.seq % 16 == 0 && (reinterpret_cast<uintptr_t>(mask) & 15) == 0;   // of sixteen
                        __syncwarp();
                        if (vectors) {
                            constexpr int PER = C::KEYS / 16;   // lanes a step
                            for (int c0 = 0; c0 < candidates * PER; c0 += 64) {
                                uint4 raw[2];
                                int left[2];
#pragma unroll
                                for (int u = 0; u < 2; ++u) {
                                    const int x = c0 + 32 * u + lane, at = base + x / PER;
                                    const int j = (at < sink_steps ? at * C::KEYS : lo + (at - sink_steps) * C::KEYS) + 16 * (x % PER);
                                    left[u] = x < candidates * PER ? (at < sink_steps ? sinks_end : hi) - j : 0;
                                    raw[u] = left[u] > 0 ? *reinterpret_cast<const uint4 *>(kept + j) : make_uint4(0, 0, 0, 0);
                                }
#pragma unroll
                                for (int u = 0; u < 2; ++u) {
                                    const int x = c0 + 32 * u + lane;
                                    const uint32_t q4[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
                                    uint32_t bits = 0;
#pragma unroll
                                    for (int e = 0; e < 4; ++e) {   // any bit of a byte -> its highest; the four highest bits side by side
                                        const uint32_t v = (((q4[e] & 0x7f7f7f7fu) + 0x7f7f7f7fu) | q4[e]) & 0x80808080u;
                                        bits |= ((v >> 7) * 0x01020408u >> 24 & 15u) << (4 * e);
                                    }
                                    bits &= left[u] >= 16 ? 0xffffu : left[u] > 0 ? (1u << left[u]) - 1u : 0u;
                                    if (x < candidates * PER) {
                                        reinterpret_cast<uint16_t *>(s_bits[x / PER])[x % PER] = (uint16_t) bits;
                                    }
                                }
                            }
                        } else {
                            for (int c0 = 0; c0 < candidates; c0 += 8) {
                                uint32_t four[8];
#pragma unroll
                                for (int u = 0; u < 8; ++u) {
                                    const int at = base + c0 + u;
                                    const int j = (at < sink_steps ? at * C::KEYS : lo + (at - sink_steps) * C::KEYS) + 4 * lane;
                                    const int left = c0 + u < candidates && 4 * lane < C::KEYS ? (at < sink_steps ? sinks_end : hi) - j : 0;
                                    four[u] = 0;
                                    if (words) {
                                        four[u] = left > 0 ? *reinterpret_cast<const uint32_t *>(kept + j) & (left >= 4 ? 0xffffffffu : (1u << (8 * left)) - 1u) : 0u;
                                    } else {
#pragma unroll
                                        for (int e = 0; e < 4; ++e) {
                                            four[u] |= e < left ? (uint32_t) (uint8_t) kept[j + e] << (8 * e) : 0u;
                                        }
                                    }
                                }
#pragma unroll
                                for (int u = 0; u < 8; ++u) {
                                    // any bit of a byte -> its lowest; the four lowest bits side by side; eight lanes' to a word
                                    uint32_t v = four[u] | four[u] >> 4;
                                    v |= v >> 2;
                                    v |= v >> 1;
                                    v = ((v & 0x01010101u) * 0x01020408u >> 24 & 15u) << (4 * (lane & 7));
                                    v |= __shfl_xor_sync(0xffffffffu, v, 1);
                                    v |= __shfl_xor_sync(0xffffffffu, v, 2);
                                    v |= __shfl_xor_sync(0xffffffffu, v, 4);
                                    if ((lane & 7) == 0 && c0 + u < candidates) {
                                        s_bits[c0 + u][lane >> 3] = v;
                                    }
                                }
                            }
                        }
                        __syncwarp();
                    }
                    const int at = base + lane;
                    const bool in_sinks = at < sink_steps;
                    const int keys = at < steps ? min((in_sinks ? sinks_end : hi) - (in_sinks ? at : at - sink_steps) * C::KEYS - (in_sinks ? 0 : lo), C::KEYS) : 0;
                    WindowStep d;
                    d.item = item;
                    d.j0 = in_sinks ? at * C::KEYS : lo + (at - sink_steps) * C::KEYS;
                    d.columns = keys == 0 ? 0 : keys <= 16 ? 16 : C::KEYS;
                    d.flags = 0;
                    int count = 0;
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        d.kept[u] = keys == 0 ? 0 : kept != nullptr ? s_bits[lane][u] & range_bits(0, keys, 32 * u) : range_bits(0, keys, 32 * u);
                        count += __popc(d.kept[u]);
                    }
#pragma unroll
                    for (int t = 0; t < NQ; ++t) {
                        const int first = w.tile_row[t], last = min(first + kTileRows, s.seq) - 1;
                        const int t_lo = first > s.before ? first - s.before : 0;
                        const int t_hi = s.after < s.seq - 1 - last ? last + s.after + 1 : s.seq;
                        if (count > 0 && first < s.seq && d.j0 < t_hi && (d.j0 + keys > t_lo || d.j0 < s.sinks)) {
                            d.flags |= 1u << t;
                        }
                        const bool whole = count == d.columns && (s.after >= s.seq || d.j0 + keys - 1 <= first + s.after) &&
                                           (last - s.before <= d.j0 || d.j0 + keys <= s.sinks);
                        if (!whole) {
                            d.flags |= 16u << t;
                        }
                    }
                    unsigned todo = __ballot_sync(0xffffffffu, (d.flags & 15u) != 0 || at == steps);
                    while (todo != 0 && ok) {
                        const int from = __ffs(todo) - 1;
                        todo &= todo - 1;
                        const int j0 = __shfl_sync(0xffffffffu, d.j0, from);
                        const bool end = base + from == steps;
                        if (end) {   // the next item: not earlier, so that blocks finish together
                            asked = __all_sync(0xffffffffu, s_stop == 0) != 0;
                            if (asked && lane == 0) {
                                mbar_arrive_expect(&s_takes, 16);
                                take_block(&s_taken[turn & 1], &s_takes);
                            }
                        }
                        const int st = step % C::STAGES;
                        const uint32_t before = (step / C::STAGES - 1) & 1;
                        if (step >= C::STAGES) {
                            ok = wait_together(&s_kempty[st], before);
                        }
                        if (lane == from) {
                            s_steps[step % kStepSlots] = d;
                        }
                        __syncwarp();
                        if (ok && lane == 0) {
                            if (!end) {
                                mbar_arrive_expect(&s_kfull[st], C::KV_BYTES);
                                for (int x = 0; x < C::HALVES; ++x) {
                                    tma_tile(s_kt + st * C::KV_BYTES + x * C::HALF_KV, &k_map, 64 * x, j0, w.kh, w.b, &s_kfull[st]);
                                }
                            } else {
                                mbar_arrive(&s_kfull[st]);
                            }
                        }
                        __syncwarp();
                        if (ok && step >= C::STAGES) {
                            ok = wait_together(&s_vempty[st], before);
                        }
                        if (ok && lane == 0) {
                            if (!end) {
                                mbar_arrive_expect(&s_vfull[st], C::KV_BYTES);
                                for (int x = 0; x < C::HALVES; ++x) {
                                    tma_tile(s_vt + st * C::KV_BYTES + x * C::HALF_KV, &v_map, 64 * x, j0, w.kh, w.b, &s_vfull[st]);
                                }
                            } else {
                                mbar_arrive(&s_vfull[st]);
                            }
                        }
                        __syncwarp();
                        step += ok ? 1 : 0;
                    }
                }
                ok = ok && (!asked || wait_together(&s_takes, turn & 1));
                item = ok && asked ? taken_block(&s_taken[turn & 1]) : -1;
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // the answer is read before its place is written again
            }
            if (ok) {   // the end of all
                const int st = step % C::STAGES;
                if (step >= C::STAGES) {
                    ok = wait_together(&s_kempty[st], (step / C::STAGES - 1) & 1);
                }
                if (ok && lane == 0) {
                    s_steps[step % kStepSlots].columns = -1;
                    s_steps[step % kStepSlots].flags = 0;
                    mbar_arrive(&s_kfull[st]);
                }
                __syncwarp();
            }
            if (!ok) {   // the copies in flight land before the block's shared memory goes
                if (turn > 0 && wait_together(&s_takes, (turn - 1) & 1) && lane == 0 && taken_block(&s_taken[(turn - 1) & 1]) >= 0) {
                    s_turns.add(turn, taken_block(&s_taken[(turn - 1) & 1]));   // taken over and not begun
                }
                for (int i = max(turn - C::QUERIES, 0); i <= turn; ++i) {
                    (void) wait_together(&s_qfull[i % C::QUERIES], (i / C::QUERIES) & 1);
                }
                for (int i = max(step - C::STAGES, 0); i <= step; ++i) {
                    (void) wait_together(&s_kfull[i % C::STAGES], (i / C::STAGES) & 1);
                    (void) wait_together(&s_vfull[i % C::STAGES], (i / C::STAGES) & 1);
                }
            }
        } else if (warp < C::SOFTMAX_WARPS + NQ) {
            // ---- matrix products of a tile: the warp walks together (its addresses stay in uniform registers), one lane issues
            const int t = warp - C::SOFTMAX_WARPS;
            const uint32_t ksteps = (uint32_t) (s.dim + 15) / 16;
            const uint32_t idesc_o = (1u << 4) | (1u << 16) | ((2 * ksteps) << 17) | ((kTileRows >> 4) << 24);   // N: the dimension, in 16s
            const bool leader = elect_one();
            const uint64_t q_desc = swizzled_desc(smem_addr(s_qt + t * C::TILE_BYTES), 16), k_desc = swizzled_desc(smem_addr(s_kt), 16);
            const uint64_t v_desc = swizzled_desc(smem_addr(s_vt), C::HALF_KV);
            const uint32_t t_s = tmem + t * C::KEYS, t_p = tmem + C::WEIGHTS + t * (C::KEYS / 2), t_o = tmem + C::CONTEXT + t * DP;
            bool ok = true, started = false;   // started: O holds something of this item
            int columns_before = 0, step = 0, turn = 0;
            uint32_t flags_before = 0;
            bool new_item = true;
            uint64_t qd = 0;
            for (; ok; ++step) {
                const int st = step % C::STAGES, st_before = (step + C::STAGES - 1) % C::STAGES, qb = turn % C::QUERIES;
                ok = wait_together(&s_kfull[st], (step / C::STAGES) & 1);
                const int columns = __shfl_sync(0xffffffffu, s_steps[step % kStepSlots].columns, 0);
                const uint32_t flags = __shfl_sync(0xffffffffu, s_steps[step % kStepSlots].flags, 0) >> t;
                if (new_item && columns >= 0) {
                    ok = ok && wait_together(&s_qfull[qb], (turn / C::QUERIES) & 1);
                    qd = q_desc + (uint64_t) (qb * NQ * (C::TILE_BYTES / 16));
                    new_item = false;
                }
                if (step > 0) {
                    ok = ok && wait_together(&s_sfree[t], (step - 1) & 1);
                    tmem_fence_after();
                }
                if (ok && leader) {
                    if ((flags & 1u) != 0) {
                        const uint64_t kd = k_desc + (uint64_t) (st * (C::KV_BYTES / 16));
                        const uint32_t idesc_s = (1u << 4) | ((uint32_t) (columns / 8) << 17) | ((kTileRows >> 4) << 24);
#pragma unroll
                        for (int kk = 0; kk < DP / 16; ++kk) {
                            if (kk < (int) ksteps) {
                                mma_ss(t_s, qd + ((kk >> 2) * kHalfTileBytes + (kk & 3) * 32) / 16, kd + ((kk >> 2) * C::HALF_KV + (kk & 3) * 32) / 16,
                                       idesc_s, kk > 0);
                            }
                        }
                    }
                    mma_commit(&s_sfull[t]);
                    mbar_arrive(&s_sfull[t]);
                    if (columns >= 0) {
                        mma_commit(&s_kempty[st]);
                    }
                    if (columns == 0) {
                        mma_commit(&s_qempty[qb]);
                    }
                }
                __syncwarp();
                if (columns < 0) {
                    break;
                }
                if (step > 0) {   // O += P.V of the step before; of one that ended an item, only the wait until O has been read
                    const bool takes_part = (flags_before & 1u) != 0;
                    ok = ok && wait_together(&s_vfull[st_before], ((step - 1) / C::STAGES) & 1);
                    if (ok && takes_part && (flags_before & 16u) != 0) {
                        clear_rows<C::KEYS, C::HALVES>(s_vt + st_before * C::KV_BYTES, s_steps[(step - 1) % kStepSlots].kept, columns_before);
                    }
                    ok = ok && wait_together(&s_pfull[t], (step - 1) & 1);
                    tmem_fence_after();
                    if (ok && leader) {
                        if (takes_part) {
                            const uint64_t vd = v_desc + (uint64_t) (st_before * (C::KV_BYTES / 16));
#pragma unroll
                            for (int kk = 0; kk < C::KEYS / 16; ++kk) {
                                if (16 * kk < columns_before) {
                                    mma_ts(t_o, t_p + 8 * kk, vd + 128 * kk, idesc_o, kk > 0 || started);
                                }
                            }
                        }
                        mma_commit(&s_ofull[t]);
                        mma_commit(&s_vempty[st_before]);
                    }
                    started = columns_before != 0 && (started || takes_part);
                    __syncwarp();
                }
                columns_before = columns;
                flags_before = flags;
                if (columns == 0) {
                    new_item = true;
                    ++turn;
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::SOFTMAX_REGS));
        // ---- softmax: a row per thread
        const int t = NQ == 1 ? 0 : warp / 4;
        const uint32_t lanes = (uint32_t) (32 * (warp & 3)) << 16;
        const uint32_t t_s = tmem + t * C::KEYS + lanes, t_p = tmem + C::WEIGHTS + t * (C::KEYS / 2) + lanes, t_o = tmem + C::CONTEXT + t * DP + lanes;
        const float c = s.scale * kLog2e;
        bool ok = true;
        int step = 0;
        for (int turn = 0;; ++step, ++turn) {
            ok = wait_together(&s_sfull[t], step & 1);   // an item's first step says which it is
            if (!ok) {
                atomicMin(&s_turns.first_bad, turn);
                break;
            }
            if (s_steps[step % kStepSlots].columns < 0) {
                break;
            }
            const WindowItem<NQ> work(s_steps[step % kStepSlots].item, s, row_blocks, pair_heads);
            bool waited = true;
            const int h = work.tile_head[t], i = work.tile_row[t] + 32 * (warp & 3) + lane;
            const int lo = i > s.before ? i - s.before : 0;
            const int hi = s.after < s.seq - 1 - i ? i + s.after + 1 : s.seq;
            const int sinks_hi = min(s.sinks, hi);
            float top = -INFINITY, total = 0.f;   // top: of q.k, unscaled
            bool first = true, any = false;       // any: the row has met a key that it sees
            // One step of this row. The number of its 16-column chunks is fixed, so that its loops have no branches and the exponentials of
            // one chunk overlap the arithmetic of the next (a branch per chunk costs a third of the rate).
            auto softmax_step = [&](auto chunks, const WindowStep *d, uint32_t flags) {
                constexpr int CHUNKS = decltype(chunks)::value;
                uint32_t r[CHUNKS][16];
#pragma unroll
                for (int w = 0; w < CHUNKS; ++w) {
                    tmem_load16(t_s + 16 * w, r[w]);
                }
                if (step > 0) {   // while they arrive: the product of the step before has read its weights and added to O
                    ok = wait_together(&s_ofull[t], (step - 1) & 1);
                    tmem_fence_after();
                }
                tmem_wait_loads();
                tmem_fence_before();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&s_sfree[t]);   // the next scores may come
                }
                if ((flags & 16u) != 0) {
                    const int j0 = d->j0;
#pragma unroll
                    for (int w = 0; w < CHUNKS; w += 2) {   // 32 columns
                        const uint32_t see = d->kept[w / 2] & (range_bits(lo, hi, j0 + 16 * w) | range_bits(0, sinks_hi, j0 + 16 * w));
                        any = any || see != 0;
#pragma unroll
                        for (int e = 0; e < (w + 1 < CHUNKS ? 32 : 16); ++e) {
                            r[w + e / 16][e % 16] = (see >> e & 1u) != 0 ? r[w + e / 16][e % 16] : 0xff800000u;
                        }
                    }
                } else {
                    any = true;
                }
                float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int w = 0; w < CHUNKS; ++w) {
#pragma unroll
                    for (int e = 0; e < 16; e += 2) {
                        m[e / 2 % 4] = max3_nan(m[e / 2 % 4], __uint_as_float(r[w][e]), __uint_as_float(r[w][e + 1]));
                    }
                }
                const float here = max3_nan(max3_nan(m[0], m[1], m[2]), m[3], m[3]);
                if (!(here < INFINITY)) {
                    total = NAN;   // an infinite score or a NaN: the row is NaN as it is
                }
                const bool raise = (here - top) * c > kRaiseBy;   // the first visible key: infinity > 8
                float shrink = 1.f;
                if (raise) {
                    shrink = fast_exp2((top - here) * c);
                    top = here;
                }
                const float2 c2 = splat2(c), nt2 = splat2(top == -INFINITY ? 0.f : fmaf(-top, c, kWeightScale));
                float2 sum0 = make_float2(0.f, 0.f), sum1 = make_float2(0.f, 0.f);
#pragma unroll
                for (int w = 0; w < CHUNKS; ++w) {
                    uint32_t p[8];
#pragma unroll
                    for (int e = 0; e < 16; e += 4) {
                        float2 a = fma2(make_float2(__uint_as_float(r[w][e]), __uint_as_float(r[w][e + 1])), c2, nt2);
                        float2 z = fma2(make_float2(__uint_as_float(r[w][e + 2]), __uint_as_float(r[w][e + 3])), c2, nt2);
                        a = make_float2(fast_exp2(a.x), fast_exp2(a.y));
                        z = make_float2(fast_exp2(z.x), fast_exp2(z.y));
                        sum0 = add2(sum0, a);
                        sum1 = add2(sum1, z);
                        const __half2 pa = __float22half2_rn(a), pz = __float22half2_rn(z);
                        p[e / 2] = *reinterpret_cast<const uint32_t *>(&pa);
                        p[e / 2 + 1] = *reinterpret_cast<const uint32_t *>(&pz);
                    }
                    tmem_store8(t_p + 8 * w, p);
                }
                sum0 = add2(sum0, sum1);
                total = fmaf(total, shrink, sum0.x + sum0.y);
                if (!first && __any_sync(0xffffffffu, raise)) {
                    const float2 sh2 = splat2(shrink);
                    for (int x = 0; x < s.dim; x += 16) {
                        uint32_t o[16];
                        tmem_load16(t_o + x, o);
                        tmem_wait_loads();
#pragma unroll
                        for (int e = 0; e < 16; e += 2) {
                            const float2 v2 = mul2(make_float2(__uint_as_float(o[e]), __uint_as_float(o[e + 1])), sh2);
                            o[e] = __float_as_uint(v2.x);
                            o[e + 1] = __float_as_uint(v2.y);
                        }
                        tmem_store16(t_o + x, o);
                    }
                }
                first = false;
                tmem_wait_stores();
            };
            for (; ok; ++step) {
                ok = waited || wait_together(&s_sfull[t], step & 1);
                waited = false;
                tmem_fence_after();
                const WindowStep *d = &s_steps[step % kStepSlots];
                const int columns = d->columns;
                const uint32_t flags = d->flags >> t;
                if (ok && (flags & 1u) != 0) {
                    if (columns == C::KEYS) {
                        softmax_step(std::integral_constant<int, C::CHUNKS>(), d, flags);
                    } else {
                        softmax_step(std::integral_constant<int, 1>(), d, flags);
                    }
                } else {
                    if (step > 0) {
                        ok = ok && wait_together(&s_ofull[t], (step - 1) & 1);
                        tmem_fence_after();
                    }
                    if (!ok || columns == 0) {
                        break;
                    }
                    if (lane == 0) {
                        mbar_arrive(&s_sfree[t]);
                    }
                }
                tmem_fence_before();
                __syncwarp();
                if (lane == 0 && ok) {
                    mbar_arrive(&s_pfull[t]);
                }
            }
            // ---- context rows (the last completion waited for covers every product into O)
            if (!ok) {
                atomicMin(&s_turns.first_bad, turn);
                break;
            }
            if (any && total == 0.f) {
                total = NAN;   // nothing but scores of minus infinity: 0 / 0
            }
            const float inv = total == 0.f ? 0.f : 1.f / total;
            float most = 0.f;
            __half *out = context + ((int64_t) work.b * s.seq + i) * s.context_stride + (int64_t) h * s.dim;
            unsigned char *q_tile = s_qt + ((turn % C::QUERIES) * NQ + t) * C::TILE_BYTES;
            uint32_t o[DP / 16][16];
#pragma unroll
            for (int x = 0; x < DP / 16; ++x) {
                if (!first && 16 * x < s.dim) {
                    tmem_load16(t_o + 16 * x, o[x]);
                } else {   // no step took part
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        o[x][e] = 0;
                    }
                }
            }
            tmem_wait_loads();
            tmem_fence_before();
            __syncwarp();
            if (lane == 0) {   // O and the scores' place are free for the next item
                mbar_arrive(&s_sfree[t]);
                mbar_arrive(&s_pfull[t]);
            }
            const float2 inv2 = splat2(inv);
#pragma unroll
            for (int x = 0; x < DP / 8; ++x) {
                if (8 * x < s.dim) {   // past the dimension V is zeros up to a whole 16 columns, and O too
                    uint32_t w[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int at = 8 * (x & 1) + 2 * e;
                        const float2 a = mul2(make_float2(__uint_as_float(o[x / 2][at]), __uint_as_float(o[x / 2][at + 1])), inv2);
                        most = max3_nan(most, fabsf(a.x), fabsf(a.y));
                        const __half2 hv = __float22half2_rn(a);
                        w[e] = *reinterpret_cast<const uint32_t *>(&hv);
                    }
                    if (C::ROWS_BY_TMA && row_vectors) {   // into the place of this item's queries, which no product reads any more
                        const int r = 32 * (warp & 3) + lane;
                        *reinterpret_cast<uint4 *>(q_tile + (x / 8) * kHalfTileBytes + r * 128 + ((x % 8) ^ (r & 7)) * 16) = make_uint4(w[0], w[1], w[2], w[3]);
                    } else if (i < s.seq && row_vectors) {
                        *reinterpret_cast<uint4 *>(out + 8 * x) = make_uint4(w[0], w[1], w[2], w[3]);
                    } else if (i < s.seq) {
                        const __half *hw = reinterpret_cast<const __half *>(w);
#pragma unroll
                        for (int u = 0; u < 8; ++u) {
                            out[8 * x + u] = hw[u];
                        }
                    }
                }
            }
            if (C::ROWS_BY_TMA) {
                const int first_row = work.tile_row[t] + 32 * (warp & 3);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) {
                    if (row_vectors && first_row < s.seq) {
                        for (int x = 0; 64 * x < s.dim; ++x) {
                            tma_rows(&o_map, q_tile + x * kHalfTileBytes + 32 * (warp & 3) * 128, 64 * x, first_row, h, work.b);
                        }
                        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                        asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                    }
                    mbar_arrive(&s_qempty[turn % C::QUERIES]);
                }
                __syncwarp();
            }
            const unsigned bad = __ballot_sync(0xffffffffu, i < s.seq && total == total && !(most <= 65504.f));
            if (bad != 0 && lane == 0) {
                const int n = s_agains[warp];
                s_again[warp][n % kAgainItems] = make_int4(work.b, i, h, (int) bad);
                s_agains[warp] = n + 1;
                s_stop = 1;
            }
            __syncwarp();
        }
        if (s_agains[warp] > 0) {
            if (C::ROWS_BY_TMA && lane == 0) {   // the rows sent have to be there before they are written again
                asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
            }
            __syncwarp();
            for (int n = 0; n < s_agains[warp]; ++n) {
                const int4 rows = s_again[warp][n % kAgainItems];
                for (unsigned bad = (unsigned) rows.w; bad != 0; bad &= bad - 1) {
                    window_row_again<DP>(q, k, v, mask, context, &s, s_row[warp], rows.x, rows.y + __ffs(bad) - 1, rows.z);
                }
            }
        }
    }
    tmem_fence_before();
    __syncthreads();
    if (threadIdx.x == 0 && s_turns.first_bad != kNoTurn) {
        atomicAdd(&g_window_give_ups, 1u);
    }
    for (int turn = s_turns.first_bad; turn < s_turns.known; ++turn) {   // after a give-up only
        const WindowItem<NQ> w(s_turns.item(turn), s, row_blocks, pair_heads);
        for (int e = threadIdx.x; e < NQ * kTileRows * s.dim; e += C::THREADS) {
            const int t = e / (kTileRows * s.dim), r = e / s.dim % kTileRows, i = w.tile_row[t] + r;
            if (i < s.seq) {
                context[((int64_t) w.b * s.seq + i) * s.context_stride + (int64_t) w.tile_head[t] * s.dim + e % s.dim] = __float2half_rn(NAN);
            }
        }
    }
    if (warp == 0) {
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t) C::TMEM_COLS) : "memory");
    }
}

typedef CUresult (*EncodeTiled)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                                const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// cuTensorMapEncodeTiled, looked up once (the library links the runtime only); null where the driver has none.
inline EncodeTiled encode_tiled() {
    static const EncodeTiled fn = [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &found) != cudaSuccess ||
            found != cudaDriverEntryPointSuccess) {
            (void) cudaGetLastError();
            p = nullptr;
        }
        return (EncodeTiled) p;
    }();
    return fn;
}

// [batch, heads, seq, dim] view of rows `stride` elements apart, read in boxes of `rows` rows x 64 columns.
inline bool window_map(CUtensorMap *map, const __half *p, int dim, int seq, int heads, int batch, int64_t stride, int rows) {
    const EncodeTiled encode = encode_tiled();
    const cuuint64_t dims[4] = {(cuuint64_t) dim, (cuuint64_t) seq, (cuuint64_t) heads, (cuuint64_t) batch};
    const cuuint64_t strides[3] = {(cuuint64_t) stride * 2, (cuuint64_t) dim * 2, (cuuint64_t) seq * (cuuint64_t) stride * 2};
    const cuuint32_t box[4] = {64, (cuuint32_t) rows, 1, 1}, step[4] = {1, 1, 1, 1};
    if (encode == nullptr || !aligned16(p) || strides[0] % 16 != 0 || strides[1] % 16 != 0 || strides[0] >= (1ull << 40) || strides[2] >= (1ull << 40)) {
        return false;
    }
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<__half *>(p), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int DP, int NQ>
int window_tc_launch(const CUtensorMap &qm, const CUtensorMap &km, const CUtensorMap &vm, const CUtensorMap &om, bool row_vectors, const __half *q, const __half *k, const __half *v,
                     const int8_t *mask, __half *context, const WindowShape &s, cudaStream_t stream) {
    typedef WindowTc<DP, NQ> C;
    static std::atomic<uint64_t> prepared{0};   // devices on which the kernel may use its shared memory
    int dev = 0;
    cudaError_t err = cudaGetDevice(&dev);
    if (err == cudaSuccess && (dev >= 64 || ((prepared.load(std::memory_order_acquire) >> dev) & 1ull) == 0)) {
        cudaFuncAttributes attr;
        err = cudaFuncGetAttributes(&attr, window_tc_kernel<DP, NQ>);
        if (err == cudaSuccess && attr.numRegs < C::LAUNCH_REGS) {
            err = cudaErrorInvalidKernelImage;   // compiled to fewer registers than its groups of warps share out among themselves: a broken build
        }
        if (err == cudaSuccess) {
            err = cudaFuncSetAttribute(window_tc_kernel<DP, NQ>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM_BYTES);
        }
        if (err == cudaSuccess && dev < 64) {
            prepared.fetch_or(1ull << dev, std::memory_order_release);
        }
    }
    if (err != cudaSuccess) {
        set_last_error(err);
        return CUBK_ERR_LAUNCH;
    }
    const int pair = NQ == 2 && (s.heads / s.kv_heads) % 2 == 0 ? 1 : 0;
    const int rows = pair ? kTileRows : NQ * kTileRows;
    const int row_blocks = (s.seq + rows - 1) / rows;
    const int64_t items = (int64_t) row_blocks * s.batch * (pair ? s.heads / 2 : s.heads);
    if (items > 0x7fffffffLL) {
        return CUBK_ERR_UNSUPPORTED;
    }
    window_tc_kernel<DP, NQ><<<(unsigned) items, C::THREADS, C::SMEM_BYTES, stream>>>(qm, km, vm, om, row_vectors, q, k, v, mask, context, s, row_blocks, pair);
    return check_launch();
}

// Binary16 on the tensor cores; CUBK_ERR_UNSUPPORTED where TMA cannot read the operands (rows or heads that do not start on
// 16-byte boundaries), the head dimension is above 128 or the scale is not positive (a row's largest score is then not its
// largest product): the caller takes another kernel.
inline int window_tc(const __half *q, const __half *k, const __half *v, const int8_t *mask, __half *context, const WindowShape &s,
                     cudaStream_t stream) {
    CUtensorMap qm, km, vm, om;
    const int keys = s.dim <= 64 ? WindowTc<64, 1>::KEYS : WindowTc<128, 2>::KEYS;
    if (s.dim > 128 || !(s.scale > 0.f) || !window_map(&qm, q, s.dim, s.seq, s.heads, s.batch, s.q_stride, kTileRows) ||
        !window_map(&km, k, s.dim, s.seq, s.kv_heads, s.batch, s.kv_stride, keys) ||
        !window_map(&vm, v, s.dim, s.seq, s.kv_heads, s.batch, s.kv_stride, keys)) {
        return CUBK_ERR_UNSUPPORTED;
    }
    // a context whose rows or heads do not start on 16-byte boundaries is written element by element
    const bool row_vectors = window_map(&om, context, s.dim, s.seq, s.heads, s.batch, s.context_stride, 32);
    if (!row_vectors) {
        om = qm;
    }
    return s.dim <= 64 ? window_tc_launch<64, 1>(qm, km, vm, om, row_vectors, q, k, v, mask, context, s, stream)
                       : window_tc_launch<128, 2>(qm, km, vm, om, row_vectors, q, k, v, mask, context, s, stream);
}

template <typename T>
int window_attention(const T *q, const T *k, const T *v, int64_t q_stride, int64_t kv_stride, const int8_t *mask, int batch, int seq,
                     int heads, int kv_heads, int dim, int before, int after, int sinks, float scale, T *context, int64_t context_stride,
                     cudaStream_t stream) {
    if (q == nullptr || k == nullptr || v == nullptr || context == nullptr || batch < 0 || seq < 0 || heads <= 0 || kv_heads <= 0 || dim <= 0 ||
        before < 0 || after < 0 || sinks < 0 || heads % kv_heads != 0 || q_stride < (int64_t) heads * dim ||
        kv_stride < (int64_t) kv_heads * dim || context_stride < (int64_t) heads * dim) {
        return CUBK_ERR_INVALID_ARG;
    }
    if (dim > kWindowMaxDim || seq > 0x3fffffff) {
        return CUBK_ERR_UNSUPPORTED;
    }
    if (batch == 0 || seq == 0) {
        return CUBK_OK;
    }
    const WindowShape s = {batch, seq, heads, kv_heads, dim, before, after, sinks, scale, q_stride, kv_stride, context_stride};
    // A tile of rows takes as long for one token as for 64 or 128; a warp per row is faster for a few. 12 heads of 64, float32: 1 x 8
    // tokens 4.8 us against 10.3 in tiles, 1024 x 16 328 against 363, but 1024 x 24 628 against 382. Binary16: 1 x 4 4.2 against 6.4,
    // 1024 x 8 96 against 124, but 1024 x 12 162 against 124.
    if (seq > (sizeof(T) == 2 ? 8 : 16)) {
        if constexpr (sizeof(T) == 2) {
            const int rc = window_tc(q, k, v, mask, context, s, stream);
            if (rc != CUBK_ERR_UNSUPPORTED) {
                return rc;
            }
        }
        const int rc = window_plain(q, k, v, mask, context, s, stream);
        if (rc != CUBK_ERR_UNSUPPORTED) {
            return rc;
        }
    }
    const int64_t groups = ((int64_t) batch * seq * heads + kWindowRowWarps - 1) / kWindowRowWarps;
    const unsigned blocks = (unsigned) (groups < 148 * 64 ? groups : 148 * 64);
    const auto kernel = dim <= 64 ? window_rows_kernel<T, 2> : dim <= 128 ? window_rows_kernel<T, 4> : window_rows_kernel<T, 8>;
    kernel<<<blocks, 32 * kWindowRowWarps, 0, stream>>>(q, k, v, mask, context, s);
    return check_launch();
}

}  // namespace cubk

extern "C" {

int cubk_window_give_ups(unsigned int *count) {
    if (count == nullptr) {
        return CUBK_ERR_INVALID_ARG;
    }
    const cudaError_t err = cudaMemcpyFromSymbol(count, cubk::g_window_give_ups, sizeof(unsigned int));
    if (err != cudaSuccess) {
        cubk::set_last_error(err);
        return CUBK_ERR_LAUNCH;
    }
    return CUBK_OK;
}

int cubk_window_attention_f32(const float *q, const float *k, const float *v, int64_t q_stride, int64_t kv_stride, const int8_t *mask,
                              int batch, int seq, int heads, int kv_heads, int head_dim, int before, int after, int sinks, float scale,
                              float *context, int64_t context_stride, void *stream) {
    return cubk::window_attention<float>(q, k, v, q_stride, kv_stride, mask, batch, seq, heads, kv_heads, head_dim, before, after, sinks,
                                         scale, context, context_stride, (cudaStream_t) stream);
}

int cubk_window_attention_f16(const void *q, const void *k, const void *v, int64_t q_stride, int64_t kv_stride, const int8_t *mask,
                              int batch, int seq, int heads, int kv_heads, int head_dim, int before, int after, int sinks, float scale,
                              void *context, int64_t context_stride, void *stream) {
    return cubk::window_attention<__half>((const __half *) q, (const __half *) k, (const __half *) v, q_stride, kv_stride, mask, batch, seq,
                                          heads, kv_heads, head_dim, before, after, sinks, scale, (__half *) context, context_stride,
                                          (cudaStream_t) stream);
}

}  // extern "C"
