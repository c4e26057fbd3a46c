// K8: attention with a sliding window and first tokens that stay visible (sinks).
//
// Whole sequences: query i sees key j when the key is kept, j <= i + after, and j >= i - before or j < sinks.
// Single tokens: keys and values live in a ring of sinks + window slots per stream; the slot of position p is p
// below sinks and sinks + (p - sinks) % window from there on, so the slots that hold anything are the first
// min(p + 1, sinks + window) and every one of them is visible to p.
// Softmax statistics and all sums are float32. A key that a query does not see contributes nothing at all, whatever
// bits its rows hold; a query that sees no key gets zeros.
#include "common.cuh"

namespace cubk {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kWindowMaxDim = 256;
constexpr int kWindowRowWarps = 4;

// ---------------------------------------------------------------- one query row per warp
// Any head dimension up to 256, any strides: 32 keys at a time, a key per lane for the scores, a column (or several)
// per lane for the context. `key(j)` and `value(j)` give the addresses of row j, `seen(j)` says whether it counts.
template <typename T, typename Key, typename Value, typename Seen>
__device__ void window_row(const T *q, float *s_q, int dim, float scale, int sinks_end, int lo, int hi, Key key, Value value, Seen seen,
                           T *context) {
    const int lane = threadIdx.x & 31;
    __syncwarp();
    for (int c = lane; c < dim; c += 32) {
        s_q[c] = to_float<T>(q[c]);
    }
    __syncwarp();
    float o[kWindowMaxDim / 32];
#pragma unroll
    for (int i = 0; i < kWindowMaxDim / 32; ++i) {
        o[i] = 0.f;
    }
    float top = -INFINITY, total = 0.f;
    for (int part = 0; part < 2; ++part) {
        const int begin = part == 0 ? 0 : lo, end = part == 0 ? sinks_end : hi;
        for (int j0 = begin; j0 < end; j0 += 32) {
            const int j = j0 + lane;
            const bool use = j < end && seen(j);
            float s = -INFINITY;
            if (use) {
                const T *kr = key(j);
                float a0 = 0.f, a1 = 0.f;
                int c = 0;
                for (; c + 1 < dim; c += 2) {
                    a0 = fmaf(s_q[c], to_float<T>(kr[c]), a0);
                    a1 = fmaf(s_q[c + 1], to_float<T>(kr[c + 1]), a1);
                }
                if (c < dim) {
                    a0 = fmaf(s_q[c], to_float<T>(kr[c]), a0);
                }
                s = scale * kLog2e * (a0 + a1);
            }
            unsigned visible = __ballot_sync(0xffffffffu, use);
            const float next = fmaxf(top, group_max<32>(s));
            if (visible == 0 || next == -INFINITY) {
                if (!__any_sync(0xffffffffu, use && !(s == -INFINITY))) {   // a NaN score goes on below
                    continue;
                }
            }
            const float shrink = top == -INFINITY ? 0.f : fast_exp2(top - next);
            const float p = use ? fast_exp2(s - next) : 0.f;
            top = next;
            total = total * shrink + group_sum<32>(p);
#pragma unroll
            for (int i = 0; i < kWindowMaxDim / 32; ++i) {
                o[i] *= shrink;
            }
            while (visible != 0) {
                const int from = __ffs(visible) - 1;
                visible &= visible - 1;
                const float w = __shfl_sync(0xffffffffu, p, from);
                const T *vr = value(j0 + from);
#pragma unroll
                for (int i = 0; i < kWindowMaxDim / 32; ++i) {
                    if (lane + 32 * i < dim) {
                        o[i] = fmaf(w, to_float<T>(vr[lane + 32 * i]), o[i]);
                    }
                }
            }
        }
    }
    const float inv = total == 0.f ? 0.f : 1.f / total;
#pragma unroll
    for (int i = 0; i < kWindowMaxDim / 32; ++i) {
        if (lane + 32 * i < dim) {
            context[lane + 32 * i] = from_float<T>(o[i] * inv);
        }
    }
}

struct WindowShape {
    int batch, seq, heads, kv_heads, dim;
    int before, after, sinks;
    float scale;
    int64_t q_stride, kv_stride, context_stride;
};

// Row (b, i) of head h of a whole sequence.
template <typename T>
__device__ __forceinline__ void window_prompt_row(const T *q, const T *k, const T *v, const int8_t *mask, T *context, const WindowShape &s,
                                                  float *s_q, int b, int i, int h) {
    const int64_t first = (int64_t) b * s.seq;
    const int kh = h / (s.heads / s.kv_heads);
    const int8_t *kept = mask != nullptr ? mask + first : nullptr;
    const T *kb = k + first * s.kv_stride + (int64_t) kh * s.dim, *vb = v + first * s.kv_stride + (int64_t) kh * s.dim;
    const int lo = i > s.before ? i - s.before : 0;
    const int hi = s.after < s.seq - 1 - i ? i + s.after + 1 : s.seq;
    window_row<T>(q + (first + i) * s.q_stride + (int64_t) h * s.dim, s_q, s.dim, s.scale, min(min(s.sinks, lo), hi), lo, hi,
                  [&](int j) { return kb + j * s.kv_stride; }, [&](int j) { return vb + j * s.kv_stride; },
                  [&](int j) { return kept == nullptr || kept[j] != 0; }, context + (first + i) * s.context_stride + (int64_t) h * s.dim);
}

template <typename T>
__global__ void __launch_bounds__(32 * kWindowRowWarps)
window_rows_kernel(const T *q, const T *k, const T *v, const int8_t *mask, T *context, WindowShape s) {
    __shared__ float s_q[kWindowRowWarps][kWindowMaxDim];
    const int warp = threadIdx.x >> 5;
    const int64_t total = (int64_t) s.batch * s.seq * s.heads;
    for (int64_t r = (int64_t) blockIdx.x * kWindowRowWarps + warp; r < total; r += (int64_t) gridDim.x * kWindowRowWarps) {
        const int64_t bh = r / s.seq;
        window_prompt_row<T>(q, k, v, mask, context, s, s_q[warp], (int) (bh / s.heads), (int) (r - bh * s.seq), (int) (bh % s.heads));
    }
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
    const int64_t groups = ((int64_t) batch * seq * heads + kWindowRowWarps - 1) / kWindowRowWarps;
    const unsigned blocks = (unsigned) (groups < 148 * 64 ? groups : 148 * 64);
    window_rows_kernel<T><<<blocks, 32 * kWindowRowWarps, 0, stream>>>(q, k, v, mask, context, s);
    return check_launch();
}

// ---------------------------------------------------------------- ring caches
struct RingShape {
    int batch, heads, kv_heads, dim;
    int window, sinks;
    float scale;
    int64_t q_stride, kv_stride, context_stride;
};

__device__ __forceinline__ int ring_slot(int p, int window, int sinks) {
    return p < sinks ? p : sinks + (p - sinks) % window;
}

// One (stream, head) per warp. The new token's key and value are read where they came from, never from the slot that the
// warp of the group's first head writes.
template <typename T>
__global__ void __launch_bounds__(32 * kWindowRowWarps)
window_step_rows_kernel(const T *q, const T *k, const T *v, const int32_t *positions, T *k_cache, T *v_cache, T *context, RingShape s) {
    __shared__ float s_q[kWindowRowWarps][kWindowMaxDim];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t total = (int64_t) s.batch * s.heads;
    const int slots = s.window + s.sinks, share = s.heads / s.kv_heads;
    for (int64_t r = (int64_t) blockIdx.x * kWindowRowWarps + warp; r < total; r += (int64_t) gridDim.x * kWindowRowWarps) {
        const int64_t b = r / s.heads;
        const int h = (int) (r - b * s.heads), kh = h / share;
        const int p = positions[b];
        if (p < 0) {
            continue;
        }
        const int slot = ring_slot(p, s.window, s.sinks);
        const int n = p < slots ? p + 1 : slots;
        const T *kn = k + b * s.kv_stride + (int64_t) kh * s.dim, *vn = v + b * s.kv_stride + (int64_t) kh * s.dim;
        T *kc = k_cache + (b * s.kv_heads + kh) * slots * s.dim, *vc = v_cache + (b * s.kv_heads + kh) * slots * s.dim;
        if (h == kh * share) {
            for (int c = lane; c < s.dim; c += 32) {
                kc[(int64_t) slot * s.dim + c] = kn[c];
                vc[(int64_t) slot * s.dim + c] = vn[c];
            }
        }
        window_row<T>(q + b * s.q_stride + (int64_t) h * s.dim, s_q[warp], s.dim, s.scale, 0, 0, n,
                      [&](int j) { return j == slot ? kn : kc + (int64_t) j * s.dim; },
                      [&](int j) { return j == slot ? vn : vc + (int64_t) j * s.dim; }, [&](int) { return true; },
                      context + b * s.context_stride + (int64_t) h * s.dim);
    }
}

template <typename T>
int window_attention_step(const T *q, const T *k, const T *v, int64_t q_stride, int64_t kv_stride, const int32_t *positions, int batch,
                          int heads, int kv_heads, int dim, int window, int sinks, float scale, T *k_cache, T *v_cache, T *context,
                          int64_t context_stride, cudaStream_t stream) {
    if (q == nullptr || k == nullptr || v == nullptr || positions == nullptr || k_cache == nullptr || v_cache == nullptr ||
        context == nullptr || batch < 0 || heads <= 0 || kv_heads <= 0 || dim <= 0 || window <= 0 || sinks < 0 || heads % kv_heads != 0 ||
        q_stride < (int64_t) heads * dim || kv_stride < (int64_t) kv_heads * dim || context_stride < (int64_t) heads * dim) {
        return CUBK_ERR_INVALID_ARG;
    }
    if (dim > kWindowMaxDim || window > 0x3fffffff || sinks > 0x3fffffff) {
        return CUBK_ERR_UNSUPPORTED;
    }
    if (batch == 0) {
        return CUBK_OK;
    }
    const RingShape s = {batch, heads, kv_heads, dim, window, sinks, scale, q_stride, kv_stride, context_stride};
    const int64_t groups = ((int64_t) batch * heads + kWindowRowWarps - 1) / kWindowRowWarps;
    const unsigned blocks = (unsigned) (groups < 148 * 64 ? groups : 148 * 64);
    window_step_rows_kernel<T><<<blocks, 32 * kWindowRowWarps, 0, stream>>>(q, k, v, positions, k_cache, v_cache, context, s);
    return check_launch();
}

// Keys and values of a prompt's last tokens (and its sinks) into the ring: one warp per (token, kv head). Of the tokens that
// share a slot only the last is written, so no two warps write the same row.
template <typename T>
__global__ void __launch_bounds__(256)
window_cache_fill_kernel(const T *k, const T *v, int64_t kv_stride, const int32_t *lengths, int batch, int seq, int kv_heads, int dim,
                         int window, int sinks, T *k_cache, T *v_cache) {
    const int lane = threadIdx.x & 31;
    const int slots = window + sinks;
    const int64_t total = (int64_t) batch * seq * kv_heads;
    for (int64_t r = (int64_t) blockIdx.x * 8 + (threadIdx.x >> 5); r < total; r += (int64_t) gridDim.x * 8) {
        const int64_t token = r / kv_heads;
        const int kh = (int) (r - token * kv_heads);
        const int64_t b = token / seq;
        const int j = (int) (token - b * seq);
        const int length = lengths != nullptr ? min(lengths[b], seq) : seq;
        if (j >= length || (j >= sinks && j < length - window)) {
            continue;
        }
        const int64_t to = ((b * kv_heads + kh) * slots + ring_slot(j, window, sinks)) * dim, from = token * kv_stride + (int64_t) kh * dim;
        for (int c = lane; c < dim; c += 32) {
            k_cache[to + c] = k[from + c];
            v_cache[to + c] = v[from + c];
        }
    }
}

template <typename T>
int window_cache_fill(const T *k, const T *v, int64_t kv_stride, const int32_t *lengths, int batch, int seq, int kv_heads, int dim,
                      int window, int sinks, T *k_cache, T *v_cache, cudaStream_t stream) {
    if (k == nullptr || v == nullptr || k_cache == nullptr || v_cache == nullptr || batch < 0 || seq < 0 || kv_heads <= 0 || dim <= 0 ||
        window <= 0 || sinks < 0 || kv_stride < (int64_t) kv_heads * dim) {
        return CUBK_ERR_INVALID_ARG;
    }
    if (dim > kWindowMaxDim || window > 0x3fffffff || sinks > 0x3fffffff) {
        return CUBK_ERR_UNSUPPORTED;
    }
    if (batch == 0 || seq == 0) {
        return CUBK_OK;
    }
    const int64_t groups = ((int64_t) batch * seq * kv_heads + 7) / 8;
    const unsigned blocks = (unsigned) (groups < 148 * 32 ? groups : 148 * 32);
    window_cache_fill_kernel<T><<<blocks, 256, 0, stream>>>(k, v, kv_stride, lengths, batch, seq, kv_heads, dim, window, sinks, k_cache,
                                                            v_cache);
    return check_launch();
}

}  // namespace cubk

extern "C" {

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

int cubk_window_attention_step_f32(const float *q, const float *k, const float *v, int64_t q_stride, int64_t kv_stride,
                                   const int32_t *positions, int batch, int heads, int kv_heads, int head_dim, int window, int sinks,
                                   float scale, float *k_cache, float *v_cache, float *context, int64_t context_stride, void *stream) {
    return cubk::window_attention_step<float>(q, k, v, q_stride, kv_stride, positions, batch, heads, kv_heads, head_dim, window, sinks,
                                              scale, k_cache, v_cache, context, context_stride, (cudaStream_t) stream);
}

int cubk_window_attention_step_f16(const void *q, const void *k, const void *v, int64_t q_stride, int64_t kv_stride,
                                   const int32_t *positions, int batch, int heads, int kv_heads, int head_dim, int window, int sinks,
                                   float scale, void *k_cache, void *v_cache, void *context, int64_t context_stride, void *stream) {
    return cubk::window_attention_step<__half>((const __half *) q, (const __half *) k, (const __half *) v, q_stride, kv_stride, positions,
                                               batch, heads, kv_heads, head_dim, window, sinks, scale, (__half *) k_cache,
                                               (__half *) v_cache, (__half *) context, context_stride, (cudaStream_t) stream);
}

int cubk_window_cache_fill_f32(const float *k, const float *v, int64_t kv_stride, const int32_t *lengths, int batch, int seq, int kv_heads,
                               int head_dim, int window, int sinks, float *k_cache, float *v_cache, void *stream) {
    return cubk::window_cache_fill<float>(k, v, kv_stride, lengths, batch, seq, kv_heads, head_dim, window, sinks, k_cache, v_cache,
                                          (cudaStream_t) stream);
}

int cubk_window_cache_fill_f16(const void *k, const void *v, int64_t kv_stride, const int32_t *lengths, int batch, int seq, int kv_heads,
                               int head_dim, int window, int sinks, void *k_cache, void *v_cache, void *stream) {
    return cubk::window_cache_fill<__half>((const __half *) k, (const __half *) v, kv_stride, lengths, batch, seq, kv_heads, head_dim,
                                           window, sinks, (__half *) k_cache, (__half *) v_cache, (cudaStream_t) stream);
}

}  // extern "C"
