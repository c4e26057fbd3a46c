// One query row of windowed attention per warp: what every shape and alignment falls back to, and what computes rows again
// that came out not finite.
#pragma once

#include "common.cuh"

namespace cubk {

constexpr float kLog2e = 1.4426950408889634f;
// Weights of binary16 products are 2^kWeightScale times what they are relative to the running maximum, and that is raised when a
// weight passes 2^kRaiseBy of it: at most 2^15, and what is smaller than 2^-32 of the largest is lost instead of 2^-25 (40000 keys of
// 2^-25.5 beside one key make 2^-10 of a row). The scale cancels in the division by the sum.
constexpr float kWeightScale = 7.f, kRaiseBy = 8.f;
constexpr int kWindowMaxDim = 256;
constexpr int kWindowRowWarps = 4;

// Head dimensions up to 32 COLS, any strides: 32 keys at a time, a key per lane for the scores, COLS columns
// per lane for the context. The values of four keys are loaded as they are stored and converted together afterwards, over a number of
// columns that the compiler knows: 1024 x 6 binary16 tokens of 12 heads of 64 take 70 us (with eight columns a lane for every dimension,
// converted one by one, 111 to 116). Bound by latency: each warp waits for its 32 key rows and then eight times for four value rows.
// `key(j)` and `value(j)` give the addresses of row j, `seen(j)` says whether it counts.
template <typename T, int COLS, typename Key, typename Value, typename Seen>
__device__ void window_row(const T *q, float *s_q, int dim, float scale, int sinks_end, int lo, int hi, Key key, Value value, Seen seen,
                           T *context) {
    const int lane = threadIdx.x & 31;
    __syncwarp();
    for (int c = lane; c < dim; c += 32) {
        s_q[c] = to_float<T>(q[c]);
    }
    __syncwarp();
    float o[COLS];
#pragma unroll
    for (int i = 0; i < COLS; ++i) {
        o[i] = 0.f;
    }
    float top = -INFINITY, total = 0.f;
    bool any = false;
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
                if ((reinterpret_cast<uintptr_t>(kr) & 15u) == 0) {
                    constexpr int E = 16 / (int) sizeof(T);
#pragma unroll 4
                    for (; c + E <= dim; c += E) {
                        const uint4 raw = *reinterpret_cast<const uint4 *>(kr + c);
                        const T *e = reinterpret_cast<const T *>(&raw);
#pragma unroll
                        for (int x = 0; x < E; x += 2) {
                            a0 = fmaf(s_q[c + x], to_float<T>(e[x]), a0);
                            a1 = fmaf(s_q[c + x + 1], to_float<T>(e[x + 1]), a1);
                        }
                    }
                }
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
            if (visible == 0) {
                continue;
            }
            any = true;
            const float next = fmaxf(top, group_max<32>(s));
            const float shrink = top == -INFINITY ? 0.f : fast_exp2(top - next);
            const float p = use ? fast_exp2(s - (next == -INFINITY ? 0.f : next)) : 0.f;   // scores of minus infinity: 0
            top = next;
            total = total * shrink + group_sum<32>(p);
#pragma unroll
            for (int i = 0; i < COLS; ++i) {
                o[i] *= shrink;
            }
            while (visible != 0) {   // the rows of four keys on their way at a time
                float w[4];
                T e[4][COLS];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const bool on = visible != 0;
                    const int from = on ? __ffs(visible) - 1 : 0;
                    visible &= visible - 1;
                    w[u] = __shfl_sync(0xffffffffu, p, from);
                    w[u] = on ? w[u] : 0.f;
                    const T *vr = value(j0 + from);
#pragma unroll
                    for (int i = 0; i < COLS; ++i) {
                        e[u][i] = on && lane + 32 * i < dim ? vr[lane + 32 * i] : T(0.f);
                    }
                }
#pragma unroll
                for (int u = 0; u < 4; ++u) {
#pragma unroll
                    for (int i = 0; i < COLS; ++i) {
                        o[i] = fmaf(w[u], to_float<T>(e[u][i]), o[i]);
                    }
                }
            }
        }
    }
    const float inv = any ? 1.f / total : 0.f;   // nothing but scores of minus infinity: 0 times infinity, NaN as 0 / 0 is
#pragma unroll
    for (int i = 0; i < COLS; ++i) {
        if (lane + 32 * i < dim) {
            context[lane + 32 * i] = from_float<T>(o[i] * inv);
        }
    }
}

}  // namespace cubk
