// K8, single tokens: attention over ring caches, with a sliding window and first tokens that stay visible (sinks).
//
// The keys and values that a stream can still see live in a ring of sinks + window slots; the slot of position p is p below sinks
// and sinks + (p - sinks) % window from there on, so the slots that hold anything are the first min(p + 1, sinks + window) and
// every one of them is visible to p. Softmax statistics and all sums are float32.
#include <cooperative_groups.h>

#include "window_row.cuh"

namespace cubk {

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
template <typename T, int COLS>
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
        window_row<T, COLS>(q + b * s.q_stride + (int64_t) h * s.dim, s_q[warp], s.dim, s.scale, 0, 0, n,
                      [&](int j) { return j == slot ? kn : kc + (int64_t) j * s.dim; },
                      [&](int j) { return j == slot ? vn : vc + (int64_t) j * s.dim; }, [&](int) { return true; },
                      context + b * s.context_stride + (int64_t) h * s.dim);
    }
}

// ---- single tokens, 16-byte rows: a cluster of blocks per (stream, kv head)
// The keys of a stream are cut into blocks that the warps of the cluster take in turn, each with a softmax of its own over
// what it took; at the end the blocks read one another's partial sums through distributed shared memory and every block
// writes its share of the context. Nothing is staged in device memory, so calls need no workspace and no order among them,
// and the sums are added in the same order every time. The kernels are bound by the cache's bytes: 32 streams of 32 / 8 heads of 128
// over 2048 slots, binary16, take 40.5 us (5.2 TB/s, 0.81 of what a copy reaches). Small grids are bound by the loads an SM has in
// flight and by two cluster barriers: one such stream with 4096 slots 10.7 us, one float32 stream of 12 heads of 64 with 512 slots 4.5.
template <int WARPS, int HEADS, int DP>
struct StepPartial {
    float o[WARPS][HEADS][DP + 2];   // two columns of padding spread the rows over the banks
    float2 stat[WARPS][HEADS];       // maximum (log2 domain) and sum
    static_assert(HEADS <= 32, "a bit a head in step_join");
};

constexpr int kStepBlocks = 8;   // of a cluster at most

// Parts (maximum, sum, weighted sum of values) joined into one; a part without keys has sums of 0 and counts for nothing. At least
// one key is visible, so a sum of 0 in the end means that all scores are minus infinity, and 0 / 0 is what the row holds then.
template <int N>
__device__ __forceinline__ float3 join_parts(const float2 (&stat)[N], const float (&o)[N]) {
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        top = fmaxf(top, stat[i].x);
    }
    float sum = 0.f, total = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float weight = stat[i].x == -INFINITY ? 0.f : fast_exp2(stat[i].x - top);
        total = fmaf(weight, stat[i].y, total);
        sum = fmaf(weight, o[i], sum);
    }
    return make_float3(top, total, sum);
}

// First the warps of a block, in its own shared memory, then the blocks: each output element's parts are loaded together. What comes back
// in the first block are the heads to compute again: not finite although their scores are, in binary16, whose products see a weight
// of 0 where float32 has a small one, and 0 times an infinite value is NaN.
template <typename T, int WARPS, int HEADS, int DP>
__device__ __forceinline__ unsigned step_join(StepPartial<WARPS, HEADS, DP> *part, unsigned *s_again, int heads_here, int dim, T *out) {
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    const int blocks = (int) cluster.num_blocks(), rank = (int) cluster.block_rank();
    constexpr int PER_THREAD = (HEADS * DP + 32 * WARPS - 1) / (32 * WARPS);
    float3 joined[PER_THREAD];
    auto store = [&](unsigned *again, int h, int at, float total, float sum) {
        const float x = sum / total;
        out[at] = from_float<T>(x);
        if (sizeof(T) == 2 && !(fabsf(x) <= 65504.f) && total > 0.f) {
            atomicOr(again, 1u << h);
        }
    };
    if (threadIdx.x == 0) {
        *s_again = 0;
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < PER_THREAD; ++u) {
        const int e = threadIdx.x + u * 32 * WARPS, h = e / DP, x = e % DP;
        if (h < heads_here) {
            float2 stat[WARPS];
            float o[WARPS];
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                stat[w] = part->stat[w][h];
                o[w] = part->o[w][h][x];
            }
            joined[u] = join_parts<WARPS>(stat, o);
        }
    }
    if (blocks == 1) {
#pragma unroll
        for (int u = 0; u < PER_THREAD; ++u) {
            const int e = threadIdx.x + u * 32 * WARPS, h = e / DP, x = e % DP;
            if (h < heads_here && x < dim) {
                store(s_again, h, h * dim + x, joined[u].y, joined[u].z);
            }
        }
        __syncthreads();
        return *s_again;
    }
    __syncthreads();   // every warp's part has been read: the first one's place takes the block's
#pragma unroll
    for (int u = 0; u < PER_THREAD; ++u) {
        const int e = threadIdx.x + u * 32 * WARPS, h = e / DP, x = e % DP;
        if (h < heads_here) {
            part->o[0][h][x] = joined[u].z;
            if (x == 0) {
                part->stat[0][h] = make_float2(joined[u].x, joined[u].y);
            }
        }
    }
    cluster.sync();
    for (int e = rank * (32 * WARPS) + threadIdx.x; e < heads_here * dim; e += blocks * 32 * WARPS) {
        const int h = e / dim, x = e - h * dim;
        float2 stat[kStepBlocks];
        float o[kStepBlocks];
#pragma unroll
        for (int r = 0; r < kStepBlocks; ++r) {
            stat[r] = make_float2(-INFINITY, 0.f);
            o[r] = 0.f;
            if (r < blocks) {
                const StepPartial<WARPS, HEADS, DP> *from = cluster.map_shared_rank(part, r);
                stat[r] = from->stat[0][h];
                o[r] = from->o[0][h][x];
            }
        }
        const float3 all = join_parts<kStepBlocks>(stat, o);
        store(cluster.map_shared_rank(s_again, 0), h, e, all.y, all.z);
    }
    cluster.sync();   // nobody leaves while its sums are read
    return rank == 0 ? *s_again : 0;
}

// One head again, by a warp of its own over every visible slot.
template <int DP>
__device__ __forceinline__ void step_row_again(const __half *q, const __half *kn, const __half *vn, const __half *kc, const __half *vc, __half *out, float *s_q,
                                            int dim, float scale, int slot, int n) {
    window_row<__half, DP / 32>(q, s_q, dim, scale, 0, 0, n, [&](int j) { return j == slot ? kn : kc + (int64_t) j * dim; },
                       [&](int j) { return j == slot ? vn : vc + (int64_t) j * dim; }, [&](int) { return true; }, out);
}

struct StepPlace {
    int b, kh, first_head, heads_here, slot, n;
    int worker, workers;   // this warp among the cluster's
};

template <int WARPS, int HEADS>
__device__ __forceinline__ bool step_place(const int32_t *positions, const RingShape &s, int chunks, StepPlace &at) {
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    const int blocks = (int) cluster.num_blocks(), rank = (int) cluster.block_rank();
    const int64_t unit = blockIdx.x / blocks;
    const int share = s.heads / s.kv_heads;
    const int chunk = (int) (unit % chunks);
    const int64_t pair = unit / chunks;
    at.b = (int) (pair / s.kv_heads);
    at.kh = (int) (pair - (int64_t) at.b * s.kv_heads);
    at.first_head = at.kh * share + chunk * HEADS;
    at.heads_here = min(HEADS, share - chunk * HEADS);
    const int p = positions[at.b];
    if (p < 0) {
        return false;
    }
    const int slots = s.window + s.sinks;
    at.slot = ring_slot(p, s.window, s.sinks);
    at.n = p < slots ? p + 1 : slots;
    at.worker = rank * WARPS + (threadIdx.x >> 5);
    at.workers = blocks * WARPS;
    return true;
}

// The new token's row into its slot, by the first chunk's first block; the readers of the slot take the token's own row.
template <typename T, int WARPS>
__device__ __forceinline__ void step_store(const T *kn, const T *vn, T *kc, T *vc, const StepPlace &at, const RingShape &s) {
    if (at.first_head == at.kh * (s.heads / s.kv_heads) && at.worker < WARPS) {
        constexpr int E = 16 / (int) sizeof(T);
        for (int c = threadIdx.x; c < s.dim / E; c += 32 * WARPS) {
            reinterpret_cast<uint4 *>(kc + (int64_t) at.slot * s.dim)[c] = reinterpret_cast<const uint4 *>(kn)[c];
            reinterpret_cast<uint4 *>(vc + (int64_t) at.slot * s.dim)[c] = reinterpret_cast<const uint4 *>(vn)[c];
        }
    }
}

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose_8x8(uint32_t a) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}

// Binary16: S^T = K.Q^T and O^T += V^T.P^T on warp-level matrix instructions, 16 keys x 8 NT heads a block of keys. Lane
// (g, t) = (lane / 4, lane % 4) reads 16 bytes (chunk t, t + 4, ..) of the K rows g and g + 8: eight columns that are two steps
// of the reduction, in an order that Q shares. Of V it reads chunk g (g + 8) of the rows 2 t, 2 t + 1, 2 t + 8, 2 t + 9 and pairs
// the halves of two rows: word i of a chunk is rows g and g + 8 of the i-th 16 output columns. So K and V go from memory to
// operands with no stop in shared memory; P^T turns around in registers. Registers are bounded so that five blocks of four warps share an SM
// for heads of 64 (16 streams of 12 heads, 1024 slots: 11.0 us, with four 15.3).
template <int WARPS, int DP, int NT>
__global__ void __launch_bounds__(32 * WARPS, (DP == 64 ? (NT == 1 ? 20 : 16) : (NT == 1 ? 12 : 8)) / WARPS)
window_step_f16_kernel(const __half *q, const __half *k, const __half *v, const int32_t *positions, __half *k_cache, __half *v_cache,
                       __half *context, const __grid_constant__ RingShape s, int chunks) {
    constexpr int HEADS = 8 * NT, KC = DP / 32, VC = DP / 64;
    __shared__ StepPartial<WARPS, HEADS, DP> part;
    __shared__ unsigned s_again;
    StepPlace at;
    if (!step_place<WARPS, HEADS>(positions, s, chunks, at)) {
        return;
    }
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int64_t slots = s.window + s.sinks;
    const __half *kn = k + at.b * s.kv_stride + (int64_t) at.kh * s.dim, *vn = v + at.b * s.kv_stride + (int64_t) at.kh * s.dim;
    __half *kc = k_cache + ((int64_t) at.b * s.kv_heads + at.kh) * slots * s.dim, *vc = v_cache + ((int64_t) at.b * s.kv_heads + at.kh) * slots * s.dim;
    step_store<__half, WARPS>(kn, vn, kc, vc, at, s);

    uint32_t qf[NT][KC][4];
#pragma unroll
    for (int m = 0; m < NT; ++m) {
#pragma unroll
        for (int c = 0; c < KC; ++c) {
            const int col = 8 * (t + 4 * c), head = 8 * m + g;
            uint4 r = make_uint4(0, 0, 0, 0);
            if (head < at.heads_here && col < s.dim) {
                r = ld_param(q + at.b * s.q_stride + (int64_t) (at.first_head + head) * s.dim + col);
            }
            qf[m][c][0] = r.x, qf[m][c][1] = r.y, qf[m][c][2] = r.z, qf[m][c][3] = r.w;
        }
    }
    float o[NT][VC][4][4];
    float top[NT][2], total[NT][2];
#pragma unroll
    for (int m = 0; m < NT; ++m) {
        top[m][0] = top[m][1] = -INFINITY;
        total[m][0] = total[m][1] = 0.f;
#pragma unroll
        for (int x = 0; x < VC; ++x) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                o[m][x][i][0] = o[m][x][i][1] = o[m][x][i][2] = o[m][x][i][3] = 0.f;
            }
        }
    }
    const float c2 = s.scale * kLog2e;
    const int key_blocks = (at.n + 15) / 16;
    for (int kb = at.worker; kb < key_blocks; kb += at.workers) {
        const int j0 = kb * 16;
        uint4 kr[2][KC], vr[4][VC];
        const bool whole = j0 + 16 <= at.n && (at.slot < j0 || at.slot >= j0 + 16);
        if (whole) {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const __half *row = kc + (int64_t) (j0 + g + 8 * r) * s.dim;
#pragma unroll
                for (int c = 0; c < KC; ++c) {
                    const int col = 8 * (t + 4 * c);
                    kr[r][c] = col < s.dim ? ld_stream(row + col) : make_uint4(0, 0, 0, 0);
                }
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const __half *row = vc + (int64_t) (j0 + 2 * t + (r & 1) + 8 * (r >> 1)) * s.dim;
#pragma unroll
                for (int x = 0; x < VC; ++x) {
                    const int col = 8 * (g + 8 * x);
                    vr[r][x] = col < s.dim ? ld_stream(row + col) : make_uint4(0, 0, 0, 0);
                }
            }
        } else {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int j = j0 + g + 8 * r;
                const __half *row = j == at.slot ? kn : kc + (int64_t) j * s.dim;
#pragma unroll
                for (int c = 0; c < KC; ++c) {
                    const int col = 8 * (t + 4 * c);
                    kr[r][c] = j < at.n && col < s.dim ? *reinterpret_cast<const uint4 *>(row + col) : make_uint4(0, 0, 0, 0);
                }
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int j = j0 + 2 * t + (r & 1) + 8 * (r >> 1);
                const __half *row = j == at.slot ? vn : vc + (int64_t) j * s.dim;
#pragma unroll
                for (int x = 0; x < VC; ++x) {
                    const int col = 8 * (g + 8 * x);
                    vr[r][x] = j < at.n && col < s.dim ? *reinterpret_cast<const uint4 *>(row + col) : make_uint4(0, 0, 0, 0);
                }
            }
        }
        float sc[NT][4];
#pragma unroll
        for (int m = 0; m < NT; ++m) {
            sc[m][0] = sc[m][1] = sc[m][2] = sc[m][3] = 0.f;
#pragma unroll
            for (int c = 0; c < KC; ++c) {
                mma_f16(sc[m], kr[0][c].x, kr[1][c].x, kr[0][c].y, kr[1][c].y, qf[m][c][0], qf[m][c][1]);
                mma_f16(sc[m], kr[0][c].z, kr[1][c].z, kr[0][c].w, kr[1][c].w, qf[m][c][2], qf[m][c][3]);
            }
        }
        bool raise = false;
#pragma unroll
        for (int m = 0; m < NT; ++m) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {   // e: head 2 t + e % 2, key g + 8 (e / 2)
                sc[m][e] = j0 + g + 8 * (e >> 1) < at.n ? sc[m][e] * c2 : -INFINITY;
                raise = raise || sc[m][e] - top[m][e & 1] > kRaiseBy + kWeightScale;
            }
        }
        if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
            for (int m = 0; m < NT; ++m) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float here = fmaxf(fmaxf(sc[m][e], sc[m][e + 2]) - kWeightScale, top[m][e]);   // 2^7 below the largest
                    here = fmaxf(here, __shfl_xor_sync(0xffffffffu, here, 4));
                    here = fmaxf(here, __shfl_xor_sync(0xffffffffu, here, 8));
                    here = fmaxf(here, __shfl_xor_sync(0xffffffffu, here, 16));
                    const float shrink = top[m][e] == here ? 1.f : fast_exp2(top[m][e] - here);
                    top[m][e] = here;
                    total[m][e] *= shrink;
#pragma unroll
                    for (int x = 0; x < VC; ++x) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            o[m][x][i][e] *= shrink;
                            o[m][x][i][e + 2] *= shrink;
                        }
                    }
                }
            }
        }
#pragma unroll
        for (int m = 0; m < NT; ++m) {
            float p[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                p[e] = sc[m][e] == -INFINITY ? 0.f : fast_exp2(sc[m][e] - top[m][e & 1]);
                total[m][e & 1] += p[e];
            }
            // each weight as two binary16 numbers: 22 bits of it, where one has 11 (32 streams of 32 / 8 heads of 128: 40.5 us, with one 40.15)
            uint32_t b[2][2];   // high and low parts, keys 0 to 7 and 8 to 15
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const __half2 high = __floats2half2_rn(p[2 * i], p[2 * i + 1]);
                const float2 back = __half22float2(high);
                const __half2 low = __floats2half2_rn(p[2 * i] - back.x, p[2 * i + 1] - back.y);
                b[0][i] = transpose_8x8(*reinterpret_cast<const uint32_t *>(&high));
                b[1][i] = transpose_8x8(*reinterpret_cast<const uint32_t *>(&low));
            }
#pragma unroll
            for (int x = 0; x < VC; ++x) {
                const uint32_t w0[4] = {vr[0][x].x, vr[0][x].y, vr[0][x].z, vr[0][x].w}, w1[4] = {vr[1][x].x, vr[1][x].y, vr[1][x].z, vr[1][x].w};
                const uint32_t w2[4] = {vr[2][x].x, vr[2][x].y, vr[2][x].z, vr[2][x].w}, w3[4] = {vr[3][x].x, vr[3][x].y, vr[3][x].z, vr[3][x].w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t a[4] = {__byte_perm(w0[i], w1[i], 0x5410), __byte_perm(w0[i], w1[i], 0x7632), __byte_perm(w2[i], w3[i], 0x5410),
                                           __byte_perm(w2[i], w3[i], 0x7632)};
                    mma_f16(o[m][x][i], a[0], a[1], a[2], a[3], b[1][0], b[1][1]);
                    mma_f16(o[m][x][i], a[0], a[1], a[2], a[3], b[0][0], b[0][1]);
                }
            }
        }
    }
#pragma unroll
    for (int m = 0; m < NT; ++m) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float sum = total[m][e];
            sum += __shfl_xor_sync(0xffffffffu, sum, 4);
            sum += __shfl_xor_sync(0xffffffffu, sum, 8);
            sum += __shfl_xor_sync(0xffffffffu, sum, 16);
            const int head = 8 * m + 2 * t + e;
            if (g == 0) {
                part.stat[warp][head] = make_float2(top[m][e], sum);
            }
#pragma unroll
            for (int x = 0; x < VC; ++x) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    *reinterpret_cast<float2 *>(&part.o[warp][head][8 * (g + 8 * x) + 2 * i]) = make_float2(o[m][x][i][e], o[m][x][i][e + 2]);
                }
            }
        }
    }
    __half *out = context + at.b * s.context_stride + (int64_t) at.first_head * s.dim;
    const unsigned again = step_join<__half, WARPS, HEADS, DP>(&part, &s_again, at.heads_here, s.dim, out);
    if (again != 0) {   // the parts have been read: their place holds the queries
        for (int h = warp; h < at.heads_here; h += WARPS) {
            if ((again >> h & 1u) != 0) {
                step_row_again<DP>(q + at.b * s.q_stride + (int64_t) (at.first_head + h) * s.dim, kn, vn, kc, vc, out + h * s.dim,
                               part.o[warp][0], s.dim, s.scale, at.slot, at.n);
            }
        }
    }
}

// float32: LPK lanes share a key, four columns each, so that a warp reads 32 / LPK whole rows per instruction; every group of
// lanes keeps a softmax of its own over its keys, HEADS heads at once. Per key and head a lane has four multiply-adds for the score
// and log2(LPK) shuffles with an addition each for its sum.
template <int WARPS, int LPK, int HEADS>
__global__ void __launch_bounds__(32 * WARPS)
window_step_f32_kernel(const float *q, const float *k, const float *v, const int32_t *positions, float *k_cache, float *v_cache, float *context,
                       const __grid_constant__ RingShape s, int chunks) {
    constexpr int DP = 4 * LPK, GROUPS = 32 / LPK, U = HEADS == 1 ? 8 : 4;   // U: rows per lane group in flight
    __shared__ StepPartial<WARPS, HEADS, DP> part;
    __shared__ unsigned s_again;
    StepPlace at;
    if (!step_place<WARPS, HEADS>(positions, s, chunks, at)) {
        return;
    }
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, group = lane / LPK, col = 4 * (lane % LPK);
    const int64_t slots = s.window + s.sinks;
    const float *kn = k + at.b * s.kv_stride + (int64_t) at.kh * s.dim, *vn = v + at.b * s.kv_stride + (int64_t) at.kh * s.dim;
    float *kc = k_cache + ((int64_t) at.b * s.kv_heads + at.kh) * slots * s.dim, *vc = v_cache + ((int64_t) at.b * s.kv_heads + at.kh) * slots * s.dim;
    step_store<float, WARPS>(kn, vn, kc, vc, at, s);
    const bool mine = col < s.dim;
    const float c2 = s.scale * kLog2e;
    float4 qf[HEADS], o[HEADS];
    float top[HEADS], total[HEADS];
#pragma unroll
    for (int h = 0; h < HEADS; ++h) {
        qf[h] = mine && h < at.heads_here
                    ? __ldg(reinterpret_cast<const float4 *>(q + at.b * s.q_stride + (int64_t) (at.first_head + h) * s.dim + col))
                    : make_float4(0.f, 0.f, 0.f, 0.f);
        o[h] = make_float4(0.f, 0.f, 0.f, 0.f);
        top[h] = -INFINITY;
        total[h] = 0.f;
    }
    const int per_block = GROUPS * U, key_blocks = (at.n + per_block - 1) / per_block;
    for (int kb = at.worker; kb < key_blocks; kb += at.workers) {
        float4 kr[U], vr[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int j = kb * per_block + u * GROUPS + group;
            const float *krow = j == at.slot ? kn : kc + (int64_t) j * s.dim, *vrow = j == at.slot ? vn : vc + (int64_t) j * s.dim;
            const bool in = mine && j < at.n;
            kr[u] = in ? *reinterpret_cast<const float4 *>(krow + col) : make_float4(0.f, 0.f, 0.f, 0.f);
            vr[u] = in ? *reinterpret_cast<const float4 *>(vrow + col) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
#pragma unroll
        for (int h = 0; h < HEADS; ++h) {
            float sc[U];
            float here = top[h];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float d = fmaf(qf[h].x, kr[u].x, qf[h].y * kr[u].y) + fmaf(qf[h].z, kr[u].z, qf[h].w * kr[u].w);
#pragma unroll
                for (int m = LPK / 2; m > 0; m >>= 1) {
                    d += __shfl_xor_sync(0xffffffffu, d, m);
                }
                sc[u] = kb * per_block + u * GROUPS + group < at.n ? d * c2 : -INFINITY;
                here = fmaxf(here, sc[u]);
            }
            const float shrink = top[h] == here ? 1.f : fast_exp2(top[h] - here);
            top[h] = here;
            total[h] *= shrink;
            o[h].x *= shrink, o[h].y *= shrink, o[h].z *= shrink, o[h].w *= shrink;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const float p = sc[u] == -INFINITY ? 0.f : fast_exp2(sc[u] - here);
                total[h] += p;
                o[h].x = fmaf(p, vr[u].x, o[h].x);
                o[h].y = fmaf(p, vr[u].y, o[h].y);
                o[h].z = fmaf(p, vr[u].z, o[h].z);
                o[h].w = fmaf(p, vr[u].w, o[h].w);
            }
        }
    }
#pragma unroll
    for (int h = 0; h < HEADS; ++h) {
        float all = top[h];
#pragma unroll
        for (int m = LPK; m < 32; m <<= 1) {
            all = fmaxf(all, __shfl_xor_sync(0xffffffffu, all, m));
        }
        const float shrink = top[h] == all ? 1.f : (top[h] == -INFINITY ? 0.f : fast_exp2(top[h] - all));
        float r[5] = {total[h] * shrink, o[h].x * shrink, o[h].y * shrink, o[h].z * shrink, o[h].w * shrink};
#pragma unroll
        for (int m = LPK; m < 32; m <<= 1) {
#pragma unroll
            for (int i = 0; i < 5; ++i) {
                r[i] += __shfl_xor_sync(0xffffffffu, r[i], m);
            }
        }
        if (group == 0) {
            if (lane == 0) {
                part.stat[warp][h] = make_float2(all, r[0]);
            }
            *reinterpret_cast<float2 *>(&part.o[warp][h][col]) = make_float2(r[1], r[2]);
            *reinterpret_cast<float2 *>(&part.o[warp][h][col + 2]) = make_float2(r[3], r[4]);
        }
    }
    step_join<float, WARPS, HEADS, DP>(&part, &s_again, at.heads_here, s.dim, context + at.b * s.context_stride + (int64_t) at.first_head * s.dim);
}

// Blocks of a cluster: doubled until the grid has two blocks per SM, and on to about five while every warp keeps 6 KB of keys (below
// that a block's start and join cost more than its share of the loads brings: 9 streams of 32 / 8 heads of 128 with 715 slots take 9.8 us
// in clusters of four, 13.9 in eights; 16 of 12 heads of 64 with 1024 slots 13.1 in twos, 11.0 in fours).
inline int step_cluster(int64_t units, int64_t slots, int64_t row_bytes) {
    int blocks = 1;
    while (blocks < kStepBlocks && slots > 64 * blocks) {
        const int64_t grid = units * blocks * 2, warp_bytes = slots * row_bytes / (blocks * 2 * 4);
        if (grid > 2 * 148 && (grid > 5 * 148 + 74 || warp_bytes < 6 * 1024)) {
            break;
        }
        blocks *= 2;
    }
    return blocks;
}

template <typename T, int HEADS, typename Kernel>
int step_launch(Kernel four, Kernel eight, bool has_eight, const T *q, const T *k, const T *v, const int32_t *positions, T *k_cache, T *v_cache, T *context,
                const RingShape &s, cudaStream_t stream) {
    const int chunks = (s.heads / s.kv_heads + HEADS - 1) / HEADS;
    const int64_t units = (int64_t) s.batch * s.kv_heads * chunks, slots = (int64_t) s.window + s.sinks;
    const int cluster = step_cluster(units, slots, (int64_t) s.dim * (int) sizeof(T));
    if (units * cluster > 0x7fffffffLL) {
        return CUBK_ERR_UNSUPPORTED;
    }
    // Eight warps a block where even full clusters leave half of the SMs without one: what a stream takes then is set by the loads an
    // SM has in flight (one stream of 32 / 8 heads of 128 with 4096 slots: 13.6 us with four warps, 10.6 with eight; with blocks on most
    // SMs four are the better: 4 streams of 16 / 4 heads, 14.2 against 17.0).
    const bool wide = has_eight && units * cluster <= 74 && slots >= 128 * cluster;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3((unsigned) (units * cluster));
    config.blockDim = dim3(wide ? 256 : 128);
    config.stream = stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned) cluster;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    config.attrs = &attr;
    config.numAttrs = 1;
    const cudaError_t err = cudaLaunchKernelEx(&config, wide ? eight : four, q, k, v, positions, k_cache, v_cache, context, s, chunks);
    if (err != cudaSuccess) {
        (void) cudaGetLastError();
        set_last_error(err);
        return CUBK_ERR_LAUNCH;
    }
    return CUBK_OK;
}

// Rows and heads that start on 16-byte boundaries, head dimension up to 128.
inline int step_vectors(const __half *q, const __half *k, const __half *v, const int32_t *positions, __half *k_cache, __half *v_cache,
                        __half *context, const RingShape &s, cudaStream_t stream) {
    const int share = s.heads / s.kv_heads;
    // the parts of eight warps with 16 heads of 128 do not fit a block's static shared memory
#define STEP_F16(DP, NT)                                                                                                                  \
    step_launch<__half, 8 * NT>(window_step_f16_kernel<4, DP, NT>, window_step_f16_kernel<DP * NT == 256 ? 4 : 8, DP, NT>, DP * NT < 256, q, \
                                k, v, positions, k_cache, v_cache, context, s, stream)
    if (s.dim <= 64) {
        return share <= 8 ? STEP_F16(64, 1) : STEP_F16(64, 2);
    }
    return share <= 8 ? STEP_F16(128, 1) : STEP_F16(128, 2);
#undef STEP_F16
}

inline int step_vectors(const float *q, const float *k, const float *v, const int32_t *positions, float *k_cache, float *v_cache, float *context,
                        const RingShape &s, cudaStream_t stream) {
    const int share = s.heads / s.kv_heads;
#define STEP_F32(LPK, HEADS)                                                                                                             \
    step_launch<float, HEADS>(window_step_f32_kernel<4, LPK, HEADS>, window_step_f32_kernel<8, LPK, HEADS>, true, q, k, v, positions,   \
                              k_cache, v_cache, context, s, stream)
    if (share == 1) {
        return s.dim <= 32 ? STEP_F32(8, 1) : s.dim <= 64 ? STEP_F32(16, 1) : STEP_F32(32, 1);
    }
    return s.dim <= 32 ? STEP_F32(8, 4) : s.dim <= 64 ? STEP_F32(16, 4) : STEP_F32(32, 4);
#undef STEP_F32
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
    constexpr int E = 16 / (int) sizeof(T);
    if (dim <= 128 && dim % E == 0 && q_stride % E == 0 && kv_stride % E == 0 && aligned16(q) && aligned16(k) && aligned16(v) &&
        aligned16(k_cache) && aligned16(v_cache)) {
        const int rc = step_vectors(q, k, v, positions, k_cache, v_cache, context, s, stream);
        if (rc != CUBK_ERR_UNSUPPORTED) {
            return rc;
        }
    }
    const int64_t groups = ((int64_t) batch * heads + kWindowRowWarps - 1) / kWindowRowWarps;
    const unsigned blocks = (unsigned) (groups < 148 * 64 ? groups : 148 * 64);
    const auto kernel = dim <= 64 ? window_step_rows_kernel<T, 2> : dim <= 128 ? window_step_rows_kernel<T, 4> : window_step_rows_kernel<T, 8>;
    kernel<<<blocks, 32 * kWindowRowWarps, 0, stream>>>(q, k, v, positions, k_cache, v_cache, context, s);
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
