// K8: attention with a sliding window and first tokens that stay visible (sinks).
//
// Whole sequences: query i sees key j when the key is kept, j <= i + after, and j >= i - before or j < sinks.
// Single tokens: keys and values live in a ring of sinks + window slots per stream; the slot of position p is p
// below sinks and sinks + (p - sinks) % window from there on, so the slots that hold anything are the first
// min(p + 1, sinks + window) and every one of them is visible to p.
// Softmax statistics and all sums are float32. A key that a query does not see contributes nothing at all, whatever
// bits its rows hold; a query that sees no key gets zeros.
#include <cuda.h>

#include <atomic>

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

// ---------------------------------------------------------------- whole sequences on tcgen05 (binary16)
// A block owns NQ tiles of 128 query rows: two heads that share their keys, or consecutive rows of one head. Per step of up
// to 128 keys and per tile: S = Q.K^T (tcgen05.mma, float32 accumulators in tensor memory), softmax by 128 threads that own
// a row each (tensor-memory lane = query row, so no shuffles), P back into tensor memory over S as binary16, O += P.V with P
// as the tensor-memory operand. Warps: 4 NQ for the softmax, one that issues the MMAs, one that chooses the steps and
// loads K and V with TMA (128-byte swizzle; V is read as it lies, as an MN-major operand).
//   * Steps: first the sinks below the window, then the window in 128s. A step whose keys are all masked is left out; one that
//     every row of a tile sees whole skips the masking.
//   * The running maximum of a row is raised only when a step's maximum exceeds it by 2^8 (a weight is then at most 256, far
//     inside binary16, and the sums are float32), so that O is read back and scaled in few steps.
//   * Weights of unseen keys are exactly 0, but 0 times an infinity or NaN in an unseen V row is NaN: a row that comes out not
//     finite is computed again by one warp over its visible keys alone.
// Every wait is bounded; a block that gives up writes NaN, frees its tensor memory and returns.
constexpr int kTileRows = 128;
constexpr int kHalfTileBytes = kTileRows * 128;    // 128 rows x 64 binary16
constexpr int kStepSlots = 8;                      // descriptors of steps in flight; more than the stages + 1
constexpr float kRaiseBy = 8.f;                    // log2 of the largest weight

struct WindowStep {
    int j0, keys;            // keys = 0: no more steps
    uint32_t kept[4];
    uint32_t flags;          // bit t: tile t takes part; bit 4 + t: some row of tile t does not see some key
};

template <int DP, int NQ>
struct WindowTc {
    static constexpr int HALVES = DP / 64;
    static constexpr int TILE_BYTES = HALVES * kHalfTileBytes;
    static constexpr int STAGES = 2;
    static constexpr int SOFTMAX_WARPS = 4 * NQ;
    static constexpr int THREADS = 32 * (SOFTMAX_WARPS + 2);
    static constexpr int TMEM_COLS = NQ == 1 ? 256 : 512;
    static constexpr int SMEM_BYTES = 1024 + (NQ + 2 * STAGES) * TILE_BYTES;   // 1024: alignment of the swizzled tiles
    static_assert(NQ * (128 + DP) <= TMEM_COLS, "scores and contexts of all tiles");
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

__device__ __forceinline__ void tmem_load32(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
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

// 128 rows x 64 columns of one head into a swizzled tile; rows and columns outside the tensor arrive as zeros.
__device__ __forceinline__ void tma_tile(void *dst, const CUtensorMap *map, int column, int row, int head, int batch, uint64_t *bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(
                     smem_addr(dst)),
                 "l"(map), "r"(column), "r"(row), "r"(head), "r"(batch), "r"(smem_addr(bar))
                 : "memory");
}

// Bits lo .. hi - 1 of a word that stands for positions base .. base + 31.
__device__ __forceinline__ uint32_t range_bits(int lo, int hi, int base) {
    const int a = min(max(lo - base, 0), 32), b = min(max(hi - base, 0), 32);
    const uint32_t below_b = b == 32 ? 0xffffffffu : (1u << b) - 1u, below_a = a == 32 ? 0xffffffffu : (1u << a) - 1u;
    return below_b & ~below_a;
}

// One row again over its visible keys alone (rows whose tile held an infinity or NaN).
__device__ __noinline__ void window_row_again(const __half *q, const __half *k, const __half *v, const int8_t *mask, __half *context,
                                              const WindowShape *s, float *s_q, int b, int i, int h) {
    window_prompt_row<__half>(q, k, v, mask, context, *s, s_q, b, i, h);
}

template <int DP, int NQ>
__global__ void __launch_bounds__(WindowTc<DP, NQ>::THREADS, NQ == 1 ? 2 : 1)
window_tc_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                 const __half *q, const __half *k, const __half *v, const int8_t *mask, __half *context, const __grid_constant__ WindowShape s,
                 int row_blocks, int pair_heads) {
    typedef WindowTc<DP, NQ> C;
    extern __shared__ unsigned char tc_raw[];
    __shared__ uint64_t s_qfull, s_kfull[C::STAGES], s_kempty[C::STAGES], s_vfull[C::STAGES], s_vempty[C::STAGES], s_sfull[NQ], s_pfull[NQ];
    __shared__ uint32_t s_tmem;
    __shared__ WindowStep s_steps[kStepSlots];
    __shared__ float s_row[C::SOFTMAX_WARPS][kWindowMaxDim];
    unsigned char *tiles = tc_raw + ((1024u - (smem_addr(tc_raw) & 1023u)) & 1023u);
    unsigned char *s_qt = tiles, *s_kt = tiles + NQ * C::TILE_BYTES, *s_vt = s_kt + C::STAGES * C::TILE_BYTES;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    // the block's tiles: last rows first (with a one-sided window that reaches far, they have the most keys)
    const int per_head = row_blocks;
    const int rb = per_head - 1 - (int) (blockIdx.x % per_head);
    const int bh = (int) (blockIdx.x / per_head);
    const int head_groups = pair_heads ? s.heads / 2 : s.heads;
    const int b = bh / head_groups;
    const int h0 = (bh - b * head_groups) * (pair_heads ? 2 : 1);
    const int row0 = rb * (pair_heads ? kTileRows : NQ * kTileRows);
    const int kh = h0 / (s.heads / s.kv_heads);
    int tile_row[NQ], tile_head[NQ];
#pragma unroll
    for (int t = 0; t < NQ; ++t) {
        tile_row[t] = pair_heads ? row0 : row0 + t * kTileRows;
        tile_head[t] = pair_heads ? h0 + t : h0;
    }

    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&s_tmem)), "r"((uint32_t) C::TMEM_COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (threadIdx.x == 32) {
        mbar_init(&s_qfull, 1);
        for (int i = 0; i < C::STAGES; ++i) {
            mbar_init(&s_kfull[i], 1);
            mbar_init(&s_kempty[i], 1);
            mbar_init(&s_vfull[i], 1);
            mbar_init(&s_vempty[i], 1);
        }
        for (int t = 0; t < NQ; ++t) {
            mbar_init(&s_sfull[t], 2);   // the MMAs' completion and the issuing thread, which read the step's descriptor
            mbar_init(&s_pfull[t], 4);
        }
        mbar_init_fence();
    }
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    const uint32_t tmem = s_tmem;

    if (warp == C::SOFTMAX_WARPS + 1) {
        // ---- steps and loads
        const int last_row = min(row0 + (pair_heads ? 1 : NQ) * kTileRows, s.seq) - 1;
        const int lo = row0 > s.before ? row0 - s.before : 0;
        const int hi = s.after < s.seq - 1 - last_row ? last_row + s.after + 1 : s.seq;
        const int sinks_end = min(s.sinks, lo);
        const int8_t *kept = mask != nullptr ? mask + (int64_t) b * s.seq : nullptr;
        if (lane == 0) {
            mbar_arrive_expect(&s_qfull, NQ * C::TILE_BYTES);
            for (int t = 0; t < NQ; ++t) {
                for (int x = 0; x < C::HALVES; ++x) {
                    tma_tile(s_qt + t * C::TILE_BYTES + x * kHalfTileBytes, &q_map, 64 * x, tile_row[t], tile_head[t], b, &s_qfull);
                }
            }
        }
        bool ok = true;
        int step = 0;
        int j0 = sinks_end > 0 ? 0 : lo;
        bool in_sinks = sinks_end > 0;
        while (ok) {
            if (in_sinks && j0 >= sinks_end) {
                in_sinks = false;
                j0 = lo;
            }
            const int keys = min((in_sinks ? sinks_end : hi) - j0, kTileRows);   // none left: 0 or less (only past the window)
            WindowStep d;
            d.j0 = j0;
            d.keys = max(keys, 0);
            d.flags = 0;
            bool all = true;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const int j = j0 + 32 * w + lane;
                const bool in = 32 * w + lane < keys;
                const bool on = in && (kept == nullptr || kept[j] != 0);
                d.kept[w] = __ballot_sync(0xffffffffu, on);
                all = all && __all_sync(0xffffffffu, on || !in);
            }
            j0 += kTileRows;
            if (keys > 0) {
                if ((d.kept[0] | d.kept[1] | d.kept[2] | d.kept[3]) == 0) {
                    continue;
                }
#pragma unroll
                for (int t = 0; t < NQ; ++t) {
                    const int first = tile_row[t], last = min(first + kTileRows, s.seq) - 1;
                    const int t_lo = first > s.before ? first - s.before : 0;
                    const int t_hi = s.after < s.seq - 1 - last ? last + s.after + 1 : s.seq;
                    if (first < s.seq && d.j0 < t_hi && (d.j0 + keys > t_lo || d.j0 < s.sinks)) {
                        d.flags |= 1u << t;
                    }
                    const bool whole = all && keys % 32 == 0 && (s.after >= s.seq || d.j0 + keys - 1 <= first + s.after) &&
                                       (last - s.before <= d.j0 || d.j0 + keys <= s.sinks);
                    if (!whole) {
                        d.flags |= 16u << t;
                    }
                }
            }
            const int st = step % C::STAGES;
            const uint32_t again = (step / C::STAGES) & 1;
            if (step >= C::STAGES) {
                ok = __all_sync(0xffffffffu, mbar_wait_bounded(&s_kempty[st], again ^ 1));
                if (!ok) {
                    break;
                }
            }
            if (lane == 0) {
                s_steps[step % kStepSlots] = d;
                if (d.keys > 0) {
                    mbar_arrive_expect(&s_kfull[st], C::TILE_BYTES);
                    for (int x = 0; x < C::HALVES; ++x) {
                        tma_tile(s_kt + st * C::TILE_BYTES + x * kHalfTileBytes, &k_map, 64 * x, d.j0, kh, b, &s_kfull[st]);
                    }
                } else {
                    mbar_arrive(&s_kfull[st]);
                }
            }
            __syncwarp();
            if (d.keys == 0) {
                break;
            }
            if (step >= C::STAGES) {
                ok = __all_sync(0xffffffffu, mbar_wait_bounded(&s_vempty[st], again ^ 1));
            }
            if (ok && lane == 0) {
                mbar_arrive_expect(&s_vfull[st], C::TILE_BYTES);
                for (int x = 0; x < C::HALVES; ++x) {
                    tma_tile(s_vt + st * C::TILE_BYTES + x * kHalfTileBytes, &v_map, 64 * x, d.j0, kh, b, &s_vfull[st]);
                }
            }
            __syncwarp();
            ++step;
        }
        if (!ok) {   // the copies in flight land before the block's shared memory goes
            (void) mbar_wait_bounded(&s_qfull, 0);
            for (int i = max(step - C::STAGES, 0); i <= step; ++i) {
                (void) mbar_wait_bounded(&s_kfull[i % C::STAGES], (i / C::STAGES) & 1);
                (void) mbar_wait_bounded(&s_vfull[i % C::STAGES], (i / C::STAGES) & 1);
            }
        }
        __syncwarp();
    } else if (warp == C::SOFTMAX_WARPS) {
        // ---- matrix products, issued by one thread
        if (lane == 0) {
            const uint32_t ksteps = (uint32_t) (s.dim + 15) / 16;
            const uint32_t idesc_o = (1u << 4) | (1u << 16) | ((2 * ksteps) << 17) | ((kTileRows >> 4) << 24);   // N: the dimension, in 16s
            bool ok = mbar_wait_bounded(&s_qfull, 0);
            bool first[NQ];
#pragma unroll
            for (int t = 0; t < NQ; ++t) {
                first[t] = true;
            }
            int keys_before = 0;
            uint32_t flags_before = 0;
            for (int step = 0; ok; ++step) {
                const int st = step % C::STAGES, st_before = (step + C::STAGES - 1) % C::STAGES;
                ok = mbar_wait_bounded(&s_kfull[st], (step / C::STAGES) & 1);
                if (!ok) {
                    break;
                }
                const int keys = s_steps[step % kStepSlots].keys;
                const uint32_t flags = s_steps[step % kStepSlots].flags;
                const uint32_t keys16 = (uint32_t) (keys + 15) / 16;
                const uint32_t idesc_s = (1u << 4) | ((2 * keys16) << 17) | ((kTileRows >> 4) << 24);
#pragma unroll
                for (int t = 0; t < NQ; ++t) {
                    if (step > 0) {
                        ok = ok && mbar_wait_bounded(&s_pfull[t], (step - 1) & 1) &&
                             mbar_wait_bounded(&s_vfull[st_before], ((step - 1) / C::STAGES) & 1);
                        tmem_fence_after();
                        if (ok && (flags_before >> t & 1u) != 0) {
                            const uint32_t vs = smem_addr(s_vt + st_before * C::TILE_BYTES);
                            for (int kk = 0; kk < (keys_before + 15) / 16; ++kk) {
                                mma_ts(tmem + NQ * 128 + t * DP, tmem + t * 128 + 8 * kk, swizzled_desc(vs + 2048 * kk, kHalfTileBytes), idesc_o,
                                       !(first[t] && kk == 0));
                            }
                            first[t] = false;
                        }
                        if (t == NQ - 1 && ok) {
                            mma_commit(&s_vempty[st_before]);
                        }
                    }
                    if (ok && (flags >> t & 1u) != 0) {
                        const uint32_t qs = smem_addr(s_qt + t * C::TILE_BYTES), ks = smem_addr(s_kt + st * C::TILE_BYTES);
                        for (uint32_t kk = 0; kk < ksteps; ++kk) {
                            const uint32_t at = (kk >> 2) * kHalfTileBytes + (kk & 3) * 32;
                            mma_ss(tmem + t * 128, swizzled_desc(qs + at, 16), swizzled_desc(ks + at, 16), idesc_s, kk > 0);
                        }
                    }
                    if (ok) {
                        mma_commit(&s_sfull[t]);
                        mbar_arrive(&s_sfull[t]);
                    }
                }
                if (keys == 0) {
                    break;
                }
                if (ok) {
                    mma_commit(&s_kempty[st]);
                }
                keys_before = keys;
                flags_before = flags;
            }
        }
        __syncwarp();
    } else {
        // ---- softmax: a row per thread
        const int t = NQ == 1 ? 0 : warp / 4;
        const int i = tile_row[t] + 32 * (warp & 3) + lane;
        const int h = tile_head[t];
        const uint32_t lanes = (uint32_t) (32 * (warp & 3)) << 16;
        const uint32_t t_s = tmem + t * 128 + lanes, t_o = tmem + NQ * 128 + t * DP + lanes;
        const int lo = i > s.before ? i - s.before : 0;
        const int hi = s.after < s.seq - 1 - i ? i + s.after + 1 : s.seq;
        const float c = s.scale * kLog2e;
        float top = -INFINITY, total = 0.f;   // top: of q.k, unscaled
        bool first = true, ok = true;
        for (int step = 0;; ++step) {
            ok = __all_sync(0xffffffffu, mbar_wait_bounded(&s_sfull[t], step & 1));
            if (!ok) {
                break;
            }
            tmem_fence_after();
            const WindowStep *d = &s_steps[step % kStepSlots];
            const int keys = d->keys;
            if (keys == 0) {
                break;
            }
            const uint32_t flags = d->flags >> t;
            if ((flags & 1u) != 0) {
                uint32_t r[4][32];
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    if (32 * w < keys) {
                        tmem_load32(t_s + 32 * w, r[w]);
                    }
                }
                tmem_wait_loads();
                if ((flags & 16u) != 0) {
                    const int j0 = d->j0;
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        if (32 * w < keys) {
                            const uint32_t see = d->kept[w] & (range_bits(lo, hi, j0 + 32 * w) | range_bits(0, min(s.sinks, hi), j0 + 32 * w));
#pragma unroll
                            for (int e = 0; e < 32; ++e) {
                                r[w][e] = (see >> e & 1u) != 0 ? r[w][e] : 0xff800000u;
                            }
                        }
                    }
                }
                float m0 = -INFINITY, m1 = -INFINITY, m2 = -INFINITY, m3 = -INFINITY;
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    if (32 * w < keys) {
#pragma unroll
                        for (int e = 0; e < 32; e += 4) {
                            m0 = fmaxf(m0, __uint_as_float(r[w][e]));
                            m1 = fmaxf(m1, __uint_as_float(r[w][e + 1]));
                            m2 = fmaxf(m2, __uint_as_float(r[w][e + 2]));
                            m3 = fmaxf(m3, __uint_as_float(r[w][e + 3]));
                        }
                    }
                }
                const float here = fmaxf(fmaxf(m0, m1), fmaxf(m2, m3));
                const bool raise = (here - top) * c > kRaiseBy;   // the first visible key: infinity > 8
                float shrink = 1.f;
                if (raise) {
                    shrink = fast_exp2((top - here) * c);
                    top = here;
                }
                if (!first && __any_sync(0xffffffffu, raise)) {
                    // the products into O are done: they were issued before this step's scores
                    const float2 sh2 = splat2(shrink);
                    for (int x = 0; x < s.dim; x += 16) {
                        uint32_t o[16];
                        asm volatile(
                            "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
                            "tcgen05.wait::ld.sync.aligned;"
                            : "=r"(o[0]), "=r"(o[1]), "=r"(o[2]), "=r"(o[3]), "=r"(o[4]), "=r"(o[5]), "=r"(o[6]), "=r"(o[7]), "=r"(o[8]),
                              "=r"(o[9]), "=r"(o[10]), "=r"(o[11]), "=r"(o[12]), "=r"(o[13]), "=r"(o[14]), "=r"(o[15])
                            : "r"(t_o + x)
                            : "memory");
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
                const float2 c2 = splat2(c), nt2 = splat2(top == -INFINITY ? 0.f : -top * c);
                float2 sum0 = make_float2(0.f, 0.f), sum1 = make_float2(0.f, 0.f);
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    if (32 * w < keys) {
                        uint32_t p[16];
#pragma unroll
                        for (int e = 0; e < 32; e += 4) {
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
                        tmem_store16(t_s + 16 * w, p);
                    }
                }
                sum0 = add2(sum0, sum1);
                total = fmaf(total, shrink, sum0.x + sum0.y);
                tmem_wait_stores();
            }
            tmem_fence_before();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&s_pfull[t]);
            }
        }
        // ---- context rows (the last completion covers every product into O)
        const float inv = !ok ? NAN : (total == 0.f ? 0.f : 1.f / total);
        bool finite = true;
        __half *out = context + ((int64_t) b * s.seq + i) * s.context_stride + (int64_t) h * s.dim;
        const bool vec = (reinterpret_cast<uintptr_t>(context) & 15) == 0 && s.context_stride % 8 == 0;
        for (int x = 0; x < s.dim; x += 32) {
            uint32_t o[32];
            if (first) {   // no step took part
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                    o[e] = 0;
                }
            } else {
                tmem_load32(t_o + x, o);
                tmem_wait_loads();
            }
            uint32_t w[16];
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
                const float a = __uint_as_float(o[e]) * inv, z = __uint_as_float(o[e + 1]) * inv;
                if (x + e < s.dim) {   // columns past the dimension hold leftovers of another block
                    finite = finite && fabsf(a) <= 65504.f && fabsf(z) <= 65504.f;
                }
                const __half2 hv = __floats2half2_rn(a, z);
                w[e / 2] = *reinterpret_cast<const uint32_t *>(&hv);
            }
            if (i < s.seq) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (x + 8 * e < s.dim) {
                        if (vec) {
                            *reinterpret_cast<uint4 *>(out + x + 8 * e) = make_uint4(w[4 * e], w[4 * e + 1], w[4 * e + 2], w[4 * e + 3]);
                        } else {
                            const __half *hw = reinterpret_cast<const __half *>(&w[4 * e]);
#pragma unroll
                            for (int u = 0; u < 8; ++u) {
                                out[x + 8 * e + u] = hw[u];
                            }
                        }
                    }
                }
            }
        }
        unsigned bad = __ballot_sync(0xffffffffu, ok && i < s.seq && !finite);
        while (bad != 0) {
            const int from = __ffs(bad) - 1;
            bad &= bad - 1;
            window_row_again(q, k, v, mask, context, &s, s_row[warp], b, i - lane + from, h);
        }
    }
    tmem_fence_before();
    __syncthreads();
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

// [batch, heads, seq, dim] view of rows `stride` elements apart, read in boxes of 128 rows x 64 columns.
inline bool window_map(CUtensorMap *map, const __half *p, int dim, int seq, int heads, int batch, int64_t stride) {
    const EncodeTiled encode = encode_tiled();
    const cuuint64_t dims[4] = {(cuuint64_t) dim, (cuuint64_t) seq, (cuuint64_t) heads, (cuuint64_t) batch};
    const cuuint64_t strides[3] = {(cuuint64_t) stride * 2, (cuuint64_t) dim * 2, (cuuint64_t) seq * (cuuint64_t) stride * 2};
    const cuuint32_t box[4] = {64, kTileRows, 1, 1}, step[4] = {1, 1, 1, 1};
    if (encode == nullptr || !aligned16(p) || strides[0] % 16 != 0 || strides[1] % 16 != 0 || strides[0] >= (1ull << 40) || strides[2] >= (1ull << 40)) {
        return false;
    }
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<__half *>(p), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int DP, int NQ>
int window_tc_launch(const CUtensorMap &qm, const CUtensorMap &km, const CUtensorMap &vm, const __half *q, const __half *k, const __half *v,
                     const int8_t *mask, __half *context, const WindowShape &s, cudaStream_t stream) {
    typedef WindowTc<DP, NQ> C;
    static std::atomic<uint64_t> prepared{0};   // devices on which the kernel may use its shared memory
    int dev = 0;
    cudaError_t err = cudaGetDevice(&dev);
    if (err == cudaSuccess && (dev >= 64 || ((prepared.load(std::memory_order_acquire) >> dev) & 1ull) == 0)) {
        err = cudaFuncSetAttribute(window_tc_kernel<DP, NQ>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM_BYTES);
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
    const int64_t blocks = (int64_t) row_blocks * s.batch * (pair ? s.heads / 2 : s.heads);
    if (blocks > 0x7fffffffLL) {
        return CUBK_ERR_UNSUPPORTED;
    }
    window_tc_kernel<DP, NQ><<<(unsigned) blocks, C::THREADS, C::SMEM_BYTES, stream>>>(qm, km, vm, q, k, v, mask, context, s, row_blocks, pair);
    return check_launch();
}

// Binary16 on the tensor cores; CUBK_ERR_UNSUPPORTED where TMA cannot read the operands (rows or heads that do not start on
// 16-byte boundaries), the head dimension is above 128 or the scale is not positive (a row's largest score is then not its
// largest product): the caller takes another kernel.
inline int window_tc(const __half *q, const __half *k, const __half *v, const int8_t *mask, __half *context, const WindowShape &s,
                     cudaStream_t stream) {
    CUtensorMap qm, km, vm;
    if (s.dim > 128 || !(s.scale > 0.f) || !window_map(&qm, q, s.dim, s.seq, s.heads, s.batch, s.q_stride) ||
        !window_map(&km, k, s.dim, s.seq, s.kv_heads, s.batch, s.kv_stride) || !window_map(&vm, v, s.dim, s.seq, s.kv_heads, s.batch, s.kv_stride)) {
        return CUBK_ERR_UNSUPPORTED;
    }
    return s.dim <= 64 ? window_tc_launch<64, 1>(qm, km, vm, q, k, v, mask, context, s, stream)
                       : window_tc_launch<128, 2>(qm, km, vm, q, k, v, mask, context, s, stream);
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
    if constexpr (sizeof(T) == 2) {
        const int rc = window_tc(q, k, v, mask, context, s, stream);
        if (rc != CUBK_ERR_UNSUPPORTED) {
            return rc;
        }
    }
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
