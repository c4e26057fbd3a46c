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
#include "common.cuh"

namespace cubk {

constexpr int kW4Tile = 16;           // weight rows of a tile
constexpr int kW4Block = 128;         // columns of a tile
constexpr int kW4TileBytes = kW4Tile * kW4Block / 2;
constexpr int kW4Warps = 16;
constexpr int kW4Ahead = 2;           // pairs of tiles a warp has in flight

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

// (w & mask) | base in one instruction (left to itself the compiler makes two of it: one immediate operand too many).
__device__ __forceinline__ uint32_t and_or(uint32_t w, uint32_t mask, uint32_t base) {
    uint32_t d;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(d) : "r"(w), "r"(mask), "r"(base));
    return d;
}

// The eight codes of a word as four pairs of the operand type (exact).
template <bool BF16>
__device__ __forceinline__ void w4_expand(uint32_t w, uint32_t (&p)[4]) {
    if (BF16) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            asm("sub.bf16x2 %0, %1, %2;" : "=r"(p[i]) : "r"(and_or(w >> (4 * i), 0x000f000fu, 0x43004300u)), "r"(0x43084308u));   // 128 + c - 136
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
            const uint32_t v = i == 0 ? w : w >> 8;
            const uint32_t lo = and_or(v, 0x000f000fu, 0x64006400u), hi = and_or(v, 0x00f000f0u, 0x64006400u);
            asm("sub.f16x2 %0, %1, %2;" : "=r"(p[i]) : "r"(lo), "r"(0x64086408u));                                 // 1024 + c - 1032
            asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(p[i + 1]) : "r"(hi), "r"(0x2c002c00u), "r"(0xd480d480u));    // (1024 + 16 c) / 16 - 72
        }
    }
}

// The x operands of one lane: eight consecutive columns from k0 of a row, loaded as Raw and then brought into SPLITS sets of
// four pairs.
template <XKind X>
struct XLoad;

template <>
struct XLoad<X_F16> {
    typedef __half Elem;
    typedef uint4 Raw;
    static constexpr int SPLITS = 1, BATCH = 8;   // BATCH: loads of a thread in flight while x is laid out
    static constexpr bool BF16 = false;
    static __device__ __forceinline__ Raw load(const __half *row, int k0, int k, bool vec) {
        if (vec) {
            return ld_param(row + k0);
        }
        const unsigned short *r = reinterpret_cast<const unsigned short *>(row);
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t lo = k0 + 2 * i < k ? r[k0 + 2 * i] : 0, hi = k0 + 2 * i + 1 < k ? r[k0 + 2 * i + 1] : 0;
            w[i] = lo | hi << 16;
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    static __device__ __forceinline__ void operands(const Raw &v, uint32_t (&b)[1][4]) {
        b[0][0] = v.x, b[0][1] = v.y, b[0][2] = v.z, b[0][3] = v.w;
    }
};

template <>
struct XLoad<X_E4M3> {
    typedef uint8_t Elem;
    typedef uint2 Raw;
    static constexpr int SPLITS = 1, BATCH = 8;
    static constexpr bool BF16 = false;
    static __device__ __forceinline__ Raw load(const uint8_t *row, int k0, int k, bool vec) {
        if (vec) {
            return __ldg(reinterpret_cast<const uint2 *>(row + k0));
        }
        uint32_t w[2] = {0, 0};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (k0 + i < k) {
                w[i / 4] |= (uint32_t) row[k0 + i] << (8 * (i % 4));
            }
        }
        return make_uint2(w[0], w[1]);
    }
    static __device__ __forceinline__ void operands(const Raw &v, uint32_t (&b)[1][4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint16_t pair = (uint16_t) ((i < 2 ? v.x : v.y) >> (16 * (i % 2)));
            asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(b[0][i]) : "h"(pair));
        }
    }
};

template <>
struct XLoad<X_F32> {
    typedef float Elem;
    struct Raw {
        float v[8];
    };
    static constexpr int SPLITS = 3, BATCH = 4;
    static constexpr bool BF16 = true;
    static __device__ __forceinline__ Raw load(const float *row, int k0, int k, bool vec) {
        Raw r;
        if (vec && k0 + 8 <= k) {
            const float4 lo = __ldg(reinterpret_cast<const float4 *>(row + k0)), hi = __ldg(reinterpret_cast<const float4 *>(row + k0) + 1);
            r.v[0] = lo.x, r.v[1] = lo.y, r.v[2] = lo.z, r.v[3] = lo.w, r.v[4] = hi.x, r.v[5] = hi.y, r.v[6] = hi.z, r.v[7] = hi.w;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                r.v[i] = k0 + i < k ? row[k0 + i] : 0.f;
            }
        }
        return r;
    }
    // the top 16 bits of a float32 are a bfloat16 (of a NaN, only with its quiet bit set; without it they may be an infinity); what is left
    // of 24 bits of mantissa after two of them fits a third
    static __device__ __forceinline__ void operands(Raw r, uint32_t (&b)[3][4]) {
#pragma unroll
        for (int s = 0; s < 3; ++s) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (s == 0) {
                    r.v[2 * i] = quiet(r.v[2 * i]);
                    r.v[2 * i + 1] = quiet(r.v[2 * i + 1]);
                }
                b[s][i] = __byte_perm(__float_as_uint(r.v[2 * i]), __float_as_uint(r.v[2 * i + 1]), 0x7632);
                r.v[2 * i] = rest(r.v[2 * i]);
                r.v[2 * i + 1] = rest(r.v[2 * i + 1]);
            }
        }
    }
    static __device__ __forceinline__ float quiet(float v) {
        return v != v ? __uint_as_float(0x7fffffffu) : v;
    }
    static __device__ __forceinline__ float rest(float v) {
        const uint32_t top = __float_as_uint(v) & 0xffff0000u;
        return (top & 0x7f800000u) == 0x7f800000u ? 0.f : v - __uint_as_float(top);   // an infinity leaves nothing
    }
};

// What a block does; see w4_plan().
struct W4Plan {
    int kblocks;        // tiles along k
    int slice;          // of them whose x operands are in shared memory at a time
    int slices;
    int round;          // rows of tiles whose sums are carried from slice to slice
};

__device__ __forceinline__ void copy_async16(void *smem, const void *global) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_addr(smem)), "l"(__cvta_generic_to_global(global)) : "memory");
}

__device__ __forceinline__ void copy_async_commit() {
    asm volatile("cp.async.commit_group;" ::: "memory");
}

// `bytes` (2 or 4) of the four come from memory, the rest are zeros.
__device__ __forceinline__ void copy_async4(void *smem, const void *global, int bytes) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_addr(smem)), "l"(__cvta_generic_to_global(global)), "r"(bytes) : "memory");
}

template <int LEFT>
__device__ __forceinline__ void copy_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory");
}

template <typename T, XKind X, int TT, int GROUP>
struct W4Smem {
    // scales of a pair of tiles, 16 for each of their groups: for binary16 as words, which start one element early in every other row
    // of an odd n
    static constexpr int SCALE_WORDS = sizeof(T) == 2 ? 9 : 16, WORDS = 2 * kW4Block / GROUP * SCALE_WORDS;
    static constexpr int PAIR = 2 * kW4TileBytes, SCALE_SLOT = (4 * WORDS + 15) / 16 * 16, SCALE_SLOTS = 2 * kW4Ahead;
    static constexpr int WARP = kW4Ahead * PAIR + SCALE_SLOTS * SCALE_SLOT;
    static constexpr int RING = kW4Warps * WARP;
    static constexpr int JOIN = kW4Warps * 2 * TT * 32 * 16;                // over the ring, once it has run dry
    static constexpr int X_TILE = XLoad<X>::SPLITS * TT * 4 * 32 * 16;      // operands of 128 columns
    static constexpr int SCALES = X == X_E4M3 ? 8 * TT * 4 : 0;             // and the scales of their x rows
    static constexpr int CARRY = TT * 32 * 16;                              // sums of a row of tiles
    static constexpr int LIMIT = 227 * 1024 - RING;
    static_assert(JOIN <= RING, "the parts of split tiles fit into the ring");
};

// A block takes a range of rows of tiles; their tiles, two by two along k, are one list that its 16 warps cut into equal pieces,
// so that every warp streams one contiguous run of memory. Each lane copies its own 64 bytes of a pair into a ring that only its warp
// reads and refills a slot as soon as it has read it, so the weights' way from memory needs few registers and no barrier; x is
// brought into operand form once (per slice where it does not fit), so that a lane's operand is one conflict-free 16-byte read. A
// row of tiles that lies in one piece is finished by its warp; the parts of one that is cut meet in shared memory and are added
// in the order of the warps.
// Bound by issue, not by memory: 204 warp instructions per KB of codes at 16 rows of x, a third of them the expansion. 4096 by 30522,
// groups of 128: 24.8 us at 16 rows (2.6 TB/s), 17.3 at one (3.7 TB/s); per KB and SM 85 and 57 cycles, where memory alone would take 44.
// At k = 4096 and one row, 4.8 us do not grow with n (launch, x to operands, the first weights, the join); 768 by 2304 takes 4.3 in
// all. At 16 rows, as the kernel was built: scales loaded a tile ahead 48 us, through the ring 46; tiles dealt to the warps one by one
// 41, in contiguous runs 36; single tiles in flight 28.8, pairs 26.4; the expansion in two logic operations 26.4, in one 24.6.
template <typename T, XKind X, int TT, int GROUP>
__global__ void __launch_bounds__(32 * kW4Warps, 1)
w4_matvec_kernel(const typename XLoad<X>::Elem *x, const float *x_scales, int x_groups, int rows, int k, const uint8_t *packed,
                 const T *scales, int n, const T *bias, T *out, bool vec, const W4Plan plan) {
    typedef W4Smem<T, X, TT, GROUP> S;
    constexpr int SPLITS = XLoad<X>::SPLITS;
    constexpr bool BF16 = XLoad<X>::BF16;
    constexpr int STEPS = GROUP / 32, PER_TILE = kW4Block / GROUP;   // 32-column steps of a group, groups of a tile
    constexpr int PASSES = (S::WORDS + 31) / 32;                     // copies of a lane for a pair's scales
    extern __shared__ __align__(16) unsigned char w4_smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
    unsigned char *ring = w4_smem + warp * S::WARP, *scale_ring = ring + kW4Ahead * S::PAIR;
    float4 *join = reinterpret_cast<float4 *>(w4_smem);                               // [warp][2][TT][lane]
    uint4 *s_x = reinterpret_cast<uint4 *>(w4_smem + S::RING);                        // [tile][32-column step][split][TT][lane]
    float *s_xs = reinterpret_cast<float *>(w4_smem + S::RING + plan.slice * S::X_TILE);   // [tile][x row]
    float4 *carry = reinterpret_cast<float4 *>(w4_smem + S::RING + plan.slice * (S::X_TILE + S::SCALES));   // [row of tiles][TT][lane]
    const int row0 = blockIdx.y * (8 * TT);
    const int tiles = (n + kW4Tile - 1) / kW4Tile;
    const int tiles_begin = (int) ((int64_t) tiles * blockIdx.x / gridDim.x), tiles_end = (int) ((int64_t) tiles * (blockIdx.x + 1) / gridDim.x);
    const int last_group = (k - 1) / GROUP;
    // a finished row of tiles: c[m] holds weight rows g and g + 8, x rows 2 t and 2 t + 1 of block m
    auto finish = [&](int tile, int m, const float4 &c) {
        const float v[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int col = tile * kW4Tile + g + 8 * (i >> 1), row = row0 + 8 * m + 2 * t + (i & 1);
            if (col < n && row < rows) {
                out[(size_t) row * n + col] = from_float<T>(v[i] + (bias != nullptr ? to_float<T>(bias[col]) : 0.f));
            }
        }
    };

    for (int round = tiles_begin; round < tiles_end; round += plan.round) {
        const int round_tiles = min(plan.round, tiles_end - round);
        for (int sl = 0; sl < plan.slices; ++sl) {
            const int first = sl * plan.slice, len = min(plan.slice, plan.kblocks - first);
            const int pairs = (len + 1) / 2, total = round_tiles * pairs;
            const int begin = (int) ((int64_t) total * warp / kW4Warps), end = (int) ((int64_t) total * (warp + 1) / kW4Warps);
            // the list as this warp copies it: the next pair, and where its tiles and this lane's words of its scales lie
            int ahead = begin, ahead_tile = round + begin / pairs, ahead_pair = begin % pairs;
            const uint8_t *src = nullptr;
            const T *src_scales[PASSES];
            bool plain = false;   // no word of the scales reaches past the matrix
            auto start_tile = [&]() {
                src = packed + ((size_t) ahead_tile * plan.kblocks + first + 2 * ahead_pair) * kW4TileBytes + lane * 16;
#pragma unroll
                for (int p = 0; p < PASSES; ++p) {
                    src_scales[p] = scales + (size_t) ((first + 2 * ahead_pair) * PER_TILE + (32 * p + lane) / S::SCALE_WORDS) * n +
                                    ahead_tile * kW4Tile;
                }
                plain = n - ahead_tile * kW4Tile >= 18;
            };
            auto fetch = [&](int slot) {
                if (ahead < end) {
                    unsigned char *to = ring + slot * S::PAIR + lane * 16;
                    copy_async16(to, src);
                    copy_async16(to + 512, src + 512);
                    if (2 * ahead_pair + 1 < len) {
                        copy_async16(to + 1024, src + 1024);
                        copy_async16(to + 1536, src + 1536);
                    }
                    unsigned char *to_scales = scale_ring + (ahead - begin) % S::SCALE_SLOTS * S::SCALE_SLOT;
#pragma unroll
                    for (int p = 0; p < PASSES; ++p) {
                        const int w = 32 * p + lane, word = w % S::SCALE_WORDS;
                        const int row = (first + 2 * ahead_pair) * PER_TILE + w / S::SCALE_WORDS;
                        if ((S::WORDS % 32 == 0 || w < S::WORDS) && row <= last_group) {
                            const T *at = src_scales[p];
                            int left = 2;   // scales of this row from the word on
                            if (sizeof(T) == 2) {
                                const int early = (int) (reinterpret_cast<uintptr_t>(at) >> 1 & 1);
                                at += 2 * word - early;
                                left = plain ? 2 : n - ahead_tile * kW4Tile - (2 * word - early);
                            } else {
                                at += word;
                                left = plain ? 2 : 2 * (n - ahead_tile * kW4Tile - word);
                            }
                            if (left > 0) {
                                copy_async4(to_scales + 4 * w, at, left == 1 ? 2 : 4);
                            }
                        }
                    }
                    ++ahead;
                    src += 2 * kW4TileBytes;
#pragma unroll
                    for (int p = 0; p < PASSES; ++p) {
                        src_scales[p] += (size_t) n * (2 * PER_TILE);
                    }
                    if (++ahead_pair == pairs) {
                        ahead_pair = 0;
                        ++ahead_tile;
                        start_tile();
                    }
                }
                copy_async_commit();
            };
            start_tile();
            for (int i = 0; i < kW4Ahead; ++i) {
                fetch(i);
            }
            if (plan.slices > 1 || round == tiles_begin) {
                // the operands of the slice before are no longer read: the joins below end in a barrier
                constexpr int THREADS = 32 * kW4Warps, BATCH = XLoad<X>::BATCH;
                for (int i0 = threadIdx.x; i0 < len * 4 * TT * 32; i0 += THREADS * BATCH) {
                    typename XLoad<X>::Raw raw[BATCH];
#pragma unroll
                    for (int u = 0; u < BATCH; ++u) {
                        const int i = i0 + u * THREADS, l = i & 31, m = (i >> 5) % TT, step = (i >> 5) / TT;
                        const int row = row0 + 8 * m + (l >> 2), k0 = first * kW4Block + 32 * step + 8 * (l & 3);
                        raw[u] = typename XLoad<X>::Raw{};
                        if (step < 4 * len && row < rows && k0 < k) {
                            raw[u] = XLoad<X>::load(x + (size_t) row * k, k0, k, vec);
                        }
                    }
#pragma unroll
                    for (int u = 0; u < BATCH; ++u) {
                        const int i = i0 + u * THREADS, l = i & 31, m = (i >> 5) % TT, step = (i >> 5) / TT;
                        uint32_t b[SPLITS][4];
                        XLoad<X>::operands(raw[u], b);
                        if (step < 4 * len) {
#pragma unroll
                            for (int p = 0; p < SPLITS; ++p) {
                                s_x[((step * SPLITS + p) * TT + m) * 32 + l] = make_uint4(b[p][0], b[p][1], b[p][2], b[p][3]);
                            }
                        }
                    }
                }
                if (X == X_E4M3) {
                    for (int i = threadIdx.x; i < len * 8 * TT; i += 32 * kW4Warps) {
                        const int row = row0 + i % (8 * TT), kb = first + i / (8 * TT);
                        s_xs[i] = row < rows ? x_scales[(size_t) row * x_groups + (x_groups > 1 ? kb : 0)] : 0.f;
                    }
                }
                __syncthreads();
            }

            // a part of a row of tiles that another warp has begun is kept for the join in slot 0, one that another will end in slot 1
            float4 kept[2][TT];
            int slot = 0;
            int tile = begin / pairs, pair = begin - tile * pairs;
            for (int at = begin; at < end;) {
                float acc[TT][4];
#pragma unroll
                for (int m = 0; m < TT; ++m) {
                    acc[m][0] = acc[m][1] = acc[m][2] = acc[m][3] = 0.f;
                }
                const bool begun = pair != 0;
                const int stop = min(pairs, pair + end - at);
                const uint4 *xt = s_x + (size_t) pair * 8 * SPLITS * TT * 32 + lane;
                for (; pair < stop; ++pair, ++at) {
                    copy_async_wait<kW4Ahead - 1>();
                    __syncwarp();   // the scales were copied by other lanes
                    const unsigned char *from = ring + slot * S::PAIR + lane * 16;
                    uint32_t words[2][2][4];   // tile, rows g and g + 8, 32-column step
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint4 r = ld_shared_vec(from + 512 * i);
                        words[i / 2][i % 2][0] = r.x, words[i / 2][i % 2][1] = r.y, words[i / 2][i % 2][2] = r.z, words[i / 2][i % 2][3] = r.w;
                    }
                    const T *pair_scales = reinterpret_cast<const T *>(scale_ring + (at - begin) % S::SCALE_SLOTS * S::SCALE_SLOT) + g;
                    fetch(slot);   // into the slot just read; the scales' ring is twice as long
                    slot = slot == kW4Ahead - 1 ? 0 : slot + 1;
                    float sum[TT][4];
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        if (j == 4 && 2 * pair + 1 >= len) {
                            break;
                        }
                        if (j % STEPS == 0) {
#pragma unroll
                            for (int m = 0; m < TT; ++m) {
                                sum[m][0] = sum[m][1] = sum[m][2] = sum[m][3] = 0.f;
                            }
                        }
                        uint32_t pa[4], pb[4];
                        w4_expand<BF16>(words[j / 4][0][j % 4], pa);
                        w4_expand<BF16>(words[j / 4][1][j % 4], pb);
                        const uint32_t a0[4] = {pa[0], pb[0], pa[1], pb[1]}, a1[4] = {pa[2], pb[2], pa[3], pb[3]};
#pragma unroll
                        for (int m = 0; m < TT; ++m) {
#pragma unroll
                            for (int p = SPLITS - 1; p >= 0; --p) {
                                const uint4 b = xt[((j * SPLITS + p) * TT + m) * 32];
                                w4_mma<BF16>(sum[m], a0, b.x, b.y);
                                w4_mma<BF16>(sum[m], a1, b.z, b.w);
                            }
                        }
                        if ((j + 1) % STEPS == 0) {
                            const int row = (first + 2 * pair) * PER_TILE + j / STEPS;
                            const T *sc = pair_scales + j / STEPS * (S::SCALE_WORDS * 4 / (int) sizeof(T));
                            if (sizeof(T) == 2) {   // the copy began one element early where the row starts in the middle of a word
                                sc += row & n & 1;
                            }
                            const bool real = PER_TILE == 1 || row <= last_group;   // groups past k: no scale was copied
                            const float ga = real ? to_float<T>(sc[0]) : 0.f, gb = real ? to_float<T>(sc[8]) : 0.f;
#pragma unroll
                            for (int m = 0; m < TT; ++m) {
                                if (X == X_E4M3) {
                                    const float2 xs = *reinterpret_cast<const float2 *>(&s_xs[(2 * pair + j / 4) * 8 * TT + 8 * m + 2 * t]);
                                    sum[m][0] *= xs.x, sum[m][1] *= xs.y, sum[m][2] *= xs.x, sum[m][3] *= xs.y;
                                }
                                acc[m][0] = fmaf(sum[m][0], ga, acc[m][0]);
                                acc[m][1] = fmaf(sum[m][1], ga, acc[m][1]);
                                acc[m][2] = fmaf(sum[m][2], gb, acc[m][2]);
                                acc[m][3] = fmaf(sum[m][3], gb, acc[m][3]);
                            }
                        }
                    }
                    xt += 8 * SPLITS * TT * 32;
                }
#pragma unroll
                for (int m = 0; m < TT; ++m) {
                    float4 c = make_float4(acc[m][0], acc[m][1], acc[m][2], acc[m][3]);
                    if (begun) {
                        kept[0][m] = c;
                    } else if (pair < pairs) {
                        kept[1][m] = c;
                    } else {
                        float4 *sums = carry + (tile * TT + m) * 32 + lane;
                        if (sl > 0) {
                            const float4 old = *sums;
                            c.x += old.x, c.y += old.y, c.z += old.z, c.w += old.w;
                        }
                        if (sl == plan.slices - 1) {
                            finish(round + tile, m, c);
                        } else {
                            *sums = c;
                        }
                    }
                }
                if (pair == pairs) {
                    pair = 0;
                    ++tile;
                }
            }
            __syncthreads();   // the ring has run dry; so have the operands, for the next slice
#pragma unroll
            for (int i = 0; i < 2; ++i) {
#pragma unroll
                for (int m = 0; m < TT; ++m) {
                    join[((warp * 2 + i) * TT + m) * 32 + lane] = kept[i][m];   // slots without a part are not read
                }
            }
            __syncthreads();
            for (int i = warp; i < round_tiles * TT; i += kW4Warps) {
                const int joined = i / TT, m = i % TT;
                const int w1 = (int) (((int64_t) (joined * pairs + 1) * kW4Warps - 1) / total);               // the warp of its first pair
                const int w2 = (int) (((int64_t) (joined * pairs + pairs) * kW4Warps - 1) / total);           // and of its last
                if (w1 == w2) {
                    continue;
                }
                float4 c = join[((w1 * 2 + 1) * TT + m) * 32 + lane];
                for (int w = w1 + 1; w <= w2; ++w) {
                    if (((int64_t) total * w / kW4Warps) == ((int64_t) total * (w + 1) / kW4Warps)) {
                        continue;   // more warps than pairs: this one had none
                    }
                    const float4 a = join[(w * 2 * TT + m) * 32 + lane];
                    c.x += a.x, c.y += a.y, c.z += a.z, c.w += a.w;
                }
                float4 *sums = carry + i * 32 + lane;
                if (sl > 0) {
                    const float4 old = *sums;
                    c.x += old.x, c.y += old.y, c.z += old.z, c.w += old.w;
                }
                if (sl == plan.slices - 1) {
                    finish(round + joined, m, c);
                } else {
                    *sums = c;
                }
            }
            __syncthreads();
        }
    }
}

// All of x in shared memory where it fits, and then a block's rows of tiles in one round; else slices of k, with the sums of 16
// rows of tiles carried between them (x is loaded again for every 16 rows of tiles then: 8 TT rows of x against 256 of weights).
inline W4Plan w4_plan(int k, int limit, int per_tile, int carry) {
    W4Plan p;
    p.kblocks = (k + kW4Block - 1) / kW4Block;
    p.slice = p.kblocks;
    p.slices = 1;
    p.round = 1 << 30;
    if ((int64_t) p.kblocks * per_tile > limit) {
        p.round = 16;
        const int most = (limit - p.round * carry) / per_tile;
        p.slices = (p.kblocks + most - 1) / most;
        p.slice = (p.kblocks + p.slices - 1) / p.slices;
        p.slice += p.slice < most ? p.slice % 2 : 0;   // whole pairs
        p.slices = (p.kblocks + p.slice - 1) / p.slice;
    }
    return p;
}

template <typename T, XKind X, int TT, int GROUP>
int w4_matvec_launch(const typename XLoad<X>::Elem *x, const float *x_scales, int x_groups, int rows, int k, const void *packed,
                     const T *scales, int n, const T *bias, T *out, bool vec, cudaStream_t stream) {
    typedef W4Smem<T, X, TT, GROUP> S;
    static OccupancyCache cache;
    // one block per SM, by its registers; asked with all of the shared memory so that the answer holds for every plan
    const int resident = resident_blocks(w4_matvec_kernel<T, X, TT, GROUP>, 32 * kW4Warps, 227 * 1024, &cache, true);
    if (resident <= 0) {
        set_last_error(cudaErrorLaunchOutOfResources);
        return CUBK_ERR_LAUNCH;
    }
    const W4Plan plan = w4_plan(k, S::LIMIT, S::X_TILE + S::SCALES, S::CARRY);
    const int smem = S::RING + plan.slice * (S::X_TILE + S::SCALES) + (plan.slices > 1 ? plan.round * S::CARRY : 0);
    const int tiles = (n + kW4Tile - 1) / kW4Tile;
    // one wave: blocks of different rows read the same codes at the same time (64 x 4096 by 11008 with a wave per 32 rows 63.1 us, in one 44.5)
    const int row_blocks = (rows + 8 * TT - 1) / (8 * TT), across = resident / row_blocks > 1 ? resident / row_blocks : 1;
    const dim3 grid((unsigned) (tiles < across ? tiles : across), (unsigned) row_blocks);
    w4_matvec_kernel<T, X, TT, GROUP><<<grid, 32 * kW4Warps, smem, stream>>>(x, x_scales, x_groups, rows, k, (const uint8_t *) packed, scales,
                                                                             n, bias, out, vec, plan);
    return check_launch();
}

// Eight rows of x a block, or sixteen (one more product per expanded code; 16 x 4096 by 30522: 24.8 us). Eight also where their blocks
// make one wave, so that more SMs share the laying out of x (24 x 6144 by 139: 30.3 us in blocks of 32 rows, 8.1 in blocks of eight), and
// where sixteen rows of x do not fit into shared memory at once and eight do (16 x 8192 by 8192: 22.7 and 20.2). More than
// sixteen are slower at every size tried: 64 x 4096 by 11008 44.5 us by 32 rows, 30.8 by 16; 32 x 768 by 2304 6.0 and 4.5.
template <typename T, XKind X, int GROUP>
int w4_matvec_rows(const typename XLoad<X>::Elem *x, const float *x_scales, int x_groups, int rows, int k, const void *packed,
                   const T *scales, int n, const T *bias, T *out, bool vec, cudaStream_t stream) {
    const int64_t tiles = (n + kW4Tile - 1) / kW4Tile, kblocks = (k + kW4Block - 1) / kW4Block, eights = ((int64_t) rows + 7) / 8;
    typedef W4Smem<T, X, 1, GROUP> One;
    typedef W4Smem<T, X, 2, GROUP> Two;
    const bool only_eight_fit = kblocks * (Two::X_TILE + Two::SCALES) > Two::LIMIT && kblocks * (One::X_TILE + One::SCALES) <= One::LIMIT;
    if (rows <= 8 || tiles * eights <= 148 || (only_eight_fit && eights <= 65535)) {
        return w4_matvec_launch<T, X, 1, GROUP>(x, x_scales, x_groups, rows, k, packed, scales, n, bias, out, vec, stream);
    }
    return w4_matvec_launch<T, X, 2, GROUP>(x, x_scales, x_groups, rows, k, packed, scales, n, bias, out, vec, stream);
}

template <typename T, XKind X>
int w4_matvec(const typename XLoad<X>::Elem *x, const float *x_scales, int x_group, int rows, int k, const void *packed,
              const T *scales, int group, int n, const T *bias, T *out, cudaStream_t stream) {
    if (x == nullptr || packed == nullptr || scales == nullptr || out == nullptr || rows < 0 || k <= 0 || n <= 0 ||
        (group != 32 && group != 64 && group != 128) || (X == X_E4M3 && (x_scales == nullptr || (x_group != 0 && x_group != 128)))) {
        return CUBK_ERR_INVALID_ARG;
    }
    if (!aligned16(packed) || (reinterpret_cast<uintptr_t>(scales) & 3u) != 0 || ((int64_t) rows + 15) / 16 > 65535 || k > (1 << 30) || n > (1 << 30)) {
        return CUBK_ERR_UNSUPPORTED;
    }
    if (rows == 0) {
        return CUBK_OK;
    }
    constexpr int kLane = 8 * (int) sizeof(*x);   // bytes of a lane's eight columns
    // whole vectors: of eight columns, of float32 four
    const bool vec = k % (X == X_F32 ? 4 : 8) == 0 && reinterpret_cast<uintptr_t>(x) % (kLane < 16 ? kLane : 16) == 0;
    const int x_groups = X == X_E4M3 && x_group != 0 ? (k + kW4Block - 1) / kW4Block : 1;
#define W4(GROUP) w4_matvec_rows<T, X, GROUP>(x, x_scales, x_groups, rows, k, packed, scales, n, bias, out, vec, stream)
    return group == 32 ? W4(32) : group == 64 ? W4(64) : W4(128);
#undef W4
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

// Codes by rounding to nearest even under the group's scale = max|w| / 7, rounded to the storage type first. A group that holds a NaN
// or an infinity gets a scale that is not finite and codes 0, so that its products are NaN.
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
        top = max_nan(top, fabsf(v[e]));
    }
    for (int o = 1; o < group / 8; o <<= 1) {
        top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
    }
    const T stored = from_float<T>(top / 7.f);
    const float scale = to_float<T>(stored);
    int c[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float q = scale > 0.f && scale < INFINITY ? rintf(v[e] / scale) : 0.f;
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
    w.kblocks = (int) (((int64_t) k + kW4Block - 1) / kW4Block);
    w.words = ((int64_t) n + kW4Tile - 1) / kW4Tile * kW4Tile * w.kblocks * 16;   // a multiple of 256
    w.ok = w.words / 256 <= 0x7fffffffLL && n <= (1 << 30) && k <= (1 << 30);
    w.blocks = (unsigned) (w.words / 256);
    return w;
}

template <typename T>
int w4_quantize(const T *weights, int n, int k, int group, void *packed, T *scales, cudaStream_t stream) {
    if (weights == nullptr || packed == nullptr || scales == nullptr || n <= 0 || k <= 0 ||
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
    if (codes == nullptr || packed == nullptr || n <= 0 || k <= 0) {
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
