// Products with 4-bit weights:  y[t, n] = sum_g sw[g, n] sx[g, t] sum_{k in group g} qw[n, k] qx[t, k].
//
// Rows qx are 8-bit with a scale per 128 elements (rows8.cu); a weight's elements are -8 .. 7 in 4 bits with a bf16 scale per 128 elements of
// a feature.  A word of four bytes holds eight elements: byte i element i in its lower half and element i + 4 in its upper one, so that
// two masks give two words of four bytes in the order in which the rows lie.  Both are padded with zeros to a multiple of 128 elements.
// The inner sums are exact (32-bit integers: |sum| <= 16 * 8 * 127 * 128 < 2^21, a weight's half byte stays in the upper half of its byte, which
// makes it sixteen times as large and spares the sign's extension), the outer ones in float: by ascending group in each of a CTA's sets of warps
// (one, or two that take the stages in turn), then over the sets and over the CTAs that share a tile's K, in order.
//
// Bound: up to eight rows the weights' bytes (1 x 3,584 x 37,888 in 13.3 us, 5.1 TB/s of packed weights; 8 x 5,120 x 27,648 14.8).  From there to 64 rows no unit of
// an SM is near its limit (24 x 5,120 x 27,648 17.2 us: issue slots 43 %, DRAM 39, tensor pipe 32, ALU 29; 64 x 3,584 x 37,888 24.0): the warps wait, on each other's
// stages by the look of it.  Above, each group's conversion and scaling, two operations or three for every sum of 128 products, beside the matrix instructions,
// which take a quarter of the time (2,048 x 3,584 x 37,888 in 483 to 509 us, by the GPU and how long it has been at it).  Below 10 us what a launch takes to
// start and to meet shows (1 x 3,584 x 4,608: 4.7 us, its bytes 1.3).  A weight that is not settled (read after the kernels in front) takes a microsecond
// more: 1 x 3,584 x 4,608 5.8, 24 x 5,120 x 27,648 18.7, 8 x 18,944 x 3,584 12.5 against 11.8.
#include <cooperative_groups.h>

#include "tensor_core.cuh"

namespace {
namespace cg = cooperative_groups;
constexpr int GROUP = 128;

__device__ __forceinline__ void mma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t lower(uint32_t w) { return (w << 4) & 0xf0f0f0f0u; }
__device__ __forceinline__ uint32_t upper(uint32_t w) { return w & 0xf0f0f0f0u; }

struct W4Params {
    const uint8_t* rows;          // [M][128 G] signed bytes
    const float* row_scales;      // [G], stride ld_scales
    long long ld_scales;
    const uint8_t* packed;        // [N][64 G]
    const __nv_bfloat16* scales;  // [G][N]
    void* out;                    // [M][N]
    int M, N, G;
    int ahead;                    // the weight may be read before the kernels in front have ended: all that wrote it had ended before this launch
    int* err_flag;
};

constexpr int ERR_TIMEOUT = 2;
constexpr int FEATURES = 128, W_BYTES = FEATURES * GROUP / 2;      // of a tile

__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* err_flag) {
    return mbar_wait_or<ERR_TIMEOUT>(bar, parity, abort_flag, err_flag);
}
// ... that does not look at the abort flag: for copies and MMAs in flight, before the CTA gives its memory back.
__device__ __forceinline__ void mbar_drain(uint32_t bar, uint32_t parity) {
    const long long t0 = clock64();
    while (!mbar_try_wait(bar, parity) && clock64() - t0 < PYRE_WAIT_CYCLES) {}
}

// What the CTAs of a cluster hold of the tile of F features from f0 and `tokens` tokens from t0 on, SETS times [token][F + 4] floats each (`stride` apart, at
// the start of shared memory), added up in order.  (A row of F + 4: what a warp stores at once falls on different banks.)
template <int SETS, int F, typename T>
__device__ __forceinline__ void add_shares(const W4Params& p, uint8_t* gen, int stride, bool failed, int f0, int t0, int tokens) {
    cg::cluster_group cluster = cg::this_cluster();
    const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    if (C > 1) cluster.sync();
    if (!failed) {      // (a CTA that gave up raised the error word: what the others write is not looked at)
        const bool vec = p.N % 4 == 0 && !((uintptr_t)p.out & (4 * sizeof(T) - 1));
        for (int i = rank * blockDim.x + threadIdx.x; i < tokens * (F / 4); i += C * blockDim.x) {
            const int t = i / (F / 4), f = i % (F / 4) * 4;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int q = 0; q < C; ++q) {
                const float* const sums = reinterpret_cast<const float*>(C > 1 ? cluster.map_shared_rank(gen, q) : gen) + t * (F + 4) + f;
#pragma unroll
                for (int e = 0; e < SETS; ++e) {
                    const float4 a = *reinterpret_cast<const float4*>(sums + e * stride);
                    v.x += a.x;
                    v.y += a.y;
                    v.z += a.z;
                    v.w += a.w;
                }
            }
            T* const out = (T*)p.out + (size_t)(t0 + t) * p.N + f0 + f;
            const Vec<T, 4> rounded = {from_f32<T>(v.x), from_f32<T>(v.y), from_f32<T>(v.z), from_f32<T>(v.w)};
            if (vec) {
                if (f0 + f < p.N) store_vec<T, 4>(out, rounded);
            } else
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (f0 + f + k < p.N) out[k] = rounded.v[k];
        }
    }
    if (C > 1) cluster.sync();      // the others' sums are read
}

// ---------------------------------------------------------------------------
// Few rows: a stream of weights from memory.  A CTA owns F features (128 or 96) and up to 8 NT tokens; the CTAs of a cluster share a tile's K.
//   two last warps     : one thread, TMA.  Two groups of 128 k at a time into a ring of STAGES: the weights as they are packed, the tokens' bytes.  (A copy of one group
//                        has rows of 64 bytes, which hold up its engine.)  And the
//                        groups' scales, of the features (a sixteenth of them: the integers are sixteen times as large) and of the tokens.
//   the others         : two sets of F / 32 that take the stages in turn; a warp owns 32 features.  Lane l holds 32 neighbouring elements (the l % 4th quarter
//                        of the group) of four features and of token l / 4: which k an MMA step sums over is free as long as both
//                        operands agree.
// The sets' and the cluster's shares meet in shared memory and are added in order.
// ---------------------------------------------------------------------------
constexpr int STREAM_STAGES = 4, PAIR = 2;

template <int NT, int F> struct Stream {
    static constexpr int WARPS = F / 32, THREADS = (2 * WARPS + 2) * 32, ROW = F + 4, W_BYTES = F * GROUP / 2;      // of a set; ...; a token's sums (see below); a group's
    static constexpr int X_BYTES = NT * 8 * GROUP;                                                    // a group's
    static constexpr int STAGE = PAIR * (W_BYTES + X_BYTES);                                          // multiples of 1,024: the swizzles' patterns
    static constexpr int SCALES = STREAM_STAGES * STAGE, SCALE = (F + NT * 8) * 4;             // [stage][group][features, tokens] floats
    static constexpr int BARS = SCALES + STREAM_STAGES * PAIR * SCALE;
    static constexpr int TOTAL = BARS + STREAM_STAGES * 16 + 16 + 1024;
    static_assert(2 * NT * 8 * ROW * 4 <= SCALES && 2 * (TOTAL + 1024) <= 233472 && STREAM_STAGES % 2 == 0, "the sets' sums take the ring's place; two CTAs");
};

template <int NT, int F, typename T>
__global__ void __launch_bounds__(2 * F + 64, 2)
w4_stream_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const W4Params p) {
    using L = Stream<NT, F>;
    constexpr int W_BYTES = L::W_BYTES, WARPS = L::WARPS, ROW = L::ROW;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* gen = smem_raw + (base - smem_u32(smem_raw));
    const uint32_t full = base + L::BARS, empty = full + 8 * STREAM_STAGES;
    volatile int* abort_flag = reinterpret_cast<volatile int*>(gen + L::BARS + 16 * STREAM_STAGES);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    cg::cluster_group cluster = cg::this_cluster();
    const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int f0 = blockIdx.x / C * F, t0 = blockIdx.y * NT * 8;
    const int first = (int)((long long)rank * p.G / C), n = (int)((rank + 1ll) * p.G / C) - first, steps = (n + PAIR - 1) / PAIR;      // four groups at least

    if (threadIdx.x == 0) {
        *abort_flag = 0;
        for (int s = 0; s < STREAM_STAGES; ++s) { mbar_init(full + 8 * s, 2); mbar_init(empty + 8 * s, WARPS); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    pdl_trigger();
    bool ok = true;
    if (warp == 2 * WARPS) {
        if (lane == 0) {
            asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_w)) : "memory");
            asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_x)) : "memory");
            const int early = min(steps, STREAM_STAGES);
            int asked = 0;
            if (!p.ahead) pdl_wait();
            auto weights = [&](int i) {
                const int s = i % STREAM_STAGES;
                mbar_expect_tx(full + 8 * s, L::STAGE);
                tma_load_2d(base + s * L::STAGE, &map_w, full + 8 * s, (first + PAIR * i) * (GROUP / 2), f0);
            };
            for (int i = 0; i < early; ++i) weights(i);
            pdl_wait();
            for (int i = 0; i < steps; ++i) {
                const int s = i % STREAM_STAGES;
                if (i >= early) {
                    if (!(ok = mbar_wait(empty + 8 * s, ((i / STREAM_STAGES) & 1) ^ 1, abort_flag, p.err_flag))) break;
                    weights(i);
                }
                for (int h = 0; h < PAIR; ++h)      // (beyond the last group: zeros)
                    tma_load_2d(base + s * L::STAGE + PAIR * W_BYTES + h * L::X_BYTES, &map_x, full + 8 * s, (first + PAIR * i + h) * GROUP, t0);
                asked = i + 1;
            }
            // the copies end before the CTA does, also where a reader's wait ran out after this thread had asked for the last of them
            for (int i = max(0, asked - STREAM_STAGES); i < asked; ++i) mbar_drain(full + 8 * (i % STREAM_STAGES), (i / STREAM_STAGES) & 1);
        }
    } else if (warp == 2 * WARPS + 1) {
        constexpr int BATCH = 4;
        static_assert(BATCH % PAIR == 0 && NT <= 4, "whole stages, a lane per token");
        bool waited = false;
        if (!p.ahead) { pdl_wait(); waited = true; }
        for (int i0 = 0; i0 < n && ok; i0 += BATCH) {
            float v[BATCH][WARPS], x[BATCH];
#pragma unroll
            for (int j = 0; j < BATCH; ++j)
#pragma unroll
                for (int q = 0; q < WARPS; ++q)
                    v[j][q] = __bfloat162float(p.scales[(size_t)(first + min(i0 + j, n - 1)) * p.N + min(f0 + q * 32 + lane, p.N - 1)]) * 0.0625f;
            if (!waited) pdl_wait();
            waited = true;
#pragma unroll
            for (int j = 0; j < BATCH; ++j) x[j] = p.row_scales[(size_t)(first + min(i0 + j, n - 1)) * p.ld_scales + min(t0 + lane, p.M - 1)];
#pragma unroll
            for (int j = 0; j < BATCH; ++j) {
                const int i = (i0 + j) / PAIR, s = i % STREAM_STAGES;
                if (i >= steps) break;
                if (j % PAIR == 0) {
                    ok = mbar_wait(empty + 8 * s, ((i / STREAM_STAGES) & 1) ^ 1, abort_flag, p.err_flag) && ok;
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                }
                float* const to = reinterpret_cast<float*>(gen + L::SCALES + (s * PAIR + j % PAIR) * L::SCALE);
#pragma unroll
                for (int q = 0; q < WARPS; ++q) to[q * 32 + lane] = v[j][q];
                if (lane < NT * 8) to[F + lane] = x[j];
                if (j % PAIR == PAIR - 1) {
                    __syncwarp();
                    if (lane == 0) mbar_arrive(full + 8 * s);
                }
            }
        }
        if (!waited) pdl_wait();
    } else {
        const int set = warp / WARPS, row0 = warp % WARPS * 32, quad = lane >> 2, c = lane & 3;
        // The feature of a lane among eight: neighbouring lanes of four read rows four apart, whose swizzles are different.
        const int row8 = (quad >> 1) | (quad & 1) << 2;
        float total[NT][2][4] = {};
        pdl_wait();      // no bounded wait should have to last as long as the kernels before
        for (int i = set; i < steps; i += 2) {
            const int s = i % STREAM_STAGES;
            ok = mbar_wait(full + 8 * s, (i / STREAM_STAGES) & 1, abort_flag, p.err_flag);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            const uint8_t* const stage = gen + s * L::STAGE;
            const int groups = min(PAIR, n - PAIR * i);
            for (int g = 0; g < groups; ++g) {
                // features row8 + 0, 8, 16, 24: the lower and the upper halves of 16 bytes
                uint32_t lo[4][4], hi[4][4];
#pragma unroll
                for (int q = 0; q < 4; ++q) {      // 128-byte swizzle: a chunk of 16 bytes by bits 7 to 9
                    const uint4 w = *reinterpret_cast<const uint4*>(stage + (row0 + q * 8 + row8) * 128 + (((4 * g + c) ^ row8) << 4));
                    const uint32_t word[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) { lo[q][j] = lower(word[j]); hi[q][j] = upper(word[j]); }
                }
                const float* const scales = reinterpret_cast<const float*>(gen + L::SCALES + (s * PAIR + g) * L::SCALE);
                float sw[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) sw[q] = scales[row0 + q * 8 + row8];
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const uint8_t* const src = stage + PAIR * W_BYTES + g * L::X_BYTES + (t * 8 + quad) * GROUP;
                    const uint4 x0 = *reinterpret_cast<const uint4*>(src + (((2 * c) ^ quad) << 4));
                    const uint4 x1 = *reinterpret_cast<const uint4*>(src + (((2 * c + 1) ^ quad) << 4));
                    const uint32_t x[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
                    const float2 sx = *reinterpret_cast<const float2*>(scales + F + t * 8 + 2 * c);
                    int d[2][4] = {};
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int h = 0; h < 2; ++h) mma_s8(d[h], lo[2 * h][j], lo[2 * h + 1][j], hi[2 * h][j], hi[2 * h + 1][j], x[2 * j], x[2 * j + 1]);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        total[t][h][0] = fmaf((float)d[h][0] * sx.x, sw[2 * h], total[t][h][0]);
                        total[t][h][1] = fmaf((float)d[h][1] * sx.y, sw[2 * h], total[t][h][1]);
                        total[t][h][2] = fmaf((float)d[h][2] * sx.x, sw[2 * h + 1], total[t][h][2]);
                        total[t][h][3] = fmaf((float)d[h][3] * sx.y, sw[2 * h + 1], total[t][h][3]);
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(empty + 8 * s);
        }
        // [set][token][feature]; the ring is free once both sets are through it
        asm volatile("bar.sync 1, %0;" ::"n"(2 * F) : "memory");
        float* const sums = reinterpret_cast<float*>(gen) + set * NT * 8 * ROW;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int e = 0; e < 4; ++e) sums[(t * 8 + 2 * c + (e & 1)) * ROW + row0 + h * 16 + (e >> 1) * 8 + row8] = total[t][h][e];
    }
    const bool failed = __syncthreads_or(!ok);
    add_shares<2, F, T>(p, gen, NT * 8 * ROW, failed, f0, t0, min(NT * 8, p.M - t0));
}

// ---------------------------------------------------------------------------
// Many rows, on the 5th-generation tensor cores.  A CTA owns 128 features (the MMA's rows) and TN tokens and takes a group of 128 k at a time:
//   warps 0, 3, a thread each : TMA.  The tokens' bytes of a group (TN x 128) into one ring, its weights as they are packed (128 x 64) into another.
//   warps 4..7         : a thread owns a feature: 64 bytes of a group to 128 (two masks and a shift per eight), stored to tensor memory, which
//                        is where the MMAs take their A operand from.
//   warp 1, one thread : four MMAs (kind::i8, 32 k each) a group, into one of two accumulators of 32-bit integers.
//   warp 2             : the scales of four groups at a time, of features and of tokens, to shared memory.
//   warps 8 to the last: a thread owns a feature and 32 of the tokens.  The group's integers come out of tensor memory, are scaled by token and by
//                        feature and added to float sums in registers, by ascending group.
// Where there are few tiles the CTAs of a cluster share a tile's K, and their sums meet in shared memory.
// Bound by the last warps: of 483 us (on the fastest GPU, as all figures here) for 2,048 x 3,584 x 37,888 some 200 go with the conversions, products and additions (with a quarter of them it takes 349), 48 with
// the reads of the tokens' scales; a quarter of the MMAs or no unpacking changes nothing.  Four warps for 128 tokens took 574 us, eight 550, sixteen 506 (then the
// tiles' copies); a third accumulator 514; sums by the MMAs' own fragments (half as many reads of scales) 508.
// ---------------------------------------------------------------------------
constexpr int EPI_WARP0 = 8, COLS = 32, A_COLS = 32;      // the first warp for the sums, the tokens of such a warp; columns of a group's weights
constexpr int W_STAGES = 6, STAGES = 6;               // packed weights; both operands of the MMAs
constexpr int BATCH = 4, S_STAGES = 2;                // groups whose scales come at a time

__device__ __forceinline__ bool elect_one() {
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one != 0;
}
// D (tensor memory, 32-bit integers) += A (tensor memory, signed bytes) * B (shared memory, signed bytes)
__device__ __forceinline__ void umma_i8(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::i8 [%0], [%1], %2, %3, p;\n\t}"
                 ::"r"(tmem_d), "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, int* r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]) : "r"(taddr));
}
// The loads before have arrived.  It takes their registers, so that nothing is done with them ahead of it (and what is not from tensor memory may be).
__device__ __forceinline__ void tmem_wait16(int* r) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]));
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};"
                 ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
                   "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr) : "memory");
}
__device__ __forceinline__ uint64_t pack2(float a, float b) {
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
    return v;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t v;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
    return v;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t v;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
    return v;
}

// A warp's part of a tile (32 features from f on, COLS tokens from t0 on) leaves from shared memory (`stage`, [token][feature]) by a copy of its own, so that
// the warp goes on with its next tile.  (By pieces of 16 bytes, stored by the warp itself, a tile took 3,100 cycles in which no sums were taken: 2,048 x
// 3,584 x 37,888 506 us.)  Rows off 16-byte boundaries leave by elements.
template <typename T>
__device__ __forceinline__ void leave(const W4Params& p, const CUtensorMap* map, T* stage, const uint64_t (&sum)[COLS / 2], int f, int t0, int vec) {
    const int lane = threadIdx.x & 31;
    if (vec) {
        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");      // the tile before has left
        __syncwarp();
#pragma unroll
        for (int q = 0; q < COLS; ++q) stage[q * 32 + lane] = from_f32<T>(__uint_as_float((uint32_t)(sum[q / 2] >> (q & 1 ? 32 : 0))));
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0 && f < p.N && t0 < p.M) {      // (what lies beyond the matrix is left out by the copy)
            asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];"
                         ::"l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(stage)), "r"(f), "r"(t0) : "memory");
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        }
    } else {
        T* const out = (T*)p.out + (size_t)t0 * p.N + f + lane;
#pragma unroll
        for (int q = 0; q < COLS; ++q)
            if (q < p.M - t0 && f + lane < p.N) ElemOps<T>::store(out + (size_t)q * p.N, __uint_as_float((uint32_t)(sum[q / 2] >> (q & 1 ? 32 : 0))));
    }
}

template <int TN, typename T> struct Many {
    static constexpr int EPI_WARPS = 4 * TN / COLS, THREADS = (EPI_WARP0 + EPI_WARPS) * 32;
    static constexpr int X_BYTES = TN * GROUP;
    static constexpr int W_OFF = 0, X_OFF = W_STAGES * W_BYTES;
    static constexpr int SX_OFF = X_OFF + STAGES * X_BYTES, SW_OFF = SX_OFF + S_STAGES * BATCH * TN * 4;      // [stage][group][token], [..][feature]
    static constexpr int OUT_OFF = SW_OFF + S_STAGES * BATCH * FEATURES * 4;      // [warp][token][32 features]
    static constexpr int BARS = OUT_OFF + EPI_WARPS * COLS * 32 * (int)sizeof(T);
    static constexpr int N_BARS = 2 * (W_STAGES + STAGES + S_STAGES + 2) + 1;
    static constexpr int TOTAL = BARS + N_BARS * 8 + 24 + 1024;
    static constexpr int A_COL0 = 2 * TN;
    static_assert(A_COL0 + STAGES * A_COLS <= 512 && TOTAL <= 232448 && TN % 64 == 0 && TN * (FEATURES + 4) * 4 <= SX_OFF && OUT_OFF % 128 == 0, "fits");
};

// SHARED: the CTAs of a cluster share a tile's K (`share` groups each), a tile each; else a CTA takes tile after tile.  vec: whole pieces of 16 bytes leave.
template <int TN, bool SHARED, typename T>
__global__ void __launch_bounds__(Many<TN, T>::THREADS, 1)
w4_many_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_out, const __grid_constant__ W4Params p, int tiles_m, int tiles, int share, int vec) {
    using L = Many<TN, T>;
    constexpr int EPI_WARPS = L::EPI_WARPS;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* gen = smem_raw + (base - smem_u32(smem_raw));
    const uint32_t w_full = base + L::BARS, w_empty = w_full + 8 * W_STAGES;
    const uint32_t ab_full = w_empty + 8 * W_STAGES, ab_empty = ab_full + 8 * STAGES;      // both operands: converted weights and the tokens' bytes
    const uint32_t s_full = ab_empty + 8 * STAGES, s_empty = s_full + 8 * S_STAGES;
    const uint32_t acc_full = s_empty + 8 * S_STAGES, acc_empty = acc_full + 16, drained = acc_empty + 16;
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(gen + L::BARS + L::N_BARS * 8);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(gen + L::BARS + L::N_BARS * 8 + 8);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int C = SHARED ? (int)cg::this_cluster().num_blocks() : 1, rank = SHARED ? (int)cg::this_cluster().block_rank() : 0;

    if (threadIdx.x == 0) {
        *abort_flag = 0;
        for (int s = 0; s < W_STAGES; ++s) { mbar_init(w_full + 8 * s, 1); mbar_init(w_empty + 8 * s, 4); }
        for (int s = 0; s < STAGES; ++s) { mbar_init(ab_full + 8 * s, 5); mbar_init(ab_empty + 8 * s, 1); }
        for (int s = 0; s < S_STAGES; ++s) { mbar_init(s_full + 8 * s, 1); mbar_init(s_empty + 8 * s, EPI_WARPS); }
        for (int s = 0; s < 2; ++s) { mbar_init(acc_full + 8 * s, 1); mbar_init(acc_empty + 8 * s, EPI_WARPS); }
        mbar_init(drained, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        __syncwarp();
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32((const void*)tmem_slot)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = *tmem_slot;
    pdl_trigger();

    int f0, t0, first, n;
    auto place = [&](int tile) {
        f0 = tile / tiles_m * FEATURES;
        t0 = tile % tiles_m * TN;
        first = rank * share;      // (the last of many CTAs may have none left)
        n = min(share, p.G - first);
    };
    if (warp == 0 || warp == 3) {
        if (lane == 0) {
            // the weights have a thread of their own: they are converted, so they are wanted well before the rows are
            const bool rows = warp == 0;
            const CUtensorMap* const map = rows ? &map_x : &map_w;
            const uint32_t full = rows ? ab_full : w_full, empty = rows ? ab_empty : w_empty, stages = rows ? STAGES : W_STAGES;
            asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
            bool waited = false, ok = true;
            uint32_t it = 0;
            for (int tile = blockIdx.x / C; tile < tiles && ok; tile += gridDim.x / C) {
                place(tile);
                for (int i = 0; i < n; ++i) {
                    if (!waited && (rows || !p.ahead || it == W_STAGES)) { pdl_wait(); waited = true; }
                    const uint32_t s = it % stages;
                    if (!(ok = mbar_wait(empty + 8 * s, ((it / stages) & 1) ^ 1, abort_flag, p.err_flag))) break;
                    mbar_expect_tx(full + 8 * s, rows ? L::X_BYTES : W_BYTES);
                    if (rows) tma_load_2d(base + L::X_OFF + s * L::X_BYTES, map, full + 8 * s, (first + i) * GROUP, t0);
                    else tma_load_2d(base + L::W_OFF + s * W_BYTES, map, full + 8 * s, (first + i) * (GROUP / 2), f0);
                    ++it;
                }
            }
            if (!waited) pdl_wait();
            // the copies end before the CTA does, also where a reader's wait ran out after this thread had asked for the last of them
            for (uint32_t at = it > stages ? it - stages : 0; at < it; ++at) mbar_drain(full + 8 * (at % stages), (at / stages) & 1);
        }
    } else if (warp == 1) {
        // D 32-bit integers (2 at bit 4), A and B signed bytes (1 at bits 7 and 10), N >> 3 at bit 17, M >> 4 at bit 24
        constexpr uint32_t idesc = (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(TN >> 3) << 17) | ((uint32_t)(FEATURES >> 4) << 24);
        const uint64_t db0 = umma_desc(base + L::X_OFF);
        const bool elected = elect_one();      // the whole warp goes through the loop, so that the operands stay in uniform registers
        int it = 0, s = 0;
        bool ok = true;
        pdl_wait();      // no bounded wait should have to last as long as the kernels before
        for (int tile = blockIdx.x / C; tile < tiles && ok; tile += gridDim.x / C) {
            place(tile);
            for (int i = 0; i < n; ++i, ++it) {
                const int d = it & 1;
                ok = mbar_wait(acc_empty + 8 * d, ((it >> 1) & 1) ^ 1, abort_flag, p.err_flag) &&
                     mbar_wait(ab_full + 8 * s, (it / STAGES) & 1, abort_flag, p.err_flag);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint64_t db = db0 + s * (L::X_BYTES >> 4);
                const uint32_t a = tmem + L::A_COL0 + s * A_COLS;
                if (elected) {
#pragma unroll
                    for (int q = 0; q < 4; ++q) umma_i8(tmem + d * TN, a + 8 * q, db + 2 * q, idesc, q > 0);      // 32 bytes of k further
                    umma_commit(acc_full + 8 * d);
                    umma_commit(ab_empty + 8 * s);
                }
                __syncwarp();
                s = s + 1 == STAGES ? 0 : s + 1;
            }
        }
        if (elected) {
            umma_commit(drained);      // the MMAs end before tensor memory is given back, also where a wait ran out
            mbar_drain(drained, 0);
        }
        __syncwarp();
    } else if (warp == 2) {
        // the scales of the tokens, and of the features (a sixteenth of them: the integers are sixteen times as large)
        bool ok = true;
        int bt = 0;
        pdl_wait();
        for (int tile = blockIdx.x / C; tile < tiles && ok; tile += gridDim.x / C) {
            place(tile);
            for (int i0 = 0; i0 < n && ok; i0 += BATCH, ++bt) {
                const int s = bt % S_STAGES;
                constexpr int F = FEATURES / 32, X = TN / 32;
                float x[BATCH][X], w[BATCH][F];
#pragma unroll
                for (int j = 0; j < BATCH; ++j) {
                    const size_t g = first + min(i0 + j, n - 1);
#pragma unroll
                    for (int q = 0; q < X; ++q) x[j][q] = p.row_scales[g * p.ld_scales + min(t0 + q * 32 + lane, p.M - 1)];
#pragma unroll
                    for (int q = 0; q < F; ++q) w[j][q] = __bfloat162float(p.scales[g * p.N + min(f0 + q * 32 + lane, p.N - 1)]) * 0.0625f;
                }
                ok = mbar_wait(s_empty + 8 * s, ((bt / S_STAGES) & 1) ^ 1, abort_flag, p.err_flag);
                ok = __all_sync(0xffffffffu, ok);
                float* const sx = reinterpret_cast<float*>(gen + L::SX_OFF) + s * BATCH * TN + lane;
                float* const sw = reinterpret_cast<float*>(gen + L::SW_OFF) + s * BATCH * FEATURES + lane;
#pragma unroll
                for (int j = 0; j < BATCH; ++j) {
#pragma unroll
                    for (int q = 0; q < X; ++q) sx[j * TN + q * 32] = x[j][q];
#pragma unroll
                    for (int q = 0; q < F; ++q) sw[j * FEATURES + q * 32] = w[j][q];
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(s_full + 8 * s);
            }
        }
    } else if (warp < EPI_WARP0) {
        const int quarter = warp & 3, row = quarter * 32 + lane;
        const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
        bool waited = false, ok = true;
        int it = 0;
        for (int tile = blockIdx.x / C; tile < tiles && ok; tile += gridDim.x / C) {
            place(tile);
            for (int i = 0; i < n && ok; ++i, ++it) {
                const int s = it % W_STAGES, sa = it % STAGES;
                if (!waited && (!p.ahead || it >= min(W_STAGES, STAGES))) { pdl_wait(); waited = true; }      // from here on the copies and the MMAs have to run
                ok = mbar_wait(w_full + 8 * s, (it / W_STAGES) & 1, abort_flag, p.err_flag);
                const uint32_t src = base + L::W_OFF + s * W_BYTES + row * 64;      // 64-byte swizzle: a chunk of 16 bytes by bits 7 and 8
                uint32_t v[16], a[32];
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v[4 * q]), "=r"(v[4 * q + 1]), "=r"(v[4 * q + 2]), "=r"(v[4 * q + 3])
                                 : "r"(src + ((q ^ ((row >> 1) & 3)) << 4)) : "memory");
#pragma unroll
                for (int q = 0; q < 16; ++q) { a[2 * q] = lower(v[q]); a[2 * q + 1] = upper(v[q]); }
                __syncwarp();
                if (lane == 0) mbar_arrive(w_empty + 8 * s);
                ok = mbar_wait(ab_empty + 8 * sa, ((it / STAGES) & 1) ^ 1, abort_flag, p.err_flag) && ok;
                ok = __all_sync(0xffffffffu, ok);
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                tmem_st16(tmem + lanes + L::A_COL0 + sa * A_COLS, a);
                tmem_st16(tmem + lanes + L::A_COL0 + sa * A_COLS + 16, a + 16);
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(ab_full + 8 * sa);
            }
        }
        if (!waited) pdl_wait();
    } else {
        const int quarter = warp & 3, row = quarter * 32 + lane, col0 = ((warp - EPI_WARP0) >> 2) * COLS;
        const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
        pdl_wait();
        bool ok = true;
        int it = 0, bt = 0;
        for (int tile = blockIdx.x / C; tile < tiles && ok; tile += gridDim.x / C) {
            place(tile);
            uint64_t sum[COLS / 2];
#pragma unroll
            for (int q = 0; q < COLS / 2; ++q) sum[q] = 0;
            for (int i0 = 0; i0 < n && ok; i0 += BATCH, ++bt) {
                const int s = bt % S_STAGES;
                ok = mbar_wait(s_full + 8 * s, (bt / S_STAGES) & 1, abort_flag, p.err_flag);
                const float* sx = reinterpret_cast<const float*>(gen + L::SX_OFF) + s * BATCH * TN + col0;
                const float* sw = reinterpret_cast<const float*>(gen + L::SW_OFF) + s * BATCH * FEATURES + row;
                const int most = min(BATCH, n - i0);
                for (int j = 0; j < most; ++j, ++it, sx += TN, sw += FEATURES) {
                    const int d = it & 1;
                    ok = mbar_wait(acc_full + 8 * d, (it >> 1) & 1, abort_flag, p.err_flag) && ok;
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint32_t from = tmem + lanes + d * TN + col0;
                    int v[2][16];
                    tmem_ld16(from, v[0]);
                    const float ws = *sw;
                    const uint64_t scale = pack2(ws, ws);
#pragma unroll
                    for (int c = 0; c < COLS; c += 16) {
                        int* const now = v[(c / 16) & 1];
                        tmem_wait16(now);
                        if (c + 16 < COLS) tmem_ld16(from + c + 16, v[(c / 16 + 1) & 1]);      // on its way while this one is worked on
                        else {
                            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                            __syncwarp();
                            if (lane == 0) mbar_arrive(acc_empty + 8 * d);
                        }
#pragma unroll
                        for (int q = 0; q < 16; q += 4) {
                            const ulonglong2 x4 = *reinterpret_cast<const ulonglong2*>(sx + c + q);
                            uint64_t &s0 = sum[(c + q) / 2], &s1 = sum[(c + q) / 2 + 1];
                            s0 = fma2(mul2(pack2((float)now[q], (float)now[q + 1]), x4.x), scale, s0);
                            s1 = fma2(mul2(pack2((float)now[q + 2], (float)now[q + 3]), x4.y), scale, s1);
                        }
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(s_empty + 8 * s);
            }
            if (!ok) break;
            if (!SHARED) {
                leave<T>(p, &map_out, reinterpret_cast<T*>(gen + L::OUT_OFF) + (warp - EPI_WARP0) * COLS * 32, sum, f0 + quarter * 32, t0 + col0, vec);
            } else {      // [token][feature], in the rings' place: all that was in them has been used
                float* const sums = reinterpret_cast<float*>(gen) + col0 * (FEATURES + 4) + row;
#pragma unroll
                for (int q = 0; q < COLS; ++q) sums[q * (FEATURES + 4)] = __uint_as_float((uint32_t)(sum[q / 2] >> (q & 1 ? 32 : 0)));
            }
        }
        if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 1) {
        __syncwarp();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
    if (SHARED) {
        place(blockIdx.x / C);
        add_shares<1, FEATURES, T>(p, gen, 0, *abort_flag != 0, f0, t0, min(TN, p.M - t0));
    }
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encode_tiled() {
    static EncodeTiledFn fn = nullptr;
    if (!fn) {
        void* ptr = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeTiledFn>(ptr);
    }
    return fn;
}
// A map of bytes [rows][pitch] in boxes of `high` rows of `wide` bytes.
bool byte_map(CUtensorMap* map, const void* p, int rows, long long pitch, int wide, int high) {
    EncodeTiledFn fn = encode_tiled();
    if (!fn) return false;
    cuuint64_t dims[2] = {(cuuint64_t)pitch, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)pitch};
    cuuint32_t box[2] = {(cuuint32_t)wide, (cuuint32_t)high}, elem[2] = {1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(p), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
              wide == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// A map of results [rows][n] in boxes of `high` rows of 32.
template <typename T>
bool result_map(CUtensorMap* map, void* p, int rows, int n, int high) {
    EncodeTiledFn fn = encode_tiled();
    if (!fn) return false;
    cuuint64_t dims[2] = {(cuuint64_t)n, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)n * sizeof(T)};
    cuuint32_t box[2] = {32, (cuuint32_t)high}, elem[2] = {1, 1};
    return fn(map, sizeof(T) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, p, dims, strides, box, elem,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Clusters of `kernel` that find room at once, by the number of their CTAs (a cluster needs its CTAs on neighbouring SMs; the driver knows how many there
// are room for).  Worked out once per kernel and device.
constexpr int MOST_SHARES = 8;
struct Room {
    int known, clusters[MOST_SHARES + 1];
};
template <typename... Args>
cudaError_t find_room(void (*kernel)(Args...), int threads, int bytes, Room& room) {
    if (room.known) return cudaSuccess;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = bytes;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    for (int c = 2; c <= MOST_SHARES; ++c) {
        attr.val.clusterDim.x = c;
        cfg.gridDim = dim3(c);
        e = cudaOccupancyMaxActiveClusters(&room.clusters[c], kernel, &cfg);
        if (e != cudaSuccess) return e;
    }
    room.known = 1;
    return cudaSuccess;
}
// CTAs that share a tile's K: as many as find room, each with four groups at least.  Two, four or eight where two CTAs are on an SM (16 x 5,120 x 7,168: 4 of
// them 8.9 us, 5 12.2; 8 x 3,584 x 4,608: 4 5.9, 7 6.7), any number where one is (64 x 5,120 x 5,120: 3 11.3, 2 12.5; 128 x 5,120 x 2,560: as many as there is room for 11.6, 4 12.2).
template <bool TWOS>
int shares_of(const Room& room, long long tiles, int G) {
    int c = MOST_SHARES;
    while (c > 1 && (tiles > room.clusters[c] || G < 4 * c)) c = TWOS ? c / 2 : c - 1;
    return c;
}
template <typename... Args>
int launch_clusters(void (*kernel)(Args...), dim3 grid, int cluster, int threads, int bytes, cudaStream_t stream, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = bytes;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = cluster > 1 ? attr : attr + 1;
    cfg.numAttrs = (cluster > 1) + pyre_pdl_enabled();
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
    if (e != cudaSuccess) return (int)e;
    PYRE_LAUNCH_CHECK();
    return 0;
}
template <int TN, typename T>
int launch_many(const W4Params& p, cudaStream_t stream) {
    using L = Many<TN, T>;
    static Room shared_room[PYRE_MAX_DEVICES] = {}, room[PYRE_MAX_DEVICES] = {};
    const int dev = pyre_current_device();
    cudaError_t e = find_room(w4_many_kernel<TN, true, T>, L::THREADS, L::TOTAL, shared_room[dev]);
    if (e == cudaSuccess) e = find_room(w4_many_kernel<TN, false, T>, L::THREADS, L::TOTAL, room[dev]);
    if (e != cudaSuccess) return (int)e;
    CUtensorMap mw, mx;
    if (!byte_map(&mw, p.packed, p.N, 64ll * p.G, 64, FEATURES) || !byte_map(&mx, p.rows, p.M, 128ll * p.G, 128, TN)) return PYRE_ERR_BAD_ARG;
    const int tiles_m = ceil_div(p.M, TN);
    const long long tiles = (long long)tiles_m * ceil_div(p.N, FEATURES);
    if (tiles > 0x7fffffffll) return PYRE_ERR_UNSUPPORTED;
    const int C = shares_of<false>(shared_room[dev], tiles, p.G), share = ceil_div(p.G, C), vec = p.N % (16 / (int)sizeof(T)) == 0 && !((uintptr_t)p.out & 15);
    CUtensorMap mo = {};      // (only the copies of whole tiles use it)
    if (C == 1 && vec && !result_map<T>(&mo, p.out, p.M, p.N, COLS)) return PYRE_ERR_BAD_ARG;
    if (C > 1) return launch_clusters(w4_many_kernel<TN, true, T>, dim3((unsigned)(tiles * C)), C, L::THREADS, L::TOTAL, stream, mw, mx, mo, p, tiles_m, (int)tiles, share, vec);
    return launch_clusters(w4_many_kernel<TN, false, T>, dim3((unsigned)min(tiles, (long long)pyre_sm_count())), 1, L::THREADS, L::TOTAL, stream, mw, mx, mo, p, tiles_m, (int)tiles, share, vec);
}
template <int NT, int F, typename T>
int launch_stream(const W4Params& p, cudaStream_t stream) {
    using L = Stream<NT, F>;
    static Room room[PYRE_MAX_DEVICES] = {};
    const int dev = pyre_current_device(), tiles = ceil_div(p.N, F), rows = ceil_div(p.M, NT * 8);
    const cudaError_t e = find_room(w4_stream_kernel<NT, F, T>, L::THREADS, L::TOTAL, room[dev]);
    if (e != cudaSuccess) return (int)e;
    CUtensorMap mw, mx;
    if (!byte_map(&mw, p.packed, p.N, 64ll * p.G, 128, F) || !byte_map(&mx, p.rows, p.M, 128ll * p.G, 128, NT * 8)) return PYRE_ERR_BAD_ARG;
    const int C = shares_of<true>(room[dev], (long long)tiles * rows, p.G);
    return launch_clusters(w4_stream_kernel<NT, F, T>, dim3((unsigned)(tiles * C), (unsigned)rows), C, L::THREADS, L::TOTAL, stream, mw, mx, p);
}
// Tiles of 96 features where those of 128 would leave an SM more of them: 24 x 5,120 x 27,648 (216 tiles, two on some SMs, or 288) 18.1 us against 22.3.
template <int NT, typename T>
int launch_tiles(const W4Params& p, cudaStream_t stream) {
    const int sms = pyre_sm_count();
    auto features = [&](int F) { return ceil_div(ceil_div(p.N, F), sms) * F; };
    return ceil_div(p.N, FEATURES) > sms && ceil_div(p.N, 96) <= 2 * sms && features(96) < features(FEATURES) ? launch_stream<NT, 96, T>(p, stream)
                                                                                                            : launch_stream<NT, FEATURES, T>(p, stream);
}
template <typename T>
int launch_few(const W4Params& p, cudaStream_t stream) {
    switch (ceil_div(p.M, 8)) {
        case 1: return launch_tiles<1, T>(p, stream);
        case 2: return launch_tiles<2, T>(p, stream);
        case 3: return launch_tiles<3, T>(p, stream);
        default: return launch_tiles<4, T>(p, stream);
    }
}
// Rows up to here take the stream.  5,120 x 27,648, us on it / on the tensor cores: 8 rows 15.8 / 31.7, 24 18.1 / 31.6, 32 23.7 / 31.7;
// 18,944 x 3,584: 16 13.5 / 18.9, 32 19.3 / 19.1; 3,584 x 3,584: 8 5.8 / 7.4.
constexpr int FEW = 32;

// A warp per group of a feature: s = bf16(max |w| / 7), q = rint(w / s) within -8 .. 7.  A group of zeros (or below 2^-100) has s = 0, one with an
// infinity or a NaN s = NaN.
template <typename T>
__global__ void w4_quantize_kernel(const T* w, long long ld, uint8_t* packed, __nv_bfloat16* scales, int N, int K) {
    pdl_trigger();
    pdl_wait();
    const int G = (K + GROUP - 1) / GROUP, lane = threadIdx.x & 31;
    const long long items = (long long)N * G, step = (long long)gridDim.x * (blockDim.x >> 5);
    for (long long item = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); item < items; item += step) {
        const int n = (int)(item / G), g = (int)(item - (long long)n * G), i = g * GROUP + lane * 4;
        float v[4];
        uint32_t most = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            v[k] = i + k < K ? to_f32<T>(w[(size_t)n * ld + i + k]) : 0.f;
            most = max(most, __float_as_uint(v[k]) & 0x7fffffffu);
        }
        most = __reduce_max_sync(0xffffffffu, most);
        const float largest = __uint_as_float(most);
        const bool bad = most >= 0x7f800000u, none = bad || largest < 7.888609052210118e-31f;
        const __nv_bfloat16 s = __float2bfloat16_rn(bad ? __uint_as_float(0x7fffffffu) : none ? 0.f : largest / 7.f);
        const float scale = __bfloat162float(s);
        uint32_t q = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) q |= ((uint32_t)(none ? 0 : max(-8, min(7, __float2int_rn(v[k] / scale)))) & 15u) << (8 * k);
        const uint32_t next = __shfl_down_sync(0xffffffffu, q, 1);      // the next four elements
        if ((lane & 1) == 0) reinterpret_cast<uint32_t*>(packed)[item * (GROUP / 8) + (lane >> 1)] = q | next << 4;
        if (lane == 0) scales[(size_t)g * N + n] = s;
    }
}

template <typename T>
__global__ void w4_values_kernel(const uint8_t* packed, const __nv_bfloat16* scales, T* out, int N, int K) {
    pdl_trigger();
    pdl_wait();
    const int G = (K + GROUP - 1) / GROUP, lane = threadIdx.x & 31;
    const long long items = (long long)N * G, step = (long long)gridDim.x * (blockDim.x >> 5);
    for (long long item = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); item < items; item += step) {
        const int n = (int)(item / G), g = (int)(item - (long long)n * G), i = g * GROUP + lane * 4;
        const uint32_t word = reinterpret_cast<const uint32_t*>(packed)[item * (GROUP / 8) + (lane >> 1)];
        const uint32_t q = lane & 1 ? upper(word) : lower(word);
        const float s = __bfloat162float(scales[(size_t)g * N + n]);
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (i + k < K) out[(size_t)n * K + i + k] = from_f32<T>((float)((int8_t)(q >> (8 * k)) >> 4) * s);
    }
}
int item_blocks(long long items) { return (int)min((long long)pyre_sm_count() * 8, ceil_div_ll(items, 8)); }
}  // namespace

// w [N, K] at a stride of ld elements -> packed [N][64 G], scales [G][N], G = ceil(K / 128)
PYRE_API int pyre_w4_quantize(const void* w, long long ld, void* packed, void* scales, int N, int K, int dtype, cudaStream_t stream) {
    if (N <= 0 || K <= 0) return 0;
    const dim3 blocks(item_blocks((long long)N * ceil_div(K, GROUP)));
    if (dtype == PYRE_F32) pyre_launch(w4_quantize_kernel<float>, blocks, dim3(256), 0, stream, (const float*)w, ld, (uint8_t*)packed, (__nv_bfloat16*)scales, N, K);
    else if (dtype == PYRE_BF16) pyre_launch(w4_quantize_kernel<__nv_bfloat16>, blocks, dim3(256), 0, stream, (const __nv_bfloat16*)w, ld, (uint8_t*)packed, (__nv_bfloat16*)scales, N, K);
    else return PYRE_ERR_BAD_ARG;
    PYRE_LAUNCH_CHECK();
    return 0;
}

PYRE_API int pyre_w4_values(const void* packed, const void* scales, void* out, int N, int K, int dtype, cudaStream_t stream) {
    if (N <= 0 || K <= 0) return 0;
    const dim3 blocks(item_blocks((long long)N * ceil_div(K, GROUP)));
    if (dtype == PYRE_F32) pyre_launch(w4_values_kernel<float>, blocks, dim3(256), 0, stream, (const uint8_t*)packed, (const __nv_bfloat16*)scales, (float*)out, N, K);
    else if (dtype == PYRE_BF16) pyre_launch(w4_values_kernel<__nv_bfloat16>, blocks, dim3(256), 0, stream, (const uint8_t*)packed, (const __nv_bfloat16*)scales, (__nv_bfloat16*)out, N, K);
    else return PYRE_ERR_BAD_ARG;
    PYRE_LAUNCH_CHECK();
    return 0;
}

// rows [M][128 G] and packed [N][64 G] on 16-byte boundaries; out [M, N] of `dtype`.  ahead: whatever wrote packed and scales had ended, waited for by the host, before
// this call; the kernel then asks for them while the kernels in front of it still run.
PYRE_API int pyre_w4_linear(const void* rows, const float* row_scales, long long ld_scales, const void* packed, const void* scales, void* out,
                            int M, int N, int G, int dtype, int ahead, int* err_flag, cudaStream_t stream) {
    if (M <= 0 || N <= 0) return 0;
    if (G <= 0 || ((uintptr_t)rows & 15) || ((uintptr_t)packed & 15)) return PYRE_ERR_BAD_ARG;
    if (dtype != PYRE_F32 && dtype != PYRE_BF16) return PYRE_ERR_BAD_ARG;
    const W4Params p = {(const uint8_t*)rows, row_scales, ld_scales, (const uint8_t*)packed, (const __nv_bfloat16*)scales, out, M, N, G, ahead, err_flag};
    if (M <= FEW) return dtype == PYRE_F32 ? launch_few<float>(p, stream) : launch_few<__nv_bfloat16>(p, stream);
    // tiles of 64 tokens / 128, us: 64 x 3,584 x 37,888 24.8 / 34.3, 64 x 3,584 x 3,584 8.0 / 9.9; 128 x 3,584 x 37,888 44.9 / 34.9, 128 x 18,944 x 3,584 32.2 / 27.4
    if (M <= 64) return dtype == PYRE_F32 ? launch_many<64, float>(p, stream) : launch_many<64, __nv_bfloat16>(p, stream);
    return dtype == PYRE_F32 ? launch_many<128, float>(p, stream) : launch_many<128, __nv_bfloat16>(p, stream);
}
