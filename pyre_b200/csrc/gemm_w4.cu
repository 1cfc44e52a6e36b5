// Products with 4-bit weights:  y[t, n] = sum_g sw[g, n] sx[g, t] sum_{k in group g} qw[n, k] qx[t, k].
//
// Rows qx are 8-bit with a scale per 128 elements (rows8.cu); a weight's elements are -8 .. 7 in 4 bits with a bf16 scale per 128 elements of
// a feature.  A word of four bytes holds eight elements: byte i element i in its lower half and element i + 4 in its upper one, so that
// two masks give two words of four bytes in the order in which the rows lie.  Both are padded with zeros to a multiple of 128 elements.
// The inner sums are exact (32-bit integers: |sum| <= 16 * 8 * 127 * 128 < 2^21, a weight's half byte stays in the upper half of its byte, which
// makes it sixteen times as large and spares the sign's extension), the outer ones in float, by ascending group in each of a CTA's warps,
// then over the warps in order.
#include "common.cuh"

namespace {
constexpr int GROUP = 128;

__device__ __forceinline__ void mma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
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
};

constexpr int WARPS = 8;

// A CTA owns 16 features and NT tiles of 8 tokens; its warps take the groups in turn.  Lane l of a warp holds 32 neighbouring elements (the
// l % 4th quarter of the group) of features l / 4 and l / 4 + 8 and of token l / 4: which k an MMA step sums over is free as long as
// both operands agree.
template <int NT, typename T>
__global__ void __launch_bounds__(WARPS * 32)
w4_few_kernel(const W4Params p) {
    __shared__ float sums[WARPS][NT * 4][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, quad = lane >> 2, c = lane & 3;
    const int f0 = blockIdx.x * 16, t0 = blockIdx.y * NT * 8;
    const int fa = min(f0 + quad, p.N - 1), fb = min(f0 + quad + 8, p.N - 1);
    const size_t pitch = (size_t)p.G * GROUP;
    const uint8_t* wa = p.packed + fa * (pitch / 2) + c * 16;
    const uint8_t* wb = p.packed + fb * (pitch / 2) + c * 16;
    const uint8_t* x[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) x[n] = p.rows + (size_t)min(t0 + n * 8 + quad, p.M - 1) * pitch + c * 32;
    pdl_trigger();
    pdl_wait();
    float total[NT][4] = {};
    for (int g = warp; g < p.G; g += WARPS) {
        const uint4 a4 = *reinterpret_cast<const uint4*>(wa + (size_t)g * (GROUP / 2));
        const uint4 b4 = *reinterpret_cast<const uint4*>(wb + (size_t)g * (GROUP / 2));
        const float sa = __bfloat162float(p.scales[(size_t)g * p.N + fa]) * 0.0625f;
        const float sb = __bfloat162float(p.scales[(size_t)g * p.N + fb]) * 0.0625f;
        const uint32_t a[4] = {a4.x, a4.y, a4.z, a4.w}, b[4] = {b4.x, b4.y, b4.z, b4.w};
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const uint4 x0 = *reinterpret_cast<const uint4*>(x[n] + (size_t)g * GROUP);
            const uint4 x1 = *reinterpret_cast<const uint4*>(x[n] + (size_t)g * GROUP + 16);
            const uint32_t xv[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
            int d[4] = {};
#pragma unroll
            for (int j = 0; j < 4; ++j) mma_s8(d, lower(a[j]), lower(b[j]), upper(a[j]), upper(b[j]), xv[2 * j], xv[2 * j + 1]);
            const float* s = p.row_scales + (size_t)g * p.ld_scales;
            const float s0 = s[min(t0 + n * 8 + 2 * c, p.M - 1)], s1 = s[min(t0 + n * 8 + 2 * c + 1, p.M - 1)];
            total[n][0] = fmaf((float)d[0] * s0, sa, total[n][0]);
            total[n][1] = fmaf((float)d[1] * s1, sa, total[n][1]);
            total[n][2] = fmaf((float)d[2] * s0, sb, total[n][2]);
            total[n][3] = fmaf((float)d[3] * s1, sb, total[n][3]);
        }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) sums[warp][n * 4 + i][lane] = total[n][i];
    __syncthreads();
    for (int e = warp; e < NT * 4; e += WARPS) {
        float v = sums[0][e][lane];
        for (int w = 1; w < WARPS; ++w) v += sums[w][e][lane];
        const int t = t0 + (e >> 2) * 8 + 2 * c + (e & 1), f = f0 + quad + (e & 2) * 4;
        if (t < p.M && f < p.N) ElemOps<T>::store((T*)p.out + (size_t)t * p.N + f, v);
    }
}

template <typename T>
int launch_few(const W4Params& p, cudaStream_t stream) {
    const int tiles = ceil_div(p.M, 8), nt = tiles >= 4 ? 4 : tiles >= 2 ? 2 : 1;
    const dim3 grid(ceil_div(p.N, 16), ceil_div(tiles, nt));
    if (nt == 4) pyre_launch(w4_few_kernel<4, T>, grid, dim3(WARPS * 32), 0, stream, p);
    else if (nt == 2) pyre_launch(w4_few_kernel<2, T>, grid, dim3(WARPS * 32), 0, stream, p);
    else pyre_launch(w4_few_kernel<1, T>, grid, dim3(WARPS * 32), 0, stream, p);
    PYRE_LAUNCH_CHECK();
    return 0;
}

// A warp per group of a feature: s = bf16(max |w| / 7), q = rint(w / s) within -8 .. 7.  A group of zeros (or below 2^-100) has s = 0, one with an
// infinity or a NaN s = NaN.
template <typename T>
__global__ void w4_quantize_kernel(const T* w, long long ld, uint8_t* packed, __nv_bfloat16* scales, int N, int K) {
    pdl_wait();      // no trigger: a product reads the weight ahead of its own wait
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

// rows [M][128 G] and packed [N][64 G] on 16-byte boundaries; out [M, N] of `dtype`
PYRE_API int pyre_w4_linear(const void* rows, const float* row_scales, long long ld_scales, const void* packed, const void* scales, void* out,
                            int M, int N, int G, int dtype, cudaStream_t stream) {
    if (M <= 0 || N <= 0) return 0;
    if (G <= 0 || ((uintptr_t)rows & 15) || ((uintptr_t)packed & 15)) return PYRE_ERR_BAD_ARG;
    const W4Params p = {(const uint8_t*)rows, row_scales, ld_scales, (const uint8_t*)packed, (const __nv_bfloat16*)scales, out, M, N, G};
    if (dtype == PYRE_F32) return launch_few<float>(p, stream);
    if (dtype == PYRE_BF16) return launch_few<__nv_bfloat16>(p, stream);
    return PYRE_ERR_BAD_ARG;
}
