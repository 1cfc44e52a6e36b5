// Rows of activations in 8 bits with a scale per 128 neighbouring elements: what a product with a 4-bit weight reads.
//
// A row of H elements y makes G = ceil(H / 128) groups (the last one may be short: its missing elements are zeros).
//   s = max |y| / 127 over the group (float), q = rint(y / s) in [-127, 127], y stands for q s.
// A group whose largest |y| is below 2^-100 counts as zeros (s = 0), one that holds an infinity or a NaN has s = NaN (and so gives NaN
// wherever it is read).  Rows lie at a pitch of 128 G bytes, scales as [G][T]: a product takes a group of all its tokens at once.
//
//   norm   x += delta (written back), y = x / sqrt(mean(x^2) + eps) * w: a block per row, a warp per group; the row stays in registers
//          between the sum of squares and the scaling (up to 8,192 elements; above, it is read again, out of L2).
//   rows   y = x as it is (attention's output), a warp per group, or four groups.
//   gate   y = act(gate) * up, likewise.
//   values the numbers that rows stand for, for a consumer that wants plain activations.
//
// Bound: memory, for many rows.  bf16, us (read and written, TB/s): norm 2,048 x 3,584 15.7 (5.2), 8,192 x 3,584 55 (5.9); rows 8,192 x 3,584 16.1 (5.5);
// gate 2,048 x 18,944 41.5 (4.7); values 8,192 x 3,584 19.7 (4.5).  With a warp per group, whose lanes have four elements each, rows took 45.6 and gate
// 98: a group's two divisions and its maximum cost more than its elements.  Few rows take what a launch and a round trip to memory take, in a captured step:
// norm 1 x 3,584 2.4 (its two reductions of a row are one round trip and a meeting of the block), rows 1.1, gate 1 x 18,944 1.4.
#include "common.cuh"

namespace {
constexpr int GROUP = 128;
constexpr float LEAST = 7.888609052210118e-31f;      // 2^-100

// The larger magnitude, NaN where one is.
__device__ __forceinline__ float larger(float most, float y) {
    float m;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(most), "f"(fabsf(y)));
    return m;
}
// The scale of a group and what its elements are multiplied by, from its largest magnitude.
__device__ __forceinline__ float group_scale(float largest, float& inverse) {
    const bool bad = __float_as_uint(largest) >= 0x7f800000u, none = bad || largest < LEAST;
    inverse = none ? 0.f : 127.f / largest;
    return bad ? __uint_as_float(0x7fffffffu) : none ? 0.f : largest / 127.f;
}
// Four elements in 8 bits: beside 1.5 2^23 the sum's last byte is the product to the nearest whole number (one fused operation in a conversion's
// place).  A group without a scale has an inverse of 0; in one that holds an infinity or a NaN the bytes do not matter, but are zeros.
__device__ __forceinline__ uint32_t four_bytes(const float* y, float inverse) {
    uint32_t b[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) b[k] = __float_as_uint(fmaf(y[k], inverse, 12582912.f));
    const uint32_t q = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
    return inverse > 0.f ? q : 0;
}

// A lane's four elements of a warp's group -> four bytes; the scale comes back in every lane.
__device__ __forceinline__ uint32_t group_bytes(const float (&y)[4], float& scale) {
    const float most = larger(larger(larger(fabsf(y[0]), y[1]), y[2]), y[3]);
    float inverse;      // (as bits: NaN above infinity above all numbers)
    scale = group_scale(__uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(most))), inverse);
    return four_bytes(y, inverse);
}

// Four neighbouring elements from i on of a row of n, zeros beyond it.  VEC: i and n are multiples of four and the row is aligned.
template <typename T, bool VEC>
__device__ __forceinline__ void load4(float (&v)[4], const T* row, int i, int n) {
    if (VEC) {
        if (i < n) {
            const Vec<T, 4> a = load_vec<T, 4>(row + i);
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = to_f32<T>(a.v[k]);
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = 0.f;
        }
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = i + k < n ? to_f32<T>(row[i + k]) : 0.f;
    }
}
template <bool VEC>
__device__ __forceinline__ void store4(float* row, int i, int n, const float (&v)[4]) {
    if (VEC) {
        if (i < n) *reinterpret_cast<float4*>(row + i) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (i + k < n) row[i + k] = v[k];
    }
}

struct Norm8Params {
    float* x;
    const void* delta;
    const float* partials;
    long long partial_stride;
    const float* w;
    int8_t* out;
    float* scales;
    const int* rows;
    int n_partials, n_rows, H, update_x;
    float eps;
};

// KEEP: groups of the row that a warp keeps in registers; 0: the row is read again for the scaling (any width).
template <typename T, bool VEC, int KEEP>
__global__ void norm8_kernel(const Norm8Params p) {
    pdl_trigger();
    pdl_wait();
    __shared__ float scratch[33];
    const int r = blockIdx.x, src = p.rows ? p.rows[r] : r;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const int H = p.H, G = (H + GROUP - 1) / GROUP;
    float* xr = p.x + (size_t)src * H;
    const T* dr = p.delta ? (const T*)p.delta + (size_t)src * H : nullptr;
    const float* pr = p.partials ? p.partials + (size_t)src * H : nullptr;
    auto stream = [&](int i, float (&v)[4]) {
        load4<float, VEC>(v, xr, i, H);
        if (pr) {
            float sum[4], more[4];
            load4<float, VEC>(sum, pr, i, H);
            for (int s = 1; s < p.n_partials; ++s) {
                load4<float, VEC>(more, pr + (size_t)s * p.partial_stride, i, H);
#pragma unroll
                for (int k = 0; k < 4; ++k) sum[k] += more[k];
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] += sum[k];
        } else if (dr) {
            float d[4];
            load4<T, VEC>(d, dr, i, H);
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] += d[k];
        }
    };
    float kept[KEEP > 0 ? KEEP : 1][4];
    float ss = 0.f;
    auto square = [&](const float (&v)[4]) {
#pragma unroll
        for (int k = 0; k < 4; ++k) ss = fmaf(v[k], v[k], ss);
    };
    if constexpr (KEEP > 0) {
#pragma unroll
        for (int j = 0; j < KEEP; ++j) stream((warp + j * warps) * GROUP + lane * 4, kept[j]);
#pragma unroll
        for (int j = 0; j < KEEP; ++j) {
            if (p.update_x) store4<VEC>(xr, (warp + j * warps) * GROUP + lane * 4, H, kept[j]);
            square(kept[j]);
        }
    } else {
        for (int g = warp; g < G; g += warps) {
            float v[4];
            stream(g * GROUP + lane * 4, v);
            if (p.update_x) store4<VEC>(xr, g * GROUP + lane * 4, H, v);
            square(v);
        }
    }
    const float rstd = 1.0f / sqrtf(block_sum(ss, scratch) / (float)H + p.eps);
    uint32_t* out = reinterpret_cast<uint32_t*>(p.out + (size_t)r * G * GROUP);
    auto finish = [&](int g, const float (&v)[4]) {
        float w[4], y[4], scale;
        load4<float, VEC>(w, p.w, g * GROUP + lane * 4, H);
#pragma unroll
        for (int k = 0; k < 4; ++k) y[k] = __fmul_rn(__fmul_rn(v[k], rstd), w[k]);
        out[g * (GROUP / 4) + lane] = group_bytes(y, scale);
        if (lane == 0) p.scales[(size_t)g * p.n_rows + r] = scale;
    };
    if constexpr (KEEP > 0) {
#pragma unroll
        for (int j = 0; j < KEEP; ++j)
            if (warp + j * warps < G) finish(warp + j * warps, kept[j]);
    } else {
        for (int g = warp; g < G; g += warps) {
            float v[4];
            const int i = g * GROUP + lane * 4;
            if (p.update_x) load4<float, VEC>(v, xr, i, H);      // the lane's own store
            else stream(i, v);
            finish(g, v);
        }
    }
}

// A warp's next U neighbouring groups of the rows: f(which of them, row, group in it).
template <int U, typename F> __device__ __forceinline__ void each_group(long long item, long long items, int G, F f) {
    int r = (int)(item / G), g = (int)(item - (long long)r * G);
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (item + u < items) f(u, r, g);
        if (++g == G) {
            g = 0;
            ++r;
        }
    }
}

// GATE: rows of [gates | ups], 2 K wide, by kind (0 silu, 1 relu, 2 clamped, see common.cuh); -1: rows as they are.  LANES lanes take a group, by pieces of
// up to 16 bytes, neighbouring lanes neighbouring pieces.
template <typename T, bool VEC, int GATE, int LANES>
__global__ void rows8_kernel(const T* x, long long ld, int8_t* out, float* scales, int n_rows, int K, float limit) {
    pdl_trigger();
    pdl_wait();
    constexpr int E = GROUP / LANES, PIECE = E * (int)sizeof(T) < 16 ? E : 16 / (int)sizeof(T), PIECES = E / PIECE;      // elements of a lane, of a piece
    const int G = (K + GROUP - 1) / GROUP, l = threadIdx.x % LANES * PIECE;
    const long long items = (long long)n_rows * G;
    const int own = threadIdx.x / LANES, first = blockIdx.x * (blockDim.x / LANES), step = gridDim.x * (blockDim.x / LANES);
    const int rows_on = step / G, groups_on = step - rows_on * G;
    int r = (first + own) / G, g = (first + own) - r * G;
    for (long long at = first; at < items; at += step) {      // (the whole block goes round as often)
        const bool live = at + own < items;
        const T* const row = x + (live ? r : 0) * ld;
        float y[E];
        auto load = [&](float* v, const T* from) {
#pragma unroll
            for (int q = 0; q < PIECES; ++q) {
                const int i = g * GROUP + q * LANES * PIECE + l;
                if (VEC) {
                    if (live && i < K) {
                        const Vec<T, PIECE> a = load_vec<T, PIECE>(from + i);
#pragma unroll
                        for (int k = 0; k < PIECE; ++k) v[q * PIECE + k] = to_f32<T>(a.v[k]);
                    } else {
#pragma unroll
                        for (int k = 0; k < PIECE; ++k) v[q * PIECE + k] = 0.f;
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < PIECE; ++k) v[q * PIECE + k] = live && i + k < K ? to_f32<T>(from[i + k]) : 0.f;
                }
            }
        };
        load(y, row);
        if (GATE >= 0) {
            float up[E];
            load(up, row + K);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                float z = y[e], u = up[e];
                if (GATE == 2) {
                    z = fminf(z, limit);
                    u = fminf(fmaxf(u, -limit), limit) + 1.0f;
                }
                const float s = GATE == 1 ? fmaxf(z, 0.f) : __fdividef(z, 1.0f + expf(GATE == 2 ? -CLAMPED_GLU_SLOPE * z : -z));      // (off by 2^-22)
                y[e] = g * GROUP + e / PIECE * LANES * PIECE + l + e % PIECE < K ? __fmul_rn(s, u) : 0.f;
            }
        }
        float most = fabsf(y[0]), inverse;
#pragma unroll
        for (int e = 1; e < E; ++e) most = larger(most, y[e]);
        if constexpr (LANES == 32)
            most = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(most)));
        else
#pragma unroll
            for (int o = LANES / 2; o > 0; o >>= 1) most = larger(most, __shfl_xor_sync(0xffffffffu, most, o));
        const float scale = group_scale(most, inverse);
        if (live) {
            uint32_t* const to = reinterpret_cast<uint32_t*>(out) + (at + own) * (GROUP / 4) + l / 4;
#pragma unroll
            for (int q = 0; q < PIECES; ++q) {
                if constexpr (PIECE == 8)
                    *reinterpret_cast<uint2*>(to + q * LANES * 2) = make_uint2(four_bytes(y + q * 8, inverse), four_bytes(y + q * 8 + 4, inverse));
                else
                    to[q * LANES] = four_bytes(y + q * 4, inverse);
            }
            if (l == 0) scales[(size_t)g * n_rows + r] = scale;
        }
        r += rows_on;
        g += groups_on;
        if (g >= G) {
            g -= G;
            ++r;
        }
    }
}

template <typename T, int U>
__global__ void rows8_values_kernel(const int8_t* rows, const float* scales, long long ld_scales, T* out, int n_rows, int K) {
    pdl_trigger();
    pdl_wait();
    const int G = (K + GROUP - 1) / GROUP, lane = threadIdx.x & 31;
    const long long items = (long long)n_rows * G, step = (long long)gridDim.x * (blockDim.x >> 5) * U;
    const bool vec = K % 4 == 0;
    for (long long item = ((long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5)) * U; item < items; item += step) {
        uint32_t q[U];
        float s[U];
        each_group<U>(item, items, G, [&](int u, int r, int g) {
            q[u] = reinterpret_cast<const uint32_t*>(rows)[(item + u) * (GROUP / 4) + lane];
            s[u] = scales[(size_t)g * ld_scales + r];
        });
        each_group<U>(item, items, G, [&](int u, int r, int g) {
            const int i = g * GROUP + lane * 4;
            Vec<T, 4> v;
#pragma unroll
            for (int k = 0; k < 4; ++k) v.v[k] = from_f32<T>((float)(int8_t)(q[u] >> (8 * k)) * s[u]);
            T* o = out + (size_t)r * K + i;
            if (vec) {
                if (i < K) store_vec<T, 4>(o, v);
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (i + k < K) o[k] = v.v[k];
            }
        });
    }
}

// Many groups: a warp takes four at a time, so that all SMs' loads fill the way to memory and four groups' scales are worked out at once (rows
// 2,048 x 3,584: 4.7 us against 11.9); where there are few it takes one, whose lanes have less to do one after the other (gate 1 x 18,944: 1.4
// against 1.9, 48 x 13,824 3.3 against 3.8).
bool many_groups(long long items) { return items >= (long long)pyre_sm_count() * 64; }
int item_blocks(long long items) { return (int)min((long long)pyre_sm_count() * 8, ceil_div_ll(items, many_groups(items) ? 32 : 8)); }
bool aligned(const void* p, int bytes) { return ((uintptr_t)p & (bytes - 1)) == 0; }
}  // namespace

// x fp32 [., H]; delta [., H] in `dtype` or fp32 partial sums [n_partials] (stride between them in elements), or neither; out [n_rows][128 G];
// scales [G][n_rows].
PYRE_API int pyre_norm_rows8(float* x, const void* delta, const float* partials, int n_partials, long long partial_stride,
                             const float* weight, void* out, float* scales, const int* rows, int n_rows, int H, float eps, int update_x,
                             int dtype, cudaStream_t stream) {
    if (n_rows <= 0) return 0;
    if (H <= 0 || (rows && update_x) || (delta && partials) || (partials && n_partials < 1)) return PYRE_ERR_BAD_ARG;
    if (dtype != PYRE_F32 && dtype != PYRE_BF16) return PYRE_ERR_BAD_ARG;
    const int G = ceil_div(H, GROUP);
    const bool vec = H % 4 == 0 && partial_stride % 4 == 0 && aligned(x, 16) && aligned(delta, dtype == PYRE_F32 ? 16 : 8) && aligned(partials, 16) && aligned(weight, 16);
    const Norm8Params p = {x, delta, partials, partial_stride, weight, (int8_t*)out, scales, rows, n_partials, n_rows, H, update_x, eps};
    const int warps = min(16, G), keep = ceil_div(G, warps);
#define LAUNCH_K(TT, V, KP) pyre_launch(norm8_kernel<TT, V, KP>, dim3(n_rows), dim3(warps * 32), 0, stream, p)
#define LAUNCH(TT, V) do { if (keep <= 2) LAUNCH_K(TT, V, 2); else if (keep <= 4) LAUNCH_K(TT, V, 4); else LAUNCH_K(TT, V, 0); } while (0)
    if (dtype == PYRE_F32) { if (vec) LAUNCH(float, true); else LAUNCH(float, false); }
    else { if (vec) LAUNCH(__nv_bfloat16, true); else LAUNCH(__nv_bfloat16, false); }
#undef LAUNCH
#undef LAUNCH_K
    PYRE_LAUNCH_CHECK();
    return 0;
}

// x [n_rows] rows of K elements (gate: of K gates and K ups) at a stride of ld elements.
PYRE_API int pyre_rows8(const void* x, long long ld, void* out, float* scales, int n_rows, int K, int gate, int kind, float limit, int dtype,
                        cudaStream_t stream) {
    if (n_rows <= 0 || K <= 0) return 0;
    if (kind < 0 || kind > 2 || (kind == 2 && !(limit > 0.f))) return PYRE_ERR_BAD_ARG;
    const long long items = (long long)n_rows * ceil_div(K, GROUP);
    const bool many = many_groups(items);
    const int size = dtype == PYRE_F32 ? 4 : 2, piece = many ? 16 / size : 4;
    const bool vec = K % piece == 0 && ld % piece == 0 && aligned(x, piece * size);
    const dim3 blocks(item_blocks(items));
#define LAUNCH_L(TT, V, GT, L) pyre_launch(rows8_kernel<TT, V, GT, L>, blocks, dim3(256), 0, stream, (const TT*)x, ld, (int8_t*)out, scales, n_rows, K, limit)
#define LAUNCH_G(TT, V, GT) do { if (many) LAUNCH_L(TT, V, GT, 8); else LAUNCH_L(TT, V, GT, 32); } while (0)
#define LAUNCH_V(TT, GT) do { if (vec) LAUNCH_G(TT, true, GT); else LAUNCH_G(TT, false, GT); } while (0)
#define LAUNCH(TT) do { if (!gate) LAUNCH_V(TT, -1); else if (kind == 0) LAUNCH_V(TT, 0); else if (kind == 1) LAUNCH_V(TT, 1); else LAUNCH_V(TT, 2); } while (0)
    if (dtype == PYRE_F32) LAUNCH(float);
    else if (dtype == PYRE_BF16) LAUNCH(__nv_bfloat16);
    else return PYRE_ERR_BAD_ARG;
#undef LAUNCH
#undef LAUNCH_G
#undef LAUNCH_V
#undef LAUNCH_L
    PYRE_LAUNCH_CHECK();
    return 0;
}

PYRE_API int pyre_rows8_values(const void* rows, const float* scales, long long ld_scales, void* out, int n_rows, int K, int dtype, cudaStream_t stream) {
    if (n_rows <= 0 || K <= 0) return 0;
    if (dtype != PYRE_F32 && dtype != PYRE_BF16) return PYRE_ERR_BAD_ARG;
    const long long items = (long long)n_rows * ceil_div(K, GROUP);
    const dim3 blocks(item_blocks(items));
#define LAUNCH(TT, U) pyre_launch(rows8_values_kernel<TT, U>, blocks, dim3(256), 0, stream, (const int8_t*)rows, scales, ld_scales, (TT*)out, n_rows, K)
    if (dtype == PYRE_F32) { if (many_groups(items)) LAUNCH(float, 4); else LAUNCH(float, 1); }
    else { if (many_groups(items)) LAUNCH(__nv_bfloat16, 4); else LAUNCH(__nv_bfloat16, 1); }
#undef LAUNCH
    PYRE_LAUNCH_CHECK();
    return 0;
}
