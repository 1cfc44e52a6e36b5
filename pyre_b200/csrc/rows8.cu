// Rows of activations in 8 bits with a scale per 128 neighbouring elements: what a product with a 4-bit weight reads.
//
// A row of H elements y makes G = ceil(H / 128) groups (the last one may be short: its missing elements are zeros).
//   s = max |y| / 127 over the group (float), q = rint(y / s) in [-127, 127], y stands for q s.
// A group whose largest |y| is below 2^-100 counts as zeros (s = 0), one that holds an infinity or a NaN has s = NaN (and so gives NaN
// wherever it is read).  Rows lie at a pitch of 128 G bytes, scales as [G][T]: a product takes a group of all its tokens at once.
//
//   norm   x += delta (written back), y = x / sqrt(mean(x^2) + eps) * w: a block per row, a warp per group; the row stays in registers
//          between the sum of squares and the scaling.
//   rows   y = x as it is (attention's output), a warp per group.
//   gate   y = act(gate) * up, a warp per group.
//   values the numbers that rows stand for, for a consumer that wants plain activations.
#include "common.cuh"

namespace {
constexpr int GROUP = 128;
constexpr float LEAST = 7.888609052210118e-31f;      // 2^-100

// A lane's four elements of a group -> four bytes; the scale comes back in every lane.
__device__ __forceinline__ uint32_t group_bytes(const float (&y)[4], float& scale) {
    uint32_t most = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) most = max(most, __float_as_uint(y[k]) & 0x7fffffffu);
    most = __reduce_max_sync(0xffffffffu, most);      // as bits: NaN above infinity above all numbers
    const float largest = __uint_as_float(most);
    if (most >= 0x7f800000u) {
        scale = __uint_as_float(0x7fffffffu);
        return 0;
    }
    if (largest < LEAST) {
        scale = 0.f;
        return 0;
    }
    scale = largest / 127.f;
    const float inverse = 127.f / largest;
    uint32_t out = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) out |= ((uint32_t)__float2int_rn(y[k] * inverse) & 0xffu) << (8 * k);
    return out;
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

// gate: rows of [gates | ups], 2 K wide (kind 0 silu, 1 relu, 2 clamped, see common.cuh); else rows as they are.  A warp per group.
template <typename T, bool VEC, bool GATE>
__global__ void rows8_kernel(const T* x, long long ld, int8_t* out, float* scales, int n_rows, int K, int kind, float limit) {
    pdl_trigger();
    pdl_wait();
    const int G = (K + GROUP - 1) / GROUP, lane = threadIdx.x & 31;
    const long long items = (long long)n_rows * G, step = (long long)gridDim.x * (blockDim.x >> 5);
    for (long long item = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); item < items; item += step) {
        const int r = (int)(item / G), g = (int)(item - (long long)r * G), i = g * GROUP + lane * 4;
        float y[4], scale;
        load4<T, VEC>(y, x + r * ld, i, K);
        if (GATE) {
            float up[4];
            load4<T, VEC>(up, x + r * ld + K, i, K);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float z = y[k], u = up[k];
                if (kind == 2) {
                    z = fminf(z, limit);
                    u = fminf(fmaxf(u, -limit), limit) + 1.0f;
                }
                const float s = kind == 1 ? fmaxf(z, 0.f) : z / (1.0f + expf(kind == 2 ? -CLAMPED_GLU_SLOPE * z : -z));
                y[k] = i + k < K ? __fmul_rn(s, u) : 0.f;
            }
        }
        const uint32_t q = group_bytes(y, scale);
        reinterpret_cast<uint32_t*>(out)[item * (GROUP / 4) + lane] = q;
        if (lane == 0) scales[(size_t)g * n_rows + r] = scale;
    }
}

template <typename T>
__global__ void rows8_values_kernel(const int8_t* rows, const float* scales, long long ld_scales, T* out, int n_rows, int K) {
    pdl_trigger();
    pdl_wait();
    const int G = (K + GROUP - 1) / GROUP, lane = threadIdx.x & 31;
    const long long items = (long long)n_rows * G, step = (long long)gridDim.x * (blockDim.x >> 5);
    const bool vec = K % 4 == 0;
    for (long long item = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); item < items; item += step) {
        const int r = (int)(item / G), g = (int)(item - (long long)r * G), i = g * GROUP + lane * 4;
        const uint32_t q = reinterpret_cast<const uint32_t*>(rows)[item * (GROUP / 4) + lane];
        const float s = scales[(size_t)g * ld_scales + r];
        Vec<T, 4> v;
#pragma unroll
        for (int k = 0; k < 4; ++k) v.v[k] = from_f32<T>((float)(int8_t)(q >> (8 * k)) * s);
        T* o = out + (size_t)r * K + i;
        if (vec) {
            if (i < K) store_vec<T, 4>(o, v);
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (i + k < K) o[k] = v.v[k];
        }
    }
}

int item_blocks(long long items, int warps) { return (int)min((long long)pyre_sm_count() * (64 / warps), ceil_div_ll(items, warps)); }
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
    const int size = dtype == PYRE_F32 ? 4 : 2;
    const bool vec = K % 4 == 0 && ld % 4 == 0 && aligned(x, 4 * size);
    const int blocks = item_blocks((long long)n_rows * ceil_div(K, GROUP), 8);
#define LAUNCH_G(TT, V, GT) pyre_launch(rows8_kernel<TT, V, GT>, dim3(blocks), dim3(256), 0, stream, (const TT*)x, ld, (int8_t*)out, scales, n_rows, K, kind, limit)
#define LAUNCH(TT) do { if (gate) { if (vec) LAUNCH_G(TT, true, true); else LAUNCH_G(TT, false, true); } else { if (vec) LAUNCH_G(TT, true, false); else LAUNCH_G(TT, false, false); } } while (0)
    if (dtype == PYRE_F32) LAUNCH(float);
    else if (dtype == PYRE_BF16) LAUNCH(__nv_bfloat16);
    else return PYRE_ERR_BAD_ARG;
#undef LAUNCH
#undef LAUNCH_G
    PYRE_LAUNCH_CHECK();
    return 0;
}

PYRE_API int pyre_rows8_values(const void* rows, const float* scales, long long ld_scales, void* out, int n_rows, int K, int dtype, cudaStream_t stream) {
    if (n_rows <= 0 || K <= 0) return 0;
    const int blocks = item_blocks((long long)n_rows * ceil_div(K, GROUP), 8);
    if (dtype == PYRE_F32) pyre_launch(rows8_values_kernel<float>, dim3(blocks), dim3(256), 0, stream, (const int8_t*)rows, scales, ld_scales, (float*)out, n_rows, K);
    else if (dtype == PYRE_BF16) pyre_launch(rows8_values_kernel<__nv_bfloat16>, dim3(blocks), dim3(256), 0, stream, (const int8_t*)rows, scales, ld_scales, (__nv_bfloat16*)out, n_rows, K);
    else return PYRE_ERR_BAD_ARG;
    PYRE_LAUNCH_CHECK();
    return 0;
}
