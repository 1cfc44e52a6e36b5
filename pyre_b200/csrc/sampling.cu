// Sampling over fp32 logits, one block per row.
//
// The reference samples greedily only: `int(logits[i, -1].argmax())` on the host
// after a device-to-host copy per request (pyre/scheduler.py:80,94).  Here both
// rules run on the device and one int per row comes back:
//   temperature == 0 : argmax, the lowest index winning a tie
//   temperature  > 0 : Gumbel-max, argmax_v(logit[v] / temperature + g(seed, index, v))
// The noise g depends only on the request's seed, the index of the token being
// generated and the vocabulary entry, never on the batch: a request draws the same
// tokens alone or beside others.  u = (23 random bits + 0.5) / 2^23 is exact in fp32
// and lies strictly inside (0, 1), so g = -log(-log(u)) is finite.
#include <cooperative_groups.h>

#include "common.cuh"

__device__ __forceinline__ unsigned long long mix64(unsigned long long z) {
    z += 0x9E3779B97F4A7C15ull;
    z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
    z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
    return z ^ (z >> 31);
}

__device__ __forceinline__ float gumbel(unsigned long long seed, unsigned int token_index, unsigned int v) {
    const unsigned long long h = mix64(seed ^ mix64(((unsigned long long)token_index << 32) | v));
    const float u = ((float)(h >> 41) + 0.5f) * (1.0f / 8388608.0f);
    return -logf(-logf(u));
}

struct Best {
    float score;
    int index;
};

__device__ __forceinline__ Best better(Best a, Best b) {
    // larger score wins; equal scores: lower index; an empty slot has index INT_MAX
    if (b.score > a.score || (b.score == a.score && b.index < a.index)) return b;
    return a;
}

__global__ void sample_kernel(const float* logits, long long ld, const float* temperature,
                              const unsigned long long* seeds, const int* token_index,
                              int* out, int V) {
    __shared__ Best warp_best[32];
    pdl_trigger();
    pdl_wait();
    const int r = blockIdx.x;
    const float* row = logits + (size_t)r * ld;
    const float temp = temperature ? temperature[r] : 0.f;
    const bool greedy = !(temp > 0.f);
    const float inv_t = greedy ? 1.f : 1.0f / temp;
    const unsigned long long seed = seeds ? seeds[r] : 0ull;
    const unsigned int tix = token_index ? (unsigned int)token_index[r] : 0u;

    Best best{-INFINITY, 0x7fffffff};
    for (int v = threadIdx.x; v < V; v += blockDim.x) {
        float s = row[v];
        if (!greedy) s = __fadd_rn(__fmul_rn(s, inv_t), gumbel(seed, tix, (unsigned int)v));
        if (s > best.score || best.index == 0x7fffffff) best = Best{s, v};
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        Best other{__shfl_xor_sync(0xffffffffu, best.score, o), __shfl_xor_sync(0xffffffffu, best.index, o)};
        best = better(best, other);
    }
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (lane == 0) warp_best[warp] = best;
    __syncthreads();
    if (warp == 0) {
        const int n_warps = (blockDim.x + 31) >> 5;
        best = lane < n_warps ? warp_best[lane] : Best{-INFINITY, 0x7fffffff};
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            Best other{__shfl_xor_sync(0xffffffffu, best.score, o), __shfl_xor_sync(0xffffffffu, best.index, o)};
            best = better(best, other);
        }
        if (lane == 0) out[r] = best.index == 0x7fffffff ? 0 : best.index;
    }
}

// Large vocabularies: stage 1 scans a slice of the row per block and leaves its best
// (score, index) in scratch; stage 2 picks the best slice.  The winner is the same as
// in the one-block kernel: largest score, lowest index on a tie.
__global__ void sample_slices_kernel(const float* logits, long long ld, const float* temperature,
                                     const unsigned long long* seeds, const int* token_index,
                                     float* slice_score, int* slice_index, int V, int slice) {
    __shared__ Best warp_best[32];
    pdl_trigger();
    pdl_wait();
    const int r = blockIdx.y, sl = blockIdx.x;
    const float* row = logits + (size_t)r * ld;
    const float temp = temperature ? temperature[r] : 0.f;
    const bool greedy = !(temp > 0.f);
    const float inv_t = greedy ? 1.f : 1.0f / temp;
    const unsigned long long seed = seeds ? seeds[r] : 0ull;
    const unsigned int tix = token_index ? (unsigned int)token_index[r] : 0u;
    const int begin = sl * slice, end = min(begin + slice, V);
    Best best{-INFINITY, 0x7fffffff};
    for (int v = begin + threadIdx.x; v < end; v += blockDim.x) {
        float s = row[v];
        if (!greedy) s = __fadd_rn(__fmul_rn(s, inv_t), gumbel(seed, tix, (unsigned int)v));
        if (s > best.score || best.index == 0x7fffffff) best = Best{s, v};
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        Best other{__shfl_xor_sync(0xffffffffu, best.score, o), __shfl_xor_sync(0xffffffffu, best.index, o)};
        best = better(best, other);
    }
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (lane == 0) warp_best[warp] = best;
    __syncthreads();
    if (warp == 0) {
        const int n_warps = (blockDim.x + 31) >> 5;
        best = lane < n_warps ? warp_best[lane] : Best{-INFINITY, 0x7fffffff};
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            Best other{__shfl_xor_sync(0xffffffffu, best.score, o), __shfl_xor_sync(0xffffffffu, best.index, o)};
            best = better(best, other);
        }
        if (lane == 0) {
            slice_score[(size_t)r * gridDim.x + sl] = best.score;
            slice_index[(size_t)r * gridDim.x + sl] = best.index;
        }
    }
}

__global__ void sample_pick_kernel(const float* slice_score, const int* slice_index,
                                   int* out, int n_slices) {
    pdl_trigger();
    pdl_wait();
    const int r = blockIdx.x;
    Best best{-INFINITY, 0x7fffffff};
    for (int i = threadIdx.x; i < n_slices; i += 32)
        best = better(best, Best{slice_score[(size_t)r * n_slices + i], slice_index[(size_t)r * n_slices + i]});
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        Best other{__shfl_xor_sync(0xffffffffu, best.score, o), __shfl_xor_sync(0xffffffffu, best.index, o)};
        best = better(best, other);
    }
    if (threadIdx.x == 0) out[r] = best.index == 0x7fffffff ? 0 : best.index;
}

// Slices the two-stage path cuts a row of V entries into (0: use the one-block kernel).
PYRE_API int pyre_sample_slices(int V) { return V >= 16384 ? (V + 4095) / 4096 : 0; }

// logits [R, V] fp32 with row stride ld; temperature [R] fp32 (null = all greedy);
// seeds [R] uint64 and token_index [R] int32 (may be null when all rows are greedy);
// out [R] int32.  scratch: R * pyre_sample_slices(V) * 2 words, needed when that is not 0.
PYRE_API int pyre_sample(const float* logits, long long ld, const float* temperature,
                         const unsigned long long* seeds, const int* token_index, int* out, int n_rows, int V,
                         void* scratch, cudaStream_t stream) {
    if (n_rows <= 0) return 0;
    if (V <= 0) return PYRE_ERR_BAD_ARG;
    const int n_slices = pyre_sample_slices(V);
    if (n_slices > 0) {
        if (!scratch) return PYRE_ERR_BAD_ARG;
        float* sc = (float*)scratch;
        int* ix = (int*)scratch + (size_t)n_rows * n_slices;
        pyre_launch(sample_slices_kernel, dim3(dim3(n_slices, n_rows)), dim3(256), 0, stream, logits, ld, temperature, seeds, token_index, sc, ix, V, 4096);
        PYRE_LAUNCH_CHECK();
        pyre_launch(sample_pick_kernel, dim3(n_rows), dim3(32), 0, stream, sc, ix, out, n_slices);
        PYRE_LAUNCH_CHECK();
        return 0;
    }
    const int threads = V >= 8192 ? 1024 : (V >= 1024 ? 256 : 64);
    pyre_launch(sample_kernel, dim3(n_rows), dim3(threads), 0, stream, logits, ld, temperature, seeds, token_index, out, V);
    PYRE_LAUNCH_CHECK();
    return 0;
}

// ---------------------------------------------------------------------------
// Sampling from the likeliest tokens of a row (temperature > 0):
//   w_i = exp((l_i - max l) / T); the order of the tokens: larger l first, of equal ones the lower index.
//   top_k  > 0 : the first k tokens            (0: all)
//   top_p  < 1 : of those the shortest prefix whose mass is at least p of theirs, one token at least
//   min_p  > 0 : of those the tokens with w_i >= min_p
// All three keep a prefix of the order.  The token is argmax over it of (l_i - max l) / T + g(seed, index, i), the noise of the kernels
// above.  A row without a filter is chosen from as above, bit for bit; a NaN counts as -inf.
//
// A cluster of CTAs shares a row; each keeps its slice in shared memory where it fits.  Masses are whole numbers
// (w 2^31, summed in 64 bits), so neither the order of the additions nor the cluster's size can move a border: results do not depend on them.
//   1. max l.
//   2. a histogram by distance from it in steps of 1/64 (count and mass per step; l decides the step alone and in order), of the tokens less than
//      NEAR steps away; the others' mass stays in registers.  The step in which the k-th token or the p-th part of the mass lies follows.
//   3. the tokens up to that step, some hundreds as a rule, go to the first CTA's list, and the others are done.  It ranks the ones of that step by
//      (l, index): the border token; and once more for p after k.  Then noise for the tokens up to the border.
// Where the border lies further away, or more tokens lie before it than the list holds (flat rows, rows of equal entries):
//   2. the histogram of all tokens,
//   3. the border step's tokens alone go to the list; if they are more than it holds, their span of (l, index) is cut into as many steps again, until
//      they fit.
//   4. all CTAs look for the tokens up to the border.
// ---------------------------------------------------------------------------
namespace {
namespace cg = cooperative_groups;
typedef unsigned long long u64;
constexpr int F_THREADS = 512, F_WARPS = F_THREADS / 32, BINS = 2048, NEAR = F_THREADS, LISTED = 512, NEAR_LISTED = 2048, MAX_CLUSTER = 8;
constexpr float BINS_PER_NAT = 64.f;

struct FilterParams {
    const float* logits;
    long long ld;
    const float* temperature;
    const u64* seeds;
    const int* token_index;
    const int* top_k;
    const float* top_p;
    const float* min_p;
    int* out;
    int V, slice;      // entries per CTA, a multiple of 4
    int resident;      // the slice lies in shared memory
};

struct FilterShared {
    unsigned near_count[NEAR], near_low[NEAR], near_high[NEAR];      // mass: high 2^32 + low
    union {
        struct {
            unsigned count[BINS], low[BINS], high[BINS];
        };
        struct {
            u64 near_list[NEAR_LISTED];
            unsigned near_mass[NEAR_LISTED];
        };
    };
    u64 list[LISTED];
    unsigned list_mass[LISTED];
    u64 slots[2][MAX_CLUSTER][2];                     // what the cluster's CTAs tell each other
    u64 warp_u64[2][F_WARPS];
    Best warp_best[F_WARPS];
    Best cluster_best[MAX_CLUSTER];
    unsigned near_listed;
    int near_step;                                    // the tokens up to this step are listed; < 0: too far or too many
    u64 rest;                                         // the mass beyond the near steps
    // the step that a search ended in (`above`: before it), or the border
    int step;
    u64 above_count, above_mass, inside, border, border_mass;
    unsigned listed;
};

// A number whose order as an unsigned integer is that of the floats (-0 and +0 are one).
__device__ __forceinline__ unsigned order_key(float l) {
    const unsigned u = __float_as_uint(l + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float entry(float l) { return l == l ? l : -INFINITY; }

__global__ void __launch_bounds__(F_THREADS)
sample_filtered_kernel(const FilterParams p) {
    extern __shared__ float4 dyn[];
    __shared__ FilterShared sh;
    cg::cluster_group cluster = cg::this_cluster();
    const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int r = blockIdx.x / C;
    pdl_trigger();
    cluster.sync();      // the others have started: their shared memory can be written to
    pdl_wait();
    const float* row = p.logits + (size_t)r * p.ld;
    const int begin = min(rank * p.slice, p.V), n = min(p.slice, p.V - begin);
    const float T = p.temperature ? p.temperature[r] : 0.f;
    const bool greedy = !(T > 0.f);
    const float inv_t = greedy ? 1.f : 1.0f / T;
    const u64 seed = p.seeds ? p.seeds[r] : 0ull;
    const unsigned tix = p.token_index ? (unsigned)p.token_index[r] : 0u;
    const int k = p.top_k ? p.top_k[r] : 0;
    const float top_p = p.top_p ? p.top_p[r] : 1.f, min_p = p.min_p ? fminf(p.min_p[r], 1.f) : 0.f;
    const bool by_count = k > 0 && k < p.V, by_mass = top_p < 1.f;
    const bool filtered = !greedy && (k > 0 || by_mass || min_p > 0.f);

    int turn = 0;
    // every CTA's pair of numbers, known to all threads of the cluster afterwards in sh.slots[returned]
    auto exchange = [&](u64 a, u64 b) {      // a, b: in the first C threads
        const int at = turn;
        turn ^= 1;
        if (tid < C) {
            FilterShared* other = cluster.map_shared_rank(&sh, tid);
            other->slots[at][rank][0] = a;
            other->slots[at][rank][1] = b;
        }
        cluster.sync();
        return at;
    };
    auto best_of_block = [&](Best& best) {      // in thread 0
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
            best = better(best, Best{__shfl_xor_sync(0xffffffffu, best.score, o), __shfl_xor_sync(0xffffffffu, best.index, o)});
        if (lane == 0) sh.warp_best[warp] = best;
        __syncthreads();
        if (tid == 0)
            for (int w = 1; w < F_WARPS; ++w) best = better(best, sh.warp_best[w]);
    };
    auto finish = [&](Best best) {
        best_of_block(best);
        if (tid == 0) cluster.map_shared_rank(&sh, 0)->cluster_best[rank] = best;
        cluster.sync();
        if (rank == 0 && tid == 0) {
            for (int c = 1; c < C; ++c) best = better(best, sh.cluster_best[c]);
            p.out[r] = best.index == 0x7fffffff ? 0 : best.index;
        }
    };
    Best best{-INFINITY, 0x7fffffff};
    if (!filtered) {
        for (int i = tid; i < n; i += F_THREADS) {
            float s = entry(row[begin + i]);
            if (!greedy) s = __fadd_rn(__fmul_rn(s, inv_t), gumbel(seed, tix, (unsigned)(begin + i)));
            if (s > best.score || best.index == 0x7fffffff) best = Best{s, begin + i};
        }
        finish(best);
        return;
    }

    // 1. the slice, and the largest entry
    const float* held = row + begin;
    float most = -INFINITY;
    const int shift16 = (int)(((uintptr_t)held >> 2) & 3), head = min(n, (4 - shift16) & 3), body = (n - head) / 4;
    // f(four entries, the index of the first) for all of the slice, by whole vectors but for its ends (of which the first entry alone counts)
    auto vectors = [&](const float* src, auto f) {
        if (tid < head) f(make_float4(entry(src[tid]), -INFINITY, -INFINITY, -INFINITY), tid, 1);
        constexpr int AHEAD = 4;
        for (int i = tid; i < body; i += AHEAD * F_THREADS) {
            float4 v[AHEAD];
#pragma unroll
            for (int q = 0; q < AHEAD; ++q)
                if (i + q * F_THREADS < body) v[q] = *reinterpret_cast<const float4*>(src + head + 4 * (i + q * F_THREADS));
#pragma unroll
            for (int q = 0; q < AHEAD; ++q)
                if (i + q * F_THREADS < body)
                    f(make_float4(entry(v[q].x), entry(v[q].y), entry(v[q].z), entry(v[q].w)), head + 4 * (i + q * F_THREADS), 4);
        }
        const int last = head + 4 * body + tid;
        if (last < n) f(make_float4(entry(src[last]), -INFINITY, -INFINITY, -INFINITY), last, 1);
    };
    {
        float* const mine = reinterpret_cast<float*>(dyn) + shift16;      // the same place within 16 bytes
        vectors(held, [&](const float4& v, int i, int count) {
            most = fmaxf(most, fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)));
            if (!p.resident) return;
            if (count == 4) *reinterpret_cast<float4*>(mine + i) = v;
            else mine[i] = v.x;
        });
        if (p.resident) held = mine;
    }
    // f(entry, its index) for all of the slice
    auto entries = [&](auto f) {
        vectors(held, [&](const float4& v, int i, int count) {
            f(v.x, i);
            if (count == 4) { f(v.y, i + 1); f(v.z, i + 2); f(v.w, i + 3); }
        });
    };
    most = warp_max(most);
    if (lane == 0) sh.warp_best[warp].score = most;
    sh.near_count[tid] = sh.near_low[tid] = sh.near_high[tid] = 0;
    if (tid == 0) {
        sh.listed = sh.near_listed = 0;
        sh.rest = 0;
    }
    __syncthreads();
    if (tid < C)
        for (int w = 0; w < F_WARPS; ++w) most = fmaxf(most, sh.warp_best[w].score);
    {
        const int at = exchange(__float_as_uint(most), 0);
        for (int c = 0; c < C; ++c) most = fmaxf(most, __uint_as_float((unsigned)sh.slots[at][c][0]));
    }
    // (the distance of the largest entry is zero even where it is infinite or the temperature's inverse is)
    auto distance = [&](float l) { return l == most ? 0.f : (most - l) * inv_t; };
    auto mass_of = [&](float d) { return __float2uint_rn(expf(-d) * 2147483648.f); };
    auto first_step = [&](float d) { return (int)fminf(d * BINS_PER_NAT, (float)(BINS - 1)); };
    auto composite = [&](float l, int i) { return (u64)order_key(l) << 32 | (unsigned)~(unsigned)(begin + i); };
    auto tally = [&](int b, unsigned f) {
        atomicAdd(&sh.count[b], 1u);
        const unsigned old = atomicAdd(&sh.low[b], f);
        if (old + f < old) atomicAdd(&sh.high[b], 1u);
    };

    // Adds up the cluster's histograms and finds the step in which the sum (of counts or masses) reaches `target`: sh.step, .above_*, .inside in every
    // CTA.  Each CTA adds up a run of steps.  target 0: only the whole mass is wanted (returned).
    auto locate = [&](bool mass, u64 target, u64 before_count, u64 before_mass, bool add) {
        const int run = BINS / C, per = (run + F_THREADS - 1) / F_THREADS, first = rank * run;
        cluster.sync();
        if (add && C > 1) {
            for (int b = first + tid; b < first + run; b += F_THREADS) {
                u64 sum = ((u64)sh.high[b] << 32) + sh.low[b];
                unsigned count = sh.count[b];
                for (int c = 1; c < C; ++c) {
                    const FilterShared* other = cluster.map_shared_rank(&sh, (rank + c) % C);
                    sum += ((u64)other->high[b] << 32) + other->low[b];
                    count += other->count[b];
                }
                sh.high[b] = (unsigned)(sum >> 32);
                sh.low[b] = (unsigned)sum;
                sh.count[b] = count;
            }
            __syncthreads();
        }
        // a thread's own steps, then the threads before it
        u64 counts = 0, masses = 0;
        for (int q = 0; q < per; ++q) {
            const int b = tid * per + q;
            if (b < run) {
                counts += sh.count[first + b];
                masses += ((u64)sh.high[first + b] << 32) + sh.low[first + b];
            }
        }
        u64 c_up = counts, m_up = masses;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 a = __shfl_up_sync(0xffffffffu, c_up, o), b = __shfl_up_sync(0xffffffffu, m_up, o);
            if (lane >= o) { c_up += a; m_up += b; }
        }
        if (lane == 31) { sh.warp_u64[0][warp] = c_up; sh.warp_u64[1][warp] = m_up; }
        __syncthreads();
        u64 c_all = 0, m_all = 0;
        for (int w = 0; w < F_WARPS; ++w) {
            if (w == warp) { c_up += c_all; m_up += m_all; }
            c_all += sh.warp_u64[0][w];
            m_all += sh.warp_u64[1][w];
        }
        const int at = exchange(c_all, m_all);
        u64 c_before = before_count, m_before = before_mass, m_whole = before_mass;
        for (int c = 0; c < C; ++c) {
            if (c < rank) { c_before += sh.slots[at][c][0]; m_before += sh.slots[at][c][1]; }
            m_whole += sh.slots[at][c][1];
        }
        if (target == 0) return m_whole;
        u64 c_at = c_before + c_up - counts, m_at = m_before + m_up - masses;      // before the thread's own
        if ((mass ? m_at : c_at) < target && (mass ? m_at + masses : c_at + counts) >= target) {
            int b = tid * per;
            for (;; ++b) {
                const u64 c = sh.count[first + b], m = ((u64)sh.high[first + b] << 32) + sh.low[first + b];
                if ((mass ? m_at + m : c_at + c) >= target) {
                    for (int q = 0; q < C; ++q) {
                        FilterShared* other = cluster.map_shared_rank(&sh, q);
                        other->step = first + b;
                        other->above_count = c_at;
                        other->above_mass = m_at;
                        other->inside = c;
                    }
                    break;
                }
                c_at += c;
                m_at += m;
            }
        }
        cluster.sync();
        return m_whole;
    };
    // From the first histogram (already added up where !add) to the border token: sh.border and, with everything before it, its mass, in every CTA.
    auto search = [&](bool mass, u64 target, bool add) {
        locate(mass, target, 0, 0, add);
        const int step0 = sh.step;
        u64 from = 0, to = ~0ull;      // the span of (l, index) left
        auto inside = [&](float l, int i) {
            const u64 key = composite(l, i);
            return first_step(distance(l)) == step0 && key >= from && key <= to;
        };
        bool spanned = false;
        for (int level = 0; sh.inside > LISTED && level < 7; ++level) {      // 64 bits, eleven a time
            if (!spanned) {
                u64 low = ~0ull, high = 0;
                entries([&](float l, int i) {
                    if (inside(l, i)) {
                        low = min(low, composite(l, i));
                        high = max(high, composite(l, i));
                    }
                });
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) {
                    low = min(low, __shfl_xor_sync(0xffffffffu, low, o));
                    high = max(high, __shfl_xor_sync(0xffffffffu, high, o));
                }
                __syncthreads();
                if (lane == 0) { sh.warp_u64[0][warp] = low; sh.warp_u64[1][warp] = high; }
                __syncthreads();
                for (int w = 0; w < F_WARPS; ++w) {
                    low = min(low, sh.warp_u64[0][w]);
                    high = max(high, sh.warp_u64[1][w]);
                }
                const int at = exchange(low, high);
                for (int c = 0; c < C; ++c) {
                    low = min(low, sh.slots[at][c][0]);
                    high = max(high, sh.slots[at][c][1]);
                }
                from = low;
                to = high;
                spanned = true;
            }
            int shift = 0;
            while ((to - from) >> shift >= BINS) ++shift;
            const u64 before_count = sh.above_count, before_mass = sh.above_mass;
            cluster.sync();      // all have read the last histogram and what it gave
            for (int b = tid; b < BINS; b += F_THREADS) sh.count[b] = sh.low[b] = sh.high[b] = 0;
            __syncthreads();
            entries([&](float l, int i) {
                if (inside(l, i)) tally((int)((to - composite(l, i)) >> shift), mass_of(distance(l)));
            });
            locate(mass, target, before_count, before_mass, true);
            to -= (u64)sh.step << shift;
            from = max(from, to - ((1ull << shift) - 1));
        }
        // the tokens of the span, ranked by the first CTA
        FilterShared* const lead = cluster.map_shared_rank(&sh, 0);
        entries([&](float l, int i) {
            if (inside(l, i)) {
                const unsigned at = atomicAdd(&lead->listed, 1u);
                if (at < LISTED) {
                    lead->list[at] = composite(l, i);
                    lead->list_mass[at] = mass_of(distance(l));
                }
            }
        });
        cluster.sync();
        if (rank == 0) {
            const int count = min((int)sh.listed, LISTED);
            for (int q = tid; q < count; q += F_THREADS) {
                const u64 key = sh.list[q], own = sh.list_mass[q];
                u64 c_at = sh.above_count, m_at = sh.above_mass;
                for (int j = 0; j < count; ++j)
                    if (sh.list[j] > key) { ++c_at; m_at += sh.list_mass[j]; }
                if (mass ? m_at < target && m_at + own >= target : c_at + 1 == target)
                    for (int c = 0; c < C; ++c) {
                        FilterShared* other = cluster.map_shared_rank(&sh, c);
                        other->border = key;
                        other->border_mass = m_at + own;
                    }
            }
            __syncthreads();
            if (tid == 0) sh.listed = 0;
        }
        cluster.sync();
    };

    u64 border = 0;
    if (most == -INFINITY) {
        if (rank == 0 && tid == 0) p.out[r] = 0;      // nothing left to choose from
        cluster.sync();
        return;
    }
    auto clear = [&]() {
        for (int b = tid; b < BINS; b += F_THREADS) sh.count[b] = sh.low[b] = sh.high[b] = 0;
        __syncthreads();
    };
    auto share = [&](u64 whole) { return max(1ull, (u64)ceil((double)top_p * (double)whole)); };
    auto score = [&](float l, unsigned index) {
        const float d = distance(l);
        if (min_p > 0.f && !(expf(-d) >= min_p)) return;
        const float s = entry(__fadd_rn(-d, gumbel(seed, tix, index)));
        best = better(best, Best{s, (int)index});
    };
    if (by_count || by_mass) {
        FilterShared* const lead = cluster.map_shared_rank(&sh, 0);
        // 2. the near steps; what lies beyond them counts where the whole mass is wanted
        u64 rest = 0;
        entries([&](float l, int) {
            const float d = distance(l);
            if (d * BINS_PER_NAT < (float)NEAR) {
                const int b = first_step(d);
                const unsigned f = mass_of(d);
                atomicAdd(&sh.near_count[b], 1u);
                const unsigned old = atomicAdd(&sh.near_low[b], f);
                if (old + f < old) atomicAdd(&sh.near_high[b], 1u);
            }
            else if (!by_count && d < 23.f) rest += mass_of(d);      // (below 2^-32 beyond)
        });
        if (!by_count) {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) rest += __shfl_xor_sync(0xffffffffu, rest, o);
            if (lane == 0 && rest) atomicAdd(&lead->rest, rest);
        }
        __syncthreads();
        if (rank != 0) {
            const unsigned count = sh.near_count[tid], low = sh.near_low[tid];
            if (count) {
                atomicAdd(&lead->near_count[tid], count);
                const unsigned old = atomicAdd(&lead->near_low[tid], low);
                const unsigned high = sh.near_high[tid] + (old + low < old);
                if (high) atomicAdd(&lead->near_high[tid], high);
            }
        }
        cluster.sync();
        // the steps' sums up to and with each one of the first CTA's threads', and the search among them
        u64 counts = 0, masses = 0, c_up = 0, m_up = 0, target = k;
        auto near_step = [&](bool mass, u64 target) {      // all threads of the first CTA; the step in sh.step, what is before it in sh.above_*
            if (tid == 0) sh.step = -1;
            __syncthreads();
            if ((mass ? m_up : c_up) >= target && (mass ? m_up - masses : c_up - counts) < target) {
                sh.step = tid;
                sh.above_count = c_up - counts;
                sh.above_mass = m_up - masses;
                sh.inside = counts;
            }
            __syncthreads();
        };
        if (rank == 0) {
            counts = c_up = sh.near_count[tid];
            masses = m_up = ((u64)sh.near_high[tid] << 32) + sh.near_low[tid];
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const u64 x = __shfl_up_sync(0xffffffffu, c_up, o), y = __shfl_up_sync(0xffffffffu, m_up, o);
                if (lane >= o) { c_up += x; m_up += y; }
            }
            if (lane == 31) { sh.warp_u64[0][warp] = c_up; sh.warp_u64[1][warp] = m_up; }
            __syncthreads();
            u64 m_all = 0;
            for (int w = 0; w < F_WARPS; ++w) {
                if (w < warp) { c_up += sh.warp_u64[0][w]; m_up += sh.warp_u64[1][w]; }
                m_all += sh.warp_u64[1][w];
            }
            if (!by_count) target = share(m_all + sh.rest);
            near_step(!by_count, target);
            if (tid < C) {
                const bool fits = sh.step >= 0 && sh.above_count + sh.inside <= NEAR_LISTED;
                cluster.map_shared_rank(&sh, tid)->near_step = fits ? sh.step : -1;
            }
        }
        cluster.sync();
        const int near = sh.near_step;
        if (near >= 0) {
            // 3. the tokens up to that step
            entries([&](float l, int i) {
                if (distance(l) * BINS_PER_NAT < (float)(near + 1)) {
                    const unsigned at = atomicAdd(&lead->near_listed, 1u);
                    if (at < NEAR_LISTED) {
                        lead->near_list[at] = composite(l, i);
                        lead->near_mass[at] = mass_of(distance(l));
                    }
                }
            });
            cluster.sync();
            if (rank != 0) return;      // nothing of theirs is read any more
            const int listed = min((int)sh.near_listed, NEAR_LISTED);
            auto value = [&](u64 key) {
                const unsigned u = (unsigned)(key >> 32);
                return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
            };
            // the border token, from the ones of sh.step alone where they fit into the short list, else from all listed ones
            auto rank_step = [&](bool mass, u64 target) {
                const bool brief = sh.inside <= LISTED;
                if (brief) {
                    for (int q = tid; q < listed; q += F_THREADS) {
                        const u64 key = sh.near_list[q];
                        if (first_step(distance(value(key))) == sh.step) {
                            const unsigned at = atomicAdd(&sh.listed, 1u);
                            if (at < LISTED) {
                                sh.list[at] = key;
                                sh.list_mass[at] = sh.near_mass[q];
                            }
                        }
                    }
                    __syncthreads();
                }
                const int count = brief ? min((int)sh.listed, LISTED) : listed;
                const u64* const keys = brief ? sh.list : sh.near_list;
                const unsigned* const of = brief ? sh.list_mass : sh.near_mass;
                for (int q = tid; q < count; q += F_THREADS) {
                    const u64 key = keys[q], own = of[q];
                    u64 c_at = brief ? sh.above_count : 0, m_at = brief ? sh.above_mass : 0;
                    for (int j = 0; j < count; ++j)
                        if (keys[j] > key) { ++c_at; m_at += of[j]; }
                    if (mass ? m_at < target && m_at + own >= target : c_at + 1 == target) {
                        sh.border = key;
                        sh.border_mass = m_at + own;
                    }
                }
                __syncthreads();
                if (tid == 0) sh.listed = 0;
                __syncthreads();
            };
            rank_step(!by_count, target);
            if (by_count && by_mass) {
                target = share(sh.border_mass);
                near_step(true, target);
                rank_step(true, target);
            }
            const u64 border = sh.border;
            for (int q = tid; q < listed; q += F_THREADS) {
                const u64 key = sh.near_list[q];
                if (key >= border) score(value(key), ~(unsigned)key);
            }
            best_of_block(best);
            if (tid == 0) p.out[r] = best.index == 0x7fffffff ? 0 : best.index;
            return;
        }
        // (flat rows) all steps
        auto histogram = [&]() {
            clear();
            entries([&](float l, int) {
                const float d = distance(l);
                tally(first_step(d), mass_of(d));
            });
        };
        histogram();
        u64 whole = 0;
        bool added = false;
        if (by_count) {
            search(false, (u64)k, true);
            border = sh.border;
            whole = sh.border_mass;
            if (by_mass) {      // the first histogram again (the search has added it up, or cut it into finer steps)
                __syncthreads();
                histogram();
            }
        } else {
            whole = locate(true, 0, 0, 0, true);
            added = true;
        }
        if (by_mass) {
            search(true, share(whole), !added);
            border = sh.border;
        }
    }
    entries([&](float l, int i) {
        if (composite(l, i) >= border) score(l, (unsigned)(begin + i));
    });
    finish(best);
}
}  // namespace

// logits [R, V] fp32 with row stride ld; temperature [R], seeds [R], token_index [R] (null where all rows are greedy); top_k [R] int32 (0: all), top_p [R]
// (1: all), min_p [R] (0: all), each may be null; out [R] int32.
// cluster: CTAs per row (1, 2, 4, 8), 0 for the kernel's own choice.
PYRE_API int pyre_sample_filtered(const float* logits, long long ld, const float* temperature, const unsigned long long* seeds,
                                  const int* token_index, const int* top_k, const float* top_p, const float* min_p, int* out, int n_rows,
                                  int V, int cluster, cudaStream_t stream) {
    if (n_rows <= 0) return 0;
    if (V <= 0 || (temperature && (!seeds || !token_index))) return PYRE_ERR_BAD_ARG;
    if (cluster < 0 || cluster > MAX_CLUSTER || (cluster & (cluster - 1))) return PYRE_ERR_BAD_ARG;
    // CTAs per row: as many as keep two to an SM busy, and as two slices in an SM's shared memory ask for
    int C = cluster > 0 ? cluster : 1;
    while (!cluster && C < MAX_CLUSTER && ((n_rows * (long long)C < 2 * pyre_sm_count() && V > 2048 * C) || ceil_div(V, C) > 76 * 256)) C *= 2;
    FilterParams p = {logits, ld, temperature, seeds, token_index, top_k, top_p, min_p, out, V, (ceil_div(V, C) + 3) / 4 * 4, 0};
    size_t bytes = (size_t)p.slice * 4 + 16;
    p.resident = bytes <= 190 * 1024;
    if (!p.resident) bytes = 0;
    static bool configured[PYRE_MAX_DEVICES] = {};      // the attribute is per device
    bool& done = configured[pyre_current_device()];
    if (!done) {
        const cudaError_t e = cudaFuncSetAttribute(sample_filtered_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 190 * 1024);
        if (e != cudaSuccess) return (int)e;
        done = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)n_rows * C);
    cfg.blockDim = dim3(F_THREADS);
    cfg.dynamicSmemBytes = bytes;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = C;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pyre_pdl_enabled() ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, sample_filtered_kernel, p);
    if (e != cudaSuccess) return (int)e;
    PYRE_LAUNCH_CHECK();
    return 0;
}
