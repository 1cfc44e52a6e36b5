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

    // (a NaN is above nothing: it counts as -inf)
    Best best{-INFINITY, (int)threadIdx.x < V ? (int)threadIdx.x : 0x7fffffff};
    for (int v = threadIdx.x; v < V; v += blockDim.x) {
        float s = row[v];
        if (!greedy) s = __fadd_rn(__fmul_rn(s, inv_t), gumbel(seed, tix, (unsigned int)v));
        if (s > best.score) best = Best{s, v};
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
    Best best{-INFINITY, begin + (int)threadIdx.x < end ? begin + (int)threadIdx.x : 0x7fffffff};
    for (int v = begin + threadIdx.x; v < end; v += blockDim.x) {
        float s = row[v];
        if (!greedy) s = __fadd_rn(__fmul_rn(s, inv_t), gumbel(seed, tix, (unsigned int)v));
        if (s > best.score) best = Best{s, v};
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
// A cluster of CTAs shares a row; each keeps its slice in shared memory where two such CTAs fit on an SM or each has one to itself, else it reads it again (out of L2).  Masses
// are whole numbers (w 2^31, summed in 64 bits), so neither the order of the additions nor the cluster's size can move a border: results do
// not depend on them.  A token's mass is off by half a unit, beside what its exponential is (see mass_of): the mass before a border by 2^-32 of the
// best token's per token at most (152,064 tokens: 3.5e-5 of it, where all are cut off alike; some 5e-8 where they differ).
//   1. max l, and the largest entry of each block of 128: what follows reads the blocks again that hold entries it looks for.
//   2. k: as many blocks as k have an entry of at least t, where t is the k-th of their largest ones (or somewhat below): no token below t is among the first
//      k.  The tokens from t on, hardly more than k, go to the first CTA's list, and the other CTAs are done.  It ranks them by (l, index), which
//      gives the border token of k and of p after k, and adds the noise.
//   2'. p alone: a histogram of masses by distance (max l - l) / T in steps of 1/64 (l decides the step alone and in order) of the tokens less than NEAR steps
//      away; the others' mass stays in registers.  It gives the step in which the p-th part of the mass lies, whose tokens go to the list and are
//      ranked.  All CTAs look for the tokens up to the border.
//   3'. The tokens up to the border are gathered before they get their noise: they are few in any 32 neighbours, and a token's noise is some
//      hundred instructions.
//   Where that does not do (the border lies further away, more equal entries than the list holds, k beyond the blocks), `far_border` finds it: a histogram of
//   all tokens, and the span of (l, index) in question cut into as many steps again until its tokens fit.
// ---------------------------------------------------------------------------
namespace {
namespace cg = cooperative_groups;
typedef unsigned long long u64;
constexpr int F_THREADS = 512, F_WARPS = F_THREADS / 32, BINS = 2048, NEAR = 2 * F_THREADS, LISTED = 512, NEAR_LISTED = 2048, MAX_CLUSTER = 16;
constexpr float BINS_PER_NAT = 64.f;
constexpr int GATHERED = 6144, BLOCKS = 1216, ALL_BLOCKS = 4096;      // of a CTA, of a row

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
    unsigned near_low[NEAR], near_high[NEAR];      // mass: high 2^32 + low
    union {
        struct {
            unsigned count[BINS], low[BINS], high[BINS];
        };
        struct {
            u64 near_list[NEAR_LISTED];
            unsigned near_mass[NEAR_LISTED];
        };
        float all_most[ALL_BLOCKS];
        unsigned gathered[GATHERED];
    };
    float block_most[BLOCKS];
    u64 list[LISTED];
    unsigned list_mass[LISTED];
    u64 slots[2][MAX_CLUSTER][2];                     // what the cluster's CTAs tell each other
    u64 warp_u64[2][F_WARPS];
    Best warp_best[F_WARPS];
    Best cluster_best[MAX_CLUSTER];
    unsigned listed;
    unsigned near_own, near_pushed, near_base;        // the list: a CTA's own tokens from its end downwards, the other CTAs' from its start
    unsigned n_gathered;
    int near_step, near_kind;                         // what the first CTA has found: the step, and whether it will do (0: no)
    float near_least;                                 // the smallest entry to list
    u64 rest;                                         // the mass beyond the near steps
    // the step that a search ended in (`above`: before it), or the border
    int step;
    u64 above_count, above_mass, inside, border, border_mass, target;
};

// A number whose order as an unsigned integer is that of the floats (-0 and +0 are one), and back.
__device__ __forceinline__ unsigned order_key(float l) {
    const unsigned u = __float_as_uint(l + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float entry_of(u64 key) {
    const unsigned u = (unsigned)(key >> 32);
    return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ float entry(float l) { return l == l ? l : -INFINITY; }
// exp(-d) 2^31 as a whole number (1.44 d is off by 2^-24 of it, so a mass by 1e-7 d)
__device__ __forceinline__ unsigned mass_of(float d) { return __float2uint_rn(exp2f(fmaf(d, -1.44269504f, 31.f))); }
__device__ __forceinline__ int first_step(float d) { return (int)fminf(d * BINS_PER_NAT, (float)(BINS - 1)); }
__device__ __forceinline__ void tally(unsigned* count, unsigned* low, unsigned* high, int b, unsigned f) {
    atomicAdd(count + b, 1u);
    const unsigned old = atomicAdd(low + b, f);
    if (old + f < old) atomicAdd(high + b, 1u);
}

// A CTA's part of a row.
struct Slice {
    FilterShared& sh;
    cg::cluster_group cluster;
    int C, rank, begin, n, head, body;      // entries: begin .. begin + n; up to a 16-byte boundary, and whole vectors after it
    int blocks;                             // whose largest entries are known
    int turn;
    const float* held;
    float most, inv_t, top_p;

    // (the distance of the largest entry is zero even where it is infinite or the temperature's inverse is)
    __device__ __forceinline__ float distance(float l) const { return l == most ? 0.f : (most - l) * inv_t; }
    __device__ __forceinline__ u64 composite(float l, int i) const { return (u64)order_key(l) << 32 | (unsigned)~(unsigned)(begin + i); }
    __device__ __forceinline__ u64 share(u64 whole) const { return max(1ull, (u64)ceil((double)top_p * (double)whole)); }
    // f(four entries as they are, the index of the first, how many count) for all of the slice
    template <typename F> __device__ __forceinline__ void vectors(F f) const {
        const int tid = threadIdx.x;
        if (tid < head) f(make_float4(held[tid], -INFINITY, -INFINITY, -INFINITY), tid, 1);
        constexpr int AHEAD = 4;
        for (int i = tid; i < body; i += AHEAD * F_THREADS) {
            float4 v[AHEAD];
#pragma unroll
            for (int q = 0; q < AHEAD; ++q)
                if (i + q * F_THREADS < body) v[q] = *reinterpret_cast<const float4*>(held + head + 4 * (i + q * F_THREADS));
#pragma unroll
            for (int q = 0; q < AHEAD; ++q)
                if (i + q * F_THREADS < body) f(v[q], head + 4 * (i + q * F_THREADS), 4);
        }
        const int last = head + 4 * body + tid;
        if (last < n) f(make_float4(held[last], -INFINITY, -INFINITY, -INFINITY), last, 1);
    }
    // f(entry as it is, its index)
    template <typename F> __device__ __forceinline__ void entries(F f) const {
        vectors([&](const float4& v, int i, int count) {
            f(v.x, i);
            if (count == 4) { f(v.y, i + 1); f(v.z, i + 2); f(v.w, i + 3); }
        });
    }
    // put(place, entry, its index) for the entries from `least` to `largest` in the blocks (of 32 whole vectors) from `from` to `to`; the places are taken
    // from `counter`, a warp's at once (no thread may be elsewhere).
    template <typename F> __device__ __forceinline__ void pick(int from, int to, float least, float largest, unsigned* counter, F put) const {
        const int lane = threadIdx.x & 31;
        constexpr int AHEAD = 4;
        for (int b0 = from + (threadIdx.x >> 5); b0 < to; b0 += 32 * F_WARPS) {      // a warp's blocks lie F_WARPS apart
            const int b = b0 + lane * F_WARPS;
            unsigned hit = __ballot_sync(0xffffffffu, b < to && (b >= blocks || sh.block_most[b] >= least));
            while (hit) {
                float4 v[AHEAD];
                int at[AHEAD];
#pragma unroll
                for (int q = 0; q < AHEAD; ++q) {
                    at[q] = hit ? 32 * (b0 + (__ffs(hit) - 1) * F_WARPS) + lane : body;
                    hit &= hit - 1;
                    v[q] = at[q] < body ? *reinterpret_cast<const float4*>(held + head + 4 * at[q]) : make_float4(NAN, NAN, NAN, NAN);
                }
#pragma unroll
                for (int q = 0; q < AHEAD; ++q) {
                    const float l[4] = {v[q].x, v[q].y, v[q].z, v[q].w};
                    unsigned hits[4], before = 0;
                    int total = 0;
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        hits[c] = __ballot_sync(0xffffffffu, l[c] >= least && l[c] <= largest);
                        total += __popc(hits[c]);
                    }
                    if (!total) continue;
                    if (lane == 0) before = atomicAdd(counter, (unsigned)total);
                    before = __shfl_sync(0xffffffffu, before, 0);
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        if (hits[c] >> lane & 1) put(before + __popc(hits[c] & ((1u << lane) - 1)), l[c], head + 4 * at[q] + c);
                        before += __popc(hits[c]);
                    }
                }
            }
        }
    }
    __device__ __forceinline__ int all_blocks() const { return (body + 31) / 32; }
    // ... and for the entries off whole vectors
    template <typename F> __device__ __forceinline__ void pick_ends(float least, float largest, unsigned* counter, F put) const {
        auto end = [&](int i) {
            if (held[i] >= least && held[i] <= largest) put(atomicAdd(counter, 1u), held[i], i);
        };
        const int tid = threadIdx.x;
        if (tid < head) end(tid);
        if (head + 4 * body + tid < n) end(head + 4 * body + tid);
    }
    // f(entry, its index) for the entries from `least` to `largest`
    template <typename F> __device__ __forceinline__ void between(float least, float largest, F f) const {
        vectors([&](const float4& v, int i, int count) {
            if (!(fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)) >= least)) return;
            const float l[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (q < count && l[q] >= least && l[q] <= largest) f(l[q], i + q);
        });
    }
    // Every CTA's pair of numbers (in its first C threads), known to all threads of the cluster afterwards in sh.slots[returned].
    __device__ __forceinline__ int exchange(u64 a, u64 b) {
        const int at = turn;
        turn ^= 1;
        if (threadIdx.x < C) {
            FilterShared* other = cluster.map_shared_rank(&sh, threadIdx.x);
            other->slots[at][rank][0] = a;
            other->slots[at][rank][1] = b;
        }
        cluster.sync();
        return at;
    }
    // Of the first CTA's `count` listed tokens (key(q), mass(q)), the one with which `target` tokens or `target` mass are reached, `above_*` lying before
    // them all.
    template <typename K, typename M>
    __device__ __forceinline__ void rank_list(K key_of, M mass_at, int count, bool mass, u64 target, u64 above_count, u64 above_mass) const {
        for (int q = threadIdx.x; q < count; q += F_THREADS) {
            const u64 key = key_of(q), own = mass_at(q);
            u64 c_at = above_count, m_at = above_mass;
#pragma unroll 8
            for (int j = 0; j < count; ++j)
                if (key_of(j) > key) { ++c_at; m_at += mass_at(j); }
            if (mass ? m_at < target && m_at + own >= target : c_at + 1 == target) {
                sh.border = key;
                sh.border_mass = m_at + own;
            }
        }
        __syncthreads();
    }
    __device__ void clear() const {
        for (int b = threadIdx.x; b < BINS; b += F_THREADS) sh.count[b] = sh.low[b] = sh.high[b] = 0;
        __syncthreads();
    }
    __device__ u64 locate(bool mass, u64 target, u64 before_count, u64 before_mass, bool add);
    __device__ void refine(bool mass, u64 target, float least, float largest);
    __device__ __forceinline__ void search(bool mass, u64 target, bool add) {      // from the histogram of all tokens (already added up where !add)
        locate(mass, target, 0, 0, add);
        refine(mass, target, -INFINITY, INFINITY);
    }
    __device__ void histogram() const {
        clear();
        entries([&](float l, int) {
            const float d = distance(entry(l));
            tally(sh.count, sh.low, sh.high, first_step(d), mass_of(d));
        });
    }
};

// Adds up the cluster's histograms and finds the step in which the sum (of counts or masses) reaches `target`: sh.step, .above_*, .inside in every
// CTA.  Each CTA adds up a run of steps.  target 0: only the whole mass is wanted (returned).
__device__ __noinline__ u64 Slice::locate(bool mass, u64 target, u64 before_count, u64 before_mass, bool add) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
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
}

// From the step in which the target lies (sh.step, .above_*, .inside in every CTA; its entries lie from `least` to `largest`) to the border token: sh.border and, with everything before it, its
// mass, in every CTA.
__device__ __noinline__ void Slice::refine(bool mass, u64 target, float least, float largest) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int step0 = sh.step;
    u64 from = 0, to = ~0ull;      // the span of (l, index) left
    auto inside = [&](float l, int i) {
        const u64 key = composite(l, i);
        return first_step(distance(l)) == step0 && key >= from && key <= to;
    };
    auto each = [&](auto f) {
        if (least == -INFINITY) entries([&](float x, int i) { f(entry(x), i); });
        else between(least, largest, f);
    };
    for (int level = 0; sh.inside > LISTED && level < 7; ++level) {      // 64 bits, eleven a time
        if (level == 0) {
            u64 low = ~0ull, high = 0;
            each([&](float l, int i) {
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
        }
        int shift = 0;
        while ((to - from) >> shift >= BINS) ++shift;
        const u64 before_count = sh.above_count, before_mass = sh.above_mass;
        cluster.sync();      // all have read the last histogram and what it gave
        clear();
        each([&](float l, int i) {
            if (inside(l, i)) tally(sh.count, sh.low, sh.high, (int)((to - composite(l, i)) >> shift), mass_of(distance(l)));
        });
        locate(mass, target, before_count, before_mass, true);
        to -= (u64)sh.step << shift;
        from = max(from, to - ((1ull << shift) - 1));
    }
    // the tokens of the span, ranked by the first CTA
    FilterShared* const lead = cluster.map_shared_rank(&sh, 0);
    each([&](float l, int i) {
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
        rank_list([&](int q) { return sh.list[q]; }, [&](int q) { return sh.list_mass[q]; }, min((int)sh.listed, LISTED), mass, target, sh.above_count,
                  sh.above_mass);
        if (tid == 0) sh.listed = 0;
        if (tid > 0 && tid < C) {
            FilterShared* other = cluster.map_shared_rank(&sh, tid);
            other->border = sh.border;
            other->border_mass = sh.border_mass;
        }
    }
    cluster.sync();
}

// The border token wherever it lies (sh.border in every CTA).
__device__ __noinline__ void far_border(Slice& s, int k, bool by_count, bool by_mass) {
    s.histogram();
    u64 whole = 0;
    bool added = false;
    if (by_count) {
        s.search(false, (u64)k, true);
        whole = s.sh.border_mass;
        if (by_mass) {      // the histogram again (the search has added it up, or cut it into finer steps)
            __syncthreads();
            s.histogram();
        }
    } else {
        whole = s.locate(true, 0, 0, 0, true);
        added = true;
    }
    if (by_mass) s.search(true, s.share(whole), !added);
}

__global__ void __launch_bounds__(F_THREADS, 2)
sample_filtered_kernel(const FilterParams p) {
    extern __shared__ float4 dyn[];
    __shared__ FilterShared sh;
    cg::cluster_group cluster = cg::this_cluster();
    const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int r = blockIdx.x / C;
    pdl_trigger();
    for (int b = tid; b < NEAR; b += F_THREADS) sh.near_low[b] = sh.near_high[b] = 0;
    if (tid == 0) {
        sh.listed = sh.near_own = sh.near_pushed = 0;
        sh.rest = 0;
    }
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
    const int head = min(n, (int)((4 - ((uintptr_t)(row + begin) >> 2)) & 3));
    Slice s = {sh, cluster, C, rank, begin, n, head, (n - head) / 4, 0, 0, row + begin, -INFINITY, inv_t, top_p};

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
        s.entries([&](float l, int i) {
            float v = entry(l);
            if (!greedy) v = __fadd_rn(__fmul_rn(v, inv_t), gumbel(seed, tix, (unsigned)(begin + i)));
            best = better(best, Best{v, begin + i});
        });
        finish(best);
        return;
    }

    // 1. the slice, and the largest entry
    float most = -INFINITY;
    {
        float* const mine = reinterpret_cast<float*>(dyn) + (((uintptr_t)s.held >> 2) & 3);      // the same place within 16 bytes
        auto end = [&](int i) {
            most = fmaxf(most, s.held[i]);      // a NaN is passed over
            if (p.resident) mine[i] = s.held[i];
        };
        if (tid < head) end(tid);
        if (head + 4 * s.body + tid < n) end(head + 4 * s.body + tid);
        constexpr int AHEAD = 4;
        s.blocks = min(s.all_blocks(), BLOCKS);
        for (int b0 = warp; b0 < s.all_blocks(); b0 += AHEAD * F_WARPS) {
            float4 v[AHEAD];
#pragma unroll
            for (int q = 0; q < AHEAD; ++q) {
                const int i = 32 * (b0 + q * F_WARPS) + lane;
                v[q] = i < s.body ? *reinterpret_cast<const float4*>(s.held + head + 4 * i) : make_float4(NAN, NAN, NAN, NAN);
            }
#pragma unroll
            for (int q = 0; q < AHEAD; ++q) {
                const int b = b0 + q * F_WARPS, i = 32 * b + lane;
                const float four = entry(fmaxf(fmaxf(v[q].x, v[q].y), fmaxf(v[q].z, v[q].w)));
                most = fmaxf(most, four);
                const unsigned key = __reduce_max_sync(0xffffffffu, order_key(four));
                if (lane == 0 && b < s.blocks) sh.block_most[b] = entry_of((u64)key << 32);
                if (p.resident && i < s.body) *reinterpret_cast<float4*>(mine + head + 4 * i) = v[q];
            }
        }
        if (p.resident) s.held = mine;
    }
    // the blocks' largest entries, side by side in the first CTA
    const int per_cta = (p.slice + 127) / 128 + 1;
    const bool by_blocks = by_count && C * per_cta <= ALL_BLOCKS && per_cta <= BLOCKS && k <= p.V / 256;
    if (by_blocks) {
        __syncthreads();
        float* const all = cluster.map_shared_rank(&sh, 0)->all_most;
        for (int b = tid; b < per_cta; b += F_THREADS) all[rank * per_cta + b] = b < s.blocks ? sh.block_most[b] : -INFINITY;
    }
    most = warp_max(most);
    if (lane == 0) sh.warp_best[warp].score = most;
    __syncthreads();
    if (tid < C)
        for (int w = 0; w < F_WARPS; ++w) most = fmaxf(most, sh.warp_best[w].score);
    {
        const int at = s.exchange(__float_as_uint(most), 0);
        for (int c = 0; c < C; ++c) most = fmaxf(most, __uint_as_float((unsigned)sh.slots[at][c][0]));
    }
    s.most = most;
    if (most == -INFINITY) {
        if (rank == 0 && tid == 0) p.out[r] = 0;      // nothing left to choose from
        return;
    }
    auto score = [&](float l, unsigned index) {
        const float d = s.distance(l);
        if (min_p > 0.f && !(expf(-d) >= min_p)) return;
        best = better(best, Best{entry(__fadd_rn(-d, gumbel(seed, tix, index))), (int)index});
    };
    u64 border = 0;
    if (by_count || by_mass) {
        FilterShared* const lead = cluster.map_shared_rank(&sh, 0);
        // The tokens with entries from `least` to `largest` go to the first CTA's list: its own from the end downwards, the others' by way of lists of
        // their own from the start on (one counter for all of them would be waited for in turn).
        auto list = [&](float least, float largest) {
            auto put = [&](unsigned at, float l, int i) {
                if (at < NEAR_LISTED) {
                    sh.near_list[NEAR_LISTED - 1 - at] = s.composite(l, i);
                    sh.near_mass[NEAR_LISTED - 1 - at] = mass_of(s.distance(l));
                }
            };
            s.pick(0, s.all_blocks(), least, largest, &sh.near_own, put);
            s.pick_ends(least, largest, &sh.near_own, put);
            __syncthreads();
            if (rank != 0) {
                const unsigned count = sh.near_own;
                if (tid == 0 && count) sh.near_base = atomicAdd(&lead->near_pushed, count);
                __syncthreads();
                for (unsigned q = tid; q < count && q < NEAR_LISTED; q += F_THREADS)
                    if (sh.near_base + q < NEAR_LISTED) {
                        lead->near_list[sh.near_base + q] = sh.near_list[NEAR_LISTED - 1 - q];
                        lead->near_mass[sh.near_base + q] = sh.near_mass[NEAR_LISTED - 1 - q];
                    }
            }
            cluster.sync();
        };
        // (the first CTA's) how many there are, and where the q-th one is
        auto listed = [&]() { return (int)(sh.near_pushed + sh.near_own); };
        auto place = [&](int q) { return q < (int)sh.near_pushed ? q : NEAR_LISTED - 1 - (q - (int)sh.near_pushed); };
        auto choose = [&](int count) {      // among the listed ones, by the first CTA
            const u64 border = sh.border;
            for (int q = tid; q < count; q += F_THREADS) {
                const u64 key = sh.near_list[place(q)];
                if (key >= border) score(entry_of(key), ~(unsigned)key);
            }
            best_of_block(best);
            if (tid == 0) p.out[r] = best.index == 0x7fffffff ? 0 : best.index;
        };
        int kind = 0;
        if (by_blocks) {
            // 2. t, by the first CTA
            if (rank == 0) {
                const float* const all = sh.all_most;
                const int values = C * per_cta;
                float least = INFINITY;
                for (int q = tid; q < values; q += F_THREADS)
                    if (all[q] > -INFINITY) least = fminf(least, all[q]);
                least = -warp_max(-least);
                if (lane == 0) sh.warp_best[warp].score = least;
                __syncthreads();
                for (int w = 0; w < F_WARPS; ++w) least = fminf(least, sh.warp_best[w].score);
                // steps from the largest to the least of them; those up to the step with which they are k
                const float width = (most - least) * (1.f / (NEAR - 1));
                auto step_of = [&](float v) { return width > 0.f ? (int)fminf((most - v) / width, (float)(NEAR - 1)) : 0; };
                for (int q = tid; q < values; q += F_THREADS)
                    if (all[q] > -INFINITY) atomicAdd(&sh.near_low[step_of(all[q])], 1u);
                if (tid == 0) sh.step = -1;
                __syncthreads();
                const int mine = sh.near_low[2 * tid] + sh.near_low[2 * tid + 1];      // two steps a thread
                int up = mine;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int x = __shfl_up_sync(0xffffffffu, up, o);
                    if (lane >= o) up += x;
                }
                if (lane == 31) sh.warp_u64[0][warp] = up;
                __syncthreads();
                for (int w = 0; w < warp; ++w) up += (int)sh.warp_u64[0][w];
                if (up >= k && up - mine < k) sh.step = 2 * tid + 1;
                __syncthreads();
                float t = INFINITY;
                for (int q = tid; q < values; q += F_THREADS)
                    if (all[q] > -INFINITY && step_of(all[q]) <= sh.step) t = fminf(t, all[q]);
                t = -warp_max(-t);
                __syncthreads();
                if (lane == 0) sh.warp_best[warp].score = t;
                __syncthreads();
                if (tid < C) {
                    for (int w = 0; w < F_WARPS; ++w) t = fminf(t, sh.warp_best[w].score);
                    FilterShared* other = cluster.map_shared_rank(&sh, tid);
                    other->near_least = t;
                    other->near_kind = sh.step >= 0 && most < INFINITY ? 2 : 0;
                }
            }
            cluster.sync();
            if (sh.near_kind == 2) {
                const float t = sh.near_least;
                list(t, most);
                const int count = rank == 0 ? listed() : 0;
                if (rank == 0 && tid < C) cluster.map_shared_rank(&sh, tid)->near_kind = count <= NEAR ? 3 : 0;
                cluster.sync();
                if (sh.near_kind == 3) {
                    if (rank != 0) return;      // nothing of the others' is read any more
                    // each token's place, and the mass before it: the k-th one, then the one with which p of the mass is reached
                    u64 keys[2], before[2], own[2];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int q = tid + h * F_THREADS;
                        keys[h] = q < count ? sh.near_list[place(q)] : 0;
                        own[h] = q < count ? sh.near_mass[place(q)] : 0;
                        before[h] = 0;
                        int places = 0;
                        if (q < count) {
                            const int pushed = (int)sh.near_pushed;
#pragma unroll 4
                            for (int j = 0; j < pushed; ++j)
                                if (sh.near_list[j] > keys[h]) { ++places; before[h] += sh.near_mass[j]; }
#pragma unroll 4
                            for (int j = NEAR_LISTED - (count - pushed); j < NEAR_LISTED; ++j)
                                if (sh.near_list[j] > keys[h]) { ++places; before[h] += sh.near_mass[j]; }
                            if (places + 1 == k) {
                                sh.border = keys[h];
                                sh.border_mass = before[h] + own[h];
                            }
                        }
                    }
                    __syncthreads();
                    if (by_mass) {
                        const u64 target = s.share(sh.border_mass);
                        __syncthreads();
#pragma unroll
                        for (int h = 0; h < 2; ++h)
                            if (tid + h * F_THREADS < count && before[h] < target && before[h] + own[h] >= target) sh.border = keys[h];
                        __syncthreads();
                    }
                    choose(count);
                    return;
                }
            }
        } else if (!by_count && most < INFINITY && inv_t < 1e37f && inv_t > 0.f) {
            // 2'. the near steps, and the mass beyond them
            const float scale = inv_t * BINS_PER_NAT;      // a power of two apart: distances in steps are rounded as they are
            u64 rest = 0;
            s.entries([&](float l, int) {
                const float d = (most - l) * scale;      // (a NaN's is one, and lies on neither side)
                if (d < 23.f * BINS_PER_NAT) {           // (below 2^-32 beyond)
                    const unsigned f = mass_of(d * (1.f / BINS_PER_NAT));
                    if (d < (float)NEAR) {
                        const unsigned old = atomicAdd(&sh.near_low[(int)d], f);
                        if (old + f < old) atomicAdd(&sh.near_high[(int)d], 1u);
                    } else rest += f;
                }
            });
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) rest += __shfl_xor_sync(0xffffffffu, rest, o);
            if (lane == 0 && rest) atomicAdd(&lead->rest, rest);
            __syncthreads();
            if (rank != 0)
                for (int b = tid; b < NEAR; b += F_THREADS) {
                    const unsigned low = sh.near_low[b];
                    if (low) {
                        const unsigned old = atomicAdd(&lead->near_low[b], low);
                        const unsigned high = sh.near_high[b] + (old + low < old);
                        if (high) atomicAdd(&lead->near_high[b], high);
                    } else if (sh.near_high[b]) atomicAdd(&lead->near_high[b], sh.near_high[b]);
                }
            cluster.sync();
            u64 target = 0;
            // (the first CTA) the near step in which the sum of the masses from `above` on reaches the target, which is p of the whole if there is none
            // yet: sh.step, and what is before it in sh.above_mass
            auto locate_near = [&](u64 above) {
                u64 masses[2], up = 0;      // two steps a thread: the sums up to and with them
#pragma unroll
                for (int q = 0; q < 2; ++q) up += masses[q] = ((u64)sh.near_high[2 * tid + q] << 32) + sh.near_low[2 * tid + q];
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const u64 x = __shfl_up_sync(0xffffffffu, up, o);
                    if (lane >= o) up += x;
                }
                if (lane == 31) sh.warp_u64[0][warp] = up;
                if (tid == 0) sh.step = -1;
                __syncthreads();
                u64 all = 0;
                for (int w = 0; w < F_WARPS; ++w) {
                    if (w < warp) up += sh.warp_u64[0][w];
                    all += sh.warp_u64[0][w];
                }
                if (target == 0) target = s.share(all + sh.rest);
                up += above;
#pragma unroll
                for (int q = 1; q >= 0; --q) {
                    if (up >= target && up - masses[q] < target) {
                        sh.step = 2 * tid + q;
                        sh.above_mass = up - masses[q];
                    }
                    up -= masses[q];
                }
                __syncthreads();
            };
            if (rank == 0) {
                locate_near(0);
                if (tid < C) cluster.map_shared_rank(&sh, tid)->near_step = sh.step;
            }
            cluster.sync();
            const int step = sh.near_step;
            if (step >= 0) {
                // the entries of the step lie within these, rounding and all; its tokens alone are ranked
                const float T_step = T * (1.f / BINS_PER_NAT), slack = 4e-7f * (fabsf(most) + (float)(step + 1) * T_step);
                const float least = most - (float)(step + 1) * T_step - slack, largest = most - (float)step * T_step + slack;
                list(least, largest);
                if (rank == 0) {
                    const int count = listed();
                    const bool fits = count <= NEAR_LISTED;
                    const u64 before = sh.above_mass;
                    if (fits) {
                        // the span of (l, index) that the step's tokens take, cut into steps until few are left (each is compared with each then)
                        auto in_step = [&](u64 key) { return (int)((most - entry_of(key)) * scale) == step; };
                        u64 from = ~0ull, to = 0, above = sh.above_mass;
                        if (count > 192) {
                            for (int q = tid; q < count; q += F_THREADS) {
                                const u64 key = sh.near_list[place(q)];
                                if (in_step(key)) { from = min(from, key); to = max(to, key); }
                            }
#pragma unroll
                            for (int o = 16; o > 0; o >>= 1) {
                                from = min(from, __shfl_xor_sync(0xffffffffu, from, o));
                                to = max(to, __shfl_xor_sync(0xffffffffu, to, o));
                            }
                            if (lane == 0) { sh.warp_u64[0][warp] = from; sh.warp_u64[1][warp] = to; }
                            __syncthreads();
                            for (int w = 0; w < F_WARPS; ++w) {
                                from = min(from, sh.warp_u64[0][w]);
                                to = max(to, sh.warp_u64[1][w]);
                            }
                            __syncthreads();      // the warps' counts take the same places
                        } else {
                            from = 0;
                            to = ~0ull;
                        }
                        auto left = [&](u64 key) { return key >= from && key <= to && in_step(key); };
                        for (int level = 0; level < 7 && count > 192; ++level) {
                            int own = 0;
                            for (int q = tid; q < count; q += F_THREADS) own += left(sh.near_list[place(q)]);
                            own = __reduce_add_sync(0xffffffffu, own);
                            if (lane == 0) sh.warp_u64[0][warp] = own;
                            for (int b = tid; b < NEAR; b += F_THREADS) sh.near_low[b] = sh.near_high[b] = 0;
                            __syncthreads();
                            int few = 0;
                            for (int w = 0; w < F_WARPS; ++w) few += (int)sh.warp_u64[0][w];
                            if (few <= 64) break;
                            int shift = 0;
                            while ((to - from) >> shift >= NEAR) ++shift;
                            for (int q = tid; q < count; q += F_THREADS) {
                                const u64 key = sh.near_list[place(q)];
                                if (!left(key)) continue;
                                const int b = (int)((to - key) >> shift);
                                const unsigned f = sh.near_mass[place(q)], old = atomicAdd(&sh.near_low[b], f);
                                if (old + f < old) atomicAdd(&sh.near_high[b], 1u);
                            }
                            __syncthreads();
                            locate_near(above);
                            above = sh.above_mass;
                            to -= (u64)sh.step << shift;
                            from = max(from, to - ((1ull << shift) - 1));
                            __syncthreads();
                        }
                        for (int q = tid; q < count; q += F_THREADS) {
                            const u64 key = sh.near_list[place(q)];
                            if (left(key)) {
                                const unsigned at = atomicAdd(&sh.listed, 1u);
                                if (at < LISTED) {
                                    sh.list[at] = key;
                                    sh.list_mass[at] = sh.near_mass[place(q)];
                                }
                            }
                        }
                        __syncthreads();
                        s.rank_list([&](int q) { return sh.list[q]; }, [&](int q) { return sh.list_mass[q]; }, min((int)sh.listed, LISTED), true, target, 0, above);
                    }
                    if (tid == 0) sh.listed = 0;
                    if (tid < C) {
                        FilterShared* other = cluster.map_shared_rank(&sh, tid);
                        other->border = sh.border;
                        other->near_kind = fits ? 1 : 2;
                        other->step = step;
                        other->above_mass = before;
                        other->above_count = 0;
                        other->inside = LISTED + 1;
                        other->target = target;
                    }
                }
                cluster.sync();
                kind = sh.near_kind;
                if (kind == 2) {      // more (equal entries, as a rule) than the list holds
                    Slice copy = s;
                    copy.refine(true, sh.target, least, largest);
                }
            }
        }
        if (kind == 0) {
            __syncthreads();
            Slice copy = s;      // (its address is taken: the original stays in registers)
            far_border(copy, k, by_count, by_mass);
        }
        border = sh.border;
    }
    // 3'. gathered, then worked on.  What min_p may leave lies within a little more than -log(min_p) T of the largest entry.
    float least = border ? entry_of(border) : -INFINITY;
    if (min_p > 0.f) least = fmaxf(least, most - (0.01f - logf(min_p)) * T - 4e-7f * fabsf(most));
    auto put = [&](unsigned at, float, int i) {
        if (at < GATHERED) sh.gathered[at] = i;
    };
    // A round takes as many blocks as the list is sure to hold (all, if they are but twice as many), the next ones as many as the last round's share of entries
    // lets expect; what does not fit after all is taken again.  256 rows of 152,064, min_p 89 us with rounds of one size, 59 with these.  (Dense rows as
    // they lie, not gathered: 358 us against 341 where 90,000 of each row stay.)
    constexpr int ROUND = GATHERED / 128 - 1;      // blocks, and the ends
    const int all = s.all_blocks();
    for (int from = 0, span = all <= 2 * ROUND ? max(all, 1) : ROUND; from == 0 || from < all;) {
        __syncthreads();
        if (tid == 0) sh.n_gathered = 0;
        __syncthreads();
        s.pick(from, min(all, from + span), least, INFINITY, &sh.n_gathered, put);
        if (from == 0) s.pick_ends(least, INFINITY, &sh.n_gathered, put);
        __syncthreads();
        const int count = (int)sh.n_gathered;
        if (count > GATHERED) {
            span = ROUND;
            continue;
        }
        for (int q = tid; q < count; q += F_THREADS) {
            const int i = sh.gathered[q];
            const float l = s.held[i];
            if (s.composite(l, i) >= border) score(l, begin + i);
        }
        from += span;
        span = max(ROUND, (int)min((long long)all, (long long)span * (GATHERED * 3 / 4) / max(count, 1)));
    }
    finish(best);
}
}  // namespace

// logits [R, V] fp32 with row stride ld; temperature [R], seeds [R], token_index [R] (null where all rows are greedy); top_k [R] int32 (0: all), top_p [R]
// (1: all), min_p [R] (0: all), each may be null; out [R] int32.
// cluster: CTAs per row (1, 2, 4, 8, 16), 0 for the kernel's own choice.
PYRE_API int pyre_sample_filtered(const float* logits, long long ld, const float* temperature, const unsigned long long* seeds,
                                  const int* token_index, const int* top_k, const float* top_p, const float* min_p, int* out, int n_rows,
                                  int V, int cluster, cudaStream_t stream) {
    if (n_rows <= 0) return 0;
    if (V <= 0 || (temperature && (!seeds || !token_index))) return PYRE_ERR_BAD_ARG;
    if (cluster < 0 || cluster > MAX_CLUSTER || (cluster & (cluster - 1))) return PYRE_ERR_BAD_ARG;
    // A slice stays in shared memory where two such CTAs fit on an SM (228 KB, 1 KB of it for each CTA: 17,700 entries a slice), or where each CTA
    // has an SM to itself (19,700).
    constexpr int SM_BYTES = 233472, OWN_BYTES = (int)sizeof(FilterShared) + 1024;
    constexpr int RESIDENT = (SM_BYTES / 2 - OWN_BYTES) / 16 * 16, RESIDENT_ALONE = 77 * 1024;
    static_assert(RESIDENT > 0 && 2 * (RESIDENT + OWN_BYTES) <= SM_BYTES && RESIDENT_ALONE + OWN_BYTES <= SM_BYTES, "two CTAs, one CTA");
    auto slice_of = [&](int ctas) { return (ceil_div(V, ctas) + 3) / 4 * 4; };
    auto bytes_of = [&](int ctas) { return (long long)slice_of(ctas) * 4 + 16; };
    // CTAs per row.  152,064 entries, p, m, k and the temperature drawn for each row, us on 1 / 2 / 4 / 8 / 16 CTAs a row:
    //   k            1 row 21 / 16 / 13 / 11 / 11, 12 rows 28 / 21 / 16 / 14 / 14, 16 30 / 22 / 18 / 21 / 21, 64 39 / 29 / 23 / 38 / 57, 100 40 / 30 / 37 / 52 / 84,
    //                148 39 / 33 / 50 / 69 / 120, 200 45 / 54 / 57, 256 48 / 58 / 72; k and p 128 42 / 32 / 41, 256 48 / 58 / 73
    //   p alone      1 134 / 75 / 45 / 29 / 22, 16 195 / 107 / 66 / 48 / 43, 28 - / - / 74 / 51 / 59, 37 220 / 120 / 78 / 64 / 74, 64 236 / 135 / 84 / 90 / 118,
    //                100 254 / 149 / 116 / 131, 200 295 / 200 / 192 / 236, 256 313 / 242 / 232 / 294; of 65,536 entries 28 38 / 26 / 38 on 4 / 8 / 16, 256 139 / 117 / 126
    //                on 1 / 2 / 4; of 24,000 256 56 / 54 / 69; of 16,000 (one CTA holds the row) 39 / 39, of 8,000 21 / 30.  (What two CTAs gain on 256 rows is the rows'
    //                difference: where all keep 30,000 tokens they take 243 on one or two, 90,000 339.)
    //   of all kinds 8 115 / 64 / 37 / 25 / 20, 32 179 / 100 / 59 / 42 / 40, 48 187 / 105 / 65 / 50 / 55, 100 210 / 122 / 82 / 81 / 102, 256 230 / 151 / 137 / 163
    // (Rows of all kinds come with all three arrays, as rows with k and p do: they go by p where there are few and by k where there are more than SMs.)
    // Slices between the two limits are halved: 150 rows of 18,500 entries, k / p / rows of all kinds, 37 / 34 / 56 us on two CTAs, 47 / 43 / 66 on one that reads its
    // row again, 39 / 42 / 55 on one that has the SM; 74 rows of 75,000 36 / 66 / 43 on eight, 29 / 60 / 44 on four that read it again, 38 / 80 / 52 on four
    // that have an SM each.  (Not those of eight: see 28 and 37 rows of p alone.)
    const int sms = pyre_sm_count();
    const bool mass_alone = top_p && !top_k;
    int C = cluster > 0 ? cluster
            : n_rows <= (mass_alone ? sms / 8 : top_p ? sms / 4 : sms / 12) ? MAX_CLUSTER
            : mass_alone && n_rows <= sms / 4 ? 8
            : n_rows <= sms / 2 ? 4 : n_rows <= sms || (mass_alone && bytes_of(1) > RESIDENT) ? 2 : 1;
    while (!cluster && C > 1 && V <= 1024 * C) C /= 2;
    if (!cluster && C <= 4 && (long long)n_rows * C > sms && bytes_of(C) > RESIDENT && bytes_of(C) <= RESIDENT_ALONE) C *= 2;
    FilterParams p = {logits, ld, temperature, seeds, token_index, top_k, top_p, min_p, out, V, slice_of(C), 0};
    p.resident = bytes_of(C) <= ((long long)n_rows * C <= sms ? RESIDENT_ALONE : RESIDENT);
    const size_t bytes = p.resident ? (size_t)bytes_of(C) : 0;
    static bool configured[PYRE_MAX_DEVICES] = {};      // the attribute is per device
    bool& done = configured[pyre_current_device()];
    if (!done) {
        cudaError_t e = cudaFuncSetAttribute(sample_filtered_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, RESIDENT_ALONE);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(sample_filtered_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
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
