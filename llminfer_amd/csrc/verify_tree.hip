// Drafted tokens against the target's logits on gfx950 (no counterpart in the reference). With x the logits behind a node, T the
// temperature, m the row's maximum: weight(t) = exp((x[t] - m) / T), p(t) = weight(t) / sum of weights. See llmi_hip_verify_tree
// for what is accepted and drawn.
//
// Two launches. The first reads every row once, a workgroup per slice of 4096 tokens: maximum, its lowest index, sum of the weights
// relative to the slice's maximum. The second, sampling, has a workgroup per slice too: each joins the slices of all rows (a few lanes a row),
// decides the nodes for itself on one wavefront (a node per lane, sets of nodes as 64-bit words), and sums what is left of
// the last accepted node's row over its slice; the one that comes last finds the slice and the token. Greedy it is one workgroup, and the
// row's maximum is the token.
//
// Weights are fp32: the exponent is formed as a pair (product and its rounding error, so that (x - m) / T is not rounded to 24
// bits before the exponential), the exponential is the hardware's. A thread adds its sixteen weights of a slice in fp32, everything above that in
// fp64: whichever of two neighbouring tokens a sum falls on then depends on the weights' own rounding alone.

// What bounds it: the stream of the rows in the first launch (26 x 151936 fp32 in 6 us), dependent trips to memory in the second. 6 rows of 32000 with
// draft logits 14 us, 26 of 151936 greedy 9.7, 64 of 151936 in bf16 sampled 18.7 (one workgroup that decides and draws: 51, 17, 191).

#include <hip/hip_runtime.h>
#include <float.h>
#include <stdint.h>

#include "llmi_internal.h"

namespace llmi {
namespace {

constexpr int kSlice = 4096;
constexpr int kThreads = 256;
constexpr int kEach = kSlice / kThreads;  // tokens of a slice per thread
constexpr int kNodes = LLMI_TREE_MAX_NODES;

struct Part {
    double sum;     // of the slice's weights, relative to its maximum
    float max;      // -inf: no weight in the slice
    int32_t arg;    // lowest index of the maximum, -1 if there is none
};

struct VerifyArgs {
    const void* target;
    const void* draft;  // optional
    int64_t target_stride, draft_stride;
    const int32_t* tokens;
    const int32_t* parents;  // optional
    const float* uniform;
    int32_t* path;
    int32_t* result;
    Part* parts;        // [rows][slices]: the target's rows, then the draft's
    double* left;       // [slices]: what is left of the last node's weights
    uint32_t* arrived;  // workgroups of the second launch that have left their sum
    int32_t nodes, vocab, slices;
    float c_hi, c_lo;   // log2(e) / temperature, as a sum of two floats; 0: greedy
};

// A logit as the definition takes it: NaN without weight (a maximum is the operand that is a number), +inf the largest finite number.
__device__ __forceinline__ float clean(float x) { return fminf(fmaxf(x, -INFINITY), FLT_MAX); }
__device__ __forceinline__ float logit(const float* row, int64_t t) { return clean(row[t]); }
__device__ __forceinline__ float logit(const uint16_t* row, int64_t t) { return clean(__builtin_bit_cast(float, (uint32_t)row[t] << 16)); }

// A thread's tokens of a slice: chunks of 16 bytes (four or eight tokens), the workgroup's chunks side by side. Token e of thread i is
// token place<T>(i, e) of the slice. Rows may start anywhere: the loads need no alignment.
template <typename T>
constexpr int kChunk = 16 / (int)sizeof(T);
template <typename T>
__device__ __forceinline__ int place(int thread, int e) {
    return ((e / kChunk<T>)*kThreads + thread) * kChunk<T> + e % kChunk<T>;
}
template <typename T>
__device__ __forceinline__ void load_slice(const T* row, int slice, int vocab, float (&v)[kEach]) {
    struct __attribute__((packed, aligned(sizeof(T)))) Chunk {
        T x[kChunk<T>];
    };
    const int64_t first = (int64_t)slice * kSlice;
#pragma unroll
    for (int c = 0; c < kEach / kChunk<T>; ++c) {
        const int64_t t = first + place<T>((int)threadIdx.x, c * kChunk<T>);
        if (t + kChunk<T> <= vocab) {
            const Chunk x = *reinterpret_cast<const Chunk*>(row + t);
#pragma unroll
            for (int e = 0; e < kChunk<T>; ++e) v[c * kChunk<T> + e] = logit(x.x, e);
        } else {
#pragma unroll
            for (int e = 0; e < kChunk<T>; ++e) v[c * kChunk<T> + e] = t + e < vocab ? logit(row, t + e) : -INFINITY;
        }
    }
}

// exp((x - m) / T). (-inf, and NaN where there is no maximum, are far below: weight 0.)
__device__ __forceinline__ float weight(float x, float m, float c_hi, float c_lo) {
    const float d = fmaxf(x - m, -1e30f);
    const float t = d * c_hi;
    const float lo = __builtin_fmaf(d, c_lo, __builtin_fmaf(d, c_hi, -t));
    const float e = __builtin_amdgcn_exp2f(t);
    return __builtin_fmaf(e, lo * 0.69314718f, e);
}

struct Top {
    float max;
    int32_t arg;
};
__device__ __forceinline__ Top better(Top a, Top b) {
    const bool b_wins = b.max > a.max || (b.max == a.max && (uint32_t)b.arg < (uint32_t)a.arg);  // (-1 is the highest)
    return b_wins ? b : a;
}

// x of a lane's partner in step S of a fold: neighbours, pairs, fours, eights of a row of 16 lanes, rows, halves of the wavefront. After step S
// all of 2^(S + 1) lanes that lie together have the fold.
template <int S>
__device__ __forceinline__ int partner(int x) {
    constexpr int ctrl[4] = {0xB1, 0x4E, 0x141, 0x140};
    if constexpr (S < 4) {
        return __builtin_amdgcn_update_dpp(0, x, ctrl[S], 0xf, 0xf, false);
    } else {
        const bool upper = threadIdx.x & (S == 4 ? 16 : 32);
        const auto h = S == 4 ? __builtin_amdgcn_permlane16_swap((unsigned)x, (unsigned)x, false, false)
                              : __builtin_amdgcn_permlane32_swap((unsigned)x, (unsigned)x, false, false);
        const unsigned h0 = h[0], h1 = h[1];  // (the lower halves' values, the upper halves')
        return (int)(upper ? h0 : h1);
    }
}
template <int S>
__device__ __forceinline__ float partner(float x) { return __builtin_bit_cast(float, partner<S>(__builtin_bit_cast(int, x))); }
template <int S>
__device__ __forceinline__ double partner(double x) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    const uint64_t lo = (uint32_t)partner<S>((int)(uint32_t)u), hi = (uint32_t)partner<S>((int)(u >> 32));
    return __builtin_bit_cast(double, hi << 32 | lo);
}
template <int S>
__device__ __forceinline__ Top partner(Top x) { return Top{partner<S>(x.max), partner<S>(x.arg)}; }

// Folds over groups of `lanes` lanes (a power of two, the same for all), the result in every lane.
template <int S = 0, typename V, typename F>
__device__ __forceinline__ V lanes_fold(V x, int lanes, F&& f) {
    if constexpr (S < 6) {
        if (lanes > 1 << S) return lanes_fold<S + 1>(f(x, partner<S>(x)), lanes, f);
    }
    return x;
}
__device__ __forceinline__ Top lanes_top(Top x, int lanes) {
    return lanes_fold(x, lanes, [](Top a, Top b) { return better(a, b); });
}
__device__ __forceinline__ double lanes_sum(double x, int lanes) {
    return lanes_fold(x, lanes, [](double a, double b) { return a + b; });
}
template <typename V>
__device__ __forceinline__ V lane_value(V x, int lane) {
    if constexpr (sizeof(V) == 8) {
        const uint64_t u = __builtin_bit_cast(uint64_t, x);
        const uint64_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)u, lane), hi = (uint32_t)__builtin_amdgcn_readlane((int)(u >> 32), lane);
        return __builtin_bit_cast(V, hi << 32 | lo);
    } else {
        return __builtin_bit_cast(V, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), lane));
    }
}

template <typename T, bool GREEDY>
__global__ __launch_bounds__(kThreads) void verify_stats_kernel(VerifyArgs a) {
    __shared__ float tops[kThreads / 64];
    __shared__ double sums[kThreads / 64];
    __shared__ uint32_t arg_s;
    const int slice = blockIdx.x, row = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const bool of_draft = row >= a.nodes;
    const T* x = static_cast<const T*>(of_draft ? a.draft : a.target) + (of_draft ? (row - a.nodes) * a.draft_stride : row * a.target_stride);
    float v[kEach];
    load_slice(x, slice, a.vocab, v);
    if (threadIdx.x == 0) {
        arg_s = ~0u;
        if (slice == 0 && row == 0) *a.arrived = 0u;
    }
    float mine = v[0];
#pragma unroll
    for (int e = 1; e < kEach; ++e) mine = fmaxf(mine, v[e]);
    float max = lanes_fold(mine, 64, [](float p, float q) { return fmaxf(p, q); });
    if (lane == 0) tops[wave] = max;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) max = fmaxf(max, tops[w]);
    if (mine == max && max > -INFINITY) {  // (the few threads that have it)
        int arg = 0;
#pragma unroll
        for (int e = kEach - 1; e >= 0; --e) arg = v[e] == max ? place<T>((int)threadIdx.x, e) : arg;  // (places ascend with e)
        atomicMin(&arg_s, (uint32_t)(slice * kSlice + arg));
    }
    double sum = 0.0;
    if constexpr (!GREEDY) {
        float s = 0.0f;
#pragma unroll
        for (int e = 0; e < kEach; ++e) s += weight(v[e], max, a.c_hi, a.c_lo);
        sum = lanes_sum(s, 64);
        if (lane == 0) sums[wave] = sum;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        if constexpr (!GREEDY) sum = (sums[0] + sums[1]) + (sums[2] + sums[3]);
        a.parts[(int64_t)row * a.slices + slice] = Part{sum, max, (int32_t)arg_s};
    }
}

// What the nodes' decision leaves for the token behind the path.
struct Walk {
    Top tops[2 * kNodes];
    double sums[2 * kNodes];
    int32_t refused[kNodes];
    uint32_t alike[kThreads / 64][kNodes];  // sixteen nodes each: same parent (low half), same token
    int32_t last, refused_n, count;
    int32_t tried;  // a draft's token was tried behind the last node, and refused
};

// All rows' slices joined, `lanes` lanes a row; then the nodes. `writes`: this workgroup writes the path.
template <typename T, bool GREEDY>
__device__ __forceinline__ void walk(const VerifyArgs& a, Walk& w, bool writes) {
    const int rows = a.draft ? 2 * a.nodes - 1 : a.nodes;
    int lanes = 64;
    while (lanes * rows > kThreads) lanes >>= 1;
    // What the nodes need is asked for ahead of the slices.
    const T* target = static_cast<const T*>(a.target);
    const T* draft = static_cast<const T*>(a.draft);
    const int i = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int parent = -1, token = -1;
    float u = 0.0f, x_p = -INFINITY, x_q = -INFINITY;
    if (i > 0 && i < a.nodes) {
        parent = a.parents ? a.parents[i] : i - 1;
        token = a.tokens[i];
    }
    const bool valid = parent >= 0 && parent < i && token >= 0 && token < a.vocab;
    const int at = valid ? parent : 0;
    if constexpr (!GREEDY) {
        if (valid && wave == 0) {
            u = a.uniform[i];
            x_p = logit(target + at * a.target_stride, token);
            if (a.draft) x_q = logit(draft + at * a.draft_stride, token);
        }
    }
    // Which nodes have this one's parent and which its token, sixteen nodes to a wavefront. (A loop over siblings on one wavefront, their
    // values handed on one by one, took 10 us at 64 nodes.)
    if (a.parents) {
        const int key = valid ? parent : -1;
        uint32_t alike = 0u;
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            alike |= lane_value(key, 16 * wave + k) == key ? 1u << k : 0u;
            if constexpr (!GREEDY) alike |= lane_value(token, 16 * wave + k) == token ? 0x10000u << k : 0u;
        }
        w.alike[wave][i] = alike;
    }
    {
        const int r = (int)threadIdx.x / lanes, l = (int)threadIdx.x % lanes;
        const bool mine = r < rows;
        const Part* parts = a.parts + (int64_t)(mine ? r : 0) * a.slices;
        // (sixteen slices at a time asked for together, the running maximum and sum of a softmax)
        Top top{-INFINITY, -1};
        double sum = 0.0;
        for (int s0 = l; s0 < a.slices; s0 += 16 * lanes) {
            Part p[16];
#pragma unroll
            for (int x = 0; x < 16; ++x) {
                const int s = s0 + x * lanes;
                p[x] = parts[min(s, a.slices - 1)];
                if (s >= a.slices) p[x] = Part{0.0, -INFINITY, -1};
            }
            const float before = top.max;
#pragma unroll
            for (int x = 0; x < 16; ++x) top = better(top, Top{p[x].max, p[x].arg});
            if constexpr (!GREEDY) {
                sum *= weight(before, top.max, a.c_hi, a.c_lo);
#pragma unroll
                for (int x = 0; x < 16; ++x) sum += p[x].sum * weight(p[x].max, top.max, a.c_hi, a.c_lo);
            }
        }
        const float own = top.max;
        top = lanes_top(top, lanes);
        if constexpr (!GREEDY) sum = lanes_sum(sum * weight(own, top.max, a.c_hi, a.c_lo), lanes);
        if (mine && l == 0) {
            w.tops[r] = top;
            w.sums[r] = sum;
        }
    }
    __syncthreads();
    if (wave == 0) {
        const uint64_t valid_set = __ballot(valid);
        uint64_t siblings = 0, equals = 0;
        if (a.parents) {
#pragma unroll
            for (int x = 0; x < kThreads / 64; ++x) {
                siblings |= (uint64_t)(w.alike[x][i] & 0xffffu) << 16 * x;
                equals |= (uint64_t)(w.alike[x][i] >> 16) << 16 * x;
            }
            siblings &= valid ? valid_set & ((1ull << i) - 1) : 0ull;  // earlier ones
        }
        bool accept = false, again = false;
        if constexpr (GREEDY) {
            accept = valid && w.tops[at].arg == token;
        } else {
            const double mass = valid ? (double)weight(x_p, w.tops[at].max, a.c_hi, a.c_lo) : 0.0;
            if (a.draft) {
                const double q = valid ? (double)weight(x_q, w.tops[a.nodes + at].max, a.c_hi, a.c_lo) : 0.0;
                accept = mass > 0.0 && (double)u * q * w.sums[at] < mass * (valid ? w.sums[a.nodes + at] : 0.0);
            } else {
                // a token that has been refused is not tried again, and its mass is taken away once
                again = valid && (siblings & equals);
                uint64_t taken = valid ? siblings & __ballot(valid && !again) : 0ull;
                double before = 0.0;
                while (__any(taken != 0)) {  // (in index order; every lane takes part in the hand-over)
                    const int j = taken ? __ffsll((unsigned long long)taken) - 1 : 0;
                    const double mass_j = __shfl(mass, j);
                    before += taken ? mass_j : 0.0;
                    taken &= taken - 1;
                }
                accept = valid && !again && mass > 0.0 && (double)u * (w.sums[at] - before) < mass;
            }
        }
        // the first accepted child of each node, then those whose parents are on the path
        const bool first = accept && !(siblings & __ballot(accept));
        uint64_t on = 1, before = 0;
        while (on != before) {  // (a step for each node of the path)
            before = on;
            on |= __ballot(first && (on >> at & 1));
        }
        const int count = __popcll(on), last = 63 - __clzll(on);
        const bool gone = valid && parent == last && !again;
        const uint64_t tried_set = __ballot(gone), gone_set = a.draft ? 0ull : tried_set;
        if (!a.draft && gone) w.refused[__popcll(gone_set & ((1ull << i) - 1))] = token;
        if (i == 0) {
            w.last = last;
            w.count = count;
            w.refused_n = __popcll(gone_set);
            w.tried = tried_set != 0;
        }
        if (writes) {
            if (on >> i & 1) a.path[__popcll(on & ((1ull << i) - 1))] = i;
            if (i >= count && i < a.nodes) a.path[i] = -1;
            if (i == 0) a.result[0] = count;
        }
    }
    __syncthreads();
}

// What is left of a thread's weights at the last accepted node. (The draft's distribution is taken away where a token that came from it has been
// refused. Behind the last node of a chain, and behind one whose child's token is outside the vocabulary, a chain shorter than its rows, none has.)
template <typename T>
__device__ __forceinline__ void left_of(const VerifyArgs& a, const Walk& w, int slice, float (&v)[kEach], double (&left)[kEach]) {
    const int last = w.last;
    const float m = w.tops[last].max;
    load_slice(static_cast<const T*>(a.target) + last * a.target_stride, slice, a.vocab, v);
    if (a.draft && w.tried) {
        float q[kEach];
        load_slice(static_cast<const T*>(a.draft) + last * a.draft_stride, slice, a.vocab, q);
        const float m_q = w.tops[a.nodes + last].max;
        const double p_1 = 1.0 / w.sums[last], q_1 = w.sums[a.nodes + last] > 0.0 ? 1.0 / w.sums[a.nodes + last] : 0.0;
#pragma unroll
        for (int e = 0; e < kEach; ++e)
            left[e] = fmax(weight(v[e], m, a.c_hi, a.c_lo) * p_1 - weight(q[e], m_q, a.c_hi, a.c_lo) * q_1, 0.0);
    } else {
#pragma unroll
        for (int e = 0; e < kEach; ++e) left[e] = weight(v[e], m, a.c_hi, a.c_lo);
        for (int i = 0; i < w.refused_n; ++i) {
            const int32_t t = w.refused[i] - slice * kSlice;
            if (t < 0 || t >= kSlice) continue;
#pragma unroll
            for (int e = 0; e < kEach; ++e)
                if (place<T>((int)threadIdx.x, e) == t) left[e] = 0.0;
        }
    }
}

// Inclusive sum over the lanes up to this one: shifts inside the rows of 16 lanes, then the rows' last values handed on.
template <int CTRL, int ROWS>
__device__ __forceinline__ double moved(double x) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    const uint64_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, ROWS, 0xf, false);
    const uint64_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(u >> 32), CTRL, ROWS, 0xf, false);
    return __builtin_bit_cast(double, hi << 32 | lo);  // (lanes without a source: 0)
}
__device__ __forceinline__ double lanes_upto(double x) {
    x += moved<0x111, 0xf>(x);
    x += moved<0x112, 0xf>(x);
    x += moved<0x114, 0xf>(x);
    x += moved<0x118, 0xf>(x);
    x += moved<0x142, 0xa>(x);  // lane 15 of rows 0 and 2 to rows 1 and 3
    x += moved<0x143, 0xc>(x);  // lane 31 to rows 2 and 3
    return x;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void verify_greedy_kernel(VerifyArgs a) {
    __shared__ Walk w;
    walk<T, true>(a, w, true);
    if (threadIdx.x == 0) a.result[1] = w.tops[w.last].arg;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void verify_draw_kernel(VerifyArgs a) {
    constexpr int kWaves = kThreads / 64, kChunks = kEach / kChunk<T>;
    __shared__ Walk w;
    __shared__ double sums[kChunks * kWaves], goal_s, before_s;
    __shared__ int32_t last_one, slice_s, token_s, positive_s;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, slice = blockIdx.x;
    walk<T, false>(a, w, slice == 0);
    if (w.tops[w.last].arg < 0) {  // (no token has a weight)
        if (slice == 0 && threadIdx.x == 0) a.result[1] = -1;
        return;
    }
    float v[kEach];
    double left[kEach];
    left_of<T>(a, w, slice, v, left);
    double sum = 0.0;
#pragma unroll
    for (int e = 0; e < kEach; ++e) sum += left[e];
    sum = lanes_sum(sum, 64);
    if (lane == 0) sums[wave] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        sum = (sums[0] + sums[1]) + (sums[2] + sums[3]);
        __hip_atomic_store(&a.left[slice], sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        last_one = __hip_atomic_fetch_add(a.arrived, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t)a.slices - 1u;
    }
    __syncthreads();
    if (!last_one) return;
    // the slice: the first one where the sum passes the goal, or the last one with a weight
    if (wave == 0) {
        auto left_in = [&](int s) { return s < a.slices ? __hip_atomic_load(&a.left[s], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0.0; };
        const double x0 = left_in(lane);
        double total = lane_value(lanes_upto(x0), 63);
        for (int s0 = 64; s0 < a.slices; s0 += 64) total = lane_value(total + lanes_upto(left_in(s0 + lane)), 63);
        const double goal = (double)a.uniform[0] * total;
        double before = 0.0, found_before = 0.0;
        int found = -1;
        for (int s0 = 0; s0 < a.slices; s0 += 64) {
            const double x = s0 ? left_in(s0 + lane) : x0;
            const double upto = before + lanes_upto(x);
            const uint64_t positive = __ballot(x > 0.0), passed = __ballot(x > 0.0 && upto > goal);
            const int l = passed ? __ffsll((unsigned long long)passed) - 1 : 63 - __clzll(positive);
            if (positive) {
                found = s0 + l;
                found_before = l ? lane_value(upto, l ? l - 1 : 0) : before;
            }
            if (passed) break;
            before = lane_value(upto, 63);
        }
        if (lane == 0) {
            slice_s = found;
            goal_s = goal;
            before_s = found_before;
            token_s = INT32_MAX;
            positive_s = -1;
        }
    }
    __syncthreads();
    const int found = slice_s;
    if (found < 0) {  // nothing is left
        if (threadIdx.x == 0) a.result[1] = w.tops[w.last].arg;
        return;
    }
    // the token, in the same way: sums in front of each chunk of each thread, in the order of the tokens
    left_of<T>(a, w, found, v, left);
    double upto[kChunks], own[kChunks];
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
        own[c] = 0.0;
#pragma unroll
        for (int e = 0; e < kChunk<T>; ++e) own[c] += left[c * kChunk<T> + e];
        upto[c] = lanes_upto(own[c]);
        if (lane == 63) sums[c * kWaves + wave] = upto[c];
    }
    __syncthreads();
    double at[kChunks], running = before_s;
#pragma unroll
    for (int c = 0; c < kChunks; ++c)
#pragma unroll
        for (int x = 0; x < kWaves; ++x) {
            at[c] = x == wave ? running + (upto[c] - own[c]) : at[c];
            running += sums[c * kWaves + x];
        }
    int token = INT32_MAX, positive = -1;  // (a thread's places ascend)
#pragma unroll
    for (int c = 0; c < kChunks; ++c)
#pragma unroll
        for (int e = 0; e < kChunk<T>; ++e) {
            const double y = left[c * kChunk<T> + e];
            const int t = place<T>((int)threadIdx.x, c * kChunk<T> + e);
            at[c] += y;
            positive = y > 0.0 ? t : positive;
            token = y > 0.0 && at[c] > goal_s ? min(token, t) : token;
        }
    token = lanes_fold(token, 64, [](int p, int q) { return min(p, q); });
    positive = lanes_fold(positive, 64, [](int p, int q) { return max(p, q); });
    if (lane == 0) {
        atomicMin(&token_s, token);
        atomicMax(&positive_s, positive);
    }
    __syncthreads();
    if (threadIdx.x == 0) a.result[1] = found * kSlice + (token_s != INT32_MAX ? token_s : positive_s);
}

template <typename T>
void launch(const VerifyArgs& a, int rows, hipStream_t stream) {
    const dim3 grid(a.slices, rows), block(kThreads);
    if (a.c_hi == 0.0f) {
        hipLaunchKernelGGL((verify_stats_kernel<T, true>), grid, block, 0, stream, a);
        hipLaunchKernelGGL((verify_greedy_kernel<T>), dim3(1), block, 0, stream, a);
    } else {
        hipLaunchKernelGGL((verify_stats_kernel<T, false>), grid, block, 0, stream, a);
        hipLaunchKernelGGL((verify_draw_kernel<T>), dim3(a.slices), block, 0, stream, a);
    }
}

}  // namespace

size_t verify_tree_workspace_bytes(int32_t node_num, int32_t vocab) {
    const size_t slices = ((size_t)vocab + kSlice - 1) / kSlice;
    return slices * (2 * (size_t)node_num * sizeof(Part) + sizeof(double)) + 16;
}

int launch_verify_tree(const llmi_verify_tree_args& args) {
    VerifyArgs a;
    a.target = args.target_logits;
    a.draft = args.node_num > 1 ? args.draft_logits : nullptr;
    a.target_stride = args.target_stride ? args.target_stride : args.vocab;
    a.draft_stride = args.draft_stride ? args.draft_stride : args.vocab;
    a.tokens = args.tokens;
    a.parents = args.parents;
    a.uniform = args.uniform;
    a.path = args.path;
    a.result = args.result;
    a.nodes = args.node_num;
    a.vocab = args.vocab;
    a.slices = (int32_t)(((int64_t)args.vocab + kSlice - 1) / kSlice);
    a.parts = static_cast<Part*>(args.workspace);
    a.left = reinterpret_cast<double*>(a.parts + (size_t)2 * a.nodes * a.slices);
    a.arrived = reinterpret_cast<uint32_t*>(a.left + a.slices);
    const double c = args.temperature > 0.0f ? 1.4426950408889634 / (double)args.temperature : 0.0;
    a.c_hi = (float)c;
    a.c_lo = (float)(c - (double)a.c_hi);
    const int rows = a.draft ? 2 * a.nodes - 1 : a.nodes;
    const hipStream_t stream = static_cast<hipStream_t>(args.stream);
    if (args.logits_type == LLMI_LOGITS_F32) launch<float>(a, rows, stream);
    else launch<uint16_t>(a, rows, stream);
    return check_launch();
}

}  // namespace llmi
