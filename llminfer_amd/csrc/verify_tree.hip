// Drafted tokens against the target's logits on gfx950 (no counterpart in the reference). With x the logits behind a node, T the
// temperature, m the row's maximum: weight(t) = exp((x[t] - m) / T), p(t) = weight(t) / sum of weights. See llmi_hip_verify_tree
// for what is accepted and drawn.
//
// Two launches. The first reads every row once, a workgroup per slice of 4096 tokens: maximum, its lowest index, sum of the weights
// relative to the slice's maximum. The second joins the slices, decides the nodes on one wavefront (a node per lane, sets of nodes as
// 64-bit words) and reads the last accepted node's row again for the token to draw.
//
// Weights are fp32: the exponent is formed as a pair (product and its rounding error, so that (x - m) / T is not rounded to 24
// bits before the exponential), the exponential is the hardware's. Their sums are fp64: whichever of two neighbouring tokens a sum
// falls on then depends on the weights' own rounding alone.

#include <hip/hip_runtime.h>
#include <float.h>
#include <stdint.h>

#include "llmi_internal.h"

namespace llmi {
namespace {

constexpr int kSlice = 4096;
constexpr int kStatThreads = 256;
constexpr int kWalkThreads = 1024;
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
    int32_t nodes, vocab, slices;
    float c_hi, c_lo;   // log2(e) / temperature, as a sum of two floats; 0: greedy
};

// A logit as the definition takes it: NaN without weight, +inf the largest finite number.
__device__ __forceinline__ float clean(float x) { return x != x ? -INFINITY : fminf(x, FLT_MAX); }
__device__ __forceinline__ float logit(const float* row, int64_t t) { return clean(row[t]); }
__device__ __forceinline__ float logit(const uint16_t* row, int64_t t) { return clean(__builtin_bit_cast(float, (uint32_t)row[t] << 16)); }

// exp((x - m) / T). Below 2^-126 there is nothing left of a weight.
__device__ __forceinline__ float weight(float x, float m, float c_hi, float c_lo) {
    const float d = x - m;
    const float t = d * c_hi;
    if (!(t >= -126.0f)) return 0.0f;  // (-inf and, with no maximum, NaN among them)
    const float lo = __builtin_fmaf(d, c_hi, -t) + d * c_lo;
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
__device__ __forceinline__ Top wave_top(Top x) {
    for (int s = 32; s; s >>= 1) x = better(x, Top{__shfl_xor(x.max, s), __shfl_xor(x.arg, s)});
    return x;
}
__device__ __forceinline__ double wave_sum64(double x) {
    for (int s = 32; s; s >>= 1) x += __shfl_xor(x, s);
    return x;
}

template <typename T>
__global__ __launch_bounds__(kStatThreads) void verify_stats_kernel(VerifyArgs a) {
    __shared__ Top tops[kStatThreads / 64];
    __shared__ double sums[kStatThreads / 64];
    const int slice = blockIdx.x, row = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const bool of_draft = row >= a.nodes;
    const T* x = static_cast<const T*>(of_draft ? a.draft : a.target) + (of_draft ? (row - a.nodes) * a.draft_stride : row * a.target_stride);
    constexpr int kEach = kSlice / kStatThreads;
    float v[kEach];
    Top top{-INFINITY, -1};
    const int64_t first = (int64_t)slice * kSlice + threadIdx.x;
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
        const int64_t t = first + e * kStatThreads;
        v[e] = t < a.vocab ? logit(x, t) : -INFINITY;
        if (v[e] > top.max) top = Top{v[e], (int32_t)t};
    }
    top = wave_top(top);
    if (lane == 0) tops[wave] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kStatThreads / 64; ++w) top = better(top, tops[w]);
    double sum = 0.0;
#pragma unroll
    for (int e = 0; e < kEach; ++e) sum += weight(v[e], top.max, a.c_hi, a.c_lo);
    sum = wave_sum64(sum);
    if (lane == 0) sums[wave] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kStatThreads / 64; ++w) sum += sums[w];
        a.parts[(int64_t)row * a.slices + slice] = Part{sum, top.max, top.arg};
    }
}

// What is left of token t's weight at the last accepted node.
struct Left {
    float m_p, m_q;
    double s_p, s_q;
    bool subtract;           // max(p - q, 0)
    int refused_n;
    const int32_t* refused;  // tokens without weight
};
template <typename T>
__device__ __forceinline__ double left_of(const VerifyArgs& a, const Left& f, const T* target, const T* draft, int64_t t) {
    double w = weight(logit(target, t), f.m_p, a.c_hi, a.c_lo);
    if (f.subtract) {
        const double q = f.s_q > 0.0 ? weight(logit(draft, t), f.m_q, a.c_hi, a.c_lo) / f.s_q : 0.0;
        w = fmax(w / f.s_p - q, 0.0);
    }
    for (int i = 0; i < f.refused_n; ++i)
        if (f.refused[i] == (int32_t)t) w = 0.0;
    return w;
}

// Sum over the lanes in front of this one.
__device__ __forceinline__ double wave_before(double x, int lane) {
    double s = x;
    for (int d = 1; d < 64; d <<= 1) {
        const double y = __shfl_up(s, d);
        if (lane >= d) s += y;
    }
    const double b = __shfl_up(s, 1);
    return lane ? b : 0.0;
}

template <typename T>
__global__ __launch_bounds__(kWalkThreads) void verify_walk_kernel(VerifyArgs a) {
    constexpr int kWaves = kWalkThreads / 64;
    __shared__ Top tops[2 * kNodes];
    __shared__ double sums[2 * kNodes];
    __shared__ int32_t refused[kNodes];
    __shared__ int32_t last_s, refused_s, slice_s;
    __shared__ double target_s, before_s;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int rows = a.draft ? 2 * a.nodes - 1 : a.nodes;
    const bool greedy = a.c_hi == 0.0f;
    for (int r = wave; r < rows; r += kWaves) {
        const Part* parts = a.parts + (int64_t)r * a.slices;
        Top top{-INFINITY, -1};
        for (int s = lane; s < a.slices; s += 64) top = better(top, Top{parts[s].max, parts[s].arg});
        top = wave_top(top);
        double sum = 0.0;
        for (int s = lane; s < a.slices; s += 64) sum += parts[s].sum * weight(parts[s].max, top.max, a.c_hi, a.c_lo);
        sum = wave_sum64(sum);
        if (lane == 0) {
            tops[r] = top;
            sums[r] = sum;
        }
    }
    __syncthreads();
    const T* target = static_cast<const T*>(a.target);
    const T* draft = static_cast<const T*>(a.draft);
    if (wave == 0) {
        const int i = lane;
        const int parent = i == 0 || i >= a.nodes ? -1 : a.parents ? a.parents[i] : i - 1;
        const int token = i > 0 && i < a.nodes ? a.tokens[i] : -1;
        const bool valid = parent >= 0 && parent < i && token >= 0 && token < a.vocab;
        const int at = valid ? parent : 0;
        bool accept = false, again = false;
        if (greedy) {
            accept = valid && tops[at].arg == token;
        } else {
            const double u = valid ? (double)a.uniform[i] : 0.0;
            const double mass = valid ? (double)weight(logit(target + at * a.target_stride, token), tops[at].max, a.c_hi, a.c_lo) : 0.0;
            if (a.draft) {
                const double q = valid ? (double)weight(logit(draft + at * a.draft_stride, token), tops[a.nodes + at].max, a.c_hi, a.c_lo) : 0.0;
                accept = mass > 0.0 && u * q * sums[at] < mass * (valid ? sums[a.nodes + at] : 0.0);
            } else {
                // earlier siblings, one after the other: whether one has this token, then what they have taken away
                // (every lane asks for lane j's values before any test: a lane that has left a test answers nobody)
                for (int j = 1; j < a.nodes; ++j) {
                    const int valid_j = __shfl((int)valid, j), parent_j = __shfl(parent, j), token_j = __shfl(token, j);
                    again |= valid && valid_j && j < i && parent_j == parent && token_j == token;
                }
                double before = 0.0;
                for (int j = 1; j < a.nodes; ++j) {
                    const int first_j = __shfl((int)(valid && !again), j), parent_j = __shfl(parent, j);
                    const double mass_j = __shfl(mass, j);
                    if (valid && first_j && j < i && parent_j == parent) before += mass_j;
                }
                accept = !again && mass > 0.0 && u * (sums[at] - before) < mass;
            }
        }
        // the first accepted child of each node, then those whose parents are on the path
        uint64_t on = 1;
        for (int j = 1; j < a.nodes; ++j) {
            const int valid_j = __shfl((int)valid, j), parent_j = __shfl(parent, j), accept_j = __shfl((int)accept, j);
            const int above = valid_j ? parent_j : -1;
            const uint64_t earlier = __ballot(lane < j && lane > 0 && parent == above && accept);
            if (above >= 0 && (on >> above & 1) && !earlier && accept_j) on |= 1ull << j;
        }
        const int count = __popcll(on), last = 63 - __clzll(on);
        if (lane < a.nodes) {
            if (on >> lane & 1) a.path[__popcll(on & ((1ull << lane) - 1))] = lane;
            if (lane >= count) a.path[lane] = -1;
        }
        const bool gone = valid && parent == last && !again;
        const uint64_t gone_set = a.draft ? 0ull : __ballot(gone);
        if (!a.draft && gone) refused[__popcll(gone_set & ((1ull << lane) - 1))] = token;
        if (lane == 0) {
            last_s = last;
            refused_s = __popcll(gone_set);
            a.result[0] = count;
        }
    }
    __syncthreads();
    const int last = last_s;
    if (greedy || tops[last].arg < 0) {
        if (threadIdx.x == 0) a.result[1] = tops[last].arg;
        return;
    }
    const bool subtract = a.draft && last < a.nodes - 1;
    const Left f{tops[last].max, subtract ? tops[a.nodes + last].max : 0.0f, sums[last], subtract ? sums[a.nodes + last] : 0.0, subtract, refused_s, refused};
    target += last * a.target_stride;
    if (subtract) draft += last * a.draft_stride;
    // what is left in each slice: sixteen wavefronts, four tokens of 4096 per thread, side by side
    for (int s = wave; s < a.slices; s += kWaves) {
        double sum = 0.0;
        for (int e = 0; e < kSlice / 64; ++e) {
            const int64_t t = (int64_t)s * kSlice + e * 64 + lane;
            if (t < a.vocab) sum += left_of(a, f, target, draft, t);
        }
        sum = wave_sum64(sum);
        if (lane == 0) a.left[s] = sum;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        double total = 0.0;
        for (int s = 0; s < a.slices; ++s) total += a.left[s];
        const double goal = (double)a.uniform[0] * total;
        double before = 0.0, found_before = 0.0;
        int found = -1;
        for (int s = 0; s < a.slices; ++s) {
            const double w = a.left[s];
            if (w > 0.0) {
                found = s;
                found_before = before;
                if (before + w > goal) break;
            }
            before += w;
        }
        slice_s = found;
        target_s = goal;
        before_s = found_before;
    }
    __syncthreads();
    if (slice_s < 0) {  // nothing is left
        if (threadIdx.x == 0) a.result[1] = tops[last].arg;
        return;
    }
    // the token: the first one of the slice where the sum passes the goal, or the slice's last one with a weight
    if (wave == 0) {
        const double goal = target_s;
        double before = before_s;
        int token = -1;
        for (int e = 0; e < kSlice / 64; ++e) {
            const int64_t t = (int64_t)slice_s * kSlice + e * 64 + lane;
            const double w = t < a.vocab ? left_of(a, f, target, draft, t) : 0.0;
            const double upto = before + wave_before(w, lane) + w;
            const uint64_t positive = __ballot(w > 0.0), passed = __ballot(w > 0.0 && upto > goal);
            if (passed) {
                token = slice_s * kSlice + e * 64 + __ffsll((unsigned long long)passed) - 1;
                break;
            }
            if (positive) token = slice_s * kSlice + e * 64 + 63 - __clzll(positive);
            before = __shfl(upto, 63);
        }
        if (lane == 0) a.result[1] = token;
    }
}

}  // namespace

size_t verify_tree_workspace_bytes(int32_t node_num, int32_t vocab) {
    const size_t slices = ((size_t)vocab + kSlice - 1) / kSlice;
    return slices * (2 * (size_t)node_num * sizeof(Part) + sizeof(double));
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
    const double c = args.temperature > 0.0f ? 1.4426950408889634 / (double)args.temperature : 0.0;
    a.c_hi = (float)c;
    a.c_lo = (float)(c - (double)a.c_hi);
    const dim3 grid(a.slices, a.draft ? 2 * a.nodes - 1 : a.nodes);
    const hipStream_t stream = static_cast<hipStream_t>(args.stream);
    if (args.logits_type == LLMI_LOGITS_F32) {
        hipLaunchKernelGGL((verify_stats_kernel<float>), grid, dim3(kStatThreads), 0, stream, a);
        hipLaunchKernelGGL((verify_walk_kernel<float>), dim3(1), dim3(kWalkThreads), 0, stream, a);
    } else {
        hipLaunchKernelGGL((verify_stats_kernel<uint16_t>), grid, dim3(kStatThreads), 0, stream, a);
        hipLaunchKernelGGL((verify_walk_kernel<uint16_t>), dim3(1), dim3(kWalkThreads), 0, stream, a);
    }
    return check_launch();
}

}  // namespace llmi
