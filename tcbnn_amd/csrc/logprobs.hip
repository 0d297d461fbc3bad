// Log probabilities of given classes with entropy, rank and the best alternatives, and their gradient
// (tcbnn_logprobs_forward / _backward).
//
//   m = max x,  s = sum exp(x - m),  logsumexp = m + log s,  entropy = log s - (sum (x - m) exp(x - m)) / s
//   dx_j = g_logprob ([j = t] - p_j) - g_entropy p_j (log p_j + entropy)
//
// Bound by memory, the forward pass nearly as much by instructions (an exponential, a maximum and a comparison a logit): every logit is
// read once.  2048 x 131072 bf16 with 8 best classes takes 121 us (537 MB, 4.4 TB/s), the gradient of 4095 x 32003 bf16 101 us
// (524 MB, 5.2 TB/s).  One row takes what its launches and the order of steps on a compute unit take: 4.3 us for 1000
// classes, 7.6 for 32000, 11 in two launches for 131072.
#include "head.h"

namespace tcbnn {
namespace {

using namespace head;

constexpr int kMaxTop = 64;
constexpr float kNear = 65536.0f;  // |m| up to which sums of exp(x - m) are taken about m log2 e, rounded
constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.69314718055994531f;

// The order of classes as one number: larger logits first (NaN before all, -0 with +0), lower indices first among equals.
// Larger keys come first; 0 is below every class's key.
__device__ __forceinline__ uint32_t ordered(float x) {
    if (x != x) return 0xffffffffu;
    const uint32_t u = __float_as_uint(x + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ uint64_t key_of(float x, int j) { return ((uint64_t)ordered(x) << 32) | (uint32_t)~j; }
__device__ __forceinline__ int class_of(uint64_t key) { return (int)~(uint32_t)key; }
__device__ __forceinline__ uint64_t next_key(uint64_t key) { return key == 0 ? 0 : key - 1; }  // the largest that comes behind it
__device__ __forceinline__ float logit_of(uint64_t key) {
    const uint32_t u = (uint32_t)(key >> 32);
    return u == 0xffffffffu ? NAN : __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ uint64_t lane_key(uint64_t v, int lane) {
    return ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32) | (uint32_t)__builtin_amdgcn_readlane((int)v, lane);
}
__device__ __forceinline__ uint64_t wave_max_key(uint64_t v) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v = max(v, (uint64_t)__shfl_xor((unsigned long long)v, d));
    return v;
}
__device__ __forceinline__ int wave_sum_int(int v) { return (int)wave_reduce((uint32_t)v, [](uint32_t a, uint32_t b) { return a + b; }); }

// 16 bytes of logits as they lie in memory (as words: the compiler keeps elements that come out of a branch in a register each).
typedef int Words __attribute__((ext_vector_type(4)));
template <typename T>
__device__ __forceinline__ Words load_words(const T* x) {
    return __builtin_bit_cast(Words, load_vec(x));
}
// n < V logits, -inf in the place of the others
template <typename T>
__device__ __forceinline__ Words load_rest(const T* x, int n) {
    Vec<T> v;
#pragma unroll
    for (int e = 0; e < Elem<T>::kVec; ++e) v[e] = e < n ? x[e] : (T)-INFINITY;
    return __builtin_bit_cast(Words, v);
}
// `kR` vectors of the n logits at x, the r-th one at (r * lanes + lane) V; -inf past the end.  Where the logits end within a
// vector, all lanes read that one, and the lane that it belongs to takes it.
template <typename T, int kR>
__device__ __forceinline__ void load_slices(const T* x, int n, int lane, int lanes, Words (&raw)[kR]) {
    constexpr int V = Elem<T>::kVec;
    const Words none = load_rest(x, 0);
#pragma unroll
    for (int r = 0; r < kR; ++r) {
        const int j = (r * lanes + lane) * V;
        raw[r] = none;
        if ((r + 1) * lanes * V <= n || j + V <= n) raw[r] = load_words(x + j);
    }
    if (n % V != 0) {
        const int last = n / V;
        const Words rest = load_rest(x + last * V, n % V);
#pragma unroll
        for (int r = 0; r < kR; ++r)
            if (r * lanes + lane == last) raw[r] = rest;
    }
}
template <typename T>
__device__ __forceinline__ float value(const Words& w, int e) {
    if constexpr (std::is_same_v<T, __bf16>)  // (of a conversion the compiler makes maxima in bf16, which take four instructions)
        return __uint_as_float(e & 1 ? (uint32_t)w[e / 2] & 0xffff0000u : (uint32_t)w[e / 2] << 16);
    else
        return (float)__builtin_bit_cast(Vec<T>, w)[e];
}

// What is known of a set of logits: the largest, sums of exp(x - m) and of (x - m) exp(x - m), how many go before the given
// class.  A NaN or infinite logit leaves s NaN; no allowed class leaves m = -inf and s = 0.
struct Part {
    float m, s, sx;
    int before;
};
__device__ __forceinline__ void rescale(Part& p, float m) {
    const float d = p.m - m, f = p.m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(d * kLog2e);
    p.sx = f == 0.0f ? p.s * 0.0f : __builtin_fmaf(d, p.s, p.sx) * f;  // (keeps a NaN)
    p.s *= f;
    p.m = m;
}
struct Answer {
    float m, logsum, logsumexp, entropy;
    bool none;  // no allowed class
    __device__ __forceinline__ explicit Answer(const Part& p) {
        none = p.m == -INFINITY && p.s == 0.0f;
        m = p.m;
        logsum = logf(p.s);
        logsumexp = none ? -INFINITY : m + logsum;
        entropy = none ? 0.0f : logsum - p.sx / p.s;
    }
    __device__ __forceinline__ float log_prob(float x) const { return none ? -INFINITY : (x - m) - logsum; }
};

struct LogProbsParams {
    const int32_t* targets;
    float *logprob, *entropy, *logsumexp, *top_logprob;
    int32_t *rank, *top_index;
    int rows, classes, top, chunks;
    long long ld;
    // rows in several chunks: a Part and `top` keys of each, best first
    Part* parts;    // [rows][chunks]
    uint64_t* keys; // [rows][top][chunks]: what comes first in its chunk is side by side, and so spread over the lanes that join them
};

__device__ __forceinline__ void write_row(const LogProbsParams& p, long long row, const Part& part, const Answer& a, bool given, float xt) {
    const int t = p.targets ? p.targets[row] : -1;
    if (p.logprob) p.logprob[row] = given ? a.log_prob(xt) : (t < 0 ? 0.0f : NAN);
    if (p.entropy) p.entropy[row] = a.entropy;
    if (p.logsumexp) p.logsumexp[row] = a.logsumexp;
    if (p.rank) p.rank[row] = given ? part.before : -1;
}
__device__ __forceinline__ void write_top(const LogProbsParams& p, long long row, const Answer& a, int place, uint64_t key) {
    if (p.top_index) p.top_index[row * p.top + place] = class_of(key);
    if (p.top_logprob) p.top_logprob[row * p.top + place] = a.log_prob(logit_of(key));
}

// A chunk of a row (the whole row, if it fits) belongs to a team of W wavefronts and stays in their registers, R vectors of 16
// bytes a lane, while it is looked at: for its largest logit, for the sums, for what goes before the given class, for the best
// classes.  Every lane number is a group of logits, and the k-th largest of the 64 groups' maxima bounds the k-th largest
// logit from below: what reaches the bound (little more than k, for logits in any usual order) is gathered in LDS and ordered
// by counting.  Many equal logits or a cluster in one group can be too much for the list: then the ones above the bound are
// taken with the first of those equal to it, and if that is too much still, or the chunk holds a NaN, the best classes are
// found one after the other.
constexpr int kList = 256;
constexpr int team_threads(int w) { return w == 1 ? 256 : 64 * w; }

template <int W>
__device__ __forceinline__ void team_sync() {
    if constexpr (W == 1) {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    } else {
        __syncthreads();
    }
}

template <int W>
struct TeamLds {
    uint64_t list[kList];
    uint64_t best[W];
    Part part[W];
    float lane_max[W][64];
    int count, waves[W];
};

template <typename T, int W, int R, bool SPLIT>
__global__ __launch_bounds__(team_threads(W)) void logprobs_kernel(const T* __restrict__ x, const LogProbsParams p) {
    constexpr int V = Elem<T>::kVec, kTeam = 64 * W, kTeams = team_threads(W) / kTeam, kStep = kTeam * V, kChunk = R * kStep;
    __shared__ TeamLds<W> lds_all[kTeams];
    const int lane = threadIdx.x & 63, tid = threadIdx.x % kTeam, wave = tid >> 6, team = threadIdx.x / kTeam;
    TeamLds<W>& lds = lds_all[team];
    const long long unit = (long long)blockIdx.x * kTeams + team;
    const long long row = SPLIT ? unit / p.chunks : unit;
    const int chunk = SPLIT ? (int)(unit - row * p.chunks) : 0;
    if (row >= p.rows) return;  // (a team alone in its workgroup always has a row)
    const int base = chunk * kChunk, n = min(kChunk, p.classes - base), top = p.top;
    x += row * p.ld + base;

    Words raw[R];
    // Short rows are dealt to the lanes one by one: in vectors, most lanes would have none, and the groups' maxima bound little.
    constexpr bool kDealt = W == 1 && R == 1;
    if constexpr (kDealt) {
        Vec<T> v;
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = e * 64 + tid < n ? x[e * 64 + tid] : (T)-INFINITY;
        raw[0] = __builtin_bit_cast(Words, v);
    } else {
        load_slices<T, R>(x, n, tid, kTeam, raw);
    }
    const int target = p.targets ? p.targets[row] : -1;
    const bool given = target >= 0 && target < p.classes;
    const int t = target - base;  // within the chunk, before it or behind it
    const float xt = given ? (float)x[t] + 0.0f : 0.0f;  // (+0 for -0: the sign of +0 - +0 and of +0 - -0 is clear)
    if (tid == 0) lds.count = 0;

    // ---- the largest logit of each vector, of the lane, of the wavefront
    float vec_max[R], lane_max = -INFINITY;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        vec_max[r] = value<T>(raw[r], 0);
#pragma unroll
        for (int e = 1; e < V; ++e) vec_max[r] = fmaxf(vec_max[r], value<T>(raw[r], e));
        lane_max = fmaxf(lane_max, vec_max[r]);
    }
    Part part = {wave_max(lane_max), 0.0f, 0.0f, 0};
    // ---- sums about it, and what goes before the given class.
    // exp(x - m) = 2^u, u = x log2 e - c with c = m log2 e rounded: one fused multiply-add, but about c: every term is
    // 2^off too large and every u off, where `off` is what c was rounded by (known exactly; 2^-8 at most up to kNear, as exact then as
    // differences of x and m).  u is held above -250, where 2^u is 0 anyway: 0 times -inf is NaN.
    // Before the class go larger logits and equal ones of lower index: whole vectors below it compare with the next lower
    // number, the equal ones in the class's own vector are counted afterwards.
    const float m = part.m == -INFINITY ? 0.0f : part.m, c = m * kLog2e, off = __builtin_fmaf(m, kLog2e, -c);
    uint32_t lower = ordered(xt) - 1;
    if (lower == 0x7fffffffu) --lower;  // (no class has the key of -0)
    const float below = logit_of((uint64_t)lower << 32);
    uint32_t signs = 0;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        float bound = r * kStep + tid * V + V <= t ? below : xt;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float v = value<T>(raw[r], e);
            const float u = __builtin_fmaf(v, kLog2e, -c);
            const float ex = __builtin_amdgcn_exp2f(u);
            part.s += ex;
            part.sx = __builtin_fmaf(ex, fmaxf(u, -250.0f), part.sx);
            if constexpr (kDealt) bound = e * 64 + tid < t ? below : xt;
            // the sign of bound - v, shifted in from below (comparisons write a scalar, which the addition then waits for)
            signs = __builtin_amdgcn_alignbit(signs, __float_as_uint(bound - v), 31);
        }
        if ((r + 1) * V % 32 == 0 || r == R - 1) part.before += __popc(signs);
        // Vector after vector, the values as fp32 made anew: all at once, as the compiler likes it, takes twice the registers.
        asm volatile("" : "+v"(part.s), "+v"(part.sx), "+v"(signs));
        if (r + 1 < R) asm volatile("" : "+v"(raw[r + 1]));
        __builtin_amdgcn_sched_barrier(0);
    }
    // Far from zero the row once more (from the cache), every logit's difference to m first, which is exact beside m: 2048 x 131072 fp32 about
    // 1e5 300 us, about 0 200.
    if (fabsf(m) > kNear) {
        part.s = part.sx = 0.0f;
#pragma unroll 1
        for (int j = tid * V; j < n; j += kStep) {
            const Words w = j + V <= n ? load_words(x + j) : load_rest(x + j, n - j);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float d = value<T>(w, e) - m, ex = __builtin_amdgcn_exp2f(d * kLog2e);
                part.s += ex;
                part.sx = __builtin_fmaf(ex, fmaxf(d, -200.0f), part.sx);
            }
        }
    } else {
        const float back = __builtin_amdgcn_exp2f(-off);
        part.sx = __builtin_fmaf(-off, part.s, part.sx) * (back * kLn2);
        part.s *= back;
    }
    if (!kDealt && wave == 0 && t >= 0 && t < n && lane < t % V) part.before += (float)x[t - 1 - lane] == xt;
    part.before = wave_sum_int(part.before);
    part.s = wave_sum(part.s);
    part.sx = wave_sum(part.sx);
    if (W > 1 || top > 0) {
        if (lane == 0) lds.part[wave] = part;
        lds.lane_max[wave][lane] = lane_max;
        team_sync<W>();
    }
    if constexpr (W > 1) {
        float most = lds.part[0].m;
#pragma unroll
        for (int w = 1; w < W; ++w) most = fmaxf(most, lds.part[w].m);
        part = {most, 0.0f, 0.0f, 0};
#pragma unroll
        for (int w = 0; w < W; ++w) {
            Part q = lds.part[w];
            rescale(q, most);
            part.s += q.s;
            part.sx += q.sx;
            part.before += q.before;
        }
    }
    const bool odd = part.s != part.s;  // a NaN, or infinity
    if (given && (odd || !(below > -INFINITY))) {  // what differences of floats do not order
        int before = 0;
        const uint64_t kt = key_of(xt, target);
#pragma unroll 1
        for (int j = tid; j < n; j += kTeam) before += key_of((float)x[j], base + j) > kt;
        before = wave_sum_int(before);
        team_sync<W>();
        lds.waves[wave] = before;
        team_sync<W>();
        part.before = 0;
#pragma unroll
        for (int w = 0; w < W; ++w) part.before += lds.waves[w];
    }
    const Answer answer(part);
    if (tid == 0) {
        if constexpr (SPLIT)
            p.parts[unit] = part;
        else
            write_row(p, row, part, answer, given, xt);
    }
    if (top == 0) return;
    auto emit = [&](int place, uint64_t key) {  // (keys within the chunk count their classes from its first)
        if constexpr (SPLIT)
            p.keys[(row * top + place) * p.chunks + chunk] = key == 0 ? 0 : key_of(logit_of(key), class_of(key) + base);
        else
            write_top(p, row, answer, place, key);
    };

    // ---- the best classes
    int count = kList + 1;
    if (!odd) {
        float group = lds.lane_max[0][lane];
#pragma unroll
        for (int w = 1; w < W; ++w) group = fmaxf(group, lds.lane_max[w][lane]);
        int larger = 0;
#pragma unroll
        for (int l = 0; l < 64; ++l) larger += __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(group), l)) > group;
        const float bound = -wave_max(larger < top ? -group : -INFINITY);
        auto push = [&](int j, float v) {
            const int at = atomicAdd(&lds.count, 1);
            if (at < kList) lds.list[at] = key_of(v, j);
        };
        if constexpr (kDealt) {
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (value<T>(raw[0], e) >= bound && e * 64 + tid < n) push(e * 64 + tid, value<T>(raw[0], e));
        } else {
            uint32_t hot = 0;  // the vectors that reach the bound: few, and read again (from the cache)
#pragma unroll
            for (int r = 0; r < R; ++r) hot |= vec_max[r] >= bound ? 1u << r : 0u;
            while (hot != 0) {
                const int j = __builtin_ctz(hot) * kStep + tid * V;
                hot &= hot - 1;
                const Words w = j + V <= n ? load_words(x + j) : load_rest(x + j, n - j);
#pragma unroll
                for (int e = 0; e < V; ++e)
                    if (value<T>(w, e) >= bound && j + e < n) push(j + e, value<T>(w, e));
            }
        }
        team_sync<W>();
        count = lds.count;
        if (count > kList) {
            team_sync<W>();
            if (tid == 0) lds.count = 0;
            team_sync<W>();
#pragma unroll 1
            for (int j = tid; j < n; j += kTeam)
                if ((float)x[j] > bound) push(j, (float)x[j]);
            team_sync<W>();
            count = lds.count;
            if (count <= kList - kMaxTop) {
                // ... and the first `top` of those equal to the bound: 64 W in a row at a time
                int found = 0;
#pragma unroll 1
                for (int first = 0; first < n && found < top; first += kTeam) {
                    const int j = first + tid;
                    const bool equal = j < n && (float)x[j] == bound;
                    const uint64_t mask = __builtin_amdgcn_ballot_w64(equal);
                    team_sync<W>();
                    if (lane == 0) lds.waves[wave] = __popcll(mask);
                    team_sync<W>();
                    int place = found + __popcll(mask & ((1ull << lane) - 1));
#pragma unroll
                    for (int w = 0; w < W; ++w) {
                        if (w < wave) place += lds.waves[w];
                        found += lds.waves[w];
                    }
                    if (equal && place < top) lds.list[count + place] = key_of(bound, j);
                }
                count += min(found, top);
                team_sync<W>();
            }
        }
    }
    if (count <= kList) {
        for (int i = tid; i < count; i += kTeam) {
            const uint64_t key = lds.list[i];
            int place = 0;
#pragma unroll 8
            for (int k = 0; k < count; ++k) place += lds.list[k] > key;
            if (place < top) emit(place, key);
        }
        if constexpr (SPLIT)
            for (int i = count + tid; i < top; i += kTeam) emit(i, 0);
        return;
    }
    uint64_t most = ~0ull;  // (a NaN in class 0 has that key)
#pragma unroll 1
    for (int i = 0; i < top; ++i) {
        uint64_t best = 0;
#pragma unroll 1
        for (int j = tid; j < n; j += kTeam) {
            const uint64_t key = key_of((float)x[j], j);
            if (key <= most) best = max(best, key);
        }
        best = wave_max_key(best);
        if constexpr (W > 1) {
            team_sync<W>();
            lds.best[wave] = best;
            team_sync<W>();
#pragma unroll
            for (int w = 0; w < W; ++w) best = max(best, lds.best[w]);
        }
        if (tid == 0) emit(i, best);
        most = next_key(best);
    }
}

// Rows in several chunks: a wavefront a row.  The same way to the best keys: the k-th largest of the lanes' largest bounds them.
constexpr int kJoinRows = 4;
template <typename T>
__global__ __launch_bounds__(64 * kJoinRows) void logprobs_join_kernel(const T* __restrict__ x, const LogProbsParams p) {
    __shared__ uint64_t lists[kJoinRows][kList];
    __shared__ int counts[kJoinRows];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long long row = (long long)blockIdx.x * kJoinRows + wave;
    if (row >= p.rows) return;
    const uint64_t* keys = p.keys + row * p.chunks * p.top;
    const int total = p.chunks * p.top;
    // the first keys are requested together and kept (all of them, in most calls), the others read as they are needed
    constexpr int kKept = 8;
    uint64_t kept[kKept], best = 0;
#pragma unroll
    for (int u = 0; u < kKept; ++u) kept[u] = lane + 64 * u < total ? keys[lane + 64 * u] : 0;
    auto each_key = [&](auto f) {
#pragma unroll
        for (int u = 0; u < kKept; ++u) f(kept[u]);
#pragma unroll 4
        for (int i = lane + 64 * kKept; i < total; i += 64) f(keys[i]);
    };
    each_key([&](uint64_t key) { best = max(best, key); });
    Part part = {-INFINITY, 0.0f, 0.0f, 0};
    for (int c = lane; c < p.chunks; c += 64) {
        Part q = p.parts[row * p.chunks + c];
        const float m = fmaxf(part.m, q.m);
        rescale(part, m);
        rescale(q, m);
        part.s += q.s;
        part.sx += q.sx;
        part.before += q.before;
    }
    rescale(part, wave_max(part.m));
    part.s = wave_sum(part.s);
    part.sx = wave_sum(part.sx);
    part.before = wave_sum_int(part.before);
    const Answer answer(part);
    if (lane == 0) {
        const int t = p.targets ? p.targets[row] : -1;
        const bool given = t >= 0 && t < p.classes;
        write_row(p, row, part, answer, given, given ? (float)x[row * p.ld + t] : 0.0f);
        counts[wave] = 0;
    }
    if (p.top == 0) return;
    int larger = 0;
#pragma unroll
    for (int l = 0; l < 64; ++l) larger += lane_key(best, l) > best;
    // (keys differ, but for those that stand for nothing: 0)
    const uint64_t bound = max((uint64_t)1, ~wave_max_key(larger < p.top ? ~best : 0));
    team_sync<1>();
    each_key([&](uint64_t key) {
        if (key >= bound) {
            const int at = atomicAdd(&counts[wave], 1);
            if (at < kList) lists[wave][at] = key;
        }
    });
    team_sync<1>();
    const int count = counts[wave];
    if (count <= kList) {
        for (int i = lane; i < count; i += 64) {
            const uint64_t key = lists[wave][i];
            int place = 0;
#pragma unroll 8
            for (int k = 0; k < count; ++k) place += lists[wave][k] > key;
            if (place < p.top) write_top(p, row, answer, place, key);
        }
        return;
    }
    uint64_t most = ~0ull;
    for (int i = 0; i < p.top; ++i) {
        best = 0;
        each_key([&](uint64_t key) {
            if (key <= most) best = max(best, key);
        });
        best = wave_max_key(best);
        if (lane == 0) write_top(p, row, answer, i, best);
        most = next_key(best);
    }
}

// How a row is shared: whole rows while a team's registers hold them, longer ones in chunks, small ones where there are too few
// of the large ones to fill the chip.  Measured (us): 2048 x 131072 bf16 in chunks of 16 / 8 / 4 vectors a lane 119 / 132 / 167, 1 x 131072
// 13.0 / 11.8 / 11.2; 64 x 32000 whole 8.2, in four chunks and a join 11.1; 8192 x 1000 fp32 with a wavefront a row 15.0, with
// four 32.9.
struct Shape {
    int w, r, chunks;
};
inline Shape shape_of(long long rows, int classes, int per_vector) {
    const int vectors = (classes + per_vector - 1) / per_vector;
    auto chunks = [&](int r) { return (vectors + 256 * r - 1) / (256 * r); };
    if (vectors <= 64) return {1, 1, 1};
    if (vectors <= 128) return {1, 2, 1};
    if (vectors <= 256) return {1, 4, 1};
    if (vectors <= 1024) return {4, 4, 1};
    if (vectors <= 2048) return {4, 8, 1};
    if (vectors > 4096 && rows * chunks(16) < 2 * kComputeUnits) return {4, 4, chunks(4)};
    return {4, 16, chunks(16)};
}
template <typename F>
void by_shape(const Shape& s, F&& f) {
    using std::integral_constant;
    if (s.w == 1 && s.r == 1) return f(integral_constant<int, 1>(), integral_constant<int, 1>());
    if (s.w == 1 && s.r == 2) return f(integral_constant<int, 1>(), integral_constant<int, 2>());
    if (s.w == 1) return f(integral_constant<int, 1>(), integral_constant<int, 4>());
    if (s.r == 4) return f(integral_constant<int, 4>(), integral_constant<int, 4>());
    if (s.r == 8) return f(integral_constant<int, 4>(), integral_constant<int, 8>());
    return f(integral_constant<int, 4>(), integral_constant<int, 16>());
}

// ---- gradient.  Bound by memory: a workgroup a piece of a row, four vectors of 16 bytes a thread, all requested first.
constexpr int kGradThreads = 256, kGradVectors = 4;

template <typename T>
__global__ __launch_bounds__(kGradThreads) void logprobs_grad_kernel(const T* x, const int32_t* __restrict__ targets,
                                                                     const float* __restrict__ logsumexp,
                                                                     const float* __restrict__ entropy,
                                                                     const float* __restrict__ g_logprob,
                                                                     const float* __restrict__ g_entropy, T* dx, int n, int pieces,
                                                                     long long x_ld, long long dx_ld) {
    constexpr int V = Elem<T>::kVec, kStep = kGradThreads * V, kPiece = kGradVectors * kStep;
    const long long row = blockIdx.x / (unsigned)pieces;
    const int base = (int)(blockIdx.x - (unsigned)row * pieces) * kPiece, left = n - base;
    x += row * x_ld + base;
    dx += row * dx_ld + base;
    Words raw[kGradVectors];
    load_slices<T, kGradVectors>(x, min(left, kPiece), threadIdx.x, kGradThreads, raw);
    const float lse = logsumexp[row];
    const int target = g_logprob ? targets[row] : -1, t = target - base;
    const float g = target >= n ? NAN : (target >= 0 ? g_logprob[row] : 0.0f);
    const float ge = g_entropy ? g_entropy[row] : 0.0f, h = g_entropy ? entropy[row] : 0.0f;
    const bool none = lse == -INFINITY;  // no allowed class: no distribution, no gradient
    // -p (g + ge (log p + h)), and g for the given class.  log p is held above -200, where p is 0 anyway.
    const float c0 = none ? (g != g ? g : 0.0f) : __builtin_fmaf(ge, h, g), c1 = none ? 0.0f : ge, shift = none ? 0.0f : lse;
#pragma unroll
    for (int r = 0; r < kGradVectors; ++r) {
        const int j = r * kStep + threadIdx.x * V;
        if (j >= left) break;
        float out[V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float lp = value<T>(raw[r], e) - shift;
            const float prob = __builtin_amdgcn_exp2f(lp * kLog2e);
            out[e] = -prob * __builtin_fmaf(c1, fmaxf(lp, -200.0f), c0);
        }
        if (j <= t && t < j + V) {
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (j + e == t && !none) out[e] += g;
        }
        if (j + V <= left) {
            Vec<T> v;
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] = (T)out[e];
            store_vec(dx + j, v);
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (j + e < left) dx[j + e] = (T)out[e];
        }
    }
}

}  // namespace
}  // namespace tcbnn

using namespace tcbnn;
using namespace tcbnn::head;

extern "C" size_t tcbnn_logprobs_workspace_bytes(int rows, int classes, int top, int dtype) {
    if (rows <= 0 || classes <= 0 || top < 0 || top > kMaxTop || !dtype_known(dtype)) return 0;
    const Shape s = shape_of(rows, classes, (int)(16 / dtype_bytes(dtype)));
    return s.chunks == 1 ? 0 : (size_t)rows * s.chunks * (sizeof(Part) + top * sizeof(uint64_t));
}

extern "C" int tcbnn_logprobs_forward(const tcbnn_logprobs_desc* d, void* stream) {
    TCBNN_NOTNULL(d);
    TCBNN_REQUIRE(dtype_known(d->dtype), "logprobs: unknown dtype");
    TCBNN_REQUIRE(d->rows >= 0 && d->classes > 0, "logprobs: bad shape");
    TCBNN_REQUIRE(d->top >= 0 && d->top <= kMaxTop && d->top <= d->classes, "logprobs: top is at most %d and the number of classes", kMaxTop);
    const long long ld = row_stride(d->logits_ld, d->classes);
    TCBNN_REQUIRE(ld > 0, "logprobs: rows overlap");
    if (d->rows == 0) return TCBNN_OK;
    TCBNN_NOTNULL(d->logits);
    if (d->logprob || d->rank) TCBNN_NOTNULL(d->targets);
    const int top = d->top_index || d->top_logprob ? d->top : 0;
    const Shape shape = shape_of(d->rows, d->classes, (int)(16 / dtype_bytes(d->dtype)));
    const long long units = (long long)d->rows * shape.chunks;
    Part* parts = nullptr;
    uint64_t* keys = nullptr;
    if (shape.chunks > 1) {
        TCBNN_NOTNULL(d->workspace);
        TCBNN_REQUIRE(d->workspace_bytes >= tcbnn_logprobs_workspace_bytes(d->rows, d->classes, top, d->dtype), "logprobs: workspace too small");
        TCBNN_REQUIRE((uintptr_t)d->workspace % 16 == 0, "logprobs: the workspace is not aligned to 16 bytes");
        parts = (Part*)d->workspace;
        keys = (uint64_t*)(parts + units);
    }
    by_dtype(d->dtype, [&](auto e) {
        using T = decltype(e);
        by_shape(shape, [&](auto w, auto r) {
            constexpr int W = w.value, R = r.value, kTeams = team_threads(W) / (64 * W);
            const long long at_once = kMaxThreads / team_threads(W) * kTeams / shape.chunks;
            for (long long row = 0; row < d->rows; row += at_once) {
                auto from = [&](auto* q, long long each) { return q ? q + row * each : q; };
                const int rows = (int)std::min(at_once, d->rows - row);
                const LogProbsParams p = {from(d->targets, 1), from(d->logprob, 1), from(d->entropy, 1), from(d->logsumexp, 1), from(d->top_logprob, top),
                                          from(d->rank, 1), from(d->top_index, top), rows, d->classes, top, shape.chunks, ld, from(parts, shape.chunks),
                                          from(keys, (long long)shape.chunks * top)};
                const T* x = (const T*)d->logits + row * ld;
                const dim3 grid((unsigned)(((long long)rows * shape.chunks + kTeams - 1) / kTeams));
                if constexpr (W > 1)
                    if (shape.chunks > 1) {
                        hipLaunchKernelGGL(HIP_KERNEL_NAME(logprobs_kernel<T, W, R, true>), grid, dim3(team_threads(W)), 0, (hipStream_t)stream, x, p);
                        hipLaunchKernelGGL(logprobs_join_kernel<T>, dim3((unsigned)((rows + kJoinRows - 1) / kJoinRows)), dim3(64 * kJoinRows), 0,
                                           (hipStream_t)stream, x, p);
                        continue;
                    }
                hipLaunchKernelGGL(HIP_KERNEL_NAME(logprobs_kernel<T, W, R, false>), grid, dim3(team_threads(W)), 0, (hipStream_t)stream, x, p);
            }
        });
    });
    TCBNN_LAUNCH_CHECK("logprobs_kernel");
    return TCBNN_OK;
}

extern "C" int tcbnn_logprobs_backward(const tcbnn_logprobs_grad_desc* d, void* stream) {
    TCBNN_NOTNULL(d);
    TCBNN_REQUIRE(dtype_known(d->dtype), "logprobs: unknown dtype");
    TCBNN_REQUIRE(d->rows >= 0 && d->classes > 0, "logprobs: bad shape");
    const long long x_ld = row_stride(d->logits_ld, d->classes), dx_ld = row_stride(d->grad_logits_ld, d->classes);
    TCBNN_REQUIRE(x_ld > 0 && dx_ld > 0, "logprobs: rows overlap");
    if (d->rows == 0) return TCBNN_OK;
    TCBNN_NOTNULL(d->logits);
    TCBNN_NOTNULL(d->logsumexp);
    TCBNN_NOTNULL(d->grad_logits);
    if (d->grad_logprob) TCBNN_NOTNULL(d->targets);
    if (d->grad_entropy) TCBNN_NOTNULL(d->entropy);
    TCBNN_REQUIRE(d->grad_logits != d->logits || d->rows == 1 || x_ld == dx_ld, "logprobs: a gradient over the logits has their stride");
    const long long piece = kGradThreads * kGradVectors * (long long)(16 / dtype_bytes(d->dtype));
    const long long pieces = (d->classes + piece - 1) / piece;
    const long long at_once = kMaxThreads / kGradThreads / pieces;
    by_dtype(d->dtype, [&](auto t) {
        using T = decltype(t);
        for (long long row = 0; row < d->rows; row += at_once) {
            auto from = [&](auto* q) { return q ? q + row : q; };
            hipLaunchKernelGGL(logprobs_grad_kernel<T>, dim3((unsigned)(pieces * std::min(at_once, d->rows - row))), dim3(kGradThreads), 0, (hipStream_t)stream,
                               (const T*)d->logits + row * x_ld, from(d->targets), from(d->logsumexp), from(d->entropy), from(d->grad_logprob),
                               from(d->grad_entropy), (T*)d->grad_logits + row * dx_ld, d->classes, (int)pieces, x_ld, dx_ld);
        }
    });
    TCBNN_LAUNCH_CHECK("logprobs_grad_kernel");
    return TCBNN_OK;
}
