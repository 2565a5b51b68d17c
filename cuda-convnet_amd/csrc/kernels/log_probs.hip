// log_probs.hip -- log probabilities of given classes with entropy and top alternatives, and their gradient.
// With m the largest logit of a case, t_j = (x_j - m) log2 e, s = sum_j 2^t_j, w = sum_j t_j 2^t_j:
//   ln p_j = (x_j - m) - ln s,   -sum_j p_j ln p_j = ln 2 (log2 s - w / s),
// and (m, s, w) of two sets of classes join into those of their union, so a case may be split over workgroups.
#include <math.h>
#include <algorithm>
#include <type_traits>
#include "mc_types.h"

namespace mc {
namespace {

constexpr int LT = 256;             // threads of a workgroup
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int kMaxOut = 1 << 30;     // classes: their indices stay within an int wherever a tile ends
constexpr float kFar = 0x1p20f;     // a maximum so far from zero takes sums of its own: see far_from_zero

struct LogProbArgs {
    const void* logits;
    size_t classStride, caseStride;
    const void* labels;
    int labelType, numCases, numOut;
    float *labelLogProbs, *entropy, *maxAndLogSum;
    int* topClasses;
    float* topLogProbs;
    int numTop;
};

// What a workgroup leaves of its classes of a case for the joining kernel; its best numTop keys follow in an array of their own.
struct Part { float m, s, w, label; };   // label: its logit where this part has it, else -inf
struct Parts {
    Part* stats;                  // (numCases, parts)
    unsigned long long* keys;     // (numCases, parts, numTop), largest first, 0 = none
    int parts;
    int span;                     // classes of a part
};

// The class that a label's 32 bits name, or -1 for "no class".
__device__ __forceinline__ int label_from(unsigned bits, int labelType, int numOut) {
    const float f = __uint_as_float(bits);
    const int y = labelType == MC_I32 ? (int)bits : f >= 0.f && f < (float)numOut ? (int)f : -1;
    return y >= 0 && y < numOut ? y : -1;
}
__device__ __forceinline__ int label_of(const void* labels, int labelType, int n, int numOut) {
    return label_from(static_cast<const unsigned*>(labels)[n], labelType, numOut);
}

// op over the lanes of a wave whose numbers agree modulo G (1, 2, 4 or 8), in each of them.  Rotations within rows of 16 lanes and swaps
// of rows: a dozen cycles a step, where a shuffle through the LDS takes a hundred.
template <int CTRL>
__device__ __forceinline__ float rotated(float v) { return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true)); }
template <class OP>
__device__ __forceinline__ float over_lanes(float v, int G, OP op) {
    v = op(v, rotated<0x128>(v));               // by 8,
    if (G <= 4) v = op(v, rotated<0x124>(v));   // by 4, ...
    if (G <= 2) v = op(v, rotated<0x122>(v));
    if (G <= 1) v = op(v, rotated<0x121>(v));
    const auto rows = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = op(__uint_as_float(rows[0]), __uint_as_float(rows[1]));
    const auto halves = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return op(__uint_as_float(halves[0]), __uint_as_float(halves[1]));
}
struct Larger { __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); } };
struct Sum { __device__ __forceinline__ float operator()(float a, float b) const { return a + b; } };

// ---------------------------------------------------------------- groups of threads that share a case
// A whole workgroup, or one wave of it (whose LDS accesses are in order: there only the compiler has to be held back).
template <int THREADS>
struct Group {
    static_assert(THREADS == LT || THREADS == 64, "");
    static constexpr int WAVES = THREADS / 64;
    __device__ static int index() { return THREADS == LT ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / THREADS); }
    __device__ static int tid() { return threadIdx.x & (THREADS - 1); }
    __device__ static void sync() {
        if (THREADS == LT) __syncthreads();
        else {
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
            __builtin_amdgcn_wave_barrier();
        }
    }
    __device__ static bool any(bool v) { return THREADS == LT ? __syncthreads_or(v) : __any(v); }
    // sh: WAVES floats of LDS that nobody else uses until the next sync
    __device__ static float max(float v, float* sh) {
        v = over_lanes(v, 1, Larger());
        if (WAVES == 1) return v;
        if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
        sync();
        v = sh[0];
#pragma unroll
        for (int i = 1; i < WAVES; ++i) v = fmaxf(v, sh[i]);
        return v;
    }
    __device__ static void sum2(float& a, float& b, float* sh) {
        a = over_lanes(a, 1, Sum());
        b = over_lanes(b, 1, Sum());
        if (WAVES == 1) return;
        if ((threadIdx.x & 63) == 0) {
            sh[threadIdx.x >> 6] = a;
            sh[WAVES + (threadIdx.x >> 6)] = b;
        }
        sync();
        a = sh[0];
        b = sh[WAVES];
#pragma unroll
        for (int i = 1; i < WAVES; ++i) {
            a += sh[i];
            b += sh[WAVES + i];
        }
    }
};

// ---------------------------------------------------------------- top alternatives
// Orders logits as the top alternatives are ordered: larger logit first, then lower class.  0 = never chosen (-inf, NaN).
__device__ __forceinline__ unsigned long long top_key(float x, unsigned j) {
    if (!(x > -INFINITY)) return 0;
    const unsigned b = __float_as_uint(x + 0.f);   // -0 and 0 are equal
    const unsigned o = b & 0x80000000u ? ~b : b | 0x80000000u;
    return (unsigned long long)o << 32 | (0xffffffffu - j);
}
__device__ __forceinline__ float key_logit(unsigned long long key) {
    const unsigned o = (unsigned)(key >> 32);
    return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ int key_class(unsigned long long key) { return (int)(0xffffffffu - (unsigned)key); }

constexpr int kCand = 256;   // candidates a group's list holds

// The sum of v over `lanes` neighbouring lanes (a power of two), in each of them.
__device__ __forceinline__ int sum_lanes(int v, int lanes) {
    v += lanes > 1 ? __builtin_amdgcn_mov_dpp(v, 0xB1, 0xf, 0xf, false) : 0;    // neighbours in pairs,
    v += lanes > 2 ? __builtin_amdgcn_mov_dpp(v, 0x4E, 0xf, 0xf, false) : 0;    // pairs in fours,
    v += lanes > 4 ? __builtin_amdgcn_mov_dpp(v, 0x141, 0xf, 0xf, false) : 0;   // fours in eights (mirrored: all four hold the sum),
    v += lanes > 8 ? __builtin_amdgcn_mov_dpp(v, 0x140, 0xf, 0xf, false) : 0;   // eights in sixteens
    if (lanes > 16) v += __shfl_xor(v, 16, 64);
    if (lanes > 32) v += __shfl_xor(v, 32, 64);
    return v;
}
// A value that at least k of a group's maxima (v, Q in each of `lanes` neighbouring lanes, the largest of them hi) reach and few more do:
// at least k classes reach it then, so no class below it is among the best k.  First down from hi in growing steps, then by bisection.
// Where ties or the step limits stop it early the value is lower than it could be, never too high.  (Lanes of other groups may be
// done earlier or later: nothing here reaches beyond a group.)
template <int Q>
__device__ __forceinline__ float top_threshold(const float (&v)[Q], int k, float hi, int lanes) {
    const auto reach = [&](float y) {
        int count = 0;
        if (lanes == 64) {   // the scalar unit counts
#pragma unroll
            for (int q = 0; q < Q; ++q) count += __popcll(__ballot(v[q] >= y));
            return count;
        }
#pragma unroll
        for (int q = 0; q < Q; ++q) count += v[q] >= y;
        return sum_lanes(count, lanes);
    };
    if (!(hi > -INFINITY)) return -INFINITY;
    float lo = hi, above = hi, step = fmaxf(1.f, fabsf(hi) * 0x1p-18f);
    int reached = reach(lo);
    for (int it = 0; it < 24 && reached < k; ++it, step *= 4.f) {
        above = lo;
        lo = hi - step;
        reached = reach(lo);
    }
    if (reached < k) return -INFINITY;
    const int enough = k + k / 4 + 1;
    for (int it = 0; it < 24 && reached > enough; ++it) {
        const float mid = 0.5f * lo + 0.5f * above;
        const int count = reach(mid);
        if (count >= k) {
            lo = mid;
            reached = count;
        } else above = mid;
    }
    return lo;
}
// So many can all be candidates: ordering them costs less than finding a threshold.  (128 class-major cases: 10 classes 5.9 us so and 7.5 with
// a threshold, 32 classes 9.4 and 7.6.)
constexpr int kFewClasses = 16;

// The k largest keys of classes [from, to) in one walk over them in order: THREADS classes at a time against the k-th best so far;
// what beats it joins the list, which is ordered again by counting, for each key, the larger ones.  Any number of ties, any order; used
// where the candidate list overflows.  best: MC_MAX_TOP keys, fresh: THREADS keys of LDS.
template <int THREADS, class T>
__device__ void top_by_scan(const T* x, size_t stride, int from, int to, int k, unsigned long long* best, unsigned long long* fresh) {
    typedef Group<THREADS> G;
    const int tid = G::tid();
    if (tid < k) best[tid] = 0;
    G::sync();
    for (int base = from; base < to; base += THREADS) {
        const int j = base + tid;
        unsigned long long key = j < to ? top_key((float)x[(size_t)j * stride], j) : 0;
        if (key <= best[k - 1]) key = 0;
        if (!G::any(key != 0)) continue;
        fresh[tid] = key;
        const unsigned long long mine = tid < k ? best[tid] : 0;
        G::sync();
        int rank = 0, mineRank = 0;
#pragma unroll 4
        for (int i = 0; i < THREADS; ++i) {
            rank += fresh[i] > key;
            mineRank += fresh[i] > mine;
        }
        for (int i = 0; i < k; ++i) rank += best[i] > key;
        G::sync();
        if (mine && tid + mineRank < k) best[tid + mineRank] = mine;
        if (key && rank < k) best[rank] = key;
        G::sync();
    }
}

// Orders `count` keys by counting, for each, the larger ones, and gives (rank, key) to `put` for the first k; ranks from count on get
// key 0.  The keys are distinct, but for zeros where ZEROS says that there may be some.  A thread takes OWN keys at a time, so that what it
// reads of the others serves as many.
template <bool ZEROS, int OWN, class F>
__device__ __forceinline__ void rank_keys(const unsigned long long* keys, int count, int k, int tid, int threads, F put) {
    for (int i = tid; i < count; i += threads * OWN) {
        unsigned long long key[OWN];
        int rank[OWN];
#pragma unroll
        for (int j = 0; j < OWN; ++j) {
            key[j] = keys[min(i + j * threads, count - 1)];
            rank[j] = 0;
        }
#pragma unroll 8   // (several reads of the LDS under way: 1 x 131072 bf16 10.3 -> 9.6 us)
        for (int c = 0; c < count; ++c) {
            const unsigned long long other = keys[c];
#pragma unroll
            for (int j = 0; j < OWN; ++j) rank[j] += other > key[j] || (ZEROS && key[j] == 0 && c < i + j * threads && other == 0);
        }
#pragma unroll
        for (int j = 0; j < OWN; ++j)
            if (i + j * threads < count && rank[j] < k) put(rank[j], key[j]);
    }
    for (int r = count + tid; r < k; r += threads) put(r, 0);
}

// ---------------------------------------------------------------- a case's results
struct CaseStats { float m, logSum, log2Sum; };

// (m, s, w) of all classes -> the outputs of case n; labelLogit: the label's logit, if there is a label.
__device__ __forceinline__ CaseStats case_stats(float m, float s) {
    const bool empty = s == 0.f;   // every class is ruled out
    const float l2 = empty ? 0.f : log2f(s);
    return {s != s && m == -INFINITY ? s : m, l2 * kLn2, l2};
}
__device__ __forceinline__ float log_prob(float x, const CaseStats& c) { return x == -INFINITY && c.logSum == c.logSum ? x : (x - c.m) - c.logSum; }
__device__ __forceinline__ void write_case(const LogProbArgs& a, int n, const CaseStats& c, float s, float w, int label, float labelLogit) {
    if (a.maxAndLogSum) {
        a.maxAndLogSum[n] = c.m;
        a.maxAndLogSum[(size_t)a.numCases + n] = c.logSum;
    }
    if (a.entropy) a.entropy[n] = s == 0.f ? 0.f : kLn2 * (c.log2Sum - w / s);
    if (a.labelLogProbs) a.labelLogProbs[n] = label < 0 ? 0.f : log_prob(labelLogit, c);
}
__device__ __forceinline__ void write_top(const LogProbArgs& a, int n, int rank, unsigned long long key, const CaseStats& c) {
    a.topClasses[(size_t)rank * a.numCases + n] = key ? key_class(key) : -1;
    a.topLogProbs[(size_t)rank * a.numCases + n] = key ? log_prob(key_logit(key), c) : -INFINITY;
}

// The largest of x(0) ... x(COUNT - 1), quiet NaN left out, two a step.  (As asm: the compiler would first quieten every operand, one more
// instruction each.  A signalling NaN hides what came before it; the sum tells that there may be one, and then number_max() is taken.)
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}
template <int COUNT, class F>
__device__ __forceinline__ float max_of(F x) {
    if (COUNT == 1) return x(0);
    float r = COUNT == 2 ? max3(x(0), x(1), x(1)) : max3(x(0), x(1), x(COUNT > 2 ? 2 : 0));
#pragma unroll
    for (int i = 3; i < COUNT; i += 2) r = max3(r, x(i), x(i + 1 < COUNT ? i + 1 : i));
    return r;
}

// Code for what hardly happens goes out of the way.
__device__ __forceinline__ bool rare(bool v) { return __builtin_expect(v, 0); }
// The largest number of x(0) ... x(COUNT - 1); -inf if there is none.
template <int COUNT, class F>
__device__ __forceinline__ float number_max(F x) {
    float r = -INFINITY;
#pragma unroll
    for (int i = 0; i < COUNT; ++i) {
        const float y = x(i);
        r = y > r ? y : r;
        asm volatile("" : "+v"(r));   // one after the other, in few registers
    }
    return r;
}

// Nothing that was formed of these elements before is kept for what follows.
template <class T, int N, int U>
__device__ __forceinline__ void hide(Words<T, N> (&v)[U]) {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < Words<T, N>::COUNT; ++i) asm volatile("" : "+v"(v[u].w[i]));
}

// t_j = (x_j - m) log2 e as fma(x_j, log2 e, -c), c = m log2 e as rounded; what the rounding of c moved every t by is known (another fma)
// and taken back once for all.  It is half a step of c at most, 1/16 for |m| < 2^20; from there on it would cost w its accuracy, and from
// 2^31 on 2^t its range, so that t is formed from x_j - m there (exact where 2^t counts), by far_sums(), and nothing is taken back.  (No half
// is as large.)  m = -inf leaves every t at -inf.
template <class T>
__device__ __forceinline__ bool far_from_zero(float m) { return !__is_same(T, _Float16) && fabsf(m) >= kFar && m != -INFINITY; }
struct Shift { float c; };
__device__ __forceinline__ Shift shift_for(float m) { return {fmaxf(m, -1e30f) * kLog2e}; }
__device__ __forceinline__ void take_back(float m, float& s, float& w) {
    if (!(fabsf(m) < kFar)) return;
    const float c = m * kLog2e, d = fmaf(m, kLog2e, -c), f = __builtin_amdgcn_exp2f(-d);
    w = (w - d * s) * f;
    s *= f;
}
// s and w of t(0) ... t(COUNT - 1).  A ruled-out class has t = -inf and 2^t = 0, and so has to have t 2^t; without that guard w is NaN where
// there is one, and guarded() forms it again.
template <bool ENT, int COUNT, class F>
__device__ __forceinline__ void sums_of(F t, float& s, float& w) {
    s = w = 0.f;
#pragma unroll
    for (int i = 0; i < COUNT; ++i) {
        const float x = t(i), e = __builtin_amdgcn_exp2f(x);
        s += e;
        if (ENT) w = fmaf(e, x, w);
    }
    asm volatile("" : "+v"(s), "+v"(w));   // here, and not with every e kept until they are used
}
template <int COUNT, class F>
__device__ __forceinline__ float guarded(F t) {
    float w = 0.f;
#pragma unroll
    for (int i = 0; i < COUNT; ++i) {
        const float x = t(i);
        w = fmaf(__builtin_amdgcn_exp2f(x), fmaxf(x, -200.f), w);
    }
    return w;
}
// s and w of the logits x(0) ... x(COUNT - 1) for a maximum far from zero.
template <bool ENT, int COUNT, class F>
__device__ __forceinline__ void far_sums(F x, float m, float& s, float& w) {
    float base = m;
    s = w = 0.f;
#pragma unroll
    for (int i = 0; i < COUNT; ++i) {
        if (i % 4 == 0) asm volatile("" : "+v"(base), "+v"(s));   // four at a time in registers, and nothing of before kept for here
        const float t = (x(i) - base) * kLog2e, e = __builtin_amdgcn_exp2f(t);
        s += e;
        if (ENT) w = fmaf(e, fmaxf(t, -200.f), w);
    }
    asm volatile("" : "+v"(s));
}

// The largest element of a pack.
template <class T, int N>
__device__ __forceinline__ float max_in(const Words<T, N>& v, Pass p) {
    if (!__is_same(T, _Float16) || N == 1) return max_of<N>([&](int k) { return v.at(k, p); });
    Words<T, 2> m;   // two at a time
    m.w[0] = v.w[0];
#pragma unroll
    for (int i = 1; i < v.COUNT; ++i) asm("v_pk_max_f16 %0, %1, %2" : "=v"(m.w[0]) : "v"(m.w[0]), "v"(v.w[i]));
    return fmaxf(m.at(0, p), m.at(1, p));
}
// Element k as fma(x, log2 e, -c); a half goes into the fma as it is (volatile: see Pass).
template <class T, int N>
__device__ __forceinline__ float shifted(const Words<T, N>& v, int k, Shift h, Pass p) {
    if (!__is_same(T, _Float16)) return fmaf(v.at(k, p), kLog2e, -h.c);
    float t;
    if (k % 2) asm volatile("v_fma_mix_f32 %0, %1, %2, -%3 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(t) : "v"(v.w[k / 2]), "v"(kLog2e), "v"(h.c));
    else asm volatile("v_fma_mix_f32 %0, %1, %2, -%3 op_sel:[0,0,0] op_sel_hi:[1,0,0]" : "=v"(t) : "v"(v.w[k / 2]), "v"(kLog2e), "v"(h.c));
    return t;
}

// ---------------------------------------------------------------- a case's classes side by side
// A workgroup (or wave) takes up to THREADS * U packs of 16 bytes of one case into registers in one burst of loads, and does all the
// rest there: the largest logit, the sums against it, the candidates for the top.  One pass over memory, and no rescaling of running
// sums.  Long cases are bound by the vector units (7 instructions an element, 90 % busy) with HBM close behind: 2048 x 131072 bf16
// (537 MB) with entropy and 20 alternatives 93.6 us back to back, joining included, 5.7 TB/s (traced one at a time 105 and 9); reading alone
// takes 78.
// Packs that may hold candidates.  A threshold lets k + k / 4 + 1 of the lanes' maxima through at most (41 for k = 32; ties aside), and
// with them, of s lanes of many packs each, s ln(s / (s - 41)) packs on average: 45 of a workgroup's, 65 of a wave's (81 the most of 4000 cases
// of normal logits).  8192 x 1000 bf16 with 32 alternatives: 105 us with lists of 32 a wave, which nearly every case overflowed.
constexpr int packs_for(int threads, int U) { return threads == LT ? 128 : U == 1 ? 64 : 112; }
template <class T, int THREADS, int U, bool ENT, bool TOP, bool NT>
__global__ void __launch_bounds__(LT) __attribute__((amdgpu_waves_per_eu(4))) k_log_probs_rows(LogProbArgs a, Parts p) {
    typedef Group<THREADS> G;
    constexpr int V = 16 / sizeof(T), GROUPS = LT / THREADS;
    __shared__ float shRed[GROUPS][3 * (G::WAVES > 1 ? G::WAVES : 1)];
    __shared__ float shMax[TOP ? LT : 1];
    __shared__ unsigned long long shCand[TOP ? GROUPS : 1][TOP ? kCand + MC_MAX_TOP : 1];
    // the packs that hold candidates, and where they are from
    constexpr int PACKS = packs_for(THREADS, U);
    static_assert(U == 1 || PACKS >= 2 * (MC_MAX_TOP + MC_MAX_TOP / 4 + 1), "");
    __shared__ unsigned shPack[TOP ? GROUPS : 1][TOP ? PACKS : 1][4], shFrom[TOP ? GROUPS : 1][TOP ? PACKS : 1];
    __shared__ int shPacks[GROUPS], shCount[GROUPS];
    const int group = G::index(), tid = G::tid();
    const unsigned item = blockIdx.x * GROUPS + group, row = item / (unsigned)p.parts;
    if (row >= (unsigned)a.numCases) return;          // (whole waves: THREADS is 64 then)
    const int n = (int)row, lo = (int)(item - row * p.parts) * p.span;
    const T* x = static_cast<const T*>(a.logits) + row * a.caseStride + lo;   // this part's classes: lo + j, j < len
    const int len = min(a.numOut - lo, p.span);
    // A pack that would reach past the end starts V before the end instead, and what it then repeats of its neighbour becomes -inf.  (A
    // last part shorter than a pack reaches back into the part before it.)
    Words<T, V> v[U];
    const int first = tid * V, last = len - V, back = max(-last, 0);
    const bool whole = THREADS == LT || a.numOut >= V;
    if (len == THREADS * U * V) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const T* base = x + u * (THREADS * V);
            asm("" : "+s"(base));   // the scalar unit's sum, and one offset for all
            v[u].template load<NT>(base + (unsigned)first);
        }
    } else if (whole) {
        const T* from = x - back;
#pragma unroll
        for (int u = 0; u < U; ++u) v[u].template load<NT>(from + (unsigned)(min(first + u * (THREADS * V), last) + back));
#pragma unroll
        for (int u = 0; u < U; ++u) v[u].fill_first(first + u * (THREADS * V) - last);
    } else {   // fewer classes than a pack holds
#pragma unroll
        for (int u = 0; u < U; ++u) v[u].fill();
#pragma unroll
        for (int k = 0; k < V; ++k)
            if (first == 0 && k < len) v[0].set(k, x[k]);
    }
    int label = -1;
    if (a.labelLogProbs) label = label_of(a.labels, a.labelType, n, a.numOut);
    const float labelLogit = label >= lo && label < lo + len ? (float)x[label - lo] : -INFINITY;

    // The packs' maxima.  (bf16 as pairs of 16-bit integers takes half the instructions, but only where the largest is not negative, and was no
    // faster: 2048 x 131072 97 ... 103 us, this 95 ... 103.)
    float pm[U];
    {
        const Pass pass;
#pragma unroll
        for (int u = 0; u < U; ++u) pm[u] = max_in(v[u], pass);
    }
    float mine = max_of<U>([&](int u) { return pm[u]; });
    float m = G::max(mine, shRed[group]);
    if (TOP) {
        shMax[threadIdx.x] = mine;
        if (tid == 0) shCount[group] = shPacks[group] = 0;
    }
    float s, w;
    const Shift h = shift_for(m);
    {
        const Pass pass;
        sums_of<ENT, U * V>([&](int i) { return shifted(v[i / V], i % V, h, pass); }, s, w);
    }
    if (rare(__any(far_from_zero<T>(m)))) {
        const Pass pass;
        far_sums<ENT, U * V>([&](int i) { return v[i / V].at(i % V, pass); }, m, s, w);
    } else if (ENT && __any(w != w)) {   // ruled-out classes (or NaN): again, with the guard that the usual case is spared
        Shift again = h;
        asm volatile("" : "+v"(again.c));   // (not the values of before, kept)
        const Pass pass;
        w = guarded<U * V>([&](int i) { return fmaf(v[i / V].at(i % V, pass), kLog2e, -again.c); });
    }
    G::sum2(s, w, shRed[group] + G::WAVES);
    take_back(m, s, w);
    if (rare(s != s)) {   // (in the whole group)
        hide(v);
        const Pass pass;
#pragma unroll
        for (int u = 0; u < U; ++u) pm[u] = number_max<V>([&](int k) { return v[u].at(k, pass); });
        mine = number_max<U>([&](int u) { return pm[u]; });
        m = G::max(mine, shRed[group]);
        if (TOP) shMax[threadIdx.x] = mine;
    }
    const CaseStats c = case_stats(m, s);
    if (tid == 0) {
        if (p.parts == 1) write_case(a, n, c, s, w, label, labelLogit);
        else p.stats[item] = {m, s, w, labelLogit};
    }
    if (!TOP) return;

    G::sync();
    float q[THREADS / 64];
#pragma unroll
    for (int i = 0; i < THREADS / 64; ++i) q[i] = shMax[group * THREADS + i * 64 + (threadIdx.x & 63)];
    const float threshold = len <= kFewClasses ? -INFINITY : top_threshold(q, a.numTop, m, 64);
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (pm[u] >= threshold && pm[u] > -INFINITY) {
            const int to = atomicAdd(&shPacks[group], 1);
            if (to < PACKS) {
#pragma unroll
                for (int i = 0; i < 4; ++i) shPack[group][to][i] = v[u].w[i];
                shFrom[group][to] = lo + (whole ? min(first + u * (THREADS * V), last) : 0);
            }
        }
    G::sync();
    const int packs = shPacks[group];
    for (int i = tid; i < min(packs, PACKS) * V; i += THREADS) {   // an element a thread
        const unsigned word = shPack[group][i / V][i % V * sizeof(T) / 4];
        Words<T, 4 / sizeof(T)> pair;
        pair.w[0] = word;
        const float y = sizeof(T) == 4 || i % 2 == 0 ? pair.at(0, Pass()) : pair.at(sizeof(T) == 4 ? 0 : 1, Pass());
        if (y >= threshold && y > -INFINITY) {
            const int to = atomicAdd(&shCount[group], 1);
            if (to < kCand) shCand[group][to] = top_key(y, shFrom[group][i / V] + i % V);
        }
    }
    G::sync();
    const int count = shCount[group];
    const auto put = [&](int rank, unsigned long long key) {
        if (p.parts == 1) write_top(a, n, rank, key, c);
        else p.keys[(size_t)item * a.numTop + rank] = key;
    };
    if (packs <= PACKS && count <= kCand) rank_keys<false, 1>(shCand[group], count, a.numTop, tid, THREADS, put);
    else {   // ties, or orders that put many of the largest into few packs' reach
        G::sync();
        top_by_scan<THREADS>(x - lo, 1, lo, lo + len, a.numTop, shCand[group] + kCand, shCand[group]);
        if (tid < a.numTop) put(tid, shCand[group][kCand + tid]);
    }
}

// ---------------------------------------------------------------- a class's cases side by side
// A workgroup takes 256 / G classes of G * P cases at a time, U times, into registers: lane (r, g) holds P neighbouring cases of class
// r of each.  P states a lane are reduced over the lanes that share them, then over the waves.  Without alternatives the loads bound it (32000 x
// 2048 bf16, 131 MB, traced 36.5 us and 5 for joining: lines in pieces of 128 bytes); with them every workgroup looks for the best of each of its
// cases among few classes, which takes the vector units longer than the loads: the same with 20 alternatives 96 and 11 (16 more for keeping the
// stretches' maxima, 7 for thresholds, 31 for collecting what reaches them, 6 for ordering it).
// LDS of the top alternatives: the candidate lists (or what top_by_scan needs), the stretches' maxima, the counts, the thresholds.  A list
// holds what a threshold lets through with room to spare: of s stretches, k of whose maxima reach it, about s ln(s / (s - k)) classes do.
__host__ __device__ constexpr int col_cand(int top) { return 2 * top + 32; }
__host__ __device__ constexpr int col_list_keys(int cases, int top) { return cases * col_cand(top) > LT + MC_MAX_TOP ? cases * col_cand(top) : LT + MC_MAX_TOP; }
constexpr size_t col_lds_bytes(int cases, int stretches, int top) {
    return col_list_keys(cases, top) * sizeof(unsigned long long) + ((size_t)cases * (stretches + 1) + 2 * cases) * sizeof(float);
}
template <class T, int P, int U, bool ENT, bool TOP, bool NT>
__global__ void __launch_bounds__(LT) k_log_probs_cols(LogProbArgs a, Parts p, int logG) {
    constexpr int WINDOWS = U >= 2 ? 2 : 1, W = U / WINDOWS;   // the top's maxima are kept for W classes at a time
    constexpr int Q = P == 1 ? 8 : WINDOWS * P;
    extern __shared__ unsigned long long shDyn[];
    __shared__ float shM[4][8 * P], shS[4][8 * P], shW[4][8 * P];
    __shared__ int shNan;
    const int G = 1 << logG, R = LT >> logG, cases = G * P;
    const int g = threadIdx.x & (G - 1), r = threadIdx.x >> logG, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int tiles = (a.numCases + cases - 1) / cases;
    const int tile = blockIdx.x % tiles, part = blockIdx.x / tiles;
    // (the last lanes of the last tile step back to the last P cases, or repeat them: the same values are written twice)
    const int n0 = min((tile * G + g) * P, a.numCases - P);
    const int lo = part * p.span, hi = min(a.numOut - lo, p.span) + lo;
    const T* x = static_cast<const T*>(a.logits) + (size_t)n0 * (P == 1 ? a.caseStride : 1);

    Words<T, P> v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u].template load<NT>(x + (size_t)min(lo + u * R + r, hi - 1) * a.classStride);
    if (hi - lo != U * R) {
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (lo + u * R + r >= hi) v[u].fill();
    }
    // what the case's own thread will write: its way to memory (the label, then its logit) is begun now
    const int mine = min((int)threadIdx.x, cases - 1), myCase = min((tile * G + mine / P) * P, a.numCases - P) + mine % P;
    int label = -1;
    float labelLogit = -INFINITY;
    if (a.labelLogProbs && (int)threadIdx.x < cases) {
        label = label_of(a.labels, a.labelType, myCase, a.numOut);
        if (label >= lo && label < hi) labelLogit = (float)static_cast<const T*>(a.logits)[(size_t)label * a.classStride + (size_t)myCase * a.caseStride];
    }
    float pm[TOP ? WINDOWS : 1][P], m[P], s[P], w[P];
    const Pass first;
#pragma unroll
    for (int k = 0; k < P; ++k) {
        m[k] = -INFINITY;
#pragma unroll
        for (int i = 0; i < WINDOWS; ++i) {
            const float y = max_of<W>([&](int u) { return v[i * W + u].at(k, first); });
            if (TOP) pm[i][k] = y;
            m[k] = fmaxf(m[k], y);
        }
    }
    // TOP: the maxima of WINDOWS * R stretches for each case, [case][stretch]
    float* shSeg = reinterpret_cast<float*>(shDyn + col_list_keys(cases, a.numTop));
    int* shCount = reinterpret_cast<int*>(shSeg + cases * (WINDOWS * R + 1));
    float* shTau = reinterpret_cast<float*>(shCount + cases);
    if (TOP) {
#pragma unroll
        for (int k = 0; k < P; ++k)
#pragma unroll
            for (int i = 0; i < WINDOWS; ++i) shSeg[(g * P + k) * (WINDOWS * R + 1) + i * R + r] = pm[i][k];
        if ((int)threadIdx.x < cases) shCount[threadIdx.x] = 0;
    }
    if (threadIdx.x == 0) shNan = 0;
#pragma unroll
    for (int k = 0; k < P; ++k) {
        m[k] = over_lanes(m[k], G, Larger());
        if (lane < G) shM[wave][g * P + k] = m[k];
    }
    __syncthreads();
    const Pass second;
    bool far = false;
#pragma unroll
    for (int k = 0; k < P; ++k) {
        m[k] = fmaxf(fmaxf(shM[0][g * P + k], shM[1][g * P + k]), fmaxf(shM[2][g * P + k], shM[3][g * P + k]));
        const Shift h = shift_for(m[k]);
        sums_of<ENT, U>([&](int i) { return shifted(v[i], k, h, second); }, s[k], w[k]);
        far |= far_from_zero<T>(m[k]);
        if (ENT && __any(w[k] != w[k])) {   // (see the rows)
            Shift again = h;
            asm volatile("" : "+v"(again.c));
            const Pass pass;
            w[k] = guarded<U>([&](int i) { return fmaf(v[i].at(k, pass), kLog2e, -again.c); });
        }
    }
    if (rare(__any(far))) {   // (lanes of several cases share a wave)
#pragma unroll
        for (int k = 0; k < P; ++k) {
            float fs, fw;
            const Pass pass;
            far_sums<ENT, U>([&](int i) { return v[i].at(k, pass); }, m[k], fs, fw);
            s[k] = far_from_zero<T>(m[k]) ? fs : s[k];
            w[k] = far_from_zero<T>(m[k]) ? fw : w[k];
        }
    }
    bool nan = false;
#pragma unroll
    for (int k = 0; k < P; ++k) {
        s[k] = over_lanes(s[k], G, Sum());
        nan |= s[k] != s[k];
        if (ENT) w[k] = over_lanes(w[k], G, Sum());
        if (lane < G) {
            shS[wave][g * P + k] = s[k];
            shW[wave][g * P + k] = w[k];
        }
    }
    if (nan) shNan = 1;
    __syncthreads();
    if (rare(shNan)) {   // (see the rows)
        hide(v);
        const Pass pass;
#pragma unroll
        for (int k = 0; k < P; ++k) {
            m[k] = -INFINITY;
#pragma unroll
            for (int i = 0; i < WINDOWS; ++i) {
                const float y = number_max<W>([&](int u) { return v[i * W + u].at(k, pass); });
                if (TOP) {
                    pm[i][k] = y;
                    shSeg[(g * P + k) * (WINDOWS * R + 1) + i * R + r] = y;
                }
                m[k] = fmaxf(m[k], y);
            }
            m[k] = over_lanes(m[k], G, Larger());
            if (lane < G) shM[wave][g * P + k] = m[k];
        }
        __syncthreads();
    }
    if ((int)threadIdx.x < cases) {
        const int cc = threadIdx.x, n = myCase;
        float M = fmaxf(fmaxf(shM[0][cc], shM[1][cc]), fmaxf(shM[2][cc], shM[3][cc]));
        float S = shS[0][cc] + shS[1][cc] + shS[2][cc] + shS[3][cc], Wt = shW[0][cc] + shW[1][cc] + shW[2][cc] + shW[3][cc];
        take_back(M, S, Wt);
        if (p.parts == 1) {
            const CaseStats c = case_stats(M, S);
            write_case(a, n, c, S, Wt, label, labelLogit);
            if (TOP) {
                shS[0][cc] = c.logSum;   // (these two are read by their own thread only until the next barrier)
                shW[0][cc] = c.m;
            }
        } else p.stats[(size_t)n * p.parts + part] = {M, S, Wt, labelLogit};
    }
    if (!TOP) return;

    const int lanes = min(64, LT / cases), owner = threadIdx.x / lanes, sub = threadIdx.x % lanes, stretches = WINDOWS * R, cap = col_cand(a.numTop);
    const int len = hi - lo;
    const bool few = len <= kFewClasses;   // then each class has a place in its cases' lists
    const Pass third;
    if (few) {
#pragma unroll
        for (int k = 0; k < P; ++k)
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (u * R + r < len) shDyn[(g * P + k) * cap + u * R + r] = top_key(v[u].at(k, third), lo + u * R + r);
    } else {
        // thresholds: `lanes` neighbouring lanes share a case's maxima
        float q[Q];
#pragma unroll
        for (int i = 0; i < Q; ++i) {
            const int at = sub + i * lanes;
            q[i] = owner < cases && at < stretches ? shSeg[owner * (stretches + 1) + at] : -INFINITY;
        }
        const int own = min(owner, cases - 1);
        const float most = fmaxf(fmaxf(shM[0][own], shM[1][own]), fmaxf(shM[2][own], shM[3][own]));
        const float tau = top_threshold(q, a.numTop, most, lanes);
        if (owner < cases && sub == 0) shTau[owner] = tau;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < P; ++k) {
            const float tau = shTau[g * P + k];
#pragma unroll
            for (int i = 0; i < WINDOWS; ++i)
                if (pm[i][k] >= tau) {
#pragma unroll
                    for (int u = 0; u < W; ++u) {
                        const float y = v[i * W + u].at(k, third);
                        if (y >= tau && y > -INFINITY) {
                            const int to = atomicAdd(&shCount[g * P + k], 1);
                            if (to < cap) shDyn[(g * P + k) * cap + to] = top_key(y, lo + (i * W + u) * R + r);
                        }
                    }
                }
        }
    }
    __syncthreads();
    const auto put = [&](int cc, int rank, unsigned long long key) {
        const int n = min((tile * G + cc / P) * P, a.numCases - P) + cc % P;
        if (p.parts == 1) write_top(a, n, rank, key, CaseStats{shW[0][cc], shS[0][cc], 0.f});
        else p.keys[((size_t)n * p.parts + part) * a.numTop + rank] = key;
    };
    const int count = owner < cases ? few ? len : shCount[owner] : 0;
    if (owner < cases && count <= cap) {
        const auto own = [&](int rank, unsigned long long key) { put(owner, rank, key); };
        if (few) rank_keys<true, 2>(shDyn + owner * cap, count, a.numTop, sub, lanes, own);
        else rank_keys<false, U == 16 ? 4 : 1>(shDyn + owner * cap, count, a.numTop, sub, lanes, own);   // (32000 x 2048 f32: 148 us with 1 at a time, 115 with 4)
    }
    if (!__syncthreads_or(count > cap)) return;
    for (int cc = 0; cc < cases; ++cc) {   // lists that overflowed: the lists' memory is free by now
        if (shCount[cc] <= cap) continue;
        const int n = min((tile * G + cc / P) * P, a.numCases - P) + cc % P;
        top_by_scan<LT>(static_cast<const T*>(a.logits) + (size_t)n * a.caseStride, a.classStride, lo, hi, a.numTop, shDyn + LT, shDyn);
        if ((int)threadIdx.x < a.numTop) put(cc, threadIdx.x, shDyn[LT + threadIdx.x]);
        __syncthreads();
    }
}

// ---------------------------------------------------------------- joining the parts of a case
// A wave joins up to 16 parts (2048 cases of 4: 8 us, a workgroup each 9), whose keys it holds at once: the threshold is found from all of them.  Beyond, a workgroup does: a first
// threshold from the parts' best keys (or their last ones, where there are few parts), a better one from what reaches that.  (Ordering what
// only the first lets through took most of the time: 16 parts of 20 keys each 19.7 us.)
constexpr int kJoinWave = 16, kJoinCand = 1024, kJoinFew = 128;
template <int THREADS>
__global__ void __launch_bounds__(LT) k_log_probs_join(LogProbArgs a, Parts p) {
    typedef Group<THREADS> G;
    constexpr int GROUPS = LT / THREADS, CAND = THREADS == 64 ? kJoinFew : kJoinCand;
    __shared__ float shRed[GROUPS][4 * G::WAVES];
    __shared__ unsigned long long shCand[GROUPS][CAND];
    __shared__ unsigned long long shBest[THREADS == LT ? kJoinFew : 1];
    __shared__ int shCount[GROUPS], shBestCount;
    const int group = G::index(), tid = G::tid();
    const size_t row = (size_t)blockIdx.x * GROUPS + group;
    if (row >= (size_t)a.numCases) return;
    const int n = (int)row;
    // All that is read is under way before anything is waited for: statistics, label, the parts' best keys, and as many of all keys as the
    // threads hold at EARLY each.
    constexpr int EARLY = THREADS == 64 ? kJoinWave * MC_MAX_TOP / 64 : 6;
    const Part* stats = p.stats + row * p.parts;
    const unsigned long long* keys = p.keys + row * p.parts * a.numTop;
    const int total = p.parts * a.numTop;
    Part part = {-INFINITY, 0.f, 0.f, -INFINITY};
    if (tid < p.parts) part = stats[tid];
    int label = -1;
    if (a.labelLogProbs) label = label_of(a.labels, a.labelType, n, a.numOut);
    const unsigned long long tail = THREADS == LT && a.numTop && tid < p.parts ? keys[(size_t)(tid + 1) * a.numTop - 1] : 0;
    unsigned long long early[EARLY];
#pragma unroll
    for (int i = 0; i < EARLY; ++i) early[i] = tid + i * THREADS < total ? keys[tid + i * THREADS] : 0;
    const bool thresholds = THREADS == LT && p.parts > a.numTop;
    constexpr int Q = 8;
    unsigned long long head[Q];
    const int heads = min(p.parts, 64 * Q);   // (beyond: the first ones' threshold holds too)
#pragma unroll
    for (int i = 0; i < Q; ++i) head[i] = thresholds && (int)(threadIdx.x & 63) + 64 * i < heads ? keys[(size_t)((threadIdx.x & 63) + 64 * i) * a.numTop] : 0;
    if (tid == 0) shCount[group] = shBestCount = 0;
    float m = part.m, labelLogit = part.label;
    for (int i = tid + THREADS; i < p.parts; i += THREADS) {
        m = fmaxf(m, stats[i].m);
        labelLogit = fmaxf(labelLogit, stats[i].label);
    }
    m = G::max(m, shRed[group]);
    float s = 0.f, w = 0.f;
    for (int i = tid; i < p.parts; i += THREADS) {
        if (i != tid) part = stats[i];
        const float d = part.m == m ? 0.f : (part.m - m) * kLog2e, f = __builtin_amdgcn_exp2f(d);
        s += part.s * f;
        w += fmaf(fmaxf(d, -200.f), part.s, part.w) * f;
    }
    G::sum2(s, w, shRed[group] + G::WAVES);
    labelLogit = G::max(labelLogit, shRed[group] + 3 * G::WAVES);
    const CaseStats c = case_stats(m, s);
    if (tid == 0) write_case(a, n, c, s, w, label, labelLogit);
    if (!a.numTop) return;

    // candidates: keys that reach a value that numTop parts' best keys reach
    float threshold = -INFINITY;
    if (THREADS == 64) {
        float q[EARLY];
#pragma unroll
        for (int i = 0; i < EARLY; ++i) q[i] = early[i] ? key_logit(early[i]) : -INFINITY;
        threshold = total > kFewClasses ? top_threshold(q, a.numTop, m, 64) : -INFINITY;
    } else if (thresholds) {
        float q[Q];
#pragma unroll
        for (int i = 0; i < Q; ++i) q[i] = head[i] ? key_logit(head[i]) : -INFINITY;
        threshold = top_threshold(q, a.numTop, m, 64);
    } else {   // few parts: the last key of any part's list has numTop keys from it up
        float last = tid < p.parts && tail ? key_logit(tail) : -INFINITY;
        threshold = over_lanes(last, 1, Larger());   // (in the first wave; parts <= numTop are all there, and the others' -inf is a threshold too)
    }
    const auto take = [&](unsigned long long key) {
        if (key && key_logit(key) >= threshold) {
            const int to = atomicAdd(&shCount[group], 1);
            if (to < CAND) shCand[group][to] = key;
        }
    };
    G::sync();
#pragma unroll
    for (int i = 0; i < EARLY; ++i) take(early[i]);
    if (THREADS == LT)
        for (int i = tid + EARLY * THREADS; i < total; i += THREADS) take(keys[i]);
    G::sync();
    int count = shCount[group];
    if (count <= CAND) {
        const unsigned long long* list = shCand[group];
        if (THREADS == LT && count > kJoinFew) {
            float q[CAND / 64];
#pragma unroll
            for (int i = 0; i < CAND / 64; ++i) {
                const int at = i * 64 + (threadIdx.x & 63);
                q[i] = at < count ? key_logit(list[at]) : -INFINITY;
            }
            const float better = top_threshold(q, a.numTop, m, 64);
            for (int i = tid; i < count; i += THREADS)
                if (key_logit(list[i]) >= better) {
                    const int to = atomicAdd(&shBestCount, 1);
                    if (to < kJoinFew) shBest[to] = list[i];
                }
            G::sync();
            if (shBestCount <= kJoinFew) {
                list = shBest;
                count = shBestCount;
            }
        }
        rank_keys<false, 1>(list, count, a.numTop, tid, THREADS, [&](int rank, unsigned long long key) { write_top(a, n, rank, key, c); });
        return;
    }
    // more ties than the list holds: the best, then the best below it, and so on
    unsigned long long last = ~0ull;
    for (int r = 0; r < a.numTop; ++r) {
        unsigned long long best = 0;
        for (int i = tid; i < total; i += THREADS) {
            const unsigned long long key = keys[i];
            if (key < last && key > best) best = key;
        }
        for (int off = 32; off > 0; off >>= 1) best = std::max(best, __shfl_xor(best, off, 64));
        if (G::WAVES > 1) {
            G::sync();
            if ((threadIdx.x & 63) == 0) shCand[group][threadIdx.x >> 6] = best;
            G::sync();
            for (int i = 0; i < G::WAVES; ++i) best = std::max(best, shCand[group][i]);
        }
        if (tid == 0) write_top(a, n, r, best, c);
        last = best;
    }
}

// ---------------------------------------------------------------- the gradient
struct LogProbGradArgs {
    const void* logits;
    size_t classStride, caseStride;
    const void* labels;
    int labelType, numCases, numOut;
    const float *maxAndLogSum, *entropy;
    const float *gradLabel, *gradEntropy, *gradLogZ;
    float scaleLabel, scaleEntropy, scaleLogZ;
    void* target;
    size_t targetClassStride, targetCaseStride;
    int add;
};

// d_j = p_j (A - h (ln p_j + H)) + [j = y] a.  Each logit is read and each gradient written once: bound by HBM.  2048 x 131072 bf16
// (1.07 GB) 176 us, 6.1 TB/s; 511 x 50021 f32 (204 MB) 38.
struct CaseGrad { float m, logSum, A, h, H, a; int y; };
// A case's weights, of N neighbouring cases.
template <int N>
__device__ __forceinline__ void load_words(const void* p, int n0, unsigned (&w)[N]) {
    constexpr int V = N % 4 == 0 ? 4 : 1;
#pragma unroll
    for (int i = 0; i < N; i += V) {
        Words<float, V> q;
        q.template load<false>(static_cast<const float*>(p) + n0 + i);
#pragma unroll
        for (int k = 0; k < V; ++k) w[i + k] = q.w[k];
    }
}
template <bool ENT, int N>
__device__ __forceinline__ void case_grads(const LogProbGradArgs& g, int n0, CaseGrad (&c)[N]) {
    unsigned m[N], logSum[N], y[N], gl[N], gz[N], ge[N], H[N];
    load_words(g.maxAndLogSum, n0, m);
    load_words(g.maxAndLogSum + g.numCases, n0, logSum);
    if (g.scaleLabel != 0.f) load_words(g.labels, n0, y);
    if (g.scaleLabel != 0.f && g.gradLabel) load_words(g.gradLabel, n0, gl);
    if (g.scaleLogZ != 0.f && g.gradLogZ) load_words(g.gradLogZ, n0, gz);
    if (ENT && g.gradEntropy) load_words(g.gradEntropy, n0, ge);
    if (ENT) load_words(g.entropy, n0, H);
#pragma unroll
    for (int k = 0; k < N; ++k) {
        c[k].m = __uint_as_float(m[k]);
        c[k].logSum = __uint_as_float(logSum[k]);
        c[k].y = g.scaleLabel != 0.f ? label_from(y[k], g.labelType, g.numOut) : -1;
        c[k].a = c[k].y >= 0 ? g.scaleLabel * (g.gradLabel ? __uint_as_float(gl[k]) : 1.f) : 0.f;
        c[k].A = (g.scaleLogZ != 0.f ? g.scaleLogZ * (g.gradLogZ ? __uint_as_float(gz[k]) : 1.f) : 0.f) - c[k].a;
        c[k].h = ENT ? g.scaleEntropy * (g.gradEntropy ? __uint_as_float(ge[k]) : 1.f) : 0.f;
        c[k].H = ENT ? __uint_as_float(H[k]) : 0.f;
        if (c[k].m == -INFINITY) {   // every class is ruled out: p = 0 throughout, and the label's term goes too
            c[k].m = c[k].logSum = c[k].a = 0.f;
            c[k].y = -1;
        }
    }
}
template <bool ENT>
__device__ __forceinline__ CaseGrad case_grad(const LogProbGradArgs& g, int n) {
    CaseGrad c[1];
    case_grads<ENT>(g, n, c);
    return c[0];
}
template <bool ENT>
__device__ __forceinline__ float grad_of(float x, const CaseGrad& c) {
    const float lp = (x - c.m) - c.logSum, p = __builtin_amdgcn_exp2f(lp * kLog2e);
    return ENT ? p * fmaf(-c.h, fmaxf(lp, -200.f) + c.H, c.A) : p * c.A;
}

// The gradient of a pack (and, with add, of what the target holds), element by element.  y: the label's place in the pack, if it is in it.
template <bool ENT, class T, int N>
__device__ __forceinline__ Pack<T, N> grad_pack(const Words<T, N>& v, const Words<T, N>& t, bool add, const CaseGrad& c, int y, Pass pass) {
    Pack<T, N> d;
    const bool here = (unsigned)y < (unsigned)N;
#pragma unroll
    for (int k = 0; k < N; ++k) {
        float x = grad_of<ENT>(v.at(k, pass), c);
        if (here && y == k) x += c.a;
        if (add) x += t.at(k, pass);
        d.v[k] = (T)x;
    }
    return d;
}

// U = 4 packs a thread: 2048 x 131072 bf16 178 us; with 2 187, with 8 183.
template <class T, int THREADS, int U, bool ENT, bool NT>
__global__ void __launch_bounds__(LT) k_log_probs_grad_rows(LogProbGradArgs g, int parts) {
    typedef Group<THREADS> G;
    constexpr int V = 16 / sizeof(T), GROUPS = LT / THREADS;
    const unsigned item = blockIdx.x * GROUPS + G::index(), row = item / (unsigned)parts;
    if (row >= (unsigned)g.numCases) return;
    const int lo = (int)(item - row * parts) * (THREADS * U * V), len = g.numOut - lo;
    const T* x = static_cast<const T*>(g.logits) + row * g.caseStride + lo;
    T* out = static_cast<T*>(g.target) + row * g.targetCaseStride + lo;
    const int first = G::tid() * V, last = len - V;
    const Pass pass;
    if (last >= 0) {   // whole packs; those past the end read the last one and write nothing
        Words<T, V> v[U], t[U];
#pragma unroll
        for (int u = 0; u < U; ++u) v[u].template load<NT>(x + (unsigned)min(first + u * (THREADS * V), last));
        if (g.add) {
#pragma unroll
            for (int u = 0; u < U; ++u) t[u].template load<NT>(out + (unsigned)min(first + u * (THREADS * V), last));
        }
        const CaseGrad c = case_grad<ENT>(g, (int)row);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int j = first + u * (THREADS * V);
            const Pack<T, V> d = grad_pack<ENT>(v[u], t[u], g.add, c, c.y - lo - j, pass);
            if (j <= last) store_pack<NT, T, V>(out + (unsigned)j, d);
        }
    }
    const int rest = len % V, at = len - rest + G::tid();   // the case's last classes, where they fill no pack
    if (len <= THREADS * U * V && G::tid() < rest) {
        const CaseGrad c = case_grad<ENT>(g, (int)row);
        Words<T, 1> v, t;
        v.template load<false>(x + at);
        if (g.add) t.template load<false>(out + at);
        store_pack<false, T, 1>(out + at, grad_pack<ENT>(v, t, g.add, c, c.y - lo - at, pass));
    }
}

// A lane takes P neighbouring cases of U classes; the cases that fill no pack are taken one a lane (P = 1) by the lanes
// behind the packs'.  What a case needs is loaded once for all of a lane's classes.  Up to 64 lanes side by side, so that a wave's accesses
// make whole lines: 50021 x 511 f32 51 us, 62 with 32 lanes, 78 with 16.  U = 2: 48, and 1000 x 128 3.3 us against 3.7 with 4 (32000 x 2048
// bf16: 49 against 47).
template <class T, int P, int U, bool ENT, bool NT>
__global__ void __launch_bounds__(LT) k_log_probs_grad_cols(LogProbGradArgs g, int logG) {
    const int G = 1 << logG, R = LT >> logG, packs = g.numCases / P, columns = packs + g.numCases % P;
    const int tiles = (columns + G - 1) >> logG;
    const int column = ((int)(blockIdx.x % tiles) << logG) + (threadIdx.x & (G - 1));
    const int j0 = (int)(blockIdx.x / tiles) * (R * U) + (threadIdx.x >> logG);
    if (column >= columns) return;
    const T* logits = static_cast<const T*>(g.logits);
    T* target = static_cast<T*>(g.target);
    const auto take = [&](auto width, int n0) {
        constexpr int N = decltype(width)::value;
        const T* x = logits + (size_t)n0 * (P == 1 ? g.caseStride : 1);
        T* out = target + (size_t)n0 * (P == 1 ? g.targetCaseStride : 1);
        Words<T, N> v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) v[u].template load<NT>(x + (size_t)min(j0 + u * R, g.numOut - 1) * g.classStride);
        CaseGrad c[N];
        case_grads<ENT>(g, n0, c);
        bool here = false;   // is a label of these cases among these classes, or between them?
#pragma unroll
        for (int k = 0; k < N; ++k) here |= (unsigned)(c[k].y - j0) < (unsigned)(R * U);
        const Pass pass;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int j = j0 + u * R;
            Words<T, N> t;
            if (g.add) t.template load<NT>(out + (size_t)min(j, g.numOut - 1) * g.targetClassStride);
            Pack<T, N> d;
            float e[N];
#pragma unroll
            for (int k = 0; k < N; ++k) e[k] = grad_of<ENT>(v[u].at(k, pass), c[k]);
            if (here) {
#pragma unroll
                for (int k = 0; k < N; ++k)
                    if (j == c[k].y) e[k] += c[k].a;
            }
#pragma unroll
            for (int k = 0; k < N; ++k) d.v[k] = (T)(g.add ? e[k] + t.at(k, pass) : e[k]);
            if (j < g.numOut) store_pack<NT, T, N>(out + (size_t)j * g.targetClassStride, d);
        }
    };
    if (P > 1 && column >= packs) take(std::integral_constant<int, 1>(), packs * P + (column - packs));
    else take(std::integral_constant<int, P>(), column * P);
}

// Element (class j, case n) at j*classStride + n*caseStride.  BY_CASE: a case's classes side by side; BY_CLASS: a class's cases.
enum { BY_CASE = 1, BY_CLASS = 2 };
int layout_kinds(long long classStride, long long caseStride, int numCases, int numOut) {
    const long long most = 1ll << 60;
    if (classStride < 1 || caseStride < 1 || classStride > most / numOut || caseStride > most / numCases) return 0;
    int kinds = 0;
    if ((classStride == 1 || numOut == 1) && (numCases == 1 || caseStride >= numOut)) kinds |= BY_CASE;
    if ((caseStride == 1 || numCases == 1) && (numOut == 1 || classStride >= numCases)) kinds |= BY_CLASS;
    return kinds;
}
#define MC_LAYOUT_RULE "strides must be positive and not too large, one of them 1 and the other at least as long as the lines it separates"

int check_labels(const char* what, const void* labels, int labelType, int numOut) {
    MC_REQUIRE(labels && ((size_t)labels & 3) == 0, "%s: labels are null or not aligned", what);
    MC_REQUIRE(labelType == MC_I32 || labelType == MC_F32, "%s: labels must be MC_I32 or MC_F32", what);
    MC_REQUIRE(labelType == MC_I32 || numOut <= 1 << 24, "%s: float32 labels cannot name %d classes", what, numOut);
    return MC_OK;
}

// ---------------------------------------------------------------- how a call is cut up
// Logits with a case's classes side by side: up to 64 * 4 packs of 16 bytes a wave takes a case, beyond a workgroup (8192 x 1000 f32:
// 12.4 us, a workgroup each 21.5), and a case is split where it is longer than 256 * 16 packs or where there are too few cases to fill
// the device: 16 packs a thread where that still makes 4 workgroups a CU, else 4 where that makes one, else 1 (257 x 50021 f16 14.3 us
// in parts of 4 packs a thread, 17.6 in parts of 16; 128 x 131072 bf16 12.6 and 13.7).  Class-major logits: see below.
struct Plan {
    bool rows;
    int threads;   // rows: of a group
    int P, logG;   // cols: cases of a lane, lanes of a class
    int U;
    Parts parts;
    size_t blocks, bytes;
};
Plan plan_log_probs(int type, int kinds, int numCases, int numOut, int numTop) {
    Plan p{};
    const int V = 16 / elem_size(type), cus = num_cus();
    p.rows = kinds & BY_CASE;
    p.parts.parts = 1;
    if (p.rows) {
        if (numOut <= 64 * V * 4) {
            p.threads = 64;
            p.U = numOut <= 64 * V ? 1 : 4;
            p.parts.span = numOut;
            p.blocks = ceil_div(numCases, LT / 64);
        } else {
            p.threads = LT;
            for (p.U = 16; p.U > 1 && (numOut <= LT * V * (p.U / 4) || (size_t)numCases * ceil_div(numOut, LT * V * p.U) < (p.U == 16 ? 4 : 1) * (size_t)cus); p.U /= 4) {}
            p.parts.parts = ceil_div(numOut, LT * V * p.U);
            p.parts.span = ceil_div(ceil_div(numOut, p.parts.parts), V) * V;
            p.parts.parts = ceil_div(numOut, p.parts.span);
            p.blocks = (size_t)numCases * p.parts.parts;
        }
    } else {
        p.P = V;
        if (numCases < p.P) p.P = 1;
        // A small matrix: every case in one part, if a workgroup of R classes by 1 ... 16 can hold it.  (Its lines are then read in short
        // pieces, which the L2 makes up for; joining costs a launch: 1000 x 128 f32 9.5 us, split 15.2; 4000 x 128 16.9 and 16.1.)
        const bool small = (size_t)numCases * numOut * elem_size(type) <= (4u << 20) && numOut <= LT * 16;
        const int most = numTop && p.P == 8 ? 2 : 3;   // (32 cases' candidates to a workgroup, of 64 classes at a time: 32000 x 2048 bf16 109 us, with 64 cases 200)
        for (p.U = small ? 1 : 16; small && LT * p.U < numOut; p.U *= 4) {}
        while (p.logG < most && (p.P << p.logG) < numCases && (!small || (LT >> (p.logG + 1)) * p.U >= numOut)) ++p.logG;
        const int R = LT >> p.logG, tiles = ceil_div(numCases, p.P << p.logG);
        if (!small)   // (up to 256 parts, or joining them takes longer than what it gains: 131072 x 4 bf16 16.4 us in 128 parts, 23.8 in 512)
            for (; p.U > 1 && (numOut <= R * (p.U / 4) || ((size_t)tiles * ceil_div(numOut, R * p.U) < 2 * (size_t)cus && ceil_div(numOut, R * (p.U / 4)) <= 256)); p.U /= 4) {}
        p.parts.span = R * p.U;
        p.parts.parts = ceil_div(numOut, p.parts.span);
        p.blocks = (size_t)tiles * p.parts.parts;
    }
    if (p.parts.parts > 1) p.bytes = (size_t)numCases * p.parts.parts * (sizeof(Part) + numTop * sizeof(unsigned long long));
    return p;
}

template <class T, bool ENT, bool TOP, bool NT>
void launch_rows(const Plan& p, const LogProbArgs& a, hipStream_t s) {
    const dim3 grid((unsigned)p.blocks), block(LT);
    if (p.threads == 64) {
        if (p.U == 1) hipLaunchKernelGGL((k_log_probs_rows<T, 64, 1, ENT, TOP, NT>), grid, block, 0, s, a, p.parts);
        else hipLaunchKernelGGL((k_log_probs_rows<T, 64, 4, ENT, TOP, NT>), grid, block, 0, s, a, p.parts);
    } else if (p.U == 1) hipLaunchKernelGGL((k_log_probs_rows<T, LT, 1, ENT, TOP, false>), grid, block, 0, s, a, p.parts);   // (few cases: little data)
    else if (p.U == 4) hipLaunchKernelGGL((k_log_probs_rows<T, LT, 4, ENT, TOP, NT>), grid, block, 0, s, a, p.parts);
    else hipLaunchKernelGGL((k_log_probs_rows<T, LT, 16, ENT, TOP, NT>), grid, block, 0, s, a, p.parts);
}
template <class T, int P, bool ENT, bool TOP, bool NT>
void launch_cols(const Plan& p, const LogProbArgs& a, hipStream_t s) {
    const dim3 grid((unsigned)p.blocks), block(LT);
    const size_t lds = TOP ? col_lds_bytes(P << p.logG, std::min(p.U, 2) * (LT >> p.logG), a.numTop) : 0;
    if (p.U == 1) hipLaunchKernelGGL((k_log_probs_cols<T, P, 1, ENT, TOP, NT>), grid, block, lds, s, a, p.parts, p.logG);
    else if (p.U == 4) hipLaunchKernelGGL((k_log_probs_cols<T, P, 4, ENT, TOP, NT>), grid, block, lds, s, a, p.parts, p.logG);
    else hipLaunchKernelGGL((k_log_probs_cols<T, P, 16, ENT, TOP, NT>), grid, block, lds, s, a, p.parts, p.logG);
}
template <class T, bool ENT, bool TOP, bool NT>
void launch_parts(const Plan& p, const LogProbArgs& a, hipStream_t s) {
    if (p.rows) launch_rows<T, ENT, TOP, NT>(p, a, s);
    else if (p.P == 1) launch_cols<T, 1, ENT, TOP, false>(p, a, s);
    else launch_cols<T, 16 / (int)sizeof(T), ENT, TOP, NT>(p, a, s);
}
template <class T, bool ENT, bool TOP>
void launch_log_probs(const Plan& p, const LogProbArgs& a, hipStream_t s) {
    if (streams((size_t)a.numCases * a.numOut * sizeof(T))) launch_parts<T, ENT, TOP, true>(p, a, s);
    else launch_parts<T, ENT, TOP, false>(p, a, s);
    if (p.parts.parts == 1) return;
    if (p.parts.parts <= kJoinWave) hipLaunchKernelGGL((k_log_probs_join<64>), dim3(ceil_div(a.numCases, LT / 64)), dim3(LT), 0, s, a, p.parts);
    else hipLaunchKernelGGL((k_log_probs_join<LT>), dim3(a.numCases), dim3(LT), 0, s, a, p.parts);
}

template <class T, bool ENT, bool NT>
bool launch_grad_rows(const LogProbGradArgs& g, hipStream_t s) {
    constexpr int V = 16 / (int)sizeof(T), U = 4;
    const dim3 block(LT);
    if (g.numOut <= 64 * V * U) {
        if (!fits_a_grid(ceil_div(g.numCases, LT / 64), LT)) return false;
        const dim3 grid(ceil_div(g.numCases, LT / 64));
        if (g.numOut <= 64 * V) hipLaunchKernelGGL((k_log_probs_grad_rows<T, 64, 1, ENT, NT>), grid, block, 0, s, g, 1);
        else hipLaunchKernelGGL((k_log_probs_grad_rows<T, 64, U, ENT, NT>), grid, block, 0, s, g, 1);
    } else {
        const int parts = ceil_div(g.numOut, LT * V * U);
        if (!fits_a_grid((size_t)g.numCases * parts, LT)) return false;
        hipLaunchKernelGGL((k_log_probs_grad_rows<T, LT, U, ENT, NT>), dim3((unsigned)((size_t)g.numCases * parts)), block, 0, s, g, parts);
    }
    return true;
}
template <class T, bool ENT, bool NT>
bool launch_grad_cols(const LogProbGradArgs& g, hipStream_t s) {
    constexpr int V = 16 / (int)sizeof(T), U = 2;
    const int columns = g.numCases < V ? g.numCases : g.numCases / V + g.numCases % V;
    int logG = 0;
    while (logG < 6 && (1 << logG) < columns) ++logG;
    const size_t tiles = ceil_div(columns, 1 << logG);
    const size_t blocks = tiles * ceil_div(g.numOut, (LT >> logG) * U);
    if (!fits_a_grid(blocks, LT)) return false;
    const dim3 block(LT), grid((unsigned)blocks);
    if (g.numCases < V) hipLaunchKernelGGL((k_log_probs_grad_cols<T, 1, U, ENT, false>), grid, block, 0, s, g, logG);
    else hipLaunchKernelGGL((k_log_probs_grad_cols<T, V, U, ENT, NT>), grid, block, 0, s, g, logG);
    return true;
}
template <class T, bool ENT>
bool launch_grad(const LogProbGradArgs& g, bool rows, hipStream_t s) {
    if (streams((size_t)g.numCases * g.numOut * sizeof(T) * 2)) return rows ? launch_grad_rows<T, ENT, true>(g, s) : launch_grad_cols<T, ENT, true>(g, s);
    return rows ? launch_grad_rows<T, ENT, false>(g, s) : launch_grad_cols<T, ENT, false>(g, s);
}

}  // namespace
}  // namespace mc
using namespace mc;

extern "C" {

size_t mc_log_probs_workspace_bytes(int type, long long classStride, long long caseStride, int numCases, int numOut, int numTop) {
    if (!float_type(type) || numCases <= 0 || numOut <= 0 || numOut > kMaxOut || numTop < 0 || numTop > MC_MAX_TOP) return 0;
    const int kinds = layout_kinds(classStride, caseStride, numCases, numOut);
    return kinds ? plan_log_probs(type, kinds, numCases, numOut, numTop).bytes : 0;
}

int mc_log_probs(const void* logits, int type, long long classStride, long long caseStride, const void* labels, int labelType, int numCases, int numOut,
                 float* labelLogProbs, float* entropy, float* maxAndLogSum, int* topClasses, float* topLogProbs, int numTop, void* workspace,
                 size_t workspaceBytes, mcStream_t s) {
    MC_REQUIRE(numCases >= 0 && numOut > 0 && numOut <= kMaxOut, "mc_log_probs: %d cases of %d classes", numCases, numOut);
    MC_REQUIRE(float_type(type), "mc_log_probs: unknown element type %d", type);
    MC_REQUIRE(numTop >= 0 && numTop <= MC_MAX_TOP, "mc_log_probs: numTop must be in [0, %d]", MC_MAX_TOP);
    if (numCases == 0) return MC_OK;
    MC_REQUIRE(logits && (size_t)logits % elem_size(type) == 0, "mc_log_probs: logits are null or not aligned to their elements");
    const int kinds = layout_kinds(classStride, caseStride, numCases, numOut);
    MC_REQUIRE(kinds, "mc_log_probs: " MC_LAYOUT_RULE);
    if (labelLogProbs) {
        const int rc = check_labels("mc_log_probs", labels, labelType, numOut);
        if (rc) return rc;
    }
    MC_REQUIRE(numTop ? topClasses && topLogProbs : !topClasses && !topLogProbs, "mc_log_probs: topClasses and topLogProbs are needed exactly where numTop > 0");
    MC_REQUIRE(labelLogProbs || entropy || maxAndLogSum || numTop, "mc_log_probs: no output asked for");
    MC_REQUIRE(stream_on_current_device(s), "mc_log_probs: the stream belongs to another device than the current one");
    Plan p = plan_log_probs(type, kinds, numCases, numOut, numTop);
    MC_REQUIRE(fits_a_grid(p.blocks, LT), "mc_log_probs: too many cases");
    if (p.bytes && (!workspace || workspaceBytes < p.bytes || !aligned16(workspace))) {
        set_error("mc_log_probs: workspace of %zu bytes, 16-byte aligned, needed", p.bytes);
        return MC_EWORKSPACE;
    }
    p.parts.stats = static_cast<Part*>(workspace);
    p.parts.keys = reinterpret_cast<unsigned long long*>(p.parts.stats + (p.bytes ? (size_t)numCases * p.parts.parts : 0));
    const LogProbArgs a{logits, (size_t)classStride, (size_t)caseStride, labels, labelType, numCases, numOut, labelLogProbs, entropy, maxAndLogSum,
                        topClasses, topLogProbs, numTop};
    with_type(type, [&](auto t) {
        typedef decltype(t) T;
        if (numTop) launch_log_probs<T, true, true>(p, a, S(s));
        else if (entropy) launch_log_probs<T, true, false>(p, a, S(s));
        else launch_log_probs<T, false, false>(p, a, S(s));
    });
    return launch_status("mc_log_probs");
}

int mc_log_probs_grad(const void* logits, int type, long long classStride, long long caseStride, const void* labels, int labelType, int numCases,
                      int numOut, const float* maxAndLogSum, const float* entropy, const float* gradLabel, float scaleLabel, const float* gradEntropy,
                      float scaleEntropy, const float* gradLogZ, float scaleLogZ, void* target, long long targetClassStride,
                      long long targetCaseStride, int add, mcStream_t s) {
    MC_REQUIRE(numCases >= 0 && numOut > 0 && numOut <= kMaxOut, "mc_log_probs_grad: %d cases of %d classes", numCases, numOut);
    MC_REQUIRE(float_type(type), "mc_log_probs_grad: unknown element type %d", type);
    if (numCases == 0) return MC_OK;
    MC_REQUIRE(logits && target && (size_t)logits % elem_size(type) == 0 && (size_t)target % elem_size(type) == 0,
               "mc_log_probs_grad: logits or target are null or not aligned to their elements");
    MC_REQUIRE(maxAndLogSum, "mc_log_probs_grad: maxAndLogSum is null");
    const int kinds = layout_kinds(classStride, caseStride, numCases, numOut), targetKinds = layout_kinds(targetClassStride, targetCaseStride, numCases, numOut);
    MC_REQUIRE(kinds, "mc_log_probs_grad: " MC_LAYOUT_RULE);
    MC_REQUIRE(targetKinds, "mc_log_probs_grad: target: " MC_LAYOUT_RULE);
    MC_REQUIRE(kinds & targetKinds, "mc_log_probs_grad: logits and target are laid out in different orders");
    const bool inPlace = logits == target && (classStride == targetClassStride || numOut == 1) && (caseStride == targetCaseStride || numCases == 1);
    const size_t size = elem_size(type), from = (size_t)logits, to = (size_t)target;
    const size_t fromEnd = from + size * (size_t)((numOut - 1) * classStride + (numCases - 1) * caseStride + 1);
    const size_t toEnd = to + size * (size_t)((numOut - 1) * targetClassStride + (numCases - 1) * targetCaseStride + 1);
    MC_REQUIRE(inPlace || from >= toEnd || to >= fromEnd, "mc_log_probs_grad: target overlaps the logits (in place needs the same pointer and strides)");
    if (scaleLabel != 0.f) {
        const int rc = check_labels("mc_log_probs_grad", labels, labelType, numOut);
        if (rc) return rc;
    }
    MC_REQUIRE(scaleEntropy == 0.f || entropy, "mc_log_probs_grad: the entropy's gradient needs the entropy");
    MC_REQUIRE(stream_on_current_device(s), "mc_log_probs_grad: the stream belongs to another device than the current one");
    const LogProbGradArgs a{logits, (size_t)classStride, (size_t)caseStride, labels, labelType, numCases, numOut, maxAndLogSum, entropy, gradLabel,
                            gradEntropy, gradLogZ, scaleLabel, scaleEntropy, scaleLogZ, target, (size_t)targetClassStride, (size_t)targetCaseStride, add};
    bool fits = true;
    with_type(type, [&](auto t) {
        typedef decltype(t) T;
        fits = scaleEntropy != 0.f ? launch_grad<T, true>(a, kinds & targetKinds & BY_CASE, S(s)) : launch_grad<T, false>(a, kinds & targetKinds & BY_CASE, S(s));
    });
    MC_REQUIRE(fits, "mc_log_probs_grad: too many cases");
    return launch_status("mc_log_probs_grad");
}

}  // extern "C"
