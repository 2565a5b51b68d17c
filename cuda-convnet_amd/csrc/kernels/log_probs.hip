// log_probs.hip -- log probabilities of given classes with entropy and top alternatives, and their gradient.
// With m the largest logit of a case, t_j = x_j - m, s = sum_j e^t_j, w = sum_j t_j e^t_j:
//   ln p_j = t_j - ln s,   -sum_j p_j ln p_j = ln s - w / s.
#include <math.h>
#include "mc_types.h"

namespace mc {
namespace {

constexpr int LT = 256;   // threads of a workgroup

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

// The label of case n, or -1 for "no class".
__device__ __forceinline__ int label_of(const void* labels, int labelType, int n, int numOut) {
    if (labelType == MC_I32) {
        const int y = static_cast<const int*>(labels)[n];
        return y >= 0 && y < numOut ? y : -1;
    }
    const float y = static_cast<const float*>(labels)[n];
    return y >= 0.f && y < (float)numOut ? (int)y : -1;
}

__device__ __forceinline__ float block_max(float v, float* sh) {
    for (int off = 32; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor(v, off, 64));
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    float r = sh[0];
    for (int i = 1; i < LT / 64; ++i) r = fmaxf(r, sh[i]);
    __syncthreads();
    return r;
}
__device__ __forceinline__ float block_sum(float v, float* sh) {
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    float r = sh[0];
    for (int i = 1; i < LT / 64; ++i) r += sh[i];
    __syncthreads();
    return r;
}

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

// The k largest keys of a case in one walk over its classes in order: 256 classes at a time against the k-th best so far; what
// beats it joins the list, which is ordered again by counting, for each key, the larger ones.
template <class T>
__device__ void top_by_scan(const T* x, size_t stride, int numOut, int k, unsigned long long* best, unsigned long long* fresh) {
    const int tid = threadIdx.x;
    if (tid < k) best[tid] = 0;
    __syncthreads();
    for (int base = 0; base < numOut; base += LT) {
        const int j = base + tid;
        unsigned long long key = j < numOut ? top_key((float)x[(size_t)j * stride], j) : 0;
        if (key <= best[k - 1]) key = 0;
        if (!__syncthreads_or(key != 0)) continue;
        fresh[tid] = key;
        const unsigned long long mine = tid < k ? best[tid] : 0;
        __syncthreads();
        int rank = 0, mineRank = 0;
        for (int i = 0; i < LT; ++i) {
            rank += fresh[i] > key;
            mineRank += fresh[i] > mine;
        }
        for (int i = 0; i < k; ++i) rank += best[i] > key;
        __syncthreads();
        if (mine && tid + mineRank < k) best[tid + mineRank] = mine;
        if (key && rank < k) best[rank] = key;
        __syncthreads();
    }
}

template <class T>
__global__ void __launch_bounds__(LT) k_log_probs(LogProbArgs a) {
    __shared__ float sh[LT / 64];
    __shared__ unsigned long long best[MC_MAX_TOP], fresh[LT];
    for (int n = blockIdx.x; n < a.numCases; n += gridDim.x) {
        const T* x = static_cast<const T*>(a.logits) + (size_t)n * a.caseStride;
        float m = -INFINITY;
        for (int j = threadIdx.x; j < a.numOut; j += LT) m = fmaxf(m, (float)x[(size_t)j * a.classStride]);
        m = block_max(m, sh);
        float s = 0.f, w = 0.f;
        for (int j = threadIdx.x; j < a.numOut; j += LT) {
            const float v = (float)x[(size_t)j * a.classStride];
            const float t = v == -INFINITY ? -INFINITY : v - m;
            const float e = expf(t);
            s += e;
            w += e * fmaxf(t, -200.f);   // e is 0 there
        }
        s = block_sum(s, sh);
        w = block_sum(w, sh);
        const bool empty = s == 0.f;   // every class is ruled out
        const float logSum = empty ? 0.f : logf(s);
        if (threadIdx.x == 0) {
            if (a.maxAndLogSum) {
                a.maxAndLogSum[n] = s != s && m == -INFINITY ? s : m;
                a.maxAndLogSum[a.numCases + n] = logSum;
            }
            if (a.entropy) a.entropy[n] = empty ? 0.f : logSum - w / s;
            if (a.labelLogProbs) {
                const int y = label_of(a.labels, a.labelType, n, a.numOut);
                const float v = y < 0 ? 0.f : (float)x[(size_t)y * a.classStride];
                a.labelLogProbs[n] = y < 0 ? 0.f : v == -INFINITY && s == s ? v : (v - m) - logSum;
            }
        }
        if (a.numTop) {
            top_by_scan(x, a.classStride, a.numOut, a.numTop, best, fresh);
            if ((int)threadIdx.x < a.numTop) {
                const unsigned long long key = best[threadIdx.x];
                a.topClasses[(size_t)threadIdx.x * a.numCases + n] = key ? key_class(key) : -1;
                a.topLogProbs[(size_t)threadIdx.x * a.numCases + n] = key ? (key_logit(key) - m) - logSum : -INFINITY;
            }
            __syncthreads();
        }
    }
}

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

template <class T>
__global__ void __launch_bounds__(LT) k_log_probs_grad(LogProbGradArgs a) {
    const size_t count = (size_t)a.numCases * a.numOut;
    for (size_t i = (size_t)blockIdx.x * LT + threadIdx.x; i < count; i += (size_t)gridDim.x * LT) {
        const int n = a.classStride == 1 ? (int)(i / a.numOut) : (int)(i % a.numCases), j = a.classStride == 1 ? (int)(i % a.numOut) : (int)(i / a.numCases);
        const float m = a.maxAndLogSum[n], logSum = a.maxAndLogSum[a.numCases + n];
        const float v = (float)static_cast<const T*>(a.logits)[j * a.classStride + n * a.caseStride];
        float d = 0.f;
        if (m != -INFINITY) {
            const float lp = (v - m) - logSum, p = expf(lp);
            const int y = a.scaleLabel != 0.f ? label_of(a.labels, a.labelType, n, a.numOut) : -1;
            const float g = y >= 0 ? a.scaleLabel * (a.gradLabel ? a.gradLabel[n] : 1.f) : 0.f;
            d = (a.scaleLogZ != 0.f ? a.scaleLogZ * (a.gradLogZ ? a.gradLogZ[n] : 1.f) : 0.f) - g;
            if (a.scaleEntropy != 0.f) d -= a.scaleEntropy * (a.gradEntropy ? a.gradEntropy[n] : 1.f) * (fmaxf(lp, -200.f) + a.entropy[n]);
            d = p * d + (j == y ? g : 0.f);
        }
        T* out = static_cast<T*>(a.target) + (j * a.targetClassStride + n * a.targetCaseStride);
        *out = (T)(a.add ? (float)*out + d : d);
    }
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

}  // namespace
}  // namespace mc
using namespace mc;

extern "C" {

size_t mc_log_probs_workspace_bytes(int type, long long classStride, long long caseStride, int numCases, int numOut, int numTop) { return 0; }

int mc_log_probs(const void* logits, int type, long long classStride, long long caseStride, const void* labels, int labelType, int numCases, int numOut,
                 float* labelLogProbs, float* entropy, float* maxAndLogSum, int* topClasses, float* topLogProbs, int numTop, void* workspace,
                 size_t workspaceBytes, mcStream_t s) {
    MC_REQUIRE(numCases >= 0 && numOut > 0, "mc_log_probs: %d cases of %d classes", numCases, numOut);
    MC_REQUIRE(float_type(type), "mc_log_probs: unknown element type %d", type);
    MC_REQUIRE(numTop >= 0 && numTop <= MC_MAX_TOP, "mc_log_probs: numTop must be in [0, %d]", MC_MAX_TOP);
    if (numCases == 0) return MC_OK;
    MC_REQUIRE(logits && (size_t)logits % elem_size(type) == 0, "mc_log_probs: logits are null or not aligned to their elements");
    MC_REQUIRE(layout_kinds(classStride, caseStride, numCases, numOut), "mc_log_probs: " MC_LAYOUT_RULE);
    if (labelLogProbs) {
        const int rc = check_labels("mc_log_probs", labels, labelType, numOut);
        if (rc) return rc;
    }
    MC_REQUIRE(numTop ? topClasses && topLogProbs : !topClasses && !topLogProbs, "mc_log_probs: topClasses and topLogProbs are needed exactly where numTop > 0");
    MC_REQUIRE(labelLogProbs || entropy || maxAndLogSum || numTop, "mc_log_probs: no output asked for");
    MC_REQUIRE(stream_on_current_device(s), "mc_log_probs: the stream belongs to another device than the current one");
    const LogProbArgs a{logits, (size_t)classStride, (size_t)caseStride, labels, labelType, numCases, numOut, labelLogProbs, entropy, maxAndLogSum,
                        topClasses, topLogProbs, numTop};
    with_type(type, [&](auto t) { hipLaunchKernelGGL(k_log_probs<decltype(t)>, dim3(numCases < 65536 ? numCases : 65536), dim3(LT), 0, S(s), a); });
    return launch_status("mc_log_probs");
}

int mc_log_probs_grad(const void* logits, int type, long long classStride, long long caseStride, const void* labels, int labelType, int numCases,
                      int numOut, const float* maxAndLogSum, const float* entropy, const float* gradLabel, float scaleLabel, const float* gradEntropy,
                      float scaleEntropy, const float* gradLogZ, float scaleLogZ, void* target, long long targetClassStride,
                      long long targetCaseStride, int add, mcStream_t s) {
    MC_REQUIRE(numCases >= 0 && numOut > 0, "mc_log_probs_grad: %d cases of %d classes", numCases, numOut);
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
    const size_t want = ((size_t)numCases * numOut + LT - 1) / LT, cap = (size_t)num_cus() * 16;
    with_type(type, [&](auto t) { hipLaunchKernelGGL(k_log_probs_grad<decltype(t)>, dim3((unsigned)(want < cap ? want : cap)), dim3(LT), 0, S(s), a); });
    return launch_status("mc_log_probs_grad");
}

}  // extern "C"
