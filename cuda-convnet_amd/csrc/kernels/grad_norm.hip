// grad_norm.hip -- the global norm of a list of gradient tensors, the clip factor, and the clipped gradients.
// norm^2 = sum_t sum_i (scale_t g_ti)^2: every gradient is read once and nothing else is large, so the norm is bound by HBM; clipping
// reads again what did not stay in the caches and writes.  Squares are summed in double: a float32 square overflows from |g| = 1.8e19
// on, and the double pipe keeps up with the loads (one conversion and one fma an element).
#include <math.h>
#include <string.h>
#include <algorithm>
#include <vector>
#include "mc_types.h"

namespace mc {
namespace {

constexpr int GT = 256;             // threads of a workgroup
constexpr int kMaxPartials = 2048;  // workgroups of the first pass = partial sums of the second

__device__ __forceinline__ double block_sum(double v, double* sh) {
    for (int off = 32; off > 0; off >>= 1) v += __shfl_down(v, off, 64);
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    if (lane == 0) sh[w] = v;
    __syncthreads();
    double r = 0.0;
    for (int i = 0; i < (int)blockDim.x / 64; ++i) r += sh[i];
    __syncthreads();
    return r;
}

template <class T>
__device__ __forceinline__ void add_square(double& acc, T x) {
    const double d = (double)(float)x;
    acc += d * d;
}
template <class T>
__device__ __forceinline__ double span_square(const T* g, unsigned n) {
    constexpr int V = 16 / sizeof(T), U = 8;   // U loads in flight a thread
    double acc[2] = {0.0, 0.0};
    unsigned i = 0;
    for (; i + GT * V * U <= n; i += GT * V * U) {
        Pack<T, V> x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) x[u] = load_pack<T, V>(g + i + (u * GT + threadIdx.x) * V);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int k = 0; k < V; ++k) add_square(acc[k & 1], x[u].v[k]);
    }
    for (; i + GT * V <= n; i += GT * V) {
        const Pack<T, V> x = load_pack<T, V>(g + i + threadIdx.x * V);
#pragma unroll
        for (int k = 0; k < V; ++k) add_square(acc[k & 1], x.v[k]);
    }
    for (i += threadIdx.x; i < n; i += GT) add_square(acc[0], g[i]);
    return acc[0] + acc[1];
}

__global__ void __launch_bounds__(GT) k_grad_square(const mcGradSpan* __restrict__ spans, int numSpans, double* __restrict__ partials) {
    __shared__ double sh[GT / 64];
    double acc = 0.0;
    mcGradSpan sp = spans[blockIdx.x];
    for (int b = blockIdx.x; b < numSpans; b += gridDim.x) {
        const mcGradSpan next = spans[min(b + (int)gridDim.x, numSpans - 1)];   // its way to memory is as long as a gradient's
        double s = 0.0;
        if (sp.gradType == MC_F32) s = span_square(static_cast<const float*>(sp.grad), sp.count);
        else if (sp.gradType == MC_F16) s = span_square(static_cast<const _Float16*>(sp.grad), sp.count);
        else s = span_square(static_cast<const __bf16*>(sp.grad), sp.count);
        acc += s * ((double)sp.scale * (double)sp.scale);
        sp = next;
    }
    acc = block_sum(acc, sh);
    if (threadIdx.x == 0) partials[blockIdx.x] = acc;
}

__global__ void __launch_bounds__(GT) k_grad_factor(const double* __restrict__ partials, int n, float maxNorm, float* __restrict__ out) {
    __shared__ double sh[GT / 64];
    double acc = 0.0;
    for (int i = threadIdx.x; i < n; i += GT) acc += partials[i];
    acc = block_sum(acc, sh);
    if (threadIdx.x == 0) {
        const double norm = sqrt(acc);
        const float f = (float)norm;
        out[0] = f;
        // a finite norm never gives factor 0, which means "drop the step"
        out[1] = isfinite(f) ? (norm > (double)maxNorm ? fmaxf((float)((double)maxNorm / norm), 1.40129846e-45f) : 1.f) : 0.f;
    }
}

template <class T, class O>
__device__ __forceinline__ void span_scale(const T* g, O* out, unsigned n, float f) {
    constexpr int V = 16 / (sizeof(T) > sizeof(O) ? sizeof(T) : sizeof(O)), U = 4;
    unsigned i = 0;
    for (; i + GT * V * U <= n; i += GT * V * U) {
        Pack<T, V> x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) x[u] = load_pack<T, V>(g + i + (u * GT + threadIdx.x) * V);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            Pack<O, V> y;
#pragma unroll
            for (int k = 0; k < V; ++k) y.v[k] = (O)((float)x[u].v[k] * f);
            store_pack<O, V>(out + i + (u * GT + threadIdx.x) * V, y);
        }
    }
    for (i += threadIdx.x; i < n; i += GT) out[i] = (O)((float)g[i] * f);
}
template <class O>
__device__ __forceinline__ void span_zero(O* out, unsigned n) {
    for (unsigned i = threadIdx.x; i < n; i += GT) out[i] = (O)0.f;
}
template <class T>
__device__ __forceinline__ void span_clip(const mcGradSpan& sp, float factor) {
    const T* g = static_cast<const T*>(sp.grad);
    const float f = factor * sp.scale;
    if (sp.outType == MC_F32) span_scale(g, static_cast<float*>(sp.out), sp.count, f);
    else if (sp.outType == MC_F16) span_scale(g, static_cast<_Float16*>(sp.out), sp.count, f);
    else span_scale(g, static_cast<__bf16*>(sp.out), sp.count, f);
}

__global__ void __launch_bounds__(GT) k_clip_grads(const mcGradSpan* __restrict__ spans, int numSpans, const float* __restrict__ normAndFactor) {
    const float factor = normAndFactor[1];
    mcGradSpan next = spans[numSpans - 1 - blockIdx.x];
    for (int b = blockIdx.x; b < numSpans; b += gridDim.x) {   // (from the end: what the norm read last is still in the caches)
        const mcGradSpan sp = next;
        next = spans[max(numSpans - 1 - b - (int)gridDim.x, 0)];
        if (!sp.out || (sp.out == sp.grad && factor * sp.scale == 1.f)) continue;
        if (factor == 0.f) {   // not a product: the gradients hold what made the norm infinite
            if (sp.outType == MC_F32) span_zero(static_cast<float*>(sp.out), sp.count);
            else span_zero(static_cast<_Float16*>(sp.out), sp.count);
        } else if (sp.gradType == MC_F32) span_clip<float>(sp, factor);
        else if (sp.gradType == MC_F16) span_clip<_Float16>(sp, factor);
        else span_clip<__bf16>(sp, factor);
    }
}

// inc = mom*inc + factor*grad; inc += wceps*W; W += inc, in the order (and, at factor 1, with the bits) of mc_weights_update_spans.
__device__ __forceinline__ void step(float& w, float& i, float g, float f, float mom, float wceps) {
    i = fmaf(mom, i, f * g);
    if (wceps != 0.f) i = fmaf(wceps, w, i);
    w += i;
}
__global__ void __launch_bounds__(GT) k_weights_update_clipped(float* w, float* inc, const float* __restrict__ grad, const mcUpdateSpan* __restrict__ spans,
                                                               int numSpans, const float* __restrict__ normAndFactor) {
    const float f = normAndFactor[1];
    if (f == 0.f) return;   // the norm is not finite: the step is dropped
    mcUpdateSpan next = spans[numSpans - 1 - blockIdx.x];
    for (int b = blockIdx.x; b < numSpans; b += gridDim.x) {   // (from the end, as above)
        const mcUpdateSpan sp = next;
        next = spans[max(numSpans - 1 - b - (int)gridDim.x, 0)];
        float *W = w + sp.start, *I = inc + sp.start;
        const float* G = grad + sp.start;
        constexpr int U = 4;
        unsigned v = 0;
        for (; v + GT * 4 * U <= sp.count; v += GT * 4 * U) {
            Pack<float, 4> ww[U], ii[U], gg[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const unsigned at = v + (u * GT + threadIdx.x) * 4;
                ww[u] = load_pack<float, 4>(W + at);
                ii[u] = load_pack<float, 4>(I + at);
                gg[u] = load_pack<float, 4>(G + at);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const unsigned at = v + (u * GT + threadIdx.x) * 4;
#pragma unroll
                for (int k = 0; k < 4; ++k) step(ww[u].v[k], ii[u].v[k], gg[u].v[k], f, sp.mom, sp.wceps);
                store_pack<float, 4>(I + at, ii[u]);
                store_pack<float, 4>(W + at, ww[u]);
            }
        }
        for (v += threadIdx.x; v < sp.count; v += GT) step(W[v], I[v], G[v], f, sp.mom, sp.wceps);
    }
}

int partials_for(int numSpans) { return std::max(1, std::min(numSpans, kMaxPartials)); }

struct Range { size_t lo, hi; bool out; };

// Whether something that is written overlaps anything else (gradients alone may: a shared one counts as often as it is listed).
bool ranges_clash(std::vector<Range>& r) {
    std::sort(r.begin(), r.end(), [](const Range& a, const Range& b) { return a.lo < b.lo; });
    size_t outHi = 0, anyHi = 0;
    for (const Range& x : r) {
        if (x.lo < (x.out ? anyHi : outHi)) return true;
        anyHi = std::max(anyHi, x.hi);
        if (x.out) outHi = std::max(outHi, x.hi);
    }
    return false;
}

}  // namespace
}  // namespace mc
using namespace mc;

extern "C" {

int mc_grad_spans(const mcGradTensor* tensors, int numTensors, mcGradSpan* spans, int maxSpans, int* numSpans) {
    MC_REQUIRE(numSpans && numTensors >= 0 && (tensors || numTensors == 0), "mc_grad_spans: bad arguments");
    *numSpans = 0;
    try {
        unsigned long long total = 0;
        std::vector<Range> ranges;
        for (int i = 0; i < numTensors; ++i) {
            const mcGradTensor& t = tensors[i];
            MC_REQUIRE(float_type(t.gradType) && float_type(t.outType), "mc_grad_spans: tensor %d: unknown element type", i);
            MC_REQUIRE(isfinite(t.scale), "mc_grad_spans: tensor %d: scale is not finite", i);
            if (t.count == 0) continue;
            MC_REQUIRE(t.grad, "mc_grad_spans: tensor %d: null gradient", i);
            MC_REQUIRE(t.count <= (1ull << 48), "mc_grad_spans: tensor %d: %llu elements", i, t.count);
            const size_t gs = elem_size(t.gradType), os = elem_size(t.outType);
            MC_REQUIRE((size_t)t.grad % gs == 0 && (size_t)t.out % os == 0, "mc_grad_spans: tensor %d is not aligned to its elements", i);
            MC_REQUIRE(t.out != t.grad || t.gradType == t.outType, "mc_grad_spans: tensor %d: in place needs one element type", i);
            ranges.push_back({(size_t)t.grad, (size_t)t.grad + t.count * gs, t.out == t.grad});
            if (t.out && t.out != t.grad) ranges.push_back({(size_t)t.out, (size_t)t.out + t.count * os, true});
            total += t.count;
        }
        MC_REQUIRE(!ranges_clash(ranges), "mc_grad_spans: an output overlaps another output or gradient");
        // Spans of a power of two elements: at least 4096 (a span's descriptor and its workgroup cost then less than its bytes), and about
        // 8192 spans in all, four rounds of the first pass's workgroups, so that a large list's last round is short.
        unsigned long long per = 4096;
        while (per < 65536 && per * 8192 < total) per *= 2;
        unsigned long long n = 0;
        for (int i = 0; i < numTensors; ++i) n += (tensors[i].count + per - 1) / per;
        MC_REQUIRE(n <= 0x7fffffffull, "mc_grad_spans: too many elements");
        *numSpans = (int)n;
        if (!spans) return MC_OK;
        MC_REQUIRE((unsigned long long)std::max(maxSpans, 0) >= n, "mc_grad_spans: %llu spans, room for %d", n, maxSpans);
        int at = 0;
        for (int i = 0; i < numTensors; ++i) {
            const mcGradTensor& t = tensors[i];
            for (unsigned long long done = 0; done < t.count; done += per) {
                mcGradSpan sp;
                sp.grad = static_cast<const char*>(t.grad) + done * elem_size(t.gradType);
                sp.out = t.out ? static_cast<char*>(t.out) + done * elem_size(t.outType) : nullptr;
                sp.count = (unsigned)std::min(per, t.count - done);
                sp.scale = t.scale;
                sp.gradType = t.gradType;
                sp.outType = t.outType;
                spans[at++] = sp;
            }
        }
    } catch (const std::exception& e) {
        set_error("mc_grad_spans: %s", e.what());
        return MC_EINVAL;
    }
    return MC_OK;
}

size_t mc_grad_norm_workspace_bytes(int numSpans) { return (size_t)partials_for(numSpans) * sizeof(double); }

int mc_grad_norm(const mcGradSpan* spansDevice, int numSpans, float maxNorm, float* normAndFactor, void* workspace, size_t workspaceBytes,
                 mcStream_t s) {
    MC_REQUIRE(normAndFactor && numSpans >= 0 && (spansDevice || numSpans == 0), "mc_grad_norm: bad arguments");
    MC_REQUIRE(maxNorm > 0.f, "mc_grad_norm: maxNorm must be positive");
    MC_REQUIRE(stream_on_current_device(s), "mc_grad_norm: the stream belongs to another device than the current one");
    if (!workspace || workspaceBytes < mc_grad_norm_workspace_bytes(numSpans) || !aligned16(workspace)) {
        set_error("mc_grad_norm: workspace of %zu bytes, 16-byte aligned, needed", mc_grad_norm_workspace_bytes(numSpans));
        return MC_EWORKSPACE;
    }
    double* partials = static_cast<double*>(workspace);
    const int n = numSpans ? partials_for(numSpans) : 0;
    if (n) hipLaunchKernelGGL(k_grad_square, dim3(n), dim3(GT), 0, S(s), spansDevice, numSpans, partials);
    hipLaunchKernelGGL(k_grad_factor, dim3(1), dim3(GT), 0, S(s), partials, n, maxNorm, normAndFactor);
    return launch_status("mc_grad_norm");
}

int mc_clip_grads(const mcGradSpan* spansDevice, int numSpans, const float* normAndFactor, mcStream_t s) {
    MC_REQUIRE(normAndFactor && numSpans >= 0 && (spansDevice || numSpans == 0), "mc_clip_grads: bad arguments");
    MC_REQUIRE(stream_on_current_device(s), "mc_clip_grads: the stream belongs to another device than the current one");
    if (numSpans == 0) return MC_OK;
    hipLaunchKernelGGL(k_clip_grads, dim3(std::min(numSpans, 8 * num_cus())), dim3(GT), 0, S(s), spansDevice, numSpans, normAndFactor);
    return launch_status("mc_clip_grads");
}

int mc_weights_update_spans_clipped(float* weights, float* inc, const float* grad, const mcUpdateSpan* spansDevice, int numSpans, const float* normAndFactor,
                                    mcStream_t s) {
    MC_REQUIRE(weights && inc && grad && spansDevice && normAndFactor, "mc_weights_update_spans_clipped: null pointer");
    MC_REQUIRE(aligned16(weights) && aligned16(inc) && aligned16(grad), "mc_weights_update_spans_clipped: arenas must be 16-byte aligned");
    MC_REQUIRE(stream_on_current_device(s), "mc_weights_update_spans_clipped: the stream belongs to another device than the current one");
    if (numSpans <= 0) return MC_OK;
    hipLaunchKernelGGL(k_weights_update_clipped, dim3(std::min(numSpans, 8 * num_cus())), dim3(GT), 0, S(s), weights, inc, grad, spansDevice, numSpans,
                       normAndFactor);
    return launch_status("mc_weights_update_spans_clipped");
}

}  // extern "C"
