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
constexpr int kSpan = 4096;         // elements of a span, at most
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

// The squares of a pack.  Those of 16-bit numbers are exact in float32, and a tree of 8 of them is off by at most 3 half steps there: one
// conversion to double for the pack, where the double pipe would take longer than the loads (2^28 bf16: 114 us in double throughout).
// bf16 has float32's range, though: where the sum is infinite or might have lost bits below, doubles form it.
template <class T, int V>
__device__ __forceinline__ double pack_square(const Words<T, V>& x, Pass pass) {
    if constexpr (sizeof(T) == 2) {
        float p[V / 2];
#pragma unroll
        for (int k = 0; k < V / 2; ++k) {
            const float a = x.at(2 * k, pass), b = x.at(2 * k + 1, pass);
            p[k] = fmaf(b, b, a * a);
        }
#pragma unroll
        for (int n = V / 4; n > 0; n /= 2)
#pragma unroll
            for (int k = 0; k < n; ++k) p[k] += p[k + n];
        if (!__is_same(T, __bf16) || (p[0] > 0x1p-80f && p[0] < INFINITY)) return (double)p[0];
    }
    double s = 0.0;
#pragma unroll
    for (int k = 0; k < V; ++k) {
        const double d = (double)x.at(k, pass);
        s += d * d;
    }
    return s;
}

// The packs of a span, U loads in flight a thread: past the end the last pack is loaded again and not counted.
template <class T, bool NT>
__device__ __forceinline__ double span_square(const T* g, unsigned n) {
    constexpr int V = 16 / sizeof(T), U = 4;
    const unsigned packs = n / V;
    double acc = 0.0;
    for (unsigned at = threadIdx.x; at - threadIdx.x < packs; at += GT * U) {
        Words<T, V> x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) x[u].template load<NT>(g + min(at + u * GT, packs - 1) * V);
        const Pass pass;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const double s = pack_square(x[u], pass);
            acc += at + u * GT < packs ? s : 0.0;
            asm volatile("" : "+v"(acc));   // one pack's doubles in registers at a time
        }
    }
    if (threadIdx.x < n - packs * V) {
        const double d = (double)(float)load_pack<NT, T, 1>(g + packs * V + threadIdx.x).v[0];
        acc += d * d;
    }
    return acc;
}
template <class T>
__device__ __forceinline__ double span_square(const mcGradSpan& sp, bool nt) {
    const T* g = static_cast<const T*>(sp.grad);
    return nt ? span_square<T, true>(g, sp.count) : span_square<T, false>(g, sp.count);
}

// One read of every gradient, bound by HBM: 2^28 bf16 in 300 tensors 87 us (6.2 TB/s), 2^27 f32 in 120 82 (6.6).  (16-bit numbers: the vector
// units are nearly as busy.)  As many workgroups as the second pass can add up in one go, each over spans a grid apart.
__global__ void __launch_bounds__(GT) k_grad_square(const mcGradSpan* __restrict__ spans, int numSpans, double* __restrict__ partials, bool nt) {
    __shared__ double sh[GT / 64];
    double acc = 0.0;
    mcGradSpan sp = spans[blockIdx.x];
    for (int b = blockIdx.x; b < numSpans; b += gridDim.x) {
        const mcGradSpan next = spans[min(b + (int)gridDim.x, numSpans - 1)];   // its way to memory is as long as a gradient's
        double s = 0.0;
        if (sp.gradType == MC_F32) s = span_square<float>(sp, nt);
        else if (sp.gradType == MC_F16) s = span_square<_Float16>(sp, nt);
        else s = span_square<__bf16>(sp, nt);
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

// kClipPacks packs of 4 elements a thread: a workgroup takes a part of a span.  (Streams of small tiles in the order of memory copy faster
// than workgroups that walk through stretches of their own.)  2^28 bf16 into f32 (1.6 GB) 267 us, 6.0 TB/s.
constexpr int kClipPacks = 2, kClipTile = GT * 4 * kClipPacks;
template <bool NT, class T, class O>
__device__ __forceinline__ void tile_scale(const T* g, O* out, unsigned at, unsigned n, float f) {
    at += threadIdx.x * 4;
    Pack<T, 4> x[kClipPacks];
#pragma unroll
    for (int u = 0; u < kClipPacks; ++u)
        if (at + u * GT * 4 + 4 <= n) x[u] = load_pack<NT, T, 4>(g + at + u * GT * 4);
#pragma unroll
    for (int u = 0; u < kClipPacks; ++u) {
        unsigned j = at + u * GT * 4;
        if (j + 4 <= n) {
            Pack<O, 4> y;
#pragma unroll
            for (int k = 0; k < 4; ++k) y.v[k] = f == 0.f ? (O)0.f : (O)((float)x[u].v[k] * f);
            store_pack<NT, O, 4>(out + j, y);
        } else
            for (; j < n; ++j) {
                const float v = (float)load_pack<false, T, 1>(g + j).v[0];
                Pack<O, 1> y;
                y.v[0] = f == 0.f ? (O)0.f : (O)(v * f);
                store_pack<false, O, 1>(out + j, y);
            }
    }
}
template <bool NT, class T>
__device__ __forceinline__ void tile_clip(const mcGradSpan& sp, unsigned at, float f) {
    const T* g = static_cast<const T*>(sp.grad);
    if (sp.outType == MC_F32) tile_scale<NT>(g, static_cast<float*>(sp.out), at, sp.count, f);
    else if (sp.outType == MC_F16) tile_scale<NT>(g, static_cast<_Float16*>(sp.out), at, sp.count, f);
    else tile_scale<NT>(g, static_cast<__bf16*>(sp.out), at, sp.count, f);
}

// Factor 0 writes zeros and not products: the gradients hold what made the norm infinite.
template <bool NT>
__global__ void __launch_bounds__(GT) k_clip_grads(const mcGradSpan* __restrict__ spans, const float* __restrict__ normAndFactor) {
    const mcGradSpan sp = spans[blockIdx.x / (kSpan / kClipTile)];
    const unsigned at = blockIdx.x % (kSpan / kClipTile) * kClipTile;
    if (at >= sp.count || !sp.out) return;
    const float f = normAndFactor[1] == 0.f ? 0.f : normAndFactor[1] * sp.scale;
    if (sp.out == sp.grad && f == 1.f) return;
    if (sp.gradType == MC_F32) tile_clip<NT, float>(sp, at, f);
    else if (sp.gradType == MC_F16) tile_clip<NT, _Float16>(sp, at, f);
    else tile_clip<NT, __bf16>(sp, at, f);
}

// inc = mom*inc + factor*grad; inc += wceps*W; W += inc, in the order (and, at factor 1, with the bits) of mc_weights_update_spans.
__device__ __forceinline__ void step(float& w, float& i, float g, float f, float mom, float wceps) {
    i = fmaf(mom, i, f * g);
    if (wceps != 0.f) i = fmaf(wceps, w, i);
    w += i;
}
// A workgroup takes a span, with up to 12 loads in flight a thread.  Three reads and two writes of HBM: 2^27 weights (2.7 GB) 469 us, 5.7 TB/s.
template <bool NT>
__global__ void __launch_bounds__(GT) __attribute__((amdgpu_waves_per_eu(8)))
k_weights_update_clipped(float* w, float* inc, const float* __restrict__ grad, const mcUpdateSpan* __restrict__ spans, const float* __restrict__ normAndFactor) {
    const mcUpdateSpan sp = spans[blockIdx.x];
    const float f = normAndFactor[1];
    if (f == 0.f) return;   // the norm is not finite: the step is dropped
    float *W = w + sp.start, *I = inc + sp.start;
    const float* G = grad + sp.start;
    constexpr int U = 4;
    const unsigned packs = sp.count / 4;
    for (unsigned at = threadIdx.x; at - threadIdx.x < packs; at += GT * U) {   // past the end the last pack is loaded again, and not stored
        Words<float, 4> ww[U], ii[U], gg[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const unsigned j = min(at + u * GT, packs - 1) * 4;
            ww[u].load<NT>(W + j);
            ii[u].load<NT>(I + j);
            gg[u].load<NT>(G + j);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            Pack<float, 4> nw, ni;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                nw.v[k] = __uint_as_float(ww[u].w[k]);
                ni.v[k] = __uint_as_float(ii[u].w[k]);
                step(nw.v[k], ni.v[k], __uint_as_float(gg[u].w[k]), f, sp.mom, sp.wceps);
            }
            if (at + u * GT < packs) {
                store_pack<NT, float, 4>(I + (at + u * GT) * 4, ni);
                store_pack<NT, float, 4>(W + (at + u * GT) * 4, nw);
            }
        }
    }
    const unsigned rest = packs * 4 + threadIdx.x;
    if (rest < sp.count) step(W[rest], I[rest], G[rest], f, sp.mom, sp.wceps);
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
        }
        MC_REQUIRE(!ranges_clash(ranges), "mc_grad_spans: an output overlaps another output or gradient");
        // Spans of kSpan elements, cut so that all but a tensor's first begin on a 128-byte line of what is written (of what is read, where
        // nothing is): lines that two workgroups write in halves cost a fifth of the copy's time.
        unsigned long long n = 0;
        for (int i = 0; i < numTensors; ++i) {
            const mcGradTensor& t = tensors[i];
            for (unsigned long long done = 0; done < t.count;) {
                mcGradSpan sp;
                sp.grad = static_cast<const char*>(t.grad) + done * elem_size(t.gradType);
                sp.out = t.out ? static_cast<char*>(t.out) + done * elem_size(t.outType) : nullptr;
                const unsigned past = sp.out ? (size_t)sp.out % 128 / elem_size(t.outType) : (size_t)sp.grad % 128 / elem_size(t.gradType);
                sp.count = (unsigned)std::min<unsigned long long>(kSpan - past, t.count - done);
                sp.scale = t.scale;
                sp.gradType = t.gradType;
                sp.outType = t.outType;
                if (spans && n < (unsigned long long)std::max(maxSpans, 0)) spans[n] = sp;
                ++n;
                done += sp.count;
                MC_REQUIRE(fits_a_grid(n * (kSpan / kClipTile), GT), "mc_grad_spans: too many elements");
            }
        }
        *numSpans = (int)n;
        MC_REQUIRE(!spans || (unsigned long long)std::max(maxSpans, 0) >= n, "mc_grad_spans: %llu spans, room for %d", n, maxSpans);
    } catch (const std::exception& e) {
        set_error("mc_grad_spans: %s", e.what());
        return MC_EINVAL;
    }
    return MC_OK;
}

// Spans are nearly all of kSpan elements where there are so many that streaming pays, and what a step touches besides the gradients is
// about as much again (norm and update after a pass that wrote the gradients: 2^24 elements 87 us without and 92 with nt, 2^25 187 and 173).
static bool spans_stream(int numSpans) { return streams((size_t)numSpans * kSpan * 8); }

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
    if (n) hipLaunchKernelGGL(k_grad_square, dim3(n), dim3(GT), 0, S(s), spansDevice, numSpans, partials, spans_stream(numSpans));
    hipLaunchKernelGGL(k_grad_factor, dim3(1), dim3(GT), 0, S(s), partials, n, maxNorm, normAndFactor);
    return launch_status("mc_grad_norm");
}

int mc_clip_grads(const mcGradSpan* spansDevice, int numSpans, const float* normAndFactor, mcStream_t s) {
    MC_REQUIRE(normAndFactor && numSpans >= 0 && (spansDevice || numSpans == 0), "mc_clip_grads: bad arguments");
    MC_REQUIRE(stream_on_current_device(s), "mc_clip_grads: the stream belongs to another device than the current one");
    if (numSpans == 0) return MC_OK;
    MC_REQUIRE(fits_a_grid((size_t)numSpans * (kSpan / kClipTile), GT), "mc_clip_grads: too many spans");
    const dim3 grid(numSpans * (kSpan / kClipTile)), block(GT);
    if (spans_stream(numSpans)) hipLaunchKernelGGL(k_clip_grads<true>, grid, block, 0, S(s), spansDevice, normAndFactor);
    else hipLaunchKernelGGL(k_clip_grads<false>, grid, block, 0, S(s), spansDevice, normAndFactor);
    return launch_status("mc_clip_grads");
}

int mc_weights_update_spans_clipped(float* weights, float* inc, const float* grad, const mcUpdateSpan* spansDevice, int numSpans, const float* normAndFactor,
                                    mcStream_t s) {
    MC_REQUIRE(weights && inc && grad && spansDevice && normAndFactor, "mc_weights_update_spans_clipped: null pointer");
    MC_REQUIRE(aligned16(weights) && aligned16(inc) && aligned16(grad), "mc_weights_update_spans_clipped: arenas must be 16-byte aligned");
    MC_REQUIRE(stream_on_current_device(s), "mc_weights_update_spans_clipped: the stream belongs to another device than the current one");
    if (numSpans <= 0) return MC_OK;
    MC_REQUIRE(fits_a_grid(numSpans, GT), "mc_weights_update_spans_clipped: too many spans");
    if (spans_stream(numSpans)) hipLaunchKernelGGL(k_weights_update_clipped<true>, dim3(numSpans), dim3(GT), 0, S(s), weights, inc, grad, spansDevice, normAndFactor);
    else hipLaunchKernelGGL(k_weights_update_clipped<false>, dim3(numSpans), dim3(GT), 0, S(s), weights, inc, grad, spansDevice, normAndFactor);
    return launch_status("mc_weights_update_spans_clipped");
}

}  // extern "C"
