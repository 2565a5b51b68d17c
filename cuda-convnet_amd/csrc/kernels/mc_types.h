// Element types of the entry points that take one (MC_F32 / MC_F16 / MC_BF16): vectors of them that need no more than an
// element's alignment (the hardware takes 16-byte global accesses at any element address), and conversions.
#pragma once
#include "mc_common.h"

namespace mc {

// A pointer that was itself loaded from memory, as one to global memory (the compiler would use flat accesses, which wait for the
// scalar loads beside them).
template <class T>
using GlobalPtr = __attribute__((address_space(1))) T*;

inline int elem_size(int type) { return type == MC_F32 ? 4 : 2; }
inline bool float_type(int type) { return type == MC_F32 || type == MC_F16 || type == MC_BF16; }

// V elements, aligned like one of them
template <class T, int V>
struct __attribute__((packed, aligned(sizeof(T)))) Pack { T v[V]; };

template <int BYTES, int ALIGN>
struct Raw;   // BYTES bytes as a register vector, at any address that is a multiple of ALIGN (2 or 4)
template <> struct Raw<16, 4> { typedef unsigned type __attribute__((ext_vector_type(4), aligned(4))); };
template <> struct Raw<16, 2> { typedef unsigned type __attribute__((ext_vector_type(4), aligned(2))); };
template <> struct Raw<8, 4> { typedef unsigned type __attribute__((ext_vector_type(2), aligned(4))); };
template <> struct Raw<8, 2> { typedef unsigned type __attribute__((ext_vector_type(2), aligned(2))); };
template <> struct Raw<4, 4> { typedef unsigned type; };
template <> struct Raw<4, 2> { typedef unsigned type __attribute__((aligned(2))); };
template <> struct Raw<2, 2> { typedef unsigned short type; };

// Streaming accesses (nt) keep data that is read or written once, and is larger than the caches, from displacing the rest and itself: on
// 512 MiB reads reach 6.9 TB/s against 6.3 with ordinary loads, copies 6.2 against 5.8.  Data that fits the 256 MiB last-level cache is
// better left to it: what the kernel before wrote is still there, and the kernel after finds what this one leaves.  Logits written, read
// for the log probabilities, replaced by their gradient and read again: 154 us without and 169 with nt at 134 MB, 347 and 333 at 268 MB.
inline bool streams(size_t bytes) { return bytes > ((size_t)192 << 20); }

// (NT is a template parameter throughout: of two branches that differ in the hint alone the compiler makes one without it.)
template <bool NT, class T, int V>
__device__ __forceinline__ Pack<T, V> load_pack(const T* p) {
    typedef typename Raw<sizeof(T) * V, sizeof(T)>::type R;
    const GlobalPtr<const R> q = (GlobalPtr<const R>)p;
    const R r = NT ? __builtin_nontemporal_load(q) : *q;
    Pack<T, V> v;
    __builtin_memcpy(&v, &r, sizeof(v));
    return v;
}
template <bool NT, class T, int V>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, V>& v) {
    typedef typename Raw<sizeof(T) * V, sizeof(T)>::type R;
    R r;
    __builtin_memcpy(&r, &v, sizeof(v));
    if (NT) __builtin_nontemporal_store(r, (GlobalPtr<R>)p);
    else *(GlobalPtr<R>)p = r;
}

// Elements stay in the registers that they were loaded into and are converted where they are used.  A Pass holds the constants that
// takes, anew for each pass over them and hidden from the compiler, which would hold the converted values from one pass to the next
// otherwise: twice the registers for 16-bit types.
struct Pass {
    unsigned high = 0xffff0000u, by = 16;
    __device__ __forceinline__ Pass() { asm volatile("" : "+s"(high), "+s"(by)); }
};
// N elements of type T
template <class T, int N>
struct Words {
    static constexpr int COUNT = N * sizeof(T) < 4 ? 1 : N * sizeof(T) / 4;
    unsigned w[COUNT];
    template <bool NT>
    __device__ __forceinline__ void load(const T* p) {
        typedef typename Raw<N * sizeof(T), sizeof(T)>::type R;
        const GlobalPtr<const R> q = (GlobalPtr<const R>)p;
        const R r = NT ? __builtin_nontemporal_load(q) : *q;
        w[0] = 0;
        __builtin_memcpy(w, &r, N * sizeof(T));
    }
    __device__ __forceinline__ void fill() {   // -inf
        const unsigned inf = sizeof(T) == 4 ? 0xff800000u : __is_same(T, _Float16) ? 0xfc00fc00u : 0xff80ff80u;
#pragma unroll
        for (int i = 0; i < COUNT; ++i) w[i] = inf;
    }
    __device__ __forceinline__ void fill_first(int n) {   // -inf in the first n of them
        const unsigned inf = sizeof(T) == 4 ? 0xff800000u : __is_same(T, _Float16) ? 0xfc00fc00u : 0xff80ff80u;
        constexpr int PER = sizeof(T) == 4 ? 1 : 2;
#pragma unroll
        for (int i = 0; i < COUNT; ++i) {
            if (PER == 2 && n == 2 * i + 1) w[i] = (w[i] & 0xffff0000u) | (inf & 0xffffu);
            if (n >= PER * (i + 1)) w[i] = inf;
        }
    }
    __device__ __forceinline__ void set(int k, T v) {
        unsigned short h = 0;
        if (sizeof(T) == 4) {
            __builtin_memcpy(&w[k], &v, sizeof(T));
            return;
        }
        __builtin_memcpy(&h, &v, 2);
        w[k / 2] = k % 2 ? (w[k / 2] & 0xffffu) | (unsigned)h << 16 : (w[k / 2] & 0xffff0000u) | h;
    }
    __device__ __forceinline__ float at(int k, Pass p) const {
        if (sizeof(T) == 4) return __uint_as_float(w[k]);
        const unsigned u = w[k / 2];
        if (__is_same(T, __bf16)) return __uint_as_float(k % 2 ? u & p.high : u << p.by);
        const unsigned short h = (unsigned short)(k % 2 ? u >> p.by : u);
        _Float16 v;
        __builtin_memcpy(&v, &h, 2);
        return (float)v;
    }
};

// Calls f with a value of the element type that `type` names; false if it names none.
template <class F>
inline bool with_type(int type, F f) {
    switch (type) {
        case MC_F32: f(float()); return true;
        case MC_F16: f(_Float16()); return true;
        case MC_BF16: f(__bf16()); return true;
    }
    return false;
}

// A launch counts its threads in 32 bits.
inline bool fits_a_grid(size_t blocks, int threads) { return blocks <= 0xffffffffu / (unsigned)threads; }

// The stream a call names must belong to the current device: every pointer is taken to live there, and grids are sized for it.
// Where the runtime cannot tell, the launch says; the error of asking is not left for launch_status to find (one that was there before is).
inline bool stream_on_current_device(mcStream_t s) {
    if (!s) return true;
    int dev = 0;
    hipDevice_t of = 0;
    const bool clean = hipPeekAtLastError() == hipSuccess;
    if (hipGetDevice(&dev) == hipSuccess && hipStreamGetDevice(S(s), &of) == hipSuccess) return dev == (int)of;
    if (clean) (void)hipGetLastError();
    return true;
}

}  // namespace mc
