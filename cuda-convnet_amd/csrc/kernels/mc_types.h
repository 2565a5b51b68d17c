// Element types of the entry points that take one (MC_F32 / MC_F16 / MC_BF16): vectors of them that need no more than an
// element's alignment (the hardware takes 16-byte global accesses at any element address), and conversions.
#pragma once
#include "mc_common.h"

namespace mc {

inline int elem_size(int type) { return type == MC_F32 ? 4 : 2; }
inline bool float_type(int type) { return type == MC_F32 || type == MC_F16 || type == MC_BF16; }

// V elements, aligned like one of them
template <class T, int V>
struct __attribute__((packed, aligned(sizeof(T)))) Pack { T v[V]; };

// Streaming accesses: data that is read or written once and is larger than the caches.  (On 512 MiB: reads 6.9 TB/s against 6.3 with
// ordinary loads, copies 6.2 against 5.8.)
template <int BYTES, int ALIGN>
struct Raw;   // BYTES bytes as a register vector, at any address that is a multiple of ALIGN (2 or 4)
template <> struct Raw<16, 4> { typedef unsigned type __attribute__((ext_vector_type(4), aligned(4))); };
template <> struct Raw<16, 2> { typedef unsigned type __attribute__((ext_vector_type(4), aligned(2))); };
template <> struct Raw<8, 4> { typedef unsigned type __attribute__((ext_vector_type(2), aligned(4))); };
template <> struct Raw<8, 2> { typedef unsigned type __attribute__((ext_vector_type(2), aligned(2))); };
template <> struct Raw<4, 4> { typedef unsigned type; };
template <> struct Raw<4, 2> { typedef unsigned type __attribute__((aligned(2))); };
template <> struct Raw<2, 2> { typedef unsigned short type; };

template <class T, int V>
__device__ __forceinline__ Pack<T, V> load_pack(const T* p) {
    typedef typename Raw<sizeof(T) * V, sizeof(T)>::type R;
    const R r = __builtin_nontemporal_load(reinterpret_cast<const R*>(p));
    Pack<T, V> v;
    __builtin_memcpy(&v, &r, sizeof(v));
    return v;
}
template <class T, int V>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, V>& v) {
    typedef typename Raw<sizeof(T) * V, sizeof(T)>::type R;
    R r;
    __builtin_memcpy(&r, &v, sizeof(v));
    __builtin_nontemporal_store(r, reinterpret_cast<R*>(p));
}

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

// The stream a call names must belong to the current device: every pointer is taken to live there, and grids are sized for it.
inline bool stream_on_current_device(mcStream_t s) {
    if (!s) return true;
    int dev = 0;
    hipDevice_t of = 0;
    if (hipGetDevice(&dev) != hipSuccess || hipStreamGetDevice(S(s), &of) != hipSuccess) return true;   // cannot tell: the launch says
    return dev == (int)of;
}

}  // namespace mc
