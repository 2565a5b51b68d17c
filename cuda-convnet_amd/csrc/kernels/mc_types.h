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

template <class T, int V>
__device__ __forceinline__ Pack<T, V> load_pack(const T* p) { return *reinterpret_cast<const Pack<T, V>*>(p); }
template <class T, int V>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, V>& v) { *reinterpret_cast<Pack<T, V>*>(p) = v; }

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
