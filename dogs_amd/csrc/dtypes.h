// dtypes.h -- the element types of the tensor operators (DG_F32 / DG_F16 / DG_BF16) and their 16-byte vectors.
#pragma once
#include <stdint.h>

namespace gs {

template <int DT> struct Elem;
template <> struct Elem<0> { typedef float T; };
template <> struct Elem<1> { typedef _Float16 T; };
template <> struct Elem<2> { typedef __bf16 T; };

// 16 bytes of T at any multiple of sizeof(T): rows of an odd width and slices of a larger tensor start at no aligned
// place, and the global path of gfx950 takes dword loads and stores at any address (unaligned access mode)
template <typename T> struct Vec {
    static constexpr int W = 16 / (int)sizeof(T);
    typedef T type __attribute__((ext_vector_type(W), aligned(sizeof(T))));
};

inline uint32_t elem_bytes(int dtype) { return dtype == 0 ? 4u : 2u; }

}  // namespace gs
