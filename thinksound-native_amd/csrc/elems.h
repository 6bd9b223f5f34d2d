// elems.h — element types of the block operators: f32, f16 and bf16 rows as floats, and host checks
// that two strided row windows share no element.
#pragma once
#include <numeric>

#include "tsn_common.h"

namespace tsn {

typedef __bf16 bf16_t;

inline size_t elem_bytes(int dt) { return dt == DT_F32 ? 4 : 2; }
inline bool is_elem(int dt) { return dt == DT_F32 || dt == DT_F16 || dt == DT_BF16; }

// element i of a row of type dt; the type is the same for a whole launch, so the branch is uniform
__device__ __forceinline__ float load_elem(const void *p, int dt, long long i) {
    if (dt == DT_F32) return ((const float *)p)[i];
    if (dt == DT_F16) return (float)((const half_t *)p)[i];
    return (float)((const bf16_t *)p)[i];
}
__device__ __forceinline__ void store_elem(void *p, int dt, long long i, float v) {
    if (dt == DT_F32) ((float *)p)[i] = v;
    else if (dt == DT_F16) ((half_t *)p)[i] = (half_t)v;
    else ((bf16_t *)p)[i] = (bf16_t)v;
}

// eight elements at a 16-byte aligned place (f32: 32 bytes from it)
typedef float floatx8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8_e __attribute__((ext_vector_type(8)));
template <typename T> struct Eight;
template <> struct Eight<float> { typedef floatx8 type; };
template <> struct Eight<half_t> { typedef half8 type; };
template <> struct Eight<bf16_t> { typedef bf16x8_e type; };
template <typename T, typename ONCE>
__device__ __forceinline__ void store8(T *p, const floatx8 &v, ONCE) {   // true_type: past the caches
    const auto w = __builtin_convertvector(v, typename Eight<T>::type);
    if constexpr (ONCE::value) __builtin_nontemporal_store(w, (typename Eight<T>::type *)p);
    else *(typename Eight<T>::type *)p = w;
}

// rows of `width` bytes, `ld` bytes apart, in samples `bs` bytes apart
struct Window {
    const void *p;
    unsigned long long width, ld, rows, bs, samples;
    unsigned __int128 end() const {   // strides and counts of any size: more than 64 bits
        return (unsigned __int128)(unsigned long long)p + (unsigned __int128)(samples - 1) * bs + (unsigned __int128)(rows - 1) * ld + width;
    }
};
inline Window window(const void *p, size_t elem, unsigned long long width, unsigned long long ld,
                     unsigned long long rows, unsigned long long bs = 0, unsigned long long samples = 1) {
    return Window{p, width * elem, ld * elem, rows, bs * elem, samples};
}
// Whether two windows may share bytes. They do not if they are apart from each other, or if all rows of both begin at one
// place each within g bytes, g dividing every stride that is taken, and these column ranges do not meet (columns of the same
// rows; samples between each other's rows).
inline bool windows_meet(const Window &a, const Window &b) {
    const unsigned long long pa = (unsigned long long)a.p, pb = (unsigned long long)b.p;
    if (pa >= b.end() || pb >= a.end()) return false;
    unsigned long long g = 0;
    for (const Window *w : {&a, &b}) {
        if (w->rows > 1) g = std::gcd(g, w->ld);
        if (w->samples > 1) g = std::gcd(g, w->bs);
    }
    if (g == 0) return true;   // a row each
    const unsigned long long d = (pb >= pa ? pb - pa : g - (pa - pb) % g) % g;   // b's first column after a's
    return !(d >= a.width && d + b.width <= g);
}

} // namespace tsn
