// Element types of the training operators (MG_TYPE_*), their loads and stores
// in 16-byte vectors, and the argument checks that the operators share.
#pragma once
#include <hip/hip_fp16.h>

#include "internal.h"

namespace mg {
namespace dev {

template <class T>
struct TypeOf;
template <>
struct TypeOf<float> {
    static constexpr uint32_t type = MG_TYPE_FP32;
};
template <>
struct TypeOf<__bf16> {
    static constexpr uint32_t type = MG_TYPE_BF16;
};
template <>
struct TypeOf<_Float16> {
    static constexpr uint32_t type = MG_TYPE_FP16;
};

// Vector v (16 bytes, E elements) of a row of cols elements as floats, zeros
// past the row's end. The row may begin at any element: the hardware takes
// 16-byte loads and stores at any byte address, so odd widths and offset views
// run the same instructions as aligned ones.
template <bool EXACT, class T, int E>
__device__ __forceinline__ void load_vec(const T* row, uint32_t v, uint32_t cols, float (&x)[E]) {
    static_assert(E * sizeof(T) == 16, "16-byte vectors");
    const uint32_t c = v * E;
    if (EXACT || c + E <= cols) {
        T t[E];
        __builtin_memcpy(t, row + c, 16);
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = (float)t[e];
        return;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = c + e < cols ? (float)row[c + e] : 0.0f;
}

// Rounds x to T and writes it; nothing past the row's end.
template <bool EXACT, class T, int E>
__device__ __forceinline__ void store_vec(T* row, uint32_t v, uint32_t cols, const float (&x)[E]) {
    const uint32_t c = v * E;
    if (EXACT || c + E <= cols) {
        T t[E];
#pragma unroll
        for (int e = 0; e < E; ++e) t[e] = (T)x[e];
        __builtin_memcpy(row + c, t, 16);
        return;
    }
#pragma unroll
    for (int e = 0; e < E; ++e)
        if (c + e < cols) row[c + e] = (T)x[e];
}

}  // namespace dev

inline bool type_known(uint32_t type) { return type <= MG_TYPE_FP16; }
inline uint32_t type_bytes(uint32_t type) { return type == MG_TYPE_FP32 ? 4 : 2; }
inline bool aligned(const void* p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

// Makes a stream's device current for the launches of one call.
class StreamDevice {
   public:
    int enter(hipStream_t st, const char* what) {
        if (!st) return MG_OK;
        hipDevice_t dev = 0;
        int cur = 0;
        MG_HIP(hipStreamGetDevice(st, &dev), what);
        MG_HIP(hipGetDevice(&cur), what);
        if (cur != dev) {
            MG_HIP(hipSetDevice(dev), what);
            back_ = cur;
        }
        return MG_OK;
    }
    ~StreamDevice() {
        if (back_ >= 0) (void)hipSetDevice(back_);
    }

   private:
    int back_ = -1;
};

}  // namespace mg
