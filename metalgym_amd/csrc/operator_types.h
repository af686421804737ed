// Element types of the training operators (MG_TYPE_*), their loads and stores
// in 16-byte vectors, and the argument checks that the operators share.
#pragma once
#include <hip/hip_fp16.h>

#include "internal.h"

namespace mg {
namespace dev {

// How rows of cols elements lie in vectors of 16 bytes (E elements).
enum Fit {
    kFull,  // every vector that is asked for is whole
    kTail,  // the row's last may be short, those past it are empty; cols >= E
    kTiny,  // cols < E
};

// Vector v of a row as floats, zeros past the row's end. The row may begin at any
// element: the hardware takes 16-byte loads and stores at any byte address, so odd
// widths and offset views run the same instructions as aligned ones. A short vector is
// read as the row's last 16 bytes and shifted: element by element, in a branch, every
// vector's load was waited for before the next was issued (LayerNorm of 40000 x 1001
// binary16: 50 us, so 30).
template <int FIT, class T, int E>
__device__ __forceinline__ void load_vec(const T* row, uint32_t v, uint32_t cols, float (&x)[E]) {
    static_assert(E * sizeof(T) == 16, "16-byte vectors");
    const uint32_t c = v * E;
    if constexpr (FIT == kTiny) {
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = c + e < cols ? (float)row[c + e] : 0.0f;
        return;
    }
    const uint32_t from = FIT == kTail && c > cols - E ? cols - E : c;
    // one load: an array of T filled by memcpy is taken apart into 2- and 4-byte loads
    // in places (LayerNorm of 32768 x 1024 bf16 with a residual: 47.7 us, so 42.2)
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4), aligned(2)));
    u32x4 w = *reinterpret_cast<const u32x4*>(row + from);
    if constexpr (FIT == kTail) {
        const uint32_t shift = (c - from) * sizeof(T);  // bytes; past 15 nothing is left
        w[0] = shift & 8 ? w[2] : w[0], w[1] = shift & 8 ? w[3] : w[1];
        w[0] = shift & 4 ? w[1] : w[0], w[1] = shift & 4 ? w[2] : w[1], w[2] = shift & 4 ? w[3] : w[2];
        if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int k = 0; k < 3; ++k) w[k] = __builtin_amdgcn_alignbyte(w[k + 1], w[k], shift & 2);
            w[3] >>= 8 * (shift & 2);
        }
    }
    typedef T vec __attribute__((ext_vector_type(E)));
    const vec t = __builtin_bit_cast(vec, w);
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = FIT == kFull || c + e < cols ? (float)t[e] : 0.0f;
}

// Rounds x to T and writes it; nothing past the row's end.
template <int FIT, class T, int E>
__device__ __forceinline__ void store_vec(T* row, uint32_t v, uint32_t cols, const float (&x)[E]) {
    const uint32_t c = v * E;
    if (FIT == kFull || c + E <= cols) {
        typedef T vec __attribute__((ext_vector_type(E)));
        vec t;
#pragma unroll
        for (int e = 0; e < E; ++e) t[e] = (T)x[e];
        __builtin_memcpy(row + c, &t, 16);
        return;
    }
#pragma unroll
    for (int e = 0; e < E; ++e)
        if (c + e < cols) row[c + e] = (T)x[e];
}

// Workgroups go to the 8 XCDs in turn, each of which has its own L2: gives every XCD
// one run of tiles.
__device__ __forceinline__ uint32_t xcd_run(uint32_t b, uint32_t count) {
    const uint32_t x = b & 7, each = count >> 3, more = count & 7;
    return x * each + (x < more ? x : more) + (b >> 3);
}

// Lane q of each four lanes holds four 16-bit values of column 4 a + q; gives it value q
// of the four columns 4 a .. 4 a + 3. Byte permutes with a lane's own selectors:
// selects become branches here.
template <class V>
__device__ __forceinline__ V quad_transpose(V v) {
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
    const uint32_t q = threadIdx.x & 3;
    const uint32_t halves = q & 1 ? 0x03020706u : 0x05040100u;  // (partner's high, own high) or (own low, partner's low)
    const uint32_t first = q & 2 ? 0x07060504u : 0x03020100u;   // the permute's first operand, or its second
    const u32x2 w = __builtin_bit_cast(u32x2, v);  // values (0, 1), (2, 3)
    // lanes q and q ^ 1 trade halves: even lanes get value 0 of both columns, then 2
    const uint32_t n0 = __builtin_amdgcn_mov_dpp(w[0], 0xB1, 0xF, 0xF, true);
    const uint32_t n1 = __builtin_amdgcn_mov_dpp(w[1], 0xB1, 0xF, 0xF, true);
    const uint32_t p0 = __builtin_amdgcn_perm(n0, w[0], halves), p1 = __builtin_amdgcn_perm(n1, w[1], halves);
    // lanes q and q ^ 2 trade words: the lower two lanes keep values 0 and 1
    const uint32_t got = __builtin_amdgcn_mov_dpp(__builtin_amdgcn_perm(p0, p1, first), 0x4E, 0xF, 0xF, true);
    const u32x2 out = {__builtin_amdgcn_perm(got, p0, first), __builtin_amdgcn_perm(p1, got, first)};
    return __builtin_bit_cast(V, out);
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
