// Vectors of fp32, bf16 or fp16 values as one access moves them, and their conversion to fp32.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstddef>
#include <cstdint>
#include <type_traits>

namespace scx {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ void from_f32(float& o, float v) { o = v; }
__device__ __forceinline__ void from_f32(__nv_bfloat16& o, float v) { o = __float2bfloat16_rn(v); }
__device__ __forceinline__ void from_f32(__half& o, float v) { o = __float2half_rn(v); }

// V values of type T.  Two-byte types are held as words of two, whose halves are the upper and lower bits
// of two fp32 values (bf16) or convert together (fp16): arrays of the types themselves move as 16-bit
// pieces (a step from 139 to 129 us on 8192 x 2048 bf16 tokens with a gate, forward and backward).
template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
    static constexpr bool kWordsOfTwo = sizeof(T) == 2 && V >= 2;
    using Word = std::conditional_t<kWordsOfTwo, uint32_t, T>;
    static constexpr int kWords = kWordsOfTwo ? V / 2 : V;
    Word w[kWords];

    // values 2i and 2i + 1
    __device__ __forceinline__ float2 pair(int i) const {
        if constexpr (!kWordsOfTwo) {
            return make_float2(to_f32(w[2 * i % kWords]), to_f32(w[(2 * i + 1) % kWords]));
        } else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
            return make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
        } else {
            return __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        }
    }
    __device__ __forceinline__ void set_pair(int i, float2 v) {
        if constexpr (!kWordsOfTwo) {
            from_f32(w[2 * i % kWords], v.x);
            from_f32(w[(2 * i + 1) % kWords], v.y);
        } else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
            const __nv_bfloat162 o = __floats2bfloat162_rn(v.x, v.y);
            w[i] = *reinterpret_cast<const uint32_t*>(&o);
        } else {
            const __half2 o = __floats2half2_rn(v.x, v.y);
            w[i] = *reinterpret_cast<const uint32_t*>(&o);
        }
    }
    // the value of a vector of one
    __device__ __forceinline__ float one() const {
        static_assert(V == 1, "more than one value");
        return to_f32(w[0]);
    }
    __device__ __forceinline__ void set_one(float v) {
        static_assert(V == 1, "more than one value");
        from_f32(w[0], v);
    }
};

template <typename T, int V>
__device__ __forceinline__ Vec<T, V> load_vec(const void* p, size_t e) {
    return *reinterpret_cast<const Vec<T, V>*>(static_cast<const T*>(p) + e);
}

template <typename T, int V>
__device__ __forceinline__ void store_vec(void* p, size_t e, const Vec<T, V>& v) {
    *reinterpret_cast<Vec<T, V>*>(static_cast<T*>(p) + e) = v;
}

}  // namespace scx
