// What the kernels share that walk rows of logits: how logits are stored, and keys that order as they do.
#pragma once
#include "common.h"

namespace {

// Logits as stored, 16 bytes at a time
struct LogitF32 {
    static constexpr int VEC = 4, BYTES = 4, VECS = 4;        // VECS: 16-byte loads a lane and step
    static __device__ __forceinline__ void unpack(const u32x4& v, float* f) {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(v[i]);
    }
    static __device__ __forceinline__ float at(const void* p, int64_t i) { return ((const float*)p)[i]; }
};
template <typename T>
struct Logit16 {
    static constexpr int VEC = 8, BYTES = 2, VECS = 2;
    static __device__ __forceinline__ void unpack(const u32x4& v, float* f) { unpack8<T>(v, f); }
    static __device__ __forceinline__ float at(const void* p, int64_t i) { return T::to_float(((const uint16_t*)p)[i]); }
};

// keys that order as the values do
__device__ __forceinline__ uint32_t order32(float f) {
    const uint32_t u = __float_as_uint(f);
    return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float order32_back(uint32_t k) { return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu)); }

}  // namespace
