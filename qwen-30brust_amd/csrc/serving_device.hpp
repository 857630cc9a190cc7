// Device helpers of the operators on device tensors (serving.hpp).
#pragma once
#include "qh_device.hpp"
#include "serving.hpp"

namespace qh {

typedef __bf16 bf16_t;

// Element i of p; Q8_0 codes as whole numbers.
template <uint32_t K> __device__ __forceinline__ float elem(const uint8_t* p, size_t i) {
    if constexpr (K == F32) return gld<float>(p + 4 * i);
    else if constexpr (K == F16) return (float)gld<_Float16>(p + 2 * i);
    else if constexpr (K == BF16) return __uint_as_float((uint32_t)gld<uint16_t>(p + 2 * i) << 16);
    else return (float)gld<int8_t>(p + i);
}
// x rounded once, to the nearest (ties to even).
template <uint32_t K> __device__ __forceinline__ void put(uint8_t* p, size_t i, float x) {
    if constexpr (K == F32) reinterpret_cast<float*>(p)[i] = x;
    else if constexpr (K == F16) reinterpret_cast<_Float16*>(p)[i] = (_Float16)x;
    else reinterpret_cast<bf16_t*>(p)[i] = (bf16_t)x;
}
__device__ __forceinline__ void put_kind(uint32_t kind, uint8_t* p, size_t i, float x) {
    if (kind == F32) put<F32>(p, i, x);
    else if (kind == F16) put<F16>(p, i, x);
    else put<BF16>(p, i, x);
}
__device__ __forceinline__ float elem_kind(uint32_t kind, const uint8_t* p, size_t i) {
    return kind == F32 ? elem<F32>(p, i) : kind == F16 ? elem<F16>(p, i) : elem<BF16>(p, i);
}

// Unsigned key with the order of f32::total_cmp, and back.
__device__ __forceinline__ uint32_t order_key(float x) {
    const uint32_t b = __float_as_uint(x);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t u) {
    return __uint_as_float(u ^ ((uint32_t)((int32_t)~u >> 31) | 0x80000000u));
}

// The keys of sequence b, or -1 where its length is not in [0, most].
__device__ __forceinline__ int32_t length_of(const Rows& r, uint32_t b) {
    const int32_t n = gld<int32_t>(r.length + b);
    return n < 0 || (uint32_t)n > r.most ? -1 : n;
}

}  // namespace qh
