// Values of the three storage types (float32, bfloat16, float16) as float32 and back: one rounding, to nearest even.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "crystalformer_b200.h"

namespace cf {

inline bool known_type(int type) { return type == CF_FLOAT32 || type == CF_BFLOAT16 || type == CF_FLOAT16; }
inline int type_size(int type) { return type == CF_FLOAT32 ? 4 : 2; }

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <class T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

// the largest finite value
template <class T> __device__ __forceinline__ float largest();
template <> __device__ __forceinline__ float largest<__nv_bfloat16>() { return __uint_as_float(0x7f7f0000u); }
template <> __device__ __forceinline__ float largest<__half>() { return 65504.f; }

// two values of 16 bits in one word, the first in the lower half
template <class T> __device__ __forceinline__ uint32_t pack_two(float a, float b);
template <> __device__ __forceinline__ uint32_t pack_two<__nv_bfloat16>(float a, float b)
{
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&v);
}
template <> __device__ __forceinline__ uint32_t pack_two<__half>(float a, float b)
{
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&v);
}
template <class T> __device__ __forceinline__ float2 unpack_two(uint32_t w);
template <> __device__ __forceinline__ float2 unpack_two<__nv_bfloat16>(uint32_t w)
{
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <> __device__ __forceinline__ float2 unpack_two<__half>(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2 *>(&w)); }

// VEC neighbouring values, VEC * sizeof(T) in {2, 4, 8, 16} bytes and aligned to that
template <class T, int VEC>
__device__ __forceinline__ void load_values(const T *p, float (&v)[VEC])
{
    if constexpr (VEC == 1) {
        v[0] = to_float(*p);
    } else if constexpr (sizeof(T) == 4) {
        static_assert(VEC == 4, "four floats");
        const float4 w = *reinterpret_cast<const float4 *>(p);
        v[0] = w.x; v[1] = w.y; v[2] = w.z; v[3] = w.w;
    } else {
        static_assert(VEC == 4 || VEC == 8, "eight or sixteen bytes");
        uint32_t w[VEC / 2];
        if constexpr (VEC == 8) {
            const uint4 u = *reinterpret_cast<const uint4 *>(p);
            w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
        } else {
            const uint2 u = *reinterpret_cast<const uint2 *>(p);
            w[0] = u.x; w[1] = u.y;
        }
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i) {
            const float2 f = unpack_two<T>(w[i]);
            v[2 * i] = f.x; v[2 * i + 1] = f.y;
        }
    }
}
template <class T, int VEC>
__device__ __forceinline__ void store_values(T *p, const float (&v)[VEC])
{
    if constexpr (VEC == 1) {
        *p = from_float<T>(v[0]);
    } else if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
    } else if constexpr (VEC == 8) {
        *reinterpret_cast<uint4 *>(p) = make_uint4(pack_two<T>(v[0], v[1]), pack_two<T>(v[2], v[3]), pack_two<T>(v[4], v[5]), pack_two<T>(v[6], v[7]));
    } else {
        *reinterpret_cast<uint2 *>(p) = make_uint2(pack_two<T>(v[0], v[1]), pack_two<T>(v[2], v[3]));
    }
}

// ... held as they lie in memory, to be converted when they are needed
template <int BYTES> struct RawBytes;
template <> struct RawBytes<16> { using type = uint4; };
template <> struct RawBytes<8> { using type = uint2; };
template <> struct RawBytes<4> { using type = uint32_t; };
template <> struct RawBytes<2> { using type = uint16_t; };
template <class T, int VEC> using Raw = typename RawBytes<VEC * sizeof(T)>::type;
template <class T, int VEC> __device__ __forceinline__ Raw<T, VEC> load_raw(const T *p) { return *reinterpret_cast<const Raw<T, VEC> *>(p); }
template <class T> __device__ __forceinline__ float value_of(uint32_t w) { return __uint_as_float(w); }  // of a word with one value
template <> __device__ __forceinline__ float value_of<__nv_bfloat16>(uint32_t w) { return __uint_as_float(w << 16); }
template <> __device__ __forceinline__ float value_of<__half>(uint32_t w) { return __half2float(__ushort_as_half((unsigned short)w)); }
template <class T, int VEC>
__device__ __forceinline__ void expand(const Raw<T, VEC> &raw, float (&v)[VEC])
{
    if constexpr (VEC == 1) {
        v[0] = value_of<T>(raw);
    } else if constexpr (sizeof(T) == 4) {
        v[0] = __uint_as_float(raw.x); v[1] = __uint_as_float(raw.y); v[2] = __uint_as_float(raw.z); v[3] = __uint_as_float(raw.w);
    } else {
        const float2 f = unpack_two<T>(raw.x), g = unpack_two<T>(raw.y);
        v[0] = f.x; v[1] = f.y; v[2] = g.x; v[3] = g.y;
        if constexpr (VEC == 8) {
            const float2 h = unpack_two<T>(raw.z), i = unpack_two<T>(raw.w);
            v[4] = h.x; v[5] = h.y; v[6] = i.x; v[7] = i.y;
        }
    }
}

// 32 neighbouring bytes, aligned to that, in one store
__device__ __forceinline__ void store_32(void *p, const uint32_t (&w)[8])
{
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]),
                 "r"(w[6]), "r"(w[7])
                 : "memory");
}

inline bool aligned_to(const void *p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

}  // namespace cf
