// checkers_amd/csrc/ckr_kv.h — device helpers shared by the cache, norm and
// attention kernels: element conversion, the row quantiser, the batch's layout.
#pragma once
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <cstdint>

#include "checkers_amd.h"

namespace ckr {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// ---- element types by their tags
struct ElemF32 { static constexpr int tag = CKR_F32, bytes = 4; };
struct ElemBF16 { static constexpr int tag = CKR_BF16, bytes = 2; };
struct ElemF16 { static constexpr int tag = CKR_F16, bytes = 2; };
struct ElemI8 { static constexpr int tag = CKR_I8, bytes = 1; };
struct ElemF8 { static constexpr int tag = CKR_F8, bytes = 1; };

__device__ __forceinline__ float as_f32(uint32_t u) { return __builtin_bit_cast(float, u); }
__device__ __forceinline__ uint32_t as_u32(float f) { return __builtin_bit_cast(uint32_t, f); }

// Two floats rounded to two 16-bit values in one dword (ties to even).
template <typename E> __device__ __forceinline__ uint32_t pack16(float a, float b);
template <> __device__ __forceinline__ uint32_t pack16<ElemBF16>(float a, float b) {
    typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
    const bf2 v = {(__bf16)a, (__bf16)b};
    return __builtin_bit_cast(uint32_t, v);
}
template <> __device__ __forceinline__ uint32_t pack16<ElemF16>(float a, float b) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    const h2 v = {(_Float16)a, (_Float16)b};
    return __builtin_bit_cast(uint32_t, v);
}
template <typename E> __device__ __forceinline__ float lo16(uint32_t v);
template <typename E> __device__ __forceinline__ float hi16(uint32_t v);
template <> __device__ __forceinline__ float lo16<ElemBF16>(uint32_t v) { return as_f32(v << 16); }
template <> __device__ __forceinline__ float hi16<ElemBF16>(uint32_t v) { return as_f32(v & 0xffff0000u); }
template <> __device__ __forceinline__ float lo16<ElemF16>(uint32_t v) {
    return (float)__builtin_bit_cast(_Float16, (uint16_t)v);
}
template <> __device__ __forceinline__ float hi16<ElemF16>(uint32_t v) {
    return (float)__builtin_bit_cast(_Float16, (uint16_t)(v >> 16));
}
// Four codes of a dword as floats (exact).
template <typename E> __device__ __forceinline__ f32x4 codes4(uint32_t v);
template <> __device__ __forceinline__ f32x4 codes4<ElemF8>(uint32_t v) {
    const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)v, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)v, true);
    return f32x4{a.x, a.y, b.x, b.y};
}
template <> __device__ __forceinline__ f32x4 codes4<ElemI8>(uint32_t v) {
    return f32x4{(float)(int8_t)v, (float)(int8_t)(v >> 8), (float)(int8_t)(v >> 16), (float)((int32_t)v >> 24)};
}
// Four floats as codes (ties to even); their magnitude is at most the type's largest value.
template <typename E> __device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d);
template <> __device__ __forceinline__ uint32_t encode4<ElemF8>(float a, float b, float c, float d) {
    const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, lo, true);
}
template <> __device__ __forceinline__ uint32_t encode4<ElemI8>(float a, float b, float c, float d) {
    const uint32_t x = (uint32_t)(int)__builtin_rintf(a) & 0xffu, y = (uint32_t)(int)__builtin_rintf(b) & 0xffu;
    const uint32_t z = (uint32_t)(int)__builtin_rintf(c) & 0xffu, w = (uint32_t)(int)__builtin_rintf(d);
    return x | y << 8 | z << 16 | w << 24;
}

// The same vectors at any address: global memory takes them whole.
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(1)));
typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(1)));
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(1)));
template <bool ALIGNED> struct Vecs { typedef u32x4 U4; typedef u32x2 U2; typedef f32x4 F4; };
template <> struct Vecs<false> { typedef u32x4_any U4; typedef u32x2_any U2; typedef f32x4_any F4; };

// N elements (a multiple of 8) at p, ALIGNED: for 16-byte loads (8-bit: N bytes).
template <typename E, int N, bool ALIGNED = true> __device__ __forceinline__ void load_vec(const void* p, float* x) {
    if constexpr (E::bytes == 4) {
#pragma unroll
        for (int i = 0; i < N / 4; i++) {
            const f32x4 v = reinterpret_cast<const typename Vecs<ALIGNED>::F4*>(p)[i];
#pragma unroll
            for (int j = 0; j < 4; j++) x[4 * i + j] = v[j];
        }
    } else if constexpr (E::bytes == 2) {
#pragma unroll
        for (int i = 0; i < N / 8; i++) {
            const u32x4 v = reinterpret_cast<const typename Vecs<ALIGNED>::U4*>(p)[i];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                x[8 * i + 2 * j] = lo16<E>(v[j]);
                x[8 * i + 2 * j + 1] = hi16<E>(v[j]);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < N / 8; i++) {
            const u32x2 v = reinterpret_cast<const typename Vecs<ALIGNED>::U2*>(p)[i];
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const f32x4 c = codes4<E>(v[j]);
#pragma unroll
                for (int k = 0; k < 4; k++) x[8 * i + 4 * j + k] = c[k];
            }
        }
    }
}
template <typename E, int N, bool ALIGNED = true> __device__ __forceinline__ void store_vec(void* p, const float* x) {
    if constexpr (E::bytes == 4) {
#pragma unroll
        for (int i = 0; i < N / 4; i++)
            reinterpret_cast<typename Vecs<ALIGNED>::F4*>(p)[i] = f32x4{x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]};
    } else if constexpr (E::bytes == 2) {
#pragma unroll
        for (int i = 0; i < N / 8; i++) {
            u32x4 v;
#pragma unroll
            for (int j = 0; j < 4; j++) v[j] = pack16<E>(x[8 * i + 2 * j], x[8 * i + 2 * j + 1]);
            reinterpret_cast<typename Vecs<ALIGNED>::U4*>(p)[i] = v;
        }
    } else if constexpr (N % 16 == 0) {
#pragma unroll
        for (int i = 0; i < N / 16; i++) {
            u32x4 v;
#pragma unroll
            for (int j = 0; j < 4; j++) v[j] = encode4<E>(x[16 * i + 4 * j], x[16 * i + 4 * j + 1], x[16 * i + 4 * j + 2], x[16 * i + 4 * j + 3]);
            reinterpret_cast<typename Vecs<ALIGNED>::U4*>(p)[i] = v;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N / 8; i++) {
            const float* y = x + 8 * i;
            reinterpret_cast<typename Vecs<ALIGNED>::U2*>(p)[i] = u32x2{encode4<E>(y[0], y[1], y[2], y[3]), encode4<E>(y[4], y[5], y[6], y[7])};
        }
    }
}
// One element (a row's last ones).
template <typename E> __device__ __forceinline__ float load_one(const void* p, int64_t i) {
    if constexpr (E::bytes == 4) return reinterpret_cast<const float*>(p)[i];
    else return lo16<E>(reinterpret_cast<const uint16_t*>(p)[i]);
}
template <typename E> __device__ __forceinline__ void store_one(void* p, int64_t i, float x) {
    if constexpr (E::bytes == 4) reinterpret_cast<float*>(p)[i] = x;
    else if constexpr (E::bytes == 2) reinterpret_cast<uint16_t*>(p)[i] = (uint16_t)pack16<E>(x, 0.f);
    else reinterpret_cast<uint8_t*>(p)[i] = (uint8_t)encode4<E>(x, 0.f, 0.f, 0.f);
}

// ---- the row quantiser.  The largest magnitude is taken over the bit patterns
// of |x| as integers: the order is that of the values, infinities are above
// every finite value and NaN above infinity, so a row that holds either shows it.
__device__ __forceinline__ uint32_t abs_bits(float x) { return as_u32(x) & 0x7fffffffu; }
struct RowScale { float scale, inv; };
template <typename E> __device__ __forceinline__ RowScale row_scale(uint32_t top) {
    constexpr float T = E::tag == CKR_F8 ? 448.f : 127.f;
    if (top >= 0x7f800000u) return {as_f32(0x7fc00000u), 0.f};
    const float a = as_f32(top);
    if (a < 0x1p-100f) return {0.f, 0.f};
    return {a / T, T / a};
}
// x * inv, and zero (not NaN) where inv is zero.
__device__ __forceinline__ float scaled(float x, float inv) { return inv == 0.f ? 0.f : x * inv; }

// ---- the batch
struct KvBatch {
    const int32_t* table;
    const int32_t* starts;
    const int32_t* offsets;
    int64_t table_stride;
    uint32_t width, n_seqs, n_tokens;
};

// The cache page of a sequence's position, or -1 when it is unmapped.
__device__ __forceinline__ int32_t page_of(const KvBatch& b, uint32_t seq, int64_t pos, uint32_t page_shift,
                                           uint32_t n_pages) {
    if (pos < 0) return -1;
    const uint64_t col = (uint64_t)pos >> page_shift;
    if (col >= b.width) return -1;
    const int32_t p = b.table[(int64_t)seq * b.table_stride + (int64_t)col];
    return (uint32_t)p < n_pages ? p : -1;
}

}  // namespace ckr
