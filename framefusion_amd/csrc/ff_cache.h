// The paged cache of decoded tokens: where a position lies, and what a stored code stands for.  Shared by the kernels that
// write, read, move (ff_cache.hip) and attend to it (ff_attend.hip).
#pragma once

#include "ff_common.h"
#include "ff_place.h"

namespace ff {

constexpr int kStoreSame = 0;   // template value: the cache holds T itself

typedef float f32x2 __attribute__((ext_vector_type(2)));

// 2^(byte - 127); 255 stands for a block of NaN, 0 for a row that was never written (its codes are zeros)
__device__ inline float block_scale(uint32_t byte) { return __uint_as_float(byte == 255u ? 0x7fc00000u : byte << 23); }

// bytes of one row of `dh` channels
template <int DT, int STORE> __device__ inline int row_bytes(int dh) {
    return STORE == FF_STORE_E4M3 ? dh : STORE == FF_STORE_E2M1 ? dh / 2 : dh * Act<DT>::kBytes;
}

// 8 consecutive channels of T as floats
template <int DT> __device__ inline void load8(const void* p, float* f) {
    if constexpr (DT == FF_F32) {
        Act<DT>::unpack(*(const uint4*)p, f);
        Act<DT>::unpack(((const uint4*)p)[1], f + 4);
    } else {
        Act<DT>::unpack(*(const uint4*)p, f);
    }
}
// (rounded to T)
template <int DT> __device__ inline void store8(void* p, const float* f) {
    if constexpr (DT == FF_F32) {
        *(uint4*)p = Act<DT>::pack(f);
        ((uint4*)p)[1] = Act<DT>::pack(f + 4);
    } else if constexpr (DT == FF_BF16) {
        *(uint4*)p = Act<DT>::pack_rne(f);
    } else {
        *(uint4*)p = Act<DT>::pack(f);
    }
}
// 8 codes -> the values they stand for (exact in fp32)
__device__ inline void decode8_e4m3(uint2 w, float s, float* f) {
    const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w.x, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w.x, true);
    const f32x2 c = __builtin_amdgcn_cvt_pk_f32_fp8((int)w.y, false), d = __builtin_amdgcn_cvt_pk_f32_fp8((int)w.y, true);
    f[0] = a.x * s; f[1] = a.y * s; f[2] = b.x * s; f[3] = b.y * s;
    f[4] = c.x * s; f[5] = c.y * s; f[6] = d.x * s; f[7] = d.y * s;
}
__device__ inline void decode8_e2m1(uint32_t w, float s, float* f) {
    const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 1);
    const f32x2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 3);
    f[0] = a.x * s; f[1] = a.y * s; f[2] = b.x * s; f[3] = b.y * s;
    f[4] = c.x * s; f[5] = c.y * s; f[6] = d.x * s; f[7] = d.y * s;
}
// channels [8 u, 8 u + 8) of stored row `row`
template <int DT, int STORE>
__device__ inline void fetch8(const void* codes, const uint8_t* scales, int64_t row, int dh, int u, float* f) {
    const char* p = (const char*)codes + row * row_bytes<DT, STORE>(dh);
    if constexpr (STORE == FF_STORE_E4M3) {
        decode8_e4m3(((const uint2*)p)[u], block_scale(scales[row * (dh / 32) + u / 4]), f);
    } else if constexpr (STORE == FF_STORE_E2M1) {
        decode8_e2m1(((const uint32_t*)p)[u], block_scale(scales[row * (dh / 32) + u / 4]), f);
    } else {
        load8<DT>(p + u * 8 * Act<DT>::kBytes, f);
    }
}

// channels [4 u, 4 u + 4), T of 16 bits
template <int DT, int STORE>
__device__ inline void fetch4(const void* codes, const uint8_t* scales, int64_t row, int dh, int u, float* f) {
    const char* p = (const char*)codes + row * row_bytes<DT, STORE>(dh);
    float x[8];
    if constexpr (STORE == FF_STORE_E4M3) decode8_e4m3(make_uint2(((const uint32_t*)p)[u], 0), block_scale(scales[row * (dh / 32) + u / 8]), x);
    else if constexpr (STORE == FF_STORE_E2M1) decode8_e2m1(((const uint16_t*)p)[u], block_scale(scales[row * (dh / 32) + u / 8]), x);
    else Act<DT>::unpack(make_uint4(((const uint2*)p)[u].x, ((const uint2*)p)[u].y, 0, 0), x);
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = x[e];
}

inline bool cache_aligned(const void* p) { return ((uintptr_t)p & 15) == 0; }
// FF_OK, or what is wrong with the part of a call that names the cache
int cache_check(const ff_cache_t* c);

}  // namespace ff
