// points8.h -- points held in 8 bits: the store, its element types, the helpers its kernels share.
#pragma once
#include "internal.h"
#include "points8_plan.h"

struct ae_points8 {
    uint64_t capacity = 0, dim = 0;
    uint64_t row_bytes = 0;      // dim rounded up to 16: every row starts on 16 bytes; the bytes beyond dim stay 0
    uint32_t blocks = 0;         // ceil(dim / 128)
    uint64_t scale_stride = 0;   // scales[block][row]: from block to block; the rows of a block lie together, as the matrix cores take them
    int device = 0;
    ae::DevBuf<uint8_t> codes, scales;
    ae::DevBuf<uint32_t> owner;  // per row: which row of the running write holds it (0 between writes)
};

namespace ae {

struct Rows8 {   // rows of codes with their scales: part of a store, or quantised rows in scratch memory
    const uint8_t* codes;
    const uint8_t* scales;
    uint64_t row_bytes;
    uint64_t scale_stride;
    uint64_t rows;
};

// bytes from block to block of the scales of `rows` rows, and what lies behind the last one: a tile takes the bytes of rows that do not exist
// along (they multiply zeros, and no result of theirs is written)
inline uint64_t points8_scale_stride(uint64_t rows) { return (rows + 15) / 16 * 16; }
constexpr uint64_t kScaleSlack = 512;
inline uint64_t type_size(uint32_t type) { return type == AE_TYPE_F32 ? 4 : 2; }
inline void check_type(uint32_t type, const char* what) {
    if (type > AE_TYPE_F16) fail(AE_ERR_INVALID_ARG, "%s: unknown element type %u (AE_TYPE_F32, AE_TYPE_BF16, AE_TYPE_F16)", what, type);
}
inline void check_aligned(const void* ptr, uint64_t bytes, const char* what) {
    if ((uintptr_t)ptr % bytes) fail(AE_ERR_INVALID_ARG, "%s is not aligned to %llu bytes", what, (unsigned long long)bytes);
}
// rows of `len` elements `ld` apart at `ptr`; rows > 0
inline void check_rows(const void* ptr, uint32_t type, uint64_t rows, uint64_t len, uint64_t ld, const char* what) {
    check_type(type, what);
    if (!ptr) fail(AE_ERR_INVALID_ARG, "%s is NULL", what);
    if (ld < len) fail(AE_ERR_INVALID_ARG, "%s: a stride of %llu is shorter than the row's %llu elements", what, (unsigned long long)ld, (unsigned long long)len);
    if (ld > (1ull << 40) / rows) fail(AE_ERR_INVALID_ARG, "%s: %llu rows of stride %llu are out of range", what, (unsigned long long)rows, (unsigned long long)ld);
    check_aligned(ptr, type_size(type), what);
}
void check_points8(const ae_points8* p, uint64_t first, uint64_t n, const char* what);   // on the current device, rows in range
inline Rows8 points8_rows(const ae_points8* p, uint64_t first, uint64_t n) {
    return Rows8{p->codes.p + first * p->row_bytes, p->scales.p + first, p->row_bytes, p->scale_stride, n};
}
// n rows of x into codes[n][row_bytes] / scales[blocks][scale_stride]
void points8_quantise(const void* d_x, uint32_t type, uint64_t n, uint64_t ldx, uint64_t dim, uint8_t* codes, uint8_t* scales, uint64_t scale_stride, hipStream_t s);

template <int TYPE> struct Elem;
template <> struct Elem<AE_TYPE_F32> { using T = float; };
template <> struct Elem<AE_TYPE_BF16> { using T = __bf16; };
template <> struct Elem<AE_TYPE_F16> { using T = _Float16; };

// f(std::integral_constant<int, TYPE>) for the run-time type
template <class F>
inline void by_type(uint32_t type, F&& f) {
    switch (type) {
        case AE_TYPE_F32: f(std::integral_constant<int, AE_TYPE_F32>{}); break;
        case AE_TYPE_BF16: f(std::integral_constant<int, AE_TYPE_BF16>{}); break;
        default: f(std::integral_constant<int, AE_TYPE_F16>{}); break;
    }
}

using f32x2 = __attribute__((ext_vector_type(2))) float;
using f32x4 = __attribute__((ext_vector_type(4))) float;
using u32x2 = __attribute__((ext_vector_type(2))) uint32_t;
using u32x4 = __attribute__((ext_vector_type(4))) uint32_t;
using bf16x8 = __attribute__((ext_vector_type(8))) __bf16;

// 16 bytes at any address of a 16-bit element: the memory pipeline takes vectors at any alignment, at the price of the lines that they cross
typedef uint32_t Piece __attribute__((ext_vector_type(4), aligned(2)));

// eight consecutive elements, or `count` of them (the others 0)
template <int TYPE>
__device__ __forceinline__ void load8(const typename Elem<TYPE>::T* __restrict__ p, int count, float (&v)[8]) {
    using T = typename Elem<TYPE>::T;
    constexpr int W = 16 / sizeof(T);
    using V = __attribute__((ext_vector_type(W))) T;
    if (count == 8) {
#pragma unroll
        for (int q = 0; q < 8 / W; q++) {
            const V a = __builtin_bit_cast(V, reinterpret_cast<const Piece*>(p)[q]);
#pragma unroll
            for (int t = 0; t < W; t++) v[q * W + t] = (float)a[t];
        }
    } else {
#pragma unroll
        for (int t = 0; t < 8; t++) v[t] = t < count ? (float)p[t] : 0.f;
    }
}
// one rounding, to nearest even, where T is narrower than f32
template <int TYPE>
__device__ __forceinline__ void store8(typename Elem<TYPE>::T* __restrict__ p, int count, const float (&v)[8]) {
    using T = typename Elem<TYPE>::T;
    constexpr int W = 16 / sizeof(T);
    using V = __attribute__((ext_vector_type(W))) T;
    if (count == 8) {
#pragma unroll
        for (int q = 0; q < 8 / W; q++) {
            V a;
#pragma unroll
            for (int t = 0; t < W; t++) a[t] = (T)v[q * W + t];
            reinterpret_cast<Piece*>(p)[q] = __builtin_bit_cast(Piece, a);
        }
    } else {
#pragma unroll
        for (int t = 0; t < 8; t++)
            if (t < count) p[t] = (T)v[t];
    }
}

// maximum over the 16 lanes of a row of the wave (every lane gets it)
__device__ __forceinline__ uint32_t max16(uint32_t v) {
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xF, 0xF, true));   // row_ror:8
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x124, 0xF, 0xF, true));
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x122, 0xF, 0xF, true));
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x121, 0xF, 0xF, true));
}
// the scale byte of a block whose largest finite magnitude has these bits: exponent + 127 of the smallest 2^e, e >= -126, with a <= 448 * 2^e
// = 1.75 * 2^(e + 8)
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax_bits) {
    const int b = (int)(amax_bits >> 23) - 8 + ((amax_bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    return (uint32_t)max(b, 1);
}
// the largest finite magnitude among v, as bits (non-negative floats order like their bits)
__device__ __forceinline__ uint32_t amax8(const float (&v)[8]) {
    uint32_t a = 0;
#pragma unroll
    for (int t = 0; t < 8; t++) {
        const uint32_t u = __float_as_uint(v[t]) & 0x7FFFFFFFu;
        a = max(a, u < 0x7F800000u ? u : 0u);
    }
    return a;
}
// the codes of eight values under a scale byte.  x * 2^-e is exact (or below every code), |.| <= 448: one rounding, the conversion's.  Under the largest
// scale, 2^120, the codes from 256 on would stand for 2^128 and more, which f32 does not have: 240 is the largest there, what is finite stays finite.
__device__ __forceinline__ uint2 encode8(const float (&v)[8], uint32_t byte) {
    const float shrink = __uint_as_float((254u - byte) << 23);
    float y[8];
#pragma unroll
    for (int t = 0; t < 8; t++) {
        const bool finite = (__float_as_uint(v[t]) & 0x7FFFFFFFu) < 0x7F800000u;
        y[t] = finite ? v[t] * shrink : __uint_as_float(0x7FC00000u);
    }
    if (byte == 247u) {
#pragma unroll
        for (int t = 0; t < 8; t++) y[t] = y[t] != y[t] ? y[t] : __builtin_amdgcn_fmed3f(y[t], -240.f, 240.f);
    }
    int lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], lo, true);
    int hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[4], y[5], 0, false);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[6], y[7], hi, true);
    return make_uint2((uint32_t)lo, (uint32_t)hi);
}
// the values of eight codes: exact products with a power of two (byte 0, a row never written, holds zeros only)
__device__ __forceinline__ void decode8(uint2 c, uint32_t byte, float (&v)[8]) {
    const float scale = __uint_as_float(byte << 23);
    const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)c.x, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)c.x, true);
    const f32x2 d = __builtin_amdgcn_cvt_pk_f32_fp8((int)c.y, false), e = __builtin_amdgcn_cvt_pk_f32_fp8((int)c.y, true);
    v[0] = a[0] * scale; v[1] = a[1] * scale; v[2] = b[0] * scale; v[3] = b[1] * scale;
    v[4] = d[0] * scale; v[5] = d[1] * scale; v[6] = e[0] * scale; v[7] = e[1] * scale;
}

// the values of eight codes as bf16, exact (to a multiple of 2^-133, its smallest number): widened with the block's power of two in one step
__device__ __forceinline__ bf16x8 widen8(uint32_t lo, uint32_t hi, uint32_t byte) {
    using bf16x2 = __attribute__((ext_vector_type(2))) __bf16;
    const float scale = __uint_as_float(byte << 23);
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
    return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

}  // namespace ae
