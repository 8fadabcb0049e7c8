// Row operators in 32 bits over fp32 / bf16 / fp16 rows, and the 8-bit form of a row (layer_norm.hip, act8.hip).
//
// 8-bit rows: 32 consecutive columns share one power of two,
//     scale = 2^(byte - 127),  byte = max(E - 8, 10),  E = biased exponent of max |x| (+ 1 where its significand exceeds 1.75),
// so |x| / scale <= 448 and a value is its nearest OCP e4m3 multiple of the scale (ties to even).  A power of two costs e4m3 no
// significand bit, makes the division exact - the rounding of the code is the only one - and keeps every value a bf16 as well: byte >= 10
// keeps the smallest code (2^-9 scale) at 2^-126, a normal number.  Two additions serve the backward pass: a positive value never becomes
// zero (it becomes the smallest code), so "x > 0" - LeakyReLU's derivative - reads off the code exactly; and NaN / +-inf become the NaN
// code and stay out of the maximum, so one bad value does not hide its 31 neighbours.  |x| is held at 1.875 * 2^127, in rows of fp16 at
// 1.875 * 2^15: the type's largest values would round to 2^128 / 2^16 and come back as infinities.
#pragma once
#include "common.h"
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

namespace pcvae {

constexpr int kAct8Block = 32;
typedef float f32x4_t __attribute__((ext_vector_type(4)));

// a 16-byte (8-byte, 4-byte) piece of memory at any alignment: rows of odd widths start anywhere.  One load / store instruction -
// the global path takes unaligned accesses.
template <int BYTES>
struct __attribute__((packed)) Raw { uint32_t w[BYTES / 4]; };

template <typename T> struct RowType;
constexpr uint32_t kAct8Cap = 0x7f700000u;      // 1.875 * 2^127
constexpr uint32_t kAct8CapHalf = 0x47700000u;  // 1.875 * 2^15
template <> struct RowType<float> {
    static constexpr int VW = 4;
    static constexpr uint32_t CAP = kAct8Cap;   // (bits of) the largest magnitude an 8-bit row of this type holds
    static __device__ __forceinline__ float one(const float* p) { return *p; }
    static __device__ __forceinline__ void put(float* p, float v) { *p = v; }
    static __device__ __forceinline__ void widen(const Raw<16>& r, float (&v)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(r.w[i]);
    }
    static __device__ __forceinline__ void narrow(const float (&v)[4], Raw<16>& r) {
#pragma unroll
        for (int i = 0; i < 4; ++i) r.w[i] = __float_as_uint(v[i]);
    }
};
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));

template <> struct RowType<__bf16> {
    static constexpr int VW = 8;
    static constexpr uint32_t CAP = kAct8Cap;
    static __device__ __forceinline__ float one(const __bf16* p) {
        return __uint_as_float((uint32_t)*reinterpret_cast<const uint16_t*>(p) << 16);
    }
    static __device__ __forceinline__ void put(__bf16* p, float v) { *p = (__bf16)v; }
    static __device__ __forceinline__ void widen(const Raw<16>& r, float (&v)[8]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(r.w[i] << 16);
            v[2 * i + 1] = __uint_as_float(r.w[i] & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ void narrow(const float (&v)[8], Raw<16>& r) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bf16x2_t h = __builtin_convertvector((f32x2_t{v[2 * i], v[2 * i + 1]}), bf16x2_t);
            r.w[i] = __builtin_bit_cast(uint32_t, h);
        }
    }
};
template <> struct RowType<_Float16> {
    static constexpr int VW = 8;
    static constexpr uint32_t CAP = kAct8CapHalf;
    static __device__ __forceinline__ float one(const _Float16* p) { return (float)*p; }
    static __device__ __forceinline__ void put(_Float16* p, float v) { *p = (_Float16)v; }
    static __device__ __forceinline__ void widen(const Raw<16>& r, float (&v)[8]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f16x2_t h = __builtin_bit_cast(f16x2_t, r.w[i]);
            v[2 * i] = (float)h[0];
            v[2 * i + 1] = (float)h[1];
        }
    }
    static __device__ __forceinline__ void narrow(const float (&v)[8], Raw<16>& r) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f16x2_t h = {(_Float16)v[2 * i], (_Float16)v[2 * i + 1]};
            r.w[i] = __builtin_bit_cast(uint32_t, h);
        }
    }
};

// ---- 16-byte pieces of a row of D columns, a lane's piece at column c (a multiple of VW) -------------------------------------------
// How a row ends (template argument of the kernels, from row_end()):
enum RowEnd {
    ROW_FULL = 0,    // every lane's every piece lies inside the row
    ROW_RAGGED = 1,  // pieces end anywhere; D >= VW: the last piece is the 16 bytes that END the row, moved down by the missing values -
                     // one load per piece, whatever the width
    ROW_TINY = 2     // D < VW: value by value
};
template <typename T>
__device__ __forceinline__ Raw<16> piece_load(const T* row, int c, int D, int end) {
    constexpr int VW = RowType<T>::VW;
    if (end == ROW_TINY) return Raw<16>{};
    return *reinterpret_cast<const Raw<16>*>(row + (end == ROW_FULL ? c : (c < D - VW ? c : D - VW)));
}
// the loaded piece's values; 0 from column D on.  last: this piece may hold the row's end (uniform over the lanes)
template <typename T>
__device__ __forceinline__ void piece_values(Raw<16> r, const T* row, int c, int D, int end, bool last, float (&v)[RowType<T>::VW]) {
    constexpr int VW = RowType<T>::VW;
    if (end == ROW_TINY) {
#pragma unroll
        for (int i = 0; i < VW; ++i) v[i] = c + i < D ? RowType<T>::one(row + c + i) : 0.f;
        return;
    }
    if (end == ROW_RAGGED && last) {
        const int missing = (VW - D % VW) % VW;   // uniform
        Raw<16> m = r;
        if (missing & (VW / 2)) m = Raw<16>{m.w[2], m.w[3], 0, 0};
        if (missing & (VW / 4)) m = Raw<16>{m.w[1], m.w[2], m.w[3], 0};
        if (VW == 8 && (missing & 1))
            m = Raw<16>{__builtin_amdgcn_alignbit(m.w[1], m.w[0], 16), __builtin_amdgcn_alignbit(m.w[2], m.w[1], 16),
                        __builtin_amdgcn_alignbit(m.w[3], m.w[2], 16), m.w[3] >> 16};
#pragma unroll
        for (int i = 0; i < 4; ++i) r.w[i] = c + VW <= D ? r.w[i] : (c < D ? m.w[i] : 0u);
    }
    RowType<T>::widen(r, v);
}
template <typename T>
__device__ __forceinline__ void piece_store(T* row, int c, int D, int end, const float (&v)[RowType<T>::VW]) {
    constexpr int VW = RowType<T>::VW;
    if (end == ROW_FULL || (end == ROW_RAGGED && c + VW <= D)) {
        Raw<16> r;
        RowType<T>::narrow(v, r);
        *reinterpret_cast<Raw<16>*>(row + c) = r;
    } else {
#pragma unroll
        for (int i = 0; i < VW; ++i)
            if (c + i < D) RowType<T>::put(row + c + i, v[i]);
    }
}
// VW fp32 parameters at a lane's columns; `none` without an array, 0 from column D on
template <int VW>
__device__ __forceinline__ void param_load(const float* p, int c, int D, int end, bool last, float none, float (&v)[VW]) {
    if (!p) {
#pragma unroll
        for (int i = 0; i < VW; ++i) v[i] = end == ROW_FULL || c + i < D ? none : 0.f;
        return;
    }
#pragma unroll
    for (int h = 0; h < VW; h += 4) {
        if (end == ROW_FULL || (D >= 4 && end == ROW_RAGGED)) {
            float q[4];
            piece_values<float>(piece_load<float>(p, c + h, D, end), p, c + h, D, end, last, q);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[h + i] = q[i];
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[h + i] = c + h + i < D ? p[c + h + i] : 0.f;
        }
    }
}
static inline int row_end(int D, int vw, int columns_of_all_lanes) {
    return D < vw ? ROW_TINY : (D == columns_of_all_lanes ? ROW_FULL : ROW_RAGGED);
}

// ---- reductions over 2^k neighbouring lanes, every lane gets the result ------------------------------------------------------------
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xf, 0xf, true);
}
template <int LANES, typename OP>
__device__ __forceinline__ uint32_t lanes_reduce(uint32_t v, OP op) {
    if constexpr (LANES >= 2) v = op(v, dpp<0xB1>(v));        // quad_perm 1,0,3,2
    if constexpr (LANES >= 4) v = op(v, dpp<0x4E>(v));        // quad_perm 2,3,0,1
    if constexpr (LANES >= 8) v = op(v, dpp<0x141>(v));       // row_half_mirror: the other quad of 8 (all lanes of a quad agree)
    if constexpr (LANES >= 16) v = op(v, dpp<0x140>(v));      // row_mirror: the other half of 16
    if constexpr (LANES >= 32) {
        const auto p = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        v = op(p[0], p[1]);
    }
    if constexpr (LANES >= 64) {
        const auto p = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        v = op(p[0], p[1]);
    }
    return v;
}
template <int LANES>
__device__ __forceinline__ float lanes_sum(float v) {
    return __uint_as_float(lanes_reduce<LANES>(__float_as_uint(v), [](uint32_t a, uint32_t b) {
        return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
    }));
}
template <int LANES>
__device__ __forceinline__ uint32_t lanes_max(uint32_t v) {
    return lanes_reduce<LANES>(v, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
}

// ---- 8-bit blocks -----------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t act8_byte(uint32_t top) {
    const uint32_t e = (top + 0x1fffffu) >> 23;
    return e > 18u ? e - 8u : 10u;
}
__device__ __forceinline__ float act8_inverse(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }
__device__ __forceinline__ float act8_scale(uint32_t byte) { return __uint_as_float(byte << 23); }

// four values -> four codes (the lowest byte is the first).  Any values:
__device__ __forceinline__ uint32_t act8_codes_any(const float* x, float inv, float cap) {
    float v[4];
    uint32_t bad = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if ((__float_as_uint(x[i]) & 0x7fffffffu) >= 0x7f800000u) bad |= 0x7fu << (8 * i);
        v[i] = fminf(fmaxf(x[i], -cap), cap) * inv;
        v[i] = v[i] > 0.f ? fmaxf(v[i], 0x1p-9f) : v[i];
    }
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
    r = __builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], r, true);
    return (uint32_t)r | bad;
}
// ... all of them finite, at most the cap and at least 2^-9 of the scale: the conversion alone
__device__ __forceinline__ uint32_t act8_codes_plain(const float* x, float inv) {
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(x[0] * inv, x[1] * inv, 0, false);
    r = __builtin_amdgcn_cvt_pk_fp8_f32(x[2] * inv, x[3] * inv, r, true);
    return (uint32_t)r;
}
// four codes -> their values
__device__ __forceinline__ void act8_values(uint32_t codes, float scale, float* v) {
    const f32x2_t a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(codes, scale, false), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(codes, scale, true);
    v[0] = a[0];
    v[1] = a[1];
    v[2] = b[0];
    v[3] = b[1];
}

// where a block's scale byte lies: 8 rows side by side ([ceil(M / 8)][blocks][8 rows], ld bytes per 8 rows), so that the weight gradient's
// lane - one block, 8 rows - reads its scales in one piece
template <typename B>
__device__ __forceinline__ B* act8_scale_at(B* scales, int64_t ld, int64_t row, int c) {
    return scales + (row >> 3) * ld + (c / kAct8Block) * 8 + (row & 7);
}

// a lane's VW values of type T at columns [c, c + VW) of a block it shares with its 32 / VW - 1 neighbours -> codes and (first lane) the scale byte.
// Every lane of the block takes part, whatever its columns (values from D on are zeros); columns from D on get code 0.
template <typename T>
__device__ __forceinline__ void act8_store(const float (&v)[RowType<T>::VW], int c, int Dp, uint8_t* codes, uint8_t* scale) {
    constexpr int VW = RowType<T>::VW;
    constexpr uint32_t CAP = RowType<T>::CAP;
    // magnitudes as integers: NaN and infinity are the largest.  3.5 vector operations per value unless a lane of the wave holds a bad, a
    // huge or a tiny (zero) value; then the block's maximum is taken again over the finite ones.
    uint32_t top = 0, low = 0xffffffffu;
#pragma unroll
    for (int i = 0; i < VW; ++i) {
        const uint32_t a = __float_as_uint(v[i]) & 0x7fffffffu;
        top = a > top ? a : top;
        low = a < low ? a : low;
    }
    top = lanes_max<kAct8Block / VW>(top);
    const bool odd = top > CAP;   // (uniform over the block's lanes)
    if (odd) {
        top = 0;
#pragma unroll
        for (int i = 0; i < VW; ++i) {
            uint32_t a = __float_as_uint(v[i]) & 0x7fffffffu;
            a = a >= 0x7f800000u ? 0u : (a < CAP ? a : CAP);
            top = a > top ? a : top;
        }
        top = lanes_max<kAct8Block / VW>(top);
    }
    const uint32_t byte = act8_byte(top);
    const float inv = act8_inverse(byte);
    uint32_t w[VW / 4];
    if (odd || low < (byte - 9u) << 23) {
#pragma unroll
        for (int h = 0; h < VW / 4; ++h) w[h] = act8_codes_any(v + 4 * h, inv, __uint_as_float(CAP));
    } else {
#pragma unroll
        for (int h = 0; h < VW / 4; ++h) w[h] = act8_codes_plain(v + 4 * h, inv);
    }
    if (c < Dp) {
        if constexpr (VW == 4) *reinterpret_cast<uint32_t*>(codes + c) = w[0];
        else *reinterpret_cast<uint2*>(codes + c) = make_uint2(w[0], w[1]);
        if ((c & (kAct8Block - 1)) == 0) *scale = (uint8_t)byte;
    }
}

// host: the types of a row
static inline int row_type_size(int t) { return t == PCVAE_ROW_F32 ? 4 : 2; }
// codes [M, ldc >= ceil(D / 32) * 32] at a multiple of 16 bytes, scale bytes [ceil(M / 8), lds >= 8 ceil(D / 32)] at a
// multiple of 8 (error.cpp)
int act8_check(const char* who, const uint8_t* codes, int64_t ldc, const uint8_t* scales, int64_t lds, int64_t M, int64_t D);
static inline bool row_type_ok(int t) { return t == PCVAE_ROW_F32 || t == PCVAE_ROW_BF16 || t == PCVAE_ROW_F16; }

}  // namespace pcvae
