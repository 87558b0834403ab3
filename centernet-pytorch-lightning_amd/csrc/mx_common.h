// Block-scaled ("MX") storage: up to 32 consecutive channels of a row share one power-of-two scale.
//
//   scale byte b: 2^(b - 127), 255 = not a number (the block held an infinity or a NaN: every value it stands for is a NaN)
//   e4m3 codes: 1 byte, sign / 4 exponent / 3 significand bits, largest finite 448
//   e2m1 codes: 4 bits (two to a byte, the even channel in the low half), values 0 .5 1 1.5 2 3 4 6
//   codes [rows][Cp * bits / 8] with Cp = C rounded up to 32 (the filler stands for zeros), scales [rows][Cp / 32],
//   sign bits (optional) [rows][Cp / 8]: bit j of byte i = (source[8 i + j] > 0)
#pragma once
#include "common.h"

#define MX_BLOCK 32
#define MX_MAX_C 65536            // chunk arithmetic below stays in 32 bits

typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef unsigned short u16x2_t __attribute__((ext_vector_type(2)));
// 16 bytes at any 2- / 4-byte aligned address: rows of an odd number of channels start anywhere, and the hardware loads and stores
// such vectors in one instruction all the same
typedef uint32_t u32x4_a2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));

// Exponent byte of a block's scale from the bits of its largest magnitude a (as float): the least power of two for which a / scale
// rounds to a finite element.  The elements' top binade ends where rounding would carry past the largest one — at 1.75 * 2^emax for
// e2m1 (the tie 7 would go to 8), just above 1.8125 * 2^emax for e4m3 (the tie 464 goes to 448) — so adding the distance from there to
// 2 makes the significand carry into the exponent exactly when the next scale is needed.
template <int FMT> __device__ static inline uint32_t mx_scale_byte(uint32_t abs_bits) {
    constexpr uint32_t carry = FMT == CN_MX_E2M1 ? 0x200000u : 0x17ffffu;
    constexpr int emax = FMT == CN_MX_E2M1 ? 2 : 8;
    const int e = (int)((abs_bits + carry) >> 23) - emax;
    return abs_bits >= 0x7f800000u ? 255u : (uint32_t)(e > 0 ? e : 0);
}
// 2^(b - 127) as float (b = 0: subnormal; 255: NaN)
__device__ static inline float mx_scale_value(uint32_t b) {
    return __uint_as_float(b == 255u ? 0x7fc00000u : (b == 0u ? 0x00400000u : b << 23));
}
// 2^(127 - b) for a finite scale byte (b <= 253 by construction: normal)
__device__ static inline float mx_scale_inverse(uint32_t b) { return __uint_as_float((254u - b) << 23); }

// bitwise maximum over the four lanes of a quad
__device__ static inline uint32_t quad_max_u(uint32_t v) {
    const uint32_t a = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, true);      // quad_perm [1,0,3,2]
    v = a > v ? a : v;
    const uint32_t b = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, true);      // quad_perm [2,3,0,1]
    return b > v ? b : v;
}

// eight consecutive elements of a row as floats, zero behind the row's end (`left` = channels from here to the end, may be <= 0)
__device__ static inline void mx_load8(const float* p, int left, float (&v)[8]) {
    if (left >= 8) {
        const u32x4_t a = *reinterpret_cast<const u32x4_a4*>(p), b = *reinterpret_cast<const u32x4_a4*>(p + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) { v[i] = __uint_as_float(a[i]); v[4 + i] = __uint_as_float(b[i]); }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < left ? p[i] : 0.f;
    }
}
__device__ static inline void mx_load8(const bf16_t* p, int left, float (&v)[8]) {
    if (left >= 8) {
        const u32x4_t a = *reinterpret_cast<const u32x4_a2*>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(a[i] << 16); v[2 * i + 1] = __uint_as_float(a[i] & 0xffff0000u); }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < left ? bf2f(p[i]) : 0.f;
    }
}
__device__ static inline void mx_store8(float* p, int left, const float (&v)[8]) {
    if (left >= 8) {
        *reinterpret_cast<u32x4_a4*>(p) = u32x4_t{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
        *reinterpret_cast<u32x4_a4*>(p + 4) = u32x4_t{__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7])};
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) if (i < left) p[i] = v[i];
    }
}
__device__ static inline void mx_store8(bf16_t* p, int left, const float (&v)[8]) {
    if (left >= 8) {
        *reinterpret_cast<u32x4_a2*>(p) = u32x4_t{pk_bf16(v[0], v[1]), pk_bf16(v[2], v[3]), pk_bf16(v[4], v[5]), pk_bf16(v[6], v[7])};
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) if (i < left) p[i] = f2bf(v[i]);
    }
}

__device__ static inline uint32_t mx_absmax8(const float (&v)[8]) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) { const uint32_t a = __float_as_uint(v[i]) & 0x7fffffffu; m = a > m ? a : m; }
    return m;
}
// codes of eight values on scale byte b (255: zeros); e2m1 -> 4 bytes, e4m3 -> 8 bytes.  Both conversions round to nearest even, and
// the scale is an exact power of two: one rounding in all.
__device__ static inline uint32_t mx_codes_e2m1(const float (&v)[8], uint32_t b) {
    const float s = mx_scale_value(b);
    uint32_t r = 0;
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[0], v[1], s, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[2], v[3], s, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[4], v[5], s, 2);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[6], v[7], s, 3);
    return b == 255u ? 0u : r;
}
__device__ static inline uint2 mx_codes_e4m3(const float (&v)[8], uint32_t b) {
    const float s = b == 255u ? 0.f : mx_scale_inverse(b);
    int lo = 0, hi = 0;
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * s, v[1] * s, lo, false);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[2] * s, v[3] * s, lo, true);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[4] * s, v[5] * s, hi, false);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[6] * s, v[7] * s, hi, true);
    return b == 255u ? make_uint2(0u, 0u) : make_uint2((uint32_t)lo, (uint32_t)hi);
}
// Eight consecutive elements as they lie in memory, so that several loads can be in flight before the first is unpacked (an exec-masked
// branch would make the compiler wait for every load before the next: these have none).  `left`: channels of the row from here on (may
// be <= 0), `ok`: the row exists; what is not there reads as zero.  FULL: the row has a multiple of 8 channels, so a chunk lies inside
// it or outside.  Otherwise the row's last chunk is read eight elements before the row's end and shifted down; rows of fewer than eight
// channels (C < 8, the same for all lanes) are read element by element.
// A load leaves raw bits and what is wrong with them (s: elements to shift down, 8: nothing was there); `fix` puts that right, at the time
// of use — done at once it would make every load wait for the one before.
__device__ static inline u32x4_t mx_pick(bool c, u32x4_t a, u32x4_t b) { return u32x4_t{c ? a.x : b.x, c ? a.y : b.y, c ? a.z : b.z, c ? a.w : b.w}; }
// MX_LOADS_OUT() ends a batch of loads: without it the scheduler moves a first use between them, and its wait with it.
#define MX_LOADS_OUT() __builtin_amdgcn_sched_barrier(0)
template <typename T> struct MxRaw8;
template <> struct MxRaw8<bf16_t> {
    u32x4_t a;
    int s;
    template <bool FULL> __device__ inline void load(const bf16_t* base, int64_t at, int left, bool ok, int C) {
        ok = ok && left > 0;
        if (!FULL && C < 8) {
            uint32_t e[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) e[i] = ok && i < left ? base[at + i] : 0u;
            a = u32x4_t{e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16};
            s = 0;
            return;
        }
        s = !ok ? 8 : (FULL || left >= 8 ? 0 : 8 - left);
        a = *reinterpret_cast<const u32x4_a2*>(base + (ok ? at - s : 0));
    }
    template <bool FULL> __device__ inline void fix() {
        const uint32_t m = s & 8 ? 0u : 0xffffffffu;
        if (!FULL) {
            u32x4_t v = mx_pick(s & 4, u32x4_t{a.z, a.w, 0u, 0u}, a);
            v = mx_pick(s & 2, u32x4_t{v.y, v.z, v.w, 0u}, v);
            const uint32_t h = (s & 1) * 16;
            a = u32x4_t{__builtin_amdgcn_alignbit(v.y, v.x, h), __builtin_amdgcn_alignbit(v.z, v.y, h), __builtin_amdgcn_alignbit(v.w, v.z, h), v.w >> h};
        }
        a = u32x4_t{a.x & m, a.y & m, a.z & m, a.w & m};
    }
    __device__ inline void get(float (&f)[8]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) { f[2 * i] = __uint_as_float(a[i] << 16); f[2 * i + 1] = __uint_as_float(a[i] & 0xffff0000u); }
    }
    // bits (as float) of the largest magnitude: the order of the 16-bit magnitudes is theirs
    __device__ inline uint32_t absmax() const {
        u16x2_t m = {0, 0};
#pragma unroll
        for (int i = 0; i < 4; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2_t, a[i] & 0x7fff7fffu));
        return (uint32_t)(m.x > m.y ? m.x : m.y) << 16;
    }
    __device__ inline uint32_t codes_e2m1(uint32_t scale) const {
        float f[8];
        get(f);
        return mx_codes_e2m1(f, scale);
    }
};
template <> struct MxRaw8<float> {
    u32x4_t a, b;
    int s;
    template <bool FULL> __device__ inline void load(const float* base, int64_t at, int left, bool ok, int C) {
        ok = ok && left > 0;
        if (!FULL && C < 8) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                a[i] = ok && i < left ? __float_as_uint(base[at + i]) : 0u;
                b[i] = ok && i + 4 < left ? __float_as_uint(base[at + i + 4]) : 0u;
            }
            s = 0;
            return;
        }
        s = !ok ? 8 : (FULL || left >= 8 ? 0 : 8 - left);
        const float* p = base + (ok ? at - s : 0);
        a = *reinterpret_cast<const u32x4_a4*>(p);
        b = *reinterpret_cast<const u32x4_a4*>(p + 4);
    }
    template <bool FULL> __device__ inline void fix() {
        const u32x4_t z = {0u, 0u, 0u, 0u};
        if (!FULL) {
            a = mx_pick(s & 4, b, a);
            b = mx_pick(s & 4, z, b);
            const u32x4_t a2 = {a.z, a.w, b.x, b.y}, b2 = {b.z, b.w, 0u, 0u};
            a = mx_pick(s & 2, a2, a);
            b = mx_pick(s & 2, b2, b);
            const u32x4_t a1 = {a.y, a.z, a.w, b.x}, b1 = {b.y, b.z, b.w, 0u};
            a = mx_pick(s & 1, a1, a);
            b = mx_pick(s & 1, b1, b);
        }
        const uint32_t m = s & 8 ? 0u : 0xffffffffu;
        a = u32x4_t{a.x & m, a.y & m, a.z & m, a.w & m};
        b = u32x4_t{b.x & m, b.y & m, b.z & m, b.w & m};
    }
    __device__ inline void get(float (&f)[8]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) { f[i] = __uint_as_float(a[i]); f[4 + i] = __uint_as_float(b[i]); }
    }
    __device__ inline uint32_t absmax() const {
        float f[8];
        get(f);
        return mx_absmax8(f);
    }
    __device__ inline uint32_t codes_e2m1(uint32_t scale) const {
        float f[8];
        get(f);
        return mx_codes_e2m1(f, scale);
    }
};
// store of eight elements of such a row (FULL as above)
template <bool FULL, typename T> __device__ static inline void mx_store8f(T* p, int left, const float (&v)[8]) {
    if (FULL) { if (left > 0) mx_store8(p, 8, v); }
    else mx_store8(p, left, v);
}

// the eight values that 8 bytes of e4m3 codes stand for
__device__ static inline void mx_values_e4m3(uint32_t lo, uint32_t hi, float s, float (&v)[8]) {
    f32x2_t p = __builtin_amdgcn_cvt_pk_f32_fp8((int)lo, false); v[0] = p.x * s; v[1] = p.y * s;
    p = __builtin_amdgcn_cvt_pk_f32_fp8((int)lo, true);          v[2] = p.x * s; v[3] = p.y * s;
    p = __builtin_amdgcn_cvt_pk_f32_fp8((int)hi, false);         v[4] = p.x * s; v[5] = p.y * s;
    p = __builtin_amdgcn_cvt_pk_f32_fp8((int)hi, true);          v[6] = p.x * s; v[7] = p.y * s;
}
__device__ static inline void mx_values_e2m1(uint32_t c, float s, float (&v)[8]) {
    f32x2_t p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.f, 0); v[0] = p.x * s; v[1] = p.y * s;
    p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.f, 1);         v[2] = p.x * s; v[3] = p.y * s;
    p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.f, 2);         v[4] = p.x * s; v[5] = p.y * s;
    p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.f, 3);         v[6] = p.x * s; v[7] = p.y * s;
}

// a launch has less than 2^32 threads along x (the runtime's limit); what would need more is refused before anything runs
static inline bool mx_grid_fits(int64_t workgroups, int threads) { return workgroups < ((int64_t)1 << 32) / threads; }

// n / d for n * d < 2^32 by one high multiplication (m = ceil(2^32 / d); d = 1 has m = 0)
struct MxDiv { uint32_t d, m; };
static inline MxDiv mx_div(uint32_t d) { return MxDiv{d, d == 1 ? 0u : (uint32_t)(((1ull << 32) + d - 1) / d)}; }
__device__ static inline uint32_t mx_quot(uint32_t n, MxDiv v) { return v.m ? __umulhi(n, v.m) : n; }
