// The 8-bit KV cache's pages: their layout, their scales and the exact conversions.
//
// A page holds bs tokens of one kv-head: K, then V, each bs * D bytes of q + 128 with q in
// [-127, 127], and one code byte for each of the two. A value is q * 2^(code - 127):
//   * code = e + 127 for the smallest e with rne(amax / 2^e) <= 127, amax the page's largest
//     magnitude, within the range whose multiples up to 127 are all numbers of the element type
//     (fp16: e in [-24, 9], bf16: e in [-126, 121]). With a power of two the division, the product
//     and the growth of a scale are exact, a value read back is exact in 16 bits, and tokens kept
//     while a scale grows (by a factor of two at least each time) are off by less than one step of
//     the last scale in all: 1/2 (1 + 1/2 + 1/4 + ...). A free scale amax / 127 would save up to a
//     bit once, but costs half a step at every growth, and a page of 16 tokens may grow 15 times.
//   * code 255: a value that is not finite was written; every value of the page is NaN.
//   * code 0: nothing was written; every value is 0.
//
// K is stored [D / 64][bs][64] (64 dims of a token are one 64-byte run, a 16-token load of the
// attention is contiguous per page), V token-minor [D][bs]: the attention contracts P.V over tokens,
// and a lane's operand there is consecutive tokens of one dim.
#pragma once

#include "common.h"
#include "w8a16_tiles.h"

namespace mx {
namespace kv8 {

struct Pages {
    uint8_t* data;   // [num_blocks][Hkv][2][bs * D]
    uint8_t* codes;  // [num_blocks][Hkv][2]
    int Hkv, num_blocks;
};

// Byte offset of the K run (kind 0) or V run (kind 1) of page (phys, head); its code is at
// (phys * Hkv + head) * 2 + kind.
template <int D, int BS>
__device__ __forceinline__ int64_t run_offset(const Pages& p, int phys, int head, int kind) {
    return (((int64_t)phys * p.Hkv + head) * 2 + kind) * (BS * D);
}
__device__ __forceinline__ int64_t code_offset(const Pages& p, int phys, int head, int kind) {
    return ((int64_t)phys * p.Hkv + head) * 2 + kind;
}

constexpr int kPoison = 255;

// The scale of a code as fp32: 2^(code - 127), 0 for 0, NaN for 255.
__device__ __forceinline__ float scale_of(int code) {
    return __uint_as_float(code == kPoison ? 0x7fc00000u : (uint32_t)code << 23);
}

// The code of a page whose largest magnitude has the 16-bit pattern `bits` (sign cleared).
template <bool BF16>
__device__ __forceinline__ int code_of(uint32_t bits) {
    constexpr uint32_t kInf = BF16 ? 0x7f80u : 0x7c00u;
    constexpr int kLo = BF16 ? 1 : 103, kHi = BF16 ? 248 : 136;
    const uint32_t f = BF16 ? bits << 16 : __float_as_uint((float)__builtin_bit_cast(_Float16, (uint16_t)bits));
    // m 2^k, m in [1, 2): m 2^6 rounds to at most 127 below m = 1 + 127/128 (127.5 goes to 128).
    const int code = (int)(f >> 23) - 6 + ((f & 0x7fffffu) >= 0x7f0000u ? 1 : 0);
    return bits >= kInf ? kPoison : (code < kLo ? kLo : (code > kHi ? kHi : code));
}

// 16-bit pattern -> fp32.
template <bool BF16>
__device__ __forceinline__ float widen(uint32_t bits) {
    if constexpr (BF16) return __uint_as_float(bits << 16);
    return (float)__builtin_bit_cast(_Float16, (uint16_t)bits);
}

// Quantising at a run's scale: q = rne(x / 2^e), at most 127 in magnitude. x is clamped to 127 * 2^e
// first (only the largest fp16 numbers need it, where e has reached its cap; a NaN comes out finite), then
// one fused multiply-add puts q + 128 into the low byte: its product is exact and its sum is rounded, to
// nearest even, at the units' place. A poisoned run stores q = 0.
struct Quant {
    float inv, lim;
    __device__ __forceinline__ explicit Quant(int code) {
        const bool poisoned = code == kPoison;
        inv = __uint_as_float(poisoned ? 0u : (uint32_t)(254 - code) << 23);
        lim = poisoned ? 0.0f : 127.0f * __uint_as_float((uint32_t)code << 23);
    }
    __device__ __forceinline__ uint32_t byte(float x) const {  // in the low byte; the others are not 0
        constexpr float kUnits = 12582912.0f + 128.0f;  // 1.5 * 2^23: units' place is the last bit
        return __float_as_uint(__builtin_fmaf(__builtin_amdgcn_fmed3f(x, -lim, lim), inv, kUnits));
    }
    __device__ __forceinline__ uint32_t word(float x0, float x1, float x2, float x3) const {
        const uint32_t lo = __builtin_amdgcn_perm(byte(x1), byte(x0), 0x00000400u);
        const uint32_t hi = __builtin_amdgcn_perm(byte(x3), byte(x2), 0x00000400u);
        return __builtin_amdgcn_perm(hi, lo, 0x05040100u);
    }
};

// Four kept bytes at a run's new, larger scale: rne(q 2^(old - now)). old = 0: nothing was there.
__device__ __forceinline__ uint32_t requant4(uint32_t w, float factor) {
    uint32_t out = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float q = (float)((w >> (8 * i)) & 0xffu) - 128.0f;
        out |= (uint32_t)((int)__builtin_rintf(q * factor) + 128) << (8 * i);
    }
    return out;
}
__device__ __forceinline__ float growth_factor(int old, int now) {
    const int e = 127 + old - now;
    return old == 0 || e <= 0 ? 0.0f : __uint_as_float((uint32_t)e << 23);
}

// 8 bytes -> the 8 integers q as numbers of the element type, exact: a byte permute and half a packed add
// per pair in fp16, a conversion and half a permute per byte in bf16.
template <bool BF16>
__device__ __forceinline__ half8v ints8(uint32_t d0, uint32_t d1) {
    if constexpr (!BF16) {
        return w8a16::dequant8(d0, d1);
    } else {
        uint32_t out[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t w = (i < 2 ? d0 : d1) ^ 0x80808080u;  // q + 128 -> q in two's complement
            const uint32_t lo = __float_as_uint((float)(int8_t)(w >> (16 * (i & 1))));
            const uint32_t hi = __float_as_uint((float)(int8_t)(w >> (16 * (i & 1) + 8)));
            out[i] = __builtin_amdgcn_perm(hi, lo, 0x07060302u);
        }
        return __builtin_bit_cast(half8v, uint4{out[0], out[1], out[2], out[3]});
    }
}

// What a byte stands for in an operand of one permute or conversion: q + kRawBias (0x64nn is the fp16
// number 1024 + nn).
template <bool BF16>
constexpr float kRawBias = BF16 ? 128.0f : 1152.0f;

// A page's scale as a multiplier of such numbers: (q + kRawBias) s - kRawBias s, fused, is q s exactly
// while kRawBias s is a finite number of the type: e <= 5 in fp16, e <= 120 in bf16. `excess` is the rest
// of a larger scale (at most 2^4), for the other operand.
template <bool BF16>
struct RawScale {
    float s, bias, excess;
    RawScale() = default;
    __device__ __forceinline__ explicit RawScale(int code) {
        constexpr int kMost = BF16 ? 127 + 120 : 127 + 5;
        const int c = code == kPoison || code <= kMost ? code : kMost;
        s = scale_of(c);
        bias = -kRawBias<BF16> * s;
        excess = __uint_as_float((uint32_t)(127 + (code == kPoison ? 0 : code - c)) << 23);
    }
};

// 4 bytes at page scale a and 4 at b -> 8 values of the element type (but for the scales' excess), exact.
template <bool BF16>
__device__ __forceinline__ half8v scaled4x2(uint32_t d0, uint32_t d1, const RawScale<BF16>& a, const RawScale<BF16>& b) {
    if constexpr (!BF16) {
        const _Float16 sa = (_Float16)a.s, sb = (_Float16)b.s, ba = (_Float16)a.bias, bb = (_Float16)b.bias;
        const uint4 raw{__builtin_amdgcn_perm(w8a16::kMagic, d0, w8a16::kSelLo),
                        __builtin_amdgcn_perm(w8a16::kMagic, d0, w8a16::kSelHi),
                        __builtin_amdgcn_perm(w8a16::kMagic, d1, w8a16::kSelLo),
                        __builtin_amdgcn_perm(w8a16::kMagic, d1, w8a16::kSelHi)};
        return __builtin_elementwise_fma(__builtin_bit_cast(half8v, raw), half8v{sa, sa, sa, sa, sb, sb, sb, sb},
                                         half8v{ba, ba, ba, ba, bb, bb, bb, bb});
    } else {
        // q s has at most 8 significant bits: the upper half of its fp32 pattern is the bf16 value.
        uint32_t out[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t w = i < 2 ? d0 : d1;
            const RawScale<BF16>& r = i < 2 ? a : b;
            const float lo = __builtin_fmaf((float)((w >> (16 * (i & 1))) & 0xffu), r.s, r.bias);
            const float hi = __builtin_fmaf((float)((w >> (16 * (i & 1) + 8)) & 0xffu), r.s, r.bias);
            out[i] = __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
        }
        return __builtin_bit_cast(half8v, uint4{out[0], out[1], out[2], out[3]});
    }
}

// 4 bytes at scale s0 and 4 at s1 (scale_of) -> 8 values of the element type, exact.
template <bool BF16>
__device__ __forceinline__ half8v values4x2(uint32_t d0, uint32_t d1, float s0, float s1) {
    if constexpr (!BF16) {
        const _Float16 a = (_Float16)s0, b = (_Float16)s1;
        return w8a16::dequant8(d0, d1) * half8v{a, a, a, a, b, b, b, b};
    } else {
        // q s has at most 8 significant bits: the upper half of its fp32 pattern is the bf16 value.
        uint32_t out[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t w = i < 2 ? d0 : d1;
            const float s = i < 2 ? s0 : s1;
            const float lo = ((float)((w >> (16 * (i & 1))) & 0xffu) - 128.0f) * s;
            const float hi = ((float)((w >> (16 * (i & 1) + 8)) & 0xffu) - 128.0f) * s;
            out[i] = __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
        }
        return __builtin_bit_cast(half8v, uint4{out[0], out[1], out[2], out[3]});
    }
}
template <bool BF16>
__device__ __forceinline__ half8v values8(uint32_t d0, uint32_t d1, float s) {
    return values4x2<BF16>(d0, d1, s, s);
}

// Largest 16-bit half of v over the wave (every lane gets it): row rotations, then row exchanges.
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_max(uint32_t m) {
    const uint32_t t = (uint32_t)__builtin_amdgcn_mov_dpp((int)m, CTRL, 0xf, 0xf, false);
    return t > m ? t : m;
}
__device__ __forceinline__ uint32_t wave_max_u16x2(uint32_t v) {
    uint32_t m = (v & 0xffffu) > (v >> 16) ? (v & 0xffffu) : v >> 16;
    m = dpp_max<0x128>(m);  // row_ror:8, 4, 2, 1
    m = dpp_max<0x124>(m);
    m = dpp_max<0x122>(m);
    m = dpp_max<0x121>(m);
    float a = __uint_as_float(m), b = a;
    row_swap16(a, b);
    m = __float_as_uint(a) > __float_as_uint(b) ? __float_as_uint(a) : __float_as_uint(b);
    a = b = __uint_as_float(m);
    row_swap32(a, b);
    return __float_as_uint(a) > __float_as_uint(b) ? __float_as_uint(a) : __float_as_uint(b);
}
typedef uint16_t u16x2v __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
    const u16x2v x = __builtin_bit_cast(u16x2v, a), y = __builtin_bit_cast(u16x2v, b);
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(x, y));
}

// Host: whether the kernels hold these pages, whose byte offsets are 64-bit.
inline int check_pages(const char* what, const void* data, const void* codes, int32_t Hkv, int32_t D, int32_t bs,
                       int32_t num_blocks) {
    if (!data || !codes) return fail(MX_ERR_NULL, "%s: null pointer", what);
    if (D != 64 && D != 128) return fail(MX_ERR_UNSUPPORTED, "%s: head_dim %d unsupported (64 or 128)", what, D);
    if (bs != 4 && bs != 8 && bs != 16 && bs != 32)
        return fail(MX_ERR_UNSUPPORTED, "%s: block_size %d unsupported (4, 8, 16 or 32)", what, bs);
    if (Hkv < 1 || num_blocks < 1) return fail(MX_ERR_INVALID, "%s: Hkv and num_blocks must be >= 1", what);
    if ((double)num_blocks * Hkv * 2 * bs * D > 9e18) return fail(MX_ERR_UNSUPPORTED, "%s: too many pages", what);
    if (!aligned(data, 16)) return fail(MX_ERR_ALIGNMENT, "%s: pages must be 16-byte aligned", what);
    return MX_OK;
}

// CALL(D, BS) with the pages' sizes as constants (check_pages has passed).
#define MX_KV8_DISPATCH(D, BS, CALL)                                  \
    switch ((D) * 100 + (BS)) {                                       \
        case 12804: { CALL(128, 4); break; }                          \
        case 12808: { CALL(128, 8); break; }                          \
        case 12816: { CALL(128, 16); break; }                         \
        case 12832: { CALL(128, 32); break; }                         \
        case 6404: { CALL(64, 4); break; }                            \
        case 6408: { CALL(64, 8); break; }                            \
        case 6416: { CALL(64, 16); break; }                           \
        case 6432: { CALL(64, 32); break; }                           \
    }

}  // namespace kv8
}  // namespace mx
