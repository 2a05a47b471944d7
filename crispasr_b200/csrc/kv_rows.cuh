// kv_rows.cuh — eight values of a row per lane into a row of a KV cache (F16, Q8_0, Q4_0), and out of one.
#pragma once

#include "fattn_common.cuh"

namespace b200 {

constexpr size_t kv_row_bytes(int type, int hd) {
    return type == B200_TYPE_F16 ? (size_t)hd * 2 : (size_t)hd / 32 * (type == B200_TYPE_Q8_0 ? 34 : 18);
}

// (int)roundf(t) for |t| < 2^22 without either unit's conversions: |t| + 1/2 truncated to an integer by two additions that
// round towards zero (the first cannot reach an integer the exact sum does not reach), then the sign; NaN gives 0.  In a block
// of values below 4e-37 1/d is beyond a float and t infinite: the low byte is that of the saturated conversion, 0xFF for
// +inf, 0 for -inf (a branch for such blocks cost 0.2 us per launch).
__device__ __forceinline__ uint32_t round_away(float t) {
    asm("min.NaN.f32 %0, %0, 0f437F0000;" : "+f"(t));   // 255; a NaN stays one
    const float m = fmaxf(fabsf(t), 0.0f);
    const int32_t k = __float_as_int(__fadd_rz(__fadd_rz(m, 0.5f), 8388608.0f)), sign = __float_as_int(t) >> 31;
    return (uint32_t)((k ^ sign) - sign);
}
// Low bytes of four words.
__device__ __forceinline__ uint32_t low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}
// Four Q4_0 nibbles in the low halves of a word's bytes: trunc(x * id + 8.5), at most 15, for x * id in [-8, 8] up to a rounding.
// The sum is formed on top of 2^22 and rounded towards zero, which leaves a whole number of halves (bit 0 of the result) and cannot
// reach an integer that the exact sum does not reach; 16 becomes 15.  (A NaN gets nibble 14.)
__device__ __forceinline__ uint32_t nibbles_of(float x0, float x1, float x2, float x3, float id) {
    constexpr float kBase = 4194304.0f + 8.5f;
    const uint32_t w = low_bytes(__float_as_uint(__fmaf_rz(x0, id, kBase)), __float_as_uint(__fmaf_rz(x1, id, kBase)), __float_as_uint(__fmaf_rz(x2, id, kBase)),
                                 __float_as_uint(__fmaf_rz(x3, id, kBase)));
    const uint32_t n = (w >> 1) & 0x1F1F1F1Fu;
    return (n - ((n >> 4) & 0x01010101u)) & 0x0F0F0F0Fu;
}
// Whether the first of a block's values of largest magnitude `amax` is negative.  Its values are N in each of LANES neighbouring lanes, in the
// lanes' order, the lane's largest and smallest being hi and lo.
template <int N, int LANES>
__device__ __forceinline__ bool largest_is_negative(const float* x, float hi, float lo, float amax) {
    const int base = threadIdx.x & (32 - LANES);
    const uint32_t pos = __ballot_sync(0xffffffffu, hi == amax) >> base & ((1u << LANES) - 1), neg = __ballot_sync(0xffffffffu, lo == -amax) >> base & ((1u << LANES) - 1);
    bool negative = neg && !pos;
    if (__any_sync(0xffffffffu, pos && neg)) {   // both signs, or nothing but zeros
        uint32_t sign = 0;
#pragma unroll
        for (int i = N - 1; i >= 0; i--)
            if (fabsf(x[i]) == amax) sign = __float_as_uint(x[i]) >> 31;
        sign = __shfl_sync(0xffffffffu, sign, pos | neg ? __ffs(pos | neg) - 1 : 0, LANES);
        if (pos && neg) negative = sign;
    }
    return negative;
}

// Eight values f of a row, [c, c + 8), into the cache row at row_out.  All lanes of the warp call it, four neighbouring lanes
// (from a multiple of four) having the values of a block of 32; a lane that is not `live` stores nothing.
//
// Q8_0 blocks, bit-identical to gguf-py quantize_blocks: d = amax/127 (fp32), stored as fp16; q = roundf(x * (1/d)) with
// 1/d = 0 for d == 0.  A block is 34 bytes.  In a row of an even number of blocks (head_dim 64 / 128: rows start on a 4-byte
// boundary) the quants of the odd blocks fill aligned words and those of the even ones straddle them by two bytes; there a lane
// takes the upper half of its left neighbour's last word (the first lane the scale) and the row leaves in 32-bit stores.
//
// Q4_0 blocks: d = m / -8 (fp32), stored as fp16, m the first of the values of largest magnitude; q = trunc(x * (1/d) + 8.5), at
// most 15.  Byte i holds values i and 16 + i: the lanes with values 0..15 and 16..31 exchange half of their nibbles, after which
// each of the four has a word of the block's 16 bytes.
template <int TYPE>
__device__ __forceinline__ void store_row8(uint8_t* row_out, int c, const float (&f)[8], bool live, int hd) {
    if constexpr (TYPE == B200_TYPE_F16) {
        if (live)
            *reinterpret_cast<uint4*>(row_out + c * 2) =
                make_uint4(pack_half2(f[0], f[1]), pack_half2(f[2], f[3]), pack_half2(f[4], f[5]), pack_half2(f[6], f[7]));
    } else {
        float amax = 0.0f, hi = f[0], lo = f[0];
        if constexpr (TYPE == B200_TYPE_Q4_0) {
#pragma unroll
            for (int i = 1; i < 8; i++) hi = fmaxf(hi, f[i]), lo = fminf(lo, f[i]);
            amax = fmaxf(hi, -lo);
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) amax = fmaxf(amax, fabsf(f[i]));
        }
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        const int blk = c >> 5, i4 = (c & 31) >> 3;   // lane i4 of the block's four
        if constexpr (TYPE == B200_TYPE_Q8_0) {
            const float d = __fdiv_rn(amax, 127.0f);
            const float id = d != 0.0f ? __frcp_rn(d) : 0.0f;
            uint32_t q[8];
#pragma unroll
            for (int i = 0; i < 8; i++) q[i] = round_away(__fmul_rn(f[i], id));
            const uint32_t w0 = low_bytes(q[0], q[1], q[2], q[3]), w1 = low_bytes(q[4], q[5], q[6], q[7]);
            const uint32_t dbits = __half_as_ushort(__float2half_rn(d));
            const uint32_t left = __shfl_up_sync(0xffffffffu, w1, 1);
            if (!live) return;
            uint8_t* out = row_out + blk * 34 + 8 * i4;
            if ((hd & 63) == 0) {
                if (blk & 1) {
                    *reinterpret_cast<uint32_t*>(out + 2) = w0;
                    *reinterpret_cast<uint32_t*>(out + 6) = w1;
                    if (i4 == 0) *reinterpret_cast<uint16_t*>(out) = (uint16_t)dbits;
                } else {
                    *reinterpret_cast<uint32_t*>(out) = (w0 << 16) | (i4 == 0 ? dbits : left >> 16);
                    *reinterpret_cast<uint32_t*>(out + 4) = __funnelshift_l(w0, w1, 16);
                    if (i4 == 3) *reinterpret_cast<uint16_t*>(out + 8) = (uint16_t)(w1 >> 16);
                }
            } else {   // an odd number of blocks: rows are only 2-byte aligned
                *reinterpret_cast<uint16_t*>(out + 2) = (uint16_t)w0;
                *reinterpret_cast<uint16_t*>(out + 4) = (uint16_t)(w0 >> 16);
                *reinterpret_cast<uint16_t*>(out + 6) = (uint16_t)w1;
                *reinterpret_cast<uint16_t*>(out + 8) = (uint16_t)(w1 >> 16);
                if (i4 == 0) *reinterpret_cast<uint16_t*>(out) = (uint16_t)dbits;
            }
        } else {
            // (m / -8 is exact but for denormals, where d is 0 in fp16)
            const float d = amax * (largest_is_negative<8, 4>(f, hi, lo, amax) ? 0.125f : -0.125f);
            const float id = d != 0.0f ? __frcp_rn(d) : 0.0f;
            const uint32_t w0 = nibbles_of(f[0], f[1], f[2], f[3], id), w1 = nibbles_of(f[4], f[5], f[6], f[7], id);
            const bool high = i4 & 2;
            const uint32_t other = __shfl_xor_sync(0xffffffffu, high ? w0 : w1, 2);
            const uint32_t w = high ? other | (w1 << 4) : w0 | (other << 4);
            if (!live) return;
            uint8_t* out = row_out + blk * 18 + 2 + 8 * (i4 & 1) + (high ? 4 : 0);
            if ((hd & 63) == 0 && (blk & 1)) {
                *reinterpret_cast<uint32_t*>(out) = w;
            } else {   // two bytes off a word's boundary
                *reinterpret_cast<uint16_t*>(out) = (uint16_t)w;
                *reinterpret_cast<uint16_t*>(out + 2) = (uint16_t)(w >> 16);
            }
            if (i4 == 0) *reinterpret_cast<uint16_t*>(row_out + blk * 18) = __half_as_ushort(__float2half_rn(d));
        }
    }
}

// The same for lanes that hold four values of each half of a row, f[0..3] = [4 l, 4 l + 4) and f[4..7] = hd/2 + [4 l, 4 l + 4): eight lanes
// (from a multiple of eight) share a block of either half.  hd is 64 or 128, l the lane's place in its row.
template <int TYPE>
__device__ __forceinline__ void store_row4x2(uint8_t* row_out, int l, const float (&f)[8], bool live, int hd) {
    const int i8 = l & 7;
#pragma unroll
    for (int part = 0; part < 2; part++) {
        const float* x = f + 4 * part;
        if constexpr (TYPE == B200_TYPE_F16) {
            if (live) *reinterpret_cast<uint2*>(row_out + part * hd + 8 * l) = make_uint2(pack_half2(x[0], x[1]), pack_half2(x[2], x[3]));
            continue;
        }
        const int blk = (l >> 3) + part * (hd / 64);
        const float hi = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), lo = fminf(fminf(x[0], x[1]), fminf(x[2], x[3]));
        float amax = fmaxf(hi, -lo);
#pragma unroll
        for (int m = 1; m < 8; m <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, m));
        if constexpr (TYPE == B200_TYPE_Q8_0) {
            const float d = __fdiv_rn(amax, 127.0f);
            const float id = d != 0.0f ? __frcp_rn(d) : 0.0f;
            const uint32_t w = low_bytes(round_away(__fmul_rn(x[0], id)), round_away(__fmul_rn(x[1], id)), round_away(__fmul_rn(x[2], id)), round_away(__fmul_rn(x[3], id)));
            const uint32_t dbits = __half_as_ushort(__float2half_rn(d)), left = __shfl_up_sync(0xffffffffu, w, 1);
            if (!live) continue;
            uint8_t* out = row_out + blk * 34 + 4 * i8;
            if (blk & 1) {
                *reinterpret_cast<uint32_t*>(out + 2) = w;
                if (i8 == 0) *reinterpret_cast<uint16_t*>(out) = (uint16_t)dbits;
            } else {   // (the block's quants are two bytes off the words' boundaries)
                *reinterpret_cast<uint32_t*>(out) = (w << 16) | (i8 == 0 ? dbits : left >> 16);
                if (i8 == 7) *reinterpret_cast<uint16_t*>(out + 4) = (uint16_t)(w >> 16);
            }
        } else if constexpr (TYPE == B200_TYPE_Q4_0) {
            const float d = amax * (largest_is_negative<4, 8>(x, hi, lo, amax) ? 0.125f : -0.125f);
            const float id = d != 0.0f ? __frcp_rn(d) : 0.0f;
            uint32_t w = nibbles_of(x[0], x[1], x[2], x[3], id);
            const uint32_t other = __shfl_xor_sync(0xffffffffu, w, 4);   // values 16.. of the block are lanes 4..7's
            w = i8 < 4 ? w | (other << 4) : other | (w << 4);
            if (!live) continue;
            uint8_t* out = row_out + blk * 18;
            *reinterpret_cast<uint16_t*>(out + 2 + 4 * (i8 & 3) + (i8 < 4 ? 0 : 2)) = (uint16_t)(i8 < 4 ? w : w >> 16);
            if (i8 == 0) *reinterpret_cast<uint16_t*>(out) = __half_as_ushort(__float2half_rn(d));
        }
    }
}

// Eight values [c, c + 8) of a row of blocks as they lie in memory, loaded and then converted, so that the loads of several rows can be in flight.  The
// kernel before this one may have written the row.  WORDS: rows on 4-byte boundaries.  The eight quants start 2 + 8 i bytes into
// their block, in odd blocks (34 and 18 bytes) on a word's boundary, in even ones two bytes off one, where a third word makes them up.
template <int TYPE, bool WORDS, bool SHARED = false>
struct Row8 {
    uint32_t w[TYPE == B200_TYPE_F16 ? 4 : 2];
    uint16_t d;

    // (from global memory behind griddepcontrol.wait, or from shared memory)
    template <typename T>
    static __device__ __forceinline__ T get(const T* p) {
        if constexpr (SHARED) return *p;
        else return load_global(p);
    }
    __device__ __forceinline__ void load(const uint8_t* row, int c) {
        if constexpr (TYPE == B200_TYPE_F16) {
            const uint4 u = get(reinterpret_cast<const uint4*>(row + 2 * c));
            w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
        } else {
            const int blk = c >> 5, odd = blk & 1, first = TYPE == B200_TYPE_Q8_0 ? c & 31 : c & 15;
            const uint8_t* p = row + (TYPE == B200_TYPE_Q8_0 ? 34 : 18) * blk;
            if constexpr (WORDS) {
                const uint32_t* x = reinterpret_cast<const uint32_t*>(p + first + 2 * odd);
                w[0] = get(x), w[1] = get(x + 1);
                if (!odd) {
                    const uint32_t last = get(reinterpret_cast<const uint16_t*>(x + 2));
                    w[0] = __funnelshift_r(w[0], w[1], 16), w[1] = __byte_perm(w[1], last, 0x5432);
                }
            } else {
                const uint16_t* x = reinterpret_cast<const uint16_t*>(p + 2 + first);
                w[0] = get(x) | (uint32_t)get(x + 1) << 16, w[1] = get(x + 2) | (uint32_t)get(x + 3) << 16;
            }
            d = get(reinterpret_cast<const uint16_t*>(p));
        }
    }
    __device__ __forceinline__ void values(int c, float (&f)[8]) const {
        if constexpr (TYPE == B200_TYPE_F16) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
                f[2 * i] = p.x, f[2 * i + 1] = p.y;
            }
        } else {
            const float scale = __half2float(__ushort_as_half(d));
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const uint32_t x = w[i >> 2] >> (8 * (i & 3));
                f[i] = scale * (float)(TYPE == B200_TYPE_Q8_0 ? (int)(int8_t)x : (int)(x >> (c & 16 ? 4 : 0) & 15u) - 8);
            }
        }
    }
    // The same rounded to F16 (blocks only): the quants as exact halves, one product, one rounding.
    __device__ __forceinline__ uint4 halves(int c) const {
        uint32_t o[4];
        const __half2 d2 = __half2half2(__ushort_as_half(d));
        // halves 0x64xx = 1024 + xx, less 1152 (int8 with its sign bit flipped) or 1032 (nibbles)
        const __half2 bias = __float2half2_rn(TYPE == B200_TYPE_Q8_0 ? 1152.0f : 1032.0f);
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const uint32_t q = TYPE == B200_TYPE_Q8_0 ? w[k] ^ 0x80808080u : (c & 16 ? w[k] >> 4 : w[k]) & 0x0F0F0F0Fu;
            const uint32_t h01 = __byte_perm(q, 0x64646464u, 0x4140), h23 = __byte_perm(q, 0x64646464u, 0x4342);
            const __half2 v01 = __hmul2(__hsub2(*reinterpret_cast<const __half2*>(&h01), bias), d2);
            const __half2 v23 = __hmul2(__hsub2(*reinterpret_cast<const __half2*>(&h23), bias), d2);
            o[2 * k] = *reinterpret_cast<const uint32_t*>(&v01), o[2 * k + 1] = *reinterpret_cast<const uint32_t*>(&v23);
        }
        return make_uint4(o[0], o[1], o[2], o[3]);
    }
};

// Eight consecutive values out, rounded to F16 or as they are; V16: 16-byte aligned addresses.
template <bool F32, bool V16>
__device__ __forceinline__ void store8(uint8_t* p, const float (&f)[8]) {
    if constexpr (F32 && V16) {
        reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
        reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
    } else if constexpr (F32) {
#pragma unroll
        for (int i = 0; i < 8; i++) reinterpret_cast<float*>(p)[i] = f[i];
    } else if constexpr (V16) {
        *reinterpret_cast<uint4*>(p) = make_uint4(pack_half2(f[0], f[1]), pack_half2(f[2], f[3]), pack_half2(f[4], f[5]), pack_half2(f[6], f[7]));
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) reinterpret_cast<__half*>(p)[i] = __float2half_rn(f[i]);
    }
}

}  // namespace b200
