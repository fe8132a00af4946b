// Cache pages held in 4 bits: where a number lies, how a block is rounded, how codes become numbers again.
//
// Every 32 channels of a head's key or value at one position are a block with one scale, a power of two 2^e kept as the byte
// e + 127; a number is a code of sign, two bits of exponent and one of fraction, 0, 0.5, 1, 1.5, 2, 3, 4 or 6, times the scale.
// (The OCP's MXFP4.  gfx950 converts two such codes to bfloat16 or 32 bits with their scale in one instruction, exactly, which is
// what keeps attention over them bound by memory: 4.65 cycles a SIMD for 128 numbers, measured.)
//
// e is the exponent of the block's largest magnitude less 2, and one more where that magnitude in units of 2^e would be over 7:
// such a number would round to 8, which there is none of; from 6 to 7 it rounds to 6.  (Relative error of N(0, 1): 0.112 so, 0.115
// with the exponent as it is, where 7.9 becomes 6, and 0.116 where nothing over 6 is ever cut.)  It is held within -119 .. 125: no
// number that is read back is subnormal or infinite.  A block that holds a NaN or an infinity has the byte 255 and reads as NaN.
// Rounding is to the nearest number, ties to the even code.
//
// Pages of P positions (a power of two, at least 8), bytes:
//     key codes     [page][head][position][D / 2]              channel 2 j in the low half of byte j
//     value codes   [page][head][P / 8][Dv / 2][8]             the same bytes of 8 positions side by side
//     scales        [page][head][P / 8][blocks][8]             of keys and of values, blocks = ceil(channels / 32)
// A key is read whole by the lanes that multiply it; of values a lane wants 8 positions of a few channels.  A position's bytes are
// its own in both, so tokens are written without reading what lies beside them.
#pragma once

#include "common.h"

#define XR_BLOCK4 32

struct Pages4 {
    uint8_t* kc;
    uint8_t* ks;
    uint8_t* vc;
    uint8_t* vs;
};

// what a product's caller passes beside its rotation to have keys and values go to 4-bit pages
struct XrGemmPages4 {
    void *kc, *ks, *vc, *vs;
    int n_pages, n_requests, table_width;
};

struct Write4Sums {
    const float* sums;      // [ranges][T][(H + 2 Hk) * D], 32-bit
    const float* bias;      // [(H + 2 Hk) * D] or null
    int ranges;
    const XrGemmPages4* pages;
    const int* positions;
    const int* req_of_token;
    const int* block_table;
    int table_stride;       // (from a request's row to the next's: a table may be a view of a wider one)
    const float* inv_freq;
    void* q_out;            // [T, H * D] bfloat16
    int T, H, Hk, D, rot, interleaved;     // (pairs that are not neighbours: in paired order)
    float mscale;
    int page_size;
};
// xr_rope_kv_write4 behind a product whose K ranges are still to be added up
int rope_kv_write4_sums(const Write4Sums& w, hipStream_t stream);

__host__ __device__ inline int blocks4(int channels) { return (channels + XR_BLOCK4 - 1) / XR_BLOCK4; }

// byte of a page's scale: `pb` = page * heads + head
__host__ __device__ inline size_t scale_at4(size_t pb, int page_size, int blocks, int off, int block) {
    return ((pb * (size_t)(page_size >> 3) + (off >> 3)) * blocks + block) * 8 + (off & 7);
}
__host__ __device__ inline size_t key_at4(size_t pb, int page_size, int D, int off) { return (pb * page_size + off) * (size_t)(D >> 1); }
// the byte of channel pair `pair`
__host__ __device__ inline size_t value_at4(size_t pb, int page_size, int Dv, int off, int pair) {
    return ((pb * (size_t)(page_size >> 3) + (off >> 3)) * (size_t)(Dv >> 1) + pair) * 8 + (off & 7);
}

// the scale's byte for a block whose largest magnitude has these bits (sign cleared; NaNs are the largest of all)
__device__ inline uint32_t scale_byte4(uint32_t bits) {
    if (bits >= 0x7F800000u) return 255u;
    const int b = (int)((bits + 0x1FFFFFu) >> 23) - 2;
    return (uint32_t)(b < 8 ? 8 : b > 252 ? 252 : b);
}

#if defined(__HIP_DEVICE_COMPILE__)
typedef __bf16 xr_pair_bf16 __attribute__((ext_vector_type(2)));
typedef float xr_pair_f32 __attribute__((ext_vector_type(2)));
// (of the scale's bits only the exponent counts: a byte shifted into place, whatever lies beside it)
template <int BYTE> __device__ __forceinline__ uint32_t pair4_bf16(uint32_t codes, uint32_t scale_bits) {
    union { xr_pair_bf16 b; uint32_t u; } c;
    c.b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, __uint_as_float(scale_bits), BYTE);
    return c.u;
}
template <int BYTE> __device__ __forceinline__ float2 pair4_f32(uint32_t codes, uint32_t scale_bits) {
    const xr_pair_f32 v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, __uint_as_float(scale_bits), BYTE);
    return make_float2(v[0], v[1]);
}
// 8 numbers as a word of codes in units of the scale (0 where the block reads as NaN)
__device__ __forceinline__ uint32_t codes4(const float* x, uint32_t byte) {
    const float s = __uint_as_float(byte << 23);
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], s, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], s, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], s, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], s, 3);
    return byte == 255u ? 0u : w;
}
#else   // the host pass only parses the callers
template <int BYTE> __host__ __device__ inline uint32_t pair4_bf16(uint32_t, uint32_t) { return 0; }
template <int BYTE> __host__ __device__ inline float2 pair4_f32(uint32_t, uint32_t) { return make_float2(0.f, 0.f); }
__host__ __device__ inline uint32_t codes4(const float*, uint32_t) { return 0; }
#endif
