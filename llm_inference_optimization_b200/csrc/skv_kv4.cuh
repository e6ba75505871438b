// The 4-bit page record, shared by the kernels that write, read and attend to it, and the rotary angle.
//
// A record holds 16 tokens of one kv-head in 18 * D bytes: 8 D of key codes, 8 D of value codes, 2 D of scales.  Every
// 32 channels of a row share one bf16 scale = bf16(amax * fp32(1 / 7)) (bf16: as wide a range as fp32, so no row over- or
// underflows it; the codes are made with the ROUNDED scale, so its 8 bits cost nothing but a sliver of the code range);
// code = clamp(rne(x / scale), -7, 7), stored as the nibble code + 8, even nibble low.  An all-zero group has scale 0
// (and one whose scale is below fp32's normal range all codes 0);
// a group that holds a NaN or an infinity has scale NaN, so that whoever attends to it gets NaN and not a plausible number.
//
// The order inside a record is that of the attention kernel's matrix fragments, so that its lanes fetch their operands
// with plain wide shared-memory loads (contiguous over a warp, no bank conflicts, no swizzle, no ldmatrix).  Token
// t = 4i + 2j + e of the page takes row place 8j + 2i + e:
//   keys    byte place * D/2 + c * D/8 + 4w + n/2                       channel 32w + 8c + n   (c < 4, n < 8)
//   values  byte j * 4D + g * D/2 + i * D/8 + e * D/16 + 2w + n/2       channel 32w + 4g + n   (g < 8, n < 4)
//   scales  bf16 element place * D/16 + w (keys), + D/32 (values)       group w < D/32
// One token's bytes are its own: no byte is shared between tokens, so tokens are appended without read-modify-write.
#pragma once

#include "skv_common.cuh"

#define SKV_KV_INT4 3   // kv_dtype: keys and values in 4 bits, page records as above

namespace skv {

constexpr int KV4_PAGE = 16;
template <int D> __host__ __device__ constexpr int kv4_record_bytes() { return 18 * D; }

__device__ __forceinline__ int kv4_place(int t) { return ((t >> 1) & 1) * 8 + (t >> 2) * 2 + (t & 1); }
template <int D> __device__ __forceinline__ int kv4_v_row(int t) {   // byte of token t's first value chunk (g = 0)
    return 8 * D + ((t >> 1) & 1) * 4 * D + (t >> 2) * (D / 8) + (t & 1) * (D / 16);
}
template <int D> __device__ __forceinline__ int kv4_scales(int t) { return 16 * D + kv4_place(t) * (D / 8); }

// cos and sin of position * f times factor, f given as a 64-bit fixed-point fraction of a turn (see rotary.cu).  In 64 bits,
// rounded once: rows quantised behind the rotation then take the same codes as rows rotated by the formula in 64-bit angles
// (a last-bit difference moves one value in ten million over the border between two codes).  One thread of a block works a
// pair out for all heads, so this is a hundredth of the kernels' work.
__device__ __forceinline__ float2 rotary_cos_sin(long long pos, unsigned long long f, double factor) {
    const long long phase = (long long)((unsigned long long)pos * f);
    double sn, cs;
    sincospi((double)phase * 1.0842021724855044e-19, &sn, &cs);   // 2^-63: half turns in [-1, 1)
    return make_float2((float)(cs * factor), (float)(sn * factor));
}
// One pair turned; every product and sum is rounded by itself, in every kernel and at every vector width, as the formula
// written in torch does it.
__device__ __forceinline__ void rotary_turn(float x, float y, float sn, float cs, float& u, float& w) {
    u = __fsub_rn(__fmul_rn(x, cs), __fmul_rn(y, sn));
    w = __fadd_rn(__fmul_rn(y, cs), __fmul_rn(x, sn));
}

}  // namespace skv
