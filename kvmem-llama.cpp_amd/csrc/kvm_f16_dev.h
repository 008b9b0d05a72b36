// kvm_f16_dev.h -- quantised window tiles as f16 matrix-core operands.
#pragma once
#include "kvm_internal.h"

// A byte under 0x64 is the f16 number 1024 + byte, so four values take two v_perm and two
// packed subtractions (exact); the packed product with the f16 scale rounds once, as
// (f16)((float)q * d) does.
__device__ __forceinline__ kvm_f16x2 pf_bits2(uint32_t u) {
    kvm_f16x2 v;
    __builtin_memcpy(&v, &u, 4);
    return v;
}
__device__ __forceinline__ void pf_pairs(uint32_t bytes, kvm_f16x2 &a, kvm_f16x2 &b) {
    a = pf_bits2(__builtin_amdgcn_perm(0x64646464u, bytes, 0x04010400u));
    b = pf_bits2(__builtin_amdgcn_perm(0x64646464u, bytes, 0x04030402u));
}
// 8 int8 quants times one scale
__device__ __forceinline__ kvm_f16x8 pf_q8(uint32_t w0, uint32_t w1, uint32_t dbits) {
    const _Float16 d1 = __builtin_bit_cast(_Float16, (uint16_t)dbits);
    const kvm_f16x2 off = {(_Float16)1152.0f, (_Float16)1152.0f}, d = {d1, d1};
    kvm_f16x2 r[4];
    pf_pairs(w0 ^ 0x80808080u, r[0], r[1]);
    pf_pairs(w1 ^ 0x80808080u, r[2], r[3]);
    kvm_f16x8 o;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        r[i] = (r[i] - off) * d;
        o[2 * i] = r[i][0];
        o[2 * i + 1] = r[i][1];
    }
    return o;
}
// the 8 q4_0 nibbles of a V word (kvm_vq_nib_shift) times their keys' scales
__device__ __forceinline__ kvm_f16x8 pf_q4(uint32_t w, kvm_u32x4 scales) {
    const kvm_f16x2 off = {(_Float16)1032.0f, (_Float16)1032.0f};
    kvm_f16x2 r[4];
    pf_pairs(w & 0x0f0f0f0fu, r[0], r[1]);
    pf_pairs((w >> 4) & 0x0f0f0f0fu, r[2], r[3]);
    kvm_f16x8 o;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        r[i] = (r[i] - off) * pf_bits2(scales[i]);
        o[2 * i] = r[i][0];
        o[2 * i + 1] = r[i][1];
    }
    return o;
}
