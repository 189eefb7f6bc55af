// Shared by the block operators (decay.hip, blocknorm.hip, rows8.hip), which take the element type per call: both library
// builds carry bfloat16, IEEE half and float forms of them, so the storage-type switch of vdmi_common.h is undone here.
#pragma once
#include "vdmi_common.h"
#ifdef VDMI_F16
#undef __bf16
#undef __builtin_amdgcn_mfma_f32_32x32x16_bf16
#endif

// a launch has less than 2^32 threads along x
inline bool launch_fits(long long workgroups, int threads) { return workgroups <= 0xffffffffLL / threads; }

template <typename T>
struct Pack;
template <>
struct Pack<__bf16> {
    typedef __attribute__((ext_vector_type(8))) __bf16 x8;
    static constexpr unsigned EXP = 0x7f80u;       // exponent field: all ones in infinities and NaN
};
template <>
struct Pack<_Float16> {
    typedef __attribute__((ext_vector_type(8))) _Float16 x8;
    static constexpr unsigned EXP = 0x7c00u;
};
template <typename T>
using x8_t = typename Pack<T>::x8;

__device__ __forceinline__ f32x16 mfma16(const Pack<__bf16>::x8& a, const Pack<__bf16>::x8& b, const f32x16& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma16(const Pack<_Float16>::x8& a, const Pack<_Float16>::x8& b, const f32x16& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ f32x16 zero16() {
    f32x16 z;
#pragma unroll
    for (int r = 0; r < 16; ++r) z[r] = 0.f;
    return z;
}

// registers 8 s .. 8 s + 7 of an accumulator as a 16-bit operand: 8 contraction values in accumulator-row order
template <typename T>
__device__ __forceinline__ x8_t<T> acc_operand(const f32x16& a, int s) {
    x8_t<T> f;
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = (T)a[8 * s + j];
    return f;
}

// LDS that a wave writes for its own lanes: LDS instructions of a wave execute in order, so all that is needed between the
// writes and the reads of other lanes (and before the next writes) is that the compiler keeps that order, which it need
// not where no lane reads what it wrote itself.
__device__ __forceinline__ void wave_lds_order() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); }

typedef short vdmi_s4 __attribute__((ext_vector_type(4)));

// ds_read_b64_tr_b16: the 16 lanes of a group supply four rows x four 8-byte pieces, and each lane receives one column's
// four values.  Here: contraction values from the four rows at `base` and the four rows `step` bytes further on.
template <typename T>
__device__ __forceinline__ x8_t<T> tr_operand(const char* base, int step) {
    typedef __attribute__((address_space(3))) vdmi_s4* lds_s4;
    const vdmi_s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(base));
    const vdmi_s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(base + step));
    return __builtin_bit_cast(x8_t<T>, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}

// Buffer resources: 32-bit byte offsets from a base; what lies at or past `bytes` loads as zero and is not stored.  NOWHERE:
// an offset past the end of any resource made here (they stay under 2^31 bytes).
constexpr unsigned NOWHERE = 0x80000000u;
typedef __attribute__((ext_vector_type(4))) unsigned vdmi_u4;
typedef __attribute__((ext_vector_type(2))) unsigned vdmi_u2;
__device__ __forceinline__ __amdgpu_buffer_rsrc_t vdmi_rsrc(const void* p, unsigned bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, bytes, 0x00020000);
}
template <typename T>
__device__ __forceinline__ x8_t<T> load16(__amdgpu_buffer_rsrc_t r, unsigned off) {
    return __builtin_bit_cast(x8_t<T>, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0));
}
template <typename T>
__device__ __forceinline__ void store16(__amdgpu_buffer_rsrc_t r, unsigned off, const x8_t<T>& v) {
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(vdmi_u4, v), r, off, 0, 0);
}
