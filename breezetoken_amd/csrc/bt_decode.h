// Device helpers of the decode kernels (gqa_decode.hip, gqa_paged.hip).
#pragma once

#include "bt_common.h"

namespace bt {

__device__ __forceinline__ int swz(int row, int slots) { return ((row & 7) * 2) & (slots - 1); }

template <int V>
struct IntConst {
  static constexpr int value = V;
};

// Raw buffer resource over [base, base + bytes): loads past the end return 0,
// so tokens past the valid length need no clamping.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t make_rsrc(const void* base, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), (short)0, (int)bytes, 0x00020000);
}
// K/V are streamed once per call: the non-temporal policy (nt) keeps them from
// displacing reusable lines and measurably raises the stream rate on gfx950.
constexpr int kPolicyStream = 2;  // gfx940+ cache-policy bits: nt
__device__ __forceinline__ u32x4 buf_load16(__amdgpu_buffer_rsrc_t r, uint32_t voff, uint32_t soff) {
  return __builtin_amdgcn_raw_buffer_load_b128(r, (int)voff, (int)soff, kPolicyStream);
}

typedef short short4_t __attribute__((ext_vector_type(4)));

// Scalar (constant-cache) read of a wave-uniform value written by an earlier
// kernel: issued as s_load, so its wait lands at the first use instead of
// forcing a vector load + readfirstlane right away.
template <typename T>
__device__ __forceinline__ T uniform_load(const T* p, int i) {
  return ((const __attribute__((address_space(4))) T*)(p))[i];
}

__device__ __forceinline__ floatx4 mfma16k16(const u32x2& a, const u32x2& b, const floatx4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(short4_t, a),
                                                  __builtin_bit_cast(short4_t, b), c, 0, 0, 0);
}

__device__ __forceinline__ u32x2 lds_read_tr4(const BT_LDS uint16_t* p) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4bf16((BT_LDS bf16x4*)p));
}

}  // namespace bt
