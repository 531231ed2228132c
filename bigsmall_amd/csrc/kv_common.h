// What the paged KV cache's kernels share: element conversions between the
// stored 8-bit types, f16 and bf16, wave reductions, and a step's bounds.
#pragma once

#include <stdint.h>

#include "bigsmall_kv.h"
#include "simt.h"

namespace bs_kv {

constexpr uint32_t PAGE = BS_KV_PAGE;

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef _Float16 half8v __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

__device__ __forceinline__ float bf16_to_f32(uint32_t bits) { return __uint_as_float(bits << 16); }

// Round to nearest even; NaN stays NaN (the canonical one).
__device__ __forceinline__ uint16_t f32_to_bf16(float x) {
  const uint32_t u = __float_as_uint(x);
  return x != x ? (uint16_t)0x7FC0u : (uint16_t)((u + 0x7FFFu + ((u >> 16) & 1u)) >> 16);
}

__device__ __forceinline__ bool bf16_finite(uint32_t bits) { return (bits & 0x7F80u) != 0x7F80u; }

// Four stored codes (a dword) as four f16 values, exactly: both types' values
// need 8 significant bits or fewer and lie below 448. e4m3: one conversion
// instruction per pair. int8: a biased byte u = code + 128 under the f16
// exponent of 1024 is the number 1024 + u; one packed subtraction gives the code.
template <int KIND>
__device__ __forceinline__ void codes_to_f16(uint32_t w, half2v& lo, half2v& hi) {
  if constexpr (KIND == BS_KV_FP8) {
    lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false);
    hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true);
  } else {
    const uint32_t u = w ^ 0x80808080u;
    const half2v off = {(_Float16)1152.0f, (_Float16)1152.0f};
    lo = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) - off;
    hi = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) - off;
  }
}

template <int KIND>
__device__ __forceinline__ half8v codes8_to_f16(uint32_t w0, uint32_t w1) {
  half2v a, b, c, d;
  codes_to_f16<KIND>(w0, a, b);
  codes_to_f16<KIND>(w1, c, d);
  return half8v{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

// A workgroup barrier for LDS only: loads from memory that are under way stay so (__syncthreads waits for them).
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) x = fmaxf(x, __shfl_xor(x, d));
  return x;
}

// p[i] of an array that no kernel of the call writes, at an index that is the same in all lanes: a load through the
// scalar cache, which does not stand in line with the vector loads under way.
template <class T>
__device__ __forceinline__ T uniform_load(const T* p, size_t i) {
  return ((const CST T*)(uintptr_t)p)[i];
}

// The bounds of sequence b in a step, held to what the batch's arrays can hold;
// false (and n = 0) if they make no sense.
struct SeqStep {
  int t0, n, start, len;  // first new row, new rows, cached tokens before, tokens after
};
// SAME: b is the same in all lanes.
template <bool SAME = false>
__device__ __forceinline__ bool seq_step(const bs_kv_batch& B, uint32_t b, SeqStep& s) {
  s.t0 = SAME ? uniform_load(B.cu, b) : B.cu[b];
  const int t1 = SAME ? uniform_load(B.cu, (size_t)b + 1) : B.cu[b + 1];
  s.start = SAME ? uniform_load(B.start, b) : B.start[b];
  const int room = (int)(B.table_cols * PAGE);
  const bool ok = s.t0 >= 0 && t1 >= s.t0 && t1 <= (int)B.n_rows && s.start >= 0 && s.start <= room && t1 - s.t0 <= room - s.start;
  if (!ok) s.start = 0;
  s.n = ok ? t1 - s.t0 : 0;
  s.len = s.start + s.n;
  return ok;
}

__device__ __forceinline__ void report(int32_t* status, int bit) {
  if (status) atomicOr(status, bit);
}

}  // namespace bs_kv
