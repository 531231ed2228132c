// Products of e4m3 weights with a scale for each block of 128.
//
// bs_fp8_quantise: sixteen lanes hold a block of 128 columns, eight each; the largest
// |x| goes round among them and gives the scale. The bound is memory: two bytes in, one out.
//
// bs_fp8_linear: one matrix instruction multiplies 16 rows of the weight by 16 rows of x over
// a whole block of 128 columns, so its result is scaled in registers (the row's scale times the
// block's) and added to f32 sums. The weight is the instruction's first operand: a lane then holds
// four outputs of one row of x, which share their scale. The instruction adds eight neighbouring products at a time,
// taken to the exponent 2^e of the largest and cut off at 2^(e - 13) (all e4m3 forms do); a product is itself off by up to
// 2^-3 of its size from the two codes' rounding, so that is 1/1,000 of what 8 bits cost. Sums of the groups, of blocks
// and their scaling are f32. Products exact in f16 would be summed in f32 throughout, at half the rate and less, with
// every code converted first.
#include <math.h>

#include "bigsmall_fp8.h"
#include "simt.h"

namespace {

constexpr uint32_t BLOCK = BS_FP8_BLOCK;

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

template <int TYPE>
__device__ __forceinline__ float load16(uint16_t bits) {
  if constexpr (TYPE == BS_FP8_BF16)
    return __uint_as_float((uint32_t)bits << 16);
  else
    return (float)__builtin_bit_cast(_Float16, bits);
}

// Round to nearest even; NaN stays NaN.
template <int TYPE>
__device__ __forceinline__ uint16_t store16(float x) {
  if constexpr (TYPE == BS_FP8_BF16)
    return __builtin_bit_cast(uint16_t, (__bf16)x);
  else
    return __builtin_bit_cast(uint16_t, (_Float16)x);
}

// ---- quantising

constexpr uint32_t Q_THREADS = 256, Q_ROWS = Q_THREADS / 16, Q_BLOCKS = 4;  // of one workgroup

// Blocks with an |x| below this are scaled as if they had it: scales and their inverses stay normal f32 numbers.
constexpr float AMAX_LO = 0x1p-100f;

// 448 x / a for |x| <= a, so exact that its rounding to e4m3 is the quotient's own. x and a have 11 significant bits or
// fewer, so a quotient is a border between two codes exactly or misses it by 2^-16 of itself and more; q is within 2^-22,
// and one step of the division (the remainder is exact) makes an exactly representable quotient exact.
__device__ __forceinline__ float quotient(float v, float a, float inv) {
#pragma clang fp contract(off)
  const float q = v * inv;
  return __builtin_fmaf(__builtin_fmaf(-q, a, v), inv, q);
}

template <int TYPE, bool WIDE>
__global__ __launch_bounds__(Q_THREADS) void quantise_kernel(const uint16_t* x, int64_t x_stride, bs_fp8_rows R) {
  const uint32_t lane = threadIdx.x % 16, blocks = R.code_stride / BLOCK;
  const uint64_t t = (uint64_t)blockIdx.y * Q_ROWS + threadIdx.x / 16;
  if (t >= R.rows) return;
  const uint16_t* row = x + (int64_t)t * x_stride;
  const uint32_t j0 = blockIdx.x * Q_BLOCKS;
  uint16_t v[Q_BLOCKS][8] = {};
#pragma unroll
  for (uint32_t i = 0; i < Q_BLOCKS; ++i) {
    const uint32_t k = (j0 + i) * BLOCK + lane * 8;
    if (WIDE && k + 8 <= R.cols) {
      *(uint4*)v[i] = *(const uint4*)(row + k);
    } else {
#pragma unroll
      for (uint32_t e = 0; e < 8; ++e)
        if (k + e < R.cols) v[i][e] = row[k + e];
    }
  }
#pragma unroll
  for (uint32_t i = 0; i < Q_BLOCKS; ++i) {
    const uint32_t j = j0 + i;
    if (j >= blocks) break;
    float f[8], a = 0;
    bool bad = false;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      f[e] = load16<TYPE>(v[i][e]);
      bad = bad || !(fabsf(f[e]) < INFINITY);
      a = fmaxf(a, fabsf(f[e]));
    }
    a = bad ? INFINITY : a;
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) a = fmaxf(a, __shfl_xor(a, d));
    bad = a == INFINITY;
    a = fmaxf(a, AMAX_LO);
    // near the end of f32's range both sides are taken by 2^-16
    const float down = a > 0x1p100f ? 0x1p-16f : 1.0f, b = a * down, inv = 1.0f / b;
    uint32_t w[2];
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      float y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = quotient(f[4 * p + e] * down * 448.0f, b, inv);
      w[p] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
      w[p] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], (int)w[p], true);
      w[p] = bad ? 0u : w[p];
    }
    *(uint2*)(R.codes + t * R.code_stride + j * BLOCK + lane * 8) = make_uint2(w[0], w[1]);
    if (lane == 0) R.scales[(uint64_t)j * R.scale_stride + t] = bad ? __uint_as_float(0x7FC00000u) : a / 448.0f;
  }
}

template <int TYPE>
int quantise_launch(const void* x, int64_t stride, const bs_fp8_rows& R, hipStream_t s) {
  const dim3 grid((R.code_stride / BLOCK + Q_BLOCKS - 1) / Q_BLOCKS, (R.rows + Q_ROWS - 1) / Q_ROWS);
  if (((uintptr_t)x & 15) == 0 && stride % 8 == 0)
    quantise_kernel<TYPE, true><<<grid, Q_THREADS, 0, s>>>((const uint16_t*)x, stride, R);
  else
    quantise_kernel<TYPE, false><<<grid, Q_THREADS, 0, s>>>((const uint16_t*)x, stride, R);
  return hipGetLastError() == hipSuccess ? BS_OK : BS_ERR_HIP;
}

// ---- the product

__device__ __forceinline__ f32x4 product(i32x8 w, i32x8 x) {
  // (scales of 0 name the form without scales: e4m3 as it is)
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, f32x4{0, 0, 0, 0}, 0, 0, 0, 0, 0, 0);
}

__device__ __forceinline__ i32x8 load_operand(const uint8_t* p) {
  const i32x4 lo = *(const i32x4*)p, hi = *(const i32x4*)(p + 16);
  return i32x8{lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
}

constexpr uint32_t THREADS = 256;

// A wave: 16 rows of the weight by 16 rows of x.
template <int TYPE>
__global__ __launch_bounds__(THREADS) void linear_kernel(bs_fp8_rows X, bs_fp8_weight W, uint16_t* y, int64_t y_stride) {
  const uint32_t lane = threadIdx.x % 64;
  const uint32_t n0 = (blockIdx.x * (THREADS / 64) + threadIdx.x / 64) * 16;
  const uint64_t t0 = (uint64_t)blockIdx.y * 16;
  if (n0 >= W.outer) return;
  const uint64_t t = t0 + lane % 16 < X.rows ? t0 + lane % 16 : X.rows - 1;
  const uint32_t n = min(n0 + lane % 16, W.outer - 1);
  const uint8_t* wp = W.codes + (uint64_t)n * W.stride + lane / 16 * 32;
  const uint8_t* xp = X.codes + t * X.code_stride + lane / 16 * 32;
  const float* ws = W.scales + (uint64_t)(n0 / BLOCK) * W.scale_stride;
  f32x4 sum = {0, 0, 0, 0};
  for (uint32_t j = 0; j < X.code_stride / BLOCK; ++j) {
    const f32x4 d = product(load_operand(wp + (uint64_t)j * BLOCK), load_operand(xp + (uint64_t)j * BLOCK));
    const float s = ws[j] * X.scales[(uint64_t)j * X.scale_stride + t];
#pragma unroll
    for (int r = 0; r < 4; ++r) sum[r] = __builtin_fmaf(s, d[r], sum[r]);
  }
  if (t0 + lane % 16 >= X.rows) return;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const uint32_t o = n0 + lane / 16 * 4 + r;
    if (o < W.outer) y[(int64_t)t * y_stride + o] = store16<TYPE>(sum[r]);
  }
}

template <int TYPE>
int linear_launch(const bs_fp8_rows& X, const bs_fp8_weight& W, void* y, int64_t y_stride, hipStream_t s) {
  const dim3 grid((W.outer + 63) / 64, (X.rows + 15) / 16);
  linear_kernel<TYPE><<<grid, THREADS, 0, s>>>(X, W, (uint16_t*)y, y_stride);
  return hipGetLastError() == hipSuccess ? BS_OK : BS_ERR_HIP;
}

bool aligned(const void* p) { return p && ((uintptr_t)p & 15) == 0; }

// A grid has at most 65,535 workgroups in its second dimension, 16 rows each; code offsets of a row stay below 2^31.
constexpr uint32_t MOST_ROWS = 65535 * 16, MOST_COLS = 1u << 24;

bool rows_ok(const bs_fp8_rows* r) {
  return r && r->rows <= MOST_ROWS && r->cols > 0 && r->cols <= MOST_COLS && r->code_stride % BLOCK == 0 &&
         r->code_stride >= r->cols && r->code_stride - r->cols < BLOCK && r->scale_stride >= r->rows &&
         (r->rows == 0 || (aligned(r->codes) && aligned(r->scales)));
}

bool weight_ok(const bs_fp8_weight* w) {
  return w && w->outer > 0 && w->outer <= MOST_COLS && w->inner > 0 && w->inner <= MOST_COLS && w->stride % BLOCK == 0 &&
         w->stride >= w->inner && w->scale_stride >= (w->inner + BLOCK - 1) / BLOCK && aligned(w->codes) && w->scales &&
         ((uintptr_t)w->scales & 3) == 0;
}

}  // namespace

extern "C" int bs_fp8_quantise(const void* x, uint32_t type, int64_t x_stride, const bs_fp8_rows* out, void* stream) {
  if (!rows_ok(out) || type > BS_FP8_F16 || x_stride < 0) return BS_ERR_ARG;
  if (out->rows == 0) return BS_OK;
  if (!x || ((uintptr_t)x & 1)) return BS_ERR_ARG;
  return type == BS_FP8_BF16 ? quantise_launch<BS_FP8_BF16>(x, x_stride, *out, (hipStream_t)stream)
                             : quantise_launch<BS_FP8_F16>(x, x_stride, *out, (hipStream_t)stream);
}

extern "C" uint64_t bs_fp8_linear_work_bytes(const bs_fp8_rows* x, const bs_fp8_weight* w) {
  (void)x, (void)w;
  return 0;
}

extern "C" int bs_fp8_linear(const bs_fp8_rows* x, const bs_fp8_weight* w, void* y, uint32_t type, int64_t y_stride, void* d_work,
                             uint64_t work_bytes, void* stream) {
  if (!rows_ok(x) || !weight_ok(w) || type > BS_FP8_F16 || x->cols != w->inner || y_stride < (int64_t)w->outer) return BS_ERR_ARG;
  if (x->rows == 0) return BS_OK;
  if (!y || ((uintptr_t)y & 1)) return BS_ERR_ARG;
  const uint64_t need = bs_fp8_linear_work_bytes(x, w);
  if (work_bytes < need || (need && !aligned(d_work))) return BS_ERR_CAP;
  return type == BS_FP8_BF16 ? linear_launch<BS_FP8_BF16>(*x, *w, y, y_stride, (hipStream_t)stream)
                             : linear_launch<BS_FP8_F16>(*x, *w, y, y_stride, (hipStream_t)stream);
}
