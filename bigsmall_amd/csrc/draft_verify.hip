// Verification of drafted tokens against the target's probabilities.
//
// parts_kernel: a workgroup per part of a sequence's vocabulary. Each finds the row at which the drafts end (a test a
// lane; three dependent reads) and sums that row's weights over its part. pick_kernel: a workgroup per sequence finds
// the part, the thread and the token at which the running sum passes the given share. Only that one row of p (and of
// q where a draft was refused) is read. Sums are f64: with f32 the token drawn would hang on their order wherever the
// share falls near a border, and a vocabulary has 100,000 of them. They are made in an order that depends on the
// sizes alone, so the same numbers give the same tokens.
#include <float.h>

#include <algorithm>

#include "bigsmall_draft.h"
#include "simt.h"

namespace {

constexpr uint32_t THREADS = 256, WAVES = THREADS / 64;
constexpr uint32_t MOST_PARTS = THREADS, PART_MIN = 4096;

struct Work {
  double* sums;   // [n_seqs][parts]
  int32_t* taken; // [n_seqs] drafts taken, -1: no rows
  uint32_t parts, len;  // elements of a part
};

template <int TYPE>
__device__ __forceinline__ float value(const void* p, uint64_t i) {
  if constexpr (TYPE == BS_DRAFT_F32) return ((const float*)p)[i];
  if constexpr (TYPE == BS_DRAFT_BF16) return __uint_as_float((uint32_t)((const uint16_t*)p)[i] << 16);
  if constexpr (TYPE == BS_DRAFT_F16) return (float)((const _Float16*)p)[i];
}

__device__ __forceinline__ double weight(double d) { return d > 0 ? (d < (double)FLT_MAX ? d : (double)FLT_MAX) : 0.0; }

// The weights of a sequence's last row, w(j).
template <int TYPE>
struct Row {
  const bs_draft_batch& D;
  uint64_t p, q;   // where the row begins
  int64_t without; // the token left out, -1: none
  bool minus;      // q is taken off
  __device__ Row(const bs_draft_batch& batch, uint64_t row, bool refused)
      : D(batch), p(row * (uint64_t)batch.p_stride), q(row * (uint64_t)batch.q_stride),
        without(refused && !batch.q ? batch.draft[row] : -1), minus(refused && batch.q) {}
  __device__ __forceinline__ double operator()(uint32_t j) const {
    double d = (double)value<TYPE>(D.p, p + j);
    if (minus) d -= (double)value<TYPE>(D.q, q + j);
    return (int64_t)j == without ? 0.0 : weight(d);
  }
};

// Drafts that are taken, by every wave for itself; -1: no rows.
template <int TYPE>
__device__ int32_t taken_drafts(const bs_draft_batch& D, uint32_t b, int32_t* status) {
  const int32_t r0 = D.cu[b], r1 = D.cu[b + 1];
  if (r0 < 0 || r1 < r0 || r1 > (int32_t)D.n_rows || r1 - r0 > (int32_t)D.max_drafts + 1) {
    if (status) atomicOr(status, BS_DEV_ERR_BOUNDS);
    return -1;
  }
  const int32_t n = r1 - r0 - 1;
  for (int32_t i0 = 0; i0 < n; i0 += 64) {
    const int32_t i = i0 + (int32_t)(threadIdx.x % 64);
    bool refused = false;
    if (i < n) {
      const uint64_t r = (uint64_t)(r0 + i);
      const int64_t x = D.draft[r];
      if (x < 0 || x >= (int64_t)D.vocab) {
        refused = true;
        if (status) atomicOr(status, BS_DEV_ERR_BOUNDS);
      } else {
        const double q = D.q ? (double)value<TYPE>(D.q, r * (uint64_t)D.q_stride + (uint64_t)x) : 1.0;
        refused = !((double)D.accept[r] * q < (double)value<TYPE>(D.p, r * (uint64_t)D.p_stride + (uint64_t)x));
      }
    }
    const uint64_t at = __ballot(refused);
    if (at) return i0 + __builtin_ctzll(at);
  }
  return n;
}

__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) x += __shfl_xor(x, d);
  return x;
}

// Sum of the threads' x up to and including one's own.
__device__ double block_scan(double x, double* lds) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const double up = __shfl_up(x, d);
    if (threadIdx.x % 64 >= (uint32_t)d) x += up;
  }
  __syncthreads();
  if (threadIdx.x % 64 == 63) lds[threadIdx.x / 64] = x;
  __syncthreads();
  for (uint32_t w = 0; w < threadIdx.x / 64; ++w) x += lds[w];
  return x;
}

template <int TYPE>
__global__ __launch_bounds__(THREADS) void parts_kernel(bs_draft_batch D, Work W, int32_t* status) {
  __shared__ double sums[WAVES];
  const uint32_t b = blockIdx.x / W.parts, part = blockIdx.x % W.parts;
  const int32_t a = taken_drafts<TYPE>(D, b, part == 0 ? status : nullptr);
  if (part == 0 && threadIdx.x == 0) W.taken[b] = a;
  if (a < 0) return;
  const int32_t row = D.cu[b] + a;
  const Row<TYPE> w(D, (uint64_t)row, row + 1 < D.cu[b + 1]);
  const uint32_t end = min(D.vocab, (part + 1) * W.len);
  double sum = 0;
  for (uint32_t j = part * W.len + threadIdx.x; j < end; j += THREADS) sum += w(j);
  sum = wave_sum(sum);
  if (threadIdx.x % 64 == 0) sums[threadIdx.x / 64] = sum;
  __syncthreads();
  if (threadIdx.x == 0) W.sums[(uint64_t)b * W.parts + part] = (sums[0] + sums[1]) + (sums[2] + sums[3]);
}

// The first token in [lo, hi) at which `before` plus the weights up to it exceed `share`; if rounding leaves none, the
// last one with a weight (0 if there is no such one either). Every thread gets it.
template <int TYPE>
__device__ uint32_t find(const Row<TYPE>& w, uint32_t lo, uint32_t hi, double before, double share, double* lds, uint32_t* lds_at) {
  const uint32_t each = (hi - lo + THREADS - 1) / THREADS;
  const uint32_t j0 = min(hi, lo + threadIdx.x * each), j1 = min(hi, j0 + each);
  double own = 0;
  for (uint32_t j = j0; j < j1; ++j) own += w(j);
  const double upto = before + block_scan(own, lds);
  if (threadIdx.x == 0) lds_at[0] = THREADS, lds_at[1] = 0;
  __syncthreads();
  if (own > 0 && upto > share) atomicMin(&lds_at[0], threadIdx.x);
  if (own > 0) atomicMax(&lds_at[1], threadIdx.x);
  __syncthreads();
  if (threadIdx.x == (lds_at[0] < THREADS ? lds_at[0] : lds_at[1])) {
    double sum = upto - own;
    uint32_t last = 0;
    for (uint32_t j = j0; j < j1; ++j) {
      const double x = w(j);
      sum += x;
      if (x > 0) last = j;
      if (x > 0 && sum > share) break;
    }
    lds_at[2] = last;
  }
  __syncthreads();
  return lds_at[2];
}

template <int TYPE>
__global__ __launch_bounds__(THREADS) void pick_kernel(bs_draft_batch D, Work W, int32_t* status) {
  __shared__ double lds[WAVES], total[2];
  __shared__ uint32_t at[3];
  const uint32_t b = blockIdx.x, tid = threadIdx.x;
  const int32_t a = W.taken[b];
  int64_t* out = D.tokens + (uint64_t)b * (D.max_drafts + 1);
  uint32_t token = 0;
  if (a >= 0) {
    const int32_t row = D.cu[b] + a;
    const Row<TYPE> w(D, (uint64_t)row, row + 1 < D.cu[b + 1]);
    const double own = tid < W.parts ? W.sums[(uint64_t)b * W.parts + tid] : 0.0;
    const double upto = block_scan(own, lds);
    if (tid == THREADS - 1) total[0] = upto;
    if (tid == 0) at[0] = THREADS, at[1] = 0;
    __syncthreads();
    if (total[0] > 0) {
      const double share = (double)D.pick[b] * total[0];
      if (own > 0 && upto > share) atomicMin(&at[0], tid);
      if (own > 0) atomicMax(&at[1], tid);
      __syncthreads();
      const uint32_t part = at[0] < THREADS ? at[0] : at[1];
      if (tid == part) total[1] = upto - own;
      __syncthreads();
      token = find(w, part * W.len, min(D.vocab, (part + 1) * W.len), total[1], share, lds, at);
    } else {
      // nothing is left of the row (or it holds no probability): the target's own
      const Row<TYPE> plain(D, (uint64_t)row, false);
      double sum = 0;
      for (uint32_t j = tid; j < D.vocab; j += THREADS) sum += plain(j);
      sum = block_scan(sum, lds);
      if (tid == THREADS - 1) total[1] = sum;
      __syncthreads();
      if (total[1] > 0)
        token = find(plain, 0, D.vocab, 0.0, (double)D.pick[b] * total[1], lds, at);
      else if (tid == 0 && status)
        atomicOr(status, BS_DEV_ERR_COUNT);
    }
  }
  for (uint32_t i = tid; i <= D.max_drafts; i += THREADS)
    out[i] = (int32_t)i < a ? D.draft[D.cu[b] + (int32_t)i] : (int32_t)i == a ? (int64_t)token : -1;
  if (tid == 0) D.counts[b] = a + 1;
}

Work layout(uint32_t n_seqs, uint32_t vocab, void* d_work) {
  Work w;
  // enough workgroups to fill the card, parts of 4,096 elements at least
  w.parts = std::max(1u, std::min({MOST_PARTS, 2048 / std::max(1u, n_seqs), (vocab + PART_MIN - 1) / PART_MIN}));
  w.len = (vocab + w.parts - 1) / w.parts;
  w.sums = (double*)d_work;
  w.taken = (int32_t*)(w.sums + (uint64_t)n_seqs * w.parts);
  return w;
}

template <int TYPE>
int launch(const bs_draft_batch& D, const Work& w, int32_t* status, hipStream_t s) {
  parts_kernel<TYPE><<<D.n_seqs * w.parts, THREADS, 0, s>>>(D, w, status);
  pick_kernel<TYPE><<<D.n_seqs, THREADS, 0, s>>>(D, w, status);
  return hipGetLastError() == hipSuccess ? BS_OK : BS_ERR_HIP;
}

}  // namespace

extern "C" uint64_t bs_draft_verify_work_bytes(uint32_t n_seqs, uint32_t vocab) {
  return (uint64_t)n_seqs * (layout(n_seqs, vocab, nullptr).parts * 8ull + 4ull);
}

extern "C" int bs_draft_verify(const bs_draft_batch* D, void* d_work, uint64_t work_bytes, int32_t* d_status, void* stream) {
  if (!D || D->type > BS_DRAFT_F16 || D->vocab == 0 || D->vocab > (1u << 30) || D->max_drafts > BS_DRAFT_MOST ||
      D->n_seqs > (1u << 20) || D->n_rows > (1u << 30) || D->p_stride < 0 || D->q_stride < 0)
    return BS_ERR_ARG;
  if (D->n_seqs == 0) return BS_OK;
  if (!D->cu || !D->pick || !D->tokens || !D->counts || (D->n_rows && (!D->p || !D->draft || !D->accept))) return BS_ERR_ARG;
  const uintptr_t size = D->type == BS_DRAFT_F32 ? 3 : 1;
  if (((uintptr_t)D->p & size) || ((uintptr_t)D->q & size)) return BS_ERR_ARG;
  if (!d_work || ((uintptr_t)d_work & 15) || work_bytes < bs_draft_verify_work_bytes(D->n_seqs, D->vocab)) return BS_ERR_CAP;
  const Work w = layout(D->n_seqs, D->vocab, d_work);
  hipStream_t s = (hipStream_t)stream;
  return D->type == BS_DRAFT_F32 ? launch<BS_DRAFT_F32>(*D, w, d_status, s)
         : D->type == BS_DRAFT_BF16 ? launch<BS_DRAFT_BF16>(*D, w, d_status, s)
                                    : launch<BS_DRAFT_F16>(*D, w, d_status, s);
}
