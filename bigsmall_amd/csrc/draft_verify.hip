// Verification of drafted tokens against the target's probabilities.
//
// A sequence's vocabulary is cut into pieces, at most 256 and of 1,024 weights or a multiple. sums_kernel: each workgroup finds the row
// at which the drafts end (a test a lane; three dependent reads), and each of its waves sums that row's weights over pieces
// of its own. pick_kernel: a workgroup per sequence finds the piece, then the token at which the running sum passes the given
// share; it is one wave, so nothing waits at a barrier. Small vocabularies and many sequences are one launch: a workgroup of
// 16 waves for each sequence. Only that one row of p (and of q where a draft was refused) is read, and one piece of it twice. Sums
// are f64: with f32 the token drawn would hang on their order wherever the share falls near a border, and a vocabulary has
// 100,000 of them. They are made in an order that depends on the sizes alone, so the same numbers give the same tokens.
//
// The bound is memory once there is enough to read: 128 sequences of 128,256 weights, f32, p and q: 18 us for up to 131 MB, then 5 to pick. One
// sequence: 4 and 4, a launch and dependent reads each.
#include <float.h>

#include <algorithm>

#include "bigsmall_draft.h"
#include "simt.h"

namespace {

constexpr uint32_t THREADS = 256, WAVES = THREADS / 64;
constexpr uint32_t MOST_PIECES = THREADS, PIECE = 1024;
// One launch up to this many pieces, or from this many sequences on (one a compute unit). f32, one / two launches: 16,000 weights
// 8.6 / 9.9 us for 8 sequences; 32,000 9.9 / 9.1 for 8, 11.9 / 12.9 for 128, and a call is 3 us less of the host's time; 128,256 21.7 / 9.1
// for 8, 28.5 / 30.0 for 128, 39.7 / 47.9 for 256.
constexpr uint32_t ALONE_PIECES = 32, ALONE_SEQS = 256, ALONE_THREADS = 1024;

struct Work {
  double* sums;          // [n_seqs][pieces]
  int32_t* taken;        // [n_seqs] drafts taken, -1: no rows
  uint32_t pieces, len;  // of a sequence; weights of a piece
  uint32_t groups;       // workgroups of a sequence
};

template <int TYPE>
__device__ __forceinline__ float of16(uint32_t bits) {
  if constexpr (TYPE == BS_DRAFT_BF16) return __uint_as_float(bits << 16);
  return (float)__builtin_bit_cast(_Float16, (uint16_t)bits);
}

template <int TYPE>
__device__ __forceinline__ float value(const void* p, uint64_t i) {
  if constexpr (TYPE == BS_DRAFT_F32) return ((const float*)p)[i];
  return of16<TYPE>(((const uint16_t*)p)[i]);
}

template <int TYPE>
__device__ __forceinline__ void values4(const void* p, uint64_t i, float (&v)[4]) {
  // (rows start at any multiple of a weight's size; loads may too)
  if constexpr (TYPE == BS_DRAFT_F32) {
    __builtin_memcpy(v, (const float*)p + i, 16);
  } else {
    uint2 u;
    __builtin_memcpy(&u, (const uint16_t*)p + i, 8);
    v[0] = of16<TYPE>(u.x & 0xFFFFu), v[1] = of16<TYPE>(u.x >> 16), v[2] = of16<TYPE>(u.y & 0xFFFFu), v[3] = of16<TYPE>(u.y >> 16);
  }
}

// (a difference with a NaN in it is not above 0; p = inf less q = inf is one)
__device__ __forceinline__ double weight(double d) { return d > 0 ? (d < (double)FLT_MAX ? d : (double)FLT_MAX) : 0.0; }

// The weights of a sequence's last row.
template <int TYPE>
struct Row {
  const void *p, *q;  // the row; q NULL: not taken off
  uint32_t vocab;
  int64_t without;    // the token left out, -1: none
  __device__ Row(const bs_draft_batch& D, uint64_t row, bool refused) : vocab(D.vocab), without(refused && !D.q ? D.draft[row] : -1) {
    const uint32_t size = TYPE == BS_DRAFT_F32 ? 4 : 2;
    p = (const uint8_t*)D.p + row * (uint64_t)D.p_stride * size;
    q = refused && D.q ? (const uint8_t*)D.q + row * (uint64_t)D.q_stride * size : nullptr;
  }
  __device__ __forceinline__ double of(uint32_t j, float a, float b) const { return (int64_t)j == without ? 0.0 : weight((double)a - (double)b); }
  // w(j) .. w(j + 3), 0 past the end
  __device__ __forceinline__ void four(uint32_t j, double (&w)[4]) const {
    float a[4] = {}, b[4] = {};
    if (j + 4 <= vocab) {
      values4<TYPE>(p, j, a);
      if (q) values4<TYPE>(q, j, b);
    } else {
#pragma unroll
      for (uint32_t e = 0; e < 4; ++e)
        if (j + e < vocab) {
          a[e] = value<TYPE>(p, j + e);
          if (q) b[e] = value<TYPE>(q, j + e);
        }
    }
#pragma unroll
    for (uint32_t e = 0; e < 4; ++e) w[e] = of(j + e, a[e], b[e]);
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

// The sum of a piece, by one wave: every lane has it.
template <int TYPE>
__device__ __forceinline__ double piece_sum(const Row<TYPE>& w, uint32_t piece, uint32_t len) {
  const uint32_t lane = threadIdx.x % 64, lo = piece * len, hi = min(w.vocab, lo + len);
  double sum[4] = {0, 0, 0, 0};
#pragma unroll 4
  for (uint32_t j = lo + lane * 4; j < hi; j += 256) {
    double x[4];
    w.four(j, x);
#pragma unroll
    for (int e = 0; e < 4; ++e) sum[e] += x[e];
  }
  return wave_sum((sum[0] + sum[1]) + (sum[2] + sum[3]));
}

template <int TYPE>
__global__ __launch_bounds__(THREADS) void sums_kernel(bs_draft_batch D, Work W, int32_t* status) {
  const uint32_t b = blockIdx.x / W.groups, group = blockIdx.x % W.groups;
  const int32_t a = taken_drafts<TYPE>(D, b, group == 0 ? status : nullptr);
  if (group == 0 && threadIdx.x == 0) W.taken[b] = a;
  if (a < 0) return;
  const int32_t row = D.cu[b] + a;
  const Row<TYPE> w(D, (uint64_t)row, row + 1 < D.cu[b + 1]);
  for (uint32_t piece = group * WAVES + threadIdx.x / 64; piece < W.pieces; piece += W.groups * WAVES) {
    const double sum = piece_sum(w, piece, W.len);
    if (threadIdx.x % 64 == 0) W.sums[(uint64_t)b * W.pieces + piece] = sum;
  }
}

__device__ __forceinline__ double lane_of(double x, uint32_t lane) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)u, lane), hi = __builtin_amdgcn_readlane((uint32_t)(u >> 32), lane);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// The running sum over the lanes, with this one's x.
__device__ __forceinline__ double running(double x) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const double up = __shfl_up(x, d);
    if (threadIdx.x % 64 >= (uint32_t)d) x += up;
  }
  return x;
}

// The lane whose x takes the running sum `upto` past `share`; if rounding leaves none, the last one with an x above 0.
__device__ __forceinline__ uint32_t passing(double x, double upto, double share) {
  const uint64_t some = __ballot(x > 0), past = __ballot(x > 0 && upto > share);
  return past ? (uint32_t)__builtin_ctzll(past) : some ? 63u - (uint32_t)__builtin_clzll(some) : 0u;
}

// The same among a lane's own four numbers, which begin at `run`: `at` of them is where, `run` the sum before it.
__device__ __forceinline__ void passing4(const double (&x)[4], double share, double& run, uint32_t& at, bool& done) {
  double sum = run;
#pragma unroll
  for (uint32_t e = 0; e < 4; ++e) {
    if (!done && x[e] > 0) at = e, run = sum, done = sum + x[e] > share;
    sum += x[e];
  }
}

// The token at which the running sum of a row's weights passes `part` of their whole sum, by one wave; false if the whole is 0. sums: of
// the pieces.
template <int TYPE>
__device__ bool pick(const Row<TYPE>& w, const Work& W, const double* sums, double part, uint32_t& token) {
  const uint32_t lane = threadIdx.x % 64;
  double s[4];
#pragma unroll
  for (uint32_t e = 0; e < 4; ++e) s[e] = lane * 4 + e < W.pieces ? sums[lane * 4 + e] : 0.0;
  double own = (s[0] + s[1]) + (s[2] + s[3]);
  double upto = running(own);
  const double total = lane_of(upto, 63), share = part * total;
  if (!(total > 0)) return false;
  uint32_t found = passing(own, upto, share), at = 0;
  bool done = false;
  double run = upto - own;
  passing4(s, share, run, at, done);
  const uint32_t piece = found * 4 + __builtin_amdgcn_readlane(at, found);
  const double before = lane_of(run, found);
  // the piece's weights, a run of them to each lane
  const uint32_t each = W.len / 64, j0 = piece * W.len + lane * each;
  own = 0;
  for (uint32_t j = j0; j < j0 + each; j += 16) {
    double x[4][4];
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) w.four(j + i * 4, x[i]);
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) own += (x[i][0] + x[i][1]) + (x[i][2] + x[i][3]);
  }
  upto = running(own) + before;
  found = passing(own, upto, share);
  run = upto - own, done = false;
  uint32_t last = j0;
  double sum = run;
  for (uint32_t j = j0; j < j0 + each && !done; j += 4) {
    double x[4];
    w.four(j, x);
#pragma unroll
    for (uint32_t e = 0; e < 4; ++e) {
      sum += x[e];
      if (!done && x[e] > 0) last = j + e, done = sum > share;
    }
  }
  token = __builtin_amdgcn_readlane(last, found);
  return true;
}

// LONE: the pieces' sums are made here too, by all waves; else there is one.
template <int TYPE, bool LONE>
__global__ __launch_bounds__(LONE ? ALONE_THREADS : 64) void pick_kernel(bs_draft_batch D, Work W, int32_t* status) {
  __shared__ double sums[MOST_PIECES];
  const uint32_t b = blockIdx.x, lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const int32_t a = LONE ? taken_drafts<TYPE>(D, b, wave == 0 ? status : nullptr) : W.taken[b];
  const int32_t r0 = D.cu[b], row = r0 + a;
  int64_t* out = D.tokens + (uint64_t)b * (D.max_drafts + 1);
  // the first drafts are read now and written with the token: waiting for them here would hold up the sums
  const int64_t early = wave == 0 && (int32_t)lane < a ? D.draft[r0 + (int32_t)lane] : -1;
  const auto write = [&](uint32_t token) {
    if (lane <= D.max_drafts) out[lane] = (int32_t)lane == a ? (int64_t)token : early;
    for (uint32_t i = lane + 64; i <= D.max_drafts; i += 64) out[i] = (int32_t)i < a ? D.draft[r0 + (int32_t)i] : (int32_t)i == a ? (int64_t)token : -1;
    if (lane == 0) D.counts[b] = a + 1;
  };
  if (a < 0) {
    if (wave == 0) write(0);
    return;
  }
  const Row<TYPE> w(D, (uint64_t)row, row + 1 < D.cu[b + 1]);
  if constexpr (LONE) {
    for (uint32_t piece = wave; piece < W.pieces; piece += ALONE_THREADS / 64) {
      const double sum = piece_sum(w, piece, W.len);
      if (lane == 0) sums[piece] = sum;
    }
    __syncthreads();
    if (wave != 0) return;
  }
  uint32_t token = 0;
  if (!pick(w, W, LONE ? sums : W.sums + (uint64_t)b * W.pieces, (double)D.pick[b], token)) {
    // nothing is left of the row: once more with the target's own
    const Row<TYPE> plain(D, (uint64_t)row, false);
    for (uint32_t piece = 0; piece < W.pieces; ++piece) {
      const double sum = piece_sum(plain, piece, W.len);
      if (lane == 0) sums[piece] = sum;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (!pick(plain, W, sums, (double)D.pick[b], token) && lane == 0 && status) atomicOr(status, BS_DEV_ERR_COUNT);
  }
  write(token);
}

Work layout(uint32_t n_seqs, uint32_t vocab, void* d_work) {
  Work w;
  w.len = PIECE * ((vocab + MOST_PIECES * PIECE - 1) / (MOST_PIECES * PIECE));
  w.pieces = (vocab + w.len - 1) / w.len;
  // 2,048 workgroups fill the card; more of them would look for the drafts' end once more each
  w.groups = std::max(1u, std::min((w.pieces + WAVES - 1) / WAVES, 2048 / std::max(1u, n_seqs)));
  w.sums = (double*)d_work;
  w.taken = (int32_t*)(w.sums + (uint64_t)n_seqs * w.pieces);
  return w;
}

bool alone(uint32_t n_seqs, uint32_t pieces) { return pieces <= ALONE_PIECES || n_seqs >= ALONE_SEQS; }

template <int TYPE>
int launch(const bs_draft_batch& D, const Work& w, int32_t* status, hipStream_t s) {
  if (alone(D.n_seqs, w.pieces)) {
    pick_kernel<TYPE, true><<<D.n_seqs, ALONE_THREADS, 0, s>>>(D, w, status);
  } else {
    sums_kernel<TYPE><<<D.n_seqs * w.groups, THREADS, 0, s>>>(D, w, status);
    pick_kernel<TYPE, false><<<D.n_seqs, 64, 0, s>>>(D, w, status);
  }
  return hipGetLastError() == hipSuccess ? BS_OK : BS_ERR_HIP;
}

}  // namespace

extern "C" uint64_t bs_draft_verify_work_bytes(uint32_t n_seqs, uint32_t vocab) {
  const uint32_t pieces = layout(n_seqs, vocab, nullptr).pieces;
  return alone(n_seqs, pieces) ? 0 : (uint64_t)n_seqs * (pieces * 8ull + 4ull);
}

extern "C" int bs_draft_verify(const bs_draft_batch* D, void* d_work, uint64_t work_bytes, int32_t* d_status, void* stream) {
  if (!D || D->type > BS_DRAFT_F16 || D->vocab == 0 || D->vocab > (1u << 30) || D->max_drafts > BS_DRAFT_MOST ||
      D->n_seqs > (1u << 20) || D->n_rows > (1u << 30) || D->p_stride < 0 || D->q_stride < 0)
    return BS_ERR_ARG;
  if (D->n_seqs == 0) return BS_OK;
  if (!D->cu || !D->pick || !D->tokens || !D->counts || (D->n_rows && (!D->p || !D->draft || !D->accept))) return BS_ERR_ARG;
  const uintptr_t size = D->type == BS_DRAFT_F32 ? 3 : 1;
  if (((uintptr_t)D->p & size) || ((uintptr_t)D->q & size)) return BS_ERR_ARG;
  const uint64_t need = bs_draft_verify_work_bytes(D->n_seqs, D->vocab);
  if (work_bytes < need || (need && (!d_work || ((uintptr_t)d_work & 15)))) return BS_ERR_CAP;
  const Work w = layout(D->n_seqs, D->vocab, d_work);
  hipStream_t s = (hipStream_t)stream;
  return D->type == BS_DRAFT_F32 ? launch<BS_DRAFT_F32>(*D, w, d_status, s)
         : D->type == BS_DRAFT_BF16 ? launch<BS_DRAFT_BF16>(*D, w, d_status, s)
                                    : launch<BS_DRAFT_F16>(*D, w, d_status, s);
}
