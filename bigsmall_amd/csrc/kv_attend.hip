// Attention over the paged 8-bit KV cache.
//
// The rows of a sequence and kv head are its new tokens times the q heads of
// the group, row r = token r / G, head r % G. A step whose sequences have few
// rows goes to rows_kernel, any other to prompt_kernel (both take any number);
// join_kernel puts together what was split over the cache's length.
//
// rows_kernel: tiles of 16 rows. A wave takes one page at a time:
//   S^T = K Q^T   (64 keys x 16 rows; K's codes as f16, exactly)
//   softmax over keys with a running maximum and sum
//   O^T += V^T P^T
// in 16x16x32 products. Keys are numbered so that the 16 keys of a lane in S^T
// (4 products of 16 keys, 4 accumulators each) are the 16 consecutive ones
// 16g..16g+15 of its lane group g = lane / 16; that is what the lane needs as
// the right operand of the second product, and 16 consecutive tokens of a
// channel of V are 16 bytes of the page. So P stays in registers and K and V
// go from memory to the matrix unit without LDS.
//
// Scales: a page's K scale multiplies the scores; its V scale goes into the
// exponent, p' = 2^(s + log2(vs) - m) with m the running maximum of s +
// log2(vs), so that O adds up codes * p' over pages of different scales, and
// the denominator adds up (sum of p' in the page) / vs. Scores and log2 in base
// 2, sums and maxima all in f32. p' goes to the product as f16, multiplied by 2^12
// so that weights down to 2^-26 of the largest keep all 11 bits: an eighth of what
// rounding the output to bf16 takes, and a second part of 11 more would double the
// second product. q goes as f16 after a power of two: exact down to 2^-14 of the
// row's largest channel, below that within 2^-25 of it, the size of the rounding in
// the f32 sum.
//
// A row sees one interval of keys [lo, hi), whatever masks are set. A page that
// lies inside the interval of all rows needs no comparison.
#include "kv_common.h"

#include <algorithm>

#include "lds_limit.h"

namespace bs_kv {
bool check_pool(const bs_kv_pool* p);
bool check_batch(const bs_kv_batch* b);
}  // namespace bs_kv

namespace {

using namespace bs_kv;

constexpr float LOG2E = 1.44269504088896340736f;
constexpr float LN2 = 0.69314718055994530942f;
constexpr float P_SHIFT = 12.0f;
constexpr float NEG_INF = -__builtin_inff();

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

constexpr int WAVES = 4;      // of a workgroup of rows_kernel

// Split results: per part and row O (f32, not divided), m, l. All parts of a
// row are marked: those without keys with m = -inf and l = 0; a row that was not
// split is written by its kernel itself, which leaves l = -1 in the first.
struct Work {
  float* o;
  float2* ml;
  uint32_t parts;      // that the pages which a tile of rows sees are cut into at most: 1 if nothing is split
  int piece;           // rows_kernel: pages of a part
  bool ranked;         // rows_kernel: more workgroups than run at once
};

// Interval of keys that row (token i of the sequence) sees.
__device__ __forceinline__ int2 seen_by(const bs_kv_query& A, const SeqStep& s, uint32_t b, int i) {
  const int pos = s.start + i;
  int lo = 0, hi = pos + 1;
  if (A.prefix) hi = max(hi, min(uniform_load(A.prefix, b), s.len));
  if (A.first) lo = max(lo, A.first[s.t0 + i]);
  if (A.window && (uint32_t)pos >= A.window) lo = max(lo, pos - (int)A.window + 1);
  return make_int2(min(lo, hi), hi);
}

// What turns products into scores (base 2) besides the per-row and per-page scales.
struct Score {
  float scale;    // of q.k: times log2 e without a cap, divided by the cap with one
  float cap;      // softcap * log2 e, 0: none
};

// cap * tanh(x), two ways. Up to QUICK_CAP: cap - 2 cap / (e^2x + 1), off by 2^-22 of the cap, so by 2^-16 at most, a
// sixteenth of what rounding the weights to f16 takes. Larger caps: within 2^-21 of its own value. 1 - 2 / (e^2|x| + 1)
// takes small results from two ones, so that below 1/2 an odd polynomial stands in for it (x + x^3 P(x^2), P of degree 3
// with the least largest relative error there, 2^-25.9). (us with quick / whole:
// one row over 1,024 tokens 13.1 / 15.1, an 8,192-token prompt with heads of 128 690 / 829, 500 tokens over a window of
// 16,384 with heads of 256 222 / 284.)
constexpr float QUICK_CAP = 64.0f;
__device__ __forceinline__ float quick_capped(float x, float cap) {
  const float e = exp2_fast(x * (2.0f * LOG2E));
  return cap - cap * 2.0f * __builtin_amdgcn_rcpf(e + 1.0f);
}
__device__ __forceinline__ float whole_tanh(float x) {
  const float a = fabsf(x), t = x * x;
  const float p = fmaf(t, fmaf(t, fmaf(t, 0.017241491f, -0.053045493f), 0.13325879f), -0.33333144f);
  const float far = 1.0f - 2.0f * __builtin_amdgcn_rcpf(exp2_fast(a * (2.0f * LOG2E)) + 1.0f);
  return a < 0.5f ? fmaf(x * t, p, x) : copysignf(far, x);
}

template <int D>
struct Dims {
  static constexpr int PAIRS = D / 64;              // 64 channels: two products of 32
  static constexpr bool REST = D % 64 != 0;         // 16 or 32 more: one product
  static constexpr int REST_GROUPS = (D % 64) / 8;  // lane groups that hold channels of it
  static constexpr int STEPS = 2 * PAIRS + (REST ? 1 : 0);
  static constexpr int TILES = D / 16;              // of 16 channels of O^T
};

// Channel that element 0 of product `step` holds in lane group g.
template <int D>
__device__ __forceinline__ int channel_of(int step, int g) {
  return step < 2 * Dims<D>::PAIRS ? 64 * (step / 2) + 16 * g + 8 * (step % 2) : 64 * Dims<D>::PAIRS + 8 * g;
}

// A page's bytes are used once in a call (128 sequences of 16,000 tokens, GB/s: 5,700 through the caches as usual, 6,130
// as a stream).
// `page` is the same in all lanes, so that an address is a scalar and a 32-bit offset.
__device__ __forceinline__ uint4 stream16(const uint8_t* page, uint32_t at) {
  const uint8_t* p = page + at;
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  const u32x4 v = __builtin_nontemporal_load((const u32x4*)p);
  return make_uint4(v.x, v.y, v.z, v.w);
}

template <int D, int KIND>
struct PageK {       // a lane's part of a K page: 4 keys
  uint4 w[4][Dims<D>::PAIRS];
  uint2 r[4];
  __device__ __forceinline__ void load(const uint8_t* page, int lane) {
    const uint32_t g = (uint32_t)lane >> 4, row = (16 * ((lane & 15) >> 2) + (lane & 3)) * D;
#pragma unroll
    for (uint32_t t = 0; t < 4; ++t) {
#pragma unroll
      for (uint32_t c = 0; c < Dims<D>::PAIRS; ++c) w[t][c] = stream16(page, row + 16 * g + (4 * t * D + 64 * c));
      if constexpr (Dims<D>::REST)
        r[t] = g < (uint32_t)Dims<D>::REST_GROUPS ? *(const uint2*)(page + (row + 8 * g + (4 * t * D + 64 * Dims<D>::PAIRS))) : make_uint2(0, 0);
    }
  }
  __device__ __forceinline__ half8v operand(int t, int step) const {
    if (step >= 2 * Dims<D>::PAIRS) {
      half8v x = codes8_to_f16<KIND>(r[t].x, r[t].y);
      return x;
    }
    const uint4 x = w[t][step / 2];
    return step % 2 ? codes8_to_f16<KIND>(x.z, x.w) : codes8_to_f16<KIND>(x.x, x.y);
  }
};

template <int D, int KIND>
struct PageV {
  uint4 w[Dims<D>::TILES];
  __device__ __forceinline__ void load(const uint8_t* page, int lane) {
    const uint32_t at = (uint32_t)(lane & 15) * PAGE + 16 * ((uint32_t)lane >> 4);
#pragma unroll
    for (uint32_t d = 0; d < Dims<D>::TILES; ++d) w[d] = stream16(page, at + 16 * d * PAGE);
  }
  __device__ __forceinline__ half8v operand(int d, int u) const {
    return u ? codes8_to_f16<KIND>(w[d].z, w[d].w) : codes8_to_f16<KIND>(w[d].x, w[d].y);
  }
};

// Running softmax of one row tile in a wave: this lane's row is lane & 15.
template <int D>
struct State {
  f32x4 o[Dims<D>::TILES];
  float m, l;        // m: over all keys so far; l: of this lane's keys
};

// Scores of a page from its products: s[t][i] belongs to key j0 + 4 t + i (j0: the lane group's first).
template <int N>
__device__ __forceinline__ void scores(f32x4 (&s)[N], const Score& sc, float row_scale, float page_scale, float shift,
                                       int j0, int2 see, bool inside, bool biased, float slope, int pos) {
  float c = row_scale * (page_scale * sc.scale);
  if (sc.cap > QUICK_CAP * LOG2E) {
#pragma unroll
    for (int t = 0; t < N; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[t][i] = sc.cap * whole_tanh(s[t][i] * c);
    c = 1.0f;
  }
  int lo = see.x - j0, hi = see.y - j0;
  float d = (float)(pos - j0);
  BS_OPAQUE(lo);
  BS_OPAQUE(hi);
  BS_OPAQUE(d);
#pragma unroll
  for (int t = 0; t < N; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float x = s[t][i] * c;
      if (sc.cap != 0.0f && sc.cap <= QUICK_CAP * LOG2E) x = quick_capped(x, sc.cap);
      const int j = 4 * t + i;
      if (biased) x -= slope * fabsf(d - (float)j);
      x += shift;
      if (!inside) x = (j >= lo && j < hi) ? x : NEG_INF;
      s[t][i] = x;
    }
}

// Weights from scores; rescales what is already there.
template <int D, int N>
__device__ __forceinline__ void weights(f32x4 (&s)[N], State<D>& st, float inv_vs) {
  float top = NEG_INF;
#pragma unroll
  for (int t = 0; t < N; ++t) top = fmaxf(top, fmaxf(fmaxf(s[t][0], s[t][1]), fmaxf(s[t][2], s[t][3])));
  top = fmaxf(top, __shfl_xor(top, 16));
  top = fmaxf(top, __shfl_xor(top, 32));
  const float m = fmaxf(st.m, top);
  const float base = (m == NEG_INF ? 0.0f : m) - P_SHIFT;
  const float alpha = exp2_fast(st.m - (m == NEG_INF ? 0.0f : m));
  st.m = m;
  float sum = 0;
#pragma unroll
  for (int t = 0; t < N; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s[t][i] = exp2_fast(s[t][i] - base);
      sum += s[t][i];
    }
  // a page that the row does not see adds nothing, whatever its scale
  st.l = st.l * alpha + (sum == 0.0f ? 0.0f : sum * inv_vs);
#pragma unroll
  for (int d = 0; d < Dims<D>::TILES; ++d) st.o[d] *= alpha;
}

// One row's m and l after its keys of part `slot` of `parts`; if that is all of them, its lse.
__device__ __forceinline__ void mark_row(const bs_kv_query& A, const bs_kv_batch& B, const Work& W, uint32_t slot, uint32_t parts, size_t row,
                                         float m, float l) {
  const size_t n = (size_t)B.n_rows * A.n_q_heads;
  if (parts > 1) {
    W.ml[slot * n + row] = make_float2(m, l);
    if (slot == 0)
      for (uint32_t k = parts; k < W.parts; ++k) W.ml[k * n + row] = make_float2(NEG_INF, 0.0f);
  } else {
    if (A.lse) A.lse[row] = l == 0.0f ? NEG_INF : (m - P_SHIFT + __builtin_amdgcn_logf(l)) * LN2;
    if (W.parts > 1) W.ml[row] = make_float2(NEG_INF, -1.0f);
  }
}

// 64 of a wave's pages at a time, one a lane: number (or ~0: no such page) and scales.
struct PageList {
  uint32_t id;
  float ks, vs;
  __device__ __forceinline__ void load(const bs_kv_pool& P, const int32_t* table, uint32_t h, int page, int end, int32_t* status) {
    id = ~0u;
    ks = vs = 0.0f;
    if (page >= end) return;
    id = (uint32_t)table[page];
    if (id >= P.n_pages) {
      report(status, BS_DEV_ERR_BOUNDS);
      id = ~0u;
      return;
    }
    ks = P.k_scale[(size_t)id * P.n_kv_heads + h];
    vs = P.v_scale[(size_t)id * P.n_kv_heads + h];
  }
  __device__ __forceinline__ uint32_t number(int i) const { return (uint32_t)__builtin_amdgcn_readlane((int)id, i); }
  __device__ __forceinline__ float scale_k(int i) const { return __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(ks), i)); }
  __device__ __forceinline__ float scale_v(int i) const { return __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(vs), i)); }
};

// A tile of 16 rows of a sequence and kv head, and a part of the pages that it sees: about `piece` pages each, one size
// for all sequences, so that long ones do not make long parts. The workgroup deals its pages to the four waves in turn.
// A wave reads the next page's K as soon as this one's is multiplied, and its V after this one's: between 8 and 16 KiB a
// wave are always under way (heads of 128), 64 to 128 KiB a compute unit. The bound is memory: 2 D bytes a key against
// 4 D flops a row, and at 16 rows the matrix unit and the conversions still take a quarter of the time that the bytes
// do. 128 sequences of 15,000 to 16,383 tokens, 8 kv heads of 128: 639 us, 6.4 TB/s; 64 sequences of up to 8,192: 129 us,
// 4.2 TB/s (one workgroup a sequence and head just fills the card, and the longest goes on alone); a single row over
// 1,024 tokens 13 us, which is the chain of dependent reads: the step, page numbers, pages. 168 registers a wave, for
// three waves a SIMD instead of two, spill and cost a third.
template <int D, int KIND>
__global__ __launch_bounds__(64 * WAVES, D <= 128 ? 2 : 1) void rows_kernel(bs_kv_pool P, bs_kv_batch B, bs_kv_query A, Work W,
                                                                           int32_t* status) {
  constexpr int STEPS = Dims<D>::STEPS, TILES = Dims<D>::TILES;
  constexpr int PART = D < 128 ? D : 128, PARTS = D / PART;      // channels joined at a time
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4;
  // Consecutive workgroups go to the eight dies in turn, which so get heads and not sequences. Where not all run at once,
  // the longest start first: the later parts of long sequences, then sequences by length, among 64 at a time.
  const uint32_t h = blockIdx.x, slot = gridDim.z - 1 - blockIdx.z;
  const uint32_t group = A.n_q_heads / P.n_kv_heads;
  uint32_t b = blockIdx.y;
  __shared__ __attribute__((aligned(16))) float part_o[WAVES][16][PART + 4];
  __shared__ float part_m[WAVES][16], part_l[WAVES][16];
  const float sign = A.scale < 0.0f ? -1.0f : 1.0f;
  const Score sc = {fabsf(A.softcap != 0.0f ? A.scale / A.softcap : A.scale * LOG2E), A.softcap * LOG2E};
  const bool biased = A.slopes != nullptr;
  const size_t unit = (size_t)P.n_kv_heads * PAGE * D, head = (size_t)h * PAGE * D;

  SeqStep s;
  bool sound;
  if (W.ranked) {
    const uint32_t b0 = b & ~63u, n = min(B.n_seqs - b0, 64u);
    s = {0, 0, 0, 0};
    sound = (uint32_t)lane >= n || seq_step(B, b0 + (uint32_t)lane, s);
    // no two keys are alike, whatever the lengths: each rank below n is one lane's
    const uint32_t key = (uint32_t)s.len * 64 + 63 - (uint32_t)lane;
    uint32_t rank = 0;
    for (uint32_t j = 0; j < n; ++j) rank += (uint32_t)__builtin_amdgcn_readlane((int)key, (int)j) > key;
    const int l = __builtin_ctzll(__ballot(rank == b - b0 && (uint32_t)lane < n));
    sound = __builtin_amdgcn_readlane((int)sound, l) != 0;
    s = {__builtin_amdgcn_readlane(s.t0, l), __builtin_amdgcn_readlane(s.n, l), __builtin_amdgcn_readlane(s.start, l),
         __builtin_amdgcn_readlane(s.len, l)};
    b = b0 + (uint32_t)l;
  } else {
    sound = seq_step<true>(B, b, s);
  }
  if (!sound) {
    if (threadIdx.x == 0) report(status, BS_DEV_ERR_BOUNDS);
    return;
  }
  const int rows = s.n * (int)group;
  const int32_t* table = B.table + (size_t)b * B.table_stride;

  for (int tile = 0; tile * 16 < rows; ++tile) {
    const int r = tile * 16 + (lane & 15);
    const bool real = r < rows;
    const int i = real ? r / (int)group : 0;
    const uint32_t hq = h * group + (uint32_t)(real ? r % (int)group : 0);
    const int pos = s.start + i;
    const int2 see = real ? seen_by(A, s, b, i) : make_int2(0, 0);

    // pages that any row of the tile sees, and this workgroup's piece of them
    int lo = see.x < see.y ? see.x : 0x7FFFFFFF, hi = see.x < see.y ? see.y : 0;
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) {
      lo = min(lo, __shfl_xor(lo, d));
      hi = max(hi, __shfl_xor(hi, d));
    }
    const int page_lo = __builtin_amdgcn_readfirstlane(lo >= hi ? 0 : lo / (int)PAGE);
    const int page_hi = __builtin_amdgcn_readfirstlane(lo >= hi ? 0 : (hi + (int)PAGE - 1) / (int)PAGE);
    const uint32_t parts = min((uint32_t)max((page_hi - page_lo + W.piece - 1) / W.piece, 1), W.parts);
    if (slot >= parts) continue;
    const int piece = (page_hi - page_lo + (int)parts - 1) / (int)parts;
    const int mine = min(page_lo + piece * (int)slot, page_hi), end = min(mine + piece, page_hi);
    const int full_pages = s.len / (int)PAGE, full_end = min(end, full_pages);      // pages from full_pages on are the tail

    // The tail, 16 keys of it a wave, and the first page are on their way before q is looked at. Key 4 g + e of the
    // wave's 16 belongs to lane group g, in S^T and as the right operand of the second product (of whose eight elements
    // a lane the last four are 0). Slots after the sequence's end hold anything: they count as 0.
    // (mine < end: a part that is left without pages, where there are more than the plan was made for, has no tail either.)
    const bool tailed = mine < end && end > full_pages;
    uint32_t tail = 0;
    if (tailed) {
      tail = (uint32_t)uniform_load(B.tails, 2 * (size_t)b + 1);
      if (tail >= P.n_tails && threadIdx.x == 0) report(status, BS_DEV_ERR_BOUNDS);
    }
    // of this wave's 16; a tail that does not exist is left out
    const int used = tailed && tail < P.n_tails ? s.len - full_pages * (int)PAGE - 16 * wave : 0;
    uint4 kt[STEPS];
    uint2 vt[TILES];
    const uint4 none = make_uint4(0, 0, 0, 0);
    if (used > 0) {
      const uint16_t *const kr = P.k_tail + tail * unit + head + 16 * wave * D, *const vr = P.v_tail + tail * unit + head + 16 * wave;
      const uint32_t row = (uint32_t)(lane & 15) * D, ahead = (uint32_t)(lane & 15) * PAGE + 4 * (uint32_t)g;
#pragma unroll
      for (int c = 0; c < STEPS; ++c) {
        const int ch = channel_of<D>(c, g);
        kt[c] = ((lane & 15) < used && ch < D) ? *(const uint4*)(kr + (row + (uint32_t)ch)) : none;
      }
#pragma unroll
      for (int d = 0; d < TILES; ++d) vt[d] = 4 * g < used ? *(const uint2*)(vr + (ahead + 16 * (uint32_t)d * PAGE)) : make_uint2(0, 0);
    }
    PageList list;
    list.load(P, table, h, mine + wave + WAVES * lane, full_end, status);
    const uint8_t *const kp = (const uint8_t*)P.k + head, *const vp = (const uint8_t*)P.v + head;
    PageK<D, KIND> k;
    PageV<D, KIND> v;
    uint32_t id = list.number(0);
    if (mine + wave < full_end) {
      k.load(kp + (id == ~0u ? 0 : id * unit), lane);
      v.load(vp + (id == ~0u ? 0 : id * unit), lane);
    }

    const float slope = biased ? A.slopes[hq] * LOG2E : 0.0f;
    // the row of q as f16, scaled by a power of two to lie below 2 (exact for what is within 2^-14 of the largest)
    const uint16_t* q = A.q + (int64_t)(s.t0 + i) * A.q_token + (int64_t)hq * A.q_head;
    half8v q16[STEPS];
    float row_scale;
    State<D> st;
#pragma unroll
    for (int d = 0; d < TILES; ++d) st.o[d] = f32x4{0, 0, 0, 0};
    st.m = NEG_INF;
    st.l = 0;
    {
      uint4 raw[STEPS];
      float top = 0;
      bool fine = true;
#pragma unroll
      for (int c = 0; c < STEPS; ++c) {
        const int ch = channel_of<D>(c, g);
        raw[c] = (real && ch < D) ? *(const uint4*)(q + ch) : none;
        uint16_t x[8];
        __builtin_memcpy(x, &raw[c], 16);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          fine = fine && bf16_finite(x[e]);
          top = fmaxf(top, fabsf(bf16_to_f32(x[e])));
        }
      }
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32));
      int ok = fine;
      ok &= __shfl_xor(ok, 16);
      ok &= __shfl_xor(ok, 32);
      const int e2 = (top == 0.0f || !ok) ? 0 : max((int)((__float_as_uint(top) >> 23) & 255) - 127, -100);
      row_scale = ok ? ldexpf(1.0f, e2) : __uint_as_float(0x7FC00000u);
#pragma unroll
      for (int c = 0; c < STEPS; ++c) {
        uint16_t x[8];
        __builtin_memcpy(x, &raw[c], 16);
#pragma unroll
        for (int e = 0; e < 8; ++e) q16[c][e] = ok ? (_Float16)(sign * ldexpf(bf16_to_f32(x[e]), -e2)) : (_Float16)0.0f;
      }
      // the tail: bf16 as it is; p' in two bf16 parts keeps 16 bits of it
      if (used > 0) {
        f32x4 acc[1] = {f32x4{0, 0, 0, 0}};
#pragma unroll
        for (int c = 0; c < STEPS; ++c)
          acc[0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, kt[c]), __builtin_bit_cast(bf16x8, raw[c]), acc[0], 0, 0, 0);
        scores(acc, sc, ok ? sign : row_scale, 1.0f, 0.0f, full_pages * (int)PAGE + 16 * wave + 4 * g, see, false, biased, slope, pos);
        weights<D>(acc, st, 1.0f);
        bf16x8 p_hi, p_lo;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          p_hi[e] = (__bf16)acc[0][e];
          p_lo[e] = (__bf16)(acc[0][e] - (float)p_hi[e]);
          p_hi[e + 4] = p_lo[e + 4] = (__bf16)0.0f;
        }
#pragma unroll
        for (int d = 0; d < TILES; ++d) {
          bf16x8 vb = __builtin_bit_cast(bf16x8, make_uint4(vt[d].x, vt[d].y, 0, 0));
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (4 * g + e >= used) vb[e] = (__bf16)0.0f;
          st.o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vb, p_hi, st.o[d], 0, 0, 0);
          st.o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vb, p_lo, st.o[d], 0, 0, 0);
        }
      }
    }

    if (mine + wave < full_end) {
      int at = 0;                       // place in the list
      for (int page = mine + wave; page < full_end; page += WAVES) {
        const bool ok = id != ~0u;
        const float ks = list.scale_k(at), shift = __builtin_amdgcn_logf(list.scale_v(at));
        f32x4 acc[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          acc[t] = f32x4{0, 0, 0, 0};
#pragma unroll
          for (int c = 0; c < STEPS; ++c) acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k.operand(t, c), q16[c], acc[t], 0, 0, 0);
        }
        // the next page (past the end: this one again)
        if (page + WAVES < full_end) {
          if (++at == 64) {
            at = 0;
            list.load(P, table, h, page + WAVES + WAVES * lane, full_end, status);
          }
          id = list.number(at);
        }
        const size_t next = id == ~0u ? 0 : id * unit;
        k.load(kp + next, lane);
        const int j0 = page * (int)PAGE;
        const bool inside = ok && __ballot(real && (j0 < see.x || j0 + (int)PAGE > see.y)) == 0;
        scores(acc, sc, row_scale, ks, shift, j0 + 16 * g, ok ? see : make_int2(0, 0), inside, biased, slope, pos);
        weights<D>(acc, st, exp2_fast(-shift));
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          half8v p;
#pragma unroll
          for (int e = 0; e < 8; ++e) p[e] = (_Float16)acc[2 * u + e / 4][e % 4];
#pragma unroll
          for (int d = 0; d < TILES; ++d) st.o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v.operand(d, u), p, st.o[d], 0, 0, 0);
        }
        v.load(vp + next, lane);
      }
    }

    // join the waves: rows' m and l, then O. A thread has eight channels of row tid / 16.
    st.l += __shfl_xor(st.l, 16);
    st.l += __shfl_xor(st.l, 32);
    __syncthreads();
    if (lane < 16) part_m[wave][lane] = st.m, part_l[wave][lane] = st.l;
    const int wr = (int)threadIdx.x >> 4, wc = (int)threadIdx.x & 15, wrow = tile * 16 + wr;
    const size_t out_row = (size_t)(s.t0 + (wrow < rows ? wrow / (int)group : 0)) * A.n_q_heads + h * group + (uint32_t)(wrow < rows ? wrow % (int)group : 0);
    const size_t split_row = (size_t)slot * B.n_rows * A.n_q_heads + out_row;
#pragma unroll
    for (int part = 0; part < PARTS; ++part) {
      if (part) __syncthreads();
#pragma unroll
      for (int d = 0; d < PART / 16; ++d) *(f32x4*)&part_o[wave][lane & 15][16 * d + 4 * g] = st.o[part * (PART / 16) + d];
      __syncthreads();
      float m = NEG_INF, l = 0, f[WAVES];
#pragma unroll
      for (int w = 0; w < WAVES; ++w) m = fmaxf(m, part_m[w][wr]);
#pragma unroll
      for (int w = 0; w < WAVES; ++w) {
        f[w] = exp2_fast(part_m[w][wr] - (m == NEG_INF ? 0.0f : m));
        l += part_l[w][wr] * f[w];
      }
      if (wrow >= rows) continue;
      if (part == 0 && wc == 0) mark_row(A, B, W, slot, parts, out_row, m, l);
      if (8 * wc >= PART) continue;
      float x[8] = {};
#pragma unroll
      for (int w = 0; w < WAVES; ++w)
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] += part_o[w][wr][8 * wc + e] * f[w];
      if (parts > 1) {
        float* to = W.o + split_row * D + part * PART + 8 * wc;
        *(float4*)to = make_float4(x[0], x[1], x[2], x[3]);
        *(float4*)(to + 4) = make_float4(x[4], x[5], x[6], x[7]);
      } else {
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        uint32_t y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = f32_to_bf16(x[2 * e] * inv) | ((uint32_t)f32_to_bf16(x[2 * e + 1] * inv) << 16);
        *(uint4*)(A.out + out_row * D + part * PART + 8 * wc) = make_uint4(y[0], y[1], y[2], y[3]);
      }
    }
  }
}

// Many rows: a workgroup of four waves takes 128 rows of a sequence and kv head, 32 a wave, and goes through their pages
// together. Each page is converted to f16 once, on its way into LDS (two buffers, one barrier a page, the next page's
// loads in flight meanwhile), and read from there by all four waves as the left operand of 32x32x16 products. Keys are
// numbered so that the 16 keys of a lane in a 32-key S^T tile are two runs of 8, which are its part of the right operand
// of two products with V^T: key bits 2 and 3 change places between a tile's row and the key in it. LDS rows have an odd
// number of 16-byte pieces, so that the 8 lanes of one LDS cycle hit different banks.
//
// Two workgroups a compute unit (one with heads of 256, whose o alone is 128 registers a lane). A page costs a wave 32
// products (heads of 128), about 500 ns of the matrix unit, and some 260 other vector instructions, 32 exponentials and 32
// conversions among them; the bound is how far the two waves of a SIMD run one beside the other. 8,192-token causal prompt,
// 32 and 8 heads of 128, e4m3: 565 to 585 us from run to run, 0.95 PFLOP/s, where a large f16 product of the library
// reaches 1.23; the products alone take 320. 500 tokens over a window of 16,384, heads of 256, capped: 224 us, 0.6 PFLOP/s
// (all 512 registers are in use there, and 10 to 18 more spill once a cap or a bias is set). Eight waves and 256 rows a
// workgroup, on one card: 573 us where four waves took 578, but 90 us instead of 46 for short documents. One wave a SIMD
// with the next page's scores woven into this page's weights: 800 us.
constexpr int PROMPT_WAVES = 4, PROMPT_ROWS = 32 * PROMPT_WAVES, PROMPT_THREADS = 64 * PROMPT_WAVES;

// The maximum of x over the two lanes that share a row (32 apart).
__device__ __forceinline__ float pair_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float pair_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

template <int D>
struct Tile {
  static constexpr int STEPS = D / 16;            // products over channels
  static constexpr int TILES = (D + 31) / 32;     // of 32 channels of O^T (the last may be half empty)
  static constexpr int K_ROW = D * 2 + 16;        // bytes
  static constexpr int V_ROW = PAGE * 2 + 16;
  static constexpr int K_BYTES = PAGE * K_ROW, V_BYTES = TILES * 32 * V_ROW;
  static constexpr int BYTES = K_BYTES + V_BYTES;
  static constexpr int LOADS = (PAGE * D / 16 + PROMPT_THREADS - 1) / PROMPT_THREADS;   // 16-byte loads of a thread, for K and for V
};

template <int D, int KIND>
struct Staged {      // a thread's part of a page on its way to LDS
  uint4 k[Tile<D>::LOADS], v[Tile<D>::LOADS];
  __device__ __forceinline__ void load(const uint8_t* kp, const uint8_t* vp, int tid) {
#pragma unroll
    for (int i = 0; i < Tile<D>::LOADS; ++i) {
      const int at = (tid + PROMPT_THREADS * i) * 16;
      if (PAGE * D % (16 * PROMPT_THREADS) == 0 || at < (int)PAGE * D) {
        k[i] = *(const uint4*)(kp + at);
        v[i] = *(const uint4*)(vp + at);
      }
    }
  }
  __device__ __forceinline__ void store(uint8_t* lds, int tid) const {
#pragma unroll
    for (int i = 0; i < Tile<D>::LOADS; ++i) {
      const int at = (tid + PROMPT_THREADS * i) * 16;
      if (PAGE * D % (16 * PROMPT_THREADS) == 0 || at < (int)PAGE * D) {
        const int key = at / D, ch = at % D;
        const int row = (key & 0x33) | ((key & 4) << 1) | ((key & 8) >> 1);
        uint8_t* to = lds + row * Tile<D>::K_ROW + ch * 2;
        *(half8v*)to = codes8_to_f16<KIND>(k[i].x, k[i].y);
        *(half8v*)(to + 16) = codes8_to_f16<KIND>(k[i].z, k[i].w);
        to = lds + Tile<D>::K_BYTES + at / (int)PAGE * Tile<D>::V_ROW + at % (int)PAGE * 2;
        *(half8v*)to = codes8_to_f16<KIND>(v[i].x, v[i].y);
        *(half8v*)(to + 16) = codes8_to_f16<KIND>(v[i].z, v[i].w);
      }
    }
  }
};

// N products whose left operands come from LDS, in groups of four: the next group's reads are under way while one
// group is multiplied. Left alone the compiler waits for every read right before its product.
template <int N, class Read, class Multiply>
__device__ __forceinline__ void products(Read read, Multiply multiply) {
  constexpr int G = 4;
  half8v a[2][G];
#pragma unroll
  for (int i = 0; i < G && i < N; ++i) a[0][i] = read(i);
#pragma unroll
  for (int g = 0; g * G < N; ++g) {
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < G; ++i)
      if ((g + 1) * G + i < N) a[(g + 1) & 1][i] = read((g + 1) * G + i);
#pragma unroll
    for (int i = 0; i < G; ++i)
      if (g * G + i < N) multiply(g * G + i, a[g & 1][i]);
  }
  __builtin_amdgcn_sched_barrier(0);
}

// What prompt_kernel is compiled for: no cap and no bias; a cap of at most QUICK_CAP, a bias or both; a larger cap.
enum Caps { PLAIN, QUICK, WHOLE };

// Scores of 64 keys (two S^T tiles) as they come from the products, into what is left to multiply by c and to add to
// (QUICK: the cap): caps, biases and masks where there are any. j0: this lane's first key.
template <int CAPS>
__device__ __forceinline__ void prompt_scores(f32x16 (&s)[2], float& c, const Score& sc, bool inside, int j0, int2 see, bool biased,
                                              float slope, int pos) {
  if constexpr (CAPS == WHOLE) {
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[t][i] = whole_tanh(s[t][i] * c);
    c = sc.cap;
  }
  if constexpr (CAPS != PLAIN) {
    if (CAPS == QUICK && sc.cap != 0.0f) {       // the quotient here, cap in the last step
      const float k = c * (2.0f * LOG2E);
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[t][i] = __builtin_amdgcn_rcpf(-1.0f - exp2_fast(s[t][i] * k));
      c = 2.0f * sc.cap;
    }
    if (biased) {
      float d = (float)(pos - j0);
      BS_OPAQUE(d);
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[t][i] = s[t][i] * c - slope * fabsf(d - (float)(32 * t + 16 * (i >> 3) + (i & 7)));
      c = 1.0f;
    }
  }
  if (!inside) {
    // made here and nowhere earlier: left to itself the compiler keeps 64 bounds in registers through the whole loop
    int lo = see.x - j0, hi = see.y - j0;
    BS_OPAQUE(lo);
    BS_OPAQUE(hi);
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int j = 32 * t + 16 * (i >> 3) + (i & 7);
        s[t][i] = (j >= lo && j < hi) ? s[t][i] * c : NEG_INF;
      }
    c = 1.0f;
  }
}

// Weights 2^(s c + add - m + SHIFT) from scores; m, l and o move on. The exponents are made with the maximum of the
// pages before, and only if some row's largest is over 2^SLACK times that (or the row had seen nothing) does the
// maximum move and o get rescaled: hardly ever. Weights then reach 2^(SHIFT + SLACK), inside f16, and those down to
// 2^-(SHIFT + 14) of the largest keep all 11 bits.
constexpr float SLACK = 8.0f, SHIFT = 7.0f;
template <int D>
__device__ __forceinline__ void prompt_weights(f32x16 (&s)[2], f32x16 (&o)[Tile<D>::TILES], float& m, float& l, float c, float add, float inv_vs) {
  const float base = add + SHIFT - (m == NEG_INF ? 0.0f : m);
  float top = NEG_INF;
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) s[t][i] = fmaf(s[t][i], c, base);
#pragma unroll
  for (int i = 0; i < 16; ++i) top = fmaxf(top, fmaxf(s[0][i], s[1][i]));
  top = pair_max(top);
  if (__ballot(top > (m == NEG_INF ? NEG_INF : SHIFT + SLACK))) {
    const float was = m == NEG_INF ? 0.0f : m, grown = top - SHIFT + was;      // the row's largest score
    const float now = fmaxf(m, grown);
    const float alpha = exp2_fast(m - (now == NEG_INF ? 0.0f : now));
    const float down = was - (now == NEG_INF ? 0.0f : now);
    m = now;
    l *= alpha;
#pragma unroll
    for (int d = 0; d < Tile<D>::TILES; ++d) o[d] *= alpha;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[t][i] += down;
  }
  float sum[4] = {0, 0, 0, 0};
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s[t][i] = exp2_fast(s[t][i]);
      sum[i & 3] += s[t][i];
    }
  const float all = (sum[0] + sum[1]) + (sum[2] + sum[3]);
  l += all == 0.0f ? 0.0f : all * inv_vs;
}

template <int D, int KIND, int CAPS>
__global__ __launch_bounds__(PROMPT_THREADS, D <= 128 ? 8 / PROMPT_WAVES : 1) void prompt_kernel(bs_kv_pool P, bs_kv_batch B, bs_kv_query A, Work W,
                                                                      int32_t* status) {
  constexpr int STEPS = Tile<D>::STEPS, TILES = Tile<D>::TILES;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  __shared__ int bounds[2][PROMPT_WAVES];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, half = lane >> 5;
  const uint32_t h = blockIdx.x % P.n_kv_heads, split = blockIdx.x / P.n_kv_heads, b = blockIdx.z;
  const uint32_t group = A.n_q_heads / P.n_kv_heads;
  SeqStep s;
  if (!seq_step<true>(B, b, s)) {
    if (tid == 0) report(status, BS_DEV_ERR_BOUNDS);
    return;
  }
  const int rows = s.n * (int)group;
  const float sign = A.scale < 0.0f ? -1.0f : 1.0f;
  const Score sc = {fabsf(A.softcap != 0.0f ? A.scale / A.softcap : A.scale * LOG2E), A.softcap * LOG2E};
  const bool biased = A.slopes != nullptr;
  const size_t unit = (size_t)P.n_kv_heads * PAGE * D, head = (size_t)h * PAGE * D;
  const int full_pages = s.len / (int)PAGE, row_tiles = (rows + PROMPT_ROWS - 1) / PROMPT_ROWS;

  // the last tiles, which see most under a causal mask, come first
  for (int tile = row_tiles - 1 - (int)blockIdx.y; tile >= 0; tile -= (int)gridDim.y) {
    const int r = tile * PROMPT_ROWS + wave * 32 + (lane & 31);
    const bool real = r < rows;
    const int i = real ? r / (int)group : 0;
    const uint32_t hq = h * group + (uint32_t)(real ? r % (int)group : 0);
    const int pos = s.start + i;
    int2 see = real ? seen_by(A, s, b, i) : make_int2(0, 0);
    const float slope = CAPS != PLAIN && biased ? A.slopes[hq] * LOG2E : 0.0f;

    const uint16_t* q = A.q + (int64_t)(s.t0 + i) * A.q_token + (int64_t)hq * A.q_head;
    uint4 raw[STEPS];
#pragma unroll
    for (int c = 0; c < STEPS; ++c) raw[c] = real ? *(const uint4*)(q + 16 * c + 8 * half) : make_uint4(0, 0, 0, 0);

    // keys that any row of the wave, and of the workgroup, sees
    int lo = see.x < see.y ? see.x : 0x7FFFFFFF, hi = see.x < see.y ? see.y : 0;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      lo = min(lo, __shfl_xor(lo, d));
      hi = max(hi, __shfl_xor(hi, d));
    }
    const int wave_lo = __builtin_amdgcn_readfirstlane(lo), wave_hi = __builtin_amdgcn_readfirstlane(hi);
    lds_barrier();
    if (lane == 0) bounds[0][wave] = lo, bounds[1][wave] = hi;
    lds_barrier();
#pragma unroll
    for (int w = 0; w < PROMPT_WAVES; ++w) lo = min(lo, bounds[0][w]), hi = max(hi, bounds[1][w]);
    const int page_lo = lo >= hi ? 0 : lo / (int)PAGE, page_hi = lo >= hi ? 0 : (hi + (int)PAGE - 1) / (int)PAGE;
    const int per = (page_hi - page_lo + (int)W.parts - 1) / (int)W.parts;
    const int begin = __builtin_amdgcn_readfirstlane(page_lo + per * (int)split);
    const int end = __builtin_amdgcn_readfirstlane(min(begin + per, page_hi));
    const int full_end = min(end, full_pages);

    // Page numbers and scales come through vector loads, in line with the pages' own: number n is asked for with page
    // n - 1, scales with their page, so that nothing waits for them. Past the end: the last page again.
    const int32_t* table = B.table + (size_t)b * B.table_stride;
    int zero = 0;
    BS_OPAQUE(zero);                          // (an index of the lanes' own keeps the loads out of the scalar cache)
    const auto number = [&](int page) { return table[min(page, full_end - 1) + zero]; };
    Staged<D, KIND> st;
    uint32_t id = 0;
    int coming = 0;
    float next_ks = 0, next_vs = 1;
    const auto fetch = [&](int page) {
      id = (uint32_t)__builtin_amdgcn_readfirstlane(coming);
      const uint32_t real_id = id < P.n_pages ? id : 0;
      next_ks = P.k_scale[(size_t)real_id * P.n_kv_heads + h + zero];
      next_vs = P.v_scale[(size_t)real_id * P.n_kv_heads + h + zero];
      coming = number(page + 1);
      st.load((const uint8_t*)P.k + real_id * unit + head, (const uint8_t*)P.v + real_id * unit + head, tid);
    };
    if (begin < full_end) {
      coming = number(begin);
      fetch(begin);
    }
    // with the first page on its way: the row of q as f16, scaled by a power of two to lie below 2
    half8v q16[STEPS];
    float row_scale;
    {
      uint16_t x[STEPS][8];
      float top = 0;
      bool fine = true;
#pragma unroll
      for (int c = 0; c < STEPS; ++c) {
        __builtin_memcpy(x[c], &raw[c], 16);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          fine = fine && bf16_finite(x[c][e]);
          top = fmaxf(top, fabsf(bf16_to_f32(x[c][e])));
        }
      }
      top = pair_max(top);
      const bool ok = pair_max(fine ? 0.0f : 1.0f) == 0.0f;
      const int e2 = (top == 0.0f || !ok) ? 0 : max((int)((__float_as_uint(top) >> 23) & 255) - 127, -100);
      row_scale = ok ? ldexpf(1.0f, e2) : __uint_as_float(0x7FC00000u);
#pragma unroll
      for (int c = 0; c < STEPS; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) q16[c][e] = ok ? (_Float16)(sign * ldexpf(bf16_to_f32(x[c][e]), -e2)) : (_Float16)0.0f;
    }

    f32x16 o[TILES];
#pragma unroll
    for (int d = 0; d < TILES; ++d)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[d][e] = 0;
    float m = NEG_INF, l = 0;

    for (int page = begin; page < full_end; ++page) {
      uint8_t* buf = lds + ((page - begin) & 1) * Tile<D>::BYTES;
      st.store(buf, tid);
      const bool ok = id < P.n_pages;
      if (!ok && tid == 0) report(status, BS_DEV_ERR_BOUNDS);
      const float ks = next_ks, shift = __builtin_amdgcn_logf(next_vs);
      fetch(page + 1);
      lds_barrier();
      const int j0 = page * (int)PAGE;
      if (!ok || j0 >= wave_hi || j0 + (int)PAGE <= wave_lo) continue;
      f32x16 acc[2];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[t][e] = 0;
      const uint8_t* kr = buf + (lane & 31) * Tile<D>::K_ROW + 16 * half;
      products<2 * STEPS>([&](int n) { return *(const half8v*)(kr + n % 2 * 32 * Tile<D>::K_ROW + n / 2 * 32); },
                          [&](int n, half8v a) { acc[n % 2] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, q16[n / 2], acc[n % 2], 0, 0, 0); });
      const bool inside = __ballot(real && (j0 < see.x || j0 + (int)PAGE > see.y)) == 0;
      float c = row_scale * (ks * sc.scale);
      prompt_scores<CAPS>(acc, c, sc, inside, j0 + 8 * half, see, biased, slope, pos);
      prompt_weights<D>(acc, o, m, l, c, CAPS == WHOLE ? shift : shift + sc.cap, exp2_fast(-shift));
      half8v p[4];
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int e = 0; e < 8; ++e) p[u][e] = (_Float16)acc[u >> 1][8 * (u & 1) + e];
      const uint8_t* vr = buf + Tile<D>::K_BYTES + (lane & 31) * Tile<D>::V_ROW + 16 * half;
      products<4 * TILES>([&](int n) { return *(const half8v*)(vr + n % TILES * 32 * Tile<D>::V_ROW + n / TILES * 32); },
                          [&](int n, half8v a) { o[n % TILES] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, p[n / TILES], o[n % TILES], 0, 0, 0); });
    }

    // the tail: bf16 as it is; p' in two bf16 parts keeps 16 bits of it. Slots after the sequence's end hold anything.
    if (begin < end && end > full_pages && full_pages * (int)PAGE < wave_hi) {
      const uint32_t id = (uint32_t)uniform_load(B.tails, 2 * (size_t)b + 1);
      if (id >= P.n_tails) {
        if (lane == 0) report(status, BS_DEV_ERR_BOUNDS);
      } else {
        const uint16_t* kt = P.k_tail + id * unit + head;
        const uint16_t* vt = P.v_tail + id * unit + head;
        const int used = s.len - full_pages * (int)PAGE;
        const uint4 none = make_uint4(0, 0, 0, 0);
        f32x16 acc[2];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[t][e] = 0;
        const int row = lane & 31, key0 = (row & 0x13) | ((row & 4) << 1) | ((row & 8) >> 1);
#pragma unroll
        for (int c = 0; c < STEPS; ++c) {
          const bf16x8 qb = __builtin_bit_cast(bf16x8, real ? *(const uint4*)(q + 16 * c + 8 * half) : none);
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const int key = 32 * t + key0;
            const bf16x8 kb = __builtin_bit_cast(bf16x8, key < used ? *(const uint4*)(kt + key * D + 16 * c + 8 * half) : none);
            acc[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kb, qb, acc[t], 0, 0, 0);
          }
        }
        if (sign < 0.0f)
#pragma unroll
          for (int t = 0; t < 2; ++t) acc[t] = -acc[t];
        float c = row_scale == row_scale ? sc.scale : row_scale;
        prompt_scores<CAPS>(acc, c, sc, false, full_pages * (int)PAGE + 8 * half, see, biased, slope, pos);
        prompt_weights<D>(acc, o, m, l, c, CAPS == WHOLE ? 0.0f : sc.cap, 1.0f);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          bf16x8 p_hi, p_lo;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float x = acc[u >> 1][8 * (u & 1) + e];
            p_hi[e] = (__bf16)x;
            p_lo[e] = (__bf16)(x - (float)p_hi[e]);
          }
          const int key = 16 * u + 8 * half;
#pragma unroll
          for (int d = 0; d < TILES; ++d) {
            const int ch = 32 * d + (lane & 31);
            bf16x8 vb = __builtin_bit_cast(bf16x8, ch < D ? *(const uint4*)(vt + ch * PAGE + key) : none);
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (key + e >= used) vb[e] = (__bf16)0.0f;
            o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vb, p_hi, o[d], 0, 0, 0);
            o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vb, p_lo, o[d], 0, 0, 0);
          }
        }
      }
    }

    l = pair_sum(l);
    if (real) {
      const size_t out_row = (size_t)(s.t0 + i) * A.n_q_heads + hq;
      if (half == 0) mark_row(A, B, W, split, W.parts, out_row, m + (P_SHIFT - SHIFT), l);
      if (W.parts == 1 || begin < end) {
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        float* part = W.o + ((size_t)split * B.n_rows * A.n_q_heads + out_row) * D;
#pragma unroll
        for (int d = 0; d < TILES; ++d)
#pragma unroll
          for (int a = 0; a < 4; ++a) {
            const int ch = 32 * d + 8 * a + 4 * half;
            if (ch >= D) continue;
            if (W.parts > 1) {
              *(float4*)(part + ch) = make_float4(o[d][4 * a], o[d][4 * a + 1], o[d][4 * a + 2], o[d][4 * a + 3]);
            } else {
              uint2 w;
              w.x = f32_to_bf16(o[d][4 * a] * inv) | ((uint32_t)f32_to_bf16(o[d][4 * a + 1] * inv) << 16);
              w.y = f32_to_bf16(o[d][4 * a + 2] * inv) | ((uint32_t)f32_to_bf16(o[d][4 * a + 3] * inv) << 16);
              *(uint2*)(A.out + out_row * D + ch) = w;
            }
          }
      }
    }
  }
}

// Rows' parts into the output, WAVES_A_ROW waves (1 or 4) a row: they deal the parts among them, 64 at a time; lane k
// looks at its wave's k-th, then all lanes add up those that hold something, eight loads at a time. Latency: 3 to 5 us.
template <int D, int WAVES_A_ROW>
__global__ __launch_bounds__(256) void join_kernel(bs_kv_query A, Work W, uint32_t n) {
  constexpr int EACH = (D + 63) / 64, AT_ONCE = 8;
  __shared__ float part_x[4][EACH * 64], part_m[4], part_l[4];
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t share = WAVES_A_ROW == 4 ? wave : 0;
  const uint32_t row = WAVES_A_ROW == 4 ? blockIdx.x : blockIdx.x * 4 + wave;
  if (row >= n || W.ml[row].y < 0.0f) return;            // none, or written by its kernel
  float m = NEG_INF, l = 0, x[EACH] = {};
  for (uint32_t k0 = 0; k0 < W.parts; k0 += 64 * WAVES_A_ROW) {
    const uint32_t mine = k0 + lane * WAVES_A_ROW + share;
    float2 ml = make_float2(NEG_INF, 0.0f);
    if (mine < W.parts) ml = W.ml[(size_t)mine * n + row];
    const float now = fmaxf(m, wave_max(ml.x)), ref = now == NEG_INF ? 0.0f : now;
    const float back = exp2_fast(m - ref), f = exp2_fast(ml.x - ref);
    m = now;
    l = l * back + ml.y * f;                             // (of this lane's slots)
#pragma unroll
    for (int c = 0; c < EACH; ++c) x[c] *= back;
    uint64_t some = __ballot(!(ml.x == NEG_INF && ml.y == 0.0f));
    while (some) {
      float fk[AT_ONCE], o[AT_ONCE][EACH];
#pragma unroll
      for (int u = 0; u < AT_ONCE; ++u) {
        const bool any = some != 0;
        const int k = any ? __builtin_ctzll(some) : 0;
        some &= some - 1;
        fk[u] = any ? __shfl(f, k) : 0.0f;
        const float* from = W.o + ((size_t)(k0 + (uint32_t)k * WAVES_A_ROW + share) * n + row) * D;
#pragma unroll
        for (int c = 0; c < EACH; ++c) o[u][c] = any && (int)lane + 64 * c < D ? from[lane + 64 * c] : 0.0f;
      }
#pragma unroll
      for (int u = 0; u < AT_ONCE; ++u)
#pragma unroll
        for (int c = 0; c < EACH; ++c) x[c] += o[u][c] * fk[u];
    }
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) l += __shfl_xor(l, d);
  if constexpr (WAVES_A_ROW == 4) {
#pragma unroll
    for (int c = 0; c < EACH; ++c) part_x[wave][lane + 64 * c] = x[c];
    if (lane == 0) part_m[wave] = m, part_l[wave] = l;
    __syncthreads();
    if (wave) return;
    m = fmaxf(fmaxf(part_m[0], part_m[1]), fmaxf(part_m[2], part_m[3]));
    l = 0;
#pragma unroll
    for (int c = 0; c < EACH; ++c) x[c] = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = exp2_fast(part_m[w] - (m == NEG_INF ? 0.0f : m));
      l += part_l[w] * f;
#pragma unroll
      for (int c = 0; c < EACH; ++c) x[c] += part_x[w][lane + 64 * c] * f;
    }
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
  for (int c = 0; c < EACH; ++c)
    if ((int)lane + 64 * c < D) A.out[(size_t)row * D + lane + 64 * c] = f32_to_bf16(x[c] * inv);
  if (A.lse && lane == 0) A.lse[row] = l == 0.0f ? NEG_INF : (m - P_SHIFT + __builtin_amdgcn_logf(l)) * LN2;
}

// Launch shapes of a call. FEW_ROWS: rows of a sequence and kv head up to which rows_kernel takes a step. (64 sequences
// of up to 8,192 tokens, 4 rows, us: 131 there, 193 in prompt_kernel; of up to 12,000, 4 to 16 rows: 206 and 265. With
// more than one tile of rows it would read every page again. Where sequences differ, prompt_kernel takes all of them: the
// same caches with 4 to 32 rows 275 us, against 410 with the two kernels one after the other. That holds for caches of
// that size: a prompt of 2,048 tokens beside 63 single tokens on caches of 1,000 to 100,000 takes 3,380 us, where the two
// alone take 66 and 729, because the prompt's tiles fill the card and the long caches are not split.)
constexpr uint32_t FEW_ROWS = 16;

struct Plan {
  bool few;              // rows_kernel, else prompt_kernel
  uint32_t tiles;        // of 16 or PROMPT_ROWS rows, of the sequence that has most
  uint32_t parts, piece; // pages are cut into at most so many parts; rows_kernel: of so many pages
};

constexpr uint64_t RESIDENT = 512;       // workgroups of 256 threads that run at once, two on each of 256 compute units

uint32_t split_for(uint64_t blocks, uint64_t want, uint64_t pages, uint64_t least) {
  const uint64_t n = blocks >= want ? 1 : (want + blocks - 1) / blocks;
  return (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>(n, pages / least));
}

// Pieces of a cache of `pages` pages, `blocks` tiles of rows in all: as many as fill the card, of 4 pages (one a wave)
// at least, and of 16 once there are 32, since every piece costs the joining kernel. Up to 16 pages a workgroup is done
// before a second kernel has begun. Not where sequences differ: with blocks enough for the card a step is not split, and
// 63 sequences near 1,000 tokens with one of 131,072 take 890 us, where the two alone take 50 and 59. (One row, heads of 128, 8 kv heads, us a call with one piece / pieces of 4 / 8 / 16
// pages: 1,000 tokens 13.5 / 16.2 / 16.3 / 13.5, 4,000 tokens 36.8 / 17.0 / 18.9 / 23.5, 16,000 tokens - / 22.1 / 20.2 / 22.5,
// 32,000 tokens - / 26.8 / 28.6 / 24.4. As the rule has it: 256 tokens 9.5, 512 10.5, 1,024 14.0, 1,500 14.1, 2,048 13.3, 3,000 14.7.)
uint32_t pieces_for(uint64_t blocks, uint64_t pages) {
  if (pages <= 16) return 1;
  return split_for(blocks, RESIDENT, std::min<uint64_t>(pages / 4, std::max<uint64_t>(32, pages / 16)), 1);
}

Plan make_plan(const bs_kv_pool* P, const bs_kv_batch* B, uint32_t n_q_heads) {
  const uint64_t group = n_q_heads / P->n_kv_heads, heads = P->n_kv_heads, seqs = B->n_seqs;
  const uint64_t rows = std::max<uint64_t>(B->max_new * group, 1), pages = std::max<uint64_t>((B->max_len + PAGE - 1) / PAGE, 1);
  Plan p = {rows <= FEW_ROWS, 1, 1, 0};
  if (p.few) {
    p.parts = pieces_for(heads * seqs, pages);
    p.piece = (uint32_t)((pages + p.parts - 1) / p.parts);
  } else {
    p.tiles = (uint32_t)std::min<uint64_t>((rows + PROMPT_ROWS - 1) / PROMPT_ROWS, 65535);
    // tiles that the sequences can have in all, if max_new is what it says; one workgroup a compute unit with heads of 256
    const uint64_t tiles = std::max<uint64_t>(std::min<uint64_t>(p.tiles * seqs, B->n_rows * group / PROMPT_ROWS + seqs), 1);
    p.parts = split_for(tiles * heads, P->head_dim > 128 ? RESIDENT / 2 : RESIDENT, pages, 8);
  }
  return p;
}

uint64_t split_rows(const bs_kv_batch* B, uint32_t n_q_heads, const Plan& p) {
  return p.parts > 1 ? (uint64_t)p.parts * B->n_rows * n_q_heads : 0;
}

template <int D, int KIND, int CAPS>
void prompt_launch(const bs_kv_pool* P, const bs_kv_batch* B, const bs_kv_query* Q, const Work& w, int32_t* status, hipStream_t stream,
                   dim3 grid) {
  static std::atomic<uint64_t> done{0};
  bs_internal::ensure_lds_limit((const void*)prompt_kernel<D, KIND, CAPS>, 2 * Tile<D>::BYTES, done);
  prompt_kernel<D, KIND, CAPS><<<grid, PROMPT_THREADS, 2 * Tile<D>::BYTES, stream>>>(*P, *B, *Q, w, status);
}

template <int D, int KIND>
int launch(const bs_kv_pool* P, const bs_kv_batch* B, const bs_kv_query* given, void* work, int32_t* status, hipStream_t stream) {
  // A cap outside [2^-60, 2^60] does to f32 scores what the nearer end does (below 2^48 they pass whole; all become 0), and
  // the quotients by it would leave f32's range.
  bs_kv_query query = *given;
  if (query.softcap != 0.0f) query.softcap = std::min(std::max(query.softcap, 0x1p-60f), 0x1p60f);
  const bs_kv_query* const Q = &query;
  const Plan p = make_plan(P, B, Q->n_q_heads);
  const uint64_t rows = split_rows(B, Q->n_q_heads, p);
  const bool ranked = (uint64_t)P->n_kv_heads * B->n_seqs * p.parts > RESIDENT && B->n_seqs > 1;
  const Work w = {(float*)work, (float2*)((char*)work + rows * D * 4), p.parts, (int)p.piece, ranked};
  if (p.few) {
    rows_kernel<D, KIND><<<dim3(P->n_kv_heads, B->n_seqs, p.parts), 64 * WAVES, 0, stream>>>(*P, *B, *Q, w, status);
  } else {
    const dim3 grid(P->n_kv_heads * p.parts, p.tiles, B->n_seqs);
    if (Q->softcap > QUICK_CAP) prompt_launch<D, KIND, WHOLE>(P, B, Q, w, status, stream, grid);
    else if (Q->softcap != 0.0f || Q->slopes) prompt_launch<D, KIND, QUICK>(P, B, Q, w, status, stream, grid);
    else prompt_launch<D, KIND, PLAIN>(P, B, Q, w, status, stream, grid);
  }
  if (p.parts > 1) {
    const uint32_t n = B->n_rows * Q->n_q_heads;
    // Four waves a row from 8 parts on (64 rows of 64 parts: 5 us, with one wave 25).
    if (p.parts > 8) join_kernel<D, 4><<<n, 256, 0, stream>>>(*Q, w, n);
    else join_kernel<D, 1><<<(n + 3) / 4, 256, 0, stream>>>(*Q, w, n);
  }
  return hipGetLastError() == hipSuccess ? BS_OK : BS_ERR_HIP;
}

bool heads_ok(const bs_kv_pool* P, uint32_t n_q_heads) { return n_q_heads > 0 && n_q_heads % P->n_kv_heads == 0; }

}  // namespace

extern "C" uint64_t bs_kv_attend_work_bytes(const bs_kv_pool* P, const bs_kv_batch* B, uint32_t n_q_heads) {
  if (!check_pool(P) || !check_batch(B) || !heads_ok(P, n_q_heads) || B->n_rows == 0 || B->n_seqs == 0) return 0;
  return split_rows(B, n_q_heads, make_plan(P, B, n_q_heads)) * (P->head_dim * 4ull + 8);
}

extern "C" int bs_kv_attend(const bs_kv_pool* P, const bs_kv_batch* B, const bs_kv_query* Q, void* d_work, uint64_t work_bytes,
                            int32_t* d_status, void* stream) {
  if (!check_pool(P) || !check_batch(B) || !Q || !heads_ok(P, Q->n_q_heads)) return BS_ERR_ARG;
  if (B->n_rows == 0 || B->n_seqs == 0) return BS_OK;
  if (!Q->q || !Q->out || (((uintptr_t)Q->q | (uintptr_t)Q->out) & 15) || (Q->q_token & 7) || (Q->q_head & 7)) return BS_ERR_ARG;
  if (!(Q->softcap >= 0.0f) || B->n_seqs > 65535) return BS_ERR_ARG;
  if (bs_kv_attend_work_bytes(P, B, Q->n_q_heads) > work_bytes || (work_bytes && (!d_work || ((uintptr_t)d_work & 15)))) return BS_ERR_CAP;
  hipStream_t s = (hipStream_t)stream;
#define BS_KV_GO(D)                                                                     \
  return P->kind == BS_KV_FP8 ? launch<D, BS_KV_FP8>(P, B, Q, d_work, d_status, s)      \
                              : launch<D, BS_KV_INT8>(P, B, Q, d_work, d_status, s)
  switch (P->head_dim) {
    case 64: BS_KV_GO(64);
    case 80: BS_KV_GO(80);
    case 96: BS_KV_GO(96);
    case 128: BS_KV_GO(128);
    default: BS_KV_GO(256);
  }
#undef BS_KV_GO
}
