// Filling and reading back the paged 8-bit KV cache.
//
// bs_kv_append: one workgroup per (page that the step touches, kv head). It
// rotates the q rows of the head's group and the K rows, and holds the page's K
// in registers and its V, as bf16, in LDS, where V turns from rows of channels
// into rows of tokens. If the step completes the page, the largest |x| of K and
// of V give its scales and both go out as codes; the page's earlier tokens come
// from the sequence's old tail. Otherwise the new tokens go into the tail. A
// page is written by one workgroup in one go, so nothing is summed across
// workgroups and a step run again writes the same bytes. The bound is memory: q
// in and out, k and v in, 8-bit codes out. 32,768 tokens of 32 and 8 heads of 128:
// 161 us, 4.7 TB/s, where a large copy reaches 5.1. One token: 4.5 us of kernel,
// two dependent reads (the step's lengths, then rows and angles) and the launch.
//
// bs_kv_read: one workgroup per (page, kv head), codes times scale; V turns back
// in LDS. 32,768 tokens, 8 heads of 128: 45 us from memory, 4.5 TB/s.
#include "kv_common.h"

#include <algorithm>

namespace {

using namespace bs_kv;

constexpr uint32_t THREADS = 256, DIES = 8;

// Largest |x| of a page held to this range: a scale stays a normal f32 number,
// and so do its inverse and the products of attention's weights with it.
constexpr float AMAX_LO = 0x1p-40f, AMAX_HI = 0x1p60f;

template <int KIND>
__device__ __forceinline__ float qmax() { return KIND == BS_KV_FP8 ? 448.0f : 127.0f; }

// Two values as two codes in the low 16 bits.
template <int KIND>
__device__ __forceinline__ uint32_t quantise2(float x, float y, float inv) {
#pragma clang fp contract(off)
  const float q = qmax<KIND>();
  x = fminf(fmaxf(x * inv, -q), q);
  y = fminf(fmaxf(y * inv, -q), q);
  if constexpr (KIND == BS_KV_FP8)
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x, y, 0, false) & 0xFFFFu;
  else
    return ((uint32_t)(int)rintf(x) & 0xFFu) | (((uint32_t)(int)rintf(y) & 0xFFu) << 8);
}

template <int N>
struct alignas(2 * N) Half {
  uint16_t x[N];
};

// The page numbered `unit` among all pages that the step touches, sequence by
// sequence: its sequence and its place in it. Every wave counts for itself, 64
// sequences at a time; those of the first page, where a status is asked for, go on to
// the last sequence to report lengths and offsets that make no sense.
__device__ bool find_unit(const bs_kv_batch& B, uint32_t unit, uint32_t& b, uint32_t& page, SeqStep& step, int32_t* status) {
  const uint32_t lane = threadIdx.x & 63;
  uint32_t base = 0;
  bool found = false;
  for (uint32_t b0 = 0; b0 < B.n_seqs; b0 += 64) {
    uint32_t pages = 0, at = 0;
    SeqStep s = {0, 0, 0, 0};
    if (b0 + lane < B.n_seqs) {
      if (!seq_step(B, b0 + lane, s) && unit == 0) report(status, BS_DEV_ERR_BOUNDS);
      at = (uint32_t)s.start / PAGE;
      if (s.n > 0) pages = (uint32_t)(s.len - 1) / PAGE - at + 1;
    }
    uint32_t incl = pages;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const uint32_t up = __shfl_up(incl, d);
      if (lane >= (uint32_t)d) incl += up;
    }
    const uint64_t past = __ballot(base + incl > unit);
    if (past && !found) {
      const int l = __builtin_ctzll(past);
      b = b0 + (uint32_t)l;
      page = (uint32_t)__builtin_amdgcn_readlane((int)(at + unit - (base + incl - pages)), l);
      step.t0 = __builtin_amdgcn_readlane(s.t0, l), step.n = __builtin_amdgcn_readlane(s.n, l);
      step.start = __builtin_amdgcn_readlane(s.start, l), step.len = __builtin_amdgcn_readlane(s.len, l);
      if (unit != 0 || !status) return true;
      found = true;
    }
    base += (uint32_t)__builtin_amdgcn_readlane((int)incl, 63);
  }
  return found;
}

// One token's 2 * VEC channels: VEC pairs that turn together, or as many channels that do not turn.
template <int VEC>
struct Item {
  int a, b;   // channels of the two vectors
  int angle;  // column of cos and sin, -1: no turn
};
template <int VEC>
__device__ __forceinline__ Item<VEC> item_at(const bs_kv_rows& R, uint32_t it) {
  const int i = (int)it * VEC;
  if (2 * i < (int)R.rot) return R.interleaved ? Item<VEC>{2 * i, 2 * i + VEC, i} : Item<VEC>{i, i + (int)R.rot / 2, i};
  return {2 * i, 2 * i + VEC, -1};
}

// x[0..2V) of an item turned by cos, sin and rounded to bf16. The products and the sum round one by one, as separate
// f32 operations do.
template <int VEC>
__device__ __forceinline__ void turn(const float* c, const float* s, bool interleaved, Half<VEC>& va, Half<VEC>& vb) {
#pragma clang fp contract(off)
  uint16_t* e[2] = {va.x, vb.x};
  if (interleaved) {
#pragma unroll
    for (int p = 0; p < VEC; ++p) {
      uint16_t &x = e[2 * p / VEC][2 * p % VEC], &y = e[(2 * p + 1) / VEC][(2 * p + 1) % VEC];
      const float a = bf16_to_f32(x), b = bf16_to_f32(y);
      x = f32_to_bf16(a * c[p] - b * s[p]);
      y = f32_to_bf16(b * c[p] + a * s[p]);
    }
  } else {
#pragma unroll
    for (int p = 0; p < VEC; ++p) {
      const float a = bf16_to_f32(va.x[p]), b = bf16_to_f32(vb.x[p]);
      va.x[p] = f32_to_bf16(a * c[p] - b * s[p]);
      vb.x[p] = f32_to_bf16(b * c[p] + a * s[p]);
    }
  }
}

template <int VEC>
__device__ __forceinline__ Half<VEC> load_half(const uint16_t* p) {
  return *(const Half<VEC>*)p;
}

template <int VEC>
__device__ __forceinline__ void load_angles(const bs_kv_rows& R, int pos, int column, float* c, float* s) {
  const size_t at = (size_t)pos * (R.rot / 2) + (size_t)column;
#pragma unroll
  for (int i = 0; i < VEC; i += 4) {      // rot is a multiple of 8, so rows of angles are multiples of 16 bytes
    *(float4*)(c + i) = *(const float4*)(R.cos + at + i);
    *(float4*)(s + i) = *(const float4*)(R.sin + at + i);
  }
}

template <int D, int VEC, int KIND>
__global__ __launch_bounds__(THREADS) void append_kernel(bs_kv_pool P, bs_kv_batch B, bs_kv_rows R, int32_t* status) {
  constexpr uint32_t ITEMS = D / (2 * VEC);                       // of one token
  constexpr uint32_t NI = (PAGE * ITEMS + THREADS - 1) / THREADS; // of one thread, for a whole page
  constexpr uint32_t ROW = D / 2 + 1;                             // dwords of a token's V in LDS: rows start in different banks
  __shared__ uint32_t vt[PAGE * ROW];
  __shared__ int poisoned[PAGE];
  __shared__ float tops[2][THREADS / 64];
  // Consecutive workgroups go to the eight dies in turn. The heads of one page go to one die, one after another, which
  // then reads their tokens' angles once (32,768 tokens: with the heads of a page on eight dies a tenth more time).
  const uint32_t tid = threadIdx.x, turn_of = blockIdx.x / DIES, h = turn_of % P.n_kv_heads;
  uint32_t b, page;
  SeqStep s;
  if (!find_unit(B, turn_of / P.n_kv_heads * DIES + blockIdx.x % DIES, b, page, s, status)) return;
  const int p0 = (int)(page * PAGE);
  const int old = max(s.start - p0, 0), have = min(s.len - p0, (int)PAGE);  // slots [0, old) are in the tail, [old, have) are new
  const bool full = have == (int)PAGE;
  const int t_first = s.t0 + p0 - s.start;                                  // the row of slot 0 (old slots have none)
  const uint32_t tail_in = (uint32_t)uniform_load(B.tails, 2 * (size_t)b), tail_out = (uint32_t)uniform_load(B.tails, 2 * (size_t)b + 1);
  const uint32_t id = (uint32_t)uniform_load(B.table, (size_t)b * B.table_stride + page);
  // the page's earlier tokens are needed to quantise it, or where the tail moves without a page being completed
  const bool from_tail = old > 0 && (full || tail_in != tail_out);
  const int lo = from_tail ? 0 : old;
  bool ok = (full ? id < P.n_pages : tail_out < P.n_tails) && (!from_tail || tail_in < P.n_tails);
  if (R.rot && (uint32_t)s.len > R.n_pos) ok = false;
  if (!ok) {
    if (tid == 0) report(status, BS_DEV_ERR_BOUNDS);
    return;
  }
  const size_t head = (size_t)h * PAGE * D;
  const size_t unit_elems = (size_t)P.n_kv_heads * PAGE * D;
  const uint16_t* kt_in = P.k_tail + (from_tail ? tail_in * unit_elems : 0) + head;
  const uint16_t* vt_in = P.v_tail + (from_tail ? tail_in * unit_elems : 0) + head;

  if (tid < PAGE) poisoned[tid] = 0;
  __syncthreads();

  // The q heads of the group, new tokens only. With few tokens the heads go to different threads, with many one thread
  // turns its channels in every head by the angles it has loaded. From the last thread on down: of a single token, q is
  // the last waves' and k and v the first one's, side by side.
  if (R.q) {
    const uint32_t group = R.n_q_heads / P.n_kv_heads, tokens = (uint32_t)(have - old);
    const uint32_t spread = tokens * ITEMS >= THREADS ? 1 : group;
    for (uint32_t idx = THREADS - 1 - tid; idx < tokens * spread * ITEMS; idx += THREADS) {
      const Item<VEC> it = item_at<VEC>(R, idx % ITEMS);
      const uint32_t rest = idx / ITEMS;
      const int slot = old + (int)(rest / spread);
      const int64_t t = t_first + slot;
      float c[VEC], sn[VEC];
      if (it.angle >= 0) load_angles<VEC>(R, p0 + slot, it.angle, c, sn);
      for (uint32_t g = rest % spread; g < group; g += spread) {
        const int64_t hq = (int64_t)h * group + g;
        const uint16_t* q = R.q + t * R.q_token + hq * R.q_head;
        uint16_t* o = R.q_out + (t * R.n_q_heads + hq) * D;
        Half<VEC> a = load_half<VEC>(q + it.a), e = load_half<VEC>(q + it.b);
        if (it.angle >= 0) turn<VEC>(c, sn, R.interleaved, a, e);
        *(Half<VEC>*)(o + it.a) = a;
        *(Half<VEC>*)(o + it.b) = e;
      }
    }
  }

  // K into registers, V into LDS
  Half<VEC> ka[NI], kb[NI];
  float kmax = 0, vmax = 0;
#pragma unroll
  for (uint32_t i = 0; i < NI; ++i) {
    const uint32_t idx = tid + i * THREADS;
    const int slot = (int)(idx / ITEMS);
    if (slot < lo || slot >= have) continue;
    const Item<VEC> it = item_at<VEC>(R, idx % ITEMS);
    bool fine = true;
    if (slot < old) {
      ka[i] = load_half<VEC>(kt_in + slot * D + it.a);
      kb[i] = load_half<VEC>(kt_in + slot * D + it.b);
    } else {
      const int64_t t = t_first + slot;
      const uint16_t* k = R.k + t * R.k_token + (int64_t)h * R.k_head;
      const uint16_t* v = R.v + t * R.v_token + (int64_t)h * R.v_head;
      ka[i] = load_half<VEC>(k + it.a);
      kb[i] = load_half<VEC>(k + it.b);
      // of V any two vectors of the token will do: the same channels keep the loads alike
      Half<VEC> v2[2] = {load_half<VEC>(v + it.a), load_half<VEC>(v + it.b)};
      if (it.angle >= 0) {
        float c[VEC], sn[VEC];
        load_angles<VEC>(R, p0 + slot, it.angle, c, sn);
        turn<VEC>(c, sn, R.interleaved, ka[i], kb[i]);
      }
#pragma unroll
      for (int p = 0; p < 2; ++p) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          if (!bf16_finite(v2[p].x[e])) {
            fine = false;
            v2[p].x[e] = 0;
          }
          vmax = fmaxf(vmax, fabsf(bf16_to_f32(v2[p].x[e])));
        }
        uint32_t* row = vt + slot * ROW + (p ? it.b : it.a) / 2;
#pragma unroll
        for (int e = 0; e < VEC / 2; ++e) row[e] = v2[p].x[2 * e] | ((uint32_t)v2[p].x[2 * e + 1] << 16);
      }
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      fine = fine && bf16_finite(ka[i].x[e]) && bf16_finite(kb[i].x[e]);
      kmax = fmaxf(kmax, fmaxf(fabsf(bf16_to_f32(ka[i].x[e])), fabsf(bf16_to_f32(kb[i].x[e]))));
    }
    if (!fine) poisoned[slot] = 1;
  }
  if (from_tail) {
    uint16_t* v16 = (uint16_t*)vt;
    for (uint32_t idx = tid; idx < D * (PAGE / 8); idx += THREADS) {
      const int d = (int)(idx / (PAGE / 8)), slot = (int)(idx % (PAGE / 8)) * 8;
      if (slot >= old) continue;
      const Half<8> x = load_half<8>(vt_in + d * PAGE + slot);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (slot + e < old) {
          v16[(slot + e) * 2 * ROW + d] = x.x[e];
          vmax = fmaxf(vmax, fabsf(bf16_to_f32(x.x[e])));
        }
    }
  }
  kmax = wave_max(kmax);
  vmax = wave_max(vmax);
  if ((tid & 63) == 0) tops[0][tid / 64] = kmax, tops[1][tid / 64] = vmax;
  __syncthreads();

  if (full) {
    const bool bad = __ballot(poisoned[tid % PAGE] != 0) != 0;      // every wave looks at all 64 tokens
    kmax = fminf(fmaxf(fmaxf(fmaxf(tops[0][0], tops[0][1]), fmaxf(tops[0][2], tops[0][3])), AMAX_LO), AMAX_HI);
    vmax = fminf(fmaxf(fmaxf(fmaxf(tops[1][0], tops[1][1]), fmaxf(tops[1][2], tops[1][3])), AMAX_LO), AMAX_HI);
    const float kinv = bad ? 0.0f : (1.0f / kmax) * qmax<KIND>(), vinv = (1.0f / vmax) * qmax<KIND>();
    if (tid == 0) {
      P.k_scale[(size_t)id * P.n_kv_heads + h] = bad ? __uint_as_float(0x7FC00000u) : kmax * (1.0f / qmax<KIND>());
      P.v_scale[(size_t)id * P.n_kv_heads + h] = vmax * (1.0f / qmax<KIND>());
    }
    uint8_t* kp = (uint8_t*)P.k + id * unit_elems + head;
#pragma unroll
    for (uint32_t i = 0; i < NI; ++i) {
      const uint32_t idx = tid + i * THREADS;
      if (idx >= PAGE * ITEMS) continue;
      const Item<VEC> it = item_at<VEC>(R, idx % ITEMS);
      uint8_t* row = kp + (idx / ITEMS) * D;
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const Half<VEC>& x = p ? kb[i] : ka[i];
        uint32_t w[VEC / 4];
#pragma unroll
        for (int e = 0; e < VEC / 4; ++e)
          w[e] = bad ? 0u
                     : quantise2<KIND>(bf16_to_f32(x.x[4 * e]), bf16_to_f32(x.x[4 * e + 1]), kinv) |
                           (quantise2<KIND>(bf16_to_f32(x.x[4 * e + 2]), bf16_to_f32(x.x[4 * e + 3]), kinv) << 16);
#pragma unroll
        for (int e = 0; e < VEC / 4; ++e) ((uint32_t*)(row + (p ? it.b : it.a)))[e] = w[e];
      }
    }
    // two channels of 16 tokens each
    uint8_t* vp = (uint8_t*)P.v + id * unit_elems + head;
    for (uint32_t idx = tid; idx < D / 2 * (PAGE / 16); idx += THREADS) {
      const uint32_t d2 = idx / (PAGE / 16), slot = idx % (PAGE / 16) * 16;
      uint32_t a[4], c[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        uint32_t x[4];
#pragma unroll
        for (int f = 0; f < 4; ++f) x[f] = vt[(slot + 4 * e + f) * ROW + d2];
        a[e] = quantise2<KIND>(bf16_to_f32(x[0] & 0xFFFFu), bf16_to_f32(x[1] & 0xFFFFu), vinv) |
               (quantise2<KIND>(bf16_to_f32(x[2] & 0xFFFFu), bf16_to_f32(x[3] & 0xFFFFu), vinv) << 16);
        c[e] = quantise2<KIND>(bf16_to_f32(x[0] >> 16), bf16_to_f32(x[1] >> 16), vinv) |
               (quantise2<KIND>(bf16_to_f32(x[2] >> 16), bf16_to_f32(x[3] >> 16), vinv) << 16);
      }
      *(uint4*)(vp + (2 * d2) * PAGE + slot) = make_uint4(a[0], a[1], a[2], a[3]);
      *(uint4*)(vp + (2 * d2 + 1) * PAGE + slot) = make_uint4(c[0], c[1], c[2], c[3]);
    }
  } else {
    uint16_t* kt = P.k_tail + tail_out * unit_elems + head;
    uint16_t* vo = P.v_tail + tail_out * unit_elems + head;
#pragma unroll
    for (uint32_t i = 0; i < NI; ++i) {
      const uint32_t idx = tid + i * THREADS;
      const int slot = (int)(idx / ITEMS);
      if (slot < lo || slot >= have) continue;
      const Item<VEC> it = item_at<VEC>(R, idx % ITEMS);
      if (poisoned[slot]) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) ka[i].x[e] = kb[i].x[e] = 0x7FC0u;
      }
      *(Half<VEC>*)(kt + slot * D + it.a) = ka[i];
      *(Half<VEC>*)(kt + slot * D + it.b) = kb[i];
    }
    const uint16_t* v16 = (const uint16_t*)vt;
    const uint32_t count = (uint32_t)(have - lo);
    for (uint32_t idx = tid; idx < D * count; idx += THREADS) {
      const uint32_t d = idx / count, slot = (uint32_t)lo + idx % count;
      vo[d * PAGE + slot] = v16[slot * 2 * ROW + d];
    }
  }
}

template <int D, int KIND>
__global__ __launch_bounds__(THREADS) void read_kernel(bs_kv_pool P, const int32_t* pages, uint32_t n_cols,
                                                       const int32_t* tail, uint32_t n, uint16_t* k_out, uint16_t* v_out,
                                                       int32_t* status) {
#pragma clang fp contract(off)
  constexpr uint32_t ROW = D / 2 + 1;
  __shared__ uint32_t vt[PAGE * ROW];     // V, bf16, rows of tokens
  const uint32_t tid = threadIdx.x, page = blockIdx.x, h = blockIdx.y;
  const uint32_t p0 = page * PAGE, have = min(n - p0, PAGE);
  const bool full = have == PAGE;
  const uint32_t id = (uint32_t)(full ? uniform_load(pages, page) : uniform_load(tail, 0));
  if (id >= (full ? P.n_pages : P.n_tails)) {
    if (tid == 0) report(status, BS_DEV_ERR_BOUNDS);
    return;
  }
  const size_t base = ((size_t)id * P.n_kv_heads + h) * PAGE * D;
  uint16_t* ko = k_out + ((size_t)h * n + p0) * D;
  uint16_t* vo = v_out + ((size_t)h * n + p0) * D;
  uint16_t* v16 = (uint16_t*)vt;
  if (full) {
    const float ks = uniform_load(P.k_scale, (size_t)id * P.n_kv_heads + h), vs = uniform_load(P.v_scale, (size_t)id * P.n_kv_heads + h);
    constexpr uint32_t LOADS = (PAGE * D / 16 + THREADS - 1) / THREADS;
    const uint4 *const kp = (const uint4*)((const uint8_t*)P.k + base), *const vp = (const uint4*)((const uint8_t*)P.v + base);
    uint4 kw[LOADS], vw[LOADS];
#pragma unroll
    for (uint32_t l = 0; l < LOADS; ++l) {
      const uint32_t i = tid + l * THREADS;
      if (PAGE * D % (16 * THREADS) == 0 || i < PAGE * D / 16) kw[l] = kp[i], vw[l] = vp[i];
    }
#pragma unroll
    for (uint32_t l = 0; l < LOADS; ++l) {
      const uint32_t i = tid + l * THREADS;
      if (PAGE * D % (16 * THREADS) != 0 && i >= PAGE * D / 16) continue;
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const half8v x = p ? codes8_to_f16<KIND>(kw[l].z, kw[l].w) : codes8_to_f16<KIND>(kw[l].x, kw[l].y);
        const half8v z = p ? codes8_to_f16<KIND>(vw[l].z, vw[l].w) : codes8_to_f16<KIND>(vw[l].x, vw[l].y);
        const uint32_t d = i / (PAGE / 16), slot = i % (PAGE / 16) * 16 + 8 * p;
        Half<8> y;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          y.x[e] = f32_to_bf16((float)x[e] * ks);
          v16[(slot + e) * 2 * ROW + d] = f32_to_bf16((float)z[e] * vs);
        }
        *(Half<8>*)(ko + 16 * i + 8 * p) = y;
      }
    }
  } else {
    for (uint32_t i = tid; i < have * D / 8; i += THREADS) *(Half<8>*)(ko + 8 * i) = load_half<8>(P.k_tail + base + 8 * i);
    for (uint32_t i = tid; i < D * PAGE; i += THREADS) {
      const uint32_t d = i / PAGE, slot = i % PAGE;
      if (slot < have) v16[slot * 2 * ROW + d] = P.v_tail[base + d * PAGE + slot];
    }
  }
  __syncthreads();
  for (uint32_t i = tid; i < have * D / 8; i += THREADS) {
    const uint32_t slot = i / (D / 8), c = i % (D / 8);
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = vt[slot * ROW + 4 * c + e];
    *(uint4*)(vo + 8 * i) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

bool pool_ok(const bs_kv_pool* p) {
  if (!p || !p->k || !p->v || !p->k_scale || !p->v_scale || !p->k_tail || !p->v_tail) return false;
  if ((((uintptr_t)p->k | (uintptr_t)p->v | (uintptr_t)p->k_tail | (uintptr_t)p->v_tail) & 15) != 0) return false;
  const uint32_t d = p->head_dim;
  return p->n_kv_heads >= 1 && p->n_kv_heads <= 65535 && p->kind <= BS_KV_FP8 &&
         (d == 64 || d == 80 || d == 96 || d == 128 || d == 256);
}

bool batch_ok(const bs_kv_batch* b) {
  return b && b->start && b->cu && b->table && b->tails && b->table_cols <= (1u << 24) && b->table_stride >= b->table_cols &&
         b->n_rows <= (1u << 30) && b->n_seqs <= (1u << 24) && (uint64_t)b->n_seqs * b->table_cols <= (1u << 30);
}

bool rows_ok(const void* p, int64_t token, int64_t head) {
  return p && ((uintptr_t)p & 15) == 0 && (token & 7) == 0 && (head & 7) == 0;
}

template <int D, int VEC, int KIND>
int append_launch(const bs_kv_pool* P, const bs_kv_batch* B, const bs_kv_rows* R, int32_t* status, hipStream_t stream) {
  // n new tokens touch at most (n + 62) / 64 + 1 pages, and no more than n: enough workgroups for any sequence lengths
  const uint64_t units = std::min<uint64_t>(B->n_rows, (B->n_rows + 62ull * B->n_seqs) / 64 + B->n_seqs);
  const uint64_t blocks = (units + DIES - 1) / DIES * DIES * P->n_kv_heads;
  if (blocks > 0x7FFFFFFF) return BS_ERR_ARG;
  append_kernel<D, VEC, KIND><<<(uint32_t)blocks, THREADS, 0, stream>>>(*P, *B, *R, status);
  return hipGetLastError() == hipSuccess ? BS_OK : BS_ERR_HIP;
}

template <int D, int KIND>
int read_launch(const bs_kv_pool* P, const int32_t* pages, uint32_t n_cols, const int32_t* tail, uint32_t n, uint16_t* k,
                uint16_t* v, int32_t* status, hipStream_t stream) {
  read_kernel<D, KIND><<<dim3((n + PAGE - 1) / PAGE, P->n_kv_heads), THREADS, 0, stream>>>(*P, pages, n_cols, tail, n, k, v, status);
  return hipGetLastError() == hipSuccess ? BS_OK : BS_ERR_HIP;
}

}  // namespace

namespace bs_kv {
bool check_pool(const bs_kv_pool* p) { return pool_ok(p); }
bool check_batch(const bs_kv_batch* b) { return batch_ok(b); }
}  // namespace bs_kv

extern "C" int bs_kv_append(const bs_kv_pool* P, const bs_kv_batch* B, const bs_kv_rows* R, int32_t* d_status, void* stream) {
  if (!pool_ok(P) || !batch_ok(B) || !R) return BS_ERR_ARG;
  if (R->rot % 8 || R->rot > P->head_dim) return BS_ERR_ARG;
  if (R->rot && (!R->cos || !R->sin || (((uintptr_t)R->cos | (uintptr_t)R->sin) & 15))) return BS_ERR_ARG;
  if (B->n_rows == 0 || B->n_seqs == 0) return BS_OK;
  if (!rows_ok(R->k, R->k_token, R->k_head) || !rows_ok(R->v, R->v_token, R->v_head)) return BS_ERR_ARG;
  if (R->q && (!rows_ok(R->q, R->q_token, R->q_head) || !rows_ok(R->q_out, 0, 0) || R->n_q_heads == 0 ||
               R->n_q_heads % P->n_kv_heads))
    return BS_ERR_ARG;
  hipStream_t s = (hipStream_t)stream;
  // Eight pairs an item (16-byte loads) where the turned channels divide by it, else four (2,048 tokens,
  // heads of 128: 17 us, by fours 21; 32,768 tokens: by fours 2 % more).
  const bool wide = R->rot % 16 == 0;
#define BS_KV_GO(D, K) return wide ? append_launch<D, 8, K>(P, B, R, d_status, s) : append_launch<D, 4, K>(P, B, R, d_status, s)
#define BS_KV_DIMS(K)              \
  switch (P->head_dim) {           \
    case 64: BS_KV_GO(64, K);      \
    case 80: BS_KV_GO(80, K);      \
    case 96: BS_KV_GO(96, K);      \
    case 128: BS_KV_GO(128, K);    \
    default: BS_KV_GO(256, K);     \
  }
  if (P->kind == BS_KV_FP8) BS_KV_DIMS(BS_KV_FP8)
  BS_KV_DIMS(BS_KV_INT8)
#undef BS_KV_GO
#undef BS_KV_DIMS
}

extern "C" int bs_kv_read(const bs_kv_pool* P, const int32_t* d_pages, uint32_t n_cols, const int32_t* d_tail, uint32_t n,
                          uint16_t* d_k, uint16_t* d_v, int32_t* d_status, void* stream) {
  if (!pool_ok(P)) return BS_ERR_ARG;
  if (n == 0) return BS_OK;
  if (n > (1u << 30) || n / PAGE > n_cols || (n >= PAGE && !d_pages) || (n % PAGE && !d_tail)) return BS_ERR_ARG;
  if (!rows_ok(d_k, 0, 0) || !rows_ok(d_v, 0, 0)) return BS_ERR_ARG;
  hipStream_t s = (hipStream_t)stream;
#define BS_KV_GO(D) \
  return P->kind == BS_KV_FP8 ? read_launch<D, BS_KV_FP8>(P, d_pages, n_cols, d_tail, n, d_k, d_v, d_status, s) \
                              : read_launch<D, BS_KV_INT8>(P, d_pages, n_cols, d_tail, n, d_k, d_v, d_status, s)
  switch (P->head_dim) {
    case 64: BS_KV_GO(64);
    case 80: BS_KV_GO(80);
    case 96: BS_KV_GO(96);
    case 128: BS_KV_GO(128);
    default: BS_KV_GO(256);
  }
#undef BS_KV_GO
}
