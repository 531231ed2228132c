// The paged KV cache's books on the GPU.
//
// step_kernel: a step's tables from the lengths alone. Every workgroup counts all sequences for itself (rows and pages
// of those before its own, and of all, since a step is made whole or not at all) and then writes what belongs to its
// own sequences: nothing passes between workgroups, so it is one launch, and the books stay as they were, so it can be
// made again. The bound of the usual step is the launch and three dependent reads (place, length, page): 128 sequences of
// up to 16,383 tokens, 5 new ones each, 5 us for 131 KB of tables; 32 prompts of up to 8,192 tokens 6 us for 2 MB of rows.
// (The counts one after another over the workgroup, and a sequence looked up again for its tables: 6 and 7.)
//
// keep_kernel enters a step into the books: 3 us, a launch and two dependent reads. drop is one workgroup for a few places, else two
// launches: pages go onto the stack while lengths still stand, then the places are emptied.
#include <algorithm>

#include "kv_common.h"

namespace {

using namespace bs_kv;

constexpr uint32_t THREADS = 256, WAVES = THREADS / 64, MOST_PLACES = 65536;
// Workgroups count all sequences each, so beyond 512 of them they take several sequences.
constexpr uint32_t MOST_GROUPS = 512;

// Sums of N numbers over the workgroup, side by side, and the bits of `bits` that any thread has.
template <int N>
struct Totals {
  int64_t sum[WAVES][N];
  int bits[WAVES];
};
template <int N>
__device__ int totals(int64_t (&x)[N], int bits, Totals<N>& lds) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] += __shfl_xor(x[i], d);
  const int any = (__ballot(bits & BS_DEV_ERR_BOUNDS) ? BS_DEV_ERR_BOUNDS : 0) | (__ballot(bits & BS_DEV_ERR_COUNT) ? BS_DEV_ERR_COUNT : 0);
  const uint32_t wave = threadIdx.x / 64;
  if (threadIdx.x % 64 == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) lds.sum[wave][i] = x[i];
    lds.bits[wave] = any;
  }
  __syncthreads();
  int all = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = 0;
#pragma unroll
  for (uint32_t w = 0; w < WAVES; ++w) {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] += lds.sum[w][i];
    all |= lds.bits[w];
  }
  return all;
}

// What a step wants of one sequence.
struct Want {
  int32_t place, start, n, pages;  // pages: taken anew
  int bad;                         // BS_DEV_ERR_* bits
};

__device__ Want want(const bs_kv_books& K, const bs_kv_tables& S, const int32_t* d_new, const int32_t* d_sure, uint32_t b) {
  Want w = {S.seqs[b], 0, 0, 0, 0};
  if ((uint32_t)w.place >= K.n_places) {
    w.bad = BS_DEV_ERR_BOUNDS;
    return w;
  }
  const int64_t room = (int64_t)K.cols * PAGE, fresh = d_new[b], start = K.length[w.place];
  int64_t sure = d_sure ? (int64_t)d_sure[b] : fresh;
  if (fresh < 0 || sure < 0 || start < 0 || start > room) {
    w.bad = BS_DEV_ERR_BOUNDS;
    return w;
  }
  w.start = (int32_t)start;
  sure = sure < fresh ? sure : fresh;
  if (start + sure > room) {
    w.bad = BS_DEV_ERR_COUNT;
    return w;
  }
  int64_t end = start + fresh;
  if (d_sure) {  // the last token that completes a page is a certain one
    const int64_t most = ((start + sure) / PAGE + 1) * PAGE - 1;
    end = end < most ? end : most;
    end = end < room ? end : room;
  }
  w.n = (int32_t)(end - start);
  w.pages = (int32_t)(end / PAGE - start / PAGE);
  return w;
}

__global__ __launch_bounds__(THREADS) void step_kernel(bs_kv_books K, bs_kv_tables S, const int32_t* d_new, const int32_t* d_sure,
                                                       uint32_t each, int32_t* status) {
  __shared__ uint32_t seen[MOST_PLACES / 32];
  __shared__ Totals<4> lds;
  __shared__ Want own[MOST_PLACES / MOST_GROUPS];
  const uint32_t tid = threadIdx.x, first = blockIdx.x * each, last = min(S.n_seqs, first + each);
  for (uint32_t i = tid; i < (K.n_places + 31) / 32; i += THREADS) seen[i] = 0;
  __syncthreads();
  int64_t sums[4] = {0, 0, 0, 0};  // rows and pages, and those of the sequences before this workgroup's
  const int32_t n_free = *K.n_free;
  int bad = 0;
  for (uint32_t b = tid; b < S.n_seqs; b += THREADS) {
    const Want w = want(K, S, d_new, d_sure, b);
    bad |= w.bad;
    sums[0] += w.n, sums[1] += w.pages;
    if (b < first) sums[2] += w.n, sums[3] += w.pages;
    if (b >= first && b < last) own[b - first] = w;
    if (!(w.bad & BS_DEV_ERR_BOUNDS)) {
      const uint32_t bit = 1u << (w.place % 32);
      if (atomicOr(&seen[w.place / 32], bit) & bit) bad |= BS_DEV_ERR_BOUNDS;
    }
  }
  bad = totals(sums, bad, lds);
  int64_t rows = sums[0], pages = sums[1], rows_before = sums[2], pages_before = sums[3];
  if (n_free < 0 || n_free > (int32_t)K.n_pages) bad |= BS_DEV_ERR_BOUNDS;
  if (rows > (int64_t)S.n_rows || pages > (int64_t)n_free) bad |= BS_DEV_ERR_COUNT;
  if (bad && blockIdx.x == 0 && blockIdx.y == 0 && tid == 0) report(status, bad);
  if (bad) rows = rows_before = 0;

  // rows are dealt to the workgroups of a sequence in strips, and so are the columns of its table
  const uint32_t strip = blockIdx.y * THREADS + tid, strips = gridDim.y * THREADS;
  int32_t at = (int32_t)rows_before, from = n_free - 1 - (int32_t)pages_before;
  for (uint32_t b = first; b < last; ++b) {
    const Want w = own[b - first];
    const int32_t n = bad ? 0 : w.n, taken = bad ? 0 : w.pages, held = w.start / (int32_t)PAGE;
    const bool place = (uint32_t)w.place < K.n_places;
    if (strip == 0) {
      const int32_t which = place ? K.which[w.place] & 1 : 0, tail = place ? K.tails[w.place] : 0;
      S.start[b] = w.start;
      S.cu[b] = at;
      S.tails[2 * (size_t)b] = tail + which;
      S.tails[2 * (size_t)b + 1] = tail + (taken ? which ^ 1 : which);
    }
    const int32_t* held_pages = K.table + (size_t)(place ? w.place : 0) * K.cols;
    int32_t* row = S.table + (size_t)b * K.cols;
    for (int32_t c = (int32_t)strip; c < (int32_t)K.cols; c += (int32_t)strips)
      row[c] = c < held ? held_pages[c] : c < held + taken ? K.free[from - (c - held)] : 0;
    for (int32_t i = (int32_t)strip; i < n; i += (int32_t)strips) {
      S.owner[at + i] = (int32_t)b;
      S.position[at + i] = w.start + i;
      S.slot[at + i] = ((int64_t)w.place * K.cols) * PAGE + w.start + i;
    }
    at += n, from -= taken;
  }
  const uint32_t all = gridDim.x * strips;
  for (uint32_t r = (uint32_t)rows + blockIdx.x * strips + strip; r < S.n_rows; r += all) S.owner[r] = -1, S.position[r] = -1, S.slot[r] = -1;
  if (blockIdx.x == 0 && strip == 0) S.cu[S.n_seqs] = (int32_t)rows;
}

__global__ __launch_bounds__(THREADS) void keep_kernel(bs_kv_books K, bs_kv_tables S, const int32_t* d_sure, const int32_t* d_kept) {
  __shared__ Totals<1> lds;
  const uint32_t tid = threadIdx.x;
  if (blockIdx.x == S.n_seqs) {  // one more workgroup for the stack
    int64_t pages[1] = {0};
    for (uint32_t b = tid; b < S.n_seqs; b += THREADS) {
      const int32_t start = S.start[b], end = start + S.cu[b + 1] - S.cu[b];
      pages[0] += end / (int32_t)PAGE - start / (int32_t)PAGE;
    }
    totals(pages, 0, lds);
    if (tid == 0) *K.n_free -= (int32_t)pages[0];
    return;
  }
  const uint32_t b = blockIdx.x;
  const int32_t n = S.cu[b + 1] - S.cu[b];
  if (n <= 0) return;
  const int32_t place = S.seqs[b], start = S.start[b], held = start / (int32_t)PAGE, have = (start + n) / (int32_t)PAGE;
  if ((uint32_t)place >= K.n_places || start < 0 || have > (int32_t)K.cols) return;  // (not what the step was made of)
  for (int32_t c = held + (int32_t)tid; c < have; c += THREADS) K.table[(size_t)place * K.cols + c] = S.table[(size_t)b * K.cols + c];
  if (tid == 0) {
    int32_t kept = d_kept ? d_kept[b] : n;
    kept = max(kept, d_sure ? d_sure[b] : n);
    K.length[place] = start + min(kept, n);
    if (have > held) K.which[place] ^= 1;
  }
}

// Pages of the places before `first`, and of all; 0 and an error's bit if the places are not to be dropped together.
__device__ int count_pages(const bs_kv_books& K, const int32_t* seqs, uint32_t n_seqs, uint32_t first, int64_t& before, int64_t& total,
                           uint32_t* seen, Totals<2>& lds) {
  const uint32_t tid = threadIdx.x;
  for (uint32_t i = tid; i < (K.n_places + 31) / 32; i += THREADS) seen[i] = 0;
  __syncthreads();
  int bad = 0;
  int64_t sums[2] = {0, 0};
  const int32_t n_free = *K.n_free;
  for (uint32_t b = tid; b < n_seqs; b += THREADS) {
    const uint32_t place = (uint32_t)seqs[b];
    if (place >= K.n_places) {
      bad = BS_DEV_ERR_BOUNDS;
      continue;
    }
    const uint32_t bit = 1u << (place % 32);
    const int32_t length = K.length[place];
    if ((atomicOr(&seen[place / 32], bit) & bit) || length < 0 || length > (int32_t)(K.cols * PAGE)) {
      bad = BS_DEV_ERR_BOUNDS;
      continue;
    }
    sums[0] += length / (int32_t)PAGE;
    if (b < first) sums[1] += length / (int32_t)PAGE;
  }
  bad = totals(sums, bad, lds);
  total = sums[0], before = sums[1];
  return n_free < 0 || total + n_free > (int64_t)K.n_pages ? BS_DEV_ERR_BOUNDS : bad;
}

__global__ __launch_bounds__(THREADS) void push_kernel(bs_kv_books K, const int32_t* seqs, uint32_t n_seqs, uint32_t each, int32_t* status) {
  __shared__ uint32_t seen[MOST_PLACES / 32];
  __shared__ Totals<2> lds;
  const uint32_t first = blockIdx.x * each, last = min(n_seqs, first + each);
  int64_t before, total;
  if (const int bad = count_pages(K, seqs, n_seqs, first, before, total, seen, lds)) {
    if (blockIdx.x == 0 && threadIdx.x == 0) report(status, bad);
    return;
  }
  int32_t to = *K.n_free + (int32_t)total - 1 - (int32_t)before;
  for (uint32_t b = first; b < last; ++b) {
    const int32_t place = seqs[b], pages = K.length[place] / (int32_t)PAGE;
    for (int32_t c = (int32_t)threadIdx.x; c < pages; c += THREADS) K.free[to - c] = K.table[(size_t)place * K.cols + c];
    to -= pages;
  }
}

__global__ __launch_bounds__(THREADS) void empty_kernel(bs_kv_books K, const int32_t* seqs, uint32_t n_seqs) {
  __shared__ uint32_t seen[MOST_PLACES / 32];
  __shared__ Totals<2> lds;
  int64_t before, total;
  if (count_pages(K, seqs, n_seqs, 0, before, total, seen, lds)) return;
  for (uint32_t b = threadIdx.x; b < n_seqs; b += THREADS) K.length[seqs[b]] = 0, K.which[seqs[b]] = 0;
  if (threadIdx.x == 0) *K.n_free += (int32_t)total;
}

// Both in one launch, by one workgroup: a wave a place.
constexpr uint32_t D_THREADS = 1024, D_PAGES = 16384;
__global__ __launch_bounds__(D_THREADS) void drop_kernel(bs_kv_books K, const int32_t* seqs, uint32_t n_seqs, int32_t* status) {
  __shared__ uint32_t seen[MOST_PLACES / 32];
  __shared__ int32_t upto[D_THREADS / 64];
  __shared__ int32_t pages[D_THREADS], to[D_THREADS];
  __shared__ int any_bad;
  const uint32_t tid = threadIdx.x, lane = tid % 64, wave = tid / 64;
  for (uint32_t i = tid; i < (K.n_places + 31) / 32; i += D_THREADS) seen[i] = 0;
  if (tid == 0) any_bad = 0;
  __syncthreads();
  const int32_t n_free = *K.n_free;
  const uint32_t place = tid < n_seqs ? (uint32_t)seqs[tid] : 0;
  int32_t own = 0;
  if (tid < n_seqs) {
    bool bad = place >= K.n_places;
    if (!bad) {
      const uint32_t bit = 1u << (place % 32);
      const int32_t length = K.length[place];
      bad = (atomicOr(&seen[place / 32], bit) & bit) || length < 0 || length > (int32_t)(K.cols * PAGE);
      own = bad ? 0 : length / (int32_t)PAGE;
    }
    if (bad) any_bad = 1;
  }
  int32_t before = own;  // pages up to and with this thread's
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int32_t up = __shfl_up(before, d);
    if (lane >= (uint32_t)d) before += up;
  }
  if (lane == 63) upto[wave] = before;
  __syncthreads();
  int32_t total = 0;
  for (uint32_t w = 0; w < D_THREADS / 64; ++w) {
    if (w < wave) before += upto[w];
    total += upto[w];
  }
  if (any_bad || n_free < 0 || (int64_t)total + n_free > (int64_t)K.n_pages) {
    if (tid == 0) report(status, BS_DEV_ERR_BOUNDS);
    return;
  }
  pages[tid] = own;
  to[tid] = n_free + total - 1 - (before - own);
  __syncthreads();
  for (uint32_t b = wave; b < n_seqs; b += D_THREADS / 64) {
    const int32_t* from = K.table + (size_t)(uint32_t)seqs[b] * K.cols;
    for (int32_t c = (int32_t)lane; c < pages[b]; c += 64) K.free[to[b] - c] = from[c];
  }
  if (tid < n_seqs) K.length[place] = 0, K.which[place] = 0;
  if (tid == 0) *K.n_free = n_free + total;
}

bool books_ok(const bs_kv_books* k) {
  return k && k->length && k->which && k->table && k->free && k->n_free && k->tails && k->n_places > 0 && k->n_places <= MOST_PLACES &&
         k->cols > 0 && k->cols < (1u << 24) && k->n_pages > 0 && k->n_pages < (1u << 30);
}

bool step_ok(const bs_kv_books* k, const bs_kv_tables* s) {
  return s && s->n_seqs <= k->n_places && s->n_rows < (1u << 30) &&
         (s->n_seqs == 0 || (s->seqs && s->start && s->cu && s->tails && s->table)) &&
         (s->n_rows == 0 || (s->owner && s->position && s->slot && ((uintptr_t)s->slot & 7) == 0));
}

int done() { return hipGetLastError() == hipSuccess ? BS_OK : BS_ERR_HIP; }

}  // namespace

extern "C" int bs_kv_books_step(const bs_kv_books* K, const bs_kv_tables* S, const int32_t* d_new, const int32_t* d_sure,
                                int32_t* d_status, void* stream) {
  if (!books_ok(K) || !step_ok(K, S) || (S->n_seqs && !d_new)) return BS_ERR_ARG;
  if (S->n_seqs == 0) return BS_OK;
  const uint32_t each = (S->n_seqs + MOST_GROUPS - 1) / MOST_GROUPS, groups = (S->n_seqs + each - 1) / each;
  const uint32_t strips = std::min({16u, std::max(1u, S->max_new / 2048), std::max(1u, 1024 / groups)});
  step_kernel<<<dim3(groups, strips), THREADS, 0, (hipStream_t)stream>>>(*K, *S, d_new, d_sure, each, d_status);
  return done();
}

extern "C" int bs_kv_books_keep(const bs_kv_books* K, const bs_kv_tables* S, const int32_t* d_sure, const int32_t* d_kept, void* stream) {
  if (!books_ok(K) || !step_ok(K, S)) return BS_ERR_ARG;
  if (S->n_seqs == 0) return BS_OK;
  keep_kernel<<<S->n_seqs + 1, THREADS, 0, (hipStream_t)stream>>>(*K, *S, d_sure, d_kept);
  return done();
}

extern "C" int bs_kv_books_drop(const bs_kv_books* K, const int32_t* d_seqs, uint32_t n_seqs, int32_t* d_status, void* stream) {
  if (!books_ok(K) || n_seqs > K->n_places || (n_seqs && !d_seqs)) return BS_ERR_ARG;
  if (n_seqs == 0) return BS_OK;
  if (n_seqs <= D_THREADS && (uint64_t)n_seqs * K->cols <= D_PAGES) {  // 32 places of 256 pages at most: 4 us, in two launches 8
    drop_kernel<<<1, D_THREADS, 0, (hipStream_t)stream>>>(*K, d_seqs, n_seqs, d_status);
    return done();
  }
  const uint32_t each = (n_seqs + MOST_GROUPS - 1) / MOST_GROUPS;
  push_kernel<<<(n_seqs + each - 1) / each, THREADS, 0, (hipStream_t)stream>>>(*K, d_seqs, n_seqs, each, d_status);
  empty_kernel<<<1, THREADS, 0, (hipStream_t)stream>>>(*K, d_seqs, n_seqs);
  return done();
}
