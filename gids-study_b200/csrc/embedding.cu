// Embedding lookup with scaling and its gradient by sorted ids, for sm_100a.
//
// Lookup: out[i, :] = round(scale * weight[id_i, :]). One thread moves
// EMB_UNROLL vectors of a flat (row, vector) index space, so rows of any width
// fill the warps; an id outside the table gives a zero row and sets the device's
// error word. Rows that are not aligned to vectors come through shared memory
// instead. Bound by HBM: 1,000,003 rows of 768 fp16 take 519 us, 0.92 of the
// measured copy rate for the 3.07 GB they read and write (545 us when the output
// stays in L2 and pushes out rows of the table).
//
// Gradient: dweight[v, :] = round(scale * sum over {i : id_i = v} of grad[i, :]).
// The ids are sorted (LSD radix sort of (id, position) words, stable, so equal
// ids stay in position order) and the sorted list is cut into chunks whose runs
// of equal ids are summed by a team of lanes each; sums of runs that cross
// chunks are joined in a fixed order. Nothing is accumulated with atomics, so
// results repeat bit for bit. Padding and bad ids sort behind every row and are
// left out: their gradients are not read.
#include <algorithm>
#include <atomic>
#include <map>
#include <mutex>
#include <type_traits>
#include <vector>

#include "layers.hpp"
#include "rows.cuh"

namespace gids {
namespace {

// ---------------------------------------------------------------- the lookup
constexpr int EMB_THREADS = 256;
constexpr int EMB_UNROLL = 4;

struct EmbArgs {
  void* out;
  const void* weight;
  const void* ids;
  long long out_stride, weight_stride;
  unsigned long long num_rows, total;  // total = n * vectors per row
  unsigned long long vpr;              // vectors per row
  FastDiv vdiv;
  float scale;
  int* err;
};

template <typename ID>
__device__ __forceinline__ unsigned long long load_id(const void* ids, unsigned long long i) {
  // a negative id becomes a large unsigned one: outside every table
  return (unsigned long long)(long long)__ldg(reinterpret_cast<const ID*>(ids) + i);
}

template <typename W, typename O, int VEC, typename ID>
__global__ void __launch_bounds__(EMB_THREADS) embedding_kernel(EmbArgs a) {
  const unsigned long long base = (unsigned long long)blockIdx.x * (EMB_THREADS * EMB_UNROLL);
  const unsigned long long row0 = base / a.vpr;
  const unsigned int col0 = (unsigned int)(base - row0 * a.vpr);
  RowVec<W, VEC> v[EMB_UNROLL];
  unsigned long long row[EMB_UNROLL];
  unsigned int col[EMB_UNROLL];
  bool on[EMB_UNROLL], good[EMB_UNROLL];
#pragma unroll
  for (int u = 0; u < EMB_UNROLL; u++) {
    const unsigned int t = threadIdx.x + u * EMB_THREADS;
    on[u] = base + t < a.total;
    const unsigned int q = a.vdiv.div(col0 + t);
    row[u] = row0 + q;
    col[u] = col0 + t - q * a.vdiv.d;
    good[u] = false;
    if (on[u]) {
      const unsigned long long id = load_id<ID>(a.ids, row[u]);
      good[u] = id < a.num_rows;
      if (good[u])
        v[u] = load_vec<W, VEC>(reinterpret_cast<const W*>(a.weight) + (long long)id * a.weight_stride +
                                (long long)col[u] * VEC);
    }
  }
#pragma unroll
  for (int u = 0; u < EMB_UNROLL; u++) {
    if (!on[u]) continue;
    O* o = reinterpret_cast<O*>(a.out) + (long long)row[u] * a.out_stride + (long long)col[u] * VEC;
    if constexpr (std::is_same<W, O>::value) {
      if (a.scale == 1.0f && good[u]) {  // a copy, NaN bits included
        store_stream(o, v[u]);
        continue;
      }
    }
    RowVec<O, VEC> r;
#pragma unroll
    for (int j = 0; j < VEC; j++) r.v[j] = from_f32<O>(good[u] ? a.scale * to_f32(v[u].v[j]) : 0.0f);
    if (!good[u]) *reinterpret_cast<volatile int*>(a.err) = 1;
    store_stream(o, r);
  }
}

// Rows that do not start on vectors: a warp fetches slabs of SLAB columns by the
// aligned 16-byte pieces that cover them, ODD_STAGES - 1 slabs ahead, and
// passes the elements on from shared memory. (200,000 rows of 1,001 bf16: 424 us
// by single elements.)
constexpr int ODD_SLAB = 512;
constexpr int ODD_STAGES = 4;
constexpr int ODD_THREADS = 256;

template <typename W, typename O, typename ID>
__global__ void __launch_bounds__(ODD_THREADS) embedding_odd_kernel(EmbArgs a, unsigned long long n, long long dim,
                                                                    unsigned int slabs) {
  constexpr int PITCH = ODD_SLAB * (int)sizeof(W) + 16;  // 16 bytes more, for a start inside a piece
  extern __shared__ uint4 dyn[];
  const unsigned int lane = threadIdx.x & 31;
  char* ring = reinterpret_cast<char*>(dyn) + (threadIdx.x >> 5) * (PITCH * ODD_STAGES);
  const unsigned long long total = n * slabs;
  const unsigned long long step = (unsigned long long)gridDim.x * (ODD_THREADS / 32);
  const unsigned long long first = (unsigned long long)blockIdx.x * (ODD_THREADS / 32) + (threadIdx.x >> 5);
  const auto source = [&](unsigned long long unit, int& len) -> const char* {  // null: a bad id
    const unsigned long long row = unit / slabs;
    const long long c0 = (long long)(unit - row * slabs) * ODD_SLAB;
    len = (int)min((long long)ODD_SLAB, dim - c0);
    const unsigned long long id = load_id<ID>(a.ids, row);
    if (id >= a.num_rows) return nullptr;
    return reinterpret_cast<const char*>(reinterpret_cast<const W*>(a.weight) + (long long)id * a.weight_stride + c0);
  };
  const auto fetch = [&](unsigned long long unit, int stage) {
    if (unit < total) {
      int len;
      const char* src = source(unit, len);
      if (src) {
        const int early = (int)(reinterpret_cast<uintptr_t>(src) & 15), span = early + len * (int)sizeof(W);
        for (int q = (int)lane * 16; q < span; q += 512)
          copy_async_tail(ring + stage * PITCH + q, src - early + q, min(16, span - q));
      }
    }
    copies_commit();
  };
  for (int i = 0; i < ODD_STAGES - 1; i++) fetch(first + i * step, i);
  int stage = 0;
  for (unsigned long long unit = first; unit < total; unit += step) {
    __syncwarp();  // the slot that fetch() refills has been read
    fetch(unit + (ODD_STAGES - 1) * step, stage == 0 ? ODD_STAGES - 1 : stage - 1);
    copies_wait<ODD_STAGES - 1>();
    __syncwarp();
    int len;
    const char* src = source(unit, len);
    const unsigned long long row = unit / slabs;
    O* out = reinterpret_cast<O*>(a.out) + (long long)row * a.out_stride + (long long)(unit - row * slabs) * ODD_SLAB;
    const W* in = reinterpret_cast<const W*>(ring + stage * PITCH + (reinterpret_cast<uintptr_t>(src) & 15));
    if (!src && lane == 0) *reinterpret_cast<volatile int*>(a.err) = 1;
    const auto value = [&](int e) -> O {
      if constexpr (std::is_same<W, O>::value) {
        if (a.scale == 1.0f && src) return in[e];  // a copy, NaN bits included
      }
      return from_f32<O>(src ? a.scale * to_f32(in[e]) : 0.0f);
    };
    if constexpr (sizeof(O) == 4) {
#pragma unroll 4
      for (int e = (int)lane; e < len; e += 32) out[e] = value(e);
    } else {  // pairs, from the first element on a 4-byte boundary
      const int head = (reinterpret_cast<uintptr_t>(out) & 2) ? 1 : 0;
      if (head && lane == 0) out[0] = value(0);
#pragma unroll 4
      for (int e = head + 2 * (int)lane; e + 1 < len; e += 64) {
        RowVec<O, 2> two;
        two.v[0] = value(e);
        two.v[1] = value(e + 1);
        store_raw(out + e, two);
      }
      if (((len - head) & 1) && lane == 31) out[len - 1] = value(len - 1);
    }
    stage = stage + 1 == ODD_STAGES ? 0 : stage + 1;
  }
  copies_wait<0>();
}

// ------------------------------------------------------------------ the sort
// A chain of small kernels. Each is launched while the one before it drains
// (programmatic launch) and waits for its results here.
__device__ __forceinline__ void chain_wait() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

constexpr int SORT_ITEMS = 4;
constexpr int MAX_DIGIT_BITS = 9;
constexpr int MAX_RADIX = 1 << MAX_DIGIT_BITS;
constexpr int MAX_TILES = 148;

// The word that is sorted: key in the high half, position in the low half.
// Keys are the ids; padding and bad ids get the key `num_rows`.
struct IdSource {
  const void* ids;
  int id_bytes;  // 0: `words` holds sorted words of the pass before
  const unsigned long long* words;
  unsigned long long num_rows;
  long long padding;
  int* err;
};

__device__ __forceinline__ unsigned long long source_word(const IdSource& s, unsigned int i) {
  if (s.id_bytes == 0) return s.words[i];
  const long long id = s.id_bytes == 4 ? (long long)__ldg(reinterpret_cast<const int*>(s.ids) + i)
                                       : __ldg(reinterpret_cast<const long long*>(s.ids) + i);
  unsigned long long key = (unsigned long long)id;
  if (key >= s.num_rows) {
    *reinterpret_cast<volatile int*>(s.err) = 1;
    key = s.num_rows;
  } else if (id == s.padding) {
    key = s.num_rows;
  }
  return (key << 32) | i;
}

// Zeros for the rows of a dense gradient, written while the sort leaves the
// memory idle: every kernel of the sort takes a share, as bulk copies of a zero
// block of shared memory that run beside its own work. `bytes` and the
// address are multiples of 16; `tail` bytes more (a multiple of 2) follow.
constexpr int ZERO_BYTES = 8192;
struct ZeroFill {
  char* p;
  unsigned long long bytes;
  unsigned int tail;
};
__device__ __forceinline__ void zero_tail(const ZeroFill& z) {
  if (blockIdx.x == 0 && threadIdx.x < z.tail / 2) reinterpret_cast<unsigned short*>(z.p + z.bytes)[threadIdx.x] = 0;
}
__device__ __forceinline__ void zero_begin(const ZeroFill& z, uint4* zeros) {
  zero_tail(z);
  if (!z.bytes) return;
  for (int i = threadIdx.x; i < ZERO_BYTES / 16; i += blockDim.x) zeros[i] = make_uint4(0, 0, 0, 0);
  // the copies read shared memory through the asynchronous proxy
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncthreads();
  if (threadIdx.x != 0) return;
  const unsigned int src = (unsigned int)__cvta_generic_to_shared(zeros);
  for (unsigned long long at = (unsigned long long)blockIdx.x * ZERO_BYTES; at < z.bytes;
       at += (unsigned long long)gridDim.x * ZERO_BYTES) {
    const unsigned int b = (unsigned int)min((unsigned long long)ZERO_BYTES, z.bytes - at);
    asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(z.p + at), "r"(src), "r"(b)
                 : "memory");
  }
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
__device__ __forceinline__ void zero_end(const ZeroFill& z) {
  if (z.bytes && threadIdx.x == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
}

// A pass sorts by one digit of the keys: the bits [shift, shift + bits) of the
// words. Tile t covers the words [t * per, (t + 1) * per).
struct Pass {
  unsigned int n, per, tiles;
  int shift, bits;
  unsigned int* counts;  // [tile][digit, at least 4] words
};

template <int THREADS>
__global__ void __launch_bounds__(THREADS) count_kernel(IdSource src, Pass p, ZeroFill zero) {
  __shared__ unsigned int hist[MAX_RADIX];
  __shared__ alignas(128) uint4 zeros[ZERO_BYTES / 16];
  chain_wait();
  zero_begin(zero, zeros);
  if (blockIdx.x < p.tiles) {
    const int radix = 1 << p.bits;
    const int row = max(radix, 4);
    for (int d = threadIdx.x; d < row; d += THREADS) hist[d] = 0;
    __syncthreads();
    const unsigned int lo = blockIdx.x * p.per, hi = min(p.n, lo + p.per);
    for (unsigned int i0 = lo + threadIdx.x; i0 < hi; i0 += (THREADS * SORT_ITEMS)) {
      unsigned int digit[SORT_ITEMS];
#pragma unroll
      for (int k = 0; k < SORT_ITEMS; k++) {
        const unsigned int i = i0 + k * THREADS;
        digit[k] = i < hi ? (unsigned int)(source_word(src, i) >> p.shift) & (radix - 1) : (unsigned int)radix;
      }
#pragma unroll
      for (int k = 0; k < SORT_ITEMS; k++)
        if (digit[k] < (unsigned int)radix) atomicAdd(&hist[digit[k]], 1u);  // integers: the order does not matter
    }
    __syncthreads();
    for (int d = threadIdx.x; d < row; d += THREADS) p.counts[blockIdx.x * row + d] = hist[d];
  }
  zero_end(zero);
}

template <int THREADS>
struct SortShared {
  unsigned int base[MAX_RADIX];                    // next output index of each digit
  unsigned int before[MAX_RADIX];                  // words of the digit in earlier tiles
  unsigned short wcount[THREADS / 32][MAX_RADIX];  // digits of this step, by warp
  unsigned short part[4][MAX_RADIX];
  unsigned int wsum[THREADS / 32];
};

// base[d] = (words of smaller digits) + s.before[d], where thread d < radix
// knows the number `total` of words of digit d
template <int THREADS>
__device__ __forceinline__ void digit_bases(SortShared<THREADS>& s, int radix, unsigned int total) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  unsigned int incl = total;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned int v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) s.wsum[warp] = incl;
  __syncthreads();
  unsigned int off = 0;
  for (int w = 0; w < warp && w < MAX_RADIX / 32; w++) off += s.wsum[w];
  if (tid < radix) s.base[tid] = off + incl - total + s.before[tid];
}

// Ranks `items` words a thread among the words of the same digit in this
// step, in the order (warp, item, lane); returns the step's count of digit d to
// thread d and leaves the warps' offsets in s.wcount.
template <int THREADS>
__device__ __forceinline__ unsigned int rank_step(SortShared<THREADS>& s, int radix, int items,
                                                  const unsigned int (&digit)[SORT_ITEMS],
                                                  unsigned int (&rank)[SORT_ITEMS]) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  for (int i = lane; i < (radix + 1) / 2; i += 32) reinterpret_cast<unsigned int*>(s.wcount[warp])[i] = 0;
  __syncwarp();
  // lanes with the same digit: one ballot a bit
  unsigned int peers[SORT_ITEMS];
#pragma unroll
  for (int k = 0; k < SORT_ITEMS; k++) peers[k] = __ballot_sync(0xffffffffu, digit[k] != 0xffffffffu);
  for (int b = 0; (1 << b) < radix; b++) {
#pragma unroll
    for (int k = 0; k < SORT_ITEMS; k++) {
      if (k >= items) break;
      const bool one = (digit[k] >> b) & 1u;
      const unsigned int vote = __ballot_sync(0xffffffffu, one);
      peers[k] &= one ? vote : ~vote;
    }
  }
#pragma unroll
  for (int k = 0; k < SORT_ITEMS; k++) {
    if (k >= items) break;
    const bool in = digit[k] != 0xffffffffu;
    const unsigned int prior = in ? s.wcount[warp][digit[k]] : 0u;
    __syncwarp();
    rank[k] = prior + __popc(peers[k] & ((1u << lane) - 1u));
    if (in && (peers[k] >> lane) == 1u) s.wcount[warp][digit[k]] = (unsigned short)(prior + __popc(peers[k]));
    __syncwarp();
  }
  __syncthreads();
  // the warps' counts become offsets: up to 4 threads to a digit, each with a
  // share of the warps
  const int parts = min(4, THREADS / radix), share = (THREADS / 32) / parts;
  const int d = tid & (radix - 1), q = tid / radix;
  constexpr int MOST = (THREADS / 32) * MAX_RADIX / THREADS;
  unsigned short c[MOST];
  unsigned int sum = 0;
  if (q < parts) {
#pragma unroll
    for (int w = 0; w < MOST; w++)
      if (w < share) {
        c[w] = s.wcount[q * share + w][d];
        sum += c[w];
      }
    s.part[q][d] = (unsigned short)sum;
  }
  __syncthreads();
  unsigned int total = 0;
  if (q < parts) {
    unsigned int run = 0;
    for (int k = 0; k < parts; k++) {
      const unsigned int v = s.part[k][d];
      run += k < q ? v : 0u;
      total += v;
    }
#pragma unroll
    for (int w = 0; w < MOST; w++)
      if (w < share) {
        s.wcount[q * share + w][d] = (unsigned short)run;
        run += c[w];
      }
  }
  __syncthreads();
  return total;
}

// Stable scatter of tile blockIdx.x by one digit, ITEMS words a thread at a time.
template <int THREADS, int ITEMS>
__global__ void __launch_bounds__(THREADS) scatter_kernel(IdSource src, Pass p,
                                                               unsigned long long* __restrict__ out, ZeroFill zero) {
  extern __shared__ uint4 dyn[];
  SortShared<THREADS>& s = *reinterpret_cast<SortShared<THREADS>*>(dyn);
  // shares of all words of 4 digits, and of those in earlier tiles
  uint4(*sum)[THREADS] = reinterpret_cast<uint4(*)[THREADS]>(dyn + (sizeof(SortShared<THREADS>) + 15) / 16);
  __shared__ alignas(128) uint4 zeros[ZERO_BYTES / 16];
  chain_wait();
  zero_begin(zero, zeros);
  if (blockIdx.x < p.tiles) {
    const int radix = 1 << p.bits;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const unsigned int lo = blockIdx.x * p.per, hi = min(p.n, lo + p.per);
    unsigned long long word[SORT_ITEMS];
    unsigned int rank[SORT_ITEMS], digit[SORT_ITEMS];
    const auto load = [&](unsigned int step) {
#pragma unroll
      for (int k = 0; k < SORT_ITEMS; k++) {
        const unsigned int i = step + warp * (32 * ITEMS) + k * 32 + lane;
        const bool in = k < ITEMS && i < hi;
        word[k] = in ? source_word(src, i) : 0ull;
        digit[k] = in ? (unsigned int)(word[k] >> p.shift) & (radix - 1) : 0xffffffffu;
      }
    };
    load(lo);
    // words of every digit in all tiles and in the earlier ones: a thread takes
    // 4 digits and a share of the tiles (a digit's few instructions count here:
    // one digit a thread took 3.5 us, this way 1.5)
    const int quads = radix < 4 ? 1 : radix / 4, parts = THREADS / quads;
    {
      const int d = tid & (quads - 1), q = tid / quads;
      uint4 all = make_uint4(0, 0, 0, 0), early = all;
#pragma unroll 6
      for (unsigned int t = q; t < p.tiles; t += parts) {
        const uint4 v = reinterpret_cast<const uint4*>(p.counts)[t * quads + d];
        all.x += v.x, all.y += v.y, all.z += v.z, all.w += v.w;
        if (t < blockIdx.x) early.x += v.x, early.y += v.y, early.z += v.z, early.w += v.w;
      }
      sum[0][tid] = all;
      sum[1][tid] = early;
    }
    __syncthreads();
    unsigned int all = 0;
    if (tid < radix) {
      unsigned int early = 0;
      const unsigned int* shares = reinterpret_cast<const unsigned int*>(sum);
      for (int k = 0; k < parts && k < (int)p.tiles; k++) {
        all += shares[k * quads * 4 + tid];
        early += shares[(THREADS + k * quads) * 4 + tid];
      }
      s.before[tid] = early;
    }
    digit_bases(s, radix, all);
    for (unsigned int step = lo; step < hi; step += THREADS * ITEMS) {
      if (step != lo) load(step);
      const unsigned int total = rank_step(s, radix, ITEMS, digit, rank);
#pragma unroll
      for (int k = 0; k < SORT_ITEMS; k++) {
        if (digit[k] == 0xffffffffu) continue;
        out[s.base[digit[k]] + s.wcount[warp][digit[k]] + rank[k]] = word[k];
      }
      __syncthreads();
      if (tid < radix) s.base[tid] += total;
      __syncthreads();
    }
  }
  zero_end(zero);
}

// Runs: rank[i] = the runs of equal keys that start at or before word i, less
// one, which is the result row of word i. Only words with a row (key <
// num_rows) count.
__device__ __forceinline__ bool is_head(const unsigned long long* w, unsigned int i, unsigned long long num_rows) {
  const unsigned long long k = w[i] >> 32;
  return k < num_rows && (i == 0 || (w[i - 1] >> 32) != k);
}

template <int THREADS>
__global__ void __launch_bounds__(THREADS) head_count_kernel(const unsigned long long* w, unsigned int n,
                                                                  unsigned int per, unsigned long long num_rows,
                                                                  unsigned int* __restrict__ tile_heads) {
  __shared__ unsigned int sum;
  chain_wait();
  if (threadIdx.x == 0) sum = 0;
  __syncthreads();
  const unsigned int lo = blockIdx.x * per, hi = min(n, lo + per);
  unsigned int c = 0;
#pragma unroll 4
  for (unsigned int i = lo + threadIdx.x; i < hi; i += THREADS) c += is_head(w, i, num_rows) ? 1u : 0u;
  for (int o = 16; o; o >>= 1) c += __shfl_xor_sync(0xffffffffu, c, o);
  if ((threadIdx.x & 31) == 0) atomicAdd(&sum, c);  // integers: the order does not matter
  __syncthreads();
  if (threadIdx.x == 0) tile_heads[blockIdx.x] = sum;
}

// Ranks of words [lo, hi) after `run` runs. Every
// warp takes an equal stretch of words, counts its heads and then ranks them.
template <int THREADS>
__device__ __forceinline__ void rank_runs(const unsigned long long* w, unsigned int lo, unsigned int hi,
                                                  unsigned long long num_rows, unsigned int run, unsigned int* wsum,
                                                  unsigned int* rank) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const unsigned int stretch = ((hi - lo + (THREADS / 32) - 1) / (THREADS / 32) + 31) / 32 * 32;
  const unsigned int a = min(hi, lo + warp * stretch), b = min(hi, a + stretch);
  unsigned int mine = 0;
#pragma unroll 4
  for (unsigned int i = a; i < b; i += 32)
    mine += __popc(__ballot_sync(0xffffffffu, i + lane < b && is_head(w, i + lane, num_rows)));
  if (lane == 0) wsum[warp] = mine;
  __syncthreads();
  unsigned int before = run;
#pragma unroll
  for (int k = 0; k < (THREADS / 32); k++) before += k < warp ? wsum[k] : 0u;
#pragma unroll 4
  for (unsigned int i = a; i < b; i += 32) {
    const unsigned int vote = __ballot_sync(0xffffffffu, i + lane < b && is_head(w, i + lane, num_rows));
    if (i + lane < b) rank[i + lane] = before + __popc(vote & (0xffffffffu >> (31 - lane))) - 1u;
    before += __popc(vote);
  }
}

template <int THREADS>
__global__ void __launch_bounds__(THREADS) head_rank_kernel(const unsigned long long* w, unsigned int n,
                                                                 unsigned int per, unsigned int tiles,
                                                                 unsigned long long num_rows,
                                                                 const unsigned int* tile_heads,
                                                                 unsigned int* __restrict__ rank,
                                                                 unsigned long long* count,
                                                                 volatile unsigned long long* host_count) {
  __shared__ unsigned int wsum[THREADS / 32];
  __shared__ unsigned int heads, all;
  chain_wait();
  if (threadIdx.x == 0) heads = all = 0;
  __syncthreads();
  if (threadIdx.x < tiles) {  // integers: the order does not matter
    const unsigned int t = tile_heads[threadIdx.x];
    if (threadIdx.x < blockIdx.x) atomicAdd(&heads, t);
    if (blockIdx.x == 0) atomicAdd(&all, t);
  }
  __syncthreads();
  if (blockIdx.x == 0 && threadIdx.x == 0) {  // first of all: the host may wait for it
    *count = all;
    if (host_count) *host_count = all;
  }
  const unsigned int lo = blockIdx.x * per, hi = min(n, lo + per);
  rank_runs<THREADS>(w, lo, hi, num_rows, heads, wsum, rank);
}

// A short list: the blocks of a cluster sort it in their shared memory, with the
// counts of a pass and then the words themselves exchanged between them, and
// rank its runs (if `rank` is not null). Block c of the cluster has the words [c * tile, (c + 1) * tile), tile =
// items * CLUSTER_THREADS.
constexpr int CLUSTER_THREADS = 1024;
constexpr int CLUSTER_BLOCKS = 8;
struct ClusterShared {
  SortShared<CLUSTER_THREADS> s;
  unsigned int counts[MAX_RADIX];
  unsigned int heads;
  unsigned long long list[CLUSTER_THREADS * SORT_ITEMS];
};

__global__ void __launch_bounds__(CLUSTER_THREADS) cluster_sort_kernel(IdSource src, unsigned int n, int key_bits,
                                                                       int items, unsigned int blocks,
                                                                       unsigned long long* __restrict__ out,
                                                                       unsigned int* __restrict__ rank,
                                                                       unsigned long long* count,
                                                                       volatile unsigned long long* host_count) {
  extern __shared__ uint4 dyn[];
  ClusterShared& c = *reinterpret_cast<ClusterShared*>(dyn);
  SortShared<CLUSTER_THREADS>& s = c.s;
  chain_wait();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const unsigned int me = blockIdx.x, tile = (unsigned int)items * CLUSTER_THREADS;
  const unsigned int lo = me * tile;
  const unsigned int mine = n > lo ? min(tile, n - lo) : 0;
  const auto index = [&](int k) { return (unsigned int)(warp * 32 * items + k * 32 + lane); };
  unsigned long long word[SORT_ITEMS];
#pragma unroll
  for (int k = 0; k < SORT_ITEMS; k++) word[k] = k < items && index(k) < mine ? source_word(src, lo + index(k)) : ~0ull;
  const int passes = (key_bits + MAX_DIGIT_BITS - 1) / MAX_DIGIT_BITS;
  int done = 0;
  for (int p = 0; p < passes; p++) {
    const int bits = (key_bits - done + (passes - p) - 1) / (passes - p), radix = 1 << bits;
    unsigned int r[SORT_ITEMS], digit[SORT_ITEMS];
#pragma unroll
    for (int k = 0; k < SORT_ITEMS; k++)
      digit[k] = k < items && index(k) < mine ? (unsigned int)(word[k] >> (32 + done)) & (radix - 1) : 0xffffffffu;
    const unsigned int total = rank_step(s, radix, items, digit, r);
    if (tid < radix) c.counts[tid] = total;
    cluster_sync();  // the counts are there; every list has been read
    unsigned int all = 0;
    if (tid < radix) {
      unsigned int early = 0;
#pragma unroll
      for (unsigned int q = 0; q < CLUSTER_BLOCKS; q++) {
        if (q >= blocks) break;
        const unsigned int v = peer_load(&c.counts[tid], q);
        all += v;
        early += q < me ? v : 0u;
      }
      s.before[tid] = early;
    }
    digit_bases(s, radix, all);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < SORT_ITEMS; k++) {
      if (digit[k] == 0xffffffffu) continue;
      const unsigned int to = s.base[digit[k]] + s.wcount[warp][digit[k]] + r[k];  // < n
      const unsigned int q = to / tile;
      asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(peer(&c.list[to - q * tile], q)), "l"(word[k]) : "memory");
    }
    cluster_sync();
#pragma unroll
    for (int k = 0; k < SORT_ITEMS; k++)
      if (k < items && index(k) < mine) word[k] = c.list[index(k)];
    done += bits;
  }
#pragma unroll
  for (int k = 0; k < SORT_ITEMS; k++)
    if (k < items && index(k) < mine) out[lo + index(k)] = word[k];
  if (rank) {
    unsigned int votes[SORT_ITEMS], sum = 0;
#pragma unroll
    for (int k = 0; k < SORT_ITEMS; k++) {
      bool head = false;
      if (k < items && index(k) < mine) {
        const unsigned int key = (unsigned int)(word[k] >> 32);
        unsigned int before = 0xffffffffu;  // no key
        if (index(k) > 0)
          before = (unsigned int)(c.list[index(k) - 1] >> 32);
        else if (me > 0)  // the high half of the last word of the block before
          before = peer_load(reinterpret_cast<const unsigned int*>(&c.list[tile - 1]) + 1, me - 1);
        head = key < src.num_rows && key != before;
      }
      votes[k] = __ballot_sync(0xffffffffu, head);
      sum += __popc(votes[k]);
    }
    if (lane == 0) s.wsum[warp] = sum;
    __syncthreads();
    unsigned int run = 0, heads = 0;
#pragma unroll
    for (int w = 0; w < CLUSTER_THREADS / 32; w++) {
      run += w < warp ? s.wsum[w] : 0u;
      heads += s.wsum[w];
    }
    if (tid == 0) c.heads = heads;
    cluster_sync();
    heads = 0;
    for (unsigned int q = 0; q < blocks; q++) {
      const unsigned int v = peer_load(&c.heads, q);
      run += q < me ? v : 0u;
      heads += v;
    }
    if (me == 0 && tid == 0) {
      *count = heads;
      if (host_count) *host_count = heads;
    }
#pragma unroll
    for (int k = 0; k < SORT_ITEMS; k++) {
      if (k < items && index(k) < mine)
        rank[lo + index(k)] = run + __popc(votes[k] & (0xffffffffu >> (31 - lane))) - 1u;
      run += __popc(votes[k]);
    }
  }
  cluster_sync();  // no block leaves while another may read its memory
}

// The zeros of a dense gradient beside cluster_sort_kernel, which leaves most
// SMs free: this kernel starts with it and ends after it, so that the next one
// in the chain finds both done.
__global__ void __launch_bounds__(256) zero_kernel(ZeroFill z) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  zero_tail(z);
  const uint4 zero = make_uint4(0, 0, 0, 0);
  for (unsigned long long at = ((unsigned long long)blockIdx.x * 256 + threadIdx.x) * 16; at < z.bytes;
       at += (unsigned long long)gridDim.x * 256 * 16)
    *reinterpret_cast<uint4*>(z.p + at) = zero;
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// ------------------------------------------------------------ sums over runs
// A team of lanes walks a chunk of the sorted words for one slab of columns (16 or 32
// bytes of the gradient's row to a lane), with the running sum in registers,
// and stores a row of the result where the id changes. Rows of the gradient
// arrive through a ring of asynchronous copies, some rows ahead, which
// keeps about 128 KB an SM in flight at few registers. Sums of runs that cross
// the chunks of a block meet in shared memory; those that cross blocks are left
// in the workspace for join_kernel.
constexpr int SEG_THREADS = 256;
constexpr unsigned int SEG_MAX_ROWS = 1024;  // words of a block
// Rows of the ring, a power of two (with one vector a thread, 4 are as fast; 16
// are 10 to 20 % slower, as fewer blocks fit), and the ring's bytes.
__host__ __device__ constexpr int seg_depth(int vec, int k) { return vec > 1 && k == 2 ? 4 : 8; }
__host__ __device__ constexpr int seg_ring_bytes(int vec, int k, int teams) {
  return seg_depth(vec, k) * 16 * (vec == 1 ? SEG_THREADS + teams : SEG_THREADS * k);
}

struct SegArgs {
  const unsigned long long* words;  // sorted
  const unsigned int* rank;         // null: result rows are the keys (dense)
  void* out;
  const void* grad;
  float* head;  // [blocks][dim] sums of runs that began in an earlier block
  float* tail;  // [blocks][dim] sums of runs that go on in the next block
  long long out_stride, grad_stride;
  unsigned int num_rows, capacity;
  long long dim;
  long long* rows_out;  // with rank: the distinct keys
  unsigned int n, blocks, chunk, team, slabs;  // team: lanes, a power of two
  float scale;
};

__device__ __forceinline__ unsigned int key_of(const SegArgs& a, unsigned int i) {
  return (unsigned int)(a.words[i] >> 32);
}

// A thread has K vectors of VEC columns, vector k at column first + k * step: one
// or two of 16 bytes of the gradient where rows are aligned to them, else single
// elements of 16 bytes together.
template <int VEC, int K>
struct Columns {
  long long first;
  int step;
  __device__ Columns(const SegArgs& a, unsigned int slab) {
    first = ((long long)slab * a.team * K + (threadIdx.x & (a.team - 1))) * VEC;
    step = (int)a.team * VEC;
  }
  __device__ __forceinline__ long long col(int k) const { return first + (long long)k * step; }
};

// the result row of the run that holds word `at`
template <typename W, int VEC, int K>
__device__ __forceinline__ void store_result(const SegArgs& a, const Columns<VEC, K>& c, unsigned int key,
                                             unsigned int at, const F2 (&acc)[VEC * K / 2]) {
  const unsigned int row = a.rank ? a.rank[at] : key;
  if (row >= a.capacity) return;
  if (a.rank && c.first == 0) a.rows_out[row] = (long long)key;
  W* out = reinterpret_cast<W*>(a.out) + (long long)row * a.out_stride;
  const F2 scale(a.scale);
#pragma unroll
  for (int k = 0; k < K; k++) {
    if (c.col(k) >= a.dim) continue;
    float f[VEC];
#pragma unroll
    for (int j = 0; j < VEC; j++) {
      const F2 v = mul2(scale, acc[(k * VEC + j) / 2]);
      f[j] = (k * VEC + j) & 1 ? v.hi() : v.lo();
    }
    store_vec<W, VEC>(out + c.col(k), f);
  }
}

template <int VEC, int K>
__device__ __forceinline__ void store_partial(const SegArgs& a, const Columns<VEC, K>& c, float* row,
                                              const F2 (&acc)[VEC * K / 2]) {
#pragma unroll
  for (int k = 0; k < K; k++) {
    if (c.col(k) >= a.dim) continue;
    float f[VEC];
#pragma unroll
    for (int j = 0; j < VEC; j++) f[j] = (k * VEC + j) & 1 ? acc[(k * VEC + j) / 2].hi() : acc[(k * VEC + j) / 2].lo();
    store_vec<float, VEC>(row + c.col(k), f);
  }
}

template <typename G, typename W, int VEC, int K>
__global__ void __launch_bounds__(SEG_THREADS, 4) segment_kernel(SegArgs a) {
  constexpr bool STAGED = VEC == 1;  // a team copies the 16-byte pieces that cover its columns
  constexpr int P = VEC * K / 2, D = seg_depth(VEC, K);
  constexpr unsigned int NONE = 0xffffffffu;
  enum : unsigned char { CONT = 1, WHOLE = 2, TAIL = 4 };
  constexpr bool WIDE = VEC > 1 && K == 2;
  extern __shared__ uint4 ring[];
  // the words of the block, with the one before and the one behind; behind the
  // ring in the wide kernel (378,383 ids x 5440 fp16: 658 us, 693 in an array)
  __shared__ unsigned long long word_array[WIDE ? 1 : SEG_MAX_ROWS + 2];
  unsigned long long* words = word_array;
  if constexpr (WIDE)
    words = reinterpret_cast<unsigned long long*>(reinterpret_cast<char*>(ring) + seg_ring_bytes(VEC, K, 0));
  __shared__ F2 heads[P][SEG_THREADS];                    // sums of the runs that chunks start inside
  // CONT: the chunk starts inside a run; WHOLE: and the run goes on behind it;
  // TAIL: a run that starts in the chunk goes on behind it
  __shared__ unsigned char flags[SEG_THREADS];
  const unsigned int block = blockIdx.x / a.slabs, slab = blockIdx.x - block * a.slabs;
  const unsigned int teams = SEG_THREADS / a.team, me = threadIdx.x / a.team, lane = threadIdx.x & (a.team - 1);
  const unsigned int rows = a.chunk * teams;
  const unsigned int b0 = block * rows;  // < n
  const unsigned int here = min(rows, a.n - b0);
  chain_wait();
  // words[1 + i] is word b0 + i; a word without a row gets the key NONE (and one
  // of another call's list, whose position is not one of this gradient)
  for (unsigned int i = threadIdx.x; i < rows + 2; i += SEG_THREADS) {
    const bool in = i <= here + 1 && (i > 0 || b0 > 0) && (i <= here || b0 + here < a.n);
    const unsigned long long w = in ? a.words[b0 + i - 1] : ~0ull;
    words[i] = (unsigned int)(w >> 32) < a.num_rows && (unsigned int)w < a.n ? w : ~0ull;
  }
  __syncthreads();
  const Columns<VEC, K> c(a, slab);
  const unsigned long long* mine = words + 1 + me * a.chunk;
  // ring slots: a thread's own vector, or its team's row of the slab
  const int pitch = STAGED ? (SEG_THREADS + (int)teams) * 16 : K * SEG_THREADS * 16;
  char* slot0 = reinterpret_cast<char*>(ring) + (STAGED ? me * (a.team + 1) * 16 : threadIdx.x * 16);
  const char* g0 = reinterpret_cast<const char*>(a.grad) + (STAGED ? c.first - lane : c.first) * (long long)sizeof(G);
  const long long row_bytes = a.grad_stride * (long long)sizeof(G);
  const int slab_bytes = (int)min((long long)a.team * 16, (a.dim - (c.first - (STAGED ? lane : 0))) * (long long)sizeof(G));
  const bool active = STAGED || c.first < a.dim;
  bool also = false;  // the second vector
  if constexpr (!STAGED && K == 2) also = c.col(1) < a.dim;
  const auto fetch = [&](unsigned int i) {
    if (i < a.chunk) {
      const unsigned long long w = mine[i];
      if ((unsigned int)(w >> 32) != NONE && active) {
        const char* src = g0 + (long long)(unsigned int)w * row_bytes;
        char* dst = slot0 + (i & (D - 1)) * pitch;
        if constexpr (STAGED) {
          const int early = (int)(reinterpret_cast<uintptr_t>(src) & 15);
          for (int q = (int)lane * 16; q < early + slab_bytes; q += (int)a.team * 16)
            copy_async_tail(dst + q, src - early + q, min(16, early + slab_bytes - q));
        } else {
          copy_async(dst, src, true);
          if constexpr (K == 2) {
            if (also) copy_async(dst + SEG_THREADS * 16, src + a.team * 16, true);
          }
        }
      }
    }
    copies_commit();
  };
  F2 acc[P];
#pragma unroll
  for (int p = 0; p < P; p++) acc[p] = F2(0.0f);
#pragma unroll 1
  for (unsigned int i = 0; i < D - 1; i++) fetch(i);
  unsigned int cur = (unsigned int)(mine[0] >> 32);
  bool cont = cur != NONE && (unsigned int)(mine[-1] >> 32) == cur;
  unsigned char flag = cont ? CONT : 0;
  // word i + 1 of the chunk decides what becomes of the sum after word i
#pragma unroll 1
  for (unsigned int i = 0; i < a.chunk; i++) {
    if (STAGED) __syncwarp();  // the slot that fetch() refills has been read
    fetch(i + D - 1);
    copies_wait<D - 1>();
    if (STAGED) __syncwarp();
    if (cur == NONE) continue;
    RowVec<G, VEC> v[K];
    const char* src = slot0 + (i & (D - 1)) * pitch;
    if constexpr (STAGED) {
      const int early = (int)(((unsigned int)reinterpret_cast<uintptr_t>(g0) +
                               (unsigned int)mine[i] * (unsigned int)row_bytes) & 15);
#pragma unroll
      for (int k = 0; k < K; k++)
        v[k].v[0] = c.col(k) < a.dim
                        ? *reinterpret_cast<const G*>(src + early + (k * a.team + lane) * (int)sizeof(G))
                        : from_f32<G>(0.0f);
    } else {
#pragma unroll
      for (int k = 0; k < K; k++) v[k] = *reinterpret_cast<const RowVec<G, VEC>*>(src + k * SEG_THREADS * 16);
    }
#pragma unroll
    for (int p = 0; p < P; p++) acc[p] = add2(acc[p], pair_of(v, p));
    const unsigned int next = (unsigned int)(mine[i + 1] >> 32);
    const bool last = i + 1 == a.chunk;
    if (next == cur && !last) continue;
    // the run ends here, or leaves the chunk
    if (cont) {
#pragma unroll
      for (int p = 0; p < P; p++) heads[p][threadIdx.x] = acc[p];
      if (next == cur) flag |= WHOLE;
    } else if (next == cur) {
      flag |= TAIL;
      break;  // acc is the run's sum up to here
    } else if (active) {
      store_result<W, VEC, K>(a, c, cur, b0 + me * a.chunk + i, acc);
    }
    cont = false;
    cur = next;
#pragma unroll
    for (int p = 0; p < P; p++) acc[p] = F2(0.0f);
  }
  copies_wait<0>();
  if (lane == 0) flags[me] = flag;
  __syncthreads();
  // adds the head sums of chunks k, k + 1, ... to acc up to the run's end;
  // false if the run goes on behind the block
  const auto follow = [&](unsigned int k) {
    for (; k < teams; k++) {
#pragma unroll
      for (int p = 0; p < P; p++) acc[p] = add2(acc[p], heads[p][k * a.team + lane]);
      if (!(flags[k] & WHOLE)) return true;
    }
    return false;
  };
  if (flag & TAIL) {
    const unsigned int at = b0 + (me + 1) * a.chunk - 1;  // the chunk's last word
    if (follow(me + 1)) {
      if (active) store_result<W, VEC, K>(a, c, (unsigned int)(words[1 + at - b0] >> 32), at, acc);
    } else if (active) {
      store_partial<VEC, K>(a, c, a.tail + (size_t)block * a.dim, acc);
    }
  }
  if (me == 0 && (flag & CONT)) {
#pragma unroll
    for (int p = 0; p < P; p++) acc[p] = heads[p][threadIdx.x];
    if (flag & WHOLE) follow(1);
    if (active) store_partial<VEC, K>(a, c, a.head + (size_t)block * a.dim, acc);
  }
}

// Runs that cross blocks: the block where a run starts has its tail; the heads
// of the blocks it goes on in are shared out over the teams and added in a
// fixed order.
template <typename W, int VEC, int K>
__global__ void __launch_bounds__(SEG_THREADS) join_kernel(SegArgs a) {
  constexpr int P = VEC * K / 2;
  __shared__ F2 sums[P][SEG_THREADS];
  const unsigned int block = blockIdx.x / a.slabs, slab = blockIdx.x - block * a.slabs;
  chain_wait();
  if (block + 1 >= a.blocks) return;  // the last block's runs end in it
  const unsigned int teams = SEG_THREADS / a.team, me = threadIdx.x / a.team;
  const unsigned int rows = a.chunk * teams;
  const unsigned int b0 = block * rows, b1 = b0 + rows;
  const unsigned int cur = key_of(a, b1);
  if (cur >= a.num_rows || key_of(a, b1 - 1) != cur) return;
  if (b0 > 0 && key_of(a, b0) == cur && key_of(a, b0 - 1) == cur) return;  // it began earlier
  // the blocks it goes on in: those that start with its key
  unsigned int more = 0;
  for (unsigned int base = block + 1;; base += SEG_THREADS) {
    const unsigned int k = base + threadIdx.x;
    const unsigned int some = __syncthreads_count(k < a.blocks && key_of(a, k * rows) == cur);
    more += some;
    if (some < SEG_THREADS) break;
  }
  const Columns<VEC, K> c(a, slab);
  const auto add_row = [&](const float* row, F2 (&acc)[P]) {
    RowVec<float, VEC> v[K];
#pragma unroll
    for (int k = 0; k < K; k++) {
      if (c.col(k) < a.dim) {
        v[k] = load_row<float, VEC>(row + c.col(k));
      } else {
#pragma unroll
        for (int j = 0; j < VEC; j++) v[k].v[j] = 0.0f;
      }
    }
#pragma unroll
    for (int p = 0; p < P; p++) acc[p] = add2(acc[p], pair_of(v, p));
  };
  F2 acc[P];
#pragma unroll
  for (int p = 0; p < P; p++) acc[p] = F2(0.0f);
#pragma unroll 4
  for (unsigned int h = me; h < more; h += teams) add_row(a.head + (size_t)(block + 1 + h) * a.dim, acc);
#pragma unroll
  for (int p = 0; p < P; p++) sums[p][threadIdx.x] = acc[p];
  __syncthreads();
  if (me != 0 || c.first >= a.dim) return;
#pragma unroll
  for (int p = 0; p < P; p++) acc[p] = F2(0.0f);
  add_row(a.tail + (size_t)block * a.dim, acc);
  for (unsigned int t = 0; t < teams && t < more; t++)
#pragma unroll
    for (int p = 0; p < P; p++) acc[p] = add2(acc[p], sums[p][t * a.team + threadIdx.x]);
  store_result<W, VEC, K>(a, c, cur, b1 - 1, acc);
}

// The gradient of a few ids in one kernel: every warp looks for its ids in the
// whole list instead of in a sorted one. A warp takes an id's first position and
// a slab of columns and adds the rows of the positions that share the id. Dense:
// it also zeroes table rows that no id names. Distinct rows: an id's
// row is the number of smaller ids. The additions are those of
// segment_kernel and join_kernel, chunk by chunk and block by block of the
// sorted list, so that the dense form and the distinct rows hold the same bits.
constexpr unsigned int TINY_IDS = GIDS_FEW_IDS;
constexpr int TINY_THREADS = 256;

struct TinyArgs {
  IdSource src;
  void* out;
  const void* grad;
  long long out_stride, grad_stride, dim;
  unsigned int n, slabs;
  unsigned int chunk, rows;  // words of a chunk and of a block (powers of two)
  float scale;
  unsigned int zero_rows;  // dense: rows that a warp zeroes at a time
  bool distinct;
  unsigned int capacity;
  long long* rows_out;                      // of the distinct rows
  volatile unsigned long long* host_count;  // how many there are
};

template <typename G, typename W, int VEC>
__global__ void __launch_bounds__(TINY_THREADS) tiny_grad_kernel(TinyArgs a) {
  constexpr int P = (VEC + 1) / 2, WORDS = TINY_IDS / 32;
  __shared__ unsigned int keys[TINY_IDS];
  const unsigned int none = (unsigned int)a.src.num_rows;  // padding, bad ids and the list's end
  for (unsigned int i = threadIdx.x; i < TINY_IDS; i += TINY_THREADS)
    keys[i] = i < a.n ? (unsigned int)(source_word(a.src, i) >> 32) : none;
  __syncthreads();
  const unsigned int lane = threadIdx.x & 31;
  const unsigned int warp = blockIdx.x * (TINY_THREADS / 32) + (threadIdx.x >> 5);
  const unsigned int warps = gridDim.x * (TINY_THREADS / 32);
  unsigned int mine[WORDS];
  bool lead[WORDS];  // first of its id
#pragma unroll
  for (int w = 0; w < WORDS; w++) {
    mine[w] = keys[w * 32 + lane];
    lead[w] = mine[w] != none;
    if (a.distinct)
      for (unsigned int j = 0; j < w * 32 + lane; j++) lead[w] = lead[w] && keys[j] != mine[w];
  }
  if (a.distinct && blockIdx.x == 0 && threadIdx.x < 32) {
    unsigned int all = 0;
#pragma unroll
    for (int w = 0; w < WORDS; w++) all += __popc(__ballot_sync(0xffffffffu, lead[w]));
    if (threadIdx.x == 0) *a.host_count = all;
  }
  const auto lookup = [&](unsigned int key, unsigned int (&at)[WORDS]) {  // the positions of `key`
#pragma unroll
    for (int w = 0; w < WORDS; w++) at[w] = __ballot_sync(0xffffffffu, mine[w] == key);
  };
  for (unsigned long long task = warp; task < (unsigned long long)a.n * a.slabs; task += warps) {
    const unsigned int i = (unsigned int)(task / a.slabs);
    const long long col = ((long long)(task - (unsigned long long)i * a.slabs) * 32 + lane) * VEC;
    const unsigned int key = keys[i];
    unsigned int at[WORDS];
    lookup(key, at);
    // index: where the id's run starts in the sorted list; row: of the result
    unsigned int first = TINY_IDS, left = 0, index = 0, row = a.distinct ? 0 : key;
#pragma unroll
    for (int w = WORDS - 1; w >= 0; w--) {
      if (at[w]) first = w * 32 + __ffs(at[w]) - 1;
      left += __popc(at[w]);
      index += __popc(__ballot_sync(0xffffffffu, mine[w] < key));
      if (a.distinct) row += __popc(__ballot_sync(0xffffffffu, lead[w] && mine[w] < key));
    }
    if (key == none || first != i || col >= a.dim || row >= a.capacity) continue;  // (no shuffles below)
    if (a.distinct && col == 0) a.rows_out[row] = (long long)key;
    // sums of the chunk, of the block up to the chunk, of the run up to the block
    F2 acc[P], blk[P], tot[P];
    bool in_blk = false, in_tot = false;
    const auto clear = [&](F2 (&v)[P]) {
#pragma unroll
      for (int p = 0; p < P; p++) v[p] = F2(0.0f);
    };
    const auto plus = [&](F2 (&v)[P], const F2 (&w)[P]) {
#pragma unroll
      for (int p = 0; p < P; p++) v[p] = add2(v[p], w[p]);
    };
    const auto close_chunk = [&] {
      if (in_blk) {
        plus(blk, acc);
      } else {
#pragma unroll
        for (int p = 0; p < P; p++) blk[p] = acc[p];
      }
      in_blk = true;
      clear(acc);
    };
    const auto close_block = [&] {  // (join_kernel's sums start from zero)
      F2 v[P];
      clear(v);
      plus(v, blk);
      if (in_tot) {
        plus(tot, v);
      } else {
#pragma unroll
        for (int p = 0; p < P; p++) tot[p] = v[p];
      }
      in_tot = true;
      in_blk = false;
    };
    clear(acc);
    clear(blk);
    clear(tot);
    const G* g = reinterpret_cast<const G*>(a.grad) + col;
    unsigned int pos = i;
    for (bool begun = false; left; begun = true) {
      RowVec<G, VEC> v[4][1];
      const unsigned int some = min(left, 4u);
#pragma unroll
      for (unsigned int u = 0; u < 4; u++) {
        if (u >= some) break;
        while (keys[pos] != key) pos++;  // `left` of them are still to come
        v[u][0] = load_row<G, VEC>(g + (long long)pos * a.grad_stride);
        pos++;
      }
#pragma unroll
      for (unsigned int u = 0; u < 4; u++) {
        if (u >= some) break;
        if (begun || u > 0) {
          if ((index & (a.chunk - 1)) == 0) close_chunk();
          if ((index & (a.rows - 1)) == 0) close_block();
        }
        index++;
#pragma unroll
        for (int p = 0; p < P; p++) {
          if constexpr (VEC == 1)
            acc[p] = add2(acc[p], F2(to_f32(v[u][0].v[0]), 0.0f));
          else
            acc[p] = add2(acc[p], pair_of(v[u], p));
        }
      }
      left -= some;
    }
    close_chunk();
    if (in_tot) close_block();
#pragma unroll
    for (int p = 0; p < P; p++) acc[p] = in_tot ? tot[p] : blk[p];
    float f[VEC];
#pragma unroll
    for (int j = 0; j < VEC; j++) f[j] = a.scale * (j & 1 ? acc[j / 2].hi() : acc[j / 2].lo());
    store_vec<W, VEC>(reinterpret_cast<W*>(a.out) + (long long)row * a.out_stride + col, f);
  }
  if (a.distinct) return;
  W* table = reinterpret_cast<W*>(a.out);
  const auto clear_span = [&](W* out, long long left) {
    if constexpr (VEC == 1) {  // the elements before the first boundary of 16 bytes
      const int early = (int)(-reinterpret_cast<uintptr_t>(out) & 15) / (int)sizeof(W);
      const int head = (int)min((long long)early, left);
      if ((int)lane < head) out[lane] = from_f32<W>(0.0f);
      out += head;
      left -= head;
    }
    constexpr int PER = 16 / (int)sizeof(W);
    const long long pieces = left / PER;
    for (long long c = lane; c < pieces; c += 32) reinterpret_cast<uint4*>(out)[c] = make_uint4(0, 0, 0, 0);
    if (VEC == 1 && (int)lane < (int)(left - pieces * PER)) out[pieces * PER + lane] = from_f32<W>(0.0f);
  };
  // zero_rows rows at a time, in the stretches between those that an id names
  const unsigned long long step = (unsigned long long)warps * a.zero_rows;
  for (unsigned long long base = (unsigned long long)warp * a.zero_rows; base < none; base += step) {
    const unsigned int count = (unsigned int)min((unsigned long long)a.zero_rows, none - base);
    for (unsigned int start = 0; start < count;) {
      unsigned int next = count;
#pragma unroll
      for (int w = 0; w < WORDS; w++) {
        const unsigned int d = mine[w] - (unsigned int)base;  // (of `none`: behind)
        if (d >= start && d < next) next = d;
      }
      next = __reduce_min_sync(0xffffffffu, next);
      if (a.out_stride == a.dim)
        clear_span(table + (long long)(base + start) * a.dim, (long long)(next - start) * a.dim);
      else
        for (unsigned int r = start; r < next; r++) clear_span(table + (long long)(base + r) * a.out_stride, a.dim);
      start = next + 1;
    }
  }
}

// ------------------------------------------------------------------ host side
std::mutex g_err_mu;
constexpr int MAX_DEVICES = 64;
std::atomic<int*> g_err_host[MAX_DEVICES] = {};
int* g_err_dev[MAX_DEVICES] = {};  // under g_err_mu

unsigned int bit_length(unsigned long long v) {
  unsigned int b = 0;
  while (v) b++, v >>= 1;
  return b;
}

void check_ids(const void* ids, int id_bytes, int64_t n, int64_t num_rows, int64_t dim) {
  GIDS_CHECK(n >= 0 && n < (1ll << 31), GIDS_E_INVAL, "n must be in [0, 2^31)");
  GIDS_CHECK(num_rows >= 0 && num_rows < (1ll << 32) - 1, GIDS_E_INVAL, "num_rows must be in [0, 2^32 - 1)");
  GIDS_CHECK(dim >= 1 && dim < (1ll << 31), GIDS_E_INVAL, "dim must be in [1, 2^31)");
  GIDS_CHECK(id_bytes == 4 || id_bytes == 8, GIDS_E_INVAL, "id_bytes must be 4 or 8");
  GIDS_CHECK(n == 0 || ids, GIDS_E_INVAL, "ids is null");
  GIDS_CHECK(((uintptr_t)ids) % (uintptr_t)id_bytes == 0, GIDS_E_INVAL, "ids: address not aligned to its elements");
}

void check_device(int device) {
  GIDS_CHECK(device >= 0 && device < MAX_DEVICES, GIDS_E_INVAL, "bad device");
}

// How the sums are cut: teams of lanes, and chunks of words for a team.
struct SegPlan {
  unsigned int team, slabs, chunk, rows, blocks;  // rows: words of a block (all its teams)
};
SegPlan seg_plan(uint64_t n, uint64_t dim, int elem_bytes) {
  SegPlan p;
  const uint64_t lanes = (dim * elem_bytes + 15) / 16;  // 16 bytes of a row to a lane
  p.team = 1;
  while (p.team < 32 && p.team < lanes) p.team <<= 1;
  p.slabs = (unsigned int)((lanes + p.team - 1) / p.team);
  const unsigned int teams = SEG_THREADS / p.team;
  // long chunks leave fewer partial sums, short ones more work to share out:
  // the longest that gives every SM three blocks
  p.chunk = std::min(32u, SEG_MAX_ROWS / teams);
  while (p.chunk > 4 && (n + p.chunk * teams - 1) / (p.chunk * teams) * p.slabs < 148 * 3) p.chunk >>= 1;
  p.rows = p.chunk * teams;
  p.blocks = (unsigned int)((n + p.rows - 1) / p.rows);
  return p;
}

struct Workspace {
  uint64_t words_a, words_b, counts, tile_heads, count, rank, head, tail, bytes;
  Workspace(uint64_t n, uint64_t dim) {
    const uint64_t blocks = std::max(seg_plan(n, dim, 2).blocks, seg_plan(n, dim, 4).blocks);
    uint64_t at = 0;
    const auto take = [&](uint64_t b) {
      const uint64_t here = at;
      at += (b + 255) / 256 * 256;
      return here;
    };
    count = take(8);
    words_a = take(n * 8);
    words_b = take(n * 8);
    counts = take((uint64_t)MAX_TILES * MAX_RADIX * 4);
    tile_heads = take(MAX_TILES * 4);
    rank = take(n * 4);
    head = take(blocks * dim * 4);
    tail = take(blocks * dim * 4);
    bytes = at;
  }
};

// One kernel of a chain: all but the first start while the one before drains.
struct Cluster {
  unsigned int blocks;
};
template <typename... P, typename... A>
void chain(bool first, void (*kernel)(P...), unsigned int grid, unsigned int block, size_t smem, cudaStream_t st,
           Cluster cluster, A... args) {
  if (smem > 24 * 1024) allow_smem(reinterpret_cast<const void*>(kernel), smem);
  cudaLaunchAttribute attr[2]{};
  unsigned int attrs = 0;
  if (!first) {
    attr[attrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[attrs++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster.blocks > 1) {
    attr[attrs].id = cudaLaunchAttributeClusterDimension;
    attr[attrs].val.clusterDim.x = cluster.blocks;
    attr[attrs].val.clusterDim.y = attr[attrs].val.clusterDim.z = 1;
    attrs++;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = attrs;
  GIDS_CUDA(cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...));
}
template <typename... P, typename... A>
void chain(bool first, void (*kernel)(P...), unsigned int grid, unsigned int block, size_t smem, cudaStream_t st,
           A... args) {
  chain(first, kernel, grid, block, smem, st, Cluster{1}, args...);
}

// Threads of the sort's blocks: more where every SM has more words than a step
// of 512 threads takes (500,009 ids of 24 bits: 64 us with 1,024 threads, 73 with
// 512; 16,384 tokens of 17 bits, dense: 76 and 66 us).
bool wide_sort(uint64_t n) { return n > (uint64_t)MAX_TILES * 512 * SORT_ITEMS; }
constexpr uint64_t SMALL_LIST = (uint64_t)CLUSTER_BLOCKS * CLUSTER_THREADS * SORT_ITEMS;  // for one cluster

// Words of a thread in a step of a scatter: one where that leaves a block to an
// SM (33,000 ids of 23 bits, sort alone: 32 us, 40 with four; 131,072: 43 and 39).
int sort_items(uint64_t n) { return n <= (uint64_t)MAX_TILES * 512 ? 1 : SORT_ITEMS; }

// tiles and words per tile of the sort of n words
void sort_shape(uint64_t n, unsigned int* tiles, unsigned int* per) {
  const uint64_t threads = wide_sort(n) ? 1024 : 512, step = threads * sort_items(n);
  const uint64_t want = std::min<uint64_t>(MAX_TILES, (n + step - 1) / step);
  const uint64_t p = ((n + want - 1) / want + threads - 1) / threads * threads;
  *per = (unsigned int)p;
  *tiles = (unsigned int)((n + p - 1) / p);
}

int key_bits_of(uint64_t num_rows) { return std::max(1u, bit_length(num_rows)); }  // the largest key is num_rows
int passes_of(uint64_t n, uint64_t num_rows) {
  return n <= SMALL_LIST ? 1 : (key_bits_of(num_rows) + MAX_DIGIT_BITS - 1) / MAX_DIGIT_BITS;
}
uint64_t sorted_at(uint64_t n, uint64_t num_rows, const Workspace& lay) {
  return (passes_of(n, num_rows) - 1) & 1 ? lay.words_b : lay.words_a;
}

// Sorts the ids into the workspace, writes `zero` meanwhile and, if asked,
// ranks and counts the runs.
template <int THREADS, int ITEMS>
void sort_ids_by(const IdSource& ids, uint64_t n, char* ws, const Workspace& lay, ZeroFill zero, bool ranks,
                 unsigned long long* count, unsigned long long* host_count, int sms, cudaStream_t st) {
  unsigned int* rank = reinterpret_cast<unsigned int*>(ws + lay.rank);
  if (n <= SMALL_LIST) {
    // few words to a thread first, more blocks next, then more words
    unsigned int items = 1, blocks = 1;
    while (blocks < CLUSTER_BLOCKS && (uint64_t)blocks * CLUSTER_THREADS < n) blocks *= 2;
    while ((uint64_t)blocks * CLUSTER_THREADS * items < n) items *= 2;
    chain(true, cluster_sort_kernel, blocks, CLUSTER_THREADS, sizeof(ClusterShared), st, Cluster{blocks}, ids,
          (unsigned int)n, key_bits_of(ids.num_rows), (int)items, blocks,
          reinterpret_cast<unsigned long long*>(ws + lay.words_a), ranks ? rank : nullptr, count, host_count);
    if (zero.bytes || zero.tail) chain(false, zero_kernel, (unsigned int)sms * 4, 256, 0, st, zero);
    return;
  }
  unsigned int tiles, per;
  sort_shape(n, &tiles, &per);
  const int key_bits = key_bits_of(ids.num_rows), passes = passes_of(n, ids.num_rows);
  const unsigned int grid = std::max(tiles, zero.bytes ? (unsigned int)sms : 1u);
  unsigned long long* buf[2] = {reinterpret_cast<unsigned long long*>(ws + lay.words_a),
                                reinterpret_cast<unsigned long long*>(ws + lay.words_b)};
  // an equal share of the zeros to every kernel
  const uint64_t share = (zero.bytes / (2 * passes) + 15) / 16 * 16;
  const auto next_share = [&] {
    ZeroFill z{zero.p, std::min<uint64_t>(share, zero.bytes), 0};
    zero.p += z.bytes;
    zero.bytes -= z.bytes;
    if (!zero.bytes) std::swap(z.tail, zero.tail);  // the last share
    return z;
  };
  IdSource src = ids;
  Pass pass{(unsigned int)n, per, tiles, 32, 0, reinterpret_cast<unsigned int*>(ws + lay.counts)};
  for (int p = 0; p < passes; p++) {
    pass.shift += pass.bits;
    pass.bits = (32 + key_bits - pass.shift + (passes - p) - 1) / (passes - p);
    chain(p == 0, count_kernel<THREADS>, grid, THREADS, 0, st, src, pass, next_share());
    chain(false, scatter_kernel<THREADS, ITEMS>, grid, THREADS,
          sizeof(SortShared<THREADS>) + 16 + 2 * 16 * THREADS, st, src, pass, buf[p & 1], next_share());
    src.id_bytes = 0;
    src.words = buf[p & 1];
  }
  if (!ranks) return;
  unsigned int* heads = reinterpret_cast<unsigned int*>(ws + lay.tile_heads);
  chain(false, head_count_kernel<THREADS>, tiles, THREADS, 0, st, src.words, (unsigned int)n, per, ids.num_rows, heads);
  chain(false, head_rank_kernel<THREADS>, tiles, THREADS, 0, st, src.words, (unsigned int)n, per, tiles, ids.num_rows,
        (const unsigned int*)heads, rank, count, host_count);
}

void sort_ids(const IdSource& ids, uint64_t n, char* ws, const Workspace& lay, ZeroFill zero, bool ranks,
              unsigned long long* count, unsigned long long* host_count, int sms, cudaStream_t st) {
  if (wide_sort(n))
    sort_ids_by<1024, SORT_ITEMS>(ids, n, ws, lay, zero, ranks, count, host_count, sms, st);
  else if (sort_items(n) == 1)
    sort_ids_by<512, 1>(ids, n, ws, lay, zero, ranks, count, host_count, sms, st);
  else
    sort_ids_by<512, SORT_ITEMS>(ids, n, ws, lay, zero, ranks, count, host_count, sms, st);
}

template <typename G, typename W, int VEC, int K>
void launch_segments_k(SegArgs a, const SegPlan& p, bool first, cudaStream_t st) {
  const uint64_t grid = (uint64_t)p.blocks * a.slabs;
  GIDS_CHECK(grid < (1ull << 31), GIDS_E_UNSUPPORTED, "too many rows x columns for one launch");
  const size_t smem = seg_ring_bytes(VEC, K, SEG_THREADS / (int)p.team) +
                      (VEC > 1 && K == 2 ? (p.rows + 2) * sizeof(unsigned long long) : 0);
  chain(first, segment_kernel<G, W, VEC, K>, (unsigned int)grid, SEG_THREADS, smem, st, a);
  if (p.blocks > 1) chain(false, join_kernel<W, VEC, K>, (unsigned int)grid, SEG_THREADS, 0, st, a);
}

template <typename G, typename W, int VEC>
void launch_segments(SegArgs a, bool first, cudaStream_t st) {
  const SegPlan p = seg_plan(a.n, (uint64_t)a.dim, sizeof(G));
  a.team = p.team;
  a.slabs = p.slabs;
  a.chunk = p.chunk;
  a.blocks = p.blocks;
  if constexpr (VEC > 1) {
    // Two vectors a thread, where that leaves every SM eight blocks: the work on
    // a row's word serves twice the columns. (The sums are bound by instructions
    // else: 378,383 ids x 5440 fp16, dense, 775 us by one vector a thread, 658 by two.
    // With four blocks to an SM, 131,072 x 1024 bf16, both take 78 us.)
    const unsigned int half = (p.slabs + 1) / 2;
    if (p.slabs > 1 && (uint64_t)p.blocks * half >= 148 * 8) {
      a.slabs = half;
      return launch_segments_k<G, W, VEC, 2>(a, p, first, st);
    }
    launch_segments_k<G, W, VEC, 1>(a, p, first, st);
  } else {
    launch_segments_k<G, W, 1, 16 / (int)sizeof(G)>(a, p, first, st);
  }
}

template <typename G, typename W>
void launch_segments_vec(const SegArgs& a, const Rows& out, const Rows& grad, bool first, cudaStream_t st) {
  constexpr int BIG = 16 / (int)sizeof(G);  // a 16-byte vector of the gradient
  if (vec_ok(out, a.dim, BIG) && vec_ok(grad, a.dim, BIG))
    launch_segments<G, W, BIG>(a, first, st);
  else
    launch_segments<G, W, 1>(a, first, st);
}

// first: nothing of this call was launched just before (the workspace is ready)
void segments(const SegArgs& a, const Rows& out, const Rows& grad, bool first, cudaStream_t st) {
  if (out.type == GIDS_F32) {
    if (grad.type == GIDS_F32) return launch_segments_vec<float, float>(a, out, grad, first, st);
    if (grad.type == GIDS_F16) return launch_segments_vec<__half, float>(a, out, grad, first, st);
    return launch_segments_vec<__nv_bfloat16, float>(a, out, grad, first, st);
  }
  if (out.type == GIDS_F16) return launch_segments_vec<__half, __half>(a, out, grad, first, st);
  return launch_segments_vec<__nv_bfloat16, __nv_bfloat16>(a, out, grad, first, st);
}

template <typename G, typename W, int VEC>
void launch_tiny(TinyArgs a, int sms, cudaStream_t st) {
  a.slabs = (unsigned int)((a.dim + 32 * VEC - 1) / (32 * VEC));
  const SegPlan plan = seg_plan(a.n, (uint64_t)a.dim, sizeof(G));
  a.chunk = plan.chunk;
  a.rows = plan.rows;
  // about 2 KB of zeros at a time (64 ids into 10,000,000 x 1 fp32: 52 us by 32 rows at most, 17 us)
  a.zero_rows = (unsigned int)std::clamp<int64_t>(2048 / (a.dim * (int64_t)sizeof(W)), 1, 128);
  const uint64_t tasks =
      std::max<uint64_t>((uint64_t)a.n * a.slabs, a.distinct ? 0 : (a.src.num_rows + a.zero_rows - 1) / a.zero_rows);
  const unsigned int grid = (unsigned int)std::min<uint64_t>((tasks + 7) / 8, (uint64_t)sms * 8);
  tiny_grad_kernel<G, W, VEC><<<grid, TINY_THREADS, 0, st>>>(a);
  GIDS_CUDA(cudaGetLastError());
}

template <typename G, typename W>
void launch_tiny_vec(const TinyArgs& a, const Rows& out, const Rows& grad, int sms, cudaStream_t st) {
  constexpr int BIG = 16 / (int)sizeof(G);
  if (vec_ok(out, a.dim, BIG) && vec_ok(grad, a.dim, BIG)) return launch_tiny<G, W, BIG>(a, sms, st);
  launch_tiny<G, W, 1>(a, sms, st);
}

// (64 ids into 5,000 x 128 fp32, dense: 16 us a pass by the sorted list, 12 this
// way, and 9 since it needs no workspace.)
void tiny(const TinyArgs& a, const Rows& out, const Rows& grad, int sms, cudaStream_t st) {
  if (out.type == GIDS_F32) {
    if (grad.type == GIDS_F32) return launch_tiny_vec<float, float>(a, out, grad, sms, st);
    if (grad.type == GIDS_F16) return launch_tiny_vec<__half, float>(a, out, grad, sms, st);
    return launch_tiny_vec<__nv_bfloat16, float>(a, out, grad, sms, st);
  }
  if (out.type == GIDS_F16) return launch_tiny_vec<__half, __half>(a, out, grad, sms, st);
  launch_tiny_vec<__nv_bfloat16, __nv_bfloat16>(a, out, grad, sms, st);
}

template <typename W, typename O, int VEC>
void launch_embedding(EmbArgs a, uint64_t n, int64_t dim, int id_bytes, cudaStream_t st) {
  a.vpr = (unsigned long long)dim / VEC;
  a.vdiv = FastDiv((unsigned int)a.vpr);
  a.total = n * a.vpr;
  const uint64_t blocks = (a.total + EMB_THREADS * EMB_UNROLL - 1) / (EMB_THREADS * EMB_UNROLL);
  GIDS_CHECK(blocks < (1ull << 31), GIDS_E_UNSUPPORTED, "too many rows x columns for one launch");
  if (id_bytes == 4)
    embedding_kernel<W, O, VEC, int><<<(unsigned int)blocks, EMB_THREADS, 0, st>>>(a);
  else
    embedding_kernel<W, O, VEC, long long><<<(unsigned int)blocks, EMB_THREADS, 0, st>>>(a);
  GIDS_CUDA(cudaGetLastError());
}

template <typename W, typename O>
void launch_embedding_vec(const EmbArgs& a, const Rows& out, const Rows& weight, uint64_t n, int64_t dim, int id_bytes,
                          cudaStream_t st) {
  constexpr int BIG = 16 / (int)sizeof(W);  // a 16-byte vector of the table
  if (vec_ok(out, dim, BIG) && vec_ok(weight, dim, BIG)) return launch_embedding<W, O, BIG>(a, n, dim, id_bytes, st);
  if (vec_ok(out, dim, BIG / 2) && vec_ok(weight, dim, BIG / 2))
    return launch_embedding<W, O, BIG / 2>(a, n, dim, id_bytes, st);
  // a warp to a slab pays off from a few hundred bytes of row on
  if (dim * (int64_t)sizeof(W) < 256) return launch_embedding<W, O, 1>(a, n, dim, id_bytes, st);
  const uint64_t slabs = ((uint64_t)dim + ODD_SLAB - 1) / ODD_SLAB;
  int dev = 0;
  GIDS_CUDA(cudaGetDevice(&dev));
  const size_t smem = (size_t)(ODD_SLAB * sizeof(W) + 16) * ODD_STAGES * (ODD_THREADS / 32);
  const uint64_t want = (n * slabs + ODD_THREADS / 32 - 1) / (ODD_THREADS / 32);
  const unsigned int grid =
      (unsigned int)std::min<uint64_t>(want, (uint64_t)device_sms(dev) * (sizeof(W) == 4 ? 3 : 6));
  const auto kernel = id_bytes == 4 ? embedding_odd_kernel<W, O, int> : embedding_odd_kernel<W, O, long long>;
  if (smem > 40 * 1024) allow_smem(reinterpret_cast<const void*>(kernel), smem);
  kernel<<<grid, ODD_THREADS, smem, st>>>(a, n, dim, (unsigned int)slabs);
  GIDS_CUDA(cudaGetLastError());
}

// A new word of mapped host memory, and its address on the device.
template <typename T>
T* mapped_word(T** dev) {
  RelaxedCapture any;
  T* host = nullptr;
  GIDS_CUDA(cudaHostAlloc(&host, sizeof(T), cudaHostAllocMapped | cudaHostAllocPortable));
  const cudaError_t e = cudaHostGetDevicePointer(dev, host, 0);
  if (e != cudaSuccess) cudaFreeHost(host);
  GIDS_CUDA(e);
  return host;
}

// A word of mapped host memory for the time of a call that waits for a number
// from its kernels. They store it once, as soon as they know it, so the call
// returns while they still work (500,009 ids x 128 fp32: 171 us a pass by waiting
// for the stream, 160 this way).
std::mutex g_words_mu;
std::vector<unsigned long long*> g_words;
struct HostWord {
  static constexpr unsigned long long NONE = ~0ull;
  unsigned long long *host = nullptr, *dev = nullptr;
  bool done = false;  // no kernel is left that writes it
  explicit HostWord(bool wanted) {
    if (!wanted) return;
    {
      std::lock_guard<std::mutex> lk(g_words_mu);
      if (!g_words.empty()) {
        host = g_words.back();
        g_words.pop_back();
      }
    }
    if (host)
      GIDS_CUDA(cudaHostGetDevicePointer(&dev, host, 0));
    else
      host = mapped_word(&dev);
    __atomic_store_n(host, NONE, __ATOMIC_RELEASE);
  }
  unsigned long long wait(cudaStream_t st) {
    unsigned long long v = NONE;
    for (int i = 0; i < 20000 && v == NONE; i++) {  // about a millisecond
#if defined(__x86_64__)
      __builtin_ia32_pause();
#endif
      v = __atomic_load_n(host, __ATOMIC_ACQUIRE);
    }
    if (v == NONE) {
      RelaxedCapture any;
      GIDS_CUDA(cudaStreamSynchronize(st));
      v = __atomic_load_n(host, __ATOMIC_ACQUIRE);
    }
    done = true;
    return v;
  }
  ~HostWord() {
    if (!done) return;  // a call that failed half way: another one must not get this word
    std::lock_guard<std::mutex> lk(g_words_mu);
    g_words.push_back(host);
  }
};

IdSource id_source(const void* ids, int id_bytes, int64_t num_rows, int64_t padding_idx, int* err) {
  IdSource s{};
  s.ids = ids;
  s.id_bytes = id_bytes;
  s.num_rows = (unsigned long long)num_rows;
  s.padding = padding_idx;
  s.err = err;
  return s;
}

// few: the call's kernel needs none, so there may be none (null, 0 bytes)
void check_workspace(const void* ws, uint64_t ws_bytes, const Workspace& lay, bool few = false) {
  if (few && !ws && !ws_bytes) return;
  GIDS_CHECK(ws && ((uintptr_t)ws) % 256 == 0, GIDS_E_INVAL, "workspace is null or not aligned to 256 bytes");
  GIDS_CHECK(ws_bytes >= lay.bytes, GIDS_E_INVAL,
             "workspace too small: " + std::to_string(lay.bytes) + " bytes are needed");
}

}  // namespace

void allow_smem(const void* kernel, size_t bytes) {
  static std::mutex mu;
  static std::map<std::pair<int, const void*>, size_t> allowed;
  int dev = 0;
  GIDS_CUDA(cudaGetDevice(&dev));
  std::lock_guard<std::mutex> lk(mu);
  size_t& most = allowed[{dev, kernel}];
  if (bytes <= most) return;
  GIDS_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
  most = bytes;
}

int* id_error_word(int device) {
  std::lock_guard<std::mutex> lk(g_err_mu);
  if (!g_err_dev[device]) {
    int* d = nullptr;
    int* h = mapped_word(&d);
    *h = 0;
    g_err_dev[device] = d;
    g_err_host[device].store(h, std::memory_order_release);
  }
  return g_err_dev[device];
}

void check_id_errors(int device) {
  int* h = g_err_host[device].load(std::memory_order_acquire);
  if (h && *reinterpret_cast<volatile int*>(h) && __atomic_exchange_n(h, 0, __ATOMIC_ACQ_REL))
    throw Error(GIDS_E_RANGE,
                "an id of an earlier embedding call lay outside its table (its output row is zero, its gradient is "
                "left out)");
}

void embedding(int device, Rows out, Rows weight, int64_t num_rows, int64_t dim, const void* ids, int id_bytes,
               int64_t n, float scale, cudaStream_t st) {
  check_device(device);
  check_ids(ids, id_bytes, n, num_rows, dim);
  check_rows(out, "out", n, dim, true);
  check_rows(weight, "weight", n && num_rows ? 1 : 0, dim, false);
  GIDS_CHECK(out.type == weight.type || weight.type == GIDS_F32, GIDS_E_UNSUPPORTED,
             "out must have the table's type, or the table be float32");
  check_id_errors(device);
  if (n == 0) return;
  DeviceGuard dg(device);
  EmbArgs a{};
  a.out = out.p;
  a.weight = weight.p;
  a.ids = ids;
  a.out_stride = out.stride;
  a.weight_stride = weight.stride;
  a.num_rows = (unsigned long long)num_rows;
  a.scale = scale;
  a.err = id_error_word(device);
  if (weight.type == GIDS_F32) {
    if (out.type == GIDS_F32) return launch_embedding_vec<float, float>(a, out, weight, n, dim, id_bytes, st);
    if (out.type == GIDS_F16) return launch_embedding_vec<float, __half>(a, out, weight, n, dim, id_bytes, st);
    return launch_embedding_vec<float, __nv_bfloat16>(a, out, weight, n, dim, id_bytes, st);
  }
  if (weight.type == GIDS_F16) return launch_embedding_vec<__half, __half>(a, out, weight, n, dim, id_bytes, st);
  return launch_embedding_vec<__nv_bfloat16, __nv_bfloat16>(a, out, weight, n, dim, id_bytes, st);
}

uint64_t embedding_grad_workspace(int64_t n, int64_t num_rows, int64_t dim) {
  check_ids(reinterpret_cast<const void*>(256), 8, n, num_rows, dim);
  return Workspace((uint64_t)n, (uint64_t)dim).bytes;
}

void embedding_grad(int device, Rows dweight, int64_t num_rows, int64_t dim, Rows grad, const void* ids, int id_bytes,
                    int64_t n, int64_t padding_idx, float scale, void* ws, uint64_t ws_bytes, cudaStream_t st) {
  check_device(device);
  check_ids(ids, id_bytes, n, num_rows, dim);
  check_rows(dweight, "dweight", num_rows, dim, true);
  check_rows(grad, "grad", n, dim, false);
  GIDS_CHECK(dweight.type == grad.type || dweight.type == GIDS_F32, GIDS_E_UNSUPPORTED,
             "dweight must have the gradient's type or be float32");
  GIDS_CHECK(padding_idx >= -1 && padding_idx < std::max<int64_t>(num_rows, 1), GIDS_E_INVAL,
             "padding_idx must be -1 (none) or a row");
  const Workspace lay((uint64_t)n, (uint64_t)dim);
  if (n) check_workspace(ws, ws_bytes, lay, n <= (int64_t)TINY_IDS);
  check_id_errors(device);
  if (num_rows == 0 && n == 0) return;
  DeviceGuard dg(device);
  if (n > 0 && n <= (int64_t)TINY_IDS) {
    TinyArgs t{};
    t.src = id_source(ids, id_bytes, num_rows, padding_idx, id_error_word(device));
    t.out = dweight.p;
    t.grad = grad.p;
    t.out_stride = dweight.stride;
    t.grad_stride = grad.stride;
    t.dim = dim;
    t.n = (unsigned int)n;
    t.scale = scale;
    t.capacity = (unsigned int)num_rows;
    return tiny(t, dweight, grad, device_sms(device), st);
  }
  const size_t eb = (size_t)type_bytes(dweight.type);
  const uint64_t total = (uint64_t)num_rows * (uint64_t)dim * eb;
  ZeroFill zero{static_cast<char*>(dweight.p), total / 16 * 16, (unsigned int)(total % 16)};
  // the zeros go out beside the sort if they are one stretch of memory
  const bool stretch = num_rows <= 1 || dweight.stride == dim;
  if (n == 0 || !stretch || ((uintptr_t)dweight.p) % 16) {
    zero = ZeroFill{};
    if (stretch)
      GIDS_CUDA(cudaMemsetAsync(dweight.p, 0, total, st));
    else
      GIDS_CUDA(cudaMemset2DAsync(dweight.p, (size_t)dweight.stride * eb, 0, (size_t)dim * eb, (size_t)num_rows, st));
  }
  if (n == 0) return;
  char* base = static_cast<char*>(ws);
  sort_ids(id_source(ids, id_bytes, num_rows, padding_idx, id_error_word(device)), (uint64_t)n, base, lay, zero, false,
           nullptr, nullptr, device_sms(device), st);
  SegArgs a{};
  a.words = reinterpret_cast<const unsigned long long*>(base + sorted_at((uint64_t)n, (uint64_t)num_rows, lay));
  a.out = dweight.p;
  a.grad = grad.p;
  a.head = reinterpret_cast<float*>(base + lay.head);
  a.tail = reinterpret_cast<float*>(base + lay.tail);
  a.out_stride = dweight.stride;
  a.grad_stride = grad.stride;
  a.num_rows = a.capacity = (unsigned int)num_rows;
  a.dim = dim;
  a.n = (unsigned int)n;
  a.scale = scale;
  segments(a, dweight, grad, false, st);
}

namespace {
// Checks of the calls that return the number of distinct rows to the host.
void check_group(int device, const void* ids, int id_bytes, int64_t n, int64_t num_rows, int64_t padding_idx,
                 int64_t dim, const void* ws, uint64_t ws_bytes, bool few) {
  check_device(device);
  check_ids(ids, id_bytes, n, num_rows, dim);
  GIDS_CHECK(padding_idx >= -1 && padding_idx < std::max<int64_t>(num_rows, 1), GIDS_E_INVAL,
             "padding_idx must be -1 (none) or a row");
  check_workspace(ws, ws_bytes, Workspace((uint64_t)n, (uint64_t)dim), few);
}
void check_not_capturing(cudaStream_t st) {
  cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
  GIDS_CUDA(cudaStreamIsCapturing(st, &cap));
  GIDS_CHECK(cap == cudaStreamCaptureStatusNone, GIDS_E_STATE,
             "count_host makes the call wait for the stream, which is being captured into a graph");
}
void check_values(const int64_t* rows, const Rows& values, int64_t capacity, const Rows& grad, int64_t n,
                  int64_t dim) {
  GIDS_CHECK(capacity >= 0, GIDS_E_INVAL, "capacity must be >= 0");
  GIDS_CHECK(capacity == 0 || rows, GIDS_E_INVAL, "rows is null");
  GIDS_CHECK(((uintptr_t)rows) % 8 == 0, GIDS_E_INVAL, "rows: address not aligned to its elements");
  check_rows(values, "values", capacity, dim, true);
  check_rows(grad, "grad", n, dim, false);
  GIDS_CHECK(values.type == grad.type || values.type == GIDS_F32, GIDS_E_UNSUPPORTED,
             "values must have the gradient's type or be float32");
}
// the sums of the sorted words in the workspace
void sum_rows(int64_t* rows, const Rows& values, int64_t capacity, int64_t num_rows, int64_t dim, const Rows& grad,
              int64_t n, float scale, char* base, const Workspace& lay, bool first, cudaStream_t st) {
  SegArgs a{};
  a.words = reinterpret_cast<const unsigned long long*>(base + sorted_at((uint64_t)n, (uint64_t)num_rows, lay));
  a.rank = reinterpret_cast<const unsigned int*>(base + lay.rank);
  a.rows_out = reinterpret_cast<long long*>(rows);
  a.out = values.p;
  a.grad = grad.p;
  a.head = reinterpret_cast<float*>(base + lay.head);
  a.tail = reinterpret_cast<float*>(base + lay.tail);
  a.out_stride = values.stride;
  a.grad_stride = grad.stride;
  a.num_rows = (unsigned int)num_rows;
  a.capacity = (unsigned int)std::min<int64_t>(capacity, n);
  a.dim = dim;
  a.n = (unsigned int)n;
  a.scale = scale;
  segments(a, values, grad, first, st);
}
}  // namespace

void embedding_group(int device, const void* ids, int id_bytes, int64_t n, int64_t num_rows, int64_t padding_idx,
                     int64_t dim, void* ws, uint64_t ws_bytes, uint64_t* count_dev, uint64_t* count_host,
                     cudaStream_t st) {
  check_group(device, ids, id_bytes, n, num_rows, padding_idx, dim, ws, ws_bytes, false);
  GIDS_CHECK(((uintptr_t)count_dev) % 8 == 0, GIDS_E_INVAL, "count_dev: address not aligned to its element");
  check_id_errors(device);
  DeviceGuard dg(device);
  if (count_host) check_not_capturing(st);
  if (n == 0) {
    if (count_dev) GIDS_CUDA(cudaMemsetAsync(count_dev, 0, sizeof(*count_dev), st));
    if (count_host) *count_host = 0;
    return;
  }
  const Workspace lay((uint64_t)n, (uint64_t)dim);
  char* base = static_cast<char*>(ws);
  HostWord word(count_host != nullptr);
  unsigned long long* count =
      count_dev ? reinterpret_cast<unsigned long long*>(count_dev) : reinterpret_cast<unsigned long long*>(base + lay.count);
  sort_ids(id_source(ids, id_bytes, num_rows, padding_idx, id_error_word(device)), (uint64_t)n, base, lay, ZeroFill{},
           true, count, word.dev, 1, st);
  if (count_host) *count_host = word.wait(st);
}

void embedding_grad_rows(int device, int64_t* rows, Rows values, int64_t capacity, int64_t num_rows, int64_t dim,
                         Rows grad, int64_t n, float scale, void* ws, uint64_t ws_bytes, cudaStream_t st) {
  check_device(device);
  check_ids(reinterpret_cast<const void*>(256), 8, n, num_rows, dim);
  check_values(rows, values, capacity, grad, n, dim);
  const Workspace lay((uint64_t)n, (uint64_t)dim);
  check_workspace(ws, ws_bytes, lay);
  if (n == 0 || capacity == 0) return;
  DeviceGuard dg(device);
  sum_rows(rows, values, capacity, num_rows, dim, grad, n, scale, static_cast<char*>(ws), lay, true, st);
}

void embedding_grad_distinct(int device, int64_t* rows, Rows values, int64_t capacity, int64_t num_rows, int64_t dim,
                             Rows grad, const void* ids, int id_bytes, int64_t n, int64_t padding_idx, float scale,
                             void* ws, uint64_t ws_bytes, uint64_t* count_host, cudaStream_t st) {
  check_group(device, ids, id_bytes, n, num_rows, padding_idx, dim, ws, ws_bytes, n <= (int64_t)TINY_IDS);
  check_values(rows, values, capacity, grad, n, dim);
  GIDS_CHECK(capacity >= std::min(n, num_rows), GIDS_E_INVAL, "capacity must be at least min(n, num_rows)");
  check_id_errors(device);
  DeviceGuard dg(device);
  check_not_capturing(st);
  *count_host = 0;
  if (n == 0) return;
  HostWord word(true);
  if (n <= (int64_t)TINY_IDS) {
    TinyArgs t{};
    t.src = id_source(ids, id_bytes, num_rows, padding_idx, id_error_word(device));
    t.out = values.p;
    t.grad = grad.p;
    t.out_stride = values.stride;
    t.grad_stride = grad.stride;
    t.dim = dim;
    t.n = (unsigned int)n;
    t.scale = scale;
    t.distinct = true;
    t.rows_out = reinterpret_cast<long long*>(rows);
    t.capacity = (unsigned int)std::min<int64_t>(capacity, n);
    t.host_count = word.dev;
    tiny(t, values, grad, device_sms(device), st);
    *count_host = word.wait(st);
    return;
  }
  const Workspace lay((uint64_t)n, (uint64_t)dim);
  char* base = static_cast<char*>(ws);
  sort_ids(id_source(ids, id_bytes, num_rows, padding_idx, id_error_word(device)), (uint64_t)n, base, lay, ZeroFill{},
           true, reinterpret_cast<unsigned long long*>(base + lay.count), word.dev, 1, st);
  if (capacity) sum_rows(rows, values, capacity, num_rows, dim, grad, n, scale, base, lay, false, st);
  *count_host = word.wait(st);
}

void embedding_check(int device, cudaStream_t st) {
  check_device(device);
  DeviceGuard dg(device);
  cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
  GIDS_CUDA(cudaStreamIsCapturing(st, &cap));
  GIDS_CHECK(cap == cudaStreamCaptureStatusNone, GIDS_E_STATE,
             "the check waits for the stream, which is being captured into a graph");
  {
    RelaxedCapture any;
    GIDS_CUDA(cudaStreamSynchronize(st));
  }
  check_id_errors(device);
}

}  // namespace gids
