// Embedding lookup with scaling and its gradient by sorted ids, for sm_100a.
//
// Lookup: out[i, :] = round(scale * weight[id_i, :]). One thread moves UNROLL
// vectors of a flat (row, vector) index space, so rows of any width fill the
// warps; an id outside the table gives a zero row and sets the device's error
// word.
//
// Gradient: dweight[v, :] = round(scale * sum over {i : id_i = v} of grad[i, :]).
// The ids are sorted (LSD radix sort of (id, position) words, stable, so equal
// ids stay in position order), and the sorted list is cut into chunks of
// CHUNK entries. A team of lanes owns one chunk and one slab of columns, walks
// its entries with the running sum in registers, and stores a row of the
// result whenever the id changes. A run of equal ids that crosses a chunk's
// border leaves float32 partial sums in the workspace, which a second kernel
// adds in chunk order. Nothing is accumulated with atomics, so results repeat
// bit for bit. Padding and bad ids sort behind every row and are left out.
#include <algorithm>
#include <atomic>
#include <mutex>
#include <type_traits>

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
        store_raw(o, v[u]);
        continue;
      }
    }
    float f[VEC];
#pragma unroll
    for (int j = 0; j < VEC; j++) f[j] = good[u] ? a.scale * to_f32(v[u].v[j]) : 0.0f;
    if (!good[u]) *reinterpret_cast<volatile int*>(a.err) = 1;
    store_vec<O, VEC>(o, f);
  }
}

// ------------------------------------------------------------------ the sort
constexpr int SORT_THREADS = 512;
constexpr int SORT_WARPS = SORT_THREADS / 32;
constexpr int SORT_ITEMS = 4;
constexpr int SORT_STEP = SORT_THREADS * SORT_ITEMS;
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

// counts[tile][digit] of one digit of the keys; tile t covers `per` words
__global__ void __launch_bounds__(SORT_THREADS) count_kernel(IdSource src, unsigned int n, unsigned int per, int shift,
                                                             int bits, unsigned int* __restrict__ counts) {
  __shared__ unsigned int hist[MAX_RADIX];
  const int radix = 1 << bits;
  for (int d = threadIdx.x; d < radix; d += SORT_THREADS) hist[d] = 0;
  __syncthreads();
  const unsigned int lo = blockIdx.x * per, hi = min(n, lo + per);
  for (unsigned int i = lo + threadIdx.x; i < hi; i += SORT_THREADS) {
    const unsigned long long w = source_word(src, i);
    atomicAdd(&hist[(unsigned int)(w >> shift) & (radix - 1)], 1u);
  }
  __syncthreads();
  for (int d = threadIdx.x; d < radix; d += SORT_THREADS) counts[(size_t)blockIdx.x * radix + d] = hist[d];
}

// Stable scatter of tile blockIdx.x by one digit: word order within a tile is
// (step, warp, item, lane), which is the order of the positions.
__global__ void __launch_bounds__(SORT_THREADS) scatter_kernel(IdSource src, unsigned int n, unsigned int per,
                                                               unsigned int tiles, int shift, int bits,
                                                               const unsigned int* __restrict__ counts,
                                                               unsigned long long* __restrict__ out) {
  __shared__ unsigned int base[MAX_RADIX];                   // next output index of each digit
  __shared__ unsigned short wcount[SORT_WARPS][MAX_RADIX];   // digits of this step, by warp
  __shared__ unsigned int wsum[SORT_WARPS];
  const int radix = 1 << bits;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // base[d] = words of smaller digits + words of digit d in earlier tiles
  unsigned int before = 0, total = 0;
  if (tid < radix) {
#pragma unroll 16
    for (unsigned int t = 0; t < tiles; t++) {
      const unsigned int c = counts[(size_t)t * radix + tid];
      total += c;
      before += t < blockIdx.x ? c : 0u;
    }
  }
  unsigned int incl = total;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned int v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) wsum[warp] = incl;
  __syncthreads();
  unsigned int off = 0;
  for (int w = 0; w < warp; w++) off += wsum[w];
  if (tid < radix) base[tid] = off + incl - total + before;

  const unsigned int lo = blockIdx.x * per, hi = min(n, lo + per);
  for (unsigned int step = lo; step < hi; step += SORT_STEP) {
    __syncthreads();
    for (int i = tid; i < SORT_WARPS * MAX_RADIX / 2; i += SORT_THREADS)
      reinterpret_cast<unsigned int*>(&wcount[0][0])[i] = 0;
    __syncthreads();
    unsigned long long word[SORT_ITEMS];
    unsigned int rank[SORT_ITEMS];
    unsigned int digit[SORT_ITEMS];
#pragma unroll
    for (int k = 0; k < SORT_ITEMS; k++) {
      const unsigned int i = step + warp * (32 * SORT_ITEMS) + k * 32 + lane;
      word[k] = i < hi ? source_word(src, i) : 0ull;
      digit[k] = i < hi ? (unsigned int)(word[k] >> shift) & (radix - 1) : 0xffffffffu;
    }
#pragma unroll
    for (int k = 0; k < SORT_ITEMS; k++) {
      const unsigned int peers = __match_any_sync(0xffffffffu, digit[k]);
      const bool in = digit[k] != 0xffffffffu;
      const unsigned int prior = in ? wcount[warp][digit[k]] : 0u;
      __syncwarp();
      rank[k] = prior + __popc(peers & ((1u << lane) - 1u));
      if (in && (peers >> lane) == 1u) wcount[warp][digit[k]] = (unsigned short)(prior + __popc(peers));
      __syncwarp();
    }
    __syncthreads();
    // by digit: warps' counts -> offsets within the step; base moves on
    if (tid < radix) {
      unsigned int run = 0;
#pragma unroll
      for (int w = 0; w < SORT_WARPS; w++) {
        const unsigned int c = wcount[w][tid];
        wcount[w][tid] = (unsigned short)run;
        run += c;
      }
      total = run;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < SORT_ITEMS; k++)
      if (digit[k] != 0xffffffffu) out[base[digit[k]] + wcount[warp][digit[k]] + rank[k]] = word[k];
    __syncthreads();
    if (tid < radix) base[tid] += total;
  }
}

// --------------------------------------------------- the distinct ids, in order
// A head is the first word of a run of equal keys (of rows: key < num_rows).
__device__ __forceinline__ bool is_head(const unsigned long long* w, unsigned int i, unsigned int n,
                                        unsigned long long num_rows) {
  if (i >= n) return false;
  const unsigned long long k = w[i] >> 32;
  return k < num_rows && (i == 0 || (w[i - 1] >> 32) != k);
}

__global__ void __launch_bounds__(SORT_THREADS) head_count_kernel(const unsigned long long* __restrict__ w,
                                                                  unsigned int n, unsigned int per,
                                                                  unsigned long long num_rows,
                                                                  unsigned int* __restrict__ tile_heads) {
  __shared__ unsigned int sum;
  if (threadIdx.x == 0) sum = 0;
  __syncthreads();
  const unsigned int lo = blockIdx.x * per, hi = min(n, lo + per);
  unsigned int c = 0;
  for (unsigned int i = lo + threadIdx.x; i < hi; i += SORT_THREADS) c += is_head(w, i, n, num_rows) ? 1u : 0u;
  for (int o = 16; o; o >>= 1) c += __shfl_xor_sync(0xffffffffu, c, o);
  if ((threadIdx.x & 31) == 0) atomicAdd(&sum, c);  // integers: the order does not matter
  __syncthreads();
  if (threadIdx.x == 0) tile_heads[blockIdx.x] = sum;
}

// chunk_rank[c] = heads before word c * chunk; *count = all heads
__global__ void __launch_bounds__(SORT_THREADS) head_rank_kernel(const unsigned long long* __restrict__ w,
                                                                 unsigned int n, unsigned int per, unsigned int tiles,
                                                                 unsigned long long num_rows, unsigned int chunk_shift,
                                                                 const unsigned int* __restrict__ tile_heads,
                                                                 unsigned int* __restrict__ chunk_rank,
                                                                 unsigned long long* __restrict__ count) {
  __shared__ unsigned int wsum[SORT_WARPS];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  unsigned int run = 0, all = 0;
  for (unsigned int t = 0; t < tiles; t++) {
    const unsigned int c = tile_heads[t];
    run += t < blockIdx.x ? c : 0u;
    all += c;
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) *count = all;
  const unsigned int lo = blockIdx.x * per, hi = min(n, lo + per);
  for (unsigned int step = lo; step < hi; step += SORT_THREADS) {
    const unsigned int i = step + threadIdx.x;
    const bool head = i < hi && is_head(w, i, n, num_rows);
    const unsigned int vote = __ballot_sync(0xffffffffu, head);
    __syncthreads();
    if (lane == 0) wsum[warp] = __popc(vote);
    __syncthreads();
    unsigned int before = run, sum = 0;
#pragma unroll
    for (int k = 0; k < SORT_WARPS; k++) {
      before += k < warp ? wsum[k] : 0u;
      sum += wsum[k];
    }
    const unsigned int rank = before + __popc(vote & ((1u << lane) - 1u));
    if (i < hi && (i & ((1u << chunk_shift) - 1u)) == 0) chunk_rank[i >> chunk_shift] = rank;
    run += sum;
  }
}

// ------------------------------------------------------------ sums over runs
constexpr int SEG_THREADS = 256;
constexpr int SEG_UNROLL = 8;

struct SegArgs {
  const unsigned long long* words;  // sorted
  const unsigned int* chunk_rank;   // null: result rows are the keys (dense)
  void* out;
  const void* grad;
  float* head;  // [chunks][dim] sums of runs that began in an earlier chunk
  float* tail;  // [chunks][dim] sums of runs that go on in the next chunk
  long long out_stride, grad_stride;
  unsigned long long num_rows, capacity;
  long long dim;
  long long* rows_out;  // with chunk_rank: the distinct keys, widened
  unsigned int n, chunks, chunk_shift, team, slabs;
  float scale;
};

template <typename W, int VEC>
__device__ __forceinline__ void store_result(const SegArgs& a, unsigned long long row, long long col,
                                             const float (&acc)[VEC]) {
  float f[VEC];
#pragma unroll
  for (int j = 0; j < VEC; j++) f[j] = a.scale * acc[j];
  store_vec<W, VEC>(reinterpret_cast<W*>(a.out) + (long long)row * a.out_stride + col, f);
}

template <typename G, typename W, int VEC>
__global__ void __launch_bounds__(SEG_THREADS) segment_kernel(SegArgs a) {
  const unsigned long long item = ((unsigned long long)blockIdx.x * SEG_THREADS + threadIdx.x) / a.team;
  const unsigned long long chunk64 = item / a.slabs;
  if (chunk64 >= a.chunks) return;
  const unsigned int chunk = (unsigned int)chunk64;
  const unsigned int slab = (unsigned int)(item - chunk64 * a.slabs);
  const long long col = ((long long)slab * a.team + (threadIdx.x & (a.team - 1))) * VEC;
  if (col >= a.dim) return;
  const unsigned int i0 = chunk << a.chunk_shift;
  const unsigned int i1 = (unsigned int)min((unsigned long long)a.n, (unsigned long long)i0 + (1ull << a.chunk_shift));
  unsigned long long cur = a.words[i0] >> 32;
  if (cur >= a.num_rows) return;  // sorted: only padding and bad ids from here on
  bool cont = i0 > 0 && (a.words[i0 - 1] >> 32) == cur;
  // row of the run in hand; a run that began earlier is stored by the joiner
  unsigned long long rank = a.chunk_rank ? a.chunk_rank[chunk] : 0ull;
  if (cont) rank--;
  float acc[VEC];
#pragma unroll
  for (int j = 0; j < VEC; j++) acc[j] = 0.0f;
  const G* g = reinterpret_cast<const G*>(a.grad);
  const auto flush = [&] {
    if (cont) {
      store_vec<float, VEC>(a.head + (size_t)chunk * a.dim + col, acc);
    } else {
      const unsigned long long row = a.chunk_rank ? rank : cur;
      if (row < a.capacity) {
        store_result<W, VEC>(a, row, col, acc);
        if (a.chunk_rank && col == 0) a.rows_out[row] = (long long)cur;
      }
    }
  };
  for (unsigned int i = i0; i < i1; i += SEG_UNROLL) {
    unsigned long long w[SEG_UNROLL];
    RowVec<G, VEC> v[SEG_UNROLL];
#pragma unroll
    for (int u = 0; u < SEG_UNROLL; u++) w[u] = i + u < i1 ? a.words[i + u] : ~0ull;
#pragma unroll
    for (int u = 0; u < SEG_UNROLL; u++)
      if ((w[u] >> 32) < a.num_rows)
        v[u] = load_vec<G, VEC>(g + (long long)(unsigned int)w[u] * a.grad_stride + col);
#pragma unroll
    for (int u = 0; u < SEG_UNROLL; u++) {
      const unsigned long long key = w[u] >> 32;
      if (i + u < i1 && key != cur) {
        flush();
        cont = false;
        cur = key;
        rank++;
#pragma unroll
        for (int j = 0; j < VEC; j++) acc[j] = 0.0f;
        if (cur >= a.num_rows) return;
      }
      if (i + u < i1) {
#pragma unroll
        for (int j = 0; j < VEC; j++) acc[j] += to_f32(v[u].v[j]);
      }
    }
  }
  const bool goes_on = i1 < a.n && (a.words[i1] >> 32) == cur;
  if (goes_on && !cont)
    store_vec<float, VEC>(a.tail + (size_t)chunk * a.dim + col, acc);
  else
    flush();  // the run ends here, or fills the chunk between two others
}

// Runs that cross chunks: the team of the chunk where a run starts adds its
// tail and the heads of the chunks it goes on in, in chunk order.
template <typename W, int VEC>
__global__ void __launch_bounds__(SEG_THREADS) join_kernel(SegArgs a) {
  const unsigned long long item = ((unsigned long long)blockIdx.x * SEG_THREADS + threadIdx.x) / a.team;
  const unsigned long long chunk64 = item / a.slabs;
  if (chunk64 + 1 >= a.chunks) return;  // the last chunk's runs end in it
  const unsigned int chunk = (unsigned int)chunk64;
  const unsigned int slab = (unsigned int)(item - chunk64 * a.slabs);
  const long long col = ((long long)slab * a.team + (threadIdx.x & (a.team - 1))) * VEC;
  if (col >= a.dim) return;
  const unsigned int i0 = chunk << a.chunk_shift, i1 = (chunk + 1) << a.chunk_shift;
  const unsigned long long cur = a.words[i1] >> 32;
  if (cur >= a.num_rows || (a.words[i1 - 1] >> 32) != cur) return;
  if ((a.words[i0] >> 32) == cur && i0 > 0 && (a.words[i0 - 1] >> 32) == cur) return;  // began earlier
  float acc[VEC];
  RowVec<float, VEC> v = load_vec<float, VEC>(a.tail + (size_t)chunk * a.dim + col);
#pragma unroll
  for (int j = 0; j < VEC; j++) acc[j] = v.v[j];
  for (unsigned int c = chunk + 1; c < a.chunks && (a.words[(size_t)c << a.chunk_shift] >> 32) == cur; c++) {
    v = load_vec<float, VEC>(a.head + (size_t)c * a.dim + col);
#pragma unroll
    for (int j = 0; j < VEC; j++) acc[j] += v.v[j];
  }
  unsigned long long row = cur;
  if (a.chunk_rank) {  // heads up to and with this run's, less one
    const unsigned int next = a.chunk_rank[chunk + 1];
    row = (unsigned long long)next - 1ull;
  }
  if (row < a.capacity) {
    store_result<W, VEC>(a, row, col, acc);
    if (a.chunk_rank && col == 0) a.rows_out[row] = (long long)cur;
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

// Entries of a chunk: a border costs a partial row written and read, so longer
// chunks for long lists; short ones where there are few words to share out.
unsigned int chunk_shift_of(uint64_t n) { return n >= (1u << 18) ? 6 : 5; }

struct Workspace {
  uint64_t words_a, words_b, counts, tile_heads, count, chunk_rank, head, tail, bytes;
  uint32_t chunks, chunk_shift;
  Workspace(uint64_t n, uint64_t dim) {
    chunk_shift = chunk_shift_of(n);
    chunks = (uint32_t)((n + (1ull << chunk_shift) - 1) >> chunk_shift);
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
    chunk_rank = take(((uint64_t)chunks + 1) * 4);
    head = take((uint64_t)chunks * dim * 4);
    tail = take((uint64_t)chunks * dim * 4);
    bytes = at;
  }
};

// tiles and words per tile of the sort of n words
void sort_shape(uint64_t n, unsigned int* tiles, unsigned int* per) {
  const uint64_t want = std::min<uint64_t>(MAX_TILES, (n + SORT_STEP - 1) / SORT_STEP);
  const uint64_t p = ((n + want - 1) / want + SORT_THREADS - 1) / SORT_THREADS * SORT_THREADS;
  *per = (unsigned int)p;
  *tiles = (unsigned int)((n + p - 1) / p);
}

int passes_of(uint64_t num_rows) {  // the largest key is num_rows
  return std::max(1u, (bit_length(num_rows) + MAX_DIGIT_BITS - 1) / MAX_DIGIT_BITS);
}

// Sorts the ids into the workspace; returns where the sorted words are.
unsigned long long* sort_ids(const IdSource& ids, uint64_t n, char* ws, const Workspace& lay, cudaStream_t st) {
  unsigned int tiles, per;
  sort_shape(n, &tiles, &per);
  const int key_bits = std::max(1u, bit_length(ids.num_rows));
  const int passes = passes_of(ids.num_rows);
  unsigned long long* buf[2] = {reinterpret_cast<unsigned long long*>(ws + lay.words_a),
                                reinterpret_cast<unsigned long long*>(ws + lay.words_b)};
  unsigned int* counts = reinterpret_cast<unsigned int*>(ws + lay.counts);
  IdSource src = ids;
  int done = 0;
  for (int p = 0; p < passes; p++) {
    const int bits = (key_bits - done + (passes - p) - 1) / (passes - p);
    count_kernel<<<tiles, SORT_THREADS, 0, st>>>(src, (unsigned int)n, per, 32 + done, bits, counts);
    scatter_kernel<<<tiles, SORT_THREADS, 0, st>>>(src, (unsigned int)n, per, tiles, 32 + done, bits, counts,
                                                   buf[p & 1]);
    src.id_bytes = 0;
    src.words = buf[p & 1];
    done += bits;
  }
  return buf[(passes - 1) & 1];
}

template <typename G, typename W, int VEC>
void launch_segments(SegArgs a, cudaStream_t st) {
  const uint64_t vecs = (uint64_t)a.dim / VEC;
  a.team = 1;
  while (a.team < 32 && a.team < vecs) a.team <<= 1;
  a.slabs = (unsigned int)((vecs + a.team - 1) / a.team);
  const uint64_t threads = (uint64_t)a.chunks * a.slabs * a.team;
  const uint64_t blocks = (threads + SEG_THREADS - 1) / SEG_THREADS;
  GIDS_CHECK(blocks < (1ull << 31), GIDS_E_UNSUPPORTED, "too many rows x columns for one launch");
  segment_kernel<G, W, VEC><<<(unsigned int)blocks, SEG_THREADS, 0, st>>>(a);
  if (a.chunks > 1) join_kernel<W, VEC><<<(unsigned int)blocks, SEG_THREADS, 0, st>>>(a);
  GIDS_CUDA(cudaGetLastError());
}

template <typename G, typename W>
void launch_segments_vec(const SegArgs& a, const Rows& out, const Rows& grad, cudaStream_t st) {
  constexpr int BIG = 16 / (int)sizeof(G);  // a 16-byte vector of the gradient
  if (vec_ok(out, a.dim, BIG) && vec_ok(grad, a.dim, BIG))
    launch_segments<G, W, BIG>(a, st);
  else if (vec_ok(out, a.dim, 2) && vec_ok(grad, a.dim, 2))
    launch_segments<G, W, 2>(a, st);
  else
    launch_segments<G, W, 1>(a, st);
}

void segments(const SegArgs& a, const Rows& out, const Rows& grad, cudaStream_t st) {
  if (out.type == GIDS_F32) {
    if (grad.type == GIDS_F32) return launch_segments_vec<float, float>(a, out, grad, st);
    if (grad.type == GIDS_F16) return launch_segments_vec<__half, float>(a, out, grad, st);
    return launch_segments_vec<__nv_bfloat16, float>(a, out, grad, st);
  }
  if (out.type == GIDS_F16) return launch_segments_vec<__half, __half>(a, out, grad, st);
  return launch_segments_vec<__nv_bfloat16, __nv_bfloat16>(a, out, grad, st);
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
  if (vec_ok(out, dim, BIG) && vec_ok(weight, dim, BIG))
    launch_embedding<W, O, BIG>(a, n, dim, id_bytes, st);
  else if (vec_ok(out, dim, 2) && vec_ok(weight, dim, 2))
    launch_embedding<W, O, 2>(a, n, dim, id_bytes, st);
  else
    launch_embedding<W, O, 1>(a, n, dim, id_bytes, st);
}

IdSource id_source(const void* ids, int id_bytes, int64_t num_rows, int64_t padding_idx, int* err) {
  IdSource s{};
  s.ids = ids;
  s.id_bytes = id_bytes;
  s.num_rows = (unsigned long long)num_rows;
  s.padding = padding_idx;
  s.err = err;
  return s;
}

void check_workspace(const void* ws, uint64_t ws_bytes, const Workspace& lay) {
  GIDS_CHECK(ws && ((uintptr_t)ws) % 256 == 0, GIDS_E_INVAL, "workspace is null or not aligned to 256 bytes");
  GIDS_CHECK(ws_bytes >= lay.bytes, GIDS_E_INVAL,
             "workspace too small: " + std::to_string(lay.bytes) + " bytes are needed");
}

}  // namespace

int* id_error_word(int device) {
  std::lock_guard<std::mutex> lk(g_err_mu);
  if (!g_err_dev[device]) {
    // allocation is allowed while the calling thread captures a stream: the
    // word is not part of the graph
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    GIDS_CUDA(cudaThreadExchangeStreamCaptureMode(&mode));
    int* h = nullptr;
    cudaError_t e = cudaHostAlloc(&h, sizeof(int), cudaHostAllocMapped | cudaHostAllocPortable);
    cudaThreadExchangeStreamCaptureMode(&mode);
    GIDS_CUDA(e);
    *h = 0;
    int* d = nullptr;
    GIDS_CUDA(cudaHostGetDevicePointer(&d, h, 0));
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
  if (n) check_workspace(ws, ws_bytes, lay);
  check_id_errors(device);
  if (num_rows == 0 && n == 0) return;
  DeviceGuard dg(device);
  const size_t eb = (size_t)type_bytes(dweight.type);
  if (num_rows > 0)
    GIDS_CUDA(cudaMemset2DAsync(dweight.p, (num_rows > 1 ? (size_t)dweight.stride : (size_t)dim) * eb, 0,
                                (size_t)dim * eb, (size_t)num_rows, st));
  if (n == 0) return;
  char* base = static_cast<char*>(ws);
  SegArgs a{};
  a.words = sort_ids(id_source(ids, id_bytes, num_rows, padding_idx, id_error_word(device)), (uint64_t)n, base, lay, st);
  a.out = dweight.p;
  a.grad = grad.p;
  a.head = reinterpret_cast<float*>(base + lay.head);
  a.tail = reinterpret_cast<float*>(base + lay.tail);
  a.out_stride = dweight.stride;
  a.grad_stride = grad.stride;
  a.num_rows = a.capacity = (unsigned long long)num_rows;
  a.dim = dim;
  a.n = (unsigned int)n;
  a.chunks = lay.chunks;
  a.chunk_shift = lay.chunk_shift;
  a.scale = scale;
  segments(a, dweight, grad, st);
}

void embedding_group(int device, const void* ids, int id_bytes, int64_t n, int64_t num_rows, int64_t padding_idx,
                     int64_t dim, void* ws, uint64_t ws_bytes, uint64_t* count_dev, uint64_t* count_host,
                     cudaStream_t st) {
  check_device(device);
  check_ids(ids, id_bytes, n, num_rows, dim);
  GIDS_CHECK(padding_idx >= -1 && padding_idx < std::max<int64_t>(num_rows, 1), GIDS_E_INVAL,
             "padding_idx must be -1 (none) or a row");
  const Workspace lay((uint64_t)n, (uint64_t)dim);
  check_workspace(ws, ws_bytes, lay);
  check_id_errors(device);
  DeviceGuard dg(device);
  if (count_host) {
    cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
    GIDS_CUDA(cudaStreamIsCapturing(st, &cap));
    GIDS_CHECK(cap == cudaStreamCaptureStatusNone, GIDS_E_STATE,
               "count_host waits for the stream, which is being captured into a graph");
  }
  char* base = static_cast<char*>(ws);
  unsigned long long* count = reinterpret_cast<unsigned long long*>(base + lay.count);
  if (n == 0) {
    GIDS_CUDA(cudaMemsetAsync(count, 0, sizeof(*count), st));
  } else {
    const unsigned long long* w =
        sort_ids(id_source(ids, id_bytes, num_rows, padding_idx, id_error_word(device)), (uint64_t)n, base, lay, st);
    unsigned int tiles, per;
    sort_shape((uint64_t)n, &tiles, &per);
    unsigned int* th = reinterpret_cast<unsigned int*>(base + lay.tile_heads);
    head_count_kernel<<<tiles, SORT_THREADS, 0, st>>>(w, (unsigned int)n, per, (unsigned long long)num_rows, th);
    head_rank_kernel<<<tiles, SORT_THREADS, 0, st>>>(
        w, (unsigned int)n, per, tiles, (unsigned long long)num_rows, lay.chunk_shift, th,
        reinterpret_cast<unsigned int*>(base + lay.chunk_rank), count);
    GIDS_CUDA(cudaGetLastError());
  }
  if (count_dev) GIDS_CUDA(cudaMemcpyAsync(count_dev, count, sizeof(*count), cudaMemcpyDeviceToDevice, st));
  if (count_host) {
    unsigned long long c = 0;
    GIDS_CUDA(cudaMemcpyAsync(&c, count, sizeof(c), cudaMemcpyDeviceToHost, st));
    GIDS_CUDA(cudaStreamSynchronize(st));
    *count_host = c;
  }
}

void embedding_grad_rows(int device, int64_t* rows, Rows values, int64_t capacity, int64_t num_rows, int64_t dim,
                         Rows grad, int64_t n, float scale, void* ws, uint64_t ws_bytes, cudaStream_t st) {
  check_device(device);
  check_ids(reinterpret_cast<const void*>(256), 8, n, num_rows, dim);
  GIDS_CHECK(capacity >= 0, GIDS_E_INVAL, "capacity must be >= 0");
  GIDS_CHECK(capacity == 0 || rows, GIDS_E_INVAL, "rows is null");
  GIDS_CHECK(((uintptr_t)rows) % 8 == 0, GIDS_E_INVAL, "rows: address not aligned to its elements");
  check_rows(values, "values", capacity, dim, true);
  check_rows(grad, "grad", n, dim, false);
  GIDS_CHECK(values.type == grad.type || values.type == GIDS_F32, GIDS_E_UNSUPPORTED,
             "values must have the gradient's type or be float32");
  const Workspace lay((uint64_t)n, (uint64_t)dim);
  check_workspace(ws, ws_bytes, lay);
  if (n == 0 || capacity == 0) return;
  DeviceGuard dg(device);
  char* base = static_cast<char*>(ws);
  const int passes = passes_of((uint64_t)num_rows);
  SegArgs a{};
  a.words = reinterpret_cast<const unsigned long long*>(base + ((passes - 1) & 1 ? lay.words_b : lay.words_a));
  a.chunk_rank = reinterpret_cast<const unsigned int*>(base + lay.chunk_rank);
  a.rows_out = reinterpret_cast<long long*>(rows);
  a.out = values.p;
  a.grad = grad.p;
  a.head = reinterpret_cast<float*>(base + lay.head);
  a.tail = reinterpret_cast<float*>(base + lay.tail);
  a.out_stride = values.stride;
  a.grad_stride = grad.stride;
  a.num_rows = (unsigned long long)num_rows;
  a.capacity = (unsigned long long)capacity;
  a.dim = dim;
  a.n = (unsigned int)n;
  a.chunks = lay.chunks;
  a.chunk_shift = lay.chunk_shift;
  a.scale = scale;
  segments(a, values, grad, st);
}

void embedding_check(int device, cudaStream_t st) {
  check_device(device);
  DeviceGuard dg(device);
  GIDS_CUDA(cudaStreamSynchronize(st));
  check_id_errors(device);
}

}  // namespace gids
