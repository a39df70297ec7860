// Layer norm and its gradient, for sm_100a.
//
// Forward: m = mean(x), v = mean((x - m)^2), r = 1 / sqrt(v + eps),
// y = round((x - m) r w + b). A group of threads holds a row in registers, so
// x is read once and the variance is the sum of squared differences from the
// mean, not a difference of sums.
//
// Backward, with xh = (x - m) r and t = g w:
//   dx = round(r (t - mean(t) - xh mean(t xh))), dw = sum g xh, db = sum g.
// The threads of a group keep the sums of their columns in float32 registers
// while the group walks over rows; every block leaves one partial row of dw and
// of db in the workspace, and a second kernel adds them in block order. No
// atomics: results repeat bit for bit.
//
// Both are bound by HBM (4 to 12 bytes an element, 10 to 20 float32
// operations). What it takes to stay there: rows in flight (about 128 KB an SM,
// in shared memory rather than registers, by asynchronous copies), few
// instructions an element (packed float32 arithmetic, parameters in registers
// for the life of a block), and few shuffles and barriers (R rows are reduced
// together).
#include <algorithm>

#include "layers.hpp"
#include "rows.cuh"

namespace gids {
namespace {

constexpr int LN_THREADS = 512;       // threads of a block, and of the largest group
constexpr int LN_LONG_THREADS = 512;  // rows that do not fit the registers of a group

// What the walk over the rows needs, in the kernel's parameters (constant memory
// rather than registers).
struct RowWalk {
  long long n;       // rows
  long long total;   // groups of the launch
  const char* safe;  // an aligned address for copies of nothing
  int dim;
};

struct LnArgs {
  RowWalk walk;
  void* y;
  const void* x;
  float* mean;
  float* rstd;
  const void* w;
  const void* b;
  long long y_stride, x_stride, n;
  long long y_jump, x_jump;  // bytes from a row of a group to its next
  int dim, w_type;
  float eps, inv_dim;
};

struct LnGradArgs {
  RowWalk walk;
  void* dx;
  const void* g;
  const void* x;
  const float* mean;
  const float* rstd;
  const void* w;
  float* part;  // [blocks][2][dim], or null: no weight gradient, or one cluster's
  void *dw, *db;
  long long dx_stride, g_stride, x_stride, n;
  long long dx_jump, g_jump, x_jump;  // bytes from a row of a group to its next
  int dim, w_type;
  float inv_dim;
};

template <typename P, int VEC>
__device__ __forceinline__ void load_param_of(const void* p, long long i, float (&f)[VEC]) {
  const RowVec<P, VEC> v = load_vec<P, VEC>(reinterpret_cast<const P*>(p) + i);
#pragma unroll
  for (int j = 0; j < VEC; j++) f[j] = to_f32(v.v[j]);
}
// VEC elements of weight or bias (type code `type`), or `fill` where there is none
template <int VEC>
__device__ __forceinline__ void load_param(const void* p, int type, long long i, float fill, float (&f)[VEC]) {
  if (p) {
    if (type == GIDS_F32)
      load_param_of<float, VEC>(p, i, f);
    else if (type == GIDS_F16)
      load_param_of<__half, VEC>(p, i, f);
    else
      load_param_of<__nv_bfloat16, VEC>(p, i, f);
  } else {
#pragma unroll
    for (int j = 0; j < VEC; j++) f[j] = fill;
  }
}

__device__ __forceinline__ void store_param(void* p, int type, long long i, float v) {
  if (type == GIDS_F32)
    static_cast<float*>(p)[i] = v;
  else if (type == GIDS_F16)
    static_cast<__half*>(p)[i] = from_f32<__half>(v);
  else
    static_cast<__nv_bfloat16*>(p)[i] = from_f32<__nv_bfloat16>(v);
}

// ------------------------------------------------------------- rows of a group
// Sums N values (a power of two) over `width` >= N lanes (a power of two) in
// N - 1 + log2(width / N) shuffles instead of N log2(width): every step halves
// the values that a lane still adds up. Lane l ends with the sum of value
// (l % width) / (width / N).
template <int N>
__device__ __forceinline__ float lane_sums(float (&v)[N], int lane, int width) {
  int o = width >> 1;
#pragma unroll
  for (int n = N; n > 1; n >>= 1, o >>= 1) {
    const bool hi = (lane & o) != 0;
#pragma unroll
    for (int i = 0; i < n / 2; i++) {
      const float send = hi ? v[i] : v[i + n / 2], keep = hi ? v[i + n / 2] : v[i];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, send, o);
    }
  }
  for (; o; o >>= 1) v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
  return v[0];
}

// Sums of N values over the threads of the caller's group, to every thread.
// Groups of a warp or less use shuffles. Larger ones exchange their warps'
// sums in shared memory and add them in warp order; `red` holds two buffers,
// used in turn, so one barrier is enough. The barrier is the group's own:
// groups of a block do not wait for one another.
__device__ __forceinline__ void group_barrier(int group) {
  asm volatile("bar.sync %0, %1;" ::"r"(threadIdx.y + 1), "r"(group) : "memory");
}
template <int N, int WARPS, int WIDTH>
__device__ __forceinline__ void group_sums(float (&s)[N], int group, int lane, int warp, float4 (&red)[2][WARPS][WIDTH],
                                           int& turn) {
  static_assert(N <= 4 * WIDTH, "the exchange buffer holds N values a warp");
  if (group < N) {
#pragma unroll
    for (int o = N / 2; o; o >>= 1)
      if (o < group) {
#pragma unroll
        for (int i = 0; i < N; i++) s[i] += __shfl_xor_sync(0xffffffffu, s[i], o);
      }
  } else if (group <= 32) {
    const float v = lane_sums<N>(s, lane, group);
    if (N == 1) return;  // every lane has it
    const int first = lane & ~(group - 1);
#pragma unroll
    for (int i = 0; i < N; i++) s[i] = __shfl_sync(0xffffffffu, v, first + i * (group / N));
  } else {
    const float v = lane_sums<N>(s, lane, 32);
    if (lane % (32 / N) == 0) reinterpret_cast<float*>(red[turn][warp])[lane / (32 / N)] = v;
    group_barrier(group);
    const int warps = group >> 5, warp0 = (threadIdx.y * group) >> 5;
#pragma unroll
    for (int i = 0; i < N; i++) s[i] = 0.0f;
    for (int k = 0; k < warps; k++) {
      float4 part[(N + 3) / 4];
#pragma unroll
      for (int i = 0; i < (N + 3) / 4; i++) part[i] = red[turn][warp0 + k][i];
#pragma unroll
      for (int i = 0; i < N; i++) s[i] += reinterpret_cast<const float*>(part)[i];
    }
    turn ^= 1;
  }
}

// A group's walk over the rows. Global group g of G takes the rows g, g + G,
// g + 2 G, ..., R at a time. A thread has K vectors of VEC elements of a row.
//
// VEC > 1: 16-byte vectors of memory. Rows need not start on one: the vectors
// of a row begin at the 16-byte boundary before it, `lead` elements early, and
// the elements of the first and last vector that are not the row's are set to
// zero (they lie inside the aligned 16 bytes of the row's first or last element,
// so reading them stays inside its allocation). G is a multiple of the period with
// which rows meet the boundary again, so `lead` is the same for all rows of a
// group and a thread keeps its columns: rows of any width and stride move in
// full vectors, if all matrices of the call meet the boundary alike.
// VEC = 1: where they do not. The group copies rows by the pieces of 16 bytes that
// cover them and reads elements after a barrier.
//
// Rows arrive through a ring in shared memory by asynchronous copies, STAGES - 1
// iterations ahead of their use. With VEC > 1 a thread copies its own vectors to
// slots that only it reads, so there is no barrier.
// MODE: how a thread's vectors lie to the row. FULL_ROWS: all K are the row's;
// WHOLE_VECS: each is, or has no column of it (aligned rows); EDGES: any.
constexpr int EDGES = 0, WHOLE_VECS = 1, FULL_ROWS = 2;
template <typename X, int VEC, int K, int R, int A, int STAGES, int MODE, int THREADS, int GROUP>
struct RowRing {
  static constexpr bool STAGED = VEC == 1;
  const RowWalk& walk;
  char* mem;  // this group's part (STAGED), or this thread's first slot
  int t, group, lead = 0;  // group: threads of a group (GROUP, if that is not 0)
  int rows, steps;  // rows of this group, and of the block's first group, which has the most
  int ahead = 0, stage = 0;
  // EDGES, where registers allow it: the bits of each vector that are the row's,
  // by 32-bit words. Gradient of 300,000 x 1001 bf16: 468 us by comparisons for
  // every element, 385 us with masks; the forward pass, which holds more, spills with
  // them (237 and 296 us).
  static constexpr bool MASKED = MODE == EDGES && !STAGED && A == 2 && K <= 2;
  unsigned int mask[MASKED ? K : 1][4];

  __host__ __device__ static int pitch(int dim) { return (dim * (int)sizeof(X) + 31) / 16 * 16; }
  __host__ __device__ static size_t bytes(int groups, int dim) {
    if (STAGED) return (size_t)groups * STAGES * R * A * pitch(dim);
    return (size_t)STAGES * R * K * A * 16 * THREADS;
  }
  __device__ RowRing(void* dyn, const RowWalk& w, const void* x, long long stride)
      : walk(w), t(threadIdx.x), group(GROUP ? GROUP : blockDim.x) {
    const long long first = this->first(), block = (long long)blockIdx.x * blockDim.y;
    rows = first < w.n ? (int)((w.n - first + w.total - 1) / w.total) : 0;
    steps = block < w.n ? (int)((w.n - block + w.total - 1) / w.total) : 0;
    if constexpr (!STAGED && MODE == EDGES)
      lead = (int)((reinterpret_cast<uintptr_t>(x) + first * stride * sizeof(X)) & 15) / (int)sizeof(X);
    if constexpr (STAGED)
      mem = static_cast<char*>(dyn) + (size_t)threadIdx.y * STAGES * R * A * pitch(w.dim);
    else
      mem = static_cast<char*>(dyn) + (threadIdx.y * group + t) * 16;
    if constexpr (MASKED) {
#pragma unroll
      for (int k = 0; k < K; k++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          constexpr int PER = 4 / (int)sizeof(X);  // elements of a word
          unsigned int m = 0;
#pragma unroll
          for (int j = 0; j < PER; j++)
            if (col(k) + i * PER + j >= 0 && col(k) + i * PER + j < w.dim)
              m |= (PER == 1 ? 0xffffffffu : 0xffffu) << (16 * j);
          mask[k][i] = m;
        }
    }
  }
  // this group's first row
  __device__ __forceinline__ long long first() const { return (long long)blockIdx.x * blockDim.y + threadIdx.y; }
  // first column of vector k; the columns that a thread has of it are in [0, dim)
  __device__ __forceinline__ int col(int k) const { return (k * group + t) * VEC - lead; }
  // whether vector k has elements that are not the row's
  __device__ __forceinline__ bool partial(int k) const {
    return MODE == EDGES && (col(k) < 0 || col(k) + VEC > walk.dim);
  }
  // whether element j of vector k is the row's (EDGES)
  __device__ __forceinline__ bool valid(int k, int j) const {
    if constexpr (MASKED) return sizeof(X) == 4 ? mask[k][j & 3] != 0 : (mask[k][(j / 2) & 3] >> (16 * (j & 1))) & 1u;
    return col(k) + j >= 0 && col(k) + j < walk.dim;
  }
  // whether vector k has none that are
  __device__ __forceinline__ bool absent(int k) const { return MODE != FULL_ROWS && col(k) >= walk.dim; }
  // where this thread starts in a matrix: its first column (STAGED: the row) of the group's first row
  __device__ __forceinline__ char* start(const void* p, long long stride) const {
    return reinterpret_cast<char*>(const_cast<void*>(p)) +
           (first() * stride + (STAGED ? 0 : col(0))) * (long long)sizeof(X);
  }

  __device__ __forceinline__ char* slot(int s, int r, int k, int which) const {
    if constexpr (STAGED) return mem + ((s * R + r) * A + which) * pitch(walk.dim);
    return mem + s * (R * K * A * THREADS * 16) + ((r * K + k) * A + which) * (THREADS * 16);
  }
  // row r of the stage `ahead` from `src` (start() and jumps); nothing is read where `on` is false
  __device__ __forceinline__ void fetch(int r, int which, const char* src, bool on) const {
    if constexpr (STAGED) {
      if (!on) return;  // take() does not read it
      const int early = (int)(reinterpret_cast<uintptr_t>(src) & 15);
      const int span = early + walk.dim * (int)sizeof(X);
      char* dst = slot(ahead, r, 0, which);
      for (int i = t * 16; i < span; i += group * 16) copy_async_tail(dst + i, src - early + i, min(16, span - i));
    } else {
#pragma unroll
      for (int k = 0; k < K; k++) {
        const bool in = on && !absent(k);
        copy_async(slot(ahead, r, k, which), in ? src + k * group * 16 : walk.safe, in);
      }
    }
  }
  __device__ __forceinline__ void fetched() {
    copies_commit();
    ahead = ahead + 1 == STAGES ? 0 : ahead + 1;
  }
  __device__ __forceinline__ void sync() const {
    if constexpr (STAGED) {
      if (group > 32)
        group_barrier(group);
      else
        __syncwarp();
    }
  }
  // this thread's elements of row r of the stage in use, the group's m-th row
  // (zeros for elements that are not the row's)
  __device__ __forceinline__ void take(int r, int which, const void* p, long long stride, int m, RowVec<X, VEC> (&v)[K]) const {
    if constexpr (STAGED) {
      const unsigned int row = (unsigned int)first() + (unsigned int)m * (unsigned int)walk.total;
      const int early = (int)(((unsigned int)reinterpret_cast<uintptr_t>(p) +
                               row * (unsigned int)stride * (unsigned int)sizeof(X)) & 15);
#pragma unroll
      for (int k = 0; k < K; k++)
        v[k].v[0] = m < rows && !partial(k) ? *reinterpret_cast<const X*>(slot(stage, r, 0, which) + early +
                                                                          col(k) * (int)sizeof(X))
                                            : from_f32<X>(0.0f);
    } else {
#pragma unroll
      for (int k = 0; k < K; k++) {
        v[k] = *reinterpret_cast<const RowVec<X, VEC>*>(slot(stage, r, k, which));
        if constexpr (MASKED) {
#pragma unroll
          for (int i = 0; i < 4; i++) reinterpret_cast<unsigned int*>(&v[k])[i] &= mask[k][i];
        } else if (partial(k)) {
#pragma unroll
          for (int j = 0; j < VEC; j++)
            if (!valid(k, j)) v[k].v[j] = from_f32<X>(0.0f);
        }
      }
    }
  }
  __device__ __forceinline__ void taken() { stage = stage + 1 == STAGES ? 0 : stage + 1; }
  // weight or bias of this thread's columns, in pairs
  __device__ __forceinline__ void params(const void* p, int type, float fill, F2 (&out)[VEC * K / 2]) const {
    float f[K][VEC];
#pragma unroll
    for (int k = 0; k < K; k++) {
      if (MODE != EDGES) {
        load_param<VEC>(absent(k) ? nullptr : p, type, col(k), fill, f[k]);
      } else {
#pragma unroll
        for (int j = 0; j < VEC; j++) {
          float one[1];
          const int c = col(k) + j;
          load_param<1>(c >= 0 && c < walk.dim ? p : nullptr, type, c, fill, one);
          f[k][j] = one[0];
        }
      }
    }
#pragma unroll
    for (int i = 0; i < VEC * K / 2; i++)
      out[i] = F2(f[2 * i / VEC][2 * i % VEC], f[(2 * i + 1) / VEC][(2 * i + 1) % VEC]);
  }
  // vector k of a row of the result (`dst`: start() and jumps)
  __device__ __forceinline__ void store(char* dst, int k, const float (&f)[VEC]) const {
    X* p = reinterpret_cast<X*>(dst) + (STAGED ? col(k) : k * group * VEC);
    if (MODE != EDGES) {
      if (!absent(k)) store_vec<X, VEC>(p, f);
    } else if (!partial(k)) {
      store_vec<X, VEC>(p, f);
    } else if constexpr (!STAGED) {
#pragma unroll
      for (int j = 0; j < VEC; j++)
        if (valid(k, j)) p[j] = from_f32<X>(f[j]);
    }
  }
};

// ------------------------------------------------------------------- forward
// The rounded mean is off by up to half a step of the mean, which is not small
// beside the differences when the mean is large against them. `off` is the
// mean of the differences from it: the second pass takes it out again.
// (Not fmaxf, which would turn the NaN of a row with NaN or infinities into 0.)
__device__ __forceinline__ float variance(float mean_sq, float off) {
  const float v = mean_sq - off * off;
  return v < 0.0f ? 0.0f : v;
}

// blockDim = (threads of a group, groups).
template <typename X, int VEC, int K, int R, int STAGES, int MODE, int THREADS, int GROUP>
__global__ void __launch_bounds__(THREADS) ln_kernel(LnArgs a) {
  extern __shared__ uint4 dyn[];
  constexpr int N = 2 * R, P = VEC * K / 2;
  __shared__ float4 red[2][THREADS / 32][(N + 3) / 4];
  const int group = GROUP ? GROUP : blockDim.x;
  const int lin = threadIdx.y * group + threadIdx.x, lane = lin & 31, warp = lin >> 5;
  int turn = 0;
  RowRing<X, VEC, K, R, 1, STAGES, MODE, THREADS, GROUP> ring(dyn, a.walk, a.x, a.x_stride);
  const char* xp = ring.start(a.x, a.x_stride);
  char* yp = ring.start(a.y, a.y_stride);
  const auto fetch = [&](int m) {
#pragma unroll
    for (int r = 0; r < R; r++) ring.fetch(r, 0, xp + (m + r) * a.x_jump, m + r < ring.rows);
    ring.fetched();
  };
#pragma unroll
  for (int i = 0; i < STAGES - 1; i++) fetch(i * R);
  F2 w[P], b[P];
  ring.params(a.w, a.w_type, 1.0f, w);
  ring.params(a.b, a.w_type, 0.0f, b);
  for (int m = 0; m < ring.steps; m += R) {
    fetch(m + (STAGES - 1) * R);
    copies_wait<STAGES - 1>();
    ring.sync();
    F2 f[R][P];
    float s[R];
#pragma unroll
    for (int r = 0; r < R; r++) {
      RowVec<X, VEC> v[K];
      ring.take(r, 0, a.x, a.x_stride, m + r, v);
      F2 sum(0.0f);
#pragma unroll
      for (int p = 0; p < P; p++) {
        f[r][p] = pair_of(v, p);
        sum = add2(sum, f[r][p]);
      }
      s[r] = sum.lo() + sum.hi();
    }
    ring.taken();
    group_sums(s, group, lane, warp, red, turn);
    float mean[R], d[N];  // d: sums of x - mean and of its square
#pragma unroll
    for (int r = 0; r < R; r++) {
      mean[r] = s[r] * a.inv_dim;
      const F2 m(-mean[r]);
      F2 d0(0.0f), d1(0.0f);
#pragma unroll
      for (int p = 0; p < P; p++) f[r][p] = add2(f[r][p], m);
      // elements that are not the row's stay zero
      if constexpr (VEC == 1) {
#pragma unroll
        for (int p = 0; p < P; p++)
          f[r][p] = F2(ring.partial(2 * p) ? 0.0f : f[r][p].lo(), ring.partial(2 * p + 1) ? 0.0f : f[r][p].hi());
      } else if constexpr (MODE != FULL_ROWS) {
#pragma unroll
        for (int k = 0; k < K; k++) {
          if (ring.absent(k)) {
#pragma unroll
            for (int j = 0; j < VEC; j += 2) f[r][(k * VEC + j) / 2] = F2(0.0f);
          } else if (ring.partial(k)) {
#pragma unroll
            for (int j = 0; j < VEC; j += 2) {
              F2& c = f[r][(k * VEC + j) / 2];
              c = F2(ring.valid(k, j) ? c.lo() : 0.0f, ring.valid(k, j + 1) ? c.hi() : 0.0f);
            }
          }
        }
      }
#pragma unroll
      for (int p = 0; p < P; p++) {
        d0 = add2(d0, f[r][p]);
        d1 = fma2(f[r][p], f[r][p], d1);
      }
      d[2 * r] = d0.lo() + d0.hi();
      d[2 * r + 1] = d1.lo() + d1.hi();
    }
    group_sums(d, group, lane, warp, red, turn);
#pragma unroll
    for (int r = 0; r < R; r++) {
      if (m + r >= ring.rows) continue;
      const float off = d[2 * r] * a.inv_dim;
      const float rstd = rsqrtf(variance(d[2 * r + 1] * a.inv_dim, off) + a.eps);
      if (threadIdx.x == 0 && a.mean) {
        const long long i = ring.first() + (m + r) * a.walk.total;
        a.mean[i] = mean[r] + off;
        a.rstd[i] = rstd;
      }
      const F2 q(rstd), o(-off * rstd);
#pragma unroll
      for (int k = 0; k < K; k++) {
        float out[VEC];
#pragma unroll
        for (int j = 0; j < VEC; j++) {
          const int p = (k * VEC + j) / 2;
          const F2 h = fma2(fma2(f[r][p], q, o), w[p], b[p]);
          out[j] = (k * VEC + j) & 1 ? h.hi() : h.lo();
        }
        ring.store(yp + (m + r) * a.y_jump, k, out);
      }
    }
  }
  copies_wait<0>();
}

// Sums over a block of LN_LONG_THREADS threads, in warp order. `red` holds two
// buffers of 2 x 32 floats, used in turn, so one barrier is enough.
template <int N>
__device__ __forceinline__ void block_sum(float (&v)[N], float* red, int& turn) {
#pragma unroll
  for (int o = 16; o; o >>= 1) {
#pragma unroll
    for (int i = 0; i < N; i++) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  }
  float* buf = red + turn * 64;
  turn ^= 1;
  if ((threadIdx.x & 31) == 0) {
#pragma unroll
    for (int i = 0; i < N; i++) buf[i * 32 + (threadIdx.x >> 5)] = v[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; i++) {
    float s = 0.0f;
    for (int k = 0; k < LN_LONG_THREADS / 32; k++) s += buf[i * 32 + k];
    v[i] = s;
  }
}

// Rows longer than a group's registers: the row is read three times, the
// second and third time from L2.
template <typename X, int VEC>
__global__ void __launch_bounds__(LN_LONG_THREADS) ln_long_kernel(LnArgs a) {
  __shared__ float red[2 * 32 * 2];
  int turn = 0;
  for (long long row = blockIdx.x; row < a.n; row += gridDim.x) {
    const X* x = reinterpret_cast<const X*>(a.x) + row * a.x_stride;
    float s[1] = {0.0f};
    for (int q = threadIdx.x; q < a.dim / VEC; q += LN_LONG_THREADS) {
      const RowVec<X, VEC> v = load_row<X, VEC>(x + (long long)q * VEC);
#pragma unroll
      for (int j = 0; j < VEC; j++) s[0] += to_f32(v.v[j]);
    }
    block_sum(s, red, turn);
    const float mean = s[0] * a.inv_dim;
    float d[2] = {0.0f, 0.0f};
    for (int q = threadIdx.x; q < a.dim / VEC; q += LN_LONG_THREADS) {
      const RowVec<X, VEC> v = load_row<X, VEC>(x + (long long)q * VEC);
#pragma unroll
      for (int j = 0; j < VEC; j++) {
        const float c = to_f32(v.v[j]) - mean;
        d[0] += c;
        d[1] += c * c;
      }
    }
    block_sum(d, red, turn);
    const float off = d[0] * a.inv_dim;
    const float rstd = rsqrtf(variance(d[1] * a.inv_dim, off) + a.eps);
    if (threadIdx.x == 0 && a.mean) {
      a.mean[row] = mean + off;
      a.rstd[row] = rstd;
    }
    X* y = reinterpret_cast<X*>(a.y) + row * a.y_stride;
    for (int q = threadIdx.x; q < a.dim / VEC; q += LN_LONG_THREADS) {
      const RowVec<X, VEC> v = load_row<X, VEC>(x + (long long)q * VEC);
      float w[VEC], b[VEC];
      load_param<VEC>(a.w, a.w_type, (long long)q * VEC, 1.0f, w);
      load_param<VEC>(a.b, a.w_type, (long long)q * VEC, 0.0f, b);
#pragma unroll
      for (int j = 0; j < VEC; j++) w[j] = (to_f32(v.v[j]) - mean - off) * rstd * w[j] + b[j];
      store_vec<X, VEC>(y + (long long)q * VEC, w);
    }
  }
}

// ------------------------------------------------------------------ backward
// The rows of a block's groups, with dx, and the block's partial dw and db, laid
// out as in the forward pass.
// SMALL: the blocks are one cluster, which adds up dw and db itself.
template <typename X, int VEC, int K, int R, int STAGES, int MODE, int THREADS, int GROUP, bool SMALL>
__global__ void __launch_bounds__(THREADS) ln_grad_kernel(LnGradArgs a) {
  extern __shared__ uint4 dyn[];
  constexpr int N = 2 * R, P = VEC * K / 2;
  __shared__ float4 red[2][THREADS / 32][(N + 3) / 4];
  const int group = GROUP ? GROUP : blockDim.x, groups = blockDim.y;
  const int lin = threadIdx.y * group + threadIdx.x, lane = lin & 31, warp = lin >> 5;
  int turn = 0;
  RowRing<X, VEC, K, R, 2, STAGES, MODE, THREADS, GROUP> ring(dyn, a.walk, a.x, a.x_stride);
  const char* xp = ring.start(a.x, a.x_stride);
  const char* gp = ring.start(a.g, a.g_stride);
  char* dp = ring.start(a.dx, a.dx_stride);
  const auto fetch = [&](int m) {
#pragma unroll
    for (int r = 0; r < R; r++) {
      ring.fetch(r, 0, xp + (m + r) * a.x_jump, m + r < ring.rows);
      ring.fetch(r, 1, gp + (m + r) * a.g_jump, m + r < ring.rows);
    }
    ring.fetched();
  };
  float mean[R], rstd[R];
  const auto load_stats = [&](int m) {
#pragma unroll
    for (int r = 0; r < R; r++) {
      const long long i = ring.first() + (m + r) * a.walk.total;
      mean[r] = m + r < ring.rows ? __ldg(a.mean + i) : 0.0f;
      rstd[r] = m + r < ring.rows ? __ldg(a.rstd + i) : 0.0f;
    }
  };
#pragma unroll
  for (int i = 0; i < STAGES - 1; i++) fetch(i * R);
  load_stats(0);
  F2 w[P], dw[P], db[P];
  ring.params(a.w, a.w_type, 1.0f, w);
#pragma unroll
  for (int p = 0; p < P; p++) dw[p] = db[p] = F2(0.0f);
  for (int m = 0; m < ring.steps; m += R) {
    fetch(m + (STAGES - 1) * R);
    copies_wait<STAGES - 1>();
    ring.sync();
    F2 xh[R][P], tw[VEC == 1 ? R : 1][P];
    float s[N];  // sums of t and of t * xh, for each of the rows
    float rs[R];
#pragma unroll
    for (int r = 0; r < R; r++) {
      RowVec<X, VEC> vx[K], vg[K];
      ring.take(r, 0, a.x, a.x_stride, m + r, vx);
      ring.take(r, 1, a.g, a.g_stride, m + r, vg);
      const F2 m(-mean[r]), q(rstd[r]);
      F2 s0(0.0f), s1(0.0f);
#pragma unroll
      for (int p = 0; p < P; p++) {  // elements that are not the row's have g = 0: they add nothing
        const F2 g = pair_of(vg, p);
        xh[r][p] = mul2(add2(pair_of(vx, p), m), q);
        const F2 t = mul2(g, w[p]);
        dw[p] = fma2(g, xh[r][p], dw[p]);
        db[p] = add2(db[p], g);
        s0 = add2(s0, t);
        s1 = fma2(t, xh[r][p], s1);
        if (VEC == 1) tw[r][p] = t;
      }
      s[2 * r] = s0.lo() + s0.hi();
      s[2 * r + 1] = s1.lo() + s1.hi();
      rs[r] = rstd[r];
    }
    load_stats(m + R);
    if (!a.dx) {
      ring.taken();
      ring.sync();  // the slots are free for the next rows (the sums' barrier does this else)
      continue;
    }
    group_sums(s, group, lane, warp, red, turn);
#pragma unroll
    for (int r = 0; r < R; r++) {
      if (m + r >= ring.rows) continue;
      // dx = r t - r mean(t) - xh r mean(t xh)
      const F2 q(rs[r]), c0(-rs[r] * (s[2 * r] * a.inv_dim)), c1(-rs[r] * (s[2 * r + 1] * a.inv_dim));
      RowVec<X, VEC> vg[K];
      if constexpr (VEC > 1) {  // t again, from this thread's own slots: registers are scarcer
        ring.take(r, 1, a.g, a.g_stride, m + r, vg);
#pragma unroll
        for (int p = 0; p < P; p++) tw[0][p] = mul2(pair_of(vg, p), w[p]);
      }
#pragma unroll
      for (int k = 0; k < K; k++) {
        float f[VEC];
#pragma unroll
        for (int j = 0; j < VEC; j++) {
          const int p = (k * VEC + j) / 2;
          const F2 d = fma2(xh[r][p], c1, fma2(tw[VEC == 1 ? r : 0][p], q, c0));
          f[j] = (k * VEC + j) & 1 ? d.hi() : d.lo();
        }
        ring.store(dp + (m + r) * a.dx_jump, k, f);
      }
    }
    ring.taken();
  }
  copies_wait<0>();
  if (!SMALL && !a.part) return;
  float* cols = reinterpret_cast<float*>(dyn);  // [2][dim], in the ring's place
  float* part = SMALL ? cols : a.part + (size_t)blockIdx.x * 2 * a.dim;
  // the groups of a block add their sums in shared memory, one after another
  for (int r = 0; r < groups; r++) {
    __syncthreads();
    if ((int)threadIdx.y != r) continue;
#pragma unroll
    for (int k = 0; k < K; k++) {
#pragma unroll
      for (int j = 0; j < VEC; j++) {
        const int c = ring.col(k) + j, p = (k * VEC + j) / 2;
        if (MODE != FULL_ROWS && (c < 0 || c >= a.dim)) continue;
        const float w1 = (k * VEC + j) & 1 ? dw[p].hi() : dw[p].lo();
        const float b1 = (k * VEC + j) & 1 ? db[p].hi() : db[p].lo();
        const float pw = r ? cols[c] : 0.0f, pb = r ? cols[a.dim + c] : 0.0f;
        if (r + 1 < groups) {
          cols[c] = pw + w1;
          cols[a.dim + c] = pb + b1;
        } else {
          part[c] = pw + w1;
          part[a.dim + c] = pb + b1;
        }
      }
    }
  }
  if (!SMALL) return;
  cluster_sync();
  // every block adds up a share of the columns over the blocks, in their order
  for (int c = blockIdx.x * group * groups + lin; c < 2 * a.dim; c += gridDim.x * group * groups) {
    float v = 0.0f;
    for (unsigned int q = 0; q < gridDim.x; q++)
      v += __uint_as_float(peer_load(reinterpret_cast<const unsigned int*>(cols + c), q));
    void* out = c < a.dim ? a.dw : a.db;
    if (out) store_param(out, a.w_type, c < a.dim ? c : c - a.dim, v);
  }
  cluster_sync();  // no block leaves while another may read its memory
}

// Long rows: dx by a block per row (the row is read twice) ...
template <typename X, int VEC>
__global__ void __launch_bounds__(LN_LONG_THREADS) ln_grad_long_kernel(LnGradArgs a) {
  __shared__ float red[2 * 32 * 2];
  int turn = 0;
  for (long long row = blockIdx.x; row < a.n; row += gridDim.x) {
    const X* x = reinterpret_cast<const X*>(a.x) + row * a.x_stride;
    const X* g = reinterpret_cast<const X*>(a.g) + row * a.g_stride;
    const float mean = a.mean[row], rstd = a.rstd[row];
    float s[2] = {0.0f, 0.0f};
    for (int q = threadIdx.x; q < a.dim / VEC; q += LN_LONG_THREADS) {
      const RowVec<X, VEC> vx = load_row<X, VEC>(x + (long long)q * VEC);
      const RowVec<X, VEC> vg = load_row<X, VEC>(g + (long long)q * VEC);
      float w[VEC];
      load_param<VEC>(a.w, a.w_type, (long long)q * VEC, 1.0f, w);
#pragma unroll
      for (int j = 0; j < VEC; j++) {
        const float t = to_f32(vg.v[j]) * w[j];
        s[0] += t;
        s[1] += t * ((to_f32(vx.v[j]) - mean) * rstd);
      }
    }
    block_sum(s, red, turn);
    const float c0 = s[0] * a.inv_dim, c1 = s[1] * a.inv_dim;
    X* dx = reinterpret_cast<X*>(a.dx) + row * a.dx_stride;
    for (int q = threadIdx.x; q < a.dim / VEC; q += LN_LONG_THREADS) {
      const RowVec<X, VEC> vx = load_row<X, VEC>(x + (long long)q * VEC);
      const RowVec<X, VEC> vg = load_row<X, VEC>(g + (long long)q * VEC);
      float w[VEC];
      load_param<VEC>(a.w, a.w_type, (long long)q * VEC, 1.0f, w);
#pragma unroll
      for (int j = 0; j < VEC; j++)
        w[j] = rstd * (to_f32(vg.v[j]) * w[j] - c0 - (to_f32(vx.v[j]) - mean) * rstd * c1);
      store_vec<X, VEC>(dx + (long long)q * VEC, w);
    }
  }
}

// ... and partial sums of dw and db over slices of the rows, by column.
template <typename X>
__global__ void __launch_bounds__(LN_LONG_THREADS) ln_grad_cols_kernel(LnGradArgs a) {
  const long long c = (long long)blockIdx.y * LN_LONG_THREADS + threadIdx.x;
  if (c >= a.dim) return;
  const X* x = reinterpret_cast<const X*>(a.x) + c;
  const X* g = reinterpret_cast<const X*>(a.g) + c;
  float dw = 0.0f, db = 0.0f;
  for (long long row = blockIdx.x; row < a.n; row += gridDim.x) {
    const float gv = to_f32(g[row * a.g_stride]);
    dw += gv * ((to_f32(x[row * a.x_stride]) - a.mean[row]) * a.rstd[row]);
    db += gv;
  }
  a.part[(size_t)blockIdx.x * 2 * a.dim + c] = dw;
  a.part[((size_t)blockIdx.x * 2 + 1) * a.dim + c] = db;
}

// dweight and dbias: the blocks' partial rows, added in a fixed order
__global__ void __launch_bounds__(1024) ln_param_kernel(const float* __restrict__ part, int parts, int dim, int type,
                                                        void* dw, void* db) {
  __shared__ float s[32][33];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const long long c = (long long)blockIdx.x * 32 + tx;  // column of the two rows laid end to end
  float v = 0.0f;
  if (c < 2ll * dim)
    for (int p = ty; p < parts; p += 32) v += part[(size_t)p * 2 * dim + c];
  s[ty][tx] = v;
  __syncthreads();
  v = s[tx][ty];  // warp ty holds column ty
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const long long col = (long long)blockIdx.x * 32 + ty;
  if (tx == 0 && col < 2ll * dim) {
    void* out = col < dim ? dw : db;
    if (out) store_param(out, type, col < dim ? col : col - dim, v);
  }
}

// ------------------------------------------------------------------ host side
constexpr int MAX_SMS = 256;  // the workspace is sized without a device
// Partial rows of dw and db: one per block.
int max_parts(int sms) { return std::min(sms, MAX_SMS); }

// How the rows of a call's matrices meet 16-byte boundaries.
struct Layout {
  bool alike = true;  // every matrix the same way
  int period = 1;     // rows after which they meet them again
  bool aligned = true;
  bool params = true;  // weight and bias can be read in the same vectors
  void add(const Rows& r, const Rows& first) {
    if (!r.p) return;
    const int64_t b = type_bytes(r.type);
    alike = alike && (((uintptr_t)r.p ^ (uintptr_t)first.p) & 15) == 0 && ((r.stride - first.stride) * b) % 16 == 0;
    aligned = aligned && ((uintptr_t)r.p & 15) == 0 && (r.stride * b) % 16 == 0;
    int p = 1;
    while ((r.stride * b * p) % 16) p++;
    period = std::max(period, p);  // powers of two
  }
};

struct Plan {
  int group, groups;
  unsigned int grid;
  int mode;
};
// Threads of a group when each has k vectors of VEC elements: part of a warp (a
// power of two) or whole warps; whole warps where the group stages rows.
template <int VEC>
int group_of(int dim, int k, const Layout& l) {
  // a row that does not start on a boundary may touch one vector more
  const int vecs = VEC == 1 ? dim : (dim + (l.aligned ? 0 : VEC - 1) + VEC - 1) / VEC;
  const int t = (vecs + k - 1) / k;
  if (t > 32 || VEC == 1) return (t + 31) / 32 * 32;
  int g = 1;
  while (g < t) g <<= 1;
  return g;
}
template <int VEC>
Plan plan_of(int64_t n, int dim, int k, int rows, int threads, const Layout& l, int sms, int max_grid) {
  Plan p;
  p.group = group_of<VEC>(dim, k, l);
  // groups of a block: as many as fit, unless there are too few rows for the
  // SMs. Each group of several warps has a barrier of its own, of which a block
  // has 15 besides the first.
  const int most = std::min(threads / p.group, p.group > 32 ? 15 : threads);
  p.groups = (int)std::max<int64_t>(1, std::min<int64_t>(most, n / ((int64_t)rows * sms)));
  if (p.group < 32) p.groups = std::max(p.groups / (32 / p.group), 1) * (32 / p.group);  // whole warps
  int64_t grid = std::min<int64_t>((n + (int64_t)p.groups * rows - 1) / (p.groups * rows), max_grid);
  if (VEC > 1) {  // all groups together: a multiple of the rows' period
    while (grid * p.groups % l.period && grid + 1 <= max_grid && grid < l.period) grid++;
    while (grid * p.groups % l.period) grid--;
  }
  p.grid = (unsigned int)grid;
  p.mode = VEC == 1 || !l.aligned || !l.params || dim % VEC ? EDGES
           : (int64_t)p.group * k * VEC == dim              ? FULL_ROWS
                                                            : WHOLE_VECS;
  return p;
}

// Stages of the ring: about 256 bytes a thread, of which one stage is in use.
constexpr int stages_of(int stage) { return 256 / stage < 2 ? 2 : 256 / stage > 8 ? 8 : 256 / stage; }

RowWalk walk_of(const Plan& p, int64_t n, int dim, const void* x) {
  return {n, (long long)p.grid * p.groups,
          reinterpret_cast<const char*>(reinterpret_cast<uintptr_t>(x) & ~(uintptr_t)15), dim};
}

template <typename X, int VEC, int K, int R, int GROUP = 0>
void launch_ln_k(LnArgs a, const Layout& l, int sms, cudaStream_t st) {
  constexpr int STAGES = stages_of(VEC * (int)sizeof(X) * K * R);
  const Plan p = plan_of<VEC>(a.n, a.dim, K, R, LN_THREADS, l, sms, sms);
  a.walk = walk_of(p, a.n, a.dim, a.x);
  a.x_jump = a.walk.total * a.x_stride * (long long)sizeof(X);
  a.y_jump = a.walk.total * a.y_stride * (long long)sizeof(X);
  const size_t smem = RowRing<X, VEC, K, R, 1, STAGES, EDGES, LN_THREADS, GROUP>::bytes(p.groups, a.dim);
  auto kernel = ln_kernel<X, VEC, K, R, STAGES, EDGES, LN_THREADS, GROUP>;
  if constexpr (VEC > 1) {
    if (p.mode == FULL_ROWS) kernel = ln_kernel<X, VEC, K, R, STAGES, FULL_ROWS, LN_THREADS, GROUP>;
    if (p.mode == WHOLE_VECS) kernel = ln_kernel<X, VEC, K, R, STAGES, WHOLE_VECS, LN_THREADS, GROUP>;
  }
  if (smem > 40 * 1024) allow_smem(reinterpret_cast<const void*>(kernel), smem);
  kernel<<<p.grid, dim3(p.group, p.groups), smem, st>>>(a);
}

template <typename X, int VEC>
void launch_ln(const LnArgs& a, const Layout& l, int sms, cudaStream_t st) {
  const auto group = [&](int k) { return group_of<VEC>(a.dim, k, l); };
  // A warp to a row, without barriers, as long as a thread then has 32 columns
  // at most; several warps with 32 columns a thread for longer rows. (262,144 x
  // 1024 bf16: 186 us; 254 us as groups of 4 warps with 8 columns a thread and 4
  // rows to a barrier. Narrow rows go 4 at a time: 1,000,000 x 128 bf16 94 us, 158 us
  // one at a time.)
  constexpr int U = VEC == 1 ? 16 / (int)sizeof(X) : 1, E = VEC * U;  // columns of 16 bytes
  constexpr int MOST = 32 / E;
  if (group(U) <= 32) return launch_ln_k<X, VEC, U, 4>(a, l, sms, st);
  if (group(2 * U) <= 32) return launch_ln_k<X, VEC, 2 * U, 16 / E, 32>(a, l, sms, st);
  if constexpr (MOST == 4) {
    if (group(3 * U) <= 32) return launch_ln_k<X, VEC, 3 * U, 1, 32>(a, l, sms, st);
  } else {
    if (group(4 * U) <= 32) return launch_ln_k<X, VEC, 4 * U, 2, 32>(a, l, sms, st);
    if (group(6 * U) <= 32) return launch_ln_k<X, VEC, 6 * U, 1, 32>(a, l, sms, st);
  }
  if (group(MOST * U) <= 32) return launch_ln_k<X, VEC, MOST * U, 1, 32>(a, l, sms, st);
  launch_ln_k<X, VEC, MOST * U, 1>(a, l, sms, st);
}

// Few rows go to one cluster, which also adds up dw and db: a launch less (129 x
// 768 fp16: 18.7 us a pass by two kernels, 17.2 this way, and 14.7 since it needs no
// workspace). Those that `few` names go there for certain, so a call may leave the
// workspace out; others where a group has up to CLUSTER_STEPS steps.
constexpr int CLUSTER = 8, CLUSTER_STEPS = 4;
bool few(int64_t n, int64_t dim) { return dim <= 4096 && n <= GIDS_FEW_NORM / std::max<int64_t>(dim, 128); }

// Returns the partial rows left in a.part.
template <typename X, int VEC, int K, int R, int GROUP = 0>
int launch_ln_grad_k(LnGradArgs a, const Layout& l, int sms, cudaStream_t st) {
  constexpr int STAGES = stages_of(2 * VEC * (int)sizeof(X) * K * R);
  Plan p = plan_of<VEC>(a.n, a.dim, K, R, LN_THREADS, l, sms, max_parts(sms));
  const int most = std::min(LN_THREADS / p.group, p.group > 32 ? 15 : LN_THREADS);
  const bool small =
      (a.dw || a.db) && (few(a.n, a.dim) || a.n <= (int64_t)CLUSTER_STEPS * CLUSTER * most * R);
  if (small) {
    a.part = nullptr;
    p.groups = most;
    p.grid = 1;
    while (p.grid < CLUSTER && (l.period > 1 || (int64_t)p.grid * most * R < a.n)) p.grid *= 2;
  }
  a.walk = walk_of(p, a.n, a.dim, a.x);
  a.x_jump = a.walk.total * a.x_stride * (long long)sizeof(X);
  a.g_jump = a.walk.total * a.g_stride * (long long)sizeof(X);
  a.dx_jump = a.walk.total * a.dx_stride * (long long)sizeof(X);
  const size_t smem = std::max(RowRing<X, VEC, K, R, 2, STAGES, EDGES, LN_THREADS, GROUP>::bytes(p.groups, a.dim),
                               p.groups > 1 || small ? (size_t)a.dim * 2 * sizeof(float) : 0);
  const auto of_mode = [&](auto mode) {
    return small ? ln_grad_kernel<X, VEC, K, R, STAGES, decltype(mode)::value, LN_THREADS, GROUP, true>
                 : ln_grad_kernel<X, VEC, K, R, STAGES, decltype(mode)::value, LN_THREADS, GROUP, false>;
  };
  auto kernel = of_mode(std::integral_constant<int, EDGES>());
  if constexpr (VEC > 1) {
    if (p.mode == FULL_ROWS) kernel = of_mode(std::integral_constant<int, FULL_ROWS>());
    if (p.mode == WHOLE_VECS) kernel = of_mode(std::integral_constant<int, WHOLE_VECS>());
  }
  if (smem > 40 * 1024) allow_smem(reinterpret_cast<const void*>(kernel), smem);
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = p.grid;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = p.grid;
  cfg.blockDim = dim3(p.group, p.groups);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = &attr;
  cfg.numAttrs = small && p.grid > 1 ? 1 : 0;
  GIDS_CUDA(cudaLaunchKernelEx(&cfg, kernel, a));
  return a.part ? (int)p.grid : 0;
}

template <typename X, int VEC>
int launch_ln_grad(const LnGradArgs& a, const Layout& l, int sms, cudaStream_t st) {
  const auto group = [&](int k) { return group_of<VEC>(a.dim, k, l); };
  constexpr int U = VEC == 1 ? 16 / (int)sizeof(X) : 1;
  // Few columns a thread (their sums, the parameters and R rows are all in
  // registers) and R rows to a barrier, as long as a block has two groups to
  // overlap: 262,144 x 1024 bf16 253 us with 4 rows of one vector, 281 us with 2
  // rows; 65,536 x 4096 bf16 358 us as one group of 512 threads with 4 rows, 298 us as
  // two of 256 with one row of two vectors, 272 us with two rows (which spill where the
  // edges of odd rows take registers too).
  if (group(U) <= LN_THREADS / 2) return launch_ln_grad_k<X, VEC, U, 4>(a, l, sms, st);
  if (group(2 * U) <= LN_THREADS)
    return l.aligned ? launch_ln_grad_k<X, VEC, 2 * U, 2>(a, l, sms, st)
                     : launch_ln_grad_k<X, VEC, 2 * U, 1>(a, l, sms, st);
  return launch_ln_grad_k<X, VEC, 4 * U, 1>(a, l, sms, st);
}

// Rows that do not fit the registers of a block.
template <typename X, int VEC>
int launch_ln_grad_long(const LnGradArgs& a, int sms, cudaStream_t st) {
  int parts = 0;
  if (a.part) {
    parts = (int)std::min<int64_t>(a.n, std::min(max_parts(sms), 64));
    const dim3 grid((unsigned int)parts, (unsigned int)((a.dim + LN_LONG_THREADS - 1) / LN_LONG_THREADS));
    ln_grad_cols_kernel<X><<<grid, LN_LONG_THREADS, 0, st>>>(a);
  }
  if (a.dx)  // last: dx may be written over x or grad
    ln_grad_long_kernel<X, VEC><<<(unsigned int)std::min<int64_t>(a.n, (int64_t)sms * 4), LN_LONG_THREADS, 0, st>>>(a);
  return parts;
}

void check_norm(int device, int64_t n, int64_t dim, int x_type, int param_type) {
  GIDS_CHECK(device >= 0, GIDS_E_INVAL, "bad device");
  GIDS_CHECK(n >= 0 && n < (1ll << 38), GIDS_E_INVAL, "n must be in [0, 2^38)");
  GIDS_CHECK(dim >= 1 && dim <= (1ll << 24), GIDS_E_INVAL, "dim must be in [1, 2^24]");
  GIDS_CHECK(param_type == x_type || param_type == GIDS_F32, GIDS_E_UNSUPPORTED,
             "weight and bias must have the rows' type or be float32");
}

bool param_ok(const void* p, int param_type, int vec) {
  const int64_t b = (int64_t)type_bytes(param_type) * vec;
  return !p || ((uintptr_t)p) % (uintptr_t)(b < 16 ? b : 16) == 0;
}
void check_param(const void* p, int param_type, const char* what) {
  GIDS_CHECK(param_ok(p, param_type, 1), GIDS_E_INVAL, std::string(what) + ": address not aligned to its elements");
}

template <typename X>
void ln_typed(const LnArgs& a, const Layout& l, int sms, cudaStream_t st) {
  constexpr int BIG = 16 / (int)sizeof(X);
  const unsigned int long_grid = (unsigned int)std::min<int64_t>(a.n, (int64_t)sms * 4);
  if (l.alike && l.period <= sms && group_of<BIG>(a.dim, 32 / BIG, l) <= LN_THREADS)
    launch_ln<X, BIG>(a, l, sms, st);
  else if (group_of<1>(a.dim, 32, l) <= LN_THREADS)
    launch_ln<X, 1>(a, l, sms, st);
  else if (l.aligned && l.params && a.dim % BIG == 0)
    ln_long_kernel<X, BIG><<<long_grid, LN_LONG_THREADS, 0, st>>>(a);
  else
    ln_long_kernel<X, 1><<<long_grid, LN_LONG_THREADS, 0, st>>>(a);
  GIDS_CUDA(cudaGetLastError());
}

template <typename X>
void ln_grad_typed(const LnGradArgs& a, const Layout& l, int sms, cudaStream_t st) {
  constexpr int BIG = 16 / (int)sizeof(X);
  int parts;
  if (l.alike && l.period <= sms && group_of<BIG>(a.dim, 4, l) <= LN_THREADS)
    parts = launch_ln_grad<X, BIG>(a, l, sms, st);
  else if (group_of<1>(a.dim, 4 * BIG, l) <= LN_THREADS)
    parts = launch_ln_grad<X, 1>(a, l, sms, st);
  else if (l.aligned && l.params && a.dim % BIG == 0)
    parts = launch_ln_grad_long<X, BIG>(a, sms, st);
  else
    parts = launch_ln_grad_long<X, 1>(a, sms, st);
  GIDS_CUDA(cudaGetLastError());
  if (!a.part || !parts) return;
  ln_param_kernel<<<(unsigned int)((2ll * a.dim + 31) / 32), 1024, 0, st>>>(a.part, parts, a.dim, a.w_type, a.dw, a.db);
  GIDS_CUDA(cudaGetLastError());
}

}  // namespace

void layer_norm(int device, Rows y, float* mean, float* rstd, Rows x, const void* weight, const void* bias,
                int param_type, int64_t n, int64_t dim, float eps, cudaStream_t st) {
  check_norm(device, n, dim, x.type, param_type);
  check_rows(y, "y", n, dim, true);
  check_rows(x, "x", n, dim, false);
  GIDS_CHECK(y.type == x.type, GIDS_E_UNSUPPORTED, "y must have the rows' type");
  check_param(weight, param_type, "weight");
  check_param(bias, param_type, "bias");
  GIDS_CHECK((mean == nullptr) == (rstd == nullptr), GIDS_E_INVAL, "mean and rstd come together or not at all");
  check_param(mean, GIDS_F32, "mean");
  check_param(rstd, GIDS_F32, "rstd");
  GIDS_CHECK(eps >= 0.0f, GIDS_E_INVAL, "eps must be >= 0");
  if (n == 0) return;
  DeviceGuard dg(device);
  LnArgs a{};
  a.y = y.p;
  a.x = x.p;
  a.mean = mean;
  a.rstd = rstd;
  a.w = weight;
  a.b = bias;
  a.y_stride = y.stride;
  a.x_stride = x.stride;
  a.n = n;
  a.dim = (int)dim;
  a.eps = eps;
  a.inv_dim = 1.0f / (float)dim;
  a.w_type = param_type;
  Layout l;
  l.add(x, x);
  l.add(y, x);
  l.params = param_ok(weight, param_type, 16 / type_bytes(x.type)) && param_ok(bias, param_type, 16 / type_bytes(x.type));
  const int sms = device_sms(device);
  if (x.type == GIDS_F32) return ln_typed<float>(a, l, sms, st);
  if (x.type == GIDS_F16) return ln_typed<__half>(a, l, sms, st);
  return ln_typed<__nv_bfloat16>(a, l, sms, st);
}

uint64_t layer_norm_grad_workspace(int64_t n, int64_t dim) {
  check_norm(0, n, dim, GIDS_F32, GIDS_F32);
  // a block to every row at least, and to every row of a period
  return (uint64_t)std::min<int64_t>(std::max<int64_t>(n, 8), MAX_SMS) * 2 * (uint64_t)dim * sizeof(float);
}

void layer_norm_grad(int device, Rows dx, void* dweight, void* dbias, Rows grad, Rows x, const float* mean,
                     const float* rstd, const void* weight, int param_type, int64_t n, int64_t dim, void* ws,
                     uint64_t ws_bytes, cudaStream_t st) {
  check_norm(device, n, dim, x.type, param_type);
  check_rows(grad, "grad", n, dim, false);
  check_rows(x, "x", n, dim, false);
  GIDS_CHECK(grad.type == x.type && dx.type == x.type, GIDS_E_UNSUPPORTED, "grad and dx must have the rows' type");
  if (dx.p) check_rows(dx, "dx", n, dim, true);
  check_param(weight, param_type, "weight");
  check_param(dweight, param_type, "dweight");
  check_param(dbias, param_type, "dbias");
  GIDS_CHECK(n == 0 || (mean && rstd), GIDS_E_INVAL, "mean or rstd is null");
  check_param(mean, GIDS_F32, "mean");
  check_param(rstd, GIDS_F32, "rstd");
  const bool params = dweight || dbias;
  if (params && n && !(few(n, dim) && !ws && !ws_bytes)) {
    GIDS_CHECK(ws && ((uintptr_t)ws) % 256 == 0, GIDS_E_INVAL, "workspace is null or not aligned to 256 bytes");
    GIDS_CHECK(ws_bytes >= layer_norm_grad_workspace(n, dim), GIDS_E_INVAL,
               "workspace too small: " + std::to_string(layer_norm_grad_workspace(n, dim)) + " bytes are needed");
  }
  if (!params && (n == 0 || !dx.p)) return;
  DeviceGuard dg(device);
  if (n == 0) {  // sums over no rows
    const size_t b = (size_t)dim * type_bytes(param_type);
    if (dweight) GIDS_CUDA(cudaMemsetAsync(dweight, 0, b, st));
    if (dbias) GIDS_CUDA(cudaMemsetAsync(dbias, 0, b, st));
    return;
  }
  LnGradArgs a{};
  a.dx = dx.p;
  a.g = grad.p;
  a.x = x.p;
  a.mean = mean;
  a.rstd = rstd;
  a.w = weight;
  a.part = params ? static_cast<float*>(ws) : nullptr;
  a.dw = dweight;
  a.db = dbias;
  a.dx_stride = dx.stride;
  a.g_stride = grad.stride;
  a.x_stride = x.stride;
  a.n = n;
  a.dim = (int)dim;
  a.inv_dim = 1.0f / (float)dim;
  a.w_type = param_type;
  Layout l;
  l.add(x, x);
  l.add(grad, x);
  l.add(dx, x);
  l.params = param_ok(weight, param_type, 16 / type_bytes(x.type));
  const int sms = device_sms(device);
  if (x.type == GIDS_F32) return ln_grad_typed<float>(a, l, sms, st);
  if (x.type == GIDS_F16) return ln_grad_typed<__half>(a, l, sms, st);
  return ln_grad_typed<__nv_bfloat16>(a, l, sms, st);
}

}  // namespace gids
