// Layer norm and its gradient, for sm_100a.
//
// Forward: m = mean(x), v = mean((x - m)^2), r = 1 / sqrt(v + eps),
// y = round((x - m) r w + b). A group of threads holds one row in registers,
// so x is read once and the variance is the sum of squared differences from
// the mean, not a difference of sums.
//
// Backward, with xh = (x - m) r and t = g w:
//   dx = round(r (t - mean(t) - xh mean(t xh))), dw = sum g xh, db = sum g.
// Groups walk over rows with the sums of their columns in float32 registers;
// every block leaves one partial row of dw and of db in the workspace, and a
// second kernel adds them in block order. No atomics: results repeat bit for
// bit.
#include <algorithm>

#include "layers.hpp"
#include "rows.cuh"

namespace gids {
namespace {

constexpr int LN_THREADS = 128;      // threads of a block whose groups are a warp or less
constexpr int LN_MAX_GROUP = 1024;   // threads of the largest group
constexpr int LN_LONG_THREADS = 512; // rows that do not fit the registers of a group

struct LnArgs {
  void* y;
  const void* x;
  float* mean;
  float* rstd;
  const void* w;
  const void* b;
  long long y_stride, x_stride, n;
  int dim, vecs, group;  // group: threads per row, a power of two
  float eps, inv_dim;
};

struct LnGradArgs {
  void* dx;
  const void* g;
  const void* x;
  const float* mean;
  const float* rstd;
  const void* w;
  float* part;  // [blocks][2][dim], or null: no weight gradient
  long long dx_stride, g_stride, x_stride, n;
  int dim, vecs, group;
  float inv_dim;
};

// Sum over the threads of a group. Groups of a warp or less use shuffles;
// larger ones are the whole block and add their warps' sums in warp order.
// `red` holds two buffers of 2 x 32 floats, used in turn, so one barrier is
// enough.
template <int N>
__device__ __forceinline__ void group_sum(float (&v)[N], int group, float* red, int& turn) {
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    if (o < group) {
#pragma unroll
      for (int i = 0; i < N; i++) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    }
  }
  if (group > 32) {
    float* buf = red + turn * 64;
    turn ^= 1;
    const int warps = group >> 5;
    if ((threadIdx.x & 31) == 0) {
#pragma unroll
      for (int i = 0; i < N; i++) buf[i * 32 + (threadIdx.x >> 5)] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; i++) {
      float s = 0.0f;
      for (int k = 0; k < warps; k++) s += buf[i * 32 + k];
      v[i] = s;
    }
  }
}

template <typename P, int VEC>
__device__ __forceinline__ void load_param(const void* p, long long i, float fill, float (&f)[VEC]) {
  if (p) {
    const RowVec<P, VEC> v = load_vec<P, VEC>(reinterpret_cast<const P*>(p) + i);
#pragma unroll
    for (int j = 0; j < VEC; j++) f[j] = to_f32(v.v[j]);
  } else {
#pragma unroll
    for (int j = 0; j < VEC; j++) f[j] = fill;
  }
}

// The rounded mean is off by up to half a step of the mean, which is not small
// beside the differences when the mean is large against them. `off` is the
// mean of the differences from it: the second pass takes it out again.
__device__ __forceinline__ float variance(float mean_sq, float off) { return fmaxf(mean_sq - off * off, 0.0f); }

template <typename X, typename P, int VEC, int K>
__global__ void __launch_bounds__(LN_MAX_GROUP) ln_kernel(LnArgs a) {
  __shared__ float red[2 * 32 * 2];
  int turn = 0;
  const int t = threadIdx.x & (a.group - 1);
  const int rpb = blockDim.x / a.group;
  for (long long base = (long long)blockIdx.x * rpb; base < a.n; base += (long long)gridDim.x * rpb) {
    const long long row = base + threadIdx.x / a.group;
    const bool on = row < a.n;
    const X* x = reinterpret_cast<const X*>(a.x) + row * a.x_stride;
    float f[K][VEC];
    float s[1] = {0.0f};
#pragma unroll
    for (int k = 0; k < K; k++) {
      const int q = k * a.group + t;
      if (on && q < a.vecs) {
        const RowVec<X, VEC> v = load_row<X, VEC>(x + (long long)q * VEC);
#pragma unroll
        for (int j = 0; j < VEC; j++) f[k][j] = to_f32(v.v[j]);
      } else {
#pragma unroll
        for (int j = 0; j < VEC; j++) f[k][j] = 0.0f;
      }
    }
#pragma unroll
    for (int k = 0; k < K; k++)
#pragma unroll
      for (int j = 0; j < VEC; j++) s[0] += f[k][j];
    group_sum(s, a.group, red, turn);
    const float mean = s[0] * a.inv_dim;
    float d[2] = {0.0f, 0.0f};  // sums of x - mean and of its square
#pragma unroll
    for (int k = 0; k < K; k++) {
      const bool in = k * a.group + t < a.vecs;
#pragma unroll
      for (int j = 0; j < VEC; j++) {
        f[k][j] = in ? f[k][j] - mean : 0.0f;
        d[0] += f[k][j];
        d[1] += f[k][j] * f[k][j];
      }
    }
    group_sum(d, a.group, red, turn);
    const float off = d[0] * a.inv_dim;
    const float rstd = 1.0f / sqrtf(variance(d[1] * a.inv_dim, off) + a.eps);
    if (!on) continue;
    if (t == 0 && a.mean) {
      a.mean[row] = mean + off;
      a.rstd[row] = rstd;
    }
    X* y = reinterpret_cast<X*>(a.y) + row * a.y_stride;
#pragma unroll
    for (int k = 0; k < K; k++) {
      const int q = k * a.group + t;
      if (q >= a.vecs) continue;
      float w[VEC], b[VEC];
      load_param<P, VEC>(a.w, (long long)q * VEC, 1.0f, w);
      load_param<P, VEC>(a.b, (long long)q * VEC, 0.0f, b);
#pragma unroll
      for (int j = 0; j < VEC; j++) w[j] = (f[k][j] - off) * rstd * w[j] + b[j];
      store_vec<X, VEC>(y + (long long)q * VEC, w);
    }
  }
}

// Rows longer than a group's registers: the row is read three times, the
// second and third time from L2.
template <typename X, typename P, int VEC>
__global__ void __launch_bounds__(LN_LONG_THREADS) ln_long_kernel(LnArgs a) {
  __shared__ float red[2 * 32 * 2];
  int turn = 0;
  for (long long row = blockIdx.x; row < a.n; row += gridDim.x) {
    const X* x = reinterpret_cast<const X*>(a.x) + row * a.x_stride;
    float s[1] = {0.0f};
    for (int q = threadIdx.x; q < a.vecs; q += LN_LONG_THREADS) {
      const RowVec<X, VEC> v = load_row<X, VEC>(x + (long long)q * VEC);
#pragma unroll
      for (int j = 0; j < VEC; j++) s[0] += to_f32(v.v[j]);
    }
    group_sum(s, LN_LONG_THREADS, red, turn);
    const float mean = s[0] * a.inv_dim;
    float d[2] = {0.0f, 0.0f};
    for (int q = threadIdx.x; q < a.vecs; q += LN_LONG_THREADS) {
      const RowVec<X, VEC> v = load_row<X, VEC>(x + (long long)q * VEC);
#pragma unroll
      for (int j = 0; j < VEC; j++) {
        const float c = to_f32(v.v[j]) - mean;
        d[0] += c;
        d[1] += c * c;
      }
    }
    group_sum(d, LN_LONG_THREADS, red, turn);
    const float off = d[0] * a.inv_dim;
    const float rstd = 1.0f / sqrtf(variance(d[1] * a.inv_dim, off) + a.eps);
    if (threadIdx.x == 0 && a.mean) {
      a.mean[row] = mean + off;
      a.rstd[row] = rstd;
    }
    X* y = reinterpret_cast<X*>(a.y) + row * a.y_stride;
    for (int q = threadIdx.x; q < a.vecs; q += LN_LONG_THREADS) {
      const RowVec<X, VEC> v = load_row<X, VEC>(x + (long long)q * VEC);
      float w[VEC], b[VEC];
      load_param<P, VEC>(a.w, (long long)q * VEC, 1.0f, w);
      load_param<P, VEC>(a.b, (long long)q * VEC, 0.0f, b);
#pragma unroll
      for (int j = 0; j < VEC; j++) w[j] = (to_f32(v.v[j]) - mean - off) * rstd * w[j] + b[j];
      store_vec<X, VEC>(y + (long long)q * VEC, w);
    }
  }
}

// ------------------------------------------------------------------ backward
// The rows of a block's groups, with dx, and the block's partial dw and db.
template <typename X, typename P, int VEC, int K>
__global__ void __launch_bounds__(512) ln_grad_kernel(LnGradArgs a) {
  extern __shared__ float cols[];  // [2][dim], for blocks of several groups
  __shared__ float red[2 * 32 * 2];
  int turn = 0;
  const int t = threadIdx.x & (a.group - 1);
  const int rpb = blockDim.x / a.group;
  float w[K][VEC], dw[K][VEC], db[K][VEC];
#pragma unroll
  for (int k = 0; k < K; k++) {
    const int q = k * a.group + t;
    load_param<P, VEC>(q < a.vecs ? a.w : nullptr, (long long)q * VEC, 1.0f, w[k]);
#pragma unroll
    for (int j = 0; j < VEC; j++) dw[k][j] = db[k][j] = 0.0f;
  }
  for (long long base = (long long)blockIdx.x * rpb; base < a.n; base += (long long)gridDim.x * rpb) {
    const long long row = base + threadIdx.x / a.group;
    const bool on = row < a.n;
    const X* x = reinterpret_cast<const X*>(a.x) + row * a.x_stride;
    const X* g = reinterpret_cast<const X*>(a.g) + row * a.g_stride;
    const float mean = on ? __ldg(a.mean + row) : 0.0f;
    const float rstd = on ? __ldg(a.rstd + row) : 0.0f;
    float xh[K][VEC], gv[K][VEC];
    float s[2] = {0.0f, 0.0f};  // sums of t and of t * xh
#pragma unroll
    for (int k = 0; k < K; k++) {
      const int q = k * a.group + t;
      if (on && q < a.vecs) {
        const RowVec<X, VEC> vx = load_row<X, VEC>(x + (long long)q * VEC);
        const RowVec<X, VEC> vg = load_row<X, VEC>(g + (long long)q * VEC);
#pragma unroll
        for (int j = 0; j < VEC; j++) {
          xh[k][j] = (to_f32(vx.v[j]) - mean) * rstd;
          gv[k][j] = to_f32(vg.v[j]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < VEC; j++) xh[k][j] = gv[k][j] = 0.0f;
      }
    }
#pragma unroll
    for (int k = 0; k < K; k++)
#pragma unroll
      for (int j = 0; j < VEC; j++) {
        dw[k][j] += gv[k][j] * xh[k][j];
        db[k][j] += gv[k][j];
        gv[k][j] *= w[k][j];
        s[0] += gv[k][j];
        s[1] += gv[k][j] * xh[k][j];
      }
    if (!a.dx) continue;
    group_sum(s, a.group, red, turn);
    if (!on) continue;
    const float c0 = s[0] * a.inv_dim, c1 = s[1] * a.inv_dim;
    X* dx = reinterpret_cast<X*>(a.dx) + row * a.dx_stride;
#pragma unroll
    for (int k = 0; k < K; k++) {
      const int q = k * a.group + t;
      if (q >= a.vecs) continue;
      float f[VEC];
#pragma unroll
      for (int j = 0; j < VEC; j++) f[j] = rstd * (gv[k][j] - c0 - xh[k][j] * c1);
      store_vec<X, VEC>(dx + (long long)q * VEC, f);
    }
  }
  if (!a.part) return;
  float* part = a.part + (size_t)blockIdx.x * 2 * a.dim;
  // the groups of a block add their sums in shared memory, one after another
  for (int r = 0; r < rpb; r++) {
    if ((int)threadIdx.x / a.group == r) {
#pragma unroll
      for (int k = 0; k < K; k++) {
        const int q = k * a.group + t;
        if (q >= a.vecs) continue;
#pragma unroll
        for (int j = 0; j < VEC; j++) {
          const int c = q * VEC + j;
          const float pw = r ? cols[c] : 0.0f, pb = r ? cols[a.dim + c] : 0.0f;
          if (r + 1 < rpb) {
            cols[c] = pw + dw[k][j];
            cols[a.dim + c] = pb + db[k][j];
          } else {
            part[c] = pw + dw[k][j];
            part[a.dim + c] = pb + db[k][j];
          }
        }
      }
    }
    if (rpb > 1) __syncthreads();
  }
}

// Long rows: dx by a block per row (the row is read twice) ...
template <typename X, typename P, int VEC>
__global__ void __launch_bounds__(LN_LONG_THREADS) ln_grad_long_kernel(LnGradArgs a) {
  __shared__ float red[2 * 32 * 2];
  int turn = 0;
  for (long long row = blockIdx.x; row < a.n; row += gridDim.x) {
    const X* x = reinterpret_cast<const X*>(a.x) + row * a.x_stride;
    const X* g = reinterpret_cast<const X*>(a.g) + row * a.g_stride;
    const float mean = a.mean[row], rstd = a.rstd[row];
    float s[2] = {0.0f, 0.0f};
    for (int q = threadIdx.x; q < a.vecs; q += LN_LONG_THREADS) {
      const RowVec<X, VEC> vx = load_row<X, VEC>(x + (long long)q * VEC);
      const RowVec<X, VEC> vg = load_row<X, VEC>(g + (long long)q * VEC);
      float w[VEC];
      load_param<P, VEC>(a.w, (long long)q * VEC, 1.0f, w);
#pragma unroll
      for (int j = 0; j < VEC; j++) {
        const float t = to_f32(vg.v[j]) * w[j];
        s[0] += t;
        s[1] += t * ((to_f32(vx.v[j]) - mean) * rstd);
      }
    }
    group_sum(s, LN_LONG_THREADS, red, turn);
    const float c0 = s[0] * a.inv_dim, c1 = s[1] * a.inv_dim;
    X* dx = reinterpret_cast<X*>(a.dx) + row * a.dx_stride;
    for (int q = threadIdx.x; q < a.vecs; q += LN_LONG_THREADS) {
      const RowVec<X, VEC> vx = load_row<X, VEC>(x + (long long)q * VEC);
      const RowVec<X, VEC> vg = load_row<X, VEC>(g + (long long)q * VEC);
      float w[VEC];
      load_param<P, VEC>(a.w, (long long)q * VEC, 1.0f, w);
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
template <typename P>
__global__ void __launch_bounds__(1024) ln_param_kernel(const float* __restrict__ part, int parts, int dim, P* dw,
                                                        P* db) {
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
    P* out = col < dim ? dw : db;
    if (out) out[col < dim ? col : col - dim] = from_f32<P>(v);
  }
}

// ------------------------------------------------------------------ host side
// Partial rows of dw and db: one per block; few where a row is long.
int max_parts(int64_t n, int64_t dim) { return (int)std::min<int64_t>(n, dim <= 2048 ? 148 * 4 : 148 * 2); }

// Threads per row: a warp (less for short rows) while a thread then holds at
// most `most` vectors, else as many warps as it takes. Returns 0 if a row does
// not fit `most` vectors of `limit` threads.
int group_of(int vecs, int most, int limit) {
  int g = 1;
  while (g < 32 && g < vecs) g <<= 1;
  while (g < limit && (vecs + g - 1) / g > most) g <<= 1;
  return (vecs + g - 1) / g <= most ? g : 0;
}

struct Shape {
  int group, block, rpb;
  unsigned int grid;
};
Shape shape_of(int group, int64_t n, int64_t max_blocks) {
  Shape s;
  s.group = group;
  s.block = std::max(group, group <= 32 ? LN_THREADS : group);
  s.rpb = s.block / group;
  s.grid = (unsigned int)std::max<int64_t>(1, std::min<int64_t>((n + s.rpb - 1) / s.rpb, max_blocks));
  return s;
}

template <typename X, typename P, int VEC, int K>
void launch_ln_k(LnArgs a, int group, int sms, cudaStream_t st) {
  const Shape s = shape_of(group, a.n, (int64_t)sms * 64);
  a.group = group;
  ln_kernel<X, P, VEC, K><<<s.grid, s.block, 0, st>>>(a);
}

template <typename X, typename P, int VEC>
void launch_ln(LnArgs a, int sms, cudaStream_t st) {
  constexpr int MOST = VEC == 1 ? 16 : 32 / VEC;
  a.vecs = a.dim / VEC;
  const int group = group_of(a.vecs, MOST, LN_MAX_GROUP);
  if (!group) {
    ln_long_kernel<X, P, VEC><<<(unsigned int)std::min<int64_t>(a.n, (int64_t)sms * 4), LN_LONG_THREADS, 0, st>>>(a);
  } else {
    const int k = (a.vecs + group - 1) / group;
    if (k <= 1)
      launch_ln_k<X, P, VEC, 1>(a, group, sms, st);
    else if (k <= 2)
      launch_ln_k<X, P, VEC, 2>(a, group, sms, st);
    else if (k <= 4)
      launch_ln_k<X, P, VEC, 4>(a, group, sms, st);
    else if constexpr (MOST > 4) {
      if (k <= 8)
        launch_ln_k<X, P, VEC, 8>(a, group, sms, st);
      else if constexpr (MOST > 8)
        launch_ln_k<X, P, VEC, 16>(a, group, sms, st);
    }
  }
  GIDS_CUDA(cudaGetLastError());
}

template <typename X, typename P, int VEC, int K>
void launch_ln_grad_k(LnGradArgs a, int group, cudaStream_t st, int* parts) {
  const Shape s = shape_of(group, a.n, max_parts(a.n, a.dim));
  a.group = group;
  const size_t smem = s.rpb > 1 ? (size_t)a.dim * 2 * sizeof(float) : 0;
  *parts = (int)s.grid;
  ln_grad_kernel<X, P, VEC, K><<<s.grid, s.block, smem, st>>>(a);
}

template <typename X, typename P, int VEC>
void launch_ln_grad(LnGradArgs a, P* dw, P* db, int sms, cudaStream_t st) {
  constexpr int MOST = VEC == 1 ? 8 : 16 / VEC;
  a.vecs = a.dim / VEC;
  int parts = 0;
  const int group = group_of(a.vecs, MOST, 512);
  if (!group) {
    if (a.part) {
      parts = (int)std::min<int64_t>(max_parts(a.n, a.dim), 64);
      const dim3 grid((unsigned int)parts, (unsigned int)((a.dim + LN_LONG_THREADS - 1) / LN_LONG_THREADS));
      ln_grad_cols_kernel<X><<<grid, LN_LONG_THREADS, 0, st>>>(a);
    }
    if (a.dx)  // last: dx may be written over x or grad
      ln_grad_long_kernel<X, P, VEC><<<(unsigned int)std::min<int64_t>(a.n, (int64_t)sms * 4), LN_LONG_THREADS, 0, st>>>(
          a);
  } else {
    const int k = (a.vecs + group - 1) / group;
    if (k <= 1)
      launch_ln_grad_k<X, P, VEC, 1>(a, group, st, &parts);
    else if (k <= 2)
      launch_ln_grad_k<X, P, VEC, 2>(a, group, st, &parts);
    else if constexpr (MOST > 2) {
      if (k <= 4)
        launch_ln_grad_k<X, P, VEC, 4>(a, group, st, &parts);
      else if constexpr (MOST > 4)
        launch_ln_grad_k<X, P, VEC, 8>(a, group, st, &parts);
    }
  }
  GIDS_CUDA(cudaGetLastError());
  if (a.part)
    ln_param_kernel<P><<<(unsigned int)((2ll * a.dim + 31) / 32), 1024, 0, st>>>(a.part, parts, a.dim, dw, db);
  GIDS_CUDA(cudaGetLastError());
}

void check_norm(int device, int64_t n, int64_t dim, int x_type, int param_type) {
  GIDS_CHECK(device >= 0, GIDS_E_INVAL, "bad device");
  GIDS_CHECK(n >= 0 && n < (1ll << 40), GIDS_E_INVAL, "n must be in [0, 2^40)");
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

template <typename X, typename P>
void ln_typed(LnArgs a, const Rows& y, const Rows& x, int pt, int sms, cudaStream_t st) {
  constexpr int BIG = 16 / (int)sizeof(X);
  if (vec_ok(y, a.dim, BIG) && vec_ok(x, a.dim, BIG) && param_ok(a.w, pt, BIG) && param_ok(a.b, pt, BIG))
    launch_ln<X, P, BIG>(a, sms, st);
  else
    launch_ln<X, P, 1>(a, sms, st);
}

template <typename X, typename P>
void ln_grad_typed(LnGradArgs a, const Rows& dx, const Rows& g, const Rows& x, int pt, void* dw, void* db, int sms,
                   cudaStream_t st) {
  constexpr int BIG = 16 / (int)sizeof(X);
  if (vec_ok(dx, a.dim, BIG) && vec_ok(g, a.dim, BIG) && vec_ok(x, a.dim, BIG) && param_ok(a.w, pt, BIG))
    launch_ln_grad<X, P, BIG>(a, static_cast<P*>(dw), static_cast<P*>(db), sms, st);
  else
    launch_ln_grad<X, P, 1>(a, static_cast<P*>(dw), static_cast<P*>(db), sms, st);
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
  const int sms = device_sms(device);
  if (x.type == GIDS_F32) return ln_typed<float, float>(a, y, x, param_type, sms, st);
  if (x.type == GIDS_F16) {
    if (param_type == GIDS_F32) return ln_typed<__half, float>(a, y, x, param_type, sms, st);
    return ln_typed<__half, __half>(a, y, x, param_type, sms, st);
  }
  if (param_type == GIDS_F32) return ln_typed<__nv_bfloat16, float>(a, y, x, param_type, sms, st);
  return ln_typed<__nv_bfloat16, __nv_bfloat16>(a, y, x, param_type, sms, st);
}

uint64_t layer_norm_grad_workspace(int64_t n, int64_t dim) {
  check_norm(0, n, dim, GIDS_F32, GIDS_F32);
  return (uint64_t)max_parts(n, dim) * 2 * (uint64_t)dim * sizeof(float);
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
  const bool params = dweight || dbias;
  if (params && n) {
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
  a.dx_stride = dx.stride;
  a.g_stride = grad.stride;
  a.x_stride = x.stride;
  a.n = n;
  a.dim = (int)dim;
  a.inv_dim = 1.0f / (float)dim;
  const int sms = device_sms(device);
  if (x.type == GIDS_F32) return ln_grad_typed<float, float>(a, dx, grad, x, param_type, dweight, dbias, sms, st);
  if (x.type == GIDS_F16) {
    if (param_type == GIDS_F32)
      return ln_grad_typed<__half, float>(a, dx, grad, x, param_type, dweight, dbias, sms, st);
    return ln_grad_typed<__half, __half>(a, dx, grad, x, param_type, dweight, dbias, sms, st);
  }
  if (param_type == GIDS_F32)
    return ln_grad_typed<__nv_bfloat16, float>(a, dx, grad, x, param_type, dweight, dbias, sms, st);
  return ln_grad_typed<__nv_bfloat16, __nv_bfloat16>(a, dx, grad, x, param_type, dweight, dbias, sms, st);
}

}  // namespace gids
