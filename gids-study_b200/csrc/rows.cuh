// Device helpers of the row kernels (embedding.cu, layer_norm.cu): element
// types, vector loads and stores of rows, and a division by a launch constant.
// Arithmetic is float32 throughout; a value is rounded to its type once, when
// it is stored (round to nearest even).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

namespace gids {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) {
  return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

// VEC consecutive elements, moved in pieces of at most 16 bytes; the address
// is aligned to min(16, sizeof(T) * VEC).
template <typename T, int VEC>
struct alignas(sizeof(T) * VEC < 16 ? sizeof(T) * VEC : 16) RowVec {
  T v[VEC];
};

template <int BYTES>
struct Piece;
template <>
struct Piece<2> {
  using type = unsigned short;
};
template <>
struct Piece<4> {
  using type = unsigned int;
};
template <>
struct Piece<8> {
  using type = uint2;
};
template <>
struct Piece<16> {
  using type = uint4;
};

template <typename T, int VEC>
__device__ __forceinline__ RowVec<T, VEC> load_vec(const T* p) {
  constexpr int B = sizeof(T) * VEC < 16 ? (int)sizeof(T) * VEC : 16;
  using P = typename Piece<B>::type;
  constexpr int N = (int)sizeof(T) * VEC / B;
  RowVec<T, VEC> r;
#pragma unroll
  for (int i = 0; i < N; i++) reinterpret_cast<P*>(&r)[i] = __ldg(reinterpret_cast<const P*>(p) + i);
  return r;
}

// The same for rows that are read once, and that the kernel may overwrite
// (a coherent load, which evicts first).
template <typename T, int VEC>
__device__ __forceinline__ RowVec<T, VEC> load_row(const T* p) {
  constexpr int B = sizeof(T) * VEC < 16 ? (int)sizeof(T) * VEC : 16;
  using P = typename Piece<B>::type;
  constexpr int N = (int)sizeof(T) * VEC / B;
  RowVec<T, VEC> r;
#pragma unroll
  for (int i = 0; i < N; i++) reinterpret_cast<P*>(&r)[i] = __ldcs(reinterpret_cast<const P*>(p) + i);
  return r;
}

template <typename T, int VEC>
__device__ __forceinline__ void store_raw(T* p, const RowVec<T, VEC>& r) {
  constexpr int B = sizeof(T) * VEC < 16 ? (int)sizeof(T) * VEC : 16;
  using P = typename Piece<B>::type;
  constexpr int N = (int)sizeof(T) * VEC / B;
  if constexpr (N == 2) {
    // 32 bytes in one instruction where they are aligned: two stores of 16 bytes
    // leave a warp's sectors half written each
    if ((reinterpret_cast<uintptr_t>(p) & 31) == 0) {
      const unsigned long long* v = reinterpret_cast<const unsigned long long*>(&r);
      asm volatile("st.global.v4.b64 [%0], {%1, %2, %3, %4};" ::"l"(p), "l"(v[0]), "l"(v[1]), "l"(v[2]), "l"(v[3])
                   : "memory");
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < N; i++) reinterpret_cast<P*>(p)[i] = reinterpret_cast<const P*>(&r)[i];
}

// The same for results that are not read again soon: they leave the L2 cache first.
template <typename T, int VEC>
__device__ __forceinline__ void store_stream(T* p, const RowVec<T, VEC>& r) {
  constexpr int B = sizeof(T) * VEC < 16 ? (int)sizeof(T) * VEC : 16;
  using P = typename Piece<B>::type;
  constexpr int N = (int)sizeof(T) * VEC / B;
#pragma unroll
  for (int i = 0; i < N; i++) __stcs(reinterpret_cast<P*>(p) + i, reinterpret_cast<const P*>(&r)[i]);
}

template <typename T, int VEC>
__device__ __forceinline__ void store_vec(T* p, const float (&v)[VEC]) {
  RowVec<T, VEC> r;
#pragma unroll
  for (int i = 0; i < VEC; i++) r.v[i] = from_f32<T>(v[i]);
  store_raw(p, r);
}

// Asynchronous copy of 16 bytes to shared memory; zeros instead, and nothing
// read, where `on` is false.
__device__ __forceinline__ void copy_async(void* smem, const void* gmem, bool on) {
  const unsigned int dst = (unsigned int)__cvta_generic_to_shared(smem);
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(gmem), "r"(on ? 16 : 0) : "memory");
}
// The first `bytes` of 16, and zeros behind them.
__device__ __forceinline__ void copy_async_tail(void* smem, const void* gmem, int bytes) {
  const unsigned int dst = (unsigned int)__cvta_generic_to_shared(smem);
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(gmem), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory");
}

// Blocks of a cluster and their shared memory.
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}
// the address of `p` (of this block's shared memory) in block `rank` of the cluster
__device__ __forceinline__ unsigned int peer(const void* p, unsigned int rank) {
  unsigned int r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
               : "=r"(r)
               : "r"((unsigned int)__cvta_generic_to_shared(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ unsigned int peer_load(const unsigned int* p, unsigned int rank) {
  unsigned int v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(peer(p, rank)) : "memory");
  return v;
}

// Two float32 values in one register pair: sm_100a adds, multiplies and fuses
// both with one instruction, each half rounded as the scalar instruction does.
struct F2 {
  unsigned long long v;
  F2() = default;
  __device__ __forceinline__ F2(float lo, float hi) {
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi));
  }
  __device__ __forceinline__ explicit F2(float both) : F2(both, both) {}
  __device__ __forceinline__ float lo() const { return __uint_as_float((unsigned int)v); }
  __device__ __forceinline__ float hi() const { return __uint_as_float((unsigned int)(v >> 32)); }
};
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}

// Elements 2 p and 2 p + 1 of K vectors laid end to end.
template <typename T, int VEC, int K>
__device__ __forceinline__ F2 pair_of(const RowVec<T, VEC> (&v)[K], int p) {
  if constexpr (VEC >= 2 && sizeof(T) == 2) {
    const unsigned int u = reinterpret_cast<const unsigned int*>(&v[2 * p / VEC])[(2 * p % VEC) / 2];
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      return F2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u));
      return F2(f.x, f.y);
    }
  } else {
    return F2(to_f32(v[2 * p / VEC].v[2 * p % VEC]), to_f32(v[(2 * p + 1) / VEC].v[(2 * p + 1) % VEC]));
  }
}

// n / d for 32-bit n by a multiplication (d >= 1 fixed at launch): with
// l = ceil(log2 d) and m = floor(2^32 (2^l - d) / d) + 1,
// n / d = (t + ((n - t) >> min(l, 1))) >> max(l - 1, 0), t = mulhi(m, n)
// (Granlund and Montgomery, "Division by invariant integers using
// multiplication", PLDI 1994).
struct FastDiv {
  unsigned int d = 1, m = 1, s1 = 0, s2 = 0;
  FastDiv() = default;
  explicit FastDiv(unsigned int div) : d(div) {
    unsigned int l = 0;
    while (l < 32 && (1ull << l) < div) l++;
    m = (unsigned int)((((1ull << l) - div) << 32) / div + 1ull);
    s1 = l < 1 ? l : 1;
    s2 = l < 1 ? 0 : l - 1;
  }
  __device__ __forceinline__ unsigned int div(unsigned int n) const {
    const unsigned int t = __umulhi(m, n);
    return (t + ((n - t) >> s1)) >> s2;
  }
};

}  // namespace gids
