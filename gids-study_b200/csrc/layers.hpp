// Host side of the input-layer operators (embedding.cu, layer_norm.cu), called
// by the C ABI (abi.cpp). Every function checks its arguments before it
// touches the GPU and throws gids::Error.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>
#include <string>

#include "gids_internal.hpp"

namespace gids {

// A matrix of rows in device memory: `stride` elements from row to row, the
// columns of a row consecutive.
struct Rows {
  void* p = nullptr;
  int type = 0;        // GIDS_F32, GIDS_F16 or GIDS_BF16
  int64_t stride = 0;  // elements
};

inline int type_bytes(int type) { return type == GIDS_F32 ? 4 : 2; }

// Device word in mapped host memory that the embedding kernels of `device` set
// when an id lies outside its table; allocated on first use, for the process.
int* id_error_word(int device);
// Throws GIDS_E_RANGE, once, if an earlier embedding call on `device` met one.
void check_id_errors(int device);

void embedding(int device, Rows out, Rows weight, int64_t num_rows, int64_t dim, const void* ids, int id_bytes,
               int64_t n, float scale, cudaStream_t st);
uint64_t embedding_grad_workspace(int64_t n, int64_t num_rows, int64_t dim);
void embedding_grad(int device, Rows dweight, int64_t num_rows, int64_t dim, Rows grad, const void* ids, int id_bytes,
                    int64_t n, int64_t padding_idx, float scale, void* ws, uint64_t ws_bytes, cudaStream_t st);
void embedding_group(int device, const void* ids, int id_bytes, int64_t n, int64_t num_rows, int64_t padding_idx,
                     int64_t dim, void* ws, uint64_t ws_bytes, uint64_t* count_dev, uint64_t* count_host,
                     cudaStream_t st);
void embedding_grad_rows(int device, int64_t* rows, Rows values, int64_t capacity, int64_t num_rows, int64_t dim,
                         Rows grad, int64_t n, float scale, void* ws, uint64_t ws_bytes, cudaStream_t st);
void embedding_grad_distinct(int device, int64_t* rows, Rows values, int64_t capacity, int64_t num_rows, int64_t dim,
                             Rows grad, const void* ids, int id_bytes, int64_t n, int64_t padding_idx, float scale,
                             void* ws, uint64_t ws_bytes, uint64_t* count_host, cudaStream_t st);
void embedding_check(int device, cudaStream_t st);

void layer_norm(int device, Rows y, float* mean, float* rstd, Rows x, const void* weight, const void* bias,
                int param_type, int64_t n, int64_t dim, float eps, cudaStream_t st);
uint64_t layer_norm_grad_workspace(int64_t n, int64_t dim);
void layer_norm_grad(int device, Rows dx, void* dweight, void* dbias, Rows grad, Rows x, const float* mean,
                     const float* rstd, const void* weight, int param_type, int64_t n, int64_t dim, void* ws,
                     uint64_t ws_bytes, cudaStream_t st);

// ------------------------------------------------------------- for the above
inline void check_rows(const Rows& r, const char* what, int64_t n, int64_t dim, bool output) {
  GIDS_CHECK(r.type == GIDS_F32 || r.type == GIDS_F16 || r.type == GIDS_BF16, GIDS_E_INVAL,
             std::string(what) + ": unknown element type");
  GIDS_CHECK(r.stride >= 0, GIDS_E_INVAL, std::string(what) + ": negative row stride");
  GIDS_CHECK(n == 0 || r.p, GIDS_E_INVAL, std::string(what) + " is null");
  GIDS_CHECK(((uintptr_t)r.p) % (uintptr_t)type_bytes(r.type) == 0, GIDS_E_INVAL,
             std::string(what) + ": address not aligned to its elements");
  GIDS_CHECK(!output || n <= 1 || r.stride >= dim, GIDS_E_INVAL,
             std::string(what) + ": rows of an output must not overlap (row stride < dim)");
}

// Whether rows of `r` can be moved in vectors of `vec` elements: dim, stride
// and address are multiples of the vector (of 16 bytes where it is longer).
inline bool vec_ok(const Rows& r, int64_t dim, int vec) {
  const int64_t b = (int64_t)type_bytes(r.type) * vec;
  const int64_t a = b < 16 ? b : 16;
  return dim % vec == 0 && (r.stride * type_bytes(r.type)) % a == 0 && ((uintptr_t)r.p) % (uintptr_t)a == 0;
}

// Lets `kernel` use `bytes` of dynamic shared memory on the current device.
// What was allowed is remembered, for the runtime's call costs more than a launch.
void allow_smem(const void* kernel, size_t bytes);

inline int device_sms(int dev) {
  int sms = 0;
  GIDS_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
  return sms;
}

}  // namespace gids
