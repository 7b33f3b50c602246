// Host helpers of tj_api.cu that the library's other translation units use.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace tj_host {

// Records the message for tj_last_error() on this thread and returns status.
int fail(int status, const char* fmt, ...) __attribute__((format(printf, 2, 3)));

// Current device (must be sm_100) and its SM count.
int device(int* index, int* sms);

// Row-major [rows, cols] matrix of elt_bytes-wide elements (1: uint8, 2: 16 bits, 4: float), box
// [box_rows, box_cols] with the 128-byte swizzle, zero fill past the edges.
int make_map(CUtensorMap* map, const void* base, int elt_bytes, uint64_t rows, uint64_t cols, uint32_t box_rows,
             uint32_t box_cols);

// tj_set_wait_limit's part for tj_train.cu (each translation unit's kernels read their own copy).
int set_train_wait_limit(unsigned long long ns);

}  // namespace tj_host

#define TJH_CUDA(call)                                                                              \
  do {                                                                                              \
    cudaError_t e_ = (call);                                                                        \
    if (e_ != cudaSuccess)                                                                          \
      return tj_host::fail(TJ_ERR_CUDA, "%s: %s (%s:%d)", #call, cudaGetErrorString(e_), __FILE__, __LINE__); \
  } while (0)

#define TJH_CHECK(status)       \
  do {                          \
    int s_ = (status);          \
    if (s_ != TJ_OK) return s_; \
  } while (0)
