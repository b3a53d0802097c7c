// Status and message plumbing of the C entry points: no exception leaves one,
// and the last failure of a thread is what duck_last_error() returns there.
#pragma once
#include "../../include/duck_b200.h"

#include <cuda_runtime.h>

#include <stdexcept>
#include <string>

namespace duckb200 {

inline thread_local std::string lastError;

struct CudaError : std::runtime_error {
  using std::runtime_error::runtime_error;
};
inline void check(cudaError_t e, const char *what) {
  if (e != cudaSuccess) throw CudaError(std::string(what) + ": " + cudaGetErrorString(e));
}
inline void require(bool c, const char *msg) {
  if (!c) throw std::invalid_argument(msg);
}

template <class F> int guarded(F &&f) {
  try {
    f();
    return DUCK_OK;
  } catch (const std::invalid_argument &e) {
    lastError = e.what();
    return DUCK_EINVAL;
  } catch (const CudaError &e) {
    lastError = e.what();
    return DUCK_ECUDA;
  } catch (const std::exception &e) {
    lastError = e.what();
    return DUCK_EMODEL;
  }
}

}  // namespace duckb200
