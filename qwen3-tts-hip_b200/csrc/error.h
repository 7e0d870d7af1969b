// Errors of the C entry points: a QttsError carries the qtts_status that the
// call returns; guard() turns exceptions into a status and a message for
// qtts_last_error().
#pragma once

#include <cuda_runtime.h>

#include <new>
#include <stdexcept>
#include <string>

#include "qtts_b200.h"

namespace qtts {

std::string& last_error();  // of the calling thread

struct QttsError : std::runtime_error {
  int code;
  QttsError(int c, const std::string& m) : std::runtime_error(m), code(c) {}
};
[[noreturn]] inline void fail(int code, const std::string& m) { throw QttsError(code, m); }
[[noreturn]] inline void invalid(const std::string& m) { fail(QTTS_ERR_INVALID_INPUT, m); }

#define QCK(expr)                                                                     \
  do {                                                                                \
    cudaError_t e_ = (expr);                                                          \
    if (e_ != cudaSuccess)                                                            \
      ::qtts::fail(QTTS_ERR_CUDA, std::string(#expr) + ": " + cudaGetErrorString(e_)); \
  } while (0)

template <typename F>
int32_t guard(F&& f) {
  try {
    f();
    return QTTS_OK;
  } catch (const QttsError& e) {
    last_error() = e.what();
    return e.code;
  } catch (const std::bad_alloc&) {
    last_error() = "out of host memory";
    return QTTS_ERR_CUDA;
  } catch (const std::exception& e) {
    last_error() = e.what();
    return QTTS_ERR_INVALID_INPUT;
  }
}

inline void need(const void* p, const char* what) {
  if (!p) invalid(std::string(what) + " must not be null");
}

}  // namespace qtts
