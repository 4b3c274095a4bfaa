// The error type of the library's host code and the text behind s1c_create_error(), shared by the
// translation units.
#pragma once
#include <cuda_runtime.h>

#include <stdexcept>
#include <string>

#include "../../include/s1c.h"

namespace s1c {

struct S1cError : std::runtime_error {
  s1c_status code;
  S1cError(s1c_status c, const std::string& m) : std::runtime_error(m), code(c) {}
};

// Sets the calling thread's s1c_create_error() text (defined in s1c.cu).
void set_create_error(const char* text);

}  // namespace s1c

#define CK(call)                                                                                  \
  do {                                                                                            \
    cudaError_t e_ = (call);                                                                      \
    if (e_ != cudaSuccess)                                                                        \
      throw s1c::S1cError(S1C_ERR_CUDA, std::string(#call) + ": " + cudaGetErrorString(e_));     \
  } while (0)
