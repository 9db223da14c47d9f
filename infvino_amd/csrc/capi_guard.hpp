// What the C entry points share: exceptions become a status code and a thread-local message.
#pragma once

#include <hip/hip_runtime.h>

#include <cstring>
#include <exception>
#include <stdexcept>
#include <string>

#include "../../include/ivh.h"

namespace ivh {

std::string & last_error();  // of the calling thread

template <class F>
int guard(F && f)
{
  try {
    f();
    return IVH_OK;
  } catch (const std::invalid_argument & e) {
    last_error() = e.what();
    return IVH_ERR_INVALID;
  } catch (const std::runtime_error & e) {
    last_error() = e.what();
    return std::strncmp(e.what(), "HIP error", 9) == 0 ? IVH_ERR_DEVICE : IVH_ERR_INVALID;
  } catch (const std::exception & e) {
    last_error() = e.what();
    return IVH_ERR_INTERNAL;
  } catch (...) {
    last_error() = "unknown error";
    return IVH_ERR_INTERNAL;
  }
}

inline void check_launch(const char * what)
{
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) throw std::runtime_error(std::string("HIP error in ") + what + ": " + hipGetErrorString(e));
}

}  // namespace ivh
