// What every C entry point shares: the calling thread's last error and the translation of
// exceptions to hllm_status (none crosses the boundary).
#pragma once

#include <exception>
#include <new>
#include <string>

#include "common.hpp"

namespace hllm_rocm {

// The message of the calling thread's last failed call.
std::string& last_error();

template <typename F>
hllm_status guarded(F&& f) {
  try {
    f();
    return HLLM_OK;
  } catch (const Failure& e) {
    last_error() = e.what();
    return e.status;
  } catch (const std::bad_alloc&) {
    last_error() = "host allocation failed";
    return HLLM_RESOURCE_EXHAUSTED;
  } catch (const std::exception& e) {
    last_error() = e.what();
    return HLLM_INTERNAL;
  } catch (...) {
    last_error() = "unknown failure";
    return HLLM_INTERNAL;
  }
}

}  // namespace hllm_rocm
