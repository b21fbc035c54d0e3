// The library's error state: every int entry point returns 0 or a negative
// TF_E_* code and leaves the message for tf_last_error() (per thread).
#pragma once

#include <exception>
#include <new>
#include <string>

#include "tforge_hip.h"

namespace tfk {

// Keeps `m` for tf_last_error() and returns `code`.
int fail(int code, const std::string &m);

// Runs an entry point's body; a C++ exception (an allocation failure, say)
// becomes an error code and message instead of unwinding into the caller.
template <typename F>
int guarded(F &&body) {
  try {
    return body();
  } catch (const std::bad_alloc &) {
    return fail(TF_E_ARG, "out of host memory");
  } catch (const std::exception &e) {
    return fail(TF_E_ARG, std::string("internal error: ") + e.what());
  } catch (...) {
    return fail(TF_E_ARG, "internal error");
  }
}

}  // namespace tfk
