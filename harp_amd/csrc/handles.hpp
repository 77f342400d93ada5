// The C handles behind include/eclat_hip.h and what every entry point does with a C++ exception:
// shared by the translation units that implement the ABI.
#pragma once

#include <exception>
#include <memory>
#include <new>
#include <string>
#include <vector>

#include "../../include/eclat_hip.h"
#include "backend.hpp"

struct eh_device {
  eh::HipDevice dev;
  explicit eh_device(int i) : dev(i) {}
  eh_device(int i, hipStream_t s) : dev(i, s) {}
};
struct eh_buffer {
  eh::HipBuffer buf;
  eh_buffer(eh::HipDevice* d, size_t n) : buf(d, n) {}
};

namespace eh {

int fail(int code, const std::string& msg);    // records the calling thread's last error, returns the code
int classify(const std::string& msg);          // EH_ERR_* of an exception's text

template <class F> int guard(F&& f) {
  try {
    f();
    return EH_OK;
  } catch (const Error& e) {
    return fail(classify(e.what()), e.what());
  } catch (const std::bad_alloc&) {
    return fail(EH_ERR_INVALID, "out of host memory");
  } catch (const std::exception& e) {
    return fail(EH_ERR_INVALID, e.what());
  }
}

}  // namespace eh
