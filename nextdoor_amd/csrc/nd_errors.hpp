// How every C entry reports failure: a return code, and a text for nd_last_error().
#pragma once

#include <exception>
#include <new>
#include <string>

namespace nd {

// One per host thread, shared by all translation units of the library.
inline std::string& last_error_text() {
  static thread_local std::string text;
  return text;
}

inline int fail(const std::string& msg, int code = -1) {
  last_error_text() = msg;
  return code;
}

// No exception leaves the library: a body that throws (host memory, a container's range
// check) reports through the error text like any other failure.
template <class Body>
int guarded(Body body) {
  try {
    return body();
  } catch (const std::bad_alloc&) {
    return fail("out of host memory");
  } catch (const std::exception& e) {
    return fail(std::string("internal error: ") + e.what());
  } catch (...) {
    return fail("internal error");
  }
}

}  // namespace nd
