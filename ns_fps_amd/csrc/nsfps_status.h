// Statuses, messages and injected failures of the host library, shared by its
// translation units (defined in nsfps_host.cpp).  Not part of the C ABI.
#pragma once

#include "nsfps.h"

#include <hip/hip_runtime.h>

#include <exception>
#include <new>
#include <stdint.h>

namespace nsfps {

// Leaves the message for nsfps_last_error() and returns s.
nsfps_status fail(nsfps_status s, const char *fmt, ...);

// Failure injection (NSFPS_INJECT): the kinds of HIP operation, the one armed
// in the current call, and whether this operation is the one to fail.
enum InjectKind : int { kInjNone = 0, kInjAlloc, kInjLaunch, kInjCopy, kInjSync, kInjAny };
extern thread_local int g_inj_kind;
void arm_injection();
int op_kind(const char *expr);
hipError_t injected(int kind);

#define HIP_TRY(expr)                                                                        \
  do {                                                                                       \
    hipError_t e_ = g_inj_kind ? injected(op_kind(#expr)) : hipSuccess;                      \
    const bool inj_ = e_ != hipSuccess;                                                      \
    if (!inj_) {                                                                             \
      e_ = (expr);                                                                           \
    }                                                                                        \
    if (e_ != hipSuccess)                                                                    \
      return fail(e_ == hipErrorOutOfMemory ? NSFPS_ENOMEM : NSFPS_EDEVICE, "%s: %s (%s:%d)", \
                  #expr, inj_ ? "injected failure (NSFPS_INJECT)" : hipGetErrorString(e_),   \
                  __FILE__, __LINE__);                                                       \
  } while (0)

// No C++ exception crosses the C ABI: host allocation failures and any other
// exception become a status with a message.
template <class F>
nsfps_status guarded(F &&f) {
  try {
    arm_injection();
    return f();
  } catch (const std::bad_alloc &) {
    return fail(NSFPS_ENOMEM, "host allocation failed");
  } catch (const std::exception &e) {
    return fail(NSFPS_EDEVICE, "internal error: %s", e.what());
  } catch (...) {
    return fail(NSFPS_EDEVICE, "internal error");
  }
}

}  // namespace nsfps
