// Error reporting of the C-ABI entry points.
#ifndef OS_ERROR_H_
#define OS_ERROR_H_

#include <hip/hip_runtime.h>

#include <string>

#include "../../include/os_mcts.h"

namespace osx {

// Thread-local message of the last failed C-ABI call (os_last_error).
extern thread_local std::string g_err;
inline int Fail(int code, const std::string& msg) {
  g_err = msg;
  return code;
}

}  // namespace osx

#define HIP_TRY(expr)                                                        \
  do {                                                                       \
    hipError_t _e = (expr);                                                  \
    if (_e != hipSuccess)                                                    \
      return ::osx::Fail(OS_ERR_DEVICE, std::string(#expr " failed: ") +    \
                                            hipGetErrorString(_e));          \
  } while (0)

#endif  // OS_ERROR_H_
