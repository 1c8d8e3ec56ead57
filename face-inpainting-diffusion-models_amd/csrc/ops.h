// Host-side pieces shared by the operators of include/ifd_ops.h.
#pragma once
#include "../../include/ifd_ops.h"
#include "common.h"

namespace ifd {

inline int64_t dtype_bytes(int dt) { return dt == IFD_F32 ? 4 : 2; }
inline bool dtype_ok(int dt) { return dt == IFD_F32 || dt == IFD_BF16 || dt == IFD_F16; }
inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// An entry point refuses a call: the message names it.
#define IFD_OP_REQUIRE(cond, msg)                                                        \
  do {                                                                                   \
    if (!(cond)) {                                                                       \
      ::ifd::set_error(std::string(__func__) + ": " + (msg));                            \
      return 2;                                                                          \
    }                                                                                    \
  } while (0)

// p is null or starts on a multiple of n bytes
inline bool on(const void* p, int64_t n) { return ((uintptr_t)p & (uintptr_t)(n - 1)) == 0; }

// The checks that both directions of attention share; nullptr, or what is wrong.
const char* attention_check(const ifd_attention_args& a);

}  // namespace ifd
