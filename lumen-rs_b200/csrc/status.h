// What kernels tell the host outside their outputs: words that they set, and the
// code and message that a handle's status call makes of them.
#pragma once

#include "lumen_cuda.h"

namespace lc {

enum StatusBit { kBadInput, kTimedOut, kStatusBits };  // each a word: kernels store, they need not agree on one

inline int status_code(const volatile int* words) {
  return words[kTimedOut] ? LC_ERR_TIMEOUT : words[kBadInput] ? LC_ERR_INVALID : LC_OK;
}

inline const char* status_message(int code) {
  return code == LC_ERR_TIMEOUT   ? "a copy into shared memory did not end in time: outputs of that call are NaN or without candidates"
         : code == LC_ERR_INVALID ? "a call met a length beyond its table, a page id outside the pool or a parent outside its group"
                                  : "";
}

}  // namespace lc
