// The calling thread's error message, shared by the files of the C ABI.
#pragma once

#include <cstring>

namespace fa {

// Sets the message fa_sm75_last_error returns; the result is `status`.
int capi_fail(int status, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
char* capi_error_buffer();  // kCapiErrorBytes long
constexpr int kCapiErrorBytes = 512;
inline void capi_clear_error() { capi_error_buffer()[0] = '\0'; }

// Puts the message back as it was.
struct SavedError {
  char message[kCapiErrorBytes];
  SavedError() { std::memcpy(message, capi_error_buffer(), kCapiErrorBytes); }
  ~SavedError() { std::memcpy(capi_error_buffer(), message, kCapiErrorBytes); }
};

}  // namespace fa
