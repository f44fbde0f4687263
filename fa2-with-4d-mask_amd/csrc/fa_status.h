// Status and argument checks shared by the files of the C ABI (defined in fa_api.cpp).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace fa {

int fail(int code, const char* fmt, ...);   // sets fa_last_error's text, returns code
bool aligned16(const void* p);
int check_operand(const char* name, const void* p, int64_t sb, int64_t st, int64_t sh);
int launch_status(hipError_t e, const char* what);
constexpr int64_t kCus = 256;
// Key ranges of the 256-row forward (fa_api.cpp).
int fwd_key_split(int64_t base, int64_t nt, int64_t rows, int D, bool prec, bool shared);

}  // namespace fa
