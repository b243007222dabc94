// Host-side helpers shared by the C-ABI translation units of libsafattn.so
// (defined in saf_capi.hip).
#pragma once
#include "saf_attn.h"
#include "saf_kernels.h"

namespace saf {

// Sets the calling thread's error message and returns `code`.
int fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
bool present(const saf_tensor_t& t);
int elem_size(int dtype);
const char* dtype_name(int dtype);
bool supported_hd(int64_t hd);
int cu_count();
int launched(hipError_t e, const char* what);

}  // namespace saf
