// sb_error.h -- host helpers shared by the library's translation units.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace sb {

// Store the calling thread's message for sb_last_error() and return `code`.
int fail(int code, const char* fmt, ...);
int cuda_fail(cudaError_t e, const char* what);

// Streaming multiprocessors of a device (looked up once per device).
int sm_count(int dev, int* out);

inline bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

}  // namespace sb
