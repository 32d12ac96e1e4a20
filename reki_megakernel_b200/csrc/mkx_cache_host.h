// Host helpers shared by the translation units of the paged episode cache.
#pragma once
#include <cuda_runtime.h>

namespace mkxc {

constexpr int MAX_DEVICES = 64;
extern thread_local const char* last_error;  // last CUDA error string of a cache entry point
bool cuda_ok(cudaError_t e);                 // records the string of a failure
int page_shift(int page_rows);               // log2 of a page size, -1 for sizes that are refused
int sm_count(int device);                    // 0: failed, or no device of 0 .. MAX_DEVICES - 1

}  // namespace mkxc
