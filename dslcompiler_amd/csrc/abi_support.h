// abi_support.h -- what the C entry points outside llk_abi.cpp share with it:
// the thread's error message, the device check and the library's workspaces.
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>

#include "llk/llk_abi.h"

namespace llk {

// Records the calling thread's message and returns `code`.
int setError(int code, const char* msg);

// The current device, verified to be gfx950.
int current_gfx950(int* dev);

// A workspace of `bytes` for one call: the caller's (ctx->scratch) or the
// library's own of ctx's stream.  end() gives it back once the call's
// launches are enqueued.
class CallWorkspace {
 public:
  int begin(int dev, size_t bytes, llk_kernel_context* ctx);
  void end();
  void* ptr() const { return ptr_; }

 private:
  int dev_ = -1;
  void* ptr_ = nullptr;
  void* held_ = nullptr;
  hipStream_t stream_ = nullptr;
};

}  // namespace llk
