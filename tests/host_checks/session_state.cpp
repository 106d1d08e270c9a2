// What the tests of a session's inner state reach into: addresses of its error word and of its arrival counts, and a step that
// fails.  Built by the test against the package's own headers.
#include <functional>
#include <map>
#include <memory>
#include <mutex>
#include <set>
#include <string>
#include <unordered_map>
#include <vector>

#include <cuda_runtime.h>

#define private public
#include "../../oxionnx_b200/csrc/abi_internal.hpp"
#undef private

extern "C" {

int* error_word(oxb200_ctx* ctx) { return ctx->impl.session->err_flag_; }

uint32_t arrival_counts(oxb200_ctx* ctx, void** ptr, uint64_t* bytes, uint32_t most) {
  const auto& all = ctx->impl.session->arrival_counts_;
  for (uint32_t i = 0; i < all.size() && i < most; ++i) ptr[i] = all[i].ptr, bytes[i] = all[i].bytes;
  return (uint32_t)all.size();
}

void add_failing_step(oxb200_ctx* ctx) {
  oxb::Step st;
  st.launch = [](cudaStream_t) { throw oxb::Error{OXB200_FAILED, "a step that fails"}; };
  ctx->impl.session->steps_.push_back(st);
}
void drop_last_step(oxb200_ctx* ctx) { ctx->impl.session->steps_.pop_back(); }

}  // extern "C"
