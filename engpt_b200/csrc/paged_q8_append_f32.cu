// paged_q8_append.cu: fp32 rows.
#include "paged_q8_store.cuh"

namespace engpt {
namespace paged {

int launch_append_f32(const StoreArgs& a, int code, bool vec, cudaStream_t st) {
  return launch_store<float, true>(a, code, vec, "qkv_append_q8", st);
}

}  // namespace paged
}  // namespace engpt
