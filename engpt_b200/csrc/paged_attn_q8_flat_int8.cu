// paged_attn_q8.cuh: the flat form of int8 codes.
#include "paged_attn_q8.cuh"

namespace engpt {
namespace paged {

int launch_flat_int8(const Q8AttnArgs& a, int Hkv, bool f32, cudaStream_t st) {
  return f32 ? launch_flat<Int8Code, float>(a, Hkv, st) : launch_flat<Int8Code, __nv_bfloat16>(a, Hkv, st);
}

}  // namespace paged
}  // namespace engpt
