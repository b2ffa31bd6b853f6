// paged_attn_q8.cuh: the flat form of e4m3 codes.
#include "paged_attn_q8.cuh"

namespace engpt {
namespace paged {

int launch_flat_e4m3(const Q8AttnArgs& a, int Hkv, bool f32, cudaStream_t st) {
  return f32 ? launch_flat<E4m3Code, float>(a, Hkv, st) : launch_flat<E4m3Code, __nv_bfloat16>(a, Hkv, st);
}

}  // namespace paged
}  // namespace engpt
