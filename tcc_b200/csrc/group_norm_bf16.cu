// group_norm_bf16.cu -- the group norm kernels for bf16 features (a file per
// type, so that they compile side by side).
#include "group_norm.cuh"

namespace tcc {

void group_norm_bf16(const GroupNormArgs& a, char* scratch, bool backward, cudaStream_t s) {
    norm_by_width<__nv_bfloat16>(a, scratch, backward, s);
}

}  // namespace tcc
