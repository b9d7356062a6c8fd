// group_norm_f32.cu -- the group norm kernels for fp32 features (a file per
// type, so that they compile side by side).
#include "group_norm.cuh"

namespace tcc {

void group_norm_f32(const GroupNormArgs& a, char* scratch, bool backward, cudaStream_t s) {
    norm_by_width<float>(a, scratch, backward, s);
}

}  // namespace tcc
