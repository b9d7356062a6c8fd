// group_norm_f16.cu -- the group norm kernels for fp16 features (a file per
// type, so that they compile side by side).
#include "group_norm.cuh"

namespace tcc {

void group_norm_f16(const GroupNormArgs& a, char* scratch, bool backward, cudaStream_t s) {
    norm_by_width<__half>(a, scratch, backward, s);
}

}  // namespace tcc
