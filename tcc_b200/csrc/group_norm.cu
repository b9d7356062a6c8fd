// group_norm.cu -- group norm with an activation: scratch, checks and the
// choice of the element type's kernels (group_norm.cuh).
#include "group_norm.cuh"

namespace tcc {

void group_norm_f32(const GroupNormArgs& a, char* scratch, bool backward, cudaStream_t s);
void group_norm_f16(const GroupNormArgs& a, char* scratch, bool backward, cudaStream_t s);
void group_norm_bf16(const GroupNormArgs& a, char* scratch, bool backward, cudaStream_t s);

// The most that any vector width and element type would take, so that the
// size depends neither on the type nor on the pointers' alignment.
size_t group_norm_scratch_bytes(uint64_t N, uint64_t S, uint32_t C, uint32_t G, bool backward) {
    if (N == 0 || S == 0 || C == 0 || G == 0 || C % G) return 0;
    const uint64_t stats = 2 * align256(N * G * 4);
    uint64_t bytes = 0;
    for (int V = 1; V <= 8 && (C / G) % V == 0; V <<= 1)
        for (uint32_t es = 2; es <= 4 && es * V <= 16; es += 2) {
            if (rows_form(S, C, G, V)) {
                if (backward) bytes = std::max(bytes, rows_blocks(rows_shape(S, C, G, V), N, G) * S * 2 * C * 4);
                continue;
            }
            const SplitShape held = resident_shape(N, S, C, G, V, es * V, backward ? 2 : 1);
            if (held.chunks) {
                if (backward) bytes = std::max(bytes, resident_grid(N, held.chunks) * 2 * C * 4);
                continue;
            }
            const SplitShape sh = split_shape(N, S, C, G, V);
            bytes = std::max(bytes, backward ? split_grad_plan(N, C, G, sh).bytes
                                             : stats + align256(N * sh.chunks * G * sh.SUB * sizeof(Moments)));
        }
    return (size_t)bytes;
}

namespace {

void check_norm(const GroupNormArgs& a, void* scratch, size_t scratch_bytes, bool backward) {
    TCC_REQUIRE(valid_type(a.type), "unknown element type");
    TCC_REQUIRE(valid_type(a.param_type), "unknown parameter type");
    TCC_REQUIRE(a.act >= TCC_ACT_NONE && a.act <= TCC_ACT_GELU, "unknown activation");
    TCC_REQUIRE(a.C > 0 && a.G > 0 && a.C % a.G == 0, "C must be a positive multiple of G");
    TCC_REQUIRE(a.C <= (1u << 20), "at most 2^20 channels");
    TCC_REQUIRE(a.N < (1ull << 31) && a.S < (1ull << 31), "fewer than 2^31 samples and rows");
    TCC_REQUIRE(a.eps >= 0.f, "eps must not be negative");
    if (a.N == 0 || a.S == 0) return;
    const uint32_t es = type_bytes(a.type), ps = type_bytes(a.param_type);
    TCC_REQUIRE(a.x && (uintptr_t)a.x % es == 0 && a.ldx >= a.C, "x: NULL, misaligned, or a stride below C");
    TCC_REQUIRE((uintptr_t)a.weight % ps == 0 && (uintptr_t)a.bias % ps == 0 && (uintptr_t)a.dweight % ps == 0 &&
                    (uintptr_t)a.dbias % ps == 0,
                "a parameter is not aligned to its type");
    if (backward) {
        TCC_REQUIRE(a.dy && (uintptr_t)a.dy % es == 0 && a.lddy >= a.C, "dy: NULL, misaligned, or a stride below C");
        TCC_REQUIRE((uintptr_t)a.dx % es == 0 && (!a.dx || a.lddx >= a.C), "dx: misaligned, or a stride below C");
        TCC_REQUIRE(a.mean && a.rstd, "mean and rstd must not be NULL");
    } else {
        TCC_REQUIRE(a.y && (uintptr_t)a.y % es == 0 && a.ldy >= a.C, "y: NULL, misaligned, or a stride below C");
        TCC_REQUIRE(!a.mean == !a.rstd, "give both mean and rstd, or neither");
    }
    const size_t need = group_norm_scratch_bytes(a.N, a.S, a.C, a.G, backward);
    if (need == 0) return;
    TCC_REQUIRE(scratch && (uintptr_t)scratch % 256 == 0, "scratch must be 256-byte aligned");
    if (scratch_bytes < need)
        throw Error(TCC_ERR_CAPACITY, "scratch is smaller than tcc_group_norm_scratch_bytes");
}

void norm_by_type(const GroupNormArgs& a, void* scratch, bool backward, cudaStream_t s) {
    char* p = static_cast<char*>(scratch);
    if (a.type == TCC_F32) group_norm_f32(a, p, backward, s);
    else if (a.type == TCC_F16) group_norm_f16(a, p, backward, s);
    else group_norm_bf16(a, p, backward, s);
}

}  // namespace

void group_norm_forward(const GroupNormArgs& a, void* scratch, size_t scratch_bytes, cudaStream_t s) {
    check_norm(a, scratch, scratch_bytes, false);
    if (a.N == 0 || a.S == 0) return;
    norm_by_type(a, scratch, false, s);
}

void group_norm_backward(const GroupNormArgs& a, void* scratch, size_t scratch_bytes, cudaStream_t s) {
    check_norm(a, scratch, scratch_bytes, true);
    if (a.N == 0 || a.S == 0) {  // nothing reaches the parameters
        const size_t bytes = (size_t)a.C * type_bytes(a.param_type);
        if (a.dweight) TCC_CUDA(cudaMemsetAsync(a.dweight, 0, bytes, s));
        if (a.dbias) TCC_CUDA(cudaMemsetAsync(a.dbias, 0, bytes, s));
        return;
    }
    norm_by_type(a, scratch, true, s);
}

}  // namespace tcc
