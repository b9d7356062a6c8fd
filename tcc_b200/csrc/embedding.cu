// embedding.cu -- rows of a learned table by index, scaled, and the table's
// gradient summed by sorted index.
//
//   out[i, :]   = scale * table[idx[i], :]            (padding, out of range: 0)
//   dtable[v,:] = scale * sum over i with idx[i] = v, ascending i, of dout[i, :]
//
// Both are bound by memory: one product or sum per element moved.
#include "elem.cuh"
#include "primitives.cuh"
#include "train_ops.cuh"

#include <algorithm>

namespace tcc {

namespace {

constexpr uint32_t kMaxWidth = 1u << 20;

__device__ __forceinline__ int64_t load_index(const void* idx, int type, uint64_t i) {
    return type == TCC_I64 ? __ldg(static_cast<const long long*>(idx) + i)
                           : (int64_t)__ldg(static_cast<const int*>(idx) + i);
}

// ---------------------------------------------------------------- lookup --

constexpr int kLookupThreads = 256;
constexpr int kLookupUnroll = 4;

// A CTA owns `tile` consecutive rows of the output and walks their packs in
// memory order, so stores are contiguous at any width; the four loads of a
// step are independent.
template <typename TT, typename TO, int V>
__global__ void __launch_bounds__(kLookupThreads) lookup_kernel(
    const TT* __restrict__ table, uint64_t ldt, uint64_t num_rows, const void* __restrict__ idx,
    int idx_type, uint64_t n, int64_t padding, float scale, TO* __restrict__ out, uint64_t ldo,
    uint32_t packs, uint32_t tile, uint64_t div_magic, uint32_t* __restrict__ bad) {
    const uint64_t row0 = (uint64_t)blockIdx.x * tile;
    const uint32_t rows = (uint32_t)min((uint64_t)tile, n - row0);
    const uint32_t total = rows * packs;
    for (uint32_t base = threadIdx.x; base < total; base += kLookupThreads * kLookupUnroll) {
        Pack<TT, V> val[kLookupUnroll];
        uint32_t r[kLookupUnroll], c[kLookupUnroll];
        int64_t id[kLookupUnroll];
#pragma unroll
        for (int u = 0; u < kLookupUnroll; ++u) {
            const uint32_t q = base + u * kLookupThreads;
            r[u] = tile == 1 ? 0 : (uint32_t)((q * div_magic) >> 32);
            c[u] = q - r[u] * packs;
            id[u] = q < total ? load_index(idx, idx_type, row0 + r[u]) : -1;
        }
#pragma unroll
        for (int u = 0; u < kLookupUnroll; ++u) {
            const uint32_t q = base + u * kLookupThreads;
            if (q >= total) continue;
            const bool inside = id[u] >= 0 && (uint64_t)id[u] < num_rows;
            if (inside && id[u] != padding) {
                val[u] = load_pack_nc<TT, V>(table + (uint64_t)id[u] * ldt + (uint64_t)c[u] * V);
            } else {
#pragma unroll
                for (int k = 0; k < V; ++k) val[u].v[k] = from_f32<TT>(0.f);
                if (!inside && id[u] != padding && c[u] == 0 && bad) atomicExch(bad, 1u);
            }
        }
#pragma unroll
        for (int u = 0; u < kLookupUnroll; ++u) {
            const uint32_t q = base + u * kLookupThreads;
            if (q >= total) continue;
            // padded rows are zero whatever the scale (an infinite scale too)
            const bool zero = id[u] == padding || id[u] < 0 || (uint64_t)id[u] >= num_rows;
            Pack<TO, V> o;
#pragma unroll
            for (int k = 0; k < V; ++k)
                o.v[k] = from_f32<TO>(zero ? 0.f : to_f32(val[u].v[k]) * scale);
            store_pack_cs<TO, V>(out + (row0 + r[u]) * ldo + (uint64_t)c[u] * V, o);
        }
    }
}

template <typename TT, typename TO, int V>
void launch_lookup(const EmbeddingArgs& a, cudaStream_t s) {
    const uint32_t packs = a.F / V;
    // about eight packs a thread; whole rows per CTA
    const uint32_t tile = std::max(1u, (uint32_t)(kLookupThreads * 8) / packs);
    const uint64_t blocks = (a.n + tile - 1) / tile;
    TCC_REQUIRE(blocks < (1ull << 31), "too many indices for one call");
    const uint64_t magic = (1ull << 32) / packs + 1;  // exact for q < tile * packs <= 2048, or tile 1
    lookup_kernel<TT, TO, V><<<(unsigned)blocks, kLookupThreads, 0, s>>>(
        static_cast<const TT*>(a.table), a.ldt, a.num_rows, a.idx, a.idx_type, a.n, a.padding,
        a.scale, static_cast<TO*>(a.rows), a.ldr, packs, tile, magic, a.bad);
    TCC_CUDA(cudaGetLastError());
}

template <typename TT, typename TO>
void lookup_by_width(const EmbeddingArgs& a, cudaStream_t s) {
    VecRule rule;
    rule.count(a.F);
    rule.count(a.ldt);
    rule.count(a.ldr);
    rule.pointer(a.table, sizeof(TT));
    rule.pointer(a.rows, sizeof(TO));
    switch (rule.width()) {
        case 8:
            if constexpr (sizeof(TT) == 2 && sizeof(TO) == 2) launch_lookup<TT, TO, 8>(a, s);
            break;
        case 4: launch_lookup<TT, TO, 4>(a, s); break;
        case 2: launch_lookup<TT, TO, 2>(a, s); break;
        default: launch_lookup<TT, TO, 1>(a, s);
    }
}

// -------------------------------------------------------------- gradient --

// Sort keys: the table row, or num_rows for an index that has no row.
__global__ void grad_keys_kernel(const void* __restrict__ idx, int idx_type, uint64_t n,
                                 uint64_t num_rows, int64_t padding, uint64_t* __restrict__ keys,
                                 uint32_t* __restrict__ vals, uint32_t* __restrict__ bad) {
    const uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= n) return;
    const int64_t id = load_index(idx, idx_type, i);
    const bool inside = id >= 0 && (uint64_t)id < num_rows;
    if (!inside && id != padding && bad) atomicExch(bad, 1u);
    keys[i] = inside && id != padding ? (uint64_t)id : num_rows;
    vals[i] = (uint32_t)i;
}

__device__ __forceinline__ uint32_t lower_bound(const uint64_t* keys, uint32_t n, uint64_t v) {
    uint32_t lo = 0, hi = n;
    while (lo < hi) {
        const uint32_t mid = (lo + hi) >> 1;
        if (keys[mid] < v) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}

// A warp per table row: its run of the sorted keys, summed in order.
template <typename TG, typename TT, int V>
__global__ void __launch_bounds__(256) grad_rows_kernel(
    const TG* __restrict__ grad, uint64_t ldg, const uint64_t* __restrict__ keys,
    const uint32_t* __restrict__ order, uint32_t n, float scale, TT* __restrict__ dtable,
    uint64_t ldt, uint64_t num_rows, uint32_t packs) {
    const int lane = threadIdx.x & 31;
    const uint64_t warps = ((uint64_t)gridDim.x * blockDim.x) >> 5;
    for (uint64_t v = ((uint64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5; v < num_rows; v += warps) {
        const uint32_t lo = lower_bound(keys, n, v), hi = lower_bound(keys, n, v + 1);
        for (uint32_t c = lane; c < packs; c += 32) {
            float acc[V];
#pragma unroll
            for (int k = 0; k < V; ++k) acc[k] = 0.f;
            for (uint32_t j = lo; j < hi; ++j) {
                const Pack<TG, V> g = load_pack_cs<TG, V>(grad + (uint64_t)order[j] * ldg + (uint64_t)c * V);
#pragma unroll
                for (int k = 0; k < V; ++k) acc[k] += to_f32(g.v[k]);
            }
            Pack<TT, V> o;
#pragma unroll
            for (int k = 0; k < V; ++k) o.v[k] = from_f32<TT>(acc[k] * scale);
            store_pack<TT, V>(dtable + v * ldt + (uint64_t)c * V, o);
        }
    }
}

uint64_t align256(uint64_t b) { return (b + 255) / 256 * 256; }

template <typename TG, typename TT, int V>
void launch_grad(const EmbeddingArgs& a, const uint64_t* keys, const uint32_t* order, cudaStream_t s) {
    const unsigned blocks = (unsigned)std::min<uint64_t>((a.num_rows + 7) / 8, 148 * 64);
    grad_rows_kernel<TG, TT, V><<<blocks, 256, 0, s>>>(
        static_cast<const TG*>(a.rows), a.ldr, keys, order, (uint32_t)a.n, a.scale,
        static_cast<TT*>(a.table), a.ldt, a.num_rows, a.F / V);
    TCC_CUDA(cudaGetLastError());
}

template <typename TG, typename TT>
void grad_by_width(const EmbeddingArgs& a, const uint64_t* keys, const uint32_t* order, cudaStream_t s) {
    VecRule rule;
    rule.count(a.F);
    rule.count(a.ldt);
    rule.count(a.ldr);
    rule.pointer(a.table, sizeof(TT));
    rule.pointer(a.rows, sizeof(TG));
    switch (rule.width()) {
        case 8:
            if constexpr (sizeof(TT) == 2 && sizeof(TG) == 2) launch_grad<TG, TT, 8>(a, keys, order, s);
            break;
        case 4: launch_grad<TG, TT, 4>(a, keys, order, s); break;
        case 2: launch_grad<TG, TT, 2>(a, keys, order, s); break;
        default: launch_grad<TG, TT, 1>(a, keys, order, s);
    }
}

// fn(table type tag, row type tag); the rows are of the table's type or fp32.
template <typename Fn>
void with_types(const EmbeddingArgs& a, Fn&& fn) {
    const bool same = a.row_type == a.table_type;
    if (a.table_type == TCC_F32) fn(float{}, float{});
    else if (a.table_type == TCC_F16) same ? fn(__half{}, __half{}) : fn(__half{}, float{});
    else same ? fn(__nv_bfloat16{}, __nv_bfloat16{}) : fn(__nv_bfloat16{}, float{});
}

void check_embedding(const EmbeddingArgs& a) {
    TCC_REQUIRE(valid_type(a.table_type) && valid_type(a.row_type), "unknown element type");
    TCC_REQUIRE(a.row_type == a.table_type || a.row_type == TCC_F32,
                "rows must have the table's type or fp32");
    TCC_REQUIRE(a.idx_type == TCC_I32 || a.idx_type == TCC_I64, "unknown index type");
    TCC_REQUIRE(a.F > 0 && a.F <= kMaxWidth, "F must be in [1, 2^20]");
    TCC_REQUIRE(a.ldt >= a.F && a.ldr >= a.F, "row strides must be >= F");
    TCC_REQUIRE(a.n < (1ull << 31) && a.num_rows < (1ull << 31),
                "fewer than 2^31 indices and table rows are supported");
    TCC_REQUIRE(a.n == 0 || (a.idx && a.rows), "indices and rows must not be NULL");
    TCC_REQUIRE(a.num_rows == 0 || a.table, "the table must not be NULL");
    TCC_REQUIRE((uintptr_t)a.table % type_bytes(a.table_type) == 0 &&
                    (uintptr_t)a.rows % type_bytes(a.row_type) == 0 &&
                    (uintptr_t)a.idx % (a.idx_type == TCC_I64 ? 8 : 4) == 0,
                "a pointer is not aligned to its element type");
}

}  // namespace

void embedding_forward(const EmbeddingArgs& a, cudaStream_t s) {
    check_embedding(a);
    if (a.n == 0) return;
    with_types(a, [&](auto tt, auto to) { lookup_by_width<decltype(tt), decltype(to)>(a, s); });
}

size_t embedding_backward_scratch_bytes(uint64_t n, uint64_t num_rows, uint32_t F) {
    (void)num_rows;
    (void)F;
    return (size_t)(2 * align256(n * 8) + 2 * align256(n * 4) + radix_tmp_bytes(n) + 256);
}

void embedding_backward(const EmbeddingArgs& a, void* scratch, size_t scratch_bytes, cudaStream_t s) {
    check_embedding(a);
    if (a.num_rows == 0) return;
    TCC_REQUIRE(scratch && (uintptr_t)scratch % 256 == 0, "scratch must be 256-byte aligned");
    if (scratch_bytes < embedding_backward_scratch_bytes(a.n, a.num_rows, a.F))
        throw Error(TCC_ERR_CAPACITY, "scratch is smaller than tcc_embedding_backward_scratch_bytes");
    char* p = static_cast<char*>(scratch);
    uint64_t* keys = reinterpret_cast<uint64_t*>(p);
    uint64_t* keys2 = reinterpret_cast<uint64_t*>(p += align256(a.n * 8));
    uint32_t* vals = reinterpret_cast<uint32_t*>(p += align256(a.n * 8));
    uint32_t* vals2 = reinterpret_cast<uint32_t*>(p += align256(a.n * 4));
    void* tmp = p + align256(a.n * 4);
    bool alt = false;
    if (a.n) {
        grad_keys_kernel<<<ceil_div(a.n, 256), 256, 0, s>>>(a.idx, a.idx_type, a.n, a.num_rows, a.padding,
                                                            keys, vals, a.bad);
        TCC_CUDA(cudaGetLastError());
        alt = radix_sort_pairs(keys, vals, keys2, vals2, a.n, bits_for(a.num_rows + 1), tmp, s);
    }
    const uint64_t* k = alt ? keys2 : keys;
    const uint32_t* o = alt ? vals2 : vals;
    with_types(a, [&](auto tt, auto tg) { grad_by_width<decltype(tg), decltype(tt)>(a, k, o, s); });
}

}  // namespace tcc
