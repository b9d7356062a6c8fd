// clip.cu -- the 2-norm of all gradients of a model, and their clipping.
//
//   norm = sqrt(sum over tensors and elements of g^2)
//   g *= min(1, max_norm / (norm + eps))
//
// Bound by memory: the norm reads every gradient once, the clipping reads and
// writes it once.  The tensors' addresses travel in the kernel's parameters,
// so a call copies nothing to the device first and can be captured in a graph.
// Every CTA writes one partial sum in a fixed order and the sums are added in a
// fixed order: the same gradients give the same norm, bit for bit.
#include "elem.cuh"
#include "train_ops.cuh"

#include <algorithm>
#include <vector>

namespace tcc {

namespace {

constexpr int kThreads = 256;
constexpr uint32_t kChunkBytes = 32768;  // of one tensor, for one CTA at a time
// One CTA clips up to TCC_CLIP_SMALL_BYTES: teams of kTeam threads, a shorter
// chunk each.  At 150 KB in four tensors a call then takes 15.3 us of host time
// (which is what counts outside a graph) in place of 17.6, and 5.2 us of the GPU
// in place of 3.9; the GPU's side grows with the bytes (6.8 against 4.3 us at
// 256 KB), so the limit lies where a launch's worth is used up.
constexpr int kOneThreads = 1024, kTeam = 128;
constexpr uint32_t kOneChunkBytes = 8192;
constexpr uint32_t kMaxBlocks = 148 * 8;

// Tensors of a launch: over few of them its parameters are short (0.7, 2.7 and
// 10 KB).
constexpr int kSmall = TCC_CLIP_SMALL_TENSORS, kMiddle = 128, kLarge = 480;

// K tensors of one launch; chunk i of the launch belongs to the tensor t with
// first[t] <= i < first[t + 1].
template <int K>
struct TensorTable {
    uint32_t count, chunk_bytes;
    void* data[K];
    uint64_t n[K];
    uint32_t first[K + 1];
    uint8_t type[K];
};

struct Span {
    void* data;  // first element of the chunk
    uint32_t n;  // elements
    int type;
};

template <int K>
__device__ __forceinline__ Span chunk_span(const TensorTable<K>& t, uint32_t chunk) {
    uint32_t lo = 0, hi = t.count;  // last tensor with first <= chunk
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) >> 1;
        if (t.first[mid] <= chunk) lo = mid;
        else hi = mid;
    }
    Span s;
    s.type = t.type[lo];
    const uint32_t bytes = s.type == TCC_F32 ? 4 : 2;
    const uint64_t per = t.chunk_bytes / bytes, at = (uint64_t)(chunk - t.first[lo]) * per;
    s.data = static_cast<char*>(t.data[lo]) + at * bytes;
    s.n = (uint32_t)min(per, t.n[lo] - at);
    return s;
}

// Sum of squares of one pack.  fp32 inside a pack where that is safe; where a
// square could leave fp32's range (or all are zero) the pack is summed in
// 64 bits, so a norm of 1e30 or 1e-30 comes out right.
template <typename T, int V>
__device__ __forceinline__ double pack_squares(const Pack<T, V>& p) {
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < V; ++k) {
        const float v = to_f32(p.v[k]);
        s = fmaf(v, v, s);
    }
    if (s > 1e-25f && s < 1e37f) return (double)s;
    double d = 0.0;
#pragma unroll
    for (int k = 0; k < V; ++k) {
        const double v = (double)to_f32(p.v[k]);
        d += v * v;
    }
    return d;
}

template <int THREADS>
__device__ __forceinline__ double block_sum(double v) {
    __shared__ double ws[THREADS / 32];
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) == 0) ws[threadIdx.x >> 5] = v;
    __syncthreads();
    double t = 0.0;
#pragma unroll
    for (int i = 0; i < THREADS / 32; ++i) t += ws[i];
    __syncthreads();
    return t;
}

// Elements before the first 16-byte boundary.
__device__ __forceinline__ uint32_t head_of(const void* p, uint32_t n, uint32_t bytes) {
    const uint32_t off = (uint32_t)(reinterpret_cast<uintptr_t>(p) & 15u);
    return min(n, off ? (16 - off) / bytes : 0u);
}

template <typename T, int THREADS>
__device__ __forceinline__ double span_squares(const Span& sp) {
    constexpr int V = 16 / sizeof(T);
    const uint32_t tid = threadIdx.x % THREADS;
    const T* p = static_cast<const T*>(sp.data);
    const uint32_t head = head_of(p, sp.n, sizeof(T));
    const uint32_t packs = (sp.n - head) / V, body = head + packs * V;
    double s = 0.0;
#pragma unroll 4
    for (uint32_t q = tid; q < packs; q += THREADS)
        s += pack_squares<T, V>(load_pack<T, V>(p + head + (uint64_t)q * V));
    if (tid < head) s += pack_squares<T, 1>(load_pack<T, 1>(p + tid));
    if (body + tid < sp.n) s += pack_squares<T, 1>(load_pack<T, 1>(p + body + tid));
    return s;
}

template <int THREADS>
__device__ __forceinline__ double squares_of(const Span& sp) {
    if (sp.type == TCC_F32) return span_squares<float, THREADS>(sp);
    if (sp.type == TCC_F16) return span_squares<__half, THREADS>(sp);
    return span_squares<__nv_bfloat16, THREADS>(sp);
}

template <int K>
__global__ void __launch_bounds__(kThreads) squares_kernel(const __grid_constant__ TensorTable<K> t,
                                                           double* partial, bool add) {
    after_previous();
    double s = 0.0;
    const uint32_t chunks = t.first[t.count];
    for (uint32_t c = blockIdx.x; c < chunks; c += gridDim.x) {
        const Span sp = chunk_span<K>(t, c);
        s += squares_of<kThreads>(sp);
    }
    s = block_sum<kThreads>(s);
    if (threadIdx.x == 0) partial[blockIdx.x] = add ? partial[blockIdx.x] + s : s;
}

__device__ __forceinline__ float norm_of(const double* partial, uint32_t blocks) {
    double s = 0.0;
    for (uint32_t i = threadIdx.x; i < blocks; i += kThreads) s += partial[i];
    return (float)sqrt(block_sum<kThreads>(s));
}

__global__ void __launch_bounds__(kThreads) norm_kernel(const double* partial, uint32_t blocks, float* norm) {
    after_previous();
    const float n = norm_of(partial, blocks);
    if (threadIdx.x == 0) *norm = n;
}

template <typename T, int THREADS>
__device__ __forceinline__ void span_scale(const Span& sp, float f) {
    constexpr int V = 16 / sizeof(T);
    const uint32_t tid = threadIdx.x % THREADS;
    T* p = static_cast<T*>(sp.data);
    const uint32_t head = head_of(p, sp.n, sizeof(T));
    const uint32_t packs = (sp.n - head) / V, body = head + packs * V;
#pragma unroll 4
    for (uint32_t q = tid; q < packs; q += THREADS) {
        Pack<T, V> v = load_pack<T, V>(p + head + (uint64_t)q * V);
#pragma unroll
        for (int k = 0; k < V; ++k) v.v[k] = from_f32<T>(to_f32(v.v[k]) * f);
        store_pack<T, V>(p + head + (uint64_t)q * V, v);
    }
    if (tid < head) p[tid] = from_f32<T>(to_f32(p[tid]) * f);
    if (body + tid < sp.n) {
        T* e = p + body + tid;
        *e = from_f32<T>(to_f32(*e) * f);
    }
}

// A factor of 1 changes no value.  One that is NaN spreads, as a NaN norm should,
// but for 0 / 0, where there is nothing to clip.
__device__ __forceinline__ bool must_scale(float norm, float factor) {
    return factor < 1.f || (factor != factor && norm != 0.f);
}

template <int THREADS>
__device__ __forceinline__ void scale_by(const Span& sp, float f) {
    if (sp.type == TCC_F32) span_scale<float, THREADS>(sp, f);
    else if (sp.type == TCC_F16) span_scale<__half, THREADS>(sp, f);
    else span_scale<__nv_bfloat16, THREADS>(sp, f);
}

// Scales in the reverse of the order in which the norm was read: what was read
// last is still in L2.  partial == NULL: the norm is read from norm_in.
template <int K>
__global__ void __launch_bounds__(kThreads) scale_kernel(const __grid_constant__ TensorTable<K> t,
                                                         const double* partial, uint32_t blocks,
                                                         const float* norm_in, float* norm_out, float max_norm,
                                                         float eps) {
    after_previous();
    const float norm = partial ? norm_of(partial, blocks) : *norm_in;
    if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = norm;
    const float f = max_norm / (norm + eps);
    if (!must_scale(norm, f)) return;
    const uint32_t chunks = t.first[t.count];
    for (uint32_t i = blockIdx.x; i < chunks; i += gridDim.x) {
        const Span sp = chunk_span<K>(t, chunks - 1 - i);
        scale_by<kThreads>(sp, f);
    }
}

// Norm and clipping of few bytes by one CTA: one launch in place of two, and
// the second reading comes from the SM's own cache.
__global__ void __launch_bounds__(kOneThreads) clip_one_kernel(const __grid_constant__ TensorTable<kSmall> t,
                                                               float* norm_out, float max_norm, float eps) {
    double s = 0.0;
    const uint32_t chunks = t.first[t.count];
    for (uint32_t c = threadIdx.x / kTeam; c < chunks; c += kOneThreads / kTeam)
        s += squares_of<kTeam>(chunk_span<kSmall>(t, c));
    const float norm = (float)sqrt(block_sum<kOneThreads>(s)), f = max_norm / (norm + eps);
    if (threadIdx.x == 0) *norm_out = norm;
    if (!must_scale(norm, f)) return;
    for (uint32_t c = threadIdx.x / kTeam; c < chunks; c += kOneThreads / kTeam)
        scale_by<kTeam>(chunk_span<kSmall>(t, c), f);
}

// Fills a table from the tensors at `at` on (empty ones are skipped); returns
// where the next launch starts.
template <int K>
uint32_t fill(const tcc_tensor* t, uint32_t count, uint32_t at, TensorTable<K>& out,
              uint32_t chunk_bytes = kChunkBytes) {
    out.count = 0;
    out.chunk_bytes = chunk_bytes;
    uint64_t chunks = 0;
    for (; at < count && out.count < (uint32_t)K; ++at) {
        if (t[at].n == 0) continue;
        const uint64_t per = chunk_bytes / type_bytes(t[at].type);
        const uint64_t c = (t[at].n + per - 1) / per;
        if (chunks + c >= (1ull << 32)) {
            TCC_REQUIRE(out.count, "a tensor is too large");
            break;
        }
        out.data[out.count] = t[at].data;
        out.n[out.count] = t[at].n;
        out.type[out.count] = (uint8_t)t[at].type;
        out.first[out.count++] = (uint32_t)chunks;
        chunks += c;
    }
    out.first[out.count] = (uint32_t)chunks;
    return at;
}

void check_tensors(const tcc_tensor* t, uint32_t count, bool written) {
    TCC_REQUIRE(count == 0 || t, "tensors must not be NULL");
    for (uint32_t i = 0; i < count; ++i) {
        TCC_REQUIRE(valid_type(t[i].type), "unknown element type");
        TCC_REQUIRE(t[i].n == 0 || (t[i].data && (uintptr_t)t[i].data % type_bytes(t[i].type) == 0),
                    "a tensor is NULL or not aligned to its type");
        TCC_REQUIRE(t[i].n < (1ull << 46), "a tensor is too large");
    }
    if (!written) return;
    // a value that two tensors share would be scaled twice, by two CTAs at once
    std::vector<std::pair<uintptr_t, uintptr_t>> spans;
    for (uint32_t i = 0; i < count; ++i)
        if (t[i].n)
            spans.emplace_back((uintptr_t)t[i].data, (uintptr_t)t[i].data + t[i].n * type_bytes(t[i].type));
    if (!std::is_sorted(spans.begin(), spans.end())) std::sort(spans.begin(), spans.end());
    for (size_t i = 1; i < spans.size(); ++i)
        TCC_REQUIRE(spans[i - 1].second <= spans[i].first, "two tensors share memory");
}

// fn(table) for each launch's tensors.
template <int K, typename Fn>
void each_launch_of(const tcc_tensor* t, uint32_t count, Fn&& fn) {
    TensorTable<K> tab;
    for (uint32_t at = 0; at < count;) {
        at = fill<K>(t, count, at, tab);
        if (tab.count) fn(tab);
    }
}
template <typename Fn>
void each_launch(const tcc_tensor* t, uint32_t count, Fn&& fn) {
    if (count <= (uint32_t)kSmall) each_launch_of<kSmall>(t, count, fn);
    else if (count <= (uint32_t)kMiddle) each_launch_of<kMiddle>(t, count, fn);
    else each_launch_of<kLarge>(t, count, fn);
}

template <int K>
void launch_squares(const TensorTable<K>& tab, double* partial, unsigned blocks, bool add, cudaStream_t s) {
    if (add) {
        launch_after(squares_kernel<K>, blocks, kThreads, 0, s, tab, partial, add);
    } else {
        squares_kernel<K><<<blocks, kThreads, 0, s>>>(tab, partial, add);
        TCC_CUDA(cudaGetLastError());
    }
}

// Partial sums of every tensor; returns how many there are.
uint32_t squares(const tcc_tensor* t, uint32_t count, double* partial, cudaStream_t s) {
    uint32_t blocks = 0;
    each_launch(t, count, [&](const auto& tab) {
        const uint32_t chunks = tab.first[tab.count];
        // a later launch adds to the partial sums of the first, so all use its grid
        if (blocks == 0) {
            blocks = std::min(chunks, kMaxBlocks);
            launch_squares(tab, partial, blocks, false, s);
        } else {
            launch_squares(tab, partial, blocks, true, s);
        }
    });
    return blocks;
}

double* partials(void* scratch, size_t scratch_bytes) {
    TCC_REQUIRE(scratch && (uintptr_t)scratch % 256 == 0, "scratch must be 256-byte aligned");
    if (scratch_bytes < grad_norm_scratch_bytes())
        throw Error(TCC_ERR_CAPACITY, "scratch is smaller than tcc_grad_norm_scratch_bytes");
    return static_cast<double*>(scratch);
}

template <int K>
void scale_after(const TensorTable<K>& tab, unsigned grid, const double* partial, uint32_t blocks,
                 const float* norm_in, float* norm_out, float max_norm, float eps, cudaStream_t s) {
    launch_after(scale_kernel<K>, grid, kThreads, 0, s, tab, partial, blocks, norm_in, norm_out, max_norm, eps);
}

void scale(const tcc_tensor* t, uint32_t count, const double* partial, uint32_t blocks, const float* norm_in,
           float* norm_out, float max_norm, float eps, cudaStream_t s) {
    each_launch(t, count, [&](const auto& tab) {
        const unsigned grid = std::min(tab.first[tab.count], kMaxBlocks);
        scale_after(tab, grid, partial, blocks, norm_in, norm_out, max_norm, eps, s);
    });
}

void check_clip(float max_norm, float eps) {
    TCC_REQUIRE(max_norm >= 0.f, "max_norm must not be negative");
    TCC_REQUIRE(eps >= 0.f, "eps must not be negative");
}

}  // namespace

size_t grad_norm_scratch_bytes() { return kMaxBlocks * sizeof(double); }

void grad_norm(const tcc_tensor* t, uint32_t count, float* norm, void* scratch, size_t scratch_bytes,
               cudaStream_t s) {
    check_tensors(t, count, false);
    TCC_REQUIRE(norm, "norm must not be NULL");
    double* partial = partials(scratch, scratch_bytes);
    const uint32_t blocks = squares(t, count, partial, s);
    launch_after(norm_kernel, 1, kThreads, 0, s, partial, blocks, norm);
}

void clip_grads_with_norm(const tcc_tensor* t, uint32_t count, const float* norm, float max_norm, float eps,
                          cudaStream_t s) {
    check_tensors(t, count, true);
    check_clip(max_norm, eps);
    TCC_REQUIRE(norm, "norm must not be NULL");
    scale(t, count, nullptr, 0, norm, nullptr, max_norm, eps, s);
}

void clip_grad_norm(const tcc_tensor* t, uint32_t count, float max_norm, float eps, float* norm, void* scratch,
                    size_t scratch_bytes, cudaStream_t s) {
    check_tensors(t, count, true);
    check_clip(max_norm, eps);
    TCC_REQUIRE(norm, "norm must not be NULL");
    uint64_t bytes = 0;
    for (uint32_t i = 0; i < count; ++i) bytes += t[i].n * type_bytes(t[i].type);
    if (bytes == 0) {  // no elements: the norm is 0
        TCC_CUDA(cudaMemsetAsync(norm, 0, sizeof(float), s));
        return;
    }
    if (count <= (uint32_t)kSmall && bytes <= TCC_CLIP_SMALL_BYTES) {
        TensorTable<kSmall> tab;
        fill<kSmall>(t, count, 0, tab, kOneChunkBytes);
        clip_one_kernel<<<1, kOneThreads, 0, s>>>(tab, norm, max_norm, eps);
        TCC_CUDA(cudaGetLastError());
        return;
    }
    double* partial = partials(scratch, scratch_bytes);
    const uint32_t blocks = squares(t, count, partial, s);
    scale(t, count, partial, blocks, nullptr, norm, max_norm, eps, s);
}

}  // namespace tcc
