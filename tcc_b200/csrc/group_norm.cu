// group_norm.cu -- group norm over channels-last features, then an activation,
// and its backward.
//
// x is [N samples, S rows, C channels], G groups of Cg = C / G neighbouring
// channels.  Per (sample, group), over its m = S * Cg values:
//   mean, var = population moments;  rstd = 1 / sqrt(var + eps)
//   h = (x - mean) * rstd;  z = h * weight[c] + bias[c];  y = act(z)
// Backward, with dz = dy * act'(z):
//   dbias[c] = sum dz;  dweight[c] = sum dz * h   (over samples and rows)
//   dx = rstd * (dz * weight - (a + h * b) / m),
//   a = sum over the group of dz * weight,  b = sum of dz * weight * h
// All of it is bound by memory.  The variance is taken around a mean, never as
// the difference of two large sums: moments of small blocks, each around its
// own mean, are merged pairwise (Chan, Golub and LeVeque, 1979).
//
// Two forms:
//  * rows  (S = 1, a group within a warp): every group of a row is reduced by
//    a few lanes of one warp, x is read once.
//  * split (any other): the rows of a sample are cut into chunks, a CTA each;
//    moments (or channel sums) per chunk, a merge over the chunks, and a
//    second pass that normalises, in reverse order, so that what the first
//    pass read last is still in L2.
#include "elem.cuh"
#include "train_ops.cuh"

#include <algorithm>

namespace tcc {

namespace {

constexpr int kThreads = 256;
constexpr uint64_t kSms = 148;

// ------------------------------------------------------------ activation --

__device__ __forceinline__ float sigmoid(float z) { return __fdividef(1.f, 1.f + expf(-z)); }

template <int V>
__device__ __forceinline__ void activate(int act, float (&z)[V]) {
    if (act == TCC_ACT_RELU) {
#pragma unroll
        for (int k = 0; k < V; ++k) z[k] = z[k] <= 0.f ? 0.f : z[k];
    } else if (act == TCC_ACT_SILU) {
#pragma unroll
        for (int k = 0; k < V; ++k) z[k] *= sigmoid(z[k]);
    } else if (act == TCC_ACT_GELU) {
#pragma unroll
        for (int k = 0; k < V; ++k) z[k] *= 0.5f * (1.f + erff(z[k] * 0.70710678118654752f));
    }
}

// d *= act'(z)
template <int V>
__device__ __forceinline__ void activate_grad(int act, const float (&z)[V], float (&d)[V]) {
    if (act == TCC_ACT_RELU) {
#pragma unroll
        for (int k = 0; k < V; ++k) d[k] = z[k] <= 0.f ? 0.f : d[k];
    } else if (act == TCC_ACT_SILU) {
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const float s = sigmoid(z[k]);
            d[k] *= s * (1.f + z[k] * (1.f - s));
        }
    } else if (act == TCC_ACT_GELU) {
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const float cdf = 0.5f * (1.f + erff(z[k] * 0.70710678118654752f));
            d[k] *= cdf + z[k] * 0.39894228040143268f * expf(-0.5f * z[k] * z[k]);
        }
    }
}

// ------------------------------------------------------------- rows form --

// A slot is L lanes (a power of two) that hold one group of one row as J packs
// each; a CTA's 256 / L slots are GB groups x RB rows.  A thread keeps its
// group for the whole kernel: its parameters and their gradients stay in
// registers.
struct RowsShape {
    uint32_t L, GB, RB, packs;  // packs: of one group
};

template <int U>
__device__ __forceinline__ void lane_sum(float (&v)[U], uint32_t L) {
    for (uint32_t o = L >> 1; o; o >>= 1) {
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] += __shfl_xor_sync(0xffffffffu, v[u], o);
    }
}

template <int V>
__device__ __forceinline__ void load_params(const GroupNormArgs& a, uint64_t c, bool on, float (&w)[V],
                                            float (&b)[V]) {
#pragma unroll
    for (int k = 0; k < V; ++k) {
        w[k] = on && a.weight ? load_typed(a.weight, a.param_type, c + k) : 1.f;
        b[k] = on && a.bias ? load_typed(a.bias, a.param_type, c + k) : 0.f;
    }
}

template <typename T, int V, int J, int U>
__global__ void __launch_bounds__(kThreads) rows_forward_kernel(const GroupNormArgs a, const RowsShape sh) {
    const uint32_t slot = threadIdx.x / sh.L, lane = threadIdx.x % sh.L;
    const uint32_t g = blockIdx.y * sh.GB + slot % sh.GB, rb = slot / sh.GB;
    const bool on = rb < sh.RB && g < a.G;
    const uint32_t Cg = a.C / a.G;
    const float inv = 1.f / (float)Cg;
    const T* x = static_cast<const T*>(a.x);
    T* y = static_cast<T*>(a.y);
    bool ok[J];
    uint64_t c[J];
    float w[J][V], b[J][V];
#pragma unroll
    for (int j = 0; j < J; ++j) {
        const uint32_t p = j * sh.L + lane;
        ok[j] = on && p < sh.packs;
        c[j] = (uint64_t)g * Cg + (uint64_t)p * V;
        load_params<V>(a, c[j], ok[j], w[j], b[j]);
    }
    const uint64_t stride = (uint64_t)gridDim.x * sh.RB;
    for (uint64_t row0 = (uint64_t)blockIdx.x * sh.RB; row0 < a.N; row0 += stride * U) {
        float v[U][J][V], s[U], q[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint64_t row = row0 + u * stride + rb;
#pragma unroll
            for (int j = 0; j < J; ++j) {
                Pack<T, V> pk;
                const bool in = ok[j] && row < a.N;
                if (in) pk = load_pack_cs<T, V>(x + row * a.ldx + c[j]);
#pragma unroll
                for (int k = 0; k < V; ++k) v[u][j][k] = in ? to_f32(pk.v[k]) : 0.f;
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            s[u] = 0.f;
#pragma unroll
            for (int j = 0; j < J; ++j)
#pragma unroll
                for (int k = 0; k < V; ++k) s[u] += v[u][j][k];
        }
        lane_sum<U>(s, sh.L);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            s[u] *= inv;
            q[u] = 0.f;
#pragma unroll
            for (int j = 0; j < J; ++j)
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    v[u][j][k] -= s[u];
                    q[u] += ok[j] ? v[u][j][k] * v[u][j][k] : 0.f;
                }
        }
        lane_sum<U>(q, sh.L);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint64_t row = row0 + u * stride + rb;
            const float r = __frsqrt_rn(q[u] * inv + a.eps);
            if (on && row < a.N && lane == 0 && a.mean) {
                a.mean[row * a.G + g] = s[u];
                a.rstd[row * a.G + g] = r;
            }
#pragma unroll
            for (int j = 0; j < J; ++j) {
                if (!ok[j] || row >= a.N) continue;
                float z[V];
#pragma unroll
                for (int k = 0; k < V; ++k) z[k] = v[u][j][k] * r * w[j][k] + b[j][k];
                activate<V>(a.act, z);
                Pack<T, V> o;
#pragma unroll
                for (int k = 0; k < V; ++k) o.v[k] = from_f32<T>(z[k]);
                store_pack_cs<T, V>(y + row * a.ldy + c[j], o);
            }
        }
    }
}

// Parameter gradients: a thread's sums over its rows (kept in two levels, so
// that the rounding error does not grow with the number of rows), then over
// the CTA's RB rows in shared memory; one partial row per CTA of the grid's x.
template <typename T, int V, int J, int U>
__global__ void __launch_bounds__(kThreads) rows_backward_kernel(const GroupNormArgs a, const RowsShape sh,
                                                                 float* __restrict__ partial) {
    const uint32_t slot = threadIdx.x / sh.L, lane = threadIdx.x % sh.L;
    const uint32_t g = blockIdx.y * sh.GB + slot % sh.GB, rb = slot / sh.GB;
    const bool on = rb < sh.RB && g < a.G;
    const uint32_t Cg = a.C / a.G;
    const float inv = 1.f / (float)Cg;
    const T* x = static_cast<const T*>(a.x);
    const T* dy = static_cast<const T*>(a.dy);
    T* dx = static_cast<T*>(a.dx);
    bool ok[J];
    uint64_t c[J];
    float w[J][V], b[J][V], dw[J][V], db[J][V], dw2[J][V], db2[J][V];
#pragma unroll
    for (int j = 0; j < J; ++j) {
        const uint32_t p = j * sh.L + lane;
        ok[j] = on && p < sh.packs;
        c[j] = (uint64_t)g * Cg + (uint64_t)p * V;
        load_params<V>(a, c[j], ok[j], w[j], b[j]);
#pragma unroll
        for (int k = 0; k < V; ++k) dw[j][k] = db[j][k] = dw2[j][k] = db2[j][k] = 0.f;
    }
    const uint64_t stride = (uint64_t)gridDim.x * sh.RB;
    uint32_t since = 0;
    for (uint64_t row0 = (uint64_t)blockIdx.x * sh.RB; row0 < a.N; row0 += stride * U) {
        float h[U][J][V], d[U][J][V], s[U], q[U], r[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint64_t row = row0 + u * stride + rb;
            const bool live = on && row < a.N;
            const float mean = live ? a.mean[row * a.G + g] : 0.f;
            r[u] = live ? a.rstd[row * a.G + g] : 0.f;
#pragma unroll
            for (int j = 0; j < J; ++j) {
                const bool in = ok[j] && row < a.N;
                Pack<T, V> px, pd;
                if (in) {
                    px = load_pack_cs<T, V>(x + row * a.ldx + c[j]);
                    pd = load_pack_cs<T, V>(dy + row * a.lddy + c[j]);
                }
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    h[u][j][k] = in ? (to_f32(px.v[k]) - mean) * r[u] : 0.f;
                    d[u][j][k] = in ? to_f32(pd.v[k]) : 0.f;
                }
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            s[u] = q[u] = 0.f;
#pragma unroll
            for (int j = 0; j < J; ++j) {
                float z[V];
#pragma unroll
                for (int k = 0; k < V; ++k) z[k] = h[u][j][k] * w[j][k] + b[j][k];
                activate_grad<V>(a.act, z, d[u][j]);
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    db[j][k] += d[u][j][k];
                    dw[j][k] += d[u][j][k] * h[u][j][k];
                    d[u][j][k] *= w[j][k];
                    s[u] += d[u][j][k];
                    q[u] += d[u][j][k] * h[u][j][k];
                }
            }
        }
        lane_sum<U>(s, sh.L);
        lane_sum<U>(q, sh.L);
        if (dx) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const uint64_t row = row0 + u * stride + rb;
#pragma unroll
                for (int j = 0; j < J; ++j) {
                    if (!ok[j] || row >= a.N) continue;
                    Pack<T, V> o;
#pragma unroll
                    for (int k = 0; k < V; ++k)
                        o.v[k] = from_f32<T>(r[u] * (d[u][j][k] - (s[u] + h[u][j][k] * q[u]) * inv));
                    store_pack_cs<T, V>(dx + row * a.lddx + c[j], o);
                }
            }
        }
        if ((since += U) >= 32) {
            since = 0;
#pragma unroll
            for (int j = 0; j < J; ++j)
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    dw2[j][k] += dw[j][k];
                    db2[j][k] += db[j][k];
                    dw[j][k] = db[j][k] = 0.f;
                }
        }
    }
    if (!partial) return;
    __shared__ float sm[2][kThreads * V];
#pragma unroll
    for (int j = 0; j < J; ++j) {
        __syncthreads();
#pragma unroll
        for (int k = 0; k < V; ++k) {
            sm[0][threadIdx.x * V + k] = dw2[j][k] + dw[j][k];
            sm[1][threadIdx.x * V + k] = db2[j][k] + db[j][k];
        }
        __syncthreads();
        if (rb == 0 && ok[j]) {
            float* out = partial + (uint64_t)blockIdx.x * 2 * a.C;
#pragma unroll
            for (int k = 0; k < V; ++k) {
                float tw = 0.f, tb = 0.f;
                for (uint32_t i = 0; i < sh.RB; ++i) {
                    const uint32_t t = (threadIdx.x + i * sh.GB * sh.L) * V + k;
                    tw += sm[0][t];
                    tb += sm[1][t];
                }
                out[c[j] + k] = tw;
                out[a.C + c[j] + k] = tb;
            }
        }
    }
}

// dweight, dbias [C] = column sums of partial [rows][2][C], in 64 bits.
__global__ void __launch_bounds__(1024) param_grad_kernel(const float* __restrict__ partial, uint64_t rows,
                                                          uint32_t C, void* dweight, void* dbias, int type) {
    __shared__ double sm[32][33];
    const uint32_t tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const uint64_t c = (uint64_t)blockIdx.x * 32 + tx;  // of 2 C
    double s = 0.0;
    if (c < 2ull * C) {
#pragma unroll 4
        for (uint64_t r = ty; r < rows; r += 32) s += (double)partial[r * 2 * C + c];
    }
    sm[ty][tx] = s;
    __syncthreads();
    if (ty == 0 && c < 2ull * C) {
        double t = 0.0;
        for (int i = 0; i < 32; ++i) t += sm[i][tx];
        void* out = c < C ? dweight : dbias;
        if (out) store_typed(out, type, c < C ? c : c - C, (float)t);
    }
}

// ------------------------------------------------------------ split form --

// Columns: a block of the grid's y covers GPB whole groups (SUB = 1) or one of
// the SUB parts of a group wider than the block; TX threads across, RB rows.
struct SplitShape {
    uint32_t PG, GPB, TX, RB, SUB, cols;  // PG: packs of a group; cols: the grid's y
    uint32_t chunks;
    uint64_t chunk_rows;
};

struct SplitPlace {
    bool on;
    uint32_t g, gi, len, slot;  // group, pack within the block's part of it, that part's length
    uint64_t c;                 // first channel
    uint32_t rb;
    uint64_t n, row0, row1;
    uint32_t chunk;
};

template <int V>
__device__ __forceinline__ SplitPlace split_place(const GroupNormArgs& a, const SplitShape& sh, bool reverse) {
    SplitPlace p;
    const uint32_t tx = threadIdx.x % sh.TX;
    p.rb = threadIdx.x / sh.TX;
    if (sh.SUB == 1) {
        const uint32_t i = tx / sh.PG;
        p.g = blockIdx.y * sh.GPB + i;
        p.gi = tx - i * sh.PG;
        p.len = sh.PG;
        p.on = p.g < a.G;
        p.slot = p.g;
        p.c = ((uint64_t)p.g * sh.PG + p.gi) * V;
    } else {
        p.g = blockIdx.y / sh.SUB;
        const uint32_t first = (blockIdx.y - p.g * sh.SUB) * sh.TX;
        p.gi = tx;
        p.len = min(sh.TX, sh.PG - first);
        p.on = tx < p.len;
        p.slot = blockIdx.y;
        p.c = ((uint64_t)p.g * sh.PG + first + tx) * V;
    }
    p.on = p.on && p.rb < sh.RB;
    const uint32_t block = reverse ? gridDim.x - 1 - blockIdx.x : blockIdx.x;
    p.n = block / sh.chunks;
    p.chunk = block - (uint32_t)p.n * sh.chunks;
    p.row0 = p.chunk * sh.chunk_rows;
    p.row1 = min(p.row0 + sh.chunk_rows, a.S);
    return p;
}

struct Moments {
    float n, mean, m2;
};

__device__ __forceinline__ Moments merge(const Moments& a, const Moments& b) {
    Moments o;
    o.n = a.n + b.n;
    const float f = o.n > 0.f ? b.n / o.n : 0.f;
    const float d = b.mean - a.mean;
    o.mean = a.mean + d * f;
    o.m2 = a.m2 + b.m2 + d * d * a.n * f;
    return o;
}

constexpr int kBlockRows = 4;  // rows of a thread's block of values

template <typename T, int V>
__global__ void __launch_bounds__(kThreads) split_moments_kernel(const GroupNormArgs a, const SplitShape sh,
                                                                 Moments* __restrict__ partial) {
    const SplitPlace p = split_place<V>(a, sh, false);
    const T* x = static_cast<const T*>(a.x) + p.n * a.S * a.ldx + p.c;
    Moments m{0.f, 0.f, 0.f};
    if (p.on) {
        for (uint64_t r = p.row0 + p.rb; r < p.row1; r += (uint64_t)sh.RB * kBlockRows) {
            float v[kBlockRows][V], s = 0.f, q = 0.f;
            int rows = 0;
#pragma unroll
            for (int u = 0; u < kBlockRows; ++u) {
                const uint64_t row = r + (uint64_t)u * sh.RB;
                Pack<T, V> pk;
                if (row < p.row1) {
                    pk = load_pack<T, V>(x + row * a.ldx);
                    ++rows;
                }
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    v[u][k] = row < p.row1 ? to_f32(pk.v[k]) : 0.f;
                    s += v[u][k];
                }
            }
            const float n = (float)(rows * V);
            const float mean = s / n;
#pragma unroll
            for (int u = 0; u < kBlockRows; ++u)
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    const float d = v[u][k] - mean;
                    q += u < rows ? d * d : 0.f;
                }
            m = merge(m, Moments{n, mean, q});
        }
    }
    __shared__ Moments sm[kThreads];
    sm[threadIdx.x] = m;
    __syncthreads();
    for (uint32_t h = sh.RB; h > 1;) {  // over the rows of the block
        const uint32_t half = (h + 1) / 2;
        if (p.on && p.rb < half && p.rb + half < h)
            sm[threadIdx.x] = merge(sm[threadIdx.x], sm[threadIdx.x + half * sh.TX]);
        h = half;
        __syncthreads();
    }
    for (uint32_t h = min(sh.PG, sh.TX); h > 1;) {  // over the packs of a group
        const uint32_t half = (h + 1) / 2;
        if (p.on && p.rb == 0 && p.gi < half && p.gi + half < min(h, p.len))
            sm[threadIdx.x] = merge(sm[threadIdx.x], sm[threadIdx.x + half]);
        h = half;
        __syncthreads();
    }
    if (p.on && p.rb == 0 && p.gi == 0)
        partial[(p.n * sh.chunks + p.chunk) * ((uint64_t)a.G * sh.SUB) + p.slot] = sm[threadIdx.x];
}

// A warp per (sample, group) merges its partial moments.
__global__ void __launch_bounds__(kThreads) split_stats_kernel(const Moments* __restrict__ partial,
                                                               uint64_t N, uint32_t G, uint32_t SUB,
                                                               uint32_t chunks, float eps,
                                                               float* __restrict__ mean,
                                                               float* __restrict__ rstd) {
    const uint64_t i = ((uint64_t)blockIdx.x * kThreads + threadIdx.x) >> 5;
    if (i >= N * G) return;
    const uint32_t lane = threadIdx.x & 31;
    const uint64_t n = i / G;
    const uint32_t g = (uint32_t)(i - n * G);
    Moments m{0.f, 0.f, 0.f};
    for (uint32_t k = lane; k < chunks * SUB; k += 32) {
        const uint32_t ch = k / SUB;
        m = merge(m, partial[(n * chunks + ch) * ((uint64_t)G * SUB) + g * SUB + (k - ch * SUB)]);
    }
    for (int o = 16; o; o >>= 1) {
        Moments t;
        t.n = __shfl_down_sync(0xffffffffu, m.n, o);
        t.mean = __shfl_down_sync(0xffffffffu, m.mean, o);
        t.m2 = __shfl_down_sync(0xffffffffu, m.m2, o);
        m = merge(m, t);
    }
    if (lane == 0) {
        mean[i] = m.mean;
        rstd[i] = __frsqrt_rn(m.m2 / m.n + eps);
    }
}

template <typename T, int V>
__global__ void __launch_bounds__(kThreads) split_apply_kernel(const GroupNormArgs a, const SplitShape sh,
                                                               const float* __restrict__ mean_,
                                                               const float* __restrict__ rstd_) {
    const SplitPlace p = split_place<V>(a, sh, true);
    if (!p.on) return;
    const T* x = static_cast<const T*>(a.x) + p.n * a.S * a.ldx + p.c;
    T* y = static_cast<T*>(a.y) + p.n * a.S * a.ldy + p.c;
    const float mean = mean_[p.n * a.G + p.g], rstd = rstd_[p.n * a.G + p.g];
    float w[V], b[V];
    load_params<V>(a, p.c, true, w, b);
#pragma unroll 4
    for (uint64_t r = p.row0 + p.rb; r < p.row1; r += sh.RB) {
        const Pack<T, V> pk = load_pack<T, V>(x + r * a.ldx);
        float z[V];
#pragma unroll
        for (int k = 0; k < V; ++k) z[k] = (to_f32(pk.v[k]) - mean) * rstd * w[k] + b[k];
        activate<V>(a.act, z);
        Pack<T, V> o;
#pragma unroll
        for (int k = 0; k < V; ++k) o.v[k] = from_f32<T>(z[k]);
        store_pack_cs<T, V>(y + r * a.ldy, o);
    }
}

// Per chunk and channel: sums of dz * h and of dz -> partial [N][chunks][2][C].
template <typename T, int V>
__global__ void __launch_bounds__(kThreads) split_sums_kernel(const GroupNormArgs a, const SplitShape sh,
                                                              float* __restrict__ partial) {
    const SplitPlace p = split_place<V>(a, sh, false);
    float dw[V], db[V];
#pragma unroll
    for (int k = 0; k < V; ++k) dw[k] = db[k] = 0.f;
    if (p.on) {
        const T* x = static_cast<const T*>(a.x) + p.n * a.S * a.ldx + p.c;
        const T* dy = static_cast<const T*>(a.dy) + p.n * a.S * a.lddy + p.c;
        const float mean = a.mean[p.n * a.G + p.g], rstd = a.rstd[p.n * a.G + p.g];
        float w[V], b[V];
        load_params<V>(a, p.c, true, w, b);
#pragma unroll 4
        for (uint64_t r = p.row0 + p.rb; r < p.row1; r += sh.RB) {
            const Pack<T, V> px = load_pack<T, V>(x + r * a.ldx);
            const Pack<T, V> pd = load_pack<T, V>(dy + r * a.lddy);
            float h[V], z[V], d[V];
#pragma unroll
            for (int k = 0; k < V; ++k) {
                h[k] = (to_f32(px.v[k]) - mean) * rstd;
                z[k] = h[k] * w[k] + b[k];
                d[k] = to_f32(pd.v[k]);
            }
            activate_grad<V>(a.act, z, d);
#pragma unroll
            for (int k = 0; k < V; ++k) {
                db[k] += d[k];
                dw[k] += d[k] * h[k];
            }
        }
    }
    __shared__ float sm[2][kThreads * V];
#pragma unroll
    for (int k = 0; k < V; ++k) {
        sm[0][threadIdx.x * V + k] = dw[k];
        sm[1][threadIdx.x * V + k] = db[k];
    }
    __syncthreads();
    if (p.on && p.rb == 0) {
        float* out = partial + (p.n * sh.chunks + p.chunk) * 2 * a.C + p.c;
#pragma unroll
        for (int k = 0; k < V; ++k) {
            float tw = 0.f, tb = 0.f;
            for (uint32_t i = 0; i < sh.RB; ++i) {
                tw += sm[0][(threadIdx.x + i * sh.TX) * V + k];
                tb += sm[1][(threadIdx.x + i * sh.TX) * V + k];
            }
            out[k] = tw;
            out[a.C + k] = tb;
        }
    }
}

// sums [N][2][C] over the chunks.
__global__ void __launch_bounds__(kThreads) split_fold_kernel(const float* __restrict__ partial, uint64_t N,
                                                              uint32_t C, uint32_t chunks,
                                                              float* __restrict__ sums) {
    const uint64_t i = (uint64_t)blockIdx.x * kThreads + threadIdx.x;
    if (i >= N * 2 * C) return;
    const uint64_t n = i / (2ull * C), c = i - n * 2 * C;
    double s = 0.0;
#pragma unroll 8
    for (uint32_t k = 0; k < chunks; ++k) s += (double)partial[(n * chunks + k) * 2 * C + c];
    sums[i] = (float)s;
}

// group_sums [N][G][2]: a = sum of weight * (sum dz), b = sum of weight * (sum dz * h); a warp each.
__global__ void __launch_bounds__(kThreads) split_groups_kernel(const GroupNormArgs a,
                                                                const float* __restrict__ sums,
                                                                float* __restrict__ group_sums) {
    const uint64_t i = ((uint64_t)blockIdx.x * kThreads + threadIdx.x) >> 5;
    if (i >= a.N * a.G) return;
    const uint32_t lane = threadIdx.x & 31;
    const uint64_t n = i / a.G;
    const uint32_t g = (uint32_t)(i - n * a.G), Cg = a.C / a.G;
    float s = 0.f, q = 0.f;
    for (uint32_t k = lane; k < Cg; k += 32) {
        const uint32_t c = g * Cg + k;
        const float w = a.weight ? load_typed(a.weight, a.param_type, c) : 1.f;
        q += w * sums[n * 2 * a.C + c];
        s += w * sums[n * 2 * a.C + a.C + c];
    }
    for (int o = 16; o; o >>= 1) {
        s += __shfl_xor_sync(0xffffffffu, s, o);
        q += __shfl_xor_sync(0xffffffffu, q, o);
    }
    if (lane == 0) {
        group_sums[2 * i] = s;
        group_sums[2 * i + 1] = q;
    }
}

template <typename T, int V>
__global__ void __launch_bounds__(kThreads) split_grad_kernel(const GroupNormArgs a, const SplitShape sh,
                                                              const float* __restrict__ group_sums) {
    const SplitPlace p = split_place<V>(a, sh, true);
    if (!p.on) return;
    const T* x = static_cast<const T*>(a.x) + p.n * a.S * a.ldx + p.c;
    const T* dy = static_cast<const T*>(a.dy) + p.n * a.S * a.lddy + p.c;
    T* dx = static_cast<T*>(a.dx) + p.n * a.S * a.lddx + p.c;
    const uint64_t i = p.n * a.G + p.g;
    const float inv = 1.f / ((float)a.S * (float)(a.C / a.G));
    const float mean = a.mean[i], rstd = a.rstd[i], s = group_sums[2 * i] * inv, q = group_sums[2 * i + 1] * inv;
    float w[V], b[V];
    load_params<V>(a, p.c, true, w, b);
#pragma unroll 4
    for (uint64_t r = p.row0 + p.rb; r < p.row1; r += sh.RB) {
        const Pack<T, V> px = load_pack<T, V>(x + r * a.ldx);
        const Pack<T, V> pd = load_pack<T, V>(dy + r * a.lddy);
        float h[V], z[V], d[V];
#pragma unroll
        for (int k = 0; k < V; ++k) {
            h[k] = (to_f32(px.v[k]) - mean) * rstd;
            z[k] = h[k] * w[k] + b[k];
            d[k] = to_f32(pd.v[k]);
        }
        activate_grad<V>(a.act, z, d);
        Pack<T, V> o;
#pragma unroll
        for (int k = 0; k < V; ++k) o.v[k] = from_f32<T>(rstd * (d[k] * w[k] - (s + h[k] * q)));
        store_pack_cs<T, V>(dx + r * a.lddx, o);
    }
}

// ------------------------------------------------------------------ host --

uint64_t align256(uint64_t b) { return (b + 255) / 256 * 256; }

int pick_width(const GroupNormArgs& a) {
    const uint32_t es = type_bytes(a.type);
    VecRule rule;
    rule.count(a.C / a.G);
    const void* ptrs[] = {a.x, a.y, a.dy, a.dx};
    const uint64_t lds[] = {a.ldx, a.ldy, a.lddy, a.lddx};
    for (int i = 0; i < 4; ++i) {
        rule.pointer(ptrs[i], es);
        if (ptrs[i]) rule.count(lds[i]);
    }
    return rule.width();
}

// The rows form holds up to 8 packs a lane.
bool rows_form(uint64_t S, uint32_t Cg, int V) { return S == 1 && Cg <= 32u * 8u * (uint32_t)V; }

RowsShape rows_shape(uint32_t C, uint32_t G, int V) {
    RowsShape sh;
    sh.packs = C / G / V;
    sh.L = 1;
    while (sh.L < 32 && sh.L < sh.packs) sh.L <<= 1;
    const uint32_t slots = kThreads / sh.L;
    sh.GB = std::min(G, slots);
    sh.RB = slots / sh.GB;
    return sh;
}

// Enough CTAs in x to fill the GPU with eight per SM, whole passes over the rows.
uint64_t rows_blocks(const RowsShape& sh, uint64_t N, uint32_t G, uint64_t per_sm) {
    const uint64_t y = (G + sh.GB - 1) / sh.GB;
    return std::max<uint64_t>(1, std::min((N + sh.RB - 1) / sh.RB, kSms * per_sm / std::min(kSms, y)));
}

// Chunks of a sample: about eight CTAs per SM over all samples, at least eight
// rows a thread, at most 512 chunks to merge.
SplitShape split_shape(uint64_t N, uint64_t S, uint32_t C, uint32_t G, int V) {
    SplitShape sh;
    sh.PG = C / G / V;
    if (sh.PG <= (uint32_t)kThreads) {
        sh.GPB = std::min(G, kThreads / sh.PG);
        sh.TX = sh.GPB * sh.PG;
        sh.RB = kThreads / sh.TX;
        sh.SUB = 1;
        sh.cols = (G + sh.GPB - 1) / sh.GPB;
    } else {
        sh.GPB = 1;
        sh.TX = kThreads;
        sh.RB = 1;
        sh.SUB = (sh.PG + kThreads - 1) / kThreads;
        sh.cols = G * sh.SUB;
    }
    const uint64_t want = std::max<uint64_t>(1, kSms * 8 / std::max<uint64_t>(1, std::min(N, kSms * 8) * sh.cols));
    const uint64_t most = std::max<uint64_t>(1, S / (8 * sh.RB));
    const uint64_t chunks = std::min<uint64_t>(512, std::min(want, most));
    sh.chunk_rows = (S + chunks - 1) / chunks;
    sh.chunks = (uint32_t)((S + sh.chunk_rows - 1) / sh.chunk_rows);
    return sh;
}

uint32_t sub_slots(uint32_t C, uint32_t G) { return (C / G + kThreads - 1) / kThreads; }

// Upper bounds over every vector width, so that the size does not depend on
// the pointers' alignment.
constexpr uint64_t kRowsPerSm = 8;

}  // namespace

size_t group_norm_scratch_bytes(uint64_t N, uint64_t S, uint32_t C, uint32_t G, bool backward) {
    if (N == 0 || S == 0 || C == 0 || G == 0 || C % G) return 0;
    uint64_t rows = 0, chunks = 1;
    for (int V = 1; V <= 8; V <<= 1) {
        if ((C / G) % V) break;
        if (rows_form(S, C / G, V)) rows = std::max(rows, rows_blocks(rows_shape(C, G, V), N, G, kRowsPerSm));
        chunks = std::max<uint64_t>(chunks, split_shape(N, S, C, G, V).chunks);
    }
    if (!backward && rows_form(S, C / G, 1)) return 0;  // whichever width is picked
    const uint64_t stats = 2 * align256(N * G * 4);
    if (!backward) return (size_t)(align256(N * chunks * G * sub_slots(C, G) * sizeof(Moments)) + stats);
    return (size_t)(align256(std::max(rows, N * chunks) * 2 * C * 4) + align256(N * 2 * C * 4) + stats);
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

template <typename T, int V, int J>
void rows_launch(const GroupNormArgs& a, float* partial, bool backward, cudaStream_t s) {
    const RowsShape sh = rows_shape(a.C, a.G, V);
    const dim3 grid((unsigned)rows_blocks(sh, a.N, a.G, kRowsPerSm), (a.G + sh.GB - 1) / sh.GB);
    TCC_REQUIRE(grid.y <= 65535, "too many groups for one-row samples");
    constexpr int U = V * J <= 4 ? 4 : V * J <= 8 ? 2 : 1;
    if (backward) rows_backward_kernel<T, V, J, U><<<grid, kThreads, 0, s>>>(a, sh, partial);
    else rows_forward_kernel<T, V, J, U><<<grid, kThreads, 0, s>>>(a, sh);
    TCC_CUDA(cudaGetLastError());
    if (backward && partial) {
        param_grad_kernel<<<(2 * a.C + 31) / 32, 1024, 0, s>>>(partial, grid.x, a.C, a.dweight, a.dbias,
                                                              a.param_type);
        TCC_CUDA(cudaGetLastError());
    }
}

template <typename T, int V>
void rows_by_packs(const GroupNormArgs& a, float* partial, bool backward, cudaStream_t s) {
    const RowsShape sh = rows_shape(a.C, a.G, V);
    const uint32_t per_lane = (sh.packs + sh.L - 1) / sh.L;
    if (per_lane <= 1) rows_launch<T, V, 1>(a, partial, backward, s);
    else if (per_lane <= 2) rows_launch<T, V, 2>(a, partial, backward, s);
    else if (per_lane <= 4) rows_launch<T, V, 4>(a, partial, backward, s);
    else rows_launch<T, V, 8>(a, partial, backward, s);
}

template <typename T, int V>
void norm_launch(const GroupNormArgs& a, char* scratch, bool backward, cudaStream_t s) {
    const bool params = backward && (a.dweight || a.dbias);
    if (rows_form(a.S, a.C / a.G, V)) {
        rows_by_packs<T, V>(a, params ? reinterpret_cast<float*>(scratch) : nullptr, backward, s);
        return;
    }
    const SplitShape sh = split_shape(a.N, a.S, a.C, a.G, V);
    TCC_REQUIRE(a.N * sh.chunks < (1ull << 31) && sh.cols <= 65535, "too many samples or groups for one call");
    const dim3 grid((unsigned)(a.N * sh.chunks), sh.cols);
    const unsigned warps = ceil_div(a.N * a.G, kThreads / 32);
    if (!backward) {
        Moments* partial = reinterpret_cast<Moments*>(scratch);
        float* mean = a.mean;
        float* rstd = a.rstd;
        if (!mean) {
            mean = reinterpret_cast<float*>(scratch + align256(a.N * sh.chunks * a.G * sh.SUB * sizeof(Moments)));
            rstd = mean + align256(a.N * a.G * 4) / 4;
        }
        split_moments_kernel<T, V><<<grid, kThreads, 0, s>>>(a, sh, partial);
        split_stats_kernel<<<warps, kThreads, 0, s>>>(partial, a.N, a.G, sh.SUB, sh.chunks, a.eps, mean, rstd);
        split_apply_kernel<T, V><<<grid, kThreads, 0, s>>>(a, sh, mean, rstd);
    } else {
        float* partial = reinterpret_cast<float*>(scratch);
        float* sums = partial + align256(a.N * sh.chunks * 2 * a.C * 4) / 4;
        float* group_sums = sums + align256(a.N * 2 * a.C * 4) / 4;
        split_sums_kernel<T, V><<<grid, kThreads, 0, s>>>(a, sh, partial);
        split_fold_kernel<<<ceil_div(a.N * 2 * a.C, kThreads), kThreads, 0, s>>>(partial, a.N, a.C, sh.chunks, sums);
        if (params)
            param_grad_kernel<<<(2 * a.C + 31) / 32, 1024, 0, s>>>(sums, a.N, a.C, a.dweight, a.dbias, a.param_type);
        if (a.dx) {
            split_groups_kernel<<<warps, kThreads, 0, s>>>(a, sums, group_sums);
            split_grad_kernel<T, V><<<grid, kThreads, 0, s>>>(a, sh, group_sums);
        }
    }
    TCC_CUDA(cudaGetLastError());
}

template <typename T>
void norm_by_width(const GroupNormArgs& a, char* scratch, bool backward, cudaStream_t s) {
    switch (std::min<int>(pick_width(a), 16 / (int)sizeof(T))) {
        case 8:
            if constexpr (sizeof(T) == 2) norm_launch<T, 8>(a, scratch, backward, s);
            break;
        case 4: norm_launch<T, 4>(a, scratch, backward, s); break;
        case 2: norm_launch<T, 2>(a, scratch, backward, s); break;
        default: norm_launch<T, 1>(a, scratch, backward, s);
    }
}

void norm_by_type(const GroupNormArgs& a, void* scratch, bool backward, cudaStream_t s) {
    char* p = static_cast<char*>(scratch);
    if (a.type == TCC_F32) norm_by_width<float>(a, p, backward, s);
    else if (a.type == TCC_F16) norm_by_width<__half>(a, p, backward, s);
    else norm_by_width<__nv_bfloat16>(a, p, backward, s);
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
