// group_norm.cuh -- group norm over channels-last features, then an activation,
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
// Three forms:
//  * rows  (up to 32 rows a sample, S = 1 above all; a sample's group within a
//    warp, which is 1,024 values in packs of four or more, 512 in packs of two, 256
//    value by value): every (sample, group) is reduced by a few lanes of one warp,
//    x is read once; the next samples are on their way into a ring in shared
//    memory meanwhile.
//  * resident (a sample that fits the shared memory of at most eight SMs): a
//    cluster of CTAs holds a sample, x (and dy) are read once, the CTAs exchange
//    their moments or sums through distributed shared memory.
//  * split (any other): the rows of a sample are cut into chunks, a CTA each;
//    moments (or channel sums) per chunk, a merge over the chunks, and a
//    second pass that normalises, walking each chunk from its end, so that what
//    the first pass read last is still in L2.
#pragma once

#include "elem.cuh"
#include "train_ops.cuh"

#include <cooperative_groups.h>

#include <algorithm>
#include <type_traits>

namespace tcc {

namespace {

constexpr int kThreads = 256;
constexpr uint64_t kSms = 148;

// ---------------------------------------------------------------- values --

// V fp32 values of one thread; pairs go through the two-wide fp32
// instructions of sm_100 (one issue slot for two values).
template <int V>
struct Vec {
    float v[V];
};

#define TCC_PAIRWISE(NAME, OP, SCALAR)                                                                     \
    template <int V>                                                                                       \
    __device__ __forceinline__ Vec<V> NAME(const Vec<V>& a, const Vec<V>& b) {                             \
        Vec<V> o;                                                                                          \
        if constexpr (V % 2 == 0) {                                                                        \
            _Pragma("unroll") for (int k = 0; k < V; k += 2)                                               \
                asm("{.reg .b64 x, y, z;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n " OP              \
                    ".rn.f32x2 z, x, y;\n mov.b64 {%0, %1}, z;}"                                           \
                    : "=f"(o.v[k]), "=f"(o.v[k + 1])                                                       \
                    : "f"(a.v[k]), "f"(a.v[k + 1]), "f"(b.v[k]), "f"(b.v[k + 1]));                         \
        } else {                                                                                           \
            _Pragma("unroll") for (int k = 0; k < V; ++k) o.v[k] = SCALAR;                                 \
        }                                                                                                  \
        return o;                                                                                          \
    }
TCC_PAIRWISE(add, "add", a.v[k] + b.v[k])
TCC_PAIRWISE(mul, "mul", a.v[k] * b.v[k])
#undef TCC_PAIRWISE

// a * b + c
template <int V>
__device__ __forceinline__ Vec<V> fma(const Vec<V>& a, const Vec<V>& b, const Vec<V>& c) {
    Vec<V> o;
    if constexpr (V % 2 == 0) {
#pragma unroll
        for (int k = 0; k < V; k += 2)
            asm("{.reg .b64 x, y, z;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mov.b64 z, {%6, %7};\n "
                "fma.rn.f32x2 z, x, y, z;\n mov.b64 {%0, %1}, z;}"
                : "=f"(o.v[k]), "=f"(o.v[k + 1])
                : "f"(a.v[k]), "f"(a.v[k + 1]), "f"(b.v[k]), "f"(b.v[k + 1]), "f"(c.v[k]), "f"(c.v[k + 1]));
    } else {
#pragma unroll
        for (int k = 0; k < V; ++k) o.v[k] = fmaf(a.v[k], b.v[k], c.v[k]);
    }
    return o;
}

template <int V>
__device__ __forceinline__ Vec<V> splat(float x) {
    Vec<V> o;
#pragma unroll
    for (int k = 0; k < V; ++k) o.v[k] = x;
    return o;
}
template <int V>
__device__ __forceinline__ float sum(const Vec<V>& a) {
    if constexpr (V == 1) {
        return a.v[0];
    } else if constexpr (V == 2) {
        return a.v[0] + a.v[1];
    } else {
        Vec<V / 2> lo, hi;
#pragma unroll
        for (int k = 0; k < V / 2; ++k) {
            lo.v[k] = a.v[k];
            hi.v[k] = a.v[V / 2 + k];
        }
        return sum(add(lo, hi));
    }
}
// sum of a * b
template <int V>
__device__ __forceinline__ float dot(const Vec<V>& a, const Vec<V>& b) {
    if constexpr (V <= 2) {
        return sum(mul(a, b));
    } else {
        Vec<2> s{{a.v[0] * b.v[0], a.v[1] * b.v[1]}};
#pragma unroll
        for (int k = 2; k < V; k += 2)
            s = fma(Vec<2>{{a.v[k], a.v[k + 1]}}, Vec<2>{{b.v[k], b.v[k + 1]}}, s);
        return s.v[0] + s.v[1];
    }
}
template <typename T, int V>
__device__ __forceinline__ Vec<V> widen(const Pack<T, V>& p) {
    Vec<V> o;
#pragma unroll
    for (int k = 0; k < V; ++k) o.v[k] = to_f32(p.v[k]);
    return o;
}
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> narrow(const Vec<V>& a) {
    Pack<T, V> p;
    if constexpr (sizeof(T) == 2 && V % 2 == 0) {  // one conversion for two values
#pragma unroll
        for (int k = 0; k < V; k += 2) {
            if constexpr (std::is_same_v<T, __half>) {
                const __half2 h = __floats2half2_rn(a.v[k], a.v[k + 1]);
                p.v[k] = h.x, p.v[k + 1] = h.y;
            } else {
                const __nv_bfloat162 h = __floats2bfloat162_rn(a.v[k], a.v[k + 1]);
                p.v[k] = h.x, p.v[k + 1] = h.y;
            }
        }
    } else {
#pragma unroll
        for (int k = 0; k < V; ++k) p.v[k] = from_f32<T>(a.v[k]);
    }
    return p;
}

// ------------------------------------------------------------ activation --

// The hardware's exponential and reciprocal, which take one issue slot each: off by
// 4 u and 2 u of their results (u = 2^-24).
template <int V>
__device__ __forceinline__ void exp2_of(Vec<V>& a) {
#pragma unroll
    for (int k = 0; k < V; ++k) asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(a.v[k]));
}
template <int V>
__device__ __forceinline__ void reciprocal_of(Vec<V>& a) {
#pragma unroll
    for (int k = 0; k < V; ++k) asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(a.v[k]));
}

// 1 / (1 + 2^(-z log2 e)).  The product is rounded, so for z < 0 the result is off by
// up to (10 + |z|) u of itself (measured: 15 u at -10, 63 u at -80, where it is 1e-35);
// for z > 0 by 5 u.  Taking the exponent in two parts instead keeps 10 u everywhere but
// takes 13 % more time (2.4 M x 256 fp32: 1020 us forward in place of 898).
template <int V>
__device__ __forceinline__ Vec<V> sigmoid(const Vec<V>& z) {
    Vec<V> e = mul(z, splat<V>(-1.4426950408889634f));
    exp2_of(e);
    e = add(e, splat<V>(1.f));
    reciprocal_of(e);
    return e;
}

// The normal distribution function Phi(z), and e = exp(-z^2 / 2) for its
// density: Phi(-|z|) = e * t * P(t) with t = 1 / (1 + p |z|), the form of Abramowitz and
// Stegun (Handbook of Mathematical Functions, 7.1.26).  (erff and expf in its place:
// 1095 us against 650 for 2.4 M x 256 bf16 values.)
//  * 16-bit features: their p and five terms, off by 0.75e-7 in exact arithmetic and
//    by up to 3e-7 with fp32's roundings, far below the features' own.
//  * fp32 features (FINE): six terms, fitted here to erfcx(|z| / sqrt 2) / 2 over
//    |z| <= 13.5 with the relative error weighted by 1 / (1 + z^4): Phi(-|z|) is off by
//    at most (16 + 1.5 z^2 + 1.5 z^4) u of itself, the second part from the rounded
//    exponent, where the five terms reach 870 u at -3 and 7,800 u at -4.  1 to 2 % more time
//    (2.4 M x 256: backward 1325 -> 1343 us).
template <bool FINE, int V>
__device__ __forceinline__ Vec<V> normal_cdf(const Vec<V>& z, Vec<V>& e) {
    Vec<V> t, q;
#pragma unroll
    for (int k = 0; k < V; ++k) t.v[k] = fabsf(z.v[k]);
    t = fma(t, splat<V>(FINE ? 0.4f : 0.3275911f * 0.70710678118654752f), splat<V>(1.f));
    reciprocal_of(t);
    e = mul(mul(z, splat<V>(-0.72134752044448170f)), z);  // log2(e) / 2
    exp2_of(e);
    if constexpr (FINE) {
        q = fma(t, splat<V>(0.0550596827387823f), splat<V>(-0.24951052190289993f));
        q = fma(q, t, splat<V>(0.33170637217092475f));
        q = fma(q, t, splat<V>(0.0192833073779339f));
        q = fma(q, t, splat<V>(0.18641695632855948f));
        q = fma(q, t, splat<V>(0.15704418169723153f));
    } else {
        q = fma(t, splat<V>(0.5f * 1.061405429f), splat<V>(-0.5f * 1.453152027f));
        q = fma(q, t, splat<V>(0.5f * 1.421413741f));
        q = fma(q, t, splat<V>(-0.5f * 0.284496736f));
        q = fma(q, t, splat<V>(0.5f * 0.254829592f));
    }
    q = mul(mul(q, t), e);  // Phi(-|z|)
#pragma unroll
    for (int k = 0; k < V; ++k) q.v[k] = z.v[k] < 0.f ? q.v[k] : 1.f - q.v[k];
    return q;
}

// act(z) of features of type T
template <typename T, int V>
__device__ __forceinline__ Vec<V> activate(int act, Vec<V> z) {
    if (act == TCC_ACT_RELU) {
#pragma unroll
        for (int k = 0; k < V; ++k) z.v[k] = z.v[k] <= 0.f ? 0.f : z.v[k];
    } else if (act == TCC_ACT_SILU) {
        z = mul(z, sigmoid(z));
    } else if (act == TCC_ACT_GELU) {
        Vec<V> e;
        z = mul(z, normal_cdf<sizeof(T) == 4>(z, e));
    }
    return z;
}

// d * act'(z)
template <typename T, int V>
__device__ __forceinline__ Vec<V> activate_grad(int act, const Vec<V>& z, Vec<V> d) {
    if (act == TCC_ACT_RELU) {
#pragma unroll
        for (int k = 0; k < V; ++k) d.v[k] = z.v[k] <= 0.f ? 0.f : d.v[k];
    } else if (act == TCC_ACT_SILU) {  // s + z s (1 - s)
        const Vec<V> s = sigmoid(z), rest = fma(s, splat<V>(-1.f), splat<V>(1.f));
        d = mul(d, fma(mul(z, s), rest, s));
    } else if (act == TCC_ACT_GELU) {  // Phi(z) + z phi(z)
        Vec<V> e;
        const Vec<V> cdf = normal_cdf<sizeof(T) == 4>(z, e);
        d = mul(d, fma(mul(z, splat<V>(0.39894228040143268f)), e, cdf));
    }
    return d;
}

template <typename P, int V>
__device__ __forceinline__ Vec<V> load_param(const void* p, uint64_t c) {
    Vec<V> o;
#pragma unroll
    for (int k = 0; k < V; ++k) o.v[k] = to_f32(static_cast<const P*>(p)[c + k]);
    return o;
}
template <int V>
__device__ __forceinline__ void load_params(const GroupNormArgs& a, uint64_t c, bool on, Vec<V>& w, Vec<V>& b) {
    w = splat<V>(1.f);
    b = splat<V>(0.f);
    if (!on) return;
    if (a.param_type == TCC_F32) {
        if (a.weight) w = load_param<float, V>(a.weight, c);
        if (a.bias) b = load_param<float, V>(a.bias, c);
    } else if (a.param_type == TCC_F16) {
        if (a.weight) w = load_param<__half, V>(a.weight, c);
        if (a.bias) b = load_param<__half, V>(a.bias, c);
    } else {
        if (a.weight) w = load_param<__nv_bfloat16, V>(a.weight, c);
        if (a.bias) b = load_param<__nv_bfloat16, V>(a.bias, c);
    }
}

// 1 / sqrt(x), off by about one unit in the last place (the hardware's, and a
// Newton step); one form for every path.
__device__ __forceinline__ float inverse_root(float x) {
    float r;
    asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    const float e = fmaf(-x * r, r, 1.f);
    return fabsf(x) < 1e-30f || x > 1e37f ? rsqrtf(x) : fmaf(0.5f * r, e, r);
}

// ------------------------------------------------------------- rows form --

// A slot is L lanes (a power of two) that hold one group of one sample (of its
// S rows) as J packs each; a CTA's 256 / L slots are GB groups x RB samples.  A
// thread keeps its channels for the whole kernel: their parameters and the
// parameters' gradients stay in registers.
struct RowsShape {
    uint32_t L, log_L, GB, RB, PG, packs;  // packs of a group in a row, in a sample
    uint32_t level;                        // passes of the backward's first level of sums
    // bytes from one pass to the next, computed here so that they are constants there
    uint64_t x_step, y_step, dy_step, dx_step, stats_step;
};

template <typename T>
__device__ __forceinline__ T* advance(T* p, uint64_t bytes) {
    return reinterpret_cast<T*>(reinterpret_cast<uintptr_t>(p) + bytes);
}

// Sum over the L lanes of a slot.
__device__ __forceinline__ float lane_sum(float v, uint32_t L) {
    if (L > 1) v += __shfl_xor_sync(0xffffffffu, v, 1);
    if (L > 2) v += __shfl_xor_sync(0xffffffffu, v, 2);
    if (L > 4) v += __shfl_xor_sync(0xffffffffu, v, 4);
    if (L > 8) v += __shfl_xor_sync(0xffffffffu, v, 8);
    if (L > 16) v += __shfl_xor_sync(0xffffffffu, v, 16);
    return v;
}

// n floats, `stride` apart, by four sums at a time: no chain of more than n / 4 + 4 additions.
__device__ __forceinline__ float strided_sum(const float* p, uint32_t stride, uint32_t n) {
    float t[4] = {0.f, 0.f, 0.f, 0.f};
    uint32_t r = 0;
    for (; r + 4 <= n; r += 4)
#pragma unroll
        for (int u = 0; u < 4; ++u) t[u] += p[(r + u) * stride];
    for (; r < n; ++r) t[0] += p[r * stride];
    return (t[0] + t[1]) + (t[2] + t[3]);
}

// Long fp32 sums are kept in two levels: a thread adds kLevel rows (or blocks of
// rows, or samples), then that sum to a second one, and takes at most kLongest
// in all, so that no chain of additions grows with the data.  (The row form,
// which leaves a row of sums per thread row, takes as many as there are: its
// levels are the square root of that, 130 each for 10 M rows.)
constexpr uint32_t kLevel = 32, kLongest = 2048;

// The place of a thread: its slot's group and sample, its packs' rows and
// channels in them.
template <int V, int J>
struct RowsPlace {
    uint32_t lane, g, rb;
    bool on, ok[J];
    uint32_t row[J], c[J];
    Vec<V> w[J], b[J];
    __device__ __forceinline__ RowsPlace(const GroupNormArgs& a, const RowsShape& sh) {
        const uint32_t slot = threadIdx.x >> sh.log_L;
        lane = threadIdx.x & (sh.L - 1);
        rb = slot / sh.GB;
        g = blockIdx.y * sh.GB + slot - rb * sh.GB;
        on = rb < sh.RB && g < a.G;
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const uint32_t p = j * sh.L + lane;
            ok[j] = on && p < sh.packs;
            row[j] = p / sh.PG;
            c[j] = g * (a.C / a.G) + (p - row[j] * sh.PG) * V;
            load_params<V>(a, c[j], ok[j], w[j], b[j]);
        }
    }
    __device__ __forceinline__ uint64_t at(int j, uint64_t ld) const { return row[j] * ld + c[j]; }
};

// wait_copies with a pass number that is a constant once the loop is unrolled.
template <int D>
__device__ __forceinline__ void wait_pass(uint32_t d) {
    if (d == 0) wait_copies<D - 1>();
    else if (d == 1) wait_copies<(D > 2 ? D - 2 : 0)>();
    else if (d == 2) wait_copies<(D > 3 ? D - 3 : 0)>();
    else if (d == 3) wait_copies<(D > 4 ? D - 4 : 0)>();
    else if (d == 4) wait_copies<(D > 5 ? D - 5 : 0)>();
    else if (d == 5) wait_copies<(D > 6 ? D - 6 : 0)>();
    else if (d == 6) wait_copies<(D > 7 ? D - 7 : 0)>();
    else wait_copies<0>();
}

// Ring of the packs of the next rows: D rows of J packs of A arrays.  A thread
// copies and reads its own packs only.
template <typename T, int V, int J, int A>
struct RowsRing {
    static constexpr int D = J >= 8 ? 1 : 8 / (J * A) > 2 ? 8 / (J * A) : 2;
    static constexpr bool kAsync = sizeof(Pack<T, V>) >= 4;
    Pack<T, V> slot[D][A][J][kThreads];
};

// A CTA takes `passes` times RB neighbouring rows, at most what its ring holds:
// it asks for all of them at once and is done, so reads and writes of many CTAs
// mix.  mean and rstd are staged and leave in whole sectors (written from the
// lanes that hold them they cost 70 us at 2.4 M x 256 fp32).  There it takes
// 744 us for 5.2 GB, a copy of x 780; it was bound by instructions first (975 us
// at 190 a pack, now about 140, 85 % of the issue slots), not by memory.
template <typename T, int V, int J>
__global__ void __launch_bounds__(kThreads) rows_forward_kernel(const GroupNormArgs a, const RowsShape sh,
                                                                uint32_t passes) {
    using Ring = RowsRing<T, V, J, 1>;
    extern __shared__ uint4 smem[];
    Ring& ring = *reinterpret_cast<Ring*>(smem);
    float* stats = reinterpret_cast<float*>(smem + sizeof(Ring) / 16);  // [2][passes][RB][GB]
    const RowsPlace<V, J> p(a, sh);
    const float inv = 1.f / ((float)a.S * (float)(a.C / a.G));
    const uint64_t first = (uint64_t)blockIdx.x * passes * sh.RB;
    const uint32_t rows = (uint32_t)min((uint64_t)passes * sh.RB, a.N - first);  // of the CTA
    const T* x = static_cast<const T*>(a.x) + (first + p.rb) * a.S * a.ldx;
    T* y = static_cast<T*>(a.y) + (first + p.rb) * a.S * a.ldy;
    if constexpr (Ring::kAsync) {
        const T* at = x;
#pragma unroll
        for (uint32_t d = 0; d < Ring::D; ++d) {
            if (d * sh.RB + p.rb < rows)
#pragma unroll
                for (int j = 0; j < J; ++j)
                    if (p.ok[j]) copy_pack_async<T, V>(&ring.slot[d][0][j][threadIdx.x], at + p.at(j, a.ldx));
            commit_copies();
            at = advance(at, sh.x_step);
        }
    }
#pragma unroll
    for (uint32_t d = 0; d < Ring::D; ++d) {
        if (d >= passes) break;
        const bool on = d * sh.RB + p.rb < rows;
        Vec<V> v[J];
        if constexpr (Ring::kAsync) wait_pass<Ring::D>(d);
#pragma unroll
        for (int j = 0; j < J; ++j) {
            v[j] = splat<V>(0.f);
            if (p.ok[j] && on) {
                if constexpr (Ring::kAsync) v[j] = widen<T, V>(load_pack<T, V>(ring.slot[d][0][j][threadIdx.x].v));
                else v[j] = widen<T, V>(load_pack_cs<T, V>(x + p.at(j, a.ldx)));
            }
        }
        x = advance(x, sh.x_step);
        float s = 0.f, q = 0.f;
#pragma unroll
        for (int j = 0; j < J; ++j) s += sum(v[j]);
        const float mean = lane_sum(s, sh.L) * inv;
#pragma unroll
        for (int j = 0; j < J; ++j) {
            v[j] = add(v[j], splat<V>(-mean));
            if (p.ok[j]) q += dot(v[j], v[j]);
        }
        const float r = inverse_root(lane_sum(q, sh.L) * inv + a.eps);
        if (on && p.on && p.lane == 0 && a.mean) {
            const uint32_t at = (d * sh.RB + p.rb) * sh.GB + (p.g - blockIdx.y * sh.GB);
            stats[at] = mean;
            stats[passes * sh.RB * sh.GB + at] = r;
        }
#pragma unroll
        for (int j = 0; j < J; ++j)
            if (p.ok[j] && on)
                store_pack_cs<T, V>(y + p.at(j, a.ldy),
                                    narrow<T, V>(activate<T, V>(a.act, fma(mul(v[j], splat<V>(r)), p.w[j], p.b[j]))));
        y = advance(y, sh.y_step);
    }
    if (!a.mean) return;
    __syncthreads();
    const uint32_t g0 = blockIdx.y * sh.GB, groups = min(sh.GB, a.G - g0);
    for (uint32_t i = threadIdx.x; i < rows * groups; i += kThreads) {
        const uint32_t row = i / groups, g = i - row * groups;
        const uint64_t to = (first + row) * a.G + g0 + g;
        a.mean[to] = stats[row * sh.GB + g];
        a.rstd[to] = stats[passes * sh.RB * sh.GB + row * sh.GB + g];
    }
}

// Parameter gradients: a thread's sums over its rows (kept in two levels, so
// that the rounding error does not grow with the number of rows), then over
// the CTA's RB samples in shared memory; S partial rows per CTA of the grid's x.
// 2.4 M x 256 fp32: 1142 us for 7.7 GB, 6.7 TB/s; in bf16 782 us, 5.0 TB/s (there
// a lane holds 8 values: 120 registers, two CTAs per SM).
template <typename T, int V, int J>
__global__ void __launch_bounds__(kThreads, V * J <= 4 ? 4 : V * J <= 8 ? 2 : 1) rows_backward_kernel(const GroupNormArgs a, const RowsShape sh,
                                                                 float* __restrict__ partial) {
    after_previous();
    using Ring = RowsRing<T, V, J, 2>;
    extern __shared__ uint4 smem[];
    Ring& ring = *reinterpret_cast<Ring*>(smem);
    const RowsPlace<V, J> p(a, sh);
    const float inv = 1.f / ((float)a.S * (float)(a.C / a.G));
    const T* x = static_cast<const T*>(a.x);
    const T* dy = static_cast<const T*>(a.dy);
    T* dx = static_cast<T*>(a.dx);
    Vec<V> dw[J], db[J], dw2[J], db2[J];
#pragma unroll
    for (int j = 0; j < J; ++j) dw[j] = db[j] = dw2[j] = db2[j] = splat<V>(0.f);
    const uint64_t stride = (uint64_t)gridDim.x * sh.RB, first = (uint64_t)blockIdx.x * sh.RB;
    // passes of the CTA, and of this thread (the last may end before its row)
    const uint32_t passes = first < a.N ? (uint32_t)((a.N - 1 - first) / stride) + 1 : 0;
    const uint32_t mine = p.on && first + p.rb < a.N ? (uint32_t)((a.N - 1 - first - p.rb) / stride) + 1 : 0;
    // with one pack a lane the pointers hold its place already
    auto from = [&](int j, uint64_t ld) { return J == 1 ? 0 : p.at(j, ld); };
    auto start = [&](uint64_t ld) { return (first + p.rb) * a.S * ld + (J == 1 ? p.at(0, ld) : 0); };
    const T* x_next = x + start(a.ldx);
    const T* dy_next = dy + start(a.lddy);
    T* dx_now = dx + start(a.lddx);
    const float* stats_next = a.mean + (first + p.rb) * a.G + p.g;
    const int64_t to_rstd = a.rstd - a.mean;
    auto fetch = [&](uint32_t k, uint32_t d) {
        if (k < mine)
#pragma unroll
            for (int j = 0; j < J; ++j)
                if (p.ok[j]) {
                    copy_pack_async<T, V>(&ring.slot[d][0][j][threadIdx.x], x_next + from(j, a.ldx));
                    copy_pack_async<T, V>(&ring.slot[d][1][j][threadIdx.x], dy_next + from(j, a.lddy));
                }
        commit_copies();
        x_next = advance(x_next, sh.x_step);
        dy_next = advance(dy_next, sh.dy_step);
    };
    // the statistics of the next row, one row ahead
    float mean_next = 0.f, rstd_next = 0.f;
    auto fetch_stats = [&](uint32_t k) {
        if (k < mine) {
            mean_next = *stats_next;
            rstd_next = stats_next[to_rstd];
        }
        stats_next = advance(stats_next, sh.stats_step);
    };
    // a slot is filled again one row after it was read, when its values are in use already
    if constexpr (Ring::kAsync)
        for (uint32_t d = 0; d + 1 < Ring::D; ++d) fetch(d, d);
    fetch_stats(0);
    uint32_t d = 0, put = Ring::D - 1, since = 0;
#pragma unroll 1
    for (uint32_t k = 0; k < passes; ++k) {
        const bool live = k < mine;
        const float mean = mean_next, r = rstd_next;
        fetch_stats(k + 1);
        Vec<V> h[J], g[J];
        if constexpr (Ring::kAsync) {
            fetch(k + Ring::D - 1, put);
            put = put + 1 == Ring::D ? 0 : put + 1;
            wait_copies<Ring::D - 1>();
        }
#pragma unroll
        for (int j = 0; j < J; ++j) {
            h[j] = g[j] = splat<V>(0.f);
            if (p.ok[j] && live) {
                if constexpr (Ring::kAsync) {
                    h[j] = widen<T, V>(load_pack<T, V>(ring.slot[d][0][j][threadIdx.x].v));
                    g[j] = widen<T, V>(load_pack<T, V>(ring.slot[d][1][j][threadIdx.x].v));
                } else {
                    h[j] = widen<T, V>(load_pack_cs<T, V>(x_next + from(j, a.ldx)));
                    g[j] = widen<T, V>(load_pack_cs<T, V>(dy_next + from(j, a.lddy)));
                }
                h[j] = mul(add(h[j], splat<V>(-mean)), splat<V>(r));
            }
        }
        if constexpr (Ring::kAsync) {
            d = d + 1 == Ring::D ? 0 : d + 1;
        } else {
            x_next = advance(x_next, sh.x_step);
            dy_next = advance(dy_next, sh.dy_step);
        }
        float s = 0.f, q = 0.f;
#pragma unroll
        for (int j = 0; j < J; ++j) {
            if (a.act != TCC_ACT_NONE) g[j] = activate_grad<T, V>(a.act, fma(h[j], p.w[j], p.b[j]), g[j]);
            db[j] = add(db[j], g[j]);
            dw[j] = fma(g[j], h[j], dw[j]);
            g[j] = mul(g[j], p.w[j]);
            s += sum(g[j]);
            q += dot(g[j], h[j]);
        }
        if (dx) {
            s = lane_sum(s, sh.L) * inv;
            q = lane_sum(q, sh.L) * inv;
#pragma unroll
            for (int j = 0; j < J; ++j)
                if (p.ok[j] && live)
                    store_pack_cs<T, V>(dx_now + from(j, a.lddx),
                                        narrow<T, V>(mul(splat<V>(r), fma(h[j], splat<V>(-q),
                                                                          add(g[j], splat<V>(-s))))));
            dx_now = advance(dx_now, sh.dx_step);
        }
        if (++since == sh.level) {
            since = 0;
#pragma unroll
            for (int j = 0; j < J; ++j) {
                dw2[j] = add(dw2[j], dw[j]);
                db2[j] = add(db2[j], db[j]);
                dw[j] = db[j] = splat<V>(0.f);
            }
        }
    }
    if (!partial) return;
    if constexpr (Ring::kAsync) wait_copies<0>();
    float* sm = reinterpret_cast<float*>(smem);  // [2][kThreads][V], in the ring's place
    static_assert(sizeof(Ring) >= 2 * kThreads * V * sizeof(float) || !Ring::kAsync, "sums fit");
    // Where the lanes of a slot meet a channel again in other rows of a sample
    // at a power of two apart, they add up first; else each row is left by itself.
    const bool fold = a.S > 1 && sh.PG <= sh.L && (sh.PG & (sh.PG - 1)) == 0;
#pragma unroll
    for (int j = 0; j < J; ++j) {
        dw[j] = add(dw2[j], dw[j]);
        db[j] = add(db2[j], db[j]);
    }
    if (fold) {
#pragma unroll
        for (int j = 1; j < J; ++j) {
            dw[0] = add(dw[0], dw[j]);
            db[0] = add(db[0], db[j]);
        }
        for (uint32_t o = sh.PG; o < sh.L; o <<= 1) {
#pragma unroll
            for (int k = 0; k < V; ++k) {
                dw[0].v[k] += __shfl_xor_sync(0xffffffffu, dw[0].v[k], o);
                db[0].v[k] += __shfl_xor_sync(0xffffffffu, db[0].v[k], o);
            }
        }
    }
    const uint32_t across = sh.GB * sh.L * V;  // values of a row of slots
#pragma unroll
    for (int j = 0; j < J; ++j) {
        if (fold && j) break;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < V; ++k) {
            sm[threadIdx.x * V + k] = dw[j].v[k];
            sm[(kThreads + threadIdx.x) * V + k] = db[j].v[k];
        }
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < 2 * across; i += kThreads) {
            const uint32_t which = i >= across, e = i - which * across;
            const uint32_t slot = e / V >> sh.log_L, lane = (e / V) & (sh.L - 1);
            const uint32_t g = blockIdx.y * sh.GB + slot, pk = j * sh.L + lane, row = pk / sh.PG;
            if (g >= a.G || pk >= (fold ? sh.PG : sh.packs)) continue;
            const float t = strided_sum(sm + which * kThreads * V + e, across, sh.RB);
            const uint64_t to = fold ? blockIdx.x : (uint64_t)blockIdx.x * a.S + row;
            partial[(to * 2 + which) * a.C + g * (a.C / a.G) + (pk - row * sh.PG) * V + e % V] = t;
        }
    }
}

// dweight, dbias [C] = column sums of partial [rows][2][C], in 64 bits; a CTA
// takes 8 columns (a sector of a row) by 128 rows of threads.
__global__ void __launch_bounds__(1024) param_grad_kernel(const float* partial, uint64_t rows, uint32_t C,
                                                          void* dweight, void* dbias, int type) {
    after_previous();
    __shared__ double sm[32][8];
    const uint32_t tx = threadIdx.x & 7, ty = threadIdx.x >> 3;
    const uint64_t c = (uint64_t)blockIdx.x * 8 + tx;  // of 2 C
    double s = 0.0;
    if (c < 2ull * C) {
#pragma unroll 4
        for (uint64_t r = ty; r < rows; r += 128) s += (double)partial[r * 2 * C + c];
    }
    s += __shfl_xor_sync(0xffffffffu, s, 8);
    s += __shfl_xor_sync(0xffffffffu, s, 16);
    if ((threadIdx.x & 31) < 8) sm[threadIdx.x >> 5][tx] = s;
    __syncthreads();
    if (threadIdx.x < 8 && c < 2ull * C) {
        double t = 0.0;
        for (int i = 0; i < 32; ++i) t += sm[i][tx];
        void* out = c < C ? dweight : dbias;
        if (out) store_typed(out, type, c < C ? c : c - C, (float)t);
    }
}

inline void launch_param_grad(const GroupNormArgs& a, const float* partial, uint64_t rows, cudaStream_t s) {
    launch_after(param_grad_kernel, (2 * a.C + 7) / 8, 1024, 0, s, partial, rows, a.C, a.dweight, a.dbias,
                 a.param_type);
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

// `item`: of the N * chunks chunks of all samples.
template <int V>
__device__ __forceinline__ SplitPlace split_place(const GroupNormArgs& a, const SplitShape& sh, uint32_t item) {
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
    p.n = item / sh.chunks;
    p.chunk = item - (uint32_t)p.n * sh.chunks;
    p.row0 = p.chunk * sh.chunk_rows;
    p.row1 = min(p.row0 + sh.chunk_rows, a.S);
    return p;
}

// First channel of the grid's block of columns.
template <int V>
__device__ __forceinline__ uint32_t block_channel(const SplitShape& sh) {
    if (sh.SUB == 1) return blockIdx.y * sh.GPB * sh.PG * V;
    const uint32_t g = blockIdx.y / sh.SUB;
    return (g * sh.PG + (blockIdx.y - g * sh.SUB) * sh.TX) * V;
}

struct Moments {
    float n, mean, m2;
};

// The division is the hardware's, off by two units in the last place: what it
// weighs is a difference of means, so it costs no more than the sums' own roundings.

__device__ __forceinline__ Moments merge(const Moments& a, const Moments& b) {
    Moments o;
    o.n = a.n + b.n;
    const float f = o.n > 0.f ? __fdividef(b.n, o.n) : 0.f;
    const float d = b.mean - a.mean;
    o.mean = a.mean + d * f;
    o.m2 = a.m2 + b.m2 + d * d * a.n * f;
    return o;
}

// Calls body(packs[B][A], how many of the B rows there are) for `count` rows of
// A arrays, `inc` elements from one row to the next, B rows at a time; the next
// D rows are on their way into the thread's part of `ring` ([D][A][kThreads])
// meanwhile.  Registers hold B rows only, so that enough warps fit to hide the
// exponentials and the memory (rows prefetched into registers: 128 registers,
// 100 us in place of 52 for the sums of 232,965 x 256 bf16).  Of the four passes
// over that graph the first takes 25 us, the others 41, 50 and 55, at 54 to 67 %
// of the issue slots; in the last three the pipe of the exponentials is 54 to 73 %
// busy, with 20 of 64 warps.
template <typename T, int V, int A, int D, int B, typename Body>
__device__ __forceinline__ void stream_rows(void* smem, const T* const (&from)[A], const int64_t (&inc)[A],
                                            uint32_t count, Body&& body) {
    constexpr bool kAsync = sizeof(Pack<T, V>) >= 4;
    Pack<T, V>* ring = static_cast<Pack<T, V>*>(smem) + threadIdx.x;
    const T* at[A];
#pragma unroll
    for (int i = 0; i < A; ++i) at[i] = from[i];
    auto fetch = [&](uint32_t k) {
        if (k < count)
#pragma unroll
            for (int i = 0; i < A; ++i) {
                copy_pack_async<T, V>(ring + ((k & (D - 1)) * A + i) * kThreads, at[i]);
                at[i] += inc[i];
            }
        commit_copies();
    };
    // a slot is filled again one step after it was read, when its values are in use already
    if constexpr (kAsync)
        for (uint32_t k = 0; k < D - B; ++k) fetch(k);
#pragma unroll 1
    for (uint32_t k = 0; k < count; k += B) {
        Pack<T, V> v[B][A];
        if constexpr (kAsync) {
#pragma unroll
            for (int u = 0; u < B; ++u) fetch(k + D - B + u);
            wait_copies<D - B>();
        }
#pragma unroll
        for (int u = 0; u < B; ++u)
            if (k + u < count)
#pragma unroll
                for (int i = 0; i < A; ++i) {
                    if constexpr (kAsync) {
                        v[u][i] = load_pack<T, V>(ring[(((k + u) & (D - 1)) * A + i) * kThreads].v);
                    } else {
                        v[u][i] = load_pack<T, V>(at[i]);
                        at[i] += inc[i];
                    }
                }
        body(v, min((uint32_t)B, count - k));
    }
    if constexpr (kAsync) wait_copies<0>();
}

// Rows of this thread in its chunk.
__device__ __forceinline__ uint32_t own_rows(const SplitPlace& p, const SplitShape& sh) {
    const uint64_t first = p.row0 + p.rb;
    return p.on && first < p.row1 ? (uint32_t)((p.row1 - 1 - first) / sh.RB) + 1 : 0;
}

constexpr int kBlockRows = 4;               // rows of a thread's block of values
constexpr int kDepth1 = 8, kDepth2 = 4;     // rows ahead of one array, of two
template <typename T, int V, int A>
constexpr size_t ring_bytes() {
    return (A == 1 ? kDepth1 : kDepth2) * A * kThreads * sizeof(Pack<T, V>);
}

// The threads' sums of split_sums_kernel take the ring's place.
template <typename T, int V>
constexpr size_t sums_bytes() {
    return std::max(ring_bytes<T, V, 2>(), 2 * kThreads * V * sizeof(float));
}

// Moments of a thread's block of up to kBlockRows rows, around the block's own mean.
template <typename T, int V, typename Packs>
__device__ __forceinline__ Moments block_of(const Packs& pk, uint32_t rows) {
    Vec<V> v[kBlockRows], t = splat<V>(0.f);
    if (rows == kBlockRows) {  // all but a chunk's last: no row to leave out
#pragma unroll
        for (int u = 0; u < kBlockRows; ++u) {
            v[u] = widen<T, V>(pk[u][0]);
            t = add(t, v[u]);
        }
        const Vec<V> less = splat<V>(sum(t) * (-1.f / (kBlockRows * V)));
        t = splat<V>(0.f);
#pragma unroll
        for (int u = 0; u < kBlockRows; ++u) {
            const Vec<V> e = add(v[u], less);
            t = fma(e, e, t);
        }
        return Moments{(float)(kBlockRows * V), -less.v[0], sum(t)};
    }
#pragma unroll
    for (uint32_t u = 0; u < kBlockRows; ++u) {
        v[u] = u < rows ? widen<T, V>(pk[u][0]) : splat<V>(0.f);
        t = add(t, v[u]);
    }
    const float n = (float)(rows * V), mean = __fdividef(sum(t), n);
    t = splat<V>(0.f);
#pragma unroll
    for (uint32_t u = 0; u < kBlockRows; ++u)
        if (u < rows) {
            const Vec<V> e = add(v[u], splat<V>(-mean));
            t = fma(e, e, t);
        }
    return Moments{n, mean, sum(t)};
}

// The threads' moments merged per group part: at sm[thread] of its first pack, row 0.
__device__ __forceinline__ void block_moments(const SplitPlace& p, const SplitShape& sh, const Moments& m,
                                              Moments* sm) {
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
}

template <typename T, int V>
__global__ void __launch_bounds__(kThreads, 3) split_moments_kernel(const GroupNormArgs a, const SplitShape sh,
                                                                    Moments* __restrict__ partial) {
    after_previous();
    extern __shared__ uint4 smem[];
    const SplitPlace p = split_place<V>(a, sh, blockIdx.x);
    const T* const from[1] = {static_cast<const T*>(a.x) + (p.n * a.S + p.row0 + p.rb) * a.ldx + p.c};
    const int64_t inc[1] = {(int64_t)(sh.RB * a.ldx)};
    __shared__ Moments sm[kThreads];  // the second level, then the CTA's
    Moments m{0.f, 0.f, 0.f};
    sm[threadIdx.x] = m;
    uint32_t since = 0;
    stream_rows<T, V, 1, kDepth1, kBlockRows>(smem, from, inc, own_rows(p, sh), [&](const auto& pk, uint32_t rows) {
        m = merge(m, block_of<T, V>(pk, rows));
        if (++since == kLevel) {
            since = 0;
            sm[threadIdx.x] = merge(sm[threadIdx.x], m);
            m = Moments{0.f, 0.f, 0.f};
        }
    });
    block_moments(p, sh, merge(sm[threadIdx.x], m), sm);
    if (p.on && p.rb == 0 && p.gi == 0)
        partial[(p.n * sh.chunks + p.chunk) * ((uint64_t)a.G * sh.SUB) + p.slot] = sm[threadIdx.x];
}

// A CTA of 1, 8 or 32 warps per (sample, group) merges its partial moments.
__global__ void split_stats_kernel(const Moments* partial, uint32_t G, uint32_t SUB, uint32_t chunks, float eps, float* mean,
                                   float* rstd) {
    after_previous();
    __shared__ Moments sm[32];
    const uint64_t n = blockIdx.x / G;
    const uint32_t g = (uint32_t)(blockIdx.x - n * G);
    Moments m{0.f, 0.f, 0.f};
    for (uint32_t k = threadIdx.x; k < chunks * SUB; k += blockDim.x) {
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
    if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = m;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (uint32_t w = 1; w < blockDim.x / 32; ++w) m = merge(m, sm[w]);
        mean[blockIdx.x] = m.mean;
        rstd[blockIdx.x] = inverse_root(m.m2 / m.n + eps);
    }
}

template <typename T, int V>
__global__ void __launch_bounds__(kThreads) split_apply_kernel(const GroupNormArgs a, const SplitShape sh,
                                                               const float* mean_, const float* rstd_) {
    after_previous();
    extern __shared__ uint4 smem[];
    const SplitPlace p = split_place<V>(a, sh, gridDim.x - 1 - blockIdx.x);
    const uint32_t count = own_rows(p, sh);
    if (!count) return;
    const uint64_t last = p.n * a.S + p.row0 + p.rb + (uint64_t)(count - 1) * sh.RB;
    const T* const from[1] = {static_cast<const T*>(a.x) + last * a.ldx + p.c};
    const int64_t inc[1] = {-(int64_t)(sh.RB * a.ldx)};
    T* y = static_cast<T*>(a.y) + last * a.ldy + p.c;
    const Vec<V> less = splat<V>(-mean_[p.n * a.G + p.g]), rstd = splat<V>(rstd_[p.n * a.G + p.g]);
    Vec<V> w, b;
    load_params<V>(a, p.c, true, w, b);
    stream_rows<T, V, 1, kDepth1, 1>(smem, from, inc, count, [&](const auto& pk, uint32_t) {
        const Vec<V> h = mul(add(widen<T, V>(pk[0][0]), less), rstd);
        store_pack_cs<T, V>(y, narrow<T, V>(activate<T, V>(a.act, fma(h, w, b))));
        y -= sh.RB * a.ldy;
    });
}

// Per chunk and channel: sums of dz * h and of dz -> partial [N][chunks][2][C].
template <typename T, int V>
__global__ void __launch_bounds__(kThreads, 3) split_sums_kernel(const GroupNormArgs a, const SplitShape sh,
                                                                 float* __restrict__ partial) {
    after_previous();
    const SplitPlace p = split_place<V>(a, sh, blockIdx.x);
    extern __shared__ uint4 smem[];
    float(*all)[kThreads] = reinterpret_cast<float(*)[kThreads]>(
        reinterpret_cast<char*>(smem) + sums_bytes<T, V>());  // [2 V]: the second level
#pragma unroll
    for (int k = 0; k < 2 * V; ++k) all[k][threadIdx.x] = 0.f;
    Vec<V> dw = splat<V>(0.f), db = dw;
    if (const uint32_t count = own_rows(p, sh)) {
        const uint64_t first = p.n * a.S + p.row0 + p.rb;
        const T* const from[2] = {static_cast<const T*>(a.x) + first * a.ldx + p.c,
                                  static_cast<const T*>(a.dy) + first * a.lddy + p.c};
        const int64_t inc[2] = {(int64_t)(sh.RB * a.ldx), (int64_t)(sh.RB * a.lddy)};
        const Vec<V> less = splat<V>(-a.mean[p.n * a.G + p.g]), rstd = splat<V>(a.rstd[p.n * a.G + p.g]);
        Vec<V> w, b;
        load_params<V>(a, p.c, true, w, b);
        uint32_t since = 0;
        stream_rows<T, V, 2, kDepth2, 1>(smem, from, inc, count, [&](const auto& pk, uint32_t) {
            const Vec<V> h = mul(add(widen<T, V>(pk[0][0]), less), rstd);
            const Vec<V> d = activate_grad<T, V>(a.act, fma(h, w, b), widen<T, V>(pk[0][1]));
            db = add(db, d);
            dw = fma(d, h, dw);
            if (++since == kLevel) {
                since = 0;
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    all[k][threadIdx.x] += dw.v[k];
                    all[V + k][threadIdx.x] += db.v[k];
                }
                dw = db = splat<V>(0.f);
            }
        });
    }
    __syncthreads();
    float(*sm)[kThreads * V] = reinterpret_cast<float(*)[kThreads * V]>(smem);  // [2], in the ring's place
#pragma unroll
    for (int k = 0; k < V; ++k) {
        sm[0][threadIdx.x * V + k] = all[k][threadIdx.x] + dw.v[k];
        sm[1][threadIdx.x * V + k] = all[V + k][threadIdx.x] + db.v[k];
    }
    __syncthreads();
    // channels of the block, then the rows of threads
    const uint32_t across = sh.TX * V, c0 = block_channel<V>(sh);
    const uint32_t c1 = min(c0 + across, sh.SUB == 1 ? a.C : (blockIdx.y / sh.SUB + 1) * (a.C / a.G));
    float* out = partial + (p.n * sh.chunks + p.chunk) * 2 * a.C;
    for (uint32_t i = threadIdx.x; i < 2 * across; i += kThreads) {
        const uint32_t which = i >= across, e = i - which * across;
        if (c0 + e >= c1) continue;
        out[which * a.C + c0 + e] = strided_sum(&sm[which][e], across, sh.RB);
    }
}

// group_sums [N][G][2]: a = sum of weight * (sum dz), b = sum of weight * (sum
// dz * h), from the chunks' sums; a CTA per (sample, group), `cw` channels at a
// time (a power of two up to a warp) by blockDim.x / cw threads over the
// chunks.  With one sample the channels' sums are the parameters' gradients.
__global__ void split_groups_kernel(const GroupNormArgs a, const float* partial, uint32_t chunks, uint32_t cw,
                                    float* group_sums, bool params) {
    after_previous();
    __shared__ double sm[2][32][32];
    const uint64_t n = blockIdx.x / a.G;
    const uint32_t g = (uint32_t)(blockIdx.x - n * a.G), Cg = a.C / a.G;
    const uint32_t tx = threadIdx.x % cw, ty = threadIdx.x / cw, rows = blockDim.x / cw, warps = blockDim.x / 32;
    double s = 0.0, q = 0.0;  // of the group; in the first cw threads
    for (uint32_t k0 = 0; k0 < Cg; k0 += cw) {
        const uint32_t c = g * Cg + k0 + tx;
        const bool on = k0 + tx < Cg;
        double tw = 0.0, tb = 0.0;
        if (on) {
#pragma unroll 4
            for (uint32_t i = ty; i < chunks; i += rows) {
                const float* row = partial + (n * chunks + i) * 2 * a.C + c;
                tw += (double)row[0];
                tb += (double)row[a.C];
            }
        }
        for (uint32_t o = 16; o >= cw; o >>= 1) {  // the rows of threads in a warp
            tw += __shfl_xor_sync(0xffffffffu, tw, o);
            tb += __shfl_xor_sync(0xffffffffu, tb, o);
        }
        __syncthreads();
        if ((threadIdx.x & 31) < cw) {
            sm[0][threadIdx.x >> 5][tx] = tw;
            sm[1][threadIdx.x >> 5][tx] = tb;
        }
        __syncthreads();
        if (threadIdx.x < cw && on) {
            for (uint32_t i = 1; i < warps; ++i) {
                tw += sm[0][i][tx];
                tb += sm[1][i][tx];
            }
            const double w = a.weight ? (double)load_typed(a.weight, a.param_type, c) : 1.0;
            q += w * tw;
            s += w * tb;
            if (params && a.dweight) store_typed(a.dweight, a.param_type, c, (float)tw);
            if (params && a.dbias) store_typed(a.dbias, a.param_type, c, (float)tb);
        }
    }
    if (threadIdx.x < 32) {
        for (int o = 16; o; o >>= 1) {
            s += __shfl_xor_sync(0xffffffffu, s, o);
            q += __shfl_xor_sync(0xffffffffu, q, o);
        }
        if (threadIdx.x == 0) {
            group_sums[2 * blockIdx.x] = (float)s;
            group_sums[2 * blockIdx.x + 1] = (float)q;
        }
    }
}

// The sums of many samples: a CTA takes every gridDim.x-th chunk of its columns and
// keeps the parameters' sums to itself, in 64 bits, so that it leaves one row of
// partial [grid][2][C] (or NULL) however many samples there are; the row per chunk of
// split_sums_kernel would be twice the input for samples of one row.  What dx
// needs of a chunk are two sums per part of a group: parts [N][chunks][G * SUB] =
// (sum of weight * dz, sum of weight * dz * h), or NULL.
template <typename T, int V>
__global__ void __launch_bounds__(kThreads, 3) split_samples_kernel(const GroupNormArgs a, const SplitShape sh,
                                                                    float* __restrict__ partial,
                                                                    float2* __restrict__ parts) {
    after_previous();
    extern __shared__ uint4 smem[];
    double(*all)[kThreads] = reinterpret_cast<double(*)[kThreads]>(
        reinterpret_cast<char*>(smem) + ring_bytes<T, V, 2>());  // [2 V]: this thread's dweight, dbias
    __shared__ float2 sums[kThreads];
    const uint32_t items = (uint32_t)a.N * sh.chunks, lane = threadIdx.x & 31;
    SplitPlace p = split_place<V>(a, sh, 0);
    Vec<V> w, b;
    load_params<V>(a, p.c, p.on, w, b);
#pragma unroll
    for (int k = 0; k < 2 * V; ++k) all[k][threadIdx.x] = 0.0;
    for (uint32_t item = blockIdx.x; item < items; item += gridDim.x) {
        p = split_place<V>(a, sh, item);
        float s = 0.f, q = 0.f;
        if (const uint32_t count = own_rows(p, sh)) {
            const uint64_t first = p.n * a.S + p.row0 + p.rb;
            const T* const from[2] = {static_cast<const T*>(a.x) + first * a.ldx + p.c,
                                      static_cast<const T*>(a.dy) + first * a.lddy + p.c};
            const int64_t inc[2] = {(int64_t)(sh.RB * a.ldx), (int64_t)(sh.RB * a.lddy)};
            const Vec<V> less = splat<V>(-a.mean[p.n * a.G + p.g]), rstd = splat<V>(a.rstd[p.n * a.G + p.g]);
            Vec<V> dw = splat<V>(0.f), db = dw;
            auto keep = [&] {
                s += dot(db, w);
                q += dot(dw, w);
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    all[k][threadIdx.x] += (double)dw.v[k];
                    all[V + k][threadIdx.x] += (double)db.v[k];
                }
                dw = db = splat<V>(0.f);
            };
            uint32_t since = 0;
            stream_rows<T, V, 2, kDepth2, 1>(smem, from, inc, count, [&](const auto& pk, uint32_t) {
                const Vec<V> h = mul(add(widen<T, V>(pk[0][0]), less), rstd);
                const Vec<V> d = activate_grad<T, V>(a.act, fma(h, w, b), widen<T, V>(pk[0][1]));
                db = add(db, d);
                dw = fma(d, h, dw);
                if (++since == kLevel) {
                    since = 0;
                    keep();
                }
            });
            keep();
        }
        if (!parts) continue;
        sums[threadIdx.x] = make_float2(s, q);
        __syncthreads();
        // entry e of group i: row e / len of the block's threads, pack e % len of the group's part
        const uint32_t len = sh.SUB == 1 ? sh.PG : p.len, entries = len * sh.RB;
        const uint32_t slots = a.G * sh.SUB, first = blockIdx.y * sh.GPB;  // GPB = 1 where SUB > 1
        const bool alone = entries <= 32;  // a thread a group, or else a warp
        for (uint32_t i = alone ? threadIdx.x : threadIdx.x >> 5; i < sh.GPB && first + i < slots;
             i += alone ? kThreads : kThreads / 32) {
            float2 t = make_float2(0.f, 0.f);
            for (uint32_t e = alone ? 0 : lane; e < entries; e += alone ? 1 : 32) {
                const uint32_t r = e / len;
                const float2 o = sums[r * sh.TX + i * sh.PG + (e - r * len)];
                t.x += o.x;
                t.y += o.y;
            }
            if (!alone) {
                t.x = lane_sum(t.x, 32);
                t.y = lane_sum(t.y, 32);
            }
            if (alone || lane == 0) parts[(uint64_t)item * slots + first + i] = t;
        }
        __syncthreads();
    }
    if (!partial) return;
    __syncthreads();
    const uint32_t across = sh.TX * V, c0 = block_channel<V>(sh);
    const uint32_t c1 = min(c0 + across, sh.SUB == 1 ? a.C : (blockIdx.y / sh.SUB + 1) * (a.C / a.G));
    float* out = partial + (uint64_t)blockIdx.x * 2 * a.C;
    for (uint32_t i = threadIdx.x; i < 2 * across; i += kThreads) {
        const uint32_t which = i >= across, e = i - which * across;
        if (c0 + e >= c1) continue;
        double t = 0.0;
        for (uint32_t r = 0; r < sh.RB; ++r) t += all[which * V + e % V][r * sh.TX + e / V];
        out[which * a.C + c0 + e] = (float)t;
    }
}

// group_sums [N][G][2] from the parts of split_samples_kernel, a warp per (sample, group).
__global__ void __launch_bounds__(kThreads) split_parts_kernel(const float2* parts, uint32_t groups, uint32_t G,
                                                               uint32_t SUB, uint32_t chunks, float* group_sums) {
    after_previous();
    const uint32_t i = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (i >= groups) return;
    const uint32_t n = i / G, g = i - n * G;
    double s = 0.0, q = 0.0;
    for (uint32_t k = lane; k < chunks * SUB; k += 32) {
        const uint32_t ch = k / SUB;
        const float2 t = parts[(((uint64_t)n * chunks + ch) * G + g) * SUB + (k - ch * SUB)];
        s += (double)t.x;
        q += (double)t.y;
    }
    for (int o = 16; o; o >>= 1) {
        s += __shfl_xor_sync(0xffffffffu, s, o);
        q += __shfl_xor_sync(0xffffffffu, q, o);
    }
    if (lane == 0) {
        group_sums[2ull * i] = (float)s;
        group_sums[2ull * i + 1] = (float)q;
    }
}

template <typename T, int V>
__global__ void __launch_bounds__(kThreads, 3) split_grad_kernel(const GroupNormArgs a, const SplitShape sh,
                                                                 const float* group_sums) {
    after_previous();
    extern __shared__ uint4 smem[];
    const SplitPlace p = split_place<V>(a, sh, gridDim.x - 1 - blockIdx.x);
    const uint32_t count = own_rows(p, sh);
    if (!count) return;
    const uint64_t last = p.n * a.S + p.row0 + p.rb + (uint64_t)(count - 1) * sh.RB;
    const T* const from[2] = {static_cast<const T*>(a.x) + last * a.ldx + p.c,
                              static_cast<const T*>(a.dy) + last * a.lddy + p.c};
    const int64_t inc[2] = {-(int64_t)(sh.RB * a.ldx), -(int64_t)(sh.RB * a.lddy)};
    T* dx = static_cast<T*>(a.dx) + last * a.lddx + p.c;
    const uint64_t i = p.n * a.G + p.g;
    const float inv = 1.f / ((float)a.S * (float)(a.C / a.G));
    const Vec<V> less = splat<V>(-a.mean[i]), rstd = splat<V>(a.rstd[i]);
    const Vec<V> s = splat<V>(-group_sums[2 * i] * inv), q = splat<V>(-group_sums[2 * i + 1] * inv);
    Vec<V> w, b;
    load_params<V>(a, p.c, true, w, b);
    stream_rows<T, V, 2, kDepth2, 1>(smem, from, inc, count, [&](const auto& pk, uint32_t) {
        const Vec<V> h = mul(add(widen<T, V>(pk[0][0]), less), rstd);
        const Vec<V> d = activate_grad<T, V>(a.act, fma(h, w, b), widen<T, V>(pk[0][1]));
        store_pack_cs<T, V>(dx, narrow<T, V>(mul(rstd, fma(h, q, fma(d, w, s)))));
        dx -= sh.RB * a.lddx;
    });
}

// --------------------------------------------------------- resident form --

namespace cg = cooperative_groups;

// A cluster of sh.chunks CTAs holds a sample, a chunk each; all of a row's
// packs are in one block (sh.cols = 1).  A thread keeps its packs of its rows
// at store[(k * A + array) * kThreads] and reads back only what it copied.  The
// store is followed by the threads' and the groups' sums.
constexpr uint32_t kMaxCluster = 8;

template <int V>
__host__ __device__ __forceinline__ uint32_t resident_store(const SplitShape& sh, uint32_t pack_bytes, uint32_t arrays) {
    return (uint32_t)((sh.chunk_rows + sh.RB - 1) / sh.RB) * kThreads * pack_bytes * arrays;
}

template <typename T, int V, int A>
__device__ __forceinline__ void fetch_resident(Pack<T, V>* store, const T* const (&from)[A],
                                               const uint64_t (&step)[A], uint32_t count) {
    for (uint32_t k = 0; k < count; ++k)
#pragma unroll
        for (int i = 0; i < A; ++i) {
            const T* at = from[i] + k * step[i];
            if constexpr (sizeof(Pack<T, V>) >= 4) copy_pack_async<T, V>(store + (k * A + i) * kThreads, at);
            else store[(k * A + i) * kThreads] = load_pack<T, V>(at);
        }
    commit_copies();
}

template <typename T, int V>
__global__ void __launch_bounds__(kThreads) resident_forward_kernel(const GroupNormArgs a, const SplitShape sh) {
    extern __shared__ uint4 smem[];
    __shared__ Moments sm[kThreads];
    __shared__ Moments group[kThreads];  // of this CTA's chunk; G <= kThreads
    __shared__ float2 stats[kThreads];   // mean and rstd of the sample's groups
    cg::cluster_group cluster = cg::this_cluster();
    const SplitPlace p = split_place<V>(a, sh, blockIdx.x);
    const uint32_t count = own_rows(p, sh);
    Pack<T, V>* store = reinterpret_cast<Pack<T, V>*>(smem) + threadIdx.x;
    const uint64_t first = p.n * a.S + p.row0 + p.rb;
    const T* const from[1] = {static_cast<const T*>(a.x) + first * a.ldx + p.c};
    const uint64_t step[1] = {sh.RB * a.ldx};
    fetch_resident<T, V, 1>(store, from, step, count);
    Vec<V> w, b;
    load_params<V>(a, p.c, p.on, w, b);
    wait_copies<0>();
    Moments m{0.f, 0.f, 0.f};
    for (uint32_t k = 0; k < count; k += kBlockRows) {
        Pack<T, V> pk[kBlockRows][1];
        const uint32_t rows = min((uint32_t)kBlockRows, count - k);
#pragma unroll
        for (uint32_t u = 0; u < kBlockRows; ++u)
            if (u < rows) pk[u][0] = load_pack<T, V>(store[(k + u) * kThreads].v);
        m = merge(m, block_of<T, V>(pk, rows));
    }
    block_moments(p, sh, m, sm);
    if (p.on && p.rb == 0 && p.gi == 0) group[p.g] = sm[threadIdx.x];
    cluster.sync();
    if (threadIdx.x < a.G) {
        Moments t = *cluster.map_shared_rank(group + threadIdx.x, 0);
        for (uint32_t r = 1; r < sh.chunks; ++r) t = merge(t, *cluster.map_shared_rank(group + threadIdx.x, r));
        const float rstd = inverse_root(t.m2 / t.n + a.eps);
        stats[threadIdx.x] = make_float2(t.mean, rstd);
        if (a.mean && p.chunk == 0) {
            a.mean[p.n * a.G + threadIdx.x] = t.mean;
            a.rstd[p.n * a.G + threadIdx.x] = rstd;
        }
    }
    cluster.sync();  // stats are written, and nobody reads this CTA's moments any more
    if (!count) return;
    T* y = static_cast<T*>(a.y) + first * a.ldy + p.c;
    const Vec<V> less = splat<V>(-stats[p.g].x), rstd = splat<V>(stats[p.g].y);
    for (uint32_t k = 0; k < count; ++k) {
        const Vec<V> h = mul(add(widen<T, V>(load_pack<T, V>(store[k * kThreads].v)), less), rstd);
        store_pack_cs<T, V>(y, narrow<T, V>(activate<T, V>(a.act, fma(h, w, b))));
        y += sh.RB * a.ldy;
    }
}

// A cluster takes every (grid / chunks)-th sample and keeps the sums for the
// parameters' gradients: one row of partial [grid][2][C] per CTA, or NULL.
template <typename T, int V>
__global__ void __launch_bounds__(kThreads) resident_backward_kernel(const GroupNormArgs a, const SplitShape sh,
                                                                     float* __restrict__ partial) {
    after_previous();
    extern __shared__ uint4 smem[];
    float(*sums)[kThreads * V] = reinterpret_cast<float(*)[kThreads * V]>(
        reinterpret_cast<char*>(smem) + resident_store<V>(sh, sizeof(Pack<T, V>), 2));  // [2]: per thread, then channel
    float2* group = reinterpret_cast<float2*>(sums + 2);  // [G]: of this CTA's chunk
    float2* total = group + a.G;                          // [G]: of the sample
    cg::cluster_group cluster = cg::this_cluster();
    SplitPlace p = split_place<V>(a, sh, blockIdx.x);
    const uint32_t count = own_rows(p, sh);
    Pack<T, V>* store = reinterpret_cast<Pack<T, V>*>(smem) + threadIdx.x;
    const uint64_t step[2] = {sh.RB * a.ldx, sh.RB * a.lddy};
    const uint32_t Cg = a.C / a.G, lane = threadIdx.x & 31;
    const float inv = 1.f / ((float)a.S * (float)Cg);
    Vec<V> w, b, all_dw = splat<V>(0.f), all_db = all_dw;
    load_params<V>(a, p.c, p.on, w, b);
    // use(array, channel, sum over the rows of threads); TX * V = C
    auto over_rows = [&](const Vec<V>& dw, const Vec<V>& db, auto&& use) {
#pragma unroll
        for (int k = 0; k < V; ++k) {
            sums[0][threadIdx.x * V + k] = dw.v[k];
            sums[1][threadIdx.x * V + k] = db.v[k];
        }
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < 2 * a.C; i += kThreads) {
            const uint32_t which = i >= a.C, c = i - which * a.C;
            use(which, c, strided_sum(&sums[which][c], a.C, sh.RB));
        }
    };
    // the parameters' sums of up to kLevel samples go to the CTA's row of partial, each by one thread
    float* out = partial + (uint64_t)blockIdx.x * 2 * a.C;
    uint32_t since = 0;
    bool kept = false;
    auto keep = [&] {
        over_rows(all_dw, all_db, [&](uint32_t which, uint32_t c, float t) {
            out[which * a.C + c] = kept ? out[which * a.C + c] + t : t;
        });
        kept = true;
        since = 0;
        all_dw = all_db = splat<V>(0.f);
        __syncthreads();
    };
    for (; p.n < a.N; p.n += gridDim.x / sh.chunks) {  // the same for the whole cluster
        const uint64_t first = p.n * a.S + p.row0 + p.rb;
        const T* const from[2] = {static_cast<const T*>(a.x) + first * a.ldx + p.c,
                                  static_cast<const T*>(a.dy) + first * a.lddy + p.c};
        fetch_resident<T, V, 2>(store, from, step, count);
        const Vec<V> less = splat<V>(p.on ? -a.mean[p.n * a.G + p.g] : 0.f);
        const Vec<V> rstd = splat<V>(p.on ? a.rstd[p.n * a.G + p.g] : 0.f);
        auto row = [&](uint32_t k, Vec<V>& h, Vec<V>& d) {
            h = mul(add(widen<T, V>(load_pack<T, V>(store[(2 * k) * kThreads].v)), less), rstd);
            d = activate_grad<T, V>(a.act, fma(h, w, b), widen<T, V>(load_pack<T, V>(store[(2 * k + 1) * kThreads].v)));
        };
        wait_copies<0>();
        Vec<V> dw = splat<V>(0.f), db = dw;
        for (uint32_t k = 0; k < count; ++k) {
            Vec<V> h, d;
            row(k, h, d);
            db = add(db, d);
            dw = fma(d, h, dw);
        }
        all_dw = add(all_dw, dw);
        all_db = add(all_db, db);
        if (++since == kLevel && partial) keep();
        if (!a.dx) continue;
        // row 0 of the sums becomes the channels' sums: each is read by the thread that writes it
        over_rows(dw, db, [&](uint32_t which, uint32_t c, float t) {
            sums[which][c] = t * (a.weight ? load_typed(a.weight, a.param_type, c) : 1.f);
        });
        __syncthreads();
        for (uint32_t g = threadIdx.x >> 5; g < a.G; g += kThreads / 32) {
            float q = 0.f, t = 0.f;
            for (uint32_t k = lane; k < Cg; k += 32) {
                q += sums[0][g * Cg + k];
                t += sums[1][g * Cg + k];
            }
            q = lane_sum(q, 32);
            t = lane_sum(t, 32);
            if (lane == 0) group[g] = make_float2(t, q);
        }
        cluster.sync();
        if (threadIdx.x < a.G) {
            float2 t = make_float2(0.f, 0.f);
            for (uint32_t i = 0; i < sh.chunks; ++i) {
                const float2 o = *cluster.map_shared_rank(group + threadIdx.x, i);
                t.x += o.x;
                t.y += o.y;
            }
            total[threadIdx.x] = t;
        }
        cluster.sync();  // totals are written, and nobody reads this CTA's sums any more
        if (!count) continue;
        T* dx = static_cast<T*>(a.dx) + first * a.lddx + p.c;
        const Vec<V> s = splat<V>(-total[p.g].x * inv), q = splat<V>(-total[p.g].y * inv);
        for (uint32_t k = 0; k < count; ++k) {
            Vec<V> h, d;
            row(k, h, d);
            store_pack_cs<T, V>(dx, narrow<T, V>(mul(rstd, fma(h, q, fma(d, w, s)))));
            dx += sh.RB * a.lddx;
        }
    }
    if (!partial || (kept && !since)) return;
    __syncthreads();
    keep();
}

// ------------------------------------------------------------------ host --

inline uint64_t align256(uint64_t b) { return (b + 255) / 256 * 256; }

inline int pick_width(const GroupNormArgs& a) {
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

inline RowsShape rows_shape(uint64_t S, uint32_t C, uint32_t G, int V) {
    RowsShape sh{};
    sh.PG = C / G / V;
    sh.packs = (uint32_t)S * sh.PG;
    sh.log_L = 0;
    while (sh.log_L < 5 && (1u << sh.log_L) < sh.packs) ++sh.log_L;
    sh.L = 1u << sh.log_L;
    const uint32_t slots = kThreads / sh.L;
    sh.GB = std::min(G, slots);
    sh.RB = slots / sh.GB;
    return sh;
}

// The rows form: up to 8 packs and 32 values a lane, up to 32 rows; groups that
// fit the grid's y (1 M groups of 32 rows do not).
inline bool rows_form(uint64_t S, uint32_t C, uint32_t G, int V) {
    const uint32_t Cg = C / G;
    if (S > 32 || S * Cg > 32u * std::min(8u * (uint32_t)V, 32u)) return false;
    const RowsShape sh = rows_shape(S, C, G, V);
    return (G + sh.GB - 1) / sh.GB <= 65535;
}

// CTAs in x of the backward: four per SM, which is a whole number of waves (a
// CTA's registers let four, two or one run at once); each leaves one row of
// sums for the parameters' gradients per row of a sample.
inline bool rows_fold(const RowsShape& sh) { return sh.PG <= sh.L && (sh.PG & (sh.PG - 1)) == 0; }
inline uint64_t rows_blocks(const RowsShape& sh, uint64_t N, uint32_t G) {
    const uint64_t y = (G + sh.GB - 1) / sh.GB;
    return std::max<uint64_t>(1, std::min((N + sh.RB - 1) / sh.RB, kSms * 4 / std::min(kSms, y)));
}

// Chunks of a sample: three CTAs per SM over all samples, which run at once (a
// whole number of waves for each of the four kernels; 185 us for 232,965 x 256
// bf16 in place of 195 with eight per SM); at least eight rows a thread, at most
// kLongest.
inline SplitShape split_shape(uint64_t N, uint64_t S, uint32_t C, uint32_t G, int V) {
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
    const uint64_t want = std::max<uint64_t>(1, kSms * 3 / std::max<uint64_t>(1, std::min(N, kSms * 3) * sh.cols));
    const uint64_t most = std::max<uint64_t>(1, S / (8 * sh.RB));
    const uint64_t chunks = std::max(std::min(want, most), (S + (uint64_t)sh.RB * kLongest - 1) / (sh.RB * kLongest));
    sh.chunk_rows = (S + chunks - 1) / chunks;
    sh.chunks = (uint32_t)((S + sh.chunk_rows - 1) / sh.chunk_rows);
    return sh;
}

// Scratch of the split form's backward: rows of [2][C] for the parameters'
// gradients, and two sums per (sample, group), of parts of it first where
// there are several.  A row per chunk while there are few chunks (30 MB at most;
// with one sample split_groups_kernel then gives the parameters' gradients
// too) or long ones (a row is then at most a 64th of a 16-bit chunk, and CTAs that
// the hardware hands out balance better than fixed turns: 3,000 x 2048 x 128 bf16
// 1271 us, a row per CTA 1383); else a row per CTA (1,780 x 33 x 1040 fp32: 230 us, a
// row per chunk 724; 232,965 x 602 fp32 in one group 3.25 and 6.04 ms).
constexpr uint64_t kFewChunks = kSms * 12, kLongChunk = 256;
struct SplitGradPlan {
    bool few;
    uint64_t rows;                             // of [2][C]
    uint64_t parts_bytes, group_bytes, bytes;  // parts_bytes = 0: the sums themselves
};
inline SplitGradPlan split_grad_plan(uint64_t N, uint32_t C, uint32_t G, const SplitShape& sh) {
    SplitGradPlan p{};
    const uint64_t items = N * sh.chunks;
    p.few = items * sh.cols <= kFewChunks || sh.chunk_rows >= kLongChunk;
    p.rows = p.few ? items : std::max<uint64_t>(1, kSms * 3 / sh.cols);
    p.parts_bytes = p.few || sh.chunks * sh.SUB == 1 ? 0 : align256(items * G * sh.SUB * 8);
    p.group_bytes = align256(N * G * 8);
    p.bytes = align256(p.rows * 2 * C * 4) + p.parts_bytes + p.group_bytes;
    return p;
}

// The resident form's cluster, or chunks = 0 where a sample does not fit: two
// CTAs per SM; more CTAs than a sample needs only until every SM has one, and
// while a thread has rows left to share.
constexpr uint64_t kResidentBytes = 112 << 10;

inline uint64_t resident_bytes(const SplitShape& sh, int V, uint32_t G, uint32_t pack_bytes, uint32_t arrays) {
    const uint64_t deep = (sh.chunk_rows + sh.RB - 1) / sh.RB;
    // the forward's sums are in static shared memory, 8 KB
    return deep * kThreads * pack_bytes * arrays + (arrays == 2 ? 2 * kThreads * V * 4 + 2 * G * 8 : 0);
}

inline SplitShape resident_shape(uint64_t N, uint64_t S, uint32_t C, uint32_t G, int V, uint32_t pack_bytes,
                          uint32_t arrays) {
    SplitShape sh{};
    if (C / V > (uint32_t)kThreads || N >= (1ull << 27)) return sh;
    SplitShape r;
    r.PG = C / G / V;
    r.GPB = G;
    r.TX = C / V;
    r.RB = kThreads / r.TX;
    r.SUB = 1;
    r.cols = 1;
    for (uint32_t k = 1; k <= kMaxCluster; k <<= 1) {
        r.chunk_rows = (S + k - 1) / k;
        r.chunks = k;
        if (resident_bytes(r, V, G, pack_bytes, arrays) + (arrays == 1 ? 8 << 10 : 0) > kResidentBytes) continue;
        // a sample alone on few SMs is slower than its chunks on all of them
        // (1 x 4000 x 47 fp32: 17.7 against 9.9 us) unless its threads have little to do
        if (N * k < kSms && r.chunk_rows > 16ull * r.RB) continue;
        sh = r;
        if (N * k >= kSms || r.chunk_rows <= 8ull * r.RB) break;
    }
    return sh;
}
// CTAs of the backward: a cluster goes on with another sample.
inline uint64_t resident_grid(uint64_t N, uint32_t chunks) {
    return std::max(std::min(N, kSms * 8 / chunks), (N + kLevel * kLevel - 1) / (kLevel * kLevel)) * chunks;
}

template <typename T, int V, int J>
void rows_launch(const GroupNormArgs& a, float* partial, bool backward, cudaStream_t s) {
    RowsShape sh = rows_shape(a.S, a.C, a.G, V);
    const uint32_t cols = (a.G + sh.GB - 1) / sh.GB;
    dim3 grid(1, cols);
    if (backward) {
        using Ring = RowsRing<T, V, J, 2>;
        grid.x = (unsigned)rows_blocks(sh, a.N, a.G);
        const uint64_t samples = (uint64_t)grid.x * sh.RB, bytes = samples * a.S * sizeof(T);
        sh.x_step = bytes * a.ldx;
        sh.dy_step = bytes * a.lddy;
        sh.dx_step = bytes * a.lddx;
        sh.stats_step = samples * a.G * sizeof(float);
        sh.level = kLevel;
        while ((uint64_t)sh.level * sh.level * samples < a.N) ++sh.level;
        // where nothing is copied ahead, room for the sums alone
        const size_t smem = std::max<size_t>(Ring::kAsync ? sizeof(Ring) : 0, 2 * kThreads * V * sizeof(float));
        static std::atomic<uint64_t> done{0};
        if (smem > 48 * 1024) allow_smem(rows_backward_kernel<T, V, J>, smem, done);
        rows_backward_kernel<T, V, J><<<grid, kThreads, smem, s>>>(a, sh, partial);
    } else {
        using Ring = RowsRing<T, V, J, 1>;
        // fewer rows a CTA where the ring's would leave SMs idle
        const uint64_t row_passes = (a.N + sh.RB - 1) / sh.RB;
        const uint32_t passes = (uint32_t)std::max<uint64_t>(
            1, std::min<uint64_t>(Ring::D, row_passes * cols / (kSms * 4)));
        grid.x = ceil_div(row_passes, passes);
        sh.x_step = sh.RB * a.S * a.ldx * sizeof(T);
        sh.y_step = sh.RB * a.S * a.ldy * sizeof(T);
        const size_t smem = sizeof(Ring) + (a.mean ? 2 * passes * sh.RB * sh.GB * sizeof(float) : 0);
        static std::atomic<uint64_t> done{0};
        // the statistics take at most 2 D floats a slot
        if (smem > 48 * 1024) allow_smem(rows_forward_kernel<T, V, J>, sizeof(Ring) + 2 * Ring::D * kThreads * 4, done);
        rows_forward_kernel<T, V, J><<<grid, kThreads, smem, s>>>(a, sh, passes);
    }
    TCC_CUDA(cudaGetLastError());
    if (backward && partial) {
        launch_param_grad(a, partial, grid.x * (rows_fold(sh) ? 1 : a.S), s);
    }
}

template <typename T, int V>
void rows_by_packs(const GroupNormArgs& a, float* partial, bool backward, cudaStream_t s) {
    const RowsShape sh = rows_shape(a.S, a.C, a.G, V);
    const uint32_t per_lane = (sh.packs + sh.L - 1) / sh.L;
    if (per_lane <= 1) rows_launch<T, V, 1>(a, partial, backward, s);
    else if (per_lane <= 2) rows_launch<T, V, 2>(a, partial, backward, s);
    else if (per_lane <= 4) rows_launch<T, V, 4>(a, partial, backward, s);
    else if constexpr (V <= 4) rows_launch<T, V, 8>(a, partial, backward, s);
}

template <typename T, int V>
void resident_launch(const GroupNormArgs& a, const SplitShape& sh, float* partial, bool backward, cudaStream_t s) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(backward ? resident_grid(a.N, sh.chunks) : a.N * sh.chunks));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = resident_bytes(sh, V, a.G, sizeof(Pack<T, V>), backward ? 2 : 1);
    cfg.stream = s;
    cudaLaunchAttribute cluster{};
    cluster.id = cudaLaunchAttributeClusterDimension;
    cluster.val.clusterDim.x = sh.chunks;
    cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
    cfg.attrs = &cluster;
    cfg.numAttrs = 1;
    static std::atomic<uint64_t> forward_done{0}, backward_done{0};
    if (backward) {
        allow_smem(resident_backward_kernel<T, V>, kResidentBytes, backward_done);
        TCC_CUDA(cudaLaunchKernelEx(&cfg, resident_backward_kernel<T, V>, a, sh, partial));
        if (partial)
            launch_param_grad(a, partial, cfg.gridDim.x, s);
    } else {
        allow_smem(resident_forward_kernel<T, V>, kResidentBytes, forward_done);
        TCC_CUDA(cudaLaunchKernelEx(&cfg, resident_forward_kernel<T, V>, a, sh));
    }
    TCC_CUDA(cudaGetLastError());
}

template <typename T, int V>
void norm_launch(const GroupNormArgs& a, char* scratch, bool backward, cudaStream_t s) {
    const bool params = backward && (a.dweight || a.dbias);
    if (rows_form(a.S, a.C, a.G, V)) {
        rows_by_packs<T, V>(a, params ? reinterpret_cast<float*>(scratch) : nullptr, backward, s);
        return;
    }
    const uint32_t arrays = backward ? 2 : 1;
    const SplitShape held = resident_shape(a.N, a.S, a.C, a.G, V, sizeof(Pack<T, V>), arrays);
    if (held.chunks) {
        resident_launch<T, V>(a, held, params ? reinterpret_cast<float*>(scratch) : nullptr, backward, s);
        return;
    }
    const SplitShape sh = split_shape(a.N, a.S, a.C, a.G, V);
    TCC_REQUIRE(a.N * sh.chunks < (1ull << 31) && a.N * a.G < (1ull << 31) && sh.cols <= 65535, "too many samples or groups for one call");
    const dim3 grid((unsigned)(a.N * sh.chunks), sh.cols);
    const unsigned groups = (unsigned)(a.N * a.G);
    const bool many = sh.chunks * sh.SUB > 64;  // partial results of a group
    constexpr size_t ring1 = ring_bytes<T, V, 1>(), ring2 = ring_bytes<T, V, 2>();
    if (!backward) {
        Moments* partial = reinterpret_cast<Moments*>(scratch);
        float* mean = a.mean;
        float* rstd = a.rstd;
        if (!mean) {
            mean = reinterpret_cast<float*>(scratch + align256(a.N * sh.chunks * a.G * sh.SUB * sizeof(Moments)));
            rstd = mean + align256(a.N * a.G * 4) / 4;
        }
        split_moments_kernel<T, V><<<grid, kThreads, ring1, s>>>(a, sh, partial);
        const uint32_t merged = sh.chunks * sh.SUB;
        launch_after(split_stats_kernel, groups, merged > 16384 ? 1024 : many ? kThreads : 32, 0, s, partial, a.G, sh.SUB, sh.chunks, a.eps,
                     mean, rstd);
        launch_after(split_apply_kernel<T, V>, grid, kThreads, ring1, s, a, sh, mean, rstd);
    } else {
        const SplitGradPlan plan = split_grad_plan(a.N, a.C, a.G, sh);
        float* partial = reinterpret_cast<float*>(scratch);
        char* after = scratch + align256(plan.rows * 2 * a.C * 4);
        float* group_sums = reinterpret_cast<float*>(after + plan.parts_bytes);
        const bool one = plan.few && params && a.N == 1;  // one sample: its channels' sums are the parameters' gradients
        if (plan.few) {
            split_sums_kernel<T, V><<<grid, kThreads, sums_bytes<T, V>() + 2 * V * kThreads * sizeof(float), s>>>(a, sh, partial);
            if (a.dx || one) {
                uint32_t cw = 1;
                while (cw < 32 && cw < a.C / a.G) cw <<= 1;
                launch_after(split_groups_kernel, groups, many ? 1024 : 128, 0, s, a, partial, sh.chunks, cw,
                             group_sums, one);
            }
        } else {
            constexpr size_t smem = ring2 + 2 * V * kThreads * sizeof(double);
            static std::atomic<uint64_t> done{0};
            if (smem > 46 * 1024) allow_smem(split_samples_kernel<T, V>, smem, done);  // beside 2 KB of static ones
            float2* parts = plan.parts_bytes ? reinterpret_cast<float2*>(after) : reinterpret_cast<float2*>(group_sums);
            split_samples_kernel<T, V><<<dim3((unsigned)plan.rows, sh.cols), kThreads, smem, s>>>(
                a, sh, params ? partial : nullptr, a.dx ? parts : nullptr);
            if (a.dx && plan.parts_bytes)
                launch_after(split_parts_kernel, ceil_div(groups, kThreads / 32), kThreads, 0, s, parts, groups, a.G,
                             sh.SUB, sh.chunks, group_sums);
        }
        if (a.dx) launch_after(split_grad_kernel<T, V>, grid, kThreads, ring2, s, a, sh, group_sums);
        if (params && !one) launch_param_grad(a, partial, plan.rows, s);
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

}  // namespace

}  // namespace tcc
