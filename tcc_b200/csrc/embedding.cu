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

#include <cooperative_groups.h>

#include <algorithm>

namespace tcc {

namespace {

namespace cg = cooperative_groups;

constexpr uint32_t kMaxWidth = 1u << 20;

__device__ __forceinline__ int64_t load_index(const void* idx, int type, uint64_t i) {
    return type == TCC_I64 ? __ldg(static_cast<const long long*>(idx) + i)
                           : (int64_t)__ldg(static_cast<const int*>(idx) + i);
}

// What is the padding of a call without one, INT64_MIN, is an index like any other.
__device__ __forceinline__ bool is_padding(int64_t id, int64_t padding) {
    return id == padding && padding != TCC_NO_PADDING;
}

// ---------------------------------------------------------------- lookup --

constexpr int kLookupThreads = 256;
constexpr uint32_t kLookupRows = 1024;  // of a CTA, at most
constexpr uint32_t kZeroRow = 0xFFFFFFFFu;  // of padding and of bad indices

// A CTA's indices, checked, in shared memory.
__device__ __forceinline__ void load_ids(uint32_t* ids, const void* idx, int idx_type, uint32_t first, uint32_t rows,
                                         int64_t padding, uint32_t num_rows, uint32_t* bad) {
    for (uint32_t i = threadIdx.x; i < rows; i += kLookupThreads) {
        const int64_t id = load_index(idx, idx_type, first + i);
        uint32_t row = kZeroRow;
        if (!is_padding(id, padding)) {
            if (id >= 0 && id < (int64_t)num_rows) row = (uint32_t)id;
            else if (bad) atomicExch(bad, 1u);
        }
        ids[i] = row;
    }
    __syncthreads();
}

// The packs of a CTA's rows in order, whatever a row's length, so that rows of 25
// packs leave no lane idle.  A thread loads its next kAhead packs (32 bytes) while
// it writes those before: 65,537 x 602 fp32 take 55 us, 2 M power-law rows of
// 100 266 at 6.1 TB/s of what they move (a team of lanes per row: 59 and 270).
// Loads go through L1, so that a row that many indices share is not fetched from
// one place of L2 each time (2 M lookups of one row of 400 bytes: 135 us, past L1
// 2141).
template <typename TT, typename TO, int V>
__global__ void __launch_bounds__(kLookupThreads) lookup_kernel(
    const TT* __restrict__ table, uint32_t table_stride, uint32_t num_rows, const void* __restrict__ idx,
    int idx_type, uint32_t n, int64_t padding, float scale, TO* __restrict__ out, uint32_t out_stride,
    uint32_t packs, uint32_t per_pack, uint32_t rows, uint32_t* __restrict__ bad) {
    constexpr int kAhead = sizeof(Pack<TT, V>) == 16 ? 2 : sizeof(Pack<TT, V>) == 8 ? 4 : 8;
    __shared__ uint32_t ids[kLookupRows];
    const uint32_t first = blockIdx.x * rows;
    rows = min(rows, n - first);
    load_ids(ids, idx, idx_type, first, rows, padding, num_rows, bad);
    const char* from = reinterpret_cast<const char*>(table);
    char* to = reinterpret_cast<char*>(out) + (uint64_t)first * out_stride;
    const uint32_t total = rows * packs;
    auto fetch = [&](Pack<TT, V>(&v)[kAhead], uint32_t e0) {
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const uint32_t e = e0 + u * kLookupThreads, row = __umulhi(2 * e, per_pack), c = e - row * packs;
            const uint32_t id = e < total ? ids[row] : kZeroRow;
            v[u] = Pack<TT, V>{};
            if (id != kZeroRow)
                v[u] = load_pack_nc<TT, V>(
                    reinterpret_cast<const TT*>(from + (uint64_t)id * table_stride + c * (uint32_t)sizeof(v[u])));
        }
    };
    auto write = [&](const Pack<TT, V>(&v)[kAhead], uint32_t e0) {
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const uint32_t e = e0 + u * kLookupThreads, row = __umulhi(2 * e, per_pack), c = e - row * packs;
            if (e >= total) break;
            const float f = ids[row] != kZeroRow ? scale : 0.f;  // zeros, whatever the scale
            Pack<TO, V> o;
#pragma unroll
            for (int k = 0; k < V; ++k) o.v[k] = from_f32<TO>(to_f32(v[u].v[k]) * f);
            store_pack_cs<TO, V>(reinterpret_cast<TO*>(to + (uint64_t)row * out_stride + c * (uint32_t)sizeof(o)), o);
        }
    };
    constexpr uint32_t kStep = kAhead * kLookupThreads;
    Pack<TT, V> v[kAhead], w[kAhead];
    uint32_t e = threadIdx.x;
    fetch(v, e);
#pragma unroll 1
    while (e < total) {
        fetch(w, e + kStep);
        write(v, e);
        if (e + kStep >= total) break;
        fetch(v, e + 2 * kStep);
        write(w, e + kStep);
        e += 2 * kStep;
    }
}

// Rows whose width or place no wider pack divides go value by value, where the flat
// order is bound by its index arithmetic (300,000 rows of 333 values out of 50: 182 us).
// Here a team of lanes takes whole rows, PARTS values of each a lane at a time and
// as many rows as make eight: 74 us.
template <typename TT, typename TO, int PARTS>
__global__ void __launch_bounds__(kLookupThreads) lookup_odd_kernel(
    const TT* __restrict__ table, uint32_t table_stride, uint32_t num_rows, const void* __restrict__ idx,
    int idx_type, uint32_t n, int64_t padding, float scale, TO* __restrict__ out, uint32_t out_stride,
    uint32_t width, uint32_t lanes, uint32_t rows, uint32_t* __restrict__ bad) {
    constexpr int kRows = 8 / PARTS;
    __shared__ uint32_t ids[kLookupRows];
    const uint32_t first = blockIdx.x * rows;
    rows = min(rows, n - first);
    load_ids(ids, idx, idx_type, first, rows, padding, num_rows, bad);
    const uint32_t teams = kLookupThreads / lanes, team = threadIdx.x / lanes, step = kRows * teams;
    // with more than one part the team is a warp
#pragma unroll 1
    for (uint32_t c = threadIdx.x % lanes; c - threadIdx.x % lanes < width; c += PARTS * lanes) {
        const char* from = reinterpret_cast<const char*>(table + c);
        char* to = reinterpret_cast<char*>(out + c) + (uint64_t)first * out_stride;
        auto fetch = [&](TT(&v)[8], uint32_t r0) {
#pragma unroll
            for (int q = 0; q < kRows; ++q) {
                const uint32_t r = r0 + q * teams, id = r < rows ? ids[r] : kZeroRow;
                const TT* at = reinterpret_cast<const TT*>(from + (uint64_t)id * table_stride);
#pragma unroll
                for (int p = 0; p < PARTS; ++p) {
                    v[q * PARTS + p] = from_f32<TT>(0.f);
                    if (id != kZeroRow && c + p * 32 < width) v[q * PARTS + p] = __ldg(at + p * 32);
                }
            }
        };
        auto write = [&](const TT(&v)[8], uint32_t r0) {
#pragma unroll
            for (int q = 0; q < kRows; ++q) {
                const uint32_t r = r0 + q * teams;
                if (r >= rows) break;
                TO* at = reinterpret_cast<TO*>(to + (uint64_t)r * out_stride);
                const float f = ids[r] != kZeroRow ? scale : 0.f;  // zeros, whatever the scale
#pragma unroll
                for (int p = 0; p < PARTS; ++p)
                    if (c + p * 32 < width) __stcs(at + p * 32, from_f32<TO>(to_f32(v[q * PARTS + p]) * f));
            }
        };
        TT v[8], w[8];
        uint32_t r = team;
        fetch(v, r);
#pragma unroll 1
        while (r < rows) {
            fetch(w, r + step);
            write(v, r);
            if (r + step >= rows) break;
            fetch(v, r + 2 * step);
            write(w, r + step);
            r += 2 * step;
        }
    }
}

// Teams of at least as many lanes as rows in flight: narrower packs for
// narrow rows.
inline int team_width(int width, uint32_t F) {
    while (width > 1 && F / width < 8) width >>= 1;
    return width;
}

// As many rows a CTA as are asked for, fewer where that would leave less than eight CTAs per SM.
inline uint32_t lookup_rows(uint64_t n, uint32_t rows) {
    rows = std::clamp(rows, 1u, kLookupRows);
    while (rows > 1 && n / rows < 148 * 8) rows >>= 1;
    return rows;
}

template <typename TT, typename TO, int V>
void launch_lookup(const EmbeddingArgs& a, cudaStream_t s) {
    const uint32_t packs = a.F / V;
    const uint32_t rows = lookup_rows(a.n, 4096 / packs);  // of 16,384 packs a CTA: 60 us in place of 53
    // a pack's row is e / packs = the high half of 2 e * per_pack, exact for the e < 2^13 of several rows
    const uint32_t per_pack = rows > 1 ? (uint32_t)(((1ull << 31) + packs - 1) / packs) : 0;
    lookup_kernel<TT, TO, V><<<ceil_div(a.n, rows), kLookupThreads, 0, s>>>(
        static_cast<const TT*>(a.table), (uint32_t)(a.ldt * sizeof(TT)), (uint32_t)a.num_rows, a.idx, a.idx_type,
        (uint32_t)a.n, a.padding, a.scale, static_cast<TO*>(a.rows), (uint32_t)(a.ldr * sizeof(TO)), packs, per_pack,
        rows, a.bad);
    TCC_CUDA(cudaGetLastError());
}

template <typename TT, typename TO, int PARTS>
void launch_lookup_odd(const EmbeddingArgs& a, cudaStream_t s) {
    uint32_t lanes = 8;
    while (lanes < 32 && lanes < a.F) lanes <<= 1;
    const uint32_t rows = lookup_rows(a.n, 4 * (8 / PARTS) * kLookupThreads / lanes);
    lookup_odd_kernel<TT, TO, PARTS><<<ceil_div(a.n, rows), kLookupThreads, 0, s>>>(
        static_cast<const TT*>(a.table), (uint32_t)(a.ldt * sizeof(TT)), (uint32_t)a.num_rows, a.idx, a.idx_type,
        (uint32_t)a.n, a.padding, a.scale, static_cast<TO*>(a.rows), (uint32_t)(a.ldr * sizeof(TO)), a.F, lanes, rows,
        a.bad);
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
        default:
            // whole rows by teams where at least two thirds of their places are taken: of 2 M rows
            // 15 values wide in 64 us (in flat order 72), 1 M of 47 in 84 (98); 9 wide 53 (49), 17 92 (78)
            if (uint32_t places = 8; a.F <= 128) {
                while (places < a.F) places <<= 1;
                if (3 * a.F < 2 * places) return launch_lookup<TT, TO, 1>(a, s);
            }
            if (a.F <= 32) launch_lookup_odd<TT, TO, 1>(a, s);
            else if (a.F <= 64) launch_lookup_odd<TT, TO, 2>(a, s);
            else if (a.F <= 128) launch_lookup_odd<TT, TO, 4>(a, s);
            else launch_lookup_odd<TT, TO, 8>(a, s);
    }
}

// -------------------------------------------------------------- gradient --
//
// The entries (row, position) are put in order of row, then position, and a row
// of the gradient is the sum of its run of entries, read in that order.  With
// few indices (owner form) each CTA owns a range of table rows, collects the
// indices that fall into it and sorts them in shared memory: one launch, no
// scratch.  With many (sorted form) the entries are radix sorted, cut into
// equal ranges of entries whatever the rows' counts (a hub's run crosses many
// ranges), and the partial sums of runs that cross a border are added in order
// by a last small kernel.  Nothing depends on the order in which CTAs run.

constexpr int kThreads = 256;
constexpr uint32_t kUnroll = 8;  // gradient rows in flight per team

using Entry = unsigned long long;  // row << 32 | position
__device__ __forceinline__ uint32_t row_of(Entry e) { return (uint32_t)(e >> 32); }

// Lanes of a team (8, 16 or 32): one pack of a gradient row each (grid.y covers
// the rest).
struct TeamShape {
    uint32_t lanes, teams, packs, blocks;  // blocks: the grid's y
};

TeamShape team_shape(uint32_t packs) {
    TeamShape t;
    t.packs = packs;
    t.lanes = kUnroll;
    while (t.lanes < 32 && t.lanes < packs) t.lanes <<= 1;
    t.teams = kThreads / t.lanes;
    t.blocks = (packs + t.lanes - 1) / t.lanes;
    return t;
}

// What a CTA leaves of the runs that cross its borders.
constexpr uint32_t kHead = 1, kThrough = 2, kTail = 4;
struct Border {
    uint32_t flags;  // kHead: its first run began earlier; kThrough: and goes on; kTail: its last run goes on
    uint32_t row;    // of the tail
};

// A lane's packs of the next kUnroll rows lie in a ring in shared memory, which
// asynchronous copies fill while earlier rows are added; a lane reads back only
// what it copied itself.  (Rows held in registers instead took 64 to 200
// registers a thread: 199 us for the sums of 1 M x 128 alone, in place of 182
// with the zeroing of the other rows beside them.)
template <typename TG, int V>
struct Ring {
    Pack<TG, V> slot[kUnroll][kThreads];
};

// Sums the runs of `count` entries in shared memory, team t the entries
// [t * per, (t + 1) * per).  ent[-1] and ent[count] are the entries before and
// after them (~0: none).  Rows whose run lies inside are written; for the
// others head / tail (fp32, [F]) and *border are, where they are given.  Entries
// of rows >= num_rows, which are the last, are passed over.
template <typename TG, typename TT, int V>
struct RunSums {
    const Entry* ent;
    uint32_t count, per;
    const TG* grad;
    uint32_t grad_stride;  // bytes
    float scale;
    TT* dtable;
    uint64_t ldt;
    uint32_t num_rows;
    TeamShape sh;
    Ring<TG, V>* ring;  // afterwards the teams' heads and tails

    static_assert(sizeof(Ring<TG, V>) >= 2 * kThreads * V * sizeof(float), "heads and tails fit");
    static constexpr bool kAsync = sizeof(Pack<TG, V>) >= 4;

    bool on;
    uint64_t col;
    float acc[V], kept[V];  // kept: the head, while the ring is in use
    uint32_t cur;
    bool open, begun;  // a run is open; it began in this team's range

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int k = 0; k < V; ++k) acc[k] = 0.f;
    }
    __device__ __forceinline__ void write_row() {
        if (!on) return;
        Pack<TT, V> o;
#pragma unroll
        for (int k = 0; k < V; ++k) o.v[k] = from_f32<TT>(acc[k] * scale);
        store_pack_cs<TT, V>(dtable + (uint64_t)cur * ldt + col, o);
    }
    __device__ __forceinline__ const TG* source(Entry e) const {
        return reinterpret_cast<const TG*>(reinterpret_cast<const char*>(grad) +
                                           (uint64_t)(uint32_t)e * grad_stride) + col;
    }
    __device__ __forceinline__ void consume(uint32_t i, uint32_t slot) {
        const uint32_t row = row_of(ent[i]);
        if (row != cur) {
            if (open) {
                if (begun) {
                    write_row();
                } else {
#pragma unroll
                    for (int k = 0; k < V; ++k) kept[k] = acc[k];
                }
            }
            open = begun = true;
            cur = row;
            clear();
        }
        const Pack<TG, V> g = load_pack<TG, V>(ring->slot[slot][threadIdx.x].v);
#pragma unroll
        for (int k = 0; k < V; ++k) acc[k] += to_f32(g.v[k]);
    }

    __device__ __forceinline__ void run(float* head, float* tail, Border* border) {
        __shared__ uint8_t sm_flags[kThreads];
        const uint32_t team = threadIdx.x / sh.lanes, lane = threadIdx.x % sh.lanes;
        const uint32_t pack = blockIdx.y * sh.lanes + lane;
        on = pack < sh.packs;
        col = (uint64_t)pack * V;
        const uint32_t e0 = min(team * per, count);
        uint32_t e1 = min(e0 + per, count);
        while (e1 > e0 && row_of(ent[e1 - 1]) >= num_rows) --e1;  // at the end of the whole list only
        clear();
#pragma unroll
        for (int k = 0; k < V; ++k) kept[k] = 0.f;
        uint32_t flags = 0;
        cur = row_of(ent[(int)e0 - 1]);
        open = begun = false;
        if (e0 < e1 && row_of(ent[e0]) == cur) {  // goes on from an earlier team
            open = true;
            flags = kHead;
        }
        if constexpr (kAsync) {
            auto fetch = [&](uint32_t i) {
                if (i < e1 && on)
                    copy_pack_async<TG, V>(&ring->slot[(i - e0) % kUnroll][threadIdx.x], source(ent[i]));
                commit_copies();
            };
            // a slot is filled again one row after it was read, when its values are in use already
            for (uint32_t u = 0; u + 1 < kUnroll; ++u) fetch(e0 + u);
#pragma unroll 1
            for (uint32_t i = e0; i < e1; ++i) {
                fetch(i + kUnroll - 1);
                wait_copies<kUnroll - 1>();
                consume(i, (i - e0) % kUnroll);
            }
            wait_copies<0>();
        } else {
#pragma unroll 1
            for (uint32_t i = e0; i < e1; i += kUnroll) {
                Pack<TG, V> g[kUnroll];
#pragma unroll
                for (uint32_t u = 0; u < kUnroll; ++u)
                    if (i + u < e1 && on) g[u] = load_pack_cs<TG, V>(source(ent[i + u]));
#pragma unroll
                for (uint32_t u = 0; u < kUnroll; ++u) ring->slot[u][threadIdx.x] = g[u];
                for (uint32_t u = 0; u < kUnroll && i + u < e1; ++u) consume(i + u, u);
            }
        }
        __syncthreads();  // the ring is free
        float* sm_head = reinterpret_cast<float*>(ring);
        float* sm_tail = sm_head + kThreads * V;
        bool is_tail = false;
        if (open) {
            const bool goes_on = row_of(ent[e1]) == cur;
            if (!begun) {
#pragma unroll
                for (int k = 0; k < V; ++k) kept[k] = acc[k];
                if (goes_on) flags |= kThrough;
            } else if (goes_on) {
                is_tail = true;
                flags |= kTail;
            } else {
                write_row();
            }
        }
#pragma unroll
        for (int k = 0; k < V; ++k) {
            if (flags & kHead) sm_head[threadIdx.x * V + k] = kept[k];
            if (is_tail) sm_tail[threadIdx.x * V + k] = acc[k];
        }
        if (lane == 0) sm_flags[team] = (uint8_t)flags;
        __syncthreads();
        // runs that cross teams: the team where a run begins adds the others' parts
        const uint32_t used = min(sh.teams, (count + per - 1) / per);
        auto add_heads = [&](uint32_t u) {  // from team u on; true where the run ends before `used`
            for (; u < used; ++u) {
#pragma unroll
                for (int k = 0; k < V; ++k) acc[k] += sm_head[(u * sh.lanes + lane) * V + k];
                if (!(sm_flags[u] & kThrough)) return true;
            }
            return false;
        };
        auto to_global = [&](float* out) {
            if (!on || !out) return;
#pragma unroll
            for (int k = 0; k < V; ++k) out[col + k] = acc[k];
        };
        uint32_t left = 0;
        if (is_tail) {
            if (add_heads(team + 1)) {
                write_row();
            } else {
                to_global(tail);
                if (lane == 0 && blockIdx.y == 0 && border) border->row = cur;
                left |= kTail;
            }
        }
        if (team == 0 && (flags & kHead)) {
            clear();
            left |= kHead | (add_heads(0) ? 0u : kThrough);
            to_global(head);
        }
        if (border) {
            __shared__ uint32_t sm_left;
            if (threadIdx.x == 0) sm_left = 0;
            __syncthreads();
            if (left && lane == 0) atomicOr(&sm_left, left);
            __syncthreads();
            if (threadIdx.x == 0 && blockIdx.y == 0) border->flags = sm_left;
        }
    }
};

// The table's gradient as bytes, for rows that become zero: `step` is the
// widest store (16, 8, 4 or 2 bytes) that rows and stride are multiples of.
struct ZeroRows {
    char* base;
    uint64_t stride;
    uint32_t bytes, step;
};

template <typename W>
__device__ __forceinline__ void zero_rows_by(const uint8_t* touched, uint32_t r0, uint32_t r1, const ZeroRows& z) {
    // the range's words in order, whatever a row's length: neighbouring threads, neighbouring words
    const uint32_t words = z.bytes / (uint32_t)sizeof(W), rows_on = blockDim.x / words;
    const uint32_t on = blockDim.x - rows_on * words;
    uint32_t r = threadIdx.x / words, c = threadIdx.x - r * words;
    char* at = z.base + (uint64_t)r0 * z.stride;
#pragma unroll 4
    while (r < r1 - r0) {
        if (!touched[r]) __stcs(reinterpret_cast<W*>(at + r * z.stride) + c, W{});
        r += rows_on;
        c += on;
        if (c >= words) {
            c -= words;
            ++r;
        }
    }
}

// Rows [r0, r1) whose flag is 0, by the whole CTA.
__device__ __forceinline__ void zero_rows(const uint8_t* touched, uint32_t r0, uint32_t r1, const ZeroRows& z) {
    if (z.step == 16) zero_rows_by<uint4>(touched, r0, r1, z);
    else if (z.step == 8) zero_rows_by<uint2>(touched, r0, r1, z);
    else if (z.step == 4) zero_rows_by<uint32_t>(touched, r0, r1, z);
    else zero_rows_by<uint16_t>(touched, r0, r1, z);
}

ZeroRows rows_to_zero(const EmbeddingArgs& a) {
    const uint64_t es = type_bytes(a.table_type);
    ZeroRows z{static_cast<char*>(a.table), a.ldt * es, (uint32_t)(a.F * es), 16};
    while (((uintptr_t)z.base | z.stride | z.bytes) & (z.step - 1)) z.step >>= 1;
    return z;
}

// Words of the table's gradient that become zero beside a kernel of the sort,
// which leaves the memory idle: CTAs of its own, after the kernel's.
struct EarlyZero {
    uint4* at;
    uint64_t words;
    uint32_t ctas;
};

__device__ __forceinline__ void zero_words(const EarlyZero& z, uint32_t cta) {
    const uint64_t step = (uint64_t)z.ctas * blockDim.x;
#pragma unroll 4
    for (uint64_t i = (uint64_t)cta * blockDim.x + threadIdx.x; i < z.words; i += step)
        __stcs(z.at + i, make_uint4(0, 0, 0, 0));
}

// ------------------------------------------------------------ owner form --

// Indices of the owner form, at most: 1,000 spread ones take 7 us, in the sorted
// form 20; but 2,000 of one row are one CTA's work, 73 us, there 28.
constexpr uint32_t kOwnerMax = 1024;
constexpr uint32_t kOwnerRows = 8192;      // table rows of a CTA, at most
constexpr int kOwnerEach = kOwnerMax / kThreads;

template <typename TG, typename TT, int V>
__global__ void __launch_bounds__(kThreads) grad_owner_kernel(
    const TG* __restrict__ grad, uint32_t grad_stride, const void* __restrict__ idx, int idx_type, uint32_t n,
    int64_t padding, float scale, TT* __restrict__ dtable, uint64_t ldt, uint32_t num_rows, uint32_t rows,
    const TeamShape sh, const ZeroRows zero, uint32_t* __restrict__ bad) {
    extern __shared__ uint4 smem[];
    Ring<TG, V>* ring = reinterpret_cast<Ring<TG, V>*>(smem);
    Entry* entries = reinterpret_cast<Entry*>(ring + 1) + 1;  // one before, one after
    uint8_t* touched = reinterpret_cast<uint8_t*>(entries + kOwnerMax + 1);
    __shared__ uint32_t warp_hits[kThreads / 32];
    const uint32_t r0 = blockIdx.x * rows, r1 = min(r0 + rows, num_rows);
    for (uint32_t i = threadIdx.x; i < r1 - r0; i += kThreads) touched[i] = 0;
    // this thread's indices, in order of position
    Entry mine[kOwnerEach];
    uint32_t hits = 0;
#pragma unroll
    for (int k = 0; k < kOwnerEach; ++k) {
        const uint32_t i = threadIdx.x * kOwnerEach + k;
        mine[k] = ~0ull;
        if (i < n) {
            const int64_t id = load_index(idx, idx_type, i);
            const bool inside = id >= 0 && id < (int64_t)num_rows;
            if (!inside && !is_padding(id, padding) && bad && blockIdx.x == 0) atomicExch(bad, 1u);
            if (inside && id != padding && id >= (int64_t)r0 && id < (int64_t)r1) {
                mine[k] = (Entry)id << 32 | i;
                ++hits;
            }
        }
    }
    uint32_t before = hits;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t t = __shfl_up_sync(0xffffffffu, before, o);
        if ((threadIdx.x & 31) >= (uint32_t)o) before += t;
    }
    if ((threadIdx.x & 31) == 31) warp_hits[threadIdx.x >> 5] = before;
    __syncthreads();
    uint32_t total = 0, base = before - hits;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
        if (w < (int)(threadIdx.x >> 5)) base += warp_hits[w];
        total += warp_hits[w];
    }
    if (total) {  // the same for the whole CTA
#pragma unroll
        for (int k = 0; k < kOwnerEach; ++k)
            if (mine[k] != ~0ull) {
                entries[base++] = mine[k];
                touched[(uint32_t)(mine[k] >> 32) - r0] = 1;
            }
        uint32_t size = 1;  // bitonic sort of the power of two above `total`
        while (size < total) size <<= 1;
        for (uint32_t i = total + threadIdx.x; i < size; i += kThreads) entries[i] = ~0ull;
        __syncthreads();
        for (uint32_t k = 2; k <= size; k <<= 1)
            for (uint32_t j = k >> 1; j; j >>= 1) {
                for (uint32_t i = threadIdx.x; i < size; i += kThreads) {
                    const uint32_t p = i ^ j;
                    if (p > i) {
                        const Entry a = entries[i], b = entries[p];
                        if ((a > b) == ((i & k) == 0)) {
                            entries[i] = b;
                            entries[p] = a;
                        }
                    }
                }
                __syncthreads();
            }
        if (threadIdx.x == 0) entries[-1] = entries[total] = ~0ull;  // the padding of the sort is read no more
        __syncthreads();
        RunSums<TG, TT, V> sums{entries, total, (total + sh.teams - 1) / sh.teams, grad, grad_stride, scale,
                                dtable,  ldt,   num_rows, sh, ring};
        sums.run(nullptr, nullptr, nullptr);
    }
    // the CTAs of the other columns take their share of the rows
    const uint32_t share = (r1 - r0 + gridDim.y - 1) / gridDim.y;
    const uint32_t z0 = min(r0 + blockIdx.y * share, r1), z1 = min(z0 + share, r1);
    zero_rows(touched + (z0 - r0), z0, z1, zero);
}

template <typename TG, typename TT, int V>
void launch_owner(const EmbeddingArgs& a, cudaStream_t s) {
    const TeamShape sh = team_shape(a.F / V);
    const uint32_t num_rows = (uint32_t)a.num_rows;
    // four CTAs per SM, of at most 64 rows each or else sixteen per SM
    const uint32_t rows =
        std::min(kOwnerRows, std::max(ceil_div(num_rows, 148 * 16), std::min(64u, ceil_div(num_rows, 148 * 4))));
    const dim3 grid(ceil_div(num_rows, rows), sh.blocks);
    const size_t smem = sizeof(Ring<TG, V>) + (kOwnerMax + 2) * sizeof(Entry) + (rows + 15) / 16 * 16;
    static std::atomic<uint64_t> done{0};
    allow_smem(grad_owner_kernel<TG, TT, V>, sizeof(Ring<TG, V>) + (kOwnerMax + 2) * sizeof(Entry) + kOwnerRows, done);
    grad_owner_kernel<TG, TT, V><<<grid, kThreads, smem, s>>>(
        static_cast<const TG*>(a.rows), (uint32_t)(a.ldr * sizeof(TG)), a.idx, a.idx_type, (uint32_t)a.n,
        a.padding, a.scale, static_cast<TT*>(a.table), a.ldt, num_rows, rows, sh, rows_to_zero(a), a.bad);
    TCC_CUDA(cudaGetLastError());
}

// ----------------------------------------------------------- sorted form --
//
// LSD radix sort of the entries by row, at most 11 bits a pass (two passes up to
// 4 M rows), three kernels a pass: digit counts per tile, offsets, scatter.  No
// CTA waits for another.

constexpr int kSortThreads = 512;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kTileEach = 8;
constexpr uint32_t kTile = kSortThreads * kTileEach;  // entries of a tile
constexpr int kMinDigitBits = 8, kMaxDigitBits = 11;
constexpr uint32_t kMaxDigits = 1u << kMaxDigitBits;

struct IndexSource {  // pass 0: the indices themselves; rows without a gradient sort last
    static constexpr bool kGiven = true;  // before the call's first kernel
    const void* idx;
    int type;
    int64_t padding;
    uint32_t num_rows;
    uint32_t* bad;
    __device__ __forceinline__ Entry load(uint32_t i) const {
        const int64_t id = load_index(idx, type, i);
        const bool real = id >= 0 && id < (int64_t)num_rows && id != padding;
        return (Entry)(real ? (uint32_t)id : num_rows) << 32 | i;
    }
    __device__ __forceinline__ void note(uint32_t i, Entry e) const {
        if (bad && row_of(e) == num_rows && !is_padding(load_index(idx, type, i), padding)) atomicExch(bad, 1u);
    }
};

struct EntrySource {
    static constexpr bool kGiven = false;
    const Entry* entries;
    __device__ __forceinline__ Entry load(uint32_t i) const { return entries[i]; }
    __device__ __forceinline__ void note(uint32_t, Entry) const {}
};

// counts [tile][digit], totals [digit] (zero before).
template <typename Source>
__global__ void __launch_bounds__(kSortThreads) digit_counts_kernel(const Source src, uint32_t n, int shift,
                                                                    uint32_t digits, uint32_t* __restrict__ counts,
                                                                    uint32_t* __restrict__ totals) {
    after_previous();
    __shared__ uint32_t hist[kMaxDigits];
    for (uint32_t d = threadIdx.x; d < digits; d += kSortThreads) hist[d] = 0;
    const uint32_t base = blockIdx.x * kTile + threadIdx.x;
    Entry e[kTileEach];
#pragma unroll
    for (int k = 0; k < kTileEach; ++k)
        if (base + k * kSortThreads < n) e[k] = src.load(base + k * kSortThreads);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kTileEach; ++k)
        if (base + k * kSortThreads < n) {
            atomicAdd(&hist[(row_of(e[k]) >> shift) & (digits - 1)], 1u);
            src.note(base + k * kSortThreads, e[k]);
        }
    __syncthreads();
    for (uint32_t d = threadIdx.x; d < digits; d += kSortThreads) {
        counts[(uint64_t)blockIdx.x * digits + d] = hist[d];
        if (hist[d]) atomicAdd(&totals[d], hist[d]);
    }
}

// counts -> where a tile's first entry of each digit goes.  A CTA takes 32
// digits; 32 rows of threads share the tiles.
__global__ void __launch_bounds__(1024) digit_offsets_kernel(uint32_t* counts, uint32_t tiles, uint32_t digits,
                                                             const uint32_t* totals) {
    after_previous();
    __shared__ uint32_t part[32][33];
    __shared__ uint32_t below[32];
    const uint32_t lane = threadIdx.x & 31, row = threadIdx.x >> 5;
    const uint32_t d0 = blockIdx.x * 32, d = d0 + lane;
    uint32_t s = 0;
    for (uint32_t i = threadIdx.x; i < d0; i += 1024) s += totals[i];
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) below[row] = s;
    const uint32_t per = (tiles + 31) / 32, t0 = min(row * per, tiles), t1 = min(t0 + per, tiles);
    uint32_t sum = 0;
    if (d < digits) {
#pragma unroll 8
        for (uint32_t t = t0; t < t1; ++t) sum += counts[(uint64_t)t * digits + d];
    }
    part[row][lane] = sum;
    __syncthreads();
    if (row == 0) {
        uint32_t base = below[lane];  // the totals of the digits before d0
        for (int o = 16; o; o >>= 1) base += __shfl_xor_sync(0xffffffffu, base, o);
        const uint32_t mine = d < digits ? totals[d] : 0;
        uint32_t inc = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t t = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= (uint32_t)o) inc += t;
        }
        uint32_t run = base + inc - mine;
        for (int r = 0; r < 32; ++r) {
            const uint32_t c = part[r][lane];
            part[r][lane] = run;
            run += c;
        }
    }
    __syncthreads();
    if (d < digits) {
        uint32_t run = part[row][lane];
#pragma unroll 8
        for (uint32_t t = t0; t < t1; ++t) {
            const uint64_t at = (uint64_t)t * digits + d;
            const uint32_t c = counts[at];
            counts[at] = run;
            run += c;
        }
    }
}

// Lanes of the warp with the same digit: a vote for each of its bits (the
// warp's own match instruction took 17 us in place of 15 for a pass over 1 M).
template <int BITS>
__device__ __forceinline__ unsigned same_digit(uint32_t d, bool in) {
    unsigned same = __ballot_sync(0xffffffffu, in);
#pragma unroll
    for (int bit = 0; bit < BITS; ++bit) {
        const unsigned set = __ballot_sync(0xffffffffu, d >> bit & 1u);
        same &= d >> bit & 1u ? set : ~set;
    }
    return same;
}

// Stable: warp w ranks the tile's entries [w * 256, (w + 1) * 256) against its
// own digit counts; a prefix over the warps puts them in order.
template <typename Source, int BITS>
__global__ void __launch_bounds__(kSortThreads) digit_scatter_kernel(const Source src, uint32_t n, int shift,
                                                                     const uint32_t* offsets, Entry* out) {
    if constexpr (!Source::kGiven) after_previous();
    constexpr uint32_t digits = 1u << BITS;
    extern __shared__ uint4 smem[];
    uint16_t* all = reinterpret_cast<uint16_t*>(smem);  // [kSortWarps][digits]
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint16_t* cnt = all + warp * digits;
    const uint32_t base = blockIdx.x * kTile + warp * (kTile / kSortWarps) + lane;
    Entry e[kTileEach];
    uint32_t place[kTileEach];  // digit, and the rank among the warp's entries of that digit
#pragma unroll
    for (int k = 0; k < kTileEach; ++k) {
        const uint32_t i = base + k * 32;
        e[k] = i < n ? src.load(i) : ~0ull;
    }
    for (uint32_t i = threadIdx.x; i < kSortWarps * digits / 8; i += kSortThreads) smem[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kTileEach; ++k) {
        const bool in = base + k * 32 < n;
        const uint32_t d = in ? (row_of(e[k]) >> shift) & (digits - 1) : kMaxDigits;
        const unsigned peers = same_digit<BITS>(d, in);
        const uint32_t rank = __popc(peers & lanemask_lt());
        const uint32_t seen = in ? cnt[d] : 0;
        __syncwarp();
        if (in && rank == 0) cnt[d] = (uint16_t)(seen + __popc(peers));
        __syncwarp();
        place[k] = d << 16 | (seen + rank);
    }
    __syncthreads();
    // two digits at a time, one in each half of a word (a tile has 2^12 entries)
    for (uint32_t d = threadIdx.x; d < digits / 2; d += kSortThreads) {
        uint32_t* col = reinterpret_cast<uint32_t*>(all) + d;
        uint32_t run = 0;
#pragma unroll
        for (int w = 0; w < kSortWarps; ++w) {
            const uint32_t c = col[w * (digits / 2)];
            col[w * (digits / 2)] = run;
            run += c;
        }
    }
    if constexpr (Source::kGiven) after_previous();  // the ranks took the indices alone
    const uint32_t* offset = offsets + (uint64_t)blockIdx.x * digits;
    uint32_t start[kTileEach];
#pragma unroll
    for (int k = 0; k < kTileEach; ++k) start[k] = base + k * 32 < n ? offset[place[k] >> 16] : 0;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kTileEach; ++k)
        if (base + k * 32 < n) out[start[k] + cnt[place[k] >> 16] + (place[k] & 0xFFFFu)] = e[k];
}

// The whole sort by one cluster of CTAs for up to kClusterMax entries: each CTA
// holds `each` of them, ranks them by digit, and writes them to their places in
// the CTAs' shared memory.  One launch in place of seven: the gradient of 8,193
// indices in a table of 10,000 x 64 takes 26 us in place of 38, of 40,000 40
// in place of 44, of 65,536 52 in place of 44: the sort is then bound by what
// eight SMs can do.  From about 100 MB of table on it wins up to 65,536 all the
// same, by what the other SMs zero meanwhile (1 M x 128: 136 in place of 140).
constexpr uint32_t kCluster = 8;
constexpr int kHeldEach = 16;  // entries of a thread
constexpr uint32_t kHeld = kSortThreads * kHeldEach;
constexpr uint32_t kClusterMax = kCluster * kHeld, kClusterSmall = 40960;
constexpr uint64_t kClusterTable = 100000000;

bool by_cluster(const EmbeddingArgs& a) {
    return a.n <= kClusterSmall ||
           (a.n <= kClusterMax && a.num_rows * a.F * type_bytes(a.table_type) >= kClusterTable);
}

size_t cluster_smem(uint32_t each, uint32_t digits) {
    return 2 * (size_t)each * sizeof(Entry) + (size_t)kSortWarps * digits * 2 + (size_t)digits * 12;
}

template <int BITS>
__global__ void __launch_bounds__(kSortThreads) cluster_sort_kernel(const IndexSource src, uint32_t n, uint32_t each,
                                                                    int passes, Entry* __restrict__ out,
                                                                    const EarlyZero zero) {
    after_previous();
    if (blockIdx.x >= kCluster) return zero_words(zero, blockIdx.x - kCluster);  // whole clusters
    extern __shared__ uint4 smem[];
    __shared__ uint32_t warp_sums[kSortWarps];
    cg::cluster_group cluster = cg::this_cluster();
    constexpr uint32_t digits = 1u << BITS;
    const uint32_t rank_cta = cluster.block_rank();
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    Entry* held = reinterpret_cast<Entry*>(smem);  // [2][each]
    uint16_t* all = reinterpret_cast<uint16_t*>(held + 2 * each);             // [kSortWarps][digits]
    uint32_t* hist = reinterpret_cast<uint32_t*>(all + kSortWarps * digits);  // [digits]: of this CTA
    uint32_t* total = hist + digits;  // [digits]: of the cluster
    uint32_t* start = total + digits;  // [digits]: where this CTA's first entry of a digit goes
    uint16_t* cnt = all + warp * digits;
    const uint32_t first = min(rank_cta * each, n), count = min(each, n - first);
    // a warp ranks `steps` times 32 neighbouring entries
    const uint32_t steps = (each + kSortThreads - 1) / kSortThreads, base = warp * steps * 32 + lane;
    Entry e[kHeldEach];
#pragma unroll
    for (int k = 0; k < kHeldEach; ++k) {
        const uint32_t i = base + k * 32;
        e[k] = ~0ull;
        if (k < (int)steps && i < count) {
            e[k] = src.load(first + i);
            src.note(first + i, e[k]);
        }
    }
#pragma unroll 1
    for (int pass = 0; pass < passes; ++pass) {
        const int shift = pass * BITS;
        for (uint32_t i = threadIdx.x; i < kSortWarps * digits / 8; i += kSortThreads)
            reinterpret_cast<uint4*>(all)[i] = make_uint4(0, 0, 0, 0);
        __syncthreads();
        uint32_t place[kHeldEach];
#pragma unroll
        for (int k = 0; k < kHeldEach; ++k) {
            if (k >= (int)steps) break;
            const bool in = base + k * 32 < count;
            const uint32_t d = in ? (row_of(e[k]) >> shift) & (digits - 1) : kMaxDigits;
            const unsigned peers = same_digit<BITS>(d, in);
            const uint32_t rank = __popc(peers & lanemask_lt());
            const uint32_t seen = in ? cnt[d] : 0;
            __syncwarp();
            if (in && rank == 0) cnt[d] = (uint16_t)(seen + __popc(peers));
            __syncwarp();
            place[k] = d << 16 | (seen + rank);
        }
        __syncthreads();
        for (uint32_t d = threadIdx.x; d < digits / 2; d += kSortThreads) {
            uint32_t* col = reinterpret_cast<uint32_t*>(all) + d;
            uint32_t run = 0;
#pragma unroll
            for (int w = 0; w < kSortWarps; ++w) {
                const uint32_t c = col[w * (digits / 2)];
                col[w * (digits / 2)] = run;
                run += c;
            }
            hist[2 * d] = run & 0xFFFFu;
            hist[2 * d + 1] = run >> 16;
        }
        cluster.sync();  // every CTA's counts are there
        for (uint32_t d = threadIdx.x; d < digits; d += kSortThreads) {
            uint32_t c[kCluster], before = 0, sum = 0;
#pragma unroll
            for (uint32_t r = 0; r < kCluster; ++r) c[r] = *cluster.map_shared_rank(hist + d, r);
#pragma unroll
            for (uint32_t r = 0; r < kCluster; ++r) {
                if (r < rank_cta) before += c[r];
                sum += c[r];
            }
            total[d] = sum;
            start[d] = before;
        }
        __syncthreads();
        // exclusive sums of the totals: a thread takes neighbouring digits
        const uint32_t per = (digits + kSortThreads - 1) / kSortThreads, d0 = threadIdx.x * per;
        uint32_t mine = 0;
        for (uint32_t i = 0; i < per && d0 + i < digits; ++i) mine += total[d0 + i];
        uint32_t inc = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t t = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= (uint32_t)o) inc += t;
        }
        if (lane == 31) warp_sums[warp] = inc;
        __syncthreads();
        uint32_t below = inc - mine;
        for (uint32_t w = 0; w < warp; ++w) below += warp_sums[w];
        for (uint32_t i = 0; i < per && d0 + i < digits; ++i) {
            start[d0 + i] += below;
            below += total[d0 + i];
        }
        __syncthreads();
        if (pass + 1 == passes) {
#pragma unroll
            for (int k = 0; k < kHeldEach; ++k)
                if (k < (int)steps && base + k * 32 < count) {
                    const uint32_t d = place[k] >> 16;
                    out[start[d] + cnt[d] + (place[k] & 0xFFFFu)] = e[k];
                }
            break;
        }
        Entry* next = held + (pass & 1) * each;
#pragma unroll
        for (int k = 0; k < kHeldEach; ++k)
            if (k < (int)steps && base + k * 32 < count) {
                const uint32_t d = place[k] >> 16, to = start[d] + cnt[d] + (place[k] & 0xFFFFu);
                const uint32_t cta = to / each;
                *cluster.map_shared_rank(next + (to - cta * each), cta) = e[k];
            }
        cluster.sync();  // every entry is in its place, and nobody reads the counts any more
#pragma unroll
        for (int k = 0; k < kHeldEach; ++k)
            if (k < (int)steps && base + k * 32 < count) e[k] = next[base + k * 32];
    }
    cluster.sync();  // no CTA's counts go while another reads them
}

// The rows of a table range that have no entry become zero; the range's
// entries are found by search, and rows looked up in them one by one where
// they are too many to walk (a hub's).
constexpr uint32_t kFillRows = 1024;  // at most
constexpr uint32_t kFillWalk = 16384;

__device__ __forceinline__ uint32_t first_of(const Entry* entries, uint32_t lo, uint32_t hi, uint32_t row) {
    while (lo < hi) {
        const uint32_t mid = lo + (hi - lo) / 2;
        if (row_of(entries[mid]) < row) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}

__device__ __forceinline__ void fill_range(const Entry* entries, uint32_t n, uint32_t r0, uint32_t r1,
                                           const ZeroRows& zero, uint8_t* touched, uint32_t* bounds) {
    if (threadIdx.x < 2) bounds[threadIdx.x] = first_of(entries, 0, n, threadIdx.x ? r1 : r0);
    for (uint32_t i = threadIdx.x; i < r1 - r0; i += kThreads) touched[i] = 0;
    __syncthreads();
    const uint32_t lo = bounds[0], hi = bounds[1];
    if (hi - lo <= kFillWalk) {
#pragma unroll 4
        for (uint32_t i = lo + threadIdx.x; i < hi; i += kThreads) touched[row_of(entries[i]) - r0] = 1;
    } else {
        for (uint32_t r = r0 + threadIdx.x; r < r1; r += kThreads) {
            const uint32_t at = first_of(entries, lo, hi, r);
            touched[r - r0] = at < hi && row_of(entries[at]) == r;
        }
    }
    __syncthreads();
    zero_rows(touched, r0, r1, zero);
}

// CTAs [0, fills) of the grid's x fill; of the others i takes range i of the entries.
struct SortedShape {
    uint32_t per, range, sums;  // entries of a team, of a CTA; CTAs
    uint32_t fill_rows, fills;  // table rows of a CTA that fills; CTAs
    uint32_t zeroed;            // rows that are zero already
};

template <typename TG, typename TT, int V>
__global__ void __launch_bounds__(kThreads) grad_sorted_kernel(
    const TG* __restrict__ grad, uint32_t grad_stride, const Entry* entries, uint32_t n, float scale, TT* dtable,
    uint64_t ldt, uint32_t num_rows, const TeamShape sh, const SortedShape so, const ZeroRows zero, float* heads,
    float* tails, Border* borders) {
    after_previous();
    extern __shared__ uint4 smem[];
    if (blockIdx.x < so.fills) {
        __shared__ uint32_t bounds[2];
        static_assert(kFillRows <= sizeof(Ring<TG, V>), "flags fit");
        // the CTAs of the other columns take their share of the rows
        const uint32_t share = (so.fill_rows + gridDim.y - 1) / gridDim.y;
        const uint32_t f0 = so.zeroed + blockIdx.x * so.fill_rows;
        const uint32_t r0 = f0 + min(blockIdx.y * share, so.fill_rows);
        const uint32_t r1 = min(min(r0 + share, f0 + so.fill_rows), num_rows);
        if (r0 < r1) fill_range(entries, n, r0, r1, zero, reinterpret_cast<uint8_t*>(smem), bounds);
        return;
    }
    const uint32_t i = blockIdx.x - so.fills, width = sh.packs * V;
    const uint32_t lo = i * so.range, count = min(so.range, n - lo);
    Ring<TG, V>* ring = reinterpret_cast<Ring<TG, V>*>(smem);
    Entry* ent = reinterpret_cast<Entry*>(ring + 1);  // the entry before, the range, the entry after
    for (uint32_t k = threadIdx.x; k < count + 2; k += kThreads)
        ent[k] = lo + k > 0 && lo + k <= n ? entries[lo + k - 1] : ~0ull;
    __syncthreads();
    RunSums<TG, TT, V> sums{ent + 1, count, so.per, grad, grad_stride, scale, dtable, ldt, num_rows, sh, ring};
    sums.run(heads + (uint64_t)i * width, tails + (uint64_t)i * width, borders + i);
}

// A block per range: where a run begins in it and goes on, its parts are added.
// The threads are columns (of W floats) times groups; a group adds a contiguous
// part of the ranges, and the groups' sums are added in order, in 64 bits: a hub's
// run has as many parts as its rows allow, and a wide row one group.
template <typename TT, int W>
__global__ void __launch_bounds__(kThreads) grad_join_kernel(const Border* borders, uint32_t sums, const float* heads,
                                                             const float* tails, uint32_t width, float scale,
                                                             TT* dtable, uint64_t ldt, uint32_t num_rows) {
    after_previous();
    const Border b = borders[blockIdx.x];
    if (!(b.flags & kTail) || b.row >= num_rows) return;
    // the ranges after it that hold a part: up to the first that is not passed through
    __shared__ uint32_t last;
    __shared__ double part[W][kThreads];
    const uint32_t begin = blockIdx.x + 1;
    if (threadIdx.x == 0) last = sums;
    for (uint32_t from = begin;; from += kThreads) {
        const uint32_t i = from + threadIdx.x;
        const bool ends = i >= sums || !(borders[i].flags & kThrough);
        __syncthreads();
        if (ends) atomicMin(&last, min(i, sums - 1));
        __syncthreads();
        if (last < sums) break;
    }
    const uint32_t cols = width / W, parts = last + 1 - begin;
    uint32_t across = 1;  // columns side by side
    while (across < kThreads && across < cols) across <<= 1;
    const uint32_t groups = kThreads / across, group = threadIdx.x / across;
    const uint32_t each = (parts + groups - 1) / groups;
    const uint32_t p0 = begin + min(group * each, parts), p1 = begin + min((group + 1) * each, parts);
    for (uint32_t c0 = 0; c0 < cols; c0 += across) {
        const uint32_t c = c0 + threadIdx.x % across;
        double acc[W];
#pragma unroll
        for (int k = 0; k < W; ++k) acc[k] = 0.0;
        if (c < cols) {
            if (group == 0) {
                const Pack<float, W> t = load_pack<float, W>(tails + (uint64_t)blockIdx.x * width + c * W);
#pragma unroll
                for (int k = 0; k < W; ++k) acc[k] = (double)t.v[k];
            }
#pragma unroll 4
            for (uint32_t i = p0; i < p1; ++i) {
                const Pack<float, W> h = load_pack<float, W>(heads + (uint64_t)i * width + c * W);
#pragma unroll
                for (int k = 0; k < W; ++k) acc[k] += (double)h.v[k];
            }
        }
#pragma unroll
        for (int k = 0; k < W; ++k) part[k][threadIdx.x] = acc[k];
        __syncthreads();
        if (group == 0 && c < cols) {
            for (uint32_t g = 1; g < groups && g * each < parts; ++g)
#pragma unroll
                for (int k = 0; k < W; ++k) acc[k] += part[k][g * across + threadIdx.x];
#pragma unroll
            for (int k = 0; k < W; ++k)
                dtable[(uint64_t)b.row * ldt + c * W + k] = from_f32<TT>((float)(acc[k] * (double)scale));
        }
        __syncthreads();
    }
}

uint64_t align256(uint64_t b) { return (b + 255) / 256 * 256; }

struct SortPlan {
    int passes, bits;  // digit bits of a pass
    uint32_t tiles, digits;
};

SortPlan sort_plan(uint64_t n, uint64_t num_rows) {
    SortPlan p;
    const int total = std::max(1, bits_for(num_rows + 1));
    p.passes = (total + kMaxDigitBits - 1) / kMaxDigitBits;
    p.bits = std::max(kMinDigitBits, (total + p.passes - 1) / p.passes);
    p.digits = 1u << p.bits;
    p.tiles = ceil_div(n, kTile);
    return p;
}

// Entries of a team: about 16 CTAs per SM over the whole list (ranges long
// enough that few runs cross), at least 16; of a CTA at most 1024.
constexpr uint32_t kRangeMax = 1024;
SortedShape sorted_shape(uint64_t n, uint64_t num_rows, const TeamShape& sh, uint64_t zeroed = 0) {
    SortedShape so;
    const uint64_t per = (n / (148 * 16) + sh.teams - 1) / sh.teams;
    so.per = (uint32_t)std::min<uint64_t>(kRangeMax / sh.teams, std::max<uint64_t>(16, per));
    so.range = so.per * sh.teams;
    so.sums = ceil_div(n, so.range);
    // about four such CTAs per SM, so that a small table's rows are spread too
    so.fill_rows = (uint32_t)std::min<uint64_t>(kFillRows, std::max<uint64_t>(16, num_rows / (148 * 4)));
    so.fills = ceil_div(num_rows - zeroed, so.fill_rows);
    so.zeroed = (uint32_t)zeroed;
    return so;
}

// Ranges of any vector width.
uint64_t max_sums(uint64_t n, uint64_t num_rows, uint32_t F) {
    uint64_t most = 1;
    for (uint32_t width = 1; width <= 8 && F % width == 0; width <<= 1)
        most = std::max<uint64_t>(most, sorted_shape(n, num_rows, team_shape(F / width)).sums);
    return most;
}

struct GradScratch {
    Entry *a, *b;
    uint32_t* counts;
    uint32_t* totals;  // [passes][digits], zero before
    float *heads, *tails;
    Border* borders;
    size_t total_bytes, bytes;
};

GradScratch lay_out(uint64_t n, uint64_t num_rows, uint32_t F, char* base) {
    GradScratch g;
    const SortPlan p = sort_plan(n, num_rows);
    const uint64_t sums = max_sums(n, num_rows, F);
    uint64_t at = 0;
    auto take = [&](uint64_t bytes) {
        char* q = base + at;
        at += align256(bytes);
        return q;
    };
    g.a = reinterpret_cast<Entry*>(take(n * 8));
    g.b = reinterpret_cast<Entry*>(take(n * 8));
    g.counts = reinterpret_cast<uint32_t*>(take((uint64_t)p.tiles * p.digits * 4));
    g.total_bytes = (size_t)p.passes * p.digits * 4;
    g.totals = reinterpret_cast<uint32_t*>(take(g.total_bytes));
    g.heads = reinterpret_cast<float*>(take(sums * F * 4));
    g.tails = reinterpret_cast<float*>(take(sums * F * 4));
    g.borders = reinterpret_cast<Border*>(take(sums * sizeof(Border)));
    g.bytes = at;
    return g;
}

// Rows that become zero beside the cluster's sort, which leaves most SMs idle:
// about what is written in its time (more delays the sums: all 537 MB of 1 M x 128
// first took 167 us for 65,536 indices, none 161, these 136; for 2,049 157, 132
// and 107).  Beside the tiles' kernels the stores slow the sort by more than they
// save (1 M indices: 277 to 300 us in place of 261).
uint64_t early_rows(const EmbeddingArgs& a) {
    if (!by_cluster(a) || a.ldt != a.F || (uintptr_t)a.table % 16) return 0;
    const uint64_t most = 80000000 + 2000 * a.n;
    return std::min<uint64_t>(a.num_rows, most / (a.F * type_bytes(a.table_type))) & ~7ull;  // of whole words
}

template <int BITS>
const Entry* sort_by_cluster(const IndexSource& src, uint32_t n, const SortPlan& p, const GradScratch& g,
                             EarlyZero zero, cudaStream_t s) {
    const uint32_t each = (n + kCluster - 1) / kCluster;
    static std::atomic<uint64_t> done{0};
    allow_smem(cluster_sort_kernel<BITS>, cluster_smem(kHeld, p.digits), done);
    cudaLaunchConfig_t cfg{};
    // 264 CTAs, and only as many as find work.  They carry the sort's shared memory: two to an
    // SM up to about 12,000 indices with 11-bit digits, above that one, in two turns.
    zero.ctas = (uint32_t)std::min<uint64_t>(33, (zero.words + 8191) / 8192) * kCluster;
    cfg.gridDim = dim3(kCluster + zero.ctas);
    cfg.blockDim = dim3(kSortThreads);
    cfg.dynamicSmemBytes = cluster_smem(each, p.digits);
    cfg.stream = s;
    cudaLaunchAttribute cluster{};
    cluster.id = cudaLaunchAttributeClusterDimension;
    cluster.val.clusterDim.x = kCluster;
    cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
    cfg.attrs = &cluster;
    cfg.numAttrs = 1;
    TCC_CUDA(cudaLaunchKernelEx(&cfg, cluster_sort_kernel<BITS>, src, n, each, p.passes, g.a, zero));
    return g.a;
}

template <int BITS>
const Entry* sort_by_tiles(const IndexSource& src, uint32_t n, const SortPlan& p, const GradScratch& g,
                           cudaStream_t s) {
    TCC_CUDA(cudaMemsetAsync(g.totals, 0, g.total_bytes, s));
    const size_t smem = (size_t)kSortWarps * p.digits * sizeof(uint16_t);
    static std::atomic<uint64_t> first_done{0}, next_done{0};
    allow_smem(digit_scatter_kernel<IndexSource, BITS>, smem, first_done);
    allow_smem(digit_scatter_kernel<EntrySource, BITS>, smem, next_done);
    Entry* in = g.b;
    Entry* out = g.a;
    for (int pass = 0; pass < p.passes; ++pass) {
        const int shift = pass * BITS;
        uint32_t* totals = g.totals + (size_t)pass * p.digits;
        const EntrySource from_entries{in};
        if (pass == 0)
            digit_counts_kernel<<<p.tiles, kSortThreads, 0, s>>>(src, n, shift, p.digits, g.counts, totals);
        else
            launch_after(digit_counts_kernel<EntrySource>, p.tiles, kSortThreads, 0, s, from_entries, n, shift,
                         p.digits, g.counts, totals);
        launch_after(digit_offsets_kernel, ceil_div(p.digits, 32), 1024, 0, s, g.counts, p.tiles, p.digits, totals);
        if (pass == 0)
            launch_after(digit_scatter_kernel<IndexSource, BITS>, p.tiles, kSortThreads, smem, s, src, n, shift,
                         g.counts, out);
        else
            launch_after(digit_scatter_kernel<EntrySource, BITS>, p.tiles, kSortThreads, smem, s, from_entries, n,
                         shift, g.counts, out);
        std::swap(in, out);
    }
    TCC_CUDA(cudaGetLastError());
    return in;
}

template <int BITS>
const Entry* sort_entries(const IndexSource& src, uint32_t n, const SortPlan& p, const GradScratch& g,
                          bool cluster, const EarlyZero& zero, cudaStream_t s) {
    return cluster ? sort_by_cluster<BITS>(src, n, p, g, zero, s) : sort_by_tiles<BITS>(src, n, p, g, s);
}

template <typename TG, typename TT, int V>
void launch_sorted(const EmbeddingArgs& a, char* scratch, cudaStream_t s) {
    const uint32_t n = (uint32_t)a.n, num_rows = (uint32_t)a.num_rows;
    const GradScratch g = lay_out(n, num_rows, a.F, scratch);
    const SortPlan p = sort_plan(n, num_rows);
    const TeamShape sh = team_shape(a.F / V);
    const uint64_t early = early_rows(a), row = a.F * type_bytes(a.table_type);
    const EarlyZero zero{static_cast<uint4*>(a.table), early * row / 16, 0};
    const SortedShape so = sorted_shape(n, num_rows, sh, early);
    const IndexSource from_idx{a.idx, a.idx_type, a.padding, num_rows, a.bad};
    const bool cluster = by_cluster(a);
    const Entry* in = p.bits == 8    ? sort_entries<8>(from_idx, n, p, g, cluster, zero, s)
                      : p.bits == 9  ? sort_entries<9>(from_idx, n, p, g, cluster, zero, s)
                      : p.bits == 10 ? sort_entries<10>(from_idx, n, p, g, cluster, zero, s)
                                     : sort_entries<11>(from_idx, n, p, g, cluster, zero, s);
    static std::atomic<uint64_t> sums_done{0};
    const size_t sum_smem = sizeof(Ring<TG, V>) + (so.range + 2) * sizeof(Entry);
    allow_smem(grad_sorted_kernel<TG, TT, V>, sizeof(Ring<TG, V>) + (kRangeMax + 2) * sizeof(Entry), sums_done);
    launch_after(grad_sorted_kernel<TG, TT, V>, dim3(so.fills + so.sums, sh.blocks), kThreads, sum_smem, s,
                 static_cast<const TG*>(a.rows), (uint32_t)(a.ldr * sizeof(TG)), in, n, a.scale,
                 static_cast<TT*>(a.table), a.ldt, num_rows, sh, so, rows_to_zero(a), g.heads, g.tails, g.borders);
    if (so.sums > 1) {
        auto join = a.F % 4 ? grad_join_kernel<TT, 1> : grad_join_kernel<TT, 4>;
        launch_after(join, so.sums, kThreads, 0, s, g.borders, so.sums, g.heads, g.tails, a.F, a.scale,
                     static_cast<TT*>(a.table), a.ldt, num_rows);
    }
    TCC_CUDA(cudaGetLastError());
}

bool owner_form(uint64_t n) { return n <= kOwnerMax; }

template <typename TG, typename TT, int V>
void launch_grad(const EmbeddingArgs& a, char* scratch, cudaStream_t s) {
    if (owner_form(a.n)) launch_owner<TG, TT, V>(a, s);
    else launch_sorted<TG, TT, V>(a, scratch, s);
}

template <typename TG, typename TT>
void grad_by_width(const EmbeddingArgs& a, char* scratch, cudaStream_t s) {
    VecRule rule;
    rule.count(a.F);
    rule.count(a.ldt);
    rule.count(a.ldr);
    rule.pointer(a.table, sizeof(TT));
    rule.pointer(a.rows, sizeof(TG));
    switch (team_width(rule.width(), a.F)) {
        case 8:
            if constexpr (sizeof(TT) == 2 && sizeof(TG) == 2) launch_grad<TG, TT, 8>(a, scratch, s);
            break;
        case 4: launch_grad<TG, TT, 4>(a, scratch, s); break;
        case 2: launch_grad<TG, TT, 2>(a, scratch, s); break;
        default: launch_grad<TG, TT, 1>(a, scratch, s);
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
    TCC_REQUIRE(a.ldr < (1ull << 30) && a.ldt < (1ull << 30), "row strides are too large");
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
    if (owner_form(n) || num_rows == 0) return 0;
    return lay_out(n, num_rows, F, nullptr).bytes;
}

void embedding_backward(const EmbeddingArgs& a, void* scratch, size_t scratch_bytes, cudaStream_t s) {
    check_embedding(a);
    if (a.num_rows == 0) return;
    const size_t need = embedding_backward_scratch_bytes(a.n, a.num_rows, a.F);
    if (need) {
        TCC_REQUIRE(scratch && (uintptr_t)scratch % 256 == 0, "scratch must be 256-byte aligned");
        if (scratch_bytes < need)
            throw Error(TCC_ERR_CAPACITY, "scratch is smaller than tcc_embedding_backward_scratch_bytes");
    }
    char* p = static_cast<char*>(scratch);
    with_types(a, [&](auto tt, auto tg) { grad_by_width<decltype(tg), decltype(tt)>(a, p, s); });
}

}  // namespace tcc
