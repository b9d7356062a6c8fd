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
constexpr int kUnroll = 8;  // gradient rows in flight per team
constexpr uint32_t kNoRow = 0xFFFFFFFFu;

using Entry = unsigned long long;  // row << 32 | position
__device__ __forceinline__ uint32_t row_of(Entry e) { return (uint32_t)(e >> 32); }

// Lanes of a team: one pack of a gradient row each (grid.y covers the rest).
struct TeamShape {
    uint32_t lanes, teams, packs, blocks;  // blocks: the grid's y
};

TeamShape team_shape(uint32_t packs) {
    TeamShape t;
    t.packs = packs;
    t.lanes = 1;
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

// Sums the runs of entries [lo, hi) of `entries`, team t the entries
// [lo + t * per, lo + (t + 1) * per).  Rows whose run lies inside are written;
// for the others head / tail (fp32, [F]) and *border are, where they are given
// (entries then go on outside [lo, hi) within [0, end)).  Entries of rows >=
// num_rows are passed over.
template <typename TG, typename TT, int V>
__device__ __forceinline__ void sum_runs(const Entry* entries, uint32_t lo, uint32_t hi, uint32_t end, uint32_t per,
                                         const TG* __restrict__ grad, uint64_t ldg, float scale,
                                         TT* __restrict__ dtable, uint64_t ldt, uint32_t num_rows,
                                         const TeamShape& sh, float* head, float* tail, Border* border) {
    __shared__ float sm_head[kThreads * V], sm_tail[kThreads * V];
    __shared__ uint8_t sm_flags[kThreads];
    const uint32_t team = threadIdx.x / sh.lanes, lane = threadIdx.x % sh.lanes;
    const uint32_t pack = blockIdx.y * sh.lanes + lane;
    const bool on = pack < sh.packs;
    const uint64_t col = (uint64_t)pack * V;
    const uint64_t first = (uint64_t)lo + (uint64_t)team * per;
    const uint32_t e0 = (uint32_t)min(first, (uint64_t)hi), e1 = (uint32_t)min(first + per, (uint64_t)hi);
    float acc[V];
    auto clear = [&] {
#pragma unroll
        for (int k = 0; k < V; ++k) acc[k] = 0.f;
    };
    auto write_row = [&](uint32_t row) {
        if (!on || row >= num_rows) return;
        Pack<TT, V> o;
#pragma unroll
        for (int k = 0; k < V; ++k) o.v[k] = from_f32<TT>(acc[k] * scale);
        store_pack_cs<TT, V>(dtable + (uint64_t)row * ldt + col, o);
    };
    auto to_shared = [&](float* s) {
#pragma unroll
        for (int k = 0; k < V; ++k) s[threadIdx.x * V + k] = acc[k];
    };
    clear();
    uint32_t flags = 0, cur = kNoRow;
    bool begun = true;  // the current run began in this team's range
    if (e0 < e1) {
        cur = row_of(entries[e0]);
        if (e0 > 0 && row_of(entries[e0 - 1]) == cur) {
            flags |= kHead;
            begun = false;
        }
        for (uint32_t j = e0; j < e1; j += kUnroll) {
            uint32_t row[kUnroll];
            Pack<TG, V> g[kUnroll];
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                const Entry e = j + u < e1 ? entries[j + u] : ~0ull;
                row[u] = row_of(e);
                if (on && row[u] < num_rows)
                    g[u] = load_pack_cs<TG, V>(grad + (uint64_t)(uint32_t)e * ldg + col);
            }
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                if (j + u >= e1) break;
                if (row[u] != cur) {
                    if (begun) write_row(cur);
                    else to_shared(sm_head);
                    begun = true;
                    cur = row[u];
                    clear();
                }
                if (row[u] < num_rows) {
#pragma unroll
                    for (int k = 0; k < V; ++k) acc[k] += to_f32(g[u].v[k]);
                }
            }
        }
        const bool goes_on = e1 < end && row_of(entries[e1]) == cur;
        if (!begun) {
            to_shared(sm_head);
            if (goes_on) flags |= kThrough;
        } else if (goes_on) {
            to_shared(sm_tail);
            flags |= kTail;
        } else {
            write_row(cur);
        }
    }
    if (lane == 0) sm_flags[team] = (uint8_t)flags;
    __syncthreads();
    // runs that cross teams: the team where a run begins adds the others' parts
    const uint32_t used = min(sh.teams, (hi - lo + per - 1) / per);
    auto add_heads = [&](uint32_t u) {  // from team u on; true where the run ends before `used`
        while (u < used) {
#pragma unroll
            for (int k = 0; k < V; ++k) acc[k] += sm_head[(u * sh.lanes + lane) * V + k];
            if (!(sm_flags[u] & kThrough)) return true;
            ++u;
        }
        return false;
    };
    auto to_global = [&](float* out) {
        if (!on || !out) return;
#pragma unroll
        for (int k = 0; k < V; ++k) out[col + k] = acc[k];
    };
    uint32_t left = 0;
    if (team < used && (flags & kTail)) {
#pragma unroll
        for (int k = 0; k < V; ++k) acc[k] = sm_tail[threadIdx.x * V + k];
        if (add_heads(team + 1)) {
            write_row(cur);
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

// Zeroes the rows [r0, r1) whose flag is 0: a team's lanes the same packs as above.
template <typename TT, int V>
__device__ __forceinline__ void zero_rows(const uint8_t* touched, uint32_t r0, uint32_t r1, const TeamShape& sh,
                                          TT* __restrict__ dtable, uint64_t ldt) {
    Pack<TT, V> z;
#pragma unroll
    for (int k = 0; k < V; ++k) z.v[k] = from_f32<TT>(0.f);
    const uint32_t pack = blockIdx.y * sh.lanes + threadIdx.x % sh.lanes;
    if (pack >= sh.packs) return;
    for (uint32_t r = r0 + threadIdx.x / sh.lanes; r < r1; r += sh.teams)
        if (!touched[r - r0]) store_pack_cs<TT, V>(dtable + (uint64_t)r * ldt + (uint64_t)pack * V, z);
}

// ------------------------------------------------------------ owner form --

constexpr uint32_t kOwnerMax = 2048;       // indices
constexpr uint32_t kOwnerRows = 8192;      // table rows of a CTA, at most
constexpr int kOwnerEach = kOwnerMax / kThreads;

template <typename TG, typename TT, int V>
__global__ void __launch_bounds__(kThreads) grad_owner_kernel(
    const TG* __restrict__ grad, uint64_t ldg, const void* __restrict__ idx, int idx_type, uint32_t n,
    int64_t padding, float scale, TT* __restrict__ dtable, uint64_t ldt, uint32_t num_rows, uint32_t rows,
    const TeamShape sh, uint32_t* __restrict__ bad) {
    __shared__ Entry entries[kOwnerMax];
    __shared__ uint8_t touched[kOwnerRows];
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
            if (!inside && id != padding && bad && blockIdx.x == 0) atomicExch(bad, 1u);
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
        sum_runs<TG, TT, V>(entries, 0, total, total, (total + sh.teams - 1) / sh.teams, grad, ldg, scale, dtable,
                            ldt, num_rows, sh, nullptr, nullptr, nullptr);
    }
    zero_rows<TT, V>(touched, r0, r1, sh, dtable, ldt);
}

template <typename TG, typename TT, int V>
void launch_owner(const EmbeddingArgs& a, cudaStream_t s) {
    const TeamShape sh = team_shape(a.F / V);
    const uint32_t num_rows = (uint32_t)a.num_rows;
    // four CTAs per SM, or what a CTA can own at most
    const uint32_t rows = std::min(kOwnerRows, std::max(1u, ceil_div(num_rows, 148 * 4)));
    const dim3 grid(ceil_div(num_rows, rows), sh.blocks);
    grad_owner_kernel<TG, TT, V><<<grid, kThreads, 0, s>>>(
        static_cast<const TG*>(a.rows), a.ldr, a.idx, a.idx_type, (uint32_t)a.n, a.padding, a.scale,
        static_cast<TT*>(a.table), a.ldt, num_rows, rows, sh, a.bad);
    TCC_CUDA(cudaGetLastError());
}

// ----------------------------------------------------------- sorted form --
//
// LSD radix sort of the entries by row, at most 11 bits a pass (two passes up to
// 4 M rows), three kernels a pass: digit counts per tile, offsets, scatter.  No
// CTA waits for another.

constexpr int kTileEach = 16;
constexpr uint32_t kTile = kThreads * kTileEach;  // entries of a tile
constexpr int kMaxDigitBits = 11;
constexpr uint32_t kMaxDigits = 1u << kMaxDigitBits;
constexpr int kWarps = kThreads / 32;

struct IndexSource {  // pass 0: the indices themselves; rows without a gradient sort last
    const void* idx;
    int type;
    int64_t padding;
    uint32_t num_rows;
    uint8_t* touched;
    uint32_t* bad;
    __device__ __forceinline__ Entry load(uint32_t i, bool note) const {
        const int64_t id = load_index(idx, type, i);
        const bool inside = id >= 0 && id < (int64_t)num_rows;
        const bool real = inside && id != padding;
        if (note) {
            if (!inside && id != padding && bad) atomicExch(bad, 1u);
            if (real) touched[id] = 1;
        }
        return (Entry)(real ? (uint32_t)id : num_rows) << 32 | i;
    }
};

struct EntrySource {
    const Entry* entries;
    __device__ __forceinline__ Entry load(uint32_t i, bool) const { return entries[i]; }
};

// counts [tile][digit], totals [digit] (zero before).
template <typename Source>
__global__ void __launch_bounds__(kThreads) digit_counts_kernel(const Source src, uint32_t n, int shift,
                                                                uint32_t digits, uint32_t* __restrict__ counts,
                                                                uint32_t* __restrict__ totals) {
    __shared__ uint32_t hist[kMaxDigits];
    for (uint32_t d = threadIdx.x; d < digits; d += kThreads) hist[d] = 0;
    __syncthreads();
    const uint32_t base = blockIdx.x * kTile;
#pragma unroll 8
    for (int k = 0; k < kTileEach; ++k) {
        const uint32_t i = base + k * kThreads + threadIdx.x;
        if (i < n) atomicAdd(&hist[(row_of(src.load(i, true)) >> shift) & (digits - 1)], 1u);
    }
    __syncthreads();
    for (uint32_t d = threadIdx.x; d < digits; d += kThreads) {
        counts[(uint64_t)blockIdx.x * digits + d] = hist[d];
        if (hist[d]) atomicAdd(&totals[d], hist[d]);
    }
}

// counts -> where a tile's first entry of each digit goes.  A CTA takes 32
// digits; 32 rows of threads share the tiles.
__global__ void __launch_bounds__(1024) digit_offsets_kernel(uint32_t* __restrict__ counts, uint32_t tiles,
                                                             uint32_t digits, const uint32_t* __restrict__ totals) {
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

// Stable: warp w ranks the tile's entries [w * 512, (w + 1) * 512) against its
// own digit counts; a prefix over the warps puts them in order.
template <typename Source>
__global__ void __launch_bounds__(kThreads) digit_scatter_kernel(const Source src, uint32_t n, int shift,
                                                                 uint32_t digits,
                                                                 const uint32_t* __restrict__ offsets,
                                                                 Entry* __restrict__ out) {
    __shared__ uint16_t cnt[kWarps][kMaxDigits];
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (uint32_t d = lane; d < digits; d += 32) cnt[warp][d] = 0;
    __syncwarp();
    const uint32_t base = blockIdx.x * kTile + warp * (kTile / kWarps) + lane;
    Entry e[kTileEach];
    uint32_t place[kTileEach];  // digit, and the rank among the warp's entries of that digit
#pragma unroll
    for (int k = 0; k < kTileEach; ++k) {
        const uint32_t i = base + k * 32;
        e[k] = i < n ? src.load(i, false) : ~0ull;
    }
#pragma unroll
    for (int k = 0; k < kTileEach; ++k) {
        const bool in = base + k * 32 < n;
        const uint32_t d = in ? (row_of(e[k]) >> shift) & (digits - 1) : kMaxDigits;
        const unsigned peers = __match_any_sync(0xffffffffu, d);
        const uint32_t rank = __popc(peers & lanemask_lt());
        const uint32_t seen = in ? cnt[warp][d] : 0;
        __syncwarp();
        if (in && rank == 0) cnt[warp][d] = (uint16_t)(seen + __popc(peers));
        __syncwarp();
        place[k] = d << 16 | (seen + rank);
    }
    __syncthreads();
    const uint32_t* offset = offsets + (uint64_t)blockIdx.x * digits;
    for (uint32_t d = threadIdx.x; d < digits; d += kThreads) {
        uint32_t run = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const uint32_t c = cnt[w][d];
            cnt[w][d] = (uint16_t)run;
            run += c;
        }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kTileEach; ++k) {
        if (base + k * 32 >= n) continue;
        const uint32_t d = place[k] >> 16;
        out[__ldg(offset + d) + cnt[warp][d] + (place[k] & 0xFFFFu)] = e[k];
    }
}

// Blocks [0, sums) of the grid's x: ranges of entries.  The others: rows
// without an entry, which become zero.
struct SortedShape {
    uint32_t per, range, sums, fill_rows;  // entries of a team, of a CTA; CTAs; rows of a fill CTA
};

template <typename TG, typename TT, int V>
__global__ void __launch_bounds__(kThreads) grad_sorted_kernel(
    const TG* __restrict__ grad, uint64_t ldg, const Entry* __restrict__ entries, uint32_t n, float scale,
    TT* __restrict__ dtable, uint64_t ldt, uint32_t num_rows, const TeamShape sh, const SortedShape so,
    const uint8_t* __restrict__ touched, float* __restrict__ heads, float* __restrict__ tails,
    Border* __restrict__ borders) {
    const uint32_t width = sh.packs * V;
    if (blockIdx.x < so.sums) {
        const uint32_t lo = blockIdx.x * so.range, hi = min(lo + so.range, n);
        sum_runs<TG, TT, V>(entries, lo, hi, n, so.per, grad, ldg, scale, dtable, ldt, num_rows, sh,
                            heads + (uint64_t)blockIdx.x * width, tails + (uint64_t)blockIdx.x * width,
                            borders + blockIdx.x);
    } else {
        const uint32_t r0 = (blockIdx.x - so.sums) * so.fill_rows;
        zero_rows<TT, V>(touched + r0, r0, min(r0 + so.fill_rows, num_rows), sh, dtable, ldt);
    }
}

// A block per range: where a run begins in it and goes on, its parts are added.
template <typename TT>
__global__ void __launch_bounds__(128) grad_join_kernel(const Border* __restrict__ borders, uint32_t sums,
                                                        const float* __restrict__ heads,
                                                        const float* __restrict__ tails, uint32_t width, float scale,
                                                        TT* __restrict__ dtable, uint64_t ldt, uint32_t num_rows) {
    const Border b = borders[blockIdx.x];
    if (!(b.flags & kTail) || b.row >= num_rows) return;
    // the ranges after it that hold a part: up to the first that is not passed through
    __shared__ uint32_t last;
    uint32_t from = blockIdx.x + 1;
    if (threadIdx.x == 0) last = sums;
    for (;; from += 128) {
        const uint32_t i = from + threadIdx.x;
        const bool ends = i >= sums || !(borders[i].flags & kThrough);
        __syncthreads();
        if (ends) atomicMin(&last, min(i, sums - 1));
        __syncthreads();
        if (last < sums) break;
    }
    for (uint32_t f = threadIdx.x; f < width; f += 128) {
        float acc = tails[(uint64_t)blockIdx.x * width + f];
#pragma unroll 8
        for (uint32_t i = blockIdx.x + 1; i <= last; ++i) acc += heads[(uint64_t)i * width + f];
        dtable[(uint64_t)b.row * ldt + f] = from_f32<TT>(acc * scale);
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
    p.bits = (total + p.passes - 1) / p.passes;
    p.digits = 1u << p.bits;
    p.tiles = ceil_div(n, kTile);
    return p;
}

// Entries of a team: about 16 CTAs per SM over the whole list (ranges long
// enough that few runs cross), at least 16.
SortedShape sorted_shape(uint64_t n, uint64_t num_rows, const TeamShape& sh) {
    SortedShape so;
    const uint64_t per = (n / (148 * 16) + sh.teams - 1) / sh.teams;
    so.per = (uint32_t)std::max<uint64_t>(16, (per + kUnroll - 1) / kUnroll * kUnroll);
    so.range = so.per * sh.teams;
    so.sums = ceil_div(n, so.range);
    so.fill_rows = 64;
    while (num_rows / so.fill_rows > (1u << 16)) so.fill_rows <<= 1;
    return so;
}

// Ranges whatever the vector width: a range is never below 16 entries of the
// eight teams that full warps give.
uint64_t max_sums(uint64_t n) { return n / (16 * kWarps) + 1; }

struct GradScratch {
    Entry *a, *b;
    uint32_t* counts;
    uint32_t* totals;   // [passes][digits], then `touched`: zeroed together
    uint8_t* touched;
    float *heads, *tails;
    Border* borders;
    size_t zero_bytes, bytes;
};

GradScratch lay_out(uint64_t n, uint64_t num_rows, uint32_t F, char* base) {
    GradScratch g;
    const SortPlan p = sort_plan(n, num_rows);
    uint64_t at = 0;
    auto take = [&](uint64_t bytes) {
        char* q = base + at;
        at += align256(bytes);
        return q;
    };
    g.a = reinterpret_cast<Entry*>(take(n * 8));
    g.b = reinterpret_cast<Entry*>(take(n * 8));
    g.counts = reinterpret_cast<uint32_t*>(take((uint64_t)p.tiles * p.digits * 4));
    const uint64_t zero = at;
    g.totals = reinterpret_cast<uint32_t*>(take((uint64_t)p.passes * p.digits * 4));
    g.touched = reinterpret_cast<uint8_t*>(take(num_rows));
    g.zero_bytes = at - zero;
    g.heads = reinterpret_cast<float*>(take(max_sums(n) * F * 4));
    g.tails = reinterpret_cast<float*>(take(max_sums(n) * F * 4));
    g.borders = reinterpret_cast<Border*>(take(max_sums(n) * sizeof(Border)));
    g.bytes = at;
    return g;
}

template <typename TG, typename TT, int V>
void launch_sorted(const EmbeddingArgs& a, char* scratch, cudaStream_t s) {
    const uint32_t n = (uint32_t)a.n, num_rows = (uint32_t)a.num_rows;
    const GradScratch g = lay_out(n, num_rows, a.F, scratch);
    const SortPlan p = sort_plan(n, num_rows);
    const TeamShape sh = team_shape(a.F / V);
    const SortedShape so = sorted_shape(n, num_rows, sh);
    TCC_CUDA(cudaMemsetAsync(g.totals, 0, g.zero_bytes, s));
    const IndexSource from_idx{a.idx, a.idx_type, a.padding, num_rows, g.touched, a.bad};
    Entry* in = g.b;
    Entry* out = g.a;
    for (int pass = 0; pass < p.passes; ++pass) {
        const int shift = pass * p.bits;
        uint32_t* totals = g.totals + (size_t)pass * p.digits;
        const EntrySource from_entries{in};
        if (pass == 0)
            digit_counts_kernel<<<p.tiles, kThreads, 0, s>>>(from_idx, n, shift, p.digits, g.counts, totals);
        else
            digit_counts_kernel<<<p.tiles, kThreads, 0, s>>>(from_entries, n, shift, p.digits, g.counts, totals);
        digit_offsets_kernel<<<ceil_div(p.digits, 32), 1024, 0, s>>>(g.counts, p.tiles, p.digits, totals);
        if (pass == 0)
            digit_scatter_kernel<<<p.tiles, kThreads, 0, s>>>(from_idx, n, shift, p.digits, g.counts, out);
        else
            digit_scatter_kernel<<<p.tiles, kThreads, 0, s>>>(from_entries, n, shift, p.digits, g.counts, out);
        std::swap(in, out);
    }
    const uint32_t fills = ceil_div(num_rows, so.fill_rows);
    grad_sorted_kernel<TG, TT, V><<<dim3(so.sums + fills, sh.blocks), kThreads, 0, s>>>(
        static_cast<const TG*>(a.rows), a.ldr, in, n, a.scale, static_cast<TT*>(a.table), a.ldt, num_rows, sh, so,
        g.touched, g.heads, g.tails, g.borders);
    if (so.sums > 1)
        grad_join_kernel<TT><<<so.sums, 128, 0, s>>>(g.borders, so.sums, g.heads, g.tails, a.F, a.scale,
                                                     static_cast<TT*>(a.table), a.ldt, num_rows);
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
    switch (rule.width()) {
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
