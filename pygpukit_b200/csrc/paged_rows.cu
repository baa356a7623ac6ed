// paged_rows.cu -- the positions of a cache that stay when it is cut, and rows of the pages that move together.
//
// Selection.  Of a sequence's positions the first, the recent and the ones of the largest weights stay, per key head, `budget` in all, in ascending order.  A block has one head, a
// warp a run of its positions, a weight as an ordered 32-bit number in a register.  The least that stays is found in four digits of eight bits, a histogram each, in which every lane
// has a column of its own: weights are alike in their upper digits, and a warp's 32 additions to one place would take turns.  Then a warp counts what stays of its run and writes it
// behind what the warps before it have.  A digit that nothing below the least shares ends the search.  Bound by its passes' latencies, 4 bytes a position being little: 2048 of 4096
// positions of 8 heads 7.1 us, 4096 of 8192 of 128 heads 12.0.
//
// Moving.  Row start + i of a sequence becomes, in place, what row start + from[i] was, from[i] >= i.  What is written lies before everything that is still to be read, from[i'] >= i' > i,
// but for the rows that are moved at the same time: a tile's rows are read by all of the cluster before any is written, and the next tile's are on their way
// meanwhile.  Bound by memory (2048 of 4096 rows of 128 heads and keys and values, 550 MB, 126 us) or, of few rows, by the chain from position to page to row: 4 rows in 16 layers 6.3 us.
#include "paged.cuh"
#include "../../include/pgk_b200.h"

namespace pgk {

namespace {

constexpr int C_THREADS = 1024, C_WARPS = C_THREADS / 32, C_BINS = 256;

struct SelectParams {
    const float* weights; long ld;
    const int32_t* seq_slots; const int32_t* contexts;
    int slots, kv_heads, budget, first, recent, most;
    int32_t* kept; int32_t* counts;
};

// a float's order as a number; the positions that stay in any case above all, NaN below all, one zero
__device__ __forceinline__ uint32_t ordered(float x) {
    if (x != x) return 0u;
    const uint32_t u = __float_as_uint(x + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// K: positions of a lane that stay in registers; 0: looked at anew in every pass
template <int K>
__global__ void __launch_bounds__(C_THREADS) select_kernel(const __grid_constant__ SelectParams p) {
    __shared__ int bins[C_BINS][32];
    __shared__ int sums[C_BINS], over[C_WARPS], same[C_WARPS];
    __shared__ int found, left, whole;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, head = blockIdx.x, seq = blockIdx.y;
    griddep_wait();
    griddep_launch();
    const int slot = __ldcg(p.seq_slots + seq);
    const bool there = (unsigned)slot < (unsigned)p.slots;
    const int ctx = there ? min(max(0, __ldcg(p.contexts + seq)), p.most) : 0, count = min(ctx, p.budget);
    int32_t* const kept = p.kept + ((size_t)seq * p.kv_heads + head) * p.budget;
    if (head == 0 && tid == 0) p.counts[seq] = count;
    for (int i = count + tid; i < p.budget; i += C_THREADS) kept[i] = -1;
    if (ctx <= p.budget) {
        for (int i = tid; i < count; i += C_THREADS) kept[i] = i;
        return;
    }
    const float* const w = p.weights + ((size_t)slot * p.kv_heads + head) * p.ld;
    const int recent = ctx - p.recent;
    const int run = K > 0 ? 32 * K : ((ctx + C_WARPS - 1) / C_WARPS + 31) & ~31, from = warp * run, to = min(ctx, from + run), n = to > from ? (to - from + 31) / 32 : 0;
    auto key = [&](int j) { return j >= to ? 0u : (j < p.first || j >= recent ? 0xffffffffu : ordered(__ldcg(w + j))); };
    uint32_t held[K > 0 ? K : 1];
    if constexpr (K > 0) {
#pragma unroll
        for (int i = 0; i < K; ++i) held[i] = key(from + 32 * i + lane);
    }
    // f(position, its key) for the run's positions, 32 at a time
    auto each = [&](auto f) {
        if constexpr (K > 0) {
#pragma unroll
            for (int i = 0; i < K; ++i)
                if (i < n) f(from + 32 * i + lane, held[i]);
        } else
            for (int i = 0; i < n; ++i) f(from + 32 * i + lane, key(from + 32 * i + lane));
    };
    // the least key that stays: digit by digit, `need` of those that share the digits so far
    uint32_t least = 0;
    int need = count;
#pragma unroll 1
    for (int shift = 24; shift >= 0; shift -= 8) {
        const uint32_t above = shift == 24 ? 0u : 0xffffffffu << (shift + 8);
#pragma unroll
        for (int i = 0; i < C_BINS / C_WARPS; ++i) bins[warp + C_WARPS * i][lane] = 0;
        __syncthreads();
        each([&](int j, uint32_t x) {
            if (j < to && (x & above) == least) atomicAdd(&bins[(x >> shift) & 255u][lane], 1);
        });
        __syncthreads();
        int x[C_BINS / C_WARPS];
#pragma unroll
        for (int i = 0; i < C_BINS / C_WARPS; ++i) x[i] = bins[warp + C_WARPS * i][lane];
        const int sum = reduce_lanes<C_BINS / C_WARPS>(x, lane, [](int a, int b) { return a + b; });
        if (lane < C_BINS / C_WARPS) sums[warp + C_WARPS * lane] = sum;
        __syncthreads();
        if (warp == 0) {                                      // the bin with the need-th from above: lane l has bins 8 l ... 8 l + 7
            int mine[8], all = 0;
#pragma unroll
            for (int i = 7; i >= 0; --i) mine[i] = all += sums[8 * lane + i];         // of it and the lane's higher ones
            int after = all;
#pragma unroll
            for (int x = 1; x < 32; x <<= 1) {
                const int got = __shfl_down_sync(0xffffffffu, after, x);
                if (lane + x < 32) after += got;
            }
            after -= all;                                     // keys in the bins of the lanes after this one
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int higher = after + (i < 7 ? mine[i + 1] : 0);
                if (higher < need && need <= after + mine[i]) {
                    found = 8 * lane + i;
                    left = need - higher;
                    whole = need == after + mine[i];
                }
            }
        }
        __syncthreads();
        least |= (uint32_t)found << shift;
        need = left;
        if (whole) break;                                     // all that share the digits stay; what they have behind them does not count
    }
    // those above the least, and the first `need` of its equals
    int n_over = 0, n_same = 0;
    each([&](int j, uint32_t x) {
        n_over += __popc(__ballot_sync(0xffffffffu, j < to && x > least));
        n_same += __popc(__ballot_sync(0xffffffffu, j < to && x == least));
    });
    if (lane == 0) { over[warp] = n_over; same[warp] = n_same; }
    __syncthreads();
    static_assert(C_WARPS == 32);
    int seen = __reduce_add_sync(0xffffffffu, lane < warp ? same[lane] : 0), at = __reduce_add_sync(0xffffffffu, lane < warp ? over[lane] : 0) + min(seen, need);
    each([&](int j, uint32_t x) {
        const uint32_t eq = __ballot_sync(0xffffffffu, j < to && x == least), below = (1u << lane) - 1u;
        const bool stays = j < to && (x > least || (x == least && seen + __popc(eq & below) < need));
        const uint32_t all = __ballot_sync(0xffffffffu, stays);
        if (stays) kept[at + __popc(all & below)] = j;
        at += __popc(all);
        seen += __popc(eq);
    });
}

constexpr int M_THREADS = 256, M_UNITS = 8, M_TILE = M_THREADS * M_UNITS, M_ARRAYS = 192, M_CLUSTER = 8;

struct MoveParams {
    void* arrays[M_ARRAYS];
    int n, bytes, chunk;                  // arrays, bytes of a row, arrays of a block
    const int32_t* table;
    int pages, page_size, slots, max_pages, kv_heads;
    const int32_t* seq_slots; const int32_t* starts;
    const int32_t* from; const int32_t* counts;
    int width, by_head;                   // from [sequences][kv_heads if by_head][width]
    float* weights; long weights_ld;      // moved as well, [slots][kv_heads][weights_ld]; what is behind the last row up to the context becomes zero
    const int32_t* contexts;
    PagedDiv by_page, by_units;
};

template <int V> struct Unit;
template <> struct Unit<16> { using T = uint4; };
template <> struct Unit<4> { using T = uint32_t; };
template <> struct Unit<2> { using T = uint16_t; };
__device__ __forceinline__ uint4 load_unit(const uint4* p) { return ld_act16(p); }
__device__ __forceinline__ uint32_t load_unit(const uint32_t* p) { return __ldcg(p); }
__device__ __forceinline__ uint16_t load_unit(const uint16_t* p) { return ld_act2(p); }

// A block has a head of a sequence in `chunk` arrays.  Rows of a tile: their places, looked up while the tile before is on its way, are the same in all arrays, and with
// few rows several arrays' make a tile.
template <int V>
__global__ void __launch_bounds__(M_THREADS, 3) move_kernel(const __grid_constant__ MoveParams p) {
    using T = typename Unit<V>::T;
    __shared__ int2 places[2][M_TILE];                        // of a tile's rows: from, to; from below 0: in its place, or not at all
    const int tid = threadIdx.x, rank = blockIdx.x, blocks = gridDim.x, chunk = blockIdx.y / p.kv_heads, head = blockIdx.y - chunk * p.kv_heads, seq = blockIdx.z;
    griddep_wait();
    griddep_launch();
    const int slot = __ldcg(p.seq_slots + seq);
    const bool there = (unsigned)slot < (unsigned)p.slots;                // the same in all of the cluster
    const int count = there ? max(0, min(__ldcg(p.counts + seq), p.width)) : 0, start = p.starts ? __ldcg(p.starts + seq) : 0;
    const int32_t* const from = p.from + ((size_t)seq * (p.by_head ? p.kv_heads : 1) + (p.by_head ? head : 0)) * p.width;
    auto all = [&]() {
        if (blocks > 1) paged_cluster_sync();
        else __syncthreads();
    };
    const int a0 = chunk * p.chunk, arrays = min(p.chunk, p.n - a0);
    if (arrays > 0) {
        const int32_t* const table = p.table + (there ? (size_t)slot * p.max_pages : 0);
        auto row_of = [&](long long j) {
            if (j < 0 || j >= (long long)p.max_pages * p.page_size) return -1;
            const int pg = paged_div((int)j, p.by_page), page = __ldcg(table + pg);
            return (unsigned)page >= (unsigned)p.pages ? -1 : (page * p.kv_heads + head) * p.page_size + ((int)j - pg * p.page_size);
        };
        const uint32_t units = (uint32_t)(p.bytes / V);
        // rows of a tile: of one array as many as it has units for, or all there are and as many arrays
        const int per = max(1, (int)(M_TILE / units)), rows = min(per, count), group = count <= per && blocks == 1 ? max(1, per / max(1, count)) : 1;
        const int tiles = rows > 0 ? (count + rows * blocks - 1) / (rows * blocks) : 0;
        const uint32_t per_array = (1u << 22) / (uint32_t)max(1, rows) + 1u;                // exact for ar < 2^11
        auto look = [&](int tile) {
            const int i0 = (tile * blocks + rank) * rows;
            for (int r = tid; r < rows; r += M_THREADS) {
                const int i = i0 + r, f = i < count ? __ldcg(from + i) : -1;
                int2 x = make_int2(-1, -1);
                if (f > i) x = make_int2(row_of((long long)start + f), row_of((long long)start + i));           // (before it nothing is moved from)
                if (x.y < 0) x.x = -1;
                places[tile & 1][r] = x;
            }
        };
        if (tiles > 0) look(0);
        __syncthreads();
        for (int a = 0; a < arrays; a += group) {
            const int n = min(group, arrays - a);
            for (int t = 0; t < tiles; ++t) {
                // rows of more units than a tile has go piece by piece
                for (uint32_t c0 = 0; c0 < units; c0 += M_TILE) {
                    const uint32_t wide = min(units - c0, (uint32_t)M_TILE), total = wide * (uint32_t)rows * (uint32_t)n;
                    T x[M_UNITS];
                    T *to[M_UNITS], *at[M_UNITS];
#pragma unroll
                    for (int q = 0; q < M_UNITS; ++q) {               // all addresses before the first load: no branch between
                        const uint32_t e = (uint32_t)(q * M_THREADS + tid), ar = units > M_TILE ? 0u : (uint32_t)paged_div((int)e, p.by_units), c = c0 + (e - ar * wide);
                        const uint32_t k = group > 1 ? min(__umulhi(ar << 10, per_array), (uint32_t)n - 1u) : 0u;         // ar / rows
                        const int2 row = places[t & 1][min(ar - k * (uint32_t)rows, (uint32_t)M_TILE - 1u)];
                        T* const base = (T*)p.arrays[a0 + a + (int)k];
                        at[q] = base + (size_t)max(row.x, 0) * units + c;
                        to[q] = e < total && row.x >= 0 ? base + (size_t)max(row.y, 0) * units + c : nullptr;
                    }
#pragma unroll
                    for (int q = 0; q < M_UNITS; ++q)
                        if (to[q]) x[q] = load_unit(at[q]);
                    if (c0 + M_TILE >= units) {
                        if (t + 1 < tiles) look(t + 1);
                        else if (tiles % 2 == 0) look(0);         // for the next array; this tile is in the other buffer
                    }
                    all();
#pragma unroll
                    for (int q = 0; q < M_UNITS; ++q)
                        if (to[q]) *to[q] = x[q];
                }
            }
            if (tiles > 1 && tiles % 2 && a + group < arrays) {           // this tile was in tile 0's buffer
                __syncthreads();
                look(0);
                __syncthreads();
            }
        }
        return;
    }
    if (!there) return;
    float* const w = p.weights + ((size_t)slot * p.kv_heads + head) * p.weights_ld;
    for (long long i0 = 0; i0 < count; i0 += (long long)M_TILE * blocks) {
        float x[M_UNITS];
        long long to[M_UNITS];
#pragma unroll
        for (int q = 0; q < M_UNITS; ++q) {
            const long long i = i0 + ((long long)rank * M_UNITS + q) * M_THREADS + tid;
            to[q] = -1;
            if (i >= count) continue;
            const int f = __ldcg(from + i);
            const long long src = (long long)start + f, dst = (long long)start + i;
            if (f <= i || dst < 0 || src >= p.weights_ld) continue;
            x[q] = __ldcg(w + src);
            to[q] = dst;
        }
        all();
#pragma unroll
        for (int q = 0; q < M_UNITS; ++q)
            if (to[q] >= 0) w[to[q]] = x[q];
    }
    all();                                         // all rows are read
    const long long end = min((long long)__ldcg(p.contexts + seq), (long long)p.weights_ld);
    for (long long j = max(0ll, (long long)start + count) + rank * M_THREADS + tid; j < end; j += blocks * M_THREADS) w[j] = 0.f;
}

}  // namespace

}  // namespace pgk

using namespace pgk;

extern "C" int pgk_select_rows(const float* weights, long weights_ld, const int32_t* seq_slots, const int32_t* context_lens, int seqs, int slots, int kv_heads, int max_context,
                               int budget, int first, int recent, int32_t* kept, int32_t* counts, void* stream) {
    PGK_REQUIRE(seqs >= 0 && seqs <= 65535 && slots > 0 && kv_heads > 0 && max_context >= 0 && max_context <= PAGED_MOST && weights_ld >= max_context, "select_rows failed: %d sequences, %d slots of %d heads, %d of %ld positions",
                seqs, slots, kv_heads, max_context, weights_ld);
    PGK_REQUIRE(budget > 0 && first >= 0 && recent >= 0 && (long long)first + recent <= budget, "select_rows failed: a budget of %d with %d first and %d recent positions", budget, first, recent);
    if (seqs == 0) return 0;
    PGK_REQUIRE(weights && seq_slots && context_lens && kept && counts, "select_rows failed: an array is missing");
    SelectParams p = {weights, weights_ld, seq_slots, context_lens, slots, kv_heads, budget, first, recent, max_context, kept, counts};
    const auto kernel = max_context <= 4 * C_THREADS ? select_kernel<4> : (max_context <= 8 * C_THREADS ? select_kernel<8> :
                        (max_context <= 16 * C_THREADS ? select_kernel<16> : select_kernel<0>));
    PGK_CUDA(launch_waiting(kernel, dim3(kv_heads, seqs), dim3(C_THREADS), 0, (cudaStream_t)stream, p));
    return 0;
}

extern "C" int pgk_move_rows(void* const* host_arrays, const int32_t* host_row_bytes, int n_arrays, const int32_t* page_table, int pages, int page_size, int slots, int max_pages,
                             int kv_heads, const int32_t* seq_slots, const int32_t* starts, const int32_t* from, const int32_t* counts, int seqs, int width, int by_head, float* weights,
                             long weights_ld, const int32_t* context_lens, void* stream) {
    PGK_REQUIRE(n_arrays >= 0 && pages > 0 && page_size > 0 && slots > 0 && max_pages > 0 && kv_heads > 0 && seqs >= 0 && seqs <= 65535 && width >= 0 && width <= PAGED_MOST && weights_ld >= 0,
                "move_rows failed: %d arrays of %d pages of %d positions, %d slots of %d pages, %d heads, %d sequences", n_arrays, pages, page_size, slots, max_pages, kv_heads, seqs);
    PGK_REQUIRE((long long)pages * kv_heads * page_size <= 0x7fffffffll && (long long)max_pages * page_size <= 0x7fffffffll && kv_heads <= 65535,
                "move_rows failed: too many rows or heads");
    if (seqs == 0 || (width == 0 && !weights) || (n_arrays == 0 && !weights)) return 0;
    PGK_REQUIRE(page_table && seq_slots && from && counts && (n_arrays == 0 || (host_arrays && host_row_bytes)) && (!weights || context_lens), "move_rows failed: an array is missing");
    MoveParams p = {};
    p.table = page_table; p.pages = pages; p.page_size = page_size; p.slots = slots; p.max_pages = max_pages; p.kv_heads = kv_heads;
    p.seq_slots = seq_slots; p.starts = starts; p.from = from; p.counts = counts; p.width = width; p.by_head = by_head;
    p.weights_ld = weights_ld; p.contexts = context_lens;
    p.by_page = paged_divisor(page_size);
    const cudaStream_t st = (cudaStream_t)stream;
    for (int a = 0; a < n_arrays; ++a)
        PGK_REQUIRE(host_arrays[a] && host_row_bytes[a] > 0 && host_row_bytes[a] % 2 == 0, "move_rows failed: rows of %d bytes", host_row_bytes[a]);
    auto move = [&]() -> int {
        uintptr_t low = (uintptr_t)p.bytes;
        for (int a = 0; a < p.n; ++a) low |= (uintptr_t)p.arrays[a];
        const int unit = low % 16 == 0 ? 16 : (low % 4 == 0 ? 4 : 2);
        p.by_units = paged_divisor(p.bytes / unit);
        // arrays of a block: as many as leave four blocks a SM, where there are so many
        p.chunk = (int)((long long)p.n * kv_heads * seqs / (4 * sm_count()));
        if (p.chunk < 1) p.chunk = 1;
        const int chunks = (p.n + p.chunk - 1) / p.chunk + (p.weights ? 1 : 0);
        PGK_REQUIRE((long long)chunks * kv_heads <= 65535, "move_rows failed: too many heads");
        // blocks that share a head's rows: until there are twelve a SM, which even out (256 heads of 4096 rows, 1 / 2 / 4 / 8 blocks, before the addresses came before the loads: 139 / 148 / 132 / 147 us; now 126 with 4), none with less than a tile
        const long long items = (long long)chunks * kv_heads * seqs;
        int blocks = 1;
        while (blocks < M_CLUSTER && items * blocks * 2 <= 12 * sm_count() && (long long)width * (p.bytes / unit) > (long long)M_TILE * blocks) blocks *= 2;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(blocks, (unsigned)(chunks * kv_heads), (unsigned)seqs);
        cfg.blockDim = dim3(M_THREADS);
        cfg.stream = st;
        cudaLaunchAttribute attr[2];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        attr[1].id = cudaLaunchAttributeClusterDimension;
        attr[1].val.clusterDim.x = (unsigned)blocks;
        attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 2;
        count_launch();
        PGK_CUDA(unit == 16 ? cudaLaunchKernelEx(&cfg, move_kernel<16>, p) : (unit == 4 ? cudaLaunchKernelEx(&cfg, move_kernel<4>, p) : cudaLaunchKernelEx(&cfg, move_kernel<2>, p)));
        p.weights = nullptr;
        p.n = 0;
        return 0;
    };
    // a launch has arrays of one row size, the first one the weights as well
    p.weights = weights;
    for (int a = 0; a < n_arrays; ++a) {
        bool before = false;
        for (int e = 0; e < a && !before; ++e) before = host_row_bytes[e] == host_row_bytes[a];
        if (before) continue;
        p.bytes = host_row_bytes[a];
        for (int e = a; e < n_arrays; ++e) {
            if (host_row_bytes[e] != p.bytes) continue;
            p.arrays[p.n++] = host_arrays[e];
            if (p.n == M_ARRAYS)
                if (int rc = move()) return rc;
        }
        if (p.n > 0)
            if (int rc = move()) return rc;
    }
    if (n_arrays == 0) {
        p.bytes = 2;
        return move();
    }
    return 0;
}
