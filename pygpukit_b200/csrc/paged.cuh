// paged.cuh -- a key / value cache of 16 or 32 bits in pages [pages][kv_heads][page_size][dim] behind a page table [slots][pages of a slot], and the steps of
// sequences that attend over it: what paged_few.cu, paged_tc.cu, paged_f32.cu (attention) and paged_weigh.cu (weights by position) share.
//
// A sequence has n rows of the queries, which are the last n of its context's positions: step row t lies at position context - n + t.  Row i sees every position
// before context - n and, of the step's, those whose bit is set in its mask, or without masks the rows 0 ... i.  Slots, contexts, row starts and page numbers are
// data of the device: whatever they say, nothing outside the arrays is touched.
#pragma once
#include <mutex>

#include "tc_common.cuh"

namespace pgk {

// n / d = hi(n mul) >> shift for n < 2^31; mul 0: d = 1
struct PagedDiv { uint32_t mul, shift; };
inline PagedDiv paged_divisor(int d) {
    if (d <= 1) return {0u, 0u};
    uint32_t log = 0;                     // the least with d <= 2^log
    while ((1ull << log) < (uint64_t)d) ++log;
    return {(uint32_t)((1ull << (31 + log)) / (uint64_t)d + 1), log - 1};
}

struct PagedParams {
    const void* q; void* out;
    long q_ld, o_ld;                      // elements
    const void* k_data; const void* v_data;
    const int32_t* table;
    int pages, page_size, slots, max_pages, kv_heads, dim;
    const int32_t* seq_slots; const int32_t* contexts; const int32_t* starts;      // starts NULL: a row a sequence
    int seqs, tokens, max_rows, max_keys, heads, rep, tiles, splits;
    float scale_log2;                     // scale log2 e
    float zero;                           // what a product is added to so that it is rounded: of a product and a sum alone the compiler makes one multiply-add
    const int32_t* masks;                 // [tokens][words], or NULL
    int words;
    float* lse;                           // [tokens][heads] natural logarithms, or NULL
    float* partial;                       // NULL: the blocks that share a sequence's keys are a cluster; otherwise where each leaves its sums, [item][head][split][ROWS][DN + 4]
    float* weights; long weights_ld;      // paged_weigh.cu: [slots][kv_heads][weights_ld]
    bool wide_q, wide_o;                  // rows on 16-byte boundaries
    PagedDiv by_page, by_rep, by_seqs, by_splits;
};

// paged_tc.cu: whether it serves the call, and the call; paged_few.cu: what it does not; paged_f32.cu
bool paged_tc_serves(const PagedParams& p, int dtype);
int paged_tc(const PagedParams& p, int dtype, cudaStream_t st);
int paged_few(const PagedParams& p, int dtype, cudaStream_t st);
int paged_f32(const PagedParams& p, cudaStream_t st);

constexpr int PAGED_MOST = 0x7fff0000;       // of what a kernel counts in steps of up to 2^15: the count behind the last stays in 32 bits
constexpr int PAGED_CLUSTER = 16, PAGED_APART = 32;       // blocks that share a sequence's keys, at most: of a cluster, and one by one
static_assert(PAGED_APART <= 32);          // a lane of the join has one

// How many clusters of a kernel run at once: of eight blocks, one a SM, fewer than 148 / 8; 0: none of that size runs
template <typename... KArgs>
inline cudaError_t clusters_at_once(int* out, void (*kernel)(KArgs...), int threads, size_t smem, int blocks) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = (unsigned)blocks;
    cfg.gridDim = dim3(1, 1, (unsigned)blocks);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    *out = 0;
    const cudaError_t e = cudaOccupancyMaxActiveClusters(out, kernel, &cfg);
    if (e == cudaSuccess || blocks == 1) return e;
    cudaGetLastError();
    *out = 0;
    return cudaSuccess;
}
// What a launcher has asked once, by the first thread that comes: a call's split, and with it its bits, is the same in all
struct PagedOccupancy {
    std::mutex mutex;
    bool asked = false;
    int at_once[PAGED_CLUSTER + 1] = {};
    template <typename F> cudaError_t once(F ask) {
        std::lock_guard<std::mutex> lock(mutex);
        if (asked) return cudaSuccess;
        const cudaError_t e = ask(at_once);
        asked = e == cudaSuccess;
        return e;
    }
};
// Blocks that share a sequence's tiles.  As a cluster, which folds through shared memory: rounds of clusters times (a block's tiles + what it costs besides, in tiles).  Or one by
// one, which leave their sums in memory for another launch (half as much again): where clusters do not fill the SMs.  One sequence of 8 key heads, us: 1 row over 4096 keys, clusters
// of 10 11.5 and 18 blocks apart 11.6; over 8000 15.2 and 13.6, over 32000 37 and 32; 208 rows over 32000 in two tiles, clusters of 6 54 and 9 blocks apart 45.
// Eight trees of 128 float32 rows over 4000 keys, 1 / 2 / 3 blocks: 379 / 316 / 360.
struct PagedSplit { int splits; bool apart; };
inline PagedSplit paged_split(const PagedParams& p, int keys, const int* at_once, int most, int ends) {
    const int nt = (p.max_keys + keys - 1) / keys;
    const long long items = (long long)p.seqs * p.tiles * p.kv_heads;
    long long least = 0;
    PagedSplit best = {1, false};
    for (int s = 1; s <= most; ++s) {
        if (s > 1 && at_once[s] <= 0) continue;                                            // none of that size runs: its launch would fail
        const int fit = at_once[s] > 0 ? at_once[s] : 1;
        long long rounds = (8 * items + fit - 1) / fit;                                    // in eighths, whole ones up to two: then blocks no longer end together
        if (rounds <= 16) rounds = (rounds + 7) & ~7ll;
        const long long cost = rounds * ((nt + s - 1) / s + ends);
        if (s == 1 || cost < least) { best = {s, false}; least = cost; }
    }
    for (int s = 2; s <= PAGED_APART && items * s <= at_once[1]; ++s) {
        const long long cost = 8 * ((nt + s - 1) / s) + 12 * ends;
        if (cost < least) { best = {s, true}; least = cost; }
    }
    return best;
}

// blocks of a cluster along z, and the launch that waits for the kernel before it
template <typename... KArgs, typename... Args>
inline cudaError_t launch_clusters(void (*kernel)(KArgs...), dim3 grid, bool apart, int threads, size_t smem, cudaStream_t st, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = 1;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = apart ? 1u : grid.z;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    count_launch();
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
}

#ifdef __CUDACC__

constexpr float PAGED_LOG2E = 1.4426950408889634f, PAGED_LN2 = 0.6931471805599453f, PAGED_LAZY = 8.f;
// A row's reference m from its largest score (log2).  A weight is 2^(x - m) with x, the score times the factor, rounded as m is: left exact in one multiply-add, the rounding of m would
// be a factor of all weights of the row, 2^(2^-2) at 2^22 but 2^256 at 2^32.  (Two instructions for two scores where one would do: 8 x 64 rows over 4100 keys 49.5 -> 51.9 us, 13 rows of 16
// sequences 25.6 -> 26.0, few rows as before; a second form of a tile behind a branch 52.4 and more.)  float16 weights go from 2^6 down, so that small ones keep their bits, and grow to 2^14; where a
// reference has no bits for that, from 1.
template <int DT> __device__ __forceinline__ float paged_reference(float top) { return DT == 1 && fabsf(top) < 4194304.f ? top - 6.f : top; }

__device__ __forceinline__ int paged_div(int n, PagedDiv d) { return d.mul ? (int)(__umulhi((uint32_t)n, d.mul) >> d.shift) : n; }       // n not negative

// A block's rows -- ROWS of one sequence's, a token's query heads of one key head beside each other -- and the keys that they see between them, cut over the blocks of a
// cluster in units of UNIT keys.
template <int ROWS, int UNIT> struct PagedBlock {
    int seq, head, split, slot, ctx, first, n_rows, f0, live, base, end, ubeg, uend;       // base: the position of the step's row 0
    const int32_t* table;
    __device__ __forceinline__ PagedBlock(const PagedParams& p, int item, int head_, int split_) : head(head_), split(split_) {
        const int turn = paged_div(item, p.by_seqs);
        seq = item - turn * p.seqs;
        f0 = (p.tiles - 1 - turn) * ROWS;
        slot = __ldcg(p.seq_slots + seq);
        ctx = max(0, __ldcg(p.contexts + seq));
        first = p.starts ? __ldcg(p.starts + seq) : seq;
        n_rows = p.starts ? max(0, __ldcg(p.starts + seq + 1) - first) : 1;
        const int rows = min(n_rows, p.max_rows) * p.rep;                                // fits: checked by the host
        const bool work = f0 < rows && (unsigned)slot < (unsigned)p.slots && ctx > 0;
        live = f0 < rows && (unsigned)slot < (unsigned)p.slots ? min(ROWS, rows - f0) : 0;
        base = ctx - n_rows;                                                             // may lie before position 0: those rows have no key
        const int last = p.masks ? ctx : base + paged_div(f0 + max(live, 1) - 1, p.by_rep) + 1;      // behind the last key that a row sees
        end = work ? max(0, min(min(last, ctx), p.max_keys)) : 0;
        const int nu = (end + UNIT - 1) / UNIT, per = paged_div(nu + p.splits - 1, p.by_splits);
        ubeg = min(nu, split * per);
        uend = min(nu, ubeg + per);
        table = p.table + (work ? (size_t)slot * p.max_pages : 0);
    }
    // the cache row (of dim elements) that holds position j of the head, or -1
    __device__ __forceinline__ int row_of(const PagedParams& p, int j) const {
        if (j < 0 || j >= end) return -1;
        const int pg = paged_div(j, p.by_page);
        const int page = __ldcg(table + pg);
        if ((unsigned)page >= (unsigned)p.pages) return -1;
        return (page * p.kv_heads + head) * p.page_size + (j - pg * p.page_size);
    }
    __device__ __forceinline__ int token(const PagedParams& p, int r) const { return first + paged_div(f0 + r, p.by_rep); }
};

// Whether step row i sees step row t
__device__ __forceinline__ bool paged_sees(const PagedParams& p, int tok, int i, int t) {
    if (!p.masks) return t <= i;
    return (unsigned)tok < (unsigned)p.tokens && t < 32 * p.words && ((uint32_t)__ldcg(p.masks + (size_t)tok * p.words + (t >> 5)) >> (t & 31)) & 1u;
}
// of step rows t ... t + 31 the ones that row i sees; those before the step (t < 0) all
__device__ __forceinline__ uint32_t paged_window(const PagedParams& p, int tok, int i, int t) {
    if (t <= -32) return 0xffffffffu;
    if (!p.masks) return t > i ? 0u : (i - t >= 31 ? 0xffffffffu : (2u << (i - t)) - 1u);
    if ((unsigned)tok >= (unsigned)p.tokens) return 0u;        // nobody's row
    const int32_t* row = p.masks + (size_t)tok * p.words;
    const int w = t >> 5;                                     // floor
    const uint32_t lo = w < 0 ? 0xffffffffu : (w < p.words ? (uint32_t)__ldcg(row + w) : 0u);
    const uint32_t hi = w + 1 < p.words ? (uint32_t)__ldcg(row + w + 1) : 0u;
    return __funnelshift_r(lo, hi, (uint32_t)t & 31u);
}

__device__ __forceinline__ void paged_cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t paged_remote(uint32_t at, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(at), "r"(rank));
    return r;
}
__device__ __forceinline__ float paged_remote_float(uint32_t at) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
    return v;
}
template <int DT> __device__ __forceinline__ uint32_t paged_pack2(float lo, float hi) {
    if constexpr (DT == 1) {
        const __half2 h = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&h);
    } else
        return pack_bf16x2(lo, hi);
}
// Two weights (not negative) as one word.  bfloat16: rounded up from the half on by integers, since the conversion shares its unit with the exponentials: of a tile of 128 x 128
// scores 512 cycles beside their 1024.  (A NaN may get lost; the row's sum has it.)
template <int DT> __device__ __forceinline__ uint32_t paged_weights2(float a, float b) {
    if constexpr (DT == 1) return paged_pack2<1>(a, b);
    else return __byte_perm(__float_as_uint(a) + 0x8000u, __float_as_uint(b) + 0x8000u, 0x7632);
}
// the same as two terms: what is left of the first one's cut
template <int DT> __device__ __forceinline__ void paged_weights2x2(float a, float b, uint32_t& hi, uint32_t& lo) {
    if constexpr (DT == 1) {
        hi = paged_pack2<1>(a, b);
        const float2 back = __half22float2(*reinterpret_cast<const __half2*>(&hi));
        lo = paged_pack2<1>(a - back.x, b - back.y);
    } else {
        const uint32_t x = __float_as_uint(a), y = __float_as_uint(b);
        hi = __byte_perm(x, y, 0x7632);
        const float u = a - __uint_as_float(x & 0xffff0000u), v = b - __uint_as_float(y & 0xffff0000u);
        lo = __byte_perm(__float_as_uint(u) + 0x8000u, __float_as_uint(v) + 0x8000u, 0x7632);
    }
}
template <int DT> __device__ __forceinline__ float paged_float(const void* base, size_t at) {
    if constexpr (DT == 0) return __ldcg((const float*)base + at);
    else if constexpr (DT == 1) return __half2float(__ushort_as_half(ld_act2((const uint16_t*)base + at)));
    else return bf16_bits_to_f32(ld_act2((const uint16_t*)base + at));
}
// an infinity or NaN among the two 16-bit numbers of a word: those halves' bits
template <int DT> __device__ __forceinline__ uint32_t paged_unfinite(uint32_t w) {
    constexpr uint32_t E = DT == 1 ? 0x7c00u : 0x7f80u;
    return ((w & E) == E ? 0xffffu : 0u) | ((w & (E << 16)) == (E << 16) ? 0xffff0000u : 0u);
}
// pairs of float32 in a register pair: one instruction for two products or sums
__device__ __forceinline__ uint64_t pair(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpair(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
// the lanes' N values (a power of two up to 32) reduced over the warp: lane l ends with value l % N
template <int N, typename T, typename F> __device__ __forceinline__ T reduce_lanes(T (&v)[N], int lane, F f) {
#pragma unroll
    for (int w = N / 2; w > 0; w >>= 1) {
        const bool up = lane & w;
#pragma unroll
        for (int j = 0; j < w; ++j) {
            const T got = __shfl_xor_sync(0xffffffffu, up ? v[j] : v[j + w], w);
            v[j] = f(up ? v[j + w] : v[j], got);
        }
    }
    T x = v[0];
#pragma unroll
    for (int w = N; w < 32; w <<= 1) x = f(x, __shfl_xor_sync(0xffffffffu, x, w));
    return x;
}
// 2^(s - m) for a reference that is not there yet (m = -infinity)
__device__ __forceinline__ float paged_neg(float m) { return m == -INFINITY ? 0.f : -m; }

// A tile of V in shared memory, `chunks` of 64 elements (128 bytes a key, `chunk` bytes each), keys j0 on, as a warp has fetched it in pieces of bp positions: the values of positions
// [from, end) that are not finite become zeros -- true where there were any --, and what lies behind the end in the last piece as well (what was not fetched is zeros).
template <int DT> __device__ __forceinline__ bool paged_fix_values(uint32_t tile, int chunks, uint32_t chunk, int j0, int from, int end, int bp, int lane) {
    const int k0 = max(0, from - j0), k1 = min(128, end - j0);
    auto unit = [&](uint32_t a, uint32_t (&x)[4]) {
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]) : "r"(a) : "memory");
    };
    auto put = [&](uint32_t a, const uint32_t (&x)[4]) {
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" :: "r"(a), "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]) : "memory");
    };
    uint32_t most = 0;                                        // the largest magnitude says whether there are any
#pragma unroll 4
    for (int e = k0 * 8 + lane; e < k1 * 8; e += 32)
        for (int c = 0; c < chunks; ++c) {
            uint32_t x[4];
            unit(tile + (uint32_t)c * chunk + (uint32_t)e * 16u, x);
#pragma unroll
            for (int y = 0; y < 4; ++y) most = __vmaxu2(most, x[y] & 0x7fff7fffu);
        }
    const bool bad = __any_sync(0xffffffffu, paged_unfinite<DT>(most) != 0);
    if (bad)
        for (int e = k0 * 8 + lane; e < k1 * 8; e += 32)
            for (int c = 0; c < chunks; ++c) {
                const uint32_t a = tile + (uint32_t)c * chunk + (uint32_t)e * 16u;
                uint32_t x[4];
                unit(a, x);
#pragma unroll
                for (int y = 0; y < 4; ++y) x[y] &= ~paged_unfinite<DT>(x[y]);
                put(a, x);
            }
    const uint32_t none[4] = {0, 0, 0, 0};
    const int z1 = bp ? min(128, (max(0, k1) + bp - 1) & ~(bp - 1)) : 0;
    for (int e = max(0, k1) * 8 + lane; e < z1 * 8; e += 32)
        for (int c = 0; c < chunks; ++c) put(tile + (uint32_t)c * chunk + (uint32_t)e * 16u, none);
    return bad;
}

// A row's outputs d ... d + 3, rounded and written
template <int DT> __device__ __forceinline__ void paged_put(const PagedParams& p, size_t at, float4 o) {
    if constexpr (DT == 0) {
        float* dst = (float*)p.out + at;
        if (p.wide_o) *(float4*)dst = o;
        else { dst[0] = o.x; dst[1] = o.y; dst[2] = o.z; dst[3] = o.w; }
    } else {
        uint16_t* dst = (uint16_t*)p.out + at;
        const uint32_t x = paged_pack2<DT>(o.x, o.y), y = paged_pack2<DT>(o.z, o.w);
        if (p.wide_o) *(uint2*)dst = make_uint2(x, y);
        else { dst[0] = (uint16_t)x; dst[1] = (uint16_t)(x >> 16); dst[2] = (uint16_t)y; dst[3] = (uint16_t)(y >> 16); }
    }
}

// The values that are not finite of the positions from `from` on that row r sees: where there are any, they are the row's element.  Among the step's rows they were taken as zero, since
// a weight of zero times them would reach rows that do not see them; those before the step were multiplied, but an infinity times a weight's second term, or a weight that is
// zero for being small, is a NaN.  (Element by element, since such values are rare.)
template <int ROWS, int UNIT, int DT>
__device__ __noinline__ void paged_unfinite_values(const PagedParams& p, const PagedBlock<ROWS, UNIT>& b, int r, int d, int from, float4& o) {
    const int step = paged_div(b.f0 + r, p.by_rep);
    float4 u = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int j = max(0, from); j < b.end; ++j) {
        if (j >= b.base && !paged_sees(p, b.first + step, step, j - b.base)) continue;
        const int row = b.row_of(p, j);
        if (row < 0) continue;
        float* x = &u.x;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float v = paged_float<DT>(p.v_data, (size_t)row * p.dim + d + e);
            if (!(fabsf(v) < INFINITY)) x[e] += v;
        }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if ((&u.x)[e] != 0.f) (&o.x)[e] = (&u.x)[e];
}
// A row's outputs behind its factor 1 / sum (zero: it sees nothing).  bad: values of the step's rows were taken as zero
template <int ROWS, int UNIT, int DT>
__device__ __forceinline__ void paged_settle(const PagedParams& p, const PagedBlock<ROWS, UNIT>& b, int r, int d, bool bad, float factor, float4& o) {
    if (factor == 0.f) o = make_float4(0.f, 0.f, 0.f, 0.f);
    else if (factor == factor) {                              // (a NaN among the scores is in all)
        const bool fine = fabsf(o.x) < INFINITY && fabsf(o.y) < INFINITY && fabsf(o.z) < INFINITY && fabsf(o.w) < INFINITY;
        if (bad || !fine) paged_unfinite_values<ROWS, UNIT, DT>(p, b, r, d, fine ? b.base : 0, o);
    }
}

// What a block says of its rows: references (log2) and sums, and whether a value of the step's rows that is not finite was taken as zero
template <int ROWS> struct PagedFold {
    float m[ROWS], l[ROWS];
    int bad;
};

// What a part's sums are multiplied by: without a maximum nothing was seen, or all was NaN, which the sum knows
__device__ __forceinline__ float paged_factor(float m, float l, float top) { return m == -INFINITY ? l - l : ex2(m - top); }

// The end of every kernel, whose block leaves its rows' sums at stage + r (DN + 4).  begin(), with all threads, when nothing of the shared memory is in use any more; join(), with
// all threads, when sums, references and so on are there.  Row r belongs to block r % splits of the cluster, which gets it from all blocks and joins them (fetching from the
// others as one goes waited for each load of a row and for a barrier before leaving: 7900 of a block's 17,000 cycles for a tree of 8 over 1000 keys; sent element by element 25
// cycles a store).  Or the rows go to memory for paged_join_kernel.
template <int ROWS, int UNIT, int DT, int DN> struct PagedOut {
    static constexpr int LD = DN + 4, BYTES = (2 * ROWS + PAGED_CLUSTER - 1) * LD * 4;
    const PagedParams& p;
    const PagedBlock<ROWS, UNIT>& b;
    const PagedFold<ROWS>& f;
    float* const stage;
    __device__ __forceinline__ PagedOut(const PagedParams& p_, const PagedBlock<ROWS, UNIT>& b_, const PagedFold<ROWS>& f_, float* stage_) : p(p_), b(b_), f(f_), stage(stage_) {}
    __device__ __forceinline__ void begin() {
        __syncthreads();
        if (p.splits > 1 && !p.partial) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    }
    template <typename Then> __device__ __forceinline__ void join(Then then) {
        const int tid = (int)threadIdx.x, threads = (int)blockDim.x, lane = tid & 31, warps = threads >> 5, slots = paged_div(ROWS + p.splits - 1, p.by_splits);
        for (int r = tid; r < b.live; r += threads) *(float4*)(stage + r * LD + DN) = make_float4(f.m[r], f.l[r], f.bad ? 1.f : 0.f, 0.f);
        __syncthreads();
        then();                                    // the sums have been read
        float* room = stage;
        if (p.splits > 1) {
            room += ROWS * LD;
            float* const global = p.partial ? p.partial + ((size_t)(blockIdx.x * gridDim.y + blockIdx.y) * p.splits + b.split) * (ROWS * LD) : nullptr;
            if (!global) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
#pragma unroll 1
            for (int r = tid >> 5; r < b.live; r += warps) {
                const int slot = paged_div(r, p.by_splits);
                const uint32_t to = paged_remote(smem_u32(room) + (uint32_t)((b.split * slots + slot) * LD) * 4u, global ? 0u : (uint32_t)(r - slot * p.splits));
#pragma unroll
                for (int c = 0; c < LD / 4; c += 32)
                    if (c + lane < LD / 4) {
                        const float4 v = *(const float4*)(stage + r * LD + 4 * (c + lane));
                        if (global) __stcg((float4*)(global + r * LD) + c + lane, v);
                        else asm volatile("st.shared::cluster.v4.f32 [%0], {%1,%2,%3,%4};" :: "r"(to + 16u * (uint32_t)(c + lane)), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
                    }
            }
            if (global) return;
            paged_cluster_sync();
        }
        // ---------------- rows split, split + splits, ...: a part's factor goes where its reference was; beside the first one's where the row goes (and whether values were
        // taken as zero), and what all is multiplied by
        const int mine = b.live > b.split ? paged_div(b.live - b.split + p.splits - 1, p.by_splits) : 0, ld = slots * LD;
        for (int slot = tid; slot < mine; slot += threads) {
            const int x = b.f0 + b.split + slot * p.splits, i = paged_div(x, p.by_rep), tok = b.first + i, h = b.head * p.rep + x - i * p.rep;
            float* const tail = room + slot * LD + DN;
            float top = -INFINITY, sum = 0.f, bad = 0.f;
            for (int s0 = 0; s0 < p.splits; s0 += 4) {
                float m[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) m[u] = s0 + u < p.splits ? tail[(s0 + u) * ld] : -INFINITY;
#pragma unroll
                for (int u = 0; u < 4; ++u) top = fmaxf(top, m[u]);
            }
            for (int s0 = 0; s0 < p.splits; s0 += 4) {
                float4 v[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) v[u] = s0 + u < p.splits ? *(const float4*)(tail + (s0 + u) * ld) : make_float4(-INFINITY, 0.f, 0.f, 0.f);
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const float w = paged_factor(v[u].x, v[u].y, top);
                    sum = fmaf(v[u].y, w, sum);
                    bad += v[u].z;
                    if (s0 + u < p.splits) tail[(s0 + u) * ld] = w;
                }
            }
            const bool any = sum > 0.f || sum != sum, there = tok >= 0 && tok < p.tokens;
            tail[1] = __int_as_float(there ? tok : -1);
            tail[2] = __int_as_float(bad != 0.f ? ~h : h);
            tail[3] = any ? 1.f / sum : 0.f;
            if (p.lse && there) p.lse[(size_t)tok * p.heads + h] = any ? (top + log2f(sum)) * PAGED_LN2 : -INFINITY;
        }
        __syncthreads();
#pragma unroll 2
        for (int i = tid; i < mine * (DN / 4); i += threads) {
            const int slot = i / (DN / 4), d = (i - slot * (DN / 4)) * 4;
            const float* const from = room + slot * LD;
            const float4 t = *(const float4*)(from + DN), first = *(const float4*)(from + d);
            const int tok = __float_as_int(t.y), where = __float_as_int(t.z), h = where < 0 ? ~where : where;
            if (d >= p.dim || tok < 0) continue;
            float4 o = make_float4(t.x * first.x, t.x * first.y, t.x * first.z, t.x * first.w);
#pragma unroll 4
            for (int s = 1; s < p.splits; ++s) {
                const float w = from[s * ld + DN];
                const float4 v = *(const float4*)(from + s * ld + d);
                o.x = fmaf(w, v.x, o.x); o.y = fmaf(w, v.y, o.y); o.z = fmaf(w, v.z, o.z); o.w = fmaf(w, v.w, o.w);
            }
            o.x *= t.w; o.y *= t.w; o.z *= t.w; o.w *= t.w;
            paged_settle<ROWS, UNIT, DT>(p, b, b.split + slot * p.splits, d, where < 0, t.w, o);
            paged_put<DT>(p, (size_t)tok * p.o_ld + (size_t)h * p.dim + d, o);
        }
    }
};

// What blocks that are no cluster have left becomes one: a warp a row
template <int ROWS, int UNIT, int DT, int DN>
__global__ void __launch_bounds__(256) paged_join_kernel(const __grid_constant__ PagedParams p) {
    const PagedBlock<ROWS, UNIT> b(p, (int)blockIdx.x, (int)blockIdx.y, 0);          // what the kernel before has read as well: it is there
    const int r = (int)blockIdx.z * 8 + (int)(threadIdx.x >> 5);
    griddep_wait();
    griddep_launch();
    if (r >= b.live) return;
    constexpr int LD = DN + 4, STEP = ROWS * LD;
    const int lane = (int)threadIdx.x & 31, x = b.f0 + r, i = paged_div(x, p.by_rep), tok = b.first + i, h = b.head * p.rep + x - i * p.rep;
    if (tok < 0 || tok >= p.tokens) return;
    const float* const from = p.partial + ((size_t)(blockIdx.x * gridDim.y + blockIdx.y) * p.splits * ROWS + r) * LD;
    float4 v[8];                                                          // eight parts on their way, the first ones beside the references
    auto load = [&](int d, int s0) {
#pragma unroll
        for (int u = 0; u < 8; ++u) v[u] = d < p.dim && s0 + u < p.splits ? __ldcg((const float4*)(from + (size_t)(s0 + u) * STEP + d)) : make_float4(0.f, 0.f, 0.f, 0.f);
    };
    const float4 tail = lane < p.splits ? __ldcg((const float4*)(from + (size_t)lane * STEP + DN)) : make_float4(-INFINITY, 0.f, 0.f, 0.f);       // lane s knows part s
    load(4 * lane, 0);
    const float top = warp_max(tail.x);
    float w = paged_factor(tail.x, tail.y, top);
    const float sum = warp_sum(tail.y * w);
    const bool bad = __any_sync(0xffffffffu, tail.z != 0.f), any = sum > 0.f || sum != sum;
    const float factor = any ? 1.f / sum : 0.f;
    w *= factor;
    if (lane == 0 && p.lse) p.lse[(size_t)tok * p.heads + h] = any ? (top + log2f(sum)) * PAGED_LN2 : -INFINITY;
#pragma unroll
    for (int d = 4 * lane; d < (DN + 127) / 128 * 128; d += 128) {
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
        for (int s0 = 0; s0 < p.splits; s0 += 8) {
            if (d >= 128 || s0 > 0) load(d, s0);
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const float y = __shfl_sync(0xffffffffu, w, (s0 + u) & 31);
                o.x = fmaf(y, v[u].x, o.x); o.y = fmaf(y, v[u].y, o.y); o.z = fmaf(y, v[u].z, o.z); o.w = fmaf(y, v[u].w, o.w);
            }
        }
        if (d >= p.dim) continue;
        paged_settle<ROWS, UNIT, DT>(p, b, r, d, bad, factor, o);
        paged_put<DT>(p, (size_t)tok * p.o_ld + (size_t)h * p.dim + d, o);
    }
}

// The launch of an attention kernel with the split that it takes, and of the join behind blocks that are no cluster
template <int ROWS, int UNIT, int DT, int DN, typename Launch>
int paged_launch(PagedParams p, PagedSplit split, cudaStream_t st, Launch launch) {
    p.splits = split.splits;
    p.by_splits = paged_divisor(p.splits);
    const dim3 grid((unsigned)(p.seqs * p.tiles), p.kv_heads, p.splits);
    void* ws = nullptr;
    if (split.apart) {
        if (int rc = scratch_alloc(&ws, (size_t)grid.x * grid.y * grid.z * ROWS * (DN + 4) * 4, st)) return rc;
        p.partial = (float*)ws;
    }
    cudaError_t e = launch(p, grid, split.apart);
    if (e == cudaSuccess && ws) {
        const long long most = (long long)p.max_rows * p.rep;
        e = launch_waiting(paged_join_kernel<ROWS, UNIT, DT, DN>, dim3(grid.x, grid.y, (unsigned)((most < ROWS ? most : ROWS) + 7) / 8), dim3(256), 0, st, p);
    }
    if (int rc = scratch_free(ws, st)) return rc;
    PGK_CUDA(e);
    return 0;
}

#endif  // __CUDACC__

}  // namespace pgk
