// paged_tc.cu -- attention of many rows a sequence (trees of drafts, portions of prompts) over 16-bit pages on tcgen05; the mathematics of paged_few.cu.
//
// A block has 128 (row, head) rows and walks over tiles of 128 keys:
//   * one warp fetches tiles of K and V by turns into a ring of six, by TMA in pieces of as many positions as divide a page;
//   * one thread issues S = Q K^T, queries in tensor memory, and O += P V.  Products run in the order in which they were issued, so that the scores of tile i + 2 may
//     follow the product that reads the weights of tile i in their place;
//   * four warps, a lane a row, have the even tiles, four the odd ones: the maxima of one are looked for while the other's weights are formed.  A row's reference, which
//     both share, moves when its maximum has grown by 2^8; it passes from tile to tile before the weights are formed.  A weight is rounded to the cache's type once:
//     outputs are off by 1.4 times what their own rounding makes.  (Two terms, half as many products again, leave only that: 8 x 64 rows over 4100 keys 49.6 -> 61 us.)
//   * only tiles that hold the step's rows, or the context's end, look at masks.  What lies behind the end is zeroed in V by the copying warp, and values of the step's
//     rows that are not finite are taken as zero there (a weight of zero times them would reach rows that do not see them) and added in the end.
// Bound by the copies: a SM takes in about 32 bytes a clock, 64 KB of a tile a microsecond, whatever the others do; its products and exponentials need half of that.  (256 rows
// a block, two sets of rows over the same tiles, halves the copies, but has room for one tile of scores a set: 3500 cycles for what are 2 x 2000 here, and a longer way in and
// out: 8 x 64 rows over 4100 keys 54 us where this took 47; it is 49.6 since scores of any size have weights, see paged_reference.)
// Blocks of a cluster share a sequence's keys.
#include "paged.cuh"
#include "tc_common.cuh"
#include "tma.cuh"
#include "../../include/pgk_b200.h"

namespace pgk {

namespace {

constexpr int T_ROWS = 128, T_KEYS = 128, T_SOFT = 8, T_THREADS = (T_SOFT + 2) * 32, T_SLOTS = 6;
constexpr uint32_t T_CHUNK = T_KEYS * 128;                         // 64 elements of 128 keys
constexpr uint32_t T_O = 0, T_Q = 128, T_S = 256;                  // TMEM columns: outputs, queries, two tiles of scores

struct Copies {
    int bp;                  // positions a copy, a power of two that divides the page
    int rows;                // of the cache: coordinates from here on read zeros
    int* err;
};

// C: 64-element chunks of a head
template <int C> struct Tile {
    static constexpr int DN = 64 * C;
    static constexpr uint32_t BYTES = C * T_CHUNK;
    // Half of a SM's shared memory at least: a block takes all of tensor memory, and two of unlike kernels on a SM, each of a cluster whose others wait for tensor memory
    // on the other's SMs, would wait for ever.
    static constexpr int RING = T_SLOTS * (int)BYTES, FOLD = (2 * T_ROWS + PAGED_CLUSTER - 1) * (DN + 4) * 4, HALF = 116 * 1024, MOST = RING > FOLD ? RING : FOLD,
                         SMEM = (MOST > HALF ? MOST : HALF) + 1024;
};

// 32 weights 2^(s scale + neg) to TMEM column `to`; their sum is of the unrounded ones
template <int DT>
__device__ __forceinline__ void weights32(const float* s, float scale, float zero, float neg, uint32_t to, uint64_t& l) {
    uint32_t y[16];
    const uint64_t scale2 = pair(scale, scale), zero2 = pair(zero, zero), neg2 = pair(neg, neg);
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        float a, b;
        unpair(add2(fma2(pair(s[2 * e], s[2 * e + 1]), scale2, zero2), neg2), a, b);
        a = ex2(a);
        b = ex2(b);
        l = add2(l, pair(a, b));
        y[e] = paged_weights2<DT>(a, b);
    }
    __syncwarp();
    tmem_st16u(to, y);
}

template <int C, int DT>
__global__ void __launch_bounds__(T_THREADS, 1) paged_tc_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                                                                const __grid_constant__ PagedParams p, const __grid_constant__ Copies cp) {
    using X = Tile<C>;
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ __align__(8) uint64_t full[T_SLOTS], empty[T_SLOTS], land, sfull[2], pready[2], pvdone[2];
    __shared__ uint32_t tmem_base_s;
    __shared__ float refs[2][T_ROWS], half_m[2][T_ROWS], half_l[2][T_ROWS];
    __shared__ PagedFold<T_ROWS> f;
    __shared__ int missing;
    int* const err = cp.err;
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), D = p.dim;
    const uint32_t ring = (smem_u32(smem) + 1023u) & ~1023u;

    if (warp == T_SOFT) tmem_alloc(&tmem_base_s, 512);
    if (tid == 0) {
        for (int s = 0; s < T_SLOTS; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
        mbar_init(&land, 1);
        for (int g = 0; g < 2; ++g) { mbar_init(&sfull[g], 1); mbar_init(&pready[g], 4); mbar_init(&pvdone[g], 1); }
        mbar_fence_init();
        missing = f.bad = 0;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_base_s;
    griddep_wait();
    griddep_launch();

    const PagedBlock<T_ROWS, T_KEYS> b(p, (int)blockIdx.x, (int)blockIdx.y, (int)blockIdx.z);
    const int n = b.uend - b.ubeg, steps = (D + 15) / 16;
    const int quad = warp & 3, side = (warp >> 2) & 1, row = quad * 32 + lane;
    const int step_row = paged_div(b.f0 + row, p.by_rep), tok = b.first + step_row;
    const bool live = warp < T_SOFT && row < b.live && tok >= 0 && tok < p.tokens;

    // Queries, zeros behind the head's end: rows as they lie through the ring's last place, which the copying warp has not come to, to tensor memory, a lane a row
    if (warp < T_SOFT) {
        const int last = min(b.end, b.uend * T_KEYS);
        int j = b.ubeg * T_KEYS + cp.bp * tid;
        const int page = j < last ? __ldcg(b.table + paged_div(j, p.by_page)) : 0;    // looked at behind the queries
        const uint32_t qs = ring + (T_SLOTS - 1) * X::BYTES;
#pragma unroll
        for (int i = tid; i < T_ROWS * C * 8; i += T_SOFT * 32) {
            const int r = i / (C * 8), u = i - r * (C * 8), x = b.f0 + r, step = paged_div(x, p.by_rep), t = b.first + step;
            uint4 v = make_uint4(0, 0, 0, 0);
            if (r < b.live && u * 8 < D && t >= 0 && t < p.tokens) {
                const uint16_t* const src = (const uint16_t*)p.q + (size_t)t * p.q_ld + (size_t)(b.head * p.rep + x - step * p.rep) * D + u * 8;
                if (p.wide_q) v = ld_act16(src);
                else {
                    uint32_t w[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) w[e] = (uint32_t)ld_act2(src + 2 * e) | (uint32_t)ld_act2(src + 2 * e + 1) << 16;
                    v = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" :: "r"(qs + (uint32_t)r * (C * 128u) + (uint32_t)((u ^ (r & 7)) << 4)), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
        }
        bool gone = (unsigned)page >= (unsigned)p.pages;
        for (j += cp.bp * T_SOFT * 32; j < last; j += cp.bp * T_SOFT * 32) gone |= b.row_of(p, j) < 0;
        if (gone) missing = 1;
        __syncwarp();
        asm volatile("bar.sync 10, %0;" :: "n"(T_SOFT * 32) : "memory");
        uint32_t x[X::DN / 4];                     // a half of the row
#pragma unroll
        for (int i = 0; i < C * 4; ++i) {
            const uint32_t u = (uint32_t)(side * C * 4 + i);
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(x[4 * i]), "=r"(x[4 * i + 1]), "=r"(x[4 * i + 2]), "=r"(x[4 * i + 3])
                         : "r"(qs + (uint32_t)row * (C * 128u) + ((u ^ (uint32_t)(row & 7)) << 4)) : "memory");
        }
        __syncwarp();
#pragma unroll
        for (int c = 0; c < C; ++c) tmem_st16u(tmem + ((uint32_t)(quad * 32) << 16) + T_Q + (uint32_t)(side * C + c) * 16u, *(uint32_t (*)[16])(x + 16 * c));
        tmem_st_wait();
        fence_proxy_async();                       // the place goes back to the copies
        tc_fence_before();
    }
    // The copying warp comes when all other places are on their way.  (That the rest waits for it, instead of it alone for the queries, took 46.5 us where 50 went by: 512 rows of
    // eight sequences over 4100 keys.)
    auto queries_there = [] {
        __syncwarp();
        asm volatile("bar.sync 9, %0;" :: "n"(T_THREADS) : "memory");
        tc_fence_after();
    };
    if (warp <= T_SOFT) queries_there();

    if (warp == T_SOFT) {
        // ---------------- MMAs, from one thread.  The ring has K 0, K 1, V 0, K 2, V 1, ...
        if (elect_one()) {
            constexpr uint32_t types = DT == 1 ? ~((1u << 7) | (1u << 10)) : ~0u;        // both operands float16, or both bfloat16
            constexpr uint32_t id_s = umma_idesc_bf16(T_KEYS) & types, id_o = (umma_idesc_bf16(X::DN) | (1u << 16)) & types;   // values: the elements are contiguous
            RingPos at;
            bool ok = true;
            auto scores = [&](int i) {             // where the weights of tile i - 2 were
                ok = ok && bar_wait(err, smem_u32(&full[at.s]), at.round);
                if (!ok) return;
                tc_fence_after();
                const uint64_t d = desc_sw128(ring + at.s * X::BYTES);
                const uint32_t to = tmem + T_S + (uint32_t)(i & 1) * 128u;
#pragma unroll
                for (int k = 0; k < X::DN / 16; ++k)
                    if (k < steps)
                        umma_bf16_ta(to, tmem + T_Q + (uint32_t)k * 8u, d + (uint64_t)((k >> 2) * (T_CHUNK / 16) + (k & 3) * 2), id_s, k ? 1u : 0u);
                umma_commit(&sfull[i & 1]);
                umma_commit(&empty[at.s]);
                at.next(T_SLOTS);
            };
            if (n > 0) scores(0);
            if (n > 1) scores(1);
            int made = 0;
            for (int i = 0; ok && i < n; ++i) {
                ok = bar_wait(err, smem_u32(&full[at.s]), at.round) && bar_wait(err, smem_u32(&pready[i & 1]), (uint32_t)(i >> 1) & 1u);
                if (!ok) break;
                tc_fence_after();
                const uint64_t d = desc_mn_sw128(ring + at.s * X::BYTES, T_CHUNK);
                const uint32_t from = tmem + T_S + (uint32_t)(i & 1) * 128u;
#pragma unroll
                for (int k = 0; k < T_KEYS / 16; ++k)              // 16 keys: 2048 bytes of V
                    umma_bf16_ta(tmem + T_O, from + (uint32_t)(k >> 2) * 64u + (uint32_t)(k & 3) * 8u, d + (uint64_t)(k * 128), id_o, (i | k) ? 1u : 0u);
                umma_commit(&pvdone[i & 1]);
                umma_commit(&empty[at.s]);
                at.next(T_SLOTS);
                made = i + 1;
                if (i + 2 < n) scores(i + 2);
            }
            if (made) bar_wait(err, smem_u32(&pvdone[(made - 1) & 1]), (uint32_t)((made - 1) >> 1) & 1u);
        }
        __syncwarp();
    } else if (warp == T_SOFT + 1) {
        // ---------------- copies: lane l has piece l of a tile
        const int pieces = T_KEYS / cp.bp, from = min(b.base, b.end);      // from `from` on values are looked at
        bool ok = true, bad = false, met = false;
        int issued = 0;
        uint32_t landed = 0;
        RingPos at;
        auto where = [&](int i) {                  // no such position or page: zeros
            const int r = lane < pieces && i < n ? b.row_of(p, (b.ubeg + i) * T_KEYS + lane * cp.bp) : -1;
            return r < 0 ? cp.rows : r;
        };
        auto fetch = [&](const CUtensorMap* map, int i, int at_row, bool fix) {
            if (issued == T_SLOTS - 1 && !met) {
                met = true;
                queries_there();
            }
            ok = ok && __all_sync(0xffffffffu, bar_wait(err, smem_u32(&empty[at.s]), at.round ^ 1u));
            if (!ok) return;
            const uint32_t bar = smem_u32(fix ? &land : &full[at.s]), tile = ring + at.s * X::BYTES;
            if (lane == 0) mbar_expect_tx(bar, X::BYTES);
            __syncwarp();
            if (lane < pieces)
#pragma unroll
                for (int c = 0; c < C; ++c) tma_load_2d(tile + (uint32_t)c * T_CHUNK + (uint32_t)(lane * cp.bp) * 128u, map, c * 64, at_row, bar);
            ++issued;
            if (fix) {
                ok = __all_sync(0xffffffffu, bar_wait(err, smem_u32(&land), landed));
                landed ^= 1u;
                if (!ok) return;
                bad |= paged_fix_values<DT>(tile, C, T_CHUNK, (b.ubeg + i) * T_KEYS, from, b.end, cp.bp, lane);
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(&full[at.s]);
            }
            at.next(T_SLOTS);
        };
        int r0 = where(0), r1 = where(1);
        if (n > 0) fetch(&kmap, 0, r0, false);
        if (ok && n > 1) fetch(&kmap, 1, r1, false);
        for (int i = 0; ok && i < n; ++i) {
            const int r2 = where(i + 2);
            fetch(&vmap, i, r0, (b.ubeg + i + 1) * T_KEYS > from);
            if (ok && i + 2 < n) fetch(&kmap, i + 2, r2, false);
            r0 = r1;
            r1 = r2;
        }
        if (!met) queries_there();
        if (bad) f.bad = 1;
        if (lane == 0)
            for (int j = max(0, issued - T_SLOTS); j < issued; ++j)       // whoever gave up: do not leave with copies in flight
                bar_wait(err, smem_u32(&full[j % T_SLOTS]), (uint32_t)(j / T_SLOTS) & 1u);
        __syncwarp();
    } else {
        // ---------------- weights: tiles of the warp's side, lane = row
        const uint32_t lanes = tmem + ((uint32_t)(quad * 32) << 16), at = lanes + T_S + (uint32_t)side * 128u;
        const int clean = missing ? 0 : min(b.base, b.end);               // keys before this one are seen by all
        float m = -INFINITY, l = 0.f;                                     // the reference of this side's last tile, and its share of the sum
        bool ok = true;
        for (int i = side; i < n; i += 2) {
            const int j0 = (b.ubeg + i) * T_KEYS;
            const bool edge = j0 + T_KEYS > clean;
            uint32_t see[4];
            if (edge) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int j = j0 + 32 * e;
                    see[e] = live && j < b.end ? paged_window(p, tok, step_row, j - b.base) : 0u;
                    if (b.end - j < 32) see[e] &= b.end > j ? (1u << (b.end - j)) - 1u : 0u;
                    if (missing)
                        for (int x = 0; x < 32; x += 8)                   // a copy has 8 positions at least
                            if (b.row_of(p, j + x) < 0) see[e] &= ~(0xffu << x);
                }
            }
            ok = ok && __all_sync(0xffffffffu, bar_wait(err, smem_u32(&sfull[side]), (uint32_t)(i >> 1) & 1u));
            __syncwarp();
            tc_fence_after();
            float s[64];
            auto load = [&](int half) {                                   // half of the tile's scores, -infinity where the row does not see
#pragma unroll
                for (int c = 0; c < 64; c += 16) tmem_ld16_async(at + (uint32_t)(half * 64 + c), *(float (*)[16])(s + c));
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                for (int c = 0; c < 64; c += 16) tmem_pass(*(float (*)[16])(s + c));
                if (edge) {
                    const uint32_t lo = half ? see[2] : see[0], hi = half ? see[3] : see[1];
#pragma unroll
                    for (int e = 0; e < 64; ++e)
                        if (!(((e < 32 ? lo : hi) >> (e & 31)) & 1u)) s[e] = -INFINITY;
                }
            };
            float t[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int half = 0; half < 2; ++half) {                        // the second one stays
                load(half);
#pragma unroll
                for (int e = 0; e < 64; ++e) t[e & 3] = fmaxf(t[e & 3], s[e]);
            }
            const float top = paged_reference<DT>(fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3])) * p.scale_log2);
            // the reference passes from the other side's warp, which has the tile before, and on to it
            float was = -INFINITY;
            if (i > 0) {
                asm volatile("bar.sync %0, 64;" :: "r"(1 + 2 * quad + (side ^ 1)) : "memory");
                was = refs[side ^ 1][row];
            }
            const float now = top > was + PAGED_LAZY ? top : was;         // (also the first finite maximum)
            refs[side][row] = now;
            __syncwarp();
            if (i + 1 < n) asm volatile("bar.arrive %0, 64;" :: "r"(1 + 2 * quad + side) : "memory");
            if (__any_sync(0xffffffffu, now != m)) {
                if (now != m) l *= m == -INFINITY ? 0.f : exp2f(m - now);
                m = now;
            }
            if (i > 0 && __any_sync(0xffffffffu, now != was)) {
                const float fix = now == was ? 1.f : (was == -INFINITY ? 0.f : exp2f(was - now));
                ok = ok && __all_sync(0xffffffffu, bar_wait(err, smem_u32(&pvdone[side ^ 1]), (uint32_t)((i - 1) >> 1) & 1u));
                __syncwarp();
                tc_fence_after();
#pragma unroll 1
                for (int c = 0; c < X::DN; c += 16) {
                    float o[16];
                    const uint32_t to = lanes + T_O + (uint32_t)c;
                    tmem_ld16(to, o);
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[e] *= fix;
                    tmem_st16(to, o);
                }
            }
            const float neg = paged_neg(now);
            uint64_t l2 = pair(0.f, 0.f);
            weights32<DT>(s, p.scale_log2, p.zero, neg, at + 64u, l2);    // each half to where its scores were
            weights32<DT>(s + 32, p.scale_log2, p.zero, neg, at + 80u, l2);
            load(0);
            weights32<DT>(s, p.scale_log2, p.zero, neg, at, l2);
            weights32<DT>(s + 32, p.scale_log2, p.zero, neg, at + 16u, l2);
            float la, lb;
            unpair(l2, la, lb);
            l += la + lb;
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&pready[side]);
        }
        half_m[side][row] = m;
        half_l[side][row] = l;
    }
    PagedOut<T_ROWS, T_KEYS, DT, X::DN> out(p, b, f, (float*)smem);
    out.begin();                                   // nobody's tile is read or written any more
    tc_fence_after();
    if (tid < T_ROWS) {                            // references only grow: the larger one is the outputs'
        const float m0 = half_m[0][tid], m1 = half_m[1][tid], l0 = half_l[0][tid], l1 = half_l[1][tid], m = fmaxf(m0, m1);
        f.m[tid] = m;
        f.l[tid] = (m0 == -INFINITY ? l0 : l0 * exp2f(m0 - m)) + (m1 == -INFINITY ? l1 : l1 * exp2f(m1 - m));
    }
    if (warp < T_SOFT) {
        float* const to = out.stage + row * out.LD;
#pragma unroll 1
        for (int c = side * (X::DN / 2); c < (side + 1) * (X::DN / 2); c += 16) {
            float o[16];
            if (n > 0) tmem_ld16(tmem + ((uint32_t)(quad * 32) << 16) + T_O + (uint32_t)c, o);
            else {
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] = 0.f;
            }
#pragma unroll
            for (int e = 0; e < 16; e += 4) *(float4*)(to + c + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
            __syncwarp();
        }
    }
    tc_fence_before();
    __syncthreads();
    out.join([&] {
        if (warp == T_SOFT) tmem_dealloc(tmem, 512);
    });
}

template <int C, int DT>
int launch_tiles(PagedParams p, cudaStream_t st) {
    using X = Tile<C>;
    static PagedOccupancy fits;
    const auto kernel = paged_tc_kernel<C, DT>;
    PGK_CUDA(fits.once([&](int* at_once) {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, X::SMEM);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        for (int i = 1; e == cudaSuccess && i <= PAGED_CLUSTER; ++i) e = clusters_at_once(&at_once[i], kernel, T_THREADS, X::SMEM, i);
        return e;
    }));
    Copies cp = {};
    cp.bp = p.page_size & -p.page_size;
    if (cp.bp > T_KEYS) cp.bp = T_KEYS;
    cp.rows = p.pages * p.kv_heads * p.page_size;
    cp.err = wait_word(kWaitPaged);
    PGK_REQUIRE(cp.err, "paged_attention failed: no pinned host memory");
    CUtensorMap kmap{}, vmap{};
    PGK_REQUIRE(tma_map_bf16_2d(&kmap, p.k_data, (uint64_t)p.dim, (uint64_t)cp.rows, (uint64_t)p.dim * 2, 64, (uint32_t)cp.bp) &&
                    tma_map_bf16_2d(&vmap, p.v_data, (uint64_t)p.dim, (uint64_t)cp.rows, (uint64_t)p.dim * 2, 64, (uint32_t)cp.bp),
                "paged_attention failed: no tensor map of %d rows of %d elements", cp.rows, p.dim);
    p.tiles = (int)(((long long)p.max_rows * p.rep + T_ROWS - 1) / T_ROWS);
    return paged_launch<T_ROWS, T_KEYS, DT, X::DN>(p, paged_split(p, T_KEYS, fits.at_once, PAGED_CLUSTER, 4), st, [&](const PagedParams& q, dim3 grid, bool apart) {
        return launch_clusters(kernel, grid, apart, T_THREADS, (size_t)X::SMEM, st, kmap, vmap, q, cp);
    });
}

}  // namespace

// More rows than a block of the other kernel has; copies of eight positions and more, 16 bytes at a time
bool paged_tc_serves(const PagedParams& p, int dtype) {
    return dtype != 0 && p.dim >= 64 && p.dim <= 128 && p.page_size % 8 == 0 && (long long)p.max_rows * p.rep > 32 && tma_encode_fn() != nullptr;
}
int paged_tc(const PagedParams& p, int dtype, cudaStream_t st) {
    if (p.dim == 64) return dtype == 1 ? launch_tiles<1, 1>(p, st) : launch_tiles<1, 2>(p, st);
    return dtype == 1 ? launch_tiles<2, 1>(p, st) : launch_tiles<2, 2>(p, st);
}

}  // namespace pgk
