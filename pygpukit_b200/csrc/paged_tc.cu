// paged_tc.cu -- attention of many rows a sequence (trees of drafts, portions of prompts) over 16-bit pages on tcgen05; the mathematics of paged_few.cu.
//
// A block has 128 (row, head) rows and walks over tiles of 128 keys, three of K and V in shared memory, fetched by TMA in pieces of as many positions as divide a page:
//   * one thread issues S = Q K^T, queries in tensor memory, and O += P V, the scores of tile i + 1 before the weights of tile i are waited for;
//   * eight warps, a lane a row and two warps a row, turn scores into weights, rounded to the cache's type once, in the scores' place; a row's reference moves when
//     its maximum has grown by 2^8;
//   * only tiles that hold the step's rows, or the context's end, look at masks.  What lies behind the end is zeroed in V by the copying warp, and values of the step's
//     rows that are not finite are taken as zero there (a weight of zero times them would reach rows that do not see them) and added in the end.
// Bound by the chain of a row's warps: of a tile the products take 512 cycles, the exponentials 1024 of the special unit.
// Blocks of a cluster share a sequence's keys and fold through distributed shared memory.
#include "paged.cuh"
#include "tc_common.cuh"
#include "tma.cuh"
#include "../../include/pgk_b200.h"

namespace pgk {

namespace {

constexpr int T_ROWS = 128, T_KEYS = 128, T_SOFT = 8, T_THREADS = (T_SOFT + 2) * 32, T_STAGES = 3;
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
    static constexpr int RING = 2 * T_STAGES * (int)BYTES, FOLD = T_ROWS * (DN + 4) * 4, HALF = 116 * 1024, MOST = RING > FOLD ? RING : FOLD,
                         SMEM = (MOST > HALF ? MOST : HALF) + 1024;
};

__device__ __forceinline__ bool all_wait(int* err, uint64_t* bar, uint32_t parity) {
    const bool ok = bar_wait(err, smem_u32(bar), parity);
    return __all_sync(0xffffffffu, ok);
}
// 32 weights 2^(s scale + neg) to TMEM column `to`; their sum is of the unrounded ones
template <int DT>
__device__ __forceinline__ void weights32(const float* s, float scale, float neg, uint32_t to, uint64_t& l) {
    uint32_t y[16];
    const uint64_t scale2 = pair(scale, scale), neg2 = pair(neg, neg);
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        float a, b;
        unpair(fma2(pair(s[2 * e], s[2 * e + 1]), scale2, neg2), a, b);
        a = ex2(a);
        b = ex2(b);
        l = add2(l, pair(a, b));
        y[e] = paged_pack2<DT>(a, b);
    }
    __syncwarp();
    tmem_st16u(to, y);
}

template <int C, int DT>
__global__ void __launch_bounds__(T_THREADS, 1) paged_tc_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                                                                const __grid_constant__ PagedParams p, const __grid_constant__ Copies cp) {
    using X = Tile<C>;
    constexpr float TOP = DT == 1 ? 6.f : 0.f;                     // as in paged_few.cu
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ __align__(8) uint64_t full[T_STAGES], empty[T_STAGES], land, sfull[2], pready[2], pvdone;
    __shared__ uint32_t tmem_base_s;
    __shared__ float wmax[2][2][T_ROWS];
    __shared__ PagedFold<T_ROWS> f;
    __shared__ int missing;
    int* const err = cp.err;
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), D = p.dim;
    const uint32_t ks = (smem_u32(smem) + 1023u) & ~1023u, vs = ks + T_STAGES * X::BYTES;

    if (warp == T_SOFT) tmem_alloc(&tmem_base_s, 512);
    if (tid == 0) {
        for (int s = 0; s < T_STAGES; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
        mbar_init(&land, 1);
        mbar_init(&sfull[0], 1); mbar_init(&sfull[1], 1);
        mbar_init(&pready[0], T_SOFT); mbar_init(&pready[1], T_SOFT); mbar_init(&pvdone, 1);
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
    const int quad = warp & 3, half = (warp >> 2) & 1, row = quad * 32 + lane;
    const int step_row = (b.f0 + row) / p.rep, tok = b.first + step_row;
    const bool live = warp < T_SOFT && row < b.live && tok >= 0 && tok < p.tokens;

    if (warp < 4) {                                // queries to tensor memory, zeros behind the head's end
        const uint16_t* const src = (const uint16_t*)p.q + (live ? (size_t)tok * p.q_ld + (size_t)(b.head * p.rep + b.f0 + row - step_row * p.rep) * D : 0);
        uint32_t x[X::DN / 32][16];
#pragma unroll
        for (int c = 0; c < X::DN / 32; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint4 v = make_uint4(0, 0, 0, 0);
                const int d = 32 * c + 8 * i;
                if (live && d < D) {
                    if (p.wide_q) v = ld_act16(src + d);
                    else {
                        uint32_t w[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) w[e] = (uint32_t)ld_act2(src + d + 2 * e) | (uint32_t)ld_act2(src + d + 2 * e + 1) << 16;
                        v = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
                x[c][4 * i] = v.x; x[c][4 * i + 1] = v.y; x[c][4 * i + 2] = v.z; x[c][4 * i + 3] = v.w;
            }
        __syncwarp();
#pragma unroll
        for (int c = 0; c < X::DN / 32; ++c) tmem_st16u(tmem + ((uint32_t)(quad * 32) << 16) + T_Q + (uint32_t)c * 16u, x[c]);
        tmem_st_wait();
    } else if (warp <= T_SOFT) {
        const int last = min(b.end, b.uend * T_KEYS);
        bool gone = false;
        for (int j = b.ubeg * T_KEYS + cp.bp * (tid - 128); j < last; j += cp.bp * (T_SOFT + 1 - 4) * 32) gone |= b.row_of(p, j) < 0;
        if (gone) missing = 1;
    }
    if (warp <= T_SOFT) {                          // the copies are on their way meanwhile
        tc_fence_before();
        __syncwarp();
        asm volatile("bar.sync 5, %0;" :: "n"((T_SOFT + 1) * 32) : "memory");
        tc_fence_after();
    }

    if (warp == T_SOFT) {
        // ---------------- MMAs, from one thread
        if (elect_one()) {
            constexpr uint32_t types = DT == 1 ? ~((1u << 7) | (1u << 10)) : ~0u;        // both operands float16, or both bfloat16
            constexpr uint32_t id_s = umma_idesc_bf16(T_KEYS) & types, id_o = (umma_idesc_bf16(X::DN) | (1u << 16)) & types;   // values: the elements are contiguous
            const uint64_t kd = desc_sw128(ks), vd = desc_mn_sw128(vs, T_CHUNK);
            bool ok = true;
            auto scores = [&](int i) {             // where the weights of tile i - 2 were
                const int s = i % T_STAGES;
                ok = ok && bar_wait(err, smem_u32(&full[s]), (uint32_t)(i / T_STAGES) & 1u);
                if (!ok) return;
                tc_fence_after();
                const uint64_t d = kd + (uint64_t)(s * (X::BYTES / 16));
                const uint32_t to = tmem + T_S + (uint32_t)(i & 1) * 128u;
#pragma unroll
                for (int k = 0; k < X::DN / 16; ++k)
                    if (k < steps)
                        umma_bf16_ta(to, tmem + T_Q + (uint32_t)k * 8u, d + (uint64_t)((k >> 2) * (T_CHUNK / 16) + (k & 3) * 2), id_s, k ? 1u : 0u);
                umma_commit(&sfull[i & 1]);
            };
            if (n > 0) scores(0);
            int made = 0;
            for (int i = 0; ok && i < n; ++i) {
                const int s = i % T_STAGES;
                if (i > 0) ok = bar_wait(err, smem_u32(&pvdone), (uint32_t)((i - 1) & 1));
                if (ok && i + 1 < n) scores(i + 1);
                ok = ok && bar_wait(err, smem_u32(&pready[i & 1]), (uint32_t)(i >> 1) & 1u);
                if (!ok) break;
                tc_fence_after();
                const uint64_t d = vd + (uint64_t)(s * (X::BYTES / 16));
                const uint32_t at = tmem + T_S + (uint32_t)(i & 1) * 128u;
#pragma unroll
                for (int k = 0; k < T_KEYS / 16; ++k)              // 16 keys: 2048 bytes of V
                    umma_bf16_ta(tmem + T_O, at + (uint32_t)(k >> 2) * 64u + (uint32_t)(k & 3) * 8u, d + (uint64_t)(k * 128), id_o, (i | k) ? 1u : 0u);
                umma_commit(&pvdone);
                umma_commit(&empty[s]);
                made = i + 1;
            }
            if (made) bar_wait(err, smem_u32(&pvdone), (uint32_t)((made - 1) & 1));
        }
        __syncwarp();
    } else if (warp == T_SOFT + 1) {
        // ---------------- copies: lane l has piece l of a tile
        const int pieces = T_KEYS / cp.bp;
        bool ok = true, bad = false;
        int made = 0;
        uint32_t landed = 0;
        auto where = [&](int i) {                  // no such position or page: zeros
            const int r = lane < pieces && i < n ? b.row_of(p, (b.ubeg + i) * T_KEYS + lane * cp.bp) : -1;
            return r < 0 ? cp.rows : r;
        };
        int at = where(0);
        for (; made < n; ++made) {
            const int s = made % T_STAGES, j0 = (b.ubeg + made) * T_KEYS, next = where(made + 1);
            const int from = min(b.base, b.end);   // from here on values are looked at
            const bool fix = j0 + T_KEYS > from;
            ok = ok && all_wait(err, &empty[s], (((uint32_t)made / T_STAGES) & 1u) ^ 1u);
            if (!ok) break;
            const uint32_t bar = smem_u32(fix ? &land : &full[s]);
            if (lane == 0) mbar_expect_tx(bar, 2 * X::BYTES);
            __syncwarp();
            if (lane < pieces) {
                const uint32_t to = (uint32_t)s * X::BYTES + (uint32_t)(lane * cp.bp) * 128u;
#pragma unroll
                for (int c = 0; c < C; ++c) tma_load_2d(ks + to + (uint32_t)c * T_CHUNK, &kmap, c * 64, at, bar);
#pragma unroll
                for (int c = 0; c < C; ++c) tma_load_2d(vs + to + (uint32_t)c * T_CHUNK, &vmap, c * 64, at, bar);
            }
            if (fix) {
                ok = all_wait(err, &land, landed);
                landed ^= 1u;
                if (!ok) break;
                // values of the step's rows: is any not finite?  The largest exponent of a lane's says
                const int k0 = max(0, from - j0), k1 = min(T_KEYS, b.end - j0);
                const uint32_t tile = vs + (uint32_t)s * X::BYTES;
                auto unit = [&](uint32_t a, uint32_t (&x)[4]) {
                    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]) : "r"(a) : "memory");
                };
                auto put = [&](uint32_t a, const uint32_t (&x)[4]) {
                    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" :: "r"(a), "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]) : "memory");
                };
                uint32_t most = 0;
#pragma unroll 4
                for (int i = k0 * 8 + lane; i < k1 * 8; i += 32)
#pragma unroll
                    for (int c = 0; c < C; ++c) {
                        uint32_t x[4];
                        unit(tile + (uint32_t)c * T_CHUNK + (uint32_t)i * 16u, x);
#pragma unroll
                        for (int e = 0; e < 4; ++e) most = __vmaxu2(most, x[e] & 0x7fff7fffu);
                    }
                if (__any_sync(0xffffffffu, paged_unfinite<DT>(most) != 0)) {
                    bad = true;
                    for (int i = k0 * 8 + lane; i < k1 * 8; i += 32)
                        for (int c = 0; c < C; ++c) {
                            const uint32_t a = tile + (uint32_t)c * T_CHUNK + (uint32_t)i * 16u;
                            uint32_t x[4];
                            unit(a, x);
#pragma unroll
                            for (int e = 0; e < 4; ++e) x[e] &= ~paged_unfinite<DT>(x[e]);
                            put(a, x);
                        }
                }
                // what lies behind the end in the last copy (what was not copied is zeros)
                const uint32_t none[4] = {0, 0, 0, 0};
                for (int i = max(0, k1) * 8 + lane; i < min(T_KEYS, (max(0, k1) + cp.bp - 1) & ~(cp.bp - 1)) * 8; i += 32)
#pragma unroll
                    for (int c = 0; c < C; ++c) put(tile + (uint32_t)c * T_CHUNK + (uint32_t)i * 16u, none);
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(&full[s]);
            }
            at = next;
        }
        if (bad) f.bad = 1;
        if (lane == 0)
            for (int j = max(0, made - T_STAGES); j < made; ++j)          // whoever gave up: do not leave with copies in flight
                bar_wait(err, smem_u32(&full[j % T_STAGES]), (uint32_t)(j / T_STAGES) & 1u);
        __syncwarp();
    } else {
        // ---------------- weights
        const uint32_t lanes = tmem + ((uint32_t)(quad * 32) << 16);
        const int clean = missing ? 0 : min(b.base, b.end);               // keys before this one are seen by all
        float m = -INFINITY, l = 0.f;
        bool ok = true;
        for (int i = 0; i < n; ++i) {
            const uint32_t at = lanes + T_S + (uint32_t)(i & 1) * 128u + (uint32_t)(half * 64);
            const int j0 = (b.ubeg + i) * T_KEYS + half * 64;
            uint32_t see[2] = {0xffffffffu, 0xffffffffu};
            const bool edge = j0 + 64 > clean;
            if (edge) {
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const int j = j0 + 32 * u;
                    see[u] = live && j < b.end ? paged_window(p, tok, step_row, j - b.base) : 0u;
                    if (b.end - j < 32) see[u] &= b.end > j ? (1u << (b.end - j)) - 1u : 0u;
                    if (missing)
                        for (int e = 0; e < 32; e += 8)                   // a copy has 8 positions at least
                            if (b.row_of(p, j + e) < 0) see[u] &= ~(0xffu << e);
                }
            }
            ok = ok && all_wait(err, &sfull[i & 1], (uint32_t)((i >> 1) & 1));
            __syncwarp();
            tc_fence_after();
            float s[64], top = -INFINITY;
#pragma unroll
            for (int c = 0; c < 64; c += 16) tmem_ld16_async(at + (uint32_t)c, *(float (*)[16])(s + c));
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
            for (int c = 0; c < 64; c += 16) tmem_pass(*(float (*)[16])(s + c));
            if (edge) {
#pragma unroll
                for (int e = 0; e < 64; ++e)
                    if (!((see[e >> 5] >> (e & 31)) & 1u)) s[e] = -INFINITY;
            }
#pragma unroll
            for (int e = 0; e < 64; ++e) top = fmaxf(top, s[e]);
            top = top * p.scale_log2 - TOP;
            wmax[i & 1][half][row] = top;
            __syncwarp();
            asm volatile("bar.sync %0, 64;" :: "r"(1 + quad) : "memory");          // the row's two warps
            top = fmaxf(top, wmax[i & 1][half ^ 1][row]);
            const bool up = top > m + PAGED_LAZY;                 // (also the first finite maximum)
            if (__any_sync(0xffffffffu, up)) {                    // the same in both warps: each has half of the outputs
                const float fix = !up ? 1.f : (m == -INFINITY ? 0.f : exp2f(m - top));
                if (up) m = top;
                l *= fix;
                if (i > 0) {
                    ok = ok && all_wait(err, &pvdone, (uint32_t)((i - 1) & 1));
                    __syncwarp();
                    tc_fence_after();
#pragma unroll 1
                    for (int c = 0; c < X::DN / 2; c += 16) {
                        float o[16];
                        const uint32_t to = lanes + T_O + (uint32_t)(half * (X::DN / 2) + c);
                        tmem_ld16(to, o);
#pragma unroll
                        for (int e = 0; e < 16; ++e) o[e] *= fix;
                        tmem_st16(to, o);
                    }
                }
            }
            const float neg = paged_neg(m);
            uint64_t l2 = pair(0.f, 0.f);
            weights32<DT>(s, p.scale_log2, neg, at, l2);          // to where the warp's own scores were
            weights32<DT>(s + 32, p.scale_log2, neg, at + 16u, l2);
            float la, lb;
            unpair(l2, la, lb);
            l += la + lb;
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&pready[i & 1]);           // a barrier each: weights of two tiles may be ready before the first is looked for
        }
        asm volatile("bar.sync %0, 64;" :: "r"(1 + quad) : "memory");              // the last tile's maxima are read
        wmax[0][half][row] = l;
        __syncwarp();
        asm volatile("bar.sync %0, 64;" :: "r"(1 + quad) : "memory");
        if (half == 0) { f.m[row] = m; f.l[row] = wmax[0][0][row] + wmax[0][1][row]; }
    }
    __syncthreads();                               // nobody's tile is read or written any more
    tc_fence_after();
    float* const sums = (float*)smem;              // [128][DN + 4]
    if (warp < T_SOFT) {
#pragma unroll 1
        for (int c = half * (X::DN / 2); c < (half + 1) * (X::DN / 2); c += 16) {
            float o[16];
            if (n > 0) tmem_ld16(tmem + ((uint32_t)(quad * 32) << 16) + T_O + (uint32_t)c, o);
            else {
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] = 0.f;
            }
#pragma unroll
            for (int e = 0; e < 16; e += 4) *(float4*)(sums + (size_t)row * (X::DN + 4) + c + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
            __syncwarp();
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == T_SOFT) tmem_dealloc(tmem, 512);
    paged_fold<T_ROWS, T_KEYS, DT, X::DN>(p, b, sums, f);
}

template <int C, int DT>
int launch_tiles(PagedParams p, cudaStream_t st) {
    static bool configured = false;
    static int at_once[PAGED_CLUSTER + 1] = {};
    const auto kernel = paged_tc_kernel<C, DT>;
    if (!configured) {
        PGK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Tile<C>::SMEM));
        PGK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        for (int i = 1; i <= PAGED_CLUSTER; ++i) PGK_CUDA(clusters_at_once(&at_once[i], kernel, T_THREADS, Tile<C>::SMEM, i));
        configured = true;
    }
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
    p.splits = paged_clusters(p, T_KEYS, at_once, PAGED_CLUSTER, 4);
    PGK_CUDA(launch_clusters(kernel, dim3((unsigned)(p.seqs * p.tiles), p.kv_heads, p.splits), T_THREADS, (size_t)Tile<C>::SMEM, st, kmap, vmap, p, cp));
    return 0;
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
