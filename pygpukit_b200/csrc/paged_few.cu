// paged_few.cu -- attention of few rows a sequence over 16-bit pages: decoded tokens, small trees of drafts, and whatever the tiles of 128 rows of paged_tc.cu do not serve
// (heads above 128 elements, small pages).
//
// One pass over the keys with the running maximum and sum of a softmax, on tcgen05 with the keys as the products' 128 lanes: a block has NR = 16, 32 or 64 (row, head) rows,
// S^T[128 keys, NR] = K Q^T, and O^T[128 elements, 2 NR] += V^T P^T, so that few rows cost few columns and K and V are read from shared memory as TMA left them.  (With mma.sync
// and K and V in registers, 64 tokens over 8192 keys took 390 us, 550 instructions for 16 keys of a warp; with rows copied to shared memory one by one 455, 15 cycles a
// copy of 256 bytes.)
//   * one warp fetches tiles of K and V by turns into a ring, in pieces of as many positions as divide a page, four rows at a time where that is fewer than eight;
//   * one thread issues the products, the scores of tile i + 1 before the weights of tile i are waited for;
//   * eight warps, a lane a key, two halves of the rows: maxima meet by shuffles and one exchange among a half's four warps; a row's reference moves when its
//     maximum has grown by 2^8.  A weight is two terms of the cache's type (bfloat16 2^-17 of it; one term left an output 1.4 times as far off), whose products have
//     accumulators of their own; its sum is float32 of the unrounded one.
// Only tiles that hold the step's rows, or the context's end, look at masks; values there as in paged_tc.cu.  Blocks of a cluster share a sequence's keys.
// Bound by the bytes of the keys and, for one request, by the chain from launch to fold.
#include "paged.cuh"
#include "tc_common.cuh"
#include "tma.cuh"
#include "../../include/pgk_b200.h"

namespace pgk {

namespace {

constexpr int W_KEYS = 128, W_SOFT = 8, W_THREADS = (W_SOFT + 2) * 32;
constexpr uint32_t W_CHUNK = W_KEYS * 128;                         // 64 elements of 128 keys

struct FewCopies {
    int bp;                  // positions a copy, a power of two that divides the page; 0: four rows wherever they are
    int rows;                // of the cache: coordinates from here on read zeros
    int* err;
};

// NR: rows; C: 64-element chunks of a head
template <int NR, int C> struct Few {
    static constexpr int R = NR / 2, DG = (C + 1) / 2, DN = 64 * C, PBUF = NR == 64 ? 1 : 2;
    static constexpr uint32_t TILE = C * W_CHUNK, QCHUNK = NR * 128, Q = C * QCHUNK, P = W_KEYS * 4 * NR;
    static constexpr int ROOM = 218 * 1024 - 1024 - (int)(Q + PBUF * P), FIT = ROOM / (int)TILE, SLOTS = FIT < 8 ? FIT : 8;
    static constexpr int BYTES = SLOTS * (int)TILE + (int)(Q + PBUF * P) + 1024;
    static constexpr uint32_t COLUMNS = 2 * NR + DG * 2 * NR, TMEM = COLUMNS <= 64 ? 64 : (COLUMNS <= 128 ? 128 : (COLUMNS <= 256 ? 256 : 512));
    static_assert(SLOTS >= 2 && COLUMNS <= 512 && (2 * NR + PAGED_CLUSTER - 1) * (DN + 4) * 4 <= BYTES - 1024);
};

__device__ __forceinline__ bool all_wait(int* err, uint64_t* bar, uint32_t parity) {
    const bool ok = bar_wait(err, smem_u32(bar), parity);
    return __all_sync(0xffffffffu, ok);
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const float* v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
                 :: "r"(taddr), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]) : "memory");
}
template <int NR, int C, int DT>
__global__ void __launch_bounds__(W_THREADS, 1) paged_few_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                                                                 const __grid_constant__ PagedParams p, const __grid_constant__ FewCopies cp) {
    using X = Few<NR, C>;
    constexpr int R = X::R, SLOTS = X::SLOTS;
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ __align__(8) uint64_t full[SLOTS], empty[SLOTS], land, sfull[2], pready[2], pvdone[2];        // a barrier each: of two tiles both may have come before the first is looked for
    __shared__ uint32_t tmem_base_s;
    __shared__ __align__(16) float wmax[2][NR][4];
    __shared__ PagedFold<NR> f;
    __shared__ int missing;
    int* const err = cp.err;
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), D = p.dim;
    const uint32_t ring = (smem_u32(smem) + 1023u) & ~1023u, ps = ring + SLOTS * X::TILE, qs = ps + X::PBUF * X::P;

    if (warp == W_SOFT) tmem_alloc(&tmem_base_s, X::TMEM);
    if (tid == 0) {
        for (int s = 0; s < SLOTS; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
        mbar_init(&land, 1);
        mbar_init(&sfull[0], 1); mbar_init(&sfull[1], 1);
        mbar_init(&pready[0], W_SOFT); mbar_init(&pready[1], W_SOFT);
        mbar_init(&pvdone[0], 1); mbar_init(&pvdone[1], 1);
        mbar_fence_init();
        missing = f.bad = 0;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_base_s, tmem_o = tmem + 2 * NR;
    griddep_wait();
    griddep_launch();

    const PagedBlock<NR, W_KEYS> b(p, (int)blockIdx.x, (int)blockIdx.y, (int)blockIdx.z);
    const int n = b.uend - b.ubeg, steps = (D + 15) / 16;
    const int quad = warp & 3, half = (warp >> 2) & 1, r0 = half * R;

    if (warp < W_SOFT) {
        const int last = min(b.end, b.uend * W_KEYS), step = cp.bp ? cp.bp : 1;
        int j = b.ubeg * W_KEYS + step * tid;
        int page = j < last ? __ldcg(b.table + paged_div(j, p.by_page)) : 0;          // looked at behind the queries
        // ---------------- queries: rows of 128 bytes, 64 elements each, zeros behind the head's end
#pragma unroll 4
        for (int i = tid; i < NR * C * 8; i += W_SOFT * 32) {
            const int r = i / (C * 8), u = i - r * (C * 8), d = u * 8, x = b.f0 + r, row = paged_div(x, p.by_rep), tok = b.first + row;
            uint4 v = make_uint4(0, 0, 0, 0);
            if (r < b.live && d < D && tok >= 0 && tok < p.tokens) {
                const uint16_t* src = (const uint16_t*)p.q + (size_t)tok * p.q_ld + (size_t)(b.head * p.rep + x - row * p.rep) * D + d;
                if (p.wide_q) v = ld_act16(src);
                else {
                    uint32_t w[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) w[e] = (uint32_t)ld_act2(src + 2 * e) | (uint32_t)ld_act2(src + 2 * e + 1) << 16;
                    v = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};"
                         :: "r"(qs + (uint32_t)(u >> 3) * X::QCHUNK + (uint32_t)r * 128u + (uint32_t)(((u & 7) ^ (r & 7)) << 4)), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
        }
        bool gone = (unsigned)page >= (unsigned)p.pages;
        for (j += step * W_SOFT * 32; j < last; j += step * W_SOFT * 32) gone |= b.row_of(p, j) < 0;
        if (gone) missing = 1;
        fence_proxy_async();
    }
    if (warp <= W_SOFT) {                          // the copies are on their way meanwhile
        __syncwarp();
        asm volatile("bar.sync 5, %0;" :: "n"((W_SOFT + 1) * 32) : "memory");
    }

    if (warp == W_SOFT) {
        // ---------------- MMAs, from one thread; the ring has K 0, K 1, V 0, K 2, V 1, ...
        if (elect_one()) {
            constexpr uint32_t types = DT == 1 ? ~((1u << 7) | (1u << 10)) : ~0u;        // both operands float16, or both bfloat16
            constexpr uint32_t id_s = umma_idesc_bf16(NR) & types, id_o = umma_idesc_bf16_mn(2 * NR) & types;
            RingPos at;
            bool ok = true;
            auto scores = [&](int i) {
                ok = ok && bar_wait(err, smem_u32(&full[at.s]), at.round);
                if (!ok) return;
                tc_fence_after();
                const uint64_t dk = desc_sw128(ring + at.s * X::TILE), dq = desc_sw128(qs);
                const uint32_t to = tmem + (uint32_t)(i & 1) * NR;
#pragma unroll
                for (int k = 0; k < 4 * C; ++k)
                    if (k < steps)
                        umma_bf16(to, dk + (uint64_t)((k >> 2) * (W_CHUNK / 16) + (k & 3) * 2), dq + (uint64_t)((k >> 2) * (X::QCHUNK / 16) + (k & 3) * 2), id_s, k ? 1u : 0u);
                umma_commit(&sfull[i & 1]);
                umma_commit(&empty[at.s]);
                at.next(SLOTS);
            };
            if (n > 0) scores(0);
            int made = 0;
            for (int i = 0; ok && i < n; ++i) {
                if (i + 1 < n) scores(i + 1);      // where the scores of tile i - 1 were, whose weights have been waited for
                ok = ok && bar_wait(err, smem_u32(&pready[i & 1]), (uint32_t)(i >> 1) & 1u) && bar_wait(err, smem_u32(&full[at.s]), at.round);
                if (!ok) break;
                tc_fence_after();
                const uint32_t from = ps + (X::PBUF == 2 ? (uint32_t)(i & 1) * X::P : 0u);
                const uint64_t dv = desc_mn_sw128(ring + at.s * X::TILE, W_CHUNK);
                const uint64_t dp = NR == 16 ? desc_mn_sw64(from, X::P) : desc_mn_sw128(from, W_CHUNK);
#pragma unroll
                for (int g = 0; g < X::DG; ++g)
#pragma unroll
                    for (int k = 0; k < W_KEYS / 16; ++k)          // 16 keys: 2048 bytes of V, 1024 or 2048 of the weights
                        umma_bf16(tmem_o + (uint32_t)g * (2 * NR), dv + (uint64_t)(g * (2 * W_CHUNK / 16) + k * 128), dp + (uint64_t)(k * (NR == 16 ? 64 : 128)), id_o, (i | k) ? 1u : 0u);
                umma_commit(&pvdone[i & 1]);
                umma_commit(&empty[at.s]);
                at.next(SLOTS);
                made = i + 1;
            }
            if (made) bar_wait(err, smem_u32(&pvdone[(made - 1) & 1]), (uint32_t)((made - 1) >> 1) & 1u);
        }
        __syncwarp();
    } else if (warp == W_SOFT + 1) {
        // ---------------- copies
        const int pieces = cp.bp ? W_KEYS / cp.bp : 32;
        bool ok = true, bad = false;
        int issued = 0;
        uint32_t landed = 0;
        RingPos at;
        const int from = min(b.base, b.end);       // from here on values are looked at
        // this lane's piece of tile i: no such position or page: zeros
        auto where = [&](int i, int e) {
            const int r = lane < pieces && i < n ? b.row_of(p, (b.ubeg + i) * W_KEYS + (cp.bp ? lane * cp.bp : 4 * lane + e)) : -1;
            return r < 0 ? cp.rows : r;
        };
        int even[4], odd[4];                       // of tiles i and i + 1 by turns
        auto look = [&](int i) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (e == 0 || !cp.bp) {
                    const int r = where(i, e);
                    if (i & 1) odd[e] = r;
                    else even[e] = r;
                }
        };
        auto fetch = [&](const CUtensorMap* map, int i, bool fix) {
            ok = ok && all_wait(err, &empty[at.s], at.round ^ 1u);
            if (!ok) return;
            const uint32_t bar = smem_u32(fix ? &land : &full[at.s]), tile = ring + at.s * X::TILE;
            if (lane == 0) mbar_expect_tx(bar, X::TILE);
            __syncwarp();
            const int x0 = i & 1 ? odd[0] : even[0];
            if (cp.bp) {
                if (lane < pieces)
#pragma unroll
                    for (int c = 0; c < C; ++c) tma_load_2d(tile + (uint32_t)c * W_CHUNK + (uint32_t)(lane * cp.bp) * 128u, map, c * 64, x0, bar);
            } else {
                const int x1 = i & 1 ? odd[1] : even[1], x2 = i & 1 ? odd[2] : even[2], x3 = i & 1 ? odd[3] : even[3];
#pragma unroll
                for (int c = 0; c < C; ++c) tma_gather4(tile + (uint32_t)c * W_CHUNK + (uint32_t)lane * 512u, map, c * 64, x0, x1, x2, x3, bar);
            }
            ++issued;
            if (fix) {
                ok = all_wait(err, &land, landed);
                landed ^= 1u;
                if (!ok) return;
                bad |= paged_fix_values<DT>(tile, C, W_CHUNK, (b.ubeg + i) * W_KEYS, from, b.end, cp.bp, lane);
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(&full[at.s]);
            }
            at.next(SLOTS);
        };
        if (n > 0) {
            look(0);
            fetch(&kmap, 0, false);
            look(1);
            for (int i = 0; ok && i < n; ++i) {
                if (i + 1 < n) fetch(&kmap, i + 1, false);
                if (ok) fetch(&vmap, i, (b.ubeg + i + 1) * W_KEYS > from);
                look(i + 2);
            }
        }
        if (bad) f.bad = 1;
        if (lane == 0)
            for (int j = max(0, issued - SLOTS); j < issued; ++j)         // whoever gave up: do not leave with copies in flight
                bar_wait(err, smem_u32(&full[j % SLOTS]), (uint32_t)(j / SLOTS) & 1u);
        __syncwarp();
    } else {
        // ---------------- weights: lane = key, rows r0 ... r0 + R - 1
        const uint32_t lanes = tmem + ((uint32_t)(quad * 32) << 16);
        const int clean = missing ? 0 : min(b.base, b.end);               // keys before this one are seen by all
        const int key = quad * 32 + lane, mine = r0 + (lane & (R - 1));    // the row whose reference the lane keeps
        const int step_row = paged_div(b.f0 + mine, p.by_rep), tok = b.first + step_row;
        const bool live = mine < b.live && tok >= 0 && tok < p.tokens;
        float m_r = -INFINITY, nm[R], l[R];
#pragma unroll
        for (int r = 0; r < R; ++r) nm[r] = l[r] = 0.f;
        bool ok = true;
        for (int i = 0; i < n; ++i) {
            const int j0 = (b.ubeg + i) * W_KEYS + quad * 32, j = j0 + lane;
            const bool edge = j0 + 32 > clean;
            uint32_t see = 0;                      // of the warp's keys the ones that the lane's row sees
            bool there = true;
            if (edge) {
                see = live && j0 < b.end ? paged_window(p, tok, step_row, j0 - b.base) : 0u;
                there = missing ? b.row_of(p, j) >= 0 : j < b.end;
            }
            ok = ok && all_wait(err, &sfull[i & 1], (uint32_t)((i >> 1) & 1));
            __syncwarp();
            tc_fence_after();
            float s[R];
            tmem_columns<R>(lanes + (uint32_t)(i & 1) * NR + (uint32_t)r0, s);
            if (edge) {
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const uint32_t bits = __shfl_sync(0xffffffffu, see, r);
                    if (!there || !((bits >> lane) & 1u)) s[r] = -INFINITY;
                }
            }
            float v[R];
#pragma unroll
            for (int r = 0; r < R; ++r) v[r] = s[r];
            const float top = reduce_lanes<R>(v, lane, [](float x, float y) { return fmaxf(x, y); });
            if (lane < R) wmax[i & 1][r0 + lane][quad] = top;
            __syncwarp();
            asm volatile("bar.sync %0, 128;" :: "r"(1 + half) : "memory");
            const float4 w = *(const float4*)wmax[i & 1][mine];
            const float mt = paged_reference<DT>(fmaxf(fmaxf(w.x, w.y), fmaxf(w.z, w.w)) * p.scale_log2);
            const bool up = mt > m_r + PAGED_LAZY;                // (also the first finite maximum)
            bool waited = false;
            if (__any_sync(0xffffffffu, up)) {                    // the same in the half's four warps: its columns of O^T move along
                const float f_r = !up ? 1.f : (m_r == -INFINITY ? 0.f : exp2f(m_r - mt));
                if (up) m_r = mt;
                float fix[R];
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    nm[r] = paged_neg(__shfl_sync(0xffffffffu, m_r, r));
                    fix[r] = __shfl_sync(0xffffffffu, f_r, r);
                    l[r] *= fix[r];
                }
                if (i > 0) {
                    ok = ok && all_wait(err, &pvdone[(i - 1) & 1], (uint32_t)((i - 1) >> 1) & 1u);
                    __syncwarp();
                    waited = true;
                    tc_fence_after();
#pragma unroll 1
                    for (int g = 0; g < 2 * X::DG; ++g) {
                        const uint32_t to = lanes + 2 * NR + (uint32_t)g * NR + (uint32_t)r0;
                        float o[R];
                        tmem_columns<R>(to, o);
#pragma unroll
                        for (int r = 0; r < R; ++r) o[r] *= fix[r];
#pragma unroll
                        for (int r = 0; r < R; r += 8) tmem_st8(to + (uint32_t)r, o + r);
                    }
                    tmem_st_wait();
                }
            }
            const uint64_t scale2 = pair(p.scale_log2, p.scale_log2), zero2 = pair(p.zero, p.zero);
            uint32_t hi[R / 2], lo[R / 2];
#pragma unroll
            for (int e = 0; e < R / 2; ++e) {
                float a, c;
                unpair(add2(fma2(pair(s[2 * e], s[2 * e + 1]), scale2, zero2), pair(nm[2 * e], nm[2 * e + 1])), a, c);
                a = ex2(a);
                c = ex2(c);
                l[2 * e] += a;
                l[2 * e + 1] += c;
                paged_weights2x2<DT>(a, c, hi[e], lo[e]);
            }
            // the product that has read what was here: of the tile before, or the one before that
            if (i >= X::PBUF && !waited) {
                ok = ok && all_wait(err, &pvdone[(i - X::PBUF) & 1], (uint32_t)((i - X::PBUF) >> 1) & 1u);
                __syncwarp();
            }
            const uint32_t to = ps + (X::PBUF == 2 ? (uint32_t)(i & 1) * X::P : 0u);
            auto put = [&](int term, int u, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
                uint32_t a;
                if constexpr (NR == 16) a = to + (uint32_t)key * 64u + (uint32_t)(((2 * term + half) ^ ((key >> 1) & 3)) << 4);
                else if constexpr (NR == 32) a = to + (uint32_t)key * 128u + (uint32_t)(((4 * term + 2 * half + u) ^ (key & 7)) << 4);
                else a = to + (uint32_t)term * W_CHUNK + (uint32_t)key * 128u + (uint32_t)(((4 * half + u) ^ (key & 7)) << 4);
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" :: "r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
            };
#pragma unroll
            for (int u = 0; u < R / 8; ++u) {
                put(0, u, hi[4 * u], hi[4 * u + 1], hi[4 * u + 2], hi[4 * u + 3]);
                put(1, u, lo[4 * u], lo[4 * u + 1], lo[4 * u + 2], lo[4 * u + 3]);
            }
            fence_proxy_async();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&pready[i & 1]);
        }
        // ---------------- a row's reference and sum
        const float sum = reduce_lanes<R>(l, lane, [](float x, float y) { return x + y; });
        asm volatile("bar.sync %0, 128;" :: "r"(1 + half) : "memory");             // the last tile's maxima are read
        if (lane < R) wmax[0][r0 + lane][quad] = sum;
        __syncwarp();
        asm volatile("bar.sync %0, 128;" :: "r"(1 + half) : "memory");
        if (quad == 0 && lane < R) {
            const float4 w = *(const float4*)wmax[0][mine];
            f.m[mine] = m_r;
            f.l[mine] = (w.x + w.y) + (w.z + w.w);
        }
    }
    PagedOut<NR, W_KEYS, DT, X::DN> out(p, b, f, (float*)(smem + (ring - smem_u32(smem))));
    out.begin();                                   // nobody's tile is read or written any more
    tc_fence_after();
    if (warp < W_SOFT) {
#pragma unroll 1
        for (int g = 0; g < X::DG; ++g) {
            const int d = g * 128 + quad * 32 + lane;
            const uint32_t at = tmem_o + ((uint32_t)(quad * 32) << 16) + (uint32_t)g * (2 * NR) + (uint32_t)r0;
            float x[R], y[R];
            if (n > 0) {
                tmem_columns<R>(at, x);
                tmem_columns<R>(at + NR, y);
            } else {
#pragma unroll
                for (int r = 0; r < R; ++r) x[r] = y[r] = 0.f;
            }
            if (d < X::DN) {
#pragma unroll
                for (int r = 0; r < R; ++r)
                    out.stage[(r0 + r) * out.LD + d] = x[r] + y[r];
            }
            __syncwarp();
        }
    }
    tc_fence_before();
    out.join([&] {
        if (warp == W_SOFT) tmem_dealloc(tmem, X::TMEM);
    });
}

template <int NR, int C, int DT>
int launch_few(PagedParams p, cudaStream_t st) {
    using X = Few<NR, C>;
    static PagedOccupancy fits;
    const auto kernel = paged_few_kernel<NR, C, DT>;
    PGK_CUDA(fits.once([&](int* at_once) {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, X::BYTES);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        for (int i = 1; e == cudaSuccess && i <= PAGED_CLUSTER; ++i) e = clusters_at_once(&at_once[i], kernel, W_THREADS, X::BYTES, i);
        return e;
    }));
    FewCopies cp = {};
    cp.bp = p.page_size & -p.page_size;
    if (cp.bp > W_KEYS) cp.bp = W_KEYS;
    if (cp.bp < 8) cp.bp = 0;
    cp.rows = p.pages * p.kv_heads * p.page_size;
    cp.err = wait_word(kWaitPagedFew);
    PGK_REQUIRE(cp.err, "paged_attention failed: no pinned host memory");
    CUtensorMap kmap{}, vmap{};
    const uint32_t box = cp.bp ? (uint32_t)cp.bp : 1u;
    PGK_REQUIRE(tma_encode_fn() && tma_map_bf16_2d(&kmap, p.k_data, (uint64_t)p.dim, (uint64_t)cp.rows, (uint64_t)p.dim * 2, 64, box) &&
                    tma_map_bf16_2d(&vmap, p.v_data, (uint64_t)p.dim, (uint64_t)cp.rows, (uint64_t)p.dim * 2, 64, box),
                "paged_attention failed: no tensor map of %d rows of %d elements", cp.rows, p.dim);
    p.tiles = (int)(((long long)p.max_rows * p.rep + NR - 1) / NR);
    return paged_launch<NR, W_KEYS, DT, X::DN>(p, paged_split(p, W_KEYS, fits.at_once, PAGED_CLUSTER, 4), st, [&](const PagedParams& q, dim3 grid, bool apart) {
        return launch_clusters(kernel, grid, apart, W_THREADS, (size_t)X::BYTES, st, kmap, vmap, q, cp);
    });
}
template <int C, int DT>
int launch_few_rows(const PagedParams& p, cudaStream_t st) {
    const long long rows = (long long)p.max_rows * p.rep;
    if (rows <= 16) return launch_few<16, C, DT>(p, st);
    return rows <= 32 ? launch_few<32, C, DT>(p, st) : launch_few<64, C, DT>(p, st);
}
template <int DT>
int launch_few_dim(const PagedParams& p, cudaStream_t st) {
    switch ((p.dim + 63) / 64) {
        case 1: return launch_few_rows<1, DT>(p, st);
        case 2: return launch_few_rows<2, DT>(p, st);
        case 3: return launch_few_rows<3, DT>(p, st);
        default: return launch_few_rows<4, DT>(p, st);
    }
}

}  // namespace

int paged_few(const PagedParams& p, int dtype, cudaStream_t st) { return dtype == 1 ? launch_few_dim<1>(p, st) : launch_few_dim<2>(p, st); }

}  // namespace pgk
