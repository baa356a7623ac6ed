// paged_weigh.cu -- the attention weights that a cached position gets, summed over a step's rows and the query heads of its key head: what decides which positions of a
// cache stay when it is cut.  weights[slot][g][j] += sum over rows i and heads h of g of exp(scale q_ih . k_j - lse_ih), lse from the attention over the same rows.
//
// 16-bit pages: scores S^T[128 keys, NR rows] = K Q^T by tcgen05 as in paged_few.cu, tiles of K through a ring, the step's rows in shared memory (as many as 64 KB hold at a
// time); eight warps, a lane a key and half of the rows each, sum the weights as they come.  32-bit pages: multiply-adds, a lane a key.  A position's sum is one
// thread's until it is added, so that the same call gives the same bits.  Decoding is bound by the bytes of the keys, windows of a prompt's last tokens by the exponentials.
#include <type_traits>

#include "paged.cuh"
#include "tc_common.cuh"
#include "tma.cuh"
#include "../../include/pgk_b200.h"

namespace pgk {

namespace {

constexpr int H_ALL = 1 << 30;                                // rows of a "block": all of the sequence's
constexpr int H_KEYS = 128, H_SOFT = 8, H_THREADS = (H_SOFT + 2) * 32, H_QBYTES = 64 * 1024;
constexpr uint32_t H_CHUNK = H_KEYS * 128;                    // 64 elements of 128 keys
constexpr int G_WARPS = 4, G_THREADS = G_WARPS * 32, G_KEYS = G_WARPS * 32, G_ROWS = 16;

using Keys = PagedBlock<H_ALL, H_KEYS>;
static_assert(H_KEYS == G_KEYS);

// minus a row's logarithm (log2); for rows that see nothing a number that leaves no weight
constexpr float H_NONE = -3e38f;
__device__ __forceinline__ float row_neg(const PagedParams& p, const Keys& b, int r) {
    const int tok = b.token(p, r);
    if (r >= b.live || tok < 0 || tok >= p.tokens) return H_NONE;
    const float z = __ldcg(p.lse + (size_t)tok * p.heads + b.head * p.rep + r - paged_div(r, p.by_rep) * p.rep);
    return z == -INFINITY ? H_NONE : -z * PAGED_LOG2E;
}
__device__ __forceinline__ void add_weight(const PagedParams& p, const Keys& b, int j, float w) {
    atomicAdd(p.weights + ((size_t)b.slot * p.kv_heads + b.head) * p.weights_ld + j, w);
}

struct WeighCopies {
    int bp, rows;            // as in paged_few.cu
    int groups;              // of NR rows, in shared memory at a time
    int* err;
};

// NR: rows of a product; C: 64-element chunks of a head
template <int NR, int C> struct Weigh {
    static constexpr int R = NR / 2, SLOTS = C == 1 ? 4 : (C == 2 ? 3 : 2);
    static constexpr uint32_t TILE = C * H_CHUNK, QCHUNK = NR * 128, Q = C * QCHUNK, TMEM = 2 * NR < 32 ? 32 : 2 * NR;
    static constexpr int MOST = H_QBYTES / (int)Q;
    static int bytes(int groups) { return SLOTS * (int)TILE + groups * ((int)Q + NR * 4) + 1024; }
};

template <int NR, int C, int DT>
__global__ void __launch_bounds__(H_THREADS) paged_weigh_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ PagedParams p, const __grid_constant__ WeighCopies cp) {
    using X = Weigh<NR, C>;
    constexpr int R = X::R, SLOTS = X::SLOTS;
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ __align__(8) uint64_t full[SLOTS], empty[SLOTS], sfull[2], sread[2];
    __shared__ uint32_t tmem_base_s;
    __shared__ float other[2][H_KEYS];
    __shared__ int missing;
    int* const err = cp.err;
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), D = p.dim;
    const uint32_t ring = (smem_u32(smem) + 1023u) & ~1023u, qs = ring + SLOTS * X::TILE;
    float* const negs = (float*)(smem + (qs - smem_u32(smem)) + (size_t)cp.groups * X::Q);        // [groups][NR]

    if (warp == H_SOFT) tmem_alloc(&tmem_base_s, X::TMEM);
    if (tid == 0) {
        for (int s = 0; s < SLOTS; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
        for (int s = 0; s < 2; ++s) { mbar_init(&sfull[s], 1); mbar_init(&sread[s], H_SOFT); }
        mbar_fence_init();
        missing = 0;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_base_s;
    griddep_wait();
    griddep_launch();

    const Keys b(p, (int)blockIdx.z, (int)blockIdx.y, (int)blockIdx.x);
    const int n = b.live > 0 ? b.uend - b.ubeg : 0, steps = (D + 15) / 16, batch = cp.groups * NR, batches = (b.live + batch - 1) / batch;
    const int quad = warp & 3, half = (warp >> 2) & 1, r0 = half * R;

    if (warp < H_SOFT) {
        const int last = min(b.end, b.uend * H_KEYS), step = cp.bp ? cp.bp : 1;
        bool gone = false;
        for (int j = b.ubeg * H_KEYS + step * tid; j < last; j += step * H_SOFT * 32) gone |= b.row_of(p, j) < 0;
        if (gone) missing = 1;
    }
    int turns = 0, tiles = 0;                      // of the batches before: score buffers and ring places that were used
    bool ok = true;
    for (int y = 0; y < batches; ++y) {
        const int f0 = y * batch, groups = min(cp.groups, (b.live - f0 + NR - 1) / NR);
        int turn = turns;
        RingPos at;
        at.s = (uint32_t)(tiles % SLOTS);
        at.round = (uint32_t)(tiles / SLOTS) & 1u;
        if (warp < H_SOFT) {
            // ---------------- the batch's rows
#pragma unroll 4
            for (int i = tid; i < groups * NR * C * 8; i += H_SOFT * 32) {
                const int r = i / (C * 8), u = i - r * (C * 8), d = u * 8, x = f0 + r, row = paged_div(x, p.by_rep), tok = b.first + row, g = r / NR, rr = r - g * NR;
                uint4 v = make_uint4(0, 0, 0, 0);
                if (x < b.live && d < D && tok >= 0 && tok < p.tokens) {
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
                             :: "r"(qs + (uint32_t)g * X::Q + (uint32_t)(u >> 3) * X::QCHUNK + (uint32_t)rr * 128u + (uint32_t)(((u & 7) ^ (rr & 7)) << 4)), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
                             : "memory");
            }
            for (int i = tid; i < groups * NR; i += H_SOFT * 32) negs[i] = row_neg(p, b, f0 + i);
            fence_proxy_async();
        }
        if (warp <= H_SOFT) {                      // the copies are on their way meanwhile
            __syncwarp();
            asm volatile("bar.sync 5, %0;" :: "n"((H_SOFT + 1) * 32) : "memory");
        }
        if (warp == H_SOFT) {
            // ---------------- MMAs, from one thread
            if (elect_one()) {
                for (int i = 0; ok && i < n; ++i) {
                    ok = bar_wait(err, smem_u32(&full[at.s]), at.round);
                    const uint64_t dk = desc_sw128(ring + at.s * X::TILE);
                    for (int g = 0; ok && g < groups; ++g, ++turn) {
                        ok = bar_wait(err, smem_u32(&sread[turn & 1]), ((uint32_t)(turn >> 1) & 1u) ^ 1u);
                        if (!ok) break;
                        tc_fence_after();
                        const uint64_t dq = desc_sw128(qs + (uint32_t)g * X::Q);
                        constexpr uint32_t types = DT == 1 ? ~((1u << 7) | (1u << 10)) : ~0u, id = umma_idesc_bf16(NR) & types;
#pragma unroll
                        for (int k = 0; k < 4 * C; ++k)
                            if (k < steps)
                                umma_bf16(tmem + (uint32_t)(turn & 1) * NR, dk + (uint64_t)((k >> 2) * (H_CHUNK / 16) + (k & 3) * 2),
                                          dq + (uint64_t)((k >> 2) * (X::QCHUNK / 16) + (k & 3) * 2), id, k ? 1u : 0u);
                        umma_commit(&sfull[turn & 1]);
                    }
                    if (ok) umma_commit(&empty[at.s]);
                    at.next(SLOTS);
                }
            }
            __syncwarp();
        } else if (warp == H_SOFT + 1) {
            // ---------------- copies, as in paged_few.cu
            const int pieces = cp.bp ? H_KEYS / cp.bp : 32;
            int row[4];
            auto look = [&](int i) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (e > 0 && cp.bp) continue;
                    const int r = lane < pieces && i < n ? b.row_of(p, (b.ubeg + i) * H_KEYS + (cp.bp ? lane * cp.bp : 4 * lane + e)) : -1;
                    row[e] = r < 0 ? cp.rows : r;
                }
            };
            look(0);
            for (int i = 0; ok && i < n; ++i) {
                ok = __all_sync(0xffffffffu, bar_wait(err, smem_u32(&empty[at.s]), at.round ^ 1u));
                if (!ok) break;
                const uint32_t bar = smem_u32(&full[at.s]), tile = ring + at.s * X::TILE;
                if (lane == 0) mbar_expect_tx(bar, X::TILE);
                __syncwarp();
                if (cp.bp) {
                    if (lane < pieces)
#pragma unroll
                        for (int c = 0; c < C; ++c) tma_load_2d(tile + (uint32_t)c * H_CHUNK + (uint32_t)(lane * cp.bp) * 128u, &kmap, c * 64, row[0], bar);
                } else {
#pragma unroll
                    for (int c = 0; c < C; ++c) tma_gather4(tile + (uint32_t)c * H_CHUNK + (uint32_t)lane * 512u, &kmap, c * 64, row[0], row[1], row[2], row[3], bar);
                }
                look(i + 1);
                at.next(SLOTS);
            }
        } else {
            // ---------------- weights: lane = key, rows r0 ... r0 + R - 1 of every group
            const uint32_t lanes = tmem + ((uint32_t)(quad * 32) << 16);
            const int clean = missing ? 0 : min(b.base, b.end), key = quad * 32 + lane;
            for (int i = 0; i < n; ++i) {
                const int j0 = (b.ubeg + i) * H_KEYS + quad * 32, j = j0 + lane;
                const bool edge = j0 + 32 > clean, there = edge && missing ? b.row_of(p, j) >= 0 : j < b.end;
                float sum = 0.f;
                for (int g = 0; g < groups; ++g, ++turn) {
                    const int rows = b.live - f0 - g * NR - r0;    // of this half's; where there are fewer than R, the rest's queries are zeros, which times an infinite key are NaN
                    const bool mixed = edge || rows < R;
                    uint32_t see = 0;
                    if (mixed) {
                        const int x = f0 + g * NR + r0 + (lane & (R - 1)), row = paged_div(x, p.by_rep);
                        see = x < b.live && j0 < b.end ? paged_window(p, b.first + row, row, j0 - b.base) : 0u;
                    }
                    ok = ok && __all_sync(0xffffffffu, bar_wait(err, smem_u32(&sfull[turn & 1]), (uint32_t)(turn >> 1) & 1u));
                    __syncwarp();
                    tc_fence_after();
                    float s[R];
                    tmem_columns<R>(lanes + (uint32_t)(turn & 1) * NR + (uint32_t)r0, s);
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sread[turn & 1]);
                    if (rows <= 0) continue;
                    const float4* const neg = (const float4*)(negs + g * NR + r0);
                    auto add = [&](auto masked) {          // apart from each other: a branch at every weight is 1340 cycles for 64 rows
                        const uint64_t scale2 = pair(p.scale_log2, p.scale_log2);
                        uint64_t sum2 = pair(sum, 0.f);
#pragma unroll
                        for (int r = 0; r < R; r += 4) {
                            const float4 x = neg[r / 4];
                            float w[4];
                            unpair(fma2(pair(s[r], s[r + 1]), scale2, pair(x.x, x.y)), w[0], w[1]);
                            unpair(fma2(pair(s[r + 2], s[r + 3]), scale2, pair(x.z, x.w)), w[2], w[3]);
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                w[e] = ex2(w[e]);
                                if constexpr (masked.value) {
                                    const uint32_t bits = __shfl_sync(0xffffffffu, see, r + e);
                                    if (!there || !((bits >> lane) & 1u)) w[e] = 0.f;
                                }
                            }
                            sum2 = add2(sum2, pair(w[0], w[1]));
                            sum2 = add2(sum2, pair(w[2], w[3]));
                        }
                        float u, v;
                        unpair(sum2, u, v);
                        sum = u + v;
                    };
                    if (mixed) add(std::true_type{});
                    else add(std::false_type{});
                }
                if (half == 1) other[i & 1][key] = sum;
                asm volatile("bar.sync %0, 64;" :: "r"(1 + quad) : "memory");      // a key's two warps; two turns of places, so that none is overwritten unread
                if (half == 0 && j < b.end) add_weight(p, b, j, sum + other[i & 1][key]);
            }
        }
        turns += n * groups;
        tiles += n;
        if (warp <= H_SOFT && y + 1 < batches) {   // the rows are read
            __syncwarp();
            asm volatile("bar.sync 5, %0;" :: "n"((H_SOFT + 1) * 32) : "memory");
        }
    }
    if (warp == H_SOFT + 1 && lane == 0 && !ok)    // whoever gave up: do not leave with copies in flight
        for (int s = 0; s < SLOTS; ++s) {
            bar_wait(err, smem_u32(&full[s]), 0u);
            bar_wait(err, smem_u32(&full[s]), 1u);
        }
    tc_fence_before();
    __syncthreads();
    if (warp == H_SOFT) tmem_dealloc(tmem, X::TMEM);
}

__global__ void __launch_bounds__(G_THREADS) paged_weigh_f32_kernel(const __grid_constant__ PagedParams p) {
    extern __shared__ __align__(16) float smf[];
    __shared__ float negs[G_ROWS];
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), D = p.dim, D4 = D / 4, DF = D + 4;
    float* const qs = smf;                                    // [G_ROWS][D]
    float* const ks = qs + G_ROWS * D + warp * 32 * DF;
    griddep_wait();
    griddep_launch();
    const Keys b(p, (int)blockIdx.z, (int)blockIdx.y, 0);        // all positions; the block's are the next line's
    const int k0 = (int)blockIdx.x * G_KEYS, j0 = k0 + 32 * warp, j = j0 + lane;
    if (k0 >= b.end || b.live == 0) return;

    const int rows = b.row_of(p, j);
    for (int r = 0; r < 32; ++r) {
        const int row = __shfl_sync(0xffffffffu, rows, r);
        for (int c = lane; c < D4; c += 32)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;"
                         :: "r"(smem_u32(ks + r * DF + 4 * c)), "l"((const float*)p.k_data + (size_t)max(row, 0) * D + 4 * c), "r"(row >= 0 ? 16u : 0u) : "memory");
    }
    cp_async_commit();
    const bool edge = __any_sync(0xffffffffu, rows < 0) || j0 + 32 > b.base;
    float sum = 0.f;
#pragma unroll 1
    for (int f0 = 0; f0 < b.live; f0 += G_ROWS) {
        __syncthreads();
        for (int i = tid; i < G_ROWS * D; i += G_THREADS) {
            const int r = i / D, f = f0 + r, row = paged_div(f, p.by_rep), tok = b.first + row;
            qs[i] = f < b.live && tok >= 0 && tok < p.tokens ? __ldcg((const float*)p.q + (size_t)tok * p.q_ld + (size_t)(b.head * p.rep + f - row * p.rep) * D + (i - r * D)) : 0.f;
        }
        if (tid < G_ROWS) negs[tid] = row_neg(p, b, f0 + tid);
        cp_async_wait<0>();
        __syncthreads();
        const int n = min(G_ROWS, b.live - f0);
#pragma unroll 1
        for (int r0 = 0; r0 < n; r0 += 4) {
            float s[4] = {};
            const float* const kr = ks + lane * DF;
#pragma unroll 4
            for (int c = 0; c < D4; ++c) {
                const float4 x = *(const float4*)(kr + 4 * c);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float4 q = *(const float4*)(qs + (r0 + r) * D + 4 * c);
                    s[r] = fmaf(q.x, x.x, fmaf(q.y, x.y, fmaf(q.z, x.z, fmaf(q.w, x.w, s[r]))));
                }
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float w = ex2(fmaf(s[r], p.scale_log2, negs[r0 + r]));
                bool sees = f0 + r0 + r < b.live;          // (other rows' queries are zeros: an infinite key makes NaN of them)
                if (edge && sees) {
                    const int i = paged_div(f0 + r0 + r, p.by_rep);
                    sees = rows >= 0 && (j < b.base || paged_sees(p, b.first + i, i, j - b.base));
                }
                if (sees) sum += w;
            }
        }
    }
    if (j < b.end) add_weight(p, b, j, sum);
}

template <int NR, int C, int DT> int launch_weigh(PagedParams p, cudaStream_t st) {
    using X = Weigh<NR, C>;
    static bool configured = false;
    if (!configured) {
        PGK_CUDA(cudaFuncSetAttribute(paged_weigh_kernel<NR, C, DT>, cudaFuncAttributeMaxDynamicSharedMemorySize, X::bytes(X::MOST)));
        configured = true;
    }
    WeighCopies cp = {};
    cp.bp = p.page_size & -p.page_size;
    if (cp.bp > H_KEYS) cp.bp = H_KEYS;
    if (cp.bp < 8) cp.bp = 0;
    cp.rows = p.pages * p.kv_heads * p.page_size;
    const long long groups = ((long long)p.max_rows * p.rep + NR - 1) / NR;
    cp.groups = (int)(groups < X::MOST ? groups : X::MOST);
    cp.err = wait_word(kWaitWeigh);
    PGK_REQUIRE(cp.err, "paged_weigh failed: no pinned host memory");
    CUtensorMap kmap{};
    PGK_REQUIRE(tma_encode_fn() && tma_map_bf16_2d(&kmap, p.k_data, (uint64_t)p.dim, (uint64_t)cp.rows, (uint64_t)p.dim * 2, 64, cp.bp ? (uint32_t)cp.bp : 1u),
                "paged_weigh failed: no tensor map of %d rows of %d elements", cp.rows, p.dim);
    // blocks that share a sequence's positions: rounds of all SMs times (a block's tiles + what it costs besides, about three of them)
    const int smem = X::bytes(cp.groups), resident = smem > 112 * 1024 ? 1 : (smem > 74 * 1024 ? 2 : 3), nt = (p.max_keys + H_KEYS - 1) / H_KEYS;
    const long long items = (long long)p.seqs * p.kv_heads, slots = (long long)resident * sm_count();
    long long least = 0;
    for (int s = 1; s <= nt && s <= 1024; ++s) {
        const long long cost = ((items * s + slots - 1) / slots) * ((nt + s - 1) / s + 3);
        if (s == 1 || cost < least) { p.splits = s; least = cost; }
    }
    p.by_splits = paged_divisor(p.splits);
    PGK_CUDA(launch_waiting(paged_weigh_kernel<NR, C, DT>, dim3(p.splits, p.kv_heads, p.seqs), dim3(H_THREADS), (size_t)smem, st, kmap, p, cp));
    return 0;
}
template <int C, int DT> int launch_weigh_rows(const PagedParams& p, cudaStream_t st) {
    const long long rows = (long long)p.max_rows * p.rep;
    if (rows <= 16) return launch_weigh<16, C, DT>(p, st);
    return rows <= 32 ? launch_weigh<32, C, DT>(p, st) : launch_weigh<64, C, DT>(p, st);
}
template <int DT> int launch_weigh_dim(const PagedParams& p, cudaStream_t st) {
    switch ((p.dim + 63) / 64) {
        case 1: return launch_weigh_rows<1, DT>(p, st);
        case 2: return launch_weigh_rows<2, DT>(p, st);
        case 3: return launch_weigh_rows<3, DT>(p, st);
        default: return launch_weigh_rows<4, DT>(p, st);
    }
}

int weigh(PagedParams p, int dtype, cudaStream_t st) {
    p.tiles = 1;
    if (p.max_keys == 0) return 0;
    if (dtype == 1) return launch_weigh_dim<1>(p, st);
    if (dtype == 2) return launch_weigh_dim<2>(p, st);
    p.splits = 1;
    const dim3 grid((unsigned)((p.max_keys + G_KEYS - 1) / G_KEYS), p.kv_heads, p.seqs);
    static bool configured = false;
    if (!configured) {
        PGK_CUDA(cudaFuncSetAttribute(paged_weigh_f32_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (G_ROWS * 256 + G_WARPS * 32 * 260) * 4));
        configured = true;
    }
    PGK_CUDA(launch_waiting(paged_weigh_f32_kernel, grid, dim3(G_THREADS), (size_t)(G_ROWS * p.dim + G_WARPS * 32 * (p.dim + 4)) * 4, st, p));
    return 0;
}

// what all calls over such a cache have to fulfil, and their parameters
int paged_params(const char* fn, PagedParams* out, const void* q, long q_ld, const void* k_cache, const void* v_cache, int pages, int page_size, const int32_t* page_table, int slots,
                 int max_pages, const int32_t* seq_slots, const int32_t* context_lens, const int32_t* row_starts, int seqs, int tokens, int max_rows, int max_context, int heads,
                 int kv_heads, int dim, float scale, const int32_t* masks, int mask_words, int dtype) {
    PGK_REQUIRE(dtype >= 0 && dtype <= 2, "%s failed: unknown type %d", fn, dtype);
    PGK_REQUIRE(dim >= 8 && dim <= 256 && dim % 8 == 0, "%s failed: heads of %d elements (multiples of 8 up to 256)", fn, dim);
    PGK_REQUIRE(pages > 0 && page_size > 0 && slots > 0 && max_pages > 0 && kv_heads > 0 && kv_heads <= 65535 && heads > 0 && heads % kv_heads == 0,
                "%s failed: %d pages of %d positions, %d slots of %d pages, %d query heads over %d", fn, pages, page_size, slots, max_pages, heads, kv_heads);
    PGK_REQUIRE((long long)pages * kv_heads * page_size <= 0x7fffffffll && (long long)max_pages * page_size <= 0x7fffffffll, "%s failed: more than 2^31 rows of a cache", fn);
    PGK_REQUIRE(q_ld >= (long)heads * dim, "%s failed: rows of %ld for %d heads of %d", fn, q_ld, heads, dim);
    PGK_REQUIRE(seqs >= 0 && seqs <= 65535 && tokens >= 0 && max_rows > 0 && max_context >= 0 && (row_starts || (tokens >= seqs && max_rows == 1)) &&
                    (long long)max_rows * (heads / kv_heads) <= 1 << 24 && (long long)seqs * max_rows * (heads / kv_heads) <= 0x7fffffffll,
                "%s failed: %d sequences of up to %d rows in %d, %d keys", fn, seqs, max_rows, tokens, max_context);
    PGK_REQUIRE(scale >= 0.f && scale < 1e38f, "%s failed: scale %g", fn, scale);
    PGK_REQUIRE(mask_words >= 0 && (!masks || mask_words > 0) && mask_words <= 1 << 20, "%s failed: masks of %d words", fn, mask_words);
    PGK_REQUIRE(seqs == 0 || tokens == 0 || (q && k_cache && v_cache && page_table && seq_slots && context_lens), "%s failed: an array is missing", fn);
    PGK_REQUIRE((uintptr_t)k_cache % 16 == 0 && (uintptr_t)v_cache % 16 == 0 && (uintptr_t)q % (dtype ? 2 : 4) == 0, "%s failed: a cache that does not start on 16 bytes", fn);
    PagedParams p = {};
    p.q = q; p.q_ld = q_ld;
    p.k_data = k_cache; p.v_data = v_cache; p.table = page_table;
    p.pages = pages; p.page_size = page_size; p.slots = slots; p.max_pages = max_pages; p.kv_heads = kv_heads; p.dim = dim;
    p.seq_slots = seq_slots; p.contexts = context_lens; p.starts = row_starts;
    p.seqs = seqs; p.tokens = tokens; p.heads = heads; p.rep = heads / kv_heads;
    p.max_rows = max_rows < tokens ? max_rows : tokens;
    p.max_keys = max_context < max_pages * page_size ? max_context : max_pages * page_size;
    p.scale_log2 = (scale > 0.f ? scale : 1.f / sqrtf((float)dim)) * PAGED_LOG2E;
    p.masks = masks; p.words = mask_words;
    p.by_page = paged_divisor(page_size);
    p.by_rep = paged_divisor(p.rep);
    p.by_seqs = paged_divisor(p.seqs);
    const int size = dtype == 0 ? 4 : 2;
    p.wide_q = (uintptr_t)q % 16 == 0 && q_ld * size % 16 == 0;
    *out = p;
    return 0;
}

}  // namespace

}  // namespace pgk

using namespace pgk;

extern "C" int pgk_paged_attention(const void* q, long q_ld, const void* k_cache, const void* v_cache, void* out, long o_ld, int pages, int page_size,
                                   const int32_t* page_table, int slots, int max_pages, const int32_t* seq_slots, const int32_t* context_lens, const int32_t* row_starts,
                                   int seqs, int tokens, int max_rows, int max_context, int heads, int kv_heads, int dim, float scale, const int32_t* masks, int mask_words,
                                   float* lse, int dtype, void* stream) {
    PagedParams p;
    if (int rc = paged_params("paged_attention", &p, q, q_ld, k_cache, v_cache, pages, page_size, page_table, slots, max_pages, seq_slots, context_lens, row_starts, seqs, tokens,
                              max_rows, max_context, heads, kv_heads, dim, scale, masks, mask_words, dtype))
        return rc;
    PGK_REQUIRE(o_ld >= (long)heads * dim, "paged_attention failed: output rows of %ld for %d heads of %d", o_ld, heads, dim);
    if (seqs == 0 || tokens == 0) return 0;
    PGK_REQUIRE(out, "paged_attention failed: no output");
    const int size = dtype == 0 ? 4 : 2;
    p.out = out; p.o_ld = o_ld; p.lse = lse;
    p.wide_o = (uintptr_t)out % 16 == 0 && o_ld * size % 16 == 0;
    const cudaStream_t st = (cudaStream_t)stream;
    if (dtype == 0) return paged_f32(p, st);
    return paged_tc_serves(p, dtype) ? paged_tc(p, dtype, st) : paged_few(p, dtype, st);
}

extern "C" int pgk_paged_weigh(const void* q, long q_ld, const void* k_cache, const float* lse, float* weights, long weights_ld, int pages, int page_size,
                               const int32_t* page_table, int slots, int max_pages, const int32_t* seq_slots, const int32_t* context_lens, const int32_t* row_starts, int seqs,
                               int tokens, int max_rows, int max_context, int heads, int kv_heads, int dim, float scale, const int32_t* masks, int mask_words, int dtype,
                               void* stream) {
    PagedParams p;
    if (int rc = paged_params("paged_weigh", &p, q, q_ld, k_cache, k_cache, pages, page_size, page_table, slots, max_pages, seq_slots, context_lens, row_starts, seqs, tokens,
                              max_rows, max_context, heads, kv_heads, dim, scale, masks, mask_words, dtype))
        return rc;
    PGK_REQUIRE(weights_ld >= max_context, "paged_weigh failed: weights of %ld positions for %d", weights_ld, max_context);
    if (seqs == 0 || tokens == 0) return 0;
    PGK_REQUIRE(lse && weights, "paged_weigh failed: an array is missing");
    p.lse = const_cast<float*>(lse); p.weights = weights; p.weights_ld = weights_ld;
    return weigh(p, dtype, (cudaStream_t)stream);
}
