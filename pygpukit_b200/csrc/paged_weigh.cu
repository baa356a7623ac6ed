// paged_weigh.cu -- the attention weights that a cached position gets, summed over a step's rows and the query heads of its key head: what decides which positions of a
// cache stay when it is cut.  weights[slot][g][j] += sum over rows i and heads h of g of exp(scale q_ih . k_j - lse_ih), lse from the attention over the same rows.
//
// Scores by mma.sync m16n8k16 with the keys as its 16, as in paged_few.cu, in float32 by multiply-adds.  A block has the step's rows in shared memory (all of them, or as many
// as fit at a time) and a share of the positions; a warp walks over its own 16 by 16, the next on their way from memory to registers meanwhile.  A
// position's sum is one thread's until it is added, so that the same call gives the same bits.  Decoding is bound by the bytes of the keys, windows of a prompt's last tokens by
// products and exponentials.
#include "paged.cuh"
#include "tc_common.cuh"
#include "../../include/pgk_b200.h"

namespace pgk {

namespace {

constexpr int H_ALL = 1 << 30;                                // rows of a "block": all of the sequence's
constexpr int H_WARPS = 4, H_THREADS = H_WARPS * 32, H_KEYS = 16, H_RESIDENT = 4;
constexpr int H_QBYTES = 48 * 1024;                           // queries of a block at a time: four blocks a SM
constexpr int G_WARPS = 4, G_THREADS = G_WARPS * 32, G_KEYS = G_WARPS * 32, G_ROWS = 16;

using Keys = PagedBlock<H_ALL, H_KEYS>;

template <int DT>
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (DT == 1)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// minus a row's logarithm (log2): -infinity for rows that do not exist or see nothing
__device__ __forceinline__ float row_neg(const PagedParams& p, const Keys& b, int r) {
    const int tok = b.token(p, r);
    if (r >= b.live || tok < 0 || tok >= p.tokens) return -INFINITY;
    const float z = __ldcg(p.lse + (size_t)tok * p.heads + b.head * p.rep + r % p.rep);
    return z == -INFINITY ? -INFINITY : -z * PAGED_LOG2E;
}
__device__ __forceinline__ float weight(float s, float scale, float neg) { return neg == -INFINITY ? 0.f : ex2(fmaf(s, scale, neg)); }
__device__ __forceinline__ void add_weight(const PagedParams& p, const Keys& b, int j, float w) {
    atomicAdd(p.weights + ((size_t)b.slot * p.kv_heads + b.head) * p.weights_ld + j, w);
}

// N: 32-element pieces of a head
template <int N, int DT>
__global__ void __launch_bounds__(H_THREADS, N <= 4 ? H_RESIDENT : 2) paged_weigh_kernel(const __grid_constant__ PagedParams p, int most) {
    extern __shared__ __align__(16) unsigned char smem[];
    uint4* const qs = (uint4*)smem;                           // [tiles of eight rows][N][32]: lane (gl, t)'s elements 32 s + 8 t ... + 7 of row 8 n + gl
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), gl = lane >> 2, t = lane & 3, D = p.dim;
    griddep_wait();
    griddep_launch();
    const Keys b(p, (int)blockIdx.z, (int)blockIdx.y, (int)blockIdx.x);
    float* const negs = (float*)(qs + (size_t)most * N * 32);
    if (b.ubeg >= b.uend || b.live == 0) return;

    const char* const kb = (const char*)p.k_data;
    const size_t stride = (size_t)D * 2;
    uint4 kk[N][2], ahead[N][2];
    auto load_k = [&](int rows, uint4 (&x)[N][2]) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int row = __shfl_sync(0xffffffffu, rows, 8 * u + gl);
            const char* const src = kb + (size_t)max(row, 0) * stride + 16 * t;
#pragma unroll
            for (int s = 0; s < N; ++s) {
                x[s][u] = make_uint4(0, 0, 0, 0);
                if (row >= 0 && 32 * s + 8 * t < D) x[s][u] = ld_act16(src + 64 * s);
            }
        }
    };
    auto look = [&](int k) { return k < b.uend ? b.row_of(p, k * H_KEYS + (lane & 15)) : -1; };
#pragma unroll 1
    for (int f0 = 0; f0 < b.live; f0 += 8 * most) {
        const int tiles = min(most, (b.live - f0 + 7) / 8);
        int k = b.ubeg + warp, rows = look(k), next = look(k + H_WARPS);
        load_k(rows, kk);
        if (f0 > 0) __syncthreads();
        for (int i = warp; i < tiles * N; i += H_WARPS) {
            const int n = i / N, s = i - n * N, x = f0 + 8 * n + gl, d = 32 * s + 8 * t, row = x / p.rep, tok = b.first + row;
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
            qs[i * 32 + lane] = v;
        }
        for (int i = tid; i < 8 * tiles; i += H_THREADS) negs[i] = row_neg(p, b, f0 + i);
        __syncthreads();
#pragma unroll 1
        for (; k < b.uend; k += H_WARPS) {
            const int j0 = k * H_KEYS;
            const uint32_t there = __ballot_sync(0xffffffffu, rows >= 0);
            const bool edge = (there & 0xffffu) != 0xffffu || j0 + H_KEYS > b.base;
            rows = next;
            load_k(rows, ahead);
            next = look(k + 2 * H_WARPS);
            float sum0 = 0.f, sum1 = 0.f;                     // of keys gl and gl + 8: this lane's rows
#pragma unroll 1
            for (int n = 0; n < tiles; ++n) {
                float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int q = 0; q < N; ++q) {
                    const uint4 a = qs[(n * N + q) * 32 + lane];
                    mma16816<DT>(s, kk[q][0].x, kk[q][1].x, kk[q][0].y, kk[q][1].y, a.x, a.y);
                    mma16816<DT>(s, kk[q][0].z, kk[q][1].z, kk[q][0].w, kk[q][1].w, a.z, a.w);
                }
                const float2 neg = *(const float2*)(negs + 8 * n + 2 * t);
                const float w0 = weight(s[0], p.scale_log2, neg.x), w1 = weight(s[1], p.scale_log2, neg.y), w2 = weight(s[2], p.scale_log2, neg.x),
                            w3 = weight(s[3], p.scale_log2, neg.y);
                if (edge) {
                    const int i0 = (f0 + 8 * n + 2 * t) / p.rep, i1 = (f0 + 8 * n + 2 * t + 1) / p.rep, at = j0 - b.base;
                    const uint32_t see0 = paged_window(p, b.first + i0, i0, at) & there, see1 = paged_window(p, b.first + i1, i1, at) & there;
                    sum0 += ((see0 >> gl) & 1u ? w0 : 0.f) + ((see1 >> gl) & 1u ? w1 : 0.f);
                    sum1 += ((see0 >> (gl + 8)) & 1u ? w2 : 0.f) + ((see1 >> (gl + 8)) & 1u ? w3 : 0.f);
                } else {
                    sum0 += w0 + w1;
                    sum1 += w2 + w3;
                }
            }
#pragma unroll
            for (int x = 1; x <= 2; x <<= 1) {
                sum0 += __shfl_xor_sync(0xffffffffu, sum0, x);
                sum1 += __shfl_xor_sync(0xffffffffu, sum1, x);
            }
            const int j = j0 + gl + 8 * t;                    // lanes 0 and 1 of a group write
            if (t < 2 && j < b.end) add_weight(p, b, j, t ? sum1 : sum0);
#pragma unroll
            for (int s = 0; s < N; ++s) { kk[s][0] = ahead[s][0]; kk[s][1] = ahead[s][1]; }
        }
    }
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
            const int r = i / D, f = f0 + r, row = f / p.rep, tok = b.first + row;
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
                const float w = weight(s[r], p.scale_log2, negs[r0 + r]);
                bool sees = true;
                if (edge) {
                    const int i = (f0 + r0 + r) / p.rep;
                    sees = rows >= 0 && (j < b.base || paged_sees(p, b.first + i, i, j - b.base));
                }
                if (sees) sum += w;
            }
        }
    }
    if (j < b.end) add_weight(p, b, j, sum);
}

template <int N, int DT> int launch_weigh(PagedParams p, cudaStream_t st) {
    static bool configured = false;
    if (!configured) {
        PGK_CUDA(cudaFuncSetAttribute(paged_weigh_kernel<N, DT>, cudaFuncAttributeMaxDynamicSharedMemorySize, H_QBYTES));
        configured = true;
    }
    // tiles of eight rows that fit, and blocks that share a sequence's positions: four rounds of all SMs, none with less than two turns of its warps
    const long long tiles = ((long long)p.max_rows * p.rep + 7) / 8, fit = H_QBYTES / (N * 512 + 32);
    const int most = (int)(tiles < fit ? tiles : fit);
    const long long items = (long long)p.kv_heads * p.seqs, wanted = (4ll * H_RESIDENT * sm_count() + items - 1) / items, turns = (p.max_keys + 2 * H_WARPS * H_KEYS - 1) / (2 * H_WARPS * H_KEYS);
    p.splits = (int)(wanted < turns ? wanted : turns);
    PGK_CUDA(launch_waiting(paged_weigh_kernel<N, DT>, dim3(p.splits, p.kv_heads, p.seqs), dim3(H_THREADS), (size_t)most * (N * 512 + 32), st, p, most));
    return 0;
}
template <int DT> int launch_weigh_dim(const PagedParams& p, cudaStream_t st) {
    switch ((p.dim + 31) / 32) {
        case 1: case 2: return launch_weigh<2, DT>(p, st);
        case 3: return launch_weigh<3, DT>(p, st);
        case 4: return launch_weigh<4, DT>(p, st);
        case 5: case 6: return launch_weigh<6, DT>(p, st);
        default: return launch_weigh<8, DT>(p, st);
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
    if (page_size > 1) {                                      // log: the least with page_size <= 2^log
        uint32_t log = 0;
        while ((1ull << log) < (uint64_t)page_size) ++log;
        p.page_shift = log - 1;
        p.page_mul = (uint32_t)((1ull << (31 + log)) / (uint64_t)page_size + 1);
    }
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
