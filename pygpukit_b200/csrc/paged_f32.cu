// paged_f32.cu -- attention over pages of 32 bits: products and sums are float32, nothing is rounded between.
//
// A block has R (row, head) rows (4, 8 or 16: as many as a token's heads need), each of its warps walks over its own blocks of 32 keys, whose K and V it fetches to
// shared memory by itself, K of the next block while this one's values are summed and V while its scores are formed.  Scores: a lane a key, the queries' elements are
// broadcast; values: a lane four neighbouring elements (and four 128 on), the weights are broadcast.  A row costs 2 instructions' issue a key and
// element quartet beside the loads, so that few rows are bound by the cache's bytes and trees by the multiply-adds.  Blocks of a cluster share a sequence's keys.
#include <type_traits>

#include "paged.cuh"
#include "tc_common.cuh"
#include "../../include/pgk_b200.h"

namespace pgk {

namespace {

constexpr int S_KEYS = 32;

__device__ __forceinline__ void cp_async16_or_zero(void* dst, const void* src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" :: "r"(smem_u32(dst)), "l"(src), "r"(there ? 16u : 0u) : "memory");
}

// PC: quartets of elements a lane has of an output row; W: warps
template <int R, int PC, int W> struct Single {
    static int warp_floats(int D) { return S_KEYS * (D + 4) + S_KEYS * D + R * S_KEYS; }
    static int bytes(int D) {
        const int run = (R * D + W * warp_floats(D)) * 4, fold = W * R * (128 * PC + 4) * 4;
        return run > fold ? run : fold;
    }
};

template <int R, int PC, int W>
__global__ void __launch_bounds__(W * 32, 1) paged_f32_kernel(const __grid_constant__ PagedParams p) {
    extern __shared__ __align__(16) float smf[];
    __shared__ float wm[W][R], wl[W][R];
    __shared__ PagedFold<R> f;
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), D = p.dim, D4 = D / 4, DF = D + 4;
    float* const qs = smf;                                    // [R][D]
    float* const ks = qs + R * D + warp * (S_KEYS * DF + S_KEYS * D + R * S_KEYS);
    float* const vs = ks + S_KEYS * DF;
    float* const ps = vs + S_KEYS * D;                        // [R][32]
    if (tid == 0) f.bad = 0;
    griddep_wait();
    griddep_launch();
    const PagedBlock<R, S_KEYS> b(p, (int)blockIdx.x, (int)blockIdx.y, (int)blockIdx.z);

    auto fetch = [&](const void* base, float* to, int ld, int rows) {
        const float* const src = (const float*)base;
        if (D4 <= 16) {                                       // two keys at a time
            for (int r = 0; r < S_KEYS; r += 2) {
                const int key = r + (lane >> 4), c = lane & 15, row = __shfl_sync(0xffffffffu, rows, key);
                if (c < D4) cp_async16_or_zero(to + key * ld + 4 * c, src + (size_t)max(row, 0) * D + 4 * c, row >= 0);
            }
        } else {
            for (int r = 0; r < S_KEYS; ++r) {
                const int row = __shfl_sync(0xffffffffu, rows, r);
                for (int c = lane; c < D4; c += 32) cp_async16_or_zero(to + r * ld + 4 * c, src + (size_t)max(row, 0) * D + 4 * c, row >= 0);
            }
        }
        cp_async_commit();
    };
    int k = b.ubeg + warp;
    int rows = k < b.uend ? b.row_of(p, k * S_KEYS + lane) : -1;
    if (k < b.uend) {
        fetch(p.k_data, ks, DF, rows);
        fetch(p.v_data, vs, D, rows);
    }
    for (int i = tid; i < R * D; i += W * 32) {
        const int r = i / D, x = b.f0 + r, tok = b.first + x / p.rep;
        qs[i] = r < b.live && tok >= 0 && tok < p.tokens ? __ldcg((const float*)p.q + (size_t)tok * p.q_ld + (size_t)(b.head * p.rep + x % p.rep) * D + (i - r * D)) : 0.f;
    }
    __syncthreads();

    float4 o[R][PC];
    float m[R], l[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        m[r] = -INFINITY;
        l[r] = 0.f;
#pragma unroll
        for (int c = 0; c < PC; ++c) o[r][c] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    bool bad = false;
#pragma unroll 1
    for (; k < b.uend; k += W) {
        const int j0 = k * S_KEYS, next = k + W < b.uend ? b.row_of(p, (k + W) * S_KEYS + lane) : -1;
        cp_async_wait<1>();                                   // K is here
        __syncwarp();
        float s[R];
#pragma unroll
        for (int r = 0; r < R; ++r) s[r] = 0.f;
        const float* const kr = ks + lane * DF;
#pragma unroll 2
        for (int c = 0; c < D4; ++c) {
            const float4 x = *(const float4*)(kr + 4 * c);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const float4 q = *(const float4*)(qs + r * D + 4 * c);
                s[r] = fmaf(q.x, x.x, fmaf(q.y, x.y, fmaf(q.z, x.z, fmaf(q.w, x.w, s[r]))));
            }
        }
        __syncwarp();
        if (k + W < b.uend) fetch(p.k_data, ks, DF, next);
        else cp_async_commit();
        const bool edge = __any_sync(0xffffffffu, rows < 0) || j0 + S_KEYS > b.base;
        const int at = j0 - b.base;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float x = s[r] * p.scale_log2;
            if (edge) {
                const int i = (b.f0 + r) / p.rep, t = at + lane;
                if (rows < 0 || r >= b.live || (t >= 0 && !paged_sees(p, b.first + i, i, t))) x = -INFINITY;
            }
            const float top = warp_max(x);
            if (top > m[r] + PAGED_LAZY) {                    // the same in all lanes; also the first finite maximum
                const float fix = m[r] == -INFINITY ? 0.f : exp2f(m[r] - top);
                m[r] = top;
                l[r] *= fix;
#pragma unroll
                for (int c = 0; c < PC; ++c) { o[r][c].x *= fix; o[r][c].y *= fix; o[r][c].z *= fix; o[r][c].w *= fix; }
            }
            const float w = ex2(x + paged_neg(m[r]));
            l[r] += w;
            ps[r * S_KEYS + lane] = w;
        }
        cp_async_wait<1>();                                   // V is here
        __syncwarp();
        auto values = [&](auto step) {
#pragma unroll 1
            for (int key = 0; key < S_KEYS; key += 4) {
                float4 v[4][PC];
#pragma unroll
                for (int u = 0; u < 4; ++u)
#pragma unroll
                    for (int c = 0; c < PC; ++c) {
                        v[u][c] = lane + 32 * c < D4 ? *(const float4*)(vs + (key + u) * D + 4 * (lane + 32 * c)) : make_float4(0.f, 0.f, 0.f, 0.f);
                        if constexpr (step.value)
                            if (at + key + u >= 0) {          // values of the step's rows, which not all rows see
                                float* const x = &v[u][c].x;
#pragma unroll
                                for (int e = 0; e < 4; ++e)
                                    if (!(fabsf(x[e]) < INFINITY)) { bad = true; x[e] = 0.f; }
                            }
                    }
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const float4 w = *(const float4*)(ps + r * S_KEYS + key);
                    const float wu[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                    for (int u = 0; u < 4; ++u)
#pragma unroll
                        for (int c = 0; c < PC; ++c) {
                            o[r][c].x = fmaf(wu[u], v[u][c].x, o[r][c].x); o[r][c].y = fmaf(wu[u], v[u][c].y, o[r][c].y);
                            o[r][c].z = fmaf(wu[u], v[u][c].z, o[r][c].z); o[r][c].w = fmaf(wu[u], v[u][c].w, o[r][c].w);
                        }
                }
            }
        };
        if (at + S_KEYS > 0) values(std::true_type{});
        else values(std::false_type{});
        __syncwarp();
        rows = next;
        if (k + W < b.uend) fetch(p.v_data, vs, D, rows);
        else cp_async_commit();
    }
    cp_async_wait<0>();

    // ---------------- the warps' sums into one
    if (bad) f.bad = 1;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        l[r] = warp_sum(l[r]);
        if (lane == 0) { wm[warp][r] = m[r]; wl[warp][r] = l[r]; }
    }
    __syncthreads();
    float* const fold = smf;                                  // [W][R][FS]
    constexpr int FS = 128 * PC + 4;
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int c = 0; c < PC; ++c)
            if (lane + 32 * c < D4) *(float4*)(fold + (warp * R + r) * FS + 4 * (lane + 32 * c)) = o[r][c];
    __syncthreads();
    if (tid < R) {
        float top = -INFINITY, sum = 0.f;
        for (int w = 0; w < W; ++w) top = fmaxf(top, wm[w][tid]);
        for (int w = 0; w < W; ++w) {
            const float x = wm[w][tid] == -INFINITY ? wl[w][tid] - wl[w][tid] : exp2f(wm[w][tid] - top);
            sum = fmaf(wl[w][tid], x, sum);
            wm[w][tid] = x;
        }
        f.m[tid] = top;
        f.l[tid] = sum;
    }
    __syncthreads();
    for (int i = tid; i < b.live * D4; i += W * 32) {
        const int r = i / D4, d = (i - r * D4) * 4;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int w = 0; w < W; ++w) {
            const float y = wm[w][r];
            const float4 v = *(const float4*)(fold + (w * R + r) * FS + d);
            x.x = fmaf(y, v.x, x.x); x.y = fmaf(y, v.y, x.y); x.z = fmaf(y, v.z, x.z); x.w = fmaf(y, v.w, x.w);
        }
        *(float4*)(fold + r * FS + d) = x;
    }
    paged_fold<R, S_KEYS, 0, 128 * PC>(p, b, fold, f);
}

template <int R, int PC, int W>
int launch_single(PagedParams p, cudaStream_t st) {
    static bool configured = false;
    if (!configured) {
        PGK_CUDA(cudaFuncSetAttribute(paged_f32_kernel<R, PC, W>, cudaFuncAttributeMaxDynamicSharedMemorySize, Single<R, PC, W>::bytes(128 * PC)));
        PGK_CUDA(cudaFuncSetAttribute(paged_f32_kernel<R, PC, W>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        configured = true;
    }
    const int smem = Single<R, PC, W>::bytes(p.dim), resident = smem > 110 * 1024 ? 1 : (smem > 72 * 1024 ? 2 : 3);
    p.tiles = (int)(((long long)p.max_rows * p.rep + R - 1) / R);
    p.splits = paged_cut(p, (long long)p.seqs * p.tiles * p.kv_heads, S_KEYS, W, resident, 3.f, PAGED_CLUSTER);
    PGK_CUDA(launch_clusters(paged_f32_kernel<R, PC, W>, dim3((unsigned)(p.seqs * p.tiles), p.kv_heads, p.splits), W * 32, (size_t)smem, st, p));
    return 0;
}

}  // namespace

int paged_f32(const PagedParams& p, cudaStream_t st) {
    const long long rows = (long long)p.max_rows * p.rep;
    if (p.dim > 128) return rows <= 4 ? launch_single<4, 2, 2>(p, st) : launch_single<8, 2, 2>(p, st);
    if (rows <= 4) return launch_single<4, 1, 4>(p, st);
    return rows <= 8 ? launch_single<8, 1, 4>(p, st) : launch_single<16, 1, 4>(p, st);
}

}  // namespace pgk
