// paged_f32.cu -- attention over pages of 32 bits: products and sums are float32, nothing is rounded between.
//
// A block has R (row, head) rows (4, 8 or 16: as many as a token's heads need), each of its warps walks over its own blocks of 32 keys, whose K and V it fetches to
// shared memory by itself, K of the next block while this one's values are summed and V while its scores are formed.  Scores: a lane a key, the queries' elements are
// broadcast; values: a lane four neighbouring elements (and four 128 on), the weights are broadcast.  Products are
// pairs of float32 in one instruction.  Few rows are bound by the instructions that fetch and the chain of a turn, trees by the multiply-adds and what feeds them.  Blocks of a cluster share a sequence's keys.
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
    static int warp_floats(int D) { return S_KEYS * (D + 4) + S_KEYS * D + 2 * R * S_KEYS; }
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
    float* const ks = qs + R * D + warp * (S_KEYS * DF + S_KEYS * D + 2 * R * S_KEYS);
    float* const vs = ks + S_KEYS * DF;
    float2* const ps = (float2*)(vs + S_KEYS * D);            // [R][32], each weight twice
    if (tid == 0) f.bad = 0;
    griddep_wait();
    griddep_launch();
    const PagedBlock<R, S_KEYS> b(p, (int)blockIdx.x, (int)blockIdx.y, (int)blockIdx.z);

    auto fetch = [&](const void* base, float* to, int ld, int rows) {
        const float* const src = (const float*)base + 4 * (D4 <= 16 ? lane & 15 : lane);
        if (D4 <= 16) {                                       // two keys at a time
            float* dst = to + (lane >> 4) * ld + 4 * (lane & 15);
#pragma unroll 8
            for (int r = 0; r < S_KEYS; r += 2, dst += 2 * ld) {
                const int row = __shfl_sync(0xffffffffu, rows, r + (lane >> 4));
                if ((lane & 15) < D4) cp_async16_or_zero(dst, src + (size_t)max(row, 0) * D, row >= 0);
            }
        } else {
            float* dst = to + 4 * lane;
#pragma unroll 8
            for (int r = 0; r < S_KEYS; ++r, dst += ld) {
                const int row = __shfl_sync(0xffffffffu, rows, r);
                const float* const from = src + (size_t)max(row, 0) * D;
#pragma unroll
                for (int c = 0; c < PC; ++c)
                    if (lane + 32 * c < D4) cp_async16_or_zero(dst + 128 * c, from + 128 * c, row >= 0);
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

    uint64_t o[R][PC][2];                                     // pairs of elements
    float m_r = -INFINITY, nm[R], l[R];                      // lane r keeps row r's reference
#pragma unroll
    for (int r = 0; r < R; ++r) {
        nm[r] = l[r] = 0.f;
#pragma unroll
        for (int c = 0; c < PC; ++c) o[r][c][0] = o[r][c][1] = pair(0.f, 0.f);
    }
    bool bad = false;
#pragma unroll 1
    for (; k < b.uend; k += W) {
        const int j0 = k * S_KEYS, next = k + W < b.uend ? b.row_of(p, (k + W) * S_KEYS + lane) : -1;
        cp_async_wait<1>();                                   // K is here
        __syncwarp();
        uint64_t s2[R];
#pragma unroll
        for (int r = 0; r < R; ++r) s2[r] = pair(0.f, 0.f);
        const float* const kr = ks + lane * DF;
#pragma unroll 4
        for (int c = 0; c < D4; ++c) {
            const ulonglong2 x = *(const ulonglong2*)(kr + 4 * c);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const ulonglong2 q = *(const ulonglong2*)(qs + r * D + 4 * c);
                s2[r] = fma2(q.x, x.x, s2[r]);
                s2[r] = fma2(q.y, x.y, s2[r]);
            }
        }
        __syncwarp();
        if (k + W < b.uend) fetch(p.k_data, ks, DF, next);
        else cp_async_commit();
        const bool edge = __any_sync(0xffffffffu, rows < 0) || j0 + S_KEYS > b.base;
        const int at = j0 - b.base;
        float s[R], v[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float a, c;
            unpair(s2[r], a, c);
            s[r] = (a + c) * p.scale_log2;
            if (edge) {
                const int i = (b.f0 + r) / p.rep, t = at + lane;
                if (rows < 0 || r >= b.live || (t >= 0 && !paged_sees(p, b.first + i, i, t))) s[r] = -INFINITY;
            }
            v[r] = s[r];
        }
        const float top = reduce_lanes<R>(v, lane, [](float x, float y) { return fmaxf(x, y); });
        const bool up = top > m_r + PAGED_LAZY;               // (also the first finite maximum)
        if (__any_sync(0xffffffffu, up)) {
            const float f_r = !up ? 1.f : (m_r == -INFINITY ? 0.f : exp2f(m_r - top));
            if (up) m_r = top;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const float fix = __shfl_sync(0xffffffffu, f_r, r);
                nm[r] = paged_neg(__shfl_sync(0xffffffffu, m_r, r));
                l[r] *= fix;
#pragma unroll
                for (int c = 0; c < PC; ++c) { o[r][c][0] = mul2(o[r][c][0], pair(fix, fix)); o[r][c][1] = mul2(o[r][c][1], pair(fix, fix)); }
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const float w = ex2(s[r] + nm[r]);
            l[r] += w;
            ps[r * S_KEYS + lane] = make_float2(w, w);
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
                    const ulonglong2 w0 = *(const ulonglong2*)(ps + r * S_KEYS + key), w1 = *(const ulonglong2*)(ps + r * S_KEYS + key + 2);
                    const uint64_t w[4] = {w0.x, w0.y, w1.x, w1.y};
#pragma unroll
                    for (int u = 0; u < 4; ++u)
#pragma unroll
                        for (int c = 0; c < PC; ++c) {
                            o[r][c][0] = fma2(w[u], pair(v[u][c].x, v[u][c].y), o[r][c][0]);
                            o[r][c][1] = fma2(w[u], pair(v[u][c].z, v[u][c].w), o[r][c][1]);
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
    if (lane < R) wm[warp][lane] = m_r;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        l[r] = warp_sum(l[r]);
        if (lane == 0) wl[warp][r] = l[r];
    }
    __syncthreads();
    float* const fold = smf;                                  // [W][R][FS]
    constexpr int FS = 128 * PC + 4;
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int c = 0; c < PC; ++c)
            if (lane + 32 * c < D4) *(ulonglong2*)(fold + (warp * R + r) * FS + 4 * (lane + 32 * c)) = make_ulonglong2(o[r][c][0], o[r][c][1]);
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
    const int smem = Single<R, PC, W>::bytes(p.dim), kind = smem > 113 * 1024 ? 0 : (smem > 75 * 1024 ? 1 : 2);       // one, two, three blocks a SM
    static int at_once[3][PAGED_CLUSTER + 1] = {};
    if (at_once[kind][1] == 0)
        for (int i = 1; i <= PAGED_CLUSTER; ++i) PGK_CUDA(clusters_at_once(&at_once[kind][i], paged_f32_kernel<R, PC, W>, W * 32, (size_t)smem, i));
    p.tiles = (int)(((long long)p.max_rows * p.rep + R - 1) / R);
    p.splits = paged_clusters(p, S_KEYS * W, at_once[kind], PAGED_CLUSTER, 2);
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
