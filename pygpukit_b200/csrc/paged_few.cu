// paged_few.cu -- attention of few rows a sequence over 16-bit pages: decoded tokens, small trees of drafts, and whatever the large tiles of paged_tc.cu do not serve
// (heads above 128 elements, pages that no copy of eight positions fits).
//
// One pass over the keys with the running maximum and sum of a softmax.  A block has 16 (row, head) rows, each of its warps walks over its own blocks of 16 keys:
// S = Q K^T and O += P V by mma.sync m16n8k16, K and V straight from memory to registers, sixteen bytes a lane.  The order of a head's elements in the score's sum is free, so a
// lane takes the eight that follow each other in one key; V wants pairs of keys in a register, which byte permutations of two keys' loads make.  Keys of a block of
// 16 are on their way while those before are multiplied; weights are rounded to the cache's type once (bfloat16 2^-9 of each, independent from key to key, beside
// the output's own 2^-9), their sum is float32 of the unrounded ones.  Blocks of a cluster share a sequence's keys and fold through distributed shared memory.
// Bound by the bytes of the keys and, for one request, by the chain from launch to fold.
#include "paged.cuh"
#include "tc_common.cuh"
#include "../../include/pgk_b200.h"

namespace pgk {

namespace {

constexpr int W_KEYS = 16, W_WARPS = 4, W_THREADS = W_WARPS * 32, W_ROWS = 16;

// sixteen bytes of the cache, each read once by a block
__device__ __forceinline__ uint4 ld_cache16(const void* p) {
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
template <int DT>
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (DT == 1)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// N: 32-element pieces of a head
template <int N> struct Few {
    static constexpr int DP = 32 * N, CH = (DP + 63) / 64, DF = DP + 4;
    static constexpr int QBYTES = N * 2 * 32 * 16, FOLD = W_WARPS * W_ROWS * DF * 4, BYTES = QBYTES > FOLD ? QBYTES : FOLD;
    static constexpr int RESIDENT = N <= 2 ? 4 : (N <= 4 ? 3 : 2);
};

template <int N, int DT>
__global__ void __launch_bounds__(W_THREADS, Few<N>::RESIDENT) paged_few_kernel(const __grid_constant__ PagedParams p) {
    using F = Few<N>;
    constexpr int CH = F::CH;
    // float16 weights: from 2^6 down, so that those 2^-20 of the largest still have all their bits; they grow to 2^14 before the reference moves
    constexpr float TOP = DT == 1 ? 6.f : 0.f;
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ float wm[W_WARPS][W_ROWS], wl[W_WARPS][W_ROWS], row_m[W_ROWS], row_l[W_ROWS];
    __shared__ int flag;
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), gl = lane >> 2, t = lane & 3;
    if (tid == 0) flag = 0;
    griddep_wait();
    griddep_launch();
    const PagedBlock<W_ROWS, W_KEYS> b(p, (int)blockIdx.x, (int)blockIdx.y, (int)blockIdx.z);
    const int D = p.dim;

    // ---------------- queries: piece s, half r: this lane's eight elements 32 s + 8 t of row gl + 8 r
    uint4* const qs = (uint4*)smem;
    for (int i = warp; i < 2 * N; i += W_WARPS) {
        const int r = gl + 8 * (i & 1), d = 32 * (i >> 1) + 8 * t;
        uint4 v = make_uint4(0, 0, 0, 0);
        const int f = b.f0 + r, tok = b.first + f / p.rep;
        if (r < b.live && d < D && tok >= 0 && tok < p.tokens) {
            const uint16_t* src = (const uint16_t*)p.q + (size_t)tok * p.q_ld + (size_t)(b.head * p.rep + f % p.rep) * D + d;
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
    __syncthreads();

    float o[CH][8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[c][j][e] = 0.f;
    const int row0 = (b.f0 + gl) / p.rep, row1 = (b.f0 + gl + 8) / p.rep;         // the step's rows of this lane's two
    const char* const kb = (const char*)p.k_data;
    const char* const vb = (const char*)p.v_data;
    const size_t stride = (size_t)D * 2;
    bool bad = false;

    uint4 kk[N][2];
    auto load_k = [&](int rows) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int row = __shfl_sync(0xffffffffu, rows, 8 * u + gl);
            const char* const src = kb + (size_t)max(row, 0) * stride + 16 * t;
#pragma unroll
            for (int s = 0; s < N; ++s) {
                kk[s][u] = make_uint4(0, 0, 0, 0);
                if (row >= 0 && 32 * s + 8 * t < D) kk[s][u] = ld_cache16(src + 64 * s);
            }
        }
    };
    int k = b.ubeg + warp;
    int rows = k < b.uend ? b.row_of(p, k * W_KEYS + (lane & 15)) : -1;
    int next = k + W_WARPS < b.uend ? b.row_of(p, (k + W_WARPS) * W_KEYS + (lane & 15)) : -1;
    if (k < b.uend) load_k(rows);
#pragma unroll 1
    for (; k < b.uend; k += W_WARPS) {
        const int j0 = k * W_KEYS;
        // values of keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9: eight elements from 64 c + 8 gl on
        uint4 vv[CH][4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int row = __shfl_sync(0xffffffffu, rows, 2 * t + (u & 1) + 8 * (u >> 1));
            const char* const src = vb + (size_t)max(row, 0) * stride + 16 * gl;
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                vv[c][u] = make_uint4(0, 0, 0, 0);
                if (row >= 0 && 64 * c + 8 * gl < D) vv[c][u] = ld_cache16(src + 128 * c);
            }
        }
        float s[2][4] = {};
#pragma unroll
        for (int q = 0; q < N; ++q) {
            const uint4 a = qs[(2 * q) * 32 + lane], c = qs[(2 * q + 1) * 32 + lane];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                mma16816<DT>(s[u], a.x, c.x, a.y, c.y, kk[q][u].x, kk[q][u].y);
                mma16816<DT>(s[u], a.z, c.z, a.w, c.w, kk[q][u].z, kk[q][u].w);
            }
        }
        const uint32_t there = __ballot_sync(0xffffffffu, rows >= 0);
        const bool edge = (there & 0xffffu) != 0xffffu || j0 + W_KEYS > b.base;
        rows = next;
        if (k + W_WARPS < b.uend) load_k(rows);
        next = k + 2 * W_WARPS < b.uend ? b.row_of(p, (k + 2 * W_WARPS) * W_KEYS + (lane & 15)) : -1;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[u][e] *= p.scale_log2;
        if (edge) {
            const int at = j0 - b.base;                       // the step's row of the block's first key, below 0 before the step
            const uint32_t see0 = paged_window(p, b.first + row0, row0, at) & there, see1 = paged_window(p, b.first + row1, row1, at) & there;
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int bit = 8 * u + 2 * t + e;
                    if (!((see0 >> bit) & 1u)) s[u][e] = -INFINITY;
                    if (!((see1 >> bit) & 1u)) s[u][2 + e] = -INFINITY;
                }
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (at + 2 * t + (u & 1) + 8 * (u >> 1) >= 0) {            // values of the step's rows, which not all rows see
#pragma unroll
                    for (int c = 0; c < CH; ++c) {
                        uint32_t* const w = &vv[c][u].x;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const uint32_t x = paged_unfinite<DT>(w[e]);
                            bad |= x != 0;
                            w[e] &= ~x;
                        }
                    }
                }
        }
        float top0 = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[1][0], s[1][1])), top1 = fmaxf(fmaxf(s[0][2], s[0][3]), fmaxf(s[1][2], s[1][3]));
#pragma unroll
        for (int x = 1; x <= 2; x <<= 1) {
            top0 = fmaxf(top0, __shfl_xor_sync(0xffffffffu, top0, x));
            top1 = fmaxf(top1, __shfl_xor_sync(0xffffffffu, top1, x));
        }
        top0 -= TOP;
        top1 -= TOP;
        const bool up0 = top0 > m[0] + PAGED_LAZY, up1 = top1 > m[1] + PAGED_LAZY;          // (also the first finite maximum)
        if (__any_sync(0xffffffffu, up0 || up1)) {
            const float f0 = !up0 ? 1.f : (m[0] == -INFINITY ? 0.f : exp2f(m[0] - top0)), f1 = !up1 ? 1.f : (m[1] == -INFINITY ? 0.f : exp2f(m[1] - top1));
            if (up0) m[0] = top0;
            if (up1) m[1] = top1;
            l[0] *= f0;
            l[1] *= f1;
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    o[c][j][0] *= f0; o[c][j][1] *= f0;
                    o[c][j][2] *= f1; o[c][j][3] *= f1;
                }
        }
        const float n0 = paged_neg(m[0]), n1 = paged_neg(m[1]);
        uint32_t a[4];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const float w0 = ex2(s[u][0] + n0), w1 = ex2(s[u][1] + n0), w2 = ex2(s[u][2] + n1), w3 = ex2(s[u][3] + n1);
            l[0] += w0 + w1;
            l[1] += w2 + w3;
            a[2 * u] = paged_pack2<DT>(w0, w1);
            a[2 * u + 1] = paged_pack2<DT>(w2, w3);
        }
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const uint32_t* const v0 = &vv[c][0].x;
            const uint32_t* const v1 = &vv[c][1].x;
            const uint32_t* const v2 = &vv[c][2].x;
            const uint32_t* const v3 = &vv[c][3].x;
#pragma unroll
            for (int j = 0; j < 8; ++j) {                     // element 64 c + 8 gl + j of the key pairs
                const uint32_t sel = j & 1 ? 0x7632u : 0x5410u;
                mma16816<DT>(o[c][j], a[0], a[1], a[2], a[3], __byte_perm(v0[j >> 1], v1[j >> 1], sel), __byte_perm(v2[j >> 1], v3[j >> 1], sel));
            }
        }
    }

    // ---------------- the warps' sums into one: column n of o[c][j] is element 64 c + 8 n + j
    if (bad) flag = 1;
#pragma unroll
    for (int x = 1; x <= 2; x <<= 1) {
        l[0] += __shfl_xor_sync(0xffffffffu, l[0], x);
        l[1] += __shfl_xor_sync(0xffffffffu, l[1], x);
    }
    if (t == 0) {
        wm[warp][gl] = m[0]; wm[warp][gl + 8] = m[1];
        wl[warp][gl] = l[0]; wl[warp][gl + 8] = l[1];
    }
    __syncthreads();                                          // the queries are read
    float* const fold = (float*)smem;
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int r = gl + 8 * (e >> 1), d = 64 * c + 16 * t + 8 * (e & 1);
            if (d < F::DP) {
                float* const dst = fold + ((size_t)warp * W_ROWS + r) * F::DF + d;
                *(float4*)dst = make_float4(o[c][0][e], o[c][1][e], o[c][2][e], o[c][3][e]);
                *(float4*)(dst + 4) = make_float4(o[c][4][e], o[c][5][e], o[c][6][e], o[c][7][e]);
            }
        }
    __syncthreads();
    if (tid < W_ROWS) {
        float top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int w = 0; w < W_WARPS; ++w) top = fmaxf(top, wm[w][tid]);
#pragma unroll
        for (int w = 0; w < W_WARPS; ++w) {
            const float f = wm[w][tid] == -INFINITY ? wl[w][tid] - wl[w][tid] : exp2f(wm[w][tid] - top);
            sum = fmaf(wl[w][tid], f, sum);
            wm[w][tid] = f;
        }
        row_m[tid] = top;
        row_l[tid] = sum;
    }
    __syncthreads();
    for (int i = tid; i < b.live * (F::DP / 4); i += W_THREADS) {
        const int r = i / (F::DP / 4), d = (i - r * (F::DP / 4)) * 4;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < W_WARPS; ++w) {
            const float f = wm[w][r];
            const float4 v = *(const float4*)(fold + ((size_t)w * W_ROWS + r) * F::DF + d);
            x.x = fmaf(f, v.x, x.x); x.y = fmaf(f, v.y, x.y); x.z = fmaf(f, v.z, x.z); x.w = fmaf(f, v.w, x.w);
        }
        *(float4*)(fold + (size_t)r * F::DF + d) = x;
    }
    paged_fold<W_ROWS, W_KEYS, DT>(p, b, fold, F::DF, row_m, row_l, &flag);
}

template <int N, int DT>
int launch_few(PagedParams p, cudaStream_t st) {
    static bool configured = false;
    if (!configured) {
        PGK_CUDA(cudaFuncSetAttribute(paged_few_kernel<N, DT>, cudaFuncAttributeMaxDynamicSharedMemorySize, Few<N>::BYTES));
        PGK_CUDA(cudaFuncSetAttribute(paged_few_kernel<N, DT>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        configured = true;
    }
    p.tiles = (int)(((long long)p.max_rows * p.rep + W_ROWS - 1) / W_ROWS);
    p.splits = paged_cut(p, (long long)p.seqs * p.tiles * p.kv_heads, W_KEYS, W_WARPS, Few<N>::RESIDENT, 6.f, PAGED_CLUSTER);
    PGK_CUDA(launch_clusters(paged_few_kernel<N, DT>, dim3((unsigned)(p.seqs * p.tiles), p.kv_heads, p.splits), W_THREADS, Few<N>::BYTES, st, p));
    return 0;
}
template <int DT>
int launch_few_dim(const PagedParams& p, cudaStream_t st) {
    switch ((p.dim + 31) / 32) {
        case 1: case 2: return launch_few<2, DT>(p, st);
        case 3: return launch_few<3, DT>(p, st);
        case 4: return launch_few<4, DT>(p, st);
        case 5: case 6: return launch_few<6, DT>(p, st);
        default: return launch_few<8, DT>(p, st);
    }
}

}  // namespace

int paged_few(const PagedParams& p, int dtype, cudaStream_t st) { return dtype == 1 ? launch_few_dim<1>(p, st) : launch_few_dim<2>(p, st); }

}  // namespace pgk
