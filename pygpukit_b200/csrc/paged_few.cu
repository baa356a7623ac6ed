// paged_few.cu -- attention of few rows a sequence over 16-bit pages: decoded tokens, small trees of drafts, and whatever the large tiles of paged_tc.cu do not serve
// (heads above 128 elements, pages that no copy of eight positions fits).
//
// One pass over the keys with the running maximum and sum of a softmax.  A block has 8 or 16 (row, head) rows, each of its warps walks over its own blocks of 16 keys by
// mma.sync m16n8k16, the keys and then the values' elements as its 16: S^T = K Q^T, O^T += V^T P^T, so that eight rows cost half of what sixteen do.  K and V go straight
// from memory to registers, sixteen bytes a lane: the order of a head's elements in the score's sum is free, so a lane takes the eight that follow each other in one
// key; V wants pairs of keys in a register, which byte permutations of two keys' loads make.  The next 16 keys are fetched as soon as a product has read these.
// Weights become two terms of bfloat16 (2^-17 of each; one left an output 1.4 times as far off), one of float16 (2^-12); their sum is float32 of the unrounded ones.
// Blocks of a cluster share a sequence's keys and fold through distributed shared memory.
// Bound by the bytes of the keys and, for one request, by the chain from launch to fold.
#include "paged.cuh"
#include "tc_common.cuh"
#include "../../include/pgk_b200.h"

namespace pgk {

namespace {

constexpr int W_KEYS = 16, W_WARPS = 4, W_THREADS = W_WARPS * 32;

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
// an 8 x 8 matrix of 16-bit numbers, a register a lane, transposed
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}

// N: 32-element pieces of a head; NT: tiles of eight rows
template <int N, int NT> struct Few {
    static constexpr int DP = 32 * N, CH = (DP + 63) / 64, ROWS = 8 * NT, DF = DP + 4;
    static constexpr int QBYTES = N * NT * 32 * 16, FOLD = W_WARPS * ROWS * DF * 4, BYTES = QBYTES > FOLD ? QBYTES : FOLD;
    static constexpr int RESIDENT = N <= 2 ? (NT == 1 ? 5 : 4) : (N <= 4 ? 3 : 2);
};

template <int N, int NT, int DT>
__global__ void __launch_bounds__(W_THREADS, Few<N, NT>::RESIDENT) paged_few_kernel(const __grid_constant__ PagedParams p) {
    using F = Few<N, NT>;
    constexpr int CH = F::CH, ROWS = F::ROWS, TERMS = DT == 1 ? 1 : 2;
    // float16 weights: from 2^6 down, so that those 2^-20 of the largest still have all their bits; they grow to 2^14 before the reference moves
    constexpr float TOP = DT == 1 ? 6.f : 0.f;
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ float wm[W_WARPS][ROWS], wl[W_WARPS][ROWS];
    __shared__ PagedFold<ROWS> f;
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), gl = lane >> 2, t = lane & 3;
    if (tid == 0) f.bad = 0;
    griddep_wait();
    griddep_launch();
    const PagedBlock<ROWS, W_KEYS> b(p, (int)blockIdx.x, (int)blockIdx.y, (int)blockIdx.z);
    const int D = p.dim;
    const char* const kb = (const char*)p.k_data;
    const char* const vb = (const char*)p.v_data;
    const size_t stride = (size_t)D * 2;

    uint4 kk[N][2], vv[CH][4];
    auto load_k = [&](int rows) {                             // key gl, gl + 8: elements 32 s + 8 t ... + 7
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
    auto load_v = [&](int rows) {                             // keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9: elements 64 c + 8 gl ... + 7
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
    };
    int k = b.ubeg + warp;
    int rows = k < b.uend ? b.row_of(p, k * W_KEYS + (lane & 15)) : -1;
    int next = k + W_WARPS < b.uend ? b.row_of(p, (k + W_WARPS) * W_KEYS + (lane & 15)) : -1;

    // ---------------- queries: piece s, tile n: this lane's eight elements 32 s + 8 t of row 8 n + gl
    uint4* const qs = (uint4*)smem;
    for (int i = warp; i < N * NT; i += W_WARPS) {
        const int r = gl + 8 * (i % NT), d = 32 * (i / NT) + 8 * t, x = b.f0 + r, tok = b.first + x / p.rep;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (r < b.live && d < D && tok >= 0 && tok < p.tokens) {
            const uint16_t* src = (const uint16_t*)p.q + (size_t)tok * p.q_ld + (size_t)(b.head * p.rep + x % p.rep) * D + d;
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
    if (k < b.uend) {
        load_k(rows);
        load_v(rows);
    }
    __syncthreads();

    float o[CH][4][NT][4], m[NT][2], l[NT][2];               // of rows 8 n + 2 t, + 1
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        m[n][0] = m[n][1] = -INFINITY;
        l[n][0] = l[n][1] = 0.f;
    }
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[c][j][n][e] = 0.f;
    bool bad = false;
#pragma unroll 1
    for (; k < b.uend; k += W_WARPS) {
        const int j0 = k * W_KEYS;
        float s[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
#pragma unroll
        for (int q = 0; q < N; ++q)
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const uint4 a = qs[(q * NT + n) * 32 + lane];
                mma16816<DT>(s[n], kk[q][0].x, kk[q][1].x, kk[q][0].y, kk[q][1].y, a.x, a.y);
                mma16816<DT>(s[n], kk[q][0].z, kk[q][1].z, kk[q][0].w, kk[q][1].w, a.z, a.w);
            }
        const uint32_t there = __ballot_sync(0xffffffffu, rows >= 0);
        const bool edge = (there & 0xffffu) != 0xffffu || j0 + W_KEYS > b.base;
        const bool more = k + W_WARPS < b.uend;
        rows = next;
        if (more) load_k(rows);
        next = k + 2 * W_WARPS < b.uend ? b.row_of(p, (k + 2 * W_WARPS) * W_KEYS + (lane & 15)) : -1;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[n][e] *= p.scale_log2;
        if (edge) {
            const int at = j0 - b.base;                       // the step's row of the block's first key, below 0 before the step
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int i = (b.f0 + 8 * n + 2 * t + e) / p.rep;
                    const uint32_t see = paged_window(p, b.first + i, i, at) & there;
                    if (!((see >> gl) & 1u)) s[n][e] = -INFINITY;
                    if (!((see >> (gl + 8)) & 1u)) s[n][2 + e] = -INFINITY;
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
        float top[NT][2];
        bool up = false;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float x = fmaxf(s[n][e], s[n][2 + e]);
#pragma unroll
                for (int y = 4; y <= 16; y <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, y));
                top[n][e] = x - TOP;
                up |= top[n][e] > m[n][e] + PAGED_LAZY;       // (also the first finite maximum)
            }
        if (__any_sync(0xffffffffu, up)) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    if (!(top[n][e] > m[n][e] + PAGED_LAZY)) continue;
                    const float fix = m[n][e] == -INFINITY ? 0.f : exp2f(m[n][e] - top[n][e]);
                    m[n][e] = top[n][e];
                    l[n][e] *= fix;
#pragma unroll
                    for (int c = 0; c < CH; ++c)
#pragma unroll
                        for (int j = 0; j < 4; ++j) { o[c][j][n][e] *= fix; o[c][j][n][2 + e] *= fix; }
                }
        }
        uint32_t w[NT][TERMS][2];                             // weights of row 8 n + gl: keys 2 t, 2 t + 1 and 2 t + 8, 2 t + 9
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const float n0 = paged_neg(m[n][0]), n1 = paged_neg(m[n][1]);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const float a = ex2(s[n][2 * u] + n0), c = ex2(s[n][2 * u + 1] + n1);
                l[n][0] += a;
                l[n][1] += c;
                const uint32_t x = paged_pack2<DT>(a, c);
                w[n][0][u] = transposed(x);
                if constexpr (TERMS == 2) w[n][1][u] = transposed(pack_bf16x2(a - bf16lo(x), c - bf16hi(x)));
            }
        }
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const uint32_t* const v0 = &vv[c][0].x;
            const uint32_t* const v1 = &vv[c][1].x;
            const uint32_t* const v2 = &vv[c][2].x;
            const uint32_t* const v3 = &vv[c][3].x;
#pragma unroll
            for (int j = 0; j < 4; ++j) {                     // elements 64 c + 8 gl + 2 j, + 1 of the key pairs
                const uint32_t a0 = __byte_perm(v0[j], v1[j], 0x5410), a1 = __byte_perm(v0[j], v1[j], 0x7632), a2 = __byte_perm(v2[j], v3[j], 0x5410),
                               a3 = __byte_perm(v2[j], v3[j], 0x7632);
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int x = 0; x < TERMS; ++x) mma16816<DT>(o[c][j][n], a0, a1, a2, a3, w[n][x][0], w[n][x][1]);
            }
        }
        if (more) load_v(rows);
    }

    // ---------------- the warps' sums into one
    if (bad) f.bad = 1;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float x = l[n][e];
#pragma unroll
            for (int y = 4; y <= 16; y <<= 1) x += __shfl_xor_sync(0xffffffffu, x, y);
            if (gl == 0) { wm[warp][8 * n + 2 * t + e] = m[n][e]; wl[warp][8 * n + 2 * t + e] = x; }
        }
    __syncthreads();                                          // the queries are read
    float* const sums = (float*)smem;                         // [warps][rows][DF]
#pragma unroll
    for (int c = 0; c < CH; ++c)
        if (64 * c + 8 * gl < F::DP) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float* const dst = sums + ((size_t)warp * ROWS + 8 * n + 2 * t + e) * F::DF + 64 * c + 8 * gl;
                    *(float4*)dst = make_float4(o[c][0][n][e], o[c][0][n][2 + e], o[c][1][n][e], o[c][1][n][2 + e]);
                    *(float4*)(dst + 4) = make_float4(o[c][2][n][e], o[c][2][n][2 + e], o[c][3][n][e], o[c][3][n][2 + e]);
                }
        }
    if (tid < ROWS) {
        float top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int x = 0; x < W_WARPS; ++x) top = fmaxf(top, wm[x][tid]);
#pragma unroll
        for (int x = 0; x < W_WARPS; ++x) {
            const float y = wm[x][tid] == -INFINITY ? wl[x][tid] - wl[x][tid] : exp2f(wm[x][tid] - top);
            sum = fmaf(wl[x][tid], y, sum);
            wm[x][tid] = y;
        }
        f.m[tid] = top;
        f.l[tid] = sum;
    }
    __syncthreads();
    for (int i = tid; i < b.live * (F::DP / 4); i += W_THREADS) {
        const int r = i / (F::DP / 4), d = (i - r * (F::DP / 4)) * 4;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int y = 0; y < W_WARPS; ++y) {
            const float z = wm[y][r];
            const float4 v = *(const float4*)(sums + ((size_t)y * ROWS + r) * F::DF + d);
            x.x = fmaf(z, v.x, x.x); x.y = fmaf(z, v.y, x.y); x.z = fmaf(z, v.z, x.z); x.w = fmaf(z, v.w, x.w);
        }
        *(float4*)(sums + (size_t)r * F::DF + d) = x;
    }
    paged_fold<ROWS, W_KEYS, DT, F::DP>(p, b, sums, f);
}

template <int N, int NT, int DT>
int launch_few(PagedParams p, cudaStream_t st) {
    using F = Few<N, NT>;
    static bool configured = false;
    if (!configured) {
        PGK_CUDA(cudaFuncSetAttribute(paged_few_kernel<N, NT, DT>, cudaFuncAttributeMaxDynamicSharedMemorySize, F::BYTES));
        PGK_CUDA(cudaFuncSetAttribute(paged_few_kernel<N, NT, DT>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        configured = true;
    }
    p.tiles = (int)(((long long)p.max_rows * p.rep + F::ROWS - 1) / F::ROWS);
    p.splits = paged_cut(p, (long long)p.seqs * p.tiles * p.kv_heads, W_KEYS, W_WARPS, F::RESIDENT, 6.f, PAGED_CLUSTER);
    PGK_CUDA(launch_clusters(paged_few_kernel<N, NT, DT>, dim3((unsigned)(p.seqs * p.tiles), p.kv_heads, p.splits), W_THREADS, F::BYTES, st, p));
    return 0;
}
template <int DT>
int launch_few_dim(const PagedParams& p, cudaStream_t st) {
    const bool two = (long long)p.max_rows * p.rep > 8;
    switch ((p.dim + 31) / 32) {
        case 1: case 2: return two ? launch_few<2, 2, DT>(p, st) : launch_few<2, 1, DT>(p, st);
        case 3: return two ? launch_few<3, 2, DT>(p, st) : launch_few<3, 1, DT>(p, st);
        case 4: return two ? launch_few<4, 2, DT>(p, st) : launch_few<4, 1, DT>(p, st);
        case 5: case 6: return launch_few<6, 1, DT>(p, st);
        default: return launch_few<8, 1, DT>(p, st);
    }
}

}  // namespace

int paged_few(const PagedParams& p, int dtype, cudaStream_t st) { return dtype == 1 ? launch_few_dim<1>(p, st) : launch_few_dim<2>(p, st); }

}  // namespace pgk
