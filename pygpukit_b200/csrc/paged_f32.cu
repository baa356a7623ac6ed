// paged_f32.cu -- attention over pages of 32 bits: products and sums are float32, nothing is rounded between.
//
// A block has R (row, head) rows (4, 8 or 16: as many as a token's heads need), each of its warps walks over its own blocks of 32 keys, whose K and V it fetches to
// shared memory by itself, K of the next block while this one's values are summed and V while its scores are formed.  Scores: a lane has two keys and half of the rows; values: a
// lane has every 16th quartet of elements and half of the rows.  Both load the next operands while these are multiplied.  (A lane a key and all rows: 67 us where this
// takes 35, four sequences of 84 rows over 1500 keys of 64 elements; four keys and 32 rows a block 36.)  Bound by the latency of shared memory: a block of 32 keys and 16
// rows of 64 elements takes a warp 6500 cycles, of which its multiply-adds need 2000, and a SM has two warps for each of its schedulers.
// Blocks of a cluster share a sequence's keys.
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

// E: quartets of elements a lane has of an output row; W: warps.  What the halves of a warp read at once lies four banks apart.
template <int R, int E, int W> struct Single {
    static constexpr int DN = 64 * E, FS = DN + 4;
    static int warp_floats(int D) { return S_KEYS * (D + 4) + S_KEYS * D + 2 * R * S_KEYS + 4; }
    static int bytes(int D) {
        const int run = (R * D + 4 + W * warp_floats(D)) * 4, fold = (W * R + R + PAGED_CLUSTER - 1) * FS * 4;
        return run > fold ? run : fold;
    }
};

// N values of each of 16 lanes into the lanes' results: lane l of the 16 gets that of value l / (16 / N)
template <int N, typename Op> __device__ __forceinline__ float reduce_half(float (&v)[N], int lane, Op op) {
    int off = 8;
#pragma unroll
    for (int n = N / 2; n >= 1; n /= 2, off /= 2)
#pragma unroll
        for (int i = 0; i < n; ++i) {
            const float mine = lane & off ? v[i + n] : v[i], other = lane & off ? v[i] : v[i + n];
            v[i] = op(mine, __shfl_xor_sync(0xffffffffu, other, off));
        }
#pragma unroll
    for (int o = 8 / N; o >= 1; o /= 2) v[0] = op(v[0], __shfl_xor_sync(0xffffffffu, v[0], o));
    return v[0];
}

template <int R, int E, int W>
__global__ void __launch_bounds__(W * 32, 1) paged_f32_kernel(const __grid_constant__ PagedParams p) {
    using X = Single<R, E, W>;
    constexpr int H = R / 2, EACH = 16 / H;                    // rows of a half; lanes that know a row's reference
    extern __shared__ __align__(16) float smf[];
    __shared__ float wm[W][R], wl[W][R];
    __shared__ PagedFold<R> f;
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), D = p.dim, D4 = D / 4, DF = D + 4;
    const int half = lane >> 4, sub = lane & 15, r0 = half * H;
    float* const qs = smf;                                    // [2][H][D] and 4 between the halves
    float* const ks = qs + R * D + 4 + warp * (S_KEYS * DF + S_KEYS * D + 2 * R * S_KEYS + 4);
    float* const vs = ks + S_KEYS * DF;
    float2* const ps = (float2*)(vs + S_KEYS * D) + half * (H * S_KEYS + 2);       // the half's [H][32], each weight twice
    if (tid == 0) f.bad = 0;
    griddep_wait();
    griddep_launch();
    const PagedBlock<R, S_KEYS> b(p, (int)blockIdx.x, (int)blockIdx.y, (int)blockIdx.z);

    auto fetch = [&](const void* base, float* to, int ld, int rows) {
        const float* const src = (const float*)base + 4 * (E == 1 ? lane & 15 : lane);
        if constexpr (E == 1) {                                       // two keys at a time
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
                for (int c = 0; c < E / 2; ++c)
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
#pragma unroll
    for (int r = warp; r < R; r += W) {
        const int x = b.f0 + r, step = paged_div(x, p.by_rep), tok = b.first + step;
        const bool live = r < b.live && tok >= 0 && tok < p.tokens;
        const float* const src = (const float*)p.q + (live ? (size_t)tok * p.q_ld + (size_t)(b.head * p.rep + x - step * p.rep) * D : 0);
        float* const dst = qs + r * D + (r >= H ? 4 : 0);
        if (p.wide_q) {
#pragma unroll
            for (int c = 0; c < (E + 1) / 2; ++c)
                if (lane + 32 * c < D4) *(float4*)(dst + 4 * (lane + 32 * c)) = live ? __ldcg((const float4*)src + lane + 32 * c) : make_float4(0.f, 0.f, 0.f, 0.f);
        } else
            for (int d = lane; d < D; d += 32) dst[d] = live ? __ldcg(src + d) : 0.f;
    }
    __syncthreads();

    uint64_t o[H][E][2];                                      // pairs of elements
    float m_r = -INFINITY, nm[H], l[H];                       // a lane keeps row r0 + sub / EACH's reference
#pragma unroll
    for (int r = 0; r < H; ++r) {
        nm[r] = l[r] = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) o[r][e][0] = o[r][e][1] = pair(0.f, 0.f);
    }
    bool bad = false;
#pragma unroll 1
    for (; k < b.uend; k += W) {
        const int j0 = k * S_KEYS, next = k + W < b.uend ? b.row_of(p, (k + W) * S_KEYS + lane) : -1;
        cp_async_wait<1>();                                   // K is here
        __syncwarp();
        uint64_t s2[H][2];
#pragma unroll
        for (int r = 0; r < H; ++r) s2[r][0] = s2[r][1] = pair(0.f, 0.f);
        const float* const kr = ks + sub * DF;
        const float* const qr = qs + r0 * D + 4 * half;
        ulonglong2 x[2], y[2], q[2][H];                       // the next ones on their way while these are multiplied
        auto load = [&](int u, int c) {
            x[u] = *(const ulonglong2*)(kr + 4 * c);
            y[u] = *(const ulonglong2*)(kr + 16 * DF + 4 * c);
#pragma unroll
            for (int r = 0; r < H; ++r) q[u][r] = *(const ulonglong2*)(qr + r * D + 4 * c);
        };
        load(0, 0);
#pragma unroll 1
        for (int c = 0; c < D4; c += 2)                       // (a multiple of two)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                load(u ^ 1, min(c + u + 1, D4 - 1));
#pragma unroll
                for (int r = 0; r < H; ++r) {
                    s2[r][0] = fma2(q[u][r].x, x[u].x, s2[r][0]);
                    s2[r][1] = fma2(q[u][r].x, y[u].x, s2[r][1]);
                }
#pragma unroll
                for (int r = 0; r < H; ++r) {
                    s2[r][0] = fma2(q[u][r].y, x[u].y, s2[r][0]);
                    s2[r][1] = fma2(q[u][r].y, y[u].y, s2[r][1]);
                }
            }
        __syncwarp();
        if (k + W < b.uend) fetch(p.k_data, ks, DF, next);
        else cp_async_commit();
        const bool edge = __any_sync(0xffffffffu, rows < 0) || j0 + S_KEYS > b.base;
        const int at = j0 - b.base;
        float s[H][2], v[H];
#pragma unroll
        for (int r = 0; r < H; ++r) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                float a, c;
                unpair(s2[r][u], a, c);
                s[r][u] = (a + c) * p.scale_log2;
            }
        }
        if (edge) {
            const unsigned there = __ballot_sync(0xffffffffu, rows >= 0);
#pragma unroll
            for (int r = 0; r < H; ++r) {
                const int i = paged_div(b.f0 + r0 + r, p.by_rep);
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const int key = sub + 16 * u, t = at + key;
                    if (!((there >> key) & 1u) || r0 + r >= b.live || (t >= 0 && !paged_sees(p, b.first + i, i, t))) s[r][u] = -INFINITY;
                }
            }
        }
#pragma unroll
        for (int r = 0; r < H; ++r) v[r] = fmaxf(s[r][0], s[r][1]);
        const float top = reduce_half<H>(v, lane, [](float x, float y) { return fmaxf(x, y); });
        const bool up = top > m_r + PAGED_LAZY;               // (also the first finite maximum)
        if (__any_sync(0xffffffffu, up)) {
            const float f_r = !up ? 1.f : (m_r == -INFINITY ? 0.f : exp2f(m_r - top));
            if (up) m_r = top;
#pragma unroll
            for (int r = 0; r < H; ++r) {
                const float fix = __shfl_sync(0xffffffffu, f_r, half * 16 + r * EACH);
                nm[r] = paged_neg(__shfl_sync(0xffffffffu, m_r, half * 16 + r * EACH));
                l[r] *= fix;
#pragma unroll
                for (int e = 0; e < E; ++e) { o[r][e][0] = mul2(o[r][e][0], pair(fix, fix)); o[r][e][1] = mul2(o[r][e][1], pair(fix, fix)); }
            }
        }
#pragma unroll
        for (int r = 0; r < H; ++r)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const float w = ex2(s[r][u] + nm[r]);
                l[r] += w;
                ps[r * S_KEYS + sub + 16 * u] = make_float2(w, w);
            }
        cp_async_wait<1>();                                   // V is here
        __syncwarp();
        auto values = [&](auto step) {
            float4 v[2][2][E];
            ulonglong2 w[2][H];                               // of two keys
            auto load = [&](int u, int key) {
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        float4& x = v[u][j][e];
                        x = sub + 16 * e < D4 ? *(const float4*)(vs + (key + j) * D + 4 * (sub + 16 * e)) : make_float4(0.f, 0.f, 0.f, 0.f);
                        if constexpr (step.value)
                            if (at + key + j >= 0) {          // values of the step's rows, which not all rows see
#pragma unroll
                                for (int i = 0; i < 4; ++i)
                                    if (!(fabsf((&x.x)[i]) < INFINITY)) { bad = true; (&x.x)[i] = 0.f; }
                            }
                    }
#pragma unroll
                for (int r = 0; r < H; ++r) w[u][r] = *(const ulonglong2*)(ps + r * S_KEYS + key);
            };
            load(0, 0);
#pragma unroll 1
            for (int key = 0; key < S_KEYS; key += 4)
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    load(u ^ 1, min(key + 2 * u + 2, S_KEYS - 2));
#pragma unroll
                    for (int r = 0; r < H; ++r)
#pragma unroll
                        for (int e = 0; e < E; ++e) {
                            o[r][e][0] = fma2(w[u][r].x, pair(v[u][0][e].x, v[u][0][e].y), o[r][e][0]);
                            o[r][e][1] = fma2(w[u][r].x, pair(v[u][0][e].z, v[u][0][e].w), o[r][e][1]);
                        }
#pragma unroll
                    for (int r = 0; r < H; ++r)
#pragma unroll
                        for (int e = 0; e < E; ++e) {
                            o[r][e][0] = fma2(w[u][r].y, pair(v[u][1][e].x, v[u][1][e].y), o[r][e][0]);
                            o[r][e][1] = fma2(w[u][r].y, pair(v[u][1][e].z, v[u][1][e].w), o[r][e][1]);
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
    const float sum_r = reduce_half<H>(l, lane, [](float x, float y) { return x + y; });
    if (sub % EACH == 0) {
        wm[warp][r0 + sub / EACH] = m_r;
        wl[warp][r0 + sub / EACH] = sum_r;
    }
    __syncthreads();
    constexpr int FS = X::FS;
    float* const fold = smf;                                  // [W][R][FS]
#pragma unroll
    for (int r = 0; r < H; ++r)
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (sub + 16 * e < D4) *(ulonglong2*)(fold + (warp * R + r0 + r) * FS + 4 * (sub + 16 * e)) = make_ulonglong2(o[r][e][0], o[r][e][1]);
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
    PagedOut<R, S_KEYS, 0, X::DN> out(p, b, f, fold + (W - 1) * R * FS);       // the last warp's place, and what is behind it
    out.begin();
    for (int i = tid; i < b.live * D4; i += W * 32) {
        const int r = i / D4, d = (i - r * D4) * 4;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int w = 0; w < W; ++w) {
            const float y = wm[w][r];
            const float4 v = *(const float4*)(fold + (w * R + r) * FS + d);
            x.x = fmaf(y, v.x, x.x); x.y = fmaf(y, v.y, x.y); x.z = fmaf(y, v.z, x.z); x.w = fmaf(y, v.w, x.w);
        }
        *(float4*)(out.stage + r * FS + d) = x;
    }
    out.join([] {});
}

template <int R, int E, int W>
int launch_single(PagedParams p, cudaStream_t st) {
    const int smem = Single<R, E, W>::bytes(p.dim), kind = smem > 113 * 1024 ? 0 : (smem > 75 * 1024 ? 1 : 2);       // one, two, three blocks a SM
    static PagedOccupancy fits[3];
    PGK_CUDA(fits[kind].once([&](int* at_once) {
        const auto kernel = paged_f32_kernel<R, E, W>;
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Single<R, E, W>::bytes(64 * E));
        if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        for (int i = 1; e == cudaSuccess && i <= PAGED_CLUSTER; ++i) {
            e = clusters_at_once(&at_once[i], kernel, W * 32, (size_t)smem, i);
            if (kind) at_once[i] += at_once[i] / 16;          // a few more than fit run beside the others' second half: 96 of three blocks, 93 fit, 35 us, of two blocks 45
        }
        return e;
    }));
    p.tiles = (int)(((long long)p.max_rows * p.rep + R - 1) / R);
    return paged_launch<R, S_KEYS, 0, 64 * E>(p, paged_split(p, S_KEYS * W, fits[kind].at_once, PAGED_CLUSTER, 2), st, [&](const PagedParams& q, dim3 grid, bool apart) {
        return launch_clusters(paged_f32_kernel<R, E, W>, grid, apart, W * 32, (size_t)smem, st, q);
    });
}

}  // namespace

int paged_f32(const PagedParams& p, cudaStream_t st) {
    const long long rows = (long long)p.max_rows * p.rep;
    if (p.dim > 128) return rows <= 4 ? launch_single<4, 4, 2>(p, st) : launch_single<8, 4, 2>(p, st);
    if (p.dim > 64) return rows <= 4 ? launch_single<4, 2, 4>(p, st) : (rows <= 8 ? launch_single<8, 2, 4>(p, st) : launch_single<16, 2, 4>(p, st));
    return rows <= 4 ? launch_single<4, 1, 4>(p, st) : (rows <= 8 ? launch_single<8, 1, 4>(p, st) : launch_single<16, 1, 4>(p, st));
}

}  // namespace pgk
