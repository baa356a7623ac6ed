// tree.cu -- trees of drafted tokens: which rows of a step see each other, and which drafts the model accepts.
//
// A sequence's rows are a tree by their parents (row numbers of the same sequence, smaller than the row's own; others make a root).  Row i's mask has its own bit and its
// ancestors', its depth is how many those are.  A thread walks one row's ancestors for one word of its mask: they descend, so that it stops below its word.
//
// Acceptance: row 0 is the last token that was accepted before the step; of a row's children the lowest one whose token is what the model chose behind the row is accepted next.
// What the model chose is the largest logit, the lowest index of equal ones (NaN counts as none); a cluster of blocks reads a row, bound by the bytes of the logits; a second
// launch walks the trees, a warp a sequence.
#include "paged.cuh"
#include "../../include/pgk_b200.h"

namespace pgk {

namespace {

__global__ void __launch_bounds__(256) tree_masks_kernel(const int32_t* parents, const int32_t* starts, int tokens, int max_rows, int words, int32_t* masks, int32_t* depths) {
    extern __shared__ int up[];
    griddep_wait();
    griddep_launch();
    const int seq = blockIdx.x, first = __ldcg(starts + seq), n = min(max(0, __ldcg(starts + seq + 1) - first), max_rows);
    if (first < 0 || (long long)first + n > tokens) return;
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
        const int x = __ldcg(parents + first + i);
        up[i] = x >= 0 && x < i ? x : -1;
    }
    __syncthreads();
    for (int x = blockIdx.y * blockDim.x + threadIdx.x; x < n * words; x += blockDim.x * gridDim.y) {
        const int i = x / words, w = x - i * words;
        uint32_t bits = 0;
        int j = i, depth = 0;
        for (; j >= 32 * w; j = up[j]) {
            if (j >> 5 == w) bits |= 1u << (j & 31);
            ++depth;
        }
        masks[(size_t)(first + i) * words + w] = (int32_t)bits;
        if (w == 0) depths[first + i] = depth - 1;
    }
}

constexpr int A_THREADS = 512, A_CLUSTER = 8;
struct Best { float v; int at; };
__device__ __forceinline__ Best better(Best a, Best b) { return b.v > a.v || (b.v == a.v && b.at < a.at) ? b : a; }

template <int DT>
__global__ void __launch_bounds__(A_THREADS) choose_kernel(const void* logits, long ld, int vocab, int wide, int32_t* chosen) {
    constexpr int E = DT == 0 ? 4 : 8;                        // elements of 16 bytes
    __shared__ float vs[A_THREADS / 32];
    __shared__ int is[A_THREADS / 32];
    __shared__ float bv;
    __shared__ int bi;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, blocks = gridDim.x, row = blockIdx.y;
    griddep_wait();
    griddep_launch();
    Best best = {-INFINITY, 0x7fffffff};
    const char* const src = (const char*)logits + (size_t)row * ld * (DT == 0 ? 4 : 2);
    auto take = [&](float v, int i) {
        if (v > best.v) best = {v, i};                        // a thread's indexes ascend
    };
    if (wide) {
        const int n = vocab / E;
#pragma unroll 4
        for (int c = blockIdx.x * A_THREADS + tid; c < n; c += blocks * A_THREADS) {
            const uint4 x = ldg_stream(src + (size_t)c * 16);
            const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if constexpr (DT == 0) take(__uint_as_float(w[e]), c * E + e);
                else if constexpr (DT == 1) {
                    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[e]));
                    take(f.x, c * E + 2 * e);
                    take(f.y, c * E + 2 * e + 1);
                } else {
                    take(bf16lo(w[e]), c * E + 2 * e);
                    take(bf16hi(w[e]), c * E + 2 * e + 1);
                }
            }
        }
        if (blockIdx.x == 0 && tid < vocab - n * E) take(paged_float<DT>(src, (size_t)n * E + tid), n * E + tid);
    } else
        for (int i = blockIdx.x * A_THREADS + tid; i < vocab; i += blocks * A_THREADS) take(paged_float<DT>(src, (size_t)i), i);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) best = better(best, {__shfl_xor_sync(0xffffffffu, best.v, x), __shfl_xor_sync(0xffffffffu, best.at, x)});
    if (lane == 0) { vs[warp] = best.v; is[warp] = best.at; }
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < A_THREADS / 32; ++w) best = better(best, {vs[w], is[w]});
        bv = best.v;
        bi = best.at;
    }
    if (blocks > 1) paged_cluster_sync();
    if (blockIdx.x == 0 && tid == 0) {
        for (int s = 1; s < blocks; ++s)
            best = better(best, {paged_remote_float(paged_remote(smem_u32(&bv), s)), __float_as_int(paged_remote_float(paged_remote(smem_u32(&bi), s)))});
        chosen[row] = best.at == 0x7fffffff ? 0 : best.at;    // nothing above -infinity: the first
    }
    if (blocks > 1) paged_cluster_sync();
}

__global__ void __launch_bounds__(32) accept_kernel(const int32_t* chosen, const int32_t* tokens, const int32_t* parents, const int32_t* starts, int total, int max_rows, int32_t* rows,
                                                    int32_t* counts, int32_t* next) {
    extern __shared__ int sh[];
    const int lane = threadIdx.x, seq = blockIdx.x;
    griddep_wait();
    griddep_launch();
    const int first = __ldcg(starts + seq);
    int n = min(max(0, __ldcg(starts + seq + 1) - first), max_rows);
    if (first < 0 || (long long)first + n > total) n = 0;
    int* const tok = sh;
    int* const up = sh + max_rows;
    int* const want = sh + 2 * max_rows;
    for (int i = lane; i < n; i += 32) {
        tok[i] = __ldcg(tokens + first + i);
        up[i] = __ldcg(parents + first + i);
        want[i] = __ldcg(chosen + first + i);
    }
    __syncwarp();
    int32_t* const out = rows + (size_t)seq * max_rows;
    int count = 0, cur = n > 0 ? 0 : -1, last = -1;
    while (cur >= 0) {
        if (lane == 0) out[count] = cur;
        ++count;
        last = cur;
        int child = -1;
        for (int j = (last + 1) & ~31; j < n && child < 0; j += 32) {
            const int i = j + lane;
            const uint32_t hit = __ballot_sync(0xffffffffu, i > last && i < n && up[i] == last && tok[i] == want[last]);
            if (hit) child = j + __ffs((int)hit) - 1;
        }
        cur = child;
    }
    for (int i = count + lane; i < max_rows; i += 32) out[i] = -1;
    if (lane == 0) {
        counts[seq] = count;
        next[seq] = last >= 0 ? want[last] : -1;
    }
}

}  // namespace

}  // namespace pgk

using namespace pgk;

extern "C" int pgk_tree_masks(const int32_t* parents, const int32_t* row_starts, int seqs, int tokens, int max_rows, int words, int32_t* masks, int32_t* depths, void* stream) {
    PGK_REQUIRE(seqs >= 0 && tokens >= 0 && max_rows > 0 && max_rows <= 4096 && words * 32ll >= max_rows && words <= 1 << 18, "tree_masks failed: %d sequences of up to %d rows in %d, masks of %d words", seqs, max_rows,
                tokens, words);
    if (seqs == 0 || tokens == 0) return 0;
    PGK_REQUIRE(parents && row_starts && masks && depths, "tree_masks failed: an array is missing");
    const int blocks = (int)(((long long)max_rows * words + 255) / 256);
    PGK_CUDA(launch_waiting(tree_masks_kernel, dim3(seqs, blocks < 64 ? blocks : 64), dim3(256), (size_t)max_rows * 4, (cudaStream_t)stream, parents, row_starts, tokens, max_rows, words, masks,
                            depths));
    return 0;
}

extern "C" int pgk_accept_tree(const void* logits, long ld, int dtype, int vocab, const int32_t* chosen, const int32_t* tokens, const int32_t* parents, const int32_t* row_starts, int seqs,
                               int total, int max_rows, int32_t* rows, int32_t* counts, int32_t* next_tokens, void* stream) {
    PGK_REQUIRE(seqs >= 0 && total >= 0 && total <= 65535 && max_rows > 0 && max_rows <= 4096, "accept_tree failed: %d sequences of up to %d rows in %d", seqs, max_rows, total);
    PGK_REQUIRE(chosen || (dtype >= 0 && dtype <= 2 && vocab > 0 && vocab <= PAGED_MOST && ld >= vocab), "accept_tree failed: type %d, vocabulary %d in rows of %ld", dtype, vocab, ld);
    if (seqs == 0) return 0;
    PGK_REQUIRE((logits || chosen || total == 0) && tokens && parents && row_starts && rows && counts && next_tokens, "accept_tree failed: an array is missing");
    const cudaStream_t st = (cudaStream_t)stream;
    void* ws = nullptr;
    if (!chosen && total > 0) {
        if (int rc = scratch_alloc(&ws, (size_t)total * 4, st)) return rc;
        const int size = dtype == 0 ? 4 : 2, wide = (uintptr_t)logits % 16 == 0 && ld * size % 16 == 0;
        int blocks = 1;                                       // a row's: until there are 16 a SM, which even out, none with less than four rounds
        while (blocks < A_CLUSTER && (long long)total * blocks <= 8 * sm_count() && (long long)vocab * size > 4ll * 16 * A_THREADS * blocks) blocks *= 2;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(blocks, total);
        cfg.blockDim = dim3(A_THREADS);
        cfg.stream = st;
        cudaLaunchAttribute attr[2];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        attr[1].id = cudaLaunchAttributeClusterDimension;
        attr[1].val.clusterDim.x = (unsigned)blocks;
        attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 2;
        count_launch();
        const auto kernel = dtype == 0 ? choose_kernel<0> : (dtype == 1 ? choose_kernel<1> : choose_kernel<2>);
        const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, logits, ld, vocab, wide, (int32_t*)ws);
        if (e != cudaSuccess) scratch_free(ws, st);
        PGK_CUDA(e);
        chosen = (const int32_t*)ws;
    }
    const cudaError_t e = launch_waiting(accept_kernel, dim3(seqs), dim3(32), (size_t)max_rows * 12, st, chosen, tokens, parents, row_starts, total, max_rows, rows, counts, next_tokens);
    if (int rc = scratch_free(ws, st)) return rc;
    PGK_CUDA(e);
    return 0;
}
