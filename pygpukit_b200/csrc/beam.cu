// beam.cu -- a step of beam search: the best continuations of every group of beams, and the rows of memory that follow them.
//
//   c[k, v] = score[k] + (x[k, v] - log sum_u exp x[k, u]);  the n largest of a group's beams x vocabulary, ties to the lowest (beam, token)
//
// What bounds the selection: the logits, read once.  A block takes up to 8192 logits of a row into registers: their maximum, the sum of their
// exponentials, and their n best by the key (value, token), which no two share.  The n-th largest of the block's 256 per-thread maxima is a bound
// that at least n elements reach, and at most n threads' elements (n x 32) can: those few are ranked by counting.  A block per group then
// forms the rows' logarithms and ranks the survivors in float64, so that beams whose candidates lie within float32 rounding of each other
// keep their order.
#include "common.cuh"
#include "tc_common.cuh"
#include "../../include/pgk_b200.h"

#include <cmath>

namespace pgk {

namespace {

constexpr int B_THREADS = 256, B_EPT = 32, B_SLICE = B_THREADS * B_EPT;
constexpr int B_MAX_N = 64, B_MAX_BEAMS = 64;
constexpr int B_LIST = B_MAX_N * B_EPT;

struct BeamParams {
    const void* x; long ld;
    const float* scores; const int32_t* finished;
    int pad, beams, vocab, n, slices;
    float2* part;                         // [row][slice]: maximum, sum
    unsigned long long* keys;             // [row][slice][n], best first; 0: none
    float* out_scores; int32_t* parents; int32_t* tokens;
};

// larger key: larger value, then lower token; 0 is below every key
__device__ __forceinline__ unsigned long long beam_key(float v, uint32_t token) {
    const uint32_t u = __float_as_uint(v + 0.f);                  // -0 is 0
    return (unsigned long long)(u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u)) << 32 | (uint32_t)~token;
}
__device__ __forceinline__ float beam_value(unsigned long long key) {
    const uint32_t u = (uint32_t)(key >> 32);
    return __uint_as_float(u ^ ((u >> 31) ? 0x80000000u : 0xffffffffu));
}

template <int DT>
__device__ __forceinline__ float beam_logit(const void* x, size_t i) {
    float v;
    if constexpr (DT == 0) v = __ldcg((const float*)x + i);
    else if constexpr (DT == 1) { const uint16_t h = ld_act2((const uint16_t*)x + i); v = __half2float(__ushort_as_half(h)); }
    else v = bf16_bits_to_f32(ld_act2((const uint16_t*)x + i));
    return v;
}

// the place of `mine` among the block's values: how many are larger (they are all different, or 0)
__device__ __forceinline__ int rank_of(const unsigned long long* all, int count, unsigned long long mine) {
    int r = 0;
    for (int i = 0; i < count; ++i) r += all[i] > mine;
    return r;
}

template <int DT>
__global__ void __launch_bounds__(B_THREADS) beam_rows_kernel(const __grid_constant__ BeamParams p) {
    __shared__ unsigned long long best[B_THREADS], list[B_LIST];
    __shared__ float red[B_THREADS / 32];
    __shared__ int count;
    __shared__ unsigned long long bound;
    griddep_wait();
    griddep_launch();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, slice = blockIdx.x, row = blockIdx.y;
    if (p.finished && __ldcg(p.finished + row) != 0) return;
    const int from = slice * B_SLICE, n_here = min(B_SLICE, p.vocab - from);
    const char* x = (const char*)p.x + (size_t)row * p.ld * (DT == 0 ? 4 : 2);
    float v[B_EPT];
    float top = -INFINITY;
    bool bad = false;
#pragma unroll
    for (int e = 0; e < B_EPT; ++e) {
        const int i = e * B_THREADS + tid;
        v[e] = i < n_here ? beam_logit<DT>(x, (size_t)from + i) : -INFINITY;
    }
#pragma unroll
    for (int e = 0; e < B_EPT; ++e) {
        bad |= v[e] != v[e];
        top = fmaxf(top, v[e]);
    }
    if (tid == 0) { count = 0; bound = 0; }
    const float mine = top;
    top = warp_max(top);
    if (lane == 0) red[warp] = top;
    bad = __syncthreads_or(bad);
#pragma unroll
    for (int w = 0; w < B_THREADS / 32; ++w) top = fmaxf(top, red[w]);
    // exponentials; the thread's best key
    float sum = 0.f;
    const float base = top == -INFINITY ? 0.f : top;
    unsigned long long key = 0;
#pragma unroll
    for (int e = 0; e < B_EPT; ++e) {
        const int i = e * B_THREADS + tid;
        sum += expf(v[e] - base);
        if (v[e] == mine && key == 0 && i < n_here) key = beam_key(v[e], (uint32_t)(from + i));
    }
    sum = warp_sum(sum);
    __syncthreads();
    if (lane == 0) red[warp] = sum;
    best[tid] = key;
    __syncthreads();
    if (tid == 0) {
        sum = 0.f;
        for (int w = 0; w < B_THREADS / 32; ++w) sum += red[w];
        // a row with a NaN, or with +infinity, has no candidates: its logarithm says so
        p.part[(size_t)row * p.slices + slice] = make_float2(bad ? NAN : top, sum);
    }
    // the n-th largest of the threads' best keys (0 when fewer threads have any)
    if (key && rank_of(best, B_THREADS, key) == p.n - 1) bound = key;
    __syncthreads();
    const unsigned long long cut = bound;
#pragma unroll
    for (int e = 0; e < B_EPT; ++e) {
        const int i = e * B_THREADS + tid;
        if (i < n_here && v[e] == v[e]) {
            const unsigned long long k = beam_key(v[e], (uint32_t)(from + i));
            if (k >= cut) {
                const int at = atomicAdd(&count, 1);
                if (at < B_LIST) list[at] = k;
            }
        }
    }
    __syncthreads();
    const int m = min(count, B_LIST);
    unsigned long long* out = p.keys + ((size_t)row * p.slices + slice) * p.n;
    for (int i = tid; i < m; i += B_THREADS) {
        const int r = rank_of(list, m, list[i]);
        if (r < p.n) out[r] = list[i];
    }
    for (int i = m + tid; i < p.n; i += B_THREADS) out[i] = 0;
}

// A group's candidates, ordered by (score, lower beam, lower token).  A candidate's place: score in float64, then its flat index.
__device__ __forceinline__ bool ahead(double c, uint32_t beam, uint32_t token, double d, uint32_t beam2, uint32_t token2) {
    return c > d || (c == d && (beam < beam2 || (beam == beam2 && token < token2)));
}

__global__ void __launch_bounds__(B_THREADS) beam_merge_kernel(const __grid_constant__ BeamParams p) {
    __shared__ double lse[B_MAX_BEAMS];
    __shared__ int state[B_MAX_BEAMS];             // 0: candidates from the row's lists; 1: finished; 2: nothing but -infinity
    __shared__ double bc[B_THREADS / 32];
    __shared__ uint32_t bb[B_THREADS / 32], bt[B_THREADS / 32];
    griddep_wait();
    griddep_launch();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = blockIdx.x, K = p.beams;
    for (int k = warp; k < K; k += B_THREADS / 32) {
        const int row = g * K + k;
        const float score = __ldcg(p.scores + row);
        int st = !(score > -1e30f) ? 2 : 0;
        if (p.finished && __ldcg(p.finished + row) != 0) st = score != score ? 2 : 1;
        double l = 0.0;
        if (st == 0) {
            float top = -INFINITY;
            bool bad = false;
            for (int s = lane; s < p.slices; s += 32) {
                const float m = __ldcg(p.part + (size_t)row * p.slices + s).x;
                bad |= m != m;
                top = fmaxf(top, m);
            }
            top = warp_max(top);
            bad = __any_sync(0xffffffffu, bad) || top == INFINITY || top == -INFINITY;
            double sum = 0.0;
            for (int s = lane; s < p.slices; s += 32) {
                const float2 q = __ldcg(p.part + (size_t)row * p.slices + s);
                if (!bad && q.x > -INFINITY) sum += (double)q.y * exp((double)q.x - (double)top);
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (bad) st = 2;
            else l = (double)top + log(sum);
        }
        if (lane == 0) { lse[k] = l; state[k] = st; }
    }
    __syncthreads();
    const int each = p.slices * p.n, total = K * each;
    double last_c = INFINITY;
    uint32_t last_b = 0, last_t = 0;
    for (int place = 0; place < p.n; ++place) {
        double c = -INFINITY;
        uint32_t b = 0xffffffffu, t = 0xffffffffu;                 // behind every candidate
        for (int i = tid; i < total; i += B_THREADS) {
            const uint32_t k = (uint32_t)(i / each), j = (uint32_t)(i - (int)k * each);
            const int row = g * K + (int)k;
            double cc = -INFINITY;
            uint32_t tt = j;
            if (state[k] == 0) {
                const unsigned long long key = __ldcg(p.keys + (size_t)row * each + j);
                if (key == 0) continue;
                tt = ~(uint32_t)key;
                cc = (double)__ldcg(p.scores + row) + ((double)beam_value(key) - lse[k]);
            } else {                                               // the first tokens, all at -infinity; a finished beam's pad at its score
                if (j > (uint32_t)p.n) continue;
                if (state[k] == 1) {
                    tt = j == 0 ? (uint32_t)p.pad : (j - 1 < (uint32_t)p.pad ? j - 1 : j);
                    if (j == 0) cc = (double)__ldcg(p.scores + row);
                }
                if (tt >= (uint32_t)p.vocab) continue;
            }
            if (place > 0 && !ahead(last_c, last_b, last_t, cc, k, tt)) continue;
            if (ahead(cc, k, tt, c, b, t)) { c = cc; b = k; t = tt; }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const double c2 = __shfl_xor_sync(0xffffffffu, c, o);
            const uint32_t b2 = __shfl_xor_sync(0xffffffffu, b, o), t2 = __shfl_xor_sync(0xffffffffu, t, o);
            if (ahead(c2, b2, t2, c, b, t)) { c = c2; b = b2; t = t2; }
        }
        __syncthreads();
        if (lane == 0) { bc[warp] = c; bb[warp] = b; bt[warp] = t; }
        __syncthreads();
        c = bc[0]; b = bb[0]; t = bt[0];
        for (int w = 1; w < B_THREADS / 32; ++w)
            if (ahead(bc[w], bb[w], bt[w], c, b, t)) { c = bc[w]; b = bb[w]; t = bt[w]; }
        last_c = c; last_b = b; last_t = t;
        if (tid == 0) {
            const size_t at = (size_t)g * p.n + place;
            p.out_scores[at] = (float)c;
            p.parents[at] = (int32_t)b;
            p.tokens[at] = (int32_t)t;
        }
    }
}

// ---------------------------------------------------------------- rows that follow their beams
// A thread has one word of every row of its group: it loads them all, then stores the ones that change, so that a row may be parent and
// child at once, and two children may have one parent.
constexpr int R_ARRAYS = 64, R_REGS = 16, R_THREADS = 256, R_SMEM_THREADS = 128, R_MAX = 64;

struct RowsParams {
    unsigned char* data[R_ARRAYS];
    long long words[R_ARRAYS];            // of a row
    const int32_t* src; const int32_t* dst;        // dst NULL: group g's rows g group ... take row src[i] of the group
    int rows, pairs, group;
};

template <typename W, bool SMEM>
__global__ void __launch_bounds__(SMEM ? R_SMEM_THREADS : R_THREADS) rows_kernel(const __grid_constant__ RowsParams p) {
    extern __shared__ __align__(16) unsigned char held[];
    __shared__ int from[R_MAX], to[R_MAX];
    griddep_wait();
    griddep_launch();
    const int tid = threadIdx.x, T = SMEM ? R_SMEM_THREADS : R_THREADS, first = blockIdx.y * p.group, n = min(p.group, p.pairs - first);
    if (tid < n) {
        int s = __ldcg(p.src + first + tid), d = first + tid;
        if (p.dst) {
            d = __ldcg(p.dst + first + tid);
            if ((unsigned)s >= (unsigned)p.rows) s = -1;
        } else
            s = (unsigned)s < (unsigned)p.group ? first + s : -1;
        if ((unsigned)d >= (unsigned)p.rows || s == d) s = -1;
        from[tid] = s;
        to[tid] = d;
    }
    __syncthreads();
    const long long words = p.words[blockIdx.z];
    W* data = reinterpret_cast<W*>(p.data[blockIdx.z]);
    for (long long c = (long long)blockIdx.x * T + tid; c < words; c += (long long)gridDim.x * T) {
        if constexpr (SMEM) {
            W* mine = reinterpret_cast<W*>(held) + tid;
            for (int i = 0; i < n; ++i)
                if (from[i] >= 0) mine[i * T] = __ldcg(data + from[i] * words + c);
            for (int i = 0; i < n; ++i)
                if (from[i] >= 0) data[to[i] * words + c] = mine[i * T];
        } else {
            W v[R_REGS];
#pragma unroll
            for (int i = 0; i < R_REGS; ++i)
                if (i < n && from[i] >= 0) v[i] = __ldcg(data + from[i] * words + c);
#pragma unroll
            for (int i = 0; i < R_REGS; ++i)
                if (i < n && from[i] >= 0) data[to[i] * words + c] = v[i];
        }
    }
}

template <typename W>
cudaError_t launch_rows(RowsParams& p, int arrays, cudaStream_t st) {
    long long most = 0;
    for (int a = 0; a < arrays; ++a) most = p.words[a] > most ? p.words[a] : most;
    const int blocks_y = (p.pairs + p.group - 1) / p.group;
    const bool smem = p.group > R_REGS;
    const int T = smem ? R_SMEM_THREADS : R_THREADS;
    long long x = (most + T - 1) / T;
    if (x > 65535) x = 65535;
    const size_t bytes = smem ? (size_t)p.group * T * sizeof(W) : 0;
    if (smem) {
        if (cudaError_t e = cudaFuncSetAttribute(rows_kernel<W, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)((size_t)R_MAX * T * sizeof(W)))) return e;
        return launch_waiting(rows_kernel<W, true>, dim3((unsigned)x, blocks_y, arrays), dim3(T), bytes, st, p);
    }
    return launch_waiting(rows_kernel<W, false>, dim3((unsigned)x, blocks_y, arrays), dim3(T), 0, st, p);
}

}  // namespace

}  // namespace pgk

using namespace pgk;

extern "C" {

int pgk_beam_select(const void* logits, long ld, int dtype, const float* scores, const int32_t* finished, int pad_token, int groups, int beams, int vocab, int n,
                    float* out_scores, int32_t* out_parents, int32_t* out_tokens, void* stream) {
    PGK_REQUIRE(dtype >= 0 && dtype <= 2, "beam_select failed: unknown type %d", dtype);
    PGK_REQUIRE(groups >= 0 && beams > 0 && beams <= B_MAX_BEAMS && vocab > 0 && ld >= vocab, "beam_select failed: %d groups of %d beams (64 at most), %d tokens in rows of %ld", groups,
                beams, vocab, ld);
    PGK_REQUIRE(n > 0 && n <= B_MAX_N && (long long)n <= (long long)beams * vocab, "beam_select failed: %d of %d x %d candidates (64 at most)", n, beams, vocab);
    PGK_REQUIRE(!finished || (pad_token >= 0 && pad_token < vocab), "beam_select failed: pad token %d outside the vocabulary", pad_token);
    PGK_REQUIRE((long long)groups * beams <= 65535, "beam_select failed: %d groups of %d beams (65535 rows at most)", groups, beams);
    if (groups == 0) return 0;
    PGK_REQUIRE(logits && scores && out_scores && out_parents && out_tokens, "beam_select failed: no logits, scores or outputs");
    const cudaStream_t st = (cudaStream_t)stream;
    BeamParams p = {};
    p.x = logits; p.ld = ld; p.scores = scores; p.finished = finished;
    p.pad = pad_token; p.beams = beams; p.vocab = vocab; p.n = n;
    p.slices = (vocab + B_SLICE - 1) / B_SLICE;
    p.out_scores = out_scores; p.parents = out_parents; p.tokens = out_tokens;
    const size_t rows = (size_t)groups * beams, parts = rows * p.slices * sizeof(float2), keys = rows * p.slices * n * sizeof(unsigned long long);
    void* ws = nullptr;
    if (int rc = scratch_alloc(&ws, keys + parts, st)) return rc;
    p.keys = (unsigned long long*)ws;
    p.part = (float2*)((char*)ws + keys);
    auto kernel = dtype == 0 ? beam_rows_kernel<0> : (dtype == 1 ? beam_rows_kernel<1> : beam_rows_kernel<2>);
    cudaError_t e = launch_waiting(kernel, dim3(p.slices, (unsigned)rows), dim3(B_THREADS), 0, st, p);
    if (e == cudaSuccess) e = launch_waiting(beam_merge_kernel, dim3(groups), dim3(B_THREADS), 0, st, p);
    if (int rc = scratch_free(ws, st)) return rc;
    PGK_CUDA(e);
    return 0;
}

int pgk_copy_rows(void* const* host_arrays, const int64_t* host_row_bytes, int n_arrays, int rows, const int32_t* src, const int32_t* dst, int pairs, int group,
                  void* stream) {
    PGK_REQUIRE(n_arrays >= 0 && rows >= 0 && pairs >= 0, "copy_rows failed: %d arrays of %d rows, %d pairs", n_arrays, rows, pairs);
    if (n_arrays == 0 || pairs == 0) return 0;
    PGK_REQUIRE(host_arrays && host_row_bytes && src, "copy_rows failed: no arrays or rows");
    PGK_REQUIRE(group > 0 && group <= R_MAX, "copy_rows failed: groups of %d rows (64 at most)", group);
    PGK_REQUIRE(dst || (pairs <= rows && pairs % group == 0), "copy_rows failed: %d rows in groups of %d of %d", pairs, group, rows);
    PGK_REQUIRE((pairs + group - 1) / group <= 65535, "copy_rows failed: %d pairs", pairs);
    uintptr_t bits = 0;
    for (int a = 0; a < n_arrays; ++a) {
        PGK_REQUIRE(host_arrays[a] && host_row_bytes[a] >= 0, "copy_rows failed: array %d is missing", a);
        bits |= (uintptr_t)host_arrays[a] | (uintptr_t)host_row_bytes[a];
    }
    const int size = bits % 16 == 0 ? 16 : (bits % 4 == 0 ? 4 : 1);
    RowsParams p = {};
    p.src = src; p.dst = dst; p.rows = rows; p.pairs = pairs; p.group = group;
    for (int a = 0; a < n_arrays; a += R_ARRAYS) {
        const int m = n_arrays - a < R_ARRAYS ? n_arrays - a : R_ARRAYS;
        long long most = 0;
        for (int i = 0; i < m; ++i) {
            p.data[i] = (unsigned char*)host_arrays[a + i];
            p.words[i] = host_row_bytes[a + i] / size;
            most = p.words[i] > most ? p.words[i] : most;
        }
        if (most == 0) continue;
        const cudaStream_t st = (cudaStream_t)stream;
        PGK_CUDA(size == 16 ? launch_rows<uint4>(p, m, st) : (size == 4 ? launch_rows<uint32_t>(p, m, st) : launch_rows<unsigned char>(p, m, st)));
    }
    return 0;
}

}  // extern "C"
