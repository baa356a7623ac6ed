// beam.cu -- a step of beam search: the best continuations of every group of beams, and the rows of memory that follow them.
//
//   c[k, v] = score[k] + (x[k, v] - log sum_u exp x[k, u]);  the n largest of a group's beams x vocabulary, ties to the lowest (beam, token)
//
// What bounds the selection: the logits, read once, and two launches.  A block takes up to 8192 logits of a row into registers: their maximum, the sum of
// their exponentials, and their n best by the key (value, token), which no two share.  Elements below a bound are left out: with k = ceil(n / 8), the
// smallest of its eight warps' k-th largest per-thread maxima, which at least n elements reach; what passes, some dozens of random logits, is ranked by
// counting.  Where more pass than the list holds (logits that are all the same, say) the bound is the n-th largest of the 256 per-thread maxima
// by key, which n threads' elements at most can reach.  A slice's sum is float32 (its 8192 terms: 4e-8 of a score).  A block per group then forms the rows' logarithms and takes the best of the sorted lists'
// heads n times, in float64, so that beams whose candidates lie within float32 rounding of each other keep their order.
// Measured: 4 beams of 32768 tokens 8.8 to 9.3 us, 128 of 151936 27.6 to 28.4: 17 for the rows (78 MB, 4.6 TB/s; half of the issue slots), the rest one warp a group
// over the heads.
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
    uint32_t beam_mul;                    // i / (slices n) = hi(i beam_mul) for as many entries as fit shared memory
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
    if constexpr (DT == 0) return __ldcg((const float*)x + i);
    else if constexpr (DT == 1) return __half2float(__ushort_as_half(ld_act2((const uint16_t*)x + i)));
    else return bf16_bits_to_f32(ld_act2((const uint16_t*)x + i));
}
// four neighbouring logits; `wide`: they start on a 16-byte (8-byte, of 16 bits) boundary and all exist
template <int DT>
__device__ __forceinline__ void beam_load4(const void* x, size_t i, bool wide, int exist, float (&v)[4]) {
    if constexpr (DT == 0) {
        const float* p = (const float*)x + i;
        if (wide) {
            const uint4 w = ldg_stream(p);
            v[0] = __uint_as_float(w.x); v[1] = __uint_as_float(w.y); v[2] = __uint_as_float(w.z); v[3] = __uint_as_float(w.w);
        } else {
#pragma unroll
            for (int c = 0; c < 4; ++c) v[c] = c < exist ? __ldcg(p + c) : -INFINITY;
        }
    } else {
        const uint16_t* p = (const uint16_t*)x + i;
        uint16_t h[4] = {};
        if (wide) {
            const uint2 w = __ldcg((const uint2*)p);
            h[0] = (uint16_t)w.x; h[1] = (uint16_t)(w.x >> 16); h[2] = (uint16_t)w.y; h[3] = (uint16_t)(w.y >> 16);
        } else {
#pragma unroll
            for (int c = 0; c < 4; ++c)
                if (c < exist) h[c] = ld_act2(p + c);
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) v[c] = c < exist ? (DT == 1 ? __half2float(__ushort_as_half(h[c])) : bf16_bits_to_f32(h[c])) : -INFINITY;
    }
}

// the place of `mine` among the block's values: how many are larger (they are all different, or 0)
__device__ __forceinline__ int rank_of(const unsigned long long* all, int count, unsigned long long mine) {
    int r = 0;
    for (int i = 0; i < count; ++i) r += all[i] > mine;
    return r;
}

template <int DT>
__global__ void __launch_bounds__(B_THREADS, 4) beam_rows_kernel(const __grid_constant__ BeamParams p) {
    constexpr int WARPS = B_THREADS / 32;
    __shared__ unsigned long long best[B_THREADS], list[B_LIST], bound;
    __shared__ float red[WARPS];
    __shared__ uint32_t kth[WARPS];
    __shared__ int count;
    griddep_wait();
    griddep_launch();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, slice = blockIdx.x, row = blockIdx.y;
    if (p.finished && __ldcg(p.finished + row) != 0) return;
    const int from = slice * B_SLICE, n_here = min(B_SLICE, p.vocab - from);
    const char* x = (const char*)p.x + (size_t)row * p.ld * (DT == 0 ? 4 : 2);
    const bool aligned = ((uintptr_t)x & (DT == 0 ? 15 : 7)) == 0;
    // element 4 (256 e + tid) + c of the slice is v[4 e + c]
    float v[B_EPT];
#pragma unroll
    for (int e = 0; e < B_EPT / 4; ++e) {
        const int i = 4 * (e * B_THREADS + tid);
        beam_load4<DT>(x, (size_t)from + i, aligned && i + 4 <= n_here, n_here - i, *(float (*)[4])(v + 4 * e));
    }
    float four[B_EPT / 4], top = -INFINITY;                        // the maxima of neighbouring fours
#pragma unroll
    for (int e = 0; e < B_EPT / 4; ++e) {
        four[e] = fmaxf(fmaxf(v[4 * e], v[4 * e + 1]), fmaxf(v[4 * e + 2], v[4 * e + 3]));
        top = fmaxf(top, four[e]);
    }
    if (tid == 0) { count = 0; bound = 0; }
    // the warp's k-th largest maximum, as ordered bits; 0 where fewer lanes have an element
    {
        const float mine = top;
        uint32_t left = 4 * tid < n_here ? (uint32_t)(beam_key(mine, 0) >> 32) : 0u, got = 0;
        const int k = (p.n + WARPS - 1) / WARPS;
        for (int i = 0; i < k; ++i) {
            got = __reduce_max_sync(0xffffffffu, left);
            const uint32_t who = __ballot_sync(0xffffffffu, left == got);
            if (lane == __ffs(who) - 1) left = 0;
        }
        if (lane == 0) kth[warp] = got;
    }
    top = warp_max(top);
    if (lane == 0) red[warp] = top;
    __syncthreads();
    uint32_t low = 0xffffffffu;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
        top = fmaxf(top, red[w]);
        low = min(low, kth[w]);
    }
    __syncthreads();
    float sum = 0.f;
    const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int e = 0; e < B_EPT; ++e) sum += ex2((v[e] - base) * 1.4426950408889634f);      // off by 2^-24 of the distance: terms that count lie near the maximum
    const float cut = low == 0 ? -INFINITY : __uint_as_float(low ^ ((low >> 31) ? 0x80000000u : 0xffffffffu));
#pragma unroll
    for (int e = 0; e < B_EPT / 4; ++e)
        if (four[e] >= cut) {
            const int i = 4 * (e * B_THREADS + tid);
#pragma unroll
            for (int c = 0; c < 4; ++c)
                if (v[4 * e + c] >= cut && i + c < n_here) {
                    const int at = atomicAdd(&count, 1);
                    if (at < B_LIST) list[at] = beam_key(v[4 * e + c], (uint32_t)(from + i + c));
                }
        }
    sum = warp_sum(sum);
    if (lane == 0) red[warp] = sum;
    __syncthreads();
    if (tid == 0) {
        sum = 0.f;
        for (int w = 0; w < WARPS; ++w) sum += red[w];
        // a row with a NaN or +infinity has no candidates: its sum is NaN, and its maximum says so
        p.part[(size_t)row * p.slices + slice] = make_float2(sum != sum ? NAN : top, sum);
    }
    if (count > B_LIST) {                                          // the whole block; the logits once more, element i by thread i % 256
        unsigned long long key = 0;
        __syncthreads();
        for (int i = tid; i < n_here; i += B_THREADS) {
            const float y = beam_logit<DT>(x, (size_t)from + i);
            if (y == y) key = max(key, beam_key(y, (uint32_t)(from + i)));
        }
        best[tid] = key;
        if (tid == 0) count = 0;
        __syncthreads();
        if (key && rank_of(best, B_THREADS, key) == p.n - 1) bound = key;
        __syncthreads();
        const unsigned long long least = bound;
        for (int i = tid; i < n_here; i += B_THREADS) {
            const float y = beam_logit<DT>(x, (size_t)from + i);
            const unsigned long long k = beam_key(y, (uint32_t)(from + i));
            if (y == y && k >= least) {
                const int at = atomicAdd(&count, 1);
                if (at < B_LIST) list[at] = k;
            }
        }
        __syncthreads();
    }
    const int m = min(count, B_LIST);
    unsigned long long* out = p.keys + ((size_t)row * p.slices + slice) * p.n;
    for (int i = tid; i < m; i += B_THREADS) {
        const int r = rank_of(list, m, list[i]);
        if (r < p.n) out[r] = list[i];
    }
    for (int i = m + tid; i < p.n; i += B_THREADS) out[i] = 0;
}

// float64 as ordered bits, 0 below all (NaN is -infinity)
__device__ __forceinline__ unsigned long long ordered(double c) {
    const unsigned long long u = (unsigned long long)__double_as_longlong(c == c ? c : -INFINITY);
    return u ^ ((u >> 63) ? ~0ull : 1ull << 63);
}
__device__ __forceinline__ double unordered(unsigned long long k) { return __longlong_as_double((long long)(k ^ ((k >> 63) ? 1ull << 63 : ~0ull))); }

// A list per (beam, slice), best first; lists in the order of their tokens, so that of equal heads the lowest list's wins.  HELD: all scores in shared memory.
template <bool HELD>
__global__ void __launch_bounds__(B_THREADS) beam_merge_kernel(const __grid_constant__ BeamParams p) {
    constexpr int WARPS = B_THREADS / 32;
    extern __shared__ __align__(16) unsigned char smem[];          // heads [lists], next [lists], then scores [lists][n]
    __shared__ double lse[B_MAX_BEAMS], base[B_MAX_BEAMS];
    __shared__ int state[B_MAX_BEAMS];             // 0: candidates from the row's lists; 1: finished; 2: nothing but -infinity
    __shared__ unsigned long long won_key[B_MAX_N];
    __shared__ int won_list[B_MAX_N], won_at[B_MAX_N];
    griddep_wait();
    griddep_launch();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = blockIdx.x, K = p.beams, lists = K * p.slices;
    unsigned long long* const heads = (unsigned long long*)smem;
    int* const next = (int*)(heads + lists);
    unsigned long long* const held = (unsigned long long*)(smem + (((size_t)lists * 12 + 15) & ~(size_t)15));
    if constexpr (HELD) {                          // the lists come while the logarithms are formed (those of beams that have none: anything)
        for (int i = tid; i < lists * p.n; i += B_THREADS)
            asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(smem_u32(held + i)), "l"(p.keys + (size_t)g * lists * p.n + i) : "memory");
        cp_async_commit();
    }
    for (int k = warp; k < K; k += WARPS) {
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
                if (!bad && q.x > -INFINITY) sum += (double)q.y * (double)expf(q.x - top);
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (bad) st = 2;
            else l = (double)top + log(sum);
        }
        if (lane == 0) { lse[k] = l; base[k] = (double)score; state[k] = st; }
    }
    for (int i = tid; i < lists; i += B_THREADS) next[i] = 0;
    __syncthreads();
    // entry j of list i: its score and its token
    auto token_of = [&](int i, int j) -> uint32_t {
        const int st = state[i / p.slices];
        if (st == 0) return ~(uint32_t)__ldcg(p.keys + ((size_t)g * lists + i) * p.n + j);
        if (st == 2) return (uint32_t)j;
        return j == 0 ? (uint32_t)p.pad : (uint32_t)(j - 1 < p.pad ? j - 1 : j);
    };
    auto score_of = [&](unsigned long long key, int k, bool first_list, int j) -> unsigned long long {
        const int st = state[k];
        if (st == 0) return key ? ordered(base[k] + ((double)beam_value(key) - lse[k])) : 0;
        if (!first_list || j >= p.vocab) return 0;                 // the first tokens, all at -infinity; a finished beam's pad at its score
        return ordered(st == 1 && j == 0 ? base[k] : -INFINITY);
    };
    if constexpr (HELD) {
        cp_async_wait<0>();
        __syncthreads();
        for (int i = tid; i < lists * p.n; i += B_THREADS) {
            const int k = p.beam_mul ? (int)__umulhi((uint32_t)i, p.beam_mul) : i, in_beam = i - k * p.slices * p.n;
            held[i] = score_of(held[i], k, in_beam < p.n, in_beam);
        }
        __syncthreads();
    }
    auto head = [&](int i) -> unsigned long long {
        const int j = next[i];
        if (j >= p.n) return 0;
        if constexpr (HELD) return held[i * p.n + j];
        else return score_of(__ldcg(p.keys + ((size_t)g * lists + i) * p.n + j), i / p.slices, i % p.slices == 0, j);
    };
    for (int i = tid; i < lists; i += B_THREADS) heads[i] = head(i);
    __syncthreads();
    if (warp == 0) {                               // one warp: its lanes have every 32nd list, and no barrier stands between two places
        unsigned long long mine = 0;
        int which = 0;
        auto look = [&] {                          // the best head of this lane's lists
            mine = 0;
            for (int i = lane; i < lists; i += 32) {
                const unsigned long long h = heads[i];
                if (h > mine) { mine = h; which = i; }
            }
        };
        look();
        for (int place = 0; place < p.n; ++place) {
            const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(mine >> 32));
            const bool in = (uint32_t)(mine >> 32) == hi;
            const uint32_t lo = __reduce_max_sync(0xffffffffu, in ? (uint32_t)mine : 0u);
            const int list = (int)__reduce_min_sync(0xffffffffu, in && (uint32_t)mine == lo ? (uint32_t)which : 0x7fffffffu);       // of equals the lowest
            if (in && (uint32_t)mine == lo && which == list) {
                won_key[place] = mine;
                won_list[place] = list;
                won_at[place] = next[list]++;
                heads[list] = head(list);
                look();
            }
            __syncwarp();
        }
    }
    __syncthreads();
    if (tid < p.n) {
        const size_t at = (size_t)g * p.n + tid;
        p.out_scores[at] = (float)unordered(won_key[tid]);
        p.parents[at] = won_list[tid] / p.slices;
        p.tokens[at] = (int32_t)token_of(won_list[tid], won_at[tid]);
    }
}

// ---------------------------------------------------------------- rows that follow their beams
// A thread has one word of every row of its group: it loads them all, then stores the ones that change, so that a row may be parent and
// child at once, and two children may have one parent.
// What bounds it: memory (16 arrays of 32 rows of 1 MB in groups of 8: 84.3 us, 6.0 TB/s of what is read and written).  Groups of up to 16 rows go through
// registers, as many as a group of 4, 8 or 16 needs, larger ones through shared memory, which is slower where both would do (us, 8 arrays of 32 rows of 1 MB,
// groups of 8 58.9 / 68, of 16 65 / 104); its copies are asynchronous, all of a thread's on their way at once (64 rows, 815 waited for one by one, 144 so), in
// small blocks, so that a block's loads run beside another's stores (64 rows in blocks of 128 / 64 / 32 threads 183 / 144 / 152).
constexpr int R_ARRAYS = 64, R_REGS = 16, R_THREADS = 256, R_SMEM_THREADS = 64, R_MAX = 64;

struct RowsParams {
    unsigned char* data[R_ARRAYS];
    long long words[R_ARRAYS];            // of a row
    const int32_t* src; const int32_t* dst;        // dst NULL: group g's rows g group ... take row src[i] of the group
    int rows, pairs, group;
};

template <typename W, int REGS>
__global__ void __launch_bounds__(REGS ? R_THREADS : R_SMEM_THREADS) rows_kernel(const __grid_constant__ RowsParams p) {
    extern __shared__ __align__(16) unsigned char held[];
    __shared__ int from[R_MAX], to[R_MAX];
    griddep_wait();
    griddep_launch();
    const int tid = threadIdx.x, T = REGS ? R_THREADS : R_SMEM_THREADS, first = blockIdx.y * p.group, n = min(p.group, p.pairs - first);
    for (int i = tid; i < n; i += T) {
        int s = __ldcg(p.src + first + i), d = first + i;
        if (p.dst) {
            d = __ldcg(p.dst + first + i);
            if ((unsigned)s >= (unsigned)p.rows) s = -1;
        } else
            s = (unsigned)s < (unsigned)p.group ? first + s : -1;
        if ((unsigned)d >= (unsigned)p.rows || s == d) s = -1;
        from[i] = s;
        to[i] = d;
    }
    __syncthreads();
    const long long words = p.words[blockIdx.z];
    W* data = reinterpret_cast<W*>(p.data[blockIdx.z]);
    for (long long c = (long long)blockIdx.x * T + tid; c < words; c += (long long)gridDim.x * T) {
        if constexpr (REGS == 0) {
            W* mine = reinterpret_cast<W*>(held) + tid;
            for (int i = 0; i < n; ++i) {
                if (from[i] < 0) continue;
                if constexpr (sizeof(W) == 16) cp_async16(mine + i * T, data + from[i] * words + c);
                else if constexpr (sizeof(W) == 4) cp_async4(mine + i * T, data + from[i] * words + c);
                else mine[i * T] = __ldcg(data + from[i] * words + c);
            }
            if constexpr (sizeof(W) >= 4) {
                cp_async_commit();
                cp_async_wait<0>();                        // a thread reads what it has copied itself
            }
            for (int i = 0; i < n; ++i)
                if (from[i] >= 0) data[to[i] * words + c] = mine[i * T];
        } else {
            W v[REGS];
#pragma unroll
            for (int i = 0; i < REGS; ++i)
                if (i < n && from[i] >= 0) v[i] = __ldcg(data + from[i] * words + c);
#pragma unroll
            for (int i = 0; i < REGS; ++i)
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
        static bool configured = false;
        if (!configured) {
            if (cudaError_t e = cudaFuncSetAttribute(rows_kernel<W, 0>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)((size_t)R_MAX * T * sizeof(W)))) return e;
            configured = true;
        }
        return launch_waiting(rows_kernel<W, 0>, dim3((unsigned)x, blocks_y, arrays), dim3(T), bytes, st, p);
    }
    auto kernel = p.group <= 4 ? rows_kernel<W, 4> : (p.group <= 8 ? rows_kernel<W, 8> : rows_kernel<W, 16>);
    return launch_waiting(kernel, dim3((unsigned)x, blocks_y, arrays), dim3(T), 0, st, p);
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
    PGK_REQUIRE((long long)vocab <= 250ll * B_SLICE, "beam_select failed: %d tokens (%lld at most)", vocab, 250ll * B_SLICE);
    if (groups == 0) return 0;
    PGK_REQUIRE(logits && scores && out_scores && out_parents && out_tokens, "beam_select failed: no logits, scores or outputs");
    const cudaStream_t st = (cudaStream_t)stream;
    BeamParams p = {};
    p.x = logits; p.ld = ld; p.scores = scores; p.finished = finished;
    p.pad = pad_token; p.beams = beams; p.vocab = vocab; p.n = n;
    p.slices = (vocab + B_SLICE - 1) / B_SLICE;
    p.beam_mul = p.slices * n > 1 ? (uint32_t)((1ull << 32) / (unsigned)(p.slices * n)) + 1 : 0;
    p.out_scores = out_scores; p.parents = out_parents; p.tokens = out_tokens;
    const size_t rows = (size_t)groups * beams, parts = rows * p.slices * sizeof(float2), keys = rows * p.slices * n * sizeof(unsigned long long);
    void* ws = nullptr;
    if (int rc = scratch_alloc(&ws, keys + parts, st)) return rc;
    p.keys = (unsigned long long*)ws;
    p.part = (float2*)((char*)ws + keys);
    auto kernel = dtype == 0 ? beam_rows_kernel<0> : (dtype == 1 ? beam_rows_kernel<1> : beam_rows_kernel<2>);
    cudaError_t e = launch_waiting(kernel, dim3(p.slices, (unsigned)rows), dim3(B_THREADS), 0, st, p);
    const size_t next = ((size_t)beams * p.slices * 12 + 15) & ~(size_t)15, held = next + (size_t)beams * p.slices * n * 8;
    const size_t most = 200 * 1024;
    static bool configured = false;
    if (!configured && e == cudaSuccess) {
        e = cudaFuncSetAttribute(beam_merge_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(beam_merge_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most);
        configured = e == cudaSuccess;
    }
    if (e == cudaSuccess)
        e = held <= most ? launch_waiting(beam_merge_kernel<true>, dim3(groups), dim3(B_THREADS), held, st, p)
                         : launch_waiting(beam_merge_kernel<false>, dim3(groups), dim3(B_THREADS), next, st, p);
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
