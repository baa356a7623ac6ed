// kv4_attention.cu -- attention over the four-bit paged cache (kv4.cuh has the format): decoded tokens, and a few rows a sequence.
//
//   o[t, h, :] = sum_j w_j v_j / (sum_j w_j + exp(sink_h - m)),   w_j = exp(x_j - m),   x_j = scale q[t, h, :] . k_j, capped c tanh(x_j / c)
//   over the keys j <= pos(t), with a window also j > pos(t) - window;  pos(t) = context - rows + (t's place among its sequence's rows)
//
// With k_j = s (c - z) per group of 32 elements, both sums run over codes: q . k = sum_g s_g (q_g . c_g - z_g sum q_g), and of a group's values
// sum_j w_j v_j = sum_j (w_j s_j) c_j - sum_j (w_j s_j) z_j.  What this makes of the work:
//   * codes go to the tensor cores (mma.sync m16n8k16) as they are.  Four bits in the lowest places of a float16 are c 2^-24, four bits above them c 2^-20,
//     of a bfloat16 c 2^-133 and c 2^-129: subnormal numbers, which the products take exactly (tested), so that two elements cost one AND.
//     The query carries 2^-4 where the code carries 2^4, and a power of two that brings its largest element below 2^10 (2^11).
//   * A is 16 keys of codes, B eight query rows: float16 queries (rows of 16 bits: exact for elements above 2^-22 of their row's largest, bfloat16, or 2^-19, float16,
//     and within 2^-30 of it below; float32 rows: two terms, 22 bits of the largest), a group's sum starts at -z sum q_g, and a group's scale is one
//     multiply-add per (key, row).
//   * of the values A is 16 elements by 16 keys -- a lane's bytes of two keys, merged by one permutation --, B the weights times the group's scale and 2^64
//     (which keeps products with c 2^-133 normal), rounded to bfloat16 once for rows of that type; float16 rows have two such terms, 16 bits (one left
//     2^-9 of a weight beside an output's own 2^-12), float32 rows three, 24 bits.  The sum of w s z is
//     a product over the same rounded weights, so that what rounding does to codes of up to 15 is done to (c - z) only.
//   * S comes out as [key][row] and is needed as [key][row] operand of the other layout: movmatrix, two cycles for 64 numbers.
// What bounds it: with 64 and more sequences instructions, 340 for 16 keys of 128 elements and 8 rows, which would alone be issued in the time that the cache's
// bytes take (64 over 8192 keys, 64 / 8 heads of 128: 81 us), but are in 149 to 152: a scheduler has one to issue in 61 % of a SM's active cycles (latencies of
// dependent ones, the integer units 59 % taken), and SMs are active 88 % of the time, with 1024 blocks on 592 places.  With one sequence the chain of a
// launch, a page number, the rows and the fold (4096 keys: 9.6 us).  The same 64 with float16 rows 190 us, with float32 ones 279.
// A warp takes 32 keys at a time through a ring of its own in shared memory (cp.async, no barrier among warps), with its own maximum and sums;
// the warps fold in shared memory, and where a sequence's keys are cut over the blocks of a cluster, these fold through distributed shared memory.
//
// A row that sees no key gives zeros.
#include "kv4_attention.cuh"
#include "tc_common.cuh"
#include "../../include/pgk_b200.h"

namespace pgk {

int kv4_check(const char* fn, const void* data, int pages, int page_size, const void* table, int slots, int max_pages, int kv_heads, int dim);

namespace {

constexpr int F_KEYS = 32, F_STAGES = 2, F_CLUSTER = 8;
constexpr float F_LIFT = 18446744073709551616.f;                   // 2^64

// W warps a block; the rings, and behind them (float32 rows: in their place, afterwards) the warps' sums; queries in fragments; sums of queries
template <int G, int NT, int DT, int W> struct Few {
    static constexpr int THREADS = W * 32, RESIDENT = G * NT <= 4 ? 16 / W : 8 / W;
    static constexpr int STAGE = F_KEYS * 36 * G;                  // codes of K, of V, words of K, of V
    static constexpr int RINGS = W * F_STAGES * STAGE, FOLD = W * 8 * NT * (32 * G + 4) * 4;
    static constexpr bool RUNS = DT != 0;
    static constexpr int RUN = DT == 1 ? 8 : 16;                   // blocks whose values one accumulator sums: 32 products, with two terms or one
    static constexpr int SUMS = RUNS ? RINGS : 0, FRAG = RUNS ? RINGS + FOLD : (RINGS > FOLD ? RINGS : FOLD), QSUM = FRAG + G * 2 * NT * (DT == 0 ? 2 : 1) * 256, BYTES = QSUM + G * NT * (DT == 0 ? 2 : 1) * 128;
};

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16_k8(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t b0) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(b0));
}
__device__ __forceinline__ uint32_t transposed(uint32_t v) {       // an 8 x 8 matrix of 16-bit numbers over the warp
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
// A row of codes in the ring is G pieces of 16 bytes, in an order that keeps the lanes of one load off each other's banks: those of a quad's keys
// (rows r ... r + 7, all pieces) as well as those of a value's (every second row, one place).
template <int G>
__device__ __forceinline__ int piece(int row, int i) {
    if constexpr (G == 2) return i ^ ((row >> 2) & 1);
    else if constexpr (G == 4) return i ^ ((row >> 1) & 3);
    else if constexpr (G == 8) return i ^ ((row >> 1) & 3) << 1 ^ (row & 1);
    else return i;
}
// the G words that lane t of a quad has of a row
template <int G>
__device__ __forceinline__ void lds_codes(const unsigned char* rows, int row, int t, uint32_t (&w)[G]) {
    const unsigned char* at = rows + row * 16 * G;
    if constexpr (G % 4 == 0) {
#pragma unroll
        for (int i = 0; i < G; i += 4) {
            const uint4 v = *(const uint4*)(at + 16 * piece<G>(row, t * (G / 4) + i / 4));
            w[i] = v.x; w[i + 1] = v.y; w[i + 2] = v.z; w[i + 3] = v.w;
        }
    } else if constexpr (G == 2) {
        const uint2 v = *(const uint2*)(at + 16 * piece<G>(row, t >> 1) + 8 * (t & 1));
        w[0] = v.x; w[1] = v.y;
    } else if constexpr (G % 2 == 0) {
#pragma unroll
        for (int i = 0; i < G; i += 2) {
            const uint2 v = *(const uint2*)(at + 4 * (t * G + i));
            w[i] = v.x; w[i + 1] = v.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < G; ++i) w[i] = *(const uint32_t*)(at + 4 * (t * G + i));
    }
}
// the G group words of a row, two to a register
template <int G>
__device__ __forceinline__ void lds_groups(const unsigned char* p, uint32_t (&m)[(G + 1) / 2]) {
    if constexpr (G == 8) {
        const uint4 v = *(const uint4*)p;
        m[0] = v.x; m[1] = v.y; m[2] = v.z; m[3] = v.w;
    } else if constexpr (G == 4) {
        const uint2 v = *(const uint2*)p;
        m[0] = v.x; m[1] = v.y;
    } else if constexpr (G % 2 == 0) {
#pragma unroll
        for (int i = 0; i < G / 2; ++i) m[i] = *(const uint32_t*)(p + 4 * i);
    } else {
#pragma unroll
        for (int i = 0; i < G; ++i) {
            const uint32_t h = *(const uint16_t*)(p + 2 * i);
            m[i / 2] = i % 2 ? m[i / 2] | h << 16 : h;
        }
    }
}
__device__ __forceinline__ float group_scale(uint32_t m, int odd) { return __uint_as_float(odd ? m & 0x7ff00000u : (m << 16) & 0x7ff00000u); }
__device__ __forceinline__ void cp_async16_at(uint32_t smem, const void* g) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem), "l"(g) : "memory");
}

template <int DT>
__device__ __forceinline__ float row_element(const void* q, size_t i) {
    if constexpr (DT == 0) return __ldcg((const float*)q + i);
    else if constexpr (DT == 1) return __half2float(__ushort_as_half(ld_act2((const uint16_t*)q + i)));
    else return bf16_bits_to_f32(ld_act2((const uint16_t*)q + i));
}
struct Yes { static constexpr bool value = true; };
struct No { static constexpr bool value = false; };
__device__ __forceinline__ float finite(float v) { return fabsf(v) < INFINITY ? v : 0.f; }
template <int G, int NT, int DT, int W>
__global__ void __launch_bounds__(Few<G, NT, DT, W>::THREADS, Few<G, NT, DT, W>::RESIDENT) kv4_few_kernel(const __grid_constant__ Kv4AttnParams p) {
    using Smem = Few<G, NT, DT, W>;
    constexpr int D = 32 * G, DP = D + 4, ROWS = 8 * NT, WARPS = W, THREADS = Smem::THREADS, STAGE = Smem::STAGE;
    constexpr int QT = DT == 0 ? 2 : 1, PT = 3 - DT, MW = (G + 1) / 2;
    // Rows of 16 bits take a byte, c + 16 c' (a bfloat16 too, subnormal or of the first exponent), where they would take its lower four bits, and subtract the
    // product of the upper ones in the end: one operation in five less.  The difference costs four bits of the sums' 24, which therefore are short ones (RUN).
    constexpr bool BYTES = DT != 0;
    constexpr uint32_t LOW = BYTES ? 0x00ff00ffu : 0x000f000fu;
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ float fac_s[ROWS], wm[WARPS][ROWS], wl[WARPS][ROWS], block_m[ROWS], block_l[ROWS];
    __shared__ int lim_s[ROWS];
    griddep_wait();
    griddep_launch();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, gl = lane >> 2, t = lane & 3;
    const int seq = blockIdx.x / p.tiles, f0 = (blockIdx.x - seq * p.tiles) * ROWS, head = blockIdx.y, split = blockIdx.z;
    const int slot = __ldcg(p.seq_slots + seq), ctx = __ldcg(p.contexts + seq);
    const int first = p.starts ? __ldcg(p.starts + seq) : seq, n = p.starts ? __ldcg(p.starts + seq + 1) - first : 1;
    const int rows = min(min(n, p.max_rows), 0x7fffffff / p.rep) * p.rep;                  // of this head's group
    if (f0 >= rows || (unsigned)slot >= (unsigned)p.k.slots) return;                       // the whole cluster
    const int live = min(ROWS, rows - f0), i0 = f0 / p.rep, i1 = (f0 + live - 1) / p.rep;
    const int pos0 = ctx - n + i0, pos1 = ctx - n + i1;
    const int begin = kv4_first_key(p, pos0), end = min(min(pos1 + 1, ctx), p.max_keys);
    const int b0 = begin / F_KEYS, nb = max(0, (end + F_KEYS - 1) / F_KEYS - b0);
    const int per = (nb + p.splits - 1) / p.splits, bend = min(nb, (split + 1) * per) + b0;
    const int lo_max = kv4_first_key(p, pos1), hi_min = min(pos0 + 1, end);

    // ---------------- the ring: 32 keys of K and V, their words behind them
    unsigned char* const ring = smem + (size_t)warp * F_STAGES * STAGE;
    const uint32_t ring_at = smem_u32(ring);
    const int32_t* table = p.k.table + (size_t)slot * p.k.max_pages;
    const unsigned char* const khead = p.k.data + (size_t)head * p.head_bytes + lane * 16;
    const unsigned char* const vhead = p.v_data + (size_t)head * p.head_bytes + lane * 16;
    const int code_bytes = p.k.page_size * 16 * G;
    auto page_of = [&](uint32_t n) { return kv4_page_of(p, n); };
    auto pages_of = [&](int b, int (&pg)[2]) {                     // of the block's two halves; -1: nothing to see there
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int n = 2 * b + u;
            pg[u] = b < bend && 16 * n < end ? __ldcg(table + page_of(n)) : -1;
        }
    };
    auto fetch = [&](int b, int stage, const int (&pg)[2]) {       // returns which halves have a page
        const uint32_t to = ring_at + stage * STAGE;
        uint32_t ok = 0;
        long long at[2];                                           // of the half's codes, and of its words behind the page's codes
        int words[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const bool good = (unsigned)pg[u] < (unsigned)p.k.pages;
            const uint32_t n = 2 * b + u;
            const int row = good ? (int)(16u * n - page_of(n) * (uint32_t)p.k.page_size) : 0;
            ok |= (uint32_t)good << u;
            at[u] = (good ? pg[u] : 0) * p.page_bytes + row * (16 * G);
            words[u] = code_bytes - row * (14 * G);
        }
        if (b < bend) {
#pragma unroll
            for (int i = 0; i < G; ++i) {                          // 16 G copies a half: of either side G a lane
                const int c = i * 32 + lane, key = c / G, x = key * G + piece<G>(key, c - key * G);
                const bool second = G % 2 == 0 ? i >= G / 2 : c >= 16 * G;
                const long long from = (second ? at[1] - 256 * G : at[0]) + i * 512;
                cp_async16_at(to + x * 16, khead + from);
                cp_async16_at(to + F_KEYS * 16 * G + x * 16, vhead + from);
            }
#pragma unroll
            for (int i = 0; i < (8 * G + 31) / 32; ++i) {          // words: 4 G copies a side, 2 G of either half
                const int c = i * 32 + lane, side = c >= 4 * G, u = (c - side * 4 * G) >= 2 * G;
                if (c < 8 * G)
                    cp_async16_at(to + F_KEYS * 32 * G + c * 16, (side ? vhead : khead) + (u ? at[1] + words[1] : at[0] + words[0]) + i * 512 - (side * 4 * G + u * 2 * G) * 16);
            }
        }
        cp_async_commit();
        return ok;
    };
    int block, ahead[2];
    uint32_t have[F_STAGES];
    auto start = [&] {
        int now[2];
        block = b0 + split * per + warp;
        pages_of(block, now);
        pages_of(block + WARPS, ahead);
        have[0] = fetch(block, 0, now);
    };
    start();

    // ---------------- queries into fragments
    unsigned char* const frag = smem + Smem::FRAG;
    unsigned char* const qsum = smem + Smem::QSUM;                 // [G][NT][term][lane]: -sum of the group's queries, in a term of float16 a quad's lane
    for (int c = warp; c < ROWS; c += WARPS) {
        const int f = f0 + c, i = f / p.rep, tok = first + i;
        const bool there = c < live && tok >= 0 && tok < p.tokens;
        float x[G], top = 0.f;
#pragma unroll
        for (int g = 0; g < G; ++g) {
            x[g] = there ? row_element<DT>(p.q, (size_t)tok * p.q_ld + (size_t)(head * p.rep + f - i * p.rep) * D + 32 * g + lane) : 0.f;
            top = fmaxf(top, fabsf(x[g]));
        }
        top = warp_max(top);
        // 2^9 <= top 2^(e - 127) < 2^10: 32 of them have a sum in float16; of float32 rows 2^10 <= ... < 2^11
        const uint32_t e = min(max((DT == 0 ? 264u : 263u) - min(__float_as_uint(top) >> 23, 262u), 4u), 250u);
        const float mult = __uint_as_float(e << 23);
        const int w = lane, qt = w >> 3, nib = w & 7, pr = nib & 3;
#pragma unroll
        for (int g = 0; g < G; ++g) {
            // Terms of float32 rows are integers of 11 bits, the second of 2^-12: their products' sums have 20 bits and are exact, each in an accumulator of
            // its own (sums of floating terms in one, truncated at every product, were off by 2e-6 of a score, ten times float32's own).
            const float y = x[g] * mult, first = DT == 0 ? rintf(y) : y, f = pr & 1 ? 0.0625f : 1.f;
#pragma unroll
            for (int term = 0; term < QT; ++term) {
                const float part = term == 0 ? first : rintf((y - first) * 4096.f) * (1.f / 4096.f);
                const __half h = __float2half_rn(part * f);
                *(uint16_t*)(frag + ((((size_t)(g * 2 + (pr >> 1)) * NT + (c >> 3)) * QT + term) * 32 + (c & 7) * 4 + qt) * 8 + (pr & 1) * 4 + (nib >> 2) * 2) =
                    __half_as_ushort(h);
                float sum = -warp_sum(__half2float(h) * (pr & 1 ? 16.f : 1.f));
                // the lane i of a quad multiplies its copy of z by piece i; an even group's z is in a word's lower half, an odd one's in the upper
                for (int i = 0; i < 4; ++i) {
                    const __half piece = __float2half_rn(DT == 0 ? fminf(fmaxf(sum, -32768.f), 32768.f) : sum);
                    sum -= __half2float(piece);
                    if (lane == i) *(uint32_t*)(qsum + ((size_t)((g * NT + (c >> 3)) * QT + term) * 32 + (c & 7) * 4 + i) * 4) = (uint32_t)__half_as_ushort(piece) << (g & 1 ? 16 : 0);
                }
            }
        }
        if (lane == 0) {
            fac_s[c] = fminf(p.scale_log2 * __uint_as_float((254u - e) << 23) * 16777216.f, 3.4028235e38f);       // (scores of 10^36: no infinity that a zero meets)
            lim_s[c] = there ? ctx - n + i : -1;
        }
    }
    __syncthreads();
    float fac[NT][2], m[NT][2], l[NT][2], acc[2 * G][NT][4], zac[NT][4];
    int lim[NT][2];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            fac[j][c] = p.cap_log2 > 0.f ? 1.f : fac_s[8 * j + 2 * t + c];
            lim[j][c] = lim_s[8 * j + 2 * t + c];
        }
    const uint32_t half_sel = gl & 1 ? 0x7632u : 0x5410u;
    bool careful = false, huge = false, bad, fresh;
    // The accumulators into the warp's sums.  A lane has columns 8 j + 2 t + c, elements 32 g + 4 gl ... + 3 of them, and nobody else does before the warps fold.
    float* const fold = (float*)(smem + Smem::SUMS);               // [WARPS][ROWS][DP]
    auto sum_at = [&](int j, int c, int g) { return (float4*)(fold + ((size_t)warp * ROWS + 8 * j + 2 * t + c) * DP + 32 * g + 4 * gl); };
    auto put = [&] {
        const float even = 5.9029581035870565e20f, odd = 3.6893488147419103e19f;  // 2^133 / 2^64 and 2^129 / 2^64
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            bad |= zac[j][0] != zac[j][0] || zac[j][1] != zac[j][1];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    const float z = __shfl_sync(0xffffffffu, zac[j][c], g * 4 + t) * even;
                    const float a0 = BYTES ? acc[2 * g][j][c] - acc[2 * g][j][2 + c] : acc[2 * g][j][c];
                    const float a2 = BYTES ? acc[2 * g + 1][j][c] - acc[2 * g + 1][j][2 + c] : acc[2 * g + 1][j][c];
                    float4 o = make_float4(fmaf(a0, even, -z), fmaf(acc[2 * g][j][2 + c], odd, -z), fmaf(a2, even, -z), fmaf(acc[2 * g + 1][j][2 + c], odd, -z));
                    float4* const at = sum_at(j, c, g);
                    if (!fresh) {
                        const float4 v = *at;
                        o.x += v.x; o.y += v.y; o.z += v.z; o.w += v.w;
                    }
                    *at = o;
                }
                float sum = l[j][c] * (1.f / F_LIFT);
#pragma unroll
                for (int o = 4; o <= 16; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                if (gl == 0) wl[warp][8 * j + 2 * t + c] = fresh ? sum : wl[warp][8 * j + 2 * t + c] + sum;
                l[j][c] = 0.f;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) zac[j][i] = 0.f;
#pragma unroll
            for (int i = 0; i < 2 * G; ++i)
#pragma unroll
                for (int c = 0; c < 4; ++c) acc[i][j][c] = 0.f;
        }
        fresh = false;
    };
again:
    bad = false;
    fresh = true;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            m[j][c] = -INFINITY;
            l[j][c] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) zac[j][i] = 0.f;
#pragma unroll
        for (int i = 0; i < 2 * G; ++i)
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[i][j][c] = 0.f;
    }

    for (int k = 0; block < bend; ++k, block += WARPS) {
        const int stage = k % F_STAGES;
        __syncwarp();                                              // the other stage has been read
        {
            int next[2];
            pages_of(block + 2 * WARPS, next);
            have[(k + 1) % F_STAGES] = fetch(block + WARPS, (k + 1) % F_STAGES, ahead);
            ahead[0] = next[0]; ahead[1] = next[1];
        }
        cp_async_wait<F_STAGES - 1>();
        __syncwarp();
        const unsigned char* const kc = ring + stage * STAGE;
        const unsigned char* const vc = kc + F_KEYS * 16 * G;
        const unsigned char* const kwords = kc + F_KEYS * 32 * G;
        const unsigned char* const vwords = kwords + F_KEYS * 2 * G;
        const int key0 = block * F_KEYS;
        const bool edge = key0 < lo_max || key0 + F_KEYS > hi_min || have[stage] != 3u;

        // ---------------- scores
        float s[2][NT][4];
        {
            uint32_t kw[2][2][G], km[2][2][MW], kz[2][2][MW];
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const int row = 16 * u + 8 * r + gl;
                    lds_codes<G>(kc, row, t, kw[u][r]);
                    lds_groups<G>(kwords + row * 2 * G, km[u][r]);
#pragma unroll
                    for (int i = 0; i < MW; ++i) kz[u][r][i] = km[u][r][i] & 0x000f000fu;
                }
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[u][j][i] = 0.f;
#pragma unroll
            for (int g = 0; g < G; ++g) {
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    uint32_t qs[QT];
                    uint2 b[2][QT];
#pragma unroll
                    for (int term = 0; term < QT; ++term) qs[term] = *(const uint32_t*)(qsum + (((g * NT + j) * QT + term) * 32 + lane) * 4);
#pragma unroll
                    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
                        for (int term = 0; term < QT; ++term)
                            b[ks][term] = *(const uint2*)(frag + ((((size_t)(g * 2 + ks) * NT + j) * QT + term) * 32 + lane) * 8);
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const float s0 = group_scale(km[u][0][g / 2], g & 1), s1 = group_scale(km[u][1][g / 2], g & 1);
                        float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int term = QT - 1; term >= 0; --term) {
                            float a[4] = {0.f, 0.f, 0.f, 0.f};
                            mma_f16_k8(a, kz[u][0][g / 2], kz[u][1][g / 2], qs[term]);
#pragma unroll
                            for (int ks = 0; ks < 2; ++ks) {
                                const uint32_t w0 = ks ? kw[u][0][g] >> 8 : kw[u][0][g], w1 = ks ? kw[u][1][g] >> 8 : kw[u][1][g];
                                mma_f16(a, w0 & 0x000f000fu, w1 & 0x000f000fu, w0 & 0x00f000f0u, w1 & 0x00f000f0u, b[ks][term].x, b[ks][term].y);
                            }
#pragma unroll
                            for (int i = 0; i < 4; ++i) c[i] = term == QT - 1 ? a[i] : c[i] + a[i];
                        }
                        s[u][j][0] = fmaf(s0, c[0], s[u][j][0]);
                        s[u][j][1] = fmaf(s0, c[1], s[u][j][1]);
                        s[u][j][2] = fmaf(s1, c[2], s[u][j][2]);
                        s[u][j][3] = fmaf(s1, c[3], s[u][j][3]);
                    }
                }
            }
        }
        // ---------------- weights
        if (p.cap_log2 > 0.f) {                                    // (fac is 1 then)
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {                  // float32 rows: 2^-22 of a cap of 50 would be a weight's 17th bit
                        float& x = s[u][j][i];
                        x *= fac_s[8 * j + 2 * t + (i & 1)];
                        if constexpr (DT == 0) x = p.cap_log2 * tanhf(x / p.cap_log2);
                        else x = p.cap_log2 * (p.cap_log2 > KV4_CAP_WIDE ? kv4_tanh_wide(x * kv4_cap_in(1.f, p.cap_log2)) : kv4_tanh(x * kv4_cap_in(1.f, p.cap_log2)));
                    }
        }
        uint32_t unseen = 0;                                       // of this lane's 8 NT (key, row)
        if (edge) {
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int key = key0 + 16 * u + 8 * (i >> 1) + gl, last = lim[j][i & 1];
                        if (key > last || key >= end || (p.window > 0 && last - key >= p.window) || !((have[stage] >> u) & 1u)) {
                            s[u][j][i] = -INFINITY;
                            unseen |= 1u << ((u * NT + j) * 4 + i);
                        }
                    }
        }
        bool up = false;
        float top[NT][2];
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                top[j][c] = fmaxf(fmaxf(s[0][j][c], s[0][j][2 + c]), fmaxf(s[1][j][c], s[1][j][2 + c])) * fac[j][c];
                up |= top[j][c] > m[j][c] + 8.f;
            }
        if (__any_sync(0xffffffffu, up)) {                         // a reference moves when its maximum has grown by 2^8 (or at all at first)
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                float f[2];
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    float best = top[j][c];
#pragma unroll
                    for (int o = 4; o <= 16; o <<= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, o));
                    best = fmaxf(best, m[j][c]);
                    f[c] = m[j][c] == -INFINITY ? 0.f : ex2(m[j][c] - best);
                    m[j][c] = best;
                    huge |= fabsf(best) > KV4_HUGE && best > -INFINITY;
                    l[j][c] *= f[c];
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) zac[j][i] *= f[i & 1];
#pragma unroll
                for (int i = 0; i < 2 * G; ++i)
#pragma unroll
                    for (int c = 0; c < 4; ++c) acc[i][j][c] *= f[c & 1];
                if (Smem::RUNS && !fresh) {
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
#pragma unroll
                        for (int g = 0; g < G; ++g) {
                            float4* const at = sum_at(j, c, g);
                            const float4 v = *at;
                            *at = make_float4(v.x * f[c], v.y * f[c], v.z * f[c], v.w * f[c]);
                        }
                        if (gl == 0) wl[warp][8 * j + 2 * t + c] *= f[c];
                    }
                }
            }
            huge = __any_sync(0xffffffffu, huge);
        }
        if (huge) {                                                // x - m of rounded x then: what rounding m left of a multiply-add's exact product may be anything
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[u][j][i] *= fac[j][i & 1];
        }
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                // Weights are 2^64 times theirs.  In rows of 16 bits the exponent has it, whose rounding then is 2^-18.
                const float base = (m[j][c] == -INFINITY ? 0.f : -m[j][c]) + (DT == 0 ? 0.f : 64.f);
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        float w = ex2(fmaf(s[u][j][2 * r + c], huge ? 1.f : fac[j][c], base));
                        if constexpr (DT == 0) w *= F_LIFT;
                        l[j][c] += w;
                        s[u][j][2 * r + c] = w;
                    }
            }
        // ---------------- values: one run of instructions for blocks without an edge
        auto values = [&](auto special) {
            constexpr bool SPECIAL = decltype(special)::value;
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                uint32_t vw[4][G], vz[4][MW], vm[2][MW];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int row = 16 * u + 2 * t + (i & 1) + 8 * (i >> 1);
                    lds_codes<G>(vc, row, gl >> 1, vw[i]);
                    lds_groups<G>(vwords + row * 2 * G, vz[i]);
                }
#pragma unroll
                for (int r = 0; r < 2; ++r) lds_groups<G>(vwords + (16 * u + 8 * r + gl) * 2 * G, vm[r]);
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    const uint32_t v0 = __byte_perm(vw[0][g], vw[1][g], half_sel), v1 = __byte_perm(vw[2][g], vw[3][g], half_sel);
                    const uint32_t v2 = BYTES ? __byte_perm(v0, 0, 0x4341) : v0 >> 8, v3 = BYTES ? __byte_perm(v1, 0, 0x4341) : v1 >> 8;
                    const uint32_t zmask = gl == g ? 0x000f000fu : 0u;
                    const uint32_t z0 = __byte_perm(vz[0][g / 2], vz[1][g / 2], g & 1 ? 0x7632 : 0x5410) & zmask;
                    const uint32_t z1 = __byte_perm(vz[2][g / 2], vz[3][g / 2], g & 1 ? 0x7632 : 0x5410) & zmask;
                    const float s0 = group_scale(vm[0][g / 2], g & 1), s1 = group_scale(vm[1][g / 2], g & 1);
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        // Float32 rows sum 16 keys here and add these sums: the products' own additions truncate, which made 1.6e-6 of an output over
                        // 15751 keys, and 3e-7 this way.
                        float part[3][4] = {};
                        float (&low)[4] = DT == 0 ? part[0] : acc[2 * g][j], (&high)[4] = DT == 0 ? part[1] : acc[2 * g + 1][j], (&zsum)[4] = DT == 0 ? part[2] : zac[j];
                        float w[4] = {s[u][j][0] * s0, s[u][j][1] * s0, s[u][j][2] * s1, s[u][j][3] * s1};
                        if constexpr (SPECIAL) {                   // a key that is not seen may have any bytes for a scale (one that is, with a weight of zero too, has its NaN)
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                if ((unseen >> ((u * NT + j) * 4 + i)) & 1u) w[i] = 0.f;
                        }
#pragma unroll
                        for (int term = 0; term < PT; ++term) {
                            const uint32_t lo = pack_bf16x2(w[0], w[1]), hi = pack_bf16x2(w[2], w[3]);
                            const uint32_t p0 = transposed(lo), p1 = transposed(hi);
                            mma_bf16(low, v0 & LOW, v0 & 0x00f000f0u, v1 & LOW, v1 & 0x00f000f0u, p0, p1);
                            mma_bf16(high, BYTES ? v2 : v2 & LOW, v2 & 0x00f000f0u, BYTES ? v3 : v3 & LOW, v3 & 0x00f000f0u, p0, p1);
                            if constexpr (SPECIAL) {
                                float y[4];
#pragma unroll
                                for (int i = 0; i < 4; ++i) y[i] = careful ? finite(w[i]) : w[i];
                                mma_bf16(zsum, z0, 0u, z1, 0u, transposed(pack_bf16x2(y[0], y[1])), transposed(pack_bf16x2(y[2], y[3])));
                            } else
                                mma_bf16(zsum, z0, 0u, z1, 0u, p0, p1);
                            if (term + 1 < PT) {
                                w[0] -= bf16lo(lo); w[1] -= bf16hi(lo);
                                w[2] -= bf16lo(hi); w[3] -= bf16hi(hi);
                            }
                        }
                        if constexpr (DT == 0) {
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                acc[2 * g][j][i] += part[0][i];
                                acc[2 * g + 1][j][i] += part[1][i];
                                zac[j][i] += part[2][i];
                            }
                        }
                    }
                }
            }
        };
        if (edge || careful) values(Yes{});
        else values(No{});
        // Products add into their accumulator truncated.  Over all of a warp's keys that was 4e-3 of an output over 131072 keys (48 sequences, rows of 16 bits), what the
        // upper codes' sums are subtracted for above all; 32 products at a time leave nothing beside the output's own rounding (float16 2.06e-4 for 2.05e-4).
        // Time: 64 sequences over 8192 keys 148 -> 151 us; 153 with 16 products at a time.
        if (Smem::RUNS && (k % Smem::RUN == Smem::RUN - 1 || block + WARPS >= bend)) put();
    }
    cp_async_wait<0>();
    if constexpr (!Smem::RUNS) {
#pragma unroll
        for (int j = 0; j < NT; ++j) bad |= zac[j][0] != zac[j][0] || zac[j][1] != zac[j][1];
    }
    // The groups' sums of w s z share a product's rows: a scale that is NaN, in one group, would reach the others as 0 NaN.  Then once more, without it there.
    if (!careful && __any_sync(0xffffffffu, bad)) {
        careful = true;
        __syncwarp();
        start();
        goto again;
    }

    // ---------------- the warps' sums into one
    if constexpr (!Smem::RUNS) {
        __syncthreads();                                           // the rings are read
        put();
    } else if (fresh) {                                            // a warp without keys
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
#pragma unroll
                for (int g = 0; g < G; ++g) *sum_at(j, c, g) = make_float4(0.f, 0.f, 0.f, 0.f);
                if (gl == 0) wl[warp][8 * j + 2 * t + c] = 0.f;
            }
    }
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int c = 0; c < 2; ++c)
            if (gl == 0) wm[warp][8 * j + 2 * t + c] = m[j][c];
    __syncthreads();
    if (tid < ROWS) {
        float top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) top = fmaxf(top, wm[w][tid]);
        for (int w = 0; w < WARPS; ++w) {
            // a warp whose scores are all NaN has no maximum and a sum of NaN
            const float f = wm[w][tid] == -INFINITY ? wl[w][tid] - wl[w][tid] : exp2f(wm[w][tid] - top);
            sum += wl[w][tid] * f;
            wm[w][tid] = f;
        }
        block_m[tid] = top;
        block_l[tid] = sum;
    }
    __syncthreads();
    for (int i = tid; i < live * (D / 4); i += THREADS) {
        const int col = i / (D / 4), d = (i - col * (D / 4)) * 4;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const float f = wm[w][col];
            const float4 v = *(const float4*)(fold + ((size_t)w * ROWS + col) * DP + d);
            o.x = fmaf(f, v.x, o.x); o.y = fmaf(f, v.y, o.y); o.z = fmaf(f, v.z, o.z); o.w = fmaf(f, v.w, o.w);
        }
        *(float4*)(fold + (size_t)col * DP + d) = o;
    }
    // ---------------- the cluster's into one: block r has every `splits`-th piece
    if (p.splits > 1) cluster_sync();
    else __syncthreads();
    const uint32_t fold_at = smem_u32(fold), m_at = smem_u32(block_m), l_at = smem_u32(block_l);
    for (int i = split * THREADS + tid; i < live * (D / 4); i += p.splits * THREADS) {
        const int col = i / (D / 4), d = (i - col * (D / 4)) * 4;
        const int f = f0 + col, row = f / p.rep, tok = first + row, h = head * p.rep + f - row * p.rep;
        if (tok < 0 || tok >= p.tokens) continue;
        const float sink = p.sinks ? __ldcg(p.sinks + h) * 1.4426950408889634f : -INFINITY;
        float top = sink, sum = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        if (p.splits > 1) {
            for (int s = 0; s < p.splits; ++s) top = fmaxf(top, remote_float(remote(m_at + 4 * col, s)));
            for (int s = 0; s < p.splits; ++s) {
                const float ms = remote_float(remote(m_at + 4 * col, s)), ls = remote_float(remote(l_at + 4 * col, s));
                const float w = ms == -INFINITY ? ls - ls : exp2f(ms - top);
                const float4 v = remote_float4(remote(fold_at + (col * DP + d) * 4, s));
                sum = fmaf(w, ls, sum);
                o.x = fmaf(w, v.x, o.x); o.y = fmaf(w, v.y, o.y); o.z = fmaf(w, v.z, o.z); o.w = fmaf(w, v.w, o.w);
            }
        } else {
            top = fmaxf(top, block_m[col]);
            const float w = block_m[col] == -INFINITY ? block_l[col] - block_l[col] : exp2f(block_m[col] - top);
            const float4 v = *(const float4*)(fold + (size_t)col * DP + d);
            sum = w * block_l[col];
            o = make_float4(w * v.x, w * v.y, w * v.z, w * v.w);
        }
        if (sink != -INFINITY) sum += exp2f(sink - top);
        const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
        const size_t at = (size_t)tok * p.o_ld + (size_t)h * D + d;
        o.x *= inv; o.y *= inv; o.z *= inv; o.w *= inv;
        if constexpr (DT == 0) {
            float* dst = (float*)p.out + at;
            if (p.wide_o) *(float4*)dst = o;
            else { dst[0] = o.x; dst[1] = o.y; dst[2] = o.z; dst[3] = o.w; }
        } else {
            uint16_t* dst = (uint16_t*)p.out + at;
            const uint32_t a = kv4_pack2<DT>(o.x, o.y), b = kv4_pack2<DT>(o.z, o.w);
            if (p.wide_o) *(uint2*)dst = make_uint2(a, b);
            else { dst[0] = (uint16_t)a; dst[1] = (uint16_t)(a >> 16); dst[2] = (uint16_t)b; dst[3] = (uint16_t)(b >> 16); }
        }
    }
    if (p.splits > 1) cluster_sync();                              // nobody leaves while another reads
}

// Blocks of a cluster that share a sequence's keys.  Time in a warp's blocks of 32 keys (2.3 us with all warps at work): a block's own, and what it
// spends at its two ends, about five of them, or the SMs' share of all blocks.  Measured (us, 1 / 2 / 4 / 8 of four warps): 64 sequences over 8192 keys, 8
// heads 161 / 146 / 153 / 173; 8 with five rows over 3000 51.7 / 31.9 / 38.3 / 44.2; one over 4096 36.4 / 22.1 / 14.3 / 10.7, of eight warps 9.8.
struct Cut { int splits; float cost; };
Cut few_cut(const Kv4AttnParams& p, int rows, int warps, int resident) {
    const long long tiles = ((long long)p.max_rows * p.rep + rows - 1) / rows, items = p.seqs * tiles * p.k.kv_heads;
    const int keys = p.window > 0 && p.window < p.max_keys - p.max_rows ? p.window + p.max_rows : p.max_keys;
    const int nb = (keys + F_KEYS - 1) / F_KEYS;
    Cut best = {1, 0.f};
    for (int s = 1; s <= F_CLUSTER; s *= 2) {
        const float each = (float)(((nb + s - 1) / s + warps - 1) / warps + 5), all = (float)(items * s) * each / (float)(sm_count() * resident);
        const float cost = each > all ? each : all;
        if (s == 1 || cost < best.cost) best = {s, cost};
    }
    return best;
}

template <int G, int NT, int DT, int W>
cudaError_t launch_few(Kv4AttnParams p, cudaStream_t st) {
    using Smem = Few<G, NT, DT, W>;
    static_assert(Smem::BYTES <= 220 * 1024);
    static bool configured = false;
    if (!configured) {
        if (cudaError_t e = cudaFuncSetAttribute(kv4_few_kernel<G, NT, DT, W>, cudaFuncAttributeMaxDynamicSharedMemorySize, Smem::BYTES)) return e;
        configured = true;
    }
    p.tiles = (int)(((long long)p.max_rows * p.rep + 8 * NT - 1) / (8 * NT));
    p.splits = few_cut(p, 8 * NT, W, Smem::RESIDENT).splits;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(p.seqs * p.tiles), p.k.kv_heads, p.splits);
    cfg.blockDim = dim3(Smem::THREADS);
    cfg.dynamicSmemBytes = Smem::BYTES;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = 1;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = (unsigned)p.splits;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    count_launch();
    return cudaLaunchKernelEx(&cfg, kv4_few_kernel<G, NT, DT, W>, p);
}

// Eight rows a column block: as many blocks as the rows of a sequence's group need, up to what the accumulators' registers allow (G NT <= 8)
template <int G, int DT>
cudaError_t launch_few_rows(const Kv4AttnParams& p, cudaStream_t st) {
    const long long rows = (long long)p.max_rows * p.rep;
    if constexpr (G <= 2) {
        if (rows > 16) return launch_few<G, 4, DT, 4>(p, st);
    }
    if constexpr (G <= 4) {
        if (rows > 8) return launch_few<G, 2, DT, 4>(p, st);
        if (few_cut(p, 8, 8, Few<G, 1, DT, 8>::RESIDENT).cost < few_cut(p, 8, 4, Few<G, 1, DT, 4>::RESIDENT).cost) return launch_few<G, 1, DT, 8>(p, st);
    }
    return launch_few<G, 1, DT, 4>(p, st);
}
template <int DT>
cudaError_t launch_few_dim(const Kv4AttnParams& p, cudaStream_t st) {
    switch (p.k.dim) {
        case 64: return launch_few_rows<2, DT>(p, st);
        case 96: return launch_few_rows<3, DT>(p, st);
        case 128: return launch_few_rows<4, DT>(p, st);
        case 192: return launch_few_rows<6, DT>(p, st);
        default: return launch_few_rows<8, DT>(p, st);
    }
}

}  // namespace

}  // namespace pgk

using namespace pgk;

extern "C" int pgk_kv4_attention(const void* q, long q_ld, const void* k_cache, const void* v_cache, void* out, long o_ld, int pages, int page_size,
                                 const int32_t* page_table, int slots, int max_pages, const int32_t* seq_slots, const int32_t* context_lens,
                                 const int32_t* row_starts, int seqs, int tokens, int max_rows, int max_context, int heads, int kv_heads, int dim, float scale,
                                 int window, float softcap, const float* sinks, int dtype, void* stream) {
    const char* fn = "kv4_attention";
    if (int rc = kv4_check(fn, k_cache, pages, page_size, page_table, slots, max_pages, kv_heads, dim)) return rc;
    if (int rc = kv4_check(fn, v_cache, pages, page_size, page_table, slots, max_pages, kv_heads, dim)) return rc;
    PGK_REQUIRE(dtype >= 0 && dtype <= 2, "kv4_attention failed: unknown type %d", dtype);
    PGK_REQUIRE(heads > 0 && heads % kv_heads == 0 && kv_heads <= 65535 && q_ld >= (long)heads * dim && o_ld >= (long)heads * dim,
                "kv4_attention failed: %d query heads over %d, rows of %ld and %ld", heads, kv_heads, q_ld, o_ld);
    PGK_REQUIRE(seqs >= 0 && tokens >= 0 && max_rows > 0 && max_context >= 0 && (row_starts || (tokens >= seqs && max_rows == 1)) &&
                    (long long)seqs * max_rows * (heads / kv_heads) <= 0x7fffffffll,
                "kv4_attention failed: %d sequences of up to %d rows in %d, %d keys", seqs, max_rows, tokens, max_context);
    PGK_REQUIRE(window >= 0 && softcap >= 0.f && softcap < 1e38f && scale >= 0.f && scale < 1e38f, "kv4_attention failed: window %d, cap %g, scale %g", window, softcap, scale);
    if (seqs == 0 || tokens == 0) return 0;
    PGK_REQUIRE(q && out && seq_slots && context_lens, "kv4_attention failed: no queries, output, slots or contexts");
    Kv4AttnParams p = {};
    p.q = q; p.out = out; p.q_ld = q_ld; p.o_ld = o_ld;
    p.k = {(unsigned char*)k_cache, page_table, pages, page_size, slots, max_pages, kv_heads, dim};
    p.v_data = (const unsigned char*)v_cache;
    p.seq_slots = seq_slots; p.contexts = context_lens; p.starts = row_starts;
    p.seqs = seqs; p.tokens = tokens; p.heads = heads; p.rep = heads / kv_heads;
    p.max_rows = max_rows < tokens ? max_rows : tokens;
    p.max_keys = max_context < max_pages * page_size ? max_context : max_pages * page_size;
    p.scale_log2 = (scale > 0.f ? scale : 1.f / sqrtf((float)dim)) * 1.4426950408889634f;
    p.cap_log2 = softcap > 0.f ? fmaxf(softcap, 1e-30f) * 1.4426950408889634f : 0.f;          // (scores within 1e-30 of zero, and a weight of 1, in any case)
    p.window = window; p.sinks = sinks;
    p.head_bytes = (long long)page_size * kv4_row_bytes(dim);
    p.page_bytes = p.head_bytes * kv_heads;
    const uint32_t sub = (uint32_t)page_size / 16;                 // n < 2^27 and sub <= 2^8: exact with a multiplier of 32 bits
    if (sub > 1) {
        uint32_t log = 0;
        while ((1u << log) < sub) ++log;
        p.page_shift = log > 5 ? log - 5 : 0;
        p.page_mul = (uint32_t)((1ull << (32 + p.page_shift)) / sub) + 1;
    }
    const int size = dtype == 0 ? 4 : 2;
    p.wide_q = (uintptr_t)q % 16 == 0 && q_ld * size % 16 == 0;
    p.wide_o = (uintptr_t)out % 16 == 0 && o_ld * size % 16 == 0;
    const cudaStream_t st = (cudaStream_t)stream;
    if (kv4_prompt_serves(p, dtype)) return kv4_prompt(p, dtype, st);
    PGK_CUDA(dtype == 0 ? launch_few_dim<0>(p, st) : (dtype == 1 ? launch_few_dim<1>(p, st) : launch_few_dim<2>(p, st)));
    return 0;
}
