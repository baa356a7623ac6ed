// kv4_prompt.cu -- attention of many rows a sequence (prompts, portions of them) over the four-bit paged cache on tcgen05; the mathematics of
// kv4_attention.cu, for rows of 16 bits and heads of 64, 96 and 128 elements.
//
// A block has 128 rows (a token's query heads of one key head beside each other) and walks over tiles of 128 keys:
//   * eight warps expand a tile of K, then of V, to bfloat16 in shared memory -- s (c - z) is a bfloat16 number, nothing is rounded: a nibble under
//     the exponent of 128 is 128 + c, one subtraction and one product for two elements.  Their loads run one tile ahead, in registers;
//   * one thread issues S = Q K^T (queries in tensor memory, float16 ones as two bfloat16 terms) and O += P V, the scores of tile i + 1 before the
//     weights of tile i are waited for; three tiles of K and V are in shared memory;
//   * eight warps, a lane a row and two warps a row, turn scores into weights; a weight is rounded to bfloat16 once (2^-9 of it, independent from
//     key to key, beside the output's own 2^-9), for float16 rows to two such terms (2^-17), their sum is float32 of the unrounded ones.  A row's
//     reference moves when its maximum has grown by 2^8.  Products add into tensor memory truncated: over 131072 keys an output is small by 1e-4 of itself.
// The eight elements of a word of codes keep the order (0, 4, 1, 5, 2, 6, 3, 7) that its nibbles fall into: queries are brought into it, outputs back.
// What bounds it: the chain of a row's warps.  Of 128 x 128 x 128 the products take 512 cycles and the exponentials 1024 of the special unit; measured are 1890 a
// tile (scores ready, maxima 180 cycles, exchange between a row's warps 240, weights 1160, arrival) where tiles were made before, 2750 where the block
// makes them (K 800 to 1200, V 800, what lies between 400 each: two warps a scheduler, latency), and 13600 at a block's two ends.  Measured: 512 rows over 16384
// keys, 32 / 4 heads of 128, 147 to 154 us (0.9 PFLOP/s), 2000 rows over themselves, 32 / 8 heads, 73 to 78 us, 8 sequences of 5 rows over 3000 keys 28 us;
// float16 rows, twice the products and a second term a weight, 200, 97 and 36.
// Few blocks share a sequence's keys within a cluster and fold through distributed shared memory.
//
// A value of NaN counts as zero in the products (0 NaN would reach rows that do not see it); where any was met, rows look for the ones they see
// in the end.
#include "kv4_attention.cuh"
#include "tc_common.cuh"
#include "../../include/pgk_b200.h"

namespace pgk {

namespace {

constexpr int P_ROWS = 128, P_KEYS = 128, P_SOFT = 8, P_EXPAND = 8, P_THREADS = (P_SOFT + 1 + P_EXPAND) * 32, P_STAGES = 3, P_CLUSTER = 8;
constexpr uint32_t P_CHUNK = P_KEYS * 128;                         // 64 elements of 128 keys
constexpr uint32_t P_O = 0, P_Q = 128, P_S = 256;                  // TMEM columns: outputs, queries (two terms of 64), two tiles of scores
constexpr float P_LAZY = 8.f;
// Rows of a sequence and head from which its tiles are made once.  Measured (us, made by each block / once, 8 heads of 128 elements): one sequence over 16384
// keys, 512 rows 58.6 / 62.4, 768 140 / 130, 1024 104 / 95; 8 over 3000, 512 82.9 / 84.2, 768 116 / 111; 32 over 2000, 512 219 / 228, 768 299 / 294.
constexpr int P_IMAGES_FROM = 768;
constexpr long long P_IMAGES_MOST = 1ll << 30;

// Tiles as they lie in shared memory, made ahead of the products: [sequence][head][tile][K, V], and per tile whether a value is NaN.  Tile 0 is the one
// that holds the first key of the sequence's first row.
struct Images {
    unsigned char* data;
    int32_t* nans;
    int tiles;
};
__device__ __forceinline__ int first_tile(const Kv4AttnParams& p, int ctx, int n_rows) { return kv4_first_key(p, ctx - n_rows) / P_KEYS; }

template <int G> struct Prompt {
    static constexpr int D = 32 * G, DN = G == 2 ? 64 : 128;       // 96 elements: the products go on to 128 over zeros
    static constexpr uint32_t TILE = (DN / 64) * P_CHUNK;
    static constexpr int RING = 2 * P_STAGES * TILE, FOLD = P_ROWS * (D + 4) * 4, BYTES = (RING > FOLD ? RING : FOLD) + 1024;
};

__device__ __forceinline__ bool all_wait(int* err, uint64_t* bar, uint32_t parity) {
    const bool ok = bar_wait(err, smem_u32(bar), parity);
    return __all_sync(0xffffffffu, ok);
}
__device__ __forceinline__ uint32_t bf2_add(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("add.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint32_t bf2_mul(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

// Sixteen keys of a warp: this lane's bytes of two of them (keys kq and kq + 8; two quads of an access are keys 4 apart, so that stores meet all banks)
template <int G> struct Raw {
    uint32_t c[2][G], m[2][(G + 1) / 2];
    __device__ __forceinline__ void load(const unsigned char* codes, const unsigned char* words, const bool (&there)[2]) {
#pragma unroll
        for (int it = 0; it < 2; ++it) {
#pragma unroll
            for (int g = 0; g < G; ++g) c[it][g] = 0;
#pragma unroll
            for (int g = 0; g < (G + 1) / 2; ++g) m[it][g] = 0;
            if (there[it]) {
                const unsigned char* const x = codes + it * 128 * G;
                const unsigned char* const y = words + it * 16 * G;
                if constexpr (G == 4) {
                    const uint4 v = ld_act16(x);
                    c[it][0] = v.x; c[it][1] = v.y; c[it][2] = v.z; c[it][3] = v.w;
                    const uint2 u = __ldcg((const uint2*)y);
                    m[it][0] = u.x; m[it][1] = u.y;
                } else if constexpr (G == 2) {
                    const uint2 v = __ldcg((const uint2*)x);
                    c[it][0] = v.x; c[it][1] = v.y;
                    m[it][0] = __ldcg((const uint32_t*)y);
                } else {
#pragma unroll
                    for (int g = 0; g < G; ++g) {
                        c[it][g] = __ldcg((const uint32_t*)x + g);
                        m[it][g / 2] |= (uint32_t)ld_act2((const uint16_t*)y + g) << (16 * (g & 1));
                    }
                }
            }
        }
    }
    // put(it, g, four words): elements 32 g + 8 t ... + 7 of the lane's key, in the order of its nibbles.  Values that are NaN become zeros: true
    template <typename Put> __device__ __forceinline__ bool expand(bool values, Put put) const {
        bool nan = false;
#pragma unroll
        for (int it = 0; it < 2; ++it)
#pragma unroll
            for (int g = 0; g < G; ++g) {
                uint32_t w = __byte_perm(m[it][g / 2], 0, g & 1 ? 0x3232 : 0x1010);
                if (values && (w & 0x7f80u) == 0x7f80u) { nan = true; w = 0; }
                const uint32_t zero = (w & 0x000f000fu) | 0xc300c300u, scale = w & 0x7ff07ff0u;        // -(128 + z), s
                const uint32_t x = c[it][g];
                uint32_t y[4] = {x, x >> 4, x >> 8, x >> 12};
#pragma unroll
                for (int e = 0; e < 4; ++e) y[e] = bf2_mul(bf2_add((y[e] & 0x000f000fu) | 0x43004300u, zero), scale);
                put(it, g, make_uint4(y[0], y[1], y[2], y[3]));
            }
        return nan;
    }
};
__device__ __forceinline__ int lane_key(int lane) { return (lane >> 3) + 4 * ((lane >> 2) & 1); }
// where a lane's eight elements of group g of key `key` (16 w + kq, 8 on with it = 1) lie in a tile
template <int G>
__device__ __forceinline__ uint32_t tile_place(int key, int t, int it, int g) {
    return (uint32_t)key * 128u + ((uint32_t)(((4 * (g & 1) + t) ^ (key & 7)) * 16)) + (uint32_t)(g >> 1) * P_CHUNK + (uint32_t)it * 1024u;
}

// tiles of K and V, a block each
template <int G>
__global__ void __launch_bounds__(P_EXPAND * 32) kv4_images_kernel(const __grid_constant__ Kv4AttnParams p, const __grid_constant__ Images im) {
    using C = Prompt<G>;
    griddep_wait();
    griddep_launch();
    const int tile = blockIdx.x, head = blockIdx.y, seq = blockIdx.z, tid = threadIdx.x, lane = tid & 31, w = tid >> 5, t = lane & 3;
    const int slot = __ldcg(p.seq_slots + seq), ctx = __ldcg(p.contexts + seq);
    const int n_rows = p.starts ? __ldcg(p.starts + seq + 1) - __ldcg(p.starts + seq) : 1;
    const int base = first_tile(p, ctx, n_rows), end = min(ctx, p.max_keys), j = (base + tile) * P_KEYS + 16 * w + lane_key(lane);
    if (base + tile >= (end + P_KEYS - 1) / P_KEYS || (unsigned)slot >= (unsigned)p.k.slots) return;
    const uint32_t run = (uint32_t)((base + tile) * P_KEYS + 16 * w) >> 4, in_slot = kv4_page_of(p, run);
    const int page = (int)(run << 4) < end ? __ldcg(p.k.table + (size_t)slot * p.k.max_pages + in_slot) : -1, in_page = j - (int)(in_slot * (uint32_t)p.k.page_size);
    const bool good = (unsigned)page < (unsigned)p.k.pages, there[2] = {good && j < end, good && j + 8 < end};
    const long long at = page * p.page_bytes + (long long)head * p.head_bytes;
    Raw<G> k, v;
    k.load(p.k.data + at + in_page * (16 * G) + t * 4 * G, p.k.data + at + p.k.page_size * (16 * G) + in_page * (2 * G), there);
    v.load(p.v_data + at + in_page * (16 * G) + t * 4 * G, p.v_data + at + p.k.page_size * (16 * G) + in_page * (2 * G), there);
    const size_t n = ((size_t)seq * p.k.kv_heads + head) * im.tiles + tile;
    unsigned char* const to = im.data + n * (2 * C::TILE);
    const int key = 16 * w + lane_key(lane);
    k.expand(false, [&](int it, int g, uint4 x) { *(uint4*)(to + tile_place<G>(key, t, it, g)) = x; });
    const bool nan = v.expand(true, [&](int it, int g, uint4 x) { *(uint4*)(to + C::TILE + tile_place<G>(key, t, it, g)) = x; });
    if constexpr (G == 3) {                        // elements 96 ... 127 of V
        for (int i = tid; i < P_KEYS * 4; i += P_EXPAND * 32)
            *(uint4*)(to + C::TILE + P_CHUNK + (i / 4) * 128 + (((4 + i % 4) ^ (i / 4 & 7)) * 16)) = make_uint4(0, 0, 0, 0);
    }
    const int any = __syncthreads_or(nan);
    if (tid == 0) im.nans[n] = any;
}

// A block's rows -- ROWS of one sequence's, a token's query heads of one key head beside each other -- and the tiles that they see between them.  Blocks
// come with the longest rows first.
template <int ROWS> struct Block {
    int seq, head, split, slot, ctx, first, n_rows, f0, live, pos0, pos1, begin, end, tbeg, n;
    const int32_t* table;
    __device__ __forceinline__ explicit Block(const Kv4AttnParams& p) {
        seq = blockIdx.x % p.seqs;
        f0 = (p.tiles - 1 - (int)(blockIdx.x / p.seqs)) * ROWS;
        head = blockIdx.y;
        split = blockIdx.z;
        slot = __ldcg(p.seq_slots + seq);
        ctx = __ldcg(p.contexts + seq);
        first = p.starts ? __ldcg(p.starts + seq) : seq;
        n_rows = p.starts ? __ldcg(p.starts + seq + 1) - first : 1;
        const int rows = min(min(n_rows, p.max_rows), 0x7fffffff / p.rep) * p.rep;
        const bool work = f0 < rows && (unsigned)slot < (unsigned)p.k.slots;               // the same in all of the cluster
        live = work ? min(ROWS, rows - f0) : 0;
        pos0 = ctx - n_rows + f0 / p.rep;
        pos1 = ctx - n_rows + (f0 + max(live, 1) - 1) / p.rep;
        begin = kv4_first_key(p, pos0);
        end = work ? min(min(pos1 + 1, ctx), p.max_keys) : 0;
        const int t0 = begin / P_KEYS, nt = max(0, (end + P_KEYS - 1) / P_KEYS - t0), per = (nt + p.splits - 1) / p.splits;
        tbeg = t0 + split * per;
        n = max(0, min(nt, (split + 1) * per) - split * per);
        table = p.k.table + (work ? (size_t)slot * p.k.max_pages : 0);
    }
    // whether a page of the keys does not exist, by `count` threads of which this is number i
    __device__ __forceinline__ bool gone(const Kv4AttnParams& p, int i, int count) const {
        bool g = false;
        const int last = min(end, (tbeg + n) * P_KEYS);
        for (int j = tbeg * P_KEYS + 16 * i; j < last; j += 16 * count) g |= (unsigned)__ldcg(table + kv4_page_of(p, (uint32_t)j >> 4)) >= (unsigned)p.k.pages;
        return g;
    }
};
// Row r of a block: whose it is, and what it sees: keys in (under, limit]
struct Row {
    int tok, h, pos, limit, under;
    bool live;
    template <int ROWS> __device__ __forceinline__ Row(const Kv4AttnParams& p, const Block<ROWS>& b, int r) {
        const int f = b.f0 + r, i = f / p.rep;
        tok = b.first + i;
        h = b.head * p.rep + f - i * p.rep;
        pos = b.ctx - b.n_rows + i;
        live = r < b.live && tok >= 0 && tok < p.tokens;
        limit = live ? min(pos, b.end - 1) : -1;
        under = kv4_first_key(p, pos) - 1;
    }
};
// eight query elements in the order of a word's nibbles, as one or two bfloat16 terms
template <int DT>
__device__ __forceinline__ void query8(const Kv4AttnParams& p, const Row& r, int at, uint32_t* a, uint32_t* b) {
    uint32_t w[4] = {};
    if (r.live) {
        const uint16_t* src = (const uint16_t*)p.q + (size_t)r.tok * p.q_ld + at;
        if (p.wide_q) {
            const uint4 v = ld_act16(src);
            w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = (uint32_t)ld_act2(src + 2 * e) | (uint32_t)ld_act2(src + 2 * e + 1) << 16;
        }
    }
    const uint32_t v[4] = {__byte_perm(w[0], w[2], 0x5410), __byte_perm(w[0], w[2], 0x7632), __byte_perm(w[1], w[3], 0x5410), __byte_perm(w[1], w[3], 0x7632)};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if constexpr (DT == 1) {
            const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&v[e]));
            a[e] = pack_bf16x2(x.x, x.y);
            b[e] = pack_bf16x2(x.x - bf16lo(a[e]), x.y - bf16hi(a[e]));
        } else
            a[e] = v[e];
    }
}
// N scores of a row, from TMEM column `at`, key j0: capped (or, if they are huge, with their factor), and -infinity where the row does not see; `off`: runs of 16 keys without a page
template <int N>
__device__ __forceinline__ void row_scores(const Kv4AttnParams& p, uint32_t at, int j0, bool edge, bool huge, const Row& r, uint32_t off, float (&s)[N]) {
#pragma unroll
    for (int c = 0; c < N; c += 16) tmem_ld16_async(at + (uint32_t)c, *(float (*)[16])(s + c));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int c = 0; c < N; c += 16) tmem_pass(*(float (*)[16])(s + c));
    if (p.cap_log2 > 0.f || huge) {
        if (p.cap_log2 > 0.f) {
            const float in = kv4_cap_in(p.scale_log2, p.cap_log2);
#pragma unroll
            for (int e = 0; e < N; ++e) s[e] = p.cap_log2 * kv4_tanh(s[e] * in);
        } else {
#pragma unroll
            for (int e = 0; e < N; ++e) s[e] *= p.scale_log2;
        }
    }
    if (edge) {
        const int hi = r.limit - j0, lo = r.under - j0;
#pragma unroll
        for (int e = 0; e < N; ++e)
            if (e > hi || e <= lo || ((off >> (e / 16)) & 1u)) s[e] = -INFINITY;
    }
}
// of `runs` runs of 16 keys from j0 on, the ones without a page
template <int ROWS>
__device__ __forceinline__ uint32_t runs_gone(const Kv4AttnParams& p, const Block<ROWS>& b, int j0, int runs) {
    uint32_t off = 0;
    for (int u = 0; u < runs; ++u)
        if (j0 + 16 * u < b.end && (unsigned)__ldcg(b.table + kv4_page_of(p, (uint32_t)(j0 + 16 * u) >> 4)) >= (unsigned)p.k.pages) off |= 1u << u;
    return off;
}
// pairs of float32 in a register pair: one instruction for two products or sums
__device__ __forceinline__ uint64_t pair(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpair(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
// 32 weights 2^(s fac + neg) to TMEM column `to`, as one bfloat16 term or two (the second 32 columns on); their sum is of the unrounded ones
template <int TERMS>
__device__ __forceinline__ void weights32(const float* s, float fac, float neg, uint32_t to, uint64_t& l) {
    uint32_t y[16], z[16];
    const uint64_t fac2 = pair(fac, fac), neg2 = pair(neg, neg);
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        const uint64_t x = fma2(pair(s[2 * e], s[2 * e + 1]), fac2, neg2);
        float a, b;
        unpair(x, a, b);
        a = ex2(a);
        b = ex2(b);
        l = add2(l, pair(a, b));
        y[e] = pack_bf16x2(a, b);
        if constexpr (TERMS == 2) z[e] = pack_bf16x2(a - bf16lo(y[e]), b - bf16hi(y[e]));
    }
    __syncwarp();
    tmem_st16u(to, y);
    if constexpr (TERMS == 2) tmem_st16u(to + 32u, z);
}
__device__ __forceinline__ void rescale(uint32_t at, int columns, float f) {
#pragma unroll 1
    for (int c = 0; c < columns; c += 16) {
        float o[16];
        tmem_ld16(at + (uint32_t)c, o);
#pragma unroll
        for (int e = 0; e < 16; ++e) o[e] *= f;
        tmem_st16(at + (uint32_t)c, o);
    }
}
// what a row's outputs are multiplied by, whose weights have the reference `top` and the sum `sum`: the sink joins
__device__ __forceinline__ float row_factor(const Kv4AttnParams& p, int h, float top, float sum) {
    const float sink = p.sinks ? __ldcg(p.sinks + h) * 1.4426950408889634f : -INFINITY, all = fmaxf(top, sink);
    const float w = top == -INFINITY ? 1.f : exp2f(top - all);             // (no maximum: nothing seen, or all NaN, which the sum knows)
    sum *= w;
    if (sink != -INFINITY) sum += exp2f(sink - all);
    return sum > 0.f || sum != sum ? w / sum : 0.f;
}
// groups of which the row sees a value that is NaN, in the block's tiles
template <int G, int ROWS>
__device__ __forceinline__ uint32_t lost_groups(const Kv4AttnParams& p, const Block<ROWS>& b, const Row& r) {
    uint32_t lost = 0;
    const int last = min(r.limit, (b.tbeg + b.n) * P_KEYS - 1);
    for (int j = max(max(b.begin, b.tbeg * P_KEYS), r.under + 1); j <= last; ++j) {
        const uint32_t in_slot = kv4_page_of(p, (uint32_t)j >> 4);
        const int page = __ldcg(b.table + in_slot);
        if ((unsigned)page >= (unsigned)p.k.pages) continue;
        const uint16_t* words = (const uint16_t*)(p.v_data + page * p.page_bytes + (size_t)b.head * p.head_bytes + (size_t)p.k.page_size * (16 * G)) +
                                (size_t)(j - (int)(in_slot * (uint32_t)p.k.page_size)) * G;
        for (int g = 0; g < G; ++g)
            if ((ld_act2(words + g) & 0x7f80u) == 0x7f80u) lost |= 1u << g;
    }
    return lost;
}
// outputs [from, to) of a row, from TMEM column `at`: to memory, or to the fold
template <int DT>
__device__ __forceinline__ void outputs(const Kv4AttnParams& p, const Row& r, int dim, int from, int to, uint32_t at, bool any, uint32_t lost, float factor, float* fold) {
#pragma unroll 1
    for (int c = from; c < to; c += 16) {
        float o[16], x[16];
        __syncwarp();
        if (any) tmem_ld16(at + (uint32_t)c, o);
        else {
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = 0.f;
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] = o[(e & 8) + (e & 4 ? 2 * (e & 3) + 1 : 2 * (e & 3))];
        if ((lost >> (c / 32)) & 1u) {
#pragma unroll
            for (int e = 0; e < 16; ++e) x[e] = NAN;
        }
        if (fold) {
#pragma unroll
            for (int e = 0; e < 16; e += 4) *(float4*)(fold + c + e) = make_float4(x[e], x[e + 1], x[e + 2], x[e + 3]);
        } else if (r.live) {
            uint16_t* dst = (uint16_t*)p.out + (size_t)r.tok * p.o_ld + (size_t)r.h * dim + c;
            uint32_t y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = kv4_pack2<DT>(x[2 * e] * factor, x[2 * e + 1] * factor);
            if (p.wide_o) {
                *(uint4*)dst = make_uint4(y[0], y[1], y[2], y[3]);
                *(uint4*)(dst + 8) = make_uint4(y[4], y[5], y[6], y[7]);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) { dst[2 * e] = (uint16_t)y[e]; dst[2 * e + 1] = (uint16_t)(y[e] >> 16); }
            }
        }
    }
    __syncwarp();
}
// the cluster's blocks into one, rows of D + 4 floats each: block r has every `splits`-th piece
template <int D, int DT, int ROWS>
__device__ __forceinline__ void fold_cluster(const Kv4AttnParams& p, const Block<ROWS>& b, const float* fold, const float* row_m, const float* row_l) {
    cluster_sync();
    const uint32_t fold_at = smem_u32(fold), m_at = smem_u32(row_m), l_at = smem_u32(row_l);
    for (int i = b.split * (int)blockDim.x + (int)threadIdx.x; i < b.live * (D / 4); i += p.splits * (int)blockDim.x) {
        const int r = i / (D / 4), d = (i - r * (D / 4)) * 4;
        const Row row(p, b, r);
        if (!row.live) continue;
        float top = -INFINITY, sum = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int s = 0; s < p.splits; ++s) top = fmaxf(top, remote_float(remote(m_at + 4 * r, s)));
        for (int s = 0; s < p.splits; ++s) {
            const float ms = remote_float(remote(m_at + 4 * r, s)), ls = remote_float(remote(l_at + 4 * r, s));
            const float w = ms == -INFINITY ? ls - ls : exp2f(ms - top);
            const float4 v = remote_float4(remote(fold_at + (r * (D + 4) + d) * 4, s));
            sum = fmaf(w, ls, sum);
            o.x = fmaf(w, v.x, o.x); o.y = fmaf(w, v.y, o.y); o.z = fmaf(w, v.z, o.z); o.w = fmaf(w, v.w, o.w);
        }
        const float factor = row_factor(p, row.h, top, sum);
        const uint32_t x = kv4_pack2<DT>(o.x * factor, o.y * factor), y = kv4_pack2<DT>(o.z * factor, o.w * factor);
        uint16_t* dst = (uint16_t*)p.out + (size_t)row.tok * p.o_ld + (size_t)row.h * D + d;
        if (p.wide_o) *(uint2*)dst = make_uint2(x, y);
        else { dst[0] = (uint16_t)x; dst[1] = (uint16_t)(x >> 16); dst[2] = (uint16_t)y; dst[3] = (uint16_t)(y >> 16); }
    }
    cluster_sync();                                // nobody leaves while another reads
}

// IMAGES: one warp copies tiles that kv4_images_kernel has made; otherwise P_EXPAND warps make them
template <int G, int DT, bool IMAGES>
__global__ void __launch_bounds__(IMAGES ? (P_SOFT + 2) * 32 : P_THREADS, 1) kv4_prompt_kernel(const __grid_constant__ Kv4AttnParams p, const __grid_constant__ Images im, int* err) {
    using C = Prompt<G>;
    constexpr int THREADS = IMAGES ? (P_SOFT + 2) * 32 : P_THREADS, FILLS = IMAGES ? 1 : P_EXPAND;
    constexpr int D = C::D, DN = C::DN, QT = DT == 1 ? 2 : 1;
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ __align__(8) uint64_t full[P_STAGES], empty[P_STAGES], sfull[2], pready[2], pvdone;
    __shared__ uint32_t tmem_base_s;
    __shared__ float wmax[2][2][P_ROWS], row_m[P_ROWS], row_l[P_ROWS];
    __shared__ int missing, nans;
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    const uint32_t ks = (smem_u32(smem) + 1023u) & ~1023u, vs = ks + P_STAGES * C::TILE;

    if (warp == P_SOFT) tmem_alloc(&tmem_base_s, 512);
    if (tid == 0) {
        for (int s = 0; s < P_STAGES; ++s) {
            mbar_init(&full[s], FILLS); mbar_init(&empty[s], 1);
        }
        mbar_init(&sfull[0], 1); mbar_init(&sfull[1], 1);
        mbar_init(&pready[0], P_SOFT); mbar_init(&pready[1], P_SOFT); mbar_init(&pvdone, 1);
        mbar_fence_init();
        missing = nans = 0;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_base_s;
    griddep_wait();
    griddep_launch();

    const Block<P_ROWS> b(p);
    const int n = b.n, begin = b.begin, end = b.end, tbeg = b.tbeg, head = b.head;
    const size_t image = ((size_t)b.seq * p.k.kv_heads + head) * im.tiles + (tbeg - first_tile(p, b.ctx, b.n_rows));        // the block's first tile
    const int32_t* const table = b.table;
    const int quad = warp & 3, half = (warp >> 2) & 1, row = quad * 32 + lane;
    const Row r(p, b, warp < P_SOFT ? row : P_ROWS);

    if (warp < 4) {                                // queries to tensor memory
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
            uint32_t x[16], y[16];
#pragma unroll
            for (int i = 0; i < 4; ++i) query8<DT>(p, r, r.h * D + c + 8 * i, x + 4 * i, y + 4 * i);
            __syncwarp();
            const uint32_t to = tmem + ((uint32_t)(quad * 32) << 16) + P_Q + (uint32_t)c / 2u;
            tmem_st16u(to, x);
            if constexpr (QT == 2) tmem_st16u(to + 64u, y);
        }
        tmem_st_wait();
    } else {
        if (b.gone(p, tid - 128, THREADS - 128)) missing = 1;
        if constexpr (IMAGES) {
            for (int i = tid - 128; i < n; i += THREADS - 128)
                if (__ldcg(im.nans + image + i)) nans = 1;
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();

    if (warp == P_SOFT) {
        // ---------------- MMAs, from one thread: votes and elections of a whole warp between them took 250 cycles a wait
        if (elect_one()) {
            constexpr uint32_t id_s = umma_idesc_bf16(P_KEYS), id_o = umma_idesc_bf16(DN) | (1u << 16);   // values: the elements are contiguous
            const uint64_t kd = desc_sw128(ks), vd = desc_mn_sw128(vs, P_CHUNK);
            bool ok = true;
            auto scores = [&](int i) {             // where the weights of tile i - 2 were
                const int s = i % P_STAGES;
                ok = ok && bar_wait(err, smem_u32(&full[s]), (uint32_t)(i / P_STAGES) & 1u);
                if (!ok) return;
                tc_fence_after();
                const uint64_t d = kd + (uint64_t)(s * (C::TILE / 16));
                const uint32_t to = tmem + P_S + (uint32_t)(i & 1) * 128u;
#pragma unroll
                for (int term = QT - 1; term >= 0; --term)
#pragma unroll
                    for (int k = 0; k < D / 16; ++k)
                        umma_bf16_ta(to, tmem + P_Q + (uint32_t)term * 64u + (uint32_t)k * 8u, d + (uint64_t)((k >> 2) * (P_CHUNK / 16) + (k & 3) * 2), id_s, k || term < QT - 1 ? 1u : 0u);
                umma_commit(&sfull[i & 1]);
            };
            if (n > 0) scores(0);
            int made = 0;
            for (int i = 0; ok && i < n; ++i) {
                const int s = i % P_STAGES;
                if (i > 0) ok = bar_wait(err, smem_u32(&pvdone), (uint32_t)((i - 1) & 1));
                if (ok && i + 1 < n) scores(i + 1);
                ok = ok && bar_wait(err, smem_u32(&pready[i & 1]), (uint32_t)(i >> 1) & 1u);
                if (!ok) break;
                tc_fence_after();
                const uint64_t d = vd + (uint64_t)(s * (C::TILE / 16));
                const uint32_t at = tmem + P_S + (uint32_t)(i & 1) * 128u;
#pragma unroll
                for (int term = 0; term < QT; ++term)
#pragma unroll
                    for (int k = 0; k < P_KEYS / 16; ++k)          // 16 keys: 2048 bytes of V
                        umma_bf16_ta(tmem + P_O, at + (uint32_t)term * 32u + (uint32_t)(k >> 2) * 64u + (uint32_t)(k & 3) * 8u, d + (uint64_t)(k * 128), id_o, (i | k | term) ? 1u : 0u);
                umma_commit(&pvdone);
                umma_commit(&empty[s]);
                made = i + 1;
            }
            if (made) bar_wait(err, smem_u32(&pvdone), (uint32_t)((made - 1) & 1));           // here, where each was waited for: others might take the last but two for it
        }
        __syncwarp();
    } else if (warp > P_SOFT) {
        if constexpr (IMAGES) {
            // ---------------- tiles of K and V, copied
            if (elect_one()) {
                bool ok = true;
                int made = 0;
                for (; made < n; ++made) {
                    const int s = made % P_STAGES;
                    ok = ok && bar_wait(err, smem_u32(&empty[s]), (((uint32_t)made / P_STAGES) & 1u) ^ 1u);
                    if (!ok) break;
                    const unsigned char* const from = im.data + (image + made) * (2 * C::TILE);
                    mbar_arrive_expect_tx(&full[s], 2 * C::TILE);
                    bulk_copy_g2s(smem + (ks - smem_u32(smem)) + s * C::TILE, from, C::TILE, &full[s]);
                    bulk_copy_g2s(smem + (vs - smem_u32(smem)) + s * C::TILE, from + C::TILE, C::TILE, &full[s]);
                }
                for (int j = max(0, made - P_STAGES); j < made; ++j)        // whoever gave up: do not leave with copies in flight
                    bar_wait(err, smem_u32(&full[j % P_STAGES]), (uint32_t)(j / P_STAGES) & 1u);
            }
            __syncwarp();
        } else {
            // ---------------- tiles of K and V, expanded
            const int w = warp - P_SOFT - 1, t = lane & 3, key = 16 * w + lane_key(lane);
            const unsigned char* const khead = p.k.data + (size_t)head * p.head_bytes;
            const unsigned char* const vhead = p.v_data + (size_t)head * p.head_bytes;
            const int code_bytes = p.k.page_size * 16 * G;
            if constexpr (G == 3) {                    // elements 96 ... 127 of V
                for (int i = tid - (P_SOFT + 1) * 32; i < P_STAGES * P_KEYS * 4; i += P_EXPAND * 32) {
                    const int s = i / (P_KEYS * 4), k = i / 4 % P_KEYS;
                    asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" :: "r"(vs + s * C::TILE + P_CHUNK + k * 128 + (((4 + i % 4) ^ (k & 7)) * 16)), "r"(0) : "memory");
                }
            }
            Raw<G> kr, vr;
            int page, ahead;                           // of the warp's 16 keys; of the tile after
            long long codes = 0, words = 0;            // this lane's places in the head's pages
            bool there[2] = {false, false}, nan = false;
            auto page_at = [&](int i) {
                const int j = (tbeg + i) * P_KEYS + 16 * w;
                return i < n && j < end ? __ldcg(table + kv4_page_of(p, (uint32_t)j >> 4)) : -1;
            };
            auto place = [&](int i) {
                const int j = (tbeg + i) * P_KEYS + key;
                const int in_page = j - (int)(kv4_page_of(p, (uint32_t)j >> 4) * (uint32_t)p.k.page_size);
                const bool good = (unsigned)page < (unsigned)p.k.pages;
                there[0] = good && j >= begin && j < end;
                there[1] = good && j + 8 >= begin && j + 8 < end;
                codes = page * p.page_bytes + in_page * (16 * G) + t * 4 * G;
                words = page * p.page_bytes + code_bytes + in_page * (2 * G);
            };
            const uint32_t to_even = tile_place<G>(key, t, 0, 0), to_odd = to_even ^ 64u;                 // groups of a chunk's first and second half
            auto store = [&](uint32_t tile) {
                return [=](int it, int g, uint4 x) {
                    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};"
                                 :: "r"(tile + (g & 1 ? to_odd : to_even) + (uint32_t)(g >> 1) * P_CHUNK + (uint32_t)it * 1024u), "r"(x.x), "r"(x.y), "r"(x.z), "r"(x.w) : "memory");
                };
            };
            page = page_at(0);
            place(0);
            kr.load(khead + codes, khead + words, there);
            vr.load(vhead + codes, vhead + words, there);
            ahead = page_at(1);
            bool ok = true;
            for (int i = 0; i < n; ++i) {
                const int s = i % P_STAGES;
                const uint32_t free = (((uint32_t)i / P_STAGES) & 1u) ^ 1u;
                ok = ok && all_wait(err, &empty[s], free);
                if (!ok) break;
                kr.expand(false, store(ks + s * C::TILE));
                page = ahead;
                place(i + 1);
                if (i + 1 < n) kr.load(khead + codes, khead + words, there);
                ahead = page_at(i + 2);
                nan |= vr.expand(true, store(vs + s * C::TILE));
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(&full[s]);
                if (i + 1 < n) vr.load(vhead + codes, vhead + words, there);
            }
            if (nan) nans = 1;
        }
    } else {
        // ---------------- weights
        const uint32_t lanes = tmem + ((uint32_t)(quad * 32) << 16);
        const int clean_lo = kv4_first_key(p, b.pos1) - 1, clean_hi = missing ? -1 : min(b.pos0, end - 1);
        float m = -INFINITY, neg = 0.f, l = 0.f, fac = p.cap_log2 > 0.f ? 1.f : p.scale_log2;
        bool ok = true, huge = false;
        for (int i = 0; i < n; ++i) {
            const uint32_t at = lanes + P_S + (uint32_t)(i & 1) * 128u;
            const int j0 = (tbeg + i) * P_KEYS + half * 64;
            ok = ok && all_wait(err, &sfull[i & 1], (uint32_t)((i >> 1) & 1));
            __syncwarp();
            tc_fence_after();
            const bool edge = j0 <= clean_lo || j0 + 63 > clean_hi;
            const uint32_t off = edge && missing ? runs_gone(p, b, j0, 4) : 0u;
            float s[64], top = -INFINITY;
            row_scores(p, at + (uint32_t)(half * 64), j0, edge, QT == 1 && huge, r, off, s);
#pragma unroll
            for (int e = 0; e < 64; ++e) top = fmaxf(top, s[e]);
            top *= fac;
            wmax[i & 1][half][row] = top;
            __syncwarp();
            asm volatile("bar.sync %0, 64;" :: "r"(1 + quad) : "memory");          // the row's two warps
            top = fmaxf(top, wmax[i & 1][half ^ 1][row]);
            const bool up = top > m + P_LAZY;                     // (also the first finite maximum)
            if (__any_sync(0xffffffffu, up)) {                    // the same in both warps: each has half of the outputs
                const float fix = !up ? 1.f : (m == -INFINITY ? 0.f : exp2f(m - top));
                if (up) { m = top; neg = -top; }
                l *= fix;
                // From here on x - m of rounded x, as in the other kernel: in this place, where nothing is in a hurry, or, where registers are scarce (two terms a
                // weight: spills, 8 x 5 rows 34 us -> 42, so 36), in a run of weights of their own (whose branch costs one-term rows 3 %).
                if (!huge && p.cap_log2 <= 0.f && __any_sync(0xffffffffu, fabsf(neg) > KV4_HUGE)) {
                    huge = true;
                    if constexpr (QT == 1) {
#pragma unroll
                        for (int e = 0; e < 64; ++e) s[e] *= fac;
                        fac = 1.f;
                    }
                }
                if (i > 0) {
                    ok = ok && all_wait(err, &pvdone, (uint32_t)((i - 1) & 1));
                    __syncwarp();
                    tc_fence_after();
                    rescale(lanes + P_O + (uint32_t)(half * (DN / 2)), DN / 2, fix);
                }
            }
            uint64_t l2 = pair(0.f, 0.f);
            if (QT == 2 && huge) {
#pragma unroll
                for (int e = 0; e < 64; ++e) s[e] *= fac;
                weights32<QT>(s, 1.f, neg, at + (uint32_t)(half * 64), l2);
                weights32<QT>(s + 32, 1.f, neg, at + (uint32_t)(half * 64 + 16), l2);
            } else {
                weights32<QT>(s, fac, neg, at + (uint32_t)(half * 64), l2);           // to where the warp's own scores were
                weights32<QT>(s + 32, fac, neg, at + (uint32_t)(half * 64 + 16), l2);
            }
            float la, lb;
            unpair(l2, la, lb);
            l += la + lb;
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&pready[i & 1]);           // a barrier each: weights of two tiles may be ready before the first is looked for
        }
        asm volatile("bar.sync %0, 64;" :: "r"(1 + quad) : "memory");              // the last tile's maxima are read
        wmax[0][half][row] = l;
        __syncwarp();
        asm volatile("bar.sync %0, 64;" :: "r"(1 + quad) : "memory");
        if (half == 0) { row_m[row] = m; row_l[row] = wmax[0][0][row] + wmax[0][1][row]; }
    }
    __syncthreads();                               // nobody's tile is read or written any more
    tc_fence_after();
    float* const fold = (float*)smem;              // [128][D + 4], with more than one block a sequence
    if (warp < P_SOFT)
        outputs<DT>(p, r, D, half * (DN / 2), min(D, (half + 1) * (DN / 2)), tmem + ((uint32_t)(quad * 32) << 16) + P_O, n > 0, nans && r.live ? lost_groups<G>(p, b, r) : 0u,
                    p.splits > 1 ? 0.f : row_factor(p, r.h, row_m[row], row_l[row]), p.splits > 1 ? fold + (size_t)row * (D + 4) : nullptr);
    tc_fence_before();
    __syncthreads();
    if (warp == P_SOFT) tmem_dealloc(tmem, 512);
    if (p.splits > 1) fold_cluster<D, DT>(p, b, fold, row_m, row_l);
}

// The blocks' launch: blocks of rows, and how many blocks of a cluster share a sequence's keys: rounds of clusters times (a block's tiles + what it costs
// besides, about four of them).  How many clusters run at once is asked for: of eight blocks, one a SM, fewer than 148 / 8.  (Taking the SMs for it, 256
// rows of eight heads over 3000 keys were cut into 16 clusters of eight, two rounds: 34.5 us; four blocks a cluster: 21.6.)
template <int THREADS, int SMEM>
cudaError_t launch_blocks(void (*kernel)(Kv4AttnParams, Images, int*), Kv4AttnParams p, cudaStream_t st, int (&at_once)[4], Images im, int* err) {
    p.tiles = (int)(((long long)p.max_rows * p.rep + P_ROWS - 1) / P_ROWS);
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = SMEM;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 1;
    attr[0].val.clusterDim.y = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    const int keys = p.window > 0 && p.window < p.max_keys - P_ROWS ? p.window + P_ROWS : p.max_keys, nt = (keys + P_KEYS - 1) / P_KEYS;
    const long long items = (long long)p.seqs * p.tiles * p.k.kv_heads;
    long long least = 0;
    for (int i = 0; 1 << i <= P_CLUSTER; ++i) {
        const int s = 1 << i;
        if (at_once[i] == 0) {
            attr[0].val.clusterDim.z = (unsigned)s;
            cfg.gridDim = dim3(1, 1, s);
            cfg.numAttrs = 1;
            int n = 0;
            if (cudaError_t e = cudaOccupancyMaxActiveClusters(&n, kernel, &cfg)) return e;
            at_once[i] = n > 0 ? n : 1;
        }
        const long long cost = ((items + at_once[i] - 1) / at_once[i]) * ((nt + s - 1) / s + 4);
        if (s == 1 || cost < least) { p.splits = s; least = cost; }
    }
    attr[0].val.clusterDim.z = (unsigned)p.splits;
    cfg.gridDim = dim3((unsigned)(p.seqs * p.tiles), p.k.kv_heads, p.splits);
    cfg.numAttrs = 2;
    count_launch();
    return cudaLaunchKernelEx(&cfg, kernel, p, im, err);
}

template <int G, int DT>
int launch_prompt(Kv4AttnParams p, cudaStream_t st) {
    static bool configured = false;
    static int at_once[2][4] = {};
    if (!configured) {
        PGK_CUDA(cudaFuncSetAttribute(kv4_prompt_kernel<G, DT, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, Prompt<G>::BYTES));
        PGK_CUDA(cudaFuncSetAttribute(kv4_prompt_kernel<G, DT, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, Prompt<G>::BYTES));
        configured = true;
    }
    int* err = wait_word(kWaitKv4);
    PGK_REQUIRE(err, "kv4_attention failed: no pinned host memory");
    Images im = {};
    im.tiles = (p.max_keys + P_KEYS - 1) / P_KEYS;
    if (p.window > 0 && (long long)p.window + p.max_rows < p.max_keys) {
        const int few = (p.window + p.max_rows) / P_KEYS + 2;
        if (few < im.tiles) im.tiles = few;
    }
    const long long count = (long long)p.seqs * p.k.kv_heads * im.tiles, bytes = count * (2 * Prompt<G>::TILE + 4);
    void* ws = nullptr;
    if ((long long)p.max_rows * p.rep >= P_IMAGES_FROM && im.tiles > 0 && p.k.kv_heads <= 65535 && p.seqs <= 65535 && bytes <= P_IMAGES_MOST) {
        const int rc = scratch_alloc(&ws, (size_t)bytes, st);
        if (rc == (int)cudaErrorMemoryAllocation) set_error("");      // no room: the blocks make their tiles
        else if (rc) return rc;
    }
    cudaError_t e = cudaSuccess;
    if (ws) {
        im.data = (unsigned char*)ws;
        im.nans = (int32_t*)((unsigned char*)ws + count * (2 * Prompt<G>::TILE));
        e = launch_waiting(kv4_images_kernel<G>, dim3(im.tiles, p.k.kv_heads, p.seqs), dim3(P_EXPAND * 32), 0, st, p, im);
        if (e == cudaSuccess) e = launch_blocks<(P_SOFT + 2) * 32, Prompt<G>::BYTES>(kv4_prompt_kernel<G, DT, true>, p, st, at_once[1], im, err);
    } else {
        e = launch_blocks<P_THREADS, Prompt<G>::BYTES>(kv4_prompt_kernel<G, DT, false>, p, st, at_once[0], im, err);
    }
    if (int rc = scratch_free(ws, st)) return rc;
    PGK_CUDA(e);
    return 0;
}
template <int DT>
int launch_prompt_dim(const Kv4AttnParams& p, cudaStream_t st) {
    return p.k.dim == 64 ? launch_prompt<2, DT>(p, st) : (p.k.dim == 96 ? launch_prompt<3, DT>(p, st) : launch_prompt<4, DT>(p, st));
}

}  // namespace

// More rows than a block of the other kernel has (32 of 64 elements, 16 of more).  Measured there / here (us, 8 heads, 16 and 20 rows): 128 elements, one
// sequence over 3000 keys 14.2 / 15.6 and 15.6 / 15.5, 8 over 3000 21.7 / 28.0 and 32.1 / 27.9, 32 over 2000 39.4 / 60.7 and 66.5 / 60.8; 64 elements,
// 32 and 48 rows, 8 over 3000 24.8 / 23.6 and 35.8 / 23.8, 32 over 2000 42.4 / 49.7 and 77.3 / 49.4.  Caps that want the series of tanh stay there: its code
// would cost every call here 1 % (76.8 -> 77.5 us, 152.9 -> 154.7).
bool kv4_prompt_serves(const Kv4AttnParams& p, int dtype) {
    return dtype != 0 && p.k.dim <= 128 && p.cap_log2 <= KV4_CAP_WIDE && (long long)p.max_rows * p.rep > (p.k.dim == 64 ? 32 : 16);
}
int kv4_prompt(const Kv4AttnParams& p, int dtype, cudaStream_t st) { return dtype == 1 ? launch_prompt_dim<1>(p, st) : launch_prompt_dim<2>(p, st); }

}  // namespace pgk
