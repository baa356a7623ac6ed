// kv4_cache.cu -- rows into the four-bit paged cache (kv4.cuh has the format), the position rotation on the way, and back out of it.
//
//   q[t, h, :], k[t, h, :] rotated by the angles of positions[t] over their first R elements:  (a, b) -> (a cos - b sin, b cos + a sin)
//   for the pairs (i, i + R / 2), or (2 i, 2 i + 1);  q in place, k and v rounded to four bits into the page that holds the position.
//
// What bounds them: for prompts instructions, 61 % of the issue slots (4000 tokens of 32 and 8 heads of 128: 29.9 us, 2.9 TB/s of queries read and written, keys and
// values read, 9 / 16 byte an element written), for decoded tokens the launch (8: 2.2 us); reading back, memory and the launch (4000 tokens 5.2 us).
// A lane has eight neighbouring elements, one 32-bit word of codes; four lanes a group, D / 8 lanes a row; a rotation's other half comes
// from another lane of the warp, so that all of a row is loaded before any of it is written.  A warp keeps its token's angles and takes
// several of the token's heads.  Products and sums are rounded one by one (no fused multiply-add): a key on the border between two codes then
// falls where elementary float32 operations put it.
#include "kv4.cuh"
#include "../../include/pgk_b200.h"

namespace pgk {

namespace {

constexpr int A_WARPS = 4;

struct AppendParams {
    void* q; const void* k; const void* v;
    long q_ld, k_ld, v_ld;                // elements from token to token
    const float* cos; const float* sin;   // [table_rows][rot]
    int table_rows, rot, pairs;
    Kv4Pages kc;
    unsigned char* v_data;
    const int32_t* slots; const int32_t* positions;
    int tokens, heads;
    bool wide_q, wide_k, wide_v, wide_t;
};

template <int DT, int PER>
__global__ void __launch_bounds__(A_WARPS * 32) kv4_append_kernel(const __grid_constant__ AppendParams p) {
    griddep_wait();
    griddep_launch();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, token = blockIdx.x;
    const int D = p.kc.dim, W = D / 8, G = D / 32, side = 32 / W;         // side: rows of a warp at a time
    const int w = lane % W, which = lane / W, i0 = 8 * w, half = p.rot / 2;
    const int rows = p.heads + 2 * p.kc.kv_heads, first = (blockIdx.y * A_WARPS + warp) * PER * side;
    if (first >= rows) return;                                             // the whole warp
    const int pos = __ldcg(p.positions + token), slot = __ldcg(p.slots + token);
    // q heads, then k, then v
    auto place = [&](int r, int& kind, int& h) -> size_t {
        kind = r < p.heads ? 0 : (r < p.heads + p.kc.kv_heads ? 1 : 2);
        h = kind == 0 ? r : r - p.heads - (kind == 2 ? p.kc.kv_heads : 0);
        return (size_t)token * (kind == 0 ? p.q_ld : (kind == 1 ? p.k_ld : p.v_ld)) + (size_t)h * D + i0;
    };
    Kv4Eight<DT> raw[PER];
#pragma unroll
    for (int n = 0; n < PER; ++n) {
        const int r = first + n * side + which;
        int kind, h;
        const size_t at = place(r, kind, h);
        raw[n] = {};
        if (which < side && r < rows) raw[n].load(kind == 0 ? p.q : (kind == 1 ? p.k : p.v), at, kind == 0 ? p.wide_q : (kind == 1 ? p.wide_k : p.wide_v));
    }
    if (p.rot > 0 && (unsigned)pos >= (unsigned)p.table_rows) return;      // the whole block
    const bool turns = i0 < p.rot;
    const int other = p.pairs ? lane : (i0 < half ? lane + half / 8 : lane - half / 8);
    Kv4Eight<0> c8 = {}, s8 = {};                                          // in pairs: the first four
    if (turns) {
        const size_t at = (size_t)pos * p.rot + (p.pairs ? i0 / 2 : (i0 < half ? i0 : i0 - half));
        if (p.pairs) {
#pragma unroll
            for (int e = 0; e < 4; ++e) { c8.w[e] = __ldcg((const uint32_t*)p.cos + at + e); s8.w[e] = __ldcg((const uint32_t*)p.sin + at + e); }
        } else {
            c8.load(p.cos, at, p.wide_t);
            s8.load(p.sin, at, p.wide_t);
        }
    }
    const int page = kv4_page(p.kc, slot, pos);
    if (page < 0) return;
    float cs[8], sn[8];
    c8.floats(cs);
    s8.floats(sn);
    if (!p.pairs && i0 < half) {                                           // a cos - b sin as a cos + b (-sin): the same bits
#pragma unroll
        for (int e = 0; e < 8; ++e) sn[e] = -sn[e];
    }
    const int row = pos % p.kc.page_size;
#pragma unroll
    for (int n = 0; n < PER; ++n) {
        if (first + n * side >= rows) break;                               // the whole warp
        const int r = first + n * side + which;
        const bool live = which < side && r < rows;
        int kind, h;
        const size_t at = place(r, kind, h);
        float x[8], y[8];
        Kv4Eight<DT> far = raw[n];
        if (p.rot > 0 && !p.pairs) {
#pragma unroll
            for (int e = 0; e < (DT == 0 ? 8 : 4); ++e) far.w[e] = __shfl_sync(0xffffffffu, far.w[e], other & 31);
        }
        raw[n].floats(x);
        far.floats(y);
        if (turns && kind != 2) {
            if (p.pairs) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float a = x[2 * e], b = x[2 * e + 1];
                    x[2 * e] = __fsub_rn(__fmul_rn(a, cs[e]), __fmul_rn(b, sn[e]));
                    x[2 * e + 1] = __fadd_rn(__fmul_rn(b, cs[e]), __fmul_rn(a, sn[e]));
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = __fadd_rn(__fmul_rn(x[e], cs[e]), __fmul_rn(y[e], sn[e]));
            }
        }
        if (live && kind == 0) kv4_store8<DT>(p.q, at, p.wide_q, x);
        if (!__any_sync(0xffffffffu, live && kind != 0)) continue;
        uint32_t codes, word;
        kv4_encode(x, codes, word);
        if (live && kind != 0) {
            unsigned char* base = (kind == 1 ? p.kc.data : p.v_data) + ((size_t)page * p.kc.kv_heads + h) * ((size_t)p.kc.page_size * kv4_row_bytes(D));
            const int t = w & 3, g = w >> 2;
            *(uint32_t*)(base + (size_t)row * (D / 2) + 4 * (t * G + g)) = codes;
            if (t == 0) *(uint16_t*)(base + (size_t)p.kc.page_size * (D / 2) + ((size_t)row * G + g) * 2) = (uint16_t)word;
        }
    }
}

// a thread a word of codes of up to R_HEADS heads
constexpr int R_HEADS = 4;
template <int DT>
__global__ void __launch_bounds__(256) kv4_read_kernel(const __grid_constant__ Kv4Pages c, const int32_t* slots, const int32_t* positions, void* out, int tokens,
                                                       bool wide) {
    griddep_wait();
    griddep_launch();
    const int D = c.dim, W = D / 8, G = D / 32, parts = (c.kv_heads + R_HEADS - 1) / R_HEADS;
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= (long long)tokens * parts * W) return;
    const int w = (int)(i % W), h0 = (int)(i / W % parts) * R_HEADS, token = (int)(i / W / parts);
    const int pos = __ldcg(positions + token), page = kv4_page(c, __ldcg(slots + token), pos);
    uint32_t codes[R_HEADS] = {}, word[R_HEADS] = {};
    if (page >= 0) {
        const unsigned char* base = kv4_page_head(c, page, h0);
        const int row = pos % c.page_size, t = w & 3, g = w >> 2;
        const size_t head = (size_t)c.page_size * kv4_row_bytes(D), at = (size_t)row * (D / 2) + 4 * (t * G + g), words = (size_t)c.page_size * (D / 2) + 2 * ((size_t)row * G + g);
#pragma unroll
        for (int h = 0; h < R_HEADS; ++h)
            if (h0 + h < c.kv_heads) {
                codes[h] = __ldcg((const uint32_t*)(base + h * head + at));
                word[h] = ld_act2((const uint16_t*)(base + h * head + words));
            }
    }
#pragma unroll
    for (int h = 0; h < R_HEADS; ++h)
        if (h0 + h < c.kv_heads) {
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = kv4_value(codes[h], e, word[h]);
            kv4_store8<DT>(out, (((size_t)token * c.kv_heads + h0 + h) * W + w) * 8, wide, x);
        }
}

}  // namespace

// What both sides of the library check of a cache and its table.
int kv4_check(const char* fn, const void* data, int pages, int page_size, const void* table, int slots, int max_pages, int kv_heads, int dim) {
    PGK_REQUIRE(kv4_dim_ok(dim), "%s failed: heads of %d elements (64, 96, 128, 192 and 256 are served)", fn, dim);
    PGK_REQUIRE(page_size > 0 && page_size % 16 == 0 && page_size <= 4096, "%s failed: pages of %d positions (multiples of 16 up to 4096)", fn, page_size);
    PGK_REQUIRE(pages > 0 && slots > 0 && max_pages > 0 && kv_heads > 0 && (long long)max_pages * page_size <= 0x7fffffffll - 4096, "%s failed: %d pages, %d slots of %d, %d heads", fn,
                pages, slots, max_pages, kv_heads);
    PGK_REQUIRE(data && table && (uintptr_t)data % 16 == 0 && (uintptr_t)table % 4 == 0, "%s failed: the cache has to start on a 16-byte boundary", fn);
    return 0;
}

}  // namespace pgk

using namespace pgk;

extern "C" {

int pgk_kv4_append(void* q, const void* k, const void* v, long q_ld, long k_ld, long v_ld, const float* cos_table, const float* sin_table, int table_rows, int rot,
                   int interleaved, void* k_cache, void* v_cache, int pages, int page_size, const int32_t* page_table, int slots, int max_pages,
                   const int32_t* row_slots, const int32_t* positions, int tokens, int heads, int kv_heads, int dim, int dtype, void* stream) {
    const char* fn = "kv4_append";
    if (int rc = kv4_check(fn, k_cache, pages, page_size, page_table, slots, max_pages, kv_heads, dim)) return rc;
    if (int rc = kv4_check(fn, v_cache, pages, page_size, page_table, slots, max_pages, kv_heads, dim)) return rc;
    PGK_REQUIRE(dtype >= 0 && dtype <= 2, "kv4_append failed: unknown type %d", dtype);
    PGK_REQUIRE(rot >= 0 && rot <= dim && rot % 16 == 0, "kv4_append failed: a rotation of %d elements (multiples of 16 up to %d)", rot, dim);
    PGK_REQUIRE(rot == 0 || (cos_table && sin_table && table_rows > 0), "kv4_append failed: a rotation needs its tables");
    PGK_REQUIRE(tokens >= 0 && heads >= 0 && (heads == 0 || q) && k && v && k_ld >= (long)kv_heads * dim && v_ld >= (long)kv_heads * dim &&
                    (heads == 0 || q_ld >= (long)heads * dim) && (long long)heads + 2ll * kv_heads <= 65536,
                "kv4_append failed: %d tokens of %d and %d heads, rows of %ld, %ld and %ld", tokens, heads, kv_heads, q_ld, k_ld, v_ld);
    if (tokens == 0) return 0;
    PGK_REQUIRE(row_slots && positions, "kv4_append failed: no slots or positions");
    AppendParams p = {};
    p.q = q; p.k = k; p.v = v;
    p.q_ld = q_ld; p.k_ld = k_ld; p.v_ld = v_ld;
    p.cos = cos_table; p.sin = sin_table; p.table_rows = table_rows; p.rot = rot; p.pairs = interleaved != 0;
    p.kc = {(unsigned char*)k_cache, page_table, pages, page_size, slots, max_pages, kv_heads, dim};
    p.v_data = (unsigned char*)v_cache;
    p.slots = row_slots; p.positions = positions;
    p.tokens = tokens;
    p.heads = rot > 0 ? heads : 0;                              // queries that do not turn stay where they are
    const int size = dtype == 0 ? 4 : 2;
    auto wide = [&](const void* x, long ld) { return (uintptr_t)x % 16 == 0 && ld * size % 16 == 0; };
    p.wide_q = wide(q, q_ld); p.wide_k = wide(k, k_ld); p.wide_v = wide(v, v_ld);
    const int side = 32 / (dim / 8), steps = (p.heads + 2 * kv_heads + side - 1) / side;
    p.wide_t = rot > 0 && ((uintptr_t)cos_table | (uintptr_t)sin_table) % 16 == 0;
    // Prompts: a warp takes up to three steps of its token, whose loads are on their way together and share its page and angles; never so many that a block's
    // warps have none (us, one / two / three / six steps a warp: 32 and 8 heads of 128, 128 tokens 3.3 / 3.2 / 3.7 / 5.4, 512 7.0 / 6.7 / 5.7 / 7.8, 4000
    // 39.1 / 32.1 / 29.9 / 31.2; keys and values alone, 512 5.2 / 3.8 / 4.0 / 5.9; 8 and 1 heads of 64, 4000 7.3 / 7.8 / 8.8 / 10.2).
    const int full = (steps + A_WARPS - 1) / A_WARPS, per = (long long)tokens * steps < 4096 ? 1 : (full < 3 ? full : 3);
    const dim3 grid(tokens, (steps + A_WARPS * per - 1) / (A_WARPS * per));
    auto of = [&](auto* one, auto* two, auto* three) { return per == 1 ? one : (per == 2 ? two : three); };
    auto kernel = dtype == 0 ? of(kv4_append_kernel<0, 1>, kv4_append_kernel<0, 2>, kv4_append_kernel<0, 3>)
                             : (dtype == 1 ? of(kv4_append_kernel<1, 1>, kv4_append_kernel<1, 2>, kv4_append_kernel<1, 3>)
                                           : of(kv4_append_kernel<2, 1>, kv4_append_kernel<2, 2>, kv4_append_kernel<2, 3>));
    PGK_CUDA(launch_waiting(kernel, grid, dim3(A_WARPS * 32), 0, (cudaStream_t)stream, p));
    return 0;
}

int pgk_kv4_read(const void* cache, int pages, int page_size, const int32_t* page_table, int slots, int max_pages, const int32_t* row_slots,
                 const int32_t* positions, void* out, int tokens, int kv_heads, int dim, int dtype, void* stream) {
    if (int rc = kv4_check("kv4_read", cache, pages, page_size, page_table, slots, max_pages, kv_heads, dim)) return rc;
    PGK_REQUIRE(dtype >= 0 && dtype <= 2, "kv4_read failed: unknown type %d", dtype);
    PGK_REQUIRE(tokens >= 0, "kv4_read failed: %d rows", tokens);
    if (tokens == 0) return 0;
    PGK_REQUIRE(row_slots && positions && out, "kv4_read failed: no slots, positions or output");
    const Kv4Pages c = {(unsigned char*)cache, page_table, pages, page_size, slots, max_pages, kv_heads, dim};
    const long long blocks = ((long long)tokens * ((kv_heads + R_HEADS - 1) / R_HEADS) * (dim / 8) + 255) / 256;
    PGK_REQUIRE(blocks <= 0x7fffffffll, "kv4_read failed: %d rows", tokens);
    auto kernel = dtype == 0 ? kv4_read_kernel<0> : (dtype == 1 ? kv4_read_kernel<1> : kv4_read_kernel<2>);
    PGK_CUDA(launch_waiting(kernel, dim3((unsigned)blocks), dim3(256), 0, (cudaStream_t)stream, c, row_slots, positions, out, tokens, (uintptr_t)out % 16 == 0));
    return 0;
}

}  // extern "C"
