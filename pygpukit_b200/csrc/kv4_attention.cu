// kv4_attention.cu -- attention over the four-bit paged cache (kv4.cuh has the format).
//
//   o[t, h, :] = sum_j w_j v_j / (sum_j w_j + exp(sink_h - m)),   w_j = exp(x_j - m),   x_j = scale q[t, h, :] . k_j, capped c tanh(x_j / c)
//   over the keys j <= pos(t), with a window also j > pos(t) - window;  pos(t) = context - rows + (t's place among its sequence's rows)
//
// A row that sees no key gives zeros.
#include "kv4.cuh"
#include "../../include/pgk_b200.h"

namespace pgk {

int kv4_check(const char* fn, const void* data, int pages, int page_size, const void* table, int slots, int max_pages, int kv_heads, int dim);

namespace {

struct Kv4AttnParams {
    const void* q; void* out;
    long q_ld, o_ld;
    Kv4Pages k;
    const unsigned char* v_data;
    const int32_t* seq_slots; const int32_t* contexts; const int32_t* starts;      // starts NULL: a row a sequence
    int seqs, tokens, max_rows, max_keys, heads;
    float scale, softcap;
    int window;
    const float* sinks;
};

template <int DT>
__global__ void __launch_bounds__(128) kv4_attention_plain_kernel(const __grid_constant__ Kv4AttnParams p) {
    __shared__ float qs[4][256];
    griddep_wait();
    griddep_launch();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, h = blockIdx.y * 4 + warp;
    const int seq = blockIdx.x / p.max_rows, r = blockIdx.x - seq * p.max_rows;
    const int first = p.starts ? __ldcg(p.starts + seq) : seq, last = p.starts ? __ldcg(p.starts + seq + 1) : seq + 1;
    const int t = first + r;
    const int slot = __ldcg(p.seq_slots + seq), ctx = __ldcg(p.contexts + seq);
    if (h >= p.heads || t >= last || t < 0 || t >= p.tokens || (unsigned)slot >= (unsigned)p.k.slots) return;
    const int D = p.k.dim, G = D / 32, g = h / (p.heads / p.k.kv_heads);
    const int pos = ctx - (last - first) + r;
    for (int i = lane; i < D / 8; i += 32) {
        float x[8];
        kv4_load8<DT>(p.q, (size_t)t * p.q_ld + (size_t)h * D + 8 * i, false, x);
        for (int e = 0; e < 8; ++e) qs[warp][8 * i + e] = x[e];
    }
    __syncwarp();
    float m = p.sinks ? __ldcg(p.sinks + h) : -INFINITY, l = m == -INFINITY ? 0.f : 1.f, acc[8] = {};
    const int begin = p.window > 0 ? max(0, pos - p.window + 1) : 0, end = min(min(pos + 1, ctx), p.max_keys);
    for (int j0 = begin; j0 < end; j0 += 32) {
        const int j = j0 + lane, page = j < end ? kv4_page(p.k, slot, j) : -1, row = j % p.k.page_size;
        const size_t at = page < 0 ? 0 : ((size_t)page * p.k.kv_heads + g) * ((size_t)p.k.page_size * kv4_row_bytes(D));
        float x = -INFINITY;
        if (page >= 0) {
            const unsigned char* base = p.k.data + at;
            x = 0.f;
            for (int gi = 0; gi < G; ++gi) {
                const uint32_t word = ld_act2((const uint16_t*)(base + (size_t)p.k.page_size * (D / 2)) + (size_t)row * G + gi);
                for (int w = 0; w < 4; ++w) {
                    const uint32_t codes = __ldcg((const uint32_t*)(base + (size_t)row * (D / 2)) + w * G + gi);
                    for (int e = 0; e < 8; ++e) x = fmaf(qs[warp][32 * gi + 8 * w + e], kv4_value(codes, e, word), x);
                }
            }
            x *= p.scale;
            if (p.softcap > 0.f) x = p.softcap * tanhf(x / p.softcap);
        }
        const float top = fmaxf(m, warp_max(x));
        const bool nan = __any_sync(0xffffffffu, x != x);
        const float f = m == -INFINITY ? 0.f : expf(m - top);
        const float w = x == -INFINITY ? 0.f : expf(x - top);
        l = l * f + warp_sum(w);
        if (nan) l = NAN;
        for (int gi = 0; gi < G; ++gi) acc[gi] *= f;
        m = top;
        for (int n = 0; n < 32 && j0 + n < end; ++n) {
            const float wn = __shfl_sync(0xffffffffu, w, n);
            const size_t atn = __shfl_sync(0xffffffffu, (unsigned long long)at, n);
            const int pg = __shfl_sync(0xffffffffu, page, n);
            if (pg < 0) continue;
            const int rn = (j0 + n) % p.k.page_size;
            const unsigned char* base = p.v_data + atn;
            for (int gi = 0; gi < G; ++gi) {
                const uint32_t word = ld_act2((const uint16_t*)(base + (size_t)p.k.page_size * (D / 2)) + (size_t)rn * G + gi);
                const uint32_t codes = __ldcg((const uint32_t*)(base + (size_t)rn * (D / 2)) + (lane >> 3) * G + gi);
                acc[gi] = fmaf(wn, kv4_value(codes, lane & 7, word), acc[gi]);
            }
        }
    }
    const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
    for (int gi = 0; gi < G; ++gi) {
        const size_t at = (size_t)t * p.o_ld + (size_t)h * D + 32 * gi + lane;
        const float o = acc[gi] * inv;
        if constexpr (DT == 0) ((float*)p.out)[at] = o;
        else ((uint16_t*)p.out)[at] = (uint16_t)kv4_pack2<DT>(o, 0.f);
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
    PGK_REQUIRE(heads > 0 && heads % kv_heads == 0 && heads <= 65535 && q_ld >= (long)heads * dim && o_ld >= (long)heads * dim,
                "kv4_attention failed: %d query heads over %d, rows of %ld and %ld", heads, kv_heads, q_ld, o_ld);
    PGK_REQUIRE(seqs >= 0 && tokens >= 0 && max_rows > 0 && max_context >= 0 && (row_starts || (tokens >= seqs && max_rows == 1)) && (long long)seqs * max_rows <= 0x7fffffffll,
                "kv4_attention failed: %d sequences of up to %d rows in %d, %d keys", seqs, max_rows, tokens, max_context);
    PGK_REQUIRE(window >= 0 && softcap >= 0.f && scale == scale, "kv4_attention failed: window %d, cap %g, scale %g", window, softcap, scale);
    if (seqs == 0 || tokens == 0) return 0;
    PGK_REQUIRE(q && out && seq_slots && context_lens, "kv4_attention failed: no queries, output, slots or contexts");
    Kv4AttnParams p = {};
    p.q = q; p.out = out; p.q_ld = q_ld; p.o_ld = o_ld;
    p.k = {(unsigned char*)k_cache, page_table, pages, page_size, slots, max_pages, kv_heads, dim};
    p.v_data = (const unsigned char*)v_cache;
    p.seq_slots = seq_slots; p.contexts = context_lens; p.starts = row_starts;
    p.seqs = seqs; p.tokens = tokens; p.max_rows = max_rows; p.heads = heads;
    p.max_keys = max_context < max_pages * page_size ? max_context : max_pages * page_size;
    p.scale = scale > 0.f ? scale : 1.f / sqrtf((float)dim);
    p.window = window; p.softcap = softcap; p.sinks = sinks;
    auto kernel = dtype == 0 ? kv4_attention_plain_kernel<0> : (dtype == 1 ? kv4_attention_plain_kernel<1> : kv4_attention_plain_kernel<2>);
    PGK_CUDA(launch_waiting(kernel, dim3((unsigned)seqs * max_rows, (heads + 3) / 4), dim3(128), 0, (cudaStream_t)stream, p));
    return 0;
}
