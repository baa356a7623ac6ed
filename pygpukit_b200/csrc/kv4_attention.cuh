// kv4_attention.cuh -- what the kernels of attention over the four-bit cache share: kv4_attention.cu (a few rows a sequence), kv4_prompt.cu (many).
#pragma once
#include "kv4.cuh"
#include "tc_common.cuh"

namespace pgk {

struct Kv4AttnParams {
    const void* q; void* out;
    long q_ld, o_ld;
    Kv4Pages k;
    const unsigned char* v_data;
    const int32_t* seq_slots; const int32_t* contexts; const int32_t* starts;      // starts NULL: a row a sequence
    int seqs, tokens, max_rows, max_keys, heads, rep, tiles, splits;
    float scale_log2, cap_log2;           // scale log2 e; cap log2 e or 0
    int window;
    const float* sinks;
    bool wide_q, wide_o;                  // rows on 16-byte boundaries
    uint32_t page_mul, page_shift;        // n / (page_size / 16) = hi(n page_mul) >> page_shift; page_mul 0: pages of 16
    long long page_bytes, head_bytes;
};

constexpr float KV4_CAP_WIDE = 256.f;      // a cap (times log2 e) from which tanh is wanted to float32 of itself, not of 1

// kv4_prompt.cu: whether it serves the call, and the call
bool kv4_prompt_serves(const Kv4AttnParams& p, int dtype);
int kv4_prompt(const Kv4AttnParams& p, int dtype, cudaStream_t st);

#ifdef __CUDACC__

constexpr float KV4_HUGE = 268435456.f;                            // a reference of 2^28: float32 has steps of 32 there

// The first key that the row of position `pos` sees.  Windows and contexts are any 32-bit numbers, and a sequence may have rows before its position 0:
// pos - window + 1 of such a row may lie below -2^31, and is not formed.
__device__ __forceinline__ int kv4_first_key(const Kv4AttnParams& p, int pos) { return p.window > 0 && pos >= p.window ? pos - p.window + 1 : 0; }

// the page that holds the 16 positions n
__device__ __forceinline__ uint32_t kv4_page_of(const Kv4AttnParams& p, uint32_t n) { return p.page_mul ? __umulhi(n, p.page_mul) >> p.page_shift : n; }

// A capped score is cap tanh(y), y = z ln 2 / 2 with z the score times kv4_cap_in.  As 1 - 2 / (1 + e^2y) tanh is off by 2^-22 whatever y is: of a cap of KV4_CAP_WIDE
// (in units of log2 e: 177) that is 6e-5 of a weight, and everything of much wider ones, which take its series below y = 0.3 (to y^9: 5e-8 of it).
__device__ __forceinline__ float kv4_tanh(float z) { return 1.f - __fdividef(2.f, 1.f + ex2(z)); }
// (a call: inline it costs every kernel's other paths 1 %, 152 -> 154 us)
static __device__ __noinline__ float kv4_tanh_wide(float z) {
    const float y = z * 0.34657359f, y2 = y * y;
    return fabsf(y) < 0.3f ? fmaf(y * y2, fmaf(y2, fmaf(y2, fmaf(y2, 62.f / 2835.f, -17.f / 315.f), 2.f / 15.f), -1.f / 3.f), y) : kv4_tanh(z);
}
__device__ __forceinline__ float kv4_cap_in(float scale, float cap) { return fminf(scale * 2.885390043f / cap, 3.4028235e38f); }     // (no infinity that a zero meets)

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t remote(uint32_t at, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(at), "r"(rank));
    return r;
}
__device__ __forceinline__ float remote_float(uint32_t at) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ float4 remote_float4(uint32_t at) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
    return v;
}

#endif  // __CUDACC__

}  // namespace pgk
