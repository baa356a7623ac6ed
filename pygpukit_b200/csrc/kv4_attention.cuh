// kv4_attention.cuh -- what the kernels of attention over the four-bit cache share: kv4_attention.cu (a few rows a sequence), kv4_prompt.cu (many).
#pragma once
#include "kv4.cuh"

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
