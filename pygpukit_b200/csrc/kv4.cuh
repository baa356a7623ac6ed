// kv4.cuh -- keys and values in four bits: the format, and the paged cache that holds it.
//
// A group is 32 neighbouring elements of one head's row.  With lo = min(0, min x) and hi = max(0, max x) of the group,
//     s = (hi - lo) / 15, rounded up to four significant bits;  z = rint(-lo / s);  c = clip(rint(x / s) + z, 0, 15);  x ~ s (c - z).
// (c - z) has four bits and a sign and s four: what the cache stands for is a bfloat16 number exactly, so that nothing is lost when a
// kernel hands it to the tensor cores, and 0 is 0.  A group's word is 16 bits: the scale as a bfloat16 in bits 4 to 14 (its lower four bits of
// mantissa are zero) and z in bits 0 to 3.  Scales are 0 or 2^-40 ... 2^53: smaller groups are zeros (word 0); a group that holds a NaN, an
// infinity or a magnitude of 2^56 has a NaN scale (kKv4Nan), and whoever sees the row gets NaN, as from a row of floats.
//
// A page of one head is one run of bytes: page_size rows of D / 2 bytes of codes, then page_size rows of D / 32 words.  With G = D / 32 the
// 32-bit word t G + g of a row holds elements 32 g + 8 t ... 32 g + 8 t + 7 (element e in nibble e): the lanes t = 0 ... 3 of a quad
// of an m16n8k16 product then find the words of all groups side by side, and two products of 16 elements are one group.
#pragma once
#include "common.cuh"

namespace pgk {

constexpr uint32_t kKv4Nan = 0x7fc0u;

struct Kv4Pages {                         // one cache (keys or values) and the table that orders its pages
    unsigned char* data;
    const int32_t* table;                 // [slots][max_pages]
    int pages, page_size, slots, max_pages, kv_heads, dim;
};
__host__ __device__ constexpr int kv4_row_bytes(int dim) { return dim / 2 + dim / 16; }
inline bool kv4_dim_ok(int dim) { return dim == 64 || dim == 96 || dim == 128 || dim == 192 || dim == 256; }

#ifdef __CUDACC__

// the page that holds a position, or -1: whatever a slot, a position or the table says, nothing outside the cache is touched
__device__ __forceinline__ int kv4_page(const Kv4Pages& c, int slot, int pos) {
    if ((unsigned)slot >= (unsigned)c.slots || pos < 0) return -1;
    const int i = pos / c.page_size;
    if (i >= c.max_pages) return -1;
    const int p = __ldcg(c.table + (size_t)slot * c.max_pages + i);
    return (unsigned)p < (unsigned)c.pages ? p : -1;
}
__device__ __forceinline__ unsigned char* kv4_page_head(const Kv4Pages& c, int page, int head) {
    return c.data + ((size_t)page * c.kv_heads + head) * ((size_t)c.page_size * kv4_row_bytes(c.dim));
}

__device__ __forceinline__ float kv4_scale(uint32_t word) { return __uint_as_float((word & 0x7ff0u) << 16); }
__device__ __forceinline__ float kv4_value(uint32_t codes, int e, uint32_t word) {
    return kv4_scale(word) * (float)((int)((codes >> (4 * e)) & 15u) - (int)(word & 15u));
}

// Eight elements of a group that lies in four neighbouring lanes (32-lane converged call): the codes, and the group's word.
__device__ __forceinline__ void kv4_encode(const float (&x)[8], uint32_t& codes, uint32_t& word) {
    float lo = 0.f, hi = 0.f;
    bool bad = false;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        lo = fminf(lo, x[e]);
        hi = fmaxf(hi, x[e]);
        bad |= !(fabsf(x[e]) < 7.2057594e16f);                 // 2^56, and NaN
    }
#pragma unroll
    for (int o = 1; o <= 2; o <<= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        bad |= (bool)__shfl_xor_sync(0xffffffffu, (int)bad, o);
    }
    const float s = __uint_as_float((__float_as_uint(__fdiv_rn(hi - lo, 15.f)) + 0xfffffu) & ~0xfffffu);
    codes = 0;
    word = 0;
    if (bad) { word = kKv4Nan; return; }
    if (!(s >= 9.094947e-13f)) return;                         // 2^-40
    // x / s by a product with the rounded reciprocal and one residual: correctly rounded (Markstein, IBM J. Res. Dev. 34, 1990), 3 operations where a
    // division of its own takes about ten.  Adding 1.5 2^23 leaves a quotient of 15 at most rounded to the nearest integer in the lowest bits.
    const float r = __frcp_rn(s), magic = 12582912.f;
    auto rounded = [&](float x) {
        const float q = x * r;
        return __float_as_uint(__fadd_rn(fmaf(fmaf(-s, q, x), r, q), magic)) - 0x4b400000u;
    };
    const int z = (int)rounded(-lo);
    word = (__float_as_uint(s) >> 16) | (uint32_t)z;
#pragma unroll
    for (int e = 0; e < 8; ++e) codes |= (uint32_t)min(max((int)rounded(x[e]) + z, 0), 15) << (4 * e);
}

// eight neighbouring elements of type DT (0 f32, 1 f16, 2 bf16) as they lie in memory; `wide`: they start on a 16-byte boundary
template <int DT> struct Kv4Eight {
    uint32_t w[DT == 0 ? 8 : 4];
    __device__ __forceinline__ void load(const void* base, size_t at, bool wide) {
        if constexpr (DT == 0) {
            const uint32_t* p = (const uint32_t*)base + at;
            if (wide) {
                const uint4 a = ld_act16(p), b = ld_act16(p + 4);
                w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
                w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) w[e] = __ldcg(p + e);
            }
        } else {
            const uint16_t* p = (const uint16_t*)base + at;
            if (wide) {
                const uint4 a = ld_act16(p);
                w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = (uint32_t)ld_act2(p + 2 * e) | (uint32_t)ld_act2(p + 2 * e + 1) << 16;
            }
        }
    }
    __device__ __forceinline__ void floats(float (&x)[8]) const {
        if constexpr (DT == 0) {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = __uint_as_float(w[e]);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if constexpr (DT == 2) {
                    x[2 * e] = bf16lo(w[e]);
                    x[2 * e + 1] = bf16hi(w[e]);
                } else {
                    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[e]));
                    x[2 * e] = f.x;
                    x[2 * e + 1] = f.y;
                }
            }
        }
    }
};
template <int DT>
__device__ __forceinline__ uint32_t kv4_pack2(float lo, float hi) {
    if constexpr (DT == 2) return pack_bf16x2(lo, hi);
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <int DT>
__device__ __forceinline__ void kv4_store8(void* base, size_t at, bool wide, const float (&x)[8]) {
    if constexpr (DT == 0) {
        float* p = (float*)base + at;
        if (wide) {
            *(float4*)p = make_float4(x[0], x[1], x[2], x[3]);
            *(float4*)(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) p[e] = x[e];
        }
    } else {
        uint16_t* p = (uint16_t*)base + at;
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = kv4_pack2<DT>(x[2 * e], x[2 * e + 1]);
        if (wide) {
            *(uint4*)p = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                p[2 * e] = (uint16_t)w[e];
                p[2 * e + 1] = (uint16_t)(w[e] >> 16);
            }
        }
    }
}

#endif  // __CUDACC__

}  // namespace pgk
