// The paged key/value cache as the kernels see it: a pool of pages, keys and values each [pages, kv_heads, page_size,
// head_dim], and the sequences of a call.  Everything that the device holds about the sequences is taken as it comes:
// whatever the numbers say, no access leaves the row buffers, the page table or the pool.
#pragma once

#include "common.cuh"
#include "kernels.h"

namespace b200exl3 {

// New tokens of one sequence: rows first_row .. first_row + n - 1, token i of them at position first_pos + i.
struct KvSeq {
    int first_row, n, first_pos;
};

__device__ __forceinline__ int kv_clamp_row(const KvArgs& p, int r) {
    return r < 0 ? 0 : (r > p.rows ? static_cast<int>(p.rows) : r);
}
__device__ __forceinline__ int kv_clamp_length(int n) { return n < 0 ? 0 : (n > kKvMaxTokens ? kKvMaxTokens : n); }

__device__ __forceinline__ int kv_page_index(const KvArgs& p, int pos) {
    return p.page_shift >= 0 ? pos >> p.page_shift : pos / p.page_size;
}

// The vector of (page, head 0, row of the page) counted in vectors of the pool, head h another h * page_size on; -1 where the
// table or the pool ends.
__device__ __forceinline__ int64_t kv_place(const KvArgs& p, int b, int pos) {
    const int index = kv_page_index(p, pos);
    if (pos < 0 || index >= p.table_width) return -1;
    const int page = __ldg(p.table + static_cast<int64_t>(b) * p.table_width + index);
    if (page < 0 || page >= p.pages) return -1;
    return static_cast<int64_t>(page) * p.kv_heads * p.page_size + (pos - index * p.page_size);
}

template <typename T> struct KvType;
template <> struct KvType<__half> {
    using Two = __half2;
    static constexpr uint32_t kExponent = 0x7c007c00u, kExponentStep = 0x04000400u;
    static __device__ __forceinline__ float2 unpack(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
};
template <> struct KvType<__nv_bfloat16> {
    using Two = __nv_bfloat162;
    static constexpr uint32_t kExponent = 0x7f807f80u, kExponentStep = 0x00800080u;
    static __device__ __forceinline__ float2 unpack(uint32_t w) { return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w)); }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
};
// Adds zero times two numbers: a sum that began at zero stays there unless one of them is an infinity or NaN.
template <typename T>
__device__ __forceinline__ void kv_look(uint32_t& sum, uint32_t w) {
    using Two = typename KvType<T>::Two;
    const uint32_t zero = 0;
    const Two s = __hfma2(*reinterpret_cast<const Two*>(&w), *reinterpret_cast<const Two*>(&zero), *reinterpret_cast<const Two*>(&sum));
    sum = *reinterpret_cast<const uint32_t*>(&s);
}
__device__ __forceinline__ bool kv_found(uint32_t sum) { return (sum & 0x7fff7fffu) != 0; }
// The top bit of each of two numbers that is an infinity or NaN: one step more than the largest exponent.
template <typename T>
__device__ __forceinline__ uint32_t kv_not_finite(uint32_t w) { return ((w & KvType<T>::kExponent) + KvType<T>::kExponentStep) & 0x80008000u; }
// The two numbers with zeros in those places
__device__ __forceinline__ uint32_t kv_without(uint32_t w, uint32_t top_bits) { return w & ~((top_bits >> 15) * 0xffffu); }

}  // namespace b200exl3
