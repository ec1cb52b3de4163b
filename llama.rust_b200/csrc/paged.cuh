// What the operators over a paged cache share: argument checks, page look-ups.
#pragma once
#include <cuda_bf16.h>

#include "common.cuh"
#include "paged_b200.h"

namespace b200 {

constexpr int ERR_PAGED = 7;   // error code of a kernel that met a page, sequence, position or parent outside its range

// The cache as kernels read it
struct PagedCache {
    uint8_t *k, *v;
    int64_t page_stride;
    const int32_t *tables;
    int64_t table_ld, n_pages;
    int page_log2, n_head_kv, d, n_seq;
};

int paged_check_cache(const b200_paged_cache &c, const char *op, PagedCache *out);   // paged_append.cu
// refuses operands (null: not given) that are not aligned to their elements, and those that no kernel of the current device may touch: another device's memory, the host's
// pageable memory
struct PagedOperand {
    const void *p;
    const char *name;
    unsigned align = 1;   // bytes of an element, where nothing else has looked at it
};
int paged_check_device(const PagedOperand *operands, int n, const char *op);
inline bool paged_overlap(const void *a, size_t na, const void *b, size_t nb) { return (uintptr_t)a < (uintptr_t)b + nb && (uintptr_t)b < (uintptr_t)a + na; }

// Byte offset of position p of sequence s in the cache (K and V alike), or -1 where the table or a page id does not reach
__device__ __forceinline__ int64_t paged_row(const PagedCache &c, int s, int p) {
    const int i = p >> c.page_log2;
    if (i >= c.table_ld) return -1;
    const int32_t page = __ldg(c.tables + (int64_t)s * c.table_ld + i);
    if (page < 0 || page >= c.n_pages) return -1;
    return page * c.page_stride + (int64_t)(p & ((1 << c.page_log2) - 1)) * c.n_head_kv * c.d * 2;
}

template <typename T>
__device__ __forceinline__ float paged_f32(T v) { return (float)v; }
template <typename T>
__device__ __forceinline__ T paged_from(float v);
template <>
__device__ __forceinline__ __half paged_from<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 paged_from<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
// two values of a word, low half first
template <typename T>
__device__ __forceinline__ uint32_t paged_pack(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t paged_pack<__half>(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *(const uint32_t *)&h;
}
template <>
__device__ __forceinline__ uint32_t paged_pack<__nv_bfloat16>(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *(const uint32_t *)&h;
}
template <typename T>
__device__ __forceinline__ float2 paged_two(uint32_t w);
template <>
__device__ __forceinline__ float2 paged_two<__half>(uint32_t w) { return __half22float2(*(const __half2 *)&w); }
template <>
__device__ __forceinline__ float2 paged_two<__nv_bfloat16>(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }

}  // namespace b200
