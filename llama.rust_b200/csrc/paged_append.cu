// Keys and values of a step into a paged cache, keys and queries rotated on the way (b200_paged_append).
//
//   y[e0] = x[e0] cos - x[e1] sin,  y[e1] = x[e0] sin + x[e1] cos     for the channel pairs (e0, e1) of the first n_dims channels
//
// in F32, rounded once to the cache's 16 bits.  Bound by memory: every element is read once and written once, and nothing but a table row of (cos, sin)
// is read twice (by the heads of a token, from L1 and L2).  A thread takes 16 channels of one head of one token: the eight that a rotation
// brings together with eight others and these, so that F32 rows are read 32 bytes at a time, 16-bit rows and the cache 16.
// Rows whose addresses do not allow that, or whose rotating channels are no multiple of 16, go pair by pair.
// Measured on the device, 32 heads on 8 of 128, F32 into BF16: 8192 tokens 51.5 us (306 MB: 5.9 TB/s, 0.92 of the measured copy rate; 58 us with two 16-byte loads in the
// place of one of 32), four tokens 1.8 us.
#include "paged.cuh"

namespace b200 {

int paged_check_device(const PagedOperand *operands, int n, const char *op) {
    for (int i = 0; i < n; i++) B200_REQUIRE((uintptr_t)operands[i].p % operands[i].align == 0, "%s: %s must be aligned to %u bytes", op, operands[i].name, operands[i].align);
    int dev = 0;
    B200_CUDA(cudaGetDevice(&dev));
    for (int i = 0; i < n; i++) {
        const char *const what = operands[i].name;
        if (operands[i].p == nullptr) continue;
        cudaPointerAttributes at;
        if (cudaPointerGetAttributes(&at, operands[i].p) != cudaSuccess) {
            cudaGetLastError();
            B200_REQUIRE(false, "%s: %s is not memory that a kernel can touch", op, what);
        }
        B200_REQUIRE(at.type != cudaMemoryTypeUnregistered, "%s: %s is pageable host memory", op, what);
        B200_REQUIRE(at.type != cudaMemoryTypeDevice || at.device == dev, "%s: %s is memory of device %d, the current device is %d", op, what, at.device, dev);
    }
    return B200_STATUS_SUCCESS;
}

int paged_check_cache(const b200_paged_cache &c, const char *op, PagedCache *out) {
    B200_REQUIRE(c.type == B200_TYPE_F16 || c.type == B200_TYPE_BF16, "%s: cache type %d is neither F16 nor BF16", op, c.type);
    B200_REQUIRE(c.page_size >= 16 && c.page_size <= 256 && (c.page_size & (c.page_size - 1)) == 0, "%s: pages of %d positions (16, 32, 64, 128 or 256 are served)", op, c.page_size);
    B200_REQUIRE(c.n_head_kv > 0 && c.n_head_kv <= 65535, "%s: %lld key heads", op, (long long)c.n_head_kv);
    B200_REQUIRE(c.d > 0 && c.d <= 1024 && c.d % 16 == 0, "%s: heads of %lld channels (a multiple of 16 up to 1024 is wanted)", op, (long long)c.d);
    B200_REQUIRE(c.k != nullptr && c.v != nullptr && c.tables != nullptr, "%s: null cache operand", op);
    B200_REQUIRE((((uintptr_t)c.k | (uintptr_t)c.v) & 15) == 0, "%s: pages must be 16-byte aligned", op);
    B200_REQUIRE(c.n_pages > 0 && c.n_pages <= 0x7fffffffLL && c.table_ld > 0 && c.table_ld <= 0x7fffffffLL && c.n_seq > 0 && c.n_seq <= 0x7fffffffLL, "%s: empty or too large a cache (%lld pages, %lld table entries, %lld sequences)", op,
                 (long long)c.n_pages, (long long)c.table_ld, (long long)c.n_seq);
    const int64_t page = (int64_t)c.page_size * c.n_head_kv * c.d * 2, stride = c.page_stride ? c.page_stride : page;
    B200_REQUIRE(stride >= page && stride % 16 == 0 && stride < (1LL << 40), "%s: a page stride of %lld bytes (at least %lld, a multiple of 16, below 2^40)", op, (long long)stride, (long long)page);
    out->k = (uint8_t *)c.k;
    out->v = (uint8_t *)c.v;
    out->page_stride = stride;
    out->tables = c.tables;
    out->table_ld = c.table_ld;
    out->n_pages = c.n_pages;
    out->page_log2 = __builtin_ctz((unsigned)c.page_size);
    out->n_head_kv = (int)c.n_head_kv;
    out->d = (int)c.d;
    out->n_seq = (int)c.n_seq;
    return B200_STATUS_SUCCESS;
}

namespace {

struct AppendArgs {
    PagedCache cache;
    const int32_t *pos, *seq;
    const uint8_t *x[3];             // q, k, v
    int64_t x_nb1[3], x_nb2[3];
    uint8_t *q_out;
    int64_t q_out_nb1, q_out_nb2;
    const float *rope;
    int64_t rope_rows, rope_ld;
    int n_head, n_dims, neox;
    unsigned per_tok, units;         // threads of a token, of a head
    int64_t n_tok;
    int *err;
};
constexpr int AP_NT = 128;

template <typename XT>
__device__ __forceinline__ void load8(const XT *p, float (&v)[8]) {
    const uint4 a = *(const uint4 *)p;
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 f = paged_two<XT>(w[i]);
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}
template <>
__device__ __forceinline__ void load8<float>(const float *p, float (&v)[8]) {
    if (((uintptr_t)p & 31) == 0) {   // a sector at once
        asm volatile("ld.global.v8.f32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];" : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]) : "l"(p) : "memory");
        return;
    }
    const float4 a = *(const float4 *)p, b = *(const float4 *)(p + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
template <typename CT>
__device__ __forceinline__ void store8(CT *p, const float (&v)[8]) {
    *(uint4 *)p = make_uint4(paged_pack<CT>(v[0], v[1]), paged_pack<CT>(v[2], v[3]), paged_pack<CT>(v[4], v[5]), paged_pack<CT>(v[6], v[7]));
}
__device__ __forceinline__ void turn(float &a, float &b, float c, float s) {
    const float x0 = a, x1 = b;
    a = __fmaf_rn(x0, c, -__fmul_rn(x1, s));
    b = __fmaf_rn(x0, s, __fmul_rn(x1, c));
}

// A thread has one unit of one head of one token (a CTA a token, or 128 units of it; two or four tokens a thread, their rows on the way together, took longer:
// 58 and 68 us for 55).  VEC: a unit is 16 channels, else one pair
template <typename XT, typename CT, bool VEC>
__global__ void __launch_bounds__(AP_NT) paged_append_kernel(const AppendArgs a) {
    constexpr int W = VEC ? 8 : 1;
    pdl_trigger();
    const unsigned in_tok = blockIdx.y * AP_NT + threadIdx.x, slot = in_tok / a.units, u = in_tok - slot * a.units;
    if (in_tok >= a.per_tok) return;
    const int64_t t = blockIdx.x;
    const int what = (int)slot < a.n_head ? 0 : (int)slot < a.n_head + a.cache.n_head_kv ? 1 : 2;
    const int h = what == 0 ? (int)slot : what == 1 ? (int)slot - a.n_head : (int)slot - a.n_head - a.cache.n_head_kv;
    const bool turns = what < 2 && 2 * W * (int)u < a.n_dims;
    const int e0 = turns && a.neox ? W * u : 2 * W * u, e1 = turns && a.neox ? e0 + a.n_dims / 2 : e0 + W;
    const XT *const src = (const XT *)(a.x[what] + t * a.x_nb1[what] + h * a.x_nb2[what]);
    pdl_wait();
    const int32_t p = a.pos[t], s = a.seq ? a.seq[t] : (int32_t)t;
    float x0[W], x1[W];
    if constexpr (VEC) {   // on the way before the position is known
        load8<XT>(src + e0, x0);
        load8<XT>(src + e1, x1);
    } else {
        x0[0] = paged_f32(src[e0]);
        x1[0] = paged_f32(src[e1]);
    }
    if (p < 0) return;
    // where it goes; what has no place is left out, of a token as a whole
    const int64_t row = s >= 0 && s < a.cache.n_seq ? paged_row(a.cache, s, p) : -1;
    if (row < 0 || (a.n_dims > 0 && p >= a.rope_rows)) {
        if (in_tok == 0) atomicExch(a.err, ERR_PAGED);
        return;
    }
    CT *const dst = what == 0 ? (CT *)(a.q_out + t * a.q_out_nb1 + h * a.q_out_nb2) : (CT *)((what == 1 ? a.cache.k : a.cache.v) + row) + (int64_t)h * a.cache.d;
    const float *const table = a.rope + p * a.rope_ld + 2 * W * u;
    if constexpr (VEC) {
        if (turns) {
            float c0[8], c1[8];
            load8<float>(table, c0);
            load8<float>(table + 8, c1);
            if (a.neox) {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    turn(x0[e], x1[e], c0[2 * e], c0[2 * e + 1]);
                    turn(x0[4 + e], x1[4 + e], c1[2 * e], c1[2 * e + 1]);
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    turn(x0[e], x0[e + 1], c0[e], c0[e + 1]);
                    turn(x1[e], x1[e + 1], c1[e], c1[e + 1]);
                }
            }
        }
        store8<CT>(dst + e0, x0);
        store8<CT>(dst + e1, x1);
    } else {
        if (turns) turn(x0[0], x1[0], table[0], table[1]);
        dst[e0] = paged_from<CT>(x0[0]);
        dst[e1] = paged_from<CT>(x1[0]);
    }
}

template <typename XT, typename CT>
int launch_append(AppendArgs a, bool vec, cudaStream_t s) {
    a.units = (unsigned)(a.cache.d / (vec ? 16 : 2));
    a.per_tok = a.units * (unsigned)(a.n_head + 2 * a.cache.n_head_kv);
    const unsigned y = (a.per_tok + AP_NT - 1) / AP_NT;
    B200_REQUIRE(y <= 65535, "paged_append: too many heads for one launch");
    if (vec) return launch_pdl(paged_append_kernel<XT, CT, true>, dim3((unsigned)a.n_tok, y), dim3(AP_NT), 0, s, a);
    return launch_pdl(paged_append_kernel<XT, CT, false>, dim3((unsigned)a.n_tok, y), dim3(AP_NT), 0, s, a);
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" int b200_paged_append(const struct b200_paged_append_args *args, void *stream) {
    B200_REQUIRE(args != nullptr, "paged_append: null arguments");
    const b200_paged_append_args &g = *args;
    AppendArgs a;
    int rc = paged_check_cache(g.cache, "paged_append", &a.cache);
    if (rc != B200_STATUS_SUCCESS) return rc;
    const int xs = g.x_type == B200_TYPE_F32 ? 4 : 2;
    B200_REQUIRE(g.x_type == B200_TYPE_F32 || g.x_type == B200_TYPE_F16 || g.x_type == B200_TYPE_BF16, "paged_append: input type %d is not F32, F16 or BF16", g.x_type);
    B200_REQUIRE(g.n_tok >= 0 && g.n_tok <= 0x7fffffffLL, "paged_append: %lld tokens", (long long)g.n_tok);
    B200_REQUIRE(g.n_head >= 0 && g.n_head <= 65535, "paged_append: %d query heads", g.n_head);
    B200_REQUIRE(g.n_dims >= 0 && g.n_dims % 2 == 0 && g.n_dims <= g.cache.d, "paged_append: %d rotating channels of %lld", g.n_dims, (long long)g.cache.d);
    B200_REQUIRE(g.mode == 0 || g.mode == 2, "paged_append: mode %d is neither NORMAL (0) nor NEOX (2)", g.mode);
    if (g.n_tok == 0) return B200_STATUS_SUCCESS;
    B200_REQUIRE(g.pos != nullptr && g.k != nullptr && g.v != nullptr && (g.n_head == 0 || (g.q != nullptr && g.q_out != nullptr)), "paged_append: null operand");
    B200_REQUIRE(g.n_dims == 0 || (g.rope != nullptr && g.rope_rows > 0 && g.rope_ld >= g.n_dims), "paged_append: a rotation needs its table (rows of %d floats and more)", g.n_dims);
    const int64_t nb[8] = {g.k_nb1, g.k_nb2, g.v_nb1, g.v_nb2, g.n_head ? g.q_nb1 : 0, g.n_head ? g.q_nb2 : 0, g.n_head ? g.q_out_nb1 : 0, g.n_head ? g.q_out_nb2 : 0};
    uint64_t all = (uintptr_t)g.k | (uintptr_t)g.v;
    for (int i = 0; i < 6; i++) all |= (uint64_t)nb[i];
    if (g.n_head) all |= (uintptr_t)g.q;
    const uint64_t out = g.n_head ? (uintptr_t)g.q_out | (uint64_t)nb[6] | (uint64_t)nb[7] : 0;
    B200_REQUIRE(all % xs == 0 && out % 2 == 0, "paged_append: rows and strides must be aligned to their elements");
    const PagedOperand mem[10] = {{g.cache.k, "the cache's keys"}, {g.cache.v, "the cache's values"}, {g.cache.tables, "tables", 4}, {g.pos, "pos", 4}, {g.seq, "seq", 4},
                                  {g.k, "k"}, {g.v, "v"}, {g.n_head ? g.q : nullptr, "q"}, {g.n_head ? g.q_out : nullptr, "q_out"}, {g.n_dims ? g.rope : nullptr, "rope", 4}};
    if ((rc = paged_check_device(mem, 10, "paged_append")) != B200_STATUS_SUCCESS) return rc;
    a.n_tok = g.n_tok;
    a.pos = g.pos;
    a.seq = g.seq;
    a.x[0] = (const uint8_t *)g.q; a.x[1] = (const uint8_t *)g.k; a.x[2] = (const uint8_t *)g.v;
    a.x_nb1[0] = g.q_nb1; a.x_nb1[1] = g.k_nb1; a.x_nb1[2] = g.v_nb1;
    a.x_nb2[0] = g.q_nb2; a.x_nb2[1] = g.k_nb2; a.x_nb2[2] = g.v_nb2;
    a.q_out = (uint8_t *)g.q_out;
    a.q_out_nb1 = g.q_out_nb1;
    a.q_out_nb2 = g.q_out_nb2;
    a.rope = g.rope;
    a.rope_rows = g.rope_rows;
    a.rope_ld = g.rope_ld;
    a.n_head = g.n_head;
    a.n_dims = g.n_dims;
    a.neox = g.mode == 2;
    if ((rc = device_error_word(&a.err)) != B200_STATUS_SUCCESS) return rc;
    const bool vec = all % 16 == 0 && out % 16 == 0 && g.n_dims % 16 == 0 && (g.n_dims == 0 || (((uintptr_t)g.rope | (uint64_t)(g.rope_ld * 4)) & 15) == 0);
    const cudaStream_t s = (cudaStream_t)stream;
    const bool bf = g.cache.type == B200_TYPE_BF16;
    if (g.x_type == B200_TYPE_F32) return bf ? launch_append<float, __nv_bfloat16>(a, vec, s) : launch_append<float, __half>(a, vec, s);
    if (g.x_type == B200_TYPE_F16) return bf ? launch_append<__half, __nv_bfloat16>(a, vec, s) : launch_append<__half, __half>(a, vec, s);
    return bf ? launch_append<__nv_bfloat16, __nv_bfloat16>(a, vec, s) : launch_append<__nv_bfloat16, __half>(a, vec, s);
}
