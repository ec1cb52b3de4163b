// Attention of one row per sequence over a paged cache, positions that a group of sequences shares read once for the group (b200_prefix_attn).
//
//   o = sum_p w_p v_p / (sum_p w_p + exp(sink)),  w_p = exp(scale q k_p - max)          softmax in one pass, running maximum and sum in F32
//
// Rows that share positions share key heads too.  The shared part (prefix_attn_tcgen05.cu) takes the whole tiles of 128 positions that a sequence shares, all rows
// of a group and key head together; the own part (prefix_attn_own.cuh) what is left of a sequence, the query heads of a key head together.  Either cuts its positions
// into parts that leave (accumulator, maximum, sum) in the workspace; one launch has the CTAs of both, prefix_merge_kernel joins a row's parts, a warp each.
// Measured on the device, 32 heads on 8 of 128, BF16 (other where it says so), of the bytes that each cached position costs once at the copy rate:
//   a group of 64 rows, 32768 shared positions, up to 512 of a row's own     60.6 us, 252 MB: 4.2 TB/s, 0.64; 34.3 GFLOP: 566 TFLOP/s
//   4 groups of 16 rows, 4096 shared, up to 128 own                         24.6 us, 97 MB: 4.0 TB/s, 0.61
//   3 groups of 7 rows, 2047 shared, up to 333 own, F16, 16 key heads of 64 21 us, 49 MB: 2.3 TB/s, 0.36
//   a group of 8 rows, 1000 shared, up to 24 own, F16                       9.5 us, of which the second launch 4.6
// Above a few thousand positions the chain of a tile bounds it (scores, weights, products: prefix_attn_tcgen05.cu), below that beginnings and ends: 5 us of a CTA, the
// second launch.
#include <cmath>

#include "prefix_attn_own.cuh"

namespace b200 {

namespace {

constexpr int PX_MAX_PARTS = 64;   // of the shared positions, and of a row's own

// A warp a row: its parts joined, the sink, the division, the only rounding.  A row that does not come out finite is computed again from what it sees
// alone: products run over whole tiles, where a position that another row of the block sees meets this one with weight 0, and 0 * Inf is NaN.  So is one whose
// shared part met a page out of range, or scores that F32 holds whole steps of only (maximum NaN, sum 0).  A row whose shared part gave up waiting (both NaN) is not stored.
template <typename T, int D>
__global__ void __launch_bounds__(128) prefix_merge_kernel(const PrefixArgs a) {
    constexpr int C = D / 32, AT_ONCE = 8;   // channels of a lane: C lane ..; parts whose loads are under way together
    pdl_trigger();
    const int lane = threadIdx.x & 31;
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (row >= (int64_t)a.n_seq * a.n_head) return;
    const int s = (int)(row / a.n_head), h = (int)(row - (int64_t)s * a.n_head);
    const int parts = a.shared_parts + PX_WARPS * a.own_parts;
    const float2 *const ml = a.ml + row * parts;
    pdl_wait();
    const int n = a.lens[s];
    float sink = a.sinks ? a.sinks[h] * PX_LOG2E : -INFINITY;
    if (sink > 3.402823466e38f) sink = 3.402823466e38f;   // the largest sinks: no weight is left beside them
    // the first parts' outputs are asked for before it is known which of them there are
    const float *const acc = a.acc + row * parts * D + C * lane;
    auto load = [&](int i, float (&u)[C]) {
        if constexpr (C == 4) {
            const float4 y = i < parts ? *(const float4 *)(acc + (int64_t)i * D) : make_float4(0.f, 0.f, 0.f, 0.f);
            u[0] = y.x; u[1] = y.y; u[2] = y.z; u[3] = y.w;
        } else {
            const float2 y = i < parts ? *(const float2 *)(acc + (int64_t)i * D) : make_float2(0.f, 0.f);
            u[0] = y.x; u[1] = y.y;
        }
    };
    float u[AT_ONCE][C];
#pragma unroll
    for (int k = 0; k < AT_ONCE; k++) load(k, u[k]);
    float M = sink;
    bool again = false, lost = false;
    for (int i = lane; i < parts; i += 32) {
        const float2 x = ml[i];
        M = fmaxf(M, x.x);
        if (x.x != x.x) {
            if (x.y != x.y) lost = true;
            else again = true;
        }
    }
    if (__any_sync(0xffffffffu, lost)) return;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    float v[C], L = 0.0f;
#pragma unroll
    for (int c = 0; c < C; c++) v[c] = 0.0f;
    if (n > 0 && M > -INFINITY) {
        for (int base = 0; base < parts; base += 32) {
            const float2 x = base + lane < parts ? ml[base + lane] : make_float2(-INFINITY, 0.0f);
            const float f = x.x == -INFINITY ? 0.0f : pa_ex2(x.x - M);
            if (x.x != -INFINITY) L = fmaf(f, x.y, L);
            const unsigned in = __ballot_sync(0xffffffffu, x.x != -INFINITY);   // the others' outputs were not written: whatever is read there is not used
            for (int i = 0; i < min(parts - base, 32); i += AT_ONCE) {
                float w[AT_ONCE][C];
#pragma unroll
                for (int k = 0; k < AT_ONCE; k++)
#pragma unroll
                    for (int c = 0; c < C; c++) w[k][c] = in >> (i + k) & 1u ? u[k][c] : 0.0f;
#pragma unroll
                for (int k = 0; k < AT_ONCE; k++) load(base + i + AT_ONCE + k, u[k]);
#pragma unroll
                for (int k = 0; k < AT_ONCE; k++) {
                    const float g = __shfl_sync(0xffffffffu, f, i + k);
#pragma unroll
                    for (int c = 0; c < C; c++) v[c] = fmaf(g, w[k][c], v[c]);
                }
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
        if (sink > -INFINITY) L += pa_ex2(sink - M);
    }
    bool fine = !again && L < INFINITY;
#pragma unroll
    for (int c = 0; c < C; c++) fine &= fabsf(v[c]) < INFINITY;
    if (!__all_sync(0xffffffffu, fine)) {   // again, position by position
        const T *const q = (const T *)(a.q + (int64_t)s * a.q_nb1 + (int64_t)h * a.q_nb2) + C * lane;
        int first, end;
        prefix_group(a, s, &first, &end);
        const int shared = a.n_group ? a.shared[s] : 0;
        float m = sink;
        L = sink > -INFINITY ? 1.0f : 0.0f;
#pragma unroll
        for (int c = 0; c < C; c++) v[c] = 0.0f;
        for (int p = 0; p < n; p++) {
            const int64_t at = paged_row(a.cache, p < shared ? first : s, p);
            if (at < 0) {
                if ((p >> a.cache.page_log2) >= a.cache.table_ld) break;
                continue;
            }
            const int64_t mine = at + ((int64_t)(h / a.each) * D + C * lane) * 2;
            const T *const k = (const T *)(a.cache.k + mine), *const val = (const T *)(a.cache.v + mine);
            float dot = 0.0f;
#pragma unroll
            for (int c = 0; c < C; c++) dot = fmaf(paged_f32(q[c]), paged_f32(k[c]), dot);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
            dot *= a.scale_log2;
            if (!(dot < INFINITY)) {   // NaN, or a weight of exp(inf - inf)
                L = NAN;
                break;
            }
            if (dot == -INFINITY) continue;
            const float mn = fmaxf(m, dot), al = m == -INFINITY ? 0.0f : pa_ex2(m - mn), w = pa_ex2(dot - mn);
            m = mn;
            L = fmaf(L, al, w);
#pragma unroll
            for (int c = 0; c < C; c++) v[c] = fmaf(w, paged_f32(val[c]), v[c] * al);
        }
    }
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    T *const out = (T *)(a.dst + (int64_t)s * a.dst_nb1 + (int64_t)h * a.dst_nb2) + C * lane;
    if constexpr (C == 4) *(uint2 *)out = make_uint2(paged_pack<T>(v[0] * inv, v[1] * inv), paged_pack<T>(v[2] * inv, v[3] * inv));
    else *(uint32_t *)out = paged_pack<T>(v[0] * inv, v[1] * inv);
}

struct PrefixPlan {
    PrefixArgs a;
    int64_t rows;
    size_t ml_bytes, bytes;
};

// Into how many parts the positions are cut, and how the SMs are dealt out between the shared part (a CTA a part, one an SM, first) and the own part
// (CTAs that walk the items, three at a time): what takes least by a model of the launch.  Times in ns, measured with 8 key heads of 128 and of 64
// channels: a CTA of the shared part about 10000 and, a tile, 1850 with two blocks of rows, 6000 and 1250 with one (5000 and 850 with 64 channels); a unit of the own part
// 4000, 1500 an item and, a tile, 580 for each of the SM's units (an SM takes in 50 GB/s), at least 900; a row's partial output crosses L2 twice at about 5 bytes a
// picosecond.
struct PartsPlan {
    int64_t d, rows, shared_items, shared_tiles, own_items, own_tiles;
    bool two_blocks;
    int shared_parts, own_parts, own_ctas;
};
void plan_parts(PartsPlan *p, int64_t sms) {
    static const int counts[] = {1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11, 12, 14, 16, 18, 24, 32, 48, 64};
    static_assert(PX_MAX_PARTS == 64, "the most parts there are");
    const int64_t wide = p->d == 128, c_shared = p->two_blocks ? (wide ? 1850 : 1300) : (wide ? 1250 : 850), f_shared = p->two_blocks ? 10000 : wide ? 6000 : 5000;
    int64_t best = INT64_MAX;
    p->shared_parts = p->own_parts = p->own_ctas = 1;
    if (p->own_items == 0) return;
    for (int ns : counts) {
        if (ns > 1 && ns > p->shared_tiles) break;
        const int64_t n1 = p->shared_tiles ? p->shared_items * ns : 0, t1 = n1 ? f_shared + c_shared * ((p->shared_tiles + ns - 1) / ns) : 0;
        const int64_t waves = n1 / sms, left = sms - (n1 - waves * sms);   // SMs that the last wave leaves
        if (ns > 1 && n1 > 2 * sms) break;
        for (int no : counts) {
            if (no > 1 && no > p->own_tiles) break;
            const int64_t items = p->own_items * no, ctas = items < left ? items : left, units = items < 3 * ctas ? (items + ctas - 1) / ctas : 3;
            const int64_t each = (items + ctas * units - 1) / (ctas * units), tile = (wide ? 580 : 290) * units > 900 ? (wide ? 580 : 290) * units : 900;
            const int64_t t2 = 4000 + each * ((wide ? 1500 : 1000) + tile * ((p->own_tiles + no - 1) / no));
            const int64_t shared = (waves + (n1 > waves * sms)) * t1, own = waves * t1 + t2;
            const int64_t time = (shared > own ? shared : own) + p->rows * (PX_WARPS * no + (n1 ? ns : 0)) * p->d * 8 / 5000;
            if (time < best) {
                best = time;
                p->shared_parts = ns;
                p->own_parts = no;
                p->own_ctas = (int)ctas;
            }
        }
    }
}

int prefix_plan(const b200_prefix_attn_args &g, PrefixPlan *p) {
    PrefixArgs &a = p->a;
    int rc = paged_check_cache(g.cache, "prefix_attn", &a.cache);
    if (rc != B200_STATUS_SUCCESS) return rc;
    B200_REQUIRE(g.cache.d == 64 || g.cache.d == 128, "prefix_attn: heads of %lld channels (64 and 128 are served)", (long long)g.cache.d);
    B200_REQUIRE(g.n_seq >= 0 && g.n_seq <= g.cache.n_seq, "prefix_attn: %lld rows, the cache has tables for %lld sequences", (long long)g.n_seq, (long long)g.cache.n_seq);
    B200_REQUIRE(g.n_head > 0 && g.n_head <= 65535 && g.n_head % g.cache.n_head_kv == 0, "prefix_attn: %d heads over %lld key heads", g.n_head, (long long)g.cache.n_head_kv);
    B200_REQUIRE(g.n_group >= 0 && g.n_group <= g.n_seq, "prefix_attn: %d groups of %lld sequences", g.n_group, (long long)g.n_seq);
    B200_REQUIRE(g.max_len >= 0 && g.max_shared >= 0 && g.max_group >= 0, "prefix_attn: negative sizes");
    B200_REQUIRE(fabsf(g.scale * PX_LOG2E) < INFINITY, "prefix_attn: the scale %g, or log2(e) times it, is not finite", g.scale);
    a.n_seq = (int)g.n_seq;
    a.n_head = g.n_head;
    a.n_group = g.n_group;
    a.each = g.n_head / (int)g.cache.n_head_kv;
    const int64_t kv = g.cache.n_head_kv;
    p->rows = (int64_t)g.n_seq * g.n_head;
    // one sequence shares nothing, and less than a tile is no shared part
    const int64_t shared_tiles = g.n_group && g.max_group > 1 ? g.max_shared / PX_TILE : 0;
    a.served = shared_tiles > 0 ? (int)(g.max_group < g.n_seq ? g.max_group : g.n_seq) : 0;
    a.shared_blocks = 0;
    const int64_t shared_rows = (int64_t)a.served * a.each, block_rows = prefix_shared_rows(shared_rows);
    if (a.served) {
        B200_REQUIRE(shared_rows < (1 << 28), "prefix_attn: groups of %d sequences are too large", g.max_group);
        a.shared_blocks = (int)((shared_rows + block_rows - 1) / block_rows);
    }
    a.own_blocks = (a.each + PX_BM - 1) / PX_BM;
    PartsPlan pp;
    pp.d = g.cache.d;
    pp.rows = p->rows;
    pp.two_blocks = block_rows > 128;
    pp.shared_items = (int64_t)g.n_group * kv * a.shared_blocks;
    pp.shared_tiles = shared_tiles;
    pp.own_items = (int64_t)g.n_seq * kv * a.own_blocks;
    const int64_t own = g.max_len - shared_tiles * PX_TILE;
    pp.own_tiles = own > PX_BN ? (own + PX_BN - 1) / PX_BN : 1;
    plan_parts(&pp, sm_count());
    a.shared_parts = a.served ? pp.shared_parts : 0;
    a.own_parts = pp.own_parts;
    a.own_ctas = pp.own_ctas;
    B200_REQUIRE(pp.shared_items < (1 << 24) && pp.own_items < (1 << 23), "prefix_attn: too many rows for one launch");
    const int64_t slots = p->rows * (a.shared_parts + PX_WARPS * a.own_parts);
    p->ml_bytes = ((size_t)slots * sizeof(float2) + 255) & ~(size_t)255;
    p->bytes = p->ml_bytes + (size_t)slots * (size_t)g.cache.d * 4;
    return B200_STATUS_SUCCESS;
}

template <typename T, int D>
int launch_merge(const PrefixPlan &p, cudaStream_t s) {
    return launch_pdl(prefix_merge_kernel<T, D>, dim3((unsigned)((p.rows + 3) / 4)), dim3(128), 0, s, p.a);
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" {

size_t b200_prefix_attn_workspace_nbytes(const struct b200_prefix_attn_args *args) {
    PrefixPlan p;
    if (args == nullptr || prefix_plan(*args, &p) != B200_STATUS_SUCCESS) return 0;
    return p.bytes;
}

int b200_prefix_attn(const struct b200_prefix_attn_args *args, void *stream) {
    B200_REQUIRE(args != nullptr, "prefix_attn: null arguments");
    const b200_prefix_attn_args &g = *args;
    PrefixPlan p;
    int rc = prefix_plan(g, &p);
    if (rc != B200_STATUS_SUCCESS) return rc;
    if (g.n_seq == 0) return B200_STATUS_SUCCESS;
    B200_REQUIRE(g.q != nullptr && g.dst != nullptr && g.lens != nullptr && (g.n_group == 0 || (g.shared != nullptr && g.group_first != nullptr)), "prefix_attn: null operand");
    B200_REQUIRE((((uintptr_t)g.q | (uintptr_t)g.dst | (uint64_t)g.q_nb1 | (uint64_t)g.q_nb2 | (uint64_t)g.dst_nb1 | (uint64_t)g.dst_nb2) & 15) == 0,
                 "prefix_attn: q, dst and their strides must be multiples of 16 bytes");
    B200_REQUIRE(g.workspace != nullptr && (uintptr_t)g.workspace % 256 == 0 && g.workspace_nbytes >= p.bytes, "prefix_attn: a workspace of %zu bytes, 256-byte aligned, is needed (%zu given)", p.bytes,
                 g.workspace_nbytes);
    const PagedOperand mem[10] = {{g.cache.k, "the cache's keys"}, {g.cache.v, "the cache's values"}, {g.cache.tables, "tables", 4}, {g.q, "q"}, {g.dst, "dst"}, {g.lens, "lens", 4},
                                  {g.n_group ? g.shared : nullptr, "shared", 4}, {g.n_group ? g.group_first : nullptr, "group_first", 4}, {g.sinks, "sinks", 4}, {g.workspace, "the workspace"}};
    if ((rc = paged_check_device(mem, 10, "prefix_attn")) != B200_STATUS_SUCCESS) return rc;
    PrefixArgs &a = p.a;
    if ((rc = device_error_word(&a.err)) != B200_STATUS_SUCCESS) return rc;
    a.q = (const uint8_t *)g.q;
    a.dst = (uint8_t *)g.dst;
    a.q_nb1 = g.q_nb1;
    a.q_nb2 = g.q_nb2;
    a.dst_nb1 = g.dst_nb1;
    a.dst_nb2 = g.dst_nb2;
    a.lens = g.lens;
    a.shared = g.shared;
    a.group_first = g.group_first;
    a.sinks = g.sinks;
    a.scale_log2 = g.scale * PX_LOG2E;
    a.ml = (float2 *)g.workspace;
    a.acc = (float *)((uint8_t *)g.workspace + p.ml_bytes);
    const cudaStream_t s = (cudaStream_t)stream;
    if ((rc = launch_prefix_parts(a, g.cache.type, s)) != B200_STATUS_SUCCESS) return rc;
    if (g.cache.type == B200_TYPE_F16) return g.cache.d == 128 ? launch_merge<__half, 128>(p, s) : launch_merge<__half, 64>(p, s);
    return g.cache.d == 128 ? launch_merge<__nv_bfloat16, 128>(p, s) : launch_merge<__nv_bfloat16, 64>(p, s);
}

}  // extern "C"
