// Attention of one row per sequence over a paged cache, positions that a group of sequences shares read once for the group (b200_prefix_attn).
//
//   o = sum_p w_p v_p / (sum_p w_p + exp(sink)),  w_p = exp(scale q k_p - max)          softmax in one pass, running maximum and sum in F32
//
// Rows that share positions share key heads too: for the shared part a block of rows is (sequences of a group) x (query heads of a key head), for
// the others the query heads of a key head of one sequence.  Positions are cut into parts that leave (accumulator, maximum, sum) in the workspace;
// prefix_merge_kernel joins a row's parts, a warp each.
#include <cmath>

#include "paged.cuh"

namespace b200 {

namespace {

constexpr int PX_BM = 16, PX_BN = 64, PX_WARPS = 4, PX_NT = PX_WARPS * 32;
constexpr int PX_MAX_PARTS = 64;
constexpr float PX_LOG2E = 1.4426950408889634f;

struct PrefixArgs {
    PagedCache cache;
    const uint8_t *q;
    uint8_t *dst;
    int64_t q_nb1, q_nb2, dst_nb1, dst_nb2;
    const int32_t *lens, *shared, *group_first;
    const float *sinks;
    float scale_log2;
    int n_seq, n_head, n_group, each;         // each: query heads of a key head
    int shared_parts, own_parts, shared_blocks, own_blocks;   // parts of positions; blocks of PX_BM rows of a (group, key head), of a (sequence, key head)
    int64_t shared_units;                     // CTAs of the shared part
    float2 *ml;                               // [row][part]: maximum (log2 units), sum
    float *acc;                               // [row][part][d]
    int *err;
};

__device__ __forceinline__ uint32_t px_smem(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void px_cp16(void *dst, const void *src, bool there) {   // zeros where there is nothing to read
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(px_smem(dst)), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void px_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void px_wait_but_one() { asm volatile("cp.async.wait_group 1;" ::: "memory"); }
__device__ __forceinline__ void px_ldsm(uint32_t (&r)[4], const void *p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(px_smem(p)));
}
__device__ __forceinline__ void px_ldsm_t(uint32_t (&r)[4], const void *p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(px_smem(p)));
}
template <typename T>
__device__ __forceinline__ void px_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void px_mma<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void px_mma<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// two weights as the second product takes them; the sum takes them as they were (their rounding errors have no common sign)
template <typename T>
__device__ __forceinline__ uint32_t px_weights(float lo, float hi, float *sum) {
    *sum += lo + hi;
    return paged_pack<T>(lo, hi);
}

// A CTA: up to 16 rows against one part of their positions.  Warp w has positions 16 w .. + 15 of every tile of 64 (its own maximum and sum), the four are joined at the end.
template <typename T, int D>
__global__ void __launch_bounds__(PX_NT) prefix_rows_kernel(const PrefixArgs a) {
    constexpr int PITCH = D * 2 + 16, KS = D / 16, DB = D / 8, TILE = PX_BN * PITCH;
    extern __shared__ __align__(16) unsigned char smem[];   // K [2][PX_BN][PITCH], V the same
    __shared__ int64_t cell_of[2][PX_BN];                   // byte offset of a tile's positions, -1: not there
    __shared__ float wm[PX_WARPS][PX_BM], wl[PX_WARPS][PX_BM];
    pdl_trigger();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    // what this CTA is: rows r0 .. of `rows` (row x: sequence s0 + x / each, head hk * each + x % each), positions lo .. of the table of sequence `table`
    int64_t id = blockIdx.x;
    int hk, s0, x0, n_rows, table, part, parts;
    const bool shared_part = id < a.shared_units;
    pdl_wait();
    if (shared_part) {
        part = (int)(id % a.shared_parts); id /= a.shared_parts;
        parts = a.shared_parts;
        const int blk = (int)(id % a.shared_blocks); id /= a.shared_blocks;
        hk = (int)(id % a.cache.n_head_kv);
        const int g = (int)(id / a.cache.n_head_kv);
        int first = a.group_first[g], end = a.group_first[g + 1];
        if (first < 0 || end < first || end > a.n_seq || (g == 0 && first != 0) || (g == a.n_group - 1 && end != a.n_seq)) {
            if (tid == 0) atomicExch(a.err, ERR_PAGED);
            return;
        }
        s0 = table = first;
        x0 = blk * PX_BM;
        n_rows = (end - first) * a.each;
    } else {
        id -= a.shared_units;
        part = (int)(id % a.own_parts); id /= a.own_parts;
        parts = a.own_parts;
        x0 = (int)(id % a.own_blocks) * PX_BM; id /= a.own_blocks;
        hk = (int)(id % a.cache.n_head_kv);
        s0 = table = (int)(id / a.cache.n_head_kv);
        n_rows = a.each;
    }
    const int row_step = shared_part ? a.shared_blocks * PX_BM : a.own_blocks * PX_BM;
    const int capacity = (int)(a.cache.table_ld < (0x7fffff00 >> a.cache.page_log2) ? a.cache.table_ld << a.cache.page_log2 : 0x7fffff00);
    // more sequences in a group than the launch was shaped for: another turn
    for (; x0 < n_rows; x0 += row_step) {
        const int live = n_rows - x0 < PX_BM ? n_rows - x0 : PX_BM;
        // what the rows see: lo .. of all, up to end_a, end_b of this thread's rows lane / 4 and + 8
        auto end_of = [&](int x) {   // of row x
            const int s = s0 + x / a.each;
            const int n = a.lens[s];
            const int f = a.shared ? max(a.shared[s], 0) : 0;
            return shared_part ? min(n, f) : n;
        };
        const int r_a = lane >> 2, r_b = r_a + 8;
        int end_a = r_a < live ? end_of(x0 + r_a) : 0, end_b = r_b < live ? end_of(x0 + r_b) : 0;
        const int lo = shared_part || !a.shared ? 0 : max(a.shared[s0], 0);
        int end = max(end_a, end_b);
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) end = max(end, __shfl_xor_sync(0xffffffffu, end, o));
        if (end > capacity) {
            if (tid == 0) atomicExch(a.err, ERR_PAGED);
            end = capacity;
        }
        const int t_lo = lo / PX_BN, t_hi = end > lo ? (end + PX_BN - 1) / PX_BN : t_lo;
        const int per = (t_hi - t_lo + parts - 1) / parts;
        const int t0 = t_lo + part * per, t1 = min(t0 + per, t_hi), n_walk = max(t1 - t0, 0);
        const int64_t head = (int64_t)hk * D * 2;
        // a thread's pieces of a tile: 16 bytes tid % PIECES of rows tid / PIECES + RSTEP j
        constexpr int PIECES = D / 8, RSTEP = PX_NT / PIECES, PASSES = PX_BN / RSTEP;
        auto look_up = [&](int tile, int buf) {   // the threads of the first two warps: a position each
            if (tid < PX_BN) {
                const int p = tile * PX_BN + tid;
                int64_t at = -1;
                if (p >= lo && p < end) {
                    at = paged_row(a.cache, table, p);
                    if (at < 0) atomicExch(a.err, ERR_PAGED);
                }
                cell_of[buf][tid] = at;
            }
        };
        auto stage = [&](int buf) {
            unsigned char *const kd = smem + buf * TILE + (tid / PIECES) * PITCH + (tid % PIECES) * 16, *const vd = kd + 2 * TILE;
#pragma unroll
            for (int j = 0; j < PASSES; j++) {
                const int64_t at = cell_of[buf][tid / PIECES + j * RSTEP];
                const int64_t from = (at < 0 ? 0 : at + head) + (tid % PIECES) * 16;
                px_cp16(kd + j * RSTEP * PITCH, a.cache.k + from, at >= 0);
                px_cp16(vd + j * RSTEP * PITCH, a.cache.v + from, at >= 0);
            }
            px_commit();
        };
        __syncthreads();   // of the turn before
        if (n_walk > 0) look_up(t0, 0);
        if (n_walk > 1) look_up(t0 + 1, 1);
        __syncthreads();
        if (n_walk > 0) stage(0); else px_commit();
        if (n_walk > 1) stage(1); else px_commit();
        uint32_t qf[KS][4];
        {
            const int xa = x0 + (r_a < live ? r_a : 0), xb = x0 + (r_b < live ? r_b : 0), c0 = 4 * (lane & 3);
            const uint8_t *const qa = a.q + (int64_t)(s0 + xa / a.each) * a.q_nb1 + (int64_t)(hk * a.each + xa % a.each) * a.q_nb2 + c0;
            const uint8_t *const qb = a.q + (int64_t)(s0 + xb / a.each) * a.q_nb1 + (int64_t)(hk * a.each + xb % a.each) * a.q_nb2 + c0;
#pragma unroll
            for (int s = 0; s < KS; s++) {
                qf[s][0] = *(const uint32_t *)(qa + 32 * s);
                qf[s][1] = *(const uint32_t *)(qb + 32 * s);
                qf[s][2] = *(const uint32_t *)(qa + 32 * s + 16);
                qf[s][3] = *(const uint32_t *)(qb + 32 * s + 16);
            }
        }
        float o[DB][4];
#pragma unroll
        for (int j = 0; j < DB; j++) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f;
        float m_a = -INFINITY, m_b = -INFINITY, l_a = 0.0f, l_b = 0.0f;
        const int k_row = (lane & 7) + ((lane >> 4) << 3), k_col = ((lane >> 3) & 1) * 16;
        const int v_row = (lane & 7) + (((lane >> 3) & 1) << 3), v_col = (lane >> 4) * 16;
        const int pw = 16 * warp;
        for (int it = 0; it < n_walk; it++) {
            const int buf = it & 1;
            px_wait_but_one();
            __syncthreads();
            const unsigned char *const kt = smem + buf * TILE, *const vt = kt + 2 * TILE;
            float s[2][4];
#pragma unroll
            for (int n = 0; n < 2; n++) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f;
#pragma unroll
            for (int st = 0; st < KS; st++) {
                uint32_t b[4];
                px_ldsm(b, kt + (pw + k_row) * PITCH + st * 32 + k_col);
                px_mma<T>(s[0], qf[st], b[0], b[1]);
                px_mma<T>(s[1], qf[st], b[2], b[3]);
            }
            float mx_a = -INFINITY, mx_b = -INFINITY;
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const int in = pw + n * 8 + 2 * (lane & 3) + e, p = (t0 + it) * PX_BN + in;
                    const bool there = cell_of[buf][in] >= 0;
                    s[n][e] = there && p < end_a ? s[n][e] * a.scale_log2 : -INFINITY;
                    s[n][2 + e] = there && p < end_b ? s[n][2 + e] * a.scale_log2 : -INFINITY;
                    mx_a = fmaxf(mx_a, s[n][e]);
                    mx_b = fmaxf(mx_b, s[n][2 + e]);
                }
            mx_a = fmaxf(mx_a, __shfl_xor_sync(0xffffffffu, mx_a, 1)); mx_a = fmaxf(mx_a, __shfl_xor_sync(0xffffffffu, mx_a, 2));
            mx_b = fmaxf(mx_b, __shfl_xor_sync(0xffffffffu, mx_b, 1)); mx_b = fmaxf(mx_b, __shfl_xor_sync(0xffffffffu, mx_b, 2));
            const float mn_a = fmaxf(m_a, mx_a), mn_b = fmaxf(m_b, mx_b);
            const float al_a = m_a == -INFINITY ? 0.0f : exp2f(m_a - mn_a), al_b = m_b == -INFINITY ? 0.0f : exp2f(m_b - mn_b);
            const float sub_a = mn_a == -INFINITY ? 0.0f : mn_a, sub_b = mn_b == -INFINITY ? 0.0f : mn_b;
            m_a = mn_a; m_b = mn_b;
            float ps_a = 0.0f, ps_b = 0.0f;
            uint32_t pf[4];
            pf[0] = px_weights<T>(exp2f(s[0][0] - sub_a), exp2f(s[0][1] - sub_a), &ps_a);
            pf[1] = px_weights<T>(exp2f(s[0][2] - sub_b), exp2f(s[0][3] - sub_b), &ps_b);
            pf[2] = px_weights<T>(exp2f(s[1][0] - sub_a), exp2f(s[1][1] - sub_a), &ps_a);
            pf[3] = px_weights<T>(exp2f(s[1][2] - sub_b), exp2f(s[1][3] - sub_b), &ps_b);
            l_a = fmaf(l_a, al_a, ps_a);
            l_b = fmaf(l_b, al_b, ps_b);
#pragma unroll
            for (int j = 0; j < DB; j++) {
                o[j][0] *= al_a; o[j][1] *= al_a; o[j][2] *= al_b; o[j][3] *= al_b;
            }
#pragma unroll
            for (int e = 0; e < DB; e += 2) {
                uint32_t b[4];
                px_ldsm_t(b, vt + (pw + v_row) * PITCH + e * 16 + v_col);
                px_mma<T>(o[e], pf, b[0], b[1]);
                px_mma<T>(o[e + 1], pf, b[2], b[3]);
            }
            __syncthreads();   // everyone is done with this buffer
            if (it + 2 < n_walk) look_up(t0 + it + 2, buf);
            __syncthreads();
            if (it + 2 < n_walk) stage(buf); else px_commit();
        }
        // the four warps joined
        l_a += __shfl_xor_sync(0xffffffffu, l_a, 1); l_a += __shfl_xor_sync(0xffffffffu, l_a, 2);
        l_b += __shfl_xor_sync(0xffffffffu, l_b, 1); l_b += __shfl_xor_sync(0xffffffffu, l_b, 2);
        if (l_a != l_a) m_a = fmaxf(m_a, 0.0f);   // a NaN score is no maximum, but the row has seen it
        if (l_b != l_b) m_b = fmaxf(m_b, 0.0f);
        float *const oacc = (float *)smem;   // [PX_WARPS][PX_BM][D]; every copy has landed
        if ((lane & 3) == 0) {
            wm[warp][r_a] = m_a; wl[warp][r_a] = l_a;
            wm[warp][r_b] = m_b; wl[warp][r_b] = l_b;
        }
#pragma unroll
        for (int j = 0; j < DB; j++) {
            *(float2 *)(oacc + (warp * PX_BM + r_a) * D + j * 8 + 2 * (lane & 3)) = make_float2(o[j][0], o[j][1]);
            *(float2 *)(oacc + (warp * PX_BM + r_b) * D + j * 8 + 2 * (lane & 3)) = make_float2(o[j][2], o[j][3]);
        }
        __syncthreads();
        const int all_parts = a.shared_parts + a.own_parts, my_part = shared_part ? part : a.shared_parts + part;
        for (int i = tid; i < live * (D / 4); i += PX_NT) {
            const int r = i / (D / 4), c = 4 * (i % (D / 4)), x = x0 + r;
            float M = -INFINITY;
#pragma unroll
            for (int w = 0; w < PX_WARPS; w++) M = fmaxf(M, wm[w][r]);
            const int64_t out = ((int64_t)(s0 + x / a.each) * a.n_head + hk * a.each + x % a.each) * all_parts + my_part;
            if (M == -INFINITY) {
                if (c == 0) a.ml[out] = make_float2(-INFINITY, 0.0f);
                continue;
            }
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            float L = 0.0f;
#pragma unroll
            for (int w = 0; w < PX_WARPS; w++) {
                const float f = wm[w][r] == -INFINITY ? 0.0f : exp2f(wm[w][r] - M);
                const float4 u = *(const float4 *)(oacc + (w * PX_BM + r) * D + c);
                v.x = fmaf(f, u.x, v.x); v.y = fmaf(f, u.y, v.y); v.z = fmaf(f, u.z, v.z); v.w = fmaf(f, u.w, v.w);
                L = fmaf(f, wl[w][r], L);
            }
            *(float4 *)(a.acc + out * D + c) = v;
            if (c == 0) a.ml[out] = make_float2(M, L);
        }
    }
}

// A warp a row: its parts joined, the sink, the division, the only rounding.  A row that does not come out finite is computed again from what it sees
// alone: products run over whole tiles, where a position that another row of the block sees meets this one with weight 0, and 0 * Inf is NaN.
template <typename T, int D>
__global__ void __launch_bounds__(128) prefix_merge_kernel(const PrefixArgs a) {
    constexpr int C = D / 32;   // channels of a lane: C lane ..
    pdl_trigger();
    const int lane = threadIdx.x & 31;
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (row >= (int64_t)a.n_seq * a.n_head) return;
    const int s = (int)(row / a.n_head), h = (int)(row - (int64_t)s * a.n_head);
    const int parts = a.shared_parts + a.own_parts;
    pdl_wait();
    float M = -INFINITY;
    const float sink = a.sinks ? a.sinks[h] * PX_LOG2E : -INFINITY;
    for (int i = lane; i < parts; i += 32) M = fmaxf(M, a.ml[row * parts + i].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    M = fmaxf(M, sink);
    float v[C], L = 0.0f;
#pragma unroll
    for (int c = 0; c < C; c++) v[c] = 0.0f;
    const int n = a.lens[s];
    if (n > 0 && M > -INFINITY) {
        for (int i = 0; i < parts; i++) {
            const float2 ml = a.ml[row * parts + i];
            if (ml.x == -INFINITY) continue;
            const float f = exp2f(ml.x - M);
            const float *const acc = a.acc + (row * parts + i) * D + C * lane;
            L = fmaf(f, ml.y, L);
#pragma unroll
            for (int c = 0; c < C; c++) v[c] = fmaf(f, acc[c], v[c]);
        }
        if (sink > -INFINITY) L += exp2f(sink - M);
    }
    bool fine = true;
#pragma unroll
    for (int c = 0; c < C; c++) fine &= fabsf(v[c]) < INFINITY;
    if (!__all_sync(0xffffffffu, fine && L < INFINITY)) {   // again, position by position
        const T *const q = (const T *)(a.q + (int64_t)s * a.q_nb1 + (int64_t)h * a.q_nb2) + C * lane;
        int g = 0;
        while (g + 1 < a.n_group && a.group_first[g + 1] <= s) g++;
        int first = a.n_group ? a.group_first[g] : s;
        if (first < 0 || first > s) first = s;   // groups that the other kernel has reported
        const int shared = a.shared ? max(a.shared[s], 0) : 0;
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
            if (!(dot < INFINITY)) {
                L = NAN;
                break;
            }
            if (dot == -INFINITY) continue;
            const float mn = fmaxf(m, dot), al = m == -INFINITY ? 0.0f : exp2f(m - mn), w = exp2f(dot - mn);
            m = mn;
            L = fmaf(L, al, w);
#pragma unroll
            for (int c = 0; c < C; c++) v[c] = fmaf(w, paged_f32(val[c]), v[c] * al);
        }
    }
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    T *const out = (T *)(a.dst + (int64_t)s * a.dst_nb1 + (int64_t)h * a.dst_nb2) + C * lane;
#pragma unroll
    for (int c = 0; c < C; c += 2) *(uint32_t *)(out + c) = paged_pack<T>(v[c] * inv, v[c + 1] * inv);
}

struct PrefixPlan {
    PrefixArgs a;
    int64_t rows;
    size_t ml_bytes, bytes;
};

int prefix_plan(const b200_prefix_attn_args &g, PrefixPlan *p) {
    PrefixArgs &a = p->a;
    int rc = paged_check_cache(g.cache, "prefix_attn", &a.cache);
    if (rc != B200_STATUS_SUCCESS) return rc;
    B200_REQUIRE(g.cache.d == 64 || g.cache.d == 128, "prefix_attn: heads of %lld channels (64 and 128 are served)", (long long)g.cache.d);
    B200_REQUIRE(g.n_seq >= 0 && g.n_seq <= g.cache.n_seq, "prefix_attn: %lld rows, the cache has tables for %lld sequences", (long long)g.n_seq, (long long)g.cache.n_seq);
    B200_REQUIRE(g.n_head > 0 && g.n_head <= 65535 && g.n_head % g.cache.n_head_kv == 0, "prefix_attn: %d heads over %lld key heads", g.n_head, (long long)g.cache.n_head_kv);
    B200_REQUIRE(g.n_group >= 0 && g.n_group <= g.n_seq, "prefix_attn: %d groups of %lld sequences", g.n_group, (long long)g.n_seq);
    B200_REQUIRE(g.max_len >= 0 && g.max_shared >= 0 && g.max_group >= 0, "prefix_attn: negative sizes");
    B200_REQUIRE(fabsf(g.scale) < INFINITY, "prefix_attn: the scale is not finite");
    a.n_seq = (int)g.n_seq;
    a.n_head = g.n_head;
    a.n_group = g.n_group;
    a.each = g.n_head / (int)g.cache.n_head_kv;
    const int64_t per = g.max_group > 0 ? g.max_group : 1;
    a.shared_blocks = (int)((per * a.each + PX_BM - 1) / PX_BM);
    a.own_blocks = (a.each + PX_BM - 1) / PX_BM;
    // parts so that some four CTAs an SM have about the same number of tiles
    const int64_t kv = g.cache.n_head_kv;
    const int64_t shared_tiles = g.n_group ? (g.max_shared + PX_BN - 1) / PX_BN : 0, own_tiles = (g.max_len > (g.n_group ? g.max_shared : 0) ? g.max_len - (g.n_group ? g.max_shared : 0) + PX_BN - 1 : PX_BN) / PX_BN;
    const int64_t shared_ctas = (int64_t)g.n_group * kv * a.shared_blocks, own_ctas = (int64_t)g.n_seq * kv * a.own_blocks;
    const int64_t work = shared_ctas * shared_tiles + own_ctas * own_tiles, each = work / (4 * sm_count()) + 1;   // tiles a CTA
    auto parts = [&](int64_t tiles) {
        int64_t n = (tiles + each - 1) / each;
        return (int)(n < 1 ? 1 : n > PX_MAX_PARTS ? PX_MAX_PARTS : n);
    };
    a.shared_parts = g.n_group ? parts(shared_tiles) : 0;
    a.own_parts = parts(own_tiles);
    a.shared_units = shared_ctas * a.shared_parts;
    B200_REQUIRE(a.shared_units + own_ctas * a.own_parts < 0x7fffffffLL, "prefix_attn: too many rows for one launch");
    p->rows = (int64_t)g.n_seq * g.n_head;
    const int64_t slots = p->rows * (a.shared_parts + a.own_parts);
    p->ml_bytes = ((size_t)slots * sizeof(float2) + 255) & ~(size_t)255;
    p->bytes = p->ml_bytes + (size_t)slots * (size_t)g.cache.d * 4;
    return B200_STATUS_SUCCESS;
}

template <typename T, int D>
int launch_prefix(const PrefixPlan &p, cudaStream_t s) {
    const PrefixArgs &a = p.a;
    constexpr int SMEM = 4 * PX_BN * (D * 2 + 16);
    const int64_t ctas = a.shared_units + (int64_t)a.n_seq * a.cache.n_head_kv * a.own_blocks * a.own_parts;
    B200_CUDA(cudaFuncSetAttribute(prefix_rows_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM));
    const int rc = launch_pdl(prefix_rows_kernel<T, D>, dim3((unsigned)ctas), dim3(PX_NT), SMEM, s, a);
    if (rc != B200_STATUS_SUCCESS) return rc;
    return launch_pdl(prefix_merge_kernel<T, D>, dim3((unsigned)((p.rows + 3) / 4)), dim3(128), 0, s, a);
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
    const void *mem[4] = {g.cache.k, g.q, g.dst, g.workspace};
    const char *names[4] = {"the cache", "q", "dst", "the workspace"};
    for (int i = 0; i < 4; i++)
        if ((rc = paged_check_device(mem[i], "prefix_attn", names[i])) != B200_STATUS_SUCCESS) return rc;
    PrefixArgs &a = p.a;
    if ((rc = device_error_word(&a.err)) != B200_STATUS_SUCCESS) return rc;
    a.q = (const uint8_t *)g.q;
    a.dst = (uint8_t *)g.dst;
    a.q_nb1 = g.q_nb1;
    a.q_nb2 = g.q_nb2;
    a.dst_nb1 = g.dst_nb1;
    a.dst_nb2 = g.dst_nb2;
    a.lens = g.lens;
    a.shared = g.n_group ? g.shared : nullptr;
    a.group_first = g.group_first;
    a.sinks = g.sinks;
    a.scale_log2 = g.scale * PX_LOG2E;
    a.ml = (float2 *)g.workspace;
    a.acc = (float *)((uint8_t *)g.workspace + p.ml_bytes);
    const cudaStream_t s = (cudaStream_t)stream;
    if (g.cache.type == B200_TYPE_F16) return g.cache.d == 128 ? launch_prefix<__half, 128>(p, s) : launch_prefix<__half, 64>(p, s);
    return g.cache.d == 128 ? launch_prefix<__nv_bfloat16, 128>(p, s) : launch_prefix<__nv_bfloat16, 64>(p, s);
}

}  // extern "C"
