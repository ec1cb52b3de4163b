// Attention of one row per sequence over a paged cache, positions that a group of sequences shares read once for the group (b200_prefix_attn).
//
//   o = sum_p w_p v_p / (sum_p w_p + exp(sink)),  w_p = exp(scale q k_p - max)          softmax in one pass, running maximum and sum in F32
//
// Rows that share positions share key heads too.  prefix_shared_kernel (prefix_attn_tcgen05.cu) takes the whole tiles of 128 positions that a sequence shares, all rows
// of a group and key head together; prefix_own_kernel here takes what is left of a sequence, the query heads of a key head together.  Either cuts its positions
// into parts that leave (accumulator, maximum, sum) in the workspace; prefix_merge_kernel joins a row's parts, a warp each.
#include <cmath>

#include "attn_tcgen05.cuh"
#include "prefix_attn.cuh"

namespace b200 {

namespace {

constexpr int PX_BM = 16, PX_BN = 64, PX_WARPS = 4, PX_NT = PX_WARPS * 32;
constexpr int PX_MAX_PARTS = 64;   // of the shared positions, and of a row's own
template <int D>
constexpr int PX_STAGES = D == 128 ? 2 : 4;   // 64 KB of tiles under way or at work: a CTA then fits an SM beside one of the shared part's (161 KB, and 128 registers a thread each)

__device__ __forceinline__ uint32_t px_smem(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void px_cp16(void *dst, const void *src, bool there) {   // zeros where there is nothing to read
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(px_smem(dst)), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void px_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void px_wait_but() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
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

// The group that sequence s stands in, by a whole warp: its first sequence, or s itself where no group holds it (that is reported).  *served: whether
// the shared part has computed its whole shared tiles.  A search that looks at 32 places at a time
__device__ __forceinline__ int prefix_first(const PrefixArgs &a, int s, bool *served) {
    *served = false;
    if (a.n_group == 0) return s;
    const int lane = threadIdx.x & 31;
    int g = 0, n = a.n_group;
    while (n > 1) {
        const int step = (n + 31) / 32, at = lane * step;
        const bool behind = at < n && a.group_first[g + at] <= s;
        const int last = 31 - __clz(__ballot_sync(0xffffffffu, behind) | 1u);
        g += last * step;
        n = min(step, n - last * step);
    }
    const int first = a.group_first[g], end = a.group_first[g + 1];
    if (!prefix_group_fits(first, end, a.n_seq) || s < first || s >= end) {
        if (lane == 0) atomicExch(a.err, ERR_PAGED);
        return s;
    }
    *served = s - first < a.served;
    return first;
}

// A CTA: up to 16 query heads of a sequence and key head against one part of its positions behind those that the shared part covers.  Warp w has positions
// 16 w .. + 15 of every tile of 64 (its own maximum and sum), the four are joined at the end.  Positions that the sequence does not see are zeros in
// shared memory, whatever the page holds.
template <typename T, int D>
__global__ void __launch_bounds__(PX_NT, 4) prefix_own_kernel(const PrefixArgs a, bool after_shared) {
    constexpr int ROW = D * 2, KS = D / 16, DB = D / 8, TILE = PX_BN * ROW, NST = PX_STAGES<D>;
    extern __shared__ __align__(128) unsigned char smem[];   // K [NST][PX_BN][ROW], V the same; 16-byte piece u of row r lies at u ^ (r % 8)
    __shared__ int64_t cell_of[NST][PX_BN];                  // byte offset of a tile's positions, -1: not there
    __shared__ float wm[PX_WARPS][PX_BM], wl[PX_WARPS][PX_BM];
    pdl_trigger();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int64_t id = blockIdx.x;
    const int part = (int)(id % a.own_parts); id /= a.own_parts;
    const int x0 = (int)(id % a.own_blocks) * PX_BM; id /= a.own_blocks;
    const int hk = (int)(id % a.cache.n_head_kv), s = (int)(id / a.cache.n_head_kv);
    if (!after_shared) pdl_wait();   // else the kernel in front has waited for what was before it, and this one reads nothing of its
    const int rows = min(a.each - x0, PX_BM);
    const int len = a.lens[s], shared = a.n_group ? a.shared[s] : 0;
    bool served;
    const int first = prefix_first(a, s, &served);
    const int capacity = (int)(a.cache.table_ld < (0x7fffff00 >> a.cache.page_log2) ? a.cache.table_ld << a.cache.page_log2 : 0x7fffff00);
    if (len > capacity && tid == 0) atomicExch(a.err, ERR_PAGED);
    const int end = min(len, capacity), lo = served ? min(max(min(len, shared), 0), capacity) / PX_TILE * PX_TILE : 0;
    const int tiles = end > lo ? (end - lo + PX_BN - 1) / PX_BN : 0, per = (tiles + a.own_parts - 1) / a.own_parts;
    const int n_walk = max(min(per, tiles - part * per), 0), p0 = lo + part * per * PX_BN;
    const int64_t head = (int64_t)hk * D * 2;
    // a thread's pieces of a tile: 16 bytes tid % PIECES of rows tid / PIECES + RSTEP j
    constexpr int PIECES = D / 8, RSTEP = PX_NT / PIECES, PASSES = PX_BN / RSTEP;
    static_assert(RSTEP % 8 == 0, "a thread's rows have one place for their piece");
    auto look_up = [&](int tile) -> int64_t {   // the threads of the first two warps: a position each
        const int p = p0 + tile * PX_BN + tid;
        if (tid >= PX_BN || tile >= n_walk || p >= end) return -1;
        const int64_t at = paged_row(a.cache, p < shared ? first : s, p);
        if (at < 0) atomicExch(a.err, ERR_PAGED);
        return at;
    };
    auto stage = [&](int buf) {
        unsigned char *const kd = smem + buf * TILE + (tid / PIECES) * ROW + (((tid % PIECES) ^ (tid / PIECES & 7)) << 4), *const vd = kd + NST * TILE;
#pragma unroll
        for (int j = 0; j < PASSES; j++) {
            const int64_t at = cell_of[buf][tid / PIECES + j * RSTEP];
            const int64_t from = (at < 0 ? 0 : at + head) + (tid % PIECES) * 16;
            px_cp16(kd + j * RSTEP * ROW, a.cache.k + from, at >= 0);
            px_cp16(vd + j * RSTEP * ROW, a.cache.v + from, at >= 0);
        }
    };
    {
        int64_t c[NST];
#pragma unroll
        for (int i = 0; i < NST; i++) c[i] = look_up(i);
        if (tid < PX_BN) {
#pragma unroll
            for (int i = 0; i < NST; i++) cell_of[i][tid] = c[i];
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NST; i++) {
        if (i < n_walk) stage(i);
        px_commit();
    }
    const int r_a = lane >> 2, r_b = r_a + 8;   // this thread's rows
    uint32_t qf[KS][4];
    {
        const int xa = x0 + (r_a < rows ? r_a : 0), xb = x0 + (r_b < rows ? r_b : 0), c0 = 4 * (lane & 3);
        const uint8_t *const qs = a.q + (int64_t)s * a.q_nb1 + c0;
        const uint8_t *const qa = qs + (int64_t)(hk * a.each + xa) * a.q_nb2, *const qb = qs + (int64_t)(hk * a.each + xb) * a.q_nb2;
#pragma unroll
        for (int k = 0; k < KS; k++) {
            qf[k][0] = *(const uint32_t *)(qa + 32 * k);
            qf[k][1] = *(const uint32_t *)(qb + 32 * k);
            qf[k][2] = *(const uint32_t *)(qa + 32 * k + 16);
            qf[k][3] = *(const uint32_t *)(qb + 32 * k + 16);
        }
    }
    float o[DB][4];
#pragma unroll
    for (int j = 0; j < DB; j++) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f;
    float m_a = -INFINITY, m_b = -INFINITY, l_a = 0.0f, l_b = 0.0f;
    const int k_row = (lane & 7) + ((lane >> 4) << 3), k_piece = (lane >> 3) & 1;
    const int v_row = (lane & 7) + (((lane >> 3) & 1) << 3), v_piece = lane >> 4, turn = lane & 7;   // rows' places modulo 8
    const int pw = 16 * warp;
    for (int it = 0; it < n_walk; it++) {
        const int buf = it % NST;
        const int64_t next = look_up(it + NST);
        px_wait_but<NST - 1>();
        __syncthreads();
        const unsigned char *const kt = smem + buf * TILE + (pw + k_row) * ROW, *const vt = smem + (NST + buf) * TILE + (pw + v_row) * ROW;
        float sc[2][4];
#pragma unroll
        for (int n = 0; n < 2; n++) sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.0f;
#pragma unroll
        for (int st = 0; st < KS; st++) {
            uint32_t b[4];
            px_ldsm(b, kt + (((2 * st + k_piece) ^ turn) << 4));
            px_mma<T>(sc[0], qf[st], b[0], b[1]);
            px_mma<T>(sc[1], qf[st], b[2], b[3]);
        }
        float mx_a = -INFINITY, mx_b = -INFINITY;
#pragma unroll
        for (int n = 0; n < 2; n++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const bool there = cell_of[buf][pw + n * 8 + 2 * (lane & 3) + e] >= 0;
                sc[n][e] = there ? sc[n][e] * a.scale_log2 : -INFINITY;
                sc[n][2 + e] = there ? sc[n][2 + e] * a.scale_log2 : -INFINITY;
                mx_a = fmaxf(mx_a, sc[n][e]);
                mx_b = fmaxf(mx_b, sc[n][2 + e]);
            }
        mx_a = fmaxf(mx_a, __shfl_xor_sync(0xffffffffu, mx_a, 1)); mx_a = fmaxf(mx_a, __shfl_xor_sync(0xffffffffu, mx_a, 2));
        mx_b = fmaxf(mx_b, __shfl_xor_sync(0xffffffffu, mx_b, 1)); mx_b = fmaxf(mx_b, __shfl_xor_sync(0xffffffffu, mx_b, 2));
        const float mn_a = fmaxf(m_a, mx_a), mn_b = fmaxf(m_b, mx_b);
        const float al_a = m_a == -INFINITY ? 0.0f : pa_ex2(m_a - mn_a), al_b = m_b == -INFINITY ? 0.0f : pa_ex2(m_b - mn_b);
        const float sub_a = mn_a == -INFINITY ? 0.0f : mn_a, sub_b = mn_b == -INFINITY ? 0.0f : mn_b;
        const bool same = m_a == mn_a && m_b == mn_b;
        m_a = mn_a; m_b = mn_b;
        float ps_a = 0.0f, ps_b = 0.0f;
        uint32_t pf[4];
        pf[0] = px_weights<T>(pa_ex2(sc[0][0] - sub_a), pa_ex2(sc[0][1] - sub_a), &ps_a);
        pf[1] = px_weights<T>(pa_ex2(sc[0][2] - sub_b), pa_ex2(sc[0][3] - sub_b), &ps_b);
        pf[2] = px_weights<T>(pa_ex2(sc[1][0] - sub_a), pa_ex2(sc[1][1] - sub_a), &ps_a);
        pf[3] = px_weights<T>(pa_ex2(sc[1][2] - sub_b), pa_ex2(sc[1][3] - sub_b), &ps_b);
        l_a = fmaf(l_a, al_a, ps_a);
        l_b = fmaf(l_b, al_b, ps_b);
        if (!__all_sync(0xffffffffu, same)) {
#pragma unroll
            for (int j = 0; j < DB; j++) {
                o[j][0] *= al_a; o[j][1] *= al_a; o[j][2] *= al_b; o[j][3] *= al_b;
            }
        }
#pragma unroll
        for (int e = 0; e < DB; e += 2) {
            uint32_t b[4];
            px_ldsm_t(b, vt + (((e + v_piece) ^ turn) << 4));
            px_mma<T>(o[e], pf, b[0], b[1]);
            px_mma<T>(o[e + 1], pf, b[2], b[3]);
        }
        __syncthreads();   // everyone is done with this buffer
        if (tid < PX_BN) cell_of[buf][tid] = next;
        __syncthreads();
        if (it + NST < n_walk) stage(buf);
        px_commit();
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
    const int all_parts = a.shared_parts + a.own_parts;
    for (int i = tid; i < rows * (D / 4); i += PX_NT) {
        const int r = i / (D / 4), c = 4 * (i % (D / 4));
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < PX_WARPS; w++) M = fmaxf(M, wm[w][r]);
        const int64_t row = (int64_t)s * a.n_head + hk * a.each + x0 + r, out = row * all_parts + a.shared_parts + part;
        if (c == 0 && part == 0 && !served)
            for (int q = 0; q < a.shared_parts; q++) a.ml[row * all_parts + q] = make_float2(-INFINITY, 0.0f);   // nobody else writes them
        if (M == -INFINITY) {
            if (c == 0) a.ml[out] = make_float2(-INFINITY, 0.0f);
            continue;
        }
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        float L = 0.0f;
#pragma unroll
        for (int w = 0; w < PX_WARPS; w++) {
            const float f = wm[w][r] == -INFINITY ? 0.0f : pa_ex2(wm[w][r] - M);
            const float4 u = *(const float4 *)(oacc + (w * PX_BM + r) * D + c);
            v.x = fmaf(f, u.x, v.x); v.y = fmaf(f, u.y, v.y); v.z = fmaf(f, u.z, v.z); v.w = fmaf(f, u.w, v.w);
            L = fmaf(f, wl[w][r], L);
        }
        *(float4 *)(a.acc + out * D + c) = v;
        if (c == 0) a.ml[out] = make_float2(M, L);
    }
    // the merge waits for this kernel alone: it must not be over before the shared part is
    if (after_shared && blockIdx.x == 0) pdl_wait();
}

// A warp a row: its parts joined, the sink, the division, the only rounding.  A row that does not come out finite is computed again from what it sees
// alone: products run over whole tiles, where a position that another row of the block sees meets this one with weight 0, and 0 * Inf is NaN.  So is one whose
// shared part met a page out of range (maximum NaN, sum 0).  A row whose shared part gave up waiting (both NaN) is not stored.
template <typename T, int D>
__global__ void __launch_bounds__(128) prefix_merge_kernel(const PrefixArgs a) {
    constexpr int C = D / 32, AT_ONCE = 4;   // channels of a lane: C lane ..; parts whose loads are under way together
    pdl_trigger();
    const int lane = threadIdx.x & 31;
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (row >= (int64_t)a.n_seq * a.n_head) return;
    const int s = (int)(row / a.n_head), h = (int)(row - (int64_t)s * a.n_head);
    const int parts = a.shared_parts + a.own_parts;
    const float2 *const ml = a.ml + row * parts;
    pdl_wait();
    const int n = a.lens[s];
    const float sink = a.sinks ? a.sinks[h] * PX_LOG2E : -INFINITY;
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
            const unsigned in = __ballot_sync(0xffffffffu, x.x != -INFINITY);
            for (int i = 0; i < min(parts - base, 32); i += AT_ONCE) {
                float w[AT_ONCE], u[AT_ONCE][C];
#pragma unroll
                for (int k = 0; k < AT_ONCE; k++) {
                    w[k] = __shfl_sync(0xffffffffu, f, (i + k) & 31);
                    const float *const acc = a.acc + (row * parts + base + i + k) * D + C * lane;
                    const bool there = i + k < 32 && (in >> (i + k) & 1u);
                    if constexpr (C == 4) {
                        const float4 y = there ? *(const float4 *)acc : make_float4(0.f, 0.f, 0.f, 0.f);
                        u[k][0] = y.x; u[k][1] = y.y; u[k][2] = y.z; u[k][3] = y.w;
                    } else {
                        const float2 y = there ? *(const float2 *)acc : make_float2(0.f, 0.f);
                        u[k][0] = y.x; u[k][1] = y.y;
                    }
                    if (!there) w[k] = 0.0f;
                }
#pragma unroll
                for (int k = 0; k < AT_ONCE; k++)
#pragma unroll
                    for (int c = 0; c < C; c++) v[c] = fmaf(w[k], u[k][c], v[c]);
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
        bool served;
        const int first = prefix_first(a, s, &served), shared = a.n_group ? a.shared[s] : 0;
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
    const int64_t kv = g.cache.n_head_kv, sms = sm_count();
    // parts that take the fewest tile steps in all waves of CTAs; a CTA costs about four steps besides its tiles (its beginning, its partial output)
    auto parts = [&](int64_t items, int64_t tiles, int64_t at_once) {
        int best = 1;
        int64_t cost = INT64_MAX;
        for (int n = 1; n <= PX_MAX_PARTS && n <= tiles; n++) {
            const int64_t c = ((items * n + at_once - 1) / at_once) * ((tiles + n - 1) / n + 4);
            if (c < cost) {
                cost = c;
                best = n;
            }
        }
        return best;
    };
    // one sequence shares nothing, and less than a tile is no shared part
    const int64_t shared_tiles = g.n_group && g.max_group > 1 ? g.max_shared / PX_TILE : 0;
    a.served = shared_tiles > 0 ? g.max_group : 0;
    a.shared_blocks = a.shared_parts = 0;
    if (a.served) {
        const int64_t rows = (int64_t)a.served * a.each;
        B200_REQUIRE(rows < (1 << 28), "prefix_attn: groups of %d sequences are too large", g.max_group);
        a.shared_blocks = (int)((rows + prefix_shared_rows(rows) - 1) / prefix_shared_rows(rows));
        const int64_t items = (int64_t)g.n_group * kv * a.shared_blocks;
        a.shared_parts = parts(items, shared_tiles, sms);
        B200_REQUIRE(items * a.shared_parts < 0x7fffffffLL, "prefix_attn: too many groups for one launch");
    }
    a.own_blocks = (a.each + PX_BM - 1) / PX_BM;
    const int64_t own_items = (int64_t)g.n_seq * kv * a.own_blocks, own = g.max_len - shared_tiles * PX_TILE;
    a.own_parts = parts(own_items, own > PX_BN ? (own + PX_BN - 1) / PX_BN : 1, sms * 3);
    B200_REQUIRE(own_items * a.own_parts < 0x7fffffffLL, "prefix_attn: too many rows for one launch");
    p->rows = (int64_t)g.n_seq * g.n_head;
    const int64_t slots = p->rows * (a.shared_parts + a.own_parts);
    p->ml_bytes = ((size_t)slots * sizeof(float2) + 255) & ~(size_t)255;
    p->bytes = p->ml_bytes + (size_t)slots * (size_t)g.cache.d * 4;
    return B200_STATUS_SUCCESS;
}

template <typename T, int D>
int launch_prefix(const PrefixPlan &p, int type, cudaStream_t s) {
    const PrefixArgs &a = p.a;
    constexpr int SMEM = 2 * PX_STAGES<D> * PX_BN * D * 2;
    int rc = a.shared_parts ? launch_prefix_shared(a, type, s) : B200_STATUS_SUCCESS;
    if (rc != B200_STATUS_SUCCESS) return rc;
    const int64_t ctas = (int64_t)a.n_seq * a.cache.n_head_kv * a.own_blocks * a.own_parts;
    B200_CUDA(cudaFuncSetAttribute(prefix_own_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM));
    if ((rc = launch_pdl(prefix_own_kernel<T, D>, dim3((unsigned)ctas), dim3(PX_NT), SMEM, s, a, a.shared_parts > 0)) != B200_STATUS_SUCCESS) return rc;
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
    a.shared = g.shared;
    a.group_first = g.group_first;
    a.sinks = g.sinks;
    a.scale_log2 = g.scale * PX_LOG2E;
    a.ml = (float2 *)g.workspace;
    a.acc = (float *)((uint8_t *)g.workspace + p.ml_bytes);
    const cudaStream_t s = (cudaStream_t)stream;
    if (g.cache.type == B200_TYPE_F16) return g.cache.d == 128 ? launch_prefix<__half, 128>(p, g.cache.type, s) : launch_prefix<__half, 64>(p, g.cache.type, s);
    return g.cache.d == 128 ? launch_prefix<__nv_bfloat16, 128>(p, g.cache.type, s) : launch_prefix<__nv_bfloat16, 64>(p, g.cache.type, s);
}

}  // extern "C"
