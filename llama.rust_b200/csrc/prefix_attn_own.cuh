// The own part of b200_prefix_attn: what a sequence does not share, by mma.sync: the query heads of a key head are few rows, and the cache is read once.
// Bound by what an SM takes in from memory, about 50 GB/s (a tile of 64 positions, 32 KB, in 580 ns), which three units of four warps with 64 KB of tiles under way
// or at work each come near; a CTA's few or short items by the latency of their look-ups, about 5 us.
#pragma once
#include "attn_tcgen05.cuh"
#include "prefix_attn.cuh"

namespace b200 {

constexpr int PX_BM = 16, PX_BN = 64, PX_NT = PX_WARPS * 32;
// F16 has no weights below 2^-24: there a row's maximum counts 15 steps of log2 less, so that its largest weight is 2^15 and one of 2^-29 of it loses nothing
template <typename T>
constexpr float PX_LIFT = std::is_same<T, __half>::value ? 15.0f : 0.0f;
template <int D>
constexpr int PX_STAGES = D == 128 ? 2 : 4;   // 64 KB of tiles under way or at work
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
// two weights as the second product takes them, in the cache's 16 bits; the sum takes them as they were (their rounding errors have no common sign).  Weights in two parts would
// bring the outputs from 2.3e-3 of their norm (BF16; F16 2.8e-4) to the 1.7e-3 (2.1e-4) of their own rounding, for a second product that is twice as long
template <typename T>
__device__ __forceinline__ uint32_t px_weights(float lo, float hi, float *sum) {
    *sum += lo + hi;
    return paged_pack<T>(lo, hi);
}

// One part of a sequence's own positions for up to 16 query heads of a key head
struct PxItem {
    int s, hk, x0, rows, part;   // rows: query heads hk * each + x0 ..
    int p0, n, end;              // first position, tiles, behind the last position
    int first, shared;           // positions below `shared` are in the table of sequence `first`
};
struct PxTask {                  // what the multiplying side keeps of it
    int64_t row;                 // of its first query head
    int rows, part, n;
};

template <int D>
struct alignas(128) PxUnit {                  // shared memory of four warps
    unsigned char k[PX_STAGES<D>][PX_BN][D * 2], v[PX_STAGES<D>][PX_BN][D * 2];   // 16-byte piece u of row r lies at u ^ (r % 8)
    unsigned char q[PX_STAGES<D>][PX_BM][D * 2];
    int64_t cell_of[PX_STAGES<D>][PX_BN];   // byte offset of a tile's positions, -1: not there
    PxTask task[8];
};

// Four warps walk the items unit, unit + n_units, ..: a stream of tiles of 64 positions, PX_STAGES ahead of the products, whichever items they belong to, so
// that an item costs little besides its tiles (item by item, its look-ups, queries and first tile in front of each, took twice the time on four tiles; items handed to a CTA's units as they come to them were no faster).  Warp w has positions 16 w .. + 15 of
// every tile, its own maximum and sum, and leaves a part of its own for the merge.  Positions that the sequence does not see are zeros in shared memory,
// whatever the page holds.  tid: 0 .. 127; barrier: a named one of these four warps
template <typename T, int D>
__device__ __forceinline__ void prefix_own_stream(const PrefixArgs &a, int unit, int n_units, PxUnit<D> &sh, int tid, int barrier) {
    constexpr int KS = D / 16, DB = D / 8, NST = PX_STAGES<D>;
    constexpr int PIECES = D / 8, RSTEP = PX_NT / PIECES, PASSES = PX_BN / RSTEP;   // a thread's pieces of a tile: 16 bytes tid % PIECES of rows tid / PIECES + RSTEP j
    static_assert(RSTEP % 8 == 0, "a thread's rows have one place for their piece");
    const int lane = tid & 31, warp = tid >> 5;
    const int n_items = a.n_seq * a.cache.n_head_kv * a.own_blocks * a.own_parts, of_seq = a.cache.n_head_kv * a.own_blocks * a.own_parts;   // below 2^30
    const int all_parts = a.shared_parts + PX_WARPS * a.own_parts;
    const int capacity = (int)(a.cache.table_ld < (0x7fffff00 >> a.cache.page_log2) ? a.cache.table_ld << a.cache.page_log2 : 0x7fffff00);
    auto sync = [&]() { asm volatile("bar.sync %0, %1;" ::"r"(barrier), "n"(PX_NT) : "memory"); };

    // ---- the loading side: item `next_item`'s tile `tile` comes next
    PxItem it;
    it.n = 0;
    int next_item = unit - n_units;
    int tile = 0, tasks = 0;   // tasks: items handed to the multiplying side so far
    // an item's length and shared positions are read an item ahead
    int ahead_len = 0, ahead_shared = 0, grp_first = 0, grp_end = 0;   // the group of the item before: most likely this one's too
    bool in_group = false;
    // up to 32 groups are looked through in registers (two trips to memory an item otherwise, 1 us)
    const int my_first = lane < a.n_group ? a.group_first[lane] : 0, my_end = lane < a.n_group ? a.group_first[lane + 1] : 0;
    auto find_group = [&](int s) -> bool {
        if (a.n_group == 0 || a.n_group > 32) return prefix_group(a, s, &grp_first, &grp_end);
        const int g = 31 - __clz(__ballot_sync(0xffffffffu, lane < a.n_group && my_first <= s) | 1u);
        grp_first = __shfl_sync(0xffffffffu, my_first, g);
        grp_end = __shfl_sync(0xffffffffu, my_end, g);
        if (prefix_group_fits(grp_first, grp_end, a.n_seq) && s >= grp_first && s < grp_end) return true;
        if (lane == 0) atomicExch(a.err, ERR_PAGED);
        grp_first = s;
        grp_end = s + 1;
        return false;
    };
    auto read_ahead = [&](int item) {
        if (item < n_items) {
            ahead_len = a.lens[item / of_seq];
            ahead_shared = a.n_group ? a.shared[item / of_seq] : 0;
        }
    };
    read_ahead(unit);
    // on to the next item with tiles; false: there is none
    auto advance = [&]() -> bool {
        while (tile >= it.n) {
            next_item = min(next_item + n_units, n_items);
            if (next_item == n_items) return false;
            it.s = next_item / of_seq;
            int id = next_item - it.s * of_seq;
            it.part = id % a.own_parts; id /= a.own_parts;
            it.x0 = id % a.own_blocks * PX_BM;
            it.hk = id / a.own_blocks;
            it.rows = min(a.each - it.x0, PX_BM);
            const int len = ahead_len;
            it.shared = ahead_shared;
            read_ahead(next_item + n_units);
            if (it.s < grp_first || it.s >= grp_end) in_group = find_group(it.s);
            it.first = grp_first;
            const bool served = in_group && it.s - grp_first < a.served;
            if (len > capacity && tid == 0) atomicExch(a.err, ERR_PAGED);
            it.end = min(len, capacity);
            const int lo = served ? min(max(min(len, it.shared), 0), capacity) / PX_TILE * PX_TILE : 0;
            const int tiles = it.end > lo ? (it.end - lo + PX_BN - 1) / PX_BN : 0, per = (tiles + a.own_parts - 1) / a.own_parts;
            it.n = max(min(per, tiles - it.part * per), 0);
            it.p0 = lo + it.part * per * PX_BN;
            tile = 0;
            const int64_t row = (int64_t)it.s * a.n_head + it.hk * a.each + it.x0;
            if (!served && it.part == 0)   // nobody else writes them
                for (int i = tid; i < it.rows * a.shared_parts; i += PX_NT) a.ml[(row + i / a.shared_parts) * all_parts + i % a.shared_parts] = make_float2(-INFINITY, 0.0f);
            if (it.n == 0) {
                if (tid < it.rows * PX_WARPS) a.ml[(row + tid / PX_WARPS) * all_parts + a.shared_parts + PX_WARPS * it.part + tid % PX_WARPS] = make_float2(-INFINITY, 0.0f);
            } else {
                if (tid == 0) sh.task[tasks % 8] = {row, it.rows, it.part, it.n};
                tasks++;
            }
        }
        return true;
    };
    // the cell of position tid of that tile (the threads of the first two warps)
    auto look_up = [&]() -> int64_t {
        const int p = it.p0 + tile * PX_BN + tid;
        if (tid >= PX_BN || p >= it.end) return -1;
        const int64_t at = paged_row(a.cache, p < it.shared ? it.first : it.s, p);
        if (at < 0) atomicExch(a.err, ERR_PAGED);
        return at;
    };
    // its copies, and with the item's first tile its queries (zeros behind the last)
    auto stage = [&](int buf) {
        const int r = tid / PIECES, u = tid % PIECES, to = (u ^ (r & 7)) << 4;
        const int64_t head = (int64_t)it.hk * D * 2 + u * 16;
#pragma unroll
        for (int j = 0; j < PASSES; j++) {
            const int64_t at = sh.cell_of[buf][r + j * RSTEP], from = at < 0 ? 0 : at + head;
            px_cp16(&sh.k[buf][r + j * RSTEP][to], a.cache.k + from, at >= 0);
            px_cp16(&sh.v[buf][r + j * RSTEP][to], a.cache.v + from, at >= 0);
        }
        if (tile == 0) {
#pragma unroll
            for (int y = r; y < PX_BM; y += RSTEP)
                px_cp16(&sh.q[(tasks - 1) % NST][y][to], a.q + (int64_t)it.s * a.q_nb1 + (int64_t)(it.hk * a.each + it.x0 + (y < it.rows ? y : 0)) * a.q_nb2 + u * 16, y < it.rows);
        }
        tile++;
    };
#pragma unroll 1
    for (int i = 0; i < NST; i++) {
        const bool more = advance();
        if (more && tid < PX_BN) sh.cell_of[i][tid] = look_up();
        sync();
        if (more) stage(i);
        px_commit();
    }

    // ---- the multiplying side
    const int r_a = lane >> 2, r_b = r_a + 8;   // this thread's rows
    const int k_row = 16 * warp + (lane & 7) + ((lane >> 4) << 3), k_piece = (lane >> 3) & 1;
    const int v_row = 16 * warp + (lane & 7) + (((lane >> 3) & 1) << 3), v_piece = lane >> 4, turn = lane & 7;   // rows' places modulo 8
    int buf = 0;
#pragma unroll 1
    for (int done = 0; done < tasks; done++) {   // `tasks` grows while there are items
        const PxTask task = sh.task[done % 8];
        uint32_t qf[KS][4];
        float o[DB][4];
#pragma unroll
        for (int j = 0; j < DB; j++) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f;
        float m_a = -INFINITY, m_b = -INFINITY, l_a = 0.0f, l_b = 0.0f;
#pragma unroll 1
        for (int t = 0; t < task.n; t++) {
            const bool more = advance();
            const int64_t next = more ? look_up() : -1;
            px_wait_but<NST - 1>();
            sync();
            if (t == 0) {
#pragma unroll
                for (int k = 0; k < KS; k++) px_ldsm(qf[k], &sh.q[done % NST][lane & 15][((2 * k + (lane >> 4)) ^ turn) << 4]);
            }
            float sc[2][4];
#pragma unroll
            for (int n = 0; n < 2; n++) sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.0f;
#pragma unroll
            for (int k = 0; k < KS; k++) {
                uint32_t b[4];
                px_ldsm(b, &sh.k[buf][k_row][((2 * k + k_piece) ^ turn) << 4]);
                px_mma<T>(sc[0], qf[k], b[0], b[1]);
                px_mma<T>(sc[1], qf[k], b[2], b[3]);
            }
            float mx_a = -INFINITY, mx_b = -INFINITY;
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const bool there = sh.cell_of[buf][16 * warp + n * 8 + 2 * (lane & 3) + e] >= 0;
                    sc[n][e] = there ? sc[n][e] * a.scale_log2 : -INFINITY;
                    sc[n][2 + e] = there ? sc[n][2 + e] * a.scale_log2 : -INFINITY;
                    mx_a = fmaxf(mx_a, sc[n][e]);
                    mx_b = fmaxf(mx_b, sc[n][2 + e]);
                }
            mx_a = fmaxf(mx_a, __shfl_xor_sync(0xffffffffu, mx_a, 1)); mx_a = fmaxf(mx_a, __shfl_xor_sync(0xffffffffu, mx_a, 2));
            mx_b = fmaxf(mx_b, __shfl_xor_sync(0xffffffffu, mx_b, 1)); mx_b = fmaxf(mx_b, __shfl_xor_sync(0xffffffffu, mx_b, 2));
            const float mn_a = fmaxf(m_a, mx_a - PX_LIFT<T>), mn_b = fmaxf(m_b, mx_b - PX_LIFT<T>);
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
                px_ldsm_t(b, &sh.v[buf][v_row][((e + v_piece) ^ turn) << 4]);
                px_mma<T>(o[e], pf, b[0], b[1]);
                px_mma<T>(o[e + 1], pf, b[2], b[3]);
            }
            sync();   // everyone is done with this buffer
            if (more && tid < PX_BN) sh.cell_of[buf][tid] = next;
            sync();
            if (more) stage(buf);
            px_commit();
            buf = buf + 1 == NST ? 0 : buf + 1;
        }
        // this warp's part of the rows
        l_a += __shfl_xor_sync(0xffffffffu, l_a, 1); l_a += __shfl_xor_sync(0xffffffffu, l_a, 2);
        l_b += __shfl_xor_sync(0xffffffffu, l_b, 1); l_b += __shfl_xor_sync(0xffffffffu, l_b, 2);
        if (l_a != l_a) m_a = fmaxf(m_a, 0.0f);   // a NaN score is no maximum, but the row has seen it
        if (l_b != l_b) m_b = fmaxf(m_b, 0.0f);
#pragma unroll
        for (int half = 0; half < 2; half++) {
            const int r = half ? r_b : r_a;
            const float m = half ? m_b : m_a, l = half ? l_b : l_a;
            if (r >= task.rows) continue;
            const int64_t out = (task.row + r) * all_parts + a.shared_parts + PX_WARPS * task.part + warp;
            if ((lane & 3) == 0) a.ml[out] = make_float2(m, l);
            if (m == -INFINITY) continue;
            float *const acc = a.acc + out * D + 2 * (lane & 3);
#pragma unroll
            for (int j = 0; j < DB; j++) *(float2 *)(acc + 8 * j) = make_float2(o[j][2 * half], o[j][2 * half + 1]);
        }
    }
}

}  // namespace b200
