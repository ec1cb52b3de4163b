// The shared part of b200_prefix_attn: all rows of a group against the positions they share, on the tcgen05 tensor cores.
//
//   acc = sum_p w_p v_p,  sum = sum_p w_p,  w_p = exp2(scale log2(e) q k_p - m)       over the whole tiles of 128 positions that a row shares, per part
//
//   * A CTA takes up to 128 rows (sequence of the group, query head of the key head), or 256 as two blocks, and a part of the tiles.  Row r of a block is lane r of tensor memory.
//     Up to 64 (32) rows stand there twice (four times): products of 128 rows cost the same whatever they hold, and each copy takes the exponentials of half (a quarter) of a
//     tile's positions, its weights of the others zero, so that all four warps of a softmax group have work; the copies' outputs are added at the end.
//   * K and V come in tiles of 128 positions by TMA, a box a page (or as much of a page as a tile holds), the pages' ids read a tile ahead; K is a K-major
//     and V an MN-major B operand, so neither is transposed.  A page id out of range is loaded from behind the last page (zeros), and the part's rows are marked to be
//     computed again without it.
//   * Two groups of four softmax warps work in turn: with one block of rows they take the tiles alternately, each with
//     an output of its own; with two blocks each has its block and both read every tile.  While one computes weights the tensor cores have the other's
//     products.  A thread owns a row; weights go back into tensor memory over the scores they came from, as the A operand of the second product.
//   * A row sees a tile as a whole or not at all, so that no score is masked one by one.
//   * A tile's weights are taken under the maximum in use without a look at its scores; only where their sum exceeds TC_MOST (or the row has seen nothing yet) are they taken
//     again under the tile's own maximum, and the output rescaled: the weights' rounding is relative, so nothing is lost.
//   * Weights enter the second product in the cache's 16 bits, as in the own part (what that costs the outputs stands there).
// Bound by the chain of a tile: scores of a block in (a product of 128 x 128 x 128 and the way to tensor memory), 128 exponentials a thread, weights back, the second product.  Two blocks take
// 1.85 us a tile (2 x 8.4 MFLOP and 64 KB: 1.3 PFLOP/s and 5.2 TB/s while 148 SMs are at it), one block 1.25 us.  Under ncu (64 rows behind 32768 positions, two blocks of 128) the tensor cores are busy 28 % of
// the launch, memory 44 %, issue slots 24 %; the beginning (page ids, queries, first tile) and the end (outputs of 256 rows) are 10 us of 55.  (There 96 CTAs take in 35 GB/s each and 52 of the own part 50: 6 TB/s.)
// Every wait is bounded; a wait that runs out raises the CTA's abort flag and the device error word, and its rows are marked so that none is stored.
#include "prefix_attn_own.cuh"

namespace b200 {

namespace {

constexpr int TC_M = 128, TC_N = PX_TILE, TC_THREADS = 384, TC_SM_WARP0 = 4, TC_SLOTS_MAX = 8;
constexpr int TC_REGS = 168, TC_FEW_REGS = 56, TC_MANY_REGS = 216;   // a thread's at launch, then of the loading and of the softmax warps
constexpr int TC_ERR_WAIT = 4;
// F16 has no weights below 2^-24: there the maximum in use is 8 steps of log2 below the row's, so that a weight loses nothing down to 2^-22 of the largest and is dropped below
// 2^-33 (without it 2^-14 and 2^-25: behind one outstanding position a tail of 65536 equal ones was lost as a whole)
template <typename T>
constexpr float TC_LIFT = std::is_same<T, __half>::value ? 8.0f : 0.0f;
// sum of a tile's weights up to which the maximum in use is kept: no weight of F16 overflows, and 128 equal ones of a first tile stay below it
template <typename T>
constexpr float TC_MOST = std::is_same<T, __half>::value ? 61440.0f : 4096.0f;
// A maximum is rounded, a weight's exponent is not: the largest weight is 2^e with e up to half a step of the maximum.  From this one on that is 1 and more (2^31: weights
// of the best positions are all zero, or infinite), and the row is computed again position by position
constexpr float TC_FAR = 16777216.0f;
static_assert(TC_FEW_REGS * TC_SM_WARP0 * 32 + TC_MANY_REGS * (TC_THREADS - TC_SM_WARP0 * 32) <= TC_REGS * TC_THREADS, "register shares");

template <typename T, int D, int ROWS>
struct TcCfg {
    static constexpr bool TWO = ROWS == 256;
    static constexpr int BLOCK = TWO ? 128 : ROWS, COPIES = TC_M / BLOCK, COLS = TC_N / COPIES;   // rows of a block; its copies in the lanes of tensor memory; positions that each copy answers for
    static constexpr int CHUNKS = D / 64;               // 64 elements = one 128-byte swizzled box
    static constexpr int TILE = TC_N * D * 2, Q = TC_M * D * 2 * (TWO ? 2 : 1);
    static constexpr int SLOTS = D == 128 ? (TWO ? 4 : 5) : TC_SLOTS_MAX;
    static constexpr int SHARED = Q + SLOTS * TILE + 256, OWN = PX_OWN_UNITS * (int)sizeof(PxUnit<D>), SMEM = SHARED > OWN ? SHARED : OWN;   // the barriers behind the operands: nothing is static, so that the operands begin where shared memory does
    static constexpr uint32_t O_COL = 2 * TC_N;         // tensor memory: two score tiles, then two outputs
    static constexpr uint32_t TYPES = sizeof(T) == 2 && !std::is_same<T, __half>::value ? (1u << 7) | (1u << 10) : 0u;   // A and B are BF16
    static constexpr uint32_t IDESC_S = (1u << 4) | TYPES | ((uint32_t)(TC_N >> 3) << 17) | ((uint32_t)(TC_M >> 4) << 24);
    static constexpr uint32_t IDESC_O = (1u << 4) | TYPES | (1u << 16) | ((uint32_t)(D >> 3) << 17) | ((uint32_t)(TC_M >> 4) << 24);   // B is MN-major
};
struct TcShared {
    uint64_t full[TC_SLOTS_MAX], empty[TC_SLOTS_MAX];
    uint64_t sfull[2], pready[2];                       // scores of a softmax group stand; its weights stand
    uint64_t qready, done;
    uint32_t tmem_base;
    int abort_flag, n_tiles, bad;
};
struct TcArgs {
    uint32_t wait_limit;
    int mute;   // test hook: this tile's values are not asked for by the first CTA
    int box;    // positions of a box
};

__device__ __forceinline__ void tc_tma(uint32_t dst, const CUtensorMap *map, int x, int head, int pos, int page, uint64_t *bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst), "l"(map), "r"(x), "r"(head), "r"(pos), "r"(page),
                 "r"(pa_smem(bar))
                 : "memory");
}

__device__ __forceinline__ void tc_st16(uint32_t taddr, const uint32_t *r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
                 "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
                 : "memory");
}

template <typename T, int D, int ROWS>
__global__ void __launch_bounds__(TC_THREADS, 1)
prefix_parts_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, const PrefixArgs a, const TcArgs ta) {
    using C = TcCfg<T, D, ROWS>;
    constexpr bool TWO = C::TWO;
    constexpr int COPIES = C::COPIES, COLS = C::COLS;
    extern __shared__ __align__(1024) uint8_t tc_raw[];
    const int64_t shared_ctas = (int64_t)a.n_group * a.cache.n_head_kv * a.shared_blocks * a.shared_parts;
    if (blockIdx.x >= shared_ctas) {
        static_assert(PX_OWN_UNITS * PX_NT == TC_THREADS && sizeof(PxUnit<D>) % 128 == 0, "units of a CTA");
        const int unit = threadIdx.x / PX_NT;
        pdl_wait();
        pdl_trigger();
        prefix_own_stream<T, D>(a, (int)(blockIdx.x - shared_ctas) + unit * a.own_ctas, a.own_ctas * PX_OWN_UNITS, ((PxUnit<D> *)tc_raw)[unit], threadIdx.x % PX_NT, 1 + unit);
        return;
    }
    static_assert(sizeof(TcShared) <= 256, "barriers");
    TcShared &sh = *(TcShared *)(tc_raw + C::Q + C::SLOTS * C::TILE);
    const uint32_t q_s = pa_smem(tc_raw), kv_s = q_s + C::Q;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    volatile int *abort_flag = &sh.abort_flag;
    int64_t id = blockIdx.x;
    const int part = (int)(id % a.shared_parts); id /= a.shared_parts;
    const int blk = (int)(id % a.shared_blocks); id /= a.shared_blocks;
    const int hk = (int)(id % a.cache.n_head_kv), grp = (int)(id / a.cache.n_head_kv);

    if (tid == 0) {
        for (int i = 0; i < C::SLOTS; i++) {
            pa_init(&sh.full[i], 1);
            pa_init(&sh.empty[i], 1);
        }
        for (int g = 0; g < 2; g++) {
            pa_init(&sh.sfull[g], 1);
            pa_init(&sh.pready[g], 4);
        }
        pa_init(&sh.qready, 8);
        pa_init(&sh.done, 1);
        sh.abort_flag = 0;
        sh.n_tiles = sh.bad = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(pa_smem(&sh.tmem_base)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    pa_fence_before();
    __syncthreads();
    pa_fence_after();
    const uint32_t tmem = sh.tmem_base;
    pdl_wait();      // q, the cache rows of this step and the lengths come from earlier kernels
    pdl_trigger();
    // the group's rows: row x is sequence first + x / each, head hk * each + x % each
    int first = a.group_first[grp], end = a.group_first[grp + 1];
    const bool fits = prefix_group_fits(first, end, a.n_seq);
    if (!fits) {
        if (tid == 0) atomicExch(a.err, ERR_PAGED);
        first = end = 0;
    }
    const int x0 = blk * ROWS, n_rows = min(end - first, a.served) * a.each - x0;   // may be negative
    // the tiles that any of this CTA's rows sees, and this part's share of them
    if (tid < ROWS && tid < n_rows) atomicMax(&sh.n_tiles, prefix_cover(a, first + (x0 + tid) / a.each) / PX_TILE);
    __syncthreads();
    const int capacity = (int)min(a.cache.table_ld << a.cache.page_log2 >> 7, (int64_t)0xffffff);
    int n_all = sh.n_tiles;
    if (n_all > capacity) {   // the own part reports it
        n_all = capacity;
    }
    const int per = (n_all + a.shared_parts - 1) / a.shared_parts, t0 = min(part * per, n_all), n_tiles = min(per, n_all - t0);
    const int steps = TWO ? 2 * n_tiles : n_tiles;

    if (warp < TC_SM_WARP0) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(TC_FEW_REGS));
        if ((warp == 0 || warp == 2) && n_tiles > 0) {
            // warp 0 asks for the keys, warp 2 for the values: a box costs the asking warp some 115 clocks, and a tile of small pages has 16
            const bool keys = warp == 0;
            const CUtensorMap *const map = keys ? &kmap : &vmap;
            const int boxes = TC_N / ta.box, my_box = lane % boxes, my_chunk = lane / boxes;   // up to 8 boxes x 2 chunks
            const bool mine = lane < boxes * C::CHUNKS;
            const int32_t *const table = a.cache.tables + (int64_t)first * a.cache.table_ld;
            const int page_mask = (1 << a.cache.page_log2) - 1;
            // page id of this lane's box of a tile; what is out of range is read from behind the last page (zeros)
            auto page_of = [&](int t) -> int {
                if (!mine || t >= n_tiles) return 0;
                const int32_t p = __ldg(table + (((int64_t)(t0 + t) * TC_N + my_box * ta.box) >> a.cache.page_log2));
                if (p < 0 || p >= a.cache.n_pages) {
                    atomicExch(a.err, ERR_PAGED);
                    *(volatile int *)&sh.bad = 1;   // in front of this tile's arrival: the rows' last barrier comes behind it
                    return (int)min(a.cache.n_pages, (int64_t)0x7fffffff);
                }
                return p;
            };
            const int mute = !keys && blockIdx.x == 0 ? ta.mute : -1;
            bool ok = true;
            int page = page_of(0), t = 0, begun = -1;
            for (; t < n_tiles; t++) {
                const int next = page_of(t + 1);
                // the order in which the products read them: with two blocks K 0, V 0, K 1, .., with one K 0, K 1, V 0, K 2, V 1, ..
                const int seq = TWO ? 2 * t + !keys : keys ? (t < 2 ? t : 2 * t - 1) : min(2 * t + 2, n_tiles + t), s = seq % C::SLOTS;
                ok = ok && pa_wait(&sh.empty[s], ((uint32_t)(seq / C::SLOTS) & 1u) ^ 1u, abort_flag, ta.wait_limit);
                if (t == (keys ? 1 : 0)) ok = ok && pa_wait(&sh.qready, 0, abort_flag, ta.wait_limit);   // the queries are needed before these are
                if (!ok) break;
                if (lane == 0) pa_expect(&sh.full[s], C::TILE);
                __syncwarp();
                if (mine && t != mute)
                    tc_tma(kv_s + (uint32_t)(s * C::TILE + my_chunk * (TC_N * 128) + my_box * ta.box * 128), map, 64 * my_chunk, hk, ((t0 + t) * TC_N + my_box * ta.box) & page_mask, page, &sh.full[s]);
                begun = seq;
                page = next;
            }
            // a CTA that gives up still waits (bounded) for the copies it has in flight: those since the slots' last turn
            if (*abort_flag)
                for (int q = max(begun - C::SLOTS + 1, 0); q <= begun; q++) pa_drain(&sh.full[q % C::SLOTS], (uint32_t)(q / C::SLOTS) & 1u, ta.wait_limit);
        } else if (warp == 1 && n_tiles > 0) {
            // the whole warp waits, one elected lane issues: descriptors then stay in uniform registers
            const bool leader = pa_elect();
            int seq = 0, k_slot = 0, v_slot = 0;
            const uint64_t q_desc = pa_desc(q_s, 16), k_desc = pa_desc(kv_s, 16), v_desc = pa_desc(kv_s, TC_N * 128);
            bool ok = pa_wait(&sh.qready, 0, abort_flag, ta.wait_limit);
            auto arrived = [&](int *slot) {   // the next tile in the ring
                *slot = seq % C::SLOTS;
                ok = ok && pa_wait(&sh.full[*slot], (uint32_t)(seq / C::SLOTS) & 1u, abort_flag, ta.wait_limit);
                seq++;
            };
            // scores of step n, for softmax group n % 2: over its former weights, whose product was issued before (products complete in order)
            auto scores = [&](int n) {
                const int g = n & 1;
                if (!TWO || g == 0) arrived(&k_slot);
                if (!ok) return;
                pa_fence_after();
                if (leader) {
#pragma unroll
                    for (int ks = 0; ks < D / 16; ks++) {
                        const uint32_t off = (uint32_t)((ks >> 2) * TC_M * 128 + (ks & 3) * 32) >> 4;
                        pa_mma_ss(tmem + (uint32_t)(g * TC_N), q_desc + off + (uint32_t)(TWO ? g * (TC_M * D * 2 >> 4) : 0), k_desc + (uint32_t)(k_slot * (C::TILE >> 4)) + off, C::IDESC_S, ks > 0);
                    }
                    if (!TWO || g == 1) pa_commit(&sh.empty[k_slot]);
                    pa_commit(&sh.sfull[g]);
                }
            };
            for (int n = 0; n < 2 && n < steps && ok; n++) scores(n);
            for (int n = 0; n < steps && ok; n++) {
                const int g = n & 1, j = n >> 1;
                if (!TWO || g == 0) arrived(&v_slot);
                ok = ok && pa_wait(&sh.pready[g], (uint32_t)j & 1u, abort_flag, ta.wait_limit);
                if (!ok) break;
                pa_fence_after();
                if (leader) {
#pragma unroll
                    for (int ks = 0; ks < TC_N / 16; ks++)
                        pa_mma_ts(tmem + C::O_COL + (uint32_t)(g * D), tmem + (uint32_t)(g * TC_N + ks * 8), v_desc + (uint32_t)(v_slot * (C::TILE >> 4) + ks * 128), C::IDESC_O, j > 0 || ks > 0);
                    if (!TWO || g == 1) pa_commit(&sh.empty[v_slot]);
                }
                if (n + 2 < steps) scores(n + 2);
            }
            if (leader) pa_commit(&sh.done);
            // the operands and tensor memory stay until the products are through, whatever the other roles do
            pa_drain(&sh.done, 0, ta.wait_limit);
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(TC_MANY_REGS));
        const int g = (warp - TC_SM_WARP0) >> 2, r = (warp & 3) * 32 + lane;   // softmax group, row of its block: a warp reaches the tensor-memory lanes of its number modulo 4
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t t_s = tmem + lanes + (uint32_t)(g * TC_N), t_o = tmem + lanes + C::O_COL + (uint32_t)(g * D);
        const int copy = r / C::BLOCK, x = TWO ? g * TC_M + r : r % C::BLOCK;
        const bool live = x < n_rows;
        const int seq = first + (live ? (x0 + x) / a.each : 0), head = hk * a.each + (live ? (x0 + x) % a.each : 0);
        const int64_t out = ((int64_t)seq * a.n_head + head) * (a.shared_parts + PX_WARPS * a.own_parts) + part;
        const int my_tiles = live ? min(prefix_cover(a, seq) / PX_TILE, n_all) - t0 : 0;   // tiles of this part that the row sees
        if (n_tiles > 0) {
            // q into the swizzled K-major operand, zeros behind the last row: a warp takes an eighth of the rows, a lane 16 bytes at a time, all under way at once (row by row
            // through registers this took 14 us of a launch)
            constexpr int LANES = D / 8, PER = 32 / LANES, RW = (TWO ? 2 : 1) * TC_M / 8;   // lanes of a row, rows at a time
            const int e = lane % LANES, c = e >> 3, u = e & 7;
#pragma unroll
            for (int h = 0; h < RW; h += PER) {
                const int y = (warp - TC_SM_WARP0) * RW + h + lane / LANES, yb = y % TC_M, yr = TWO ? y : y % C::BLOCK, row = x0 + (yr < n_rows ? yr : 0), i = row / a.each;
                const uint8_t *const src = a.q + (int64_t)(first + i) * a.q_nb1 + (int64_t)(hk * a.each + row - i * a.each) * a.q_nb2 + 16 * e;
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(q_s + (uint32_t)((y / TC_M) * (TC_M * D * 2) + c * (TC_M * 128) + (yb >> 3) * 1024 + (yb & 7) * 128 + ((u ^ (yb & 7)) << 4))),
                             "l"(src), "r"(yr < n_rows ? 16 : 0)
                             : "memory");
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) pa_arrive(&sh.qready);
        }
        float m = -INFINITY, l = 0.0f;   // the maximum in use (log2 units) and the sum of the weights under it
        const bool warp_live = __any_sync(0xffffffffu, live);
        const int turns = TWO ? n_tiles : (n_tiles + 1 - g) / 2;
        for (int j = 0; j < turns; j++) {
            if (!pa_wait(&sh.sfull[g], (uint32_t)j & 1u, abort_flag, ta.wait_limit)) break;
            if (warp_live) {
                pa_fence_after();
                const bool sees = (TWO ? j : 2 * j + g) < my_tiles;
                const float sc = a.scale_log2;
                uint32_t p[COLS / 2];
                const uint32_t t_mine = t_s + (uint32_t)(copy * COLS);   // the warp's: a copy's rows are whole warps
                // the weights under the maximum in use; where their sum says that it has grown too much, and where there is none yet, once more under the tile's own
                bool anew = __any_sync(0xffffffffu, sees && m == -INFINITY);
                for (;;) {
                    uint32_t s[COLS];
#pragma unroll
                    for (int c = 0; c < COLS; c += 32) pa_ld32(s + c, t_mine + (uint32_t)c);
                    pa_wait_ld();
                    if (anew) {
                        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                        const float sign = sc < 0.0f ? -1.0f : 1.0f;   // under a negative scale the smallest score is the largest
#pragma unroll
                        for (int c = 0; c < COLS; c += 4)
#pragma unroll
                            for (int e = 0; e < 4; e++) mx[e] = fmaxf(mx[e], sign * __uint_as_float(s[c + e]));
                        float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
                        top = top == -INFINITY ? -INFINITY : top * fabsf(sc) - TC_LIFT<T>;
                        const float al = sees && top > m ? pa_ex2(m - top) : 1.0f;
                        if (sees) m = fmaxf(m, top);
                        l *= al;
                        if (j > 0 && __any_sync(0xffffffffu, al != 1.0f)) {
                            // the group's former product is complete: the scores that were waited for were issued behind it
#pragma unroll 1
                            for (int c = 0; c < D; c += 32) {
                                uint32_t o[32];
                                pa_ld32(o, t_o + (uint32_t)c);
                                pa_wait_ld();
#pragma unroll
                                for (int e = 0; e < 32; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * al);
                                pa_st32(t_o + (uint32_t)c, o);
                            }
                            pa_wait_st();
                        }
                    }
                    uint64_t ps[2] = {0, 0};   // two running sums each
                    const float sub = m == -INFINITY ? 0.0f : -m;
                    const uint64_t sc2 = pa_pair(sc, sc), sub2 = pa_pair(sub, sub);
#pragma unroll
                    for (int c = 0; c < COLS / 2; c++) {
                        const uint64_t y = pa_fma2(pa_pair(__uint_as_float(s[2 * c]), __uint_as_float(s[2 * c + 1])), sc2, sub2);
                        // (three in eight by multiply-adds, a polynomial of degree 4, were no faster: 16 a clock and SM are not what a tile waits for)
                        const float2 x = pa_split(y);
                        const float e0 = pa_ex2(x.x), e1 = pa_ex2(x.y);
                        p[c] = paged_pack<T>(e0, e1);
                        ps[c & 1] = pa_add2(ps[c & 1], pa_pair(e0, e1));
                    }
                    const float2 p0 = pa_split(ps[0]), p1 = pa_split(ps[1]);
                    const float sum = (p0.x + p1.x) + (p0.y + p1.y);
                    if (anew || !__any_sync(0xffffffffu, sees && !(sum <= TC_MOST<T>))) {
                        if (sees && m > -INFINITY) l += sum;
                        else if (sees && sum != sum) l = sum;   // NaN scores alone
                        break;
                    }
                    anew = true;
                }
                if (!sees || m == -INFINITY) {   // weights of zero, whatever the scores were
#pragma unroll
                    for (int c = 0; c < COLS / 2; c++) p[c] = 0u;
                }
                if constexpr (COPIES == 4) {
                    const uint32_t none[16] = {};
#pragma unroll
                    for (int c = 0; c < 4; c++) tc_st16(t_s + (uint32_t)(16 * c), c == copy ? p : none);
                } else if constexpr (COPIES == 2) {
                    const uint32_t none[32] = {};
#pragma unroll
                    for (int c = 0; c < 2; c++) pa_st32(t_s + (uint32_t)(32 * c), c == copy ? p : none);
                } else {
                    pa_st32(t_s, p);
                    pa_st32(t_s + 32u, p + 32);
                }
                pa_wait_st();
                pa_fence_before();
            }
            __syncwarp();
            if (lane == 0) pa_arrive(&sh.pready[g]);
        }
        if (l != l) m = fmaxf(m, 0.0f);   // a NaN score is no maximum, but the row has seen it
        if (n_tiles == 0) {
            if (live && copy == 0 && (TWO || g == 0)) a.ml[out] = make_float2(-INFINITY, 0.0f);
        } else {
            const bool finished = __all_sync(0xffffffffu, pa_wait(&sh.done, 0, abort_flag, ta.wait_limit) && !*abort_flag);
            pa_fence_after();
            // All products are through, or nothing will be stored: the operands' memory takes maxima and sums (over the queries) and the outputs (over the slots, row
            // after row, 16-byte piece u of row y at u ^ (y % 32)), so that rows go out whole
            float2 *const ml = (float2 *)tc_raw, *const fin = ml + 2 * TC_M;   // of both softmax groups, of a lane
            int64_t *const outs = (int64_t *)(fin + TC_M);
            float4 *const rows = (float4 *)(tc_raw + C::Q);
            float wa = 1.0f, wb = 0.0f;
            bool ina = m != -INFINITY, inb = false;
            int c0 = 0, c1 = D;
            if (!TWO) {   // the two groups' outputs under their common maximum, half the channels each
                ml[g * TC_M + r] = make_float2(m, l);
                asm volatile("bar.sync 1, 256;" ::: "memory");
                const float2 la = ml[r], lb = ml[TC_M + r];
                const float ma = la.x, mb = lb.x;
                m = fmaxf(ma, mb);
                ina = ma != -INFINITY;   // no output where the group had no tile or the row saw none of them
                inb = mb != -INFINITY;
                wa = ina ? pa_ex2(ma - m) : 0.0f;
                wb = inb ? pa_ex2(mb - m) : 0.0f;
                l = (ina ? wa * la.y : 0.0f) + (inb ? wb * lb.y : 0.0f);
                c0 = g * (D / 2);
                c1 = c0 + D / 2;
                if (COPIES > 1) {   // the copies' too
                    if (g == 0) fin[r] = make_float2(m, l);
                    asm volatile("bar.sync 1, 256;" ::: "memory");
                    float top = -INFINITY, sum = 0.0f;
#pragma unroll
                    for (int q = 0; q < COPIES; q++) top = fmaxf(top, fin[q * C::BLOCK + x].x);
#pragma unroll
                    for (int q = 0; q < COPIES; q++) {
                        const float2 f = fin[q * C::BLOCK + x];
                        if (f.x != -INFINITY) sum += pa_ex2(f.x - top) * f.y;
                    }
                    const float f = m == -INFINITY ? 0.0f : pa_ex2(m - top);
                    wa *= f;
                    wb *= f;
                    m = top;
                    l = sum;
                }
            }
            if (copy == 0 && c0 == 0) {
                outs[x] = live ? out : -1;
                if (live) a.ml[out] = !finished ? make_float2(NAN, NAN) : *(volatile int *)&sh.bad || (fabsf(m) >= TC_FAR && m > -INFINITY) ? make_float2(NAN, 0.0f) : make_float2(m, l);
            }
            const int y = TWO ? g * TC_M + r : r;
            if (warp_live) {
#pragma unroll 1
                for (int c = c0; c < c1; c += 32) {
                    uint32_t u[32], v[TWO ? 1 : 32];
                    pa_ld32(u, tmem + lanes + C::O_COL + (uint32_t)((TWO ? g * D : 0) + c));
                    if constexpr (!TWO) pa_ld32(v, tmem + lanes + C::O_COL + (uint32_t)(D + c));
                    pa_wait_ld();
#pragma unroll
                    for (int e = 0; e < 32; e++) {
                        float z = ina ? (TWO ? __uint_as_float(u[e]) : wa * __uint_as_float(u[e])) : 0.0f;
                        if constexpr (!TWO) z += inb ? wb * __uint_as_float(v[e]) : 0.0f;
                        u[e] = __float_as_uint(z);
                    }
#pragma unroll
                    for (int e = 0; e < 32; e += 4)
                        rows[y * (D / 4) + (((c + e) / 4) ^ (y & (D / 4 - 1)))] = make_float4(__uint_as_float(u[e]), __uint_as_float(u[e + 1]), __uint_as_float(u[e + 2]), __uint_as_float(u[e + 3]));
                }
            }
            asm volatile("bar.sync 1, 256;" ::: "memory");
            if (!*abort_flag) {
                const int n = min(n_rows, TWO ? 2 * TC_M : C::BLOCK);
                for (int i = tid - TC_SM_WARP0 * 32; i < n * (D / 4); i += 256) {
                    const int z = i / (D / 4), u = i % (D / 4);
                    float4 f = rows[z * (D / 4) + (u ^ (z & (D / 4 - 1)))];
#pragma unroll
                    for (int q = 1; q < COPIES; q++) {
                        const int zq = q * C::BLOCK + z;
                        const float4 h = rows[zq * (D / 4) + (u ^ (zq & (D / 4 - 1)))];
                        f.x += h.x; f.y += h.y; f.z += h.z; f.w += h.w;
                    }
                    *(float4 *)(a.acc + outs[z] * D + 4 * u) = f;
                }
            }
        }
        pa_fence_before();
    }
    __syncthreads();
    pa_fence_after();
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    if (*abort_flag && tid == 0) atomicExch(a.err, TC_ERR_WAIT);
}

template <typename T, int D, int ROWS>
int launch(const PrefixArgs &a, CUtensorMapDataType type, cudaStream_t s) {
    using C = TcCfg<T, D, ROWS>;
    TcArgs ta;
    attn_wait_hook(&ta.wait_limit, &ta.mute);
    const int page = 1 << a.cache.page_log2;
    ta.box = page < TC_N ? page : TC_N;
    CUtensorMap km, vm;
    B200_REQUIRE(paged_tile_map(&km, type, a.cache.k, D, a.cache.n_head_kv, page, a.cache.n_pages, a.cache.page_stride, ta.box) &&
                     paged_tile_map(&vm, type, a.cache.v, D, a.cache.n_head_kv, page, a.cache.n_pages, a.cache.page_stride, ta.box),
                 "prefix_attn: tensor maps over %lld pages of %d positions refused", (long long)a.cache.n_pages, page);
    B200_CUDA(cudaFuncSetAttribute(prefix_parts_kernel<T, D, ROWS>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
    // the warps' register shares come out of what the block is launched with; the swizzle counts in 1024 bytes, where shared memory begins
    static const cudaFuncAttributes built = [] {
        cudaFuncAttributes fa = {};
        if (cudaFuncGetAttributes(&fa, prefix_parts_kernel<T, D, ROWS>) != cudaSuccess) fa.numRegs = 0;
        return fa;
    }();
    B200_REQUIRE(built.numRegs >= TC_REGS && built.sharedSizeBytes == 0, "prefix_attn: a build with %d registers a thread and %zu bytes of static shared memory cannot be served", built.numRegs,
                 built.sharedSizeBytes);
    const int64_t ctas = (int64_t)a.n_group * a.cache.n_head_kv * a.shared_blocks * a.shared_parts + a.own_ctas;
    return launch_pdl(prefix_parts_kernel<T, D, ROWS>, dim3((unsigned)ctas), dim3(TC_THREADS), C::SMEM, s, km, vm, a, ta);
}

}  // namespace

int prefix_shared_rows(int64_t rows) { return rows > 128 ? 256 : rows > 64 ? 128 : rows > 32 ? 64 : 32; }

template <typename T, int D>
static int launch_rows(const PrefixArgs &a, CUtensorMapDataType type, cudaStream_t s) {
    switch (prefix_shared_rows((int64_t)a.served * a.each)) {
        case 32: return launch<T, D, 32>(a, type, s);
        case 64: return launch<T, D, 64>(a, type, s);
        case 128: return launch<T, D, 128>(a, type, s);
        default: return launch<T, D, 256>(a, type, s);
    }
}

int launch_prefix_parts(const PrefixArgs &a, int type, cudaStream_t s) {
    if (type == B200_TYPE_F16) return a.cache.d == 128 ? launch_rows<__half, 128>(a, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, s) : launch_rows<__half, 64>(a, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, s);
    return a.cache.d == 128 ? launch_rows<__nv_bfloat16, 128>(a, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, s) : launch_rows<__nv_bfloat16, 64>(a, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, s);
}

}  // namespace b200
