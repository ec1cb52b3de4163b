// What the beams of a request hold, moved to the beams that were chosen (b200_beam_reorder).
//
// Nothing is moved that a table can say: a parent's first child takes over its row of the table (pages, state slots), so that only the second and
// further children of a parent need a copy, into the pages of beams that nobody continues.  Sources are then always rows that keep their contents
// and destinations rows that nobody reads, so that copies need no order and no second buffer.
//
// Bound by memory: 2 bytes of traffic for each byte of a page that moves.  Every CTA works out the request's plan from its parents (at most 64: two
// ballots a group), so that there is one launch: grid (sequences x shares of a sequence's pages, pools).  The CTAs of beams that take over
// a row leave at once.  Measured on the device: 8 requests of 8 beams, 300 positions of their own in pages of 16, 32 pools (638 MB copied) 196.6 us, 0.99 of the measured copy rate;
// 4 beams' states of 2 MB in 24 pools 30.3 us.  About 32 CTAs an SM in all: with 16 29.2 and 201, with 8 31 and 215.
#include "paged.cuh"

namespace b200 {

namespace {

constexpr int BR_NT = 256, BR_MAX_POOLS = 128, BR_MAX_BEAM = 64, BR_PIECE = 32768;

struct ReorderArgs {
    const int32_t *parents, *tables_in, *lens_in;
    int32_t *tables_out, *lens_out, *row_of;
    int64_t table_ld, n_pages, page_bytes, page_stride;
    int n_beam, page_size, n_pools, shares;
    int64_t pieces;                      // a page's, of up to BR_PIECE bytes
    int *err;
    uint8_t *pool[BR_MAX_POOLS];
};

__global__ void __launch_bounds__(BR_NT) beam_reorder_kernel(const __grid_constant__ ReorderArgs a) {
    pdl_trigger();
    __shared__ int par[BR_MAX_BEAM];
    __shared__ unsigned long long alive_s, first_s, used_s;
    const int tid = threadIdx.x;
    const int share = (int)(blockIdx.x % a.shares);
    const int64_t seq = blockIdx.x / a.shares, row0 = seq / a.n_beam * a.n_beam;
    const int j = (int)(seq - row0);
    if (tid == 0) alive_s = first_s = used_s = 0;
    __syncthreads();
    pdl_wait();
    if (tid < BR_MAX_BEAM) {
        int p = tid < a.n_beam ? a.parents[row0 + tid] : -1;
        if (p >= a.n_beam) {
            if (tid == j && blockIdx.y == 0 && share == 0) atomicExch(a.err, ERR_PAGED);
            p = -1;
        }
        par[tid] = p;
    }
    __syncthreads();
    if (tid < a.n_beam && par[tid] >= 0) {
        const int p = par[tid];
        bool first = true;
        for (int i = 0; i < tid; i++) first &= par[i] != p;
        atomicOr(&used_s, 1ull << tid);
        atomicOr(&alive_s, 1ull << p);
        if (first) atomicOr(&first_s, 1ull << tid);
    }
    __syncthreads();
    const unsigned long long all = a.n_beam == 64 ? ~0ull : (1ull << a.n_beam) - 1, used = used_s, first = first_s, extra = used & ~first, below = (1ull << j) - 1;
    const int p = par[j];
    int row = p;
    if (!(first >> j & 1)) {   // the n-th of the beams that nobody continues
        int n = used >> j & 1 ? __popcll(extra & below) : __popcll(extra) + __popcll(all & ~used & below);
        unsigned long long free = all & ~alive_s;
        while (n-- > 0) free &= free - 1;
        row = __ffsll((long long)free) - 1;
    }
    const int32_t *const to = a.tables_in + (row0 + row) * a.table_ld;
    const int32_t len = p >= 0 ? a.lens_in[row0 + p] : 0;
    if (blockIdx.y == 0) {
        for (int64_t i = (int64_t)share * BR_NT + tid; i < a.table_ld; i += (int64_t)a.shares * BR_NT) a.tables_out[seq * a.table_ld + i] = to[i];
        if (share == 0 && tid == 0) {
            a.lens_out[seq] = len;
            if (a.row_of) a.row_of[seq] = row;
        }
    }
    if (!(extra >> j & 1) || len <= 0 || (int)blockIdx.y >= a.n_pools) return;
    const int32_t *const from = a.tables_in + (row0 + p) * a.table_ld;
    int64_t pages = ((int64_t)len + a.page_size - 1) / a.page_size;
    if (pages > a.table_ld) {
        if (blockIdx.y == 0 && share == 0 && tid == 0) atomicExch(a.err, ERR_PAGED);
        pages = a.table_ld;
    }
    uint8_t *const pool = a.pool[blockIdx.y];
    for (int64_t w = share; w < pages * a.pieces; w += a.shares) {
        const int64_t i = a.pieces == 1 ? w : w / a.pieces, at = (w - i * a.pieces) * BR_PIECE;
        const int32_t f = from[i], t = to[i];
        if (f == t) continue;
        if (f < 0 || f >= a.n_pages || t < 0 || t >= a.n_pages) {
            if (tid == 0) atomicExch(a.err, ERR_PAGED);
            continue;
        }
        const uint4 *const src = (const uint4 *)(pool + f * a.page_stride + at);
        uint4 *const dst = (uint4 *)(pool + t * a.page_stride + at);
        const int n = (int)((a.page_bytes - at < BR_PIECE ? a.page_bytes - at : BR_PIECE) / 16);
        int e = tid;
        for (; e + 3 * BR_NT < n; e += 4 * BR_NT) {
            const uint4 v0 = __ldcs(src + e), v1 = __ldcs(src + e + BR_NT), v2 = __ldcs(src + e + 2 * BR_NT), v3 = __ldcs(src + e + 3 * BR_NT);
            dst[e] = v0;
            dst[e + BR_NT] = v1;
            dst[e + 2 * BR_NT] = v2;
            dst[e + 3 * BR_NT] = v3;
        }
        for (; e < n; e += BR_NT) dst[e] = src[e];
    }
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" int b200_beam_reorder(const struct b200_beam_reorder_args *args, void *stream) {
    B200_REQUIRE(args != nullptr, "beam_reorder: null arguments");
    const b200_beam_reorder_args &g = *args;
    B200_REQUIRE(g.n_request >= 0 && g.n_beam >= 1 && g.n_beam <= BR_MAX_BEAM, "beam_reorder: %d requests of %d beams (up to %d)", g.n_request, g.n_beam, BR_MAX_BEAM);
    B200_REQUIRE(g.n_pools >= 0 && (g.n_pools == 0 || g.pools != nullptr), "beam_reorder: %d pools", g.n_pools);
    B200_REQUIRE(g.table_ld > 0 && g.page_size > 0, "beam_reorder: rows of %lld pages of %d positions", (long long)g.table_ld, g.page_size);
    const int64_t stride = g.page_stride ? g.page_stride : g.page_bytes;
    B200_REQUIRE(g.n_pools == 0 || (g.n_pages > 0 && g.page_bytes > 0 && g.page_bytes % 16 == 0 && stride % 16 == 0 && stride >= g.page_bytes),
                 "beam_reorder: %lld pages of %lld bytes, %lld apart (multiples of 16)", (long long)g.n_pages, (long long)g.page_bytes, (long long)stride);
    if (g.n_request == 0) return B200_STATUS_SUCCESS;
    B200_REQUIRE(g.parents != nullptr && g.tables_in != nullptr && g.tables_out != nullptr && g.lens_in != nullptr && g.lens_out != nullptr, "beam_reorder: null operand");
    const int64_t n = (int64_t)g.n_request * g.n_beam;
    B200_REQUIRE(n < (1 << 24), "beam_reorder: %lld beams are too many for one launch", (long long)n);
    const size_t ids = (size_t)n * 4, tables = ids * (size_t)g.table_ld;
    const void *in[3] = {g.parents, g.tables_in, g.lens_in}, *out[3] = {g.tables_out, g.lens_out, g.row_of};
    const size_t in_bytes[3] = {ids, tables, ids}, out_bytes[3] = {tables, ids, g.row_of ? ids : 0};
    for (int o = 0; o < 3; o++)
        for (int i = 0; i < 3; i++)
            B200_REQUIRE(!paged_overlap(in[i], in_bytes[i], out[o], out_bytes[o]) && (i >= o || !paged_overlap(out[i], out_bytes[i], out[o], out_bytes[o])), "beam_reorder: an output overlaps another operand");
    for (int i = 0; i < g.n_pools; i++) B200_REQUIRE(g.pools[i] != nullptr && (uintptr_t)g.pools[i] % 16 == 0, "beam_reorder: pool %d is null or not 16-byte aligned", i);
    const PagedOperand mem[6] = {{g.parents, "parents", 4}, {g.tables_in, "tables_in", 4}, {g.tables_out, "tables_out", 4}, {g.lens_in, "lens_in", 4}, {g.lens_out, "lens_out", 4}, {g.row_of, "row_of", 4}};
    int rc = paged_check_device(mem, 6, "beam_reorder");
    for (int i = 0; i < g.n_pools && rc == B200_STATUS_SUCCESS; i++) {
        const PagedOperand pool = {g.pools[i], "a pool"};
        rc = paged_check_device(&pool, 1, "beam_reorder");
    }
    if (rc != B200_STATUS_SUCCESS) return rc;
    ReorderArgs a;
    if ((rc = device_error_word(&a.err)) != B200_STATUS_SUCCESS) return rc;
    a.parents = g.parents;
    a.tables_in = g.tables_in;
    a.lens_in = g.lens_in;
    a.tables_out = g.tables_out;
    a.lens_out = g.lens_out;
    a.row_of = g.row_of;
    a.table_ld = g.table_ld;
    a.n_pages = g.n_pages;
    a.page_bytes = g.page_bytes;
    a.page_stride = stride;
    a.n_beam = g.n_beam;
    a.page_size = g.page_size;
    a.pieces = (g.page_bytes + BR_PIECE - 1) / BR_PIECE;
    // shares of a beam's pages: about 32 CTAs an SM over all beams and pools, no more than there are pieces
    const int64_t shares = (32 * (int64_t)sm_count() + n * (g.n_pools > 0 ? g.n_pools : 1) - 1) / (n * (g.n_pools > 0 ? g.n_pools : 1)), most = g.table_ld * (a.pieces > 0 ? a.pieces : 1);
    a.shares = (int)(shares < most ? shares : most);
    for (int at = 0; at == 0 || at < g.n_pools; at += BR_MAX_POOLS) {
        a.n_pools = g.n_pools - at < BR_MAX_POOLS ? g.n_pools - at : BR_MAX_POOLS;
        for (int i = 0; i < a.n_pools; i++) a.pool[i] = (uint8_t *)g.pools[at + i];
        rc = launch_pdl(beam_reorder_kernel, dim3((unsigned)(n * a.shares), (unsigned)(a.n_pools > 0 ? a.n_pools : 1)), dim3(BR_NT), 0, (cudaStream_t)stream, a);
        if (rc != B200_STATUS_SUCCESS) return rc;
    }
    return B200_STATUS_SUCCESS;
}
