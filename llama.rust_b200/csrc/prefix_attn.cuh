// What the kernels of b200_prefix_attn share: the launch's arguments, which sequences stand together, parts of a row.
#pragma once
#include "paged.cuh"

namespace b200 {

constexpr int PX_TILE = 128;   // positions of a tile of the shared part: it ends at a multiple of this, what is left of it belongs to the rows' own part
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
    int served;                               // sequences of a group that the shared part takes; further ones read their shared positions with their own
    int shared_parts, shared_blocks;          // CTAs that a (group, key head)'s positions and rows are dealt to
    int own_parts, own_blocks;                // parts and blocks of 16 rows of a (sequence, key head)
    int own_ctas;                             // CTAs that walk them
    float2 *ml;                               // [row][part]: maximum (log2 units), sum; the shared parts first, then PX_WARPS for each of a row's own
    float *acc;                               // [row][part][d]
    int *err;
};

__device__ __forceinline__ bool prefix_group_fits(int first, int end, int n_seq) { return first >= 0 && end >= first && end <= n_seq; }
// positions of sequence s that the shared part covers, were it served there
__device__ __forceinline__ int prefix_cover(const PrefixArgs &a, int s) { return max(min(a.lens[s], a.shared[s]), 0) / PX_TILE * PX_TILE; }

// prefix_attn_tcgen05.cu: all parts of all rows, in one launch
int launch_prefix_parts(const PrefixArgs &a, int type, cudaStream_t s);
constexpr int PX_WARPS = 4, PX_OWN_UNITS = 3;   // warps that share a part of a row's own positions; such parts that a CTA has at work at a time
int prefix_shared_rows(int64_t rows);      // rows a CTA of the shared part takes where a (group, key head) has so many

#ifdef __CUDACC__
// The group that sequence s stands in, by a whole warp: its first sequence and the one behind its last; s alone where nothing is shared, and where no group holds it
// (that is reported: false).  A search that looks at 32 places at a time
__device__ __forceinline__ bool prefix_group(const PrefixArgs &a, int s, int *first, int *end) {
    *first = s;
    *end = s + 1;
    if (a.n_group == 0) return false;
    const int lane = threadIdx.x & 31;
    int g = 0, n = a.n_group;
    while (n > 1) {
        const int step = (n + 31) / 32, at = lane * step;
        const bool behind = at < n && a.group_first[g + at] <= s;
        const int last = 31 - __clz(__ballot_sync(0xffffffffu, behind) | 1u);
        g += last * step;
        n = min(step, n - last * step);
    }
    const int f = a.group_first[g], e = a.group_first[g + 1];
    if (!prefix_group_fits(f, e, a.n_seq) || s < f || s >= e) {
        if (lane == 0) atomicExch(a.err, ERR_PAGED);
        return false;
    }
    *first = f;
    *end = e;
    return true;
}
#endif

}  // namespace b200
