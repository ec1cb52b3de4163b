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
    int own_parts, own_blocks;                // the same of a (sequence, key head)
    float2 *ml;                               // [row][part]: maximum (log2 units), sum; the shared parts first
    float *acc;                               // [row][part][d]
    int *err;
};

__device__ __forceinline__ bool prefix_group_fits(int first, int end, int n_seq) { return first >= 0 && end >= first && end <= n_seq; }
// positions of sequence s that the shared part covers, were it served there
__device__ __forceinline__ int prefix_cover(const PrefixArgs &a, int s) { return max(min(a.lens[s], a.shared[s]), 0) / PX_TILE * PX_TILE; }

int launch_prefix_shared(const PrefixArgs &a, int type, cudaStream_t s);   // prefix_attn_tcgen05.cu
int prefix_shared_rows(int64_t rows);                                      // rows a CTA takes where a (group, key head) has so many

}  // namespace b200
