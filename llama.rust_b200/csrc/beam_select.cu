// The k best continuations of a request's beams (b200_beam_select): log softmax over every beam's logits, the beam's score added, and the k
// best of beams x vocabulary in the order of (score in 64 bits, beam, logit, token).
//
//   score(b, w) = scores[b] + ((x_w - m) - log sum_v exp(x_v - m)),   m = max_v x_v        (m = +inf: x_w - m is 0 where x_w = m, -inf elsewhere)
//
// Bound by reading the logits once, but for the latency of what follows the read.  Two launches, or one of clusters for few requests of up to 16 chunks:
//   * beam_rows_kernel: a CTA holds a chunk of a row in registers (512 threads x EPT values), so that maximum, sum of exponentials and the chunk's k best come of
//     one read.  The k best: the k-th largest of the maxima of groups of threads, of which there are 2 k and more, is a bound that at least k values reach and
//     few more do; those are listed and ordered by counting the better ones of each.  Where more than 512 reach it (equal values), bisections over counts find the k-th value
//     and, of its equals, the last token.
//   * beam_merge_kernel: a CTA per request joins the chunks' sums in 64 bits and selects among beams x chunks x k candidates the same way, the scores
//     in 64 bits: two candidates of different beams are told apart unless their scores agree to about 1e-7.
//   * beam_cluster_kernel: a CTA a chunk leaves its candidates in the first one's shared memory, which merges them.
// Measured on the device: 64 rows of 128256 F32 (33 MB, 16 candidates) 17.4 us, 160 of 50001 BF16 14.8 us, 4 of 32000 F32 6.1 us.  The chunks' read takes a third of the first; the rest
// is the latency of barriers and counting, of which an SM overlaps three CTAs.
// Sums: F32 over a thread's values, 64 bits from there (1e-7 of the sum, so 1e-7 of a score).  Equal rows of one call give the same bits wherever they lie: which thread
// sums which value is the same for all of them, also where rows do not begin at 16-byte boundaries (their values are then shifted into place).  Calls of other numbers of
// rows may cut a vocabulary into other chunks, and differ in the last bits of a sum.
#include <cuda_bf16.h>

#include "paged.cuh"

namespace b200 {

namespace {

constexpr int BS_NT = 512, BS_MAX_K = 128, BS_MAX_BEAM = 64;
constexpr int BS_LIST = 512;            // candidates that are ordered by counting
constexpr int BS_CLUSTER = 16;          // chunks of a request that one launch takes
constexpr int BS_MERGE_NT = 512, BS_HELD = 4;   // threads of the merge; candidates each keeps in registers

struct Cand {                            // of a chunk, in descending order; behind its last one -inf
    float value;
    int token;
};
struct SelectArgs {
    const uint8_t *logits, *logits_end;
    const float *scores;
    const uint8_t *done;
    int64_t ld, n_vocab;
    int n_beam, k, chunks, end_token;
    Cand *cand;                          // [row][chunk][k]
    float *top;                          // [row][chunk]
    double *sum;                         // [row][chunk]
    float *out_scores;
    int32_t *out_tokens, *out_parents;
};

// an integer in the order of the float (no NaN; -0 is +0)
__device__ __forceinline__ uint32_t order32(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint64_t order64(double x) {
    const uint64_t b = (uint64_t)__double_as_longlong(x + 0.0);
    return b >> 63 ? ~b : b | (1ull << 63);
}
__device__ __forceinline__ float value32(uint32_t o) { return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o); }
__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
constexpr float LOG2E = 1.4426950408889634f, LOWEST = -3.402823466e38f;   // the least finite value
// Maxima up to which a chunk's exponentials are one multiply-add each, exp2(x log2(e) - c) with c = m log2(e) rounded: c is then below 2^13, off by 2^-12 at most, and
// what the merge's first-order correction leaves, (ln 2 2^-12)^2 / 2 = 1.4e-8, is less than half a step of F32.  Above it m is subtracted first
constexpr float NEAR_ZERO = 4096.0f;
constexpr uint64_t ORDER64_NONE = 0x000fffffffffffffull;

__device__ __forceinline__ int block_total(int v, int *part) {   // sum over the block; part: one int per warp
    v = __reduce_add_sync(0xffffffffu, v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    int t = 0;
    for (int i = 0; i < (int)(blockDim.x >> 5); i++) t += part[i];
    return t;
}

// the 16 bytes `shift` bytes into two neighbouring vectors; shift is the same for a whole row
__device__ __forceinline__ void shifted16(const uint4 &v0, const uint4 &v1, int shift, uint32_t (&w)[4]) {
    const uint32_t in[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
    const int words = shift >> 2, bits = (shift & 3) * 8;
    uint32_t s[5];
#pragma unroll
    for (int i = 0; i < 5; i++) s[i] = words == 0 ? in[i] : words == 1 ? in[i + 1] : words == 2 ? in[i + 2] : (i + 3 < 8 ? in[i + 3] : 0u);
#pragma unroll
    for (int i = 0; i < 4; i++) w[i] = __funnelshift_r(s[i], s[i + 1], bits);
}
// the 16 bytes at p, which need not be aligned; [lo, hi): the bytes that may be read in whole words around them
template <typename T>
__device__ __forceinline__ void load16(const uint8_t *p, const uint8_t *row_end, const uint8_t *lo, const uint8_t *hi, uint32_t (&w)[4]) {
    constexpr int N = 16 / (int)sizeof(T);
    const int shift = (int)((uintptr_t)p & 15);
    if (shift == 0 && p + 16 <= row_end) {
        const uint4 v = ld_stream16(p);
        w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
        return;
    }
    const uint8_t *const a = p - shift;
    if (p + 16 <= row_end && a >= lo && a + 32 <= hi) {
        const uint4 v0 = *(const uint4 *)a, v1 = *(const uint4 *)(a + 16);
        shifted16(v0, v1, shift, w);
        return;
    }
    // value by value at the tensor's ends
    const T none = (T)(-INFINITY);
    __align__(16) T e[N];
#pragma unroll
    for (int i = 0; i < N; i++) e[i] = p + (i + 1) * (int)sizeof(T) <= row_end ? ((const T *)p)[i] : none;
#pragma unroll
    for (int i = 0; i < 4; i++) w[i] = ((const uint32_t *)e)[i];
}

template <typename T>
struct Unpack;
template <>
struct Unpack<float> {
    static constexpr int N = 4;
    __device__ static void get(const uint32_t (&w)[4], float *v) {
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = __uint_as_float(w[i]);
    }
};
template <typename T>
struct Unpack {
    static constexpr int N = 8;
    __device__ static void get(const uint32_t (&w)[4], float *v) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 f = paged_two<T>(w[i]);
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    }
};

// threads of a group of which one maximum is taken: 16, fewer for more candidates
__device__ __forceinline__ int group_width(int k) { return k <= 16 ? 16 : k <= 32 ? 8 : k <= 64 ? 4 : 2; }
static_assert(BS_NT >= 4 * BS_MAX_K && BS_MERGE_NT == BS_NT, "two groups of two threads a candidate");

struct ChunkShared {
    __align__(16) float group_top[32], small_top[BS_NT / 2];
    float bound;
    double warp_sum[BS_NT / 32];
    uint64_t list[BS_LIST];                  // order of the value, then the complement of the token: larger is better
    int n_list, part[BS_NT / 32];
};

// A chunk of a row: its k best (behind the last one -inf), its maximum, its sum of exponentials.  EPT values a thread, a vector of 16 bytes at a time: value N j + i of
// vector v of thread t is element chunk * BS_NT * EPT + (v * BS_NT + t) * N + i
template <typename T, int EPT>
__device__ __forceinline__ void beam_chunk(const SelectArgs &a, int64_t row, int chunk, Cand *out, float *out_top, double *out_sum, ChunkShared &sh) {
    constexpr int N = Unpack<T>::N, VECS = EPT / N;
    const int tid = threadIdx.x;
    const uint8_t *const base = a.logits + row * a.ld * (int64_t)sizeof(T), *const row_end = base + a.n_vocab * (int64_t)sizeof(T);
    const int first = chunk * BS_NT * EPT;   // the vocabulary is below 2^31
    float x[EPT];
    const bool whole = (int64_t)first + BS_NT * EPT <= a.n_vocab;
    const int shift = (int)((uintptr_t)base & 15);
    const uint8_t *const from = base - shift + (int64_t)first * (int)sizeof(T);   // whole vectors around the chunk
    if (whole && shift == 0) {
        uint4 w[VECS];
#pragma unroll
        for (int v = 0; v < VECS; v++) w[v] = ld_stream16(from + (v * BS_NT + tid) * 16);
#pragma unroll
        for (int v = 0; v < VECS; v++) {
            const uint32_t u[4] = {w[v].x, w[v].y, w[v].z, w[v].w};
            Unpack<T>::get(u, x + v * N);
        }
    } else if (whole && from >= a.logits && from + (BS_NT * VECS + 1) * 16 <= a.logits_end) {   // a row that begins anywhere: the vector behind is a neighbour's, from L1
        uint4 w[VECS], next[VECS];
#pragma unroll
        for (int v = 0; v < VECS; v++) {
            w[v] = __ldg((const uint4 *)(from + (v * BS_NT + tid) * 16));
            next[v] = __ldg((const uint4 *)(from + (v * BS_NT + tid + 1) * 16));
        }
#pragma unroll
        for (int v = 0; v < VECS; v++) {
            uint32_t u[4];
            shifted16(w[v], next[v], shift, u);
            Unpack<T>::get(u, x + v * N);
        }
    } else {   // the row's end, and the tensor's
#pragma unroll
        for (int v = 0; v < VECS; v++) {
            const int64_t e = (int64_t)first + (int64_t)(v * BS_NT + tid) * N;
            if (e < a.n_vocab) {
                uint32_t w[4];
                load16<T>(base + e * (int64_t)sizeof(T), row_end, base, row_end, w);
                Unpack<T>::get(w, x + v * N);
            } else {
#pragma unroll
                for (int i = 0; i < N; i++) x[v * N + i] = -INFINITY;
            }
        }
    }
    float mine = -INFINITY, four[EPT / 4];   // maxima of all its values, of each four
#pragma unroll
    for (int i = 0; i < EPT; i += 4) {
#pragma unroll
        for (int e = 0; e < 4; e++) x[i + e] = fmaxf(x[i + e], -INFINITY);   // a NaN counts as -inf
        four[i / 4] = fmaxf(max3(x[i], x[i + 1], x[i + 2]), x[i + 3]);
        mine = fmaxf(mine, four[i / 4]);
    }
    // maxima of 32 groups of 16 threads, then of the chunk; for more than 16 candidates those of smaller groups too
    const int lane = tid & 31, width = group_width(a.k);
    float g = mine;
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) {
        if (o == width && (tid & (width - 1)) == 0) sh.small_top[tid / width] = g;
        g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, o));
    }
    if ((tid & 15) == 0) sh.group_top[tid >> 4] = g;
    if (tid == 0) sh.n_list = 0;
    __syncthreads();
    const float mine_g = sh.group_top[lane];
    float m = mine_g;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    // sum of exponentials; what the rounding of c is off by, the merge puts right
    float s = 0.0f;
    if (fabsf(m) <= NEAR_ZERO) {
        const float c = m * LOG2E;
        float s4[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < EPT; i++) s4[i & 3] += fast_exp2(fmaf(x[i], LOG2E, -c));
        s = (s4[0] + s4[1]) + (s4[2] + s4[3]);
    } else if (m > -INFINITY) {
#pragma unroll
        for (int i = 0; i < EPT; i++) s += x[i] == m ? 1.0f : exp2f((x[i] - m) * LOG2E);
    }
    double ds = (double)s;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ds += __shfl_xor_sync(0xffffffffu, ds, o);
    if (lane == 0) sh.warp_sum[tid >> 5] = ds;
    // A bound that k values of the chunk reach and few more do: the k-th largest of the groups' maxima, of which there are 2 k and more (independent values:
    // at most 1.4 k above it).  A group's threads share the comparisons.  Where fewer than k maxima are finite it lets every finite value pass
    if (width == 16) {   // (by the loop below: 64 rows of 128256 18.9 us, so 17.2)
        const int j = 2 * (lane & 15), me = tid >> 4;
        const float2 o = *(const float2 *)(sh.group_top + j);
        int better = (o.x > g || (o.x == g && j < me)) + (o.y > g || (o.y == g && j + 1 < me));
#pragma unroll
        for (int s16 = 8; s16 > 0; s16 >>= 1) better += __shfl_xor_sync(0xffffffffu, better, s16);
        if (better == a.k - 1) sh.bound = g;   // sixteen threads, one value
    } else {
        const int me = tid / width;
        const float own = sh.small_top[me];
        int better = 0;
        for (int j = tid & (width - 1); j < BS_NT / width; j += width) {
            const float other = sh.small_top[j];
            better += other > own || (other == own && j < me);
        }
        for (int o = width / 2; o > 0; o >>= 1) better += __shfl_xor_sync(0xffffffffu, better, o);
        if (better == a.k - 1) sh.bound = own;
    }
    __syncthreads();
    const float bound = fmaxf(sh.bound, LOWEST);
    // (hits counted by warp and stored without the additions' answers: more instructions, slower)
#pragma unroll
    for (int f = 0; f < EPT / 4; f++)
        if (four[f] >= bound) {
#pragma unroll
            for (int i = 4 * f; i < 4 * f + 4; i++)
                if (x[i] >= bound) {
                    const int at = atomicAdd(&sh.n_list, 1);
                    if (at < BS_LIST) sh.list[at] = (uint64_t)order32(x[i]) << 32 | (uint32_t)~(first + ((i / N) * BS_NT + tid) * N + i % N);
                }
        }
    __syncthreads();
    int n = sh.n_list;
    if (n > BS_LIST) {           // too many reach it: the k-th largest value itself, and of its equals the first
        uint32_t lo = order32(bound), top = order32(m);
        while (lo < top) {
            const uint32_t at = lo + (top - lo + 1) / 2;
            int c = 0;
#pragma unroll
            for (int i = 0; i < EPT; i++) c += order32(x[i]) >= at;
            if (block_total(c, sh.part) >= a.k) lo = at;
            else top = at - 1;
        }
        int above = 0;
#pragma unroll
        for (int i = 0; i < EPT; i++) above += order32(x[i]) > lo;
        const int want = a.k - block_total(above, sh.part);
        int l = first, h = (int)(a.n_vocab - 1 < (int64_t)first + BS_NT * EPT - 1 ? a.n_vocab - 1 : (int64_t)first + BS_NT * EPT - 1);
        while (l < h) {
            const int at = l + (h - l) / 2;
            int c = 0;
#pragma unroll
            for (int i = 0; i < EPT; i++) c += order32(x[i]) == lo && first + ((i / N) * BS_NT + tid) * N + i % N <= at;
            if (block_total(c, sh.part) >= want) h = at;
            else l = at + 1;
        }
        if (tid == 0) sh.n_list = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < EPT; i++) {
            const uint32_t o = order32(x[i]);
            if (o > lo || (o == lo && first + ((i / N) * BS_NT + tid) * N + i % N <= l)) sh.list[atomicAdd(&sh.n_list, 1)] = (uint64_t)o << 32 | (uint32_t)~(first + ((i / N) * BS_NT + tid) * N + i % N);
        }
        __syncthreads();
        n = sh.n_list;
    }
    for (int at_warp = (tid >> 5) * 8; at_warp < n; at_warp += BS_NT / 4) {   // four threads a value, eight values a warp
        const int i = at_warp + (lane >> 2);
        const uint64_t me = i < n ? sh.list[i] : 0;
        int better = 0;
#pragma unroll 4
        for (int j = tid & 3; j < n; j += 4) better += sh.list[j] > me;
        better += __shfl_xor_sync(0xffffffffu, better, 1);
        better += __shfl_xor_sync(0xffffffffu, better, 2);
        if (i < n && (tid & 3) == 0 && better < a.k) out[better] = {value32((uint32_t)(me >> 32)), (int)~(uint32_t)me};
    }
    for (int i = n + tid; i < a.k; i += BS_NT) out[i] = {-INFINITY, 0};
    if (tid == BS_NT - 1) {
        *out_top = m;
        double t = 0.0;
#pragma unroll
        for (int i = 0; i < BS_NT / 32; i++) t += sh.warp_sum[i];
        *out_sum = t;
    }
}

template <typename T, int EPT>
__global__ void __launch_bounds__(BS_NT, 3) beam_rows_kernel(const SelectArgs a) {
    pdl_trigger();
    __shared__ ChunkShared sh;
    const int64_t row = blockIdx.y, slot = row * a.chunks + blockIdx.x;
    pdl_wait();
    if (a.done && a.done[row]) return;       // the merge does not ask for this beam
    beam_chunk<T, EPT>(a, row, blockIdx.x, a.cand + slot * a.k, a.top + slot, a.sum + slot, sh);
}

// One candidate of a request: its place among them (beam, chunk, place in the chunk's list) gives the beam
struct MergeView {
    const double *offset;
    const float *top;
    int per_beam;
    __device__ __forceinline__ uint64_t order(int i, float value) const {
        const int b = i / per_beam;
        const float m = top[b];
        const double off = offset[b];
        if (off == -INFINITY) return ORDER64_NONE;
        if (m != m) return i == b * per_beam ? order64(off) : ORDER64_NONE;   // an ended beam's only one
        const double score = value == m ? off : off + ((double)value - (double)m);
        return score > -INFINITY ? order64(score) : ORDER64_NONE;   // beside a logit of +inf a word has none, and inf - inf is no score
    }
};

struct MergeShared {
    double offset[BS_MAX_BEAM];              // score of a beam less the logarithm of its sum
    float top[BS_MAX_BEAM];
    uint64_t key[BS_LIST];
    uint64_t where[BS_LIST];                 // what comes first among equal scores is less
    uint64_t bound, best;
    int n_list, part[BS_MERGE_NT / 32];
};

// Request r of its beams' chunks: candidates, maxima and sums [beam][chunk]
__device__ __forceinline__ void beam_merge(const SelectArgs &a, int64_t r, const Cand *cand, const float *tops, const double *sums, MergeShared &sh) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t row0 = r * a.n_beam;
    const int per_beam = a.chunks * a.k, total = a.n_beam * per_beam;
    if (tid == 0) sh.n_list = 0;
    // the first candidates are on their way while the beams' sums are joined
    Cand mine[BS_HELD];
#pragma unroll
    for (int u = 0; u < BS_HELD; u++) mine[u] = tid + u * BS_MERGE_NT < total ? cand[tid + u * BS_MERGE_NT] : Cand{-INFINITY, 0};
    for (int b = warp; b < a.n_beam; b += BS_MERGE_NT / 32) {
        const int64_t row = row0 + b;
        float t = lane < a.chunks ? tops[b * a.chunks + lane] : -INFINITY;   // of an ended beam whatever stands there: not used
        double part_sum = lane < a.chunks ? sums[b * a.chunks + lane] : 0.0;
        const float score = a.scores[row];
        const bool off = !(score > -INFINITY), ended = a.done && a.done[row];   // off: -inf or NaN
        float m = -INFINITY;
        double s = 0.0;
        if (!ended) {
            m = t;
            for (int c = lane + 32; c < a.chunks; c += 32) m = fmaxf(m, tops[b * a.chunks + c]);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
            for (int c = lane;;) {
                // exp(t - m), and what c = t log2(e) was off by when the chunk's exponentials were taken
                if (t > -INFINITY) {
                    const double back = fabsf(t) <= NEAR_ZERO ? 1.0 - 0.6931471805599453 * (double)fmaf(t, LOG2E, -(t * LOG2E)) : 1.0;
                    s += part_sum * back * (t == m ? 1.0 : fabsf(m) < 1e30f ? (double)fast_exp2((t - m) * LOG2E) : exp((double)t - (double)m));
                }
                c += 32;
                if (c >= a.chunks) break;
                t = tops[b * a.chunks + c];
                part_sum = sums[b * a.chunks + c];
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        }
        if (lane == 0) {
            sh.offset[b] = off || (!ended && m == -INFINITY) ? -INFINITY : ended ? (double)score : (double)score - log(s);
            sh.top[b] = ended ? NAN : m;
        }
    }
    __syncthreads();
    const MergeView view = {sh.offset, sh.top, per_beam};
    uint64_t held[BS_HELD], most = ORDER64_NONE;
#pragma unroll
    for (int u = 0; u < BS_HELD; u++) {
        const int i = tid + u * BS_MERGE_NT;
        held[u] = i < total ? view.order(i, mine[u].value) : ORDER64_NONE;
        most = held[u] > most ? held[u] : most;
    }
    for (int i = tid + BS_HELD * BS_MERGE_NT; i < total; i += BS_MERGE_NT) {
        const uint64_t o = view.order(i, cand[i].value);
        most = o > most ? o : most;
    }
    // count of a thread's own candidates for which f(order, candidate, place) holds
    auto count = [&](auto f) -> int {
        int c = 0;
#pragma unroll
        for (int u = 0; u < BS_HELD; u++) c += held[u] > ORDER64_NONE && f(held[u], mine[u], tid + u * BS_MERGE_NT);
        for (int i = tid + BS_HELD * BS_MERGE_NT; i < total; i += BS_MERGE_NT) {
            const Cand cd = cand[i];
            const uint64_t o = view.order(i, cd.value);
            c += o > ORDER64_NONE && f(o, cd, i);
        }
        return c;
    };
    // beam (6 bits), then the complement of the logit's order (a beam's larger logits come first, also where 64 bits do not tell their scores apart), then token (24
    // bits; of an ended beam's only candidate logit and token are whatever stands there)
    auto place = [&](const Cand &cd, int i) -> uint64_t { return (uint64_t)(i / per_beam) << 56 | (uint64_t)~order32(cd.value) << 24 | (cd.token & 0xffffff); };
    // Bound: k candidates reach lo, as above.  Fewer than k groups have any: every candidate passes
    const int width = group_width(a.k), groups = BS_MERGE_NT / width;
    for (int o = width / 2; o > 0; o >>= 1) {
        const uint64_t v = __shfl_xor_sync(0xffffffffu, most, o);
        most = v > most ? v : most;
    }
    if (tid % width == 0) sh.key[tid / width] = most;
    __syncthreads();
    {
        int better = 0;   // the threads of a group share the comparisons
#pragma unroll 2
        for (int j = tid % width; j < groups; j += width) {
            const uint64_t other = sh.key[j];
            better += other > most || (other == most && j < tid / width);
        }
        for (int o = width / 2; o > 0; o >>= 1) better += __shfl_xor_sync(0xffffffffu, better, o);
        if (better == a.k - 1) sh.bound = most;
        if (better == 0) sh.best = most;
    }
    __syncthreads();
    uint64_t lo = sh.bound > ORDER64_NONE ? sh.bound : ORDER64_NONE + 1;
    auto list = [&](uint64_t o, const Cand &cd, int i) {
        const int e = atomicAdd(&sh.n_list, 1);
        if (e < BS_LIST) {
            sh.key[e] = o;
            sh.where[e] = place(cd, i);
        }
        return true;
    };
    count([&](uint64_t o, const Cand &cd, int i) { return o >= lo && list(o, cd, i); });
    __syncthreads();
    int n = sh.n_list;
    if (n > BS_LIST) {   // too many reach it: the k-th score itself, and of its equals the first by beam, logit and token
        uint64_t up = sh.best;
        while (lo < up) {
            const uint64_t mid = lo + (up - lo) / 2 + ((up - lo) & 1);
            if (block_total(count([&](uint64_t o, const Cand &, int) { return o >= mid; }), sh.part) >= a.k) lo = mid;
            else up = mid - 1;
        }
        const int want = a.k - block_total(count([&](uint64_t o, const Cand &, int) { return o > lo; }), sh.part);
        uint64_t l = 0, h = ((uint64_t)a.n_beam << 56) - 1;
        while (l < h) {
            const uint64_t mid = l + (h - l) / 2;
            if (block_total(count([&](uint64_t o, const Cand &cd, int i) { return o == lo && place(cd, i) <= mid; }), sh.part) >= want) h = mid;
            else l = mid + 1;
        }
        if (tid == 0) sh.n_list = 0;
        __syncthreads();
        count([&](uint64_t o, const Cand &cd, int i) { return (o > lo || (o == lo && place(cd, i) <= l)) && list(o, cd, i); });
        __syncthreads();
        n = sh.n_list;
    }
    for (int at_warp = warp * 4; at_warp < n; at_warp += BS_MERGE_NT / 8) {   // eight threads a candidate, four candidates a warp
        const int i = at_warp + (lane >> 3);
        const uint64_t me = i < n ? sh.key[i] : 0;
        const uint64_t at = i < n ? sh.where[i] : 0;
        int better = 0;
#pragma unroll 2
        for (int j = tid & 7; j < n; j += 8) better += sh.key[j] > me || (sh.key[j] == me && sh.where[j] < at);
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) better += __shfl_xor_sync(0xffffffffu, better, o);
        if (i < n && (tid & 7) == 0 && better < a.k) {
            const int64_t e = r * a.k + better;
            const uint64_t bits = me >> 63 ? me & ~(1ull << 63) : ~me;
            a.out_scores[e] = (float)__longlong_as_double((long long)bits);
            const int b = (int)(at >> 56);
            a.out_parents[e] = b;
            a.out_tokens[e] = sh.top[b] != sh.top[b] ? a.end_token : (int32_t)(at & 0xffffff);
        }
    }
    for (int i = n + tid; i < a.k; i += BS_MERGE_NT) {
        a.out_scores[r * a.k + i] = -INFINITY;
        a.out_tokens[r * a.k + i] = -1;
        a.out_parents[r * a.k + i] = -1;
    }
}

__global__ void __launch_bounds__(BS_MERGE_NT) beam_merge_kernel(const SelectArgs a) {
    pdl_trigger();
    __shared__ MergeShared sh;
    const int64_t r = blockIdx.x, slot0 = r * a.n_beam * a.chunks;
    pdl_wait();
    beam_merge(a, r, a.cand + slot0 * a.k, a.top + slot0, a.sum + slot0, sh);
}

// Both in one launch, for few requests of up to 16 chunks in all: a cluster a request.  Every CTA leaves its chunk's candidates in the first one's shared memory, which
// merges them (4 beams x 32000: 6.0 us of the device, 6.5 in two launches, and 2 us less of the host)
template <typename T, int EPT>
__global__ void __launch_bounds__(BS_NT) beam_cluster_kernel(const SelectArgs a) {
    pdl_trigger();
    __shared__ union {
        ChunkShared chunk;
        MergeShared merge;
    } sh;
    __shared__ Cand cand[BS_CLUSTER * BS_MAX_K];
    __shared__ float top[BS_CLUSTER];
    __shared__ double sum[BS_CLUSTER];
    const int size = a.n_beam * a.chunks, rank = blockIdx.x % size, beam = rank / a.chunks;
    const int64_t r = blockIdx.x / size, row = r * a.n_beam + beam;
    asm volatile("barrier.cluster.arrive.relaxed.aligned;\nbarrier.cluster.wait.aligned;" ::: "memory");   // the first CTA's shared memory is there
    pdl_wait();
    if (!(a.done && a.done[row]))
        beam_chunk<T, EPT>(a, row, rank - beam * a.chunks, (Cand *)__cluster_map_shared_rank(cand, 0) + rank * a.k, (float *)__cluster_map_shared_rank(top, 0) + rank,
                           (double *)__cluster_map_shared_rank(sum, 0) + rank, sh.chunk);
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (rank == 0) beam_merge(a, r, cand, top, sum, sh.merge);
}

// values a thread: 16, or 8 where that would leave SMs without a chunk (and 4 of F32).  (256 threads with 32 values each were 24 warps an SM and waited more:
// 64 rows of 128256 17.2 us then, 16.7 so)
int select_ept(int64_t rows, int64_t n_vocab, int type) {
    const int sms = sm_count(), least = type == B200_TYPE_F32 ? 4 : 8;
    for (int ept = 16; ept > least; ept /= 2)
        if (rows * ((n_vocab + BS_NT * ept - 1) / (BS_NT * ept)) >= 2 * sms) return ept;
    return least;
}

// The same for the form with clusters: the fewest values a thread with which a request has no more chunks than that; 0: two launches.  Clusters are quicker while all of
// them are at work at once, two CTAs an SM (larger ones leave SMs of a group over), and wait for one another beyond; F32, us of the device, clusters and two launches:
//   CTAs of a request  requests                       requests
//                   1  296       6.5    8.9             400   11.7   11.6
//                   2  148       6.5    7.9             160   11.2    8.0
//                   4   64       6.8    7.5              74    8.6    7.7
//                   8   18       7.1    7.8              37    9.9    9.0
//                  16   14       7.5    8.6 (32000 x 4)  16   10.7    9.4 (64: 18.8 and 9.4 at 32000, 114 and 15 at 8 x 5000)
int select_cluster_ept(int n_request, int n_beam, int64_t n_vocab, int type) {
    for (int ept = type == B200_TYPE_F32 ? 4 : 8; ept <= 16; ept *= 2) {
        const int64_t size = n_beam * ((n_vocab + BS_NT * ept - 1) / (BS_NT * ept)), ctas = n_request * size;
        if (size <= BS_CLUSTER) return 4 * ctas <= (size <= 2 ? 8 : size <= 4 ? 7 : 6) * (int64_t)sm_count() ? ept : 0;
    }
    return 0;
}

struct SelectPlan {
    bool cluster;
    int ept;
    int64_t rows, chunks;
    size_t cand, top, sum, bytes;     // offsets in the workspace
};
size_t up256(size_t v) { return (v + 255) & ~(size_t)255; }

int select_plan(const b200_beam_select_args &g, SelectPlan *p) {
    B200_REQUIRE(g.logits_type == B200_TYPE_F32 || g.logits_type == B200_TYPE_F16 || g.logits_type == B200_TYPE_BF16, "beam_select: logits of type %d are not F32, F16 or BF16", g.logits_type);
    B200_REQUIRE(g.n_request >= 0 && g.n_request <= 65535 && g.n_beam >= 1 && g.n_beam <= BS_MAX_BEAM, "beam_select: %d requests of %d beams (up to 65535 of up to %d)", g.n_request, g.n_beam, BS_MAX_BEAM);
    B200_REQUIRE(g.k >= 1 && g.k <= BS_MAX_K, "beam_select: %d candidates (1 to %d)", g.k, BS_MAX_K);
    B200_REQUIRE(g.n_vocab >= 1 && g.n_vocab <= (1 << 24) && g.logits_ld >= g.n_vocab, "beam_select: a vocabulary of %lld in rows %lld apart (up to 2^24)", (long long)g.n_vocab, (long long)g.logits_ld);
    p->rows = (int64_t)g.n_request * g.n_beam;
    p->ept = select_cluster_ept(g.n_request, g.n_beam, g.n_vocab, g.logits_type);
    p->cluster = p->ept > 0;
    if (!p->cluster) p->ept = select_ept(p->rows, g.n_vocab, g.logits_type);
    p->chunks = (g.n_vocab + BS_NT * p->ept - 1) / (BS_NT * p->ept);
    B200_REQUIRE(p->rows <= 65535, "beam_select: %lld rows are too many for one launch", (long long)p->rows);
    B200_REQUIRE(p->chunks * g.k * g.n_beam < 0x7fffffffLL, "beam_select: too many candidates of a request");
    const size_t slots = (size_t)(p->rows * p->chunks);
    p->cand = 0;
    p->top = p->cand + up256(slots * g.k * sizeof(Cand));
    p->sum = p->top + up256(slots * 4);
    p->bytes = p->sum + up256(slots * 8);
    return B200_STATUS_SUCCESS;
}

template <typename T, int EPT>
int launch_select(const SelectArgs &a, const SelectPlan &p, int n_request, cudaStream_t s) {
    if (p.cluster) {
        const unsigned size = (unsigned)(a.n_beam * a.chunks);
        if (size > 8) B200_CUDA(cudaFuncSetAttribute(beam_cluster_kernel<T, EPT>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        return launch_pdl_cluster(beam_cluster_kernel<T, EPT>, dim3((unsigned)n_request * size), dim3(BS_NT), size, 0, s, a);
    }
    const int rc = launch_pdl(beam_rows_kernel<T, EPT>, dim3((unsigned)p.chunks, (unsigned)p.rows), dim3(BS_NT), 0, s, a);
    if (rc != B200_STATUS_SUCCESS) return rc;
    return launch_pdl(beam_merge_kernel, dim3((unsigned)n_request), dim3(BS_MERGE_NT), 0, s, a);
}
template <typename T>
int launch_select(const SelectArgs &a, const SelectPlan &p, int n_request, cudaStream_t s) {
    if (p.ept == 16) return launch_select<T, 16>(a, p, n_request, s);
    if constexpr (sizeof(T) == 4)
        if (p.ept == 4) return launch_select<T, 4>(a, p, n_request, s);
    return launch_select<T, 8>(a, p, n_request, s);
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" {

size_t b200_beam_select_workspace_nbytes(const struct b200_beam_select_args *args) {
    SelectPlan p;
    if (args == nullptr || select_plan(*args, &p) != B200_STATUS_SUCCESS) return 0;
    return p.bytes ? p.bytes : 256;
}

int b200_beam_select(const struct b200_beam_select_args *args, void *stream) {
    B200_REQUIRE(args != nullptr, "beam_select: null arguments");
    const b200_beam_select_args &g = *args;
    SelectPlan p;
    int rc = select_plan(g, &p);
    if (rc != B200_STATUS_SUCCESS) return rc;
    if (g.n_request == 0) return B200_STATUS_SUCCESS;
    B200_REQUIRE(g.logits != nullptr && g.scores != nullptr && g.out_scores != nullptr && g.out_tokens != nullptr && g.out_parents != nullptr, "beam_select: null operand");
    B200_REQUIRE(g.done == nullptr || (g.end_token >= 0 && g.end_token < g.n_vocab), "beam_select: end token %d is outside the vocabulary", g.end_token);
    const int size = g.logits_type == B200_TYPE_F32 ? 4 : 2;
    B200_REQUIRE((uintptr_t)g.logits % size == 0, "beam_select: logits must be aligned to their type");
    B200_REQUIRE(g.workspace != nullptr && (uintptr_t)g.workspace % 256 == 0 && g.workspace_nbytes >= p.bytes, "beam_select: a workspace of %zu bytes, 256-byte aligned, is needed (%zu given)", p.bytes,
                 g.workspace_nbytes);
    // A request's scores are read until its choice is made: another's results must not lie on them.  Its own may, where there are as many
    const size_t rows4 = (size_t)p.rows * 4, outs = (size_t)g.n_request * g.k * 4;
    const void *const in[3] = {g.logits, g.scores, g.done}, *const out[4] = {g.out_scores, g.out_tokens, g.out_parents, g.workspace};
    const size_t in_bytes[3] = {(size_t)((p.rows - 1) * g.logits_ld + g.n_vocab) * size, rows4, g.done ? (size_t)p.rows : 0}, out_bytes[4] = {outs, outs, outs, p.bytes};
    for (int o = 0; o < 4; o++) {
        for (int i = 0; i < 3; i++)
            B200_REQUIRE(!paged_overlap(in[i], in_bytes[i], out[o], out_bytes[o]) || (i == 1 && o == 0 && g.scores == g.out_scores && g.k == g.n_beam),
                         "beam_select: an output or the workspace overlaps another operand");
        for (int i = 0; i < o; i++) B200_REQUIRE(!paged_overlap(out[i], out_bytes[i], out[o], out_bytes[o]), "beam_select: an output or the workspace overlaps another operand");
    }
    const PagedOperand mem[7] = {{g.logits, "logits"}, {g.scores, "scores", 4}, {g.done, "done"}, {g.out_scores, "out_scores", 4}, {g.out_tokens, "out_tokens", 4}, {g.out_parents, "out_parents", 4},
                                 {g.workspace, "the workspace"}};
    if ((rc = paged_check_device(mem, 7, "beam_select")) != B200_STATUS_SUCCESS) return rc;
    uint8_t *const ws = (uint8_t *)g.workspace;
    SelectArgs a;
    a.logits = (const uint8_t *)g.logits;
    a.logits_end = a.logits + ((p.rows - 1) * g.logits_ld + g.n_vocab) * size;
    a.scores = g.scores;
    a.done = g.done;
    a.ld = g.logits_ld;
    a.n_vocab = g.n_vocab;
    a.n_beam = g.n_beam;
    a.k = g.k;
    a.chunks = (int)p.chunks;
    a.end_token = g.end_token;
    a.cand = (Cand *)(ws + p.cand);
    a.top = (float *)(ws + p.top);
    a.sum = (double *)(ws + p.sum);
    a.out_scores = g.out_scores;
    a.out_tokens = g.out_tokens;
    a.out_parents = g.out_parents;
    const cudaStream_t s = (cudaStream_t)stream;
    if (g.logits_type == B200_TYPE_F32) return launch_select<float>(a, p, g.n_request, s);
    if (g.logits_type == B200_TYPE_F16) return launch_select<__half>(a, p, g.n_request, s);
    return launch_select<__nv_bfloat16>(a, p, g.n_request, s);
}

}  // extern "C"
