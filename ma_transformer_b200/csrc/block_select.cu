// Which blocks of keys a query reads, by a cheap score; over the pages of a paged cache (one new token per sequence) and
// over the blocks of whole sequences (prompts and training).
//
// With lo and hi the smallest and largest key of a block column by column, the G query heads of a key head score it
//     sum_g sum_d max(q_gd lo_d, q_gd hi_d) = sum_d up_d hi_d + down_d lo_d,
//     up_d = sum_g max(q_gd, 0), down_d = sum_g min(q_gd, 0):
// one dot product of 2 D terms whatever G is, and an upper bound of the group's summed q . k over the block's keys.
// Bounds are exact in the keys' type, and a selection is the one that scores in 64 bits give, so it does not depend on how
// sums are split: two blocks change places only where their true scores agree to about 1e-15.
//
// Few scores are needed to 64 bits, and all of them in 64 bits cost more than the rest of a selection (159 us of 221 for
// 65536 rows of up to 128 blocks of 64-column keys, where fp32 takes 22).  So scores are first formed in fp32 with a bound eps on their error; what lies more than 2 eps
// above or below the topk-th largest is decided by that, and the rest is scored again in 64 bits.  Where the two scores
// at the border are nearer than 2 eps to many others (equal keys, say), all of those are scored again: slower, not
// different.  A 64-bit score becomes a key whose order as an integer is the score's (NaN lowest, the query's own block
// highest); ties go to the lower index.
#include <limits.h>

#include "paged.cuh"
#include "pdl.cuh"
#include "ptx.cuh"

namespace mat {
namespace {

constexpr uint64_t kOwnKey = ~0ull;
constexpr int kWarpRow = 1024;      // keys a row may have to be held by one warp's registers

__device__ __forceinline__ uint64_t key_of(double x) {
    if (x != x) return 0;
    const uint64_t u = (uint64_t)__double_as_longlong(x);
    return (u >> 63) ? ~u : u | 0x8000000000000000ull;
}

// fp32 scores as integers of the same order (NaN lowest)
__device__ __forceinline__ uint32_t key32_of(float x) {
    if (x != x) return 0;
    const uint32_t u = __float_as_uint(x);
    return (u >> 31) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float of_key32(uint32_t k) {
    return __uint_as_float((k >> 31) ? k & 0x7fffffffu : ~k);
}

// The product form above is the definition's sum where all is finite.  Infinite bounds need its terms as they stand: a head
// that takes a bound with weight zero would make 0 x inf of it.
template <typename T> __device__ double score_by_terms(const T *q, const T *low, const T *high, int64_t G, int D) {
    double s = 0;
    for (int64_t g = 0; g < G; ++g)
        for (int d = 0; d < D; ++d) {
            const double w = (double)Elem<T>::to_f(q[g * D + d]), x = w * (double)Elem<T>::to_f(low[d]), y = w * (double)Elem<T>::to_f(high[d]);
            if (x != x || y != y) return NAN;
            s += x > y ? x : y;
        }
    return s;
}

// ---- bounds of the blocks of whole sequences ------------------------------------------------------------------------
// One CTA per block and 64 bytes x 8 of its columns: 32 vectors of columns, 8 threads each taking every 8th token, four
// tokens in flight.  A NaN key makes its column's bounds NaN.
template <typename T>
__global__ void __launch_bounds__(256) block_bounds_kernel(const T *k, T *bounds, int64_t S, int64_t nb, int block, int64_t HD) {
    pdl_trigger();
    constexpr int W = Vec16<T>::N;
    __shared__ float red[2][8][32 * W];
    const int64_t n = blockIdx.x, b = blockIdx.z, c = ((int64_t)blockIdx.y * 32 + threadIdx.x % 32) * W;
    const int part = threadIdx.x / 32;
    const int64_t s0 = n * block, s1 = s0 + block < S ? s0 + block : S;
    float lo[W], hi[W];
#pragma unroll
    for (int j = 0; j < W; ++j) { lo[j] = INFINITY; hi[j] = -INFINITY; }
    if (c < HD)
#pragma unroll 4
        for (int64_t s = s0 + part; s < s1; s += 8) {
            float x[W];
            Vec16<T>::unpack(__ldg(reinterpret_cast<const uint4 *>(k + (b * S + s) * HD + c)), x);
#pragma unroll
            for (int j = 0; j < W; ++j) { lo[j] = ptx::min_nan(lo[j], x[j]); hi[j] = ptx::max_nan(hi[j], x[j]); }
        }
#pragma unroll
    for (int j = 0; j < W; ++j) {
        red[0][part][j * 32 + threadIdx.x % 32] = lo[j];
        red[1][part][j * 32 + threadIdx.x % 32] = hi[j];
    }
    __syncthreads();
    if (part < 2 && c < HD) {          // warp 0 joins the smallest, warp 1 the largest
        float m[W];
#pragma unroll
        for (int j = 0; j < W; ++j) {
            m[j] = red[part][0][j * 32 + threadIdx.x % 32];
            for (int x = 1; x < 8; ++x) {
                const float y = red[part][x][j * 32 + threadIdx.x % 32];
                m[j] = part ? ptx::max_nan(m[j], y) : ptx::min_nan(m[j], y);
            }
        }
        *reinterpret_cast<uint4 *>(bounds + ((b * nb + n) * 2 + part) * HD + c) = Vec16<T>::pack(m);
    }
}

// ---- scores of whole sequences: a 64 x 64 tile of (queries, blocks) per CTA -----------------------------------------
template <typename T>
__global__ void __launch_bounds__(256) block_scores_kernel(const T *q, const T *bounds, uint64_t *keys, int64_t S, int64_t H, int64_t Hkv,
                                                           int64_t D, int64_t nb, int block, int causal, int64_t s_lo, int64_t s_hi) {
    const int64_t b = blockIdx.z / Hkv, h = blockIdx.z % Hkv, G = H / Hkv;
    const int64_t s0 = s_lo + (int64_t)blockIdx.y * 64, n0 = (int64_t)blockIdx.x * 64;
    const int64_t s_last = (s0 + 63 < s_hi ? s0 + 63 : s_hi - 1);
    pdl_trigger();
    pdl_wait();
    if (causal && n0 > s_last / block) return;
    __shared__ double up[16][65], down[16][65], hi[16][65], lo[16][65];
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    double acc[4][4] = {};
    for (int64_t d0 = 0; d0 < D; d0 += 16) {
        for (int i = threadIdx.x; i < 64 * 16; i += 256) {
            const int c = i % 16, r = i / 16;
            const int64_t d = d0 + c, s = s0 + r, n = n0 + r;
            double u = 0, w = 0, l = 0, x = 0;
            if (d < D && s < s_hi)
                for (int64_t g = 0; g < G; ++g) {
                    const double y = (double)Elem<T>::to_f(q[((b * S + s) * H + h * G + g) * D + d]);
                    if (y > 0) u += y; else w += y;       // a NaN lands in w and makes the row's scores NaN
                }
            if (d < D && n < nb) {
                const T *row = bounds + ((b * nb + n) * 2 * Hkv + h) * D + d;
                l = (double)Elem<T>::to_f(row[0]);
                x = (double)Elem<T>::to_f(row[Hkv * D]);
            }
            up[c][r] = u; down[c][r] = w; lo[c][r] = l; hi[c][r] = x;
        }
        __syncthreads();
#pragma unroll 4
        for (int c = 0; c < 16; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const double u = up[c][ty + 16 * i], w = down[c][ty + 16 * i];
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] += u * hi[c][tx + 16 * j] + w * lo[c][tx + 16 * j];
            }
        __syncthreads();
    }
    for (int i = 0; i < 4; ++i) {
        const int64_t s = s0 + ty + 16 * i;
        if (s >= s_hi) continue;
        for (int j = 0; j < 4; ++j) {
            const int64_t n = n0 + tx + 16 * j;
            if (n >= nb) continue;
            if (!(fabs(acc[i][j]) < INFINITY)) {
                const T *low = bounds + ((b * nb + n) * 2 * Hkv + h) * D;
                acc[i][j] = score_by_terms(q + ((b * S + s) * H + h * G) * D, low, low + Hkv * D, G, (int)D);
            }
            keys[((s - s_lo) * gridDim.z + blockIdx.z) * nb + n] = n == s / block ? kOwnKey : key_of(acc[i][j]);
        }
    }
}

// ---- the same for 16-bit types on the tensor cores, in fp32 ---------------------------------------------------------
// With q+ = max(q, 0) and q- = min(q, 0) a score is [q+ q-] . [hi lo], products of 16-bit numbers that the tensor cores
// form exactly; heads of a group follow each other in the same accumulator.  64 queries x 64 blocks per CTA, a warp per
// 16 queries.  Leaves the score and, per row, the sum of its heads' norms (times a block's norm: a bound of the terms).
template <typename T, int DP>
__global__ void __launch_bounds__(128) block_scores_mma_kernel(const T *q, const T *bounds, float *scores, float *norms, int64_t S, int64_t H, int64_t Hkv,
                                                               int64_t D_, int64_t nb, int block, int causal, int64_t s_lo, int64_t s_hi) {
    constexpr int PITCH = DP + 8;
    __shared__ __align__(16) T hi[64 * PITCH], lo[64 * PITCH];
    extern __shared__ __align__(16) char smem[];
    T *qs = (T *)smem;
    const int64_t b = blockIdx.z / Hkv, h = blockIdx.z % Hkv, G = H / Hkv;
    const int64_t s0 = s_lo + (int64_t)blockIdx.y * 64, n0 = (int64_t)blockIdx.x * 64;
    const int64_t s_last = (s0 + 63 < s_hi ? s0 + 63 : s_hi - 1);
    const int D = (int)D_, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    pdl_trigger();
    pdl_wait();
    if (causal && n0 > s_last / block) return;
    const uint4 zero = make_uint4(0, 0, 0, 0);
    for (int i = threadIdx.x; i < 64 * (DP / 8); i += 128) {
        const int r = i / (DP / 8), c = i % (DP / 8) * 8;
        const bool in = n0 + r < nb && c < D;
        const T *src = bounds + ((b * nb + n0 + r) * 2 * Hkv + h) * D + c;
        *reinterpret_cast<uint4 *>(lo + r * PITCH + c) = in ? __ldg(reinterpret_cast<const uint4 *>(src)) : zero;
        *reinterpret_cast<uint4 *>(hi + r * PITCH + c) = in ? __ldg(reinterpret_cast<const uint4 *>(src + Hkv * D)) : zero;
    }
    float s[8][4] = {}, norm0 = 0.f, norm1 = 0.f;
    for (int64_t g = 0; g < G; ++g) {
        __syncthreads();
        for (int i = threadIdx.x; i < 64 * (DP / 8); i += 128) {
            const int r = i / (DP / 8), c = i % (DP / 8) * 8;
            const bool in = s0 + r < s_hi && c < D;
            *reinterpret_cast<uint4 *>(qs + r * PITCH + c) = in ? __ldg(reinterpret_cast<const uint4 *>(q + ((b * S + s0 + r) * H + h * G + g) * D + c)) : zero;
        }
        __syncthreads();
        float sq0 = 0.f, sq1 = 0.f;
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk) {
            uint32_t a[4], up[4], down[4];
            ptx::ldmatrix_x4(a, ptx::smem_u32(qs + (warp * 16 + lane % 16) * PITCH + kk * 16 + (lane / 16) * 8));
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                const uint32_t neg = ((a[y] >> 15) & 0x00010001u) * 0xffffu;      // ones where the half is negative
                up[y] = a[y] & ~neg;
                down[y] = a[y] & neg;
                const float x0 = ptx::Mma<T>::lo(a[y]), x1 = ptx::Mma<T>::hi(a[y]);
                if (y % 2 == 0) sq0 += x0 * x0 + x1 * x1; else sq1 += x0 * x0 + x1 * x1;
            }
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                uint32_t r[4];
                const int at = (c * 16 + lane % 8 + (lane / 16) * 8) * PITCH + kk * 16 + (lane / 8 % 2) * 8;
                ptx::ldmatrix_x4(r, ptx::smem_u32(hi + at));
                ptx::Mma<T>::run(s[2 * c], up, r[0], r[1]);
                ptx::Mma<T>::run(s[2 * c + 1], up, r[2], r[3]);
                ptx::ldmatrix_x4(r, ptx::smem_u32(lo + at));
                ptx::Mma<T>::run(s[2 * c], down, r[0], r[1]);
                ptx::Mma<T>::run(s[2 * c + 1], down, r[2], r[3]);
            }
        }
#pragma unroll
        for (int y = 1; y < 4; y <<= 1) {
            sq0 += __shfl_xor_sync(0xffffffffu, sq0, y);
            sq1 += __shfl_xor_sync(0xffffffffu, sq1, y);
        }
        norm0 += sqrtf(sq0);
        norm1 += sqrtf(sq1);
    }
    const int64_t r0 = s0 + warp * 16 + lane / 4, r1 = r0 + 8;
    const int64_t row0 = (r0 - s_lo) * gridDim.z + blockIdx.z, row1 = (r1 - s_lo) * gridDim.z + blockIdx.z;
    if (blockIdx.x == 0 && lane % 4 == 0) {
        if (r0 < s_hi) norms[row0] = norm0;
        if (r1 < s_hi) norms[row1] = norm1;
    }
#pragma unroll
    for (int c = 0; c < 8; ++c)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
            const int64_t n = n0 + c * 8 + (lane % 4) * 2 + y;
            if (n >= nb) continue;
            if (r0 < s_hi) scores[row0 * nb + n] = s[c][y];
            if (r1 < s_hi) scores[row1 * nb + n] = s[c][2 + y];
        }
}

// Euclidean norm of max(|lo|, |hi|) of every block and head, one warp each; norms: [B, H_kv, blocks]
template <typename T>
__global__ void __launch_bounds__(128) block_norms_kernel(const T *bounds, float *norms, int64_t rows, int64_t nb, int64_t Hkv, int64_t D) {
    const int64_t r = (int64_t)blockIdx.x * 4 + threadIdx.x / 32;      // (b * nb + n) * Hkv + h
    pdl_trigger();
    pdl_wait();
    if (r >= rows) return;
    const T *lo = bounds + (r / Hkv * 2 * Hkv + r % Hkv) * D, *hi = lo + Hkv * D;
    float s = 0.f;
    for (int d = threadIdx.x % 32; d < D; d += 32) {
        const float x = fabsf(Elem<T>::to_f(lo[d])), y = fabsf(Elem<T>::to_f(hi[d]));
        s += x > y || x != x ? x * x : y * y;          // a NaN must show
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (threadIdx.x % 32 == 0) norms[(r / Hkv / nb * Hkv + r % Hkv) * nb + r / Hkv % nb] = sqrtf(s);
}

// ---- scores of a cache's pages ---------------------------------------------------------------------------------------
// Bound by latency at the sizes that occur: 16 us for 15625 pages x 8 heads of 64 (32 MB: 5 us), most of it the chain
// length -> table -> bounds -> sum over lanes.
//
// LP lanes share a page: a lane holds the weights of its NV vectors (of the 2 D bounds: smallest keys, then largest) in
// registers and reads four pages' vectors at once.  Leaves (score, sum of the terms' absolute values) in fp32 for pages
// first, first + step, ... of a row; `threads` threads take part.
template <typename T, int LP, int NV>
__device__ __forceinline__ void score_pages(const PagedView &c, const T *bounds, const T *q, int64_t H, int64_t Hkv, int64_t D, int64_t b, int64_t h,
                                            int n, int first, int step, float2 *scores) {
    constexpr int W = Vec16<T>::N, U = NV >= 4 ? 1 : NV == 2 ? 2 : 4;
    const int64_t G = H / Hkv;
    const int part = threadIdx.x % LP, vecs = (int)D / W;
    float w[NV][W];
    int off[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int v = i * LP + part;
        const bool high = v >= vecs;
        const int col = (high ? v - vecs : v) * W;
        off[i] = v < 2 * vecs ? (int)((high ? Hkv * D : 0) + h * D + col) : -1;
#pragma unroll
        for (int j = 0; j < W; ++j) w[i][j] = 0.f;
        if (off[i] >= 0)
            for (int64_t g = 0; g < G; ++g) {
                float x[W];
                Vec16<T>::unpack(__ldg(reinterpret_cast<const uint4 *>(q + (h * G + g) * D + col)), x);
#pragma unroll
                for (int j = 0; j < W; ++j)
                    if ((x[j] > 0) == high) w[i][j] += x[j];       // a NaN lands among the smallest keys' weights
            }
    }
    // the table is read a step ahead; the trip count is the same for all lanes of a warp (they shuffle together)
    int next[U];
    auto look_up = [&](int p0) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int p = p0 + u * step + threadIdx.x / LP;
            next[u] = p < n ? table_entry(c, b, p) : -1;
        }
    };
    look_up(first);
    for (int p0 = first; p0 < n; p0 += U * step) {
        uint4 x[U][NV];
        int64_t phys[U];
#pragma unroll
        for (int u = 0; u < U; ++u) phys[u] = next[u] < c.n_pages ? next[u] : -1;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < NV; ++i)
                x[u][i] = phys[u] >= 0 && off[i] >= 0 ? __ldg(reinterpret_cast<const uint4 *>(bounds + phys[u] * 2 * Hkv * D + off[i])) : make_uint4(0, 0, 0, 0);
        look_up(p0 + U * step);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float s = 0.f, size = 0.f;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                float y[W];
                Vec16<T>::unpack(x[u][i], y);
#pragma unroll
                for (int j = 0; j < W; ++j) {
                    s = fmaf(w[i][j], y[j], s);
                    size = fmaf(fabsf(w[i][j]), fabsf(y[j]), size);
                }
            }
#pragma unroll
            for (int o = LP / 2; o > 0; o >>= 1) {
                s += __shfl_xor_sync(0xffffffffu, s, o);
                size += __shfl_xor_sync(0xffffffffu, size, o);
            }
            const int p = p0 + u * step + threadIdx.x / LP;
            // a page outside the cache is no number: it sends its row to the 64-bit scores, which report it and rank it last
            if (part == 0 && p < n) scores[p] = make_float2(phys[u] < 0 ? -INFINITY : s, size);
        }
    }
}

template <typename T, int LP, int NV>
__global__ void __launch_bounds__(256) page_scores_kernel(PagedView c, const T *bounds, const T *q, int64_t q_stride, int64_t H, int64_t Hkv, int64_t D,
                                                          const int32_t *lengths, float2 *scores) {
    constexpr int GROUPS = 256 / LP;
    const int64_t b = blockIdx.z, h = blockIdx.y;
    pdl_trigger();
    const int64_t len = lengths[b];
    if (len <= 0) return;
    const int64_t held = ((len - 1) >> c.page_shift) + 1;      // pages that hold tokens; the last is the token's own
    const int n = (int)(held < c.width ? held : c.width), first = blockIdx.x * GROUPS;
    if (first < n)
        score_pages<T, LP, NV>(c, bounds, q + b * q_stride, H, Hkv, D, b, h, n, first, gridDim.x * GROUPS, scores + (b * Hkv + h) * c.width);
}

// ---- the topk of a row -----------------------------------------------------------------------------------------------
// Rows of whole sequences: row r = (s - s_lo, b, h), its eligible keys are [0, own] (causal) or [0, nb).
struct RowsOfBlocks {
    int B, S, Hkv, nb, s_lo, block, causal;     // 32-bit: a 64-bit division is some 100 instructions
    __device__ __forceinline__ int query(uint32_t r) const { return s_lo + (int)(r / (uint32_t)(B * Hkv)); }
    __device__ __forceinline__ int count(uint32_t r) const { return causal ? query(r) / block + 1 : nb; }
    __device__ __forceinline__ int64_t stride() const { return nb; }
    __device__ __forceinline__ int64_t out_row(uint32_t r) const {
        const int bh = (int)(r % (uint32_t)(B * Hkv)), b = bh / Hkv;
        return ((int64_t)b * S + query(r)) * Hkv + bh - b * Hkv;
    }
};

// The k largest of a row's n keys, held by one warp: key[j] of lane l is number 32 j + l (0 past n).
template <int PER> __device__ __forceinline__ void topk_of_warp(const uint64_t (&key)[PER], int n, int k, int topk, int32_t *o) {
    const int lane = threadIdx.x % 32;
    uint64_t cut = 0;
    if (k < n) {
        for (int bit = 63; bit >= 0; --bit) {
            const uint64_t want = cut | (1ull << bit);
            int c = 0;
#pragma unroll
            for (int j = 0; j < PER; ++j) c += key[j] >= want;
            c = __reduce_add_sync(0xffffffffu, c);
            if (c >= k) cut = want;
            if (c == k) break;
        }
    }
    int above = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) above += key[j] > cut && j * 32 + lane < n;
    int ties = k - __reduce_add_sync(0xffffffffu, above), done = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const bool in = j * 32 + lane < n, tie = in && key[j] == cut;
        const uint32_t tied = __ballot_sync(0xffffffffu, tie), below = (1u << lane) - 1;
        const bool take = in && (key[j] > cut || (tie && __popc(tied & below) < ties));
        const uint32_t taken = __ballot_sync(0xffffffffu, take);
        if (take) o[done + __popc(taken & below)] = j * 32 + lane;
        done += __popc(taken);
        ties -= __popc(tied) < ties ? __popc(tied) : ties;
    }
    for (int i = done + lane; i < topk; i += 32) o[i] = -1;
}

template <int PER, typename Rows>
__global__ void __launch_bounds__(128) topk_warp_kernel(const uint64_t *keys, int32_t *out, int64_t rows, int topk, Rows of) {
    const uint32_t r = blockIdx.x * 4 + threadIdx.x / 32;
    pdl_trigger();
    pdl_wait();
    if (r >= rows) return;
    const int lane = threadIdx.x % 32;
    const int n = (int)of.count(r), k = topk < n ? topk : n;
    const uint64_t *row = keys + (int64_t)r * of.stride();
    uint64_t key[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) key[j] = j * 32 + lane < n ? row[j * 32 + lane] : 0;
    topk_of_warp<PER>(key, n, k, topk, out + of.out_row(r) * topk);
}

// One warp per row over fp32 scores: the topk-th largest by halving the interval of the scores' integers (about ten
// counts: any value between the topk-th and the next will do), the border again in 64 bits where it is too close.
// 65536 rows of up to 128 blocks: 60 us, 640 instructions a row at 2.5 a clock (64 steps over 64-bit keys: 65 us, behind
// scores that took 159 us in 64 bits where these take 22).
template <int PER, typename T>
__global__ void __launch_bounds__(128, PER <= 4 ? 8 : 1) select_rows_kernel(const T *q, const T *bounds, const float *scores, const float *q_norms, const float *block_norms,
                                                          int32_t *out, int64_t rows, int topk, int64_t H, int64_t D, RowsOfBlocks of) {
    const uint32_t r = blockIdx.x * 4 + threadIdx.x / 32;
    pdl_trigger();
    pdl_wait();
    if (r >= rows) return;
    const int lane = threadIdx.x % 32, bh = (int)(r % (uint32_t)(of.B * of.Hkv)), G = (int)H / of.Hkv;
    const int64_t s = of.query(r), b = bh / of.Hkv, h = bh - b * of.Hkv;
    const int own = (int)s / of.block, n = of.causal ? own + 1 : of.nb, k = topk < n ? topk : n;
    const float *row = scores + (int64_t)r * of.nb;
    const float q_norm = q_norms[r];
    uint32_t key[PER];
    float size = 0.f;
    bool odd = false;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int i = j * 32 + lane;
        key[j] = 0;
        if (i < n) {
            const float x = row[i], y = block_norms[(b * of.Hkv + h) * of.nb + i];
            key[j] = i == own ? 0xffffffffu : key32_of(x);
            if (i != own) {                        // its score decides nothing
                size = fmaxf(size, y);
                odd |= !(fabsf(x) < INFINITY && y < INFINITY);
            }
        }
    }
    int32_t *o = out + ((b * of.S + s) * of.Hkv + h) * topk;
    uint32_t cut = 0;                       // taken: key >= cut
    bool close = false;
    if (k < n) {
        if (k == 1) {
            cut = 0xffffffffu;
        } else {
            uint32_t lo = 0xffffffffu, hi = 0;
#pragma unroll
            for (int j = 0; j < PER; ++j)
                if (j * 32 + lane < n && key[j] != 0xffffffffu) { lo = min(lo, key[j]); hi = max(hi, key[j]); }
            lo = __reduce_min_sync(0xffffffffu, lo);
            hi = __reduce_max_sync(0xffffffffu, hi) + 1;
            bool met = false;               // count(key >= lo) == k, else it is more and count(key >= hi) is less
            while (hi - lo > 1) {
                const uint32_t mid = lo + (hi - lo) / 2;
                int c = 0;
#pragma unroll
                for (int j = 0; j < PER; ++j) c += key[j] >= mid;
                c = __reduce_add_sync(0xffffffffu, c);
                if (c >= k) lo = mid; else hi = mid;
                met = c == k;
                if (met) break;
            }
            cut = lo;
            size = fmaxf(size, 0.f);
#pragma unroll
            for (int x = 16; x > 0; x >>= 1) size = fmaxf(size, __shfl_xor_sync(0xffffffffu, size, x));
            odd = __any_sync(0xffffffffu, odd);
            // A product step adds 16 products to the accumulator; aligned to the largest and cut at 24 bits, each of the
            // 17 terms may lose 2^-23 of the largest: 2.1e-6 of the terms' size per step.  Squares and terms below the least
            // normal number, 1.2e-38, may be lost altogether: up to 2e-18 of a norm of 128 columns, 2.1e-37 of a step.
            const float eps = (float)(2 * G * ((D + 15) / 16) + 1) * (2.1e-6f * (q_norm + (float)G * 2e-18f) * (size + 2e-18f) + 2.1e-37f);
            // the least that is taken and the most that is not
            uint32_t in = 0xffffffffu, not_in = 0;
#pragma unroll
            for (int j = 0; j < PER; ++j)
                if (j * 32 + lane < n) { if (key[j] >= cut) in = min(in, key[j]); else not_in = max(not_in, key[j]); }
            in = __reduce_min_sync(0xffffffffu, in);
            not_in = __reduce_max_sync(0xffffffffu, not_in);
            odd |= !(eps < INFINITY);
            const float kth = of_key32(in);
            close = odd || !met || !(kth - of_key32(not_in) > 2.f * eps);
            if (close) {
                // 64-bit keys: certain ones highest, hopeless ones lowest, the border by its scores
                uint64_t exact[PER];
#pragma unroll
                for (int j = 0; j < PER; ++j) {
                    const int i = j * 32 + lane;
                    const float x = of_key32(key[j]);
                    const bool sure = i == own || (!odd && x > kth + 2.f * eps);
                    exact[j] = i < n && sure ? kOwnKey : 0;
                    uint32_t border = __ballot_sync(0xffffffffu, i < n && !sure && (odd || x >= kth - 2.f * eps));
                    while (border) {
                        const int who = __ffs(border) - 1;
                        border &= border - 1;
                        const T *low = bounds + ((b * of.nb + j * 32 + who) * 2 * of.Hkv + h) * D, *high = low + of.Hkv * D;
                        double t = 0;
                        for (int d = lane; d < D; d += 32) {
                            double u = 0, w = 0;
                            for (int g = 0; g < G; ++g) {
                                const double y = (double)Elem<T>::to_f(q[((b * of.S + s) * H + h * G + g) * D + d]);
                                if (y > 0) u += y; else w += y;
                            }
                            t += u * (double)Elem<T>::to_f(high[d]) + w * (double)Elem<T>::to_f(low[d]);
                        }
#pragma unroll
                        for (int x2 = 16; x2 > 0; x2 >>= 1) t += __shfl_xor_sync(0xffffffffu, t, x2);
                        if (lane == who) {
                            if (!(fabs(t) < INFINITY)) t = score_by_terms(q + ((b * of.S + s) * H + h * G) * D, low, high, G, (int)D);
                            exact[j] = key_of(t);
                        }
                    }
                }
                topk_of_warp<PER>(exact, n, k, topk, o);
                return;
            }
        }
    }
    int done = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const bool take = j * 32 + lane < n && key[j] >= cut;
        const uint32_t taken = __ballot_sync(0xffffffffu, take);
        if (take) o[done + __popc(taken & ((1u << lane) - 1))] = j * 32 + lane;
        done += __popc(taken);
    }
    for (int i = done + lane; i < topk; i += 32) o[i] = -1;
}

// One CTA per row of any length: THREADS x PER keys in registers, the rest read again for every bit.
template <int THREADS> __device__ __forceinline__ int block_sum(int x, int *of_warp) {
    x = __reduce_add_sync(0xffffffffu, x);
    __syncthreads();
    if (threadIdx.x % 32 == 0) of_warp[threadIdx.x / 32] = x;
    __syncthreads();
    return __reduce_add_sync(0xffffffffu, threadIdx.x % 32 < THREADS / 32 ? of_warp[threadIdx.x % 32] : 0);
}

// The k largest of n keys, k < n or not, by a whole CTA.
template <int THREADS> __device__ void topk_of_row(const uint64_t *row, int64_t n, int topk, int32_t *o, int *of_warp, int *tied_of) {
    constexpr int PER = 16;
    const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
    const int k = topk < n ? topk : (int)n;
    uint64_t key[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) key[j] = j * THREADS + tid < n ? row[j * THREADS + tid] : 0;
    auto count = [&](auto &&test) {
        int c = 0;
#pragma unroll
        for (int j = 0; j < PER; ++j) c += test(key[j]) && j * THREADS + tid < n;
        for (int64_t i = (int64_t)PER * THREADS + tid; i < n; i += THREADS) c += test(row[i]);
        return block_sum<THREADS>(c, of_warp);
    };
    uint64_t cut = 0;
    if (k < n)
        for (int bit = 63; bit >= 0; --bit) {
            const uint64_t want = cut | (1ull << bit);
            const int c = count([&](uint64_t x) { return x >= want; });
            if (c >= k) cut = want;
            if (c == k) break;
        }
    int ties = k - count([&](uint64_t x) { return x > cut; }), done = 0;
    for (int64_t base = 0; base < n; base += THREADS) {
        const int64_t i = base + tid;
        const uint64_t x = i < n ? row[i] : 0;
        const bool tie = i < n && x == cut;
        // most stretches of a long row hold nothing that is taken
        if (!__syncthreads_or(i < n && x >= cut)) continue;
        const uint32_t tied = __ballot_sync(0xffffffffu, tie), below = (1u << lane) - 1;
        if (lane == 0) tied_of[warp] = __popc(tied);
        __syncthreads();
        int before = 0, all = 0;
        for (int w = 0; w < THREADS / 32; ++w) { if (w < warp) before += tied_of[w]; all += tied_of[w]; }
        const bool take = i < n && (x > cut || (tie && before + __popc(tied & below) < ties));
        const uint32_t taken = __ballot_sync(0xffffffffu, take);
        if (lane == 0) of_warp[warp] = __popc(taken);
        __syncthreads();
        int at = done, total = 0;
        for (int w = 0; w < THREADS / 32; ++w) { if (w < warp) at += of_warp[w]; total += of_warp[w]; }
        if (take) o[at + __popc(taken & below)] = (int32_t)i;
        done += total;
        ties -= all < ties ? all : ties;
    }
    for (int i = done + tid; i < topk; i += THREADS) o[i] = -1;
}

template <int THREADS, typename Rows>
__global__ void __launch_bounds__(THREADS) topk_block_kernel(const uint64_t *keys, int32_t *out, int topk, Rows of) {
    __shared__ int of_warp[32], tied_of[32];
    const uint32_t r = blockIdx.x;
    pdl_trigger();
    pdl_wait();
    topk_of_row<THREADS>(keys + (int64_t)r * of.stride(), of.count(r), topk, out + of.out_row(r) * topk, of_warp, tied_of);
}

// ---- the topk pages of a row: one CTA -------------------------------------------------------------------------------
// 1. Every thread takes the largest fp32 score of its share of the pages; the (topk - 1)-th largest of those maxima is
//    a floor under the (topk - 1)-th largest score (the token's own page is taken anyway), so no page more than 2 eps
//    below it can be chosen.  With 256 or 1024 threads and few pages wanted, little more than topk pages remain.
// 2. Of the remaining pages, up to kCandidates, those more than 2 eps above or below the wanted rank's score are decided;
//    the others, where there are more of them than places, are scored again in 64 bits, one warp each.
// 3. Each candidate counts the candidates that beat it; the winners count the winners before them: their place.
// Rows where more remain (many equal pages; topk above the number of threads) are scored in 64 bits throughout, by the
// same warps, and searched bit by bit.
constexpr int kCandidates = 1024;

// LP > 0: the CTA scores its row's pages itself first (rows enough to fill the GPU with one CTA each).
template <typename T, int THREADS, int LP, int NV>
__global__ void __launch_bounds__(THREADS, THREADS == 512 ? 2 : 1) select_pages_kernel(PagedView c, const T *bounds, const T *q, int64_t q_stride, int64_t H, int64_t Hkv, int64_t D,
                                                               const int32_t *lengths, float2 *scores, int32_t *out, int topk, int *status) {
    constexpr int W = Vec16<T>::N;
    const int64_t b = blockIdx.y, h = blockIdx.x, G = H / Hkv, row = b * Hkv + h;
    const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32, vecs = (int)D / W;
    __shared__ double up[256], down[256];
    __shared__ uint64_t key[kCandidates];
    __shared__ int page_of[kCandidates];
    __shared__ float score_of[kCandidates], s_kth;
    __shared__ int of_warp[32], tied_of[32], s_count;
    __shared__ uint32_t s_cut;
    __shared__ float f_warp[32];
    pdl_trigger();
    pdl_wait();
    const int64_t len = lengths[b];
    const int64_t held = len <= 0 ? 0 : ((len - 1) >> c.page_shift) + 1;
    const int n = (int)(held < c.width ? held : c.width);
    int32_t *o = out + row * topk;
    if (n <= topk) {
        for (int i = tid; i < topk; i += THREADS) o[i] = i < n ? i : -1;
        return;
    }
    // the token's own page is in (where the table reaches it); `want` of the `others` before it
    const int others = held <= c.width ? n - 1 : n, want = topk - (n - others);
    for (int d = tid; d < D; d += THREADS) {
        double u = 0, w = 0;
        for (int64_t g = 0; g < G; ++g) {
            const double y = (double)Elem<T>::to_f(q[b * q_stride + (h * G + g) * D + d]);
            if (y > 0) u += y; else w += y;
        }
        up[d] = u; down[d] = w;
    }
    if (LP > 0) {
        score_pages<T, LP ? LP : 32, NV>(c, bounds, q + b * q_stride, H, Hkv, D, b, h, n, 0, THREADS / (LP ? LP : 32), scores + row * c.width);
        __syncthreads();
    }
    const float2 *mine = scores + row * c.width;
    float best = -INFINITY, size = 0.f;
    bool odd = false;
    for (int i = tid; i < others; i += THREADS) {
        const float2 x = mine[i];
        best = fmaxf(best, x.x);
        size = fmaxf(size, x.y);
        odd |= !(fabsf(x.x) < INFINITY && x.y < INFINITY);
    }
    if (tid == 0) s_count = 0;
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) size = fmaxf(size, __shfl_xor_sync(0xffffffffu, size, x));
    if (lane == 0) f_warp[warp] = size;
    odd = __syncthreads_or(odd);
    size = f_warp[lane % (THREADS / 32)];
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) size = fmaxf(size, __shfl_xor_sync(0xffffffffu, size, x));
    // a lane adds up to 32 products, the lanes 5 times; the weights are rounded (G times): 2^-24 each of the terms' sizes
    const float eps = (float)(64 + G) * 5.9604645e-8f * size + 1e-42f;
    // The want-th largest of the threads' maxima, by one warp halving their interval: counts without a barrier (16 warps
    // that searched bit by bit waited at 64 barriers, a quarter of the kernel).
    uint32_t *maxima = reinterpret_cast<uint32_t *>(page_of);        // THREADS of them
    maxima[tid] = tid < others ? key32_of(best) : 0;
    __syncthreads();
    if (warp == 0) {
        uint32_t k32[THREADS / 32], lo = 0xffffffffu, hi = 0;
#pragma unroll
        for (int j = 0; j < THREADS / 32; ++j) {
            k32[j] = maxima[j * 32 + lane];
            if (k32[j]) { lo = min(lo, k32[j]); hi = max(hi, k32[j]); }
        }
        lo = __reduce_min_sync(0xffffffffu, lo);
        hi = __reduce_max_sync(0xffffffffu, hi) + 1;
        // count(>= hi) = 0; count(>= lo) is the number of maxima: a search is of use where that reaches want
        int c = 0;
#pragma unroll
        for (int j = 0; j < THREADS / 32; ++j) c += k32[j] > 0;
        c = __reduce_add_sync(0xffffffffu, c);
        if (want < 1 || c < want) lo = 0;
        else
            while (hi - lo > 1 && c != want) {
                const uint32_t mid = lo + (hi - lo) / 2;
                int x = 0;
#pragma unroll
                for (int j = 0; j < THREADS / 32; ++j) x += k32[j] >= mid;
                x = __reduce_add_sync(0xffffffffu, x);
                if (x >= want) { lo = mid; c = x; } else hi = mid;
            }
        if (lane == 0) s_cut = lo;
    }
    __syncthreads();
    const uint32_t cut = s_cut;
    // cut 0: fewer maxima than wanted.  cut is at or below the want-th maximum: at worst a lower floor.
    const float floor = cut == 0 || odd ? -INFINITY : of_key32(cut) - 2.f * eps;
    // 64-bit score of a page, by a warp
    auto exact = [&](int p) {
        const int64_t phys = physical_page(c, b, p, status);
        if (phys < 0) return (uint64_t)0;
        double s = 0;
        for (int v = lane; v < 2 * vecs; v += 32) {
            const bool high = v >= vecs;
            const int col = (high ? v - vecs : v) * W;
            float x[W];
            Vec16<T>::unpack(__ldg(reinterpret_cast<const uint4 *>(bounds + ((phys * 2 + high) * Hkv + h) * D + col)), x);
            const double *w = high ? up : down;
#pragma unroll
            for (int j = 0; j < W; ++j) s += w[col + j] * (double)x[j];
        }
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
        if (!(fabs(s) < INFINITY)) {
            const T *low = bounds + (phys * 2 * Hkv + h) * D;
            s = score_by_terms(q + b * q_stride + h * G * D, low, low + Hkv * D, G, (int)D);
        }
        return key_of(s);
    };
    if (want > 0)
        for (int i = tid; i < others; i += THREADS)
            if (const float x = mine[i].x; odd || x >= floor) {
                const int at = atomicAdd(&s_count, 1);       // the order in the list does not matter: ranks are counted
                if (at < kCandidates) { page_of[at] = i; score_of[at] = x; }
            }
    __syncthreads();
    const int m = s_count;
    if (m <= kCandidates) {
        // the score at the wanted rank, in fp32
        if (!odd)
            for (int i = tid; i < m; i += THREADS) {
                const float x = score_of[i];
                const int p = page_of[i];
                int before = 0;
#pragma unroll 8
                for (int j = 0; j < m; ++j) before += score_of[j] > x || (score_of[j] == x && page_of[j] < p);
                if (before == want - 1) s_kth = x;
            }
        __syncthreads();
        const float kth = odd || m == 0 ? 0.f : s_kth;
        int sure = 0, near = 0;
        for (int i = tid; i < m; i += THREADS) {
            const float x = score_of[i];
            const bool above = !odd && x > kth + 2.f * eps, below = !odd && x < kth - 2.f * eps;
            sure += above;
            near += !above && !below;
            key[i] = above ? kOwnKey : below ? 0 : kOwnKey - 1;
        }
        sure = block_sum<THREADS>(sure, of_warp);
        near = block_sum<THREADS>(near, of_warp);
        __syncthreads();
        if (sure + near > want) {
            for (int i = warp; i < m; i += THREADS / 32) {
                if (key[i] != kOwnKey - 1) continue;
                const uint64_t k = exact(page_of[i]);
                if (lane == 0) key[i] = k;
            }
            __syncthreads();
        }
        // rank of each candidate, then (marked by a set sign of its page) its place among the winners
        bool wins[(kCandidates + THREADS - 1) / THREADS];
#pragma unroll
        for (int y = 0; y < (kCandidates + THREADS - 1) / THREADS; ++y) {
            const int i = y * THREADS + tid;
            wins[y] = false;
            if (i < m) {
                const uint64_t k = key[i];
                const int p = page_of[i];
                int before = 0;
#pragma unroll 8
                for (int j = 0; j < m; ++j) before += key[j] > k || (key[j] == k && page_of[j] < p);
                wins[y] = before < want;
            }
        }
        __syncthreads();
#pragma unroll
        for (int y = 0; y < (kCandidates + THREADS - 1) / THREADS; ++y) {
            const int i = y * THREADS + tid;
            if (i < m && !wins[y]) page_of[i] = INT_MAX;
        }
        __syncthreads();
#pragma unroll
        for (int y = 0; y < (kCandidates + THREADS - 1) / THREADS; ++y) {
            const int i = y * THREADS + tid;
            if (i < m && wins[y]) {
                const int p = page_of[i];
                int before = 0;
#pragma unroll 8
                for (int j = 0; j < m; ++j) before += page_of[j] < p;
                o[before] = p;
            }
        }
        if (tid == 0 && others < n) o[want] = others;
        return;
    }
    // everything in 64 bits, over the fp32 scores
    uint64_t *keys = reinterpret_cast<uint64_t *>(scores + row * c.width);
    for (int i = warp; i < n; i += THREADS / 32) {
        const uint64_t k = i == held - 1 ? kOwnKey : exact(i);
        if (lane == 0) keys[i] = k;
    }
    __syncthreads();
    topk_of_row<THREADS>(keys, n, topk, o, of_warp, tied_of);
}

template <typename Rows>
int launch_topk(const uint64_t *keys, int32_t *out, int64_t rows, int64_t most, int64_t topk, const Rows &of, cudaStream_t s) {
    const unsigned grid = (unsigned)((rows + 3) / 4);
    cudaError_t e;
    if (most <= 128) e = launch_after(topk_warp_kernel<4, Rows>, dim3(grid), dim3(128), 0, s, keys, out, rows, (int)topk, of);
    else if (most <= 512) e = launch_after(topk_warp_kernel<16, Rows>, dim3(grid), dim3(128), 0, s, keys, out, rows, (int)topk, of);
    else if (most <= kWarpRow) e = launch_after(topk_warp_kernel<32, Rows>, dim3(grid), dim3(128), 0, s, keys, out, rows, (int)topk, of);
    else e = launch_after(topk_block_kernel<1024, Rows>, dim3((unsigned)rows), dim3(1024), 0, s, keys, out, (int)topk, of);
    return e == cudaSuccess ? MAT_OK : cuda_fail(e, "launching the selection");
}

size_t align256(size_t x) { return (x + 255) / 256 * 256; }

// Queries whose scores are held at a time: at most about 64 MiB of keys, in steps of a score tile.
int64_t rows_at_a_time(int64_t B, int64_t S, int64_t Hkv, int64_t nb) {
    int64_t n = (64ll << 20) / (B * Hkv * nb * 8) / 64 * 64;
    if (n < 64) n = 64;
    return n < S ? n : S;
}

int check_select(int64_t B, int64_t S, int64_t H, int64_t Hkv, int64_t D, int dtype, int64_t block, int64_t topk) {
    if (dtype != MAT_F32 && dtype != MAT_BF16 && dtype != MAT_F16) return fail(MAT_ERR_INVALID, "unknown dtype %d", dtype);
    if (B < 1 || S < 1 || H < 1 || Hkv < 1 || D < 1) return fail(MAT_ERR_INVALID, "all tensor dimensions must be > 0");
    if (H % Hkv) return fail(MAT_ERR_INVALID, "H = %lld query heads do not divide over H_kv = %lld key heads", (long long)H, (long long)Hkv);
    if (D % 8 || D > 128) return fail(MAT_ERR_UNSUPPORTED, "block selection takes head widths that are multiples of 8 up to 128, got %lld", (long long)D);
    if (block < 16 || block > 128 || block % 16) return fail(MAT_ERR_UNSUPPORTED, "block must be a multiple of 16 from 16 to 128, got %lld", (long long)block);
    if (topk < 1 || topk > 1024) return fail(MAT_ERR_UNSUPPORTED, "topk must be in [1, 1024], got %lld", (long long)topk);
    if (B > 65535 || Hkv > 65535 || B * Hkv > 65535) return fail(MAT_ERR_UNSUPPORTED, "B * H_kv must be at most 65535");
    if (H > INT_MAX || S > (1ll << 30) / block * block) return fail(MAT_ERR_UNSUPPORTED, "the sequence is too long");
    return MAT_OK;
}

// 16-bit rows of up to kWarpRow blocks: fp32 scores on the tensor cores, one warp per row.
bool scores_in_fp32(int dtype, int64_t nb) { return dtype != MAT_F32 && nb <= kWarpRow; }

struct SelectPlan {
    int64_t nb, step;          // blocks, queries whose scores are held at a time
    size_t norms, q_norms, scores, total;
};

SelectPlan select_plan(int64_t B, int64_t S, int64_t Hkv, int64_t D, int dtype, int64_t block) {
    SelectPlan p;
    p.nb = (S + block - 1) / block;
    p.step = rows_at_a_time(B, S, Hkv, p.nb);
    p.norms = align256((size_t)B * p.nb * 2 * Hkv * D * dtype_size(dtype));      // the blocks' bounds lie first
    p.q_norms = p.norms + align256((size_t)B * p.nb * Hkv * 4);
    p.scores = p.q_norms + align256((size_t)p.step * B * Hkv * 4);
    p.total = p.scores + (size_t)p.step * B * Hkv * p.nb * (scores_in_fp32(dtype, p.nb) ? 4 : 8);
    return p;
}

template <typename T, int DP>
cudaError_t launch_scores_mma(dim3 grid, cudaStream_t s, const T *q, const T *bounds, float *scores, float *norms, int64_t S, int64_t H, int64_t Hkv,
                              int64_t D, int64_t nb, int block, int causal, int64_t s0, int64_t s1) {
    const size_t smem = 64 * (DP + 8) * sizeof(T);
    if (ensure_dynamic_smem((const void *)block_scores_mma_kernel<T, DP>, smem, "shared memory of the block scores")) return cudaErrorInvalidValue;
    return launch_after(block_scores_mma_kernel<T, DP>, grid, dim3(128), smem, s, q, bounds, scores, norms, S, H, Hkv, D, nb, block, causal, s0, s1);
}

template <typename T>
int select_in_fp32(const T *q, const T *bounds, int64_t B, int64_t S, int64_t H, int64_t Hkv, int64_t D, int64_t block, int64_t topk, int causal,
                   int32_t *blocks, char *ws, const SelectPlan &p, cudaStream_t s) {
    float *norms = (float *)(ws + p.norms), *q_norms = (float *)(ws + p.q_norms), *scores = (float *)(ws + p.scores);
    const int64_t all = B * p.nb * Hkv;
    cudaError_t e = launch_after(block_norms_kernel<T>, dim3((unsigned)((all + 3) / 4)), dim3(128), 0, s, bounds, norms, all, p.nb, Hkv, D);
    for (int64_t s0 = 0; s0 < S && e == cudaSuccess; s0 += p.step) {
        const int64_t s1 = s0 + p.step < S ? s0 + p.step : S, seen = causal ? (s1 - 1) / block + 1 : p.nb, rows = (s1 - s0) * B * Hkv;
        const dim3 grid((unsigned)((seen + 63) / 64), (unsigned)((s1 - s0 + 63) / 64), (unsigned)(B * Hkv));
        e = D <= 64 ? launch_scores_mma<T, 64>(grid, s, q, bounds, scores, q_norms, S, H, Hkv, D, p.nb, (int)block, causal, s0, s1)
                    : launch_scores_mma<T, 128>(grid, s, q, bounds, scores, q_norms, S, H, Hkv, D, p.nb, (int)block, causal, s0, s1);
        if (e != cudaSuccess) break;
        const RowsOfBlocks of{(int)B, (int)S, (int)Hkv, (int)p.nb, (int)s0, (int)block, causal};
        const dim3 ctas((unsigned)((rows + 3) / 4));
#define SELECT_ROWS(PER) e = launch_after(select_rows_kernel<PER, T>, ctas, dim3(128), 0, s, q, bounds, scores, q_norms, norms, blocks, rows, (int)topk, H, D, of)
        if (seen <= 128) SELECT_ROWS(4);
        else if (seen <= 256) SELECT_ROWS(8);
        else if (seen <= 512) SELECT_ROWS(16);
        else SELECT_ROWS(32);
#undef SELECT_ROWS
    }
    return e == cudaSuccess ? MAT_OK : cuda_fail(e, "launching the block selection");
}
template <>
int select_in_fp32<float>(const float *, const float *, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int, int32_t *, char *,
                          const SelectPlan &, cudaStream_t) {
    return fail(MAT_ERR_UNSUPPORTED, "fp32 inputs are scored in 64 bits");
}

template <typename T>
int run_select_blocks(const T *q, const T *k, int64_t B, int64_t S, int64_t H, int64_t Hkv, int64_t D, int dtype, int64_t block, int64_t topk,
                      int causal, int32_t *blocks, void *ws, cudaStream_t s) {
    const SelectPlan p = select_plan(B, S, Hkv, D, dtype, block);
    T *bounds = (T *)ws;
    block_bounds_kernel<T><<<dim3((unsigned)p.nb, (unsigned)((Hkv * D + 32 * Vec16<T>::N - 1) / (32 * Vec16<T>::N)), (unsigned)B), 256, 0, s>>>(k, bounds, S, p.nb, (int)block, Hkv * D);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return cuda_fail(e, "launching the block bounds");
    if (scores_in_fp32(dtype, p.nb)) return select_in_fp32<T>(q, bounds, B, S, H, Hkv, D, block, topk, causal, blocks, (char *)ws, p, s);
    uint64_t *keys = (uint64_t *)((char *)ws + p.scores);
    for (int64_t s0 = 0; s0 < S; s0 += p.step) {
        const int64_t s1 = s0 + p.step < S ? s0 + p.step : S;
        const int64_t seen = causal ? (s1 - 1) / block + 1 : p.nb;
        dim3 grid((unsigned)((seen + 63) / 64), (unsigned)((s1 - s0 + 63) / 64), (unsigned)(B * Hkv));
        e = launch_after(block_scores_kernel<T>, grid, dim3(256), 0, s, q, (const T *)bounds, keys, S, H, Hkv, D, p.nb, (int)block, causal, s0, s1);
        if (e != cudaSuccess) return cuda_fail(e, "launching the block scores");
        RowsOfBlocks of{(int)B, (int)S, (int)Hkv, (int)p.nb, (int)s0, (int)block, causal};
        if (int rc = launch_topk(keys, blocks, (s1 - s0) * B * Hkv, seen, topk, of, s)) return rc;
    }
    return MAT_OK;
}

int check_paged_select(const mat_paged_cache *c, int64_t B, int64_t H, int64_t width, int64_t topk) {
    if (!c->key_bounds) return fail(MAT_ERR_INVALID, "selecting pages needs the cache's key_bounds");
    if (H < c->H_kv || H % c->H_kv) return fail(MAT_ERR_INVALID, "H = %lld query heads do not divide over H_kv = %lld key heads", (long long)H, (long long)c->H_kv);
    if (topk < 1 || topk > 65536) return fail(MAT_ERR_UNSUPPORTED, "topk must be in [1, 65536], got %lld", (long long)topk);
    (void)B; (void)width;
    return MAT_OK;
}

template <typename T>
int run_select_pages(const mat_paged_cache *c, const PagedView &v, const T *q, int64_t q_stride, int64_t B, int64_t H, const int32_t *lengths,
                     int64_t topk, int32_t *pages, float2 *scores, int *status, cudaStream_t s) {
    const int vecs = 2 * (int)c->D / Vec16<T>::N;            // of one page and head
    const int lp = vecs <= 8 ? 8 : vecs <= 32 ? 16 : 32;
    const T *bounds = (const T *)c->key_bounds;
    const dim3 rows((unsigned)c->H_kv, (unsigned)B);
    cudaError_t e;
    if (B * c->H_kv >= 148) {
#define SELECT_PAGES(LP, NV) select_pages_kernel<T, 512, LP, NV><<<rows, 512, 0, s>>>(v, bounds, q, q_stride, H, c->H_kv, c->D, lengths, scores, pages, (int)topk, status)
        if (lp == 8) SELECT_PAGES(8, 1);
        else if (vecs <= 16) SELECT_PAGES(16, 1);
        else if (vecs <= 32) SELECT_PAGES(16, 2);
        else if (vecs <= 64) SELECT_PAGES(32, 2);
        else SELECT_PAGES(32, 4);
#undef SELECT_PAGES
        e = cudaGetLastError();
        return e == cudaSuccess ? MAT_OK : cuda_fail(e, "launching the selection");
    }
    int64_t gx = (v.width * lp + 4 * 256 - 1) / (4 * 256);
    const int64_t cap = 148 * 8 / (B * c->H_kv) + 1;         // enough CTAs to fill the GPU; each walks several pages
    if (gx > cap) gx = cap;
    const dim3 grid((unsigned)gx, (unsigned)c->H_kv, (unsigned)B);
#define PAGE_SCORES(LP, NV) page_scores_kernel<T, LP, NV><<<grid, 256, 0, s>>>(v, bounds, q, q_stride, H, c->H_kv, c->D, lengths, scores)
    if (lp == 8) PAGE_SCORES(8, 1);
    else if (vecs <= 16) PAGE_SCORES(16, 1);
    else if (vecs <= 32) PAGE_SCORES(16, 2);
    else if (vecs <= 64) PAGE_SCORES(32, 2);
    else PAGE_SCORES(32, 4);
#undef PAGE_SCORES
    e = cudaGetLastError();
    if (e != cudaSuccess) return cuda_fail(e, "launching the page scores");
    // few pages per row: a small CTA, whose steps wait for fewer warps (1000 pages x 8 heads, 16 wanted: 6.9 us with 256 threads,
    // 8.9 with 1024; 64 of 512 pages x 128 rows: 15.5 and 15.7; 128 of 2048 pages: 25 and 22)
    if (v.width <= 2048 && topk <= 128) e = launch_after(select_pages_kernel<T, 256, 0, 1>, rows, dim3(256), 0, s, v, bounds, q, q_stride, H, c->H_kv, c->D, lengths, scores, pages, (int)topk, status);
    else e = launch_after(select_pages_kernel<T, 1024, 0, 1>, rows, dim3(1024), 0, s, v, bounds, q, q_stride, H, c->H_kv, c->D, lengths, scores, pages, (int)topk, status);
    return e == cudaSuccess ? MAT_OK : cuda_fail(e, "launching the selection");
}

}  // namespace
}  // namespace mat

using namespace mat;

extern "C" size_t mat_select_blocks_workspace_bytes(int64_t B, int64_t S, int64_t H, int64_t H_kv, int64_t D, int dtype, int64_t block, int64_t topk) {
    if (check_select(B, S, H, H_kv, D, dtype, block, topk)) return 0;
    return select_plan(B, S, H_kv, D, dtype, block).total;
}

extern "C" int mat_select_blocks(const void *q, const void *k, int64_t B, int64_t S, int64_t H, int64_t H_kv, int64_t D, int dtype, int64_t block,
                                 int64_t topk, int causal, int32_t *blocks, void *workspace, size_t workspace_bytes, void *stream) {
    if (int rc = check_select(B, S, H, H_kv, D, dtype, block, topk)) return rc;
    if (!q || !k || !blocks) return fail(MAT_ERR_INVALID, "q, k and blocks must be non-NULL");
    if (((uintptr_t)q | (uintptr_t)k) % 16) return fail(MAT_ERR_INVALID, "q and k must be 16-byte aligned");
    const size_t need = mat_select_blocks_workspace_bytes(B, S, H, H_kv, D, dtype, block, topk);
    if (!workspace || workspace_bytes < need || (uintptr_t)workspace % 256)
        return fail(MAT_ERR_WORKSPACE, "workspace of %zu bytes (256-byte aligned) required, got %zu", need, workspace ? workspace_bytes : (size_t)0);
    note_kernel("select_blocks");
    cudaStream_t s = (cudaStream_t)stream;
    causal = causal != 0;
    switch (dtype) {
        case MAT_F32: return run_select_blocks((const float *)q, (const float *)k, B, S, H, H_kv, D, dtype, block, topk, causal, blocks, workspace, s);
        case MAT_BF16: return run_select_blocks((const __nv_bfloat16 *)q, (const __nv_bfloat16 *)k, B, S, H, H_kv, D, dtype, block, topk, causal, blocks, workspace, s);
        default: return run_select_blocks((const __half *)q, (const __half *)k, B, S, H, H_kv, D, dtype, block, topk, causal, blocks, workspace, s);
    }
}

extern "C" size_t mat_paged_select_workspace_bytes(const mat_paged_cache *cache, int64_t B, int64_t H, int64_t table_width, int64_t topk) {
    if (check_paged_cache(cache) || B < 1 || table_width < 1 || check_paged_select(cache, B, H, table_width, topk)) return 0;
    return (size_t)B * cache->H_kv * table_width * 8;
}

extern "C" int mat_paged_select(const mat_paged_cache *cache, const void *q, int64_t q_stride, int64_t B, int64_t H, const int32_t *page_table,
                                int64_t table_width, int64_t table_stride, const int32_t *lengths, int64_t topk, int32_t *pages,
                                void *workspace, size_t workspace_bytes, void *stream) {
    if (int rc = check_paged_cache(cache)) return rc;
    if (int rc = check_page_table(page_table, table_width, table_stride, B)) return rc;
    if (int rc = check_paged_select(cache, B, H, table_width, topk)) return rc;
    if (!q || !lengths || !pages) return fail(MAT_ERR_INVALID, "q, lengths and pages must be non-NULL");
    if ((uintptr_t)q % 16 || q_stride < 0 || q_stride * (int64_t)dtype_size(cache->dtype) % 16)
        return fail(MAT_ERR_INVALID, "q must be 16-byte aligned and its stride a multiple of 16 bytes");
    const size_t need = mat_paged_select_workspace_bytes(cache, B, H, table_width, topk);
    if (!workspace || workspace_bytes < need || (uintptr_t)workspace % 256)
        return fail(MAT_ERR_WORKSPACE, "workspace of %zu bytes (256-byte aligned) required, got %zu", need, workspace ? workspace_bytes : (size_t)0);
    const PagedView v = paged_view(cache, page_table, table_width, table_stride);
    int *status = paged_status_word();
    if (!status) return fail(MAT_ERR_CUDA, "no device status word");
    note_kernel("paged_select");
    cudaStream_t s = (cudaStream_t)stream;
    float2 *scores = (float2 *)workspace;      // and 64-bit keys in their place where a row needs them
    switch (cache->dtype) {
        case MAT_F32: return run_select_pages(cache, v, (const float *)q, q_stride, B, H, lengths, topk, pages, scores, status, s);
        case MAT_BF16: return run_select_pages(cache, v, (const __nv_bfloat16 *)q, q_stride, B, H, lengths, topk, pages, scores, status, s);
        default: return run_select_pages(cache, v, (const __half *)q, q_stride, B, H, lengths, topk, pages, scores, status, s);
    }
}
