// Which blocks of keys a query reads, by a cheap score; over the pages of a paged cache (one new token per sequence) and
// over the blocks of whole sequences (prompts and training).
//
// With lo and hi the smallest and largest key of a block column by column, the G query heads of a key head score it
//     sum_g sum_d max(q_gd lo_d, q_gd hi_d) = sum_d up_d hi_d + down_d lo_d,
//     up_d = sum_g max(q_gd, 0), down_d = sum_g min(q_gd, 0):
// one dot product of 2 D terms whatever G is, and an upper bound of the group's summed q . k over the block's keys.
// Bounds are exact in the keys' type, and scores are formed and compared in 64 bits, so a selection does not depend on
// how the sums are split: two blocks change places only where their true scores agree to about 1e-15.
//
// A score becomes a 64-bit key whose order as an integer is the score's (NaN lowest, the query's own block highest); the
// topk-th largest key is found bit by bit (byte by byte for long rows), ties go to the lower index.
#include <limits.h>

#include "paged.cuh"
#include "pdl.cuh"

namespace mat {
namespace {

constexpr uint64_t kOwnKey = ~0ull;
constexpr int kWarpRow = 1024;      // keys a row may have to be held by one warp's registers

__device__ __forceinline__ uint64_t key_of(double x) {
    if (x != x) return 0;
    const uint64_t u = (uint64_t)__double_as_longlong(x);
    return (u >> 63) ? ~u : u | 0x8000000000000000ull;
}

// ---- bounds of the blocks of whole sequences ------------------------------------------------------------------------
// One CTA per block and 64 bytes x 8 of its columns: 32 vectors of columns, 8 threads each taking every 8th token, four
// tokens in flight.
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
            for (int j = 0; j < W; ++j) { lo[j] = fminf(lo[j], x[j]); hi[j] = fmaxf(hi[j], x[j]); }
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
                m[j] = part ? fmaxf(m[j], y) : fminf(m[j], y);
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
            if (n < nb) keys[((s - s_lo) * gridDim.z + blockIdx.z) * nb + n] = n == s / block ? kOwnKey : key_of(acc[i][j]);
        }
    }
}

// ---- scores of a cache's pages ---------------------------------------------------------------------------------------
// LP lanes share a page: a lane holds the weights of its NV vectors (of the 2 D bounds: smallest keys, then largest) in
// 64 bits in registers and reads four pages' vectors at once.
template <typename T, int LP, int NV>
__global__ void __launch_bounds__(256) page_scores_kernel(PagedView c, const T *bounds, const T *q, int64_t q_stride, int64_t H, int64_t Hkv, int64_t D,
                                                          const int32_t *lengths, uint64_t *keys, int *status) {
    constexpr int W = Vec16<T>::N, GROUPS = 256 / LP, U = NV >= 4 ? 2 : 4;
    const int64_t b = blockIdx.z, h = blockIdx.y, G = H / Hkv;
    pdl_trigger();
    const int64_t len = lengths[b];
    if (len <= 0) return;
    const int64_t held = ((len - 1) >> c.page_shift) + 1;      // pages that hold tokens; the last is the token's own
    const int64_t n = held < c.width ? held : c.width;
    if ((int64_t)blockIdx.x * GROUPS >= n) return;
    const int part = threadIdx.x % LP, vecs = (int)D / W;
    double w[NV][W];
    int64_t off[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int v = i * LP + part;
        const bool high = v >= vecs;
        const int col = (high ? v - vecs : v) * W;
        off[i] = v < 2 * vecs ? (high ? Hkv * D : 0) + h * D + col : -1;
#pragma unroll
        for (int j = 0; j < W; ++j) w[i][j] = 0;
        if (off[i] >= 0)
            for (int64_t g = 0; g < G; ++g) {
                float x[W];
                Vec16<T>::unpack(__ldg(reinterpret_cast<const uint4 *>(q + b * q_stride + (h * G + g) * D + col)), x);
#pragma unroll
                for (int j = 0; j < W; ++j)
                    if ((x[j] > 0) == high) w[i][j] += (double)x[j];       // a NaN lands among the smallest keys' weights
            }
    }
    const int64_t step = (int64_t)gridDim.x * GROUPS;
    // the trip count is the same for all lanes of a warp (they shuffle together): bounded by the CTA's first group
    for (int64_t p0 = (int64_t)blockIdx.x * GROUPS; p0 < n; p0 += U * step) {
        uint4 x[U][NV];
        int64_t phys[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t p = p0 + u * step + threadIdx.x / LP;
            phys[u] = p < n ? physical_page(c, b, p, status) : -1;
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < NV; ++i)
                x[u][i] = phys[u] >= 0 && off[i] >= 0 ? __ldg(reinterpret_cast<const uint4 *>(bounds + phys[u] * 2 * Hkv * D + off[i])) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            double s = 0;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                float y[W];
                Vec16<T>::unpack(x[u][i], y);
#pragma unroll
                for (int j = 0; j < W; ++j) s += w[i][j] * (double)y[j];
            }
#pragma unroll
            for (int o = LP / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
            const int64_t p = p0 + u * step + threadIdx.x / LP;
            if (part == 0 && p < n) keys[(b * Hkv + h) * c.width + p] = p == held - 1 ? kOwnKey : phys[u] < 0 ? 0 : key_of(s);
        }
    }
}

// ---- the topk of a row -----------------------------------------------------------------------------------------------
// Rows of whole sequences: row r = (s - s_lo, b, h), its eligible keys are [0, own] (causal) or [0, nb).
struct RowsOfBlocks {
    int64_t B, S, Hkv, nb, s_lo;
    int block, causal;
    __device__ __forceinline__ int64_t count(int64_t r) const { return causal ? (s_lo + r / (B * Hkv)) / block + 1 : nb; }
    __device__ __forceinline__ int64_t stride() const { return nb; }
    __device__ __forceinline__ int64_t out_row(int64_t r) const {
        const int64_t s = s_lo + r / (B * Hkv), b = r / Hkv % B, h = r % Hkv;
        return (b * S + s) * Hkv + h;
    }
};
// Rows of a cache: row r = (b, h).
struct RowsOfPages {
    const int32_t *lengths;
    int64_t Hkv, width;
    int page_shift;
    __device__ __forceinline__ int64_t count(int64_t r) const {
        const int64_t len = lengths[r / Hkv];
        const int64_t n = len <= 0 ? 0 : ((len - 1) >> page_shift) + 1;
        return n < width ? n : width;
    }
    __device__ __forceinline__ int64_t stride() const { return width; }
    __device__ __forceinline__ int64_t out_row(int64_t r) const { return r; }
};

// One warp per row, its keys in registers.
template <int PER, typename Rows>
__global__ void __launch_bounds__(128) topk_warp_kernel(const uint64_t *keys, int32_t *out, int64_t rows, int topk, Rows of) {
    const int64_t r = (int64_t)blockIdx.x * 4 + threadIdx.x / 32;
    pdl_trigger();
    pdl_wait();
    if (r >= rows) return;
    const int lane = threadIdx.x % 32;
    const int n = (int)of.count(r), k = topk < n ? topk : n;
    const uint64_t *row = keys + r * of.stride();
    uint64_t key[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) key[j] = j * 32 + lane < n ? row[j * 32 + lane] : 0;
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
    int32_t *o = out + of.out_row(r) * topk;
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

// One CTA per row of any length: THREADS x PER keys in registers, the rest read again for every bit.
template <int THREADS> __device__ __forceinline__ int block_sum(int x, int *of_warp) {
    x = __reduce_add_sync(0xffffffffu, x);
    __syncthreads();
    if (threadIdx.x % 32 == 0) of_warp[threadIdx.x / 32] = x;
    __syncthreads();
    return __reduce_add_sync(0xffffffffu, threadIdx.x % 32 < THREADS / 32 ? of_warp[threadIdx.x % 32] : 0);
}

template <int THREADS, int PER, typename Rows>
__global__ void __launch_bounds__(THREADS) topk_block_kernel(const uint64_t *keys, int32_t *out, int topk, Rows of) {
    const int64_t r = blockIdx.x;
    const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
    pdl_trigger();
    pdl_wait();
    const int64_t n = of.count(r);
    const int k = topk < n ? topk : (int)n;
    const uint64_t *row = keys + r * of.stride();
    int32_t *o = out + of.out_row(r) * topk;
    __shared__ int of_warp[32], tied_of[32];
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

template <typename Rows>
int launch_topk(const uint64_t *keys, int32_t *out, int64_t rows, int64_t most, int64_t topk, const Rows &of, cudaStream_t s) {
    const unsigned grid = (unsigned)((rows + 3) / 4);
    cudaError_t e;
    if (most <= 128) e = launch_after(topk_warp_kernel<4, Rows>, dim3(grid), dim3(128), 0, s, keys, out, rows, (int)topk, of);
    else if (most <= 512) e = launch_after(topk_warp_kernel<16, Rows>, dim3(grid), dim3(128), 0, s, keys, out, rows, (int)topk, of);
    else if (most <= kWarpRow) e = launch_after(topk_warp_kernel<32, Rows>, dim3(grid), dim3(128), 0, s, keys, out, rows, (int)topk, of);
    else e = launch_after(topk_block_kernel<1024, 16, Rows>, dim3((unsigned)rows), dim3(1024), 0, s, keys, out, (int)topk, of);
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
    if (B * Hkv > 65535 || B > 65535) return fail(MAT_ERR_UNSUPPORTED, "B * H_kv must be at most 65535");
    if (S > (1ll << 30) / block * block) return fail(MAT_ERR_UNSUPPORTED, "the sequence is too long");
    return MAT_OK;
}

template <typename T>
int run_select_blocks(const T *q, const T *k, int64_t B, int64_t S, int64_t H, int64_t Hkv, int64_t D, int64_t block, int64_t topk,
                      int causal, int32_t *blocks, void *ws, cudaStream_t s) {
    const int64_t nb = (S + block - 1) / block, step = rows_at_a_time(B, S, Hkv, nb);
    T *bounds = (T *)ws;
    uint64_t *keys = (uint64_t *)((char *)ws + align256((size_t)B * nb * 2 * Hkv * D * sizeof(T)));
    block_bounds_kernel<T><<<dim3((unsigned)nb, (unsigned)((Hkv * D + 32 * Vec16<T>::N - 1) / (32 * Vec16<T>::N)), (unsigned)B), 256, 0, s>>>(k, bounds, S, nb, (int)block, Hkv * D);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return cuda_fail(e, "launching the block bounds");
    for (int64_t s0 = 0; s0 < S; s0 += step) {
        const int64_t s1 = s0 + step < S ? s0 + step : S;
        const int64_t seen = causal ? (s1 - 1) / block + 1 : nb;
        dim3 grid((unsigned)((seen + 63) / 64), (unsigned)((s1 - s0 + 63) / 64), (unsigned)(B * Hkv));
        e = launch_after(block_scores_kernel<T>, grid, dim3(256), 0, s, q, (const T *)bounds, keys, S, H, Hkv, D, nb, (int)block, causal, s0, s1);
        if (e != cudaSuccess) return cuda_fail(e, "launching the block scores");
        RowsOfBlocks of{B, S, Hkv, nb, s0, (int)block, causal};
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
                     int64_t topk, int32_t *pages, uint64_t *keys, int *status, cudaStream_t s) {
    const int vecs = 2 * (int)c->D / Vec16<T>::N;            // of one page and head
    const int lp = vecs <= 8 ? 8 : vecs <= 16 ? 16 : 32;
    int64_t gx = (v.width * lp + 4 * 256 - 1) / (4 * 256);
    const int64_t cap = 148 * 8 / (B * c->H_kv) + 1;         // enough CTAs to fill the GPU; each walks several pages
    if (gx > cap) gx = cap;
    const dim3 grid((unsigned)gx, (unsigned)c->H_kv, (unsigned)B);
#define PAGE_SCORES(LP, NV) page_scores_kernel<T, LP, NV><<<grid, 256, 0, s>>>(v, (const T *)c->key_bounds, q, q_stride, H, c->H_kv, c->D, lengths, keys, status)
    if (lp == 8) PAGE_SCORES(8, 1);
    else if (lp == 16) PAGE_SCORES(16, 1);
    else if (vecs <= 32) PAGE_SCORES(32, 1);
    else if (vecs <= 64) PAGE_SCORES(32, 2);
    else PAGE_SCORES(32, 4);
#undef PAGE_SCORES
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return cuda_fail(e, "launching the page scores");
    RowsOfPages of{lengths, c->H_kv, v.width, v.page_shift};
    return launch_topk(keys, pages, B * c->H_kv, v.width, topk, of, s);
}

}  // namespace
}  // namespace mat

using namespace mat;

extern "C" size_t mat_select_blocks_workspace_bytes(int64_t B, int64_t S, int64_t H, int64_t H_kv, int64_t D, int dtype, int64_t block, int64_t topk) {
    if (check_select(B, S, H, H_kv, D, dtype, block, topk)) return 0;
    const int64_t nb = (S + block - 1) / block;
    return align256((size_t)B * nb * 2 * H_kv * D * dtype_size(dtype)) + (size_t)rows_at_a_time(B, S, H_kv, nb) * B * H_kv * nb * 8;
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
        case MAT_F32: return run_select_blocks((const float *)q, (const float *)k, B, S, H, H_kv, D, block, topk, causal, blocks, workspace, s);
        case MAT_BF16: return run_select_blocks((const __nv_bfloat16 *)q, (const __nv_bfloat16 *)k, B, S, H, H_kv, D, block, topk, causal, blocks, workspace, s);
        default: return run_select_blocks((const __half *)q, (const __half *)k, B, S, H, H_kv, D, block, topk, causal, blocks, workspace, s);
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
    uint64_t *keys = (uint64_t *)workspace;
    switch (cache->dtype) {
        case MAT_F32: return run_select_pages(cache, v, (const float *)q, q_stride, B, H, lengths, topk, pages, keys, status, s);
        case MAT_BF16: return run_select_pages(cache, v, (const __nv_bfloat16 *)q, q_stride, B, H, lengths, topk, pages, keys, status, s);
        default: return run_select_pages(cache, v, (const __half *)q, q_stride, B, H, lengths, topk, pages, keys, status, s);
    }
}
