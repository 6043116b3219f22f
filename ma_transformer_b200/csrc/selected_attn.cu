// Attention over selected blocks of keys and its gradients: the C entry points and the lists of the queries that chose a
// block.  The tiles are in selected_tiles.cu.
//
//   forward   o_i = sum_j p_ij v_j, p_ij = exp(scale q_i . k_j - lse_i) over the keys j of the query's blocks
//   backward  delta_i = do_i . o_i, ds_ij = p_ij (do_i . v_j - delta_i),
//             dq_i = scale sum_j ds_ij k_j, dk_j = scale sum_i ds_ij q_i, dv_j = sum_i p_ij do_i
// dk and dv are sums over the queries that chose the key's block, in ascending order: no atomics.
#include <limits.h>

#include <cmath>

#include "paged.cuh"
#include "pdl.cuh"
#include "selected_attn.cuh"

namespace mat {
namespace {

constexpr int kTile = 256;          // queries per tile of the lists
constexpr int kRange = 1024;        // blocks per CTA of the lists: 32 KB of bit masks

// ---- lists: per tile of queries a count per block, then where each run starts, then the entries ----------------------------------------------------------------------------------------------------------
// mask[n][w]: the tile's queries that chose block n, a bit each.  A bit set does not depend on the order of the writers,
// so the lists come out the same every time.
__device__ __forceinline__ int own_limit(const SelProblem &p, int64_t i) {
    return p.causal ? (int)(i / p.block) + 1 : (int)p.nb;
}

// A tile's lists come through shared memory, kStage entries of every query at a time: read one by one from global memory
// they lived off the L1, which the next kernel's waiting CTAs take away (fill: 62 us instead of 19 at 8192 x 8 x 16).
constexpr int kStage = 16;

struct TileLists {
    const SelProblem &p;
    const int32_t *first;       // of the tile's first query
    int rows;                   // queries of the tile that exist
    int (*stage)[kStage + 1];
    __device__ __forceinline__ void load(int s0) {
        __syncthreads();
        const int cnt = min(kStage, (int)p.topk - s0);
        for (int x = threadIdx.x; x < rows * kStage; x += kTile) {
            const int r = x / kStage, c = x % kStage;
            if (c < cnt) stage[r][c] = __ldg(first + (int64_t)r * p.Hkv * p.topk + s0 + c);
        }
        __syncthreads();
    }
    // calls f(block, place in the list) for this thread's entries that count and lie in [n0, n1)
    template <typename F> __device__ __forceinline__ void each(int limit, int n0, int n1, F &&f) {
        int prev = -1;
        for (int s0 = 0; s0 < p.topk; s0 += kStage) {
            load(s0);
            const int cnt = min(kStage, (int)p.topk - s0);
            if ((int)threadIdx.x < rows)
                for (int c = 0; c < cnt; ++c) {
                    const int n = stage[threadIdx.x][c];
                    if (sel_entry_counts(n, prev, limit) && n >= n0 && n < n1) f(n, s0 + c);
                }
        }
    }
};

__device__ __forceinline__ TileLists tile_lists(const SelProblem &p, int64_t tile, int64_t bh, int (*stage)[kStage + 1]) {
    const int64_t b = bh / p.Hkv, h = bh % p.Hkv, i0 = tile * kTile;
    return TileLists{p, p.blocks + ((b * p.S + i0) * p.Hkv + h) * p.topk, (int)min((int64_t)kTile, p.S - i0), stage};
}

__global__ void __launch_bounds__(kTile) lists_count_kernel(const SelProblem p, const SelLists l, int64_t bh0) {
    __shared__ int hist[kRange], stage[kTile][kStage + 1];
    const int64_t tile = blockIdx.x, bh = blockIdx.z;
    const int n0 = blockIdx.y * kRange, n1 = min(n0 + kRange, (int)p.nb), tid = threadIdx.x;
    pdl_trigger();
    for (int i = tid; i < n1 - n0; i += kTile) hist[i] = 0;
    pdl_wait();
    tile_lists(p, tile, bh0 + bh, stage).each(own_limit(p, tile * kTile + tid), n0, n1, [&](int n, int) { atomicAdd(&hist[n - n0], 1); });
    __syncthreads();
    for (int n = n0 + tid; n < n1; n += kTile) l.counts[(bh * l.tiles + tile) * p.nb + n] = hist[n - n0];
}

__global__ void __launch_bounds__(kTile) lists_fill_kernel(const SelProblem p, const SelLists l, int64_t bh0) {
    extern __shared__ int fill_smem[];
    uint32_t (*mask)[kTile / 32] = (uint32_t (*)[kTile / 32])fill_smem;            // [kRange][kTile / 32]
    int *start = fill_smem + kRange * (kTile / 32);                                // [kRange]
    int (*stage)[kStage + 1] = (int (*)[kStage + 1])(start + kRange);              // [kTile][kStage + 1]
    const int64_t tile = blockIdx.x, bh = blockIdx.z;
    const int n0 = blockIdx.y * kRange, n1 = min(n0 + kRange, (int)p.nb), tid = threadIdx.x;
    pdl_trigger();
    for (int i = tid; i < (n1 - n0) * (kTile / 32); i += kTile) (&mask[0][0])[i] = 0;
    pdl_wait();
    for (int i = tid; i < n1 - n0; i += kTile) start[i] = l.base[bh * (p.nb + 1) + n0 + i] + l.counts[(bh * l.tiles + tile) * p.nb + n0 + i];
    const int limit = own_limit(p, tile * kTile + tid);
    TileLists lists = tile_lists(p, tile, bh0 + bh, stage);
    lists.each(limit, n0, n1, [&](int n, int) { atomicOr(&mask[n - n0][tid / 32], 1u << (tid % 32)); });
    __syncthreads();
    int32_t *entries = l.entry + bh * p.S * p.topk;
    const int i = (int)(tile * kTile) + tid;
    lists.each(limit, n0, n1, [&](int n, int s) {
        const uint32_t *m = mask[n - n0];
        int rank = __popc(m[tid / 32] & ((1u << (tid % 32)) - 1));
#pragma unroll
        for (int w = 0; w < kTile / 32 - 1; ++w) rank += w < tid / 32 ? __popc(m[w]) : 0;
        entries[start[n - n0] + rank] = i * (int)p.topk + s;
    });
}

// inclusive sum over the CTA's 1024 threads
__device__ __forceinline__ int block_scan(int x, int *of_warp) {
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();                 // of_warp may still be read from the scan before
    if (lane == 31) of_warp[warp] = x;
    __syncthreads();
    int before = 0;
    for (int w = 0; w < warp; ++w) before += of_warp[w];
    return x + before;
}

// counts of a block's tiles -> offsets within its list; totals of the blocks -> where each list starts, and the items of
// its rows: one CTA per bh
__global__ void __launch_bounds__(1024) lists_base_kernel(SelLists l, int64_t nb, int G, int2 *items, int32_t *item_base, int64_t max_items, int rows_per_item) {
    __shared__ int of_warp[32], carry[2];
    const int64_t bh = blockIdx.x;
    pdl_trigger();
    pdl_wait();
    int entries = 0, before = 0;
    for (int64_t n0 = 0; n0 < nb; n0 += 1024) {
        const int64_t n = n0 + threadIdx.x;
        int x = 0;
        if (n < nb) {
            int32_t *c = l.counts + bh * l.tiles * nb + n;
            for (int64_t t0 = 0; t0 < l.tiles; t0 += 8) {       // eight tiles' counts in flight
                int y[8];
#pragma unroll
                for (int u = 0; u < 8; ++u) y[u] = t0 + u < l.tiles ? c[(t0 + u) * nb] : 0;
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    if (t0 + u < l.tiles) c[(t0 + u) * nb] = x;
                    x += y[u];
                }
            }
        }
        const int sum = block_scan(x, of_warp);
        if (n < nb) l.base[bh * (nb + 1) + n] = entries + sum - x;
        const int mine = (int)(((int64_t)x * G + rows_per_item - 1) / rows_per_item);
        const int isum = block_scan(mine, of_warp);
        if (n < nb) {
            const int at = before + isum - mine;
            item_base[bh * (nb + 1) + n] = at;
            for (int i = 0; i < mine; ++i) items[bh * max_items + at + i] = make_int2((int)n, i * rows_per_item);
        }
        if (threadIdx.x == 1023) { carry[0] = sum; carry[1] = isum; }
        __syncthreads();
        entries += carry[0];
        before += carry[1];
    }
    if (threadIdx.x == 0) {
        l.base[bh * (nb + 1) + nb] = entries;
        item_base[bh * (nb + 1) + nb] = before;
    }
}

int launched(const char *what) {
    cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? MAT_OK : cuda_fail(e, what);
}

int check_selected(int64_t B, int64_t S, int64_t H, int64_t Hkv, int64_t D, int dtype, int64_t block, int64_t topk) {
    if (dtype != MAT_F32 && dtype != MAT_BF16 && dtype != MAT_F16) return fail(MAT_ERR_INVALID, "unknown dtype %d", dtype);
    if (B < 1 || S < 1 || H < 1 || Hkv < 1 || D < 1) return fail(MAT_ERR_INVALID, "all tensor dimensions must be > 0");
    if (H % Hkv) return fail(MAT_ERR_INVALID, "H = %lld query heads do not divide over H_kv = %lld key heads", (long long)H, (long long)Hkv);
    if (D % 8 || D > 128) return fail(MAT_ERR_UNSUPPORTED, "block-selected attention takes head widths that are multiples of 8 up to 128, got %lld", (long long)D);
    if (block < 16 || block > 128 || block % 16) return fail(MAT_ERR_UNSUPPORTED, "block must be a multiple of 16 from 16 to 128, got %lld", (long long)block);
    if (topk < 1 || topk > 1024) return fail(MAT_ERR_UNSUPPORTED, "topk must be in [1, 1024], got %lld", (long long)topk);
    if (B > 65535 || Hkv > 65535 || B * Hkv > 65535) return fail(MAT_ERR_UNSUPPORTED, "B * H_kv must be at most 65535");
    if (S > INT_MAX || H > INT_MAX || S * topk > INT_MAX / (H / Hkv) || S * H > INT_MAX || B * S * H > (int64_t)INT_MAX * 2) return fail(MAT_ERR_UNSUPPORTED, "the sequence is too long for its topk");
    return MAT_OK;
}

}  // namespace

size_t sel_lists_bytes(int64_t pairs, int64_t S, int64_t nb, int64_t topk) {
    const int64_t tiles = (S + kTile - 1) / kTile;
    return sel_align((size_t)pairs * nb * tiles * 4) + sel_align((size_t)pairs * (nb + 1) * 4) + sel_align((size_t)pairs * S * topk * 4);
}

SelLists sel_lists_at(void *ws, int64_t pairs, int64_t S, int64_t nb, int64_t topk) {
    SelLists l;
    l.tiles = (S + kTile - 1) / kTile;
    char *at = (char *)ws;
    l.counts = (int32_t *)at; at += sel_align((size_t)pairs * nb * l.tiles * 4);
    l.base = (int32_t *)at;   at += sel_align((size_t)pairs * (nb + 1) * 4);
    l.entry = (int32_t *)at;
    return l;
}

int launch_sel_lists(const SelProblem &p, const SelLists &l, int64_t bh0, int64_t pairs, int2 *items, int32_t *item_base, int64_t max_items,
                     int rows_per_item) {
    const dim3 grid((unsigned)l.tiles, (unsigned)((p.nb + kRange - 1) / kRange), (unsigned)pairs);
    lists_count_kernel<<<grid, kTile, 0, p.stream>>>(p, l, bh0);
    launch_after(lists_base_kernel, dim3((unsigned)pairs), dim3(1024), 0, p.stream, l, p.nb, (int)(p.H / p.Hkv), items, item_base, max_items, rows_per_item);
    const size_t smem = (kRange * (kTile / 32 + 1) + kTile * (kStage + 1)) * sizeof(int);
    if (int rc = ensure_dynamic_smem((const void *)lists_fill_kernel, smem, "shared memory of the lists of a block selection")) return rc;
    launch_after(lists_fill_kernel, grid, dim3(kTile), smem, p.stream, p, l, bh0);
    return launched("launching the lists of a block selection");
}

}  // namespace mat

using namespace mat;

static int have_workspace(size_t need, const void *workspace, size_t bytes) {
    if (workspace && bytes >= need && (uintptr_t)workspace % 256 == 0) return MAT_OK;
    return fail(MAT_ERR_WORKSPACE, "workspace of %zu bytes (256-byte aligned) required, got %zu", need, workspace ? bytes : (size_t)0);
}

extern "C" size_t mat_selected_attn_fwd_workspace_bytes(int64_t B, int64_t S, int64_t H, int64_t H_kv, int64_t D, int dtype, int64_t block, int64_t topk) {
    return check_selected(B, S, H, H_kv, D, dtype, block, topk) ? 0 : sel_workspace_bytes(B, S, H, H_kv, D, dtype, block, topk, false);
}

extern "C" int mat_selected_attn_fwd(const void *q, const void *k, const void *v, void *o, float *lse, int64_t B, int64_t S, int64_t H,
                                     int64_t H_kv, int64_t D, int dtype, const int32_t *blocks, int64_t block, int64_t topk, int causal,
                                     float scale, void *workspace, size_t workspace_bytes, void *stream) {
    if (int rc = check_selected(B, S, H, H_kv, D, dtype, block, topk)) return rc;
    if (!q || !k || !v || !o || !lse || !blocks) return fail(MAT_ERR_INVALID, "q, k, v, o, lse and blocks must be non-NULL");
    if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)o) % 16) return fail(MAT_ERR_INVALID, "q, k, v and o must be 16-byte aligned");
    SelProblem p{};
    p.q = q; p.k = k; p.v = v; p.out = o; p.lse = lse;
    p.B = B; p.S = S; p.H = H; p.Hkv = H_kv; p.D = D; p.dtype = dtype;
    p.blocks = blocks; p.block = block; p.topk = topk; p.nb = (S + block - 1) / block; p.causal = causal != 0;
    p.scale = scale > 0.f ? scale : 1.0f / std::sqrt((float)D);
    p.stream = (cudaStream_t)stream;
    if (int rc = have_workspace(sel_workspace_bytes(B, S, H, H_kv, D, dtype, block, topk, false), workspace, workspace_bytes)) return rc;
    note_kernel(dtype == MAT_F32 ? "selected_f32" : "selected_mma");
    return launch_sel(p, workspace, false);
}

extern "C" size_t mat_selected_attn_bwd_workspace_bytes(int64_t B, int64_t S, int64_t H, int64_t H_kv, int64_t D, int dtype, int64_t block, int64_t topk) {
    return check_selected(B, S, H, H_kv, D, dtype, block, topk) ? 0 : sel_workspace_bytes(B, S, H, H_kv, D, dtype, block, topk, true);
}

extern "C" int mat_selected_attn_bwd(const void *q, const void *k, const void *v, const void *o, const float *lse, const void *dout, void *dq,
                                     void *dk, void *dv, int64_t B, int64_t S, int64_t H, int64_t H_kv, int64_t D, int dtype,
                                     const int32_t *blocks, int64_t block, int64_t topk, int causal, float scale, void *workspace,
                                     size_t workspace_bytes, void *stream) {
    if (int rc = check_selected(B, S, H, H_kv, D, dtype, block, topk)) return rc;
    if (!q || !k || !v || !o || !lse || !dout || !dq || !dk || !dv || !blocks) return fail(MAT_ERR_INVALID, "all tensors must be non-NULL");
    if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)o | (uintptr_t)dout | (uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv) % 16)
        return fail(MAT_ERR_INVALID, "all tensors must be 16-byte aligned");
    if (int rc = have_workspace(sel_workspace_bytes(B, S, H, H_kv, D, dtype, block, topk, true), workspace, workspace_bytes)) return rc;
    SelProblem p{};
    p.q = q; p.k = k; p.v = v; p.o = o; p.dout = dout; p.lse_in = lse; p.dq = dq; p.dk = dk; p.dv = dv;
    p.B = B; p.S = S; p.H = H; p.Hkv = H_kv; p.D = D; p.dtype = dtype;
    p.blocks = blocks; p.block = block; p.topk = topk; p.nb = (S + block - 1) / block; p.causal = causal != 0;
    p.scale = scale > 0.f ? scale : 1.0f / std::sqrt((float)D);
    p.stream = (cudaStream_t)stream;
    note_kernel(dtype == MAT_F32 ? "selected_bwd_f32" : "selected_bwd_mma");
    return launch_sel(p, workspace, true);
}
