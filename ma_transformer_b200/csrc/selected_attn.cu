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

// ---- lists ----------------------------------------------------------------------------------------------------------
// mask[n][w]: the tile's queries that chose block n, a bit each.  A bit set does not depend on the order of the writers,
// so the lists come out the same every time.
__device__ __forceinline__ int own_limit(const SelProblem &p, int64_t i) {
    return p.causal ? (int)(i / p.block) + 1 : (int)p.nb;
}

template <bool FILL> __global__ void __launch_bounds__(kTile) lists_kernel(const SelProblem p, const SelLists l) {
    __shared__ uint32_t mask[kRange][kTile / 32];
    const int64_t tile = blockIdx.x, bh = blockIdx.z, b = bh / p.Hkv, h = bh % p.Hkv;
    const int n0 = blockIdx.y * kRange, n1 = min(n0 + kRange, (int)p.nb);
    const int tid = threadIdx.x;
    pdl_trigger();
    for (int i = tid; i < (n1 - n0) * (kTile / 32); i += kTile) (&mask[0][0])[i] = 0;
    pdl_wait();
    __syncthreads();
    const int64_t i = tile * kTile + tid;
    const int32_t *row = p.blocks + ((b * p.S + i) * p.Hkv + h) * p.topk;
    const int limit = i < p.S ? own_limit(p, i) : 0;
    if (i < p.S) {
        int prev = -1;
#pragma unroll 8
        for (int s = 0; s < p.topk; ++s) {
            const int n = row[s];
            if (sel_entry_counts(n, prev, limit) && n >= n0 && n < n1) atomicOr(&mask[n - n0][tid / 32], 1u << (tid % 32));
        }
    }
    __syncthreads();
    if (!FILL) {
        for (int n = n0 + tid; n < n1; n += kTile) {
            int c = 0;
#pragma unroll
            for (int w = 0; w < kTile / 32; ++w) c += __popc(mask[n - n0][w]);
            l.counts[(bh * p.nb + n) * l.tiles + tile] = c;
        }
    } else if (i < p.S) {
        int prev = -1;
        int32_t *entries = l.entry + bh * p.S * p.topk;
        for (int s0 = 0; s0 < p.topk; s0 += 8) {       // eight entries' offsets in flight
            int n[8], at[8];
#pragma unroll
            for (int y = 0; y < 8; ++y) n[y] = s0 + y < p.topk ? row[s0 + y] : -1;
#pragma unroll
            for (int y = 0; y < 8; ++y) {
                if (!sel_entry_counts(n[y], prev, limit) || n[y] < n0 || n[y] >= n1) n[y] = -1;
                at[y] = n[y] < 0 ? 0 : l.base[bh * (p.nb + 1) + n[y]] + l.counts[(bh * p.nb + n[y]) * l.tiles + tile];
            }
#pragma unroll
            for (int y = 0; y < 8; ++y) {
                if (n[y] < 0) continue;
                const uint32_t *m = mask[n[y] - n0];
                int rank = __popc(m[tid / 32] & ((1u << (tid % 32)) - 1));
                for (int w = 0; w < tid / 32; ++w) rank += __popc(m[w]);
                entries[at[y] + rank] = (int32_t)(i * p.topk + s0 + y);
            }
        }
    }
}

// counts of a block's tiles -> offsets within its list, one warp per (bh, block)
__global__ void __launch_bounds__(128) lists_offsets_kernel(SelLists l, int64_t rows) {
    const int64_t r = (int64_t)blockIdx.x * 4 + threadIdx.x / 32;
    pdl_trigger();
    pdl_wait();
    if (r >= rows) return;
    const int lane = threadIdx.x % 32;
    int32_t *c = l.counts + r * l.tiles;
    int total = 0;
    for (int64_t t0 = 0; t0 < l.tiles; t0 += 32) {
        const int x = t0 + lane < l.tiles ? c[t0 + lane] : 0;
        int sum = x;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += y;
        }
        if (t0 + lane < l.tiles) c[t0 + lane] = total + sum - x;
        total += __shfl_sync(0xffffffffu, sum, 31);
    }
    if (lane == 0) l.totals[r] = total;
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

// totals of the blocks -> where each list starts, and the items of its rows: one CTA per bh
__global__ void __launch_bounds__(1024) lists_base_kernel(SelLists l, int64_t nb, int G, int2 *items, int32_t *item_base, int64_t max_items, int rows_per_item) {
    __shared__ int of_warp[32], carry[2];
    const int64_t bh = blockIdx.x;
    pdl_trigger();
    pdl_wait();
    int entries = 0, before = 0;
    for (int64_t n0 = 0; n0 < nb; n0 += 1024) {
        const int64_t n = n0 + threadIdx.x;
        const int x = n < nb ? l.totals[bh * nb + n] : 0;
        const int sum = block_scan(x, of_warp);
        if (n < nb) l.base[bh * (nb + 1) + n] = entries + sum - x;
        const int mine = (int)(((int64_t)x * G + rows_per_item - 1) / rows_per_item);
        const int isum = block_scan(mine, of_warp);
        if (items && n < nb) {
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
        if (items) item_base[bh * (nb + 1) + nb] = before;
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
    if (B * Hkv > 65535) return fail(MAT_ERR_UNSUPPORTED, "B * H_kv must be at most 65535");
    if (S * topk > INT_MAX / (H / Hkv) || S * H > INT_MAX || B * S * H > (int64_t)INT_MAX * 2) return fail(MAT_ERR_UNSUPPORTED, "the sequence is too long for its topk");
    return MAT_OK;
}

}  // namespace

size_t sel_lists_bytes(int64_t B, int64_t S, int64_t Hkv, int64_t nb, int64_t topk) {
    const int64_t tiles = (S + kTile - 1) / kTile, bh = B * Hkv;
    return sel_align((size_t)bh * nb * tiles * 4) + sel_align((size_t)bh * nb * 4) + sel_align((size_t)bh * (nb + 1) * 4) +
           sel_align((size_t)bh * S * topk * 4);
}

SelLists sel_lists_at(void *ws, int64_t B, int64_t S, int64_t Hkv, int64_t nb, int64_t topk) {
    SelLists l;
    l.tiles = (S + kTile - 1) / kTile;
    const int64_t bh = B * Hkv;
    char *at = (char *)ws;
    l.counts = (int32_t *)at; at += sel_align((size_t)bh * nb * l.tiles * 4);
    l.totals = (int32_t *)at; at += sel_align((size_t)bh * nb * 4);
    l.base = (int32_t *)at;   at += sel_align((size_t)bh * (nb + 1) * 4);
    l.entry = (int32_t *)at;
    return l;
}

int launch_sel_lists(const SelProblem &p, const SelLists &l, int2 *items, int32_t *item_base, int64_t max_items, int rows_per_item) {
    const unsigned bh = (unsigned)(p.B * p.Hkv);
    const dim3 grid((unsigned)l.tiles, (unsigned)((p.nb + kRange - 1) / kRange), bh);
    lists_kernel<false><<<grid, kTile, 0, p.stream>>>(p, l);
    const int64_t rows = (int64_t)bh * p.nb;
    launch_after(lists_offsets_kernel, dim3((unsigned)((rows + 3) / 4)), dim3(128), 0, p.stream, l, rows);
    launch_after(lists_base_kernel, dim3(bh), dim3(1024), 0, p.stream, l, p.nb, (int)(p.H / p.Hkv), items, item_base, max_items, rows_per_item);
    launch_after(lists_kernel<true>, grid, dim3(kTile), 0, p.stream, p, l);
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
