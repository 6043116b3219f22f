// Attention over selected blocks of keys and its gradients: the C entry points, the lists of the queries that chose a
// block, and the kernels that serve every type and width: one warp per row with fp32 arithmetic.
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

// ---- one warp per row -----------------------------------------------------------------------------------------------
__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}
__device__ __forceinline__ float warp_max(float x) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
    return x;
}

// dot of a row in shared memory (fp32) with a row of elements
template <typename T> __device__ __forceinline__ float dot_row(const float *a, const T *x, int D) {
    constexpr int W = Vec16<T>::N;
    float s = 0.f;
    for (int d = 0; d < D; d += W) {
        float y[W];
        Vec16<T>::unpack(__ldg(reinterpret_cast<const uint4 *>(x + d)), y);
#pragma unroll
        for (int j = 0; j < W; ++j) s = fmaf(a[d + j], y[j], s);
    }
    return s;
}

// BWD false: o and lse of row (b, i, head).  BWD true: dq of the row; delta is left in delta_out for the key pass.
template <typename T, bool BWD> __global__ void __launch_bounds__(128) sel_rows_kernel(const SelProblem p, float *delta_out) {
    __shared__ float qs[4][128], ds_row[4][128];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, D = (int)p.D;
    const int64_t r = (int64_t)blockIdx.x * 4 + warp;       // (b, i, head)
    if (r >= p.B * p.S * p.H) return;
    const int64_t head = r % p.H, i = r / p.H % p.S, b = r / p.H / p.S, h = head / (p.H / p.Hkv);
    float delta = 0.f;
    for (int d = lane; d < D; d += 32) {
        qs[warp][d] = Elem<T>::to_f(((const T *)p.q)[r * D + d]);
        if (BWD) {
            const float g = Elem<T>::to_f(((const T *)p.dout)[r * D + d]);
            ds_row[warp][d] = g;
            delta = fmaf(g, Elem<T>::to_f(((const T *)p.o)[r * D + d]), delta);
        }
    }
    __syncwarp();
    const float lse = BWD ? p.lse_in[r] : 0.f;
    if (BWD) {
        delta = warp_sum(delta);
        if (lane == 0) delta_out[r] = delta;
    }
    float m = -INFINITY, l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
    const int32_t *list = p.blocks + ((b * p.S + i) * p.Hkv + h) * p.topk;
    const int limit = p.causal ? (int)(i / p.block) + 1 : (int)p.nb;
    int prev = -1;
    for (int s = 0; s < p.topk; ++s) {
        const int n = list[s];
        if (!sel_entry_counts(n, prev, limit)) continue;
        const int64_t j0 = n * p.block;
        int64_t j1 = j0 + p.block < p.S ? j0 + p.block : p.S;
        if (p.causal && j1 > i + 1) j1 = i + 1;
        for (int64_t base = j0; base < j1; base += 32) {
            const int64_t j = base + lane;
            const bool in = j < j1;
            const int64_t at = ((b * p.S + (in ? j : j0)) * p.Hkv + h) * D;
            const float x = dot_row<T>(qs[warp], (const T *)p.k + at, D) * p.scale;
            float w;     // the weight of this lane's key in the sum below
            if (BWD) {
                const float dp = dot_row<T>(ds_row[warp], (const T *)p.v + at, D);
                w = in && lse != -INFINITY ? expf(x - lse) * (dp - delta) : 0.f;
            } else {
                const float top = fmaxf(m, warp_max(in ? x : -INFINITY)), ref = top == -INFINITY ? 0.f : top;
                const float keep = expf(m - ref);
                w = in ? expf(x - ref) : 0.f;
                m = top;
                l = l * keep + warp_sum(w);
#pragma unroll
                for (int c = 0; c < 4; ++c) acc[c] *= keep;
            }
            const int64_t row0 = ((b * p.S + base) * p.Hkv + h) * D;
            const int cnt = (int)(j1 - base < 32 ? j1 - base : 32);
            const T *src = (const T *)(BWD ? p.k : p.v) + row0;
            for (int t = 0; t < cnt; ++t) {
                const float wt = __shfl_sync(0xffffffffu, w, t);
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (c * 32 + lane < D) acc[c] = fmaf(wt, Elem<T>::to_f(src[t * p.Hkv * D + c * 32 + lane]), acc[c]);
            }
        }
    }
    T *out = (T *)(BWD ? p.dq : p.out) + r * D;
    const float f = BWD ? p.scale : (l == 0.f ? 0.f : 1.f / l);
#pragma unroll
    for (int c = 0; c < 4; ++c)
        if (c * 32 + lane < D) out[c * 32 + lane] = Elem<T>::from_f(l == 0.f && !BWD ? 0.f : acc[c] * f);
    if (!BWD && lane == 0) p.lse[r] = l == 0.f ? -INFINITY : m + logf(l);
}

// dk and dv of one key: one warp, lanes over columns
template <typename T> __global__ void __launch_bounds__(128) sel_keys_kernel(const SelProblem p, const SelLists l, const float *delta) {
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, D = (int)p.D, G = (int)(p.H / p.Hkv);
    const int64_t r = (int64_t)blockIdx.x * 4 + warp;       // (b, j, h)
    if (r >= p.B * p.S * p.Hkv) return;
    const int64_t h = r % p.Hkv, j = r / p.Hkv % p.S, b = r / p.Hkv / p.S, bh = b * p.Hkv + h, n = j / p.block;
    float k[4], v[4], dk[4] = {0.f, 0.f, 0.f, 0.f}, dv[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        const bool in = c * 32 + lane < D;
        k[c] = in ? Elem<T>::to_f(((const T *)p.k)[r * D + c * 32 + lane]) : 0.f;
        v[c] = in ? Elem<T>::to_f(((const T *)p.v)[r * D + c * 32 + lane]) : 0.f;
    }
    const int32_t *list = l.entry + bh * p.S * p.topk;
    for (int e = l.base[bh * (p.nb + 1) + n]; e < l.base[bh * (p.nb + 1) + n + 1]; ++e) {
        const int64_t i = list[e] / p.topk;
        if (p.causal && i < j) continue;
        for (int g = 0; g < G; ++g) {
            const int64_t row = (b * p.S + i) * p.H + h * G + g;
            float q[4], o[4], x = 0.f, dp = 0.f;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const bool in = c * 32 + lane < D;
                q[c] = in ? Elem<T>::to_f(((const T *)p.q)[row * D + c * 32 + lane]) : 0.f;
                o[c] = in ? Elem<T>::to_f(((const T *)p.dout)[row * D + c * 32 + lane]) : 0.f;
                x = fmaf(q[c], k[c], x);
                dp = fmaf(o[c], v[c], dp);
            }
            x = warp_sum(x) * p.scale;
            dp = warp_sum(dp);
            const float w = expf(x - p.lse_in[row]), d = w * (dp - delta[row]);
#pragma unroll
            for (int c = 0; c < 4; ++c) { dv[c] = fmaf(w, o[c], dv[c]); dk[c] = fmaf(d, q[c], dk[c]); }
        }
    }
#pragma unroll
    for (int c = 0; c < 4; ++c)
        if (c * 32 + lane < D) {
            ((T *)p.dk)[r * D + c * 32 + lane] = Elem<T>::from_f(dk[c] * p.scale);
            ((T *)p.dv)[r * D + c * 32 + lane] = Elem<T>::from_f(dv[c]);
        }
}

int launched(const char *what) {
    cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? MAT_OK : cuda_fail(e, what);
}

template <typename T> int run_fwd(const SelProblem &p) {
    sel_rows_kernel<T, false><<<(unsigned)((p.B * p.S * p.H + 3) / 4), 128, 0, p.stream>>>(p, nullptr);
    return launched("launching the selected attention");
}

template <typename T> int run_bwd(const SelProblem &p, const SelLists &l, float *delta) {
    if (int rc = launch_sel_lists(p, l, nullptr, nullptr, 0, 1)) return rc;
    sel_rows_kernel<T, true><<<(unsigned)((p.B * p.S * p.H + 3) / 4), 128, 0, p.stream>>>(p, delta);
    if (int rc = launched("launching the selected attention's query gradient")) return rc;
    sel_keys_kernel<T><<<(unsigned)((p.B * p.S * p.Hkv + 3) / 4), 128, 0, p.stream>>>(p, l, delta);
    return launched("launching the selected attention's key gradients");
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

extern "C" size_t mat_selected_attn_fwd_workspace_bytes(int64_t B, int64_t S, int64_t H, int64_t H_kv, int64_t D, int dtype, int64_t block, int64_t topk) {
    if (check_selected(B, S, H, H_kv, D, dtype, block, topk) || dtype == MAT_F32) return 0;
    return sel_mma_workspace_bytes(B, S, H, H_kv, D, block, topk, false);
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
    const size_t need = mat_selected_attn_fwd_workspace_bytes(B, S, H, H_kv, D, dtype, block, topk);
    if (need > 0 && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 256))
        return fail(MAT_ERR_WORKSPACE, "workspace of %zu bytes (256-byte aligned) required, got %zu", need, workspace ? workspace_bytes : (size_t)0);
    note_kernel(dtype == MAT_F32 ? "selected_rows" : "selected_mma");
    return dtype == MAT_F32 ? run_fwd<float>(p) : launch_sel_mma(p, workspace, false);
}

extern "C" size_t mat_selected_attn_bwd_workspace_bytes(int64_t B, int64_t S, int64_t H, int64_t H_kv, int64_t D, int dtype, int64_t block, int64_t topk) {
    if (check_selected(B, S, H, H_kv, D, dtype, block, topk)) return 0;
    if (dtype != MAT_F32) return sel_mma_workspace_bytes(B, S, H, H_kv, D, block, topk, true);
    return sel_align((size_t)B * S * H * 4) + sel_lists_bytes(B, S, H_kv, (S + block - 1) / block, topk);
}

extern "C" int mat_selected_attn_bwd(const void *q, const void *k, const void *v, const void *o, const float *lse, const void *dout, void *dq,
                                     void *dk, void *dv, int64_t B, int64_t S, int64_t H, int64_t H_kv, int64_t D, int dtype,
                                     const int32_t *blocks, int64_t block, int64_t topk, int causal, float scale, void *workspace,
                                     size_t workspace_bytes, void *stream) {
    if (int rc = check_selected(B, S, H, H_kv, D, dtype, block, topk)) return rc;
    if (!q || !k || !v || !o || !lse || !dout || !dq || !dk || !dv || !blocks) return fail(MAT_ERR_INVALID, "all tensors must be non-NULL");
    if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)o | (uintptr_t)dout | (uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv) % 16)
        return fail(MAT_ERR_INVALID, "all tensors must be 16-byte aligned");
    const size_t need = mat_selected_attn_bwd_workspace_bytes(B, S, H, H_kv, D, dtype, block, topk);
    if (!workspace || workspace_bytes < need || (uintptr_t)workspace % 256)
        return fail(MAT_ERR_WORKSPACE, "workspace of %zu bytes (256-byte aligned) required, got %zu", need, workspace ? workspace_bytes : (size_t)0);
    SelProblem p{};
    p.q = q; p.k = k; p.v = v; p.o = o; p.dout = dout; p.lse_in = lse; p.dq = dq; p.dk = dk; p.dv = dv;
    p.B = B; p.S = S; p.H = H; p.Hkv = H_kv; p.D = D; p.dtype = dtype;
    p.blocks = blocks; p.block = block; p.topk = topk; p.nb = (S + block - 1) / block; p.causal = causal != 0;
    p.scale = scale > 0.f ? scale : 1.0f / std::sqrt((float)D);
    p.stream = (cudaStream_t)stream;
    note_kernel(dtype == MAT_F32 ? "selected_bwd_rows" : "selected_bwd_mma");
    if (dtype != MAT_F32) return launch_sel_mma(p, workspace, true);
    return run_bwd<float>(p, sel_lists_at((char *)workspace + sel_align((size_t)B * S * H * 4), B, S, H_kv, p.nb, topk), (float *)workspace);
}
