// Attention of one new token per sequence over a paged cache: split over the cache's length, then joined.
//
// A row is (sequence, key head) with the G query heads that read it, so every key and value leaves HBM once for all of
// them.  What a row sees is a list of n virtual tokens: the whole cache (t -> position t), a window of the framework's
// kind (t -> first + t * dilation) or a list of pages (t -> slot t mod page of page entry t / page).  The list is cut
// into chunks of c tokens, one CTA each; a CTA keeps the running maximum and sum of its softmax and one output row per
// query head, and rows of several chunks leave (maximum, sum, unnormalised output) in the workspace in fp32 for
// join_kernel, which adds them up in chunk order: nothing depends on timing.  How a row is cut follows from its length, the
// number of rows (sequences x key heads) and the width of the page table or the window or list (plan() below), so a
// sequence may round differently in another batch or under a wider table.
#include <limits.h>

#include <cmath>

#include "paged.cuh"
#include "pdl.cuh"
#include "ptx.cuh"

namespace mat {
namespace {

constexpr int kSms = 148;

struct DecodeArgs {
    PagedView c;
    const void *q;
    void *o;
    int64_t q_stride, B, H, Hkv, D;
    const int32_t *lengths;
    int64_t left, dilation;
    const int32_t *pages;
    int64_t n_sel;
    float scale_log2;
    int G, nsplit, min_chunk, tiles;   // tiles: groups of query heads per key head
    int cluster;                    // the chunks of a row are one cluster
    int aligned;                    // the kernel reads 16 neighbouring positions at a time: first is a multiple of 16
    float2 *stats;                  // [B, H, nsplit] (maximum, sum)
    float *part;                    // [B, H, nsplit, D]
    int *status;
};

// The virtual tokens of one row.
struct RowTokens {
    int64_t len, first, lo, dil;   // positions below lo belong to the alignment, not to the row
    const int32_t *list;
    int64_t n;
    __device__ __forceinline__ RowTokens(const DecodeArgs &a, int64_t b, int64_t h) {
        len = a.lengths[b];
        first = lo = 0; dil = 1; list = nullptr;
        if (len <= 0) {
            n = 0;
        } else if (a.pages) {
            list = a.pages + (b * a.Hkv + h) * a.n_sel;
            n = a.n_sel << a.c.page_shift;
        } else {
            // tokens past the end of the table are absent
            const int64_t cap = a.c.width << a.c.page_shift;
            if (len > cap && threadIdx.x == 0) atomicOr(a.status, kPagedOutside);
            if (a.left < 0) {
                n = len < cap ? len : cap;
            } else {
                dil = a.dilation;
                const int64_t back = dil == 1 ? len - 1 : (len - 1) / dil;
                n = (a.left < back ? a.left : back) + 1;
                first = lo = len - 1 - (n - 1) * dil;
                if (len > cap) n = first < cap ? (cap - first + dil - 1) / dil : 0;
                if (a.aligned) {
                    first = lo / 16 * 16;
                    n += n > 0 ? lo - first : 0;
                }
            }
        }
    }
    // tokens per chunk; rows of up to c tokens are one chunk
    __device__ __forceinline__ int64_t chunk(const DecodeArgs &a) const {
        if (n <= a.min_chunk) return a.min_chunk;
        // as few chunks as min_chunk allows, all of one size
        const uint32_t most = (uint32_t)a.nsplit, m = (uint32_t)n, want = (m + a.min_chunk - 1) / a.min_chunk, k = want < most ? want : most;
        return (int64_t)(((m + k - 1) / k + 63) / 64 * 64);
    }
    // position of virtual token t, or -1
    __device__ __forceinline__ int64_t position(const DecodeArgs &a, int64_t t) const {
        if (!list) return first + t * dil;
        const int64_t p = list[t >> a.c.page_shift];
        const int64_t pos = (p << a.c.page_shift) + (t & ((1 << a.c.page_shift) - 1));
        return p >= 0 && pos < len ? pos : -1;
    }
};

// Rows of few chunks: the chunks' CTAs form a cluster and join through each other's shared memory, without a workspace
// and a second launch (8 rows of 777 tokens: a call of 10.6 us against 15.2).  Every CTA of the cluster stays to the end,
// so this is for launches that fit the GPU at once.  `mine`: [heads][cols + 4] unnormalised outputs, then maximum and sum
// in the last columns; the CTAs share the (head, 4 columns) items.
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t peer_smem(const void *p, uint32_t rank) {
    uint32_t a;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(ptx::smem_u32(p)), "r"(rank));
    return a;
}
__device__ __forceinline__ float4 peer_load(uint32_t a) {
    float4 x;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w) : "r"(a) : "memory");
    return x;
}
template <typename T> __device__ __forceinline__ void cluster_join(const DecodeArgs &a, const float *mine, int heads, int pitch, int64_t head0) {
    __syncthreads();
    cluster_sync();
    const int vecs = (int)a.D / 4, n = a.nsplit;
    for (int x = blockIdx.y * 128 + threadIdx.x; x < heads * vecs; x += n * 128) {
        const int g = x / vecs, col = x % vecs * 4;
        const float *row = mine + g * pitch;
        float4 st[8], u[8];
        float top = -INFINITY;
#pragma unroll
        for (int r = 0; r < 8; ++r)
            if (r < n) {
                st[r] = peer_load(peer_smem(row + pitch - 4, r));
                u[r] = peer_load(peer_smem(row + col, r));
                top = fmaxf(top, st[r].x);
            }
        const float ref = top == -INFINITY ? 0.f : top;
        float sum = 0.f;
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int r = 0; r < 8; ++r)
            if (r < n) {
                const float e = exp2f(st[r].x - ref);
                sum += st[r].y * e;
                y.x = fmaf(u[r].x, e, y.x); y.y = fmaf(u[r].y, e, y.y); y.z = fmaf(u[r].z, e, y.z); y.w = fmaf(u[r].w, e, y.w);
            }
        const float f = sum == 0.f ? 0.f : 1.f / sum;
        T *o = (T *)a.o + (head0 + g) * a.D + col;
        o[0] = Elem<T>::from_f(y.x * f); o[1] = Elem<T>::from_f(y.y * f); o[2] = Elem<T>::from_f(y.z * f); o[3] = Elem<T>::from_f(y.w * f);
    }
    __syncthreads();
    cluster_sync();                                  // nobody leaves while its shared memory is read
}

// ---- one warp per few keys, fp32 arithmetic: any type ---------------------------------------------------------------
// LPK lanes hold one key's columns, NV 16-byte vectors each (lanes past D idle); a warp scores 32 / LPK keys at a time,
// U times unrolled so that their loads are in flight together.  GT query heads per CTA.
template <typename T, int LPK, int NV, int GT, int U, bool CLUSTER>
__global__ void __launch_bounds__(128) decode_simt_kernel(const DecodeArgs a) {
    constexpr int W = Vec16<T>::N, KPW = 32 / LPK, C = NV * W, NVAL = U * GT;
    constexpr int NR = NVAL > LPK ? NVAL / LPK : 1;                  // scores a lane is left with
    constexpr int ULANE = LPK / U;                                   // lowest lane bit that tells keys apart
    const int64_t b = blockIdx.z, h = blockIdx.x / (unsigned)a.tiles, g0 = (int64_t)(blockIdx.x % (unsigned)a.tiles) * GT;
    const int64_t G = a.G;
    const int D = (int)a.D;
    pdl_trigger();
    const RowTokens row(a, b, h);
    const int64_t chunk = row.chunk(a), t0 = blockIdx.y * chunk;
    const int64_t t1 = t0 + chunk < row.n ? t0 + chunk : row.n;
    if (!CLUSTER && t0 >= row.n && blockIdx.y > 0) return;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, part = lane % LPK, key = lane / LPK;

    const int group0 = lane - part;
    const int first_value = part * NVAL / LPK;                       // of the scores this lane is left with
    auto lane_of = [](int value) { return value * LPK / NVAL; };     // lane of a group that is left with it
    float q[GT][C], acc[GT][C], m[NR], l[NR];
#pragma unroll
    for (int i = 0; i < NR; ++i) { m[i] = -INFINITY; l[i] = 0.f; }
#pragma unroll
    for (int g = 0; g < GT; ++g) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int col = (i * LPK + part) * W;
            if (g0 + g < G && col < D) {
                Vec16<T>::unpack(*reinterpret_cast<const uint4 *>((const T *)a.q + b * a.q_stride + (h * G + g0 + g) * D + col), &q[g][i * W]);
            } else {
#pragma unroll
                for (int j = 0; j < W; ++j) q[g][i * W + j] = 0.f;
            }
        }
#pragma unroll
        for (int j = 0; j < C; ++j) { q[g][j] *= a.scale_log2; acc[g][j] = 0.f; }
    }

    // positions and table entries of the next keys are read while the present ones are worked on
    int64_t at[U];
    int32_t entry[U];
    auto look_up = [&](int64_t base) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t t = base + u * KPW + key;
            at[u] = t < t1 ? row.position(a, t) : -1;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) entry[u] = at[u] >= 0 ? table_entry(a.c, b, at[u] >> a.c.page_shift) : -1;
    };
    look_up(t0 + warp * (KPW * U));
    for (int64_t base = t0 + warp * (KPW * U); base < t1; base += 4 * KPW * U) {
        uint4 kv[U][NV], vv[U][NV];
        bool ok[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            ok[u] = entry[u] >= 0 && entry[u] < a.c.n_pages;
            const int64_t phys = entry[u], slot = at[u] & ((1 << a.c.page_shift) - 1);
            const T *kr = (const T *)a.c.k + phys * a.c.k_page + slot * a.c.k_tok + h * a.c.k_head;
            const T *vr = (const T *)a.c.v + phys * a.c.v_page + slot * a.c.v_tok + h * a.c.v_head;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int col = (i * LPK + part) * W;
                const bool in = ok[u] && col < D;
                kv[u][i] = in ? __ldg(reinterpret_cast<const uint4 *>(kr + col)) : make_uint4(0, 0, 0, 0);
                vv[u][i] = in ? __ldg(reinterpret_cast<const uint4 *>(vr + col)) : make_uint4(0, 0, 0, 0);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (at[u] >= 0 && !ok[u]) atomicOr(a.status, kPagedOutside);
        look_up(base + 4 * KPW * U);
        // Scores of U keys x GT heads, NV values per group of lanes.  Halving the set at every step of the sum over lanes
        // takes NV - 1 exchanges instead of NV log2(LPK), and leaves each lane with its own NR scores: one exponential
        // per score instead of one per lane, and the weights go back by a shuffle each.
        float s[NVAL];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float k[C];
#pragma unroll
            for (int i = 0; i < NV; ++i) Vec16<T>::unpack(kv[u][i], k + i * W);
#pragma unroll
            for (int g = 0; g < GT; ++g) {
                float d = 0.f;
#pragma unroll
                for (int j = 0; j < C; ++j) d = fmaf(q[g][j], k[j], d);
                s[u * GT + g] = d;
            }
        }
        int left = NVAL;
#pragma unroll
        for (int o = LPK / 2; o > 0; o >>= 1) {
            if (left > 1) {
                left /= 2;
#pragma unroll
                for (int i = 0; i < NVAL / 2; ++i)
                    if (i < left) {
                        const float send = lane & o ? s[i] : s[i + left], keep = lane & o ? s[i + left] : s[i];
                        s[i] = keep + __shfl_xor_sync(0xffffffffu, send, o);
                    }
            } else {
                s[0] += __shfl_xor_sync(0xffffffffu, s[0], o);
            }
        }
        uint32_t seen = 0;                               // keys of this group's U that count
#pragma unroll
        for (int u = 0; u < U; ++u) seen |= (ok[u] ? 1u : 0u) << u;
        bool moved = false;
        float keep[NR];
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            if (!(seen >> ((first_value + i) / GT) & 1)) s[i] = -INFINITY;
            float top = s[i];
#pragma unroll
            for (int o = ULANE; o < LPK; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));   // over the keys
            top = fmaxf(top, m[i]);
            const float ref = top == -INFINITY ? 0.f : top;   // nothing seen yet: every weight below is 2^-inf = 0
            keep[i] = exp2f(m[i] - ref);
            moved |= top != m[i];
            m[i] = top;
            s[i] = exp2f(s[i] - ref);
            l[i] = l[i] * keep[i] + s[i];
        }
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
            for (int g = 0; g < GT; ++g) {
                const float f = __shfl_sync(0xffffffffu, keep[g % NR], group0 + lane_of(g));
#pragma unroll
                for (int j = 0; j < C; ++j) acc[g][j] *= f;
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float v[C];
#pragma unroll
            for (int i = 0; i < NV; ++i) Vec16<T>::unpack(vv[u][i], v + i * W);
#pragma unroll
            for (int g = 0; g < GT; ++g) {
                const float w = __shfl_sync(0xffffffffu, s[(u * GT + g) % NR], group0 + lane_of(u * GT + g));
#pragma unroll
                for (int j = 0; j < C; ++j) acc[g][j] = fmaf(w, v[j], acc[g][j]);
            }
        }
    }
    // every lane: maximum and sum of every head of its group
    float m_all[GT], l_all[GT];
#pragma unroll
    for (int i = 0; i < NR; ++i)
#pragma unroll
        for (int o = ULANE; o < LPK; o <<= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], o);
#pragma unroll
    for (int g = 0; g < GT; ++g) {
        m_all[g] = __shfl_sync(0xffffffffu, m[g % NR], group0 + lane_of(g));
        l_all[g] = __shfl_sync(0xffffffffu, l[g % NR], group0 + lane_of(g));
    }
    // join the key lanes of a warp, then the warps
    extern __shared__ __align__(16) float sm[];        // [4][GT][D + 2], then for a cluster [GT][D + 4]
#pragma unroll
    for (int g = 0; g < GT; ++g) {
#pragma unroll
        for (int o = LPK; o < 32; o <<= 1) {
            const float m2 = __shfl_xor_sync(0xffffffffu, m_all[g], o), l2 = __shfl_xor_sync(0xffffffffu, l_all[g], o);
            const float top = fmaxf(m_all[g], m2), ref = top == -INFINITY ? 0.f : top;
            const float e1 = exp2f(m_all[g] - ref), e2 = exp2f(m2 - ref);
            l_all[g] = l_all[g] * e1 + l2 * e2;
            m_all[g] = top;
#pragma unroll
            for (int j = 0; j < C; ++j) acc[g][j] = acc[g][j] * e1 + __shfl_xor_sync(0xffffffffu, acc[g][j], o) * e2;
        }
        float *w = sm + (warp * GT + g) * (D + 2);
        if (key == 0) {
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int j = 0; j < W; ++j)
                    if ((i * LPK + part) * W < D) w[2 + (i * LPK + part) * W + j] = acc[g][i * W + j];
            if (part == 0) { w[0] = m_all[g]; w[1] = l_all[g]; }
        }
    }
    __syncthreads();
    const bool whole = chunk >= row.n;
    for (int g = 0; g < GT && g0 + g < G; ++g) {
        const float *w = sm + g * (D + 2);
        const int stride = GT * (D + 2);
        float top = -INFINITY, sum = 0.f, e[4];
        for (int i = 0; i < 4; ++i) top = fmaxf(top, w[i * stride]);
        const float ref = top == -INFINITY ? 0.f : top;
        for (int i = 0; i < 4; ++i) { e[i] = exp2f(w[i * stride] - ref); sum += w[i * stride + 1] * e[i]; }
        const int64_t head = b * a.H + h * G + g0 + g;
        const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
        for (int d = threadIdx.x; d < D; d += 128) {
            float x = 0.f;
            for (int i = 0; i < 4; ++i) x += w[i * stride + 2 + d] * e[i];
            if (CLUSTER) sm[4 * GT * (D + 2) + g * (D + 4) + d] = x;
            else if (whole) ((T *)a.o)[head * D + d] = Elem<T>::from_f(sum == 0.f ? 0.f : x * inv);
            else a.part[(head * a.nsplit + blockIdx.y) * D + d] = x;
        }
        if (CLUSTER && threadIdx.x < 2) sm[4 * GT * (D + 2) + g * (D + 4) + D + threadIdx.x] = threadIdx.x ? sum : top;
        else if (!whole && threadIdx.x == 0) a.stats[head * a.nsplit + blockIdx.y] = make_float2(top, sum);
    }
    if (CLUSTER) cluster_join<T>(a, sm + 4 * GT * (D + 2), (int)(G - g0 < GT ? G - g0 : GT), D + 4, b * a.H + h * G + g0);
}

// ---- 16-bit types on the tensor cores ---------------------------------------------------------------------------------
// One warp per 16 neighbouring tokens against up to 16 query heads of a key head: S = Q K^T and O += P V are m16n8k16
// products whose rows are the heads, so a group of 1 to 16 heads costs the same and the kernel stays bound by memory.
// What it needs is bytes in flight: every warp has a ring of NS tiles of its own, filled by cp.async NS - 1 tiles ahead
// (128 KB a SM with two CTAs) and waited for without a CTA barrier.  A tile never crosses a page (pages of 16 tokens and
// more), so its 16 rows share one table lookup, a warp looks up 32 tiles at a time, and rows are stepped through: forming
// every copy's address took more issue slots than the mathematics (150 us instead of 140).
// 64 sequences of up to 8192 tokens, 32 heads on 8 of 128 columns, 861 MB: 140 us = 6.15 TB/s by ncu, 95 % of the measured
// copy rate; a call of 154 to 158 us with its join over states that L2 does not hold (5.5 TB/s).  4 of up to 131072, 1254 MB:
// a call of 217 to 220 us (5.7 TB/s).
__device__ __forceinline__ void cp_async16(void *dst, const void *src, bool in) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(ptx::smem_u32(dst)), "l"(src), "r"(in ? 16 : 0) : "memory");
}

template <typename T, int DP, int NS, bool CLUSTER> __global__ void __launch_bounds__(128) decode_mma_kernel(const DecodeArgs a) {
    constexpr int PITCH = DP + 8, TILE = 16 * PITCH, CH = DP / 8;
    const int64_t b = blockIdx.z, h = blockIdx.x / (unsigned)a.tiles, G = a.G;
    const int g0 = (int)(blockIdx.x % (unsigned)a.tiles) * 16, heads = min(16, (int)G - g0);
    const int D = (int)a.D;
    pdl_trigger();
    const RowTokens row(a, b, h);
    const int64_t chunk = row.chunk(a), t0 = blockIdx.y * chunk;
    const int64_t t1 = t0 + chunk < row.n ? t0 + chunk : row.n;
    if (!CLUSTER && t0 >= row.n && blockIdx.y > 0) return;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    extern __shared__ __align__(16) char smem[];
    T *ring = (T *)smem + warp * NS * 2 * TILE;          // NS x (16 keys, 16 values)
    const int tiles = t1 > t0 ? (int)((t1 - t0 + 15) / 16) : 0, mine = (tiles - warp + 3) / 4;   // tiles warp, warp + 4, ...

    // queries: through this warp's ring into registers
    uint32_t qf[DP / 16][4];
    for (int c = lane; c < 16 * CH; c += 32) {
        const int r = c / CH, col = c % CH * 8;
        const bool in = r < heads && col < D;
        const T *src = (const T *)a.q + b * a.q_stride + (h * G + g0 + (in ? r : 0)) * D + (in ? col : 0);
        *reinterpret_cast<uint4 *>(ring + r * PITCH + col) = in ? __ldg(reinterpret_cast<const uint4 *>(src)) : make_uint4(0, 0, 0, 0);
    }
    __syncwarp();
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk)
        ptx::ldmatrix_x4(qf[kk], ptx::smem_u32(ring + (lane % 16) * PITCH + kk * 16 + (lane / 16) * 8));
    __syncwarp();

    // lane x of a batch of 32 tiles: physical page (-1: none) and first position of this warp's tile 32 * batch + x
    int phys_of = -1, pos_of = 0;
    auto look_up = [&](int batch) {
        const int x = batch * 32 + lane;
        phys_of = -1;
        if (x < mine) {
            const int64_t t = t0 + (int64_t)(warp + 4 * x) * 16;
            const int64_t pos = row.position(a, t);     // -1: a list entry that counts for nothing
            if (pos >= 0) {
                phys_of = (int)physical_page(a.c, b, pos >> a.c.page_shift, a.status);
                pos_of = (int)pos;
            }
        }
    };
    // this lane's 16 bytes of every row it copies; a lane past D copies zeros
    constexpr int RS = 32 / CH > 0 ? 32 / CH : 1;        // rows a warp copies at a time
    const int r0 = lane / CH, col = lane % CH * 8, bytes = col < D ? 16 : 0;
    const int64_t k_lane = col < D ? r0 * a.c.k_tok + h * a.c.k_head + col : 0, v_lane = col < D ? r0 * a.c.v_tok + h * a.c.v_head + col : 0;
    const int64_t k_step = col < D ? RS * a.c.k_tok : 0, v_step = col < D ? RS * a.c.v_tok : 0;
    const uint32_t lane_dst = ptx::smem_u32(ring + r0 * PITCH + col);
    int fill = 0;                                        // place of the ring that the next load goes to
    auto load = [&](int x) {                             // tile x into its place of the ring
        const int phys = __shfl_sync(0xffffffffu, phys_of, x % 32), pos = __shfl_sync(0xffffffffu, pos_of, x % 32);
        if (x < mine) {
            uint32_t dst = lane_dst + fill * (2 * TILE * (int)sizeof(T));
            const int64_t slot = pos & ((1 << a.c.page_shift) - 1);
            const int lo = (int)(row.lo - pos), hi = phys < 0 ? 0 : (int)(row.len - pos < 16 ? row.len - pos : 16);
            const T *k = (const T *)a.c.k, *v = (const T *)a.c.v;
            if (phys >= 0) {
                k += phys * a.c.k_page + slot * a.c.k_tok;
                v += phys * a.c.v_page + slot * a.c.v_tok;
            }
            if (lo <= 0 && hi == 16) {                   // all but the ends of a row
                k += k_lane;
                v += v_lane;
#pragma unroll
                for (int i = 0; i < 16 / RS; ++i) {
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(k), "r"(bytes) : "memory");
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + TILE * (int)sizeof(T)), "l"(v), "r"(bytes) : "memory");
                    dst += RS * PITCH * sizeof(T);
                    k += k_step;
                    v += v_step;
                }
            } else {
                // rows outside the sequence arrive as zeros: a weight of zero would not silence what such a row holds
                T *at = ring + fill * 2 * TILE;
                for (int r = r0; r < 16; r += RS) {
                    const bool in = r >= lo && r < hi && col < D;
                    cp_async16(at + r * PITCH + col, in ? k + r * a.c.k_tok + h * a.c.k_head + col : k, in);
                    cp_async16(at + TILE + r * PITCH + col, in ? v + r * a.c.v_tok + h * a.c.v_head + col : v, in);
                }
            }
        }
        fill = fill == NS - 1 ? 0 : fill + 1;
        asm volatile("cp.async.commit_group;" ::: "memory");
    };

    float o[DP / 8][4], m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
#pragma unroll
    for (int c = 0; c < DP / 8; ++c) o[c][0] = o[c][1] = o[c][2] = o[c][3] = 0.f;
    look_up(0);
    int phys_now = phys_of, pos_now = pos_of;            // of the batch being computed; loads may be a batch ahead
#pragma unroll
    for (int x = 0; x < NS - 1; ++x) load(x);
    int place = 0;
    for (int x = 0; x < mine; ++x) {
        if (x % 32 == 0) { phys_now = phys_of; pos_now = pos_of; }
        if ((x + NS - 1) % 32 == 0) look_up((x + NS - 1) / 32);
        load(x + NS - 1);
        asm volatile("cp.async.wait_group %0;" ::"n"(NS - 1) : "memory");
        __syncwarp();
        const T *k = ring + place * 2 * TILE, *v = k + TILE;
        place = place == NS - 1 ? 0 : place + 1;
        const int phys = __shfl_sync(0xffffffffu, phys_now, x % 32), pos = __shfl_sync(0xffffffffu, pos_now, x % 32);
        if (phys >= 0) {
            float s[2][4] = {};
#pragma unroll
            for (int kk = 0; kk < DP / 16; ++kk) {
                uint32_t r[4];
                ptx::ldmatrix_x4(r, ptx::smem_u32(k + (lane % 8 + (lane / 16) * 8) * PITCH + kk * 16 + (lane / 8 % 2) * 8));
                ptx::Mma<T>::run(s[0], qf[kk], r[0], r[1]);
                ptx::Mma<T>::run(s[1], qf[kk], r[2], r[3]);
            }
            const int lo = (int)(row.lo - pos), hi = (int)(row.len - pos < 16 ? row.len - pos : 16);
            if (lo > 0 || hi < 16)
#pragma unroll
                for (int c = 0; c < 2; ++c)
#pragma unroll
                    for (int y = 0; y < 4; ++y) {
                        const int col = c * 8 + (lane % 4) * 2 + y % 2;
                        if (col < lo || col >= hi) s[c][y] = -INFINITY;
                    }
            float t0m = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[1][0], s[1][1]));
            float t1m = fmaxf(fmaxf(s[0][2], s[0][3]), fmaxf(s[1][2], s[1][3]));
#pragma unroll
            for (int y = 1; y < 4; y <<= 1) {
                t0m = fmaxf(t0m, __shfl_xor_sync(0xffffffffu, t0m, y));
                t1m = fmaxf(t1m, __shfl_xor_sync(0xffffffffu, t1m, y));
            }
            t0m = fmaxf(m0, t0m * a.scale_log2);
            t1m = fmaxf(m1, t1m * a.scale_log2);
            if (__any_sync(0xffffffffu, t0m != m0 || t1m != m1)) {       // a new maximum somewhere: rescale
                const float e0 = ptx::ex2(m0 - (t0m == -INFINITY ? 0.f : t0m)), e1 = ptx::ex2(m1 - (t1m == -INFINITY ? 0.f : t1m));
                m0 = t0m; m1 = t1m;
                l0 *= e0; l1 *= e1;
#pragma unroll
                for (int c = 0; c < DP / 8; ++c) { o[c][0] *= e0; o[c][1] *= e0; o[c][2] *= e1; o[c][3] *= e1; }
            }
            const float r0 = m0 == -INFINITY ? 0.f : m0, r1 = m1 == -INFINITY ? 0.f : m1;
            // the weights are rounded to the cache's type for the tensor cores, one rounding of the kind the output has;
            // their sum stays in fp32
            uint32_t pf[4];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const float w = ptx::ex2(fmaf(s[c][0], a.scale_log2, -r0)), x1 = ptx::ex2(fmaf(s[c][1], a.scale_log2, -r0));
                const float y = ptx::ex2(fmaf(s[c][2], a.scale_log2, -r1)), z = ptx::ex2(fmaf(s[c][3], a.scale_log2, -r1));
                l0 += w + x1;
                l1 += y + z;
                pf[2 * c] = ptx::Mma<T>::pack(w, x1);
                pf[2 * c + 1] = ptx::Mma<T>::pack(y, z);
            }
#pragma unroll
            for (int c = 0; c < DP / 16; ++c) {
                uint32_t r[4];
                ptx::ldmatrix_x4_trans(r, ptx::smem_u32(v + (lane % 16) * PITCH + c * 16 + (lane / 16) * 8));
                ptx::Mma<T>::run(o[2 * c], pf, r[0], r[1]);
                ptx::Mma<T>::run(o[2 * c + 1], pf, r[2], r[3]);
            }
        }
        __syncwarp();                                    // the tile's place may be filled again
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
    for (int y = 1; y < 4; y <<= 1) {
        l0 += __shfl_xor_sync(0xffffffffu, l0, y);
        l1 += __shfl_xor_sync(0xffffffffu, l1, y);
    }
    __syncthreads();                                     // the rings become the warps' results
    float *sm = (float *)smem;                           // [4][16][DP + 4], then [4][16] maxima and sums
    float *ms = sm + 4 * 16 * (DP + 4), *ls = ms + 64;
    const int gr = lane / 4;
    if (lane % 4 == 0) {
        ms[warp * 16 + gr] = m0; ms[warp * 16 + gr + 8] = m1;
        ls[warp * 16 + gr] = l0; ls[warp * 16 + gr + 8] = l1;
    }
#pragma unroll
    for (int c = 0; c < DP / 8; ++c) {
        float *w = sm + (warp * 16 + gr) * (DP + 4) + c * 8 + (lane % 4) * 2;
        *reinterpret_cast<float2 *>(w) = make_float2(o[c][0], o[c][1]);
        *reinterpret_cast<float2 *>(w + 8 * (DP + 4)) = make_float2(o[c][2], o[c][3]);
    }
    __syncthreads();
    const bool whole = chunk >= row.n;
    const int vecs = D / 4;
    for (int x = threadIdx.x; x < heads * vecs; x += 128) {
        const int g = x / vecs, col = x % vecs * 4;
        float top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, ms[i * 16 + g]);
        const float ref = top == -INFINITY ? 0.f : top;
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float e = ptx::ex2(ms[i * 16 + g] - ref);
            sum += ls[i * 16 + g] * e;
            const float4 u = *reinterpret_cast<const float4 *>(sm + (i * 16 + g) * (DP + 4) + col);
            y.x = fmaf(u.x, e, y.x); y.y = fmaf(u.y, e, y.y); y.z = fmaf(u.z, e, y.z); y.w = fmaf(u.w, e, y.w);
        }
        const int64_t head = b * a.H + h * G + g0 + g;
        if (CLUSTER) {
            float *mine_row = ls + 64 + g * (DP + 4);
            *reinterpret_cast<float4 *>(mine_row + col) = y;
            if (col == 0) *reinterpret_cast<float4 *>(mine_row + DP) = make_float4(top, sum, 0.f, 0.f);
        } else if (whole) {
            const float f = sum == 0.f ? 0.f : 1.f / sum;
            T z[4] = {Elem<T>::from_f(y.x * f), Elem<T>::from_f(y.y * f), Elem<T>::from_f(y.z * f), Elem<T>::from_f(y.w * f)};
            *reinterpret_cast<uint2 *>((T *)a.o + head * D + col) = *reinterpret_cast<uint2 *>(z);
        } else {
            *reinterpret_cast<float4 *>(a.part + (head * a.nsplit + blockIdx.y) * D + col) = y;
            if (col == 0) a.stats[head * a.nsplit + blockIdx.y] = make_float2(top, sum);
        }
    }
    if (CLUSTER) cluster_join<T>(a, ls + 64, heads, DP + 4, b * a.H + h * G + g0);
}

// ---- joining the chunks of a row -------------------------------------------------------------------------------------
// Up to 32 chunks: one warp per (sequence, query head), a lane per chunk for the weights, then lanes over columns.
template <typename T> __global__ void __launch_bounds__(128) join_few_kernel(const DecodeArgs a) {
    const int lane = threadIdx.x % 32, D = (int)a.D;
    const uint32_t x = blockIdx.x * 4 + threadIdx.x / 32, b = x / (uint32_t)a.H, hq = x - b * (uint32_t)a.H;
    pdl_wait();
    if (b >= (uint32_t)a.B) return;
    const int64_t head = x;
    const RowTokens row(a, b, hq / (uint32_t)a.G);
    const int64_t chunk = row.chunk(a);
    if (chunk >= row.n) return;                      // written by its only chunk
    const int n = (int)((uint32_t)(row.n + chunk - 1) / (uint32_t)chunk);
    const float2 st = lane < n ? a.stats[head * a.nsplit + lane] : make_float2(-INFINITY, 0.f);
    float top = st.x;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float w = exp2f(st.x - (top == -INFINITY ? 0.f : top));
    float sum = st.y * w;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const float f = sum == 0.f ? 0.f : 1.f / sum;
    const float *part = a.part + head * a.nsplit * D;
    for (int c0 = 0; c0 < D; c0 += 128) {
        const int col = c0 + lane * 4;
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int i = 0; i < n; ++i) {
            const float e = __shfl_sync(0xffffffffu, w, i);
            const float4 u = col < D ? *reinterpret_cast<const float4 *>(part + i * D + col) : make_float4(0.f, 0.f, 0.f, 0.f);
            y.x = fmaf(u.x, e, y.x); y.y = fmaf(u.y, e, y.y); y.z = fmaf(u.z, e, y.z); y.w = fmaf(u.w, e, y.w);
        }
        if (col >= D) continue;
        T *o = (T *)a.o + head * D + col;
        o[0] = Elem<T>::from_f(y.x * f); o[1] = Elem<T>::from_f(y.y * f); o[2] = Elem<T>::from_f(y.z * f); o[3] = Elem<T>::from_f(y.w * f);
    }
}

// More: CTAs of 32 columns of a (sequence, query head), the chunks' weights first, then the sum; the threads' sums are
// added in a fixed order.
template <typename T> __global__ void __launch_bounds__(256) join_kernel(const DecodeArgs a) {
    constexpr int vecs = 8, lanes = 32;             // 32 columns a CTA, every 32nd chunk a thread
    __shared__ float4 acc[256];
    __shared__ float red[8], weight[256];
    const int64_t b = blockIdx.y, head = b * a.H + blockIdx.x, h = blockIdx.x / (unsigned)a.G;
    const int tid = threadIdx.x, D = (int)a.D, v = blockIdx.z * vecs + tid % vecs, k = tid / vecs;
    // Ahead of the wait: the lengths were complete before the decode kernel began, which is a plain launch, and that kernel
    // sets the same status bit (1.6 us of 106 for 4 sequences of 32768 tokens).
    const RowTokens row(a, b, h);
    const int64_t chunk = row.chunk(a);
    pdl_wait();
    if (chunk >= row.n) return;                      // written by its only chunk
    const int n = (int)((row.n + chunk - 1) / chunk);
    const float2 *st = a.stats + head * a.nsplit;
    const float *part = a.part + head * a.nsplit * D;
    const float2 first = tid < n ? st[tid] : make_float2(-INFINITY, 0.f);
    float top = first.x;
    for (int i = tid + 256; i < n; i += 256) top = fmaxf(top, st[i].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (tid % 32 == 0) red[tid / 32] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) top = fmaxf(top, red[i]);
    const float ref = top == -INFINITY ? 0.f : top;
    float sum = 0.f;                                 // this thread's chunks; added up below
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i0 = 0; i0 < n; i0 += 256) {
        const float2 mine = i0 == 0 ? first : i0 + tid < n ? st[i0 + tid] : make_float2(-INFINITY, 0.f);
        const float w0 = exp2f(mine.x - ref);
        sum += mine.y * w0;
        __syncthreads();
        weight[tid] = w0;
        __syncthreads();
        const int m = min(256, n - i0);
        if (v * 4 < D)
#pragma unroll 4
            for (int i = k; i < m; i += lanes) {
                const float4 y = *reinterpret_cast<const float4 *>(part + (int64_t)(i0 + i) * D + v * 4);
                const float w = weight[i];
                x.x = fmaf(y.x, w, x.x); x.y = fmaf(y.y, w, x.y); x.z = fmaf(y.z, w, x.z); x.w = fmaf(y.w, w, x.w);
            }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    acc[tid] = x;
    __syncthreads();
    if (tid % 32 == 0) red[tid / 32] = sum;
    __syncthreads();
    if (k > 0 || v * 4 >= D) return;
    sum = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += red[i];
    for (int i = 1; i < lanes; ++i) {
        const float4 y = acc[i * vecs + tid];
        x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
    }
    const float f = sum == 0.f ? 0.f : 1.f / sum;
    T *o = (T *)a.o + head * D + v * 4;
    o[0] = Elem<T>::from_f(x.x * f); o[1] = Elem<T>::from_f(x.y * f); o[2] = Elem<T>::from_f(x.z * f); o[3] = Elem<T>::from_f(x.w * f);
}

int launch_rows(void (*kernel)(const DecodeArgs), const DecodeArgs &a, size_t smem, cudaStream_t s) {
    if (int rc = ensure_dynamic_smem((const void *)kernel, smem, "shared memory of the paged decode")) return rc;
    cudaLaunchConfig_t cfg = {};
    // heads fastest: the CTAs that read neighbouring rows of a page run side by side
    cfg.gridDim = dim3((unsigned)(a.Hkv * a.tiles), (unsigned)a.nsplit, (unsigned)a.B);
    cfg.blockDim = dim3(128);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 1;
    attr[0].val.clusterDim.y = (unsigned)a.nsplit;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = a.cluster ? 1 : 0;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a);
    return e == cudaSuccess ? MAT_OK : cuda_fail(e, "launching the paged decode");
}

template <typename T, int LPK, int NV, int GT> int launch_simt(const DecodeArgs &a, cudaStream_t s) {
    constexpr int U = NV == 1 ? 4 : 2;
    const size_t smem = (4 * GT * (a.D + 2) + (a.cluster ? GT * (a.D + 4) : 0)) * sizeof(float);
    return launch_rows(a.cluster ? decode_simt_kernel<T, LPK, NV, GT, U, true> : decode_simt_kernel<T, LPK, NV, GT, U, false>, a, smem, s);
}

template <typename T, int LPK, int NV> int launch_simt_heads(const DecodeArgs &a, int gt, cudaStream_t s) {
    switch (gt) {
        case 1: return launch_simt<T, LPK, NV, 1>(a, s);
        case 2: return launch_simt<T, LPK, NV, 2>(a, s);
        case 8: if constexpr (sizeof(T) == 4 && NV == 1) return launch_simt<T, LPK, NV, 8>(a, s);
        default: return launch_simt<T, LPK, NV, 4>(a, s);
    }
}

template <typename T, int DP, int NS> int launch_mma(const DecodeArgs &a, cudaStream_t s) {
    const size_t ring = 4 * NS * 2 * 16 * (DP + 8) * sizeof(T), res = ((a.cluster ? 5 : 4) * 16 * (DP + 4) + 128) * sizeof(float);
    return launch_rows(a.cluster ? decode_mma_kernel<T, DP, NS, true> : decode_mma_kernel<T, DP, NS, false>, a, ring > res ? ring : res, s);
}

template <typename T> int run_simt(DecodeArgs &a, cudaStream_t s) {
    const int64_t G = a.H / a.Hkv;
    const int vecs = (int)(a.D * sizeof(T) / 16);
    // eight heads a CTA where the registers allow it: 306 us against 362 for 32 fp32 sequences of up to 8192 tokens with 64
    // heads on 8 of 128 columns
    const int gt = G >= 8 && sizeof(T) == 4 && vecs <= 32 ? 8 : G >= 4 ? 4 : (G >= 2 ? 2 : 1);
    a.tiles = (int)((G + gt - 1) / gt);
    return vecs <= 8 ? launch_simt_heads<T, 8, 1>(a, gt, s)
         : vecs <= 16 ? launch_simt_heads<T, 16, 1>(a, gt, s)
         : vecs <= 32 ? launch_simt_heads<T, 32, 1>(a, gt, s) : launch_simt_heads<T, 32, 2>(a, gt, s);
}

// Ring places: at 256 columns three fit as well (one CTA a SM either way) but start later: one sequence of 4000 tokens x
// 4 heads of 256 takes 20.4 us with three and 18.8 with two, 64 of 8192 x 8 heads 663 and 667.
template <typename T> int run_mma(DecodeArgs &a, cudaStream_t s) {
    a.tiles = (int)((a.H / a.Hkv + 15) / 16);
    return a.D <= 64 ? launch_mma<T, 64, 3>(a, s) : a.D <= 128 ? launch_mma<T, 128, 3>(a, s) : launch_mma<T, 256, 2>(a, s);
}
template <> int run_mma<float>(DecodeArgs &a, cudaStream_t s) { return run_simt<float>(a, s); }

template <typename T> int launch_decode(DecodeArgs &a, cudaStream_t s) {
    const int rc = a.aligned ? run_mma<T>(a, s) : run_simt<T>(a, s);
    if (rc || a.nsplit == 1 || a.cluster) return rc;
    const cudaError_t e = a.nsplit <= 32 ? launch_after(join_few_kernel<T>, dim3((unsigned)((a.H * a.B + 3) / 4)), dim3(128), 0, s, a)
                                         : launch_after(join_kernel<T>, dim3((unsigned)a.H, (unsigned)a.B, (unsigned)((a.D + 31) / 32)), dim3(256), 0, s, a);
    return e == cudaSuccess ? MAT_OK : cuda_fail(e, "launching the paged decode's join");
}

// How many chunks a row may have, and their least size.  The lengths are on the device, so both come from the page
// table's width; the kernels shorten the chunks' number, not their size, for shorter rows.  One sequence of 777 tokens x 8
// heads of 64 takes 9.8 us under a table for up to 8192 tokens and 13.9 under any wider one.
struct DecodePlan { int nsplit, min_chunk, cluster; };

DecodePlan plan(const mat_paged_cache *c, int64_t B, int64_t width, int64_t left, int64_t n_sel) {
    int64_t most = width * c->page_size;
    if (n_sel > 0) most = n_sel * c->page_size;
    else if (left >= 0 && left < most - 16) most = left + 16;   // up to 15 tokens before the window's first
    const int64_t rows = B * c->H_kv;
    DecodePlan p;
    if (rows * 8 <= kSms && most <= 8192) {       // one cluster of at most eight chunks per row, all of them resident
        p.min_chunk = 64;
        p.nsplit = (int)(most >= 8 * 64 ? 8 : (most + 63) / 64);
        p.cluster = p.nsplit > 1;
        return p;
    }
    // Every CTA pays some 4 us to look up its pages, fill its rings and write its result.  64 sequences of up to 8192
    // tokens x 8 key heads of 128: 172 us with chunks of 512 tokens and more, 163 with 1024, 159 with 2048; 32 x 2048
    // chosen tokens x 8: 78, 61, 53 us.  Few rows need the shorter chunks to fill the GPU, and below 16 rows of up to 65536
    // tokens chunks of 128: 46 us against 56 with 512 for one fp32 sequence of 60000 tokens x 1 head of 128 (16-bit: 24 us
    // either way; 8 heads of 64: 37 against 33).  Elsewhere 512: 131072 tokens x 1 head 24 against 41 with 128, 16 x 2048 x 8
    // heads 35 against 56, 4 x 9000 x 4 heads 26 against 31 (fp32, 4 x 16000 x 8 heads: 136 against 128).
    p.min_chunk = rows >= kSms ? 2048 : rows >= 16 || most > 65536 ? 512 : 128;
    int64_t cap = 16 * kSms / rows;
    if (cap < 8) cap = 8;
    const int64_t n = (most + p.min_chunk - 1) / p.min_chunk;
    p.nsplit = (int)(n < 1 ? 1 : n > cap ? cap : n);
    p.cluster = p.nsplit > 1 && p.nsplit <= 8 && rows * p.nsplit <= kSms;
    return p;
}

int check_decode(const mat_paged_cache *c, int64_t B, int64_t H, int64_t left, int64_t n_sel) {
    if (H < c->H_kv || H % c->H_kv) return fail(MAT_ERR_INVALID, "H = %lld query heads do not divide over H_kv = %lld key heads", (long long)H, (long long)c->H_kv);
    if (H > 65535) return fail(MAT_ERR_UNSUPPORTED, "at most 65535 query heads");
    if (n_sel < 0 || n_sel > INT_MAX / c->page_size) return fail(MAT_ERR_INVALID, "the list of pages is too long");
    (void)B; (void)left;
    return MAT_OK;
}

size_t align256(size_t x) { return (x + 255) / 256 * 256; }

}  // namespace
}  // namespace mat

using namespace mat;

extern "C" size_t mat_paged_decode_workspace_bytes(const mat_paged_cache *cache, int64_t B, int64_t H, int64_t table_width,
                                                   int64_t left, int64_t n_sel) {
    if (check_paged_cache(cache) || B < 1 || H < 1 || table_width < 1 || check_decode(cache, B, H, left, n_sel)) return 0;
    const DecodePlan p = plan(cache, B, table_width, left, n_sel);
    if (p.nsplit == 1 || p.cluster) return 0;
    return align256((size_t)B * H * p.nsplit * sizeof(float2)) + (size_t)B * H * p.nsplit * cache->D * sizeof(float);
}

extern "C" int mat_paged_decode(const mat_paged_cache *cache, const void *q, int64_t q_stride, void *o, int64_t B, int64_t H,
                                const int32_t *page_table, int64_t table_width, int64_t table_stride,
                                const int32_t *lengths, int64_t left, int64_t dilation, const int32_t *pages,
                                int64_t n_sel, float scale, void *workspace, size_t workspace_bytes, void *stream) {
    if (int rc = check_paged_cache(cache)) return rc;
    if (int rc = check_page_table(page_table, table_width, table_stride, B)) return rc;
    if (int rc = check_decode(cache, B, H, left, n_sel)) return rc;
    if (!q || !o || !lengths) return fail(MAT_ERR_INVALID, "q, o and lengths must be non-NULL");
    if (((uintptr_t)q | (uintptr_t)o) % 16 || q_stride < 0 || q_stride * (int64_t)dtype_size(cache->dtype) % 16)
        return fail(MAT_ERR_INVALID, "q and o must be 16-byte aligned and q's stride a multiple of 16 bytes");
    if (left >= 0 && dilation < 1) return fail(MAT_ERR_INVALID, "dilation must be >= 1");
    if (pages && n_sel < 1) return fail(MAT_ERR_INVALID, "a list of pages needs at least one entry per row");
    if (pages && left >= 0) return fail(MAT_ERR_INVALID, "a list of pages and a window cannot be combined");
    const size_t need = mat_paged_decode_workspace_bytes(cache, B, H, table_width, left, pages ? n_sel : 0);
    if (need > 0 && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 256))
        return fail(MAT_ERR_WORKSPACE, "workspace of %zu bytes (256-byte aligned) required, got %zu", need, workspace ? workspace_bytes : (size_t)0);
    DecodeArgs a;
    a.c = paged_view(cache, page_table, table_width, table_stride);
    a.q = q; a.o = o; a.q_stride = q_stride;
    a.B = B; a.H = H; a.Hkv = cache->H_kv; a.D = cache->D;
    a.G = (int)(H / cache->H_kv);
    a.lengths = lengths; a.left = left; a.dilation = dilation;
    a.pages = pages; a.n_sel = n_sel;
    a.scale_log2 = (scale > 0.f ? scale : 1.0f / std::sqrt((float)cache->D)) * 1.4426950408889634f;
    const DecodePlan w = plan(cache, B, table_width, left, pages ? n_sel : 0);
    a.nsplit = w.nsplit; a.min_chunk = w.min_chunk; a.cluster = w.cluster;
    a.stats = (float2 *)workspace;
    a.part = (float *)((char *)workspace + align256((size_t)B * H * a.nsplit * sizeof(float2)));
    if (!(a.status = paged_status_word())) return fail(MAT_ERR_CUDA, "no device status word");
    // 16 neighbouring tokens at a time on the tensor cores: 16-bit types, pages of 16 tokens and more, no dilation
    a.aligned = cache->dtype != MAT_F32 && cache->page_size >= 16 && (left < 0 || dilation == 1);
    note_kernel(a.aligned ? "paged_decode_mma" : "paged_decode_simt");
    cudaStream_t s = (cudaStream_t)stream;
    switch (cache->dtype) {
        case MAT_F32: return launch_decode<float>(a, s);
        case MAT_BF16: return launch_decode<__nv_bfloat16>(a, s);
        default: return launch_decode<__half>(a, s);
    }
}
