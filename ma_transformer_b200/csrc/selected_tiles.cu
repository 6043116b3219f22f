// Block-selected attention in tiles: 16-bit types on the warp-level tensor-core instructions (here), fp32 on the FMA pipe
// (selected_f32.cuh).
//
// Queries of one sequence choose different blocks, so a tile of neighbouring queries shares no keys.  The selection is
// turned round instead: per block the list of the rows (query, head) that chose it, gathered 16 or 64 at a time into
// dense tiles against the block's keys, which stay in shared memory.  A row meets its blocks in different CTAs, so each
// leaves a partial result in fp32 (forward: maximum, sum, unnormalised output; backward: its share of dq), and a second
// kernel joins a row's partials in the order of its list.  dk and dv of a block are summed over its rows by one CTA per
// `rows per item` rows and then over the items in order: nothing depends on timing, there are no atomics.
//
// The partials are the traffic: 4 D bytes written and read per (row, block) against 2 D for the gathered query, so the
// (batch, key head) pairs are worked off in groups whose partials and lists take at most kPairBudget bytes (one pair where
// that takes more; beside them the backward holds 4 bytes a row).  Groups small enough for
// L2 (64 MB) were slower than all pairs at once, for the tails of their launches: 281 + 446 against 247 + 377 us forward
// and backward at 8192 tokens x 8 heads of 64 x 16 blocks, so the budget only bounds the workspace.
#include <cmath>

#include "paged.cuh"
#include "selected_attn.cuh"
#include "pdl.cuh"
#include "ptx.cuh"

namespace mat {
namespace {

constexpr int kFwdRows = 256;        // rows per forward item (a multiple of 64)
// rows per item in fp32.  Backward: 64 instead of 128 rows, twice the CTAs: 563 -> 462 us at 4096 x 8 heads of 64 x 8 blocks
// of 64, 75 -> 62 at 2 x 1000 x 4 heads of 32; forward with 64: 241 -> 259.
constexpr int kF32Rows = 128, kF32BwdRows = 64;
constexpr int kBwdRows = 512;        // rows per backward item
constexpr size_t kPairBudget = 1024ull << 20;

struct SelTile {                     // what the kernels need beside SelProblem
    SelLists l;
    int2 *items;                     // [group bh][max_items] (block, first row)
    int32_t *item_base;              // [group bh][nb + 1]
    int64_t max_items;
    float2 *stats;                   // [group rows][slots]
    float *part;                     // [group rows][slots][D]
    float *kv_part;                  // [group bh][max_items][nsub][2][kv_rows][D]
    const float *delta;
    float *delta_part;               // [group rows][slots][nsub]: shares of delta (few keys a row)
    int64_t bh0;                     // first (batch, key head) of the group
    int G, nsub, kv_rows;            // kv_rows: keys of a (sub-)block, 64 at most
    float scale_log2;
};

template <typename T> __device__ __forceinline__ void store4(T *at, const float4 &x) {
    T y[4] = {Elem<T>::from_f(x.x), Elem<T>::from_f(x.y), Elem<T>::from_f(x.z), Elem<T>::from_f(x.w)};
    if (sizeof(T) == 4) *reinterpret_cast<float4 *>(at) = *reinterpret_cast<const float4 *>(&x);
    else *reinterpret_cast<uint2 *>(at) = *reinterpret_cast<uint2 *>(y);
}
__device__ __forceinline__ void cp_async16(void *dst, const void *src, bool in) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(ptx::smem_u32(dst)), "l"(src), "r"(in ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// rows [0, n) of `rows` into shared memory, the rest zeros; columns from D on are zeros
template <typename T, int DP>
__device__ __forceinline__ void stage_keys(T *dst, const T *src, int64_t row_stride, int n, int rows, int D) {
    for (int i = threadIdx.x; i < rows * (DP / 8); i += 128) {
        const int r = i / (DP / 8), c = i % (DP / 8) * 8;
        const bool in = r < n && c < D;
        cp_async16(dst + r * (DP + 8) + c, in ? src + r * row_stride + c : src, in);
    }
}

// Zero does not silence an infinity or a NaN, so the zero weights of pairs that do not see each other need finite factors.
// Only tiles whose rows see part of the keys (the queries of a causal block itself) have such pairs, and there a value of
// that kind shows in the tile's scores or dP.  Such a tile forms its gradients from zeros in those values' place, and this
// says what the pairs that see them get: rows see the first `vis` keys, so it is enough to know, column by column, the first
// such key, and how many keys the rows with such a value see.  Looking for them takes 9 of 252 us of the backward tiles at
// 8192 tokens x 8 heads of 64 x 16 blocks of 64 (2 of 460 at 4096 x 2 x 16 heads of 128).
template <int DP> struct OddColumns {
    int key[DP];                         // first key with such a value; 64: none
    int q[DP];                           // keys that see such a query: NaN in dk (the row's weights are NaN)
    int nan[DP], up[DP], down[DP];       // keys that see such an output gradient: a NaN, an infinity of either sign, in dv
    __device__ __forceinline__ void clear(int threads) {
        for (int x = threadIdx.x; x < DP; x += threads) {
            key[x] = 64;
            q[x] = nan[x] = up[x] = down[x] = 0;
        }
    }
    __device__ __forceinline__ void see_key(int row, int col) { atomicMin(&key[col], row); }
    __device__ __forceinline__ void see_query(int vis, int col) { atomicMax(&q[col], vis); }
    __device__ __forceinline__ void see_grad(float x, int vis, int col) { atomicMax(x != x ? &nan[col] : x > 0.f ? &up[col] : &down[col], vis); }
    __device__ __forceinline__ float dq(float x, int vis, int col) const { return vis > key[col] ? NAN : x; }
    __device__ __forceinline__ float dk(float x, int row, int col) const { return row < q[col] ? NAN : x; }
    __device__ __forceinline__ float dv(float x, int row, int col) const {
        return x + (row < nan[col] ? NAN : 0.f) + (row < up[col] ? INFINITY : 0.f) - (row < down[col] ? INFINITY : 0.f);
    }
};

}  // namespace
}  // namespace mat
#include "selected_f32.cuh"
namespace mat {
namespace {

// ---- forward ----------------------------------------------------------------------------------------------------------
// One warp per 16 rows, NKP keys at a time; keys and values of the block are shared by the CTA's warps, each warp's
// queries have two buffers of their own.  120 to 129 us at 8192 tokens x 8 heads of 64 x 16 blocks of 64 (ncu: L1 73 % busy,
// tensor pipe 25 to 27 %, DRAM 23 %), where the partials alone are 268 MB written (41 us).  Tried and not faster: 32 rows a
// warp sharing each key fragment (126 us at 168 registers), partials leaving through shared memory as bulk copies of a
// row each (135 us).  NKP = 32 instead of 64 in the exact kernels: 220 against 226 us for the whole forward.
// EXACT: D == DP and a block is a whole number of NKP keys, known to the compiler.
template <typename T, int DP, int NKP, bool EXACT> __global__ void __launch_bounds__(128, DP == 64 ? 4 : 3) sel_fwd_mma_kernel(const SelProblem p, const SelTile t) {
    constexpr int PITCH = DP + 8, NF = NKP / 8;
    const int64_t bhl = blockIdx.y;
    const int bh = (int)t.bh0 + blockIdx.y;
    const int64_t b = bh / (int)p.Hkv, h = bh - b * p.Hkv;
    pdl_trigger();
    pdl_wait();
    if ((int)blockIdx.x >= t.item_base[bhl * (p.nb + 1) + p.nb]) return;
    const int2 item = t.items[bhl * t.max_items + blockIdx.x];
    const int n = item.x, e0 = t.l.base[bhl * (p.nb + 1) + n];
    const int rows_all = (t.l.base[bhl * (p.nb + 1) + n + 1] - e0) * t.G;
    const int r_end = min(item.y + kFwdRows, rows_all);
    const int D = EXACT ? DP : (int)p.D, d16 = EXACT ? DP / 16 : (D + 15) / 16, block = (int)p.block, T_ = (int)p.topk;
    const int64_t j0 = (int64_t)n * block;
    const int held = (int)min((int64_t)block, p.S - j0);
    extern __shared__ __align__(16) char smem[];
    const int key_rows = (block + NKP - 1) / NKP * NKP;
    T *ks = (T *)smem, *vs = ks + key_rows * PITCH;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    T *qs = vs + key_rows * PITCH + warp * 2 * 16 * PITCH;
    const int64_t krow = p.Hkv * D;
    const T *kg = (const T *)p.k + ((b * p.S + j0) * p.Hkv + h) * D, *vg = (const T *)p.v + ((b * p.S + j0) * p.Hkv + h) * D;
    stage_keys<T, DP>(ks, kg, krow, held, key_rows, D);
    stage_keys<T, DP>(vs, vg, krow, held, key_rows, D);
    cp_async_commit();
    // the item's rows: query (-1 past the end), row of q within the batch item, place of the partial within the pair
    __shared__ int row_q[kFwdRows], row_src[kFwdRows], row_at[kFwdRows];
    for (int x = threadIdx.x; x < kFwdRows; x += 128) {
        const int r = item.y + x;
        int i = -1, src = 0, at = 0;
        if (r < r_end) {
            const int e = r / t.G, g = r - e * t.G, entry = t.l.entry[bhl * p.S * T_ + e0 + e];
            i = entry / T_;
            src = i * (int)p.H + g;
            at = (i * t.G + g) * T_ + entry - i * T_;
        }
        row_q[x] = i; row_src[x] = src; row_at[x] = at;
    }
    const int64_t part0 = (int64_t)blockIdx.y * p.S * t.G * T_;
    const T *q0 = (const T *)p.q + (b * p.S * p.H + h * t.G) * D;
    auto stage_rows = [&](T *dst, int x) {
#pragma unroll
        for (int c = lane; c < 16 * (DP / 8); c += 32) {
            const int r = c / (DP / 8), col = c % (DP / 8) * 8;
            const bool in = row_q[x + r] >= 0 && (EXACT || col < D);
            cp_async16(dst + r * PITCH + col, q0 + (int64_t)row_src[x + r] * D + (in ? col : 0), in);
        }
    };
    __shared__ uint32_t odd_keys[4];
    if (threadIdx.x < 4) odd_keys[threadIdx.x] = 0;
    __syncthreads();
    int first = item.y + warp * 16, cur = 0;
    if (first < r_end) stage_rows(qs, first - item.y);
    cp_async_commit();
    cp_async_wait<1>();          // the block's keys and values
    __syncthreads();
    // A weight of zero does not silence a value that is infinite or NaN (a padded token behind the query, say), so such
    // values go into the product as zeros and are added to the rows that see them.
    constexpr uint32_t kExp = sizeof(T) == 2 && ptx::Mma<T>::kOnes == 0x3F803F80u ? 0x7f80u : 0x7c00u;
    for (int x = threadIdx.x; x < held * (DP / 8); x += 128) {
        T *at = vs + x / (DP / 8) * PITCH + x % (DP / 8) * 8;
        const uint4 u = *reinterpret_cast<const uint4 *>(at);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
        bool any = false;
#pragma unroll
        for (int y = 0; y < 4; ++y) any |= (w[y] & kExp) == kExp || (w[y] >> 16 & kExp) == kExp;
        if (any) {
            for (int y = 0; y < 8; ++y) {
                const float f = Elem<T>::to_f(at[y]);
                if (f - f != 0.f) at[y] = Elem<T>::from_f(0.f);
            }
            atomicOr(&odd_keys[x / (DP / 8) / 32], 1u << (x / (DP / 8) % 32));
        }
    }
    __syncthreads();
    const bool odd = (odd_keys[0] | odd_keys[1] | odd_keys[2] | odd_keys[3]) != 0;
    for (; first < r_end; first += 64) {
        if (first + 64 < r_end) stage_rows(qs + (cur ^ 1) * 16 * PITCH, first + 64 - item.y);
        cp_async_commit();
        cp_async_wait<1>();
        __syncwarp();
        const T *q = qs + cur * 16 * PITCH;
        uint32_t qf[DP / 16][4];
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk)
            if (kk < d16) ptx::ldmatrix_x4(qf[kk], ptx::smem_u32(q + (lane % 16) * PITCH + kk * 16 + (lane / 16) * 8));
        // keys of the block that a row sees: the first `vis`
        const int i = row_q[first - item.y + lane % 16];
        const int mine = i < 0 ? 0 : p.causal ? min(held, (int)(i + 1 - j0)) : held;
        const int vis0 = __shfl_sync(0xffffffffu, mine, lane / 4), vis1 = __shfl_sync(0xffffffffu, mine, lane / 4 + 8);
        const bool full = __all_sync(0xffffffffu, mine == block);
        float o[DP / 8][4];
#pragma unroll
        for (int c = 0; c < DP / 8; ++c) o[c][0] = o[c][1] = o[c][2] = o[c][3] = 0.f;
        float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
        for (int base = 0; base < held; base += NKP) {
            const int n16 = EXACT ? NKP / 16 : min(NKP, block - base) / 16;
            float s[NF][4];
#pragma unroll
            for (int c = 0; c < NF; ++c) s[c][0] = s[c][1] = s[c][2] = s[c][3] = 0.f;
#pragma unroll
            for (int kk = 0; kk < DP / 16; ++kk)
                if (kk < d16)
#pragma unroll
                    for (int c = 0; c < NF / 2; ++c)
                        if (c < n16) {
                            uint32_t r[4];
                            ptx::ldmatrix_x4(r, ptx::smem_u32(ks + (base + c * 16 + lane % 8 + (lane / 16) * 8) * PITCH + kk * 16 + (lane / 8 % 2) * 8));
                            ptx::Mma<T>::run(s[2 * c], qf[kk], r[0], r[1]);
                            ptx::Mma<T>::run(s[2 * c + 1], qf[kk], r[2], r[3]);
                        }
            float t0 = -INFINITY, t1 = -INFINITY;
#pragma unroll
            for (int c = 0; c < NF; ++c) {
                if (!full) {
                    const int col = base + c * 8 + (lane % 4) * 2;
                    if (col >= vis0) s[c][0] = -INFINITY;
                    if (col + 1 >= vis0) s[c][1] = -INFINITY;
                    if (col >= vis1) s[c][2] = -INFINITY;
                    if (col + 1 >= vis1) s[c][3] = -INFINITY;
                } else if (!EXACT && c / 2 >= n16) {
                    s[c][0] = s[c][1] = s[c][2] = s[c][3] = -INFINITY;
                }
                t0 = fmaxf(t0, fmaxf(s[c][0], s[c][1]));
                t1 = fmaxf(t1, fmaxf(s[c][2], s[c][3]));
            }
#pragma unroll
            for (int x = 1; x < 4; x <<= 1) {
                t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, x));
                t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, x));
            }
            t0 = fmaxf(m0, t0 * t.scale_log2);
            t1 = fmaxf(m1, t1 * t.scale_log2);
            const float ref0 = t0 == -INFINITY ? 0.f : t0, ref1 = t1 == -INFINITY ? 0.f : t1;
            const float keep0 = ptx::ex2(m0 - ref0), keep1 = ptx::ex2(m1 - ref1);
            m0 = t0; m1 = t1;
            l0 *= keep0; l1 *= keep1;
            if (base > 0)
#pragma unroll
                for (int c = 0; c < DP / 8; ++c) { o[c][0] *= keep0; o[c][1] *= keep0; o[c][2] *= keep1; o[c][3] *= keep1; }
            uint32_t pf[NF / 2][4];
#pragma unroll
            for (int c = 0; c < NF; ++c) {
                const float a = ptx::ex2(fmaf(s[c][0], t.scale_log2, -ref0)), bb = ptx::ex2(fmaf(s[c][1], t.scale_log2, -ref0));
                const float cc = ptx::ex2(fmaf(s[c][2], t.scale_log2, -ref1)), d = ptx::ex2(fmaf(s[c][3], t.scale_log2, -ref1));
                l0 += a + bb;
                l1 += cc + d;
                // the weights are rounded to the inputs' type for the tensor cores: one more rounding of the kind the
                // output has; their sum is kept in fp32
                pf[c / 2][(c % 2) * 2] = ptx::Mma<T>::pack(a, bb);
                pf[c / 2][(c % 2) * 2 + 1] = ptx::Mma<T>::pack(cc, d);
            }
#pragma unroll
            for (int kk = 0; kk < NF / 2; ++kk)
                if (kk < n16)
#pragma unroll
                    for (int c = 0; c < DP / 16; ++c)
                        if (c < d16) {
                            uint32_t r[4];
                            ptx::ldmatrix_x4_trans(r, ptx::smem_u32(vs + (base + kk * 16 + lane % 16) * PITCH + c * 16 + (lane / 16) * 8));
                            ptx::Mma<T>::run(o[2 * c], pf[kk], r[0], r[1]);
                            ptx::Mma<T>::run(o[2 * c + 1], pf[kk], r[2], r[3]);
                        }
        }
        if (odd)
            for (int j = 0; j < held; ++j) {
                if (!(odd_keys[j / 32] >> (j % 32) & 1)) continue;
#pragma unroll
                for (int c = 0; c < DP / 8; ++c)
#pragma unroll
                    for (int y = 0; y < 4; ++y) {
                        const int col = c * 8 + (lane % 4) * 2 + y % 2;
                        if (col >= D || j >= (y < 2 ? vis0 : vis1)) continue;
                        const float f = Elem<T>::to_f(vg[j * krow + col]);
                        if (f - f != 0.f) o[c][y] += f;
                    }
            }
#pragma unroll
        for (int x = 1; x < 4; x <<= 1) {
            l0 += __shfl_xor_sync(0xffffffffu, l0, x);
            l1 += __shfl_xor_sync(0xffffffffu, l1, x);
        }
        const int64_t at0 = part0 + row_at[first - item.y + lane / 4], at1 = part0 + row_at[first - item.y + lane / 4 + 8];
        const bool in0 = vis0 > 0, in1 = vis1 > 0;
        if (lane % 4 == 0) {
            if (in0) t.stats[at0] = make_float2(m0, l0);
            if (in1) t.stats[at1] = make_float2(m1, l1);
        }
#pragma unroll
        for (int c = 0; c < DP / 8; ++c) {
            const int col = c * 8 + (lane % 4) * 2;
            if (c * 8 < D) {
                if (in0) *reinterpret_cast<float2 *>(t.part + at0 * D + col) = make_float2(o[c][0], o[c][1]);
                if (in1) *reinterpret_cast<float2 *>(t.part + at1 * D + col) = make_float2(o[c][2], o[c][3]);
            }
        }
        __syncwarp();
        cur ^= 1;
    }
    cp_async_wait<0>();
}

// Joins a row's partials in the order of its list: LPR lanes of 4 columns per row.  The lanes look at LPR entries of the
// list together (which count, and with what weight) while the first AHEAD partials are on their way.
// BWD: the sum of a row's shares of dq.
template <typename T, int LPR, int AHEAD, bool BWD> __global__ void __launch_bounds__(128) sel_join_kernel(const SelProblem p, const SelTile t) {
    const uint32_t x0 = blockIdx.x * (128u / LPR) + threadIdx.x / LPR, G = t.G;                 // (i, g) of the pair; S G < 2^31
    const int lane = threadIdx.x % LPR, col = lane * 4, D = (int)p.D, T_ = (int)p.topk;
    pdl_trigger();
    pdl_wait();
    const bool live = x0 < (uint32_t)p.S * G, in = live && col < D;
    const uint32_t x = live ? x0 : 0;
    const int i = (int)(x / G), g = (int)(x - i * G);
    const int bh = (int)t.bh0 + blockIdx.y;
    const int64_t b = bh / (int)p.Hkv, h = bh - b * p.Hkv;
    const int64_t rr = (int64_t)blockIdx.y * p.S * G + x;                                       // among the group's rows
    const int32_t *list = p.blocks + ((b * p.S + i) * p.Hkv + h) * T_;
    const int limit = p.causal ? i / (int)p.block + 1 : (int)p.nb;
    const int64_t out = ((b * p.S + i) * p.H + h * G + g);
    const float *part = t.part + rr * T_ * t.nsub * D + col;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float m = -INFINITY, l = 0.f;
    int prev = -1;
    const int subs = BWD ? t.nsub : 1;
    for (int s0 = 0; s0 < T_; s0 += LPR) {
        const int s = s0 + lane, cnt = min(LPR, T_ - s0);
        // the first partials are read before it is known whether they count: three dependent reads become two
        float4 ahead[AHEAD];
#pragma unroll
        for (int y = 0; y < AHEAD; ++y)
            ahead[y] = in && y < cnt ? *reinterpret_cast<const float4 *>(part + (s0 + y) * subs * (int64_t)D) : make_float4(0.f, 0.f, 0.f, 0.f);
        const float2 st0 = !BWD && live && s < T_ ? t.stats[rr * T_ + s] : make_float2(-INFINITY, 0.f);
        const int n = s < T_ ? list[s] : -1;
        int top = n;                                   // largest entry up to this lane's
#pragma unroll
        for (int x = 1; x < LPR; x <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, top, x, LPR);
            if (lane >= x) top = max(top, y);
        }
        int before = __shfl_up_sync(0xffffffffu, top, 1, LPR);
        before = lane == 0 ? prev : max(prev, before);
        const bool counts = n > before && n < limit;
        prev = max(prev, __shfl_sync(0xffffffffu, top, LPR - 1, LPR));
        // BWD: how many sub-blocks of the block hold keys
        int uses = counts ? 1 : 0;
        float w = counts ? 1.f : 0.f;
        if (BWD) {
            if (counts) uses = min(t.nsub, (int)((p.S - (int64_t)n * p.block + 63) / 64));
        } else {
            const float2 st = counts ? st0 : make_float2(-INFINITY, 0.f);
            float mx = st.x;
#pragma unroll
            for (int x = LPR / 2; x > 0; x >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x, LPR));
            const float now = fmaxf(m, mx), ref = now == -INFINITY ? 0.f : now, keep = exp2f(m - ref);
            m = now;
            w = exp2f(st.x - ref);
            float sum = st.y * w;
#pragma unroll
            for (int x = LPR / 2; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x, LPR);
            l = l * keep + sum;
            acc.x *= keep; acc.y *= keep; acc.z *= keep; acc.w *= keep;
        }
        auto add = [&](const float4 &x, float f) {
            acc.x = fmaf(x.x, f, acc.x); acc.y = fmaf(x.y, f, acc.y); acc.z = fmaf(x.z, f, acc.z); acc.w = fmaf(x.w, f, acc.w);
        };
#pragma unroll
        for (int y = 0; y < AHEAD; ++y) {
            const int use = __shfl_sync(0xffffffffu, uses, y, LPR);
            const float f = __shfl_sync(0xffffffffu, w, y, LPR);
            if (use) add(ahead[y], f);                 // what nobody wrote may be NaN: skipped, not weighted with zero
            if (BWD)
                for (int u = 1; u < use; ++u)
                    if (in) add(*reinterpret_cast<const float4 *>(part + ((s0 + y) * subs + u) * (int64_t)D), 1.f);
        }
#pragma unroll 8
        for (int y = AHEAD; y < cnt; ++y) {
            const int use = __shfl_sync(0xffffffffu, uses, y, LPR);
            const float f = __shfl_sync(0xffffffffu, w, y, LPR);
            for (int u = 0; u < use; ++u)
                if (in) add(*reinterpret_cast<const float4 *>(part + ((s0 + y) * subs + u) * (int64_t)D), f);
        }
    }
    if (!in) return;
    float f = BWD ? p.scale : 1.f / l;
    if (!BWD && l == 0.f) {                            // no keys: zeros; keys that all score -inf: NaN, the softmax of such a row
        f = 0.f;
        prev = -1;
        for (int s = 0; s < T_; ++s)
            if (sel_entry_counts(list[s], prev, limit)) f = NAN;
    }
    if (!BWD && lane == 0) p.lse[out] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f;
    store4((T *)(BWD ? p.dq : p.out) + out * D + col, make_float4(acc.x * f, acc.y * f, acc.z * f, acc.w * f));
}

// ---- backward ---------------------------------------------------------------------------------------------------------
// A tile is 64 rows against up to NKP keys of one (sub-)block.  Warp w scores rows 16 w .. 16 w + 15 and writes their
// share of dq; for dk and dv the weights and dS go through shared memory and warp w owns 16 keys (NKP = 64), or 16 keys
// and half of the columns (NKP = 32).  Seven products of 16 x 64 x 64 per 16 rows (dq and dk count twice): 252 us at 8192 tokens x
// 8 heads of 64 x 16 blocks of 64, tensor pipe 44 %, L1 67 % busy (fragments, P and dS, gathered rows), two CTAs a SM by
// registers.  fp16 gradients want the loss scale that the library's other 16-bit backward kernels want: dS is held in
// the inputs' type.
// DELTA: the tile leaves each row's share of delta = sum p dp instead of gradients.  Where a row has few keys its output is
// as large as a value, and delta taken from the rounded output is off by as much as dS's own rounding: dq and dk of rows
// of up to 16 keys were 1.8 and 1.7 times as far off as a rounding of the result alone (of 553 rows that see their own
// block of 128 only, 1.6 times), against 1.1 to 1.4 where rows see two blocks and more.
template <typename T, int DP, int NKP, bool EXACT, bool DELTA> __global__ void __launch_bounds__(128, 2) sel_bwd_mma_kernel(const SelProblem p, const SelTile t) {
    constexpr int PITCH = DP + 8, NF = NKP / 8, WP = NKP + 8, KW = NKP / 16, CW = 4 / KW, CF = DP / 16 / CW, NBUF = DP == 64 ? 2 : 1;
    const int64_t bhl = blockIdx.z;
    const int bh = (int)t.bh0 + blockIdx.z;
    const int64_t b = bh / (int)p.Hkv, h = bh - b * p.Hkv;
    pdl_trigger();
    pdl_wait();
    if ((int)blockIdx.x >= t.item_base[bhl * (p.nb + 1) + p.nb]) return;
    const int2 item = t.items[bhl * t.max_items + blockIdx.x];
    const int n = item.x, e0 = t.l.base[bhl * (p.nb + 1) + n], sub = blockIdx.y;
    const int rows_all = (t.l.base[bhl * (p.nb + 1) + n + 1] - e0) * t.G;
    const int r_end = min(item.y + kBwdRows, rows_all);
    const int D = EXACT ? DP : (int)p.D, d16 = EXACT ? DP / 16 : (D + 15) / 16, T_ = (int)p.topk;
    const int64_t j0 = (int64_t)n * p.block + sub * 64;
    const int keys = min((int)p.block - sub * 64, 64);                       // of the sub-block
    const int held = (int)max((int64_t)0, min((int64_t)keys, p.S - j0)), n16 = EXACT ? NKP / 16 : (keys + 15) / 16;
    if (held == 0) return;                                                    // the sequence ends before this half
    extern __shared__ __align__(16) char smem[];
    T *ks = (T *)smem, *vs = ks + NKP * PITCH, *qs = vs + NKP * PITCH, *ps = qs + NBUF * 128 * PITCH, *ds = ps + 64 * WP, *dr = ds + 64 * WP;
    int *row_q = (int *)(dr + 64 * WP), *row_at = row_q + kBwdRows;
    int *row_src = row_at + kBwdRows;
    float *row_lse = (float *)(row_src + kBwdRows), *row_delta = row_lse + kBwdRows;
    OddColumns<DP> &odd = *(OddColumns<DP> *)(row_delta + kBwdRows);
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int64_t krow = p.Hkv * D;
    stage_keys<T, DP>(ks, (const T *)p.k + ((b * p.S + j0) * p.Hkv + h) * D, krow, held, NKP, D);
    stage_keys<T, DP>(vs, (const T *)p.v + ((b * p.S + j0) * p.Hkv + h) * D, krow, held, NKP, D);
    cp_async_commit();
    for (int x = threadIdx.x; x < kBwdRows; x += 128) {
        const int r = item.y + x;
        int i = -1, at = 0, src = 0;
        float lse = 0.f, delta = 0.f;
        if (r < r_end) {
            const int e = r / t.G, g = r - e * t.G, entry = t.l.entry[bhl * p.S * T_ + e0 + e];
            i = entry / T_;
            at = (i * t.G + g) * T_ + entry - i * T_;
            src = i * (int)p.H + g;
            const int64_t row = b * p.S * p.H + h * t.G + src;
            lse = p.lse_in[row] * 1.4426950408889634f;
            if (!DELTA) delta = t.delta[row];
        }
        row_q[x] = i; row_at[x] = at; row_src[x] = src; row_lse[x] = lse; row_delta[x] = delta;
    }
    const int64_t part0 = (int64_t)bhl * p.S * t.G * T_;
    // queries and output gradients of 64 rows: warp w gathers (and scores) rows 16 w .. 16 w + 15
    const int64_t src0 = (b * p.S * p.H + h * t.G) * D;
    auto stage_rows = [&](T *dst, int x) {
#pragma unroll
        for (int c = lane; c < 16 * (DP / 8); c += 32) {
            const int r = warp * 16 + c / (DP / 8), col = c % (DP / 8) * 8;
            const bool in = row_q[x + r] >= 0 && (EXACT || col < D);
            const int64_t off = src0 + (int64_t)row_src[x + r] * D + (in ? col : 0);
            cp_async16(dst + r * PITCH + col, (const T *)p.q + off, in);
            cp_async16(dst + (64 + r) * PITCH + col, (const T *)p.dout + off, in);
        }
        cp_async_commit();
    };
    __syncthreads();
    stage_rows(qs, 0);
    float dk[CF][2][4], dv[CF][2][4];
#pragma unroll
    for (int c = 0; c < CF; ++c)
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int y = 0; y < 4; ++y) dk[c][x][y] = dv[c][x][y] = 0.f;
    const int kg = warp % KW, cg = warp / KW;          // this warp's keys and column half in the key pass
    const int ragged_end = p.causal ? (int)(j0 + held) - 1 : 0;        // queries below it see part of the keys
    bool odd_rows = false;                             // `odd` is in use
    int cur = 0;
    for (int first = item.y; first < r_end; first += 64, cur ^= NBUF - 1) {
        const T *qt = qs + cur * 128 * PITCH, *ot = qt + 64 * PITCH;
        cp_async_wait<0>();
        __syncthreads();                 // this tile is in; the other buffer, ps and ds are free again
        if (NBUF == 2 && first + 64 < r_end) stage_rows(qs + (cur ^ 1) * 128 * PITCH, first + 64 - item.y);
        const int x0 = first - item.y + warp * 16 + lane / 4, x1 = x0 + 8, i0 = row_q[x0], i1 = row_q[x1];
        const int vis0 = i0 < 0 ? 0 : p.causal ? max(0, (int)min((int64_t)held, i0 + 1 - j0)) : held;
        const int vis1 = i1 < 0 ? 0 : p.causal ? max(0, (int)min((int64_t)held, i1 + 1 - j0)) : held;
        const float lse0 = row_lse[x0], lse1 = row_lse[x1], del0 = row_delta[x0], del1 = row_delta[x1];
        float s[NF][4], dp[NF][4];
#pragma unroll
        for (int c = 0; c < NF; ++c)
#pragma unroll
            for (int y = 0; y < 4; ++y) s[c][y] = dp[c][y] = 0.f;
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk)
            if (kk < d16) {
                uint32_t qf[4], of[4];
                ptx::ldmatrix_x4(qf, ptx::smem_u32(qt + (warp * 16 + lane % 16) * PITCH + kk * 16 + (lane / 16) * 8));
                ptx::ldmatrix_x4(of, ptx::smem_u32(ot + (warp * 16 + lane % 16) * PITCH + kk * 16 + (lane / 16) * 8));
#pragma unroll
                for (int c = 0; c < NF / 2; ++c)
                    if (c < n16) {
                        uint32_t x[4];
                        const int row = c * 16 + lane % 8 + (lane / 16) * 8, col = kk * 16 + (lane / 8 % 2) * 8;
                        ptx::ldmatrix_x4(x, ptx::smem_u32(ks + row * PITCH + col));
                        ptx::Mma<T>::run(s[2 * c], qf, x[0], x[1]);
                        ptx::Mma<T>::run(s[2 * c + 1], qf, x[2], x[3]);
                        ptx::ldmatrix_x4(x, ptx::smem_u32(vs + row * PITCH + col));
                        ptx::Mma<T>::run(dp[2 * c], of, x[0], x[1]);
                        ptx::Mma<T>::run(dp[2 * c + 1], of, x[2], x[3]);
                    }
            }
        if constexpr (DELTA) {
            float sum0 = 0.f, sum1 = 0.f;
#pragma unroll
            for (int c = 0; c < NF; ++c) {
                const int col = c * 8 + (lane % 4) * 2;
                if (col < vis0) sum0 = fmaf(ptx::ex2(fmaf(s[c][0], t.scale_log2, -lse0)), dp[c][0], sum0);
                if (col + 1 < vis0) sum0 = fmaf(ptx::ex2(fmaf(s[c][1], t.scale_log2, -lse0)), dp[c][1], sum0);
                if (col < vis1) sum1 = fmaf(ptx::ex2(fmaf(s[c][2], t.scale_log2, -lse1)), dp[c][2], sum1);
                if (col + 1 < vis1) sum1 = fmaf(ptx::ex2(fmaf(s[c][3], t.scale_log2, -lse1)), dp[c][3], sum1);
            }
#pragma unroll
            for (int x = 1; x < 4; x <<= 1) {
                sum0 += __shfl_xor_sync(0xffffffffu, sum0, x);
                sum1 += __shfl_xor_sync(0xffffffffu, sum1, x);
            }
            if (lane % 4 == 0) {
                if (i0 >= 0) t.delta_part[(part0 + row_at[x0]) * t.nsub + sub] = sum0;
                if (i1 >= 0) t.delta_part[(part0 + row_at[x1]) * t.nsub + sub] = sum1;
            }
            if (NBUF == 1) {
                __syncthreads();
                if (first + 64 < r_end) stage_rows(qs, first + 64 - item.y);
            }
            continue;
        }
        const bool ragged = row_q[first - item.y] < ragged_end;        // a tile's first row has its lowest query
        float zero = 0.f;                              // NaN: a score or dP of a ragged tile is not finite
        if (ragged) {
#pragma unroll
            for (int c = 0; c < NF; ++c)
#pragma unroll
                for (int y = 0; y < 4; ++y) zero = fmaf(s[c][y], 0.f, zero);
            zero = fmaf(dp[0][0], 0.f, fmaf(dp[0][2], 0.f, zero));      // an output gradient shows in every column
        }
        uint32_t df[NF / 2][4], dl[NF / 2][4];
#pragma unroll
        for (int c = 0; c < NF; ++c) {
            const int col = c * 8 + (lane % 4) * 2;
            const float a = col < vis0 ? ptx::ex2(fmaf(s[c][0], t.scale_log2, -lse0)) : 0.f;
            const float bb = col + 1 < vis0 ? ptx::ex2(fmaf(s[c][1], t.scale_log2, -lse0)) : 0.f;
            const float cc = col < vis1 ? ptx::ex2(fmaf(s[c][2], t.scale_log2, -lse1)) : 0.f;
            const float d = col + 1 < vis1 ? ptx::ex2(fmaf(s[c][3], t.scale_log2, -lse1)) : 0.f;
            // Weights are rounded to the inputs' type for dv, one rounding of the kind the result has.  dq and dk also
            // have the rounded output's error in delta, so dS goes into them as two halves, rounded value and rest: for
            // bf16 1.9e-3 off instead of 2.6e-3 (dq), 1.9e-3 instead of 2.4e-3 (dk; 12 us of 350
            // at 8192 tokens x 8 heads of 64).
            const float ea = col < vis0 ? a * (dp[c][0] - del0) : 0.f, eb = col + 1 < vis0 ? bb * (dp[c][1] - del0) : 0.f;
            const float ec = col < vis1 ? cc * (dp[c][2] - del1) : 0.f, ed = col + 1 < vis1 ? d * (dp[c][3] - del1) : 0.f;
            const uint32_t p0 = ptx::Mma<T>::pack(a, bb), p1 = ptx::Mma<T>::pack(cc, d);
            const uint32_t d0 = ptx::Mma<T>::pack(ea, eb), d1 = ptx::Mma<T>::pack(ec, ed);
            df[c / 2][(c % 2) * 2] = d0;
            df[c / 2][(c % 2) * 2 + 1] = d1;
            dl[c / 2][(c % 2) * 2] = ptx::Mma<T>::pack(ea - ptx::Mma<T>::lo(d0), eb - ptx::Mma<T>::hi(d0));
            dl[c / 2][(c % 2) * 2 + 1] = ptx::Mma<T>::pack(ec - ptx::Mma<T>::lo(d1), ed - ptx::Mma<T>::hi(d1));
            const int row = warp * 16 + lane / 4;
            *reinterpret_cast<uint32_t *>(ps + row * WP + col) = p0;
            *reinterpret_cast<uint32_t *>(ps + (row + 8) * WP + col) = p1;
            *reinterpret_cast<uint32_t *>(ds + row * WP + col) = d0;
            *reinterpret_cast<uint32_t *>(ds + (row + 8) * WP + col) = d1;
            *reinterpret_cast<uint32_t *>(dr + row * WP + col) = dl[c / 2][(c % 2) * 2];
            *reinterpret_cast<uint32_t *>(dr + (row + 8) * WP + col) = dl[c / 2][(c % 2) * 2 + 1];
        }
        bool odd_tile = false;
        if (ragged) odd_tile = __syncthreads_or(zero != 0.f);
        else __syncthreads();
        if (odd_tile) {
            if (!odd_rows) odd.clear(128);
            odd_rows = true;
            __syncthreads();
            T *rows = qs + cur * 128 * PITCH;          // 64 queries, then their output gradients
            for (int x = threadIdx.x; x < (128 + held) * (DP / 8); x += 128) {
                const int r = x / (DP / 8), c = x % (DP / 8) * 8, i = r < 128 ? row_q[first - item.y + r % 64] : 0;
                T *at = (r < 128 ? rows + r * PITCH : ks + (r - 128) * PITCH) + c;
                if (i < 0) continue;
                const int vis = max(0, (int)min((int64_t)held, i + 1 - j0));
                for (int y = 0; y < 8; ++y) {
                    const float f = Elem<T>::to_f(at[y]);
                    if (f - f == 0.f) continue;
                    at[y] = Elem<T>::from_f(0.f);
                    if (r >= 128) odd.see_key(r - 128, c + y);
                    else if (r < 64) odd.see_query(vis, c + y);
                    else odd.see_grad(f, vis, c + y);
                }
            }
            __syncthreads();
        }
        // dq share of this warp's rows, 16 columns at a time
        const int64_t at0 = (part0 + row_at[x0]) * t.nsub + sub, at1 = (part0 + row_at[x1]) * t.nsub + sub;
#pragma unroll
        for (int c = 0; c < DP / 16; ++c)
            if (c < d16) {
                float q0[4] = {0.f, 0.f, 0.f, 0.f}, q1[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int kk = 0; kk < NF / 2; ++kk)
                    if (kk < n16) {
                        uint32_t x[4];
                        ptx::ldmatrix_x4_trans(x, ptx::smem_u32(ks + (kk * 16 + lane % 16) * PITCH + c * 16 + (lane / 16) * 8));
                        ptx::Mma<T>::run(q0, df[kk], x[0], x[1]);
                        ptx::Mma<T>::run(q1, df[kk], x[2], x[3]);
                        ptx::Mma<T>::run(q0, dl[kk], x[0], x[1]);
                        ptx::Mma<T>::run(q1, dl[kk], x[2], x[3]);
                    }
                const int col = c * 16 + (lane % 4) * 2;
                if (i0 >= 0) {
                    *reinterpret_cast<float2 *>(t.part + at0 * D + col) = make_float2(q0[0], q0[1]);
                    if (c * 16 + 8 < D) *reinterpret_cast<float2 *>(t.part + at0 * D + col + 8) = make_float2(q1[0], q1[1]);
                }
                if (i1 >= 0) {
                    *reinterpret_cast<float2 *>(t.part + at1 * D + col) = make_float2(q0[2], q0[3]);
                    if (c * 16 + 8 < D) *reinterpret_cast<float2 *>(t.part + at1 * D + col + 8) = make_float2(q1[2], q1[3]);
                }
            }
        // dv += P^T dO, dk += dS^T Q for this warp's keys and columns
        if (kg < n16)
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) {
                uint32_t pa[4], da[4], ra[4];
                const int row = kk * 16 + (lane / 16) * 8 + lane % 8, col = kg * 16 + (lane / 8 % 2) * 8;
                ptx::ldmatrix_x4_trans(pa, ptx::smem_u32(ps + row * WP + col));
                ptx::ldmatrix_x4_trans(da, ptx::smem_u32(ds + row * WP + col));
                ptx::ldmatrix_x4_trans(ra, ptx::smem_u32(dr + row * WP + col));
#pragma unroll
                for (int c = 0; c < CF; ++c)
                    if (cg * CF + c < d16) {
                        uint32_t x[4];
                        const int dc = (cg * CF + c) * 16 + (lane / 16) * 8;
                        ptx::ldmatrix_x4_trans(x, ptx::smem_u32(ot + (kk * 16 + lane % 16) * PITCH + dc));
                        ptx::Mma<T>::run(dv[c][0], pa, x[0], x[1]);
                        ptx::Mma<T>::run(dv[c][1], pa, x[2], x[3]);
                        ptx::ldmatrix_x4_trans(x, ptx::smem_u32(qt + (kk * 16 + lane % 16) * PITCH + dc));
                        ptx::Mma<T>::run(dk[c][0], da, x[0], x[1]);
                        ptx::Mma<T>::run(dk[c][1], da, x[2], x[3]);
                        ptx::Mma<T>::run(dk[c][0], ra, x[0], x[1]);
                        ptx::Mma<T>::run(dk[c][1], ra, x[2], x[3]);
                    }
            }
        if (odd_tile) {
            __syncthreads();                 // also puts the shares above before what follows
            for (int x = threadIdx.x; x < 64 * D; x += 128) {
                const int r = first - item.y + x / D, col = x % D, i = row_q[r];
                if (i < 0 || min((int64_t)held, i + 1 - j0) <= odd.key[col]) continue;
                t.part[((part0 + row_at[r]) * t.nsub + sub) * D + col] = NAN;       // zero times such a key
            }
            // the keys as they are
            stage_keys<T, DP>(ks, (const T *)p.k + ((b * p.S + j0) * p.Hkv + h) * D, krow, held, NKP, D);
            cp_async_commit();
        }
        if (NBUF == 1) {
            __syncthreads();             // every warp is done with the tile
            if (first + 64 < r_end) stage_rows(qs, first + 64 - item.y);
        }
    }
    if (DELTA) return;
    cp_async_wait<0>();
    float *out = t.kv_part + (((bhl * t.max_items + blockIdx.x) * t.nsub + sub) * 2) * t.kv_rows * D, *out_v = out + t.kv_rows * D;
    if (kg < n16)
#pragma unroll
        for (int c = 0; c < CF; ++c)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int col = (cg * CF + c) * 16 + x * 8 + (lane % 4) * 2, row = kg * 16 + lane / 4;
                if ((cg * CF + c) * 16 + x * 8 < D) {
                    *reinterpret_cast<float2 *>(out + row * D + col) = make_float2(dk[c][x][0], dk[c][x][1]);
                    *reinterpret_cast<float2 *>(out + (row + 8) * D + col) = make_float2(dk[c][x][2], dk[c][x][3]);
                    *reinterpret_cast<float2 *>(out_v + row * D + col) = make_float2(dv[c][x][0], dv[c][x][1]);
                    *reinterpret_cast<float2 *>(out_v + (row + 8) * D + col) = make_float2(dv[c][x][2], dv[c][x][3]);
                }
            }
    if (odd_rows) {
        __syncthreads();
        for (int x = threadIdx.x; x < keys * D; x += 128) {
            const int row = x / D, col = x - row * D;
            out[x] = odd.dk(out[x], row, col);
            out_v[x] = odd.dv(out_v[x], row, col);
        }
    }
}

// dk and dv of a (sub-)block: the sum of its items' shares in order; zeros for a block that nobody chose
template <typename T> __global__ void __launch_bounds__(128) sel_kv_join_kernel(const SelProblem p, const SelTile t) {
    const int64_t bhl = blockIdx.y;
    const int bh = (int)t.bh0 + blockIdx.y;
    const int64_t b = bh / (int)p.Hkv, h = bh - b * p.Hkv;
    pdl_trigger();
    pdl_wait();
    const int n = blockIdx.x / t.nsub, sub = blockIdx.x % t.nsub, D = (int)p.D;
    const int64_t j0 = (int64_t)n * p.block + sub * 64;
    const int held = (int)min((int64_t)min((int)p.block - sub * 64, 64), p.S - j0);
    const int i0 = t.item_base[bhl * (p.nb + 1) + n], i1 = t.item_base[bhl * (p.nb + 1) + n + 1];
    const int x = blockIdx.z * 128 + threadIdx.x;
    if (x < held * D / 4) {
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f), c = a;
#pragma unroll 4
        for (int i = i0; i < i1; ++i) {
            const float *src = t.kv_part + (((bhl * t.max_items + i) * t.nsub + sub) * 2) * t.kv_rows * D;
            const float4 u = *reinterpret_cast<const float4 *>(src + x * 4), w = *reinterpret_cast<const float4 *>(src + t.kv_rows * D + x * 4);
            a.x += u.x; a.y += u.y; a.z += u.z; a.w += u.w;
            c.x += w.x; c.y += w.y; c.z += w.z; c.w += w.w;
        }
        const int64_t at = ((b * p.S + j0 + x * 4 / D) * p.Hkv + h) * D + x * 4 % D;
        store4((T *)p.dk + at, make_float4(a.x * p.scale, a.y * p.scale, a.z * p.scale, a.w * p.scale));
        store4((T *)p.dv + at, c);
    }
}

// delta of every row as the sum of its shares, in the order of its list
__global__ void __launch_bounds__(128) sel_delta_join_kernel(const SelProblem p, const SelTile t, float *delta) {
    const uint32_t x = blockIdx.x * 128u + threadIdx.x, G = t.G;
    pdl_trigger();
    pdl_wait();
    if (x >= (uint32_t)p.S * G) return;
    const int i = (int)(x / G), g = (int)(x - i * G), bh = (int)t.bh0 + blockIdx.y, T_ = (int)p.topk;
    const int64_t b = bh / (int)p.Hkv, h = bh - b * p.Hkv;
    const int32_t *list = p.blocks + ((b * p.S + i) * p.Hkv + h) * T_;
    const int limit = p.causal ? i / (int)p.block + 1 : (int)p.nb;
    const float *part = t.delta_part + ((int64_t)blockIdx.y * p.S * G + x) * T_ * t.nsub;
    float sum = 0.f;
    int prev = -1;
    for (int s = 0; s < T_; ++s) {
        if (!sel_entry_counts(list[s], prev, limit)) continue;
        const int uses = min(t.nsub, (int)((p.S - (int64_t)prev * p.block + 63) / 64));
        for (int u = 0; u < uses; ++u) sum += part[s * t.nsub + u];
    }
    delta[(b * p.S + i) * p.H + h * G + g] = sum;
}

// delta = dO . O of every row: LPR lanes of 16 bytes
template <typename T, int LPR> __global__ void __launch_bounds__(128) sel_delta_kernel(const T *o, const T *dout, float *delta, int64_t rows, int D) {
    constexpr int W = Vec16<T>::N;
    const int64_t r = (int64_t)blockIdx.x * (128 / LPR) + threadIdx.x / LPR;
    const int col = (threadIdx.x % LPR) * W;
    pdl_trigger();
    pdl_wait();
    float s = 0.f;
    if (r < rows && col < D) {
        float x[W], y[W];
        Vec16<T>::unpack(__ldg(reinterpret_cast<const uint4 *>(o + r * D + col)), x);
        Vec16<T>::unpack(__ldg(reinterpret_cast<const uint4 *>(dout + r * D + col)), y);
#pragma unroll
        for (int j = 0; j < W; ++j) s = fmaf(x[j], y[j], s);
    }
#pragma unroll
    for (int x = 1; x < LPR; x <<= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    if (r < rows && col == 0) delta[r] = s;
}

template <typename T> void launch_delta(const SelProblem &p, float *delta) {
    const int64_t all = p.B * p.S * p.H;
    const int lanes = (int)p.D * (int)sizeof(T) / 16 <= 8 ? 8 : (int)p.D * (int)sizeof(T) / 16 <= 16 ? 16 : 32;
    const dim3 grid((unsigned)((all + 128 / lanes - 1) / (128 / lanes)));
    const T *o = (const T *)p.o, *g = (const T *)p.dout;
    if (lanes == 8) launch_after(sel_delta_kernel<T, 8>, grid, dim3(128), 0, p.stream, o, g, delta, all, (int)p.D);
    else if (lanes == 16) launch_after(sel_delta_kernel<T, 16>, grid, dim3(128), 0, p.stream, o, g, delta, all, (int)p.D);
    else launch_after(sel_delta_kernel<T, 32>, grid, dim3(128), 0, p.stream, o, g, delta, all, (int)p.D);
}

// AHEAD covers the whole list where that has up to 16 entries: with 8 for 16 the backward of 8192 x 8 heads of 64 took 374 us
// instead of 346, with 16 for 8 that of 4096 x 16 heads of 128 took 664 instead of 595.
template <typename T, bool BWD> void launch_join(const SelProblem &p, const SelTile &t, int64_t pairs) {
    const int64_t rows = p.S * t.G;
    const dim3 narrow((unsigned)((rows + 7) / 8), (unsigned)pairs), wide((unsigned)((rows + 3) / 4), (unsigned)pairs);
    if (p.D <= 64) {
        if (p.topk <= 8) launch_after(sel_join_kernel<T, 16, 8, BWD>, narrow, dim3(128), 0, p.stream, p, t);
        else launch_after(sel_join_kernel<T, 16, 16, BWD>, narrow, dim3(128), 0, p.stream, p, t);
    } else {
        if (p.topk <= 8) launch_after(sel_join_kernel<T, 32, 8, BWD>, wide, dim3(128), 0, p.stream, p, t);
        else launch_after(sel_join_kernel<T, 32, 16, BWD>, wide, dim3(128), 0, p.stream, p, t);
    }
}

template <typename T> void launch_kv_join(const SelProblem &p, const SelTile &t, int64_t pairs) {
    launch_after(sel_kv_join_kernel<T>, dim3((unsigned)(p.nb * t.nsub), (unsigned)pairs, (unsigned)((64 * p.D / 4 + 127) / 128)), dim3(128), 0, p.stream, p, t);
}

int launched(const char *what) {
    cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? MAT_OK : cuda_fail(e, what);
}

// What lies where in the workspace.
struct Plan {
    int64_t max_items, group;       // items per (batch, key head); pairs worked off together
    int nsub, kv_rows;
    size_t lists, items, base, stats, part, kv, delta, delta_part, total;
};

// Rows of so few keys that delta is summed from the tiles (16-bit types); with one block a causal row may see a key or two.
bool few_keys(int64_t block, int64_t topk) { return topk == 1 || block * topk <= 64; }

int rows_per_item(int dtype, bool bwd) { return dtype == MAT_F32 ? (bwd ? kF32BwdRows : kF32Rows) : bwd ? kBwdRows : kFwdRows; }

Plan plan(int64_t B, int64_t S, int64_t H, int64_t Hkv, int64_t D, int dtype, int64_t block, int64_t topk, bool bwd) {
    Plan w;
    const int64_t nb = (S + block - 1) / block, G = H / Hkv, bh = B * Hkv;
    w.nsub = bwd ? (int)((block + 63) / 64) : 1;
    const int64_t rows = rows_per_item(dtype, bwd);
    w.max_items = S * topk * G / rows + nb;
    w.kv_rows = (int)(block < 64 ? block : 64);
    const size_t part = (size_t)S * G * topk * w.nsub * D * 4, kv = bwd ? (size_t)w.max_items * w.nsub * 2 * w.kv_rows * D * 4 : 0;
    const size_t stats = bwd ? 0 : (size_t)S * G * topk * sizeof(float2);
    const size_t shares = bwd && dtype != MAT_F32 && few_keys(block, topk) ? (size_t)S * G * topk * w.nsub * 4 : 0;
    const size_t pair = part + kv + stats + shares + (size_t)w.max_items * sizeof(int2) + (size_t)(nb + 1) * 4 + sel_lists_bytes(1, S, nb, topk);
    w.group = pair >= kPairBudget ? 1 : (int64_t)(kPairBudget / pair);
    if (w.group > bh) w.group = bh;
    size_t at = 0;
    auto take = [&](size_t n) { const size_t x = at; at += sel_align(n); return x; };
    w.lists = take(sel_lists_bytes(w.group, S, nb, topk));
    w.items = take((size_t)w.group * w.max_items * sizeof(int2));
    w.base = take((size_t)w.group * (nb + 1) * 4);
    w.stats = take(w.group * stats);
    w.part = take(w.group * part);
    w.kv = take(w.group * kv);
    w.delta = take(bwd ? (size_t)B * S * H * 4 : 0);
    w.delta_part = take(w.group * shares);
    w.total = at;
    return w;
}

SelTile tile_args(const SelProblem &p, const Plan &w, void *ws) {
    SelTile t{};
    char *at = (char *)ws;
    t.l = sel_lists_at(at + w.lists, w.group, p.S, p.nb, p.topk);
    t.items = (int2 *)(at + w.items);
    t.item_base = (int32_t *)(at + w.base);
    t.max_items = w.max_items;
    t.stats = (float2 *)(at + w.stats);
    t.part = (float *)(at + w.part);
    t.kv_part = (float *)(at + w.kv);
    t.delta = (const float *)(at + w.delta);
    t.delta_part = (float *)(at + w.delta_part);
    t.G = (int)(p.H / p.Hkv);
    t.nsub = w.nsub;
    t.kv_rows = w.kv_rows;
    t.scale_log2 = p.scale * 1.4426950408889634f;
    return t;
}

// The groups of pairs in turn: their lists, their tiles, then their joins.
template <bool BWD, typename T, typename Launch> int over_groups(const SelProblem &p, const Plan &w, SelTile &t, Launch &&tiles) {
    const int64_t bh = p.B * p.Hkv;
    for (t.bh0 = 0; t.bh0 < bh; t.bh0 += w.group) {
        const int64_t n = bh - t.bh0 < w.group ? bh - t.bh0 : w.group;
        if (int rc = launch_sel_lists(p, t.l, t.bh0, n, t.items, t.item_base, t.max_items, rows_per_item(p.dtype, BWD))) return rc;
        tiles((unsigned)n);
        launch_join<T, BWD>(p, t, n);
        if (BWD) launch_kv_join<T>(p, t, n);
    }
    return launched(BWD ? "launching the selected attention's backward" : "launching the selected attention");
}

template <typename T, int DP, int NKP, bool EXACT> int fwd(const SelProblem &p, const Plan &w, SelTile &t) {
    const size_t smem = ((p.block + NKP - 1) / NKP * NKP * 2 + 4 * 2 * 16) * (DP + 8) * sizeof(T);
    if (int rc = ensure_dynamic_smem((const void *)sel_fwd_mma_kernel<T, DP, NKP, EXACT>, smem, "shared memory of the selected attention")) return rc;
    return over_groups<false, T>(p, w, t, [&](unsigned n) {
        launch_after(sel_fwd_mma_kernel<T, DP, NKP, EXACT>, dim3((unsigned)w.max_items, n), dim3(128), smem, p.stream, p, t);
    });
}

template <typename T, int DP, int NKP, bool EXACT> int bwd(const SelProblem &p, const Plan &w, SelTile &t) {
    const size_t smem = ((2 * NKP + (DP == 64 ? 4 : 2) * 64) * (DP + 8) + 3 * 64 * (NKP + 8)) * sizeof(T) + kBwdRows * 20 + sizeof(OddColumns<DP>);
    const auto grads = sel_bwd_mma_kernel<T, DP, NKP, EXACT, false>, shares = sel_bwd_mma_kernel<T, DP, NKP, EXACT, true>;
    const bool few = few_keys(p.block, p.topk);
    if (int rc = ensure_dynamic_smem((const void *)grads, smem, "shared memory of the selected attention's backward")) return rc;
    if (int rc = few ? ensure_dynamic_smem((const void *)shares, smem, "shared memory of the selected attention's backward") : MAT_OK) return rc;
    float *delta = const_cast<float *>(t.delta);
    return over_groups<true, T>(p, w, t, [&](unsigned n) {
        const dim3 grid((unsigned)w.max_items, (unsigned)w.nsub, n);
        if (!few && t.bh0 == 0) launch_delta<T>(p, delta);             // of all pairs
        if (few) {
            launch_after(shares, grid, dim3(128), smem, p.stream, p, t);
            launch_after(sel_delta_join_kernel, dim3((unsigned)((p.S * t.G + 127) / 128), n), dim3(128), 0, p.stream, p, t, delta);
        }
        launch_after(grads, grid, dim3(128), smem, p.stream, p, t);
    });
}

int run_f32(const SelProblem &p, void *ws, bool back) {
    const Plan w = plan(p.B, p.S, p.H, p.Hkv, p.D, p.dtype, p.block, p.topk, back);
    SelTile t = tile_args(p, w, ws);
    const size_t pitch = p.D + 4, key_rows = (p.block + 63) / 64 * 64;
    const size_t smem = ((back ? 4 * 64 : 2 * key_rows + 64) * pitch + (back ? 2 : 1) * 64 * kWPitch) * sizeof(float);
    if (int rc = ensure_dynamic_smem(back ? (const void *)sel_bwd_f32_kernel : (const void *)sel_fwd_f32_kernel, smem, "shared memory of the selected attention in fp32")) return rc;
    if (!back)
        return over_groups<false, float>(p, w, t, [&](unsigned n) {
            launch_after(sel_fwd_f32_kernel, dim3((unsigned)w.max_items, n), dim3(kF32Threads), smem, p.stream, p, t);
        });
    return over_groups<true, float>(p, w, t, [&](unsigned n) {
        if (t.bh0 == 0) launch_delta<float>(p, const_cast<float *>(t.delta));       // of all pairs
        launch_after(sel_bwd_f32_kernel, dim3((unsigned)w.max_items, (unsigned)w.nsub, n), dim3(kF32Threads), smem, p.stream, p, t);
    });
}

template <typename T> int run(const SelProblem &p, void *ws, bool back) {
    const Plan w = plan(p.B, p.S, p.H, p.Hkv, p.D, p.dtype, p.block, p.topk, back);
    SelTile t = tile_args(p, w, ws);
    const int dp = p.D <= 64 ? 64 : 128, nkp = p.block <= 32 ? 32 : 64;
    const bool exact = p.D == dp && p.block % nkp == 0;
#define SEL_CASE(DP, NKP)                                                                        \
    if (dp == DP && nkp == NKP)                                                                  \
        return back ? (exact ? bwd<T, DP, NKP, true>(p, w, t) : bwd<T, DP, NKP, false>(p, w, t)) \
                    : (exact ? fwd<T, DP, 32, true>(p, w, t) : fwd<T, DP, NKP, false>(p, w, t))
    SEL_CASE(64, 32);
    SEL_CASE(64, 64);
    SEL_CASE(128, 32);
    SEL_CASE(128, 64);
#undef SEL_CASE
    return fail(MAT_ERR_UNSUPPORTED, "no kernel for this width");
}

}  // namespace

size_t sel_workspace_bytes(int64_t B, int64_t S, int64_t H, int64_t Hkv, int64_t D, int dtype, int64_t block, int64_t topk, bool bwd) {
    return plan(B, S, H, Hkv, D, dtype, block, topk, bwd).total;
}

int launch_sel(const SelProblem &p, void *workspace, bool bwd) {
    if (p.dtype == MAT_F32) return run_f32(p, workspace, bwd);
    return p.dtype == MAT_BF16 ? run<__nv_bfloat16>(p, workspace, bwd) : run<__half>(p, workspace, bwd);
}

}  // namespace mat
