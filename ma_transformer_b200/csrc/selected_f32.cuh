// fp32 tiles of block-selected attention: the plan of the 16-bit kernels (rows gathered by the block they chose, partials
// joined in list order) with fp32 products on the FMA pipe.  The tensor cores' TF32 products, three to one fp32 product,
// are 1.2e-6 to 2.4e-6 off on this kind of sum; these stay at fp32's own 4e-7.
//
// A tile is 64 rows x 64 keys, 256 threads of 4 rows x 4 keys (rows ty + 16 i, keys tx + 16 j).  Rows of shared memory
// are D + 4 floats: an odd number of 16-byte units for every D that is a multiple of 8, so 16-byte reads down a column
// meet no bank twice.
#pragma once

namespace mat {
namespace {

constexpr int kF32Threads = 256, kWPitch = 68;

// acc[i][j] += a[row ty + 16 i] . x[key tx + 16 j] over D columns
__device__ __forceinline__ void tile_dot(float (&acc)[4][4], const float *a, const float *x, int D, int pitch) {
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    for (int d = 0; d < D; d += 4) {
        float4 u[4], w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            u[i] = *reinterpret_cast<const float4 *>(a + (ty + 16 * i) * pitch + d);
            w[i] = *reinterpret_cast<const float4 *>(x + (tx + 16 * i) * pitch + d);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                acc[i][j] = fmaf(u[i].x, w[j].x, acc[i][j]);
                acc[i][j] = fmaf(u[i].y, w[j].y, acc[i][j]);
                acc[i][j] = fmaf(u[i].z, w[j].z, acc[i][j]);
                acc[i][j] = fmaf(u[i].w, w[j].w, acc[i][j]);
            }
    }
}

__device__ __forceinline__ void fma4(float4 &y, float a, const float4 &x) {
    y.x = fmaf(a, x.x, y.x); y.y = fmaf(a, x.y, y.y); y.z = fmaf(a, x.z, y.z); y.w = fmaf(a, x.w, y.w);
}

// y[r] = sum over keys of w[4 rg + r][key] * x[key][col .. col + 3]
__device__ __forceinline__ void tile_times(float4 (&y)[4], const float *w, const float *x, int keys, int rg, int col, int pitch) {
    for (int k = 0; k < keys; k += 4) {
        float4 u[4], z[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            u[i] = *reinterpret_cast<const float4 *>(w + (4 * rg + i) * kWPitch + k);
            z[i] = *reinterpret_cast<const float4 *>(x + (k + i) * pitch + col);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            fma4(y[i], u[i].x, z[0]);
            fma4(y[i], u[i].y, z[1]);
            fma4(y[i], u[i].z, z[2]);
            fma4(y[i], u[i].w, z[3]);
        }
    }
}

__device__ __forceinline__ void stage_f32(float *dst, const float *src, int64_t row_stride, int n, int rows, int D) {
    const int vecs = D / 4, pitch = D + 4;
    for (int i = threadIdx.x; i < rows * vecs; i += kF32Threads) {
        const int r = i / vecs, c = (i - r * vecs) * 4;
        cp_async16(dst + r * pitch + c, r < n ? src + r * row_stride + c : src, r < n);
    }
}

__global__ void __launch_bounds__(kF32Threads) sel_fwd_f32_kernel(const SelProblem p, const SelTile t) {
    const int64_t bhl = blockIdx.y;
    const int bh = (int)t.bh0 + blockIdx.y;
    const int64_t b = bh / (int)p.Hkv, h = bh - b * p.Hkv;
    pdl_trigger();
    pdl_wait();
    if ((int)blockIdx.x >= t.item_base[bhl * (p.nb + 1) + p.nb]) return;
    const int2 item = t.items[bhl * t.max_items + blockIdx.x];
    const int n = item.x, e0 = t.l.base[bhl * (p.nb + 1) + n], D = (int)p.D, pitch = D + 4, T_ = (int)p.topk, block = (int)p.block;
    const int rows_all = (t.l.base[bhl * (p.nb + 1) + n + 1] - e0) * t.G, r_end = min(item.y + kF32Rows, rows_all);
    const int64_t j0 = (int64_t)n * block;
    const int held = (int)min((int64_t)block, p.S - j0), key_rows = (block + 63) / 64 * 64;
    extern __shared__ __align__(16) char smem[];
    float *ks = (float *)smem, *vs = ks + key_rows * pitch, *qs = vs + key_rows * pitch, *ws = qs + 64 * pitch;   // ws: [64][kWPitch]
    __shared__ int row_q[64], row_at[64];
    __shared__ uint32_t odd_keys[4];
    const float *kg = (const float *)p.k + ((b * p.S + j0) * p.Hkv + h) * D, *vg = (const float *)p.v + ((b * p.S + j0) * p.Hkv + h) * D;
    stage_f32(ks, kg, p.Hkv * D, held, key_rows, D);
    stage_f32(vs, vg, p.Hkv * D, held, key_rows, D);
    cp_async_commit();
    const int tid = threadIdx.x, tx = tid % 16, ty = tid / 16;
    if (tid < 4) odd_keys[tid] = 0;
    cp_async_wait<0>();
    __syncthreads();
    // infinite and NaN values go into the product as zeros and are added to the rows that see them
    for (int x = tid; x < held * D; x += kF32Threads) {
        const int r = x / D;
        float *at = vs + r * pitch + x - r * D;
        if (!(fabsf(*at) < INFINITY)) {
            *at = 0.f;
            atomicOr(&odd_keys[r / 32], 1u << (r % 32));
        }
    }
    const int64_t part0 = (int64_t)blockIdx.y * p.S * t.G * T_;
    const float *q0 = (const float *)p.q + (b * p.S * p.H + h * t.G) * D;
    for (int first = item.y; first < r_end; first += 64) {
        __syncthreads();
        if (tid < 64) {
            const int r = first + tid;
            int i = -1, at = 0;
            if (r < r_end) {
                const int e = r / t.G, entry = t.l.entry[bhl * p.S * T_ + e0 + e];
                i = entry / T_;
                at = (i * t.G + r - e * t.G) * T_ + entry - i * T_;
            }
            row_q[tid] = i; row_at[tid] = at;
        }
        __syncthreads();
        const int vecs = D / 4;
        for (int x = tid; x < 64 * vecs; x += kF32Threads) {
            const int r = x / vecs, c = (x - r * vecs) * 4, i = row_q[r];
            cp_async16(qs + r * pitch + c, i < 0 ? q0 : q0 + ((int64_t)i * p.H + (first + r) % t.G) * D + c, i >= 0);
        }
        cp_async_commit();
        cp_async_wait<0>();
        __syncthreads();
        float m[4], l[4];
        int vis[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int q = row_q[ty + 16 * i];
            vis[i] = q < 0 ? 0 : p.causal ? min(held, (int)(q + 1 - j0)) : held;
            m[i] = -INFINITY; l[i] = 0.f;
        }
        float4 y[2][4];       // output of up to two (4 rows x 4 columns) items
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) y[u][i] = make_float4(0.f, 0.f, 0.f, 0.f);
        __shared__ float keep_of[64];
        for (int base = 0; base < held; base += 64) {
            float s[4][4] = {};
            tile_dot(s, qs, ks + base * pitch, D, pitch);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float top = -INFINITY;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    s[i][j] = base + tx + 16 * j < vis[i] ? s[i][j] * t.scale_log2 : -INFINITY;
                    top = fmaxf(top, s[i][j]);
                }
#pragma unroll
                for (int x = 1; x < 16; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
                top = fmaxf(top, m[i]);
                const float ref = top == -INFINITY ? 0.f : top, keep = exp2f(m[i] - ref);
                m[i] = top;
                l[i] *= keep;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float w = exp2f(s[i][j] - ref);
                    l[i] += w;
                    ws[(ty + 16 * i) * kWPitch + tx + 16 * j] = w;
                }
                if (tx == 0) keep_of[ty + 16 * i] = keep;
            }
            __syncthreads();
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int x = tid + u * kF32Threads, rg = x / vecs, col = (x - rg * vecs) * 4;
                if (rg >= 16) continue;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float keep = keep_of[4 * rg + i];
                    y[u][i].x *= keep; y[u][i].y *= keep; y[u][i].z *= keep; y[u][i].w *= keep;
                }
                tile_times(y[u], ws, vs + base * pitch, min(64, block - base), rg, col, pitch);
            }
            __syncthreads();
        }
        const bool odd = (odd_keys[0] | odd_keys[1] | odd_keys[2] | odd_keys[3]) != 0;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int x = tid + u * kF32Threads, rg = x / vecs, col = (x - rg * vecs) * 4;
            if (rg >= 16) continue;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int q = row_q[4 * rg + i];
                if (q < 0) continue;
                if (odd) {
                    const int see = p.causal ? min(held, (int)(q + 1 - j0)) : held;
                    for (int j = 0; j < see; ++j) {
                        if (!(odd_keys[j / 32] >> (j % 32) & 1)) continue;
                        const float4 z = *reinterpret_cast<const float4 *>(vg + j * p.Hkv * D + col);
                        if (!(fabsf(z.x) < INFINITY)) y[u][i].x += z.x;
                        if (!(fabsf(z.y) < INFINITY)) y[u][i].y += z.y;
                        if (!(fabsf(z.z) < INFINITY)) y[u][i].z += z.z;
                        if (!(fabsf(z.w) < INFINITY)) y[u][i].w += z.w;
                    }
                }
                *reinterpret_cast<float4 *>(t.part + (part0 + row_at[4 * rg + i]) * D + col) = y[u][i];
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int x = 1; x < 16; x <<= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], x);
            if (tx == 0 && vis[i] > 0) t.stats[part0 + row_at[ty + 16 * i]] = make_float2(m[i], l[i]);
        }
    }
}

__global__ void __launch_bounds__(kF32Threads) sel_bwd_f32_kernel(const SelProblem p, const SelTile t) {
    const int64_t bhl = blockIdx.z;
    const int bh = (int)t.bh0 + blockIdx.z, sub = blockIdx.y;
    const int64_t b = bh / (int)p.Hkv, h = bh - b * p.Hkv;
    pdl_trigger();
    pdl_wait();
    if ((int)blockIdx.x >= t.item_base[bhl * (p.nb + 1) + p.nb]) return;
    const int2 item = t.items[bhl * t.max_items + blockIdx.x];
    const int n = item.x, e0 = t.l.base[bhl * (p.nb + 1) + n], D = (int)p.D, pitch = D + 4, T_ = (int)p.topk, vecs = D / 4;
    const int rows_all = (t.l.base[bhl * (p.nb + 1) + n + 1] - e0) * t.G, r_end = min(item.y + kF32BwdRows, rows_all);
    const int64_t j0 = (int64_t)n * p.block + sub * 64;
    const int keys = min((int)p.block - sub * 64, 64), held = (int)max((int64_t)0, min((int64_t)keys, p.S - j0));
    if (held == 0) return;                                   // the sequence ends before this half
    extern __shared__ __align__(16) char smem[];
    float *ks = (float *)smem, *vs = ks + 64 * pitch, *qs = vs + 64 * pitch, *os = qs + 64 * pitch, *ps = os + 64 * pitch, *ds = ps + 64 * kWPitch;
    __shared__ int row_q[64], row_at[64];
    __shared__ float row_lse[64], row_delta[64];
    __shared__ OddColumns<128> odd;
    stage_f32(ks, (const float *)p.k + ((b * p.S + j0) * p.Hkv + h) * D, p.Hkv * D, held, 64, D);
    stage_f32(vs, (const float *)p.v + ((b * p.S + j0) * p.Hkv + h) * D, p.Hkv * D, held, 64, D);
    cp_async_commit();
    const int tid = threadIdx.x, tx = tid % 16, ty = tid / 16;
    const int64_t part0 = (int64_t)bhl * p.S * t.G * T_, src0 = (b * p.S * p.H + h * t.G) * D;
    float4 dk[2][4], dv[2][4];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) dk[u][i] = dv[u][i] = make_float4(0.f, 0.f, 0.f, 0.f);
    const int ragged_end = p.causal ? (int)(j0 + held) - 1 : 0;        // queries below it see part of the keys
    bool odd_rows = false;                               // `odd` is in use
    for (int first = item.y; first < r_end; first += 64) {
        __syncthreads();
        if (tid < 64) {
            const int r = first + tid;
            int i = -1, at = 0;
            float lse = 0.f, delta = 0.f;
            if (r < r_end) {
                const int e = r / t.G, g = r - e * t.G, entry = t.l.entry[bhl * p.S * T_ + e0 + e];
                i = entry / T_;
                at = (i * t.G + g) * T_ + entry - i * T_;
                const int64_t row = (b * p.S + i) * p.H + h * t.G + g;
                lse = p.lse_in[row];
                delta = t.delta[row];
            }
            row_q[tid] = i; row_at[tid] = at; row_lse[tid] = lse; row_delta[tid] = delta;
        }
        __syncthreads();
        for (int x = tid; x < 64 * vecs; x += kF32Threads) {
            const int r = x / vecs, c = (x - r * vecs) * 4, i = row_q[r];
            const int64_t off = i < 0 ? 0 : src0 + ((int64_t)i * p.H + (first + r) % t.G) * D + c;
            cp_async16(qs + r * pitch + c, (const float *)p.q + off, i >= 0);
            cp_async16(os + r * pitch + c, (const float *)p.dout + off, i >= 0);
        }
        cp_async_commit();
        cp_async_wait<0>();
        __syncthreads();
        float s[4][4] = {}, dp[4][4] = {};
        tile_dot(s, qs, ks, D, pitch);
        tile_dot(dp, os, vs, D, pitch);
        const bool ragged = row_q[0] < ragged_end;       // a tile's first row has its lowest query
        float zero = 0.f;                                // NaN: a score or dP of a ragged tile is not finite
        if (ragged)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
#pragma unroll
                for (int j = 0; j < 4; ++j) zero = fmaf(s[i][j], 0.f, zero);
                zero = fmaf(dp[i][0], 0.f, zero);        // an output gradient shows in every column
            }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = ty + 16 * i, q = row_q[r];
            const int vis = q < 0 ? 0 : p.causal ? max(0, (int)min((int64_t)held, q + 1 - j0)) : held;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const bool in = tx + 16 * j < vis;
                const float w = in ? expf(fmaf(s[i][j], p.scale, -row_lse[r])) : 0.f;
                ps[r * kWPitch + tx + 16 * j] = w;
                ds[r * kWPitch + tx + 16 * j] = in ? w * (dp[i][j] - row_delta[r]) : 0.f;
            }
        }
        bool odd_tile = false;
        if (ragged) odd_tile = __syncthreads_or(zero != 0.f);
        else __syncthreads();
        if (odd_tile) {
            if (!odd_rows) odd.clear(kF32Threads);
            odd_rows = true;
            __syncthreads();
            for (int x = tid; x < (128 + held) * D; x += kF32Threads) {
                const int r = x / D, c = x - r * D, i = r < 128 ? row_q[r % 64] : 0;
                float *at = (r < 64 ? qs + r * pitch : r < 128 ? os + (r - 64) * pitch : ks + (r - 128) * pitch) + c;
                const float f = *at;
                if (i < 0 || fabsf(f) < INFINITY) continue;
                const int vis = max(0, (int)min((int64_t)held, i + 1 - j0));
                *at = 0.f;
                if (r >= 128) odd.see_key(r - 128, c);
                else if (r < 64) odd.see_query(vis, c);
                else odd.see_grad(f, vis, c);
            }
            __syncthreads();
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int x = tid + u * kF32Threads, rg = x / vecs, col = (x - rg * vecs) * 4;
            if (rg >= 16) continue;
            float4 y[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) y[i] = make_float4(0.f, 0.f, 0.f, 0.f);
            tile_times(y, ds, ks, keys, rg, col, pitch);
            if (odd_tile)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int vis = max(0, (int)min((int64_t)held, row_q[4 * rg + i] + 1 - j0));
                    y[i].x = odd.dq(y[i].x, vis, col); y[i].y = odd.dq(y[i].y, vis, col + 1);
                    y[i].z = odd.dq(y[i].z, vis, col + 2); y[i].w = odd.dq(y[i].w, vis, col + 3);
                }
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (row_q[4 * rg + i] >= 0) *reinterpret_cast<float4 *>(t.part + ((part0 + row_at[4 * rg + i]) * t.nsub + sub) * D + col) = y[i];
            // keys 4 rg .. 4 rg + 3
            for (int r = 0; r < 64; ++r) {
                const float4 w = *reinterpret_cast<const float4 *>(ps + r * kWPitch + 4 * rg), e = *reinterpret_cast<const float4 *>(ds + r * kWPitch + 4 * rg);
                const float4 o = *reinterpret_cast<const float4 *>(os + r * pitch + col), q = *reinterpret_cast<const float4 *>(qs + r * pitch + col);
                fma4(dv[u][0], w.x, o); fma4(dv[u][1], w.y, o); fma4(dv[u][2], w.z, o); fma4(dv[u][3], w.w, o);
                fma4(dk[u][0], e.x, q); fma4(dk[u][1], e.y, q); fma4(dk[u][2], e.z, q); fma4(dk[u][3], e.w, q);
            }
        }
        if (odd_tile) {                                  // the keys as they are
            __syncthreads();
            stage_f32(ks, (const float *)p.k + ((b * p.S + j0) * p.Hkv + h) * D, p.Hkv * D, held, 64, D);
            cp_async_commit();
        }
    }
    cp_async_wait<0>();
    float *out = t.kv_part + (((bhl * t.max_items + blockIdx.x) * t.nsub + sub) * 2) * t.kv_rows * D;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const int x = tid + u * kF32Threads, rg = x / vecs, col = (x - rg * vecs) * 4;
        if (rg >= 16) continue;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = 4 * rg + i;
            if (r >= t.kv_rows) break;
            if (odd_rows) {
                float4 &x = dk[u][i], &y = dv[u][i];
                x.x = odd.dk(x.x, r, col); x.y = odd.dk(x.y, r, col + 1); x.z = odd.dk(x.z, r, col + 2); x.w = odd.dk(x.w, r, col + 3);
                y.x = odd.dv(y.x, r, col); y.y = odd.dv(y.y, r, col + 1); y.z = odd.dv(y.z, r, col + 2); y.w = odd.dv(y.w, r, col + 3);
            }
            *reinterpret_cast<float4 *>(out + r * D + col) = dk[u][i];
            *reinterpret_cast<float4 *>(out + (t.kv_rows + r) * D + col) = dv[u][i];
        }
    }
}

}  // namespace
}  // namespace mat
