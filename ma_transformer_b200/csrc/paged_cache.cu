// Appends new tokens to a paged key-value cache: keys (and optionally the queries of the same tokens) turned by their
// positions, values copied, and the touched pages' key bounds set.
//
// Rotation: column pair (a, b) at position p with frequency f becomes (a cos t - b sin t, b cos t + a sin t), t = p f.
// The angle is formed in 64 bits as a number of half turns, p * (f / pi), and reduced by its nearest even integer
// before it is rounded to fp32 (an fp32 product would be off by p * f * 2^-24: 0.06 rad at position 10^6).
//
// append_rows_kernel streams: a CTA takes a tile of tokens with all their heads, finds each token's sequence, page and
// angles once (a chain of five dependent reads), and then moves 2 x 16 bytes per thread and step.  7 prompts, 32768
// tokens x (12 + 2 * 4) heads of 64 in fp16, 172 MB, 27 us at the copy rate: 33 us (46 us a call with the bounds).  One
// CTA per page and key head paid that chain per 10 KB: 177 us, 100 us with 8-byte vectors and more CTAs.
//
// page_bounds_kernel follows where the cache keeps bounds: one warp owns one page and head and takes its bounds from all
// filled slots (the new ones come from L2), so there are no atomics, and a cache that was rolled back and written again
// ends with the same bits as one that never was.
#include <limits.h>

#include <atomic>

#include "paged.cuh"
#include "pdl.cuh"

namespace mat {

__device__ int g_paged_status;

int *paged_status_word() {
    static std::atomic<int *> known[64];        // by device: looking the symbol up takes longer than the rest of a launch
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0) return nullptr;
    int *p = dev < 64 ? known[dev].load(std::memory_order_acquire) : nullptr;
    if (!p) {
        void *at = nullptr;
        if (cudaGetSymbolAddress(&at, g_paged_status) != cudaSuccess) return nullptr;
        p = (int *)at;
        if (dev < 64) known[dev].store(p, std::memory_order_release);
    }
    return p;
}

int paged_status_read_and_clear(int *out) {
    int zero = 0;
    cudaError_t e = cudaMemcpyFromSymbol(out, g_paged_status, sizeof(int));
    if (e == cudaSuccess) e = cudaMemcpyToSymbol(g_paged_status, &zero, sizeof(int));
    return e == cudaSuccess ? MAT_OK : cuda_fail(e, "reading the paged cache's status word");
}

int check_paged_cache(const mat_paged_cache *c) {
    if (!c) return fail(MAT_ERR_INVALID, "cache is NULL");
    if (c->dtype != MAT_F32 && c->dtype != MAT_BF16 && c->dtype != MAT_F16)
        return fail(MAT_ERR_INVALID, "unknown dtype %d", c->dtype);
    if (!c->k || !c->v) return fail(MAT_ERR_INVALID, "the cache's k and v must be non-NULL");
    if (c->n_pages < 1 || c->n_pages > INT_MAX) return fail(MAT_ERR_INVALID, "n_pages must be in [1, 2^31)");
    if (c->page_size < 8 || c->page_size > 1024 || (c->page_size & (c->page_size - 1)))
        return fail(MAT_ERR_UNSUPPORTED, "page_size must be a power of two from 8 to 1024, got %lld", (long long)c->page_size);
    if (c->H_kv < 1 || c->H_kv > 65535) return fail(MAT_ERR_INVALID, "H_kv must be in [1, 65535]");
    if (c->D < 8 || c->D > 256 || c->D % 8)
        return fail(MAT_ERR_UNSUPPORTED, "the paged cache takes head widths that are multiples of 8 up to 256, got %lld", (long long)c->D);
    const int64_t vec = 16 / (int64_t)dtype_size(c->dtype);
    const int64_t st[6] = {c->k_page_stride, c->k_token_stride, c->k_head_stride, c->v_page_stride, c->v_token_stride, c->v_head_stride};
    for (int64_t s : st)
        if (s < 0 || s % vec) return fail(MAT_ERR_INVALID, "cache strides must be non-negative multiples of 16 bytes");
    if (((uintptr_t)c->k | (uintptr_t)c->v | (uintptr_t)c->key_bounds) % 16)
        return fail(MAT_ERR_INVALID, "cache tensors must be 16-byte aligned");
    return MAT_OK;
}

int check_page_table(const int32_t *table, int64_t width, int64_t stride, int64_t B) {
    if (!table) return fail(MAT_ERR_INVALID, "page_table is NULL");
    if (B < 1 || B > 65535) return fail(MAT_ERR_INVALID, "the number of sequences must be in [1, 65535], got %lld", (long long)B);
    if (width < 1 || stride < width) return fail(MAT_ERR_INVALID, "page_table needs a width of at least 1 and rows at least as far apart");
    if (width > INT_MAX) return fail(MAT_ERR_UNSUPPORTED, "page_table is too wide");
    return MAT_OK;
}

PagedView paged_view(const mat_paged_cache *c, const int32_t *table, int64_t width, int64_t stride) {
    PagedView p;
    p.k = c->k; p.v = c->v;
    p.k_page = c->k_page_stride; p.k_tok = c->k_token_stride; p.k_head = c->k_head_stride;
    p.v_page = c->v_page_stride; p.v_tok = c->v_token_stride; p.v_head = c->v_head_stride;
    p.n_pages = c->n_pages;
    p.page_shift = __builtin_ctzll((unsigned long long)c->page_size);
    p.table = table; p.width = width; p.table_stride = stride;
    return p;
}

namespace {

constexpr int kKnownStarts = 1024;   // sequences whose row ranges a CTA holds in shared memory

struct AppendArgs {
    PagedView c;
    const void *kn, *vn, *q;
    void *qo, *bounds;
    int64_t kn_tok, vn_tok, q_tok, N, B, H, Hkv, D;
    const int32_t *cu, *start;
    const double *inv_freq;
    int rot, interleaved, tile;     // tile: tokens per CTA of the rows kernel
    int *status;
};

__device__ __forceinline__ void angle_of(double pos, double freq, float &c, float &s) {
    const double half_turns = pos * (freq * 0.31830988618379067154);
    const double r = half_turns - 2.0 * rint(0.5 * half_turns);   // in [-1, 1]
    sincospif((float)r, &s, &c);
}

// First row of sequence b (b = B: the end of the last), inside [0, N] whatever cu_seqlens holds.
__device__ __forceinline__ int64_t first_row(const AppendArgs &a, int64_t b) {
    if (!a.cu) return b;
    const int64_t n = __ldg(a.cu + b);
    return n < 0 ? 0 : n > a.N ? a.N : n;
}

// Columns of one row in units of two vectors of W: unit u's vectors start at columns at0 and at1.  Its pairs (from
// `pair` on, -1: not rotated) are (first vector, second vector) element by element, or neighbours when interleaved.
// W = 1 serves rotations whose halves do not start on 16 bytes, pair by pair.
template <int W> struct Unit {
    int at0, at1, pair;
    __device__ __forceinline__ Unit(int u, int rot, bool interleaved) {
        if (u * 2 * W < rot) {
            pair = u * W;
            at0 = interleaved ? 2 * u * W : u * W;
            at1 = interleaved ? at0 + W : rot / 2 + u * W;
        } else {
            pair = -1;
            at0 = u * 2 * W;
            at1 = at0 + W;
        }
    }
};

// x: the 2 W values of a unit; c, s: cosine and sine of its pairs
template <int W> __device__ __forceinline__ void turn(float *x, const float *c, const float *s, bool interleaved) {
    if (interleaved) {
#pragma unroll
        for (int i = 0; i < W; ++i) {
            const float a = x[2 * i], b = x[2 * i + 1];
            x[2 * i] = a * c[i] - b * s[i];
            x[2 * i + 1] = b * c[i] + a * s[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < W; ++i) {
            const float a = x[i], b = x[W + i];
            x[i] = a * c[i] - b * s[i];
            x[W + i] = b * c[i] + a * s[i];
        }
    }
}

template <typename T, bool VEC> __global__ void __launch_bounds__(256, 4) append_rows_kernel(const AppendArgs a) {
    constexpr int W = VEC ? Vec16<T>::N : 1, U = 2;
    __shared__ int starts[kKnownStarts + 1];         // first rows of the sequences
    __shared__ int pos_of[64];
    __shared__ int64_t k_of[64], v_of[64];
    extern __shared__ __align__(16) float turns[];                 // [tile][rot / 2] cosines, then sines
    pdl_trigger();
    const int tid = threadIdx.x, D = (int)a.D, half = a.rot / 2;
    const int64_t n0 = (int64_t)blockIdx.x * a.tile;
    const int cnt = (int)(a.N - n0 < a.tile ? a.N - n0 : a.tile);
    float *cosines = turns, *sines = turns + a.tile * half;
    const bool known = a.B <= kKnownStarts;
    if (a.cu && known)
        for (int i = tid; i <= a.B; i += 256) starts[i] = (int)first_row(a, i);
    __syncthreads();
    if (tid < cnt) {
        const int64_t n = n0 + tid;
        int64_t b = n, begin = n, pos = -1, k = -1, v = -1;
        if (a.cu) {                                  // the last sequence that starts at or before n
            int64_t lo = 0, hi = a.B - 1;
            while (lo < hi) {
                const int64_t mid = (lo + hi + 1) >> 1;
                if ((known ? (int64_t)starts[mid] : first_row(a, mid)) <= n) lo = mid; else hi = mid - 1;
            }
            b = lo;
            begin = first_row(a, b);
            if (n < begin || n >= first_row(a, b + 1)) b = -1;      // padding
        }
        if (b >= 0) {
            const int64_t at = a.start[b];
            if (at < 0) {
                atomicOr(a.status, kPagedOutside);
            } else {
                pos = at + n - begin;
                if (pos > INT_MAX) atomicOr(a.status, kPagedOutside);
                const int64_t phys = pos > INT_MAX ? -1 : physical_page(a.c, b, pos >> a.c.page_shift, a.status);
                const int64_t slot = pos & ((1 << a.c.page_shift) - 1);
                if (phys >= 0) {
                    k = phys * a.c.k_page + slot * a.c.k_tok;
                    v = phys * a.c.v_page + slot * a.c.v_tok;
                }
            }
        }
        pos_of[tid] = pos > INT_MAX ? -1 : (int)pos;
        k_of[tid] = k;
        v_of[tid] = v;
    }
    __syncthreads();
    for (int i = tid; i < cnt * half; i += 256) {
        const int t = i / half;
        angle_of((double)pos_of[t], a.inv_freq[i - t * half], cosines[i], sines[i]);
    }
    __syncthreads();
    // a thread keeps its head and columns and walks over the tokens: 256 (head, unit) pairs at a time, several tokens
    // side by side where there are fewer
    const int units = (D + 2 * W - 1) / (2 * W), heads_q = a.q ? (int)a.H : 0, heads_k = (int)a.Hkv, pairs = (heads_q + 2 * heads_k) * units;
    for (int p0 = 0; p0 < pairs; p0 += 256) {
        const int width = pairs - p0 < 256 ? pairs - p0 : 256, lanes = 256 / width, lane = tid / width;
        if (lane >= lanes) continue;
        const int at = p0 + tid - lane * width, role = at / units;
        const Unit<W> u(at - role * units, a.rot, a.interleaved);
        const bool is_q = role < heads_q, is_v = role >= heads_q + heads_k, second = u.at1 < D;
        const int h = is_q ? role : is_v ? role - heads_q - heads_k : role - heads_q;
        const bool turned = u.pair >= 0 && !is_v;
        const int64_t src_tok = is_q ? a.q_tok : is_v ? a.vn_tok : a.kn_tok;
        const T *src = (const T *)(is_q ? a.q : is_v ? a.vn : a.kn) + n0 * src_tok + (int64_t)h * D;
        T *dst = is_q ? (T *)a.qo + (n0 * a.H + h) * D : is_v ? (T *)a.c.v + h * a.c.v_head : (T *)a.c.k + h * a.c.k_head;
        for (int t0 = lane; t0 < cnt; t0 += lanes * U) {
            uint4 raw[U][2];
            int64_t to[U];
#pragma unroll
            for (int y = 0; y < U; ++y) {
                const int t = t0 + y * lanes;
                to[y] = t >= cnt || pos_of[t] < 0 ? -1 : is_q ? t * a.H * D : is_v ? v_of[t] : k_of[t];
                if (to[y] < 0) continue;
                const T *from = src + t * src_tok;
                if (VEC) {
                    raw[y][0] = *reinterpret_cast<const uint4 *>(from + u.at0);
                    if (second) raw[y][1] = *reinterpret_cast<const uint4 *>(from + u.at1);
                } else {
                    raw[y][0].x = __float_as_uint(Elem<T>::to_f(from[u.at0]));
                    raw[y][1].x = __float_as_uint(Elem<T>::to_f(from[u.at1]));
                }
            }
#pragma unroll
            for (int y = 0; y < U; ++y) {
                if (to[y] < 0) continue;
                T *out = dst + to[y];
                if (turned) {
                    float x[2 * W];
                    __align__(16) float c[W >= 4 ? W : 4], s[W >= 4 ? W : 4];
                    const int first = (t0 + y * lanes) * half + u.pair;
                    if (VEC) {
#pragma unroll
                        for (int i = 0; i < W; i += 4) {      // a unit's pairs start on 16 bytes: rot is a multiple of 2 W
                            *reinterpret_cast<float4 *>(c + i) = *reinterpret_cast<const float4 *>(cosines + first + i);
                            *reinterpret_cast<float4 *>(s + i) = *reinterpret_cast<const float4 *>(sines + first + i);
                        }
                    } else {
                        c[0] = cosines[first];
                        s[0] = sines[first];
                    }
                    if (VEC) {
                        Vec16<T>::unpack(raw[y][0], x);
                        Vec16<T>::unpack(raw[y][1], x + W);
                    } else {
                        x[0] = __uint_as_float(raw[y][0].x);
                        x[W] = __uint_as_float(raw[y][1].x);
                    }
                    turn<W>(x, c, s, a.interleaved);
                    if (VEC) {
                        raw[y][0] = Vec16<T>::pack(x);
                        raw[y][1] = Vec16<T>::pack(x + W);
                    } else {
                        raw[y][0].x = __float_as_uint(x[0]);
                        raw[y][1].x = __float_as_uint(x[W]);
                    }
                }
                if (VEC) {
                    *reinterpret_cast<uint4 *>(out + u.at0) = raw[y][0];
                    if (second) *reinterpret_cast<uint4 *>(out + u.at1) = raw[y][1];
                } else {
                    out[u.at0] = Elem<T>::from_f(__uint_as_float(raw[y][0].x));
                    out[u.at1] = Elem<T>::from_f(__uint_as_float(raw[y][1].x));
                }
            }
        }
    }
}

// Bounds of one page and head from its first `filled` slots, by one warp: LV lanes of 16 bytes share a token.  A NaN key
// makes its column's bounds NaN, so that the page's score says so.
template <typename T> __device__ void page_bounds(const AppendArgs &a, int64_t phys, int h, int filled) {
    constexpr int W = Vec16<T>::N;
    const int lane = threadIdx.x % 32, D = (int)a.D, vecs = D / W;
    const int lv = vecs <= 1 ? 1 : vecs <= 2 ? 2 : vecs <= 4 ? 4 : vecs <= 8 ? 8 : vecs <= 16 ? 16 : 32, lt = 32 / lv;
    const T *rows = (const T *)a.c.k + phys * a.c.k_page + (int64_t)h * a.c.k_head;
    T *out = (T *)a.bounds + (phys * 2 * a.Hkv + h) * (int64_t)D;
    for (int v0 = 0; v0 < vecs; v0 += lv) {
        const int col = (v0 + lane % lv) * W;
        float lo[W], hi[W];
#pragma unroll
        for (int j = 0; j < W; ++j) { lo[j] = INFINITY; hi[j] = -INFINITY; }
        if (col < D)
#pragma unroll 8
            for (int s = lane / lv; s < filled; s += lt) {
                float x[W];
                Vec16<T>::unpack(*reinterpret_cast<const uint4 *>(rows + s * a.c.k_tok + col), x);
#pragma unroll
                for (int j = 0; j < W; ++j) { lo[j] = ptx::min_nan(lo[j], x[j]); hi[j] = ptx::max_nan(hi[j], x[j]); }
            }
        for (int o = lv; o < 32; o <<= 1)
#pragma unroll
            for (int j = 0; j < W; ++j) {
                lo[j] = ptx::min_nan(lo[j], __shfl_xor_sync(0xffffffffu, lo[j], o));
                hi[j] = ptx::max_nan(hi[j], __shfl_xor_sync(0xffffffffu, hi[j], o));
            }
        if (lane < lv && col < D) {
            *reinterpret_cast<uint4 *>(out + col) = Vec16<T>::pack(lo);
            *reinterpret_cast<uint4 *>(out + a.Hkv * (int64_t)D + col) = Vec16<T>::pack(hi);
        }
    }
}

// Warp x < B: the first page of sequence x; warp B + t: the pages that begin inside rows [t * page, (t + 1) * page) of
// the packed batch and are not a sequence's first.
template <typename T> __global__ void __launch_bounds__(128) page_bounds_kernel(const AppendArgs a) {
    pdl_trigger();
    pdl_wait();
    const int64_t item = (int64_t)blockIdx.x * 4 + threadIdx.x / 32;
    const int lane = threadIdx.x % 32, h = blockIdx.y, page = 1 << a.c.page_shift;
    auto one = [&](int64_t b, int64_t pos, int64_t count) {       // `count` new tokens from position pos on one page
        if (pos < 0 || pos > INT_MAX) return;
        const int64_t phys = physical_page(a.c, b, pos >> a.c.page_shift, a.status);
        if (phys >= 0) page_bounds<T>(a, phys, h, (int)((pos & (page - 1)) + count));
    };
    if (item < a.B) {
        const int64_t n0 = first_row(a, item), end = first_row(a, item + 1), pos = a.start[item], room = page - (pos & (page - 1));
        if (n0 < end) one(item, pos, room < end - n0 ? room : end - n0);
        return;
    }
    const int64_t t0 = (item - a.B) * page, t1 = t0 + page;
    if (!a.cu || t0 >= a.N) return;
    int64_t lo = 0, hi = a.B - 1;                    // the last sequence that starts at or before t0, 32 guesses at a time
    while (lo < hi) {
        const int64_t step = (hi - lo + 32) / 32, at = lo + lane * step;
        const uint32_t before = __ballot_sync(0xffffffffu, at <= hi && first_row(a, at) <= t0);
        if (!before) break;                          // only for malformed cu_seqlens
        lo += (31 - __clz(before)) * step;
        hi = hi < lo + step - 1 ? hi : lo + step - 1;
    }
    for (int64_t b0 = lo; b0 < a.B; b0 += 32) {      // 32 sequences at a time: at most one page of each begins here
        const int64_t b = b0 + lane;
        int64_t n = -1, pos = 0, count = 0;
        bool more = false;
        if (b < a.B) {
            const int64_t n0 = first_row(a, b), end = first_row(a, b + 1), at = a.start[b];
            more = n0 < t1;
            if (more && n0 < end && at >= 0) {
                n = n0 + page - (at & (page - 1));   // the first row on a page of its own
                if (n < t0) n += (t0 - n + page - 1) / page * page;
                if (n >= t1 || n >= end) n = -1;
                pos = at + n - n0;
                count = page < end - n ? page : end - n;
            }
        }
        uint32_t found = __ballot_sync(0xffffffffu, n >= 0);
        while (found) {
            const int who = __ffs(found) - 1;
            found &= found - 1;
            one(b0 + who, __shfl_sync(0xffffffffu, pos, who), __shfl_sync(0xffffffffu, count, who));
        }
        if (!__all_sync(0xffffffffu, more)) return;
    }
}

template <typename T> int launch_append(AppendArgs &a, bool vec, cudaStream_t stream) {
    // one wave of CTAs (four a SM) where a tile of at most 64 tokens and 32 KB of angles allows it
    const int64_t wave = 148 * 4, most = a.rot ? min((int64_t)64, (int64_t)32768 / (a.rot * 4)) : 64;
    a.tile = (int)min(most, (a.N + wave - 1) / wave);
    const unsigned tiles = (unsigned)((a.N + a.tile - 1) / a.tile);
    const size_t smem = (size_t)a.tile * a.rot * sizeof(float);
    if (vec) append_rows_kernel<T, true><<<tiles, 256, smem, stream>>>(a);
    else append_rows_kernel<T, false><<<tiles, 256, smem, stream>>>(a);
    cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess && a.bounds) {
        const int64_t page = 1ll << a.c.page_shift, items = a.B + (a.cu ? (a.N + page - 1) / page : 0);
        e = launch_after(page_bounds_kernel<T>, dim3((unsigned)((items + 3) / 4), (unsigned)a.Hkv), dim3(128), 0, stream, a);
    }
    return e == cudaSuccess ? MAT_OK : cuda_fail(e, "launching the paged append");
}

}  // namespace
}  // namespace mat

using namespace mat;

extern "C" int mat_paged_append(const mat_paged_cache *cache, const void *k_new, const void *v_new, int64_t k_token_stride,
                                int64_t v_token_stride, int64_t N, const int32_t *cu_seqlens, const int32_t *start,
                                const int32_t *page_table, int64_t table_width, int64_t table_stride, int64_t B,
                                const void *q, void *q_out, int64_t H, int64_t q_token_stride, const double *inv_freq,
                                int64_t rot, int interleaved, void *stream) {
    if (int rc = check_paged_cache(cache)) return rc;
    if (int rc = check_page_table(page_table, table_width, table_stride, B)) return rc;
    if (N < 0 || N > INT_MAX) return fail(MAT_ERR_INVALID, "the number of new tokens must be in [0, 2^31), got %lld", (long long)N);
    if (!cu_seqlens && N != B) return fail(MAT_ERR_INVALID, "without cu_seqlens every sequence gets one token: N = %lld, B = %lld", (long long)N, (long long)B);
    if (N == 0) return MAT_OK;
    if (!k_new || !v_new || !start) return fail(MAT_ERR_INVALID, "k_new, v_new and start must be non-NULL");
    if ((q == nullptr) != (q_out == nullptr)) return fail(MAT_ERR_INVALID, "q and q_out come together");
    const int64_t D = cache->D, Hkv = cache->H_kv, vec = 16 / (int64_t)dtype_size(cache->dtype);
    if (q && H > 65535) return fail(MAT_ERR_UNSUPPORTED, "at most 65535 query heads");
    if (q && (H < Hkv || H % Hkv)) return fail(MAT_ERR_INVALID, "H = %lld query heads do not divide over H_kv = %lld key heads", (long long)H, (long long)Hkv);
    if (rot < 0 || rot > D || rot % 2) return fail(MAT_ERR_INVALID, "the rotated width must be even and at most D, got %lld", (long long)rot);
    if (rot > 0 && !inv_freq) return fail(MAT_ERR_INVALID, "a rotation needs its frequencies");
    const int64_t ts[3] = {k_token_stride, v_token_stride, q ? q_token_stride : 0};
    for (int64_t t : ts)
        if (t < 0 || t % vec) return fail(MAT_ERR_INVALID, "token strides must be non-negative multiples of 16 bytes");
    if (((uintptr_t)k_new | (uintptr_t)v_new | (uintptr_t)q | (uintptr_t)q_out) % 16)
        return fail(MAT_ERR_INVALID, "k_new, v_new, q and q_out must be 16-byte aligned");
    AppendArgs a;
    a.c = paged_view(cache, page_table, table_width, table_stride);
    a.kn = k_new; a.vn = v_new; a.q = q; a.qo = q_out; a.bounds = cache->key_bounds;
    a.kn_tok = k_token_stride; a.vn_tok = v_token_stride; a.q_tok = q_token_stride;
    a.N = N; a.B = B; a.H = H; a.Hkv = Hkv; a.D = D;
    a.cu = cu_seqlens; a.start = start; a.inv_freq = inv_freq;
    a.rot = inv_freq ? (int)rot : 0;
    a.interleaved = interleaved != 0;
    if (!(a.status = paged_status_word())) return fail(MAT_ERR_CUDA, "no device status word");
    const bool whole = a.rot % (2 * vec) == 0;   // both halves of a rotated pair start on 16 bytes
    note_kernel(whole ? "paged_append" : "paged_append_pairs");
    cudaStream_t s = (cudaStream_t)stream;
    switch (cache->dtype) {
        case MAT_F32: return launch_append<float>(a, whole, s);
        case MAT_BF16: return launch_append<__nv_bfloat16>(a, whole, s);
        default: return launch_append<__half>(a, whole, s);
    }
}
