// Appends new tokens to a paged key-value cache: keys (and optionally the queries of the same tokens) turned by their
// positions, values copied, and the touched pages' key bounds set, in one launch.
//
// Rotation: column pair (a, b) at position p with frequency f becomes (a cos t - b sin t, b cos t + a sin t), t = p f.
// The angle is formed in 64 bits as a number of half turns, p * (f / pi), and reduced by its nearest even integer
// before it is rounded to fp32 (an fp32 product would be off by p * f * 2^-24: 0.06 rad at position 10^6).
//
// One CTA owns one page of one sequence: it writes the call's tokens of that page and then knows every filled slot, so
// the bounds (smallest and largest key per column) need no atomics.  CTA x < B takes sequence x's first page, CTA B + t
// the pages that begin inside rows [t * page, (t + 1) * page) of the packed batch; y is the key head (with the query
// heads that read it).  Bounds are taken from all filled slots, not merged with the old ones: a cache that was rolled
// back and written again ends with the same bits as one that never was.
#include <limits.h>

#include <atomic>

#include "paged.cuh"

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

constexpr int kThreads = 256;   // at least two lanes per column pair at D = 256

struct AppendArgs {
    PagedView c;
    const void *kn, *vn, *q;
    void *qo, *bounds;
    int64_t kn_tok, vn_tok, q_tok, N, B, H, Hkv, D;
    const int32_t *cu, *start;
    const double *inv_freq;
    int rot, interleaved;
    int *status;
};

__device__ __forceinline__ void angle_of(double pos, double freq, float &c, float &s) {
    const double half_turns = pos * (freq * 0.31830988618379067154);
    const double r = half_turns - 2.0 * rint(0.5 * half_turns);   // in [-1, 1]
    sincospif((float)r, &s, &c);
}

// Columns of one row in units of two vectors of four: unit u's vectors start at columns at0, at1, and its pairs are
// (first vector, second vector) element by element, or neighbours when interleaved.  Four columns (8 bytes of a 16-bit
// type) keep the kernel within 64 registers, four CTAs a SM: with 16-byte vectors it held two, and packed prompts of
// 32768 tokens x (12 + 2 * 4) heads of 64 took 177 us instead of WIDE_US.
constexpr int W = 4;
struct Unit {
    int at0, at1, pair;   // pair: index of the unit's first rotated pair, -1 for none
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

// four elements as fp32 values and back
template <typename T> struct Four {
    static __device__ __forceinline__ void load(const T *p, float *x) {
        const uint2 u = *reinterpret_cast<const uint2 *>(p);
        x[0] = Vec16<T>::one((uint16_t)(u.x & 0xffffu)); x[1] = Vec16<T>::one((uint16_t)(u.x >> 16));
        x[2] = Vec16<T>::one((uint16_t)(u.y & 0xffffu)); x[3] = Vec16<T>::one((uint16_t)(u.y >> 16));
    }
    static __device__ __forceinline__ void store(T *p, const float *x) {
        *reinterpret_cast<uint2 *>(p) = make_uint2(Vec16<T>::two(x[0], x[1]), Vec16<T>::two(x[2], x[3]));
    }
};
template <> struct Four<float> {
    static __device__ __forceinline__ void load(const float *p, float *x) { *reinterpret_cast<float4 *>(x) = *reinterpret_cast<const float4 *>(p); }
    static __device__ __forceinline__ void store(float *p, const float *x) { *reinterpret_cast<float4 *>(p) = *reinterpret_cast<const float4 *>(x); }
};

// x: the 2 N values of a unit; c, s: cosine and sine of its N pairs
template <int N> __device__ __forceinline__ void turn(float *x, const float *c, const float *s, bool interleaved) {
    if (interleaved) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float a = x[2 * i], b = x[2 * i + 1];
            x[2 * i] = a * c[i] - b * s[i];
            x[2 * i + 1] = b * c[i] + a * s[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float a = x[i], b = x[N + i];
            x[i] = a * c[i] - b * s[i];
            x[N + i] = b * c[i] + a * s[i];
        }
    }
}

// Columns that no vector path serves (a rotation whose halves do not start on 16 bytes): pair by pair.
template <typename T> __device__ __forceinline__ void pair_columns(int r, int rot, bool interleaved, int &c0, int &c1) {
    if (2 * r < rot) {
        c0 = interleaved ? 2 * r : r;
        c1 = interleaved ? 2 * r + 1 : r + rot / 2;
    } else {
        c0 = 2 * r;
        c1 = 2 * r + 1;
    }
}

// One page of one sequence: rows [n0, n0 + count) of the packed batch land in slots [slot0, slot0 + count).
template <typename T, bool VEC>
__device__ void append_page(const AppendArgs &a, int64_t b, int64_t n0, int count, int64_t pos0, float *red) {
    constexpr int N = VEC ? W : 1;
    const int h = blockIdx.y, G = a.q ? (int)(a.H / a.Hkv) : 0;
    const int D = (int)a.D;
    const int units = D / (2 * N);
    const int lanes = kThreads / units;               // rows in flight
    const int u = threadIdx.x % units, lane = threadIdx.x / units;
    const bool active = lane < lanes;
    const int page = 1 << a.c.page_shift;
    const int slot0 = (int)(pos0 & (page - 1));
    const int64_t phys = physical_page(a.c, b, pos0 >> a.c.page_shift, a.status);

    // tokens over lanes; lanes left over take the roles (key, value, query heads) of a token in turn
    int tl = 1;
    while (tl * 2 <= lanes && tl < count) tl *= 2;
    const int rl = lanes / tl, my_t = lane % tl, my_r = lane / tl;

    float lo[2 * N], hi[2 * N];
#pragma unroll
    for (int i = 0; i < 2 * N; ++i) { lo[i] = INFINITY; hi[i] = -INFINITY; }

    int c0[2] = {0, 0};
    Unit un(VEC ? u : 0, a.rot, a.interleaved);
    bool rotated = un.pair >= 0;
    if (!VEC) {
        pair_columns<T>(u, a.rot, a.interleaved, c0[0], c0[1]);
        rotated = 2 * u < a.rot;
    }
    auto load = [&](const T *row, float *x) {
        if (VEC) { Four<T>::load(row + un.at0, x); Four<T>::load(row + un.at1, x + N); }
        else { x[0] = Elem<T>::to_f(row[c0[0]]); x[N] = Elem<T>::to_f(row[c0[1]]); }
    };
    auto store = [&](T *row, const float *x) {
        if (VEC) { Four<T>::store(row + un.at0, x); Four<T>::store(row + un.at1, x + N); }
        else { row[c0[0]] = Elem<T>::from_f(x[0]); row[c0[1]] = Elem<T>::from_f(x[N]); }
    };
    T *kp = (T *)a.c.k + (phys < 0 ? 0 : phys * a.c.k_page) + (int64_t)h * a.c.k_head;
    T *vp = (T *)a.c.v + (phys < 0 ? 0 : phys * a.c.v_page) + (int64_t)h * a.c.v_head;

    if (active && my_r < rl) {
        for (int t = my_t; t < count; t += tl) {
            const int64_t n = n0 + t;
            float cs[N], sn[N];
            if (rotated) {
                const int pair = VEC ? un.pair : u;
#pragma unroll
                for (int i = 0; i < N; ++i) angle_of((double)(pos0 + t), a.inv_freq[pair + i], cs[i], sn[i]);
            }
            for (int role = my_r; role < G + 2; role += rl) {
                float x[2 * N];
                if (role == 1) {          // value
                    if (phys >= 0) {
                        load((const T *)a.vn + n * a.vn_tok + (int64_t)h * D, x);
                        store(vp + (int64_t)(slot0 + t) * a.c.v_tok, x);
                    }
                    continue;
                }
                const T *src = role == 0 ? (const T *)a.kn + n * a.kn_tok + (int64_t)h * D
                                         : (const T *)a.q + n * a.q_tok + ((int64_t)h * G + role - 2) * D;
                if (role == 0 && phys < 0) continue;
                load(src, x);
                if (rotated) turn<N>(x, cs, sn, a.interleaved);
                if (role == 0) {
                    store(kp + (int64_t)(slot0 + t) * a.c.k_tok, x);
#pragma unroll
                    for (int i = 0; i < 2 * N; ++i) {
                        const float y = Elem<T>::to_f(Elem<T>::from_f(x[i]));   // the key as the cache holds it
                        lo[i] = fminf(lo[i], y);
                        hi[i] = fmaxf(hi[i], y);
                    }
                } else {
                    store((T *)a.qo + (n * a.H + (int64_t)h * G + role - 2) * D, x);
                }
            }
        }
        if (a.bounds && phys >= 0)
            for (int s = lane; s < slot0; s += lanes) {      // slots filled by earlier calls
                float x[2 * N];
                load(kp + (int64_t)s * a.c.k_tok, x);
#pragma unroll
                for (int i = 0; i < 2 * N; ++i) {
                    lo[i] = fminf(lo[i], x[i]);
                    hi[i] = fmaxf(hi[i], x[i]);
                }
            }
    }
    if (!a.bounds) return;            // the same for the whole grid
    // join the lanes' bounds; red: [lo, hi][element of a unit][thread]
#pragma unroll
    for (int i = 0; i < 2 * N; ++i) {
        red[i * kThreads + threadIdx.x] = lo[i];
        red[(2 * N + i) * kThreads + threadIdx.x] = hi[i];
    }
    __syncthreads();
    if (phys < 0) return;
    const int used = min(lanes, max(tl, slot0));        // lanes that saw a key
    T *out = (T *)a.bounds + (phys * 2 * a.Hkv + h) * (int64_t)D;
    for (int o = threadIdx.x; o < 4 * N * units; o += kThreads) {
        const bool is_hi = o >= 2 * N * units;
        const int r = is_hi ? o - 2 * N * units : o, i = r / units, v = r % units;
        int col[2] = {0, 0};
        if (VEC) {
            const Unit w(v, a.rot, a.interleaved);
            col[0] = w.at0 + i; col[1] = w.at1 + i - N;
        } else {
            pair_columns<T>(v, a.rot, a.interleaved, col[0], col[1]);
        }
        const int c = i < N ? col[0] : col[1];
        const float *x = red + (is_hi ? 2 * N + i : i) * kThreads + v;
        float m = x[0];
        for (int l = 1; l < used; ++l) m = is_hi ? fmaxf(m, x[l * units]) : fminf(m, x[l * units]);
        out[(is_hi ? a.Hkv * (int64_t)D : 0) + c] = Elem<T>::from_f(m);
    }
}

template <typename T, bool VEC> __global__ void __launch_bounds__(kThreads, 4) append_kernel(const AppendArgs a) {
    __shared__ float red[4 * (VEC ? W : 1) * kThreads];
    const int page = 1 << a.c.page_shift;
    auto first_row = [&](int64_t b) -> int64_t {
        if (!a.cu) return b;
        const int64_t n = a.cu[b];
        return n < 0 ? 0 : (n > a.N ? a.N : n);
    };
    if (blockIdx.x < a.B) {
        const int64_t b = blockIdx.x, n0 = first_row(b), end = first_row(b + 1);
        if (n0 >= end) return;
        const int64_t pos = a.start[b];
        if (pos < 0) {
            atomicOr(a.status, kPagedOutside);
            return;
        }
        const int64_t room = page - (pos & (page - 1));
        append_page<T, VEC>(a, b, n0, (int)(room < end - n0 ? room : end - n0), pos, red);
        return;
    }
    // pages that begin inside this tile of rows and are not a sequence's first
    const int64_t t0 = (int64_t)(blockIdx.x - a.B) * page, t1 = t0 + page;
    int64_t lo = 0, hi = a.B - 1;                    // the last sequence that starts at or before t0, 32 guesses at a time
    while (lo < hi) {
        const int64_t step = (hi - lo + 32) / 32, at = lo + (threadIdx.x % 32) * step;
        const uint32_t before = __ballot_sync(0xffffffffu, at <= hi && first_row(at) <= t0);
        if (!before) break;                          // only for malformed cu_seqlens
        lo += (31 - __clz(before)) * step;
        hi = hi < lo + step - 1 ? hi : lo + step - 1;
    }
    for (int64_t b = lo; b < a.B && first_row(b) < t1; ++b) {
        const int64_t n0 = first_row(b), end = first_row(b + 1), pos = a.start[b];
        if (n0 >= end || pos < 0) continue;
        int64_t n = n0 + page - (pos & (page - 1));  // the first row on a page of its own
        if (n < t0) n += (t0 - n + page - 1) / page * page;
        if (n >= t1 || n >= end) continue;
        append_page<T, VEC>(a, b, n, (int)(page < end - n ? page : end - n), pos + n - n0, red);
        __syncthreads();
    }
}

template <typename T> int launch_append(const AppendArgs &a, bool vec, cudaStream_t stream) {
    const int64_t page = 1ll << a.c.page_shift;
    const int64_t gx = a.B + (a.cu ? (a.N + page - 1) / page : 0);
    dim3 grid((unsigned)gx, (unsigned)a.Hkv);
    if (vec) append_kernel<T, true><<<grid, kThreads, 0, stream>>>(a);
    else append_kernel<T, false><<<grid, kThreads, 0, stream>>>(a);
    cudaError_t e = cudaGetLastError();
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
    const bool v4 = a.rot % (2 * W) == 0;   // both halves of a rotated pair start on a vector
    note_kernel(v4 ? "paged_append" : "paged_append_pairs");
    cudaStream_t s = (cudaStream_t)stream;
    switch (cache->dtype) {
        case MAT_F32: return launch_append<float>(a, v4, s);
        case MAT_BF16: return launch_append<__nv_bfloat16>(a, v4, s);
        default: return launch_append<__half>(a, v4, s);
    }
}
