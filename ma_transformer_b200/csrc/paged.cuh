// Shared by the paged-cache kernels: the cache as the kernels see it, the walk from a token's position to its row, and
// 16-byte accesses as fp32 values.
#pragma once

#include "mat_common.cuh"
#include "ptx.cuh"

namespace mat {

struct PagedView {
    const void *k, *v;
    int64_t k_page, k_tok, k_head, v_page, v_tok, v_head;   // strides in elements
    int64_t n_pages;
    int page_shift;
    const int32_t *table;
    int64_t width, table_stride;
};

constexpr int kPagedOutside = 2;   // status bit: a table entry or a start position outside the cache

int check_paged_cache(const mat_paged_cache *c);
int check_page_table(const int32_t *table, int64_t width, int64_t stride, int64_t B);
PagedView paged_view(const mat_paged_cache *c, const int32_t *table, int64_t width, int64_t stride);
int *paged_status_word();                    // device address of the status word on the current device (NULL: error)
int paged_status_read_and_clear(int *out);

// Physical page of a logical one, or -1 where the table has none inside the cache.
__device__ __forceinline__ int64_t physical_page(const PagedView &c, int64_t b, int64_t logical, int *status) {
    if (logical < 0 || logical >= c.width) {
        atomicOr(status, kPagedOutside);
        return -1;
    }
    const int32_t p = __ldg(c.table + b * c.table_stride + logical);
    if (p < 0 || p >= c.n_pages) {
        atomicOr(status, kPagedOutside);
        return -1;
    }
    return p;
}

// The table's entry alone, for several pages at once: with the report in between, the reads wait for each other (a step
// of four pages took the page scores 2.6 us, 1.8 without).
__device__ __forceinline__ int32_t table_entry(const PagedView &c, int64_t b, int64_t logical) {
    return logical >= 0 && logical < c.width ? __ldg(c.table + b * c.table_stride + logical) : -1;
}
// 16 bytes of elements as fp32 values and back.
template <typename T> struct Vec16;
template <> struct Vec16<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void unpack(const uint4 &u, float *f) {
        f[0] = __uint_as_float(u.x); f[1] = __uint_as_float(u.y); f[2] = __uint_as_float(u.z); f[3] = __uint_as_float(u.w);
    }
    static __device__ __forceinline__ uint4 pack(const float *f) {
        return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
    }
};
template <typename T> struct Vec16Half {
    static constexpr int N = 8;
    static __device__ __forceinline__ void unpack(const uint4 &u, float *f) {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = ptx::Mma<T>::lo(w[i]);
            f[2 * i + 1] = ptx::Mma<T>::hi(w[i]);
        }
    }
    static __device__ __forceinline__ uint4 pack(const float *f) {
        return make_uint4(ptx::Mma<T>::pack(f[0], f[1]), ptx::Mma<T>::pack(f[2], f[3]), ptx::Mma<T>::pack(f[4], f[5]), ptx::Mma<T>::pack(f[6], f[7]));
    }
};
template <> struct Vec16<__nv_bfloat16> : Vec16Half<__nv_bfloat16> {};
template <> struct Vec16<__half> : Vec16Half<__half> {};

}  // namespace mat
