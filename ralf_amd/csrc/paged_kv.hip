// The paged key / value cache: written (quantised on the way) and read back.
//
// A row is one head's key or value of one token: dim elements, 8 to a lane.  Writing in 8 bits takes the largest magnitude over the row's lanes as an INTEGER
// maximum of the bit patterns (ordered like the values, infinities and NaN on top), takes the exponent from its bits, and scales by a power of two -- exact, so
// only the one rounding to the code remains and every reader gets the same value.  Both kernels are bound by bytes; a wave takes whole tokens, so that finding
// the sequence (64 probes in one load) and the page is paid once per token and not per row.  42 500 tokens of 2 x 8 x 128 e4m3 -> bf16: 261 MB in 53 us (4.9 TB/s);
// 10 600 tokens bf16 -> e4m3: 65 MB in 18 us behind a kernel that has filled the caches with other data, 14 alone (a wave's chain of three trips to memory; it takes one
// token's rows of all heads, so its stores are 128 bytes in as many places of a page).
#include "paged.h"

namespace {
using namespace paged;

struct WriteArgs {
    RalfPagedKV c;
    const void* k; const void* v;
    int64_t k_ts, k_hs, v_ts, v_hs, T;
    const int* q_start;
};
struct ReadArgs {
    RalfPagedKV c;
    void* k; void* v;
    int64_t rows;
    const int* start;
};

// 8 elements as loaded -> fp32 (bf16: r0 alone)
template <typename T> __device__ __forceinline__ void spread(const u32x4 r0, const u32x4 r1, float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 2) {
            f[2 * i] = __uint_as_float(r0[i] << 16);
            f[2 * i + 1] = __uint_as_float(r0[i] & 0xffff0000u);
        } else {
            f[i] = __uint_as_float(r0[i]);
            f[4 + i] = __uint_as_float(r1[i]);
        }
    }
}
template <typename T> __device__ __forceinline__ void load8(const T* p, float (&f)[8]) {
    const u32x4 r0 = *(const u32x4*)p;
    u32x4 r1 = r0;
    if constexpr (sizeof(T) == 4) r1 = *(const u32x4*)(p + 4);
    spread<T>(r0, r1, f);
}

// token `t` (the same in all lanes) -> page * (heads * page) .. row index of head 0, or -1 where nothing is to be stored / to be read
__device__ __forceinline__ int64_t place(const RalfPagedKV& c, int b, int64_t p) {
    if (p < 0 || p >= (int64_t)c.max_pages * c.page) return -1;
    const int pi = (int)(p / c.page);
    const int pg = c.table[(int64_t)b * c.table_ld + pi];
    if (pg < 0 || pg >= c.n_pages) return -1;
    return (int64_t)pg * c.heads * c.page + (p - (int64_t)pi * c.page);
}

// one row's share of a lane -> the pool
template <typename T, int STORE, int LANES, int D>
__device__ __forceinline__ void store_row(const RalfPagedKV& c, bool isv, int64_t row, int e0, const u32x4 r0, const u32x4 r1) {
    if constexpr (STORE <= RALF_KV_BF16) {
        T* dst = (T*)(isv ? c.v : c.k) + row * D + e0;
        *(u32x4*)dst = r0;
        if constexpr (sizeof(T) == 4) *(u32x4*)(dst + 4) = r1;
    } else {
        float f[8];
        spread<T>(r0, r1, f);
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) { const uint32_t u = __float_as_uint(f[i]) & 0x7fffffffu; m = m > u ? m : u; }
#pragma unroll
        for (int o = 1; o < LANES; o <<= 1) { const uint32_t u = __shfl_xor(m, o); m = m > u ? m : u; }
        const uint32_t ex = exp_byte<STORE>(m);
        u32x2 code = {0u, 0u};
        if (ex != 255u) {
            const float inv = exp_inverse(ex), top = largest_code<STORE>(ex);
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = __builtin_amdgcn_fmed3f(f[i] * inv, -top, top);       // (nothing is cut off but what would be rounded past fp32's range)
            if constexpr (STORE == RALF_KV_E4M3) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int w = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * i], f[4 * i + 1], 0, false);
                    code[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(f[4 * i + 2], f[4 * i + 3], w, true);
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) code[i >> 2] |= ((uint32_t)(int)rintf(f[i]) & 0xffu) << (8 * (i & 3));
            }
        }
        *(u32x2*)((uint8_t*)(isv ? c.v : c.k) + row * D + e0) = code;
        if (e0 == 0) ((uint8_t*)(isv ? c.v_exp : c.k_exp))[row] = (uint8_t)ex;
    }
}

template <int D, typename T, int STORE>
__global__ __launch_bounds__(256) void write_kernel(const WriteArgs a) {
    constexpr int LANES = D / 8, RI = 64 / LANES;       // lanes of a row, rows at once
    const RalfPagedKV& c = a.c;
    const int lane = threadIdx.x & 63, e0 = (lane % LANES) * 8;
    const int64_t nw = (int64_t)gridDim.x * 4;
    for (int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); t < a.T; t += nw) {
        const Owner w = owner_of(a.q_start + 1, c.kv_len, c.B, t, lane);
        if (w.b >= c.B) continue;
        const int64_t cell = place(c, w.b, (int64_t)w.len - w.end + t);
        if (cell < 0) continue;
        // (a whole row is in or out: the exchange of its largest magnitude stays within rows.  Several rows' loads in flight at once -- 2 or 4 -- measured slower,
        //  22-24 against 17 us at 10 600 tokens of 2 x 8 x 128: the registers cost more waves than the loads gained)
        for (int r = lane / LANES; r < 2 * c.heads; r += RI) {
            const bool isv = r >= c.heads;
            const int h = isv ? r - c.heads : r;
            const T* src = isv ? (const T*)a.v + t * a.v_ts + h * a.v_hs : (const T*)a.k + t * a.k_ts + h * a.k_hs;
            const u32x4 r0 = *(const u32x4*)(src + e0);
            u32x4 r1 = r0;
            if constexpr (sizeof(T) == 4) r1 = *(const u32x4*)(src + e0 + 4);
            store_row<T, STORE, LANES, D>(c, isv, cell + (int64_t)h * c.page, e0, r0, r1);
        }
    }
}

template <int D, typename T, int STORE>
__global__ __launch_bounds__(256) void read_kernel(const ReadArgs a) {
    constexpr int LANES = D / 8, RI = 64 / LANES;
    const RalfPagedKV& c = a.c;
    const int lane = threadIdx.x & 63;
    const int64_t nw = (int64_t)gridDim.x * 4;
    for (int64_t n = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); n < a.rows; n += nw) {
        const Owner w = owner_of(a.start + 1, c.kv_len, c.B, n, lane);
        if (w.b >= c.B) continue;
        const int64_t p = n - a.start[w.b];
        const int64_t cell = p < w.len ? place(c, w.b, p) : -1;
        const int e0 = (lane % LANES) * 8;
#pragma unroll 2
        for (int r = lane / LANES; r < 2 * c.heads; r += RI) {
            const int h = r < c.heads ? r : r - c.heads;
            const bool isv = r >= c.heads;
            const int64_t row = cell + (int64_t)h * c.page;
            float f[8];
            if (cell < 0) {
#pragma unroll
                for (int i = 0; i < 8; ++i) f[i] = 0.f;
            } else if constexpr (STORE == RALF_KV_F32) {
                load8((const float*)(isv ? c.v : c.k) + row * D + e0, f);
            } else if constexpr (STORE == RALF_KV_BF16) {
                load8((const bf16*)(isv ? c.v : c.k) + row * D + e0, f);
            } else {
                const u32x2 w = *(const u32x2*)((const uint8_t*)(isv ? c.v : c.k) + row * D + e0);
                const float s = exp_value(((const uint8_t*)(isv ? c.v_exp : c.k_exp))[row]);
                float g[4];
                codes_f32<STORE>(w[0], g);
#pragma unroll
                for (int i = 0; i < 4; ++i) f[i] = g[i] * s;
                codes_f32<STORE>(w[1], g);
#pragma unroll
                for (int i = 0; i < 4; ++i) f[4 + i] = g[i] * s;
            }
            T* dst = (T*)(isv ? a.v : a.k) + (n * c.heads + h) * D + e0;
            if constexpr (sizeof(T) == 2) {
                bf16x8 o;
#pragma unroll
                for (int i = 0; i < 8; ++i) o[i] = (bf16)f[i];     // (exact for every store but fp32: rounded once)
                *(bf16x8*)dst = o;
            } else {
                *(f32x4*)dst = f32x4{f[0], f[1], f[2], f[3]};
                *(f32x4*)(dst + 4) = f32x4{f[4], f[5], f[6], f[7]};
            }
        }
    }
}

inline int blocks_for(int64_t tokens) {      // a wave per token, up to 16 waves for each of the 1024 SIMDs
    const int64_t b = (tokens + 3) / 4;
    return (int)(b > 4096 ? 4096 : b);
}

template <int D>
int write_dim(const WriteArgs& a, int dtype, void* stream) {
    const int g = blocks_for(a.T);
    hipStream_t s = (hipStream_t)stream;
    if (a.c.store == RALF_KV_F32) write_kernel<D, float, RALF_KV_F32><<<g, 256, 0, s>>>(a);
    else if (a.c.store == RALF_KV_BF16) write_kernel<D, bf16, RALF_KV_BF16><<<g, 256, 0, s>>>(a);
    else if (a.c.store == RALF_KV_E4M3) {
        if (dtype == RALF_F32) write_kernel<D, float, RALF_KV_E4M3><<<g, 256, 0, s>>>(a);
        else write_kernel<D, bf16, RALF_KV_E4M3><<<g, 256, 0, s>>>(a);
    } else {
        if (dtype == RALF_F32) write_kernel<D, float, RALF_KV_INT8><<<g, 256, 0, s>>>(a);
        else write_kernel<D, bf16, RALF_KV_INT8><<<g, 256, 0, s>>>(a);
    }
    return ralf::check_launch("paged_kv_write");
}
template <int D, typename T>
int read_dim(const ReadArgs& a, void* stream) {
    const int g = blocks_for(a.rows);
    hipStream_t s = (hipStream_t)stream;
    if (a.c.store == RALF_KV_F32) read_kernel<D, T, RALF_KV_F32><<<g, 256, 0, s>>>(a);
    else if (a.c.store == RALF_KV_BF16) read_kernel<D, T, RALF_KV_BF16><<<g, 256, 0, s>>>(a);
    else if (a.c.store == RALF_KV_E4M3) read_kernel<D, T, RALF_KV_E4M3><<<g, 256, 0, s>>>(a);
    else read_kernel<D, T, RALF_KV_INT8><<<g, 256, 0, s>>>(a);
    return ralf::check_launch("paged_kv_read");
}
}  // namespace

extern "C" int ralf_paged_kv_write(const RalfPagedKV* kv, int dtype, const void* k, const void* v, int64_t k_ts, int64_t k_hs, int64_t v_ts, int64_t v_hs,
                                   const int* q_start, int64_t T, void* stream) {
    RALF_REQUIRE(kv, "paged_kv_write: null descriptor");
    const int rc = check_kv(*kv, "paged_kv_write");
    if (rc) return rc;
    RALF_REQUIRE(dtype == RALF_F32 || dtype == RALF_BF16, "paged_kv_write: dtype %d", dtype);
    RALF_REQUIRE(kv->store >= RALF_KV_E4M3 || kv->store == (dtype == RALF_F32 ? RALF_KV_F32 : RALF_KV_BF16), "paged_kv_write: a cache of store %d takes its own type", kv->store);
    RALF_REQUIRE(T >= 0 && T < ((int64_t)1 << 31), "paged_kv_write: %lld rows", (long long)T);
    if (T == 0 || kv->B == 0 || kv->max_pages == 0 || kv->n_pages == 0) return RALF_OK;
    RALF_REQUIRE(k && v && q_start, "paged_kv_write: null pointer");
    RALF_REQUIRE(k_ts % 8 == 0 && k_hs % 8 == 0 && v_ts % 8 == 0 && v_hs % 8 == 0 && (uintptr_t)k % 16 == 0 && (uintptr_t)v % 16 == 0,
                 "paged_kv_write: rows have to start at multiples of 8 elements, 16-byte aligned");
    RALF_REQUIRE(k_ts >= 0 && k_hs >= 0 && v_ts >= 0 && v_hs >= 0, "paged_kv_write: negative stride");
    const WriteArgs a = {*kv, k, v, k_ts, k_hs, v_ts, v_hs, T, q_start};
    switch (kv->dim) {
        case 32: return write_dim<32>(a, dtype, stream);
        case 64: return write_dim<64>(a, dtype, stream);
        case 128: return write_dim<128>(a, dtype, stream);
        default: return write_dim<256>(a, dtype, stream);
    }
}

extern "C" int ralf_paged_kv_read(const RalfPagedKV* kv, int dtype, void* k, void* v, const int* start, int64_t rows, void* stream) {
    RALF_REQUIRE(kv, "paged_kv_read: null descriptor");
    const int rc = check_kv(*kv, "paged_kv_read");
    if (rc) return rc;
    RALF_REQUIRE(dtype == RALF_F32 || dtype == RALF_BF16, "paged_kv_read: dtype %d", dtype);
    RALF_REQUIRE(rows >= 0 && rows < ((int64_t)1 << 31), "paged_kv_read: %lld rows", (long long)rows);
    if (rows == 0 || kv->B == 0) return RALF_OK;
    RALF_REQUIRE(k && v && start && (uintptr_t)k % 16 == 0 && (uintptr_t)v % 16 == 0, "paged_kv_read: null or unaligned pointer");
    const ReadArgs a = {*kv, k, v, rows, start};
#define RALF_READ_DIM(D) (dtype == RALF_F32 ? read_dim<D, float>(a, stream) : read_dim<D, bf16>(a, stream))
    switch (kv->dim) {
        case 32: return RALF_READ_DIM(32);
        case 64: return RALF_READ_DIM(64);
        case 128: return RALF_READ_DIM(128);
        default: return RALF_READ_DIM(256);
    }
#undef RALF_READ_DIM
}
