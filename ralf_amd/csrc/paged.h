// What the paged-cache kernels share: finding the sequence of a token, and the two 8-bit stores.
#pragma once
#include "common.h"

namespace paged {
typedef __bf16 bf16;
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// how many of key(0) .. key(n-1), ascending, are <= at.  One wave, all lanes active, `at` the same in all: 64 probes at once, so up to 64 sequences cost one load
// and up to 4096 two (a bisection would be 6 and 12 dependent ones).  Within [0, n] whatever the keys are.
template <class F>
__device__ __forceinline__ int count_le(F key, int n, int64_t at, int lane) {
    int base = 0;
    while (n > 64) {
        const int step = (n + 63) >> 6, i = (lane + 1) * step - 1;
        const bool below = i < n && key(base + (i < n ? i : 0)) <= at;
        const int c = __popcll(__ballot(below));
        base += c * step;
        n = n - c * step < step ? n - c * step : step;
    }
    const bool below = lane < n && key(base + (lane < n ? lane : 0)) <= at;
    return base + __popcll(__ballot(below));
}

// The sequence b of row t (ends: start + 1, so that rows ends[b - 1] .. ends[b] - 1 are b's; b = B behind the last), ends[b] and kv_len[b], the same in all lanes.
// Up to 64 sequences: one lane to each, everything in one trip to memory.
struct Owner { int b, end, len; };
__device__ __forceinline__ Owner owner_of(const int* ends, const int* kv_len, int B, int64_t t, int lane) {
    Owner o;
    if (B <= 64) {
        const int i = lane < B ? lane : B - 1, e = ends[i], n = kv_len[i];
        o.b = __popcll(__ballot(lane < B && e <= t));
        const int at = o.b < B ? o.b : B - 1;
        o.end = __builtin_amdgcn_readlane(e, at);
        o.len = __builtin_amdgcn_readlane(n, at);
    } else {
        o.b = count_le([&](int i) { return (int64_t)ends[i]; }, B, t, lane);
        const int at = o.b < B ? o.b : B - 1;
        o.end = ends[at];
        o.len = kv_len[at];
    }
    return o;
}

// the exponent byte of a row whose largest magnitude has the bits u: 127 + e, e the smallest integer with max <= LARGEST * 2^e and at least -100;
// 255 if the row holds an infinity or a NaN (their bits are the largest)
template <int STORE>
__device__ __forceinline__ uint32_t exp_byte(uint32_t u) {
    // 448 = 1.75 * 2^8, 127 = 1.984375 * 2^6
    const int e = (int)(u >> 23) - (STORE == RALF_KV_E4M3 ? 8 : 6) + ((u & 0x7fffffu) > (STORE == RALF_KV_E4M3 ? 0x600000u : 0x7e0000u) ? 1 : 0);
    return u >= 0x7f800000u ? 255u : (uint32_t)(e < 27 ? 27 : e);
}
// the largest code of such a row whose value fp32 holds: at the exponents of fp32's largest numbers the next code, 256 (64), would be 2^128
template <int STORE>
__device__ __forceinline__ float largest_code(uint32_t byte) {
    return STORE == RALF_KV_E4M3 ? (byte == 247u ? 240.f : 448.f) : (byte == 249u ? 63.f : 127.f);
}
__device__ __forceinline__ float exp_value(uint32_t byte) { return __builtin_bit_cast(float, byte << 23); }            // 2^(byte - 127); 255 gives inf (0 * inf = NaN)
__device__ __forceinline__ float exp_inverse(uint32_t byte) { return __builtin_bit_cast(float, (254u - byte) << 23); }  // 2^(127 - byte), byte in [1, 253]

// 4 codes of a dword -> fp32, exact
template <int STORE>
__device__ __forceinline__ void codes_f32(uint32_t w, float (&f)[4]) {
    if constexpr (STORE == RALF_KV_E4M3) {
        const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
        f[0] = a[0]; f[1] = a[1]; f[2] = b[0]; f[3] = b[1];
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = (float)(int8_t)(w >> (8 * i));
    }
}
// 4 codes -> two pairs of bf16, exact (e4m3 has 4 significant bits, |int8| 7)
template <int STORE>
__device__ __forceinline__ u32x2 codes_bf16(uint32_t w) {
    if constexpr (STORE == RALF_KV_E4M3) {
        const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, true);
        return u32x2{__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b)};
    } else {
        float f[4];
        codes_f32<STORE>(w, f);
        // the low 16 bits are zero: the high halves ARE the bf16 values
        return u32x2{__builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, f[1]), __builtin_bit_cast(uint32_t, f[0]), 0x07060302u),
                     __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, f[3]), __builtin_bit_cast(uint32_t, f[2]), 0x07060302u)};
    }
}
// host: what every entry asks of the cache
inline int check_kv(const RalfPagedKV& c, const char* what) {
    RALF_REQUIRE(c.B >= 0 && c.max_pages >= 0 && c.n_pages >= 0 && c.table_ld >= 0, "%s: negative size", what);
    RALF_REQUIRE(c.page == 16 || c.page == 32 || c.page == 64 || c.page == 128 || c.page == 256, "%s: page of %d tokens not in {16, 32, 64, 128, 256}", what, c.page);
    RALF_REQUIRE(c.dim == 32 || c.dim == 64 || c.dim == 128 || c.dim == 256, "%s: head dim %d not in {32, 64, 128, 256}", what, c.dim);
    RALF_REQUIRE(c.heads > 0 && c.heads <= 65535, "%s: %d heads", what, c.heads);
    RALF_REQUIRE(c.store >= RALF_KV_F32 && c.store <= RALF_KV_INT8, "%s: store %d", what, c.store);
    RALF_REQUIRE(c.n_pages < ((int64_t)1 << 31) && (int64_t)c.max_pages * c.page < ((int64_t)1 << 31), "%s: too many pages", what);
    RALF_REQUIRE(c.B == 0 || c.max_pages == 0 || (c.table && c.table_ld >= c.max_pages), "%s: null table, or rows shorter than max_pages", what);
    RALF_REQUIRE(c.n_pages == 0 || (c.k && c.v), "%s: null cache pointer", what);
    RALF_REQUIRE(c.B == 0 || c.kv_len, "%s: null kv_len", what);
    RALF_REQUIRE(c.store < RALF_KV_E4M3 || c.n_pages == 0 || (c.k_exp && c.v_exp), "%s: an 8-bit store needs its exponents", what);
    RALF_REQUIRE((uintptr_t)c.k % 16 == 0 && (uintptr_t)c.v % 16 == 0 && (uintptr_t)c.k_exp % 4 == 0 && (uintptr_t)c.v_exp % 4 == 0, "%s: unaligned cache", what);
    return RALF_OK;
}
}  // namespace paged
