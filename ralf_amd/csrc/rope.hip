// Rotary positions with several axes (ralf_rope_axes).
//
// Pair j of a head at token t turns by the angle pos[axis[j]][t] * freq[j]; the gradient of a rotation is the rotation by the opposite angle, so the
// backward pass is this kernel with `inverse`.
//   * the angle: a position of 2^31 times a frequency of 1 has no correct bit left in 32 bits once it is taken modulo 2 pi, so the product is formed in
//     double in TURNS (freq / 2 pi), the whole turns are dropped there and only the fraction (|f| <= 1/2) goes on in fp32 to sin / cos of pi * 2f.
//   * one thread owns VEC pairs of one token and walks over heads: its sines and cosines are computed once and stay in registers.
//   * bound by bytes: every element is read once and written once in 16-byte pieces.
#include "common.h"

namespace {
typedef __bf16 bf16;
template <typename T, int N> struct alignas(sizeof(T) * N) Vec { T v[N]; };

struct RopeArgs {
    RalfRopeDesc d;
    int rot, pass, hg;      // chunks of VEC pairs, chunks of VEC pass-through elements, head groups
};

template <typename T, int VEC, bool ADJ>
__global__ __launch_bounds__(256) void rope_kernel(const RopeArgs a) {
    const RalfRopeDesc& d = a.d;
    const uint32_t per = (uint32_t)(a.rot + a.pass) * a.hg;
    const int64_t gid = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t t = gid / per;
    if (t >= d.T) return;
    const uint32_t rem = (uint32_t)(gid - t * per);
    const int h0 = (int)(rem / (uint32_t)(a.rot + a.pass)), c = (int)(rem % (uint32_t)(a.rot + a.pass));
    const T* x = (const T*)d.x + t * d.x_ts;
    T* y = (T*)d.y + t * d.y_ts;
    typedef Vec<T, VEC> V;
    if (c >= a.rot) {                                   // dims behind the rotated ones
        const int o = d.R + (c - a.rot) * VEC;
        for (int h = h0; h < d.H; h += a.hg) *(V*)(y + h * d.y_hs + o) = *(const V*)(x + h * d.x_hs + o);
        return;
    }
    const int P = d.R >> 1, j0 = c * VEC;
    float cs[VEC], sn[VEC];
#pragma unroll
    for (int q = 0; q < VEC; ++q) {
        const int ax = d.axis[j0 + q];
        const bool ok = (unsigned)ax < (unsigned)d.A;
        const double turns = ok ? (double)d.pos[(int64_t)ax * d.pos_as + t] * (d.freq[j0 + q] * 0.15915494309189533577) : 0.0;
        const float f = (float)(turns - rint(turns));
        float s, co;
        sincospif(2.f * f, &s, &co);
        cs[q] = co;
        sn[q] = d.inverse ? -s : s;
    }
    const int o1 = ADJ ? 2 * j0 : j0, o2 = ADJ ? 2 * j0 + VEC : P + j0;
#pragma unroll 2
    for (int h = h0; h < d.H; h += a.hg) {
        const V u = *(const V*)(x + h * d.x_hs + o1), w = *(const V*)(x + h * d.x_hs + o2);
        V p, r;
        if (ADJ) {
            float e[2 * VEC];
#pragma unroll
            for (int q = 0; q < VEC; ++q) { e[q] = (float)u.v[q]; e[VEC + q] = (float)w.v[q]; }
            float o[2 * VEC];
#pragma unroll
            for (int q = 0; q < VEC; ++q) {
                o[2 * q] = e[2 * q] * cs[q] - e[2 * q + 1] * sn[q];
                o[2 * q + 1] = e[2 * q + 1] * cs[q] + e[2 * q] * sn[q];
            }
#pragma unroll
            for (int q = 0; q < VEC; ++q) { p.v[q] = (T)o[q]; r.v[q] = (T)o[VEC + q]; }
        } else {
#pragma unroll
            for (int q = 0; q < VEC; ++q) {
                const float m = (float)u.v[q], n = (float)w.v[q];
                p.v[q] = (T)(m * cs[q] - n * sn[q]);
                r.v[q] = (T)(n * cs[q] + m * sn[q]);
            }
        }
        *(V*)(y + h * d.y_hs + o1) = p;
        *(V*)(y + h * d.y_hs + o2) = r;
    }
}

template <typename T, int VEC>
int launch(const RalfRopeDesc& d, void* stream) {
    RopeArgs a;
    a.d = d;
    a.rot = d.R / 2 / VEC;
    a.pass = d.x == d.y ? 0 : (d.D - d.R) / VEC;
    // one head group = the angles once per token; more of them only as far as the launch would otherwise leave the card's 256 CUs short of threads
    const int64_t per = (int64_t)(a.rot + a.pass) * d.T;
    const int64_t want = ((int64_t)1 << 18) / per;
    a.hg = (int)(want < 1 ? 1 : want > d.H ? d.H : want);
    const int64_t blocks = (per * a.hg + 255) / 256;
    RALF_REQUIRE(blocks < ((int64_t)1 << 31) && (int64_t)(a.rot + a.pass) * a.hg < ((int64_t)1 << 31), "rope_axes: too many elements for one launch");
    if (d.adjacent) rope_kernel<T, VEC, true><<<(int)blocks, 256, 0, (hipStream_t)stream>>>(a);
    else rope_kernel<T, VEC, false><<<(int)blocks, 256, 0, (hipStream_t)stream>>>(a);
    return ralf::check_launch("rope_axes");
}
}  // namespace

extern "C" int ralf_rope_axes(const RalfRopeDesc* dp, void* stream) {
    RALF_REQUIRE(dp, "rope_axes: null descriptor");
    const RalfRopeDesc& d = *dp;
    RALF_REQUIRE(d.dtype == RALF_F32 || d.dtype == RALF_BF16, "rope_axes: dtype %d", d.dtype);
    RALF_REQUIRE(d.T >= 0 && d.H > 0 && d.D > 0 && d.A > 0, "rope_axes: bad sizes");
    RALF_REQUIRE(d.R > 0 && d.R % 2 == 0 && d.R <= d.D, "rope_axes: %d rotated dims of %d (an even number of at most the head's is needed)", d.R, d.D);
    RALF_REQUIRE(d.x_ts >= 0 && d.x_hs >= 0 && d.y_ts >= 0 && d.y_hs >= 0 && d.pos_as >= 0, "rope_axes: negative stride");
    if (d.T == 0) return RALF_OK;
    RALF_REQUIRE(d.x && d.y && d.pos && d.freq && d.axis, "rope_axes: null pointer");
    RALF_REQUIRE((d.T == 1 || d.y_ts > 0) && (d.H == 1 || d.y_hs > 0), "rope_axes: the output's rows overlap");
    RALF_REQUIRE(d.x != d.y || (d.x_ts == d.y_ts && d.x_hs == d.y_hs), "rope_axes: in place needs one set of strides");
    const int P = d.R / 2, el = d.dtype == RALF_BF16 ? 2 : 4;
    auto fits = [&](int vec) {     // every piece a whole, aligned vector
        const uintptr_t by = (uintptr_t)vec * el;
        return P % vec == 0 && (d.D - d.R) % vec == 0 && d.x_ts % vec == 0 && d.x_hs % vec == 0 && d.y_ts % vec == 0 && d.y_hs % vec == 0 &&
               (uintptr_t)d.x % by == 0 && (uintptr_t)d.y % by == 0;
    };
    if (d.dtype == RALF_BF16) {
        if (fits(8)) return launch<bf16, 8>(d, stream);
        if (fits(4)) return launch<bf16, 4>(d, stream);
        return launch<bf16, 1>(d, stream);
    }
    if (fits(4)) return launch<float, 4>(d, stream);
    return launch<float, 1>(d, stream);
}
