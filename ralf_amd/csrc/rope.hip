// Rotary positions with several axes (ralf_rope_axes).
//
// Pair j of a head at token t turns by the angle pos[axis[j]][t] * freq[j]; the gradient of a rotation is the rotation by the opposite angle, so the
// backward pass is this kernel with `inverse`.
//   * the angle: a position of 2^31 times a frequency of 1 has no correct bit left in 32 bits once it is taken modulo 2 pi, so the product is formed in
//     double in TURNS (freq / 2 pi), the whole turns are dropped there and only the fraction (|f| <= 1/2) goes on in fp32 to sin / cos of pi * 2f.
//   * one thread owns 16 bytes' worth of pairs of one token and walks over heads: its sines and cosines are computed once and stay in registers.
//   * bound by bytes: every element is read once and written once in 16-byte pieces: 16384 tokens of 40 heads of 128 in bf16, 336 MB in 74 us (4.5 TB/s); heads of 134 dims
//     (rows at any element) 3.4 TB/s against 1.8 with single elements.
#include "common.h"
#include "rows.h"

namespace {
typedef __bf16 bf16;
// 16 bytes of elements, wherever they start: heads of an odd width put rows at any element, which the memory takes at full width
template <typename T> struct Piece { static constexpr int N = 16 / sizeof(T); typedef T V __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T)))); };

struct RopeArgs {
    RalfRopeDesc d;
    int rot, pass, hg;      // pieces of rotated pairs and of dims passed through, head groups
};

// a pair's turn, in fp32, rounded once
__device__ __forceinline__ void turn(float a, float b, float c, float s, float& x, float& y) {
    x = a * c - b * s;
    y = b * c + a * s;
}

template <typename T, bool ADJ>
__global__ __launch_bounds__(256) void rope_kernel(const RopeArgs a) {
    constexpr int N = Piece<T>::N;
    typedef typename Piece<T>::V V;
    typedef T V4 __attribute__((ext_vector_type(4), aligned(sizeof(T))));
    typedef T V2 __attribute__((ext_vector_type(2), aligned(sizeof(T))));
    const RalfRopeDesc& d = a.d;
    const uint32_t per = (uint32_t)(a.rot + a.pass) * a.hg;
    const int64_t gid = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t t = gid / per;
    if (t >= d.T) return;
    const uint32_t rem = (uint32_t)(gid - t * per);
    const int h0 = (int)(rem / (uint32_t)(a.rot + a.pass)), c = (int)(rem % (uint32_t)(a.rot + a.pass));
    const T* x = (const T*)d.x + t * d.x_ts;
    T* y = (T*)d.y + t * d.y_ts;
    if (c >= a.rot) {                                   // dims behind the rotated ones
        const int o = d.R + (c - a.rot) * N;
        for (int h = h0; h < d.H; h += a.hg) {
            if (o + N <= d.D) *(V*)(y + h * d.y_hs + o) = *(const V*)(x + h * d.x_hs + o);
            else {                                      // fewer than a piece: by halves of one
                const T* xh = x + h * d.x_hs;
                T* yh = y + h * d.y_hs;
                int i = o;
                if (d.D - i >= 4) { *(V4*)(yh + i) = *(const V4*)(xh + i); i += 4; }
                if (d.D - i >= 2) { *(V2*)(yh + i) = *(const V2*)(xh + i); i += 2; }
                if (d.D - i >= 1) yh[i] = xh[i];
            }
        }
        return;
    }
    const int P = d.R >> 1, j0 = c * N, n = P - j0 < N ? P - j0 : N;
    float cs[N], sn[N];
    uint32_t stay = 0u;                                 // bit q: the pair's axis has no positions, its elements are copied (1 * a - 0 * b would carry b's infinities and NaN to a)
#pragma unroll
    for (int q = 0; q < N; ++q) {
        if (q >= n) { cs[q] = 1.f; sn[q] = 0.f; continue; }
        const int ax = d.axis[j0 + q];
        const bool ok = (unsigned)ax < (unsigned)d.A;
        stay |= (ok ? 0u : 1u) << q;
        const double turns = ok ? (double)d.pos[(int64_t)ax * d.pos_as + t] * (d.freq[j0 + q] * 0.15915494309189533577) : 0.0;
        const float f = (float)(turns - rint(turns));
        float s, co;
        sincospif(2.f * f, &s, &co);
        cs[q] = co;
        sn[q] = d.inverse ? -s : s;
    }
    const int o1 = ADJ ? 2 * j0 : j0, o2 = ADJ ? 2 * j0 + N : P + j0;
    if (n == N) {
#pragma unroll 2
        for (int h = h0; h < d.H; h += a.hg) {
            const V u = *(const V*)(x + h * d.x_hs + o1), w = *(const V*)(x + h * d.x_hs + o2);
            V p, r;
#pragma unroll
            for (int q = 0; q < N; ++q) {
                float e, f;
                if constexpr (ADJ) {
                    // pair q: elements 2 q, 2 q + 1 of the two pieces one behind the other
                    turn((float)(q < N / 2 ? u[2 * q % N] : w[2 * q % N]), (float)(q < N / 2 ? u[2 * q % N + 1] : w[2 * q % N + 1]), cs[q], sn[q], e, f);
                    if (q < N / 2) { p[2 * q % N] = (T)e; p[2 * q % N + 1] = (T)f; }
                    else { r[2 * q % N] = (T)e; r[2 * q % N + 1] = (T)f; }
                } else {
                    turn((float)u[q], (float)w[q], cs[q], sn[q], e, f);
                    p[q] = (T)e;
                    r[q] = (T)f;
                }
            }
            if (stay) {
#pragma unroll
                for (int q = 0; q < N; ++q) {           // element q of the two pieces: of pairs q / 2 and (q + N) / 2 where pairs are adjacent
                    p[q] = (stay >> (ADJ ? q / 2 : q)) & 1u ? u[q] : p[q];
                    r[q] = (stay >> (ADJ ? (q + N) / 2 : q)) & 1u ? w[q] : r[q];
                }
            }
            *(V*)(y + h * d.y_hs + o1) = p;
            *(V*)(y + h * d.y_hs + o2) = r;
        }
    } else {                                            // the last pairs of a number that is no multiple of a piece
        for (int h = h0; h < d.H; h += a.hg) {
            const T* xh = x + h * d.x_hs;
            T* yh = y + h * d.y_hs;
#pragma unroll
            for (int q = 0; q < N; ++q) {
                if (q >= n) continue;
                const int i1 = ADJ ? 2 * (j0 + q) : j0 + q, i2 = ADJ ? i1 + 1 : P + j0 + q;
                float e, f;
                const T u = xh[i1], w = xh[i2];
                const bool keep = (stay >> q) & 1u;
                turn((float)u, (float)w, cs[q], sn[q], e, f);
                yh[i1] = keep ? u : (T)e;
                yh[i2] = keep ? w : (T)f;
            }
        }
    }
}

template <typename T>
int launch(const RalfRopeDesc& d, void* stream) {
    RopeArgs a;
    a.d = d;
    const int n = Piece<T>::N;
    a.rot = (d.R / 2 + n - 1) / n;
    a.pass = d.x == d.y ? 0 : (d.D - d.R + n - 1) / n;
    // one head group = the angles once per token; more of them only as far as the launch would otherwise leave the card's 256 CUs short of threads
    const ralf::wide per = (ralf::wide)(a.rot + a.pass) * d.T;
    const int64_t want = (int64_t)(((int64_t)1 << 18) / per);
    a.hg = (int)(want < 1 ? 1 : want > d.H ? d.H : want);
    const ralf::wide blocks = (per * a.hg + 255) / 256;
    RALF_REQUIRE(blocks < ((int64_t)1 << 31) && (int64_t)(a.rot + a.pass) * a.hg < ((int64_t)1 << 31), "rope_axes: too many elements for one launch");
    RALF_REQUIRE(d.x == d.y || ralf::rows_disjoint({d.x, d.x_ts, d.x_hs}, {d.y, d.y_ts, d.y_hs}, d.T, d.H, d.D, sizeof(T)), "rope_axes: the output overlaps x without being x");
    if (d.adjacent) rope_kernel<T, true><<<(int)blocks, 256, 0, (hipStream_t)stream>>>(a);
    else rope_kernel<T, false><<<(int)blocks, 256, 0, (hipStream_t)stream>>>(a);
    return ralf::check_launch("rope_axes");
}
}  // namespace

extern "C" int ralf_rope_axes(const RalfRopeDesc* dp, void* stream) {
    RALF_REQUIRE(dp, "rope_axes: null descriptor");
    const RalfRopeDesc& d = *dp;
    RALF_REQUIRE(d.dtype == RALF_F32 || d.dtype == RALF_BF16, "rope_axes: dtype %d", d.dtype);
    RALF_REQUIRE(d.T >= 0 && d.H > 0 && d.D > 0 && d.D < (1 << 30) && d.A > 0, "rope_axes: bad sizes");
    RALF_REQUIRE(d.R > 0 && d.R % 2 == 0 && d.R <= d.D, "rope_axes: %d rotated dims of %d (an even number of at most the head's is needed)", d.R, d.D);
    RALF_REQUIRE(d.x_ts >= 0 && d.x_hs >= 0 && d.y_ts >= 0 && d.y_hs >= 0 && d.pos_as >= 0, "rope_axes: negative stride");
    if (d.T == 0) return RALF_OK;
    RALF_REQUIRE(d.x && d.y && d.pos && d.freq && d.axis, "rope_axes: null pointer");
    RALF_REQUIRE(ralf::rows_apart(d.T, d.y_ts, d.H, d.y_hs, d.D), "rope_axes: the output's rows overlap");
    RALF_REQUIRE(d.x != d.y || (d.x_ts == d.y_ts && d.x_hs == d.y_hs), "rope_axes: in place needs one set of strides");
    return d.dtype == RALF_BF16 ? launch<bf16>(d, stream) : launch<float>(d, stream);
}
