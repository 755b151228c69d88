// Penalties for repeated tokens, biases and grammar masks on logits (ralf_logits_process), in front of the token choice.
//
// A workgroup owns a tile of one row's vocabulary: it counts the row's history into LDS counters of its tile (integer LDS atomics: the order does not change
// the result; bit 31 = seen at all, the low bits = occurrences behind the prompt), then streams its logits once.  No count leaves the chip and nothing has to be
// kept between steps.  Bound by bytes: logits read and written once, the bias and the mask read once; the history is read once per TILE, from L2 behind the
// first, which is why the tile is as wide as leaves every CU workgroups.  64 rows of 130 001 fp32 logits with biases by row and 4096 tokens of history: 103 MB in 24 us
// (4.3 TB/s; 45 us with single-element loads behind the counting).
#include "common.h"
#include "rows.h"

namespace {
typedef __bf16 bf16;
constexpr int THREADS = 512;
constexpr int MAX_TILE = 8192;      // 32 KiB of counters: four workgroups, 32 waves, to a CU
// (rows of an odd vocabulary start anywhere: the vectors are of their elements' alignment, which the memory takes at full width)
template <typename T> struct Piece { static constexpr int N = 16 / sizeof(T); typedef T V __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T)))); };
typedef float F4 __attribute__((ext_vector_type(4), aligned(4)));

template <typename T>
__global__ __launch_bounds__(THREADS) void logits_kernel(const RalfLogitsDesc d, int tile, int tiles) {
    typedef typename Piece<T>::V V;
    constexpr int N = Piece<T>::N, PIECES = MAX_TILE / (THREADS * N);
    extern __shared__ uint32_t cnt[];
    const int b = blockIdx.x / tiles, v0 = (blockIdx.x % tiles) * tile;
    const int n = d.V - v0 < tile ? d.V - v0 : tile;
    const T* in = (const T*)d.logits + (int64_t)b * d.ld_in + v0;
    T* out = (T*)d.out + (int64_t)b * d.ld_out + v0;
    const float* bias = d.bias ? d.bias + (int64_t)b * d.bias_ld + v0 : nullptr;
    // all of the thread's logits and biases are on their way while the history is counted
    V x[PIECES];
    F4 bb[PIECES][N / 4];
#pragma unroll
    for (int k = 0; k < PIECES; ++k) {
        const int i = (k * THREADS + threadIdx.x) * N;
        if (i + N <= n) {
            x[k] = *(const V*)(in + i);
            if (bias)
#pragma unroll
                for (int q = 0; q < N / 4; ++q) bb[k][q] = *(const F4*)(bias + i + 4 * q);
        }
    }
    const bool hist = d.repetition || d.presence || d.frequency;
    if (hist) {
        for (int i = threadIdx.x; i < n; i += THREADS) cnt[i] = 0u;
        __syncthreads();
        int len = d.len[b];
        len = len < 0 ? 0 : len > d.L ? d.L : len;
        const int plen = d.prompt_len ? d.prompt_len[b] : 0;
        const int64_t* tok = d.tokens + (int64_t)b * d.tok_ld;
#pragma unroll 4
        for (int i = threadIdx.x; i < len; i += THREADS) {
            const int64_t v = tok[i] - v0;
            if (v >= 0 && v < n) {
                if (i >= plen) atomicAdd(&cnt[v], 1u);
                else atomicOr(&cnt[v], 0x80000000u);
            }
        }
        __syncthreads();
    }
    const float rep = d.repetition ? d.repetition[b] : 1.f, pre = d.presence ? d.presence[b] : 0.f, frq = d.frequency ? d.frequency[b] : 0.f;
    const int* mask = nullptr;
    if (d.mask) {
        const int mr = d.mask_row ? d.mask_row[b] : b;
        if (mr >= 0 && mr < d.mask_rows) mask = d.mask + (int64_t)mr * d.mask_ld + (v0 >> 5);       // (a tile starts on a word)
    }
    auto one = [&](float f, int i, float add, bool allowed) {
        if (hist) {
            const uint32_t c = cnt[i];
            if (c) {
                f = f > 0.f ? f / rep : f * rep;
                const uint32_t k = c & 0x7fffffffu;
                if (k) f = f - frq * (float)k - pre;
            }
        }
        if (bias) f += add;
        return allowed ? f : -__builtin_inff();
    };
#pragma unroll
    for (int k = 0; k < PIECES; ++k) {
        const int i = (k * THREADS + threadIdx.x) * N;
        if (i + N <= n) {
            const uint32_t word = mask ? (uint32_t)mask[i >> 5] >> (i & 31) : ~0u;
            V y;
#pragma unroll
            for (int q = 0; q < N; ++q) y[q] = (T)one((float)x[k][q], i + q, bias ? bb[k][q >> 2][q & 3] : 0.f, (word >> q) & 1u);
            *(V*)(out + i) = y;
        } else {
            for (int q = i; q < n; ++q) out[q] = (T)one((float)in[q], q, bias ? bias[q] : 0.f, mask ? ((uint32_t)mask[q >> 5] >> (q & 31)) & 1u : true);
        }
    }
}

template <typename T>
int launch(const RalfLogitsDesc& d, void* stream) {
    // the widest tile (the history is read once per tile) that leaves the 256 CUs two workgroups each
    int tiles = 512 / d.B;
    const int most = (d.V + 1023) / 1024, least = (d.V + MAX_TILE - 1) / MAX_TILE;
    tiles = tiles > most ? most : tiles;
    tiles = tiles < least ? least : tiles;
    int tile = (d.V + tiles - 1) / tiles;
    tile = (tile + 31) & ~31;
    tiles = (d.V + tile - 1) / tile;
    RALF_REQUIRE((int64_t)d.B * tiles < ((int64_t)1 << 31), "logits_process: too many rows");
    logits_kernel<T><<<d.B * tiles, THREADS, (size_t)tile * 4, (hipStream_t)stream>>>(d, tile, tiles);
    return ralf::check_launch("logits_process");
}
}  // namespace

extern "C" int ralf_logits_process(const RalfLogitsDesc* dp, void* stream) {
    RALF_REQUIRE(dp, "logits_process: null descriptor");
    const RalfLogitsDesc& d = *dp;
    RALF_REQUIRE(d.dtype == RALF_F32 || d.dtype == RALF_BF16, "logits_process: dtype %d", d.dtype);
    RALF_REQUIRE(d.B >= 0 && d.V > 0 && d.L >= 0 && d.mask_rows >= 0 && d.V < (1 << 30), "logits_process: bad sizes");
    if (d.B == 0) return RALF_OK;
    RALF_REQUIRE(d.logits && d.out && d.ld_in >= d.V && d.ld_out >= d.V, "logits_process: null logits, or rows shorter than V");
    RALF_REQUIRE(d.logits != d.out || d.ld_in == d.ld_out, "logits_process: in place needs one row stride");
    RALF_REQUIRE(d.logits == d.out || ralf::rows_disjoint({d.logits, d.ld_in, 0}, {d.out, d.ld_out, 0}, d.B, 1, d.V, d.dtype == RALF_BF16 ? 2 : 4), "logits_process: the output overlaps the logits without being them");
    if (d.repetition || d.presence || d.frequency)
        RALF_REQUIRE(d.len && (d.L == 0 || d.tokens) && d.tok_ld >= d.L, "logits_process: penalties need the history and its lengths");
    RALF_REQUIRE(!d.bias || d.bias_ld == 0 || d.bias_ld >= d.V, "logits_process: bias rows shorter than V");
    RALF_REQUIRE(!d.mask || d.mask_ld >= (d.V + 31) / 32, "logits_process: mask rows shorter than V bits");
    RALF_REQUIRE(!d.mask || d.mask_row || d.mask_rows >= d.B, "logits_process: without mask_row every row needs a mask of its own");
    return d.dtype == RALF_BF16 ? launch<bf16>(d, stream) : launch<float>(d, stream);
}
