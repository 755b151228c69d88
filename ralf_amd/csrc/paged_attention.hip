// Attention of each sequence's newest tokens over the paged cache (ralf_paged_attention).
//
// Rows and tiles.  The q_heads / heads = G query heads that share a key head are rows of one product: row r of sequence b under key head hk is token r / G,
// query head hk * G + r % G.  A tile is BM consecutive rows; it sees the keys up to its last row's position.
//
// Products, transposed so that a lane owns one row (lane & 15) throughout: S^T[key][row] = K Q^T, then O^T[dim][row] = V^T P^T.  The accumulators of the first
// are the operand of the second as they stand (the matrix instruction's contraction slots are named after the keys the lane holds), row maxima need
// two exchanges (lanes 16 and 32 apart), and every rescaling is lane-local.
//   bf16: v_mfma_f32_16x16x32_bf16, keys and values rounded to bf16 already (8-bit codes are exact in it, their powers of two go to the scores and the
//         probabilities in fp32).  few_kernel takes a probability as two bf16 parts (2^-16 of it left out), so that a result is off by its own rounding alone: up to
//         8 % of the time at dims 32 and 64 and where 8-bit codes are unpacked, nothing where bytes bound it.  many_kernel rounds it to one (half a step: 2^-8; the sum is taken in fp32
//         before that rounding): two parts are half as many matrix instructions again and took 429 us against 320 (2048 new on 8192 cached tokens, 32 / 8 heads of 128),
//         for results that are off by 0.0017 (their own rounding to bf16) instead of 0.0023 of their size.
//   fp32: v_mfma_f32_16x16x4_f32 on an fp32 cache; on 8-bit codes three bf16 products, the query and the probabilities in three bf16 parts (split3).
// Running maximum and sum of the softmax in fp32; exponentials base 2 with log2(e) folded into the scale.
//
// Masks.  A row that has seen no key keeps max = -inf, sum = 0 and gives zeros.  Values behind kv_len and on bad pages count as zeros; a later
// token's or an out-of-window value that is an infinity or a NaN must not reach a row through 0 * inf: such values are taken out of the products of partly visible
// blocks and added, behind the loop, to the rows that see them.
#include "paged.h"
#include "rows.h"

namespace {
using namespace paged;

constexpr int MAX_SPLITS = 128;
constexpr float LOG2E = 1.4426950408889634f;
// The reference of the exponentials (log2 units) stays so far above the row's largest score that weights are at most 1, 2^-8 as a rule: 256 keys of equal weight may hold fp32's
// largest number before an unnormalised sum leaves its range.  (More of it would take as much from the other end: sums of values below 2^-118 already leave the normal range.)
constexpr float HEADROOM = 8.f;

// What a kernel leaves of rows whose keys it cuts into several pieces (splits > 1): o [splits][rows][dim] unnormalised, ml [splits][rows][2] reference (log2 units) and sum
struct Part {
    float* o;
    float* ml;
    int64_t rows;       // row t * q_heads + h of all T * q_heads; or `slots`, of few_kernel beside many_kernel where that is fewer:
    int splits;
    bool slots;         // row (b * few_rows + r) * heads + hk of all B * few_rows * heads, r of sequence b under key head hk
    __host__ __device__ size_t bytes(int dim) const { return splits > 1 ? (size_t)splits * rows * (dim + 2) * sizeof(float) : 0; }
};
struct Args {
    RalfPagedAttnDesc d;
    int G, page_log2;
    int few_rows;       // sequences of at most so many rows go to few_kernel, the others to many_kernel
    int few_tiles;      // tiles of a sequence in few_kernel's grid where few_rows bounds them; 0: found from q_start
    float qscale;       // scale * log2(e)
    Part few, many;
};

__device__ __forceinline__ float exp2f_(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float sum4(float v) { v += __shfl_xor(v, 16); return v + __shfl_xor(v, 32); }

struct Tile { int b, tok0, row0, rows, first, L; bool ok; };  // sequence, its first token's row of q, first row, its rows, the position of its first new token, its keys

// the first key that a row at position pos sees
__device__ __forceinline__ int behind(int pos, int window) {
    const int64_t k = window > 0 ? (int64_t)pos - window + 1 : 0;
    return k < 0 ? 0 : (int)k;
}

// tile w of BM rows: sequence b's tiles start at q_start[b] * G / BM + b, which leaves every sequence room for ceil(n * G / BM) of them
template <int BM>
__device__ __forceinline__ Tile find_tile(const Args& a, int w, int lane, int per_seq) {
    Tile t;
    const int B = a.d.kv.B, G = a.G;
    t.ok = false;
    int64_t s, e0, L;
    if (B <= 64 && !per_seq) {          // one lane to a sequence: everything in one trip to memory
        const int i = lane < B ? lane : B - 1;
        const int s_ = a.d.q_start[i], e_ = a.d.q_start[i + 1], l_ = a.d.kv.kv_len[i];
        t.b = __popcll(__ballot(lane < B && (int64_t)s_ * G / BM + lane <= w)) - 1;
        if (t.b < 0) return t;
        s = __builtin_amdgcn_readlane(s_, t.b);
        e0 = __builtin_amdgcn_readlane(e_, t.b);
        L = __builtin_amdgcn_readlane(l_, t.b);
    } else {
        t.b = per_seq ? w / per_seq : count_le([&](int i) { return (int64_t)a.d.q_start[i] * G / BM + i; }, B, w, lane) - 1;
        if (t.b < 0) return t;
        s = a.d.q_start[t.b];
        e0 = a.d.q_start[t.b + 1];
        L = a.d.kv.kv_len[t.b];
    }
    const int64_t e = e0 < a.d.T ? e0 : a.d.T;
    if (s < 0 || e <= s) return t;
    const int64_t row0 = (per_seq ? w % per_seq : w - (s * G / BM + t.b)) * BM, rows = (e - s) * G;
    if (row0 >= rows) return t;
    t.row0 = (int)row0;
    t.rows = (int)rows;
    const int64_t most = (int64_t)a.d.kv.max_pages * a.d.kv.page;
    t.L = (int)(L < most ? L : most);
    t.first = (int)(L - (e0 - s));
    t.tok0 = (int)s;
    t.ok = true;
    return t;
}

// ------------------------------------------------------------------------------------------------
// few rows: 16 to a workgroup, its 4 waves take blocks of 32 or 64 keys in turn (a long axis and few rows: the keys are what there is to divide).
// K and V go from memory straight into registers, each byte once per 16 rows; a block's loads are issued a block ahead of its products and its pages looked up
// two ahead, which keeps 60 - 130 KB in flight to a CU.  Bound by bytes: 64 sequences of 2048 - 8192 tokens, 8 key heads of 128: e4m3 684 MB in 153 us (4.5 TB/s; without
// the loads ahead 450 us), bf16 4.8 TB/s (282 us); a copy reaches 4.9 on this card.
// ------------------------------------------------------------------------------------------------
// The shapes of a lane's share of a block of NT sixteens of keys.  Of a key row it holds EPL consecutive elements (16 bytes) of every 4 EPL -- the contraction over
// dims may run in any order, as long as the query's registers follow the same one -- and of four value rows of each sixteen CPL columns.
template <int D, int STORE, bool F32>
struct Few {
    static constexpr int ESZ = STORE == RALF_KV_F32 ? 4 : STORE == RALF_KV_BF16 ? 2 : 1;
    static constexpr int CPL = D / 16;
    static constexpr int EPL = 16 / ESZ > D / 4 ? D / 4 : 16 / ESZ;
    static constexpr int NK = D / 4 / EPL;                          // loads of a key row
    static constexpr int KW = EPL * ESZ / 4;                        // dwords of each
    static constexpr int VW = CPL * ESZ < 4 ? 1 : CPL * ESZ / 4;    // dwords of a value row's columns
    // keys of a block: enough bytes in flight with two blocks' registers (loaded one ahead) in 256, the scores' exchanges paid for many keys
    static constexpr bool FP32 = STORE == RALF_KV_F32;              // fp32 products; otherwise bf16 ones, of fp32 queries in three parts
    static constexpr int PARTS = F32 && !FP32 ? 3 : 1;
    static constexpr int WPARTS = F32 && !FP32 ? 3 : 2;             // of the weights: split2 leaves 2^-16 of one, so that a bf16 result is off by its own rounding alone
    static constexpr int NT = FP32 ? (D * ESZ >= 512 ? 1 : 2) : (D * ESZ >= 128 ? 2 : 4);
    static constexpr int REGS = NT * (NK * KW + 4 * VW);
    static constexpr bool TWO = REGS <= 80;                         // two blocks' registers
    static constexpr int WAVES = TWO && D < 256 ? 2 : 1;            // waves to a SIMD that the registers have to leave room for
};

template <int W>
__device__ __forceinline__ void load_words(const uint8_t* p, uint32_t (&w)[W], int bytes) {
    if constexpr (W >= 4) {
#pragma unroll
        for (int i = 0; i < W / 4; ++i) {
            const u32x4 v = ((const u32x4*)p)[i];
#pragma unroll
            for (int j = 0; j < 4; ++j) w[4 * i + j] = v[j];
        }
    } else if constexpr (W == 2) {
        const u32x2 v = *(const u32x2*)p;
        w[0] = v[0]; w[1] = v[1];
    } else {
        w[0] = bytes == 4 ? *(const uint32_t*)p : *(const uint16_t*)p;
    }
}

// does a dword of values hold an infinity or a NaN; the dword without them
template <int STORE>
__device__ __forceinline__ bool odd_word(uint32_t w) {
    if constexpr (STORE == RALF_KV_F32) return (w & 0x7f800000u) == 0x7f800000u;
    else if constexpr (STORE == RALF_KV_BF16) return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u;
    else if constexpr (STORE == RALF_KV_E4M3) return (w & 0x7fu) == 0x7fu || (w & 0x7f00u) == 0x7f00u || (w & 0x7f0000u) == 0x7f0000u || (w & 0x7f000000u) == 0x7f000000u;
    else return false;
}
template <int STORE>
__device__ __forceinline__ uint32_t finite_word(uint32_t w) {
    if constexpr (STORE == RALF_KV_F32) return odd_word<STORE>(w) ? 0u : w;
    else if constexpr (STORE == RALF_KV_BF16) return ((w & 0x7f80u) == 0x7f80u ? 0u : w & 0xffffu) | ((w & 0x7f800000u) == 0x7f800000u ? 0u : w & 0xffff0000u);
    else {
        uint32_t r = 0u;
        for (int i = 0; i < 4; ++i) r |= ((w >> (8 * i)) & 0x7fu) == 0x7fu ? 0u : w & (0xffu << (8 * i));
        return r;
    }
}
// element i of a row of values: itself if it is an infinity or a NaN, else 0
template <int STORE>
__device__ __forceinline__ float odd_value(const uint8_t* row, int i) {
    float x;
    if constexpr (STORE == RALF_KV_F32) x = ((const float*)row)[i];
    else if constexpr (STORE == RALF_KV_BF16) x = __uint_as_float((uint32_t)((const uint16_t*)row)[i] << 16);
    else x = (row[i] & 0x7fu) == 0x7fu ? __builtin_nanf("") : 0.f;
    return fabsf(x) < __builtin_inff() ? 0.f : x;
}

// Eight fp32 values as sums of three bf16 ones, by cutting off: 8 + 8 + 8 significant bits, so nothing is left out (but what falls below the smallest number).  An
// 8-bit code is exact in bf16, so three bf16 products of 16 cycles each stand for the fp32 product of 32 dims that takes the fp32 instruction 256.
__device__ __forceinline__ void split3(const float* f, bf16x8 (&part)[3]) {
    uint32_t w[3][8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        w[0][i] = __float_as_uint(f[i]) & 0xffff0000u;
        const float a = __uint_as_float(w[0][i]);
        const float r1 = fabsf(a) < __builtin_inff() ? f[i] - a : f[i] != f[i] ? f[i] : 0.f;
        w[1][i] = __float_as_uint(r1) & 0xffff0000u;
        w[2][i] = __float_as_uint(r1 - __uint_as_float(w[1][i]));
    }
#pragma unroll
    for (int x = 0; x < 3; ++x) {
        u32x4 v;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = __builtin_amdgcn_perm(w[x][2 * i + 1], w[x][2 * i], 0x07060302u);
        part[x] = __builtin_bit_cast(bf16x8, v);
    }
}

// Eight weights as sums of two bf16 values, 2^-16 of a weight left out.
//   INF (values that may be infinite: weight times infinity has to be infinity in both parts): the first part by cutting off, so that the rest is not negative, and 2^-22 of the weight
//     more than the rest, so that it is zero only where the weight is.
//   otherwise (8-bit codes; their NaN is NaN for any weight): both parts rounded to nearest.
// On bf16 caches of dims 32 and 64 the first form also holds few_kernel to 128 registers, four waves to a SIMD (134 with the conversion: 64 sequences with 12 new on 2048 keys at
// dim 32 34 us, 30 so); on 8-bit ones of dim 32 it is the second that leaves a wave more (163 registers against 171: 46 us against 50).
template <bool INF>
__device__ __forceinline__ void split2(const float* f, bf16x8 (&part)[2]) {
    u32x4 hi, lo;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float x = f[2 * i], y = f[2 * i + 1];
        bf16x2 rest;
        if constexpr (INF) {
            constexpr float MORE = 1.f + 0x1p-22f;
            hi[i] = __builtin_amdgcn_perm(__float_as_uint(y), __float_as_uint(x), 0x07060302u);
            rest = bf16x2{(bf16)fmaf(x, MORE, -__uint_as_float(__float_as_uint(x) & 0xffff0000u)), (bf16)fmaf(y, MORE, -__uint_as_float(__float_as_uint(y) & 0xffff0000u))};
        } else {
            const bf16x2 h = {(bf16)x, (bf16)y};
            hi[i] = __builtin_bit_cast(uint32_t, h);
            rest = bf16x2{(bf16)(x - (float)h[0]), (bf16)(y - (float)h[1])};
        }
        lo[i] = __builtin_bit_cast(uint32_t, rest);
    }
    part[0] = __builtin_bit_cast(bf16x8, hi);
    part[1] = __builtin_bit_cast(bf16x8, lo);
}

template <int D, int STORE, bool F32>
struct FewBuf {
    typedef Few<D, STORE, F32> S;
    uint32_t k[S::NT][S::NK][S::KW], v[4 * S::NT][S::VW], ke[S::NT], ve[S::NT];
    uint32_t bad;           // bit s: the block's sixteen s is not there (behind the end, or on a bad page)
};

template <int D, int STORE, bool F32>
__global__ __launch_bounds__(256, (Few<D, STORE, F32>::WAVES)) void few_kernel(const Args a) {
    typedef Few<D, STORE, F32> S;
    typedef FewBuf<D, STORE, F32> Buf;
    constexpr int BM = 16, NT = S::NT, KB = 16 * NT, CPL = S::CPL, ESZ = S::ESZ;
    extern __shared__ float sm[];                       // [4][16][D]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r16 = lane & 15, kg = lane >> 4;
    const RalfPagedKV& c = a.d.kv;
    const int split = blockIdx.x % a.few.splits;
    const int hk = (blockIdx.x / a.few.splits) % c.heads;
    const Tile t = find_tile<BM>(a, blockIdx.x / a.few.splits / c.heads, lane, a.few_tiles);
    if (!t.ok || t.rows > a.few_rows) return;
    const int64_t tok0 = t.tok0;
    const int row = t.row0 + r16;
    const bool live = row < t.rows;
    const int ti = (live ? row : t.row0) / a.G, hq = hk * a.G + (live ? row : t.row0) % a.G;
    // the keys this lane's row sees: lo .. hi
    const int pos = t.first + ti;
    const int hi = !live ? -1 : a.d.causal && pos < t.L - 1 ? pos : t.L - 1;
    const int lo = behind(pos, a.d.window);
    // the tile's keys: positions grow with the row
    const int last = (t.row0 + BM < t.rows ? t.row0 + BM : t.rows) - 1;
    const int p0 = t.first + t.row0 / a.G, p1 = t.first + last / a.G;
    const int kbeg = behind(p0, a.d.window), kend = a.d.causal && p1 < t.L ? p1 + 1 : t.L;
    const int full_lo = behind(p1, a.d.window), full_hi = a.d.causal && p0 < t.L - 1 ? p0 : t.L - 1;   // keys that every row of the tile sees
    // this split's blocks of KB keys
    const int blk0 = kbeg / KB, nblk = kend > kbeg ? (kend + KB - 1) / KB - blk0 : 0;
    const int per = (nblk + a.few.splits - 1) / a.few.splits;
    const int sb = blk0 + split * per, se = sb + per < blk0 + nblk ? sb + per : blk0 + nblk;

    const int64_t qoff = (tok0 + ti) * a.d.q_ts + hq * a.d.q_hs;
    float qf[S::FP32 ? D / 4 : 1];
    u32x4 qb[S::PARTS][S::FP32 ? 1 : D / 32];
#pragma unroll
    for (int j = 0; j < S::NK; ++j) {
        const int64_t at = qoff + (4 * j + kg) * S::EPL;
        if constexpr (F32) {
            float f[S::EPL];
#pragma unroll
            for (int i = 0; i < S::EPL / 4; ++i) {
                const f32x4 v = live ? *(const f32x4*)((const float*)a.d.q + at + 4 * i) : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int q = 0; q < 4; ++q) f[4 * i + q] = v[q];
            }
            if constexpr (S::FP32) {
#pragma unroll
                for (int i = 0; i < S::EPL; ++i) qf[j * S::EPL + i] = f[i];
            } else {
#pragma unroll
                for (int i = 0; i < S::EPL / 8; ++i) {
                    bf16x8 part[3];
                    split3(&f[8 * i], part);
#pragma unroll
                    for (int x = 0; x < 3; ++x) qb[x][j * (S::EPL / 8) + i] = __builtin_bit_cast(u32x4, part[x]);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < S::EPL / 8; ++i) qb[0][j * (S::EPL / 8) + i] = live ? *(const u32x4*)((const bf16*)a.d.q + at + 8 * i) : u32x4{0u, 0u, 0u, 0u};
        }
    }

    f32x4 acc[CPL];
#pragma unroll
    for (int i = 0; i < CPL; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = -__builtin_inff(), l = 0.f;
    const int* table = c.table + (int64_t)t.b * c.table_ld;
    const int64_t head_rows = (int64_t)c.heads * c.page;
    const uint8_t* kbase = (const uint8_t*)c.k + ((int64_t)hk * c.page + r16) * (D * ESZ) + kg * (S::EPL * ESZ);
    const uint8_t* vbase = (const uint8_t*)c.v + ((int64_t)hk * c.page + 4 * kg) * (D * ESZ) + r16 * (CPL * ESZ);
    const uint8_t* kebase = (const uint8_t*)c.k_exp + (int64_t)hk * c.page + 4 * kg;
    const uint8_t* vebase = (const uint8_t*)c.v_exp + (int64_t)hk * c.page + 4 * kg;

    int pages[NT];          // looked up one block ahead of their loads: the loads' addresses wait for nothing
    auto look = [&](int blk) {
#pragma unroll
        for (int s = 0; s < NT; ++s) {
            const int k0 = blk * KB + 16 * s;
            pages[s] = blk < se && k0 < t.L ? table[k0 >> a.page_log2] : -1;
        }
    };
    auto load = [&](Buf& w, int blk) {
        w.bad = 0u;
#pragma unroll
        for (int s = 0; s < NT; ++s) {
            const bool ok = pages[s] >= 0 && pages[s] < c.n_pages;
            w.bad |= (ok ? 0u : 1u) << s;
            // (a sixteen that is not there is read from page 0 and left out afterwards)
            const int64_t row0 = (ok ? pages[s] : 0) * head_rows + ((blk * KB + 16 * s) & (c.page - 1));
            const uint8_t* kp = kbase + row0 * (D * ESZ);
            const uint8_t* vp = vbase + row0 * (D * ESZ);
#pragma unroll
            for (int j = 0; j < S::NK; ++j) load_words<S::KW>(kp + j * (4 * S::EPL * ESZ), w.k[s][j], S::KW * 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) load_words<S::VW>(vp + i * (D * ESZ), w.v[4 * s + i], CPL * ESZ);
            if constexpr (STORE >= RALF_KV_E4M3) {
                w.ke[s] = *(const uint32_t*)(kebase + row0);
                w.ve[s] = *(const uint32_t*)(vebase + row0);
            }
        }
    };
    auto is_mixed = [&](int blk, uint32_t bad) { return blk * KB < full_lo || blk * KB + KB - 1 > full_hi || bad; };   // some row does not see some key of the block
    bool odd = false;
    auto compute = [&](Buf& w, int blk) {
        const int key0 = blk * KB;
        float p[4 * NT];
#pragma unroll
        for (int s = 0; s < NT; ++s) {
            f32x4 st = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < S::NK; ++j) {
                if constexpr (S::FP32) {
#pragma unroll
                    for (int x = 0; x < S::KW; ++x) st = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(w.k[s][j][x]), qf[j * S::EPL + x], st, 0, 0, 0);
                } else {
#pragma unroll
                    for (int x = 0; x < S::EPL / 8; ++x) {
                        u32x4 kv;
                        if constexpr (STORE == RALF_KV_BF16) kv = u32x4{w.k[s][j][0], w.k[s][j][1], w.k[s][j][2], w.k[s][j][3]};
                        else {
                            const u32x2 u = codes_bf16<STORE>(w.k[s][j][2 * x]), v = codes_bf16<STORE>(w.k[s][j][2 * x + 1]);
                            kv = u32x4{u[0], u[1], v[0], v[1]};
                        }
#pragma unroll
                        for (int y = S::PARTS - 1; y >= 0; --y)
                            st = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, kv), __builtin_bit_cast(bf16x8, qb[y][j * (S::EPL / 8) + x]), st, 0, 0, 0);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float x = st[i] * a.qscale;
                if constexpr (STORE >= RALF_KV_E4M3) x *= exp_value((w.ke[s] >> (8 * i)) & 0xffu);
                p[4 * s + i] = x;
            }
        }
        const bool mixed = is_mixed(blk, w.bad);
        uint32_t seen = ~0u;        // bit 4 s + i: the row sees that key
        if (mixed) {
            seen = 0u;
#pragma unroll
            for (int s = 0; s < NT; ++s)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int key = key0 + 16 * s + 4 * kg + i;
                    const bool see = key >= lo && key <= hi && !((w.bad >> s) & 1u);
                    seen |= (see ? 1u : 0u) << (4 * s + i);
                    p[4 * s + i] = see ? p[4 * s + i] : -__builtin_inff();
                    if (key >= t.L || ((w.bad >> s) & 1u)) {        // nobody's values
#pragma unroll
                        for (int q = 0; q < S::VW; ++q) w.v[4 * s + i][q] = 0u;
                    }
                }
        }
        // running maximum and sum
        float mx = p[0];
#pragma unroll
        for (int i = 1; i < 4 * NT; ++i) mx = fmaxf(mx, p[i]);
        mx = fmaxf(m, wave::max_x16_x32(mx) + HEADROOM);
        const float base = mx == -__builtin_inff() ? 0.f : mx;
        if (__any(mx > m)) {
            const float alpha = exp2f_(m - base);          // (m = -inf: 0)
            l *= alpha;
            m = mx;
#pragma unroll
            for (int i = 0; i < CPL; ++i) acc[i] *= alpha;
        }
        float sum = 0.f;                                    // (this lane's keys only: summed over the four lane groups at the end)
#pragma unroll
        for (int i = 0; i < 4 * NT; ++i) { p[i] = exp2f_(p[i] - base); sum += p[i]; }
        l += sum;
        if constexpr (STORE >= RALF_KV_E4M3) {
#pragma unroll
            for (int i = 0; i < 4 * NT; ++i) {
                const float e = exp_value((w.ve[i >> 2] >> (8 * (i & 3))) & 0xffu);
                p[i] = (seen >> i) & 1u ? p[i] * e : 0.f;       // (a hidden row's exponent may stand for NaN)
            }
        }
        // A hidden value that is an infinity or a NaN would reach the rows that do not see it as 0 * inf: such values are taken out of the product (and given to the
        // rows that do see them when the loop is done)
        if (STORE != RALF_KV_INT8 && mixed) {
            bool any = false;
#pragma unroll
            for (int e = 0; e < 4 * NT; ++e)
#pragma unroll
                for (int q = 0; q < S::VW; ++q) any |= odd_word<STORE>(w.v[e][q]);
            if (__any(any)) {
                odd = true;
#pragma unroll
                for (int e = 0; e < 4 * NT; ++e)
#pragma unroll
                    for (int q = 0; q < S::VW; ++q) w.v[e][q] = finite_word<STORE>(w.v[e][q]);
            }
        }
        // values
        if constexpr (S::FP32) {
#pragma unroll
            for (int e = 0; e < 4 * NT; ++e)
#pragma unroll
                for (int q = 0; q < CPL; ++q) acc[q] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(w.v[e][q]), p[e], acc[q], 0, 0, 0);
        } else {
#pragma unroll
            for (int g = 0; g < NT / 2; ++g) {
                bf16x8 pb[S::WPARTS];
                if constexpr (S::WPARTS == 3) split3(&p[8 * g], pb);
                else split2<STORE == RALF_KV_BF16>(&p[8 * g], pb);
#pragma unroll
                for (int q = 0; q < CPL; q += 2) {
                    // columns q, q + 1 of the lane, keys in the order of pb: pairs of keys side by side
                    u32x4 v0, v1;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if constexpr (STORE == RALF_KV_BF16) {
                            const uint32_t lo2 = w.v[8 * g + 2 * e][q >> 1], hi2 = w.v[8 * g + 2 * e + 1][q >> 1];
                            v0[e] = __builtin_amdgcn_perm(hi2, lo2, 0x05040100u);
                            v1[e] = __builtin_amdgcn_perm(hi2, lo2, 0x07060302u);
                        } else {
                            const u32x2 u = codes_bf16<STORE>(__builtin_amdgcn_perm(w.v[8 * g + 2 * e + 1][q >> 2], w.v[8 * g + 2 * e][q >> 2], (q & 2) ? 0x07030602u : 0x05010400u));
                            v0[e] = u[0];
                            v1[e] = u[1];
                        }
                    }
#pragma unroll
                    for (int y = S::WPARTS - 1; y >= 0; --y) {
                        acc[q] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, v0), pb[y], acc[q], 0, 0, 0);
                        acc[q + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, v1), pb[y], acc[q + 1], 0, 0, 0);
                    }
                }
            }
        }
    };
    int blk = sb + wave;
    look(blk);
    if constexpr (S::TWO) {
        // two blocks' registers in turn: the next block's loads are in flight while this one is computed
        Buf w0, w1;
        if (blk < se) load(w0, blk);
        look(blk + 4);
        while (blk < se) {
            if (blk + 4 < se) load(w1, blk + 4);
            look(blk + 8);
            compute(w0, blk);
            blk += 4;
            if (blk >= se) break;
            if (blk + 4 < se) load(w0, blk + 4);
            look(blk + 8);
            compute(w1, blk);
            blk += 4;
        }
    } else {
        Buf w0;
        for (; blk < se; blk += 4) {
            load(w0, blk);
            look(blk + 4);
            compute(w0, blk);
        }
    }

    // The values taken out above, to the rows that see them: their weights are positive, so the sum is the value itself.  Rare, so short in registers.
    if (odd) {
        for (blk = sb + wave; blk < se; blk += 4) {
            look(blk);
            uint32_t bad = 0u;
#pragma unroll
            for (int s = 0; s < NT; ++s) bad |= (pages[s] >= 0 && pages[s] < c.n_pages ? 0u : 1u) << s;
            if (!is_mixed(blk, bad)) continue;
            for (int k = 0; k < KB; ++k) {
                const int key = blk * KB + k;
                if (key >= t.L || ((bad >> (k >> 4)) & 1u)) continue;
                const uint8_t* vrow = (const uint8_t*)c.v + (table[key >> a.page_log2] * head_rows + (int64_t)hk * c.page + (key & (c.page - 1))) * (D * ESZ);
                const bool see = key >= lo && key <= hi;
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int q = 0; q < CPL; ++q) {
                        const float x = odd_value<STORE>(vrow, (4 * kg + i) * CPL + q);
                        if (see) acc[q][i] += x;
                        asm volatile("" ::: "memory");      // (one load at a time)
                    }
            }
        }
    }

    // join the four waves through LDS: first the maxima and sums, then in the same place the accumulators (lane: row r16, columns (4 kg + i) * CPL + q);
    // 16 threads to a row
    l = sum4(l);
    const int orow = threadIdx.x >> 4, oc = threadIdx.x & 15;
    if (kg == 0) { sm[(wave * 16 + r16) * 2] = m; sm[(wave * 16 + r16) * 2 + 1] = l; }
    __syncthreads();
    float mm = -__builtin_inff(), ll = 0.f, fw[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) { fw[w] = sm[(w * 16 + orow) * 2]; mm = fmaxf(mm, fw[w]); }
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        fw[w] = exp2f_(fw[w] - (mm == -__builtin_inff() ? 0.f : mm));
        ll += fw[w] * sm[(w * 16 + orow) * 2 + 1];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int q = 0; q < CPL; ++q) sm[(wave * 16 + r16) * D + (4 * kg + i) * CPL + q] = acc[q][i];
    __syncthreads();
    if (t.row0 + orow >= t.rows) return;
    float o[CPL];
#pragma unroll
    for (int q = 0; q < CPL; ++q) o[q] = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w)
#pragma unroll
        for (int q = 0; q < CPL; ++q) o[q] += fw[w] * sm[(w * 16 + orow) * D + oc + 16 * q];
    const int oti = (t.row0 + orow) / a.G, ohq = hk * a.G + (t.row0 + orow) % a.G;
    if (a.few.splits > 1) {
        const int64_t own = a.few.slots ? ((int64_t)t.b * a.few_rows + t.row0 + orow) * c.heads + hk : (tok0 + oti) * a.d.q_heads + ohq, at = split * a.few.rows + own;
#pragma unroll
        for (int q = 0; q < CPL; ++q) a.few.o[at * D + oc + 16 * q] = o[q];
        if (oc == 0) { a.few.ml[at * 2] = mm; a.few.ml[at * 2 + 1] = ll; }
    } else {
        const float inv = ll == 0.f ? 0.f : 1.f / ll;
        const int64_t at = (tok0 + oti) * a.d.o_ts + ohq * a.d.o_hs;
#pragma unroll
        for (int q = 0; q < CPL; ++q) {
            const float x = ll == 0.f ? 0.f : o[q] * inv;
            if constexpr (F32) ((float*)a.d.o)[at + oc + 16 * q] = x;
            else ((bf16*)a.d.o)[at + oc + 16 * q] = (bf16)x;
        }
    }
}

// ------------------------------------------------------------------------------------------------
// many rows: 32 to a wave, 8 (4) waves share tiles of 64 keys in LDS, each byte from memory once per 256 (128) rows.
// v_mfma_f32_32x32x16_bf16: a lane owns row (lane & 31) and of every 32 keys the sixteen 8 (i / 4) + 4 (lane / 32) + i % 4.
//   * a tile's loads are issued a tile ahead into registers and stored to the other LDS buffer behind the products: one barrier a tile.  8-bit codes become
//     bf16 values there, once for all waves.
//   * LDS rows of dim elements without padding, their 16-byte chunks swizzled (kswz, vswz).
//   * scores run half a tile ahead of their weights and products half a tile behind, step by step in one stream of instructions: the vector unit's 16 exponentials a
//     lane and half (as long as 8 matrix instructions) run in the matrix unit's shadow.
// 2048 new on 8192 cached tokens, 32 / 8 heads of 128: 302 - 330 us from card to card, 1020 - 940 TFLOP/s (a large plain product: 1611), both units half busy at a clock of 2.0 GHz.  Left out one at a
// time: staging - 46 us, weights - 43, settling - 11; bare matrix instructions, LDS reads and barriers 229 us.  Loads straight into LDS (6 us slower), fragments 4 or 6
// steps ahead, two workgroups of 4 waves to a CU (+ 23) and other wave priorities gained nothing.
// ------------------------------------------------------------------------------------------------
template <int N> struct Const { static constexpr int value = N; };
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
#define LDS_PTR(T, p) ((__attribute__((address_space(3))) T*)(p))

template <int D, int W>
struct Many {
    static constexpr int WAVES = W, BM = 32 * WAVES, KB = 64;
    static constexpr int TPK = WAVES;                               // threads of a key row
    static constexpr int EPT = D / TPK, CH = EPT < 8 ? EPT : 8, NCH = EPT / CH;     // a thread's elements, in chunks of CH
    static constexpr int CPR = D / 8;                               // 16-byte chunks of an LDS row
    static constexpr int LDS = 2 * 2 * KB * D * 2;                  // bytes: K and V, two buffers
    // where 16-byte chunk c of a row lies: c ^ kswz(key), c ^ vswz(key).  Sixteen lanes reading one chunk of sixteen keys, and 32 lanes reading 4 chunks of 4 values
    // (the transposing read), so touch each of the 64 banks once.
    static __device__ __forceinline__ int kswz(int key) { return D >= 128 ? key & 15 : D == 64 ? (key >> 1) & 7 : (key >> 2) & 3; }
    static __device__ __forceinline__ int vswz(int key) { return D >= 128 ? 4 * (key & 3) : D == 64 ? 4 * ((key >> 1) & 1) : 0; }
};

// CH codes / values of a chunk, bf16 pairs
template <int STORE, int CH>
__device__ __forceinline__ void chunk_bf16(const uint32_t (&raw)[STORE == RALF_KV_BF16 ? CH / 2 : CH / 4], uint32_t ex, uint32_t (&w)[CH / 2]) {
    if constexpr (STORE == RALF_KV_BF16) {
#pragma unroll
        for (int i = 0; i < CH / 2; ++i) w[i] = raw[i];
    } else {
        const float sc = exp_value(ex);
#pragma unroll
        for (int i = 0; i < CH / 4; ++i) {
            if constexpr (STORE == RALF_KV_E4M3) {
                w[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(raw[i], sc, false));
                w[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(raw[i], sc, true));
            } else {
                float f[4];
                codes_f32<STORE>(raw[i], f);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const bf16x2 b = {(bf16)(f[2 * j] * sc), (bf16)(f[2 * j + 1] * sc)};        // (7 significant bits: exact)
                    w[2 * i + j] = __builtin_bit_cast(uint32_t, b);
                }
            }
        }
        if (ex == 255u) {
#pragma unroll
            for (int i = 0; i < CH / 2; ++i) w[i] = 0x7fc07fc0u;
        }
    }
}

template <int D, int STORE, int W>
__global__ __launch_bounds__(64 * W, (D == 256 ? 1 : 2)) void many_kernel(const Args a, int ntiles) {
    typedef Many<D, W> M;
    constexpr int KB = M::KB, ESZ = STORE == RALF_KV_BF16 ? 2 : 1, RW = M::CH * ESZ / 4;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    __shared__ int s_odd;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r32 = lane & 31, h = lane >> 5;
    const RalfPagedKV& c = a.d.kv;
    // tiles of one key head and split side by side on one XCD (workgroups are dealt to the 8 XCDs in turn): they read the same keys
    const int nwg = gridDim.x, q8 = nwg >> 3, r8 = nwg & 7, xcd = blockIdx.x & 7;
    const int vid = (xcd < r8 ? xcd * (q8 + 1) : r8 * (q8 + 1) + (xcd - r8) * q8) + (blockIdx.x >> 3);
    const int hk = vid / ntiles / a.many.splits, split = vid / ntiles % a.many.splits;
    const Tile t = find_tile<M::BM>(a, vid % ntiles, lane, 0);
    if (!t.ok || t.rows <= a.few_rows) return;
    if (threadIdx.x == 0) s_odd = 0;        // (a barrier ahead of the first value stored)
    const int64_t tok0 = t.tok0;
    const int row = t.row0 + 32 * wave + r32;
    const bool live = row < t.rows;
    const int ti = (live ? row : t.row0) / a.G, hq = hk * a.G + (live ? row : t.row0) % a.G;
    const int pos = t.first + ti;
    const int hi = !live ? -1 : a.d.causal && pos < t.L - 1 ? pos : t.L - 1;
    const int lo = behind(pos, a.d.window);
    struct Range { int kbeg, kend, lo, hi; };
    auto range = [&](int r0, int n) {     // the keys that some (kbeg .. kend - 1) and that every one (lo .. hi) of n rows from r0 on sees
        const int last = (r0 + n < t.rows ? r0 + n : t.rows) - 1;
        const int p0 = t.first + r0 / a.G, p1 = t.first + last / a.G;
        return Range{behind(p0, a.d.window), a.d.causal && p1 < t.L ? p1 + 1 : t.L, behind(p1, a.d.window), a.d.causal && p0 < t.L - 1 ? p0 : t.L - 1};
    };
    const Range all = range(t.row0, M::BM);
    const int w0 = t.row0 + 32 * wave;
    const Range own = w0 < t.rows ? range(w0, 32) : Range{0, 0, 0, -1};
    const int kbeg = all.kbeg, kend = all.kend, wg_lo = all.lo, wg_hi = all.hi, full_lo = own.lo, full_hi = own.hi;
    const int blk0 = kbeg / KB, nblk = kend > kbeg ? (kend + KB - 1) / KB - blk0 : 0;
    const int per = (nblk + a.many.splits - 1) / a.many.splits;
    const int sb = blk0 + split * per, se = sb + per < blk0 + nblk ? sb + per : blk0 + nblk;

    u32x4 q[D / 16];
    {
        const bf16* qp = (const bf16*)a.d.q + (tok0 + ti) * a.d.q_ts + hq * a.d.q_hs + 8 * h;
        const uint32_t flip = a.qscale < 0.f ? 0x80008000u : 0u;      // (a negative scale goes into the query, so that the largest score has the largest weight)
#pragma unroll
        for (int j = 0; j < D / 16; ++j) {
            q[j] = live ? *(const u32x4*)(qp + 16 * j) : u32x4{0u, 0u, 0u, 0u};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (a.qscale == 0.f) q[j][i] = ((q[j][i] & 0x7f80u) == 0x7f80u ? 0x7fc0u : 0u) | ((q[j][i] & 0x7f800000u) == 0x7f800000u ? 0x7fc00000u : 0u);
                q[j][i] ^= flip;
            }
        }
    }
    const float qs = a.qscale == 0.f ? 1.f : fabsf(a.qscale);          // (a scale of 0 is a query of 0, and of NaN where it was not finite: hidden scores are -inf, and stay so)
    f32x16 acc[D / 32];
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) acc[i][j] = 0.f;
    // the reference of the exponentials, in log2 units and always a whole number, so that moving it scales what has been summed up exactly; set HEADROOM above the largest
    // score it stays until a score passes it (a weight is then 1 at most)
    float m2 = -__builtin_inff(), l = 0.f;

    const int* table = c.table + (int64_t)t.b * c.table_ld;
    const int64_t head_rows = (int64_t)c.heads * c.page;
    const int skey = threadIdx.x / M::TPK, spart = threadIdx.x % M::TPK, s4 = skey >> 4;        // the key row and part of it that this thread brings in
    // pages of a tile's four sixteens, one to a lane (lane & 3); the keys that a wave brings in lie in one of them
    const int lane4 = lane & 3, mine = __builtin_amdgcn_readfirstlane(s4);
    auto look = [&](int blk) {
        const int k0 = blk * KB + 16 * lane4;
        const bool in = blk < se && k0 < t.L;
        const int pg = table[in ? k0 >> a.page_log2 : 0];
        return in && pg >= 0 && pg < c.n_pages ? pg : -1;
    };
    auto bad_of = [&](int pages) { return (uint32_t)__ballot(pages < 0) & 15u; };
    // the pool's row of the first key that this wave brings in (of page 0 if its page is not there): the same for all its lanes
    auto row_of = [&](int blk, int pages) {
        const int pg = __builtin_amdgcn_readlane(pages, mine);
        return (pg < 0 ? 0 : pg) * head_rows + (int64_t)hk * c.page + ((blk * KB + 16 * mine) & (c.page - 1));
    };
    const uint32_t lane_row = skey & 15, lane_at = (lane_row * D + spart * M::CH) * ESZ;
    uint32_t kr[M::NCH][RW], vr[M::NCH][RW], kex = 127u, vex = 127u;
    auto load = [&](const void* base, const void* exps, int64_t row, uint32_t (&w)[M::NCH][RW], uint32_t& ex) {
        const uint8_t* p = (const uint8_t*)base + row * (D * ESZ);
#pragma unroll
        for (int i = 0; i < M::NCH; ++i) load_words<RW>(p + lane_at + i * (M::TPK * M::CH * ESZ), w[i], 4);
        if constexpr (STORE >= RALF_KV_E4M3) ex = ((const uint8_t*)exps + row)[lane_row];
    };
    uint8_t* const ks = lds;
    uint8_t* const vs = lds + 2 * KB * D * 2;
    auto put = [&](uint8_t* row, int ch, int off, const uint32_t (&w)[M::CH / 2]) {
        uint8_t* p = row + (ch << 4) + off;
        if constexpr (M::CH == 8) *(u32x4*)p = u32x4{w[0], w[1], w[2], w[3]};
        else *(u32x2*)p = u32x2{w[0], w[1]};
    };
    auto store_k = [&](int buf) {
#pragma unroll
        for (int i = 0; i < M::NCH; ++i) {
            uint32_t w[M::CH / 2];
            chunk_bf16<STORE, M::CH>(kr[i], kex, w);
            const int e = (i * M::TPK + spart) * M::CH;
            put(ks + (buf * KB + skey) * (D * 2), (e >> 3) ^ M::kswz(skey), (e & 7) * 2, w);
        }
    };
    auto store_v = [&](int buf, int blk, uint32_t bad) {
        const bool mixed = blk * KB < wg_lo || blk * KB + KB - 1 > wg_hi || bad;     // some row of the workgroup does not see some key of the tile
        const bool gone = ((bad >> mine) & 1u) || blk * KB + skey >= t.L;
#pragma unroll
        for (int i = 0; i < M::NCH; ++i) {
            uint32_t w[M::CH / 2];
            chunk_bf16<STORE, M::CH>(vr[i], vex, w);
            if (mixed) {
                // values that are not there: 0.  Infinities and NaN, which 0 * inf would carry to rows that do not see them: taken out, and given to the rows that do
                // see them when the loop is done
#pragma unroll
                for (int x = 0; x < M::CH / 2; ++x) {
                    if (gone) w[x] = 0u;
                    else if (odd_word<RALF_KV_BF16>(w[x])) { w[x] = finite_word<RALF_KV_BF16>(w[x]); s_odd = 1; }
                }
            }
            const int e = (i * M::TPK + spart) * M::CH;
            put(vs + (buf * KB + skey) * (D * 2), (e >> 3) ^ M::vswz(skey), (e & 7) * 2, w);
        }
    };
    // LDS addresses of a lane's fragments (the swizzles are exclusive ors, so a fragment's place is its number's exclusive or with the lane's own)
    const uint32_t kaddr = r32 * (D * 2) + ((h ^ M::kswz(r32)) << 4);
    uint32_t vaddr;
    {
        const int Ls = lane & 15, vkey = 4 * h + (Ls >> 2), vcol = 16 * ((lane >> 4) & 1) + (Ls & 3) * 4;
        vaddr = 2 * KB * D * 2 + vkey * (D * 2) + (((vcol >> 3) ^ M::vswz(vkey)) << 4) + (vcol & 7) * 2;
    }
    auto key_frag = [&](int j, int at) { return *(const bf16x8*)(lds + (kaddr ^ (j << 5)) + at * (D * 2)); };       // at: buffer * KB + first key
    auto value_frag = [&](int ct, int at) {
        const uint8_t* p = lds + (vaddr ^ (ct << 6)) + at * (D * 2);
        const bf16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(LDS_PTR(bf16x4, p)), v1 = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(LDS_PTR(bf16x4, p + 8 * D * 2));
        return __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7);
    };
    // what the scores are masked with and the reference follows, before their weights are taken; pb: weights taken already and not yet summed up
    auto largest = [&](const f32x16& st) {
        float mx = st[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) mx = __builtin_elementwise_maximum(mx, st[i]);
        return mx;
    };
    auto settle = [&](f32x16& st, float mx, int key0, uint32_t bad2, bf16x8 (&pb)[2]) __attribute__((always_inline)) {
        if (key0 < full_lo || key0 + 31 > full_hi || bad2) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int key = key0 + 8 * (i >> 2) + 4 * h + (i & 3);
                const bool see = key >= lo && key <= hi && !((bad2 >> (i >> 3)) & 1u);
                st[i] = see ? st[i] : -__builtin_inff();
            }
            mx = largest(st);
        }
        float mo = mx;
        wave::swap32(mx, mo);
        mx = __builtin_elementwise_maximum(mx, mo) * qs;
        const bool need = mx > m2;
        if (__any(need)) {
            const float mn = need ? ceilf(mx) + HEADROOM : m2;
            const float alpha = mn == -__builtin_inff() ? 1.f : exp2f_(m2 - mn);       // (m2 = -inf: 0; unchanged: 1)
            m2 = mn;
            l *= alpha;
#pragma unroll
            for (int i = 0; i < D / 32; ++i)
#pragma unroll
                for (int j = 0; j < 16; ++j) acc[i][j] *= alpha;
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int e = 0; e < 8; ++e) pb[u][e] = (bf16)((float)pb[u][e] * alpha);
        }
    };
    // One half's turn: the weights pb of its scores st; beside them the scores sn of the half at `knext` and the products of the weights pp with the values at `vprev`.
    // Written in the order that it is to run in, a scheduling fence behind each step: one matrix instruction, the fragment of the step after next, now and then two
    // weights.  The scores come first, so that their largest (-> the lane's, before any mask) is known when the products are through.
    auto turn = [&](const f32x16& st, bf16x8 (&pb)[2], f32x16& sn, int knext, const bf16x8 (&pp)[2], int vprev) __attribute__((always_inline)) {
        constexpr int S = D / 16, STEPS = 2 * S;
        const float base = m2 == -__builtin_inff() ? 0.f : -m2;
        float s0 = 0.f, s1 = 0.f, mx = 0.f;
        uint32_t w[8];
        bf16x8 f[3];
        auto fetch = [&](int i) { f[i % 3] = i < S ? key_frag(i, knext) : value_frag((i - S) % (D / 32), vprev + 16 * ((i - S) / (D / 32))); };
        fetch(0);
        fetch(1);
#pragma unroll
        for (int i = 0; i < 16; ++i) sn[i] = 0.f;
        __builtin_amdgcn_s_setprio(1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
            if (i < S) sn = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f[i % 3], __builtin_bit_cast(bf16x8, q[i]), sn, 0, 0, 0);
            else {
                const int u = (i - S) / (D / 32), ct = (i - S) % (D / 32);
                acc[ct] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f[i % 3], pp[u], acc[ct], 0, 0, 0);
            }
            if (i + 2 < STEPS) fetch(i + 2);
#pragma unroll
            for (int e = i * 8 / STEPS; e < (i + 1) * 8 / STEPS; ++e) {
                const float x = exp2f_(fmaf(st[2 * e], qs, base)), y = exp2f_(fmaf(st[2 * e + 1], qs, base));
                s0 += x;
                s1 += y;
                const bf16x2 xy = {(bf16)x, (bf16)y};
                w[e] = __builtin_bit_cast(uint32_t, xy);
                asm volatile("" : "+v"(w[e]), "+v"(s0), "+v"(s1));         // (here, in the matrix instructions' shadow, and not where the weights are used)
            }
            if (i == S + S / 2) {
                mx = largest(sn);             // (NaN is carried along: the row's weights are NaN whatever the reference)
                asm volatile("" : "+v"(mx));
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_s_setprio(0);
        pb[0] = __builtin_bit_cast(bf16x8, u32x4{w[0], w[1], w[2], w[3]});
        pb[1] = __builtin_bit_cast(bf16x8, u32x4{w[4], w[5], w[6], w[7]});
        l += s0 + s1;               // (this half's keys only: the two are added at the end)
        return mx;
    };

    // The loop runs over halves of 32 keys: while the weights of one half are taken (vector unit), the scores of the next and the products of the weights before it
    // are made (matrix unit).  Scores so run half a tile ahead and products half a tile behind: in tile j's turn K tiles j and j + 1 and V tiles j - 1 and j are in LDS,
    // K tile j + 1 and V tile j stored there in its first half, with the one barrier behind it.
    const int nt = se > sb ? se - sb : 0;
    if (nt) {
        int pages = look(sb), pages1 = look(sb + 1);
        int64_t row = row_of(sb, pages);
        load(c.k, c.k_exp, row, kr, kex);
        for (int i = threadIdx.x; i < KB * D / 8; i += 64 * M::WAVES) ((u32x4*)(vs + KB * D * 2))[i] = u32x4{0u, 0u, 0u, 0u};      // ("tile -1": values for weights of 0)
        store_k(0);
        load(c.v, c.v_exp, row, vr, vex);
        uint32_t bad0 = bad_of(pages), bad1 = bad_of(pages1);
        row = row_of(sb + 1, pages1);
        load(c.k, c.k_exp, row, kr, kex);           // (behind the last tile: a row that is not there, read from page 0 and never used)
        __syncthreads();
        f32x16 sa, sc;
        bf16x8 pa[2], pc[2];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int e = 0; e < 8; ++e) pa[u][e] = pc[u][e] = (bf16)0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) sa[i] = 0.f;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) sa = __builtin_amdgcn_mfma_f32_32x32x16_bf16(key_frag(i, 0), __builtin_bit_cast(bf16x8, q[i]), sa, 0, 0, 0);
        settle(sa, largest(sa), sb * KB, bad0 & 3u, pa);
        // (one tile with buffer 0 and one with buffer 1 current, so that LDS addresses are constants apart: 24 vector additions a tile less)
        auto tile = [&](auto which, int j) __attribute__((always_inline)) {
            const int BUF = which.value, cur = BUF * KB, oth = KB - cur;
            const int blk = sb + j;
            pages = look(blk + 2);
            // first half: its weights; the scores of the second; the products of the tile before
            const float mc = turn(sa, pa, sc, cur + 32, pc, oth + 32);
            store_k(BUF ^ 1);
            store_v(BUF, blk, bad0);
            load(c.v, c.v_exp, row, vr, vex);
            row = row_of(blk + 2, pages);
            load(c.k, c.k_exp, row, kr, kex);
            settle(sc, mc, blk * KB + 32, bad0 >> 2, pa);
            __syncthreads();
            // second half: its weights; the scores of the next tile's first (of stale keys behind the last tile: not used); the products of this tile's first
            const float ma = turn(sc, pc, sa, oth, pa, cur);
            bad0 = bad1;
            bad1 = bad_of(pages);
            if (j + 1 < nt) settle(sa, ma, (blk + 1) * KB, bad0 & 3u, pc);
        };
        if constexpr (D < 256) {
            for (int j = 0; j < nt; j += 2) {
                tile(Const<0>{}, j);
                if (j + 1 < nt) tile(Const<1>{}, j + 1);
            }
        } else {                // (no registers for two copies)
            struct Which { int value; };
            for (int j = 0; j < nt; ++j) tile(Which{j & 1}, j);
        }
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
            const int u = i / (D / 32), ct = i % (D / 32);
            acc[ct] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(value_frag(ct, ((nt - 1) & 1) * KB + 32 + 16 * u), pc[u], acc[ct], 0, 0, 0);
        }
    }
    __syncthreads();            // (s_odd)

    if (nt) {
        if (s_odd) {            // the values taken out, to the rows that see them
            for (int key = sb * KB; key < se * KB && key < t.L; ++key) {
                const int pg = table[key >> a.page_log2];
                if (pg < 0 || pg >= c.n_pages) continue;
                const int k0 = key & ~(KB - 1);
                uint32_t b = 0u;
                for (int s = 0; s < 4; ++s) {
                    const int p = k0 + 16 * s < t.L ? table[(k0 + 16 * s) >> a.page_log2] : -1;
                    b |= p >= 0 && p < c.n_pages ? 0u : 1u;
                }
                if (!(k0 < wg_lo || k0 + KB - 1 > wg_hi || b)) continue;        // (a tile that all see kept them)
                const int64_t at = pg * head_rows + (int64_t)hk * c.page + (key & (c.page - 1));
                const uint8_t* vrow = (const uint8_t*)c.v + at * (D * ESZ);
                float scale = 1.f;
                if constexpr (STORE >= RALF_KV_E4M3) scale = exp_value(((const uint8_t*)c.v_exp)[at]);
                const bool see = key >= lo && key <= hi;
#pragma unroll
                for (int ct = 0; ct < D / 32; ++ct)
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int col = 32 * ct + 8 * (i >> 2) + 4 * h + (i & 3);
                        float x;
                        if constexpr (STORE == RALF_KV_BF16) x = odd_value<STORE>(vrow, col);
                        else {          // (an exponent of 255, a NaN code, a product behind fp32's range)
                            float f[4];
                            codes_f32<STORE>(vrow[col], f);
                            x = f[0] * scale;
                            x = fabsf(x) < __builtin_inff() ? 0.f : x;
                        }
                        if (see) acc[ct][i] += x;
                        asm volatile("" ::: "memory");      // (one load at a time)
                    }
            }
        }
    }

    if (!live) return;
    float lo2 = l;
    wave::swap32(l, lo2);
    l += lo2;
    if (a.many.splits > 1) {
        const int64_t at = split * a.many.rows + (tok0 + ti) * a.d.q_heads + hq;
#pragma unroll
        for (int ct = 0; ct < D / 32; ++ct)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                *(f32x4*)(a.many.o + at * D + 32 * ct + 8 * g + 4 * h) = f32x4{acc[ct][4 * g], acc[ct][4 * g + 1], acc[ct][4 * g + 2], acc[ct][4 * g + 3]};
        if (h == 0) { a.many.ml[at * 2] = m2; a.many.ml[at * 2 + 1] = l; }
    } else {
        const float inv = l == 0.f ? 0.f : 1.f / l;
        bf16* op = (bf16*)a.d.o + (tok0 + ti) * a.d.o_ts + hq * a.d.o_hs;
#pragma unroll
        for (int ct = 0; ct < D / 32; ++ct)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                bf16x4 o;
#pragma unroll
                for (int i = 0; i < 4; ++i) o[i] = (bf16)(l == 0.f ? 0.f : acc[ct][4 * g + i] * inv);
                *(bf16x4*)(op + 32 * ct + 8 * g + 4 * h) = o;
            }
    }
}

// The splits of one kernel's rows joined, a workgroup to a row of its Part: the splits' maxima and sums give each its weight (LDS), then their sums are added up, several splits at once
// and eight loads of each in flight.  Registers for 8 waves to a SIMD: the 2048 rows of 64 decoded tokens run in one round (with 66 registers 6.2 us instead of 5).
enum JoinRows { ALL, FEW_BESIDE_MANY, MANY_BESIDE_FEW };      // whose rows: of the one kernel that runs, or of one of the two
template <int D, bool F32, JoinRows ROWS>
__global__ __launch_bounds__(256, 8) void join_kernel(const Args a, const Part p) {
    constexpr int LANES = D / 4;                                    // threads of a split's row, 4 columns each
    constexpr int WAYS = 256 / LANES;                               // splits at once
    __shared__ float so[WAYS][D], weight[MAX_SPLITS], red[4][2];
    uint32_t r = blockIdx.x;            // (FEW_BESIDE_MANY: a slot, whichever way the rows lie)
    const int64_t R = p.rows;
    int64_t t;
    int h;
    if constexpr (ROWS == FEW_BESIDE_MANY) {
        const uint32_t br = r / (uint32_t)a.d.kv.heads;
        const int hk = (int)(r - br * (uint32_t)a.d.kv.heads), b = (int)(br / (uint32_t)a.few_rows), row = (int)(br % (uint32_t)a.few_rows);
        const int64_t s = a.d.q_start[b], e0 = a.d.q_start[b + 1], e = e0 < a.d.T ? e0 : a.d.T, rows = (e - s) * a.G;
        if (s < 0 || row >= rows || rows > a.few_rows) return;
        t = s + row / a.G;
        h = hk * a.G + row % a.G;
        if (!p.slots) r = (uint32_t)(t * a.d.q_heads + h);
    } else {
        t = r / (uint32_t)a.d.q_heads;
        h = (int)(r - (uint32_t)t * (uint32_t)a.d.q_heads);
        if (t < a.d.q_start[0] || t >= a.d.q_start[a.d.kv.B]) return;
        if constexpr (ROWS == MANY_BESIDE_FEW) {        // (not few_kernel's)
            const Owner w = owner_of(a.d.q_start + 1, a.d.kv.kv_len, a.d.kv.B, t, threadIdx.x & 63);
            const int64_t e = w.end < a.d.T ? w.end : a.d.T;
            if (w.b >= a.d.kv.B || (e - a.d.q_start[w.b]) * a.G <= a.few_rows) return;
        }
    }
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    static_assert(MAX_SPLITS <= 256, "one thread to a split's maximum");
    const bool have = tid < p.splits;
    const float ms = have ? p.ml[((int64_t)tid * R + r) * 2] : -__builtin_inff(), ls = have ? p.ml[((int64_t)tid * R + r) * 2 + 1] : 0.f;
    const float wm = wave::max64(ms);
    if (lane == 0) red[wave][0] = wm;
    __syncthreads();
    const float mm = fmaxf(fmaxf(red[0][0], red[1][0]), fmaxf(red[2][0], red[3][0])), base = mm == -__builtin_inff() ? 0.f : mm;
    const float f = exp2f_(ms - base);
    if (have) weight[tid] = f;
    const float wl = wave::sum64(f * ls);
    if (lane == 0) red[wave][1] = wl;
    __syncthreads();
    const float ll = (red[0][1] + red[1][1]) + (red[2][1] + red[3][1]);
    const int way = tid / LANES, ln = tid % LANES;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    const float* src = p.o + (int64_t)r * D + 4 * ln;
#pragma unroll 8
    for (int s = way; s < p.splits; s += WAYS) o += *(const f32x4*)(src + (int64_t)s * R * D) * weight[s];
    *(f32x4*)&so[way][4 * ln] = o;
    __syncthreads();
    if (tid >= D) return;
    float x = 0.f;
#pragma unroll
    for (int w = 0; w < WAYS; ++w) x += so[w][tid];
    x = ll == 0.f ? 0.f : x / ll;
    const int64_t at = t * a.d.o_ts + h * a.d.o_hs + tid;
    if constexpr (F32) ((float*)a.d.o)[at] = x;
    else ((bf16*)a.d.o)[at] = (bf16)x;
}

// How a call is laid out.  A sequence of more than `few` rows under a key head goes to many_kernel: few_kernel reads the keys again for every 16 rows, a tile of
// many_kernel costs the same whether it holds 32 rows or 256.
struct Plan {
    int few_splits, many_splits, few_rows, few_tiles, many_waves;
    int64_t few_grid, many_tiles;       // tiles of 16 and of 32 * many_waves rows; 0: the kernel is not launched
};
inline Plan plan_for(const RalfPagedAttnDesc& d) {
    Plan p = {};
    const int64_t G = d.q_heads / d.kv.heads, B = d.kv.B, rows = d.T * G, heads = d.kv.heads;
    const int64_t most_rows = d.max_q > 0 && d.max_q < d.T ? d.max_q * G : rows;       // (a wrong bound costs time only: each kernel alone takes every sequence)
    int64_t keys = (int64_t)d.kv.max_pages * d.kv.page;
    if (d.max_kv > 0 && d.max_kv < keys) keys = d.max_kv;
    if (d.causal && d.window > 0 && d.window + (int64_t)256 < keys) keys = d.window + (int64_t)256;      // (what a tile can see of them)
    // 64 rows; 32 where the keys are few and a tile's prologue is most of either kernel (64 sequences on 300 keys, us with 32 against 64: 41 / 62 at up to 96 rows, 42 / 53
    // at up to 128, but 48 / 42 at up to 48; on 2048 keys 64 is the better one, 115 against 156 at up to 48 rows, on e4m3 87 against 147), and for a single sequence,
    // which takes one of the kernels alone (48 rows on 32768 keys: 40 against 61, on e4m3 40 against 44)
    const int few = keys <= 512 || B == 1 ? 32 : 64;
    // Splits of few_kernel's keys between wgs workgroups.  A wave takes `turns` blocks of 32 keys one behind the other; two workgroups to a CU run at once.  Splitting costs the
    // join (5 us, some 6 turns), so short axes stay whole; longer ones are cut until the card is full or a wave has two turns left, and to 16 turns at most, so that
    // sequences of different lengths even out (64 sequences of 2048 - 8192: 154 us against 162 in one piece) -- but no further than 4096 workgroups, which even out by
    // themselves.
    auto few_splits = [&](int64_t wgs) {
        const int64_t turns = (keys + 127) / 128;
        const int64_t fill = (512 + wgs - 1) / wgs, enough = (4096 + wgs - 1) / wgs, even = (turns + 15) / 16 < enough ? (turns + 15) / 16 : enough;
        const int64_t s = fill < turns / 2 ? fill : turns / 2;
        return turns < 8 ? 1 : s > even ? s : even;
    };
    auto bounded = [](int64_t s) { return (int)(s > MAX_SPLITS ? MAX_SPLITS : s < 1 ? 1 : s); };
    p.few_splits = p.many_splits = 1;
    if (d.dtype == RALF_F32 || most_rows <= few) {
        p.few_rows = 0x7fffffff;
        p.few_grid = rows / 16 + B;
        const int64_t tiles = d.T * ((G + 15) / 16);
        p.few_splits = bounded(few_splits((p.few_grid < tiles ? p.few_grid : tiles) * heads));
    } else {
        // 256 rows to a workgroup, one of them to a CU; 128 and two to a CU where no sequence has more (half of the waves would only wait: 64 chunks of 32 tokens on
        // 2048, 216 -> 132 us; at 8192 rows 356 us against 333).  At dim 256 the accumulators leave room for 128 rows and one workgroup.
        p.many_waves = d.kv.dim == 256 || most_rows <= 128 ? 4 : 8;
        const int64_t bm = 32 * p.many_waves, slots = d.kv.dim < 256 && p.many_waves == 4 ? 512 : 256;
        p.many_tiles = rows / bm + B;
        // Sequences of few rows beside those of many: single tokens as a rule, one tile to a key head.  Their keys are cut as if they were alone -- few_kernel runs behind
        // many_kernel and has the card to itself (2048 new tokens on 10 240 and one on 131 072: 417 us, 303 and 103 alone; with many_kernel's one piece 2258) -- and not at all
        // if the host's bound leaves no such sequence.  Four prompts of up to 512 tokens on 4096, none of them short, pay 5 us of 152 for the workgroups that find nothing to do.
        if (B > 1 && (d.max_q <= 0 || d.T - (B - 1) * d.max_q <= few / G)) {
            p.few_rows = few;
            p.few_tiles = few / 16;
            p.few_grid = B * (few / 16);
            p.few_splits = bounded(few_splits(B * heads));
        }
        // cut the keys only as far as leaves every CU its workgroups, in pieces of 4 tiles at least
        const int64_t bound = B * ((most_rows + bm - 1) / bm), other = rows / bm + (B < rows / few ? B : rows / few);
        const int64_t wgs = (bound < other ? bound : other) * heads;
        const int64_t s = slots / (wgs > 0 ? wgs : 1);
        p.many_splits = bounded(s > keys / 256 ? keys / 256 : s);
    }
    return p;
}
inline Part part_few(const RalfPagedAttnDesc& d, const Plan& p) {
    const int64_t all = d.T * d.q_heads, slots = (int64_t)d.kv.B * p.few_rows * d.kv.heads;
    const bool fewer = p.few_tiles && slots < all;
    return Part{nullptr, nullptr, fewer ? slots : all, p.few_grid ? p.few_splits : 1, fewer};
}
inline Part part_many(const RalfPagedAttnDesc& d, const Plan& p) { return Part{nullptr, nullptr, d.T * d.q_heads, p.many_splits, false}; }

template <int D, int STORE, int W>
int launch_many(const Args& a, const Plan& p, hipStream_t st) {
    constexpr int lds = Many<D, W>::LDS;
    if (lds >= 65536) (void)hipFuncSetAttribute(reinterpret_cast<const void*>(many_kernel<D, STORE, W>), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    many_kernel<D, STORE, W><<<(int)(p.many_tiles * a.d.kv.heads * a.many.splits), 64 * W, lds, st>>>(a, (int)p.many_tiles);
    return ralf::check_launch("paged_attention (many rows)");
}
template <int D, int STORE, bool F32>
int launch(const Args& a, const Plan& p, void* stream) {
    const int64_t heads = a.d.kv.heads;
    RALF_REQUIRE(p.few_grid * heads * a.few.splits < ((int64_t)1 << 31) && p.many_tiles * heads * a.many.splits < ((int64_t)1 << 31), "paged_attention: too many tiles");
    hipStream_t st = (hipStream_t)stream;
    // (a workgroup to a row: T * q_heads < 2^31 of them; few rows beside many are cut up only where B * heads < 4096)
    auto join = [&](const Part& part, auto rows) {
        const int64_t wgs = rows.value == FEW_BESIDE_MANY ? a.d.kv.B * (int64_t)a.few_rows * heads : part.rows;
        join_kernel<D, F32, (JoinRows)rows.value><<<(int)wgs, 256, 0, st>>>(a, part);
        return ralf::check_launch("paged_attention (join)");
    };
    if constexpr (!F32) {
        if (p.many_tiles) {
            int rc = D < 256 && p.many_waves == 8 ? launch_many<D, STORE, D < 256 ? 8 : 4>(a, p, st) : launch_many<D, STORE, 4>(a, p, st);
            if (!rc && a.many.splits > 1) rc = a.few_tiles ? join(a.many, Const<MANY_BESIDE_FEW>{}) : join(a.many, Const<ALL>{});
            if (rc) return rc;
        }
    }
    if (p.few_grid) {
        few_kernel<D, STORE, F32><<<(int)(p.few_grid * heads * a.few.splits), 256, 4 * 16 * D * sizeof(float), st>>>(a);
        int rc = ralf::check_launch("paged_attention");
        if (!rc && a.few.splits > 1) rc = a.few_tiles ? join(a.few, Const<FEW_BESIDE_MANY>{}) : join(a.few, Const<ALL>{});
        if (rc) return rc;
    }
    return RALF_OK;
}
template <int D>
int launch_dim(const Args& a, const Plan& p, void* stream) {
    if (a.d.dtype == RALF_F32) {
        if (a.d.kv.store == RALF_KV_F32) return launch<D, RALF_KV_F32, true>(a, p, stream);
        if (a.d.kv.store == RALF_KV_E4M3) return launch<D, RALF_KV_E4M3, true>(a, p, stream);
        return launch<D, RALF_KV_INT8, true>(a, p, stream);
    }
    if (a.d.kv.store == RALF_KV_BF16) return launch<D, RALF_KV_BF16, false>(a, p, stream);
    if (a.d.kv.store == RALF_KV_E4M3) return launch<D, RALF_KV_E4M3, false>(a, p, stream);
    return launch<D, RALF_KV_INT8, false>(a, p, stream);
}

int check(const RalfPagedAttnDesc& d) {
    const int rc = check_kv(d.kv, "paged_attention");
    if (rc) return rc;
    RALF_REQUIRE(d.dtype == RALF_F32 || d.dtype == RALF_BF16, "paged_attention: dtype %d", d.dtype);
    RALF_REQUIRE(d.kv.store >= RALF_KV_E4M3 || d.kv.store == (d.dtype == RALF_F32 ? RALF_KV_F32 : RALF_KV_BF16), "paged_attention: a cache of store %d takes queries of its own type", d.kv.store);
    RALF_REQUIRE(d.q_heads > 0 && d.q_heads % d.kv.heads == 0, "paged_attention: %d query heads on %d key heads", d.q_heads, d.kv.heads);
    RALF_REQUIRE(d.T >= 0 && d.T < ((int64_t)1 << 31) && d.T * d.q_heads < ((int64_t)1 << 31), "paged_attention: %lld rows", (long long)d.T);
    RALF_REQUIRE(fabsf(d.scale * LOG2E) < __builtin_inff(), "paged_attention: a scale of %g", d.scale);
    RALF_REQUIRE(d.window >= 0 && d.max_q >= 0 && d.max_kv >= 0, "paged_attention: negative window or bound");
    return RALF_OK;
}
}  // namespace

extern "C" size_t ralf_paged_attention_workspace_bytes(const RalfPagedAttnDesc* d) {
    if (!d || check(*d) || d->T == 0 || d->kv.B == 0) return 0;
    const Plan p = plan_for(*d);
    return part_few(*d, p).bytes(d->kv.dim) + part_many(*d, p).bytes(d->kv.dim);
}

extern "C" int ralf_paged_attention(const RalfPagedAttnDesc* dp, void* workspace, size_t workspace_bytes, void* stream) {
    RALF_REQUIRE(dp, "paged_attention: null descriptor");
    const RalfPagedAttnDesc& d = *dp;
    const int rc = check(d);
    if (rc) return rc;
    if (d.T == 0 || d.kv.B == 0) return RALF_OK;
    RALF_REQUIRE(d.q && d.o && d.q_start, "paged_attention: null pointer");
    RALF_REQUIRE(d.q_ts % 8 == 0 && d.q_hs % 8 == 0 && d.o_ts % 8 == 0 && d.o_hs % 8 == 0 && (uintptr_t)d.q % 16 == 0 && (uintptr_t)d.o % 16 == 0 &&
                     d.q_ts >= 0 && d.q_hs >= 0 && d.o_ts >= 0 && d.o_hs >= 0,
                 "paged_attention: rows have to start at multiples of 8 elements, 16-byte aligned");
    RALF_REQUIRE(ralf::rows_apart(d.T, d.o_ts, d.q_heads, d.o_hs, d.kv.dim), "paged_attention: the output's rows overlap");
    RALF_REQUIRE((d.q == d.o && d.q_ts == d.o_ts && d.q_hs == d.o_hs) || ralf::rows_disjoint({d.q, d.q_ts, d.q_hs}, {d.o, d.o_ts, d.o_hs}, d.T, d.q_heads, d.kv.dim, d.dtype == RALF_BF16 ? 2 : 4),
                 "paged_attention: the output overlaps the queries without being them");
    Args a;
    a.d = d;
    a.G = d.q_heads / d.kv.heads;
    const Plan p = plan_for(d);
    a.few = part_few(d, p);
    a.many = part_many(d, p);
    a.few_rows = p.few_rows;
    a.few_tiles = p.few_tiles;
    a.page_log2 = __builtin_ctz(d.kv.page);
    if (d.kv.n_pages == 0) a.d.kv.max_pages = 0;        // (no page to look at: every row is empty)
    a.qscale = d.scale * LOG2E;
    const size_t need = ralf_paged_attention_workspace_bytes(dp);
    if (need && (!workspace || workspace_bytes < need)) {
        ralf::set_error("paged_attention: workspace of %zu bytes, %zu needed", workspace_bytes, need);
        return RALF_ERR_WORKSPACE;
    }
    float* at = (float*)workspace;      // the sums (of whole 128-byte rows) of both in front of the references
    for (Part* part : {&a.many, &a.few}) {
        if (part->splits == 1) continue;
        part->o = at;
        at += (size_t)part->splits * part->rows * d.kv.dim;
    }
    for (Part* part : {&a.many, &a.few}) {
        if (part->splits == 1) continue;
        part->ml = at;
        at += (size_t)part->splits * part->rows * 2;
    }
    switch (d.kv.dim) {
        case 32: return launch_dim<32>(a, p, stream);
        case 64: return launch_dim<64>(a, p, stream);
        case 128: return launch_dim<128>(a, p, stream);
        default: return launch_dim<256>(a, p, stream);
    }
}
