// Attention of each sequence's newest tokens over the paged cache (ralf_paged_attention).
//
// Rows and tiles.  The q_heads / heads = G query heads that share a key head are rows of one product: row r of sequence b under key head hk is token r / G,
// query head hk * G + r % G.  A tile is BM consecutive rows; it sees the keys up to its last row's position.
//
// Products, transposed so that a lane owns one row (lane & 15) throughout: S^T[key][row] = K Q^T, then O^T[dim][row] = V^T P^T.  The accumulators of the first
// are the operand of the second as they stand (the matrix instruction's contraction slots are named after the keys the lane holds), row maxima need
// two exchanges (lanes 16 and 32 apart), and every rescaling is lane-local.
//   bf16: v_mfma_f32_16x16x32_bf16, keys and values rounded to bf16 already (8-bit codes are exact in it, their powers of two go to the scores and the
//         probabilities in fp32), probabilities rounded to bf16 (relative 2^-9; the sum is taken before that rounding in fp32).
//   fp32: v_mfma_f32_16x16x4_f32 throughout.
// Running maximum and sum of the softmax in fp32; exponentials base 2 with log2(e) folded into the scale.
//
// Masks.  A row that has seen no key keeps max = -inf, sum = 0 and gives zeros.  Keys behind kv_len and keys on bad pages are zeroed as they are loaded; a later
// token's or an out-of-window value that is an infinity or a NaN must not reach a row through 0 * inf: see below.
#include "paged.h"

namespace {
using namespace paged;

struct Args {
    RalfPagedAttnDesc d;
    int G, splits, page_log2;
    float qscale;       // scale * log2(e)
    float* part_o;      // [splits][T * q_heads][dim] unnormalised
    float* part_ml;     // [splits][T * q_heads][2] running maximum (log2 units), sum
};

__device__ __forceinline__ float exp2f_(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float sum4(float v) { v += __shfl_xor(v, 16); return v + __shfl_xor(v, 32); }

struct Tile { int b, row0, rows, first, L; bool ok; };  // sequence, first row, its rows, the position of its first new token, its keys

// the first key that a row at position pos sees
__device__ __forceinline__ int behind(int pos, int window) {
    const int64_t k = window > 0 ? (int64_t)pos - window + 1 : 0;
    return k < 0 ? 0 : (int)k;
}

// tile w of BM rows: sequence b's tiles start at q_start[b] * G / BM + b, which leaves every sequence room for ceil(n * G / BM) of them
template <int BM>
__device__ __forceinline__ Tile find_tile(const Args& a, int w, int lane) {
    Tile t;
    const int B = a.d.kv.B, G = a.G;
    const int c = count_le([&](int i) { return (int64_t)a.d.q_start[i] * G / BM + i; }, B, w, lane);
    t.b = c - 1;
    t.ok = false;
    if (c == 0) return t;
    const int64_t s = a.d.q_start[t.b], e0 = a.d.q_start[t.b + 1], e = e0 < a.d.T ? e0 : a.d.T;
    if (s < 0 || e <= s) return t;
    const int64_t row0 = (w - (s * G / BM + t.b)) * BM, rows = (e - s) * G;
    if (row0 >= rows) return t;
    t.row0 = (int)row0;
    t.rows = (int)rows;
    const int64_t most = (int64_t)a.d.kv.max_pages * a.d.kv.page, L = a.d.kv.kv_len[t.b];
    t.L = (int)(L < most ? L : most);
    t.first = (int)(L - (e0 - s));
    t.ok = true;
    return t;
}

// ------------------------------------------------------------------------------------------------
// few rows: 16 to a workgroup, its 4 waves take blocks of 32 keys in turn (a long axis and few rows: the keys are what there is to divide).
// K and V go from memory straight into registers, each byte once per 16 rows.
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
    static constexpr int NT = F32 ? (D * ESZ >= 512 ? 1 : 2) : (D * ESZ >= 128 ? 2 : 4);
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
    const int split = blockIdx.x % a.splits;
    const int hk = (blockIdx.x / a.splits) % c.heads;
    const Tile t = find_tile<BM>(a, blockIdx.x / a.splits / c.heads, lane);
    if (!t.ok) return;
    const int64_t tok0 = a.d.q_start[t.b];
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
    const int per = (nblk + a.splits - 1) / a.splits;
    const int sb = blk0 + split * per, se = sb + per < blk0 + nblk ? sb + per : blk0 + nblk;

    const int64_t qoff = (tok0 + ti) * a.d.q_ts + hq * a.d.q_hs;
    float qf[F32 ? D / 4 : 1];
    u32x4 qb[F32 ? 1 : D / 32];
#pragma unroll
    for (int j = 0; j < S::NK; ++j) {
        const int64_t at = qoff + (4 * j + kg) * S::EPL;
        if constexpr (F32) {
#pragma unroll
            for (int i = 0; i < S::EPL / 4; ++i) {
                const f32x4 v = live ? *(const f32x4*)((const float*)a.d.q + at + 4 * i) : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int q = 0; q < 4; ++q) qf[j * S::EPL + 4 * i + q] = v[q];
            }
        } else {
#pragma unroll
            for (int i = 0; i < S::EPL / 8; ++i) qb[j * (S::EPL / 8) + i] = live ? *(const u32x4*)((const bf16*)a.d.q + at + 8 * i) : u32x4{0u, 0u, 0u, 0u};
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
                if constexpr (F32) {
#pragma unroll
                    for (int x = 0; x < S::KW; ++x) {
                        if constexpr (STORE == RALF_KV_F32) st = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(w.k[s][j][x]), qf[j * S::EPL + x], st, 0, 0, 0);
                        else {
                            float f[4];
                            codes_f32<STORE>(w.k[s][j][x], f);
#pragma unroll
                            for (int i = 0; i < 4; ++i) st = __builtin_amdgcn_mfma_f32_16x16x4f32(f[i], qf[j * S::EPL + 4 * x + i], st, 0, 0, 0);
                        }
                    }
                } else {
#pragma unroll
                    for (int x = 0; x < S::EPL / 8; ++x) {
                        u32x4 kv;
                        if constexpr (STORE == RALF_KV_BF16) kv = u32x4{w.k[s][j][0], w.k[s][j][1], w.k[s][j][2], w.k[s][j][3]};
                        else {
                            const u32x2 u = codes_bf16<STORE>(w.k[s][j][2 * x]), v = codes_bf16<STORE>(w.k[s][j][2 * x + 1]);
                            kv = u32x4{u[0], u[1], v[0], v[1]};
                        }
                        st = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, kv), __builtin_bit_cast(bf16x8, qb[j * (S::EPL / 8) + x]), st, 0, 0, 0);
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
        mx = fmaxf(m, wave::max_x16_x32(mx));
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
        if constexpr (F32) {
#pragma unroll
            for (int e = 0; e < 4 * NT; ++e) {
                float f[CPL];
                if constexpr (STORE == RALF_KV_F32) {
#pragma unroll
                    for (int q = 0; q < CPL; ++q) f[q] = __uint_as_float(w.v[e][q]);
                } else {
#pragma unroll
                    for (int x = 0; x < S::VW; ++x) {
                        float g[4];
                        codes_f32<STORE>(w.v[e][x], g);
#pragma unroll
                        for (int i = 0; i < (CPL < 4 ? CPL : 4); ++i) f[4 * x + i] = g[i];
                    }
                }
#pragma unroll
                for (int q = 0; q < CPL; ++q) acc[q] = __builtin_amdgcn_mfma_f32_16x16x4f32(f[q], p[e], acc[q], 0, 0, 0);
            }
        } else {
#pragma unroll
            for (int g = 0; g < NT / 2; ++g) {
                bf16x8 pb;
#pragma unroll
                for (int i = 0; i < 8; ++i) pb[i] = (bf16)p[8 * g + i];
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
                    acc[q] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, v0), pb, acc[q], 0, 0, 0);
                    acc[q + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, v1), pb, acc[q + 1], 0, 0, 0);
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
    if (a.splits > 1) {
        const int64_t at = ((int64_t)split * a.d.T + tok0 + oti) * a.d.q_heads + ohq;
#pragma unroll
        for (int q = 0; q < CPL; ++q) a.part_o[at * D + oc + 16 * q] = o[q];
        if (oc == 0) { a.part_ml[at * 2] = mm; a.part_ml[at * 2 + 1] = ll; }
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

// the splits of a row joined: a workgroup to a row, its waves take splits in turn
template <int D, bool F32>
__global__ __launch_bounds__(256) void join_kernel(const Args a) {
    constexpr int LANES = D / 4 < 64 ? D / 4 : 64;                  // lanes of a row, 4 columns each
    constexpr int WAYS = 256 / LANES;                               // splits at once
    __shared__ float so[WAYS][D];
    __shared__ float sf[WAYS];
    const int64_t R = a.d.T * a.d.q_heads, r = blockIdx.x;
    const int64_t t = r / a.d.q_heads;
    const int h = (int)(r - t * a.d.q_heads);
    if (t < a.d.q_start[0] || t >= a.d.q_start[a.d.kv.B]) return;
    const int way = threadIdx.x / LANES, ln = threadIdx.x % LANES;
    float mm = -__builtin_inff(), ll = 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    for (int s = way; s < a.splits; s += WAYS) {
        const float ms = a.part_ml[((int64_t)s * R + r) * 2], ls = a.part_ml[((int64_t)s * R + r) * 2 + 1];
        const f32x4 v = *(const f32x4*)(a.part_o + ((int64_t)s * R + r) * D + 4 * ln);
        const float mn = fmaxf(mm, ms), base = mn == -__builtin_inff() ? 0.f : mn, f0 = exp2f_(mm - base), f1 = exp2f_(ms - base);
        ll = ll * f0 + ls * f1;
        o = o * f0 + v * f1;
        mm = mn;
    }
    *(f32x4*)&so[way][4 * ln] = o;
    __shared__ float sl[WAYS];
    if (ln == 0) { sf[way] = mm; sl[way] = ll; }
    __syncthreads();
    if (threadIdx.x >= D) return;
    mm = sf[0];
#pragma unroll
    for (int w = 1; w < WAYS; ++w) mm = fmaxf(mm, sf[w]);
    const float base = mm == -__builtin_inff() ? 0.f : mm;
    float x = 0.f;
    ll = 0.f;
#pragma unroll
    for (int w = 0; w < WAYS; ++w) {
        const float f = exp2f_(sf[w] - base);
        ll += f * sl[w];
        x += f * so[w][threadIdx.x];
    }
    x = ll == 0.f ? 0.f : x / ll;
    const int64_t at = t * a.d.o_ts + h * a.d.o_hs + threadIdx.x;
    if constexpr (F32) ((float*)a.d.o)[at] = x;
    else ((bf16*)a.d.o)[at] = (bf16)x;
}

inline int64_t few_tiles(const RalfPagedAttnDesc& d) { return d.T * (d.q_heads / d.kv.heads) / 16 + d.kv.B; }
// Workgroups of a key axis: as many as give each CU several (their lengths differ), of 256 keys at least, and no more than the join reads quickly
inline int splits_for(const RalfPagedAttnDesc& d) {
    int64_t keys = (int64_t)d.kv.max_pages * d.kv.page;
    if (d.max_kv > 0 && d.max_kv < keys) keys = d.max_kv;
    const int64_t tiles = few_tiles(d) < d.T ? few_tiles(d) : d.T;
    const int64_t wgs = tiles * d.kv.heads;
    int64_t s = (2048 + wgs - 1) / wgs;
    const int64_t most = (keys + 255) / 256;
    s = s > most ? most : s;
    s = s > 128 ? 128 : s;
    return (int)(s < 1 ? 1 : s);
}

template <int D, int STORE, bool F32>
int launch(const Args& a, void* stream) {
    const int64_t grid = few_tiles(a.d) * a.d.kv.heads * a.splits;
    RALF_REQUIRE(grid < ((int64_t)1 << 31), "paged_attention: too many tiles");
    const size_t lds = 4 * 16 * D * sizeof(float);
    few_kernel<D, STORE, F32><<<(int)grid, 256, lds, (hipStream_t)stream>>>(a);
    int rc = ralf::check_launch("paged_attention");
    if (rc || a.splits == 1) return rc;
    const int64_t R = a.d.T * a.d.q_heads;
    join_kernel<D, F32><<<(int)R, 256, 0, (hipStream_t)stream>>>(a);
    return ralf::check_launch("paged_attention (join)");
}
template <int D>
int launch_dim(const Args& a, void* stream) {
    if (a.d.dtype == RALF_F32) {
        if (a.d.kv.store == RALF_KV_F32) return launch<D, RALF_KV_F32, true>(a, stream);
        if (a.d.kv.store == RALF_KV_E4M3) return launch<D, RALF_KV_E4M3, true>(a, stream);
        return launch<D, RALF_KV_INT8, true>(a, stream);
    }
    if (a.d.kv.store == RALF_KV_BF16) return launch<D, RALF_KV_BF16, false>(a, stream);
    if (a.d.kv.store == RALF_KV_E4M3) return launch<D, RALF_KV_E4M3, false>(a, stream);
    return launch<D, RALF_KV_INT8, false>(a, stream);
}

int check(const RalfPagedAttnDesc& d) {
    const int rc = check_kv(d.kv, "paged_attention");
    if (rc) return rc;
    RALF_REQUIRE(d.dtype == RALF_F32 || d.dtype == RALF_BF16, "paged_attention: dtype %d", d.dtype);
    RALF_REQUIRE(d.kv.store >= RALF_KV_E4M3 || d.kv.store == (d.dtype == RALF_F32 ? RALF_KV_F32 : RALF_KV_BF16), "paged_attention: a cache of store %d takes queries of its own type", d.kv.store);
    RALF_REQUIRE(d.q_heads > 0 && d.q_heads % d.kv.heads == 0, "paged_attention: %d query heads on %d key heads", d.q_heads, d.kv.heads);
    RALF_REQUIRE(d.T >= 0 && d.T * d.q_heads < ((int64_t)1 << 31), "paged_attention: %lld rows", (long long)d.T);
    RALF_REQUIRE(d.window >= 0 && d.max_q >= 0 && d.max_kv >= 0, "paged_attention: negative window or bound");
    return RALF_OK;
}
}  // namespace

extern "C" size_t ralf_paged_attention_workspace_bytes(const RalfPagedAttnDesc* d) {
    if (!d || check(*d) || d->T == 0 || d->kv.B == 0) return 0;
    const int s = splits_for(*d);
    return s > 1 ? (size_t)s * d->T * d->q_heads * (d->kv.dim + 2) * sizeof(float) : 0;
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
    Args a;
    a.d = d;
    a.G = d.q_heads / d.kv.heads;
    a.splits = splits_for(d);
    a.page_log2 = __builtin_ctz(d.kv.page);
    if (d.kv.n_pages == 0) a.d.kv.max_pages = 0;        // (no page to look at: every row is empty)
    a.qscale = d.scale * 1.4426950408889634f;
    const size_t need = ralf_paged_attention_workspace_bytes(dp);
    if (need && (!workspace || workspace_bytes < need)) {
        ralf::set_error("paged_attention: workspace of %zu bytes, %zu needed", workspace_bytes, need);
        return RALF_ERR_WORKSPACE;
    }
    a.part_o = (float*)workspace;
    a.part_ml = need ? (float*)workspace + (size_t)a.splits * d.T * d.q_heads * d.kv.dim : nullptr;
    switch (d.kv.dim) {
        case 32: return launch_dim<32>(a, stream);
        case 64: return launch_dim<64>(a, stream);
        case 128: return launch_dim<128>(a, stream);
        default: return launch_dim<256>(a, stream);
    }
}
