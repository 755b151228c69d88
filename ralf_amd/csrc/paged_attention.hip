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
// token's or an out-of-window value that is an infinity or a NaN must not reach a row through 0 * inf: see fix_hidden().
#include "paged.h"

namespace {
using namespace paged;

struct Args {
    RalfPagedAttnDesc d;
    int G, splits;
    float qscale;       // scale * log2(e)
    float* part_o;      // [splits][T * q_heads][dim] unnormalised
    float* part_ml;     // [splits][T * q_heads][2] running maximum (log2 units), sum
};

__device__ __forceinline__ float exp2f_(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float max4(float v) { v = fmaxf(v, __shfl_xor(v, 16)); return fmaxf(v, __shfl_xor(v, 32)); }
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
// A block in which some row does not see some key, with an infinity or a NaN among its values: 0 * inf would carry it to the rows that do not see it.  Those
// values are taken out of the product; how many of each kind a (row, column) sees comes from products of indicators, and is put onto the accumulators here.
__device__ __forceinline__ void fix_hidden(f32x4& acc, const f32x4 nan, const f32x4 pos, const f32x4 neg) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (pos[i] > 0.f) acc[i] += __builtin_inff();
        if (neg[i] > 0.f) acc[i] -= __builtin_inff();
        if (nan[i] > 0.f) acc[i] = __builtin_nanf("");
    }
}

template <int D, int STORE, bool F32>
struct Few {
    static constexpr int CPL = D / 16;       // value columns of a lane
    static constexpr int ESZ = STORE == RALF_KV_F32 ? 4 : STORE == RALF_KV_BF16 ? 2 : 1;
};

// CPL consecutive values of one key at byte address p -> fp32
template <int N, int STORE>
__device__ __forceinline__ void load_f32(const uint8_t* p, float (&f)[N]) {
    if constexpr (STORE == RALF_KV_F32) {
        if constexpr (N == 2) { const f32x2 v = *(const f32x2*)p; f[0] = v[0]; f[1] = v[1]; }
        else {
#pragma unroll
            for (int i = 0; i < N / 4; ++i) { const f32x4 v = ((const f32x4*)p)[i]; f[4 * i] = v[0]; f[4 * i + 1] = v[1]; f[4 * i + 2] = v[2]; f[4 * i + 3] = v[3]; }
        }
    } else if constexpr (N == 2) {
        float g[4];
        codes_f32<STORE>(*(const uint16_t*)p, g);
        f[0] = g[0]; f[1] = g[1];
    } else {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) {
            float g[4];
            codes_f32<STORE>(((const uint32_t*)p)[i], g);
#pragma unroll
            for (int j = 0; j < 4; ++j) f[4 * i + j] = g[j];
        }
    }
}
// N consecutive values of one key -> packed bf16 pairs
template <int N, int STORE>
__device__ __forceinline__ void load_b16(const uint8_t* p, uint32_t (&w)[N / 2]) {
    if constexpr (STORE == RALF_KV_BF16) {
        if constexpr (N == 2) w[0] = *(const uint32_t*)p;
        else if constexpr (N == 4) { const u32x2 v = *(const u32x2*)p; w[0] = v[0]; w[1] = v[1]; }
        else {
#pragma unroll
            for (int i = 0; i < N / 8; ++i) { const u32x4 v = ((const u32x4*)p)[i]; w[4 * i] = v[0]; w[4 * i + 1] = v[1]; w[4 * i + 2] = v[2]; w[4 * i + 3] = v[3]; }
        }
    } else if constexpr (N == 2) {
        w[0] = codes_bf16<STORE>(*(const uint16_t*)p)[0];
    } else if constexpr (N == 4) {
        const u32x2 v = codes_bf16<STORE>(*(const uint32_t*)p);
        w[0] = v[0]; w[1] = v[1];
    } else if constexpr (N == 8) {
        const u32x2 r = *(const u32x2*)p;
#pragma unroll
        for (int i = 0; i < 2; ++i) { const u32x2 v = codes_bf16<STORE>(r[i]); w[2 * i] = v[0]; w[2 * i + 1] = v[1]; }
    } else {
#pragma unroll
        for (int h = 0; h < N / 16; ++h) {
            const u32x4 r = ((const u32x4*)p)[h];
#pragma unroll
            for (int i = 0; i < 4; ++i) { const u32x2 v = codes_bf16<STORE>(r[i]); w[8 * h + 2 * i] = v[0]; w[8 * h + 2 * i + 1] = v[1]; }
        }
    }
}

template <int D, int STORE, bool F32>
__global__ __launch_bounds__(256) void few_kernel(const Args a) {
    constexpr int BM = 16, KB = 32, CPL = D / 16;
    typedef Few<D, STORE, F32> Fw;
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
    const int full_lo = behind(p1, a.d.window), full_hi = a.d.causal ? p0 : t.L - 1;   // keys that every row of the tile sees
    // this split's blocks of KB keys
    const int blk0 = kbeg / KB, nblk = kend > kbeg ? (kend + KB - 1) / KB - blk0 : 0;
    const int per = (nblk + a.splits - 1) / a.splits;
    const int sb = blk0 + split * per, se = sb + per < blk0 + nblk ? sb + per : blk0 + nblk;

    const int64_t qoff = (tok0 + ti) * a.d.q_ts + hq * a.d.q_hs;
    constexpr int QN = F32 ? D / 4 : 1, QB = F32 ? 1 : D / 32;
    float qf[QN];
    u32x4 qb[QB];
    if constexpr (F32) {
#pragma unroll
        for (int j = 0; j < D / 16; ++j) {
            const f32x4 v = live ? *(const f32x4*)((const float*)a.d.q + qoff + 16 * j + 4 * kg) : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < 4; ++i) qf[4 * j + i] = v[i];
        }
    } else {
#pragma unroll
        for (int j = 0; j < D / 32; ++j) qb[j] = live ? *(const u32x4*)((const bf16*)a.d.q + qoff + 32 * j + 8 * kg) : u32x4{0u, 0u, 0u, 0u};
    }

    f32x4 acc[CPL];
#pragma unroll
    for (int i = 0; i < CPL; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = -__builtin_inff(), l = 0.f;
    const int* table = c.table + (int64_t)t.b * c.table_ld;
    const int64_t head_rows = (int64_t)c.heads * c.page;

    for (int blk = sb + wave; blk < se; blk += 4) {
        const int key0 = blk * KB;
        int64_t cell[2];            // first pool row of each 16 keys (a page holds whole sixteens), -1: none
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const int k0 = key0 + 16 * s, pi = k0 / c.page;
            const int pg = k0 < t.L ? table[pi] : -1;
            cell[s] = pg >= 0 && pg < c.n_pages ? pg * head_rows + (int64_t)hk * c.page + (k0 - pi * c.page) : -1;
        }
        const bool whole = key0 + KB <= t.L && cell[0] >= 0 && cell[1] >= 0;       // every key of the block is there
        float p[8];
        // scores
        f32x4 st[2];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            st[s] = f32x4{0.f, 0.f, 0.f, 0.f};
            const uint8_t* kp = (const uint8_t*)c.k + ((cell[s] < 0 ? 0 : cell[s]) + r16) * (int64_t)(D * Fw::ESZ);
            if (cell[s] < 0) continue;          // (uniform)
            if constexpr (F32) {
#pragma unroll
                for (int j = 0; j < D / 16; ++j) {
                    float f[4];
                    load_f32<4, STORE>(kp + (16 * j + 4 * kg) * Fw::ESZ, f);
#pragma unroll
                    for (int i = 0; i < 4; ++i) st[s] = __builtin_amdgcn_mfma_f32_16x16x4f32(f[i], qf[4 * j + i], st[s], 0, 0, 0);
                }
            } else {
#pragma unroll
                for (int j = 0; j < D / 32; ++j) {
                    uint32_t w[4];
                    load_b16<8, STORE>(kp + (32 * j + 8 * kg) * Fw::ESZ, w);
                    const u32x4 wv = {w[0], w[1], w[2], w[3]};
                    st[s] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, wv), __builtin_bit_cast(bf16x8, qb[j]), st[s], 0, 0, 0);
                }
            }
        }
        float vs[8];
        uint32_t seen = 0u;         // bit 4 s + i: the row sees that key
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            uint32_t ke = 0x7f7f7f7fu, ve = 0x7f7f7f7fu;
            if constexpr (STORE >= RALF_KV_E4M3) {
                if (cell[s] >= 0) {
                    ke = *(const uint32_t*)((const uint8_t*)c.k_exp + cell[s] + 4 * kg);
                    ve = *(const uint32_t*)((const uint8_t*)c.v_exp + cell[s] + 4 * kg);
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int key = key0 + 16 * s + 4 * kg + i;
                float x = st[s][i];
                if constexpr (STORE >= RALF_KV_E4M3) {
                    x *= exp_value((ke >> (8 * i)) & 0xffu);
                    vs[4 * s + i] = exp_value((ve >> (8 * i)) & 0xffu);
                }
                const bool see = key >= lo && key <= hi && cell[s] >= 0;
                p[4 * s + i] = see ? x * a.qscale : -__builtin_inff();
                seen |= (see ? 1u : 0u) << (4 * s + i);
            }
        }
        // running maximum and sum
        float mx = p[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) mx = fmaxf(mx, p[i]);
        mx = max4(mx);
        const float mn = fmaxf(m, mx), base = mn == -__builtin_inff() ? 0.f : mn;
        const float alpha = exp2f_(m - base);          // (m = -inf: 0)
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) { p[i] = exp2f_(p[i] - base); sum += p[i]; }
        l = l * alpha + sum;                            // (this lane's keys only: summed over the four lane groups at the end)
        m = mn;
#pragma unroll
        for (int i = 0; i < CPL; ++i) acc[i] *= alpha;
        if constexpr (STORE >= RALF_KV_E4M3) {
#pragma unroll
            for (int i = 0; i < 8; ++i) p[i] = (seen >> i) & 1u ? p[i] * vs[i] : 0.f;       // (a hidden row's exponent may stand for NaN)
        }
        const bool mixed = key0 < full_lo || key0 + KB - 1 > full_hi || !whole;     // some row does not see some key of the block
        // values
        if constexpr (F32) {
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                if (cell[s] < 0) continue;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int key = key0 + 16 * s + 4 * kg + i;
                    float f[CPL];
                    load_f32<CPL, STORE>((const uint8_t*)c.v + ((cell[s] + 4 * kg + i) * (int64_t)D + r16 * CPL) * Fw::ESZ, f);
                    if (mixed && key >= t.L) {
#pragma unroll
                        for (int q = 0; q < CPL; ++q) f[q] = 0.f;
                    }
                    if (mixed) {
                        bool odd = false;
#pragma unroll
                        for (int q = 0; q < CPL; ++q) odd |= !(fabsf(f[q]) < __builtin_inff());
                        if (__any(odd)) {
                            const float one = (seen >> (4 * s + i)) & 1u ? 1.f : 0.f;
#pragma unroll
                            for (int q = 0; q < CPL; ++q) {
                                const float x = f[q];
                                const bool ok = fabsf(x) < __builtin_inff();
                                auto count = [&](bool is) { return __builtin_amdgcn_mfma_f32_16x16x4f32(is ? 1.f : 0.f, one, f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0); };
                                fix_hidden(acc[q], count(x != x), count(!ok && x > 0.f), count(!ok && x < 0.f));
                                f[q] = ok ? x : 0.f;
                            }
                        }
                    }
#pragma unroll
                    for (int q = 0; q < CPL; ++q) acc[q] = __builtin_amdgcn_mfma_f32_16x16x4f32(f[q], p[4 * s + i], acc[q], 0, 0, 0);
                }
            }
        } else {
            uint32_t w[8][CPL / 2];
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int key = key0 + 16 * s + 4 * kg + i;
                    if (cell[s] >= 0) load_b16<CPL, STORE>((const uint8_t*)c.v + ((cell[s] + 4 * kg + i) * (int64_t)D + r16 * CPL) * Fw::ESZ, w[4 * s + i]);
                    if (cell[s] < 0 || (mixed && key >= t.L)) {
#pragma unroll
                        for (int q = 0; q < CPL / 2; ++q) w[4 * s + i][q] = 0u;
                    }
                }
            bf16x8 pb;
#pragma unroll
            for (int i = 0; i < 8; ++i) pb[i] = (bf16)p[i];
            if (mixed) {
                bool odd = false;
#pragma unroll
                for (int i = 0; i < 8; ++i)
#pragma unroll
                    for (int q = 0; q < CPL / 2; ++q) odd |= (w[i][q] & 0x7f80u) == 0x7f80u || (w[i][q] & 0x7f800000u) == 0x7f800000u;
                if (__any(odd)) {
                    bf16x8 one;
#pragma unroll
                    for (int i = 0; i < 8; ++i) one[i] = (bf16)((seen >> i) & 1u ? 1.f : 0.f);
#pragma unroll
                    for (int q = 0; q < CPL; ++q) {
                        bf16x8 nan, pos, neg;
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const float x = __builtin_bit_cast(float, (q & 1) ? w[i][q >> 1] & 0xffff0000u : w[i][q >> 1] << 16);
                            const bool ok = fabsf(x) < __builtin_inff();
                            nan[i] = (bf16)(x != x ? 1.f : 0.f);
                            pos[i] = (bf16)(!ok && x > 0.f ? 1.f : 0.f);
                            neg[i] = (bf16)(!ok && x < 0.f ? 1.f : 0.f);
                            if (!ok) w[i][q >> 1] &= (q & 1) ? 0x0000ffffu : 0xffff0000u;
                        }
                        auto count = [&](bf16x8 v) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, one, f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0); };
                        fix_hidden(acc[q], count(nan), count(pos), count(neg));
                    }
                }
            }
#pragma unroll
            for (int q = 0; q < CPL; ++q) {
                u32x4 av;
#pragma unroll
                for (int e = 0; e < 4; ++e) av[e] = __builtin_amdgcn_perm(w[2 * e + 1][q >> 1], w[2 * e][q >> 1], (q & 1) ? 0x07060302u : 0x05040100u);
                acc[q] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, av), pb, acc[q], 0, 0, 0);
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

// the splits of a row joined: one wave per row
template <int D, bool F32>
__global__ __launch_bounds__(256) void join_kernel(const Args a) {
    const int lane = threadIdx.x & 63;
    const int64_t R = a.d.T * a.d.q_heads, r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (r >= R) return;
    const int64_t t = r / a.d.q_heads;
    const int h = (int)(r - t * a.d.q_heads);
    if (t < a.d.q_start[0] || t >= a.d.q_start[a.d.kv.B]) return;
    float mm = -__builtin_inff();
    for (int s = 0; s < a.splits; ++s) mm = fmaxf(mm, a.part_ml[((int64_t)s * R + r) * 2]);
    const float base = mm == -__builtin_inff() ? 0.f : mm;
    float ll = 0.f, o[(D + 63) / 64] = {};
    for (int s = 0; s < a.splits; ++s) {
        const float f = exp2f_(a.part_ml[((int64_t)s * R + r) * 2] - base);
        ll += f * a.part_ml[((int64_t)s * R + r) * 2 + 1];
#pragma unroll
        for (int q = 0; q < (D + 63) / 64; ++q)
            if (D >= 64 || lane < D) o[q] += f * a.part_o[((int64_t)s * R + r) * D + 64 * q + lane];
    }
#pragma unroll
    for (int q = 0; q < (D + 63) / 64; ++q) {
        if (D < 64 && lane >= D) continue;
        const float x = ll == 0.f ? 0.f : o[q] / ll;
        const int64_t at = t * a.d.o_ts + h * a.d.o_hs + 64 * q + lane;
        if constexpr (F32) ((float*)a.d.o)[at] = x;
        else ((bf16*)a.d.o)[at] = (bf16)x;
    }
}

inline int64_t few_tiles(const RalfPagedAttnDesc& d) { return d.T * (d.q_heads / d.kv.heads) / 16 + d.kv.B; }
inline int splits_for(const RalfPagedAttnDesc& d) {
    int64_t keys = (int64_t)d.kv.max_pages * d.kv.page;
    if (d.max_kv > 0 && d.max_kv < keys) keys = d.max_kv;
    const int64_t wgs = few_tiles(d) * d.kv.heads;
    int64_t s = 1024 / (wgs > 0 ? wgs : 1);
    const int64_t most = (keys + 255) / 256;      // two blocks of 32 keys to a wave
    s = s > most ? most : s;
    s = s > 64 ? 64 : s;
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
    join_kernel<D, F32><<<(int)((R + 3) / 4), 256, 0, (hipStream_t)stream>>>(a);
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
