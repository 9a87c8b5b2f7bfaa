// Attention over the paged key-value cache (attention_n of the reference, src/es_engine.c:975, whose loops over a host cache
// this replaces): out = softmax(scale q k^T) v with one pass over the keys, keeping per query the running maximum m, the sum
// l of 2^(s - m) and the weighted sum of v rows, all in fp32; an m that moves scales l and the sum by 2^(m_old - m_new).
//
// Rows. The G = heads / kv heads query heads that share a K/V head are rows of one product, for every token of a tile: row r of
// a sequence is query r / G, head r % G. A prompt's tile is then 128 rows of few tokens (little lost to causality) and a decode
// tile the G heads of the one token, and each K or V element that is read serves all of them.
//
// Orientation. Both products run transposed, S^T = K q^T and O^T = V^T P^T: a query is a column, so that its m, l and scale
// live in the lanes of that column, and the layout in which the matrix cores leave S^T is the one in which they take P^T as the
// second operand, up to an order of the keys that V^T is given too: the weights never leave their registers.
//
// fp32 queries. q is split into as many terms of the cache's type as carry fp32's 24 bits (two of fp16 after scaling the row to
// 2^14, 22 bits; three of bf16), one product each, and so are the weights. K and V are exact as they are.
// Queries of the cache's own type go in as they are. Their weights are two terms in decode, which waits for memory: errors against 64 bits
// are those of out's own rounding (131072 tokens, fp16, 2.1e-4; 47.85 us, and with one term 2.6e-4 and 47.7). A prompt rounds them once to
// the type, as out will be: half a step of it relative to each, no more than storing the weights would cost. Its matrix cores are
// what it waits for: two terms would take 2.91 ms, not 2.13, for 16384 tokens of fp16 (error 1.9e-4, not 2.5e-4), 340 us, not
// 264, for 8 prompts of 99 to 3333 in bf16. Who needs more brings q as fp32. l adds up the unrounded weights.
//
// Caches in 8 bits (E8). Their numbers, times the power of two that 16 tokens of a head share, are numbers of bf16, and without it of fp16: one
// instruction turns two of them into either, exactly. bf16 queries take them with their scales, and all else is as over bf16. fp32 and fp16
// queries (UNSCALED) take K as the numbers are, in fp16, so that fp32 needs two terms and not three; K's scales are factors of the scores. V is taken
// with its scales, in bf16, by decode, whose weights are cut into two or three terms of bf16, and without, in fp16, by prompts, whose scales of
// V become factors of the weights (see attn_prompt_kernel). The errors against 64 bits of the cache's numbers: fp32 2.0e-7 to 3.9e-7.
// Half the bytes, and more instructions to a byte: 131072 tokens of one sequence, 4 heads of 128, 32.0 us (134 MB; over bf16 48.1), where decode's
// own kernel takes 27.3 (4.9 TB/s); 4096 prompt tokens, 32 heads of 128 over 8, bf16 157 us (over bf16 150), fp32 269 (over fp16 261).
//
// Sinks (SINKS). A window leaves the first `sinks` tokens of a sequence in sight. Keys are numbered without those between: the sinks rounded up to 64
// (a.kept), then the window's steps, so that chunks, blocks and steps go over both without a gap.
#pragma once
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "es_hip_attn.h"

namespace {

using namespace esq;

// ---- which work a prompt's workgroup takes ---------------------------------------------------------------------------------------
// A tile is PM rows of one sequence and K/V head; a part is a tile's chunk of keys. Chunks have one length for the whole call,
// from the lengths on the device: the least that leaves about `target` parts, so that few rows over many keys fill the device
// and a captured call adapts to later lengths. Every wave finds its part by a scan over the sequences, 64 at a time.
constexpr int PM = 128, PN = 64;   // rows of a tile, keys of a step
// workgroups that a CU holds at once (registers and LDS), with queries of nq terms and heads of dim elements
constexpr int prompt_per_cu(int nq, int dim) { return dim > 128 || (nq == 3 && dim > 64) ? 1 : 2; }
constexpr int PARTS = 256, MOST_PARTS = 512;   // parts that a call is split into, per workgroup that a CU holds; and at most

struct Seq {
    int t0, n, len;      // first query row, queries, tokens
    int base, tiles;     // keys left out before the first chunk's, or behind the first tokens kept (a multiple of 64); tiles of PM rows
};
__device__ Seq seq_of(const AttnArgs &a, int b) {
    Seq s;
    s.t0 = min(max(a.start[b], 0), a.ntok);
    s.n = min(max(a.start[b + 1], s.t0), a.ntok) - s.t0;
    s.len = a.c.tokens(b);
    s.base = a.window ? max(0, (max(0, s.len - s.n - a.window + 1) & ~63) - a.kept) : 0;
    s.tiles = (int)(((long long)s.n * a.G + PM - 1) / PM);
    return s;
}

constexpr int CHUNK_MIN = 128, CHUNK_SAVES = 512, CHUNK_PAIRS = 384;   // keys

// The chunk's keys; 2^30: tiles are whole, which they stay unless chunks shorten the longest by more than CHUNK_SAVES: the
// parts' sums go through memory and a second launch joins them. us, whole and in chunks, 32 heads over 8, fp16: a prompt of 700
// tokens, heads of 64 16 and 19, of 128 22 and 25, of 256 40 and 42; of 1000 21 and 26, 29 and 41, 51 and 51 (fp32 over bf16 34 and 38,
// 54 and 53, 131 and 131); the last 16 of 1500 tokens 27 and 11, 34 and 13, 62 and 19 (44 and 13, 68 and 17, 167 and 31). One
// number for all errs where rows are few, their parts soon joined: the last 16 of 700 stay whole, 15 and 10 for heads of
// 64 in fp16, 26 and 14 for 128 in fp32 over fp16.
// One sequence: its tiles' chunks are as many as there is room for (target), and half as many where that is two to a CU and they
// are of CHUNK_PAIRS keys or less, since twice the parts cost more than the second workgroup of a CU gains. The last 64 of so many
// tokens, 32 heads of 128 over 4, us, in half the chunks and in all: 3000 fp16 20 and 22, fp32 23 and 27; 8001 26 and 29, 32 and 36; 12000 (the
// last that has half) 30 and 32, 39 and 43; 16000 35 and 37, 47 and 50; 30000 53 and 51, 75 and 76. The last 256 of 8001 over 8 57 and
// 53, 80 and 79; heads of 64 the same within 2 us.
// Several: the mean share of a place, and, where a CU holds but one workgroup, longer until the sequences' last chunks find room
// too. Two to a CU even out by themselves, with chunks of whole 128s. us, in bf16 of 256 elements, where one fits, longer and
// not: 3 sequences of 1250 to 2500 tokens, the last 300 new, 107 and 188; in fp16 of 128, where two fit: 16 of 1500 to 3000, the
// last 16 new, longer 48 and not 43, with chunks of whole 64s 59.
__device__ int chunk_of(const AttnArgs &a) {
    if (!a.target) return 1 << 30;
    int chunk, longest = 0;
    if (a.nseq == 1) {
        const Seq s = seq_of(a, 0);
        longest = s.len - s.base;
        const float chunks = fmaxf(1.0f, floorf((float)a.target / (float)max(s.tiles, 1)));
        chunk = (int)((float)longest / chunks + PN) & -PN;
        chunk = max(a.pairs && chunk <= CHUNK_PAIRS ? chunk * 2 : chunk, CHUNK_MIN);
    } else {
        const unsigned step = a.pairs ? CHUNK_MIN : PN;
        auto rounded = [&](unsigned long long keys) {
            return (int)min(max((keys + step - 1) / step * step, (unsigned long long)CHUNK_MIN), 1ull << 30);
        };
        int tiles = 0, span = 0;   // this lane's sequence, where there are no more than 64
        unsigned long long all = 0;
        for (int b = threadIdx.x & 63; b < a.nseq; b += 64) {
            const Seq s = seq_of(a, b);
            tiles = s.tiles;
            span = s.len - s.base;
            all += (unsigned long long)tiles * (unsigned)span;
            if (tiles) longest = max(longest, span);
        }
#pragma unroll
        for (int d = 32; d; d >>= 1) {
            all += __shfl_xor(all, d);
            longest = max(longest, __shfl_xor(longest, d));
        }
        chunk = rounded((all + a.target - 1) / a.target);
        for (int i = 0; i < 8 && !a.pairs && a.nseq <= 64 && chunk < 1 << 30; i++) {
            uint32_t parts = (uint32_t)tiles * (uint32_t)max(1, (span + chunk - 1) / chunk);
#pragma unroll
            for (int d = 32; d; d >>= 1) parts += __shfl_xor(parts, d);
            if (parts <= (uint32_t)a.target) break;
            chunk = max(chunk + PN, rounded((unsigned long long)chunk * parts / a.target));
        }
    }
    return __builtin_amdgcn_readfirstlane((long long)longest <= (long long)chunk + CHUNK_SAVES ? 1 << 30 : chunk);
}
__device__ int chunks_of(const Seq &s, int chunk) { return max(1, (s.len - s.base + chunk - 1) / chunk); }

struct Part {
    int b, tile, chunk, chunks;   // chunks: of the tile
    uint32_t first;               // number of the sequence's first part
    Seq s;
};
// over the lanes up to this one, by lane moves: from 1, 2, 4 and 8 below within a row of 16, a row's last lane to the next row,
// of rows 1 and 3, and the second row's to the upper two
__device__ uint32_t sum_up_to(uint32_t n) {
    int x = (int)n;
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);
    return (uint32_t)x;
}
// The part with number `item` (within one K/V head), or, TILES, the tile with that number and `chunk` 0; false if there is
// none. Starts that are out of order may give any number of parts: they are counted modulo 2^32.
template <bool TILES> __device__ bool part_of(const AttnArgs &a, int item, int chunk, Part &p) {
    const int lane = threadIdx.x & 63;
    uint32_t tiles_before = 0, parts_before = 0;
    if (a.nseq == 1) {
        p.b = 0;
        p.s = seq_of(a, 0);
        p.chunks = chunks_of(p.s, chunk);
        p.first = 0;
    } else {
        for (int g = 0;; g += 64) {
            if (g >= a.nseq) return false;
            Seq s{};
            int chunks = 1;
            uint32_t parts = 0;
            if (g + lane < a.nseq) {
                s = seq_of(a, g + lane);
                chunks = chunks_of(s, chunk);
                parts = (uint32_t)s.tiles * (uint32_t)chunks;
            }
            const uint32_t mine = TILES ? (uint32_t)s.tiles : parts, upto = sum_up_to(mine);
            const uint32_t parts_upto = TILES ? sum_up_to(parts) : upto;
            uint32_t &before = TILES ? tiles_before : parts_before;
            const unsigned long long past = __ballot((uint32_t)item < before + upto);
            if (past) {
                const int w = __builtin_ctzll(past);
                p.b = g + w;
                p.s.t0 = __builtin_amdgcn_readlane(s.t0, w);
                p.s.n = __builtin_amdgcn_readlane(s.n, w);
                p.s.len = __builtin_amdgcn_readlane(s.len, w);
                p.s.base = __builtin_amdgcn_readlane(s.base, w);
                p.s.tiles = __builtin_amdgcn_readlane(s.tiles, w);
                p.chunks = __builtin_amdgcn_readlane(chunks, w);
                p.first = parts_before + (uint32_t)__builtin_amdgcn_readlane((int)(parts_upto - parts), w);
                item = (int)((uint32_t)item - before - (uint32_t)__builtin_amdgcn_readlane((int)(upto - mine), w));
                break;
            }
            tiles_before += TILES ? (uint32_t)__builtin_amdgcn_readlane((int)upto, 63) : 0;
            parts_before += (uint32_t)__builtin_amdgcn_readlane((int)parts_upto, 63);
        }
    }
    p.tile = TILES ? item : item / p.chunks;
    p.chunk = TILES ? 0 : item - p.tile * p.chunks;
    return item >= 0 && p.tile < p.s.tiles;
}

// ---- arithmetic --------------------------------------------------------------------------------------------------------------
template <bool BF> __device__ f4 mfma16(u4 x, u4 y, f4 c) {
    if constexpr (BF) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, x), __builtin_bit_cast(b8, y), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, x), __builtin_bit_cast(h8, y), c, 0, 0, 0);
}
template <bool BF> __device__ f16v mfma32(u4 x, u4 y, f16v c) {
    if constexpr (BF) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8, x), __builtin_bit_cast(b8, y), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, x), __builtin_bit_cast(h8, y), c, 0, 0, 0);
}

// x as the sum of N values of the cache's type, each the nearest to what is left
template <bool BF, int N> __device__ void split(const float (&x)[8], u4 (&y)[N]) {
    using T = std::conditional_t<BF, __bf16, _Float16>;
    using V = T __attribute__((ext_vector_type(8)));
    float r[8];
#pragma unroll
    for (int i = 0; i < 8; i++) r[i] = x[i];
#pragma unroll
    for (int t = 0; t < N; t++) {
        V v;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            v[i] = static_cast<T>(r[i]);
            if (t + 1 < N) r[i] -= static_cast<float>(v[i]);
        }
        y[t] = __builtin_bit_cast(u4, v);
    }
}

constexpr float LOWEST = -INFINITY;
// Weights are 2^SHIFT p, p relative to m, which in fp16 keeps all bits of keys down to 2^-29 of the largest (bf16 has fp32's range).
template <bool BF> constexpr int SHIFT = BF ? 0 : 15;
// A prompt's m may lie below the largest score by up to LAG (in powers of two), and moves, with the sums so far, only past that; its
// weights are 2^(SHIFT - LAG) p. us, so and where m follows every maximum: 16384 tokens, 32 heads of 128 over 4, fp16, 2135
// and 2211; 8 prompts of 99 to 3333 tokens, bf16, 268 and 281. (Decode waits for memory: no difference.)
template <bool BF, int NQ> constexpr int LAG = BF && NQ == 1 ? 8 : 3;
// the exponent that weights are taken relative to: a row that has seen no key (or only minus infinity) keeps zeros, not NaN
__device__ float reference(float m) { return m == LOWEST ? 0.0f : m; }

// A constant in the exponent rounds it: between 8 and 16 half a step of fp32 is 2^-21, 3.3e-7 of the weight, more than the weights'
// terms lose (2^-22); between 2 and 4 it is 8e-8. So the two terms of fp16, which need a 2^BY of 12 or 15, take it as a factor, when
// they are rounded, and their l at the end: exact, and no instruction more than without (decode of 500 tokens 6.66 us and, in the exponent,
// 6.62; 64 prompt tokens behind 7937 31.0 and 30.8). Three terms of bf16 keep the constant small. With 16-bit queries, whose out is rounded to 2^-9 or
// 2^-12, any goes into the exponent.
template <int NQ> constexpr bool FACTOR = NQ == 2;
template <int NQ, int BY> __device__ float weights_sum(float l) { return FACTOR<NQ> ? l * (1 << (BY & 31)) : l; }
template <int NQ, int BY> __device__ float weight(float s, float cs, float ref) {
    return __builtin_amdgcn_exp2f(__builtin_fmaf(s, cs, FACTOR<NQ> ? -ref : BY - ref));
}
template <bool BF, int NQ, int BY, int NP> __device__ void split_weights(const float (&x)[8], u4 (&y)[NP]) {   // NP terms
    if constexpr (NQ == 1 && NP == 2) {
        // Both terms cut off, the second's last bit set: it is off by less than its last place (2^-14 of the weight in bf16, 2^-20 in fp16),
        // to either side, and greater than 0, so that an infinity in V comes out as one.
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            if constexpr (BF) {
                const uint32_t a = __float_as_uint(x[i]), b = __float_as_uint(x[i + 1]);
                const float ra = x[i] - __uint_as_float(a & 0xffff0000u), rb = x[i + 1] - __uint_as_float(b & 0xffff0000u);
                y[0][i / 2] = __builtin_amdgcn_perm(b, a, 0x07060302u);
                y[1][i / 2] = __builtin_amdgcn_perm(__float_as_uint(rb), __float_as_uint(ra), 0x07060302u) | 0x00010001u;
            } else {
                const auto v = __builtin_amdgcn_cvt_pkrtz(x[i], x[i + 1]);
                const auto w = __builtin_amdgcn_cvt_pkrtz(x[i] - static_cast<float>(v[0]), x[i + 1] - static_cast<float>(v[1]));
                y[0][i / 2] = __builtin_bit_cast(uint32_t, v);
                y[1][i / 2] = __builtin_bit_cast(uint32_t, w) | 0x00010001u;
            }
        }
    } else if constexpr (!FACTOR<NQ>) {
        split<BF, NP>(x, y);
    } else {
        static_assert(!BF && NP == 2);
        constexpr float f = 1 << BY;
        h8 v, w;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            v[i] = static_cast<_Float16>(__builtin_fmaf(x[i], f, 0.0f));
            w[i] = static_cast<_Float16>(__builtin_fmaf(x[i], f, -static_cast<float>(v[i])));
        }
        y[0] = __builtin_bit_cast(u4, v);
        y[1] = __builtin_bit_cast(u4, w);
    }
}

// fp32 weights as three bf16 terms, exactly: 24 bits cut off 8 at a time
__device__ void split_whole(const float (&x)[8], u4 (&y)[3]) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        float r[2] = {x[i], x[i + 1]};
#pragma unroll
        for (int t = 0; t < 3; t++) {
            const uint32_t a = __float_as_uint(r[0]), b = __float_as_uint(r[1]);
            y[t][i / 2] = __builtin_amdgcn_perm(b, a, 0x07060302u);
            r[0] -= __uint_as_float(a & 0xffff0000u);
            r[1] -= __uint_as_float(b & 0xffff0000u);
        }
    }
}

// Eight elements of a query row, from d on (zeros past dim): fp32 or 16 bits.
__device__ void load8(const uint8_t *row, int d, int dim, float (&x)[8]) {
    struct __attribute__((packed, aligned(4))) F8 { float x[8]; };
    if (d < dim) {
        const F8 f = *reinterpret_cast<const F8 *>(row + (size_t)d * 4);
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = f.x[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = 0.0f;
    }
}
__device__ u4 load8(const uint8_t *row, int d, int dim) {
    struct __attribute__((packed, aligned(2))) H8 { uint32_t x[4]; };
    u4 y = {0, 0, 0, 0};
    if (d < dim) {
        const H8 f = *reinterpret_cast<const H8 *>(row + (size_t)d * 2);
#pragma unroll
        for (int i = 0; i < 4; i++) y[i] = f.x[i];
    }
    return y;
}

// A query row's terms for the K steps of a product of KS * KL elements a step (lane group g of the row holds elements g * 8 of
// each), and what the row's scores are multiplied by. The lanes that share a row are XOR, 2 XOR, ... apart (XOR: 16 or 32).
// E8: a step's elements as 16 bytes of an 8-bit row hold two steps' (see attn_decode_kernel).
template <int KL, bool E8> __device__ constexpr int query_at(int s, int g) { return E8 ? (s >> 1) * 2 * KL + g * 16 + (s & 1) * 8 : s * KL + g * 8; }
template <bool BF, int NQ, int KS, int KL, int XOR, bool E8 = false>
__device__ float load_query(const uint8_t *row, bool valid, int g, int dim, float c2, u4 (&q)[KS][NQ]) {
    if constexpr (NQ == 1) {
#pragma unroll
        for (int s = 0; s < KS; s++) q[s][0] = valid ? load8(row, query_at<KL, E8>(s, g), dim) : u4{0, 0, 0, 0};
        return c2;
    } else {
        float x[KS][8];
        float big = 0.0f;
#pragma unroll
        for (int s = 0; s < KS; s++) {
            load8(row, valid ? query_at<KL, E8>(s, g) : dim, dim, x[s]);
#pragma unroll
            for (int i = 0; i < 8; i++) big = fmaxf(big, fabsf(x[s][i]));
        }
        int e = 0;
        if constexpr (!BF) {   // to 2^14 <= the largest < 2^15: both terms far from fp16's limits
            if constexpr (XOR == 16) big = with_lane<16>(big, Max());
            big = with_lane<32>(big, Max());
            if (big > 0.0f && big < INFINITY) e = 14 - (static_cast<int>(__float_as_uint(big) >> 23) - 127);
            e = min(e, 126);
        }
#pragma unroll
        for (int s = 0; s < KS; s++) {
            if constexpr (!BF) {
#pragma unroll
                for (int i = 0; i < 8; i++) x[s][i] = ldexpf(x[s][i], e);
            }
            split<BF, NQ>(x[s], q[s]);
        }
        return fmaxf(ldexpf(c2, -e), 1.17549435e-38f);   // (never 0, which would turn a hidden key's score into NaN)
    }
}

// what a query's scores against a run of an 8-bit cache are multiplied by (never 0, as above, nor infinite, which would turn a score of 0 into NaN)
__device__ float times_scale(float cs, float ks) { return __builtin_amdgcn_fmed3f(cs * ks, 1.17549435e-38f, 3.40282347e38f); }

template <bool F32, bool BF> __device__ void store4(uint8_t *row, int d, const float (&x)[4]) {
    if constexpr (F32) {
        struct __attribute__((packed, aligned(4))) F4 { float x[4]; };
        F4 f;
#pragma unroll
        for (int i = 0; i < 4; i++) f.x[i] = x[i];
        *reinterpret_cast<F4 *>(row + (size_t)d * 4) = f;
    } else {
        using T = std::conditional_t<BF, __bf16, _Float16>;
        struct __attribute__((packed, aligned(2))) H4 { T x[4]; };
        H4 f;
#pragma unroll
        for (int i = 0; i < 4; i++) f.x[i] = static_cast<T>(x[i]);
        *reinterpret_cast<H4 *>(row + (size_t)d * 2) = f;
    }
}

// Where runs of 16 keys of a sequence and head begin, one run per lane, in bytes from a pool's start; the upper half is negative
// where the run is in no page, or not asked for. An 8-bit cache's have their scales with them; the scale of a run that nobody sees, which shares
// a step with those that are seen, is 1: its page may be another's by now, and hold a scale that nobody has written.
template <bool E8> struct Runs {
    int lo, hi;
    float ks, vs;
    __device__ Runs(const KvView &c, const int *table, int head, int run, bool asked, bool seen) {
        const int page = asked ? table[run >> (c.shift - 4)] : -1;
        const bool none = page < 0 || page >= c.npages;
        const size_t row = c.row_at(page, head, (run & ((1 << (c.shift - 4)) - 1)) << 4), at = row * c.dim * (E8 ? 1 : 2);
        lo = (int)(uint32_t)at;
        hi = none ? -1 : (int)(at >> 32);
        if constexpr (E8) {
            const bool known = seen && !none;
            const size_t i = known ? row >> 4 : 0;
            ks = known ? c.ks[i] : 1.0f;
            vs = known ? c.vs[i] : 1.0f;
        }
    }
    __device__ bool none(int lane) const { return __builtin_amdgcn_readlane(hi, lane) < 0; }
    __device__ float k_scale(int lane) const { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(ks), lane)); }
    __device__ float v_scale(int lane) const { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(vs), lane)); }
};
// A buffer descriptor of one of them, for loads whose offsets count from its first row: the loads check their own bounds, so that
// what lies past its `bytes` reads as zeros, and so does all of a run that is in no page, and no lane holds an address, only
// its offset. run_of gives it as four words, for asm; Run loads by it, past the caches, as nobody else reads a decode call's keys
// soon. us so and through the caches: 131072 tokens, 4 heads of 128, 49 and 55; 32 sequences of 77 to 8192 tokens 35.9 and 36.4; what
// the last-level cache holds whole gains nothing (48 windows of 4096 tokens, 2 heads of 64, 79 MB: 21.6 and 21.4).
template <bool E8> __device__ u4 run_of(const uint8_t *pool, const Runs<E8> &all, int lane, int bytes) {
    const int hi = __builtin_amdgcn_readlane(all.hi, lane);
    const uint64_t at = reinterpret_cast<uint64_t>(pool) + ((uint64_t)(uint32_t)max(hi, 0) << 32 | (uint32_t)__builtin_amdgcn_readlane(all.lo, lane));
    return u4{(uint32_t)at, (uint32_t)(at >> 32) & 0xffff, hi < 0 ? 0 : (uint32_t)bytes, 0x00020000};
}
template <bool ONCE> struct Run {   // ONCE: past the caches
    __amdgpu_buffer_rsrc_t r;
    template <bool E8> __device__ Run(const uint8_t *pool, const Runs<E8> &all, int lane, int bytes) {
        const int hi = __builtin_amdgcn_readlane(all.hi, lane);
        const uint64_t at = (uint64_t)(uint32_t)max(hi, 0) << 32 | (uint32_t)__builtin_amdgcn_readlane(all.lo, lane);
        r = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(pool + at), (short)0, hi < 0 ? 0 : bytes, 0x00020000);
    }
    __device__ u4 load16(int lane_offset, int offset) const {
        return __builtin_bit_cast(u4, __builtin_amdgcn_raw_buffer_load_b128(r, lane_offset, offset, ONCE ? 2 : 0));
    }
    __device__ u2 load8(int lane_offset, int offset) const {
        return __builtin_bit_cast(u2, __builtin_amdgcn_raw_buffer_load_b64(r, lane_offset, offset, ONCE ? 2 : 0));
    }
    __device__ uint32_t load4(int lane_offset, int offset) const {
        return __builtin_amdgcn_raw_buffer_load_b32(r, lane_offset, offset, ONCE ? 2 : 0);
    }
};

// numbers of 8 bits, times a power of two, as bf16 (or, times 1, as fp16): exact
template <bool BF, bool UPPER> __device__ uint32_t two_of(uint32_t x, float scale) {
    if constexpr (BF) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, scale, UPPER));
    else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, 1.0f, UPPER));
}
template <bool BF> __device__ u4 eight_of(uint32_t x, uint32_t y, float scale) {
    return u4{two_of<BF, false>(x, scale), two_of<BF, true>(x, scale), two_of<BF, false>(y, scale), two_of<BF, true>(y, scale)};
}

// two rows' elements j of 2 packed elements, as a pair
template <int J> __device__ uint32_t pair(uint32_t first, uint32_t second) {
    return __builtin_amdgcn_perm(second, first, J & 1 ? 0x07060302u : 0x05040100u);
}

// ---- one query per sequence ----------------------------------------------------------------------------------------------------
// A tile is the G query heads of a sequence's K/V head (16 of them, where there are more, and every 16 read K and V for themselves: 32
// sequences of 4096 tokens, 2 K/V heads of 128, 8 to 64 heads each, fp16: 8 28 us, 16 30, 17 41, 32 42, 64 78), its keys blocks of 128. The tiles'
// blocks, one after another, are dealt out evenly: workgroup w of a K/V head takes blocks [w * each, (w + 1) * each) of them,
// whatever sequences they are of, so that a ragged batch keeps every workgroup busy to the end. What a workgroup has of a tile
// that others have parts of goes to the workspace, and a second launch joins them. (The last workgroup of a tile to arrive
// could do that in the same launch, but 128 of them counting in one word and one CU reading all their sums took 78 us for one
// sequence of 131072 tokens, where the two launches take 48.) Where no table row holds more than 512 tokens, a tile is one block and one launch does:
// one sequence of 500 tokens, 32 heads of 64 over 8, 6.6 us, in blocks of 128 with the second launch 9.7.
//
// Inside: four waves, each 32 keys at a time in turn, joined in LDS at the end. Nothing is staged: a lane loads its K fragments
// as the matrix cores take them (key lane % 16, 8 elements) and, of V, the DP / 16 elements from (lane % 16) * DP / 16 on of
// the 8 keys whose weights it holds, which it turns into 8 keys of one element each with byte permutes. A fragment read this
// way is used once, so that LDS would only add a copy. Bound by HBM where the caches are long: 131072 tokens of 4 heads of 128,
// fp16, 268 MB in 48 us (5.6 TB/s, joined; 42, 6.4 TB/s, before that), where a plain read reaches 6.2.
constexpr int BLOCK = 7, BLOCK_WHOLE = 9, DECODE_M = 16;   // (log2)
constexpr int DECODE_PARTS = 512;   // parts of a tile that can be joined, and so workgroups of a K/V head, at most
// workgroups that a CU holds at once (8 bits, heads of 64: 64 sequences of 1000 to 9000 tokens, 8 heads, fp32, with two 60 us, three 57, four 58)
constexpr int decode_per_cu(int dim, bool eight) { return eight && dim <= 64 ? 3 : dim <= 128 ? 2 : 1; }
// Workgroups, all heads together: as many as fit the device at once and bring it to the memory's rate; half of that for one
// sequence, whose tiles have the more parts to join: 20000 and 131072 tokens of 8 heads of 128, us, 21 and 87 with 256,
// 23 and 90 with 512. 8 bits, fp32 queries, 5000, 20000 and 131072 tokens, with 256 and with 512: 8 heads of 64 11.2 and 11.9, 14.8 and 15.7, 41.1 and
// 33.2 (the longest would gain); 4 of 128 11.8 and 11.7, 15.1 and 16.5, 32.2 and 33.7; 8 of 256 17.3 and 21.8, 25.5 and 34.6, 91.4 and 100.5.
constexpr int decode_groups(int dim, int nseq, bool eight) { return nseq > 1 ? 256 * decode_per_cu(dim, eight) : 256; }

// the sequences' blocks: lane i has those of sequence g + i, and `extra` more for each of its tiles
struct Blocks {
    int len;
    uint32_t mine, upto;   // of the sequence; of the group's sequences up to it
};
__device__ int blocks_of(const AttnArgs &a, int len, int &base) {   // of one tile; an empty one has a block too: somebody writes its zeros
    base = a.window ? max(0, (max(0, len - a.window) & ~63) - a.kept) : 0;
    return max(1, (len - base + (1 << a.block) - 1) >> a.block);
}
__device__ Blocks blocks_from(const AttnArgs &a, int g, int tiles, int extra) {
    Blocks x{0, 0, 0};
    const int b = g + (threadIdx.x & 63);
    int base;
    if (b < a.nseq) {
        x.len = a.c.tokens(b);
        x.mine = (uint32_t)tiles * (uint32_t)(blocks_of(a, x.len, base) + extra);
    }
    x.upto = a.nseq == 1 ? (uint32_t)__builtin_amdgcn_readfirstlane((int)x.mine) : sum_up_to(x.mine);
    return x;
}

// Every workgroup's way to its blocks: lane i holds those of the sequences `group` + i, of which there are `before` before. Blocks are dealt out
// evenly, `each` to a workgroup. 8 bits (a.weigh): beginning another tile costs a workgroup about what a block does (its pages, its query and its keys
// are waited for, its sums joined), which shows where a workgroup's share would hold three of the shortest tiles: then every tile counts `extra` = 1
// block more, ahead of its own. us, without and with, where that is so: 32 sequences of 77 to 8192 tokens, 4 heads of 128, 27.3 and 23.7; 64 of 300
// to 6000 38.8 and 37.2; 16 of 200 to 20000, 8 heads of 128, 40.0 and 37.8, 256 of 600 72.4 and 72.7; 64 of 100 to 1500, 8 of 64, 22.2 and 20.6. Where
// it is not: 32 of 4096, 8 of 128, 50.2 and 51.9, 100 of 600 36.8 and 36.9; but 160 of 600 53.4 and 50.7, 16 of 300 to 6000, 4 of 128, 19.7 and
// 17.8, 16 of 1000 to 9000, 4 of 256, 36.7 and 34.3, which would gain. To look for the shortest tile takes 0.2 us for up to 64 sequences, 0.9 for 100,
// 1.6 for 256, 7 for 512.
template <bool WEIGH> struct Deal {
    Blocks bl;
    uint32_t total, each, before = 0;
    int group = 0, extra = 0;
    __device__ static uint32_t share(const AttnArgs &a, uint32_t total) {
        const uint32_t n = total + a.target - 1;
        const uint32_t each = __umulhi(n, a.inverse);   // n / target, or one less
        return each + (n - each * a.target >= (uint32_t)a.target);
    }
    __device__ Deal(const AttnArgs &a, int tiles) : bl(blocks_from(a, 0, tiles, 0)) {
        total = (uint32_t)__builtin_amdgcn_readlane((int)bl.upto, 63);
        for (int g = 64; g < a.nseq; g += 64) total += (uint32_t)__builtin_amdgcn_readlane((int)blocks_from(a, g, tiles, 0).upto, 63);
        each = share(a, total);
        if (WEIGH && a.weigh) {
            const int lane = threadIdx.x & 63;
            uint32_t least = lane < a.nseq ? bl.mine : ~0u;
            for (int g = 64 + lane; g < a.nseq; g += 64) {
                int base;
                least = min(least, (uint32_t)tiles * (uint32_t)blocks_of(a, a.c.tokens(g), base));
            }
            if (__any(3 * (uint64_t)least <= (uint64_t)each * tiles)) {
                extra = 1;
                total += (uint32_t)tiles * a.nseq;
                each = share(a, total);
                bl.upto += (uint32_t)tiles * min(lane + 1, a.nseq);
                bl.mine += lane < a.nseq ? tiles : 0;
            }
        }
    }
    // on to the sequences from g on (a multiple of 64)
    __device__ void next(const AttnArgs &a, int tiles) {
        before += (uint32_t)__builtin_amdgcn_readlane((int)bl.upto, 63);
        group += 64;
        bl = blocks_from(a, group, tiles, extra);
    }
    __device__ uint32_t first_of(int in) const { return before + (uint32_t)__builtin_amdgcn_readlane((int)(bl.upto - bl.mine), in); }
};

// AHEAD: steps of a wave's keys on their way. One is enough where other workgroups' are on theirs, and leaves more registers; with 8 bits, a
// step of heads of 64, or one workgroup to a CU, two are better (decode_ahead). us with one and two, fp32: 131072 tokens of one sequence, 4 heads
// of 128, 33.9 and 32.2 (20000 14.6 and 15.1; 20000 and 131072 of 8 heads of 256 23.6 and 25.5, 89.2 and 91.3: one would do there); 32 sequences of 77 to
// 8192 27.1 and 28.6; 64 sequences of 1000 to 9000, 8 heads of 64, 64.6 and 60.3.
constexpr int decode_ahead(int dim, int nseq) { return dim <= 64 || nseq == 1 ? 2 : 1; }
template <bool BF, int NQ, int DP, bool E8 = false, bool SINKS = false, int AHEAD = 1>
__global__ __launch_bounds__(256, DP == 64 && NQ < 3 ? 3 : decode_per_cu(DP, E8)) void attn_decode_kernel(AttnArgs a) {
    constexpr int KS = DP / 32, DL = DP / 16, BM = DECODE_M;
    constexpr bool UNSCALED = E8 && !BF;     // K goes into the product without its scales, which the scores take
    constexpr bool WBF = BF || E8;           // weights and V are bf16
    constexpr int ES = E8 ? 1 : 2;           // bytes of an element
    constexpr int NP = NQ == 1 ? 2 : E8 ? 3 : NQ;   // terms of the weights
    constexpr bool F32 = NQ > 1;
    __shared__ float lm[4][BM], ll[4][BM];
    __shared__ __attribute__((aligned(16))) float lo_acc[4][BM][DP + 4];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int head = blockIdx.x % a.c.heads, group = blockIdx.x / a.c.heads;
    const int rows = a.G, tiles = (a.G + BM - 1) / BM, dim = a.c.dim;

    Deal<E8> deal(a, tiles);
    const uint32_t each = deal.each, end = min(deal.total, (group + 1) * each);
    for (uint32_t pos = group * each; pos < end;) {
        int tid = threadIdx.x;
        asm volatile("" : "+v"(tid));   // (or every address that depends on it is computed ahead of the loop, and kept in registers that the loop lacks)
        const int lane = tid & 63, col = lane & 15, g = lane >> 4;
        unsigned long long past;
        while (!(past = __ballot(pos < deal.before + deal.bl.upto))) {
            deal.next(a, tiles);
            if (deal.group >= a.nseq) return;   // (not while the lengths stay)
        }
        const int in = __builtin_ctzll(past), seq = deal.group + in;
        const int len = __builtin_amdgcn_readlane(deal.bl.len, in);
        const uint32_t s0 = deal.first_of(in);
        int base;
        const int blocks = blocks_of(a, len, base);
        // SINKS: keys are numbered without the `base` that lie behind the first a.kept and before the window
        const int hi = SINKS ? len - base : len;
        const int extra = E8 ? deal.extra : 0, tile = tiles == 1 ? 0 : (int)((pos - s0) / (blocks + extra));
        int block = (int)((pos - s0) - (uint32_t)tile * (blocks + extra)) - extra;
        if (E8 && block < 0) {
            if (++pos >= end) break;
            block = 0;
        }
        const int here = (int)min((uint32_t)(blocks - block), end - pos);
        const uint32_t tile_at = pos - block;   // the tile's first block among all
        pos += here;
        const int lo = max(a.window ? len - a.window : 0, 0) - (SINKS ? base : 0), first = (SINKS ? 0 : base) + (block << a.block), last = min(hi, first + (here << a.block));
        const int r = tile * BM + col;
        const int *table = a.c.table + (size_t)max(a.c.row(seq), 0) * a.c.max_pages;

        f4 acc[DL];
#pragma unroll
        for (int j = 0; j < DL; j++) acc[j] = f4{0, 0, 0, 0};
        float m = LOWEST, l = 0.0f;

        // This wave's keys of step n: 32 from first + (4 n + wave) * 32 on, two runs of 16. Lane 2 i + h holds where run h of
        // step 32 s + i begins, of the 32 steps at hand and of the 32 after them.
        auto fetch = [&](int n) {
            const int run = (first >> 4) + ((n + (lane >> 1)) * 4 + wave) * 2 + (lane & 1);
            return Runs<E8>(a.c, table, head, SINKS && run * 16 >= a.kept ? run + (base >> 4) : run, run * 16 < last,
                            run * 16 + 16 > lo || (SINKS && run * 16 < a.sinks));
        };
        Runs<E8> pg = fetch(0), pgn = fetch(32);
        u4 q[KS][NQ];
        const float q_scale = load_query<BF, NQ, KS, 32, 16, E8>(a.q + (size_t)seq * a.qstride + (size_t)(head * a.G + r) * dim * (F32 ? 4 : 2),
                                                        r < rows, g, dim, a.c2, q);
        // A lane's 16 bytes of an 8-bit row are the elements that its group has of two steps.
        const int kd = (col * dim + g * (16 / ES)) * ES, vd = (g * 4 * dim + col * DL) * ES;
        u4 kr[AHEAD][2][KS * ES / 2];         // run h, elements s * 32 + g * 8 of key col (8 bits: s * 64 + g * 16)
        uint32_t vr[AHEAD][8][DL * ES / 4];   // DL elements of the keys g * 4 + i (first four) and 16 + g * 4 + i
        float ks[AHEAD][2], vs[AHEAD][2];     // the runs' scales
        bool ok[AHEAD][2];                    // the runs are in pages
        auto run = [&](const uint8_t *pool, int n, int h) {
            return Run<true>(pool, pg, (n & 31) * 2 + h, min(last - (first + (n * 4 + wave) * 32 + h * 16), 16) * dim * ES);
        };
        auto load_k = [&](auto at, int n) {
            constexpr int A = decltype(at)::value;
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const Run<true> r = run(a.c.k, n, h);
                ok[A][h] = !pg.none((n & 31) * 2 + h);
                if constexpr (E8) ks[A][h] = pg.k_scale((n & 31) * 2 + h);
#pragma unroll
                for (int s = 0; s < KS * ES / 2; s++) kr[A][h][s] = r.load16(kd + s * 64, 0);
            }
        };
        auto load_v = [&](auto at, int n) {
            constexpr int A = decltype(at)::value;
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const Run<true> r = run(a.c.v, n, h);
                if constexpr (E8) vs[A][h] = pg.v_scale((n & 31) * 2 + h);
#pragma unroll
                for (int i = 0; i < 4; i++) {   // (elements past dim: others' in their place, in sums that are not written)
                    if constexpr (DL * ES == 4) {
                        vr[A][h * 4 + i][0] = r.load4(vd, i * dim * ES);
                    } else if constexpr (DL * ES == 8) {
                        const u2 y = r.load8(vd, i * dim * ES);
                        vr[A][h * 4 + i][0] = y[0];
                        vr[A][h * 4 + i][1] = y[1];
                    } else {
#pragma unroll
                        for (int w = 0; w < DL * ES / 4; w += 4) {
                            const u4 y = r.load16(vd + w * 4, i * dim * ES);
#pragma unroll
                            for (int k = 0; k < 4; k++) vr[A][h * 4 + i][w + k] = y[k];
                        }
                    }
                }
            }
        };
        // The K of the step AHEAD is loaded once this one's scores are there and its V once this one's is summed, into the same
        // registers.
        const int mine = first + wave * 32, steps = mine < last ? (last - mine + 127) / 128 : 0;
        auto step = [&](auto at, int n) {
            constexpr int A = decltype(at)::value;
            const int t0 = mine + n * 128;
            f4 s[2];
            if (dim < DP) {   // elements past dim: zeros, which the query's zeros keep
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int k = 0; k < KS * ES / 2; k++)
                        if ((k * 64 + g * 16) / ES >= dim) kr[A][h][k] = u4{0, 0, 0, 0};
            }
            u4 kf[2][KS];
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int k = 0; k < KS; k++) {
                    if constexpr (E8) kf[h][k] = eight_of<BF>(kr[A][h][k / 2][k % 2 * 2], kr[A][h][k / 2][k % 2 * 2 + 1], ks[A][h]);
                    else kf[h][k] = kr[A][h][k];
                }
            // A sum for each term, the smallest added first: the matrix cores round a sum after every 8 products, which loses small terms'
            // next to a large one's one by one. fp32 over fp16, error against 64 bits, so and with all terms in one sum: 500 keys of 64
            // 2.3e-7 to 2.5e-7 and 2.8e-7 to 4.2e-7, 32 sequences of 128 2.3e-7 and 3.3e-7 (us 6.67 and 6.63, 36.0 and 35.9)
#pragma unroll
            for (int t = NQ - 1; t >= 0; t--) {
                f4 part[2] = {f4{0, 0, 0, 0}, f4{0, 0, 0, 0}};
#pragma unroll
                for (int k = 0; k < KS; k++)
#pragma unroll
                    for (int h = 0; h < 2; h++) part[h] = mfma16<BF>(kf[h][k], q[k][t], part[h]);
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int i = 0; i < 4; i++) s[h][i] = t == NQ - 1 ? part[h][i] : s[h][i] + part[h][i];
            }
            float cs[2] = {q_scale, q_scale};   // what the runs' scores are multiplied by
            if constexpr (UNSCALED) {
                cs[0] = times_scale(q_scale, ks[A][0]);
                cs[1] = times_scale(q_scale, ks[A][1]);
            }
            const bool ok0 = ok[A][0], ok1 = ok[A][1], more = n + AHEAD < steps;
            if (more) {
                if (((n + AHEAD) & 31) == 0) {
                    pg = pgn;
                    pgn = fetch(n + AHEAD + 32);
                }
                load_k(at, n + AHEAD);
            }
            const int sinks = SINKS ? a.sinks : 0;
            if ((t0 < lo && t0 + 32 > sinks) || t0 + 32 > last || !ok0 || !ok1) {   // what is not to be seen: no score, and zeros for whatever V holds
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const int t = t0 + (i >> 2) * 16 + g * 4 + (i & 3);
                    const bool before = t < lo && t >= sinks;
                    if (before || t >= last || !(i < 4 ? ok0 : ok1)) s[i >> 2][i & 3] = LOWEST;
                    if (before) {
#pragma unroll
                        for (int w = 0; w < DL * ES / 4; w++) vr[A][i][w] = 0;
                    }
                }
            }
            float big = LOWEST;
            if constexpr (UNSCALED) {
                big = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])) * cs[0], fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])) * cs[1]);
                big = with_lane<32>(with_lane<16>(big, Max()), Max());
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++) big = fmaxf(big, s[i >> 2][i & 3]);
                big = with_lane<32>(with_lane<16>(big, Max()), Max()) * q_scale;
            }
            if (__any(big > m)) {
                const float now = fmaxf(m, big), f = __builtin_amdgcn_exp2f(m - reference(now));
                m = now;
                l *= f;
#pragma unroll
                for (int j = 0; j < DL; j++)
#pragma unroll
                    for (int i = 0; i < 4; i++) acc[j][i] *= f;
            }
            const float ref = reference(m);
            float w8[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                w8[i] = weight<NQ, SHIFT<WBF>>(s[i >> 2][i & 3], cs[i >> 2], ref);
                l += w8[i];
            }
            u4 pt[NP];
            if constexpr (NP == 3 && E8) split_whole(w8, pt);
            else split_weights<WBF, NQ, SHIFT<WBF>>(w8, pt);
#pragma unroll
            for (int j = 0; j < DL; j += 2) {
                u4 v0, v1;
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    if constexpr (E8) {   // two keys' elements j and j + 1 in a word, key by key
                        const uint32_t x = __builtin_amdgcn_perm(vr[A][2 * k + 1][j / 4], vr[A][2 * k][j / 4], j & 2 ? 0x07030602u : 0x05010400u);
                        v0[k] = two_of<true, false>(x, vs[A][k / 2]);
                        v1[k] = two_of<true, true>(x, vs[A][k / 2]);
                    } else {
                        v0[k] = pair<0>(vr[A][2 * k][j / 2], vr[A][2 * k + 1][j / 2]);
                        v1[k] = pair<1>(vr[A][2 * k][j / 2], vr[A][2 * k + 1][j / 2]);
                    }
                }
#pragma unroll
                for (int t = 0; t < NP; t++) {
                    acc[j] = mfma16<WBF>(v0, pt[t], acc[j]);
                    acc[j + 1] = mfma16<WBF>(v1, pt[t], acc[j + 1]);
                }
            }
            if (more) load_v(at, n + AHEAD);
        };
        using First = std::integral_constant<int, 0>;
        using Second = std::integral_constant<int, AHEAD - 1>;
        if (steps > 0) {
            load_k(First(), 0);
            load_v(First(), 0);
        }
        if (AHEAD > 1 && steps > 1) {
            load_k(Second(), 1);
            load_v(Second(), 1);
        }
        for (int n = 0; n < steps; n += AHEAD) {
            step(First(), n);
            if (AHEAD > 1 && n + 1 < steps) step(Second(), n + 1);
        }
        l = weights_sum<NQ, SHIFT<WBF>>(with_lane<32>(with_lane<16>(l, Sum()), Sum()));

        // the four waves' m, l and sums; lane (g, col) holds elements (g * 4 + i) * DL + j of head col
        if (g == 0) {
            lm[wave][col] = m;
            ll[wave][col] = l;
        }
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int j = 0; j < DL; j += 4)
                *reinterpret_cast<f4 *>(&lo_acc[wave][col][(g * 4 + i) * DL + j]) = f4{acc[j][i], acc[j + 1][i], acc[j + 2][i], acc[j + 3][i]};
        __syncthreads();
        const bool whole = here == blocks;
        // a group's part of a tile that it begins is its second in the workspace, of one that it goes on with its first
        const size_t part = (size_t)head * BM * 2 * a.target + (size_t)group * 2 + (group == (int)(tile_at / each) ? 1 : 0);
        uint8_t *out = a.out + (size_t)seq * a.ostride + (size_t)(head * a.G + tile * BM) * dim * (F32 ? 4 : 2);
        for (int e = tid; e < BM * (DP / 4); e += 256) {
            const int row = e / (DP / 4), d = e % (DP / 4) * 4;
            if (tile * BM + row >= rows || d >= dim) continue;
            float mm = LOWEST;
#pragma unroll
            for (int w = 0; w < 4; w++) mm = fmaxf(mm, lm[w][row]);
            float sum = 0.0f, x[4] = {0, 0, 0, 0};
#pragma unroll
            for (int w = 0; w < 4; w++) {
                const float f = __builtin_amdgcn_exp2f(lm[w][row] - reference(mm));
                sum += f * ll[w][row];
#pragma unroll
                for (int i = 0; i < 4; i++) x[i] += f * lo_acc[w][row][d + i];
            }
            if (whole) {
                const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
                for (int i = 0; i < 4; i++) x[i] = sum == 0.0f ? 0.0f : x[i] * inv;
                store4<F32, BF>(out + (size_t)row * dim * (F32 ? 4 : 2), d, x);
            } else {
                const size_t at = part + (size_t)row * 2 * a.target;
                if (d == 0) a.pml[at] = float2{mm, sum};
                *reinterpret_cast<f4 *>(a.po + at * dim + d) = f4{x[0], x[1], x[2], x[3]};
            }
        }
        __syncthreads();   // the next tile's sums go where these were
    }
}

// The parts of `together` rows of a tile a workgroup (a power of two), dim / 4 threads (rounded up to 16, 32 or 64) to a row
// and the 256 / that / together such groups of a row sharing its parts: each group finds the weights 2^(m - the largest m) for
// itself, in LDS. The sums' first loads, which need no weights, go out before them; what order they are added in, the lengths
// alone give.
template <bool F32, bool BF> __global__ __launch_bounds__(256) void attn_decode_join_kernel(AttnArgs a, int together) {
    constexpr int BM = DECODE_M, AHEAD = 16, MOST = DECODE_PARTS;
    const int tiles = (a.G + BM - 1) / BM, dim = a.c.dim, quads = dim / 4;
    const int w = quads <= 16 ? 16 : quads <= 32 ? 32 : 64, d = threadIdx.x % w, k = threadIdx.x / w, shares = 256 / w / together;
    const int blocks_per_head = (a.G + together - 1) / together;
    const int seq = blockIdx.x / (a.c.heads * blocks_per_head), rest = blockIdx.x - seq * (a.c.heads * blocks_per_head);
    const int head = rest / blocks_per_head, r0 = (rest - head * blocks_per_head) * together;   // (together divides 16: rows of one tile)
    Deal<true> deal(a, tiles);
    while (seq >= deal.group + 64) deal.next(a, tiles);
    int base;
    const int blocks = blocks_of(a, __builtin_amdgcn_readlane(deal.bl.len, seq - deal.group), base);
    const uint32_t at = deal.first_of(seq - deal.group) + (uint32_t)(r0 / BM) * (blocks + deal.extra) + deal.extra;
    const uint32_t from = at / deal.each, parts = (at + blocks - 1) / deal.each - from + 1;
    if (parts == 1 || parts > MOST || from + parts > (uint32_t)a.target) return;   // (one: written already; the others cannot be while the lengths stay)
    const int r = r0 + k % together, share = k / together;
    // the row's part in group from + n: the first is its group's second
    const size_t part0 = ((size_t)head * BM + min(r, a.G - 1) % BM) * 2 * a.target + (size_t)from * 2;
    auto part = [&](uint32_t n) { return part0 + (n ? n * 2 : 1); };
    const float *sums = a.po + min(d, quads - 1) * 4;
    f4 v[AHEAD];   // (a part that there is not: the last again, at weight 0)
#pragma unroll
    for (int i = 0; i < AHEAD; i++) v[i] = *reinterpret_cast<const f4 *>(sums + part(min((uint32_t)(share + i * shares), parts - 1)) * dim);

    __shared__ float wt[16][MOST];
    __shared__ f4 sx[256];
    float m = LOWEST, l = 0.0f;
    for (uint32_t n = d; n < parts; n += w) {
        const float2 ml = a.pml[part(n)];
        if (ml.y != 0.0f) m = fmaxf(m, ml.x);
    }
    m = over_lanes(m, w, Max());
    for (uint32_t n = d; n < parts; n += w) {
        const float2 ml = a.pml[part(n)];
        const float f = ml.y != 0.0f ? __builtin_amdgcn_exp2f(ml.x - reference(m)) : 0.0f;
        wt[k][n] = f;
        l += f * ml.y;
    }
    l = over_lanes(l, w, Sum());
    __syncthreads();
    f4 x = {0, 0, 0, 0};
#pragma unroll
    for (int n = 0; n < AHEAD; n++) {
        const int i = share + n * shares;
        const float f = i < (int)parts ? wt[k][i] : 0.0f;
#pragma unroll
        for (int j = 0; j < 4; j++) x[j] = __builtin_fmaf(f, v[n][j], x[j]);
    }
    for (uint32_t n = share + AHEAD * shares; n < parts; n += shares) {
        const f4 y = *reinterpret_cast<const f4 *>(sums + part(n) * dim);
#pragma unroll
        for (int j = 0; j < 4; j++) x[j] = __builtin_fmaf(wt[k][n], y[j], x[j]);
    }
    sx[threadIdx.x] = x;
    __syncthreads();
    if (share || d >= quads || r >= a.G) return;
    for (int g = 1; g < shares; g++)
#pragma unroll
        for (int j = 0; j < 4; j++) x[j] += sx[(g * together + k) * w + d][j];
    float o[4];
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int j = 0; j < 4; j++) o[j] = l == 0.0f ? 0.0f : x[j] * inv;
    store4<F32, BF>(a.out + (size_t)seq * a.ostride + (size_t)(head * a.G + r) * dim * (F32 ? 4 : 2), d * 4, o);
}

// ---- a tile of prompt rows -------------------------------------------------------------------------------------------------------
// A workgroup of four waves takes 128 rows, 32 a wave, against its keys, 64 at a time in LDS, where the next 64 go while these
// are multiplied: straight from memory (a wave's instruction brings 64 pieces of 16 bytes to consecutive places; which piece,
// each lane says). K and V lie as in the pools, key after key, but the pieces of a key are exchanged among themselves, so that
// the lanes of a read (16 keys' pieces of K; of V, the 4 keys of a transposing read, 32 elements of each) fall on different
// banks: piece c of key t is at c ^ k_turn(t), c ^ v_turn(t).
//
// Keys that a row does not see have weight 0, and 0 times an infinity or NaN is not 0: V rows that no row sees are zeros in LDS,
// and so are such elements of keys that only some rows see; where there were any, they are added to those rows at the end.
//
// Bound by the matrix cores and their power: 16384 tokens, 32 heads of 128 over 4, fp16, 2.19 ms, 1005 TFLOP/s counted causally. The
// waves of a SIMD together keep the matrix cores busy for 57% of the cycles, at 1.9 to 2 GHz; a large library product, busy for
// 70%, is clocked at 1.4 and gives 1320. Two workgroups a CU: with 64 rows a wave, which halves the reads of LDS, only one
// fits, and the exponentials of one wave no longer pass under the products of another: 2.94 ms where this had 2.25. Tiles of
// 256 rows in eight waves: within 2%.
template <int DP> __device__ constexpr int k_turn(int t) { return DP == 64 ? t >> 1 & 7 : t & 15; }
// (8 bits: the last bit too, for the writes to LDS, see settle)
template <int DP, bool E8> __device__ constexpr int v_turn(int t) { return DP == 64 ? (t >> 1 & 1) * (E8 ? 5 : 4) : (t & 3) * 4 + (E8 ? t & 1 : 0); }

// 64 pieces of 16 bytes from a run into LDS: lane i's, at `lane_offset` + `offset` from the run's first row, to lds + 16 i;
// zeros past the run's end
__device__ void run_to_lds(u4 r, int lane_offset, int offset, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %3\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, %2 offen lds" ::"v"(lane_offset), "s"(r), "s"(offset), "s"(lds) : "memory");
}
using s4 = short __attribute__((ext_vector_type(4)));
// of 4 keys, one element each: lane i of 16 gives where 4 elements of key i / 4 are and takes element i of the 16
__device__ u2 transposed(uint32_t lds) {
    return __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<__attribute__((address_space(3))) s4 *>(lds)));
}

template <bool BF, int NQ, int DP, bool E8 = false, bool SINKS = false>
__global__ __launch_bounds__(256, E8 && NQ == 2 && DP == 64 ? 3 : prompt_per_cu(NQ, DP)) void attn_prompt_kernel(AttnArgs a) {
    constexpr bool UNSCALED = E8 && !BF;                     // (see below)
    constexpr bool SHORT = E8 && NQ == 2;                    // of registers: what can be computed anew is not kept
    constexpr int NB = DP == 64 && !E8 ? 3 : 2;              // steps of keys in LDS
    constexpr int ES = E8 ? 1 : 2;                           // bytes of an element in the pools
    constexpr int KS = DP / 16, DT = DP / 32, CH = DP / 8;   // CH: pieces of a key
    constexpr int NI = CH / 4;                               // a wave's instructions for its 16 keys
    constexpr int ROWS = 64 / CH;                            // keys of one
    constexpr uint32_t TILE = PN * DP * 2;                   // bytes of K, or V, of a step
    constexpr bool F32 = NQ > 1;
    constexpr int BY = SHIFT<BF> - LAG<BF, NQ>;              // weights are 2^BY p
    __shared__ __attribute__((aligned(1024))) uint8_t lds[2 * NB * TILE];   // K of NB steps, V of them
    __shared__ int odd;                                      // elements of V were left out
    // UNSCALED: of each step's four runs the scales of K and of V, and the exponents of the latter (a wave writes its run's)
    __shared__ __attribute__((aligned(16))) float run_ks[UNSCALED ? NB : 1][4], run_vs[UNSCALED ? NB : 1][4], run_ve[UNSCALED ? NB : 1][4];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 31, half = lane >> 5;
    const int head = blockIdx.x % a.c.heads, item = blockIdx.x / a.c.heads;
    const int chunk = chunk_of(a);
    Part p;
    if (!part_of<false>(a, item, chunk, p)) return;
    const bool whole = chunk == 1 << 30;
    const int tile = p.s.tiles - 1 - p.tile;   // the tiles that see most keys first
    const int rows = min(PM, p.s.n * a.G - tile * PM);
    const int back = p.s.len - p.s.n;          // query i stands at back + i
    const int pos_lo = back + tile * PM / a.G, pos_hi = back + (tile * PM + rows - 1) / a.G;
    const int see_lo = a.window ? max(0, pos_lo - a.window + 1) : 0, see_hi = pos_hi + 1;   // keys that some row sees
    int first = (SINKS ? 0 : p.s.base) + (whole ? 0 : p.chunk * chunk);
    int last = SINKS ? see_hi - p.s.base : see_hi;
    if (!whole) last = min(last, first + chunk);
    // SINKS: keys are numbered without the `left` that lie behind the first a.kept and before what the tile, or the part, sees
    // of the window (the parts' share them out without p.s.base of them)
    int left = 0;
    if constexpr (SINKS) {
        const int windows = max(a.kept + p.s.base, see_lo & ~(PN - 1)) - p.s.base;   // the tile's first, as parts number them
        if (first < a.kept) {
            left = p.s.base + windows - a.kept;
            last = max(min(last, a.kept), last - (windows - a.kept));
        } else {
            left = p.s.base;
            first = max(first, windows);
        }
    } else {
        first = max(first, see_lo & ~(PN - 1));
    }
    auto at_key = [&](int n) { return SINKS && n >= a.kept ? n + left : n; };   // the token that key n is
    // every row sees all sinks, and none of the keys behind them in their last step, which are then not brought: zeros
    const bool sinks_alone = SINKS && see_lo >= a.kept;
    const int sinks_end = SINKS ? __builtin_amdgcn_readfirstlane(sinks_alone ? min(a.sinks, last) : last) : 0;
    auto in_sight = [&](int n) { return SINKS && n < a.kept ? sinks_end : last; };   // the end of the keys to bring from n on
    const int *table = a.c.table + (size_t)max(a.c.row(p.b), 0) * a.c.max_pages;
    const int dim = a.c.dim;

    const int r = min(tile * PM + wave * 32 + col, tile * PM + rows - 1);   // lanes past the last row repeat it
    const int query = r / a.G, pos = back + query, from = a.window ? pos - a.window + 1 : 0;
    const size_t qoff = (size_t)(head * a.G + r - query * a.G) * dim * (F32 ? 4 : 2);
    u4 q[KS][NQ];
    const float cs = load_query<BF, NQ, KS, 16, 32>(a.q + (size_t)(p.s.t0 + query) * a.qstride + qoff, true, half, dim, a.c2, q);
    const int wpos_lo = __builtin_amdgcn_readlane(pos, 0), wpos_hi = __builtin_amdgcn_readlane(pos, 31);
    const int from_hi = a.window ? pos_hi - a.window + 1 : 0, wfrom_hi = a.window ? wpos_hi - a.window + 1 : 0;
    const bool idle = wave * 32 >= rows;

    f16v acc[DT];
#pragma unroll
    for (int j = 0; j < DT; j++)
#pragma unroll
        for (int i = 0; i < 16; i++) acc[j][i] = 0.0f;
    float m = LOWEST, l = 0.0f;
    // UNSCALED: K and V go into the products as the numbers are, in fp16, which takes fp32 queries in two terms, not bf16's three (4096 tokens, 32
    // heads of 128 over 8: 298 us with two, 458 with three). K's scales are factors of the scores. V's are factors of the weights, and as fp16
    // has not the range for both, the sums have a reference of their own: m2, the maximum of score plus exponent of the run's scale, which
    // keeps the bits of what weighs most in a row's sum, whatever the scales. by_scale is 2^(BY + m - m2).
    float m2 = LOWEST, by_scale = 1 << (BY & 31);

    // where 64 runs of 16 keys from run `pb` on begin, one per lane, and the 64 after them
    auto fetch = [&](int u) {
        const int t = at_key(u * 16);
        return Runs<E8>(a.c, table, head, t >> 4, u * 16 < last, t + 16 > see_lo || (SINKS && t < a.sinks));
    };
    int pb = first >> 4;
    Runs<E8> pg = fetch(pb + lane), pgn = fetch(pb + 64 + lane);

    // This wave brings run `wave` of each step: key n * ROWS + lane / CH of it and place lane % CH of that key by instruction n
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)lds;
    constexpr int VN = DP == 256 ? 2 : 1;   // instructions after which V's pieces are exchanged the same way again
    int k_from[NI], v_from[VN];
#pragma unroll
    for (int n = 0; n < NI; n++) {
        const int t = n * ROWS + lane / CH, c = lane % CH ^ k_turn<DP>(t);
        k_from[n] = c * 8 < dim ? (t * dim + c * 8) * 2 : 0x40000000;   // (elements past dim: past the run's end)
    }
#pragma unroll
    for (int n = 0; n < VN; n++) {
        const int t = n * ROWS + lane / CH, c = lane % CH ^ v_turn<DP, E8>(t);
        v_from[n] = c * 8 < dim ? (t * dim + c * 8) * 2 : 0x40000000;
    }
    // the window of runs moved on to the one from t0 on: its number there; `holes` gets which of the step's four are in no page
    auto seek = [&](int t0, int &none) {
        int u0 = (t0 >> 4) - pb;
        if (u0 >= 64) {
            pb += 64;
            u0 -= 64;
            pg = pgn;
            pgn = fetch(pb + 64 + lane);
        }
        none = (int)(__ballot(pg.hi < 0) >> u0 & 15);
        return u0 + wave;
    };
    auto bytes_of = [&](int n) { return __builtin_amdgcn_readfirstlane((SINKS ? max(min(in_sight(n) - n - wave * 16, 16), 0) : min(last - n - wave * 16, 16)) * dim * ES); };
    // brings the keys from t0 on to LDS; which of their four runs are in no page
    auto load = [&](int t0, int buf) {
        int none;
        const int u = seek(t0, none);
        const u4 k = run_of(a.c.k, pg, u, bytes_of(t0)), v = run_of(a.c.v, pg, u, bytes_of(t0));
        const uint32_t to = lds0 + buf * TILE + wave * NI * 1024;
#pragma unroll
        for (int n = 0; n < NI; n++) run_to_lds(k, k_from[n], 0, to + n * 1024);
#pragma unroll
        for (int n = 0; n < NI; n++) run_to_lds(v, v_from[n % VN], n / VN * VN * ROWS * dim * 2, to + NB * TILE + n * 1024);
        return none;
    };
    // 8 bits: the next step's keys wait in registers, 16 bytes of key n * ROWS8 + t8 in each, and are turned into 16 bits on their way
    // to LDS, where they lie as a 16-bit cache's do: at the beginning of a step, with the step after it asked for then; or, SHARED, K there and
    // V at the end, in the same registers, with V asked for at the beginning and K at the end, where both do not fit. us, so and SHARED, fp32, 32 heads
    // over 8: of 256, 2048 tokens, 207 and 181, of 128, 4096 tokens, 267 and 271.
    constexpr bool SHARED = NQ == 2 && DP == 256;
    //
    // A lane has 16 bytes, two pieces, of a key. Eight lanes in a row have 4 such of two keys whose pieces are exchanged differently in the last
    // bit, so that their first pieces, and their second ones, fall on different banks.
    constexpr int CH8 = DP / 16, ROWS8 = 64 / CH8, R8 = E8 ? DP / 64 : 1;
    const int c8 = DP == 64 ? lane & 3 : DP == 128 ? (lane & 3) + (lane >> 3 & 1) * 4 : (lane & 3) + (lane >> 3 & 3) * 4;
    const int t8 = DP == 64 ? (lane >> 3 & 1) + (lane >> 2 & 1) * 2 + (lane >> 4) * 4 : DP == 128 ? (lane >> 2 & 1) + (lane >> 4) * 2 : (lane >> 2 & 1) + (lane >> 5) * 2;
    u4 x8[SHARED ? 1 : 2][R8];
    float scale8[SHARED ? 1 : 2];
    auto load8 = [&](auto is_v, int t0, int u) {
        const int from = c8 * 16 < dim ? t8 * dim + c8 * 16 : 0x40000000;   // (elements past dim: past the run's end)
        const Run<false> r(is_v ? a.c.v : a.c.k, pg, u, bytes_of(t0));
        constexpr int W = !SHARED && is_v;
#pragma unroll
        for (int n = 0; n < R8; n++) x8[W][n] = r.load16(from, n * ROWS8 * dim);
        scale8[W] = is_v ? pg.v_scale(u) : pg.k_scale(u);
    };
    auto settle = [&](auto is_v, int buf) {
        constexpr int W = !SHARED && is_v;
        const float scale = scale8[W];
#pragma unroll
        for (int n = 0; n < R8; n++) {
            const int t = n * ROWS8 + t8, c = c8 * 2, turn = is_v ? v_turn<DP, E8>(t) : k_turn<DP>(t);
            uint8_t *key = lds + ((is_v ? NB : 0) + buf) * TILE + (wave * 16 + t) * DP * 2;
            *reinterpret_cast<u4 *>(key + (c ^ turn) * 16) = eight_of<BF>(x8[W][n][0], x8[W][n][1], scale);
            *reinterpret_cast<u4 *>(key + (c + 1 ^ turn) * 16) = eight_of<BF>(x8[W][n][2], x8[W][n][3], scale);
        }
        if (UNSCALED && lane == 0) {
            if (is_v) {
                run_vs[buf][wave] = scale;
                run_ve[buf][wave] = (float)((int)(__float_as_uint(scale) >> 23 & 255) - 127);
            } else {
                run_ks[buf][wave] = scale;
            }
        }
    };
    using K8 = std::false_type;
    using V8 = std::true_type;
    int u8 = 0;   // the number of the run whose K is in registers
    auto load_k8 = [&](int t0) {
        int none;
        u8 = seek(t0, none);
        load8(K8(), t0, u8);
        return none;
    };
    auto some_hidden = [&](int t0) { return (t0 + PN > pos_lo + 1 || t0 < from_hi) && !(sinks_alone && t0 < a.kept); };   // of the step's keys, from some row
    // V of the step from t0 on, where some row does not see all of its keys: zeros for what none sees or must not be multiplied
    // by 0
    auto clean = [&](int t0, int buf) {
        constexpr uint32_t E = BF ? 0x7f80u : 0x7c00u;   // an exponent of ones
        bool left = false;
#pragma unroll 1
        for (int i = tid; i < PN * CH; i += 256) {
            u4 *at = reinterpret_cast<u4 *>(lds + (NB + buf) * TILE) + i;
            u4 x = *at;
            const bool none = t0 + i / CH < see_lo && !(SINKS && t0 + i / CH < a.sinks);
            bool write = none;
#pragma unroll
            for (int w = 0; w < 4; w++) {
                const uint32_t bad = ((x[w] & E) == E ? 0xffffu : 0) | ((x[w] >> 16 & E) == E ? 0xffff0000u : 0);
                left |= bad && !none;
                write |= bad != 0;
                x[w] = none ? 0 : x[w] & ~bad;
            }
            if (write) *at = x;
        }
        if (left) odd = 1;
    };
    auto arrived = [&](bool all) {   // the next step's keys are in LDS (all: of every step asked for), then those that the other waves brought
        if (all) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        else asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NB - 2) * 2 * NI) : "memory");   // (what was asked for last comes last)
        __syncthreads();
    };
    // reads: K piece (k * 2 + half) of key h * 32 + col; of V, as transposed() takes them, 4 elements of key u * 16 + r * 8 +
    // half * 4 + lane % 16 / 4
    constexpr int KA = KS < 8 ? KS : 8, VA = DT < 4 ? DT : 4;   // (addresses that are not another's at a constant distance)
    // Reads of K, and fragments of V, under way ahead of the products: as the compiler left them, each product waited for its own. Where
    // registers are SHORT, more than they have room for would be none (the compiler then drops the order): us with these and with none, 4096 tokens,
    // heads of 128, 267 and 294, of 64 166 and 172, 2048 of 256 181 and 232, a prompt's last 64 of 8001 33.2 and 38.1. In a 16-bit cache's
    // kernels, 8192 tokens: heads of 256, fp16 1330 and 1534, fp32 2017 and 2363; of 128 555 and 563.
    constexpr int AHEAD_K = SHORT ? 4 : 6, AHEAD_V = !SHORT ? 4 : DP == 256 ? 1 : 2;
    uint32_t k_at[KA], v_at[VA];
#pragma unroll
    for (int k = 0; k < KA; k++) k_at[k] = lds0 + col * DP * 2 + ((k * 2 + half) ^ k_turn<DP>(col)) * 16;
#pragma unroll
    for (int j = 0; j < VA; j++) {
        const int t = half * 4 + (lane & 15) / 4, e = j * 32 + (lane >> 4 & 1) * 16 + (lane & 3) * 4;
        v_at[j] = lds0 + NB * TILE + t * DP * 2 + ((e / 8) ^ v_turn<DP, E8>(t)) * 16 + e % 8 * 2;
    }
    if (tid == 0) odd = 0;
    __syncthreads();
    int holes = 0, buf = 0;   // holes: four bits a step, this one's lowest
    if constexpr (E8) {
        if (first < last) {
            holes = load_k8(first);
            if (!SHARED) load8(V8(), first, u8);
            settle(K8(), 0);
            if (SHARED) load8(V8(), first, u8);
            settle(V8(), 0);
            if (first + PN < last) {
                holes |= load_k8(first + PN) << 4;
                if (!SHARED) load8(V8(), first + PN, u8);
            }
        }
        __syncthreads();
    } else {
#pragma unroll
        for (int n = 0; n < NB - 1; n++)
            if (first + n * PN < last) holes |= load(first + n * PN, n) << 4 * n;
        arrived(true);
    }
    for (int n0 = first; n0 < last; n0 += PN) {
        const int t0 = at_key(n0);
        const bool more = n0 + (NB - 1) * PN < last;
        if constexpr (E8) {
            if (more) {
                settle(K8(), buf ^ 1);
                if constexpr (SHARED) {
                    load8(V8(), n0 + PN, u8);
                } else {
                    settle(V8(), buf ^ 1);
                    if (n0 + 2 * PN < last) {
                        holes |= load_k8(n0 + 2 * PN) << 8;
                        load8(V8(), n0 + 2 * PN, u8);
                    }
                }
            }
        } else {
            if (more) holes |= load(n0 + (NB - 1) * PN, buf == 0 ? NB - 1 : buf - 1) << 4 * (NB - 1);
        }
        if (some_hidden(t0)) {
            clean(t0, buf);
            __syncthreads();
        }
        if (!(idle || t0 > wpos_hi || (a.window && t0 + PN <= wpos_lo - a.window + 1 && !(SINKS && t0 < a.sinks)))) {
            // (kept as they are, so that what is added to them goes into the instructions; where registers are short, each is the first with
            // its piece's number exchanged into it)
            uint32_t k_now[KA], v_now[VA];
#pragma unroll
            for (int k = 0; k < KA; k++) {
                k_now[k] = SHORT ? (k_at[0] + buf * TILE) ^ k * 32 : k_at[k] + buf * TILE;
                if constexpr (!SHORT) asm volatile("" : "+v"(k_now[k]));
            }
#pragma unroll
            for (int j = 0; j < VA; j++) {
                v_now[j] = SHORT ? (v_at[0] + buf * TILE) ^ j * 64 : v_at[j] + buf * TILE;
                if constexpr (!SHORT) asm volatile("" : "+v"(v_now[j]));
            }
            f16v s[2];
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int i = 0; i < 16; i++) s[h][i] = 0.0f;
#pragma unroll
            for (int k = 0; k < KS; k++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const u4 kf = *reinterpret_cast<__attribute__((address_space(3))) const u4 *>(k_now[k % KA] + h * 32 * DP * 2 + k / KA * 256);
#pragma unroll
                    for (int t = 0; t < NQ; t++) s[h] = mfma32<BF>(kf, q[k][t], s[h]);
                }
            // (with three terms the products are long enough)
            if constexpr (NQ < 3) {
                __builtin_amdgcn_sched_group_barrier(0x100, AHEAD_K, 0);
#pragma unroll
                for (int i = 0; i < 2 * KS - AHEAD_K; i++) {
                    __builtin_amdgcn_sched_group_barrier(0x8, NQ, 0);
                    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                }
                __builtin_amdgcn_sched_group_barrier(0x8, AHEAD_K * NQ, 0);
            }
            if (t0 + PN > wpos_lo + 1 || t0 < wfrom_hi) {
                const int to = pos - t0 - half * 4, since = from - t0 - half * 4, sinks = SINKS ? a.sinks - t0 - half * 4 : 0;
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        const int t = h * 32 + i / 4 * 8 + (i & 3);
                        if (t > to || (t < since && !(SINKS && t < sinks))) s[h][i] = LOWEST;
                    }
            }
            if (holes & 15) {
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int i = 0; i < 16; i++)
                        if (holes >> (h * 2 + i / 8) & 1) s[h][i] = LOWEST;
            }
            u4 pt[4][NQ];
            if constexpr (UNSCALED) {
                auto four = [&](const float (&x)[4]) { return *reinterpret_cast<const f4 *>(x); };
                const f4 k4 = four(run_ks[buf]), v4 = four(run_vs[buf]), e4 = four(run_ve[buf]);
                float big = LOWEST, big2 = LOWEST, csr[4];
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    float x = LOWEST;
#pragma unroll
                    for (int i = 0; i < 8; i++) x = fmaxf(x, s[u >> 1][(u & 1) * 8 + i]);
                    csr[u] = times_scale(cs, k4[u]);
                    x *= csr[u];
                    big = fmaxf(big, x);
                    big2 = fmaxf(big2, x + e4[u]);
                }
                big = with_lane<32>(big, Max());
                big2 = with_lane<32>(big2, Max());
                if (__any(big > m + LAG<BF, NQ> || big2 > m2 + LAG<BF, NQ>)) {
                    const float now = fmaxf(m, big), now2 = fmaxf(m2, big2), f = __builtin_amdgcn_exp2f(m2 - reference(now2));
                    l *= __builtin_amdgcn_exp2f(m - reference(now));
                    m = now;
                    m2 = now2;
                    by_scale = __builtin_amdgcn_exp2f(BY + (reference(m) - reference(m2)));
#pragma unroll
                    for (int j = 0; j < DT; j++)
#pragma unroll
                        for (int i = 0; i < 16; i++) acc[j][i] *= f;
                }
                const float ref = reference(m);
                // Below a `by` of 2^100, p's that fp32 has lost would be less than 2^-26 as weights, below fp16's range. Above it none is over
                // 2^-85, which l does not show, and as fp32 may have lost what is to be a large weight, the exponents take the power of two.
                float by[4];
#pragma unroll
                for (int u = 0; u < 4; u++) by[u] = by_scale * v4[u];
                if (__any(fmaxf(fmaxf(by[0], by[1]), fmaxf(by[2], by[3])) > 0x1p100f)) {
#pragma unroll
                    for (int u = 0; u < 4; u++) {
                        const bool far = by[u] > 0x1p100f;
                        const float up = e4[u] + (BY - 100 + (ref - reference(m2)));
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            const float x = s[u >> 1][(u & 1) * 8 + i];
                            s[u >> 1][(u & 1) * 8 + i] = far ? __builtin_fmaf(x, csr[u], up) : x;
                        }
                        csr[u] = far ? 1.0f : csr[u];
                        by[u] = far ? 0x1p100f : by[u];
                    }
                }
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    h8 v, w;
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u >> 1][(u & 1) * 8 + i], csr[u], -ref));
                        l += x;
                        v[i] = static_cast<_Float16>(__builtin_fmaf(x, by[u], 0.0f));
                        if constexpr (NQ == 2) w[i] = static_cast<_Float16>(__builtin_fmaf(x, by[u], -static_cast<float>(v[i])));
                    }
                    pt[u][0] = __builtin_bit_cast(u4, v);
                    if constexpr (NQ == 2) pt[u][1] = __builtin_bit_cast(u4, w);
                }
            } else {
                float big = LOWEST;
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int i = 0; i < 16; i++) big = fmaxf(big, s[h][i]);
                big = with_lane<32>(big, Max()) * cs;
                if (__any(big > m + LAG<BF, NQ>)) {
                    const float now = fmaxf(m, big), f = __builtin_amdgcn_exp2f(m - reference(now));
                    m = now;
                    l *= f;
#pragma unroll
                    for (int j = 0; j < DT; j++)
#pragma unroll
                        for (int i = 0; i < 16; i++) acc[j][i] *= f;
                }
                const float ref = reference(m);
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    float w8[8];
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        w8[i] = weight<NQ, BY>(s[u >> 1][(u & 1) * 8 + i], cs, ref);
                        l += w8[i];
                    }
                    split_weights<BF, NQ, BY>(w8, pt[u]);
                }
            }
#pragma unroll
            for (int u = 0; u < 4; u++)
#pragma unroll
                for (int j = 0; j < DT; j++) {
                    const uint32_t at = v_now[j % VA] + u * 16 * DP * 2 + j / VA * 256;
                    const u2 v0 = transposed(at), v1 = transposed(at + 8 * DP * 2);
                    const u4 vf = {v0[0], v0[1], v1[0], v1[1]};
#pragma unroll
                    for (int t = 0; t < NQ; t++) acc[j] = mfma32<BF>(vf, pt[u][t], acc[j]);
                }
            if constexpr (NQ < 3) {
                __builtin_amdgcn_sched_group_barrier(0x100, 2 * AHEAD_V, 1);
#pragma unroll
                for (int i = 0; i < 4 * DT - AHEAD_V; i++) {
                    __builtin_amdgcn_sched_group_barrier(0x8, NQ, 1);
                    __builtin_amdgcn_sched_group_barrier(0x100, 2, 1);
                }
                __builtin_amdgcn_sched_group_barrier(0x8, AHEAD_V * NQ, 1);
            }
        }
        holes >>= 4;
        buf = buf == NB - 1 ? 0 : buf + 1;
        if constexpr (E8) {
            if constexpr (SHARED) {
                if (more) settle(V8(), buf);
                if (n0 + 2 * PN < last) holes |= load_k8(n0 + 2 * PN) << 4;
            }
            __syncthreads();
        } else {
            arrived(!more);
        }
    }
    l = with_lane<32>(l, Sum());
    if constexpr (!UNSCALED) l = weights_sum<NQ, BY>(l);

    if (wave * 32 + col >= rows) return;
    // acc[j][i] is element j * 32 + i / 4 * 8 + half * 4 + i % 4
    if (odd) {   // what was left out, for the keys of the steps that were looked through (an infinity or NaN, whatever its weight)
        for (int n = SINKS ? first : max(first, see_lo); n < last; n++) {
            const int t = at_key(n), t0 = t & ~(PN - 1);
            if (!some_hidden(t0) || t > pos || (t < from && !(SINKS && t < a.sinks))) continue;
            const int page = table[t >> a.c.shift];
            if (page < 0 || page >= a.c.npages) continue;
            const size_t at = a.c.row_at(page, head, t & ((1 << a.c.shift) - 1));
            const uint8_t *row = a.c.v + at * dim * ES;
            const float scale = E8 && !UNSCALED ? a.c.vs[at >> 4] : 1.0f;
            int lane_d = half * 4;
            asm volatile("" : "+v"(lane_d));   // (or what depends on it is computed ahead of the loop, for all elements)
#pragma unroll
            for (int j = 0; j < DT; j++) {
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    using T = std::conditional_t<BF, __bf16, _Float16>;
                    const int d = j * 32 + i / 4 * 8 + lane_d + (i & 3);
                    float v = 0.0f;
                    if constexpr (E8) v = d < dim ? __builtin_amdgcn_cvt_f32_fp8(row[d], 0) * scale : 0.0f;
                    else v = d < dim ? static_cast<float>(*reinterpret_cast<const T *>(row + d * 2)) : 0.0f;
                    if (!(fabsf(v) < INFINITY)) acc[j][i] += v;
                }
                __builtin_amdgcn_sched_barrier(0);   // (not all of the row's loads at once, for which there are no registers)
            }
        }
    }
    const bool done = p.chunks == 1;
    const size_t at = ((size_t)item * a.c.heads + head) * PM + wave * 32 + col;
    float inv = !done ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
    if constexpr (UNSCALED) inv *= __builtin_amdgcn_exp2f(reference(m2) - reference(m) - BY);   // the sums relative to m
    if (!done && half == 0) a.pml[at] = float2{m, l};
    uint8_t *row = a.out + (size_t)(p.s.t0 + query) * a.ostride + qoff;
#pragma unroll
    for (int j = 0; j < DT; j++)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const int d = j * 32 + i * 2 + half * 4;
            if (d >= dim) continue;
            float x[4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                x[k] = acc[j][i + k] * inv;
                if (done && l == 0.0f) x[k] = 0.0f;
            }
            if (done) store4<F32, BF>(row, d, x);
            else *reinterpret_cast<f4 *>(a.po + at * dim + d) = f4{x[0], x[1], x[2], x[3]};
        }
}

// ---- parts joined ------------------------------------------------------------------------------------------------------------
// out of a prompt's row = sum over its parts of 2^(m of the part - the largest m) * (the part's sum), over the same of l: the
// weights first, in LDS, then the sums in the order of the parts, dim / 4 threads (rounded up to 16, 32 or 64) a row, as many
// rows as that gives a workgroup at a time, of `blocks` workgroups to a tile in turn.
template <bool F32, bool BF> __global__ __launch_bounds__(256) void attn_join_kernel(AttnArgs a, int blocks) {
    const int quads = a.c.dim / 4, w = quads <= 16 ? 16 : quads <= 32 ? 32 : 64;   // threads per row
    const int d = threadIdx.x % w, k = threadIdx.x / w, groups = 256 / w;
    const int head = blockIdx.x % a.c.heads, block = blockIdx.x / a.c.heads % blocks;
    const int chunk = chunk_of(a);
    Part p;
    if (!part_of<true>(a, blockIdx.x / a.c.heads / blocks, chunk, p) || p.chunks == 1) return;   // (one part: written already)
    const uint32_t first = p.first + (uint32_t)p.tile * (uint32_t)p.chunks;
    const int tile = p.s.tiles - 1 - p.tile;
    const int rows = min(PM, p.s.n * a.G - tile * PM);
    if (p.chunks > MOST_PARTS + 1 || (size_t)first + p.chunks > (size_t)a.items) return;   // (starts out of order)
    __shared__ float wt[16][MOST_PARTS + 1];
    float *f = wt[k];
    for (int row0 = block * groups; row0 < rows; row0 += blocks * groups) {
        const int row = row0 + k;
        const size_t at = ((size_t)first * a.c.heads + head) * PM + min(row, rows - 1), step = (size_t)a.c.heads * PM;
        float m = LOWEST;
        for (int c = d; c < p.chunks; c += w) {
            const float2 ml = a.pml[at + c * step];
            if (ml.y != 0.0f) m = fmaxf(m, ml.x);
        }
        m = over_lanes(m, w, Max());
        float l = 0.0f;
        for (int c = d; c < p.chunks; c += w) {
            const float2 ml = a.pml[at + c * step];
            const float x = ml.y != 0.0f ? __builtin_amdgcn_exp2f(ml.x - reference(m)) : 0.0f;
            f[c] = x;
            l += x * ml.y;
        }
        l = over_lanes(l, w, Sum());
        __syncthreads();
        if (d < quads && row < rows) {
            f4 x = {0, 0, 0, 0};
            const float *y = a.po + at * a.c.dim + d * 4;
            const size_t pitch = step * a.c.dim;
#pragma unroll 8
            for (int c = 0; c < p.chunks; c++) {
                const f4 v = *reinterpret_cast<const f4 *>(y + c * pitch);
#pragma unroll
                for (int i = 0; i < 4; i++) x[i] = __builtin_fmaf(f[c], v[i], x[i]);
            }
            const int r = tile * PM + row, query = r / a.G;
            float o[4];
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
            for (int i = 0; i < 4; i++) o[i] = l == 0.0f ? 0.0f : x[i] * inv;
            store4<F32, BF>(a.out + (size_t)(p.s.t0 + query) * a.ostride + (size_t)(head * a.G + r - query * a.G) * a.c.dim * (F32 ? 4 : 2), d * 4, o);
        }
        __syncthreads();   // the next rows' weights go where these were
    }
}

}  // namespace
