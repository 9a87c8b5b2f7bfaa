// Shared by the paged key-value cache's translation units: the cache as the kernels see it, which part of a call a workgroup
// takes, and the matrix-core types. A page holds, per K/V head, `page` token rows of dim elements, so a (page, head) is one
// contiguous run and 16 tokens (the least page) never span two pages. Elements are of 16 bits, or of 8 with a scale for every 16 tokens.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "es_hip_quant.h"

namespace esq {

struct KvView {
    uint8_t *k, *v;
    const float *ks, *vs;   // an 8-bit cache's scales
    const int *table, *len, *seq;
    int heads, dim, shift;   // page = 1 << shift tokens
    int npages, rows, max_pages;

    __device__ int row(int b) const {   // the table row of the call's sequence b, or -1
        const int r = seq ? seq[b] : b;
        return r >= 0 && r < rows ? r : -1;
    }
    __device__ int tokens(int b) const {   // never more than the table has room for
        const int r = row(b);
        if (r < 0) return 0;
        const int n = len[r], most = max_pages << shift;
        return n < 0 ? 0 : n < most ? n : most;
    }
    // token rows from a pool's start to (page, head, token): times dim the element, and an 8-bit cache's scale every 16th
    __device__ size_t row_at(int page, int head, int token) const { return (((size_t)page * heads + head) << shift) + token; }
};

// A view checked on the host; records the reason and returns ES_HIP_EINVAL where kv cannot be used for nseq sequences.
int kv_check(const es_hip_kv *kv, int nseq, KvView &v, bool paged);

using h8 = _Float16 __attribute__((ext_vector_type(8)));
using b8 = __bf16 __attribute__((ext_vector_type(8)));
using f4 = float __attribute__((ext_vector_type(4)));
using f16v = float __attribute__((ext_vector_type(16)));
using u2 = uint32_t __attribute__((ext_vector_type(2)));
using u4 = uint32_t __attribute__((ext_vector_type(4)));

// f of a lane's value and that of the lane D (16 or 32) away, the same on both sides
template <int D, class F> __device__ float with_lane(float x, F f) {
    static_assert(D == 16 || D == 32);
    const uint32_t b = __float_as_uint(x);
    if constexpr (D == 32) {
        const auto r = __builtin_amdgcn_permlane32_swap(b, b, false, false);
        return f(__uint_as_float(r[0]), __uint_as_float(r[1]));
    } else {
        const auto r = __builtin_amdgcn_permlane16_swap(b, b, false, false);
        return f(__uint_as_float(r[0]), __uint_as_float(r[1]));
    }
}
struct Max { __device__ float operator()(float a, float b) const { return fmaxf(a, b); } };
struct Sum { __device__ float operator()(float a, float b) const { return a + b; } };
// f over w = 16, 32 or 64 lanes in a row, to all of them
template <class F> __device__ float over_lanes(float x, int w, F f) {
    auto moved = [&](auto ctrl) { return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), decltype(ctrl)::value, 0xf, 0xf, false)); };
    x = f(x, moved(std::integral_constant<int, 0xb1>()));    // the neighbour, the other pair of four, and, once fours and eights agree,
    x = f(x, moved(std::integral_constant<int, 0x4e>()));    // the mirror image in eight and in sixteen
    x = f(x, moved(std::integral_constant<int, 0x141>()));
    x = f(x, moved(std::integral_constant<int, 0x140>()));
    if (w >= 32) x = with_lane<16>(x, f);
    if (w == 64) x = with_lane<32>(x, f);
    return x;
}

struct AttnArgs {
    KvView c;
    const int *start;          // null: one query per sequence
    const uint8_t *q;
    uint8_t *out;
    float2 *pml;               // parts' m and l: [part][head][row of the tile] (one query per sequence: [head][row][part])
    float *po;                 // parts' sums: [dim] for each of those
    size_t qstride, ostride;   // bytes
    int nseq, ntok, G;
    int window;                // below the tokens that a table row holds; 0: none
    int sinks, kept;           // first tokens that the window leaves in sight; those rounded up to a multiple of 64 (no window: 0)
    float c2;                  // scale * log2(e)
    int target;                // parts aimed for per K/V head; 0: every tile is one part. One query per sequence: workgroups
    bool pairs;                // target is two workgroups a CU
    uint32_t inverse;          // 2^32 / target, rounded down (2^32 - 1 for 1)
    int block;                 // one query per sequence: log2 of the keys of a block
    int items;                 // parts per K/V head that there is room for
    bool weigh;                // one query per sequence: beginning a tile is counted too
};

// the kernels of caches in 8 bits (type: of the queries), and of 16-bit caches with sinks, which are compiled in files of their own
using AttnKernel = void (*)(AttnArgs);
AttnKernel attn_f8_decode_kernel(uint32_t type, int dim, bool sinks, int nseq);
AttnKernel attn_f8_prompt_kernel(uint32_t type, int dim, bool sinks);
AttnKernel attn_sinks_kernel(bool prompt, bool bf16, bool fp32, int dim);

}  // namespace esq
