// The paged key-value cache: new tokens' rows into their pages, pages copied, and the bookkeeping of sequences and pages.
// The reference's cache is two host arrays per layer, one sequence long (src/es_engine.c, attention_n at :975); pages let
// sequences of any length share one pool and a common beginning.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstddef>
#include <cstring>
#include <functional>
#include <new>
#include <vector>

#include "es_hip_attn.h"
#include "es_hip_host.h"

namespace esq {

int kv_check(const es_hip_kv *kv, int nseq, KvView &v, bool paged) {
    if (!kv) return host_fail(ES_HIP_EINVAL, "null cache");
    const bool eight = kv->type == ES_HIP_F8;
    if (kv->type != ES_HIP_F16 && kv->type != ES_HIP_BF16 && !eight) return host_fail(ES_HIP_EINVAL, "the cache's type is F16, BF16 or F8");
    if (kv->heads < 1 || kv->heads > 4096 || kv->dim < 8 || kv->dim > 256 || kv->dim % 8)
        return host_fail(ES_HIP_EINVAL, "1 to 4096 K/V heads of a multiple of 8 up to 256 elements");
    if (eight && kv->dim % 16) return host_fail(ES_HIP_EINVAL, "an F8 cache's heads have a multiple of 16 elements");
    if (kv->page < 16 || kv->page > 1024 || (kv->page & (kv->page - 1)))
        return host_fail(ES_HIP_EINVAL, "a page is a power of two from 16 to 1024 tokens");
    if (kv->npages < 1) return host_fail(ES_HIP_EINVAL, "no pages");
    if (!kv->k || !kv->v || ((reinterpret_cast<uintptr_t>(kv->k) | reinterpret_cast<uintptr_t>(kv->v)) & 15))
        return host_fail(ES_HIP_EINVAL, "null or misaligned pools (16 bytes)");
    // (the scales' fields are read for F8 alone: a program built when the struct ended before them has none)
    if (eight && (!kv->k_scale || !kv->v_scale || ((reinterpret_cast<uintptr_t>(kv->k_scale) | reinterpret_cast<uintptr_t>(kv->v_scale)) & 3)))
        return host_fail(ES_HIP_EINVAL, "null or misaligned scales of an F8 cache");
    v.k = static_cast<uint8_t *>(kv->k);
    v.v = static_cast<uint8_t *>(kv->v);
    v.ks = eight ? kv->k_scale : nullptr;
    v.vs = eight ? kv->v_scale : nullptr;
    v.heads = kv->heads;
    v.dim = kv->dim;
    v.shift = __builtin_ctz((unsigned)kv->page);
    v.npages = kv->npages;
    v.table = kv->table;
    v.len = kv->len;
    v.seq = kv->seq;
    v.rows = kv->rows;
    v.max_pages = kv->max_pages;
    if (!paged) return ES_HIP_OK;
    if (nseq < 0) return host_fail(ES_HIP_EINVAL, "negative number of sequences");
    if (nseq == 0) return ES_HIP_OK;
    if (!kv->table || !kv->len || kv->rows < 1 || kv->max_pages < 1)
        return host_fail(ES_HIP_EINVAL, "null or empty page table or lengths");
    if (!kv->seq && kv->rows < nseq) return host_fail(ES_HIP_EINVAL, "fewer table rows than sequences");
    if ((long long)kv->max_pages * kv->page > 1 << 30) return host_fail(ES_HIP_EINVAL, "max_pages * page exceeds 2^30 tokens");
    if ((reinterpret_cast<uintptr_t>(kv->table) | reinterpret_cast<uintptr_t>(kv->len) | reinterpret_cast<uintptr_t>(kv->seq)) & 3)
        return host_fail(ES_HIP_EINVAL, "table, len and seq must be 4-byte aligned");
    return ES_HIP_OK;
}

}  // namespace esq

namespace {

using namespace esq;

// ---- new rows ------------------------------------------------------------------------------------------------------------
// One thread per 8 elements of K and the same of V: 16 bytes of each pool. Where its token goes are three dependent loads
// (start, len, table), the same ones for all threads of the row, under which the elements' own loads are on their way. Bound by
// its reads and writes where it is long (71 MB, fp32 to bf16, in 12.7 us), by its launch where it is short (one token 4.1 us,
// of which its kernel 2).
struct AppendArgs {
    KvView c;
    const int *start;
    const uint8_t *k, *v;
    size_t kstride, vstride;   // bytes
    int nseq, token0, ntok;    // tokens of this launch and the first of them
    int all;                   // tokens of the call
    int per;                   // threads per token: heads * dim / 8
};

template <bool BF> __device__ uint32_t round2(float a, float b) {
    if constexpr (BF) {
        using b2 = __bf16 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, b2{static_cast<__bf16>(a), static_cast<__bf16>(b)});
    } else {
        using h2 = _Float16 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, h2{static_cast<_Float16>(a), static_cast<_Float16>(b)});
    }
}

// 8 elements in the cache's type
template <bool F32, bool BF> struct Eight {
    struct __attribute__((packed, aligned(F32 ? 4 : 2))) Raw { uint32_t x[F32 ? 8 : 4]; } raw;
    __device__ explicit Eight(const uint8_t *p) : raw(*reinterpret_cast<const Raw *>(p)) {}
    __device__ u4 value() const {
        u4 w;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if constexpr (F32) w[j] = round2<BF>(__uint_as_float(raw.x[2 * j]), __uint_as_float(raw.x[2 * j + 1]));
            else w[j] = raw.x[j];
        }
        return w;
    }
};

template <bool F32, bool BF> __global__ __launch_bounds__(256) void kv_append_kernel(AppendArgs a) {
    const uint32_t i = blockIdx.x * 256u + threadIdx.x;
    const int t = a.token0 + (int)(i / a.per), c = (int)(i % a.per);
    if (t >= a.token0 + a.ntok) return;
    int b = t, back = 1;   // the token is the back-th last of sequence b
    if (a.start) {         // b: the last sequence that starts at or before t
        int lo = 0, hi = a.nseq;
        while (hi - lo > 1) {
            const int m = (lo + hi) >> 1;
            if (a.start[m] <= t) lo = m; else hi = m;
        }
        b = lo;
        const int end = min(a.start[b + 1], a.all);
        if (a.start[b] > t || end <= t) return;   // (rows that are no sequence's are not read)
        back = end - t;
    }
    const Eight<F32, BF> k(a.k + (size_t)t * a.kstride + (size_t)c * (F32 ? 32 : 16)), v(a.v + (size_t)t * a.vstride + (size_t)c * (F32 ? 32 : 16));
    const int r = a.c.row(b), pos = a.c.tokens(b) - back;
    const int page = r < 0 || pos < 0 ? -1 : a.c.table[(size_t)r * a.c.max_pages + (pos >> a.c.shift)];
    const u4 kw = k.value(), vw = v.value();
    if (page < 0 || page >= a.c.npages) return;
    const int dc = a.c.dim >> 3, head = c / dc, d = (c - head * dc) * 8;
    const size_t at = (a.c.row_at(page, head, pos & ((1 << a.c.shift) - 1)) * a.c.dim + d) * 2;
    *reinterpret_cast<u4 *>(a.c.k + at) = kw;
    *reinterpret_cast<u4 *>(a.c.v + at) = vw;
}

// ---- new rows in 8 bits --------------------------------------------------------------------------------------------------------
// A wave per run of 16 tokens and K/V head that gets tokens, of K or of V: its elements in registers, 8 a lane at a time, their
// largest over the lanes, the scale, and the numbers. A run that had tokens before the call keeps them: its scale never
// shrinks, and where it grows they are rounded once more to the new one, which is exact but for what falls below 2^-6 of it (so that
// adding tokens one by one and all at once differ there alone). Powers of two make all of this exact arithmetic: no result hangs
// on how a division was rounded.
//
// Runs are found by slots: sequence b has those from start[b] / 16 + 2 b on, at least as many as the runs that its tokens can touch
// ((n + 14) / 16 + 1 of n), and a wave finds its sequence by 64 probes at a time.
//
// Bound by its launch where it is short (a token 4.6 us, of which its kernel 3), by its reads and writes where it is long: 6700 tokens of 8 heads of 64
// from fp32, 59 MB, in 11.8 us; 4096 of 8 heads of 128, 42 MB, in 9.4. (A wave for K and V of its run together: 11.4 and 9.6, short calls 0.1 us more.)
constexpr int E_LEAST = -100, E_MOST = 120;   // the scales' exponents
__device__ int exponent(float scale) { return min(max((int)(__float_as_uint(scale) >> 23 & 255) - 127, E_LEAST), E_MOST); }
__device__ float power(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
// the least e with largest <= 448 * 2^e = 1.75 * 2^(e + 8)
__device__ int exponent_for(float largest) {
    const uint32_t u = __float_as_uint(largest);
    return min(max((int)(u >> 23) - 127 - 8 + ((u & 0x7fffff) > 0x600000), E_LEAST), E_MOST);
}
__device__ bool finite(float x) { return fabsf(x) < INFINITY; }

enum { ROW_F32, ROW_F16, ROW_BF16 };
// 8 elements as they come
template <int ROW> struct Row8 {
    struct __attribute__((packed, aligned(ROW == ROW_F32 ? 4 : 2))) Raw { uint32_t x[ROW == ROW_F32 ? 8 : 4]; } raw;
    __device__ void load(const uint8_t *p) { raw = *reinterpret_cast<const Raw *>(p); }
    __device__ float get(int i) const {
        if constexpr (ROW == ROW_F32) return __uint_as_float(raw.x[i]);
        else if constexpr (ROW == ROW_BF16) return __uint_as_float(i & 1 ? raw.x[i / 2] & 0xffff0000u : raw.x[i / 2] << 16);
        else return static_cast<float>(__builtin_bit_cast(_Float16, (uint16_t)(raw.x[i / 2] >> (i & 1) * 16)));
    }
};
__device__ u2 eight_numbers(const float (&x)[8]) {
    u2 y;
#pragma unroll
    for (int i = 0; i < 2; i++)
        y[i] = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i + 2], x[4 * i + 3], __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i], x[4 * i + 1], 0, false), true);
    return y;
}

struct AppendArgs8 {
    KvView c;
    float *ks, *vs;
    const int *start;
    const uint8_t *k, *v;
    size_t kstride, vstride;   // bytes
    int nseq, ntok, slots;
};

template <int ROW, int DP> __global__ __launch_bounds__(256) void kv_append8_kernel(AppendArgs8 a) {
    constexpr int NI = DP / 32, ES = ROW == ROW_F32 ? 4 : 2;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long long item = (long long)blockIdx.x * 4 + wave;
    const int slot = (int)(item / a.c.heads), head = (int)(item - (long long)slot * a.c.heads);
    if (slot >= a.slots) return;
    int b = slot, t0 = slot, n = 1, j = 0;   // the sequence, its rows, the number of the run among those it may touch
    if (a.start) {
        int at = 0, end = a.nseq;
        for (;;) {
            const int step = (end - at + 63) >> 6, i = min(at + lane * step, a.nseq - 1);
            const int from = a.start[i], to = a.start[i + 1];
            const int before = __builtin_popcountll(__ballot(at + lane * step < end && (from >> 4) + 2 * i <= slot));
            if (!before) return;
            at += (before - 1) * step;
            if (step == 1) {
                b = at;
                t0 = __builtin_amdgcn_readlane(from, before - 1);
                j = slot - (t0 >> 4) - 2 * b;
                n = __builtin_amdgcn_readlane(to, before - 1);
                break;
            }
            end = min(end, at + step);
        }
        t0 = min(max(t0, 0), a.ntok);
        n = min(max(n, t0), a.ntok) - t0;
    }
    const int r = a.c.row(b), len = a.c.tokens(b), first = len - n;
    const int begin = (max(first, 0) & -16) + j * 16, lo = max(max(first, 0), begin), hi = min(len, begin + 16);
    if (r < 0 || (unsigned)j > 1u << 26 || lo >= hi) return;
    const int page = a.c.table[(size_t)r * a.c.max_pages + (begin >> a.c.shift)];
    if (page < 0 || page >= a.c.npages) return;
    const bool is_v = blockIdx.y;
    const size_t row = a.c.row_at(page, head, begin & ((1 << a.c.shift) - 1));
    uint8_t *pool = (is_v ? a.c.v : a.c.k) + row * a.c.dim;
    float *scale = (is_v ? a.vs : a.ks) + (row >> 4);
    const uint8_t *src = (is_v ? a.v : a.k) + (size_t)(t0 + lo - first) * (is_v ? a.vstride : a.kstride) + (size_t)head * a.c.dim * ES;
    const size_t stride = is_v ? a.vstride : a.kstride;
    const int per = a.c.dim >> 3, mine = (hi - lo) * per;   // eights of elements
    const bool more = lo > begin;
    const int e_old = more ? exponent(*scale) : E_LEAST;

    Row8<ROW> x[NI];
    float largest = 0.0f;
#pragma unroll
    for (int i = 0; i < NI; i++) {
        const int id = lane + i * 64, t = id / per, d = (id - t * per) * 8;
        if (id < mine) {
            x[i].load(src + t * stride + d * ES);
#pragma unroll
            for (int k = 0; k < 8; k++) largest = fmaxf(largest, finite(x[i].get(k)) ? fabsf(x[i].get(k)) : 0.0f);
        }
    }
    largest = over_lanes(largest, 64, Max());
    const int e = max(exponent_for(largest), e_old);
    if (more && e > e_old) {
        const float by = power(max(e_old - e, -32));   // (2^-32: every number to 0)
        for (int id = lane; id < (lo - begin) * per; id += 64) {
            u2 *p = reinterpret_cast<u2 *>(pool) + id;
            const u2 w = *p;
            float y[8];
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const auto y0 = __builtin_amdgcn_cvt_pk_f32_fp8(w[i], false), y1 = __builtin_amdgcn_cvt_pk_f32_fp8(w[i], true);
                y[i * 4] = y0[0] * by;
                y[i * 4 + 1] = y0[1] * by;
                y[i * 4 + 2] = y1[0] * by;
                y[i * 4 + 3] = y1[1] * by;
            }
            *p = eight_numbers(y);
        }
    }
    const float by = power(-e);
    u2 *to = reinterpret_cast<u2 *>(pool + (size_t)(lo - begin) * a.c.dim);
#pragma unroll
    for (int i = 0; i < NI; i++) {
        if (lane + i * 64 < mine) {
            float y[8];
#pragma unroll
            for (int k = 0; k < 8; k++) y[k] = finite(x[i].get(k)) ? x[i].get(k) * by : __uint_as_float(0x7fc00000u);
            to[lane + i * 64] = eight_numbers(y);
        }
    }
    if (lane == 0) *scale = power(e);
}

// ---- pages copied ----------------------------------------------------------------------------------------------------------
// The pairs travel with the launch (a kernel's arguments hold 4 KB): no list in memory, nothing to wait for. 16 KB per
// workgroup, four loads in flight per thread. Bound by HBM where it is long: copies of COPY_ONCE bytes and more go past the
// caches (ONCE). us past them and through them, bytes read and written: 63 MB 12.4 and 10.8, 126 MB 24.5 and 29.3, 786 MB 159
// (4.9 TB/s) and 175.
constexpr int COPY_PAIRS = 448, COPY_BYTES = 16384;
constexpr size_t COPY_ONCE = 96u << 20;   // bytes read and written
struct CopyArgs {
    uint8_t *k, *v;
    float *ks, *vs;        // an 8-bit cache's scales
    size_t layer_bytes, layer_scales;
    int page_scales;
    uint32_t page_bytes;   // a multiple of 256
    int src[COPY_PAIRS], dst[COPY_PAIRS];
};

template <bool ONCE, bool E8> __global__ __launch_bounds__(256) void kv_copy_kernel(CopyArgs a) {
    const int layer = blockIdx.z >> 1;
    uint8_t *pool = (blockIdx.z & 1 ? a.v : a.k) + (size_t)layer * a.layer_bytes;
    const uint8_t *s = pool + (size_t)a.src[blockIdx.y] * a.page_bytes;
    uint8_t *d = pool + (size_t)a.dst[blockIdx.y] * a.page_bytes;
    const uint32_t at = blockIdx.x * COPY_BYTES + threadIdx.x * 16;
    u4 x[4];
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (at + i * 4096 < a.page_bytes) {
            const u4 *p = reinterpret_cast<const u4 *>(s + at + i * 4096);
            x[i] = ONCE ? __builtin_nontemporal_load(p) : *p;
        }
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (at + i * 4096 < a.page_bytes) {
            u4 *p = reinterpret_cast<u4 *>(d + at + i * 4096);
            if constexpr (ONCE) __builtin_nontemporal_store(x[i], p);
            else *p = x[i];
        }
    if constexpr (E8) {   // this workgroup's share of the page's scales
        float *scales = (blockIdx.z & 1 ? a.vs : a.ks) + (size_t)layer * a.layer_scales;
        const int share = (a.page_scales + gridDim.x - 1) / gridDim.x, first = blockIdx.x * share;
        for (int i = first + threadIdx.x; i < min(first + share, a.page_scales); i += 256)
            scales[(size_t)a.dst[blockIdx.y] * a.page_scales + i] = scales[(size_t)a.src[blockIdx.y] * a.page_scales + i];
    }
}

// the pools of nlayers layers: where the first one's are, and how far apart the layers are
struct Layers {
    uint8_t *k, *v;
    float *ks, *vs;   // null: a 16-bit cache
    size_t layer_bytes, page_bytes, page_scales;   // page_scales: scales of a page
    int nlayers;
    size_t layer_scales() const { return page_scales ? layer_bytes / (page_bytes / page_scales) : 0; }
};

hipError_t copy_pages(const Layers &c, const int *src, const int *dst, int n, hipStream_t s) {
    CopyArgs a;
    a.layer_bytes = c.layer_bytes;
    a.layer_scales = c.layer_scales();
    a.page_bytes = (uint32_t)c.page_bytes;
    a.page_scales = (int)c.page_scales;
    const bool once = (double)c.page_bytes * c.nlayers * n * 4 >= COPY_ONCE;
    const auto f = c.ks ? (once ? kv_copy_kernel<true, true> : kv_copy_kernel<false, true>) : (once ? kv_copy_kernel<true, false> : kv_copy_kernel<false, false>);
    for (int l = 0; l < c.nlayers; l += 16384)   // (a grid's z ends at 65535)
        for (int i = 0; i < n; i += COPY_PAIRS) {
            const int m = std::min(COPY_PAIRS, n - i);
            std::copy(src + i, src + i + m, a.src);
            std::copy(dst + i, dst + i + m, a.dst);
            a.k = c.k + (size_t)l * c.layer_bytes;
            a.v = c.v + (size_t)l * c.layer_bytes;
            a.ks = c.ks ? c.ks + (size_t)l * a.layer_scales : nullptr;
            a.vs = c.vs ? c.vs + (size_t)l * a.layer_scales : nullptr;
            f<<<dim3((unsigned)((c.page_bytes + COPY_BYTES - 1) / COPY_BYTES), m, 2 * std::min(16384, c.nlayers - l)), 256, 0, s>>>(a);
            if (hipError_t e = hipGetLastError()) return e;
        }
    return hipSuccess;
}

// ---- the pool's tables -----------------------------------------------------------------------------------------------------
// Entries written to the table (at >= 0) or to the lengths (at < 0: length ~at), sent with the launch.
constexpr int SET_MAX = 448;
struct SetArgs {
    int *table, *len;
    int n;
    int64_t at[SET_MAX / 2];
    int value[SET_MAX / 2];
};
__global__ __launch_bounds__(256) void kv_set_kernel(SetArgs a) {
    const int i = threadIdx.x;
    if (i >= a.n) return;
    if (a.at[i] >= 0) a.table[a.at[i]] = a.value[i];
    else a.len[~a.at[i]] = a.value[i];
}
// A fork's table row: the first n entries of one row into another's.
__global__ __launch_bounds__(256) void kv_row_kernel(const int *src, int *dst, int n) {
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i < n) dst[i] = src[i];
}

}  // namespace

struct es_hip_kv_pool {
    struct Seq {
        bool live = false;
        int len = 0;
        std::vector<int> pages;
    };
    uint32_t type = 0;
    int nlayers = 0, heads = 0, dim = 0, page = 0, npages = 0, max_seqs = 0, max_pages = 0;
    size_t page_bytes = 0, layer_bytes = 0;
    size_t page_scales = 0;   // an 8-bit cache's scales of a page
    uint8_t *mem = nullptr;   // K of every layer, then V; an 8-bit cache: then the scales of K, and of V
    int *table = nullptr, *len = nullptr;
    std::vector<int> refs;    // sequences that hold the page
    std::vector<int> spare;   // a heap, the lowest number first
    std::vector<Seq> seqs;

    int take() {
        std::pop_heap(spare.begin(), spare.end(), std::greater<int>());
        const int p = spare.back();
        spare.pop_back();
        return p;
    }
    void give(int p) {   // never allocates: spare has room for every page
        spare.push_back(p);
        std::push_heap(spare.begin(), spare.end(), std::greater<int>());
    }
    bool has(int s) const { return s >= 0 && s < max_seqs && seqs[s].live; }
    size_t pool_bytes() const { return layer_bytes * nlayers; }
    size_t layer_scales() const { return page_scales * npages; }
    float *scales(int layer, bool v) const {
        if (!page_scales) return nullptr;
        return reinterpret_cast<float *>(mem + 2 * pool_bytes()) + ((size_t)(v ? nlayers : 0) + layer) * layer_scales();
    }
    Layers layers() const;
};

Layers es_hip_kv_pool::layers() const {
    return {mem, mem + pool_bytes(), scales(0, false), scales(0, true), layer_bytes, page_bytes, page_scales, nlayers};
}

namespace {

struct Sets {   // table and length entries to send
    std::vector<int64_t> at;
    std::vector<int> value;
    void reserve(size_t n) {
        at.reserve(n);
        value.reserve(n);
    }
    void entry(const es_hip_kv_pool *p, int s, size_t j, int page) {
        at.push_back((int64_t)s * p->max_pages + (int64_t)j);
        value.push_back(page);
    }
    void length(int s, int n) {
        at.push_back(~(int64_t)s);
        value.push_back(n);
    }
    hipError_t send(const es_hip_kv_pool *p, hipStream_t st) const {
        SetArgs a;
        a.table = p->table;
        a.len = p->len;
        for (size_t i = 0; i < at.size(); i += SET_MAX / 2) {
            a.n = (int)std::min<size_t>(SET_MAX / 2, at.size() - i);
            std::copy(at.begin() + i, at.begin() + i + a.n, a.at);
            std::copy(value.begin() + i, value.begin() + i + a.n, a.value);
            kv_set_kernel<<<1, 256, 0, st>>>(a);
            if (hipError_t e = hipGetLastError()) return e;
        }
        return hipSuccess;
    }
};

// the checks of every call that sends something
int ready(const es_hip_kv_pool *p, void *stream) {
    if (!p) return host_fail(ES_HIP_EINVAL, "null pool");
    if (!p->mem) return ES_HIP_OK;
    if (int rc = host_need_device()) return rc;
    hipStreamCaptureStatus cap = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing(static_cast<hipStream_t>(stream), &cap) == hipSuccess && cap != hipStreamCaptureStatusNone)
        return host_fail(ES_HIP_EINVAL, "a pool's bookkeeping cannot be captured");
    return ES_HIP_OK;
}

int no_memory() { return host_fail(ES_HIP_ENOMEM, "out of host memory"); }

int set_len(es_hip_kv_pool *p, int s, int n, hipStream_t st) {
    if (!p->mem) return ES_HIP_OK;
    SetArgs a;
    a.table = p->table;
    a.len = p->len;
    a.n = 1;
    a.at[0] = ~(int64_t)s;
    a.value[0] = n;
    kv_set_kernel<<<1, 256, 0, st>>>(a);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? ES_HIP_OK : host_hip_fail(e, "length launch");
}

void drop_pages(es_hip_kv_pool *p, es_hip_kv_pool::Seq &q, size_t keep) {
    while (q.pages.size() > keep) {
        const int g = q.pages.back();
        q.pages.pop_back();
        if (--p->refs[g] == 0) p->give(g);
    }
}

int extend(es_hip_kv_pool *p, const int *seqs, const int *n, int count, hipStream_t st) {
    std::vector<char> named(p->max_seqs, 0);
    size_t need = 0;
    std::vector<int> refs_down;   // shared last pages, once per sequence that will copy its own
    for (int i = 0; i < count; i++) {
        if (!p->has(seqs[i])) return host_fail(ES_HIP_EINVAL, "no such sequence");
        if (named[seqs[i]]) return host_fail(ES_HIP_EINVAL, "a sequence is named twice");
        named[seqs[i]] = 1;
        const es_hip_kv_pool::Seq &q = p->seqs[seqs[i]];
        if (n[i] < 0 || (long long)q.len + n[i] > (long long)p->max_pages * p->page)
            return host_fail(ES_HIP_EINVAL, "negative number of tokens, or more than max_pages pages hold");
        need += (size_t)(((long long)q.len + n[i] + p->page - 1) / p->page) - q.pages.size();
        if (n[i] && q.len % p->page) {   // the last page is written to: alone, or on a copy
            const int g = q.pages.back();
            const int before = (int)std::count(refs_down.begin(), refs_down.end(), g);
            if (p->refs[g] - before > 1) {
                refs_down.push_back(g);
                need++;
            }
        }
    }
    if (need > p->spare.size()) return host_fail(ES_HIP_EBUSY, "too few free pages");
    // everything that can fail for want of host memory comes before the first change
    std::vector<int> src, dst;
    Sets sets;
    src.reserve(refs_down.size());
    dst.reserve(refs_down.size());
    sets.reserve(need + (size_t)count);
    for (int i = 0; i < count; i++) {
        es_hip_kv_pool::Seq &q = p->seqs[seqs[i]];
        q.pages.reserve((size_t)(((long long)q.len + n[i] + p->page - 1) / p->page));
    }
    for (int i = 0; i < count; i++) {
        if (!n[i]) continue;
        es_hip_kv_pool::Seq &q = p->seqs[seqs[i]];
        if (q.len % p->page && p->refs[q.pages.back()] > 1) {
            const int g = p->take();
            src.push_back(q.pages.back());
            dst.push_back(g);
            p->refs[q.pages.back()]--;
            p->refs[g] = 1;
            q.pages.back() = g;
            sets.entry(p, seqs[i], q.pages.size() - 1, g);
        }
        q.len += n[i];
        while ((long long)q.pages.size() * p->page < q.len) {
            const int g = p->take();
            p->refs[g] = 1;
            q.pages.push_back(g);
            sets.entry(p, seqs[i], q.pages.size() - 1, g);
        }
        sets.length(seqs[i], q.len);
    }
    if (!p->mem) return ES_HIP_OK;
    hipError_t e = copy_pages(p->layers(), src.data(), dst.data(), (int)src.size(), st);
    if (e == hipSuccess) e = sets.send(p, st);
    return e == hipSuccess ? ES_HIP_OK : host_hip_fail(e, "page launch");
}

int fork(es_hip_kv_pool *p, int seq, hipStream_t st) {
    if (!p->has(seq)) return host_fail(ES_HIP_EINVAL, "no such sequence");
    int f = 0;
    while (f < p->max_seqs && p->seqs[f].live) f++;
    if (f == p->max_seqs) return host_fail(ES_HIP_EBUSY, "every sequence number is in use");
    es_hip_kv_pool::Seq &q = p->seqs[f];
    std::vector<int> pages(p->seqs[seq].pages);
    q.pages.swap(pages);
    q.len = p->seqs[seq].len;
    q.live = true;
    for (int g : q.pages) p->refs[g]++;
    if (!p->mem) return f;
    const int n = (int)q.pages.size();
    if (n) {
        kv_row_kernel<<<(n + 255) / 256, 256, 0, st>>>(p->table + (size_t)seq * p->max_pages, p->table + (size_t)f * p->max_pages, n);
        if (hipError_t e = hipGetLastError()) return host_hip_fail(e, "table launch");
    }
    const int rc = set_len(p, f, q.len, st);
    return rc ? rc : f;
}

int compact(es_hip_kv_pool *p, hipStream_t st) {
    const int used = p->npages - (int)p->spare.size();
    std::vector<int> src, dst, to(p->npages);
    for (int g = 0, hole = 0; g < p->npages; g++) {
        to[g] = g;
        if (g < used || !p->refs[g]) continue;
        while (p->refs[hole]) hole++;   // as many holes below `used` as pages in use from there on
        to[g] = hole++;
        src.push_back(g);
        dst.push_back(to[g]);
    }
    Sets sets;
    size_t moved = 0;
    for (const auto &q : p->seqs)
        for (int g : q.pages) moved += to[g] != g;
    sets.reserve(moved);
    for (size_t i = 0; i < src.size(); i++) {
        p->refs[dst[i]] = p->refs[src[i]];
        p->refs[src[i]] = 0;
    }
    for (int s = 0; s < p->max_seqs; s++)
        for (size_t j = 0; j < p->seqs[s].pages.size(); j++) {
            int &g = p->seqs[s].pages[j];
            if (to[g] == g) continue;
            g = to[g];
            sets.entry(p, s, j, g);
        }
    p->spare.clear();
    for (int g = used; g < p->npages; g++) p->spare.push_back(g);   // ascending: a heap as it is
    if (!p->mem || src.empty()) return used;
    hipError_t e = copy_pages(p->layers(), src.data(), dst.data(), (int)src.size(), st);
    if (e == hipSuccess) e = sets.send(p, st);
    return e == hipSuccess ? used : host_hip_fail(e, "page launch");
}

}  // namespace

extern "C" {

int es_hip_kv_append_dev(const es_hip_kv *kv, int nseq, const int *start, int ntok, uint32_t src_type, const void *k,
                         size_t kstride, const void *v, size_t vstride, void *stream) {
    if (int rc = host_need_device()) return rc;
    AppendArgs a;
    if (int rc = kv_check(kv, nseq, a.c, true)) return rc;
    const bool eight = kv->type == ES_HIP_F8;
    if (src_type != ES_HIP_F32 && (eight ? src_type != ES_HIP_F16 && src_type != ES_HIP_BF16 : src_type != kv->type))
        return host_fail(ES_HIP_EINVAL, "rows are F32 or of the cache's type (an F8 cache: F32, F16 or BF16)");
    if (ntok < 0 || (!start && ntok != nseq)) return host_fail(ES_HIP_EINVAL, "ntok is negative, or not nseq without start");
    if (ntok == 0 || nseq == 0) return ES_HIP_OK;
    const size_t es = src_type == ES_HIP_F32 ? 4 : 2, row = (size_t)kv->heads * kv->dim;
    if (!k || !v || ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & (es - 1)) ||
        (reinterpret_cast<uintptr_t>(start) & 3))
        return host_fail(ES_HIP_EINVAL, "null or misaligned k, v or start");
    if (!kstride) kstride = row;
    if (!vstride) vstride = row;
    if (ntok > 1 && (kstride < row || vstride < row)) return host_fail(ES_HIP_EINVAL, "rows overlap (stride below heads * dim)");
    if (eight) {
        AppendArgs8 e;
        e.c = a.c;
        e.ks = kv->k_scale;
        e.vs = kv->v_scale;
        e.start = start;
        e.k = static_cast<const uint8_t *>(k);
        e.v = static_cast<const uint8_t *>(v);
        e.kstride = kstride * es;
        e.vstride = vstride * es;
        e.nseq = nseq;
        e.ntok = ntok;
        const long long slots = start ? (long long)ntok / 16 + 2LL * nseq + 1 : nseq, waves = slots * kv->heads;
        // (four waves a workgroup, and a launch has less than 2^32 threads)
        if (waves > (1LL << 26) - 4) return host_fail(ES_HIP_EINVAL, "an F8 cache: (ntok / 16 + 2 nseq + 1) heads, or nseq heads without start, exceed 2^26 - 4");
        e.slots = (int)slots;
        const int dp = kv->dim <= 64 ? 0 : kv->dim <= 128 ? 1 : 2;
        static constexpr void (*kernels[3][3])(AppendArgs8) = {
            {kv_append8_kernel<ROW_F32, 64>, kv_append8_kernel<ROW_F32, 128>, kv_append8_kernel<ROW_F32, 256>},
            {kv_append8_kernel<ROW_F16, 64>, kv_append8_kernel<ROW_F16, 128>, kv_append8_kernel<ROW_F16, 256>},
            {kv_append8_kernel<ROW_BF16, 64>, kv_append8_kernel<ROW_BF16, 128>, kv_append8_kernel<ROW_BF16, 256>}};
        const auto f = kernels[src_type == ES_HIP_F32 ? ROW_F32 : src_type == ES_HIP_F16 ? ROW_F16 : ROW_BF16][dp];
        f<<<dim3((unsigned)((waves + 3) / 4), 2), 256, 0, static_cast<hipStream_t>(stream)>>>(e);
        const hipError_t err = hipGetLastError();
        return err == hipSuccess ? ES_HIP_OK : host_hip_fail(err, "append launch");
    }
    a.start = start;
    a.k = static_cast<const uint8_t *>(k);
    a.v = static_cast<const uint8_t *>(v);
    a.kstride = kstride * es;
    a.vstride = vstride * es;
    a.nseq = nseq;
    a.all = ntok;
    a.per = (int)(row / 8);
    const int most = (1 << 30) / a.per;   // tokens per launch: thread numbers stay within 32 bits
    for (a.token0 = 0; a.token0 < ntok; a.token0 += a.ntok) {
        a.ntok = std::min(most, ntok - a.token0);
        const unsigned grid = (unsigned)(((size_t)a.ntok * a.per + 255) / 256);
        const bool bf = kv->type == ES_HIP_BF16;
        auto f = src_type == ES_HIP_F32 ? (bf ? kv_append_kernel<true, true> : kv_append_kernel<true, false>) : kv_append_kernel<false, false>;
        f<<<grid, 256, 0, static_cast<hipStream_t>(stream)>>>(a);
        if (hipError_t e = hipGetLastError()) return host_hip_fail(e, "append launch");
    }
    return ES_HIP_OK;
}

int es_hip_kv_copy_pages_dev(const es_hip_kv *kv, int nlayers, size_t layer_bytes, const int *src, const int *dst, int n,
                             void *stream) {
    if (int rc = host_need_device()) return rc;
    KvView c;
    if (int rc = kv_check(kv, 0, c, false)) return rc;
    if (nlayers < 0 || n < 0 || (n && (!src || !dst))) return host_fail(ES_HIP_EINVAL, "bad page list or number of layers");
    if (nlayers == 0 || n == 0) return ES_HIP_OK;
    const bool eight = kv->type == ES_HIP_F8;
    const size_t page_bytes = (size_t)kv->heads * kv->page * kv->dim * (eight ? 1 : 2), page_scales = eight ? (size_t)kv->heads * kv->page / 16 : 0;
    if (!layer_bytes) layer_bytes = page_bytes * kv->npages;
    if (nlayers > 1 && (layer_bytes < page_bytes * kv->npages || layer_bytes % (eight ? 16 * kv->dim : 16)))
        return host_fail(ES_HIP_EINVAL, "layers overlap, or a layer is not a multiple of 16 bytes (F8: of 16 tokens)");
    try {
        std::vector<uint64_t> is_src((kv->npages + 63) / 64, 0), is_dst((kv->npages + 63) / 64, 0);
        for (int i = 0; i < n; i++) {
            if (src[i] < 0 || src[i] >= kv->npages || dst[i] < 0 || dst[i] >= kv->npages)
                return host_fail(ES_HIP_EINVAL, "a page number is outside the pools");
            const uint64_t bit = 1ull << (dst[i] & 63);
            if (is_dst[dst[i] >> 6] & bit) return host_fail(ES_HIP_EINVAL, "a page is a destination twice");
            is_dst[dst[i] >> 6] |= bit;
            is_src[src[i] >> 6] |= 1ull << (src[i] & 63);
        }
        for (size_t w = 0; w < is_src.size(); w++)
            if (is_src[w] & is_dst[w]) return host_fail(ES_HIP_EINVAL, "a page is a source and a destination");
    } catch (const std::bad_alloc &) {
        return no_memory();
    }
    const Layers layers = {c.k, c.v, eight ? kv->k_scale : nullptr, eight ? kv->v_scale : nullptr, layer_bytes, page_bytes, page_scales, nlayers};
    const hipError_t e = copy_pages(layers, src, dst, n, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? ES_HIP_OK : host_hip_fail(e, "page copy launch");
}

int es_hip_kv_pool_create(es_hip_kv_pool **out, uint32_t type, int nlayers, int heads, int dim, int page, int npages,
                          int max_seqs, int max_pages) {
    if (!out) return host_fail(ES_HIP_EINVAL, "null output pointer");
    *out = nullptr;
    if (nlayers < 0 || max_seqs < 1 || max_pages < 1) return host_fail(ES_HIP_EINVAL, "bad number of layers, sequences or pages");
    if ((long long)max_seqs * max_pages > 1LL << 40) return host_fail(ES_HIP_EINVAL, "max_seqs * max_pages exceeds 2^40");
    es_hip_kv kv = {type, heads, dim, page, npages, reinterpret_cast<void *>(16), reinterpret_cast<void *>(16),
                    reinterpret_cast<const int *>(16), reinterpret_cast<const int *>(16), nullptr, max_seqs, max_pages,
                    reinterpret_cast<float *>(16), reinterpret_cast<float *>(16)};
    KvView v;
    if (int rc = kv_check(&kv, 1, v, true)) return rc;
    if (nlayers)
        if (int rc = host_need_device()) return rc;
    es_hip_kv_pool *p = nullptr;
    try {
        p = new es_hip_kv_pool;
        p->type = type;
        p->nlayers = nlayers;
        p->heads = heads;
        p->dim = dim;
        p->page = page;
        p->npages = npages;
        p->max_seqs = max_seqs;
        p->max_pages = max_pages;
        p->page_bytes = (size_t)heads * page * dim * (type == ES_HIP_F8 ? 1 : 2);
        p->page_scales = type == ES_HIP_F8 ? (size_t)heads * page / 16 : 0;
        p->layer_bytes = p->page_bytes * npages;
        p->refs.assign(npages, 0);
        p->spare.resize(npages);
        for (int g = 0; g < npages; g++) p->spare[g] = g;
        p->seqs.resize(max_seqs);
    } catch (const std::bad_alloc &) {
        delete p;
        return no_memory();
    }
    if (nlayers) {
        size_t all;
        hipError_t e = hipErrorOutOfMemory;
        if (!__builtin_mul_overflow(p->layer_bytes + p->layer_scales() * sizeof(float), (size_t)nlayers * 2, &all)) e = hipMalloc(reinterpret_cast<void **>(&p->mem), all);
        if (e == hipSuccess) e = hipMalloc(reinterpret_cast<void **>(&p->table), (size_t)max_seqs * max_pages * sizeof(int));
        if (e == hipSuccess) e = hipMalloc(reinterpret_cast<void **>(&p->len), (size_t)max_seqs * sizeof(int));
        if (e == hipSuccess) e = hipMemset(p->len, 0, (size_t)max_seqs * sizeof(int));
        if (e == hipSuccess) e = hipDeviceSynchronize();   // the first call may come on any stream
        if (e != hipSuccess) {
            es_hip_kv_pool_destroy(p);
            return host_hip_fail(e, "pool allocation");
        }
    }
    *out = p;
    return ES_HIP_OK;
}

void es_hip_kv_pool_destroy(es_hip_kv_pool *p) {
    if (!p) return;
    if (p->mem) (void)hipFree(p->mem);
    if (p->table) (void)hipFree(p->table);
    if (p->len) (void)hipFree(p->len);
    delete p;
}

int es_hip_kv_pool_view(const es_hip_kv_pool *p, int layer, es_hip_kv *out) {
    if (!p || !out || layer < 0 || layer >= p->nlayers) return host_fail(ES_HIP_EINVAL, "null pool or output, or no such layer");
    uint8_t *k = p->mem + (size_t)layer * p->layer_bytes;
    const es_hip_kv kv = {p->type, p->heads, p->dim, p->page, p->npages, k, k + p->pool_bytes(), p->table, p->len, nullptr, p->max_seqs, p->max_pages,
                          p->scales(layer, false), p->scales(layer, true)};
    // (the scales' fields are written for F8 alone, as they are read)
    memcpy(out, &kv, p->page_scales ? sizeof(kv) : offsetof(es_hip_kv, k_scale));
    return ES_HIP_OK;
}

int es_hip_kv_pool_free_pages(const es_hip_kv_pool *p) {
    return p ? (int)p->spare.size() : host_fail(ES_HIP_EINVAL, "null pool");
}

int es_hip_kv_seq_create(es_hip_kv_pool *p, void *stream) {
    if (int rc = ready(p, stream)) return rc;
    for (int s = 0; s < p->max_seqs; s++)
        if (!p->seqs[s].live) {
            if (int rc = set_len(p, s, 0, static_cast<hipStream_t>(stream))) return rc;
            p->seqs[s].live = true;
            p->seqs[s].len = 0;
            return s;
        }
    return host_fail(ES_HIP_EBUSY, "every sequence number is in use");
}

int es_hip_kv_seq_extend(es_hip_kv_pool *p, const int *seqs, const int *n, int count, void *stream) {
    if (int rc = ready(p, stream)) return rc;
    if (count < 0 || (count && (!seqs || !n))) return host_fail(ES_HIP_EINVAL, "null list of sequences");
    try {
        return extend(p, seqs, n, count, static_cast<hipStream_t>(stream));
    } catch (const std::bad_alloc &) {
        return no_memory();
    }
}

int es_hip_kv_seq_fork(es_hip_kv_pool *p, int seq, void *stream) {
    if (int rc = ready(p, stream)) return rc;
    try {
        return fork(p, seq, static_cast<hipStream_t>(stream));
    } catch (const std::bad_alloc &) {
        return no_memory();
    }
}

int es_hip_kv_seq_truncate(es_hip_kv_pool *p, int seq, int len, void *stream) {
    if (int rc = ready(p, stream)) return rc;
    if (!p->has(seq) || len < 0 || len > p->seqs[seq].len) return host_fail(ES_HIP_EINVAL, "no such sequence, or not that many tokens");
    if (int rc = set_len(p, seq, len, static_cast<hipStream_t>(stream))) return rc;
    p->seqs[seq].len = len;
    drop_pages(p, p->seqs[seq], ((size_t)len + p->page - 1) / p->page);
    return ES_HIP_OK;
}

int es_hip_kv_seq_free(es_hip_kv_pool *p, int seq, void *stream) {
    if (int rc = es_hip_kv_seq_truncate(p, seq, 0, stream)) return rc;
    p->seqs[seq].live = false;
    return ES_HIP_OK;
}

int es_hip_kv_seq_len(const es_hip_kv_pool *p, int seq) {
    return p && p->has(seq) ? p->seqs[seq].len : host_fail(ES_HIP_EINVAL, "null pool or no such sequence");
}

int es_hip_kv_seq_pages(const es_hip_kv_pool *p, int seq, int *out, int cap) {
    if (!p || !p->has(seq) || cap < 0 || (cap && !out)) return host_fail(ES_HIP_EINVAL, "null pool or output, or no such sequence");
    const std::vector<int> &g = p->seqs[seq].pages;
    std::copy(g.begin(), g.begin() + std::min<size_t>(cap, g.size()), out);
    return (int)g.size();
}

int es_hip_kv_pool_compact(es_hip_kv_pool *p, void *stream) {
    if (int rc = ready(p, stream)) return rc;
    try {
        return compact(p, static_cast<hipStream_t>(stream));
    } catch (const std::bad_alloc &) {
        return no_memory();
    }
}

}  // extern "C"
