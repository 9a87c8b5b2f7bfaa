// Attention over the paged key-value cache: argument checks, workspaces, which kernel a call takes and its launches. The kernels
// are in es_hip_attn_kernels.h; those of 8-bit caches and of windows with sinks are compiled in files of their own.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "es_hip_attn_kernels.h"
#include "es_hip_host.h"

namespace {

// ---- host ------------------------------------------------------------------------------------------------------------------------
struct Shape {
    size_t items;      // prompt: the most parts per K/V head that the call's lengths can give; else workgroups per K/V head
    size_t tiles;      // prompt: the most tiles
    int target;        // AttnArgs::target
    bool pairs;        // AttnArgs::pairs
    int block;         // AttnArgs::block
    size_t slots;      // parts per K/V head that the workspace holds
    int bm;
    size_t sums(const es_hip_kv *kv) const { return slots * kv->heads * bm * (size_t)kv->dim * sizeof(float); }
    size_t workspace(const es_hip_kv *kv) const { return sums(kv) + slots * kv->heads * bm * sizeof(float2); }
};
Shape shape_of(const es_hip_kv *kv, int nseq, int ntok, int heads, uint32_t type, bool prompt) {
    const int G = heads / kv->heads;
    const long long most = (long long)kv->max_pages * kv->page;
    const int nq = type != ES_HIP_F32 ? 1 : kv->type == ES_HIP_BF16 ? 3 : 2;
    Shape s{};
    if (prompt) {
        const int per_cu = prompt_per_cu(nq, kv->dim);
        const int parts = std::max(PARTS * per_cu / kv->heads, 1);
        s.pairs = per_cu == 2;
        s.bm = PM;
        s.tiles = (size_t)ntok * G / PM + nseq;
        s.target = s.tiles >= (size_t)parts || most <= CHUNK_MIN + CHUNK_SAVES ? 0 : parts;
        s.items = s.tiles + s.target;   // sum of tiles * ceil(span / chunk) <= tiles + target
        s.slots = s.target ? s.items : 0;
    } else {
        s.bm = DECODE_M;
        s.target = std::min(std::max(decode_groups(kv->dim, nseq, kv->type == ES_HIP_F8) / kv->heads, 1), DECODE_PARTS);
        s.items = s.target;
        s.block = most <= 1 << BLOCK_WHOLE ? BLOCK_WHOLE : BLOCK;
        s.slots = most > 1 << s.block ? 2 * s.items : 0;   // (0: every tile is one block)
    }
    return s;
}

int check_heads(const es_hip_kv *kv, int nseq, int ntok, int heads, KvView &v) {
    if (int rc = kv_check(kv, nseq, v, true)) return rc;
    if (heads < 1 || heads % kv->heads || heads > 65536) return host_fail(ES_HIP_EINVAL, "heads: a multiple of the cache's, up to 65536");
    if (ntok < 0) return host_fail(ES_HIP_EINVAL, "negative number of tokens");
    // (a launch holds 2^24 workgroups of 256)
    if ((long long)ntok * heads > 1 << 29 || (long long)nseq * heads > 1 << 23)
        return host_fail(ES_HIP_EINVAL, "more than 2^29 query rows, or 2^23 sequences times heads");
    if (nseq && ((long long)kv->max_pages * kv->page / (1 << BLOCK) + 2) * nseq * (heads / kv->heads / DECODE_M + 1) > 1LL << 31)
        return host_fail(ES_HIP_EINVAL, "more than 2^31 blocks of 128 keys");
    return ES_HIP_OK;
}

int check_type(const es_hip_kv *kv, uint32_t type) {
    const bool fits = kv->type == ES_HIP_F8 ? type == ES_HIP_F16 || type == ES_HIP_BF16 : type == kv->type;
    return type == ES_HIP_F32 || fits ? ES_HIP_OK : host_fail(ES_HIP_EINVAL, "q and out are F32 or of the cache's type (an F8 cache: F32, F16 or BF16)");
}

template <bool BF, int NQ> AttnKernel kernel_of(bool prompt, int dim) {
    if (prompt) return dim <= 64 ? attn_prompt_kernel<BF, NQ, 64> : dim <= 128 ? attn_prompt_kernel<BF, NQ, 128> : attn_prompt_kernel<BF, NQ, 256>;
    return dim <= 64 ? attn_decode_kernel<BF, NQ, 64> : dim <= 128 ? attn_decode_kernel<BF, NQ, 128> : attn_decode_kernel<BF, NQ, 256>;
}

template <bool F32, bool BF> hipError_t launch(AttnKernel f, const AttnArgs &a, const Shape &s, bool prompt, hipStream_t st) {
    f<<<(unsigned)(s.items * a.c.heads), 256, 0, st>>>(a);
    if (hipError_t e = hipGetLastError()) return e;
    if (!s.slots) return hipSuccess;
    const int groups = a.c.dim <= 64 ? 16 : a.c.dim <= 128 ? 8 : 4;   // rows that a workgroup's threads join at once
    if (!prompt) {
        // one row a workgroup where that leaves few of them, as many as it has groups of threads where there are many
        int together = 1;
        while (together < groups && together < a.G && (long long)a.nseq * a.c.heads * ((a.G + together - 1) / together) > 256) together *= 2;
        attn_decode_join_kernel<F32, BF><<<(unsigned)((size_t)a.nseq * a.c.heads * ((a.G + together - 1) / together)), 256, 0, st>>>(a, together);
        return hipGetLastError();
    }
    const int blocks = (int)std::min<size_t>(PM / groups, std::max<size_t>(1, 1024 / (s.tiles * a.c.heads)));   // workgroups per tile: many tiles have one part each
    attn_join_kernel<F32, BF><<<(unsigned)(s.tiles * a.c.heads * blocks), 256, 0, st>>>(a, blocks);
    return hipGetLastError();
}

int attention(const es_hip_kv *kv, int nseq, const int *start, int ntok, int heads, uint32_t type, const void *q, size_t qstride,
              float scale, int window, int sinks, void *out, size_t ostride, void *ws, size_t ws_bytes, void *stream) {
    if (int rc = host_need_device()) return rc;
    AttnArgs a;
    const bool prompt = start != nullptr;
    if (int rc = check_heads(kv, nseq, ntok, heads, a.c)) return rc;
    if (int rc = check_type(kv, type)) return rc;
    if (!(scale > 0.0f) || !std::isfinite(scale * 1.5f)) return host_fail(ES_HIP_EINVAL, "scale is positive and finite");
    if (window < 0 || sinks < 0) return host_fail(ES_HIP_EINVAL, "negative window or sinks");
    if (nseq == 0 || ntok == 0) return ES_HIP_OK;
    const size_t es = type == ES_HIP_F32 ? 4 : 2, row = (size_t)heads * kv->dim;
    if (!q || !out || ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & (es - 1)) || (reinterpret_cast<uintptr_t>(start) & 3))
        return host_fail(ES_HIP_EINVAL, "null or misaligned q, out or start");
    if (!qstride) qstride = row;
    if (!ostride) ostride = row;
    if (ntok > 1 && (qstride < row || ostride < row)) return host_fail(ES_HIP_EINVAL, "rows overlap (stride below heads * dim)");
    const Shape s = shape_of(kv, nseq, ntok, heads, type, prompt);
    const size_t need = s.workspace(kv);
    if (need && (!ws || ws_bytes < need || (reinterpret_cast<uintptr_t>(ws) & 15)))
        return host_fail(ES_HIP_EINVAL, "workspace missing, too small or misaligned (16 bytes)");
    a.start = start;
    a.q = static_cast<const uint8_t *>(q);
    a.out = static_cast<uint8_t *>(out);
    a.po = static_cast<float *>(ws);
    a.pml = reinterpret_cast<float2 *>(static_cast<uint8_t *>(ws) + s.sums(kv));
    a.qstride = qstride * es;
    a.ostride = ostride * es;
    a.nseq = nseq;
    a.ntok = ntok;
    a.G = heads / kv->heads;
    const int most = kv->max_pages * kv->page;
    a.window = window >= most ? 0 : window;   // (len - n - window then fits an int, whatever n)
    if (sinks >= most) a.window = 0;   // (every token stays in sight)
    a.sinks = a.window ? sinks : 0;
    a.kept = (a.sinks + PN - 1) & -PN;
    a.c2 = std::max(scale * 1.44269504088896340736f, 1.17549435e-38f);
    a.target = s.target;
    a.pairs = s.pairs;
    a.inverse = s.target > 1 ? (uint32_t)((1ull << 32) / s.target) : ~0u;
    a.block = s.block;
    a.items = (int)s.items;
    a.weigh = kv->type == ES_HIP_F8 && nseq > 1;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const bool f32 = type == ES_HIP_F32, bf = kv->type == ES_HIP_BF16;
    const AttnKernel f = kv->type == ES_HIP_F8 ? (prompt ? attn_f8_prompt_kernel(type, kv->dim, a.sinks > 0) : attn_f8_decode_kernel(type, kv->dim, a.sinks > 0, nseq))
                         : a.sinks             ? attn_sinks_kernel(prompt, bf, f32, kv->dim)
                         : bf                  ? (f32 ? kernel_of<true, 3>(prompt, kv->dim) : kernel_of<true, 1>(prompt, kv->dim))
                                               : (f32 ? kernel_of<false, 2>(prompt, kv->dim) : kernel_of<false, 1>(prompt, kv->dim));
    const hipError_t e = f32 ? launch<true, true>(f, a, s, prompt, st) : type == ES_HIP_BF16 ? launch<false, true>(f, a, s, prompt, st) : launch<false, false>(f, a, s, prompt, st);
    return e == hipSuccess ? ES_HIP_OK : host_hip_fail(e, "attention launch");
}

}  // namespace

extern "C" {

size_t es_hip_attn_decode_workspace(const es_hip_kv *kv, int nseq, int heads) {
    KvView v;
    if (check_heads(kv, nseq, nseq, heads, v) || !nseq) return 0;
    return shape_of(kv, nseq, nseq, heads, kv->type, false).workspace(kv);   // (fp32 queries need as much, or less)
}

size_t es_hip_attn_prompt_workspace(const es_hip_kv *kv, int nseq, int ntok, int heads, uint32_t type) {
    KvView v;
    if (check_heads(kv, nseq, ntok, heads, v) || check_type(kv, type) || !nseq || !ntok) return 0;
    return shape_of(kv, nseq, ntok, heads, type, true).workspace(kv);
}

size_t es_hip_attn_workspace_upto(const es_hip_kv *kv, int nseq, int ntok, int heads) {
    KvView v;
    if (check_heads(kv, nseq, ntok, heads, v) || !nseq) return 0;
    size_t most = shape_of(kv, nseq, nseq, heads, kv->type, false).workspace(kv);   // (decode: never less for more sequences)
    for (uint32_t type : {(uint32_t)ES_HIP_F32, kv->type}) {
        // a prompt's slots are its tiles plus the parts aimed for, as long as the tiles are fewer than those
        Shape s = shape_of(kv, 1, 1, heads, type, true);
        const size_t tiles = shape_of(kv, nseq, ntok, heads, type, true).tiles;
        if (!ntok || !s.target) continue;   // (no call has parts if one of a token has none)
        s.slots = std::min(tiles, (size_t)s.target - 1) + s.target;
        most = std::max(most, s.workspace(kv));
    }
    return most;
}

int es_hip_attn_decode_sinks_dev(const es_hip_kv *kv, int nseq, int heads, uint32_t type, const void *q, size_t qstride, float scale,
                                 int window, int sinks, void *out, size_t ostride, void *ws, size_t ws_bytes, void *stream) {
    return attention(kv, nseq, nullptr, nseq, heads, type, q, qstride, scale, window, sinks, out, ostride, ws, ws_bytes, stream);
}

int es_hip_attn_decode_dev(const es_hip_kv *kv, int nseq, int heads, uint32_t type, const void *q, size_t qstride, float scale,
                           int window, void *out, size_t ostride, void *ws, size_t ws_bytes, void *stream) {
    return es_hip_attn_decode_sinks_dev(kv, nseq, heads, type, q, qstride, scale, window, 0, out, ostride, ws, ws_bytes, stream);
}

int es_hip_attn_prompt_sinks_dev(const es_hip_kv *kv, int nseq, const int *start, int ntok, int heads, uint32_t type, const void *q,
                                 size_t qstride, float scale, int window, int sinks, void *out, size_t ostride, void *ws,
                                 size_t ws_bytes, void *stream) {
    if (!start && ntok > 0 && nseq > 0) {
        if (int rc = host_need_device()) return rc;
        return host_fail(ES_HIP_EINVAL, "null start");
    }
    return attention(kv, nseq, start, ntok, heads, type, q, qstride, scale, window, sinks, out, ostride, ws, ws_bytes, stream);
}

int es_hip_attn_prompt_dev(const es_hip_kv *kv, int nseq, const int *start, int ntok, int heads, uint32_t type, const void *q,
                           size_t qstride, float scale, int window, void *out, size_t ostride, void *ws, size_t ws_bytes,
                           void *stream) {
    return es_hip_attn_prompt_sinks_dev(kv, nseq, start, ntok, heads, type, q, qstride, scale, window, 0, out, ostride, ws, ws_bytes, stream);
}

}  // extern "C"
