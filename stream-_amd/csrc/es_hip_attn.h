// Shared by the paged key-value cache's translation units: the cache as the kernels see it, which part of a call a workgroup
// takes, and the matrix-core types. A page holds, per K/V head, `page` token rows of dim elements, so a (page, head) is one
// contiguous run and 16 tokens (the least page) never span two pages.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "es_hip_quant.h"

namespace esq {

struct KvView {
    uint8_t *k, *v;
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
    // bytes from a pool's start to (page, head, token)
    __device__ size_t at(int page, int head, int token) const {
        return ((((size_t)page * heads + head) << shift) + token) * dim * 2;
    }
};

// A view checked on the host; records the reason and returns ES_HIP_EINVAL where kv cannot be used for nseq sequences.
int kv_check(const es_hip_kv *kv, int nseq, KvView &v, bool paged);

using h8 = _Float16 __attribute__((ext_vector_type(8)));
using b8 = __bf16 __attribute__((ext_vector_type(8)));
using f4 = float __attribute__((ext_vector_type(4)));
using f16v = float __attribute__((ext_vector_type(16)));
using u2 = uint32_t __attribute__((ext_vector_type(2)));
using u4 = uint32_t __attribute__((ext_vector_type(4)));

}  // namespace esq
