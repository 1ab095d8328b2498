// q38_paged.hpp — the batched token mixers' descriptors and the index arithmetic that host and
// device share (rows of a ragged batch, pages of a cache), so that a CPU test can check it.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace q38 {

constexpr int kBatchMaxSeqs = 4096;
constexpr int kBatchMaxRows = 1 << 24;

struct PagedCacheDev {
    void *keys, *values;   // [pages][hkv][1 << shift][d] bf16 or int8
    float *ks, *vs;        // [pages][hkv][1 << shift] (int8), else null
    int pages, shift, hkv, d;
};
struct PagedBatchDev {
    const int32_t *off, *tokens, *table;
    int seqs, rows, width;  // width: columns of the page table
};
struct DeltaBatchDev {
    const int32_t *off, *origin, *last, *ckpt;  // origin, last, ckpt may be null
    float* states;
    int seqs, rows, slots;
};
struct DeltaDev {
    const uint16_t *q, *k, *v;
    const float *g, *beta;
    uint16_t* out;
    int64_t qs, ks, vs;  // row strides in elements
    int hk, hv, dk, dv;
    float scale;
};

// The rows of sequence i: [begin, end) within the tensors, whatever the offsets hold.
struct RowSpan {
    int begin, end;
};
__host__ __device__ inline RowSpan row_span(const int32_t* off, int i, int rows) {
    int b = off[i], e = off[i + 1];
    b = b < 0 ? 0 : b;
    e = e > rows ? rows : e;
    return RowSpan{b, e < b ? b : e};
}
// The sequence that owns row r (the last one that begins at or before it), or -1: for ascending
// offsets; any others end the search too, at some sequence of the batch.
__host__ __device__ inline int row_sequence(const int32_t* off, int seqs, int r) {
    int lo = 0, hi = seqs;  // off[lo] <= r < off[hi], with off[-1] and off[seqs + 1] taken as infinities
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (off[mid] <= r) lo = mid;
        else hi = mid;
    }
    return seqs > 0 && off[lo] <= r && r < off[lo + 1] ? lo : -1;
}
// Element index of a token's head row in the cache (its scale's index times d), or -1 where the
// page is out of range. 64 bits: a cache may hold more than 2^31 elements.
__host__ __device__ inline int64_t cache_row(int32_t page, int pages, int hkv, int head, int shift, int t) {
    if (static_cast<uint32_t>(page) >= static_cast<uint32_t>(pages)) return -1;
    return ((static_cast<int64_t>(page) * hkv + head) << shift) + (t & ((1 << shift) - 1));
}

hipError_t launch_paged_append(const PagedCacheDev& C, bool q8, const PagedBatchDev& B, const uint16_t* k, int64_t ks,
                               const uint16_t* v, int64_t vs, hipStream_t st);
size_t paged_attention_ws(const PagedCacheDev& C, const PagedBatchDev& B, int max_rows, int hq);
hipError_t launch_paged_attention(const PagedCacheDev& C, bool q8, const PagedBatchDev& B, int max_rows,
                                  const uint16_t* q, int64_t qs, int hq, float scale, uint16_t* out, int64_t os,
                                  void* ws, hipStream_t st);
size_t delta_ws(const DeltaDev& D, const DeltaBatchDev& B, int max_rows);
hipError_t launch_delta(const DeltaDev& D, const DeltaBatchDev& B, int max_rows, void* ws, hipStream_t st);

} // namespace q38
