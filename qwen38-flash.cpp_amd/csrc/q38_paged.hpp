// q38_paged.hpp — the batched token mixers' descriptors and the index arithmetic that host and
// device share (rows of a ragged batch, pages of a cache), so that a CPU test can check it.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace q38 {

constexpr int kBatchMaxSeqs = 4096;
constexpr int kBatchMaxRows = 1 << 19;  // (a launch has less than 2^32 threads)

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

// ---- how attention's work is split. A batch's work per kv head is a list of items, one per
// (sequence, tile of M of its rows x group queries), each of so many steps of T tokens (at least
// one: a tile that sees nothing still writes its zeros). The list of steps is cut into equal
// shares, one per workgroup, whatever sequences they belong to, so that one long sequence or many
// ragged ones load the chip evenly. An item inside one share is finished there; the pieces of the
// others are joined by a second kernel.
struct AttnItem {
    int seq, tile;       // sequence, tile of its queries
    int rows;            // the sequence's rows
    int first;           // its first row in the tensors
    int tokens;          // its tokens (0 where they are negative or behind the table)
    int see;             // tokens that the tile's last row sees
    int steps;           // max(1, ceil(see / T))
    bool bad;            // tokens behind the table
};
struct AttnSplit {
    int G, M, T;  // queries per kv head and row; queries per tile; tokens per step
};
__host__ __device__ inline int attn_tiles(const AttnSplit& S, int rows) { return (rows * S.G + S.M - 1) / S.M; }
__host__ __device__ inline void attn_sequence(const PagedBatchDev& B, int shift, int seq, AttnItem* it) {
    const RowSpan span = row_span(B.off, seq, B.rows);
    it->seq = seq;
    it->first = span.begin;
    it->rows = span.end - span.begin;
    const int t = B.tokens[seq];
    it->bad = t > static_cast<int64_t>(B.width) << shift;
    it->tokens = t < 0 || it->bad ? 0 : t;
}
// Tokens that the sequence's row r sees.
__host__ __device__ inline int attn_see(const AttnItem& it, int r) {
    const int n = it.tokens - it.rows + r + 1;
    return n < 0 ? 0 : n;
}
__host__ __device__ inline void attn_tile(const AttnSplit& S, int tile, AttnItem* it) {
    const int last = (tile + 1) * S.M - 1, end = it->rows * S.G - 1;
    it->tile = tile;
    it->see = attn_see(*it, (last < end ? last : end) / S.G);
    it->steps = it->see > S.T ? (it->see + S.T - 1) / S.T : 1;
}
// Steps of all tiles of a sequence.
__host__ __device__ inline int attn_weight(const AttnSplit& S, const PagedBatchDev& B, int shift, int seq) {
    AttnItem it;
    attn_sequence(B, shift, seq, &it);
    int sum = 0;
    for (int j = 0, n = attn_tiles(S, it.rows); j < n; ++j) {
        attn_tile(S, j, &it);
        sum += it.steps;
    }
    return sum;
}
// A share's next piece: `it` and its steps [from, to), the item's first step at `start` of the
// whole list. Call with *pos inside sequence seq, whose first step is at seq_start; moves *pos, and
// *seq and *seq_start with it.
struct AttnPiece {
    AttnItem it;
    int from, to;
    int64_t start;
};
__host__ __device__ inline bool attn_next(const AttnSplit& S, const PagedBatchDev& B, int shift, int64_t end, int* seq,
                                          int64_t* seq_start, int64_t* pos, AttnPiece* out) {
    while (*pos < end && *seq < B.seqs) {
        attn_sequence(B, shift, *seq, &out->it);
        int64_t at = *seq_start;
        for (int j = 0, n = attn_tiles(S, out->it.rows); j < n; ++j) {
            attn_tile(S, j, &out->it);
            if (*pos < at + out->it.steps) {
                out->start = at;
                out->from = static_cast<int>(*pos - at);
                out->to = static_cast<int>((end < at + out->it.steps ? end : at + out->it.steps) - at);
                *pos = at + out->to;
                return true;
            }
            at += out->it.steps;
        }
        *seq_start = at;
        ++*seq;
    }
    return false;
}
// The piece's place among its share's two partial results: one for an item that began before the
// share, one for an item that goes on behind it.
__host__ __device__ inline int attn_slot(int64_t item_start, int64_t share, int64_t w) {
    return item_start < w * share ? 0 : 1;
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
