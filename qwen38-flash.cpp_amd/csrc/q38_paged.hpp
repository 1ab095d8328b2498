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
// (sequence, tile of R of its rows), each of so many steps of T tokens (at least one: a tile that
// sees nothing still writes its zeros). The list of steps is cut into equal shares, one per
// workgroup, whatever sequences they belong to, so that one long sequence, many ragged ones or the
// tiles of a prompt, each a little longer than the one before, load the chip evenly. An item inside
// one share is finished there; the pieces of the others are joined by a second kernel.
struct AttnSplit {
    int G, M, T;  // queries per kv head and row; queries per tile (the tile's rows: M / G >= 1); tokens per step
    __host__ __device__ int rows() const { return M / G; }
};
struct AttnItem {
    int seq = -1, tile;
    int rows;    // the sequence's rows
    int first;   // its first row in the tensors
    int tokens;  // its tokens (0 where they are negative or behind the table)
    int see;     // tokens that the tile's last row sees
    int steps;   // max(1, ceil(see / T))
    bool bad;    // tokens behind the table
};
__host__ __device__ inline int attn_tiles(const AttnSplit& S, int rows) { return (rows + S.rows() - 1) / S.rows(); }
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
    const int behind = (tile + 1) * S.rows();
    it->tile = tile;
    it->see = attn_see(*it, (behind < it->rows ? behind : it->rows) - 1);
    it->steps = it->see > S.T ? (it->see + S.T - 1) / S.T : 1;
}
// sum over i < n of floor((a i + b) / m). Whole parts of a / m and b / m come out of the sum; what is left, a and
// b below m, counts for every height j = 1 .. top (the last term) the i with a i + b >= m j, n - ceil((m j - b) / a)
// of them, so it is n top less a sum of the same kind over the heights, with a and m exchanged as in Euclid's
// algorithm (counting the points under a line by rows in place of columns: Graham, Knuth, Patashnik,
// Concrete Mathematics, chapter 3).
__host__ __device__ inline int64_t floor_sum(uint32_t n, uint32_t m, uint32_t a, uint32_t b) {
    int64_t sum = 0;
    for (bool less = false;; less = !less) {
        const int64_t pairs = static_cast<int64_t>(n) * (static_cast<int64_t>(n) - 1) / 2;
        int64_t part = pairs * (a / m) + static_cast<int64_t>(n) * (b / m);
        a %= m;
        b %= m;
        const uint32_t top = n ? (a * (n - 1) + b) / m : 0;
        part += static_cast<int64_t>(n) * top;
        sum += less ? -part : part;
        if (top == 0) return sum;
        // (j = heights + 1: ceil((m (heights + 1) - b) / a) = floor((m heights + m - b + a - 1) / a))
        b = m - b + a - 1;
        const uint32_t columns = a;
        a = m;
        m = columns;
        n = top;
    }
}
// Steps of the sequence's tiles 0 .. n - 1 (n <= its tiles; all but its last tile have their R rows).
__host__ __device__ inline int64_t attn_before(const AttnSplit& S, const AttnItem& it, int n) {
    const int R = S.rows(), seen = it.tokens - it.rows;  // tokens in front of the first row
    int64_t sum = 0;
    if (n == attn_tiles(S, it.rows) && n > 0) {
        AttnItem last = it;
        attn_tile(S, --n, &last);
        sum = last.steps;
    }
    const int blind = seen < 0 ? (-seen / R < n ? -seen / R : n) : 0;  // tiles that see nothing
    return sum + blind + floor_sum(n - blind, S.T, R, seen + (blind + 1) * R + S.T - 1);
}
// All steps of the sequence.
__host__ __device__ inline int64_t attn_weight(const AttnSplit& S, const AttnItem& it) {
    return attn_before(S, it, attn_tiles(S, it.rows));
}
// A place in the list: an item and its first step.
struct AttnCursor {
    int seq, tile;
    int64_t start;
};
// The item that holds step pos, inside the sequence of `it`, whose first step is seq_start.
__host__ __device__ inline AttnCursor attn_seek(const AttnSplit& S, const AttnItem& it, int64_t seq_start, int64_t pos) {
    int lo = 0, hi = attn_tiles(S, it.rows);
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (seq_start + attn_before(S, it, mid) <= pos) lo = mid;
        else hi = mid;
    }
    return AttnCursor{it.seq, lo, seq_start + (lo ? attn_before(S, it, lo) : 0)};
}
// A share's next piece: an item's steps [from, to), the item's first step at `start` of the list. The
// cursor stands at the item that holds step *pos and moves with it. out->it: the piece before, whose
// sequence need not be read again, or seq -1.
struct AttnPiece {
    AttnItem it;
    int from, to;
    int64_t start;
};
__host__ __device__ inline bool attn_next(const AttnSplit& S, const PagedBatchDev& B, int shift, int64_t end,
                                          AttnCursor* at, int64_t* pos, AttnPiece* out) {
    while (*pos < end && at->seq < B.seqs) {
        if (out->it.seq != at->seq) attn_sequence(B, shift, at->seq, &out->it);
        if (at->tile < attn_tiles(S, out->it.rows)) {
            attn_tile(S, at->tile, &out->it);
            const int64_t behind = at->start + out->it.steps;
            out->start = at->start;
            out->from = static_cast<int>(*pos - at->start);
            out->to = static_cast<int>((end < behind ? end : behind) - at->start);
            *pos = at->start + out->to;
            if (*pos == behind) {
                at->start = behind;
                ++at->tile;
            }
            return true;
        }
        ++at->seq;
        at->tile = 0;
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
