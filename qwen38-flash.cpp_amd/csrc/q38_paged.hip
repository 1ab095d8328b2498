// q38_paged.hip — the paged key-value cache of many requests: the append of a batch's new keys
// and values, and causal attention of the new rows over the cache.
//
//   k_paged_append   per (row, kv head, keys / values): the copy into the token's place, or its
//                    8-bit codes and scale
//   k_paged_attn     per (row, query head): one pass over the row's tokens with the running
//                    maximum and sum of the softmax
#include "q38_device.hpp"
#include "q38_paged.hpp"
#include "q38_internal.hpp"

namespace q38 {

namespace {

// D / 8 lanes take one head row, 16 bytes each. The offsets are staged in LDS: one round trip to
// memory, then the search for the row's sequence runs there.
template <int D, bool Q8>
__global__ __launch_bounds__(256) void k_paged_append(PagedCacheDev C, PagedBatchDev B, const uint16_t* __restrict__ k,
                                                      int64_t ks, const uint16_t* __restrict__ v, int64_t vs) {
    extern __shared__ int32_t off[];
    constexpr int L = D / 8;
    for (int i = threadIdx.x; i <= B.seqs; i += 256) off[i] = B.off[i];
    __syncthreads();
    const int64_t unit = static_cast<int64_t>(blockIdx.x) * (256 / L) + threadIdx.x / L;
    const int lane = threadIdx.x % L;
    const int row = static_cast<int>(unit / (2 * C.hkv));
    const int part = static_cast<int>(unit % (2 * C.hkv));
    if (row >= B.rows) return;
    const int head = part >> 1, which = part & 1;
    const int s = row_sequence(off, B.seqs, row);
    if (s < 0) return;
    const RowSpan span = row_span(off, s, B.rows);
    const int64_t t = static_cast<int64_t>(B.tokens[s]) - (span.end - row);
    if (t < 0 || (t >> C.shift) >= B.width) return;
    const int32_t page = B.table[static_cast<int64_t>(s) * B.width + (t >> C.shift)];
    const int64_t at = cache_row(page, C.pages, C.hkv, head, C.shift, static_cast<int>(t));
    if (at < 0) return;
    const uint16_t* src = which ? v + row * vs : k + row * ks;
    const uint4 x = *reinterpret_cast<const uint4*>(src + head * D + lane * 8);
    void* dst = which ? C.values : C.keys;
    if constexpr (!Q8) {
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(dst) + at * D + lane * 8) = x;
    } else {
        // the largest magnitude as a bit pattern: ordered as the values are, infinities and NaN on top
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) top = max(top, max(w[i] & 0x7fffu, (w[i] >> 16) & 0x7fffu));
#pragma unroll
        for (int m = L / 2; m >= 1; m >>= 1) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), m, L)));
        const bool finite = top < 0x7f80u;
        const float a = bf2f(static_cast<uint16_t>(top));
        // x * 127 would overflow for the largest x: both are brought down by a power of two
        const float down = a > 0x1.0p+100f ? 0x1.0p-64f : 1.0f;
        const float b = a * down;
        uint32_t code[2] = {0, 0};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float f = (i & 1 ? bfhi(w[i >> 1]) : bflo(w[i >> 1])) * down;
            // (127 x is exact in 24 bits and the quotient rounded once: never across a tie)
            const int c = finite && a > 0.0f ? static_cast<int>(rintf(f * 127.0f / b)) : 0;
            code[i >> 2] |= (static_cast<uint32_t>(c) & 0xffu) << (8 * (i & 3));
        }
        *reinterpret_cast<uint2*>(static_cast<int8_t*>(dst) + at * D + lane * 8) = make_uint2(code[0], code[1]);
        if (lane == 0) (which ? C.vs : C.ks)[at] = finite ? a / 127.0f : __uint_as_float(0x7fc00000u);
    }
}

// One wave per (row, query head); lane l holds dims l D/64 .. of the query, the output and each
// token's key and value.
template <int D, bool Q8>
__global__ __launch_bounds__(64) void k_paged_attn(PagedCacheDev C, PagedBatchDev B, const uint16_t* __restrict__ q,
                                                   int64_t qs, int hq, float scale, uint16_t* __restrict__ out,
                                                   int64_t os) {
    constexpr int E = D / 64;
    const int row = blockIdx.x, h = blockIdx.y, lane = threadIdx.x;
    const int s = row_sequence(B.off, B.seqs, row);
    if (s < 0) return;
    const RowSpan span = row_span(B.off, s, B.rows);
    const int head = h / (hq / C.hkv);
    int64_t see = static_cast<int64_t>(B.tokens[s]) - (span.end - row) + 1;
    bool bad = false;
    if (B.tokens[s] > (static_cast<int64_t>(B.width) << C.shift)) bad = true, see = 0;
    float qv[E], o[E] = {};
#pragma unroll
    for (int e = 0; e < E; ++e) qv[e] = bf2f(q[row * qs + h * D + lane * E + e]);
    float m = -INFINITY, sum = 0.0f;
    for (int64_t t = 0; t < see; ++t) {
        const int32_t page = B.table[static_cast<int64_t>(s) * B.width + (t >> C.shift)];
        const int64_t at = cache_row(page, C.pages, C.hkv, head, C.shift, static_cast<int>(t));
        if (at < 0) {
            bad = true;
            break;
        }
        float kv[E], vv[E], dot = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int64_t i = at * D + lane * E + e;
            kv[e] = Q8 ? static_cast<const int8_t*>(C.keys)[i] : bf2f(static_cast<const uint16_t*>(C.keys)[i]);
            vv[e] = Q8 ? static_cast<const int8_t*>(C.values)[i] : bf2f(static_cast<const uint16_t*>(C.values)[i]);
            dot = fmaf(qv[e], kv[e], dot);
        }
        dot = wave_sum_xor(dot) * scale;
        if (Q8) dot *= C.ks[at];
        const float top = fmaxf(m, dot);
        // (a score of -inf leaves the row as it was; NaN reaches the sum)
        const float keep = top == -INFINITY ? 1.0f : expf(m - top);
        const float p = dot == -INFINITY ? 0.0f : expf(dot - top);
        m = top;
        sum = sum * keep + p;
        const float pv = Q8 ? p * C.vs[at] : p;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = fmaf(pv, vv[e], o[e] * keep);
    }
    const float inv = bad ? __uint_as_float(0x7fc00000u) : see > 0 ? 1.0f / sum : 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) out[row * os + h * D + lane * E + e] = f2bf(see > 0 || bad ? o[e] * inv : 0.0f);
}

} // namespace

hipError_t launch_paged_append(const PagedCacheDev& C, bool q8, const PagedBatchDev& B, const uint16_t* k, int64_t ks,
                               const uint16_t* v, int64_t vs, hipStream_t st) {
    const int64_t units = static_cast<int64_t>(B.rows) * 2 * C.hkv;
    const dim3 grid(static_cast<unsigned>((units * (C.d / 8) + 255) / 256));
    const size_t lds = (static_cast<size_t>(B.seqs) + 1) * 4;
    auto go = [&](auto kern) { return launch(kern, grid, dim3(256), lds, st, C, B, k, ks, v, vs); };
    if (q8) return C.d == 64 ? go(k_paged_append<64, true>) : C.d == 128 ? go(k_paged_append<128, true>) : go(k_paged_append<256, true>);
    return C.d == 64 ? go(k_paged_append<64, false>) : C.d == 128 ? go(k_paged_append<128, false>) : go(k_paged_append<256, false>);
}

size_t paged_attention_ws(const PagedCacheDev&, const PagedBatchDev&, int, int) { return 0; }

hipError_t launch_paged_attention(const PagedCacheDev& C, bool q8, const PagedBatchDev& B, int, const uint16_t* q,
                                  int64_t qs, int hq, float scale, uint16_t* out, int64_t os, void*, hipStream_t st) {
    const dim3 grid(B.rows, hq);
    auto go = [&](auto kern) { return launch(kern, grid, dim3(64), 0, st, C, B, q, qs, hq, scale, out, os); };
    if (q8) return C.d == 64 ? go(k_paged_attn<64, true>) : C.d == 128 ? go(k_paged_attn<128, true>) : go(k_paged_attn<256, true>);
    return C.d == 64 ? go(k_paged_attn<64, false>) : C.d == 128 ? go(k_paged_attn<128, false>) : go(k_paged_attn<256, false>);
}

} // namespace q38
