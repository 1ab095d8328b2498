// q38_paged.hip — the paged key-value cache of many requests: the append of a batch's new keys
// and values, and causal attention of the new rows over the cache.
//
//   k_paged_append   per (row, kv head, keys / values): the copy into the token's place, or its
//                    8-bit codes and scale
//   k_paged_split    attention of few queries per sequence: equal shares of all sequences' tokens,
//                    one pass with the running maximum and sum of the softmax
//   k_paged_tile     attention of many queries per sequence: tiles of 128 or 256 of them over keys
//                    and values staged in LDS
//   k_paged_join     the pieces of a sequence that several workgroups worked on
#include "q38_device.hpp"
#include "q38_paged.hpp"
#include "q38_internal.hpp"

#include <algorithm>
#include <type_traits>

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

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float floatx2 __attribute__((ext_vector_type(2)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef uint32_t uintx4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((floatx2){lo, hi}, bf16x2));
}
__device__ __forceinline__ float code_f(uint32_t w, int b) { return static_cast<float>(static_cast<int8_t>(w >> (8 * b))); }
__device__ __forceinline__ floatx4 mfma(uintx4 a, uintx4 b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
constexpr float kNan = __builtin_nanf("");
// The largest of the values of lanes u, 16 + u, 32 + u and 48 + u (a swap with itself leaves the lower
// and the upper of two rows' values in both: their order does not matter here).
__device__ __forceinline__ float quarters_max(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// ---- the register layout of the attention products.
// A wave works transposed, on 32 tokens and 16 queries (a column each) at a time: S^T = K Q^T,
// then O^T += V^T P^T, with 16x16x32 products (A: row lane % 16, k 8 (lane / 16) + j; B the same by
// column; result: column lane % 16, rows 4 (lane / 16) + r). The order of a product's rows and of
// its k index is free as long as both operands agree, and it is chosen so that nothing has to
// move between lanes, with u = lane % 16, w = lane / 16:
//   scores   two products per 32 dims: product a (0, 1) has token 8 (u / 4) + 4 a + u % 4 in row u,
//            so that a lane's results, rows 4 w + r of both, are tokens 8 w .. 8 w + 7 of its query:
//            just the k index that the second product wants of its B operand. Keys are read as
//            16-byte runs of a row straight into the operand.
//   values   lane (u, w) reads the rows of tokens 8 w .. 8 w + 7, E = D / 16 dims of each, 16 bytes at
//            a time; pairs of rows are interleaved by byte permutes into E operands of 8 tokens,
//            operand o covering dim o of every lane's run. Results: dims of 4 w + r's runs.
// The softmax statistics of a query live in its column's lanes: rescaling is lane-local too.
template <int D, bool Q8>
struct AttnGeo {
    static constexpr int E = D / 16;                  // dims of a lane's run in the values
    static constexpr int VD = Q8 ? E / 4 : E / 2;     // its dwords
    static constexpr int KS = D / 32;                 // 32-dim products of a score
    static constexpr int KD = Q8 ? D / 64 : D / 32;   // 16-byte loads of a key row and lane
    static constexpr int EC = (Q8 ? 16 : 8) < E ? (Q8 ? 16 : 8) : E;  // dims of one load of the values
    // dim of operand o in the run of lane u (or result row u)
    __device__ static int dim(int u, int o) { return (o / EC) * 16 * EC + EC * u + o % EC; }
};

// 32 tokens' keys of a lane (with their scales), or their values.
template <int D, bool Q8>
struct KeyTile {
    uintx4 k[2][AttnGeo<D, Q8>::KD];
    floatx4 s[2];
};
template <int D, bool Q8>
struct ValueTile {
    uint32_t v[8][AttnGeo<D, Q8>::VD];
    floatx4 s[2];
};

// First cache rows (head rows) of the two 16-token halves of 32 tokens.
struct HalfRows {
    int64_t lo, hi;
    __device__ __forceinline__ int64_t of(int half) const {
        const int64_t a = lo, b = hi;  // (values: a select of addresses would put them in memory)
        return half ? b : a;
    }
};
// A sequence's pages. The 32 tokens from `base` lie in the pages of their two 16-token halves (one
// page, for pages of 32 and more): the numbers are uniform over the wave.
struct PageWalk {
    const int32_t* table;  // the sequence's row, read through the scalar cache: a vector load's wait
                           // would also be one for all keys and values in flight
    int shift, pages, hkv, head, see;
    bool bad;
    // (a page out of range counts as page 0, a half behind the last seen token as that token's page)
    __device__ __forceinline__ int64_t half(int t) {
        typedef const __attribute__((address_space(4))) int32_t scalar_t;
        int page = ((scalar_t*)(reinterpret_cast<uintptr_t>(table)))[min(t, see - 1) >> shift];
        if (static_cast<uint32_t>(page) >= static_cast<uint32_t>(pages)) {
            bad = true;
            page = 0;
        }
        return ((static_cast<int64_t>(page) * hkv + head) << shift) + (t & ((1 << shift) - 1));
    }
    __device__ __forceinline__ HalfRows rows(int base) { return HalfRows{half(base), half(base + 16)}; }
};

template <int D, bool Q8>
__device__ __forceinline__ void load_keys(const PagedCacheDev& C, HalfRows at, int lane, KeyTile<D, Q8>& t) {
    using Geo = AttnGeo<D, Q8>;
    const int u = lane & 15, w = lane >> 4;
    const int64_t row = at.of(u >> 3) + (8 * (u >> 2) & 15) + (u & 3);
    const char* p = static_cast<const char*>(C.keys) + row * (D * (Q8 ? 1 : 2)) + 16 * w;
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int c = 0; c < Geo::KD; ++c)
            t.k[a][c] = *reinterpret_cast<const uintx4*>(p + 4 * a * D * (Q8 ? 1 : 2) + 64 * c);
    if constexpr (Q8) {
        const float* s = C.ks + at.of(w >> 1) + (8 * w & 15);
        t.s[0] = *reinterpret_cast<const floatx4*>(s);
        t.s[1] = *reinterpret_cast<const floatx4*>(s + 4);
    }
}
template <int D, bool Q8>
__device__ __forceinline__ void load_values(const PagedCacheDev& C, HalfRows at, int lane, ValueTile<D, Q8>& t) {
    using Geo = AttnGeo<D, Q8>;
    const int u = lane & 15, w = lane >> 4;
    const int64_t row = at.of(w >> 1) + (8 * w & 15);
    constexpr int B = Q8 ? 1 : 2;
    const char* p = static_cast<const char*>(C.values) + row * (D * B) + Geo::EC * B * u;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        if constexpr (Geo::VD == 1) {
            t.v[j][0] = *reinterpret_cast<const uint32_t*>(p + j * D * B);
        } else if constexpr (Geo::VD == 2) {
            const uint2 x = *reinterpret_cast<const uint2*>(p + j * D * B);
            t.v[j][0] = x.x, t.v[j][1] = x.y;
        } else {
#pragma unroll
            for (int c = 0; c < Geo::VD / 4; ++c) {
                const uintx4 x = *reinterpret_cast<const uintx4*>(p + j * D * B + 256 * c);
#pragma unroll
                for (int i = 0; i < 4; ++i) t.v[j][4 * c + i] = x[i];
            }
        }
    }
    if constexpr (Q8) {
        t.s[0] = *reinterpret_cast<const floatx4*>(C.vs + row);
        t.s[1] = *reinterpret_cast<const floatx4*>(C.vs + row + 4);
    }
}

// The queries of a tile as B operands: column lane % 16 of each group of 16.
template <int D, bool Q8, int MT>
struct QueryTile {
    uintx4 q[MT][AttnGeo<D, Q8>::KS];
    // (a negative scale turns the queries' signs, so that the softmax's factor is not negative)
    __device__ __forceinline__ void load(const uint16_t* q0, int64_t qs, const AttnItem& it, const AttnSplit& S, int head,
                                         int m0, bool negate, int lane) {
        const int u = lane & 15, w = lane >> 4;
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            const int idx = it.tile * S.M + m0 + 16 * m + u;
            const bool live = idx < it.rows * S.G;
            const uint16_t* p = q0 + (it.first + (live ? idx / S.G : 0)) * qs + (head * S.G + (live ? idx % S.G : 0)) * D;
#pragma unroll
            for (int c = 0; c < AttnGeo<D, Q8>::KS; ++c) {
                // (the keys' 16-byte loads hold 16 dims of an 8-bit row, 8 of a bf16 one)
                const int d = Q8 ? 64 * (c >> 1) + 16 * w + 8 * (c & 1) : 32 * c + 8 * w;
                q[m][c] = live ? *reinterpret_cast<const uintx4*>(p + d) ^ (negate ? 0x80008000u : 0u) : (uintx4){0, 0, 0, 0};
            }
        }
    }
};

// The running softmax of a wave's queries and its sum of the values.
template <int D, bool Q8, int MT>
struct AttnState {
    using Geo = AttnGeo<D, Q8>;
    floatx4 o[MT][Geo::E];
    // the sum of the probabilities. bf16 caches: of the rounded ones, by a product with ones (every
    // result row is the sum over all tokens), so that a row whose weight lies on one token gives
    // its value without their rounding; Q8: of the lane's own tokens (all[m][0]).
    floatx4 all[MT];
    float top[MT];
    int lim[MT];             // tokens that the query sees

    __device__ __forceinline__ void clear(const AttnItem& it, const AttnSplit& S, int m0, int lane) {
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            const int idx = it.tile * S.M + m0 + 16 * m + (lane & 15);
            lim[m] = idx < it.rows * S.G ? attn_see(it, idx / S.G) : 0;
            top[m] = -INFINITY;
            all[m] = (floatx4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int o_ = 0; o_ < Geo::E; ++o_) o[m][o_] = (floatx4){0.0f, 0.0f, 0.0f, 0.0f};
        }
    }

    // From the 32 tokens' products of query group m: the new maximum, the probabilities as the
    // second product's B operand, and their sum. MASKED steps: some query does not see all tokens.
    __device__ __forceinline__ void soften(int m, const floatx4 (&s)[2], const floatx4 (&ks)[2], float c, int base,
                                           bool masked, int lane, float (&p)[8]) {
        const int first = base + 8 * (lane >> 4);
        float best = -INFINITY;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            p[j] = s[j >> 2][j & 3];
            if constexpr (Q8) p[j] *= ks[j >> 2][j & 3];
        }
        if (masked) {
#pragma unroll
            for (int j = 0; j < 8; ++j) p[j] = first + j < lim[m] ? p[j] : -INFINITY;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) best = fmaxf(best, p[j]);
        best = quarters_max(best);
        best = best == -INFINITY ? best : best * c;  // (c may be 0)
        if (__any(best > top[m])) {  // rare after the first tokens: the sums are brought to the new maximum
            const float now = fmaxf(best, top[m]);
            const float keep = now == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(top[m] - now);
            top[m] = now;
            all[m] *= keep;
#pragma unroll
            for (int o_ = 0; o_ < Geo::E; ++o_) o[m][o_] *= keep;
        }
        // (no seen token yet: the scores are -inf, and so are their differences from 0)
        const float ref = top[m] == -INFINITY ? 0.0f : top[m];
#pragma unroll
        for (int j = 0; j < 8; ++j) p[j] = __builtin_amdgcn_exp2f(fmaf(p[j], c, -ref));
        if (masked) {
#pragma unroll
            for (int j = 0; j < 8; ++j) p[j] = first + j < lim[m] ? p[j] : 0.0f;
        }
        if constexpr (Q8) {
#pragma unroll
            for (int j = 0; j < 8; ++j) all[m][0] += p[j];
        }
    }
    // The sum over all tokens, the same in the four lanes of a query.
    __device__ __forceinline__ float total(int m) const {
        float v = all[m][0];
        if constexpr (Q8) {
            v += xor_lane_f<16>(v);
            v += xor_lane_f<32>(v);
        }
        return v;
    }

    __device__ __forceinline__ void scores(const KeyTile<D, Q8>& k, const QueryTile<D, Q8, MT>& q, float c, int base,
                                           bool masked, int lane, float (&p)[MT][8]) {
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            floatx4 s[2];
#pragma unroll
            for (int a = 0; a < 2; ++a) {
                s[a] = (floatx4){0.0f, 0.0f, 0.0f, 0.0f};
                if constexpr (!Q8) {
#pragma unroll
                    for (int i = 0; i < Geo::KS; ++i) s[a] = mfma(k.k[a][i], q.q[m][i], s[a]);
                } else {
#pragma unroll
                    for (int i = 0; i < Geo::KS; ++i) {
                        // codes are integers of at most 8 bits: exact in bf16
                        const uint32_t x = k.k[a][i >> 1][2 * (i & 1)], y = k.k[a][i >> 1][2 * (i & 1) + 1];
                        const uintx4 b = {pack_bf16(code_f(x, 0), code_f(x, 1)), pack_bf16(code_f(x, 2), code_f(x, 3)),
                                          pack_bf16(code_f(y, 0), code_f(y, 1)), pack_bf16(code_f(y, 2), code_f(y, 3))};
                        s[a] = mfma(b, q.q[m][i], s[a]);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
            }
            soften(m, s, k.s, c, base, masked, lane, p[m]);
        }
    }

    // O^T += V^T P^T; the probabilities, at most 1, are rounded to bf16 for it (with the value's
    // scale in a Q8 cache): half a step of each against the value it multiplies, as the output's
    // own rounding.
    __device__ __forceinline__ void weights(const float (&p)[MT][8], const floatx4 (&vs)[2], int base, int lane,
                                            uintx4 (&b)[MT]) {
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                x[j] = p[m][j];
                // (an unseen token's scale may be anything)
                if constexpr (Q8) x[j] = base + 8 * (lane >> 4) + j < lim[m] ? x[j] * vs[j >> 2][j & 3] : 0.0f;
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) b[m][j] = pack_bf16(x[2 * j], x[2 * j + 1]);
        }
    }
    template <bool CODES>  // the values as 8-bit codes, not as bf16
    __device__ __forceinline__ void products(const ValueTile<D, CODES>& t, const uintx4 (&b)[MT]) {
        if constexpr (!Q8) {
            constexpr uint32_t one = 0x3f803f80u;
#pragma unroll
            for (int m = 0; m < MT; ++m) all[m] = mfma((uintx4){one, one, one, one}, b[m], all[m]);
        }
#pragma unroll
        for (int o_ = 0; o_ < Geo::E; ++o_) {
            uintx4 a;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (CODES)
                    a[j] = pack_bf16(code_f(t.v[2 * j][o_ >> 2], o_ & 3), code_f(t.v[2 * j + 1][o_ >> 2], o_ & 3));
                else
                    a[j] = __builtin_amdgcn_perm(t.v[2 * j + 1][o_ >> 1], t.v[2 * j][o_ >> 1],
                                                 o_ & 1 ? 0x07060302u : 0x05040100u);
            }
#pragma unroll
            for (int m = 0; m < MT; ++m) o[m][o_] = mfma(a, b[m], o[m][o_]);
            // (an operand or two at a time: formed all at once they would take the tile's size again)
            if (o_ & 1) __builtin_amdgcn_sched_barrier(0);
        }
    }
    __device__ __forceinline__ void values(const ValueTile<D, Q8>& t, const float (&p)[MT][8], int base, int lane) {
        uintx4 b[MT];
        weights(p, t.s, base, lane, b);
        products<Q8>(t, b);
    }
    // the same for values widened to bf16 on their way, with their scales beside them
    __device__ __forceinline__ void values16(const ValueTile<D, false>& t, const floatx4 (&vs)[2], const float (&p)[MT][8],
                                             int base, int lane) {
        uintx4 b[MT];
        weights(p, vs, base, lane, b);
        products<false>(t, b);
    }
};

// bf16 values in steps that not every query of a tile sees whole. A product of a probability 0 and
// an infinity or NaN is NaN, so tokens that nobody sees and elements that are not finite are
// cleared; true where a seen one was not finite (never, in a healthy model): the outputs of the
// queries that see it take it at the end (add_special).
__device__ __forceinline__ uint32_t special_mask(uint32_t x) {
    return ((x & 0x7f80u) == 0x7f80u ? 0xffffu : 0u) | ((x & 0x7f800000u) == 0x7f800000u ? 0xffff0000u : 0u);
}
template <int D>
__device__ __forceinline__ bool clean_values(ValueTile<D, false>& t, int base, int see, int lane) {
    uint32_t any = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const bool dead = base + 8 * (lane >> 4) + j >= see;
#pragma unroll
        for (int i = 0; i < AttnGeo<D, false>::VD; ++i) {
            const uint32_t x = dead ? 0u : t.v[j][i], m = special_mask(x);
            any |= m;
            t.v[j][i] = x & ~m;
        }
    }
    return __any(any != 0);
}
// The first token of the steps that a tile's queries do not see whole.
__device__ __forceinline__ int special_from(int all) { return all & ~31; }
// Dims d .. d + 3 of a query's sum, with the non-finite values of the tokens t0 .. lim - 1 (their
// weights are positive: an infinity or NaN comes out whatever they are).
template <int D>
__device__ __forceinline__ floatx4 add_special(const PagedCacheDev& C, const int32_t* table, int head, int t0, int lim,
                                               int d, floatx4 x) {
    for (int t = t0; t < lim; ++t) {
        const int64_t at = cache_row(table[t >> C.shift], C.pages, C.hkv, head, C.shift, t);
        if (at < 0) continue;
        const uint2 v = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(C.values) + at * D + d);
        const uint32_t m0 = special_mask(v.x), m1 = special_mask(v.y);
        x[0] += bflo(v.x & m0), x[1] += bfhi(v.x & m0), x[2] += bflo(v.y & m1), x[3] += bfhi(v.y & m1);
    }
    return x;
}

constexpr int kSplitWaves = 4;                 // waves of a workgroup
constexpr int kSplitTokens = 32 * kSplitWaves; // tokens of a step

__device__ __forceinline__ int64_t uniform(int64_t v) {  // a value that every lane holds, in scalar registers
    const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v));
    const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(static_cast<uint64_t>(v) >> 32));
    return static_cast<int64_t>((static_cast<uint64_t>(hi) << 32) | lo);
}
// Where the share's first step lies: the sequence that holds step w * share of the list, and that
// sequence's first step; returns the list's length. Every wave finds it by itself, 64 sequences a
// round (a scan over the workgroup took two barriers and 2 us of the smallest calls); up to 64 sequences
// are weighed once.
__device__ __forceinline__ int64_t find_share(const AttnSplit& S, const PagedBatchDev& B, int shift, int64_t w, int64_t W,
                                              int* seq, int64_t* seq_start, int64_t* share) {
    const int lane = threadIdx.x & 63;
    auto weight = [&](int s) { return s < B.seqs ? static_cast<int64_t>(attn_weight(S, B, shift, s)) : 0; };
    int64_t mine = 0, sum = 0;
    for (int s0 = 0; s0 < B.seqs; s0 += 64) sum += mine = weight(s0 + lane);
    for (int d = 32; d >= 1; d >>= 1) sum += __shfl_xor(sum, d);
    sum = uniform(sum);
    *share = (sum + W - 1) / W;
    const int64_t want = w * *share;
    int64_t before = 0;
    for (int s0 = 0; s0 < B.seqs && want < sum; s0 += 64) {
        if (B.seqs > 64) mine = weight(s0 + lane);
        int64_t upto = mine;
        for (int d = 1; d < 64; d <<= 1) {
            const int64_t x = __shfl_up(upto, d);
            if (lane >= d) upto += x;
        }
        const uint64_t past = __ballot(before + upto > want);
        if (past) {
            const int l = __builtin_ctzll(past);
            *seq = __builtin_amdgcn_readfirstlane(s0 + l);
            *seq_start = before + uniform(__shfl(upto - mine, l));
            break;
        }
        before += uniform(__shfl(upto, 63));
    }
    return sum;
}

// A workgroup's share of a kv head's steps; wave i takes tokens 32 i .. 32 i + 31 of every step, the
// next step's keys and values in flight, and the waves' sums are joined through LDS at the end of
// a piece. Few queries per token: bound by the cache's bytes.
template <int D, bool Q8, int MT>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void k_paged_split(PagedCacheDev C, PagedBatchDev B, int G,
                                                                           const uint16_t* __restrict__ q, int64_t qs,
                                                                           float c, uint16_t* __restrict__ out, int64_t os,
                                                                           float* __restrict__ part) {
    using Geo = AttnGeo<D, Q8>;
    constexpr int M = 16 * MT, LR = D + 4;  // (rows of the waves' sums padded: 16 bytes move the banks)
    extern __shared__ float lds[];          // [waves][M][LR], then [waves][M] maxima and sums
    __shared__ int flags[kSplitWaves];
    const AttnSplit S{G, M, kSplitTokens};
    const int w = blockIdx.x, W = gridDim.x, head = blockIdx.y;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int seq = 0;
    int64_t seq_start = 0, share = 0;
    const int64_t total = find_share(S, B, C.shift, w, W, &seq, &seq_start, &share);
    int64_t pos = w * share;
    const int64_t end = min(total, pos + share);
    AttnPiece pc;
    while (attn_next(S, B, C.shift, end, &seq, &seq_start, &pos, &pc)) {
        const AttnItem& it = pc.it;
        PageWalk walk{B.table + static_cast<int64_t>(it.seq) * B.width, C.shift, C.pages, C.hkv, head, it.see, it.bad};
        // tokens that every query of the tile sees: steps below need no mask
        const int all = attn_see(it, it.tile * M / G);
        QueryTile<D, Q8, MT> qt;
        AttnState<D, Q8, MT> st;
        qt.load(q, qs, it, S, head, 0, c < 0.0f, lane);
        st.clear(it, S, 0, lane);
        KeyTile<D, Q8> kt;
        ValueTile<D, Q8> vt;
        int base = pc.from * kSplitTokens + 32 * wave;
        const int stop = min(pc.to * kSplitTokens, it.see);
        HalfRows at{0, 0};
        bool special = false;
        if (base < stop) {
            at = walk.rows(base);
            load_keys<D, Q8>(C, at, lane, kt);
            load_values<D, Q8>(C, at, lane, vt);
            if (base + kSplitTokens < stop) at = walk.rows(base + kSplitTokens);
        }
        for (; base < stop; base += kSplitTokens) {
            const bool more = base + kSplitTokens < stop, masked = base + 32 > all;
            float p[MT][8];
            st.scores(kt, qt, fabsf(c), base, masked, lane, p);
            if (more) load_keys<D, Q8>(C, at, lane, kt);
            if constexpr (!Q8)
                if (masked) special |= clean_values<D>(vt, base, it.see, lane);
            st.values(vt, p, base, lane);
            if (more) load_values<D, Q8>(C, at, lane, vt);
            if (base + 2 * kSplitTokens < stop) at = walk.rows(base + 2 * kSplitTokens);
        }
        // join the waves
        float* stats = lds + kSplitWaves * M * LR;
        __syncthreads();  // (the previous piece's sums have been read)
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            float sum = st.total(m);
            if (walk.bad) sum = kNan;
            const int row = 16 * m + (lane & 15);
            if (lane < 16) {
                stats[wave * M + row] = st.top[m];
                stats[(kSplitWaves + wave) * M + row] = sum;
            }
            float* dst = lds + (wave * M + row) * LR;
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int o = 0; o < Geo::E; o += 4)
                    *reinterpret_cast<floatx4*>(dst + Geo::dim(4 * (lane >> 4) + r, o)) =
                        (floatx4){st.o[m][o][r], st.o[m][o + 1][r], st.o[m][o + 2][r], st.o[m][o + 3][r]};
        }
        if (lane == 0) flags[wave] = special;
        __syncthreads();
        special = (flags[0] | flags[1] | flags[2] | flags[3]) != 0;
        const bool whole = pc.to - pc.from == it.steps;
        float* pd = nullptr;
        if (!whole) pd = part + ((static_cast<int64_t>(head) * W + w) * 2 + attn_slot(pc.start, share, w)) * (M * (D + 2));
        for (int e = threadIdx.x; e < M * D / 4; e += 256) {
            const int row = e / (D / 4), d = e % (D / 4) * 4, idx = it.tile * M + row;
            if (idx >= it.rows * G) continue;
            float top = stats[row];
#pragma unroll
            for (int i = 1; i < kSplitWaves; ++i) top = fmaxf(top, stats[i * M + row]);
            const float ref = top == -INFINITY ? 0.0f : top;
            float sum = 0.0f;
            floatx4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < kSplitWaves; ++i) {
                const float f = __builtin_amdgcn_exp2f(stats[i * M + row] - ref);
                sum += stats[(kSplitWaves + i) * M + row] * f;
                o += *reinterpret_cast<const floatx4*>(lds + (i * M + row) * LR + d) * f;
            }
            if constexpr (!Q8)
                if (special)
                    o = add_special<D>(C, walk.table, head, max(special_from(all), pc.from * kSplitTokens),
                                       min(stop, attn_see(it, idx / G)), d, o);
            if (whole) {
                const float inv = it.bad || attn_see(it, idx / G) > 0 ? 1.0f / sum : 0.0f;
                const uint2 x = make_uint2(pack_bf16(o[0] * inv, o[1] * inv), pack_bf16(o[2] * inv, o[3] * inv));
                *reinterpret_cast<uint2*>(out + (it.first + idx / G) * os + (head * G + idx % G) * D + d) = x;
            } else {
                *reinterpret_cast<floatx4*>(pd + row * D + d) = o;
                if (d == 0) pd[M * D + row] = top, pd[M * D + M + row] = sum;
            }
        }
    }
}

// ---- many queries per sequence. A workgroup takes M = 32 x waves queries of one item and one of
// `splits` equal ranges of its tokens; keys and values go through LDS, TB tokens at a time and the
// next ones in flight (an 8-bit cache is converted on the way: its codes are exact in bf16), and
// every wave multiplies them with its own 32 queries. Bound by the matrix cores, by the
// exponentials beside them (8 per lane for 16 products of 128 dims) and by LDS reads, which 32
// queries per wave bring to the matrix cores' own time.
template <int D>
struct TileGeo {
    static constexpr int WAVES = 4;
    static constexpr int M = 32 * WAVES;
    static constexpr int TB = D == 64 ? 64 : 32;
    static constexpr int CH = D / 8;                       // 16-byte chunks of a bf16 row
    static constexpr int PIECES = TB * CH / (64 * WAVES);  // chunks per thread
    static constexpr size_t kLds = 2 * (2 * static_cast<size_t>(TB) * D * 2 + 2 * TB * 4);
};
// Place of a token's chunk in its tile: a wave's 16-byte reads of the keys go down 16 rows, 8 of
// which (token % 4, token / 8 % 2) get chunks of their own banks.
template <int D>
__device__ __forceinline__ int tile_at(int token, int chunk) {
    return token * (D / 8) + (chunk ^ ((token & 3) | ((token >> 1) & 4)));
}

// Which item a workgroup takes: the sequences' tiles in order, a sequence's last (longest) first.
__device__ __forceinline__ bool find_tile(const AttnSplit& S, const PagedBatchDev& B, int shift, int want, AttnItem* it) {
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int s0 = 0; s0 < B.seqs; s0 += 64) {
        const int s = s0 + lane;
        int n = 0;
        if (s < B.seqs) {
            const RowSpan span = row_span(B.off, s, B.rows);
            n = attn_tiles(S, span.end - span.begin);
        }
        int upto = n;
        for (int d = 1; d < 64; d <<= 1) {
            const int x = __shfl_up(upto, d);
            if (lane >= d) upto += x;
        }
        const uint64_t past = __ballot(before + upto > want);
        if (past) {
            const int l = __builtin_ctzll(past);
            attn_sequence(B, shift, __builtin_amdgcn_readfirstlane(s0 + l), it);
            const int tiles = __builtin_amdgcn_readfirstlane(__shfl(n, l));
            const int start = before + __builtin_amdgcn_readfirstlane(__shfl(upto, l)) - tiles;
            attn_tile(S, tiles - 1 - (want - start), it);
            return true;
        }
        before += __builtin_amdgcn_readfirstlane(__shfl(upto, 63));
    }
    return false;
}

template <int D, bool Q8>
__global__ __launch_bounds__(64 * TileGeo<D>::WAVES, D == 256 ? 1 : 2) void k_paged_tile(
    PagedCacheDev C, PagedBatchDev B, int G, const uint16_t* __restrict__ q, int64_t qs, float c, uint16_t* __restrict__ out,
    int64_t os, float* __restrict__ part) {
    using Geo = AttnGeo<D, false>;
    using TG = TileGeo<D>;
    constexpr int TB = TG::TB, NT = 64 * TG::WAVES, CH = TG::CH, PC = TG::PIECES, MT = 2;
    extern __shared__ uintx4 tiles[];  // [2][keys, values][TB][CH], then [2][key, value scales][TB]
    float* const scales = reinterpret_cast<float*>(tiles + 4 * TB * CH);
    const AttnSplit S{G, TG::M, TB};
    const int head = blockIdx.y, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int u = lane & 15, w = lane >> 4;
    AttnItem it;
    if (!find_tile(S, B, C.shift, blockIdx.x, &it)) return;
    // (read by vector loads: told to be the same for all lanes, for scalar branches)
    it.first = __builtin_amdgcn_readfirstlane(it.first);
    it.rows = __builtin_amdgcn_readfirstlane(it.rows);
    it.tokens = __builtin_amdgcn_readfirstlane(it.tokens);
    it.bad = __builtin_amdgcn_readfirstlane(it.bad);
    attn_tile(S, __builtin_amdgcn_readfirstlane(it.tile), &it);
    const int per = (it.steps + gridDim.z - 1) / gridDim.z, from = blockIdx.z * per, to = min(it.steps, from + per);
    if (from >= to) return;
    const int m0 = wave * 32, i0 = it.tile * TG::M + m0, rows = it.rows * G;
    QueryTile<D, false, MT> qt;
    AttnState<D, Q8, MT> st;
    qt.load(q, qs, it, S, head, m0, c < 0.0f, lane);
    st.clear(it, S, m0, lane);
    c = fabsf(c);
    // tokens that all, and any, of the wave's queries see
    const int all = i0 < rows ? attn_see(it, i0 / G) : 0;
    const int any = i0 < rows ? attn_see(it, min(i0 + 31, rows - 1) / G) : 0;
    const int stop = min(to * TB, it.see);
    const int32_t* table = B.table + static_cast<int64_t>(it.seq) * B.width;
    PageWalk walk{table, C.shift, C.pages, C.hkv, head, max(it.see, 1), it.bad};
    bool special = false;

    // Staging. A wave's piece of a tile lies in 16 tokens of one page: uniform addresses and a lane's
    // own offset. What lies behind the seen tokens is read with them and masked by its reader.
    constexpr int EL = Q8 ? 1 : 2;
    const int ch = threadIdx.x % CH, wt = wave * 64 / CH;  // the wave's first token of a piece
    const uint32_t lane_off = ((lane / CH) * D + 8 * ch) * EL;
    typedef typename std::conditional<Q8, uint2, uintx4>::type raw_t;
    raw_t kr[PC], vr[PC];
    float sr[2] = {0.0f, 0.0f};
    auto fetch = [&](int t0) {
#pragma unroll
        for (int i = 0; i < PC; ++i) {
            const int64_t at = walk.half(t0 + i * (NT / CH) + wt) * (D * EL);
            kr[i] = *reinterpret_cast<const raw_t*>(static_cast<const char*>(C.keys) + at + lane_off);
            vr[i] = *reinterpret_cast<const raw_t*>(static_cast<const char*>(C.values) + at + lane_off);
        }
        if constexpr (Q8)
            if (wave < TB / 16) {  // 16 tokens' scales per wave
                const int64_t at = walk.half(t0 + 16 * wave);
                sr[0] = C.ks[at + u], sr[1] = C.vs[at + u];
            }
    };
    auto widen = [](raw_t x) {
        if constexpr (Q8)
            return (uintx4){pack_bf16(code_f(x.x, 0), code_f(x.x, 1)), pack_bf16(code_f(x.x, 2), code_f(x.x, 3)),
                            pack_bf16(code_f(x.y, 0), code_f(x.y, 1)), pack_bf16(code_f(x.y, 2), code_f(x.y, 3))};
        else
            return x;
    };
    auto stage = [&](int buf) {
#pragma unroll
        for (int i = 0; i < PC; ++i) {
            const int at = tile_at<D>(i * (NT / CH) + wt + lane / CH, ch);
            tiles[(2 * buf) * TB * CH + at] = widen(kr[i]);
            tiles[(2 * buf + 1) * TB * CH + at] = widen(vr[i]);
        }
        if constexpr (Q8)
            if (wave < TB / 16 && lane < 16) {
                scales[2 * buf * TB + 16 * wave + u] = sr[0];
                scales[(2 * buf + 1) * TB + 16 * wave + u] = sr[1];
            }
    };
    // 32 tokens of a staged tile
    auto half = [&](int base, int sub, const uintx4* kt, const uintx4* vt, const float* sc) {
        const bool masked = base + 32 > all;
        auto key = [&](int a, int i) { return kt[tile_at<D>(32 * sub + 8 * (u >> 2) + 4 * a + (u & 3), 4 * i + w)]; };
        ValueTile<D, false> v;
        auto read_values = [&] {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int t = 32 * sub + 8 * w + j;
                if constexpr (D == 64) {
                    const uint2 x = reinterpret_cast<const uint2*>(vt + tile_at<D>(t, u >> 1))[u & 1];
                    v.v[j][0] = x.x, v.v[j][1] = x.y;
                } else {
#pragma unroll
                    for (int b = 0; b < D / 128; ++b) {
                        const uintx4 x = vt[tile_at<D>(t, 16 * b + u)];
#pragma unroll
                        for (int i = 0; i < 4; ++i) v.v[j][4 * b + i] = x[i];
                    }
                }
            }
        };
        floatx4 s[MT][2], ks[2], vs[2];
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
            for (int m = 0; m < MT; ++m) s[m][a] = (floatx4){0.0f, 0.0f, 0.0f, 0.0f};
        if constexpr (D < 256) {  // all reads in flight before the first product, the values' before the softmax
            uintx4 k[2][Geo::KS];
#pragma unroll
            for (int a = 0; a < 2; ++a)
#pragma unroll
                for (int i = 0; i < Geo::KS; ++i) k[a][i] = key(a, i);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int a = 0; a < 2; ++a)
#pragma unroll
                for (int i = 0; i < Geo::KS; ++i)
#pragma unroll
                    for (int m = 0; m < MT; ++m) s[m][a] = mfma(k[a][i], qt.q[m][i], s[m][a]);
            read_values();
        } else {  // (256 dims: no registers for them)
#pragma unroll
            for (int a = 0; a < 2; ++a)
#pragma unroll
                for (int i = 0; i < Geo::KS; ++i) {
                    const uintx4 k = key(a, i);
#pragma unroll
                    for (int m = 0; m < MT; ++m) s[m][a] = mfma(k, qt.q[m][i], s[m][a]);
                }
        }
        if constexpr (Q8)
#pragma unroll
            for (int a = 0; a < 2; ++a) {
                ks[a] = *reinterpret_cast<const floatx4*>(sc + 32 * sub + 8 * w + 4 * a);
                vs[a] = *reinterpret_cast<const floatx4*>(sc + TB + 32 * sub + 8 * w + 4 * a);
            }
        float p[MT][8];
#pragma unroll
        for (int m = 0; m < MT; ++m) st.soften(m, s[m], ks, c, base, masked, lane, p[m]);
        if constexpr (D == 256) read_values();
        if constexpr (!Q8)
            if (masked) special |= clean_values<D>(v, base, any, lane);
        st.values16(v, vs, p, base, lane);
    };
    fetch(from * TB);
    stage(0);
    __syncthreads();
    for (int step = from; step < to; ++step) {
        const int buf = (step - from) & 1;
        fetch(min(step + 1, to - 1) * TB);
        const uintx4* kt = tiles + (2 * buf) * TB * CH;
#pragma unroll
        for (int sub = 0; sub < TB / 32; ++sub)
            if (step * TB + 32 * sub < any) half(step * TB + 32 * sub, sub, kt, kt + TB * CH, scales + 2 * buf * TB);
        stage(buf ^ 1);
        lds_barrier();
    }
    const bool bad = __syncthreads_or(it.bad || (it.see > 0 && walk.bad));
    const bool whole = per >= it.steps;
    float* pd = nullptr;
    if (!whole) pd = part + ((static_cast<int64_t>(blockIdx.x) * C.hkv + head) * gridDim.z + blockIdx.z) * (TG::M * (D + 2));
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        float sum = st.total(m);
        if (bad) sum = kNan;
        const int idx = i0 + 16 * m + u;
        if (idx >= rows) continue;
        const float inv = bad || st.lim[m] > 0 ? 1.0f / sum : 0.0f;
        const int row = m0 + 16 * m + u;
        uint16_t* dst = out + (it.first + idx / G) * os + (head * G + idx % G) * D;
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int o = 0; o < Geo::E; o += 4) {
                const int d = Geo::dim(4 * w + r, o);
                floatx4 x = {st.o[m][o][r], st.o[m][o + 1][r], st.o[m][o + 2][r], st.o[m][o + 3][r]};
                if constexpr (!Q8)
                    if (special)
                        x = add_special<D>(C, table, head, max(special_from(all), from * TB), min(stop, st.lim[m]), d, x);
                if (whole)
                    *reinterpret_cast<uint2*>(dst + d) = make_uint2(pack_bf16(x[0] * inv, x[1] * inv), pack_bf16(x[2] * inv, x[3] * inv));
                else
                    *reinterpret_cast<floatx4*>(pd + row * D + d) = x;
            }
        if (!whole && w == 0) pd[TG::M * D + row] = st.top[m], pd[TG::M * D + TG::M + row] = sum;
    }
}

// Joins the pieces of an item that several workgroups worked on, a workgroup per (row, query head),
// each of its waves every fourth piece, eight in flight. TILES: pieces of k_paged_tile, W ranges per
// item; else those of k_paged_split, W shares.
template <int D, bool TILES>
__global__ __launch_bounds__(256) void k_paged_join(PagedCacheDev C, PagedBatchDev B, AttnSplit S, int W,
                                                    int items, const float* __restrict__ part,
                                                    uint16_t* __restrict__ out, int64_t os) {
    constexpr int E = D / 64;
    __shared__ float sums[4][D + 2];
    const int row = blockIdx.x, lane = threadIdx.x & 63, G = S.G, M = S.M;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = blockIdx.y;
    const int seq = row_sequence(B.off, B.seqs, row);
    if (seq < 0) return;
    // what lies in front of the sequence: steps (and the list's length), or tiles
    int64_t total = 0, start = 0;
    for (int s = lane; s < (TILES ? seq : B.seqs); s += 64) {
        int n;
        if constexpr (TILES) {
            const RowSpan span = row_span(B.off, s, B.rows);
            n = attn_tiles(S, span.end - span.begin);
        } else {
            n = attn_weight(S, B, C.shift, s);
        }
        total += n;
        if (s < seq) start += n;
    }
    for (int d = 32; d >= 1; d >>= 1) {
        total += __shfl_xor(total, d);
        start += __shfl_xor(start, d);
    }
    AttnItem it;
    attn_sequence(B, C.shift, seq, &it);
    const int idx = (row - it.first) * G + h % G, head = h / G, at = idx % M;
    int64_t first, step;  // the first piece, and from one to the next
    int n;
    if constexpr (TILES) {
        attn_tile(S, idx / M, &it);
        const int per = (it.steps + W - 1) / W;
        n = (it.steps + per - 1) / per;
        const int64_t item = start + attn_tiles(S, it.rows) - 1 - it.tile;
        if (item >= items) return;  // (offsets that do not ascend: more tiles than rows)
        first = (item * C.hkv + head) * W;
        step = 1;
    } else {
        const int64_t share = (total + W - 1) / W;
        for (int j = 0; j < idx / M; ++j) {
            attn_tile(S, j, &it);
            start += it.steps;
        }
        attn_tile(S, idx / M, &it);
        const int64_t w0 = start / share, w1 = (start + it.steps - 1) / share;
        n = static_cast<int>(w1 - w0) + 1;
        // (an item goes on behind its first share, whose second slot it takes; it began before the others)
        first = (static_cast<int64_t>(head) * W + w0) * 2 + 1;
        step = 2;
    }
    if (n == 1) return;
    auto piece = [&](int i) { return part + (first + i * step - (!TILES && i > 0)) * (M * (D + 2)); };
    float top = -INFINITY;
    for (int i = lane; i < n; i += 64) top = fmaxf(top, piece(i)[M * D + at]);
    top = wave_max(top);
    const float ref = top == -INFINITY ? 0.0f : top;
    float sum = 0.0f, o[E] = {};
#pragma unroll 8
    for (int i = wave; i < n; i += 4) {
        const float* src = piece(i);
        const float f = __builtin_amdgcn_exp2f(src[M * D + at] - ref);
        sum = fmaf(src[M * D + M + at], f, sum);
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = fmaf(src[at * D + lane * E + e], f, o[e]);
    }
#pragma unroll
    for (int e = 0; e < E; ++e) sums[wave][lane * E + e] = o[e];
    if (lane == 0) sums[wave][D] = sum;
    __syncthreads();
    if (wave) return;
    sum = sums[0][D] + sums[1][D] + sums[2][D] + sums[3][D];
    const float inv = it.bad || attn_see(it, idx / G) > 0 ? 1.0f / sum : 0.0f;
    uint16_t* dst = out + row * os + h * D + lane * E;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int d = lane * E + e;
        dst[e] = f2bf((sums[0][d] + sums[1][d] + sums[2][d] + sums[3][d]) * inv);
    }
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

namespace {

// Up to 32 queries per sequence and kv head the split kernel reads every token once; above, the tile
// kernel does so once per 128 or 256 queries.
struct AttnPlan {
    bool tiles;
    int mt;         // split: 16-query groups
    int W;          // split: workgroups per kv head; tiles: ranges per item
    int items;      // tiles: items at most
    bool joined;
    int M;
};
AttnPlan attn_plan(const PagedCacheDev& C, const PagedBatchDev& B, int max_rows, int hq) {
    AttnPlan p{};
    const int64_t G = hq / C.hkv, queries = max_rows * G, span = static_cast<int64_t>(B.width) << C.shift;
    p.tiles = queries > 32;
    if (!p.tiles) {
        p.mt = queries <= 16 ? 1 : 2;
        p.M = 16 * p.mt;
        p.W = std::max(1, 256 * (C.d == 256 ? 1 : 2) / C.hkv);  // the chip's 256 CUs at the kernel's occupancy
        p.joined = span > kSplitTokens;  // (no sequence of the table is longer than a step: nothing is split)
    } else {
        p.M = TileGeo<64>::M;
        p.items = static_cast<int>(std::min<int64_t>(B.rows * G / p.M + B.seqs, B.rows * G));
        // ranges of at least 256 tokens, until there are about two workgroups per CU
        const int64_t blocks = std::max<int64_t>(1, static_cast<int64_t>(p.items) * C.hkv);
        p.W = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(512 / blocks, (span + 255) / 256)));
        p.joined = p.W > 1;
    }
    return p;
}

template <int D, bool Q8, int MT>
hipError_t launch_split(const PagedCacheDev& C, const PagedBatchDev& B, const AttnPlan& p, const uint16_t* q, int64_t qs,
                        int hq, float c, uint16_t* out, int64_t os, float* part, hipStream_t st) {
    constexpr size_t lds = (static_cast<size_t>(kSplitWaves) * 16 * MT * (D + 4) + 2 * kSplitWaves * 16 * MT) * 4;
    const hipError_t e = ensure_lds<k_paged_split<D, Q8, MT>>(lds);
    if (e != hipSuccess) return e;
    return launch(k_paged_split<D, Q8, MT>, dim3(p.W, C.hkv), dim3(256), lds, st, C, B, hq / C.hkv, q, qs, c, out, os, part);
}
template <int D, bool Q8>
hipError_t launch_attention(const PagedCacheDev& C, const PagedBatchDev& B, const AttnPlan& p, const uint16_t* q, int64_t qs,
                            int hq, float scale, uint16_t* out, int64_t os, float* part, hipStream_t st) {
    const float c = scale * 1.44269504088896341f;  // exponents of 2
    hipError_t e;
    if (!p.tiles) {
        e = p.mt == 1 ? launch_split<D, Q8, 1>(C, B, p, q, qs, hq, c, out, os, part, st)
                      : launch_split<D, Q8, 2>(C, B, p, q, qs, hq, c, out, os, part, st);
    } else {
        e = ensure_lds<k_paged_tile<D, Q8>>(TileGeo<D>::kLds);
        if (e == hipSuccess)
            e = launch(k_paged_tile<D, Q8>, dim3(p.items, C.hkv, p.W), dim3(64 * TileGeo<D>::WAVES), TileGeo<D>::kLds, st, C, B,
                       hq / C.hkv, q, qs, c, out, os, part);
    }
    if (e != hipSuccess || !p.joined) return e;
    const AttnSplit S{hq / C.hkv, p.M, p.tiles ? TileGeo<D>::TB : kSplitTokens};
    const dim3 grid(B.rows, hq);
    return p.tiles ? launch(k_paged_join<D, true>, grid, dim3(256), 0, st, C, B, S, p.W, p.items, part, out, os)
                   : launch(k_paged_join<D, false>, grid, dim3(256), 0, st, C, B, S, p.W, p.items, part, out, os);
}

} // namespace

size_t paged_attention_ws(const PagedCacheDev& C, const PagedBatchDev& B, int max_rows, int hq) {
    const AttnPlan p = attn_plan(C, B, max_rows, hq);
    const size_t pieces = static_cast<size_t>(C.hkv) * p.W * (p.tiles ? p.items : 2);
    return p.joined ? pieces * p.M * (C.d + 2) * 4 : 0;
}

hipError_t launch_paged_attention(const PagedCacheDev& C, bool q8, const PagedBatchDev& B, int max_rows, const uint16_t* q,
                                  int64_t qs, int hq, float scale, uint16_t* out, int64_t os, void* ws, hipStream_t st) {
    const AttnPlan p = attn_plan(C, B, max_rows, hq);
    auto go = [&](auto kern) { return kern(C, B, p, q, qs, hq, scale, out, os, static_cast<float*>(ws), st); };
    if (q8)
        return C.d == 64    ? go(launch_attention<64, true>)
               : C.d == 128 ? go(launch_attention<128, true>)
                            : go(launch_attention<256, true>);
    return C.d == 64    ? go(launch_attention<64, false>)
           : C.d == 128 ? go(launch_attention<128, false>)
                        : go(launch_attention<256, false>);
}

} // namespace q38
