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
// memory, then the search for the row's sequence runs there. Decode steps take a launch's latency, long
// prompts the bytes' time.
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

// The sequence's row of query i of a tile (query i % G of the row's group), or -1 behind the tile's rows.
__device__ __forceinline__ int tile_row(const AttnSplit& S, const AttnItem& it, int i) {
    const int r = i / S.G, row = it.tile * S.rows() + r;
    return r < S.rows() && row < it.rows ? row : -1;
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
            const int row = tile_row(S, it, m0 + 16 * m + u);
            const bool live = row >= 0;
            const uint16_t* p = q0 + (it.first + (live ? row : 0)) * qs + (head * S.G + (m0 + 16 * m + u) % S.G) * D;
#pragma unroll
            for (int c = 0; c < AttnGeo<D, Q8>::KS; ++c) {
                // (the keys' 16-byte loads hold 16 dims of an 8-bit row, 8 of a bf16 one)
                const int d = Q8 ? 64 * (c >> 1) + 16 * w + 8 * (c & 1) : 32 * c + 8 * w;
                q[m][c] = live ? *reinterpret_cast<const uintx4*>(p + d) ^ (negate ? 0x80008000u : 0u) : (uintx4){0, 0, 0, 0};
            }
        }
    }
};

// The running softmax of a wave's queries and its sum of the values, the probabilities in P bf16 parts.
template <int D, bool Q8, int MT, int P>
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
            const int row = tile_row(S, it, m0 + 16 * m + (lane & 15));
            lim[m] = row >= 0 ? attn_see(it, row) : 0;
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
        // (opaque: the compiler would share the comparisons of the two masks and make them in front of the branches, in
        // every step, or not, by what else the kernel holds: five ragged prompts 453 us in place of 430. With 256
        // dims, 16 queries per wave, sharing is better: ragged prompts 341 us against 344, in 8 bits 319 against 322.)
        auto seen_from = [&] {
            int first = base + 8 * (lane >> 4) - lim[m];
            if constexpr (D < 256) asm volatile("" : "+v"(first));
            return first;
        };
        float best = -INFINITY;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            p[j] = s[j >> 2][j & 3];
            if constexpr (Q8) p[j] *= ks[j >> 2][j & 3];
        }
        if (masked) {
            const int first = seen_from();
#pragma unroll
            for (int j = 0; j < 8; ++j) p[j] = first + j < 0 ? p[j] : -INFINITY;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) best = fmaxf(best, p[j]);
        best = quarters_max(best);
        best = best == -INFINITY ? best : best * c;  // (c may be 0)
        // `top` is what exponents are taken from, and need not be the maximum itself: below 2^8 above it
        // the probabilities and their sums are as exact. Rare after the first tokens, then: the sums
        // brought to a new one.
        if (__any(best > top[m] + 8.0f)) {
            const float now = best > top[m] + 8.0f ? best : top[m];  // (a query's own need alone moves it)
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
            const int first = seen_from();
#pragma unroll
            for (int j = 0; j < 8; ++j) p[j] = first + j < 0 ? p[j] : 0.0f;
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
                                           bool masked, int lane, const floatx4 (&vs)[2], uintx4 (&b)[MT][P]) {
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
                        const uintx4 kc = {pack_bf16(code_f(x, 0), code_f(x, 1)), pack_bf16(code_f(x, 2), code_f(x, 3)),
                                          pack_bf16(code_f(y, 0), code_f(y, 1)), pack_bf16(code_f(y, 2), code_f(y, 3))};
                        s[a] = mfma(kc, q.q[m][i], s[a]);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
            }
            float p[8];
            soften(m, s, k.s, c, base, masked, lane, p);
            weights(m, p, vs, base, lane, b[m]);
        }
    }

    // O^T += V^T P^T; the probabilities (with the value's scale in a Q8 cache) are rounded to P bf16 parts
    // for it. One: each is off by up to 2^-8 of itself, as the output by its own rounding (k_paged_tile, many
    // queries of a sequence; a second part took five ragged prompts from 432 to 535 us). Two: by 2^-17
    // (sequences of few queries: k_paged_split, bound by bytes, at most 2.5% of its time, and in k_paged_tile a
    // second wave, whose one part is what the first part leaves: `low`).
    __device__ __forceinline__ void weights(int m, const float (&p)[8], const floatx4 (&vs)[2], int base, int lane,
                                            uintx4 (&b)[P], bool low = false) {
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            x[j] = p[j];
            // (an unseen token's scale may be anything)
            if constexpr (Q8) x[j] = base + 8 * (lane >> 4) + j < lim[m] ? x[j] * vs[j >> 2][j & 3] : 0.0f;
        }
#pragma unroll
        for (int n = 0; n < P; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                b[n][i] = pack_bf16(x[2 * i], x[2 * i + 1]);
                if (n + 1 < P) x[2 * i] -= bflo(b[n][i]), x[2 * i + 1] -= bfhi(b[n][i]);
            }
        if (low)
#pragma unroll
            for (int i = 0; i < 4; ++i) b[0][i] = pack_bf16(x[2 * i] - bflo(b[0][i]), x[2 * i + 1] - bfhi(b[0][i]));
    }
    template <bool CODES>  // the values as 8-bit codes, not as bf16
    __device__ __forceinline__ void products(const ValueTile<D, CODES>& t, const uintx4 (&b)[MT][P]) {
        if constexpr (!Q8) {
            constexpr uint32_t one = 0x3f803f80u;
#pragma unroll
            for (int n = 0; n < P; ++n)
#pragma unroll
                for (int m = 0; m < MT; ++m) all[m] = mfma((uintx4){one, one, one, one}, b[m][n], all[m]);
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
            for (int n = 0; n < P; ++n)
#pragma unroll
                for (int m = 0; m < MT; ++m) o[m][o_] = mfma(a, b[m][n], o[m][o_]);
            // (an operand or two at a time: formed all at once they would take the tile's size again)
            if (o_ & 1) __builtin_amdgcn_sched_barrier(0);
        }
    }
};

// bf16 values in steps that not every query of a tile sees whole. A product of a probability 0 and
// an infinity or NaN is NaN, so tokens that nobody sees and elements that are not finite are
// cleared; true where a seen one was not finite (never, in a healthy model): the outputs of the
// queries that see it take it at the end (add_special).
// All ones in each half of x that is an infinity or NaN (its exponent's carry into the sign's place).
__device__ __forceinline__ uint32_t special_mask(uint32_t x) {
    const uint32_t m = ((x & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
    return m | (m - (m >> 15));
}
template <int D>
__device__ __forceinline__ bool clean_values(ValueTile<D, false>& t, int base, int see, int lane) {
    uint32_t any = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const uint32_t seen = static_cast<uint32_t>((base + 8 * (lane >> 4) + j - see) >> 31);
#pragma unroll
        for (int i = 0; i < AttnGeo<D, false>::VD; ++i) {
            const uint32_t x = t.v[j][i] & seen, m = special_mask(x);
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

constexpr int kSplitQueries = 32;              // queries per sequence and kv head that it is for
constexpr int kSplitWaves = 4;                 // waves of a workgroup
constexpr int kSplitTokens = 32 * kSplitWaves; // tokens of a step

__device__ __forceinline__ int64_t uniform(int64_t v) {  // a value that every lane holds, in scalar registers
    const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v));
    const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(static_cast<uint64_t>(v) >> 32));
    return static_cast<int64_t>((static_cast<uint64_t>(hi) << 32) | lo);
}
// (the 64-bit division's steps are worth avoiding in the smallest calls)
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
    return (a | b) >> 32 ? a / b : static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
}
// The list's length and a share's size, and the item that holds step w * share with its sequence (if the
// list is that long). Every wave finds it by itself, 64 sequences a round, from one load of their lengths (a
// scan over the workgroup took two barriers and 2 us of the smallest calls); up to 64 sequences are weighed
// once.
__device__ __forceinline__ int64_t find_share(const AttnSplit& S, const PagedBatchDev& B, int shift, int64_t w, int64_t W,
                                              AttnCursor* at, AttnItem* seq, int64_t* share) {
    const int lane = threadIdx.x & 63;
    AttnItem it;
    int64_t mine = 0, upto = 0, sum = 0;
    auto weigh = [&](int s) {
        mine = 0;
        if (s < B.seqs) {
            attn_sequence(B, shift, s, &it);
            mine = attn_weight(S, it);
        }
    };
    auto scan = [&] {
        upto = mine;
        for (int d = 1; d < 64; d <<= 1) {
            const int64_t x = __shfl_up(upto, d);
            if (lane >= d) upto += x;
        }
        return uniform(__shfl(upto, 63));
    };
    if (B.seqs <= 64) {
        weigh(lane);
        sum = scan();
    } else {
        for (int s0 = 0; s0 < B.seqs; s0 += 64) weigh(s0 + lane), sum += mine;
        for (int d = 32; d >= 1; d >>= 1) sum += __shfl_xor(sum, d);
        sum = uniform(sum);
    }
    *share = quotient(sum + W - 1, W);
    const int64_t want = w * *share;
    int64_t before = 0;
    for (int s0 = 0; s0 < B.seqs && want < sum; s0 += 64) {
        int64_t these = sum;
        if (B.seqs > 64) {
            weigh(s0 + lane);
            these = scan();
        }
        const uint64_t past = __ballot(before + upto > want);
        if (past) {
            const int l = __builtin_ctzll(past);
            seq->seq = __builtin_amdgcn_readfirstlane(s0 + l);
            seq->first = __builtin_amdgcn_readlane(it.first, l);
            seq->rows = __builtin_amdgcn_readlane(it.rows, l);
            seq->tokens = __builtin_amdgcn_readlane(it.tokens, l);
            seq->bad = __builtin_amdgcn_readlane(it.bad, l);
            const AttnCursor c = attn_seek(S, *seq, before + uniform(__shfl(upto - mine, l)), want);
            *at = AttnCursor{c.seq, __builtin_amdgcn_readfirstlane(c.tile), uniform(c.start)};
            break;
        }
        before += these;
    }
    return sum;
}
// A wave's walk through its share. It lies in LDS between the pieces: nothing of it is needed while a
// piece is worked on, and in registers it cost the inner loops theirs.
struct ShareWalk {
    AttnCursor at;
    int64_t pos, end, share, start;  // start: the current piece's item
    int first, rows, tokens, bad, tile, from, to;

    // false where the share is empty
    __device__ __forceinline__ bool open(const AttnSplit& S, const PagedBatchDev& B, int shift, int64_t w, int64_t W) {
        AttnCursor c{0, 0, 0};
        AttnItem it;
        int64_t sh = 0;
        const int64_t total = find_share(S, B, shift, w, W, &c, &it, &sh);
        if (w * sh >= total) return false;
        if ((threadIdx.x & 63) == 0) {
            at = c, share = sh, pos = w * sh, end = min(total, (w + 1) * sh);
            seq_ = it.seq, first = it.first, rows = it.rows, tokens = it.tokens, bad = it.bad;
        }
        return true;
    }
    // The next piece; the same for all lanes.
    __device__ __forceinline__ bool next(const AttnSplit& S, const PagedBatchDev& B, int shift) {
        AttnCursor c{__builtin_amdgcn_readfirstlane(at.seq), __builtin_amdgcn_readfirstlane(at.tile), uniform(at.start)};
        int64_t p = uniform(pos);
        AttnPiece pc;
        pc.it = sequence();
        if (!attn_next(S, B, shift, uniform(end), &c, &p, &pc)) return false;
        if ((threadIdx.x & 63) == 0) {
            at = c, pos = p, start = pc.start, seq_ = pc.it.seq;
            first = pc.it.first, rows = pc.it.rows, tokens = pc.it.tokens, bad = pc.it.bad, tile = pc.it.tile;
            from = pc.from, to = pc.to;
        }
        return true;
    }
    __device__ __forceinline__ AttnItem sequence() const {
        AttnItem it;
        it.seq = seq();
        it.first = __builtin_amdgcn_readfirstlane(first);
        it.rows = __builtin_amdgcn_readfirstlane(rows);
        it.tokens = __builtin_amdgcn_readfirstlane(tokens);
        it.bad = __builtin_amdgcn_readfirstlane(bad);
        return it;
    }
    __device__ __forceinline__ AttnItem item(const AttnSplit& S) const {
        AttnItem it = sequence();
        attn_tile(S, __builtin_amdgcn_readfirstlane(tile), &it);
        return it;
    }
    __device__ __forceinline__ int seq() const { return __builtin_amdgcn_readfirstlane(seq_); }
    int seq_;
};
// What a share leaves for the join: the item that goes on behind it, if it began in it, and the
// number of its pieces (0: none). They lie at the workspace's start, which is 16-byte aligned.
struct alignas(16) CutItem {
    int pieces, first, rows, tokens, tile, bad, unused[2];
};
static_assert(sizeof(CutItem) == 32 && alignof(CutItem) <= 16, "the partial sums behind them keep the workspace's alignment");
__device__ __forceinline__ void note_cut(CutItem* cut, const ShareWalk& sw, const AttnItem& it) {
    *cut = CutItem{static_cast<int>(quotient(sw.start + it.steps - 1, sw.share) - quotient(sw.start, sw.share)) + 1, it.first, it.rows,
                   it.tokens, it.tile, it.bad};
}

// A workgroup's share of a kv head's steps; wave i takes tokens 32 i .. 32 i + 31 of every step, the
// next step's keys and values in flight, and the waves' sums are joined through LDS at the end of
// a piece. Few queries per token: bound by the cache's bytes (64 ragged requests of one row: 87 us,
// 4.8 TB/s), one request by the latency of its few steps (4,001 tokens: 11.5 us).
template <int D, bool Q8, int MT>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void k_paged_split(PagedCacheDev C, PagedBatchDev B, int G,
                                                                           const uint16_t* __restrict__ q, int64_t qs,
                                                                           float c, uint16_t* __restrict__ out, int64_t os,
                                                                           float* __restrict__ part,
                                                                           CutItem* __restrict__ cuts) {
    using Geo = AttnGeo<D, Q8>;
    constexpr int M = 16 * MT, LR = D + 4;  // (rows of the waves' sums padded: 16 bytes move the banks)
    extern __shared__ float lds[];          // [waves][M][LR], then [waves][M] maxima and sums
    __shared__ int flags[kSplitWaves];
    const AttnSplit S{G, M, kSplitTokens};
    const int w = blockIdx.x, W = gridDim.x, head = blockIdx.y;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    __shared__ ShareWalk walks[kSplitWaves];
    ShareWalk& sw = walks[wave];
    CutItem* const cut = cuts + head * W + w;
    if (threadIdx.x == 0) cut->pieces = 0;
    if (!sw.open(S, B, C.shift, w, W)) return;
    while (sw.next(S, B, C.shift)) {
        // (opaque: what follows from the lane is formed anew per piece, not kept in registers for the next)
        int lane = threadIdx.x & 63;
        asm volatile("" : "+v"(lane));
        AttnItem it = sw.item(S);
        PageWalk walk{B.table + static_cast<int64_t>(sw.seq()) * B.width, C.shift, C.pages, C.hkv, head, it.see, it.bad};
        // tokens that every query of the tile sees: steps below need no mask
        const int all = attn_see(it, it.tile * S.rows());
        QueryTile<D, Q8, MT> qt;
        AttnState<D, Q8, MT, 2> st;
        qt.load(q, qs, it, S, head, 0, c < 0.0f, lane);
        st.clear(it, S, 0, lane);
        KeyTile<D, Q8> kt;
        ValueTile<D, Q8> vt;
        int base = __builtin_amdgcn_readfirstlane(sw.from) * kSplitTokens + 32 * wave;
        const int stop = min(__builtin_amdgcn_readfirstlane(sw.to) * kSplitTokens, it.see);
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
            uintx4 b[MT][2];
            st.scores(kt, qt, fabsf(c), base, masked, lane, vt.s, b);
            if (more) load_keys<D, Q8>(C, at, lane, kt);
            if constexpr (!Q8)
                if (masked) special |= clean_values<D>(vt, base, it.see, lane);
            st.template products<Q8>(vt, b);
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
        asm volatile("" ::: "memory");  // (read anew: see ShareWalk)
        it = sw.item(S);
        const int from = sw.from;
        const bool whole = sw.to - from == it.steps;
        float* pd = nullptr;
        if (!whole) {
            const int slot = attn_slot(sw.start, sw.share, w);
            pd = part + ((static_cast<int64_t>(head) * W + w) * 2 + slot) * (M * (D + 2));
            if (slot && threadIdx.x == 0) note_cut(cut, sw, it);
        }
        for (int e = threadIdx.x; e < M * D / 4; e += 256) {
            const int i = e / (D / 4), d = e % (D / 4) * 4, row = tile_row(S, it, i);
            if (row < 0) continue;
            float top = stats[i];
#pragma unroll
            for (int n = 1; n < kSplitWaves; ++n) top = fmaxf(top, stats[n * M + i]);
            const float ref = top == -INFINITY ? 0.0f : top;
            float sum = 0.0f;
            floatx4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int n = 0; n < kSplitWaves; ++n) {
                const float f = __builtin_amdgcn_exp2f(stats[n * M + i] - ref);
                sum += stats[(kSplitWaves + n) * M + i] * f;
                o += *reinterpret_cast<const floatx4*>(lds + (n * M + i) * LR + d) * f;
            }
            if constexpr (!Q8)
                if (special)
                    o = add_special<D>(C, walk.table, head, max(special_from(all), from * kSplitTokens),
                                       min(stop, attn_see(it, row)), d, o);
            if (whole) {
                const float inv = it.bad || attn_see(it, row) > 0 ? 1.0f / sum : 0.0f;
                const uint2 x = make_uint2(pack_bf16(o[0] * inv, o[1] * inv), pack_bf16(o[2] * inv, o[3] * inv));
                *reinterpret_cast<uint2*>(out + (it.first + row) * os + (head * G + i % G) * D + d) = x;
            } else {
                *reinterpret_cast<floatx4*>(pd + i * D + d) = o;
                if (d == 0) pd[M * D + i] = top, pd[M * D + M + i] = sum;
            }
        }
    }
}

// ---- many queries per sequence. Tiles of 256 queries (128 of 256 dims) in equal shares as above;
// keys and values go through LDS, TB tokens at a time and the next ones in flight (an 8-bit cache is
// converted on the way: its codes are exact in bf16), and every wave multiplies them with its own 32
// queries. Bound by the matrix cores, by the exponentials beside them (8 per lane for 16 products of 128
// dims) and by LDS reads, which 32 queries per wave bring to the matrix cores' own time: five ragged
// prompts, 5,647 rows of 32 heads of 128 over 20,306 tokens, in 430 us with their join, 697 TFLOP/s (4.9 ms
// with k_paged_split).
template <int D>
struct TileGeo {
    // One workgroup of two waves per SIMD fills a CU: two workgroups of one each share it unevenly (the
    // older one's waves go first: done after 430 us, the other's after 525) and leave it half empty at the
    // end, 24% longer for five ragged prompts. 16-query groups per wave (MT): 256 dims take the
    // registers of two.
    static constexpr int MT = D == 256 ? 1 : 2, WAVES = 8, M = 16 * MT * WAVES;
    static constexpr int TB = D == 256 ? 32 : 64;
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

template <int D, bool Q8>
__global__ __launch_bounds__(64 * TileGeo<D>::WAVES, 2) void k_paged_tile(
    PagedCacheDev C, PagedBatchDev B, int G, int shares, const uint16_t* __restrict__ q, int64_t qs, float c,
    uint16_t* __restrict__ out, int64_t os, float* __restrict__ part, CutItem* __restrict__ cuts) {
    using Geo = AttnGeo<D, false>;
    using TG = TileGeo<D>;
    constexpr int TB = TG::TB, NT = 64 * TG::WAVES, CH = TG::CH, PC = TG::PIECES, MT = TG::MT;
    constexpr int F = kSplitQueries / (16 * MT);
    extern __shared__ uintx4 tiles[];  // [2][keys, values][TB][CH], then [2][key, value scales][TB]
    float* const scales = reinterpret_cast<float*>(tiles + 4 * TB * CH);
    const AttnSplit S{G, TG::M, kSplitTokens};
    // Workgroups go to the 8 XCDs in turn, each with an L2 of its own: an XCD takes neighbouring shares of
    // one head, whose tiles read the same keys and values at about the same time.
    const int per_xcd = gridDim.x / 8, n = blockIdx.x % 8 * per_xcd + blockIdx.x / 8;
    if (n >= shares * C.hkv) return;
    const int head = n / shares, place = n % shares, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const bool negate = c < 0.0f;
    c = fabsf(c);
    __shared__ ShareWalk walks[TG::WAVES];
    ShareWalk& sw = walks[wave];
    CutItem* const cut = cuts + n;
    if (threadIdx.x == 0) cut->pieces = 0;
    if (!sw.open(S, B, C.shift, place, shares)) return;
    while (sw.next(S, B, C.shift)) {
        // (opaque: what follows from the lane is formed anew per piece, not kept in registers for the next)
        int lane = threadIdx.x & 63;
        asm volatile("" : "+v"(lane));
        const int u = lane & 15, w = lane >> 4;
        AttnItem it = sw.item(S);
        // A sequence of few queries, beside a longer one that brought the batch here, has its probabilities in two
        // bf16 parts as in k_paged_split (its error must not grow when a prompt joins its batch): the first F waves
        // hold its queries, the next F, idle otherwise, the same queries with the parts that the first ones'
        // rounding leaves, and the sums are added at the end (33 requests of a row or two in a batch that came
        // here: 100 -> 113 us; both parts in one wave's loop 120 us, and the prompts' loop 5% slower).
        const bool few = it.rows * G <= kSplitQueries, low = few && wave >= F && wave < 2 * F;
        const int m0 = (low ? wave - F : wave) * 16 * MT;
        QueryTile<D, false, MT> qt;
        AttnState<D, Q8, MT, 1> st;
        qt.load(q, qs, it, S, head, m0, negate, lane);
        st.clear(it, S, m0, lane);
        // tokens that all, and any, of the wave's queries see (a wave without queries has nothing to mask)
        const int r0 = tile_row(S, it, m0), rows_left = min(it.rows, (it.tile + 1) * S.rows());
        const int all = r0 >= 0 ? attn_see(it, r0) : 1 << 30;
        const int any = r0 >= 0 ? attn_see(it, min(it.tile * S.rows() + (m0 + 16 * MT - 1) / G, rows_left - 1)) : 0;
        const int from = __builtin_amdgcn_readfirstlane(sw.from) * (kSplitTokens / TB);
        const int stop = min(__builtin_amdgcn_readfirstlane(sw.to) * kSplitTokens, it.see);
        const int to = max(from + 1, (stop + TB - 1) / TB);
        PageWalk walk{B.table + static_cast<int64_t>(sw.seq()) * B.width, C.shift, C.pages, C.hkv, head, max(it.see, 1), it.bad};
        bool special = false;

        // Staging. A wave's piece of a tile lies in 16 tokens of one page: uniform addresses and a lane's
        // own offset. What lies behind the seen tokens is read with them and masked by its reader.
        constexpr int EL = Q8 ? 1 : 2;
        const int ch = lane % CH, wt = wave * 64 / CH;  // the wave's first token of a piece
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
            uintx4 b[MT][1];
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                float p[8];
                st.soften(m, s[m], ks, c, base, masked, lane, p);
                st.weights(m, p, vs, base, lane, b[m], low);
            }
            if constexpr (D == 256) read_values();
            if constexpr (!Q8)
                if (masked) special |= clean_values<D>(v, base, any, lane);
            st.template products<false>(v, b);
        };
        fetch(from * TB);
        stage(0);
        __syncthreads();
        // a wave without queries only stages (33 requests of a row or two in a batch that came here: 133 -> 100 us;
        // ragged prompts of 256 dims, which gain nothing, 325 -> 329)
        if (r0 < 0) {
            for (int step = from; step < to; ++step) {
                fetch(min(step + 1, to - 1) * TB);
                stage(((step - from) & 1) ^ 1);
                lds_barrier();
            }
        } else {
            for (int step = from; step < to; ++step) {
                const int buf = (step - from) & 1;
                fetch(min(step + 1, to - 1) * TB);
                // (waves whose queries see nothing of the tile's end multiply it all the same: a branch around
                // the products made the compiler move every sum once per step)
                const uintx4* kt = tiles + (2 * buf) * TB * CH;
#pragma unroll
                for (int sub = 0; sub < TB / 32; ++sub)
                    half(step * TB + 32 * sub, sub, kt, kt + TB * CH, scales + 2 * buf * TB);
                stage(buf ^ 1);
                lds_barrier();
            }
        }
        const bool bad = __syncthreads_or(it.bad || (it.see > 0 && walk.bad));
        if (few) {
            static_assert(F * MT * (Geo::E + 1) * 64 <= 4 * TB * CH, "the staged tiles' place holds the sums");
            uintx4* const place = tiles + (low ? wave - F : wave) * MT * (Geo::E + 1) * 64 + lane;
            if (low)
#pragma unroll
                for (int m = 0; m < MT; ++m) {
#pragma unroll
                    for (int o = 0; o < Geo::E; ++o)
                        place[(m * (Geo::E + 1) + o) * 64] = __builtin_bit_cast(uintx4, st.o[m][o]);
                    place[(m * (Geo::E + 1) + Geo::E) * 64] = __builtin_bit_cast(uintx4, st.all[m]);
                }
            __syncthreads();
            if (wave < F)
#pragma unroll
                for (int m = 0; m < MT; ++m) {
#pragma unroll
                    for (int o = 0; o < Geo::E; ++o)
                        st.o[m][o] += __builtin_bit_cast(floatx4, place[(m * (Geo::E + 1) + o) * 64]);
                    // (in a Q8 cache the sum is of the probabilities themselves)
                    if constexpr (!Q8) st.all[m] += __builtin_bit_cast(floatx4, place[(m * (Geo::E + 1) + Geo::E) * 64]);
                }
            __syncthreads();
        }
        asm volatile("" ::: "memory");  // (read anew: see ShareWalk)
        it = sw.item(S);
        const bool whole = sw.to - sw.from == it.steps;
        float* pd = nullptr;
        if (!whole) {
            const int slot = attn_slot(sw.start, sw.share, place);
            pd = part + (static_cast<int64_t>(n) * 2 + slot) * (TG::M * (D + 2));
            if (slot && threadIdx.x == 0) note_cut(cut, sw, it);
        }
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            float sum = st.total(m);
            if (bad) sum = kNan;
            const int i = m0 + 16 * m + u, row = low ? -1 : tile_row(S, it, i);
            if (row < 0) continue;
            const float inv = bad || st.lim[m] > 0 ? 1.0f / sum : 0.0f;
            uint16_t* dst = out + (it.first + row) * os + (head * G + i % G) * D;
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int o = 0; o < Geo::E; o += 4) {
                    const int d = Geo::dim(4 * w + r, o);
                    const floatx4 x = {st.o[m][o][r], st.o[m][o + 1][r], st.o[m][o + 2][r], st.o[m][o + 3][r]};
                    if (whole)
                        *reinterpret_cast<uint2*>(dst + d) = make_uint2(pack_bf16(x[0] * inv, x[1] * inv), pack_bf16(x[2] * inv, x[3] * inv));
                    else
                        *reinterpret_cast<floatx4*>(pd + i * D + d) = x;
                }
            if (!whole && w == 0) pd[TG::M * D + i] = st.top[m], pd[TG::M * D + TG::M + i] = sum;
        }
        if constexpr (!Q8)
            if (special && !low) {  // to what the lane has just written
#pragma unroll 1
                for (int n = 0; n < MT * Geo::E; ++n) {
                    const int i = m0 + 16 * (n / Geo::E) + u, row = tile_row(S, it, i);
                    if (row < 0) continue;
                    const int d = Geo::dim(4 * w + n % Geo::E / (Geo::E / 4), 0) + n % (Geo::E / 4) * 4 % Geo::EC +
                                  n % (Geo::E / 4) * 4 / Geo::EC * 16 * Geo::EC;
                    const int t0 = max(special_from(all), from * TB), lim = min(stop, attn_see(it, row));
                    if (whole) {
                        uint2* p = reinterpret_cast<uint2*>(out + (it.first + row) * os + (head * G + i % G) * D + d);
                        const floatx4 x = add_special<D>(C, walk.table, head, t0, lim, d,
                                                         (floatx4){bflo(p->x), bfhi(p->x), bflo(p->y), bfhi(p->y)});
                        *p = make_uint2(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]));
                    } else {
                        floatx4* p = reinterpret_cast<floatx4*>(pd + i * D + d);
                        *p = add_special<D>(C, walk.table, head, t0, lim, d, *p);
                    }
                }
            }
    }
}

// Joins the pieces of the items that the shares' ends cut: a workgroup per (share that an item goes on
// from, kv head, QB of the tile's queries), WQ waves per query, each with every WQ-th run of PB pieces in
// flight. Bound by the latency of its rounds. Prompts cut many queries into few pieces: a wave per query
// (five prompts: 19 us). Long contexts cut few queries into many: four waves per query (three contexts of
// up to 131,072 tokens 6.1 us, a wave per query 12.9; one of 4,001 3.8 us and 6.1).
template <int D, int WQ, int QB, int PB>
__global__ __launch_bounds__(256) void k_paged_join(AttnSplit S, int W, const float* __restrict__ part,
                                                    const CutItem* __restrict__ cuts, uint16_t* __restrict__ out,
                                                    int64_t os) {
    static_assert(WQ == 1 || (WQ == 4 && QB == 1), "waves of a query meet once");
    constexpr int E = D / 64;
    typedef float vec_t __attribute__((ext_vector_type(E)));
    __shared__ vec_t sums[WQ][64];
    __shared__ float2 stats[WQ];
    const int lane = threadIdx.x & 63, head = blockIdx.y, G = S.G, M = S.M;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), place = head * W + blockIdx.x, turn = wave % WQ;
    const CutItem cut = cuts[place];
    const int n = __builtin_amdgcn_readfirstlane(cut.pieces);
    if (n == 0) return;
    AttnItem it;
    it.first = __builtin_amdgcn_readfirstlane(cut.first);
    it.rows = __builtin_amdgcn_readfirstlane(cut.rows);
    it.tokens = __builtin_amdgcn_readfirstlane(cut.tokens);
    it.tile = __builtin_amdgcn_readfirstlane(cut.tile);
    it.bad = __builtin_amdgcn_readfirstlane(cut.bad);
    // (it is the second slot of its first share and the first of the others)
    const float* first = part + (static_cast<int64_t>(place) * 2 + 1) * (M * (D + 2));
    auto piece = [&](int i) { return first + static_cast<int64_t>(2 * i - (i > 0)) * (M * (D + 2)); };
#pragma unroll 2
    for (int j = wave / WQ; j < QB; j += 4 / WQ) {
        const int i = blockIdx.z * QB + j, row = tile_row(S, it, i);
        if (WQ == 1 && row < 0) continue;
        float top = -INFINITY, sum = 0.0f;
        vec_t o = {};
        for (int p0 = turn * PB; p0 < n && row >= 0; p0 += WQ * PB) {
            float t[PB], l[PB], now = top;
            vec_t x[PB];
#pragma unroll
            for (int p = 0; p < PB; ++p) {
                const float* src = piece(min(p0 + p, n - 1));
                t[p] = src[M * D + i];
                l[p] = src[M * D + M + i];
                x[p] = *reinterpret_cast<const vec_t*>(src + i * D + lane * E);
                if (p0 + p >= n) t[p] = -INFINITY;
                now = fmaxf(now, t[p]);
            }
            const float ref = now == -INFINITY ? 0.0f : now, keep = __builtin_amdgcn_exp2f(top - ref);
            top = now;
            sum *= keep;
            o *= keep;
#pragma unroll
            for (int p = 0; p < PB; ++p) {
                // (a repeated piece counts nothing, also where it holds a NaN)
                const float f = p0 + p < n ? __builtin_amdgcn_exp2f(t[p] - ref) : 0.0f;
                sum = p0 + p < n ? fmaf(l[p], f, sum) : sum;
                o = p0 + p < n ? o + x[p] * f : o;
            }
        }
        if constexpr (WQ > 1) {
            sums[wave][lane] = o;
            if (lane == 0) stats[wave] = make_float2(top, sum);
            __syncthreads();
            if (turn || row < 0) return;
#pragma unroll
            for (int k = 1; k < WQ; ++k) top = fmaxf(top, stats[k].x);
            const float ref = top == -INFINITY ? 0.0f : top;
            sum = 0.0f;
            o = vec_t{};
#pragma unroll
            for (int k = 0; k < WQ; ++k) {
                const float f = __builtin_amdgcn_exp2f(stats[k].x - ref);
                sum = fmaf(stats[k].y, f, sum);
                o += sums[k][lane] * f;
            }
        }
        const float inv = it.bad || attn_see(it, row) > 0 ? 1.0f / sum : 0.0f;
        uint16_t* dst = out + (it.first + row) * os + (head * G + i % G) * D + lane * E;
#pragma unroll
        for (int e = 0; e < E; ++e) dst[e] = f2bf(o[e] * inv);
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
// kernel does so once per 128 or 256.
struct AttnPlan {
    bool tiles, joined;
    int mt;  // split: 16-query groups
    int M;   // queries per tile
    int W;   // shares per kv head
};
AttnPlan attn_plan(const PagedCacheDev& C, const PagedBatchDev& B, int max_rows, int hq) {
    AttnPlan p{};
    const int G = hq / C.hkv;
    const int64_t queries = static_cast<int64_t>(max_rows) * G;
    p.tiles = queries > kSplitQueries;
    p.mt = queries <= 16 ? 1 : 2;
    p.M = !p.tiles ? 16 * p.mt : C.d == 256 ? TileGeo<256>::M : TileGeo<128>::M;
    p.W = std::max(1, 256 * (p.tiles || C.d == 256 ? 1 : 2) / C.hkv);  // the chip's 256 CUs at the kernels' occupancy
    // (no sequence is longer than a step, or a share holds its head's whole list: nothing is cut inside an item)
    p.joined = p.W > 1 && (static_cast<int64_t>(B.width) << C.shift) > kSplitTokens;
    return p;
}

template <int D, bool Q8, int MT>
hipError_t launch_split(const PagedCacheDev& C, const PagedBatchDev& B, const AttnPlan& p, const uint16_t* q, int64_t qs,
                        int hq, float c, uint16_t* out, int64_t os, float* part, CutItem* cuts, hipStream_t st) {
    constexpr size_t lds = (static_cast<size_t>(kSplitWaves) * 16 * MT * (D + 4) + 2 * kSplitWaves * 16 * MT) * 4;
    const hipError_t e = ensure_lds<k_paged_split<D, Q8, MT>>(lds);
    if (e != hipSuccess) return e;
    return launch(k_paged_split<D, Q8, MT>, dim3(p.W, C.hkv), dim3(256), lds, st, C, B, hq / C.hkv, q, qs, c, out, os, part,
                  cuts);
}
template <int D, bool Q8>
hipError_t launch_attention(const PagedCacheDev& C, const PagedBatchDev& B, const AttnPlan& p, const uint16_t* q, int64_t qs,
                            int hq, float scale, uint16_t* out, int64_t os, void* ws, hipStream_t st) {
    const float c = scale * 1.44269504088896341f;  // exponents of 2
    CutItem* const cuts = static_cast<CutItem*>(ws);
    float* const part = reinterpret_cast<float*>(cuts + static_cast<size_t>(C.hkv) * p.W);
    hipError_t e;
    if (!p.tiles) {
        e = p.mt == 1 ? launch_split<D, Q8, 1>(C, B, p, q, qs, hq, c, out, os, part, cuts, st)
                      : launch_split<D, Q8, 2>(C, B, p, q, qs, hq, c, out, os, part, cuts, st);
    } else {
        e = ensure_lds<k_paged_tile<D, Q8>>(TileGeo<D>::kLds);
        if (e == hipSuccess)
            e = launch(k_paged_tile<D, Q8>, dim3((p.W * C.hkv + 7) / 8 * 8), dim3(64 * TileGeo<D>::WAVES), TileGeo<D>::kLds,
                       st, C, B, hq / C.hkv, p.W, q, qs, c, out, os, part, cuts);
    }
    if (e != hipSuccess || !p.joined) return e;
    const AttnSplit S{hq / C.hkv, p.M, kSplitTokens};
    if (p.tiles)
        return launch(k_paged_join<D, 1, 32, 2>, dim3(p.W - 1, C.hkv, p.M / 32), dim3(256), 0, st, S, p.W, part, cuts, out, os);
    return launch(k_paged_join<D, 4, 1, 8>, dim3(p.W - 1, C.hkv, p.M), dim3(256), 0, st, S, p.W, part, cuts, out, os);
}

} // namespace

size_t paged_attention_ws(const PagedCacheDev& C, const PagedBatchDev& B, int max_rows, int hq) {
    const AttnPlan p = attn_plan(C, B, max_rows, hq);
    const size_t shares = static_cast<size_t>(C.hkv) * p.W;
    return shares * sizeof(CutItem) + (p.joined ? shares * 2 * p.M * (C.d + 2) * 4 : 0);
}

hipError_t launch_paged_attention(const PagedCacheDev& C, bool q8, const PagedBatchDev& B, int max_rows, const uint16_t* q,
                                  int64_t qs, int hq, float scale, uint16_t* out, int64_t os, void* ws, hipStream_t st) {
    const AttnPlan p = attn_plan(C, B, max_rows, hq);
    auto go = [&](auto kern) { return kern(C, B, p, q, qs, hq, scale, out, os, ws, st); };
    if (q8)
        return C.d == 64    ? go(launch_attention<64, true>)
               : C.d == 128 ? go(launch_attention<128, true>)
                            : go(launch_attention<256, true>);
    return C.d == 64    ? go(launch_attention<64, false>)
           : C.d == 128 ? go(launch_attention<128, false>)
                        : go(launch_attention<256, false>);
}

} // namespace q38
