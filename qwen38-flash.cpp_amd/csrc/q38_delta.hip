// q38_delta.hip — the gated delta rule of many requests over a pool of float states:
//   S <- exp(g) S,  S <- S + beta (v - S k) k^T,  o = scale * S q      per row and value head.
//
//   k_delta_rows     short sequences and checkpoints: row by row, the state in registers
//   k_delta_system   long sequences, in chunks of 32 rows: every chunk's triangular system and scores
//   k_delta_chunks   the walk over a sequence's chunks, the state in registers
#include "q38_device.hpp"
#include "q38_paged.hpp"
#include "q38_internal.hpp"

namespace q38 {

namespace {

__device__ __forceinline__ float sum8(float v) {  // over 8 neighbouring lanes, the same in all of them
    v += xor_lane_f<1>(v);
    v += xor_lane_f<2>(v);
    v += xor_lane_f<4>(v);
    return v;
}

// A value that is the same for the whole wave, through the scalar cache: its wait is not one for the
// vector loads in flight.
template <typename T>
__device__ __forceinline__ T uniform_load(const T* p) {
    typedef const __attribute__((address_space(4))) T scalar_t;
    return *((scalar_t*)(reinterpret_cast<uintptr_t>(p)));
}

// A wave takes 8 R value rows of one head of one sequence: 8 lanes per value row, lane `sub` of them
// key dims 32 c + 4 sub .. + 3 (16-byte state accesses, 128 bytes together per row). Single tokens are
// bound by the states' bytes: 104 us for 128 requests of 32 heads [128][128], 5.2 TB/s, a copy's rate,
// and 4.8 us for one request. Longer sequences are a chain of two sums over lanes per row; the next row's
// operands are in flight during a row.
template <int DK, int R>
__device__ __forceinline__ void walk_rows(const DeltaDev& D, const DeltaBatchDev& B, int s, int h, int dv0) {
    constexpr int C = DK / 32;
    const int lane = threadIdx.x & 63, sub = lane & 7;
    const int dv = dv0 + (lane >> 3);  // the lane's first value row, the next 8 on
    const int hk = h / (D.hv / D.hk);
    const int first = uniform_load(B.off + s), behind = uniform_load(B.off + s + 1);
    const int from = B.origin ? uniform_load(B.origin + s) : -1, last = B.last ? uniform_load(B.last + s) : -1;
    const int begin = max(first, 0), end = min(behind, B.rows);
    const size_t elems = static_cast<size_t>(D.hv) * D.dv * DK;
    const size_t lane_at = (static_cast<size_t>(h) * D.dv + dv) * DK + 4 * sub;
    float4 st[R][C];
    const float fill = from >= B.slots ? __builtin_nanf("") : 0.0f;
    if (from >= 0 && from < B.slots) {
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int c = 0; c < C; ++c)
                st[i][c] = *reinterpret_cast<const float4*>(B.states + from * elems + lane_at + i * 8 * DK + 32 * c);
    } else {
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int c = 0; c < C; ++c) st[i][c] = make_float4(fill, fill, fill, fill);
    }
    auto store = [&](int slot) {
        if (slot < 0 || slot >= B.slots) return;
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int c = 0; c < C; ++c)
                *reinterpret_cast<float4*>(B.states + slot * elems + lane_at + i * 8 * DK + 32 * c) = st[i][c];
    };
    struct RowIn {
        uint2 k[C], q[C];
        uint16_t v[R];
        float g, b;
    };
    auto load = [&](int r, RowIn& x) {
        r = min(r, end - 1);
#pragma unroll
        for (int c = 0; c < C; ++c) {
            x.k[c] = *reinterpret_cast<const uint2*>(D.k + r * D.ks + hk * DK + 32 * c + 4 * sub);
            x.q[c] = *reinterpret_cast<const uint2*>(D.q + r * D.qs + hk * DK + 32 * c + 4 * sub);
        }
#pragma unroll
        for (int i = 0; i < R; ++i) x.v[i] = D.v[r * D.vs + h * D.dv + dv + 8 * i];
        x.g = uniform_load(D.g + static_cast<size_t>(r) * D.hv + h);
        x.b = uniform_load(D.beta + static_cast<size_t>(r) * D.hv + h);
    };
    auto row = [&](int r, const RowIn& x) {
        const float decay = expf(x.g);
        float hit[R] = {}, o[R] = {};
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int c = 0; c < C; ++c) {
                float4& t = st[i][c];
                t.x *= decay, t.y *= decay, t.z *= decay, t.w *= decay;
                hit[i] = fmaf(t.x, bflo(x.k[c].x), hit[i]);
                hit[i] = fmaf(t.y, bfhi(x.k[c].x), hit[i]);
                hit[i] = fmaf(t.z, bflo(x.k[c].y), hit[i]);
                hit[i] = fmaf(t.w, bfhi(x.k[c].y), hit[i]);
            }
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const float u = x.b * (bf2f(x.v[i]) - sum8(hit[i]));
#pragma unroll
            for (int c = 0; c < C; ++c) {
                float4& t = st[i][c];
                t.x = fmaf(u, bflo(x.k[c].x), t.x);
                t.y = fmaf(u, bfhi(x.k[c].x), t.y);
                t.z = fmaf(u, bflo(x.k[c].y), t.z);
                t.w = fmaf(u, bfhi(x.k[c].y), t.w);
                o[i] = fmaf(t.x, bflo(x.q[c].x), o[i]);
                o[i] = fmaf(t.y, bfhi(x.q[c].x), o[i]);
                o[i] = fmaf(t.z, bflo(x.q[c].y), o[i]);
                o[i] = fmaf(t.w, bfhi(x.q[c].y), o[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < R; ++i) {
            o[i] = sum8(o[i]);
            if (sub == 0) D.out[(static_cast<size_t>(r) * D.hv + h) * D.dv + dv + 8 * i] = f2bf(o[i] * D.scale);
        }
        if (B.ckpt) store(uniform_load(B.ckpt + r));
    };
    if (begin < end) {
        RowIn a, b;
        load(begin, a);
        for (int r = begin; r < end; r += 2) {
            load(r + 1, b);
            row(r, a);
            if (r + 1 >= end) break;
            load(r + 2, a);
            row(r + 1, b);
        }
    }
    store(last);
}

template <int DK, int R>
__global__ __launch_bounds__(256) void k_delta_rows(DeltaDev D, DeltaBatchDev B) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    walk_rows<DK, R>(D, B, blockIdx.z, blockIdx.y, (blockIdx.x * 4 + wave) * 8 * R);
}

// ---- the chunked form. Within a chunk of C rows, with G_i the sums of its log decays up to row i,
// A_ij = beta_i (k_i . k_j) exp(G_i - G_j) for j < i and T = (I + A)^-1, the rows' updates
// u_i = beta_i (v_i - S k_i) solve a triangular system:
//   U   = T diag(beta) Y,  Y_i = v_i - exp(G_i) S k_i           (S: the state before the chunk)
//   o_i = exp(G_i) S q_i + sum_{j <= i} (q_i . k_j) exp(G_i - G_j) U_j
//   S  <- exp(G_C) S + sum_j exp(G_C - G_j) U_j k_j^T
// k_delta_system forms T diag(beta), the scores and the decays of every chunk at once;
// k_delta_chunks walks a sequence's chunks with the state in registers.
//
// The products run on the bf16 matrix cores. q, k and v are bf16 already: k . k and q . k are exact
// products with float sums. Float operands are split into bf16 parts, x = hi + mid + lo: three parts
// (24 bits) of all that the state is made of, T, Y, U and the state itself in S k, whose error Y takes into U
// and so back into the state, multiplied part by part (for two split operands the six products down to
// 2^-24); two (16 bits) of what only the outputs, rounded to bf16, are made of: the state in S q, the scores
// and U beside them. The states are as far from 64 bits as those of float rows: of 128 rows without decay
// 1.5e-7 of their norm (float rows 2.3e-7; the state in two parts 9e-7, U in two 5e-6). The third part of the
// state costs about 4% of a prompt's time (4,001 rows 188 -> 196 us in a pass).
constexpr int kChunk = 32;
constexpr double kFloor = -1e4;  // exp() of it is 0; log decays below (-inf) are taken as this

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float floatx2 __attribute__((ext_vector_type(2)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef uint32_t uintx4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((floatx2){lo, hi}, bf16x2));
}
__device__ __forceinline__ floatx4 mfma(uintx4 a, uintx4 b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
// Eight floats as an operand, in P parts.
template <int P>
struct Parts {
    uintx4 p[P];
    __device__ __forceinline__ void split(const float (&x)[8]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float a = x[2 * i], b = x[2 * i + 1];
#pragma unroll
            for (int n = 0; n < P; ++n) {
                const uint32_t w = pack_bf16(a, b);
                p[n][i] = w;
                if (n + 1 < P) a -= bflo(w), b -= bfhi(w);
            }
        }
    }
};

// What k_delta_system leaves of a (chunk, value head): T diag(beta) in three parts and the scores,
// both as operands (16 bytes per lane, two row tiles), then exp(G_i) and exp(G_C - G_i).
struct alignas(16) ChunkSystem {
    uintx4 t[3][2][64];
    uintx4 m[2][2][64];
    float into[kChunk], left[kChunk];
};

// Row of tile a's operand row (or result row) u: a lane's result rows 4 w + r of both tiles are the
// chunk's rows 8 w .. 8 w + 7, the k index that the next product wants of it.
__device__ __forceinline__ int chunk_row(int u, int a) { return 8 * (u >> 2) + 4 * a + (u & 3); }

// The chunk of the whole batch's list, and its sequence's first row and rows from the chunk's on.
__device__ __forceinline__ bool find_chunk(const DeltaBatchDev& B, int want, int* row, int* rows) {
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int s0 = 0; s0 < B.seqs; s0 += 64) {
        RowSpan span{0, 0};
        if (s0 + lane < B.seqs) span = row_span(B.off, s0 + lane, B.rows);
        const int n = (span.end - span.begin + kChunk - 1) / kChunk;
        int upto = n;
        for (int d = 1; d < 64; d <<= 1) {
            const int x = __shfl_up(upto, d);
            if (lane >= d) upto += x;
        }
        const uint64_t past = __ballot(before + upto > want);
        if (past) {
            const int l = __builtin_ctzll(past), at = want - before - __shfl(upto, l) + __shfl(n, l);
            *row = __shfl(span.begin, l) + at * kChunk;
            *rows = min(kChunk, __shfl(span.end, l) - *row);
            return true;
        }
        before += __shfl(upto, 63);
    }
    return false;
}
// The sequence that the slot-th group of workgroups takes. A walk is one chain per head, so the longest
// sequences begin first (eight ragged prompts of 32 heads in their own order 368 us, so 348); where all
// groups are on the chip at once, two workgroups per CU, those of the second half join the first half's in
// the opposite order, the shortest beside the longest (eight of 16 heads in their own order 168 us, longest
// first 158, so 156). Up to 64 sequences; more fill the chip in any order.
__device__ __forceinline__ int nth_sequence(const DeltaBatchDev& B, int slot, int groups_per_round) {
    if (B.seqs > 64 || B.seqs == 1) return slot;
    const int lane = threadIdx.x & 63;
    int length = -1;
    if (lane < B.seqs) {
        const RowSpan span = row_span(B.off, lane, B.rows);
        length = span.end - span.begin;
    }
    int rank = 0;
    for (int s = 0; s < B.seqs; ++s) {
        const int other = __builtin_amdgcn_readlane(length, s);
        rank += other > length || (other == length && s < lane);
    }
    if (B.seqs <= 2 * groups_per_round && slot >= groups_per_round) slot = B.seqs - 1 - (slot - groups_per_round);
    return __builtin_ctzll(__ballot(lane < B.seqs && rank == slot));
}
// The sequence's first chunk in the list.
__device__ __forceinline__ int first_chunk(const DeltaBatchDev& B, int seq) {
    int n = 0;
    for (int s = threadIdx.x & 63; s < seq; s += 64) {
        const RowSpan span = row_span(B.off, s, B.rows);
        n += (span.end - span.begin + kChunk - 1) / kChunk;
    }
    for (int d = 32; d >= 1; d >>= 1) n += __shfl_xor(n, d);
    return n;
}

// One wave per chunk and value head, or two value heads of one key head (N = 2): their products are the
// same, and the substitution of one head's diagonal blocks fills half a wave (eight ragged prompts, 16,320
// systems: 86 us with one, 75 with two). Bound by bytes where there are many chunks: those systems are 171 MB
// behind 133 MB of queries and keys, 4.1 TB/s (half the LDS, for twice the waves, changed nothing).
template <int DK, int N>
__global__ __launch_bounds__(64) void k_delta_system(DeltaDev D, DeltaBatchDev B, ChunkSystem* __restrict__ sys) {
    constexpr int KS = DK / 32, LD = kChunk + 4;
    __shared__ __align__(16) float As[N][kChunk][LD];  // A, then T in its place, then the scores
    __shared__ double Gs[N][kChunk];
    __shared__ float Bs[N][kChunk];
    const int h0 = blockIdx.y * N, lane = threadIdx.x, u = lane & 15, w = lane >> 4, hk = h0 / (D.hv / D.hk);
    int r0 = 0, n = 0;
    if (!find_chunk(B, blockIdx.x, &r0, &n)) return;
    // the decay sums, in double: differences of far sums must keep a weak decay's digits (lanes 32 e .. of head e)
    {
        const int e = N == 2 ? lane >> 5 : 0, i = lane & 31;
        const bool mine = i < n;
        const size_t at = static_cast<size_t>(r0 + i) * D.hv + h0 + e;
        const float g = mine ? D.g[at] : 0.0f;
        double G = g < kFloor ? kFloor : g;
        for (int d = 1; d < kChunk; d <<= 1) {
            const double x = __shfl_up(G, d, 32);
            if (i >= d) G += x;
        }
        if (N == 2 || lane < kChunk) {
            Gs[e][i] = G;
            Bs[e][i] = mine ? D.beta[at] : 0.0f;
        }
    }
    // operands: row 16 t + u, dims 32 s + 8 w ..; rows behind the sequence are zeros
    uintx4 kop[2][KS], qop[2][KS];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const int r = 16 * t + u;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            kop[t][s] = qop[t][s] = (uintx4){0, 0, 0, 0};
            if (r < n) {
                kop[t][s] = *reinterpret_cast<const uintx4*>(D.k + (r0 + r) * D.ks + hk * DK + 32 * s + 8 * w);
                qop[t][s] = *reinterpret_cast<const uintx4*>(D.q + (r0 + r) * D.qs + hk * DK + 32 * s + 8 * w);
            }
        }
    }
    __syncthreads();
    floatx4 qk[N][2][2];
#pragma unroll
    for (int ti = 0; ti < 2; ++ti)
#pragma unroll
        for (int tj = 0; tj <= ti; ++tj) {
            floatx4 kk = {0.0f, 0.0f, 0.0f, 0.0f}, qq = kk;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                kk = mfma(kop[ti][s], kop[tj][s], kk);
                qq = mfma(qop[ti][s], kop[tj][s], qq);
            }
#pragma unroll
            for (int e = 0; e < N; ++e)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int i = 16 * ti + 4 * w + r, j = 16 * tj + u;
                    const float d = j <= i ? expf(static_cast<float>(Gs[e][i] - Gs[e][j])) : 0.0f;
                    As[e][i][j] = j < i ? Bs[e][i] * kk[r] * d : 0.0f;
                    qk[e][ti][tj][r] = j <= i ? qq[r] * d : 0.0f;
                }
        }
    __syncthreads();
    // the two diagonal blocks' inverses, a column per lane, by substitution
    {
        const int b = 16 * (w & 1), e = N == 2 ? w >> 1 : 0;
        float t[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            float x = 0.0f;
#pragma unroll
            for (int j = 0; j < 16; j += 4) {
                if (j >= i) break;
                const floatx4 a = *reinterpret_cast<const floatx4*>(&As[e][b + i][b + j]);
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (j + c < i) x = fmaf(a[c], t[j + c], x);
            }
            t[i] = i == u ? 1.0f : -x;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            As[e][b + i][b + u] = t[i];
        }
    }
    __syncthreads();
    // the block below them: -T22 (A21 T11), float products (A21 T11 stands above for a while)
    floatx4 x[N];
#pragma unroll
    for (int e = 0; e < N; ++e) {
        x[e] = (floatx4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < 16; k += 4)
            x[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(As[e][16 + u][k + w], As[e][k + w][u], x[e], 0, 0, 0);
#pragma unroll
        for (int r = 0; r < 4; ++r) As[e][4 * w + r][16 + u] = x[e][r];
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < N; ++e) {
        x[e] = (floatx4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < 16; k += 4)
            x[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(As[e][16 + u][16 + k + w], As[e][k + w][16 + u], x[e], 0, 0, 0);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            As[e][16 + 4 * w + r][u] = -x[e][r];
            As[e][4 * w + r][16 + u] = 0.0f;
        }
    }
    __syncthreads();
    ChunkSystem* const out0 = sys + static_cast<size_t>(blockIdx.x) * D.hv + h0;
#pragma unroll
    for (int e = 0; e < N; ++e)
#pragma unroll
        for (int a = 0; a < 2; ++a) {
            float row[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) row[j] = As[e][chunk_row(u, a)][8 * w + j] * Bs[e][8 * w + j];
            Parts<3> t;
            t.split(row);
#pragma unroll
            for (int p = 0; p < 3; ++p) out0[e].t[p][a][lane] = t.p[p];
        }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < N; ++e)
#pragma unroll
        for (int ti = 0; ti < 2; ++ti)
#pragma unroll
            for (int tj = 0; tj < 2; ++tj)
#pragma unroll
                for (int r = 0; r < 4; ++r) As[e][16 * ti + 4 * w + r][16 * tj + u] = tj <= ti ? qk[e][ti][tj][r] : 0.0f;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < N; ++e) {
        ChunkSystem& out = out0[e];
#pragma unroll
        for (int a = 0; a < 2; ++a) {
            float row[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) row[j] = As[e][16 * a + u][8 * w + j];
            Parts<2> m;
            m.split(row);
#pragma unroll
            for (int p = 0; p < 2; ++p) out.m[p][a][lane] = m.p[p];
        }
        if (lane < kChunk) {
            out.into[lane] = expf(static_cast<float>(Gs[e][lane]));
            out.left[lane] = expf(static_cast<float>(Gs[e][kChunk - 1] - Gs[e][lane]));
        }
    }
}

// The walk. A state wave holds 16 value columns of a head's state, transposed: S^T tile o (o < E =
// DK / 16) has key dim E (4 w + r) + o in its result row 4 w + r and the value dim in its column. Lane
// (u, w) thus holds key dims 4 E w .. 4 E (w + 1) - 1 of value dim u, eight of them in a row being an
// operand of S k and S q with keys and queries read as stored: no value moves between lanes. A sequence is
// one chain of chunks per head, and a wave issues an instruction every four cycles at best, so what the chain
// does not need is left to a second wave on another SIMD: two state waves (32 value columns) go with two output
// waves, of 16 rows of the chunk each, which take the operands of S and U through LDS a chunk later, load the
// keys and values and stage them as the state waves want them (the keys as stored and, pairs of rows
// interleaved, as operands of K^T). A prompt of 4,001 rows: 170 us, 1.35 us a chunk, bound by the state wave's
// own 500 instructions (161 us with two parts of the state; one wave doing all, before, took 80 us more). Eight
// ragged prompts, 16,192 rows, two workgroups per CU: 339 us with their systems, bound by the vector memory
// path, which takes a cycle per row that neighbouring lanes do not share (output waves by columns, each with
// all queries, scores and short stores of its own, took 8% longer).
template <int DK>
struct WalkGeo {
    static constexpr int E = DK / 16, KS = DK / 32, CH = DK / 8;
    static constexpr int NW = 2;                              // state waves of a workgroup, and output waves
    static constexpr int PC = kChunk * CH / (64 * NW);        // an output thread's rows of the keys, 16 bytes of each
    static constexpr int kKeys = kChunk * CH, kParts = NW * KS * 2 * 64, kUpd = NW * 2 * 64;
    static constexpr size_t kLds = 2 * 16 * static_cast<size_t>(2 * kKeys + kParts + 2 * kUpd);  // (128 dims: half a CU's)
};

template <int DK>
__global__ __launch_bounds__(128 * WalkGeo<DK>::NW, 2) void k_delta_chunks(DeltaDev D, DeltaBatchDev B,
                                                                           const ChunkSystem* __restrict__ sys, int bound) {
    using Geo = WalkGeo<DK>;
    constexpr int E = Geo::E, KS = Geo::KS, CH = Geo::CH, NW = Geo::NW, PC = Geo::PC, KB = KS < 4 ? KS : 4;
    extern __shared__ uintx4 walk_lds[];  // [2] of: keys, K^T's operands, the state's parts, U, V
    uintx4* const keys_lds = walk_lds;
    uintx4* const turned_lds = walk_lds + 2 * Geo::kKeys;
    uintx4* const parts_lds = walk_lds + 4 * Geo::kKeys;
    floatx4* const upd_lds = reinterpret_cast<floatx4*>(walk_lds + 2 * (2 * Geo::kKeys + Geo::kParts));
    floatx4* const val_lds = upd_lds + 2 * Geo::kUpd;
    const int lane = threadIdx.x & 63, u = lane & 15, w = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int part = wave % NW;  // a state wave's 16 columns, an output wave's 16 rows of the chunk
    const bool outputs = wave >= NW;
    // Workgroups go to the 8 XCDs in turn, each with an L2 of its own: those of one head, which read the
    // same chunk systems, keys and queries, are one XCD's (spread over the XCDs eight ragged prompts take
    // 393 us in place of 348).
    const int groups = D.dv / (16 * NW), turn = blockIdx.x / 8, chain = turn / groups * 8 + blockIdx.x % 8;
    if (chain >= D.hv * B.seqs) return;
    const int h = chain % D.hv, hk = h / (D.hv / D.hk);
    const int s = nth_sequence(B, chain / D.hv, max(1, 256 / (groups * D.hv)));
    const int dv = turn % groups * NW * 16;  // the workgroup's first value dim
    const RowSpan span = row_span(B.off, s, B.rows);
    const int length = __builtin_amdgcn_readfirstlane(span.end - span.begin), begin = __builtin_amdgcn_readfirstlane(span.begin);
    const int c0 = __builtin_amdgcn_readfirstlane(first_chunk(B, s));
    // (offsets that do not ascend could name more chunks than the workspace holds)
    const int chunks = max(0, min((length + kChunk - 1) / kChunk, bound - c0));
    const ChunkSystem* const sys0 = sys + static_cast<size_t>(c0) * D.hv + h;
    auto system = [&](int n) -> const ChunkSystem& { return sys0[static_cast<size_t>(min(n, chunks - 1)) * D.hv]; };
    // keys: swizzled for reads down chunk_row()'s rows
    auto key_at = [](int row, int ch) { return row * CH + (ch ^ ((row & 3) | ((row >> 1) & 4))); };
    // V and U: rows 8 w + 4 a .. of column u in a slot of their own, so that the writes of V, down the columns,
    // get banks of their own
    auto slot = [](int columns, int column, int block, int a) {
        return 128 * columns + 64 * a + 16 * block + (column ^ (2 * block + a) ^ (4 * columns));
    };
    // Loads of a next chunk are made always, of the last one's again behind it, and their number is the same
    // on every path, so that a wait counts only the loads that it needs. Rows behind the sequence: its last
    // row again, whose update is nothing (its beta in the system is 0).

    // A row's products with the matrices' zeros do not hide an infinity or NaN of a later row of its chunk: U, and
    // with it the outputs, would be NaN from the chunk's first row on, where the rule is causal. Such a U is in the
    // state for good, so the state tells at the end: the workgroup then runs its part of the sequence again from
    // the origin, which nothing has overwritten, row by row (in a healthy model never; 4,001 rows 2.4 ms).
    int* const flags = reinterpret_cast<int*>(upd_lds + (chunks & 1) * Geo::kUpd);  // (not in use at the end)
    auto again = [&] {
        if (chunks == 0) return false;
        int any = 0;
#pragma unroll
        for (int i = 0; i < NW; ++i) any |= flags[i];
        if (__builtin_amdgcn_readfirstlane(any) == 0) return false;
        __threadfence();  // (the outputs so far are behind those that replace them)
        __syncthreads();
        walk_rows<DK, 1>(D, B, s, h, dv + 8 * wave);
        return true;
    };

    if (outputs) {
        const char* const kb = reinterpret_cast<const char*>(D.k + begin * D.ks + hk * DK);
        const char* const vb = reinterpret_cast<const char*>(D.v + begin * D.vs + h * D.dv + dv);
        const char* const qb = reinterpret_cast<const char*>(D.q + begin * D.qs + hk * DK);
        char* const ob = reinterpret_cast<char*>(D.out + (static_cast<size_t>(begin) * D.hv + h) * D.dv + dv);
        const int tid = part * 64 + lane;
        uintx4 kr[PC], vr, qr[KS], mop[2];
        float eg;
        auto fetch_keys = [&](int chunk) {
#pragma unroll
            for (int i = 0; i < PC; ++i) {
                const int64_t row = min(chunk * kChunk + tid / CH * PC + i, length - 1);
                kr[i] = *reinterpret_cast<const uintx4*>(kb + 2 * row * D.ks + 16 * (tid % CH));
            }
            const int64_t row = min(chunk * kChunk + 16 * part + lane / 4, length - 1);
            vr = *reinterpret_cast<const uintx4*>(vb + 2 * (row * D.vs + 8 * (lane & 3)));
        };
        auto stage_keys = [&](int buf) {
            const int r0 = tid / CH * PC;
#pragma unroll
            for (int i = 0; i < PC; ++i) keys_lds[buf * Geo::kKeys + key_at(r0 + i, tid % CH)] = kr[i];
            // operand o of K^T: dim E u + o of rows 8 w ..
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int d = 8 * (tid % CH) + e;
                typedef uint32_t pairs_t __attribute__((ext_vector_type(PC / 2)));
                uint32_t x[PC / 2];
#pragma unroll
                for (int j = 0; j < PC / 2; ++j)
                    x[j] = __builtin_amdgcn_perm(kr[2 * j + 1][e >> 1], kr[2 * j][e >> 1], e & 1 ? 0x07060302u : 0x05040100u);
                uintx4* const at = turned_lds + buf * Geo::kKeys + d % E * 64 + r0 / 8 * 16 + d / E;
                uint32_t* const to = reinterpret_cast<uint32_t*>(at) + r0 % 8 / 2;
                if constexpr (PC == 2) {
                    *to = x[0];
                } else {
                    pairs_t all;
#pragma unroll
                    for (int j = 0; j < PC / 2; ++j) all[j] = x[j];
                    *reinterpret_cast<pairs_t*>(to) = all;
                }
            }
            const int row = 16 * part + lane / 4;
            float* to = reinterpret_cast<float*>(val_lds + buf * Geo::kUpd) + (row & 3);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                to[4 * slot(lane >> 1 & 1, 8 * (lane & 1) + i, row >> 3, row >> 2 & 1)] =
                    i & 1 ? bfhi(vr[i >> 1]) : bflo(vr[i >> 1]);
        };
        auto fetch_queries = [&](int chunk) {  // operands: row u of the wave's, dims 4 E w + 8 k ..
            const int64_t row = min(chunk * kChunk + 16 * part + u, length - 1);
#pragma unroll
            for (int k = 0; k < KS; ++k) qr[k] = *reinterpret_cast<const uintx4*>(qb + 2 * row * D.qs + 16 * (KS * w + k));
        };
        auto fetch_scores = [&](const ChunkSystem& cs) {
#pragma unroll
            for (int p = 0; p < 2; ++p) mop[p] = cs.m[p][part][lane];
            eg = cs.into[16 * part + u];
        };
        if (chunks > 0) {
            fetch_keys(0);
            fetch_queries(0);
            fetch_scores(system(0));
            stage_keys(0);
        }
        lds_barrier();
        for (int n = 0; n <= chunks && chunks > 0; ++n) {  // the keys of chunk n + 1, the outputs of chunk n - 1
            fetch_keys(min(n + 1, chunks - 1));
            if (n > 0) {
                const uintx4* parts = parts_lds + ((n - 1) & 1) * Geo::kParts + lane;
                const floatx4* upd = upd_lds + ((n - 1) & 1) * Geo::kUpd;
                // O^T = exp(G) S q + U^T M^T, transposed: value dims by the wave's rows
                floatx4 ot[NW];
#pragma unroll
                for (int c = 0; c < NW; ++c) ot[c] = (floatx4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int k = 0; k < KS; ++k)
#pragma unroll
                    for (int p = 1; p >= 0; --p)
#pragma unroll
                        for (int c = 0; c < NW; ++c) ot[c] = mfma(parts[((c * KS + k) * 2 + p) * 64], qr[k], ot[c]);
                Parts<2> up[NW];
#pragma unroll
                for (int c = 0; c < NW; ++c) {
                    const floatx4 un[2] = {upd[slot(c, u, w, 0)], upd[slot(c, u, w, 1)]};
                    float x[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) x[j] = un[j >> 2][j & 3];
                    up[c].split(x);
                }
#pragma unroll
                for (int c = 0; c < NW; ++c) ot[c] = mfma(up[c].p[0], mop[1], ot[c] * eg);
#pragma unroll
                for (int p = 1; p >= 0; --p)
#pragma unroll
                    for (int c = 0; c < NW; ++c) ot[c] = mfma(up[c].p[p], mop[0], ot[c]);
                fetch_queries(n);
                fetch_scores(system(n));
                // lane L stores 16 bytes of row L / 4: what lanes (L / 4, 2 (L % 2)) and the next w have of its columns
                uint32_t x[4];
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int d = 0; d < 2; ++d) {
                        const int from = 4 * (lane / 4 + 16 * (2 * (lane & 1) + i));
                        uint32_t y[NW];
#pragma unroll
                        for (int c = 0; c < NW; ++c)
                            y[c] = __builtin_amdgcn_ds_bpermute(
                                from, pack_bf16(ot[c][2 * d] * D.scale, ot[c][2 * d + 1] * D.scale));
                        x[2 * i + d] = lane & 2 ? y[1] : y[0];
                    }
                const int row = (n - 1) * kChunk + 16 * part + lane / 4;
                if (row < length)
                    *reinterpret_cast<uintx4*>(ob + 2 * (static_cast<int64_t>(row) * D.hv * D.dv + 8 * (lane & 3))) =
                        (uintx4){x[0], x[1], x[2], x[3]};
            }
            stage_keys((n + 1) & 1);
            lds_barrier();  // (the next chunk's loads stay in flight)
        }
        again();
        return;
    }

    const size_t elems = static_cast<size_t>(D.hv) * D.dv * DK;
    const int from = B.origin ? uniform_load(B.origin + s) : -1;
    floatx4 st[E];
    auto state_at = [&](int slot, int r) {  // E consecutive key dims
        return B.states + slot * elems + (static_cast<size_t>(h) * D.dv + dv + 16 * part + u) * DK + E * (4 * w + r);
    };
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int o = 0; o < E; o += 4) {
            floatx4 x = {0.0f, 0.0f, 0.0f, 0.0f};
            if (from >= B.slots) x = x + __builtin_nanf("");
            else if (from >= 0) x = *reinterpret_cast<const floatx4*>(state_at(from, r) + o);
#pragma unroll
            for (int e = 0; e < 4; ++e) st[o + e][r] = x[e];
        }
    // a chunk's system in registers, every part loaded anew as soon as its chunk is done with it
    uintx4 top[3][2];
    floatx4 into[2], left[2];
    float whole = 1.0f;
    auto load_t = [&](const ChunkSystem& cs) {
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
            for (int p = 0; p < 3; ++p) top[p][a] = cs.t[p][a][lane];
    };
    auto load_into = [&](const ChunkSystem& cs) {
#pragma unroll
        for (int a = 0; a < 2; ++a) into[a] = *reinterpret_cast<const floatx4*>(cs.into + 8 * w + 4 * a);
    };
    auto load_left = [&](const ChunkSystem& cs) {
#pragma unroll
        for (int a = 0; a < 2; ++a) left[a] = *reinterpret_cast<const floatx4*>(cs.left + 8 * w + 4 * a);
        whole = cs.into[kChunk - 1];
    };
    if (chunks > 0) {
        load_into(system(0));
        load_t(system(0));
        load_left(system(0));
    }
    lds_barrier();
    for (int n = 0; n < chunks; ++n) {
        const uintx4* kt = keys_lds + (n & 1) * Geo::kKeys;
        const uintx4* turned = turned_lds + (n & 1) * Geo::kKeys + lane;
        uintx4* parts = parts_lds + (n & 1) * Geo::kParts + part * KS * 2 * 64 + lane;
        floatx4* upd = upd_lds + (n & 1) * Geo::kUpd;
        const floatx4* val = val_lds + (n & 1) * Geo::kUpd;
        const ChunkSystem& next = system(n + 1);
        // P = K S^T (chunk rows by value dims)
        floatx4 pr[2] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
        for (int k0 = 0; k0 < KS; k0 += KB) {
            uintx4 kb[KB][2];
#pragma unroll
            for (int k = 0; k < KB; ++k)
#pragma unroll
                for (int a = 0; a < 2; ++a) kb[k][a] = kt[key_at(chunk_row(u, a), KS * w + k0 + k)];
            __builtin_amdgcn_sched_barrier(0);  // (all reads in flight before the first product)
#pragma unroll
            for (int k = 0; k < KB; ++k) {
                float x[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = st[(8 * (k0 + k) + j) % E][(8 * (k0 + k) + j) / E];
                Parts<3> sp;
                sp.split(x);
#pragma unroll
                for (int p = 2; p >= 0; --p) {
                    if (p < 2) parts[((k0 + k) * 2 + p) * 64] = sp.p[p];
#pragma unroll
                    for (int a = 0; a < 2; ++a) pr[a] = mfma(kb[k][a], sp.p[p], pr[a]);
                }
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        // V, K^T and the state's decay, beside the products' end (the reads first: left to the compiler some
        // came after the sums that need them, 2% of the walk)
        const floatx4 vv[2] = {val[slot(part, u, w, 0)], val[slot(part, u, w, 1)]};
        constexpr int KT = E < 8 ? E : 8;
        uintx4 kv[KT];
#pragma unroll
        for (int o = 0; o < KT; ++o) kv[o] = turned[o * 64];
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int o = 0; o < E; ++o) st[o] *= whole;
        // U = T diag(beta) Y, Y = V - exp(G) P (chains of products that add to one result wait for each
        // other: two or more take turns)
        Parts<3> yp;
        {
            float y[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = vv[j >> 2][j & 3] - into[j >> 2][j & 3] * pr[j >> 2][j & 3];
            yp.split(y);
        }
        load_into(next);
        floatx4 un[2] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
        for (int order = 2; order >= 0; --order)
#pragma unroll
            for (int i = 0; i <= order; ++i)
#pragma unroll
                for (int a = 0; a < 2; ++a) un[a] = mfma(top[order - i][a], yp.p[i], un[a]);
        load_t(next);
        // S^T = exp(G_C) S^T + K^T (exp(G_C - G) U)
        Parts<3> zp;
        {
            float z[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) z[j] = left[j >> 2][j & 3] * un[j >> 2][j & 3];
            zp.split(z);
        }
#pragma unroll
        for (int a = 0; a < 2; ++a) upd[slot(part, u, w, a)] = un[a];
        load_left(next);
#pragma unroll
        for (int o = 0; o < E; o += 2) {
#pragma unroll
            for (int p = 2; p >= 0; --p)
#pragma unroll
                for (int i = 0; i < 2; ++i) st[o + i] = mfma(kv[(o + i) % KT], zp.p[p], st[o + i]);
            if (o + KT < E) kv[o] = turned[(o + KT) * 64], kv[o + 1] = turned[(o + 1 + KT) * 64];
        }
        lds_barrier();  // (the next chunk's loads stay in flight)
    }
    if (chunks > 0) {
        float sum = 0.0f;  // 0 or NaN
#pragma unroll
        for (int o = 0; o < E; ++o)
#pragma unroll
            for (int r = 0; r < 4; ++r) sum = fmaf(st[o][r], 0.0f, sum);
        const bool strange = __any(sum != 0.0f) && from < B.slots;  // (an origin out of range: NaN as it is)
        if (lane == 0) flags[part] = strange;
        lds_barrier();  // the output waves' last chunk
    }
    if (again()) return;
    const int to = B.last ? uniform_load(B.last + s) : -1;
    if (to < 0 || to >= B.slots) return;
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int o = 0; o < E; o += 4)
            *reinterpret_cast<floatx4*>(state_at(to, r) + o) =
                (floatx4){st[o][r], st[o + 1][r], st[o + 2][r], st[o + 3][r]};
}

// Sequences of up to so many rows go row by row. By rows and in chunks, us, 32 heads [128][128] / 16 [256][256] /
// 8 [64][64]: one sequence of 24 rows 18.6 and 15.2 / 26.5 and 18.2 / 13.1 and 13.3; eight of 16 rows 21.9 and
// 27.7 / 33.0 and 49.2 / 9.7 and 14.4, of 24 rows 28.0 and 28.0 / 43.4 and 49.8 / 13.1 and 14.2; 64 of 24 rows
// 158 and 172 / 318 and 391 / 18.3 and 27.5, of 28 rows 178 and 175 / 358 and 393 / 20.8 and 27.5, of 32 rows
// 196 and 179 / 398 and 395 / 23.2 and 27.7. (Few small heads would go by rows a little longer: 4 us of one call,
// which the rule leaves out.)
bool by_rows(const DeltaBatchDev& B, int max_rows) {
    return B.ckpt || B.rows == 0 || max_rows <= (B.seqs < 32 ? 16 : 28);
}
int chunk_bound(const DeltaBatchDev& B) { return B.rows / kChunk + (B.seqs < B.rows ? B.seqs : B.rows); }

template <int DK>
hipError_t launch_chunks(const DeltaDev& D, const DeltaBatchDev& B, ChunkSystem* sys, hipStream_t st) {
    const int bound = chunk_bound(B);
    const hipError_t e = D.hv / D.hk % 2 ? launch(k_delta_system<DK, 1>, dim3(bound, D.hv), dim3(64), 0, st, D, B, sys)
                                         : launch(k_delta_system<DK, 2>, dim3(bound, D.hv / 2), dim3(64), 0, st, D, B, sys);
    if (e != hipSuccess) return e;
    using Geo = WalkGeo<DK>;
    if (const hipError_t l = ensure_lds<k_delta_chunks<DK>>(Geo::kLds); l != hipSuccess) return l;
    const dim3 grid(D.dv / (16 * Geo::NW) * ((D.hv * B.seqs + 7) / 8 * 8));
    return launch(k_delta_chunks<DK>, grid, dim3(128 * Geo::NW), Geo::kLds, st, D, B, static_cast<const ChunkSystem*>(sys),
                  bound);
}

} // namespace

size_t delta_ws(const DeltaDev& D, const DeltaBatchDev& B, int max_rows) {
    return by_rows(B, max_rows) ? 0 : static_cast<size_t>(chunk_bound(B)) * D.hv * sizeof(ChunkSystem);
}

hipError_t launch_delta(const DeltaDev& D, const DeltaBatchDev& B, int max_rows, void* ws, hipStream_t st) {
    if (!by_rows(B, max_rows)) {
        ChunkSystem* sys = static_cast<ChunkSystem*>(ws);
        return D.dk == 64    ? launch_chunks<64>(D, B, sys, st)
               : D.dk == 128 ? launch_chunks<128>(D, B, sys, st)
                             : launch_chunks<256>(D, B, sys, st);
    }
    constexpr int R = 2;
    const dim3 grid(D.dv / (32 * R), D.hv, B.seqs);
    return D.dk == 64    ? launch(k_delta_rows<64, R>, grid, dim3(256), 0, st, D, B)
           : D.dk == 128 ? launch(k_delta_rows<128, R>, grid, dim3(256), 0, st, D, B)
                         : launch(k_delta_rows<256, R>, grid, dim3(256), 0, st, D, B);
}

} // namespace q38
