// q38_delta.hip — the gated delta rule of many requests over a pool of float states:
//   S <- exp(g) S,  S <- S + beta (v - S k) k^T,  o = scale * S q      per row and value head.
//
//   k_delta_rows   row by row, the state in registers across a sequence's rows
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

// Four waves take 32 value rows of one head of one sequence: 8 lanes per value row, lane `sub`
// of them key dims 32 c + 4 sub .. + 3 (16-byte state accesses, 128 bytes together per row).
template <int DK>
__global__ __launch_bounds__(256) void k_delta_rows(DeltaDev D, DeltaBatchDev B) {
    constexpr int C = DK / 32;
    const int s = blockIdx.z, h = blockIdx.y, sub = threadIdx.x & 7;
    const int dv = blockIdx.x * 32 + (threadIdx.x >> 3);
    const int hk = h / (D.hv / D.hk);
    const RowSpan span = row_span(B.off, s, B.rows);
    const int from = B.origin ? B.origin[s] : -1;
    const size_t elems = static_cast<size_t>(D.hv) * D.dv * DK;
    const size_t lane_at = (static_cast<size_t>(h) * D.dv + dv) * DK + 4 * sub;
    float4 st[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        st[c] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (from >= B.slots) st[c].x = st[c].y = st[c].z = st[c].w = __uint_as_float(0x7fc00000u);
        else if (from >= 0) st[c] = *reinterpret_cast<const float4*>(B.states + from * elems + lane_at + 32 * c);
    }
    auto store = [&](int slot) {
        if (slot < 0 || slot >= B.slots) return;
#pragma unroll
        for (int c = 0; c < C; ++c) *reinterpret_cast<float4*>(B.states + slot * elems + lane_at + 32 * c) = st[c];
    };
    struct RowIn {
        uint2 k[C], q[C];
        float v, g, b;
        int to;
    };
    auto load = [&](int r) {
        RowIn x;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            x.k[c] = *reinterpret_cast<const uint2*>(D.k + r * D.ks + hk * DK + 32 * c + 4 * sub);
            x.q[c] = *reinterpret_cast<const uint2*>(D.q + r * D.qs + hk * DK + 32 * c + 4 * sub);
        }
        x.v = bf2f(D.v[r * D.vs + h * D.dv + dv]);
        x.g = D.g[static_cast<size_t>(r) * D.hv + h];
        x.b = D.beta[static_cast<size_t>(r) * D.hv + h];
        x.to = B.ckpt ? B.ckpt[r] : -1;
        return x;
    };
    RowIn next;
    if (span.begin < span.end) next = load(span.begin);
    for (int r = span.begin; r < span.end; ++r) {
        const RowIn x = next;
        if (r + 1 < span.end) next = load(r + 1);
        const float decay = expf(x.g);
        float hit = 0.0f;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            st[c].x *= decay, st[c].y *= decay, st[c].z *= decay, st[c].w *= decay;
            hit = fmaf(st[c].x, bflo(x.k[c].x), hit);
            hit = fmaf(st[c].y, bfhi(x.k[c].x), hit);
            hit = fmaf(st[c].z, bflo(x.k[c].y), hit);
            hit = fmaf(st[c].w, bfhi(x.k[c].y), hit);
        }
        const float u = x.b * (x.v - sum8(hit));
        float o = 0.0f;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            st[c].x = fmaf(u, bflo(x.k[c].x), st[c].x);
            st[c].y = fmaf(u, bfhi(x.k[c].x), st[c].y);
            st[c].z = fmaf(u, bflo(x.k[c].y), st[c].z);
            st[c].w = fmaf(u, bfhi(x.k[c].y), st[c].w);
            o = fmaf(st[c].x, bflo(x.q[c].x), o);
            o = fmaf(st[c].y, bfhi(x.q[c].x), o);
            o = fmaf(st[c].z, bflo(x.q[c].y), o);
            o = fmaf(st[c].w, bfhi(x.q[c].y), o);
        }
        o = sum8(o);
        if (sub == 0) D.out[(static_cast<size_t>(r) * D.hv + h) * D.dv + dv] = f2bf(o * D.scale);
        store(x.to);
    }
    if (B.last) store(B.last[s]);
}

} // namespace

size_t delta_ws(const DeltaDev&, const DeltaBatchDev&, int) { return 0; }

hipError_t launch_delta(const DeltaDev& D, const DeltaBatchDev& B, int, void*, hipStream_t st) {
    const dim3 grid(D.dv / 32, D.hv, B.seqs);
    return D.dk == 64    ? launch(k_delta_rows<64>, grid, dim3(256), 0, st, D, B)
           : D.dk == 128 ? launch(k_delta_rows<128>, grid, dim3(256), 0, st, D, B)
                         : launch(k_delta_rows<256>, grid, dim3(256), 0, st, D, B);
}

} // namespace q38
