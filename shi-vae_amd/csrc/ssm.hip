// Selective state-space scan, forward, backward and single token:
//   s = softplus(dt + dt_bias), a[n] = exp(s A[n]), h[n] = a[n] h[n] + s u B[n], y = (sum_n C[n] h[n] + Dp u) silu(z)
// Backward, with g[n] = dL/dh[n] running from the last row to the first and dy' = dy silu(z):
//   g[n] = C[n] dy' + (a g)[n] of the next row;  dC[n] = sum_d dy' h[n];  dB[n] = sum_d g[n] s u
//   ds = sum_n (a g)[n] h_prev[n] A[n] + u sum_n g[n] B[n];  du = s sum_n g[n] B[n] + Dp dy';  dA[n] = sum_t (a g)[n] h_prev[n] s
// A is general (one number per channel and state), so the recurrence is element-wise in (d, n) and has no matrix form:
// one exponential, one product and two fused multiply-adds per (row, channel, state).  A wave64 instruction takes 4 cycles,
// the exponential 16, so 16 states cost 512 cycles per row and 64 channels, softplus and the gate about 160 more: the
// whole card does 235 G (row, channel) pairs a second, which is 1.9 TB/s of bf16 traffic.  Bound by vector instructions,
// not by memory.
//
// Layout: lane = channel (64 neighbouring channels per workgroup, one cache line of bf16), the states of a channel are dealt
// to the workgroup's waves, S to each.  Rows come in tiles of 16: all threads together load u, dt, z, B, C of the next tile
// while the present one runs, and put s and s u (once per channel, not once per wave) and fp32 copies of B and C into LDS;
// every wave then runs its states through the tile and leaves its part of y in LDS; all threads add the parts, gate, store.
// Where B * D is small, the time axis is split into pieces: a first launch runs each piece from a zero state and keeps its
// last state and sum of s; since prod_t exp(s_t A) = exp(A sum_t s_t), a piece of the second launch gets its first state
// from those of the pieces in front of it.
#include <algorithm>

#include "common.h"
#include "elem.h"

namespace shivae {

size_t sum_parts_floats(int64_t n, int64_t cols);
int launch_sum_parts(const float* part, int64_t n, int cols, float* mid, float* out0, int split, float* out1, hipStream_t stream);

constexpr int TT = SHIVAE_SCAN_CKPT;  // rows per tile

struct SsmP {
    shivae_ssm_args a;
    int E, tiles_g, tiles;  // channels per group, 64-channel tiles per group and in all
    int np, plen;           // pieces of the time axis, rows per piece (a multiple of TT)
    float* hend;            // [np][B][N][D] a piece's last state (backward: the adjoint that leaves it at its first row)
    float* ssum;            // [np][B][D] sum of s over a piece
    float *pbc, *pA, *pD;   // backward: partial sums [tiles][T * B][2][N], [np * B][N][D], [np * B][2][D]
};

__device__ __forceinline__ int ssm_len(const SsmP& p, int b) {
    if (!p.a.lengths) return p.a.T;
    const int n = p.a.lengths[b];
    return n < 0 ? 0 : (n < p.a.T ? n : p.a.T);
}

// One workgroup's place: piece, sequence, group, and this lane's channel.
struct Place {
    int piece, b, g, tile, d;
    bool ok;
};
__device__ __forceinline__ Place ssm_place(const SsmP& p, int lane) {
    Place q;
    unsigned i = blockIdx.x;
    q.tile = i % p.tiles;
    i /= p.tiles;
    q.b = i % p.a.B;
    q.piece = i / p.a.B;
    q.g = q.tile / p.tiles_g;
    const int e = (q.tile - q.g * p.tiles_g) * 64 + lane;
    q.ok = e < p.E;
    q.d = q.g * p.E + (q.ok ? e : 0);
    return q;
}

// FIRST: the launch that finds the pieces' last states (no y).
template <class E, int S, int NW, bool FIRST>
__global__ __launch_bounds__(64 * NW) void ssm_fwd_kernel(SsmP p) {
    constexpr int NP = S * NW, KT = TT / NW, NB = (TT * NP + 64 * NW - 1) / (64 * NW);
    __shared__ float2 sd[TT][64];
    __shared__ __attribute__((aligned(16))) float sB[TT][NP], sC[FIRST ? 1 : TT][NP];
    __shared__ float sy[FIRST ? 1 : NW][TT][64];
    const shivae_ssm_args& a = p.a;
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const Place q = ssm_place(p, lane);
    const int n = ssm_len(p, q.b), t0 = q.piece * p.plen, t1 = min(a.T, t0 + p.plen), tn = min(t1, n);

    float h[S], A2[S];
#pragma unroll
    for (int j = 0; j < S; ++j) {
        const int s = w * S + j;
        const bool live = q.ok && s < a.N;
        const int64_t o = ((int64_t)q.b * a.N + s) * a.D + q.d;
        A2[j] = live ? a.A[(int64_t)s * a.D + q.d] * kLog2e : 0.f;
        h[j] = live && q.piece == 0 && a.state ? a.state[o] : 0.f;
        if (!FIRST && live)
            for (int c = 0; c < q.piece; ++c) {
                const float sum = p.ssum[((int64_t)c * a.B + q.b) * a.D + q.d];
                h[j] = fmaf(__builtin_amdgcn_exp2f(A2[j] * sum), h[j], p.hend[(int64_t)c * a.B * a.N * a.D + o]);
            }
    }
    const float bias = a.dt_bias ? a.dt_bias[q.d] : 0.f, Dp = (!FIRST && a.Dp) ? a.Dp[q.d] : 0.f;
    const E* u = static_cast<const E*>(a.u) + (int64_t)q.b * a.u_sb + q.d;
    const E* dt = static_cast<const E*>(a.dt) + (int64_t)q.b * a.dt_sb + q.d;
    const E* z = a.z && !FIRST ? static_cast<const E*>(a.z) + (int64_t)q.b * a.z_sb + q.d : nullptr;
    E* y = FIRST ? nullptr : static_cast<E*>(a.y) + (int64_t)q.b * a.y_sb + q.d;
    const E* Bm = static_cast<const E*>(a.Bm) + (int64_t)q.b * a.B_sb + (int64_t)q.g * a.B_sg;
    const E* Cm = static_cast<const E*>(a.Cm) + (int64_t)q.b * a.C_sb + (int64_t)q.g * a.C_sg;

    // The next tile's operands, requested while the present one runs.
    E ru[KT], rd[KT], rz[KT], rB[NB], rC[NB];
    auto request = [&](int tb) {
#pragma unroll
        for (int k = 0; k < KT; ++k) {
            const int t = tb + w + NW * k;
            ru[k] = rd[k] = rz[k] = (E)0.f;
            if (t < tn && q.ok) {
                ru[k] = u[(int64_t)t * a.u_st];
                rd[k] = dt[(int64_t)t * a.dt_st];
                if (z) rz[k] = z[(int64_t)t * a.z_st];
            }
        }
#pragma unroll
        for (int k = 0; k < NB; ++k) {
            const int e = tid + 64 * NW * k, r = e / NP, s = e % NP;
            rB[k] = rC[k] = (E)0.f;
            if (r < TT && tb + r < tn && s < a.N) {
                rB[k] = Bm[(int64_t)(tb + r) * a.B_st + s];
                if (!FIRST) rC[k] = Cm[(int64_t)(tb + r) * a.C_st + s];
            }
        }
    };
    float total = 0.f;
    if (t0 < tn) request(t0);
    for (int tb = t0; tb < tn; tb += TT) {
        float ku[KT], kz[KT];
#pragma unroll
        for (int k = 0; k < KT; ++k) {
            const int r = w + NW * k;
            float s = elem_f(rd[k]) + bias;
            if (a.softplus) s = seq_softplus(s);
            ku[k] = elem_f(ru[k]);
            kz[k] = elem_f(rz[k]);
            if (tb + r >= tn) s = 0.f;  // rows behind the sequence leave the state as it is
            sd[r][lane] = make_float2(s, s * ku[k]);
        }
#pragma unroll
        for (int k = 0; k < NB; ++k) {
            const int e = tid + 64 * NW * k, r = e / NP, s = e % NP;
            if (r < TT) {
                sB[r][s] = elem_f(rB[k]);
                if constexpr (!FIRST) sC[r][s] = elem_f(rC[k]);
            }
        }
        __syncthreads();
        if (tb + TT < tn) request(tb + TT);
        if (!FIRST && a.ckpt && q.ok) {
#pragma unroll
            for (int j = 0; j < S; ++j)
                if (w * S + j < a.N) a.ckpt[(((int64_t)(tb / TT) * a.B + q.b) * a.N + w * S + j) * a.D + q.d] = h[j];
        }
#pragma unroll
        for (int r = 0; r < TT; ++r) {
            const float2 s = sd[r][lane];
            float acc = 0.f;
#pragma unroll
            for (int j = 0; j < S; ++j) {
                h[j] = fmaf(__builtin_amdgcn_exp2f(s.x * A2[j]), h[j], s.y * sB[r][w * S + j]);
                if constexpr (!FIRST) acc = fmaf(sC[r][w * S + j], h[j], acc);
            }
            if constexpr (FIRST) total += s.x;
            else sy[w][r][lane] = acc;
        }
        __syncthreads();
        if constexpr (!FIRST) {
#pragma unroll
            for (int k = 0; k < KT; ++k) {
                const int r = w + NW * k;
                float v = Dp * ku[k];
#pragma unroll
                for (int i = 0; i < NW; ++i) v += sy[i][r][lane];
                if (z) v *= kz[k] * seq_sigmoid(kz[k]);
                if (tb + r < tn && q.ok) y[(int64_t)(tb + r) * a.y_st] = f_elem<E>(v);
            }
        }
    }
    if (!q.ok) return;
    if (!FIRST)
        for (int t = max(t0, n) + w; t < t1; t += NW) y[(int64_t)t * a.y_st] = (E)0.f;
    float* out = FIRST ? p.hend + (int64_t)q.piece * a.B * a.N * a.D : (q.piece == p.np - 1 ? a.state_out : nullptr);
    if (out)
#pragma unroll
        for (int j = 0; j < S; ++j)
            if (w * S + j < a.N) out[((int64_t)q.b * a.N + w * S + j) * a.D + q.d] = h[j];
    if (FIRST && w == 0) p.ssum[((int64_t)q.piece * a.B + q.b) * a.D + q.d] = total;
}

// One row.  A thread owns V neighbouring channels of one sequence and walks the states: the fp32 state is read and written
// once, 16 bytes a lane, and is nearly all of the traffic.
template <class E, int V>
__global__ __launch_bounds__(256) void ssm_token_kernel(SsmP p, int nvec) {
    const shivae_ssm_args& a = p.a;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= (int64_t)a.B * nvec) return;
    const int b = (int)(i / nvec), d = (int)(i - (int64_t)b * nvec) * V, g = d / p.E;
    const bool live = ssm_len(p, b) > 0;
    const E* Bm = static_cast<const E*>(a.Bm) + (int64_t)b * a.B_sb + (int64_t)g * a.B_sg;
    const E* Cm = static_cast<const E*>(a.Cm) + (int64_t)b * a.C_sb + (int64_t)g * a.C_sg;
    float s[V], u[V], z[V], y[V];
    const Pack<E, V> ru = *reinterpret_cast<const Pack<E, V>*>(static_cast<const E*>(a.u) + (int64_t)b * a.u_sb + d);
    const Pack<E, V> rd = *reinterpret_cast<const Pack<E, V>*>(static_cast<const E*>(a.dt) + (int64_t)b * a.dt_sb + d);
    Pack<E, V> rz = {};
    if (a.z) rz = *reinterpret_cast<const Pack<E, V>*>(static_cast<const E*>(a.z) + (int64_t)b * a.z_sb + d);
#pragma unroll
    for (int c = 0; c < V; ++c) {
        u[c] = elem_f(ru.v[c]);
        z[c] = elem_f(rz.v[c]);
        s[c] = elem_f(rd.v[c]) + (a.dt_bias ? a.dt_bias[d + c] : 0.f);
        if (a.softplus) s[c] = seq_softplus(s[c]);
        y[c] = a.Dp ? a.Dp[d + c] * u[c] : 0.f;
    }
    const int64_t o = (int64_t)b * a.N * a.D + d;
#pragma unroll 8
    for (int n = 0; n < a.N; ++n) {
        Pack<float, V> h = {}, A = *reinterpret_cast<const Pack<float, V>*>(a.A + (int64_t)n * a.D + d);
        if (a.state) h = *reinterpret_cast<const Pack<float, V>*>(a.state + o + (int64_t)n * a.D);
        if (live) {
            const float Bn = elem_f(Bm[n]), Cn = elem_f(Cm[n]);
#pragma unroll
            for (int c = 0; c < V; ++c) {
                h.v[c] = fmaf(__builtin_amdgcn_exp2f(s[c] * (A.v[c] * kLog2e)), h.v[c], s[c] * u[c] * Bn);
                y[c] = fmaf(Cn, h.v[c], y[c]);
            }
        }
        if (a.state_out) *reinterpret_cast<Pack<float, V>*>(a.state_out + o + (int64_t)n * a.D) = h;
    }
    Pack<E, V> ry;
#pragma unroll
    for (int c = 0; c < V; ++c) {
        if (a.z) y[c] *= z[c] * seq_sigmoid(z[c]);
        ry.v[c] = live ? f_elem<E>(y[c]) : (E)0.f;
    }
    *reinterpret_cast<Pack<E, V>*>(static_cast<E*>(a.y) + (int64_t)b * a.y_sb + d) = ry;
}

// Sums eight values over the wave's 64 lanes.  v_permlane32_swap / v_permlane16_swap put two values' halves into one register,
// so a step halves the registers and not only the lanes; the last four steps rotate within rows of 16 lanes.  Afterwards every
// lane of 16-lane row r holds the sum of v[R(r)] in lo and of v[4 + R(r)] in hi, R = 0, 2, 1, 3.
__device__ __forceinline__ float swap32_add(float x, float y) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(y), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float swap16_add(float x, float y) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(y), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
template <int CTRL>
__device__ __forceinline__ float dpp_add(float x) {
    return x + __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), CTRL, 0xf, 0xf, false));
}
__device__ __forceinline__ float row16_sum(float x) {
    x = dpp_add<0x128>(x);  // row_ror:8, 4, 2, 1
    x = dpp_add<0x124>(x);
    x = dpp_add<0x122>(x);
    return dpp_add<0x121>(x);
}

// FIRST: the launch that finds what each piece hands to the one in front of it, (a g) at its first row, from nothing behind.
// Q passes of NW * S states each run through a tile one after another (Q > 1: more than 16 states).
template <class E, int S, int Q, bool FIRST>
__global__ __launch_bounds__(256, 2) void ssm_bwd_kernel(SsmP p) {
    constexpr int NW = 4, NP = S * NW * Q, KT = TT / NW, NB = (TT * NP + 255) / 256;
    __shared__ float2 sd[TT][64];
    __shared__ float sg[TT][64];
    __shared__ __attribute__((aligned(16))) float sB[TT][NP], sC[TT][NP];
    __shared__ float part[FIRST ? 1 : 3][FIRST ? 1 : NW][TT][64];  // of y, of sum g B, of sum (a g) h_prev A
    const shivae_ssm_args& a = p.a;
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const Place q = ssm_place(p, lane);
    const int n = ssm_len(p, q.b), t0 = q.piece * p.plen, t1 = min(a.T, t0 + p.plen), tn = min(t1, n);

    float ag[Q][S], A2[Q][S], dA[Q][S];
#pragma unroll
    for (int k = 0; k < Q; ++k)
#pragma unroll
        for (int j = 0; j < S; ++j) {
            const int s = (k * NW + w) * S + j;
            const bool live = q.ok && s < a.N;
            const int64_t o = ((int64_t)q.b * a.N + s) * a.D + q.d;
            A2[k][j] = live ? a.A[(int64_t)s * a.D + q.d] * kLog2e : 0.f;
            dA[k][j] = 0.f;
            ag[k][j] = live && q.piece == p.np - 1 && a.dstate_out ? a.dstate_out[o] : 0.f;
            if (!FIRST && live)
                for (int c = p.np - 1; c > q.piece; --c) {
                    const float sum = p.ssum[((int64_t)c * a.B + q.b) * a.D + q.d];
                    ag[k][j] = fmaf(__builtin_amdgcn_exp2f(A2[k][j] * sum), ag[k][j], p.hend[(int64_t)c * a.B * a.N * a.D + o]);
                }
        }
    const float bias = a.dt_bias ? a.dt_bias[q.d] : 0.f, Dp = a.Dp ? a.Dp[q.d] : 0.f;
    const E* u = static_cast<const E*>(a.u) + (int64_t)q.b * a.u_sb + q.d;
    const E* dt = static_cast<const E*>(a.dt) + (int64_t)q.b * a.dt_sb + q.d;
    const E* z = a.z ? static_cast<const E*>(a.z) + (int64_t)q.b * a.z_sb + q.d : nullptr;
    const E* dy = static_cast<const E*>(a.dy) + (int64_t)q.b * a.dy_sb + q.d;
    const E* Bm = static_cast<const E*>(a.Bm) + (int64_t)q.b * a.B_sb + (int64_t)q.g * a.B_sg;
    const E* Cm = static_cast<const E*>(a.Cm) + (int64_t)q.b * a.C_sb + (int64_t)q.g * a.C_sg;
    const int64_t orow = (int64_t)a.B * a.D, obase = (int64_t)q.b * a.D + q.d;

    E ru[KT], rd[KT], rz[KT], rg[KT], rB[NB], rC[NB];
    auto request = [&](int tb) {
#pragma unroll
        for (int k = 0; k < KT; ++k) {
            const int t = tb + w + NW * k;
            ru[k] = rd[k] = rz[k] = rg[k] = (E)0.f;
            if (t < tn && q.ok) {
                if (!FIRST) ru[k] = u[(int64_t)t * a.u_st];
                rd[k] = dt[(int64_t)t * a.dt_st];
                if (z) rz[k] = z[(int64_t)t * a.z_st];
                rg[k] = dy[(int64_t)t * a.dy_st];
            }
        }
#pragma unroll
        for (int k = 0; k < NB; ++k) {
            const int e = tid + 256 * k, r = e / NP, s = e % NP;
            rB[k] = rC[k] = (E)0.f;
            if (r < TT && tb + r < tn && s < a.N) {
                if (!FIRST) rB[k] = Bm[(int64_t)(tb + r) * a.B_st + s];
                rC[k] = Cm[(int64_t)(tb + r) * a.C_st + s];
            }
        }
    };
    float total = 0.f, dDp = 0.f, dbias = 0.f;
    const int last = t0 < tn ? (tn - 1) / TT * TT : t0;
    if (t0 < tn) request(last);
    for (int tb = last; tb >= t0 && t0 < tn; tb -= TT) {
        float ku[KT], kx[KT], kz[KT], ky[KT], ks[KT];  // u, dt + bias, z, dy, s of this thread's rows
#pragma unroll
        for (int k = 0; k < KT; ++k) {
            const int r = w + NW * k;
            ku[k] = elem_f(ru[k]);
            kz[k] = elem_f(rz[k]);
            ky[k] = elem_f(rg[k]);
            kx[k] = elem_f(rd[k]) + bias;
            ks[k] = a.softplus ? seq_softplus(kx[k]) : kx[k];
            if (tb + r >= tn) ks[k] = 0.f;
            sd[r][lane] = make_float2(ks[k], ks[k] * ku[k]);
            sg[r][lane] = z ? ky[k] * (kz[k] * seq_sigmoid(kz[k])) : ky[k];
        }
#pragma unroll
        for (int k = 0; k < NB; ++k) {
            const int e = tid + 256 * k, r = e / NP, s = e % NP;
            if (r < TT) {
                if (!FIRST) sB[r][s] = elem_f(rB[k]);
                sC[r][s] = elem_f(rC[k]);
            }
        }
        __syncthreads();
        if (tb - TT >= t0) request(tb - TT);
#pragma unroll
        for (int k = 0; k < Q; ++k) {
            const int s0 = (k * NW + w) * S;
            if constexpr (FIRST) {
#pragma unroll
                for (int r = TT - 1; r >= 0; --r) {
                    const float s = sd[r][lane].x, gy = sg[r][lane];
#pragma unroll
                    for (int j = 0; j < S; ++j) ag[k][j] = __builtin_amdgcn_exp2f(s * A2[k][j]) * fmaf(sC[r][s0 + j], gy, ag[k][j]);
                    if (k == 0) total += s;
                }
            } else {
            // forward through the tile again: states and decays stay in registers
            float h[TT][S], e[TT][S], first[S];
#pragma unroll
            for (int j = 0; j < S; ++j) {
                first[j] = 0.f;
                if (q.ok && s0 + j < a.N) first[j] = a.ckpt[(((int64_t)(tb / TT) * a.B + q.b) * a.N + s0 + j) * a.D + q.d];
            }
#pragma unroll
            for (int r = 0; r < TT; ++r) {
                const float2 s = sd[r][lane];
                float acc = 0.f;
#pragma unroll
                for (int j = 0; j < S; ++j) {
                    e[r][j] = __builtin_amdgcn_exp2f(s.x * A2[k][j]);
                    h[r][j] = fmaf(e[r][j], r ? h[r ? r - 1 : 0][j] : first[j], s.y * sB[r][s0 + j]);
                    acc = fmaf(sC[r][s0 + j], h[r][j], acc);
                }
                if (z) part[0][w][r][lane] = k ? part[0][w][r][lane] + acc : acc;
            }
            // and back
            float outB = 0.f, outC = 0.f;
#pragma unroll
            for (int r = TT - 1; r >= 0; --r) {
                const float2 s = sd[r][lane];
                const float gy = sg[r][lane];
                float gb = 0.f, gs = 0.f, vB[4] = {0.f, 0.f, 0.f, 0.f}, vC[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = 0; j < S; ++j) {
                    const float g = fmaf(sC[r][s0 + j], gy, ag[k][j]);
                    vC[j] = gy * h[r][j];
                    vB[j] = g * s.y;
                    gb = fmaf(g, sB[r][s0 + j], gb);
                    ag[k][j] = e[r][j] * g;
                    const float m = ag[k][j] * (r ? h[r ? r - 1 : 0][j] : first[j]);
                    gs = fmaf(m, A2[k][j], gs);
                    dA[k][j] = fmaf(m, s.x, dA[k][j]);
                }
                part[1][w][r][lane] = k ? part[1][w][r][lane] + gb : gb;
                part[2][w][r][lane] = k ? part[2][w][r][lane] + gs : gs;
                const float xB = swap16_add(swap32_add(vB[0], vB[1]), S > 2 ? swap32_add(vB[2], vB[3]) : 0.f);
                const float xC = swap16_add(swap32_add(vC[0], vC[1]), S > 2 ? swap32_add(vC[2], vC[3]) : 0.f);
                const float cB = row16_sum(xB), cC = row16_sum(xC);
                if ((lane & 15) == r) {
                    outB = cB;
                    outC = cC;
                }
            }
            const int r = lane & 15, row = lane >> 4, j = (row & 1) * 2 + (row >> 1);  // 16-lane row -> state
            if (tb + r < tn && j < S && s0 + j < a.N) {
                float* o = p.pbc + (((int64_t)q.tile * a.T + tb + r) * a.B + q.b) * 2 * a.N + s0 + j;
                o[0] = outB;
                o[a.N] = outC;
            }
            }
        }
        __syncthreads();
        if constexpr (!FIRST) {
#pragma unroll
            for (int k = 0; k < KT; ++k) {
                const int r = w + NW * k;
                if (tb + r >= tn || !q.ok) continue;
                float gb = 0.f, gs = 0.f;
#pragma unroll
                for (int i = 0; i < NW; ++i) {
                    gb += part[1][i][r][lane];
                    gs += part[2][i][r][lane];
                }
                const float gy = sg[r][lane];
                float ds = fmaf(ku[k], gb, gs * kLn2);
                if (a.softplus) ds *= seq_sigmoid(kx[k]);
                const int64_t o = (int64_t)(tb + r) * orow + obase;
                static_cast<E*>(a.du)[o] = f_elem<E>(fmaf(ks[k], gb, Dp * gy));
                static_cast<E*>(a.ddt)[o] = f_elem<E>(ds);
                dbias += ds;
                dDp = fmaf(gy, ku[k], dDp);
                if (z) {
                    float y = Dp * ku[k];
#pragma unroll
                    for (int i = 0; i < NW; ++i) y += part[0][i][r][lane];
                    const float sig = seq_sigmoid(kz[k]);
                    static_cast<E*>(a.dz)[o] = f_elem<E>(ky[k] * y * fmaf(kz[k] * sig, 1.f - sig, sig));
                }
            }
            __syncthreads();  // sg and part are written again by the next tile
        }
    }
    if constexpr (FIRST) {
        if (!q.ok) return;
#pragma unroll
        for (int k = 0; k < Q; ++k)
#pragma unroll
            for (int j = 0; j < S; ++j) {
                const int s = (k * NW + w) * S + j;
                if (s < a.N) p.hend[(((int64_t)q.piece * a.B + q.b) * a.N + s) * a.D + q.d] = ag[k][j];
            }
        if (w == 0) p.ssum[((int64_t)q.piece * a.B + q.b) * a.D + q.d] = total;
    } else {
    __syncthreads();
    part[0][w][0][lane] = dDp;
    part[0][w][1][lane] = dbias;
    __syncthreads();
    if (!q.ok) return;
    const int64_t pb = (int64_t)q.piece * a.B + q.b;
    if (w < 2) {
        float v = 0.f;
#pragma unroll
        for (int i = 0; i < NW; ++i) v += part[0][i][w][lane];
        p.pD[(pb * 2 + w) * a.D + q.d] = v;
    }
#pragma unroll
    for (int k = 0; k < Q; ++k)
#pragma unroll
        for (int j = 0; j < S; ++j) {
            const int s = (k * NW + w) * S + j;
            if (s >= a.N) continue;
            p.pA[(pb * a.N + s) * a.D + q.d] = dA[k][j];
            if (q.piece == 0 && a.dstate) a.dstate[((int64_t)q.b * a.N + s) * a.D + q.d] = ag[k][j];
        }
    for (int t = max(t0, n) + w; t < t1; t += NW) {
        const int64_t o = (int64_t)t * orow + obase;
        static_cast<E*>(a.du)[o] = (E)0.f;
        static_cast<E*>(a.ddt)[o] = (E)0.f;
        if (z) static_cast<E*>(a.dz)[o] = (E)0.f;
    }
    }
}

// dB, dC = the sums of the channel tiles' parts, rounded once; 0 behind a sequence's last row.
template <class E>
__global__ __launch_bounds__(256) void ssm_dbc_kernel(SsmP p) {
    const shivae_ssm_args& a = p.a;
    const int64_t rows = (int64_t)a.T * a.B, total = rows * a.G * 2 * a.N;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= total) return;
    const int w2 = 2 * a.N, k = (int)(i % w2);
    const int64_t rg = i / w2, row = rg % rows;
    const int g = (int)(rg / rows), t = (int)(row / a.B), b = (int)(row - (int64_t)t * a.B);
    float v = 0.f;
    if (t < ssm_len(p, b))
        for (int c = 0; c < p.tiles_g; ++c) v += p.pbc[((int64_t)(g * p.tiles_g + c) * rows + row) * w2 + k];
    const bool isC = k >= a.N;
    static_cast<E*>(isC ? a.dC : a.dB)[(row * a.G + g) * a.N + (isC ? k - a.N : k)] = f_elem<E>(v);
}

static int ssm_check(const shivae_ssm_args* a, const char* who) {
    SV_REQUIRE(a, "%s: null argument block", who);
    SV_REQUIRE(a->T > 0 && a->B > 0 && a->D > 0, "%s: T, B, D must be positive (%d, %d, %d)", who, a->T, a->B, a->D);
    SV_REQUIRE(a->N >= 1 && a->N <= 64, "%s: %d states per channel, 1..64 are supported", who, a->N);
    SV_REQUIRE(a->G >= 1 && a->D % a->G == 0, "%s: %d groups do not divide %d channels", who, a->G, a->D);
    SV_REQUIRE(a->dtype == SHIVAE_F32 || a->dtype == SHIVAE_BF16 || a->dtype == SHIVAE_F16, "%s: unknown dtype %d", who, a->dtype);
    SV_REQUIRE(a->T <= 1 << 30 && a->D <= 1 << 24, "%s: T or D is too large", who);
    SV_REQUIRE(a->u && a->dt && a->A && a->Bm && a->Cm, "%s: u, dt, A, B and C are required", who);
    return SHIVAE_OK;
}

// Pieces of the time axis.  A split costs the second launch's work again without y (about 0.9 of it), so it is taken only
// where the unsplit grid leaves most of the card idle: pieces until there are `want` workgroups, at least 64 rows each.
static void ssm_split(SsmP& p, int64_t want) {
    const shivae_ssm_args& a = p.a;
    p.E = a.D / a.G;
    p.tiles_g = ceil_div(p.E, 64);
    p.tiles = p.tiles_g * a.G;
    const int64_t groups = (int64_t)p.tiles * a.B;
    int64_t np = 1;
    if (2 * groups <= want) np = std::min<int64_t>({want / groups, 32, ceil_div(a.T, 64)});
    p.plen = np > 1 ? round_up(ceil_div(a.T, (int)np), TT) : round_up(a.T, TT);
    p.np = ceil_div(a.T, p.plen);
}
constexpr int64_t kFwdWant = 512, kBwdWant = 512;

static size_t piece_floats(const SsmP& p) { return p.np > 1 ? (size_t)p.np * p.a.B * (p.a.N + 1) * p.a.D : 0; }

template <class E>
static void launch_ssm_fwd(const SsmP& p, bool first, int pieces, hipStream_t s) {
    const dim3 grid((unsigned)((int64_t)p.tiles * p.a.B * pieces));
#define SV_SSM(S, NW)                                                                                   \
    if (first) hipLaunchKernelGGL((ssm_fwd_kernel<E, S, NW, true>), grid, dim3(64 * NW), 0, s, p);      \
    else hipLaunchKernelGGL((ssm_fwd_kernel<E, S, NW, false>), grid, dim3(64 * NW), 0, s, p)
    const int N = p.a.N;
    if (N <= 4) { SV_SSM(1, 4); }
    else if (N <= 8) { SV_SSM(2, 4); }
    else if (N <= 16) { SV_SSM(4, 4); }
    else if (N <= 32) { SV_SSM(4, 8); }
    else { SV_SSM(8, 8); }
#undef SV_SSM
}

template <class E>
static void launch_ssm_bwd(const SsmP& p, bool first, hipStream_t s) {
    const dim3 grid((unsigned)((int64_t)p.tiles * p.a.B * p.np));
#define SV_SSM(S, Q)                                                                                  \
    if (first) hipLaunchKernelGGL((ssm_bwd_kernel<E, S, Q, true>), grid, dim3(256), 0, s, p);         \
    else hipLaunchKernelGGL((ssm_bwd_kernel<E, S, Q, false>), grid, dim3(256), 0, s, p)
    const int N = p.a.N;
    if (N <= 8) { SV_SSM(2, 1); }
    else if (N <= 16) { SV_SSM(4, 1); }
    else if (N <= 32) { SV_SSM(4, 2); }
    else { SV_SSM(4, 4); }
#undef SV_SSM
}

}  // namespace shivae

using namespace shivae;

extern "C" {

size_t shivae_selective_scan_fwd_ws(const shivae_ssm_args* args) {
    if (ssm_check(args, "selective_scan_fwd_ws") != SHIVAE_OK) return 0;
    SsmP p{*args};
    ssm_split(p, kFwdWant);
    return piece_floats(p) * sizeof(float);
}

int shivae_selective_scan_fwd(const shivae_ssm_args* args, void* ws_dev, size_t ws_bytes, shivae_stream stream) {
    SV_TRY(ssm_check(args, "selective_scan_fwd"));
    SsmP p{*args};
    const shivae_ssm_args& a = p.a;
    SV_REQUIRE(a.y, "selective_scan_fwd: y is required");
    SV_REQUIRE(!a.state || a.state != a.state_out || a.T <= TT, "selective_scan_fwd: the state can be updated in place for up to %d rows only", TT);
    ssm_split(p, kFwdWant);
    SV_REQUIRE((int64_t)p.tiles * a.B * p.np < (int64_t)1 << 31, "selective_scan_fwd: B * D is too large");
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (a.T == 1 && !a.ckpt) {
        const int V = 4;
        const bool vec = p.E % V == 0 && a.u_sb % V == 0 && a.dt_sb % V == 0 && a.z_sb % V == 0 && a.y_sb % V == 0 && aligned_to(a.u, 16) && aligned_to(a.dt, 16) &&
                         aligned_to(a.z, 16) && aligned_to(a.y, 16) && aligned_to(a.A, 16) && aligned_to(a.state, 16) && aligned_to(a.state_out, 16);
        const int nvec = vec ? a.D / V : a.D;
        const dim3 grid((unsigned)(((int64_t)a.B * nvec + 255) / 256));
        SV_BY_DTYPE(a.dtype, {
            if (vec) hipLaunchKernelGGL((ssm_token_kernel<E, 4>), grid, dim3(256), 0, s, p, nvec);
            else hipLaunchKernelGGL((ssm_token_kernel<E, 1>), grid, dim3(256), 0, s, p, nvec);
        });
        SV_CHECK_HIP(hipGetLastError());
        return SHIVAE_OK;
    }
    const size_t need = piece_floats(p) * sizeof(float);
    SV_REQUIRE(need == 0 || (ws_dev && ws_bytes >= need), "selective_scan_fwd: workspace of %zu bytes is smaller than %zu", ws_bytes, need);
    p.hend = static_cast<float*>(ws_dev);
    p.ssum = p.hend + (size_t)p.np * a.B * a.N * a.D;
    if (p.np > 1) SV_BY_DTYPE(a.dtype, launch_ssm_fwd<E>(p, true, p.np - 1, s));
    SV_BY_DTYPE(a.dtype, launch_ssm_fwd<E>(p, false, p.np, s));
    SV_CHECK_HIP(hipGetLastError());
    return SHIVAE_OK;
}

static size_t bwd_floats(const SsmP& p) {
    const shivae_ssm_args& a = p.a;
    return piece_floats(p) + (size_t)p.tiles * a.T * a.B * 2 * a.N + (size_t)p.np * a.B * (a.N + 2) * a.D +
           sum_parts_floats((int64_t)p.np * a.B, (int64_t)std::max(a.N, 2) * a.D);
}

size_t shivae_selective_scan_bwd_ws(const shivae_ssm_args* args) {
    if (ssm_check(args, "selective_scan_bwd_ws") != SHIVAE_OK) return 0;
    SsmP p{*args};
    ssm_split(p, kBwdWant);
    return bwd_floats(p) * sizeof(float);
}

int shivae_selective_scan_bwd(const shivae_ssm_args* args, void* ws_dev, size_t ws_bytes, shivae_stream stream) {
    SV_TRY(ssm_check(args, "selective_scan_bwd"));
    SsmP p{*args};
    const shivae_ssm_args& a = p.a;
    SV_REQUIRE(a.dy && a.du && a.ddt && a.dB && a.dC && a.dA && a.ckpt, "selective_scan_bwd: dy, du, ddt, dB, dC, dA and the forward's ckpt are required");
    SV_REQUIRE((!a.z || a.dz) && (!a.Dp || a.dDp) && (!a.dt_bias || a.ddt_bias), "selective_scan_bwd: z, Dp and dt_bias need buffers for their gradients");
    ssm_split(p, kBwdWant);
    SV_REQUIRE((int64_t)p.tiles * a.B * p.np < (int64_t)1 << 31, "selective_scan_bwd: B * D is too large");
    const size_t need = bwd_floats(p) * sizeof(float);
    SV_REQUIRE(ws_dev && ws_bytes >= need, "selective_scan_bwd: workspace of %zu bytes is smaller than %zu", ws_bytes, need);
    hipStream_t s = static_cast<hipStream_t>(stream);
    p.hend = static_cast<float*>(ws_dev);
    p.ssum = p.hend + (p.np > 1 ? (size_t)p.np * a.B * a.N * a.D : 0);
    p.pbc = p.hend + piece_floats(p);
    p.pA = p.pbc + (size_t)p.tiles * a.T * a.B * 2 * a.N;
    p.pD = p.pA + (size_t)p.np * a.B * a.N * a.D;
    if (p.np > 1) SV_BY_DTYPE(a.dtype, launch_ssm_bwd<E>(p, true, s));
    SV_BY_DTYPE(a.dtype, launch_ssm_bwd<E>(p, false, s));
    SV_CHECK_HIP(hipGetLastError());
    const int64_t total = (int64_t)a.T * a.B * a.G * 2 * a.N;
    const dim3 grid((unsigned)((total + 255) / 256));
    SV_REQUIRE((total + 255) / 256 < (int64_t)1 << 31, "selective_scan_bwd: T * B * G * N is too large");
    SV_BY_DTYPE(a.dtype, hipLaunchKernelGGL((ssm_dbc_kernel<E>), grid, dim3(256), 0, s, p));
    SV_CHECK_HIP(hipGetLastError());
    float* mid = p.pD + (size_t)p.np * a.B * 2 * a.D;
    SV_TRY(launch_sum_parts(p.pA, (int64_t)p.np * a.B, a.N * a.D, mid, a.dA, a.N * a.D, nullptr, s));
    if (a.Dp || a.dt_bias) return launch_sum_parts(p.pD, (int64_t)p.np * a.B, 2 * a.D, mid, a.dDp, a.D, a.ddt_bias, s);
    return SHIVAE_OK;
}

}  // extern "C"
