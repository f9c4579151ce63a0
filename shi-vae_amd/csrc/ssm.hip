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
#include <utility>

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
    int vec;                // B and C can be read S states at a time
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
    int piece, b, g, tile;
    int d0;        // the tile's first channel
    unsigned lo;   // this lane's channel from there (0 where the tile has none for it)
    int d;
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
    const int e0 = (q.tile - q.g * p.tiles_g) * 64;
    q.ok = e0 + lane < p.E;
    q.d0 = q.g * p.E + e0;
    q.lo = q.ok ? lane : 0;
    q.d = q.d0 + (int)q.lo;
    return q;
}

// B and C of a row are the same for all channels of a group.  A wave needs S states of each for the 16 rows of a tile: lane l holds
// row l mod 16, one register per state, and v_mul / v_fmac take row r from there with row_newbcast:r at no extra instruction.  (From
// LDS a broadcast read still returns 64 lanes: 64 of 96 LDS cycles per row and 64 channels.  With scalar loads every row waited for
// its own: 757 us against 404 for LDS at T 2048, B 16, D 2048, N 16.)
template <int R>
__device__ __forceinline__ float row_of(float v) {
    return __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(v), 0x150 + R, 0xf, 0xf, true));
}
// acc + sum_j row_of<R>(c[j]) h[j], j < 3 or 4.  hipcc folds the row selection into a product but not into a fused multiply-add; a VGPR
// needs two wait states between being written and being read through DPP.
template <int R>
__device__ __forceinline__ void row_fmac3(float& acc, const float* c, const float* h) {
    asm("s_nop 1\n\t"
        "v_fmac_f32_dpp %0, %1, %4 row_newbcast:%7 row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f32_dpp %0, %2, %5 row_newbcast:%7 row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f32_dpp %0, %3, %6 row_newbcast:%7 row_mask:0xf bank_mask:0xf"
        : "+v"(acc) : "v"(c[0]), "v"(c[1]), "v"(c[2]), "v"(h[0]), "v"(h[1]), "v"(h[2]), "n"(R));
}
template <int R>
__device__ __forceinline__ void row_fmac4(float& acc, const float* c, const float* h) {
    asm("s_nop 1\n\t"
        "v_fmac_f32_dpp %0, %1, %5 row_newbcast:%9 row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f32_dpp %0, %2, %6 row_newbcast:%9 row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f32_dpp %0, %3, %7 row_newbcast:%9 row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f32_dpp %0, %4, %8 row_newbcast:%9 row_mask:0xf bank_mask:0xf"
        : "+v"(acc) : "v"(c[0]), "v"(c[1]), "v"(c[2]), "v"(c[3]), "v"(h[0]), "v"(h[1]), "v"(h[2]), "v"(h[3]), "n"(R));
}
template <int R, int S>
__device__ __forceinline__ float row_dot(const float (&c)[S], const float (&h)[S]) {
    float acc = row_of<R>(c[0]) * h[0];
    if constexpr (S == 2) acc = fmaf(row_of<R>(c[1]), h[1], acc);
    if constexpr (S >= 4) row_fmac3<R>(acc, c + 1, h + 1);
    if constexpr (S >= 8) row_fmac4<R>(acc, c + 4, h + 4);
    if constexpr (S >= 16) {
        row_fmac4<R>(acc, c + 8, h + 8);
        row_fmac4<R>(acc, c + 12, h + 12);
    }
    return acc;
}

template <class E>
__device__ __forceinline__ E at(const E* base, unsigned off) {  // off in bytes: a uniform base and a 32-bit offset per lane
    return *reinterpret_cast<const E*>(reinterpret_cast<const char*>(base) + off);
}
template <class E>
__device__ __forceinline__ void put(E* base, unsigned off, E v) {
    *reinterpret_cast<E*>(reinterpret_cast<char*>(base) + off) = v;
}

template <class E, int S>
struct RowRegs {
    float v[S];
    // base: row tb of this group's matrix; s0: first state; rows tb + (lane mod 16), 0 at and behind tn, states 0 at and behind N
    __device__ __forceinline__ void load(const E* base, unsigned stb, int s0, int N, bool vec, int left, int lane) {
        const int r = lane & 15;
        const unsigned off = (unsigned)min(r, left - 1) * stb;
        E e[S];
        if (vec) {
            const Pack<E, S> q = *reinterpret_cast<const Pack<E, S>*>(reinterpret_cast<const char*>(base + s0) + off);
#pragma unroll
            for (int j = 0; j < S; ++j) e[j] = q.v[j];
        } else {
#pragma unroll
            for (int j = 0; j < S; ++j) e[j] = at(base + min(s0 + j, N - 1), off);
        }
#pragma unroll
        for (int j = 0; j < S; ++j) v[j] = r < left && s0 + j < N ? elem_f(e[j]) : 0.f;
    }
};

// Rows r0, r0 + 4, r0 + 8, r0 + 12 of a tile of one [T][B][D] operand, as byte offsets from the tile's first row (the uniform base
// moves).  With fewer than 16 rows left the last one is read again.
struct TileRows {
    unsigned off[4];
    __device__ __forceinline__ void set(unsigned stb, int r0, unsigned lo_bytes, int left = TT) {
#pragma unroll
        for (int k = 0; k < 4; ++k) off[k] = (unsigned)min(r0 + 4 * k, left - 1) * stb + lo_bytes;
    }
    template <class E>
    __device__ __forceinline__ void load(E (&o)[4], const E* base) const {
#pragma unroll
        for (int k = 0; k < 4; ++k) o[k] = at(base, off[k]);
    }
};

// v_permlane32_swap / v_permlane16_swap put halves of two registers into one, so that adding the two sums both values over half of
// the lanes and halves the registers as well: swap16_add(swap32_add(a, b), swap32_add(c, d)) holds, in the 16-lane rows 0 to 3, the sums
// over the four rows of a, c, b, d.
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

template <int N, class F>
__device__ __forceinline__ void unroll(F f) {  // f(0), f(1), ... with the number as a constant
    [&]<int... I>(std::integer_sequence<int, I...>) { (f(std::integral_constant<int, I>{}), ...); }(std::make_integer_sequence<int, N>{});
}

// A wave owns 16 channels: lane = (state group g4 = lane / 16, channel lane % 16), S states of the channel per lane.  Of a tile's 16
// rows the lane prepares row 4 k + g4 for its channel (k = 0..3: softplus, s u, later the gate and the store), so that this work is done
// once per channel; the state groups get s and s u through the wave's own 2 KiB of LDS, and y's parts come back summed, row 4 k + g4 in
// lane row g4.  No barrier: a wave waits for nobody.
// FIRST: the launch that finds the pieces' last states (no y).
template <class E, int S, bool FIRST>
__global__ __launch_bounds__(256) void ssm_fwd_kernel(SsmP p) {
    const shivae_ssm_args& a = p.a;
    __shared__ float2 rows_s[4][TT][16];
    const int lane = threadIdx.x & 63, g4 = lane >> 4;
    float2 (&row)[TT][16] = rows_s[threadIdx.x >> 6];  // this wave's own: s, s u of 16 rows and channels
    const Place q = ssm_place(p, (int)(threadIdx.x >> 6) * 16 + (lane & 15));
    if (!__any(q.ok)) return;
    const int n = ssm_len(p, q.b), t0 = q.piece * p.plen, t1 = min(a.T, t0 + p.plen), tn = min(t1, n);
    const int64_t state0 = ((int64_t)q.b * a.N + g4 * S) * a.D + q.d, statep = (int64_t)a.B * a.N * a.D;

    float h[S], A2[S];
#pragma unroll
    for (int j = 0; j < S; ++j) {
        const bool live = q.ok && g4 * S + j < a.N;
        const int64_t o = state0 + (int64_t)j * a.D;
        A2[j] = live ? a.A[(int64_t)(g4 * S + j) * a.D + q.d] * kLog2e : 0.f;
        h[j] = live && q.piece == 0 && a.state ? a.state[o] : 0.f;
        if (!FIRST && live)
            for (int c = 0; c < q.piece; ++c) {
                const float sum = p.ssum[((int64_t)c * a.B + q.b) * a.D + q.d];
                h[j] = fmaf(__builtin_amdgcn_exp2f(A2[j] * sum), h[j], p.hend[c * statep + o]);
            }
    }
    const float bias = a.dt_bias ? a.dt_bias[q.d] : 0.f, Dp = (!FIRST && a.Dp) ? a.Dp[q.d] : 0.f;
    const unsigned le = q.lo * (unsigned)sizeof(E);
    const unsigned us = (unsigned)a.u_st * sizeof(E), ds = (unsigned)a.dt_st * sizeof(E), zs = (unsigned)a.z_st * sizeof(E), ys = (unsigned)a.y_st * sizeof(E);
    const unsigned Bs = (unsigned)a.B_st * sizeof(E), Cs = (unsigned)a.C_st * sizeof(E);
    const E* u = static_cast<const E*>(a.u) + (int64_t)q.b * a.u_sb + q.d0 + t0 * a.u_st;
    const E* dt = static_cast<const E*>(a.dt) + (int64_t)q.b * a.dt_sb + q.d0 + t0 * a.dt_st;
    const E* z = static_cast<const E*>(a.z) + (int64_t)q.b * a.z_sb + q.d0 + t0 * a.z_st;
    const E* Bm = static_cast<const E*>(a.Bm) + (int64_t)q.b * a.B_sb + (int64_t)q.g * a.B_sg + t0 * a.B_st;
    const E* Cm = static_cast<const E*>(a.Cm) + (int64_t)q.b * a.C_sb + (int64_t)q.g * a.C_sg + t0 * a.C_st;
    E* y = static_cast<E*>(a.y) + (int64_t)q.b * a.y_sb + q.d0 + t0 * a.y_st;
    const bool gate = !FIRST && a.z;
    TileRows ou, od, oz, oy;
    ou.set(us, g4, le);
    od.set(ds, g4, le);
    if (!FIRST) oz.set(zs, g4, le);
    if (!FIRST) oy.set(ys, g4, le);

    E ru[4], rd[4], rz[4];  // the next tile's operands, requested while the present one runs
    RowRegs<E, S> nB, nC;
    auto request = [&](int left) {
        if (left < TT) {
            ou.set(us, g4, le, left);
            od.set(ds, g4, le, left);
            if (!FIRST) oz.set(zs, g4, le, left);
        }
        ou.load(ru, u);
        od.load(rd, dt);
        if (gate) oz.load(rz, z);
        nB.load(Bm, Bs, g4 * S, a.N, p.vec, left, lane);
        if (!FIRST) nC.load(Cm, Cs, g4 * S, a.N, p.vec, left, lane);
        u += TT * a.u_st;
        dt += TT * a.dt_st;
        z += TT * a.z_st;
        Bm += TT * a.B_st;
        Cm += TT * a.C_st;
    };
    float total = 0.f;
    int left = tn - t0;  // rows from the present tile's first one
    float* ckpt = a.ckpt && !FIRST ? a.ckpt + (int64_t)(t0 / TT) * statep + state0 : nullptr;
    if (left > 0) request(left);
    for (; left > 0; left -= TT) {
        float s[4], ku[4], kz[4], v[4];
        // (flags outside of the loops over k: a branch between them would run the four chains of dependent operations in turn)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            s[k] = elem_f(rd[k]) + bias;
            ku[k] = elem_f(ru[k]);
        }
        if (gate)
#pragma unroll
            for (int k = 0; k < 4; ++k) kz[k] = elem_f(rz[k]);
        if (a.softplus)
#pragma unroll
            for (int k = 0; k < 4; ++k) s[k] = seq_softplus(s[k]);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const bool in = 4 * k + g4 < left;  // rows behind the sequence leave the state as it is
            s[k] = in ? s[k] : 0.f;
            if (FIRST) total += s[k];
            row[4 * k + g4][lane & 15] = make_float2(s[k], in ? s[k] * ku[k] : 0.f);
        }
        const RowRegs<E, S> vB = nB, vC = nC;
        if (left > TT) request(left - TT);
        if (ckpt) {
#pragma unroll
            for (int j = 0; j < S; ++j)
                if (q.ok && g4 * S + j < a.N) ckpt[(int64_t)j * a.D] = h[j];
            ckpt += statep;
        }
        float2 x[TT];
#pragma unroll
        for (int r = 0; r < TT; ++r) x[r] = row[r][lane & 15];
        unroll<4>([&](auto K) {
            constexpr int k = K;
            float acc[4];
            unroll<4>([&](auto I) {
                constexpr int i = I, r = 4 * k + i;
#pragma unroll
                for (int j = 0; j < S; ++j) h[j] = fmaf(__builtin_amdgcn_exp2f(x[r].x * A2[j]), h[j], row_of<r>(vB.v[j]) * x[r].y);
                if constexpr (!FIRST) acc[i] = row_dot<r>(vC.v, h);
            });
            if constexpr (!FIRST) v[k] = fmaf(Dp, ku[k], swap16_add(swap32_add(acc[0], acc[2]), swap32_add(acc[1], acc[3])));
        });
        if constexpr (!FIRST) {
            if (gate)
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] *= kz[k] * seq_sigmoid(kz[k]);
            if (q.ok) {
                if (left >= TT) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) put(y, oy.off[k], f_elem<E>(v[k]));
                } else {
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (4 * k + g4 < left) put(y, oy.off[k], f_elem<E>(v[k]));
                }
            }
            y += TT * a.y_st;
        }
    }
    if constexpr (!FIRST) {
        if (q.ok)
            for (int t = max(t0, n) + g4; t < t1; t += 4) (static_cast<E*>(a.y) + (int64_t)q.b * a.y_sb + q.d0 + t * a.y_st)[q.lo] = (E)0.f;
    }
    float* out = FIRST ? p.hend + q.piece * statep : (q.piece == p.np - 1 ? a.state_out : nullptr);
    if (out)
#pragma unroll
        for (int j = 0; j < S; ++j)
            if (q.ok && g4 * S + j < a.N) out[state0 + (int64_t)j * a.D] = h[j];
    if (FIRST) {
        total = swap32_add(total, total);
        total = swap16_add(total, total);  // over the four rows of lanes
        if (q.ok && g4 == 0) p.ssum[((int64_t)q.piece * a.B + q.b) * a.D + q.d] = total;
    }
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

// FIRST: the launch that finds what each piece hands to the one in front of it, (a g) at its first row, from nothing behind.
// Q passes of NW * S states each run through a tile one after another (Q > 1: more than 16 states).
template <class E, int S, int Q, bool FIRST>
__global__ __launch_bounds__(256, 2) void ssm_bwd_kernel(SsmP p) {
    constexpr int NW = 4, KT = TT / NW;
    __shared__ float2 sd[TT][64];
    __shared__ float sg[TT][64];
    __shared__ float part[FIRST ? 1 : 3][FIRST ? 1 : NW][TT][64];  // of y, of sum g B, of sum (a g) h_prev A
    const shivae_ssm_args& a = p.a;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
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
    const int64_t c0 = q.d0;
    const int last = t0 < tn ? (tn - 1) / TT * TT : t0;  // the last tile; from there to the front
    const unsigned le = q.lo * (unsigned)sizeof(E);
    const unsigned us = (unsigned)a.u_st * sizeof(E), ds = (unsigned)a.dt_st * sizeof(E), zs = (unsigned)a.z_st * sizeof(E), gs_ = (unsigned)a.dy_st * sizeof(E);
    const unsigned Bs = (unsigned)a.B_st * sizeof(E), Cs = (unsigned)a.C_st * sizeof(E), os = (unsigned)((int64_t)a.B * a.D * sizeof(E));
    const E* u = static_cast<const E*>(a.u) + (int64_t)q.b * a.u_sb + c0 + last * a.u_st;
    const E* dt = static_cast<const E*>(a.dt) + (int64_t)q.b * a.dt_sb + c0 + last * a.dt_st;
    const E* z = static_cast<const E*>(a.z) + (int64_t)q.b * a.z_sb + c0 + last * a.z_st;
    const E* dy = static_cast<const E*>(a.dy) + (int64_t)q.b * a.dy_sb + c0 + last * a.dy_st;
    const E* Bm = static_cast<const E*>(a.Bm) + (int64_t)q.b * a.B_sb + (int64_t)q.g * a.B_sg + last * a.B_st;
    const E* Cm = static_cast<const E*>(a.Cm) + (int64_t)q.b * a.C_sb + (int64_t)q.g * a.C_sg + last * a.C_st;
    const bool gate = a.z;
    TileRows ou, od, oz, og, oo;
    auto offsets = [&](int left) {
        if (!FIRST) ou.set(us, w, le, left);
        od.set(ds, w, le, left);
        oz.set(zs, w, le, left);
        og.set(gs_, w, le, left);
    };
    oo.set(os, w, le);

    E ru[KT], rd[KT], rz[KT], rg[KT];
    auto request = [&]() {
        if (!FIRST) ou.load(ru, u);
        od.load(rd, dt);
        if (gate) oz.load(rz, z);
        og.load(rg, dy);
        u -= TT * (int64_t)a.u_st;
        dt -= TT * (int64_t)a.dt_st;
        z -= TT * (int64_t)a.z_st;
        dy -= TT * (int64_t)a.dy_st;
    };
    float total = 0.f, dDp = 0.f, dbias = 0.f;
    int left = tn - last;
    if (left > 0) {
        offsets(min(left, TT));
        request();
        offsets(TT);
    }
    for (int tb = last; tb >= t0 && t0 < tn; tb -= TT, left = TT) {
        float ku[KT], kx[KT], kz[KT], ky[KT], ks[KT];  // u, dt + bias, z, dy, s of this thread's rows
#pragma unroll
        for (int k = 0; k < KT; ++k) {
            const int r = w + NW * k;
            const bool in = r < left && q.ok;  // (a lane without a channel adds nothing to dB and dC)
            ku[k] = FIRST ? 0.f : elem_f(ru[k]);
            kx[k] = elem_f(rd[k]) + bias;
            ks[k] = a.softplus ? seq_softplus(kx[k]) : kx[k];
            ky[k] = elem_f(rg[k]);
            float gy = ky[k];
            if (gate) {
                kz[k] = elem_f(rz[k]);
                gy *= kz[k] * seq_sigmoid(kz[k]);
            }
            if (!in) ks[k] = 0.f;
            sd[r][lane] = make_float2(ks[k], in ? ks[k] * ku[k] : 0.f);
            sg[r][lane] = in ? gy : 0.f;
        }
        __syncthreads();
        if (tb - TT >= t0) request();
#pragma unroll
        for (int k = 0; k < Q; ++k) {
            const int s0 = (k * NW + w) * S;
            RowRegs<E, S> vB, vC;
            vC.load(Cm, Cs, s0, a.N, p.vec, left, lane);
            if (!FIRST) vB.load(Bm, Bs, s0, a.N, p.vec, left, lane);
            if constexpr (FIRST) {
                unroll<TT>([&](auto I) {
                    constexpr int r = TT - 1 - I;
                    const float s = sd[r][lane].x, gy = sg[r][lane];
#pragma unroll
                    for (int j = 0; j < S; ++j) ag[k][j] = __builtin_amdgcn_exp2f(s * A2[k][j]) * fmaf(row_of<r>(vC.v[j]), gy, ag[k][j]);
                    if (k == 0) total += s;
                });
            } else {
            // forward through the tile again: states and decays stay in registers
            float h[TT][S], e[TT][S], first[S];
#pragma unroll
            for (int j = 0; j < S; ++j) {
                first[j] = 0.f;
                if (q.ok && s0 + j < a.N) first[j] = (a.ckpt + (((int64_t)(tb / TT) * a.B + q.b) * a.N + s0 + j) * a.D + c0)[q.lo];
            }
            unroll<TT>([&](auto R) {
                constexpr int r = R;
                const float2 s = sd[r][lane];
#pragma unroll
                for (int j = 0; j < S; ++j) {
                    e[r][j] = __builtin_amdgcn_exp2f(s.x * A2[k][j]);
                    h[r][j] = fmaf(e[r][j], r ? h[r ? r - 1 : 0][j] : first[j], row_of<r>(vB.v[j]) * s.y);
                }
                const float acc = row_dot<r>(vC.v, h[r]);
                if (gate) part[0][w][r][lane] = k ? part[0][w][r][lane] + acc : acc;
            });
            // and back
            float outB = 0.f, outC = 0.f;
            unroll<TT>([&](auto I) {
                constexpr int r = TT - 1 - I;
                const float2 s = sd[r][lane];
                const float gy = sg[r][lane];
                float g[S], gs = 0.f, xB[4] = {0.f, 0.f, 0.f, 0.f}, xC[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = 0; j < S; ++j) {
                    g[j] = ag[k][j] + row_of<r>(vC.v[j]) * gy;
                    xC[j] = gy * h[r][j];
                    xB[j] = g[j] * s.y;
                    ag[k][j] = e[r][j] * g[j];
                    const float m = ag[k][j] * (r ? h[r ? r - 1 : 0][j] : first[j]);
                    gs = fmaf(m, A2[k][j], gs);
                    dA[k][j] = fmaf(m, s.x, dA[k][j]);
                }
                const float gb = row_dot<r>(vB.v, g);
                part[1][w][r][lane] = k ? part[1][w][r][lane] + gb : gb;
                part[2][w][r][lane] = k ? part[2][w][r][lane] + gs : gs;
                const float yB = swap16_add(swap32_add(xB[0], xB[1]), S > 2 ? swap32_add(xB[2], xB[3]) : 0.f);
                const float yC = swap16_add(swap32_add(xC[0], xC[1]), S > 2 ? swap32_add(xC[2], xC[3]) : 0.f);
                const float cB = row16_sum(yB), cC = row16_sum(yC);
                if ((lane & 15) == r) {
                    outB = cB;
                    outC = cC;
                }
            });
            const int r = lane & 15, row = lane >> 4, j = (row & 1) * 2 + (row >> 1);  // 16-lane row -> state
            if (r < left && j < S && s0 + j < a.N) {
                float* o = p.pbc + (((int64_t)q.tile * a.T + tb + r) * a.B + q.b) * 2 * a.N + s0 + j;
                o[0] = outB;
                o[a.N] = outC;
            }
            if (Q > 1) __builtin_amdgcn_sched_barrier(0);  // one pass's registers at a time
            }
        }
        Bm -= TT * (int64_t)a.B_st;
        Cm -= TT * (int64_t)a.C_st;
        __syncthreads();
        if constexpr (!FIRST) {
#pragma unroll
            for (int k = 0; k < KT; ++k) {
                const int r = w + NW * k;
                if (r >= left) continue;
                float gb = 0.f, gs = 0.f;
#pragma unroll
                for (int i = 0; i < NW; ++i) {
                    gb += part[1][i][r][lane];
                    gs += part[2][i][r][lane];
                }
                const float gy = sg[r][lane];
                float ds = fmaf(ku[k], gb, gs * kLn2);
                if (a.softplus) ds *= seq_sigmoid(kx[k]);
                const int64_t o = (int64_t)tb * a.B * a.D + (int64_t)q.b * a.D + c0;
                if (q.ok) {
                    put(static_cast<E*>(a.du) + o, oo.off[k], f_elem<E>(fmaf(ks[k], gb, Dp * gy)));
                    put(static_cast<E*>(a.ddt) + o, oo.off[k], f_elem<E>(ds));
                }
                dbias += ds;
                dDp = fmaf(gy, ku[k], dDp);
                if (gate) {
                    float y = Dp * ku[k];
#pragma unroll
                    for (int i = 0; i < NW; ++i) y += part[0][i][r][lane];
                    const float sig = seq_sigmoid(kz[k]);
                    const float dz = ky[k] * y * fmaf(kz[k] * sig, 1.f - sig, sig);
                    if (q.ok) put(static_cast<E*>(a.dz) + o, oo.off[k], f_elem<E>(dz));
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
        const int64_t o = ((int64_t)t * a.B + q.b) * a.D + c0;
        (static_cast<E*>(a.du) + o)[q.lo] = (E)0.f;
        (static_cast<E*>(a.ddt) + o)[q.lo] = (E)0.f;
        if (gate) (static_cast<E*>(a.dz) + o)[q.lo] = (E)0.f;
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
    // (rows of a tile are addressed by 32-bit byte offsets)
    for (int64_t st : {a->u_st, a->dt_st, a->z_st, a->y_st, a->dy_st, a->B_st, a->C_st, (int64_t)a->B * a->D})
        SV_REQUIRE(st >= 0 && st * elem_bytes(a->dtype) < (int64_t)1 << 28, "%s: rows %lld elements apart, less than 2^28 bytes are supported", who, (long long)st);
    return SHIVAE_OK;
}

// Pieces of the time axis.  A split costs the second launch's work again without y (about 0.9 of it), so it is taken only
// where the unsplit grid leaves at least half of the card's SIMDs with one wave: then pieces of at least 64 rows until there are
// about 1024 workgroups.
static void ssm_split(SsmP& p) {
    const shivae_ssm_args& a = p.a;
    p.E = a.D / a.G;
    p.tiles_g = ceil_div(p.E, 64);
    p.tiles = p.tiles_g * a.G;
    const int64_t groups = (int64_t)p.tiles * a.B;
    int64_t np = 1;
    if (groups <= 256) np = std::min<int64_t>({1024 / groups, 32, ceil_div(a.T, 64)});
    p.plen = np > 1 ? round_up(ceil_div(a.T, (int)np), TT) : round_up(a.T, TT);
    p.np = ceil_div(a.T, p.plen);
}
// May a lane read its S states of a row of B or C at once?
static void ssm_vec(SsmP& p, int S) {
    const shivae_ssm_args& a = p.a;
    p.vec = a.N % S == 0 && aligned_to(a.Bm, 16) && aligned_to(a.Cm, 16);
    for (int64_t st : {a.B_st, a.B_sb, a.B_sg, a.C_st, a.C_sb, a.C_sg}) p.vec = p.vec && st % S == 0;
}

static size_t piece_floats(const SsmP& p) { return p.np > 1 ? (size_t)p.np * p.a.B * (p.a.N + 1) * p.a.D : 0; }
static bool a_token(const SsmP& p) { return p.a.T == 1 && !p.a.ckpt; }

template <class E>
static void launch_ssm_fwd(SsmP& p, bool first, int pieces, hipStream_t s) {
    const dim3 grid((unsigned)((int64_t)p.tiles * p.a.B * pieces));
#define SV_SSM(S)                                                                                   \
    if (first) hipLaunchKernelGGL((ssm_fwd_kernel<E, S, true>), grid, dim3(256), 0, s, p);      \
    else hipLaunchKernelGGL((ssm_fwd_kernel<E, S, false>), grid, dim3(256), 0, s, p)
    const int N = p.a.N;
    ssm_vec(p, N <= 4 ? 1 : N <= 8 ? 2 : N <= 16 ? 4 : N <= 32 ? 8 : 16);
    if (N <= 4) { SV_SSM(1); }
    else if (N <= 8) { SV_SSM(2); }
    else if (N <= 16) { SV_SSM(4); }
    else if (N <= 32) { SV_SSM(8); }
    else { SV_SSM(16); }
#undef SV_SSM
}

template <class E>
static void launch_ssm_bwd(SsmP& p, bool first, hipStream_t s) {
    const dim3 grid((unsigned)((int64_t)p.tiles * p.a.B * p.np));
#define SV_SSM(S, Q)                                                                                  \
    if (first) hipLaunchKernelGGL((ssm_bwd_kernel<E, S, Q, true>), grid, dim3(256), 0, s, p);         \
    else hipLaunchKernelGGL((ssm_bwd_kernel<E, S, Q, false>), grid, dim3(256), 0, s, p)
    const int N = p.a.N;
    ssm_vec(p, N <= 8 ? 2 : 4);
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
    ssm_split(p);
    return a_token(p) ? 0 : piece_floats(p) * sizeof(float);
}

int shivae_selective_scan_fwd(const shivae_ssm_args* args, void* ws_dev, size_t ws_bytes, shivae_stream stream) {
    SV_TRY(ssm_check(args, "selective_scan_fwd"));
    SsmP p{*args};
    const shivae_ssm_args& a = p.a;
    SV_REQUIRE(a.y, "selective_scan_fwd: y is required");
    SV_REQUIRE(!a.state || a.state != a.state_out || a.T <= TT, "selective_scan_fwd: the state can be updated in place for up to %d rows only", TT);
    ssm_split(p);
    SV_REQUIRE((int64_t)p.tiles * a.B * p.np < (int64_t)1 << 31, "selective_scan_fwd: B * D is too large");
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (a_token(p)) {
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
    SV_REQUIRE(need == 0 || (ws_dev && ws_bytes >= need && aligned_to(ws_dev, 16)), "selective_scan_fwd: a 16-byte aligned workspace of %zu bytes is needed, not %zu", need, ws_bytes);
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
    ssm_split(p);
    return bwd_floats(p) * sizeof(float);
}

int shivae_selective_scan_bwd(const shivae_ssm_args* args, void* ws_dev, size_t ws_bytes, shivae_stream stream) {
    SV_TRY(ssm_check(args, "selective_scan_bwd"));
    SsmP p{*args};
    const shivae_ssm_args& a = p.a;
    SV_REQUIRE(a.dy && a.du && a.ddt && a.dB && a.dC && a.dA && a.ckpt, "selective_scan_bwd: dy, du, ddt, dB, dC, dA and the forward's ckpt are required");
    SV_REQUIRE((!a.z || a.dz) && (!a.Dp || a.dDp) && (!a.dt_bias || a.ddt_bias), "selective_scan_bwd: z, Dp and dt_bias need buffers for their gradients");
    ssm_split(p);
    SV_REQUIRE((int64_t)p.tiles * a.B * p.np < (int64_t)1 << 31, "selective_scan_bwd: B * D is too large");
    const size_t need = bwd_floats(p) * sizeof(float);
    SV_REQUIRE(ws_dev && ws_bytes >= need && aligned_to(ws_dev, 16), "selective_scan_bwd: a 16-byte aligned workspace of %zu bytes is needed, not %zu", need, ws_bytes);
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
