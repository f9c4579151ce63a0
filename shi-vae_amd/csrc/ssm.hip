// Selective state-space scan, forward, backward and single token:
//   s = softplus(dt + dt_bias), a[n] = exp(s A[n]), h[n] = a[n] h[n] + s u B[n], y = (sum_n C[n] h[n] + Dp u) silu(z)
// Backward, with g[n] = dL/dh[n] running from the last row to the first and dy' = dy silu(z):
//   g[n] = C[n] dy' + (a g)[n] of the next row;  dC[n] = sum_d dy' h[n];  dB[n] = sum_d g[n] s u
//   ds = sum_n (a g)[n] h_prev[n] A[n] + u sum_n g[n] B[n];  du = s sum_n g[n] B[n] + Dp dy';  dA[n] = sum_t (a g)[n] h_prev[n] s
// A is general (one number per channel and state), so the recurrence is element-wise in (d, n) and has no matrix form: one exponential,
// two products and two fused multiply-adds per (row, channel, state).  Measured here a vector instruction of a wave takes 4 cycles, an
// exponential 8, so the forward pass of 16 states is 16 * 24 = 384 cycles per row and 64 channels, softplus and the gate about 100 more:
// at most 325 G (row, channel) pairs a second on the whole card, 2.6 TB/s of bf16 traffic.  Bound by vector instructions, not by memory.
//
// Layout: lane = (state group, channel): a wave owns 16 neighbouring channels and all their states, a workgroup 64 channels of a sequence
// (one cache line of bf16).  Rows come in tiles of 16, requested a tile ahead.  Where B * D is small the time axis is split into pieces: a
// first launch runs each piece from a zero state and keeps its last state and sum of s; since prod_t exp(s_t A) = exp(A sum_t s_t), a piece
// of the second launch gets its first state from those of the pieces in front of it (backward: the adjoint from those behind).
// Measured (MI355X, us a call, GPU time of captured calls): T 2048, B 16, D 2048, N 16, bf16, gate: 328 (1.65 TB/s); at B 64 1057, 254 G
// pairs a second, 0.78 of the bound: at B 16 a SIMD has two waves, whose dependent exponentials are not covered.  T 8192, B 1: 139 in 32
// pieces; in 16 pieces 151.  With 32 and 64 states: 502 and 1004; T 8192, B 1 with 64 539.
// Earlier forms of the same kernel, at B 16: 64 channels a wave and the states over four waves, s, B and C from LDS: 404 (64 of its 96 LDS
// cycles per row were broadcasts of B and C); B and C by scalar loads: 757; by row_newbcast: 415; waves that share nothing: 350.
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

// A log2(e), infinities made finite: an A of -inf (no memory) has to give exp(0 A) = 1 behind a sequence's end, and 0 where a step is
// positive.  A NaN stays one (v_maximum3_f32; fminf and fmaxf return the other operand).
__device__ __forceinline__ float scale_A(float A) { return __builtin_elementwise_minimum(__builtin_elementwise_maximum(A * kLog2e, -3.4e38f), 3.4e38f); }

// 2^x v + add, where 2^x alone may leave the range of fp32: x is the sum of a piece's log2 decays, and decays that grow (s A > 0) take a
// state of 0, or a small one, through a piece without ever leaving the range.
__device__ __forceinline__ float decay_add(float x, float v, float add) {
    const float k = fabsf(x) <= 126.f ? 0.f : rintf(fminf(fmaxf(x, -1e4f), 1e4f)), f = __builtin_elementwise_minimum(x, 1e4f) - k;
    return fmaf(__builtin_amdgcn_exp2f(f), __builtin_amdgcn_ldexpf(v, (int)k), add);
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

// (Whole words, so that the compiler does not merge the wide load with the element loads of the other branch into element loads.)
template <int BYTES>
struct Words {
    typedef unsigned T __attribute__((ext_vector_type(BYTES >= 16 ? 4 : BYTES / 4)));
    static constexpr int n = BYTES >= 16 ? BYTES / 16 : 1;
    T v[n];
};
template <>
struct Words<2> {
    unsigned short v[1];
};
// What a lane needs of B or C for a tile: S states of row (lane mod 16), as loaded.
template <class E, int S>
struct RowRegs {
    Pack<E, S> e;
    // base: the tile's row 0 of this group's matrix; s0: first state; left: rows from there to the sequence's end
    __device__ __forceinline__ void load(const E* base, unsigned stb, int s0, int N, bool vec, int left, int lane) {
        const unsigned off = (unsigned)min(lane & 15, left - 1) * stb;
        if (vec) {
            using W = Words<S * sizeof(E)>;
            const W w = *reinterpret_cast<const W*>(reinterpret_cast<const char*>(base) + (off + (unsigned)(min(s0, N - S) * sizeof(E))));
            __builtin_memcpy(&e, &w, sizeof(e));
        } else {
#pragma unroll
            for (int j = 0; j < S; ++j) e.v[j] = at(base, off + (unsigned)(min(s0 + j, N - 1) * sizeof(E)));
        }
    }
    // as fp32; rows at and behind `left` and states at and behind N are 0
    __device__ __forceinline__ void get(float (&v)[S], int s0, int N, int left, int lane) const {
#pragma unroll
        for (int j = 0; j < S; ++j) v[j] = elem_f(e.v[j]);
        if (left >= TT && N % (4 * S) == 0) return;  // (a whole tile of whole states: uniform, and the usual case)
#pragma unroll
        for (int j = 0; j < S; ++j) v[j] = (lane & 15) < left && s0 + j < N ? v[j] : 0.f;
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
// The sums over the four state groups of four rows' parts, row i in lane row i.  The swaps read a VGPR two wait states after a vector
// instruction wrote it at the earliest, and the compiler does not see the last instruction of row_dot's assembly (S >= 4).
template <int S>
__device__ __forceinline__ float sum_groups(float (&v)[4]) {
    if constexpr (S >= 4) asm("s_nop 1" : "+v"(v[0]), "+v"(v[1]), "+v"(v[2]), "+v"(v[3]));
    return swap16_add(swap32_add(v[0], v[2]), swap32_add(v[1], v[3]));
}
template <int N, class F>
__device__ __forceinline__ void unroll(F f) {  // f(0), f(1), ... with the number as a constant
    [&]<int... I>(std::integer_sequence<int, I...>) { (f(std::integral_constant<int, I>{}), ...); }(std::make_integer_sequence<int, N>{});
}

// What the pieces hand on to each other, S states of a lane's channel at a time (states at and behind N are read as the last one).
template <int S>
struct PieceStates {
    const SsmP& p;
    const float *hend, *ssum;  // of this sequence and channel
    int s0;
    __device__ __forceinline__ PieceStates(const SsmP& p, const Place& q, int s0)
        : p(p), hend(p.hend + (int64_t)q.b * p.a.N * p.a.D + q.d), ssum(p.ssum + (int64_t)q.b * p.a.D + q.d), s0(s0) {}
    __device__ __forceinline__ const float* state(int c, int j) const { return hend + ((int64_t)c * p.a.B * p.a.N + min(s0 + j, p.a.N - 1)) * p.a.D; }
    __device__ __forceinline__ void load(float (&v)[S], int c) const {
#pragma unroll
        for (int j = 0; j < S; ++j) v[j] = *state(c, j);
    }
    // v through piece c: prod_t exp(s_t A) = exp(A sum_t s_t), and what the piece itself left.
    __device__ __forceinline__ void pass(float (&v)[S], const float (&A2)[S], int c) const {
        const float sum = ssum[(int64_t)c * p.a.B * p.a.D];
#pragma unroll
        for (int j = 0; j < S; ++j) v[j] = decay_add(A2[j] * sum, v[j], *state(c, j));
    }
    __device__ __forceinline__ void clear(float (&v)[S], bool ok) const {
#pragma unroll
        for (int j = 0; j < S; ++j) v[j] = ok && s0 + j < p.a.N ? v[j] : 0.f;
    }
};

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
    const int pieces = (n + p.plen - 1) / p.plen;  // that hold rows of the sequence

    float h[S], A2[S];
#pragma unroll
    for (int j = 0; j < S; ++j) {
        const bool live = q.ok && g4 * S + j < a.N;
        const int64_t o = state0 + (int64_t)j * a.D;
        A2[j] = live ? scale_A(a.A[(int64_t)(g4 * S + j) * a.D + q.d]) : 0.f;
        h[j] = live && q.piece == 0 && a.state ? a.state[o] : 0.f;
    }
    if (!FIRST && q.piece) {
        PieceStates<S> in(p, q, g4 * S);
        in.load(h, 0);
        for (int c = 1; c < min(q.piece, pieces); ++c) in.pass(h, A2, c);
        in.clear(h, q.ok);
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
    float total = 0.f, ku[4], kz[4], vB[S], vC[S];
    // A tile's operands as the rows below take them, from what request() loaded.
    auto prepare = [&](int left) {
        float s[4];
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
        float su[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) su[k] = s[k] * ku[k];
        if (left < TT)  // rows behind the sequence leave the state as it is
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const bool in = 4 * k + g4 < left;
                s[k] = in ? s[k] : 0.f;
                su[k] = in ? su[k] : 0.f;
            }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (FIRST) total += s[k];
            row[4 * k + g4][lane & 15] = make_float2(s[k], su[k]);
        }
        nB.get(vB, g4 * S, a.N, left, lane);
        if (!FIRST) nC.get(vC, g4 * S, a.N, left, lane);
    };
    int left = tn - t0;  // rows from the present tile's first one
    float* ckpt = a.ckpt && !FIRST ? a.ckpt + (int64_t)(t0 / TT) * statep + state0 : nullptr;
    if (left > 0) {
        request(left);
        prepare(left);
        if (left > TT) request(left - TT);
    }
    for (; left > 0; left -= TT) {
        float2 x[TT];
#pragma unroll
        for (int r = 0; r < TT; ++r) x[r] = row[r][lane & 15];
        if (ckpt) {
#pragma unroll
            for (int j = 0; j < S; ++j)
                if (q.ok && g4 * S + j < a.N) ckpt[(int64_t)j * a.D] = h[j];
            ckpt += statep;
        }
        float v[4], pz[4];
        unroll<4>([&](auto K) {
            constexpr int k = K;
            float acc[4];
            unroll<4>([&](auto I) {
                constexpr int i = I, r = 4 * k + i;
#pragma unroll
                for (int j = 0; j < S; ++j) h[j] = fmaf(__builtin_amdgcn_exp2f(x[r].x * A2[j]), h[j], row_of<r>(vB[j]) * x[r].y);
                if constexpr (!FIRST) acc[i] = row_dot<r>(vC, h);
            });
            if constexpr (!FIRST) v[k] = fmaf(Dp, ku[k], sum_groups<S>(acc));
            pz[k] = kz[k];
        });
        // The next tile is taken over in front of this one's stores: stores and loads share a counter that is waited for in order.
        if (left > TT) prepare(left - TT);
        if constexpr (!FIRST) {
            if (gate)
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] *= pz[k] * seq_sigmoid(pz[k]);
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
        if (left > 2 * TT) request(left - 2 * TT);
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
// once, 16 bytes a lane, and is nearly all of the traffic: B 256, D 2048, N 16, bf16: 17 us for 67 MB of it, 3.9 TB/s; with 64 states 52.
// Channels that are not 16-byte aligned, one a thread, cost nothing: slices 8 bytes off 16 us, D 2046 17.
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
                h.v[c] = fmaf(__builtin_amdgcn_exp2f(s[c] * scale_A(A.v[c])), h.v[c], s[c] * u[c] * Bn);
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

// The adjoint of a piece's last state: the gradient of state_out for the last piece, otherwise what the pieces behind it hand down (those
// behind the sequence's end what they get).
template <int S>
__device__ __forceinline__ void piece_adjoints(const SsmP& p, const Place& q, int n, int s0, const float (&A2)[S], float (&v)[S]) {
    const shivae_ssm_args& a = p.a;
    PieceStates<S> in(p, q, s0);
    if (q.piece == p.np - 1) {
#pragma unroll
        for (int j = 0; j < S; ++j) v[j] = a.dstate_out ? a.dstate_out[((int64_t)q.b * a.N + min(s0 + j, a.N - 1)) * a.D + q.d] : 0.f;
    } else {
        in.load(v, p.np - 1);
        for (int c = min(p.np - 1, (n + p.plen - 1) / p.plen) - 1; c > q.piece; --c) in.pass(v, A2, c);
    }
    in.clear(v, q.ok);
}

// The operands of the backward kernels: 16-row tiles from a piece's last to its first, requested a tile ahead.
template <class E, bool FIRST>
struct BwdRows {
    const E *u, *dt, *z, *dy;
    E ru[4], rd[4], rz[4], rg[4];
    bool gate;
    __device__ __forceinline__ BwdRows(const shivae_ssm_args& a, const Place& q, int64_t last) {
        u = static_cast<const E*>(a.u) + (int64_t)q.b * a.u_sb + q.d0 + last * a.u_st;
        dt = static_cast<const E*>(a.dt) + (int64_t)q.b * a.dt_sb + q.d0 + last * a.dt_st;
        z = static_cast<const E*>(a.z) + (int64_t)q.b * a.z_sb + q.d0 + last * a.z_st;
        dy = static_cast<const E*>(a.dy) + (int64_t)q.b * a.dy_sb + q.d0 + last * a.dy_st;
        gate = a.z != nullptr;
    }
    __device__ __forceinline__ void request(const shivae_ssm_args& a, int g4, unsigned lo, int left) {
        const unsigned le = lo * (unsigned)sizeof(E);
        TileRows o;
        if (!FIRST) {
            o.set((unsigned)a.u_st * sizeof(E), g4, le, left);
            o.load(ru, u);
            u -= TT * a.u_st;
        }
        o.set((unsigned)a.dt_st * sizeof(E), g4, le, left);
        o.load(rd, dt);
        dt -= TT * a.dt_st;
        o.set((unsigned)a.dy_st * sizeof(E), g4, le, left);
        o.load(rg, dy);
        dy -= TT * a.dy_st;
        if (gate) {
            o.set((unsigned)a.z_st * sizeof(E), g4, le, left);
            o.load(rz, z);
            z -= TT * a.z_st;
        }
    }
};

// What each piece hands to the one in front of it: (a g) at its first row, from nothing behind (the last piece: from dstate_out).
template <class E, int S>
__global__ __launch_bounds__(256) void ssm_bwd_first_kernel(SsmP p) {
    __shared__ float2 rows_s[4][TT][16];
    const shivae_ssm_args& a = p.a;
    const int lane = threadIdx.x & 63, g4 = lane >> 4;
    float2 (&row)[TT][16] = rows_s[threadIdx.x >> 6];  // this wave's own: s, dy'
    Place q = ssm_place(p, (int)(threadIdx.x >> 6) * 16 + (lane & 15));
    if (!__any(q.ok)) return;
    q.piece += 1;  // (nothing is in front of the first piece)
    const int n = ssm_len(p, q.b), t0 = q.piece * p.plen, t1 = min(a.T, t0 + p.plen), tn = min(t1, n);
    float ag[S], A2[S];
#pragma unroll
    for (int j = 0; j < S; ++j) {
        const bool live = q.ok && g4 * S + j < a.N;
        A2[j] = live ? scale_A(a.A[(int64_t)(g4 * S + j) * a.D + q.d]) : 0.f;
        ag[j] = live && q.piece == p.np - 1 && a.dstate_out ? a.dstate_out[((int64_t)q.b * a.N + g4 * S + j) * a.D + q.d] : 0.f;
    }
    const float bias = a.dt_bias ? a.dt_bias[q.d] : 0.f;
    const int64_t last = t0 < tn ? (tn - 1) / TT * TT : t0;
    const E* Cm = static_cast<const E*>(a.Cm) + (int64_t)q.b * a.C_sb + (int64_t)q.g * a.C_sg + last * a.C_st;
    const unsigned Cs = (unsigned)a.C_st * sizeof(E);
    BwdRows<E, true> in(a, q, last);
    RowRegs<E, S> nC;
    float total = 0.f;
    int left = tn - (int)last;
    if (left > 0) {
        in.request(a, g4, q.lo, min(left, TT));
        nC.load(Cm, Cs, g4 * S, a.N, p.vec, left, lane);
    }
    for (int64_t tb = last; tb >= t0 && t0 < tn; tb -= TT, left = TT) {
        float s[4], gy[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            s[k] = elem_f(in.rd[k]) + bias;
            gy[k] = elem_f(in.rg[k]);
        }
        if (a.softplus)
#pragma unroll
            for (int k = 0; k < 4; ++k) s[k] = seq_softplus(s[k]);
        if (in.gate)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float z = elem_f(in.rz[k]);
                gy[k] *= z * seq_sigmoid(z);
            }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const bool on = 4 * k + g4 < left;
            s[k] = on ? s[k] : 0.f;
            total += s[k];
            row[4 * k + g4][lane & 15] = make_float2(s[k], on ? gy[k] : 0.f);
        }
        float vC[S];
        nC.get(vC, g4 * S, a.N, left, lane);
        if (tb > t0) {
            in.request(a, g4, q.lo, TT);
            Cm -= TT * a.C_st;
            nC.load(Cm, Cs, g4 * S, a.N, p.vec, TT, lane);
        }
        float2 x[TT];
#pragma unroll
        for (int r = 0; r < TT; ++r) x[r] = row[r][lane & 15];
        auto run = [&](auto whole) {
            unroll<TT>([&](auto I) {
                constexpr int r = TT - 1 - I;
#pragma unroll
                for (int j = 0; j < S; ++j) {
                    const float v = __builtin_amdgcn_exp2f(x[r].x * A2[j]) * (ag[j] + row_of<r>(vC[j]) * x[r].y);
                    ag[j] = whole || r < left ? v : ag[j];  // (behind the sequence's end exp(0 A) is no 1 where A is NaN)
                }
            });
        };
        if (left >= TT) run(std::true_type{});
        else run(std::false_type{});
    }
#pragma unroll
    for (int j = 0; j < S; ++j)
        if (q.ok && g4 * S + j < a.N) p.hend[(((int64_t)q.piece * a.B + q.b) * a.N + g4 * S + j) * a.D + q.d] = ag[j];
    total = swap32_add(total, total);
    total = swap16_add(total, total);
    if (q.ok && g4 == 0) p.ssum[((int64_t)q.piece * a.B + q.b) * a.D + q.d] = total;
}

// Sums over the 16 channels of a wave, for 16 rows at once.  Two rows' values are merged into one register while the lanes that still hold
// different channels' parts halve, four times; lane l of each 16-lane row ends with row bitrev4(l)'s sum, after 33 instructions for 16
// values.  Steps 1 and 2 (partner lane ^ 8, then mirrored in 8 lanes) write half of the banks from each of the two; steps 3 and 4 (^ 2, ^ 1)
// need a selection.
template <int S>
struct Sums {
    float b[S], c[S];
};
#define SV_MERGE(NAME, HOW, LO, HI)                                                                                        \
    template <int S>                                                                                                       \
    __device__ __forceinline__ void NAME(float (&o)[S], const float (&l)[S], const float (&h)[S]) {                        \
        if constexpr (S == 4)                                                                                              \
            asm("s_nop 1\n\t"                                                                                              \
                "v_add_f32_dpp %0, %4, %4 " HOW " row_mask:0xf bank_mask:" LO "\n\t"                                       \
                "v_add_f32_dpp %1, %5, %5 " HOW " row_mask:0xf bank_mask:" LO "\n\t"                                       \
                "v_add_f32_dpp %2, %6, %6 " HOW " row_mask:0xf bank_mask:" LO "\n\t"                                       \
                "v_add_f32_dpp %3, %7, %7 " HOW " row_mask:0xf bank_mask:" LO "\n\t"                                       \
                "v_add_f32_dpp %0, %8, %8 " HOW " row_mask:0xf bank_mask:" HI "\n\t"                                       \
                "v_add_f32_dpp %1, %9, %9 " HOW " row_mask:0xf bank_mask:" HI "\n\t"                                       \
                "v_add_f32_dpp %2, %10, %10 " HOW " row_mask:0xf bank_mask:" HI "\n\t"                                     \
                "v_add_f32_dpp %3, %11, %11 " HOW " row_mask:0xf bank_mask:" HI                                            \
                : "=&v"(o[0]), "=&v"(o[1]), "=&v"(o[2]), "=&v"(o[3])                                                       \
                : "v"(l[0]), "v"(l[1]), "v"(l[2]), "v"(l[3]), "v"(h[0]), "v"(h[1]), "v"(h[2]), "v"(h[3]));                 \
        else                                                                                                               \
            for (int j = 0; j < S; ++j)                                                                                    \
                asm("s_nop 1\n\t"                                                                                          \
                    "v_add_f32_dpp %0, %1, %1 " HOW " row_mask:0xf bank_mask:" LO "\n\t"                                   \
                    "v_add_f32_dpp %0, %2, %2 " HOW " row_mask:0xf bank_mask:" HI                                          \
                    : "=&v"(o[j]) : "v"(l[j]), "v"(h[j]));                                                                 \
    }
SV_MERGE(merge8, "row_ror:8", "0x3", "0xc")
SV_MERGE(merge4, "row_half_mirror", "0x5", "0xa")
#undef SV_MERGE
template <int CTRL>
__device__ __forceinline__ float merge_quad(float lo, float hi, bool upper) {  // upper: this lane keeps hi
    const float x = upper ? hi : lo, y = upper ? lo : hi;
    return x + __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(y), CTRL, 0xf, 0xf, true));
}
template <int LEVEL, int S>
__device__ __forceinline__ Sums<S> merge_rows(const Sums<S>& lo, const Sums<S>& hi, int lane) {
    Sums<S> o;
    if constexpr (LEVEL == 1) {
        merge8(o.b, lo.b, hi.b);
        merge8(o.c, lo.c, hi.c);
    } else if constexpr (LEVEL == 2) {
        merge4(o.b, lo.b, hi.b);
        merge4(o.c, lo.c, hi.c);
    } else {
        constexpr int ctrl = LEVEL == 3 ? 0x4e : 0xb1;  // quad_perm 2 3 0 1, 1 0 3 2
        const bool upper = lane & (LEVEL == 3 ? 2 : 1);
#pragma unroll
        for (int j = 0; j < S; ++j) {
            o.b[j] = merge_quad<ctrl>(lo.b[j], hi.b[j], upper);
            o.c[j] = merge_quad<ctrl>(lo.c[j], hi.c[j], upper);
        }
    }
    return o;
}
// f(row) for rows base + 2^LEVEL - 1 down to base, merged
template <int LEVEL, int S, int BASE, class F>
__device__ __forceinline__ Sums<S> sum_rows(F& f, int lane) {
    if constexpr (LEVEL == 0) return f(std::integral_constant<int, BASE>{});
    else {
        const Sums<S> hi = sum_rows<LEVEL - 1, S, BASE + (1 << (LEVEL - 1))>(f, lane);
        const Sums<S> lo = sum_rows<LEVEL - 1, S, BASE>(f, lane);
        return merge_rows<LEVEL>(lo, hi, lane);
    }
}

// The backward pass of a piece.  Lanes as in the forward kernel.  A tile's rows are run forward again from the checkpoint in front of it,
// with states and decays in registers (128 of them for S = 4), then back.  More than 16 states take several passes over a tile, 4 S
// states each, whose adjoints and sums wait in LDS.  dB and dC are sums over all channels: of the wave's 16 by sum_rows, of the
// workgroup's four waves through LDS (the one barrier of a pass), of the workgroups by ssm_dbc_kernel.
// Bound by vector instructions: 206 us (T 2048, B 4, D 1536, N 16, bf16, gate, 10 pieces), in which a SIMD issues 7.7e4 of them, 0.63 of its
// time; 222 us (T 1000, B 64, D 256, fp32).  The four passes around it: ssm_fwd_kernel 52 (FIRST) and 72, ssm_bwd_first_kernel 48,
// ssm_dbc_kernel 10 (all from a trace of 13 calls; a long run of calls takes 372 for all, 0.94 of their sum).  With 32 and 64 states, two
// and four passes over a tile: 777 and 1974 forward and backward.  The sums over channels by LDS atomics on floats instead (200 cycles each)
// took longer than all of the rest.
template <class E, int S, bool MANY>
__global__ __launch_bounds__(256, 2) void ssm_bwd_kernel(SsmP p) {
    constexpr int P = 4 * S;  // states of a pass
    __shared__ float2 rows_s[4][TT][16];
    __shared__ float rows_g[4][TT][16];
    // what the end of a tile needs again, out of the way of the 8 S TT registers in between: u, dt + bias, z, dy of a lane's four rows,
    // and the sums for y, g B and (a g) h_prev A
    __shared__ __attribute__((aligned(16))) float4 hold_s[4][4][64];
    __shared__ float sums_s[4][3][4][64];
    __shared__ __attribute__((aligned(16))) float part[2][4][TT][2][P];
    extern __shared__ __attribute__((aligned(16))) float kept[];  // [passes][3 S][256]: ag, A2, dA, where there are several passes
    const shivae_ssm_args& a = p.a;
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, g4 = lane >> 4, c16 = lane & 15;
    float2 (&row)[TT][16] = rows_s[wv];  // this wave's own: s, s u
    float (&rowg)[TT][16] = rows_g[wv];  // dy'
    float4 (&hold)[4][64] = hold_s[wv];
    float (&sum3)[3][4][64] = sums_s[wv];
    const Place q = ssm_place(p, wv * 16 + c16);
    const int n = ssm_len(p, q.b), t0 = q.piece * p.plen, t1 = min(a.T, t0 + p.plen), tn = min(t1, n);
    const int passes = MANY ? (a.N + P - 1) / P : 1;
    float ag[S], A2[S], dA[S];
    for (int k = 0; k < passes; ++k) {
#pragma unroll
        for (int j = 0; j < S; ++j) {
            const int s = k * P + g4 * S + j;
            const bool live = q.ok && s < a.N;
            A2[j] = live ? scale_A(a.A[(int64_t)s * a.D + q.d]) : 0.f;
            dA[j] = 0.f;
        }
        piece_adjoints<S>(p, q, n, k * P + g4 * S, A2, ag);
        if (MANY)
#pragma unroll
            for (int j = 0; j < S; ++j) {
                float* o = kept + (int64_t)k * 3 * S * 256 + threadIdx.x;
                o[j * 256] = ag[j];
                o[(S + j) * 256] = A2[j];
                o[(2 * S + j) * 256] = 0.f;
            }
    }
    const float bias = a.dt_bias ? a.dt_bias[q.d] : 0.f, Dp = a.Dp ? a.Dp[q.d] : 0.f;
    const int64_t last = t0 < tn ? (tn - 1) / TT * TT : t0, statep = (int64_t)a.B * a.N * a.D;
    const unsigned Bs = (unsigned)a.B_st * sizeof(E), Cs = (unsigned)a.C_st * sizeof(E);
    const E* Bm = static_cast<const E*>(a.Bm) + (int64_t)q.b * a.B_sb + (int64_t)q.g * a.B_sg;
    const E* Cm = static_cast<const E*>(a.Cm) + (int64_t)q.b * a.C_sb + (int64_t)q.g * a.C_sg;
    BwdRows<E, false> in(a, q, last);

    // B, C and the checkpoint of the next pass (of this tile or of the one in front of it)
    RowRegs<E, S> nB, nC;
    float nh[S];
    auto request_states = [&](int64_t tb, int pass, int left, int lane, int g4, unsigned lo) {
        nB.load(Bm + tb * a.B_st, Bs, pass * P + g4 * S, a.N, p.vec, left, lane);
        nC.load(Cm + tb * a.C_st, Cs, pass * P + g4 * S, a.N, p.vec, left, lane);
        const float* c = a.ckpt + tb / TT * statep + (int64_t)q.b * a.N * a.D + q.d0;
#pragma unroll
        for (int j = 0; j < S; ++j) nh[j] = at(c, (unsigned)min(pass * P + g4 * S + j, a.N - 1) * (unsigned)a.D * 4 + lo * 4);
    };
    float dDp = 0.f, dbias = 0.f;
    int left = tn - (int)last, buf = 0;
    if (left > 0) {
        in.request(a, g4, q.lo, min(left, TT));
        request_states(last, 0, left, lane, g4, q.lo);
    }
    for (int64_t tb = last; tb >= t0 && t0 < tn; tb -= TT, left = TT) {
        // Opaque once a tile, so that no address that follows from them is kept in registers over the loop.
        int lane = threadIdx.x & 63;
        unsigned lo = q.lo;
        asm volatile("" : "+v"(lane), "+v"(lo));
        const int g4 = lane >> 4, c16 = lane & 15;
        {
            float ku[4], kx[4], kz[4] = {}, ky[4], ks[4], kg[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                ku[k] = elem_f(in.ru[k]);
                kx[k] = ks[k] = elem_f(in.rd[k]) + bias;
                kg[k] = ky[k] = elem_f(in.rg[k]);
            }
            if (a.softplus)
#pragma unroll
                for (int k = 0; k < 4; ++k) ks[k] = seq_softplus(kx[k]);
            if (in.gate)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    kz[k] = elem_f(in.rz[k]);
                    kg[k] = ky[k] * (kz[k] * seq_sigmoid(kz[k]));
                }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const bool on = 4 * k + g4 < left && q.ok;  // (a lane without a channel adds nothing to dB and dC)
                ks[k] = on ? ks[k] : 0.f;
                row[4 * k + g4][c16] = make_float2(ks[k], on ? ks[k] * ku[k] : 0.f);
                rowg[4 * k + g4][c16] = on ? kg[k] : 0.f;
                hold[k][lane] = make_float4(ku[k], kx[k], kz[k], ky[k]);
            }
        }
        if (tb > t0) in.request(a, g4, lo, TT);
#pragma unroll 1
        for (int pass = 0; pass < passes; ++pass) {
            float* keep = kept + (int64_t)pass * 3 * S * 256 + threadIdx.x;
            if (MANY)
#pragma unroll
                for (int j = 0; j < S; ++j) {
                    ag[j] = keep[j * 256];
                    A2[j] = keep[(S + j) * 256];
                    dA[j] = keep[(2 * S + j) * 256];
                }
            float vB[S], vC[S], h0[S];
            nB.get(vB, pass * P + g4 * S, a.N, left, lane);
            nC.get(vC, pass * P + g4 * S, a.N, left, lane);
#pragma unroll
            for (int j = 0; j < S; ++j) h0[j] = q.ok && pass * P + g4 * S + j < a.N ? nh[j] : 0.f;
            if (pass + 1 < passes) request_states(tb, pass + 1, left, lane, g4, lo);
            else if (tb > t0) request_states(tb - TT, 0, TT, lane, g4, lo);
            float h[TT][S], e[TT][S];
            float2 x[TT];  // read from LDS four rows ahead of their use
#pragma unroll
            for (int r = 0; r < 4; ++r) x[r] = row[r][c16];
            unroll<4>([&](auto K) {
                constexpr int k = K;
                float acc[4];
                if constexpr (k < 3)
#pragma unroll
                    for (int i = 4; i < 8; ++i) x[4 * k + i] = row[4 * k + i][c16];
                unroll<4>([&](auto I) {
                    constexpr int i = I, r = 4 * k + i;
#pragma unroll
                    for (int j = 0; j < S; ++j) {
                        e[r][j] = __builtin_amdgcn_exp2f(x[r].x * A2[j]);
                        h[r][j] = fmaf(e[r][j], r ? h[r ? r - 1 : 0][j] : h0[j], row_of<r>(vB[j]) * x[r].y);
                    }
                    acc[i] = row_dot<r>(vC, h[r]);
                });
                const float y = sum_groups<S>(acc);
                sum3[0][k][lane] = MANY && pass ? sum3[0][k][lane] + y : y;
                __builtin_amdgcn_sched_barrier(0);  // (or the scheduler starts all rows at once and runs out of registers)
            });
            if (left < TT)  // (behind the sequence's end exp(0 A) is no 1 where A is NaN)
                unroll<TT>([&](auto R) {
                    constexpr int r = R;
                    if (r >= left)
#pragma unroll
                        for (int j = 0; j < S; ++j) e[r][j] = 1.f;
                });
            // Everything that the way back takes from LDS and from B and C is taken again: kept from the way there it would be 10 S + 32
            // registers that are not free.
            asm volatile("" ::: "memory");
#pragma unroll
            for (int j = 0; j < S; ++j) asm volatile("" : "+v"(vB[j]), "+v"(vC[j]), "+v"(A2[j]));
            float rb[4], rs[4], gyr[TT];
            float2 xr[TT];
#pragma unroll
            for (int r = TT - 4; r < TT; ++r) {
                xr[r] = row[r][c16];
                gyr[r] = rowg[r][c16];
            }
            auto back = [&](auto R) {
                constexpr int r = R, i = r & 3;
                if constexpr (i == 3 && r > 3)
#pragma unroll
                    for (int t = r - 7; t < r - 3; ++t) {
                        xr[t] = row[t][c16];
                        gyr[t] = rowg[t][c16];
                    }
                const float2 x = xr[r];
                const float gy = gyr[r];
                Sums<S> o;
                float g[S], gs = 0.f;
#pragma unroll
                for (int j = 0; j < S; ++j) {
                    g[j] = ag[j] + row_of<r>(vC[j]) * gy;
                    o.c[j] = gy * h[r][j];
                    o.b[j] = g[j] * x.y;
                    ag[j] = e[r][j] * g[j];
                    const float m = ag[j] * (r ? h[r ? r - 1 : 0][j] : h0[j]);
                    gs = fmaf(m, A2[j], gs);
                    dA[j] = fmaf(m, x.x, dA[j]);
                }
                rb[i] = row_dot<r>(vB, g);
                rs[i] = gs;
                if constexpr (i == 0) __builtin_amdgcn_sched_barrier(0);
                if constexpr (i == 0) {
                    const float gb = sum_groups<S>(rb);
                    const float gs4 = swap16_add(swap32_add(rs[0], rs[2]), swap32_add(rs[1], rs[3]));
                    sum3[1][r / 4][lane] = MANY && pass ? sum3[1][r / 4][lane] + gb : gb;
                    sum3[2][r / 4][lane] = MANY && pass ? sum3[2][r / 4][lane] + gs4 : gs4;
                }
                return o;
            };
            const Sums<S> sums = sum_rows<4, S, 0>(back, lane);
            const int rr = __brev((unsigned)c16) >> 28;
            *reinterpret_cast<Pack<float, S>*>(&part[buf][wv][rr][0][g4 * S]) = *reinterpret_cast<const Pack<float, S>*>(sums.b);
            *reinterpret_cast<Pack<float, S>*>(&part[buf][wv][rr][1][g4 * S]) = *reinterpret_cast<const Pack<float, S>*>(sums.c);
            if (MANY)
#pragma unroll
                for (int j = 0; j < S; ++j) {
                    keep[j * 256] = ag[j];
                    keep[(2 * S + j) * 256] = dA[j];
                }
            __syncthreads();
            for (int i = threadIdx.x; i < TT * 2 * P; i += 256) {
                const int r = i / (2 * P), kind = i / P & 1, s = i % P;
                const float v = (part[buf][0][r][kind][s] + part[buf][1][r][kind][s]) + (part[buf][2][r][kind][s] + part[buf][3][r][kind][s]);
                if (r < left && pass * P + s < a.N) p.pbc[((((int64_t)q.tile * a.T + tb + r) * a.B + q.b) * 2 + kind) * a.N + pass * P + s] = v;
            }
            buf ^= 1;  // (written again behind the next barrier's far side only)
        }
        E* const du = static_cast<E*>(a.du) + (tb * a.B + q.b) * a.D + q.d0;
        E* const ddt = static_cast<E*>(a.ddt) + (tb * a.B + q.b) * a.D + q.d0;
        float4 k4[4];  // u, dt + bias, z, dy
        float ks[4], kg[4], gb[4], ds[4];
        TileRows oo;
        oo.set((unsigned)((int64_t)a.B * a.D * sizeof(E)), g4, lo * (unsigned)sizeof(E));
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            k4[k] = hold[k][lane];
            ks[k] = row[4 * k + g4][c16].x;
            kg[k] = rowg[4 * k + g4][c16];
            gb[k] = sum3[1][k][lane];
            ds[k] = fmaf(k4[k].x, gb[k], sum3[2][k][lane] * kLn2);
        }
        if (a.softplus)
#pragma unroll
            for (int k = 0; k < 4; ++k) ds[k] *= seq_sigmoid(k4[k].y);
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (4 * k + g4 < left && q.ok) {
                put(du, oo.off[k], f_elem<E>(fmaf(ks[k], gb[k], Dp * kg[k])));
                put(ddt, oo.off[k], f_elem<E>(ds[k]));
                dbias += ds[k];
                dDp = fmaf(kg[k], k4[k].x, dDp);
            }
        if (in.gate) {
            E* const dz = static_cast<E*>(a.dz) + (tb * a.B + q.b) * a.D + q.d0;
            float v[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float sig = seq_sigmoid(k4[k].z);
                v[k] = k4[k].w * fmaf(Dp, k4[k].x, sum3[0][k][lane]) * fmaf(k4[k].z * sig, 1.f - sig, sig);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (4 * k + g4 < left && q.ok) put(dz, oo.off[k], f_elem<E>(v[k]));
        }
    }
    if (!q.ok) return;
    const int64_t pb = (int64_t)q.piece * a.B + q.b;
    dDp = swap32_add(dDp, dDp);
    dbias = swap32_add(dbias, dbias);
    dDp = swap16_add(dDp, dDp);
    dbias = swap16_add(dbias, dbias);
    if (g4 < 2) p.pD[(pb * 2 + g4) * a.D + q.d] = g4 ? dbias : dDp;
    for (int k = 0; k < passes; ++k)
#pragma unroll
        for (int j = 0; j < S; ++j) {
            const int s = k * P + g4 * S + j;
            if (s >= a.N) continue;
            const float* keep = kept + (int64_t)k * 3 * S * 256 + threadIdx.x;
            p.pA[(pb * a.N + s) * a.D + q.d] = MANY ? keep[(2 * S + j) * 256] : dA[j];
            if (q.piece == 0 && a.dstate) a.dstate[((int64_t)q.b * a.N + s) * a.D + q.d] = MANY ? keep[j * 256] : ag[j];
        }
    for (int t = max(t0, n) + g4; t < t1; t += 4) {
        const int64_t o = ((int64_t)t * a.B + q.b) * a.D + q.d;
        static_cast<E*>(a.du)[o] = (E)0.f;
        static_cast<E*>(a.ddt)[o] = (E)0.f;
        if (a.z) static_cast<E*>(a.dz)[o] = (E)0.f;
    }
}

// dB, dC = the sums of the channel tiles' parts, rounded once; 0 behind a sequence's last row.
template <class E>
__global__ __launch_bounds__(256) void ssm_dbc_kernel(SsmP p) {
    const shivae_ssm_args& a = p.a;
    const int64_t rows = (int64_t)a.T * a.B, total = rows * a.G * 2 * a.N;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int w2 = 2 * a.N, k = (int)(i % w2);
        const int64_t rg = i / w2, row = rg % rows;
        const int g = (int)(rg / rows), t = (int)(row / a.B), b = (int)(row - (int64_t)t * a.B);
        float v = 0.f;
        if (t < ssm_len(p, b))
            for (int c = 0; c < p.tiles_g; ++c) v += p.pbc[((int64_t)(g * p.tiles_g + c) * rows + row) * w2 + k];
        const bool isC = k >= a.N;
        static_cast<E*>(isC ? a.dC : a.dB)[(row * a.G + g) * a.N + (isC ? k - a.N : k)] = f_elem<E>(v);
    }
}

static int ssm_check(const shivae_ssm_args* a, const char* who) {
    SV_REQUIRE(a, "%s: null argument block", who);
    SV_REQUIRE(a->T > 0 && a->B > 0 && a->D > 0, "%s: T, B, D must be positive (%d, %d, %d)", who, a->T, a->B, a->D);
    SV_REQUIRE(a->N >= 1 && a->N <= 64, "%s: %d states per channel, 1..64 are supported", who, a->N);
    SV_REQUIRE(a->G >= 1 && a->D % a->G == 0, "%s: %d groups do not divide %d channels", who, a->G, a->D);
    SV_REQUIRE(a->dtype == SHIVAE_F32 || a->dtype == SHIVAE_BF16 || a->dtype == SHIVAE_F16, "%s: unknown dtype %d", who, a->dtype);
    SV_REQUIRE(a->T <= 1 << 30 && (int64_t)a->D * a->N <= 1 << 28, "%s: T or D * N is too large", who);
    SV_REQUIRE(a->u && a->dt && a->A && a->Bm && a->Cm, "%s: u, dt, A, B and C are required", who);
    // (rows of a tile are addressed by 32-bit byte offsets)
    for (int64_t st : {a->u_st, a->dt_st, a->z_st, a->y_st, a->dy_st, a->B_st, a->C_st, (int64_t)a->B * a->D})
        SV_REQUIRE(a->T == 1 || (st >= 0 && st * elem_bytes(a->dtype) < (int64_t)1 << 28), "%s: rows %lld elements apart, less than 2^28 bytes are supported", who, (long long)st);
    return SHIVAE_OK;
}

// Pieces of the time axis.  A split costs the second launch's work again without y (0.7 of it; backward a quarter), so it is taken only
// up to 256 workgroups, one wave a SIMD: then pieces of at least 64 rows until there are about 1024.  Measured (us, forward and backward
// together): T 1000, B 64, D 256, fp32, 256 workgroups: split 408, not 471; T 2048, B 4, D 1536, bf16, 96 workgroups: split 372, not 932.
// For 512 / 1024 / 1536 / 2048 workgroups (up to 64 pieces in the last): T 8192, B 1, D 2048 forward 151 / 139 / 141 / 154; the two above
// 417 / 408 / 396 / 397 and 390 / 372 / 357 / 372.
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
static void launch_ssm_bwd_first(SsmP& p, hipStream_t s) {
    const dim3 grid((unsigned)((int64_t)p.tiles * p.a.B * (p.np - 1)));
#define SV_SSM(S) hipLaunchKernelGGL((ssm_bwd_first_kernel<E, S>), grid, dim3(256), 0, s, p)
    const int N = p.a.N;
    ssm_vec(p, N <= 4 ? 1 : N <= 8 ? 2 : N <= 16 ? 4 : N <= 32 ? 8 : 16);
    if (N <= 4) SV_SSM(1);
    else if (N <= 8) SV_SSM(2);
    else if (N <= 16) SV_SSM(4);
    else if (N <= 32) SV_SSM(8);
    else SV_SSM(16);
#undef SV_SSM
}

template <class E>
static int launch_ssm_bwd(SsmP& p, hipStream_t s) {
    const dim3 grid((unsigned)((int64_t)p.tiles * p.a.B * p.np));
    const int N = p.a.N, S = N <= 4 ? 1 : N <= 8 ? 2 : 4, passes = ceil_div(N, 4 * S);
    constexpr size_t pass_lds = 3 * 4 * 256 * sizeof(float), most_lds = 4 * pass_lds;  // N <= 64: up to 48 KiB beside 57 of static
    const size_t lds = passes > 1 ? passes * pass_lds : 0;
    ssm_vec(p, S);
    if (lds)  // (past the default limit of 64 KiB; always to the most, since the limit is the function's and another thread may be between
              // here and its launch)
        SV_CHECK_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(ssm_bwd_kernel<E, 4, true>), hipFuncAttributeMaxDynamicSharedMemorySize, (int)most_lds));
    if (S == 1) hipLaunchKernelGGL((ssm_bwd_kernel<E, 1, false>), grid, dim3(256), 0, s, p);
    else if (S == 2) hipLaunchKernelGGL((ssm_bwd_kernel<E, 2, false>), grid, dim3(256), 0, s, p);
    else if (passes == 1) hipLaunchKernelGGL((ssm_bwd_kernel<E, 4, false>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((ssm_bwd_kernel<E, 4, true>), grid, dim3(256), lds, s, p);
    SV_CHECK_HIP(hipGetLastError());
    return SHIVAE_OK;
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
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (a_token(p)) {
        const int V = 4;
        const bool vec = p.E % V == 0 && a.u_sb % V == 0 && a.dt_sb % V == 0 && a.z_sb % V == 0 && a.y_sb % V == 0 && aligned_to(a.u, 16) && aligned_to(a.dt, 16) &&
                         aligned_to(a.z, 16) && aligned_to(a.y, 16) && aligned_to(a.A, 16) && aligned_to(a.state, 16) && aligned_to(a.state_out, 16);
        const int nvec = vec ? a.D / V : a.D;
        const int64_t blocks = ((int64_t)a.B * nvec + 255) / 256;
        SV_REQUIRE(grid_fits(blocks, 256), "selective_scan_fwd: B * D is too large (%d sequences of %d channel groups)", a.B, nvec);
        const dim3 grid((unsigned)blocks);
        SV_BY_DTYPE(a.dtype, {
            if (vec) hipLaunchKernelGGL((ssm_token_kernel<E, 4>), grid, dim3(256), 0, s, p, nvec);
            else hipLaunchKernelGGL((ssm_token_kernel<E, 1>), grid, dim3(256), 0, s, p, nvec);
        });
        SV_CHECK_HIP(hipGetLastError());
        return SHIVAE_OK;
    }
    SV_REQUIRE(grid_fits((int64_t)p.tiles * a.B * p.np, 256), "selective_scan_fwd: B * D is too large (%d sequences of %d tiles of 64 channels)", a.B, p.tiles);
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
    SV_REQUIRE(grid_fits((int64_t)p.tiles * a.B * p.np, 256), "selective_scan_bwd: B * D is too large (%d sequences of %d tiles of 64 channels)", a.B, p.tiles);
    const size_t need = bwd_floats(p) * sizeof(float);
    SV_REQUIRE(ws_dev && ws_bytes >= need && aligned_to(ws_dev, 16), "selective_scan_bwd: a 16-byte aligned workspace of %zu bytes is needed, not %zu", need, ws_bytes);
    hipStream_t s = static_cast<hipStream_t>(stream);
    p.hend = static_cast<float*>(ws_dev);
    p.ssum = p.hend + (p.np > 1 ? (size_t)p.np * a.B * a.N * a.D : 0);
    p.pbc = p.hend + piece_floats(p);
    p.pA = p.pbc + (size_t)p.tiles * a.T * a.B * 2 * a.N;
    p.pD = p.pA + (size_t)p.np * a.B * a.N * a.D;
    if (p.np > 1) SV_BY_DTYPE(a.dtype, launch_ssm_bwd_first<E>(p, s));
    SV_BY_DTYPE(a.dtype, SV_TRY(launch_ssm_bwd<E>(p, s)));
    SV_CHECK_HIP(hipGetLastError());
    const int64_t total = (int64_t)a.T * a.B * a.G * 2 * a.N;
    const dim3 grid((unsigned)std::min<int64_t>((total + 255) / 256, 1 << 22));
    SV_BY_DTYPE(a.dtype, hipLaunchKernelGGL((ssm_dbc_kernel<E>), grid, dim3(256), 0, s, p));
    SV_CHECK_HIP(hipGetLastError());
    float* mid = p.pD + (size_t)p.np * a.B * 2 * a.D;
    SV_TRY(launch_sum_parts(p.pA, (int64_t)p.np * a.B, a.N * a.D, mid, a.dA, a.N * a.D, nullptr, s));
    if (a.Dp || a.dt_bias) return launch_sum_parts(p.pD, (int64_t)p.np * a.B, 2 * a.D, mid, a.dDp, a.D, a.ddt_bias, s);
    return SHIVAE_OK;
}

}  // extern "C"
