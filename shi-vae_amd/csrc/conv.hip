// Short causal convolution over time, one filter per channel, with its activation:
//   xs = [state rows ; x rows],  pre[t] = bias + sum_j weight[j] xs[t+j],  y = silu(pre) or pre          (t >= length: 0)
//   g = dy act'(pre),  dxs[t+j] += weight[j] g[t],  dweight[j] = sum_t,b g[t] xs[t+j],  dbias = sum_t,b g
// Bound by memory traffic: 2 W + ~10 operations per element read and written.
//
// A thread owns one 16-byte group of channels of one sequence and a run of time steps, and keeps the window of the last
// W - 1 rows in registers, so that a row is read once per run (the W - 1 rows in front of a run are read again by the run
// behind them).  Neighbouring threads own neighbouring channels: every access is a contiguous 1 KiB per wave.
// Measured (W 4, silu): T 2048, B 16, D 2048, bf16 50 us, 5.4 TB/s, as fast as a copy; T 1000, B 64, D 256, fp32 18 us forward, 35 backward,
// and 2 x 5 for the partial sums.  Channels that are not 16-byte aligned are read one a thread: T 2048, B 16, D 2044 59 us, a slice of 2048
// 8 bytes off 60, D 2047 77.
#include <algorithm>

#include "common.h"
#include "elem.h"

namespace shivae {

struct ConvP {
    shivae_conv_args a;
    int nvec, run, nrun;  // channel groups per sequence, time steps per thread, runs
    float* part;          // backward: [nrun * B][W + 1][D] partial sums of dweight and dbias
};

__device__ __forceinline__ int seq_len(const int* lengths, int b, int T) {
    if (!lengths) return T;
    const int n = lengths[b];
    return n < 0 ? 0 : (n < T ? n : T);
}

template <class E, int V>
__device__ __forceinline__ void load_row(const E* p, float (&o)[V]) {
    const Pack<E, V> r = *reinterpret_cast<const Pack<E, V>*>(p);
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = elem_f(r.v[i]);
}
template <class E, int V>
__device__ __forceinline__ void store_row(E* p, const float (&v)[V]) {
    Pack<E, V> r;
#pragma unroll
    for (int i = 0; i < V; ++i) r.v[i] = f_elem<E>(v[i]);
    *reinterpret_cast<Pack<E, V>*>(p) = r;
}

// Row r of xs = [state ; x] for r < W - 1 + n: the state's rows come first, zeros where there is no state.
template <class E, int V, int W>
__device__ __forceinline__ void load_xs(const shivae_conv_args& a, int r, int b, int d, float (&o)[V]) {
    if (r >= W - 1) return load_row<E, V>(static_cast<const E*>(a.x) + (int64_t)(r - (W - 1)) * a.x_st + (int64_t)b * a.x_sb + d, o);
    if (a.state) return load_row<E, V>(static_cast<const E*>(a.state) + ((int64_t)r * a.B + b) * a.D + d, o);
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = 0.f;
}

template <class E, int V, int W>
__global__ __launch_bounds__(256) void conv_fwd_kernel(ConvP p) {
    const shivae_conv_args& a = p.a;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= (int64_t)a.B * p.nvec) return;
    const int b = (int)(i / p.nvec), d = (int)(i - (int64_t)b * p.nvec) * V;
    const int n = seq_len(a.lengths, b, a.T);
    const int t0 = blockIdx.y * p.run, t1 = min(a.T, t0 + p.run), tn = min(t1, n);
    float w[W][V], bias[V];
#pragma unroll
    for (int j = 0; j < W; ++j) load_row<float, V>(a.weight + (int64_t)j * a.D + d, w[j]);
    if (a.bias) load_row<float, V>(a.bias + d, bias);
    else
#pragma unroll
        for (int k = 0; k < V; ++k) bias[k] = 0.f;
    const E* x = static_cast<const E*>(a.x) + (int64_t)b * a.x_sb + d;
    E* y = static_cast<E*>(a.y) + (int64_t)b * a.y_sb + d;
    if (t0 < tn) {
        float win[W - 1][V];
#pragma unroll
        for (int j = 0; j < W - 1; ++j) load_xs<E, V, W>(a, t0 + j, b, d, win[j]);
        constexpr int U = 8;  // rows in flight per thread
        for (int t = t0; t < tn; t += U) {
            Pack<E, V> raw[U];
#pragma unroll
            for (int k = 0; k < U; ++k)
                if (t + k < tn) raw[k] = *reinterpret_cast<const Pack<E, V>*>(x + (int64_t)(t + k) * a.x_st);
#pragma unroll
            for (int k = 0; k < U; ++k) {
                if (t + k >= tn) break;
                float o[V];
#pragma unroll
                for (int c = 0; c < V; ++c) {
                    const float xv = elem_f(raw[k].v[c]);
                    float s = bias[c];
#pragma unroll
                    for (int j = 0; j < W - 1; ++j) s = fmaf(w[j][c], win[j][c], s);
                    s = fmaf(w[W - 1][c], xv, s);
                    o[c] = a.silu ? s * seq_sigmoid(s) : s;
#pragma unroll
                    for (int j = 0; j + 1 < W - 1; ++j) win[j][c] = win[j + 1][c];
                    win[W - 2][c] = xv;
                }
                store_row<E, V>(y + (int64_t)(t + k) * a.y_st, o);
            }
        }
    }
    const float zero[V] = {};
    for (int t = max(t0, n); t < t1; ++t) store_row<E, V>(y + (int64_t)t * a.y_st, zero);
    // The last W - 1 rows of xs.  state_out may be the state itself when there is one run: the thread has read the rows of
    // its window by now, and row j is written before only rows behind it are read.
    if (a.state_out && blockIdx.y == 0)
#pragma unroll
        for (int j = 0; j < W - 1; ++j) {
            float r[V];
            load_xs<E, V, W>(a, n + j, b, d, r);
            store_row<E, V>(static_cast<E*>(a.state_out) + ((int64_t)j * a.B + b) * a.D + d, r);
        }
}

// Rows r = t0 .. t1 + W - 2 of dy and x: g[r] needs x[r-W+1 .. r]; dx[r-W+1] needs g[r-W+1 .. r], so the run's last W - 1
// gradients come from the run behind it and are computed twice; dweight and dbias take the run's own rows only.  The first
// run also writes the rows in front of x, the state's gradient.  The gradient of state_out enters dx where the row lies.
template <class E, int V, int W>
__global__ __launch_bounds__(256) void conv_bwd_kernel(ConvP p) {
    const shivae_conv_args& a = p.a;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= (int64_t)a.B * p.nvec) return;
    const int b = (int)(i / p.nvec), d = (int)(i - (int64_t)b * p.nvec) * V;
    const int n = seq_len(a.lengths, b, a.T);
    const int t0 = blockIdx.y * p.run, t1 = min(a.T, t0 + p.run);
    float w[W][V], bias[V], dw[W][V], db[V], g[W][V], win[W][V];
#pragma unroll
    for (int j = 0; j < W; ++j) {
        load_row<float, V>(a.weight + (int64_t)j * a.D + d, w[j]);
#pragma unroll
        for (int c = 0; c < V; ++c) dw[j][c] = g[j][c] = win[j][c] = 0.f;
    }
    if (a.bias) load_row<float, V>(a.bias + d, bias);
#pragma unroll
    for (int c = 0; c < V; ++c) {
        db[c] = 0.f;
        if (!a.bias) bias[c] = 0.f;
    }
    const E* x = static_cast<const E*>(a.x) + (int64_t)b * a.x_sb + d;
    const E* dy = static_cast<const E*>(a.dy) + (int64_t)b * a.dy_sb + d;
    E* dx = static_cast<E*>(a.dx) + (int64_t)b * a.D + d;
    const int64_t rowlen = (int64_t)a.B * a.D;
    if (t0 < n) {
#pragma unroll
        for (int j = 0; j < W - 1; ++j) load_xs<E, V, W>(a, t0 + j, b, d, win[j + 1]);  // shifted down at the first row
    }
    const int rend = t1 + W - 1;
    constexpr int U = 4;
    for (int rb = t0; rb < rend; rb += U) {
        Pack<E, V> rx[U], rg[U];
#pragma unroll
        for (int k = 0; k < U; ++k)
            if (rb + k < rend && rb + k < n) {
                rx[k] = *reinterpret_cast<const Pack<E, V>*>(x + (int64_t)(rb + k) * a.x_st);
                rg[k] = *reinterpret_cast<const Pack<E, V>*>(dy + (int64_t)(rb + k) * a.dy_st);
            }
#pragma unroll
        for (int k = 0; k < U; ++k) {
            const int r = rb + k;
            if (r >= rend) break;
#pragma unroll
            for (int c = 0; c < V; ++c) {
#pragma unroll
                for (int j = 0; j + 1 < W; ++j) {
                    win[j][c] = win[j + 1][c];
                    g[j][c] = g[j + 1][c];
                }
                float gv = 0.f;
                if (r < n) {
                    win[W - 1][c] = elem_f(rx[k].v[c]);
                    gv = elem_f(rg[k].v[c]);
                    if (a.silu) {
                        float s = bias[c];
#pragma unroll
                        for (int j = 0; j < W; ++j) s = fmaf(w[j][c], win[j][c], s);
                        const float sg = seq_sigmoid(s);
                        gv *= fmaf(s * sg, 1.f - sg, sg);
                    }
                    if (r < t1) {
#pragma unroll
                        for (int j = 0; j < W; ++j) dw[j][c] = fmaf(gv, win[j][c], dw[j][c]);
                        db[c] += gv;
                    }
                }
                g[W - 1][c] = gv;
            }
            const int row = r - (W - 1);  // the row of x whose gradient is complete now (< 0: of the state)
            if (row < t0 && (blockIdx.y != 0 || !a.dstate)) continue;
            float o[V];
#pragma unroll
            for (int c = 0; c < V; ++c) {
                float s = 0.f;
#pragma unroll
                for (int j = 0; j < W; ++j) s = fmaf(w[j][c], g[W - 1 - j][c], s);
                o[c] = s;
            }
            const int so = row - (n - (W - 1));  // the row of state_out that this row of xs became
            if (a.dstate_out && so >= 0 && so < W - 1) {
                float e[V];
                load_row<E, V>(static_cast<const E*>(a.dstate_out) + ((int64_t)so * a.B + b) * a.D + d, e);
#pragma unroll
                for (int c = 0; c < V; ++c) o[c] += e[c];
            }
            if (row < 0) {
                store_row<E, V>(static_cast<E*>(a.dstate) + ((int64_t)(row + W - 1) * a.B + b) * a.D + d, o);
            } else {
                if (row >= n)
#pragma unroll
                    for (int c = 0; c < V; ++c) o[c] = 0.f;
                store_row<E, V>(dx + (int64_t)row * rowlen, o);
            }
        }
    }
    float* part = p.part + ((int64_t)blockIdx.y * a.B + b) * (W + 1) * a.D + d;
#pragma unroll
    for (int j = 0; j < W; ++j) store_row<float, V>(part + (int64_t)j * a.D, dw[j]);
    store_row<float, V>(part + (int64_t)W * a.D, db);
}

// out[c] = sum over k of part[k][c], c < cols, in a fixed order whatever the grid: a block adds `step` rows of 64 columns, its four
// waves every fourth row, wave 0 the four sums.  With more than 64 rows a first launch adds up to 64 slices of them into `mid`.
__global__ __launch_bounds__(256) void sum_parts_kernel(const float* part, int64_t n, int64_t step, int cols, float* out0, int split, float* out1) {
    __shared__ float acc[4][64];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, c = blockIdx.x * 64 + lane;
    const int64_t k0 = (int64_t)blockIdx.y * step, k1 = min(n, k0 + step);
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    if (c < cols)
        for (int64_t k = k0 + wv; k < k1; k += 16)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (k + 4 * q < k1) s[q] += part[(k + 4 * q) * cols + c];
    acc[wv][lane] = (s[0] + s[1]) + (s[2] + s[3]);
    __syncthreads();
    if (wv || c >= cols) return;
    const float v = (acc[0][lane] + acc[1][lane]) + (acc[2][lane] + acc[3][lane]);
    if (c >= split) {
        if (out1) out1[c - split] = v;
    } else if (out0) {
        out0[(int64_t)blockIdx.y * cols + c] = v;
    }
}

constexpr int kSlices = 64;
size_t sum_parts_floats(int64_t n, int64_t cols) { return n > kSlices ? (size_t)kSlices * cols : 0; }

int launch_sum_parts(const float* part, int64_t n, int cols, float* mid, float* out0, int split, float* out1, hipStream_t stream) {
    if (n > kSlices) {
        const int64_t step = (n + kSlices - 1) / kSlices;
        const int slices = (int)((n + step - 1) / step);
        hipLaunchKernelGGL(sum_parts_kernel, dim3(ceil_div(cols, 64), slices), dim3(256), 0, stream, part, n, step, cols, mid, cols, nullptr);
        part = mid;
        n = slices;
    }
    hipLaunchKernelGGL(sum_parts_kernel, dim3(ceil_div(cols, 64)), dim3(256), 0, stream, part, n, n, cols, out0, split, out1);
    SV_CHECK_HIP(hipGetLastError());
    return SHIVAE_OK;
}

// Time steps per thread.  Forward 16: longer runs read fewer rows twice, but leave fewer loads in flight (us, runs of 16 / 32 / 64: T 2048,
// B 16, D 2048, bf16 49 / 49 / 55; T 1000, B 64, D 256, fp32 23 / 24 / 30; T 256, B 4, D 512 10.7 / 12.8 / 22; T 4096, B 64 runs of 16 / 64
// 421 / 447).  Backward a run writes partial sums of the parameters' gradients, (W + 1) D fp32 numbers, as much as ten bf16 rows: as long as
// two waves are left for every SIMD, up to 256 (with 8 / 4 / 2 waves: 205 / 172 / 161; 60 / 61 / 52; 26 in all; and T 4096, B 64, up to
// 64 / 256: 1136 / 1028).
static int conv_run(const shivae_conv_args& a, int vec, bool bwd) {
    const int64_t seqs = (int64_t)a.B * ceil_div(a.D, vec);
    int run = 16;
    if (bwd)
        while (run < 256 && seqs * ceil_div(a.T, run * 2) >= 1024 * 2 * 64) run *= 2;
    while (ceil_div(a.T, run) > 65535) run *= 2;
    return run;
}

static int conv_vec(const shivae_conv_args& a, bool bwd) {
    const int v = 16 / elem_bytes(a.dtype), ib = 16;
    bool ok = a.D % v == 0 && a.x_st % v == 0 && a.x_sb % v == 0 && aligned_to(a.x, ib) && aligned_to(a.weight, ib) && aligned_to(a.bias, ib) && aligned_to(a.state, ib);
    if (bwd) ok = ok && a.dy_st % v == 0 && a.dy_sb % v == 0 && aligned_to(a.dy, ib) && aligned_to(a.dx, ib) && aligned_to(a.dstate, ib) && aligned_to(a.dstate_out, ib);
    else ok = ok && a.y_st % v == 0 && a.y_sb % v == 0 && aligned_to(a.y, ib) && aligned_to(a.state_out, ib);
    return ok ? v : 1;
}

template <class E, int V>
static void launch_conv(bool bwd, const ConvP& p, dim3 grid, hipStream_t s) {
#define SV_CONV(WW)                                                                                       \
    if (bwd) hipLaunchKernelGGL((conv_bwd_kernel<E, V, WW>), grid, dim3(256), 0, s, p);                   \
    else hipLaunchKernelGGL((conv_fwd_kernel<E, V, WW>), grid, dim3(256), 0, s, p)
    if (p.a.W == 2) { SV_CONV(2); }
    else if (p.a.W == 3) { SV_CONV(3); }
    else { SV_CONV(4); }
#undef SV_CONV
}

static int conv_check(const shivae_conv_args* a, const char* who) {
    SV_REQUIRE(a, "%s: null argument block", who);
    SV_REQUIRE(a->T > 0 && a->B > 0 && a->D > 0, "%s: T, B, D must be positive (%d, %d, %d)", who, a->T, a->B, a->D);
    SV_REQUIRE(a->W >= 2 && a->W <= 4, "%s: filter width %d is not 2, 3 or 4", who, a->W);
    SV_REQUIRE(a->dtype == SHIVAE_F32 || a->dtype == SHIVAE_BF16 || a->dtype == SHIVAE_F16, "%s: unknown dtype %d", who, a->dtype);
    SV_REQUIRE(a->x && a->weight, "%s: x and weight are required", who);
    SV_REQUIRE(a->T <= 1 << 30 && a->B <= 1 << 30 && a->D <= 1 << 24 && (int64_t)a->B * a->D < (int64_t)1 << 38, "%s: T, B or D is too large", who);
    return SHIVAE_OK;
}

}  // namespace shivae

using namespace shivae;

extern "C" {

int shivae_causal_conv_fwd(const shivae_conv_args* args, shivae_stream stream) {
    SV_TRY(conv_check(args, "causal_conv_fwd"));
    const shivae_conv_args& a = *args;
    SV_REQUIRE(a.y, "causal_conv_fwd: y is required");
    const int v = conv_vec(a, false);
    ConvP p{a, ceil_div(a.D, v), conv_run(a, v, false), 0, nullptr};
    p.nrun = ceil_div(a.T, p.run);
    SV_REQUIRE(!a.state || a.state != a.state_out || p.nrun == 1, "causal_conv_fwd: the state can be updated in place for up to %d time steps only", p.run);
    const int64_t blocks = ((int64_t)a.B * p.nvec + 255) / 256;
    SV_REQUIRE(grid_fits(blocks, 256), "causal_conv_fwd: B * D is too large (%d sequences of %d channel groups)", a.B, p.nvec);
    const dim3 grid((unsigned)blocks, p.nrun);
    SV_BY_DTYPE(a.dtype, {
        if (v > 1) launch_conv<E, 16 / (int)sizeof(E)>(false, p, grid, static_cast<hipStream_t>(stream));
        else launch_conv<E, 1>(false, p, grid, static_cast<hipStream_t>(stream));
    });
    SV_CHECK_HIP(hipGetLastError());
    return SHIVAE_OK;
}

size_t shivae_causal_conv_bwd_ws(const shivae_conv_args* args) {
    if (conv_check(args, "causal_conv_bwd_ws") != SHIVAE_OK) return 0;
    // (runs are shortest, and partials most, where a thread owns eight channels)
    const int64_t n = (int64_t)ceil_div(args->T, conv_run(*args, 8, true)) * args->B, cols = (int64_t)(args->W + 1) * args->D;
    return ((size_t)n * cols + sum_parts_floats(n, cols)) * sizeof(float);
}

int shivae_causal_conv_bwd(const shivae_conv_args* args, void* ws_dev, size_t ws_bytes, shivae_stream stream) {
    SV_TRY(conv_check(args, "causal_conv_bwd"));
    const shivae_conv_args& a = *args;
    SV_REQUIRE(a.dy && a.dx && a.dweight, "causal_conv_bwd: dy, dx and dweight are required");
    SV_REQUIRE(!a.state || a.dstate, "causal_conv_bwd: a state that came in needs a buffer for its gradient");
    SV_REQUIRE(a.dbias || !a.bias, "causal_conv_bwd: a bias needs a buffer for its gradient");
    const int v = conv_vec(a, true);
    ConvP p{a, ceil_div(a.D, v), conv_run(a, v, true), 0, static_cast<float*>(ws_dev)};
    p.nrun = ceil_div(a.T, p.run);
    const int64_t blocks = ((int64_t)a.B * p.nvec + 255) / 256;
    SV_REQUIRE(grid_fits(blocks, 256), "causal_conv_bwd: B * D is too large (%d sequences of %d channel groups)", a.B, p.nvec);
    const size_t need = shivae_causal_conv_bwd_ws(args);
    SV_REQUIRE(ws_dev && ws_bytes >= need, "causal_conv_bwd: workspace of %zu bytes is smaller than %zu", ws_bytes, need);
    SV_REQUIRE(aligned_to(ws_dev, 16), "causal_conv_bwd: the workspace must be 16-byte aligned");
    const dim3 grid((unsigned)blocks, p.nrun);
    hipStream_t s = static_cast<hipStream_t>(stream);
    SV_BY_DTYPE(a.dtype, {
        if (v > 1) launch_conv<E, 16 / (int)sizeof(E)>(true, p, grid, s);
        else launch_conv<E, 1>(true, p, grid, s);
    });
    SV_CHECK_HIP(hipGetLastError());
    const int64_t n = (int64_t)p.nrun * a.B;
    const int cols = (a.W + 1) * a.D;
    return launch_sum_parts(p.part, n, cols, p.part + n * cols, a.dweight, a.W * a.D, a.dbias, s);
}

}  // extern "C"
