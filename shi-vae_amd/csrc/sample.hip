// Drawing a category from logits with temperature, top-k, top-p and min-p, one uniform number per row.
//
//   w_i = exp((x_i - max) / temperature); order = by value descending, equal values by index ascending
//   kept: the first top_k in the order; of these the shortest lead whose weight reaches top_p of theirs; of these w >= min_p
//   token = the first index i, in index order, with  sum_{kept j <= i} w_j > u * sum_{kept j} w_j
//
// Which category is drawn hangs on comparisons of long sums, and 16-bit logits have long runs of equal values, whose errors add up
// in step.  So a weight is computed in 64 bits (a polynomial for 2^f, within 2^-38 of the weight) and held as a multiple of 2^-43 of the
// largest: sums of these are exact, independent of order (integer LDS atomics included), and fit 63 bits for 2^20 categories.  A
// weight below 2^-44 of the largest is 0 and is never drawn.  Order is by the logits' own bits, never by rounded quotients.
//
// Measured (us): 256 x 131072, bf16, top-p 0.95 133, with min-p 0.01 114, top-k 50 35, no cut 62, the largest alone 24; 1 x 32768, top-k 50
// 14, with top-p 15.6; 102400 rows of 8 9.  Where it hurts: a row stays on one compute unit, 1 x 131072 with top-p takes 118 us.
//
// A row is a workgroup's.  No row is sorted: top-k and top-p need the last element they keep.  A histogram of (max - x) /
// temperature over the range that has weight (counts, or sums of weights) finds the bin it lies in; the elements of that bin -- or
// of all bins up to it, when they are few, which leaves nothing of the row to read again -- go to a list in LDS that is sorted.  A
// bin too full for the list (runs of equal values) is resolved by four 8-bit digits of the key instead.  Bound by the row's reads
// for few kept elements (the row stays in L2 between the passes) and by vector instructions for many: about 25 for an exponential in 64
// bits, 100 per category in all with top-p.
#include <algorithm>

#include "common.h"
#include "elem.h"

namespace shivae {

using u64 = unsigned long long;

struct SampleP {
    shivae_sample_args a;
};

struct RowParams {
    float temperature, top_p, min_p, u;
    int top_k;
};
__device__ __forceinline__ RowParams row_params(const shivae_sample_args& a, int64_t r) {
    RowParams q;
    q.temperature = a.temperature_rows ? a.temperature_rows[r] : a.temperature;
    q.top_k = a.top_k_rows ? a.top_k_rows[r] : a.top_k;
    q.top_p = a.top_p_rows ? a.top_p_rows[r] : a.top_p;
    q.min_p = fminf(a.min_p_rows ? a.min_p_rows[r] : a.min_p, 1.f);  // the largest is always kept
    q.u = a.u[r];
    if (q.top_k <= 0 || q.top_k >= a.V) q.top_k = 0;
    return q;
}

// A logit as it is compared: NaN counts as -inf.
__device__ __forceinline__ float clean(float x) { return fmaxf(x, -INFINITY); }
// Unsigned keys in the order of the values (-0 as 0), and back.
__device__ __forceinline__ unsigned key_of(float x) {
    const unsigned b = __float_as_uint(x + 0.f);
    return b ^ ((unsigned)((int)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float of_key(unsigned k) { return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu)); }

constexpr int kFix = 43;
// 2^(y + SHIFT) for -900 <= y <= 0.  2^f = 1 + f P(f), |f| <= 1/2, where P, of degree 7, meets (2^f - 1) / f at the eight Chebyshev
// nodes of the interval: within 2.2e-12 = 2^-38.7 (the Taylor series needs two terms more for that).  Adding 1.5 2^52 + SHIFT rounds y to a
// whole number and leaves it, SHIFT larger, in the low word, which is added to the exponent (v_rndne_f64, v_ldexp_f64 and the conversion
// cost several fused operations each).
template <int SHIFT>
__device__ __forceinline__ double exp2_f64(double y) {
    constexpr double magic = 6755399441055744.0 + SHIFT;
    const double t = y + magic, f = y - (t - magic);
    double p = 1.3250805517502250e-06;
    p = fma(p, f, 1.5303700711365693e-05);
    p = fma(p, f, 1.5403475186530786e-04);
    p = fma(p, f, 1.3333478473685416e-03);
    p = fma(p, f, 9.6181291352361396e-03);
    p = fma(p, f, 5.5504109063258665e-02);
    p = fma(p, f, 2.4022650695888503e-01);
    p = fma(p, f, 6.9314718055683244e-01);
    p = fma(p, f, 1.0);
    const u64 b = (u64)__double_as_longlong(p);
    const unsigned hi = (unsigned)(b >> 32) + ((unsigned)__double_as_longlong(t) << 20);
    return __longlong_as_double((long long)((u64)hi << 32 | (unsigned)b));
}
// The weight of x as a multiple of 2^-43: adding 2^52 rounds to whole numbers and leaves them in the mantissa.
struct Weigh {
    double c, top;  // log2(e) / temperature, the largest logit
    double least;   // log2 of min_p, at least -44
    __device__ __forceinline__ double log2w(float x) const { return ((double)x - top) * c; }
    __device__ void set(float max, float temperature, float min_p) {
        c = 1.4426950408889634074 / (double)temperature;
        top = max;
        least = min_p > 0.f ? fmax(log2((double)min_p), -44.0) : -44.0;
    }
    __device__ __forceinline__ bool enough(float x) const { return log2w(x) >= least; }  // min-p
    // No branch: eight elements' chains of dependent operations run side by side.  -inf (and -inf * 0) become 2^-200, which rounds to 0.
    __device__ __forceinline__ u64 fix(float x) const {
        return (u64)__double_as_longlong(exp2_f64<kFix>(fmax(log2w(x), -200.0)) + 4503599627370496.0) & 0xfffffffffffffull;
    }
};

// The sum over the wave's lanes, in every lane: rotations within rows of 16 lanes, then exchanges of rows (no LDS round trips).
template <int CTRL>
__device__ __forceinline__ u64 ror_add(u64 v) {
    const unsigned lo = __builtin_amdgcn_mov_dpp((unsigned)v, CTRL, 0xf, 0xf, true), hi = __builtin_amdgcn_mov_dpp((unsigned)(v >> 32), CTRL, 0xf, 0xf, true);
    return v + ((u64)hi << 32 | lo);
}
__device__ __forceinline__ u64 wave_sum(u64 v) {
    v = ror_add<0x128>(v);
    v = ror_add<0x124>(v);
    v = ror_add<0x122>(v);
    v = ror_add<0x121>(v);
    auto l = __builtin_amdgcn_permlane16_swap((unsigned)v, (unsigned)v, false, false), h = __builtin_amdgcn_permlane16_swap((unsigned)(v >> 32), (unsigned)(v >> 32), false, false);
    v = ((u64)h[0] << 32 | l[0]) + ((u64)h[1] << 32 | l[1]);
    l = __builtin_amdgcn_permlane32_swap((unsigned)v, (unsigned)v, false, false);
    h = __builtin_amdgcn_permlane32_swap((unsigned)(v >> 32), (unsigned)(v >> 32), false, false);
    return ((u64)h[0] << 32 | l[0]) + ((u64)h[1] << 32 | l[1]);
}

// The sum over lanes 0 to this one: shifts within rows of 16 lanes (row_shr, 0 from outside), then the rows in front.
template <int CTRL>
__device__ __forceinline__ u64 shr_add(u64 v) {
    const unsigned lo = __builtin_amdgcn_update_dpp(0u, (unsigned)v, CTRL, 0xf, 0xf, false), hi = __builtin_amdgcn_update_dpp(0u, (unsigned)(v >> 32), CTRL, 0xf, 0xf, false);
    return v + ((u64)hi << 32 | lo);
}
__device__ __forceinline__ u64 lane_u64(u64 v, int l) {
    return (u64)(unsigned)__builtin_amdgcn_readlane((int)(v >> 32), l) << 32 | (unsigned)__builtin_amdgcn_readlane((int)v, l);
}
__device__ __forceinline__ u64 wave_scan(u64 v, int lane) {
    v = shr_add<0x111>(v);
    v = shr_add<0x112>(v);
    v = shr_add<0x114>(v);
    v = shr_add<0x118>(v);
    const u64 r0 = lane_u64(v, 15), r1 = lane_u64(v, 31), r2 = lane_u64(v, 47);
    return v + (lane >= 16 ? r0 : 0) + (lane >= 32 ? r1 : 0) + (lane >= 48 ? r2 : 0);
}

// ------------------------------------------------------------------------------------------------ a workgroup per row
template <class E, int NT, int CAP, int NB>
struct Sampler {
    static constexpr int VE = 16 / (int)sizeof(E), NWV = NT / 64;
    static_assert(NB >= 256 && CAP >= 128, "a digit's bins and a short row's list have to fit");
    struct Shared {
        u64 hist[NB];   // bins, or sums of 64-vector segments of the row
        u64 list[CAP];
        u64 wave[NWV + 1];
        u64 found[2];
        int count, pos;
        int rank[128];  // 0 between sorts
    };

    Shared& s;
    const int tid, lane, wv;
    const E* p;
    int V, off, nvec;
    bool has_inf;  // the largest logit is +inf: +inf reads as 0, everything else as -inf

    __device__ Sampler(Shared& sh, const E* row, int n) : s(sh), tid(threadIdx.x), lane(threadIdx.x & 63), wv(threadIdx.x >> 6), p(row), V(n) {
        off = (int)(((uintptr_t)row & 15) / sizeof(E));  // vectors are aligned; the first one may start before the row
        nvec = (n + off + VE - 1) / VE;
        has_inf = false;
    }

    // Vector i of the row: values, -inf outside the row.
    __device__ __forceinline__ void get(int i, float (&x)[VE]) const {
        const int j0 = i * VE - off;
        if (j0 >= 0 && j0 + VE <= V) {
            const Pack<E, VE> r = *reinterpret_cast<const Pack<E, VE>*>(p + j0);
#pragma unroll
            for (int k = 0; k < VE; ++k) x[k] = clean(elem_f(r.v[k]));
        } else {
#pragma unroll
            for (int k = 0; k < VE; ++k) x[k] = j0 + k >= 0 && j0 + k < V ? clean(elem_f(p[j0 + k])) : -INFINITY;
        }
        if (has_inf)
#pragma unroll
            for (int k = 0; k < VE; ++k) x[k] = x[k] == INFINITY ? 0.f : -INFINITY;
    }

    // f(i, x) for every vector of the row, by whole waves of 64 neighbouring vectors (the last wave's lanes behind the row hold -inf).  Four
    // loads of a thread are in flight at a time: with one, each pass waits 16 times for L2 at 131072 categories.
    template <class F>
    __device__ __forceinline__ void sweep(F f) const {
        constexpr int U = 4;
        const int end = (nvec + 63) & ~63;
        for (int i0 = tid; i0 < end; i0 += U * NT) {
            Pack<E, VE> raw[U];
#pragma unroll
            for (int t = 0; t < U; ++t) {
                const int j0 = (i0 + t * NT) * VE - off;
                if (j0 >= 0 && j0 + VE <= V) raw[t] = *reinterpret_cast<const Pack<E, VE>*>(p + j0);
            }
            // (one copy of f: unrolled four times the passes of a row do not fit the instruction cache)
#pragma unroll 1
            for (int i = i0; i < min(end, i0 + U * NT); i += NT) {
                const int j0 = i * VE - off;
                float x[VE];
                if (j0 >= 0 && j0 + VE <= V) {
#pragma unroll
                    for (int k = 0; k < VE; ++k) x[k] = clean(elem_f(raw[0].v[k]));
                    if (has_inf)
#pragma unroll
                        for (int k = 0; k < VE; ++k) x[k] = x[k] == INFINITY ? 0.f : -INFINITY;
                } else {
                    get(i, x);
                }
                f(i, x);
#pragma unroll
                for (int t = 0; t + 1 < U; ++t) raw[t] = raw[t + 1];
            }
        }
    }

    // Exclusive sum of v over the workgroup's threads, and the whole sum.  Ends with a barrier behind the last read.
    __device__ __forceinline__ u64 scan(u64 v, u64& total) {
        const u64 in = wave_scan(v, lane);
        if (NWV == 1) {
            total = lane_u64(in, 63);
            return in - v;
        }
        if (lane == 63) s.wave[wv] = in;
        __syncthreads();
        u64 before = 0, all = 0;
#pragma unroll
        for (int i = 0; i < NWV; ++i) {
            const u64 w = s.wave[i];
            if (i < wv) before += w;
            all += w;
        }
        total = all;
        __syncthreads();
        return before + in - v;
    }

    // The first of n items, in order, at which the running sum exceeds what goal(total) gives; -> its number (n if none), the sum in
    // front of it in `before`.
    template <class W, class G>
    __device__ __forceinline__ int first_beyond(int n, W weight, G goal, u64& before, u64& total) {
        const int per = (n + NT - 1) / NT, i0 = min(n, tid * per), i1 = min(n, i0 + per);
        u64 sum = 0;
        for (int i = i0; i < i1; ++i) sum += weight(i);
        u64 run = scan(sum, total);
        const u64 g = goal(total);
        if (tid == 0) {
            s.pos = n;
            s.found[0] = 0;
        }
        __syncthreads();
        if (run <= g && run + sum > g)
            for (int i = i0; i < i1; ++i) {
                const u64 w = weight(i);
                if (run + w > g) {
                    s.pos = i;
                    s.found[0] = run;
                    break;
                }
                run += w;
            }
        __syncthreads();
        const int at = s.pos;
        before = s.found[0];
        __syncthreads();
        return at;
    }

    // list[0, n) into descending order (entries differ, but for zeros, which end up behind the rest).  Up to 128 entries by counting what
    // is larger, at two barriers and by the waves that hold some; longer lists, padded to a power of two with zeros, by a bitonic network.
    __device__ __forceinline__ void sort(int n) {
        if (n <= 128 && n <= NT) {
            // (128 threads, or a wave, for the entries, each set of them for a part of what they are compared with)
            constexpr int SPAN = NT < 128 ? NT : 128, PARTS = NT / SPAN;
            const int i = tid & (SPAN - 1);
            u64 e = 0;
            if (i < n) {
                e = s.list[i];
                int rank = 0;
#pragma unroll 4
                for (int j = tid / SPAN; j < n; j += PARTS) {
                    const u64 o = s.list[j];
                    rank += o > e || (o == e && j < i);
                }
                atomicAdd(&s.rank[i], rank);
            }
            __syncthreads();
            if (tid < SPAN && i < n) {
                s.list[s.rank[i]] = e;
                s.rank[i] = 0;
            }
            __syncthreads();
            return;
        }
        int m = 1;
        while (m < n) m <<= 1;
        for (int i = n + tid; i < m; i += NT) s.list[i] = 0;
        __syncthreads();
        for (int k = 2; k <= m; k <<= 1)
            for (int j = k >> 1; j; j >>= 1) {
                for (int i = tid; i < m / 2; i += NT) {
                    const int a = (i & ~(j - 1)) * 2 + (i & (j - 1)), b = a + j;
                    const u64 x = s.list[a], y = s.list[b];
                    if ((x < y) == ((a & k) == 0)) {
                        s.list[a] = y;
                        s.list[b] = x;
                    }
                }
                // A wave's 64 pairs lie in 128 entries that are its own in every step with j <= 64.
                if (j > 64 || (j > 1 ? j >> 1 : k) > 64) {
                    __syncthreads();
                } else {
                    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                    __builtin_amdgcn_wave_barrier();
                }
            }
    }

    // Adds every element to its bin of the histogram: bin_of(x, index) < 0 is none, value(x) what to add.  A wave whose elements
    // all lie in one bin (runs of equal values) adds once, since additions to one address queue up.
    template <class B, class W>
    __device__ __forceinline__ void fill(int bins, B bin_of, W value) {
        clear(bins);
        sweep([&](int i, const float (&x)[VE]) {
            int b[VE];
            bool same = true;
#pragma unroll
            for (int k = 0; k < VE; ++k) {
                b[k] = bin_of(x[k], i * VE + k - off);
                same &= b[k] == b[0];
            }
            const int first = __builtin_amdgcn_readfirstlane(b[0]);
            if (__ballot(same && b[0] == first) == ~0ull) {
                if (first < 0) return;
                u64 v = 0;
#pragma unroll
                for (int k = 0; k < VE; ++k) v += value(x[k]);
                v = wave_sum(v);
                if (lane == 0) atomicAdd(&s.hist[first], v);
            } else {
                u64 v[VE];
#pragma unroll
                for (int k = 0; k < VE; ++k) v[k] = value(x[k]);
#pragma unroll
                for (int k = 0; k < VE; ++k)
                    if (b[k] >= 0) atomicAdd(&s.hist[b[k]], v[k]);
            }
        });
        __syncthreads();
    }
    // Puts the elements that take(x, index) holds into the list, in any order, as far as there is room; -> their number.
    template <class F>
    __device__ __forceinline__ int gather(F take) {
        if (tid == 0) s.count = 0;
        __syncthreads();
        sweep([&](int i, const float (&x)[VE]) {
            unsigned m = 0;
#pragma unroll
            for (int k = 0; k < VE; ++k) m |= take(x[k], i * VE + k - off) ? 1u << k : 0u;
            if (!m) return;
            int at = atomicAdd(&s.count, __popc(m));
#pragma unroll
            for (int k = 0; k < VE; ++k)
                if ((m >> k & 1) && at < CAP) s.list[at++] = place(x[k], i * VE + k - off);
        });
        __syncthreads();
        const int n = s.count;
        __syncthreads();
        return n;
    }
    __device__ __forceinline__ void clear(int n) {
        for (int i = tid; i < n; i += NT) s.hist[i] = 0;
        __syncthreads();
    }

    u64 last;  // the last kept element's place in the order; 0: everything is kept
    // A place in the order, as key << 32 | ~index: larger comes first.
    __device__ __forceinline__ static u64 place(float x, int idx) { return (u64)key_of(x) << 32 | (0xffffffffu - (unsigned)idx); }

    // (max - x) scaled to bins: monotone in x, so bins are in the order of the values.  NB - 1: no weight.
    float top, bscale;
    __device__ __forceinline__ int bin(float x) const { return (int)fminf((top - x) * bscale, (float)(NB - 1)); }  // (-inf, NaN: the last)

    __device__ __forceinline__ int has_weight(float x) const {  // its bin, or -1
        const int b = bin(x);
        return b < NB - 1 ? b : -1;
    }

    // The element at which the running sum, in the order, over the kept elements of bin b first exceeds g (sum in front of the bin:
    // `before`), by counts or by weights.
    template <class W>
    __device__ __forceinline__ u64 resolve(int b, u64 before, u64 g, W weight) {
        const auto in = [&](float x, int i) { return bin(x) == b && place(x, i) >= last; };
        const int n = gather(in);
        if (n <= CAP) {
            sort(n);
            u64 bf, total;
            const int at = first_beyond(n, [&](int i) { return weight(of_key((unsigned)(s.list[i] >> 32))); }, [&](u64) { return g - before; }, bf, total);
            const u64 e = n ? s.list[min(at, n - 1)] : last;
            __syncthreads();
            return e;
        }
        unsigned prefix = 0, mask = 0;
#pragma unroll 1
        for (int shift = 24; shift >= 0; shift -= 8) {
            fill(256, [&](float x, int i) { return in(x, i) && (key_of(x) & mask) == prefix ? 255 - (int)((key_of(x) >> shift) & 255) : -1; }, weight);
            u64 bf, total;
            const int d = min(first_beyond(256, [&](int i) { return s.hist[i]; }, [&](u64) { return g - before; }, bf, total), 255);
            before += bf;
            prefix |= (unsigned)(255 - d) << shift;
            mask |= 255u << shift;
        }
        // Equal values from here on: which of them in index order.  (Those that an earlier cut dropped lie behind its own place.)
        const float x0 = of_key(prefix);
        const u64 w = weight(x0), nth = w ? (g - before) / w : 0;
        const bool tie = last && of_key((unsigned)(last >> 32)) == x0;
        upto = tie ? (int)(0xffffffffu - (unsigned)last) : 0x7fffffff;
        low = x0;
        u64 bf, total;
        float xv;
        const int idx = locate([&](float x) { return (u64)(x == x0); }, [&](u64) { return nth; }, bf, total, xv);
        return place(x0, idx < 0 ? V - 1 : idx);
    }

    // What the draw takes: above low, and at low up to index `upto`.
    float low;
    int upto;
    __device__ __forceinline__ bool takes(float x, int idx) const { return x > low || (x == low && idx <= upto); }

    // The sum over the wave's elements whose bits in m are set goes to the sum of their segment, 64 vectors.  Where few elements are taken a
    // lane computes weights for its own only, one in each round.  (256 x 131072, us, no cut / min-p 0.01 / top-p 0.3: 62 / 49 / 98; always all
    // weights 62 / 64 / 109, always rounds 91 / 48 / 98.)
    template <class W>
    __device__ __forceinline__ void segment_sum(int i, const float (&x)[VE], unsigned m, W weight) {
        u64 sum = 0;
        if (!__any(__popc(m) > VE / 2)) {
            while (__any(m != 0)) {
                float v = x[0];
#pragma unroll
                for (int k = 1; k < VE; ++k) v = (m & ((1u << k) - 1)) ? v : x[k];  // the last k with nothing taken in front of it
                const u64 w = weight(v);
                if (m) sum += w;
                m &= m - 1;
            }
        } else {
            u64 w[VE];
#pragma unroll
            for (int k = 0; k < VE; ++k) w[k] = weight(x[k]);
#pragma unroll
            for (int k = 0; k < VE; ++k) sum += m >> k & 1 ? w[k] : 0;
        }
        if (__any(sum != 0)) sum = wave_sum(sum);
        if (lane == 0) s.hist[i >> 6] = sum;
    }
    // The first index, in index order, at which the running sum of weight(x), over what takes(x, index) holds of, exceeds goal(total); -1
    // if none.  Sums of segments first, then one wave looks into the segment.
    template <class W, class G>
    __device__ __forceinline__ int locate(W weight, G goal, u64& before, u64& total, float& value) {
        sweep([&](int i, const float (&x)[VE]) {
            unsigned m = 0;
#pragma unroll
            for (int k = 0; k < VE; ++k) m |= takes(x[k], i * VE + k - off) ? 1u << k : 0u;
            segment_sum(i, x, m, weight);
        });
        return locate_in_sums(weight, goal, before, total, value);
    }
    template <class W, class G>
    __device__ __forceinline__ int locate_in_sums(W weight, G goal, u64& before, u64& total, float& value) {
        const int nseg = (nvec + 63) / 64;
        __syncthreads();
        u64 g = 0;
        const int seg = first_beyond(nseg, [&](int i) { return s.hist[i]; }, [&](u64 t) { return g = goal(t); }, before, total);
        if (tid == 0) s.pos = -1;
        __syncthreads();
        if (seg < nseg && wv == 0) {
            const int i = seg * 64 + lane;
            float x[VE];
            u64 w[VE], sum = 0;
            if (i < nvec) get(i, x);
#pragma unroll
            for (int k = 0; k < VE; ++k) {
                w[k] = i < nvec && takes(x[k], i * VE + k - off) ? weight(x[k]) : 0;
                sum += w[k];
            }
            const u64 in = wave_scan(sum, lane);
            u64 run = before + in - sum;
            if (run <= g && run + sum > g) {
                bool open = true;
#pragma unroll
                for (int k = 0; k < VE; ++k) {
                    if (open && run + w[k] > g) {
                        open = false;
                        s.pos = i * VE + k - off;
                        s.found[1] = __float_as_uint(x[k]);
                    }
                    run += w[k];
                }
            }
        }
        __syncthreads();
        const int idx = s.pos;
        value = __uint_as_float((unsigned)s.found[1]);
        __syncthreads();
        return idx;
    }

    // Where the lead ends in bin b, in front of which it holds all (weight `before`): one pass sums what is taken of those bins by segments and
    // lists bin b; what the lead holds of the list is added to the segments.  Sets `last`; false, with nothing done, if the list is too short.
    template <class W>
    __device__ __forceinline__ bool lead_sums(int b, u64 before, u64 g, W weight) {
        if (tid == 0) s.count = 0;
        __syncthreads();
        sweep([&](int i, const float (&x)[VE]) {
            unsigned m = 0, e = 0;
#pragma unroll
            for (int k = 0; k < VE; ++k) {
                const int bk = bin(x[k]);
                m |= bk < b && x[k] >= low ? 1u << k : 0u;
                e |= bk == b && place(x[k], i * VE + k - off) >= last ? 1u << k : 0u;
            }
            segment_sum(i, x, m, weight);
            if (!e) return;
            int at = atomicAdd(&s.count, __popc(e));
#pragma unroll
            for (int k = 0; k < VE; ++k)
                if ((e >> k & 1) && at < CAP) s.list[at++] = place(x[k], i * VE + k - off);
        });
        __syncthreads();
        const int n = s.count;
        __syncthreads();
        if (n > CAP) return false;
        sort(n);
        u64 bf, total;
        const int at = first_beyond(n, [&](int i) { return weight(of_key((unsigned)(s.list[i] >> 32))); }, [&](u64) { return g - before; }, bf, total);
        if (n) last = s.list[min(at, n - 1)];
        for (int i = tid; i <= min(at, n - 1); i += NT) {
            const float x = of_key((unsigned)(s.list[i] >> 32));
            const int idx = (int)(0xffffffffu - (unsigned)s.list[i]);
            if (x >= low) atomicAdd(&s.hist[(idx + off) / VE >> 6], weight(x));
        }
        __syncthreads();
        return true;
    }

    __device__ __forceinline__ float block_max(float v) {
#pragma unroll
        for (int d = 32; d; d >>= 1) v = fmaxf(v, __shfl_xor(v, d, 64));
        if (NWV > 1) {
            if (lane == 0) s.wave[wv] = __float_as_uint(v);
            __syncthreads();
            for (int i = 0; i < NWV; ++i) v = fmaxf(v, __uint_as_float((unsigned)s.wave[i]));
            __syncthreads();
        }
        return v;
    }
    // The lowest index at which the row holds x.
    __device__ __forceinline__ int first_equal(float x0) {
        if (tid == 0) s.pos = V;
        __syncthreads();
        int at = V;
        for (int i = tid; i < nvec && at == V; i += NT) {
            float x[VE];
            get(i, x);
#pragma unroll
            for (int k = VE - 1; k >= 0; --k)
                if (x[k] == x0) at = i * VE + k - off;
        }
        if (at < V) atomicMin(&s.pos, at);
        __syncthreads();
        return s.pos;
    }

    __device__ __forceinline__ void run(const RowParams& q, int64_t* token, float* logprob) {
        for (int i = tid; i < 128; i += NT) s.rank[i] = 0;
        // 1. the largest
        float most = -INFINITY;
        sweep([&](int, const float (&x)[VE]) {
#pragma unroll
            for (int k = 0; k < VE; ++k) most = fmaxf(most, x[k]);
        });
        top = block_max(most);
        if (top == -INFINITY || !(q.temperature > 0.f)) {
            const int arg = top == -INFINITY ? -1 : first_equal(top);
            if (tid == 0) {
                *token = arg;
                if (logprob) *logprob = top == -INFINITY ? -INFINITY : 0.f;
            }
            return;
        }
        if (top == INFINITY) {  // the limit of ever larger logits: those at +inf share everything
            has_inf = true;
            top = 0.f;
            most = most == INFINITY ? 0.f : -INFINITY;
        }
        Weigh wt;
        wt.set(top, q.temperature, q.min_p);
        bscale = fminf((float)(NB - 1) / (31.f * q.temperature), 1e30f);
        last = 0;
        const auto one = [](float) { return (u64)1; };
        const auto fix = [&](float x) { return wt.fix(x); };

        // 2. all that top-k keeps, or a small row, into the list
        int n = -1;  // elements in the list, if it holds all candidates
        if (q.top_k || q.top_p < 1.f) {
            // Sorting a list of all that is kept, or the bin of the last one and then (top-p) the row's weights once more?  us: 1 x 32768, top-k 1000
            // 45 / 30, with top-p 0.5 35 / 46; 64 x 8000 51 / 23, with top-p 37 / 32; 4096 x 2048, top-k 400 90 / 38, with top-p 0.9 74 / 57.
            const u64 longest = min(CAP, q.top_p < 1.f ? 2 * NT : max(128, NT / 2));
            int bk = NB - 2;
            u64 bf = 0, total = 0, upto = 0;
            const bool small = V <= 128;  // (ranks by counting; longer rows are cheaper by the histogram: 4096 x 512, top-p, 24 us against 60)
            if (!small && q.top_k && q.top_k <= NT / 2) {
                // top_k threads whose own largest lie in the bins up to bk: so do top_k elements.  There are not many more (0.7 NT for NT / 2, if
                // they lie at random), and the row's histogram is not needed: 1 x 32768, top-k 50 13.9 us, not 20.2; 256 x 131072 35, not 54.
                clear(NB);
                const int b = has_weight(most);
                if (b >= 0) atomicAdd(&s.hist[b], (u64)1);
                __syncthreads();
                bk = first_beyond(NB - 1, [&](int i) { return s.hist[i]; }, [&](u64) { return (u64)q.top_k - 1; }, bf, total);
                if (bk < NB - 1) n = gather([&](float x, int) { return bin(x) <= bk; });
                if (n > CAP) n = -1;
            }
            if (n < 0 && !small && q.top_k) {
                fill(NB, [&](float x, int) { return has_weight(x); }, one);
                bk = first_beyond(NB - 1, [&](int i) { return s.hist[i]; }, [&](u64) { return (u64)q.top_k - 1; }, bf, total);
                // (fewer than top_k elements of any weight: top-k keeps them all)
                upto = bk < NB - 1 ? bf + s.hist[bk] : total;
            }
            if (n < 0) {
                if (small || (q.top_k && upto <= longest)) n = gather([&](float x, int) { return bin(x) <= min(bk, NB - 2); });
                else if (q.top_k && bk < NB - 1) last = resolve(bk, bf, (u64)q.top_k - 1, one);
            }
        }
        u64 before, total;
        float xv = top;
        int idx;
        if (n >= 0) {
            sort(n);
            if (q.top_k) n = min(n, q.top_k);
            if (q.top_p < 1.f) {
                const int at = first_beyond(n, [&](int i) { return wt.fix(of_key((unsigned)(s.list[i] >> 32))); },
                                            [&](u64 t) { return lead(q.top_p, t); }, before, total);
                n = min(n, at + 1);
            }
            // into index order; what min-p drops goes to the end
            for (int i = tid; i < n; i += NT) {
                const u64 e = s.list[i];
                const unsigned key = (unsigned)(e >> 32);
                s.list[i] = wt.enough(of_key(key)) ? (e << 32) | key : 0;
            }
            __syncthreads();
            sort(n);
            const int at = first_beyond(n, [&](int i) { return s.list[i] ? wt.fix(of_key((unsigned)s.list[i])) : 0; },
                                        [&](u64 t) { return draw(q.u, t); }, before, total);
            const u64 e = s.list[min(at, n - 1)];
            idx = (int)(0xffffffffu - (unsigned)(e >> 32));
            xv = of_key((unsigned)e);
        } else {
            // 3. top-p over the row: the bin in which the lead ends, then its last element
            low = smallest(wt);
            upto = 0x7fffffff;
            bool summed = false;
            if (q.top_p < 1.f) {
                fill(NB, [&](float x, int i) { return last && place(x, i) < last ? -1 : has_weight(x); }, fix);
                u64 bf, g = 0;
                const int bp = first_beyond(NB - 1, [&](int i) { return s.hist[i]; }, [&](u64 t) { return g = lead(q.top_p, t); }, bf, total);
                if (bp < NB - 1) {
                    const float least = low;
                    summed = lead_sums(bp, bf, g, fix);
                    if (!summed) last = resolve(bp, bf, g, fix);
                    low = least;
                    upto = 0x7fffffff;
                }
            }
            // 4. the draw over the row
            const float cut = last ? of_key((unsigned)(last >> 32)) : -INFINITY;
            if (cut >= low) {
                low = cut;
                upto = (int)(0xffffffffu - (unsigned)last);
            }
            const auto goal = [&](u64 t) { return draw(q.u, t); };
            idx = summed ? locate_in_sums(fix, goal, before, total, xv) : locate(fix, goal, before, total, xv);
            if (idx < 0) {  // (not reached: the largest is always kept)
                idx = first_equal(top);
                xv = top;
            }
        }
        if (tid == 0) {
            *token = idx;
            if (logprob) *logprob = (float)(wt.log2w(xv) * 0.69314718055994530942 - log(ldexp((double)total, -kFix)));
        }
    }
    // The smallest value with w >= min_p and a weight at all: between two values a step apart there is none, so comparing values is
    // comparing weights.
    __device__ __forceinline__ float smallest(const Weigh& wt) const {
        unsigned lo = key_of(-INFINITY) + 1, hi = key_of(top);  // the least key for which enough() holds is in [lo, hi]
        while (lo < hi) {
            const unsigned mid = lo + (hi - lo) / 2;
            if (wt.enough(of_key(mid))) hi = mid;
            else lo = mid + 1;
        }
        return of_key(lo);
    }
    // Running sums are whole numbers: sum >= p * total is sum > ceil(p * total) - 1, sum > u * total is sum > floor(u * total).
    __device__ static u64 lead(float p, u64 total) {
        const double g = ceil(fmax((double)p, 0.0) * (double)total);
        return g < 1.0 ? 0 : (u64)g - 1;  // (past 2^53 a double has no g - 1)
    }
    __device__ static u64 draw(float u, u64 total) {
        const u64 g = (u64)(fmax((double)u, 0.0) * (double)total);
        return g < total ? g : (total ? total - 1 : 0);
    }
};

template <class E, int NT, int CAP, int NB>
__global__ __launch_bounds__(NT) void sample_kernel(SampleP p) {
    using S = Sampler<E, NT, CAP, NB>;
    __shared__ typename S::Shared sh;
    const int64_t r = blockIdx.x;
    S s(sh, static_cast<const E*>(p.a.logits) + r * p.a.ld, p.a.V);
    s.run(row_params(p.a, r), p.a.tokens + r, p.a.logprob ? p.a.logprob + r : nullptr);
}

// ------------------------------------------------------------------------------------------------ few categories
// L lanes per row (a power of two), a lane per category.  A lane finds what precedes it in the order by looking at every other one.
// 16384 rows of 60, top-p: 32 us, against 46 by a workgroup of one wave for each (44 with exchanges through LDS instead of v_readlane);
// of 24: 14.5 against 35.  102400 rows of 8, no cut: 8.6, of which 284 vector instructions a wave (8 rows) take 5.9 to issue; the
// log-probability's logarithm in 64 bits is 2.4 of the 8.6.  With top-p 10.3.
template <class E, int L>
__global__ __launch_bounds__(256) void sample_few_kernel(SampleP p) {
    const int64_t r = ((int64_t)blockIdx.x * 256 + threadIdx.x) / L;
    const int j = threadIdx.x & (L - 1);
    const bool live = r < p.a.rows;
    const int64_t rr = live ? r : 0;
    const RowParams q = row_params(p.a, rr);
    float x = live && j < p.a.V ? clean(elem_f(static_cast<const E*>(p.a.logits)[rr * p.a.ld + j])) : -INFINITY;
    float top = x;
#pragma unroll
    for (int d = L / 2; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d, L));
    const float top0 = top;
    if (top == INFINITY) {
        x = x == INFINITY ? 0.f : -INFINITY;
        top = 0.f;
    }
    Weigh wt;
    wt.set(top, q.temperature > 0.f ? q.temperature : 1.f, q.min_p);
    u64 w = x == -INFINITY ? 0 : wt.fix(x);
    int before = 0;      // elements in front of this one in the order, and their weight
    u64 weight = 0;
    if (__any(q.top_k != 0 || q.top_p < 1.f)) {
        for (int i = 0; i < L; ++i) {
            const float xi = L == 64 ? __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), i)) : __shfl(x, i, L);
            const u64 wi = L == 64 ? lane_u64(w, i) : (u64)__shfl((long long)w, i, L);
            if (xi > x || (xi == x && i < j)) {
                ++before;
                weight += wi;
            }
        }
        if (q.top_k && before >= q.top_k) w = 0;
        u64 total = w;
#pragma unroll
        for (int d = L / 2; d; d >>= 1) total += (u64)__shfl_xor((long long)total, d, L);
        if (q.top_p < 1.f && before > 0 && (double)weight >= fmax((double)q.top_p, 0.0) * (double)total) w = 0;
    }
    if (!wt.enough(x)) w = 0;
    u64 cum = w;
#pragma unroll
    for (int d = 1; d < L; d <<= 1) {
        const u64 o = (u64)__shfl_up((long long)cum, d, L);
        if (j >= d) cum += o;
    }
    const u64 total = (u64)__shfl((long long)cum, L - 1, L);
    const u64 g0 = (u64)(fmax((double)q.u, 0.0) * (double)total), g = g0 < total ? g0 : (total ? total - 1 : 0);
    const bool greedy = !(q.temperature > 0.f);
    const bool hit = greedy ? x == top : (cum > g && cum - w <= g);
    // the group's first lane that hits
    const u64 group = L == 64 ? ~0ull : ((1ull << (L & 63)) - 1) << ((threadIdx.x & 63) & ~(L - 1));
    const u64 hits = __ballot(hit) & group;
    if (!live) return;
    if (top0 == -INFINITY) {
        if (j == 0) {
            p.a.tokens[r] = -1;
            if (p.a.logprob) p.a.logprob[r] = -INFINITY;
        }
    } else if (hit && (int)(threadIdx.x & 63) == __ffsll((long long)hits) - 1) {
        p.a.tokens[r] = j;
        if (p.a.logprob) p.a.logprob[r] = greedy ? 0.f : (float)(wt.log2w(x) * 0.69314718055994530942 - log(ldexp((double)total, -kFix)));
    }
}

template <class E>
static void launch_sample(const SampleP& p, int64_t all_rows, hipStream_t s) {
    const int V = p.a.V;
    if (V <= 64) {
        const int L = V <= 2 ? 2 : V <= 4 ? 4 : V <= 8 ? 8 : V <= 16 ? 16 : V <= 32 ? 32 : 64;
        const dim3 grid((unsigned)((p.a.rows * L + 255) / 256));
        if (L == 2) hipLaunchKernelGGL((sample_few_kernel<E, 2>), grid, dim3(256), 0, s, p);
        else if (L == 4) hipLaunchKernelGGL((sample_few_kernel<E, 4>), grid, dim3(256), 0, s, p);
        else if (L == 8) hipLaunchKernelGGL((sample_few_kernel<E, 8>), grid, dim3(256), 0, s, p);
        else if (L == 16) hipLaunchKernelGGL((sample_few_kernel<E, 16>), grid, dim3(256), 0, s, p);
        else if (L == 32) hipLaunchKernelGGL((sample_few_kernel<E, 32>), grid, dim3(256), 0, s, p);
        else hipLaunchKernelGGL((sample_few_kernel<E, 64>), grid, dim3(256), 0, s, p);
        return;
    }
    // More threads for a row while the rows alone do not fill the card, fewer once they do: barriers are cheaper, and more rows share a
    // compute unit.  Measured (bf16, us, top-p 0.95): 256 x 2048 with 64 / 256 threads 23.8 / 14.9, 4096 x 2048 44.7 / 71, 4096 x 512 23.7 / 63;
    // 256 x 16384 with 256 / 1024 threads 36 / 31.7, 256 x 8192 24.0 / 25.1, 512 x 32768 77 / 89, 1024 x 32768 119 / 176.  (A row's sums of 64
    // vectors have to fit the histogram, so that the longest rows take 1024 threads however many they are.)
    const dim3 grid((unsigned)p.a.rows);
    if (V <= 512 || (V <= 4096 && all_rows >= 2048)) hipLaunchKernelGGL((sample_kernel<E, 64, 512, 256>), grid, dim3(64), 0, s, p);
    else if (V <= 8192 || (V <= 262144 && all_rows >= 512)) hipLaunchKernelGGL((sample_kernel<E, 256, 2048, 2048>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((sample_kernel<E, 1024, 4096, 4096>), grid, dim3(1024), 0, s, p);
}

}  // namespace shivae

using namespace shivae;

extern "C" int shivae_sample_categories(const shivae_sample_args* args, shivae_stream stream) {
    SV_REQUIRE(args, "sample_categories: null argument block");
    const shivae_sample_args& a = *args;
    SV_REQUIRE(a.rows > 0 && a.rows < (int64_t)1 << 25, "sample_categories: %lld rows, 1 to 2^25 are supported", (long long)a.rows);
    SV_REQUIRE(a.V >= 1 && a.V <= SHIVAE_SAMPLE_MAX, "sample_categories: %d categories, 1 to %d are supported", a.V, SHIVAE_SAMPLE_MAX);
    SV_REQUIRE(a.dtype == SHIVAE_F32 || a.dtype == SHIVAE_BF16 || a.dtype == SHIVAE_F16, "sample_categories: unknown dtype %d", a.dtype);
    SV_REQUIRE(a.logits && a.u && a.tokens, "sample_categories: logits, u and tokens are required");
    // Pieces of the rows whose threads, up to 1024 a row, a launch can have (the choice of threads goes by all rows).
    constexpr int64_t most = (int64_t)1 << 21;
    for (int64_t r = 0; r < a.rows; r += most) {
        SampleP p{a};
        p.a.logits = static_cast<const char*>(a.logits) + r * a.ld * elem_bytes(a.dtype);
        p.a.u += r;
        if (a.temperature_rows) p.a.temperature_rows += r;
        if (a.top_k_rows) p.a.top_k_rows += r;
        if (a.top_p_rows) p.a.top_p_rows += r;
        if (a.min_p_rows) p.a.min_p_rows += r;
        p.a.tokens += r;
        if (a.logprob) p.a.logprob += r;
        p.a.rows = std::min(most, a.rows - r);
        SV_BY_DTYPE(a.dtype, launch_sample<E>(p, a.rows, static_cast<hipStream_t>(stream)));
        SV_CHECK_HIP(hipGetLastError());
    }
    return SHIVAE_OK;
}
