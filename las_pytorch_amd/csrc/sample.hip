// Drawing a token from logits with temperature, top-k, top-p and min-p, from given random numbers.
//
//   w_v = exp((z_v - max z) / T);  falling order: larger logit first, equal logits by lower index
//   kept: the first top_k of that order; of those, every candidate before which less than top_p of their mass lies; of those, w_v >= min_p
//   token: the first kept index, in vocabulary order, at which the cumulated mass exceeds u times the kept mass
//
// The answer is a whole number that hangs on borders of long sums, so the sums are exact: w is formed in fp64 and held as an integer multiple of
// 2^-s (s = 62 - bits of V, at most 50), and integers add to the same sum in any order — by atomics too.  All three limits keep a head of the
// falling order, so the kept set is "every candidate not behind one cut", and the cut is one 64-bit number: (order-preserving bits of the logit,
// inverted index).  Cuts are found without sorting the row: a histogram of the distance to the maximum finds the bin that holds the cut, the
// candidates down to that bin go to a list, and only the list is sorted.  Where a bin holds more than the list can, the cut is searched digit by
// digit over the row itself.
//
// One workgroup works at a row where rows alone fill the GPU; otherwise a row is cut into slices (a workgroup each) in four launches: slice
// maxima, histogram, candidates and slice masses, the draw.  (Letting the row's last workgroup of the third draw at once was measured: its fences
// write back and drop whole L2s, 139 us at 64 rows of 32000 where that launch now takes a few and the fourth 10.)
// Bound by latency: 32 rows of 30 logits 10 us a call, 64 rows of 32000 with top-k 15, one row of 128000 with top-p 30 (four kernels of 4 + 7 + 10 + 9.5, chains of
// dependent reads and, in the last, a sort and a scan by one workgroup); and where rows alone fill the GPU by the fp64 weights, 300 cycles of a SIMD each, which
// top-p has formed twice: 241 rows of 31183 with top-p 60 us, without a limit 33.
#include "las_common.h"
#include "las_kernels.h"
#include <math.h>

namespace las {
namespace {

typedef unsigned long long u64;

constexpr int SM_BINS = 2048, SM_CAP = 4096, SM_TABLE = 256;
constexpr double SM_RANGE = 51.0;                // log2 units below the maximum: what lies further weighs nothing (s <= 50)

template <class T> static __device__ __forceinline__ float clean(T v) {
    const float x = (float)v;
    return x == x ? x + 0.f : -INFINITY;         // NaN is never drawn; -0 and +0 are one logit
}
template <class T> static __device__ __forceinline__ float logit_at(const T* z, int i) { return clean(z[i]); }

static __device__ __forceinline__ u64 place_of(float z, int i) {     // falling order of candidates = falling order of these numbers
    const unsigned b = __float_as_uint(z), k = b & 0x80000000u ? ~b : b | 0x80000000u;
    return (u64)k << 32 | (unsigned)~i;
}
static __device__ __forceinline__ float logit_of(u64 place) {
    const unsigned k = (unsigned)(place >> 32);
    return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
static __device__ __forceinline__ int index_of(u64 place) { return (int)~(unsigned)place; }
static __device__ __forceinline__ u64 larger(u64 a, u64 b) { return a > b ? a : b; }

// floor(u n) for 0 < u < 1, exactly: 24 bits of u times 64 bits of n
static __device__ __forceinline__ u64 floor_of_product(float u, u64 n) {
    const unsigned b = __float_as_uint(u), e = b >> 23;
    const u64 m = e ? (b & 0x7fffffu) | 0x800000u : b;
    const int shift = 150 - (int)(e ? e : 1);                  // u = m 2^-shift, shift >= 24
    const u64 lo = m * n, hi = __umul64hi(m, n);
    return shift >= 128 ? 0 : shift >= 64 ? hi >> (shift - 64) : lo >> shift | hi << (64 - shift);
}

// 2^d for d <= 0 in fp64: 2^(j / 256) from a table, the remainder (at most 1/512 away) by the exponential's series to the fourth power (the fifth is
// below 4e-17), the whole part by the exponent.  A third of the instructions of the library's exp2, which a row of 10^5 logits feels.
struct Weigher {
    const double* table;       // 2^(j / SM_TABLE)
    double a, unit;            // log2(e) / T, 2^s
    float zmax, af;            // bins per logit
    __device__ __forceinline__ u64 fixed(float z) const {
        const double d = z == zmax ? 0.0 : fmax(((double)z - (double)zmax) * a, -256.0);
        const double r = __builtin_rint(d * SM_TABLE);
        const int j = (int)r;
        const double f = fma(r, -1.0 / SM_TABLE, d);
        const double p = f * fma(f, fma(f, fma(f, 0.009618129107628477, 0.05550410866482158), 0.2402265069591007), 0.6931471805599453);
        const double t = table[j & (SM_TABLE - 1)];
        return rounded(ldexp(fma(t, p, t), j >> 8) * unit);
    }
    static __device__ __forceinline__ u64 rounded(double x) {        // to the nearest integer, 0 <= x <= 2^50
        return (u64)__double_as_longlong(x + 4503599627370496.0) & 0xfffffffffffffull;
    }
    __device__ __forceinline__ int bin(float z) const {               // 0 at the maximum, monotone in z
        if (z == zmax) return 0;
        const float y = (zmax - z) * af;
        return y < (float)(SM_BINS - 1) ? (int)y : SM_BINS - 1;
    }
};
// x can lie in one of the bins up to `bin`: false only where it does not (one comparison; who finds something asks Weigher::bin).  All can where that is the
// last bin, which also takes the distances that fp32 does not hold: nothing is at least NaN.
struct Near {
    float zmax, af, most;
    __device__ __forceinline__ Near(const Weigher& w, int bin) : zmax(w.zmax), af(w.af), most(bin < SM_BINS - 1 ? (float)(bin + 1) : NAN) {}
    __device__ __forceinline__ bool operator()(float x) const { return !((zmax - x) * af >= most); }
};
static_assert(SM_TABLE == 256, "Weigher::fixed takes the low eight bits");

struct Limits {
    double temperature, top_p, min_p;
    long top_k;
    float u;
    __device__ __forceinline__ Limits(const SampleArgs& a, int row) {
        temperature = a.temperature_rows ? (double)a.temperature_rows[row] : a.temperature;
        top_k = a.top_k_rows ? (long)a.top_k_rows[row] : (long)a.top_k;
        top_p = a.top_p_rows ? (double)a.top_p_rows[row] : a.top_p;
        min_p = a.min_p_rows ? (double)a.min_p_rows[row] : a.min_p;
        u = a.u[row];
    }
    __device__ __forceinline__ bool greedy() const { return !(temperature > 0.0) || top_k == 1; }
    __device__ __forceinline__ bool by_count(int V) const { return top_k > 1 && top_k < V; }
    __device__ __forceinline__ bool by_mass() const { return top_p < 1.0; }
    // the head's mass: the first candidate at which the sum reaches this is the last that top_p keeps
    __device__ __forceinline__ u64 head(u64 total) const {
        const u64 g = top_p > 0.0 ? (u64)ceil(top_p * (double)total) : 1;
        return g < 1 ? (u64)1 : g > total ? total : g;
    }
    // cumulated > u total  <=>  cumulated >= floor(u total) + 1
    __device__ __forceinline__ u64 goal(u64 total) const { return u >= 1.f ? total : (u > 0.f ? floor_of_product(u, total) : 0) + 1; }
    __device__ __forceinline__ u64 least(double unit) const { return min_p > 0.0 ? Weigher::rounded(fmin(min_p, 1.0) * unit) : 0; }
};

static __device__ __forceinline__ Weigher weigher(const double* table, float zmax, double temperature, int V) {
    Weigher w;
    w.table = table;
    w.zmax = zmax;
    w.a = 1.4426950408889634 / temperature;
    w.unit = (double)(1ull << min(50, 62 - (32 - __clz(V))));
    w.af = (float)(w.a * ((SM_BINS - 1) / SM_RANGE));
    return w;
}

struct Powers {
    double v[SM_TABLE];
    constexpr Powers() : v() {
        for (int j = 0; j < SM_TABLE; ++j) {      // the series of exp(j / 256 ln 2), smallest term first
            double x = 1.0;
            for (int n = 24; n > 0; --n) x = 1.0 + x * (j * (0.6931471805599453 / SM_TABLE)) / n;
            v[j] = x;
        }
    }
};
__device__ const Powers POWERS;
static __device__ __forceinline__ void fill_table(double* table, int tid, int nt) {
    for (int i = tid; i < SM_TABLE; i += nt) table[i] = POWERS.v[i];
}

static __device__ __forceinline__ void answer(const SampleArgs& a, int row, int token, float logp) {
    a.tokens[row] = token;
    if (a.logp) a.logp[row] = logp;
}
static __device__ __forceinline__ float share(u64 part, u64 total) { return (float)log((double)part / (double)total); }

// ---- one wave ---------------------------------------------------------------------------------------------------------------
static __device__ __forceinline__ u64 wave_sum(u64 x) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o);
    return x;
}
static __device__ __forceinline__ u64 wave_scan(u64 x) {             // inclusive
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) { const u64 y = __shfl_up(x, o); if (lane >= o) x += y; }
    return x;
}
// falling order over the wave
static __device__ __forceinline__ u64 wave_sort(u64 x) {
    const int lane = threadIdx.x & 63;
#pragma unroll 1
    for (int size = 2; size <= 64; size <<= 1)
#pragma unroll 1
        for (int o = size >> 1; o > 0; o >>= 1) {
            const u64 y = __shfl_xor(x, o);
            const bool want_large = ((lane & o) == 0) == ((lane & size) == 0);
            x = want_large == (x > y) ? x : y;
        }
    return x;
}

// All candidates that can be kept, one per lane (0: none), drawn from by one wave.  w: of the row's maximum.
// head: the mass that top_p keeps, where the list is the head of a longer row (0: the list is all that top_k left, or all there is).
static __device__ __forceinline__ void wave_draw(const SampleArgs& a, int row, const Limits& lim, const Weigher& w, u64 mine, u64 head) {
    const int lane = threadIdx.x & 63;
    u64 p = wave_sort(mine);
    u64 x = p ? w.fixed(logit_of(p)) : 0;
    if (lim.by_count(a.V) && lane >= lim.top_k) x = p = 0;
    if (lim.by_mass()) {
        const u64 incl = wave_scan(x), total = __shfl(incl, 63);
        if (incl - x >= (head ? head : lim.head(total))) x = p = 0;
    }
    if (x < lim.least(w.unit)) x = p = 0;
    // vocabulary order: lowest index first = largest inverted index first (a dropped candidate's 0 goes last)
    p = wave_sort(p << 32 | p >> 32);
    x = p ? w.fixed(logit_of(p << 32 | p >> 32)) : 0;
    const u64 incl = wave_scan(x), total = __shfl(incl, 63), goal = lim.goal(total);
    if (incl - x < goal && goal <= incl) answer(a, row, (int)~(unsigned)(p >> 32), share(x, total));
}

// ---- one workgroup ----------------------------------------------------------------------------------------------------------
struct Shared {
    u64 mass[SM_BINS];
    unsigned count[SM_BINS];
    u64 place[SM_CAP];
    double table[SM_TABLE];
    u64 red[32];
    u64 out[4];
    unsigned n;
};

template <int NT> static __device__ __forceinline__ u64 block_sum(u64 x, Shared& s) {
    x = wave_sum(x);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s.red[threadIdx.x >> 6] = x;
    __syncthreads();
    x = 0;
#pragma unroll
    for (int i = 0; i < NT / 64; ++i) x += s.red[i];
    return x;
}
template <int NT> static __device__ __forceinline__ u64 block_max(u64 x, Shared& s) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x = larger(x, __shfl_xor(x, o));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s.red[threadIdx.x >> 6] = x;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NT / 64; ++i) x = larger(x, s.red[i]);
    return x;
}
// inclusive, and the sum over all
template <int NT> static __device__ __forceinline__ u64 block_scan(u64 x, u64& total, Shared& s) {
    x = wave_scan(x);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) s.red[threadIdx.x >> 6] = x;
    __syncthreads();
    total = 0;
    const int wave = threadIdx.x >> 6;
    u64 before = 0;
#pragma unroll
    for (int i = 0; i < NT / 64; ++i) { const u64 y = s.red[i]; if (i < wave) before += y; total += y; }
    return x + before;
}
// falling order over the workgroup, one number per thread; buf: NT numbers
template <int NT> static __device__ __forceinline__ u64 block_sort(u64 x, u64* buf) {
    const int tid = threadIdx.x;
    for (int size = 2; size <= NT; size <<= 1)
        for (int o = size >> 1; o > 0; o >>= 1) {
            u64 y;
            if (o >= 64) {
                __syncthreads();
                buf[tid] = x;
                __syncthreads();
                y = buf[tid ^ o];
            } else {
                y = __shfl_xor(x, o);
            }
            const bool want_large = ((tid & o) == 0) == ((tid & size) == 0);
            x = want_large == (x > y) ? x : y;
        }
    return x;
}

// The first entry of a table of n at which the running sum reaches `target` (>= 1, at most the table's sum): (entry, sum before it).
template <int NT, class At> static __device__ __forceinline__ void reach(int n, u64 target, At at, Shared& s, int& entry, u64& before) {
    const int tid = threadIdx.x, per = (n + NT - 1) / NT, lo = min(n, tid * per), hi = min(n, lo + per);
    u64 mine = 0;
    for (int i = lo; i < hi; ++i) mine += at(i);
    u64 total;
    const u64 incl = block_scan<NT>(mine, total, s);
    if (tid == 0) { s.out[0] = (u64)(n - 1); s.out[1] = 0; }      // (an entry of the table whatever the target)
    __syncthreads();
    u64 run = incl - mine;
    if (run < target && target <= incl) {
        for (int i = lo; i < hi; ++i) {
            const u64 v = at(i);
            if (run + v >= target) { s.out[0] = (u64)i; s.out[1] = run; break; }
            run += v;
        }
    }
    __syncthreads();
    entry = (int)s.out[0];
    before = s.out[1];
    __syncthreads();
}

// The number at which the running sum of `value` over the numbers, largest first, reaches target: eight bits at a time, `bits` of them.
// each(f): calls f(number, value) for this thread's share of the candidates.
template <int NT, class Each> static __device__ __forceinline__ u64 search(u64 target, int bits, Each each, Shared& s) {
    u64 found = 0;
    for (int shift = bits - 8; shift >= 0; shift -= 8) {
        __syncthreads();
        for (int i = threadIdx.x; i < 256; i += NT) s.mass[i] = 0;
        __syncthreads();
        each([&](u64 number, u64 value) {
            if (shift == bits - 8 || (number >> (shift + 8)) == (found >> (shift + 8))) atomicAdd(&s.mass[255 - ((number >> shift) & 255)], value);
        });
        __syncthreads();
        int digit; u64 before;
        reach<NT>(256, target, [&](int i) { return s.mass[i]; }, s, digit, before);
        target -= before;
        found |= (u64)(255 - digit) << shift;
    }
    return found;
}

// f(logit as it is, index) for this thread's share of [lo, hi) of a row: sixteen bytes at a time, four loads in flight
template <int NT, class T, class F> static __device__ __forceinline__ void each_raw(const T* z, int lo, int hi, F f) {
    constexpr int EL = 16 / (int)sizeof(T), AHEAD = 4;
    typedef T V __attribute__((ext_vector_type(EL), aligned(sizeof(T))));
    for (int i0 = lo + (int)threadIdx.x * EL; i0 < hi; i0 += AHEAD * NT * EL) {
        V x[AHEAD];
#pragma unroll
        for (int n = 0; n < AHEAD; ++n)
            if (i0 + n * NT * EL + EL <= hi) x[n] = *(const V*)(z + i0 + n * NT * EL);
#pragma unroll
        for (int n = 0; n < AHEAD; ++n) {
            const int i = i0 + n * NT * EL;
            if (i + EL <= hi) {
#pragma unroll
                for (int e = 0; e < EL; ++e) f((float)x[n][e], i + e);
            } else {
                for (int e = i; e < hi; ++e) f((float)z[e], e);
            }
        }
    }
}
// f(logit, index) for this thread's share, one at a time with the next on its way: for bodies of many instructions (a draw is over in the time that
// a hundred cache lines of instructions take to arrive, so unrolling them costs more than it hides)
template <int NT, class T, class F> static __device__ __forceinline__ void each_logit(const T* z, int lo, int hi, F f) {
    int i = lo + (int)threadIdx.x;
    float next = i < hi ? logit_at(z, i) : 0.f;
#pragma unroll 1
    for (; i < hi; i += NT) {
        const float x = next;
        next = i + NT < hi ? logit_at(z, i + NT) : 0.f;
        f(x, i);
    }
}
// found(logit, index) for the few logits of this thread's share (each_raw's) that near(logit) holds for
template <int NT, class T, class Near, class Found> static __device__ __forceinline__ void each_near(const T* z, int lo, int hi, Near near, Found found) {
    constexpr int EL = 16 / (int)sizeof(T), AHEAD = 32 / EL;
    typedef T V __attribute__((ext_vector_type(EL), aligned(sizeof(T))));
    for (int i0 = lo + (int)threadIdx.x * EL; i0 < hi; i0 += AHEAD * NT * EL) {
        V x[AHEAD];
        unsigned hits = 0;
#pragma unroll
        for (int n = 0; n < AHEAD; ++n)
            if (i0 + n * NT * EL + EL <= hi) x[n] = *(const V*)(z + i0 + n * NT * EL);
#pragma unroll
        for (int n = 0; n < AHEAD; ++n) {
            const int i = i0 + n * NT * EL;
            if (i + EL <= hi) {
#pragma unroll
                for (int e = 0; e < EL; ++e) hits |= (near((float)x[n][e]) ? 1u : 0u) << (n * EL + e);
            } else if (i < hi) {
                for (int e = 0; e < hi - i; ++e) hits |= 1u << (n * EL + e);      // (the row's end: looked at one by one below)
            }
        }
        while (hits) {
            const int bit = __ffs((int)hits) - 1, i = i0 + bit / EL * NT * EL + bit % EL;
            hits &= hits - 1;
            const float v = logit_at(z, i);
            if (near(v)) found(v, i);
        }
    }
}

// draw_listed for lists that are too long to be sorted
template <int NT>
static __device__ __attribute__((noinline)) void search_listed(SampleArgs a, int row, Limits lim, Weigher w, int n, u64 head, Shared& s) {
    const int tid = threadIdx.x;
    auto each = [&](auto f) { for (int i = tid; i < n; i += NT) f(s.place[i], w.fixed(logit_of(s.place[i]))); };
    u64 cut = 0, m = 0;
    if (lim.by_count(a.V)) cut = search<NT>((u64)min(lim.top_k, (long)n), 64, [&](auto f) { each([&](u64 p, u64) { f(p, (u64)1); }); }, s);
    if (lim.by_mass()) {
        each([&](u64 p, u64 x) { if (p >= cut) m += x; });
        const u64 total = block_sum<NT>(m, s);
        cut = search<NT>(head ? head : lim.head(total), 64, [&](auto f) { each([&](u64 p, u64 x) { if (p >= cut) f(p, x); }); }, s);
    }
    const u64 least = lim.least(w.unit);
    m = 0;
    each([&](u64 p, u64 x) { if (p >= cut && x >= least) m += x; });
    const u64 total = block_sum<NT>(m, s);
    const u64 at = search<NT>(lim.goal(total), 32, [&](auto f) { each([&](u64 p, u64 x) { if (p >= cut && x >= least) f((u64)(unsigned)p, x); }); }, s);
    const int token = (int)~(unsigned)at;
    each([&](u64 p, u64 x) { if (index_of(p) == token) answer(a, row, token, share(x, total)); });
}

// Every candidate that can be kept is in s.place[0 .. n): draw.  head: see wave_draw.
template <int NT> static __device__ void draw_listed(const SampleArgs& a, int row, const Limits& lim, const Weigher& w, int n, u64 head, Shared& s) {
    const int tid = threadIdx.x;
    if (n <= 64) {
        if (tid < 64) wave_draw(a, row, lim, w, tid < n ? s.place[tid] : 0, head);
        return;
    }
    if (n <= NT) {
        u64* buf = s.mass;                        // (NT <= SM_BINS)
        u64 total;
        u64 p = block_sort<NT>(tid < n ? s.place[tid] : 0, buf);
        u64 x = p ? w.fixed(logit_of(p)) : 0;
        if (lim.by_count(a.V) && tid >= lim.top_k) x = p = 0;
        if (lim.by_mass()) {
            const u64 incl = block_scan<NT>(x, total, s);
            if (incl - x >= (head ? head : lim.head(total))) x = p = 0;
        }
        if (x < lim.least(w.unit)) x = p = 0;
        p = block_sort<NT>(p << 32 | p >> 32, buf);
        x = p ? w.fixed(logit_of(p << 32 | p >> 32)) : 0;
        const u64 incl = block_scan<NT>(x, total, s), goal = lim.goal(total);
        if (incl - x < goal && goal <= incl) answer(a, row, (int)~(unsigned)(p >> 32), share(x, total));
        return;
    }
    search_listed<NT>(a, row, lim, w, n, head, s);
}

// The cut in a list of the candidates of one bin: the one at which the running sum (of masses, or of candidates) reaches target.
template <int NT> static __device__ __forceinline__ u64 cut_in_list(const Weigher& w, bool masses, u64 target, int n, Shared& s) {
    const int tid = threadIdx.x;
    if (n <= NT) {
        u64 total;
        const u64 p = block_sort<NT>(tid < n ? s.place[tid] : 0, s.mass), x = p ? (masses ? w.fixed(logit_of(p)) : 1) : 0;
        const u64 incl = block_scan<NT>(x, total, s);
        __syncthreads();
        if (incl - x < target && target <= incl) s.out[2] = p;
        __syncthreads();
        return s.out[2];
    }
    return search<NT>(target, 64, [&](auto f) {
        for (int i = tid; i < n; i += NT) f(s.place[i], masses ? w.fixed(logit_of(s.place[i])) : (u64)1);
    }, s);
}

// The draw within [lo, hi) of a row, of the candidates not behind the cut: target as in reach, total for the share.  Ranges of the range, one per
// wave, until every thread has one index.  total = 0: neither is known yet, the range is the whole row; the first ranges' masses give both.
template <int NT, class T>
static __device__ void draw_range(const SampleArgs& a, int row, const T* z, const Limits& lim, const Weigher& w, u64 cut, u64 least, int lo, int hi, u64 target, u64 total,
                                  Shared& s) {
    constexpr int NW = NT / 64;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    auto mass_of = [&](float x, int i) {
        if (x == -INFINITY || place_of(x, i) < cut) return (u64)0;
        const u64 f = w.fixed(x);
        return f >= least ? f : (u64)0;
    };
    bool first = total == 0;
    while (hi - lo > NT || first) {
        const int per = (hi - lo + NW - 1) / NW, x0 = min(hi, lo + wave * per), x1 = min(hi, x0 + per);
        u64 m = 0;
        float next = x0 + lane < x1 ? logit_at(z, x0 + lane) : 0.f;
#pragma unroll 1
        for (int i = x0 + lane; i < x1; i += 64) {
            const float x = next;
            next = i + 64 < x1 ? logit_at(z, i + 64) : 0.f;
            m += mass_of(x, i);
        }
        m = wave_sum(m);
        __syncthreads();
        if (lane == 0) s.mass[wave] = m;
        __syncthreads();
        if (first) {
            for (int i = 0; i < NW; ++i) total += s.mass[i];
            target = lim.goal(total);
            first = false;
        }
        int part; u64 before;
        reach<NT>(NW, target, [&](int i) { return s.mass[i]; }, s, part, before);
        target -= before;
        lo = min(hi, lo + part * per);
        hi = min(hi, lo + per);
    }
    const u64 x = lo + tid < hi ? mass_of(logit_at(z, lo + tid), lo + tid) : 0;
    u64 all;
    const u64 incl = block_scan<NT>(x, all, s);
    if (incl - x < target && target <= incl) answer(a, row, lo + tid, share(x, total));
}

// ---- the row in one workgroup -----------------------------------------------------------------------------------------------
// The cut over the whole row, for bins that hold more than a list can.
template <int NT, class T> static __device__ __forceinline__ u64 cut_in_row(const T* z, int V, const Weigher& w, u64 cut, bool masses, u64 target, Shared& s) {
    return search<NT>(target, 64, [&](auto f) {
        each_logit<NT>(z, 0, V, [&](float x, int i) {
            if (x == -INFINITY) return;
            const u64 p = place_of(x, i);
            if (p >= cut) f(p, masses ? w.fixed(x) : (u64)1);
        });
    }, s);
}

template <class T, int NT> static __device__ __attribute__((noinline)) void row_draw(SampleArgs a, int row, const T* z, Limits lim, Weigher w, Shared& s) {
    const int tid = threadIdx.x, V = a.V;
    u64 cut = 0;                                  // kept: place >= cut

    auto gather = [&](int lo, int hi) {           // candidates of bins lo..hi that are not behind the cut; their number
        __syncthreads();
        if (tid == 0) s.n = 0;
        __syncthreads();
        each_logit<NT>(z, 0, V, [&](float x, int i) {
            if (x == -INFINITY) return;
            const int b = w.bin(x);
            const u64 p = place_of(x, i);
            if (b < lo || b > hi || p < cut) return;
            const unsigned at = atomicAdd(&s.n, 1u);
            if (at < SM_CAP) s.place[at] = p;
        });
        __syncthreads();
        return min((int)s.n, SM_CAP);
    };
    // counts (masses too) of the candidates not behind the cut, by bin; the number of all
    auto histogram = [&](bool masses) {
        __syncthreads();
        for (int i = tid; i < SM_BINS; i += NT) { s.mass[i] = 0; s.count[i] = 0; }
        __syncthreads();
        each_logit<NT>(z, 0, V, [&](float x, int i) {
            if (x == -INFINITY || place_of(x, i) < cut) return;
            const int b = w.bin(x);
            atomicAdd(&s.count[b], 1u);
            if (masses) atomicAdd(&s.mass[b], w.fixed(x));
        });
        __syncthreads();
        u64 c = 0;
        for (int i = tid; i < SM_BINS; i += NT) c += s.count[i];
        return block_sum<NT>(c, s);
    };

    if (lim.by_count(V)) {
        if ((u64)lim.top_k < histogram(false)) {
            int bin; u64 before;
            reach<NT>(SM_BINS, (u64)lim.top_k, [&](int i) { return (u64)s.count[i]; }, s, bin, before);
            const unsigned here = s.count[bin];
            if (before + here <= SM_CAP) return draw_listed<NT>(a, row, lim, w, gather(0, bin), 0, s);
            if (here <= SM_CAP) cut = cut_in_list<NT>(w, false, (u64)lim.top_k - before, gather(bin, bin), s);
            else cut = cut_in_row<NT>(z, V, w, 0, false, (u64)lim.top_k, s);
        }
    }
    if (lim.by_mass()) {
        histogram(true);
        u64 m = 0;
        for (int i = tid; i < SM_BINS; i += NT) m += s.mass[i];
        const u64 target = lim.head(block_sum<NT>(m, s));
        int bin; u64 before;
        reach<NT>(SM_BINS, target, [&](int i) { return s.mass[i]; }, s, bin, before);
        const unsigned here = s.count[bin];
        u64 ahead = 0;
        for (int i = tid; i < bin; i += NT) ahead += s.count[i];
        ahead = block_sum<NT>(ahead, s);
        if (cut == 0 && ahead + here <= NT) return draw_listed<NT>(a, row, lim, w, gather(0, bin), target, s);
        if (here <= SM_CAP) cut = cut_in_list<NT>(w, true, target - before, gather(bin, bin), s);
        else cut = cut_in_row<NT>(z, V, w, cut, true, target, s);
    }
    draw_range<NT>(a, row, z, lim, w, cut, lim.least(w.unit), 0, V, 0, 0, s);
}

// top_k of a row without a pass that counts: of the maxima that the threads found in their shares of the row, the top_k-th largest has at least top_k
// candidates not behind it and, the shares being small, hardly more.  A histogram of these NT maxima alone gives its bin; the candidates down to that
// bin are the list.  False (nothing done) where the list would be too long or too few threads found a candidate.
template <class T, int NT>
static __device__ __forceinline__ bool few_draw(const SampleArgs& a, int row, const T* z, const Limits& lim, const Weigher& w, float mine, Shared& s) {
    const int tid = threadIdx.x;
    if (lim.top_k > NT) return false;
    for (int i = tid; i < SM_BINS; i += NT) s.count[i] = 0;
    if (tid == 0) s.n = 0;
    __syncthreads();
    if (mine != -INFINITY) atomicAdd(&s.count[w.bin(mine)], 1u);
    const u64 found = block_sum<NT>(mine != -INFINITY, s);
    if (found < (u64)lim.top_k) return false;
    int bin; u64 before;
    reach<NT>(SM_BINS, (u64)lim.top_k, [&](int i) { return (u64)s.count[i]; }, s, bin, before);
    if (mine != -INFINITY && w.bin(mine) <= bin) {
        each_near<NT>(z, 0, a.V, Near(w, bin), [&](float x, int i) {      // its share again
            if (x == -INFINITY || w.bin(x) > bin) return;
            const unsigned at = atomicAdd(&s.n, 1u);
            if (at < SM_CAP) s.place[at] = place_of(x, i);
        });
    }
    __syncthreads();
    const unsigned n = s.n;
    if (n > SM_CAP) return false;
    draw_listed<NT>(a, row, lim, w, (int)n, 0, s);
    return true;
}

template <class T, int NT> __global__ __launch_bounds__(NT) void sample_row_kernel(SampleArgs a) {
    __shared__ Shared s;
    const int tid = threadIdx.x, row = blockIdx.x;
    const T* z = (const T*)a.z + row * a.z_b;
    const Limits lim(a, row);
    float mine = -INFINITY;                       // (a NaN loses every comparison)
    each_raw<NT>(z, 0, a.V, [&](float x, int) { mine = fmaxf(mine, x); });
    const float zmax = logit_of(block_max<NT>(place_of(mine + 0.f, 0), s));
    if (zmax == -INFINITY) { if (tid == 0) answer(a, row, -1, -INFINITY); return; }        // nothing to draw from
    if (lim.greedy()) {
        u64 best = 0;
        each_logit<NT>(z, 0, a.V, [&](float x, int i) { best = larger(best, place_of(x, i)); });
        best = block_max<NT>(best, s);
        if (tid == 0) answer(a, row, index_of(best), 0.f);
        return;
    }
    fill_table(s.table, tid, NT);
    __syncthreads();
    const Weigher w = weigher(s.table, zmax, lim.temperature, a.V);
    if (lim.by_count(a.V) && few_draw<T, NT>(a, row, z, lim, w, mine, s)) return;
    row_draw<T, NT>(a, row, z, lim, w, s);
}

// rows of at most 64 logits: a wave each
constexpr int SW_THREADS = 256;
template <class T> __global__ __launch_bounds__(SW_THREADS) void sample_wave_kernel(SampleArgs a) {
    __shared__ double table[SM_TABLE];
    fill_table(table, threadIdx.x, SW_THREADS);
    __syncthreads();
    const int row = blockIdx.x * (SW_THREADS / 64) + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (row >= a.B) return;
    const Limits lim(a, row);
    const float x = lane < a.V ? logit_at((const T*)a.z + row * a.z_b, lane) : -INFINITY;
    u64 best = lane < a.V ? place_of(x, lane) : 0;
    const u64 mine = x > -INFINITY ? best : 0;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) best = larger(best, __shfl_xor(best, o));
    const float zmax = logit_of(best);
    if (zmax == -INFINITY) { if (lane == 0) answer(a, row, -1, -INFINITY); return; }
    if (lim.greedy()) { if (lane == 0) answer(a, row, index_of(best), 0.f); return; }
    wave_draw(a, row, lim, weigher(table, zmax, lim.temperature, a.V), mine, 0);
}

// ---- the row in slices ------------------------------------------------------------------------------------------------------
constexpr int SL_THREADS = 512, SM_CHUNK = SL_THREADS, SM_CHUNKS = SM_MOST / SM_CHUNK;

// How a row is drawn once its histogram is known: LISTED every candidate that can be kept goes to the list, CUT only those of the bin of the cut
// (the bins before it are kept whole), WHOLE everything is kept, ALONE a bin is longer than the list: one workgroup takes the row by itself.
enum Mode : int { LISTED, CUT, WHOLE, ALONE };

constexpr int SM_GROUP = SM_BINS / 64;
// workspace of one row
struct RowSpace {
    u64 mass[SM_BINS], mass_of[64];        // by bin, and by groups of SM_GROUP bins
    unsigned count[SM_BINS], count_of[64];
    u64 place[SM_CAP];
    u64 slice_max[SM_SLICES], chunk_mass[SM_CHUNKS];
    u64 target, head;              // of the first slice's verdict: mass to reach within the bin, mass that top_p keeps
    int mode;
    unsigned n;
};

// slices of whole chunks (the masses are kept by chunk, so that the draw looks into one of them alone)
static __device__ __forceinline__ void slice_of(int V, int S, int i, int& lo, int& hi) {
    const int per = ((V + S - 1) / S + SM_CHUNK - 1) / SM_CHUNK * SM_CHUNK;
    lo = min(V, i * per);
    hi = min(V, lo + per);
}

template <class T> __global__ __launch_bounds__(SL_THREADS) void sample_max_kernel(SampleArgs a, RowSpace* space, int S) {
    __shared__ u64 red[SL_THREADS / 64];
    const int tid = threadIdx.x, row = blockIdx.x / S, slice = blockIdx.x - row * S;
    RowSpace& r = space[row];
    for (int i = slice * SL_THREADS + tid; i < SM_BINS; i += S * SL_THREADS) { r.mass[i] = 0; r.count[i] = 0; }
    if (slice == 0 && tid < 64) { r.mass_of[tid] = 0; r.count_of[tid] = 0; }
    if (slice == 0 && tid == 0) r.n = 0;
    int lo, hi;
    slice_of(a.V, S, slice, lo, hi);
    u64 best = 0;
    each_logit<SL_THREADS>((const T*)a.z + row * a.z_b, lo, hi, [&](float x, int i) { best = larger(best, place_of(x, i)); });
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) best = larger(best, __shfl_xor(best, o));
    if ((tid & 63) == 0) red[tid >> 6] = best;
    __syncthreads();
    if (tid == 0) {
        for (int i = 1; i < SL_THREADS / 64; ++i) best = larger(best, red[i]);
        r.slice_max[slice] = best;
    }
}

// (every wave by itself: a barrier costs more than the reads)
static __device__ __forceinline__ u64 row_max(const RowSpace& r, int S) {
    const int lane = threadIdx.x & 63;
    u64 x = lane < S ? r.slice_max[lane] : 0;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x = larger(x, __shfl_xor(x, o));
    return x;
}
static_assert(SM_SLICES <= 64, "a lane for each slice");

// The bin in which the running sum (masses, or counts) over the row's bins reaches target, the sums of both before it.  Every wave by itself.
static __device__ __forceinline__ int reach_bin(const RowSpace& r, bool masses, u64 target, u64& mass_before, u64& count_before) {
    const int lane = threadIdx.x & 63;
    u64 m = r.mass_of[lane], c = r.count_of[lane], ms = wave_scan(m), cs = wave_scan(c);
    u64 hit = __ballot((masses ? ms : cs) >= target);
    const int group = hit ? __ffsll((long long)hit) - 1 : 63;
    mass_before = __shfl(ms - m, group);
    count_before = __shfl(cs - c, group);
    m = lane < SM_GROUP ? r.mass[group * SM_GROUP + lane] : 0;
    c = lane < SM_GROUP ? r.count[group * SM_GROUP + lane] : 0;
    ms = mass_before + wave_scan(m);
    cs = count_before + wave_scan(c);
    hit = __ballot((masses ? ms : cs) >= target);
    const int at = hit ? __ffsll((long long)hit) - 1 : SM_GROUP - 1;
    mass_before = __shfl(ms - m, at);
    count_before = __shfl(cs - c, at);
    return group * SM_GROUP + at;
}

template <class T> __global__ __launch_bounds__(SL_THREADS) void sample_histogram_kernel(SampleArgs a, RowSpace* space, int S) {
    __shared__ Shared s;
    const int tid = threadIdx.x, row = blockIdx.x / S, slice = blockIdx.x - row * S;
    RowSpace& r = space[row];
    const Limits lim(a, row);
    const bool masses = !lim.by_count(a.V);      // (with top_k the first cut is one of counts)
    const float zmax = logit_of(row_max(r, S));
    if (zmax == -INFINITY || lim.greedy() || (!lim.by_count(a.V) && !lim.by_mass())) return;
    if (masses) fill_table(s.table, tid, SL_THREADS);
    for (int i = tid; i < SM_BINS; i += SL_THREADS) { s.mass[i] = 0; s.count[i] = 0; }
    __syncthreads();
    const Weigher w = weigher(s.table, zmax, lim.temperature, a.V);
    int lo, hi;
    slice_of(a.V, S, slice, lo, hi);
    each_logit<SL_THREADS>((const T*)a.z + row * a.z_b, lo, hi, [&](float x, int) {
        if (x == -INFINITY) return;
        const int b = w.bin(x);
        atomicAdd(&s.count[b], 1u);
        if (masses) atomicAdd(&s.mass[b], w.fixed(x));
    });
    __syncthreads();
    constexpr int PER = SM_BINS / SL_THREADS;
    u64 m = 0;
    unsigned c = 0;
    for (int i = tid; i < SM_BINS; i += SL_THREADS)
        if (s.count[i]) { atomicAdd(&r.count[i], s.count[i]); if (masses) atomicAdd(&r.mass[i], s.mass[i]); }
    for (int i = tid * PER; i < (tid + 1) * PER; ++i) { c += s.count[i]; m += s.mass[i]; }
#pragma unroll
    for (int o = 1; o < SM_GROUP / PER; o <<= 1) { m += __shfl_xor(m, o); c += __shfl_xor(c, o); }
    if (tid % (SM_GROUP / PER) == 0 && c) {
        atomicAdd(&r.count_of[tid * PER / SM_GROUP], c);
        if (masses) atomicAdd(&r.mass_of[tid * PER / SM_GROUP], m);
    }
}

// this workgroup's candidates, s.place[0 .. s.n), to the row's list
template <int NT> static __device__ __forceinline__ void append(RowSpace& r, Shared& s) {
    const int tid = threadIdx.x;
    __syncthreads();
    const unsigned n = min(s.n, (unsigned)SM_CAP);
    if (tid == 0) s.out[0] = n ? atomicAdd(&r.n, n) : 0;
    __syncthreads();
    const unsigned at = (unsigned)s.out[0];
    for (unsigned i = tid; i < n && at + i < SM_CAP; i += NT) r.place[at + i] = s.place[i];
}

template <class T> __global__ __launch_bounds__(SL_THREADS) void sample_slice_kernel(SampleArgs a, RowSpace* space, int S) {
    constexpr int NT = SL_THREADS;
    __shared__ Shared s;
    const int tid = threadIdx.x, row = blockIdx.x / S, slice = blockIdx.x - row * S, V = a.V;
    RowSpace& r = space[row];
    const Limits lim(a, row);
    const T* z = (const T*)a.z + row * a.z_b;
    const u64 best = row_max(r, S);
    const float zmax = logit_of(best);
    const bool first = slice == 0 && tid == 0;
    if (zmax == -INFINITY || lim.greedy()) return;
    const Weigher w = weigher(s.table, zmax, lim.temperature, V);

    // every slice comes to the same verdict
    int mode = WHOLE, bin = SM_BINS;
    u64 target = 0, head = 0;
    if (lim.by_count(V) || lim.by_mass()) {
        const int lane = tid & 63;
        const u64 all = wave_sum(r.count_of[lane]), mass = wave_sum(r.mass_of[lane]);
        u64 ahead, before;
        if (lim.by_count(V)) {
            if ((u64)lim.top_k < all) {
                bin = reach_bin(r, false, (u64)lim.top_k, before, ahead);
                mode = ahead + r.count[bin] <= SM_CAP ? LISTED : ALONE;
            } else {
                mode = lim.by_mass() ? ALONE : WHOLE;      // (fewer candidates than top_k: no masses were counted)
            }
        } else {
            target = head = lim.head(mass);
            bin = reach_bin(r, true, target, before, ahead);
            target -= before;
            const unsigned here = r.count[bin];
            mode = ahead + here <= NT ? LISTED : here <= SM_CAP ? CUT : ALONE;
        }
    }
    if (first) { r.mode = mode; r.target = target; r.head = head; }
    if (mode == ALONE) return;
    int lo, hi;
    slice_of(V, S, slice, lo, hi);
    if (mode == LISTED) {
        // (to LDS first: one addition to the row's counter per workgroup, not one per candidate)
        if (tid == 0) s.n = 0;
        __syncthreads();
        each_near<NT>(z, lo, hi, Near(w, bin), [&](float x, int i) {
            if (x == -INFINITY || w.bin(x) > bin) return;
            const unsigned at = atomicAdd(&s.n, 1u);
            if (at < SM_CAP) s.place[at] = place_of(x, i);
        });
        append<NT>(r, s);
        return;
    }
    if (tid == 0) s.n = 0;
    fill_table(s.table, tid, NT);
    __syncthreads();
    const u64 least = lim.least(w.unit);
    constexpr int EL = SM_CHUNK / 64;             // a wave takes a chunk, a lane eight logits of it
    for (int c = lo + (tid >> 6) * SM_CHUNK; c < hi; c += NT / 64 * SM_CHUNK) {
        float v[EL];
#pragma unroll
        for (int e = 0; e < EL; ++e) {
            const int i = c + e * 64 + (tid & 63);
            v[e] = i < hi ? logit_at(z, i) : -INFINITY;
        }
        u64 m = 0;
#pragma unroll
        for (int e = 0; e < EL; ++e) {
            const int i = c + e * 64 + (tid & 63), b = v[e] == -INFINITY ? SM_BINS + 1 : w.bin(v[e]);
            if (b < bin) {
                const u64 f = w.fixed(v[e]);
                if (f >= least) m += f;
            } else if (b == bin && mode == CUT) {
                const unsigned at = atomicAdd(&s.n, 1u);
                if (at < SM_CAP) s.place[at] = place_of(v[e], i);
            }
        }
        m = wave_sum(m);
        if ((tid & 63) == 0) r.chunk_mass[c / SM_CHUNK] = m;
    }
    if (mode == CUT) append<NT>(r, s);
}

template <class T> __global__ __launch_bounds__(SL_THREADS) void sample_draw_kernel(SampleArgs a, const RowSpace* space, int S) {
    constexpr int NT = SL_THREADS;
    __shared__ Shared s;
    const int tid = threadIdx.x, row = blockIdx.x, V = a.V;
    const RowSpace& r = space[row];
    const Limits lim(a, row);
    const T* z = (const T*)a.z + row * a.z_b;
    const int mode = r.mode, n = mode == LISTED || mode == CUT ? min((int)r.n, SM_CAP) : 0;
    const u64 best = row_max(r, S);
    const float zmax = logit_of(best);
    if (zmax == -INFINITY) { if (tid == 0) answer(a, row, -1, -INFINITY); return; }
    if (lim.greedy()) { if (tid == 0) answer(a, row, index_of(best), 0.f); return; }
    fill_table(s.table, tid, NT);
    const Weigher w = weigher(s.table, zmax, lim.temperature, V);
    const u64 least = lim.least(w.unit);
    for (int i = tid; i < n; i += NT) s.place[i] = r.place[i];
    __syncthreads();
    if (mode == ALONE) return row_draw<T, NT>(a, row, z, lim, w, s);
    if (mode == LISTED) return draw_listed<NT>(a, row, lim, w, n, r.head, s);
    const u64 cut = mode == CUT ? cut_in_list<NT>(w, true, r.target, n, s) : 0;
    __syncthreads();
    const int chunks = (V + SM_CHUNK - 1) / SM_CHUNK;
    u64 m = 0;
    for (int i = tid; i < chunks; i += NT) m += s.mass[i] = r.chunk_mass[i];
    __syncthreads();
    for (int i = tid; i < n; i += NT) {           // (mode CUT) the bin of the cut, as far as it is kept
        const u64 p = s.place[i], f = p >= cut ? w.fixed(logit_of(p)) : 0;
        if (f == 0 || f < least) continue;
        m += f;
        atomicAdd(&s.mass[index_of(p) / SM_CHUNK], f);
    }
    const u64 total = block_sum<NT>(m, s), goal = lim.goal(total);
    u64 before;
    int part;
    reach<NT>(chunks, goal, [&](int i) { return s.mass[i]; }, s, part, before);
    draw_range<NT>(a, row, z, lim, w, cut, least, part * SM_CHUNK, min(V, (part + 1) * SM_CHUNK), goal - before, total, s);
}

static_assert(SM_CHUNKS <= SM_BINS, "the draw keeps the chunks' masses where the histogram was");

template <class T> int by_size(const SampleArgs& a, void* workspace, hipStream_t stream) {
    // (top_k from one scalar: a workgroup finds a short list in two reads of the row, 64 rows of 32000: 34 us in slices, 15 us here)
    const int S = a.top_k > 1 && a.top_k <= 512 && !a.top_k_rows ? 1 : sample_slices(a.B, a.V);
    if (a.V <= 64) {
        hipLaunchKernelGGL(sample_wave_kernel<T>, dim3((unsigned)((a.B + 3) / 4)), dim3(SW_THREADS), 0, stream, a);
    } else if (S > 1) {
        const dim3 grid((unsigned)(a.B * S));
        RowSpace* space = (RowSpace*)workspace;
        hipLaunchKernelGGL(sample_max_kernel<T>, grid, dim3(SL_THREADS), 0, stream, a, space, S);
        // (limits that differ by row are known on the device alone: the histogram's workgroups leave at once where a row needs none)
        if (a.top_k_rows || a.top_p_rows || (a.top_k > 1 && a.top_k < a.V) || a.top_p < 1.0)
            hipLaunchKernelGGL(sample_histogram_kernel<T>, grid, dim3(SL_THREADS), 0, stream, a, space, S);
        hipLaunchKernelGGL(sample_slice_kernel<T>, grid, dim3(SL_THREADS), 0, stream, a, space, S);
        hipLaunchKernelGGL(sample_draw_kernel<T>, dim3((unsigned)a.B), dim3(SL_THREADS), 0, stream, a, space, S);
    } else if (a.V <= 4096) {
        hipLaunchKernelGGL((sample_row_kernel<T, 256>), dim3((unsigned)a.B), dim3(256), 0, stream, a);
    } else {
        hipLaunchKernelGGL((sample_row_kernel<T, 1024>), dim3((unsigned)a.B), dim3(1024), 0, stream, a);
    }
    LAS_LAUNCH_CHECK();
    return LAS_OK;
}

}  // namespace

// Slices of a row: the GPU's 256 CUs twice over shared among the rows, no slice shorter than 4096 logits.  One (a workgroup per row, no workspace) where
// that leaves no more than one.
int sample_slices(int B, int V) {
    if (V > SM_MOST) return 1;
    const int want = B > 0 ? 512 / B : 1, most = V / 4096;
    const int S = want < most ? want : most;
    return S < 2 ? 1 : S > SM_SLICES ? SM_SLICES : S;
}
size_t sample_workspace_bytes(int B, int V) { return V > 64 && sample_slices(B, V) > 1 ? (size_t)B * sizeof(RowSpace) : 0; }

int sample(const SampleArgs& a, int dtype, void* workspace, hipStream_t stream) {
    return dtype == 0 ? by_size<float>(a, workspace, stream) : dtype == 1 ? by_size<__bf16>(a, workspace, stream) : by_size<_Float16>(a, workspace, stream);
}

}  // namespace las
