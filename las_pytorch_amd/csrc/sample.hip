// Drawing a token from logits with temperature, top-k, top-p and min-p, from given random numbers.
//
//   w_v = exp((z_v - max z) / T);  falling order: larger logit first, equal logits by lower index
//   kept: the first top_k of that order; of those, every candidate before which less than top_p of their mass lies; of those, w_v >= min_p
//   token: the first kept index, in vocabulary order, at which the cumulated mass exceeds u times the kept mass
//
// The answer is a whole number that hangs on borders of long sums, so the sums are exact: w is formed in fp64 and held as an integer multiple of
// 2^-s (s = 62 - bits of V, at most 50), and integers add to the same sum in any order — by atomics too.  All three limits keep a head of the
// falling order, so the kept set is "every candidate not behind one cut", and the cut is one 64-bit number: (order-preserving bits of the logit,
// inverted index).  Cuts are found without sorting: a histogram of the distance to the maximum finds the bin that holds the cut, the candidates
// down to that bin go to a list in LDS, and the list is searched digit by digit.  Where a bin holds more than the list, the same search runs
// over the row itself.
#include "las_common.h"
#include "las_kernels.h"
#include <math.h>

namespace las {
namespace {

typedef unsigned long long u64;

constexpr int SM_BINS = 2048, SM_CAP = 4096;
constexpr float SM_RANGE = 51.f;                 // log2 units below the maximum: what lies further weighs nothing (s <= 50)

template <class T> static __device__ __forceinline__ float logit_at(const T* z, long i) {
    const float x = (float)z[i];
    return x == x ? x + 0.f : -INFINITY;         // NaN is never drawn; -0 and +0 are one logit
}

static __device__ __forceinline__ u64 place(float z, int i) {        // falling order of candidates = falling order of these numbers
    const unsigned b = __float_as_uint(z), k = b & 0x80000000u ? ~b : b | 0x80000000u;
    return (u64)k << 32 | (unsigned)~i;
}

// floor(u n) for 0 < u < 1, exactly: 24 bits of u times 64 bits of n
static __device__ __forceinline__ u64 floor_of_product(float u, u64 n) {
    const unsigned b = __float_as_uint(u), e = b >> 23;
    const u64 m = e ? (b & 0x7fffffu) | 0x800000u : b;
    const int shift = 150 - (int)(e ? e : 1);                  // u = m 2^-shift, shift >= 24
    const u64 lo = m * n, hi = __umul64hi(m, n);
    return shift >= 128 ? 0 : shift >= 64 ? hi >> (shift - 64) : lo >> shift | hi << (64 - shift);
}

// What one row needs to weigh a logit.
struct Weigher {
    double a, unit;            // log2(e) / T, 2^s
    float zmax, af;            // bins per logit
    __device__ __forceinline__ double weight(float z) const { return z == zmax ? 1.0 : exp2(((double)z - (double)zmax) * a); }
    __device__ __forceinline__ u64 fixed(double w) const { return (u64)__double2ull_rn(w * unit); }
    __device__ __forceinline__ int bin(float z) const {               // 0 at the maximum, monotone in z
        if (z == zmax) return 0;
        const float y = (zmax - z) * af;
        return y < (float)(SM_BINS - 1) ? (int)y : SM_BINS - 1;
    }
};

struct Shared {
    u64 mass[SM_BINS];
    unsigned count[SM_BINS];
    u64 place[SM_CAP];
    u64 weight[SM_CAP];
    u64 red[32];
    u64 out[4];
    float fred[32];
    unsigned n;
};

template <int NT> static __device__ __forceinline__ u64 block_sum(u64 x, Shared& s) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o);
    if constexpr (NT == 64) return x;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s.red[threadIdx.x >> 6] = x;
    __syncthreads();
    x = 0;
    for (int i = 0; i < NT / 64; ++i) x += s.red[i];
    return x;
}

// The first entry of a table of n (n <= NT * PER) at which the running sum reaches `target` (>= 1, reached somewhere): (entry, sum before it).
template <int NT, class At> static __device__ __forceinline__ void reach(int n, u64 target, At at, Shared& s, int& entry, u64& before) {
    const int tid = threadIdx.x, per = (n + NT - 1) / NT, lo = min(n, tid * per), hi = min(n, lo + per);
    u64 mine = 0;
    for (int i = lo; i < hi; ++i) mine += at(i);
    u64 incl = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) { const u64 y = __shfl_up(incl, o); if ((tid & 63) >= o) incl += y; }
    __syncthreads();
    if ((tid & 63) == 63) s.red[tid >> 6] = incl;
    if (tid == 0) { s.out[0] = (u64)(n - 1); s.out[1] = 0; }      // (an entry of the table whatever the target)
    __syncthreads();
    for (int i = 0; i < (tid >> 6); ++i) incl += s.red[i];
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

// The number at which the running sum of `value` over the numbers, largest first, reaches target: eight bits at a time.
// each(f): calls f(number, value) for this thread's share of the candidates.
template <int NT, class Each> static __device__ __forceinline__ u64 search(u64 target, Each each, Shared& s) {
    u64 found = 0;
    for (int shift = 56; shift >= 0; shift -= 8) {
        __syncthreads();
        for (int i = threadIdx.x; i < 256; i += NT) s.mass[i] = 0;
        __syncthreads();
        each([&](u64 number, u64 value) {
            if (shift == 56 || (number >> (shift + 8)) == (found >> (shift + 8))) atomicAdd(&s.mass[255 - ((number >> shift) & 255)], value);
        });
        __syncthreads();
        int digit; u64 before;
        reach<NT>(256, target, [&](int i) { return s.mass[i]; }, s, digit, before);
        target -= before;
        found |= (u64)(255 - digit) << shift;
    }
    return found;
}

template <class T, int NT>
__global__ __launch_bounds__(NT) void sample_kernel(SampleArgs a) {
    __shared__ Shared s;
    const int tid = threadIdx.x, row = blockIdx.x, V = a.V;
    const T* z = (const T*)a.z + row * a.z_b;
    const double temperature = a.temperature_rows ? (double)a.temperature_rows[row] : a.temperature;
    const long k_arg = a.top_k_rows ? (long)a.top_k_rows[row] : (long)a.top_k;
    const double top_p = a.top_p_rows ? (double)a.top_p_rows[row] : a.top_p;
    const double min_p = a.min_p_rows ? (double)a.min_p_rows[row] : a.min_p;
    const float u = a.u[row];

    // the maximum and its first place
    u64 best = 0;
    for (int i = tid; i < V; i += NT) { const u64 p = place(logit_at(z, i), i); best = best > p ? best : p; }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) { const u64 y = __shfl_xor(best, o); best = best > y ? best : y; }
    if constexpr (NT > 64) {
        if ((tid & 63) == 0) s.red[tid >> 6] = best;
        __syncthreads();
        for (int i = 0; i < NT / 64; ++i) best = best > s.red[i] ? best : s.red[i];
        __syncthreads();
    }
    const int first = (int)~(unsigned)best;
    const float zmax = logit_at(z, first);
    auto answer = [&](int token, float logp) {
        a.tokens[row] = token;
        if (a.logp) a.logp[row] = logp;
    };
    if (zmax == -INFINITY) { if (tid == 0) answer(-1, -INFINITY); return; }        // nothing to draw from
    if (!(temperature > 0.0) || k_arg == 1) { if (tid == 0) answer(first, 0.f); return; }

    Weigher w;
    w.zmax = zmax;
    w.a = 1.4426950408889634 / temperature;
    const int bits = 32 - __clz(V);
    w.unit = (double)(1ull << min(50, 62 - bits));
    w.af = (float)(w.a * ((SM_BINS - 1) / (double)SM_RANGE));
    u64 cut = 0;                                  // kept: place >= cut
    bool listed = false;                          // the list holds every kept candidate
    int n = 0;

    auto gather = [&](int lo, int hi) {           // candidates of bins lo..hi that are not behind the cut
        __syncthreads();
        if (tid == 0) s.n = 0;
        __syncthreads();
        for (int i = tid; i < V; i += NT) {
            const float x = logit_at(z, i);
            if (x == -INFINITY) continue;
            const int b = w.bin(x);
            const u64 p = place(x, i);
            if (b < lo || b > hi || p < cut) continue;
            const unsigned at = atomicAdd(&s.n, 1u);
            if (at < SM_CAP) { s.place[at] = p; s.weight[at] = w.fixed(w.weight(x)); }
        }
        __syncthreads();
        n = min((int)s.n, SM_CAP);
        __syncthreads();
    };
    auto list_each = [&](auto f) { for (int i = tid; i < n; i += NT) f(s.place[i], s.weight[i]); };
    auto row_each = [&](auto f) {
        for (int i = tid; i < V; i += NT) {
            const float x = logit_at(z, i);
            if (x == -INFINITY) continue;
            const u64 p = place(x, i);
            if (p >= cut) f(p, w.fixed(w.weight(x)));
        }
    };
    // counts (by_mass: masses too) of the candidates not behind the cut, by bin
    auto histogram = [&](bool by_mass) {
        __syncthreads();
        for (int i = tid; i < SM_BINS; i += NT) { s.mass[i] = 0; s.count[i] = 0; }
        __syncthreads();
        for (int i = tid; i < V; i += NT) {
            const float x = logit_at(z, i);
            if (x == -INFINITY || place(x, i) < cut) continue;
            const int b = w.bin(x);
            atomicAdd(&s.count[b], 1u);
            if (by_mass) atomicAdd(&s.mass[b], w.fixed(w.weight(x)));
        }
        __syncthreads();
    };
    auto counted = [&](int bin) {                 // candidates before the bin
        u64 c = 0;
        for (int i = tid; i < bin; i += NT) c += s.count[i];
        return block_sum<NT>(c, s);
    };

    if (k_arg > 1 && k_arg < V) {
        histogram(false);
        u64 c = 0;
        for (int i = tid; i < SM_BINS; i += NT) c += s.count[i];
        const u64 all = block_sum<NT>(c, s);
        if ((u64)k_arg < all) {
            int bin; u64 before;
            reach<NT>(SM_BINS, (u64)k_arg, [&](int i) { return (u64)s.count[i]; }, s, bin, before);
            const unsigned here = s.count[bin];
            if (before + here <= SM_CAP) {
                gather(0, bin);
                listed = true;
                cut = search<NT>((u64)k_arg, [&](auto f) { list_each([&](u64 p, u64) { f(p, (u64)1); }); }, s);
            } else if (here <= SM_CAP) {
                gather(bin, bin);
                cut = search<NT>((u64)k_arg - before, [&](auto f) { list_each([&](u64 p, u64) { f(p, (u64)1); }); }, s);
            } else {
                cut = search<NT>((u64)k_arg, [&](auto f) { row_each([&](u64 p, u64) { f(p, (u64)1); }); }, s);
            }
        }
    }
    if (top_p < 1.0) {
        auto goal = [&](u64 total) {              // the head's mass: the first candidate at which the sum reaches top_p of the total is the last kept
            const double t = top_p > 0.0 ? ceil(top_p * (double)total) : 1.0;
            const u64 g = (u64)t;
            return g < 1 ? (u64)1 : g > total ? total : g;
        };
        if (listed) {
            u64 m = 0;
            list_each([&](u64 p, u64 x) { if (p >= cut) m += x; });
            const u64 total = block_sum<NT>(m, s);
            cut = search<NT>(goal(total), [&](auto f) { list_each([&](u64 p, u64 x) { if (p >= cut) f(p, x); }); }, s);
        } else {
            histogram(true);
            u64 m = 0;
            for (int i = tid; i < SM_BINS; i += NT) m += s.mass[i];
            const u64 target = goal(block_sum<NT>(m, s));
            int bin; u64 before;
            reach<NT>(SM_BINS, target, [&](int i) { return s.mass[i]; }, s, bin, before);
            const unsigned here = s.count[bin];
            const u64 head = counted(bin);
            if (head + here <= SM_CAP) {
                gather(0, bin);
                listed = true;
                cut = search<NT>(target, [&](auto f) { list_each([&](u64 p, u64 x) { f(p, x); }); }, s);
            } else if (here <= SM_CAP) {
                gather(bin, bin);
                cut = search<NT>(target - before, [&](auto f) { list_each([&](u64 p, u64 x) { f(p, x); }); }, s);
            } else {
                cut = search<NT>(target, row_each, s);
            }
        }
    }

    // the draw: mass of the kept candidates, then the first index at which the cumulated mass exceeds u of it
    const u64 least = min_p > 0.0 ? w.fixed(fmin(min_p, 1.0)) : 0;
    auto goal = [&](u64 total) {                  // cumulated > u total  <=>  cumulated >= floor(u total) + 1
        if (u >= 1.f) return total;
        return (u > 0.f ? floor_of_product(u, total) : 0) + 1;
    };
    auto keeps = [&](u64 p, u64 x) { return p >= cut && x >= least; };
    u64 total = 0;
    int token;
    if (listed) {
        list_each([&](u64 p, u64 x) { if (keeps(p, x)) total += x; });
        total = block_sum<NT>(total, s);
        // lowest index first: the inverted index, largest first
        const u64 at = search<NT>(goal(total), [&](auto f) { list_each([&](u64 p, u64 x) { if (keeps(p, x)) f((u64)(unsigned)p, x); }); }, s);
        token = (int)~(unsigned)at;
    } else {
        // ranges of the row, one per wave, then ranges of the range that holds the target, until every thread has one index
        constexpr int NW = NT / 64;
        const int wave = tid >> 6, lane = tid & 63;
        int lo = 0, hi = V;
        u64 target = 0;
        bool first_level = true;
        while (true) {
            const int per = hi - lo <= NT ? 0 : (hi - lo + NW - 1) / NW;
            if (per == 0) break;
            const int x0 = min(hi, lo + wave * per), x1 = min(hi, x0 + per);
            u64 m = 0;
            for (int i = x0 + lane; i < x1; i += 64) {
                const float x = logit_at(z, i);
                if (x == -INFINITY) continue;
                const u64 f = w.fixed(w.weight(x));
                if (keeps(place(x, i), f)) m += f;
            }
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) m += __shfl_xor(m, o);
            __syncthreads();
            if (lane == 0) s.mass[wave] = m;
            __syncthreads();
            if (first_level) {
                for (int i = 0; i < NW; ++i) total += s.mass[i];
                target = goal(total);
                first_level = false;
            }
            int part; u64 before;
            reach<NT>(NW, target, [&](int i) { return s.mass[i]; }, s, part, before);
            target -= before;
            const int next = min(hi, lo + part * per);
            hi = min(hi, next + per);
            lo = next;
        }
        u64 mine = 0;
        if (lo + tid < hi) {
            const float x = logit_at(z, lo + tid);
            if (x != -INFINITY) {
                const u64 f = w.fixed(w.weight(x));
                if (keeps(place(x, lo + tid), f)) mine = f;
            }
        }
        __syncthreads();
        s.weight[tid] = mine;
        if (first_level) { total = block_sum<NT>(mine, s); target = goal(total); }
        __syncthreads();
        int at; u64 before;
        reach<NT>(NT, target, [&](int i) { return s.weight[i]; }, s, at, before);
        token = lo + at;
    }
    if (tid == 0) answer(token, (float)log((double)w.fixed(w.weight(logit_at(z, token))) / (double)total));
}

template <class T, int NT> int launch(const SampleArgs& a, hipStream_t stream) {
    hipLaunchKernelGGL((sample_kernel<T, NT>), dim3((unsigned)a.B), dim3(NT), 0, stream, a);
    LAS_LAUNCH_CHECK();
    return LAS_OK;
}
template <class T> int by_size(const SampleArgs& a, hipStream_t stream) {
    return a.V <= 4096 ? launch<T, 256>(a, stream) : launch<T, 1024>(a, stream);
}

}  // namespace

int sample(const SampleArgs& a, int dtype, hipStream_t stream) {
    return dtype == 0 ? by_size<float>(a, stream) : dtype == 1 ? by_size<__bf16>(a, stream) : by_size<_Float16>(a, stream);
}

}  // namespace las
