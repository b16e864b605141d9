// Distillation from a teacher's top logits: loss and gradient of one row in one launch.
//
//   p = softmax over the row's K entries of t / tau,  q = softmax over the vocabulary of z / tau
//   row = tau^2 sum_k p_k (log p_k - log q[index_k]),  loss = sum_rows w row,  w = 1 / (B len_b) on the first len_b steps, else 0
//   dz_v = tau w (q_v - sum of p_k over the entries k with index v)
//
// Bound by memory: the logits are read once and their gradient written once, so a row stays in the registers of its workgroup between the
// statistics and the gradient (up to 16 sixteen-byte pieces per thread of 1024: 131072 16-bit or 65536 fp32 values; longer rows are read
// a second time).  All statistics are fp32, the sum over rows is formed in a fixed order.  4096 rows of 128000 bf16 classes, 3000 of them taught, with the
// gradient: 466 us, 4.0 TB/s of bytes read and written; behind the registers' end a step
// of 152000 classes 589 us (of 128000: 483), of 2048 rows of 128000 fp32 classes 541.
#include "las_common.h"
#include "las_kernels.h"
#include <math.h>

namespace las {
namespace {

using u32x4 = __attribute__((ext_vector_type(4))) unsigned;

template <class T> struct Vec;
// (rows of an odd vocabulary start at any element: the hardware takes 16-byte accesses at element alignment)
template <> struct Vec<float> { typedef float V __attribute__((ext_vector_type(4), aligned(4))); static constexpr int EL = 4; };
template <> struct Vec<__bf16> { typedef __bf16 V __attribute__((ext_vector_type(8), aligned(2))); static constexpr int EL = 8; };
template <> struct Vec<_Float16> { typedef _Float16 V __attribute__((ext_vector_type(8), aligned(2))); static constexpr int EL = 8; };

static __device__ __forceinline__ float teacher_at(const DistillArgs& a, long i) {
    switch (a.t_dtype) {
        case 0: return ((const float*)a.t)[i];
        case 1: return (float)((const __bf16*)a.t)[i];
        default: return (float)((const _Float16*)a.t)[i];
    }
}
// entries that name no class of the vocabulary are absent
static __device__ __forceinline__ int index_at(const DistillArgs& a, long i) {
    const long v = a.idx64 ? ((const long long*)a.idx)[i] : (long)((const int*)a.idx)[i];
    return v >= 0 && v < a.V ? (int)v : -1;
}

static __device__ __forceinline__ float wave_max(float x) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor(x, o));
    return x;
}
static __device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o);
    return x;
}
// both values reduced over the workgroup, for every thread; red: 2 NT / 64 floats
template <int NT, bool MAX> static __device__ __forceinline__ void block2(float& x, float& y, float* red) {
    constexpr int NW = NT / 64;
    x = MAX ? wave_max(x) : wave_sum(x);
    y = MAX ? wave_max(y) : wave_sum(y);
    if constexpr (NW == 1) return;
    const int tid = threadIdx.x;
    __syncthreads();
    if ((tid & 63) == 0) { red[tid >> 6] = x; red[NW + (tid >> 6)] = y; }
    __syncthreads();
    x = red[0]; y = red[NW];
#pragma unroll
    for (int i = 1; i < NW; ++i) { x = MAX ? fmaxf(x, red[i]) : x + red[i]; y = MAX ? fmaxf(y, red[NW + i]) : y + red[NW + i]; }
}

// One workgroup per row.  NV > 0: NV pieces per thread hold the row; NV = 0: the row is read again.
template <class T, int NT, int NV>
__global__ __launch_bounds__(NT) void distill_kernel(DistillArgs a) {
    using V = typename Vec<T>::V;
    constexpr int EL = Vec<T>::EL;
    extern __shared__ float dyn[];
    float* sp = dyn;                             // K: teacher probabilities
    int* si = (int*)(dyn + a.K);                 // K: classes
    __shared__ float red[2 * NT / 64];
    if (a.unless_one && *a.upstream == 1.f) return;
    const int tid = threadIdx.x;
    const long row = blockIdx.x;
    const int b = (int)(row / a.U), u = (int)(row - (long)b * a.U);
    const int len = a.lens ? min(max(a.lens[b], 0), a.U) : a.U;
    const T* z = (const T*)a.z + b * a.z_b + u * a.z_u;
    T* dz = a.dz ? (T*)a.dz + b * a.dz_b + u * a.dz_u : nullptr;
    const int nvec = (a.V + EL - 1) / EL;

    auto load = [&](int i) {                     // piece i of the row; -inf behind its end
        V x;
        if (i * EL + EL <= a.V) return *(const V*)(z + i * EL);
#pragma unroll
        for (int e = 0; e < EL; ++e) x[e] = i * EL + e < a.V ? z[i * EL + e] : (T)-INFINITY;
        return x;
    };
    auto store = [&](int i, V x) {
        if (i * EL + EL <= a.V) {
            if (a.stream_out) __builtin_nontemporal_store(x, (V*)(dz + i * EL));
            else *(V*)(dz + i * EL) = x;
            return;
        }
#pragma unroll
        for (int e = 0; e < EL; ++e) if (i * EL + e < a.V) dz[i * EL + e] = x[e];
    };
    auto zeros = [&]() {
        if (a.rows && tid == 0) a.rows[row] = 0.f;
        if (dz) for (int i = tid; i < nvec; i += NT) store(i, V{});
    };
    if (u >= len) { zeros(); return; }

    // The row as raw pieces.  `held` hides from the compiler that the passes read the same values: it would otherwise keep all of them widened to
    // fp32 from one pass to the next (spilled, at 16 pieces per thread) where unpacking again is two instructions per pair.
    u32x4 keep[NV > 0 ? NV : 1];
    auto held = [&](int j) {
        asm volatile("" : "+v"(keep[j]));
        return __builtin_bit_cast(V, keep[j]);
    };
    if constexpr (NV > 0) {
        V none;
#pragma unroll
        for (int e = 0; e < EL; ++e) none[e] = (T)-INFINITY;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int i = tid + j * NT;
            keep[j] = i < nvec ? __builtin_bit_cast(u32x4, load(i)) : __builtin_bit_cast(u32x4, none);
        }
    }
    const float c = 1.4426950408889634f / a.tau;
    // Maximum and sum are taken of each piece as it arrives, relative to the thread's own running maximum: the exponentials of one piece run while the
    // others are on their way.  (A maximum of -inf stands for an empty sum: exponentials are then taken relative to 0, where they vanish.)
    auto base = [](float m) { return m == -INFINITY ? 0.f : m; };
    float mt = -INFINITY, mine = -INFINITY, sz = 0.f, st = 0.f;
    auto add = [&](V x) {
        float mx = (float)x[0];
#pragma unroll
        for (int e = 1; e < EL; ++e) mx = fmaxf(mx, (float)x[e]);
        mx = fmaxf(mine, mx);
        const float b = base(mx);
        sz *= __builtin_amdgcn_exp2f((mine - b) * c);
        mine = mx;
#pragma unroll
        for (int e = 0; e < EL; ++e) sz += __builtin_amdgcn_exp2f(((float)x[e] - b) * c);
    };
    for (int k = tid; k < a.K; k += NT) {
        const int v = index_at(a, row * a.K + k);
        const float t = v >= 0 ? teacher_at(a, row * a.K + k) : -INFINITY;
        sp[k] = t; si[k] = v;
        mt = t == t ? fmaxf(mt, t) : INFINITY;   // (a NaN, which a maximum would pass over, makes the row's probabilities NaN: NaN - inf)
    }
    if constexpr (NV > 0) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            add(held(j));
            asm volatile("" : "+v"(sz), "+v"(mine));      // (one piece unpacked at a time: all of them at once would not fit the registers)
        }
    } else {
        for (int i = tid; i < nvec; i += NT) add(load(i));
    }
    float mz = mine;
    block2<NT, true>(mt, mz, red);
    if (mt == -INFINITY) { zeros(); return; }    // (no entry at all: nothing to learn from this row)
    for (int k = tid; k < a.K; k += NT) st += __builtin_amdgcn_exp2f((sp[k] - mt) * c);
    sz *= __builtin_amdgcn_exp2f((mine - base(mz)) * c);
    block2<NT, false>(st, sz, red);
    const float w = 1.f / ((float)a.B * (float)len);
    const float invt = 1.f / st, invz = 1.f / sz, lt = log2f(st), lz = log2f(sz);

    if (a.rows) {
        float kl = 0.f, none = 0.f;
        for (int k = tid; k < a.K; k += NT) {
            const float x = (sp[k] - mt) * c, p = __builtin_amdgcn_exp2f(x) * invt;
            if (si[k] >= 0 && p != 0.f) kl = fmaf(p, (x - lt) - (((float)z[si[k]] - mz) * c - lz), kl);
        }
        block2<NT, false>(kl, none, red);
        if (tid == 0) a.rows[row] = kl * w * 0.6931471805599453f * a.tau * a.tau;
    }
    if (!dz) return;
    const float s = a.tau * w * (a.upstream ? *a.upstream : 1.f);
    const float sq = s * invz;
    auto grad = [&](V x) {
        V g;
#pragma unroll
        for (int e = 0; e < EL; ++e) g[e] = (T)(__builtin_amdgcn_exp2f(((float)x[e] - mz) * c) * sq);
        return g;
    };
    if constexpr (NV > 0) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int i = tid + j * NT;
            if (i < nvec) store(i, grad(held(j)));
        }
    } else {
        for (int i = tid; i < nvec; i += NT) store(i, grad(load(i)));
    }
    // the taught classes again, once their other writer is done: q - p in fp32, rounded once.  A class named twice is written by its first entry,
    // which adds the entries' probabilities in their order.
    __syncthreads();
    for (int k = tid; k < a.K; k += NT) {
        const int v = si[k];
        if (v < 0) continue;
        float p = 0.f;
        bool first = true;
        for (int j = 0; j < a.K; ++j)
            if (si[j] == v) {
                if (j < k) { first = false; break; }
                p += __builtin_amdgcn_exp2f((sp[j] - mt) * c) * invt;
            }
        if (first) dz[v] = (T)(__builtin_amdgcn_exp2f(((float)z[v] - mz) * c) * sq - p * s);
    }
}

// the rows' losses in a fixed order
constexpr int SUM_THREADS = 1024;
__global__ __launch_bounds__(SUM_THREADS) void distill_sum_kernel(const float* __restrict__ rows, long n, float* __restrict__ loss) {
    __shared__ double red[SUM_THREADS / 64];
    double x = 0.0;
    for (long i = threadIdx.x; i < n; i += SUM_THREADS) x += (double)rows[i];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < SUM_THREADS / 64; ++i) x += red[i];
        loss[0] = (float)x;
    }
}

template <class T, int NT, int NV> int launch(const DistillArgs& a, hipStream_t stream) {
    hipLaunchKernelGGL((distill_kernel<T, NT, NV>), dim3((unsigned)((long)a.B * a.U)), dim3(NT), (size_t)a.K * 8, stream, a);
    LAS_LAUNCH_CHECK();
    return LAS_OK;
}

template <class T> int by_size(const DistillArgs& a, hipStream_t stream) {
    const long n = (a.V + Vec<T>::EL - 1) / Vec<T>::EL;
    if (n <= 64) return launch<T, 64, 1>(a, stream);
    if (n <= 256) return launch<T, 256, 1>(a, stream);
    if (n <= 1024) return launch<T, 256, 4>(a, stream);
    if (n <= 2048) return launch<T, 512, 4>(a, stream);
    if (n <= 4096) return launch<T, 512, 8>(a, stream);
    if (n <= 8192) return launch<T, 1024, 8>(a, stream);
    if (n <= 16384) return launch<T, 1024, 16>(a, stream);
    return launch<T, 1024, 0>(a, stream);
}

}  // namespace

int distill(const DistillArgs& args, int dtype, float* loss, hipStream_t stream) {
    DistillArgs a = args;
    // a gradient that no cache could hold until its reader comes (256 MB behind the L2s) goes past them: 475 -> 452 us at 1 GB
    a.stream_out = (double)a.B * a.U * a.V * (dtype == 0 ? 4 : 2) > 256e6;
    const int rc = dtype == 0 ? by_size<float>(a, stream) : dtype == 1 ? by_size<__bf16>(a, stream) : by_size<_Float16>(a, stream);
    if (rc != LAS_OK || !loss) return rc;
    hipLaunchKernelGGL(distill_sum_kernel, dim3(1), dim3(SUM_THREADS), 0, stream, a.rows, (long)a.B * a.U, loss);
    LAS_LAUNCH_CHECK();
    return LAS_OK;
}

}  // namespace las
