// Attention of decoder states over an encoder's states of another length: forward, one-token form, backward.
//
//   s[i][j] = scale q_i . k_j  (j < len_b),  p = softmax_j s,  o_i = sum_j p[i][j] v_j ;  len_b = 0: o = 0 and every gradient 0.
//   D_i = do_i . o_i,  ds = p (do_i . v_j - D_i),  dq_i = scale sum_j ds k_j,  dk_j = scale sum_i ds q_i,  dv_j = sum_i p do_i.
//
// Heads: H query heads share Hkv key / value heads in groups of G = H / Hkv.  The rows of one (utterance, key head) are its G U query
// rows, numbered u G + g, so a tile of rows may span heads: a decode step of grouped heads is one tile, dk / dv of a shared head are
// summed over its group inside one workgroup — no atomics anywhere, every sum has a fixed order.
//
// One pass over the keys with the running maximum and sum of the softmax (fp32).  The score tile is formed TRANSPOSED (keys x rows:
// keys along the accumulator registers, one row per lane), so a row's maximum and sum are register reductions plus one exchange
// between the wave's halves, the rescale factor is one value per lane, and the probabilities leave the matrix instruction in just
// the shape that the second product wants as its right operand once the keys are taken in the order in which they lie in registers
// (a contraction may take its index in any order, if both operands do).  The left operand of that product (V^T, and K^T / Q^T / dO^T in
// the backward) is read from the row-major tile by the transposing LDS load.
#include "las_common.h"
#include "las_kernels.h"
#include <math.h>

namespace las {
namespace {

using bf16x8 = __attribute__((ext_vector_type(8))) __bf16;
using f16x8 = __attribute__((ext_vector_type(8))) _Float16;
using f32x8 = __attribute__((ext_vector_type(8))) float;
using u32x4 = __attribute__((ext_vector_type(4))) unsigned;
using s16x4 = __attribute__((ext_vector_type(4))) short;

constexpr int CA_THREADS = 256;

// ---- operands by type ------------------------------------------------------------------------------------------------------
// Every product runs on the 32x32x16 16-bit matrix instruction (lane half h holds contraction indices 8 h .. 8 h + 7 of 16; accumulation in fp32).
// A fp32 operand is the exact sum of three bf16 terms (x1 = rne(x), x2 = rne(x - x1), x3 = x - x1 - x2); six of the nine partial products are
// formed, the other three are below 2^-26 of |a b|: the accuracy of the fp32 matrix instruction at 2.67 times its rate, as in the GEMM.  (An infinite
// operand becomes NaN on the way, inf - inf, as does one that rounds beyond bf16's largest, 3.39e38.)  The terms of a tile lie in three planes of LDS, split once per workgroup as they are stored.
template <class T> struct Term { using E = T; static constexpr int N = 1; };
template <> struct Term<float> { using E = __bf16; static constexpr int N = 3; };

// eight contraction indices of one lane, all terms
template <class T> struct Frag { u32x4 p[Term<T>::N]; };

static __device__ __forceinline__ f32x16 mma16(f32x16 c, u32x4 a, u32x4 b, __bf16) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
static __device__ __forceinline__ f32x16 mma16(f32x16 c, u32x4 a, u32x4 b, _Float16) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
template <class T> static __device__ __forceinline__ f32x16 mma(f32x16 c, const Frag<T>& a, const Frag<T>& b) {
    using E = typename Term<T>::E;
    if constexpr (Term<T>::N == 3) {
        c = mma16(c, a.p[0], b.p[2], E{});
        c = mma16(c, a.p[2], b.p[0], E{});
        c = mma16(c, a.p[1], b.p[1], E{});
        c = mma16(c, a.p[0], b.p[1], E{});
        c = mma16(c, a.p[1], b.p[0], E{});
    }
    return mma16(c, a.p[0], b.p[0], E{});
}

// eight fp32 values as an operand.  16-bit types: rounding P and dS to the inputs' type costs half a step (2^-8 bf16, 2^-11 fp16) per term of sums
// that stay in fp32: the matrix instruction takes both operands in one type, and a second term would double the product.  (fp16 below its normal range: see
// P_SHIFT and DS_SCALED.)
template <class T> static __device__ __forceinline__ Frag<T> frag_of(f32x8 x) {
    using V8 = __attribute__((ext_vector_type(8))) typename Term<T>::E;
    Frag<T> f;
    if constexpr (Term<T>::N == 3) {
        const V8 a = __builtin_convertvector(x, V8);
        x -= __builtin_convertvector(a, f32x8);
        const V8 b = __builtin_convertvector(x, V8);
        x -= __builtin_convertvector(b, f32x8);
        f.p[0] = __builtin_bit_cast(u32x4, a);
        f.p[1] = __builtin_bit_cast(u32x4, b);
        f.p[2] = __builtin_bit_cast(u32x4, __builtin_convertvector(x, V8));
    } else {
        f.p[0] = __builtin_bit_cast(u32x4, __builtin_convertvector(x, V8));
    }
    return f;
}

// geometry: a row of DP elements is CPR sixteen-byte pieces of EL elements in global memory and LD elements (a piece of padding: rows start four banks
// apart) in a plane of LDS; NCH chunks of 16 contraction indices, NDT accumulator tiles
template <class T, int DP> struct Geo {
    static constexpr int EL = 16 / (int)sizeof(T), CPR = DP / EL, LD = DP + 8, NCH = DP / 16, NDT = DP / 32;
    static constexpr int plane(int rows) { return rows * LD; }
    static constexpr int bytes(int rows) { return plane(rows) * 2 * Term<T>::N; }
};

// eight elements of a row in global memory from element d on (zeros from `D` on), as fp32 values or as an operand
template <class T> static __device__ __forceinline__ f32x8 values_at(const T* row, int d, int D) {
    f32x8 x = {0, 0, 0, 0, 0, 0, 0, 0};
    if constexpr (sizeof(T) == 4) {
        if (d < D) { const f32x4 y = *(const f32x4*)(row + d); x[0] = y[0]; x[1] = y[1]; x[2] = y[2]; x[3] = y[3]; }
        if (d + 4 < D) { const f32x4 y = *(const f32x4*)(row + d + 4); x[4] = y[0]; x[5] = y[1]; x[6] = y[2]; x[7] = y[3]; }
    } else {
        using V8 = __attribute__((ext_vector_type(8))) T;
        if (d < D) x = __builtin_convertvector(*(const V8*)(row + d), f32x8);
    }
    return x;
}
template <class T> static __device__ __forceinline__ Frag<T> frag_at(const T* row, int d, int D) {
    if constexpr (sizeof(T) == 4) {
        return frag_of<T>(values_at(row, d, D));
    } else {
        Frag<T> f;
        f.p[0] = u32x4{0, 0, 0, 0};
        if (d < D) f.p[0] = *(const u32x4*)(row + d);
        return f;
    }
}
template <class T> static __device__ __forceinline__ Frag<T> no_frag() {
    Frag<T> f;
#pragma unroll
    for (int i = 0; i < Term<T>::N; ++i) f.p[i] = u32x4{0, 0, 0, 0};
    return f;
}

// chunk c (0, 1) of the 32x32 accumulator tile as the right operand of the next product: accumulator register r of lane half h is row
// 8 (r / 4) + 4 h + r % 4, so registers 8 c .. 8 c + 7 hold rows 16 c + {4 h .. 4 h + 3, 8 + 4 h .. 8 + 4 h + 3}.  ld_t below reads the left operand in
// the same order.
template <class T> static __device__ __forceinline__ Frag<T> pack(const f32x16& x, int c) {
    return frag_of<T>(f32x8{x[8 * c], x[8 * c + 1], x[8 * c + 2], x[8 * c + 3], x[8 * c + 4], x[8 * c + 5], x[8 * c + 6], x[8 * c + 7]});
}

// fp16 keeps its full precision only above 2^-14: probabilities are formed 2^P_SHIFT times too large there (a power of two in the exponential's
// argument costs nothing) and the sums divided by it: by 2^14 in the backward, where none exceeds one (2^14 of 65504), by 2^9 in the forward, where
// the running maximum may lag by 2^P_SLACK.
template <class T> constexpr float P_SHIFT = 0.f;
template <class T> constexpr float P_SHIFT_FWD = 0.f;
template <> constexpr float P_SHIFT<_Float16> = 14.f;
template <> constexpr float P_SHIFT_FWD<_Float16> = 9.f;
constexpr float P_SLACK = 6.f;

// dS has no such bound: it is as large as the output's gradient, which a mean over many rows makes small and a loss scale large.  In fp16 it is formed
// f times its size, a power of two for each lane (a row in dq, a key in dk) that follows the largest dS of the lane's sum: it starts at 2^60, where what
// is lost is below any fp16 result, and a tile that reaches beyond 2^15 takes it, and what was summed before, down to where that tile's largest lies between
// 2^9 and 2^10.  What is rounded below fp16's normal range is then off by 2^-34 of the largest at most.  (Unscaled, a dS below 2^-25 is zero and one above
// 65504 infinite.)  Price, a maximum per dS and on the key side a product: backward of 16 x 1024 over 2048, 16 on 4 heads of 32 277 -> 298 us, of 64 460 -> 465, of
// 96 720 -> 750, of 128 933 -> 1026.
template <class T> constexpr bool DS_SCALED = false;
template <> constexpr bool DS_SCALED<_Float16> = true;
template <class T> constexpr float DS_START = DS_SCALED<T> ? 0x1p60f : 1.f;
// a tile's dS as it is formed and the sum so far: the power of two by which the scale changes
template <class T, int NDT> static __device__ __forceinline__ int follow_ds(float& f, f32x16& ds, f32x16 (&acc)[NDT]) {
    if constexpr (!DS_SCALED<T>) return 0;
    float mx = fabsf(ds[0]);
#pragma unroll
    for (int r = 1; r < 16; ++r) mx = fmaxf(mx, fabsf(ds[r]));
    if (!__any(mx > 32768.f)) return 0;
    mx = fmaxf(mx, __shfl_xor(mx, 32));         // (a lane's other half holds the rest of the same sum's terms, and the same scale)
    const int by = mx > 32768.f ? min(10 - __builtin_amdgcn_frexp_expf(mx), 0) : 0;         // (an infinity has exponent 0 here, and stays one)
    f = ldexpf(f, by);
#pragma unroll
    for (int r = 0; r < 16; ++r) ds[r] = ldexpf(ds[r], by);
#pragma unroll
    for (int i = 0; i < NDT; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][r] = ldexpf(acc[i][r], by);
    return by;
}
template <class T, int NDT> static __device__ __forceinline__ void undo_ds(float f, f32x16 (&acc)[NDT]) {
    if constexpr (!DS_SCALED<T>) return;
    const int by = 1 - __builtin_amdgcn_frexp_expf(f);
#pragma unroll
    for (int i = 0; i < NDT; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][r] = ldexpf(acc[i][r], by);
}

// A tile of ROWS rows in LDS.
template <class T, int DP, int ROWS> struct LdsTile {
    using G = Geo<T, DP>;
    using E = typename Term<T>::E;
    E* s;
    // left operand, row-major: chunk c of row `row`
    __device__ __forceinline__ Frag<T> row(int row, int c, int h) const {
        Frag<T> f;
#pragma unroll
        for (int i = 0; i < Term<T>::N; ++i) f.p[i] = *(const u32x4*)(s + i * G::plane(ROWS) + row * G::LD + c * 16 + h * 8);
        return f;
    }
    // left operand, transposed: column d0 + lane % 32 at the contraction rows of chunk c (order: see pack), counted from row0.
    // ds_read_b64_tr_b16: the 16 lanes of a group name the 16 eight-byte pieces of a 4 (rows) x 16 (columns) block; lane i receives column i.
    __device__ __forceinline__ Frag<T> column(int row0, int c, int d0, int lane) const {
        typedef __attribute__((address_space(3))) s16x4* lds_ptr;
        const int h = lane >> 5, i = lane & 15;
        E* p = s + (row0 + 16 * c + 4 * h + (i >> 2)) * G::LD + d0 + (lane & 16) + (i & 3) * 4;
        Frag<T> f;
#pragma unroll
        for (int n = 0; n < Term<T>::N; ++n) {
            struct { s16x4 a, b; } both = {__builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(p + n * G::plane(ROWS))),
                                           __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(p + n * G::plane(ROWS) + 8 * G::LD))};
            f.p[n] = __builtin_bit_cast(u32x4, both);
        }
        return f;
    }
};

// ---- tiles of rows from global memory by way of registers -------------------------------------------------------------------
// Rows of any stride (multiples of 16 bytes); what lies outside [0, nrows) x [0, D) reads as zero, so that whatever a masked place
// holds (infinities, NaN) never meets a product.
constexpr int pow2_from(int n) { int p = 1; while (p < n) p *= 2; return p; }

// P: pieces that a row takes of the threads (its CPR, or the next power of two where the threads of a row have to add something up)
template <class T, int DP, int ROWS, int P = Geo<T, DP>::CPR> struct RowTile {
    using G = Geo<T, DP>;
    using E = typename Term<T>::E;
    static constexpr int N = (ROWS * P + CA_THREADS - 1) / CA_THREADS;
    static_assert(P == G::CPR || ROWS * P % 64 == 0, "a row's threads lie in one wave");
    u32x4 r[N];
    __device__ __forceinline__ void load(const T* base, long stride, int nrows, int D, int tid) {
#pragma unroll
        for (int v = 0; v < N; ++v) {
            const int i = tid + v * CA_THREADS, row = i / P, ch = i % P;
            r[v] = u32x4{0, 0, 0, 0};
            if (row < nrows && row < ROWS && ch * G::EL < D) r[v] = *(const u32x4*)(base + row * stride + ch * G::EL);
        }
    }
    // the rows that `at` stands at, of those below nrows
    template <class Walk> __device__ __forceinline__ void load(const T* base, const long (&offset)[N], const Walk& at, int nrows, int D) {
#pragma unroll
        for (int v = 0; v < N; ++v) {
            r[v] = u32x4{0, 0, 0, 0};
            if (at.inside(v, nrows, D)) r[v] = *(const u32x4*)(base + offset[v]);
        }
    }
    __device__ __forceinline__ void store(const LdsTile<T, DP, ROWS>& t, int tid) const {
#pragma unroll
        for (int v = 0; v < N; ++v) {
            const int i = tid + v * CA_THREADS, row = i / P, ch = i % P;
            if ((ROWS * P % CA_THREADS != 0 && row >= ROWS) || (P != G::CPR && ch >= G::CPR)) continue;
            E* to = t.s + row * G::LD + ch * G::EL;
            if constexpr (Term<T>::N == 3) {
                using V4 = __attribute__((ext_vector_type(4))) E;
                f32x4 x = __builtin_bit_cast(f32x4, r[v]);
#pragma unroll
                for (int n = 0; n < 3; ++n) {
                    const V4 y = __builtin_convertvector(x, V4);
                    *(V4*)(to + n * G::plane(ROWS)) = y;
                    if (n < 2) x -= __builtin_convertvector(y, f32x4);
                }
            } else {
                *(u32x4*)to = r[v];
            }
        }
    }
    // to[row] = f times the inner product of this tile's rows with another's, in fp32 (the sum's order is that of a tree over the row's threads)
    __device__ __forceinline__ void products(const RowTile& other, float f, float* to, int tid) const {
        using V = __attribute__((ext_vector_type(G::EL))) T;
#pragma unroll
        for (int v = 0; v < N; ++v) {
            const int i = tid + v * CA_THREADS, row = i / P;
            const V x = __builtin_bit_cast(V, r[v]), y = __builtin_bit_cast(V, other.r[v]);
            float d = 0.f;
#pragma unroll
            for (int e = 0; e < G::EL; ++e) d = fmaf((float)x[e], (float)y[e], d);
#pragma unroll
            for (int o = P / 2; o > 0; o >>= 1) d += __shfl_xor(d, o);
            if (i % P == 0 && row < ROWS) to[row] = d * f;
        }
    }
};

// Where this thread's pieces of a tile of ROWS rows lie, row n = u G + g being at u su + g sg of one tensor and of another: divided out once, then carried
// from tile to tile (a division and two 64-bit products per piece and tile were a third of the key side's vector instructions).
template <int EL, int ROWS, int P> struct RowWalk {
    static constexpr int N = (ROWS * P + CA_THREADS - 1) / CA_THREADS;
    long a[N], b[N], step_a, step_b, wrap_a, wrap_b;
    int g[N], row0, rest, share, ch, row;
    __device__ __forceinline__ RowWalk(long su_a, long sg_a, long su_b, long sg_b, int share_, int from, int tid)
        : row0(from), share(share_), ch(tid % P), row(tid / P) {
        static_assert(CA_THREADS % P == 0, "a thread keeps its place in the rows");
        rest = ROWS % share;
        step_a = ROWS / share * su_a + rest * sg_a; wrap_a = su_a - share * sg_a;
        step_b = ROWS / share * su_b + rest * sg_b; wrap_b = su_b - share * sg_b;
#pragma unroll
        for (int v = 0; v < N; ++v) {
            const int n = from + row + v * (CA_THREADS / P), u = n / share;
            g[v] = n - u * share;
            a[v] = u * su_a + g[v] * sg_a + ch * EL;
            b[v] = u * su_b + g[v] * sg_b + ch * EL;
        }
    }
    __device__ __forceinline__ bool inside(int v, int nrows, int D) const {
        const int n = row + v * (CA_THREADS / P);
        return row0 + n < nrows && n < ROWS && ch * EL < D;
    }
    __device__ __forceinline__ void next() {
        row0 += ROWS;
#pragma unroll
        for (int v = 0; v < N; ++v) { a[v] += step_a; b[v] += step_b; }
        if (rest == 0) return;
#pragma unroll
        for (int v = 0; v < N; ++v) {
            g[v] += rest;
            if (g[v] >= share) { g[v] -= share; a[v] += wrap_a; b[v] += wrap_b; }
        }
    }
};

static __device__ __forceinline__ float other_half(float x) { return __shfl_xor(x, 32); }

static __device__ __forceinline__ int length_of(const CrossAttnArgs& a, int b) {
    return a.lens ? min(max(a.lens[b], 0), a.T) : a.T;
}

// The factor that makes a row's sum its output, and its statistic, from the sum l of its exponentials: no key at all gives zeros; keys whose scores are all -inf
// give NaN, as a score of NaN does.
static __device__ __forceinline__ float inverse(float l, bool any) { return l > 0.f ? 1.f / l : l == 0.f && !any ? 0.f : NAN; }
static __device__ __forceinline__ float statistic(float l, bool any, float m, float c, float shift) {
    return l > 0.f ? fmaf(m, c, log2f(l) - shift) : l == 0.f && !any ? -INFINITY : NAN;
}

// Which work a block does.  Workgroups of one (utterance, key head) read the same keys: they go to one XCD (blockIdx % 8 on this device) and share its L2.
// Where a launch takes more than one round of the GPU (`a.longest_first`), an XCD's workgroups start in falling order of their utterances' lengths and
// the XCDs take turns in that order, so that the last round fills up with the short ones (16 x 512 over ragged 1500: 259 -> 240 us a step).  A
// permutation of the work for any placement of blocks.
// TILED: the `per` workgroups lie along the keys, TILED keys each.  Those behind an utterance's end have only zeros to write and start after all others:
// the shader engines of an XCD take its workgroups in turn, so that one that is done at once leaves its place empty until the turn comes round.  (Not with
// ranges of the rows: these are for no more key workgroups than CUs, which all start at once.)
struct Work { int i, b, kvh; bool any; };      // i: which of the `per` workgroups of (b, kvh)
template <int TILED = 0> static __device__ __forceinline__ Work work_of(const CrossAttnArgs& a, int block, int per) {
    const int local = block >> 3, n = a.B * a.Hkv, xcd = block & 7;
    int at = local / per * 8 + xcd, i = local % per;
    Work w = {i, at / a.Hkv, at % a.Hkv, at < n};
    if (!a.longest_first) return w;
    // the utterance whose length is the r-th largest (equal lengths by index) in lane r; a lane for each of at most 64
    const int lane = threadIdx.x & 63, mine = lane < a.B ? length_of(a, lane) : -1;
    int rank = 0;
    for (int j = 0; j < a.B; ++j) {
        const int other = __builtin_amdgcn_readlane(mine, j);
        rank += other > mine || (other == mine && j < lane) ? 1 : 0;
    }
    const int sorted = __builtin_amdgcn_ds_permute((lane < a.B ? rank : lane) * 4, lane);
    const int groups = (n + 7) / 8;
    if (TILED > 0 && a.nk == 1 && groups <= 64) {
        // lane g: the XCD's g-th (utterance, key head), its tiles of keys and of zeros, and their sums up to here
        const bool mine_any = lane < groups && lane * 8 + xcd < n;
        const int b = __shfl(sorted, mine_any ? (lane * 8 + xcd) / a.Hkv : 0), len = __shfl(mine, b);
        const int keys = mine_any ? (len + TILED - 1) / (TILED > 0 ? TILED : 1) : 0;
        int upto = keys, zeros = mine_any ? per - keys : 0;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int x = __shfl_up(upto, o), y = __shfl_up(zeros, o);
            if (lane >= o) { upto += x; zeros += y; }
        }
        const int all = __builtin_amdgcn_readlane(upto, 63), rest = local - all;
        const bool zero = rest >= 0;
        const unsigned long long past = __ballot(zero ? zeros > rest : upto > local);
        if (past == 0) { w.any = false; return w; }
        const int g = __ffsll((long long)past) - 1;
        const int own = __builtin_amdgcn_readlane(keys, g), before = __builtin_amdgcn_readlane(zero ? zeros : upto, g) - (zero ? per - own : own);
        at = g * 8 + xcd;
        w = {zero ? own + rest - before : local - before, at / a.Hkv, at % a.Hkv, true};
    }
    if (w.any) w.b = __builtin_amdgcn_readlane(sorted, w.b);
    return w;
}
// the part-th of n ranges of [0, length): whole tiles of 32
struct Range { int begin, end; };
static __device__ __forceinline__ Range range_of(int length, int n, int part) {
    const int per = ((length + n - 1) / n + 31) & ~31, begin = min(length, part * per);
    return {begin, min(length, begin + per)};
}
// blocks of a launch of `per` workgroups for each (utterance, key head)
static long blocks_of(const CrossAttnArgs& a, long per) { return ((long)a.B * a.Hkv + 7) / 8 * 8 * per; }


// Workgroups per CU that the registers are budgeted for (as many waves per SIMD): two where a workgroup's tiles fit 256 registers (18 of them to and from
// scratch memory at 16-bit heads of 128 cost less than the second workgroup gives: backward of 16 x 1024 over 2048, 1614 -> 1161 us), else one.
template <class T, int DP> constexpr int FWD_PER_CU = sizeof(T) == 2 || DP <= 64 ? 2 : 1;
template <class T, int DP, int NW> constexpr int BWD_PER_CU = DP <= 32 || (sizeof(T) == 2 && DP <= 96) || (NW == 4 && (sizeof(T) == 2 || DP <= 64)) ? 2 : 1;
// Tiles of 32 keys (rows) that a wide workgroup's waves take at a time.  Two halve the barriers, one leaves registers for another wave per SIMD: forward, 16-bit
// heads of 64 (16 x 512 over ragged 1500: 55 -> 52 us; heads of 32 have four waves either way, 113 against 127 us at 16 x 1024 over 2048, heads of 96 three
// against two, 254 against 261); backward, all but the smallest (heads of 64: 590 -> 557 us, of 96: 1320 -> 884; fp32 heads of 64, 16 x 512 over 1000: 399 -> 316;
// heads of 32: 362 against 395).  One of fp32 is three planes.
template <class T, int DP> constexpr int DEEP_FWD = (sizeof(T) == 4 && DP > 64) || (sizeof(T) == 2 && DP == 64) ? 1 : 2;
template <class T, int DP> constexpr int DEEP_BWD = DP > 32 ? 1 : 2;

// ---- forward ----------------------------------------------------------------------------------------------------------------
// Four waves: NWQ of them side by side over rows (32 each), NWK over keys (KT tiles of 32 of every key tile each).
// Many rows: bound by the issue of the softmax's vector instructions (one exponential, three others a score) and of the products, which two to four waves
// per SIMD overlap in part: bf16, 16 x 2048 rows of 16 on 4 heads over 4096 keys, 820 TFLOP/s at heads of 64, 870 at 128; fp32, 16 x 512 over 1000 heads
// of 128, 152 TFLOP/s (the library's fp32 product: 153).  One row per head: bound by the keys' bytes, 16 x 16 heads on 4 of 128
// over ragged 30000 in 149 us, 5 TB/s.
template <class T, int DP, int NWQ, int NWK, int KT>
__global__ __launch_bounds__(CA_THREADS, (FWD_PER_CU<T, DP>)) void cross_attn_fwd_kernel(CrossAttnArgs a) {
    using G = Geo<T, DP>;
    constexpr int BK = 32 * KT * NWK;
    constexpr int RED = NWK > 1 ? 4 * (DP + 2) * 32 * 4 : 0;                    // bytes of the joining of waves
    constexpr int TILE = 2 * G::bytes(BK);
    __shared__ __attribute__((aligned(16))) char smem[TILE > RED ? TILE : RED];
    const LdsTile<T, DP, BK> sK{(typename Term<T>::E*)smem}, sV{(typename Term<T>::E*)(smem + G::bytes(BK))};
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wq = wave / NWK, wk = wave % NWK, h = lane >> 5;
    const int share = a.H / a.Hkv, R = a.U * share, ntiles = (R + 32 * NWQ - 1) / (32 * NWQ);
    const Work w = work_of(a, blockIdx.x, ntiles * a.nsplit);
    if (!w.any) return;
    const int tile = w.i % ntiles, split = w.i / ntiles, b = w.b, kvh = w.kvh;
    const int len = length_of(a, b);
    const Range keys = range_of(len, a.nsplit, split);
    const int begin = keys.begin, end = keys.end;
    const T* q = (const T*)a.q + b * a.q_b + (long)kvh * share * a.q_h;
    const T* k = (const T*)a.k + b * a.k_b + kvh * a.k_h;
    const T* v = (const T*)a.v + b * a.v_b + kvh * a.v_h;

    const int row = tile * 32 * NWQ + wq * 32 + (lane & 31), u = row / share, g = row - u * share;
    const bool live = row < R;
    Frag<T> qf[G::NCH];
#pragma unroll
    for (int c = 0; c < G::NCH; ++c) qf[c] = live ? frag_at(q + u * a.q_u + g * a.q_h, c * 16 + h * 8, a.D) : no_frag<T>();
    f32x16 acc[G::NDT];
#pragma unroll
    for (int i = 0; i < G::NDT; ++i) acc[i] = f32x16{0};
    float m = -INFINITY, l = 0.f;

    RowTile<T, DP, BK> tk, tv;
    if (begin < end) {
        tk.load(k + (long)begin * a.k_t, a.k_t, end - begin, a.D, tid);
        tv.load(v + (long)begin * a.v_t, a.v_t, end - begin, a.D, tid);
    }
    for (int k0 = begin; k0 < end; k0 += BK) {
        __syncthreads();
        tk.store(sK, tid);
        tv.store(sV, tid);
        __syncthreads();
        if (k0 + BK < end) {
            tk.load(k + (long)(k0 + BK) * a.k_t, a.k_t, end - k0 - BK, a.D, tid);
            tv.load(v + (long)(k0 + BK) * a.v_t, a.v_t, end - k0 - BK, a.D, tid);
        }
        if (k0 + wk * KT * 32 >= end) continue;      // (wave-uniform; the barriers above are met by every wave again)
        f32x16 s[KT];
#pragma unroll
        for (int t = 0; t < KT; ++t) {
            s[t] = f32x16{0};
#pragma unroll
            for (int c = 0; c < G::NCH; ++c) s[t] = mma<T>(s[t], sK.row((wk * KT + t) * 32 + (lane & 31), c, h), qf[c]);
        }
        if (k0 + (wk * KT + KT) * 32 > end) {
#pragma unroll
            for (int t = 0; t < KT; ++t)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (k0 + (wk * KT + t) * 32 + 8 * (r >> 2) + 4 * h + (r & 3) >= end) s[t][r] = -INFINITY;
        }
        float mx = s[0][0];
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[t][r]);
        mx = fmaxf(m, fmaxf(mx, other_half(mx)));
        // The maximum only has to keep the exponentials in range: it follows the true one when that has grown by more than 2^P_SLACK somewhere in the
        // wave, which is once or twice in a row of any length, not at almost every tile.
        if (__any((mx - m) * a.c > P_SLACK)) {
            const float alpha = mx == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m - mx) * a.c);
            l *= alpha;
#pragma unroll
            for (int i = 0; i < G::NDT; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[i][r] *= alpha;
            m = mx;
        }
        const float mc = (m == -INFINITY ? 0.f : m * a.c) - P_SHIFT_FWD<T>;
#pragma unroll
        for (int t = 0; t < KT; ++t) {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                s[t][r] = __builtin_amdgcn_exp2f(fmaf(s[t][r], a.c, -mc));
                l += s[t][r];
            }
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const Frag<T> p = pack<T>(s[t], c);
#pragma unroll
                for (int i = 0; i < G::NDT; ++i) acc[i] = mma<T>(acc[i], sV.column((wk * KT + t) * 32, c, i * 32, lane), p);
            }
        }
    }
    l += other_half(l);
    if constexpr (NWK > 1) {       // join the waves of one row tile, in their order
        float* red = (float*)smem;
        float* mine = red + wave * (DP + 2) * 32;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < G::NDT; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) mine[(i * 32 + 8 * (r >> 2) + 4 * h + (r & 3)) * 32 + (lane & 31)] = acc[i][r];
        if (h == 0) { mine[DP * 32 + lane] = m; mine[(DP + 1) * 32 + lane] = l; }
        __syncthreads();
        if (wk != 0) return;
        const float* first = red + wq * NWK * (DP + 2) * 32;
        float mj = -INFINITY;
#pragma unroll
        for (int x = 0; x < NWK; ++x) mj = fmaxf(mj, first[x * (DP + 2) * 32 + DP * 32 + (lane & 31)]);
        l = 0.f;
#pragma unroll
        for (int i = 0; i < G::NDT; ++i) acc[i] = f32x16{0};
#pragma unroll
        for (int x = 0; x < NWK; ++x) {
            const float* from = first + x * (DP + 2) * 32;
            const float mm = from[DP * 32 + (lane & 31)];
            const float f = mm == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((mm - mj) * a.c);
            l += f * from[(DP + 1) * 32 + (lane & 31)];
#pragma unroll
            for (int i = 0; i < G::NDT; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    acc[i][r] = fmaf(f, from[(i * 32 + 8 * (r >> 2) + 4 * h + (r & 3)) * 32 + (lane & 31)], acc[i][r]);
        }
        m = mj;
    }
    if (!live) return;
    const long out_row = ((long)b * a.U + u) * a.H + kvh * share + g;
    if (a.nsplit > 1) {
        const long at = (long)split * a.B * a.U * a.H + out_row;
        float* part = a.part + at * a.D;
#pragma unroll
        for (int i = 0; i < G::NDT; ++i)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const int d = i * 32 + 8 * x + 4 * h;
                if (d < a.D) *(f32x4*)(part + d) = f32x4{acc[i][4 * x], acc[i][4 * x + 1], acc[i][4 * x + 2], acc[i][4 * x + 3]};
            }
        if (h == 0) {
            float* ml = a.part + (long)a.nsplit * a.B * a.U * a.H * a.D + at * 2;
            ml[0] = m; ml[1] = l;
        }
        return;
    }
    const float inv = inverse(l, len > 0);
    T* o = (T*)a.o + out_row * a.D;
#pragma unroll
    for (int i = 0; i < G::NDT; ++i)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const int d = i * 32 + 8 * x + 4 * h;
            using V4 = __attribute__((ext_vector_type(4))) T;
            const f32x4 y = {acc[i][4 * x] * inv, acc[i][4 * x + 1] * inv, acc[i][4 * x + 2] * inv, acc[i][4 * x + 3] * inv};
            if (d < a.D) *(V4*)(o + d) = __builtin_convertvector(y, V4);
        }
    if (a.lse && h == 0) a.lse[out_row] = statistic(l, len > 0, m, a.c, P_SHIFT_FWD<T>);
}

// joins the key ranges of a split forward: four values of one row per thread
template <class T>
__global__ __launch_bounds__(CA_THREADS) void cross_attn_join_kernel(CrossAttnArgs a) {
    const long n = (long)a.B * a.U * a.H, per = a.D / 4, i = (long)blockIdx.x * CA_THREADS + threadIdx.x;
    if (i >= n * per) return;
    const long row = i / per;
    const int d = (int)(i - row * per) * 4;
    const float* ml = a.part + (long)a.nsplit * n * a.D;
    float mj = -INFINITY;
#pragma unroll 4
    for (int s = 0; s < a.nsplit; ++s) mj = fmaxf(mj, ml[(s * n + row) * 2]);
    f32x4 acc = {0, 0, 0, 0};
    float l = 0.f;
#pragma unroll 4
    for (int s = 0; s < a.nsplit; ++s) {
        const float m = ml[(s * n + row) * 2];
        const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - mj) * a.c);      // (an empty range: zeros)
        l += f * ml[(s * n + row) * 2 + 1];
        acc += f * *(const f32x4*)(a.part + (s * n + row) * a.D + d);
    }
    const bool any = length_of(a, (int)(row / ((long)a.U * a.H))) > 0;
    const float inv = inverse(l, any);
    using V4 = __attribute__((ext_vector_type(4))) T;
    acc *= inv;
    *(V4*)((T*)a.o + row * a.D + d) = __builtin_convertvector(acc, V4);
    if (a.lse && d == 0) a.lse[row] = statistic(l, any, mj, a.c, P_SHIFT_FWD<T>);
}

// The same where there are no more rows than CUs: a workgroup per row, its threads side by side over the ranges too (one token of 16 heads over 100000 frames
// in 128 ranges: 87 us with a thread's loop over all of them, 71 so; 3 x 4 heads over 10080: 22.4 against 17.3; but 10656 rows of 5 ranges 29.8 against 38.4).
template <class T>
__global__ __launch_bounds__(CA_THREADS) void cross_attn_join_row_kernel(CrossAttnArgs a) {
    __shared__ f32x4 sum[CA_THREADS];
    __shared__ float red[CA_THREADS], ls[CA_THREADS];
    const long n = (long)a.B * a.U * a.H, row = blockIdx.x;
    const int tid = threadIdx.x, per = a.D / 4, side = CA_THREADS / per, x = tid % per, y = tid / per;
    const float* ml = a.part + (long)a.nsplit * n * a.D;
    float mj = -INFINITY, l = 0.f;
    for (int s = tid; s < a.nsplit; s += CA_THREADS) mj = fmaxf(mj, ml[(s * n + row) * 2]);
    red[tid] = mj;
    __syncthreads();
    for (int o = CA_THREADS / 2; o > 0; o >>= 1) {
        if (tid < o) red[tid] = fmaxf(red[tid], red[tid + o]);
        __syncthreads();
    }
    mj = red[0];
    f32x4 acc = {0, 0, 0, 0};
    if (y < side) {
#pragma unroll 2
        for (int s = y; s < a.nsplit; s += side) {
            const float m = ml[(s * n + row) * 2];
            const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - mj) * a.c);      // (an empty range: zeros)
            l += f * ml[(s * n + row) * 2 + 1];
            acc += f * *(const f32x4*)(a.part + (s * n + row) * a.D + x * 4);
        }
    }
    sum[tid] = acc;
    ls[tid] = l;
    __syncthreads();
    if (y != 0) return;
    for (int i = 1; i < side; ++i) { acc += sum[i * per + x]; l += ls[i * per + x]; }
    const bool any = length_of(a, (int)(row / ((long)a.U * a.H))) > 0;
    const float inv = inverse(l, any);
    using V4 = __attribute__((ext_vector_type(4))) T;
    acc *= inv;
    *(V4*)((T*)a.o + row * a.D + x * 4) = __builtin_convertvector(acc, V4);
    if (a.lse && x == 0) a.lse[row] = statistic(l, any, mj, a.c, P_SHIFT_FWD<T>);
}

// four results of a type, or of fp32 where they are one range's
template <class T> static __device__ __forceinline__ void put(float* part, T* to, f32x4 y) {
    using V4 = __attribute__((ext_vector_type(4))) T;
    if (part) *(f32x4*)part = y;
    else *(V4*)to = __builtin_convertvector(y, V4);
}
// the sum of n ranges' results of `count` fours each, in their order
template <class T> __global__ __launch_bounds__(CA_THREADS) void cross_attn_sum_kernel(const float* part, int n, long count, T* to) {
    const long i = (long)blockIdx.x * CA_THREADS + threadIdx.x;
    if (i >= count) return;
    f32x4 y = {0, 0, 0, 0};
#pragma unroll 4
    for (int s = 0; s < n; ++s) y += *(const f32x4*)(part + (s * count + i) * 4);
    put<T>(nullptr, to + i * 4, y);
}

// ---- backward: dq -----------------------------------------------------------------------------------------------------------
// The forward's shape: one row per lane; q and do stay in registers, every key tile is read once per row tile.
// Both sides of the backward together form seven products where one with atomics would form five: the price of sums of a fixed order.  Bound like the
// forward, and by LDS, from which every left operand is read: bf16 16 x 1024 over 2048, 16 on 4 heads of 64, 557 us (617 TFLOP/s of the five products).
template <class T, int DP, int NWQ, int NWK, int KT> constexpr int DQ_BYTES() {
    const int tile = 2 * Geo<T, DP>::bytes(32 * KT * NWK), red = NWK > 1 ? 4 * DP * 32 * 4 : 0;
    return tile > red ? tile : red;
}
template <class T, int DP, int NWQ, int NWK, int KT>
static __device__ __forceinline__ void cross_attn_dq(const CrossAttnArgs& a, int block, char* smem) {
    using G = Geo<T, DP>;
    constexpr int BK = 32 * KT * NWK;
    const LdsTile<T, DP, BK> sK{(typename Term<T>::E*)smem}, sV{(typename Term<T>::E*)(smem + G::bytes(BK))};
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wq = wave / NWK, wk = wave % NWK, h = lane >> 5;
    const int share = a.H / a.Hkv, R = a.U * share, ntiles = (R + 32 * NWQ - 1) / (32 * NWQ);
    const Work w = work_of(a, block, ntiles * a.nq);
    if (!w.any) return;
    const int tile = w.i % ntiles, split = w.i / ntiles, b = w.b, kvh = w.kvh;
    const Range keys = range_of(length_of(a, b), a.nq, split);
    const int begin = keys.begin, end = keys.end;
    const T* q = (const T*)a.q + b * a.q_b + (long)kvh * share * a.q_h;
    const T* k = (const T*)a.k + b * a.k_b + kvh * a.k_h;
    const T* v = (const T*)a.v + b * a.v_b + kvh * a.v_h;
    const int row = tile * 32 * NWQ + wq * 32 + (lane & 31), u = row / share, g = row - u * share;
    const bool live = row < R;
    const long out_row = ((long)b * a.U + u) * a.H + kvh * share + g;

    RowTile<T, DP, BK> tk, tv;
    if (begin < end) {
        tk.load(k + (long)begin * a.k_t, a.k_t, end - begin, a.D, tid);
        tv.load(v + (long)begin * a.v_t, a.v_t, end - begin, a.D, tid);
    }
    Frag<T> qf[G::NCH], dof[G::NCH];
    float delta = 0.f;
#pragma unroll
    for (int c = 0; c < G::NCH; ++c) {
        qf[c] = dof[c] = no_frag<T>();
        const int d = c * 16 + h * 8;
        if (live) {
            // (D_i from the output as it was rounded: half a step of each of its values, against a second tensor in fp32 kept from the forward)
            const f32x8 x = values_at((const T*)a.o + out_row * a.D, d, a.D), y = values_at((const T*)a.dout + out_row * a.D, d, a.D);
#pragma unroll
            for (int e = 0; e < 8; ++e) delta = fmaf(x[e], y[e], delta);
            qf[c] = frag_at(q + u * a.q_u + g * a.q_h, d, a.D);
            dof[c] = frag_of<T>(y);
        }
    }
    delta += other_half(delta);
    const float lse = live ? a.lse[out_row] : INFINITY;
    float f = DS_START<T>;
    delta *= f;
    f32x16 acc[G::NDT];
#pragma unroll
    for (int i = 0; i < G::NDT; ++i) acc[i] = f32x16{0};

    for (int k0 = begin; k0 < end; k0 += BK) {
        __syncthreads();
        tk.store(sK, tid);
        tv.store(sV, tid);
        __syncthreads();
        if (k0 + BK < end) {
            tk.load(k + (long)(k0 + BK) * a.k_t, a.k_t, end - k0 - BK, a.D, tid);
            tv.load(v + (long)(k0 + BK) * a.v_t, a.v_t, end - k0 - BK, a.D, tid);
        }
#pragma unroll
        for (int t = 0; t < KT; ++t) {
            const int r0 = (wk * KT + t) * 32;
            if (k0 + r0 >= end) continue;
            f32x16 s = f32x16{0}, dp = f32x16{0};
#pragma unroll
            for (int c = 0; c < G::NCH; ++c) {
                s = mma<T>(s, sK.row(r0 + (lane & 31), c, h), qf[c]);
                dp = mma<T>(dp, sV.row(r0 + (lane & 31), c, h), dof[c]);
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], a.c, -lse)) * (DS_SCALED<T> ? fmaf(dp[r], f, -delta) : dp[r] - delta);
            if (k0 + r0 + 32 > end) {            // (the keys behind the last: zeros in K, but exp2(-lse) need not be finite)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (k0 + r0 + 8 * (r >> 2) + 4 * h + (r & 3) >= end) s[r] = 0.f;
            }
            delta = ldexpf(delta, follow_ds<T>(f, s, acc));
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const Frag<T> ds = pack<T>(s, c);
#pragma unroll
                for (int i = 0; i < G::NDT; ++i) acc[i] = mma<T>(acc[i], sK.column(r0, c, i * 32, lane), ds);
            }
        }
    }
    undo_ds<T>(f, acc);
    if constexpr (NWK > 1) {
        float* red = (float*)smem;
        __syncthreads();
        if (wk != 0) {
#pragma unroll
            for (int i = 0; i < G::NDT; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) red[(wave * DP + i * 32 + 8 * (r >> 2) + 4 * h + (r & 3)) * 32 + (lane & 31)] = acc[i][r];
        }
        __syncthreads();
        if (wk != 0) return;
#pragma unroll
        for (int x = 1; x < NWK; ++x)
#pragma unroll
            for (int i = 0; i < G::NDT; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[i][r] += red[((wave + x) * DP + i * 32 + 8 * (r >> 2) + 4 * h + (r & 3)) * 32 + (lane & 31)];
    }
    if (!live) return;
    T* o = (T*)a.dq + out_row * a.D;
    float* part = a.part_q + ((long)split * a.B * a.U * a.H + out_row) * a.D;
#pragma unroll
    for (int i = 0; i < G::NDT; ++i)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const int d = i * 32 + 8 * x + 4 * h;
            const f32x4 y = {acc[i][4 * x] * a.scale, acc[i][4 * x + 1] * a.scale, acc[i][4 * x + 2] * a.scale, acc[i][4 * x + 3] * a.scale};
            if (d < a.D) put(a.nq > 1 ? part + d : nullptr, o + d, y);
        }
}

// ---- backward: dk, dv -------------------------------------------------------------------------------------------------------
// One key per lane (k and v in registers), row tiles of q and do through LDS; NWK waves side by side over keys, NWR over rows.
// D_i is formed here once more, by the threads that bring in a row of do (and for that alone the same row of the output): the two halves of the
// backward then need nothing of each other and run in one launch, the one filling the other's last round.
template <class T, int DP, int NWK, int NWR, int RT> constexpr int DKV_BYTES() {
    const int tile = 2 * Geo<T, DP>::bytes(32 * RT * NWR) + 2 * 32 * RT * NWR * 4, red = NWR > 1 ? 4 * DP * 32 * 4 : 0;
    return tile > red ? tile : red;
}
template <class T, int DP, int NWK, int NWR, int RT>
static __device__ __forceinline__ void cross_attn_dkv(const CrossAttnArgs& a, int block, char* smem) {
    using G = Geo<T, DP>;
    constexpr int BR = 32 * RT * NWR;
    constexpr float P_BACK = P_SHIFT<T> == 0.f ? 1.f : 1.f / 16384.f;
    const LdsTile<T, DP, BR> sQ{(typename Term<T>::E*)smem}, sO{(typename Term<T>::E*)(smem + G::bytes(BR))};
    float* sL = (float*)(smem + 2 * G::bytes(BR));
    float* sD = sL + BR;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wk = wave / NWR, wr = wave % NWR, h = lane >> 5;
    const int share = a.H / a.Hkv, R = a.U * share, ntiles = (a.T + 32 * NWK - 1) / (32 * NWK);
    const Work w = work_of<32 * NWK>(a, block, ntiles * a.nk);
    if (!w.any) return;
    const int tile = w.i % ntiles, split = w.i / ntiles, b = w.b, kvh = w.kvh;
    const int len = length_of(a, b);
    const Range rows = range_of(R, a.nk, split);
    const int first = rows.begin, last = rows.end;
    const T* q = (const T*)a.q + b * a.q_b + (long)kvh * share * a.q_h;
    const long row_base = (long)b * a.U * a.H + kvh * share;
    const T *dout = (const T*)a.dout + row_base * a.D, *out = (const T*)a.o + row_base * a.D;
    const int key = tile * 32 * NWK + wk * 32 + (lane & 31);
    const bool any = tile * 32 * NWK < len;             // (workgroup-uniform)

    f32x16 dk[G::NDT], dv[G::NDT];
#pragma unroll
    for (int i = 0; i < G::NDT; ++i) dk[i] = dv[i] = f32x16{0};
    if (any) {
        constexpr int P = pow2_from(G::CPR);
        RowTile<T, DP, BR, P> tq, to, ty;
        RowWalk<G::EL, BR, P> at(a.q_u, a.q_h, (long)a.H * a.D, a.D, share, first, tid);
        RowWalk<1, BR, 1> ls(0, 0, a.H, 1, share, first, tid);         // (one row per thread)
        float rl = INFINITY;
        auto fetch = [&]() {
            tq.load(q, at.a, at, last, a.D);
            to.load(dout, at.b, at, last, a.D);
            ty.load(out, at.b, at, last, a.D);
            rl = ls.inside(0, last, 1) ? a.lse[row_base + ls.b[0]] - P_SHIFT<T> : INFINITY;      // rows behind the last: p = exp2(s - inf) = 0
            at.next();
            ls.next();
        };
        // (a tile of wider heads is asked for when it is stored: held through the products it would cost a wave per SIMD, which hides the wait better)
        constexpr bool EARLY = DP <= 32;
        if (EARLY) fetch();
        Frag<T> kf[G::NCH], vf[G::NCH];
#pragma unroll
        for (int c = 0; c < G::NCH; ++c) {
            kf[c] = vf[c] = no_frag<T>();
            if (key < len) {
                kf[c] = frag_at((const T*)a.k + b * a.k_b + kvh * a.k_h + (long)key * a.k_t, c * 16 + h * 8, a.D);
                vf[c] = frag_at((const T*)a.v + b * a.v_b + kvh * a.v_h + (long)key * a.v_t, c * 16 + h * 8, a.D);
            }
        }
        float f = DS_START<T>;
        for (int r0 = first; r0 < last; r0 += BR) {
            if (!EARLY) fetch();
            __syncthreads();
            tq.store(sQ, tid);
            to.store(sO, tid);
            to.products(ty, P_BACK, sD, tid);
            if (tid < BR) sL[tid] = rl;
            __syncthreads();
            if (EARLY && r0 + BR < last) fetch();
#pragma unroll
            for (int t = 0; t < RT; ++t) {
                const int x0 = (wr * RT + t) * 32;
                if (r0 + x0 >= last) continue;
                f32x16 s = f32x16{0}, dp = f32x16{0};
#pragma unroll
                for (int c = 0; c < G::NCH; ++c) {
                    s = mma<T>(s, sQ.row(x0 + (lane & 31), c, h), kf[c]);
                    dp = mma<T>(dp, sO.row(x0 + (lane & 31), c, h), vf[c]);
                }
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const f32x4 ls = *(const f32x4*)(sL + x0 + 8 * x + 4 * h), de = *(const f32x4*)(sD + x0 + 8 * x + 4 * h);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int r = 4 * x + e;
                        s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], a.c, -ls[e]));
                        dp[r] = s[r] * fmaf(dp[r], P_BACK, -de[e]);
                        if constexpr (DS_SCALED<T>) dp[r] *= f;
                    }
                }
                follow_ds<T>(f, dp, dk);
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const Frag<T> p = pack<T>(s, c), ds = pack<T>(dp, c);
#pragma unroll
                    for (int i = 0; i < G::NDT; ++i) {
                        dv[i] = mma<T>(dv[i], sO.column(x0, c, i * 32, lane), p);
                        dk[i] = mma<T>(dk[i], sQ.column(x0, c, i * 32, lane), ds);
                    }
                }
            }
        }
        undo_ds<T>(f, dk);
    }
    if constexpr (NWR > 1) {
        if (any) {
            float* red = (float*)smem;
            auto join = [&](f32x16* acc) {
                __syncthreads();
                if (wr != 0) {
#pragma unroll
                    for (int i = 0; i < G::NDT; ++i)
#pragma unroll
                        for (int r = 0; r < 16; ++r) red[(wave * DP + i * 32 + 8 * (r >> 2) + 4 * h + (r & 3)) * 32 + (lane & 31)] = acc[i][r];
                }
                __syncthreads();
                if (wr == 0) {
#pragma unroll
                    for (int x = 1; x < NWR; ++x)
#pragma unroll
                        for (int i = 0; i < G::NDT; ++i)
#pragma unroll
                            for (int r = 0; r < 16; ++r) acc[i][r] += red[((wave + x) * DP + i * 32 + 8 * (r >> 2) + 4 * h + (r & 3)) * 32 + (lane & 31)];
                }
            };
            join(dk);
            join(dv);
        }
        if (wr != 0) return;
    }
    if (key >= a.T) return;
    const long at = (((long)b * a.T + key) * a.Hkv + kvh) * a.D, all = (long)a.B * a.T * a.Hkv * a.D;
    float* part = a.part_k + split * all + at;
#pragma unroll
    for (int i = 0; i < G::NDT; ++i)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const int d = i * 32 + 8 * x + 4 * h;
            f32x4 y = {dk[i][4 * x], dk[i][4 * x + 1], dk[i][4 * x + 2], dk[i][4 * x + 3]};
            f32x4 z = {dv[i][4 * x], dv[i][4 * x + 1], dv[i][4 * x + 2], dv[i][4 * x + 3]};
            if (key >= len) y = z = f32x4{0, 0, 0, 0};     // (a masked key's lane held whatever the zeroed operands gave)
            if (d < a.D) {
                put(a.nk > 1 ? part + d : nullptr, (T*)a.dk + at + d, y * a.scale);
                put(a.nk > 1 ? part + a.nk * all + d : nullptr, (T*)a.dv + at + d, z * P_BACK);
            }
        }
}

// One launch: the side whose workgroups take longer first (`keys_first`, else the row side's), its `first` blocks before the other's.
template <class T, int DP, int NW, int DEPTH>
__global__ __launch_bounds__(CA_THREADS, (BWD_PER_CU<T, DP, NW>)) void cross_attn_bwd_kernel(CrossAttnArgs a, int first, int keys_first) {
    constexpr int A = DKV_BYTES<T, DP, NW, 4 / NW, DEPTH>(), B = DQ_BYTES<T, DP, NW, 4 / NW, DEPTH>();
    __shared__ __attribute__((aligned(16))) char smem[A > B ? A : B];
    const bool second = (int)blockIdx.x >= first;
    const int block = second ? blockIdx.x - first : blockIdx.x;
    if (second != (keys_first != 0)) cross_attn_dkv<T, DP, NW, 4 / NW, DEPTH>(a, block, smem);
    else cross_attn_dq<T, DP, NW, 4 / NW, DEPTH>(a, block, smem);
}

// ---- launch rules -----------------------------------------------------------------------------------------------------------
constexpr int CA_CUS = 256;

// Forward: 128 rows per workgroup read (and split into terms) every key once per 128 rows instead of once per 32: taken where that gives every CU a
// workgroup, or where the keys are long enough to be cut into ranges that do (4 x 333 rows of 8 heads over 2999 fp32 keys: 139 us at 32 rows,
// 66 us at 128 rows in five ranges).
bool fwd_wide(int B, int U, int T, int H, int Hkv) {
    const long R = (long)U * (H / Hkv), n = (long)B * Hkv * ((R + 127) / 128);
    return R > 64 && (n >= CA_CUS || T >= 1024);
}

int check_grid(long grid) { return grid <= 0x7fffffffL ? LAS_OK : fail(LAS_ERR_UNSUPPORTED, "cross attention: %s%ld workgroups", "", grid); }

template <class K> int launch(K kernel, long grid, CrossAttnArgs a, hipStream_t stream) {
    if (grid == 0) return LAS_OK;
    LAS_TRY(check_grid(grid));
    a.longest_first = a.lens && a.B > 1 && a.B <= 64 && grid > 2 * CA_CUS;
    hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(CA_THREADS), 0, stream, a);
    LAS_LAUNCH_CHECK();
    return LAS_OK;
}

// Two shapes of a workgroup's four waves: wide, 128 rows (keys) with every wave at all of a key (row) tile; narrow, fewer rows, the waves side by side over
// the key (row) tile too and joined at the end: 64 rows, in the forward of small 16-bit heads 32.  (32 rows in the backward, or of wide heads, hold
// tiles of 128 of the other side: one workgroup to a CU, 20 against 12.5 us at 8 x 128 over 375 heads of 64, 70 against 27 at 4 x 400 over 500 heads of 96.)
template <class T, int DP> constexpr int NARROW = sizeof(T) == 4 || DP > 64 ? 2 : 1;

template <class T, int DP> int fwd_dp(const CrossAttnArgs& a, hipStream_t stream) {
    constexpr int NQ = NARROW<T, DP>;
    const long R = (long)a.U * (a.H / a.Hkv);
    int rc;
    if (fwd_wide(a.B, a.U, a.T, a.H, a.Hkv)) rc = launch(cross_attn_fwd_kernel<T, DP, 4, 1, DEEP_FWD<T, DP>>, blocks_of(a, a.nsplit * ((R + 127) / 128)), a, stream);
    else rc = launch(cross_attn_fwd_kernel<T, DP, NQ, 4 / NQ, 1>, blocks_of(a, a.nsplit * ((R + 32 * NQ - 1) / (32 * NQ))), a, stream);
    if (rc != LAS_OK || a.nsplit == 1) return rc;
    if ((long)a.B * a.U * a.H <= CA_CUS) return launch(cross_attn_join_row_kernel<T>, (long)a.B * a.U * a.H, a, stream);
    const long items = (long)a.B * a.U * a.H * (a.D / 4);
    return launch(cross_attn_join_kernel<T>, (items + CA_THREADS - 1) / CA_THREADS, a, stream);
}

// Backward: both sides wide where that makes two workgroups per CU, fp32 one (its narrow shape has a CU to itself too: 41 against 56 us at 32 x 128
// over 100 heads of 128; not where most of 128 rows would be empty), else both narrow.
bool bwd_wide(int B, int U, int T, int H, int Hkv, bool fp32) {
    const long R = (long)U * (H / Hkv), n = (long)B * Hkv * ((R + 127) / 128 + (T + 127) / 128);
    return n >= 2 * CA_CUS || (fp32 && R > 64 && n >= CA_CUS);
}

// (a side whose gradients nobody wants is left out)
template <class T, int DP> int bwd_dp(const CrossAttnArgs& args, hipStream_t stream) {
    CrossAttnArgs a = args;
    const long R = (long)a.U * (a.H / a.Hkv);
    const bool wide = bwd_wide(a.B, a.U, a.T, a.H, a.Hkv, sizeof(T) == 4);
    const long per = wide ? 128 : 64, rows = a.dq ? blocks_of(a, a.nq * ((R + per - 1) / per)) : 0, keys = a.dk ? blocks_of(a, a.nk * ((a.T + per - 1) / per)) : 0;
    if (rows + keys == 0) return LAS_OK;
    LAS_TRY(check_grid(rows + keys));
    a.longest_first = a.lens && a.B > 1 && a.B <= 64 && rows + keys > 2 * CA_CUS;
    // (a workgroup of the key side goes over the rows in 16 products a tile, one of the row side over the keys in 12)
    const int keys_first = R / a.nk * 4 >= a.T / a.nq * 3, first = (int)(keys_first ? keys : rows);
    if (wide) hipLaunchKernelGGL((cross_attn_bwd_kernel<T, DP, 4, DEEP_BWD<T, DP>>), dim3((unsigned)(rows + keys)), dim3(CA_THREADS), 0, stream, a, first, keys_first);
    else hipLaunchKernelGGL((cross_attn_bwd_kernel<T, DP, 2, 1>), dim3((unsigned)(rows + keys)), dim3(CA_THREADS), 0, stream, a, first, keys_first);
    LAS_LAUNCH_CHECK();
    const long nr = (long)a.B * a.U * a.H * a.D / 4, nkv = (long)a.B * a.T * a.Hkv * a.D / 4;
    auto sum = [&](const float* part, int n, long count, void* to) -> int {
        const long grid = (count + CA_THREADS - 1) / CA_THREADS;
        if (grid == 0) return LAS_OK;
        LAS_TRY(check_grid(grid));
        hipLaunchKernelGGL(cross_attn_sum_kernel<T>, dim3((unsigned)grid), dim3(CA_THREADS), 0, stream, part, n, count, (T*)to);
        LAS_LAUNCH_CHECK();
        return LAS_OK;
    };
    if (a.dq && a.nq > 1) LAS_TRY(sum(a.part_q, a.nq, nr, a.dq));
    if (a.dk && a.nk > 1) {
        LAS_TRY(sum(a.part_k, a.nk, nkv, a.dk));
        LAS_TRY(sum(a.part_k + (long)a.nk * nkv * 4, a.nk, nkv, a.dv));
    }
    return LAS_OK;
}

template <class T> int by_dim(const CrossAttnArgs& a, bool bwd, hipStream_t stream) {
    switch ((a.D + 31) / 32) {
        case 1: return bwd ? bwd_dp<T, 32>(a, stream) : fwd_dp<T, 32>(a, stream);
        case 2: return bwd ? bwd_dp<T, 64>(a, stream) : fwd_dp<T, 64>(a, stream);
        case 3: return bwd ? bwd_dp<T, 96>(a, stream) : fwd_dp<T, 96>(a, stream);
        default: return bwd ? bwd_dp<T, 128>(a, stream) : fwd_dp<T, 128>(a, stream);
    }
}

}  // namespace

// Key ranges of a forward call: as many as fill the chip twice over where the rows alone do not, none shorter than 256 keys (512 at 128 rows, 128 of
// fp32, whose tiles take longer): a range costs its workgroups a partial result in fp32 and the joining launch.  Below 128 rows they are counted in tiles of
// 32 although fp32 and heads above 64 launch 64 rows: 33 to 64 rows to a key head count as two and are cut only where the GPU is less than half full.  Counted
// as the one workgroup that they are, heads of 128 over 900 keys: 32 x 4 x 64 rows 23.7 -> 24.4 us bf16, 71 -> 61 fp32; 40 x 4 x 64 23.4 -> 25.7, 72 -> 68; 24 x 4 x 100
// 22.9 -> 25.1, 71 -> 87; 48 x 4 x 64 over 600 18.1 -> 23.3, 52 -> 66.
int cross_attn_splits(int B, int U, int T, int H, int Hkv, int dtype) {
    const long R = (long)U * (H / Hkv), per = fwd_wide(B, U, T, H, Hkv) ? 128 : 32, wgs = (long)B * Hkv * ((R + per - 1) / per);
    const long want = wgs >= CA_CUS ? 1 : 2 * CA_CUS / (wgs > 0 ? wgs : 1), most = T / (dtype == 0 ? 128 : per == 128 ? 512 : 256);
    return (int)(want < 2 || most < 2 ? 1 : (want < most ? want : most));
}

// Ranges of a backward side that has few workgroups of long loops: of the keys for a few rows, of the rows for a few keys; as many as give every CU a
// workgroup, none shorter than 256 (128 of fp32), where that side has at most half a workgroup per CU, the key side, which has twice the partial sums, a
// quarter.  A range costs its partial sum in fp32 and the launches that add them up.  (16-bit heads of 64: 8 heads of 20 rows over 20000, 451 -> 38 us; 8 heads
// of 2000 rows on one over 50, 360 -> 58; 4 x 100 over 3000, 77 -> 36, fp32 201 -> 84.  8 x 300 rows on 2 heads of 128 over 1700, 108 key workgroups, 169 against 178.)
void cross_attn_bwd_splits(int B, int U, int T, int H, int Hkv, int dtype, int& nq, int& nk) {
    const long R = (long)U * (H / Hkv), bh = (long)B * Hkv, per = bwd_wide(B, U, T, H, Hkv, dtype == 0) ? 128 : 64;
    auto ranges = [&](long tiles, long length, int few) {
        const long wgs = bh * tiles, most = length / (dtype == 0 ? 128 : 256), want = wgs <= 0 || wgs > few ? 1 : CA_CUS / wgs;
        return (int)(want < 2 || most < 2 ? 1 : want < most ? want : most);
    };
    nq = ranges((R + per - 1) / per, T, CA_CUS / 2);
    nk = ranges((T + per - 1) / per, R, CA_CUS / 4);
}

int cross_attn(const CrossAttnArgs& a, int dtype, bool bwd, hipStream_t stream) {
    switch (dtype) {
        case 0: return by_dim<float>(a, bwd, stream);
        case 1: return by_dim<__bf16>(a, bwd, stream);
        default: return by_dim<_Float16>(a, bwd, stream);
    }
}

}  // namespace las
