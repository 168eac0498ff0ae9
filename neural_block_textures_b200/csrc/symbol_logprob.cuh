// Log probabilities of given symbols under a predictor's logits, with entropy and top alternatives, and the gradient:
// ntcb_symbol_logprobs / ntcb_symbol_logprobs_grad (include/ntc_b200.h).
//
// Forward, for a row x[0..V) and its symbol t:
//   m = max x, d = x - m, s = sum e^d, u = sum e^d d
//   lse = m + log s, logp = (x_t - m) - log s, H = log s - u / s
// and the topk largest logits in order (value first, then the lower index). One read of the logits does all of it, in 32
// bits whatever their type. Rows: no finite logit (everything masked) gives lse = logp = -inf, H = 0 and no alternatives;
// a NaN or +inf gives NaN.
//
// Approximations, by choice: 2^y is the hardware's ex2.approx.ftz (2^-22 relative; results below 2^-126 are 0), and u / s and
// a renormalised row's 1 / s are __fdividef (two units in the last place).
//
// Exponents (Scale below): e^d = 2^y with y = x L - mL in one fused multiply-add, L = log2 e and mL = m L rounded. All
// y of a row are off by the same mL - m L, which is known exactly and put back where the row is finished, so the only
// rounding is y's own. y is clamped at kYLow, where 2^y is 0 in 32 bits: -inf and the type's lowest value then add 0 to u,
// not 0 * inf; the clamp passes NaN on. Two elements share an instruction (fma.f32x2) where they can: the kernels are
// bound by instruction issue and by the exponential unit (16 a clock and SM) before they are bound by memory.
//
// Gradient: p_j = e^(x_j - lse); dx_j = [j = t] dlogp - p_j (dlogp + dH (x_j - lse + H)).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <cstring>
#include <type_traits>

#include "../../include/ntc_b200.h"
#include "symbol_logprob.h"

namespace ntcb {
namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kYLow = -200.0f;        // 2^-200 is 0 in 32 bits
constexpr float kLowest = -3.402823466e38f;
constexpr unsigned kFull = 0xffffffffu;
constexpr float kNegInf = -INFINITY;

// ------------------------------------------------------------------------------------------------------- elements

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float exp2_of(float y) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(y));
    return r;
}

__device__ __forceinline__ long long load_symbol(const void* p, int type, long long i) {
    switch (type) {
        case NTCB_SYM_U8: return static_cast<const uint8_t*>(p)[i];
        case NTCB_SYM_I16: return static_cast<const int16_t*>(p)[i];
        case NTCB_SYM_I32: return static_cast<const int32_t*>(p)[i];
        default: return static_cast<const long long*>(p)[i];
    }
}

// A vector is 16 bytes of a row: VEC elements. Rows may start anywhere, so vector c of a row holds its elements
// [c VEC - shift, (c + 1) VEC - shift) with the shift that puts vectors on 16-byte boundaries.
template <class T> constexpr int VEC = 16 / (int)sizeof(T);
template <class T>
__device__ __forceinline__ int row_shift(const T* row) { return (int)((reinterpret_cast<uintptr_t>(row) / sizeof(T)) % VEC<T>); }

// Loads of the forward pass go through the read-only path; the gradient may be written over its logits, so its loads are
// ordinary ones (streamed: nothing is read twice).
template <bool READ_ONLY, class W>
__device__ __forceinline__ W load(const W* p) {
    if constexpr (READ_ONLY) return __ldg(p);
    else return __ldcs(p);
}
template <class T> __device__ __forceinline__ uint32_t raw_of(T v) {
    if constexpr (sizeof(T) == 4) return __float_as_uint(v);
    else if constexpr (std::is_same_v<T, __half>) return __half_as_ushort(v);
    else return __bfloat16_as_ushort(v);
}
template <class T> constexpr uint32_t kRawNegInf = sizeof(T) == 4 ? 0xff800000u : std::is_same_v<T, __half> ? 0xfc00u : 0xff80u;

// Elements [j0, j0 + n) of a row one by one, -inf outside [0, V), packed into 32-bit words.
template <class T, bool READ_ONLY, int WORDS>
__device__ __forceinline__ void load_words(const T* row, int j0, int V, uint32_t (&w)[WORDS]) {
    constexpr int per = 4 / (int)sizeof(T);
#pragma unroll
    for (int i = 0; i < WORDS; i++) {
        w[i] = 0;
#pragma unroll
        for (int e = 0; e < per; e++) {
            const int j = j0 + i * per + e;
            w[i] |= (j >= 0 && j < V ? raw_of(load<READ_ONLY>(row + j)) : kRawNegInf<T>) << (16 * e);
        }
    }
}
// The vector at element j0: one load where it lies inside the row, else its halves, else its elements.
template <bool READ_ONLY, class T>
__device__ __forceinline__ uint4 load_vec(const T* row, int j0, int V) {
    constexpr int N = VEC<T>;
    if (j0 >= 0 && j0 + N <= V) return load<READ_ONLY>(reinterpret_cast<const uint4*>(row + j0));
    uint32_t h[2][2];
#pragma unroll
    for (int k = 0; k < 2; k++) {
        const int j = j0 + k * N / 2;
        if (j >= 0 && j + N / 2 <= V) {
            const uint2 a = load<READ_ONLY>(reinterpret_cast<const uint2*>(row + j));
            h[k][0] = a.x; h[k][1] = a.y;
        } else {
            load_words<T, READ_ONLY>(row, j, V, h[k]);
        }
    }
    return make_uint4(h[0][0], h[0][1], h[1][0], h[1][1]);
}
template <class T>
__device__ __forceinline__ void expand(const uint4& a, float (&v)[VEC<T>]) {
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (sizeof(T) == 4) v[i] = __uint_as_float(w[i]);
        else if constexpr (std::is_same_v<T, __nv_bfloat16>) { v[2 * i] = __uint_as_float(w[i] << 16); v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
        else { __half2 h; memcpy(&h, &w[i], 4); const float2 f = __half22float2(h); v[2 * i] = f.x; v[2 * i + 1] = f.y; }
    }
}
// The largest of a number of vectors' elements; NaN counts for nothing. 16-bit types in pairs.
template <class T, int C>
__device__ __forceinline__ float max_of(const uint4 (&a)[C]) {
    if constexpr (sizeof(T) == 4) {
        float m = kNegInf;
#pragma unroll
        for (int c = 0; c < C; c++)
            m = fmaxf(fmaxf(fmaxf(m, __uint_as_float(a[c].x)), fmaxf(__uint_as_float(a[c].y), __uint_as_float(a[c].z))), __uint_as_float(a[c].w));
        return m;
    } else {
        typedef typename std::conditional<std::is_same_v<T, __half>, __half2, __nv_bfloat162>::type P;
        const auto pair = [](uint32_t w) { P p; memcpy(&p, &w, 4); return p; };
        P m = __hmax2(__hmax2(pair(a[0].x), pair(a[0].y)), __hmax2(pair(a[0].z), pair(a[0].w)));
#pragma unroll
        for (int c = 1; c < C; c++) m = __hmax2(m, __hmax2(__hmax2(pair(a[c].x), pair(a[c].y)), __hmax2(pair(a[c].z), pair(a[c].w))));
        return fmaxf(fmaxf(to_f32(m.x), to_f32(m.y)), kNegInf);
    }
}

// ------------------------------------------------------------------------------------------------------ a row's sums

// The exponents of one maximum (or lse) m. Near zero (|m| < 4096) y = x L + b, off by `off` = mL - m L for every x (at most
// 2^-11, so that 2^off is 1 + off ln 2); far from it, where that would grow, y = (x - m) L, an instruction more and exact
// where it counts.
struct Scale {
    float m, b, off;
    bool far;
    __device__ __forceinline__ explicit Scale(float at) : m(at) {
        far = !(fabsf(at) < 4096.0f);
        b = -(at * kLog2e);
        off = far ? 0.0f : -fmaf(at, kLog2e, b);
    }
};
struct Sums { float m, s, u; };

template <bool FAR>
__device__ __forceinline__ float2 exponents(float x0, float x1, const Scale& c) {
    const float2 x = make_float2(x0, x1), L = make_float2(kLog2e, kLog2e);
    float2 y;
    if constexpr (FAR) y = __fmul2_rn(__fadd2_rn(x, make_float2(-c.m, -c.m)), L);
    else y = __ffma2_rn(x, L, make_float2(c.b, c.b));
    y.x = max_nan(y.x, kYLow); y.y = max_nan(y.y, kYLow);
    return y;
}
// Adds the elements of C vectors with the exponents of c to s and u (pairs of partial sums).
template <bool FAR, class T, int C>
__device__ __forceinline__ void add_exp(const uint4 (&raw)[C], const Scale& c, float2& s, float2& u) {
#pragma unroll
    for (int k = 0; k < C; k++) {
        float x[VEC<T>];
        expand<T>(raw[k], x);
#pragma unroll
        for (int i = 0; i < VEC<T>; i += 2) {
            const float2 y = exponents<FAR>(x[i], x[i + 1], c);
            const float2 e = make_float2(exp2_of(y.x), exp2_of(y.y));
            s = __fadd2_rn(s, e);
            u = __ffma2_rn(e, y, u);
        }
    }
}
template <class T, int C>
__device__ __forceinline__ void add_exp(const uint4 (&raw)[C], const Scale& c, float2& s, float2& u) {
    if (c.far) add_exp<true, T>(raw, c, s, u);
    else add_exp<false, T>(raw, c, s, u);
}
// s and u of one maximum, without the common offset and in natural units: the true exponents are y + off, so
// sum e^d = 2^off s and sum e^d d = 2^off ln 2 (u + off s), both with 2^off = 1 + off ln 2 (off^2 is below 2^-22).
__device__ __forceinline__ Sums sums_of(const Scale& c, float s, float u) {
    const float grow = c.off * kLn2, t = kLn2 * fmaf(s, c.off, u);
    return Sums{c.m, fmaf(s, grow, s), fmaf(t, grow, t)};
}
// Joins two partial rows: s and u are relative to m.
__device__ __forceinline__ Sums join(const Sums& a, const Sums& b) {
    const float m = fmaxf(a.m, b.m);
    const float da = max_nan(a.m - m, -150.0f), db = max_nan(b.m - m, -150.0f);
    const float ea = exp2_of(da * kLog2e), eb = exp2_of(db * kLog2e);
    Sums r;
    r.m = m;
    r.s = a.s * ea + b.s * eb;
    r.u = (a.u + a.s * da) * ea + (b.u + b.s * db) * eb;
    return r;
}

struct RowOut { float lse, entropy, log_s, m; bool empty, bad; };
__device__ __forceinline__ RowOut finish_row(const Sums& q) {
    RowOut o;
    o.bad = !(q.s == q.s);
    o.empty = q.s == 0.0f;
    o.m = q.m;
    o.log_s = logf(q.s);
    o.lse = o.empty ? kNegInf : q.m + o.log_s;
    o.entropy = o.empty ? 0.0f : o.log_s - __fdividef(q.u, q.s);
    return o;
}
// The row's scalars, by one thread; t is its symbol (fetched with the row), xt the symbol's logit, NaN where there is none.
__device__ __forceinline__ void write_row(const RowArgs& a, long long r, float xt, long long t, const RowOut& o) {
    a.logp[r] = t < 0 ? 0.0f : o.bad ? NAN : o.empty ? (t < a.V ? kNegInf : NAN) : (xt - o.m) - o.log_s;
    a.entropy[r] = o.bad ? NAN : o.entropy;
    a.lse[r] = o.bad ? NAN : o.lse;
}
// The logit is in L1 or L2 by the time the row is summed up.
template <class T>
__device__ __forceinline__ void write_row(const RowArgs& a, long long r, const T* row, long long t, const RowOut& o) {
    write_row(a, r, t >= 0 && t < a.V ? to_f32(row[t]) : NAN, t, o);
}

// ------------------------------------------------------------------------------------------------------------- keys

// A logit and its position as one integer: larger value first, then the lower position; 0 is no logit. The value part
// orders as the numbers do: all bits of a negative one turned, the sign of a positive one (-0 is made +0 first). 16-bit
// logits at up to 2^16 positions fit 32 bits (one compare, one shuffle, one warp reduction), others take 64.
template <class T, class K>
__device__ __forceinline__ K key_of(float x, int pos) {
    uint32_t b = __float_as_uint(x + 0.0f);
    if constexpr (std::is_same_v<T, __half> && sizeof(K) == 4) b = (uint32_t)__half_as_ushort(__float2half_rn(x + 0.0f)) << 16;
    const uint32_t o = b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
    if constexpr (sizeof(K) == 4) return (o & 0xffff0000u) | (0xffffu - (uint32_t)pos);
    else return ((K)o << 32) | (uint32_t)~pos;
}
template <class T, class K>
__device__ __forceinline__ float key_value(K k) {
    const uint32_t o = sizeof(K) == 4 ? (uint32_t)k & 0xffff0000u : (uint32_t)((unsigned long long)k >> 32);
    uint32_t b = o ^ ((uint32_t)((int32_t)~o >> 31) | 0x80000000u);
    if constexpr (sizeof(K) == 4) b &= 0xffff0000u;
    if constexpr (std::is_same_v<T, __half> && sizeof(K) == 4) return __half2float(__ushort_as_half((unsigned short)(b >> 16)));
    else return __uint_as_float(b);
}
template <class K>
__device__ __forceinline__ int key_index(K k) {
    if constexpr (sizeof(K) == 4) return (int)(0xffffu - (k & 0xffffu));
    else return (int)(~(uint32_t)k);
}
// The keys of a vector whose first element has position pos (known when compiled). Pairs of 16-bit logits are turned
// together, and products and sums take what they can off the logic unit, which bounds the kernels that sort.
template <class T, class K>
__device__ __forceinline__ void keys_of(const uint4& a, int pos, K* k) {
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (sizeof(T) == 4) k[i] = key_of<T, K>(__uint_as_float(w[i]), pos + i);
        else {
            typedef typename std::conditional<std::is_same_v<T, __half>, __half2, __nv_bfloat162>::type P;
            P p;
            uint32_t b;
            memcpy(&p, &w[i], 4);
            if constexpr (std::is_same_v<T, __half>) p = __hadd2(p, __float2half2_rn(0.0f)); else p = __hadd2(p, __float2bfloat162_rn(0.0f));
            memcpy(&b, &p, 4);
            const uint32_t o = b ^ (((b >> 15) & 0x00010001u) * 0x7fffu + 0x80008000u);
            k[2 * i] = o * 65536u + (0xffffu - (uint32_t)(pos + 2 * i));
            k[2 * i + 1] = (o & 0xffff0000u) | (0xffffu - (uint32_t)(pos + 2 * i + 1));
        }
    }
}
__device__ __forceinline__ void write_top(const RowArgs& a, long long r, int i, float v, int index, const RowOut& o) {
    const bool none = o.bad || v == kNegInf;
    a.top_ids[r * a.topk + i] = none ? -1 : index;
    a.top_logp[r * a.topk + i] = o.bad ? NAN : none ? kNegInf : (v - o.m) - o.log_s;
}
template <class T, class K>
__device__ __forceinline__ void write_top(const RowArgs& a, long long r, int i, K k, int shift, const RowOut& o) {
    write_top(a, r, i, k ? key_value<T, K>(k) : kNegInf, key_index(k) - shift, o);
}

// The largest key of G neighbouring lanes, in all of them.
template <int G, class K>
__device__ __forceinline__ K group_max(K k) {
    if constexpr (G == 32 && sizeof(K) == 4) return __reduce_max_sync(kFull, k);
    else if constexpr (G == 32) {
        const uint32_t hi = (uint32_t)(k >> 32), top = __reduce_max_sync(kFull, hi);
        return ((K)top << 32) | __reduce_max_sync(kFull, hi == top ? (uint32_t)k : 0u);
    } else {
#pragma unroll
        for (int w = G / 2; w; w >>= 1) k = max(k, __shfl_xor_sync(kFull, k, w));
        return k;
    }
}

// Batcher's odd-even merge sort of a thread's N keys, largest first (K. E. Batcher, "Sorting networks and their
// applications", 1968).
template <int N, class K>
__device__ __forceinline__ void sort_keys(K* a) {
#pragma unroll
    for (int p = 1; p < N; p <<= 1)
#pragma unroll
        for (int k = p; k >= 1; k >>= 1)
#pragma unroll
            for (int j = k % p; j + k < N; j += 2 * k)
#pragma unroll
                for (int i = 0; i < k; i++)
                    if (i + j + k < N && (i + j) / (2 * p) == (i + j + k) / (2 * p)) {
                        const K x = a[i + j], y = a[i + j + k];
                        a[i + j] = max(x, y);
                        a[i + j + k] = min(x, y);
                    }
}
// The L largest of a thread's E keys, in order, into k[0 .. L): lists of L are sorted and joined by their larger halves.
template <int E, int L, class K>
__device__ __forceinline__ void largest_keys(K* k) {
    if constexpr (L == 1) {
#pragma unroll
        for (int i = 1; i < E; i++) k[0] = max(k[0], k[i]);
    } else {
        sort_keys<L>(k);
#pragma unroll
        for (int c = L; c < E; c += L) {
            sort_keys<L>(k + c);
#pragma unroll
            for (int i = 0; i < L; i++) k[i] = max(k[i], k[c + L - 1 - i]);   // bitonic
#pragma unroll
            for (int h = L / 2; h; h >>= 1)
#pragma unroll
                for (int i = 0; i < L; i++)
                    if (!(i & h)) { const K x = k[i], y = k[i + h]; k[i] = max(x, y); k[i + h] = min(x, y); }
        }
    }
}

// Sorts one key per lane, largest first (bitonic).
template <class K>
__device__ __forceinline__ K sort32(K k, int lane) {
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
        for (int step = size >> 1; step; step >>= 1) {
            const K other = __shfl_xor_sync(kFull, k, step);
            const bool keep_max = ((lane & step) == 0) == ((lane & size) == 0);
            k = keep_max ? max(k, other) : min(k, other);
        }
    return k;
}
// The 32 largest of two sorted lists, sorted: the larger of a[i] and b[31 - i] is a bitonic sequence of them.
template <class K>
__device__ __forceinline__ K merge32(K a, K b, int lane) {
    K k = max(a, __shfl_sync(kFull, b, 31 - lane));
#pragma unroll
    for (int step = 16; step; step >>= 1) {
        const K other = __shfl_xor_sync(kFull, k, step);
        k = (lane & step) == 0 ? max(k, other) : min(k, other);
    }
    return k;
}

// ------------------------------------------------------------------------------------------- rows in a few registers

// The place of the first of a lane's elements that equals v (its vector's number c * G + lane times VEC, plus the
// element's): -1 where none does. 16-bit types compare in pairs.
template <class T, int G, int C>
__device__ __forceinline__ int first_equal(const uint4 (&raw)[C], float v, int lane) {
    constexpr int N = VEC<T>;
    int at = -1;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int c = C - 1; c >= 0; c--) {
            float x[N];
            expand<T>(raw[c], x);
#pragma unroll
            for (int i = N - 1; i >= 0; i--)
                if (x[i] == v) at = c * G * N + i;
        }
    } else {
        typedef typename std::conditional<std::is_same_v<T, __half>, __half2, __nv_bfloat162>::type P;
        P vv;
        if constexpr (std::is_same_v<T, __half>) vv = __float2half2_rn(v); else vv = __float2bfloat162_rn(v);   // exact, or no logit
        uint32_t hit = 0;   // bit w: the lower element of word w, bit 16 + w: the upper one
#pragma unroll
        for (int c = 0; c < C; c++) {
            const uint32_t w[4] = {raw[c].x, raw[c].y, raw[c].z, raw[c].w};
#pragma unroll
            for (int i = 0; i < 4; i++) {
                P p;
                memcpy(&p, &w[i], 4);
                hit |= __heq2_mask(p, vv) & (0x00010001u << (4 * c + i));
            }
        }
        if (hit) {
            const int lo = __ffs(hit & 0xffffu), hi = __ffs(hit >> 16);
            const int e = min(lo ? 2 * (lo - 1) : 64, hi ? 2 * (hi - 1) + 1 : 64);
            at = e / N * G * N + e % N;
        }
    }
    return at < 0 ? -1 : at + lane * N;
}

// A row as a group of G lanes fetches it.
template <class T, int C>
struct RowIn {
    uint4 raw[C];
    const T* row;
    long long r, t;
    int shift, V;   // V = 0: no row
};
template <class T, int G, int C>
__device__ __forceinline__ RowIn<T, C> fetch_row(const RowArgs& a, long long block) {
    RowIn<T, C> f;
    f.r = block * (256 / G) + threadIdx.x / G;
    const int lane = threadIdx.x % G;
    const bool live = f.r < a.rows;
    f.row = static_cast<const T*>(a.x) + (live ? f.r : 0) * a.stride;
    f.shift = row_shift(f.row);
    f.V = live ? a.V : 0;
#pragma unroll
    for (int c = 0; c < C; c++) f.raw[c] = load_vec<true>(f.row, (c * G + lane) * VEC<T> - f.shift, f.V);
    f.t = live && lane == 0 ? load_symbol(a.sym, a.sym_type, f.r * a.sym_stride) : -1;
    return f;
}

// G lanes hold one row of up to G * E elements (its shift counted in) in registers: the maximum is known before the
// exponentials, so nothing is rescaled. Alternatives (L > 0): each lane sorts the L largest of its E keys (4 for up to
// four alternatives, 8 for up to eight, E for more), and the row's next one is the largest of the lanes' first ones, which its lane then
// drops; a single alternative (L = 1) is the first logit that equals the maximum.
template <class T, int G, int E, int L>
__device__ __forceinline__ void rate_row(const RowArgs& a, const RowIn<T, E / VEC<T>>& f) {
    constexpr int N = VEC<T>, C = E / N;
    typedef typename std::conditional<sizeof(T) == 2, uint32_t, unsigned long long>::type K;
    const auto& raw = f.raw;
    const long long r = f.r, t = f.t;
    const int lane = threadIdx.x % G, shift = f.shift, V = f.V;
    const bool live = V > 0;
    float m = fmaxf(max_of<T>(raw), kLowest);   // a row of nothing but -inf keeps a finite maximum: y = -inf, e^d = 0
#pragma unroll
    for (int o = G / 2; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(kFull, m, o));
    const Scale sc(m);
    float2 s2 = make_float2(0.0f, 0.0f), u2 = s2;
    add_exp<T>(raw, sc, s2, u2);
    float2 q2 = make_float2(s2.x + s2.y, u2.x + u2.y);
#pragma unroll
    for (int o = G / 2; o; o >>= 1) q2 = __fadd2_rn(q2, make_float2(__shfl_xor_sync(kFull, q2.x, o), __shfl_xor_sync(kFull, q2.y, o)));
    const RowOut o = finish_row(sums_of(sc, q2.x, q2.y));
    if (live && lane == 0) {
        if constexpr (G == 1 && E <= 8) {   // the logit is at hand
            float xt = NAN;
#pragma unroll
            for (int c = 0; c < C; c++) {
                float x[N];
                expand<T>(raw[c], x);
#pragma unroll
                for (int i = 0; i < N; i++)
                    if (t >= 0 && t < V && c * N + i - shift == (int)t) xt = x[i];
            }
            write_row(a, r, xt, t, o);
        } else {
            write_row(a, r, f.row, t, o);
        }
    }
    if constexpr (L == 1) {
        int at = first_equal<T, G>(raw, m, lane);
#pragma unroll
        for (int w = G / 2; w; w >>= 1) at = (int)min((unsigned)at, (unsigned)__shfl_xor_sync(kFull, at, w));
        if (live && lane == 0) {
            const bool none = o.bad || o.empty;
            a.top_ids[r] = none ? -1 : at - shift;
            a.top_logp[r] = o.bad ? NAN : none ? kNegInf : -o.log_s;
        }
    } else if constexpr (L > 1 && G == 1 && C == 1 && sizeof(T) == 4) {
        // four fp32 logits: neighbours change places where the upper one is larger, which keeps equal ones in order (and
        // needs no 64-bit keys)
        float v[4];
        int id[4];
        expand<T>(raw[0], v);
#pragma unroll
        for (int i = 0; i < 4; i++) id[i] = i - shift;
#pragma unroll
        for (int n = 0; n < 4; n++)
#pragma unroll
            for (int i = n % 2; i + 1 < 4; i += 2) {
                const bool swap = v[i + 1] > v[i];
                const float x = swap ? v[i + 1] : v[i], y = swap ? v[i] : v[i + 1];
                const int ix = swap ? id[i + 1] : id[i], iy = swap ? id[i] : id[i + 1];
                v[i] = x; v[i + 1] = y; id[i] = ix; id[i + 1] = iy;
            }
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (live && j < a.topk) write_top(a, r, j, v[j], id[j], o);
    } else if constexpr (L > 1) {
        K k[E];
#pragma unroll
        for (int c = 0; c < C; c++) keys_of<T>(raw[c], c * G * N, k + c * N);
        largest_keys<E, L>(k);
#pragma unroll
        for (int i = 0; i < L; i++) k[i] -= (K)(lane * N);   // the lane's part of the positions
        if constexpr (G == 1) {
#pragma unroll
            for (int j = 0; j < L; j++)
                if (live && j < a.topk) write_top<T>(a, r, j, k[j], shift, o);
        } else {
            K mine = 0;   // the alternative that this lane writes
            for (int j = 0; j < a.topk; j++) {
                const K g = group_max<G>(k[0]);
                if (k[0] == g) {
#pragma unroll
                    for (int i = 0; i + 1 < L; i++) k[i] = k[i + 1];
                    k[L - 1] = 0;
                }
                if (lane == j % G) mine = g;
                if (j % G == G - 1 || j + 1 == a.topk) {
                    const int at = j - j % G + lane;
                    if (live && at <= j) write_top<T>(a, r, at, mine, shift, o);
                }
            }
        }
    }
}

// Measured: 2^18 x 256 bf16 29 us without alternatives (4.8 TB/s of the 6.5 that a copy reaches; the exponential and the logic
// unit each some 55 % busy), 35 with one, 73 with eight (the minima and maxima of the sorts, on the half-rate logic unit, 79 %
// busy), fp32 176 with eight (64-bit keys); 2^15 x 1024 fp32 at the memory's rate; 2^20 x 4
// fp32 9.2 and, with two alternatives, 12.4 us (instruction issue: the row's end is paid by every lane).
// One group of rows to a CTA. (CTAs that stay and fetch the next rows ahead were slower on short rows: 17 against 15 us for
// 2^20 rows of 4; the hardware's turnover of CTAs hides more.)
template <class T, int G, int E, int L>
__global__ void __launch_bounds__(256) k_logprobs_lanes(const RowArgs a) {
    static_assert(E % VEC<T> == 0, "whole vectors");
    rate_row<T, G, E, L>(a, fetch_row<T, G, E / VEC<T>>(a, blockIdx.x));
}

// ------------------------------------------------------------------------------------------------------- long rows

// Shared memory of one row's threads (W warps).
constexpr int kSlots = 16;     // parts of a thread's share of the row whose maxima are kept
constexpr int kWork = 256;     // parts that are read again
constexpr int kCand = 256;     // candidate alternatives
template <class K, int W>
struct LongShared {
    Sums part[W];
    Sums total;                 // this CTA's part of the row
    K top[32];                  // this CTA's alternatives
    K lists[W][32];             // the cluster's
    K cand[kCand];
    float most[W][32];          // the threads' maxima, sorted per warp
    float slot[kSlots][32 * W];
    unsigned short work[kWork];
    int nwork, ncand;
};

__device__ __forceinline__ unsigned cluster_rank() { unsigned r; asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.aligned;\nbarrier.cluster.wait.aligned;" ::: "memory");
}
template <class P>
__device__ __forceinline__ P peer_load(const P* p, unsigned rank) {   // a word of another CTA's shared memory
    const uint32_t local = (uint32_t)__cvta_generic_to_shared(p);
    uint32_t remote;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(rank));
    P v;
    if constexpr (sizeof(P) == 8) asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(remote));
    else if constexpr (std::is_same_v<P, float>) asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(remote));
    else asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(remote));
    return v;
}

// One row per W warps (R rows in a CTA when W = 1), or per cluster of C CTAs of one row's part each. Vector c of the row
// belongs to CTA c / per, and there to thread (c - first) % threads; a thread reads U vectors at a time.
// Alternatives: the threads keep the maxima of up to kSlots parts of their share. The topk-th largest of the threads'
// maxima bounds the row's topk-th logit from below, so only the parts whose maximum reaches it are read again (from L2,
// by all threads together) and the few logits that reach it are sorted. Where many logits equal the bound (a row of one
// value, a part masked by the lowest value) those above it are taken like this and the first equal ones in order; what
// still is too much is gone through by one warp with a running list of 32.
// Measured: 2048 x 65536 bf16 52 us (5.2 TB/s; the exponential unit alone needs 37), with 20 alternatives 62; 1024 x 65536
// fp32 50 us (5.4 TB/s); 1 x 65536 fp32 on eight CTAs 5 us, with 20 alternatives 8 (latency). Many alternatives: 30000 x 4099
// fp16 63 us without, 164 with 32; 2^25 bf16 logits in rows of 700 with 17 77 us, in rows of 1024 with 32 86 (the bound lets
// too many logits through, and one warp of a row sorts them while the others wait).
template <class T, class K, int W, int R>
__global__ void __launch_bounds__(32 * W * R) k_logprobs_long(const RowArgs a, int C) {
    constexpr int N = VEC<T>, kThreads = 32 * W, U = 4;
    __shared__ LongShared<K, W> shared[R];
    LongShared<K, W>& sh = shared[R > 1 ? threadIdx.x / kThreads : 0];
    const auto sync = [] { if constexpr (W == 1) __syncwarp(); else __syncthreads(); };
    const int tid = threadIdx.x % kThreads, lane = tid & 31, warp = tid >> 5;
    const unsigned rank = W > 1 && C > 1 ? cluster_rank() : 0;
    const long long r = R > 1 ? (long long)blockIdx.x * R + threadIdx.x / kThreads : (long long)(blockIdx.x / (unsigned)C);
    if (R > 1 && r >= a.rows) return;   // whole warps: rows of W = 1 share no barrier
    const T* row = static_cast<const T*>(a.x) + r * a.stride;
    const int shift = row_shift(row), V = a.V;
    const int nvec = (V + shift + N - 1) / N;
    const int per = (nvec + C - 1) / C, first = min(nvec, (int)rank * per), end = min(nvec, first + per);
    const int rounds = (end - first + U * kThreads - 1) / (U * kThreads);
    int lg = 0;   // rounds of a slot, as a power of two
    while ((rounds - 1) >> lg >= kSlots) lg++;
    float mine = kNegInf;                // this slot's largest logit (-inf: none)
    float most = kNegInf;                // this thread's largest logit
    int round = 0;
    Scale sc(kLowest);                   // of the running maximum
    float2 s2 = make_float2(0.0f, 0.0f), u2 = s2;
    for (int c = first + tid; c < end; c += U * kThreads) {
        uint4 raw[U];
#pragma unroll
        for (int k = 0; k < U; k++) raw[k] = load_vec<true>(row, c + k * kThreads < end ? (c + k * kThreads) * N - shift : V, V);
        const float gm = max_of<T>(raw);
        if (a.topk) {
            mine = fmaxf(mine, gm);
            if (((++round) & ((1 << lg) - 1)) == 0) {
                sh.slot[(round - 1) >> lg][tid] = mine;
                most = fmaxf(most, mine);
                mine = kNegInf;
            }
        }
        if (gm > sc.m) {   // y of what is summed so far moves
            const Scale to(gm);
            const float y = max_nan(fmaf(sc.m - gm, kLog2e, sc.off - to.off), kYLow), e = exp2_of(y);
            u2.x = (u2.x + s2.x * y) * e; u2.y = (u2.y + s2.y * y) * e;
            s2.x *= e; s2.y *= e;
            sc = to;
        }
        add_exp<T>(raw, sc, s2, u2);
    }
    Sums q = sums_of(sc, s2.x + s2.y, u2.x + u2.y);
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        const Sums p{__shfl_xor_sync(kFull, q.m, o), __shfl_xor_sync(kFull, q.s, o), __shfl_xor_sync(kFull, q.u, o)};
        q = join(q, p);
    }
    if (lane == 0) sh.part[warp] = q;
    const int slots = (rounds + (1 << lg) - 1) >> lg;
    if (a.topk) {
        for (int k = round >> lg; k < slots; k++) { sh.slot[k][tid] = mine; most = fmaxf(most, mine); mine = kNegInf; }
        if (tid == 0) sh.nwork = sh.ncand = 0;
        sh.most[warp][lane] = sort32(most, lane);
    }
    sync();
    if (a.topk) {
#pragma unroll
        for (int half = W / 2; half; half >>= 1) {
            if (warp < half) {
                const float k = merge32(sh.most[warp][lane], sh.most[warp + half][lane], lane);
                __syncwarp();
                sh.most[warp][lane] = k;
            }
            sync();
        }
        const float least = sh.most[0][a.topk - 1];   // -inf when fewer threads than topk hold a logit
        // The logits that reach `least` (STRICT: that are above it) into cand; false where the lists do not hold them.
        const auto collect = [&](auto strict) {
            const auto reaches = [&](float v) { return strict ? v > least : v >= least && v > kNegInf; };
            if (reaches(most))
                for (int k = 0; k < slots; k++)
                    if (reaches(sh.slot[k][tid])) {
                        const int p = atomicAdd(&sh.nwork, 1);
                        if (p < kWork) sh.work[p] = (unsigned short)(k * kThreads + tid);
                    }
            sync();
            const int nwork = min(sh.nwork, kWork), each = U << lg;
            for (int item = tid; item < nwork * each; item += kThreads) {
                if (*const_cast<volatile int*>(&sh.ncand) > kCand) break;   // the additions to it are one after another
                const int w = sh.work[item / each], k = item % each;
                const int c = first + w % kThreads + ((w / kThreads) * each + k) * kThreads;
                if (c >= end) continue;
                float v[N];
                expand<T>(load_vec<true>(row, c * N - shift, V), v);
#pragma unroll
                for (int i = 0; i < N; i++)
                    if (reaches(v[i])) {
                        const int p = atomicAdd(&sh.ncand, 1);
                        if (p < kCand) sh.cand[p] = key_of<T, K>(v[i], c * N + i - shift);
                    }
            }
            sync();
            return sh.nwork <= kWork && sh.ncand <= kCand;
        };
        bool held = collect(std::false_type{}), ties = false;
        if (!held) {   // many logits equal to `least`: only the first of them count, found in order below
            sync();
            if (tid == 0) sh.nwork = sh.ncand = 0;
            sync();
            held = collect(std::true_type{});
            ties = true;
        }
        if (warp == 0) {
            K top = 0;
            const int count = sh.ncand;
            if (held) {
                for (int i = 0; i < count; i += 32) {
                    const K k = sort32(i + lane < count ? sh.cand[i + lane] : (K)0, lane);
                    top = i ? merge32(top, k, lane) : k;
                }
                if (ties) {   // the first topk logits that equal `least`, already in order
                    int found = 0;
                    __syncwarp();
                    for (int c0 = first; c0 < end && found < a.topk; c0 += 32) {
                        const int c = c0 + lane;
                        float v[N];
                        expand<T>(load_vec<true>(row, c < end ? c * N - shift : V, V), v);
                        int n = 0, before = 0;
#pragma unroll
                        for (int i = 0; i < N; i++) n += v[i] == least && v[i] > kNegInf;
                        int all = n;
#pragma unroll
                        for (int o = 1; o < 32; o <<= 1) { const int b = __shfl_up_sync(kFull, all, o); if (lane >= o) all += b; }
                        before = found + all - n;
#pragma unroll
                        for (int i = 0; i < N; i++)
                            if (v[i] == least && v[i] > kNegInf) {
                                if (before < 32) sh.cand[before] = key_of<T, K>(v[i], c * N + i - shift);
                                before++;
                            }
                        found += __shfl_sync(kFull, all, 31);
                    }
                    __syncwarp();
                    top = merge32(top, lane < found ? sh.cand[lane] : (K)0, lane);
                }
            } else {
                for (int c0 = first; c0 < end; c0 += 32) {
                    const int c = c0 + lane;
                    float v[N];
                    expand<T>(load_vec<true>(row, c < end ? c * N - shift : V, V), v);
#pragma unroll
                    for (int i = 0; i < N; i++) {
                        K k = v[i] >= least && v[i] > kNegInf ? key_of<T, K>(v[i], c * N + i - shift) : (K)0;
                        if (k < __shfl_sync(kFull, top, 31)) k = 0;
                        if (__any_sync(kFull, k != 0)) top = merge32(top, sort32(k, lane), lane);
                    }
                }
            }
            sh.top[lane] = top;
        }
    }
    if (W > 1 && warp == 0) {
        q = lane < W ? sh.part[lane] : Sums{kLowest, 0.0f, 0.0f};
#pragma unroll
        for (int o = W / 2; o; o >>= 1) {
            const Sums b{__shfl_xor_sync(kFull, q.m, o), __shfl_xor_sync(kFull, q.s, o), __shfl_xor_sync(kFull, q.u, o)};
            q = join(q, b);
        }
        if (lane == 0) sh.total = q;
    }
    if (W > 1 && C > 1) {
        sync();
        cluster_sync();
        if (rank == 0) {   // a warp for each CTA's list, then joined in pairs
            if (warp < C && a.topk) sh.lists[warp][lane] = peer_load(&sh.top[lane], warp);
            if (warp == 0) {
                q = lane < C ? Sums{peer_load(&sh.total.m, lane), peer_load(&sh.total.s, lane), peer_load(&sh.total.u, lane)} : Sums{kLowest, 0.0f, 0.0f};
#pragma unroll
                for (int o = W / 2; o; o >>= 1) {
                    const Sums b{__shfl_xor_sync(kFull, q.m, o), __shfl_xor_sync(kFull, q.s, o), __shfl_xor_sync(kFull, q.u, o)};
                    q = join(q, b);
                }
            }
            if (a.topk) {
                sync();
                for (int half = C / 2; half; half >>= 1) {
                    if (warp < half) {
                        const K k = merge32(sh.lists[warp][lane], sh.lists[warp + half][lane], lane);
                        __syncwarp();
                        sh.lists[warp][lane] = k;
                    }
                    sync();
                }
                if (warp == 0) sh.top[lane] = sh.lists[0][lane];
            }
        }
        cluster_sync();   // no CTA leaves while its shared memory is read
    }
    if (rank == 0 && warp == 0) {
        if (W > 1) { q.m = __shfl_sync(kFull, q.m, 0); q.s = __shfl_sync(kFull, q.s, 0); q.u = __shfl_sync(kFull, q.u, 0); }
        const RowOut o = finish_row(q);
        if (lane == 0) write_row(a, r, row, load_symbol(a.sym, a.sym_type, r * a.sym_stride), o);
        __syncwarp();
        if (lane < a.topk) write_top<T>(a, r, lane, sh.top[lane], 0, o);
    }
}

// -------------------------------------------------------------------------------------------------------- gradient

// The sum of a row's exponentials relative to its lse, by the row's `group` threads (at most a warp's, or a CTA), which take
// four vectors at a time.
template <class T, bool CTA>
__device__ __forceinline__ float row_sum(const T* row, int V, int shift, int lane, int group, float lse) {
    constexpr int N = VEC<T>, U = CTA ? 4 : 1;
    const Scale sc(lse);
    float2 s2 = make_float2(0.0f, 0.0f), u2 = s2;
    for (int c = lane; c * N - shift < V; c += U * group) {
        uint4 raw[U];
#pragma unroll
        for (int k = 0; k < U; k++) raw[k] = load_vec<false>(row, (c + k * group) * N - shift, V);
        if constexpr (CTA) {   // a round's sum by itself: rows may be long
            float2 e2 = make_float2(0.0f, 0.0f);
            add_exp<T>(raw, sc, e2, u2);
            s2 = __fadd2_rn(s2, e2);
        } else {
            add_exp<T>(raw, sc, s2, u2);
        }
    }
    float s = s2.x + s2.y;
    if constexpr (CTA) {
        __shared__ float part[8];
#pragma unroll
        for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(kFull, s, o);
        if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = s;
        __syncthreads();
        s = 0.0f;
        for (int w = 0; w < group / 32; w++) s += part[w];
    } else {
        const unsigned mask = group == 32 ? kFull : ((1u << group) - 1u) << ((threadIdx.x & 31) & ~(group - 1));
        for (int o = group / 2; o; o >>= 1) s += __shfl_xor_sync(mask, s, o);
    }
    return s;
}

// A thread takes M vectors of a row at a time. Rows of up to 128 vectors: 2^lg threads of a warp share a row. Longer ones
// (CTA): a CTA has one row's part, `chunks` CTAs a row, or the whole row where the gradient is written over the logits.
// Four vectors share the row's scalars and keep enough loads in flight; up to eight vectors a row take one each, so that
// short rows' stores stay whole. Bound by memory: 4001 x 16411 fp32 with entropy 90 us (5.8 TB/s, 89 % of a copy's rate), 2^18
// x 256 bf16 52 us (5.3), 2^20 x 4 fp32 7.9 us (5.4, launch included); the launch bounds hold the registers that the second
// sum (below) would take (without them 8.9, 55 and 91 us; as a function of its own 8.0, 56, 90).
//
// The lse is rounded to 32 bits, which is off by 2^-24 of its size: p would be off by that, and wholly wrong where all of a
// row is masked by a large finite value (p = 1 everywhere for a row of -1e9). So rows whose lse is 256 or more in size are
// summed up once more, relative to that lse, and p is divided by the sum. All of a row's threads that may have written
// parts of it in place wait for that sum.
template <class T, int M, bool ENTROPY, bool CTA>
__global__ void __launch_bounds__(256, M == 1 ? 8 : 5) k_logprobs_grad(const GradArgs a, int lg) {
    constexpr int N = VEC<T>;
    const int group = CTA ? (int)blockDim.x : 1 << lg;
    const long long r = CTA ? (long long)(blockIdx.x / (unsigned)a.chunks) : (long long)blockIdx.x * (256 >> lg) + (threadIdx.x >> lg);
    const int lane = CTA ? (int)threadIdx.x : threadIdx.x & (group - 1);
    if (r >= a.rows) return;
    const T* row = static_cast<const T*>(a.x) + r * a.stride;
    T* out = static_cast<T*>(a.dx) + r * a.dx_stride;
    const int shift = row_shift(row), V = a.V, nvec = (V + shift + N - 1) / N;
    const int part = CTA ? (int)(blockIdx.x % (unsigned)a.chunks) : 0;
    int parts = CTA ? a.chunks : 1;   // CTAs that share the row
    int c0 = lane + part * M * group;
    uint4 raw[M];
#pragma unroll
    for (int k = 0; k < M; k++) raw[k] = load_vec<false>(row, (c0 + k * group) * N - shift, V);
    const float lse = a.lse[r];
    const long long t = load_symbol(a.sym, a.sym_type, r * a.sym_stride);
    float dl = t < 0 ? 0.0f : a.dlogp[r * a.dlogp_stride];
    if (t >= V) dl = NAN;
    const bool empty = lse == kNegInf;
    const Scale sc(empty ? 0.0f : lse);
    float p0 = -fmaf(sc.off, kLn2, 1.0f);   // p = -p0 2^y (2^off, or 1 / sum)
    float shift_nat = sc.off * kLn2;        // log p = y ln 2 + shift_nat
    if (!empty && fabsf(lse) >= 256.0f) {
        if constexpr (CTA) {
            parts = min(parts, a.far_parts);
            if (part >= parts) return;   // the whole CTA
        }
        const float s = row_sum<T, CTA>(row, V, shift, lane, group, lse);
        p0 = __fdividef(-1.0f, s);
        shift_nat = -logf(s);
        if constexpr (CTA) {   // again, rather than kept over the sum
#pragma unroll
            for (int k = 0; k < M; k++) raw[k] = load_vec<false>(row, (c0 + k * group) * N - shift, V);
        }
    }
    float dh = 0.0f, base = dl;
    if constexpr (ENTROPY) {
        dh = a.dentropy[r * a.dentropy_stride];
        base = fmaf(dh, shift_nat + a.entropy[r], dl);
        dh *= kLn2;
    }
    // the exponents of either kind of Scale without a choice per element: (x - 0) L + b or (x - m) L + 0
    const float from = sc.far ? -sc.m : 0.0f, b = sc.far ? 0.0f : sc.b;
    const float2 from2 = make_float2(from, from), b2 = make_float2(b, b), dh2 = make_float2(dh * p0, dh * p0), base2 = make_float2(base * p0, base * p0);
    for (;;) {
#pragma unroll
        for (int k = 0; k < M; k++) {
            const int j0 = (c0 + k * group) * N - shift;
            if (j0 >= V) break;
            float v[N];
            expand<T>(raw[k], v);
#pragma unroll
            for (int i = 0; i < N; i += 2) {
                float2 y = __ffma2_rn(__fadd2_rn(make_float2(v[i], v[i + 1]), from2), make_float2(kLog2e, kLog2e), b2);
                y.x = max_nan(y.x, kYLow); y.y = max_nan(y.y, kYLow);
                const float2 p = make_float2(exp2_of(y.x), exp2_of(y.y));
                const float2 g = ENTROPY ? __fmul2_rn(p, __ffma2_rn(dh2, y, base2)) : __fmul2_rn(p, base2);
                v[i] = g.x; v[i + 1] = g.y;
            }
            if (t >= j0 && t < j0 + N) {
#pragma unroll
                for (int i = 0; i < N; i++)
                    if (j0 + i == t) v[i] += dl;
            }
            if (empty) {
#pragma unroll
                for (int i = 0; i < N; i++) v[i] = 0.0f;
            }
            uint4 w;
            if constexpr (sizeof(T) == 4) w = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
            else {
                uint32_t h[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    if constexpr (std::is_same_v<T, __half>) { const __half2 e = __floats2half2_rn(v[2 * i], v[2 * i + 1]); memcpy(&h[i], &e, 4); }
                    else { const __nv_bfloat162 e = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]); memcpy(&h[i], &e, 4); }
                }
                w = make_uint4(h[0], h[1], h[2], h[3]);
            }
            if (j0 >= 0 && j0 + N <= V && (reinterpret_cast<uintptr_t>(out + j0) & 15) == 0) {
                __stcs(reinterpret_cast<uint4*>(out + j0), w);
            } else {
                const uint32_t h[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int i = 0; i < N; i++) {
                    if (j0 + i < 0 || j0 + i >= V) continue;
                    if constexpr (sizeof(T) == 4) out[j0 + i] = v[i];
                    else { const unsigned short e = (unsigned short)(h[i / 2] >> (16 * (i % 2))); memcpy(out + j0 + i, &e, 2); }
                }
            }
        }
        if constexpr (!CTA) return;
        c0 += parts * M * group;   // a CTA with more than one part of the row goes on
        if (c0 - lane >= nvec) return;
#pragma unroll
        for (int k = 0; k < M; k++) raw[k] = load_vec<false>(row, (c0 + k * group) * N - shift, V);
    }
}

// ---------------------------------------------------------------------------------------------------------- launches

long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }

// The widest a row gets with its shift. Starts lie a multiple of g elements past a 16-byte boundary, so no shift is
// above VEC - g.
template <class T>
int row_span(const void* x, long long stride, int V) {
    const long long at = (long long)(reinterpret_cast<uintptr_t>(x) % 16 / sizeof(T)) | stride | VEC<T>;
    const int g = (int)(at & -at);
    return V + VEC<T> - g;
}

template <class T, int G, int E, int L>
void launch_lanes(const RowArgs& a, cudaStream_t s) {
    k_logprobs_lanes<T, G, E, L><<<(unsigned)ceil_div(a.rows, 256 / G), 256, 0, s>>>(a);
}
// Rows of up to GMAX * E elements on G lanes or the fewest above that hold them (a row's joins and its end are paid per
// lane); false for longer ones.
template <class T, int G, int GMAX, int E, int L>
bool launch_fit(const RowArgs& a, int span, cudaStream_t s) {
    if (span <= G * E) { launch_lanes<T, G, E, L>(a, s); return true; }
    if constexpr (G < GMAX) return launch_fit<T, 2 * G, GMAX, E, L>(a, span, s);
    return false;
}
// Rows with up to eight alternatives: 64 16-bit (32 fp32) elements a lane, half of that for rows of one or two lanes. Lanes
// with more elements pay a row's joins and its end less often: 2^18 x 256 bf16 with eight took 72 us with 64 a lane, 81 with
// 32; 2^18 x 64 took 29 and 24.
template <class T, int L>
bool launch_sorted(const RowArgs& a, int span, cudaStream_t s) {
    if constexpr (sizeof(T) == 2) return span <= 64 ? launch_fit<T, 1, 2, 32, L>(a, span, s) : launch_fit<T, 2, 16, 64, L>(a, span, s);
    else return span <= 32 ? launch_fit<T, 2, 2, 16, L>(a, span, s) : launch_fit<T, 2, 8, 32, L>(a, span, s);
}
template <class T, class K, int W, int R>
cudaError_t launch_long(const RowArgs& a, int C, cudaStream_t s) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(ceil_div(a.rows, R) * C));
    cfg.blockDim = dim3(32 * W * R);
    cfg.stream = s;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = (unsigned)C; at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = C > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, k_logprobs_long<T, K, W, R>, a, C);
}

template <class T, class K>
cudaError_t launch_long(const RowArgs& a, int span, cudaStream_t s, int sms) {
    // Warps to a row: one for 1536 vectors (a warp's joins are paid once, and rows that have ended make place for others),
    // more where that would leave an SM fewer than 10, and no more than leave a thread two vectors. Measured, bf16, warps
    // 1 / 2 / 4 / 8: 12000 x 4099 29 / 38 / 41 / 66 us, 6000 x 16384 44 / 40 / 41 / 48, 2048 x 65536 74 / 54 / 55 / 52,
    // 300 x 16384 12 / 7.9 / 6.1 / 6.1. Almost as many alternatives as a warp has lanes want more maxima than one warp gives
    // (12000 x 4099: 61 us with 30; with 32 one warp 113, two 68), except where a lane holds few logits anyway (2^25 in rows
    // of 1024: 88 with one warp, 116 with two).
    const int vectors = (span + VEC<T> - 1) / VEC<T>;
    int W = a.topk > 30 && span > 1024 ? 2 : 1, C = 1;
    while (W < 8 && (vectors > 1536 * W || a.rows * W < 10ll * sms) && vectors >= 64 * W * 2) W *= 2;
    // CTAs to a row: where rows are few, parts of 8192 logits or more on up to eight CTAs. 16 x 65536 took 5.2 us with eight,
    // but 148 x 8192 8.6 us with four against 4.0 with one: clusters start slowly.
    if (W == 8)
        while (C < 8 && a.V / (C * 2) >= 8192 && a.rows * C * 2 <= 4 * sms) C *= 2;
    if constexpr (sizeof(K) == 4 || sizeof(T) == 4) {   // 16-bit rows that need 64-bit keys have over 8192 vectors: W = 8
        if (W == 1) return launch_long<T, K, 1, 4>(a, 1, s);
        if (W == 2) return launch_long<T, K, 2, 1>(a, 1, s);
        if (W == 4) return launch_long<T, K, 4, 1>(a, 1, s);
    }
    return launch_long<T, K, 8, 1>(a, C, s);
}

template <class T>
cudaError_t launch_rows(const RowArgs& a, cudaStream_t s, int sms) {
    constexpr int N = VEC<T>;
    const int span = row_span<T>(a.x, a.stride, a.V);
    // Rows in registers as far as that is the faster way: without alternatives or with one up to 1024 elements; 16-bit logits
    // with up to eight also (1024 bf16: 38 us for 2^25 logits), with more up to 512 (512 with nine: 71 us, as long rows 90);
    // fp32 logits, whose keys take 64 bits, up to 256 (257 with nine: 304 us, as long rows 162).
    bool done;
    if (a.topk == 0) {
        if (span <= N) done = launch_fit<T, 1, 1, N, 0>(a, span, s);
        else if (span <= 16) done = launch_fit<T, 1, 1, 16, 0>(a, span, s);
        else if (span <= 64) done = launch_fit<T, 4, 4, 16, 0>(a, span, s);
        else done = launch_fit<T, 4, 32, 32, 0>(a, span, s);
    } else if (a.topk == 1) {
        if (span <= N) done = launch_fit<T, 1, 1, N, 1>(a, span, s);
        else done = launch_fit<T, 1, 32, 32, 1>(a, span, s);
    } else if (a.topk <= 8) {
        if (span <= N) done = launch_fit<T, 1, 1, N, N>(a, span, s);
        else if (N < 8 && span <= 8) done = launch_fit<T, 1, 1, 8, 8>(a, span, s);
        else if (span <= 16) done = launch_fit<T, 1, 1, 16, 8>(a, span, s);
        else done = a.topk <= 4 ? launch_sorted<T, 4>(a, span, s) : launch_sorted<T, 8>(a, span, s);
    } else {
        done = launch_fit<T, 1, sizeof(T) == 2 ? 32 : 16, 16, 16>(a, span, s);
    }
    if (!done) {
        typedef typename std::conditional<sizeof(T) == 2, uint32_t, unsigned long long>::type K;
        if (sizeof(T) == 2 && a.V > 65536) return launch_long<T, unsigned long long>(a, span, s, sms);
        return launch_long<T, K>(a, span, s, sms);
    }
    return cudaGetLastError();
}

template <class T, bool ENTROPY>
cudaError_t launch_grad(GradArgs a, cudaStream_t s, int sms) {
    const int nvec = (int)ceil_div(row_span<T>(a.x, a.stride, a.V), VEC<T>);
    int lg = 0;
    a.chunks = 1;
    if (nvec <= 8) {
        while ((1 << lg) < nvec) lg++;
        k_logprobs_grad<T, 1, ENTROPY, false><<<(unsigned)ceil_div(a.rows, 256 >> lg), 256, 0, s>>>(a, lg);
    } else if (nvec <= 128) {
        lg = 1;
        while ((4 << lg) < nvec) lg++;
        k_logprobs_grad<T, 4, ENTROPY, false><<<(unsigned)ceil_div(a.rows, 256 >> lg), 256, 0, s>>>(a, lg);
    } else {
        const int threads = nvec <= 256 ? 64 : nvec <= 512 ? 128 : 256;
        if (a.dx != a.x) a.chunks = (int)ceil_div(nvec, 4 * threads);
        a.far_parts = (int)std::min<long long>(8, std::max<long long>(1, 4 * sms / a.rows));   // few rows: more of each at once
        k_logprobs_grad<T, 4, ENTROPY, true><<<(unsigned)(a.rows * a.chunks), threads, 0, s>>>(a, 0);
    }
    return cudaGetLastError();
}
template <class T>
cudaError_t launch_grad(const GradArgs& a, cudaStream_t s, int sms) {
    return a.dentropy ? launch_grad<T, true>(a, s, sms) : launch_grad<T, false>(a, s, sms);
}

}  // namespace
}  // namespace ntcb
