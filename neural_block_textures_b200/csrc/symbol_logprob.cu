// Log probabilities of given symbols under a predictor's logits, with entropy and top alternatives, and the gradient:
// ntcb_symbol_logprobs / ntcb_symbol_logprobs_grad (include/ntc_b200.h).
//
// Forward, for a row x[0..V) and its symbol t:
//   m = max x, d = x - m, s = sum e^d, u = sum e^d d
//   lse = m + log s, logp = (x_t - m) - log s, H = log s - u / s
// and the topk largest logits in order (value first, then the lower index). One read of the logits does all of it: m,
// s and u are kept online (a larger maximum rescales s and u), in 32 bits whatever the logits' type.
// Rows: no finite logit (everything masked) gives lse = logp = -inf, H = 0 and no alternatives; a NaN or +inf gives NaN.
// Masked logits take no part: e^d is 0 for -inf and for the type's lowest value, and d is clamped at kDLow so that
// e^d d is 0 there too, not 0 * inf; the clamp passes NaN on.
//
// Gradient: p_j = e^(x_j - lse); dx_j = [j = t] dlogp - p_j (dlogp + dH (x_j - lse + H)).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdio>
#include <cstring>

#include "../../include/ntc_b200.h"
#include "device_scope.h"

namespace ntcb {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kDLow = -150.0f;        // e^-150 is 0 in 32 bits
constexpr int kMaxTop = NTCB_MAX_TOPK;  // 32: one alternative per lane
constexpr unsigned kFull = 0xffffffffu;
constexpr float kNegInf = -INFINITY;

struct RowArgs {
    const void* x;
    const void* sym;
    long long rows, stride, sym_stride;
    int V, topk, sym_type;
    float *logp, *entropy, *lse, *top_logp;
    int* top_ids;
};

struct GradArgs {
    const void* x;
    const void* sym;
    const float *lse, *entropy, *dlogp, *dentropy;
    void* dx;
    long long rows, stride, sym_stride, dx_stride, dlogp_stride, dentropy_stride;
    int V, sym_type, chunks;
};

// ---------------------------------------------------------------------------------------------- elements and keys

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_f32(float v, float& o) { o = v; }
__device__ __forceinline__ void from_f32(float v, __half& o) { o = __float2half_rn(v); }
__device__ __forceinline__ void from_f32(float v, __nv_bfloat16& o) { o = __float2bfloat16_rn(v); }

__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float exp_of(float d) {   // e^d for d in [kDLow, 0]
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d * kLog2e));
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

// A logit and its index as one word: larger value first, then the lower index. 0 is no logit.
typedef unsigned long long Key;
__device__ __forceinline__ Key key_of(float x, int idx) {
    const uint32_t b = __float_as_uint(x + 0.0f);   // -0 and +0 are one value
    const uint32_t o = b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
    return ((Key)o << 32) | (uint32_t)(~(uint32_t)idx);
}
__device__ __forceinline__ float key_value(Key k) {
    const uint32_t o = (uint32_t)(k >> 32);
    return __uint_as_float(o ^ ((o >> 31) ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ int key_index(Key k) { return (int)(~(uint32_t)k); }

// Vectors of VEC elements: 16 bytes of a 16-bit type, 32 bytes of fp32 (two loads).
constexpr int VEC = 8;
template <class T> struct Align { static constexpr int elems = 16 / sizeof(T); };

// Loads of the forward pass go through the read-only path; the gradient may be written over its logits, so its loads
// are ordinary ones (streamed: nothing is read twice).
template <bool READ_ONLY, class W>
__device__ __forceinline__ W load(const W* p) {
    if constexpr (READ_ONLY) return __ldg(p);
    else return __ldcs(p);
}

// Elements [j0, j0 + VEC) of a row, -inf outside [0, V). The address of j0 is 16-byte aligned by the caller's choice of
// the shift, so a vector inside the row is loaded wide; the first and the last one element by element.
template <bool READ_ONLY = true, class T>
__device__ __forceinline__ void load_vec(const T* row, int j0, int V, float (&v)[VEC]) {
    if (j0 >= 0 && j0 + VEC <= V) {
        if constexpr (sizeof(T) == 4) {
            const float4* w = reinterpret_cast<const float4*>(row + j0);
            const float4 a = load<READ_ONLY>(w), b = load<READ_ONLY>(w + 1);
            v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        } else {
            const uint4 a = load<READ_ONLY>(reinterpret_cast<const uint4*>(row + j0));
            T e[VEC];
            memcpy(e, &a, 16);
#pragma unroll
            for (int i = 0; i < VEC; i++) v[i] = to_f32(e[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < VEC; i++) v[i] = (j0 + i >= 0 && j0 + i < V) ? to_f32(load<READ_ONLY>(row + j0 + i)) : kNegInf;
    }
}

// How many elements before the row the first 16-byte boundary at or below its start lies.
template <class T>
__device__ __forceinline__ int row_shift(const T* row) { return (int)((reinterpret_cast<uintptr_t>(row) / sizeof(T)) % Align<T>::elems); }

struct Sums { float m, s, u; };

// Joins two partial rows: s and u are relative to m. u = sum e^(x - m) (x - m).
__device__ __forceinline__ Sums join(const Sums& a, const Sums& b) {
    const float m = fmaxf(a.m, b.m);
    const float da = max_nan(a.m - m, kDLow), db = max_nan(b.m - m, kDLow);
    const float ea = exp_of(da), eb = exp_of(db);
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
    o.entropy = o.empty ? 0.0f : o.log_s - q.u / q.s;
    return o;
}
// The row's scalars, by one thread.
template <class T>
__device__ __forceinline__ void write_row(const RowArgs& a, long long r, const T* row, const RowOut& o) {
    const long long t = load_symbol(a.sym, a.sym_type, r * a.sym_stride);
    float lp;
    if (t < 0) lp = 0.0f;
    else if (t >= a.V || o.bad) lp = NAN;
    else if (o.empty) lp = kNegInf;
    else lp = (to_f32(row[t]) - o.m) - o.log_s;
    a.logp[r] = lp;
    a.entropy[r] = o.bad ? NAN : o.entropy;
    a.lse[r] = o.bad ? NAN : o.lse;
}
__device__ __forceinline__ void write_top(const RowArgs& a, long long r, int i, Key k, const RowOut& o) {
    const float v = k ? key_value(k) : kNegInf;
    const bool none = o.bad || v == kNegInf;
    a.top_ids[r * a.topk + i] = none ? -1 : key_index(k);
    a.top_logp[r * a.topk + i] = o.bad ? NAN : none ? kNegInf : (v - o.m) - o.log_s;
}

// ------------------------------------------------------------------------------------------- rows in a few registers

// G lanes hold one row of up to G * E - 7 logits (a row may start in the middle of a 16-byte word) in registers: the
// maximum is known before the exponentials, so nothing is rescaled. Alternatives are taken one at a time, each the
// largest key over the lanes' best ones.
template <class T, int G, int E>
__global__ void __launch_bounds__(256) k_logprobs_lanes(const RowArgs a) {
    static_assert(E % VEC == 0, "whole vectors");
    const long long r = (long long)blockIdx.x * (256 / G) + threadIdx.x / G;
    const int lane = threadIdx.x % G;
    const bool live = r < a.rows;
    const T* row = static_cast<const T*>(a.x) + (live ? r : 0) * a.stride;
    const int shift = row_shift(row), V = live ? a.V : 0;
    float x[E];
    float m = -3.402823466e38f;   // a row of nothing but -inf keeps a finite maximum: d = -inf, e^d = 0
#pragma unroll
    for (int c = 0; c < E / VEC; c++) {
        float v[VEC];
        load_vec(row, (c * G + lane) * VEC - shift, V, v);
#pragma unroll
        for (int i = 0; i < VEC; i++) { x[c * VEC + i] = v[i]; m = fmaxf(m, v[i]); }
    }
#pragma unroll
    for (int o = G / 2; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(kFull, m, o));
    Sums q{m, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < E; i++) {
        const float d = max_nan(x[i] - m, kDLow);
        const float e = exp_of(d);
        q.s += e;
        q.u = fmaf(e, d, q.u);
    }
#pragma unroll
    for (int o = G / 2; o; o >>= 1) { q.s += __shfl_xor_sync(kFull, q.s, o); q.u += __shfl_xor_sync(kFull, q.u, o); }
    const RowOut o = finish_row(q);
    if (live && lane == 0) write_row(a, r, row, o);
    if (a.topk == 0) return;
    uint32_t taken = 0;
    Key best = 0;
#pragma unroll
    for (int i = 0; i < E; i++) {
        const Key k = key_of(x[i], (i / VEC * G + lane) * VEC + i % VEC - shift);
        if (x[i] > kNegInf) best = max(best, k);
    }
    for (int j = 0; j < a.topk; j++) {
        Key g = best;
#pragma unroll
        for (int w = G / 2; w; w >>= 1) g = max(g, __shfl_xor_sync(kFull, g, w));
        if (live && lane == 0) write_top(a, r, j, g, o);
        if (g && g == best) {
            best = 0;
#pragma unroll
            for (int i = 0; i < E; i++) {
                const Key k = key_of(x[i], (i / VEC * G + lane) * VEC + i % VEC - shift);
                if (k == g) taken |= 1u << i;
                if (x[i] > kNegInf && !((taken >> i) & 1u)) best = max(best, k);
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------------- long rows

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kCand = 512;   // candidate alternatives held in shared memory

__device__ __forceinline__ Key shfl_key(Key k, int src_xor) { return __shfl_xor_sync(kFull, k, src_xor); }

// Sorts one key per lane, largest first (bitonic).
__device__ __forceinline__ Key sort32(Key k, int lane) {
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
        for (int step = size >> 1; step; step >>= 1) {
            const Key other = shfl_key(k, step);
            const bool keep_max = ((lane & step) == 0) == ((lane & size) == 0);
            k = (keep_max == (k > other)) ? k : other;
        }
    return k;
}
// The 32 largest of two sorted lists, sorted: the larger of a[i] and b[31 - i] is a bitonic sequence of them.
__device__ __forceinline__ Key merge32(Key a, Key b, int lane) {
    const Key rb = __shfl_sync(kFull, b, 31 - lane);
    Key k = max(a, rb);
#pragma unroll
    for (int step = 16; step; step >>= 1) {
        const Key other = shfl_key(k, step);
        k = (((lane & step) == 0) == (k > other)) ? k : other;
    }
    return k;
}

struct LongShared {
    Sums part[kWarps];
    Sums total;                 // this CTA's part of the row
    Key list[kWarps][32];
    Key top[32];                // this CTA's alternatives
    Key cand[kCand];
    int count;
};

__device__ __forceinline__ unsigned cluster_rank() { unsigned r; asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.aligned;\nbarrier.cluster.wait.aligned;" ::: "memory");
}
template <class W>
__device__ __forceinline__ W peer_load(const W* p, unsigned rank) {   // a word of another CTA's shared memory
    const uint32_t local = (uint32_t)__cvta_generic_to_shared(p);
    uint32_t remote;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(rank));
    W v;
    if constexpr (sizeof(W) == 8) asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(remote));
    else asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(remote));
    return v;
}

// One row per cluster of C CTAs. Vector c of the row belongs to CTA c / per, and there to thread (c - first) % kThreads.
// Alternatives: each thread keeps its largest logit and the vector that holds it. The topk largest of the threads'
// maxima are at least as large as the row's topk-th logit, and every logit that large lies with one of those topk
// threads; so only their vectors are read again (from L2), by all threads together, and the few logits that pass are
// sorted. Work that is far above that (a row of equal logits) is taken by one warp from a running list of 32.
template <class T>
__global__ void __launch_bounds__(kThreads) k_logprobs_long(const RowArgs a, int C) {
    __shared__ LongShared sh;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const unsigned rank = C > 1 ? cluster_rank() : 0;
    const long long r = blockIdx.x / (unsigned)C;
    const T* row = static_cast<const T*>(a.x) + r * a.stride;
    const int shift = row_shift(row), V = a.V;
    const int nvec = (V + shift + VEC - 1) / VEC;
    const int per = (nvec + C - 1) / C, first = min(nvec, (int)rank * per), end = min(nvec, first + per);
    Sums q{-3.402823466e38f, 0.0f, 0.0f};
    float mine = kNegInf;   // this thread's largest logit, and its vector (the first one that holds it)
    int at = -1;
    for (int c = first + tid; c < end; c += kThreads) {
        float v[VEC];
        load_vec(row, c * VEC - shift, V, v);
        float cm = v[0];
#pragma unroll
        for (int i = 1; i < VEC; i++) cm = fmaxf(cm, v[i]);
        if (cm > mine) { mine = cm; at = c; }
        if (cm > q.m) {
            const float d = max_nan(q.m - cm, kDLow), e = exp_of(d);
            q.u = (q.u + q.s * d) * e;
            q.s *= e;
            q.m = cm;
        }
#pragma unroll
        for (int i = 0; i < VEC; i++) {
            const float d = max_nan(v[i] - q.m, kDLow);
            const float e = exp_of(d);
            q.s += e;
            q.u = fmaf(e, d, q.u);
        }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        Sums p{__shfl_xor_sync(kFull, q.m, o), __shfl_xor_sync(kFull, q.s, o), __shfl_xor_sync(kFull, q.u, o)};
        q = join(q, p);
    }
    if (lane == 0) sh.part[warp] = q;
    if (tid == 0) sh.count = 0;
    if (a.topk) {
        Key k = 0;
        if (at >= 0) {
            float v[VEC];
            load_vec(row, at * VEC - shift, V, v);
#pragma unroll
            for (int i = VEC - 1; i >= 0; i--)
                if (v[i] == mine) k = key_of(v[i], at * VEC + i - shift);
        }
        sh.list[warp][lane] = sort32(k, lane);
    }
    __syncthreads();
    if (a.topk) {
        for (int half = kWarps / 2; half; half >>= 1) {
            if (warp < half) {
                const Key k = merge32(sh.list[warp][lane], sh.list[warp + half][lane], lane);
                __syncwarp();
                sh.list[warp][lane] = k;
            }
            __syncthreads();
        }
        const Key least = sh.list[0][a.topk - 1];   // 0 when fewer threads than topk hold a logit
        const int per_thread = (end - first + kThreads - 1) / kThreads;
        for (int item = tid; item < a.topk * per_thread; item += kThreads) {
            const Key owner = sh.list[0][item / per_thread];
            if (!owner) continue;
            const int c = first + ((key_index(owner) + shift) / VEC - first) % kThreads + (item % per_thread) * kThreads;
            if (c >= end) continue;
            float v[VEC];
            load_vec(row, c * VEC - shift, V, v);
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                const Key k = key_of(v[i], c * VEC + i - shift);
                if (v[i] > kNegInf && k >= least) {
                    const int p = atomicAdd(&sh.count, 1);
                    if (p < kCand) sh.cand[p] = k;
                }
            }
        }
        __syncthreads();
        if (warp == 0) {
            Key top = 0;
            if (sh.count <= kCand) {
                for (int i = 0; i < sh.count; i += 32) {
                    const Key k = sort32(i + lane < sh.count ? sh.cand[i + lane] : 0, lane);
                    top = merge32(top, k, lane);
                }
            } else {
                const int items = a.topk * per_thread;
                for (int i0 = 0; i0 < items; i0 += 32) {
                    const int item = i0 + lane;
                    const Key owner = item < items ? sh.list[0][item / per_thread] : 0;
                    const int c = owner ? first + ((key_index(owner) + shift) / VEC - first) % kThreads + (item % per_thread) * kThreads : end;
                    float v[VEC];
                    load_vec(row, c < end ? c * VEC - shift : V, V, v);
#pragma unroll
                    for (int i = 0; i < VEC; i++) {
                        Key k = v[i] > kNegInf ? key_of(v[i], c * VEC + i - shift) : 0;
                        const Key last = __shfl_sync(kFull, top, 31);
                        if (k < least || k < last) k = 0;
                        if (__any_sync(kFull, k != 0)) top = merge32(top, sort32(k, lane), lane);
                    }
                }
            }
            sh.top[lane] = top;
        }
    }
    if (warp == 0) {
        Sums p = lane < kWarps ? sh.part[lane] : Sums{-3.402823466e38f, 0.0f, 0.0f};
#pragma unroll
        for (int o = kWarps / 2; o; o >>= 1) {
            Sums b{__shfl_xor_sync(kFull, p.m, o), __shfl_xor_sync(kFull, p.s, o), __shfl_xor_sync(kFull, p.u, o)};
            p = join(p, b);
        }
        q = p;
        if (lane == 0) sh.total = p;
    }
    if (C > 1) {
        __syncthreads();
        cluster_sync();
        if (rank == 0 && warp == 0) {
            Key top = a.topk ? sh.top[lane] : 0;
            for (int w = 1; w < C; w++) {
                Sums b{peer_load(&sh.total.m, w), peer_load(&sh.total.s, w), peer_load(&sh.total.u, w)};
                q = join(q, b);
                if (a.topk) top = merge32(top, peer_load(&sh.top[lane], w), lane);
            }
            sh.top[lane] = top;
        }
        cluster_sync();   // no CTA leaves while its shared memory is read
    }
    if (rank == 0 && warp == 0) {
        q.m = __shfl_sync(kFull, q.m, 0); q.s = __shfl_sync(kFull, q.s, 0); q.u = __shfl_sync(kFull, q.u, 0);
        const RowOut o = finish_row(q);
        if (lane == 0) write_row(a, r, row, o);
        __syncwarp();
        if (lane < a.topk) write_top(a, r, lane, sh.top[lane], o);
    }
}

// -------------------------------------------------------------------------------------------------------- gradient

// One thread per vector of a row (CTAs of 256 over rows * chunks): G lanes share a row when it is short, else a row
// takes `chunks` CTAs of kThreads vectors.
template <class T, int G>
__global__ void __launch_bounds__(256) k_logprobs_grad(const GradArgs a) {
    long long r;
    int c;
    if constexpr (G > 0) {
        r = (long long)blockIdx.x * (256 / G) + threadIdx.x / G;
        c = threadIdx.x % G;
    } else {
        r = blockIdx.x / (unsigned)a.chunks;
        c = (int)(blockIdx.x % (unsigned)a.chunks) * 256 + threadIdx.x;
    }
    if (r >= a.rows) return;
    const T* row = static_cast<const T*>(a.x) + r * a.stride;
    T* out = static_cast<T*>(a.dx) + r * a.dx_stride;
    const int shift = row_shift(row), j0 = c * VEC - shift, V = a.V;
    if (j0 >= V) return;
    const float lse = a.lse[r];
    const long long t = load_symbol(a.sym, a.sym_type, r * a.sym_stride);
    float dl = t < 0 ? 0.0f : a.dlogp[r * a.dlogp_stride];
    if (t >= V) dl = NAN;
    const float dh = a.dentropy ? a.dentropy[r * a.dentropy_stride] : 0.0f;
    const float h = a.dentropy ? a.entropy[r] : 0.0f;
    float v[VEC];
    load_vec<false>(row, j0, V, v);
    const bool empty = lse == kNegInf;
#pragma unroll
    for (int i = 0; i < VEC; i++) {
        const float d = max_nan(v[i] - lse, kDLow);
        const float p = exp_of(d);
        float g = -p * fmaf(dh, d + h, dl);
        if (j0 + i == t) g += dl;
        v[i] = empty ? 0.0f : g;
    }
    if (j0 >= 0 && j0 + VEC <= V && (reinterpret_cast<uintptr_t>(out + j0) & 15) == 0) {
        alignas(16) T e[VEC];
#pragma unroll
        for (int i = 0; i < VEC; i++) from_f32(v[i], e[i]);
        uint4 w[sizeof(e) / 16];
        memcpy(w, e, sizeof(e));
#pragma unroll
        for (int i = 0; i < (int)(sizeof(e) / 16); i++) reinterpret_cast<uint4*>(out + j0)[i] = w[i];
    } else {
#pragma unroll
        for (int i = 0; i < VEC; i++)
            if (j0 + i >= 0 && j0 + i < V) from_f32(v[i], out[j0 + i]);
    }
}

// ---------------------------------------------------------------------------------------------------------- launches

int ceil_div(long long a, long long b) { return (int)((a + b - 1) / b); }

template <class T, int G, int E>
void launch_lanes(const RowArgs& a, cudaStream_t s) {
    k_logprobs_lanes<T, G, E><<<(unsigned)ceil_div(a.rows, 256 / G), 256, 0, s>>>(a);
}

template <class T>
cudaError_t launch_rows(const RowArgs& a, cudaStream_t s, int sms) {
    const int span = a.V + Align<T>::elems - 1;   // a row with its part of a 16-byte word before it
    if (span <= 8) launch_lanes<T, 1, 8>(a, s);
    else if (span <= 16) launch_lanes<T, 2, 8>(a, s);
    else if (span <= 32) launch_lanes<T, 4, 8>(a, s);
    else if (span <= 64) launch_lanes<T, 8, 8>(a, s);
    else if (span <= 128) launch_lanes<T, 16, 8>(a, s);
    else if (span <= 256) launch_lanes<T, 32, 8>(a, s);
    else if (span <= 512) launch_lanes<T, 32, 16>(a, s);
    else if (span <= 1024) launch_lanes<T, 32, 32>(a, s);
    else {
        int C = 1;
        while (C < 8 && a.rows * C * 2 <= 4 * sms && a.V / (C * 2) >= 2048) C *= 2;
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3((unsigned)(a.rows * C));
        cfg.blockDim = dim3(kThreads);
        cfg.stream = s;
        cudaLaunchAttribute at{};
        at.id = cudaLaunchAttributeClusterDimension;
        at.val.clusterDim.x = (unsigned)C; at.val.clusterDim.y = at.val.clusterDim.z = 1;
        cfg.attrs = &at;
        cfg.numAttrs = C > 1 ? 1 : 0;
        return cudaLaunchKernelEx(&cfg, k_logprobs_long<T>, a, C);
    }
    return cudaGetLastError();
}

template <class T>
cudaError_t launch_grad(GradArgs a, cudaStream_t s) {
    const int nvec = ceil_div((long long)a.V + Align<T>::elems - 1, VEC);
    if (nvec <= 1) k_logprobs_grad<T, 1><<<(unsigned)ceil_div(a.rows, 256), 256, 0, s>>>(a);
    else if (nvec <= 4) k_logprobs_grad<T, 4><<<(unsigned)ceil_div(a.rows, 64), 256, 0, s>>>(a);
    else if (nvec <= 16) k_logprobs_grad<T, 16><<<(unsigned)ceil_div(a.rows, 16), 256, 0, s>>>(a);
    else if (nvec <= 64) k_logprobs_grad<T, 64><<<(unsigned)ceil_div(a.rows, 4), 256, 0, s>>>(a);
    else {
        a.chunks = ceil_div(nvec, 256);
        k_logprobs_grad<T, 0><<<(unsigned)(a.rows * a.chunks), 256, 0, s>>>(a);
    }
    return cudaGetLastError();
}

// ------------------------------------------------------------------------------------------------------ the checks

const char* check_desc(const ntcb_symbol_desc* d) {
    if (!d) return "null description";
    if (d->dtype < NTCB_F32 || d->dtype > NTCB_BF16) return "unknown type of the logits";
    if (d->symbol_type < NTCB_SYM_U8 || d->symbol_type > NTCB_SYM_I64) return "unknown type of the symbols";
    if (d->rows < 0) return "negative row count";
    if (d->vocab < 1 || d->vocab > (1ll << 28)) return "vocab outside 1 .. 2^28";
    if (d->row_stride < 0 || (d->row_stride > 0 && d->row_stride < d->vocab)) return "row_stride between 0 and vocab: rows overlap";
    if (d->symbol_stride < 0) return "negative symbol_stride";
    // the largest grids: one CTA per row and up to vocab / 2048 CTAs per row (gradient), below 2^31 CTAs in all
    if (d->rows > 0x7fffffffll / 8 || d->rows * ((d->vocab + 2047) / 2048 + 1) > 0x7fffffffll) return "more than 2^31 blocks of 2048 logits";
    return nullptr;
}
bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
size_t dtype_size(int t) { return t == NTCB_F32 ? 4 : 2; }
size_t symbol_size(int t) { return t == NTCB_SYM_U8 ? 1 : t == NTCB_SYM_I16 ? 2 : t == NTCB_SYM_I32 ? 4 : 8; }

}  // namespace
}  // namespace ntcb

extern "C" int ntcb_symbol_logprobs(const ntcb_symbol_desc* d, const void* logits, const void* symbols, int topk, float* logp,
                                    float* entropy, float* lse, int* top_ids, float* top_logp, void* stream, char* why, size_t why_cap) {
    using namespace ntcb;
    const auto refuse = [&](const char* m) { set_why(why, why_cap, m); return 0; };
    if (const char* m = check_desc(d)) return refuse(m);
    if (topk < 0 || topk > kMaxTop) return refuse("topk outside 0 .. 32");
    if (topk > d->vocab) return refuse("topk above vocab");
    if (d->rows == 0) return 1;
    if (!logits || !symbols || !logp || !entropy || !lse || (topk && (!top_ids || !top_logp))) return refuse("null buffer");
    if (!aligned(logits, dtype_size(d->dtype)) || !aligned(symbols, symbol_size(d->symbol_type))) return refuse("a buffer is not aligned to its type");
    DeviceScope scope(d->device, why, why_cap);
    if (!scope.ok) return 0;
    const RowArgs a{logits, symbols, d->rows, d->row_stride, d->symbol_stride, (int)d->vocab, topk, d->symbol_type,
                    logp, entropy, lse, top_logp, top_ids};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const cudaError_t e = d->dtype == NTCB_F32 ? launch_rows<float>(a, s, scope.sms)
                          : d->dtype == NTCB_F16 ? launch_rows<__half>(a, s, scope.sms)
                                                 : launch_rows<__nv_bfloat16>(a, s, scope.sms);
    return scope.launched(e, why, why_cap);
}

extern "C" int ntcb_symbol_logprobs_grad(const ntcb_symbol_desc* d, const void* logits, const void* symbols, const float* lse,
                                         const float* entropy, const float* dlogp, long long dlogp_stride, const float* dentropy,
                                         long long dentropy_stride, void* dlogits, long long dlogits_stride, void* stream, char* why,
                                         size_t why_cap) {
    using namespace ntcb;
    const auto refuse = [&](const char* m) { set_why(why, why_cap, m); return 0; };
    if (const char* m = check_desc(d)) return refuse(m);
    if (dlogp_stride < 0 || dentropy_stride < 0) return refuse("negative stride of an incoming gradient");
    if (dlogits_stride < d->vocab) return refuse("dlogits_stride below vocab: rows overlap");
    if (d->rows == 0) return 1;
    if (!logits || !symbols || !lse || !dlogp || !dlogits || (dentropy && !entropy)) return refuse("null buffer");
    const size_t sz = dtype_size(d->dtype);
    if (!aligned(logits, sz) || !aligned(dlogits, sz) || !aligned(symbols, symbol_size(d->symbol_type))) return refuse("a buffer is not aligned to its type");
    DeviceScope scope(d->device, why, why_cap);
    if (!scope.ok) return 0;
    const GradArgs a{logits, symbols, lse, entropy, dlogp, dentropy, dlogits, d->rows, d->row_stride, d->symbol_stride, dlogits_stride,
                     dlogp_stride, dentropy_stride, (int)d->vocab, d->symbol_type, 0};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const cudaError_t e = d->dtype == NTCB_F32 ? launch_grad<float>(a, s)
                          : d->dtype == NTCB_F16 ? launch_grad<__half>(a, s)
                                                 : launch_grad<__nv_bfloat16>(a, s);
    return scope.launched(e, why, why_cap);
}
