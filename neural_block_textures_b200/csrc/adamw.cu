// AdamW over many tensors in one launch, with the moments in 32 bits or in 8 (ntcb_adamw_*, include/ntc_b200.h).
//
//   g' = s g, m = b1 m + (1 - b1) g', v = b2 v + (1 - b2) g'^2, p = (1 - lr wd) p - (lr / c1) m / (sqrt(v) / sqrt(c2) + eps)
//
// Nothing is reduced over a tensor, so the step is bound by memory: 28 bytes per fp32 element with 32-bit moments (151 M
// elements in 512 tensors: 610 us, 6.9 TB/s, above the rate of a plain copy), 16 with 8-bit ones (430 to 455 us, 5.3 to 5.6
// TB/s: some 75 instructions an element keep the SMs issuing 70 % of the time; the 48 registers that five CTAs an SM leave
// cost 84 bytes of spills). With 16-bit tensors an 8-bit step moves 10 bytes an element but takes longer (13 M bf16 elements
// 49 us, fp32 45; 151 M 624 and 484, all with the step number on the device): as many instructions, issued 55 % of the time
// behind loads. Reading the moments as floats takes 230 us (6.6 TB/s). Work is cut into chunks of one tensor; a CTA takes one
// chunk, found in a table that the plan keeps on the device, and the tensors' addresses come with the launch (by value: they
// may change from step to step).
//
// 8-bit moments. Blocks of 256 elements, one warp each. A value is held as its float's exponent and upper 3 mantissa
// bits, q = bits >> 20, counted from the base of the block's window, which ends at the block's largest q. The grid of q
// does not move with the block, so a value that stays is never rounded again. Rounding to nearest would freeze v (a step
// changes it by at most 0.1 % down, a grid step is 6 to 12 %), so it is stochastic: 16 random bits are added above the
// 4 lowest of the 20 bits that are dropped (a bias below 2^-16 of a grid step), which keeps the expected value.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cfloat>
#include <cmath>
#include <new>
#include <type_traits>
#include <vector>

#include "../../include/ntc_b200.h"
#include "device_scope.h"
#include "noise.cuh"

namespace ntcb {
namespace {

constexpr int kBlock = 256;            // elements that share a window (and start a tensor's moments)
constexpr int kChunk = 2048;           // elements of one CTA: 8 blocks, one per warp
constexpr int kVec = 8;                // elements of one lane (two quads)
constexpr uint32_t kTopM = 126, kTopV = 254;
constexpr uint32_t kStreamAdamW = 5;   // beside the trainer's noise streams (noise.cuh)
constexpr unsigned kFull = 0xffffffffu;

struct Chunk {
    long long start;      // first element within the tensor
    long long state;      // first element within the moments
    int tensor, n;        // n <= kChunk
    int param_type, grad_type;
};

struct Scalars {
    double lr, beta1, beta2, wd, log_beta1, log_beta2;   // the device-scalar path recomputes step / inv / decay from these
    float b1, omb1, b2, omb2, eps, step, inv, decay, scale, one;
    uint64_t seed;
    uint32_t it;
    const long long* it_dev;
    const float* lr_dev;
    const float* scale_dev;
};

template <int N>
struct StepArgs {
    Scalars c;
    const Chunk* chunks;
    void* state;
    long long total;
    int first;            // tensor of p[0] / g[0]
    void* p[N];
    const void* g[N];
};

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_f32(float v, float& o) { o = v; }
__device__ __forceinline__ void from_f32(float v, __half& o) { o = __float2half_rn(v); }
__device__ __forceinline__ void from_f32(float v, __nv_bfloat16& o) { o = __float2bfloat16_rn(v); }

// A lane holds two quads of its warp's block: elements lane * 4 .. + 3 and 128 + lane * 4 .. + 3, so that a warp's loads and
// stores are whole lines whatever the type. `left` is how many elements of the block exist; a quad is moved in one
// piece where all of it does and its address allows.
template <class T>
__device__ __forceinline__ void load8(const T* p, int left, float (&v)[kVec]) {
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const T* q = p + 128 * h;
        const int n = left - 128 * h;
        if (n >= 4 && (reinterpret_cast<uintptr_t>(q) & (4 * sizeof(T) - 1)) == 0) {
            typedef typename std::conditional<sizeof(T) == 4, uint4, uint2>::type W;
            const W w = __ldcs(reinterpret_cast<const W*>(q));
            alignas(16) T e[4];
            memcpy(e, &w, sizeof(w));
#pragma unroll
            for (int i = 0; i < 4; i++) v[4 * h + i] = to_f32(e[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) v[4 * h + i] = i < n ? to_f32(q[i]) : 0.0f;
        }
    }
}
template <class T>
__device__ __forceinline__ void store8(T* p, int left, const float (&v)[kVec]) {
#pragma unroll
    for (int h = 0; h < 2; h++) {
        T* q = p + 128 * h;
        const int n = left - 128 * h;
        if (n >= 4 && (reinterpret_cast<uintptr_t>(q) & (4 * sizeof(T) - 1)) == 0) {
            typedef typename std::conditional<sizeof(T) == 4, uint4, uint2>::type W;
            alignas(16) T e[4];
#pragma unroll
            for (int i = 0; i < 4; i++) from_f32(v[4 * h + i], e[i]);
            W w;
            memcpy(&w, e, sizeof(w));
            __stcs(reinterpret_cast<W*>(q), w);
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (i < n) from_f32(v[4 * h + i], q[i]);
        }
    }
}
// The same by a type known when compiled (T) or only at run time (void).
template <class T>
__device__ __forceinline__ void load8(const void* p, int type, long long at, int n, float (&v)[kVec]) {
    if constexpr (!std::is_void_v<T>) load8(static_cast<const T*>(p) + at, n, v);
    else if (type == NTCB_F32) load8(static_cast<const float*>(p) + at, n, v);
    else if (type == NTCB_F16) load8(static_cast<const __half*>(p) + at, n, v);
    else load8(static_cast<const __nv_bfloat16*>(p) + at, n, v);
}
template <class T>
__device__ __forceinline__ void store8(void* p, int type, long long at, int n, const float (&v)[kVec]) {
    if constexpr (!std::is_void_v<T>) store8(static_cast<T*>(p) + at, n, v);
    else if (type == NTCB_F32) store8(static_cast<float*>(p) + at, n, v);
    else if (type == NTCB_F16) store8(static_cast<__half*>(p) + at, n, v);
    else store8(static_cast<__nv_bfloat16*>(p) + at, n, v);
}

// The scalars of this step: as the host worked them out, or, with device scalars, the same expressions by one thread of
// the CTA (they take some hundred instructions in 64 bits; every warp working them out cost 40 % of an 8-bit step).
__device__ __forceinline__ void resolve(Scalars& c) {
    if (!c.it_dev && !c.lr_dev && !c.scale_dev) return;
    __shared__ float out[4];
    if (threadIdx.x == 0) {
        const double it = c.it_dev ? (double)*c.it_dev : (double)c.it;
        const double lr = c.lr_dev ? (double)*c.lr_dev : c.lr;
        out[0] = (float)(lr / -expm1(it * c.log_beta1));
        out[1] = (float)(1.0 / sqrt(-expm1(it * c.log_beta2)));
        out[2] = (float)(1.0 - lr * c.wd);
        out[3] = c.scale_dev ? c.scale * *c.scale_dev : c.scale;
    }
    __syncthreads();
    c.step = out[0]; c.inv = out[1]; c.decay = out[2]; c.scale = out[3];
    if (c.it_dev) c.it = (uint32_t)*c.it_dev;
}

// Products and sums of the moments are rounded one by one (no fused multiply-add), so that the 8-bit codes follow from
// elementary operations; the parameter's update uses the hardware's approximate square root and reciprocal (a few units
// in the last place of an update that is itself a small part of the parameter).
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }
template <bool FLUSH>
__device__ __forceinline__ void update2(const Scalars& c, float2& p, float2 g, float2& m, float2& v) {
    // a b + c as (a b) * one + c, one = 1 only at run time: a packed product and a packed sum would be joined to one rounding
    const float2 one = both(c.one);
    g = __fmul2_rn(g, both(c.scale));
    m = __ffma2_rn(__fmul2_rn(m, both(c.b1)), one, __fmul2_rn(g, both(c.omb1)));
    v = __ffma2_rn(__fmul2_rn(v, both(c.b2)), one, __fmul2_rn(__fmul2_rn(g, g), both(c.omb2)));
    float2 r;
    if constexpr (FLUSH) {
        asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r.x) : "f"(v.x));
        asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r.y) : "f"(v.y));
    } else {
        asm("sqrt.approx.f32 %0, %1;" : "=f"(r.x) : "f"(v.x));
        asm("sqrt.approx.f32 %0, %1;" : "=f"(r.y) : "f"(v.y));
    }
    r = __ffma2_rn(r, both(c.inv), both(c.eps));   // eps is 0 or normal and a root of v at least 2^-75, so r is 0 or normal: its
    // reciprocal needs no care for subnormals
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(r.x));
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(r.y));
    p = __ffma2_rn(__fmul2_rn(m, both(-c.step)), r, __fmul2_rn(p, both(c.decay)));
}
template <bool FLUSH>
__device__ __forceinline__ void update(const Scalars& c, float (&p)[kVec], const float (&g)[kVec], float (&m)[kVec], float (&v)[kVec]) {
#pragma unroll
    for (int i = 0; i < kVec; i += 2) {   // two elements to an instruction
        float2 p2 = make_float2(p[i], p[i + 1]), m2 = make_float2(m[i], m[i + 1]), v2 = make_float2(v[i], v[i + 1]);
        update2<FLUSH>(c, p2, make_float2(g[i], g[i + 1]), m2, v2);
        p[i] = p2.x; p[i + 1] = p2.y; m[i] = m2.x; m[i + 1] = m2.y; v[i] = v2.x; v[i + 1] = v2.y;
    }
}
// A subnormal v has a root below 2^-63, and with inv <= 2^7 (beta2 up to 0.9999 at the first step) adds less than 2^-56 to
// the denominator: nothing beside eps from 2^-33 on, so its root may be flushed to zero there (three instructions less).
__device__ __forceinline__ void update(const Scalars& c, float (&p)[kVec], const float (&g)[kVec], float (&m)[kVec], float (&v)[kVec]) {
    if (c.eps >= 1.1641532e-10f && c.inv <= 128.0f) update<true>(c, p, g, m, v);
    else update<false>(c, p, g, m, v);
}

// ---- 8-bit codes
__device__ __forceinline__ uint32_t grid_of(float x, uint32_t round) {   // q of |x|; 0 for a value that is not finite
    const uint32_t bits = __float_as_uint(x) & 0x7fffffffu;
    return bits < 0x7f800000u ? min((bits + round) >> 20, 0x7f7u) : 0u;
}
__device__ __forceinline__ uint32_t code_m(float x, uint32_t q, uint32_t base) {
    const uint32_t bits = __float_as_uint(x);
    uint32_t c = q > base ? q - base : 0u;
    if ((bits & 0x7fffffffu) >= 0x7f800000u) c = kTopM + 1;
    return c ? c | ((bits >> 24) & 0x80u) : 0u;
}
__device__ __forceinline__ uint32_t code_v(float x, uint32_t q, uint32_t base) {
    const uint32_t bits = __float_as_uint(x) & 0x7fffffffu;
    uint32_t c = q > base ? q - base : 0u;
    if (bits) c = max(c, 1u);
    return bits >= 0x7f800000u ? kTopV + 1 : c;
}
__device__ __forceinline__ float value_m(uint32_t c, uint32_t base) {
    const uint32_t k = c & 0x7fu;
    const uint32_t bits = k == 0 ? 0u : k > kTopM ? 0x7fc00000u : (k + base) << 20;
    return __uint_as_float(bits | (k ? (c & 0x80u) << 24 : 0u));
}
__device__ __forceinline__ float value_v(uint32_t c, uint32_t base) {
    return __uint_as_float(c == 0 ? 0u : c > kTopV ? 0x7fc00000u : (c + base) << 20);
}
__device__ __forceinline__ uint32_t base_of(uint32_t q, uint32_t top) {   // the warp's window: up to its largest q
    const uint32_t most = __reduce_max_sync(kFull, q);
    return most > top ? most - top : 0u;
}

struct State8 {
    uint8_t *m, *v;
    uint16_t *mb, *vb;
    __host__ __device__ State8(void* s, long long total)
        : m(static_cast<uint8_t*>(s)), v(m + total), mb(reinterpret_cast<uint16_t*>(v + total)), vb(mb + total / kBlock) {}
};

// Where the 16 random bits of each value come from: the low half of word i is m's, the high half v's.
struct Noise {          // two neighbouring elements share a 64-bit draw; i counts the lane's elements
    uint64_t first;     // key + (index of the lane's first pair) * golden: draw64(key, pair + k) = mix64(first + k golden)
    __device__ __forceinline__ uint64_t operator()(int i) const { return mix64(first + (uint64_t)(i / 4 * 64 + i % 4 / 2) * kGolden64); }
};
struct Nearest {        // half a grid step
    __device__ __forceinline__ uint64_t operator()(int) const { return 0x8000800080008000ull; }
};

// A block with values that are not finite, or that may round to infinity: value by value. Called rarely, so it keeps its
// arrays in local memory and off the common way's registers.
template <class R>
__device__ __noinline__ void encode_slow(const float* m, const float* v, R rnd, uint32_t* out) {
    uint32_t qm[kVec], qv[kVec], most_m = 0, most_v = 0;
    for (int i = 0; i < kVec; i++) {
        const uint32_t w = (uint32_t)(rnd(i) >> (32 * (i % 2)));
        qm[i] = grid_of(m[i], (w & 0xffffu) << 4); qv[i] = grid_of(v[i], (w >> 16) << 4);
        most_m = max(most_m, qm[i]); most_v = max(most_v, qv[i]);
    }
    const uint32_t bm = base_of(most_m, kTopM), bv = base_of(most_v, kTopV);
    for (int h = 0; h < 2; h++) {
        uint32_t wm = 0, wv = 0;
        for (int i = 0; i < 4; i++) {
            wm |= code_m(m[4 * h + i], qm[4 * h + i], bm) << (8 * i);
            wv |= code_v(v[4 * h + i], qv[4 * h + i], bv) << (8 * i);
        }
        out[h] = wm; out[2 + h] = wv;
    }
    out[4] = bm; out[5] = bv;
}

// Encodes one block (a warp's 256 values, eight per lane). The kernel is bound by integer and logic instructions (half
// the rate of the multiply-add pipe), so the common block takes the short way: t = |bits| + (random << 4) keeps its
// fraction, the block's largest t gives the base, and 16 (max(t, base << 20) - (base << 20)), one multiply-add, has the
// code in its top byte. A value that is not finite, or that may round to infinity, shows in the largest t.
template <class R>
__device__ __forceinline__ void encode(const State8& s, long long at, int lane, const float (&m)[kVec], const float (&v)[kVec], const R& rnd) {
    uint32_t tm[kVec], tv[kVec], most_m = 0, most_v = 0, least_v = 1;
#pragma unroll
    for (int i = 0; i < kVec; i += 2) {
        const uint64_t r = rnd(i);
        const uint32_t w[2] = {(uint32_t)r, (uint32_t)(r >> 32)};
#pragma unroll
        for (int k = 0; k < 2; k++) {
            tm[i + k] = (__float_as_uint(m[i + k]) & 0x7fffffffu) + __byte_perm(w[k], 0, 0x4410) * 16u;
            tv[i + k] = __float_as_uint(v[i + k]) + __byte_perm(w[k], 0, 0x4432) * 16u;   // v has no sign, but a NaN's
        }
        most_m = __vimax3_u32(most_m, tm[i], tm[i + 1]);
        most_v = __vimax3_u32(most_v, tv[i], tv[i + 1]);
        least_v = __vimin3_u32(least_v, __float_as_uint(v[i]), __float_as_uint(v[i + 1]));
    }
    most_m = __reduce_max_sync(kFull, most_m);
    most_v = __reduce_max_sync(kFull, most_v);
    uint32_t wm[2], wv[2], bm, bv;
    if (max(most_m, most_v) < 0x7f800000u) {
        bm = most_m >> 20; bm = bm > kTopM ? bm - kTopM : 0u;
        bv = most_v >> 20; bv = bv > kTopV ? bv - kTopV : 0u;
        const uint32_t bm20 = bm << 20, bv20 = bv << 20;
#pragma unroll
        for (int i = 0; i < kVec; i++) tm[i] = (max(tm[i], bm20) * 16u - bm20 * 16u) | (__float_as_uint(m[i]) & 0x80000000u);
        if (least_v) {   // v > 0 has at least code 1
#pragma unroll
            for (int i = 0; i < kVec; i++) tv[i] = max(tv[i], bv20 + (1u << 20)) * 16u - bv20 * 16u;
        } else {
#pragma unroll
            for (int i = 0; i < kVec; i++) tv[i] = max(tv[i], min(__float_as_uint(v[i]), 1u) * (1u << 20) + bv20) * 16u - bv20 * 16u;
        }
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const uint32_t w = __byte_perm(__byte_perm(tm[4 * h], tm[4 * h + 1], 0x0073), __byte_perm(tm[4 * h + 2], tm[4 * h + 3], 0x0073), 0x5410);
            const uint32_t some = ((w & 0x7f7f7f7fu) + 0x7f7f7f7fu) & 0x80808080u;   // zero carries no sign
            wm[h] = w & (some | 0x7f7f7f7fu);
            wv[h] = __byte_perm(__byte_perm(tv[4 * h], tv[4 * h + 1], 0x0073), __byte_perm(tv[4 * h + 2], tv[4 * h + 3], 0x0073), 0x5410);
        }
    } else {
        float am[kVec], av[kVec];
        uint32_t out[6];
#pragma unroll
        for (int i = 0; i < kVec; i++) { am[i] = m[i]; av[i] = v[i]; }
        encode_slow(am, av, rnd, out);
        wm[0] = out[0]; wm[1] = out[1]; wv[0] = out[2]; wv[1] = out[3]; bm = out[4]; bv = out[5];
    }
#pragma unroll
    for (int h = 0; h < 2; h++) {
        *reinterpret_cast<uint32_t*>(s.m + at + 128 * h + lane * 4) = wm[h];
        *reinterpret_cast<uint32_t*>(s.v + at + 128 * h + lane * 4) = wv[h];
    }
    if (lane == 0) { s.mb[at / kBlock] = (uint16_t)bm; s.vb[at / kBlock] = (uint16_t)bv; }
}
// The lane's eight values of one block: loaded (fetch) and decoded later (values), so that all loads are in flight first.
struct Codes { uint2 m, v; uint32_t bm, bv; };
__device__ __forceinline__ Codes fetch(const State8& s, long long at, int lane) {
    Codes c;
    c.m.x = *reinterpret_cast<const uint32_t*>(s.m + at + lane * 4);
    c.m.y = *reinterpret_cast<const uint32_t*>(s.m + at + 128 + lane * 4);
    c.v.x = *reinterpret_cast<const uint32_t*>(s.v + at + lane * 4);
    c.v.y = *reinterpret_cast<const uint32_t*>(s.v + at + 128 + lane * 4);
    c.bm = s.mb[at / kBlock]; c.bv = s.vb[at / kBlock];
    return c;
}
__device__ __forceinline__ void values(const Codes& c, float (&m)[kVec], float (&v)[kVec]) {
    const uint32_t wm[2] = {c.m.x, c.m.y}, wv[2] = {c.v.x, c.v.y};
    const uint32_t bm20 = c.bm << 20, bv20 = c.bv << 20;
    uint32_t nan = 0;
#pragma unroll
    for (int h = 0; h < 2; h++)
        nan |= ((wm[h] & 0x7f7f7f7fu) + 0x01010101u) | (((wv[h] & 0x7f7f7f7fu) + 0x01010101u) & wv[h]);   // a top code: bit 7 of its byte
#pragma unroll
    for (int i = 0; i < kVec; i++) {
        const uint32_t tm = __byte_perm(wm[i / 4], 0, 0x4044 | ((i % 4) << 8)), k = tm & 0x7f0000u;   // the byte at bit 16
        const uint32_t xm = (k * 16u + bm20) | ((tm * 256u) & 0x80000000u);
        m[i] = __uint_as_float(k ? xm : 0u);
        const uint32_t tv = __byte_perm(wv[i / 4], 0, 0x4044 | ((i % 4) << 8));
        v[i] = __uint_as_float(tv ? tv * 16u + bv20 : 0u);
    }
    if (nan & 0x80808080u) {
#pragma unroll
        for (int i = 0; i < kVec; i++) {
            m[i] = value_m((wm[i / 4] >> (8 * (i % 4))) & 0xffu, c.bm);
            v[i] = value_v((wv[i / 4] >> (8 * (i % 4))) & 0xffu, c.bv);
        }
    }
}

// ---- the kernels: a warp takes one block of 256 elements, a lane two quads of it
template <int BITS, class P, class G, int N>
__device__ __forceinline__ void step_block(const StepArgs<N>& a, const Scalars& c, const Chunk& ch, void* p, const void* g, int lane, int block) {
    const int left = ch.n - block - lane * 4;   // elements from this lane's first one to the end
    const long long at = ch.start + block + lane * 4;
    const long long st = ch.state + block;
    float pv[kVec], gv[kVec], m[kVec], v[kVec];
    load8<P>(p, ch.param_type, at, left, pv);
    load8<G>(g, ch.grad_type, at, left, gv);
    if constexpr (BITS == 32) {
        float* sm = static_cast<float*>(a.state) + st + lane * 4;
        float* sv = sm + a.total;
        load8(sm, kBlock, m);
        load8(sv, kBlock, v);
        update(c, pv, gv, m, v);
        store8(sm, left, m);
        store8(sv, left, v);
        store8<P>(p, ch.param_type, at, left, pv);
    } else {
        const State8 s(a.state, a.total);
        const Codes codes = fetch(s, st, lane);
        values(codes, m, v);
        update(c, pv, gv, m, v);
        store8<P>(p, ch.param_type, at, left, pv);
        if (left < 132) {
#pragma unroll
            for (int i = 0; i < kVec; i++)
                if (i / 4 * 128 + i % 4 >= left) m[i] = v[i] = 0.0f;   // behind the tensor's end
        }
        encode(s, st, lane, m, v, Noise{stream_key(c.seed, kStreamAdamW, c.it, (uint32_t)ch.tensor) + ((uint64_t)at >> 1) * kGolden64});
    }
}

// Parameters and gradients of one type are the usual case and take the compiled conversions; mixed ones choose per load.
template <int BITS, int N>
__global__ void __launch_bounds__(256, BITS == 8 ? 5 : 4) k_adamw(const __grid_constant__ StepArgs<N> a) {
    const Chunk ch = a.chunks[blockIdx.x];
    const void* g = a.g[ch.tensor - a.first];
    void* p = a.p[ch.tensor - a.first];
    if (!g) return;
    Scalars c = a.c;
    resolve(c);
    const int lane = threadIdx.x & 31, block = (threadIdx.x >> 5) * kBlock;
    if (block >= ch.n) return;
    if (ch.param_type == NTCB_F32 && ch.grad_type == NTCB_F32) step_block<BITS, float, float>(a, c, ch, p, g, lane, block);
    else if (ch.param_type == NTCB_BF16 && ch.grad_type == NTCB_BF16) step_block<BITS, __nv_bfloat16, __nv_bfloat16>(a, c, ch, p, g, lane, block);
    else step_block<BITS, void, void>(a, c, ch, p, g, lane, block);
}

__global__ void __launch_bounds__(256) k_adamw_get(const State8 s, long long total, float* __restrict__ fm, float* __restrict__ fv) {
    const int lane = threadIdx.x & 31;
    const long long at = ((long long)blockIdx.x * 8 + (threadIdx.x >> 5)) * kBlock;
    if (at >= total) return;
    float m[kVec], v[kVec];
    values(fetch(s, at, lane), m, v);
    store8(fm + at + lane * 4, kBlock, m);
    store8(fv + at + lane * 4, kBlock, v);
}
__global__ void __launch_bounds__(256) k_adamw_set(const State8 s, long long total, const float* __restrict__ fm, const float* __restrict__ fv) {
    const int lane = threadIdx.x & 31;
    const long long at = ((long long)blockIdx.x * 8 + (threadIdx.x >> 5)) * kBlock;
    if (at >= total) return;
    float m[kVec], v[kVec];
    load8(fm + at + lane * 4, kBlock, m);
    load8(fv + at + lane * 4, kBlock, v);
    encode(s, at, lane, m, v, Nearest{});
}

}  // namespace
}  // namespace ntcb

struct ntcb_adamw {
    int device = -1, bits = 32;
    std::vector<long long> size, offset;       // offset has one entry more: the total
    std::vector<int> param_type, grad_type;
    std::vector<int> first_chunk;              // per tensor, one entry more
    ntcb::Chunk* chunks = nullptr;             // device
    mutable std::atomic<bool> captured{false}; // a graph has the table's or the state's address
};

namespace ntcb {
namespace {

template <int N>
cudaError_t launch_step(const ntcb_adamw* a, const Scalars& c, void* const* params, const void* const* grads, void* state, int first,
                        int count, cudaStream_t s) {
    StepArgs<N> k;
    k.c = c;
    k.chunks = a->chunks + a->first_chunk[(size_t)first];
    k.state = state;
    k.total = a->offset.back();
    k.first = first;
    for (int i = 0; i < N; i++) {
        k.p[i] = i < count ? params[first + i] : nullptr;
        k.g[i] = i < count ? grads[first + i] : nullptr;
    }
    const int blocks = a->first_chunk[(size_t)(first + count)] - a->first_chunk[(size_t)first];
    if (blocks == 0) return cudaSuccess;
    if (a->bits == 32) k_adamw<32, N><<<(unsigned)blocks, 256, 0, s>>>(k);
    else k_adamw<8, N><<<(unsigned)blocks, 256, 0, s>>>(k);
    return cudaGetLastError();
}

// Frees (a plan may be collected while some stream of the process is being captured) must not invalidate a capture.
struct RelaxedCapture {
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    RelaxedCapture() { cudaThreadExchangeStreamCaptureMode(&mode); }
    ~RelaxedCapture() { cudaThreadExchangeStreamCaptureMode(&mode); }
};

// Whether the stream is being captured (noted in the plan); -1: it cannot be asked.
int capturing(const ntcb_adamw* a, cudaStream_t s) {
    cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
    if (cudaStreamIsCapturing(s, &cap) != cudaSuccess) { cudaGetLastError(); return -1; }
    if (cap == cudaStreamCaptureStatusNone) return 0;
    a->captured.store(true);
    return 1;
}

constexpr int kMaxPerLaunch = 1984;   // two addresses each: 31 KB of the 32 KB that a launch's arguments may take

}  // namespace
}  // namespace ntcb

extern "C" {

ntcb_adamw* ntcb_adamw_create(int device, int ntensors, const long long* sizes, const int* param_types, const int* grad_types,
                              int state_bits, char* why, size_t why_cap) {
    using namespace ntcb;
    const auto refuse = [&](const char* m) { set_why(why, why_cap, m); return static_cast<ntcb_adamw*>(nullptr); };
    if (ntensors < 1 || !sizes || !param_types || !grad_types) return refuse("no tensors");
    if (state_bits != 32 && state_bits != 8) return refuse("state_bits must be 32 or 8");
    long long total = 0, chunks = 0;   // below 2^25 + ntensors chunks
    for (int i = 0; i < ntensors; i++) {
        if (sizes[i] < 0 || sizes[i] > (1ll << 36)) return refuse("a tensor's size is outside 0 .. 2^36");
        if (param_types[i] < NTCB_F32 || param_types[i] > NTCB_BF16 || grad_types[i] < NTCB_F32 || grad_types[i] > NTCB_BF16)
            return refuse("unknown type of a parameter or a gradient");
        total += (sizes[i] + kBlock - 1) / kBlock * kBlock;
        chunks += (sizes[i] + kChunk - 1) / kChunk;
        if (total > (1ll << 36)) return refuse("more than 2^36 elements");
    }
    ntcb_adamw* a = nullptr;
    try {
        a = new ntcb_adamw;
        a->bits = state_bits;
        a->size.assign(sizes, sizes + ntensors);
        a->param_type.assign(param_types, param_types + ntensors);
        a->grad_type.assign(grad_types, grad_types + ntensors);
        std::vector<Chunk> table;
        table.reserve((size_t)chunks);
        long long at = 0;
        for (int i = 0; i < ntensors; i++) {
            a->offset.push_back(at);
            a->first_chunk.push_back((int)table.size());
            for (long long s = 0; s < sizes[i]; s += kChunk)
                table.push_back(Chunk{s, at + s, i, (int)std::min<long long>(kChunk, sizes[i] - s), param_types[i], grad_types[i]});
            at += (sizes[i] + kBlock - 1) / kBlock * kBlock;
        }
        a->offset.push_back(at);
        a->first_chunk.push_back((int)table.size());
        DeviceScope scope(device, why, why_cap);
        if (!scope.ok) { delete a; return nullptr; }
        a->device = scope.device;
        if (!table.empty()) {
            cudaError_t e = cudaMalloc(&a->chunks, table.size() * sizeof(Chunk));
            // A copy from pageable memory may return before it has reached the device, and streams that do not wait for the
            // legacy stream may take the first step: the table must be there when the plan is.
            if (e == cudaSuccess) e = cudaMemcpyAsync(a->chunks, table.data(), table.size() * sizeof(Chunk), cudaMemcpyHostToDevice, cudaStreamLegacy);
            if (e == cudaSuccess) e = cudaStreamSynchronize(cudaStreamLegacy);
            if (e != cudaSuccess) {
                cudaGetLastError();
                DeviceScope::fail("the table of work", e, why, why_cap);
                if (a->chunks) cudaFree(a->chunks);
                delete a;
                return nullptr;
            }
        }
    } catch (const std::bad_alloc&) {
        delete a;
        return refuse("out of host memory");
    }
    return a;
}

void ntcb_adamw_destroy(ntcb_adamw* a) {
    if (!a) return;
    ntcb::RelaxedCapture relaxed;
    if (a->chunks) cudaFree(a->chunks);
    delete a;
}

int ntcb_adamw_captured(const ntcb_adamw* a) { return a && a->captured.load(); }

size_t ntcb_adamw_state_bytes(const ntcb_adamw* a) {
    if (!a) return 0;
    const size_t total = (size_t)a->offset.back();
    return a->bits == 32 ? total * 8 : total * 2 + total / ntcb::kBlock * 4;
}

long long ntcb_adamw_offset(const ntcb_adamw* a, int tensor) {
    return a && tensor >= 0 && (size_t)tensor < a->offset.size() ? a->offset[(size_t)tensor] : -1;
}

int ntcb_adamw_step(const ntcb_adamw* a, void* const* params, const void* const* grads, void* state, const ntcb_adamw_args* args,
                    void* stream, char* why, size_t why_cap) {
    using namespace ntcb;
    const auto refuse = [&](const char* m) { set_why(why, why_cap, m); return 0; };
    if (!a || !params || !grads || !args) return refuse("null argument");
    const int n = (int)a->size.size();
    if (a->offset.back() && (!state || (reinterpret_cast<uintptr_t>(state) & 255))) return refuse("the state must be a 256-byte aligned buffer");
    if (!(args->beta1 >= 0.0 && args->beta1 < 1.0 && args->beta2 >= 0.0 && args->beta2 < 1.0)) return refuse("a beta is outside [0, 1)");
    if (!(args->eps >= 0.0) || !(args->weight_decay >= 0.0) || std::isinf(args->eps) || std::isinf(args->weight_decay))
        return refuse("eps and weight_decay must be finite and not negative");
    if (args->eps > 0.0 && args->eps < (double)FLT_MIN) return refuse("eps must be 0 or a normal 32-bit number (1.18e-38 or more)");
    if (!args->lr_dev && !(std::isfinite(args->lr) && args->lr >= 0.0)) return refuse("lr must be finite and not negative");
    if (!args->it_dev && (args->it < 1 || args->it > 0xffffffffll)) return refuse("it counts from 1 and stays below 2^32");
    if (reinterpret_cast<uintptr_t>(args->it_dev) % 8 || reinterpret_cast<uintptr_t>(args->lr_dev) % 4 || reinterpret_cast<uintptr_t>(args->grad_scale_dev) % 4)
        return refuse("a device scalar is not aligned to its type");
    for (int i = 0; i < n; i++) {
        if (!a->size[(size_t)i] || !grads[i]) continue;
        if (!params[i]) return refuse("null parameter");
        const size_t ps = a->param_type[(size_t)i] == NTCB_F32 ? 4 : 2, gs = a->grad_type[(size_t)i] == NTCB_F32 ? 4 : 2;
        if (reinterpret_cast<uintptr_t>(params[i]) % ps || reinterpret_cast<uintptr_t>(grads[i]) % gs) return refuse("a buffer is not aligned to its type");
    }
    DeviceScope scope(a->device, why, why_cap);
    if (!scope.ok) return 0;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int cap = capturing(a, s);
    if (cap < 0) return refuse("the stream cannot be used");
    if (cap && !args->it_dev) return refuse("a captured step must take its number from the device (it_dev)");   // a replay would repeat it
    Scalars c{};
    c.lr = args->lr; c.beta1 = args->beta1; c.beta2 = args->beta2; c.wd = args->weight_decay;
    c.log_beta1 = std::log(args->beta1); c.log_beta2 = std::log(args->beta2);
    c.b1 = (float)args->beta1; c.omb1 = (float)(1.0 - args->beta1);
    c.b2 = (float)args->beta2; c.omb2 = (float)(1.0 - args->beta2);
    c.eps = (float)args->eps; c.scale = (float)args->grad_scale; c.one = 1.0f;
    if (!args->it_dev) {
        c.step = (float)(args->lr / (1.0 - std::pow(args->beta1, (double)args->it)));
        c.inv = (float)(1.0 / std::sqrt(1.0 - std::pow(args->beta2, (double)args->it)));
    }
    c.decay = (float)(1.0 - args->lr * args->weight_decay);
    c.seed = args->seed; c.it = (uint32_t)args->it;
    c.it_dev = args->it_dev; c.lr_dev = args->lr_dev; c.scale_dev = args->grad_scale_dev;
    for (int first = 0; first < n; first += kMaxPerLaunch) {
        const int count = std::min(n - first, kMaxPerLaunch);
        const cudaError_t e = count <= 16 ? launch_step<16>(a, c, params, grads, state, first, count, s)
                              : count <= 128 ? launch_step<128>(a, c, params, grads, state, first, count, s)
                                             : launch_step<kMaxPerLaunch>(a, c, params, grads, state, first, count, s);
        if (e != cudaSuccess) return scope.launched(e, why, why_cap);
    }
    return 1;
}

int ntcb_adamw_get_moments(const ntcb_adamw* a, const void* state, float* m, float* v, void* stream, char* why, size_t why_cap) {
    using namespace ntcb;
    if (!a) { set_why(why, why_cap, "null argument"); return 0; }
    const long long total = a->offset.back();
    if (!total) return 1;
    if (!state || !m || !v || (reinterpret_cast<uintptr_t>(state) & 255) || ((reinterpret_cast<uintptr_t>(m) | reinterpret_cast<uintptr_t>(v)) & 15)) {
        set_why(why, why_cap, "null or unaligned buffer"); return 0;
    }
    DeviceScope scope(a->device, why, why_cap);
    if (!scope.ok) return 0;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (capturing(a, s) < 0) { set_why(why, why_cap, "the stream cannot be used"); return 0; }
    if (a->bits == 32) {
        cudaError_t e = cudaMemcpyAsync(m, state, (size_t)total * 4, cudaMemcpyDeviceToDevice, s);
        if (e == cudaSuccess) e = cudaMemcpyAsync(v, static_cast<const float*>(state) + total, (size_t)total * 4, cudaMemcpyDeviceToDevice, s);
        return scope.launched(e, why, why_cap);
    }
    k_adamw_get<<<(unsigned)((total + kChunk - 1) / kChunk), 256, 0, s>>>(State8(const_cast<void*>(state), total), total, m, v);
    return scope.launched(cudaGetLastError(), why, why_cap);
}

int ntcb_adamw_set_moments(const ntcb_adamw* a, const float* m, const float* v, void* state, void* stream, char* why, size_t why_cap) {
    using namespace ntcb;
    if (!a) { set_why(why, why_cap, "null argument"); return 0; }
    const long long total = a->offset.back();
    if (!total) return 1;
    if (!state || !m || !v || (reinterpret_cast<uintptr_t>(state) & 255) || ((reinterpret_cast<uintptr_t>(m) | reinterpret_cast<uintptr_t>(v)) & 15)) {
        set_why(why, why_cap, "null or unaligned buffer"); return 0;
    }
    DeviceScope scope(a->device, why, why_cap);
    if (!scope.ok) return 0;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (capturing(a, s) < 0) { set_why(why, why_cap, "the stream cannot be used"); return 0; }
    if (a->bits == 32) {
        cudaError_t e = cudaMemcpyAsync(state, m, (size_t)total * 4, cudaMemcpyDeviceToDevice, s);
        if (e == cudaSuccess) e = cudaMemcpyAsync(static_cast<float*>(state) + total, v, (size_t)total * 4, cudaMemcpyDeviceToDevice, s);
        return scope.launched(e, why, why_cap);
    }
    k_adamw_set<<<(unsigned)((total + kChunk - 1) / kChunk), 256, 0, s>>>(State8(state, total), total, m, v);
    return scope.launched(cudaGetLastError(), why, why_cap);
}

}  // extern "C"
