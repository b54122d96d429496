// Losses on rows of raw predictions that a softmax turns into probabilities, with their gradients and hessians: distillation from a
// teacher's top logits, the clipped policy loss with a KL term, the preference loss of paired log ratios (formulas: include/evb.h).
//
// All three need the same of a row z[0 .. K-1]: its maximum and the sum of 2^(c (z_k - max)), c = log2(e) / tau, a few named columns,
// and then one number A so that g_k = A 2^(c (z_k - max)) everywhere but at the named columns, which are written after the others.
// What bounds them is memory: a row is read once and its gradient written once (twice with hessians); a preference reads its rows a second time,
// because a row's factor depends on all rows of its pair.  Which kernel takes a row is a matter of its size (launch_typed):
//   k_row_few    2 to 8 classes of 32 bits: a thread per row, in registers
//   k_row_tile   up to 32 classes and slots: a thread per row, staged through shared memory
//   k_row_lanes  up to 256 granules of 16 bytes (1024 floats): some lanes of a warp
//   k_row_ctas   up to 32768 granules: a CTA, or a cluster of up to eight; with two granules a thread where there are few rows
//   k_row_walk   beyond: a CTA reads the row twice
// Sums, maxima, probabilities and losses are 32-bit floats, sums of log ratios 64-bit ones; the only rounding to 16 bits is that of the results.
#include "evb_device.cuh"
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <algorithm>
#include <atomic>
#include <math.h>

namespace {

constexpr unsigned FULL = 0xffffffffu;
constexpr int MAX_TOP = 1024;        // slots of a row
constexpr int MAX_CLASSES = 1 << 20;

enum { ROW_DISTILL = 0, ROW_POLICY = 1, ROW_LOGP = 2, ROW_COEF = 3 };

struct TaughtRow;
struct SoftArgs {
    const void *z;
    long long n, ldz;
    int K;
    float c, inv_tau, tau;  // c = log2(e) / tau
    void *g, *h;            // gradient, hessian, or null
    long long ldg, ldh;
    const float *w;         // row weights or null
    long long w_stride;
    float *loss;
    // distillation: slots of a row, ldt elements from row to row
    const uint32_t *ids;
    const void *t;
    int T, t_dtype, tail;
    long long ldt;
    const TaughtRow *taught; // per row, or null
    // policy, preference: the class taken; p_stride elements from row to row
    const uint32_t *code;
    const float *old_lp, *adv, *ref;
    long long p_stride;
    float lo, hi, beta;
    float *logp;
    // preference: maximum and 1 / sum of a row, factor of its gradient
    float2 *stat;
    const float *coef;
};

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
__device__ __forceinline__ float load_t(const void *p, int dtype, long long i) {
    if (dtype == EVB_BF16) return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
    if (dtype == EVB_F16) return __half2float(static_cast<const __half *>(p)[i]);
    return static_cast<const float *>(p)[i];
}

// Maximum m and sum of 2^(c z - M), M = round(c m), of what has been seen: a multiply-add and an exponential per term.
struct Soft { float m, s; };
__device__ __forceinline__ float base_of(float m, float c) { const float M = __fmul_rn(m, c); return M == -INFINITY ? 0.0f : M; } // nothing seen: every term is 2^-inf
__device__ __forceinline__ float rise(float m, float c, float base) { return __fmul_rn(m, c) - base; } // between two M: the product rounded, never a multiply-add
// Where M's rounding would reach the exponents, or the products overflow (masks are often made of the type's lowest value), a part of a row
// sees nothing: its terms are 2^-inf.  When that is the largest prediction of the whole row (with a tail: of the classes without a slot), it is
// looked at again, less its maximum.
__device__ __forceinline__ bool is_far(float m, float c) { return fabsf(m) * c > 1.0e9f && m != -INFINITY; }

struct RowLoss { float loss, d; }; // loss and its derivative by log p of the class taken
__device__ __forceinline__ RowLoss policy_row(float lp, float old_lp, float adv, bool has_ref, float ref, float lo, float hi, float beta) {
    const float r = expf(lp - old_lp), u = r * adv, cl = fminf(fmaxf(r, 1.0f - lo), 1.0f + hi) * adv;
    RowLoss o = {u <= cl ? -u : -cl, u <= cl ? -u : 0.0f};
    if (u != u) o = {u, u};
    if (has_ref) {
        const float x = ref - lp, e = expm1f(x);
        o.loss += beta * (e - x);
        o.d -= beta * e;
    }
    return o;
}

// ---------------------------------------------------------------------------------- rows in registers
// A row is cut into granules of 16 bytes, as memory is, not as the row begins: element k sits in granule (k + off) / E, off = elements of the
// first granule that come before the row.  The first and the last granule may belong to the row in part: their elements go one by one.
__device__ __forceinline__ float ex2(float x) { // of results below 2^-126 nothing is left
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
typedef unsigned long long f2; // two floats side by side: one instruction works on both
__device__ __forceinline__ f2 pair(float a, float b) { f2 r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ void split(f2 r, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(r)); }
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) { f2 r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c)); return r; }
__device__ __forceinline__ f2 mul2(f2 a, f2 b) { f2 r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ f2 add2(f2 a, f2 b) { f2 r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ f2 ex2_2(f2 x) {
    float a, b;
    split(x, a, b);
    return pair(ex2(a), ex2(b));
}
struct Two {
    template <typename P, int E> static __device__ __forceinline__ void get(const uint4 &r, f2 (&x)[E / 2]) {
        float y[E];
        P::get(r, y);
#pragma unroll
        for (int e = 0; e < E / 2; ++e) x[e] = pair(y[2 * e], y[2 * e + 1]);
    }
    template <typename P, int E> static __device__ __forceinline__ uint4 put(const f2 (&x)[E / 2]) {
        float y[E];
#pragma unroll
        for (int e = 0; e < E / 2; ++e) split(x[e], y[2 * e], y[2 * e + 1]);
        return P::put(y);
    }
};
template <typename ZT> struct Pack;
template <> struct Pack<float> {
    static constexpr int E = 4;
    static __device__ __forceinline__ void get2(const uint4 &r, f2 (&x)[2]) { Two::get<Pack, 4>(r, x); }
    static __device__ __forceinline__ uint4 put2(const f2 (&x)[2]) { return Two::put<Pack, 4>(x); }
    static constexpr uint32_t NONE = 0xff800000u;
    static __device__ __forceinline__ void get(const uint4 &r, float (&x)[4]) {
        x[0] = __uint_as_float(r.x); x[1] = __uint_as_float(r.y); x[2] = __uint_as_float(r.z); x[3] = __uint_as_float(r.w);
    }
    static __device__ __forceinline__ uint4 put(const float (&x)[4]) {
        return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
    }
    struct Most { // the largest of many granules
        float m = -INFINITY;
        __device__ __forceinline__ void see(const uint4 &r) {
            m = fmaxf(m, fmaxf(fmaxf(__uint_as_float(r.x), __uint_as_float(r.y)), fmaxf(__uint_as_float(r.z), __uint_as_float(r.w))));
        }
        __device__ __forceinline__ float get() const { return m; }
    };
};
template <> struct Pack<__nv_bfloat16> {
    static constexpr int E = 8;
    static __device__ __forceinline__ void get2(const uint4 &r, f2 (&x)[4]) { Two::get<Pack, 8>(r, x); }
    static __device__ __forceinline__ uint4 put2(const f2 (&x)[4]) { return Two::put<Pack, 8>(x); }
    static constexpr uint32_t NONE = 0xff80ff80u;
    static __device__ __forceinline__ void two(uint32_t w, float &a, float &b) { a = __uint_as_float(w << 16); b = __uint_as_float(w & 0xffff0000u); }
    static __device__ __forceinline__ void get(const uint4 &r, float (&x)[8]) {
        two(r.x, x[0], x[1]); two(r.y, x[2], x[3]); two(r.z, x[4], x[5]); two(r.w, x[6], x[7]);
    }
    static __device__ __forceinline__ uint32_t one(float a, float b) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&v);
    }
    static __device__ __forceinline__ uint4 put(const float (&x)[8]) { return make_uint4(one(x[0], x[1]), one(x[2], x[3]), one(x[4], x[5]), one(x[6], x[7])); }
    struct Most {
        __nv_bfloat162 m = __nv_bfloat162(__ushort_as_bfloat16(0xff80), __ushort_as_bfloat16(0xff80));
        __device__ __forceinline__ void see(const uint4 &r) {
            const __nv_bfloat162 *v = reinterpret_cast<const __nv_bfloat162 *>(&r);
            m = __hmax2(m, __hmax2(__hmax2(v[0], v[1]), __hmax2(v[2], v[3])));
        }
        __device__ __forceinline__ float get() const { const float2 f = __bfloat1622float2(m); return fmaxf(f.x, f.y); }
    };
};
template <> struct Pack<__half> {
    static constexpr int E = 8;
    static __device__ __forceinline__ void get2(const uint4 &r, f2 (&x)[4]) { Two::get<Pack, 8>(r, x); }
    static __device__ __forceinline__ uint4 put2(const f2 (&x)[4]) { return Two::put<Pack, 8>(x); }
    static constexpr uint32_t NONE = 0xfc00fc00u;
    static __device__ __forceinline__ void two(uint32_t w, float &a, float &b) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w));
        a = f.x; b = f.y;
    }
    static __device__ __forceinline__ void get(const uint4 &r, float (&x)[8]) {
        two(r.x, x[0], x[1]); two(r.y, x[2], x[3]); two(r.z, x[4], x[5]); two(r.w, x[6], x[7]);
    }
    static __device__ __forceinline__ uint32_t one(float a, float b) {
        const __half2 v = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&v);
    }
    static __device__ __forceinline__ uint4 put(const float (&x)[8]) { return make_uint4(one(x[0], x[1]), one(x[2], x[3]), one(x[4], x[5]), one(x[6], x[7])); }
    struct Most {
        __half2 m = __half2(__ushort_as_half(0xfc00), __ushort_as_half(0xfc00));
        __device__ __forceinline__ void see(const uint4 &r) {
            const __half2 *v = reinterpret_cast<const __half2 *>(&r);
            m = __hmax2(m, __hmax2(__hmax2(v[0], v[1]), __hmax2(v[2], v[3])));
        }
        __device__ __forceinline__ float get() const { const float2 f = __half22float2(m); return fmaxf(f.x, f.y); }
    };
};

// Where a row lies, and what of it belongs to one group of threads: granules v0 .. v1 - 1, of which vs .. ve - 1 are whole; `ends` elements
// of the others.
template <typename ZT> struct RowAt {
    static constexpr int E = Pack<ZT>::E;
    const ZT *z;
    ZT *g, *h;
    int K, off, v0, v1, vs, ve, head, ends;
    bool whole; // whole granules of g and h can be written: they begin where those of z do
    // `most` whole granules at most: what is left over goes with the ends
    __device__ __forceinline__ RowAt(const SoftArgs &a, long long row, int rank, int CS, int most) {
        z = static_cast<const ZT *>(a.z) + row * a.ldz;
        g = a.g ? static_cast<ZT *>(a.g) + row * a.ldg : nullptr;
        h = a.h ? static_cast<ZT *>(a.h) + row * a.ldh : nullptr;
        K = a.K;
        off = (int)((uintptr_t)z & 15) / (int)sizeof(ZT);
        const int nvec = (K + off + E - 1) / E, per = CS > 1 ? (nvec + CS - 1) / CS : nvec;
        v0 = min(rank * per, nvec);
        v1 = min(v0 + per, nvec);
        head = v0 == 0 && off > 0 ? min(K, E - off) : 0;
        vs = v0 + (head > 0);
        ve = min(max(vs, v1 - (v1 == nvec && (K + off) % E != 0)), vs + most);
        ends = head + max(0, min(K, v1 * E - off) - (ve * E - off));
        whole = (((g ? (uintptr_t)g ^ (uintptr_t)z : 0) | (h ? (uintptr_t)h ^ (uintptr_t)z : 0)) & 15) == 0;
    }
    __device__ __forceinline__ int end_at(int j) const { return j < head ? j : ve * E - off + j - head; } // element of end j
    __device__ __forceinline__ const uint4 *granules() const { return reinterpret_cast<const uint4 *>(z - off); }
    __device__ __forceinline__ uint4 load(int v) const { return __ldg(granules() + v); }
    __device__ __forceinline__ void store(ZT *o, int v, const float (&x)[E]) const {
        if (whole) { reinterpret_cast<uint4 *>(o - off)[v] = Pack<ZT>::put(x); return; }
#pragma unroll
        for (int e = 0; e < E; ++e) o[v * E - off + e] = from_f<ZT>(x[e]);
    }
    __device__ __forceinline__ void fill(int t, int nt, float value) const {
        float x[E];
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = value;
        for (int v = vs + t; v < ve; v += nt) {
            if (g) store(g, v, x);
            if (h) store(h, v, x);
        }
        for (int j = t; j < ends; j += nt) {
            if (g) g[end_at(j)] = from_f<ZT>(value);
            if (h) h[end_at(j)] = from_f<ZT>(value);
        }
    }
};

// joined by `width` lanes that lie side by side, in a fixed order; every one of them gets it
__device__ __forceinline__ float lanes_sum(float v, int width) {
    for (int o = width >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(FULL, v, o);
    return v;
}
__device__ __forceinline__ float lanes_max(float v, int width) {
    if (width == 32) {
        float m;
        asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(v));
        return m;
    }
    for (int o = width >> 1; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(FULL, v, o));
    return v;
}
__device__ __forceinline__ Soft lanes_join(Soft r, float c, int width) {
    const float m = lanes_max(r.m, width);
    return {m, lanes_sum(r.s * ex2(rise(r.m, c, base_of(m, c))), width)};
}
__device__ __forceinline__ Soft join(Soft a, Soft b, float c) {
    const float m = fmaxf(a.m, b.m), base = base_of(m, c);
    return {m, a.s * ex2(rise(a.m, c, base)) + b.s * ex2(rise(b.m, c, base))};
}
__device__ __forceinline__ bool marked(const uint32_t *bits, int b) { return bits[b >> 5] >> (b & 31) & 1u; }
template <int E> __device__ __forceinline__ unsigned granule_bits(const uint32_t *bits, int u) { return bits[u * E >> 5] >> (u * E & 31) & ((1u << E) - 1u); }

// A thread's part of a row: granules vs + t, vs + t + nt, ..
template <typename ZT, int V>
__device__ __forceinline__ void fetch(uint4 (&r)[V], const RowAt<ZT> &at, int t, int nt, bool live) {
    const uint4 *p = at.granules() + at.vs + t;
    const int left = live ? at.ve - at.vs : 0;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        if ((i + 1) * nt <= left) r[i] = __ldg(p + i * nt);        // the same for all threads of the row
        else r[i] = i * nt + t < left ? __ldg(p + i * nt) : make_uint4(Pack<ZT>::NONE, Pack<ZT>::NONE, Pack<ZT>::NONE, Pack<ZT>::NONE);
    }
}
template <typename ZT, int V>
__device__ __forceinline__ void leave_out(uint4 (&r)[V], const RowAt<ZT> &at, const uint32_t *bits, int t, int nt) {
    constexpr int E = Pack<ZT>::E;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int v = at.vs + t + i * nt;
        const unsigned b = v < at.ve ? granule_bits<E>(bits, v - at.v0) : 0u;
        if (b) {
            ZT *x = reinterpret_cast<ZT *>(&r[i]);
#pragma unroll
            for (int e = 0; e < E; ++e) if (b >> e & 1u) x[e] = from_f<ZT>(-INFINITY);
        }
    }
}
template <typename ZT, int V>
__device__ __forceinline__ float terms_of(uint4 (&r)[V], float c, float nb) {
    constexpr int E = Pack<ZT>::E;
    float s[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < V; ++i) {
        float x[E];
        Pack<ZT>::get(r[i], x);
#pragma unroll
        for (int e = 0; e < E; ++e) { x[e] = ex2(fmaf(x[e], c, nb)); s[e & 1] += x[e]; }
        if (E == 4) r[i] = Pack<ZT>::put(x);
        else asm volatile("" : "+r"(r[i].x), "+r"(r[i].y), "+r"(r[i].z), "+r"(r[i].w)); // they stay packed: unpacked they would take twice the registers
    }
    return s[0] + s[1];
}
// `bits`: null, or marks of the elements to leave out, from the first of granule v0.  32-bit elements become their terms (relative to the
// thread's maximum), so that no exponential is worked out twice; 16-bit ones stay: their terms would take twice the registers.
template <typename ZT, int V>
__device__ __forceinline__ Soft take(uint4 (&r)[V], const RowAt<ZT> &at, float c, const uint32_t *bits, int t, int nt, bool live) {
    constexpr int E = Pack<ZT>::E;
    if (bits) leave_out<ZT, V>(r, at, bits, t, nt);
    typename Pack<ZT>::Most most;
#pragma unroll
    for (int i = 0; i < V; ++i) most.see(r[i]);
    float m = most.get();
    for (int j = t; live && j < at.ends; j += nt) {
        const int k = at.end_at(j);
        if (!bits || !marked(bits, k + at.off - at.v0 * E)) m = fmaxf(m, to_f(at.z[k]));
    }
    const float nb = is_far(m, c) ? -INFINITY : -base_of(m, c);
    float sum = terms_of<ZT, V>(r, c, nb);
    for (int j = t; live && j < at.ends; j += nt) {
        const int k = at.end_at(j);
        if (!bits || !marked(bits, k + at.off - at.v0 * E)) sum += ex2(fmaf(to_f(at.z[k]), c, nb));
    }
    return {m, sum};
}
// The part again, less the row's maximum.  Differences of 16-bit numbers are rounded to their type: where |c m| is above 1e9 two of them are
// equal or 2^11 and more exponents apart, before as after.
template <typename ZT, int V>
__device__ __noinline__ void less_mem(uint4 (&r)[V], const RowAt<ZT> &at, float m, const uint32_t *bits, int t, int nt) {
    constexpr int E = Pack<ZT>::E;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int v = at.vs + t + i * nt;
        if (v >= at.ve) continue;
        r[i] = at.load(v);
        const unsigned b = bits ? granule_bits<E>(bits, v - at.v0) : 0u;
        ZT *x = reinterpret_cast<ZT *>(&r[i]);
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = from_f<ZT>(b >> e & 1u ? -INFINITY : to_f(x[e]) - m);
    }
}
template <typename ZT, int V>
__device__ __noinline__ float take_far_mem(uint4 (&r)[V], const RowAt<ZT> &at, float m, float c, const uint32_t *bits, int t, int nt) {
    constexpr int E = Pack<ZT>::E;
    less_mem<ZT, V>(r, at, m, bits, t, nt);
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        float x[E];
        Pack<ZT>::get(r[i], x);
        const bool in = at.vs + t + i * nt < at.ve;
#pragma unroll
        for (int e = 0; e < E; ++e) { x[e] = in ? ex2(x[e] * c) : 0.0f; sum += x[e]; }
        if (E == 4) r[i] = Pack<ZT>::put(x);
    }
    for (int j = t; j < at.ends; j += nt) {
        const int k = at.end_at(j);
        if (!bits || !marked(bits, k + at.off - at.v0 * E)) sum += ex2((to_f(at.z[k]) - m) * c);
    }
    return sum;
}

// calls: what they are given lies in memory, and only there does it
template <typename ZT, int V>
__device__ __forceinline__ void less(uint4 (&r)[V], const RowAt<ZT> &at, float m, const uint32_t *bits, int t, int nt) {
    uint4 q[V];
#pragma unroll
    for (int i = 0; i < V; ++i) q[i] = r[i];
    less_mem<ZT, V>(q, at, m, bits, t, nt);
#pragma unroll
    for (int i = 0; i < V; ++i) r[i] = q[i];
}
template <typename ZT, int V>
__device__ __forceinline__ float take_far(uint4 (&r)[V], const RowAt<ZT> &at, float m, float c, const uint32_t *bits, int t, int nt) {
    uint4 q[V];
#pragma unroll
    for (int i = 0; i < V; ++i) q[i] = make_uint4(0u, 0u, 0u, 0u);
    const float sum = take_far_mem<ZT, V>(q, at, m, c, bits, t, nt);
#pragma unroll
    for (int i = 0; i < V; ++i) r[i] = q[i];
    return sum;
}

// Slots of a row in shared memory
struct Slots {
    int *id;            // class, 0-based, -1: none
    float *t, *z;       // what the teacher has, the row's prediction
    float *q;           // the teacher's probability: written by teach_row
    static constexpr int BYTES = 16;
    __device__ __forceinline__ Slots(void *p, int T) {
        id = static_cast<int *>(p);
        t = reinterpret_cast<float *>(id + T);
        z = t + T; q = z + T;
    }
};
constexpr float LN2 = 0.693147180559945309f, LOG2E = 1.44269504088896341f;
struct RowOut {
    float M, A, B;      // gradient A e and probability B e of the classes that are not named, e = 2^(c (z - shift) - M)
    float shift;        // 0, or the maximum of a row that is far away
    float special;      // gradient of the class taken
    float mass;         // distillation: sum of the teacher's probabilities; else: factor of (delta - p)
    float hw;           // hessian hw p (1 - p)
    float lp;           // log p of the class taken
    float loss;
    float all_M, all_ls; // distillation: log2 of the sum over all classes, in two parts, ..
    float all_shift;     // .. of predictions less this: 0, or their maximum
};
__device__ __forceinline__ bool first_slot(const Slots &s, int j) {
    for (int i = 0; i < j; ++i) if (s.id[i] == s.id[j]) return false;
    return true;
}
// What a row's slots say by themselves, before its maximum and sum are known: the sum Q of the teacher's probabilities (1 without a tail), sum q log q,
// the largest named prediction zn, sum q (z - zn), and (tail) sum of 2^(c (z - zn)) over the classes named, each of them once
struct Teach { float Q, H, zn, qz, s; };
struct alignas(16) TaughtRow { Teach teach; int flags; float tmax, r; }; // slots' flags; their largest logit, 1 / sum
// `width` lanes share the slots; all of them get the same.  Slots without a class have id -1
__device__ __forceinline__ Teach teach_row(const SoftArgs &a, const Slots &s, bool dup, int lane, int width) {
    constexpr float SHARE = 1.0f / MAX_TOP; // the sum of slots that are not normalised yet stays within 32 bits when one of them does
    const float c = a.c;
    Teach o = {0.0f, 0.0f, -INFINITY, 0.0f, 0.0f};
    float tmax = -INFINITY;
    for (int j = lane; j < a.T; j += width) if (s.id[j] >= 0) { tmax = fmaxf(tmax, s.t[j]); o.zn = fmaxf(o.zn, s.z[j]); }
    if (!a.tail) tmax = lanes_max(tmax, width);
    o.zn = lanes_max(o.zn, width);
    const float zn = o.zn == -INFINITY ? 0.0f : o.zn;
    for (int j = lane; j < a.T; j += width) {
        if (s.id[j] < 0) continue;
        const float lt = a.tail ? s.t[j] : (s.t[j] - tmax) * a.inv_tau, e = ex2(lt * LOG2E), d = s.z[j] - zn;
        s.q[j] = e;
        o.Q += e;
        if (e != 0.0f) { o.H += e * lt; o.qz += e * (d * SHARE); }
        if (a.tail && (!dup || first_slot(s, j))) o.s += ex2(d * c);
    }
    o.Q = lanes_sum(o.Q, width); o.H = lanes_sum(o.H, width); o.qz = lanes_sum(o.qz, width);
    if (a.tail) { o.s = lanes_sum(o.s, width); o.qz /= SHARE; return o; }
    const float r = 1.0f / o.Q;
    for (int j = lane; j < a.T; j += width) if (s.id[j] >= 0) s.q[j] *= r;
    o.H = o.H * r - logf(o.Q);
    o.qz *= r / SHARE;
    o.Q = 1.0f;
    return o;
}
// tau log p = tau ln 2 y, or the difference to the row's maximum where the product with c, not that itself, is beyond 32 bits
__device__ __forceinline__ float tau_log_p(const SoftArgs &a, float y, float less_max) { return y == -INFINITY ? less_max : LN2 * a.tau * y; }
// r: maximum and sum of the row, less `shift`; with a tail of the classes that have no slot.  The named ones may lie anywhere then (masks leave
// them alone, or only them): all classes together are relative to the larger of the two maxima, those without a slot among themselves to theirs.
__device__ __forceinline__ RowOut finish_row(const SoftArgs &a, const Teach &e, Soft r, float shift, float w) {
    const float c = a.c, zn = e.zn, zr = r.m + shift;
    const bool above = a.tail && zn > zr;
    RowOut o;
    o.M = base_of(r.m, c);
    o.shift = shift;
    o.all_shift = !above ? shift : is_far(zn, c) ? zn : 0.0f;
    o.all_M = !above ? o.M : base_of(zn - o.all_shift, c);
    // The exponent that brings r.s there.  r.s is relative to c r.m rounded, e.s to c zn itself: they differ by up to half a step of the product
    const float part = !above ? 0.0f : zr == -INFINITY ? zr : fmaf(zr - o.all_shift, c, -o.all_M) - fmaf(r.m, c, -o.M);
    float sum = above ? r.s * ex2(part) : r.s;
    if (a.tail) sum += e.s * ex2(fmaf(zn - o.all_shift, c, -o.all_M));
    const float ls = o.all_ls = log2f(sum);
    // the rest, when there is any: no class is left where every one is named or ruled out
    const float qt = a.tail && r.m != -INFINITY ? fmaxf(0.0f, 1.0f - e.Q) : 0.0f;
    const float lp = tau_log_p(a, fmaf(zn - o.all_shift, c, -o.all_M) - ls, zn - (above ? zn : zr));
    o.loss = a.tau * e.H - (e.qz + (zn == -INFINITY ? e.qz == 0.0f ? 0.0f : zn : e.Q > 0.0f ? lp * e.Q : 0.0f));
    if (zn == -INFINITY && e.Q > 0.0f) o.loss = isfinite(ls) ? INFINITY : NAN; // nothing that the teacher names is possible; or they are NaN, or all is ruled out
    if (qt > 0.0f) o.loss += qt * (logf(qt) - tau_log_p(a, part + log2f(r.s) - ls, zr - (above ? zn : zr)));
    o.mass = e.Q + qt;
    o.B = r.m == -INFINITY ? 0.0f * ls : ex2(part) / sum;
    o.A = w * a.tau * (o.mass * o.B - (qt > 0.0f ? qt / r.s : 0.0f));
    o.hw = w;
    o.special = o.lp = 0.0f;
    o.loss *= w * a.tau; // up to here in units of the predictions, as are its largest parts
    return o;
}
__device__ __forceinline__ float slot_p(const SoftArgs &a, const RowOut &o, float z) { return ex2(fmaf(z - o.all_shift, a.c, -o.all_M) - o.all_ls); }
__device__ __forceinline__ float less_p(float lp) { return lp < -0.5f ? 1.0f - ex2(lp * LOG2E) : -expm1f(lp); } // 1 - p, also where p is close to 1
// what belongs to the class taken, read ahead of its use
struct Taken { float z, old_lp, adv, ref; };
template <typename ZT, int KIND>
__device__ __forceinline__ Taken taken_row(const SoftArgs &a, const RowAt<ZT> &at, long long row, int code) {
    Taken t = {to_f(at.z[code]), 0.0f, 0.0f, 0.0f};
    if (KIND == ROW_POLICY) {
        const long long i = row * a.p_stride;
        t.old_lp = a.old_lp[i]; t.adv = a.adv[i];
        if (a.ref) t.ref = a.ref[i];
    }
    return t;
}
template <int KIND>
__device__ __forceinline__ RowOut class_row(const SoftArgs &a, Soft r, float shift, const Taken &t, float w) {
    RowOut o;
    o.M = base_of(r.m, a.c);
    o.shift = shift;
    o.B = 1.0f / r.s;
    // A preference adds up hundreds of them: 64 bits, and in units of the c that the terms were made with, so that roundings which all rows share
    // do not add up too
    if (KIND == ROW_LOGP) o.lp = (float)((fma((double)(t.z - shift), (double)a.c, -(double)o.M) - log2((double)r.s)) / ((double)a.c * (double)a.tau));
    else {
        const float y = fmaf(t.z - shift, a.c, -o.M) - log2f(r.s); // as tau_log_p
        o.lp = y == -INFINITY ? (t.z - shift - r.m) * a.inv_tau : LN2 * y;
    }
    o.mass = 0.0f;
    o.loss = 0.0f;
    if (KIND == ROW_POLICY) {
        const RowLoss l = policy_row(o.lp, t.old_lp, t.adv, a.ref != nullptr, t.ref, a.lo, a.hi, a.beta);
        o.loss = w * l.loss;
        o.mass = w * l.d * a.inv_tau;
    }
    o.A = -o.mass * o.B;
    o.special = o.mass * less_p(o.lp);
    o.hw = w * a.inv_tau * a.inv_tau;
    return o;
}
// the second pass over a row of a preference; y of stat is negative for a row that is far away
__device__ __forceinline__ RowOut coef_row(const SoftArgs &a, float2 st, float lp, float w) {
    RowOut o = {};
    o.shift = st.y < 0.0f ? st.x : 0.0f;
    o.M = st.y < 0.0f ? 0.0f : base_of(st.x, a.c);
    o.B = fabsf(st.y); o.lp = lp; o.mass = w; o.A = -w * o.B;
    o.special = w * less_p(o.lp);
    return o;
}
// A thread's part of the gradient (and hessian); terms(i, x): the terms of its granule i, to be multiplied by `scale`
template <typename ZT, int KIND, int V, typename F>
__device__ __forceinline__ void give(const SoftArgs &a, const RowAt<ZT> &at, const RowOut &o, int t, int nt, float scale, int code, F terms) {
    constexpr int E = Pack<ZT>::E;
    const float A = o.A * scale, B = o.B * scale, c = a.c, nb = -o.M;
    const int special = KIND == ROW_DISTILL ? -1 : code + at.off;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int v = at.vs + t + i * nt;
        if (v >= at.ve) break;
        float x[E], y[E];
        terms(i, x);
#pragma unroll
        for (int e = 0; e < E; ++e) y[e] = x[e] * A;
        if (at.g) {
            at.store(at.g, v, y);
            if (KIND != ROW_DISTILL && (unsigned)(special - v * E) < (unsigned)E) at.g[code] = from_f<ZT>(o.special);
        }
        if (at.h) {
#pragma unroll
            for (int e = 0; e < E; ++e) { const float p = x[e] * B; y[e] = o.hw * p * (1.0f - p); }
            at.store(at.h, v, y);
        }
    }
    for (int j = t; j < at.ends; j += nt) {
        const int k = at.end_at(j);
        const float e = ex2(fmaf(to_f(at.z[k]) - o.shift, c, nb)), p = e * o.B;
        if (at.g) at.g[k] = from_f<ZT>(KIND != ROW_DISTILL && k == code ? o.special : e * o.A);
        if (at.h) at.h[k] = from_f<ZT>(o.hw * p * (1.0f - p));
    }
}
// of a part that is held in granules, as predictions or (32 bits, unless it was not summed) as terms
template <typename ZT, int KIND, int V>
__device__ __forceinline__ void give(const SoftArgs &a, const RowAt<ZT> &at, const RowOut &o, const uint4 (&r)[V], int t, int nt, float scale, int code) {
    constexpr int E = Pack<ZT>::E;
    give<ZT, KIND, V>(a, at, o, t, nt, scale, code, [&](int i, float (&x)[E]) {
        Pack<ZT>::get(r[i], x);
        if (E == 8 || KIND == ROW_COEF) {
#pragma unroll
            for (int e = 0; e < E; ++e) x[e] = ex2(fmaf(x[e], a.c, -o.M));
        }
    });
}
// the named classes, after all others have been written
template <typename ZT>
__device__ __forceinline__ void put_slot(const SoftArgs &a, const RowAt<ZT> &at, const RowOut &o, const Slots &s, int j, bool dup, float w) {
    float q = s.q[j];
    if (dup) {
        if (!first_slot(s, j)) return;
        q = 0.0f;
        for (int i = j; i < a.T; ++i) if (s.id[i] == s.id[j]) q += s.q[i];
    }
    const float p = slot_p(a, o, s.z[j]);
    if (at.g) at.g[s.id[j]] = from_f<ZT>(w * a.tau * (o.mass * p - q));
    if (at.h) at.h[s.id[j]] = from_f<ZT>(o.hw * p * (1.0f - p));
}

enum { SLOT_SOME = 1, SLOT_BAD = 2, SLOT_TWICE = 4 };
// Slot j of a row into shared memory, its prediction z given; those classes among granules v0 .. v1 - 1 are marked in `bits` (bit: element from
// the first of granule v0)
template <typename ZT>
__device__ __forceinline__ int put_slot_into(const SoftArgs &a, const RowAt<ZT> &at, const Slots &s, uint32_t *bits, int j, uint32_t id, float t, float z) {
    const bool use = id != 0u && t != -INFINITY, ok = use && id <= (uint32_t)a.K;
    s.id[j] = ok ? (int)id - 1 : -1;
    s.t[j] = t;
    s.z[j] = z;
    int flags = (use ? SLOT_SOME : 0) | (use && !ok ? SLOT_BAD : 0);
    const int b = (int)id - 1 + at.off - at.v0 * RowAt<ZT>::E;
    if (ok && b >= 0 && b < (at.v1 - at.v0) * RowAt<ZT>::E && (atomicOr(&bits[b >> 5], 1u << (b & 31)) >> (b & 31) & 1u)) flags |= SLOT_TWICE;
    return flags;
}
template <typename ZT>
__device__ __forceinline__ int put_into(const SoftArgs &a, const RowAt<ZT> &at, const Slots &s, uint32_t *bits, long long row, int j) {
    const uint32_t id = a.ids[row * a.ldt + j];
    return put_slot_into(a, at, s, bits, j, id, load_t(a.t, a.t_dtype, row * a.ldt + j), id != 0u && id <= (uint32_t)a.K ? to_f(at.z[id - 1]) : 0.0f);
}

// Rows of up to V granules for each of G lanes (a power of two up to 32): 32 / G rows a warp, 8 warps a CTA.
template <typename ZT, int KIND, int V>
// The row stays in registers between its two uses.  Measured: policy 20011 x 1000 f32 34 us (floor 24), 100k x 200 f32 with ten slots 66 (26).  At 200
// classes four rows share a warp, which takes 840 instructions for a policy (39 us), 1340 with one slot (57), 1520 with ten (66), 1870 with 32 (84):
// what slots cost is mostly the same however many there are, their loops and sums over lanes.  The issue slots are 59 % used, with 22 warps an SM (80 registers).
__global__ void __launch_bounds__(256) k_row_lanes(SoftArgs a, int G, int words) {
    extern __shared__ __align__(16) unsigned char s_raw[];
    constexpr int E = Pack<ZT>::E;
    const int lane = threadIdx.x & (G - 1), group = threadIdx.x / G;
    const long long row0 = (long long)blockIdx.x * (256 / G) + group;
    const bool there = row0 < a.n;
    const long long row = there ? row0 : a.n - 1;
    const RowAt<ZT> at(a, row, 0, 1, 0x7fffffff - (1 << 22));
    unsigned char *mine = s_raw + (size_t)group * (KIND == ROW_DISTILL ? a.T * Slots::BYTES + words * 4 : 0);
    const Slots s(mine, KIND == ROW_DISTILL ? a.T : 0);
    uint32_t *bits = reinterpret_cast<uint32_t *>(mine + (size_t)a.T * Slots::BYTES);
    float w = a.w ? a.w[row * a.w_stride] : 1.0f;
    if (KIND == ROW_COEF) w = a.coef[row];
    uint32_t id = 0u;
    if (KIND != ROW_DISTILL) id = a.code[row * a.p_stride];
    bool live = there && w != 0.0f && (KIND == ROW_DISTILL || id != 0u);
    int flags = 0;
    uint4 r[V];
    fetch<ZT, V>(r, at, lane, G, live);
    if (KIND == ROW_DISTILL) {
        for (int i = lane; i < words; i += G) bits[i] = 0u;
        __syncwarp();
        if (live) for (int j = lane; j < a.T; j += G) flags |= put_into(a, at, s, bits, row, j);
        for (int o = G >> 1; o > 0; o >>= 1) flags |= __shfl_xor_sync(FULL, flags, o);
        __syncwarp();
        live = live && (flags & SLOT_SOME);
    } else if (live && id > (uint32_t)a.K) flags = SLOT_BAD;
    const bool whole = live && !(flags & SLOT_BAD);
    const int code = whole && KIND != ROW_DISTILL ? (int)id - 1 : -1;
    const Taken taken = code >= 0 ? taken_row<ZT, KIND>(a, at, row, code) : Taken{};
    if (there && !whole) {
        const float value = live ? NAN : 0.0f;
        if (KIND != ROW_LOGP) at.fill(lane, G, value);
        if (lane == 0) {
            if (KIND != ROW_COEF && a.loss) a.loss[row] = value;
            if ((KIND == ROW_POLICY || KIND == ROW_LOGP) && a.logp) a.logp[row] = value;
            if (KIND == ROW_LOGP) a.stat[row] = make_float2(0.0f, value);
        }
    }
    Soft mine_r = {0.0f, 1.0f}, all = mine_r;
    float shift = 0.0f;
    RowOut o = {};
    if (KIND == ROW_COEF) {
        if (whole) {
            o = coef_row(a, a.stat[row], a.logp[row], w);
            if (o.shift != 0.0f) less<ZT, V>(r, at, o.shift, nullptr, lane, G);
        }
    } else {
        const uint32_t *out = KIND == ROW_DISTILL && a.tail && whole ? bits : nullptr;
        mine_r = take<ZT, V>(r, at, a.c, out, lane, G, whole);
        all = lanes_join(mine_r, a.c, G);
        const bool far = whole && is_far(all.m, a.c) && all.m != INFINITY;
        if (__any_sync(FULL, far)) {
            if (far) { shift = all.m; mine_r = {0.0f, take_far<ZT, V>(r, at, shift, a.c, out, lane, G)}; }
            all = lanes_join(mine_r, a.c, G);
        }
        if (KIND == ROW_DISTILL) {
            if (!whole) for (int j = lane; j < a.T; j += G) s.id[j] = -1;
            __syncwarp();
            o = finish_row(a, teach_row(a, s, flags & SLOT_TWICE, lane, G), all, shift, w);
        }
        else if (whole) o = class_row<KIND>(a, all, shift, taken, w);
    }
    if (whole) {
        if (lane == 0) {
            if ((KIND == ROW_DISTILL || KIND == ROW_POLICY) && a.loss) a.loss[row] = o.loss;
            if ((KIND == ROW_POLICY || KIND == ROW_LOGP) && a.logp) a.logp[row] = o.lp;
            if (KIND == ROW_LOGP) a.stat[row] = shift != 0.0f ? make_float2(shift, -o.B) : make_float2(all.m, o.B);
        }
        const float scale = E == 4 && KIND != ROW_COEF ? ex2(rise(mine_r.m, a.c, o.M)) : 1.0f;
        if (KIND != ROW_LOGP) give<ZT, KIND, V>(a, at, o, r, lane, G, scale, code);
    }
    if (KIND == ROW_DISTILL) {
        __syncwarp();
        if (whole && (at.g || at.h)) for (int j = lane; j < a.T; j += G) if (s.id[j] >= 0) put_slot(a, at, o, s, j, flags & SLOT_TWICE, w);
    }
}

// Rows of up to 32 classes: a thread per row, 128 rows a CTA, all that they hold staged through shared memory so that memory is read and written
// in order.  Rows of shared memory are an odd number of words apart: neighbours fall into different banks.
// Policy 1M x 18 with hessians: 52 us (floor 37): shared memory is busy for 82 % of them, 1110 instructions a row.
constexpr int TILE = 128, TILE_K = 32, TILE_T = 32;
struct TileGeom { int Kp, Tp; uint32_t by_K, by_T; }; // by_*: (c * by) >> 32 is c / K (c / T) for c < 2^13
template <typename T, typename F>
__device__ __forceinline__ void tile_read(const T *src, long long ld, int rows, int W, uint32_t by, F put) { // put(row, column, value)
    const int n = rows * W;
    int c0 = 0;
    if (sizeof(T) == 4 && ld == W && ((uintptr_t)src & 15) == 0) {
        c0 = n & ~3;
        for (int c = 4 * threadIdx.x; c < c0; c += 4 * TILE) {
            const uint4 v = __ldg(reinterpret_cast<const uint4 *>(src + c));
            const T *x = reinterpret_cast<const T *>(&v);
#pragma unroll
            for (int e = 0; e < 4; ++e) { const int r = W == 1 ? c + e : __umulhi(c + e, by); put(r, c + e - r * W, x[e]); }
        }
    }
    for (int c = c0 + threadIdx.x; c < n; c += TILE) { const int r = W == 1 ? c : __umulhi(c, by), k = c - r * W; put(r, k, src[r * ld + k]); }
}
template <typename T>
__device__ __forceinline__ void tile_write(T *dst, long long ld, int rows, int W, int Wp, uint32_t by, const float *s) {
    const int n = rows * W;
    int c0 = 0;
    if (sizeof(T) == 4 && ld == W && ((uintptr_t)dst & 15) == 0) {
        c0 = n & ~3;
        for (int c = 4 * threadIdx.x; c < c0; c += 4 * TILE) {
            float x[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) { const int r = W == 1 ? c + e : __umulhi(c + e, by); x[e] = s[r * Wp + c + e - r * W]; }
            *reinterpret_cast<float4 *>(dst + c) = make_float4(x[0], x[1], x[2], x[3]);
        }
    }
    for (int c = c0 + threadIdx.x; c < n; c += TILE) { const int r = W == 1 ? c : __umulhi(c, by), k = c - r * W; dst[r * ld + k] = from_f<T>(s[r * Wp + k]); }
}
template <typename ZT, int KIND>
__global__ void __launch_bounds__(TILE) k_row_tile(SoftArgs a, TileGeom ge) {
    extern __shared__ __align__(16) float s_tile[]; // predictions, then gradients [TILE][Kp]; hessians; slots: four words [TILE][Tp] each
    constexpr bool DIST = KIND == ROW_DISTILL;
    const long long row0 = (long long)blockIdx.x * TILE, row = row0 + threadIdx.x;
    const int K = a.K, Kp = ge.Kp, rows = (int)min((long long)TILE, a.n - row0);
    float *s_z = s_tile, *s_h = s_z + (a.h ? TILE * Kp : 0), *s_s = s_h + TILE * Kp;
    const int T = DIST ? a.T : 0;
    const bool here = (int)threadIdx.x < rows;
    float w = 0.0f;
    uint32_t id = 0u;
    Taken taken = {};
    float2 st = make_float2(0.0f, 0.0f);
    float st_lp = 0.0f;
    if (here) {
        w = KIND == ROW_COEF ? a.coef[row] : a.w ? a.w[row * a.w_stride] : 1.0f;
        if (!DIST) id = a.code[row * a.p_stride];
        if (KIND == ROW_POLICY) {
            const long long i = row * a.p_stride;
            taken.old_lp = a.old_lp[i]; taken.adv = a.adv[i];
            if (a.ref) taken.ref = a.ref[i];
        }
        if (KIND == ROW_COEF) { st = a.stat[row]; st_lp = a.logp[row]; }
    }
    tile_read(static_cast<const ZT *>(a.z) + row0 * a.ldz, a.ldz, rows, K, ge.by_K, [&](int r, int k, ZT v) { s_z[r * Kp + k] = to_f(v); });
    if (DIST) {
        const int Tp = ge.Tp;
        tile_read(a.ids + row0 * a.ldt, a.ldt, rows, T, ge.by_T, [&](int r, int j, uint32_t v) { reinterpret_cast<uint32_t *>(s_s)[r * Tp + j] = v; });
        float *s_t = s_s + TILE * Tp;
        if (a.t_dtype == EVB_F32) tile_read(static_cast<const float *>(a.t) + row0 * a.ldt, a.ldt, rows, T, ge.by_T, [&](int r, int j, float v) { s_t[r * Tp + j] = v; });
        else if (a.t_dtype == EVB_BF16) tile_read(static_cast<const __nv_bfloat16 *>(a.t) + row0 * a.ldt, a.ldt, rows, T, ge.by_T, [&](int r, int j, __nv_bfloat16 v) { s_t[r * Tp + j] = to_f(v); });
        else tile_read(static_cast<const __half *>(a.t) + row0 * a.ldt, a.ldt, rows, T, ge.by_T, [&](int r, int j, __half v) { s_t[r * Tp + j] = to_f(v); });
    }
    __syncthreads();
    if (here) {
        float *z = s_z + threadIdx.x * Kp, *h = s_h + threadIdx.x * Kp;
        bool live = w != 0.0f && (DIST || id != 0u);
        int flags = !DIST && live && id > (uint32_t)K ? SLOT_BAD : 0;
        uint32_t named = 0u; // a bit per class
        Slots s(s_s, 0);
        if (DIST) {
            s.id = reinterpret_cast<int *>(s_s) + threadIdx.x * ge.Tp;
            s.t = s_s + (TILE + threadIdx.x) * ge.Tp;
            s.z = s.t + TILE * ge.Tp; s.q = s.z + TILE * ge.Tp;
            for (int j = 0; j < T && live; ++j) {
                const uint32_t k = (uint32_t)s.id[j];
                const bool use = k != 0u && s.t[j] != -INFINITY, ok = use && k <= (uint32_t)K;
                flags |= use ? ok ? SLOT_SOME | (named >> (k - 1) & 1u ? SLOT_TWICE : 0) : SLOT_SOME | SLOT_BAD : 0;
                s.id[j] = ok ? (int)k - 1 : -1;
                if (ok) { named |= 1u << (k - 1); s.z[j] = z[k - 1]; }
            }
            live = live && (flags & SLOT_SOME);
        }
        float loss = 0.0f, lp = 0.0f;
        float2 stat = make_float2(0.0f, 0.0f);
        if (!live || (flags & SLOT_BAD)) {
            loss = lp = stat.y = live ? NAN : 0.0f;
            for (int k = 0; k < K; ++k) { z[k] = loss; if (a.h) h[k] = loss; }
        } else {
            const uint32_t out = DIST && a.tail ? named : 0u;
            RowOut o = {};
            float m = -INFINITY;
            if (KIND == ROW_COEF) {
                o = coef_row(a, st, st_lp, w);
                m = st.x;
            } else {
                for (int k = 0; k < K; ++k) if (!(out >> k & 1u)) m = fmaxf(m, z[k]);
            }
            // 2^(c (z - max)): differences, so that no prediction is too far away
            const float base = m == -INFINITY ? 0.0f : m;
            float sum = 0.0f;
            if (!DIST) taken.z = z[id - 1] - base;
            for (int k = 0; k < K; ++k) {
                const float e = ex2((z[k] - base) * a.c);
                if (!(out >> k & 1u)) sum += e;
                z[k] = e;
            }
            const float zero = m == -INFINITY ? m : 0.0f; // the maximum, less itself
            if (DIST) { o = finish_row(a, teach_row(a, s, flags & SLOT_TWICE, 0, 1), Soft{zero, sum}, base, w); loss = o.loss; }
            else if (KIND != ROW_COEF) {
                o = class_row<KIND>(a, Soft{zero, sum}, 0.0f, taken, w);
                loss = o.loss; lp = o.lp;
                stat = make_float2(m, is_far(m, a.c) ? -o.B : o.B);
            }
            if (KIND != ROW_LOGP) {
                for (int k = 0; k < K; ++k) {
                    const float e = z[k], p = e * o.B;
                    z[k] = e * o.A;
                    if (a.h) h[k] = o.hw * p * (1.0f - p);
                }
                if (!DIST) z[id - 1] = o.special;
                else for (int j = 0; j < T; ++j) {
                    if (s.id[j] < 0) continue;
                    float q = s.q[j];
                    if (flags & SLOT_TWICE) {
                        if (!first_slot(s, j)) continue;
                        q = 0.0f;
                        for (int i = j; i < T; ++i) if (s.id[i] == s.id[j]) q += s.q[i];
                    }
                    const float p = slot_p(a, o, s.z[j]);
                    z[s.id[j]] = w * a.tau * (o.mass * p - q);
                    if (a.h) h[s.id[j]] = o.hw * p * (1.0f - p);
                }
            }
        }
        if (KIND != ROW_COEF && a.loss) a.loss[row] = loss;
        if ((KIND == ROW_POLICY || KIND == ROW_LOGP) && a.logp) a.logp[row] = lp;
        if (KIND == ROW_LOGP) a.stat[row] = stat;
    }
    if (KIND == ROW_LOGP) return;
    __syncthreads();
    if (a.g) tile_write(static_cast<ZT *>(a.g) + row0 * a.ldg, a.ldg, rows, K, Kp, ge.by_K, s_z);
    if (a.h) tile_write(static_cast<ZT *>(a.h) + row0 * a.ldh, a.ldh, rows, K, Kp, ge.by_K, s_h);
}

// The same for 2 to 8 classes of 32 bits, their number known to the compiler: a row's predictions stay in registers, read by their thread alone (the
// rows of a warp are neighbours: what one thread leaves of a line, others take); gradients and hessians go out through shared memory.
// 2M x 5 with three slots and hessians: 65 us (floor 28), 845 instructions a row that use 77 % of the issue slots; k_row_tile takes 100 us and 1400.
template <int KIND, int K>
__global__ void __launch_bounds__(TILE) k_row_few(SoftArgs a) {
    extern __shared__ __align__(16) float s_tile[]; // gradients [TILE][K], hessians
    constexpr bool DIST = KIND == ROW_DISTILL;
    const long long row0 = (long long)blockIdx.x * TILE, row = row0 + threadIdx.x;
    const int rows = (int)min((long long)TILE, a.n - row0);
    float *s_g = s_tile + threadIdx.x * K, *s_h = s_g + TILE * K;
    if ((int)threadIdx.x < rows) {
        const float *zp = static_cast<const float *>(a.z) + row * a.ldz;
        float z[K], y[K];
#pragma unroll
        for (int k = 0; k < K; ++k) z[k] = __ldg(zp + k);
        const float w = KIND == ROW_COEF ? a.coef[row] : a.w ? a.w[row * a.w_stride] : 1.0f, c = a.c;
        const uint32_t id = DIST ? 0u : a.code[row * a.p_stride];
        Taken taken = {};
        if (KIND == ROW_POLICY) {
            const long long i = row * a.p_stride;
            taken.old_lp = a.old_lp[i]; taken.adv = a.adv[i];
            if (a.ref) taken.ref = a.ref[i];
        }
        // the teacher's probability of every class; the classes that it names
        float Q = 0.0f, entropy = 0.0f, q[K];
        uint32_t named = 0u;
        bool some = false, bad = !DIST && id > (uint32_t)K;
        if (DIST) {
            const long long at = row * a.ldt;
#pragma unroll
            for (int k = 0; k < K; ++k) q[k] = 0.0f;
            float tmax = -INFINITY;
            if (!a.tail) for (int j = 0; j < a.T; ++j) if (a.ids[at + j] != 0u) tmax = fmaxf(tmax, load_t(a.t, a.t_dtype, at + j));
            for (int j = 0; j < a.T; ++j) {
                const uint32_t k1 = a.ids[at + j];
                const float t = load_t(a.t, a.t_dtype, at + j);
                if (k1 == 0u || t == -INFINITY) continue;
                some = true;
                bad = bad || k1 > (uint32_t)K;
                named |= 1u << ((k1 - 1) & 31);
                const float lt = a.tail ? t : (t - tmax) * a.inv_tau, e = ex2(lt * LOG2E);
                Q += e;
                if (e != 0.0f) entropy += e * lt;
#pragma unroll
                for (int k = 0; k < K; ++k) if (k + 1 == (int)k1) q[k] += e;
            }
        }
        const bool live = w != 0.0f && (DIST ? some : id != 0u);
        float loss = 0.0f, lp = 0.0f;
        float2 stat = make_float2(0.0f, 0.0f);
        if (!live || bad) {
            loss = lp = stat.y = live ? NAN : 0.0f;
#pragma unroll
            for (int k = 0; k < K; ++k) y[k] = z[k] = loss;
        } else {
            // 2^(c (z - max)): differences, so that no prediction is too far away.  With a tail the classes that are not named have a maximum of their own
            const uint32_t out = DIST && a.tail ? named : 0u;
            float m = -INFINITY, all_m = -INFINITY, sum = 0.0f, rest = 0.0f;
#pragma unroll
            for (int k = 0; k < K; ++k) { all_m = fmaxf(all_m, z[k]); if (!(out >> k & 1u)) m = fmaxf(m, z[k]); }
            const float base = all_m == -INFINITY ? 0.0f : all_m;
#pragma unroll
            for (int k = 0; k < K; ++k) { y[k] = ex2((z[k] - base) * c); sum += y[k]; }
            const float zero = all_m == -INFINITY ? all_m : 0.0f;
            if (DIST) {
                const float ls = log2f(sum), lq = a.tail ? 0.0f : logf(Q), rQ = a.tail ? 1.0f : 1.0f / Q, r = 1.0f / sum;
                if (zero != 0.0f) loss = NAN;
                loss += a.tau * (entropy * rQ - (a.tail ? 0.0f : lq));
                float qt = 0.0f, rbase = 0.0f, rr = 0.0f;
                if (a.tail && m != -INFINITY) {
                    qt = fmaxf(0.0f, 1.0f - Q);
                    rbase = m;
#pragma unroll
                    for (int k = 0; k < K; ++k) if (!(out >> k & 1u)) rest += ex2((z[k] - rbase) * c);
                    rr = qt / rest;
                    if (qt > 0.0f) loss += qt * (logf(qt) - (rbase - base) - LN2 * (log2f(rest) - ls)); // tau = 1
                }
                const float mass = a.tail ? Q + qt : 1.0f, f = w * a.tau;
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    const float qk = q[k] * rQ, p = y[k] * r;
                    if (qk != 0.0f) loss -= qk * (z[k] - base - LN2 * a.tau * ls);
                    float g = mass * p - qk;
                    if (a.tail && !(out >> k & 1u) && qt > 0.0f) g = mass * p - rr * ex2((z[k] - rbase) * c);
                    z[k] = f * g;
                    y[k] = w * p * (1.0f - p);
                }
                loss *= w * a.tau;
            } else {
                RowOut o;
#pragma unroll
                for (int k = 0; k < K; ++k) if (k + 1 == (int)id) taken.z = z[k] - base;
                if (KIND == ROW_COEF) o = coef_row(a, a.stat[row], a.logp[row], w);
                else {
                    o = class_row<KIND>(a, Soft{zero, sum}, 0.0f, taken, w);
                    loss = o.loss; lp = o.lp;
                    stat = make_float2(all_m, is_far(all_m, c) ? -o.B : o.B);
                }
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    const float p = y[k] * o.B;
                    z[k] = k + 1 == (int)id ? o.special : y[k] * o.A;
                    y[k] = o.hw * p * (1.0f - p);
                }
            }
        }
        if (KIND != ROW_COEF && a.loss) a.loss[row] = loss;
        if ((KIND == ROW_POLICY || KIND == ROW_LOGP) && a.logp) a.logp[row] = lp;
        if (KIND == ROW_LOGP) a.stat[row] = stat;
#pragma unroll
        for (int k = 0; k < K; ++k) { s_g[k] = z[k]; if (a.h) s_h[k] = y[k]; }
    }
    if (KIND == ROW_LOGP) return;
    __syncthreads();
    auto give = [&](float *dst, long long ld, const float *from) {
        const int n = rows * K;
        if (ld == K && ((uintptr_t)dst & 15) == 0) {
            for (int c = threadIdx.x; c < n >> 2; c += TILE) reinterpret_cast<float4 *>(dst)[c] = reinterpret_cast<const float4 *>(from)[c];
            for (int c = (n & ~3) + threadIdx.x; c < n; c += TILE) dst[c] = from[c];
        } else {
            for (int c = threadIdx.x; c < n; c += TILE) { const int r = c / K; dst[r * ld + (c - r * K)] = from[c]; }
        }
    };
    if (a.g) give(static_cast<float *>(a.g) + row0 * a.ldg, a.ldg, s_tile);
    if (a.h) give(static_cast<float *>(a.h) + row0 * a.ldh, a.ldh, s_tile + TILE * K);
}

// What the CTAs of a cluster tell one another: maximum and sum of their parts of a row.  Each writes its words into the shared memory
// of all; a barrier there counts the bytes.
struct Mail {
    float2 word[8];
    unsigned long long bar;
};
__device__ __forceinline__ uint32_t smem_at(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void bar_init(unsigned long long *bar, int count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_at(bar)), "r"(count) : "memory"); }
__device__ __forceinline__ void bar_expect(unsigned long long *bar, int bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_at(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mail_send(Mail *m, int from, int to, Soft r) {
    uint32_t at, bar;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_at(&m->word[from])), "r"(to));
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(bar) : "r"(smem_at(&m->bar)), "r"(to));
    asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v2.b32 [%0], {%1, %2}, [%3];" ::"r"(at), "r"(__float_as_uint(r.m)),
                 "r"(__float_as_uint(r.s)), "r"(bar) : "memory");
}
// waits for a phase of a barrier, about a microsecond a try; false: it did not come within a second
__device__ __forceinline__ bool bar_wait(unsigned long long *bar, unsigned parity) {
    for (int k = 0; k < (1 << 20); ++k) {
        uint32_t done;
        asm volatile("{ .reg .pred p; mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3; selp.u32 %0, 1, 0, p; }"
                     : "=r"(done) : "r"(smem_at(bar)), "r"(parity), "r"(1000u) : "memory");
        if (done) return true;
    }
    return false;
}

// Whether a class has several slots: the classes go into an open table of at least twice as many places
__host__ __device__ constexpr int table_places(int T) { int n = 64; while (n < 2 * T) n *= 2; return n; }
__device__ __forceinline__ bool table_has(int *table, int places, int id) {
    uint32_t at = (uint32_t)id * 2654435761u >> 16 & (places - 1);
    for (int tries = 0; tries < places; ++tries) {
        const int old = atomicCAS(table + at, -1, id);
        if (old == -1) return false;
        if (old == id) return true;
        at = (at + 1) & (places - 1);
    }
    return false;
}

// One row for a CTA of NT threads, or for a cluster of 1 << lcs of them, up to V granules a thread.  The row stays in registers (16-bit predictions
// packed, their exponentials worked out twice; 32-bit ones as their terms), so it is read once.  Between loads and stores lies a chain that
// no single row can hide (the sums over lanes, warps, CTAs; the row's numbers: some 4000 of 12000 clocks), so what counts is how many rows an SM has
// in hand: eight granules a thread at 64 registers, 1024 threads.  Measured and left: rows that a CTA stays for, fetched ahead by bulk
// copies into a ring (2.4 to 3.0 TB/s instead of 4.2); independent warps in two passes, the second out of L2 (2.1); a warp more for the slots
// (three CTAs an SM instead of four: 770 us instead of 597).  4.9 TB/s for 8192 x 65537 bf16 (420 us, floor 316).
// PRE: k_row_taught has seen to the slots (4096 x 131072 bf16 with 64 and a tail: 528 us, floor 322; 597 without).
template <typename ZT, int KIND, int V, int NT, bool PRE = false>
__global__ void __launch_bounds__(NT, (V == 16 ? 512 : 1024) / NT) k_row_ctas(SoftArgs a, int lcs, int words) {
    extern __shared__ __align__(16) unsigned char s_raw[];
    __shared__ Mail s_mail[2];
    __shared__ float2 s_part[32];
    __shared__ RowOut s_out;
    __shared__ int s_flags;
    constexpr int E = Pack<ZT>::E, H = E / 2, WARPS = NT / 32;
    constexpr bool DIST = KIND == ROW_DISTILL;
    constexpr bool TERMS = E == 4 && KIND != ROW_COEF; // 32-bit predictions become their terms
    const int t = threadIdx.x, lane = t & 31, CS = 1 << lcs;
    // a second pass begins with the rows that the first one read last: they are still in L2
    const long long row = KIND == ROW_COEF ? a.n - 1 - (blockIdx.x >> lcs) : blockIdx.x >> lcs;
    const int rank = blockIdx.x & (CS - 1);
    uint32_t id = 0u;
    if (!DIST) id = a.code[row * a.p_stride];
    float w = KIND == ROW_COEF ? a.coef[row] : a.w ? a.w[row * a.w_stride] : 1.0f;
    if (CS > 1 && KIND != ROW_COEF) {
        if (t == 0) {
            for (int q = 0; q < 2; ++q) { bar_init(&s_mail[q].bar, 1); bar_expect(&s_mail[q].bar, 8 * CS); }
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        __syncthreads();
        asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    }
    const RowAt<ZT> at(a, row, rank, CS, V * NT);
    const int count = at.ve - at.vs, left = count - t; // whole granules; of them, this thread's and those behind them
    const int end = t < at.ends ? at.end_at(t) : -1; // as many as threads at most
    const Slots s(s_raw, DIST ? a.T : 0);
    uint32_t *bits = reinterpret_cast<uint32_t *>(s_raw + (PRE ? 0 : (size_t)a.T * Slots::BYTES));
    TaughtRow pre = {};
    if (DIST && PRE) pre.flags = __ldg(&a.taught[row].flags);
    bool live = w != 0.0f && (DIST ? !PRE || (pre.flags & SLOT_SOME) : id != 0u);
    uint4 r[V];
    ZT end_raw = from_f<ZT>(-INFINITY);
    {
        const uint4 *p = at.granules() + at.vs + t;
        const uint4 none = make_uint4(Pack<ZT>::NONE, Pack<ZT>::NONE, Pack<ZT>::NONE, Pack<ZT>::NONE);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            r[i] = none;
            if (live && i * NT < left) r[i] = __ldg(p + i * NT);
        }
        if (live && end >= 0) end_raw = at.z[end];
    }
    // what the class taken brings along, raw: a conversion here would wait for it
    const int code = DIST ? -1 : (int)id - 1;
    int flags = DIST ? pre.flags : live && id > (uint32_t)a.K ? SLOT_BAD : 0;
    ZT code_raw = from_f<ZT>(0.0f);
    Taken taken = {};
    float2 st = make_float2(0.0f, 0.0f);
    float st_lp = 0.0f;
    if (KIND == ROW_COEF) { st = a.stat[row]; st_lp = a.logp[row]; }
    else if (!DIST && live && !flags && t < 32) {
        code_raw = at.z[code];
        if (KIND == ROW_POLICY) {
            const long long i = row * a.p_stride;
            taken.old_lp = a.old_lp[i]; taken.adv = a.adv[i];
            if (a.ref) taken.ref = a.ref[i];
        }
    }
    Teach teach = {};
    if (DIST && PRE) {
        if (live && t < 32) {
            const float4 *from = reinterpret_cast<const float4 *>(a.taught + row);
            const float4 x = __ldg(from), y = __ldg(from + 1);
            teach = {x.x, x.y, x.z, x.w, y.x};
        }
        if (live && a.tail) { // marks of the classes named
            for (int i = t; i < words; i += NT) bits[i] = 0u;
            __syncthreads();
            for (int j = t; j < a.T; j += NT) {
                const uint32_t k = __ldg(a.ids + row * a.ldt + j);
                const int b = (int)k - 1 + at.off - at.v0 * E;
                if (k != 0u && k <= (uint32_t)a.K && b >= 0 && b < (at.v1 - at.v0) * E && load_t(a.t, a.t_dtype, row * a.ldt + j) != -INFINITY)
                    atomicOr(&bits[b >> 5], 1u << (b & 31));
            }
            __syncthreads();
        }
    } else if (DIST && live) {
        int *table = reinterpret_cast<int *>(bits + words);
        const int places = table_places(a.T);
        if (t == 0) s_flags = 0;
        for (int i = t; i < words; i += NT) bits[i] = 0u;
        for (int i = t; i < places; i += NT) table[i] = -1;
        __syncthreads();
        for (int j = t; j < a.T; j += NT) {
            flags |= put_into(a, at, s, bits, row, j);
            if (s.id[j] >= 0 && table_has(table, places, s.id[j])) flags |= SLOT_TWICE; // of all classes, where the marks are of this CTA's
        }
        flags = __reduce_or_sync(FULL, flags);
        if (lane == 0 && flags) atomicOr(&s_flags, flags);
        __syncthreads();
        flags = s_flags;
        live = flags & SLOT_SOME;
    }
    if (CS > 1 && KIND != ROW_COEF) asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); // the others' mail is open
    if (!live || (flags & SLOT_BAD)) {
        const float value = live ? NAN : 0.0f;
        if (KIND != ROW_LOGP) at.fill(t, NT, value);
        if (t == 0 && rank == 0) {
            if (KIND != ROW_COEF && a.loss) a.loss[row] = value;
            if ((KIND == ROW_POLICY || KIND == ROW_LOGP) && a.logp) a.logp[row] = value;
            if (KIND == ROW_LOGP) a.stat[row] = make_float2(0.0f, value);
        }
        return;
    }
    Soft mine = {0.0f, 1.0f};
    RowOut o;
    if (KIND == ROW_COEF) {
        o = coef_row(a, st, st_lp, w);
        if (o.shift != 0.0f) less<ZT, V>(r, at, o.shift, nullptr, t, NT);
    } else {
        const uint32_t *out = DIST && a.tail ? bits : nullptr;
        if (out) leave_out<ZT, V>(r, at, out, t, NT);
        if (out && end >= 0 && marked(out, end + at.off - at.v0 * E)) end_raw = from_f<ZT>(-INFINITY);
        typename Pack<ZT>::Most most;
#pragma unroll
        for (int i = 0; i < V; ++i) if (i * NT < count) most.see(r[i]);
        const float end_z = to_f(end_raw);
        mine.m = fmaxf(most.get(), end_z);
        {
            const float nb = is_far(mine.m, a.c) ? -INFINITY : -base_of(mine.m, a.c);
            const f2 c2 = pair(a.c, a.c), b2 = pair(nb, nb);
            f2 sum[2] = {0, 0};
#pragma unroll
            for (int i = 0; i < V; ++i) {
                if (i * NT >= count) break; // the same for all threads
                f2 x[H];
                Pack<ZT>::get2(r[i], x);
#pragma unroll
                for (int e = 0; e < H; ++e) { x[e] = ex2_2(fma2(x[e], c2, b2)); sum[e & 1] = add2(sum[e & 1], x[e]); }
                if (TERMS) r[i] = Pack<ZT>::put2(x);
                else asm volatile("" : "+r"(r[i].x), "+r"(r[i].y), "+r"(r[i].z), "+r"(r[i].w)); // they stay packed: unpacked they would take twice the registers
            }
            float lo, hi;
            split(add2(sum[0], sum[1]), lo, hi);
            mine.s = lo + hi + ex2(fmaf(end_z, a.c, nb));
        }
        // the parts of the threads, the warps and the CTAs are joined, the last two by every warp for itself
        auto whole_row = [&](Mail *mail) {
            Soft all = lanes_join(mine, a.c, 32);
            if (lane == 0) s_part[t >> 5] = make_float2(all.m, all.s);
            __syncthreads();
            const float2 p = lane < WARPS ? s_part[lane] : make_float2(-INFINITY, 0.0f);
            all = lanes_join(Soft{p.x, p.y}, a.c, 32);
            if (CS > 1) {
                if (t < CS) mail_send(mail, rank, t, all);
                const bool came = bar_wait(&mail->bar, 0u);
                const float2 q = lane < CS ? mail->word[lane] : make_float2(-INFINITY, 0.0f);
                all = lanes_join(Soft{q.x, q.y}, a.c, 32);
                if (!came) all.s = NAN;
            }
            return all;
        };
        Soft all = whole_row(&s_mail[0]);
        float shift = 0.0f;
        if (is_far(all.m, a.c) && all.m != INFINITY) { // the same for all threads of the row
            __syncthreads();
            shift = all.m;
            mine = {0.0f, take_far<ZT, V>(r, at, shift, a.c, out, t, NT)};
            all = whole_row(&s_mail[1]);
        }
        if (t < 32) {
            taken.z = to_f(code_raw);
            if (DIST) o = finish_row(a, PRE ? teach : teach_row(a, s, flags & SLOT_TWICE, lane, 32), all, shift, w);
            else o = class_row<KIND>(a, all, shift, taken, w);
            if (lane == 0) {
                s_out = o;
                if (rank == 0) {
                    if ((DIST || KIND == ROW_POLICY) && a.loss) a.loss[row] = o.loss;
                    if ((KIND == ROW_POLICY || KIND == ROW_LOGP) && a.logp) a.logp[row] = o.lp;
                    if (KIND == ROW_LOGP) a.stat[row] = shift != 0.0f ? make_float2(shift, -o.B) : make_float2(all.m, o.B);
                }
            }
        }
        if (KIND == ROW_LOGP) return;
        __syncthreads();
        o = s_out;
    }
    if (!(at.g || at.h)) return;
    if (at.whole && !at.h) {
        // nothing but the gradient, whole granules
        const float A = TERMS ? o.A * ex2(rise(mine.m, a.c, o.M)) : o.A;
        const f2 c2 = pair(a.c, a.c), b2 = pair(-o.M, -o.M), A2 = pair(A, A);
        uint4 *p = reinterpret_cast<uint4 *>(at.g - at.off) + at.vs + t;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            if (i * NT >= count) break;
            if (i * NT >= left) continue;
            f2 x[H];
            Pack<ZT>::get2(r[i], x);
#pragma unroll
            for (int e = 0; e < H; ++e) x[e] = mul2(TERMS ? x[e] : ex2_2(fma2(x[e], c2, b2)), A2);
            p[i * NT] = Pack<ZT>::put2(x);
        }
        const int k = (code + at.off) / E - at.vs - t; // the class taken, by the thread that has written its granule
        if (!DIST && k >= 0 && k < left && k % NT == 0) at.g[code] = from_f<ZT>(o.special);
        if (end >= 0) at.g[end] = from_f<ZT>(!DIST && end == code ? o.special : ex2(fmaf(to_f(end_raw) - o.shift, a.c, -o.M)) * o.A);
    } else {
        give<ZT, KIND, V>(a, at, o, r, t, NT, TERMS ? ex2(rise(mine.m, a.c, o.M)) : 1.0f, code);
    }
    if (DIST) {
        __syncthreads();
        if (PRE) {
            const float2 q = __ldg(reinterpret_cast<const float2 *>(&a.taught[row].tmax)); // the largest of its logits, 1 / sum
            for (int j = t; j < a.T; j += NT) {
                const uint32_t k = __ldg(a.ids + row * a.ldt + j);
                const int v = ((int)k - 1 + at.off) / E;
                if (k == 0u || v < at.v0 || v >= at.v1) continue;
                const float x = load_t(a.t, a.t_dtype, row * a.ldt + j);
                if (x == -INFINITY) continue;
                float qk = ex2(a.tail ? x * LOG2E : (x - q.x) * a.c) * q.y;
                if (flags & SLOT_TWICE) { // the first slot of a class writes for all of them
                    bool again = false;
                    qk = 0.0f;
                    for (int i = 0; i < a.T; ++i) {
                        const float y = load_t(a.t, a.t_dtype, row * a.ldt + i);
                        if (a.ids[row * a.ldt + i] != k || y == -INFINITY) continue;
                        again = again || i < j;
                        qk += ex2(a.tail ? y * LOG2E : (y - q.x) * a.c) * q.y;
                    }
                    if (again) continue;
                }
                const float p = slot_p(a, o, to_f(at.z[k - 1]));
                if (at.g) at.g[k - 1] = from_f<ZT>(w * a.tau * (o.mass * p - qk));
                if (at.h) at.h[k - 1] = from_f<ZT>(o.hw * p * (1.0f - p));
            }
        } else {
            for (int j = t; j < a.T; j += NT) {
                const int k = s.id[j], v = (k + at.off) / E;
                if (k >= 0 && v >= at.v0 && v < at.v1) put_slot(a, at, o, s, j, flags & SLOT_TWICE, w);
            }
        }
    }
}

// The teacher's side of rows that k_row_ctas works on next: a warp per row.
template <typename ZT>
__global__ void __launch_bounds__(256) k_row_taught(SoftArgs a, TaughtRow *to) {
    extern __shared__ __align__(16) unsigned char s_raw[];
    const int lane = threadIdx.x & 31, places = table_places(a.T);
    const long long row = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (row >= a.n) return;
    unsigned char *mine = s_raw + (size_t)(threadIdx.x >> 5) * (a.T * Slots::BYTES + places * 4);
    const Slots s(mine, a.T);
    int *table = reinterpret_cast<int *>(mine + (size_t)a.T * Slots::BYTES);
    const ZT *z = static_cast<const ZT *>(a.z) + row * a.ldz;
    const float w = a.w ? a.w[row * a.w_stride] : 1.0f;
    for (int i = lane; i < places; i += 32) table[i] = -1;
    __syncwarp();
    int flags = 0;
    float tmax = -INFINITY;
    for (int j = lane; j < a.T && w != 0.0f; j += 32) {
        const uint32_t k = __ldg(a.ids + row * a.ldt + j);
        const float t = load_t(a.t, a.t_dtype, row * a.ldt + j);
        const bool use = k != 0u && t != -INFINITY, ok = use && k <= (uint32_t)a.K;
        flags |= (use ? SLOT_SOME : 0) | (use && !ok ? SLOT_BAD : 0) | (ok && table_has(table, places, (int)k - 1) ? SLOT_TWICE : 0);
        s.id[j] = ok ? (int)k - 1 : -1;
        s.t[j] = t;
        s.z[j] = ok ? to_f(z[k - 1]) : 0.0f;
        if (ok) tmax = fmaxf(tmax, t);
    }
    flags = __reduce_or_sync(FULL, flags);
    tmax = lanes_max(tmax, 32);
    __syncwarp();
    TaughtRow o = {};
    o.flags = flags;
    if ((flags & SLOT_SOME) && !(flags & SLOT_BAD)) {
        o.teach = teach_row(a, s, flags & SLOT_TWICE, lane, 32);
        float sum = 0.0f; // as teach_row has it
        if (!a.tail) for (int j = lane; j < a.T; j += 32) if (s.id[j] >= 0) sum += ex2((s.t[j] - tmax) * a.inv_tau * LOG2E);
        o.tmax = tmax;
        o.r = a.tail ? 1.0f : 1.0f / lanes_sum(sum, 32);
    }
    if (lane == 0) {
        if (!(flags & SLOT_SOME) || (flags & SLOT_BAD)) o.teach = Teach{};
        to[row] = o;
    }
}

// Rows of more granules than a cluster holds: one CTA walks over a row twice.
template <typename ZT, int KIND>
__global__ void __launch_bounds__(512) k_row_walk(SoftArgs a, int words) {
    extern __shared__ __align__(16) unsigned char s_raw[];
    __shared__ float2 s_part[32];
    __shared__ RowOut s_out;
    __shared__ int s_flags;
    constexpr int E = Pack<ZT>::E;
    const int tid = threadIdx.x, nt = blockDim.x, lane = tid & 31, warps = nt >> 5;
    const long long row = blockIdx.x;
    const RowAt<ZT> at(a, row, 0, 1, 0x7fffffff - (1 << 22));
    const Slots s(s_raw, KIND == ROW_DISTILL ? a.T : 0);
    uint32_t *bits = reinterpret_cast<uint32_t *>(s_raw + (size_t)a.T * Slots::BYTES);
    float w = a.w ? a.w[row * a.w_stride] : 1.0f;
    if (KIND == ROW_COEF) w = a.coef[row];
    uint32_t id = 0u;
    if (KIND != ROW_DISTILL) id = a.code[row * a.p_stride];
    bool live = w != 0.0f && (KIND == ROW_DISTILL || id != 0u);
    int flags = live && KIND != ROW_DISTILL && id > (uint32_t)a.K ? SLOT_BAD : 0;
    if (KIND == ROW_DISTILL && live) {
        if (tid == 0) s_flags = 0;
        for (int i = tid; i < words; i += nt) bits[i] = 0u;
        __syncthreads();
        for (int j = tid; j < a.T; j += nt) flags |= put_into(a, at, s, bits, row, j);
        flags = __reduce_or_sync(FULL, flags);
        if (lane == 0 && flags) atomicOr(&s_flags, flags);
        __syncthreads();
        flags = s_flags;
        live = flags & SLOT_SOME;
    }
    if (!live || (flags & SLOT_BAD)) {
        const float value = live ? NAN : 0.0f;
        if (KIND != ROW_LOGP) at.fill(tid, nt, value);
        if (tid == 0) {
            if (KIND != ROW_COEF && a.loss) a.loss[row] = value;
            if ((KIND == ROW_POLICY || KIND == ROW_LOGP) && a.logp) a.logp[row] = value;
            if (KIND == ROW_LOGP) a.stat[row] = make_float2(0.0f, value);
        }
        return;
    }
    const int code = KIND != ROW_DISTILL ? (int)id - 1 : -1;
    const Taken taken = code >= 0 ? taken_row<ZT, KIND>(a, at, row, code) : Taken{};
    RowOut o = {};
    float shift = 0.0f;
    RowAt<ZT> piece = at; // 4 granules a thread at a time, the ends with the last
    const uint32_t *out = KIND == ROW_DISTILL && a.tail ? bits : nullptr;
    if (KIND == ROW_COEF) {
        o = coef_row(a, a.stat[row], a.logp[row], w);
        shift = o.shift;
    } else {
        Soft all = {-INFINITY, 0.0f};
        for (piece.vs = at.vs; piece.vs < at.ve || piece.vs == at.vs; piece.vs += 4 * nt) {
            const bool last = piece.vs + 4 * nt >= at.ve;
            piece.ends = last ? at.ends : 0;
            uint4 r[4];
            fetch<ZT, 4>(r, piece, tid, nt, true);
            all = join(all, take<ZT, 4>(r, piece, a.c, out, tid, nt, true), a.c);
        }
        auto whole_row = [&]() {
            all = lanes_join(all, a.c, 32);
            if (lane == 0) s_part[tid >> 5] = make_float2(all.m, all.s);
            __syncthreads();
            const float2 p = lane < warps ? s_part[lane] : make_float2(-INFINITY, 0.0f);
            all = lanes_join(Soft{p.x, p.y}, a.c, 32);
        };
        whole_row();
        if (is_far(all.m, a.c) && all.m != INFINITY) {
            __syncthreads();
            shift = all.m;
            all = {0.0f, 0.0f};
            for (piece.vs = at.vs; piece.vs < at.ve || piece.vs == at.vs; piece.vs += 4 * nt) {
                piece.ends = piece.vs + 4 * nt >= at.ve ? at.ends : 0;
                uint4 r[4] = {};
                all.s += take_far<ZT, 4>(r, piece, shift, a.c, out, tid, nt);
            }
            whole_row();
        }
        if (KIND == ROW_DISTILL) {
            if (tid < 32) {
                o = finish_row(a, teach_row(a, s, flags & SLOT_TWICE, lane, 32), all, shift, w);
                if (tid == 0) s_out = o;
            }
            __syncthreads();
            o = s_out;
        } else o = class_row<KIND>(a, all, shift, taken, w);
        if (KIND == ROW_LOGP && tid == 0) a.stat[row] = shift != 0.0f ? make_float2(shift, -o.B) : make_float2(all.m, o.B);
    }
    if (tid == 0) {
        if ((KIND == ROW_DISTILL || KIND == ROW_POLICY) && a.loss) a.loss[row] = o.loss;
        if ((KIND == ROW_POLICY || KIND == ROW_LOGP) && a.logp) a.logp[row] = o.lp;
    }
    if (KIND == ROW_LOGP || !(at.g || at.h)) return;
    for (piece.vs = at.vs; piece.vs < at.ve || piece.vs == at.vs; piece.vs += 4 * nt) {
        piece.ends = piece.vs + 4 * nt >= at.ve ? at.ends : 0;
        uint4 r[4];
        fetch<ZT, 4>(r, piece, tid, nt, true);
        float scale = 1.0f;
        if (E == 4 && KIND != ROW_COEF) { // terms, of the classes that were summed: a named one far above them would be the maximum of its thread's
            if (shift != 0.0f) take_far<ZT, 4>(r, piece, shift, a.c, out, tid, nt);
            else scale = ex2(rise(take<ZT, 4>(r, piece, a.c, out, tid, nt, false).m, a.c, o.M));
        } else if (shift != 0.0f) less<ZT, 4>(r, piece, shift, nullptr, tid, nt);
        give<ZT, KIND, 4>(a, piece, o, r, tid, nt, scale, code);
    }
    if (KIND == ROW_DISTILL) {
        __syncthreads();
        for (int j = tid; j < a.T; j += nt) if (s.id[j] >= 0) put_slot(a, at, o, s, j, flags & SLOT_TWICE, w);
    }
}

// Sums of the log ratios of the two sequences of a pair, its loss, and the factor of every row's gradient.  One CTA per pair; the last
// one clears the factors of rows outside of all sequences.
struct PairArgs {
    const uint32_t *label;
    const int32_t *seq;
    const float *logp, *ref, *w;
    float *loss, *margin, *coef;
    long long n;
    int P, mean;
    float beta, smooth;
};
__device__ __forceinline__ float softplus_(float x) { return fmaxf(x, 0.0f) + log1pf(expf(-fabsf(x))); }
__device__ __forceinline__ RowLoss pair_loss(float m, float w, float smooth) { // loss and its derivative by the margin
    return {w * ((1.0f - smooth) * softplus_(-m) + smooth * softplus_(m)), w * (smooth / (1.0f + expf(-m)) - (1.0f - smooth) / (1.0f + expf(m)))};
}
__global__ void __launch_bounds__(256) k_pairs(PairArgs a) {
    __shared__ double s_sum[8];
    __shared__ int s_cnt[8];
    const int tid = threadIdx.x, p = blockIdx.x;
    auto bound = [&](int s) { return min(max((long long)a.seq[s], 0ll), a.n); };
    if (p == a.P) {
        const long long b = bound(0), e = bound(2 * a.P);
        for (long long i = tid; i < b; i += 256) a.coef[i] = 0.0f;
        for (long long i = e + tid; i < a.n; i += 256) a.coef[i] = 0.0f;
        return;
    }
    double D[2], share[2];
    for (int s = 0; s < 2; ++s) {
        const long long b = bound(2 * p + s), e = bound(2 * p + s + 1);
        double v = 0.0;
        int cnt = 0;
        for (long long i = b + tid; i < e; i += 256)
            if (a.label[i]) { v += (double)a.logp[i] - (a.ref ? (double)a.ref[i] : 0.0); ++cnt; }
        v = warp_sum(v);
        cnt = __reduce_add_sync(FULL, cnt);
        __syncthreads();
        if ((tid & 31) == 0) { s_sum[tid >> 5] = v; s_cnt[tid >> 5] = cnt; }
        __syncthreads();
        v = 0.0; cnt = 0;
        for (int q = 0; q < 8; ++q) { v += s_sum[q]; cnt += s_cnt[q]; }
        share[s] = a.mean && cnt > 1 ? 1.0 / (double)cnt : 1.0;
        D[s] = v * share[s];
    }
    const float m = (float)((double)a.beta * (D[0] - D[1]));
    const RowLoss o = pair_loss(m, a.w ? a.w[p] : 1.0f, a.smooth);
    if (tid == 0) { a.loss[p] = a.w && a.w[p] == 0.0f ? 0.0f : o.loss; a.margin[p] = m; }
    for (int s = 0; s < 2; ++s) {
        const long long b = bound(2 * p + s), e = bound(2 * p + s + 1);
        const float f = a.w && a.w[p] == 0.0f ? 0.0f : (float)((s ? -1.0 : 1.0) * (double)o.d * (double)a.beta * share[s]);
        for (long long i = b + tid; i < e; i += 256) a.coef[i] = a.label[i] ? f : 0.0f;
    }
}

// What may be resident at a time, asked once for every shape of a kernel
constexpr int LANES_SMEM = 200 * 1024, WALK_SMEM = 160 * 1024, TILE_SMEM = 128 * 1024, TAUGHT_SMEM = 200 * 1024; // the attribute is set to the most a kernel is given: calls of several threads do not undo one another's
cudaError_t launch_cluster(void (*kern)(SoftArgs, int, int), long long rows, int threads, int lcs, size_t smem, cudaStream_t st, const SoftArgs &a, int words) {
    cudaLaunchConfig_t c = {};
    cudaLaunchAttribute at[1];
    c.gridDim = dim3((unsigned)(rows << lcs)); c.blockDim = dim3(threads); c.dynamicSmemBytes = smem; c.stream = st;
    if (lcs > 0) {
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim.x = 1 << lcs; at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
        c.attrs = at; c.numAttrs = 1;
    }
    return cudaLaunchKernelEx(&c, kern, a, lcs, words);
}
template <typename ZT, int KIND>
int32_t launch_typed(SoftArgs a, int sms, cudaStream_t st, void *work) {
    constexpr int E = Pack<ZT>::E;
    // granules of a row: of one that begins just before the end of its first one, unless all rows begin where a granule does
    const bool aligned = (uintptr_t)a.z % 16 == 0 && (a.ldz % E == 0 || a.n == 1);
    const int nvec = (a.K + (aligned ? 0 : E - 1) + E - 1) / E;
    const size_t slots = KIND == ROW_DISTILL ? (size_t)a.T * Slots::BYTES : 0;
    auto words_of = [&](int granules) { return KIND == ROW_DISTILL ? (granules * E + 31) / 32 : 0; };
    if constexpr (E == 4) {
        if (a.K >= 2 && a.K <= 8) {
            const size_t smem = 4 * (size_t)TILE * a.K * (a.h ? 2 : 1);
            auto go = [&](void (*kern)(SoftArgs)) { return evb_launch(kern, dim3((unsigned)((a.n + TILE - 1) / TILE)), dim3(TILE), smem, st, a); };
            switch (a.K) {
            case 2: EVB_CUDA(go(k_row_few<KIND, 2>)); break;
            case 3: EVB_CUDA(go(k_row_few<KIND, 3>)); break;
            case 4: EVB_CUDA(go(k_row_few<KIND, 4>)); break;
            case 5: EVB_CUDA(go(k_row_few<KIND, 5>)); break;
            case 6: EVB_CUDA(go(k_row_few<KIND, 6>)); break;
            case 7: EVB_CUDA(go(k_row_few<KIND, 7>)); break;
            default: EVB_CUDA(go(k_row_few<KIND, 8>));
            }
            return EVB_OK;
        }
    }
    if (a.K <= TILE_K && (KIND != ROW_DISTILL || a.T <= TILE_T)) {
        TileGeom ge;
        ge.Kp = a.K | 1; ge.Tp = a.T | 1;
        ge.by_K = (uint32_t)((0x100000000ull + a.K - 1) / a.K); // not used for 1
        ge.by_T = a.T > 0 ? (uint32_t)((0x100000000ull + a.T - 1) / a.T) : 0u;
        const size_t smem = 4 * (size_t)TILE * (ge.Kp * (a.h ? 2 : 1) + (KIND == ROW_DISTILL ? 4 * ge.Tp : 0));
        if (smem > 47 * 1024) EVB_CUDA(cudaFuncSetAttribute(k_row_tile<ZT, KIND>, cudaFuncAttributeMaxDynamicSharedMemorySize, TILE_SMEM));
        EVB_CUDA(evb_launch(k_row_tile<ZT, KIND>, dim3((unsigned)((a.n + TILE - 1) / TILE)), dim3(TILE), smem, st, a, ge));
        return EVB_OK;
    }
    if (nvec <= 256) { // within a warp
        int G = 1, V = 1;
        while (G < 32 && G * 8 < nvec) G *= 2;
        while (V * G < nvec) V *= 2;
        const int words = words_of(nvec);
        const size_t smem = (size_t)(256 / G) * (slots + words * 4);
        if (smem <= LANES_SMEM) {
            const unsigned grid = (unsigned)((a.n + 256 / G - 1) / (256 / G));
            auto go = [&](void (*kern)(SoftArgs, int, int)) {
                const cudaError_t e = smem > 47 * 1024 ? cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, LANES_SMEM) : cudaSuccess;
                return e != cudaSuccess ? e : evb_launch(kern, dim3(grid), dim3(256), smem, st, a, G, words);
            };
            EVB_CUDA(V <= 2 ? go(k_row_lanes<ZT, KIND, 2>) : V == 4 ? go(k_row_lanes<ZT, KIND, 4>) : go(k_row_lanes<ZT, KIND, 8>));
            return EVB_OK;
        }
    }
    int lcs = 0;
    auto per = [&] { return (nvec + (1 << lcs) - 1) >> lcs; };
    auto holds = [&](int threads, int V) { return per() <= threads * V + (threads - 2 * E) / E; }; // the last few as ends, an element a thread
    auto go = [&](void (*kern)(SoftArgs, int, int), int threads) {
        const size_t smem = a.taught ? 0 : slots + (KIND == ROW_DISTILL ? (size_t)table_places(a.T) * 4 : 0);
        return launch_cluster(kern, a.n, threads, lcs, smem + (size_t)words_of(per()) * 4, st, a, words_of(per()));
    };
    while (lcs < 3 && (a.n << (lcs + 1)) <= sms && per() > 256) ++lcs; // few rows: several SMs for each
    if (holds(1024, 2) && (a.n << lcs) <= 2 * sms) {
        EVB_CUDA(holds(256, 2) ? go(k_row_ctas<ZT, KIND, 2, 256>, 256) : go(k_row_ctas<ZT, KIND, 2, 1024>, 1024));
        return EVB_OK;
    }
    lcs = 0;
    while (lcs < 3 && !holds(256, 8)) ++lcs;
    // Above 131072 classes of 16 bits, 65536 of 32 bits, eight CTAs of 512 threads, two an SM.  Microseconds against k_row_walk, 1000 rows: policy 140001 bf16
    // 193 and 152, 200003 225 and 217, 262136 250 and 279, 131064 f32 218 and 275 (300 rows x 200003 bf16: 76 and 95), so of many rows the walk
    // is as good or better up to some 200000 classes of 16 bits.  It is also better without gradients (200003 bf16: 168 and 92) and with a tail (301 and 223)
    if (holds(512, 8) && (a.n << lcs) <= 0x7fffffff) {
        if constexpr (KIND == ROW_DISTILL) {
            if (work) {
                const size_t smem = 8 * (slots + (size_t)table_places(a.T) * 4);
                if (smem > 47 * 1024) EVB_CUDA(cudaFuncSetAttribute(k_row_taught<ZT>, cudaFuncAttributeMaxDynamicSharedMemorySize, TAUGHT_SMEM));
                EVB_CUDA(evb_launch(k_row_taught<ZT>, dim3((unsigned)((a.n + 7) / 8)), dim3(256), smem, st, a, static_cast<TaughtRow *>(work)));
                a.taught = static_cast<const TaughtRow *>(work);
                EVB_CUDA(holds(64, 8) ? go(k_row_ctas<ZT, KIND, 8, 64, true>, 64) : holds(128, 8) ? go(k_row_ctas<ZT, KIND, 8, 128, true>, 128)
                         : holds(256, 8) ? go(k_row_ctas<ZT, KIND, 8, 256, true>, 256) : go(k_row_ctas<ZT, KIND, 8, 512, true>, 512));
                return EVB_OK;
            }
        }
        if constexpr (KIND == ROW_LOGP || KIND == ROW_COEF) {
            // either pass of a preference on rows that several CTAs share: half the threads with twice the granules (4096 x 131072 bf16: 528 us
            // instead of 575; a policy, which does both, 220 instead of 217 at half the rows)
            if (lcs > 0) {
                const int before = lcs;
                lcs = 0;
                while (lcs < 3 && !holds(128, 16)) ++lcs;
                if (holds(128, 16)) { EVB_CUDA(go(k_row_ctas<ZT, KIND, 16, 128>, 128)); return EVB_OK; }
                lcs = before;
            }
        }
        EVB_CUDA(holds(64, 8) ? go(k_row_ctas<ZT, KIND, 8, 64>, 64) : holds(128, 8) ? go(k_row_ctas<ZT, KIND, 8, 128>, 128)
                 : holds(256, 8) ? go(k_row_ctas<ZT, KIND, 8, 256>, 256) : go(k_row_ctas<ZT, KIND, 8, 512>, 512));
        return EVB_OK;
    }
    const int words = words_of(nvec);
    const size_t smem = slots + words * 4;
    if (smem > 47 * 1024) EVB_CUDA(cudaFuncSetAttribute(k_row_walk<ZT, KIND>, cudaFuncAttributeMaxDynamicSharedMemorySize, WALK_SMEM));
    EVB_CUDA(evb_launch(k_row_walk<ZT, KIND>, dim3((unsigned)a.n), dim3(512), smem, st, a, words));
    return EVB_OK;
}
template <int KIND>
int32_t launch_rows(const SoftArgs &a, int dtype, int device, cudaStream_t st, void *work = nullptr) {
    static std::atomic<int> known[64]; // processors of a device, asked for once
    int sms = device < 64 ? known[device].load(std::memory_order_relaxed) : 0;
    if (sms == 0) {
        EVB_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device));
        if (device < 64) known[device].store(sms, std::memory_order_relaxed);
    }
    return dtype == EVB_BF16 ? launch_typed<__nv_bfloat16, KIND>(a, sms, st, work) : dtype == EVB_F16 ? launch_typed<__half, KIND>(a, sms, st, work)
                                                                                                : launch_typed<float, KIND>(a, sms, st, work);
}

// the calling thread's device is what it was when the call returns
struct OnDevice {
    int before = -1, now = -1;
    int32_t enter(const char *who, int32_t device) {
        static std::atomic<int> count{0};
        int ndev = count.load(std::memory_order_relaxed);
        const cudaError_t e = ndev > 0 ? cudaSuccess : cudaGetDeviceCount(&ndev);
        if (e == cudaSuccess) count.store(ndev, std::memory_order_relaxed);
        if (e != cudaSuccess || ndev == 0) {
            cudaGetLastError();
            evb_set_error("no CUDA device available (%s): this library has no CPU fallback", cudaGetErrorString(e));
            return EVB_ERR_CUDA;
        }
        if (device < 0 || device >= ndev) { evb_set_error("%s: device %d out of range", who, device); return EVB_ERR_ARG; }
        EVB_CUDA(cudaGetDevice(&before));
        now = device;
        if (before != now) EVB_CUDA(cudaSetDevice(now));
        return EVB_OK;
    }
    ~OnDevice() { if (before >= 0 && before != now) cudaSetDevice(before); }
};

bool known_dtype(int32_t d) { return d == EVB_F32 || d == EVB_BF16 || d == EVB_F16; }
int32_t check_rows(const char *who, const void *z, int32_t dtype, int64_t n, int32_t K, int64_t ldz, const void *g, int64_t ldg, const void *h, int64_t ldh) {
    if (!known_dtype(dtype)) { evb_set_error("%s: predictions must be EVB_F32, EVB_BF16 or EVB_F16", who); return EVB_ERR_ARG; }
    if (n < 0 || n > 2000000000ll || K < 1) { evb_set_error("%s: rows / classes out of range", who); return EVB_ERR_ARG; }
    if (K > MAX_CLASSES) { evb_set_error("%s: %d classes, the limit is %d", who, K, MAX_CLASSES); return EVB_ERR_LIMIT; }
    if (ldz < K || (g && ldg < K) || (h && ldh < K)) { evb_set_error("%s: a row stride is below the number of classes", who); return EVB_ERR_ARG; }
    const size_t es = dtype == EVB_F32 ? 4 : 2;
    if (((uintptr_t)z | (uintptr_t)g | (uintptr_t)h) % es) { evb_set_error("%s: misaligned pointer", who); return EVB_ERR_ARG; }
    if (n > 0 && !z) { evb_set_error("%s: null pointer", who); return EVB_ERR_ARG; }
    return EVB_OK;
}
SoftArgs rows_args(const void *z, int64_t n, int32_t K, int64_t ldz, const float *w, float tau, float *loss, void *g, int64_t ldg, void *h, int64_t ldh) {
    SoftArgs a = {};
    a.z = z; a.n = n; a.ldz = ldz; a.K = K;
    a.tau = tau; a.inv_tau = (float)(1.0 / (double)tau); a.c = (float)(1.4426950408889634074 / (double)tau);
    a.g = g; a.h = h; a.ldg = ldg; a.ldh = ldh; a.w = w; a.w_stride = 1; a.loss = loss;
    return a;
}
bool good_tau(double v) { return v >= 1.0e-6 && v <= 1.0e6; }

} // namespace

// ---------------------------------------------------------------------------------- as losses of a handle
namespace {
// Rows 2 p and 2 p + 1 of one output: the scores are log ratios already, less those of the reference
__global__ void __launch_bounds__(256) k_score_pairs(const float *pred, const float *ref, const float *w, long long w_stride, long long pairs, float beta, float smooth,
                                                     float *grad, int nq, float *loss) {
    const long long p = (long long)blockIdx.x * blockDim.x + threadIdx.x, i = 2 * p;
    if (p >= pairs) return;
    const float m = beta * ((pred[i] - ref[i]) - (pred[i + 1] - ref[i + 1])), wp = w ? w[i * w_stride] : 1.0f;
    const RowLoss o = pair_loss(m, wp, smooth);
    if (loss) loss[p] = o.loss;
    if (grad) {
        const float g = beta * o.d, h = wp * beta * beta / ((1.0f + expf(-m)) * (1.0f + expf(m)));
        grad[i * nq] = g; grad[i * nq + 1] = h;
        grad[(i + 1) * nq] = -g; grad[(i + 1) * nq + 1] = h;
    }
}
} // namespace

int32_t evb_check_objective(const evb_params *p, int64_t nobs, int32_t y_dtype, int32_t ycols) {
    const double *q = p->alphas;
    const bool pref = p->loss == EVB_PREFERENCE, dist = p->loss == EVB_DISTILL;
    if (pref ? p->K != 1 || y_dtype != EVB_F32 || ycols != 1 || nobs % 2 != 0 : p->K < 2 || y_dtype != EVB_U32 || (dist ? ycols < 2 || ycols % 2 != 0 || ycols > 2 * MAX_TOP : ycols != 4)) {
        evb_set_error("evb_create: K=%d / ycols=%d / y_dtype=%d / nobs=%lld inconsistent with the loss", p->K, ycols, y_dtype, (long long)nobs);
        return EVB_ERR_ARG;
    }
    const bool ok = pref ? q[0] >= 0.0 && q[0] <= 1.0e6 && q[1] >= 0.0 && q[1] <= 1.0
                  : dist ? good_tau(q[0]) && (q[1] == 0.0 || (q[1] == 1.0 && q[0] == 1.0))
                         : good_tau(q[0]) && q[1] >= 0.0 && q[1] <= 1.0 && q[2] >= 0.0 && q[2] <= 3.0e38 && q[3] >= 0.0 && q[3] <= 3.0e38;
    if (!ok) { evb_set_error("evb_create: parameters of the loss out of range (%g, %g, %g, %g)", q[0], q[1], q[2], q[3]); return EVB_ERR_ARG; }
    return EVB_OK;
}

int32_t evb_launch_objective(evb_handle *h, bool eval) {
    const double *q = h->p.alphas;
    const int64_t n = eval ? h->ev_n : h->n;
    const float *pred = eval ? h->ev_pred : h->pred, *w = eval ? h->ev_w : h->unit_w ? nullptr : h->grad + h->nq - 1;
    const void *y = eval ? h->ev_y : h->y;
    float *loss = eval ? h->ev_loss : nullptr, *grad = eval ? nullptr : h->grad;
    const long long ws = eval ? 1 : h->nq;
    if (h->objective == EVB_PREFERENCE) {
        k_score_pairs<<<(unsigned)((n / 2 + 255) / 256), 256, 0, h->st>>>(pred, static_cast<const float *>(y), w, ws, n / 2, (float)q[0], (float)q[1], grad, h->nq, loss);
        EVB_CUDA(cudaGetLastError());
        return EVB_OK;
    }
    SoftArgs a = rows_args(pred, n, h->K, h->K, w, (float)q[0], loss, grad, h->nq, grad ? grad + h->K : nullptr, h->nq);
    a.w_stride = ws;
    const uint32_t *words = static_cast<const uint32_t *>(y);
    if (h->objective == EVB_DISTILL) {
        a.T = h->ycols / 2; a.ldt = h->ycols; a.tail = q[1] != 0.0;
        a.ids = words; a.t = words + a.T; a.t_dtype = EVB_F32;
        return launch_rows<ROW_DISTILL>(a, EVB_F32, h->dev, h->st);
    }
    const float *f = reinterpret_cast<const float *>(words);
    a.code = words; a.p_stride = 4; a.old_lp = f + 1; a.adv = f + 2; a.ref = q[3] > 0.0 ? f + 3 : nullptr;
    a.lo = (float)q[1]; a.hi = (float)q[2]; a.beta = (float)q[3];
    return launch_rows<ROW_POLICY>(a, EVB_F32, h->dev, h->st);
}

extern "C" int32_t evb_distill_grads(int32_t device, void *stream, const void *z, int32_t dtype, int64_t n, int32_t K, int64_t ldz, const uint32_t *ids,
                                     const void *teacher, int32_t teacher_dtype, int32_t T, int32_t tail, const float *w, double tau, float *loss,
                                     void *grad, int64_t ldg, void *hess, int64_t ldh, void *work) {
    EVB_CHECK(check_rows("evb_distill_grads", z, dtype, n, K, ldz, grad, ldg, hess, ldh));
    if (T < 1 || !known_dtype(teacher_dtype)) { evb_set_error("evb_distill_grads: a row has at least one slot, of EVB_F32, EVB_BF16 or EVB_F16"); return EVB_ERR_ARG; }
    if (T > MAX_TOP) { evb_set_error("evb_distill_grads: %d slots, the limit is %d", T, MAX_TOP); return EVB_ERR_LIMIT; }
    if (!good_tau(tau) || (tail && tau != 1.0)) { evb_set_error("evb_distill_grads: tau must lie in [1e-6, 1e6], and be 1 with a tail (tau = %g)", tau); return EVB_ERR_ARG; }
    if (n > 0 && (!ids || !teacher)) { evb_set_error("evb_distill_grads: null pointer"); return EVB_ERR_ARG; }
    if ((uintptr_t)work % 16) { evb_set_error("evb_distill_grads: misaligned pointer"); return EVB_ERR_ARG; }
    OnDevice dev;
    EVB_CHECK(dev.enter("evb_distill_grads", device));
    if (n == 0) return EVB_OK;
    SoftArgs a = rows_args(z, n, K, ldz, w, (float)tau, loss, grad, ldg, hess, ldh);
    a.ids = ids; a.t = teacher; a.t_dtype = teacher_dtype; a.T = T; a.ldt = T; a.tail = tail != 0;
    return launch_rows<ROW_DISTILL>(a, dtype, device, (cudaStream_t)stream, work);
}

extern "C" int32_t evb_policy_grads(int32_t device, void *stream, const void *z, int32_t dtype, int64_t n, int32_t K, int64_t ldz, const uint32_t *action,
                                    const float *old_logp, const float *adv, const float *ref_logp, const float *w, double tau, double clip_low,
                                    double clip_high, double beta, float *loss, float *logp, void *grad, int64_t ldg, void *hess, int64_t ldh) {
    EVB_CHECK(check_rows("evb_policy_grads", z, dtype, n, K, ldz, grad, ldg, hess, ldh));
    if (!good_tau(tau)) { evb_set_error("evb_policy_grads: tau must lie in [1e-6, 1e6] (tau = %g)", tau); return EVB_ERR_ARG; }
    if (!(clip_low >= 0.0 && clip_low <= 1.0) || !(clip_high >= 0.0 && clip_high <= 3.0e38) || !(beta >= 0.0 && beta <= 3.0e38)) {
        evb_set_error("evb_policy_grads: the clip must be within [0, 1] below and at least 0 above, beta at least 0");
        return EVB_ERR_ARG;
    }
    if (n > 0 && (!action || !old_logp || !adv)) { evb_set_error("evb_policy_grads: null pointer"); return EVB_ERR_ARG; }
    OnDevice dev;
    EVB_CHECK(dev.enter("evb_policy_grads", device));
    if (n == 0) return EVB_OK;
    SoftArgs a = rows_args(z, n, K, ldz, w, (float)tau, loss, grad, ldg, hess, ldh);
    a.code = action; a.old_lp = old_logp; a.adv = adv; a.ref = ref_logp; a.p_stride = 1;
    a.lo = (float)clip_low; a.hi = (float)clip_high; a.beta = (float)beta; a.logp = logp;
    return launch_rows<ROW_POLICY>(a, dtype, device, (cudaStream_t)stream);
}

extern "C" int32_t evb_preference_grads(int32_t device, void *stream, const void *z, int32_t dtype, int64_t n, int32_t K, int64_t ldz, const uint32_t *label,
                                        const int32_t *seq, int32_t pairs, const float *ref_logp, const float *w, double beta, double smooth, int32_t mean,
                                        float *loss, float *margin, float *logp, void *grad, int64_t ldg, void *work) {
    EVB_CHECK(check_rows("evb_preference_grads", z, dtype, n, K, ldz, grad, ldg, nullptr, 0));
    if (pairs < 0 || pairs > 500000000) { evb_set_error("evb_preference_grads: number of pairs out of range"); return EVB_ERR_ARG; }
    if (!(beta >= 0.0 && beta <= 3.0e38) || !(smooth >= 0.0 && smooth <= 1.0)) {
        evb_set_error("evb_preference_grads: beta must be at least 0 and smooth within [0, 1]");
        return EVB_ERR_ARG;
    }
    if (!seq || (n > 0 && (!label || !logp || !work)) || (pairs > 0 && (!loss || !margin))) { evb_set_error("evb_preference_grads: null pointer"); return EVB_ERR_ARG; }
    if ((uintptr_t)work % 8) { evb_set_error("evb_preference_grads: misaligned pointer"); return EVB_ERR_ARG; }
    OnDevice dev;
    EVB_CHECK(dev.enter("evb_preference_grads", device));
    cudaStream_t st = (cudaStream_t)stream;
    SoftArgs a = rows_args(z, n, K, ldz, nullptr, 1.0f, nullptr, nullptr, 0, nullptr, 0);
    a.code = label; a.p_stride = 1; a.logp = logp;
    a.stat = static_cast<float2 *>(work);
    float *coef = reinterpret_cast<float *>(a.stat + n);
    if (n > 0) EVB_CHECK(launch_rows<ROW_LOGP>(a, dtype, device, st));
    PairArgs p;
    p.label = label; p.seq = seq; p.logp = logp; p.ref = ref_logp; p.w = w; p.loss = loss; p.margin = margin; p.coef = coef;
    p.n = n; p.P = pairs; p.mean = mean != 0; p.beta = (float)beta; p.smooth = (float)smooth;
    EVB_CUDA(evb_launch(k_pairs, dim3((unsigned)pairs + 1), dim3(256), 0, st, p));
    if (n == 0 || !grad) return EVB_OK;
    a.g = grad; a.ldg = ldg; a.coef = coef;
    return launch_rows<ROW_COEF>(a, dtype, device, st);
}
