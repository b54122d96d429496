// Losses on rows of raw predictions that a softmax turns into probabilities, with their gradients and hessians: distillation from a
// teacher's top logits, the clipped policy loss with a KL term, the preference loss of paired log ratios (formulas: include/evb.h).
//
// All three need the same of a row z[0 .. K-1]: its maximum and the sum of 2^(c (z_k - max)), c = log2(e) / tau, a few named columns,
// and then one number A so that g_k = A 2^(c (z_k - max)) everywhere but at the named columns, which are written after the others.
#include "evb_device.cuh"
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <algorithm>
#include <math.h>

namespace {

constexpr unsigned FULL = 0xffffffffu;
constexpr int MAX_TOP = 1024;        // slots of a row
constexpr int MAX_CLASSES = 1 << 20;

enum { ROW_DISTILL = 0, ROW_POLICY = 1, ROW_LOGP = 2, ROW_COEF = 3 };

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

// Maximum and sum of 2^(c (z - max)) of what has been seen.  The difference comes first: products c z of the type's lowest value, which masks
// often are made of, would be infinite
struct Soft { float m, s; };
__device__ __forceinline__ float base_of(float m) { return m == -INFINITY ? 0.0f : m; } // nothing but -inf: every term is 2^-inf
__device__ __forceinline__ float term(float z, float base, float c) { return exp2f((z - base) * c); }
__device__ __forceinline__ Soft join(Soft a, Soft b, float c) {
    const float m = fmaxf(a.m, b.m), base = base_of(m);
    return {m, a.s * term(a.m, base, c) + b.s * term(b.m, base, c)};
}

struct RowLoss { float loss, d; }; // loss and its derivative by log p of the class taken
__device__ __forceinline__ RowLoss policy_row(float lp, float old_lp, float adv, const float *ref, long long i, float lo, float hi, float beta) {
    const float r = expf(lp - old_lp), u = r * adv, cl = fminf(fmaxf(r, 1.0f - lo), 1.0f + hi) * adv;
    RowLoss o = {u <= cl ? -u : -cl, u <= cl ? -u : 0.0f};
    if (u != u) o = {u, u};
    if (ref) {
        const float x = ref[i] - lp, e = expm1f(x);
        o.loss += beta * (e - x);
        o.d -= beta * e;
    }
    return o;
}

// What the threads of a CTA find, joined in a fixed order: every thread gets it.  s_red: 33 floats
template <typename F>
__device__ __forceinline__ float block_all(float v, F f, float *s_red) {
    for (int o = 16; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(FULL, v, o));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s_red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = s_red[0];
    for (int q = 1; q < (int)(blockDim.x >> 5); ++q) v = f(v, s_red[q]);
    return v;
}
__device__ __forceinline__ float sum2(float a, float b) { return a + b; }

// One CTA walks over a row twice: maximum and sum, then gradient.
template <typename ZT, int KIND>
__global__ void __launch_bounds__(256) k_rows(SoftArgs a) {
    extern __shared__ __align__(16) unsigned char s_raw[];
    __shared__ float s_red[33];
    const int K = a.K, tid = threadIdx.x, nt = blockDim.x;
    const float c = a.c;
    // distillation: class (0-based, -1: none), probability, prediction of every slot; then a bit for every class that is named
    int *s_id = reinterpret_cast<int *>(s_raw);
    float *s_q = reinterpret_cast<float *>(s_id + a.T), *s_z = s_q + a.T;
    uint32_t *s_bits = reinterpret_cast<uint32_t *>(s_z + a.T);
    for (long long row = blockIdx.x; row < a.n; row += gridDim.x) {
        const ZT *z = static_cast<const ZT *>(a.z) + row * a.ldz;
        ZT *g = a.g ? static_cast<ZT *>(a.g) + row * a.ldg : nullptr, *h = a.h ? static_cast<ZT *>(a.h) + row * a.ldh : nullptr;
        float w = a.w ? a.w[row * a.w_stride] : 1.0f;
        bool live = w != 0.0f, bad = false;
        int code = -1;
        if (KIND == ROW_DISTILL) {
            bool some = false;
            __syncthreads();
            if (a.tail) for (int i = tid; i < (K + 31) / 32; i += nt) s_bits[i] = 0u;
            __syncthreads();
            for (int j = tid; j < a.T && live; j += nt) {
                const uint32_t id = a.ids[row * a.ldt + j];
                const float t = load_t(a.t, a.t_dtype, row * a.ldt + j);
                const bool use = id != 0u && t != -INFINITY, ok = id <= (uint32_t)K;
                some |= use; bad |= use && !ok;
                s_id[j] = use && ok ? (int)id - 1 : -1;
                s_q[j] = t;
                s_z[j] = use && ok ? to_f(z[id - 1]) : 0.0f;
                if (a.tail && use && ok) atomicOr(&s_bits[(id - 1) >> 5], 1u << ((id - 1) & 31));
            }
            live = __syncthreads_or(live && some);
            bad = __syncthreads_or(bad);
        } else {
            const uint32_t id = a.code[row * a.p_stride];
            if (KIND == ROW_COEF) w = a.coef[row];
            live = live && id != 0u && w != 0.0f;
            bad = live && id > (uint32_t)K;
            if (live && !bad) code = (int)id - 1;
        }
        if (!live || bad) { // a row that does not count; a class that there is not: NaN
            const float v = bad ? NAN : 0.0f;
            for (int k = tid; k < K; k += nt) { if (g) g[k] = from_f<ZT>(v); if (h) h[k] = from_f<ZT>(v); }
            if (tid == 0) {
                if (a.loss) a.loss[row] = v;
                if ((KIND == ROW_POLICY || KIND == ROW_LOGP) && a.logp) a.logp[row] = v;
                if (KIND == ROW_LOGP) a.stat[row] = make_float2(0.0f, v);
            }
            continue;
        }
        Soft r = {-INFINITY, 0.0f};
        if (KIND != ROW_COEF) {
            const bool tail = KIND == ROW_DISTILL && a.tail;
            for (int k = tid; k < K; k += nt) {
                if (tail && (s_bits[k >> 5] >> (k & 31) & 1u)) continue;
                r = join(r, Soft{to_f(z[k]), 1.0f}, c);
            }
            const float m = block_all(r.m, [](float x, float y) { return fmaxf(x, y); }, s_red), base = base_of(m);
            r.s = block_all(r.s * term(r.m, base, c), sum2, s_red);
            r.m = m;
        }
        float A, B; // g = A e, p = B e with e = 2^(c (z - max))
        if (KIND == ROW_DISTILL) {
            float tmax = -INFINITY, zmax = r.m, Q = 0.0f;
            for (int j = tid; j < a.T; j += nt) if (s_id[j] >= 0) { tmax = fmaxf(tmax, s_q[j]); zmax = fmaxf(zmax, s_z[j]); }
            tmax = block_all(tmax, [](float x, float y) { return fmaxf(x, y); }, s_red);
            zmax = block_all(zmax, [](float x, float y) { return fmaxf(x, y); }, s_red);
            // named classes, each of them once
            const float base = base_of(zmax);
            float s = 0.0f;
            for (int j = tid; j < a.T; j += nt) {
                if (s_id[j] < 0) continue;
                Q += a.tail ? expf(s_q[j]) : expf((s_q[j] - tmax) * a.inv_tau);
                bool first = true;
                for (int i = 0; i < j; ++i) first = first && s_id[i] != s_id[j];
                if (first) s += term(s_z[j], base, c);
            }
            Q = block_all(Q, sum2, s_red);
            s = block_all(s, sum2, s_red);
            const Soft all = a.tail ? Soft{zmax, s + r.s * term(r.m, base, c)} : r;
            const float ls = logf(all.s), lq = logf(Q);
            float loss = 0.0f;
            __syncthreads();
            for (int j = tid; j < a.T; j += nt) {
                if (s_id[j] < 0) continue;
                const float lt = a.tail ? s_q[j] : (s_q[j] - tmax) * a.inv_tau - lq, q = expf(lt);
                const float lp = (s_z[j] - all.m) * a.inv_tau - ls;
                s_q[j] = q;
                s_z[j] = lp;
                if (q != 0.0f) loss += q * (lt - lp);
            }
            float qt = 0.0f;
            if (a.tail && r.m != -INFINITY) qt = fmaxf(0.0f, 1.0f - Q);
            const float mass = a.tail ? Q + qt : 1.0f;
            loss = block_all(loss, sum2, s_red);
            if (qt > 0.0f) loss += qt * (logf(qt) - ((r.m - all.m) * a.inv_tau + logf(r.s) - ls));
            if (tid == 0 && a.loss) a.loss[row] = w * a.tau * a.tau * loss;
            B = r.m == -INFINITY ? 0.0f * ls : term(r.m, base_of(all.m), c) / all.s;
            A = w * a.tau * (mass * B - (qt > 0.0f ? qt / r.s : 0.0f));
            const float m1 = base_of(r.m);
            for (int k = tid; k < K && (g || h); k += nt) {
                const float e = term(to_f(z[k]), m1, c), p = e * B;
                if (g) g[k] = from_f<ZT>(e * A);
                if (h) h[k] = from_f<ZT>(w * p * (1.0f - p));
            }
            __syncthreads();
            for (int j = tid; j < a.T && (g || h); j += nt) {
                if (s_id[j] < 0) continue;
                bool first = true;
                for (int i = 0; i < j; ++i) first = first && s_id[i] != s_id[j];
                if (!first) continue;
                float q = 0.0f;
                for (int i = j; i < a.T; ++i) if (s_id[i] == s_id[j]) q += s_q[i];
                const float p = expf(s_z[j]);
                if (g) g[s_id[j]] = from_f<ZT>(w * a.tau * (mass * p - q));
                if (h) h[s_id[j]] = from_f<ZT>(w * p * (1.0f - p));
            }
        } else {
            const float za = to_f(z[code]);
            float lp, f; // f: factor of (delta - p)
            if (KIND == ROW_COEF) {
                const float2 st = a.stat[row];
                r.m = st.x;
                B = st.y;
                lp = a.logp[row];
                f = w;
            } else {
                lp = (za - r.m) * a.inv_tau - logf(r.s);
                B = 1.0f / r.s;
                f = 0.0f;
            }
            if (KIND == ROW_LOGP) {
                if (tid == 0) { a.logp[row] = lp; a.stat[row] = make_float2(r.m, B); }
                continue;
            }
            if (KIND == ROW_POLICY) {
                const long long i = row * a.p_stride;
                const RowLoss o = policy_row(lp, a.old_lp[i], a.adv[i], a.ref, i, a.lo, a.hi, a.beta);
                if (tid == 0) { if (a.loss) a.loss[row] = w * o.loss; if (a.logp) a.logp[row] = lp; }
                f = w * o.d * a.inv_tau;
            }
            A = -f * B;
            const float m1 = base_of(r.m), hw = w * a.inv_tau * a.inv_tau;
            for (int k = tid; k < K && (g || h); k += nt) {
                const float e = term(to_f(z[k]), m1, c), p = e * B;
                if (g) g[k] = k == code ? from_f<ZT>(-f * expm1f(lp)) : from_f<ZT>(e * A);
                if (h) h[k] = from_f<ZT>(hw * p * (1.0f - p));
            }
        }
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

template <int KIND>
int32_t launch_rows(const SoftArgs &a, int dtype, int device, cudaStream_t st) {
    int sms = 0;
    EVB_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device));
    const unsigned grid = (unsigned)std::min<long long>(a.n, (long long)sms * 8);
    const size_t smem = KIND == ROW_DISTILL ? (size_t)a.T * 12 + (a.tail ? ((size_t)a.K + 31) / 32 * 4 : 0) : 0;
    auto go = [&](void (*kern)(SoftArgs)) {
        cudaError_t e = smem > 48 * 1024 ? cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) : cudaSuccess;
        return e != cudaSuccess ? e : evb_launch(kern, dim3(grid), dim3(256), smem, st, a);
    };
    EVB_CUDA(dtype == EVB_BF16 ? go(k_rows<__nv_bfloat16, KIND>) : dtype == EVB_F16 ? go(k_rows<__half, KIND>) : go(k_rows<float, KIND>));
    return EVB_OK;
}

// the calling thread's device is what it was when the call returns
struct OnDevice {
    int before = -1, now = -1;
    int32_t enter(const char *who, int32_t device) {
        int ndev = 0;
        const cudaError_t e = cudaGetDeviceCount(&ndev);
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

extern "C" int32_t evb_distill_grads(int32_t device, void *stream, const void *z, int32_t dtype, int64_t n, int32_t K, int64_t ldz, const uint32_t *ids,
                                     const void *teacher, int32_t teacher_dtype, int32_t T, int32_t tail, const float *w, double tau, float *loss,
                                     void *grad, int64_t ldg, void *hess, int64_t ldh) {
    EVB_CHECK(check_rows("evb_distill_grads", z, dtype, n, K, ldz, grad, ldg, hess, ldh));
    if (T < 1 || !known_dtype(teacher_dtype)) { evb_set_error("evb_distill_grads: a row has at least one slot, of EVB_F32, EVB_BF16 or EVB_F16"); return EVB_ERR_ARG; }
    if (T > MAX_TOP) { evb_set_error("evb_distill_grads: %d slots, the limit is %d", T, MAX_TOP); return EVB_ERR_LIMIT; }
    if (!good_tau(tau) || (tail && tau != 1.0)) { evb_set_error("evb_distill_grads: tau must lie in [1e-6, 1e6], and be 1 with a tail (tau = %g)", tau); return EVB_ERR_ARG; }
    if (n > 0 && (!ids || !teacher)) { evb_set_error("evb_distill_grads: null pointer"); return EVB_ERR_ARG; }
    OnDevice dev;
    EVB_CHECK(dev.enter("evb_distill_grads", device));
    if (n == 0) return EVB_OK;
    SoftArgs a = rows_args(z, n, K, ldz, w, (float)tau, loss, grad, ldg, hess, ldh);
    a.ids = ids; a.t = teacher; a.t_dtype = teacher_dtype; a.T = T; a.ldt = T; a.tail = tail != 0;
    return launch_rows<ROW_DISTILL>(a, dtype, device, (cudaStream_t)stream);
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
