// K15: group norm with an activation, channels last, forward and backward.
//
// A (sample, group) is HW x Cg values (Cg = C / groups), N = HW * Cg of them:
//   mean = sum x / N;  var = sum (x - mean)^2 / N;  rstd = 1 / sqrt(var + eps);  xhat = (x - mean) * rstd
//   z = gamma[c] * xhat + beta[c];  y = act(z)
//   g = dy * act'(z);  dgamma[c] = sum g * xhat;  dbeta[c] = sum g  (over b, hw);  h = g * gamma[c]
//   dx = rstd * (h - sum h / N - xhat * sum (h * xhat) / N)
// Both directions are HBM-bound: 2 (forward) or 3 (backward) tensors moved, ~12 / ~25 operations an element.
//
// Two forms.  RESIDENT: a workgroup owns whole groups of one sample and keeps their values in registers between the sums
// and the store, so each tensor is moved once.  SPLIT, where a group does not fit a workgroup: per-channel sums over
// slices of HW, a small fold, and a second pass over the operands.
#include "common.h"

namespace {
using namespace cutie;

constexpr int GN_ACT_NONE = 0, GN_ACT_RELU = 1, GN_ACT_SIGMOID = 2, GN_ACT_SILU = 3;

template <int DT, int VEC> struct Pack {      // VEC consecutive elements as they lie in memory
    typedef typename elem<DT>::type T;
    typedef T V __attribute__((ext_vector_type(VEC)));
    V v;
    __device__ __forceinline__ void load(const T* p) { v = *reinterpret_cast<const V*>(p); }
    __device__ __forceinline__ float get(int e) const { T t = v[e]; return load_as_f32(&t); }
    __device__ __forceinline__ void set(int e, float f) { T t; store_from_f32(&t, f); v[e] = t; }
    __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<V*>(p) = v; }
};
template <int DT> struct Pack<DT, 1> {
    typedef typename elem<DT>::type T;
    T v;
    __device__ __forceinline__ void load(const T* p) { v = *p; }
    __device__ __forceinline__ float get(int) const { return load_as_f32(&v); }
    __device__ __forceinline__ void set(int, float f) { store_from_f32(&v, f); }
    __device__ __forceinline__ void store(T* p) const { *p = v; }
};

// 1 / (1 + exp(-z)).  f32: the library's expf and divide.  16-bit outputs take the hardware exponential and reciprocal
// (a few units of 2^-23): half a step of the output is 2^-11 (f16) or 2^-8 (bf16).
template <int DT> __device__ __forceinline__ float sigmoid_of(float z) {
    if constexpr (DT == CUTIE_F32) return 1.f / (1.f + expf(-z));
    else return __builtin_amdgcn_rcpf(1.f + __expf(-z));
}
template <int DT> __device__ __forceinline__ float act_of(float z, int act) {
    if (act == GN_ACT_RELU) return z < 0.f ? 0.f : z;      // NaN stays NaN
    if (act == GN_ACT_SIGMOID) return sigmoid_of<DT>(z);
    if (act == GN_ACT_SILU) return z * sigmoid_of<DT>(z);
    return z;
}

// act'(z) at z = gamma * xhat + beta.  The step of the ReLU is the one place where a rounding error of z is not a small
// error of the gradient: where |z| is within the f32 error of its own computation (d = x - mean, a product and a sum: at
// most 3 roundings, 2^-24 each, of |d * rg| + |beta|; 4e-7 > 3 * 2^-24) the sign is taken in f64.
template <int DT>
__device__ __forceinline__ float act_grad(float x, float mean, float rstd, float gamma, float beta, int act) {
    if (act == GN_ACT_NONE) return 1.f;
    const float d = x - mean, rg = rstd * gamma;
    const float z = fmaf(d, rg, beta);
    if (act == GN_ACT_RELU) {
        if (fabsf(z) <= 4e-7f * (fabsf(d * rg) + fabsf(beta))) {
            const double z64 = ((double)x - (double)mean) * (double)rstd * (double)gamma + (double)beta;
            return z64 > 0.0 ? 1.f : 0.f;
        }
        return z > 0.f ? 1.f : (z != z ? z : 0.f);
    }
    const float s = sigmoid_of<DT>(z);
    if (act == GN_ACT_SIGMOID) return s * (1.f - s);
    return s * (1.f + z * (1.f - s));
}

// ---------------------------------------------------------------------------------------------------------------- resident
struct GnShape {
    int HW, C, G, Cg;
    int gc;             // groups per workgroup
    int cv;             // vectors per pixel of a workgroup: gc * Cg / VEC
    int rows_par;       // pixels side by side: blockDim / cv
    int64_t items;      // B * G / gc
};

// Workgroups that share 128-byte lines (the groups of one pixel) go to one XCD: dispatch deals consecutive blocks to the
// eight XCDs in turn, so block i takes item (i % 8) * ceil(items / 8) + i / 8.
__device__ __forceinline__ int64_t xcd_item(int64_t items) {
    const int64_t per = (items + 7) / 8;
    return (int64_t)(blockIdx.x & 7) * per + (blockIdx.x >> 3);
}

// sum over the threads of each group: every thread leaves its value, wave w folds groups w, w + waves, ... in a fixed
// order, every thread takes its group's.  thread t's group is (t % cv) / (cv / gc).
__device__ __forceinline__ float group_sum(float v, float* sh, float* tot, int gc, int cv, int active, int my) {
    __syncthreads();
    sh[threadIdx.x] = v;
    __syncthreads();
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    const int vpg = cv / gc, n = active / gc;       // vectors of a group in a pixel; threads of a group
    for (int g = wave; g < gc; g += waves) {
        float s = 0.f;
        for (int i = lane; i < n; i += 64) {
            const int r = i / vpg;
            s += sh[r * cv + g * vpg + (i - r * vpg)];
        }
        s = wave_sum(s);
        if (lane == 0) tot[g] = s;
    }
    __syncthreads();
    return tot[my];
}

template <int DT, int VEC, int K>
__global__ __launch_bounds__(1024) void gn_fwd_resident(const typename elem<DT>::type* __restrict__ x, int ld_x,
                                                        const float* __restrict__ gamma, const float* __restrict__ beta, float eps,
                                                        int act, typename elem<DT>::type* __restrict__ y, int ld_y,
                                                        float* __restrict__ stats, GnShape s) {
    __shared__ float sh[1024];
    __shared__ float tot[1024];
    const int64_t item = xcd_item(s.items);
    if (item >= s.items) return;
    const int per = s.G / s.gc;
    const int64_t b = item / per;
    const int g0 = (int)(item - b * per) * s.gc;
    const int active = s.rows_par * s.cv;
    const bool on = (int)threadIdx.x < active;
    const int col = threadIdx.x % s.cv, row = threadIdx.x / s.cv;
    const int my = on ? col / (s.cv / s.gc) : 0;
    const int c0 = g0 * s.Cg + col * VEC;
    Pack<DT, VEC> d[K];
    const typename elem<DT>::type* px = x + (b * s.HW) * ld_x + c0;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int r = row + k * s.rows_par;
        if (on && r < s.HW) d[k].load(px + (int64_t)r * ld_x);
    }
    const float inv_n = 1.f / ((float)s.HW * (float)s.Cg);
    float a = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k)
        if (on && row + k * s.rows_par < s.HW) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) a += d[k].get(e);
        }
    const float mean0 = group_sum(a, sh, tot, s.gc, s.cv, active, my) * inv_n;
    // second moments about mean0, and what mean0 misses of the mean (its own rounding): d1
    float q1 = 0.f, q2 = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k)
        if (on && row + k * s.rows_par < s.HW) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) { const float t = d[k].get(e) - mean0; q1 += t; q2 = fmaf(t, t, q2); }
        }
    const float d1 = group_sum(q1, sh, tot, s.gc, s.cv, active, my) * inv_n;
    const float m2 = group_sum(q2, sh, tot, s.gc, s.cv, active, my) * inv_n;
    const float var = fmaxf(m2 - d1 * d1, 0.f) + (m2 - m2);      // + (m2 - m2): fmaxf drops a NaN, the group must keep it
    const float rstd = 1.f / sqrtf(var + eps);
    if (!on) return;
    if (row == 0 && col % (s.cv / s.gc) == 0) {
        float* st = stats + (b * s.G + g0 + my) * 2;
        st[0] = mean0 + d1;
        st[1] = rstd;
    }
    float rg[VEC], be[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        rg[e] = gamma ? rstd * gamma[c0 + e] : rstd;
        be[e] = fmaf(-d1, rg[e], beta ? beta[c0 + e] : 0.f);
    }
    typename elem<DT>::type* py = y + (b * s.HW) * ld_y + c0;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int r = row + k * s.rows_par;
        if (r < s.HW) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) d[k].set(e, act_of<DT>(fmaf(d[k].get(e) - mean0, rg[e], be[e]), act));
            d[k].store(py + (int64_t)r * ld_y);
        }
    }
}

// chan (nullable) f32 [B][C][2]: (sum g * xhat, sum g) of each sample and channel, folded over b by gn_fold_params
template <int DT, int VEC, int K>
__global__ __launch_bounds__(1024) void gn_bwd_resident(const typename elem<DT>::type* __restrict__ dy, int ld_dy,
                                                        const typename elem<DT>::type* __restrict__ x, int ld_x,
                                                        const float* __restrict__ gamma, const float* __restrict__ beta, int act,
                                                        const float* __restrict__ stats, typename elem<DT>::type* __restrict__ dx,
                                                        int ld_dx, float* __restrict__ chan, GnShape s) {
    extern __shared__ float part[];         // [2][blockDim][VEC] when chan is wanted
    __shared__ float sh[1024];
    __shared__ float tot[1024];
    const int64_t item = xcd_item(s.items);
    if (item >= s.items) return;
    const int per = s.G / s.gc;
    const int64_t b = item / per;
    const int g0 = (int)(item - b * per) * s.gc;
    const int active = s.rows_par * s.cv;
    const bool on = (int)threadIdx.x < active;
    const int col = threadIdx.x % s.cv, row = threadIdx.x / s.cv;
    const int my = on ? col / (s.cv / s.gc) : 0;
    const int c0 = g0 * s.Cg + col * VEC;
    Pack<DT, VEC> vx[K], vd[K];
    const typename elem<DT>::type* px = x + (b * s.HW) * ld_x + c0;
    const typename elem<DT>::type* pd = dy + (b * s.HW) * ld_dy + c0;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int r = row + k * s.rows_par;
        if (on && r < s.HW) {
            vx[k].load(px + (int64_t)r * ld_x);
            vd[k].load(pd + (int64_t)r * ld_dy);
        }
    }
    const float mean = stats[(b * s.G + g0 + my) * 2], rstd = stats[(b * s.G + g0 + my) * 2 + 1];
    float ga[VEC], be[VEC], sg[VEC], sx[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        ga[e] = on && gamma ? gamma[c0 + e] : 1.f;
        be[e] = on && beta ? beta[c0 + e] : 0.f;
        sg[e] = 0.f;
        sx[e] = 0.f;
    }
#pragma unroll
    for (int k = 0; k < K; ++k)
        if (on && row + k * s.rows_par < s.HW) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float xe = vx[k].get(e);
                const float g = vd[k].get(e) * act_grad<DT>(xe, mean, rstd, ga[e], be[e], act);
                sg[e] += g;
                sx[e] = fmaf(g, (xe - mean) * rstd, sx[e]);
            }
        }
    float h0 = 0.f, h1 = 0.f;
#pragma unroll
    for (int e = 0; e < VEC; ++e) { h0 = fmaf(sg[e], ga[e], h0); h1 = fmaf(sx[e], ga[e], h1); }
    const float inv_n = 1.f / ((float)s.HW * (float)s.Cg);
    const float s0 = group_sum(h0, sh, tot, s.gc, s.cv, active, my) * inv_n;
    const float s1 = group_sum(h1, sh, tot, s.gc, s.cv, active, my) * inv_n;
    if (chan) {
        float* p0 = part + threadIdx.x * VEC;
        float* p1 = p0 + blockDim.x * VEC;
#pragma unroll
        for (int e = 0; e < VEC; ++e) { p0[e] = sx[e]; p1[e] = sg[e]; }
        __syncthreads();
        const int n = s.cv * VEC;
        for (int i = threadIdx.x; i < 2 * n; i += blockDim.x) {
            const int k = i / n, c = i - k * n;
            const float* q = part + k * blockDim.x * VEC + c;
            float t = 0.f;
            for (int r = 0; r < s.rows_par; ++r) t += q[r * n];
            chan[(b * s.C + g0 * s.Cg + c) * 2 + k] = t;
        }
    }
    if (!on) return;
    typename elem<DT>::type* pq = dx + (b * s.HW) * ld_dx + c0;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int r = row + k * s.rows_par;
        if (r < s.HW) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float xe = vx[k].get(e);
                const float h = vd[k].get(e) * act_grad<DT>(xe, mean, rstd, ga[e], be[e], act) * ga[e];
                vd[k].set(e, rstd * (h - s0 - (xe - mean) * rstd * s1));
            }
            vd[k].store(pq + (int64_t)r * ld_dx);
        }
    }
}

// dgamma[c] (+)= sum_b chan[b][c][0], dbeta[c] (+)= sum_b chan[b][c][1]: a workgroup owns 8 values, 32 lanes each add
// every 32nd sample, the 32 sums are added in lane order
__global__ __launch_bounds__(256) void gn_fold_params(const float* __restrict__ chan, int B, int C, float* __restrict__ dgamma,
                                                      float* __restrict__ dbeta, int accumulate) {
    __shared__ float sh[32][8];
    const int el = threadIdx.x & 7, part = threadIdx.x >> 3;
    const int64_t i = (int64_t)blockIdx.x * 8 + el, n = (int64_t)C * 2;
    float t = 0.f;
    if (i < n)
        for (int b = part; b < B; b += 32) t += chan[b * n + i];
    sh[part][el] = t;
    __syncthreads();
    if (part || i >= n) return;
    t = 0.f;
#pragma unroll
    for (int k = 0; k < 32; ++k) t += sh[k][el];
    float* out = (i & 1) ? dbeta : dgamma;
    if (out) out[i >> 1] = accumulate ? out[i >> 1] + t : t;
}

// ------------------------------------------------------------------------------------------------------------------- split
// grid (T slices of HW, B, blocks of 256 vectors).  slots double [B][T][C][2].  The sums of the forward are f64: squares
// of the raw values, whatever the channel's level, and no shift to choose.
template <int VEC> struct SplitMap {
    int64_t b;
    int c0, row, rows_par, r0, r1, nv;
    bool on;
    __device__ SplitMap(int HW, int C) {
        const int v0 = blockIdx.z * 256;
        nv = min(256, C / VEC - v0);
        rows_par = 256 / nv;
        const int col = threadIdx.x % nv;
        row = threadIdx.x / nv;
        on = row < rows_par;
        b = blockIdx.y;
        c0 = (v0 + col) * VEC;
        const int per = (HW + gridDim.x - 1) / gridDim.x;
        r0 = min(HW, (int)blockIdx.x * per);
        r1 = min(HW, r0 + per);
    }
};

template <int VEC, typename R>
__device__ __forceinline__ void split_store(const R* a, const R* q, R (*red)[256 * VEC], const SplitMap<VEC>& m, int C, R* slots) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) { red[0][threadIdx.x * VEC + e] = a[e]; red[1][threadIdx.x * VEC + e] = q[e]; }
    __syncthreads();
    const int n = m.nv * VEC;
    R* out = slots + ((m.b * gridDim.x + blockIdx.x) * C + (int64_t)blockIdx.z * 256 * VEC) * 2;
    for (int i = threadIdx.x; i < 2 * n; i += 256) {
        const int k = i / n, c = i - k * n;
        R t = 0;
        for (int r = 0; r < m.rows_par; ++r) t += red[k][r * n + c];
        out[c * 2 + k] = t;
    }
}

template <int DT, int VEC>
__global__ __launch_bounds__(256) void gn_fwd_partial(const typename elem<DT>::type* __restrict__ x, int ld_x, int HW, int C,
                                                      double* __restrict__ slots) {
    __shared__ double red[2][256 * VEC];
    const SplitMap<VEC> m(HW, C);
    double a[VEC] = {}, q[VEC] = {};
    if (m.on)
#pragma unroll 4
        for (int r = m.r0 + m.row; r < m.r1; r += m.rows_par) {
            Pack<DT, VEC> v;
            v.load(x + (m.b * HW + r) * ld_x + m.c0);
#pragma unroll
            for (int e = 0; e < VEC; ++e) { const double t = v.get(e); a[e] += t; q[e] = fma(t, t, q[e]); }
        }
    split_store<VEC>(a, q, red, m, C, slots);
}

// one workgroup per (group, sample): stats, and in `low` what the f32 mean misses
__global__ __launch_bounds__(256) void gn_fwd_fold(const double* __restrict__ slots, int T, int HW, int C, int G, float eps,
                                                   float* __restrict__ stats, float* __restrict__ low) {
    __shared__ double red[2][256];
    const int Cg = C / G, g = blockIdx.x;
    const int64_t b = blockIdx.y;
    double a = 0, q = 0;
    const int64_t n = (int64_t)T * Cg;
    for (int64_t i = threadIdx.x; i < n; i += 256) {
        const int64_t t = i / Cg;
        const double2 v = *reinterpret_cast<const double2*>(slots + ((b * T + t) * C + g * Cg + (i - t * Cg)) * 2);
        a += v.x;
        q += v.y;
    }
    red[0][threadIdx.x] = a;
    red[1][threadIdx.x] = q;
    __syncthreads();
    for (int o = 128; o > 0; o >>= 1) {
        if ((int)threadIdx.x < o) {
            red[0][threadIdx.x] += red[0][threadIdx.x + o];
            red[1][threadIdx.x] += red[1][threadIdx.x + o];
        }
        __syncthreads();
    }
    if (threadIdx.x) return;
    const double N = (double)HW * Cg, mean = red[0][0] / N;
    double var = red[1][0] / N - mean * mean;
    if (var < 0) var = 0;
    stats[(b * G + g) * 2] = (float)mean;
    stats[(b * G + g) * 2 + 1] = (float)(1.0 / sqrt(var + (double)eps));
    low[b * G + g] = (float)(mean - (double)(float)mean);
}

template <int DT, int VEC>
__global__ __launch_bounds__(256) void gn_fwd_apply(const typename elem<DT>::type* __restrict__ x, int ld_x,
                                                    const float* __restrict__ gamma, const float* __restrict__ beta,
                                                    const float* __restrict__ stats, const float* __restrict__ low, int act,
                                                    typename elem<DT>::type* __restrict__ y, int ld_y, int HW, int C, int G) {
    const SplitMap<VEC> m(HW, C);
    if (!m.on) return;
    const int Cg = C / G;
    float mean[VEC], rg[VEC], be[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        const int64_t g = m.b * G + (m.c0 + e) / Cg;
        mean[e] = stats[g * 2];
        rg[e] = stats[g * 2 + 1] * (gamma ? gamma[m.c0 + e] : 1.f);
        be[e] = fmaf(-low[g], rg[e], beta ? beta[m.c0 + e] : 0.f);
    }
#pragma unroll 4
    for (int r = m.r0 + m.row; r < m.r1; r += m.rows_par) {
        Pack<DT, VEC> v;
        v.load(x + (m.b * HW + r) * ld_x + m.c0);
#pragma unroll
        for (int e = 0; e < VEC; ++e) v.set(e, act_of<DT>(fmaf(v.get(e) - mean[e], rg[e], be[e]), act));
        v.store(y + (m.b * HW + r) * ld_y + m.c0);
    }
}

template <int DT, int VEC>
__global__ __launch_bounds__(256) void gn_bwd_partial(const typename elem<DT>::type* __restrict__ dy, int ld_dy,
                                                      const typename elem<DT>::type* __restrict__ x, int ld_x,
                                                      const float* __restrict__ gamma, const float* __restrict__ beta,
                                                      const float* __restrict__ stats, int act, int HW, int C, int G,
                                                      float* __restrict__ slots) {
    __shared__ float red[2][256 * VEC];
    const SplitMap<VEC> m(HW, C);
    const int Cg = C / G;
    float sx[VEC] = {}, sg[VEC] = {};
    if (m.on) {
        float mean[VEC], rstd[VEC], ga[VEC], be[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const int64_t g = m.b * G + (m.c0 + e) / Cg;
            mean[e] = stats[g * 2];
            rstd[e] = stats[g * 2 + 1];
            ga[e] = gamma ? gamma[m.c0 + e] : 1.f;
            be[e] = beta ? beta[m.c0 + e] : 0.f;
        }
#pragma unroll 2
        for (int r = m.r0 + m.row; r < m.r1; r += m.rows_par) {
            Pack<DT, VEC> vx, vd;
            vx.load(x + (m.b * HW + r) * ld_x + m.c0);
            vd.load(dy + (m.b * HW + r) * ld_dy + m.c0);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float xe = vx.get(e);
                const float g = vd.get(e) * act_grad<DT>(xe, mean[e], rstd[e], ga[e], be[e], act);
                sg[e] += g;
                sx[e] = fmaf(g, (xe - mean[e]) * rstd[e], sx[e]);
            }
        }
    }
    split_store<VEC>(sx, sg, red, m, C, slots);
}

// one workgroup per (group, sample): chan[b][c][2] = the channel's sums over its slots (in slot order), and
// grp[b][g][2] = (mean of h, mean of h * xhat)
__global__ __launch_bounds__(256) void gn_bwd_fold(const float* __restrict__ slots, int T, int HW, int C, int G,
                                                   const float* __restrict__ gamma, float* __restrict__ chan, float* __restrict__ grp) {
    __shared__ float red[2][256];
    const int Cg = C / G, g = blockIdx.x;
    const int64_t b = blockIdx.y;
    float h0 = 0.f, h1 = 0.f;
    for (int c = threadIdx.x; c < Cg; c += 256) {
        const int cc = g * Cg + c;
        float a = 0.f, q = 0.f;
#pragma unroll 8
        for (int t = 0; t < T; ++t) {
            const float2 v = *reinterpret_cast<const float2*>(slots + ((b * T + t) * C + cc) * 2);
            a += v.x;
            q += v.y;
        }
        chan[(b * C + cc) * 2] = a;
        chan[(b * C + cc) * 2 + 1] = q;
        const float ga = gamma ? gamma[cc] : 1.f;
        h1 = fmaf(a, ga, h1);
        h0 = fmaf(q, ga, h0);
    }
    red[0][threadIdx.x] = h0;
    red[1][threadIdx.x] = h1;
    __syncthreads();
    for (int o = 128; o > 0; o >>= 1) {
        if ((int)threadIdx.x < o) {
            red[0][threadIdx.x] += red[0][threadIdx.x + o];
            red[1][threadIdx.x] += red[1][threadIdx.x + o];
        }
        __syncthreads();
    }
    if (threadIdx.x) return;
    const float inv_n = 1.f / ((float)HW * (float)Cg);
    grp[(b * G + g) * 2] = red[0][0] * inv_n;
    grp[(b * G + g) * 2 + 1] = red[1][0] * inv_n;
}

template <int DT, int VEC>
__global__ __launch_bounds__(256) void gn_bwd_apply(const typename elem<DT>::type* __restrict__ dy, int ld_dy,
                                                    const typename elem<DT>::type* __restrict__ x, int ld_x,
                                                    const float* __restrict__ gamma, const float* __restrict__ beta,
                                                    const float* __restrict__ stats, const float* __restrict__ grp, int act,
                                                    typename elem<DT>::type* __restrict__ dx, int ld_dx, int HW, int C, int G) {
    const SplitMap<VEC> m(HW, C);
    if (!m.on) return;
    const int Cg = C / G;
    float mean[VEC], rstd[VEC], ga[VEC], be[VEC], s0[VEC], s1[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        const int64_t g = m.b * G + (m.c0 + e) / Cg;
        mean[e] = stats[g * 2];
        rstd[e] = stats[g * 2 + 1];
        s0[e] = grp[g * 2];
        s1[e] = grp[g * 2 + 1];
        ga[e] = gamma ? gamma[m.c0 + e] : 1.f;
        be[e] = beta ? beta[m.c0 + e] : 0.f;
    }
#pragma unroll 2
    for (int r = m.r0 + m.row; r < m.r1; r += m.rows_par) {
        Pack<DT, VEC> vx, vd;
        vx.load(x + (m.b * HW + r) * ld_x + m.c0);
        vd.load(dy + (m.b * HW + r) * ld_dy + m.c0);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const float xe = vx.get(e);
            const float h = vd.get(e) * act_grad<DT>(xe, mean[e], rstd[e], ga[e], be[e], act) * ga[e];
            vd.set(e, rstd[e] * (h - s0[e] - (xe - mean[e]) * rstd[e] * s1[e]));
        }
        vd.store(dx + (m.b * HW + r) * ld_dx + m.c0);
    }
}

// ------------------------------------------------------------------------------------------------------------------- host
inline int elem_bytes(int dt) { return dt == CUTIE_F32 ? 4 : 2; }

// slices of HW a sample is cut into in the split form: enough workgroups for the chip, at least 32 pixels each
inline int gn_slices(int B, int HW, int C) {
    int64_t t = cdiv(2048, (int64_t)B * cdiv(C, 1024));
    const int64_t most = cdiv(HW, 32);
    if (t > most) t = most;
    if (t > 256) t = 256;
    return t < 1 ? 1 : (int)t;
}

// The widest vector that all views allow: base addresses and row strides must be multiples of it, and it must divide
// `run`, the number of consecutive channels it may not cross.
inline int gn_vec(int dt, int run, const void* const* ptrs, const int* lds, int n) {
    const int es = elem_bytes(dt);
    for (int v = 16 / es; v > 1; v >>= 1) {
        if (v == 2 && es == 2) break;       // 4-byte vectors are not built: 16, 8 (16-bit types) bytes, or single elements
        if (v == 2 && es == 4) break;
        bool ok = run % v == 0;
        for (int i = 0; i < n && ok; ++i)
            ok = (reinterpret_cast<uintptr_t>(ptrs[i]) % (uintptr_t)(v * es)) == 0 && lds[i] % v == 0;
        if (ok) return v;
    }
    return 1;
}

struct GnPlan { bool resident; int threads, K; GnShape s; };

// vectors of `vec` elements a thread may hold per tensor
inline GnPlan gn_plan(int B, int HW, int C, int G, int dt, int vec, int kmax) {
    GnPlan p = {};
    const int Cg = C / G, es = elem_bytes(dt);
    p.s.HW = HW; p.s.C = C; p.s.G = G; p.s.Cg = Cg;
    int gc = 0;
    for (int d = 1; d <= G; ++d) {
        if (G % d) continue;
        const int64_t cv = (int64_t)d * Cg / vec;
        if (cv > 1024) break;
        if (cdiv(HW, 1024 / cv) > kmax) break;                                          // does not fit the registers
        if (gc && (int64_t)gc * Cg * es >= 64 && (int64_t)gc * Cg * es * HW >= 8192) break;   // wide enough already
        if (gc && (int64_t)B * G / d < 256) break;                                       // keep a workgroup per CU
        gc = d;
    }
    if (!gc) return p;
    const int64_t cv = (int64_t)gc * Cg / vec;
    int64_t t = cdiv(cdiv((int64_t)HW * cv, 4), 64) * 64;      // about four vectors a thread
    if (t > 1024) t = 1024;
    if (t < cv) t = cdiv(cv, 64) * 64;
    if (t < 64) t = 64;
    p.threads = (int)t;
    p.s.gc = gc;
    p.s.cv = (int)cv;
    p.s.rows_par = (int)(t / cv);
    p.s.items = (int64_t)B * (G / gc);
    p.K = (int)cdiv(HW, p.s.rows_par);
    p.resident = p.K <= kmax && p.s.items <= (1 << 30);
    return p;
}

// (vec, element type) -> kernel instance
#define GN_VECS(DT, vec, VEC, ...)                                            \
    if constexpr (DT == CUTIE_F32) {                                          \
        if (vec == 4) { constexpr int VEC = 4; __VA_ARGS__; }                 \
        else { constexpr int VEC = 1; __VA_ARGS__; }                          \
    } else {                                                                  \
        if (vec == 8) { constexpr int VEC = 8; __VA_ARGS__; }                 \
        else if (vec == 4) { constexpr int VEC = 4; __VA_ARGS__; }            \
        else { constexpr int VEC = 1; __VA_ARGS__; }                          \
    }

constexpr int GN_FWD_KMAX = 16, GN_BWD_KMAX = 8;

struct GnSpace { size_t slots, low, chan, grp, total; };
inline GnSpace gn_space(int B, int HW, int C, int G) {
    GnSpace w;
    const size_t T = (size_t)gn_slices(B, HW, C), BC = (size_t)B * C, BG = (size_t)B * G;
    auto up = [](size_t n) { return (n + 255) / 256 * 256; };
    w.slots = 0;
    w.low = up(BC * T * 2 * sizeof(double));
    w.chan = w.low + up(BG * sizeof(float));
    w.grp = w.chan + up(BC * 2 * sizeof(float));
    w.total = w.grp + up(BG * 2 * sizeof(float));
    return w;
}

inline int gn_check(const char* who, int B, int HW, int C, int G, int act, int dt) {
    CUTIE_CHECK_ARG(B >= 0 && HW >= 0 && C >= 1 && G >= 1 && C % G == 0, "%s: B=%d HW=%d C=%d groups=%d (groups must divide C)", who, B,
                    HW, C, G);
    CUTIE_CHECK_ARG(B <= 65535 && G <= 65535 && C <= 65535, "%s: B=%d, groups=%d, C=%d (at most 65535 each)", who, B, G, C);
    CUTIE_CHECK_ARG(act >= GN_ACT_NONE && act <= GN_ACT_SILU, "%s: activation code %d (0 none, 1 ReLU, 2 sigmoid, 3 SiLU)", who, act);
    CUTIE_CHECK_ARG(dt == CUTIE_F32 || dt == CUTIE_BF16 || dt == CUTIE_F16, "%s: unknown dtype %d", who, dt);
    return CUTIE_OK;
}
}  // namespace

extern "C" size_t cutie_gn_workspace_bytes(int B, int HW, int C, int groups) {
    if (B < 1 || HW < 0 || C < 1 || groups < 1 || C % groups) return 0;
    return gn_space(B, HW < 1 ? 1 : HW, C, groups).total;
}

extern "C" int cutie_gn_fwd(const void* x, int ld_x, const float* gamma, const float* beta, int groups, float eps, int act, void* y,
                            int ld_y, int dtype, float* stats, int B, int HW, int C, void* workspace, size_t workspace_bytes,
                            cutie_stream_t stream_) {
    hipStream_t stream = (hipStream_t)stream_;
    if (int e = gn_check("gn_fwd", B, HW, C, groups, act, dtype)) return e;
    CUTIE_CHECK_ARG(ld_x >= C && ld_y >= C, "gn_fwd: ld_x=%d ld_y=%d must be >= C=%d", ld_x, ld_y, C);
    CUTIE_CHECK_ARG(eps > 0.f, "gn_fwd: eps=%g must be positive", (double)eps);
    if (B == 0 || HW == 0) return CUTIE_OK;
    CUTIE_CHECK_ARG(x && y && stats, "gn_fwd: null pointer");
    CUTIE_CHECK_ARG(x != y, "gn_fwd: y must not be x");
    CUTIE_CHECK_ARG(reinterpret_cast<uintptr_t>(x) % elem_bytes(dtype) == 0 && reinterpret_cast<uintptr_t>(y) % elem_bytes(dtype) == 0,
                    "gn_fwd: misaligned pointers");
    const void* ptrs[2] = {x, y};
    const int lds[2] = {ld_x, ld_y};
    const int vec = gn_vec(dtype, C / groups, ptrs, lds, 2);
    const GnPlan p = gn_plan(B, HW, C, groups, dtype, vec, GN_FWD_KMAX);
    if (p.resident) {
        const dim3 grid((unsigned)(cdiv(p.s.items, 8) * 8));
        CUTIE_DISPATCH_DTYPE(dtype, DT, {
            typedef typename elem<DT>::type E;
            GN_VECS(DT, vec, VEC, {
                auto go = [&](auto kern) {
                    hipLaunchKernelGGL(kern, grid, dim3(p.threads), 0, stream, (const E*)x, ld_x, gamma, beta, eps, act, (E*)y, ld_y,
                                       stats, p.s);
                };
                if (p.K <= 4) go(gn_fwd_resident<DT, VEC, 4>);
                else if (p.K <= 8) go(gn_fwd_resident<DT, VEC, 8>);
                else go(gn_fwd_resident<DT, VEC, 16>);
            })
        });
        CUTIE_CHECK_LAUNCH();
        return CUTIE_OK;
    }
    const GnSpace w = gn_space(B, HW, C, groups);
    if (!workspace || workspace_bytes < w.total || !aligned16(workspace)) {
        set_error("gn_fwd: workspace %zu < %zu (or not 16-byte aligned)", workspace ? workspace_bytes : 0, w.total);
        return CUTIE_E_WORKSPACE;
    }
    char* ws = (char*)workspace;
    double* slots = (double*)(ws + w.slots);
    float* low = (float*)(ws + w.low);
    const int sv = gn_vec(dtype, C, ptrs, lds, 2), T = gn_slices(B, HW, C);
    const dim3 grid((unsigned)T, (unsigned)B, (unsigned)cdiv(C / sv, 256));
    CUTIE_DISPATCH_DTYPE(dtype, DT, {
        typedef typename elem<DT>::type E;
        GN_VECS(DT, sv, VEC, {
            hipLaunchKernelGGL((gn_fwd_partial<DT, VEC>), grid, dim3(256), 0, stream, (const E*)x, ld_x, HW, C, slots);
            hipLaunchKernelGGL(gn_fwd_fold, dim3((unsigned)groups, (unsigned)B), dim3(256), 0, stream, slots, T, HW, C, groups, eps, stats,
                               low);
            hipLaunchKernelGGL((gn_fwd_apply<DT, VEC>), grid, dim3(256), 0, stream, (const E*)x, ld_x, gamma, beta, stats, low, act, (E*)y,
                               ld_y, HW, C, groups);
        })
    });
    CUTIE_CHECK_LAUNCH();
    return CUTIE_OK;
}

extern "C" int cutie_gn_bwd(const void* dy, int ld_dy, const void* x, int ld_x, const float* gamma, const float* beta, int groups,
                            int act, const float* stats, void* dx, int ld_dx, int dtype, float* dgamma, float* dbeta, int accumulate,
                            int B, int HW, int C, void* workspace, size_t workspace_bytes, cutie_stream_t stream_) {
    hipStream_t stream = (hipStream_t)stream_;
    if (int e = gn_check("gn_bwd", B, HW, C, groups, act, dtype)) return e;
    CUTIE_CHECK_ARG(ld_x >= C && ld_dy >= C && ld_dx >= C, "gn_bwd: ld_dy=%d ld_x=%d ld_dx=%d must be >= C=%d", ld_dy, ld_x, ld_dx, C);
    const bool none = B == 0 || HW == 0;
    CUTIE_CHECK_ARG(none || (dy && x && stats && dx), "gn_bwd: null pointer");
    CUTIE_CHECK_ARG(none || (dx != dy && dx != x), "gn_bwd: dx must be neither dy nor x");
    const int es = elem_bytes(dtype);
    CUTIE_CHECK_ARG(reinterpret_cast<uintptr_t>(x) % es == 0 && reinterpret_cast<uintptr_t>(dy) % es == 0 &&
                        reinterpret_cast<uintptr_t>(dx) % es == 0, "gn_bwd: misaligned pointers");
    const bool params = dgamma || dbeta;
    const GnSpace w = gn_space(B < 1 ? 1 : B, HW < 1 ? 1 : HW, C, groups);
    if (!none && (!workspace || workspace_bytes < w.total || !aligned16(workspace))) {
        set_error("gn_bwd: workspace %zu < %zu (or not 16-byte aligned)", workspace ? workspace_bytes : 0, w.total);
        return CUTIE_E_WORKSPACE;
    }
    char* ws = (char*)workspace;
    float* chan = ws ? (float*)(ws + w.chan) : nullptr;
    if (!none) {
        const void* ptrs[3] = {dy, x, dx};
        const int lds[3] = {ld_dy, ld_x, ld_dx};
        const int vec = gn_vec(dtype, C / groups, ptrs, lds, 3);
        const GnPlan p = gn_plan(B, HW, C, groups, dtype, vec, GN_BWD_KMAX);
        if (p.resident) {
            const dim3 grid((unsigned)(cdiv(p.s.items, 8) * 8));
            const size_t lds_bytes = params ? (size_t)2 * p.threads * vec * sizeof(float) : 0;
            CUTIE_DISPATCH_DTYPE(dtype, DT, {
                typedef typename elem<DT>::type E;
                GN_VECS(DT, vec, VEC, {
                    int rc = CUTIE_OK;
                    auto go = [&](auto kern) {
                        if (lds_bytes) rc = ensure_dyn_lds((const void*)kern, (int)lds_bytes);
                        if (rc == CUTIE_OK)
                            hipLaunchKernelGGL(kern, grid, dim3(p.threads), lds_bytes, stream, (const E*)dy, ld_dy, (const E*)x, ld_x,
                                               gamma, beta, act, stats, (E*)dx, ld_dx, params ? chan : nullptr, p.s);
                    };
                    if (p.K <= 4) go(gn_bwd_resident<DT, VEC, 4>);
                    else go(gn_bwd_resident<DT, VEC, 8>);
                    if (rc != CUTIE_OK) return rc;
                })
            });
            CUTIE_CHECK_LAUNCH();
        } else {
            float* slots = (float*)(ws + w.slots);
            float* grp = (float*)(ws + w.grp);
            const int sv = gn_vec(dtype, C, ptrs, lds, 3), T = gn_slices(B, HW, C);
            const dim3 grid((unsigned)T, (unsigned)B, (unsigned)cdiv(C / sv, 256));
            CUTIE_DISPATCH_DTYPE(dtype, DT, {
                typedef typename elem<DT>::type E;
                GN_VECS(DT, sv, VEC, {
                    hipLaunchKernelGGL((gn_bwd_partial<DT, VEC>), grid, dim3(256), 0, stream, (const E*)dy, ld_dy, (const E*)x, ld_x, gamma,
                                       beta, stats, act, HW, C, groups, slots);
                    hipLaunchKernelGGL(gn_bwd_fold, dim3((unsigned)groups, (unsigned)B), dim3(256), 0, stream, slots, T, HW, C, groups,
                                       gamma, chan, grp);
                    hipLaunchKernelGGL((gn_bwd_apply<DT, VEC>), grid, dim3(256), 0, stream, (const E*)dy, ld_dy, (const E*)x, ld_x, gamma,
                                       beta, stats, grp, act, (E*)dx, ld_dx, HW, C, groups);
                })
            });
            CUTIE_CHECK_LAUNCH();
        }
    }
    if (params && !(none && accumulate)) {
        hipLaunchKernelGGL(gn_fold_params, dim3((unsigned)cdiv((int64_t)C * 2, 8)), dim3(256), 0, stream, chan, none ? 0 : B, C, dgamma,
                           dbeta, accumulate);
        CUTIE_CHECK_LAUNCH();
    }
    return CUTIE_OK;
}
