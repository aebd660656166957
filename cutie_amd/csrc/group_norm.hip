// K15: group norm with an activation, channels last, forward and backward.
//
// A (sample, group) is HW x Cg values (Cg = C / groups), N = HW * Cg of them:
//   mean = sum x / N;  var = sum (x - mean)^2 / N;  rstd = 1 / sqrt(var + eps);  xhat = (x - mean) * rstd
//   z = gamma[c] * xhat + beta[c];  y = act(z)
//   g = dy * act'(z);  dgamma[c] = sum g * xhat;  dbeta[c] = sum g  (over b, hw);  h = g * gamma[c]
//   dx = rstd * (h - sum h / N - xhat * sum (h * xhat) / N)
// Both directions are HBM-bound: 2 (forward) or 3 (backward) tensors moved, ~12 / ~25 operations an element.
//
// Two forms.  RESIDENT: a workgroup owns whole groups of one sample and keeps their values in registers (and LDS) between the
// sums and the store, so each tensor is moved once.  SPLIT, where a group does not fit a workgroup, or where the pieces of a
// pixel are so narrow or the groups so few that it takes longer (gn_resident_us): per-channel sums over slices of HW, a small
// fold, and a second pass over the operands.
//
// Measured (MI355X), 32 x 64 x 64 x 256, 32 groups (134 MB forward, 201 MB backward), inputs that change from call to call: forward
// f16 33 us resident (4.1 TB/s), backward bf16 SiLU 73 us + 5 us fold (2.6 TB/s).  The same inputs again, partly in cache: 32 and
// 54 us with the fold, f32 61 and 136 (268 and 403 MB); split form 50 and 86.  What decides is the width of the piece of a pixel
// that a workgroup reads (its groups' channels): 16 bytes 50 us forward, 32 bytes 31, 64 bytes 30 - L2 hands out 64 bytes at least -
// and, backward, one exponential and one reciprocal an element instead of two (86 us when the store pass made g again).
// Non-temporal stores: 38 and 90 us (pieces of a line no longer meet in L2).  The backward keeps 128 KB of x in LDS, so a CU holds one workgroup and its loads wait
// while it makes its sums.  One document (B = 1): 12 us on 32 CUs, the latency of a load, two sums and 4 us of arithmetic.
#include "common.h"

namespace {
using namespace cutie;

constexpr int GN_ACT_NONE = 0, GN_ACT_RELU = 1, GN_ACT_SIGMOID = 2, GN_ACT_SILU = 3;

// The loops are written once per activation (with_act): the choice is uniform, and left inside a loop it costs a third of the
// instructions of a kernel whose arithmetic is as long as its memory traffic.
template <int A> struct Act { static constexpr int v = A; };
template <typename F> __device__ __forceinline__ void with_act(int act, F&& f) {
    switch (act) {
        case GN_ACT_RELU: f(Act<GN_ACT_RELU>()); break;
        case GN_ACT_SIGMOID: f(Act<GN_ACT_SIGMOID>()); break;
        case GN_ACT_SILU: f(Act<GN_ACT_SILU>()); break;
        default: f(Act<GN_ACT_NONE>());
    }
}

// 1 / (1 + exp(-z)).  f32: the library's expf and divide.  The 16-bit types take the hardware exponential and reciprocal (a few units of
// 2^-23, and |z| 2^-24 from the exponent's rounding): half a step of their outputs is 2^-11 (f16) or 2^-8 (bf16).  dgamma and dbeta are
// f32 and are made of the same values, of gradients that came in 16 bits.
template <int DT> __device__ __forceinline__ float sigmoid_of(float z) {
    if constexpr (DT == CUTIE_F32) return 1.f / (1.f + expf(-z));
    else return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z * -1.44269504f));
}
template <int DT, int A> __device__ __forceinline__ float act_of(float z) {
    if constexpr (A == GN_ACT_RELU) return z < 0.f ? 0.f : z;      // NaN stays NaN
    if constexpr (A == GN_ACT_SIGMOID) return sigmoid_of<DT>(z);
    if constexpr (A == GN_ACT_SILU) return z * sigmoid_of<DT>(z);
    return z;
}

// act'(z) at z = gamma * xhat + beta.  The step of the ReLU is the one place where a rounding error of z is not a small
// error of the gradient: where |z| is within the f32 error of its own computation (d = x - mean, a product and a sum: at
// most 3 roundings, 2^-24 each, of |d * rg| + |beta|; 4e-7 > 3 * 2^-24) the sign is taken in f64.
// gamma: the channel's, nullable (1).
// mean is the stored f32 one: what it misses of the mean (up to 2^-24 of it) is in every xhat of the group.
struct Norm1 { float mean, rstd, beta, rg; };      // of one channel; rg = rstd * gamma
template <int DT, int A> __device__ __forceinline__ float act_grad(float x, float d, const Norm1& n, const float* gamma) {
    if constexpr (A == GN_ACT_NONE) return 1.f;
    const float z = fmaf(d, n.rg, n.beta);
    if constexpr (A == GN_ACT_RELU) {
        if (__builtin_expect(fabsf(z) <= 4e-7f * (fabsf(d * n.rg) + fabsf(n.beta)), 0)) {
            const double z64 = ((double)x - (double)n.mean) * (double)n.rstd * (gamma ? (double)*gamma : 1.0) + (double)n.beta;
            return z64 > 0.0 ? 1.f : 0.f;
        }
        return z > 0.f ? 1.f : (z != z ? z : 0.f);
    }
    const float s = sigmoid_of<DT>(z), r = 1.f - s;
    if constexpr (A == GN_ACT_SIGMOID) return s * r;
    return s * fmaf(z, r, 1.f);
}

// ---------------------------------------------------------------------------------------------------------------- resident
struct GnShape {
    int HW, C, G, Cg;
    int gc;             // groups per workgroup
    int cv;             // vectors per pixel of a workgroup: gc * Cg / VEC
    int rows_par;       // pixels side by side: blockDim / cv
    int64_t items;      // B * G / gc
    bool fast;          // cv and cv / gc are powers of two up to 64: sums by lane exchanges
};

// Workgroups that share 128-byte lines (the groups of one pixel) go to one XCD: dispatch deals consecutive blocks to the
// eight XCDs in turn, so block i takes item (i % 8) * ceil(items / 8) + i / 8.
__device__ __forceinline__ int64_t xcd_item(int64_t items) {
    const int64_t per = (items + 7) / 8;
    return (int64_t)(blockIdx.x & 7) * per + (blockIdx.x >> 3);
}

// Sums of NV values over the threads of each group; thread t's group is (t % cv) / vpg, vpg = cv / gc vectors a pixel.
// Where cv and vpg are powers of two up to 64 (`fast`) the lanes of one group meet by exchanges, then the waves in LDS in wave
// order; else every thread leaves its value and wave w folds groups w, w + waves, ... in a fixed order.
// sh: 16 * 64 * NV floats (1024 * NV).  The caller synchronises before it uses sh again.
template <int NV>
__device__ __forceinline__ void group_sums(float (&v)[NV], float* sh, const GnShape& s, int my) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    const int vpg = s.cv / s.gc;
    if (s.fast) {
#pragma unroll
        for (int o = 32; o > 0; o >>= 1)
            if (o >= s.cv || o < vpg) {
#pragma unroll
                for (int k = 0; k < NV; ++k) v[k] += __shfl_xor(v[k], o, 64);
            }
        if (lane < s.cv && (lane & (vpg - 1)) == 0) {
#pragma unroll
            for (int k = 0; k < NV; ++k) sh[(my * NV + k) * 16 + wave] = v[k];
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const float* q = sh + (my * NV + k) * 16;
            float t = 0.f;
            for (int w = 0; w < waves; ++w) t += q[w];
            v[k] = t;
        }
        return;
    }
    __shared__ float tot[NV][1024];
    const int active = s.rows_par * s.cv, n = active / s.gc;       // threads that hold values; of them in one group
#pragma unroll
    for (int k = 0; k < NV; ++k) sh[k * 1024 + threadIdx.x] = v[k];
    __syncthreads();
    for (int g = wave; g < s.gc; g += waves) {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            float t = 0.f;
            for (int i = lane; i < n; i += 64) {
                const int r = i / vpg;
                t += sh[k * 1024 + r * s.cv + g * vpg + (i - r * vpg)];
            }
            t = wave_sum(t);
            if (lane == 0) tot[k][g] = t;
        }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < NV; ++k) v[k] = tot[k][my];
}

// chan[c][2] = (sum of sx, sum of sg) of each channel of the workgroup over its pixels.  fast: the pixels of a wave meet by
// exchanges that halve the values a lane holds (8 + 4 + 2 + 1 of them for 16 values), then the waves in LDS in wave order.
template <int VEC>
__device__ __forceinline__ void channel_sums(const float* sx, const float* sg, float* part, const GnShape& s, float* chan) {
    constexpr int NV = 2 * VEC;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    const int n = s.cv * VEC;
    if (s.fast) {
        float v[NV];
#pragma unroll
        for (int e = 0; e < VEC; ++e) { v[e] = sx[e]; v[VEC + e] = sg[e]; }
        int base = 0, left = NV;
#pragma unroll
        for (int st = 0; st < 6; ++st) {
            const int o = 32 >> st, half = (NV >> st) / 2;      // half: compile-time
            if (o < s.cv) break;
            if (half >= 1) {
                const bool up = lane & o;
#pragma unroll
                for (int i = 0; i < half; ++i) {
                    const float keep = up ? v[i + half] : v[i], send = up ? v[i] : v[i + half];
                    v[i] = keep + __shfl_xor(send, o, 64);
                }
                base += up ? half : 0;
                left = half;
            } else {
                v[0] += __shfl_xor(v[0], o, 64);
            }
        }
        float* q = part + (wave * NV + base) * s.cv + (lane & (s.cv - 1));
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (i < left) q[i * s.cv] = v[i];
        __syncthreads();
        for (int i = threadIdx.x; i < NV * s.cv; i += blockDim.x) {
            float t = 0.f;
            for (int w = 0; w < waves; ++w) t += part[w * NV * s.cv + i];
            const int k = i / s.cv, c = (i - k * s.cv) * VEC + (k & (VEC - 1));
            chan[c * 2 + (k >= VEC ? 1 : 0)] = t;
        }
        return;
    }
    float* p0 = part + threadIdx.x * VEC;
    float* p1 = p0 + blockDim.x * VEC;
#pragma unroll
    for (int e = 0; e < VEC; ++e) { p0[e] = sx[e]; p1[e] = sg[e]; }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * n; i += blockDim.x) {
        const int k = i / n, c = i - k * n;
        const float* q = part + k * blockDim.x * VEC + c;
        float t = 0.f;
        for (int r = 0; r < s.rows_par; ++r) t += q[r * n];
        chan[c * 2 + k] = t;
    }
}

template <int DT, int VEC, int K>
__global__ __launch_bounds__(1024) void gn_fwd_resident(const typename elem<DT>::type* __restrict__ x, int ld_x,
                                                        const float* __restrict__ gamma, const float* __restrict__ beta, float eps,
                                                        int act, typename elem<DT>::type* __restrict__ y, int ld_y,
                                                        float* __restrict__ stats, GnShape s) {
    __shared__ float sh1[1024];
    __shared__ float sh2[2 * 1024];
    const int64_t item = xcd_item(s.items);
    if (item >= s.items) return;
    const int per = s.G / s.gc;
    const int64_t b = item / per;
    const int g0 = (int)(item - b * per) * s.gc;
    const bool on = (int)threadIdx.x < s.rows_par * s.cv;
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
    float sum[1] = {0.f};
#pragma unroll
    for (int k = 0; k < K; ++k)
        if (on && row + k * s.rows_par < s.HW) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) sum[0] += d[k].get(e);
        }
    group_sums<1>(sum, sh1, s, my);
    const float mean0 = sum[0] * inv_n;
    // second moments about mean0, and what mean0 misses of the mean (its own rounding): d1
    float q[2] = {0.f, 0.f};
#pragma unroll
    for (int k = 0; k < K; ++k)
        if (on && row + k * s.rows_par < s.HW) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) { const float t = d[k].get(e) - mean0; q[0] += t; q[1] = fmaf(t, t, q[1]); }
        }
    group_sums<2>(q, sh2, s, my);
    const float d1 = q[0] * inv_n, m2 = q[1] * inv_n;
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
    with_act(act, [&](auto A) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int r = row + k * s.rows_par;
            if (r < s.HW) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) d[k].set(e, act_of<DT, decltype(A)::v>(fmaf(d[k].get(e) - mean0, rg[e], be[e])));
                d[k].store(py + (int64_t)r * ld_y);
            }
        }
    });
}

// chan (nullable) f32 [B][C][2]: (sum g * xhat, sum g) of each sample and channel, folded over b by gn_fold_params.
// dy and x are read once, four vectors ahead of their use; g = dy act'(z) stays in registers as f32 (its exponential and
// reciprocal are 32 of the 88 cycles that an element takes up to the sums), x as it came in LDS (vectors) or registers.
template <int DT, int VEC, int K>
__global__ __launch_bounds__(VEC > 1 ? 512 : 1024) void gn_bwd_resident(const typename elem<DT>::type* __restrict__ dy, int ld_dy,
                                                                        const typename elem<DT>::type* __restrict__ x, int ld_x,
                                                                        const float* __restrict__ gamma, const float* __restrict__ beta,
                                                                        int act, const float* __restrict__ stats,
                                                                        typename elem<DT>::type* __restrict__ dx, int ld_dx,
                                                                        float* __restrict__ chan, GnShape s) {
    typedef Pack<DT, VEC> P;
    constexpr bool XL = VEC > 1;
    extern __shared__ __attribute__((aligned(16))) char dyn[];      // x [K][blockDim] vectors (XL); later the channel sums
    __shared__ float sh[2 * 1024];
    const int64_t item = xcd_item(s.items);
    if (item >= s.items) return;
    const int per = s.G / s.gc;
    const int64_t b = item / per;
    const int g0 = (int)(item - b * per) * s.gc;
    const bool on = (int)threadIdx.x < s.rows_par * s.cv;
    const int col = threadIdx.x % s.cv, row = threadIdx.x / s.cv;
    const int my = on ? col / (s.cv / s.gc) : 0;
    const int c0 = g0 * s.Cg + col * VEC;
    const typename elem<DT>::type* px = x + (b * s.HW) * ld_x + c0;
    const typename elem<DT>::type* pd = dy + (b * s.HW) * ld_dy + c0;
    P* keep = reinterpret_cast<P*>(dyn) + threadIdx.x;
    P kx[XL ? 1 : K];
    const float mean = stats[(b * s.G + g0 + my) * 2], rstd = stats[(b * s.G + g0 + my) * 2 + 1];
    Norm1 ch[VEC];
    float sg[VEC], sx[VEC];      // sums of g and g * (x - mean)
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        ch[e].mean = mean;
        ch[e].rstd = rstd;
        ch[e].beta = on && beta ? beta[c0 + e] : 0.f;
        ch[e].rg = on && gamma ? rstd * gamma[c0 + e] : rstd;
        sg[e] = 0.f;
        sx[e] = 0.f;
    }
    with_act(act, [&](auto A) {
        float g[K][VEC];
        constexpr int AHEAD = K < 4 ? K : 4;
        P vx[AHEAD], vd[AHEAD];
        auto fetch = [&](int k) {
            const int r = row + k * s.rows_par;
            if (on && r < s.HW) {
                vx[k % AHEAD].load(px + (int64_t)r * ld_x);
                vd[k % AHEAD].load(pd + (int64_t)r * ld_dy);
            }
        };
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) fetch(k);
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const bool in = on && row + k * s.rows_par < s.HW;
            const P cx = vx[k % AHEAD], cd = vd[k % AHEAD];
            if (k + AHEAD < K) fetch(k + AHEAD);
            if constexpr (XL) keep[k * blockDim.x] = cx;
            else kx[k] = cx;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                g[k][e] = 0.f;
                if (in) {
                    const float xe = cx.get(e), d = xe - mean;
                    g[k][e] = cd.get(e) * act_grad<DT, decltype(A)::v>(xe, d, ch[e], gamma ? gamma + c0 + e : nullptr);
                    sg[e] += g[k][e];
                    sx[e] = fmaf(g[k][e], d, sx[e]);
                }
            }
            __builtin_amdgcn_sched_barrier(0);      // one vector at a time: unrolled freely, the registers do not hold it
        }
        float h[2] = {0.f, 0.f};
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            h[0] = fmaf(sg[e], ch[e].rg, h[0]);
            h[1] = fmaf(sx[e], ch[e].rg, h[1]);
            sx[e] *= rstd;
        }
        const float inv_n = 1.f / ((float)s.HW * (float)s.Cg);
        group_sums<2>(h, sh, s, my);
        // dx = rstd (g gamma - sum (g gamma) / N - d rstd sum (g gamma d rstd) / N), d = x - mean, rstd gamma = rg
        const float s0 = h[0] * inv_n, s1 = h[1] * inv_n * rstd * rstd;
        typename elem<DT>::type* pq = dx + (b * s.HW) * ld_dx + c0;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int r = row + k * s.rows_par;
            if (on && r < s.HW) {
                P q;
                if constexpr (XL) q = keep[k * blockDim.x];
                else q = kx[k];
#pragma unroll
                for (int e = 0; e < VEC; ++e) q.set(e, fmaf(g[k][e], ch[e].rg, -fmaf(q.get(e) - mean, s1, s0)));
                q.store(pq + (int64_t)r * ld_dx);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    });
    if (chan) {
        __syncthreads();      // x in LDS is read
        channel_sums<VEC>(sx, sg, reinterpret_cast<float*>(dyn), s, chan + (b * s.C + g0 * s.Cg) * 2);
    }
}

// dgamma[c] (+)= sum_b chan[b][c][0], dbeta[c] (+)= sum_b chan[b][c][1]: a workgroup owns 8 values, 32 lanes each add
// every 32nd sample, the 32 sums are added in lane order (f64: up to 65535 samples)
__global__ __launch_bounds__(256) void gn_fold_params(const float* __restrict__ chan, int B, int C, float* __restrict__ dgamma,
                                                      float* __restrict__ dbeta, int accumulate) {
    __shared__ double sh[32][8];
    const int el = threadIdx.x & 7, part = threadIdx.x >> 3;
    const int64_t i = (int64_t)blockIdx.x * 8 + el, n = (int64_t)C * 2;
    double t = 0;
    if (i < n)
        for (int b = part; b < B; b += 32) t += chan[b * n + i];
    sh[part][el] = t;
    __syncthreads();
    if (part || i >= n) return;
    t = 0;
#pragma unroll
    for (int k = 0; k < 32; ++k) t += sh[k][el];
    float* out = (i & 1) ? dbeta : dgamma;
    if (out) out[i >> 1] = (accumulate ? out[i >> 1] : 0.f) + (float)t;
}

// ------------------------------------------------------------------------------------------------------------------- split
// grid (T slices of HW, B, blocks of 256 vectors).  slots double [B][T][C][2].  The variance of the forward is taken about the group's
// first value s: (s - mean)^2 is one of the N squares that make up N var, so E[(x - s)^2] - E[x - s]^2 loses at most log2 N of 53 bits
// whatever the level of x (about 0: 2 log2(level / spread), and a spread of 1/4 at a level of 10^6 gives 1/sigma 19 % off).  f32
// values are added up as x - s.  16-bit ones as they are, and the fold moves the sums: where their level is far above their spread
// they are whole numbers below 2^12 of one step, so the f64 sums are exact.  (The subtraction in the pass: 512 x 512 x 1024 bf16
// 404 us in place of 338; f32 603 and 597.)
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

// slots[c][2] = the threads' sums in red, [2][thread][VEC], over the rows side by side
template <int VEC, typename R>
__device__ __forceinline__ void split_store(const double (*red)[256 * VEC], const SplitMap<VEC>& m, int C, R* slots) {
    __syncthreads();
    const int n = m.nv * VEC;
    R* out = slots + ((m.b * gridDim.x + blockIdx.x) * C + (int64_t)blockIdx.z * 256 * VEC) * 2;
    for (int i = threadIdx.x; i < 2 * n; i += 256) {
        const int k = i / n, c = i - k * n;
        double t = 0;
        for (int r = 0; r < m.rows_par; ++r) t += red[k][r * n + c];
        out[c * 2 + k] = (R)t;
    }
}

// a value that is not finite makes its group NaN through the sums; the mean is then what the values themselves give
template <typename T> __device__ __forceinline__ double gn_first(const T* x, int ld_x, int64_t b, int HW, int c) {
    const float v = load_as_f32(x + b * HW * ld_x + c);
    return fabsf(v) <= 3.4028235e38f ? v : 0.f;
}

template <int DT, int VEC>
__global__ __launch_bounds__(256) void gn_fwd_partial(const typename elem<DT>::type* __restrict__ x, int ld_x, int HW, int C, int Cg,
                                                      double* __restrict__ slots) {
    __shared__ double red[2][256 * VEC];
    const SplitMap<VEC> m(HW, C);
    double a[VEC] = {}, q[VEC] = {}, first[VEC] = {};
    if (m.on) {
        int run = m.c0 / Cg;      // the group of channel c0 + e: at most one further with every channel
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            run += m.c0 + e == (run + 1) * Cg;
            if constexpr (DT == CUTIE_F32) first[e] = gn_first(x, ld_x, m.b, HW, run * Cg);
        }
#pragma unroll 4
        for (int r = m.r0 + m.row; r < m.r1; r += m.rows_par) {
            Pack<DT, VEC> v;
            v.load(x + (m.b * HW + r) * ld_x + m.c0);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                double t = v.get(e);
                if constexpr (DT == CUTIE_F32) t -= first[e];
                a[e] += t;
                q[e] = fma(t, t, q[e]);
            }
        }
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) { red[0][threadIdx.x * VEC + e] = a[e]; red[1][threadIdx.x * VEC + e] = q[e]; }
    split_store<VEC>(red, m, C, slots);
}

// one workgroup per (group, sample): stats, and in `low` what the f32 mean misses
template <int DT>
__global__ __launch_bounds__(256) void gn_fwd_fold(const typename elem<DT>::type* __restrict__ x, int ld_x,
                                                   const double* __restrict__ slots, int T, int HW, int C, int G, float eps,
                                                   float* __restrict__ stats, float* __restrict__ low) {
    __shared__ double red[2][256];
    const int Cg = C / G, g = blockIdx.x;
    const int64_t b = blockIdx.y;
    double a = 0, q = 0;
    const unsigned n = (unsigned)T * Cg;      // T <= 256
#pragma unroll 4
    for (unsigned i = threadIdx.x; i < n; i += 256) {
        const unsigned t = i / (unsigned)Cg;
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
    const double N = (double)HW * Cg, first = gn_first(x, ld_x, b, HW, g * Cg);
    a = red[0][0];
    q = red[1][0];
    if constexpr (DT != CUTIE_F32) {
        q = fma(-2 * first, a, q) + N * first * first;
        a -= N * first;
    }
    const double off = a / N, mean = first + off;
    double var = q / N - off * off;
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
    int run = m.c0 / Cg;      // the group of channel c0 + e: at most one further with every channel
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        run += m.c0 + e == (run + 1) * Cg;
        const int64_t g = m.b * G + run;
        mean[e] = stats[g * 2];
        rg[e] = stats[g * 2 + 1] * (gamma ? gamma[m.c0 + e] : 1.f);
        be[e] = fmaf(-low[g], rg[e], beta ? beta[m.c0 + e] : 0.f);
    }
    with_act(act, [&](auto A) {
#pragma unroll 4
        for (int r = m.r0 + m.row; r < m.r1; r += m.rows_par) {
            Pack<DT, VEC> v;
            v.load(x + (m.b * HW + r) * ld_x + m.c0);
#pragma unroll
            for (int e = 0; e < VEC; ++e) v.set(e, act_of<DT, decltype(A)::v>(fmaf(v.get(e) - mean[e], rg[e], be[e])));
            v.store(y + (m.b * HW + r) * ld_y + m.c0);
        }
    });
}

template <int VEC>
__device__ __forceinline__ void norms(Norm1* ch, const SplitMap<VEC>& m, int Cg, int G, const float* stats, const float* gamma,
                                      const float* beta) {
    int run = m.c0 / Cg;      // the group of channel c0 + e: at most one further with every channel
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        run += m.c0 + e == (run + 1) * Cg;
        const int64_t g = m.b * G + run;
        ch[e].mean = stats[g * 2];
        ch[e].rstd = stats[g * 2 + 1];
        ch[e].beta = beta ? beta[m.c0 + e] : 0.f;
        ch[e].rg = gamma ? ch[e].rstd * gamma[m.c0 + e] : ch[e].rstd;
    }
}

// f32 sums of GN_RUN pixels, which go to f64 sums in LDS: no chain of f32 additions is longer, however large the plane
constexpr int GN_RUN = 64;
template <int DT, int VEC>
__global__ __launch_bounds__(256) void gn_bwd_partial(const typename elem<DT>::type* __restrict__ dy, int ld_dy,
                                                      const typename elem<DT>::type* __restrict__ x, int ld_x,
                                                      const float* __restrict__ gamma, const float* __restrict__ beta,
                                                      const float* __restrict__ stats, int act, int HW, int C, int G,
                                                      float* __restrict__ slots) {
    __shared__ double red[2][256 * VEC];
    const SplitMap<VEC> m(HW, C);
    const int Cg = C / G;
    double *tx = red[0] + threadIdx.x * VEC, *tg = red[1] + threadIdx.x * VEC;      // this thread's sums of g * xhat and g
#pragma unroll
    for (int e = 0; e < VEC; ++e) tx[e] = tg[e] = 0;
    if (m.on) {
        Norm1 ch[VEC];
        norms<VEC>(ch, m, Cg, G, stats, gamma, beta);
        with_act(act, [&](auto A) {
            for (int r = m.r0 + m.row; r < m.r1;) {
                const int stop = min(m.r1, r + GN_RUN * m.rows_par);
                float sx[VEC] = {}, sg[VEC] = {};
                auto fetch = [&](int at, Pack<DT, VEC>& vx, Pack<DT, VEC>& vd) {
                    vx.load(x + (m.b * HW + at) * ld_x + m.c0);
                    vd.load(dy + (m.b * HW + at) * ld_dy + m.c0);
                };
                auto add = [&](const Pack<DT, VEC>& vx, const Pack<DT, VEC>& vd) {
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        const float xe = vx.get(e), d = xe - ch[e].mean;
                        const float g = vd.get(e) * act_grad<DT, decltype(A)::v>(xe, d, ch[e], gamma ? gamma + m.c0 + e : nullptr);
                        sg[e] += g;
                        sx[e] = fmaf(g, d, sx[e]);
                    }
                };
                Pack<DT, VEC> vx[2], vd[2];
                // two pixels' loads together (one by one 512 x 512 x 1024 f32 takes 814 us, not 576)
                for (; r + m.rows_par < stop; r += 2 * m.rows_par) {
                    fetch(r, vx[0], vd[0]);
                    fetch(r + m.rows_par, vx[1], vd[1]);
                    add(vx[0], vd[0]);
                    add(vx[1], vd[1]);
                }
                if (r < stop) {
                    fetch(r, vx[0], vd[0]);
                    add(vx[0], vd[0]);
                    r += m.rows_par;
                }
#pragma unroll
                for (int e = 0; e < VEC; ++e) { tx[e] += (double)sx[e] * ch[e].rstd; tg[e] += sg[e]; }
            }
        });
    }
    split_store<VEC>(red, m, C, slots);
}

// one workgroup per (group, sample): chan[b][c][2] = the channel's sums over its slots (in slot order), and
// grp[b][g][2] = (mean of h, mean of h * xhat).  At most 256 slots of a channel and 256 channels of a thread: f32 will do
// (in f64 21 us in place of 12 for 4096 groups)
__global__ __launch_bounds__(256) void gn_bwd_fold(const float* __restrict__ slots, int T, int HW, int C, int G,
                                                   const float* __restrict__ gamma, float* __restrict__ chan, float* __restrict__ grp) {
    __shared__ float red[2][256];
    const int Cg = C / G, g = blockIdx.x;
    const int64_t b = blockIdx.y;
    float h0 = 0.f, h1 = 0.f;
    // `parts` threads a channel take every parts-th slot, their sums are added in order
    const int w = min(Cg, 256), parts = 256 / w, col = threadIdx.x % w, part = threadIdx.x / w;
    for (int c0 = 0; c0 < Cg; c0 += w) {
        const int c = c0 + col, cc = g * Cg + c;
        float a = 0.f, q = 0.f;
        if (part < parts && c < Cg) {
#pragma unroll 8
            for (int t = part; t < T; t += parts) {
                const float2 v = *reinterpret_cast<const float2*>(slots + ((b * T + t) * C + cc) * 2);
                a += v.x;
                q += v.y;
            }
        }
        red[0][threadIdx.x] = a;
        red[1][threadIdx.x] = q;
        __syncthreads();
        if (part == 0 && c < Cg) {
            for (int k = 1; k < parts; ++k) { a += red[0][k * w + col]; q += red[1][k * w + col]; }
            chan[(b * C + cc) * 2] = a;
            chan[(b * C + cc) * 2 + 1] = q;
            const float ga = gamma ? gamma[cc] : 1.f;
            h1 = fmaf(a, ga, h1);
            h0 = fmaf(q, ga, h0);
        }
        __syncthreads();
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
    Norm1 ch[VEC];
    float s0[VEC], s1[VEC];
    norms<VEC>(ch, m, Cg, G, stats, gamma, beta);
    int run = m.c0 / Cg;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        run += m.c0 + e == (run + 1) * Cg;
        const int64_t g = m.b * G + run;
        s0[e] = grp[g * 2] * ch[e].rstd;
        s1[e] = grp[g * 2 + 1] * ch[e].rstd * ch[e].rstd;
    }
    with_act(act, [&](auto A) {
#pragma unroll 2
        for (int r = m.r0 + m.row; r < m.r1; r += m.rows_par) {
            Pack<DT, VEC> vx, vd;
            vx.load(x + (m.b * HW + r) * ld_x + m.c0);
            vd.load(dy + (m.b * HW + r) * ld_dy + m.c0);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float xe = vx.get(e), d = xe - ch[e].mean;
                const float g = vd.get(e) * act_grad<DT, decltype(A)::v>(xe, d, ch[e], gamma ? gamma + m.c0 + e : nullptr);
                vd.set(e, fmaf(g, ch[e].rg, -fmaf(d, s1[e], s0[e])));
            }
            vd.store(dx + (m.b * HW + r) * ld_dx + m.c0);
        }
    });
}

// ------------------------------------------------------------------------------------------------------------------- host
constexpr int SLICE = 8192, ROWS = 8;      // of the split form's two passes (8 x 128 x 128 x 64 f16 backward: 29 us; 4 rows 33)
inline int elem_bytes(int dt) { return dt == CUTIE_F32 ? 4 : 2; }

// slices of HW that a sample is cut into for the sums of the split form: enough workgroups for the chip, but at least 32 pixels
// and SLICE values each
inline int gn_slices(int B, int HW, int C) {
    int64_t t = cdiv(2048, (int64_t)B * cdiv(C, 1024));
    int64_t most = cdiv(HW, 32);
    if (most > cdiv((int64_t)HW * C, SLICE)) most = cdiv((int64_t)HW * C, SLICE);
    if (t > most) t = most;
    if (t > 256) t = 256;
    return t < 1 ? 1 : (int)t;
}
// and for its second pass, whose slices leave nothing behind: ROWS pixels a thread
inline unsigned gn_apply_slices(int HW, int C, int vec) {
    const int cv = C / vec;
    const int64_t t = cdiv(HW, (int64_t)(256 / (cv < 256 ? cv : 256)) * ROWS);
    return (unsigned)(t > 65535 ? 65535 : t);
}

// Values of a vector: as many of `run` consecutive channels as 16 bytes hold, wherever a row begins (32 x 64 x 64 x 256 f16 in rows of
// 257: 47 us forward, single elements 68)
inline int gn_vec(int dt, int run) {
    if (dt == CUTIE_F32) return run % 4 == 0 ? 4 : 1;
    return run % 8 == 0 ? 8 : (run % 4 == 0 ? 4 : 1);
}

// of the split form, whose threads carry their channels' constants: four (8 x 128 x 128 x 64 f16 29 us backward, eight 35, single elements
// 32), eight of a wide row (512 x 512 x 1024 bf16: 622 us, four 713; with the sums of two pixels at a time 611)
inline int gn_split_vec(int dt, int C) {
    const int v = gn_vec(dt, C);
    return v == 8 && C < 1024 ? 4 : v;
}

struct GnPlan { bool resident; int threads, K; GnShape s; };

// What the two forms take, roughly, in us: the resident form by rounds of workgroups (a forward CU holds two of them, a backward CU
// one) and the lines that a workgroup touches - pieces of a pixel below 64 bytes move 64 all the same - the split form by its
// launches and the bytes of a tensor.  Resident / split, measured: 8 x 64 x 64 x 66 f16, 33 groups 15 / 18 forward and 24 / 27 backward,
// 16 of them 26 / 19 and 37 / 31; 32 x 64 x 64 x 256 f16, 128 groups 117 / 54 and 173 / 92, 32 groups 31 / 50 and 76 / 86;
// 4 x 128 x 128 x 64 f16, 8 groups 36 / 18 forward; 8 x 128 x 128 x 256 f16, 32 groups 65 / 50 forward; 8 x 64 x 64 x 264 f16, 33 groups 20 / 22 and 44 / 33; 32 x 64 x 64 x 24, 3 groups 12 / 18
// and 19 / 24.
inline double gn_resident_us(const GnShape& s, int es, bool bwd) {
    const double piece = (double)s.gc * s.Cg * es, rounds = (double)s.items / 256;
    if (bwd) return cdiv(s.items, 256) * (9.0 + 0.75 * piece) * s.HW / 4096;
    return 3.0 + (rounds < 1 ? 1 : rounds) * s.HW * (piece < 64 ? 64 : piece) / 25e3;
}
inline double gn_split_us(int64_t bytes, bool bwd) { return bwd ? 22 + bytes * 1e-6 : 13 + bytes * 0.45e-6; }

// kmax: vectors of `vec` elements a thread may hold; tmax: threads of a workgroup
inline GnPlan gn_plan(int B, int HW, int C, int G, int dt, int vec, int kmax, int tmax, bool bwd) {
    GnPlan p = {};
    const int Cg = C / G, es = elem_bytes(dt);
    p.s.HW = HW; p.s.C = C; p.s.G = G; p.s.Cg = Cg;
    int gc = 0;
    for (int d = 1; d <= G; ++d) {
        if (G % d) continue;
        const int64_t cv = (int64_t)d * Cg / vec;
        if (cv > tmax) break;
        if (cdiv(HW, tmax / cv) > kmax) break;                                           // does not fit the registers
        // 64 bytes of a pixel and 8 KB in all are enough (32 x 64 x 64 x 256 f16: 31 us with 32, 30 with 64)
        if (gc && (int64_t)gc * Cg * es >= 64 && (int64_t)gc * Cg * es * HW >= 8192) break;
        if (gc && (int64_t)B * G / d < 256) break;      // a workgroup for every CU comes before width (one document: 25 against 31 us)
        gc = d;
    }
    if (!gc) return p;
    const int64_t cv = (int64_t)gc * Cg / vec;
    int64_t t = cdiv(cdiv((int64_t)HW * cv, 4), 64) * 64;      // about four vectors a thread
    if (t > tmax) t = tmax;
    if (t < cv) t = cdiv(cv, 64) * 64;
    if (t < 64) t = 64;
    p.threads = (int)t;
    p.s.gc = gc;
    p.s.cv = (int)cv;
    p.s.rows_par = (int)(t / cv);
    p.s.items = (int64_t)B * (G / gc);
    p.K = (int)cdiv(HW, p.s.rows_par);
    auto pow2 = [](int64_t v) { return v <= 64 && (v & (v - 1)) == 0; };
    p.s.fast = pow2(cv) && pow2(cv / gc);
    // a launch counts its threads in 32 bits (20000 x 1 x 45023 f16 in 4093 groups: 82 million workgroups of 64)
    const bool launches = cdiv(p.s.items, 8) * 8 * p.threads <= 0xffffffffll;
    p.resident = p.K <= kmax && launches && gn_resident_us(p.s, es, bwd) <= gn_split_us((int64_t)B * HW * C * es, bwd);
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

constexpr int GN_FWD_KMAX = 16;

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

// whether [rows][ld] views of C columns share an element: slices of one wide buffer do not
inline bool gn_overlap(const void* a, int ld_a, const void* b, int ld_b, int64_t rows, int C, int es) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    const uintptr_t na = (uintptr_t)((rows - 1) * ld_a + C) * es, nb = (uintptr_t)((rows - 1) * ld_b + C) * es;
    if (x >= y + nb || y >= x + na) return false;
    if (ld_a != ld_b) return true;
    const uintptr_t row = (uintptr_t)ld_a * es, d = (x > y ? x - y : y - x) % row;
    return d < (uintptr_t)C * es || row - d < (uintptr_t)C * es;
}

// the outputs beside the activations (`outs`; the workspace, where the form uses one) meet no other tensor of the call
inline int gn_apart(const char* who, const Rows* views, int nv, const Dense* ins, int ni, const Dense* outs, int no) {
    bool bad = false;
    for (int i = 0; i < no; ++i) {
        for (int j = 0; j < nv; ++j) bad |= rows_meet(views[j], outs[i]);
        for (int j = 0; j < ni; ++j) bad |= dense_meet(ins[j], outs[i]);
        for (int j = 0; j < i; ++j) bad |= dense_meet(outs[j], outs[i]);
    }
    CUTIE_CHECK_ARG(!bad, "%s: statistics, gradients of gamma and beta or the workspace overlaps another tensor of the call", who);
    return CUTIE_OK;
}

inline int gn_check(const char* who, int B, int HW, int C, int G, int act, int dt) {
    CUTIE_CHECK_ARG(B >= 0 && HW >= 0 && C >= 1 && G >= 1 && C % G == 0, "%s: B=%d HW=%d C=%d groups=%d (groups must divide C)", who, B,
                    HW, C, G);
    CUTIE_CHECK_ARG(B <= 65535 && G <= 65535 && C <= 65535, "%s: B=%d, groups=%d, C=%d (at most 65535 each)", who, B, G, C);
    CUTIE_CHECK_ARG(HW <= (1 << 30), "%s: HW=%d (at most 2^30)", who, HW);
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
    const int vec = gn_vec(dtype, C / groups);
    const GnPlan p = gn_plan(B, HW, C, groups, dtype, vec, GN_FWD_KMAX, 1024, false);
    const GnSpace w = gn_space(B, HW, C, groups);
    if (!p.resident && (!workspace || workspace_bytes < w.total || !aligned16(workspace))) {
        set_error("gn_fwd: workspace %zu < %zu (or not 16-byte aligned)", workspace ? workspace_bytes : 0, w.total);
        return CUTIE_E_WORKSPACE;
    }
    const int es = elem_bytes(dtype);
    CUTIE_CHECK_ARG(!gn_overlap(x, ld_x, y, ld_y, (int64_t)B * HW, C, es), "gn_fwd: y overlaps x");
    const uint64_t vector = (uint64_t)C * sizeof(float), width = (uint64_t)C * es;
    const Rows views[] = {{x, (int64_t)B * HW, width, (uint64_t)ld_x * es}, {y, (int64_t)B * HW, width, (uint64_t)ld_y * es}};
    const Dense ins[] = {{gamma, vector}, {beta, vector}};
    const Dense outs[] = {{stats, (uint64_t)B * groups * 2 * sizeof(float)}, {p.resident ? nullptr : workspace, w.total}};
    if (int e = gn_apart("gn_fwd", views, 2, ins, 2, outs, 2)) return e;
    CUTIE_CHECK_ARG(!rows_meet(views[1], ins[0]) && !rows_meet(views[1], ins[1]), "gn_fwd: y overlaps gamma or beta");
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
    char* ws = (char*)workspace;
    double* slots = (double*)(ws + w.slots);
    float* low = (float*)(ws + w.low);
    const int sv = gn_split_vec(dtype, C), T = gn_slices(B, HW, C);
    const dim3 grid((unsigned)T, (unsigned)B, (unsigned)cdiv(C / sv, 256)), apply(gn_apply_slices(HW, C, sv), grid.y, grid.z);
    CUTIE_DISPATCH_DTYPE(dtype, DT, {
        typedef typename elem<DT>::type E;
        GN_VECS(DT, sv, VEC, {
            hipLaunchKernelGGL((gn_fwd_partial<DT, VEC>), grid, dim3(256), 0, stream, (const E*)x, ld_x, HW, C, C / groups, slots);
            hipLaunchKernelGGL((gn_fwd_fold<DT>), dim3((unsigned)groups, (unsigned)B), dim3(256), 0, stream, (const E*)x, ld_x, slots, T, HW,
                               C, groups, eps, stats, low);
            hipLaunchKernelGGL((gn_fwd_apply<DT, VEC>), apply, dim3(256), 0, stream, (const E*)x, ld_x, gamma, beta, stats, low, act, (E*)y,
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
    CUTIE_CHECK_ARG(none || !(gn_overlap(dy, ld_dy, dx, ld_dx, (int64_t)B * HW, C, es) || gn_overlap(x, ld_x, dx, ld_dx, (int64_t)B * HW, C, es)),
                    "gn_bwd: dx overlaps dy or x");
    const uint64_t vector = (uint64_t)C * sizeof(float), width = (uint64_t)C * es;
    const int64_t rows = (int64_t)B * HW;      // 0: no views
    const Rows views[] = {{dy, rows, width, (uint64_t)ld_dy * es}, {x, rows, width, (uint64_t)ld_x * es}, {dx, rows, width, (uint64_t)ld_dx * es}};
    const Dense ins[] = {{gamma, vector}, {beta, vector}, {stats, (uint64_t)B * groups * 2 * sizeof(float)}};
    const Dense outs[] = {{dgamma, vector}, {dbeta, vector}, {none ? nullptr : workspace, w.total}};
    if (int e = gn_apart("gn_bwd", views, 3, ins, 3, outs, 3)) return e;
    CUTIE_CHECK_ARG(!rows_meet(views[2], ins[0]) && !rows_meet(views[2], ins[1]) && !rows_meet(views[2], ins[2]),
                    "gn_bwd: dx overlaps gamma, beta or stats");
    char* ws = (char*)workspace;
    float* chan = ws ? (float*)(ws + w.chan) : nullptr;
    if (!none) {
        const int vec = gn_vec(dtype, C / groups);
        const GnPlan p = gn_plan(B, HW, C, groups, dtype, vec, vec > 1 ? 16 : 24, vec > 1 ? 512 : 1024, true);
        if (p.resident) {
            const dim3 grid((unsigned)(cdiv(p.s.items, 8) * 8));
            const size_t sums = params ? (size_t)2 * p.threads * vec * sizeof(float) : 0;
            CUTIE_DISPATCH_DTYPE(dtype, DT, {
                typedef typename elem<DT>::type E;
                GN_VECS(DT, vec, VEC, {
                    int rc = CUTIE_OK;
                    auto go = [&](auto kern, int K) {
                        const size_t held = VEC > 1 ? (size_t)K * p.threads * VEC * sizeof(E) : 0, lds = held > sums ? held : sums;
                        if (lds) rc = ensure_dyn_lds((const void*)kern, (int)lds);
                        if (rc == CUTIE_OK)
                            hipLaunchKernelGGL(kern, grid, dim3(p.threads), lds, stream, (const E*)dy, ld_dy, (const E*)x, ld_x, gamma, beta,
                                               act, stats, (E*)dx, ld_dx, params ? chan : nullptr, p.s);
                    };
                    if constexpr (VEC > 1) {
                        if (p.K <= 4) go(gn_bwd_resident<DT, VEC, 4>, 4);
                        else if (p.K <= 8) go(gn_bwd_resident<DT, VEC, 8>, 8);
                        else go(gn_bwd_resident<DT, VEC, 16>, 16);
                    } else {
                        if (p.K <= 8) go(gn_bwd_resident<DT, VEC, 8>, 8);
                        else go(gn_bwd_resident<DT, VEC, 24>, 24);
                    }
                    if (rc != CUTIE_OK) return rc;
                })
            });
            CUTIE_CHECK_LAUNCH();
        } else {
            float* slots = (float*)(ws + w.slots);
            float* grp = (float*)(ws + w.grp);
            const int sv = gn_split_vec(dtype, C), T = gn_slices(B, HW, C);
            const dim3 grid((unsigned)T, (unsigned)B, (unsigned)cdiv(C / sv, 256)), apply(gn_apply_slices(HW, C, sv), grid.y, grid.z);
            CUTIE_DISPATCH_DTYPE(dtype, DT, {
                typedef typename elem<DT>::type E;
                GN_VECS(DT, sv, VEC, {
                    hipLaunchKernelGGL((gn_bwd_partial<DT, VEC>), grid, dim3(256), 0, stream, (const E*)dy, ld_dy, (const E*)x, ld_x, gamma,
                                       beta, stats, act, HW, C, groups, slots);
                    hipLaunchKernelGGL(gn_bwd_fold, dim3((unsigned)groups, (unsigned)B), dim3(256), 0, stream, slots, T, HW, C, groups,
                                       gamma, chan, grp);
                    hipLaunchKernelGGL((gn_bwd_apply<DT, VEC>), apply, dim3(256), 0, stream, (const E*)dy, ld_dy, (const E*)x, ld_x, gamma,
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
