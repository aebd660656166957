// K17: the orthogonalised update.
//
//   X0 = U / (|U|_F + eps);   X <- X B, B = a I + b A + c A A, A = X^T X   (steps times)
// maps every singular value s of X0 to a s + b s^3 + c s^5, again and again: the quintic Newton-Schulz iteration with
// a = 3.4445, b = -4.7750, c = 2.0315, which takes (0, 1] towards 1 (0.68 .. 1.21 after five steps from s >= 1e-2).  The update
// around it: m' = mu m + g', U = g' + mu m' (or m'), p' = p (1 - lr wd) - lr k X.
//
// Number format.  Three products a step, all on the matrix cores, at f32 accuracy: a value v is held as two f16, hi = f16(v)
// and lo = f16(v - hi), 22 significant bits, and a product is hi*hi + hi*lo + lo*hi with f32 accumulation (lo*lo is below the
// 22 bits).  Against f64 the error is that of the f32 computation (2e-6 of the norm after five steps on a 256 x 1920 matrix in
// both); one f16 or bf16 term instead gives 2e-2, since small singular values are amplified up to 3.4445 ** 5 = 485 times.
// f16 has no range to spare, so each kind of matrix is kept at a fixed power of two: X (singular values at most 1.21)
// times 2^12, A (at most 1.47) and B (at most 3.4445) times 2^13: entries stay below 28300, and the smallest step of f16, 2^-24,
// is 2^-36 of X.
//
// Layout.  L = max(rows, cols) rows of S = min(rows, cols) values, both padded with zeros to multiples of 64 (the transpose of
// a wide matrix is made when it is normalised); a row is blocks of 32 values, 64 bytes hi and 64 bytes lo, so that one K step
// of a product is one 128-byte line of a row.  A and B [S][S] alike.
//
// Measured (MI355X), five steps, calls back to back on one input, all on one GPU - the figures of this file are of this kind: 14 filters
// (10 of them 3840 x 256) 355 us, of which the matrix cores need 110 for the three products at the rate of a large library product;
// 2048 x 8192 1.75 ms (1.45 ms likewise; in f32 the library's rate gives 3.6).  One call among others, on inputs that change, the
// update of the 14 filters takes 410 - 451 us, 2048 x 8192 1.77 - 1.91 ms, by the GPU.
// There are three forms: the general one of this comment, and two for fewer columns, in f32, below.
#include "conv_common.h"

namespace {
using namespace cutie;
using namespace cutie::convk;

constexpr float NS_A = 3.4445f, NS_B = -4.7750f, NS_C = 2.0315f;
constexpr float X_SCALE = 4096.f, INV_X_SCALE = 1.f / 4096.f;      // 2^12
constexpr float AB_SCALE = 8192.f;                                 // 2^13
constexpr float AB_FROM_XX = 1.f / 2048.f;                         // 2^24 (X^T X) -> 2^13 A
constexpr float AB_FROM_AA = 1.f / 8192.f;                         // 2^26 (A A)   -> 2^13 A A
constexpr float X_FROM_XB = 1.f / 8192.f;                          // 2^25 (X B)   -> 2^12 X B
constexpr int NORM_CHUNK = 8192;                                   // elements of one partial sum of squares

struct Mat {
    int rows, cols;          // as the caller holds it, contiguous
    int Lp, Sp;              // padded
    int y0, y1, a, b, slab, part;      // workspace offsets in units of 256 bytes
};
struct Io { const float *p, *g, *m; float *po, *mo; float k; };
struct Mats { Mat m[CUTIE_MAX_BATCH]; int n; };
struct Ios { Io io[CUTIE_MAX_BATCH]; };
struct Starts { int v[CUTIE_MAX_BATCH + 1]; };      // first workgroup of each matrix
struct Splits { short v[CUTIE_MAX_BATCH]; };
struct Hyper {
    float lr, mu, wd, l2, clip, grad_scale;
    int nesterov;
    const float* gnorm_sq;
    const float* loss_scale;
    const int32_t* invalid;
};

// Workgroups that read the same rows run side by side behind one L2: dispatch deals consecutive blocks to the eight XCDs in turn,
// so XCD x takes the x-th eighth of the logical ids.
__device__ __forceinline__ int xcd_id() {
    const int n = gridDim.x, q = n >> 3, r = n & 7, x = blockIdx.x & 7;
    return (x < r ? x * (q + 1) : r * (q + 1) + (x - r) * q) + (blockIdx.x >> 3);
}
__device__ __forceinline__ int find(const Starts& s, int n, int id) {
    int i = 0;
    while (i + 1 < n && id >= s.v[i + 1]) ++i;
    return i;
}
__device__ __forceinline__ char* at(char* ws, int off) { return ws + (int64_t)off * 256; }

// the step is skipped: a gradient that is not finite, or results marked invalid
__device__ __forceinline__ bool skip_step(const Hyper& h) {
    return (h.invalid && *h.invalid != 0) || (h.gnorm_sq && !(fabsf(*h.gnorm_sq) <= 3.0e38f));
}

__device__ __forceinline__ float clip_scale(const Hyper& h) {
    return h.gnorm_sq && h.clip > 0.f ? h.grad_scale * (h.clip / fmaxf(sqrtf(*h.gnorm_sq) * h.grad_scale, h.clip)) : h.grad_scale;
}

__device__ __forceinline__ void block_sum_f64(double v, double* out) {
    __shared__ double sh[4];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    if (threadIdx.x == 0) *out = ((sh[0] + sh[1]) + sh[2]) + sh[3];
}

// partial sums of squares of U, in f64 (squares of any f32 are in range), one per NORM_CHUNK elements.  MUON: U is made
// here, m' stored, U left in the buffer that the first product overwrites later.
template <bool MUON>
__global__ __launch_bounds__(256) void ns_norm_kernel(Mats ms, Ios ios, Starts st, Hyper h, char* ws) {
    const int i = find(st, ms.n, blockIdx.x), chunk = blockIdx.x - st.v[i];
    const Mat M = ms.m[i];
    const Io io = ios.io[i];
    const int64_t n = (int64_t)M.rows * M.cols, e0 = (int64_t)chunk * NORM_CHUNK;
    const int64_t e1 = min(n, e0 + NORM_CHUNK);
    double s = 0;
    if constexpr (!MUON) {
        for (int64_t e = e0 + threadIdx.x; e < e1; e += 256) {
            const double v = io.g[e];
            s = fma(v, v, s);
        }
    } else {
        float* u = (float*)at(ws, M.y1);
        const bool skip = skip_step(h);
        const float inv = h.loss_scale ? h.loss_scale[1] : 1.f;
        const float scale = clip_scale(h);
        for (int64_t e = e0 + threadIdx.x; e < e1; e += 256) {
            const float g = (io.g[e] * inv + h.l2 * io.p[e]) * scale;
            const float m0 = io.m[e];
            const float m1 = h.mu * m0 + g;
            const float v = h.nesterov ? g + h.mu * m1 : m1;
            io.mo[e] = skip ? m0 : m1;
            u[e] = v;
            s = fma((double)v, (double)v, s);
        }
    }
    block_sum_f64(s, (double*)at(ws, M.part) + chunk);
}

// v must exist as an f32 before it is narrowed.  Where it is a product the compiler may narrow straight out of the multiplier for
// the stored hi (one rounding) and from the rounded f32 for the one that lo is taken against (two): next to a tie the pair is
// then off by a whole step of f16 (one element of 8385 in the 65 x 129 test: 1.3e-5 in place of 3e-7).
__device__ __forceinline__ void split(float v, f16_t& hi, f16_t& lo) {
    asm volatile("" : "+v"(v));
    hi = (f16_t)v;
    lo = (f16_t)(v - (float)hi);
}
__device__ __forceinline__ void split4(const float* v, uint2& hi, uint2& lo) {
    half4_t h, l;
#pragma unroll
    for (int e = 0; e < 4; ++e) { f16_t a, b; split(v[e], a, b); h[e] = a; l[e] = b; }
    hi = __builtin_bit_cast(uint2, h);
    lo = __builtin_bit_cast(uint2, l);
}
__device__ __forceinline__ void join4(uint2 hi, uint2 lo, float* v) {
    const half4_t h = __builtin_bit_cast(half4_t, hi), l = __builtin_bit_cast(half4_t, lo);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = (float)h[e] + (float)l[e];
}
__device__ __forceinline__ void store4_split(char* q, const float* x) {
    uint2 hi, lo;
    split4(x, hi, lo);
    *reinterpret_cast<uint2*>(q) = hi;
    *reinterpret_cast<uint2*>(q + 64) = lo;
}
// byte offset of value c (a multiple of 4) of a row's hi part; its lo part lies 64 bytes further
__device__ __forceinline__ int64_t cell(int64_t row, int ld, int c) { return row * ((int64_t)ld * 4) + (c >> 5) * 128 + (c & 31) * 2; }

// X0 in the work layout: a workgroup makes a 64 x 64 piece of [Lp][Sp]
template <bool MUON>
__global__ __launch_bounds__(256) void ns_start_kernel(Mats ms, Ios ios, Starts st, float eps, char* ws) {
    __shared__ float tile[64][65];
    __shared__ double total;
    const int i = find(st, ms.n, blockIdx.x), id = blockIdx.x - st.v[i];
    const Mat M = ms.m[i];
    const float* src = MUON ? (const float*)at(ws, M.y1) : ios.io[i].g;
    const int nt = M.Sp >> 6, l0 = (id / nt) << 6, s0 = (id % nt) << 6;
    const bool flip = M.rows < M.cols;
    // the norm: all partial sums, in one order
    const int64_t parts = (((int64_t)M.rows * M.cols) + NORM_CHUNK - 1) / NORM_CHUNK;
    const double* part = (const double*)at(ws, M.part);
    double s = 0;
    for (int64_t k = threadIdx.x; k < parts; k += 256) s += part[k];
    block_sum_f64(s, &total);
    if (!flip) {
        // straight through: 16 lanes take a row of 64, four values each
        __syncthreads();
        const double k = (double)X_SCALE / (sqrt(total) + (double)eps);
        const int c = s0 + (threadIdx.x & 15) * 4;
        const bool wide = (M.cols & 3) == 0 && (reinterpret_cast<uintptr_t>(src) & 15) == 0 && c < M.cols;
#pragma unroll
        for (int r = threadIdx.x >> 4; r < 64; r += 16) {
            float v[4] = {0.f, 0.f, 0.f, 0.f};
            if (l0 + r < M.rows) {
                const float* p = src + (int64_t)(l0 + r) * M.cols + c;
                if (wide) {
                    const float4 f = *reinterpret_cast<const float4*>(p);
                    v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (c + e < M.cols) v[e] = p[e];
                }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = (float)((double)v[e] * k);      // 1 / norm may leave f32
            store4_split(at(ws, M.y0) + cell(l0 + r, M.Sp, c), v);
        }
        return;
    }
    const int c = threadIdx.x & 63;
    for (int r = threadIdx.x >> 6; r < 64; r += 4) {
        // read along the caller's rows
        const int row = s0 + r, col = l0 + c;
        tile[c][r] = row < M.rows && col < M.cols ? src[(int64_t)row * M.cols + col] : 0.f;
    }
    __syncthreads();
    const double k = (double)X_SCALE / (sqrt(total) + (double)eps);
    const int l = threadIdx.x >> 2, q = (threadIdx.x & 3) * 16;
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
        float v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = (float)((double)tile[l][q + e + j] * k);
        store4_split(at(ws, M.y0) + cell(l0 + l, M.Sp, s0 + q + e), v);
    }
}

// ---------------------------------------------------------------------------------------------------------------- products
// Workgroup of 4 waves, 2 x 2, tile T x T with T = 32 F, a wave F x F fragments of 16 x 16.  A K step is 32 values: the tile's
// 128-byte lines (hi and lo) go to LDS by buffer_load ... lds, STAGES of them, all but one in flight while that one is used.
template <int F> struct Shape {
    static constexpr int T = 32 * F, HALF = T * 128, STAGE = 2 * HALF;      // bytes of one operand, of both
    // F = 4: two workgroups a CU with two stages (14 filters 355 us, 2048 x 8192 1.75 ms) beat one with three (403 us, 2.27 ms).
    // F = 2: two, three and four stages are alike.
    static constexpr int STAGES = F == 4 ? 2 : 3;
    static constexpr int LDS = STAGES * STAGE;
    static constexpr int PIECES = T / 8;      // 1-KB pieces of an operand; a wave moves PIECES / 4 of each
};
__device__ __forceinline__ int tr_swz(int r) { return (r & 3) | (((r >> 3) & 1) << 2); }

template <int F> struct Frags { short8_t hi[F], lo[F]; };

template <int F>
__device__ __forceinline__ void multiply(const Frags<F>& p, const Frags<F>& q, float4_t (&acc)[F][F]) {
#pragma unroll
    for (int m = 0; m < F; ++m)
#pragma unroll
        for (int n = 0; n < F; ++n) {
            acc[m][n] = mma16<CUTIE_F16>(p.hi[m], q.hi[n], acc[m][n]);
            acc[m][n] = mma16<CUTIE_F16>(p.hi[m], q.lo[n], acc[m][n]);
            acc[m][n] = mma16<CUTIE_F16>(p.lo[m], q.hi[n], acc[m][n]);
        }
}

// my pieces of the stage have landed (N younger ones may be on their way) and my reads of the stage before are done; then
// everybody's are
template <int N> __device__ __forceinline__ void stage_ready() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}
// everything has landed: nothing may be on its way into LDS when it is used for something else or the workgroup ends
__device__ __forceinline__ void drain() {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

// acc[m][n] += sum over K steps k0 .. k1 of P[p0 + m][k] * Q[q0 + n][k]: both operands row by row along K; the steps begin `turn`
// further on and go round
template <int F>
__device__ __forceinline__ void product_rows(char* smem, const char* P, unsigned p_bytes, int p_rows, int p0, const char* Q, unsigned q_bytes,
                                             int q_rows, int q0, int ld, int k0, int k1, int turn, float4_t (&acc)[F][F]) {
    typedef Shape<F> S;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int li = lane & 15, lg = lane >> 4, wm = wave >> 1, wn = wave & 1;
    const u32x4s_t rp = make_rsrc(P, p_bytes), rq = make_rsrc(Q, q_bytes);
    const unsigned lds0 = (unsigned)(uintptr_t)((lds_void_t*)smem);
    unsigned po[S::PIECES / 4], qo[S::PIECES / 4];      // source offsets of this lane at K step 0
#pragma unroll
    for (int u = 0; u < S::PIECES / 4; ++u) {
        const int row = (wave + 4 * u) * 8 + (lane >> 3);
        const unsigned chunk = (unsigned)((lane & 7) ^ swz(row)) * 16u;
        po[u] = p0 + row < p_rows ? (unsigned)(p0 + row) * (unsigned)(ld * 4) + chunk : BUF_OOB;
        qo[u] = q0 + row < q_rows ? (unsigned)(q0 + row) * (unsigned)(ld * 4) + chunk : BUF_OOB;
    }
    // a step behind the last fetches nothing, but counts: the wait below is for a fixed number of loads
    auto issue = [&](int k, int buf) {
        const bool live = k < k1;
        k += turn;
        if (k >= k1) k -= k1 - k0;
        const unsigned d = (unsigned)k * 128u;
#pragma unroll
        for (int u = 0; u < S::PIECES / 4; ++u) {
            const unsigned dst = lds0 + buf * S::STAGE + (wave + 4 * u) * 1024;
            glds16(rp, dst, !live || po[u] == BUF_OOB ? BUF_OOB : po[u] + d);
            glds16(rq, dst + S::HALF, !live || qo[u] == BUF_OOB ? BUF_OOB : qo[u] + d);
        }
    };
    int pr[F], qr[F];
#pragma unroll
    for (int f = 0; f < F; ++f) {
        const int m = (wm * F + f) * 16 + li, n = (wn * F + f) * 16 + li;
        pr[f] = m * 128 + ((lg ^ swz(m)) << 4);
        qr[f] = S::HALF + n * 128 + ((lg ^ swz(n)) << 4);
    }
    constexpr int AHEAD = S::STAGES - 1, LOADS = 2 * (S::PIECES / 4);      // loads of a wave and stage
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) issue(k0 + a, a);
    for (int k = k0; k < k1; ++k) {
        const int buf = (k - k0) % S::STAGES;
        stage_ready<(AHEAD - 1) * LOADS>();
        issue(k + AHEAD, (k - k0 + AHEAD) % S::STAGES);
        const char* s = smem + buf * S::STAGE;
        Frags<F> p, q;
#pragma unroll
        for (int f = 0; f < F; ++f) {
            p.hi[f] = *reinterpret_cast<const short8_t*>(s + pr[f]);
            p.lo[f] = *reinterpret_cast<const short8_t*>(s + (pr[f] ^ 64));
            q.hi[f] = *reinterpret_cast<const short8_t*>(s + qr[f]);
            q.lo[f] = *reinterpret_cast<const short8_t*>(s + (qr[f] ^ 64));
        }
        multiply<F>(p, q, acc);
    }
    drain();
}

// acc[m][n] += sum over rows 32 k0 .. 32 k1 of X[r][p0 + m] * X[r][q0 + n]: K runs down the rows, so the fragments come through
// the transposing LDS read.  A staged row holds T columns (hi and lo) = T * 4 bytes as 32-byte groups, XORed by the row.  On a
// diagonal tile (p0 == q0) both operands are the same columns, staged once.
template <int F>
__device__ __forceinline__ void product_cols(char* smem, const char* X, unsigned bytes, int cols, int p0, int q0, int k0, int k1,
                                             float4_t (&acc)[F][F]) {
    typedef Shape<F> S;
    constexpr int ROWB = S::T * 4;                 // 512 or 256 bytes
    constexpr int SLOTS = ROWB / 16;               // 16-byte slots of a staged row
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int li = lane & 15, lg = lane >> 4, wm = wave >> 1, wn = wave & 1;
    const u32x4s_t rs = make_rsrc(X, bytes);
    const unsigned lds0 = (unsigned)(uintptr_t)((lds_void_t*)smem);
    unsigned po[S::PIECES / 4], qo[S::PIECES / 4];
#pragma unroll
    for (int u = 0; u < S::PIECES / 4; ++u) {
        const int slot = (wave + 4 * u) * 64 + lane, row = slot / SLOTS, w = slot % SLOTS;
        const int byte = ((((w >> 1) ^ tr_swz(row)) << 1) | (w & 1)) * 16;      // of the row's T columns: 4 bytes a column
        po[u] = p0 + byte / 4 < cols ? (unsigned)row * (unsigned)(cols * 4) + (unsigned)(p0 * 4 + byte) : BUF_OOB;
        qo[u] = q0 + byte / 4 < cols ? (unsigned)row * (unsigned)(cols * 4) + (unsigned)(q0 * 4 + byte) : BUF_OOB;
    }
    auto issue = [&](int k, int buf) {
        const bool live = k < k1;
        const unsigned d = (unsigned)k * 32u * (unsigned)(cols * 4);
#pragma unroll
        for (int u = 0; u < S::PIECES / 4; ++u) {
            const unsigned dst = lds0 + buf * S::STAGE + (wave + 4 * u) * 1024;
            glds16(rs, dst, !live || po[u] == BUF_OOB ? BUF_OOB : po[u] + d);
            if (p0 != q0) glds16(rs, dst + S::HALF, !live || qo[u] == BUF_OOB ? BUF_OOB : qo[u] + d);
        }
    };
    const int r1 = lg * 8 + (li >> 2);      // and r1 + 4, whose swizzle is the same
    unsigned pr[F], qr[F];
#pragma unroll
    for (int f = 0; f < F; ++f) {
        const int m = wm * F + f, n = wn * F + f;      // 16-column fragments: 32-byte group (m >> 1) * 4 + plane * 2 + (m & 1)
        pr[f] = lds0 + r1 * ROWB + ((((m >> 1) * 4 + (m & 1)) ^ tr_swz(r1)) * 32) + (li & 3) * 8;
        qr[f] = lds0 + (p0 != q0 ? S::HALF : 0) + r1 * ROWB + ((((n >> 1) * 4 + (n & 1)) ^ tr_swz(r1)) * 32) + (li & 3) * 8;
    }
    auto tr2 = [&](unsigned a0) {
        const short4_t a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4_t*)(uintptr_t)(a0));
        const short4_t b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4_t*)(uintptr_t)(a0 + 4 * ROWB));
        return short8_t{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    };
    constexpr int AHEAD = S::STAGES - 1, LOADS = S::PIECES / 4;      // of a wave, stage and operand
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) issue(k0 + a, a);
    for (int k = k0; k < k1; ++k) {
        const int buf = (k - k0) % S::STAGES;
        if (p0 != q0) stage_ready<(AHEAD - 1) * 2 * LOADS>();
        else stage_ready<(AHEAD - 1) * LOADS>();
        issue(k + AHEAD, (k - k0 + AHEAD) % S::STAGES);
        const unsigned o = buf * S::STAGE;
        Frags<F> p, q;
#pragma unroll
        for (int f = 0; f < F; ++f) {
            p.hi[f] = tr2(pr[f] + o);
            p.lo[f] = tr2((pr[f] ^ 64) + o);
            q.hi[f] = tr2(qr[f] + o);
            q.lo[f] = tr2((qr[f] ^ 64) + o);
        }
        multiply<F>(p, q, acc);
    }
    drain();
}

// lower-triangle tile `id` of a symmetric matrix: (row, col), col <= row
__device__ __forceinline__ void tri(int id, int& r, int& c) {
    r = (int)((sqrtf(8.f * (float)id + 1.f) - 1.f) * 0.5f);
    while (r * (r + 1) / 2 > id) --r;
    while ((r + 1) * (r + 2) / 2 <= id) ++r;
    c = id - r * (r + 1) / 2;
}

__device__ __forceinline__ float make_b(float a_old, float aa, bool diagonal) {
    return fmaf(NS_B, a_old, NS_C * (aa * AB_FROM_AA)) + (diagonal ? NS_A * AB_SCALE : 0.f);
}

// The symmetric products A = X^T X (GRAM) and A A: the tiles on and below the diagonal.  Where K is cut (`splits` parts), f32 sums
// into slabs [split][tile][T][T] for ns_fold_kernel; A A whole (splits 1) goes to B from here, both triangles.
template <int F, bool GRAM>
__global__ __launch_bounds__(256, 2) void ns_sym_kernel(Mats ms, Starts st, Splits sp, int which, char* ws) {
    typedef Shape<F> S;
    __shared__ __attribute__((aligned(1024))) char smem[S::LDS];
    const int wg = xcd_id(), i = find(st, ms.n, wg);
    const Mat M = ms.m[i];
    const int nt = (M.Sp + S::T - 1) / S::T, tiles = nt * (nt + 1) / 2;
    const int id = wg - st.v[i], sl = id / tiles, t = id % tiles, splits = sp.v[i];
    int r, c;
    tri(t, r, c);
    const int steps = (GRAM ? M.Lp : M.Sp) / 32, per = (steps + splits - 1) / splits;
    const int k0 = min(steps, sl * per), k1 = min(steps, k0 + per);
    float4_t acc[F][F];
#pragma unroll
    for (int m = 0; m < F; ++m)
#pragma unroll
        for (int n = 0; n < F; ++n) acc[m][n] = float4_t{0.f, 0.f, 0.f, 0.f};
    if constexpr (GRAM) {
        product_cols<F>(smem, at(ws, which ? M.y1 : M.y0), (unsigned)((int64_t)M.Lp * M.Sp * 4), M.Sp, r * S::T, c * S::T, k0, k1, acc);
    } else {
        const unsigned bytes = (unsigned)((int64_t)M.Sp * M.Sp * 4);
        product_rows<F>(smem, at(ws, M.a), bytes, M.Sp, r * S::T, at(ws, M.a), bytes, M.Sp, c * S::T, M.Sp, k0, k1, 0, acc);
    }
    // [n][m]: a lane holds four consecutive m of one n
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, li = lane & 15, lg = lane >> 4, wm = wave >> 1, wn = wave & 1;
    if (!GRAM && splits == 1) {
        const char* A = at(ws, M.a);
        char* B = at(ws, M.b);
#pragma unroll
        for (int n = 0; n < F; ++n) {
            __syncthreads();      // the stages (n = 0), the strip before
            float* strip = reinterpret_cast<float*>(smem) + wave * 16 * (16 * F + 1);      // a wave's 16 rows (n) of 16 F columns (m)
            const int gn = c * S::T + (wn * F + n) * 16;
#pragma unroll
            for (int m = 0; m < F; ++m) {
                const int gm = r * S::T + (wm * F + m) * 16 + lg * 4;
                float x[4] = {0.f, 0.f, 0.f, 0.f};
                if (gn < M.Sp && gm < M.Sp) {
                    const char* q = A + cell(gn + li, M.Sp, gm);
                    join4(*reinterpret_cast<const uint2*>(q), *reinterpret_cast<const uint2*>(q + 64), x);
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[e] = make_b(x[e], acc[m][n][e], gn + li == gm + e);
                    store4_split(B + cell(gn + li, M.Sp, gm), x);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) strip[li * (16 * F + 1) + m * 16 + lg * 4 + e] = x[e];
            }
            __syncthreads();
            if (r == c) continue;      // a diagonal tile holds both triangles itself
            // the mirror: rows gm .. of 16 columns gn ..
            for (int i = lane; i < 16 * F * 4; i += 64) {
                const int row = i >> 2, q4 = (i & 3) * 4, gm = r * S::T + wm * F * 16 + row;
                if (gn >= M.Sp || gm >= M.Sp) continue;
                float x[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = strip[(q4 + e) * (16 * F + 1) + row];
                store4_split(B + cell(gm, M.Sp, gn + q4), x);
            }
        }
        return;
    }
    float* out = (float*)at(ws, M.slab) + ((int64_t)sl * tiles + t) * (S::T * S::T);
#pragma unroll
    for (int m = 0; m < F; ++m)
#pragma unroll
        for (int n = 0; n < F; ++n)
            *reinterpret_cast<float4_t*>(out + ((wn * F + n) * 16 + li) * S::T + (wm * F + m) * 16 + lg * 4) = acc[m][n];
}

// slabs -> A (GRAM) or B, both triangles: a workgroup folds a 32 x 32 piece of a tile in slab order
template <int F, bool GRAM>
__global__ __launch_bounds__(256) void ns_fold_kernel(Mats ms, Starts st, Splits sp, char* ws) {
    typedef Shape<F> S;
    __shared__ float tile[32][33];
    const int i = find(st, ms.n, blockIdx.x);
    const Mat M = ms.m[i];
    const int nt = (M.Sp + S::T - 1) / S::T, tiles = nt * (nt + 1) / 2, splits = sp.v[i];
    if (!GRAM && splits == 1) return;      // B is there
    const int id = blockIdx.x - st.v[i], t = id / (F * F), piece = id % (F * F);
    int r, c;
    tri(t, r, c);
    const int n = threadIdx.x >> 3, m = (threadIdx.x & 7) * 4;      // the piece's row and column
    const int pn = (piece / F) * 32, pm = (piece % F) * 32;
    const int gn = c * S::T + pn, gm = r * S::T + pm;               // of the whole matrix
    if (gn >= M.Sp || gm >= M.Sp) return;
    const float* src = (const float*)at(ws, M.slab) + (int64_t)t * (S::T * S::T) + (pn + n) * S::T + pm + m;
    float4_t v = *reinterpret_cast<const float4_t*>(src);
    for (int k = 1; k < splits; ++k) v += *reinterpret_cast<const float4_t*>(src + (int64_t)k * tiles * (S::T * S::T));
    float x[4];
    if constexpr (GRAM) {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = v[e] * AB_FROM_XX;
    } else {
        const char* a = at(ws, M.a) + cell(gn + n, M.Sp, gm + m);
        float old[4];
        join4(*reinterpret_cast<const uint2*>(a), *reinterpret_cast<const uint2*>(a + 64), old);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = make_b(old[e], v[e], gn + n == gm + m + e);
    }
    char* dst = at(ws, GRAM ? M.a : M.b);
    store4_split(dst + cell(gn + n, M.Sp, gm + m), x);
    if (r == c) return;      // a diagonal tile holds both triangles itself
#pragma unroll
    for (int e = 0; e < 4; ++e) tile[m + e][n] = x[e];
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = tile[n][m + e];
    store4_split(dst + cell(gm + n, M.Sp, gn + m), x);
}

// X' = X B.  The last step (LAST) writes the caller's matrix: X itself, or (MUON) the parameters.
template <int F, bool LAST, bool MUON>
__global__ __launch_bounds__(256, 2) void ns_apply_kernel(Mats ms, Ios ios, Starts st, Hyper h, int which, char* ws) {
    typedef Shape<F> S;
    __shared__ __attribute__((aligned(1024))) char smem[S::LDS];
    // block order as dispatched: an XCD's workgroups share one or two column tiles of B, which stay in its L2, and stream X (2048 x 8192
    // 1.75 ms, with an XCD's blocks consecutive 1.86; 14 filters 355 us and 350)
    const int i = find(st, ms.n, blockIdx.x);
    const Mat M = ms.m[i];
    const int nt = (M.Sp + S::T - 1) / S::T, id = blockIdx.x - st.v[i];
    const int l0 = (id / nt) * S::T, s0 = (id % nt) * S::T;
    const char* X = at(ws, which ? M.y1 : M.y0);
    float4_t acc[F][F];
#pragma unroll
    for (int m = 0; m < F; ++m)
#pragma unroll
        for (int n = 0; n < F; ++n) acc[m][n] = float4_t{0.f, 0.f, 0.f, 0.f};
    // Rows of B (symmetric) against rows of X: a lane ends with four consecutive columns of one row of X.  The K steps that hold
    // this tile's part of B's diagonal, and with it a X, by far the largest term for a small singular value, come last: else every
    // later addition rounds at its size (2048 x 8192: 4.0e-6 of the result instead of 1.7e-6)
    const int steps = M.Sp / 32, turn = (s0 / 32 + S::T / 32) % steps;
    product_rows<F>(smem, at(ws, M.b), (unsigned)((int64_t)M.Sp * M.Sp * 4), M.Sp, s0, X, (unsigned)((int64_t)M.Lp * M.Sp * 4), M.Lp, l0,
                    M.Sp, 0, steps, turn, acc);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, li = lane & 15, lg = lane >> 4, wm = wave >> 1, wn = wave & 1;
    const bool flip = M.rows < M.cols;
    bool skip = false;
    if constexpr (MUON) skip = skip_step(h);
    const Io& io = ios.io[i];
    // four columns of the caller's row at once where they lie so
    const bool wide = LAST && !flip && (M.cols & 3) == 0 && ((reinterpret_cast<uintptr_t>(io.po) | (MUON ? reinterpret_cast<uintptr_t>(io.p) : 0)) & 15) == 0;
    auto update = [&](float x, float p) { return skip ? p : p * (1.f - h.lr * h.wd) - h.lr * io.k * x; };
#pragma unroll
    for (int n = 0; n < F; ++n) {
        const int l = l0 + (wn * F + n) * 16 + li;
        if (l >= (LAST ? (flip ? M.cols : M.rows) : M.Lp)) continue;
#pragma unroll
        for (int m = 0; m < F; ++m) {
            const int s = s0 + (wm * F + m) * 16 + lg * 4;
            if (s >= (LAST ? (flip ? M.rows : M.cols) : M.Sp)) continue;
            float x[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = acc[m][n][e] * (LAST ? X_FROM_XB * INV_X_SCALE : X_FROM_XB);
            if constexpr (!LAST) {
                store4_split(at(ws, which ? M.y0 : M.y1) + cell(l, M.Sp, s), x);
            } else if (wide) {
                const int64_t k = (int64_t)l * M.cols + s;
                float4 o = make_float4(x[0], x[1], x[2], x[3]);
                if constexpr (MUON) {
                    const float4 p = *reinterpret_cast<const float4*>(io.p + k);
                    o = make_float4(update(o.x, p.x), update(o.y, p.y), update(o.z, p.z), update(o.w, p.w));
                }
                *reinterpret_cast<float4*>(io.po + k) = o;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (s + e >= (flip ? M.rows : M.cols)) continue;
                    const int64_t k = flip ? (int64_t)(s + e) * M.cols + l : (int64_t)l * M.cols + s + e;
                    io.po[k] = MUON ? update(x[e], io.p[k]) : x[e];
                }
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------------------------- small
// Matrices of few rows and columns: one workgroup does everything, X, A and B as f32 in LDS, the products on the f32 matrix cores
// (16 x 16 x 4; they have a sixteenth of the f16 rate, but the launches of the general form alone take longer).  The limit is where
// the tall form below takes as long.  Five steps, one matrix: 128 x 16 16 us (tall 29, general 76), 352 x 16 35 (32), 64 x 18 17,
// 288 x 32 48 (36), 192 x 48 61 (48), 128 x 64 55 (63), 192 x 64 80 (64).
constexpr int SMALL_S = 64, SMALL_THREADS = 512, SMALL_WAVES = SMALL_THREADS / 64;
constexpr int TALL_L = 8192;
__host__ __device__ inline int up16(int v) { return (v + 15) & ~15; }
inline bool is_small(int r, int c) {
    const int L = r > c ? r : c, S = r > c ? c : r;
    return S <= SMALL_S && L <= 384 && L * up16(S) <= 8192;
}
inline size_t small_lds(int r, int c) {
    const int L = up16(r > c ? r : c), S = up16(r > c ? c : r), ld = S + 4;
    return ((size_t)L + 2 * S) * ld * sizeof(float);
}
struct Smalls { int rows[CUTIE_MAX_BATCH], cols[CUTIE_MAX_BATCH], n; };

// acc[c] += P(row m, k) Q(k, column n) over k = 0 .. K-1 for NC column blocks: pa = P's address of (m = li, k = lg), pk its
// step per k; qa = Q's address of (k = lg, n = li), qk likewise
template <int NC>
__device__ __forceinline__ void small_product(const float* pa, int pk, const float* qa, int qk, int K, int nc, float4_t (&acc)[NC]) {
    for (int k = 0; k < K; k += 16) {      // K is a multiple of 16; four steps' operands are on their way together
        float a[4], q[4][NC];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            a[j] = pa[(k + j * 4) * pk];
#pragma unroll
            for (int c = 0; c < NC; ++c) q[j][c] = c < nc ? qa[(k + j * 4) * qk + c * 16] : 0.f;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int c = 0; c < NC; ++c)
                if (c < nc) acc[c] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], q[j][c], acc[c], 0, 0, 0);
    }
}

// dst = X^T X over L rows, 16 x 16 blocks round the waves; a lane ends with rows lg * 4 .. of one column
__device__ __forceinline__ void small_gram(const float* X, int ld, int L, int S, float* dst, int ldd, int waves) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, li = lane & 15, lg = lane >> 4, sb = S / 16;
    for (int t = wave; t < sb * sb; t += waves) {
        const int m0 = t / sb * 16, n0 = t % sb * 16;
        float4_t acc[1] = {float4_t{0.f, 0.f, 0.f, 0.f}};
        small_product<1>(X + lg * ld + m0 + li, ld, X + lg * ld + n0 + li, ld, L, 1, acc);
#pragma unroll
        for (int e = 0; e < 4; ++e) dst[(m0 + lg * 4 + e) * ldd + n0 + li] = acc[0][e];
    }
}
// B = a I + b A + c A A
__device__ __forceinline__ void small_b(const float* A, float* B, int ld, int S, int waves) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, li = lane & 15, lg = lane >> 4, sb = S / 16;
    for (int t = wave; t < sb * sb; t += waves) {
        const int m0 = t / sb * 16, n0 = t % sb * 16;
        float4_t acc[1] = {float4_t{0.f, 0.f, 0.f, 0.f}};
        small_product<1>(A + (m0 + li) * ld + lg, 1, A + lg * ld + n0 + li, ld, S, 1, acc);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int m = m0 + lg * 4 + e, n = n0 + li;
            B[m * ld + n] = fmaf(NS_B, A[m * ld + n], NS_C * acc[0][e]) + (m == n ? NS_A : 0.f);
        }
    }
}
// X = X B in place: a wave's 16 rows depend on themselves alone
__device__ __forceinline__ void small_apply(float* X, const float* B, int ld, int L, int S, int waves) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, li = lane & 15, lg = lane >> 4, sb = S / 16;
    for (int t = wave; t < L / 16; t += waves) {
        float4_t acc[SMALL_S / 16];
#pragma unroll
        for (int c = 0; c < SMALL_S / 16; ++c) acc[c] = float4_t{0.f, 0.f, 0.f, 0.f};
        small_product<SMALL_S / 16>(X + (t * 16 + li) * ld + lg, 1, B + lg * ld + li, ld, S, sb, acc);
#pragma unroll
        for (int c = 0; c < SMALL_S / 16; ++c)
            if (c < sb) {
#pragma unroll
                for (int e = 0; e < 4; ++e) X[(t * 16 + lg * 4 + e) * ld + c * 16 + li] = acc[c][e];
            }
    }
}

template <bool MUON>
__global__ __launch_bounds__(SMALL_THREADS) void ns_small_kernel(Smalls sm, Ios ios, Hyper h, int steps, float eps) {
    extern __shared__ __attribute__((aligned(16))) float lds[];
    __shared__ double part[SMALL_WAVES];
    const int rows = sm.rows[blockIdx.x], cols = sm.cols[blockIdx.x];
    const Io io = ios.io[blockIdx.x];
    const bool flip = rows < cols;
    const int L = up16(flip ? cols : rows), S = up16(flip ? rows : cols), ld = S + 4;      // + 4: the 16 rows of a fragment on 64 banks
    float* X = lds;                // [L][ld]
    float* A = X + L * ld;         // [S][ld]
    float* B = A + S * ld;         // [S][ld]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const bool skip = MUON && skip_step(h);
    float inv = 1.f, scale = 1.f;
    if constexpr (MUON) {
        inv = h.loss_scale ? h.loss_scale[1] : 1.f;
        scale = clip_scale(h);
    }
    for (int i = threadIdx.x; i < L * ld; i += SMALL_THREADS) X[i] = 0.f;
    __syncthreads();
    double sum = 0;
    for (int i = threadIdx.x; i < rows * cols; i += SMALL_THREADS) {
        const int r = i / cols, c = i - r * cols;
        float v;
        if constexpr (MUON) {
            const float g = (io.g[i] * inv + h.l2 * io.p[i]) * scale, m0 = io.m[i], m1 = h.mu * m0 + g;
            v = h.nesterov ? g + h.mu * m1 : m1;
            io.mo[i] = skip ? m0 : m1;
        } else {
            v = io.g[i];
        }
        X[flip ? c * ld + r : r * ld + c] = v;
        sum = fma((double)v, (double)v, sum);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
    if (lane == 0) part[wave] = sum;
    __syncthreads();
    sum = part[0];
    for (int w = 1; w < SMALL_WAVES; ++w) sum += part[w];
    const double k = 1.0 / (sqrt(sum) + (double)eps);
    for (int i = threadIdx.x; i < L * ld; i += SMALL_THREADS) X[i] = (float)((double)X[i] * k);
    __syncthreads();
    for (int step = 0; step < steps; ++step) {
        small_gram(X, ld, L, S, A, ld, SMALL_WAVES);
        __syncthreads();
        small_b(A, B, ld, S, SMALL_WAVES);
        __syncthreads();
        small_apply(X, B, ld, L, S, SMALL_WAVES);
        __syncthreads();
    }
    for (int i = threadIdx.x; i < rows * cols; i += SMALL_THREADS) {
        const int r = i / cols, c = i - r * cols;
        const float v = X[flip ? c * ld + r : r * ld + c];
        if constexpr (MUON) {
            const float p = io.p[i];
            io.po[i] = skip ? p : p * (1.f - h.lr * h.wd) - h.lr * io.k * v;
        } else {
            io.po[i] = v;
        }
    }
}

// -------------------------------------------------------------------------------------------------------------------- tall
// S <= SMALL_S and L <= TALL_L: tiles of rows, one workgroup each, f32 products as above.  The first launch makes U and each
// tile's part of U^T U; a step is one launch, in which every workgroup adds up all parts of A, makes B, takes its rows of X through
// it and, for the step after, makes its part of X'^T X': 1 + steps launches in place of the general form's 2 + 4 steps.
// One matrix, five steps: 3 x 3552 39 us (general form 111), 1024 x 64 70 (89), 5634 x 42 84 (144), 8192 x 64 134 (173), of which
// the launches alone take 30.  At S = 64 the rest is the f32 matrix cores and, with 32 tiles, each workgroup's 512 KB of parts.
constexpr int TALL_TILES = 32, TALL_ROWS = 64;
struct Tall { int rows, cols, R, tiles, y, slab, head; };      // y [tiles R][S], slab [2][tiles][S][S], head [tiles]
struct Talls { Tall t[CUTIE_MAX_BATCH]; int n; };
// of a tile of U: the sum of squares, and the power of two above its largest value, by which U is divided in its part of U^T U: squares
// of any f32 stay in range
struct Head { double sum; int exp, pad; };

// X (LDS, [R][ld]) <-> y's rows
template <int T> __device__ __forceinline__ void tall_store(const float* X, float* y, int R, int S, int ld) {
    const int q = S / 4;
    for (int i = threadIdx.x; i < R * q; i += T) {
        const int r = i / q, c = (i - r * q) * 4;
        *reinterpret_cast<float4*>(y + (int64_t)r * S + c) = *reinterpret_cast<const float4*>(X + r * ld + c);
    }
}

// A = sum of the tiles' parts, those of the first step times ratio ** 2.  N loads are on their way together; `groups` neighbouring
// lanes (a power of two at S = 16 and 32, else one) share four values.
template <int N, int T>
__device__ __forceinline__ void tall_fold(float* A, const float* slab, const float* ratio, int tiles, int S, int ld, bool first) {
    const int q = S / 4, quads = S * q, groups = S > 32 || quads >= T ? 1 : T / quads, per = (tiles + groups - 1) / groups;
    for (int k = threadIdx.x; k < quads * groups; k += T) {
        const int c4 = k / groups, t0 = (k - c4 * groups) * per, t1 = min(tiles, t0 + per);
        float4_t v = {0.f, 0.f, 0.f, 0.f};
        for (int t = t0; t < t1; t += N) {
            float4_t w[N];
#pragma unroll
            for (int j = 0; j < N; ++j) w[j] = *reinterpret_cast<const float4_t*>(slab + c4 * 4 + (int64_t)min(t + j, t1 - 1) * S * S);
#pragma unroll
            for (int j = 0; j < N; ++j) {
                if (t + j >= t1) continue;
                if (first) w[j] = w[j] * ratio[t + j] * ratio[t + j];
                v += w[j];
            }
        }
        for (int o = 1; o < groups; o <<= 1)
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] += __shfl_xor(v[e], o, 64);
        const int r = c4 / q, c = (c4 - r * q) * 4;
        if (t0 == 0) *reinterpret_cast<float4_t*>(A + r * ld + c) = v;
    }
}

template <int T, bool MUON>
__global__ __launch_bounds__(T) void ns_tall_start_kernel(Talls ts, Ios ios, Starts st, Hyper h, char* ws) {
    extern __shared__ __attribute__((aligned(16))) float lds[];
    __shared__ double part[T / 64];
    __shared__ float top[T / 64];
    const int i = find(st, ts.n, blockIdx.x), tile = blockIdx.x - st.v[i];
    const Tall M = ts.t[i];
    const Io io = ios.io[i];
    const bool flip = M.rows < M.cols;
    const int L = flip ? M.cols : M.rows, s = flip ? M.rows : M.cols, S = up16(s), ld = S + 4;
    const int l0 = tile * M.R, live = min(M.R, L - l0);      // the plan leaves no tile empty
    float* X = lds;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const bool skip = MUON && skip_step(h);
    float inv = 1.f, scale = 1.f;
    if constexpr (MUON) {
        inv = h.loss_scale ? h.loss_scale[1] : 1.f;
        scale = clip_scale(h);
    }
    for (int k = threadIdx.x; k < M.R * ld; k += T) X[k] = 0.f;
    __syncthreads();
    double sum = 0;
    float big = 0.f;
    for (int k = threadIdx.x; k < live * s; k += T) {
        // along the caller's rows
        const int a = flip ? k / live : k / s, b = flip ? k - a * live : k - a * s;
        const int64_t e = flip ? (int64_t)a * M.cols + l0 + b : (int64_t)l0 * s + k;
        float v;
        if constexpr (MUON) {
            const float g = (io.g[e] * inv + h.l2 * io.p[e]) * scale, m0 = io.m[e], m1 = h.mu * m0 + g;
            v = h.nesterov ? g + h.mu * m1 : m1;
            io.mo[e] = skip ? m0 : m1;
        } else {
            v = io.g[e];
        }
        X[flip ? b * ld + a : a * ld + b] = v;
        big = fmaxf(big, fabsf(v));
        sum = fma((double)v, (double)v, sum);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        sum += __shfl_xor(sum, o, 64);
        big = fmaxf(big, __shfl_xor(big, o, 64));
    }
    if (lane == 0) { part[wave] = sum; top[wave] = big; }
    __syncthreads();
    sum = part[0];
    big = top[0];
    for (int w = 1; w < T / 64; ++w) { sum += part[w]; big = fmaxf(big, top[w]); }
    int exp = -200;      // of a tile of zeros: its part counts nothing whatever 1 / eps is
    if (big > 0.f && big <= 3.4028235e38f) (void)frexpf(big, &exp);
    tall_store<T>(X, (float*)at(ws, M.y) + (int64_t)l0 * S, M.R, S, ld);
    __syncthreads();
    for (int k = threadIdx.x; k < M.R * ld; k += T) X[k] = ldexpf(X[k], -exp);
    __syncthreads();
    small_gram(X, ld, M.R, S, (float*)at(ws, M.slab) + (int64_t)tile * S * S, S, T / 64);
    if (threadIdx.x == 0) ((Head*)at(ws, M.head))[tile] = Head{sum, exp, 0};
}

template <int T, bool MUON>
__global__ __launch_bounds__(T) void ns_tall_step_kernel(Talls ts, Ios ios, Starts st, Hyper h, int step, int last, float eps, char* ws) {
    extern __shared__ __attribute__((aligned(16))) float lds[];
    __shared__ float ratio[TALL_TILES];
    const int i = find(st, ts.n, blockIdx.x), tile = blockIdx.x - st.v[i];
    const Tall M = ts.t[i];
    const bool flip = M.rows < M.cols;
    const int L = flip ? M.cols : M.rows, s = flip ? M.rows : M.cols, S = up16(s), ld = S + 4, q = S / 4;
    const int l0 = tile * M.R, live = min(M.R, L - l0);
    float *X = lds, *A = X + M.R * ld, *B = A + S * ld;
    float* y = (float*)at(ws, M.y) + (int64_t)l0 * S;
    double k0 = 1.0;
    if (step == 0) {
        const Head* head = (const Head*)at(ws, M.head);
        double total = 0;
        for (int t = 0; t < M.tiles; ++t) total += head[t].sum;
        k0 = 1.0 / (sqrt(total) + (double)eps);
        if (threadIdx.x < M.tiles) ratio[threadIdx.x] = (float)ldexp(k0, head[threadIdx.x].exp);
        __syncthreads();
    }
    for (int k = threadIdx.x; k < M.R * q; k += T) {
        const int r = k / q, c = (k - r * q) * 4;
        float4 v = *reinterpret_cast<const float4*>(y + (int64_t)r * S + c);
        if (step == 0) v = make_float4((float)(v.x * k0), (float)(v.y * k0), (float)(v.z * k0), (float)(v.w * k0));
        *reinterpret_cast<float4*>(X + r * ld + c) = v;
    }
    // A: the tiles' parts, in order
    const float* slab = (const float*)at(ws, M.slab) + (int64_t)(step & 1) * M.tiles * S * S;
    if (S > 32) tall_fold<16, T>(A, slab, ratio, M.tiles, S, ld, step == 0);
    else tall_fold<4, T>(A, slab, ratio, M.tiles, S, ld, step == 0);
    __syncthreads();
    small_b(A, B, ld, S, T / 64);
    __syncthreads();
    small_apply(X, B, ld, M.R, S, T / 64);
    __syncthreads();
    if (!last) {
        tall_store<T>(X, y, M.R, S, ld);
        small_gram(X, ld, M.R, S, (float*)at(ws, M.slab) + ((int64_t)((step + 1) & 1) * M.tiles + tile) * S * S, S, T / 64);
        return;
    }
    const Io io = ios.io[i];
    const bool skip = MUON && skip_step(h);
    for (int k = threadIdx.x; k < live * s; k += T) {
        const int a = flip ? k / live : k / s, b = flip ? k - a * live : k - a * s;
        const int64_t e = flip ? (int64_t)a * M.cols + l0 + b : (int64_t)l0 * s + k;
        const float v = X[flip ? b * ld + a : a * ld + b];
        if constexpr (MUON) {
            const float p = io.p[e];
            io.po[e] = skip ? p : p * (1.f - h.lr * h.wd) - h.lr * io.k * v;
        } else {
            io.po[e] = v;
        }
    }
}

// ------------------------------------------------------------------------------------------------------------------- host
// All matrices of a call are computed in one form, the cheapest that takes every one of them: a matrix more in a form's launches costs
// little, the launches of a second form come on top (14 filters of which one is 7680 x 64 and one 64 x 18: 355 us; the twelve others
// 329, those two in launches of their own forms 128 and 17 more).
struct NsPlan {
    enum { SMALL, TALL, GENERAL } form;
    Mats ms;                 // GENERAL
    Smalls sm;               // SMALL
    Talls tall;              // TALL
    size_t lds;              // of SMALL and TALL
    bool tall_wide;          // a tall one has S > 32
    Splits gram, square;
    bool fold_square;        // some A A is cut along K
    int fg, fs, fa;          // tile factors (4: 128 x 128, 2: 64 x 64) of the three products
    size_t bytes;
};

// rows of a tile of the tall form: 64 or, where that makes more than TALL_TILES tiles (all of whose parts every workgroup reads), more
inline int tall_rows(int L) {
    int64_t tiles = cdiv(L, TALL_ROWS);
    return up16((int)cdiv(L, tiles > TALL_TILES ? TALL_TILES : tiles));
}

inline int tri_tiles(int Sp, int f) { const int nt = (int)cdiv(Sp, 32 * f); return nt * (nt + 1) / 2; }

// shapes: (rows, cols) of n matrices
inline int ns_plan(const char* who, const int* shapes, int n, NsPlan& p) {
    CUTIE_CHECK_ARG(n >= 1 && n <= CUTIE_MAX_BATCH, "%s: %d matrices (1..%d)", who, n, CUTIE_MAX_BATCH);
    p.fold_square = p.tall_wide = false;
    p.form = NsPlan::SMALL;
    p.lds = 0;
    int64_t broad = 0;      // workgroups of the tall form with S = 64
    for (int i = 0; i < n; ++i) {
        const int r = shapes[2 * i], c = shapes[2 * i + 1], L = r > c ? r : c, S = r > c ? c : r;
        CUTIE_CHECK_ARG(r >= 1 && c >= 1, "%s: matrix %d is %d x %d", who, i, r, c);
        if (S > SMALL_S || L > TALL_L) p.form = NsPlan::GENERAL;
        else if (p.form == NsPlan::SMALL && !is_small(r, c)) p.form = NsPlan::TALL;
        if (S > 48) broad += cdiv(L, tall_rows(L));
    }
    // One round of workgroups: at S = 64 the f32 products of more take longer than the general form (8192 x 64: 4 matrices 149 us,
    // general 223; 32 matrices 708, general 425.  At S = 48 32 of 7079 x 35 take 333, general 340)
    if (p.form == NsPlan::TALL && broad > 256) p.form = NsPlan::GENERAL;
    size_t off = 0;      // of the workspace, in units of 256 bytes
    auto take = [&](int64_t bytes) {
        const size_t at = off;
        off += (size_t)cdiv(bytes, 256);
        return (int)at;
    };
    p.sm.n = p.tall.n = p.ms.n = n;
    if (p.form == NsPlan::SMALL) {
        for (int i = 0; i < n; ++i) {
            p.sm.rows[i] = shapes[2 * i];
            p.sm.cols[i] = shapes[2 * i + 1];
            const size_t lds = small_lds(p.sm.rows[i], p.sm.cols[i]);
            if (lds > p.lds) p.lds = lds;
        }
        p.bytes = 256;      // none needed; a size all the same
        return CUTIE_OK;
    }
    if (p.form == NsPlan::TALL) {
        for (int i = 0; i < n; ++i) {
            const int r = shapes[2 * i], c = shapes[2 * i + 1], L = r > c ? r : c, S = up16(r > c ? c : r);
            Tall& t = p.tall.t[i];
            t.rows = r;
            t.cols = c;
            t.R = tall_rows(L);
            t.tiles = (int)cdiv(L, t.R);
            t.y = take((int64_t)t.tiles * t.R * S * 4);
            t.slab = take((int64_t)2 * t.tiles * S * S * 4);
            t.head = take((int64_t)t.tiles * sizeof(Head));
            const size_t lds = ((size_t)t.R + 2 * S) * (S + 4) * sizeof(float);
            if (lds > p.lds) p.lds = lds;
            if (S > 32) p.tall_wide = true;
        }
        p.bytes = off * 256;
        return CUTIE_OK;
    }
    for (int i = 0; i < n; ++i) {
        const int r = shapes[2 * i], c = shapes[2 * i + 1];
        const int64_t Lp = cdiv(r > c ? r : c, 64) * 64, Sp = cdiv(r > c ? c : r, 64) * 64;
        CUTIE_CHECK_ARG(Lp * Sp < ((int64_t)1 << 29), "%s: matrix %d is %d x %d (padded to multiples of 64, below 2^29 values)", who, i, r, c);
        Mat& m = p.ms.m[i];
        m.rows = r;
        m.cols = c;
        m.Lp = (int)Lp;
        m.Sp = (int)Sp;
    }
    // X B and A A: the 128 tile where it gives every CU a workgroup (A A: with K cut into pieces of eight steps; 14 filters 355 us,
    // with the 64 tile for X B 397; 2048 x 8192 1.75 ms, 2.46).  X^T X: where it gives each four (2048 x 8192 1.75 ms, 64 tile 2.05;
    // 32 of 3840 x 256 789 us, 870), else the 64 tile, which wastes less of the diagonal's tiles (14 filters 355 us, 128 tile 379;
    // two of 4608 x 512 296, 337).  K is cut for two workgroups a CU (512 / tiles: 14 filters 355 us, 2048 x 8192 1.75 ms, 32 of
    // 3840 x 256 789 us; 256 / tiles 429, 2.14, 861; 1024 / tiles 349, 1.77, 843)
    int64_t tg = 0, ts = 0, ta = 0;
    for (int i = 0; i < n; ++i) {
        const Mat& m = p.ms.m[i];
        tg += (int64_t)tri_tiles(m.Sp, 4) * cdiv(m.Lp, 256);
        ts += (int64_t)tri_tiles(m.Sp, 4) * cdiv(m.Sp, 256);
        ta += cdiv(m.Lp, 128) * cdiv(m.Sp, 128);
    }
    p.fg = tg >= 1024 ? 4 : 2;
    p.fs = ts >= 256 ? 4 : 2;
    p.fa = ta >= 256 ? 4 : 2;
    int64_t ng = 0, nq = 0;
    for (int i = 0; i < n; ++i) { ng += tri_tiles(p.ms.m[i].Sp, p.fg); nq += tri_tiles(p.ms.m[i].Sp, p.fs); }
    for (int i = 0; i < n; ++i) {
        Mat& m = p.ms.m[i];
        auto cut = [](int64_t want, int steps) {      // at least four K steps a part
            int64_t s = want < steps / 4 ? want : steps / 4;
            return (short)(s < 1 ? 1 : (s > 64 ? 64 : s));
        };
        p.gram.v[i] = cut(512 / ng, m.Lp / 32);
        // A A is cut only where K is long: at S = 256 its eight steps take less than a fold of the parts
        p.square.v[i] = m.Sp > 512 ? cut(512 / nq, m.Sp / 32) : (short)1;
        if (p.square.v[i] > 1) p.fold_square = true;
        const int64_t y = (int64_t)m.Lp * m.Sp * 4, a = (int64_t)m.Sp * m.Sp * 4;
        const int64_t sg = (int64_t)p.gram.v[i] * tri_tiles(m.Sp, p.fg) * (32 * p.fg) * (32 * p.fg) * 4;
        const int64_t ss = (int64_t)p.square.v[i] * tri_tiles(m.Sp, p.fs) * (32 * p.fs) * (32 * p.fs) * 4;
        m.y0 = take(y);
        m.y1 = take(y);
        m.a = take(a);
        m.b = take(a);
        m.slab = take(sg > ss ? sg : ss);
        m.part = take(cdiv((int64_t)m.rows * m.cols, NORM_CHUNK) * 8);
    }
    CUTIE_CHECK_ARG(off < ((size_t)1 << 31), "%s: the matrices of one call are too large together", who);
    p.bytes = off * 256;
    return CUTIE_OK;
}

template <typename Count> inline unsigned starts(const NsPlan& p, Starts& st, Count count) {
    int64_t t = 0;
    for (int i = 0; i < p.ms.n; ++i) {
        st.v[i] = (int)t;
        t += count(p.ms.m[i], i);
    }
    st.v[p.ms.n] = (int)t;
    return (unsigned)t;
}

template <int F, bool GRAM> inline void ns_sym(const NsPlan& p, int which, char* ws, hipStream_t stream) {
    const Splits& sp = GRAM ? p.gram : p.square;
    Starts st;
    const unsigned g = starts(p, st, [&](const Mat& m, int i) { return (int64_t)tri_tiles(m.Sp, F) * sp.v[i]; });
    hipLaunchKernelGGL((ns_sym_kernel<F, GRAM>), dim3(g), dim3(256), 0, stream, p.ms, st, sp, which, ws);
    if (!GRAM && !p.fold_square) return;
    const unsigned f = starts(p, st, [&](const Mat& m, int) { return (int64_t)tri_tiles(m.Sp, F) * F * F; });
    hipLaunchKernelGGL((ns_fold_kernel<F, GRAM>), dim3(f), dim3(256), 0, stream, p.ms, st, sp, ws);
}

template <int F, bool MUON>
inline void ns_apply(const NsPlan& p, const Ios& ios, const Hyper& h, int which, bool last, char* ws, hipStream_t stream) {
    Starts st;
    const unsigned g = starts(p, st, [&](const Mat& m, int) { return cdiv(m.Lp, 32 * F) * cdiv(m.Sp, 32 * F); });
    if (last) hipLaunchKernelGGL((ns_apply_kernel<F, true, MUON>), dim3(g), dim3(256), 0, stream, p.ms, ios, st, h, which, ws);
    else hipLaunchKernelGGL((ns_apply_kernel<F, false, false>), dim3(g), dim3(256), 0, stream, p.ms, ios, st, h, which, ws);
}

template <int T, bool MUON>
inline int ns_tall(const NsPlan& p, const Ios& ios, const Starts& st, const Hyper& h, int wgs, int steps, float eps, char* ws, hipStream_t stream) {
    CUTIE_ENSURE_LDS((ns_tall_start_kernel<T, MUON>), p.lds);
    CUTIE_ENSURE_LDS((ns_tall_step_kernel<T, MUON>), p.lds);
    hipLaunchKernelGGL((ns_tall_start_kernel<T, MUON>), dim3(wgs), dim3(T), p.lds, stream, p.tall, ios, st, h, ws);
    CUTIE_CHECK_LAUNCH();
    for (int k = 0; k < steps; ++k) {
        hipLaunchKernelGGL((ns_tall_step_kernel<T, MUON>), dim3(wgs), dim3(T), p.lds, stream, p.tall, ios, st, h, k, (int)(k + 1 == steps),
                           eps, ws);
        CUTIE_CHECK_LAUNCH();
    }
    return CUTIE_OK;
}

template <bool MUON>
inline int ns_run(const NsPlan& p, const Ios& ios, const Hyper& h, int steps, float eps, char* ws, hipStream_t stream) {
    static_assert(sizeof(Mats) + sizeof(Ios) + sizeof(Starts) + sizeof(Hyper) + 64 < 4096, "kernel arguments");
    static_assert(sizeof(Talls) + sizeof(Ios) + sizeof(Starts) + sizeof(Hyper) + 64 < 4096, "kernel arguments");
    if (p.form == NsPlan::SMALL) {
        CUTIE_ENSURE_LDS(ns_small_kernel<MUON>, p.lds);
        hipLaunchKernelGGL((ns_small_kernel<MUON>), dim3((unsigned)p.sm.n), dim3(SMALL_THREADS), p.lds, stream, p.sm, ios, h, steps, eps);
        CUTIE_CHECK_LAUNCH();
        return CUTIE_OK;
    }
    Starts st;
    if (p.form == NsPlan::TALL) {
        int wgs = 0;
        for (int i = 0; i < p.tall.n; ++i) {
            st.v[i] = wgs;
            wgs += p.tall.t[i].tiles;
        }
        st.v[p.tall.n] = wgs;
        // 16 waves where a workgroup has a CU to itself and its products are long enough for them (5634 x 42: 84 us, 8 waves 104;
        // 32 of 7079 x 35: 401 us, 8 waves 333; 11 x 5496: 49, 8 waves 46)
        return p.tall_wide && wgs <= 256 ? ns_tall<1024, MUON>(p, ios, st, h, wgs, steps, eps, ws, stream)
                                         : ns_tall<512, MUON>(p, ios, st, h, wgs, steps, eps, ws, stream);
    }
    const unsigned g0 = starts(p, st, [](const Mat& m, int) { return cdiv((int64_t)m.rows * m.cols, NORM_CHUNK); });
    hipLaunchKernelGGL((ns_norm_kernel<MUON>), dim3(g0), dim3(256), 0, stream, p.ms, ios, st, h, ws);
    CUTIE_CHECK_LAUNCH();
    const unsigned g1 = starts(p, st, [](const Mat& m, int) { return (int64_t)(m.Lp / 64) * (m.Sp / 64); });
    hipLaunchKernelGGL((ns_start_kernel<MUON>), dim3(g1), dim3(256), 0, stream, p.ms, ios, st, eps, ws);
    CUTIE_CHECK_LAUNCH();
    for (int k = 0; k < steps; ++k) {
        const int which = k & 1;
        if (p.fg == 4) ns_sym<4, true>(p, which, ws, stream);
        else ns_sym<2, true>(p, which, ws, stream);
        if (p.fs == 4) ns_sym<4, false>(p, which, ws, stream);
        else ns_sym<2, false>(p, which, ws, stream);
        if (p.fa == 4) ns_apply<4, MUON>(p, ios, h, which, k + 1 == steps, ws, stream);
        else ns_apply<2, MUON>(p, ios, h, which, k + 1 == steps, ws, stream);
        CUTIE_CHECK_LAUNCH();
    }
    return CUTIE_OK;
}

inline int ns_common(const char* who, int steps, float eps, const NsPlan& p, const void* ws, size_t bytes) {
    CUTIE_CHECK_ARG(steps >= 1 && steps <= 32, "%s: steps=%d (1..32)", who, steps);
    CUTIE_CHECK_ARG(eps > 0.f, "%s: eps=%g must be positive", who, (double)eps);
    if (!ws || bytes < p.bytes || (reinterpret_cast<uintptr_t>(ws) & 255)) {
        set_error("%s: workspace %zu < %zu (or not 256-byte aligned)", who, ws ? bytes : 0, p.bytes);
        return CUTIE_E_WORKSPACE;
    }
    return CUTIE_OK;
}
inline bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3) == 0; }

// An output may be the input of its own place (ins[in]), and shares no byte with any other tensor of the call.
struct Target { Dense t; int in; };
inline int ns_disjoint(const char* who, const Target* outs, int no, const Dense* ins, int ni, int per, Dense space) {
    for (int i = 0; i < no; ++i) {
        const Target& o = outs[i];
        bool bad = false;
        for (int j = 0; j < i; ++j) bad |= dense_meet(o.t, outs[j].t);
        for (int j = 0; j < ni; ++j) bad |= dense_meet(o.t, ins[j]) && !(j == o.in && ins[j].p == o.t.p);
        CUTIE_CHECK_ARG(!bad, "%s: matrix %d: an output overlaps another tensor of the call", who, i / per);
    }
    bool bad = false;
    for (int i = 0; i < no; ++i) bad |= dense_meet(space, outs[i].t);
    for (int j = 0; j < ni; ++j) bad |= dense_meet(space, ins[j]);
    CUTIE_CHECK_ARG(!bad, "%s: the workspace overlaps another tensor of the call", who);
    return CUTIE_OK;
}
}  // namespace

extern "C" size_t cutie_orthogonalize_workspace_bytes(const int* shapes, int n) {
    NsPlan p;
    if (!shapes || ns_plan("orthogonalize_workspace_bytes", shapes, n, p) != CUTIE_OK) return 0;
    return p.bytes;
}

extern "C" int cutie_orthogonalize_batched(const cutie_orth_desc* descs, int n, int steps, float eps, void* workspace,
                                           size_t workspace_bytes, cutie_stream_t stream_) {
    CUTIE_CHECK_ARG(descs && n >= 1 && n <= CUTIE_MAX_BATCH, "orthogonalize: %d matrices (1..%d)", n, CUTIE_MAX_BATCH);
    int shapes[2 * CUTIE_MAX_BATCH];
    Ios ios = {};
    for (int i = 0; i < n; ++i) {
        shapes[2 * i] = descs[i].rows;
        shapes[2 * i + 1] = descs[i].cols;
        CUTIE_CHECK_ARG(descs[i].g && descs[i].out && aligned4(descs[i].g) && aligned4(descs[i].out),
                        "orthogonalize: matrix %d: null or misaligned pointer", i);
        ios.io[i].g = descs[i].g;
        ios.io[i].po = descs[i].out;
    }
    NsPlan p;
    if (int e = ns_plan("orthogonalize", shapes, n, p)) return e;
    if (int e = ns_common("orthogonalize", steps, eps, p, workspace, workspace_bytes)) return e;
    Dense ins[CUTIE_MAX_BATCH];
    Target outs[CUTIE_MAX_BATCH];
    for (int i = 0; i < n; ++i) {
        const uint64_t size = (uint64_t)descs[i].rows * descs[i].cols * sizeof(float);
        ins[i] = Dense{descs[i].g, size};
        outs[i] = Target{{descs[i].out, size}, i};
    }
    if (int e = ns_disjoint("orthogonalize", outs, n, ins, n, 1, Dense{workspace, p.bytes})) return e;
    Hyper h = {};
    return ns_run<false>(p, ios, h, steps, eps, (char*)workspace, (hipStream_t)stream_);
}

extern "C" int cutie_muon_step(const cutie_muon_desc* descs, int n, float lr, float momentum, int nesterov, float weight_decay, float l2,
                               int steps, float eps, const float* gnorm_sq, float clip, float grad_scale, const float* loss_scale,
                               const int32_t* invalid, void* workspace, size_t workspace_bytes, cutie_stream_t stream_) {
    CUTIE_CHECK_ARG(descs && n >= 1 && n <= CUTIE_MAX_BATCH, "muon_step: %d matrices (1..%d)", n, CUTIE_MAX_BATCH);
    CUTIE_CHECK_ARG(clip >= 0.f && (clip == 0.f || gnorm_sq), "muon_step: clip=%g needs gnorm_sq (0: no clip)", (double)clip);
    int shapes[2 * CUTIE_MAX_BATCH];
    Ios ios = {};
    for (int i = 0; i < n; ++i) {
        const cutie_muon_desc& d = descs[i];
        shapes[2 * i] = d.rows;
        shapes[2 * i + 1] = d.cols;
        CUTIE_CHECK_ARG(d.p && d.g && d.m && d.p_out && d.m_out && aligned4(d.p) && aligned4(d.g) && aligned4(d.m) && aligned4(d.p_out) &&
                            aligned4(d.m_out), "muon_step: matrix %d: null or misaligned pointer", i);
        ios.io[i] = Io{d.p, d.g, d.m, d.p_out, d.m_out, d.out_scale};
    }
    NsPlan p;
    if (int e = ns_plan("muon_step", shapes, n, p)) return e;
    if (int e = ns_common("muon_step", steps, eps, p, workspace, workspace_bytes)) return e;
    Dense ins[3 * CUTIE_MAX_BATCH + 3];
    Target outs[2 * CUTIE_MAX_BATCH];
    for (int i = 0; i < n; ++i) {
        const cutie_muon_desc& d = descs[i];
        const uint64_t size = (uint64_t)d.rows * d.cols * sizeof(float);
        ins[3 * i] = Dense{d.p, size};
        ins[3 * i + 1] = Dense{d.g, size};
        ins[3 * i + 2] = Dense{d.m, size};
        outs[2 * i] = Target{{d.p_out, size}, 3 * i};
        outs[2 * i + 1] = Target{{d.m_out, size}, 3 * i + 2};
    }
    ins[3 * n] = Dense{gnorm_sq, 4};
    ins[3 * n + 1] = Dense{loss_scale, 8};
    ins[3 * n + 2] = Dense{invalid, 4};
    if (int e = ns_disjoint("muon_step", outs, 2 * n, ins, 3 * n + 3, 2, Dense{workspace, p.bytes})) return e;
    const Hyper h = {lr, momentum, weight_decay, l2, clip, grad_scale, nesterov, gnorm_sq, loss_scale, invalid};
    return ns_run<true>(p, ios, h, steps, eps, (char*)workspace, (hipStream_t)stream_);
}
