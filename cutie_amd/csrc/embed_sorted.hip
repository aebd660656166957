// K16: the embedding lookup with a scale, and its gradient by sorted tokens.
//
//   out[cell][0:E] = scale * table[ids[cell]][0:E]
//   dtable[v][0:E] (+)= scale * sum of dout[cell][0:E] over the cells with ids[cell] == v, in the order of a stable sort
//
// The lookup is a row copy (HBM).  The gradient sorts (id, cell) pairs - a stable radix sort, least significant digit
// first - and adds runs of equal ids: every output row has one owner, no float atomics, the same bits every run, and an id
// that most cells hold (the empty cell of a document grid) costs what any other cells cost.
#include "common.h"

namespace {
using namespace cutie;

template <int DT, int VEC> struct Row {      // VEC elements of a 16-bit or f32 row as f32
    typedef typename elem<DT>::type T;
    static __device__ __forceinline__ void load(const T* p, float* v) {
        if constexpr (VEC == 1) {
            v[0] = load_as_f32(p);
        } else if constexpr (VEC == 4) {
            const float4 f = load4(p);
            v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
        } else {
            typedef T V __attribute__((ext_vector_type(8)));
            const V q = *reinterpret_cast<const V*>(p);
#pragma unroll
            for (int e = 0; e < 8; ++e) { const T t = q[e]; v[e] = load_as_f32(&t); }
        }
    }
    static __device__ __forceinline__ void store(T* p, const float* v) {
        if constexpr (VEC == 1) {
            store_from_f32(p, v[0]);
        } else if constexpr (VEC == 4) {
            store4(p, make_float4(v[0], v[1], v[2], v[3]));
        } else {
            typedef T V __attribute__((ext_vector_type(8)));
            V q;
#pragma unroll
            for (int e = 0; e < 8; ++e) { T t; store_from_f32(&t, v[e]); q[e] = t; }
            *reinterpret_cast<V*>(p) = q;
        }
    }
};

// `cv` vectors a row, 256 / cv rows side by side (a row wider than 256 vectors takes gridDim.y column blocks)
template <int ODT, int VEC>
__global__ __launch_bounds__(256) void embed_scaled_kernel(const int32_t* __restrict__ ids, int64_t n, const float* __restrict__ table,
                                                           int V, int E, float scale, typename elem<ODT>::type* __restrict__ out,
                                                           int ld, int32_t* __restrict__ oob) {
    const int v0 = blockIdx.y * 256, nv = min(256, E / VEC - v0);
    const int rows = 256 / nv, col = threadIdx.x % nv, sub = threadIdx.x / nv;
    if (sub >= rows) return;
    const int c0 = (v0 + col) * VEC;
    constexpr int U = 4;
    const int64_t step = (int64_t)gridDim.x * rows;
    for (int64_t base = (int64_t)blockIdx.x * rows + sub; base < n; base += U * step) {
        int id[U];
        float v[U][VEC];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t cell = base + u * step;
            id[u] = cell < n ? ids[cell] : -1;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[u][e] = 0.f;
            if (id[u] >= 0 && id[u] < V) {
                const float* p = table + (int64_t)id[u] * E + c0;
                if constexpr (VEC == 1) Row<CUTIE_F32, 1>::load(p, v[u]);
                else if constexpr (VEC == 4) Row<CUTIE_F32, 4>::load(p, v[u]);
                else { Row<CUTIE_F32, 4>::load(p, v[u]); Row<CUTIE_F32, 4>::load(p + 4, v[u] + 4); }
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t cell = base + u * step;
            if (cell >= n) break;
            if (c0 == 0 && (id[u] < 0 || id[u] >= V)) atomicAdd(oob, 1);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                v[u][e] *= scale;
                // the product exists as an f32 before it is narrowed: else the compiler narrows some forms straight out of the
                // multiplier (one rounding instead of two, another f16 next to a tie)
                asm volatile("" : "+v"(v[u][e]));
            }
            Row<ODT, VEC>::store(out + cell * ld + c0, v[u]);
        }
    }
}

// ------------------------------------------------------------------------------------------------------------------- sort
constexpr int ITEMS = 8;                // elements a thread ranks
constexpr int TILE = 256 * ITEMS;       // elements a workgroup ranks in the many-tile form
constexpr int ONE = 1024 * ITEMS;       // elements one workgroup sorts by itself
constexpr int MAX_BITS = 10, MAX_BINS = 1 << MAX_BITS;

// An id outside [0, V) sorts behind every other as the key V and adds to nothing.
__device__ __forceinline__ uint2 first_pair(const int32_t* ids, int64_t i, int V) {
    const int id = ids[i];
    return make_uint2(id >= 0 && id < V ? (unsigned)id : (unsigned)V, (unsigned)i);
}

// lanes of the wave (among `live`) that hold the same digit
__device__ __forceinline__ unsigned long long same_digit(unsigned d, int bits, unsigned long long live) {
    unsigned long long m = live;
    for (int b = 0; b < bits; ++b) {
        const bool one = (d >> b) & 1;
        const unsigned long long bal = __ballot(one);
        m &= one ? bal : ~bal;
    }
    return m;
}

// Rank of each of a thread's elements among the tile's elements of its digit, in element order (element = wave * 64 *
// ITEMS + round * 64 + lane).  cnt[waves][bins] in LDS, cleared here; afterwards cnt[w][d] = elements of digit d in earlier
// waves and total[d] (nullable) = the tile's count.
template <int WAVES>
__device__ __forceinline__ void tile_rank(const unsigned* d, const bool* ok, int bits, unsigned short (*cnt)[MAX_BINS], int* rank,
                                          unsigned* total) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, bins = 1 << bits;
    __syncthreads();
    for (int i = threadIdx.x; i < WAVES * bins; i += WAVES * 64) cnt[i >> bits][i & (bins - 1)] = 0;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ITEMS; ++r) {
        const unsigned long long m = same_digit(d[r], bits, __ballot(ok[r]));
        const int below = __popcll(m & ((1ull << lane) - 1));
        // only this wave touches cnt[w]: the lanes of one digit read the count, then the first of them moves it on
        const int base = ok[r] ? cnt[w][d[r]] : 0;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        if (ok[r] && below == 0) cnt[w][d[r]] = (unsigned short)(base + __popcll(m));
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        rank[r] = base + below;
    }
    __syncthreads();
    for (int b = threadIdx.x; b < bins; b += WAVES * 64) {
        int run = 0;
        for (int k = 0; k < WAVES; ++k) {
            const int t = cnt[k][b];
            cnt[k][b] = (unsigned short)run;
            run += t;
        }
        if (total) total[b] = (unsigned)run;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ITEMS; ++r)
        if (ok[r]) rank[r] += cnt[w][d[r]];
}

// exclusive prefix sums of v[0..bins) in LDS, by the whole workgroup (THREADS >= 256, bins <= MAX_BINS)
template <int THREADS> __device__ __forceinline__ void bin_scan(unsigned* v, int bins, unsigned* wsum) {
    constexpr int PER = MAX_BINS / 256;       // 256 threads take part, PER bins each
    __syncthreads();
    unsigned x[PER], run = 0;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    if (threadIdx.x < 256) {
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            const int b = threadIdx.x * PER + k;
            x[k] = run;
            run += b < bins ? v[b] : 0u;
        }
        unsigned inc = run;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const unsigned t = __shfl_up(inc, o, 64);
            if (lane >= o) inc += t;
        }
        if (lane == 63) wsum[w] = inc;
        run = inc - run;
    }
    __syncthreads();
    if (threadIdx.x < 256) {
        for (int k = 0; k < w; ++k) run += wsum[k];
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            const int b = threadIdx.x * PER + k;
            if (b < bins) v[b] = run + x[k];
        }
    }
    __syncthreads();
}

__device__ __forceinline__ void clear_part(float* dtable, int64_t n, int64_t block, int64_t blocks) {
    const int64_t step = blocks * blockDim.x;
    if (((uintptr_t)dtable & 15) == 0) {
        const int64_t n4 = n >> 2;
        for (int64_t i = block * blockDim.x + threadIdx.x; i < n4; i += step)
            reinterpret_cast<float4*>(dtable)[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int64_t i = (n4 << 2) + block * blockDim.x + threadIdx.x; i < n; i += step) dtable[i] = 0.f;
    } else {
        for (int64_t i = block * blockDim.x + threadIdx.x; i < n; i += step) dtable[i] = 0.f;
    }
}

// block 0 sorts n <= ONE pairs by itself; the other blocks clear the table
__global__ __launch_bounds__(1024) void sort_one_kernel(const int32_t* __restrict__ ids, int n, int V, int passes, int bits,
                                                        uint2* __restrict__ out, float* __restrict__ dtable, int64_t clear) {
    __shared__ unsigned short cnt[16][MAX_BINS];
    __shared__ unsigned base[MAX_BINS];
    __shared__ unsigned wsum[4];
    extern __shared__ uint2 pairs[];      // [n]
    if (blockIdx.x) {
        clear_part(dtable, clear, blockIdx.x - 1, gridDim.x - 1);
        return;
    }
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    uint2 p[ITEMS];
    bool ok[ITEMS];
    unsigned d[ITEMS];
    int rank[ITEMS];
#pragma unroll
    for (int r = 0; r < ITEMS; ++r) {
        const int i = w * 64 * ITEMS + r * 64 + lane;
        ok[r] = i < n;
        p[r] = ok[r] ? first_pair(ids, i, V) : make_uint2(0, 0);
    }
    for (int pass = 0; pass < passes; ++pass) {
        const int shift = pass * bits;
#pragma unroll
        for (int r = 0; r < ITEMS; ++r) d[r] = (p[r].x >> shift) & ((1u << bits) - 1);
        tile_rank<16>(d, ok, bits, cnt, rank, base);
        bin_scan<1024>(base, 1 << bits, wsum);
        if (pass + 1 < passes) {
#pragma unroll
            for (int r = 0; r < ITEMS; ++r)
                if (ok[r]) pairs[base[d[r]] + rank[r]] = p[r];
            __syncthreads();
#pragma unroll
            for (int r = 0; r < ITEMS; ++r)
                if (ok[r]) p[r] = pairs[w * 64 * ITEMS + r * 64 + lane];
        } else {
#pragma unroll
            for (int r = 0; r < ITEMS; ++r)
                if (ok[r]) out[base[d[r]] + rank[r]] = p[r];
        }
    }
}

// counts[bin][tile] of one digit; blocks behind the tiles clear the table (first pass)
template <bool FIRST>
__global__ __launch_bounds__(256) void sort_count_kernel(const int32_t* __restrict__ ids, const uint2* __restrict__ in, int64_t n, int V,
                                                         int shift, int bits, int tiles, unsigned* __restrict__ counts,
                                                         float* __restrict__ dtable, int64_t clear) {
    __shared__ unsigned hist[4][MAX_BINS];
    if ((int)blockIdx.x >= tiles) {
        clear_part(dtable, clear, blockIdx.x - tiles, gridDim.x - tiles);
        return;
    }
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, bins = 1 << bits;
    for (int i = threadIdx.x; i < 4 * bins; i += 256) hist[i >> bits][i & (bins - 1)] = 0;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ITEMS; ++r) {
        const int64_t i = (int64_t)blockIdx.x * TILE + w * 64 * ITEMS + r * 64 + lane;
        const bool ok = i < n;
        unsigned key = 0;
        if (ok) key = FIRST ? first_pair(ids, i, V).x : in[i].x;
        const unsigned d = (key >> shift) & (bins - 1);
        const unsigned long long m = same_digit(d, bits, __ballot(ok));
        if (ok && (m & ((1ull << lane) - 1)) == 0) atomicAdd(&hist[w][d], (unsigned)__popcll(m));
    }
    __syncthreads();
    for (int b = threadIdx.x; b < bins; b += 256)
        counts[(int64_t)b * tiles + blockIdx.x] = hist[0][b] + hist[1][b] + hist[2][b] + hist[3][b];
}

// one wave per bin: counts[bin][tile] becomes the count in earlier tiles, totals[bin] the whole
__global__ __launch_bounds__(256) void sort_scan_kernel(unsigned* __restrict__ counts, int tiles, int bins, unsigned* __restrict__ totals) {
    const int lane = threadIdx.x & 63, b = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (b >= bins) return;
    unsigned run = 0;
    for (int t0 = 0; t0 < tiles; t0 += 64) {
        const int t = t0 + lane;
        const unsigned c = t < tiles ? counts[(int64_t)b * tiles + t] : 0;
        unsigned inc = c;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const unsigned u = __shfl_up(inc, o, 64);
            if (lane >= o) inc += u;
        }
        if (t < tiles) counts[(int64_t)b * tiles + t] = run + inc - c;
        run += __shfl(inc, 63, 64);
    }
    if (lane == 0) totals[b] = run;
}

template <bool FIRST>
__global__ __launch_bounds__(256) void sort_scatter_kernel(const int32_t* __restrict__ ids, const uint2* __restrict__ in, int64_t n, int V,
                                                           int shift, int bits, int tiles, const unsigned* __restrict__ counts,
                                                           const unsigned* __restrict__ totals, uint2* __restrict__ out) {
    __shared__ unsigned short cnt[4][MAX_BINS];
    __shared__ unsigned base[MAX_BINS];
    __shared__ unsigned wsum[4];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, bins = 1 << bits;
    uint2 p[ITEMS];
    bool ok[ITEMS];
    unsigned d[ITEMS];
    int rank[ITEMS];
#pragma unroll
    for (int r = 0; r < ITEMS; ++r) {
        const int64_t i = (int64_t)blockIdx.x * TILE + w * 64 * ITEMS + r * 64 + lane;
        ok[r] = i < n;
        p[r] = !ok[r] ? make_uint2(0, 0) : (FIRST ? first_pair(ids, i, V) : in[i]);
        d[r] = (p[r].x >> shift) & (bins - 1);
    }
    for (int b = threadIdx.x; b < bins; b += 256) base[b] = totals[b];
    bin_scan<256>(base, bins, wsum);
    for (int b = threadIdx.x; b < bins; b += 256) base[b] += counts[(int64_t)b * tiles + blockIdx.x];
    tile_rank<4>(d, ok, bits, cnt, rank, nullptr);
#pragma unroll
    for (int r = 0; r < ITEMS; ++r)
        if (ok[r]) out[base[d[r]] + rank[r]] = p[r];
}

// ------------------------------------------------------------------------------------------------------------------- sums
// A workgroup takes `chunk` = rows * L consecutive pairs, each of its `rows` subgroups (one lane per vector column) L of them
// in order.  A run of equal ids inside a subgroup goes straight to the table.  A run that enters from the left leaves its
// part in slot A, one that starts here and leaves to the right in slot B; the subgroups' slots meet in LDS, the workgroups'
// in the workspace (slots f32 [chunks][2][E], starts[chunk] = 1 where a run leaves to the right), and run_join_kernel adds
// the parts of a run that spans workgroups.
struct SumShape {
    int64_t n;
    int V, E, ld;
    int rows, L;          // subgroups of a workgroup, pairs of a subgroup
    float scale;
    int accumulate;
};

__device__ __forceinline__ void put(float* dtable, const SumShape& s, unsigned key, int c, float v) {
    if (key >= (unsigned)s.V) return;
    float* p = dtable + (int64_t)key * s.E + c;
    const float t = s.scale * v;
    *p = s.accumulate ? *p + t : t;
}

template <int DT, int VEC>
__global__ __launch_bounds__(256) void run_sum_kernel(const uint2* __restrict__ pairs, const typename elem<DT>::type* __restrict__ dout,
                                                      float* __restrict__ dtable, SumShape s, float* __restrict__ slots,
                                                      int* __restrict__ starts) {
    __shared__ float part[2][256 * VEC];
    __shared__ int flags[256];
    const int v0 = blockIdx.y * 256, nv = min(256, s.E / VEC - v0);
    const int col = threadIdx.x % nv, j = threadIdx.x / nv;
    const int c0 = (v0 + col) * VEC, width = nv * VEC;
    const int64_t chunk0 = (int64_t)blockIdx.x * s.rows * s.L;
    const int64_t b = chunk0 + (int64_t)j * s.L;
    if (j < s.rows) {
        int f = 0;
        if (b < s.n) {
            const int64_t e = min(s.n, b + s.L);
            float acc[VEC];
#pragma unroll
            for (int k = 0; k < VEC; ++k) acc[k] = 0.f;
            bool entered = b > 0 && pairs[b - 1].x == pairs[b].x;
            constexpr int U = 4;
            for (int64_t i0 = b; i0 < e; i0 += U) {
                uint2 p[U + 1];
                float v[U][VEC];
#pragma unroll
                for (int u = 0; u <= U; ++u) p[u] = i0 + u < s.n ? pairs[i0 + u] : make_uint2(0xffffffffu, 0);
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (i0 + u < e) Row<DT, VEC>::load(dout + (int64_t)p[u].y * s.ld + c0, v[u]);
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if (i0 + u >= e) break;
#pragma unroll
                    for (int k = 0; k < VEC; ++k) acc[k] += v[u][k];
                    const bool same = p[u].x == p[u + 1].x, end = i0 + u + 1 == e;
                    if (same && !end) continue;
                    const bool leaves = same;
                    if (entered || leaves) {
                        f |= entered ? (leaves ? 3 : 1) : 4;
                        float* q = part[entered ? 0 : 1] + j * width + col * VEC;
#pragma unroll
                        for (int k = 0; k < VEC; ++k) q[k] = acc[k];
                    } else if (p[u].x < (unsigned)s.V) {
                        float* q = dtable + (int64_t)p[u].x * s.E + c0;
                        float t[VEC];
#pragma unroll
                        for (int k = 0; k < VEC; ++k) t[k] = s.scale * acc[k];
                        if (s.accumulate) {
#pragma unroll
                            for (int k = 0; k < VEC; ++k) t[k] += q[k];
                        }
                        if constexpr (VEC == 8) {
                            Row<CUTIE_F32, 4>::store(q, t);
                            Row<CUTIE_F32, 4>::store(q + 4, t + 4);
                        } else {
                            Row<CUTIE_F32, VEC>::store(q, t);
                        }
                    }
                    entered = false;
#pragma unroll
                    for (int k = 0; k < VEC; ++k) acc[k] = 0.f;
                }
            }
        }
        if (col == 0) flags[j] = f;      // 1 slot A, 2 the whole subgroup is inside one run, 4 slot B
    }
    __syncthreads();
    // the subgroups in order: `before` = the open run began before this workgroup
    for (int c = threadIdx.x; c < width; c += 256) {
        float acc = 0.f;
        bool open = false, before = false;
        for (int k = 0; k < s.rows; ++k) {
            const int f = flags[k];
            if (f & 1) {
                if (k == 0) before = true;
                acc += part[0][k * width + c];
                open = (f & 2) != 0;
                if (!open) {
                    if (before) slots[((int64_t)blockIdx.x * 2) * s.E + v0 * VEC + c] = acc;
                    else put(dtable, s, pairs[chunk0 + (int64_t)k * s.L].x, v0 * VEC + c, acc);
                    acc = 0.f;
                    before = false;
                }
            }
            if (f & 4) {
                acc = part[1][k * width + c];
                open = true;
                before = false;
            }
        }
        if (open) slots[((int64_t)blockIdx.x * 2 + (before ? 0 : 1)) * s.E + v0 * VEC + c] = acc;
        if (c == 0 && v0 == 0) starts[blockIdx.x] = open && !before;
    }
}

// one workgroup per chunk and column block: where a run starts in this chunk and leaves it, the sum of its parts, eight
// chunks apart in each of eight lanes, the eight sums in lane order
__global__ __launch_bounds__(256) void run_join_kernel(const uint2* __restrict__ pairs, float* __restrict__ dtable, SumShape s,
                                                       const float* __restrict__ slots, const int* __restrict__ starts) {
    __shared__ float sh[8][32];
    const int64_t w = blockIdx.x, chunk = (int64_t)s.rows * s.L;
    if (!starts[w]) return;
    const unsigned key = pairs[(w + 1) * chunk - 1].x;
    if (key >= (unsigned)s.V) return;
    int64_t lo = (w + 1) * chunk, hi = s.n;      // first pair behind the run: pairs[lo] belongs to it
    while (hi - lo > 1) {
        const int64_t mid = (lo + hi) >> 1;
        if (pairs[mid].x == key) lo = mid;
        else hi = mid;
    }
    const int64_t last = lo / chunk;
    const int el = threadIdx.x & 31, part = threadIdx.x >> 5;
    const int c = blockIdx.y * 32 + el;
    float t = 0.f;
    if (c < s.E) {
        if (part == 0) t = slots[(w * 2 + 1) * s.E + c];
#pragma unroll 4
        for (int64_t k = w + 1 + part; k <= last; k += 8) t += slots[k * 2 * s.E + c];
    }
    sh[part][el] = t;
    __syncthreads();
    if (part || c >= s.E) return;
    t = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) t += sh[k][el];
    put(dtable, s, key, c, t);
}

// ------------------------------------------------------------------------------------------------------------------- host
struct SortPlan { int passes, bits, tiles; bool one; };
inline SortPlan sort_plan(int64_t n, int V) {
    SortPlan p;
    int need = 1;
    while (need < 31 && ((int64_t)1 << need) <= V) ++need;       // the keys are 0 .. V
    p.passes = (need + MAX_BITS - 1) / MAX_BITS;
    p.bits = (need + p.passes - 1) / p.passes;
    p.one = n <= ONE;
    p.tiles = (int)cdiv(n, TILE);
    return p;
}

struct SumPlan { int vec, rows, L, ncol; int64_t chunks; };
inline SumPlan sum_plan(int64_t n, int E, int vec) {
    SumPlan p;
    p.vec = vec;
    const int cv = E / vec;
    p.ncol = (int)cdiv(cv, 256);
    p.rows = 256 / (cv < 256 ? cv : 256);
    const int want = n <= 65536 ? 64 : (n <= 262144 ? 256 : 512);       // pairs of a workgroup
    p.L = (int)cdiv(want, p.rows);
    if (p.L < 4) p.L = 4;
    p.chunks = cdiv(n, (int64_t)p.rows * p.L);
    return p;
}

struct GradSpace { size_t a, b, counts, totals, slots, starts, total; };
inline GradSpace grad_space(int64_t n, int V, int E) {
    GradSpace w;
    auto up = [](size_t x) { return (x + 255) / 256 * 256; };
    const SortPlan sp = sort_plan(n, V);
    const size_t pairs = up((size_t)n * sizeof(uint2));
    int64_t chunks = 0;       // whichever vector width the call will take
    for (int vec : {1, 4, 8})
        if (E % vec == 0) {
            const int64_t c = sum_plan(n, E, vec).chunks;
            if (c > chunks) chunks = c;
        }
    w.a = 0;
    w.b = pairs;
    w.counts = w.b + (sp.one ? 0 : pairs);
    w.totals = w.counts + (sp.one ? 0 : up(((size_t)sp.tiles << sp.bits) * sizeof(unsigned)));
    w.slots = w.totals + (sp.one ? 0 : up(MAX_BINS * sizeof(unsigned)));
    w.starts = w.slots + up((size_t)chunks * 2 * E * sizeof(float));
    w.total = w.starts + up((size_t)chunks * sizeof(int));
    return w;
}

inline int row_vec(int dt, int E, const void* rows, int ld, const void* table) {
    const int es = dt == CUTIE_F32 ? 4 : 2;
    if (E % 4 || !aligned16(table)) return 1;
    if (es == 2 && E % 8 == 0 && ld % 8 == 0 && aligned16(rows)) return 8;
    return ld % 4 == 0 && reinterpret_cast<uintptr_t>(rows) % (uintptr_t)(4 * es) == 0 ? 4 : 1;
}

constexpr int64_t MAX_CELLS = (int64_t)1 << 30;

inline int embed_check(const char* who, int64_t n, int V, int E, int ld, int dt) {
    CUTIE_CHECK_ARG(n >= 0 && n <= MAX_CELLS && V >= 1 && V < (1 << 30) && E >= 1 && E <= 65536,
                    "%s: n_cells=%lld (at most 2^30) V=%d (below 2^30) E=%d (at most 65536)", who, (long long)n, V, E);
    CUTIE_CHECK_ARG(ld >= E, "%s: leading dimension %d < E=%d", who, ld, E);
    CUTIE_CHECK_ARG(dt == CUTIE_F32 || dt == CUTIE_BF16 || dt == CUTIE_F16, "%s: unknown dtype %d", who, dt);
    return CUTIE_OK;
}
}  // namespace

extern "C" int cutie_embed_scaled_fwd(const int32_t* ids, int64_t n_cells, const float* table, int V, int E, float scale, void* out,
                                      int ld_out, int out_dtype, int32_t* oob_count, cutie_stream_t stream_) {
    hipStream_t stream = (hipStream_t)stream_;
    if (int e = embed_check("embed_scaled_fwd", n_cells, V, E, ld_out, out_dtype)) return e;
    if (n_cells == 0) return CUTIE_OK;
    CUTIE_CHECK_ARG(ids && table && out && oob_count, "embed_scaled_fwd: null pointer");
    const int es = out_dtype == CUTIE_F32 ? 4 : 2;
    CUTIE_CHECK_ARG(((uintptr_t)out % es) == 0 && ((uintptr_t)table % 4) == 0 && ((uintptr_t)ids % 4) == 0,
                    "embed_scaled_fwd: misaligned pointers");
    const int vec = row_vec(out_dtype, E, out, ld_out, table);
    const int cv = E / vec, rows = 256 / (cv < 256 ? cv : 256);
    int64_t g = cdiv(n_cells, (int64_t)rows * 4);
    if (g > 8192) g = 8192;
    const dim3 grid((unsigned)g, (unsigned)cdiv(cv, 256));
    CUTIE_DISPATCH_DTYPE(out_dtype, DT, {
        typedef typename elem<DT>::type T;
        auto go = [&](auto kern) {
            hipLaunchKernelGGL(kern, grid, dim3(256), 0, stream, ids, n_cells, table, V, E, scale, (T*)out, ld_out, oob_count);
        };
        if constexpr (DT != CUTIE_F32) {
            if (vec == 8) go(embed_scaled_kernel<DT, 8>);
        }
        if (vec == 4) go(embed_scaled_kernel<DT, 4>);
        if (vec == 1) go(embed_scaled_kernel<DT, 1>);
    });
    CUTIE_CHECK_LAUNCH();
    return CUTIE_OK;
}

extern "C" size_t cutie_embed_grad_sorted_workspace_bytes(int64_t n_cells, int V, int E) {
    if (n_cells < 1 || n_cells > MAX_CELLS || V < 1 || V >= (1 << 30) || E < 1 || E > 65536) return 0;
    return grad_space(n_cells, V, E).total;
}

extern "C" int cutie_embed_grad_sorted(const int32_t* ids, int64_t n_cells, const void* dout, int ld_dout, int dout_dtype, float scale,
                                       float* dtable, int V, int E, int accumulate, void* workspace, size_t workspace_bytes,
                                       cutie_stream_t stream_) {
    hipStream_t stream = (hipStream_t)stream_;
    if (int e = embed_check("embed_grad_sorted", n_cells, V, E, ld_dout, dout_dtype)) return e;
    CUTIE_CHECK_ARG(dtable && (n_cells == 0 || (ids && dout)), "embed_grad_sorted: null pointer");
    const int es = dout_dtype == CUTIE_F32 ? 4 : 2;
    CUTIE_CHECK_ARG(((uintptr_t)dout % es) == 0 && ((uintptr_t)dtable % 4) == 0 && ((uintptr_t)ids % 4) == 0,
                    "embed_grad_sorted: misaligned pointers");
    const int64_t clear = accumulate ? 0 : (int64_t)V * E;
    int64_t fill = cdiv(clear, 4096);
    if (fill > 1024) fill = 1024;
    const GradSpace w = n_cells ? grad_space(n_cells, V, E) : GradSpace{};
    if (n_cells && (!workspace || workspace_bytes < w.total || !aligned16(workspace))) {
        set_error("embed_grad_sorted: workspace %zu < %zu (or not 16-byte aligned)", workspace ? workspace_bytes : 0, w.total);
        return CUTIE_E_WORKSPACE;
    }
    if (n_cells == 0) {
        if (fill) {
            hipLaunchKernelGGL(sort_one_kernel, dim3((unsigned)fill + 1), dim3(1024), 0, stream, ids, 0, V, 0, 1, (uint2*)nullptr, dtable, clear);
            CUTIE_CHECK_LAUNCH();
        }
        return CUTIE_OK;
    }
    char* ws = (char*)workspace;
    const SortPlan sp = sort_plan(n_cells, V);
    uint2* sorted;
    if (sp.one) {
        sorted = (uint2*)(ws + w.a);
        const size_t lds = sp.passes > 1 ? (size_t)n_cells * sizeof(uint2) : 0;
        CUTIE_ENSURE_LDS(sort_one_kernel, ONE * sizeof(uint2));
        hipLaunchKernelGGL(sort_one_kernel, dim3((unsigned)fill + 1), dim3(1024), lds, stream, ids, (int)n_cells, V, sp.passes, sp.bits,
                           sorted, dtable, clear);
        CUTIE_CHECK_LAUNCH();
    } else {
        uint2* buf[2] = {(uint2*)(ws + w.a), (uint2*)(ws + w.b)};
        unsigned* counts = (unsigned*)(ws + w.counts);
        unsigned* totals = (unsigned*)(ws + w.totals);
        const int bins = 1 << sp.bits;
        for (int pass = 0; pass < sp.passes; ++pass) {
            const uint2* in = pass ? buf[(pass - 1) & 1] : nullptr;
            uint2* out = buf[pass & 1];
            const int shift = pass * sp.bits;
            const unsigned count_blocks = (unsigned)sp.tiles + (pass == 0 ? (unsigned)fill : 0u);
            if (pass == 0)
                hipLaunchKernelGGL(sort_count_kernel<true>, dim3(count_blocks), dim3(256), 0, stream, ids, in, n_cells, V, shift, sp.bits,
                                   sp.tiles, counts, dtable, clear);
            else
                hipLaunchKernelGGL(sort_count_kernel<false>, dim3(count_blocks), dim3(256), 0, stream, ids, in, n_cells, V, shift, sp.bits,
                                   sp.tiles, counts, dtable, (int64_t)0);
            hipLaunchKernelGGL(sort_scan_kernel, dim3((unsigned)cdiv(bins, 4)), dim3(256), 0, stream, counts, sp.tiles, bins, totals);
            if (pass == 0)
                hipLaunchKernelGGL(sort_scatter_kernel<true>, dim3((unsigned)sp.tiles), dim3(256), 0, stream, ids, in, n_cells, V, shift,
                                   sp.bits, sp.tiles, counts, totals, out);
            else
                hipLaunchKernelGGL(sort_scatter_kernel<false>, dim3((unsigned)sp.tiles), dim3(256), 0, stream, ids, in, n_cells, V, shift,
                                   sp.bits, sp.tiles, counts, totals, out);
            CUTIE_CHECK_LAUNCH();
        }
        sorted = buf[(sp.passes - 1) & 1];
    }
    const SumPlan p = sum_plan(n_cells, E, row_vec(dout_dtype, E, dout, ld_dout, dtable));
    SumShape s;
    s.n = n_cells; s.V = V; s.E = E; s.ld = ld_dout; s.rows = p.rows; s.L = p.L; s.scale = scale; s.accumulate = accumulate;
    float* slots = (float*)(ws + w.slots);
    int* starts = (int*)(ws + w.starts);
    CUTIE_DISPATCH_DTYPE(dout_dtype, DT, {
        typedef typename elem<DT>::type T;
        auto go = [&](auto kern) {
            hipLaunchKernelGGL(kern, dim3((unsigned)p.chunks, (unsigned)p.ncol), dim3(256), 0, stream, sorted, (const T*)dout, dtable, s,
                               slots, starts);
        };
        if constexpr (DT != CUTIE_F32) {
            if (p.vec == 8) go(run_sum_kernel<DT, 8>);
        }
        if (p.vec == 4) go(run_sum_kernel<DT, 4>);
        if (p.vec == 1) go(run_sum_kernel<DT, 1>);
    });
    CUTIE_CHECK_LAUNCH();
    hipLaunchKernelGGL(run_join_kernel, dim3((unsigned)p.chunks, (unsigned)cdiv(E, 32)), dim3(256), 0, stream, sorted, dtable, s, slots,
                       starts);
    CUTIE_CHECK_LAUNCH();
    return CUTIE_OK;
}
