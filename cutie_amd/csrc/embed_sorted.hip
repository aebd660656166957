// K16: the embedding lookup with a scale, and its gradient by sorted tokens.
//
//   out[cell][0:E] = scale * table[ids[cell]][0:E]
//   dtable[v][0:E] (+)= scale * sum of dout[cell][0:E] over the cells with ids[cell] == v, in the order of a stable sort
//
// Measured (MI355X), inputs that change from call to call: lookup 131072 x 128 f16 9 us, 500009 x 512 bf16 187 us (4.1 TB/s of the
// 760 MB it must move; 156 us on the same inputs again); gradient 131072 x 128 f16, V 18000, 94 % of the cells on one id: 49 us in six
// launches (27 us the two passes of the sort, 15 the sums, 8 the join); 500009 x 512 bf16, V 120000: 228 us, of which the sums 155
// (4.9 TB/s of the 760 MB).  The gradient by float atomics of embed.hip is faster on the first - back to back on one input 21 us
// against 46 - in an order of its own every run; a train step of CUTIE-ASPP on 32 documents has 7.55 ms with it, 7.56 with this one.
//
// The lookup is a row copy (HBM).  The gradient sorts (id, cell) pairs - a stable radix sort, least significant digit
// first - and adds runs of equal ids: every output row has one owner, no float atomics, the same bits every run, and an id
// that most cells hold (the empty cell of a document grid) costs what any other cells cost.
#include "common.h"

namespace {
using namespace cutie;

// VEC f32 values at an address aligned to 16 bytes (VEC >= 4)
template <int VEC> __device__ __forceinline__ void load_f32(const float* p, float* v) {
    if constexpr (VEC == 1) v[0] = *p;
    else {
#pragma unroll
        for (int e = 0; e < VEC; e += 4) {
            const float4 f = *reinterpret_cast<const float4*>(p + e);
            v[e] = f.x; v[e + 1] = f.y; v[e + 2] = f.z; v[e + 3] = f.w;
        }
    }
}
template <int VEC> __device__ __forceinline__ void store_f32(float* p, const float* v) {
    if constexpr (VEC == 1) *p = v[0];
    else {
#pragma unroll
        for (int e = 0; e < VEC; e += 4) *reinterpret_cast<float4*>(p + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
    }
}

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
            if (id[u] >= 0 && id[u] < V) load_f32<VEC>(table + (int64_t)id[u] * E + c0, v[u]);
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
            Pack<ODT, VEC> q;
#pragma unroll
            for (int e = 0; e < VEC; ++e) q.set(e, v[u][e]);
            q.store_nt(out + cell * ld + c0);      // 500009 x 512 bf16: 156 us, 197 through the caches; 131072 x 128: equal
        }
    }
}

// ------------------------------------------------------------------------------------------------------------------- sort
constexpr int ITEMS = 4;                // elements a thread ranks in the many-tile form
constexpr int TILE = 1024 * ITEMS;      // elements a workgroup ranks there
constexpr int SELF_TILES = 128;         // up to so many tiles a tile adds up the counts before it by itself; more take sort_scan_kernel
constexpr int ONE = 1024 * 8;           // elements one workgroup sorts by itself (4 or 8 a thread)
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
template <int WAVES, int ITEMS>
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

// one workgroup sorts n <= 1024 ITEMS pairs
template <int ITEMS>
__global__ __launch_bounds__(1024) void sort_one_kernel(const int32_t* __restrict__ ids, int n, int V, int passes, int bits,
                                                        uint2* __restrict__ out) {
    __shared__ unsigned short cnt[16][MAX_BINS];
    __shared__ unsigned base[MAX_BINS];
    __shared__ unsigned wsum[4];
    extern __shared__ uint2 pairs[];      // [n]
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
        tile_rank<16, ITEMS>(d, ok, bits, cnt, rank, base);
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

// counts[tile][bin] of one digit
template <bool FIRST>
__global__ __launch_bounds__(1024) void sort_count_kernel(const int32_t* __restrict__ ids, const uint2* __restrict__ in, int64_t n, int V,
                                                         int shift, int bits, unsigned* __restrict__ counts) {
    __shared__ unsigned hist[4][MAX_BINS];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, bins = 1 << bits;
    for (int i = threadIdx.x; i < 4 * bins; i += 1024) hist[i >> bits][i & (bins - 1)] = 0;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ITEMS; ++r) {
        const int64_t i = (int64_t)blockIdx.x * TILE + w * 64 * ITEMS + r * 64 + lane;
        const bool ok = i < n;
        unsigned key = 0;
        if (ok) key = FIRST ? first_pair(ids, i, V).x : in[i].x;
        const unsigned d = (key >> shift) & (bins - 1);
        const unsigned long long m = same_digit(d, bits, __ballot(ok));
        if (ok && (m & ((1ull << lane) - 1)) == 0) atomicAdd(&hist[w & 3][d], (unsigned)__popcll(m));
    }
    __syncthreads();
    for (int b = threadIdx.x; b < bins; b += 1024)
        counts[((int64_t)blockIdx.x << bits) + b] = hist[0][b] + hist[1][b] + hist[2][b] + hist[3][b];
}

// counts[tile][bin] becomes the count in earlier tiles, totals[bin] the whole: a workgroup takes 16 bins, 64 lanes a bin cut the
// tiles into 64 runs, each lane adds its run, the lanes' sums are scanned, and each lane walks its run again
__global__ __launch_bounds__(1024) void sort_scan_kernel(unsigned* __restrict__ counts, int tiles, int bits, unsigned* __restrict__ totals) {
    __shared__ unsigned sh[64][17];
    const int el = threadIdx.x & 15, part = threadIdx.x >> 4, bin = blockIdx.x * 16 + el, bins = 1 << bits;
    const int per = (tiles + 63) / 64, t0 = min(tiles, part * per), t1 = min(tiles, t0 + per);
    unsigned s = 0;
    if (bin < bins)
        for (int t = t0; t < t1; ++t) s += counts[((int64_t)t << bits) + bin];
    sh[part][el] = s;
    __syncthreads();
    // 16 waves: wave w scans bin w over its 64 parts
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const unsigned own = sh[lane][w];
    unsigned inc = own;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const unsigned u = __shfl_up(inc, o, 64);
        if (lane >= o) inc += u;
    }
    sh[lane][w] = inc - own;
    if (lane == 63 && blockIdx.x * 16 + w < bins) totals[blockIdx.x * 16 + w] = inc;
    __syncthreads();
    if (bin >= bins) return;
    unsigned run = sh[part][el];
    for (int t = t0; t < t1; ++t) {
        unsigned* p = counts + ((int64_t)t << bits) + bin;
        const unsigned c = *p;
        *p = run;
        run += c;
    }
}

// totals NULL: counts are the tiles' own, and each tile adds them up; else as sort_scan_kernel left them
template <bool FIRST>
__global__ __launch_bounds__(1024) void sort_scatter_kernel(const int32_t* __restrict__ ids, const uint2* __restrict__ in, int64_t n, int V,
                                                            int shift, int bits, const unsigned* __restrict__ counts,
                                                            const unsigned* __restrict__ totals, uint2* __restrict__ out) {
    __shared__ unsigned short cnt[16][MAX_BINS];
    __shared__ unsigned base[MAX_BINS], before[MAX_BINS];
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
    if (totals) {
        for (int b = threadIdx.x; b < bins; b += 1024) {
            base[b] = totals[b];
            before[b] = counts[((int64_t)blockIdx.x << bits) + b];
        }
    } else {
        for (int b = threadIdx.x; b < bins; b += 1024) base[b] = before[b] = 0;
        __syncthreads();
        // 1024 / bins groups of threads take every so many tiles; whole numbers, so the order of the additions is no matter
        const int groups = 1024 >> bits, b = threadIdx.x & (bins - 1), tiles = gridDim.x;
        unsigned all = 0, early = 0;
#pragma unroll 8
        for (int t = threadIdx.x >> bits; t < tiles; t += groups) {
            const unsigned c = counts[((int64_t)t << bits) + b];
            all += c;
            early += t < (int)blockIdx.x ? c : 0u;
        }
        if (all) atomicAdd(&base[b], all);
        if (early) atomicAdd(&before[b], early);
    }
    bin_scan<1024>(base, bins, wsum);
    for (int b = threadIdx.x; b < bins; b += 1024) base[b] += before[b];
    tile_rank<16, ITEMS>(d, ok, bits, cnt, rank, nullptr);
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
    int64_t n, chunks;
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

// Rows that no cell names: a wave takes 64 rows, finds their pairs, and clears the rows that have none.  (Clearing the whole table
// first writes the other rows twice: 31 us of 242 at V 120000, E 512.)  The pairs' two ends are searched together, 64 places a
// step: a search is a chain of loads, two here for 4096 pairs where halving takes twelve.
__device__ __forceinline__ void clear_absent(const uint2* pairs, float* dtable, const SumShape& s, int64_t wave) {
    const int lane = threadIdx.x & 63;
    const int64_t row0 = wave * 64;
    if (row0 >= s.V) return;
    int64_t lo[2] = {0, 0}, hi[2] = {s.n, s.n};      // the first pair whose key is not below row0, row0 + 64, lies in [lo, hi]
    while (lo[0] < hi[0] || lo[1] < hi[1]) {
        int64_t step[2];
        bool below[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            step[k] = (hi[k] - lo[k] + 63) >> 6;
            const int64_t i = lo[k] + lane * step[k];
            below[k] = i < hi[k] && (int64_t)pairs[i].x < row0 + 64 * k;
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int64_t c = __popcll(__ballot(below[k])), l = lo[k];      // keys ascend: the first c places are below
            hi[k] = min(hi[k], l + c * step[k]);
            if (c) lo[k] = l + (c - 1) * step[k] + 1;
        }
    }
    unsigned long long here = 0;      // bit r: row0 + r has a pair
    const int64_t first = lo[0], last = lo[1];
    if (last - first <= 256) {
        unsigned got[2] = {0, 0};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int64_t i = first + k * 64 + lane;
            if (i < last) {
                const unsigned r = pairs[i].x - (unsigned)row0;
                got[r >> 5] |= 1u << (r & 31);
            }
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            got[0] |= __shfl_xor(got[0], o, 64);
            got[1] |= __shfl_xor(got[1], o, 64);
        }
        here = ((unsigned long long)got[1] << 32) | got[0];
    } else {      // many pairs: each lane looks for its row
        int64_t l = first, h = last;
        while (l < h) {
            const int64_t mid = (l + h) >> 1;
            if ((int64_t)pairs[mid].x < row0 + lane) l = mid + 1;
            else h = mid;
        }
        here = __ballot(l < last && (int64_t)pairs[l].x == row0 + lane);
    }
    const bool absent = row0 + lane < s.V && !((here >> lane) & 1);
    const bool wide = (s.E & 3) == 0 && (reinterpret_cast<uintptr_t>(dtable) & 15) == 0;
    for (unsigned long long m = __ballot(absent); m; m &= m - 1) {
        float* p = dtable + (wave * 64 + __builtin_ctzll(m)) * s.E;
        if (wide)
            for (int c = lane * 4; c < s.E; c += 256) *reinterpret_cast<float4*>(p + c) = make_float4(0.f, 0.f, 0.f, 0.f);
        else
            for (int c = lane; c < s.E; c += 64) p[c] = 0.f;
    }
}

constexpr int CHUNK_MAX = 1280;      // pairs of a workgroup

template <int DT, int VEC>
__global__ __launch_bounds__(256) void run_sum_kernel(const uint2* __restrict__ pairs, const typename elem<DT>::type* __restrict__ dout,
                                                      float* __restrict__ dtable, SumShape s, float* __restrict__ slots,
                                                      int* __restrict__ starts) {
    __shared__ float part[2][256 * VEC];
    __shared__ int flags[256];
    __shared__ unsigned key[CHUNK_MAX + 2], pos[CHUNK_MAX];      // key[i + 1] is the chunk's pair i; its neighbours outside
    if (blockIdx.x >= s.chunks) {      // workgroups behind the chunks: four waves of rows to clear
        if (blockIdx.y == 0) clear_absent(pairs, dtable, s, ((int64_t)blockIdx.x - s.chunks) * 4 + (threadIdx.x >> 6));
        return;
    }
    const int v0 = blockIdx.y * 256, nv = min(256, s.E / VEC - v0);
    const int col = threadIdx.x % nv, j = threadIdx.x / nv;
    const int c0 = (v0 + col) * VEC, width = nv * VEC;
    const int chunk = s.rows * s.L;
    const int64_t chunk0 = (int64_t)blockIdx.x * chunk;
    for (int i = threadIdx.x; i < chunk + 2; i += 256) {
        const int64_t g = chunk0 + i - 1;
        const uint2 p = g >= 0 && g < s.n ? pairs[g] : make_uint2(0xffffffffu, 0);      // no key: V < 2^30
        key[i] = p.x;
        if (i >= 1 && i <= chunk) pos[i - 1] = p.y;
    }
    __syncthreads();
    if (j < s.rows) {
        int f = 0;
        const int b = j * s.L;
        if (chunk0 + b < s.n) {
            const int e = (int)min((int64_t)(b + s.L), s.n - chunk0);
            float acc[VEC];
#pragma unroll
            for (int k = 0; k < VEC; ++k) acc[k] = 0.f;
            bool entered = key[b] == key[b + 1];
            constexpr int U = 8;
            for (int i0 = b; i0 < e; i0 += U) {
                Pack<DT, VEC> v[U];
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (i0 + u < e) v[u].load_nt(dout + (int64_t)pos[i0 + u] * s.ld + c0);
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int i = i0 + u;
                    if (i >= e) break;
#pragma unroll
                    for (int k = 0; k < VEC; ++k) acc[k] += v[u].get(k);
                    const unsigned id = key[i + 1];
                    const bool leaves = id == key[i + 2];
                    if (leaves && i + 1 < e) continue;
                    if (entered || leaves) {
                        f |= entered ? (leaves ? 3 : 1) : 4;
                        float* q = part[entered ? 0 : 1] + j * width + col * VEC;
#pragma unroll
                        for (int k = 0; k < VEC; ++k) q[k] = acc[k];
                    } else if (id < (unsigned)s.V) {
                        float* q = dtable + (int64_t)id * s.E + c0;
                        float t[VEC];
                        if (s.accumulate) load_f32<VEC>(q, t);
#pragma unroll
                        for (int k = 0; k < VEC; ++k) t[k] = s.accumulate ? t[k] + s.scale * acc[k] : s.scale * acc[k];
                        store_f32<VEC>(q, t);
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
                    else put(dtable, s, key[k * s.L + 1], v0 * VEC + c, acc);
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
        if (c == 0 && v0 == 0) starts[blockIdx.x] = open ? (before ? 2 : 1) : 0;
    }
}

// One workgroup per chunk (and JOIN vectors of columns): where a run starts in this chunk and leaves it (starts 1), the sum of its
// parts up to the first chunk that it does not fill (starts 2: filled).  The parts go round the subgroups that a row of columns
// leaves room for, whose sums are added in order.  In f64: a part is a sum of at most CHUNK_MAX rows in f32, but the parts of one id
// are as many as the cells make (8388608 cells on one id, 516 columns: 8192 parts).
constexpr int JOIN = 256;      // 131072 cells, most on one id: 9.3 us, 8.8 with 1024 threads; 500009 cells: 6.5 and 9.6 (sums in f32)
template <int VEC>
__global__ __launch_bounds__(JOIN) void run_join_kernel(const uint2* __restrict__ pairs, float* __restrict__ dtable, SumShape s,
                                                       const float* __restrict__ slots, const int* __restrict__ starts) {
    __shared__ double sh[JOIN * VEC];
    __shared__ int first;
    const int64_t w = blockIdx.x, tail = min(s.n, (w + 1) * s.rows * s.L) - 1;
    int64_t last = w + 1;
    // three loads that do not wait for each other
    const int mine = starts[w];
    const unsigned key = pairs[tail].x;
    int next = last + threadIdx.x < s.chunks ? starts[last + threadIdx.x] : 0;
    if (mine != 1 || key >= (unsigned)s.V) return;
    for (;; last += JOIN) {      // a run that leaves a chunk ends in a later one, so there is a first that is not filled
        if (threadIdx.x == 0) first = JOIN;
        __syncthreads();
        const int64_t k = last + threadIdx.x;
        if (last > w + 1) next = k < s.chunks ? starts[k] : 0;
        if (next != 2) atomicMin(&first, (int)threadIdx.x);
        __syncthreads();
        const int f = first;
        __syncthreads();
        if (f < JOIN) { last += f; break; }
    }
    const int v0 = blockIdx.y * JOIN, nv = min(JOIN, s.E / VEC - v0), parts = JOIN / nv;
    const int col = threadIdx.x % nv, part = threadIdx.x / nv, c = (v0 + col) * VEC;
    double t[VEC] = {};
    if (part < parts) {
        if (part == 0) {
            float v[VEC];
            load_f32<VEC>(slots + (w * 2 + 1) * s.E + c, v);
#pragma unroll
            for (int e = 0; e < VEC; ++e) t[e] = v[e];
        }
#pragma unroll 8
        for (int64_t k = w + 1 + part; k <= last; k += parts) {
            float v[VEC];
            load_f32<VEC>(slots + k * 2 * s.E + c, v);
#pragma unroll
            for (int e = 0; e < VEC; ++e) t[e] += v[e];
        }
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) sh[threadIdx.x * VEC + e] = t[e];
    __syncthreads();
    if (part) return;
    for (int q = 1; q < parts; ++q)
#pragma unroll
        for (int e = 0; e < VEC; ++e) t[e] += sh[(q * nv + col) * VEC + e];
#pragma unroll
    for (int e = 0; e < VEC; ++e) put(dtable, s, key, c + e, (float)t[e]);
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
    // pairs of a workgroup: enough workgroups for the chip first (131072 x 128: 49 us with 256), then few parts to join
    // (500009 x 512: 318 us with 128, 254 with 256, 242 with 512, 239 with 1024, 268 with 2048)
    const int want = n <= 65536 ? 64 : (n <= 262144 ? 256 : 1024);
    p.L = (int)cdiv(want, p.rows);
    if (p.L < 4) p.L = 4;                                                // rows * L < max(want + rows, 4 * 256) <= CHUNK_MAX
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

// values of a vector, wherever the rows of cells begin (500009 x 512 bf16 in rows of 513: gradient 206 us, single elements 483; lookup
// 224, 283)
inline int row_vec(int dt, int E, const void* table) {
    if (E % 4 || !aligned16(table)) return 1;
    return dt != CUTIE_F32 && E % 8 == 0 ? 8 : 4;
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
    const Dense in_ids{ids, (uint64_t)n_cells * 4}, in_table{table, (uint64_t)V * E * 4}, count{oob_count, 4};
    const Rows rows_out{out, n_cells, (uint64_t)E * es, (uint64_t)ld_out * es};
    CUTIE_CHECK_ARG(!rows_meet(rows_out, in_ids) && !rows_meet(rows_out, in_table) && !rows_meet(rows_out, count) &&
                        !dense_meet(count, in_ids) && !dense_meet(count, in_table), "embed_scaled_fwd: an output overlaps another tensor of the call");
    const int vec = row_vec(out_dtype, E, table);
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
    const GradSpace w = n_cells ? grad_space(n_cells, V, E) : GradSpace{};
    if (n_cells && (!workspace || workspace_bytes < w.total || !aligned16(workspace))) {
        set_error("embed_grad_sorted: workspace %zu < %zu (or not 16-byte aligned)", workspace ? workspace_bytes : 0, w.total);
        return CUTIE_E_WORKSPACE;
    }
    const Dense in_ids{ids, (uint64_t)n_cells * 4}, space{workspace, w.total}, sums{dtable, (uint64_t)V * E * 4};
    const Rows rows_in{dout, n_cells, (uint64_t)E * es, (uint64_t)ld_dout * es};
    CUTIE_CHECK_ARG(!rows_meet(rows_in, sums) && !rows_meet(rows_in, space) && !dense_meet(in_ids, sums) && !dense_meet(in_ids, space) &&
                        !dense_meet(sums, space), "embed_grad_sorted: dtable or the workspace overlaps another tensor of the call");
    if (n_cells == 0 && accumulate) return CUTIE_OK;
    char* ws = (char*)workspace;
    const SortPlan sp = sort_plan(n_cells, V);
    uint2* sorted = nullptr;
    if (n_cells == 0) {
    } else if (sp.one) {
        sorted = (uint2*)(ws + w.a);
        const size_t lds = sp.passes > 1 ? (size_t)n_cells * sizeof(uint2) : 0;
        auto go = [&](auto kern) {
            hipLaunchKernelGGL(kern, dim3(1), dim3(1024), lds, stream, ids, (int)n_cells, V, sp.passes, sp.bits, sorted);
        };
        if (n_cells <= 4096) {
            CUTIE_ENSURE_LDS(sort_one_kernel<4>, 4096 * sizeof(uint2));
            go(sort_one_kernel<4>);
        } else {
            CUTIE_ENSURE_LDS(sort_one_kernel<8>, ONE * sizeof(uint2));
            go(sort_one_kernel<8>);
        }
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
            auto count = pass ? sort_count_kernel<false> : sort_count_kernel<true>;
            auto scatter = pass ? sort_scatter_kernel<false> : sort_scatter_kernel<true>;
            const bool scan = sp.tiles > SELF_TILES;
            hipLaunchKernelGGL(count, dim3((unsigned)sp.tiles), dim3(1024), 0, stream, ids, in, n_cells, V, shift, sp.bits, counts);
            if (scan)
                hipLaunchKernelGGL(sort_scan_kernel, dim3((unsigned)cdiv(bins, 16)), dim3(1024), 0, stream, counts, sp.tiles, sp.bits, totals);
            hipLaunchKernelGGL(scatter, dim3((unsigned)sp.tiles), dim3(1024), 0, stream, ids, in, n_cells, V, shift, sp.bits, counts,
                               scan ? totals : nullptr, out);
            CUTIE_CHECK_LAUNCH();
        }
        sorted = buf[(sp.passes - 1) & 1];
    }
    const SumPlan p = sum_plan(n_cells, E, row_vec(dout_dtype, E, dtable));
    SumShape s;
    s.n = n_cells; s.chunks = p.chunks; s.V = V; s.E = E; s.ld = ld_dout; s.rows = p.rows; s.L = p.L; s.scale = scale; s.accumulate = accumulate;
    float* slots = (float*)(ws + w.slots);
    int* starts = (int*)(ws + w.starts);
    const int64_t blocks = p.chunks + (accumulate ? 0 : cdiv(V, 256));
    CUTIE_DISPATCH_DTYPE(dout_dtype, DT, {
        typedef typename elem<DT>::type T;
        auto go = [&](auto kern) {
            hipLaunchKernelGGL(kern, dim3((unsigned)blocks, (unsigned)p.ncol), dim3(256), 0, stream, sorted, (const T*)dout, dtable, s, slots,
                               starts);
        };
        if constexpr (DT != CUTIE_F32) {
            if (p.vec == 8) go(run_sum_kernel<DT, 8>);
        }
        if (p.vec == 4) go(run_sum_kernel<DT, 4>);
        if (p.vec == 1) go(run_sum_kernel<DT, 1>);
    });
    CUTIE_CHECK_LAUNCH();
    if (n_cells == 0) return CUTIE_OK;
    const int jv = E % 4 == 0 ? 4 : 1;
    const dim3 jgrid((unsigned)p.chunks, (unsigned)cdiv(E / jv, JOIN));
    if (jv == 4) hipLaunchKernelGGL(run_join_kernel<4>, jgrid, dim3(JOIN), 0, stream, sorted, dtable, s, slots, starts);
    else hipLaunchKernelGGL(run_join_kernel<1>, jgrid, dim3(JOIN), 0, stream, sorted, dtable, s, slots, starts);
    CUTIE_CHECK_LAUNCH();
    return CUTIE_OK;
}
