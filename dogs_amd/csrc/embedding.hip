// embedding.hip -- embedding lookup and its gradient (embedding.h).
//
//   lookup    Y[i] = s E[t_i];  a token outside [0, V) gives a row of NaN
//   gradient  dE[v] = s sum_{i: t_i = v} G[i], in an order that the tokens set;  0 for the padding token and for v without one
#include <hip/hip_runtime.h>

#include "dtypes.h"
#include "embedding.h"
#include "sortscan.h"

namespace gs {

namespace {

constexpr int EB_THREADS = 256;
constexpr uint64_t PAST_BYTES = 32ull << 20;   // the L2 caches together
constexpr uint32_t EB_MAX_BLOCKS = 1u << 20;   // then they stride: a grid holds fewer than 2^32 threads

__device__ __forceinline__ int64_t token_at(const void* t, int wide, uint32_t i) {
    return wide ? ((const int64_t*)t)[i] : (int64_t)((const int32_t*)t)[i];
}

// A lane's 16 bytes of a row.  PAST: by the caches, where what is touched once is larger than they are -- 65536 x 2048 bf16
// in 131072 rows: the sums 139 us instead of 190, the lookup 72 instead of 84; smaller results stay in the caches for the
// kernel that reads them.
template <typename T, bool PAST> struct Cols {
    typedef typename Vec<T>::type V;
    static constexpr int W = Vec<T>::W;
    uint32_t c0;     // first column of this lane
    int nc;          // its columns: W, 0 past the row, or the whole row where that is shorter than W
    template <bool ONCE>
    __device__ __forceinline__ V load(const T* row) const {
        V x = {};
        const V* q = reinterpret_cast<const V*>(row + c0);
        if (nc == W) x = PAST && ONCE ? __builtin_nontemporal_load(q) : *q;
        else
            for (int j = 0; j < nc; j++) x[j] = row[j];
        return x;
    }
    __device__ __forceinline__ void store(T* row, V x) const {
        V* q = reinterpret_cast<V*>(row + c0);
        if (nc == W) {
            if (PAST) __builtin_nontemporal_store(x, q);
            else *q = x;
        } else
            for (int j = 0; j < nc; j++) row[j] = x[j];
    }
    __device__ __forceinline__ void store(T* row, const float (&acc)[W], float scale) const {
        V x;
#pragma unroll
        for (int j = 0; j < W; j++) x[j] = (T)(acc[j] * scale);
        store(row, x);
    }
};

// The last lane of a row whose width is no multiple of W takes the row's last W columns: some are the lane's before it too, and
// both compute and store the same bits.  (Its own few columns one by one: a row of 1023 fp16 took 2.7 times as long
// as one of 1024.)
template <typename T, bool PAST>
__device__ __forceinline__ Cols<T, PAST> cols_of(uint32_t slab, int lpr, uint32_t l, uint32_t D) {
    constexpr uint32_t W = Vec<T>::W;
    const uint64_t c0 = ((uint64_t)slab * lpr + l) * W;
    if (D < W) return {0u, c0 ? 0 : (int)D};
    if (c0 >= D) return {0u, 0};
    return {c0 + W <= D ? (uint32_t)c0 : D - W, (int)W};
}

// lpr lanes (a power of two, up to a wave) per row, 256 / lpr rows per block, LOOK slabs of a row in flight: one where there
// are few rows (a block per slab: 8 x 4096 bf16 2.7 us, with four 4.5), four for a large result (65536 x 2048 72 us, with
// one slab of a whole block's lanes 102)
template <typename T, int LOOK, bool PAST>
__global__ void __launch_bounds__(EB_THREADS) k_lookup(LookupArgs a, int lpr) {
    typedef typename Vec<T>::type V;
    constexpr int W = Vec<T>::W;
    const uint32_t l = threadIdx.x & (lpr - 1), per = EB_THREADS / lpr;
    Cols<T, PAST> c[LOOK];
#pragma unroll
    for (int u = 0; u < LOOK; u++) c[u] = cols_of<T, PAST>(blockIdx.y * LOOK + u, lpr, l, a.D);
    for (uint64_t row = (uint64_t)blockIdx.x * per + threadIdx.x / lpr; row < a.n; row += (uint64_t)gridDim.x * per) {
        const int64_t tok = token_at(a.tokens, a.wide, (uint32_t)row);
        const bool bad = tok < 0 || (uint64_t)tok >= a.V;
        T* out = (T*)a.out + row * a.D;
        const T* in = (const T*)a.table + (bad ? 0 : tok) * a.row_stride;
        if (a.col_stride != 1) {
            for (uint32_t k = blockIdx.y * lpr + l; k < a.D; k += gridDim.y * lpr)
                out[k] = (T)(bad ? __builtin_nanf("") : (float)in[(int64_t)k * a.col_stride] * a.scale);
            continue;
        }
        V x[LOOK];
#pragma unroll
        for (int u = 0; u < LOOK; u++) x[u] = bad ? V{} : c[u].template load<false>(in);
#pragma unroll
        for (int u = 0; u < LOOK; u++) {
#pragma unroll
            for (int j = 0; j < W; j++) x[u][j] = (T)(bad ? __builtin_nanf("") : (float)x[u][j] * a.scale);
            c[u].store(out, x[u]);
        }
    }
}

// the row that position i adds to, or V where it adds to none
__device__ __forceinline__ uint32_t key_at(const LookupGradArgs& a, uint32_t i) {
    const int64_t t = token_at(a.tokens, a.wide, i);
    return (t < 0 || t >= (int64_t)a.V || t == a.padding) ? a.V : (uint32_t)t;
}

// the lanes of the wave that hold the same `bits`-bit digit, among the active ones
__device__ __forceinline__ uint64_t peers(uint32_t d, bool act, int bits) {
    uint64_t m = __ballot(act);
    for (int b = 0; b < bits; b++) {
        const uint64_t s = __ballot((d >> b) & 1u);
        m &= ((d >> b) & 1u) ? s : ~s;
    }
    return m;
}
// what the wave's lanes stored to LDS is what they load from here on (no barrier: one wave's accesses complete in order)
__device__ __forceinline__ void wave_lds_fence() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}
__device__ __forceinline__ uint64_t lanes_below() { return (1ull << (threadIdx.x & 63)) - 1ull; }

// exclusive scan of one value per thread over the block; s_w holds a word per wave
template <int NW>
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t* s_w) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    uint32_t x = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t y = __shfl_up(x, o);
        if (lane >= o) x += y;
    }
    if (lane == 63) s_w[w] = x;
    __syncthreads();
    uint32_t off = 0;
#pragma unroll
    for (int k = 0; k < NW; k++) off += k < w ? s_w[k] : 0u;
    return off + x - v;
}

// ---- sums over a sorted list
//
// A block holds a sorted stretch of (key, position) pairs in LDS and a slab of lpr x 16 bytes of the columns.  Its groups of
// lpr lanes walk equal parts of the stretch, eight gradient rows in flight, and keep the running sum in registers;
// a row whose entries lie within one part is stored from there.  Sums of runs that cross parts meet in LDS, in order, and
// those that cross the block's ends go to the partials of the block: `head` for the run that began before it,
// `tail` for the one that begins in it and goes on.  So a token that makes up half the batch costs no more than others.
struct Pairs {       // a list in LDS as two arrays
    const uint32_t *k, *p;
    __device__ __forceinline__ uint32_t key(uint32_t j) const { return k[j]; }
    __device__ __forceinline__ uint32_t pos(uint32_t j) const { return p[j]; }
};
struct Packed {      // as key << 16 | position
    const uint32_t* e;
    __device__ __forceinline__ uint32_t key(uint32_t j) const { return e[j] >> 16; }
    __device__ __forceinline__ uint32_t pos(uint32_t j) const { return e[j] & 0xffffu; }
};
template <typename L> struct Stretch {
    L e;                     // ascending keys
    uint32_t n;
    bool open_front, open_back;   // the first / last run goes on outside
    uint32_t row0;           // key k is row row0 + k of the table
    float *head, *tail;      // the block's partials, D floats each (null: neither end is open)
};

constexpr int WALK = 8;   // rows in flight; four are as fast, twelve or sixteen take half as long again (registers)

// THREADS threads; s_part: LDS of THREADS * 2 * W floats
template <typename T, bool PAST, int THREADS, typename L>
__device__ __forceinline__ void sum_stretch(const LookupGradArgs& a, const Stretch<L>& s, const Cols<T, PAST>& c, int lpr,
                                            float* __restrict__ s_part) {
    typedef typename Vec<T>::type V;
    constexpr int W = Vec<T>::W;
    const uint32_t groups = THREADS / lpr, g = threadIdx.x / lpr, part = (s.n + groups - 1) / groups;
    const uint32_t lo = g * part < s.n ? g * part : s.n, hi = lo + part < s.n ? lo + part : s.n;
    const T* grad = (const T*)a.grad;
    T* table = (T*)a.dtable;
    float* mine = s_part + threadIdx.x * (2 * W);   // this lane's columns of the group's head, then of its tail
    if (lo < hi) {
        const bool front = lo ? s.e.key(lo - 1) == s.e.key(lo) : s.open_front;
        const bool back = hi < s.n ? s.e.key(hi) == s.e.key(hi - 1) : s.open_back;
        float acc[W] = {};
        uint32_t cur = s.e.key(lo);
        bool first = true;
        auto flush = [&](bool last) {
            if (first && front) {
#pragma unroll
                for (int j = 0; j < W; j++) mine[j] = acc[j];
            } else if (last && back) {
#pragma unroll
                for (int j = 0; j < W; j++) mine[W + j] = acc[j];
            } else {
                c.store(table + (uint64_t)(s.row0 + cur) * a.D, acc, a.scale);
            }
        };
        for (uint32_t j0 = lo; j0 < hi; j0 += WALK) {
            V x[WALK];
            uint32_t k[WALK];
#pragma unroll
            for (int u = 0; u < WALK; u++) {
                const uint32_t j = j0 + u < hi ? j0 + u : hi - 1;
                k[u] = s.e.key(j);
                x[u] = c.template load<true>(grad + (uint64_t)s.e.pos(j) * a.D);
            }
#pragma unroll
            for (int u = 0; u < WALK; u++) {
                if (j0 + u >= hi) break;
                if (k[u] != cur) {
                    flush(false);
                    first = false;
                    cur = k[u];
#pragma unroll
                    for (int j = 0; j < W; j++) acc[j] = 0.0f;
                }
#pragma unroll
                for (int j = 0; j < W; j++) acc[j] += (float)x[u][j];
            }
        }
        flush(true);
    }
    __syncthreads();
    if (lo >= hi) return;
    // the group whose tail begins a run joins it with the heads after it; group 0 also joins the run that was open in front
    const uint32_t lane_off = (threadIdx.x - g * lpr) * (2 * W);
    auto join = [&](float (&acc)[W], uint32_t k, uint32_t h) {   // heads of parts h, h + 1, ... while they hold key k
        for (; h < groups && h * part < s.n && s.e.key(h * part) == k; h++) {
            const float* o = s_part + (uint64_t)h * lpr * (2 * W) + lane_off;
#pragma unroll
            for (int j = 0; j < W; j++) acc[j] += o[j];
        }
    };
    auto put = [&](float* dst, const float (&acc)[W]) {
#pragma unroll
        for (int j = 0; j < W; j++)
            if (j < c.nc) dst[c.c0 + j] = acc[j];
    };
    if (g == 0 && s.open_front) {
        float acc[W];
#pragma unroll
        for (int j = 0; j < W; j++) acc[j] = mine[j];
        join(acc, s.e.key(0), 1);
        put(s.head, acc);
    }
    const uint32_t k = s.e.key(hi - 1);
    const bool begins = lo ? s.e.key(lo - 1) != k : !(s.open_front && s.e.key(0) == k);
    const bool goes_on = hi < s.n ? s.e.key(hi) == k : s.open_back;
    if (begins && goes_on) {
        float acc[W];
#pragma unroll
        for (int j = 0; j < W; j++) acc[j] = mine[W + j];
        join(acc, k, g + 1);
        if (s.open_back && s.e.key(s.n - 1) == k) put(s.tail, acc);
        else c.store(table + (uint64_t)(s.row0 + k) * a.D, acc, a.scale);
    }
}

// ---- few tokens: one launch
//
// A block owns `rows` (a power of two, up to 256) rows of the table and one slab of columns.  It looks through all tokens,
// each wave through a contiguous part of them, ranks those of its rows (stable counting sort by row, in LDS), and sums.
// The list is 64 IT NW entries long at most; LDS and the tokens that a lane looks at go with it (256 tokens of 64 fp32 take 6 us
// in the kernel for 1024, 9 in that for 4096).  1024 blocks are aimed at: twice as many cost up to a third (each looks through
// all tokens), half as many up to an eighth in small tables, and save 5 % in large ones.  Stored through the caches
// whatever the size: past them a table of 50021 x 1023 fp16 took 4 to 13 us more, one of 131072 x 2048 bf16 no less.
template <typename T, int NW, int IT>
__global__ void __launch_bounds__(NW * 64) k_grad_small(LookupGradArgs a, int lpr, uint32_t rows, int row_bits, uint32_t slabs) {
    __shared__ uint32_t s_list[NW * 64 * IT];
    __shared__ uint32_t s_hist[NW][256];
    __shared__ uint32_t s_w[NW];
    __shared__ float s_part[NW * 64 * 2 * Vec<T>::W];
    const int t = threadIdx.x, lane = t & 63, w = t >> 6;
    const uint32_t v0 = (uint32_t)(blockIdx.x / slabs) * rows, slab = blockIdx.x % slabs;
    const uint32_t nrows = a.V - v0 < rows ? a.V - v0 : rows;
    for (int i = t; i < NW * 256; i += NW * 64) (&s_hist[0][0])[i] = 0u;
    uint32_t code[IT];   // row << 16 | rank among this wave's tokens of the row
    const uint32_t base = (uint32_t)w * (64 * IT) + lane;
#pragma unroll
    for (int r = 0; r < IT; r++) {
        const uint32_t i = base + 64 * r;
        code[r] = i < a.n ? key_at(a, i) - v0 : ~0u;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < IT; r++) {
        const uint32_t lr = code[r];
        const bool act = lr < nrows;
        code[r] = ~0u;
        if (!__ballot(act)) continue;
        const uint64_t m = peers(lr, act, row_bits);
        const uint32_t before = (uint32_t)__popcll(m & lanes_below());
        if (act) {
            const uint32_t had = s_hist[w][lr];
            code[r] = lr << 16 | (had + before);
            if (!(m >> lane >> 1)) s_hist[w][lr] = had + before + 1;   // the last peer publishes the count
        }
        wave_lds_fence();
    }
    __syncthreads();
    uint32_t mine = 0;
    if (t < 256)
        for (int k = 0; k < NW; k++) mine += s_hist[k][t];
    uint32_t at = block_scan<NW>(mine, s_w);
    uint32_t total = 0;
    for (int k = 0; k < NW; k++) total += s_w[k];
    if (t < 256)
        for (int k = 0; k < NW; k++) {
            const uint32_t n = s_hist[k][t];
            s_hist[k][t] = at;
            at += n;
        }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < IT; r++) {
        if (code[r] == ~0u) continue;
        const uint32_t lr = code[r] >> 16, o = s_hist[w][lr] + (code[r] & 0xffffu);
        s_list[o] = lr << 16 | (base + 64 * r);
    }
    __syncthreads();
    const Cols<T, false> c = cols_of<T, false>(slab, lpr, t & (lpr - 1), a.D);
    // rows without a token: the first wave's start of a row is the row's, and where row r + 1 begins row r ends
    for (uint32_t r = t / lpr; r < nrows; r += NW * 64 / lpr) {
        const uint32_t end = r + 1 < 256 ? s_hist[0][r + 1] : total;
        if (s_hist[0][r] == end) c.store((T*)a.dtable + (uint64_t)(v0 + r) * a.D, typename Vec<T>::type{});
    }
    const Stretch<Packed> s = {{s_list}, total, false, false, v0, nullptr, nullptr};
    sum_stretch<T, false, NW * 64>(a, s, c, lpr, s_part);
}

// ---- many tokens: sort them, sum stretches of the sorted list, join what crosses stretches

// Stable radix sort of (key, position), digits of `bits` bits, 1024 pairs per block: the launches are latency, so
// the digits are as wide as two passes need (up to 11 bits) and a pass is spread over more blocks than a sort of
// millions would take: 65536 tokens of 131072 rows 27 us, 262144 of them 36, where the 8-bit sort of the binning
// (sortscan.hip, which longer lists take) needs 82 and 86.
constexpr int TS_THREADS = 256, TS_IT = 4, TS_TILE = TS_THREADS * TS_IT, TS_MAX_BITS = 11;
constexpr uint32_t TS_MAX_N = 1u << 18;   // 256 tiles: the scan of a digit's counts over tiles is one block wide

__device__ __forceinline__ uint32_t sort_key(const LookupGradArgs& a, const uint32_t* keys, uint32_t i) {
    return keys ? keys[i] : key_at(a, i);
}

__global__ void __launch_bounds__(TS_THREADS) k_sort_count(LookupGradArgs a, const uint32_t* __restrict__ keys, int shift,
                                                           int bits, uint32_t* __restrict__ counts) {
    __shared__ uint32_t hist[1 << TS_MAX_BITS];
    const uint32_t bins = 1u << bits, base = blockIdx.x * TS_TILE + threadIdx.x;
    uint32_t k[TS_IT];
#pragma unroll
    for (int r = 0; r < TS_IT; r++) {
        const uint32_t i = base + r * TS_THREADS;
        k[r] = i < a.n ? sort_key(a, keys, i) : 0u;
    }
    for (uint32_t d = threadIdx.x; d < bins; d += TS_THREADS) hist[d] = 0u;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < TS_IT; r++)
        if (base + r * TS_THREADS < a.n) atomicAdd(&hist[(k[r] >> shift) & (bins - 1)], 1u);
    __syncthreads();
    for (uint32_t d = threadIdx.x; d < bins; d += TS_THREADS) counts[(uint64_t)d * gridDim.x + blockIdx.x] = hist[d];
}

// block d: the exclusive scan of digit d's counts over the tiles, and its total
__global__ void __launch_bounds__(TS_THREADS) k_sort_scan(uint32_t* __restrict__ counts, uint32_t tiles,
                                                          uint32_t* __restrict__ totals) {
    __shared__ uint32_t s_w[TS_THREADS / 64];
    uint32_t* c = counts + (uint64_t)blockIdx.x * tiles;
    const uint32_t v = threadIdx.x < tiles ? c[threadIdx.x] : 0u;
    const uint32_t x = block_scan<TS_THREADS / 64>(v, s_w);
    if (threadIdx.x < tiles) c[threadIdx.x] = x;
    if (threadIdx.x == TS_THREADS - 1) totals[blockIdx.x] = x + v;
}

__global__ void __launch_bounds__(TS_THREADS) k_sort_scatter(LookupGradArgs a, const uint32_t* __restrict__ keys,
                                                             const uint32_t* __restrict__ pos, int shift, int bits,
                                                             const uint32_t* __restrict__ counts,
                                                             const uint32_t* __restrict__ totals,
                                                             uint32_t* __restrict__ keys_out, uint32_t* __restrict__ pos_out) {
    constexpr int NW = TS_THREADS / 64, PER = (1 << TS_MAX_BITS) / TS_THREADS;
    __shared__ uint32_t hist[NW][1 << TS_MAX_BITS];
    __shared__ uint32_t s_w[NW];
    const int t = threadIdx.x, lane = t & 63, w = t >> 6;
    const uint32_t bins = 1u << bits, base = blockIdx.x * TS_TILE + w * (64 * TS_IT) + lane;
    uint32_t k[TS_IT], p[TS_IT], rank[TS_IT];
#pragma unroll
    for (int r = 0; r < TS_IT; r++) {
        const uint32_t i = base + 64 * r;
        k[r] = i < a.n ? sort_key(a, keys, i) : 0u;
        p[r] = i < a.n && pos ? pos[i] : i;
    }
    // bins of a thread are neighbours, so one scan over the threads orders the digits
    const uint32_t per = bins > TS_THREADS ? bins / TS_THREADS : 1u;
    uint32_t tot[PER], before[PER], sum = 0;
#pragma unroll
    for (int j = 0; j < PER; j++) {
        const uint32_t d = t * per + j;
        const bool in = (uint32_t)j < per && d < bins;
        tot[j] = in ? totals[d] : 0u;
        before[j] = in ? counts[(uint64_t)d * gridDim.x + blockIdx.x] : 0u;
        sum += tot[j];
    }
    for (uint32_t d = t; d < bins; d += TS_THREADS)
#pragma unroll
        for (int q = 0; q < NW; q++) hist[q][d] = 0u;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < TS_IT; r++) {
        const bool act = base + 64 * r < a.n;
        const uint32_t d = (k[r] >> shift) & (bins - 1);
        const uint64_t m = peers(d, act, bits);
        const uint32_t lower = (uint32_t)__popcll(m & lanes_below());
        if (act) {
            const uint32_t had = hist[w][d];
            rank[r] = had + lower;
            if (!(m >> lane >> 1)) hist[w][d] = had + lower + 1;
        }
        wave_lds_fence();
    }
    uint32_t start = block_scan<NW>(sum, s_w);   // its barrier is also the one after the ranking
#pragma unroll
    for (int j = 0; j < PER; j++) {
        const uint32_t d = t * per + j;
        if ((uint32_t)j >= per || d >= bins) continue;
        uint32_t at = start + before[j];
        start += tot[j];
#pragma unroll
        for (int q = 0; q < NW; q++) {
            const uint32_t n = hist[q][d];
            hist[q][d] = at;
            at += n;
        }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < TS_IT; r++) {
        if (base + 64 * r >= a.n) continue;
        const uint32_t o = hist[w][(k[r] >> shift) & (bins - 1)] + rank[r];
        keys_out[o] = k[r];
        pos_out[o] = p[r];
    }
}

__global__ void __launch_bounds__(EB_THREADS) k_keys(LookupGradArgs a, uint32_t* __restrict__ keys) {
    const uint32_t i = blockIdx.x * EB_THREADS + threadIdx.x;
    if (i < a.n) keys[i] = key_at(a, i);
}

__device__ __forceinline__ uint32_t lower_bound(const uint32_t* __restrict__ keys, uint32_t n, uint32_t v) {
    uint32_t lo = 0, hi = n;
    while (lo < hi) {
        const uint32_t mid = lo + ((hi - lo) >> 1);
        if (keys[mid] < v) lo = mid + 1; else hi = mid;
    }
    return lo;
}

struct SumPlan {
    const uint32_t *keys, *pos;
    float* partial;          // [stretches][2][D]: head, tail
    uint32_t stretches, entries;   // entries of a stretch
    uint32_t slabs;
    uint32_t zero_rows;      // rows of a block that clears rows without a token
    int lpr;
};
constexpr uint32_t MAX_ENTRIES = 2048;

// blocks [0, stretches * slabs): the sums; the rest: zeros in the rows that no token names
template <typename T, bool PAST>
__global__ void __launch_bounds__(EB_THREADS) k_grad_sums(LookupGradArgs a, SumPlan p) {
    __shared__ uint32_t s_key[MAX_ENTRIES], s_pos[MAX_ENTRIES];
    __shared__ float s_part[EB_THREADS * 2 * Vec<T>::W];
    const uint32_t l = threadIdx.x & (p.lpr - 1);
    const uint64_t sums = (uint64_t)p.stretches * p.slabs;
    if (blockIdx.x < sums) {
        const uint32_t c = blockIdx.x / p.slabs, slab = blockIdx.x % p.slabs;
        const uint32_t e0 = c * p.entries, e1 = e0 + p.entries < a.n ? e0 + p.entries : a.n;
        for (uint32_t j = threadIdx.x; j < e1 - e0; j += EB_THREADS) {
            s_key[j] = p.keys[e0 + j];
            s_pos[j] = p.pos[e0 + j];
        }
        const uint32_t before = e0 ? p.keys[e0 - 1] : a.V, after = e1 < a.n ? p.keys[e1] : a.V;
        __syncthreads();
        uint32_t n = e1 - e0;
        if (s_key[n - 1] == a.V) n = lower_bound(s_key, n, a.V);   // entries that add to no row are last
        if (!n) return;
        float* part = p.partial + (uint64_t)c * 2 * a.D;
        const Stretch<Pairs> s = {{s_key, s_pos}, n, before == s_key[0], n == e1 - e0 && after == s_key[n - 1], 0, part, part + a.D};
        sum_stretch<T, PAST, EB_THREADS>(a, s, cols_of<T, PAST>(slab, p.lpr, l, a.D), p.lpr, s_part);
        return;
    }
    const uint64_t v0 = (blockIdx.x - sums) * p.zero_rows;
    for (uint32_t r = threadIdx.x; r < p.zero_rows; r += EB_THREADS) {
        const uint64_t v = v0 + r;
        uint32_t empty = 0;
        if (v < a.V) {
            const uint32_t at = lower_bound(p.keys, a.n, (uint32_t)v);
            empty = at == a.n || p.keys[at] != (uint32_t)v;
        }
        s_key[r] = empty;
    }
    __syncthreads();
    const uint32_t groups = EB_THREADS / p.lpr;
    for (uint32_t r = threadIdx.x / p.lpr; r < p.zero_rows; r += groups)
        if (s_key[r])
            for (uint32_t slab = 0; slab < p.slabs; slab++)
                cols_of<T, PAST>(slab, p.lpr, l, a.D).store((T*)a.dtable + (v0 + r) * a.D, typename Vec<T>::type{});
}

// The runs that cross stretches: the block of the stretch where one begins adds the tail there and the heads after it, a
// quarter of them per wave, in order.
template <typename T>
__global__ void __launch_bounds__(EB_THREADS) k_grad_join(LookupGradArgs a, SumPlan p) {
    __shared__ float4 s[EB_THREADS];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const uint32_t c = blockIdx.x, e0 = c * p.entries, e1 = e0 + p.entries;   // never the last stretch: e1 < n
    const uint32_t k = p.keys[e1 - 1];
    if (k == a.V || p.keys[e1] != k || (e0 && p.keys[e0 - 1] == k)) return;
    uint32_t heads = 0;   // stretches after c that begin with k
    for (bool more = true; more;) {
        const uint64_t h = (uint64_t)c + 1 + heads + lane;
        const uint64_t same = __ballot(h < p.stretches && p.keys[(uint32_t)(h * p.entries)] == k);
        more = same == ~0ull;
        heads += more ? 64u : (uint32_t)__builtin_ctzll(~same);
    }
    const uint32_t per = (heads + 3) / 4, lo = w * per < heads ? w * per : heads, hi = lo + per < heads ? lo + per : heads;
    const uint64_t c0 = (uint64_t)blockIdx.y * 256 + 4 * lane;
    float acc[4] = {};
    const float* base = p.partial + (uint64_t)c * 2 * a.D;
    typedef float F4 __attribute__((ext_vector_type(4), aligned(4)));
    const int nc = c0 + 4 <= a.D ? 4 : c0 < a.D ? (int)(a.D - c0) : 0;
    auto add = [&](const float* row) {
        if (nc == 4) {
            const F4 x = *reinterpret_cast<const F4*>(row + c0);
#pragma unroll
            for (int j = 0; j < 4; j++) acc[j] += x[j];
        } else {
            for (int j = 0; j < nc; j++) acc[j] += row[c0 + j];
        }
    };
    if (w == 0) add(base + a.D);
#pragma unroll 8
    for (uint32_t h = lo; h < hi; h++) add(base + (uint64_t)(h + 1) * 2 * a.D);
    s[threadIdx.x] = make_float4(acc[0], acc[1], acc[2], acc[3]);
    __syncthreads();
    if (w) return;
#pragma unroll
    for (int q = 1; q < 4; q++) {
        const float4 x = s[q * 64 + lane];
        acc[0] += x.x; acc[1] += x.y; acc[2] += x.z; acc[3] += x.w;
    }
    T* out = (T*)a.dtable + (uint64_t)k * a.D + c0;
    for (int j = 0; j < nc; j++) out[j] = (T)(acc[j] * a.scale);
}

inline size_t pad(size_t x) { return (x + 255) & ~(size_t)255; }

int key_bits(uint32_t V) {
    int b = 1;
    while (b < 32 && (V >> b)) b++;
    return b;
}

}  // namespace

namespace {

// lanes of a row's slab: as many 16-byte pieces as the row has, up to a wave
int lanes_per_row(uint32_t D, int dtype) {
    const uint32_t W = 16 / elem_bytes(dtype), pieces = (D + W - 1) / W;
    int lpr = 1;
    while (lpr < 64 && (uint32_t)lpr < pieces) lpr <<= 1;
    return lpr;
}
uint32_t slabs_of(uint32_t D, int dtype, int lpr) {
    const uint32_t per = lpr * (16 / elem_bytes(dtype));
    return (D + per - 1) / per;
}

// As many tokens as the one-launch kernel holds.  At 8000 tokens it and the sort with what follows take about as long (64 fp32
// over 2000 rows 17 us; 1023 fp16 over 50021 rows 48 us and 50), but it is one launch, not eight; a block of 16 waves
// for 16384 tokens fills a CU alone and was slower (62 us at 8191).
constexpr uint32_t SMALL_N = 8192;

// The one-launch kernel's blocks: `rows` rows of the table (a power of two, 2^bits) and a slab of half a wave's 16-byte pieces each.
// (A whole wave's: as fast where the tokens are spread, but one token that is 40 % of 8192 takes 111 us instead of 77 in
// 50000 rows of 1024 bf16; a quarter's: 55 instead of 41 where they are spread.)
struct SmallPlan {
    int lpr, bits;
    uint32_t rows, slabs, threads;
    uint64_t blocks;
};
SmallPlan small_plan(const LookupGradArgs& a, int dtype) {
    SmallPlan p = {};
    p.lpr = lanes_per_row(a.D, dtype);
    if (p.lpr > 32) p.lpr = 32;
    p.slabs = slabs_of(a.D, dtype, p.lpr);
    p.rows = 1;
    while (p.rows < 256 && (uint64_t)((a.V + p.rows - 1) / p.rows) * p.slabs > 1024) { p.rows <<= 1; p.bits++; }
    p.blocks = ((uint64_t)a.V + p.rows - 1) / p.rows * p.slabs;
    p.threads = a.n <= 4096 ? 256u : 512u;
    return p;
}

// ... unless its few blocks would each add up a long list (a table of few rows, where a group of lanes has over 160 tokens to
// walk: 8000 tokens of 1024 bf16 in 2 rows take 100 us in one launch, 24 sorted), or its many blocks would each look through
// many tokens (8192 of 2048 bf16 in 131072 rows: 160 us, sorted 131; up to 1024 tokens a lane looks through four at most).
bool one_launch(const LookupGradArgs& a, int dtype) {
    if (a.n > SMALL_N) return false;
    const SmallPlan p = small_plan(a, dtype);
    return a.n <= 160ull * a.V * (p.threads / p.lpr) && (a.n <= 1024 || a.n * p.blocks <= (1ull << 24));
}

SumPlan plan_of(const LookupGradArgs& a, int dtype) {
    SumPlan p = {};
    p.lpr = lanes_per_row(a.D, dtype);
    p.slabs = slabs_of(a.D, dtype, p.lpr);
    const uint32_t groups = EB_THREADS / p.lpr;
    p.entries = 32 * groups < MAX_ENTRIES ? 32 * groups : MAX_ENTRIES;
    p.stretches = (a.n + p.entries - 1) / p.entries;
    const uint64_t row = (uint64_t)a.D * elem_bytes(dtype);
    p.zero_rows = row >= 32768 ? 1u : (uint32_t)(32768 / row < 256 ? 32768 / row : 256);
    return p;
}

// [keys, pos] twice, the sort's counts, the partials
struct GradScratch {
    size_t pair, counts, partial, bytes;
};
GradScratch scratch_of(const LookupGradArgs& a, const SumPlan& p) {
    GradScratch s;
    s.pair = pad(4 * (size_t)a.n);
    s.counts = 4 * s.pair;
    const size_t tiles = ((size_t)a.n + TS_TILE - 1) / TS_TILE;
    const size_t counts = a.n <= TS_MAX_N ? 4 * ((size_t)1 << TS_MAX_BITS) * (tiles + 1) : radix_sort_temp_bytes(a.n);
    s.partial = s.counts + pad(counts);
    s.bytes = s.partial + (size_t)p.stretches * 2 * a.D * 4;
    return s;
}

template <typename T>
void grad_small(const LookupGradArgs& a, int dtype, hipStream_t s) {
    const SmallPlan p = small_plan(a, dtype);
    if (a.n <= 1024) k_grad_small<T, 4, 4><<<(uint32_t)p.blocks, 256, 0, s>>>(a, p.lpr, p.rows, p.bits, p.slabs);
    else if (a.n <= 4096) k_grad_small<T, 4, 16><<<(uint32_t)p.blocks, 256, 0, s>>>(a, p.lpr, p.rows, p.bits, p.slabs);
    else k_grad_small<T, 8, 16><<<(uint32_t)p.blocks, 512, 0, s>>>(a, p.lpr, p.rows, p.bits, p.slabs);
}

bool past_caches(const LookupGradArgs& a, int dtype) {
    return ((uint64_t)a.n + a.V) * a.D * elem_bytes(dtype) >= 2 * PAST_BYTES;
}

template <typename T, bool PAST>
void grad_sums(const LookupGradArgs& a, const SumPlan& p, hipStream_t s) {
    const uint64_t blocks = (uint64_t)p.stretches * p.slabs + ((uint64_t)a.V + p.zero_rows - 1) / p.zero_rows;
    k_grad_sums<T, PAST><<<(uint32_t)blocks, EB_THREADS, 0, s>>>(a, p);
    if (p.stretches > 1) k_grad_join<T><<<dim3(p.stretches - 1, (a.D + 255) / 256), EB_THREADS, 0, s>>>(a, p);
}

}  // namespace

void launch_embedding_lookup(const LookupArgs& a, int dtype, hipStream_t s) {
    const int lpr = lanes_per_row(a.D, dtype);
    const uint32_t rows = EB_THREADS / lpr, slabs = slabs_of(a.D, dtype, lpr);
    const bool large = (uint64_t)a.n * a.D * elem_bytes(dtype) >= PAST_BYTES;
    const uint64_t blocks = ((uint64_t)a.n + rows - 1) / rows;
    const dim3 grid((uint32_t)(blocks < EB_MAX_BLOCKS ? blocks : EB_MAX_BLOCKS), large ? (slabs + 3) / 4 : slabs);
    auto go = [&](auto t) {
        typedef decltype(t) T;
        if (large) k_lookup<T, 4, true><<<grid, EB_THREADS, 0, s>>>(a, lpr);
        else k_lookup<T, 1, false><<<grid, EB_THREADS, 0, s>>>(a, lpr);
    };
    if (dtype == 0) go(float());
    else if (dtype == 1) go(_Float16());
    else go(__bf16());
}

size_t embedding_grad_scratch_bytes(uint32_t V, uint32_t D, uint32_t n, int dtype) {
    LookupGradArgs a = {};
    a.V = V; a.D = D; a.n = n;
    return one_launch(a, dtype) ? 0 : scratch_of(a, plan_of(a, dtype)).bytes;
}

void launch_embedding_grad(const LookupGradArgs& a, int dtype, void* scratch, hipStream_t s) {
    if (one_launch(a, dtype)) {
        if (dtype == 0) grad_small<float>(a, dtype, s);
        else if (dtype == 1) grad_small<_Float16>(a, dtype, s);
        else grad_small<__bf16>(a, dtype, s);
        return;
    }
    SumPlan p = plan_of(a, dtype);
    const GradScratch o = scratch_of(a, p);
    char* b = (char*)scratch;
    uint32_t *k[2], *v[2];
    for (int q = 0; q < 2; q++) {
        k[q] = (uint32_t*)(b + 2 * q * o.pair);
        v[q] = (uint32_t*)(b + (2 * q + 1) * o.pair);
    }
    int in = 0;
    const int bits = key_bits(a.V);
    if (a.n <= TS_MAX_N) {
        const uint32_t tiles = (a.n + TS_TILE - 1) / TS_TILE;
        uint32_t *counts = (uint32_t*)(b + o.counts), *totals = counts + ((size_t)tiles << TS_MAX_BITS);
        const int passes = (bits + TS_MAX_BITS - 1) / TS_MAX_BITS, digit = (bits + passes - 1) / passes;
        for (int q = 0; q < passes; q++, in ^= 1) {
            const uint32_t *ki = q ? k[in] : nullptr, *vi = q ? v[in] : nullptr;
            k_sort_count<<<tiles, TS_THREADS, 0, s>>>(a, ki, q * digit, digit, counts);
            k_sort_scan<<<1u << digit, TS_THREADS, 0, s>>>(counts, tiles, totals);
            k_sort_scatter<<<tiles, TS_THREADS, 0, s>>>(a, ki, vi, q * digit, digit, counts, totals, k[in ^ 1], v[in ^ 1]);
        }
    } else {
        k_keys<<<(uint32_t)(((uint64_t)a.n + EB_THREADS - 1) / EB_THREADS), EB_THREADS, 0, s>>>(a, k[0]);
        in = radix_sort_pairs(k[0], v[0], k[1], v[1], nullptr, a.n, 0, bits, b + o.counts, s);
    }
    p.keys = k[in];
    p.pos = v[in];
    p.partial = (float*)(b + o.partial);
    auto go = [&](auto t) {
        if (past_caches(a, dtype)) grad_sums<decltype(t), true>(a, p, s);
        else grad_sums<decltype(t), false>(a, p, s);
    };
    if (dtype == 0) go(float());
    else if (dtype == 1) go(_Float16());
    else go(__bf16());
}

}  // namespace gs
