// embedding.hip -- embedding lookup and its gradient (embedding.h).
//
//   lookup    Y[i] = s E[t_i];  a token outside [0, V) gives a row of NaN
//   gradient  dE[v] = s sum_{i: t_i = v} G[i], summed in the order of i;  0 for the padding token and for v without one
#include <hip/hip_runtime.h>

#include "dtypes.h"
#include "embedding.h"
#include "sortscan.h"

namespace gs {

namespace {

constexpr int EB_THREADS = 256;
constexpr uint32_t EB_MAX_BLOCKS = 1u << 20;   // then they stride: a grid holds fewer than 2^32 threads

__device__ __forceinline__ int64_t token_at(const void* t, int wide, uint32_t i) {
    return wide ? ((const int64_t*)t)[i] : (int64_t)((const int32_t*)t)[i];
}

// LPR lanes (a power of two) per row, 256 / LPR rows per block; each lane moves 16 bytes at a time
template <typename T>
__global__ void __launch_bounds__(EB_THREADS) k_lookup(LookupArgs a, int lpr) {
    typedef typename Vec<T>::type V;
    constexpr int W = Vec<T>::W;
    const uint32_t l = threadIdx.x & (lpr - 1), per = EB_THREADS / lpr;
    for (uint64_t row = (uint64_t)blockIdx.x * per + threadIdx.x / lpr; row < a.n; row += (uint64_t)gridDim.x * per) {
        const int64_t tok = token_at(a.tokens, a.wide, (uint32_t)row);
        T* out = (T*)a.out + row * a.D;
        if (tok < 0 || (uint64_t)tok >= a.V) {
            for (uint32_t c = l; c < a.D; c += lpr) out[c] = (T)__builtin_nanf("");
            continue;
        }
        const T* in = (const T*)a.table + tok * a.row_stride;
        if (a.col_stride != 1) {
            for (uint32_t c = l; c < a.D; c += lpr) out[c] = (T)((float)in[c * a.col_stride] * a.scale);
            continue;
        }
        const uint32_t nv = a.D / W;
        for (uint32_t c = l; c < nv; c += lpr) {
            V x = *reinterpret_cast<const V*>(in + (uint64_t)c * W);
#pragma unroll
            for (int j = 0; j < W; j++) x[j] = (T)((float)x[j] * a.scale);
            *reinterpret_cast<V*>(out + (uint64_t)c * W) = x;
        }
        for (uint32_t c = nv * W + l; c < a.D; c += lpr) out[c] = (T)((float)in[c] * a.scale);
    }
}

// the sort key of position i: its token, or V where it adds to no row
__global__ void __launch_bounds__(EB_THREADS) k_keys(LookupGradArgs a, uint32_t* __restrict__ keys) {
    const uint32_t i = blockIdx.x * EB_THREADS + threadIdx.x;
    if (i >= a.n) return;
    const int64_t t = token_at(a.tokens, a.wide, i);
    keys[i] = (t < 0 || t >= (int64_t)a.V || t == a.padding) ? a.V : (uint32_t)t;
}

__device__ __forceinline__ uint32_t lower_bound(const uint32_t* __restrict__ keys, uint32_t n, uint32_t v) {
    uint32_t lo = 0, hi = n;
    while (lo < hi) {
        const uint32_t mid = lo + ((hi - lo) >> 1);
        if (keys[mid] < v) lo = mid + 1; else hi = mid;
    }
    return lo;
}

// a block per table row: the sum of its token's gradient rows, in their order
template <typename T>
__global__ void __launch_bounds__(EB_THREADS) k_rows(LookupGradArgs a, const uint32_t* __restrict__ keys,
                                                     const uint32_t* __restrict__ pos) {
    __shared__ uint32_t range[2];
    for (uint64_t v = blockIdx.x; v < a.V; v += gridDim.x) {
        __syncthreads();
        if (threadIdx.x < 2) range[threadIdx.x] = lower_bound(keys, a.n, (uint32_t)v + threadIdx.x);
        __syncthreads();
        const uint32_t lo = range[0], hi = range[1];
        T* out = (T*)a.dtable + v * a.D;
        for (uint32_t c = threadIdx.x; c < a.D; c += EB_THREADS) {
            float acc = 0.0f;
            for (uint32_t j = lo; j < hi; j++) acc += (float)((const T*)a.grad)[(uint64_t)pos[j] * a.D + c];
            out[c] = (T)(acc * a.scale);
        }
    }
}

inline size_t pad(size_t x) { return (x + 255) & ~(size_t)255; }

int key_bits(uint32_t V) {
    int b = 1;
    while (b < 32 && (V >> b)) b++;
    return b;
}

}  // namespace

void launch_embedding_lookup(const LookupArgs& a, int dtype, hipStream_t s) {
    const uint32_t W = 16 / elem_bytes(dtype), chunks = (a.D + W - 1) / W;
    int lpr = 1;
    while (lpr < EB_THREADS && (uint32_t)lpr < chunks) lpr <<= 1;
    const uint32_t rows = EB_THREADS / lpr;
    uint32_t blocks = (uint32_t)(((uint64_t)a.n + rows - 1) / rows);
    if (blocks > EB_MAX_BLOCKS) blocks = EB_MAX_BLOCKS;
    if (dtype == 0) k_lookup<float><<<blocks, EB_THREADS, 0, s>>>(a, lpr);
    else if (dtype == 1) k_lookup<_Float16><<<blocks, EB_THREADS, 0, s>>>(a, lpr);
    else k_lookup<__bf16><<<blocks, EB_THREADS, 0, s>>>(a, lpr);
}

size_t embedding_grad_scratch_bytes(uint32_t V, uint32_t D, uint32_t n, int dtype) {
    (void)V; (void)D; (void)dtype;
    return n ? 4 * pad(4 * (size_t)n) + pad(radix_sort_temp_bytes(n)) : 256;
}

void launch_embedding_grad(const LookupGradArgs& a, int dtype, void* scratch, hipStream_t s) {
    char* b = (char*)scratch;
    const size_t step = pad(4 * (size_t)a.n);
    uint32_t *k0 = (uint32_t*)b, *v0 = (uint32_t*)(b + step), *k1 = (uint32_t*)(b + 2 * step), *v1 = (uint32_t*)(b + 3 * step);
    int which = 0;
    if (a.n) {
        k_keys<<<(uint32_t)(((uint64_t)a.n + EB_THREADS - 1) / EB_THREADS), EB_THREADS, 0, s>>>(a, k0);
        which = radix_sort_pairs(k0, v0, k1, v1, nullptr, a.n, 0, key_bits(a.V), b + 4 * step, s);
    }
    const uint32_t *keys = which ? k1 : k0, *pos = which ? v1 : v0;
    const uint32_t blocks = a.V < EB_MAX_BLOCKS ? a.V : EB_MAX_BLOCKS;
    if (dtype == 0) k_rows<float><<<blocks, EB_THREADS, 0, s>>>(a, keys, pos);
    else if (dtype == 1) k_rows<_Float16><<<blocks, EB_THREADS, 0, s>>>(a, keys, pos);
    else k_rows<__bf16><<<blocks, EB_THREADS, 0, s>>>(a, keys, pos);
}

}  // namespace gs
