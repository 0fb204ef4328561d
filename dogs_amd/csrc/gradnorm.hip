// gradnorm.hip -- norm and clipping of a set of gradients (gradnorm.h).
//
//   n = sqrt(sum over tensors and elements of g^2)  (or the sum or the maximum of |g|),  g <- g min(1, max_norm / (n + 1e-6))
//
// The squares are summed in 64 bits: every finite fp32, fp16 or bf16 square is exact in range there (1e-90 .. 1e77), so
// no gradient is too large or too small for its norm, and the vector unit's 64-bit fma runs at the unpacked 32-bit
// rate -- at 8 TB/s a CU has 20 lane operations per fp32 element, and this uses two.  Blocks own fixed byte ranges and
// their partials meet in a fixed order: the same bits every time, no atomics.  HBM-bound: the norm reads each byte
// once, the scaling reads and writes it once more, and only when there is something to clip.
#include <hip/hip_runtime.h>

#include "dtypes.h"
#include "gradnorm.h"

namespace gs {

namespace {

constexpr int GN_THREADS = 256;

template <int ORD>
__device__ __forceinline__ void take(double& acc, float x) {
    if (ORD == 2) {
        const double d = (double)x;
        acc = fma(d, d, acc);
    } else if (ORD == 1) {
        acc += (double)fabsf(x);
    } else {  // the maximum; a NaN stays
        const double d = (double)fabsf(x);
        acc = (d > acc || d != d) ? d : acc;
    }
}
template <int ORD>
__device__ __forceinline__ double join(double a, double b) {
    if (ORD != 0) return a + b;
    return (b > a || b != b) ? b : a;
}

template <int ORD>
__device__ __forceinline__ double block_join(double v, double* s) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, nw = (int)(blockDim.x >> 6);
#pragma unroll
    for (int o = 32; o; o >>= 1) v = join<ORD>(v, __shfl_down(v, o));
    if (lane == 0) s[w] = v;
    __syncthreads();
    v = s[0];
    for (int k = 1; k < nw; k++) v = join<ORD>(v, s[k]);
    return v;
}

// the tensor of block b: the table's starts ascend (an empty tensor takes no block)
__device__ __forceinline__ int tensor_of(const GradTable& t, uint32_t b) {
    int lo = 0, hi = t.count;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (t.start[mid] <= b) lo = mid; else hi = mid;
    }
    return lo;
}

// AGAIN: the tensors are read once more after this (the scaling, the clipped update): they pass through the caches then,
// which keep up to 256 MB for it.  Otherwise the loads pass by them: 1e6 x 59 floats in 34 us (6.9 TB/s) instead of 40,
// while the update after it took 259 us instead of 244.  (Above 256 MB they evict each other: 403 MB of bf16 that were just
// written 96 us instead of 65; the rule goes by use alone.)
template <int ORD, bool AGAIN, typename T>
__device__ __forceinline__ double chunk_norm(const T* __restrict__ p, uint64_t n) {
    typedef typename Vec<T>::type V;
    constexpr int W = Vec<T>::W;
    double acc[2] = {0.0, 0.0};
    const uint64_t nv = n / W;
#pragma unroll 4
    for (uint64_t i = threadIdx.x; i < nv; i += GN_THREADS) {
        const V* q = reinterpret_cast<const V*>(p + i * W);
        const V x = AGAIN ? *q : __builtin_nontemporal_load(q);
#pragma unroll
        for (int j = 0; j < W; j++) take<ORD>(acc[j & 1], (float)x[j]);
    }
    for (uint64_t i = nv * W + threadIdx.x; i < n; i += GN_THREADS) take<ORD>(acc[0], (float)p[i]);
    return join<ORD>(acc[0], acc[1]);
}

template <int ORD, bool AGAIN>
__global__ void __launch_bounds__(GN_THREADS) k_grad_partials(GradTable t, double* __restrict__ partial) {
    __shared__ double s[GN_THREADS / 64];
    const uint32_t b = blockIdx.x;
    const int k = tensor_of(t, b);
    const uint64_t per = t.dtype[k] == 0 ? t.chunk / 4 : t.chunk / 2;
    const uint64_t e0 = (uint64_t)(b - t.start[k]) * per;
    const uint64_t n = t.n[k] - e0 < per ? t.n[k] - e0 : per;
    double v;
    if (t.dtype[k] == 0) v = chunk_norm<ORD, AGAIN>((const float*)t.p[k] + e0, n);
    else if (t.dtype[k] == 1) v = chunk_norm<ORD, AGAIN>((const _Float16*)t.p[k] + e0, n);
    else v = chunk_norm<ORD, AGAIN>((const __bf16*)t.p[k] + e0, n);
    v = block_join<ORD>(v, s);
    if (threadIdx.x == 0) partial[b] = v;
}

template <int ORD>
__global__ void __launch_bounds__(1024) k_grad_norm_final(const double* __restrict__ partial, uint32_t n, double max_norm,
                                                          float* __restrict__ norm_out, double* __restrict__ coef) {
    __shared__ double s[16];
    double v = 0.0;
    for (uint32_t i = threadIdx.x; i < n; i += 1024) v = join<ORD>(v, partial[i]);
    v = block_join<ORD>(v, s);
    if (threadIdx.x) return;
    const double norm = ORD == 2 ? sqrt(v) : v;
    *norm_out = (float)norm;
    if (coef) {
        const double c = max_norm / (norm + 1e-6);
        *coef = c >= 1.0 ? 1.0 : c;  // a NaN stays: every gradient becomes NaN
    }
}

template <typename T>
__device__ __forceinline__ void chunk_scale(T* __restrict__ p, uint64_t n, double c) {
    typedef typename Vec<T>::type V;
    constexpr int W = Vec<T>::W;
    const uint64_t nv = n / W;
#pragma unroll 4
    for (uint64_t i = threadIdx.x; i < nv; i += GN_THREADS) {
        V* q = reinterpret_cast<V*>(p + i * W);
        V x = __builtin_nontemporal_load(q);
#pragma unroll
        for (int j = 0; j < W; j++) x[j] = (T)(float)((float)x[j] * c);
        __builtin_nontemporal_store(x, q);
    }
    for (uint64_t i = nv * W + threadIdx.x; i < n; i += GN_THREADS) p[i] = (T)(float)((float)p[i] * c);
}

__global__ void __launch_bounds__(GN_THREADS) k_grad_scale(GradTable t, const double* __restrict__ coef) {
    const double c = *coef;
    if (c == 1.0) return;  // x * 1 is x
    // from the back: the end is what the norm left in the caches.  (The launches of more than GN_MAX tensors go front to
    // back: in reverse 300 tensors of 240 MB took 151 us with their norm instead of 150, of 600 MB 397 instead of 394.)
    const uint32_t b = gridDim.x - 1 - blockIdx.x;
    const int k = tensor_of(t, b);
    const uint64_t per = t.dtype[k] == 0 ? t.chunk / 4 : t.chunk / 2;
    const uint64_t e0 = (uint64_t)(b - t.start[k]) * per;
    const uint64_t n = t.n[k] - e0 < per ? t.n[k] - e0 : per;
    if (t.dtype[k] == 0) chunk_scale((float*)t.p[k] + e0, n, c);
    else if (t.dtype[k] == 1) chunk_scale((_Float16*)t.p[k] + e0, n, c);
    else chunk_scale((__bf16*)t.p[k] + e0, n, c);
}

}  // namespace

uint32_t gn_chunk(uint64_t total_bytes) {
    // a power of two, so that it divides by every element size and vector width; 2^31 bytes of a block at most
    // (2^43 bytes of gradients)
    uint64_t c = GN_MIN_CHUNK;
    while (c < (1ull << 31) && total_bytes / c >= GN_MAX_BLOCKS) c <<= 1;
    return (uint32_t)c;
}

uint32_t gn_blocks(uint64_t n, int dtype, uint32_t chunk) {
    const uint64_t per = chunk / elem_bytes(dtype);
    return (uint32_t)((n + per - 1) / per);
}

template <bool AGAIN>
static void grad_partials(const GradTable& t, int ord, double* partial, hipStream_t s) {
    const uint32_t b = t.start[t.count];
    if (!b) return;
    if (ord == 2) k_grad_partials<2, AGAIN><<<b, GN_THREADS, 0, s>>>(t, partial);
    else if (ord == 1) k_grad_partials<1, AGAIN><<<b, GN_THREADS, 0, s>>>(t, partial);
    else k_grad_partials<0, AGAIN><<<b, GN_THREADS, 0, s>>>(t, partial);
}

void launch_grad_partials(const GradTable& t, int ord, bool again, double* partial, hipStream_t s) {
    if (again) grad_partials<true>(t, ord, partial, s);
    else grad_partials<false>(t, ord, partial, s);
}

void launch_grad_norm_final(const double* partial, uint32_t n, int ord, double max_norm, float* norm, double* coef,
                            hipStream_t s) {
    if (ord == 2) k_grad_norm_final<2><<<1, 1024, 0, s>>>(partial, n, max_norm, norm, coef);
    else if (ord == 1) k_grad_norm_final<1><<<1, 1024, 0, s>>>(partial, n, max_norm, norm, coef);
    else k_grad_norm_final<0><<<1, 1024, 0, s>>>(partial, n, max_norm, norm, coef);
}

void launch_grad_scale(const GradTable& t, const double* coef, hipStream_t s) {
    const uint32_t b = t.start[t.count];
    if (b) k_grad_scale<<<b, GN_THREADS, 0, s>>>(t, coef);
}

}  // namespace gs
