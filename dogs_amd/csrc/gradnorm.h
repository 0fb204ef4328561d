// gradnorm.h -- the norm of a set of tensors and the scaling of them by the clipping coefficient (gradnorm.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace gs {

// tensors of one launch; their table travels in the kernel arguments (2.7 KB of the 4 KB), so no host memory has to
// outlive the call and a captured graph holds its own copy
constexpr int GN_MAX = 128;
// at most this many blocks (= double partials) over all launches of a call, and one more per tensor: each ends in a
// block of its own
constexpr uint32_t GN_MAX_BLOCKS = 4096;
constexpr uint32_t GN_MIN_CHUNK = 16384;  // bytes of a block

struct GradTable {
    void* p[GN_MAX];
    uint64_t n[GN_MAX];           // elements
    uint32_t start[GN_MAX + 1];   // first block of tensor k (of this launch)
    uint8_t dtype[GN_MAX];        // DG_F32 / DG_F16 / DG_BF16
    int count;
    uint32_t chunk;               // bytes of a block
};

// the chunk size for that
uint32_t gn_chunk(uint64_t total_bytes);
uint32_t gn_blocks(uint64_t n, int dtype, uint32_t chunk);
// partial[b] of every block: sum of squares (ord 2), sum of |x| (1) or max |x| (0: infinity); again: the tensors will be read
// once more
void launch_grad_partials(const GradTable& t, int ord, bool again, double* partial, hipStream_t s);
// *norm from the n partials, and *coef = min(1, max_norm / (norm + 1e-6)) (coef may be null)
void launch_grad_norm_final(const double* partial, uint32_t n, int ord, double max_norm, float* norm, double* coef,
                            hipStream_t s);
// every element times *coef, in place; nothing is touched when *coef == 1
void launch_grad_scale(const GradTable& t, const double* coef, hipStream_t s);

}  // namespace gs
