// embedding.h -- lookup of table rows by token, and the table's gradient by sorted tokens (embedding.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace gs {

struct LookupArgs {
    const void* table;
    int64_t row_stride, col_stride;  // elements
    const void* tokens;
    int wide;                        // tokens are 64-bit
    uint32_t n, D;
    uint64_t V;
    float scale;
    void* out;                       // [n][D]
};
void launch_embedding_lookup(const LookupArgs& a, int dtype, hipStream_t s);

struct LookupGradArgs {
    const void* grad;                // [n][D]
    const void* tokens;
    int wide;
    uint32_t n, D, V;
    float scale;
    int64_t padding;                 // -1: none
    void* dtable;                    // [V][D]
};
size_t embedding_grad_scratch_bytes(uint32_t V, uint32_t D, uint32_t n, int dtype);
void launch_embedding_grad(const LookupGradArgs& a, int dtype, void* scratch, hipStream_t s);

}  // namespace gs
