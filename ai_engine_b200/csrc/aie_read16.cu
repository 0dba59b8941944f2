// The one-token kernels over states in 16 bits (seq_read.cuh), apart from the
// other sequence operators: their many head sizes take most of the time of a build.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "host.cuh"
#include "tc_ptx.cuh"
#include "seq_read.cuh"

cudaError_t aie::read16_run(const ReadArgs &a, int nt, cudaStream_t s)
{
    return a.bf16 ? read16_launch<__nv_bfloat16>(a, nt, s) : read16_launch<__half>(a, nt, s);
}
