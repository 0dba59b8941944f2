// The one-token kernels over the 4-bit cache, f16 (seq_read.cuh), apart from the
// other sequence operators: their many head sizes take most of the time of a build.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "host.cuh"
#include "tc_ptx.cuh"
#include "seq_read.cuh"

cudaError_t aie::read4_run_f16(const ReadArgs &a, int nt, cudaStream_t s) { return read4_launch<__half>(a, nt, s); }
