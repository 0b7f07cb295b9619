// nnb_ops.h -- library-internal helpers shared between the op translation units.
#pragma once

#include <cuda_runtime.h>

#include "../../include/nnb.h"

namespace nnb {

constexpr int kDevBadIndex = 16;   // device error word: a target or token id outside its range

// out[j] (+)= sum over rows of g[r][j] in the fixed chunked order of ops_linear.cu.
nnb_status colsum(cudaStream_t s, const float* g, long long rows, long long cols, float* out, int first);
// dX (+)= G W and dW_z (+)= G_z^T X_z (per group of rows) of a linear backward; either may be null.
nnb_status linear_bwd_gemms(cudaStream_t s, long long rows, long long K, long long n, long long groups, const float* g,
		const float* x, const void* x_pack, int x_pack_mode, const float* w, float* dx, int dx_first, float* dw,
		long long dw_stride, int dw_first);
// The same per group of rows/groups consecutive rows: out[z*out_stride + j] (+)= sum over group z's rows.
nnb_status colsum_grouped(cudaStream_t s, const float* g, long long rows, long long cols, long long groups, float* out,
		long long out_stride, int first);

// Inverted dropout's factor for kept elements, 1 / (1 - p) in float (dropout.cpp:24); 0 for p == 1.
float dropout_keep_scale(float p);

// Elementwise ceiling for 1-D grids: enough blocks for n items, at most 148 * 64 blocks.
inline unsigned grid_for(long long n, int threads) {
	long long b = (n + threads - 1) / threads;
	if (b < 1) b = 1;
	if (b > 148 * 64) b = 148 * 64;
	return (unsigned)b;
}

// Launches a kernel of a chain: it may start while the stream's previous kernel still runs, as far as its
// chain_wait (nnb_ptx.cuh), which it calls before it touches memory. Its launch and prologue then hide behind
// the previous kernel, about 2 us of each step of a chain of short kernels.
template <typename... P, typename... A>
cudaError_t launch_chained(void (*kernel)(P...), dim3 grid, unsigned threads, size_t smem, cudaStream_t s, A&&... args) {
	cudaLaunchConfig_t c = {};
	c.gridDim = grid;
	c.blockDim = dim3(threads);
	c.dynamicSmemBytes = smem;
	c.stream = s;
	cudaLaunchAttribute a[1];
	a[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
	a[0].val.programmaticStreamSerializationAllowed = 1;
	c.attrs = a;
	c.numAttrs = 1;
	const cudaError_t e = cudaLaunchKernelEx(&c, kernel, static_cast<P>(args)...);
	if (e != cudaSuccess) (void)cudaGetLastError();      // returned here, not left for the next check
	return e;
}

}  // namespace nnb
