// ops_linear_ce.cu -- the vocabulary projection joined with its softmax cross entropy: sequence_cross_entropy
// (ops.cpp:1908-1979) of linear (ops.cpp:714-745), without keeping the logits.
//
//   l = X W^T + b;  loss_p = (1 - s) (lse_p - l_pt) + s (lse_p - mean_v l_pv),  lse_p = log sum_v exp l_pv
//   G = softmax(l) - s / V - (1 - s) [v = t]   (rows that count; zero elsewhere)
//   dX = G W,  dW = G^T X,  db = column sums of G        -- of the SUM of the losses
//
// The rows go in pieces: one piece's logits are in a scratch buffer at a time. When gradients are wanted
// they are computed right there, from the same logits, so that the three products cost 6 P V D operations;
// recomputing the logits in the backward pass would cost 8. The backward pass scales them by the upstream
// gradient over the number of rows that count, which is known only at the end.
#include <algorithm>
#include <cmath>

#include "nnb_gemm.h"
#include "nnb_internal.h"
#include "nnb_ops.h"
#include "nnb_trace.h"

namespace nnb {

namespace {

constexpr int kRowThreads = 256;
constexpr size_t kPieceBytes = size_t(256) << 20;   // logits of one piece

__device__ __forceinline__ float2 combine(float2 a, float2 b) {
	// (max, sum of exp(l - max)) of two parts; an empty part is (-inf, 0)
	const float m = fmaxf(a.x, b.x);
	if (m == -INFINITY) return make_float2(m, a.y + b.y);
	return make_float2(m, a.y * expf(a.x - m) + b.y * expf(b.x - m));
}

// One CTA per row of logits: the row's loss and, when grad, its row of G in place of the logits.
__global__ void __launch_bounds__(kRowThreads) ce_row_kernel(float* __restrict__ logits, int V,
		const int64_t* __restrict__ targets, int64_t ignore_index, float ls, int grad, float* __restrict__ row_loss,
		int* __restrict__ valid, int* err) {
	__shared__ float2 part[kRowThreads / 32];
	__shared__ float part_s[kRowThreads / 32];
	const long long r = blockIdx.x;
	float* row = logits + r * V;
	const int64_t t = targets[r];
	const bool ignored = t == ignore_index;
	if (ignored || t < 0 || t >= V) {
		if (grad)
			for (int c = threadIdx.x; c < V; c += kRowThreads) row[c] = 0.0f;
		if (threadIdx.x == 0) {
			row_loss[r] = ignored ? 0.0f : __int_as_float(0x7fc00000);
			valid[r] = 0;
			if (!ignored) atomicCAS(err, 0, kDevBadIndex);
		}
		return;
	}
	const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
	float2 ms = make_float2(-INFINITY, 0.0f);
	float total = 0.0f;
	for (int c = threadIdx.x; c < V; c += kRowThreads) {
		const float l = row[c];
		total += l;
		if (l > ms.x) {
			ms.y = ms.y * expf(ms.x - l) + 1.0f;
			ms.x = l;
		} else {
			ms.y += l == -INFINITY && ms.x == -INFINITY ? 0.0f : expf(l - ms.x);
		}
	}
#pragma unroll
	for (int o = 16; o > 0; o >>= 1) {
		ms = combine(ms, make_float2(__shfl_xor_sync(0xffffffffu, ms.x, o), __shfl_xor_sync(0xffffffffu, ms.y, o)));
		total += __shfl_xor_sync(0xffffffffu, total, o);
	}
	if (lane == 0) {
		part[warp] = ms;
		part_s[warp] = total;
	}
	__syncthreads();
	ms = part[0];
	total = part_s[0];
#pragma unroll
	for (int k = 1; k < kRowThreads / 32; ++k) {
		ms = combine(ms, part[k]);
		total += part_s[k];
	}
	// a row without a finite maximum (all -inf, or an infinity or NaN in it) has no softmax: NaN
	if (!(ms.x > -INFINITY && ms.x < INFINITY)) ms.y = __int_as_float(0x7fc00000);
	const float lt = row[t];
	__syncthreads();                               // row[t] is read before its owner replaces it
	if (threadIdx.x == 0) {
		const float lse = logf(ms.y), nll = lse - (lt - ms.x);
		row_loss[r] = ls == 0.0f ? nll : (1.0f - ls) * nll + ls * (lse - (total / (float)V - ms.x));
		valid[r] = 1;
	}
	if (!grad) return;
	const float inv = 1.0f / ms.y, spread = ls / (float)V;
	for (int c = threadIdx.x; c < V; c += kRowThreads) {
		float g = expf(row[c] - ms.x) * inv - spread;
		if (c == t) g -= 1.0f - ls;
		row[c] = g;
	}
}

// loss = sum of the row losses over their count, norm = 1 / count, in a fixed order in fp64.
__global__ void __launch_bounds__(1024) ce_mean_kernel(long long rows, const float* __restrict__ row_loss,
		const int* __restrict__ valid, float* __restrict__ loss, float* __restrict__ norm) {
	__shared__ double sums[32];
	__shared__ long long counts[32];
	const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
	double s = 0.0;
	long long n = 0;
	for (long long r = threadIdx.x; r < rows; r += 1024) {
		s += (double)row_loss[r];
		n += valid[r];
	}
#pragma unroll
	for (int o = 16; o > 0; o >>= 1) {
		s += __shfl_xor_sync(0xffffffffu, s, o);
		n += __shfl_xor_sync(0xffffffffu, n, o);
	}
	if (lane == 0) {
		sums[warp] = s;
		counts[warp] = n;
	}
	__syncthreads();
	if (warp != 0) return;
	s = sums[lane];
	n = counts[lane];
#pragma unroll
	for (int o = 16; o > 0; o >>= 1) {
		s += __shfl_xor_sync(0xffffffffu, s, o);
		n += __shfl_xor_sync(0xffffffffu, n, o);
	}
	if (lane == 0) {
		*loss = n ? (float)(s / (double)n) : __int_as_float(0x7fc00000);
		*norm = n ? 1.0f / (float)n : 0.0f;
	}
}

// dst[z] (+)= src[z] * (a b) for `groups` runs of n values, dst's dst_stride apart.
__global__ void scaled_accumulate_kernel(long long n, const float* __restrict__ src, const float* __restrict__ a,
		const float* __restrict__ b, float* __restrict__ dst, long long dst_stride, int first, int vec) {
	const float k = *a * *b;
	src += blockIdx.y * n;
	dst += blockIdx.y * dst_stride;
	const long long step = (long long)gridDim.x * blockDim.x;
	long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x;
	if (vec) {
		const float4* s4 = reinterpret_cast<const float4*>(src);
		float4* d4 = reinterpret_cast<float4*>(dst);
		for (; i < n / 4; i += step) {
			const float4 v = __ldg(s4 + i);
			float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
			if (!first) o = d4[i];
			d4[i] = make_float4(o.x + v.x * k, o.y + v.y * k, o.z + v.z * k, o.w + v.w * k);
		}
	} else {
		for (; i < n; i += step) dst[i] = (first ? 0.0f : dst[i]) + __ldg(src + i) * k;
	}
}

// Rows of one piece: as many whole 128-row tiles as keep its logits within kPieceBytes.
long long piece_rows(long long rows, long long V) {
	const long long fit = std::max<long long>(128, (long long)(kPieceBytes / sizeof(float)) / V / 128 * 128);
	return std::min(rows, fit);
}

struct Call {
	long long P, D, V, groups;
	const float *x, *w, *bias;
	const int64_t* targets;
	int64_t ignore_index;
	float ls;
	float *row_loss, *loss, *norm, *dx, *dw, *db;
	long long dw_stride, db_stride;
};

nnb_status run(cudaStream_t s, const Call& c, DeviceState* dev, float* logits, float* row_loss, int* valid) {
	const int mode = math_mode();
	const bool grad = c.dx || c.dw || c.db;
	const long long rg = c.P / c.groups;             // parameter gradients are kept per group of rows
	for (long long z = 0; z < c.groups; ++z) {
		for (long long r0 = z * rg; r0 < (z + 1) * rg;) {
			const long long n = std::min(piece_rows(rg, c.V), (z + 1) * rg - r0);
			const float* x = c.x + r0 * c.D;
			GemmDesc d;
			d.tb = 1; d.m = n; d.n = c.V; d.k = c.D;
			d.a = x; d.lda = c.D; d.b = c.w; d.ldb = c.D; d.c = logits; d.ldc = c.V; d.mode = mode;
			d.epi.bias = c.bias; d.epi.bias_mode = c.bias ? kBiasCol : kBiasNone;
			NNB_TRY(gemm_run(s, d));
			{
				TraceScope ts(s, kTraceRowwise);
				ce_row_kernel<<<(unsigned)n, kRowThreads, 0, s>>>(logits, (int)c.V, c.targets + r0, c.ignore_index, c.ls, grad,
					row_loss + r0, valid + r0, dev->error_word);
			}
			NNB_TRY(cuda_status(cudaGetLastError(), "linear_ce row launch"));
			const int first = r0 == z * rg;
			if (c.dx || c.dw)
				NNB_TRY(linear_bwd_gemms(s, n, c.D, c.V, 1, logits, x, nullptr, mode, c.w, c.dx ? c.dx + r0 * c.D : nullptr, 1,
					c.dw ? c.dw + z * c.dw_stride : nullptr, 0, first));
			if (c.db) NNB_TRY(colsum(s, logits, n, c.V, c.db + z * c.db_stride, first));
			r0 += n;
		}
	}
	{
		TraceScope ts(s, kTraceRowwise);
		ce_mean_kernel<<<1, 1024, 0, s>>>(c.P, row_loss, valid, c.loss, c.norm);
	}
	return cuda_status(cudaGetLastError(), "linear_ce mean launch");
}

}  // namespace

}  // namespace nnb

extern "C" {

nnb_status nnb_linear_ce_fwd(void* stream, size_t P, size_t D, size_t V, size_t groups, const float* x, const float* w,
		const float* bias, const int64_t* targets, int64_t ignore_index, float label_smoothing, float* row_loss,
		float* loss, float* norm, float* dx, float* dw, size_t dw_stride, float* db, size_t db_stride) {
	using namespace nnb;
	const char* who = "linear_ce_fwd";
	if (P == 0 || V == 0 || D == 0) return fail(NNB_ERR_SHAPE, "%s: empty input or weight", who);
	if (groups == 0 || P % groups != 0) return fail(NNB_ERR_SHAPE, "%s: %zu rows in %zu groups", who, P, groups);
	if (!(label_smoothing >= 0.0f && label_smoothing < 1.0f))
		return fail(NNB_ERR_INVALID, "%s: label_smoothing must be in [0, 1)", who);
	if (!x || !w || !targets || !loss || !norm) return fail(NNB_ERR_INVALID, "%s: null pointer", who);
	if (db && !bias) return fail(NNB_ERR_INVALID, "%s: a bias gradient without a bias", who);
	if (groups > 1 && ((dw && dw_stride && dw_stride < V * D) || (db && db_stride && db_stride < V)))
		return fail(NNB_ERR_INVALID, "%s: the groups' gradients overlap", who);
	if (P > (size_t(1) << 31) - 1 || V > (size_t(1) << 30) || D > (size_t(1) << 30))
		return fail(NNB_ERR_UNSUPPORTED, "%s: dimension too large", who);
	DeviceState* dev = nullptr;
	NNB_TRY(device_state(&dev));
	cudaStream_t s = static_cast<cudaStream_t>(stream);
	Call c;
	c.P = (long long)P; c.D = (long long)D; c.V = (long long)V; c.groups = (long long)groups;
	c.x = x; c.w = w; c.bias = bias; c.targets = targets; c.ignore_index = ignore_index; c.ls = label_smoothing;
	c.row_loss = row_loss; c.loss = loss; c.norm = norm; c.dx = dx; c.dw = dw; c.db = db;
	c.dw_stride = (long long)(dw_stride ? dw_stride : V * D);
	c.db_stride = (long long)(db_stride ? db_stride : V);
	const long long n = piece_rows(c.P / c.groups, c.V);
	const size_t logits_bytes = ((size_t)n * V * sizeof(float) + 255) / 256 * 256;
	void* ws = nullptr;
	NNB_TRY(scratch_alloc(&ws, logits_bytes + P * (sizeof(float) + sizeof(int)), s));
	float* losses = reinterpret_cast<float*>(static_cast<unsigned char*>(ws) + logits_bytes);
	const nnb_status st = run(s, c, dev, static_cast<float*>(ws), row_loss ? row_loss : losses,
		reinterpret_cast<int*>(losses + P));
	const nnb_status st2 = scratch_free(ws, s);
	return st != NNB_OK ? st : st2;
}

nnb_status nnb_scaled_accumulate(void* stream, size_t groups, size_t n, const float* src, const float* a, const float* b,
		float* dst, size_t dst_stride, int first) {
	using namespace nnb;
	if (n == 0 || groups == 0) return NNB_OK;
	if (!src || !a || !b || !dst) return fail(NNB_ERR_INVALID, "scaled_accumulate: null pointer");
	if (groups > 65535) return fail(NNB_ERR_UNSUPPORTED, "scaled_accumulate: more than 65535 groups");
	const size_t stride = dst_stride ? dst_stride : n;
	if (groups > 1 && stride < n) return fail(NNB_ERR_INVALID, "scaled_accumulate: the groups overlap");
	const bool vec = n % 4 == 0 && stride % 4 == 0 &&
		((reinterpret_cast<uintptr_t>(src) | reinterpret_cast<uintptr_t>(dst)) & 15) == 0;
	cudaStream_t s = static_cast<cudaStream_t>(stream);
	{
		TraceScope ts(s, kTraceRowwise);
		scaled_accumulate_kernel<<<dim3(grid_for((long long)(vec ? n / 4 : n), 256), (unsigned)groups), 256, 0, s>>>(
			(long long)n, src, a, b, dst, (long long)stride, first, vec);
	}
	return cuda_status(cudaGetLastError(), "scaled_accumulate launch");
}

}  // extern "C"
