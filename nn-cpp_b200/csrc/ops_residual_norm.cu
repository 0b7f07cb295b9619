// ops_residual_norm.cu -- the residual sum after a block joined with the norm before the next one, and
// its gradients (the reference composes it from add, ops.cpp:331, and layernorm, ops.cpp:1003-1078; it
// has no RMS norm, gate or residual scale):
//
//   p = branch, or post(branch)                   a norm after the block
//   h = x + scale * gate * p                      the residual stream
//   y = norm(h)                                   the norm before the next block
//
// norm(a) = (a - mean a) / sqrt(var a + eps) * gamma + beta  (layer), a / sqrt(mean a^2 + eps) * gamma
// (rms); post has its own gamma and beta. The gate's rows each serve rows / gate_rows consecutive rows:
// one row is a parameter per channel, one per sequence a conditioning, one per token anything.
//
// Backward, with hat the normalised rows and dhat = dy gamma:
//   dt = dh + inv (dhat - [mean dhat] - hat mean(dhat hat))   ([.]: layer only);   dx = dt
//   dgate = sum over its rows of scale p dt;   dp = scale gate dt;   dbranch = dp, or post's backward
//   dgamma = sum dy hat, dbeta = sum dy, and the same of dp for post's parameters.
//
// Both directions read every row once and, for rows of up to 4096 columns, keep it in registers: 16 bytes per
// element forward, 20 to 24 backward, so HBM bounds them (with the parameter sums' kernel, about 8 us, in the
// second figure: 32768 x 512 layer 41 us and 64 us, floors 41 and 51; 8190 x 2048 rms with post and gate 43
// and 74, floors 41 and 61). Above 4096 columns a row's 1024 threads have 64 registers each, too few for the
// backward's five sums and four operands per column, and it spills: 2048 x 8192 layer 43 + 64 us, with post and
// gate 56 + 131; 1024 x 16384 48 + 87 us and 69 + 303. Rows that do not move as float4 pay for 4-byte accesses
// (16384 x 1001 layer 45 + 81 us, with post and gate 63 + 138), rows of up to 128 columns for idle lanes
// (262144 x 64 rms 53 + 87, 131072 x 128 layer with post and gate 48 + 94).
//
// T threads share a row (a power of two of warps, so that a thread holds few columns); rows whose length is a
// multiple of 4 and whose buffers are 16-byte aligned move as float4. In the backward each T-thread slot walks
// a run of consecutive rows and keeps its columns' parameter sums in registers; the CTA's slots are summed in
// shared memory, and a second kernel sums the CTAs. Run lengths and orders depend on the rows per parameter
// group, the gate's span and D only, never on the grid or the GPU, so the sums are bitwise reproducible. All
// sums are fp32.
#include <initializer_list>

#include "nnb_ops.h"
#include "nnb_residual_norm.cuh"
#include "nnb_trace.h"

namespace nnb {

namespace {

using namespace resnorm;

struct Row {
	const float *x, *branch, *post_gamma, *post_beta, *gate, *gamma, *beta;
	float *h, *y;
	float4* stats;                       // per row: mean and inverse deviation of h, then of the branch
	long long rows, gate_span;           // gate_span: rows that share a row of the gate
	int D, layer;
	float eps, scale;
};

// mean (0 for rms) and 1 / sqrt(var + eps) of the row held in a[], whose columns past D are zeros.
template <int VEC, int KV, int T>
__device__ __forceinline__ float2 row_stats(const Pack<VEC> (&a)[KV], const bool (&in)[KV], bool layer, float inv_d, float eps,
		SlotSum& sum) {
	float mu = 0.0f;
	if (layer) {
		float s = 0.0f;
#pragma unroll
		for (int u = 0; u < KV; ++u)
#pragma unroll
			for (int i = 0; i < VEC; ++i) s += a[u].v[i];
		mu = sum(s) * inv_d;
	}
	float q = 0.0f;
#pragma unroll
	for (int u = 0; u < KV; ++u)
#pragma unroll
		for (int i = 0; i < VEC; ++i) {
			const float d = in[u] ? a[u].v[i] - mu : 0.0f;
			q = __fmaf_rn(d, d, q);
		}
	return make_float2(mu, 1.0f / sqrtf(sum(q) * inv_d + eps));
}

// a = (a - mean) inv gamma + beta; columns past D become zeros.
template <int VEC, int KV, int T>
__device__ __forceinline__ void affine(Pack<VEC> (&a)[KV], const bool (&in)[KV], float2 st, const float* gamma,
		const float* beta) {
	Pack<VEC> g[KV], b[KV];
#pragma unroll
	for (int u = 0; u < KV; ++u) {
		g[u].zero();
		if (in[u]) g[u].load(gamma + u * T * VEC);
	}
#pragma unroll
	for (int u = 0; u < KV; ++u) {
		b[u].zero();
		if (beta && in[u]) b[u].load(beta + u * T * VEC);
	}
#pragma unroll
	for (int u = 0; u < KV; ++u)
#pragma unroll
		for (int i = 0; i < VEC; ++i) a[u].v[i] = in[u] ? __fmaf_rn((a[u].v[i] - st.x) * st.y, g[u].v[i], b[u].v[i]) : 0.0f;
}

// CTAs per SM that the forward's registers must allow. Short rows live on occupancy: 32 registers where a thread
// holds four columns (262144 x 64 53 us, 61 with 37 registers); two CTAs of 512 threads (2048 x 8192 49 us, 64 with
// one); 80 registers for 16 columns (8190 x 2048 with post and gate 43 us, 49 with 99).
__host__ __device__ constexpr int fwd_ctas(int cols, int t) {
	return t == 1024 ? 1 : t == 512 ? 2 : cols <= 4 ? 8 : cols <= 8 ? 5 : 3;
}

// One row per slot of T threads, T and the columns per thread known to the compiler: the row's addresses
// are one base and constant offsets, and the sums are straight code.
template <int VEC, int KV, int T>
__global__ void __launch_bounds__(T > kCta ? T : kCta, fwd_ctas(VEC * KV, T)) residual_norm_fwd_kernel(const Row p) {
	constexpr int kSlots = (T > kCta ? T : kCta) / T;
	__shared__ float2 buf[2 * 32];
	const int slot = threadIdx.x / T, t = threadIdx.x % T;
	const long long r = blockIdx.x * (long long)kSlots + slot;
	chain_wait();
	if (r >= p.rows) return;                       // whole slots leave: the barriers are per slot
	SlotSum sum(buf, T);
	const int j0 = t * VEC;
	const float inv_d = 1.0f / (float)p.D;
	const long long off = r * p.D + j0;
	Pack<VEC> a[KV], xv[KV];
	bool in[KV];
#pragma unroll
	for (int u = 0; u < KV; ++u) {
		in[u] = j0 + u * T * VEC < p.D;
		a[u].zero();
		if (in[u] && p.branch) a[u].load(p.branch + off + u * T * VEC);
	}
#pragma unroll
	for (int u = 0; u < KV; ++u) {
		xv[u].zero();
		if (in[u]) xv[u].load(p.x + off + u * T * VEC);
	}
	float2 sb = make_float2(0.0f, 0.0f);
	if (p.post_gamma) {
		sb = row_stats<VEC, KV, T>(a, in, p.layer, inv_d, p.eps, sum);
		affine<VEC, KV, T>(a, in, sb, p.post_gamma + j0, p.post_beta ? p.post_beta + j0 : nullptr);
	}
	if (p.gate) {
		const long long g = p.gate_span == p.rows ? 0 : p.gate_span == 1 ? r : p.rows < 0x7fffffffLL
			? (unsigned)r / (unsigned)p.gate_span : r / p.gate_span;
		const float* gate = p.gate + g * p.D + j0;
#pragma unroll
		for (int u = 0; u < KV; ++u) {
			Pack<VEC> gv;
			gv.zero();
			if (in[u]) gv.load(gate + u * T * VEC);
#pragma unroll
			for (int i = 0; i < VEC; ++i) a[u].v[i] *= gv.v[i];
		}
	}
#pragma unroll
	for (int u = 0; u < KV; ++u) {
#pragma unroll
		for (int i = 0; i < VEC; ++i) a[u].v[i] = __fmaf_rn(p.scale, a[u].v[i], xv[u].v[i]);
		if (in[u] && p.h) a[u].store(p.h + off + u * T * VEC);
	}
	const float2 sh = row_stats<VEC, KV, T>(a, in, p.layer, inv_d, p.eps, sum);
	affine<VEC, KV, T>(a, in, sh, p.gamma + j0, p.beta ? p.beta + j0 : nullptr);
#pragma unroll
	for (int u = 0; u < KV; ++u)
		if (in[u]) a[u].store(p.y + off + u * T * VEC);
	if (t == 0 && p.stats) p.stats[r] = make_float4(sh.x, sh.y, sb.x, sb.y);
}

// Where a group's parameter sums go: out[array] + group * stride[array], stored or added.
struct Outs {
	float* out[kArrays];
	long long stride[kArrays];
	int first[kArrays];
};

// out (+)= the sum over a group's chunks: 32 columns per CTA, warp y of its eight sums chunks y, y + 8, ...
// and the eight sums are added in order. grid = (ceil(D / 32), groups, arrays).
__global__ void __launch_bounds__(256) residual_norm_params_kernel(const float* part, int chunks, int D,
		const Outs o) {
	__shared__ float tile[8][32];
	const int array = blockIdx.z, lane = threadIdx.x & 31, y = threadIdx.x >> 5;
	float* out = o.out[array];
	if (!out) return;
	const int j = blockIdx.x * 32 + lane;
	chain_wait();
	const float* src = part + (array * (long long)gridDim.y + blockIdx.y) * chunks * D + j;
	float s = 0.0f;
	if (j < D) {
		int c = y;
		for (; c + 8 * 15 < chunks; c += 8 * 16) {       // sixteen loads in flight, added in order
			float v[16];
#pragma unroll
			for (int k = 0; k < 16; ++k) v[k] = src[(long long)(c + 8 * k) * D];
#pragma unroll
			for (int k = 0; k < 16; ++k) s += v[k];
		}
#pragma unroll 4
		for (; c < chunks; c += 8) s += src[(long long)c * D];
	}
	tile[y][lane] = s;
	__syncthreads();
	if (y != 0 || j >= D) return;
#pragma unroll
	for (int k = 1; k < 8; ++k) s += tile[k][lane];
	float* dst = out + blockIdx.y * o.stride[array] + j;
	*dst = o.first[array] ? s + 0.0f : *dst + s;
}

// dgate row = its span's pieces in order. grid-stride over spans x D.
__global__ void residual_norm_gate_kernel(const float* part, long long spans, int pieces, int D,
		float* dgate, int first) {
	const long long total = spans * D;
	chain_wait();
	for (long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x; i < total; i += (long long)gridDim.x * blockDim.x) {
		const long long s = i / D;
		const float* src = part + s * pieces * D + (i - s * D);
		float v = 0.0f;
		for (int k = 0; k < pieces; ++k) v += src[(long long)k * D];
		dgate[i] = first ? v + 0.0f : dgate[i] + v;
	}
}

// Threads per row: the fewest power-of-two warps that leave a thread at most `cols` columns, at most 1024.
int threads_per_row(int D, int cols) {
	int t = 32;
	while (t < 1024 && (long long)t * cols < D) t *= 2;
	return t;
}

bool aligned16(std::initializer_list<const void*> ps) {
	uintptr_t m = 0;
	for (const void* p : ps) m |= reinterpret_cast<uintptr_t>(p);
	return (m & 15) == 0;
}

nnb_status check_common(const char* who, size_t R, size_t D, size_t gate_rows, int kind, const float* gate, bool post,
		const float* post_beta, const float* gamma, const float* beta, bool beta_given) {
	if (kind != NNB_NORM_LAYER && kind != NNB_NORM_RMS) return fail(NNB_ERR_INVALID, "%s: unknown norm %d", who, kind);
	if (D == 0) return fail(NNB_ERR_SHAPE, "%s: empty rows", who);
	if (D > kMaxD) return fail(NNB_ERR_UNSUPPORTED, "%s: rows of %zu values, at most %d", who, D, kMaxD);
	if (R > (size_t(1) << 31) - 1) return fail(NNB_ERR_UNSUPPORTED, "%s: too many rows", who);
	if (!gamma) return fail(NNB_ERR_INVALID, "%s: gamma is null", who);
	if (beta_given && (kind == NNB_NORM_LAYER) != (beta != nullptr))
		return fail(NNB_ERR_INVALID, "%s: a layer norm needs a beta, an rms norm has none", who);
	if (post && (kind == NNB_NORM_LAYER) != (post_beta != nullptr))
		return fail(NNB_ERR_INVALID, "%s: a layer norm needs a post_beta, an rms norm has none", who);
	if (!post && post_beta) return fail(NNB_ERR_INVALID, "%s: post_beta without post_gamma", who);
	if (gate && (gate_rows == 0 || R % gate_rows != 0))
		return fail(NNB_ERR_SHAPE, "%s: %zu gate rows do not divide %zu rows", who, gate_rows, R);
	return NNB_OK;
}

template <int VEC, int KV, int T>
nnb_status launch_fwd(cudaStream_t s, const Row& p) {
	constexpr int kThreads = T > kCta ? T : kCta, kSlots = kThreads / T;
	NNB_CUDA_TRY(launch_chained(residual_norm_fwd_kernel<VEC, KV, T>, (unsigned)((p.rows + kSlots - 1) / kSlots), kThreads, 0, s, p));
	return NNB_OK;
}

// The fewest threads that leave each at most VEC * KV columns; rows that one warp holds with fewer take
// fewer.
template <int VEC, int KV>
nnb_status dispatch_fwd(cudaStream_t s, const Row& p) {
	constexpr int kCols = VEC * KV;
	if (p.D <= 32 * kCols / 4) return launch_fwd<VEC, KV / 4, 32>(s, p);
	if (p.D <= 32 * kCols) return launch_fwd<VEC, KV, 32>(s, p);
	if (p.D <= 64 * kCols) return launch_fwd<VEC, KV, 64>(s, p);
	if (p.D <= 128 * kCols) return launch_fwd<VEC, KV, 128>(s, p);
	if (p.D <= 256 * kCols) return launch_fwd<VEC, KV, 256>(s, p);
	if (p.D <= 512 * kCols) return launch_fwd<VEC, KV, 512>(s, p);
	if (p.D <= 1024 * kCols) return launch_fwd<VEC, KV, 1024>(s, p);
	return launch_fwd<VEC, kMaxD / (1024 * VEC), 1024>(s, p);
}

// The sums over no rows: stored zeros.
nnb_status zero_rows(cudaStream_t s, const nnb_grad_out& g, size_t rows, size_t D) {
	if (!g.p || !g.first || rows == 0) return NNB_OK;
	return cuda_status(cudaMemset2DAsync(g.p, (g.stride ? g.stride : D) * sizeof(float), 0, D * sizeof(float), rows, s),
		"residual_norm_bwd zero fill");
}

}  // namespace

}  // namespace nnb

extern "C" {

nnb_status nnb_residual_norm_fwd(void* stream, size_t R, size_t D, size_t gate_rows, int kind, float eps, float scale,
		const float* x, const float* branch, const float* post_gamma, const float* post_beta, const float* gate,
		const float* gamma, const float* beta, float* h, float* y, float* stats) {
	using namespace nnb;
	NNB_TRY(check_common("residual_norm_fwd", R, D, gate_rows, kind, gate, post_gamma != nullptr, post_beta, gamma, beta,
		true));
	if (R == 0) return NNB_OK;
	if (!x || !y || (!branch) != (!h)) return fail(NNB_ERR_INVALID, "residual_norm_fwd: null pointer");
	if (!branch && (gate || post_gamma)) return fail(NNB_ERR_INVALID, "residual_norm_fwd: a gate or post_gamma without a branch");
	if (reinterpret_cast<uintptr_t>(stats) & 15) return fail(NNB_ERR_INVALID, "residual_norm_fwd: stats must be 16-byte aligned");
	DeviceState* dev = nullptr;
	NNB_TRY(device_state(&dev));
	Row p;
	p.x = x; p.branch = branch; p.post_gamma = post_gamma; p.post_beta = post_beta; p.gate = gate;
	p.gamma = gamma; p.beta = beta; p.h = h; p.y = y; p.stats = reinterpret_cast<float4*>(stats);
	p.rows = (long long)R; p.gate_span = gate ? (long long)(R / gate_rows) : 1;
	p.D = (int)D; p.layer = kind == NNB_NORM_LAYER; p.eps = eps; p.scale = scale;
	cudaStream_t s = static_cast<cudaStream_t>(stream);
	TraceScope ts(s, kTraceRowwise);
	return D % 4 == 0 && aligned16({x, branch, post_gamma, post_beta, gate, gamma, beta, h, y}) ? dispatch_fwd<4, 4>(s, p)
		: dispatch_fwd<1, 8>(s, p);
}

nnb_status nnb_residual_norm_bwd(void* stream, size_t R, size_t D, size_t groups, size_t gate_rows, int kind, float scale,
		const float* dh, const float* dy, const float* h, const float* branch, const float* post_gamma,
		const float* post_beta, const float* gate, const float* gamma, const float* stats, const nnb_grad_out* grads) {
	using namespace nnb;
	const char* who = "residual_norm_bwd";
	NNB_TRY(check_common(who, R, D, gate_rows, kind, gate, post_gamma != nullptr, post_beta, gamma, nullptr, false));
	if (groups == 0 || R % groups != 0) return fail(NNB_ERR_SHAPE, "%s: %zu rows in %zu groups", who, R, groups);
	if (groups > 65535) return fail(NNB_ERR_UNSUPPORTED, "%s: more than 65535 groups", who);
	const bool gate_param = gate && gate_rows == 1;
	if (gate && !gate_param && gate_rows % groups != 0)
		return fail(NNB_ERR_SHAPE, "%s: %zu gate rows in %zu groups", who, gate_rows, groups);
	if (!grads) return fail(NNB_ERR_INVALID, "%s: null pointer", who);
	const nnb_grad_out &gx = grads[0], &gb = grads[1], &gg = grads[4];
	// the parameters' sums, in the kernel's order
	const nnb_grad_out outs[kArrays] = {grads[5], grads[6], grads[2], grads[3], gate_param ? gg : nnb_grad_out{nullptr, 0, 1}};
	if ((kind == NNB_NORM_RMS && (outs[1].p || outs[3].p)) || (!post_gamma && (outs[2].p || outs[3].p)) || (!gate && gg.p))
		return fail(NNB_ERR_INVALID, "%s: a gradient of a parameter that is not there", who);
	for (int i = 0; i < kArrays; ++i) {
		if (outs[i].p && outs[i].stride && outs[i].stride < D && groups > 1)
			return fail(NNB_ERR_INVALID, "%s: the groups' gradients overlap", who);
		for (int j = 0; j < i; ++j)
			if (outs[i].p && outs[i].p == outs[j].p)
				return fail(NNB_ERR_INVALID, "%s: two parameters share a gradient buffer", who);
	}
	cudaStream_t s = static_cast<cudaStream_t>(stream);
	if (R == 0) {
		for (const nnb_grad_out& g : outs) NNB_TRY(zero_rows(s, g, groups, D));
		return gate_param || !gate ? NNB_OK : zero_rows(s, nnb_grad_out{gg.p, D, gg.first}, gate_rows, D);
	}
	const bool needs_branch = gate || post_gamma;
	if (!stats || (!dh && !dy) || (dy && !h) || (needs_branch && !branch)) return fail(NNB_ERR_INVALID, "%s: null pointer", who);
	if (reinterpret_cast<uintptr_t>(stats) & 15) return fail(NNB_ERR_INVALID, "%s: stats must be 16-byte aligned", who);
	DeviceState* dev = nullptr;
	NNB_TRY(device_state(&dev));
	Grad p;
	p.dh = dh; p.dy = dy; p.h = h; p.branch = branch; p.post_gamma = post_gamma; p.post_beta = post_beta;
	p.gate = gate; p.gamma = gamma; p.stats = reinterpret_cast<const float4*>(stats);
	p.dx = gx.p; p.dx_first = gx.first; p.dbranch = gb.p; p.dbranch_first = gb.first;
	p.dgate = gate_param ? nullptr : gg.p; p.dgate_first = gg.first;
	p.gate_span = gate ? (long long)(R / gate_rows) : 1;
	p.D = (int)D; p.layer = kind == NNB_NORM_LAYER; p.gate_is_param = gate_param; p.scale = scale;
	const bool vec = D % 4 == 0 && aligned16({dh, dy, h, branch, post_gamma, post_beta, gate, gamma, gx.p, gb.p, p.dgate});
	p.T = threads_per_row(p.D, 8);

	// Runs: as many as one wave of the GPU has slots, over a group's rows. With a gate per span a run is
	// whole spans or a piece of one, so that a span's sum is in one or in few runs.
	const int max_t = std::max(p.T, kCta), slots = max_t / p.T;
	p.group_rows = (long long)(R / groups);
	p.span = gate && !gate_param ? p.gate_span : p.group_rows;
	const long long wave = 148LL * slots * bwd_ctas(needs_branch, max_t), spans = p.group_rows / p.span;
	if (spans >= wave) {
		p.spans_per_run = (spans + wave - 1) / wave;
		p.run_rows = 0;
		p.pieces = 1;
		p.runs = (spans + p.spans_per_run - 1) / p.spans_per_run;
	} else {
		p.spans_per_run = 0;
		p.run_rows = (p.span + std::min(p.span, wave / spans) - 1) / std::min(p.span, wave / spans);
		p.pieces = (p.span + p.run_rows - 1) / p.run_rows;
		p.runs = spans * p.pieces;
	}
	const long long chunks = (p.runs + slots - 1) / slots;
	if (chunks > INT32_MAX) return fail(NNB_ERR_UNSUPPORTED, "%s: too many rows", who);
	p.chunks = (int)chunks;

	const bool gate_pieces = gate && !gate_param && p.pieces > 1;
	const size_t part = (size_t)sum_index(kArrays, p.layer, post_gamma != nullptr, gate_param) * groups * chunks * D;
	const size_t gpart = gate_pieces ? (size_t)groups * p.runs * D : 0;
	void* ws = nullptr;
	NNB_TRY(scratch_alloc(&ws, (part + 3 + gpart) * sizeof(float), s));
	p.part = static_cast<float*>(ws);
	p.gate_part = p.part + (part + 3) / 4 * 4;
	nnb_status st;
	{
		TraceScope ts(s, kTraceRowwise);
		st = vec ? (post_gamma ? bwd_vec_post : bwd_vec)(s, p, (long long)groups)
			: (post_gamma ? bwd_scalar_post : bwd_scalar)(s, p, (long long)groups);
	}
	Outs o;
	bool any = false;
	int arrays = 0;
	const bool kept[kArrays] = {true, p.layer != 0, post_gamma != nullptr, post_gamma && p.layer, gate_param};
	for (int i = 0; i < kArrays; ++i) {
		if (!kept[i]) continue;
		o.out[arrays] = outs[i].p;
		o.stride[arrays] = (long long)(outs[i].stride ? outs[i].stride : D);
		o.first[arrays] = outs[i].first;
		any |= outs[i].p != nullptr;
		++arrays;
	}
	if (st == NNB_OK && any) {
		TraceScope ts(s, kTraceRowwise);
		st = cuda_status(launch_chained(residual_norm_params_kernel,
			dim3((unsigned)((D + 31) / 32), (unsigned)groups, (unsigned)arrays), 256, 0, s, p.part, p.chunks, p.D, o),
			"residual_norm_params launch");
	}
	if (st == NNB_OK && gate_pieces && p.dgate) {
		TraceScope ts(s, kTraceRowwise);
		st = cuda_status(launch_chained(residual_norm_gate_kernel, grid_for((long long)gate_rows * p.D, 256), 256, 0, s,
			p.gate_part, (long long)gate_rows, (int)p.pieces, p.D, p.dgate, p.dgate_first), "residual_norm_gate launch");
	}
	const nnb_status st2 = scratch_free(ws, s);
	return st != NNB_OK ? st : st2;
}

}  // extern "C"
