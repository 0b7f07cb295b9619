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
// Both directions read every row once and keep it in registers: 16 bytes per element forward, 20 to 24
// backward, so HBM bounds them. T threads share a row (a power of two of warps, so that a thread holds
// few columns); rows whose length is a multiple of 4 and whose buffers are 16-byte aligned move as
// float4. In the backward each T-thread slot walks a run of consecutive rows and keeps its columns'
// parameter sums in registers; the CTA's slots are summed in shared memory, and a second kernel sums
// the CTAs. Run lengths and orders depend on the rows per parameter group, the gate's span and D only,
// never on the grid or the GPU, so the sums are bitwise reproducible. All sums are fp32.
#include <algorithm>

#include "nnb_internal.h"
#include "nnb_ops.h"
#include "nnb_trace.h"

namespace nnb {

namespace {

constexpr int kCta = 256;                // threads of a CTA whose rows need at most that many
constexpr int kMaxD = 16384;             // columns that 1024 threads hold, 16 each
constexpr int kArrays = 5;               // parameter sums: gamma, beta, post gamma, post beta, gate
// threads of one wave of the backward, which its runs are cut for: three CTAs of 256 on each of 148 SMs
// (80 registers a thread), or 1024 threads (64 registers) where a row takes more than 256
constexpr long long wave_threads(int T) { return 148LL * (T > kCta ? 1024 : 3 * kCta); }

struct Row {
	const float *x, *branch, *post_gamma, *post_beta, *gate, *gamma, *beta;
	float *h, *y;
	float4* stats;                       // per row: mean and inverse deviation of h, then of the branch
	long long rows, gate_span;           // gate_span: rows that share a row of the gate
	int D, T, layer;
	float eps, scale;
};

struct Grad {
	const float *dh, *dy, *h, *branch, *post_gamma, *post_beta, *gate, *gamma;
	const float4* stats;
	float *dx, *dbranch, *dgate;         // dgate: one row per span (null when the gate is a parameter)
	int dx_first, dbranch_first, dgate_first;
	long long gate_span;
	int D, T, layer, gate_is_param;
	float scale;
	// runs: a group of `group_rows` rows is cut into runs; a run is `spans_per_run` whole spans, or (0)
	// one of `pieces` pieces of `run_rows` rows of one span
	long long group_rows, span, run_rows, spans_per_run, pieces, runs;
	int chunks;                          // CTAs per group
	float* part;                         // [kArrays][groups][chunks][D]
	float* gate_part;                    // [groups * runs][D], pieces of a span
};

__device__ __forceinline__ float2 shuffle_sum(float2 v) {
#pragma unroll
	for (int o = 16; o > 0; o >>= 1) {
		v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
		v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
	}
	return v;
}

// Sums over the T threads of a slot (T a multiple of 32), the same bits in every thread. One barrier per
// sum: the two halves of `buf` alternate, and a half is written again only after the barrier of the sum
// between, which every thread passes after it has read.
struct SlotSum {
	float2* buf;                         // [2][warps of the CTA]
	int T, slot, warp, lane, cta_warps, parity;
	__device__ __forceinline__ SlotSum(float2* b, int t) : buf(b), T(t), slot(threadIdx.x / t), warp(threadIdx.x >> 5),
		lane(threadIdx.x & 31), cta_warps(blockDim.x >> 5), parity(0) {}
	__device__ __forceinline__ float2 operator()(float2 v) {
		v = shuffle_sum(v);
		if (T == 32) return v;
		float2* b = buf + parity * cta_warps;
		if (lane == 0) b[warp] = v;
		asm volatile("bar.sync %0, %1;" ::"r"(1 + slot), "r"(T) : "memory");
		const int n = T >> 5;
		v = lane < n ? b[slot * n + lane] : make_float2(0.0f, 0.0f);
		parity ^= 1;
		return shuffle_sum(v);
	}
	__device__ __forceinline__ float operator()(float v) { return (*this)(make_float2(v, 0.0f)).x; }
};

// VEC consecutive floats (VEC = 4: one 16-byte access).
template <int VEC>
struct Pack {
	float v[VEC];
	__device__ __forceinline__ void load(const float* p) {
		if constexpr (VEC == 4) {
			const float4 t = __ldg(reinterpret_cast<const float4*>(p));
			v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
		} else {
			v[0] = __ldg(p);
		}
	}
	// plain load: the buffer is also written by this kernel
	__device__ __forceinline__ void load_rw(const float* p) {
		if constexpr (VEC == 4) {
			const float4 t = *reinterpret_cast<const float4*>(p);
			v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
		} else {
			v[0] = *p;
		}
	}
	__device__ __forceinline__ void store(float* p) const {
		if constexpr (VEC == 4) *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
		else *p = v[0];
	}
	__device__ __forceinline__ void zero() {
#pragma unroll
		for (int i = 0; i < VEC; ++i) v[i] = 0.0f;
	}
};

// mean (0 for rms) and 1 / sqrt(var + eps) of the row held in a[]; columns past D hold anything.
template <int VEC, int KV>
__device__ __forceinline__ float2 row_stats(const Pack<VEC> (&a)[KV], int t, int groups, int T, int layer, float inv_d,
		float eps, SlotSum& sum) {
	float mu = 0.0f;
	if (layer) {
		float s = 0.0f;
#pragma unroll
		for (int u = 0; u < KV; ++u)
			if (t + u * T < groups)
#pragma unroll
				for (int i = 0; i < VEC; ++i) s += a[u].v[i];
		mu = sum(s) * inv_d;
	}
	float q = 0.0f;
#pragma unroll
	for (int u = 0; u < KV; ++u)
		if (t + u * T < groups)
#pragma unroll
			for (int i = 0; i < VEC; ++i) {
				const float d = a[u].v[i] - mu;
				q = __fmaf_rn(d, d, q);
			}
	return make_float2(mu, 1.0f / sqrtf(sum(q) * inv_d + eps));
}

template <int VEC, int KV>
__global__ void __launch_bounds__(1024) residual_norm_fwd_kernel(const Row p) {
	__shared__ float2 buf[2 * 32];
	const int T = p.T, slot = threadIdx.x / T, t = threadIdx.x - slot * T;
	const long long r = blockIdx.x * (long long)(blockDim.x / T) + slot;
	if (r >= p.rows) return;                       // whole slots leave: the barriers are per slot
	SlotSum sum(buf, T);
	const int groups = p.D / VEC;
	const float inv_d = 1.0f / (float)p.D;
	const long long off = r * p.D;
	const float* gate = p.gate ? p.gate + (r / p.gate_span) * p.D : nullptr;
	Pack<VEC> a[KV], xv[KV];
#pragma unroll
	for (int u = 0; u < KV; ++u) {
		const int j = (t + u * T) * VEC;
		if (t + u * T < groups) {
			a[u].load(p.branch + off + j);
			xv[u].load(p.x + off + j);
		}
	}
	float2 sb = make_float2(0.0f, 0.0f);
	if (p.post_gamma) sb = row_stats<VEC, KV>(a, t, groups, T, p.layer, inv_d, p.eps, sum);
#pragma unroll
	for (int u = 0; u < KV; ++u) {
		const int j = (t + u * T) * VEC;
		if (t + u * T < groups) {
			if (p.post_gamma) {
				Pack<VEC> g, b;
				g.load(p.post_gamma + j);
				if (p.post_beta) b.load(p.post_beta + j); else b.zero();
#pragma unroll
				for (int i = 0; i < VEC; ++i) a[u].v[i] = __fmaf_rn((a[u].v[i] - sb.x) * sb.y, g.v[i], b.v[i]);
			}
			if (gate) {
				Pack<VEC> g;
				g.load(gate + j);
#pragma unroll
				for (int i = 0; i < VEC; ++i) a[u].v[i] *= g.v[i];
			}
#pragma unroll
			for (int i = 0; i < VEC; ++i) a[u].v[i] = __fmaf_rn(p.scale, a[u].v[i], xv[u].v[i]);
			a[u].store(p.h + off + j);
		}
	}
	const float2 sh = row_stats<VEC, KV>(a, t, groups, T, p.layer, inv_d, p.eps, sum);
#pragma unroll
	for (int u = 0; u < KV; ++u) {
		const int j = (t + u * T) * VEC;
		if (t + u * T < groups) {
			Pack<VEC> g, b;
			g.load(p.gamma + j);
			if (p.beta) b.load(p.beta + j); else b.zero();
#pragma unroll
			for (int i = 0; i < VEC; ++i) a[u].v[i] = __fmaf_rn((a[u].v[i] - sh.x) * sh.y, g.v[i], b.v[i]);
			a[u].store(p.y + off + j);
		}
	}
	if (t == 0 && p.stats) p.stats[r] = make_float4(sh.x, sh.y, sb.x, sb.y);
}

// dst (+)= v under the grad_accum rule.
template <int VEC>
__device__ __forceinline__ void store_grad(float* dst, Pack<VEC> v, int first) {
	if (first) {
#pragma unroll
		for (int i = 0; i < VEC; ++i) v.v[i] = v.v[i] + 0.0f;
	} else {
		Pack<VEC> o;
		o.load_rw(dst);
#pragma unroll
		for (int i = 0; i < VEC; ++i) v.v[i] = o.v[i] + v.v[i];
	}
	v.store(dst);
}

// Rows of run q of a group.
__device__ __forceinline__ void run_rows(const Grad& p, long long q, long long& lo, long long& hi) {
	if (p.spans_per_run) {
		lo = q * p.spans_per_run * p.span;
		hi = min(p.group_rows, lo + p.spans_per_run * p.span);
	} else {
		const long long s = q / p.pieces, i = q - s * p.pieces;
		lo = s * p.span + i * p.run_rows;
		hi = min((s + 1) * p.span, lo + p.run_rows);
	}
}

// kPost: post's norm and its parameters; kGate: a gate. grid = (chunks, groups); dynamic shared memory:
// (slots - 1) x D floats, one array of the CTA's sums at a time.
template <int VEC, int KV, bool kPost, bool kGate, bool kBig>
__global__ void __launch_bounds__(kBig ? 1024 : kCta, kBig ? 1 : 3) residual_norm_bwd_kernel(const Grad p) {
	extern __shared__ float4 fold4[];
	__shared__ float2 buf[2 * 32];
	const int T = p.T, slot = threadIdx.x / T, slots = blockDim.x / T, t = threadIdx.x - slot * T;
	const int D = p.D, groups = D / VEC;
	const float inv_d = 1.0f / (float)D;
	SlotSum sum(buf, T);
	Pack<VEC> sg[KV], sb[KV], spg[kPost ? KV : 1], spb[kPost ? KV : 1], sgate[kGate ? KV : 1];
#pragma unroll
	for (int u = 0; u < KV; ++u) {
		sg[u].zero();
		sb[u].zero();
		if (kPost) {
			spg[u].zero();
			spb[u].zero();
		}
		if (kGate) sgate[u].zero();
	}
	const long long q = blockIdx.x * (long long)slots + slot;
	long long lo = 0, hi = 0;
	if (q < p.runs) run_rows(p, q, lo, hi);
	const long long base = blockIdx.y * p.group_rows;
	// the gate's row and the rows left in its span, stepped along (a parameter gate has one row)
	const float* gate_row = nullptr;
	long long span_index = 0, span_left = 0;
	if (kGate && lo < hi) {
		span_index = (base + lo) / p.gate_span;
		span_left = p.gate_span - (base + lo) % p.gate_span;
		gate_row = p.gate + span_index * D;
	}
	for (long long r = base + lo; r < base + hi; ++r) {
		const long long off = r * D;
		const float4 st = p.stats[r];
		Pack<VEC> dt[KV], hat[KV], br[KV];
		float2 ab = make_float2(0.0f, 0.0f);
#pragma unroll
		for (int u = 0; u < KV; ++u) {
			const int j = (t + u * T) * VEC;
			if (t + u * T < groups) {
				if (p.dh) dt[u].load(p.dh + off + j); else dt[u].zero();
				if (kPost || kGate) br[u].load(p.branch + off + j);
				if (p.dy) {
					Pack<VEC> dy;
					dy.load(p.dy + off + j);
					hat[u].load(p.h + off + j);
					Pack<VEC> g;
					g.load(p.gamma + j);
#pragma unroll
					for (int i = 0; i < VEC; ++i) {
						const float x = (hat[u].v[i] - st.x) * st.y, d = dy.v[i] * g.v[i];
						hat[u].v[i] = x;
						ab.x += d;
						ab.y = __fmaf_rn(d, x, ab.y);
						sg[u].v[i] = __fmaf_rn(dy.v[i], x, sg[u].v[i]);
						sb[u].v[i] += dy.v[i];
						dt[u].v[i] = __fmaf_rn(st.y, d, dt[u].v[i]);   // dh + inv dhat
					}
				}
			}
		}
		if (p.dy) {                                    // the same for every thread
			ab = sum(ab);
			const float ma = p.layer ? st.y * (ab.x * inv_d) : 0.0f, mb = st.y * (ab.y * inv_d);
#pragma unroll
			for (int u = 0; u < KV; ++u)
#pragma unroll
				for (int i = 0; i < VEC; ++i) dt[u].v[i] = dt[u].v[i] - ma - hat[u].v[i] * mb;
		}
		float2 ce = make_float2(0.0f, 0.0f);
#pragma unroll
		for (int u = 0; u < KV; ++u) {
			const int j = (t + u * T) * VEC;
			if (t + u * T < groups) {
				if (p.dx) store_grad<VEC>(p.dx + off + j, dt[u], p.dx_first);
				Pack<VEC> pg, pb;
				if (kPost) {
					pg.load(p.post_gamma + j);
					if (p.post_beta) pb.load(p.post_beta + j); else pb.zero();
				}
				if (kGate) {
					Pack<VEC> gt;
					gt.load(gate_row + j);
#pragma unroll
					for (int i = 0; i < VEC; ++i) {
						const float s = p.scale * dt[u].v[i];
						const float pv = kPost ? __fmaf_rn((br[u].v[i] - st.z) * st.w, pg.v[i], pb.v[i]) : br[u].v[i];
						sgate[u].v[i] = __fmaf_rn(s, pv, sgate[u].v[i]);
						dt[u].v[i] = s * gt.v[i];
					}
				} else {
#pragma unroll
					for (int i = 0; i < VEC; ++i) dt[u].v[i] *= p.scale;
				}
				if (kPost) {
#pragma unroll
					for (int i = 0; i < VEC; ++i) {
						const float x = (br[u].v[i] - st.z) * st.w, d = dt[u].v[i] * pg.v[i];
						spg[u].v[i] = __fmaf_rn(dt[u].v[i], x, spg[u].v[i]);
						spb[u].v[i] += dt[u].v[i];
						br[u].v[i] = x;
						dt[u].v[i] = d;
						ce.x += d;
						ce.y = __fmaf_rn(d, x, ce.y);
					}
				} else if (p.dbranch) {
					store_grad<VEC>(p.dbranch + off + j, dt[u], p.dbranch_first);
				}
			}
		}
		if (kPost) {
			ce = sum(ce);
			const float mc = p.layer ? ce.x * inv_d : 0.0f, me = ce.y * inv_d;
#pragma unroll
			for (int u = 0; u < KV; ++u) {
				const int j = (t + u * T) * VEC;
				if (t + u * T < groups && p.dbranch) {
#pragma unroll
					for (int i = 0; i < VEC; ++i) dt[u].v[i] = st.w * (dt[u].v[i] - mc - br[u].v[i] * me);
					store_grad<VEC>(p.dbranch + off + j, dt[u], p.dbranch_first);
				}
			}
		}
		if (kGate && !p.gate_is_param && (--span_left == 0 || r + 1 == base + hi)) {
			// the last row of a span (or of a piece of one): its sum goes out and starts again
			const bool piece = p.pieces > 1;
			float* dst = piece ? p.gate_part + (blockIdx.y * p.runs + q) * D : p.dgate ? p.dgate + span_index * D : nullptr;
			++span_index;
			span_left = p.gate_span;
			gate_row += D;
#pragma unroll
			for (int u = 0; u < KV; ++u) {
				const int j = (t + u * T) * VEC;
				if (t + u * T < groups) {
					if (piece) sgate[u].store(dst + j);
					else if (dst) store_grad<VEC>(dst + j, sgate[u], p.dgate_first);
					sgate[u].zero();
				}
			}
		}
	}
	// the CTA's sums, slot 0 + slot 1 + ... in order, one array at a time
	float* fold = reinterpret_cast<float*>(fold4);
	auto flush = [&](Pack<VEC>(&s)[KV], int array) {
		if (slot > 0) {
#pragma unroll
			for (int u = 0; u < KV; ++u)
				if (t + u * T < groups) s[u].store(fold + (long long)(slot - 1) * D + (t + u * T) * VEC);
		}
		__syncthreads();
		if (slot == 0) {
			float* dst = p.part + ((array * (long long)gridDim.y + blockIdx.y) * p.chunks + blockIdx.x) * D;
#pragma unroll
			for (int u = 0; u < KV; ++u)
				if (t + u * T < groups) {
					const int j = (t + u * T) * VEC;
					for (int k = 0; k + 1 < slots; ++k)
#pragma unroll
						for (int i = 0; i < VEC; ++i) s[u].v[i] += fold[(long long)k * D + j + i];
					s[u].store(dst + j);
				}
		}
		__syncthreads();
	};
	flush(sg, 0);
	if (p.layer) flush(sb, 1);
	if constexpr (kPost) {
		flush(spg, 2);
		if (p.layer) flush(spb, 3);
	}
	if constexpr (kGate) {
		if (p.gate_is_param) flush(sgate, 4);
	}
}

// Where a group's parameter sums go: out[array] + group * stride[array], stored or added.
struct Outs {
	float* out[kArrays];
	long long stride[kArrays];
	int first[kArrays];
};

// out (+)= the sum over a group's chunks: 32 columns per CTA, warp y sums chunks y, y + 32, ... and the
// 32 sums are added in a fixed tree. grid = (ceil(D / 32), groups, arrays), 1024 threads.
__global__ void __launch_bounds__(1024) residual_norm_params_kernel(const float* __restrict__ part, int chunks, int D,
		const Outs o) {
	__shared__ float tile[32][33];
	const int array = blockIdx.z, lane = threadIdx.x & 31, y = threadIdx.x >> 5;
	float* out = o.out[array];
	if (!out) return;
	const int j = blockIdx.x * 32 + lane;
	const float* src = part + (array * (long long)gridDim.y + blockIdx.y) * chunks * D;
	float s = 0.0f;
	if (j < D)
		for (int c = y; c < chunks; c += 32) s += __ldg(src + (long long)c * D + j);
	tile[y][lane] = s;
	__syncthreads();
	s = tile[lane][y];                             // warp y now holds column y's 32 sums
#pragma unroll
	for (int k = 16; k > 0; k >>= 1) s += __shfl_xor_sync(0xffffffffu, s, k);
	const int jo = blockIdx.x * 32 + y;
	if (lane == 0 && jo < D) {
		float* dst = out + blockIdx.y * o.stride[array] + jo;
		*dst = o.first[array] ? s + 0.0f : *dst + s;
	}
}

// dgate row = its span's pieces in order. grid-stride over spans x D.
__global__ void residual_norm_gate_kernel(const float* __restrict__ part, long long spans, int pieces, int D,
		float* __restrict__ dgate, int first) {
	const long long total = spans * D;
	for (long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x; i < total; i += (long long)gridDim.x * blockDim.x) {
		const long long s = i / D;
		const float* src = part + s * pieces * D + (i - s * D);
		float v = 0.0f;
		for (int k = 0; k < pieces; ++k) v += __ldg(src + (long long)k * D);
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
	if (R >= (size_t(1) << 40)) return fail(NNB_ERR_UNSUPPORTED, "%s: too many rows", who);
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

template <int VEC, int KV>
void launch_fwd(cudaStream_t s, const Row& p) {
	const int cta = std::max(p.T, kCta), slots = cta / p.T;
	residual_norm_fwd_kernel<VEC, KV><<<(unsigned)((p.rows + slots - 1) / slots), cta, 0, s>>>(p);
}

template <int VEC, int KV, bool kBig>
nnb_status launch_bwd_as(cudaStream_t s, const Grad& p, long long groups) {
	const int cta = std::max(p.T, kCta), slots = cta / p.T;
	const size_t smem = (size_t)(slots - 1) * p.D * sizeof(float);    // T < 256 means D <= 2048: under 48 KB
	const dim3 grid((unsigned)p.chunks, (unsigned)groups);
	const bool post = p.post_gamma != nullptr, gate = p.gate != nullptr;
	if (post && gate) residual_norm_bwd_kernel<VEC, KV, true, true, kBig><<<grid, cta, smem, s>>>(p);
	else if (post) residual_norm_bwd_kernel<VEC, KV, true, false, kBig><<<grid, cta, smem, s>>>(p);
	else if (gate) residual_norm_bwd_kernel<VEC, KV, false, true, kBig><<<grid, cta, smem, s>>>(p);
	else residual_norm_bwd_kernel<VEC, KV, false, false, kBig><<<grid, cta, smem, s>>>(p);
	return cuda_status(cudaGetLastError(), "residual_norm_bwd launch");
}
template <int VEC, int KV>
nnb_status launch_bwd(cudaStream_t s, const Grad& p, long long groups) {
	return p.T > kCta ? launch_bwd_as<VEC, KV, true>(s, p, groups) : launch_bwd_as<VEC, KV, false>(s, p, groups);
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
	if (!x || !branch || !h || !y) return fail(NNB_ERR_INVALID, "residual_norm_fwd: null pointer");
	if (reinterpret_cast<uintptr_t>(stats) & 15) return fail(NNB_ERR_INVALID, "residual_norm_fwd: stats must be 16-byte aligned");
	Row p;
	p.x = x; p.branch = branch; p.post_gamma = post_gamma; p.post_beta = post_beta; p.gate = gate;
	p.gamma = gamma; p.beta = beta; p.h = h; p.y = y; p.stats = reinterpret_cast<float4*>(stats);
	p.rows = (long long)R; p.gate_span = gate ? (long long)(R / gate_rows) : 1;
	p.D = (int)D; p.layer = kind == NNB_NORM_LAYER; p.eps = eps; p.scale = scale;
	cudaStream_t s = static_cast<cudaStream_t>(stream);
	TraceScope ts(s, kTraceRowwise);
	if (D % 4 == 0 && aligned16({x, branch, post_gamma, post_beta, gate, gamma, beta, h, y})) {
		p.T = threads_per_row((int)D, 16);
		const int kv = (p.D / 4 + p.T - 1) / p.T;
		if (kv <= 1) launch_fwd<4, 1>(s, p);
		else if (kv <= 2) launch_fwd<4, 2>(s, p);
		else launch_fwd<4, 4>(s, p);
	} else {
		p.T = threads_per_row((int)D, 8);
		const int kv = (p.D + p.T - 1) / p.T;
		if (kv <= 4) launch_fwd<1, 4>(s, p);
		else if (kv <= 8) launch_fwd<1, 8>(s, p);
		else launch_fwd<1, 16>(s, p);
	}
	return cuda_status(cudaGetLastError(), "residual_norm_fwd launch");
}

nnb_status nnb_residual_norm_bwd(void* stream, size_t R, size_t D, size_t groups, size_t gate_rows, int kind, float scale,
		const float* dh, const float* dy, const float* h, const float* branch, const float* post_gamma,
		const float* post_beta, const float* gate, const float* gamma, const float* stats, const nnb_grad_out* dx,
		const nnb_grad_out* dbranch, const nnb_grad_out* dpost_gamma, const nnb_grad_out* dpost_beta,
		const nnb_grad_out* dgate, const nnb_grad_out* dgamma, const nnb_grad_out* dbeta) {
	using namespace nnb;
	const char* who = "residual_norm_bwd";
	NNB_TRY(check_common(who, R, D, gate_rows, kind, gate, post_gamma != nullptr, post_beta, gamma, nullptr, false));
	if (groups == 0 || R % groups != 0) return fail(NNB_ERR_SHAPE, "%s: %zu rows in %zu groups", who, R, groups);
	if (groups > 65535) return fail(NNB_ERR_UNSUPPORTED, "%s: more than 65535 groups", who);
	const bool gate_param = gate && gate_rows == 1;
	if (gate && !gate_param && gate_rows % groups != 0)
		return fail(NNB_ERR_SHAPE, "%s: %zu gate rows in %zu groups", who, gate_rows, groups);
	static const nnb_grad_out none = {nullptr, 0, 1};
	auto pick = [](const nnb_grad_out* g) { return g ? *g : none; };
	const nnb_grad_out gx = pick(dx), gb = pick(dbranch), gg = pick(dgate);
	if ((kind == NNB_NORM_RMS && (pick(dbeta).p || pick(dpost_beta).p)) || (!post_gamma && (pick(dpost_gamma).p ||
			pick(dpost_beta).p)) || (!gate && gg.p))
		return fail(NNB_ERR_INVALID, "%s: a gradient of a parameter that is not there", who);
	for (const nnb_grad_out* g : {dpost_gamma, dpost_beta, dgamma, dbeta, gate_param ? dgate : nullptr})
		if (g && g->p && g->stride && g->stride < D && groups > 1)
			return fail(NNB_ERR_INVALID, "%s: the groups' gradients overlap", who);
	const float* sums[kArrays] = {pick(dgamma).p, pick(dbeta).p, pick(dpost_gamma).p, pick(dpost_beta).p,
		gate_param ? gg.p : nullptr};
	for (int i = 0; i < kArrays; ++i)
		for (int j = 0; j < i; ++j)
			if (sums[i] && sums[i] == sums[j]) return fail(NNB_ERR_INVALID, "%s: two parameters share a gradient buffer", who);
	cudaStream_t s = static_cast<cudaStream_t>(stream);
	if (R == 0) {
		for (const nnb_grad_out* g : {dpost_gamma, dpost_beta, dgamma, dbeta, gate_param ? dgate : nullptr})
			NNB_TRY(zero_rows(s, pick(g), groups, D));
		return gate_param || !gate ? NNB_OK : zero_rows(s, nnb_grad_out{gg.p, D, gg.first}, gate_rows, D);
	}
	const bool needs_branch = gate || post_gamma;
	if (!stats || (!dh && !dy) || (dy && !h) || (needs_branch && !branch)) return fail(NNB_ERR_INVALID, "%s: null pointer", who);
	if (reinterpret_cast<uintptr_t>(stats) & 15) return fail(NNB_ERR_INVALID, "%s: stats must be 16-byte aligned", who);
	Grad p;
	p.dh = dh; p.dy = dy; p.h = h; p.branch = branch; p.post_gamma = post_gamma; p.post_beta = post_beta;
	p.gate = gate; p.gamma = gamma; p.stats = reinterpret_cast<const float4*>(stats);
	p.dx = gx.p; p.dx_first = gx.first; p.dbranch = gb.p; p.dbranch_first = gb.first;
	p.dgate = gate_param ? nullptr : gg.p; p.dgate_first = gg.first;
	p.gate_span = gate ? (long long)(R / gate_rows) : 1;
	p.D = (int)D; p.layer = kind == NNB_NORM_LAYER; p.gate_is_param = gate_param; p.scale = scale;
	const bool vec = D % 4 == 0 && aligned16({dh, dy, h, branch, post_gamma, post_beta, gate, gamma, gx.p, gb.p, p.dgate});
	p.T = threads_per_row(p.D, vec ? 8 : 4);

	// Runs. A whole wave of the GPU's threads over a group's rows, and at least one row each; with a gate
	// per span a run is whole spans or a piece of one, so that a span's sum is in one or in few runs.
	const int slots = std::max(p.T, kCta) / p.T;
	p.group_rows = (long long)(R / groups);
	p.span = gate && !gate_param ? p.gate_span : p.group_rows;
	const long long wave = wave_threads(p.T), want = std::max<long long>(1, (p.group_rows * p.T + wave - 1) / wave);
	if (p.span <= want) {
		p.spans_per_run = want / p.span;
		p.run_rows = 0;
		p.pieces = 1;
		p.runs = (p.group_rows / p.span + p.spans_per_run - 1) / p.spans_per_run;
	} else {
		p.spans_per_run = 0;
		p.run_rows = want;
		p.pieces = (p.span + want - 1) / want;
		p.runs = p.group_rows / p.span * p.pieces;
	}
	const long long chunks = (p.runs + slots - 1) / slots;
	if (chunks > INT32_MAX) return fail(NNB_ERR_UNSUPPORTED, "%s: too many rows", who);
	p.chunks = (int)chunks;

	const bool gate_pieces = gate && !gate_param && p.pieces > 1;
	const size_t part = (size_t)kArrays * groups * chunks * D, gpart = gate_pieces ? (size_t)groups * p.runs * D : 0;
	void* ws = nullptr;
	NNB_TRY(scratch_alloc(&ws, (part + 3 + gpart) * sizeof(float), s));
	p.part = static_cast<float*>(ws);
	p.gate_part = p.part + (part + 3) / 4 * 4;
	nnb_status st;
	{
		TraceScope ts(s, kTraceRowwise);
		if (vec) {
			const int kv = (p.D / 4 + p.T - 1) / p.T;
			st = kv <= 1 ? launch_bwd<4, 1>(s, p, (long long)groups) : kv <= 2 ? launch_bwd<4, 2>(s, p, (long long)groups)
				: launch_bwd<4, 4>(s, p, (long long)groups);
		} else {
			const int kv = (p.D + p.T - 1) / p.T;
			st = kv <= 4 ? launch_bwd<1, 4>(s, p, (long long)groups) : launch_bwd<1, 16>(s, p, (long long)groups);
		}
	}
	Outs o;
	const nnb_grad_out outs[kArrays] = {pick(dgamma), pick(dbeta), pick(dpost_gamma), pick(dpost_beta), gate_param ? gg : none};
	bool any = false;
	int arrays = 0;
	for (int i = 0; i < kArrays; ++i) {
		const bool computed = i < 2 || (i < 4 ? post_gamma != nullptr : gate_param);
		o.out[i] = computed ? outs[i].p : nullptr;
		o.stride[i] = (long long)(outs[i].stride ? outs[i].stride : D);
		o.first[i] = outs[i].first;
		if (o.out[i]) arrays = i + 1;
		any |= o.out[i] != nullptr;
	}
	if (st == NNB_OK && any) {
		TraceScope ts(s, kTraceRowwise);
		residual_norm_params_kernel<<<dim3((unsigned)((D + 31) / 32), (unsigned)groups, (unsigned)arrays), 1024, 0, s>>>(p.part,
			p.chunks, p.D, o);
		st = cuda_status(cudaGetLastError(), "residual_norm_params launch");
	}
	if (st == NNB_OK && gate_pieces && p.dgate) {
		TraceScope ts(s, kTraceRowwise);
		residual_norm_gate_kernel<<<grid_for((long long)gate_rows * p.D, 256), 256, 0, s>>>(p.gate_part, (long long)gate_rows,
			(int)p.pieces, p.D, p.dgate, p.dgate_first);
		st = cuda_status(cudaGetLastError(), "residual_norm_gate launch");
	}
	const nnb_status st2 = scratch_free(ws, s);
	return st != NNB_OK ? st : st2;
}

}  // extern "C"
