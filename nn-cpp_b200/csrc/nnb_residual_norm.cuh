// nnb_residual_norm.cuh -- what the residual norm's forward and backward share (ops_residual_norm.cu), and
// the backward kernel, whose many instances are compiled in four translation units of their own
// (ops_residual_norm_{vec,scalar}{,_post}.cu).
#pragma once

#include <algorithm>

#include "nnb_internal.h"
#include "nnb_ops.h"
#include "nnb_ptx.cuh"

namespace nnb {
namespace resnorm {

constexpr int kCta = 256;                // threads of a CTA whose rows need at most that many
constexpr int kMaxD = 16384;             // columns that 1024 threads hold, 16 each
constexpr int kArrays = 5;               // parameter sums: gamma, beta, post gamma, post beta, gate
// Sums of the forms are kept back to back: where the sum `array` of a form is, or how many there are (kArrays).
__host__ __device__ constexpr int sum_index(int array, bool layer, bool post, bool gate_param) {
	return (array > 0) + (array > 1 && layer) + (array > 2 && post) + (array > 3 && post && layer) + (array > 4 && gate_param);
}
// CTAs per SM that the backward's registers allow: rows of at most 256 threads three (80 registers), two
// with a gate or post's norm (128: their sums and operands); longer rows one (128 or 64 registers)
__host__ __device__ constexpr int bwd_ctas(bool sums, int max_t) { return max_t > kCta ? 1 : sums ? 2 : 3; }

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
	float* part;                         // [the form's sums][groups][chunks][D]
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

__device__ __forceinline__ float shuffle_sum(float v) {
#pragma unroll
	for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
	return v;
}

// Sums over the T threads of a slot (T a power of two of warps), the same bits in every thread. One
// barrier per sum: the two halves of `buf` alternate, and a half is written again only after the barrier
// of the sum between, which every thread passes after it has read.
struct SlotSum {
	float2* buf;                         // [2][warps of the CTA]
	int T, slot, warp, lane, cta_warps, parity;
	__device__ __forceinline__ SlotSum(float2* b, int t) : buf(b), T(t), slot(threadIdx.x / t), warp(threadIdx.x >> 5),
		lane(threadIdx.x & 31), cta_warps(blockDim.x >> 5), parity(0) {}
	template <typename V>
	__device__ __forceinline__ V operator()(V v) {
		v = shuffle_sum(v);
		if (T == 32) return v;
		V* b = reinterpret_cast<V*>(buf + parity * cta_warps);
		if (lane == 0) b[warp] = v;
		asm volatile("bar.sync %0, %1;" ::"r"(1 + slot), "r"(T) : "memory");
		const int n = T >> 5;
		v = b[slot * n + (lane & (n - 1))];
		parity ^= 1;
		for (int o = n >> 1; o > 0; o >>= 1) v = add(v, shuffle(v, o));
		return v;
	}

private:
	static __device__ __forceinline__ float shuffle(float v, int o) { return __shfl_xor_sync(0xffffffffu, v, o); }
	static __device__ __forceinline__ float2 shuffle(float2 v, int o) {
		return make_float2(__shfl_xor_sync(0xffffffffu, v.x, o), __shfl_xor_sync(0xffffffffu, v.y, o));
	}
	static __device__ __forceinline__ float add(float a, float b) { return a + b; }
	static __device__ __forceinline__ float2 add(float2 a, float2 b) { return make_float2(a.x + b.x, a.y + b.y); }
};

// VEC consecutive floats (VEC = 4: one 16-byte access).
template <int VEC>
struct Pack {
	float v[VEC];
	__device__ __forceinline__ void load(const float* p) {
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

template <int VEC>
__device__ __forceinline__ void async_copy(float* dst, const float* src) {
	const uint32_t d = smem_u32(dst);
	if constexpr (VEC == 4) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(d), "l"(src) : "memory");
	else asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(d), "l"(src) : "memory");
}

// dst (+)= v under the grad_accum rule.
template <int VEC>
__device__ __forceinline__ void store_grad(float* dst, Pack<VEC> v, int first) {
	if (first) {
#pragma unroll
		for (int i = 0; i < VEC; ++i) v.v[i] = v.v[i] + 0.0f;
	} else {
		Pack<VEC> o;
		o.load(dst);
#pragma unroll
		for (int i = 0; i < VEC; ++i) v.v[i] = o.v[i] + v.v[i];
	}
	v.store(dst);
}

// Arrays staged per row: dh, dy, h and, where it is read and a row of four fits (D <= 8192), the branch.
__host__ __device__ constexpr int staged_arrays(bool branch, int cols) { return branch && cols <= 8 ? 4 : 3; }

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

// T threads per row and KV * VEC columns per thread, known to the compiler (one base address and constant
// offsets per row); kLayer, kPost, kGate: the form. grid = (chunks, groups); dynamic shared memory: the
// slots' staged rows, then (slots - 1) x D floats, one array of the CTA's sums at a time.
template <int VEC, int KV, int T, bool kLayer, bool kPost, bool kGate>
__global__ void __launch_bounds__(T > kCta ? T : kCta, bwd_ctas(kPost || kGate, T)) residual_norm_bwd_kernel(const Grad p) {
	extern __shared__ float4 dyn4[];
	__shared__ float2 buf[2 * 32];
	constexpr int kSlots = (T > kCta ? T : kCta) / T;
	constexpr bool kBranch = kPost || kGate;       // the branch is read
	constexpr int kStaged = staged_arrays(kBranch, VEC * KV);
	constexpr int kStep = T * VEC;                 // floats between a thread's groups of VEC columns
	// No load passes the wait for the staged row or a store. Single floats, and rows of 1024 threads, which have
	// an SM to themselves, ask for gamma and the gate before those (16384 x 1001 87 -> 80 us, 2048 x 8192 103 -> 101);
	// other rows leave that to the SM's other CTAs (32768 x 512 with post and gate 96 -> 87 without).
	constexpr bool kAhead = VEC == 1 || T >= 1024;
	const int slot = threadIdx.x / T, j0 = threadIdx.x % T * VEC;
	const int D = p.D;
	const float inv_d = 1.0f / (float)D;
	SlotSum sum(buf, T);
	bool in[KV];
#pragma unroll
	for (int u = 0; u < KV; ++u) in[u] = j0 + u * kStep < D;
	Pack<VEC> sg[KV], sb[kLayer ? KV : 1], spg[kPost ? KV : 1], spb[kPost && kLayer ? KV : 1], sgate[kGate ? KV : 1];
#pragma unroll
	for (int u = 0; u < KV; ++u) {
		sg[u].zero();
		if constexpr (kLayer) sb[u].zero();
		if constexpr (kPost) spg[u].zero();
		if constexpr (kPost && kLayer) spb[u].zero();
		if constexpr (kGate) sgate[u].zero();
	}
	// The row's operands, staged by asynchronous copies: each thread copies the columns it will read
	// itself (array a of this slot at stage + a * D), so it needs no barrier, and it issues the next row's
	// copies as soon as it has taken this row into registers.
	float* const dyn = reinterpret_cast<float*>(dyn4);
	float* const stage = dyn + slot * kStaged * D + j0;
	const bool with_dh = p.dh != nullptr, with_dy = p.dy != nullptr;
	auto fetch = [&](long long off) {
		auto copy = [&](int array, const float* src) {
#pragma unroll
			for (int u = 0; u < KV; ++u)
				if (in[u]) async_copy<VEC>(stage + array * D + u * kStep, src + off + u * kStep);
		};
		if (with_dh) copy(0, p.dh);
		if (with_dy) {
			copy(1, p.dy);
			copy(2, p.h);
		}
		if constexpr (kStaged == 4) copy(3, p.branch);
		cp_async_commit();
	};
	chain_wait();
	const long long q = blockIdx.x * (long long)kSlots + slot;
	long long lo = 0, hi = 0;
	if (q < p.runs) run_rows(p, q, lo, hi);
	const long long base = blockIdx.y * p.group_rows;
	// the gate's row and the rows left in its span, stepped along (a parameter gate has one row)
	const float* gate_row = nullptr;
	long long span_index = 0, span_left = 0;
	if (kGate && lo < hi) {
		span_index = (base + lo) / p.gate_span;
		span_left = p.gate_span - (base + lo) % p.gate_span;
		gate_row = p.gate + span_index * D + j0;
	}
	if (lo < hi) fetch((base + lo) * D + j0);
	for (long long r = base + lo; r < base + hi; ++r) {
		const long long off = r * D + j0;
		const float4 st = p.stats[r];
		Pack<VEC> dt[KV], hat[KV], br[kBranch ? KV : 1];
		Pack<VEC> gm[KV];
		auto load_gamma = [&](int u) {
			gm[u].zero();
			if (in[u] && with_dy) gm[u].load(p.gamma + j0 + u * kStep);
		};
		if constexpr (kAhead) {
#pragma unroll
			for (int u = 0; u < KV; ++u) load_gamma(u);
		}
		float2 ab = make_float2(0.0f, 0.0f);
		cp_async_wait<0>();
#pragma unroll
		for (int u = 0; u < KV; ++u) {
			dt[u].zero();
			if (in[u] && with_dh) dt[u].load(stage + u * kStep);
			if constexpr (kBranch) {
				br[u].zero();
				if constexpr (kStaged == 4) {
					if (in[u]) br[u].load(stage + 3 * D + u * kStep);
				} else {
					if (in[u]) br[u].load(p.branch + off + u * kStep);
				}
			}
		}
		if (with_dy) {
#pragma unroll
			for (int u = 0; u < KV; ++u) {
				Pack<VEC> dy;
				dy.zero();
				hat[u].zero();
				if constexpr (!kAhead) load_gamma(u);
				if (in[u]) {
					dy.load(stage + D + u * kStep);
					hat[u].load(stage + 2 * D + u * kStep);
				}
#pragma unroll
				for (int i = 0; i < VEC; ++i) {
					const float x = (hat[u].v[i] - st.x) * st.y, d = dy.v[i] * gm[u].v[i];
					hat[u].v[i] = x;
					ab.x += d;
					ab.y = __fmaf_rn(d, x, ab.y);
					sg[u].v[i] = __fmaf_rn(dy.v[i], x, sg[u].v[i]);
					if constexpr (kLayer) sb[u].v[i] += dy.v[i];
					dt[u].v[i] = __fmaf_rn(st.y, d, dt[u].v[i]);       // dh + inv dhat
				}
			}
		}
		if (r + 1 < base + hi) fetch(off + D);
		if (with_dy) {
			float ma = 0.0f, mb;
			if constexpr (kLayer) {
				ab = sum(ab);
				ma = st.y * (ab.x * inv_d);
				mb = st.y * (ab.y * inv_d);
			} else {
				mb = st.y * (sum(ab.y) * inv_d);
			}
#pragma unroll
			for (int u = 0; u < KV; ++u)
#pragma unroll
				for (int i = 0; i < VEC; ++i) dt[u].v[i] = dt[u].v[i] - ma - hat[u].v[i] * mb;
		}
		Pack<VEC> gt[kGate ? KV : 1];
		auto load_gate = [&](int u) {
			gt[u].zero();
			if (in[u]) gt[u].load(gate_row + u * kStep);
		};
		if constexpr (kGate && kAhead) {
#pragma unroll
			for (int u = 0; u < KV; ++u) load_gate(u);
		}
		if (p.dx) {
#pragma unroll
			for (int u = 0; u < KV; ++u)
				if (in[u]) store_grad<VEC>(p.dx + off + u * kStep, dt[u], p.dx_first);
		}
		float2 ce = make_float2(0.0f, 0.0f);
#pragma unroll
		for (int u = 0; u < KV; ++u) {
			Pack<VEC> pg, pb;
			if constexpr (kPost) {
				pg.zero();
				pb.zero();
				if (in[u]) pg.load(p.post_gamma + j0 + u * kStep);
				if constexpr (kLayer && kGate) {
					if (in[u]) pb.load(p.post_beta + j0 + u * kStep);
				}
			}
			if constexpr (kGate) {
				if constexpr (!kAhead) load_gate(u);
#pragma unroll
				for (int i = 0; i < VEC; ++i) {
					const float s = p.scale * dt[u].v[i];
					const float pv = kPost ? __fmaf_rn((br[u].v[i] - st.z) * st.w, pg.v[i], pb.v[i]) : br[u].v[i];
					sgate[u].v[i] = __fmaf_rn(s, pv, sgate[u].v[i]);
					dt[u].v[i] = s * gt[u].v[i];
				}
			} else {
#pragma unroll
				for (int i = 0; i < VEC; ++i) dt[u].v[i] *= p.scale;
			}
			if constexpr (kPost) {
#pragma unroll
				for (int i = 0; i < VEC; ++i) {
					const float x = in[u] ? (br[u].v[i] - st.z) * st.w : 0.0f, d = dt[u].v[i] * pg.v[i];
					spg[u].v[i] = __fmaf_rn(dt[u].v[i], x, spg[u].v[i]);
					if constexpr (kLayer) spb[u].v[i] += dt[u].v[i];
					br[u].v[i] = x;
					dt[u].v[i] = d;
					ce.x += d;
					ce.y = __fmaf_rn(d, x, ce.y);
				}
			}
		}
		if constexpr (kPost) {
			float mc = 0.0f, me;
			if constexpr (kLayer) {
				ce = sum(ce);
				mc = ce.x * inv_d;
				me = ce.y * inv_d;
			} else {
				me = sum(ce.y) * inv_d;
			}
#pragma unroll
			for (int u = 0; u < KV; ++u)
#pragma unroll
				for (int i = 0; i < VEC; ++i) dt[u].v[i] = st.w * (dt[u].v[i] - mc - br[u].v[i] * me);
		}
		if (p.dbranch) {
#pragma unroll
			for (int u = 0; u < KV; ++u)
				if (in[u]) store_grad<VEC>(p.dbranch + off + u * kStep, dt[u], p.dbranch_first);
		}
		if constexpr (kGate) {
			if (!p.gate_is_param && (--span_left == 0 || r + 1 == base + hi)) {
				// the last row of a span (or of a piece of one): its sum goes out and starts again
				const bool piece = p.pieces > 1;
				float* dst = piece ? p.gate_part + (blockIdx.y * p.runs + q) * D : p.dgate ? p.dgate + span_index * D : nullptr;
				++span_index;
				span_left = p.gate_span;
				gate_row += D;
#pragma unroll
				for (int u = 0; u < KV; ++u) {
					if (in[u] && dst) {
						if (piece) sgate[u].store(dst + j0 + u * kStep);
						else store_grad<VEC>(dst + j0 + u * kStep, sgate[u], p.dgate_first);
					}
					sgate[u].zero();
				}
			}
		}
	}
	// the CTA's sums, slot 0 + slot 1 + ... in order, one array at a time
	__syncthreads();                               // the staged rows are done with
	float* const fold = dyn;
	auto flush = [&](Pack<VEC>(&s)[KV], int array) {
		if (slot > 0) {
#pragma unroll
			for (int u = 0; u < KV; ++u)
				if (in[u]) s[u].store(fold + (slot - 1) * D + j0 + u * kStep);
		}
		__syncthreads();
		if (slot == 0) {
			float* dst = p.part + ((array * (long long)gridDim.y + blockIdx.y) * p.chunks + blockIdx.x) * D + j0;
#pragma unroll
			for (int u = 0; u < KV; ++u)
				if (in[u]) {
#pragma unroll
					for (int k = 0; k + 1 < kSlots; ++k)
#pragma unroll
						for (int i = 0; i < VEC; ++i) s[u].v[i] += fold[k * D + j0 + u * kStep + i];
					s[u].store(dst + u * kStep);
				}
		}
		__syncthreads();
	};
	constexpr auto at = [](int array) { return sum_index(array, kLayer, kPost, kGate); };
	flush(sg, at(0));
	if constexpr (kLayer) flush(sb, at(1));
	if constexpr (kPost) flush(spg, at(2));
	if constexpr (kPost && kLayer) flush(spb, at(3));
	if constexpr (kGate) {
		if (p.gate_is_param) flush(sgate, at(4));
	}
}

template <int VEC, int KV, int T, bool kLayer, bool kPost, bool kGate>
nnb_status launch_bwd(cudaStream_t s, const Grad& p, long long groups) {
	constexpr int kThreads = T > kCta ? T : kCta;
	const size_t smem = (size_t)(kThreads / T) * staged_arrays(kPost || kGate, VEC * KV) * p.D * sizeof(float);  // and the fold
	auto kernel = residual_norm_bwd_kernel<VEC, KV, T, kLayer, kPost, kGate>;
	if (smem > 40 * 1024)                          // with the static part: above the default 48 KB
		NNB_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
	return cuda_status(launch_chained(kernel, dim3((unsigned)p.chunks, (unsigned)groups), kThreads, smem, s, p),
		"residual_norm_bwd launch");
}

// By the threads of a row that the host chose (p.T): eight columns per thread, 16 above 8192.
template <int VEC, bool kLayer, bool kPost, bool kGate>
nnb_status dispatch_bwd(cudaStream_t s, const Grad& p, long long groups) {
	constexpr int kKV = 8 / VEC;
	if (p.D > 8 * 1024) return launch_bwd<VEC, 2 * kKV, 1024, kLayer, kPost, kGate>(s, p, groups);
	switch (p.T) {
	case 32: return launch_bwd<VEC, kKV, 32, kLayer, kPost, kGate>(s, p, groups);
	case 64: return launch_bwd<VEC, kKV, 64, kLayer, kPost, kGate>(s, p, groups);
	case 128: return launch_bwd<VEC, kKV, 128, kLayer, kPost, kGate>(s, p, groups);
	case 256: return launch_bwd<VEC, kKV, 256, kLayer, kPost, kGate>(s, p, groups);
	case 512: return launch_bwd<VEC, kKV, 512, kLayer, kPost, kGate>(s, p, groups);
	default: return launch_bwd<VEC, kKV, 1024, kLayer, kPost, kGate>(s, p, groups);
	}
}

// The backward of rows that move as float4 (vec) or as single floats, with and without post's norm.
nnb_status bwd_vec(cudaStream_t s, const Grad& p, long long groups);
nnb_status bwd_vec_post(cudaStream_t s, const Grad& p, long long groups);
nnb_status bwd_scalar(cudaStream_t s, const Grad& p, long long groups);
nnb_status bwd_scalar_post(cudaStream_t s, const Grad& p, long long groups);

}  // namespace resnorm
}  // namespace nnb
