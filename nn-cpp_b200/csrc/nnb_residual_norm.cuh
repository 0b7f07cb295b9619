// nnb_residual_norm.cuh -- what the residual norm's forward and backward share (ops_residual_norm.cu), and
// the backward kernel, compiled for float4 rows and for single floats in translation units of their own.
#pragma once

#include <algorithm>

#include "nnb_internal.h"
#include "nnb_ptx.cuh"

namespace nnb {
namespace resnorm {

constexpr int kCta = 256;                // threads of a CTA whose rows need at most that many
constexpr int kMaxD = 16384;             // columns that 1024 threads hold, 16 each
constexpr int kArrays = 5;               // parameter sums: gamma, beta, post gamma, post beta, gate
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
		o.load_rw(dst);
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

// kLayer, kPost, kGate: the form; kMaxT: the CTA's threads, 256, or 512 or 1024 for longer rows. grid = (chunks, groups); dynamic
// shared memory: the slots' staged rows, then (slots - 1) x D floats, one array of the CTA's sums at a time.
template <int VEC, int KV, bool kLayer, bool kPost, bool kGate, int kMaxT>
__global__ void __launch_bounds__(kMaxT, bwd_ctas(kPost || kGate, kMaxT)) residual_norm_bwd_kernel(const Grad p) {
	extern __shared__ float4 dyn4[];
	__shared__ float2 buf[2 * 32];
	const int T = p.T, slot = threadIdx.x / T, slots = blockDim.x / T, t = threadIdx.x - slot * T;
	const int D = p.D, groups = D / VEC;
	const float inv_d = 1.0f / (float)D;
	SlotSum sum(buf, T);
	constexpr bool kBranch = kPost || kGate;       // the branch is read
	constexpr int kStaged = staged_arrays(kBranch, VEC * KV);
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
	float* const stage = dyn + (long long)slot * kStaged * D;
	auto fetch = [&](long long r) {
		const long long off = r * D;
#pragma unroll
		for (int u = 0; u < KV; ++u) {
			const int j = (t + u * T) * VEC;
			if (t + u * T < groups) {
				if (p.dh) async_copy<VEC>(stage + j, p.dh + off + j);
				if (p.dy) {
					async_copy<VEC>(stage + D + j, p.dy + off + j);
					async_copy<VEC>(stage + 2 * D + j, p.h + off + j);
				}
				if constexpr (kStaged == 4) async_copy<VEC>(stage + 3 * D + j, p.branch + off + j);
			}
		}
		cp_async_commit();
	};
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
	if (lo < hi) fetch(base + lo);
	for (long long r = base + lo; r < base + hi; ++r) {
		const long long off = r * D;
		const float4 st = p.stats[r];
		cp_async_wait<0>();
		Pack<VEC> dt[KV], hat[KV], br[KV];
		float2 ab = make_float2(0.0f, 0.0f);
#pragma unroll
		for (int u = 0; u < KV; ++u) {
			const int j = (t + u * T) * VEC;
			if (t + u * T < groups) {
				if (p.dh) dt[u].load_rw(stage + j); else dt[u].zero();
				if constexpr (kStaged == 4) br[u].load_rw(stage + 3 * D + j);
				else if constexpr (kBranch) br[u].load(p.branch + off + j);
				if (p.dy) {
					Pack<VEC> dy;
					dy.load_rw(stage + D + j);
					hat[u].load_rw(stage + 2 * D + j);
					Pack<VEC> g;
					g.load(p.gamma + j);
#pragma unroll
					for (int i = 0; i < VEC; ++i) {
						const float x = (hat[u].v[i] - st.x) * st.y, d = dy.v[i] * g.v[i];
						hat[u].v[i] = x;
						ab.x += d;
						ab.y = __fmaf_rn(d, x, ab.y);
						sg[u].v[i] = __fmaf_rn(dy.v[i], x, sg[u].v[i]);
						if constexpr (kLayer) sb[u].v[i] += dy.v[i];
						dt[u].v[i] = __fmaf_rn(st.y, d, dt[u].v[i]);   // dh + inv dhat
					}
				}
			}
		}
		if (r + 1 < base + hi) fetch(r + 1);
		if (p.dy) {                                    // the same for every thread
			ab = sum(ab);
			const float ma = kLayer ? st.y * (ab.x * inv_d) : 0.0f, mb = st.y * (ab.y * inv_d);
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
					if constexpr (kLayer) pb.load(p.post_beta + j); else pb.zero();
				}
				if constexpr (kGate) {
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
				if constexpr (kPost) {
#pragma unroll
					for (int i = 0; i < VEC; ++i) {
						const float x = (br[u].v[i] - st.z) * st.w, d = dt[u].v[i] * pg.v[i];
						spg[u].v[i] = __fmaf_rn(dt[u].v[i], x, spg[u].v[i]);
						if constexpr (kLayer) spb[u].v[i] += dt[u].v[i];
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
			const float mc = kLayer ? ce.x * inv_d : 0.0f, me = ce.y * inv_d;
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
	__syncthreads();                               // the staged rows are done with
	float* const fold = dyn;
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
	if constexpr (kLayer) flush(sb, 1);
	if constexpr (kPost) flush(spg, 2);
	if constexpr (kPost && kLayer) flush(spb, 3);
	if constexpr (kGate) {
		if (p.gate_is_param) flush(sgate, 4);
	}
}

template <int VEC, int KV, bool kLayer, bool kPost, bool kGate, int kMaxT>
static nnb_status launch_bwd_as(cudaStream_t s, const Grad& p, long long groups) {
	const int cta = std::max(p.T, kCta), slots = cta / p.T;
	const size_t smem = (size_t)slots * staged_arrays(kPost || kGate, VEC * KV) * p.D * sizeof(float);  // holds the fold too
	auto kernel = residual_norm_bwd_kernel<VEC, KV, kLayer, kPost, kGate, kMaxT>;
	if (smem > 48 * 1024) NNB_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
	kernel<<<dim3((unsigned)p.chunks, (unsigned)groups), cta, smem, s>>>(p);
	return cuda_status(cudaGetLastError(), "residual_norm_bwd launch");
}
template <int VEC, int KV, int kMaxT>
static nnb_status launch_bwd(cudaStream_t s, const Grad& p, long long groups) {
	const int form = (p.layer ? 4 : 0) + (p.post_gamma ? 2 : 0) + (p.gate ? 1 : 0);
	switch (form) {
	case 0: return launch_bwd_as<VEC, KV, false, false, false, kMaxT>(s, p, groups);
	case 1: return launch_bwd_as<VEC, KV, false, false, true, kMaxT>(s, p, groups);
	case 2: return launch_bwd_as<VEC, KV, false, true, false, kMaxT>(s, p, groups);
	case 3: return launch_bwd_as<VEC, KV, false, true, true, kMaxT>(s, p, groups);
	case 4: return launch_bwd_as<VEC, KV, true, false, false, kMaxT>(s, p, groups);
	case 5: return launch_bwd_as<VEC, KV, true, false, true, kMaxT>(s, p, groups);
	case 6: return launch_bwd_as<VEC, KV, true, true, false, kMaxT>(s, p, groups);
	default: return launch_bwd_as<VEC, KV, true, true, true, kMaxT>(s, p, groups);
	}
}

nnb_status residual_norm_bwd_vec(cudaStream_t s, const Grad& p, long long groups);
nnb_status residual_norm_bwd_scalar(cudaStream_t s, const Grad& p, long long groups);

}  // namespace resnorm
}  // namespace nnb
