// ops_linear_ce.cu -- the vocabulary projection joined with its softmax cross entropy: sequence_cross_entropy
// (ops.cpp:1908-1979) of linear (ops.cpp:714-745), without keeping the logits.
//
//   l = X W^T + b;  loss_p = (1 - s) (lse_p - l_pt) + s (lse_p - mean_v l_pv),  lse_p = log sum_v exp l_pv
//   G = softmax(l) - s / V - (1 - s) [v = t]   (rows that count; zero elsewhere)
//   dX = G W,  dW = G^T X,  db = column sums of G        -- of the SUM of the losses
//
// The rows go in pieces. A piece's logits come out of the tensor core (split16.cu) with their softmax
// statistics per row and 128 columns; where no gradient is wanted that is all, and the logits are never
// written. Else they go into 128 x 64 blocks, which the next kernel turns into G in place: two fp16 parts
// take the 4 bytes that an fp32 logit took. G is read twice, K-major for dX and MN-major for dW, W and X
// likewise from one pack each. The three products cost 6 P V D operations; recomputing the logits in the
// backward pass would cost 8. The backward pass only scales the gradients by the upstream gradient over
// the number of rows that count, which is known at the end.
//
// Ranges (split16): blocks of 128 x 128 of X, W and G are scaled by their largest magnitude. An entry of G below
// 2^-17 of its block's largest loses relative precision, down to an absolute 2^-40 where the block holds a target
// (whose entry, softmax - 1, is at most 1): a token that is nobody's target and has probabilities near 2^-40 keeps
// few bits in its row of dW where other tokens of its block are targets.
#include <algorithm>
#include <cmath>

#include "nnb_internal.h"
#include "nnb_ops.h"
#include "nnb_split16.cuh"
#include "nnb_trace.h"

namespace nnb {

namespace {

using split16::kBlockBytes;
using split16::kCols;
using split16::kRows;

constexpr size_t kPieceBytes = size_t(512) << 20;   // G (and the logits before it) of one piece
constexpr size_t kPartBytes = size_t(256) << 20;    // softmax statistics of one piece
constexpr float kLog2e = 1.44269504088896341f;

// What the gradient needs of a row.
struct RowInfo {
	float top, inv;      // its largest logit and 1 / sum of exp(l - top); NaN inv: the row is NaN
	int target;          // -1: the row does not count (ignored, out of range or padding)
	int unused;
};

// A row's statistics from its parts (eight rows per CTA, 32 threads to a row: few rows must fill the GPU), its
// loss and RowInfo.
__global__ void __launch_bounds__(256) ce_rows_kernel(const float2* part, const float* part_sum,
		const float* target_logit, int parts, int rows, int rows_pad, int V, const int64_t* targets,
		int64_t ignore_index, float ls, const int* x_bad, const int* w_bad,
		float* row_loss, int* valid, RowInfo* info, int* err) {
	__shared__ float2 ms[32][9];
	__shared__ float tot[32][9];
	const int x = threadIdx.x & 7, y = threadIdx.x >> 3, r = blockIdx.x * 8 + x;
	chain_wait();
	float top = -INFINITY, sum = 0.0f, total = 0.0f;
	// (an empty part is (-inf, 0); a NaN or infinite logit leaves a NaN sum, and so does +inf as a maximum)
	auto join = [&](float2 b) {
		const float m = fmaxf(top, b.x);
		if (m == -INFINITY) {
			sum += b.y;
		} else {
			sum = sum * exp2_hw((top - m) * kLog2e) + b.y * exp2_hw((b.x - m) * kLog2e);
		}
		top = m;
	};
	if (r < rows)
#pragma unroll 4
		for (int k = y; k < parts; k += 32) {
			join(part[(long long)k * rows_pad + r]);
			if (part_sum) total += part_sum[(long long)k * rows_pad + r];
		}
	ms[y][x] = make_float2(top, sum);
	tot[y][x] = total;
	__syncthreads();
	if (y != 0 || r >= rows_pad) return;
	RowInfo o = {0.0f, 0.0f, -1, 0};
	if (r < rows) {
#pragma unroll 4
		for (int k = 1; k < 32; ++k) {
			join(ms[k][x]);
			total += tot[k][x];
		}
		const int64_t t = targets[r];
		if (t == ignore_index || t < 0 || t >= V) {
			row_loss[r] = t == ignore_index ? 0.0f : __int_as_float(0x7fc00000);
			valid[r] = 0;
			if (t != ignore_index) atomicCAS(err, 0, kDevBadIndex);
		} else {
			// no finite maximum, or a value of x or w that is not finite (packed as zero): NaN
			if (!(top > -INFINITY && top < INFINITY) || x_bad[r] || *w_bad) sum = __int_as_float(0x7fc00000);
			const float lse = logf(sum), nll = lse - (target_logit[r] - top);
			row_loss[r] = ls == 0.0f ? nll : (1.0f - ls) * nll + ls * (lse - (total / (float)V - top));
			valid[r] = 1;
			o.top = top;
			o.inv = 1.0f / sum;
			o.target = (int)t;
		}
	}
	if (info) info[r] = o;
}

__device__ __forceinline__ uint32_t half2_bits(float a, float b) {
	const __half2 h = __floats2half2_rn(a, b);
	return *reinterpret_cast<const uint32_t*>(&h);
}

// One block of 128 x 128 per CTA (two packed blocks of 64 columns, or the last one), in place: logits in, G out as
// fp16 parts with the block's scale; its column sums. A warp holds 128 columns of eight rows, four per lane. HBM
// bound: 4 bytes in and 4 out per logit (196 us for 134 M logits, 5.5 TB/s).
__global__ void __launch_bounds__(512, 2) ce_grad_kernel(float* blocks, int kw, int V, const RowInfo* info, float ls,
		int two_parts, int* shifts, float* col_part) {
	__shared__ RowInfo rows[kRows];
	__shared__ float4 sums[16][32];
	__shared__ unsigned tops[16];
	const int rb = blockIdx.y, tid = threadIdx.x, q = tid & 31, r0 = tid >> 5, c64 = blockIdx.x * 2 + (q >> 4);
	const bool in = c64 < kw;
	float* block = blocks + ((long long)rb * kw + c64) * (kRows * kCols);
	const int col = blockIdx.x * 2 * kCols + q * 4;
	const float spread = ls / (float)V;
	chain_wait();
	float4 l[8];
#pragma unroll
	for (int i = 0; i < 8; ++i)
		l[i] = in ? reinterpret_cast<const float4*>(block)[(r0 + 16 * i) * (kCols / 4) + (q & 15)] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
	if (tid < kRows) rows[tid] = info[rb * kRows + tid];
	__syncthreads();
	float4 cs = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
	unsigned top = 0;
#pragma unroll
	for (int i = 0; i < 8; ++i) {
		const RowInfo row = rows[r0 + 16 * i];
		float g[4] = {l[i].x, l[i].y, l[i].z, l[i].w};
#pragma unroll
		for (int k = 0; k < 4; ++k) {
			float v = exp2_hw((g[k] - row.top) * kLog2e) * row.inv - spread;
			if (col + k == row.target) v -= 1.0f - ls;
			g[k] = row.target >= 0 && col + k < V ? v : 0.0f;
			const unsigned bits = __float_as_uint(g[k]) & 0x7fffffffu;
			if (bits < 0x7f800000u) top = max(top, bits);          // (a NaN row stays NaN at any scale)
		}
		l[i] = make_float4(g[0], g[1], g[2], g[3]);
		cs.x += g[0];
		cs.y += g[1];
		cs.z += g[2];
		cs.w += g[3];
	}
	top = __reduce_max_sync(0xffffffffu, top);
	if (q == 0) tops[r0] = top;
	sums[r0][q] = cs;
	__syncthreads();                               // every logit of the block is in registers
#pragma unroll
	for (int k = 0; k < 16; ++k) top = max(top, tops[k]);
	const int shift = split16::block_shift(top);
	const float scale = split16::exp2_int(shift);
	if (tid == 0) shifts[rb * gridDim.x + blockIdx.x] = shift;
	if (in) {
		unsigned char* out = reinterpret_cast<unsigned char*>(block);
#pragma unroll
		for (int i = 0; i < 8; ++i) {
			const float4 v = make_float4(l[i].x * scale, l[i].y * scale, l[i].z * scale, l[i].w * scale);
			const uint2 hi = make_uint2(half2_bits(v.x, v.y), half2_bits(v.z, v.w));
			unsigned char* dst = out + (r0 + 16 * i) * (kCols * 2) + (q & 15) * 8;
			*reinterpret_cast<uint2*>(dst) = hi;
			if (two_parts) {
				const float2 h0 = __half22float2(*reinterpret_cast<const __half2*>(&hi.x)),
					h1 = __half22float2(*reinterpret_cast<const __half2*>(&hi.y));
				*reinterpret_cast<uint2*>(dst + split16::kPartBytes) =
					make_uint2(half2_bits(v.x - h0.x, v.y - h0.y), half2_bits(v.z - h1.x, v.w - h1.y));
			}
		}
	}
	if (!col_part || tid >= kRows || blockIdx.x * kRows + tid >= kw * kCols) return;
	// the sixteen warps' sums, in pairs
	const float* f = reinterpret_cast<const float*>(sums);
	float s[16];
#pragma unroll
	for (int k = 0; k < 16; ++k) s[k] = f[k * kRows + tid];
#pragma unroll
	for (int o = 8; o > 0; o >>= 1)
#pragma unroll
		for (int k = 0; k < o; ++k) s[k] += s[k + o];
	col_part[(long long)rb * kw * kCols + blockIdx.x * kRows + tid] = s[0];
}

// db (+)= the row blocks' column sums: 32 columns per CTA, warp y sums blocks y, y + 8, ..., then the eight
// sums in order.
__global__ void __launch_bounds__(256) ce_bias_kernel(const float* col_part, int row_blocks, int ld, int V,
		float* db, int first) {
	__shared__ float tile[8][32];
	const int lane = threadIdx.x & 31, y = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
	chain_wait();
	float s = 0.0f;
	if (c < V)
#pragma unroll 8
		for (int k = y; k < row_blocks; k += 8) s += col_part[(long long)k * ld + c];
	tile[y][lane] = s;
	__syncthreads();
	if (y != 0 || c >= V) return;
#pragma unroll
	for (int k = 1; k < 8; ++k) s += tile[k][lane];
	db[c] = first ? s : db[c] + s;
}

// loss = sum of the row losses over their count, norm = 1 / count, in a fixed order in fp64.
__global__ void __launch_bounds__(1024) ce_mean_kernel(long long rows, const float* row_loss,
		const int* valid, float* loss, float* norm) {
	__shared__ double sums[32];
	__shared__ long long counts[32];
	const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
	chain_wait();
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

constexpr int kScaledMax = 8;
struct ScaledList {
	nnb_scaled_grad g[kScaledMax];
	int vec[kScaledMax];
	const float *a, *b;
};

// dst_z (+)= src_z (a b) for the groups z of every entry (grid.y).
__global__ void __launch_bounds__(256) scaled_accumulate_kernel(const ScaledList l) {
	const nnb_scaled_grad& e = l.g[blockIdx.y];
	const float k = *l.a * *l.b;
	const long long n = (long long)e.n, step = gridDim.x * 256LL, i0 = blockIdx.x * 256LL + threadIdx.x;
	for (size_t z = 0; z < e.groups; ++z) {
		const float* __restrict__ src = e.src + z * e.n;
		float* __restrict__ dst = e.dst + z * e.dst_stride;
		if (l.vec[blockIdx.y]) {
			const float4* s4 = reinterpret_cast<const float4*>(src);
			float4* d4 = reinterpret_cast<float4*>(dst);
			for (long long i = i0; i < n / 4; i += step) {
				const float4 v = __ldg(s4 + i);
				float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
				if (!e.first) o = d4[i];
				d4[i] = make_float4(o.x + v.x * k, o.y + v.y * k, o.z + v.z * k, o.w + v.w * k);
			}
		} else {
			for (long long i = i0; i < n; i += step) dst[i] = (e.first ? 0.0f : dst[i]) + __ldg(src + i) * k;
		}
	}
}

struct Call {
	long long P, D, V, groups;
	const float *x, *w, *bias;
	const int64_t* targets;
	int64_t ignore_index;
	float ls;
	float *row_loss, *loss, *norm, *dx, *dw, *db;
	long long dw_stride, db_stride;
	bool grad() const { return dx || dw || db; }
	long long parts() const { return 2 * ((V + split16::kBN - 1) / split16::kBN); }
	long long kw() const { return (V + kCols - 1) / kCols; }
};

// Rows of one piece of a group: whole 128-row blocks within the scratch limits, or 128.
long long piece_rows(const Call& c) {
	const long long per_row = c.grad() ? c.kw() * kCols * 4 : c.parts() * 8;
	const long long limit = (long long)(c.grad() ? kPieceBytes : kPartBytes);
	return std::min(c.P / c.groups, std::max<long long>(kRows, limit / per_row / kRows * kRows));
}

// The scratch buffer's parts, 1 KB aligned.
struct Scratch {
	size_t total = 0;
	unsigned char* base = nullptr;
	size_t take(size_t bytes) {
		const size_t at = total;
		total += (bytes + 1023) / 1024 * 1024;
		return at;
	}
	template <typename T>
	T* at(size_t off) const { return reinterpret_cast<T*>(base + off); }
};

struct Layout {
	long long piece, blocks;                  // rows of a piece, and their 128-row blocks
	int dx_splits, dw_splits;                 // depth splits of the gradients' products
	size_t flags, wpack, wshift, xpack, xshift, g, gshift, part, part_sum, target_logit, info, losses, valid, cols, slabs;
};

Layout plan(const Call& c, Scratch& s) {
	Layout l;
	l.piece = piece_rows(c);
	l.blocks = (l.piece + kRows - 1) / kRows;
	const size_t pad = (size_t)l.blocks * kRows;
	l.dx_splits = c.dx ? split16::choose_splits(l.piece, c.D, c.V) : 1;
	l.dw_splits = c.dw ? split16::choose_splits(c.V, c.D, l.piece) : 1;
	l.flags = s.take((size_t)(1 + c.P) * sizeof(int));         // w's values that are not finite, and each row of x's
	l.wpack = s.take(split16::pack_bytes(c.V, c.D));
	l.wshift = s.take(split16::shift_bytes(c.V, c.D));
	l.xpack = s.take(split16::pack_bytes(l.piece, c.D));
	l.xshift = s.take(split16::shift_bytes(l.piece, c.D));
	l.g = s.take(c.grad() ? (size_t)l.blocks * c.kw() * kBlockBytes : 0);
	l.gshift = s.take(c.grad() ? split16::shift_bytes(l.piece, c.V) : 0);
	l.part = s.take((size_t)c.parts() * pad * sizeof(float2));
	l.part_sum = s.take(c.ls != 0.0f ? (size_t)c.parts() * pad * sizeof(float) : 0);
	l.target_logit = s.take(pad * sizeof(float));
	l.info = s.take(c.grad() ? pad * sizeof(RowInfo) : 0);
	l.losses = s.take(c.row_loss ? 0 : (size_t)c.P * sizeof(float));
	l.valid = s.take((size_t)c.P * sizeof(int));
	l.cols = s.take(c.db ? (size_t)l.blocks * c.kw() * kCols * sizeof(float) : 0);
	l.slabs = s.take(std::max(l.dx_splits > 1 ? (size_t)l.dx_splits * l.piece * c.D : 0,
		l.dw_splits > 1 ? (size_t)l.dw_splits * c.V * c.D : 0) * sizeof(float));
	return l;
}

nnb_status run(cudaStream_t s, const Call& c, DeviceState* dev, const Layout& l, const Scratch& m) {
	const int parts = math_mode() == NNB_MATH_FP32X3 ? 2 : 1;
	int* w_bad = m.at<int>(l.flags);
	float* row_loss = c.row_loss ? c.row_loss : m.at<float>(l.losses);
	int* valid = m.at<int>(l.valid);
	const long long rg = c.P / c.groups;             // parameter gradients are kept per group of rows
	NNB_CUDA_TRY(cudaMemsetAsync(w_bad, 0, (size_t)(1 + c.P) * sizeof(int), s));
	split16::Pack W, X, G;
	W.buf = m.at<void>(l.wpack); W.shift = m.at<int>(l.wshift); W.rows = c.V; W.cols = c.D;
	for (long long z = 0; z < c.groups; ++z) {
		for (long long r0 = z * rg; r0 < (z + 1) * rg;) {
			const long long n = std::min(l.piece, (z + 1) * rg - r0), blocks = (n + kRows - 1) / kRows, pad = blocks * kRows;
			const int first = r0 == z * rg;
			const float* x = c.x + r0 * c.D;
			int* x_bad = w_bad + 1 + r0;
			const split16::PackJob jobs[2] = {
				{x, n, c.D, blocks, m.at<void>(l.xpack), m.at<int>(l.xshift), x_bad, 1, {c.targets + r0, c.ignore_index, c.V}},
				{c.w, c.V, c.D, split16::even_blocks(c.V), m.at<void>(l.wpack), m.at<int>(l.wshift), w_bad, 0, {}}};
			NNB_TRY(split16::pack(s, jobs, r0 == 0 ? 2 : 1, parts));           // W with the first piece
			X.buf = m.at<void>(l.xpack); X.shift = m.at<int>(l.xshift); X.rows = n; X.cols = c.D;

			split16::Product p;
			p.bias = c.bias;
			p.targets = c.targets + r0;
			p.part = m.at<float2>(l.part);
			p.part_sum = c.ls != 0.0f ? m.at<float>(l.part_sum) : nullptr;
			p.target_logit = m.at<float>(l.target_logit);
			if (c.grad()) {
				p.blocks = m.at<float>(l.g);
				p.blocks_kw = (int)c.kw();
			}
			NNB_TRY(split16::run(s, p, c.grad() ? split16::kLogits : split16::kStats, parts, X, false, W, false, n, c.V, c.D));
			RowInfo* info = c.grad() ? m.at<RowInfo>(l.info) : nullptr;
			{
				TraceScope ts(s, kTraceRowwise);
				NNB_CUDA_TRY(launch_chained(ce_rows_kernel, (unsigned)(pad / 8), 256, 0, s, p.part, p.part_sum, p.target_logit,
					(int)c.parts(), (int)n, (int)pad, (int)c.V, p.targets, c.ignore_index, c.ls, x_bad, w_bad, row_loss + r0,
					valid + r0, info, dev->error_word));
			}
			if (c.grad()) {
				float* cols = c.db ? m.at<float>(l.cols) : nullptr;
				{
					TraceScope ts(s, kTraceRowwise);
					NNB_CUDA_TRY(launch_chained(ce_grad_kernel, dim3((unsigned)((c.kw() + 1) / 2), (unsigned)blocks), 512, 0, s,
						p.blocks, (int)c.kw(), (int)c.V, info, c.ls, (int)(parts == 2), m.at<int>(l.gshift), cols));
				}
				if (c.db) {
					TraceScope ts(s, kTraceRowwise);
					NNB_CUDA_TRY(launch_chained(ce_bias_kernel, (unsigned)((c.V + 31) / 32), 256, 0, s, cols, (int)blocks,
						(int)(c.kw() * kCols), (int)c.V, c.db + z * c.db_stride, first));
				}
				G.buf = m.at<void>(l.g); G.shift = m.at<int>(l.gshift); G.rows = n; G.cols = c.V;
			}
			// a product cut along its depth leaves its pieces in slabs, summed in order
			auto product = [&](const split16::Pack& a, bool mn_a, const split16::Pack& b, long long M,
					long long K, int max_splits, float* out, int accumulate) -> nnb_status {
				split16::Product d;
				d.splits = split16::split_count(K, std::min(max_splits, split16::choose_splits(M, c.D, K)));
				const bool cut = d.splits > 1;
				d.C = cut ? m.at<float>(l.slabs) : out;
				d.ldc = c.D; d.slab = cut ? M * c.D : 0;
				d.accumulate = !cut && accumulate;
				NNB_TRY(split16::run(s, d, split16::kStore, parts, a, mn_a, b, true, M, c.D, K));
				return cut ? split16::sum_slabs(s, d.C, d.splits, M * c.D, out, accumulate) : NNB_OK;
			};
			if (c.dx) NNB_TRY(product(G, false, W, n, c.V, l.dx_splits, c.dx + r0 * c.D, 0));                        // G W
			if (c.dw) NNB_TRY(product(G, true, X, c.V, n, l.dw_splits, c.dw + z * c.dw_stride, !first));             // G^T X
			r0 += n;
		}
	}
	{
		TraceScope ts(s, kTraceRowwise);
		NNB_CUDA_TRY(launch_chained(ce_mean_kernel, 1, 1024, 0, s, c.P, row_loss, valid, c.loss, c.norm));
	}
	return NNB_OK;
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
	if (groups > 65534) return fail(NNB_ERR_UNSUPPORTED, "%s: more than 65534 groups", who);
	if (!(label_smoothing >= 0.0f && label_smoothing < 1.0f))
		return fail(NNB_ERR_INVALID, "%s: label_smoothing must be in [0, 1)", who);
	if (!x || !w || !targets || !loss || !norm) return fail(NNB_ERR_INVALID, "%s: null pointer", who);
	if (db && !bias) return fail(NNB_ERR_INVALID, "%s: a bias gradient without a bias", who);
	if (groups > 1 && ((dw && dw_stride && dw_stride < V * D) || (db && db_stride && db_stride < V)))
		return fail(NNB_ERR_INVALID, "%s: the groups' gradients overlap", who);
	if (P > (size_t(1) << 31) - 1 || V > (size_t(1) << 30) || D > (size_t(1) << 30))
		return fail(NNB_ERR_UNSUPPORTED, "%s: dimension too large", who);
	// packed rows of w and x that a tensor map can count
	if ((V + 255) / 256 * 256 * ((D + 63) / 64) * 2 > INT32_MAX || (P + 127) / 128 * 128 * ((D + 63) / 64) * 2 > INT32_MAX)
		return fail(NNB_ERR_UNSUPPORTED, "%s: more packed rows than a tensor map holds", who);
	DeviceState* dev = nullptr;
	NNB_TRY(device_state(&dev));
	cudaStream_t s = static_cast<cudaStream_t>(stream);
	Call c;
	c.P = (long long)P; c.D = (long long)D; c.V = (long long)V; c.groups = (long long)groups;
	c.x = x; c.w = w; c.bias = bias; c.targets = targets; c.ignore_index = ignore_index; c.ls = label_smoothing;
	c.row_loss = row_loss; c.loss = loss; c.norm = norm; c.dx = dx; c.dw = dw; c.db = db;
	c.dw_stride = (long long)(dw_stride ? dw_stride : V * D);
	c.db_stride = (long long)(db_stride ? db_stride : V);
	Scratch m;
	const Layout l = plan(c, m);
	void* ws = nullptr;
	NNB_TRY(scratch_alloc(&ws, m.total, s));
	m.base = static_cast<unsigned char*>(ws);
	const nnb_status st = run(s, c, dev, l, m);
	const nnb_status st2 = scratch_free(ws, s);
	return st != NNB_OK ? st : st2;
}

nnb_status nnb_scaled_accumulate(void* stream, size_t count, const nnb_scaled_grad* grads, const float* a, const float* b) {
	using namespace nnb;
	if (count == 0) return NNB_OK;
	if (count > kScaledMax) return fail(NNB_ERR_UNSUPPORTED, "scaled_accumulate: more than %d tensors", kScaledMax);
	if (!grads || !a || !b) return fail(NNB_ERR_INVALID, "scaled_accumulate: null pointer");
	ScaledList l;
	l.a = a;
	l.b = b;
	int used = 0;
	size_t most = 0;
	for (size_t i = 0; i < count; ++i) {
		nnb_scaled_grad e = grads[i];
		if (e.n == 0 || e.groups == 0) continue;
		if (!e.src || !e.dst) return fail(NNB_ERR_INVALID, "scaled_accumulate: null pointer in tensor %zu", i);
		if (e.dst_stride == 0) e.dst_stride = e.n;
		if (e.groups > 1 && e.dst_stride < e.n) return fail(NNB_ERR_INVALID, "scaled_accumulate: the groups of tensor %zu overlap", i);
		l.vec[used] = e.n % 4 == 0 && e.dst_stride % 4 == 0 &&
			((reinterpret_cast<uintptr_t>(e.src) | reinterpret_cast<uintptr_t>(e.dst)) & 15) == 0;
		l.g[used++] = e;
		most = std::max(most, e.n);
	}
	if (used == 0) return NNB_OK;
	cudaStream_t s = static_cast<cudaStream_t>(stream);
	{
		TraceScope ts(s, kTraceRowwise);
		scaled_accumulate_kernel<<<dim3(grid_for((long long)(most + 3) / 4, 256), (unsigned)used), 256, 0, s>>>(l);
	}
	return cuda_status(cudaGetLastError(), "scaled_accumulate launch");
}

}  // extern "C"
