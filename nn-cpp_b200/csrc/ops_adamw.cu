// ops_adamw.cu -- one AdamW step (src/optim/adamw.cpp:15-24 then src/optim/adam.cpp:24-43) over a whole
// list of parameters in one launch, with the moments in 32 bits or in 8.
//
// The tensors' sizes and pointers travel in the kernel's parameters (no table in device memory, nothing
// to upload, nothing two captured graphs could share): kernel parameter blocks hold up to 32764 bytes.
// Every CTA takes one chunk of one tensor; it finds the tensor by bisecting the chunks' running count, whose
// dependent loads a CTA of 1024 elements (8 bits) feels: 203 M elements in one tensor take 601 us, in 56 tensors
// 676, in 133 702 (32 bits, chunks of 4096: 842, 847 and 855).
//
// 32 bits: the element operations and their order are adamw_kernel's (ops_elementwise.cu), so the
// results are bitwise those of one nnb_adamw_step per tensor. It moves 28 bytes per element and is
// bound by HBM: 558 us for 2^27 elements, 6.7 TB/s (the measured copy rate is 6.55).
//
// 8 bits: block-wise quantised moments in the manner of Dettmers et al. (8-bit optimizers via
// block-wise quantization, 2022), with a code chosen for arithmetic instead of a table: 256 consecutive
// elements share one fp32 unit u, and the code k (signed for m, unsigned for the root r of v) stands
// for sign(k) k^2 u, u = max / 127^2 or max / 255^2 over the block. Square-law codes are fine near the
// block's largest value (half a step is 0.8 % for m, 0.4 % for r) and reach down to u; a value is
// stored as the nearest one that a code stands for, a root above zero never as zero (an update divides
// by it). The root is stored instead of v because its range is half of v's in powers of ten. Per
// element the step moves 16 bytes instead of 28.
#include <cmath>

#include "nnb_internal.h"
#include "nnb_ops.h"
#include "nnb_trace.h"

namespace nnb {

namespace {

constexpr int kThreads = 256;
constexpr int kThreads8 = 128;           // 8-bit states
constexpr int kChunk = 4096;             // elements per CTA with 32-bit states: 4 float4 per thread
constexpr int kChunk8 = kThreads8 / 32 * NNB_ADAMW8_BLOCK;   // with 8-bit states: a block per warp
constexpr int kBlock = NNB_ADAMW8_BLOCK; // elements that share a unit: one warp, 8 per lane
constexpr float kTiny = 0x1p-100f;       // blocks whose largest value is below this are stored as zeros
static_assert(kBlock == 256 && kChunk8 % kBlock == 0, "a warp takes a block as two float4 per lane");

struct Scalars {
	float shrink, lr, b1, keep1, b2, keep2, eps, c1, c2;
	float minus_lr_c1, inv_root_c2;       // -lr / c1 and 1 / sqrt(c2), the 8-bit form's
};

// The list of one launch. kCap tensors fit in the classic 4 KB of parameters (small launches stay
// cheap) or in the 32 KB that sm_70 and later take.
template <int kCap>
struct List32 {
	static constexpr int kPerChunk = kChunk;
	Scalars s;
	int count;
	unsigned first[kCap + 1];              // first[i]: chunks before tensor i
	long long n[kCap];
	float* w[kCap];
	const float* g[kCap];
	float* m[kCap];
	float* v[kCap];
};
template <int kCap>
struct List8 {
	static constexpr int kPerChunk = kChunk8;
	Scalars s;
	int count;
	unsigned first[kCap + 1];
	long long n[kCap];
	float* w[kCap];
	const float* g[kCap];
	int8_t* m[kCap];
	uint8_t* v[kCap];
	float* mu[kCap];
	float* vu[kCap];
};
constexpr int kSmall = 56, kLarge = 480;
static_assert(sizeof(List8<kSmall>) <= 4096 && sizeof(List8<kLarge>) <= 32764, "kernel parameter size");
static_assert(sizeof(List32<kSmall>) <= 4096 && sizeof(List32<kLarge>) <= 32764, "kernel parameter size");

// Tensor whose chunks hold chunk c: the last i with first[i] <= c.
template <typename L>
__device__ __forceinline__ int find_tensor(const L& l, unsigned c) {
	int lo = 0, hi = l.count;
	while (hi - lo > 1) {
		const int mid = (lo + hi) >> 1;
		if (l.first[mid] <= c) lo = mid; else hi = mid;
	}
	return lo;
}

__device__ __forceinline__ void update32(const Scalars& s, float& w, float g, float& m, float& v) {
	w = w * s.shrink;
	m = s.b1 * m + s.keep1 * g;
	v = s.b2 * v + s.keep2 * g * g;
	w -= s.lr * (m / s.c1) / (sqrtf(v / s.c2) + s.eps);
}

template <int kCap>
__global__ void __launch_bounds__(kThreads) adamw_multi_kernel(const __grid_constant__ List32<kCap> l) {
	const int ti = find_tensor(l, blockIdx.x);
	const long long base = (long long)(blockIdx.x - l.first[ti]) * kChunk;
	const int n = (int)min((long long)kChunk, l.n[ti] - base);
	float* w = l.w[ti] + base;
	const float* g = l.g[ti] ? l.g[ti] + base : nullptr;   // null: a gradient of zeros
	float* m = l.m[ti] + base;
	float* v = l.v[ti] + base;
	const Scalars& s = l.s;
	const uintptr_t bits = reinterpret_cast<uintptr_t>(w) | reinterpret_cast<uintptr_t>(g) |
		reinterpret_cast<uintptr_t>(m) | reinterpret_cast<uintptr_t>(v);
	int done = 0;
	if ((bits & 15) == 0) {
		const int n4 = n >> 2;
#pragma unroll 2
		for (int i = threadIdx.x; i < n4; i += kThreads) {
			float4 wv = reinterpret_cast<const float4*>(w)[i], mv = reinterpret_cast<const float4*>(m)[i],
				vv = reinterpret_cast<const float4*>(v)[i];
			const float4 gv = g ? __ldg(reinterpret_cast<const float4*>(g) + i) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
			update32(s, wv.x, gv.x, mv.x, vv.x);
			update32(s, wv.y, gv.y, mv.y, vv.y);
			update32(s, wv.z, gv.z, mv.z, vv.z);
			update32(s, wv.w, gv.w, mv.w, vv.w);
			reinterpret_cast<float4*>(w)[i] = wv;
			reinterpret_cast<float4*>(m)[i] = mv;
			reinterpret_cast<float4*>(v)[i] = vv;
		}
		done = n4 * 4;
	}
	for (int i = done + threadIdx.x; i < n; i += kThreads) {
		float wk = w[i], mk = m[i], vk = v[i];
		update32(s, wk, g ? g[i] : 0.0f, mk, vk);
		w[i] = wk;
		m[i] = mk;
		v[i] = vk;
	}
}

// ---- 8-bit states -----------------------------------------------------------------------------

// Value of a code: sign(k) k^2 u (k^2 is exact; one rounding).
__device__ __forceinline__ float decode(float k, float u) { return k * fabsf(k) * u; }

// The code whose square is nearest to t = x inv: k with k^2 - k + 1/2 <= t < k^2 + k + 1/2; 0 for a NaN.
// k = floor(sqrt(t - 1/4) + 1/2), and the approximate root (relative error 2^-23) of a t made smaller by
// 2^-18 (inv_low) rounds to k or to k - 1, never above: one comparison settles it, and that is exact
// (the bound is a multiple of 1/2 below 2^17), so the code depends on t alone, not on the root's
// rounding. No code exceeds `levels` because the largest t is levels^2 (1 + 2^-23).
constexpr float kRoundMagic = 12582912.0f;                  // 1.5 * 2^23: adding it rounds to whole numbers
__device__ __forceinline__ float encode(float x, float inv, float inv_low, float& t) {
	t = x * inv;
	float r;
	asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(fmaxf(__fmaf_rn(x, inv_low, -0.25f), 0.0f)));
	const float k = __fadd_rn(__fadd_rn(r, kRoundMagic), -kRoundMagic), up = k + 1.0f;
	return t >= __fmaf_rn(k, up, 0.5f) ? up : k;
}
// The low byte of a whole number in [-128, 255], two's complement.
__device__ __forceinline__ uint32_t code_bits(float k) { return __float_as_uint(k + kRoundMagic); }
__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
	return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// One block by one warp: lane l holds elements 4l .. 4l + 3 and 128 + 4l .. 128 + 4l + 3.
struct Block8 {
	float w[8], g[8];
	uint32_t m[2], v[2];
	float mu, vu;
};

__device__ __forceinline__ int elem(int lane, int q) { return (q >> 2) * 128 + lane * 4 + (q & 3); }

__device__ __forceinline__ void load_block(Block8& b, bool vec, int n, int lane, const float* w, const float* g,
		const int8_t* m, const uint8_t* v, const float* mu, const float* vu) {
	b.mu = *mu;
	b.vu = *vu;
	if (vec) {
#pragma unroll
		for (int h = 0; h < 2; ++h) {
			const float4 wv = reinterpret_cast<const float4*>(w)[lane + 32 * h];
			const float4 gv = g ? __ldg(reinterpret_cast<const float4*>(g) + lane + 32 * h)
				: make_float4(0.0f, 0.0f, 0.0f, 0.0f);
			b.w[4 * h] = wv.x; b.w[4 * h + 1] = wv.y; b.w[4 * h + 2] = wv.z; b.w[4 * h + 3] = wv.w;
			b.g[4 * h] = gv.x; b.g[4 * h + 1] = gv.y; b.g[4 * h + 2] = gv.z; b.g[4 * h + 3] = gv.w;
			b.m[h] = reinterpret_cast<const uint32_t*>(m)[lane + 32 * h];
			b.v[h] = reinterpret_cast<const uint32_t*>(v)[lane + 32 * h];
		}
		return;
	}
	b.m[0] = b.m[1] = b.v[0] = b.v[1] = 0;
#pragma unroll
	for (int q = 0; q < 8; ++q) {
		const int i = elem(lane, q);
		const bool in = i < n;
		b.w[q] = in ? w[i] : 0.0f;
		b.g[q] = in && g ? g[i] : 0.0f;
		b.m[q >> 2] |= (in ? (uint32_t)(uint8_t)m[i] : 0u) << (8 * (q & 3));
		b.v[q >> 2] |= (in ? (uint32_t)v[i] : 0u) << (8 * (q & 3));
	}
}

// The step on a loaded block, its new units and its stores. The root r' = sqrt(v') serves both the
// update, w - (lr / c1) m' / (r' / sqrt(c2) + eps), and the stored code.
//
// Units: as unsigned integers the bit patterns of magnitudes order as the values do, NaN above infinity,
// so a block that holds a NaN or an infinity gets such a unit and reads back as not finite throughout.
// The two units and their inverses are four correctly rounded divisions that every lane would repeat:
// the lower half-warp works out m's pair, the upper half v's, and two shuffles hand the inverses over.
__device__ __forceinline__ void step_block(Block8& b, const Scalars& s, bool vec, int n,
		int lane, float* w, int8_t* m, uint8_t* v, float* mu, float* vu) {
	float mv[8], rv[8];
	unsigned top_m = 0, top_r = 0;
#pragma unroll
	for (int q = 0; q < 8; ++q) {
		const float km = (float)(int8_t)(b.m[q >> 2] >> (8 * (q & 3))), kr = (float)(uint8_t)(b.v[q >> 2] >> (8 * (q & 3)));
		const float r0 = kr * kr * b.vu, g = b.g[q];
		mv[q] = s.b1 * decode(km, b.mu) + s.keep1 * g;
		rv[q] = sqrtf(s.b2 * (r0 * r0) + s.keep2 * g * g);
		b.w[q] = b.w[q] * s.shrink + s.minus_lr_c1 * mv[q] / __fmaf_rn(rv[q], s.inv_root_c2, s.eps);
		top_m = max(top_m, __float_as_uint(mv[q]) & 0x7fffffffu);
		top_r = max(top_r, __float_as_uint(rv[q]) & 0x7fffffffu);
	}
	top_m = __reduce_max_sync(0xffffffffu, top_m);
	top_r = __reduce_max_sync(0xffffffffu, top_r);
	const float top = __uint_as_float(lane < 16 ? top_m : top_r), levels2 = lane < 16 ? 16129.0f : 65025.0f;
	const float unit = top < kTiny ? 0.0f : top / levels2, inv = top < kTiny ? 0.0f : levels2 / top;
	const float im = __shfl_sync(0xffffffffu, inv, 0), ir = __shfl_sync(0xffffffffu, inv, 16);
	constexpr float kLow = 1.0f - 0x1p-18f;
	const float im_low = im * kLow, ir_low = ir * kLow;
	uint32_t cm[8], cr[8];
#pragma unroll
	for (int q = 0; q < 8; ++q) {
		float t;
		cm[q] = code_bits(copysignf(encode(fabsf(mv[q]), im, im_low, t), mv[q]));
		const float kr = encode(rv[q], ir, ir_low, t);
		cr[q] = code_bits(fmaxf(kr, t > 0.0f ? 1.0f : 0.0f));
	}
#pragma unroll
	for (int h = 0; h < 2; ++h) {
		b.m[h] = pack4(cm[4 * h], cm[4 * h + 1], cm[4 * h + 2], cm[4 * h + 3]);
		b.v[h] = pack4(cr[4 * h], cr[4 * h + 1], cr[4 * h + 2], cr[4 * h + 3]);
	}
	if (vec) {
#pragma unroll
		for (int h = 0; h < 2; ++h) {
			reinterpret_cast<float4*>(w)[lane + 32 * h] =
				make_float4(b.w[4 * h], b.w[4 * h + 1], b.w[4 * h + 2], b.w[4 * h + 3]);
			reinterpret_cast<uint32_t*>(m)[lane + 32 * h] = b.m[h];
			reinterpret_cast<uint32_t*>(v)[lane + 32 * h] = b.v[h];
		}
	} else {
#pragma unroll
		for (int q = 0; q < 8; ++q) {
			const int i = elem(lane, q);
			if (i < n) {
				w[i] = b.w[q];
				m[i] = (int8_t)(b.m[q >> 2] >> (8 * (q & 3)));
				v[i] = (uint8_t)(b.v[q >> 2] >> (8 * (q & 3)));
			}
		}
	}
	// (every lane read the old units before the warp's reductions above)
	if (lane == 0) *mu = unit;
	if (lane == 16) *vu = unit;
}

// One block per warp, in small CTAs: 56 registers leave 36 warps on an SM, whose loads cover HBM's
// latency and each other's arithmetic (about 95 instructions per element, four fifths of the issue
// slots). 2^27 elements: 398 us, 5.4 TB/s, 0.82 of the measured copy rate; with an
// approximate reciprocal in place of the update's division 371 us, but the update is held to the 32-bit
// step's roundings. Measured against it: 64 registers and 32 warps 404 us; CTAs of 256 threads 4 to 6 %
// slower; several blocks per warp, even with the next block's loads issued ahead, 8 to 130 % slower (the
// warps drift apart in a long loop body).
template <int kCap>
__global__ void __launch_bounds__(kThreads8, 9) adamw8_multi_kernel(const __grid_constant__ List8<kCap> l) {
	const int ti = find_tensor(l, blockIdx.x);
	const long long base = (long long)(blockIdx.x - l.first[ti]) * kChunk8 + (threadIdx.x >> 5) * kBlock;
	if (base >= l.n[ti]) return;                   // warp-uniform
	const int n = (int)min((long long)kBlock, l.n[ti] - base), lane = threadIdx.x & 31;
	float* w = l.w[ti] + base;
	const float* g = l.g[ti] ? l.g[ti] + base : nullptr;
	int8_t* m = l.m[ti] + base;
	uint8_t* v = l.v[ti] + base;
	float* mu = l.mu[ti] + base / kBlock;
	float* vu = l.vu[ti] + base / kBlock;
	const bool vec = n == kBlock && ((reinterpret_cast<uintptr_t>(w) | reinterpret_cast<uintptr_t>(g)) & 15) == 0 &&
		((reinterpret_cast<uintptr_t>(m) | reinterpret_cast<uintptr_t>(v)) & 3) == 0;
	Block8 b;
	load_block(b, vec, n, lane, w, g, m, v, mu, vu);
	step_block(b, l.s, vec, n, lane, w, m, v, mu, vu);
}

// The moments that the codes stand for: m = sign(k) k^2 u, v = (k^2 u)^2. Four elements per thread.
__global__ void __launch_bounds__(kThreads) adamw8_moments_kernel(long long n, const int8_t* __restrict__ m,
		const uint8_t* __restrict__ v, const float* __restrict__ mu, const float* __restrict__ vu, float* __restrict__ mo,
		float* __restrict__ vo) {
	const uintptr_t bits4 = reinterpret_cast<uintptr_t>(m) | reinterpret_cast<uintptr_t>(v);
	const uintptr_t bits16 = reinterpret_cast<uintptr_t>(mo) | reinterpret_cast<uintptr_t>(vo);
	const bool aligned = (bits4 & 3) == 0 && (bits16 & 15) == 0;
	const long long quads = (n + 3) >> 2;
	for (long long i = blockIdx.x * (long long)kThreads + threadIdx.x; i < quads; i += (long long)gridDim.x * kThreads) {
		const long long e = i * 4;
		const float um = __ldg(mu + e / kBlock), ur = __ldg(vu + e / kBlock);
		if (aligned && e + 4 <= n) {
			const uint32_t cm = __ldg(reinterpret_cast<const uint32_t*>(m) + i), cv = __ldg(reinterpret_cast<const uint32_t*>(v) + i);
			float a[4], b[4];
#pragma unroll
			for (int q = 0; q < 4; ++q) {
				a[q] = decode((float)(int8_t)(cm >> (8 * q)), um);
				const float r = decode((float)(uint8_t)(cv >> (8 * q)), ur);
				b[q] = r * r;
			}
			reinterpret_cast<float4*>(mo)[i] = make_float4(a[0], a[1], a[2], a[3]);
			reinterpret_cast<float4*>(vo)[i] = make_float4(b[0], b[1], b[2], b[3]);
		} else {
			for (long long j = e; j < min(e + 4, n); ++j) {
				mo[j] = decode((float)m[j], um);
				const float r = decode((float)v[j], ur);
				vo[j] = r * r;
			}
		}
	}
}

// Host scalars exactly as Adam::step (adam.cpp:25-27) and AdamW::step (adamw.cpp:16) compute them.
Scalars host_scalars(float lr, float b1, float b2, float eps, float wd, long long step) {
	Scalars s;
	s.c1 = 1.0f - std::pow(b1, static_cast<float>(step));
	s.c2 = 1.0f - std::pow(b2, static_cast<float>(step));
	s.shrink = 1.0f - lr * wd;
	s.lr = lr;
	s.b1 = b1;
	s.keep1 = 1.0f - b1;
	s.b2 = b2;
	s.keep2 = 1.0f - b2;
	s.eps = eps;
	s.minus_lr_c1 = -lr / s.c1;
	s.inv_root_c2 = 1.0f / std::sqrt(s.c2);
	return s;
}

struct Spec {
	size_t count;
	const size_t* n;
	float* const* w;
	const float* const* g;
	void* const* m;
	void* const* v;
	float* const* mu;
	float* const* vu;
};

template <int kCap>
void set_states(List32<kCap>& l, int k, const Spec& a, size_t i) {
	l.m[k] = static_cast<float*>(a.m[i]);
	l.v[k] = static_cast<float*>(a.v[i]);
}
template <int kCap>
void set_states(List8<kCap>& l, int k, const Spec& a, size_t i) {
	l.m[k] = static_cast<int8_t*>(a.m[i]);
	l.v[k] = static_cast<uint8_t*>(a.v[i]);
	l.mu[k] = a.mu[i];
	l.vu[k] = a.vu[i];
}
template <int kCap>
void launch(cudaStream_t s, unsigned chunks, const List32<kCap>& l) {
	adamw_multi_kernel<kCap><<<chunks, kThreads, 0, s>>>(l);
}
template <int kCap>
void launch(cudaStream_t s, unsigned chunks, const List8<kCap>& l) {
	adamw8_multi_kernel<kCap><<<chunks, kThreads8, 0, s>>>(l);
}

// Fills lists of up to kCap non-empty tensors (and 2^31 - 1 chunks) and launches each.
template <typename List, int kCap>
nnb_status run_lists(cudaStream_t s, const Scalars& sc, const Spec& a) {
	DeviceState* dev = nullptr;
	size_t i = 0;
	while (i < a.count) {
		List l;
		l.s = sc;
		int k = 0;
		unsigned long long chunks = 0;
		for (; i < a.count && k < kCap; ++i) {
			if (a.n[i] == 0) continue;
			const unsigned long long c = (a.n[i] + List::kPerChunk - 1) / List::kPerChunk;
			if (k > 0 && chunks + c > 0x7fffffffull) break;
			l.first[k] = (unsigned)chunks;
			l.n[k] = (long long)a.n[i];
			l.w[k] = a.w[i];
			l.g[k] = a.g[i];
			set_states(l, k, a, i);
			chunks += c;
			++k;
		}
		if (k == 0) return NNB_OK;                // only empty tensors were left
		l.first[k] = (unsigned)chunks;
		l.count = k;
		NNB_TRY(device_state(&dev));
		{
			TraceScope ts(s, kTraceRowwise);
			launch(s, (unsigned)chunks, l);
		}
		NNB_TRY(cuda_status(cudaGetLastError(), "adamw multi launch"));
	}
	return NNB_OK;
}

nnb_status check_list(const char* who, size_t count, const size_t* n, float* const* w, const float* const* g,
		long long step, const Spec& a, bool units) {
	if (!n || !w || !g || !a.m || !a.v || (units && (!a.mu || !a.vu))) return fail(NNB_ERR_INVALID, "%s: null list", who);
	if (step < 1) return fail(NNB_ERR_INVALID, "%s: step counts from 1", who);
	for (size_t i = 0; i < count; ++i) {
		if (n[i] == 0) continue;
		if (!w[i] || !a.m[i] || !a.v[i] || (units && (!a.mu[i] || !a.vu[i])))
			return fail(NNB_ERR_INVALID, "%s: null pointer in tensor %zu", who, i);
		if (n[i] > (size_t(1) << 40)) return fail(NNB_ERR_UNSUPPORTED, "%s: tensor %zu is too large", who, i);
	}
	return NNB_OK;
}

}  // namespace

}  // namespace nnb

extern "C" {

nnb_status nnb_adamw_multi_step(void* stream, size_t count, const size_t* n, float* const* w, const float* const* g,
		float* const* m, float* const* v, float lr, float beta1, float beta2, float eps, float weight_decay,
		long long step) {
	using namespace nnb;
	if (count == 0) return NNB_OK;
	const Spec a{count, n, w, g, reinterpret_cast<void* const*>(m), reinterpret_cast<void* const*>(v), nullptr, nullptr};
	NNB_TRY(check_list("adamw_multi_step", count, n, w, g, step, a, false));
	cudaStream_t s = static_cast<cudaStream_t>(stream);
	const Scalars sc = host_scalars(lr, beta1, beta2, eps, weight_decay, step);
	return count <= kSmall ? run_lists<List32<kSmall>, kSmall>(s, sc, a) : run_lists<List32<kLarge>, kLarge>(s, sc, a);
}

nnb_status nnb_adamw8_multi_step(void* stream, size_t count, const size_t* n, float* const* w, const float* const* g,
		int8_t* const* m, uint8_t* const* v, float* const* m_unit, float* const* v_unit, float lr, float beta1, float beta2,
		float eps, float weight_decay, long long step) {
	using namespace nnb;
	if (count == 0) return NNB_OK;
	const Spec a{count, n, w, g, reinterpret_cast<void* const*>(m), reinterpret_cast<void* const*>(v), m_unit, v_unit};
	NNB_TRY(check_list("adamw8_multi_step", count, n, w, g, step, a, true));
	cudaStream_t s = static_cast<cudaStream_t>(stream);
	const Scalars sc = host_scalars(lr, beta1, beta2, eps, weight_decay, step);
	return count <= kSmall ? run_lists<List8<kSmall>, kSmall>(s, sc, a) : run_lists<List8<kLarge>, kLarge>(s, sc, a);
}

nnb_status nnb_adamw8_moments(void* stream, size_t n, const int8_t* m, const uint8_t* v, const float* m_unit,
		const float* v_unit, float* m_out, float* v_out) {
	using namespace nnb;
	if (n == 0) return NNB_OK;
	if (!m || !v || !m_unit || !v_unit || !m_out || !v_out) return fail(NNB_ERR_INVALID, "adamw8_moments: null pointer");
	cudaStream_t s = static_cast<cudaStream_t>(stream);
	{
		TraceScope ts(s, kTraceRowwise);
		adamw8_moments_kernel<<<grid_for((long long)(n + 3) / 4, kThreads), kThreads, 0, s>>>((long long)n, m, v, m_unit,
			v_unit, m_out, v_out);
	}
	return cuda_status(cudaGetLastError(), "adamw8_moments launch");
}

}  // extern "C"
