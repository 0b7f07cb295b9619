// split16.cu -- the fp16-split product (nnb_split16.cuh): pack and the tcgen05 kernel.
//
// The kernel is warp-specialised, one CTA per SM, 12 warps:
//   warp 0     TMA producer: a stage holds a 32-deep k-block, A 128 and B 256 rows (or columns), hi[, lo];
//   warp 1     MMA issuer: kind::f16 128 x 256 x 16 into two TMEM accumulators in turn, one accumulator per
//              chunk of 128 terms (3 x 8 MMAs);
//   warps 4-11 epilogue: add each finished chunk, scaled back, into registers (128 columns per thread) while
//              the tensor core works on the next, then store or reduce.
// The 384 threads are launched with 168 registers each; warps 0-3 hand theirs down to 56 and the epilogue
// takes 224 (4 x 32 x 56 + 8 x 32 x 224 = 384 x 168), which hold the 128 sums.
// Tensor bound: 3 MMAs per 128 x 256 x 16 step, 1.6 PFLOP/s of fp16 (the measured bf16 burst rate) or 540
// TFLOP/s of the fp32 product. Measured at 137 GFLOP (32768 x 512 x 4096, each way round): 300 to 313 us (450
// TFLOP/s, the pipe 73 to 75 % active at a power-capped 1.5 GHz) where the depth is 4096 or more, 366 us with the
// depth of 512, whose epilogue writes 128 KB of logits and takes 128 exponentials per thread for every
// four chunks; 548 us for 275 GFLOP (502 TFLOP/s) with the statistics alone.
// The tile: 128 x 256 and two accumulators fill TMEM, and 128 sums per thread fill the registers. A chunk
// of 256 or 512 terms instead of 128 gains 5 % and costs 2 and 4 times the error.
#include <algorithm>
#include <atomic>

#include "nnb_ops.h"
#include "nnb_split16.cuh"
#include "nnb_trace.h"

namespace nnb {
namespace split16 {

namespace {

// ---- pack ------------------------------------------------------------------------------------

__device__ __forceinline__ uint32_t half2_bits(float a, float b) {
	const __half2 h = __floats2half2_rn(a, b);
	return *reinterpret_cast<const uint32_t*>(&h);
}

struct PackWork {
	const float* x;
	long long rows, cols;
	int kw, scale_cols, vec;
	unsigned char* out;
	int* shift;
	int* bad;
	int per_row;
	LiveRows live;
};
struct PackJobs {
	PackWork job[2];
	int first;                                 // CTAs of job 0
	int parts;
};

// One block of 128 x 128 per CTA, held in registers: 16 float4 per thread (or single floats), a warp on the 128
// columns of a row; its largest magnitude; then 8 bytes of hi and of lo out per float4. HBM bound: 4 bytes in and
// 4 out per value (131072 x 512: 97 us, 5.5 TB/s; a range pass over the matrix and a pack after it took 148; a CTA's loads and
// stores do not overlap, only those of the SM's two CTAs).
__global__ void __launch_bounds__(256, 2) pack_kernel(const PackJobs jobs) {
	__shared__ unsigned tops[8];
	const bool second = (int)blockIdx.x >= jobs.first;
	const PackWork& w = jobs.job[second];
	const int b = (int)blockIdx.x - (second ? jobs.first : 0), rb = b / w.scale_cols, cb = b - rb * w.scale_cols;
	const int q = threadIdx.x & 31, r0 = threadIdx.x >> 5;
	const long long cols = w.cols, c = cb * (long long)kRows + q * 4, row0 = rb * (long long)kRows;
	chain_wait();
	float v[16][4];
#pragma unroll
	for (int i = 0; i < 16; ++i) {
		const long long r = row0 + r0 + 8 * i;
		v[i][0] = v[i][1] = v[i][2] = v[i][3] = 0.0f;
		if (r < w.rows && c < cols) {
			const float* src = w.x + r * cols + c;
			if (w.vec) {
				const float4 t = *reinterpret_cast<const float4*>(src);
				v[i][0] = t.x; v[i][1] = t.y; v[i][2] = t.z; v[i][3] = t.w;
			} else {
#pragma unroll
				for (int k = 0; k < 4; ++k)
					if (c + k < cols) v[i][k] = src[k];
			}
		}
	}
	unsigned top = 0;
#pragma unroll
	for (int i = 0; i < 16; ++i) {
		const long long r = row0 + r0 + 8 * i;
		const bool live = r < w.rows && w.live(r);
		bool bad = false;
#pragma unroll
		for (int k = 0; k < 4; ++k) {
			const unsigned bits = __float_as_uint(v[i][k]) & 0x7fffffffu;
			bad |= bits >= 0x7f800000u;
			if (!live || bits >= 0x7f800000u) v[i][k] = 0.0f;
			else top = max(top, bits);
		}
		if (live && bad) w.bad[w.per_row ? r : 0] = 1;       // every writer writes 1
	}
	top = __reduce_max_sync(0xffffffffu, top);
	if (q == 0) tops[r0] = top;
	__syncthreads();
#pragma unroll
	for (int k = 0; k < 8; ++k) top = max(top, tops[k]);
	const int shift = block_shift(top);
	if (threadIdx.x == 0) w.shift[b] = shift;
	const int c64 = 2 * cb + (q >> 4);
	if (c64 >= w.kw) return;
	const float s = exp2_int(shift);
	unsigned char* dst = w.out + (rb * (long long)w.kw + c64) * kBlockBytes + r0 * (kCols * 2) + (q & 15) * 8;
#pragma unroll
	for (int i = 0; i < 16; ++i, dst += 8 * kCols * 2) {
		float hi[4];
#pragma unroll
		for (int k = 0; k < 4; ++k) {
			v[i][k] *= s;
			hi[k] = __half2float(__float2half_rn(v[i][k]));
		}
		*reinterpret_cast<uint2*>(dst) = make_uint2(half2_bits(hi[0], hi[1]), half2_bits(hi[2], hi[3]));
		if (jobs.parts == 2)
			*reinterpret_cast<uint2*>(dst + kPartBytes) = make_uint2(half2_bits(v[i][0] - hi[0], v[i][1] - hi[1]),
				half2_bits(v[i][2] - hi[2], v[i][3] - hi[3]));
	}
}

// ---- tcgen05 kind::f16 -----------------------------------------------------------------------

// Instruction descriptor: fp32 accumulator, fp16 A and B.
constexpr uint32_t idesc_f16(int m, int n) { return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24); }

// MN-major 16-bit operand in the 128-byte swizzle: a row of 128 bytes holds 64 consecutive M (or N) elements
// of one k; 8 k-rows form a 1024-byte group (stride byte offset to the next), and the next 64 elements sit
// `lbo` bytes further on. One MMA (K = 16) reads two groups.
__device__ __forceinline__ uint64_t smem_desc_mn_sw128(uint32_t addr, uint32_t lbo) {
	uint64_t d = 0;
	d |= (uint64_t)((addr & 0x3FFFFu) >> 4);
	d |= (uint64_t)((lbo >> 4) & 0x3FFFu) << 16;
	d |= (uint64_t)(1024u >> 4) << 32;
	d |= (uint64_t)1 << 46;
	d |= (uint64_t)2 << 61;                        // SWIZZLE_128B
	return d;
}

// mma_tf32_elect's counterpart: the whole warp executes it, one lane issues.
__device__ __forceinline__ void mma_f16_elect(uint32_t d_tmem, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
	asm volatile(
		"{\n\t.reg .pred p, e;\n\t"
		"elect.sync _|e, 0xffffffff;\n\t"
		"setp.ne.b32 p, %4, 0;\n\t"
		"@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
		"l"(a), "l"(b), "r"(idesc), "r"(accumulate)
		: "memory");
}

constexpr int kGroupM = 16;                      // row tiles walked together, for L2 reuse of B
constexpr int kAPart = kBM * kBK * 2, kBPart = kBN * kBK * 2;
constexpr int kEpiTile = 32 * 32 * 4;            // staging tile of one epilogue warp
__host__ __device__ constexpr int stage_bytes(int parts) { return parts * (kAPart + kBPart); }
__host__ __device__ constexpr int stages(int parts) { return 4 * 2 / parts; }
__host__ __device__ constexpr int smem_bytes(int parts) {
	return stages(parts) * stage_bytes(parts) + kEpiWarps * kEpiTile + 1024;
}

struct Item {
	int mt, nt, split, kb0, kb1;
};
// Item t: tiles in groups of kGroupM row tiles, all splits of a tile together.
__device__ __forceinline__ Item item_at(int t, const Product& p) {
	Item it;
	it.split = t % p.splits;
	const int tile = t / p.splits;
	const int group = tile / (kGroupM * p.tiles_n), first = group * kGroupM, size = min(p.tiles_m - first, kGroupM);
	const int in = tile - group * kGroupM * p.tiles_n;
	it.mt = first + in % size;
	it.nt = in / size;
	it.kb0 = it.split * p.split_kb;
	it.kb1 = min(p.kb, it.kb0 + p.split_kb);
	return it;
}

constexpr float kLog2e = 1.44269504088896341f;

template <int kParts, bool kMnA, bool kMnB, int kEpi>
__global__ void __launch_bounds__(kThreads, 1) split16_kernel(const __grid_constant__ CUtensorMap tm_a,
		const __grid_constant__ CUtensorMap tm_b, const __grid_constant__ Product p) {
	constexpr int kStages = stages(kParts), kStageBytes = stage_bytes(kParts);
	extern __shared__ uint8_t smem_raw[];
	uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
	__shared__ __align__(8) uint64_t full_bar[kStages], empty_bar[kStages], accf_bar[2], acce_bar[2], drain_bar;
	__shared__ uint32_t tmem_base_sh;
	__shared__ int abort_sh;
	const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
	if (threadIdx.x == 0) {
		for (int s = 0; s < kStages; ++s) {
			mbar_init(smem_u32(&full_bar[s]), 1);
			mbar_init(smem_u32(&empty_bar[s]), 1);
		}
		for (int b = 0; b < 2; ++b) {
			mbar_init(smem_u32(&accf_bar[b]), 1);
			mbar_init(smem_u32(&acce_bar[b]), kEpiWarps);
		}
		mbar_init(smem_u32(&drain_bar), 1);
		abort_sh = 0;
		fence_mbar_init();
		tma_prefetch_desc(&tm_a);
		tma_prefetch_desc(&tm_b);
	}
	if (warp == 1) {
		tmem_alloc(smem_u32(&tmem_base_sh), 2 * kBN);
		tmem_relinquish();
	}
	tc_fence_before();
	__syncthreads();
	tc_fence_after();
	chain_wait();
	const uint32_t tmem_base = tmem_base_sh;
	volatile int* abort_flag = &abort_sh;
	const int items = p.tiles_m * p.tiles_n * p.splits;
	static_assert(128 * 56 + 32 * kEpiWarps * 224 <= kThreads * 168, "registers handed over");

	if (warp < 4) {
		asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
		if (warp == 0 && lane == 0) {
			// ------------------------------ TMA producer ------------------------------
			int stage = 0;
			uint32_t phase = 0;
			bool ok = true, wrapped = false;
			for (int t = blockIdx.x; ok && t < items; t += gridDim.x) {
				const Item it = item_at(t, p);
				for (int kb = it.kb0; kb < it.kb1; ++kb) {
					if (!mbar_wait(smem_u32(&empty_bar[stage]), phase ^ 1, p.err, kDevTimeoutEmpty, abort_flag)) {
						ok = false;
						break;
					}
					const uint32_t fb = smem_u32(&full_bar[stage]);
					mbar_arrive_expect_tx(fb, kStageBytes);
					const uint32_t base = smem_u32(smem + stage * kStageBytes);
#pragma unroll
					for (int s = 0; s < kParts; ++s) {
						// K-major: half a block's 128-byte rows (32 of its 64 columns); MN-major: 32 of a block
						// row's 128 rows, 64 columns per chunk. Coordinates count 4-byte units.
						if (kMnA)
							tma_load_5d(base + s * kAPart, &tm_a, fb, 0, (kb & 3) * kBK, s, it.mt * (kBM / kCols), kb >> 2);
						else
							tma_load_2d(base + s * kAPart, &tm_a, fb, (kb & 1) * (kBK / 2),
								((it.mt * p.a_kw + (kb >> 1)) * 2 + s) * kRows);
						const uint32_t bb = base + kParts * kAPart + s * kBPart;
						if (kMnB) {
							tma_load_5d(bb, &tm_b, fb, 0, (kb & 3) * kBK, s, it.nt * (kBN / kCols), kb >> 2);
						} else {
#pragma unroll
							for (int q = 0; q < 2; ++q)
								tma_load_2d(bb + q * (kBPart / 2), &tm_b, fb, (kb & 1) * (kBK / 2),
									(((it.nt * 2 + q) * p.b_kw + (kb >> 1)) * 2 + s) * kRows);
						}
					}
					if (++stage == kStages) {
						stage = 0;
						phase ^= 1;
						wrapped = true;
					}
				}
			}
			// every issued copy has landed before the CTA can exit, on the way out of a wait that gave up too: the
			// last one into each stage, those before `stage` in this round through the stages and the rest in the last
			for (int s = 0; s < kStages; ++s)
				if (s < stage || wrapped)
					mbar_wait(smem_u32(&full_bar[s]), s < stage ? phase : phase ^ 1, p.err, kDevTimeoutDrain, nullptr);
		} else if (warp == 1) {
			// --------------------- MMA issuer (the whole warp; one elected lane issues) ---------------------
			constexpr uint32_t idesc = idesc_f16(kBM, kBN) | (kMnA ? kIdescAMajorMN : 0u) | (kMnB ? kIdescBMajorMN : 0u);
			int stage = 0;
			uint32_t phase = 0;
			int v = 0;                                     // chunks so far: accumulator v & 1
			bool ok = true;
			for (int t = blockIdx.x; ok && t < items; t += gridDim.x) {
				const Item it = item_at(t, p);
				for (int c0 = it.kb0; ok && c0 < it.kb1; c0 += kChunkKb, ++v) {
					if (!mbar_wait_warp(smem_u32(&acce_bar[v & 1]), ((v >> 1) & 1) ^ 1, p.err, kDevTimeoutAccumFree, abort_flag)) {
						ok = false;
						break;
					}
					tc_fence_after();
					const uint32_t d = tmem_base + (v & 1) * kBN;
					const int c1 = min(it.kb1, c0 + kChunkKb);
					for (int kb = c0; kb < c1; ++kb) {
						if (!mbar_wait_warp(smem_u32(&full_bar[stage]), phase, p.err, kDevTimeoutFull, abort_flag)) {
							ok = false;
							break;
						}
						tc_fence_after();
						const uint32_t a0 = smem_u32(smem + stage * kStageBytes), b0 = a0 + kParts * kAPart;
	#pragma unroll
						for (int kk = 0; kk < kBK / 16; ++kk) {
							// 16 deep: 32 bytes along a K-major row, or 16 rows of 128 bytes
							auto desc = [&](bool mn, uint32_t addr) {
								return mn ? smem_desc_mn_sw128(addr + kk * 2048, kBK * 128) : smem_desc_k_sw64(addr + kk * 32);
							};
							const uint64_t a_hi = desc(kMnA, a0), b_hi = desc(kMnB, b0);
							const uint32_t more = (kb > c0 || kk > 0) ? 1u : 0u;
							if (kParts == 2) {
								const uint64_t a_lo = desc(kMnA, a0 + kAPart), b_lo = desc(kMnB, b0 + kBPart);
								mma_f16_elect(d, a_lo, b_hi, idesc, more);
								mma_f16_elect(d, a_hi, b_lo, idesc, 1u);
								mma_f16_elect(d, a_hi, b_hi, idesc, 1u);
							} else {
								mma_f16_elect(d, a_hi, b_hi, idesc, more);
							}
						}
						mma_commit_elect(smem_u32(&empty_bar[stage]));
						if (++stage == kStages) {
							stage = 0;
							phase ^= 1;
						}
					}
					if (ok) mma_commit_elect(smem_u32(&accf_bar[v & 1]));
				}
			}
			// and every issued MMA has finished before the stages and tensor memory are released
			mma_commit_elect(smem_u32(&drain_bar));
			mbar_wait_warp(smem_u32(&drain_bar), 0, p.err, kDevTimeoutDrain, nullptr);
		}
	} else {
		asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
		// ---------------------------------- epilogue ----------------------------------
		const int quad = warp & 3, half = (warp - 4) >> 2;   // TMEM lanes and columns of this warp
		const int row = quad * 32 + lane;
		float* stage = reinterpret_cast<float*>(smem + (size_t)kStages * kStageBytes + (warp - 4) * kEpiTile);
		float4* st4 = reinterpret_cast<float4*>(stage);
		const bool vec_ok = kEpi == kStore && p.ldc % 4 == 0 && p.slab % 4 == 0 && (reinterpret_cast<uintptr_t>(p.C) & 15) == 0;
		int v = 0;
		bool ok = true;
		for (int t = blockIdx.x; ok && t < items; t += gridDim.x) {
			const Item it = item_at(t, p);
			float2 acc[kBN / 4];                           // this thread's row, 128 columns in pairs
#pragma unroll
			for (int j = 0; j < kBN / 4; ++j) acc[j] = make_float2(0.0f, 0.0f);
			const int nb = min(it.nt * 2 + half, p.b_last);      // (past the last block there are zeros, whatever their scale)
			for (int c0 = it.kb0; c0 < it.kb1; c0 += kChunkKb, ++v) {
				// the chunk's terms are scaled back by 2^e: in one factor, or two where the exponent does not fit one.
				// (The loads' latency passes in the wait.)
				const int kc = c0 / kChunkKb;
				const int e = -p.sa[kMnA ? kc * p.a_sw + it.mt : it.mt * p.a_sw + kc] -
					p.sb[kMnB ? kc * p.b_sw + nb : nb * p.b_sw + kc];
				const int e1 = max(-126, min(127, e));
				const float2 back = make_float2(exp2_int(e1), exp2_int(e1));
				if (!mbar_wait_warp(smem_u32(&accf_bar[v & 1]), (v >> 1) & 1, p.err, kDevTimeoutAccum, abort_flag)) {
					ok = false;
					break;
				}
				tc_fence_after();
				const uint32_t src = tmem_base + ((uint32_t)(quad * 32) << 16) + (v & 1) * kBN + half * (kBN / 2);
#pragma unroll
				for (int c = 0; c < kBN / 64; ++c) {
					uint32_t r[32];
					tmem_ld_32x32b_x32(src + c * 32, r);
					tmem_wait_ld();
					if (e != e1) {                             // operands beyond 2^110 or below 2^-95: warp-uniform
						const float more = exp2_int(e - e1);
#pragma unroll
						for (int j = 0; j < 32; ++j) r[j] = __float_as_uint(__uint_as_float(r[j]) * more);
					}
#pragma unroll
					for (int j = 0; j < 16; ++j)
						acc[c * 16 + j] = fma2_rn(make_float2(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1])), back, acc[c * 16 + j]);
				}
				tc_fence_before();
				__syncwarp();
				if (lane == 0) mbar_arrive(smem_u32(&acce_bar[v & 1]));
			}
			if (!ok) break;
			const int gm = it.mt * kBM + row, n0 = it.nt * kBN + half * (kBN / 2);
			// the warp's 32 x 32 values (row per lane) to rows dst + r * ld, as 128-byte row segments: through the
			// staging tile, element (r, c) at float4 r * 8 + (c / 4 ^ r % 8), without bank conflicts either way
			auto stage_rows = [&](float* dst, long long ld, int rows, int c, bool add) {
#pragma unroll
				for (int g = 0; g < 8; ++g)
					st4[lane * 8 + (g ^ (lane & 7))] =
						make_float4(acc[c * 16 + 2 * g].x, acc[c * 16 + 2 * g].y, acc[c * 16 + 2 * g + 1].x, acc[c * 16 + 2 * g + 1].y);
				__syncwarp();
				const int g = lane & 7;
#pragma unroll
				for (int k = 0; k < 8; ++k) {
					const int rr = 4 * k + (lane >> 3);
					float4 o = st4[rr * 8 + (g ^ (rr & 7))];
					if (rr < rows) {
						float4* d4 = reinterpret_cast<float4*>(dst + rr * ld) + g;
						if (add) {
							const float4 old = *d4;
							o = make_float4(old.x + o.x, old.y + o.y, old.z + o.z, old.w + o.w);
						}
						*d4 = o;
					}
				}
				__syncwarp();
			};
			const int warp_row = it.mt * kBM + quad * 32, rows_here = max(0, min(32, p.M - warp_row));
			if (kEpi == kStore) {
				float* C = p.C + it.split * p.slab;
#pragma unroll
				for (int c = 0; c < kBN / 64; ++c) {
					const int gn = n0 + c * 32;
					if (gn >= p.N) break;                  // warp-uniform
					if (vec_ok && gn + 32 <= p.N) {
						stage_rows(C + (long long)warp_row * p.ldc + gn, p.ldc, rows_here, c, p.accumulate != 0);
					} else if (gm < p.M) {
						float* dst = C + (long long)gm * p.ldc + gn;
#pragma unroll
						for (int j = 0; j < 32; ++j) {
							const float a = j & 1 ? acc[c * 16 + j / 2].y : acc[c * 16 + j / 2].x;
							if (gn + j < p.N) dst[j] = p.accumulate ? dst[j] + a : a;
						}
					}
				}
			} else {
				// l = acc + bias: the biases of the warp's 128 columns through its staging tile (one coalesced
				// load, then broadcasts)
				if (p.bias) {
					float4 b;
					b.x = n0 + 4 * lane < p.N ? p.bias[n0 + 4 * lane] : 0.0f;
					b.y = n0 + 4 * lane + 1 < p.N ? p.bias[n0 + 4 * lane + 1] : 0.0f;
					b.z = n0 + 4 * lane + 2 < p.N ? p.bias[n0 + 4 * lane + 2] : 0.0f;
					b.w = n0 + 4 * lane + 3 < p.N ? p.bias[n0 + 4 * lane + 3] : 0.0f;
					st4[lane] = b;
					__syncwarp();
#pragma unroll
					for (int j = 0; j < kBN / 8; ++j) {
						const float4 bj = st4[j];
						acc[2 * j] = add2_rn(acc[2 * j], make_float2(bj.x, bj.y));
						acc[2 * j + 1] = add2_rn(acc[2 * j + 1], make_float2(bj.z, bj.w));
					}
					__syncwarp();                          // read before the tile is written again
				}
				const long long slot = (long long)(it.nt * 2 + half) * (p.tiles_m * kBM) + gm;
				if (p.part_sum) {
					float total = 0.0f;
#pragma unroll
					for (int j = 0; j < kBN / 4; ++j) {
						if (n0 + 2 * j < p.N) total += acc[j].x;
						if (n0 + 2 * j + 1 < p.N) total += acc[j].y;
					}
					p.part_sum[slot] = total;
				}
				const int64_t target = gm < p.M ? p.targets[gm] : -1;
				const int tj = target >= n0 && target < n0 + kBN / 2 && target < p.N ? (int)(target - n0) : -1;
				if (__any_sync(0xffffffffu, tj >= 0)) {
					float at = 0.0f;
#pragma unroll
					for (int j = 0; j < kBN / 4; ++j) {
						if (tj == 2 * j) at = acc[j].x;
						if (tj == 2 * j + 1) at = acc[j].y;
					}
					if (tj >= 0) p.target_logit[gm] = at;
				}
				if (n0 + kBN / 2 > p.N) {                      // columns past N: no part of the softmax
#pragma unroll
					for (int j = 0; j < kBN / 4; ++j) {
						if (n0 + 2 * j >= p.N) acc[j].x = -INFINITY;
						if (n0 + 2 * j + 1 >= p.N) acc[j].y = -INFINITY;
					}
				}
				float2 top2 = make_float2(-INFINITY, -INFINITY);
#pragma unroll
				for (int j = 0; j < kBN / 4; ++j) {
					top2.x = fmaxf(top2.x, acc[j].x);
					top2.y = fmaxf(top2.y, acc[j].y);
				}
				const float top = fmaxf(top2.x, top2.y);
				// all -inf: an empty part (top stands in as 0, every term is 0); NaN and +inf give a NaN sum
				const float base = top == -INFINITY ? 0.0f : top;
				float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
				for (int j = 0; j < kBN / 4; ++j) {
					const float2 a = mul2_rn(add2_rn(acc[j], make_float2(-base, -base)), make_float2(kLog2e, kLog2e));
					sum = add2_rn(sum, make_float2(exp2_hw(a.x), exp2_hw(a.y)));
				}
				p.part[slot] = make_float2(top, sum.x + sum.y);
				if (kEpi == kLogits) {
#pragma unroll
					for (int c = 0; c < kBN / 64; ++c) {
						const int gn = n0 + c * 32;
						if (gn >= p.blocks_kw * kCols) break;
						stage_rows(p.blocks + ((long long)it.mt * p.blocks_kw + gn / kCols) * (kRows * kCols) + quad * 32 * kCols +
							gn % kCols, kCols, 32, c, false);
					}
				}
			}
		}
	}
	tc_fence_before();
	__syncthreads();
	if (warp == 1) {
		__syncwarp();
		tc_fence_after();
		tmem_dealloc(tmem_base, 2 * kBN);
	}
}

// c (+)= sum over slabs, in order; four floats per thread where aligned.
__global__ void __launch_bounds__(256) sum_slabs_kernel(const float* slabs, int splits, long long n,
		float* c, int accumulate, int vec) {
	chain_wait();
	const long long step = gridDim.x * 256LL;
	long long i = blockIdx.x * 256LL + threadIdx.x;
	if (vec) {
		for (; i < n / 4; i += step) {
			float4 a = reinterpret_cast<const float4*>(slabs)[i];
#pragma unroll 4
			for (int k = 1; k < splits; ++k) {
				const float4 b = reinterpret_cast<const float4*>(slabs + k * n)[i];
				a = make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w);
			}
			float4* d = reinterpret_cast<float4*>(c) + i;
			if (accumulate) {
				const float4 o = *d;
				a = make_float4(o.x + a.x, o.y + a.y, o.z + a.z, o.w + a.w);
			}
			*d = a;
		}
	} else {
		for (; i < n; i += step) {
			float a = slabs[i];
			for (int k = 1; k < splits; ++k) a += slabs[k * n + i];
			c[i] = accumulate ? c[i] + a : a;
		}
	}
}

// Tensor map of a pack read K-major: its 128-byte rows as 32 4-byte units, half a row per box.
nnb_status map_k(CUtensorMap* map, const Pack& a, long long row_blocks) {
	const long long rows = row_blocks * a.kw() * 2 * kRows;
	if (rows > INT32_MAX) return fail(NNB_ERR_UNSUPPORTED, "split product: operand too large");
	return encode_tiled_2d(map, a.buf, kCols / 2, (uint64_t)rows, kCols * 2, kBK / 2, kRows, CU_TENSOR_MAP_SWIZZLE_64B);
}
// The same read MN-major: (64 columns, 128 rows, part, packed column, row block), boxes of 32 rows and
// `chunks` packed columns.
nnb_status map_mn(CUtensorMap* map, const Pack& a, int chunks) {
	const uint64_t kw = (uint64_t)a.kw();
	const uint64_t dims[5] = {kCols / 2, kRows, 2, kw, (uint64_t)a.row_blocks()};
	const uint64_t strides[4] = {kCols * 2, kPartBytes, kBlockBytes, kw * kBlockBytes};
	const uint32_t box[5] = {kCols / 2, kBK, 1, (uint32_t)chunks, 1};
	return encode_tiled_nd(map, a.buf, 5, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <int kParts, bool kMnA, bool kMnB, int kEpi>
nnb_status launch(cudaStream_t s, const DeviceState* dev, const Product& p, const CUtensorMap& ta, const CUtensorMap& tb) {
	auto kernel = split16_kernel<kParts, kMnA, kMnB, kEpi>;
	static std::atomic<bool> ready[64];                // the attribute holds for the device once set
	if (!ready[dev->device & 63].load(std::memory_order_relaxed)) {
		NNB_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes(kParts)));
		ready[dev->device & 63].store(true, std::memory_order_relaxed);
	}
	const long long items = (long long)p.tiles_m * p.tiles_n * p.splits;
	{
		TraceScope ts(s, kTraceGemm);
		NNB_CUDA_TRY(launch_chained(kernel, (unsigned)std::min<long long>(items, dev->sm_count), kThreads, smem_bytes(kParts), s,
			ta, tb, p));
	}
	return NNB_OK;
}

template <int kParts>
nnb_status dispatch(cudaStream_t s, const DeviceState* dev, int epilogue, bool mn_a, bool mn_b, const Product& p,
		const CUtensorMap& ta, const CUtensorMap& tb) {
	if (epilogue == kStats && !mn_a && !mn_b) return launch<kParts, false, false, kStats>(s, dev, p, ta, tb);
	if (epilogue == kLogits && !mn_a && !mn_b) return launch<kParts, false, false, kLogits>(s, dev, p, ta, tb);
	if (epilogue == kStore && !mn_a && mn_b) return launch<kParts, false, true, kStore>(s, dev, p, ta, tb);
	if (epilogue == kStore && mn_a && mn_b) return launch<kParts, true, true, kStore>(s, dev, p, ta, tb);
	return fail(NNB_ERR_UNSUPPORTED, "split product: form not built");
}

}  // namespace

nnb_status pack(cudaStream_t s, const PackJob* jobs, int count, int parts) {
	PackJobs k;
	k.parts = parts;
	long long ctas[2] = {0, 0};
	for (int i = 0; i < count; ++i) {
		const PackJob& j = jobs[i];
		PackWork& w = k.job[i];
		w.x = j.x; w.rows = j.rows; w.cols = j.cols; w.live = j.live;
		w.kw = (int)((j.cols + kCols - 1) / kCols); w.scale_cols = (int)((j.cols + kRows - 1) / kRows);
		w.out = static_cast<unsigned char*>(j.buf); w.shift = j.shift; w.bad = j.bad; w.per_row = j.per_row;
		w.vec = j.cols % 4 == 0 && (reinterpret_cast<uintptr_t>(j.x) & 15) == 0;
		ctas[i] = j.row_blocks * w.scale_cols;
	}
	if (ctas[0] + ctas[1] > INT32_MAX) return fail(NNB_ERR_UNSUPPORTED, "split product: operand too large");
	k.first = (int)ctas[0];
	{
		TraceScope ts(s, kTracePack);
		NNB_CUDA_TRY(launch_chained(pack_kernel, (unsigned)(ctas[0] + ctas[1]), 256, 0, s, k));
	}
	return NNB_OK;
}

// Chunks of 128 terms in a depth of K.
static long long chunks_of(long long K) { return (K + kBK * kChunkKb - 1) / (kBK * kChunkKb); }

int split_count(long long K, int want) {
	const long long chunks = chunks_of(K), per = (chunks + want - 1) / want;
	return (int)((chunks + per - 1) / per);
}

int choose_splits(long long M, long long N, long long K) {
	// Items are worked through in waves of one per SM, so n pieces of the depth take
	// ceil(tiles n / 148) / n of a tile's time, K times 21 ns (3.1 TFLOP/s per SM); writing and reading back the
	// slabs adds tiles n times 44 ns (256 KB each at 6 TB/s). The fewest pieces of about the least cost, each of
	// at least 512 terms.
	const long long tiles = (M + kBM - 1) / kBM * ((N + kBN - 1) / kBN), chunks = chunks_of(K);
	int best = 1;
	double best_cost = 0.0;
	for (int want = 1; want <= (int)std::min<long long>(16, std::max<long long>(1, chunks / 4)); ++want) {
		const int n = split_count(K, want);
		const double waves = (double)((tiles * n + 147) / 148) * ((chunks + n - 1) / n) / chunks;
		const double cost = waves + (n > 1 ? 44.0 / 21.0 * n * tiles / K : 0.0);
		if (n == 1 || cost < 0.95 * best_cost) {
			best = n;
			best_cost = cost;
		}
	}
	return best;
}

nnb_status run(cudaStream_t s, Product p, int epilogue, int parts, const Pack& a, bool mn_a, const Pack& b, bool mn_b,
		long long M, long long N, long long K) {
	DeviceState* dev = nullptr;
	NNB_TRY(device_state(&dev));
	p.M = (int)M;
	p.N = (int)N;
	p.kb = (int)((K + kBK - 1) / kBK);
	p.tiles_m = (int)((M + kBM - 1) / kBM);
	p.tiles_n = (int)((N + kBN - 1) / kBN);
	if ((long long)p.tiles_m * p.tiles_n * p.splits > INT32_MAX) return fail(NNB_ERR_UNSUPPORTED, "split product: too many tiles");
	// whole chunks per split, and no empty split
	p.split_kb = ((p.kb + p.splits - 1) / p.splits + kChunkKb - 1) / kChunkKb * kChunkKb;
	if ((p.kb + p.split_kb - 1) / p.split_kb != p.splits) return fail(NNB_ERR_INVALID, "split product: empty depth split");
	p.a_kw = (int)a.kw();
	p.b_kw = (int)b.kw();
	p.sa = a.shift;
	p.sb = b.shift;
	p.a_sw = (int)a.scale_cols();
	p.b_sw = (int)b.scale_cols();
	p.b_last = (int)(mn_b ? b.scale_cols() : b.row_blocks()) - 1;
	p.err = dev->error_word;
	CUtensorMap ta, tb;
	if (mn_a) NNB_TRY(map_mn(&ta, a, kBM / kCols));
	else NNB_TRY(map_k(&ta, a, a.row_blocks()));
	if (mn_b) NNB_TRY(map_mn(&tb, b, kBN / kCols));
	else NNB_TRY(map_k(&tb, b, (b.row_blocks() + 1) / 2 * 2));      // a 256-row tile reads whole pairs of blocks
	return parts == 2 ? dispatch<2>(s, dev, epilogue, mn_a, mn_b, p, ta, tb) : dispatch<1>(s, dev, epilogue, mn_a, mn_b, p, ta, tb);
}

nnb_status sum_slabs(cudaStream_t s, const float* slabs, int splits, long long n, float* c, int accumulate) {
	const bool vec = n % 4 == 0 && ((reinterpret_cast<uintptr_t>(slabs) | reinterpret_cast<uintptr_t>(c)) & 15) == 0;
	{
		TraceScope ts(s, kTraceAux);
		NNB_CUDA_TRY(launch_chained(sum_slabs_kernel, grid_for(vec ? n / 4 : n, 256), 256, 0, s, slabs, splits, n, c, accumulate,
			(int)vec));
	}
	return NNB_OK;
}

}  // namespace split16
}  // namespace nnb
