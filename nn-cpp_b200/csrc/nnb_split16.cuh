// nnb_split16.cuh -- products of fp32 matrices on the 16-bit tensor-core path: every block of 128 x 128 of an
// operand is scaled by a power of two and written as two fp16 parts, x s ~= hi + lo, and
// C = Ahi Bhi + Ahi Blo + Alo Bhi in fp32.
//
// fp16 has the 11 significant bits of TF32 and twice its MMA rate, so the split carries the 22 bits of
// 3xTF32 at half the time; what fp16 lacks is range. A block's scale puts its largest magnitude into
// (2^14, 2^15]: elements down to 2^-17 of it keep their 22 bits (the low part's last bit is 2^-24), smaller
// ones an absolute error of 2^-39 of the largest. That is fp32 grade next to the sums such elements enter; it
// is not for operands whose tiny elements count alone beside large ones, and the general GEMM (gemm.cu) stays
// with TF32. With one part (TF32 mode) the 11 bits are TF32's own.
//
// The scales are per block and not per matrix so that one large value costs no bits outside its block, and so
// that the pack finds them itself: a CTA holds the block in registers, takes its maximum and scales it, and
// the matrix is read once. Blocks are 128 both ways because an accumulator holds 128 terms of the depth and
// an epilogue warp 128 columns of C: whichever way the packs are read, the scales of the two operands are one
// number for a warp and a chunk, and scaling back is part of the addition that joins the chunk to the sum.
//
// Precision of the sums: the tensor core adds with truncation, a bias that grows with the number of
// additions (measured on the TF32 path: 1e-5 of a sum of 1024 terms). So an accumulator holds kChunkKb
// k-blocks (128 terms, 24 additions) and is then added, rounded to nearest, into registers.
//
// Packed layout: blocks of 128 rows x 64 columns, hi part then lo part (16 KB each, rows of 128 bytes),
// block (rb, c) at index rb * kw + c. The same pack is read K-major (its rows are C's rows or columns) or
// MN-major (its rows are the depth).
#pragma once

#include <cuda_fp16.h>

#include "nnb_internal.h"
#include "nnb_ptx.cuh"

namespace nnb {
namespace split16 {

constexpr int kRows = 128, kCols = 64;           // of a packed block
constexpr int kPartBytes = kRows * kCols * 2;
constexpr int kBlockBytes = 2 * kPartBytes;      // also 128 x 64 floats
constexpr int kBM = 128, kBN = 256;              // tile of C
constexpr int kBK = 32;                          // depth per pipeline stage: rows of 64 bytes
constexpr int kChunkKb = 4;                      // k-blocks per accumulator
constexpr int kEpiWarps = 8;                     // two per TMEM lane quarter, 128 columns each
constexpr int kThreads = 128 + 32 * kEpiWarps;   // producer, MMA issuer, two idle warps, epilogue

// A packed matrix of `rows` x `cols`, rows padded to whole blocks of 128 (256 for a K-major B), columns to 64.
struct Pack {
	const void* buf = nullptr;
	const int* shift = nullptr;                  // [row blocks][scale_cols()]: the blocks' scales are 2^shift
	long long rows = 0, cols = 0;
	long long row_blocks() const { return (rows + kRows - 1) / kRows; }
	long long kw() const { return (cols + kCols - 1) / kCols; }
	long long scale_cols() const { return (cols + kRows - 1) / kRows; }
};
// Blocks of rows, padded to an even number, and the bytes of a pack with them and of its scales.
inline long long even_blocks(long long rows) { return (rows + 2 * kRows - 1) / (2 * kRows) * 2; }
inline size_t shift_bytes(long long rows, long long cols) {
	return (size_t)even_blocks(rows) * ((cols + kRows - 1) / kRows) * sizeof(int);
}
inline size_t pack_bytes(long long rows, long long cols) {
	return (size_t)even_blocks(rows) * ((cols + kCols - 1) / kCols) * kBlockBytes;
}

// The rows that count: those whose target is a token of the vocabulary and not `ignore` (targets null: all rows).
// What the others hold is packed as zeros, so that it touches nothing.
struct LiveRows {
	const int64_t* targets = nullptr;
	int64_t ignore = 0, V = 0;
	__device__ __forceinline__ bool operator()(long long r) const {
		if (!targets) return true;
		const int64_t t = targets[r];
		return t != ignore && t >= 0 && t < V;
	}
};
// 2^k, -126 <= k <= 127.
__device__ __forceinline__ float exp2_int(int k) { return __int_as_float((k + 127) << 23); }
// The shift that puts a largest magnitude of the given bit pattern into (2^14, 2^15]; 0 for a block of zeros. At
// most 126, which exp2_int takes (below 2^-112 the block keeps fewer bits).
__device__ __forceinline__ int block_shift(unsigned top) {
	return top == 0 ? 0 : min(126, 15 - ((int)((top + 0x7fffffu) >> 23) - 127));
}

enum Epilogue : int {
	kStore = 0,     // C (+)= acc, row-major
	kStats = 1,     // softmax statistics of acc + bias per row and 128 columns
	kLogits = 2     // the same, and acc + bias into 128 x 64 float blocks
};

struct Product {
	int M = 0, N = 0;
	int kb = 0;                       // k-blocks of 32
	int tiles_m = 0, tiles_n = 0;
	int splits = 1, split_kb = 0;     // depth splits (kStore: split i writes slab i of C), k-blocks each
	int a_kw = 0, b_kw = 0;           // packed columns of the operands
	const int *sa = nullptr, *sb = nullptr;   // their blocks' shifts, scale_cols() to a row of blocks
	int a_sw = 0, b_sw = 0;
	int b_last = 0;                   // B's last block of 128 along C's columns
	// kStore
	float* C = nullptr;
	long long ldc = 0, slab = 0;
	int accumulate = 0;
	// kStats, kLogits
	const float* bias = nullptr;
	const int64_t* targets = nullptr; // per row of C
	float2* part = nullptr;           // [2 tiles_n][rows of whole tiles]: max, sum of exp(l - max)
	float* part_sum = nullptr;        // the same: sum of l (null: not wanted)
	float* target_logit = nullptr;    // per row of C
	float* blocks = nullptr;          // kLogits: [tiles_m][blocks_kw][128][64]
	int blocks_kw = 0;
	int* err = nullptr;
};

// A matrix to pack: x [rows x cols] (row-major, dense) into buf, rows padded with zeros to `row_blocks` blocks,
// and the blocks' shifts; rows that do not count become zeros, and values of others that are not finite become
// zero and set bad[row], or bad[0] (per_row 0; the caller has zeroed them).
struct PackJob {
	const float* x;
	long long rows, cols, row_blocks;
	void* buf;
	int* shift;
	int* bad;
	int per_row;
	LiveRows live;
};
// One or two of them in one launch.
nnb_status pack(cudaStream_t s, const PackJob* jobs, int count, int parts);

// C = A B^T with A = a (K-major: rows of a) or a^T (mn_a: columns of a), B likewise; p's sizes, operands'
// widths and tile counts are filled in here. parts: 2 or 1.
nnb_status run(cudaStream_t s, Product p, int epilogue, int parts, const Pack& a, bool mn_a, const Pack& b, bool mn_b,
		long long M, long long N, long long K);
// Depth splits for an M x N product of depth K; depends on the sizes only.
int choose_splits(long long M, long long N, long long K);
// The splits, at most `want`, that cut a depth of K into whole chunks with none empty (Product::splits).
int split_count(long long K, int want);
// c (+)= sum over `splits` slabs of n floats, in order.
nnb_status sum_slabs(cudaStream_t s, const float* slabs, int splits, long long n, float* c, int accumulate);

}  // namespace split16
}  // namespace nnb
