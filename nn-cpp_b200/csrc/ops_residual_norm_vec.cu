// ops_residual_norm_vec.cu -- instances of the residual norm's backward: rows that move as float4,
// without a norm after the block.
#include "nnb_residual_norm.cuh"

namespace nnb {
namespace resnorm {

nnb_status bwd_vec(cudaStream_t s, const Grad& p, long long groups) {
	if (p.layer)
		return p.gate ? dispatch_bwd<4, true, false, true>(s, p, groups) : dispatch_bwd<4, true, false, false>(s, p, groups);
	return p.gate ? dispatch_bwd<4, false, false, true>(s, p, groups) : dispatch_bwd<4, false, false, false>(s, p, groups);
}

}  // namespace resnorm
}  // namespace nnb
