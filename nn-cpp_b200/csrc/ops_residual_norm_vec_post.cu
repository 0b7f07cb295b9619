// ops_residual_norm_vec_post.cu -- instances of the residual norm's backward: rows that move as float4,
// with a norm after the block.
#include "nnb_residual_norm.cuh"

namespace nnb {
namespace resnorm {

nnb_status bwd_vec_post(cudaStream_t s, const Grad& p, long long groups) {
	if (p.layer)
		return p.gate ? dispatch_bwd<4, true, true, true>(s, p, groups) : dispatch_bwd<4, true, true, false>(s, p, groups);
	return p.gate ? dispatch_bwd<4, false, true, true>(s, p, groups) : dispatch_bwd<4, false, true, false>(s, p, groups);
}

}  // namespace resnorm
}  // namespace nnb
